"""Chunk attention on the GPU at its edges: batches that are none, values that leave the ordinary."""
import numpy as np
import pytest
import torch

from amass.attention import chunk_scratch_bytes, paged_chunk_attention
from helpers import announce
from test_gpu_chunk import DEV, Case

pytestmark = pytest.mark.gpu


def test_starts_that_do_not_ascend_leave_other_memory_alone():
    """Requests whose rows together are several times the batch's, and a scratch that holds records of
    row tiles behind `out`: the rows there stay, and the scratch serves the next call."""
    announce("chunk attention: starts that do not ascend, a scratch of records")
    T, R = 1024, 5
    c = Case(new=[T], lens=[4000], n_kv=8)
    q, kv, table, _, _ = c.dev()
    wide = torch.full((2 * T, 32, 128), 7.0, dtype=c.dt, device=DEV)
    out = wide[:T]
    bad = dict(block_table=table.expand(R, -1).contiguous(),
               seq_lens=torch.full((R,), 4000, dtype=torch.int32, device=DEV),
               query_start=torch.tensor([0, T] * 3, dtype=torch.int32, device=DEV))
    need = chunk_scratch_bytes(q, kv, *bad.values(), out)
    # (request, row tile, parts, slot, first row, rows, tokens, 0) from byte 256 on, repeated
    record = torch.tensor([0, 0, 2, 0, T, T, 4000, 0], dtype=torch.int32)
    scratch = record.repeat(-(-need // 32) + 8).view(torch.uint8)[:need].to(DEV)
    paged_chunk_attention(q, kv, *bad.values(), out, scratch=scratch)
    torch.cuda.synchronize()
    assert (wide[T:] == 7.0).all()
    c = Case(new=[90, 3], lens=[3000, 900], n_kv=8)
    q, kv, table, lens, qs = c.dev()
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device=DEV)
    paged_chunk_attention(q, kv, table, lens, qs, out, lse=lse, scratch=scratch)
    c.check(out, lse)


@pytest.mark.parametrize("T,starts,rows", [(60, [0, 40, 20, 60], [*range(20), *range(40, 60)]),
                                           (12, [0, 9, 7, 12], [*range(7), *range(9, 12)])])
def test_rows_of_one_request_only_are_right_where_starts_do_not_ascend(T, starts, rows):
    announce(f"chunk attention: starts {starts}")
    c = Case(new=[T, 0, 0], lens=[150, 40, 230], n_kv=2)
    c.qs = torch.tensor(starts, dtype=torch.int32)
    c.check(*c.run(), rows=rows)
