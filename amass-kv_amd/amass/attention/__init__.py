"""Stage B -- sparse paged decode attention over the Stage-A-selected pages.

  sparse_paged_decode_batched(q, kv_cache, block_table, seq_lens, st, out, vsource)
  dense_paged_decode(q, kv_cache, block_table, seq_lens, st, out, scale=...)
  ResidentVSource / VSource      the fast / mem-v V-source seam
  ensure_stage_b_buffers         split-K partial buffers (allocated once)

A chunk of new tokens (prompts, drafted tokens), before and beside the decode steps:

  extend_block_tables(block_table, seq_lens, query_start, free, top, slots, positions, ...)
  rope_paged_write(q, k, v, positions, table, kv_cache, slots, q_out)
  paged_chunk_attention(q, kv_cache, block_table, seq_lens, query_start, out, ...)
  free_blocks, release_blocks, rope_table

The same over a cache in 8 bits with a scale for each block, half and kv head:

  quant_cache(num_blocks, page, n_kv, d, ...)          codes and scales
  quant_paged_write(k, v, codes, scales, slots, ...)   with rotary positions on request
  quant_chunk_attention(q, codes, scales, block_table, seq_lens, query_start, out, ...)
  quant_paged_read(codes, scales, src, kv_cache, dst)  blocks to a 16-bit cache
"""
from __future__ import annotations

from .chunk import chunk_scratch_bytes, paged_chunk_attention
from .decode import (SPLIT, ResidentVSource, VSource, _split_kv, dense_paged_decode,
                     ensure_stage_b_buffers, sparse_paged_decode_batched)
from .quant import (quant_cache, quant_chunk_attention, quant_paged_read, quant_paged_write,
                    quant_scratch_bytes)
from .rope import rope_frequencies, rope_paged_write, rope_table
from .slots import extend_block_tables, free_blocks, release_blocks

__all__ = ["sparse_paged_decode_batched", "dense_paged_decode", "ResidentVSource", "VSource",
           "ensure_stage_b_buffers", "SPLIT", "extend_block_tables", "free_blocks",
           "release_blocks", "rope_frequencies", "rope_table", "rope_paged_write",
           "paged_chunk_attention", "chunk_scratch_bytes", "quant_cache", "quant_paged_write",
           "quant_paged_read", "quant_chunk_attention", "quant_scratch_bytes"]
