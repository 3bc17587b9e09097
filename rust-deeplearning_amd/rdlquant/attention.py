"""ctypes binding of the operators for several sequences over one paged cache
in librdlquant.so (include/rdl_attention.h): page tables and slots of a step
(plan_dev), RoPE with the cache write (store_dev), attention over the paged
cache (attention_paged_dev) and over packed prompts (attention_packed_dev).

All of them take raw device pointers (ints), e.g. torch.Tensor.data_ptr(), and
a hipStream_t as int; nothing synchronises.  There is no CPU fallback.
"""
from __future__ import annotations

import ctypes as C

from . import _decl, _i32, _p, _sz, check, lib

DTYPE_F32 = 0  # RDL_DTYPE_F32
DTYPE_F16 = 1  # RDL_DTYPE_F16
PLAN_BAD_LENGTH, PLAN_TABLE_FULL, PLAN_NO_PAGES, PLAN_NO_ROWS = 1, 2, 4, 8


class KvPool(C.Structure):
    """rdl_kv_pool: a layer's paged K and V memory (strides in elements)."""
    _fields_ = [("k_dev", _p), ("v_dev", _p)] + \
               [(n, _i32) for n in ("dtype", "n_pages", "page_positions", "n_kv_heads", "head_dim")] + \
               [(n, C.c_int64) for n in ("page_stride", "head_stride", "position_stride")]


_decl("rdl_kv_plan_dev", _i32, _p, _p, _sz, _p, _sz, _sz, _p, _sz, _p, _p, _sz, _p, _p, _p, _p, _p)
_decl("rdl_kv_store_dev", _i32, C.POINTER(KvPool), _sz, _p, _sz, _p, _sz, _sz, _p, _sz, _p, _sz, _p, _p, _p, _p, _sz,
      _p)
_decl("rdl_attention_paged_dev", _i32, C.POINTER(KvPool), _p, _sz, _sz, _sz, _p, _p, _sz, _p, _sz, C.c_float, _p, _sz,
      _sz, _sz, _p)
_decl("rdl_attention_packed_dev", _i32, _p, _sz, _sz, _p, _sz, _p, _sz, _i32, _sz, _sz, _sz, _p, _sz, C.c_float, _p,
      _sz, _sz, _p)


def plan_dev(cached_ptr, new_rows_ptr, n_seq, free_pages_ptr, n_free, page_positions, tables_ptr, table_stride,
             row_start_ptr, kv_len_ptr, m, row_seq_ptr, positions_ptr, slots_ptr, summary_ptr, stream=0):
    """rdl_kv_plan_dev: page tables, row starts, positions and slots of a step
    from the lengths of its sequences (int32 arrays on the device)."""
    check(lib.rdl_kv_plan_dev(cached_ptr, new_rows_ptr, n_seq, free_pages_ptr, n_free, page_positions, tables_ptr,
                              table_stride, row_start_ptr, kv_len_ptr, m, row_seq_ptr, positions_ptr, slots_ptr,
                              summary_ptr, stream))


def store_dev(pool, m, q_ptr, q_stride, q_out_ptr, q_out_stride, n_heads, k_ptr, k_stride, v_ptr, v_stride,
              positions_ptr, slots_ptr, cos_ptr=0, sin_ptr=0, n_positions=0, stream=0):
    """rdl_kv_store_dev: RoPE of the q and k rows, k and v rows into the pool's
    slots (n_heads 0: no q; cos and sin 0: no RoPE)."""
    check(lib.rdl_kv_store_dev(C.byref(pool), m, q_ptr, q_stride, q_out_ptr, q_out_stride, n_heads, k_ptr, k_stride,
                               v_ptr, v_stride, positions_ptr, slots_ptr, cos_ptr or None, sin_ptr or None,
                               n_positions, stream))


def attention_paged_dev(pool, q_ptr, q_stride, n_heads, m, row_start_ptr, kv_len_ptr, n_seq, tables_ptr,
                        table_stride, scale, out_ptr, out_stride, max_rows=0, max_kv=0, stream=0):
    """rdl_attention_paged_dev: causal attention of a step's rows over the
    paged cache (max_rows, max_kv: what to expect, 0 unknown)."""
    check(lib.rdl_attention_paged_dev(C.byref(pool), q_ptr, q_stride, n_heads, m, row_start_ptr, kv_len_ptr, n_seq,
                                      tables_ptr, table_stride, scale, out_ptr, out_stride, max_rows, max_kv, stream))


def attention_packed_dev(q_ptr, q_stride, n_heads, k_ptr, k_stride, v_ptr, v_stride, kv_dtype, n_kv_heads, head_dim,
                         m, row_start_ptr, n_seq, scale, out_ptr, out_stride, max_rows=0, stream=0):
    """rdl_attention_packed_dev: causal attention of whole prompts packed one
    behind the other."""
    check(lib.rdl_attention_packed_dev(q_ptr, q_stride, n_heads, k_ptr, k_stride, v_ptr, v_stride, kv_dtype,
                                       n_kv_heads, head_dim, m, row_start_ptr, n_seq, scale, out_ptr, out_stride,
                                       max_rows, stream))
