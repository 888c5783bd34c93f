"""Attention over every visible key of the paged latent cache on B200, for a batch whose sequences share a prefix.

No counterpart in the reference, whose attention takes selected keys (sparse_flash_attention_triton.py:1295-1455); layouts,
lengths, statistics and checks are those of `sparse_flash_attention_triton`, with every visible key selected.
"""
import ctypes

import torch

from . import _cabi
from ._host import (current_stream, device_guard, dtype_code, int32_table, note_launch, one_device, packed, ptr, seq_tensor,
                    workspace)

_D, _D_ROPE = 512, 64
_STRUCT_SIZE = ctypes.sizeof(_cabi.DsaSpaParams)
_kernel = _cabi.KERNEL_AUTO


def set_kernel(kind):
    """"auto", "portable" (row by row) or "tensor" (tcgen05 path, error if not eligible)."""
    global _kernel
    _kernel = {"auto": _cabi.KERNEL_AUTO, "portable": _cabi.KERNEL_PORTABLE, "tensor": _cabi.KERNEL_TENSOR}[kind]


def shared_prefix_attention(
    query,
    key,
    scale_value: float = 1.0,
    block_table=None,
    actual_seq_lengths_query=None,
    actual_seq_lengths_kv=None,
    query_rope=None,
    key_rope=None,
    shared_prefix_length=0,
    layout_query: str = "BSND",
    sparse_mode: int = 3,
    return_softmax_lse: bool = False,
    block_size: int = 0,
):
    """MLA-absorb attention (one KV head, value = key) over the whole visible part of a paged cache.

    Args:
        query: [B,S1,N1,512] BSND or [T1,N1,512] TND, fp16/bf16, any number of heads
        key:   [block_num,block_size,1,512], any block size
        block_table: [B, max_blocks] int32, -1 = no block
        actual_seq_lengths_query: [B] int32 / list / None (S1 each); cumulative, and required, for TND
        actual_seq_lengths_kv: [B] int32 / list: cached keys of each sequence, the prefix counted
        query_rope / key_rope: [..., 64], required
        shared_prefix_length: how many first positions hold the same tokens in every sequence with query tokens, an int or a
            one-element int32 CUDA tensor (read when the call runs, so that a captured graph follows it).  They may be read
            through the pages of any such sequence that sees them all, so that the table has to lead each of them to the same
            keys.  Sequences that do not see the whole prefix are computed from their own pages; sequences without
            query tokens take no part, whatever their lengths and pages.  0: nothing is shared
        sparse_mode: 0 full / 3 rightDownCausal
        return_softmax_lse: also return the softmax statistics (zeros otherwise)
        block_size: paged block length (defaults to key.shape[1])

    Returns:
        (attention_out, softmax_max, softmax_sum); statistics are fp32 [B,1,S1,N1] (BSND) or [1,T1,N1] (TND).  Rows that see
        no key give zeros; rows whose softmax is no number (a score that is NaN or +infinity, or none but -infinity) give NaN in all
        three.  Serving only: paged caches are not differentiated.
    """
    if sparse_mode not in (0, 3):
        raise ValueError("Only sparse_mode 0 (full) / 3 (rightDownCausal) supported")
    if query_rope is None or key_rope is None:
        raise ValueError("query_rope and key_rope are required (no empty rope)")
    if layout_query not in ("BSND", "TND"):
        raise ValueError(f"layout_query must be BSND or TND, got {layout_query}")
    if block_table is None or actual_seq_lengths_kv is None:
        raise ValueError("block_table and actual_seq_lengths_kv are required")
    tnd = layout_query == "TND"
    if query.ndim != (3 if tnd else 4):
        raise ValueError(f"query must be {'[T1,N1,D]' if tnd else '[B,S1,N1,D]'}, got {tuple(query.shape)}")
    if tnd and actual_seq_lengths_query is None:
        raise ValueError("TND query requires cumulative actual_seq_lengths_query")
    lead, N1, D = query.shape[:-2], query.shape[-2], query.shape[-1]
    if D != _D:
        raise ValueError(f"D must be {_D}, got {D}")
    if N1 < 1:
        raise ValueError(f"N1 must be positive, got {N1}")
    if query_rope.shape != (*lead, N1, _D_ROPE):
        raise ValueError(f"query_rope must have shape {(*lead, N1, _D_ROPE)}, got {tuple(query_rope.shape)}")
    blocks, page = key.shape[0], key.shape[1]
    if key.shape != (blocks, page, 1, D) or blocks < 1 or page < 1:
        raise ValueError(f"key must be [block_num,block_size,1,{D}] with a block at least, got {tuple(key.shape)}")
    if key_rope.shape != (blocks, page, 1, _D_ROPE):
        raise ValueError(f"key_rope must have shape {(blocks, page, 1, _D_ROPE)}, got {tuple(key_rope.shape)}")
    if block_size and block_size != page:
        raise ValueError("block_size must equal the cache's block dimension")
    dtype = query.dtype
    if key.dtype is not dtype or query_rope.dtype is not dtype or key_rope.dtype is not dtype:
        raise ValueError("query, key, query_rope and key_rope must share a dtype")
    code = dtype_code(query, (torch.bfloat16, torch.float16), "query")
    prefix, prefix_t = shared_prefix_length, None
    if isinstance(prefix, torch.Tensor):
        if prefix.dtype != torch.int32 or prefix.numel() != 1:
            raise ValueError("shared_prefix_length must be an int or a one-element int32 tensor")
        prefix, prefix_t = 0, prefix
    prefix = min(int(prefix), 2**31 - 1)
    if prefix < 0:
        raise ValueError(f"shared_prefix_length must not be negative, got {prefix}")
    one_device(query, key, query_rope, key_rope, prefix_t)
    dev = query.device
    seq_q, _ = seq_tensor(actual_seq_lengths_query, dev)
    seq_k, _ = seq_tensor(actual_seq_lengths_kv, dev)
    B = seq_q.shape[0] if tnd else lead[0]
    block_table = int32_table(block_table, dev)
    if block_table.ndim != 2 or block_table.shape[0] != B or seq_k.shape != (B,) or (
            seq_q is not None and seq_q.shape != (B,)):
        raise ValueError(f"block_table and lengths must have an entry for each of the {B} sequences")
    query, query_rope, key, key_rope = packed(query), packed(query_rope), packed(key), packed(key_rope)
    s1 = lead[-1]

    out = torch.empty_like(query)
    stat_shape = (1, s1, N1) if tnd else (B, 1, s1, N1)
    sm_max = torch.empty(stat_shape, dtype=torch.float32, device=dev)
    sm_sum = torch.empty_like(sm_max)
    if out.numel() == 0:
        return out, sm_max, sm_sum
    if B == 0:      # tokens that belong to no sequence
        return out.zero_(), sm_max.zero_(), sm_sum.zero_()

    p = _cabi.DsaSpaParams(
        _STRUCT_SIZE, _kernel, query.data_ptr(), query_rope.data_ptr(), key.data_ptr(), key_rope.data_ptr(), ptr(seq_q),
        seq_k.data_ptr(), block_table.data_ptr(), ptr(prefix_t), out.data_ptr(), sm_max.data_ptr(), sm_sum.data_ptr(),
        _cabi.LAYOUTS[layout_query], code, B, s1, N1, D, _D_ROPE, page, block_table.shape[1], prefix, sparse_mode,
        bool(return_softmax_lse), scale_value, blocks * page)
    with device_guard(dev):
        nbytes = ctypes.c_size_t(0)
        _cabi.check(_cabi.lib.dsa_spa_workspace_bytes(ctypes.byref(p), ctypes.byref(nbytes)), "shared_prefix_attention")
        ws = workspace(nbytes.value, dev)
        _cabi.check(_cabi.lib.dsa_spa_forward(ctypes.byref(p), ws.data_ptr(), nbytes.value, current_stream(dev)),
                    "shared_prefix_attention")
        note_launch("shared_prefix_attention", ws, dev)
    return out, sm_max, sm_sum


class SharedPrefixAttention(torch.nn.Module):
    """Attribute holder around shared_prefix_attention."""

    def __init__(self, scale_value=1.0, layout_query="BSND", sparse_mode=3, return_softmax_lse=False, block_size=0):
        super().__init__()
        self.scale_value = scale_value
        self.layout_query = layout_query
        self.sparse_mode = sparse_mode
        self.return_softmax_lse = return_softmax_lse
        self.block_size = block_size

    def forward(self, query, key, query_rope=None, key_rope=None, actual_seq_lengths_query=None,
                actual_seq_lengths_kv=None, block_table=None, shared_prefix_length=0):
        return shared_prefix_attention(
            query, key, scale_value=self.scale_value, block_table=block_table,
            actual_seq_lengths_query=actual_seq_lengths_query, actual_seq_lengths_kv=actual_seq_lengths_kv,
            query_rope=query_rope, key_rope=key_rope, shared_prefix_length=shared_prefix_length,
            layout_query=self.layout_query, sparse_mode=self.sparse_mode, return_softmax_lse=self.return_softmax_lse,
            block_size=self.block_size)

    construct = forward
