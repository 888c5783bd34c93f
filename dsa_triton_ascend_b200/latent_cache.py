"""Append of new tokens to the paged caches on B200: latents (optionally normalised), rope keys and index keys
(rotated on the way).

No counterpart in the reference, whose operators take caches that are already filled (PA_BSND,
sparse_flash_attention_triton.py:1012-1033).  The lengths and the block table are those of the operators that read the
caches afterwards.
"""
import ctypes

import torch

from . import _cabi
from ._host import current_stream, device_guard, dtype_code, ptr, require_cuda, same_device, seq_tensor
from .rotary import check_inv_freq, check_positions, section_sizes

_VALID_D = (128, 256, 512)
_D_ROPE = 64


def _token_rows(t, step, align):
    """`t` with a contiguous last dimension, strides that are multiples of `step` elements and a start on an `align`-byte
    boundary: itself (a slice of a projection is read in place) or a copy."""
    if t.stride(-1) != 1 or any(s % step for s in t.stride()[:-2]) or t.data_ptr() % align:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def latent_cache_append(
    latent,
    key_rope,
    latent_cache,
    rope_cache,
    inv_freq,
    block_table=None,
    actual_seq_lengths_query=None,
    actual_seq_lengths_kv=None,
    index_key=None,
    index_cache=None,
    positions=None,
    axis_sections=None,
    layout: str = "BSND",
    norm_weight=None,
    norm_eps: float = 1e-6,
    interleaved: bool = True,
    index_interleaved: bool = False,
    index_rotary_offset: int = 0,
):
    """Write new tokens into the paged caches that `lightning_indexer_triton`, `sparse_flash_attention_triton` and
    `shared_prefix_attention` read (PA_BSND).

    Token i of sequence b goes to position actual_seq_lengths_kv[b] - actual_seq_lengths_query[b] + i of that sequence.

    Args:
        latent:   [B,S1,1,D] BSND or [T1,1,D] TND, bf16 / fp16, D in 128/256/512
        key_rope: the same with 64; rotated by its token's position
        latent_cache / rope_cache: [block_num,block_size,1,D] / [...,64], contiguous, updated in place
        inv_freq: float32 [32], radians per position
        block_table: [B, max_blocks] int32, -1 = no block
        actual_seq_lengths_query: [B] int32 / list / None (S1 each); cumulative, and required, for TND
        actual_seq_lengths_kv: [B] int32 / list: cached tokens of each sequence, the new ones counted
        index_key / index_cache: [...,D_idx] / [block_num,block_size,1,D_idx], D_idx even, 64 to 1024, both or neither; the
            64 features from index_rotary_offset on are rotated
        positions: int32 or int64 [B,S1] / [T1], or [axes,...] with axis_sections: the positions to rotate by in place of
            the tokens' positions in the cache
        norm_weight: [D] in the latents' dtype or float32: latents are stored as x * rsqrt(mean(x^2) + norm_eps) * weight
        interleaved / index_interleaved: pairs are neighbours (2j, 2j + 1), otherwise (j, j + 32)

    Tokens past their sequence's query length, at positions before 0 or past the table, or whose block is absent or
    beyond the cache are left out, and every other slot keeps what it holds.  No two tokens of a call may
    share a slot, and the tokens must not lie in the caches' own memory.

    Returns: (latent_cache, rope_cache, index_cache), the tensors that were passed.
    """
    if layout not in ("BSND", "TND"):
        raise ValueError(f"layout must be BSND or TND, got {layout}")
    lead = latent.ndim - 2
    if latent.ndim != (4 if layout == "BSND" else 3) or latent.shape[-2] != 1:
        raise ValueError(f"latent must be {'[B,S1,1,D]' if layout == 'BSND' else '[T1,1,D]'}, got {tuple(latent.shape)}")
    if layout == "TND" and actual_seq_lengths_query is None:
        raise ValueError("TND tokens require cumulative actual_seq_lengths_query")
    if block_table is None or actual_seq_lengths_kv is None:
        raise ValueError("block_table and actual_seq_lengths_kv are required")
    if (index_key is None) != (index_cache is None):
        raise ValueError("index_key and index_cache go together")
    D, tokens = latent.shape[-1], latent.shape[:lead]
    if D not in _VALID_D:
        raise ValueError(f"D must be one of {_VALID_D}, got {D}")
    if latent_cache.ndim != 4:
        raise ValueError("caches must be [block_num,block_size,1,D]")
    blocks, block_size = latent_cache.shape[0], latent_cache.shape[1]
    d_index = index_key.shape[-1] if index_key is not None else 0
    for new, cache, width, what in ((latent, latent_cache, D, "latent"), (key_rope, rope_cache, _D_ROPE, "key_rope"),
                                    (index_key, index_cache, d_index, "index_key")):
        if new is None:
            continue
        if tuple(new.shape) != (*tokens, 1, width):
            raise ValueError(f"{what} must have shape {(*tokens, 1, width)}, got {tuple(new.shape)}")
        if tuple(cache.shape) != (blocks, block_size, 1, width):
            raise ValueError(f"the cache of {what} must have shape {(blocks, block_size, 1, width)}, got {tuple(cache.shape)}")
        if new.dtype != latent.dtype or cache.dtype != latent.dtype:
            raise ValueError("tokens and caches must share a dtype")
        if not cache.is_contiguous():
            raise ValueError("caches must be contiguous: they are updated in place")
    if block_size < 1:
        raise ValueError("block_size must be positive")
    if index_key is not None and (d_index < 64 or d_index > 1024 or d_index % 2 or index_rotary_offset < 0 or
                                  index_rotary_offset % 2 or index_rotary_offset + _D_ROPE > d_index):
        raise ValueError(f"64 features from an even index_rotary_offset on must fit D_idx (even, 64 to 1024): got "
                         f"{index_rotary_offset} and {d_index}")
    inv_freq = check_inv_freq(inv_freq)
    if inv_freq.numel() != _D_ROPE // 2:
        raise ValueError(f"inv_freq must have {_D_ROPE // 2} entries, got {inv_freq.numel()}")
    code = dtype_code(latent, (torch.bfloat16, torch.float16), "latent")
    axes, sections = 1, (_D_ROPE // 2,)
    if positions is not None:
        axes, sections = section_sizes(axis_sections, _D_ROPE // 2)
        positions = check_positions(positions, tokens, axis_sections)
    elif axis_sections is not None:
        raise ValueError("axis_sections needs positions")
    if norm_weight is not None:
        if tuple(norm_weight.shape) != (D,) or norm_weight.dtype not in (latent.dtype, torch.float32):
            raise ValueError(f"norm_weight must be [{D}] in the latents' dtype or float32")
        norm_weight = norm_weight.contiguous()
        if norm_weight.data_ptr() % 16:
            norm_weight = norm_weight.clone()
    require_cuda(latent, key_rope, latent_cache, rope_cache, inv_freq, block_table, index_key, index_cache, positions,
                 norm_weight)
    same_device(latent, key_rope, latent_cache, rope_cache, inv_freq, index_key, index_cache, positions, norm_weight)
    dev = latent.device
    if latent_cache.data_ptr() % 16 or any(c is not None and c.data_ptr() % 4 for c in (rope_cache, index_cache)):
        raise ValueError("caches must start on 16-byte boundaries (latents) and 4-byte boundaries (the others)")
    seq_q, _ = seq_tensor(actual_seq_lengths_query, dev)
    seq_k, _ = seq_tensor(actual_seq_lengths_kv, dev)
    block_table = block_table.to(device=dev, dtype=torch.int32).contiguous()
    batch = seq_q.shape[0] if layout == "TND" else latent.shape[0]
    if block_table.ndim != 2 or block_table.shape[0] != batch or tuple(seq_k.shape) != (batch,) or (
            seq_q is not None and tuple(seq_q.shape) != (batch,)):
        raise ValueError(f"block_table and lengths must have an entry for each of the {batch} sequences")
    if latent.numel() == 0 or batch == 0 or latent_cache.numel() == 0 or block_table.shape[1] == 0:
        return latent_cache, rope_cache, index_cache
    latent, key_rope = _token_rows(latent, 8, 16), _token_rows(key_rope, 2, 4)
    if index_key is not None:
        index_key = _token_rows(index_key, 2, 4)

    p = _cabi.DsaAppendParams()
    p.struct_size = ctypes.sizeof(_cabi.DsaAppendParams)
    p.dtype = code
    p.latent, p.key_rope, p.index_key, p.norm_weight = ptr(latent), ptr(key_rope), ptr(index_key), ptr(norm_weight)
    p.positions, p.inv_freq = ptr(positions), ptr(inv_freq)
    p.seq_q, p.seq_k, p.block_table = ptr(seq_q), ptr(seq_k), ptr(block_table)
    p.latent_cache, p.rope_cache, p.index_cache = ptr(latent_cache), ptr(rope_cache), ptr(index_cache)
    p.latent_stride_b, p.latent_stride_s = latent.stride(0), latent.stride(lead - 1)
    p.rope_stride_b, p.rope_stride_s = key_rope.stride(0), key_rope.stride(lead - 1)
    if index_key is not None:
        p.index_stride_b, p.index_stride_s = index_key.stride(0), index_key.stride(lead - 1)
        p.d_index, p.index_offset = d_index, index_rotary_offset
        p.index_interleaved = 1 if index_interleaved else 0
    p.layout_q, p.batch, p.s1 = _cabi.LAYOUTS[layout], batch, latent.shape[lead - 1]
    p.d, p.d_rope = D, _D_ROPE
    p.block_size, p.max_blocks = block_size, block_table.shape[1]
    p.interleaved = 1 if interleaved else 0
    p.positions_64bit = 1 if positions is not None and positions.dtype == torch.int64 else 0
    p.dtype_w = _cabi.DTYPE_FP32 if norm_weight is not None and norm_weight.dtype == torch.float32 else code
    p.axes = axes
    for i, n in enumerate(sections):
        p.sections[i] = n
    p.norm_eps = float(norm_eps)
    p.key_rows = blocks * block_size
    with device_guard(dev):
        _cabi.check(_cabi.lib.dsa_latent_append(ctypes.byref(p), current_stream(dev)), "latent_cache_append")
    return latent_cache, rope_cache, index_cache


class LatentCacheAppend(torch.nn.Module):
    """Attribute holder around latent_cache_append."""

    def __init__(self, inv_freq, layout="BSND", norm_weight=None, norm_eps=1e-6, interleaved=True, index_interleaved=False,
                 index_rotary_offset=0, axis_sections=None):
        super().__init__()
        self.register_buffer("inv_freq", inv_freq, persistent=False)
        self.register_buffer("norm_weight", norm_weight, persistent=False)
        self.layout = layout
        self.norm_eps = norm_eps
        self.interleaved = interleaved
        self.index_interleaved = index_interleaved
        self.index_rotary_offset = index_rotary_offset
        self.axis_sections = axis_sections

    def forward(self, latent, key_rope, latent_cache, rope_cache, index_key=None, index_cache=None, positions=None,
                actual_seq_lengths_query=None, actual_seq_lengths_kv=None, block_table=None):
        return latent_cache_append(
            latent, key_rope, latent_cache, rope_cache, self.inv_freq, block_table=block_table,
            actual_seq_lengths_query=actual_seq_lengths_query, actual_seq_lengths_kv=actual_seq_lengths_kv,
            index_key=index_key, index_cache=index_cache, positions=positions, axis_sections=self.axis_sections,
            layout=self.layout, norm_weight=self.norm_weight, norm_eps=self.norm_eps, interleaved=self.interleaved,
            index_interleaved=self.index_interleaved, index_rotary_offset=self.index_rotary_offset)

    construct = forward
