"""Append of new tokens to the paged caches on B200: latents (optionally normalised), rope keys and index keys
(rotated on the way).

No counterpart in the reference, whose operators take caches that are already filled (PA_BSND,
sparse_flash_attention_triton.py:1012-1033).  The lengths and the block table are those of the operators that read the
caches afterwards.
"""
import ctypes

import torch

from . import _cabi
from ._host import KeepsFloat32, current_stream, device_guard, dtype_code, int32_table, one_device, ptr, seq_tensor
from .rotary import check_inv_freq, check_positions, section_sizes

_VALID_D = (128, 256, 512)
_D_ROPE = 64
_PAIRS = (_D_ROPE // 2,)
_STRUCT_SIZE = ctypes.sizeof(_cabi.DsaAppendParams)


def _token_rows(t, step, align):
    """(`t`, stride of a sequence, stride of a token) with a contiguous last dimension, strides that are multiples of `step`
    elements and a start on an `align`-byte boundary: itself (a slice of a projection is read in place) or a copy."""
    stride = t.stride()
    sb, ss = stride[0], stride[-3]
    if stride[-1] != 1 or sb % step or ss % step or t.data_ptr() % align:
        t = t.clone(memory_format=torch.contiguous_format)
        stride = t.stride()
        sb, ss = stride[0], stride[-3]
    return t, sb, ss


def _check_pair(new, cache, tokens, blocks, block_size, width, dtype, what):
    if new.shape != (*tokens, 1, width):
        raise ValueError(f"{what} must have shape {(*tokens, 1, width)}, got {tuple(new.shape)}")
    if cache.shape != (blocks, block_size, 1, width):
        raise ValueError(f"the cache of {what} must have shape {(blocks, block_size, 1, width)}, got {tuple(cache.shape)}")
    if new.dtype is not dtype or cache.dtype is not dtype:
        raise ValueError("tokens and caches must share a dtype")
    if not cache.is_contiguous():
        raise ValueError("caches must be contiguous: they are updated in place")


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
    tnd = layout == "TND"
    if latent.ndim != (3 if tnd else 4) or latent.shape[-2] != 1:
        raise ValueError(f"latent must be {'[T1,1,D]' if tnd else '[B,S1,1,D]'}, got {tuple(latent.shape)}")
    if tnd and actual_seq_lengths_query is None:
        raise ValueError("TND tokens require cumulative actual_seq_lengths_query")
    if block_table is None or actual_seq_lengths_kv is None:
        raise ValueError("block_table and actual_seq_lengths_kv are required")
    if (index_key is None) != (index_cache is None):
        raise ValueError("index_key and index_cache go together")
    D, tokens = latent.shape[-1], latent.shape[:-2]
    if D not in _VALID_D:
        raise ValueError(f"D must be one of {_VALID_D}, got {D}")
    if latent_cache.ndim != 4 or latent_cache.shape[1] < 1:
        raise ValueError("caches must be [block_num,block_size,1,D]")
    blocks, block_size = latent_cache.shape[0], latent_cache.shape[1]
    dtype = latent.dtype
    code = dtype_code(latent, (torch.bfloat16, torch.float16), "latent")
    _check_pair(latent, latent_cache, tokens, blocks, block_size, D, dtype, "latent")
    _check_pair(key_rope, rope_cache, tokens, blocks, block_size, _D_ROPE, dtype, "key_rope")
    d_index = 0
    if index_key is not None:
        d_index = index_key.shape[-1]
        _check_pair(index_key, index_cache, tokens, blocks, block_size, d_index, dtype, "index_key")
        if (d_index < 64 or d_index > 1024 or d_index % 2 or index_rotary_offset < 0 or index_rotary_offset % 2 or
                index_rotary_offset + _D_ROPE > d_index):
            raise ValueError(f"64 features from an even index_rotary_offset on must fit D_idx (even, 64 to 1024): got "
                             f"{index_rotary_offset} and {d_index}")
    inv_freq = check_inv_freq(inv_freq)
    if inv_freq.shape[0] != _D_ROPE // 2:
        raise ValueError(f"inv_freq must have {_D_ROPE // 2} entries, got {inv_freq.shape[0]}")
    axes, sections = 1, _PAIRS
    if positions is not None:
        axes, sections = section_sizes(axis_sections, _D_ROPE // 2)
        positions = check_positions(positions, tokens, axis_sections)
    elif axis_sections is not None:
        raise ValueError("axis_sections needs positions")
    code_w = code
    if norm_weight is not None:
        if norm_weight.shape != (D,) or (norm_weight.dtype is not dtype and norm_weight.dtype is not torch.float32):
            raise ValueError(f"norm_weight must be [{D}] in the latents' dtype or float32")
        norm_weight = norm_weight.contiguous()
        if norm_weight.data_ptr() % 16:
            norm_weight = norm_weight.clone()
        if norm_weight.dtype is torch.float32:
            code_w = _cabi.DTYPE_FP32
    one_device(latent, key_rope, latent_cache, rope_cache, inv_freq, index_key, index_cache, positions, norm_weight)
    dev = latent.device
    if latent_cache.data_ptr() % 16 or rope_cache.data_ptr() % 4 or (index_cache is not None and index_cache.data_ptr() % 4):
        raise ValueError("caches must start on 16-byte boundaries (latents) and 4-byte boundaries (the others)")
    seq_q, _ = seq_tensor(actual_seq_lengths_query, dev)
    seq_k, _ = seq_tensor(actual_seq_lengths_kv, dev)
    block_table = int32_table(block_table, dev)
    batch = seq_q.shape[0] if tnd else tokens[0]
    if block_table.ndim != 2 or block_table.shape[0] != batch or seq_k.shape != (batch,) or (
            seq_q is not None and seq_q.shape != (batch,)):
        raise ValueError(f"block_table and lengths must have an entry for each of the {batch} sequences")
    if latent.numel() == 0 or batch == 0 or blocks == 0 or block_table.shape[1] == 0:
        return latent_cache, rope_cache, index_cache
    latent, latent_b, latent_s = _token_rows(latent, 8, 16)
    key_rope, rope_b, rope_s = _token_rows(key_rope, 2, 4)
    index_b = index_s = 0
    if index_key is not None:
        index_key, index_b, index_s = _token_rows(index_key, 2, 4)

    p = _cabi.DsaAppendParams(
        _STRUCT_SIZE, code, latent.data_ptr(), key_rope.data_ptr(), ptr(index_key), ptr(norm_weight), ptr(positions),
        inv_freq.data_ptr(), ptr(seq_q), seq_k.data_ptr(), block_table.data_ptr(), latent_cache.data_ptr(), rope_cache.data_ptr(),
        ptr(index_cache), latent_b, latent_s, rope_b, rope_s, index_b, index_s, _cabi.LAYOUTS[layout], batch, tokens[-1], D,
        _D_ROPE, d_index, index_rotary_offset, block_size, block_table.shape[1], bool(interleaved), bool(index_interleaved),
        positions is not None and positions.dtype is torch.int64, code_w, axes, sections, norm_eps, blocks * block_size)
    with device_guard(dev):
        _cabi.check(_cabi.lib.dsa_latent_append(ctypes.byref(p), current_stream(dev)), "latent_cache_append")
    return latent_cache, rope_cache, index_cache


class LatentCacheAppend(KeepsFloat32):
    """Attribute holder around latent_cache_append.  inv_freq and a float32 norm_weight stay float32 when the model is cast."""

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
