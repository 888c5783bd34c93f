"""Rotary positions of queries and keys on B200, with one position axis or several, and their gradient.

No counterpart in the reference, whose operators take `query_rope`, `key_rope` and the index queries and keys already
rotated (sparse_flash_attention_triton.py:1317-1339).  Names, layouts and checks follow the other operators.
"""
import ctypes

import torch

from . import _cabi
from ._host import KeepsFloat32, current_stream, device_guard, dtype_code, one_device

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_STRUCT_SIZE = ctypes.sizeof(_cabi.DsaRopeParams)
MAX_AXES = 4


def section_sizes(axis_sections, pairs):
    """(axes, pairs per axis) of `axis_sections`; None: one axis."""
    if axis_sections is None:
        return 1, (pairs,)
    sections = tuple(int(n) for n in axis_sections)
    if not 1 <= len(sections) <= MAX_AXES or min(sections) < 0 or sum(sections) != pairs:
        raise ValueError(f"axis_sections must be 1 to {MAX_AXES} numbers of pairs whose sum is {pairs}, got {axis_sections}")
    return len(sections), sections


def check_positions(positions, tokens, axis_sections, what="positions"):
    """`positions` of shape `tokens`, or [axes, *tokens] where axis_sections are given, as a contiguous tensor."""
    want = tokens if axis_sections is None else (len(axis_sections), *tokens)
    if positions.dtype is not torch.int32 and positions.dtype is not torch.int64:
        raise ValueError(f"{what} must be int32 or int64, got {positions.dtype}")
    if positions.shape != want:
        raise ValueError(f"{what} must have shape {want}, got {tuple(positions.shape)}")
    return positions.contiguous()


def check_inv_freq(inv_freq):
    if inv_freq.dtype != torch.float32 or inv_freq.ndim != 1 or inv_freq.numel() < 1:
        raise ValueError("inv_freq must be a float32 vector with an entry per pair")
    return inv_freq.contiguous()


def _rotate(x, positions, inv_freq, layout, interleaved, rotary_offset, axis_sections, inverse, what):
    if layout == "BSND":
        if x.ndim != 4:
            raise ValueError(f"{what} must be [B,S,N,D], got {tuple(x.shape)}")
        batch, s1, n, D = x.shape
        stride_b, stride_s, stride_n, stride_d = x.stride()
        tokens = (batch, s1)
    elif layout == "TND":
        if x.ndim != 3:
            raise ValueError(f"{what} must be [T,N,D], got {tuple(x.shape)}")
        s1, n, D = x.shape
        stride_s, stride_n, stride_d = x.stride()
        batch, stride_b, tokens = 1, 0, (s1,)
    else:
        raise ValueError(f"layout must be BSND or TND, got {layout}")
    code = dtype_code(x, _DTYPES, what)
    inv_freq = check_inv_freq(inv_freq)
    pairs = inv_freq.shape[0]
    if D > 1024 or rotary_offset < 0 or rotary_offset + 2 * pairs > D:
        raise ValueError(f"{pairs} pairs from feature {rotary_offset} on do not fit {D} features (at most 1024)")
    axes, sections = section_sizes(axis_sections, pairs)
    positions = check_positions(positions, tokens, axis_sections)
    one_device(x, positions, inv_freq)
    if batch == 0 or s1 == 0 or n == 0:     # (contiguous whatever its strides are)
        return torch.empty_like(x, memory_format=torch.contiguous_format)
    if stride_d != 1:
        return _rotate(x.contiguous(), positions, inv_freq, layout, interleaved, rotary_offset, axis_sections, inverse, what)
    out = torch.empty_like(x, memory_format=torch.contiguous_format)
    p = _cabi.DsaRopeParams(
        _STRUCT_SIZE, inverse, x.data_ptr(), positions.data_ptr(), inv_freq.data_ptr(), out.data_ptr(), stride_b, stride_s,
        stride_n, code, positions.dtype is torch.int64, batch, s1, n, D, pairs, rotary_offset, bool(interleaved), axes, sections)
    dev = x.device
    with device_guard(dev):
        _cabi.check(_cabi.lib.dsa_rope(ctypes.byref(p), current_stream(dev)), "rotary_embedding")
    return out


class _Rotation(torch.autograd.Function):
    """The rotation for autograd: linear in x, and its transpose is the rotation by the opposite angles."""

    @staticmethod
    def forward(ctx, x, positions, inv_freq, layout, interleaved, rotary_offset, axis_sections, inverse):
        ctx.save_for_backward(positions, inv_freq)
        ctx.how = (layout, interleaved, rotary_offset, None if axis_sections is None else tuple(axis_sections), not inverse)
        return _rotate(x, positions, inv_freq, layout, interleaved, rotary_offset, axis_sections, inverse, "x")

    @staticmethod
    def backward(ctx, d_out):
        return (_recorded(d_out, *ctx.saved_tensors, *ctx.how, "d_out"), *[None] * 7)


def _recorded(x, positions, inv_freq, layout, interleaved, rotary_offset, axis_sections, inverse, what):
    if x.requires_grad and torch.is_grad_enabled():
        return _Rotation.apply(x, positions, inv_freq, layout, interleaved, rotary_offset, axis_sections, inverse)
    return _rotate(x, positions, inv_freq, layout, interleaved, rotary_offset, axis_sections, inverse, what)


def rotary_embedding(x, positions, inv_freq, layout: str = "BSND", interleaved: bool = True, rotary_offset: int = 0,
                     axis_sections=None):
    """Rotate features of queries or keys by their tokens' positions.

    Pair j of the rotated features, as one complex number, is multiplied by exp(i p inv_freq[j]).

    Args:
        x: [B,S,N,D] BSND or [T,N,D] TND, bf16 / fp16 / fp32, D up to 1024; any strides (a slice of a projection is read
            in place as long as its last dimension is contiguous)
        positions: int32 or int64 [B,S] / [T]; with axis_sections [axes,B,S] / [axes,T]
        inv_freq: float32 [pairs], radians per position
        interleaved: a pair is features (2j, 2j + 1) of the rotated ones; otherwise (j, j + pairs)
        rotary_offset: first rotated feature; the 2 * pairs features from there on are rotated, the others copied
        axis_sections: pairs per position axis (time, height, width, ...), in order, up to four axes; None: one axis

    Returns: a new contiguous tensor of x's shape and dtype.  Angles are taken in 64 bits, sine, cosine and the rotation
    in 32.  Autograd records the call where x requires a gradient; without it the gradient is `rotary_embedding_grad`.
    Positions and frequencies are not differentiated, and may not change before the backward pass.
    """
    return _recorded(x, positions, inv_freq, layout, interleaved, rotary_offset, axis_sections, False, "x")


def rotary_embedding_grad(d_out, positions, inv_freq, layout: str = "BSND", interleaved: bool = True,
                          rotary_offset: int = 0, axis_sections=None):
    """Gradient of `rotary_embedding` with respect to x, given the gradient of its result: the rotation by the
    opposite angles.  Arguments as there."""
    return _recorded(d_out, positions, inv_freq, layout, interleaved, rotary_offset, axis_sections, True, "d_out")


class RotaryEmbedding(KeepsFloat32):
    """Attribute holder around rotary_embedding.  inv_freq stays float32 when the model is cast."""

    def __init__(self, inv_freq, layout="BSND", interleaved=True, rotary_offset=0, axis_sections=None):
        super().__init__()
        self.register_buffer("inv_freq", inv_freq, persistent=False)
        self.layout = layout
        self.interleaved = interleaved
        self.rotary_offset = rotary_offset
        self.axis_sections = axis_sections

    def forward(self, x, positions):
        return rotary_embedding(x, positions, self.inv_freq, self.layout, self.interleaved, self.rotary_offset,
                                self.axis_sections)

    construct = forward
