"""rotary_embedding and its gradient against a 64-bit rotation: types, layouts, axes, strides, odd widths, far positions."""
import pytest
import torch

from tests.latent_ref import inv_freq, rotation_bound, turn

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _check(x, positions, freq, **kw):
    from dsa_triton_ascend_b200 import rotary_embedding, rotary_embedding_grad
    offset, inter, sections = kw.get("rotary_offset", 0), kw.get("interleaved", True), kw.get("axis_sections")
    before = x.clone()
    for f, sign in ((rotary_embedding, 1.0), (rotary_embedding_grad, -1.0)):
        out = f(x, positions, freq, **kw)
        assert out.shape == x.shape and out.dtype == x.dtype and out.is_contiguous()
        ref = turn(x, positions, freq, sections, offset, inter, sign)
        bound = rotation_bound(x, ref, x.dtype, freq.numel(), offset, inter)
        bad = (out.double() - ref).abs() > bound
        assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} features off"
        keep = torch.ones(x.shape[-1], dtype=torch.bool, device=x.device)
        keep[offset:offset + 2 * freq.numel()] = False
        assert torch.equal(out[..., keep], x[..., keep])
    assert torch.equal(x, before)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("tokens,heads,width,pairs,offset", [
    (1, 1, 64, 32, 0), (1, 128, 64, 32, 0), (777, 5, 64, 32, 0), (300, 64, 128, 32, 64), (33, 7, 128, 32, 0),
    (19, 3, 192, 64, 64), (50, 3, 66, 33, 0), (50, 3, 71, 5, 3), (4, 2, 1024, 512, 0), (3, 1, 2, 1, 0), (9, 130, 200, 32, 136),
    (2001, 1, 64, 32, 0), (5, 2, 264, 4, 8)])
def test_rotation(dtype, interleaved, tokens, heads, width, pairs, offset):
    g = torch.Generator(device="cuda").manual_seed(tokens + heads)
    x = torch.randn(tokens, heads, width, generator=g, device="cuda").to(DT[dtype])
    pos = torch.randint(0, 200000, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    _check(x, pos, inv_freq(pairs), layout="TND", interleaved=interleaved, rotary_offset=offset)


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("sections", [(32,), (8, 12, 12), (1, 31), (0, 16, 0, 16), (4, 4, 12, 12)])
def test_several_axes(sections, interleaved):
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(3, 41, 6, 128, generator=g, device="cuda").bfloat16()
    pos = torch.randint(-50, 5000, (len(sections), 3, 41), generator=g, device="cuda")
    _check(x, pos, inv_freq(), interleaved=interleaved, rotary_offset=64, axis_sections=sections)


def test_far_and_negative_positions():
    """A 32-bit product of position and frequency would be off by radians here."""
    x = torch.randn(2, 6, 4, 64, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    pos = torch.tensor([[0, 1, -1, 2**31 - 1, -2**31, 123456789], [2**40 + 1, -2**40, 999999999999, 7, 65536, 2**33]], device="cuda")
    # (64-bit angles of the plain form at 10^12 radians are themselves good to 1e-4: compare with whole turns taken off first)
    from dsa_triton_ascend_b200 import rotary_embedding
    freq = inv_freq()
    out = rotary_embedding(x, pos, freq).double().cpu()
    from fractions import Fraction
    import math
    pi = Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899862803482534211706798214808651")
    for b in range(2):
        for s in range(6):
            for j in range(32):
                angle = Fraction(int(pos[b, s])) * Fraction(float(freq[j]))
                turns = angle / (2 * pi)
                a = float((turns - round(turns)) * 2 * pi)
                # relative error of the 64-bit turns: two roundings and the constant's, 4 x 2^-53
                slack = abs(float(turns)) * 2 * math.pi * 4 * 2.0**-53 + 1e-6
                re, im = x[b, s, :, 2 * j].double().cpu(), x[b, s, :, 2 * j + 1].double().cpu()
                want = re * math.cos(a) - im * math.sin(a)
                assert ((out[b, s, :, 2 * j] - want).abs() <= slack * (re.abs() + im.abs())).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_strided_and_unaligned_inputs(dtype):
    g = torch.Generator(device="cuda").manual_seed(3)
    big = torch.randn(3, 17, 9, 200, generator=g, device="cuda").to(DT[dtype])
    pos = torch.randint(0, 4096, (3, 17), generator=g, device="cuda")
    for x in (big[..., 136:200], big[..., 3:67], big[:, ::2, 1:5, 8:72].transpose(0, 0), big[:, :, ::3, :64],
              big.transpose(0, 1)[..., :64], big[:1].expand(3, 17, 9, 200)[..., 64:128], big[..., ::2][..., :64]):
        p = pos[:, :x.shape[1]] if x.shape[0] == 3 else torch.randint(0, 99, x.shape[:2], generator=g, device="cuda")
        _check(x, p, inv_freq())
    flat = torch.randn(4 * 8 * 64 + 1, generator=g, device="cuda").to(DT[dtype])
    _check(flat[1:].view(4, 8, 64), pos[0, :4], inv_freq(), layout="TND")


def test_nothing_to_rotate():
    from dsa_triton_ascend_b200 import rotary_embedding
    for shape in ((0, 4, 2, 64), (2, 0, 2, 64), (2, 3, 0, 64)):
        x = torch.empty(shape, device="cuda", dtype=torch.bfloat16)
        assert rotary_embedding(x, torch.zeros(shape[:2], dtype=torch.int32, device="cuda"), inv_freq()).shape == shape


def test_values_that_are_not_numbers_stay_in_their_pairs():
    from dsa_triton_ascend_b200 import rotary_embedding
    x = torch.zeros(4, 2, 64, device="cuda", dtype=torch.bfloat16)
    x[1, 0, 6] = float("nan")
    x[2, 1, 9] = float("inf")
    out = rotary_embedding(x, torch.arange(4, device="cuda"), inv_freq(), layout="TND")
    bad = ~torch.isfinite(out)
    want = torch.zeros_like(bad)
    want[1, 0, 6:8] = True
    want[2, 1, 8:10] = True
    assert torch.equal(bad, want)


def test_gradient_against_differences():
    """Linear in x: the difference quotient along any direction is the product with the gradient's transpose."""
    from dsa_triton_ascend_b200 import rotary_embedding, rotary_embedding_grad
    g = torch.Generator(device="cuda").manual_seed(5)
    x, d, w = (torch.randn(37, 3, 128, generator=g, device="cuda") for _ in range(3))
    pos = torch.randint(0, 5000, (2, 37), generator=g, device="cuda")
    kw = dict(layout="TND", interleaved=False, rotary_offset=32, axis_sections=(20, 12))
    f = lambda v: (rotary_embedding(v, pos, inv_freq(), **kw).double() * w.double()).sum()
    got = (rotary_embedding_grad(w, pos, inv_freq(), **kw).double() * d.double()).sum()
    want = (f(x + d) - f(x - d)) / 2
    # 14208 products of size 1, each off by at most 3e-6: the sum of their errors stays below 0.05
    assert abs(float(got - want)) < 0.05


def test_captured_and_on_another_stream():
    from dsa_triton_ascend_b200 import rotary_embedding
    x = torch.randn(64, 16, 64, device="cuda").bfloat16()
    pos = torch.arange(64, device="cuda", dtype=torch.int32)
    freq = inv_freq()
    want = rotary_embedding(x, pos, freq, layout="TND")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = rotary_embedding(x, pos, freq, layout="TND")
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = rotary_embedding(x, pos, freq, layout="TND")
    pos.add_(5)
    want = rotary_embedding(x, pos, freq, layout="TND")
    graph.replay()
    assert torch.equal(y, want)


def test_module_holds_the_arguments():
    from dsa_triton_ascend_b200 import RotaryEmbedding, rotary_embedding
    x = torch.randn(2, 5, 3, 128, device="cuda").half()
    pos = torch.arange(10, device="cuda").view(2, 5)
    m = RotaryEmbedding(inv_freq(), interleaved=False, rotary_offset=64)
    assert torch.equal(m(x, pos), rotary_embedding(x, pos, inv_freq(), interleaved=False, rotary_offset=64))
