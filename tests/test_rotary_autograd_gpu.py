"""Gradients of rotary_embedding through torch's autograd."""
import pytest
import torch

from tests.latent_ref import inv_freq, rotation_bound, turn

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("interleaved,offset,sections", [(True, 0, None), (False, 64, (8, 12, 12)), (True, 30, (20, 12))])
def test_gradient_of_the_formula(dtype, interleaved, offset, sections):
    from dsa_triton_ascend_b200 import rotary_embedding
    g = torch.Generator(device="cuda").manual_seed(1)
    x, w = (torch.randn(3, 41, 6, 128, generator=g, device="cuda").to(DT[dtype]) for _ in range(2))
    pos = torch.randint(0, 5000, (3, 41) if sections is None else (len(sections), 3, 41), generator=g, device="cuda")
    x.requires_grad_()
    kw = dict(interleaved=interleaved, rotary_offset=offset, axis_sections=sections)
    y = rotary_embedding(x, pos, inv_freq(), **kw)
    assert y.requires_grad and torch.equal(y, rotary_embedding(x.detach(), pos, inv_freq(), **kw))
    (got,) = torch.autograd.grad(y, x, w)
    want = turn(w, pos, inv_freq(), sections, offset, interleaved, -1.0)
    assert got.dtype == x.dtype
    assert ((got.double() - want).abs() <= rotation_bound(w, want, x.dtype, 32, offset, interleaved)).all()


def test_gradient_of_differences_through_a_module_and_a_slice():
    """A projection whose slice is rotated: the gradients of what lies before the rotation, against difference quotients."""
    from dsa_triton_ascend_b200 import RotaryEmbedding
    g = torch.Generator(device="cuda").manual_seed(2)
    a, weight, v, d = (torch.randn(*s, generator=g, device="cuda") for s in ((7, 32), (32, 4 * 192), (7, 4, 64), (32, 4 * 192)))
    pos = torch.randint(0, 5000, (7,), generator=g, device="cuda")
    rotary = RotaryEmbedding(inv_freq(), layout="TND")
    f = lambda w: (rotary((a @ w).view(7, 4, 192)[..., 128:], pos).double() * v.double()).sum()
    weight.requires_grad_()
    f(weight).backward()
    got = (weight.grad.double() * d.double()).sum()
    with torch.no_grad():
        want = (f(weight + d) - f(weight - d)) / 2
        assert not rotary(a.view(7, 1, 32).repeat(1, 1, 2), pos).requires_grad
    # linear in the weight: 1792 products of size 6 x 1, each off by at most 1e-5 of 6 (sums of 32 products, a rotation)
    assert abs(float(got - want)) < 1792 * 6e-5


def test_gradient_of_the_gradient():
    from dsa_triton_ascend_b200 import rotary_embedding, rotary_embedding_grad
    x, w = (torch.randn(5, 3, 64, device="cuda", requires_grad=True) for _ in range(2))
    pos = torch.arange(5, device="cuda")
    y = rotary_embedding(x, pos, inv_freq(), layout="TND")
    (dx,) = torch.autograd.grad(y, x, w, create_graph=True)
    u = torch.randn_like(dx)
    (dw,) = torch.autograd.grad(dx, w, u)
    assert torch.equal(dw, rotary_embedding(u, pos, inv_freq(), layout="TND"))
    z = rotary_embedding_grad(w, pos, inv_freq(), layout="TND")
    assert torch.equal(z, dx) and torch.equal(torch.autograd.grad(z, w, u)[0], dw)


def test_expanded_gradients_and_nothing_to_rotate():
    from dsa_triton_ascend_b200 import rotary_embedding, rotary_embedding_grad
    x = torch.randn(5, 3, 64, device="cuda", requires_grad=True)
    pos = torch.arange(5, device="cuda")
    rotary_embedding(x, pos, inv_freq(), layout="TND").sum().backward()
    assert torch.equal(x.grad, rotary_embedding_grad(torch.ones_like(x), pos, inv_freq(), layout="TND"))
    x = torch.randn(0, 3, 64, device="cuda", requires_grad=True)
    rotary_embedding(x, pos[:0], inv_freq(), layout="TND").sum().backward()
    assert x.grad.shape == x.shape


def test_positions_that_change_before_the_backward_pass_are_refused():
    from dsa_triton_ascend_b200 import rotary_embedding
    x = torch.randn(5, 3, 64, device="cuda", requires_grad=True)
    pos = torch.arange(5, device="cuda")
    y = rotary_embedding(x, pos, inv_freq(), layout="TND")
    pos.add_(1)
    with pytest.raises(RuntimeError):
        y.sum().backward()


def test_captured_step_with_its_backward_pass_and_another_stream():
    from dsa_triton_ascend_b200 import rotary_embedding, rotary_embedding_grad
    x, w = (torch.randn(64, 16, 64, device="cuda").bfloat16() for _ in range(2))
    pos, freq = torch.arange(64, device="cuda"), inv_freq()

    def step():
        leaf = x.detach().requires_grad_()
        y = rotary_embedding(leaf, pos, freq, layout="TND")
        return y.detach(), torch.autograd.grad(y, leaf, w)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, step()):
        assert torch.equal(a, b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    pos.add_(5)
    x.mul_(-1)
    graph.replay()
    want = (rotary_embedding(x, pos, freq, layout="TND"), rotary_embedding_grad(w, pos, freq, layout="TND"))
    assert all(torch.equal(a, b) for a, b in zip(held, want))
