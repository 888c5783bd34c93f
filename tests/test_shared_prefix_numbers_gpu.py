"""shared_prefix_attention where numbers end: values that are not finite."""
import pytest
import torch

from tests.latent_ref import rows_of
from tests.test_shared_prefix_gpu import KERNELS, call, check, kernel, make, reference

pytestmark = pytest.mark.gpu


def _want(s, mode=3):
    flat = lambda t: t.reshape(-1, *t.shape[-2:])
    return reference(flat(s["q"]), flat(s["qr"]), s["cache"], s["rope"], s["table"], s["q_lens"], s["kv_lens"], s["starts"],
                     1 / 24, mode)


def _one_bad_row(s, bad, kind):
    """Feature 100 of one head of the second sequence's first token is `bad`: that row is no number, all others are right."""
    want, room = _want(s)
    token = s["starts"][1]
    s["q"].view(-1, *s["q"].shape[-2:])[token, 3, 100] = bad
    with kernel(kind):
        got = [g.reshape(w.shape).clone() for g, w in zip(call(s), want)]
    for g, name in zip(got, ("out", "max", "sum")):
        assert torch.isnan(g[token, 3]).all(), name
    for g, w in zip(got, want):
        g[token, 3] = w[token, 3].to(g.dtype)
    check(got, want, room, kind)


@pytest.mark.parametrize("kind", KERNELS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("tokens", [1, 2, 3])
@pytest.mark.parametrize("length", [5, 100, 128, 129, 290])
def test_a_query_that_is_not_a_number_spoils_its_row_at_any_length(kind, bad, tokens, length):
    s = make(length, "BSND", [tokens] * 3, [length + 3, length, length + 40], 16, 64, 0)
    first = rows_of(s["table"], 1, torch.tensor([0], device="cuda"), 64, s["cache"].shape[0])
    s["cache"].view(-1, 512)[first, 100] = 1.0          # (infinite queries: a score is +inf)
    _one_bad_row(s, bad, kind)
