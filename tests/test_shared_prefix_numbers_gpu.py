"""shared_prefix_attention where numbers end: queries, keys and scores that are not finite, exact scores, weights that fp16 hardly
holds, sequences that take no part."""
import pytest
import torch

from tests.latent_ref import rows_of
from tests.test_shared_prefix_gpu import KERNELS, call, check, kernel, make, reference, verify

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


@pytest.mark.parametrize("kind", KERNELS)
@pytest.mark.parametrize("tokens", [1, 2])
@pytest.mark.parametrize("length", [3, 100, 129, 1000, 20000])
def test_scores_of_minus_infinity_alone_are_no_number(kind, tokens, length):
    """Every key's feature 100 is negative, the query's is infinite: 0 / 0, not a row that sees nothing."""
    s = make(length, "BSND", [tokens] * 3, [length + 3, length, length + 40], 16, 64, 0)
    s["cache"][..., 100] = -s["cache"][..., 100].abs() - 1
    _one_bad_row(s, float("inf"), kind)


@pytest.mark.parametrize("kind", KERNELS)
@pytest.mark.parametrize("bad", [float("inf"), float("-inf")])
def test_an_infinite_key_that_weighs_nothing_shows_in_its_column(kind, bad):
    """Packed rows with one key of their own, whose score is -inf for some heads: 0 x infinity in the column of the value."""
    lens = [641 + (i % 3) for i in range(70)]
    hit = [b for b in (0, 33, 69)]
    assert all(lens[b] == 641 for b in hit)
    s = make(50, "BSND", [1] * 70, lens, 8, 64, 640)
    want, room = _want(s)
    without = reference(s["q"][:, 0], s["qr"][:, 0], s["cache"], s["rope"], s["table"], [1] * 70, [640] * 70, s["starts"], 1 / 24, 0)
    for b in hit:
        row = rows_of(s["table"], b, torch.tensor([640], device="cuda"), 64, s["cache"].shape[0])
        s["cache"].view(-1, 512)[row, 77] = bad
    with kernel(kind):
        got = [g.reshape(w.shape) for g, w in zip(call(s), want)]
    others = torch.ones(70, dtype=torch.bool, device="cuda")
    others[hit] = False
    check([g[others] for g in got], [w[others] for w in want], [r[others] for r in room], kind)
    low = torch.stack([s["q"][b, 0, :, 77].float() * bad < 0 for b in hit])       # heads whose score is -inf
    assert low.any() and not low.all()
    assert torch.isnan(got[0][hit][~low]).all() and torch.isnan(got[1][hit][~low]).all() and torch.isnan(got[2][hit][~low]).all()
    o = got[0][hit][low]
    assert torch.isnan(o[:, 77]).all()
    keep = torch.arange(512, device="cuda") != 77
    diff = (o[:, keep].double() - without[0][0][hit][low][:, keep]).abs()
    assert (diff <= without[1][0][hit][low][:, keep]).all()
    for k in (1, 2):
        assert ((got[k][hit][low].double() - without[0][k][hit][low]).abs() <= without[1][k][hit][low]).all()


@pytest.mark.parametrize("kind", KERNELS)
@pytest.mark.parametrize("layout", ["BSND", "TND"])
@pytest.mark.parametrize("stale", [-1, 0, 2**31 - 1])
def test_sequences_without_query_tokens_do_not_lend_the_prefix(kind, layout, stale):
    """Idle slots of a batch with lengths and table rows of before: the longest sequences, and their pages hold something else."""
    q_lens = [1] * 75
    kv = [700 + i % 50 for i in range(75)]
    s = make(51, layout, q_lens, kv, 8, 64, 640)
    blocks = s["cache"].shape[0]
    for b in (0, 20, 74):
        kv[b] = 800
        s["table"][b] = stale if stale else blocks - 1
    if layout == "BSND":
        for b in (0, 20, 74):
            q_lens[b] = 0
    else:
        for b in (0, 20, 74):
            q_lens[b] = 0
        ends = torch.tensor(q_lens).cumsum(0).tolist()
        s["starts"], s["seq_q"] = [0] + ends[:-1], ends
        s["q"], s["qr"] = s["q"][:ends[-1]].contiguous(), s["qr"][:ends[-1]].contiguous()
    verify(s, kind)


@pytest.mark.parametrize("kind", KERNELS)
def test_a_longer_sequence_of_many_tokens_beside_packed_ones(kind):
    """What is promised past the shorter sequences' ends: the packed ones meet as much as they see."""
    q_lens = [2] * 75 + [60]
    s = make(52, "TND", q_lens, [700 + i % 3 for i in range(75)] + [1500], 8, 64, 704)
    for prefix in (640, 701, 704, 1400):
        verify(s, kind, prefix=prefix)


@pytest.mark.parametrize("kind", KERNELS)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_exact_scores_keep_their_maximum(kind, dtype):
    """Queries with one feature: a score is one product, exact in 32 bits, and so is its product with a power of two.  What is left
    of a maximum's error: the score in units of log2 and its way back are rounded once each (2^-24), and the two constants
    are the nearest 32-bit numbers to log2 e and ln 2 (off by 1.4e-8 and 0.3e-8): below 2.5 x 2^-24."""
    s = make(53, "BSND", [1] * 40, [900 + 3 * i for i in range(40)], 16, 64, 0, dtype)
    s["q"].zero_()
    s["qr"].zero_()
    for h in range(16):
        s["q"][:, 0, h, 32 * h + 5] = 1.5 + h / 8
    flat = s["q"][:, 0].double()
    with kernel(kind):
        out, top, total = call(s, scale=0.25)
    worst = 0.0
    for b, n in enumerate(s["kv_lens"]):
        row = rows_of(s["table"], b, torch.arange(n, device="cuda"), 64, s["cache"].shape[0])
        score = flat[b] @ s["cache"].view(-1, 512)[row].double().T * 0.25
        m = score.amax(1)
        worst = max(worst, float(((top[b, 0, 0].double() - m).abs() / m.abs()).max()))
    assert worst <= 2.5 * 2.0**-24, worst * 2**24


@pytest.mark.parametrize("kind", KERNELS)
@pytest.mark.parametrize("below", [12.0, 14.0, 18.0])
def test_a_long_tail_under_one_dominant_key_in_fp16(kind, below):
    """4000 keys some nats below the first, which is zero as a value: the output is what the tail weighs.  P has to hold the
    tail's weights at half a step of fp16, or of its smallest numbers 2^7 below the largest of P: 2^-25 x 2^-7 a key."""
    n, B, H = 4000, 80, 128
    g = torch.Generator(device="cuda").manual_seed(54)
    table = torch.arange(63, device="cuda", dtype=torch.int32).repeat(B, 1)
    cache = (8 + torch.randn(63, 64, 1, 512, generator=g, device="cuda")).half()
    rope = torch.zeros(63, 64, 1, 64, device="cuda", dtype=torch.float16)
    rope.view(-1, 64)[:, 0] = -below - torch.randint(0, 64, (63 * 64,), generator=g, device="cuda") / 256
    cache.view(-1, 512)[0], rope.view(-1, 64)[0] = 0.0, 0.0
    q, qr = torch.zeros(B, 1, H, 512, device="cuda").half(), torch.zeros(B, 1, H, 64, device="cuda").half()
    qr[..., 0] = 1.0
    s = dict(q=q, qr=qr, cache=cache, rope=rope, table=table, q_lens=[1] * B, kv_lens=[n] * B, starts=list(range(B)), seq_q=[1] * B,
             layout="BSND", prefix=0)
    with kernel(kind):
        out = call(s, scale=1.0)[0].view(B * H, 512).double()
    score, v = rope.view(-1, 64)[:n, 0].double(), cache.view(-1, 512)[:n].double()
    e = torch.exp(score)
    want = (e[:, None] * v).sum(0) / e.sum()
    eps = torch.finfo(torch.float16).eps
    # scores are exact up to the two roundings of their product with the scale, at most 20 x 2^-23; 32-bit sums as elsewhere
    rel = eps / 2 + 20 * 2.0**-23 + (n / 16 + 64) * 2.0**-23
    room = 1.05 * ((rel + eps / 2) * want + 2.0**-32 * v.sum(0) / e.sum()) + 2.0**-25
    off = (out - want).abs() / room
    assert off.max() <= 1, float(off.max())


@pytest.mark.parametrize("kind", KERNELS)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_scores_whose_steps_are_as_large_as_the_guard(kind, dtype):
    """Scores around 4e7, where 32-bit numbers are 4 apart, that climb by 0 to 16 from tile to tile: outputs stay between the
    smallest and the largest value (a weight past the type's largest number would be infinite)."""
    n, B, H = 4000, 80, 128
    g = torch.Generator(device="cuda").manual_seed(55)
    dt = {"bf16": torch.bfloat16, "fp16": torch.float16}[dtype]
    table = torch.arange(16 * 63, device="cuda", dtype=torch.int32).view(16, 63).repeat(5, 1)
    cache = torch.rand(16 * 63, 64, 1, 512, generator=g, device="cuda").to(dt)
    rope = torch.zeros(16, 63 * 64, 64, device="cuda", dtype=dt)
    climb = (4 * torch.randint(0, 5, (16, 32), generator=g, device="cuda")).cumsum(1).repeat_interleave(128, 1)[:, :63 * 64]
    rope[..., 0] = 1220.0
    rope[..., 1], rope[..., 2] = climb // 128, climb % 128           # (exact in either type)
    q, qr = torch.zeros(B, 1, H, 512, device="cuda").to(dt), torch.zeros(B, 1, H, 64, device="cuda").to(dt)
    qr[..., 0], qr[..., 1], qr[..., 2] = 32768.0, 128.0, 1.0
    s = dict(q=q, qr=qr, cache=cache, rope=rope.view(16 * 63, 64, 1, 64), table=table, q_lens=[1] * B, kv_lens=[n] * B,
             starts=list(range(B)), seq_q=[1] * B, layout="BSND", prefix=0)
    with kernel(kind):
        out, top, total = call(s, scale=1.0)
    assert torch.isfinite(out).all() and torch.isfinite(top).all() and torch.isfinite(total).all()
    assert (out >= 0).all() and (out <= 1 + 2.0**-7).all() and (total >= 1 - 2.0**-10).all()
