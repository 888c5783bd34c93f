"""shared_prefix_attention against a 64-bit softmax over each sequence's visible keys, on both kernels."""
import contextlib

import pytest
import torch

from tests.latent_ref import inv_freq, paged, rows_of

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
KERNELS = ["portable", "tensor"]


@contextlib.contextmanager
def kernel(kind):
    from dsa_triton_ascend_b200 import prefix_attention as m
    m.set_kernel(kind)
    try:
        yield
    finally:
        m.set_kernel("auto")


def reference(q, qr, cache, rope, table, q_lens, kv_lens, starts, scale, mode):
    """Output and statistics in 64 bits over flat tokens, and what a kernel may be off by:
    - scores: 576 products summed in 32 bits, by a step of 2^-23 of the sum of magnitudes per 16 of them and the scale's two
      roundings; a weight is off by twice the largest of its row,
    - P is rounded once (half a step, or half the smallest number of fp16), P V summed in 32 bits (2^-23 per 16 keys, and
      the parts of a row joined), the result rounded once."""
    T, H = q.shape[:2]
    page, blocks = cache.shape[1], cache.shape[0]
    out = torch.zeros(T, H, 512, dtype=torch.float64, device="cuda")
    top, total = (torch.zeros(T, H, dtype=torch.float64, device="cuda") for _ in range(2))
    room, room_top, room_total = torch.zeros_like(out), torch.zeros_like(top), torch.zeros_like(top)
    info = torch.finfo(q.dtype)
    c, r = cache.view(-1, 512), rope.view(-1, 64)
    for b, (n, length) in enumerate(zip(q_lens, kv_lens)):
        length = min(length, table.shape[1] * page)
        for i in range(n):
            seen = min(length, kv_lens[b] - n + i + 1) if mode == 3 else length
            if seen <= 0:
                continue
            t = starts[b] + i
            row = rows_of(table, b, torch.arange(seen, device="cuda"), page, blocks)
            here = (row >= 0)[:, None]
            v = torch.where(here, c[row.clamp_min(0)].double(), 0.0)
            k = torch.cat([v, torch.where(here, r[row.clamp_min(0)].double(), 0.0)], 1)
            x = torch.cat([q[t], qr[t]], -1).double()
            s = x @ k.T * scale
            size = (x.abs() @ k.abs().T).amax(1) * abs(scale)
            ds = (36 + 4) * 2.0**-23 * size
            m = s.amax(1)
            e = torch.exp(s - m[:, None])
            z = e.sum(1)
            w = e / z[:, None]
            out[t], top[t], total[t] = w @ v, m, z
            a = w @ v.abs()
            tiny = info.tiny * info.eps / 2 * v.abs().sum(0)[None] / z[:, None]
            rel = info.eps / 2 + 2 * ds + (seen / 16 + 64) * 2.0**-23
            room[t] = 1.05 * (rel[:, None] * a + tiny + info.eps / 2 * out[t].abs()) + info.tiny * info.eps
            room_top[t] = ds + 1e-6
            room_total[t] = z * (2 * ds + (seen / 16 + 64) * 2.0**-23)
    return (out, top, total), (room, room_top, room_total)


def check(got, want, room, what=""):
    for name, g, w, r in zip(("out", "max", "sum"), got, want, room):
        g = g.reshape(w.shape).double()
        assert torch.isfinite(g).all(), f"{what} {name}: {int((~torch.isfinite(g)).sum())} values are not finite"
        bad = (g - w).abs() > r
        assert not bad.any(), f"{what} {name}: {int(bad.sum())} of {bad.numel()} off, worst {float(((g - w).abs() / r.clamp_min(1e-30)).max()):.2f} x"


def make(seed, layout, q_lens, kv_lens, heads, page, prefix, dtype="bf16", s1=None, tail=0, q_scale=2.0, spare=3):
    """A batch whose first min(prefix, length) positions are the same tokens; slots that hold no token are NaN."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, whole = DT[dtype], prefix // page
    table, blocks = paged(g, [max(0, n) for n in kv_lens], page, whole if any(n >= prefix for n in kv_lens) else 0, spare=spare)
    rnd = lambda *s, scale=1.0: (torch.randn(*s, generator=g, device="cuda") * scale).to(dt)
    cache, rope = (torch.full((blocks, page, 1, w), float("nan"), device="cuda", dtype=dt) for w in (512, 64))
    first = rnd(prefix, 576)
    for b, n in enumerate(kv_lens):
        if n <= 0:
            continue
        row = rows_of(table, b, torch.arange(n, device="cuda"), page, blocks)
        x = torch.cat([first[:n], rnd(max(0, n - prefix), 576)])
        cache.view(-1, 512)[row], rope.view(-1, 64)[row] = x[:, :512], x[:, 512:]
    if layout == "TND":
        ends = torch.tensor(q_lens).cumsum(0).tolist()
        starts, lead, seq_q = [0] + ends[:-1], (ends[-1] + tail,), ends
    else:
        s1 = s1 or max(q_lens)
        starts, lead, seq_q = [b * s1 for b in range(len(q_lens))], (len(q_lens), s1), q_lens
    return dict(q=rnd(*lead, heads, 512, scale=q_scale), qr=rnd(*lead, heads, 64, scale=q_scale), cache=cache, rope=rope,
                table=table, q_lens=q_lens, kv_lens=kv_lens, starts=starts, seq_q=seq_q, layout=layout, prefix=prefix)


def call(s, scale=1 / 24, mode=3, prefix=None, lse=True):
    from dsa_triton_ascend_b200 import shared_prefix_attention
    return shared_prefix_attention(
        s["q"], s["cache"], scale_value=scale, block_table=s["table"], actual_seq_lengths_query=s["seq_q"],
        actual_seq_lengths_kv=s["kv_lens"], query_rope=s["qr"], key_rope=s["rope"],
        shared_prefix_length=s["prefix"] if prefix is None else prefix, layout_query=s["layout"], sparse_mode=mode,
        return_softmax_lse=lse)


def verify(s, kind, scale=1 / 24, mode=3, prefix=None):
    from dsa_triton_ascend_b200 import check_status
    flat = lambda t: t.reshape(-1, *t.shape[-2:])
    want, room = reference(flat(s["q"]), flat(s["qr"]), s["cache"], s["rope"], s["table"], s["q_lens"], s["kv_lens"],
                           s["starts"], scale, mode)
    with kernel(kind):
        got = call(s, scale, mode, prefix)
        check_status()
    check(got, want, room, kind)
    return got


@pytest.mark.parametrize("kind", KERNELS)
@pytest.mark.parametrize("heads", [1, 5, 16, 64, 128, 130, 200])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_decode_step(kind, heads, dtype):
    verify(make(heads, "BSND", [1] * 6, [300, 257, 700, 301, 512, 256], heads, 64, 256, dtype), kind)


@pytest.mark.parametrize("kind", KERNELS)
@pytest.mark.parametrize("page", [1, 8, 16, 24, 32, 48, 64, 100, 128, 256])
@pytest.mark.parametrize("prefix", [0, 500, 768])
def test_pages(kind, page, prefix):
    verify(make(page, "BSND", [1] * 5, [prefix + n for n in (1, 17, 128, 300, 515)], 16, page, prefix), kind)


@pytest.mark.parametrize("kind", KERNELS)
@pytest.mark.parametrize("prefix", [1, 15, 16, 63, 64, 127, 128, 129, 255, 256, 257, 511, 1000, 1024, 2049])
def test_prefix_lengths(kind, prefix):
    verify(make(prefix, "BSND", [1, 1, 1], [prefix + 1, prefix + 200, prefix], 32, 64, prefix), kind)


@pytest.mark.parametrize("kind", KERNELS)
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 64, 127, 128, 129, 255, 256, 1281])
def test_one_sequence(kind, length):
    verify(make(length, "BSND", [1], [length], 128, 64, 0), kind)
    verify(make(length, "BSND", [1], [length], 3, 16, length), kind)


@pytest.mark.parametrize("kind", KERNELS)
@pytest.mark.parametrize("mode", [0, 3])
@pytest.mark.parametrize("layout", ["BSND", "TND"])
@pytest.mark.parametrize("heads", [1, 8, 20, 64, 128])
def test_several_tokens(kind, mode, layout, heads):
    """Tokens of a sequence see different numbers of keys; row tiles end inside a token and inside a sequence."""
    q_lens = [3, 1, 9, 2, 33] if layout == "TND" else [3, 1, 2, 3, 3]
    verify(make(heads, layout, q_lens, [600 + 3, 512 + 1, 700, 513, 512 + 33], heads, 64, 512), kind, mode=mode)


@pytest.mark.parametrize("kind", KERNELS)
@pytest.mark.parametrize("heads", [4, 64])
def test_padded_batches(kind, heads):
    """Sequences without tokens, rows past a sequence's query length, rows behind the last sequence, keys of length 0, more new
    tokens than keys: rows that see nothing are zeros."""
    s = make(1, "BSND", [2, 0, 4, 1], [400, 300, 2, 0], heads, 16, 300, s1=5)
    got = verify(s, kind)
    assert not got[0].view(4, 5, heads, 512)[1].any() and not got[0].view(4, 5, heads, 512)[2, :2].any()
    s = make(2, "TND", [2, 0, 4, 1], [400, 300, 2, 0], heads, 16, 300, tail=7)
    got = verify(s, kind)
    assert not got[0][7:].any() and not got[1][0, 7:].any() and not got[2][0, 7:].any()


@pytest.mark.parametrize("kind", KERNELS)
@pytest.mark.parametrize("prefix", [200, 600, 5000])
def test_sequences_shorter_than_the_prefix(kind, prefix):
    """The longest one may be shorter itself."""
    verify(make(prefix, "BSND", [1] * 5, [10, 900, 599, 601, 199], 16, 64, 600), kind, prefix=prefix)


@pytest.mark.parametrize("kind", KERNELS)
def test_a_promise_of_less_than_what_is_shared(kind):
    s = make(3, "BSND", [1] * 9, [700 + 30 * i for i in range(9)], 16, 64, 640)
    a = verify(s, kind)
    for prefix in (0, 1, 333, 576):
        b = verify(s, kind, prefix=prefix)
        assert (a[0].float() - b[0].float()).abs().max() < 0.05


@pytest.mark.parametrize("kind", KERNELS)
@pytest.mark.parametrize("heads", [16, 128])
def test_absent_blocks_read_as_zero_keys(kind, heads):
    s = make(4, "BSND", [1] * 4, [700, 650, 900, 513], heads, 64, 512)
    blocks = s["cache"].shape[0]
    s["table"][:, 2] = -1                   # inside the prefix, for everybody
    s["table"][1, 9] = blocks               # beyond the cache
    s["table"][2, 12] = 2**31 - 1
    s["table"][0, 8] = -7
    verify(s, kind)


@pytest.mark.parametrize("kind", KERNELS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("layout", ["BSND", "TND"])
def test_values_in_masked_places_do_not_count(kind, bad, layout):
    """The last token's own key and value are not finite: the tokens before it, which share its tiles, do not see it."""
    q_lens = [3, 3, 3]
    s = make(5, layout, q_lens, [403, 260, 515], 16, 64, 256)
    for b, n in enumerate(s["kv_lens"]):
        if b == 1:
            continue
        row = rows_of(s["table"], b, torch.tensor([n - 1], device="cuda"), 64, s["cache"].shape[0])
        s["cache"].view(-1, 512)[row, 5] = bad
    flat = lambda t: t.reshape(-1, *t.shape[-2:])
    want, room = reference(flat(s["q"]), flat(s["qr"]), s["cache"], s["rope"], s["table"], q_lens, s["kv_lens"], s["starts"],
                           1 / 24, 3)
    with kernel(kind):
        got = [g.reshape(w.shape) for g, w in zip(call(s), want)]
    sees = torch.tensor([False, False, True] + [False] * 3 + [False, False, True], device="cuda")
    check([g[~sees] for g in got], [w[~sees] for w in want], [r[~sees] for r in room], kind)
    assert not torch.isfinite(got[0][sees][..., 5]).any()


@pytest.mark.parametrize("kind", KERNELS)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("order", ["rising", "falling", "one"])
def test_scores_that_outgrow_the_first_tile(kind, dtype, order):
    """Later keys score higher by far more than any power of two that a type holds; or the first ones do."""
    s = make(6, "BSND", [1] * 3, [1300, 1025, 1290], 32, 64, 1024, dtype)
    n = 1300
    gain = {"rising": torch.linspace(0, 8, n), "falling": torch.linspace(8, 0, n),
            "one": torch.zeros(n).index_fill_(0, torch.tensor([777]), 9.0)}[order].cuda()
    u = torch.nn.functional.normalize(torch.randn(512, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda"), dim=0)
    s["q"] = (s["q"].float() * 0.3 + 20 * u).to(s["q"].dtype)
    for b, length in enumerate(s["kv_lens"]):
        row = rows_of(s["table"], b, torch.arange(length, device="cuda"), 64, s["cache"].shape[0])
        if b == 0:
            lo = 0
        else:
            lo, row = 1024, row[1024:]
        c = s["cache"].view(-1, 512)
        c[row] = (c[row].float() * 0.5 + gain[lo:length, None] * u).to(c.dtype)
    verify(s, kind, scale=1.0)


@pytest.mark.parametrize("kind", KERNELS)
def test_scale_zero_negative_and_large(kind):
    s = make(7, "BSND", [1] * 3, [300, 129, 513], 16, 16, 128)
    for scale in (0.0, -1 / 24, 1.0):
        verify(s, kind, scale=scale)


@pytest.mark.parametrize("kind", KERNELS)
def test_statistics_that_are_not_asked_for_are_zeros(kind):
    s = make(8, "BSND", [1] * 5, [300, 129, 513, 0, 200], 16, 16, 128)
    with kernel(kind):
        a, b = call(s), call(s, lse=False)
    assert torch.equal(a[0], b[0]) and not b[1].any() and not b[2].any()
    assert b[1].shape == a[1].shape == (5, 1, 1, 16)


@pytest.mark.parametrize("kind", KERNELS)
def test_strided_and_unaligned_operands(kind):
    s = make(9, "BSND", [1] * 3, [300, 129, 513], 16, 64, 128)
    want = verify(s, kind)
    both = torch.cat([s["q"], s["qr"]], -1)
    flat = torch.empty(s["rope"].numel() + 1, device="cuda", dtype=s["rope"].dtype)
    flat[1:] = s["rope"].view(-1)
    t = dict(s, q=both[..., :512], qr=both[..., 512:], rope=flat[1:].view(s["rope"].shape),
             cache=torch.cat([s["cache"], s["cache"]], -1)[..., :512])
    with kernel(kind):
        got = call(t)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("kind", KERNELS)
def test_many_sequences_and_long_ones(kind):
    lens = [1100 + (37 * i) % 640 for i in range(40)]
    verify(make(10, "BSND", [1] * 40, lens, 16, 64, 1088), kind)
    verify(make(11, "BSND", [1] * 2, [20000, 9000], 8, 128, 8999), kind)


@pytest.mark.parametrize("page", [1, 8, 16, 24, 32, 48, 64, 100, 128])
@pytest.mark.parametrize("prefix", [500, 768])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_packed_rows_over_pages(page, prefix, dtype):
    """Enough sequences of few rows that they meet the prefix together, in tiles that mix sequences."""
    lens = [prefix + 1 + (13 * i) % 300 for i in range(200)]
    verify(make(page, "BSND", [1] * 200, lens, 2, page, prefix, dtype), "tensor")


@pytest.mark.parametrize("prefix", [255, 256, 257, 383, 384, 1000, 1024, 2049])
@pytest.mark.parametrize("heads,batch", [(3, 299), (64, 150), (20, 290)])
def test_packed_rows_behind_prefixes(prefix, heads, batch):
    lens = [prefix + (7 * i) % 200 for i in range(batch)]       # (some hold nothing but the prefix)
    verify(make(prefix, "BSND", [1] * batch, lens, heads, 64, prefix), "tensor")


@pytest.mark.parametrize("layout", ["BSND", "TND"])
@pytest.mark.parametrize("mode", [0, 3])
def test_packed_rows_beside_others(layout, mode):
    """Sequences of one to three tokens, of none, of a whole chunk, shorter than the prefix, without keys: packed ones between them."""
    q_lens = [1 + i % 3 for i in range(80)]
    kv = [900 + (11 * i) % 333 for i in range(80)]
    q_lens[5], q_lens[17], kv[9], kv[21], kv[40] = 0, 3 if layout == "BSND" else 40, 512, 3, 0
    verify(make(31, layout, q_lens, kv, 8, 64, 896, s1=4 if layout == "BSND" else None, tail=5 if layout == "TND" else 0),
           "tensor", mode=mode)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_values_in_masked_places_of_packed_rows(bad):
    q_lens, kv = [2] * 70, [700 + i for i in range(70)]
    s = make(32, "BSND", q_lens, kv, 8, 16, 640)
    for b in (0, 33, 69):
        row = rows_of(s["table"], b, torch.tensor([kv[b] - 1], device="cuda"), 16, s["cache"].shape[0])
        s["cache"].view(-1, 512)[row, 77] = bad
    flat = lambda t: t.reshape(-1, *t.shape[-2:])
    want, room = reference(flat(s["q"]), flat(s["qr"]), s["cache"], s["rope"], s["table"], q_lens, kv, s["starts"], 1 / 24, 3)
    got = [g.reshape(w.shape) for g, w in zip(call(s), want)]
    sees = torch.zeros(140, dtype=torch.bool, device="cuda")
    sees[[1, 67, 139]] = True
    check([g[~sees] for g in got], [w[~sees] for w in want], [r[~sees] for r in room])
    assert not torch.isfinite(got[0][sees][..., 77]).any()


def test_absent_blocks_of_packed_rows():
    s = make(33, "BSND", [1] * 70, [700 + i for i in range(70)], 8, 64, 640)
    s["table"][:, 3] = -1
    s["table"][7, 10] = s["cache"].shape[0]
    verify(s, "tensor")


def test_packed_scores_that_outgrow_the_first_tile():
    s = make(34, "BSND", [1] * 70, [1300 + i for i in range(70)], 8, 64, 1280)
    u = torch.nn.functional.normalize(torch.randn(512, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda"), dim=0)
    s["q"] = (s["q"].float() * 0.3 + 20 * u).to(s["q"].dtype)
    row = rows_of(s["table"], 0, torch.arange(1280, device="cuda"), 64, s["cache"].shape[0])
    c = s["cache"].view(-1, 512)
    c[row] = (c[row].float() * 0.5 + torch.linspace(0, 8, 1280, device="cuda")[:, None] * u).to(c.dtype)
    verify(s, "tensor", scale=1.0)


def test_the_longest_sequence_lends_the_prefix():
    """The pages of the others hold other numbers where the prefix would be: what counts is the first of the longest ones'."""
    s = make(35, "BSND", [1] * 70, [700] * 30 + [900] + [701] * 39, 8, 64, 640)
    got = call(s)
    s["table"][:30, :10] = s["table"][30, 10]
    s["table"][31:, :10] = -1
    assert all(torch.equal(a, b) for a, b in zip(call(s), got))


def test_single_tokens_of_many_small_sequences():
    """130 sequences of one head: a row tile holds rows of 128 sequences."""
    lens = [257 + i for i in range(130)]
    verify(make(12, "BSND", [1] * 130, lens, 1, 16, 257), "tensor")
    lens[3] = lens[50] = 0
    lens[129] = 5
    verify(make(13, "BSND", [1] * 130, lens, 1, 16, 257), "tensor")


@pytest.mark.parametrize("heads,batch,own", [(128, 20, 300), (16, 70, 260), (32, 3, 2000)])
def test_same_call_same_bits(heads, batch, own):
    s = make(14, "BSND", [1] * batch, [1024 + own + i for i in range(batch)], heads, 64, 1024)
    a = call(s)
    for _ in range(5):
        assert all(torch.equal(x, y) for x, y in zip(a, call(s)))


def test_offsets_past_32_bits():
    """Pages at the end of a cache of 5 GB: byte offsets above 2^32."""
    s = make(15, "BSND", [1] * 3, [300, 500, 257], 16, 64, 256)
    blocks, small = 78000, s["cache"].shape[0]
    cache = torch.zeros(blocks, 64, 1, 512, device="cuda", dtype=torch.bfloat16)
    rope = torch.zeros(blocks, 64, 1, 64, device="cuda", dtype=torch.bfloat16)
    cache[-small:], rope[-small:] = s["cache"], s["rope"]
    want = {k: verify(s, k) for k in KERNELS}
    table = torch.where(s["table"] >= 0, s["table"] + (blocks - small), s["table"])
    for k in KERNELS:
        with kernel(k):
            got = call(dict(s, cache=cache, rope=rope, table=table))
        assert all(torch.equal(a, b) for a, b in zip(got, want[k]))


def test_the_prefix_length_can_live_on_the_device():
    """A captured call follows lengths, tables, queries and the prefix length that change in place."""
    from dsa_triton_ascend_b200 import shared_prefix_attention
    s = make(16, "BSND", [1] * 9, [700 + 41 * i for i in range(9)], 16, 64, 640)
    prefix = torch.tensor([640], dtype=torch.int32, device="cuda")
    lens = torch.tensor(s["kv_lens"], dtype=torch.int32, device="cuda")
    f = lambda p: shared_prefix_attention(s["q"], s["cache"], scale_value=1 / 24, block_table=s["table"],
                                          actual_seq_lengths_kv=lens, query_rope=s["qr"], key_rope=s["rope"],
                                          shared_prefix_length=p, return_softmax_lse=True)
    f(prefix)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = f(prefix)
    for p, short in ((640, 0), (0, 3), (256, 60), (5000, 1), (-5, 2), (640, 699)):
        prefix.fill_(p)
        lens.copy_(torch.tensor(s["kv_lens"]) - short)
        s["q"].mul_(-1)
        graph.replay()
        t = dict(s, kv_lens=[n - short for n in s["kv_lens"]])
        flat = lambda x: x.reshape(-1, *x.shape[-2:])
        want, room = reference(flat(s["q"]), flat(s["qr"]), s["cache"], s["rope"], s["table"], s["q_lens"], t["kv_lens"],
                               s["starts"], 1 / 24, 3)
        check(held, want, room, str(p))


@pytest.mark.parametrize("kind", KERNELS)
def test_tables_without_columns_and_batches_without_keys(kind):
    s = make(40, "BSND", [2] * 3, [50, 60, 70], 16, 16, 48)
    for t in (dict(s, table=s["table"][:, :0]), dict(s, kv_lens=[0, 0, 0]), dict(s, kv_lens=[-3, 0, -1]), dict(s, seq_q=[0, 0, 0])):
        with kernel(kind):
            got = call(t)
        assert not any(g.any() for g in got)


@pytest.mark.parametrize("kind", KERNELS)
def test_lengths_past_the_table(kind):
    """Positions behind the table's last block do not exist."""
    s = make(41, "BSND", [1] * 3, [300, 200, 320], 16, 16, 0)
    s["table"] = s["table"][:, :20].contiguous()
    lens = [2**31 - 1, 200, 5000]
    want, room = reference(s["q"][:, 0], s["qr"][:, 0], s["cache"], s["rope"],
                           torch.where(s["table"] >= 0, s["table"], torch.full_like(s["table"], 10**6)), [1] * 3, [320, 200, 320],
                           [0, 1, 2], 1 / 24, 3)
    s["table"][0, 19] = s["table"][1, 13:] = -1        # (blocks that were never filled: absent)
    with kernel(kind):
        got = call(dict(s, kv_lens=lens))
    got = [g.reshape(w.shape) for g, w in zip(got, want)]
    check([g[2:] for g in got], [w[2:] for w in want], [r[2:] for r in room], kind)
    # sequence 0 claims positions 300 .. 303 of its 19th block, which no token filled: they hold NaN and are visible
    assert torch.isnan(got[0][0]).all() and torch.isfinite(got[0][1:]).all()


@pytest.mark.parametrize("heads", [3, 33, 70, 128])
@pytest.mark.parametrize("batch,length", [(1, 20000), (1, 9473), (2, 12000), (3, 7001), (4, 6100), (5, 5200), (9, 3500)])
def test_few_rows_in_many_parts(heads, batch, length):
    """Rows with parts from one share, from every share, and from a few, with the parts joined by one warp and by eight."""
    verify(make(heads + batch, "BSND", [1] * batch, [length - 131 * i for i in range(batch)], heads, 64, 0), "tensor")


@pytest.mark.parametrize("layout", ["BSND", "TND"])
@pytest.mark.parametrize("prefix", [0, 640])
@pytest.mark.parametrize("batch", [31, 58, 60, 61, 62, 63, 64, 65, 80])
def test_around_the_row_tiles_that_are_planned_without_a_kernel(layout, prefix, batch):
    """One token and eight heads a sequence; some sequences without keys, or with fewer than the prefix."""
    kv = [prefix + (b * 37) % 290 if b % 7 else b % 3 * 100 for b in range(batch)]
    verify(make(batch, layout, [1] * batch, kv, 8, 64, prefix), "tensor")


@pytest.mark.parametrize("layout", ["BSND", "TND"])
@pytest.mark.parametrize("batch", [1, 2, 8, 16, 17])
def test_few_packed_rows_in_many_parts(layout, batch):
    s = make(batch, layout, [1 + b % 2 for b in range(batch)], [9000 + 37 * b for b in range(batch)], 8, 64, 8192)
    a, b = verify(s, "tensor"), verify(s, "tensor")
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("kind", KERNELS)
@pytest.mark.parametrize("heads", [16, 128])
def test_a_query_that_is_not_a_number_spoils_its_own_row_only(kind, heads):
    s = make(42, "BSND", [2] * 3, [300, 290, 310], heads, 64, 256)
    flat = lambda t: t.reshape(-1, *t.shape[-2:])
    want, room = reference(flat(s["q"]), flat(s["qr"]), s["cache"], s["rope"], s["table"], s["q_lens"], s["kv_lens"],
                           s["starts"], 1 / 24, 3)
    s["q"][1, 0, 3, 100] = float("nan")
    with kernel(kind):
        got = [g.reshape(w.shape).clone() for g, w in zip(call(s), want)]
    assert all(torch.isnan(g[2, 3]).all() for g in got)
    for g, w in zip(got, want):
        g[2, 3] = w[2, 3].to(g.dtype)
    check(got, want, room, kind)


@pytest.mark.parametrize("heads,batch", [(256, 3), (300, 2), (16, 700), (1, 1500)])
def test_many_heads_and_many_sequences(heads, batch):
    lens = [130 + (i * 7) % 150 for i in range(batch)]
    verify(make(43, "BSND", [1] * batch, lens, heads, 64, 128), "tensor")


@pytest.mark.parametrize("heads", [16, 128])
def test_a_prompt_of_its_own(heads):
    """One long sequence, every token a query: a causal prefill over the cache."""
    verify(make(44, "TND", [700], [700], heads, 64, 0), "tensor")
    verify(make(45, "TND", [300, 5, 200], [1100, 5, 700], heads, 32, 0), "tensor")


def test_a_captured_call_packs_and_unpacks():
    """The same graph with a prefix that is worth packing, one that is not, and lengths that move."""
    from dsa_triton_ascend_b200 import shared_prefix_attention
    B = 80
    s = make(46, "BSND", [1] * B, [700 + (5 * i) % 90 for i in range(B)], 8, 64, 640)
    prefix = torch.tensor([640], dtype=torch.int32, device="cuda")
    lens = torch.tensor(s["kv_lens"], dtype=torch.int32, device="cuda")
    f = lambda: shared_prefix_attention(s["q"], s["cache"], scale_value=1 / 24, block_table=s["table"], actual_seq_lengths_kv=lens,
                                        query_rope=s["qr"], key_rope=s["rope"], shared_prefix_length=prefix, return_softmax_lse=True)
    f()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = f()
    for p, short in ((640, 0), (128, 5), (0, 1), (640, 50), (9999, 9)):
        prefix.fill_(p)
        lens.copy_(torch.tensor(s["kv_lens"]) - short)
        graph.replay()
        want, room = reference(s["q"][:, 0], s["qr"][:, 0], s["cache"], s["rope"], s["table"], [1] * B,
                               [n - short for n in s["kv_lens"]], list(range(B)), 1 / 24, 3)
        check(held, want, room, str(p))


def test_calls_on_two_streams_at_once():
    a = make(17, "BSND", [1] * 8, [2000 + 64 * i for i in range(8)], 16, 64, 1920)
    b = make(18, "BSND", [1] * 30, [900 + 64 * i for i in range(30)], 64, 64, 832, "fp16")
    want = [call(a), call(b)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        x = call(a)
        with torch.cuda.stream(side):
            y = call(b)
        got.append((x, y))
    torch.cuda.synchronize()
    for x, y in got:
        assert all(torch.equal(p, q) for p, q in zip(x, want[0])) and all(torch.equal(p, q) for p, q in zip(y, want[1]))


def test_append_then_attend_then_index():
    """The operators as a decode loop uses them: rotate and append the new tokens, then attention over the whole cache, against
    sparse attention with every key selected, and the indexer over the appended index keys."""
    from dsa_triton_ascend_b200 import (latent_cache_append, lightning_indexer_triton, rotary_embedding,
                                        shared_prefix_attention, sparse_flash_attention_triton)
    g = torch.Generator(device="cuda").manual_seed(19)
    B, H, page, prefix, bf = 5, 32, 64, 640, torch.bfloat16
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").to(bf)
    longest = prefix + 200
    table, blocks = paged(g, [longest + b for b in range(B)], page, prefix // page)
    caches = [rnd(blocks, page, 1, w) for w in (512, 64, 128)]
    freq = inv_freq()
    lens = torch.tensor([prefix + 20 * b for b in range(B)], dtype=torch.int32, device="cuda")
    # the shared prompt is appended once, through the first sequence
    latent_cache_append(rnd(1, prefix, 1, 512), rnd(1, prefix, 1, 64), *caches[:2], freq, block_table=table[:1],
                        actual_seq_lengths_kv=[prefix], index_key=rnd(1, prefix, 1, 128), index_cache=caches[2],
                        norm_weight=torch.ones(512, device="cuda"))
    for step in range(3):
        lens += 1
        latent_cache_append(rnd(B, 1, 1, 512), rnd(B, 1, 1, 64), *caches[:2], freq, block_table=table, actual_seq_lengths_kv=lens,
                            index_key=rnd(B, 1, 1, 128), index_cache=caches[2], norm_weight=torch.ones(512, device="cuda"))
        q, qr = rnd(B, 1, H, 512), rotary_embedding(rnd(B, 1, H, 192)[..., 128:], (lens - 1)[:, None], freq)
        host = lens.tolist()
        got = shared_prefix_attention(q, caches[0], scale_value=1 / 24, block_table=table, actual_seq_lengths_kv=lens,
                                      query_rope=qr, key_rope=caches[1], shared_prefix_length=prefix, return_softmax_lse=True)
        want, room = reference(q[:, 0], qr[:, 0], caches[0], caches[1], table, [1] * B, host, list(range(B)), 1 / 24, 3)
        check(got, want, room)
        every = torch.arange(max(host), device="cuda", dtype=torch.int32).repeat(B, 1, 1, 1)
        sparse = sparse_flash_attention_triton(q, caches[0], caches[0], every, scale_value=1 / 24, block_table=table,
                                               actual_seq_lengths_kv=lens, query_rope=qr, key_rope=caches[1],
                                               layout_kv="PA_BSND", sparse_mode=3, return_softmax_lse=True)
        assert (got[0].float() - sparse[0].float()).abs().max() < 2e-2
        assert (got[1] - sparse[1]).abs().max() < 1e-3 and ((got[2] / sparse[2]) - 1).abs().max() < 1e-3
        idx, _ = lightning_indexer_triton(rnd(B, 1, 64, 128), caches[2], torch.rand(B, 1, 64, generator=g, device="cuda"),
                                          actual_seq_lengths_key=lens, block_table=table, layout_key="PA_BSND",
                                          sparse_count=1024, sparse_mode=3)
        for b, n in enumerate(host):
            assert sorted(v for v in idx[b, 0, 0].tolist() if v >= 0) == list(range(min(n, 1024)))


def test_module_holds_the_arguments():
    from dsa_triton_ascend_b200 import SharedPrefixAttention
    s = make(20, "TND", [2, 3], [300, 400], 16, 64, 256)
    m = SharedPrefixAttention(scale_value=1 / 24, layout_query="TND", return_softmax_lse=True)
    got = m(s["q"], s["cache"], s["qr"], s["rope"], s["seq_q"], s["kv_lens"], s["table"], 256)
    assert all(torch.equal(a, b) for a, b in zip(got, call(s)))
