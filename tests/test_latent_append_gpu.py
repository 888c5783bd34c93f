"""latent_cache_append against a 64-bit plain form: layouts, page sizes, strides, tokens without a slot, padded batches."""
import pytest
import torch

from tests.latent_ref import inv_freq, paged, rotation_bound, rows_of, turn

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _reference(latent, rope, index, caches, freq, table, q_lens, kv_lens, starts, positions, sections, weight, eps, inter,
               index_inter, index_offset):
    """The caches as float64 and, slot by slot, what each value may be off by; flat tokens, sequence b's from starts[b] on."""
    page, blocks = caches[0].shape[1], caches[0].shape[0]
    want = [c.double().view(-1, c.shape[-1]).clone() if c is not None else None for c in caches]
    room = [torch.zeros_like(w) if w is not None else None for w in want]
    info = torch.finfo(latent.dtype)
    for b, (n, total) in enumerate(zip(q_lens, kv_lens)):
        if n <= 0:
            continue
        at = slice(starts[b], starts[b] + n)
        p = torch.arange(n, device="cuda") + (total - n)
        row = rows_of(table, b, p, page, blocks)
        ok = row >= 0
        row = row[ok]
        turned = p if positions is None else positions[..., at]
        x = latent[at].double()
        if weight is not None:
            x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
        want[0][row] = x[ok, 0]
        # normalised: a sum of 512 squares in 32 bits, a root and two products, below 3e-6; then one rounding
        room[0][row] = (x[ok, 0].abs() * (info.eps / 2 * (1 + 3e-6) + 3e-6) + info.tiny * info.eps) if weight is not None else 0.0
        for k, (t, off, il) in enumerate(((rope, 0, inter), (index, index_offset, index_inter)), 1):
            if t is None:
                continue
            y = turn(t[at], turned, freq, sections, off, il)
            want[k][row] = y[ok, 0]
            room[k][row] = rotation_bound(t[at], y, latent.dtype, 32, off, il)[ok, 0]
    return want, room


def _run(seed, layout, q_lens, kv_lens, page, dtype="bf16", d=512, d_index=128, norm=None, sections=None, inter=True,
         index_inter=False, index_offset=0, s1=None, tail=0, mangle=None, device_lens=True, pos64=False):
    from dsa_triton_ascend_b200 import latent_cache_append
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, B = DT[dtype], len(q_lens)
    table, blocks = paged(g, [max(0, n) for n in kv_lens], page)
    if mangle is not None:
        mangle(table, blocks)
    if layout == "TND":
        ends = torch.tensor(q_lens).cumsum(0).tolist()
        starts, lead = [0] + ends[:-1], (ends[-1] + tail,)
        seq_q = ends
    else:
        s1 = s1 or max(q_lens)
        starts, lead = [b * s1 for b in range(B)], (B, s1)
        seq_q = q_lens
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dt)
    both = rnd(*lead, 1, d + 64)
    latent, rope = both[..., :d], both[..., d:]
    index = rnd(*lead, 1, d_index) if d_index else None
    caches = [rnd(blocks, page, 1, d), rnd(blocks, page, 1, 64), rnd(blocks, page, 1, d_index) if d_index else None]
    weight = None if norm is None else (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dt if norm == "io" else torch.float32)
    positions = None
    if sections is not None:
        positions = torch.randint(0, 9000, (len(sections), *lead), generator=g, device="cuda",
                                  dtype=torch.int64 if pos64 else torch.int32)
    freq = inv_freq()
    flat = lambda t: None if t is None else t.reshape(-1, 1, t.shape[-1])
    want, room = _reference(flat(latent), flat(rope), flat(index), caches, freq, table, q_lens, kv_lens, starts,
                            None if positions is None else positions.reshape(len(sections), -1), sections, weight, 1e-6,
                            inter, index_inter, index_offset)
    lens = (lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")) if device_lens else list
    got = latent_cache_append(
        latent, rope, caches[0], caches[1], freq, block_table=table, actual_seq_lengths_query=lens(seq_q),
        actual_seq_lengths_kv=lens(kv_lens), index_key=index, index_cache=caches[2], positions=positions,
        axis_sections=sections, layout=layout, norm_weight=weight, interleaved=inter, index_interleaved=index_inter,
        index_rotary_offset=index_offset)
    for k, (c, w, r) in enumerate(zip(caches, want, room)):
        assert got[k] is c
        if c is not None:
            bad = (c.double().view(w.shape) - w).abs() > r
            assert not bad.any(), f"cache {k}: {int(bad.sum())} values off"


@pytest.mark.parametrize("page", [1, 16, 24, 64, 100, 128])
@pytest.mark.parametrize("layout", ["BSND", "TND"])
def test_pages_and_layouts(page, layout):
    _run(page, layout, [3, 1, 130, 7], [3, 77, 400, 129], page)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("norm", [None, "io", "fp32"])
@pytest.mark.parametrize("d", [128, 256, 512])
def test_types_norms_and_widths(dtype, norm, d):
    _run(d, "BSND", [2] * 9, [2, 3, 64, 65, 100, 128, 257, 999, 12], 64, dtype=dtype, d=d, norm=norm)


@pytest.mark.parametrize("inter", [True, False])
@pytest.mark.parametrize("index_inter,index_offset,d_index", [(False, 0, 128), (True, 64, 128), (True, 2, 66), (False, 30, 200),
                                                              (False, 0, 64), (False, 0, 0)])
def test_pairs_and_index_keys(inter, index_inter, index_offset, d_index):
    _run(7, "TND", [5, 33], [50, 33], 16, inter=inter, index_inter=index_inter, index_offset=index_offset, d_index=d_index)


@pytest.mark.parametrize("pos64", [False, True])
@pytest.mark.parametrize("sections,layout", [((8, 12, 12), "BSND"), ((32,), "TND"), ((0, 16, 4, 12), "TND")])
def test_positions_from_outside(sections, layout, pos64):
    _run(3, layout, [4, 9, 2], [100, 9, 33], 48, sections=sections, pos64=pos64)


def test_one_token_each_of_a_full_batch():
    _run(4, "BSND", [1] * 130, [1 + 37 * i for i in range(130)], 64, norm="io", device_lens=False)


def test_padded_rows_and_rows_behind_the_last_sequence_are_left_out():
    _run(5, "BSND", [3, 0, 5, 1], [40, 17, 5, 200], 16, s1=9)
    _run(6, "TND", [3, 0, 5, 1], [40, 17, 5, 200], 16, tail=21)


def test_more_new_tokens_than_the_length_counts():
    """The first ones would lie before position 0."""
    _run(8, "BSND", [6, 6], [4, 100], 16)


def test_absent_pages_and_pages_beyond_the_cache():
    def mangle(table, blocks):
        table[0, 1] = -1
        table[1, 0] = blocks
        table[2, 2] = 2**31 - 1
        table[3] = -1
    _run(9, "TND", [40, 40, 40, 40], [64, 40, 100, 40], 16, mangle=mangle)


def test_lengths_past_the_table():
    """Sequence 0 claims 500 tokens, its table has pages for about 100."""
    from dsa_triton_ascend_b200 import latent_cache_append
    page, caches = 16, [torch.zeros(9, 16, 1, w, device="cuda", dtype=torch.bfloat16) for w in (512, 64)]
    table = torch.arange(7, device="cuda", dtype=torch.int32)[None]
    one = lambda w: torch.ones(1, 500, 1, w, device="cuda", dtype=torch.bfloat16)
    latent_cache_append(one(512), one(64), *caches, inv_freq(), block_table=table, actual_seq_lengths_kv=[500])
    assert (caches[0][:7] == 1).all() and (caches[0][7:] == 0).all()


def test_offsets_past_32_bits():
    """The last slots of a cache of 5 GB: element offsets above 2^31."""
    from dsa_triton_ascend_b200 import latent_cache_append
    page, blocks = 128, 40000
    cache = torch.zeros(blocks, page, 1, 512, device="cuda", dtype=torch.bfloat16)
    rope = torch.zeros(blocks, page, 1, 64, device="cuda", dtype=torch.bfloat16)
    table = torch.tensor([[blocks - 1, blocks - 2]], device="cuda", dtype=torch.int32)
    x = torch.randn(1, 200, 1, 512, device="cuda").bfloat16()
    r = torch.randn(1, 200, 1, 64, device="cuda").bfloat16()
    latent_cache_append(x, r, cache, rope, inv_freq(), block_table=table, actual_seq_lengths_kv=[200])
    assert torch.equal(cache[blocks - 1, :, 0], x[0, :128, 0]) and torch.equal(cache[blocks - 2, :72, 0], x[0, 128:, 0])
    assert int(cache[:blocks - 2].count_nonzero()) == 0 and int(cache[blocks - 2, 72:].count_nonzero()) == 0


def test_captured_step_follows_the_lengths():
    from dsa_triton_ascend_b200 import latent_cache_append
    g = torch.Generator(device="cuda").manual_seed(1)
    table, blocks = paged(g, [64, 64], 16)
    lens = torch.tensor([5, 9], dtype=torch.int32, device="cuda")
    x, r = torch.randn(2, 1, 1, 512, device="cuda").half(), torch.randn(2, 1, 1, 64, device="cuda").half()
    caches = [torch.zeros(blocks, 16, 1, w, device="cuda", dtype=torch.float16) for w in (512, 64)]
    step = lambda c: latent_cache_append(x, r, *c, inv, block_table=table, actual_seq_lengths_kv=lens)
    inv = inv_freq()
    step([c.clone() for c in caches])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(caches)
    plain = [c.clone() for c in caches]
    for _ in range(40):
        x.add_(0.125)
        graph.replay()
        step(plain)
        lens += 1
    assert all(torch.equal(a, b) for a, b in zip(caches, plain)) and int(caches[0].count_nonzero()) > 70 * 500


def test_module_holds_the_arguments():
    from dsa_triton_ascend_b200 import LatentCacheAppend, latent_cache_append
    g = torch.Generator(device="cuda").manual_seed(2)
    table, blocks = paged(g, [20], 16)
    x, r = torch.randn(1, 3, 1, 512, device="cuda").half(), torch.randn(1, 3, 1, 64, device="cuda").half()
    a, b = ([torch.zeros(blocks, 16, 1, w, device="cuda", dtype=torch.float16) for w in (512, 64)] for _ in range(2))
    w = torch.rand(512, device="cuda")
    LatentCacheAppend(inv_freq(), norm_weight=w, interleaved=False)(x, r, *a, block_table=table, actual_seq_lengths_kv=[20])
    latent_cache_append(x, r, *b, inv_freq(), block_table=table, actual_seq_lengths_kv=[20], norm_weight=w, interleaved=False)
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and int(a[0].count_nonzero()) > 1400
