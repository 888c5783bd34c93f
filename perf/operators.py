"""Measured work of the operators around the latent (MLA) paged cache: the rotation of queries and keys, the append of new
tokens to the caches, and dense attention of a batch whose sequences share a prefix.

`listed()` names the fixed cases, `draw(rng)` gives another one of the same ranges, `prepare(case, seed)` makes what a
serving or training program holds before the call, `run(state)` is one pass (`own`: through the framework's operators, else
in their plain form), `exact(case, seed)` what a pass returns, from the definitions in 64 bits, `work(case)` the bytes and
operations that a pass cannot do without.

Kinds of case (`op`):
  rotate        rotary positions of queries or index queries, one axis or several
  rotate_grad   the gradient of the same
  append        latents, rope keys and index keys of new tokens into their paged caches, rotated (and normalised) on the way
  attend        attention of query tokens over every visible key of the paged latent cache, whose first positions are the
                same tokens for the whole batch
"""
import math

import torch

own = False

DIM, ROPE, INDEX_DIM = 512, 64, 128
SCALE = 1.0 / math.sqrt(DIM + ROPE)
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one token for each of 64 conversations, the heads of one of eight tensor-parallel ranks: latency
        dict(name="rotate_step", op="rotate", tokens=64, heads=16, width=64, row=192, offset=0, pairs=32, axes="",
             interleaved=True, dtype="bf16"),
        # prefill of a batch of prompts: the rope part (64 wide) of queries that come as rows of 192 per head
        dict(name="rotate_prompts", op="rotate", tokens=15360, heads=128, width=64, row=192, offset=0, pairs=32, axes="",
             interleaved=True, dtype="bf16"),
        # index queries of an odd batch: 64 of 128 features rotated, the halves paired, positions of time, height and width
        dict(name="rotate_index_fp16", op="rotate", tokens=2047, heads=64, width=128, row=128, offset=0, pairs=32,
             axes="8 12 12", interleaved=False, dtype="fp16"),
        # training: the gradient back through the rotation, text and image tokens packed
        dict(name="rotate_grad_4k", op="rotate_grad", tokens=4091, heads=64, width=64, row=64, offset=0, pairs=32,
             axes="16 8 8", interleaved=True, dtype="bf16"),
        # a decode step of 64 conversations: one token each into all three caches, the latent normalised on the way
        dict(name="append_step", op="append", layout="BSND", batch=64, q_tokens=1, q_lens="", cached=4096, page=64,
             index=True, norm=True, axes="", interleaved=True, dtype="bf16"),
        # prefill of a batch of prompts, some continued
        dict(name="append_prompts", op="append", layout="TND", batch=4, q_tokens=0, q_lens="8192 4096 2048 1024",
             cached=2048, page=128, index=True, norm=True, axes="", interleaved=True, dtype="bf16"),
        # chunks of odd lengths, latents already normalised, no index keys, pages of 48, image positions
        dict(name="append_chunks_fp16", op="append", layout="TND", batch=5, q_tokens=0, q_lens="377 1029 64 1 613",
             cached=3000, page=48, index=False, norm=False, axes="8 12 12", interleaved=False, dtype="fp16"),
        # a few conversations behind a short system prompt, few heads: latency
        dict(name="attend_step_8", op="attend", layout="BSND", batch=8, q_tokens=1, q_lens="", prefix=1024, shortest=16,
             longest=256, heads=16, page=64, dtype="bf16"),
        # a full decode batch behind a long shared document
        dict(name="attend_step_64", op="attend", layout="BSND", batch=64, q_tokens=1, q_lens="", prefix=16384, shortest=64,
             longest=2048, heads=128, page=128, dtype="bf16"),
        # two tokens (one speculated) for an odd batch; the prefix ends inside a page
        dict(name="attend_spec_33_fp16", op="attend", layout="BSND", batch=33, q_tokens=2, q_lens="", prefix=5003,
             shortest=2, longest=700, heads=64, page=16, dtype="fp16"),
        # a scheduler's mixed batch behind a shared document: chunks of prompts and a lone token
        dict(name="attend_chunks", op="attend", layout="TND", batch=4, q_tokens=0, q_lens="377 64 1 129", prefix=8192,
             shortest=1, longest=600, heads=32, page=64, dtype="bf16"),
        # nothing shared: each conversation reads its own cache
        dict(name="attend_apart_16", op="attend", layout="BSND", batch=16, q_tokens=1, q_lens="", prefix=0, shortest=2048,
             longest=8192, heads=128, page=128, dtype="bf16"),
    ]


# ------------------------------------------------------------------------------------------------
# Drawn cases
# ------------------------------------------------------------------------------------------------
def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _lens(rng, total):
    parts = [rng.uniform(0.1, 1.0) for _ in range(rng.randint(1, 6))]
    return [max(1, int(total * p / sum(parts))) for p in parts]


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        kind = "rotate" if c["op"].startswith("rotate") else c["op"]
        most[kind] = max(most.get(kind, (0, 0)), (w["bytes"], w["flops"]), key=lambda v: max(v[0] / 6e12, v[1] / 1.5e15))
    while True:
        kind = rng.choice(("rotate", "append", "attend", "attend"))
        dtype = rng.choice(("bf16", "bf16", "fp16"))
        axes = rng.choice(("", "", "8 12 12", "16 8 8", "10 22", "4 4 12 12"))
        if kind == "rotate":
            width = rng.choice((64, 64, 128, 192))
            pairs = rng.choice([p for p in (32, 32, 32, 64) if 2 * p <= width])
            if pairs == 64:
                axes = rng.choice(("", "16 24 24"))
            c = dict(op=rng.choice(("rotate", "rotate", "rotate_grad")), tokens=_log_int(rng, 1, 15360),
                     heads=rng.choice((1, 5, 16, 32, 64, 128)), width=width, row=width + rng.choice((0, 0, 64, 128)),
                     offset=rng.choice((0, width - 2 * pairs)), pairs=pairs, axes=axes, interleaved=rng.random() < 0.5,
                     dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")))
        elif kind == "append":
            packed = rng.random() < 0.5
            lens = _lens(rng, _log_int(rng, 1, 15360)) if packed else []
            c = dict(op="append", layout="TND" if packed else "BSND", batch=len(lens) if packed else _log_int(rng, 1, 64),
                     q_tokens=0 if packed else rng.choice((1, 1, 2, 3)), q_lens=" ".join(map(str, lens)),
                     cached=_log_int(rng, 1, 4096), page=rng.choice((1, 16, 24, 48, 64, 100, 128)),
                     index=rng.random() < 0.7, norm=rng.random() < 0.5, axes=axes, interleaved=rng.random() < 0.5,
                     dtype=dtype)
        else:
            packed = rng.random() < 0.3
            lens = _lens(rng, _log_int(rng, 4, 700)) if packed else []
            shortest = _log_int(rng, 1, 1024)
            c = dict(op="attend", layout="TND" if packed else "BSND", batch=len(lens) if packed else _log_int(rng, 1, 64),
                     q_tokens=0 if packed else rng.choice((1, 1, 1, 2, 4)), q_lens=" ".join(map(str, lens)),
                     prefix=rng.choice((0, _log_int(rng, 1, 16384), _log_int(rng, 256, 16384), _log_int(rng, 256, 16384))),
                     shortest=shortest, longest=shortest + _log_int(rng, 1, 4096),
                     heads=rng.choice((1, 8, 16, 20, 32, 64, 128)), page=rng.choice((16, 24, 32, 48, 64, 64, 100, 128)),
                     dtype=dtype)
        w = work(c)
        if w["bytes"] <= most[kind][0] and w["flops"] <= max(most[kind][1], w["bytes"]):
            return c


# ------------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------------
def _ints(text):
    return [int(v) for v in text.split()]


def _query_lens(c):
    return _ints(c["q_lens"]) if c["layout"] == "TND" else [c["q_tokens"]] * c["batch"]


def _ends(lens):
    out, at = [], 0
    for n in lens:
        at += n
        out.append(at)
    return out


class _Draws:
    def __init__(self, seed, dtype):
        self.gen, self.dtype = torch.Generator(device="cuda").manual_seed(seed), DTYPES[dtype]

    def normal(self, *shape, scale=1.0, dtype=None):
        out = torch.empty(shape, dtype=dtype or self.dtype, device="cuda")
        flat = out.view(-1)
        for i in range(0, flat.numel(), 1 << 26):
            n = min(1 << 26, flat.numel() - i)
            flat[i:i + n] = torch.randn(n, generator=self.gen, device="cuda") * scale
        return out

    def ints(self, lo, hi, *shape):
        return torch.randint(lo, hi + 1, shape, generator=self.gen, device="cuda", dtype=torch.int32)


def _inv_freq(pairs):
    return (1.0 / 10000.0 ** (torch.arange(pairs, dtype=torch.float64) / pairs)).float().cuda()


def _table(d, totals, longest, page, shared=0):
    """Block table of sequences of `totals` tokens (at most `longest`, for which the cache has room) whose first `shared` whole
    pages are the same ones; pages in random order.  With it the number of pages of the cache."""
    need = [-(-n // page) for n in totals]
    own_pages = [max(0, n - shared) for n in need]
    blocks = shared + sum(max(0, -(-n // page) - shared) for n in longest)
    pages = torch.randperm(blocks, generator=d.gen, device="cuda").to(torch.int32)
    table = torch.full((len(totals), max(-(-n // page) for n in longest)), -1, dtype=torch.int32, device="cuda")
    at = shared
    for b, n in enumerate(need):
        table[b, :min(n, shared)] = pages[:min(n, shared)]
        if n > shared:
            table[b, shared:n] = pages[at:at + own_pages[b]]
            at += own_pages[b]
    return table, blocks


def prepare(case, seed):
    c = dict(case)
    d = _Draws(seed, c["dtype"])
    op = c["op"]
    if op in ("rotate", "rotate_grad"):
        axes = _ints(c["axes"])
        lead = (len(axes),) if axes else ()
        return dict(op=op, x=d.normal(c["tokens"], c["heads"], c["row"])[..., c["row"] - c["width"]:],
                    positions=d.ints(0, 131071, *lead, c["tokens"]), inv_freq=_inv_freq(c["pairs"]),
                    axes=tuple(axes) or None, offset=c["offset"], interleaved=c["interleaved"])
    q_lens = _query_lens(c)
    tokens, batch, tnd = sum(q_lens), c["batch"], c["layout"] == "TND"
    lead = (tokens,) if tnd else (batch, c["q_tokens"])
    s = dict(op=op, layout=c["layout"], q_lens=q_lens, page=c["page"],
             ends=torch.tensor(_ends(q_lens), dtype=torch.int32, device="cuda") if tnd else None)
    if op == "append":
        totals = [n + v for n, v in zip(q_lens, d.ints(0, c["cached"], batch).tolist())]
        s["table"], blocks = _table(d, totals, [n + c["cached"] for n in q_lens], c["page"])
        axes = _ints(c["axes"])
        projected = d.normal(*lead, 1, DIM + ROPE)      # one projection gives the latent and the rope key
        s.update(latent=projected[..., :DIM], rope=projected[..., DIM:], inv_freq=_inv_freq(ROPE // 2),
                 latent_cache=d.normal(blocks, c["page"], 1, DIM), rope_cache=d.normal(blocks, c["page"], 1, ROPE),
                 index=d.normal(*lead, 1, INDEX_DIM) if c["index"] else None,
                 index_cache=d.normal(blocks, c["page"], 1, INDEX_DIM) if c["index"] else None,
                 weight=1 + d.normal(DIM, scale=0.1) if c["norm"] else None, axes=tuple(axes) or None,
                 positions=d.ints(0, 8191, len(axes), *lead) if axes else None, interleaved=c["interleaved"])
    else:
        totals = [c["prefix"] + max(n, v) for n, v in zip(q_lens, d.ints(c["shortest"], c["longest"], batch).tolist())]
        page, whole = c["page"], c["prefix"] // c["page"]
        s["table"], blocks = _table(d, totals, [c["prefix"] + max(n, c["longest"]) for n in q_lens], page, whole)
        s.update(q=d.normal(*lead, c["heads"], DIM, scale=2.0), q_rope=d.normal(*lead, c["heads"], ROPE, scale=2.0),
                 latent_cache=d.normal(blocks, page, 1, DIM), rope_cache=d.normal(blocks, page, 1, ROPE),
                 prefix=c["prefix"])
        if c["prefix"] % page:      # the prefix ends inside a page: each sequence has a copy of that page's first tokens
            first = s["table"][:, whole].long()
            for cache in (s["latent_cache"], s["rope_cache"]):
                cache[first, :c["prefix"] % page] = cache[first[0], :c["prefix"] % page].clone()
    s.update(totals=totals, lens=torch.tensor(totals, dtype=torch.int32, device="cuda"))
    return s


# ------------------------------------------------------------------------------------------------
# One pass: the plain form
# ------------------------------------------------------------------------------------------------
def _angles(positions, inv_freq, axes):
    """cos and sin [tokens.., 1, pairs] of positions [tokens..], or of [axes, tokens..] whose pairs are dealt out in order;
    the angles of far positions are taken in 64 bits."""
    if axes is None:
        angle = positions[..., None].double() * inv_freq.double()
    else:
        angle = torch.cat([positions[i][..., None].double() * f.double()
                           for i, f in enumerate(torch.split(inv_freq, list(axes)))], dim=-1)
    return angle.cos().float().unsqueeze(-2), angle.sin().float().unsqueeze(-2)


def _rotate(x, cos, sin, offset, interleaved):
    """fp32 x [tokens.., heads, width] with the features offset .. offset + 2 pairs rotated."""
    pairs = cos.shape[-1]
    y = x.float().clone()
    part = y[..., offset:offset + 2 * pairs]
    if interleaved:
        a, b = part[..., 0::2].clone(), part[..., 1::2].clone()
        part[..., 0::2], part[..., 1::2] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = part[..., :pairs].clone(), part[..., pairs:].clone()
        part[..., :pairs], part[..., pairs:] = a * cos - b * sin, a * sin + b * cos
    return y


def _flat(x, s):
    return x.reshape(-1, *x.shape[(1 if s["layout"] == "TND" else 2):])


def _slots(s):
    """Position and cache row of every token, sequence by sequence."""
    pos, row = [], []
    for b, (n, total) in enumerate(zip(s["q_lens"], s["totals"])):
        p = torch.arange(total - n, total, device="cuda")
        pos.append(p)
        row.append(s["table"][b].long()[p // s["page"]] * s["page"] + p % s["page"])
    return torch.cat(pos), torch.cat(row)


def _run_plain(s):
    op = s["op"]
    if op in ("rotate", "rotate_grad"):
        cos, sin = _angles(s["positions"], s["inv_freq"], s["axes"])
        return _rotate(s["x"], cos, sin if op == "rotate" else -sin, s["offset"], s["interleaved"]).to(s["x"].dtype)
    if op == "append":
        pos, row = _slots(s)
        if s["positions"] is not None:
            pos = s["positions"].reshape(len(s["axes"]), -1)
        cos, sin = _angles(pos, s["inv_freq"], s["axes"])
        x = _flat(s["latent"], s).float()
        if s["weight"] is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * s["weight"].float()
        caches = [s["latent_cache"], s["rope_cache"]]
        rows = [x, _rotate(_flat(s["rope"], s), cos, sin, 0, s["interleaved"])]
        if s["index"] is not None:
            caches.append(s["index_cache"])
            rows.append(_rotate(_flat(s["index"], s), cos, sin, 0, False))
        for cache, new in zip(caches, rows):
            cache.view(-1, 1, cache.shape[-1])[row] = new.to(cache.dtype)
        return tuple(caches)
    q, q_rope = _flat(s["q"], s), _flat(s["q_rope"], s)
    out, top, total, at = [], [], [], 0
    for b, (n, length) in enumerate(zip(s["q_lens"], s["totals"])):
        p = torch.arange(length, device="cuda")
        row = s["table"][b].long()[p // s["page"]] * s["page"] + p % s["page"]
        value = s["latent_cache"].view(-1, DIM)[row].float()
        key = torch.cat([value, s["rope_cache"].view(-1, ROPE)[row].float()], dim=1)
        x = torch.cat([q[at:at + n].float(), q_rope[at:at + n].float()], dim=2)
        scores = torch.matmul(x, key.T) * SCALE                       # [n, heads, keys]
        hidden = p[None, :] > (length - n + torch.arange(n, device="cuda"))[:, None]
        scores.masked_fill_(hidden[:, None, :], -math.inf)
        m = scores.amax(-1, keepdim=True)
        e = (scores - m).exp_()
        z = e.sum(-1, keepdim=True)
        out.append((torch.matmul(e, value) / z).to(s["q"].dtype))
        top.append(m[..., 0])
        total.append(z[..., 0])
        at += n
    shape = (1,) + s["q"].shape[:2] if s["layout"] == "TND" else (s["q"].shape[0], 1) + s["q"].shape[1:3]
    return torch.cat(out).view(s["q"].shape), torch.cat(top).view(shape), torch.cat(total).view(shape)


# ------------------------------------------------------------------------------------------------
# One pass: the framework's operators
# ------------------------------------------------------------------------------------------------
def _run_own(s):
    from dsa_triton_ascend_b200 import (latent_cache_append, rotary_embedding, rotary_embedding_grad,
                                        shared_prefix_attention)
    op = s["op"]
    if op in ("rotate", "rotate_grad"):
        f = rotary_embedding if op == "rotate" else rotary_embedding_grad
        return f(s["x"], s["positions"], s["inv_freq"], layout="TND", interleaved=s["interleaved"],
                 rotary_offset=s["offset"], axis_sections=s["axes"])
    if op == "append":
        caches = latent_cache_append(
            s["latent"], s["rope"], s["latent_cache"], s["rope_cache"], s["inv_freq"], block_table=s["table"],
            actual_seq_lengths_query=s["ends"], actual_seq_lengths_kv=s["lens"], index_key=s["index"],
            index_cache=s["index_cache"], positions=s["positions"], axis_sections=s["axes"], layout=s["layout"],
            norm_weight=s["weight"], norm_eps=EPS, interleaved=s["interleaved"])
        return caches if s["index"] is not None else caches[:2]
    return shared_prefix_attention(
        s["q"], s["latent_cache"], scale_value=SCALE, block_table=s["table"], actual_seq_lengths_query=s["ends"],
        actual_seq_lengths_kv=s["lens"], query_rope=s["q_rope"], key_rope=s["rope_cache"],
        shared_prefix_length=s["prefix"], layout_query=s["layout"], sparse_mode=3, return_softmax_lse=True)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------------------
# From the definitions, in 64 bits
# ------------------------------------------------------------------------------------------------
def _turned(x, positions, inv_freq, axes, offset, interleaved, sign=1.0):
    """float64 rows [tokens, heads, width]; pair j of the rotated features, as one complex number, times e^(i position f_j)."""
    pairs = inv_freq.numel()
    axis = torch.zeros(pairs, dtype=torch.long) if axes is None else \
        torch.repeat_interleave(torch.arange(len(axes)), torch.tensor(axes))
    at = positions.reshape(1 if axes is None else len(axes), -1).double().T[:, axis.cuda()]       # [tokens, pairs]
    wheel = torch.polar(torch.ones_like(at), sign * at * inv_freq.double())[:, None, :]
    j = torch.arange(pairs, device="cuda")
    re = offset + (2 * j if interleaved else j)
    im = offset + (2 * j + 1 if interleaved else j + pairs)
    y = x.double()
    z = torch.complex(y[..., re], y[..., im]) * wheel
    return y.index_copy(-1, re, z.real).index_copy(-1, im, z.imag)


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op in ("rotate", "rotate_grad"):
        return _turned(s["x"], s["positions"], s["inv_freq"], s["axes"], s["offset"], s["interleaved"],
                       1.0 if op == "rotate" else -1.0)
    if op == "append":
        caches = [s[n].double() for n in ("latent_cache", "rope_cache", "index_cache") if s[n] is not None]
        starts = [0] + _ends(s["q_lens"])
        tokens = [s[n].reshape(starts[-1], 1, s[n].shape[-1]) if s[n] is not None else None
                  for n in ("latent", "rope", "index")]
        for b, (n, total) in enumerate(zip(s["q_lens"], s["totals"])):
            mine = slice(starts[b], starts[b] + n)
            p = torch.arange(n, device="cuda") + (total - n)
            page, at = s["table"][b][torch.div(p, s["page"], rounding_mode="floor")].long(), p.remainder(s["page"])
            turn = p if s["positions"] is None else s["positions"].reshape(len(s["axes"]), -1)[:, mine]
            x = tokens[0][mine].double()
            if s["weight"] is not None:
                x = s["weight"].double() * x / (x.pow(2).sum(-1, keepdim=True) / DIM + EPS).sqrt()
            caches[0][page, at] = x
            caches[1][page, at] = _turned(tokens[1][mine], turn, s["inv_freq"], s["axes"], 0, s["interleaved"])
            if tokens[2] is not None:
                caches[2][page, at] = _turned(tokens[2][mine], turn, s["inv_freq"], s["axes"], 0, False)
        return tuple(caches)
    starts = [0] + _ends(s["q_lens"])
    heads = s["q"].shape[-2]
    q, qr = s["q"].reshape(starts[-1], heads, DIM), s["q_rope"].reshape(starts[-1], heads, ROPE)
    out = torch.empty(starts[-1], heads, DIM, dtype=torch.float64, device="cuda")
    top = torch.empty(starts[-1], heads, dtype=torch.float64, device="cuda")
    total = torch.empty_like(top)
    for b, (n, length) in enumerate(zip(s["q_lens"], s["totals"])):
        pages = s["table"][b, :-(-length // s["page"])].long()
        c = s["latent_cache"][pages].reshape(-1, DIM)[:length].double()
        r = s["rope_cache"][pages].reshape(-1, ROPE)[:length].double()
        for i in range(n):                              # a token sees the keys up to its own position
            t, seen = starts[b] + i, length - n + i + 1
            x = (q[t].double() @ c[:seen].T + qr[t].double() @ r[:seen].T) / math.sqrt(DIM + ROPE)
            top[t] = x.max(dim=1).values
            total[t] = torch.exp(x - top[t][:, None]).sum(1)
            out[t] = torch.softmax(x, dim=1) @ c[:seen]
    stat = (1, starts[-1], heads) if s["layout"] == "TND" else (len(s["q_lens"]), 1, s["q_lens"][0], heads)
    return out.view(s["q"].shape), top.view(stat), total.view(stat)


# ------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ------------------------------------------------------------------------------------------------
def work(case):
    c, op = case, case["op"]
    size = 4 if c["dtype"] == "fp32" else 2
    axes = max(1, len(_ints(c.get("axes", ""))))
    if op in ("rotate", "rotate_grad"):     # features in and out, positions in; six operations a pair
        n = c["tokens"] * c["heads"]
        return dict(bytes=2 * size * n * c["width"] + 4 * axes * c["tokens"] + 4 * c["pairs"], flops=6.0 * n * c["pairs"])
    q_lens = _query_lens(c)
    tokens = sum(q_lens)
    if op == "append":                      # tokens in, cache rows out, the pages and lengths that say where
        width = DIM + ROPE + (INDEX_DIM if c["index"] else 0)
        pairs = ROPE // 2 * (2 if c["index"] else 1)
        return dict(bytes=2 * size * tokens * width + 4 * (tokens + 2 * c["batch"]) +
                    (4 * axes * tokens if c["axes"] else 0) + (size * DIM if c["norm"] else 0),
                    flops=tokens * (6.0 * pairs + (4.0 * DIM if c["norm"] else 0)))
    # queries in, output and statistics out, the prefix's keys once and every sequence's own keys once
    mean = (c["shortest"] + c["longest"]) // 2
    lens = [max(n, mean) for n in q_lens]
    pairs = sum(n * (c["prefix"] + k) - n * (n - 1) // 2 for n, k in zip(q_lens, lens))
    keys = c["prefix"] + sum(lens)
    return dict(bytes=size * tokens * c["heads"] * (DIM + ROPE + DIM) + 8 * tokens * c["heads"] + size * (DIM + ROPE) * keys +
                4 * (keys // c["page"] + 2 * c["batch"]), flops=2.0 * pairs * c["heads"] * (2 * DIM + ROPE))
