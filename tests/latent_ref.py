"""Plain 64-bit forms of the operators around the latent paged cache, and the paged batches that their tests share."""
import torch


def turn(x, positions, inv_freq, sections, offset, interleaved, sign=1.0):
    """float64 x [..., heads, width]; positions [...] or [axes, ...]: pair j of the rotated features times exp(i p f_j)."""
    pairs = inv_freq.numel()
    sizes = [pairs] if sections is None else list(sections)
    pos = positions[None] if sections is None else positions
    angle = torch.cat([pos[a][..., None].double() * f.double()
                       for a, f in enumerate(torch.split(inv_freq, sizes))], -1)[..., None, :] * sign
    y = x.double().clone()
    part = y[..., offset:offset + 2 * pairs]
    re, im = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :pairs], part[..., pairs:])
    re, im = re.clone(), im.clone()
    new_re, new_im = re * angle.cos() - im * angle.sin(), re * angle.sin() + im * angle.cos()
    if interleaved:
        part[..., 0::2], part[..., 1::2] = new_re, new_im
    else:
        part[..., :pairs], part[..., pairs:] = new_re, new_im
    return y


def rotation_bound(x, ref, dtype, pairs, offset, interleaved):
    """What a rotation in 32 bits rounded once to `dtype` may be off by.  The fraction of a turn is rounded to 2^-24 of at most
    1/2 (2e-7 radians), sine and cosine to 2 units in the last place (2.4e-7), two products and their sum to
    2^-24 each: together below 1e-6 of |re| + |im|."""
    a = x.double().abs()
    part = a[..., offset:offset + 2 * pairs]
    if interleaved:
        s = (part[..., 0::2] + part[..., 1::2]).repeat_interleave(2, -1)
    else:
        s = (part[..., :pairs] + part[..., pairs:]).repeat(*[1] * (part.ndim - 1), 2)
    room = torch.zeros_like(a)
    room[..., offset:offset + 2 * pairs] = 1e-6 * s
    info = torch.finfo(dtype)
    # (the rounding is half a step of what is rounded, which lies within `room` of ref)
    return (ref.abs() + room) * (info.eps / 2) + room + info.tiny * info.eps


def paged(gen, totals, page, shared=0, spare=3):
    """Block table (int32, -1 past a sequence) of sequences of `totals` tokens whose first `shared` pages are the same ones,
    pages in random order, and the number of pages of the cache (`spare` of them unused)."""
    need = [-(-n // page) for n in totals]
    blocks = shared + sum(max(0, n - shared) for n in need) + spare
    pages = torch.randperm(blocks, generator=gen, device=gen.device).to(torch.int32)
    table = torch.full((len(totals), max(need + [1]) + 1), -1, dtype=torch.int32, device=gen.device)
    at = shared
    for b, n in enumerate(need):
        table[b, :min(n, shared)] = pages[:min(n, shared)]
        if n > shared:
            table[b, shared:n] = pages[at:at + n - shared]
            at += n - shared
    return table, blocks


def rows_of(table, b, positions, page, blocks):
    """Cache row of each position of sequence b; -1 where its block is absent, past the table or beyond the cache."""
    block = torch.div(positions, page, rounding_mode="floor")
    inside = (positions >= 0) & (block < table.shape[1])
    blk = table[b].long()[block.clamp(0, table.shape[1] - 1)]
    row = blk * page + positions % page
    return torch.where(inside & (blk >= 0) & (blk < blocks), row, torch.full_like(row, -1))


def inv_freq(pairs=32, base=10000.0, device="cuda"):
    return (1.0 / base ** (torch.arange(pairs, dtype=torch.float64) / pairs)).float().to(device)
