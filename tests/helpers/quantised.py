"""The quantised cache written out plainly, in 64 bits and one element at a time where it matters: what a group of values is
held as, which byte each code lies in, and attention over what is held."""

from __future__ import annotations

import math

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
PLACE = (0, 2, 1, 3, 4, 6, 5, 7)


def token_bytes(dim, bits):
    return 2 * (dim * bits // 8) + dim // 32 * 4 + 4


def round_up_bf16(x):
    """The next bfloat16 number that is not below the float32 rounding of x >= 0 (float64 tensor)."""
    f = x.float()
    return (((f.view(torch.int32).long() + 0xFFFF) >> 16) << 16).to(torch.int32).view(torch.float32).double()


def hold(x, bits):
    """Codes, step and offset (float64) of the last dimension of x."""
    half = 2 ** (bits - 1)
    x = x.double()
    hi, lo = x.amax(-1, keepdim=True), x.amin(-1, keepdim=True)
    z = ((half * hi + (half - 1) * lo) / (2 * half - 1)).float().bfloat16().double()
    s = round_up_bf16(torch.maximum((hi - z) / (half - 1), (z - lo) / half))
    c = torch.where(s > 0, torch.round((x - z) / torch.where(s > 0, s, torch.ones_like(s))), torch.zeros_like(x)).clamp(-half, half - 1) + half
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    c = torch.where(bad, torch.full_like(c, half), c)
    nan = torch.full_like(s, math.nan)
    return c.long(), torch.where(bad, nan, s)[..., 0], torch.where(bad, nan, z)[..., 0]


def stands_for(c, s, z, bits):
    return z[..., None] + s[..., None] * (c - 2 ** (bits - 1)).double()


def _word(s, z):
    def half(x):
        return (x.to(torch.bfloat16).view(torch.int16).long() & 0xFFFF) if not math.isnan(float(x)) else torch.tensor(0x7FC0)

    w = int(half(s)) << 16 | int(half(z))
    return [(w >> (8 * i)) & 255 for i in range(4)]


def put(cache, page, slot, k, v, bits):
    """Writes one token's key and value [heads, dim] into a cache of bytes [pages, heads, head bytes] on the CPU."""
    heads, dim = k.shape
    groups = dim // 32
    P = cache.shape[2] // token_bytes(dim, bits)
    plane = P * dim * bits // 8
    for h in range(heads):
        raw = cache[page, h]
        c, s, z = hold(k[h].reshape(groups, 32), bits)
        for g in range(groups):
            for j in range(4):
                unit = (slot * 4 + j) * groups * bits + g * bits
                eight = [int(c[g, 8 * j + e]) for e in range(8)]
                if bits == 8:
                    for e in range(8):
                        raw[unit + e] = eight[e]
                else:
                    word = sum(eight[e] << (4 * (e // 2 + 4 * (e % 2))) for e in range(8))
                    for i in range(4):
                        raw[unit + i] = (word >> (8 * i)) & 255
            at = 2 * plane + (slot * groups + g) * 4
            raw[at : at + 4] = torch.tensor(_word(s[g], z[g]), dtype=torch.uint8)
        c, s, z = hold(v[h], bits)
        for d in range(0, dim, 2):
            if bits == 8:
                for i in (d, d + 1):
                    raw[plane + (slot // 8 * dim + i) * 8 + slot % 8] = int(c[i])
            else:
                raw[plane + (slot // 8 * (dim // 2) + d // 2) * 8 + PLACE[slot % 8]] = int(c[d]) | int(c[d + 1]) << 4
        at = 2 * plane + P * groups * 4 + slot * 4
        raw[at : at + 4] = torch.tensor(_word(s, z), dtype=torch.uint8)


def put_all(cache, table, seq_lens, keys, values, bits):
    """The same for whole sequences at once (keys[b] [n, heads, dim]); the layout is that of `put`, which the tests hold it to."""
    for b, n in enumerate(seq_lens):
        if n == 0:
            continue
        dim = keys[b].shape[2]
        P = cache.shape[2] // token_bytes(dim, bits)
        at = torch.arange(n)
        put_tokens(cache, table[b, at // P].long(), at % P, keys[b], values[b], bits)


def _word_bytes(s, z):
    def half(x):
        h = x.to(torch.bfloat16).view(torch.int16).long() & 0xFFFF
        return torch.where(torch.isnan(x), torch.full_like(h, 0x7FC0), h)

    w = half(s) << 16 | half(z)
    return torch.stack([(w >> (8 * i)) & 255 for i in range(4)], -1).to(torch.uint8)


def put_tokens(cache, pages, slots, k, v, bits):
    n, heads, dim = k.shape
    groups = dim // 32
    P = cache.shape[2] // token_bytes(dim, bits)
    plane = P * dim * bits // 8
    ck, sk, zk = hold(k.reshape(n, heads, groups, 4, 8).flatten(3), bits)
    ck = ck.unflatten(3, (4, 8)).transpose(2, 3)  # [n, heads, 4, groups, 8]
    cv, sv, zv = hold(v, bits)
    kb = cache[:, :, :plane].unflatten(2, (P, 4, groups, bits))
    vb = cache[:, :, plane : 2 * plane].unflatten(2, (P // 8, dim * bits // 8, 8))
    kw = cache[:, :, 2 * plane : 2 * plane + P * groups * 4].unflatten(2, (P, groups, 4))
    vw = cache[:, :, 2 * plane + P * groups * 4 :].unflatten(2, (P, 4))
    if bits == 8:
        kb[pages, :, slots] = ck.to(torch.uint8)
        vb[pages, :, slots // 8, :, slots % 8] = cv.to(torch.uint8)
    else:
        word = sum(ck[..., e] << (4 * (e // 2 + 4 * (e % 2))) for e in range(8))
        kb[pages, :, slots] = torch.stack([(word >> (8 * i)) & 255 for i in range(4)], -1).to(torch.uint8)
        vb[pages, :, slots // 8, :, torch.tensor(PLACE)[slots % 8]] = (cv[..., 0::2] | cv[..., 1::2] << 4).to(torch.uint8)
    kw[pages, :, slots] = _word_bytes(sk, zk)
    vw[pages, :, slots] = _word_bytes(sv, zv)


def turn(x, positions, inv_freq):
    """Adjacent pairs of x [T, heads, dim] turned in 64 bits, rounded once to x's type."""
    if inv_freq is None:
        return x
    angle = positions.double()[:, None] * inv_freq.double()
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    a, b = x.double()[..., 0::2], x.double()[..., 1::2]
    return torch.stack([a * c - b * s, b * c + a * s], -1).flatten(2).float().to(x.dtype)


class Step:
    """A step's lengths, a block table over a pool of pages in mixed order, and a `StepBatch` of it."""

    def __init__(self, new, kv, page, seed=0, spare=2, device="cpu"):
        g = torch.Generator().manual_seed(seed)
        self.new, self.kv, self.page = list(new), list(kv), page
        held = [-(-n // page) for n in kv]
        self.pool = sum(held) + spare
        order = torch.randperm(self.pool, generator=g).to(torch.int32)
        self.table = torch.full((len(kv), max(max(held), 1) + 1), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(held):
            self.table[b, :n] = order[at : at + n]
            at += n
        self.positions = torch.cat([torch.arange(n - m, n) for m, n in zip(new, kv)]).to(torch.int32)
        self.seq = torch.cat([torch.full((m,), b) for b, m in enumerate(new)]).to(torch.int32)
        self.cu = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32)
        self.lens = torch.tensor(list(kv), dtype=torch.int32)

    def batch(self, device):
        from cwm_amd.engine.batch import StepBatch

        to = lambda t: t.to(device)  # noqa: E731
        return StepBatch(
            n_tokens=int(self.cu[-1]), n_seqs=len(self.kv), n_logit_rows=0, tokens=to(self.positions), positions=to(self.positions),
            seq_of_token=to(self.seq), cu_q=to(self.cu), kv_len=to(self.lens), state_slots=to(self.lens), logit_rows=to(self.lens)[:0],
            block_tables=[to(self.table)], q_lens=self.new, kv_lens=self.kv, page_size=self.page,
        )


def _most_of_tile(x):
    """[n, dim] -> [n]: the largest magnitude among the 32 tokens that a token belongs to."""
    most = torch.nn.functional.pad(x.abs().amax(1), (0, -x.shape[0] % 32)).reshape(-1, 32).amax(1)
    return most.repeat_interleave(32)[: x.shape[0]]


def attention(step, q, keys, values, bits, window, scale):
    """Float64 result [T, Hq * dim] over what the cache holds of `keys` and `values`, and how far a kernel may be off it.

    A kernel's scores are float32 sums of at most dim + 40 terms of the matrix instructions and of the groups, each rounded
    (2^-24 of the largest partial sum, twice for sums whose order is the instruction's): the terms are at most
    s (143 + 136) |q| and |z| |q| with an offset of the codes (bfloat16 queries, 4 bits; 8 bits: 255 + 128), s 2 H |q| without.
    A score that is off by d moves the result by at most 2 d sum p |v|.  bfloat16: the weights p s are two parts of
    half a step of half a step together and multiply codes less H, and the result is rounded; the sums with the codes' offset, s (OFF' + c), are float32 sums of one
    term for 32 keys.  bfloat16 portions of more than 128 rows read queries, keys and values as float16 with a power of two beside them: a
    score is off by the sum of dim independent roundings of up to half a step, 2^-11 |q k| each, whose deviation is that over sqrt(3)
    (six of them are allowed), and a value by half a step; the weights p are rounded and multiply whole values.  What is smaller than
    2^-14 beside its power of two is off by 2^-25 at most: 2^-17 of the largest query of its row, the largest key or value of its
    32, and 2^-25 of a weight whose row has one of at least 1."""
    T, heads_q, dim = q.shape
    heads = keys[0].shape[1]
    group = heads_q // heads
    half, fine = 2 ** (bits - 1), q.dtype == torch.float32
    reach = 2 * half if fine else (279 if bits == 4 else 383)
    out = torch.zeros(T, heads_q, dim, dtype=torch.float64)
    limit = torch.zeros_like(out)
    t0 = 0
    for b, (m, n) in enumerate(zip(step.new, step.kv)):
        if m == 0:
            continue
        at, mine = torch.arange(n), torch.arange(n - m, n)[:, None]
        seen = at <= mine
        if window is not None:
            seen &= at > mine - window
        for h in range(heads):
            ck, sk, zk = hold(keys[b][:, h].reshape(n, dim // 32, 32), bits)
            cv, sv, zv = hold(values[b][:, h], bits)
            k, v = stands_for(ck, sk, zk, bits).flatten(1), stands_for(cv, sv, zv, bits)
            for g in range(h * group, (h + 1) * group):
                x = q[t0 : t0 + m, g].double()
                p = torch.softmax((x @ k.t() * scale).masked_fill(~seen, -math.inf), 1)
                o = p @ v
                out[t0 : t0 + m, g] = o
                size = (x.abs().reshape(m, -1, 32).sum(-1)[:, None] * (sk * reach + zk.abs())).sum(-1)  # [m, n]
                off = 2.0 * 2.0 ** -24 * (dim + 40) * scale * torch.where(seen, size, torch.zeros_like(size)).amax(1)
                spread = p @ (sv[:, None] * reach + zv[:, None].abs())
                err = 2 * off[:, None] * (p @ v.abs()) + 2.0 * 2.0 ** -24 * (n / 32 + 40) * spread
                if not fine and m * group > 128:
                    half_step, least = 2.0 ** -11, 2.0 ** -17
                    off = off + 6 / 3 ** 0.5 * half_step * scale * torch.where(seen, (x * x) @ (k * k).t(), torch.zeros_like(size)).sqrt().amax(1)
                    small = x.abs().amax(1)[:, None] * k.abs().sum(1) + x.abs().sum(1)[:, None] * _most_of_tile(k)
                    off = off + least * scale * torch.where(seen, small, torch.zeros_like(size)).amax(1)
                    err = 2 * off[:, None] * (p @ v.abs()) + 2.0 * 2.0 ** -24 * (n / 32 + 40) * spread
                    err = err + 2.01 * half_step * (p @ v.abs()) + least * (p @ _most_of_tile(v))[:, None] + 2.0 ** -25 * (seen.double() @ v.abs())
                    err = err + HALF_STEP[q.dtype] * (o.abs() + err)
                elif not fine:
                    err = err + 2.0 ** -16 * (p @ (sv[:, None] * (cv - half).abs().double()))
                    err = err + HALF_STEP[q.dtype] * (o.abs() + err)
                else:
                    err = err + 2.0 ** -23 * o.abs()
                limit[t0 : t0 + m, g] = err
        t0 += m
    return out.flatten(1), limit.flatten(1)
