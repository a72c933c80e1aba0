"""Operators of quantised serving: a paged cache of keys and values held in 4 or 8 bits (written as the tokens come,
read back, and read by the attention of decoded tokens and prompt portions), and the product of 8-bit integers with a scale
for every token and output channel.

A cached group of values x (32 neighbouring elements of a key, a whole head of a value) is held as codes c of `bits` bits, a
step s and an offset z, both bfloat16, and stands for z + s (c - H), H = 2^(bits - 1):

    z = bf16((H max x + (H - 1) min x) / (2H - 1))
    s = max((max x - z) / (H - 1), (z - min x) / H), rounded to float32 and then up to bfloat16
    c = round((x - z) / s) + H, ties to even, within 0 .. 2H - 1

A page of a layer is bytes [key/value heads, head bytes]; one head of a page of P tokens is laid out as
    keys    [P][4][D / 32][8]   codes: element 32 g + 8 j + e of the head at [j][g][e]; with 4 bits, eight codes are a little-endian
                                word in which element e has the four bits from 4 (e / 2 + 4 (e % 2)) on
    values  [P / 8][D][8]       codes, eight tokens of a dimension together; with 4 bits [P / 8][D / 2][8] bytes, an even dimension
                                in the low half of a byte and the next one in the high half, token t of eight in byte
                                (0, 2, 1, 3, 4, 6, 5, 7)[t]
    steps and offsets of the keys [P][D / 32], then of the values [P]: a 32-bit word each, s in its upper half and z in its lower

The product: a row x of activations is held as round(x / a) with a = max|x| / 127 in float32, the weight as integers with
a float32 scale a row, and y = a w (sum of the integers' products) + bias.
"""

import math

import torch

own = False

DEVICE = "cuda:0"
PAIR_OF = (0, 2, 1, 3, 4, 6, 5, 7)  # byte of token t of eight in a value block of 4 bits


# ---- the cases ----------------------------------------------------------------------- #
def listed():
    return [
        # a decode step of eight requests at very different depths: one token each, keys turned, written and read back (latency)
        {"name": "cache_write_decode_8", "op": "write", "bits": 4, "dtype": "bf16", "heads": 8, "dim": 128, "page": 256,
         "new": "1,1,1,1,1,1,1,1", "kv": "32768,20011,12289,8193,6000,4097,2500,1023"},
        # the largest portion of a prompt that one step takes
        {"name": "cache_write_prompt_4096", "op": "write", "bits": 4, "dtype": "bf16", "heads": 8, "dim": 128, "page": 256,
         "new": "4096", "kv": "12288"},
        # portions of several prompts with tokens of other requests between, 8 bits, small pages, heads of 64
        {"name": "cache_write_ragged_8bit", "op": "write", "bits": 8, "dtype": "bf16", "heads": 8, "dim": 64, "page": 64,
         "new": "613,1,130,37,1,749", "kv": "613,911,167,1061,3001,750"},
        # a short conversation taken out of the cache again, to be kept on the host in bfloat16
        {"name": "cache_read_777_8bit", "op": "read", "bits": 8, "dtype": "bf16", "heads": 8, "dim": 64, "page": 256, "kv": "777"},
        # a context of the longest length
        {"name": "cache_read_131072", "op": "read", "bits": 4, "dtype": "bf16", "heads": 8, "dim": 128, "page": 256, "kv": "131072"},
        # one user's chat
        {"name": "attend_decode_1x1000", "op": "attend", "bits": 4, "dtype": "bf16", "q_heads": 48, "heads": 8, "dim": 128, "page": 256,
         "window": 0, "new": "1", "kv": "1000"},
        # decode at batch 8 and context 32,768
        {"name": "attend_decode_8x32768", "op": "attend", "bits": 4, "dtype": "bf16", "q_heads": 48, "heads": 8, "dim": 128, "page": 256,
         "window": 0, "new": "1,1,1,1,1,1,1,1", "kv": "32768,32768,32768,32768,32768,32768,32768,32768"},
        # a prompt of 2,048 tokens
        {"name": "attend_prompt_2048", "op": "attend", "bits": 4, "dtype": "bf16", "q_heads": 48, "heads": 8, "dim": 128, "page": 256,
         "window": 0, "new": "2048", "kv": "2048"},
        # decoded tokens and portions of prompts in one step, a layer with a window, 8 bits
        {"name": "attend_mixed_window_8bit", "op": "attend", "bits": 8, "dtype": "bf16", "q_heads": 32, "heads": 8, "dim": 128, "page": 256,
         "window": 2048, "new": "1,1,301,1,77,1,1,513", "kv": "5011,911,301,4097,2125,64,7777,3585"},
        # one decoded token through the attention's output projection of the 32B shape
        {"name": "product_1_row", "op": "product", "dtype": "bf16", "rows": 1, "k": 6144, "n": 6144, "bias": False},
        # 37 decoded tokens through the joined gate and up projections of the 8B shape
        {"name": "product_37_rows", "op": "product", "dtype": "bf16", "rows": 37, "k": 4096, "n": 28672, "bias": False},
        # a prompt of 2,048 tokens through those of the 32B shape
        {"name": "product_2048_rows", "op": "product", "dtype": "bf16", "rows": 2048, "k": 6144, "n": 43008, "bias": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "read", "attend", "attend", "product"])
    dtype = "fp32" if rng.random() < 0.15 else "bf16"
    if op == "product":
        rows = _log(rng, 1, 2048)
        k = 16 * _log(rng, 4, 900)
        n = _log(rng, 100, min(43008, 2 * 10**8 // k, 5 * 10**11 // (2 * rows * k)))
        return {"op": op, "dtype": dtype, "rows": rows, "k": k, "n": n, "bias": rng.random() < 0.3}
    bits = rng.choice([4, 4, 8])
    dim = rng.choice([32, 64, 64, 96, 128, 128, 128, 192, 256])
    page = rng.choice([8, 16, 64, 128, 256, 256])
    if op in ("write", "read"):
        heads = rng.choice([1, 2, 3, 5, 8, 8, 16])
        total = max(1, _log(rng, 1, 4096 if op == "write" else 65536) * 64 // (heads * dim // 16))
        seqs = min(total, rng.randint(1, 9))
        cuts = sorted(rng.sample(range(1, total), seqs - 1)) if seqs > 1 else []
        new = [b - a for a, b in zip([0, *cuts], [*cuts, total])]
        case = {"op": op, "bits": bits, "dtype": dtype, "heads": heads, "dim": dim, "page": page}
        if op == "read":
            return {**case, "kv": ",".join(map(str, new))}
        return {**case, "new": ",".join(map(str, new)), "kv": ",".join(str(n + rng.choice([0, _log(rng, 1, 20000)])) for n in new)}
    heads = rng.choice([1, 2, 4, 8, 8])
    group = rng.choice([1, 2, 3, 4, 6, 8, 16])
    case = {"op": op, "bits": bits, "dtype": dtype, "q_heads": heads * group, "heads": heads, "dim": dim, "page": page,
            "window": rng.choice([0, 0, 0, _log(rng, 1, 8192)])}
    kind = rng.choice(["decode", "decode", "prompt", "mixed"])
    if kind == "decode":
        seqs = _log(rng, 1, 64)
        most = max(2, min(65536, 8 * 32768 * 8 * 128 // (seqs * heads * dim)))
        new, kv = [1] * seqs, [_log(rng, 1, most) for _ in range(seqs)]
    else:
        seqs = 1 if kind == "prompt" else rng.randint(2, 8)
        new = [1 if kind == "mixed" and rng.random() < 0.4 else _log(rng, 2, 1024 if kind == "prompt" else 300) for _ in range(seqs)]
        kv = [n + rng.choice([0, _log(rng, 1, 2000)]) for n in new]
    return {**case, "new": ",".join(map(str, new)), "kv": ",".join(map(str, kv))}


def _lengths(text):
    return [int(n) for n in text.split(",")]


def _type(case):
    return torch.float32 if case["dtype"] == "fp32" else torch.bfloat16


# ---- what a user's program has in hand ------------------------------------------------- #
def _sizes(bits, dim, page):
    """Bytes of one head of a page: keys' codes (the values' take as many), words of the keys, words of the values."""
    return page * dim * bits // 8, page * (dim // 32) * 4, page * 4


def _step(case, gen):
    """Lengths, block table (the pages of a pool in a random order) and each new token's place."""
    kv, page = _lengths(case["kv"]), case["page"]
    new = _lengths(case["new"]) if "new" in case else kv
    pages = [-(-n // page) for n in kv]
    pool = sum(pages) + 3
    order = torch.randperm(pool, device=DEVICE, generator=gen).to(torch.int32)
    table = torch.full((len(kv), max(pages)), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at : at + n]
        at += n
    positions = torch.cat([torch.arange(n - m, n, dtype=torch.int32, device=DEVICE) for m, n in zip(new, kv)])
    seq = torch.repeat_interleave(torch.arange(len(kv), device=DEVICE), torch.tensor(new, device=DEVICE)).to(torch.int32)
    first = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device=DEVICE)
    lengths = torch.tensor(kv, dtype=torch.int32, device=DEVICE)
    return {"q_lens": new, "kv_lens": kv, "table": table, "pool": pool, "positions": positions, "seq": seq, "first": first, "lengths": lengths}


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    dtype = _type(case)
    if case["op"] == "product":
        # activations behind a norm: a few channels much larger than the others; a weight quantised row by row
        x = torch.randn(case["rows"], case["k"], device=DEVICE, generator=gen)
        x = (x * torch.exp(0.5 * torch.randn(case["k"], device=DEVICE, generator=gen))).to(dtype)
        weight = (torch.randn(case["n"], case["k"], device=DEVICE, generator=gen) * 32).round_().clamp_(-127, 127).to(torch.int8)
        scale = (0.5 + torch.rand(case["n"], device=DEVICE, generator=gen)) * (0.02 / 32)
        bias = torch.randn(case["n"], device=DEVICE, generator=gen) if case["bias"] else None
        return {"case": case, "x": x, "weight": weight, "scale": scale, "bias": bias}
    heads, dim, page, bits = case["heads"], case["dim"], case["page"], case["bits"]
    state = {"case": case, **_step(case, gen)}
    codes, key_words, value_words = _sizes(bits, dim, page)
    cache = torch.zeros((state["pool"], heads, 2 * codes + key_words + value_words), dtype=torch.uint8, device=DEVICE)
    state["cache"] = cache
    # a few channels of the keys lie far from zero, as they do in trained models
    centre = 3.0 * torch.randn(heads, dim, device=DEVICE, generator=gen) * (torch.rand(heads, dim, device=DEVICE, generator=gen) < 0.1)
    if case["op"] == "write":
        tokens = state["positions"].numel()
        q_heads = 4 * heads
        joined = torch.randn(tokens, (q_heads + 2 * heads) * dim, device=DEVICE, generator=gen)
        joined[:, q_heads * dim : (q_heads + heads) * dim] += centre.reshape(-1)
        joined = joined.to(dtype)  # as the joined projection leaves it
        state["k"] = joined[:, q_heads * dim : (q_heads + heads) * dim].unflatten(1, (heads, dim))
        state["v"] = joined[:, (q_heads + heads) * dim :].unflatten(1, (heads, dim))
        state["table_of_angles"] = 1.0 / (500000.0 ** (torch.arange(0, dim, 2, device=DEVICE).float() / dim))
        return state
    # a cache that earlier steps have filled, every page of the pool with tokens of its own
    at_once = max(1, 16384 // page)
    for p0 in range(0, state["pool"], at_once):
        part = cache[p0 : p0 + at_once]
        slots = part.shape[0] * page
        k = (torch.randn(slots, heads, dim, device=DEVICE, generator=gen) + centre).to(dtype)
        v = torch.randn(slots, heads, dim, device=DEVICE, generator=gen).to(dtype)
        every = torch.arange(slots, device=DEVICE)
        _put(part, k, v, every // page, every % page, bits)
    if case["op"] == "attend":
        rows = torch.randn(state["positions"].numel(), case["q_heads"] * dim, device=DEVICE, generator=gen)
        state["q"] = (1.5 * rows).to(dtype).unflatten(1, (case["q_heads"], dim))
    return state


# ---- the plain forms --------------------------------------------------------------------- #
def _quantised(x, bits):
    """Codes (int64) and words (int64, step and offset) of the last dimension of float32 `x`.  In 64 bits: ties and steps that
    just fit are common among short numbers, and a quotient that is off in its last bit decides them otherwise (as does a
    quotient by a Python number, which is a product with its reciprocal)."""
    half = 1 << (bits - 1)
    hi, lo = x.amax(-1).double(), x.amin(-1).double()
    z = ((half * hi + (half - 1) * lo) / torch.full_like(hi, 2 * half - 1)).float().to(torch.bfloat16)
    zd = z.double()
    need = torch.maximum((hi - zd) / torch.full_like(hi, half - 1), (zd - lo) / half).float()
    step = ((need.view(torch.int32).long() + 0xFFFF) >> 16) << 16
    s = step.to(torch.int32).view(torch.float32).double()[..., None]
    c = torch.where(s > 0, torch.round((x.double() - zd[..., None]) / s), torch.zeros_like(s)).clamp(-half, half - 1).long() + half
    return c, step | (z.view(torch.int16).long() & 0xFFFF)


def _parts(cache, dim, bits):
    """The four regions of every head of every page: bytes of the keys and of the values, words of either."""
    per_token = 2 * (dim * bits // 8) + (dim // 32) * 4 + 4
    pages, heads, size = cache.shape
    page = size // per_token
    codes, key_words, _ = _sizes(bits, dim, page)
    k = cache[:, :, :codes].unflatten(2, (page, 4, dim // 32, bits))
    v = cache[:, :, codes : 2 * codes].unflatten(2, (page // 8, dim * bits // 8, 8))
    kw = cache[:, :, 2 * codes : 2 * codes + key_words].unflatten(2, (page, dim // 32, 4))
    vw = cache[:, :, 2 * codes + key_words :].unflatten(2, (page, 4))
    return k, v, kw, vw


def _word_bytes(w):
    return torch.stack([(w >> (8 * i)) & 255 for i in range(4)], dim=-1).to(torch.uint8)


def _put(cache, k, v, pages, slots, bits):
    """Quantises keys and values [T, heads, dim] and writes them at slot `slots` of page `pages`."""
    dim = k.shape[2]
    kp, vp, kw, vw = _parts(cache, dim, bits)
    c, words = _quantised(k.float().unflatten(2, (dim // 32, 32)), bits)
    c = c.unflatten(3, (4, 8)).transpose(2, 3)  # [T, heads, 4, dim / 32, 8]
    if bits == 4:
        # byte i of a word: its low half is bits 8 i .. 8 i + 3; element e lies at 4 (e / 2 + 4 (e % 2))
        low, high = [0, 4, 1, 5], [2, 6, 3, 7]
        c = c[..., low] | (c[..., high] << 4)
    kp[pages, :, slots] = c.to(torch.uint8)
    kw[pages, :, slots] = _word_bytes(words)
    c, words = _quantised(v.float(), bits)
    vw[pages, :, slots] = _word_bytes(words)
    if bits == 4:
        c = c[..., 0::2] | (c[..., 1::2] << 4)
        place = torch.tensor(PAIR_OF, device=c.device)[slots % 8]
    else:
        place = slots % 8
    vp[pages, :, slots // 8, :, place] = c.to(torch.uint8)


def _words_of(b):
    b = b.long()
    w = b[..., 0] | (b[..., 1] << 8) | (b[..., 2] << 16) | (b[..., 3] << 24)
    as_float = lambda bits: torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32).view(torch.float32)  # noqa: E731
    return as_float((w >> 16) << 16), as_float((w & 0xFFFF) << 16)


def _get(cache, pages, slots, dim, bits):
    """Float32 keys and values [..., heads, dim] that the cache holds at slot `slots` of page `pages`."""
    half = 1 << (bits - 1)
    kp, vp, kw, vw = _parts(cache, dim, bits)
    c = kp[pages, :, slots].int()
    if bits == 4:
        c = torch.stack([c[..., 0] & 15, c[..., 2] & 15, c[..., 0] >> 4, c[..., 2] >> 4, c[..., 1] & 15, c[..., 3] & 15, c[..., 1] >> 4, c[..., 3] >> 4], -1)
    c = c.transpose(-3, -2).flatten(-2)  # [..., heads, dim / 32, 32]
    s, z = _words_of(kw[pages, :, slots])
    k = (z[..., None] + s[..., None] * (c - half)).flatten(-2)
    place = torch.tensor(PAIR_OF, device=cache.device)[slots % 8] if bits == 4 else slots % 8
    c = vp[pages, :, slots // 8, :, place].int()
    if bits == 4:
        c = torch.stack([c & 15, c >> 4], dim=-1).flatten(-2)
    s, z = _words_of(vw[pages, :, slots])
    return k, z[..., None] + s[..., None] * (c - half)


def _turned(k, positions, table):
    angle = positions.double()[:, None] * table.double()
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    a, b = k.double().unflatten(2, (k.shape[2] // 2, 2)).unbind(-1)
    return torch.stack([a * c - b * s, b * c + a * s], dim=-1).flatten(2).float().to(k.dtype)


def _places(state):
    page = state["case"]["page"]
    positions, seq = state["positions"].long(), state["seq"].long()
    return state["table"][seq, positions // page].long(), positions % page


def _plain_write(state):
    bits = state["case"]["bits"]
    pages, slots = _places(state)
    k = _turned(state["k"], state["positions"], state["table_of_angles"])
    _put(state["cache"], k, state["v"], pages, slots, bits)
    return _plain_read(state)


def _plain_read(state):
    pages, slots = _places(state)
    k, v = _get(state["cache"], pages, slots, state["case"]["dim"], state["case"]["bits"])
    dtype = _type(state["case"])
    return k.to(dtype), v.to(dtype)


def _plain_attend(state):
    """Every sequence padded to the longest: scores, mask, softmax, sum of the values, in float32."""
    case, q = state["case"], state["q"]
    heads, dim, page = case["heads"], case["dim"], case["page"]
    lengths, first, seq = state["lengths"].long(), state["first"].long(), state["seq"].long()
    n_seq, longest, most = lengths.numel(), max(state["kv_lens"]), max(state["q_lens"])
    at = torch.arange(longest, device=q.device)
    pages = state["table"].long()[:, at // page].clamp(min=0)
    k, v = _get(state["cache"], pages, (at % page).expand_as(pages), dim, case["bits"])  # [B, S, heads, dim]
    inside = torch.arange(q.shape[0], device=q.device) - first[seq]  # the token's place in its portion
    padded = torch.zeros((n_seq, most, *q.shape[1:]), device=q.device)
    padded[seq, inside] = q.float()
    group = case["q_heads"] // heads
    rows = padded.unflatten(2, (heads, group)).permute(0, 2, 1, 3, 4).flatten(2, 3)  # [B, heads, most * group, dim]
    scores = torch.matmul(rows, k.permute(0, 2, 3, 1).contiguous()) * dim ** -0.5
    position = (lengths - (first[1:] - first[:-1]))[:, None] + torch.arange(most, device=q.device)  # [B, most]
    seen = (at <= position[..., None]) & (at < lengths[:, None, None])
    if case["window"]:
        seen &= at > position[..., None] - case["window"]
    seen = seen[:, None, :, None].expand(-1, -1, -1, group, -1).flatten(2, 3)
    scores = scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_(min=-1e30)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True).clamp_(min=1e-30)
    out = torch.matmul(p, v.permute(0, 2, 1, 3).contiguous()) / total
    out = out.unflatten(2, (most, group)).permute(0, 2, 1, 3, 4).flatten(2)  # [B, most, q_heads * dim]
    return out[seq, inside].to(q.dtype)


def _plain_product(state):
    x = state["x"].float()
    top = x.abs().amax(1, keepdim=True)
    a = top / torch.full_like(top, 127)
    codes = torch.where(a > 0, torch.round(x / a), torch.zeros_like(x))
    y = torch.matmul(codes, state["weight"].float().t()) * a * state["scale"]
    if state["bias"] is not None:
        y = y + state["bias"]
    return y.to(state["x"].dtype)


# ---- the framework's calls ----------------------------------------------------------------- #
def _batch(state):
    """The step's descriptor, made once a step and used by all of its layers."""
    from cwm_amd.engine.batch import StepBatch

    batch = state.get("batch")
    if batch is None:
        batch = state["batch"] = StepBatch(
            n_tokens=state["positions"].numel(), n_seqs=len(state["kv_lens"]), n_logit_rows=0, tokens=state["positions"],
            positions=state["positions"], seq_of_token=state["seq"], cu_q=state["first"], kv_len=state["lengths"],
            state_slots=state["lengths"], logit_rows=state["lengths"][:0], block_tables=[state["table"]],
            q_lens=state["q_lens"], kv_lens=state["kv_lens"], page_size=state["case"]["page"],
        )
    return batch


def _own_run(state):
    from cwm_amd import ops

    case = state["case"]
    if case["op"] == "product":
        return ops.linear_int8(state["x"], state["weight"], state["scale"], state["bias"])
    if case["op"] == "attend":
        return ops.quant_paged_attention(
            state["q"], state["cache"], state["table"], _batch(state), case["window"] or None, case["dim"] ** -0.5, case["bits"]
        )
    if case["op"] == "write":
        ops.quant_kv_write(
            state["k"], state["v"], state["positions"], state["table_of_angles"], state["cache"], state["table"], state["seq"], case["bits"]
        )
    return ops.quant_kv_read(state["cache"], state["table"], state["positions"], state["seq"], case["dim"], case["bits"], _type(case))


def run(state):
    if own:
        return _own_run(state)
    plain = {"write": _plain_write, "read": _plain_read, "attend": _plain_attend, "product": _plain_product}
    return plain[state["case"]["op"]](state)


# ---- what a pass cannot do without ----------------------------------------------------------- #
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "product":
        m, n, k = case["rows"], case["n"], case["k"]
        return {"bytes": m * k * size + n * k + 4 * n + m * n * size + (4 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    heads, dim = case["heads"], case["dim"]
    held = heads * (2 * (dim * case["bits"] // 8) + (dim // 32) * 4 + 4)  # bytes of a token
    kv = _lengths(case["kv"])
    new = _lengths(case["new"]) if "new" in case else kv
    tokens = sum(new)
    rows = 2 * heads * dim * size * tokens  # keys and values of the tokens as they come, or as they are given back
    if case["op"] == "write":
        return {"bytes": 2 * rows + held * tokens, "flops": 16 * heads * dim * tokens}
    if case["op"] == "read":
        return {"bytes": rows + held * tokens, "flops": 4 * heads * dim * tokens}
    pairs = keys = 0
    for m, n in zip(new, kv):
        w = case["window"] or n
        first = n - m  # the first new token's position
        keys += n - max(0, first - w + 1)
        short = max(0, min(n, w) - first)  # tokens whose window reaches past the start
        pairs += sum((first + 1, first + short)) * short // 2 + (m - short) * w
    return {"bytes": keys * held + 2 * tokens * case["q_heads"] * dim * size, "flops": 4 * pairs * case["q_heads"] * dim}


# ---- the definition in 64 bits ---------------------------------------------------------------- #
def _stands_for(x, bits):
    """What a group held in `bits` bits stands for; x is float64 [..., group]."""
    top = 2**bits - 1
    upper, lower = 2 ** (bits - 1) - 1, 2 ** (bits - 1)  # steps above and below the offset
    largest, smallest = x.max(-1, keepdim=True).values, x.min(-1, keepdim=True).values
    offset = ((lower * largest + upper * smallest) / torch.full_like(largest, top)).float().bfloat16().double()
    need = torch.maximum((largest - offset) / torch.full_like(offset, upper), (offset - smallest) / lower).float().double()
    near = need.bfloat16()  # the next one up where this is below
    step = torch.where(near.double() < need, (near.view(torch.int16) + 1).view(torch.bfloat16), near).double()
    steps = torch.where(step > 0, (x - offset) / torch.where(step > 0, step, torch.ones_like(step)), torch.zeros_like(x))
    return offset + step * torch.round(steps).clamp(-lower, upper)


def _held(cache, page, slot, head, dim, bits):
    """Keys and values in float64 [n, dim] of one head at places (page, slot), byte by byte as the layout says."""
    per_token = dim * bits // 4 + dim // 8 + 4
    size = cache.shape[2] // per_token
    flat = cache.reshape(-1)
    base = ((page * cache.shape[1] + head) * cache.shape[2])[:, None]
    slot = slot[:, None]
    plane = size * dim * bits // 8
    d = torch.arange(dim, device=cache.device)

    def byte(at):
        return flat[base + at].to(torch.int64)

    def number(at):
        return ((byte(at + 1) << 24) + (byte(at) << 16) - ((byte(at + 1) >> 7) << 32)).to(torch.int32).view(torch.float32).double()

    group, j, e = d // 32, d % 32 // 8, d % 8
    unit = (j * (dim // 32) + group) * bits  # first byte of the element's eight codes within the token's key
    if bits == 4:
        nibble = e // 2 + 4 * (e % 2)
        codes = byte(slot * (dim // 2) + unit + nibble // 2) // torch.where(nibble % 2 == 1, 16, 1) % 16
    else:
        codes = byte(slot * dim + unit + e)
    words = 2 * plane + (slot * (dim // 32) + group) * 4
    key = number(words) + number(words + 2) * (codes - 2 ** (bits - 1))
    if bits == 4:
        place = torch.tensor([0, 2, 1, 3, 4, 6, 5, 7], device=cache.device)[slot % 8]
        codes = byte(plane + (slot // 8 * (dim // 2) + d // 2) * 8 + place) // torch.where(d % 2 == 1, 16, 1) % 16
    else:
        codes = byte(plane + (slot // 8 * dim + d) * 8 + slot % 8)
    words = 2 * plane + size * (dim // 32) * 4 + slot * 4
    value = number(words) + number(words + 2) * (codes - 2 ** (bits - 1))
    return key, value


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "product":
        x = state["x"].double()
        scale = (x.abs().amax(1, keepdim=True) / 127).float().double()  # held in float32
        steps = torch.round(torch.where(scale > 0, x / scale, torch.zeros_like(x)))
        y = torch.zeros(case["rows"], case["n"], dtype=torch.float64, device=DEVICE)
        for n0 in range(0, case["n"], 8192):
            y[:, n0 : n0 + 8192] = (steps @ state["weight"][n0 : n0 + 8192].double().t()) * scale * state["scale"][n0 : n0 + 8192].double()
        return y if state["bias"] is None else y + state["bias"].double()
    heads, dim, page, bits = case["heads"], case["dim"], case["page"], case["bits"]
    if case["op"] == "write":
        turn = state["positions"].double()[:, None, None] * state["table_of_angles"].double()
        k = torch.view_as_complex(state["k"].double().unflatten(2, (dim // 2, 2)).contiguous()) * torch.polar(torch.ones_like(turn), turn)
        k = torch.view_as_real(k).flatten(2).to(torch.float32).to(_type(case)).double()  # keys are rounded to the activations' type
        return _stands_for(k.unflatten(2, (dim // 32, 32)), bits).flatten(2), _stands_for(state["v"].double(), bits)
    table, kv = state["table"].long(), state["kv_lens"]

    def sequence(b, head, lo, hi):
        at = torch.arange(lo, hi, device=DEVICE)
        parts = [_held(state["cache"], table[b, a // page], a % page, head, dim, bits) for a in at.split(4096)]
        return torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])

    if case["op"] == "read":
        got = [[sequence(b, h, 0, n) for h in range(heads)] for b, n in enumerate(kv)]
        return tuple(torch.cat([torch.stack([h[i] for h in one], dim=1) for one in got]) for i in (0, 1))
    group = case["q_heads"] // heads
    q = state["q"].double()
    out = torch.zeros(q.shape[0], case["q_heads"], dim, dtype=torch.float64, device=DEVICE)
    t0 = 0
    for m, (b, n) in zip(state["q_lens"], enumerate(kv)):
        lo = max(0, n - m - case["window"] + 1) if case["window"] else 0
        at, mine = torch.arange(lo, n, device=DEVICE), torch.arange(n - m, n, device=DEVICE)[:, None]
        hidden = at > mine
        if case["window"]:
            hidden = hidden | (mine - at >= case["window"])
        for h in range(heads):
            k, v = sequence(b, h, lo, n)
            for g in range(h * group, (h + 1) * group):
                s = (q[t0 : t0 + m, g] @ k.t()) / math.sqrt(dim)
                out[t0 : t0 + m, g] = torch.softmax(s.masked_fill(hidden, -math.inf), dim=1) @ v
        t0 += m
    return out.flatten(1)
