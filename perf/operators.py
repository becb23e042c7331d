"""What the operators around the 4-bit K/V cache are measured on: norms and rotation of queries and keys, the
cache's write and read-back, and the attention that reads it.

A case names its operator ("op"):
  rope   qk_norm_rope   rows of fused q|k|v: RMSNorm of each query and key head, then the position rotation
  cache  kv4_write, kv4_read   rows of K and V quantised into the pages, and rows read back out of them
  attend kv4_attention   each row's query heads over its sequence's cached positions

Rows belong to sequences: sequence s has the rows row_start[s] .. row_start[s+1]-1, its cache holds kv_len[s]
positions, and its rows stand at the last of them. Rows behind row_start[n_seq] are padding, left as they were.

The cache is [page][kv_head][K block | V block], 64 positions a page. A block holds 64 positions of head_dim codes
(0..15, two a byte) and then, per position and group of 64 dimensions, the fp16 pair (d, m) of x = m + d * code.
m is the largest fp16 not above the group's minimum, d the smallest fp16 that reaches its maximum in 15 steps, the
code the nearest one (ties to even).
"""
import math

import torch

own = False

PAGE, GROUP = 64, 64
F16_MAX = 65504.0
DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16}


# ---- cases -----------------------------------------------------------------
def _rope(name, rows, heads, kv, hd, dtype, norm, halves=False, n_pos=4096, pad=0):
    return {"name": name, "op": "rope", "rows": rows, "heads": heads, "kv": kv, "hd": hd, "dtype": dtype, "norm": norm,
            "halves": halves, "n_pos": n_pos, "pad": pad}


def _cache(name, seqs, rows, length, heads, kv, hd, dtype, write, spread=False):
    return {"name": name, "op": "cache", "seqs": seqs, "rows": rows, "len": length, "heads": heads, "kv": kv, "hd": hd,
            "dtype": dtype, "write": write, "spread": spread}


def _attend(name, seqs, rows, length, heads, kv, hd, dtype, spread=False):
    return {"name": name, "op": "attend", "seqs": seqs, "rows": rows, "len": length, "heads": heads, "kv": kv, "hd": hd,
            "dtype": dtype, "spread": spread}


def listed():
    return [
        # one token of the 4B shape on its way from the q|k|v product to the cache
        _rope("rope 1 row 4b", 1, 32, 8, 128, "f32", True),
        # a ragged step of the tiny shape: 100 rows, some of them padding, no norms (the Llama form)
        _rope("rope 100 rows tiny", 100, 8, 2, 64, "f32", False, n_pos=1000, pad=7),
        # a long prompt of the 27B shape in half precision, halves rotated, far positions
        _rope("rope 4096 rows 27b f16", 4096, 32, 16, 128, "f16", True, halves=True, n_pos=32768),
        # the step of a 16-sequence batch of the 8B shape: one new row each, read back
        _cache("write step 16 seqs", 16, 1, 4096, 32, 8, 128, "f32", True, spread=True),
        # prompts of eight sequences written in one call and read back
        _cache("write 8 prompts", 8, 577, 1500, 32, 8, 128, "f32", True, spread=True),
        # a whole 32768-position cache read back in half precision, as a caller that moves it elsewhere does
        _cache("read 32768 f16", 1, 32768, 32768, 32, 8, 128, "f16", False),
        # the first token of a short sequence
        _attend("attend 1 seq 65", 1, 1, 65, 8, 2, 64, "f32"),
        # batch-1 decode of the 4B shape behind a 512-token prompt
        _attend("attend 1 seq 576 4b", 1, 1, 576, 32, 8, 128, "f32"),
        # one token of each of 16 sequences, 32768 positions each: the long-context batch
        _attend("attend 16 seqs 32768", 16, 1, 32768, 32, 8, 128, "f32"),
        # a serving step with lengths from none to 8191, in half precision, 27B heads
        _attend("attend 64 ragged f16 27b", 64, 1, 8191, 32, 16, 128, "f16", spread=True),
        # verification of 8 drafted tokens for each of 4 sequences
        _attend("attend verify 4x8", 4, 8, 8192, 32, 8, 128, "f32"),
        # a prompt chunk of 64 rows behind a long context
        _attend("attend chunk 64", 1, 64, 16384, 32, 8, 128, "f32"),
    ]


SHAPES = [(8, 2, 64), (8, 8, 64), (32, 8, 128), (32, 16, 128), (16, 2, 128), (16, 4, 256)]
MOST_ROPE = 4096 * 48 * 128        # elements of the largest rope case
MOST_CACHE = 32768 * 8 * 128       # elements a side of the largest cache case
MOST_LEN = 16 * 32768 * 8 * 128    # cached elements a side of the largest attention case
MOST_PAIRS = 64 * 16384 * 32 * 128  # products a side of the largest attention case with several rows


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    heads, kv, hd = rng.choice(SHAPES)
    dtype = rng.choice(["f32", "f32", "f16"])
    op = rng.choice(["rope", "cache", "attend", "attend"])
    if op == "rope":
        rows = _log(rng, 1, MOST_ROPE // ((heads + kv) * hd))
        c = _rope("", rows, heads, kv, hd, dtype, rng.random() < 0.6, rng.random() < 0.5, _log(rng, 64, 32768),
                  rng.randrange(0, min(9, rows)))
    elif op == "cache":
        seqs, write = _log(rng, 1, 64), rng.random() < 0.7
        length = _log(rng, 1, min(32768, MOST_CACHE // (seqs * kv * hd)))
        rows = rng.choice([1, _log(rng, 1, length)]) if write else length
        c = _cache("", seqs, rows, length, heads, kv, hd, dtype, write, rng.random() < 0.5)
    else:
        seqs, rows = _log(rng, 1, 64), rng.choice([1, 1, _log(rng, 1, 64)])
        most = MOST_LEN // (seqs * kv * hd)
        if rows > 1:
            most = min(most, MOST_PAIRS // (seqs * rows * heads * hd))
        c = _attend("", seqs, rows, _log(rng, 1, max(1, min(32768, most))), heads, kv, hd, dtype, rng.random() < 0.5)
    del c["name"]
    return c


def _plan(case):
    """Cached positions and rows of every sequence, before their order is shuffled: all alike, or spread from
    nothing to the most."""
    n, length, rows = case["seqs"], case["len"], case["rows"]
    if not case["spread"] or n == 1:
        return [length] * n, [min(rows, length)] * n
    lens = [length * i // (n - 1) for i in range(n)]
    return lens, [min(rows - (rows * (i % 3)) // 4, lens[i]) for i in range(n)]


def work(case):
    hd, kv, size = case["hd"], case["kv"], 4 if case["dtype"] == "f32" else 2
    if case["op"] == "rope":
        rows = case["rows"] - case["pad"]
        n = rows * (case["heads"] + kv) * hd
        # each row's sines and cosines, the norm weights, the values in and out
        return {"bytes": 2 * n * size + rows * (hd * 4 + 4) + (8 * hd if case["norm"] else 0),
                "flops": n * (7 if case["norm"] else 3)}
    row4 = 2 * kv * (hd // 2 + 4 * (hd // GROUP))  # a position's K and V in 4 bits
    lens, rows = _plan(case)
    if case["op"] == "cache":
        n = sum(rows)
        values = 2 * n * kv * hd * size
        return {"bytes": n * row4 * (2 if case["write"] else 1) + values * (2 if case["write"] else 1),
                "flops": 2 * n * kv * hd * (6 if case["write"] else 2)}
    pairs = sum(t * L - t * (t - 1) // 2 for t, L in zip(rows, lens))
    return {"bytes": sum(L for t, L in zip(rows, lens) if t) * row4 + 2 * sum(rows) * case["heads"] * hd * size,
            "flops": 4 * pairs * case["heads"] * hd}


# ---- inputs ----------------------------------------------------------------
def _rope_tables(n_pos, hd):
    th = torch.arange(n_pos, dtype=torch.float64, device=DEV)[:, None] * torch.pow(
        torch.tensor(1e6, dtype=torch.float64, device=DEV), -torch.arange(0, hd, 2, dtype=torch.float64, device=DEV) / hd)
    return th.cos().float(), th.sin().float()


def _kv_values(g, n, kv, hd, channel, what):
    """Rows as a model has them: keys with a few channels far from zero, values with tokens of different sizes."""
    x = torch.randn(n, kv, hd, device=DEV, generator=g)
    if what == "k":
        return x + channel
    return x * torch.exp(0.5 * torch.randn(n, kv, 1, device=DEV, generator=g))


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    hd, kv, heads, dtype = case["hd"], case["kv"], case["heads"], TYPES[case["dtype"]]
    s = {"op": case["op"], "hd": hd, "kv": kv, "heads": heads, "dtype": dtype}
    if case["op"] == "rope":
        rows, n_pos = case["rows"], case["n_pos"]
        s["x"] = (2 * torch.randn(rows, (heads + 2 * kv) * hd, device=DEV, generator=g)).to(dtype)
        s["pos"] = torch.randint(0, n_pos, (rows,), device=DEV, generator=g, dtype=torch.int32)
        order = torch.randperm(rows, device=DEV, generator=g)
        s["pos"][order[:1]] = n_pos - 1
        s["pos"][order[rows - case["pad"]:]] = -1
        s["cos"], s["sin"] = _rope_tables(n_pos, hd)
        s["halves"], s["norm"] = case["halves"], case["norm"]
        s["wq"] = 1 + 0.2 * torch.randn(hd, device=DEV, generator=g) if case["norm"] else None
        s["wk"] = 1 + 0.2 * torch.randn(hd, device=DEV, generator=g) if case["norm"] else None
        s["q_out"] = torch.zeros(rows, heads, hd, dtype=dtype, device=DEV)
        s["k_out"] = torch.zeros(rows, kv, hd, dtype=dtype, device=DEV)
        return s
    lens, rows = _plan(case)
    n = len(lens)
    order = torch.randperm(n, device=DEV, generator=g)
    kv_len = torch.tensor(lens, device=DEV)[order]
    row_start = torch.zeros(n + 1, dtype=torch.int64, device=DEV)
    row_start[1:] = torch.tensor(rows, device=DEV)[order].cumsum(0)
    # every sequence's pages, scattered over the pool
    per_seq = -(-max(case["len"], 1) // PAGE)
    need = -(-kv_len // PAGE)
    used = sum(-(-L // PAGE) for L in lens)
    slot = need.cumsum(0)[:, None] - need[:, None] + torch.arange(per_seq, device=DEV)
    pages = torch.randperm(used + 3, device=DEV, generator=g)
    inside = torch.arange(per_seq, device=DEV) < need[:, None]
    s["table"] = torch.where(inside, pages[slot.clamp(max=used)], -1).int()
    s["kv_len"], s["row_start"] = kv_len.int(), row_start.int()
    s["rows"] = n * case["rows"]
    s["cache"] = torch.zeros(used + 3, kv, 2, PAGE * (hd // 2 + 4 * (hd // GROUP)), dtype=torch.uint8, device=DEV)
    channel = 3 * torch.randn(kv, hd, device=DEV, generator=g) * (torch.rand(kv, hd, device=DEV, generator=g) < 0.06)
    # what the cache holds already: whole pages of sequences (a page's positions behind its sequence's end stay zero)
    live = torch.arange(per_seq * PAGE, device=DEV).view(1, per_seq, PAGE) < kv_len[:, None, None]
    step = max(1, (1 << 28) // (PAGE * kv * hd))
    where = inside.nonzero()
    for at in range(0, used, step):
        sq, pg = where[at:at + step].unbind(1)
        ok = live[sq, pg][:, :, None, None]
        for side, what in ((0, "k"), (1, "v")):
            x = _kv_values(g, sq.numel() * PAGE, kv, hd, channel, what).half().view(-1, PAGE, kv, hd)
            code, dm = _quantise(torch.where(ok, x, 0).transpose(1, 2))
            s["cache"][s["table"][sq, pg].long(), :, side] = _pack(code, dm, side)
    if case["op"] == "cache":
        s["write"] = case["write"]
        if case["write"]:  # the new rows, where the q|k|v product left them
            row = torch.randn(s["rows"], heads * hd, device=DEV, generator=g)
            k, v = (_kv_values(g, s["rows"], kv, hd, channel, w).view(s["rows"], -1) for w in "kv")
            s["qkv"] = torch.cat([row, k, v], 1).to(dtype)
        s["k_out"] = torch.zeros(s["rows"], kv, hd, dtype=dtype, device=DEV)
        s["v_out"] = torch.zeros(s["rows"], kv, hd, dtype=dtype, device=DEV)
    else:
        s["q"] = torch.randn(s["rows"], heads, hd, device=DEV, generator=g).to(dtype)
        s["out"] = torch.zeros(s["rows"], heads, hd, dtype=dtype, device=DEV)
        s["most"] = case["rows"]
    return s


# ---- the 4-bit format, in torch --------------------------------------------
def _f16_step(x):
    """The distance of fp16 numbers around x (64 bits): a power of two, put together from its exponent."""
    return ((torch.frexp(x).exponent - 11).clamp(min=-24).long() + 1023 << 52).view(torch.float64)


def _quantise(x):
    """x [..., hd]: codes [..., hd] (bytes) and the pairs (d, m) [..., hd / 64, 2] (fp16), chosen in 64 bits."""
    x = x.double().clamp(-F16_MAX, F16_MAX).unflatten(-1, (-1, GROUP))
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    m = torch.floor(lo / _f16_step(lo)) * _f16_step(lo)
    d = (hi - m) / torch.full_like(m, 15)  # by a tensor: a division by a number becomes a product with its inverse
    d = torch.ceil(d / _f16_step(d)) * _f16_step(d)
    code = torch.where(d > 0, torch.round((x - m) / d), 0).nan_to_num(0)
    return code.to(torch.uint8).flatten(-2), torch.cat([d, m], -1).half()


def _pack(code, dm, side):
    """Codes [..., PAGE, hd] and pairs [..., PAGE, groups, 2] as a block's bytes."""
    hd = code.shape[-1]
    slab = min(hd, 128)
    if side == 0:  # K: dimension = slab, group, t, word, 8 codes of a word; a position's words go t, group, word
        c = code.view(*code.shape[:-2], PAGE, hd // slab, slab // 64, 4, 2, 4, 2)
        c = c[..., 0] | c[..., 1] << 4
        n = c.dim()
        c = c.permute(*range(n - 6), n - 5, n - 6, n - 3, n - 4, n - 2, n - 1)
    else:  # V: position = step, half, t, parity; dimension = slab, block, g, 4 codes of a half word
        c = code.view(*code.shape[:-2], 4, 2, 4, 2, hd // slab, slab // 32, 8, 2, 2)
        c = c[..., 0] | c[..., 1] << 4
        n = c.dim()
        c = c.permute(*range(n - 8), n - 4, n - 8, n - 7, n - 6, n - 2, n - 3, n - 5, n - 1)
    lead = code.shape[:-2]
    return torch.cat([c.reshape(*lead, -1), dm.contiguous().view(torch.uint8).reshape(*lead, -1)], -1)


def _unpack(block, hd, side):
    """A block's bytes [..., n] as codes [..., PAGE, hd] and pairs [..., PAGE, groups, 2]."""
    lead, slab = block.shape[:-1], min(hd, 128)
    at = PAGE * hd // 2
    c = block[..., :at]
    if side == 0:
        c = c.view(*lead, hd // slab, PAGE, 4, slab // 64, 2, 4)
        n = c.dim()
        c = c.permute(*range(n - 6), n - 5, n - 6, n - 3, n - 4, n - 2, n - 1)
    else:
        c = c.view(*lead, hd // slab, 4, 2, 4, 8, slab // 32, 2, 2)
        n = c.dim()
        c = c.permute(*range(n - 8), n - 7, n - 6, n - 5, n - 2, n - 8, n - 3, n - 4, n - 1)
    code = torch.stack([c & 15, c >> 4], -1).reshape(*lead, PAGE, hd)
    dm = block[..., at:].contiguous().view(torch.float16).view(*lead, PAGE, hd // GROUP, 2)
    return code, dm


def _values(code, dm):
    """What the codes stand for, in 32 bits."""
    dm = dm.double()
    x = code.unflatten(-1, (-1, GROUP)).double() * dm[..., :1] + dm[..., 1:]
    return x.flatten(-2).float()


# ---- plain forms -----------------------------------------------------------
def _rope_rows(s):
    rows, hd = s["x"].shape[0], s["hd"]
    x = s["x"].float().view(rows, -1, hd)
    pos = s["pos"].long()
    live = (pos >= 0)[:, None, None]
    cos, sin = (s[t][pos.clamp(min=0)][:, None] for t in ("cos", "sin"))

    def side(h, w):
        if s["norm"]:
            h = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + 1e-6) * w
        if s["halves"]:
            a, b = h[..., : hd // 2], h[..., hd // 2:]
            return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
        a, b = h[..., 0::2], h[..., 1::2]
        return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)

    q = side(x[:, : s["heads"]], s["wq"]).to(s["dtype"])
    k = side(x[:, s["heads"]: s["heads"] + s["kv"]], s["wk"]).to(s["dtype"])
    return {"q": torch.where(live, q, s["q_out"]), "k": torch.where(live, k, s["k_out"])}


def _rows_of(s):
    """Each row's sequence, its position there, and whether it is one (padding rows are none)."""
    row = torch.arange(s["rows"], device=DEV)
    start = s["row_start"].long()
    seq = torch.searchsorted(start, row, right=True) - 1
    live = row < start[-1]
    seq = torch.where(live, seq, 0)
    pos = s["kv_len"].long()[seq] - (start[seq + 1] - row)
    live = live & (pos >= 0)
    return seq, torch.where(live, pos, 0), live


def _cache_pass(s):
    seq, pos, live = _rows_of(s)
    hd, kv, rows = s["hd"], s["kv"], s["rows"]
    page, at = s["table"][seq, pos // PAGE].long().clamp(min=0), pos % PAGE
    half = PAGE * hd // 2
    got = {}
    for side, name in ((0, "k"), (1, "v")):
        where = _code_places(hd, side)[at]                      # [rows, hd]: 2 * byte + (0 low, 1 high) of a block
        pair = half + (at[:, None, None] * (hd // GROUP) + torch.arange(hd // GROUP, device=DEV)[:, None]) * 4 + torch.arange(
            4, device=DEV)                                      # [rows, groups, 4] bytes of (d, m)
        head = torch.arange(kv, device=DEV)
        blocks = s["cache"][:, :, side]
        if s["write"]:
            nq = s["heads"] * hd
            x = s["qkv"][:, nq + side * kv * hd: nq + (side + 1) * kv * hd].reshape(rows, kv, hd)
            code, dm = _quantise(x)
            ok = live.nonzero().squeeze(1)
            # two codes to a byte: a byte's low and high code belong to one row
            low, high = code[:, :, 0::2], code[:, :, 1::2]
            byte = where[:, 0::2] // 2
            blocks[page[ok][:, None, None], head[:, None], byte[ok][:, None]] = (low | high << 4)[ok]
            blocks[page[ok][:, None, None], head[:, None], pair[ok].flatten(1)[:, None]] = dm[ok].view(torch.uint8).reshape(-1, kv, 4 * (hd // GROUP))
        code = blocks[page[:, None, None], head[:, None], (where // 2)[:, None]] >> (4 * (where % 2))[:, None].to(torch.uint8) & 15
        dm = blocks[page[:, None, None], head[:, None], pair.flatten(1)[:, None]].view(torch.float16).view(rows, kv, -1, 2)
        got[name] = torch.where(live[:, None, None], _values(code, dm).to(s["dtype"]), s[name + "_out"])
    return got


def _code_places(hd, side):
    """[PAGE, hd]: where a block keeps the code of each position and dimension, as 2 * byte + half."""
    at, slab = torch.arange(PAGE * hd // 2, device=DEV), min(hd, 128)
    if side == 0:
        c = at.view(hd // slab, PAGE, 4, slab // 64, 2, 4).permute(1, 0, 3, 2, 4, 5)
    else:
        c = at.view(hd // slab, 4, 2, 4, 8, slab // 32, 2, 2).permute(1, 2, 3, 6, 0, 5, 4, 7)
    return torch.stack([2 * c, 2 * c + 1], -1).reshape(PAGE, hd)


def _attend_rows(s):
    hd, kv, heads, most = s["hd"], s["kv"], s["heads"], s["most"]
    n, per_seq = s["table"].shape
    seq, pos, live = _rows_of(s)
    at = torch.arange(s["rows"], device=DEV) - s["row_start"].long()[seq]
    at = torch.where(live, at, 0)
    # [seqs, most, heads, hd]: every sequence's rows, the absent ones with no position to see
    q = torch.zeros(n, most, heads, hd, device=DEV)
    seen = torch.full((n, most), -1, device=DEV)
    ok = live.nonzero().squeeze(1)
    q[seq[ok], at[ok]] = s["q"][ok].float()
    seen[seq[ok], at[ok]] = pos[ok]
    pages = s["cache"][s["table"].long().clamp(min=0)]          # [seqs, pages, kv, 2, bytes]
    k, v = (_values(*_unpack(pages[:, :, :, side], hd, side)) for side in (0, 1))
    k, v = (x.transpose(2, 3).reshape(n, per_seq * PAGE, kv, hd) for x in (k, v))
    q = q.view(n, most, kv, heads // kv, hd)
    score = torch.einsum("stgnd,slgd->sgntl", q, k) * (1 / math.sqrt(hd))
    hidden = torch.arange(per_seq * PAGE, device=DEV) > seen[:, None, None, :, None]
    score = score.masked_fill(hidden, -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(top == -math.inf, 0, top))
    total = weight.sum(-1)
    o = torch.einsum("sgntl,slgd->stgnd", weight, v)
    total = total.permute(0, 3, 1, 2)[..., None]
    o = torch.where(total > 0, o / total, 0).view(n, most, heads, hd).to(s["dtype"])
    inside = torch.arange(s["rows"], device=DEV) < s["row_start"][-1]
    return {"out": torch.where(inside[:, None, None], o[seq, at], s["out"])}


def run(s):
    if own:
        import rustfox_b200 as rf
        if s["op"] == "rope":
            q, k = rf.qk_norm_rope(s["x"], s["heads"], s["kv"], s["hd"], s["pos"], s["cos"], s["sin"], q_norm=s["wq"],
                                   k_norm=s["wk"], eps=1e-6, halves=s["halves"], q_out=s["q_out"], k_out=s["k_out"])
            return {"q": q, "k": k}
        if s["op"] == "cache":
            if s["write"]:
                rows, nq, nkv = s["rows"], s["heads"] * s["hd"], s["kv"] * s["hd"]
                rf.kv4_write(s["cache"], s["table"], s["row_start"], s["kv_len"], s["qkv"][:, nq:nq + nkv],
                             s["qkv"][:, nq + nkv:])
            k, v = rf.kv4_read(s["cache"], s["table"], s["row_start"], s["kv_len"], k_out=s["k_out"], v_out=s["v_out"])
            return {"k": k, "v": v}
        return {"out": rf.kv4_attention(s["q"], s["cache"], s["table"], s["row_start"], s["kv_len"], out=s["out"])}
    return {"rope": _rope_rows, "cache": _cache_pass, "attend": _attend_rows}[s["op"]](s)


# ---- the definition, in 64 bits --------------------------------------------
def _exact_rope(s):
    hd, out = s["hd"], {}
    at = s["pos"].long()
    for name, first, count, w in (("q", 0, s["heads"], s["wq"]), ("k", s["heads"], s["kv"], s["wk"])):
        h = s["x"].double()[:, first * hd:(first + count) * hd].reshape(-1, count, hd)
        if w is not None:
            h = h / torch.sqrt(h.pow(2).sum(-1, keepdim=True) / hd + 1e-6) * w.double()
        i = torch.arange(hd // 2, device=DEV)
        a, b = (i, i + hd // 2) if s["halves"] else (2 * i, 2 * i + 1)
        turn = torch.complex(s["cos"].double(), s["sin"].double())[at.clamp(min=0)][:, None, :]
        z = torch.complex(h[..., a], h[..., b]) * turn
        y = torch.zeros_like(h)
        y[..., a], y[..., b] = z.real, z.imag
        y[at < 0] = 0
        out[name] = y
    return out


def _exact_level(x, times, up):
    """The fp16 number h next to x / times (64 bits) with times * h on the side of x asked for, found by stepping
    from the nearest one."""
    bits = (x / times).float().half().view(torch.int16).int()
    rank = torch.where(bits < 0, -(bits & 0x7FFF), bits)        # order of fp16 numbers as whole numbers
    value = lambda r: times * torch.where(r < 0, -r | 0x8000, r).to(torch.int16).view(torch.float16).double()  # noqa: E731
    for _ in range(2):
        rank = torch.where(value(rank) < x, rank + 1, rank) if up else torch.where(value(rank) > x, rank - 1, rank)
    for _ in range(2):
        rank = torch.where(value(rank - 1) >= x, rank - 1, rank) if up else torch.where(value(rank + 1) <= x, rank + 1, rank)
    return value(rank) / torch.full_like(x, times)


def _exact_round_trip(x):
    g = x.double().unflatten(-1, (-1, GROUP))
    m = _exact_level(g.amin(-1), 1, False)[..., None]
    d = _exact_level(g.amax(-1) - m[..., 0], 15, True)[..., None]
    levels = m + d * torch.arange(16, device=DEV, dtype=torch.float64)
    # the nearer of the two levels around x; a tie goes to the even code
    step = (g[..., None] >= levels[..., None, 1:15]).sum(-1)
    below, above = torch.gather(levels, -1, step), torch.gather(levels, -1, step + 1)
    take = (above - g < g - below) | ((above - g == g - below) & (step % 2 == 1))
    return torch.where(take & (d > 0), above, below).flatten(-2)


def _exact_positions(s, seq, first, count):
    """K and V of a sequence's positions first .. first+count-1 in 64 bits, nibble by nibble."""
    hd, kv = s["hd"], s["kv"]
    p = torch.arange(first, first + count, device=DEV)
    blocks = s["cache"][s["table"][seq].long()[p // PAGE]]       # [count, kv, 2, bytes]
    p, d = (p % PAGE)[:, None], torch.arange(hd, device=DEV)
    slab, r = d // 128, d % 128
    wide = min(hd, 128)
    kb = slab * (PAGE * wide // 2) + p * (wide // 2) + 4 * ((r % 64 // 16) * 2 * (wide // 64) + 2 * (r // 64) + r % 16 // 8) + r % 8 // 2
    word = (((slab * 4 + p // 16) * 2 + p // 8 % 2) * 4 + p % 8 // 2) * 8 + r % 32 // 4
    vb = 4 * (word * (wide // 32) + r // 32) + 2 * (p % 2) + r % 4 // 2
    pairs = blocks[..., PAGE * hd // 2:].contiguous().view(torch.float16).view(count, kv, 2, PAGE, hd // GROUP, 2)
    pairs = pairs[torch.arange(count, device=DEV), :, :, p[:, 0]].double()      # [count, kv, 2, groups, 2]
    out = []
    for side, place in ((0, kb), (1, vb)):
        byte = torch.gather(blocks[:, :, side], 2, place[:, None].expand(count, kv, hd))
        code = torch.where(d % 2 == 0, byte % 16, byte // 16).double()
        dm = pairs[:, :, side].repeat_interleave(GROUP, -2)
        out.append(code * dm[..., 0] + dm[..., 1])
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "rope":
        return _exact_rope(s)
    hd, kv, heads, rows = s["hd"], s["kv"], s["heads"], s["rows"]
    start, lens = s["row_start"].tolist(), s["kv_len"].tolist()
    if s["op"] == "cache":
        out = {n: torch.zeros(rows, kv, hd, dtype=torch.float64, device=DEV) for n in "kv"}
        for q, L in enumerate(lens):
            a, b = start[q], start[q + 1]
            if a == b:
                continue
            if s["write"]:
                new = s["qkv"][a:b, heads * hd:].reshape(b - a, 2, kv, hd)
                out["k"][a:b], out["v"][a:b] = _exact_round_trip(new[:, 0]), _exact_round_trip(new[:, 1])
            else:
                out["k"][a:b], out["v"][a:b] = _exact_positions(s, q, L - (b - a), b - a)
        return out
    out = torch.zeros(rows, heads, hd, dtype=torch.float64, device=DEV)
    for q, L in enumerate(lens):
        a, b = start[q], start[q + 1]
        if a == b or L == 0:
            continue
        k, v = _exact_positions(s, q, 0, L)
        x = s["q"][a:b].double().view(b - a, kv, heads // kv, hd) / math.sqrt(hd)
        last = L - (b - a) + torch.arange(b - a, device=DEV)
        future = torch.arange(L, device=DEV) > last[:, None]
        for h in range(kv):
            z = torch.tensordot(x[:, h], k[:, h], dims=([2], [1])).masked_fill(future[:, None], -math.inf)
            out[a:b].view(b - a, kv, heads // kv, hd)[:, h] = torch.softmax(z, -1) @ v[:, h]
    return {"out": out}
