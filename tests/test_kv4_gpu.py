"""The 4-bit paged K/V cache (foxcuda_kv4_*) and foxcuda_qk_norm_rope against
the definition in 64 bits (tests/kv4_ref.py).

- The quantiser and the read-back are exact: every byte of the cache, and
  every fp32 value read back, is the definition's (m + d * code fits fp32's
  24 bits but for its last rounding, which the reference repeats).
- Attention. fp32 rows: q and p d enter as hi + lo fp16 (2^-22 of them), the
  products' sums round at 2^-19 of their largest addend (2^-23, times 2^4 for
  the leading zeros of a subnormal operand); over the 64 addends of a group
  those roundings are independent and the weights average them, so the result
  is within a few times 2^-19 = 2e-6 of its norm. The bound is 1e-5. fp16 rows:
  the result is rounded once, 2^-11 of a value at most, which adds 5e-4.
- Rotation: fp32 is one product, one sum and at most four roundings of the
  norm away, 8 half steps of 2^-24 of the pair's length; fp16 adds its own."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

import kv4_ref as R  # noqa: E402
import rustfox_b200 as rf  # noqa: E402

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16}
TOL = {"f32": 1e-5, "f16": 1e-5 + 2.0 ** -11}


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).to(DEV)
    return t if dtype is None else t.to(dtype)


def i32(a):
    return torch.tensor(list(a), dtype=torch.int32, device=DEV)


def host(t):
    return t.cpu().numpy()


class Cache:
    """Sequences of the given lengths over scattered pages; the bytes of the
    pool are noise (NaN parameters among them) until something is written."""

    def __init__(self, lens, kv, hd, seed=0, spare=2, fill=True, stride=None):
        rng = np.random.default_rng(seed)
        need = [-(-L // R.PAGE) for L in lens]
        stride = stride or max(max(need), 1)
        pages = rng.permutation(sum(need) + spare)
        self.table = np.full((len(lens), stride), -7, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = pages[at:at + n]
            at += n
        self.data = rng.integers(0, 256, (len(pages), kv, 2, R.block_bytes(hd)), dtype=np.uint8)
        self.lens, self.kv, self.hd, self.rng = list(lens), kv, hd, rng
        if fill:
            for s, L in enumerate(lens):
                if L:
                    k = self.values(L) + self.channel()
                    R.put(self.data, self.table, s, np.arange(L), k, self.values(L))

    def channel(self):
        return 2 * self.rng.normal(0, 1, (self.kv, self.hd)) * (self.rng.random((self.kv, self.hd)) < 0.1)

    def values(self, n):
        return self.rng.normal(0, 1, (n, self.kv, self.hd)) * np.exp(0.5 * self.rng.normal(0, 1, (n, self.kv, 1)))

    def on_device(self):
        return dev(self.data), dev(self.table)


def starts(rows):
    return np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)


# ---- write and read --------------------------------------------------------
@pytest.mark.parametrize("hd,kv", [(64, 1), (64, 8), (128, 2), (256, 3)])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_write_gives_the_definitions_bytes_and_nothing_else(hd, kv, dtype):
    lens, rows, pad = [1, 64, 0, 65, 130, 7], [1, 3, 0, 65, 66, 9], 3  # the last has more rows than positions
    c = Cache(lens, kv, hd, seed=hd + kv, fill=False)
    n = sum(rows) + pad
    start = starts(rows)
    # rows as a slice of wider rows (the fused q|k|v product's)
    wide = c.rng.normal(0, 1, (n, 64 + 2 * kv * hd + 16)) * np.exp(c.rng.normal(0, 3, (n, 1)))
    x = dev(wide, TYPES[dtype])
    k, v = x[:, 64:64 + kv * hd], x[:, 64 + kv * hd:64 + 2 * kv * hd]
    cache, table = c.on_device()
    rf.kv4_write(cache, table, i32(start), i32(lens), k, v)
    for s, L in enumerate(lens):
        a, b = start[s], start[s + 1]
        have = min(b - a, L)
        sel = slice(b - have, b)
        R.put(c.data, c.table, s, np.arange(L - have, L), host(k[sel].double()).reshape(-1, kv, hd),
              host(v[sel].double()).reshape(-1, kv, hd))
    assert np.array_equal(host(cache), c.data)
    # read back what was written
    k2, v2 = (torch.full((n, kv, hd), 7.5, dtype=TYPES[dtype], device=DEV) for _ in "kv")
    rf.kv4_read(cache, table, i32(start), i32(lens), k_out=k2, v_out=v2)
    want = [np.full((n, kv, hd), 7.5) for _ in "kv"]
    for s, L in enumerate(lens):
        b = start[s + 1]
        have = min(b - start[s], L)
        for side, x in enumerate(R.get(c.data, c.table, s, np.arange(L - have, L))):
            want[side][b - have:b] = x
    for got, w in zip((k2, v2), want):
        w = torch.from_numpy(w).float().to(TYPES[dtype])
        assert torch.equal(got.cpu(), w)
    rf.kernel_errors()


def test_groups_at_the_edges_of_the_format():
    """Equal values, zeros, values beyond fp16, infinities, NaN, subnormal
    steps, and values that lie exactly between two levels."""
    hd, kv = 128, 1
    g = []
    ramp = np.arange(64) % 16
    g += [np.zeros(64), np.full(64, -0.0), np.full(64, 3.3), np.full(64, 1e30), np.full(64, 6e-8), np.full(64, -1e-9)]
    g += [np.where(ramp == 3, np.inf, ramp), np.where(ramp == 3, -np.inf, 1.0), np.where(ramp == 5, np.nan, ramp)]
    g += [ramp * 0.25, ramp * 0.25 + 0.125, np.where(ramp == 15, 15.0, ramp % 15 + 0.5), ramp * 2.0 ** -24,
          ramp * 2.0 ** -23 + 2.0 ** -24, np.linspace(-65504, 65504, 64), np.linspace(-1e6, 1e6, 64)]
    g += [100 + ramp * 1e-3, 0.1 + np.arange(64) * 1e-9, np.nextafter(np.float32(1.5), 2) * np.ones(64),
          np.where(ramp == 0, 0.0, np.nextafter(np.float32(7.5), np.float32(8 * (ramp % 2)))),
          np.where(ramp == 0, 0.0, np.where(ramp == 1, 15.0, np.float32(0.5) + ramp // 2 * 1.0))]
    # borders met from both sides by less than fp32 keeps of x - m
    g += [np.where(ramp == 0, -1.0, np.where(ramp == 1, 14.0, (ramp - 0.5) + (-1.0) ** ramp * 1e-9))]
    if len(g) % 2:
        g.append(np.ones(64))
    x = np.array(g, np.float32).reshape(-1, kv, hd)
    n = len(x)
    c = Cache([n], kv, hd, fill=False)
    cache, table = c.on_device()
    t = dev(x)
    rf.kv4_write(cache, table, i32([0, n]), i32([n]), t, t)
    got, _ = rf.kv4_read(cache, table, i32([0, n]), i32([n]), n)
    R.put(c.data, c.table, 0, np.arange(n), x, x)
    want = R.get(c.data, c.table, 0, np.arange(n))[0].astype(np.float32)
    assert np.array_equal(host(got), want, equal_nan=True)
    assert np.isnan(want).sum() == 64 and np.isfinite(np.delete(want.reshape(-1, 64), 8, 0)).all()


def test_random_groups_bit_for_bit():
    """Many groups of every size of step, as fp32: the codes are decided
    exactly, so not one differs."""
    hd, kv, n = 256, 4, 4096
    rng = np.random.default_rng(3)
    x = rng.normal(0, 1, (n, kv, hd)) * np.exp(rng.normal(0, 4, (n, kv, 1))) + rng.normal(0, 1, (n, kv, 1)) * 10
    x = x.astype(np.float32)
    c = Cache([n], kv, hd, fill=False)
    cache, table = c.on_device()
    rf.kv4_write(cache, table, i32([0, n]), i32([n]), dev(x), dev(-x))
    k, v = rf.kv4_read(cache, table, i32([0, n]), i32([n]), n)
    for got, y in ((k, x), (v, -x)):
        want = R.values(*R.quantise(y)).astype(np.float32)
        assert np.array_equal(host(got), want), np.count_nonzero(host(got) != want)


# ---- norms and rotation ----------------------------------------------------
def _rope_want(x, heads, kv, hd, pos, cos, sin, wq, wk, eps, halves):
    out = []
    for first, count, w in ((0, heads, wq), (heads, kv, wk)):
        h = x[:, first * hd:(first + count) * hd].astype(np.float64).reshape(len(x), count, hd)
        if w is not None:
            h = h / np.sqrt((h * h).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
        c, s = (a.astype(np.float64)[np.maximum(pos, 0)][:, None] for a in (cos, sin))
        i = np.arange(hd // 2)
        a, b = (i, i + hd // 2) if halves else (2 * i, 2 * i + 1)
        y = np.empty_like(h)
        y[..., a], y[..., b] = h[..., a] * c - h[..., b] * s, h[..., a] * s + h[..., b] * c
        out.append(y)
    return out


@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("norm", ["both", "q", "none"])
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 64), (32, 8, 128), (3, 1, 256)])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_rope_against_64_bits(heads, kv, hd, norm, halves, dtype):
    rng = np.random.default_rng(heads + hd)
    n, n_pos = 37, 500
    x = dev(rng.normal(0, 2, (n, (heads + 2 * kv) * hd)), TYPES[dtype])
    x[5] = 0  # a row of zeros: its norm is eps alone
    th = np.arange(n_pos)[:, None] * 1e4 ** (-2.0 * np.arange(hd // 2) / hd)
    cos, sin = np.cos(th).astype(np.float32), np.sin(th).astype(np.float32)
    pos = rng.integers(0, n_pos, n).astype(np.int32)
    pos[[0, 9, n - 1]] = [n_pos - 1, -1, -3]
    wq, wk = (rng.normal(1, 0.3, hd).astype(np.float32) for _ in "qk")
    wq, wk = (wq if norm != "none" else None), (wk if norm == "both" else None)
    q, k = (torch.full((n, h, hd), 3.25, dtype=TYPES[dtype], device=DEV) for h in (heads, kv))
    args = (heads, kv, hd, dev(pos), dev(cos), dev(sin))
    kw = dict(q_norm=None if wq is None else dev(wq), k_norm=None if wk is None else dev(wk), eps=1e-5, halves=halves)
    rf.qk_norm_rope(x, *args, q_out=q, k_out=k, **kw)
    want = _rope_want(host(x.double()), heads, kv, hd, pos, cos, sin, wq, wk, 1e-5, halves)
    step = 2.0 ** -24 * 8 + (2.0 ** -11 if dtype == "f16" else 0)
    for got, w in zip((q, k), want):
        got = host(got.double())
        live = pos >= 0
        size = np.maximum(np.abs(w).max(-1, keepdims=True), 1e-6)
        assert (np.abs(got - w) / size)[live].max() <= step
        assert (got[~live] == 3.25).all()
    # in place, the rows of x are their own output
    y = x.clone()
    nq = heads * hd
    q2, k2 = y[:, :nq].unflatten(1, (heads, hd)), y[:, nq:nq + kv * hd].unflatten(1, (kv, hd))
    rf.qk_norm_rope(y, *args, q_out=q2, k_out=k2, **kw)
    live = torch.from_numpy(pos >= 0).to(DEV)
    assert torch.equal(q2[live], q[live]) and torch.equal(k2[live], k[live])
    assert torch.equal(y[~live], x[~live]) and torch.equal(y[:, nq + kv * hd:], x[:, nq + kv * hd:])


def test_rope_without_norms_is_the_decode_steps_rotation():
    """Each product and sum rounded by itself, as upstream (src/ops.c:56-73)."""
    heads, kv, hd, n = 4, 2, 64, 50
    rng = np.random.default_rng(8)
    x = rng.normal(0, 1, (n, (heads + kv) * hd)).astype(np.float32)
    th = np.arange(n)[:, None] * 1e6 ** (-2.0 * np.arange(hd // 2) / hd)
    cos, sin = np.cos(th).astype(np.float32), np.sin(th).astype(np.float32)
    q, k = rf.qk_norm_rope(dev(x), heads, kv, hd, i32(range(n)), dev(cos), dev(sin))
    h = x.reshape(n, heads + kv, hd)
    c, s = cos[:, None], sin[:, None]
    a, b = h[..., 0::2], h[..., 1::2]
    want = np.stack([(a * c).astype(np.float32) - (b * s).astype(np.float32),
                     (a * s).astype(np.float32) + (b * c).astype(np.float32)], -1).reshape(h.shape)
    got = np.concatenate([host(q), host(k)], 1)
    assert np.array_equal(got.view(np.uint32), want.view(np.uint32))


def test_rope_position_beyond_the_tables_is_skipped_and_reported():
    x = torch.randn(3, 6 * 64, device=DEV)
    cos = torch.ones(4, 32, device=DEV)
    q = torch.full((3, 4, 64), 9.0, device=DEV)
    rf.kernel_errors()
    rf.qk_norm_rope(x, 4, 2, 64, i32([0, 4, 3]), cos, torch.zeros_like(cos), q_out=q)
    with pytest.raises(rf.FoxError, match="outside"):
        rf.kernel_errors()
    rf.kernel_errors()  # read once
    assert (q[1] == 9).all() and torch.equal(q[[0, 2]].reshape(2, -1), x[[0, 2], :256])


# ---- attention -------------------------------------------------------------
def _attend(c, q, rows, lens, out0=None, **kw):
    cache, table = c.on_device()
    out = None if out0 is None else dev(out0, q.dtype)
    got = rf.kv4_attention(q, cache, table, i32(starts(rows)), i32(lens), out=out, **kw)
    return host(got.double())


def _close(got, want, dtype, what=""):
    assert np.isfinite(got).all(), what
    err = np.linalg.norm(got - want) / max(np.linalg.norm(want), 1e-30)
    assert err <= TOL[dtype], (what, err)
    # and each row by itself
    rows = np.linalg.norm((got - want).reshape(len(got), -1), axis=1)
    size = np.linalg.norm(want.reshape(len(want), -1), axis=1)
    assert (rows <= 3 * TOL[dtype] * size + 1e-30).all(), (what, (rows / np.maximum(size, 1e-30)).max())


SHAPES = [(8, 2, 64), (2, 2, 64), (4, 2, 128), (32, 8, 128), (16, 2, 128), (8, 1, 256), (4, 4, 256)]


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("heads,kv,hd", SHAPES)
def test_single_tokens_of_ragged_sequences(heads, kv, hd, dtype):
    lens = [1, 2, 63, 64, 65, 0, 127, 129, 300, 1000]
    rows = [1] * 9 + [1]
    rows[1] = 0  # a sequence without a row this time
    c = Cache(lens, kv, hd, seed=heads + hd)
    n = sum(rows) + 2
    q = dev(c.rng.normal(0, 1, (n, heads, hd)), TYPES[dtype])
    out0 = np.full((n, heads, hd), 0.375)
    got = _attend(c, q, rows, lens, out0)
    want = R.attend(host(q.double()), c.data, c.table, starts(rows), lens, out0)
    _close(got, want, dtype)
    assert (got[-2:] == 0.375).all()  # padding rows
    assert (got[4] == 0).all()        # the row that sees nothing (sequence 5)
    rf.kernel_errors()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("heads,kv,hd", SHAPES)
def test_chunks_of_rows(heads, kv, hd, dtype):
    """Rows see up to their own position; sequences of no rows, of one, of
    more rows than positions; row counts that end inside a tile."""
    lens, rows = [64, 200, 5, 33, 700, 0], [64, 7, 9, 1, 19, 2]
    c = Cache(lens, kv, hd, seed=heads * hd)
    n = sum(rows) + 1
    q = dev(c.rng.normal(0, 1, (n, heads, hd)), TYPES[dtype])
    out0 = np.full((n, heads, hd), -2.0)
    got = _attend(c, q, rows, lens, out0)
    want = R.attend(host(q.double()), c.data, c.table, starts(rows), lens, out0)
    _close(got, want, dtype)
    a = starts(rows)[2]
    assert (got[a:a + 4] == 0).all() and (got[-1] == -2).all()
    rf.kernel_errors()


@pytest.mark.parametrize("heads,kv,hd,length,rows", [(8, 2, 64, 20001, 1), (32, 8, 128, 9000, 3), (16, 2, 128, 6001, 70),
                                                     (8, 2, 256, 4097, 2)])
def test_long_sequences_are_split_and_joined(heads, kv, hd, length, rows):
    c = Cache([length, 130], kv, hd, seed=length)
    n = rows + 1
    q = dev(c.rng.normal(0, 1, (n, heads, hd))).float()
    got = _attend(c, q, [rows, 1], [length, 130])
    want = R.attend(host(q.double()), c.data, c.table, starts([rows, 1]), [length, 130], np.zeros((n, heads, hd)))
    _close(got, want, "f32")


@pytest.mark.parametrize("scale", [0.0, 0.02, 3.0])
@pytest.mark.parametrize("size", [1e-20, 1e-3, 1.0, 300.0, 1e15])
def test_scales_and_sizes_of_queries(scale, size):
    """Softmax from flat to one-hot. A score z is off by at most 2^-19 |z| or
    so, and the weight by as much times the score: the bound follows the
    largest score, up to the sizes where no precision is left."""
    heads, kv, hd, L = 8, 2, 128, 333
    c = Cache([L], kv, hd, seed=4)
    q = dev(size * c.rng.normal(0, 1, (1, heads, hd))).float()
    got = _attend(c, q, [1], [L], scale=scale)
    assert np.isfinite(got).all()
    want = R.attend(host(q.double()), c.data, c.table, [0, 1], [L], np.zeros((1, heads, hd)), scale=scale or None)
    k = R.get(c.data, c.table, 0, np.arange(L))[0]
    z = np.abs(np.einsum("hd,lhd->hl", np.abs(host(q.double())[0]).reshape(kv, -1, hd).max(1), np.abs(k))).max()
    tol = 1e-5 + 2.0 ** -19 * z * (scale or hd ** -0.5)
    if tol < 0.1:
        assert np.linalg.norm(got - want) <= tol * np.linalg.norm(want)


@pytest.mark.parametrize("size", [1e-7, 1e-3, 1.0, 1e3, 4e4])
def test_sizes_of_values(size):
    """The scaling of the weights follows V's steps, from fp16's smallest to
    its largest, and positions of very different size side by side."""
    heads, kv, hd, L = 4, 2, 64, 500
    c = Cache([L], kv, hd, seed=5, fill=False)
    v = size * np.clip(c.values(L), -1.5, 1.5)
    v[::7] *= 1e-3
    R.put(c.data, c.table, 0, np.arange(L), c.values(L), v)
    q = dev(c.rng.normal(0, 1, (1, heads, hd))).float()
    got = _attend(c, q, [1], [L])
    want = R.attend(host(q.double()), c.data, c.table, [0, 1], [L], np.zeros((1, heads, hd)))
    _close(got, want, "f32")


def test_hidden_positions_may_hold_anything():
    """NaN and infinities in positions a row does not see, behind a sequence's
    end and in its future, change nothing (the pool's noise holds both); in
    one it does see, a NaN reaches the rows that see it and no others."""
    heads, kv, hd, L, T = 8, 2, 128, 70, 6
    c = Cache([L], kv, hd, seed=6)
    q = dev(c.rng.normal(0, 1, (T, heads, hd))).float()
    want = R.attend(host(q.double()), c.data, c.table, [0, T], [L], np.zeros((T, heads, hd)))
    at = L - 2  # seen by the last two rows
    for side in (0, 1):
        d = c.data.copy()
        n = 4 * (hd // R.GROUP)
        p = at % R.PAGE
        c.data[c.table[0, at // R.PAGE], :, side, R.PAGE * hd // 2 + p * n: R.PAGE * hd // 2 + (p + 1) * n] = 0xFF
        got = _attend(c, q, [T], [L])
        _close(got[:T - 2], want[:T - 2], "f32")
        assert np.isnan(got[T - 2:]).all()
        c.data = d
    # NaN and infinite queries stay in their own row and head
    q[0, 0, 3], q[1, 1, 5] = float("nan"), float("inf")
    got = _attend(c, q, [T], [L])
    bad = np.zeros((T, heads), bool)
    bad[0, 0] = bad[1, 1] = True
    assert np.isnan(got[bad]).all()
    _close(got[~bad], want[~bad], "f32")


def test_the_same_call_gives_the_same_bits():
    """And a row beside other sequences what it gets alone, but for where the
    sums are split."""
    heads, kv, hd = 16, 4, 128
    lens = [777, 5, 3000, 64, 1500]
    c = Cache(lens, kv, hd, seed=9)
    q = dev(c.rng.normal(0, 1, (5, heads, hd))).float()
    cache, table = c.on_device()
    whole = rf.kv4_attention(q, cache, table, i32(range(6)), i32(lens))
    for _ in range(3):
        assert torch.equal(rf.kv4_attention(q, cache, table, i32(range(6)), i32(lens)), whole)
    for s in range(5):
        one = rf.kv4_attention(q[s:s + 1], cache, table[s:s + 1].contiguous(), i32([0, 1]), i32(lens[s:s + 1]))
        _close(host(one.double()), host(whole[s:s + 1].double()), "f32", s)


def test_many_sequences_and_shared_pages():
    """Sequences that share a prefix's pages; more sequences than a warp scans
    at once."""
    heads, kv, hd, n = 8, 2, 64, 150
    c = Cache([256], kv, hd, seed=10)
    table = np.repeat(c.table, n, 0)
    lens = c.rng.integers(0, 257, n)
    q = dev(c.rng.normal(0, 1, (n, heads, hd))).float()
    got = host(rf.kv4_attention(q, dev(c.data), dev(table), i32(range(n + 1)), i32(lens)).double())
    want = R.attend(host(q.double()), c.data, table, np.arange(n + 1), lens, np.zeros((n, heads, hd)))
    _close(got, want, "f32")
    k, v = rf.kv4_read(dev(c.data), dev(table), i32(range(n + 1)), i32(lens), n)
    for s in np.flatnonzero(lens):
        w = R.get(c.data, table, s, [lens[s] - 1])
        assert np.array_equal(host(k)[s], w[0][0].astype(np.float32)) and np.array_equal(host(v)[s], w[1][0].astype(np.float32))


def test_pages_outside_the_cache_and_lengths_outside_the_table():
    """What the device arrays place out of bounds is skipped, as if it were
    absent, and reported; the rest is as it should be."""
    heads, kv, hd = 4, 2, 128
    lens = [200, 100]
    c = Cache(lens, kv, hd, seed=11)
    bad = c.table.copy()
    bad[0, 1] = len(c.data)      # one past the last page
    bad[1, 0] = -1
    q = dev(c.rng.normal(0, 1, (2, heads, hd))).float()
    rf.kernel_errors()
    got = host(rf.kv4_attention(q, dev(c.data), dev(bad), i32([0, 1, 2]), i32(lens)).double())
    with pytest.raises(rf.FoxError, match="outside"):
        rf.kernel_errors()
    gone = {0: 1, 1: 0}
    want = R.attend(host(q.double()), c.data, c.table, [0, 1, 2], lens, np.zeros((2, heads, hd)),
                    seen=lambda s, p: p // R.PAGE != gone[s])
    _close(got, want, "f32")
    # rows of an absent page are neither written nor read back
    cache = dev(c.data)
    x = torch.ones(100, kv, hd, device=DEV)
    rf.kv4_write(cache, dev(bad), i32([0, 0, 100]), i32(lens), x, x)
    with pytest.raises(rf.FoxError):
        rf.kernel_errors()
    R.put(c.data, c.table, 1, np.arange(64, 100), *(np.ones((36, kv, hd)) for _ in "kv"))
    assert np.array_equal(host(cache), c.data)
    # a length beyond the table is held to it
    got = host(rf.kv4_attention(q, cache, dev(c.table), i32([0, 1, 2]), i32([10 ** 6, 100])).double())
    with pytest.raises(rf.FoxError):
        rf.kernel_errors()
    want = R.attend(host(q.double()), c.data, c.table, [0, 1, 2], [c.table.shape[1] * 64, 100], np.zeros((2, heads, hd)))
    assert np.allclose(got[1], want[1], rtol=0, atol=1e-4)


def test_caches_beyond_four_gigabytes():
    kv, hd, heads = 8, 128, 8
    pages = (1 << 32) // (kv * 2 * R.block_bytes(hd)) + 70
    small = Cache([150], kv, hd, seed=12)
    cache = torch.empty(pages, kv, 2, R.block_bytes(hd), dtype=torch.uint8, device=DEV)
    table = np.array([[pages - 1, 3, pages - 2]], np.int32)
    for i in range(3):
        cache[int(table[0, i])] = dev(small.data[small.table[0, i]])
    q = dev(small.rng.normal(0, 1, (1, heads, hd))).float()
    got = host(rf.kv4_attention(q, cache, dev(table), i32([0, 1]), i32([150])).double())
    want = R.attend(host(q.double()), small.data, small.table, [0, 1], [150], np.zeros((1, heads, hd)))
    _close(got, want, "f32")
    x = torch.randn(1, kv, hd, device=DEV)
    rf.kv4_write(cache, dev(table), i32([0, 1]), i32([151]), x, x)
    k, _ = rf.kv4_read(cache, dev(table), i32([0, 1]), i32([151]), 1)
    assert np.array_equal(host(k), R.values(*R.quantise(host(x))).astype(np.float32))


# ---- together --------------------------------------------------------------
def _step(st, x, pos, row_start, kv_len, work=None):
    """One layer's attention part: norms and rotation in place, the cache's
    write, the attention."""
    heads, kv, hd = st["heads"], st["kv"], st["hd"]
    nq, nk = heads * hd, kv * hd
    q, k = x[:, :nq].unflatten(1, (heads, hd)), x[:, nq:nq + nk].unflatten(1, (kv, hd))
    rf.qk_norm_rope(x, heads, kv, hd, pos, st["cos"], st["sin"], q_norm=st["wq"], k_norm=st["wk"], q_out=q, k_out=k)
    rf.kv4_write(st["cache"], st["table"], row_start, kv_len, k, x[:, nq + nk:])
    return rf.kv4_attention(q, st["cache"], st["table"], row_start, kv_len, out=st["out"], workspace=work)


def _setup(heads, kv, hd, n_seq, stride, rows, seed=1):
    rng = np.random.default_rng(seed)
    th = np.arange(stride * 64)[:, None] * 1e6 ** (-2.0 * np.arange(hd // 2) / hd)
    pages = rng.permutation(n_seq * stride).reshape(n_seq, stride).astype(np.int32)
    return dict(heads=heads, kv=kv, hd=hd, cos=dev(np.cos(th)).float(), sin=dev(np.sin(th)).float(),
                wq=dev(rng.normal(1, 0.2, hd)).float(), wk=dev(rng.normal(1, 0.2, hd)).float(),
                cache=rf.kv4_cache(n_seq * stride, kv, hd, DEV), table=dev(pages),
                out=torch.zeros(rows, heads, hd, device=DEV)), rng


def test_prompt_chunks_and_steps_against_plain_attention():
    """Two sequences, prompts in chunks and then single tokens: every row's
    output against 64 bits over the values the cache stands for, and those
    against the rotated keys within half a step."""
    heads, kv, hd = 8, 2, 64
    st, rng = _setup(heads, kv, hd, 2, 4, 40)
    have = [0, 0]
    for rows in ([40, 0], [25, 15], [1, 1], [0, 39], [1, 1], [1, 1]):
        n = 40
        x = dev(rng.normal(0, 1, (n, (heads + 2 * kv) * hd))).float()
        pos = np.full(n, -1, np.int32)
        start = starts(rows)
        for s in (0, 1):
            pos[start[s]:start[s + 1]] = have[s] + np.arange(rows[s])
            have[s] += rows[s]
        y = x.clone()
        out = _step(st, y, dev(pos), i32(start), i32(have))
        q = host(y[:, :heads * hd].double()).reshape(n, heads, hd)
        want = R.attend(q, host(st["cache"]), host(st["table"]), start, have, np.zeros((n, heads, hd)))
        m = start[-1]
        _close(host(out.double())[:m], want[:m], "f32", rows)
        wq, wk = host(st["wq"]), host(st["wk"])
        roped = _rope_want(host(x.double()), heads, kv, hd, pos, host(st["cos"]), host(st["sin"]), wq, wk, 1e-5, False)[1]
        for s in (0, 1):
            if rows[s]:
                got = R.get(host(st["cache"]), host(st["table"]), s, have[s] - rows[s] + np.arange(rows[s]))[0]
                w = roped[start[s]:start[s + 1]]
                assert np.abs(got - w).max() <= R.quantise(w)[1].max() * 0.51
    rf.kernel_errors()


def test_a_captured_step_follows_its_device_lengths():
    """rope, write and attention in one graph, replayed while the lengths and
    positions advance on the device, equal the eager calls bit for bit; a
    second graph with its own workspace runs on another stream at once."""
    heads, kv, hd, n_seq = 8, 2, 128, 3
    sets = []
    for k in range(2):
        st, rng = _setup(heads, kv, hd, n_seq, 20, n_seq, seed=20 + k)
        st.update(lens=i32([1200 - 100 * k, 3, 64]), x=torch.empty(n_seq, (heads + 2 * kv) * hd, device=DEV),
                  start=i32(range(n_seq + 1)), seed=k, eager=st["cache"].clone(),
                  work=torch.empty(rf.kv4_attention_workspace(hd, 20), dtype=torch.uint8, device=DEV))
        st["cache"].random_(0, 60), st["eager"].copy_(st["cache"])  # finite parameters
        sets.append(st)
    rf.kernel_errors()

    def body(st):
        st["lens"] += 1
        return _step(st, st["x"], st["lens"] - 1, st["start"], st["lens"], st["work"])

    graphs, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for st in sets:
        lens = st["lens"].clone()
        st["x"].normal_()
        body(st)  # warm
        st["lens"].copy_(lens)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            body(st)
        st["lens"].copy_(lens)
        st["cache"].copy_(st["eager"])
        graphs.append(g)
    torch.cuda.synchronize()
    inputs = [[torch.randn_like(st["x"]) for _ in range(6)] for st in sets]
    got = [[], []]
    for i in range(6):
        for k, st in enumerate(sets):
            with torch.cuda.stream(streams[k]):
                st["x"].copy_(inputs[k][i])
                graphs[k].replay()
                got[k].append(st["out"].clone())
    torch.cuda.synchronize()
    for k, st in enumerate(sets):
        st["cache"] = st["eager"]
        st["lens"] -= 6
        for i in range(6):
            st["x"].copy_(inputs[k][i])
            assert torch.equal(body(st), got[k][i]), (k, i)
    rf.kernel_errors()


def test_c_calls_on_the_legacy_stream():
    """The C entry points with stream NULL, as a host without torch makes them."""
    L = rf.lib()
    heads, kv, hd, n = 4, 2, 64, 80
    c = Cache([n], kv, hd, seed=30, fill=False)
    cache, table = c.on_device()
    x = dev(c.values(n)).float()
    start, lens = i32([0, n]), i32([n])
    torch.cuda.synchronize()
    v = rf.api.Kv4(cache.data_ptr(), table.data_ptr(), start.data_ptr(), lens.data_ptr(), len(c.data), kv, hd, 1,
                   c.table.shape[1], n)
    assert L.foxcuda_kv4_write(C.byref(v), 0, x.data_ptr(), kv * hd, x.data_ptr(), kv * hd, None) == 0
    out = torch.empty(n, kv, hd, device=DEV)
    out2 = torch.empty_like(out)
    assert L.foxcuda_kv4_read(C.byref(v), 0, out.data_ptr(), out2.data_ptr(), None) == 0
    assert L.foxcuda_kernel_errors(None) == 0
    want = R.values(*R.quantise(host(x))).astype(np.float32)
    assert np.array_equal(host(out), want) and np.array_equal(host(out2), want)
