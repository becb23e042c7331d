"""foxcuda_kv4_attention for many rows of a sequence, against the definition in
64 bits (tests/kv4_ref.py): the shapes here have 48 (row, head) pairs a sequence
and KV head or more, and tables of more than 16 pages or many rows, which is
where the kernel on the 5th-generation tensor cores takes over.

Tolerance, fp32 rows: q, the weights and a page's offsets are hi + lo fp16,
2^-22 each; d times a code is exact. The scores' sum truncates at most 9 times
at its full size and 16 times at 2^-11 of it, 2^-23 each: 1.1e-6 of a score,
2e-6 of a weight's exponent for scores of about 2 (what normal q and k give).
A page truncates O 12 times, and it is read out every 4 pages: 48 x 2^-24 on
average, 3e-6. Together 6e-6; the bound is 1e-5 of the result's norm, three
times that for one row. fp16 rows add half a step, 2^-11."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

import kv4_ref as R  # noqa: E402
import rustfox_b200 as rf  # noqa: E402
from test_kv4_gpu import TYPES, Cache, _attend, _close, dev, host, i32, starts  # noqa: E402

WIDE = 17  # a table of this many pages may split its runs


def _check(c, q, rows, lens, dtype="f32", fill=-2.0, **kw):
    out0 = np.full((q.shape[0], q.shape[1], q.shape[2]), fill)
    got = _attend(c, q, rows, lens, out0, **kw)
    want = R.attend(host(q.double()), c.data, c.table, starts(rows), lens, out0, **kw)
    _close(got, want, dtype, (rows, lens))
    rf.kernel_errors()
    return got


def _q(c, n, heads, hd, dtype="f32"):
    return dev(c.rng.normal(0, 1, (n, heads, hd)), TYPES[dtype])


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 64), (2, 2, 64), (4, 2, 128), (8, 1, 128), (4, 4, 128)])
def test_rows_of_ragged_sequences(heads, kv, hd, dtype):
    """Tiles that end inside a row and inside the 128 pairs, more rows than
    positions, no rows, no positions, one position, pages' edges."""
    lens = [64, 200, 5, 33, 700, 0, 1, 65, 128]
    rows = [64, 150, 9, 0, 131, 60, 1, 65, 77]
    c = Cache(lens, kv, hd, seed=heads + hd, stride=WIDE)
    got = _check(c, _q(c, sum(rows) + 3, heads, hd, dtype), rows, lens, dtype)
    a = starts(rows)
    assert (got[a[2]:a[2] + 4] == 0).all() and (got[a[5]:a[6]] == 0).all()
    assert (got[-3:] == -2).all()


@pytest.mark.parametrize("n", [47, 48, 127, 128, 129, 257])
def test_rows_about_the_tiles_edges(n):
    for hd in (64, 128):
        c = Cache([300], 1, hd, seed=n, stride=WIDE)
        _check(c, _q(c, n, 1, hd), [n], [300])


@pytest.mark.parametrize("heads,kv,hd,length,rows", [(8, 2, 64, 20001, 50), (16, 2, 128, 6001, 70), (32, 8, 128, 12000, 48),
                                                     (16, 2, 128, 3001, 4)])
def test_long_sequences_are_split_and_joined(heads, kv, hd, length, rows):
    c = Cache([length, 130], kv, hd, seed=length)
    _check(c, _q(c, rows + 9, heads, hd), [rows, 9], [length, 130])


def test_short_tables_with_rows_for_every_sm():
    lens, rows = [1000, 3, 64, 640], [70, 3, 40, 50]
    c = Cache(lens, 8, 128, seed=3)
    assert c.table.shape[1] == 16
    _check(c, _q(c, sum(rows), 32, 128), rows, lens)


@pytest.mark.parametrize("scale", [0.0, 0.02, 3.0])
@pytest.mark.parametrize("size", [1e-20, 1e-3, 1.0, 300.0, 1e15])
def test_scales_and_sizes_of_queries(scale, size):
    """As for single tokens: the bound follows the largest score."""
    heads, kv, hd, L, T = 4, 1, 128, 333, 20
    c = Cache([L], kv, hd, seed=4, stride=WIDE)
    q = dev(size * c.rng.normal(0, 1, (T, heads, hd))).float()
    got = _attend(c, q, [T], [L], scale=scale)
    assert np.isfinite(got).all()
    want = R.attend(host(q.double()), c.data, c.table, [0, T], [L], np.zeros((T, heads, hd)), scale=scale or None)
    k = R.get(c.data, c.table, 0, np.arange(L))[0]
    z = np.abs(np.einsum("td,ld->tl", np.abs(host(q.double())).max(1), np.abs(k[:, 0]))).max()
    tol = 1e-5 + 2.0 ** -19 * z * (scale or hd ** -0.5)
    if tol < 0.1:
        assert np.linalg.norm(got - want) <= tol * np.linalg.norm(want)


@pytest.mark.parametrize("side", ["k", "v"])
@pytest.mark.parametrize("size", [1e-7, 1e-3, 1.0, 1e3, 4e4])
def test_sizes_of_what_is_cached(side, size):
    """From fp16's smallest to its largest, pages of very different size side
    by side: the operands' scale changes along the walk."""
    heads, kv, hd, L, T = 12, 3, 64, 700, 30
    c = Cache([L], kv, hd, seed=5, fill=False, stride=WIDE)
    x = {"k": c.values(L), "v": c.values(L)}
    x[side] = size * np.clip(x[side], -1.5, 1.5)
    x[side][::7] *= 1e-3
    x[side][128:256] *= 1e-2
    R.put(c.data, c.table, 0, np.arange(L), x["k"], x["v"])
    q = c.rng.normal(0, 1, (T, heads, hd)) / (max(size, 1.0) if side == "k" else 1.0)
    _check(c, dev(q).float(), [T], [L])


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("side", [0, 1])
def test_hidden_positions_may_hold_anything(side, hd):
    """A NaN group reaches the rows that see its position, in V its own 64
    dimensions only; the noise behind the end reaches nobody."""
    heads, kv, L, T = 8, 2, 150, 30
    c = Cache([L], kv, hd, seed=6, stride=WIDE)
    q = _q(c, T, heads, hd)
    want = R.attend(host(q.double()), c.data, c.table, [0, T], [L], np.zeros((T, heads, hd)))
    at, group = L - 26, hd // R.GROUP - 1  # in the second of three pages, seen by the last 26 rows
    n = 4 * (hd // R.GROUP)
    o = R.PAGE * hd // 2 + (at % R.PAGE) * n + 4 * group
    c.data[c.table[0, at // R.PAGE], :, side, o:o + 4] = 0xFF
    got = _attend(c, q, [T], [L])
    _close(got[:T - 26], want[:T - 26], "f32")
    seen = got[T - 26:]
    if side == 0:
        assert np.isnan(seen).all()
    else:
        assert np.isnan(seen[..., 64 * group:64 * group + 64]).all()
        if group:
            _close(np.ascontiguousarray(seen[..., :64]), np.ascontiguousarray(want[T - 26:, :, :64]), "f32")


def test_queries_that_are_not_finite_stay_in_their_row_and_head():
    heads, kv, hd, L, T = 8, 2, 128, 400, 40
    c = Cache([L], kv, hd, seed=7, stride=WIDE)
    q = _q(c, T, heads, hd)
    want = R.attend(host(q.double()), c.data, c.table, [0, T], [L], np.zeros((T, heads, hd)))
    q[3, 0, 3], q[17, 5, 100], q[39, 7, 0] = float("nan"), float("inf"), float("-inf")
    got = _attend(c, q, [T], [L])
    bad = np.zeros((T, heads), bool)
    bad[3, 0] = bad[17, 5] = bad[39, 7] = True
    assert np.isnan(got[bad]).all()
    _close(got[~bad], want[~bad], "f32")


def test_pages_outside_the_cache():
    heads, kv, hd = 8, 2, 128
    lens, rows = [200, 100, 1200], [20, 15, 30]
    c = Cache(lens, kv, hd, seed=11)
    bad = c.table.copy()
    bad[0, 1], bad[1, 0], bad[2, 5:9] = len(c.data), -1, 1 << 30
    q = _q(c, sum(rows), heads, hd)
    got = host(rf.kv4_attention(q, dev(c.data), dev(bad), i32(starts(rows)), i32(lens)).double())
    with pytest.raises(rf.FoxError, match="outside"):
        rf.kernel_errors()
    gone = {0: (1,), 1: (0,), 2: (5, 6, 7, 8)}
    want = R.attend(host(q.double()), c.data, c.table, starts(rows), lens, np.zeros((sum(rows), heads, hd)),
                    seen=lambda s, p: ~np.isin(p // R.PAGE, gone[s]))
    _close(got, want, "f32")


def test_rows_with_strides_and_strided_tables():
    """Rows of a wider projection; a table whose rows are longer than used."""
    heads, kv, hd, lens, rows = 8, 2, 128, [90, 500], [30, 33]
    c = Cache(lens, kv, hd, seed=12, stride=40)
    wide = _q(c, 63, heads + 2 * kv, hd)
    q = wide[:, :heads]
    got = _attend(c, q, rows, lens)
    want = R.attend(host(q.double()), c.data, c.table, starts(rows), lens, np.zeros((63, heads, hd)))
    _close(got, want, "f32")


def test_the_same_call_gives_the_same_bits_many_times():
    """Hundreds of launches back to back, each stretch of pages some twenty
    long: the roles of a block run ahead of one another by all they may."""
    heads, kv, hd, L, T = 32, 8, 128, 12000, 64
    c = Cache([L], kv, hd, seed=13)
    q = _q(c, T, heads, hd)
    cache, table = c.on_device()
    first = rf.kv4_attention(q, cache, table, i32([0, T]), i32([L]))
    assert torch.isfinite(first).all()
    rs, kl = i32([0, T]), i32([L])
    for _ in range(20):
        outs = [rf.kv4_attention(q, cache, table, rs, kl) for _ in range(20)]
        assert all(torch.equal(o, first) for o in outs)
    rf.kernel_errors()


def test_a_captured_call_follows_its_device_lengths():
    heads, kv, hd, T = 16, 4, 64, 32
    c = Cache([2000, 900], kv, hd, seed=14)
    q = _q(c, 2 * T, heads, hd)
    cache, table = c.on_device()
    rs, kl = i32([0, T, 2 * T]), i32([2000, 900])
    out = torch.empty(2 * T, heads, hd, device=q.device)
    rf.kv4_attention(q, cache, table, rs, kl, out=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        rf.kv4_attention(q, cache, table, rs, kl, out=out)
    for rows, lens in (([T, T], [2000, 900]), ([60, 4], [64, 1]), ([0, 64], [5, 831]), ([10, 20], [0, 33])):
        rs.copy_(i32(starts(rows)))
        kl.copy_(i32(lens))
        out.fill_(-2.0)
        g.replay()
        want = R.attend(host(q.double()), c.data, c.table, starts(rows), lens, np.full((2 * T, heads, hd), -2.0))
        _close(host(out.double()), want, "f32", (rows, lens))


@pytest.mark.parametrize("T", [1, 5])
def test_single_tokens_and_a_group_of_v_that_is_not_a_number(T):
    """The other kernel (few rows): NaN in one group of V stays in its 64
    dimensions there too."""
    heads, kv, hd, L = 8, 2, 128, 150
    c = Cache([L], kv, hd, seed=16)
    q = _q(c, T, heads, hd)
    want = R.attend(host(q.double()), c.data, c.table, [0, T], [L], np.zeros((T, heads, hd)))
    o = R.PAGE * hd // 2 + 70 % R.PAGE * 8 + 4
    c.data[c.table[0, 1], :, 1, o:o + 4] = 0xFF
    got = _attend(c, q, [T], [L])
    assert np.isnan(got[..., 64:]).all()
    _close(np.ascontiguousarray(got[..., :64]), np.ascontiguousarray(want[..., :64]), "f32")


def test_calls_on_two_streams_with_their_own_workspaces():
    heads, kv, hd, T = 16, 4, 128, 16
    c = Cache([5000, 3500], kv, hd, seed=17)
    cache, table = c.on_device()
    q = _q(c, 2 * T, heads, hd)
    rs, kl = i32([0, T, 2 * T]), i32([5000, 3500])
    want = rf.kv4_attention(q, cache, table, rs, kl)
    one = rf.kv4_attention(q[:1], cache, table[:1].contiguous(), i32([0, 1]), i32([5000]))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(40):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(rf.kv4_attention(q, cache, table, rs, kl) if i % 4 < 2 else
                        rf.kv4_attention(q[:1], cache, table[:1].contiguous(), i32([0, 1]), i32([5000])))
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        assert torch.equal(o, want if i % 4 < 2 else one), i
    rf.kernel_errors()


def test_as_many_sequences_as_a_call_takes():
    """1024 ragged sequences of 12 rows of 4 heads that share a prefix's pages,
    some of them empty; then all of them."""
    heads, kv, hd, n, T = 4, 1, 128, 1024, 12
    c = Cache([256], kv, hd, seed=18)
    table = np.full((n, WIDE), -1, np.int32)
    table[:, :4] = c.table
    lens = c.rng.integers(0, 257, n)
    rs = np.arange(n + 1) * T
    q = _q(c, n * T, heads, hd)
    args = dev(c.data), dev(table), i32(rs)
    got = host(rf.kv4_attention(q, *args, i32(lens)).double())
    for s in range(0, n, 37):
        a, b = rs[s], rs[s + 1]
        want = R.attend(host(q[a:b].double()), c.data, table[s:s + 1], [0, T], lens[s:s + 1], np.zeros((T, heads, hd)))
        if lens[s]:
            _close(got[a:b], want, "f32", (s, lens[s]))
        else:
            assert (got[a:b] == 0).all()
    out = torch.full_like(q, 3.0)
    rf.kv4_attention(q, *args, i32([0] * n), out=out)
    assert (out == 0).all()
    rf.kernel_errors()
