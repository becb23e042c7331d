"""Where the rows of a 4-bit cache's calls stand when the device arrays name more
than there is: lengths beyond the block table, rows beyond the row arrays. Row r
of sequence s stands at kv_len[s] - (row_start[s + 1] - r), whatever is there:
a row outside its table is skipped and reported, and moves no other row.
Tolerances are test_kv4_gpu.py's."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

import kv4_ref as R  # noqa: E402
import rustfox_b200 as rf  # noqa: E402
from test_kv4_gpu import DEV, TYPES, Cache, _close, dev, host, i32, starts  # noqa: E402


def places(start, lens, n, cap):
    """(row, sequence, position) of the rows that have a place in their table."""
    return [(r, s, lens[s] - (start[s + 1] - r)) for s in range(len(lens)) for r in range(start[s], min(start[s + 1], n))
            if 0 <= lens[s] - (start[s + 1] - r) < cap]


def _write_and_read(c, start, lens, n, dtype="f32"):
    """Every byte of the cache after a write, and every value read back."""
    rf.kernel_errors()
    kv, hd = c.kv, c.hd
    k, v = (dev(c.values(n), TYPES[dtype]) for _ in "kv")
    cache, table = c.on_device()
    rf.kv4_write(cache, table, i32(start), i32(lens), k, v)
    with pytest.raises(rf.FoxError, match="outside"):
        rf.kernel_errors()
    there = places(start, lens, n, c.table.shape[1] * R.PAGE)
    for r, s, p in there:
        R.put(c.data, c.table, s, [p], host(k[r:r + 1].double()), host(v[r:r + 1].double()))
    assert np.array_equal(host(cache), c.data)
    k2, v2 = (torch.full((n, kv, hd), 7.5, dtype=TYPES[dtype], device=DEV) for _ in "kv")
    rf.kv4_read(cache, table, i32(start), i32(lens), k_out=k2, v_out=v2)
    with pytest.raises(rf.FoxError, match="outside"):
        rf.kernel_errors()
    want = [np.full((n, kv, hd), 7.5) for _ in "kv"]
    for r, s, p in there:
        for side, x in enumerate(R.get(c.data, c.table, s, [p])):
            want[side][r] = x[0]
    for got, w in zip((k2, v2), want):
        assert torch.equal(got.cpu(), torch.from_numpy(w).float().to(TYPES[dtype]))


def _attend(c, heads, start, lens, n, want_lens=None):
    """Every row's output; rows behind the arrays' end are the reference's only."""
    rf.kernel_errors()
    cap = c.table.shape[1] * R.PAGE
    q = c.rng.normal(0, 1, (max(n, start[-1]), heads, c.hd)).astype(np.float32)
    cache, table = c.on_device()
    out = torch.full((n, heads, c.hd), -2.0, device=DEV)
    rf.kv4_attention(dev(q[:n]), cache, table, i32(start), i32(lens), out=out)
    with pytest.raises(rf.FoxError, match="outside"):
        rf.kernel_errors()
    want = R.attend(q, c.data, c.table, start, want_lens or lens, np.full(q.shape, -2.0), seen=lambda s, p: p < cap)
    _close(host(out.double()), want[:n], "f32")


@pytest.mark.parametrize("over", [1, 3, 70])
@pytest.mark.parametrize("rows", [1, 4, 80])
@pytest.mark.parametrize("hd,kv", [(64, 3), (128, 2), (256, 1)])
def test_write_and_read_of_a_sequence_that_outgrew_its_table(hd, kv, rows, over):
    c = Cache([128, 128], kv, hd, seed=hd + rows + over, fill=False)
    for dtype in ("f32", "f16"):
        _write_and_read(c, starts([rows, 5]).tolist(), [128 + over, 100], rows + 7, dtype)


@pytest.mark.parametrize("over", [1, 3, 70])
@pytest.mark.parametrize("rows", [1, 4, 9, 80])
@pytest.mark.parametrize("heads,kv,hd", [(2, 2, 64), (8, 2, 128), (4, 2, 256)])
def test_attention_of_a_sequence_that_outgrew_its_table(heads, kv, hd, rows, over):
    """Rows inside the table see up to their own position, those outside all of
    the table's."""
    c = Cache([128, 128], kv, hd, seed=hd + rows + over)
    _attend(c, heads, starts([rows, 5]).tolist(), [128 + over, 100], rows + 7)


@pytest.mark.parametrize("over", [1, 30, 200])
def test_attention_of_many_rows_that_outgrew_their_table(over):
    c = Cache([1088, 900], 2, 128, seed=over)
    assert c.table.shape[1] == 17
    _attend(c, 4, starts([90, 20]).tolist(), [1088 + over, 900], 112)


def test_the_largest_lengths():
    c = Cache([128, 128], 2, 64, seed=1)
    _write_and_read(c, [0, 4, 9], [2 ** 31 - 1, 100], 9)
    c = Cache([128, 128], 2, 64, seed=2)
    _attend(c, 4, [0, 4, 9], [2 ** 31 - 1, 100], 9, want_lens=[200, 100])
