"""What stands in positions that a row does not see does not reach it through
the positions that it shares a tile with: infinities, and values so large that
a scale common to the tile would take the small ones' bits. One and two query
heads a KV head put several rows into a tile of either attention kernel.
Tolerances are test_kv4_gpu.py's."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

import kv4_ref as R  # noqa: E402
import rustfox_b200 as rf  # noqa: E402
from test_kv4_gpu import Cache, _attend, _close, dev, host  # noqa: E402

# heads, KV heads, head dimension, rows, pages of the table: few rows, then many
FEW = [(2, 2, 64, 4, 3), (4, 2, 64, 2, 3), (2, 2, 128, 4, 3), (2, 1, 128, 9, 3), (2, 2, 256, 5, 3)]
MANY = [(2, 2, 64, 60, 17), (4, 2, 128, 40, 17)]


def _case(heads, kv, hd, rows, stride, size=1.0, seed=1):
    L = 150
    c = Cache([L], kv, hd, seed=seed, fill=False, stride=stride)
    R.put(c.data, c.table, 0, np.arange(L), c.values(L), size * c.values(L))
    q = dev(c.rng.normal(0, 1, (rows, heads, hd))).float()
    return c, q, L


@pytest.mark.parametrize("what", ["d", "m", "both"])
@pytest.mark.parametrize("case", FEW + MANY)
def test_an_infinity_reaches_who_sees_it(case, what):
    """In one group of V of the last position, which the last row sees, in the
    group's dimensions only."""
    heads, kv, hd, rows, stride = case
    c, q, L = _case(*case)
    want = R.attend(host(q.double()), c.data, c.table, [0, rows], [L], np.zeros((rows, heads, hd)))
    at, group = L - 1, hd // R.GROUP - 1
    n = 4 * (hd // R.GROUP)
    o = R.PAGE * hd // 2 + at % R.PAGE * n + 4 * group
    blk = c.data[c.table[0, at // R.PAGE], :, 1]
    if what != "m":
        blk[:, o:o + 2] = [0x00, 0x7C]
    if what != "d":
        blk[:, o + 2:o + 4] = [0x00, 0x7C]
    got = _attend(c, q, [rows], [L])
    _close(got[:-1], want[:-1], "f32")
    assert not np.isfinite(got[-1, :, 64 * group:]).any()
    if group:
        _close(np.ascontiguousarray(got[-1:, :, :64 * group]), np.ascontiguousarray(want[-1:, :, :64 * group]), "f32")
    rf.kernel_errors()


@pytest.mark.parametrize("size", [1.0, 1e-2])
@pytest.mark.parametrize("case", FEW + MANY)
def test_large_values_of_a_later_row_take_no_bits(case, size):
    """V of up to fp16's largest in the last position: steps of 8000 beside steps
    of 0.2, and of 0.002, which the rows before the last see."""
    heads, kv, hd, rows, stride = case
    c, q, L = _case(*case, size=size, seed=2)
    big = np.linspace(-6e4, 6e4, kv * hd).reshape(1, kv, hd)[..., np.random.default_rng(0).permutation(hd)]
    big[..., ::R.GROUP], big[..., 1::R.GROUP] = -6e4, 6e4
    R.put(c.data, c.table, 0, [L - 1], c.values(1), big)
    got = _attend(c, q, [rows], [L])
    want = R.attend(host(q.double()), c.data, c.table, [0, rows], [L], np.zeros((rows, heads, hd)))
    assert R.get(c.data, c.table, 0, [L - 1])[1].max() > 5.9e4
    _close(got[:-1], want[:-1], "f32")
    _close(got[-1:], want[-1:], "f32")
    rf.kernel_errors()


@pytest.mark.parametrize("case", FEW + MANY)
def test_steps_that_no_write_gives(case):
    """A cache filled by other means: finite steps of 60000 and offsets of fp16's
    largest in one group of the last position, values of up to 965504."""
    heads, kv, hd, rows, stride = case
    c, q, L = _case(*case, seed=3)
    n = 4 * (hd // R.GROUP)
    o = R.PAGE * hd // 2 + (L - 1) % R.PAGE * n
    for side in (0, 1):
        blk = c.data[c.table[0, (L - 1) // R.PAGE], :, side]
        blk[:, o:o + 4] = np.array([60000, 65504], np.float16).view(np.uint8)
    got = _attend(c, q, [rows], [L])
    want = R.attend(host(q.double()), c.data, c.table, [0, rows], [L], np.zeros((rows, heads, hd)))
    _close(got[:-1], want[:-1], "f32")
    # the last row's score there is beyond all others, above or below
    _close(got[-1:], want[-1:], "f32")
    rf.kernel_errors()
