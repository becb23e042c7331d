"""row_start that names more rows than the row arrays hold: every call places
the rows that are there alike, and reports the others."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

import rustfox_b200 as rf  # noqa: E402
from test_kv4_gpu import DEV, Cache, dev, host, i32  # noqa: E402
from test_kv4_places_gpu import _attend, _write_and_read  # noqa: E402

CASES = [([0, 10], 8, [10]), ([0, 10, 30], 22, [64, 100]), ([0, 22, 40, 45], 22, [30, 64, 64]),
         ([0, 40, 40, 140], 100, [128, 3, 110]), ([3, 9, 1 << 30], 50, [128, 1 << 30])]


@pytest.mark.parametrize("start,n,lens", CASES)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_write_and_read(hd, start, n, lens):
    c = Cache([128] * len(lens), 2, hd, seed=n + hd, fill=False)
    _write_and_read(c, start, lens, n)


@pytest.mark.parametrize("start,n,lens", CASES[:-1])
@pytest.mark.parametrize("heads,kv,hd", [(2, 2, 64), (8, 2, 128), (4, 2, 256)])
def test_attention(heads, kv, hd, start, n, lens):
    c = Cache([128] * len(lens), kv, hd, seed=n + hd)
    _attend(c, heads, start, lens, n)


def test_attention_of_many_rows():
    c = Cache([300, 500], 2, 128, seed=3, stride=17)
    _attend(c, 4, [0, 60, 140], [300, 500], 100)


@pytest.mark.parametrize("start", [[0, 60, 0, 60], [0, 40, 39], [100, 99], [0] * 40 + [50, 0, 50], [2, -5, 3]])
@pytest.mark.parametrize("heads,stride", [(2, 3), (4, 17)])
def test_a_falling_row_start_is_refused_by_attention(heads, stride, start):
    """Rows that two sequences would have: none is touched, and the calls after
    are as ever. (Rows counted twice are also how the units of a call could pass
    the bound that the host checks.)"""
    n_seq, n = len(start) - 1, 110
    c = Cache([150] * n_seq, 2, 128, seed=stride, stride=stride)
    q = dev(c.rng.normal(0, 1, (n, heads, 128))).float()
    cache, table = c.on_device()
    out = torch.full((n, heads, 128), -2.0, device=DEV)
    rf.kernel_errors()
    rf.kv4_attention(q, cache, table, i32(start), i32(c.lens), out=out)
    with pytest.raises(rf.FoxError, match="outside"):
        rf.kernel_errors()
    assert (host(out) == -2.0).all()
    rf.kv4_attention(q, cache, table, i32([0, 5] + [5] * (n_seq - 1)), i32(c.lens), out=out)
    rf.kernel_errors()
    assert np.isfinite(host(out)).all() and (host(out[5:]) == -2.0).all() and (host(out[:5]) != -2.0).any()
