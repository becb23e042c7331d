"""Query heads per KV head that do not divide the attention kernels' tiles of 4
and 128 (row, head) pairs, as many as the engine's own attention takes: a row's
heads stand in two tiles, tiles hold parts of rows. Tolerances are
test_kv4_gpu.py's."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

import kv4_ref as R  # noqa: E402
import rustfox_b200 as rf  # noqa: E402
from test_kv4_gpu import TYPES, Cache, _attend, _close, dev, host, starts  # noqa: E402


def _check(c, heads, rows, lens, dtype):
    n = sum(rows) + 2
    q = dev(c.rng.normal(0, 1, (n, heads, c.hd)), TYPES[dtype])
    out0 = np.full((n, heads, c.hd), -2.0)
    got = _attend(c, q, rows, lens, out0)
    want = R.attend(host(q.double()), c.data, c.table, starts(rows), lens, out0)
    _close(got, want, dtype)
    assert (got[-2:] == -2).all()
    rf.kernel_errors()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("group", [3, 5, 6, 7])
def test_single_tokens_and_short_chunks(group, hd, dtype):
    lens, rows = [1, 64, 65, 0, 129, 300, 1000, 5, 40], [1, 1, 2, 1, 3, 1, 1, 9, 7]
    _check(Cache(lens, 2, hd, seed=group + hd), 2 * group, rows, lens, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("group", [3, 5, 6, 7])
def test_many_rows(group, hd, dtype):
    lens, rows = [64, 200, 5, 700, 0, 1, 1900], [64, 43, 9, 128, 30, 1, 37]
    c = Cache(lens, 2, hd, seed=group + hd)
    assert c.table.shape[1] > 16 and sum(rows) * group >= 48 * len(rows)
    _check(c, 2 * group, rows, lens, dtype)


@pytest.mark.parametrize("group", [3, 7])
def test_long_sequences_are_split_and_joined(group):
    lens, rows = [9001, 130], [2, 3]
    _check(Cache(lens, 1, 128, seed=group), group, rows, lens, "f32")
    lens, rows = [9001, 130], [45, 60]
    _check(Cache(lens, 1, 128, seed=group + 1), group, rows, lens, "f32")
