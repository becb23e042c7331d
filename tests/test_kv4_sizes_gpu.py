"""Queries and scales at the ends of what fp32 holds, for both attention kernels."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

import kv4_ref as R  # noqa: E402
import rustfox_b200 as rf  # noqa: E402
from test_kv4_gpu import Cache, _attend, _close, dev, host  # noqa: E402

# heads, KV heads, head dimension, rows, pages of the table: few rows, then many
CASES = [(2, 2, 64, 4, 3), (8, 2, 128, 3, 3), (4, 2, 256, 5, 3), (2, 2, 64, 60, 17), (4, 2, 128, 40, 17)]


@pytest.mark.parametrize("scale", [1e-5, 1e-10, 1e-20, 1e-38, 1e-45])
@pytest.mark.parametrize("size", [0.0, 1e-30, 1.0])
@pytest.mark.parametrize("v", [1.0, 1e-3])
@pytest.mark.parametrize("case", CASES)
def test_scores_of_nothing_weigh_every_seen_position_alike(case, v, size, scale):
    """Scores of zero, or too small for fp32: the mean of what each row sees, and
    nothing of what it does not."""
    heads, kv, hd, rows, stride = case
    L = 150
    c = Cache([L], kv, hd, seed=3, fill=False, stride=stride)
    # (keys that are all small have another scale)
    R.put(c.data, c.table, 0, np.arange(L), v * np.clip(c.values(L), -3, 3), c.values(L))
    q = dev(size * c.rng.normal(0, 1, (rows, heads, hd))).float()
    got = _attend(c, q, [rows], [L], scale=scale)
    want = R.attend(host(q.double()), c.data, c.table, [0, rows], [L], np.zeros((rows, heads, hd)), scale=scale)
    _close(got, want, "f32")
    rf.kernel_errors()


@pytest.mark.parametrize("size,scale", [(1e33, 0.0), (1e35, 0.0), (1e36, 0.0), (1e36, 1e-36), (3e37, 1e-37), (3e37, 1e-30)])
@pytest.mark.parametrize("case", CASES)
def test_queries_near_the_end_of_fp32(case, size, scale):
    """Finite queries give finite results: softmax's ordinary ones where the scale
    makes up for their size, and otherwise the value whose score is the largest
    (where no other comes within 2^-15 of the scores' size, the bound of
    test_kv4_gpu.py 16 times over)."""
    heads, kv, hd, rows, stride = case
    L = 150
    c = Cache([L], kv, hd, seed=4, stride=stride)
    q = dev(size * c.rng.uniform(-1, 1, (rows, heads, hd))).float()
    got = _attend(c, q, [rows], [L], scale=scale)
    assert np.isfinite(got).all()
    want = R.attend(host(q.double()), c.data, c.table, [0, rows], [L], np.zeros((rows, heads, hd)), scale=scale or None)
    if size * scale and size * scale <= 10:
        _close(got, want, "f32")
        return
    k = R.get(c.data, c.table, 0, np.arange(L))[0]
    x = host(q.double()).reshape(rows, kv, heads // kv, hd)
    z = np.einsum("rkgd,lkd->rkgl", x, k).reshape(rows, heads, L)
    z[np.broadcast_to((np.arange(L) > L - rows + np.arange(rows)[:, None])[:, None], z.shape)] = -np.inf
    top = np.sort(z, -1)[..., -2:]
    most = np.einsum("rkgd,lkd->rkgl", np.abs(x), np.abs(k)).reshape(rows, heads, L).max(-1)
    clear = top[..., 1] - top[..., 0] > 2.0 ** -15 * most
    assert clear.mean() > 0.9
    _close(got[clear], want[clear], "f32")
    rf.kernel_errors()
