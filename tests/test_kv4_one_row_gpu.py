"""A single row has no stride: a slice of a tensor with any row stride is taken."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

import kv4_ref as R  # noqa: E402
import rustfox_b200 as rf  # noqa: E402
from test_kv4_gpu import DEV, Cache, dev, host, i32  # noqa: E402


def _row(values, stride):
    """values [n] as the first columns of the first of three rows of `stride`."""
    t = torch.zeros(3, stride, device=DEV)
    t[0, :len(values)] = dev(values).float()
    return t[:1, :len(values)]


@pytest.mark.parametrize("more", [1, 3, 64])
def test_one_row_of_wider_rows(more):
    heads, kv, hd, L = 4, 2, 64, 100
    c = Cache([L], kv, hd, seed=5)
    rng = np.random.default_rng(more)
    q, k = (rng.normal(0, 1, h * hd).astype(np.float32) for h in (heads, kv))
    cache, table = c.on_device()
    rows, lens = i32([0, 1]), i32([L])
    want = rf.kv4_attention(dev(q).view(1, heads, hd), cache, table, rows, lens)
    got = rf.kv4_attention(_row(q, heads * hd + more), cache, table, rows, lens, out=_row(q, heads * hd + more))
    assert torch.equal(got.view(1, heads, hd), want)
    rf.kv4_write(cache, table, rows, lens, _row(k, kv * hd + more), _row(-k, kv * hd + more))
    k2, v2 = rf.kv4_read(cache, table, rows, lens, k_out=_row(k, kv * hd + more), v_out=_row(k, kv * hd + more))
    for got, x in ((k2, k), (v2, -k)):
        x = R.values(*R.quantise(x.reshape(kv, hd))).astype(np.float32)
        assert np.array_equal(host(got).reshape(kv, hd), x)
    x = np.concatenate([q, k])
    cos, sin, pos = torch.ones(2, hd // 2, device=DEV), torch.zeros(2, hd // 2, device=DEV), i32([1])
    q3, k3 = rf.qk_norm_rope(_row(x, len(x) + more), heads, kv, hd, pos, cos, sin, q_out=_row(q, heads * hd + more),
                             k_out=_row(k, kv * hd + more))
    assert np.array_equal(host(q3)[0], q) and np.array_equal(host(k3)[0], k)
    y = _row(x, len(x) + more)  # in place
    rf.qk_norm_rope(y, heads, kv, hd, pos, cos, sin, q_out=y[:, :heads * hd], k_out=y[:, heads * hd:])
    assert np.array_equal(host(y)[0], x)
    rf.kernel_errors()
