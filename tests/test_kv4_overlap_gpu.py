"""Rows that stand between one another's without overlapping are taken: the
rotation in place, over columns that are not read, into columns of one buffer;
keys and values of one tensor. Results are those of rows by themselves."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

import rustfox_b200 as rf  # noqa: E402
from test_kv4_gpu import DEV, TYPES, Cache, dev, i32  # noqa: E402

HEADS, KV = 4, 2


def _cols(t, at, heads, hd):
    return t[:, at:at + heads * hd].unflatten(1, (heads, hd))


@pytest.mark.parametrize("rows", [1, 50])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_rotation(hd, dtype, rows):
    rng = np.random.default_rng(hd + rows)
    nq, nk = HEADS * hd, KV * hd
    x = dev(rng.normal(0, 1, (rows, nq + 2 * nk)), TYPES[dtype])
    th = rng.normal(0, 1, (8, hd // 2))
    cos, sin, pos = dev(np.cos(th)).float(), dev(np.sin(th)).float(), i32(rng.integers(0, 8, rows))
    w = dev(rng.normal(1, 0.1, hd)).float()

    def call(t, **kw):
        return rf.qk_norm_rope(t, HEADS, KV, hd, pos, cos, sin, q_norm=w, k_norm=w, halves=True, **kw)

    q, k = call(x)
    both, flipped = (torch.zeros(rows, nq + 2 * nk, dtype=x.dtype, device=DEV) for _ in "ab")
    inplace, over, only_q, only_k = (x.clone() for _ in range(4))
    cases = [
        (x, _cols(both, 0, HEADS, hd), _cols(both, nq, KV, hd)),
        (x, _cols(flipped, nk, HEADS, hd), _cols(flipped, 0, KV, hd)),
        (inplace, _cols(inplace, 0, HEADS, hd), _cols(inplace, nq, KV, hd)),
        (over, _cols(over, 0, HEADS, hd), _cols(over, nq + nk, KV, hd)),  # where the values stood
        (only_q, _cols(only_q, 0, HEADS, hd), None),
        (only_k, None, _cols(only_k, nq, KV, hd)),
    ]
    for i, (src, qo, ko) in enumerate(cases):
        got = call(src, q_out=qo, k_out=ko)
        assert torch.equal(got[0], q) and torch.equal(got[1], k), i
    assert torch.equal(over[:, nq:nq + nk], x[:, nq:nq + nk])
    if rows > 1:
        shifted = torch.zeros(rows * (nq + 2 * nk) + 64, dtype=x.dtype, device=DEV)
        flat = shifted[:x.numel()].view_as(x)
        with pytest.raises(rf.FoxError, match="overlap"):
            call(flat, q_out=shifted[16:16 + rows * nq].view(rows, HEADS, hd))
    rf.kernel_errors()


def test_keys_and_values_of_one_tensor():
    n, hd = 70, 128
    c = Cache([n], KV, hd, seed=2, fill=False)
    x = dev(c.values(n)).float()
    cache, table = c.on_device()
    rf.kv4_write(cache, table, i32([0, n]), i32([n]), x, x)
    k, v = rf.kv4_read(cache, table, i32([0, n]), i32([n]), n)
    assert torch.equal(k, v)
    two = torch.full((2, n, KV, hd), 7.5, device=DEV)
    rf.kv4_read(cache, table, i32([0, n]), i32([n]), k_out=two[0], v_out=two[1])
    assert torch.equal(two[0], k) and torch.equal(two[1], v)
    rf.kernel_errors()
