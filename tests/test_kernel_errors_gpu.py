"""The device error word keeps a wait that gave up when a later call names a
position outside its arrays. The word is set from the host, as a kernel that gave
up leaves it; nothing waits here."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

import rustfox_b200 as rf  # noqa: E402
from test_kv4_gpu import Cache, dev, i32  # noqa: E402


def _set_word(code):
    rf.kernel_errors()  # (the word is found on its first use)
    where = rf.lib()._ZN3fox14kernel_err_ptrEv
    where.restype, where.argtypes = C.c_void_p, []
    at = where()
    assert at
    torch.cuda.synchronize()
    assert C.CDLL("libcuda.so.1").cuMemsetD32_v2(C.c_uint64(at), C.c_uint(code), C.c_size_t(1)) == 0
    torch.cuda.synchronize()


def _outside(op):
    """A call with a page, or a position, that is not there."""
    c = Cache([100], 2, 64, seed=1)
    x, q = dev(c.values(1)).float(), dev(c.rng.normal(0, 1, (60, 4, 64))).float()
    cache, table = c.on_device()
    table[0, 1] = len(c.data)
    if op == "write":
        rf.kv4_write(cache, table, i32([0, 1]), i32([100]), x, x)
    elif op == "read":
        rf.kv4_read(cache, table, i32([0, 1]), i32([129]), 1)
    elif op == "rope":
        cos = torch.ones(4, 32, device=x.device)
        rf.qk_norm_rope(torch.zeros(1, 6 * 64, device=x.device), 4, 2, 64, i32([4]), cos, cos)
    elif op == "few":
        rf.kv4_attention(q[:1], cache, table, i32([0, 1]), i32([100]))
    else:
        wide = torch.cat([table, torch.full((1, 20), -1, dtype=torch.int32, device=x.device)], 1)
        rf.kv4_attention(q, cache, wide, i32([0, 60]), i32([100]))


@pytest.mark.parametrize("op", ["write", "read", "rope", "few", "many"])
@pytest.mark.parametrize("code", [1, 2])
def test_a_wait_that_gave_up_is_not_hidden(op, code):
    _set_word(code)
    _outside(op)
    with pytest.raises(rf.FoxError, match=rf"gave up \(code {code}\).*not valid.*skipped"):
        rf.kernel_errors()
    rf.kernel_errors()  # read once
    _outside(op)
    with pytest.raises(rf.FoxError, match="outside") as e:
        rf.kernel_errors()
    assert "not valid" not in str(e.value)
    rf.kernel_errors()
