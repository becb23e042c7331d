"""Index arrays at addresses that no int32 has are refused, before any device
call reads them (host addresses stand in for the device's; nothing is read)."""
import ctypes as C

import pytest


@pytest.fixture()
def buf():
    b = C.create_string_buffer(1 << 16)
    yield (C.addressof(b) + 15) // 16 * 16
    del b


@pytest.mark.parametrize("by", [1, 2, 3])
@pytest.mark.parametrize("name", ["table", "row_start", "kv_len"])
def test_the_caches_arrays(buf, name, by):
    import rustfox_b200 as rf
    L = rf.lib()
    at = dict(cache=buf, table=buf + 32768, row_start=buf + 33000, kv_len=buf + 33400)
    at[name] += by
    c = C.byref(rf.api.Kv4(*at.values(), 1, 1, 64, 1, 2, 1))
    k, v = buf + 40000, buf + 44096
    for st in (L.foxcuda_kv4_write(c, 0, k, 64, v, 64, None), L.foxcuda_kv4_read(c, 0, k, v, None),
               L.foxcuda_kv4_attention(c, 0, k, 64, 1, 0.0, None, 0, v, None)):
        assert st == 1 and "4-byte aligned" in rf.last_error()


@pytest.mark.parametrize("by", [1, 2, 3])
def test_the_rotations_positions(buf, by):
    import rustfox_b200 as rf
    st = rf.lib().foxcuda_qk_norm_rope(0, buf, 128, 2, 1, 1, 64, None, None, 1e-5, buf + 8192, buf + 16384, 4, 0,
                                       buf + 20480 + by, buf + 24576, 64, buf + 28672, 64, None)
    assert st == 1 and "4-byte aligned" in rf.last_error()
