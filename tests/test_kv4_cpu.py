"""The 4-bit K/V cache without a GPU: the definition's own properties, and
the refusals of its entry points (which come before any device call; host
buffers stand in for device pointers)."""
import ctypes as C

import numpy as np
import pytest

import kv4_ref as R


def _values(rng, n, hd):
    x = rng.normal(0, 1, (n, hd)) * np.exp(rng.normal(0, 2, (n, 1))) + rng.normal(0, 3, (n, 1))
    return x.astype(np.float32)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_every_value_reads_back_within_half_a_step(hd):
    x = _values(np.random.default_rng(1), 200, hd)
    code, d, m = R.quantise(x)
    got = R.values(code, d, m)
    step = np.repeat(d, R.GROUP, -1)
    assert (np.abs(got - x) <= step / 2 * (1 + 1e-12)).all()
    top = (m + 15 * d)[..., None]
    g = x.reshape(200, -1, R.GROUP)
    assert (g >= m[..., None]).all() and (g <= top).all()  # every value lies between the first and last level


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_block_layout_is_a_permutation(hd):
    for side in (0, 1):
        p, d = np.meshgrid(np.arange(R.PAGE), np.arange(hd), indexing="ij")
        byte, high = R.code_at(hd, side, p, d)
        assert np.array_equal(np.sort((2 * byte + high).ravel()), np.arange(R.PAGE * hd))
        # two codes of a byte belong to one position
        owner = np.full(R.PAGE * hd // 2, -1)
        for half in (0, 1):
            pos, at = p[high == half], byte[high == half]
            assert half == 0 or (owner[at] == pos).all()
            owner[at] = pos


def test_put_get_round_trip():
    rng = np.random.default_rng(2)
    cache = rng.integers(0, 256, (5, 2, 2, R.block_bytes(128)), dtype=np.uint8)
    table = np.array([[3, 0, 4]], np.int32)
    pos = np.arange(60, 140)
    k, v = (_values(rng, len(pos) * 2, 128).reshape(len(pos), 2, 128) for _ in "kv")
    R.put(cache, table, 0, pos, k, v)
    for got, x in zip(R.get(cache, table, 0, pos), (k, v)):
        assert np.array_equal(got, R.values(*R.quantise(x)))


def _lib():
    import rustfox_b200 as rf
    return rf, rf.lib()


def _view(rf, p, **kw):
    a = dict(cache=p, table=p, row_start=p, kv_len=p, n_pages=4, n_head_kv=2, head_dim=64, n_seq=1, table_stride=2,
             n_rows=3)
    a.update(kw)
    return rf.api.Kv4(**a)


@pytest.fixture()
def buf():
    b = C.create_string_buffer(1 << 14)
    base = (C.addressof(b) + 15) // 16 * 16
    yield base
    del b


CACHE_CASES = [
    (dict(head_dim=96), 5), (dict(head_dim=0), 5), (dict(n_head_kv=0), 1), (dict(n_seq=1025), 1),
    (dict(n_rows=(1 << 20) + 1), 1), (dict(table_stride=(1 << 24) + 1), 1), (dict(n_pages=1 << 31), 1),
    (dict(cache=None), 1), (dict(table=None), 1), (dict(row_start=None), 1), (dict(kv_len=None), 1),
    (dict(cache="odd"), 1),
]


@pytest.mark.parametrize("change,want", CACHE_CASES)
def test_every_call_refuses_a_bad_cache(buf, change, want):
    rf, L = _lib()
    if change.get("cache") == "odd":
        change = dict(cache=buf + 4)
    c = _view(rf, buf, **change)
    calls = [L.foxcuda_kv4_write(C.byref(c), 0, buf, 1024, buf, 1024, None),
             L.foxcuda_kv4_read(C.byref(c), 0, buf, buf, None),
             L.foxcuda_kv4_attention(C.byref(c), 0, buf, 1024, 4, 0.0, buf, 1 << 40, buf, None)]
    assert calls == [want] * 3 and rf.last_error()


def test_rows_types_and_strides_are_refused(buf):
    rf, L = _lib()
    c = C.byref(_view(rf, buf))
    w = C.byref(_view(rf, buf, table_stride=17))
    huge = C.byref(_view(rf, buf, n_rows=1 << 20, table_stride=1 << 12))  # 2^31 pages of tiles
    odd = buf + 8
    cases = [
        (L.foxcuda_kv4_write(None, 0, buf, 128, buf, 128, None), 1),
        (L.foxcuda_kv4_write(c, 8, buf, 128, buf, 128, None), 5),       # Q8_0 rows
        (L.foxcuda_kv4_write(c, 0, None, 128, buf, 128, None), 1),
        (L.foxcuda_kv4_write(c, 0, odd, 128, buf, 128, None), 1),
        (L.foxcuda_kv4_write(c, 0, buf, 127, buf, 128, None), 1),       # shorter than a row
        (L.foxcuda_kv4_write(c, 0, buf, 130, buf, 128, None), 1),       # 520 bytes: unaligned rows
        (L.foxcuda_kv4_write(c, 1, buf, 132, buf, 128, None), 1),       # 264 bytes
        (L.foxcuda_kv4_read(c, 0, buf, odd, None), 1),
        (L.foxcuda_kv4_read(c, 34, buf, buf, None), 5),
        (L.foxcuda_kv4_attention(c, 0, buf, 256, 3, 0.0, buf, 1 << 40, buf, None), 5),   # 3 heads over 2
        (L.foxcuda_kv4_attention(c, 0, buf, 256, 0, 0.0, buf, 1 << 40, buf, None), 5),
        (L.foxcuda_kv4_attention(c, 0, buf, 2048, 32, 0.0, buf, 1 << 40, buf, None), 5),  # 16 to a KV head
        (L.foxcuda_kv4_attention(c, 0, buf, 256, 4, -1.0, buf, 1 << 40, buf, None), 1),
        (L.foxcuda_kv4_attention(c, 0, buf, 256, 4, float("nan"), buf, 1 << 40, buf, None), 1),
        (L.foxcuda_kv4_attention(c, 0, buf, 256, 4, float("inf"), buf, 1 << 40, buf, None), 1),
        (L.foxcuda_kv4_attention(w, 0, buf, 256, 4, 0.0, buf, 16, buf, None), 1),         # workspace too small
        (L.foxcuda_kv4_attention(w, 0, buf, 256, 4, 0.0, None, 1 << 40, buf, None), 1),
        (L.foxcuda_kv4_attention(huge, 0, buf, 256, 4, 0.0, buf, 1 << 40, buf, None), 1),
        (L.foxcuda_kv4_attention(c, 0, buf, 256, 4, 0.0, buf, 1 << 40, odd, None), 1),
    ]
    for i, (got, want) in enumerate(cases):
        assert got == want, i
    assert L.foxcuda_kv4_block_bytes(96) == 0 and L.foxcuda_kv4_block_bytes(128) == R.block_bytes(128)
    assert L.foxcuda_kv4_attention_workspace(96, 100) == 0
    assert L.foxcuda_kv4_attention_workspace(128, 16) == 0 < L.foxcuda_kv4_attention_workspace(128, 17)
    assert rf.api.KV4_WHOLE_PAGES == 16


def test_a_call_without_rows_or_sequences_does_nothing(buf):
    rf, L = _lib()
    for change in (dict(n_rows=0), dict(n_seq=0)):
        c = C.byref(_view(rf, buf, **change))
        assert L.foxcuda_kv4_write(c, 0, buf, 128, buf, 128, None) == 0
        assert L.foxcuda_kv4_read(c, 0, buf, buf, None) == 0
        assert L.foxcuda_kv4_attention(c, 0, buf, 256, 4, 0.0, buf, 0, buf, None) == 0


def test_rope_refusals(buf):
    rf, L = _lib()
    ok = dict(type=0, x=buf, xs=512, rows=2, h=4, kv=2, hd=64, qn=None, kn=None, eps=1e-5, cos=buf, sin=buf, n_pos=4,
              halves=0, pos=buf, q=buf, qs=256, k=buf, ks=128, stream=None)

    def call(**kw):
        return L.foxcuda_qk_norm_rope(*{**ok, **kw}.values())

    odd = buf + 4
    for kw, want in [(dict(type=12), 5), (dict(hd=80), 5), (dict(h=0), 1), (dict(kv=0), 1), (dict(halves=2), 1),
                     (dict(rows=(1 << 20) + 1), 1), (dict(n_pos=1 << 31), 1), (dict(x=None), 1), (dict(cos=None), 1),
                     (dict(pos=None), 1), (dict(k=None), 1), (dict(x=odd), 1), (dict(sin=odd), 1), (dict(qn=odd), 1),
                     (dict(xs=383), 1), (dict(qs=255), 1), (dict(ks=130), 1)]:
        assert call(**kw) == want, kw
    assert call(rows=0) == 0


def test_python_wrappers_check_their_tensors():
    torch = pytest.importorskip("torch")
    rf, _ = _lib()
    cache = torch.zeros(4, 2, 2, R.block_bytes(64), dtype=torch.uint8)
    table = torch.zeros(1, 2, dtype=torch.int32)
    start, lens = torch.tensor([0, 3], dtype=torch.int32), torch.tensor([3], dtype=torch.int32)
    x = torch.zeros(3, 2, 64)
    good = dict(cache=cache, table=table, row_start=start, kv_len=lens, k=x, v=x)
    bad = [dict(cache=cache.int()), dict(cache=cache[:, :, :1]), dict(table=table.long()), dict(table=table[0]),
           dict(row_start=start[:1]), dict(kv_len=lens.long()), dict(k=x[:2]), dict(v=x.half()),
           dict(k=x[:, :1], v=x[:, :1]), dict(k=x.transpose(1, 2).contiguous().transpose(1, 2)),
           dict()]  # the last: tensors of the host
    for change in bad:
        with pytest.raises(rf.FoxError):
            rf.kv4_write(**{**good, **change})
    with pytest.raises(rf.FoxError):
        rf.kv4_read(cache, table, start, lens)
    with pytest.raises(rf.FoxError):
        rf.kv4_attention(torch.zeros(3, 4, 64), cache, table, start, lens, out=torch.zeros(3, 4, 64).half())
    with pytest.raises(rf.FoxError):
        rf.kv4_cache(1, 1, 96, device="cpu")
    pos = torch.zeros(3, dtype=torch.int32)
    cos = torch.zeros(8, 32)
    rows = torch.zeros(3, 512)
    for change in (dict(x=rows[:, :300]), dict(pos=pos.long()), dict(cos=cos.double()), dict(cos=cos[:, :16]),
                   dict(q_norm=torch.ones(32)), dict(q_out=torch.zeros(3, 4, 64).half()), dict()):
        with pytest.raises(rf.FoxError):
            rf.qk_norm_rope(**{**dict(x=rows, n_head=4, n_head_kv=2, head_dim=64, pos=pos, cos=cos, sin=cos), **change})


def test_the_struct_is_laid_out_as_the_header_says(tmp_path):
    import pathlib
    import subprocess

    import rustfox_b200.api as api
    names = [f[0] for f in api.Kv4._fields_]
    src = tmp_path / "kv4.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "foxcuda.h"\nint main(void) {\n'
                   + "".join(f'  printf("%zu\\n", offsetof(foxcuda_kv4, {n}));\n' for n in names)
                   + '  printf("%zu\\n", sizeof(foxcuda_kv4));\n  return 0;\n}\n')
    include = pathlib.Path(__file__).resolve().parent.parent / "include"
    subprocess.run(["gcc", "-I", str(include), "-o", str(tmp_path / "kv4"), str(src)], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "kv4")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [getattr(api.Kv4, n).offset for n in names] + [C.sizeof(api.Kv4)]


def test_outputs_that_overlap_are_refused(buf):
    """Other blocks of the launch may still read what one writes."""
    rf, L = _lib()
    c = _view(rf, buf)
    rows = c.n_rows * c.n_head_kv * c.head_dim * 4
    assert L.foxcuda_kv4_read(C.byref(c), 0, buf, buf + rows - 16, None) == 1
    assert b"overlap" in L.foxcuda_last_error()
    assert L.foxcuda_kv4_attention(C.byref(c), 0, buf, 256, 4, 0.0, buf, 1 << 40, buf, None) == 1
    assert b"overlap" in L.foxcuda_last_error()
