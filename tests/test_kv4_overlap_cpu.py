"""Outputs that overlap what a call of the 4-bit cache reads, or one another, are
refused: other blocks of the launch may still read what one writes. The rule is
compiled and compared with the sets of bytes here, the calls' refusals come
before any device call; what they let through runs in
test_kv4_overlap_gpu.py."""
import ctypes as C
import os
import random
import subprocess

import pytest

import kv4_ref as R

N, KV, HD, HEADS, PAGES, SEQS, STRIDE = 3, 2, 64, 4, 4, 2, 20
CACHE = PAGES * KV * 2 * R.block_bytes(HD)
TABLE, STARTS, LENS = SEQS * STRIDE * 4, (SEQS + 1) * 4, SEQS * 4
ROW, QROW = KV * HD * 4, HEADS * HD * 4
ARG = 1


@pytest.fixture(scope="module")
def at():
    """16-byte aligned addresses of arrays that do not overlap, none of which is
    ever read or written here."""
    import rustfox_b200 as rf
    need = rf.lib().foxcuda_kv4_attention_workspace(HD, STRIDE)
    sizes = dict(cache=CACHE, table=TABLE, starts=STARTS, lens=LENS, k=N * ROW, v=N * ROW, q=N * QROW, out=N * QROW,
                 work=need, cos=8 * HD // 2 * 4, sin=8 * HD // 2 * 4, pos=N * 4, wq=HD * 4, wk=HD * 4,
                 x=N * (QROW + 2 * ROW), spare=1 << 16)
    b = C.create_string_buffer(sum(sizes.values()) + 64 * len(sizes))
    p, base = {}, (C.addressof(b) + 15) // 16 * 16
    for name, n in sizes.items():
        p[name] = base
        base += (n + 31) // 16 * 16
    p["need"] = need
    yield p
    del b


def _call(op, p, change):
    """Status of a call with the addresses of p but for `change`."""
    import rustfox_b200 as rf
    L = rf.lib()
    a = {**p, **change}
    c = C.byref(rf.api.Kv4(a["cache"], a["table"], a["starts"], a["lens"], PAGES, KV, HD, SEQS, STRIDE, N))
    if op == "write":
        return L.foxcuda_kv4_write(c, 0, a["k"], ROW // 4, a["v"], ROW // 4, None)
    if op == "read":
        return L.foxcuda_kv4_read(c, 0, a["k"], a["v"], None)
    return L.foxcuda_kv4_attention(c, 0, a["q"], QROW // 4, HEADS, 0.0, a["work"], a["need"], a["out"], None)


@pytest.mark.parametrize("op,change", [
    ("write", lambda p: dict(k=p["cache"] + CACHE - 16)), ("write", lambda p: dict(v=p["cache"] - N * ROW + 16)),
    ("write", lambda p: dict(k=p["cache"] + 32)), ("write", lambda p: dict(table=p["cache"] + 4)),
    ("write", lambda p: dict(starts=p["cache"] + CACHE - 4)), ("write", lambda p: dict(lens=p["cache"])),
    ("read", lambda p: dict(k=p["v"] + N * ROW - 16)), ("read", lambda p: dict(v=p["k"])),
    ("read", lambda p: dict(k=p["cache"] + CACHE - 16)), ("read", lambda p: dict(v=p["cache"] - N * ROW + 16)),
    ("read", lambda p: dict(table=p["k"] + 4)), ("read", lambda p: dict(lens=p["v"])),
    ("read", lambda p: dict(starts=p["v"] + N * ROW - 4)),
    ("attention", lambda p: dict(q=p["out"])), ("attention", lambda p: dict(q=p["out"] + N * QROW - 16)),
    ("attention", lambda p: dict(out=p["cache"] + CACHE - 16)), ("attention", lambda p: dict(work=p["cache"] + 16)),
    ("attention", lambda p: dict(work=p["out"] + N * QROW - 16)), ("attention", lambda p: dict(out=p["work"] + p["need"] - 16)),
    ("attention", lambda p: dict(q=p["work"])), ("attention", lambda p: dict(table=p["out"])),
    ("attention", lambda p: dict(lens=p["work"] + 8)), ("attention", lambda p: dict(starts=p["out"] + 4)),
])
def test_what_overlaps_is_refused(at, op, change):
    import rustfox_b200 as rf
    assert _call(op, at, change(at)) == ARG
    assert "overlap" in rf.last_error()


X = (QROW + 2 * ROW) // 4  # elements of a row of x


@pytest.mark.parametrize("change", [
    lambda p: dict(q=p["x"], qs=QROW // 4),                                      # another stride
    lambda p: dict(q=p["x"], qs=X + 4),
    lambda p: dict(q=p["x"] + 16, qs=X),                                         # shifted
    lambda p: dict(q=p["x"] + QROW - 16, qs=X), lambda p: dict(k=p["x"], ks=X),
    lambda p: dict(k=p["x"] + QROW - 16, ks=X), lambda p: dict(k=p["x"] + 4 * X - 16, ks=X),
    lambda p: dict(q=p["x"] + 4 * X, qs=X),                                      # the next row's queries
    lambda p: dict(k=p["x"] + 4 * X + QROW, ks=X),
    lambda p: dict(rows=1, q=p["x"] + 16),
    lambda p: dict(k=p["q"] + N * QROW - 16), lambda p: dict(q=p["spare"], qs=X, k=p["spare"] + QROW - 16, ks=X),
    lambda p: dict(q=p["spare"] + ROW - 16, qs=X, k=p["spare"], ks=X),
    lambda p: dict(q=p["spare"], qs=X, k=p["spare"] + 4 * X, ks=X),
    lambda p: dict(cos=p["q"]), lambda p: dict(sin=p["k"]), lambda p: dict(pos=p["q"] + N * QROW - 4),
    lambda p: dict(wq=p["k"]), lambda p: dict(wk=p["q"] + 16),
])
def test_rotation_refuses_all_but_its_own_rows(at, change):
    import rustfox_b200 as rf
    p = {**at, "rows": N, "qs": QROW // 4, "ks": ROW // 4}
    p.update(change(at))
    st = rf.lib().foxcuda_qk_norm_rope(0, p["x"], X, p["rows"], HEADS, KV, HD, p["wq"], p["wk"], 1e-5, p["cos"], p["sin"], 8, 0,
                                       p["pos"], p["q"], p["qs"], p["k"], p["ks"], None)
    assert st == ARG and "overlap" in rf.last_error()


RULE = r"""
#include "%s/rustfox_b200/csrc/host.cuh"
int* fox::kernel_err_ptr() { return nullptr; }
int main() {
  size_t v[8];
  while (scanf("%%zu %%zu %%zu %%zu %%zu %%zu %%zu %%zu", v, v + 1, v + 2, v + 3, v + 4, v + 5, v + 6, v + 7) == 8)
    printf("%%d", (int)fox::overlap(fox::Rows{(void*)v[0], v[1], v[2], v[3]}, fox::Rows{(void*)v[4], v[5], v[6], v[7]}));
}
"""


def test_the_rule_against_sets_of_bytes(tmp_path):
    """Rows of one stride are told apart exactly, and so are single pieces of
    memory; of different strides, the ranges are."""
    from rustfox_b200 import build
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    (tmp_path / "rule.cu").write_text(RULE % root)
    subprocess.run([build.nvcc(), "-std=c++17", "-cudart", "static", "-o", str(tmp_path / "rule"), str(tmp_path / "rule.cu")],
                   check=True, capture_output=True)
    rng, cases = random.Random(1), []
    for _ in range(20000):
        s = rng.randint(1, 12)
        a, b = ([rng.randint(1, 60), rng.randint(0, s), rng.randint(0, 4), s] for _ in "ab")
        if rng.random() < 0.3:
            b[3] = max(b[1], rng.randint(1, 12))
        if rng.random() < 0.1:
            (a if rng.random() < 0.5 else b)[0] = 0  # no array
        cases.append((a, b))
    got = subprocess.run([str(tmp_path / "rule")], input="\n".join(" ".join(map(str, a + b)) for a, b in cases), text=True,
                         check=True, capture_output=True).stdout
    assert len(got) == len(cases)

    def held(r, whole=False):
        p, row, n, stride = r
        if not p or not row or not n:
            return set()
        return set(range(p, p + (n - 1) * stride + row)) if whole else {p + i * stride + j for i in range(n) for j in range(row)}

    for (a, b), g in zip(cases, got):
        ranges = a[3] != b[3] or a[2] < 2 or b[2] < 2
        assert (g == "1") == bool(held(a, ranges) & held(b, ranges)), (a, b)
