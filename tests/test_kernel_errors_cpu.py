"""What foxcuda_kernel_errors says of the device error word's codes: a wait that
gave up (the output is not valid) is never hidden by a position that was
skipped. The host function is compiled and called here without a device."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC = r"""
#include "%s/rustfox_b200/csrc/host.cuh"
int* fox::kernel_err_ptr() { return nullptr; }
int main() {
  const int codes[] = {0, fox::KERR_WAIT, 2, fox::KERR_PAGES, fox::KERR_WAIT | fox::KERR_PAGES, 2 | fox::KERR_PAGES};
  for (int c : codes) {
    fox::g_err[0] = 0;
    const int st = fox::kernel_err_status(c);
    printf("%%d|%%s\n", st, fox::g_err);
  }
}
"""


@pytest.fixture(scope="module")
def answers(tmp_path_factory):
    from rustfox_b200 import build
    at = tmp_path_factory.mktemp("err")
    (at / "err.cu").write_text(SRC % ROOT)
    subprocess.run([build.nvcc(), "-std=c++17", "-cudart", "static", "-o", str(at / "err"), str(at / "err.cu")], check=True)
    out = subprocess.run([str(at / "err")], check=True, capture_output=True, text=True).stdout
    return [(int(x.split("|")[0]), x.split("|")[1]) for x in out.splitlines()]


def test_each_code(answers):
    none, wait, two, pages, both, two_pages = answers
    assert none == (0, "")
    for st, text in (wait, two, both, two_pages):
        assert st == 7 and "gave up" in text and "not valid" in text
    assert "code 1" in wait[1] and "code 2" in two[1] and "code 1" in both[1] and "code 2" in two_pages[1]
    assert pages[0] == 1 and "skipped" in pages[1] and "not valid" not in pages[1]
    assert "skipped" in both[1] and "skipped" in two_pages[1] and "skipped" not in wait[1]
