"""row_start that names more rows than the row arrays hold: every call places
the rows that are there alike, and reports the others."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from test_kv4_gpu import Cache  # noqa: E402
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
