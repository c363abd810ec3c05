"""Keys in parts, and their joining by one wave a row and by four, at every padded size of a head, on and off alignment; some parts empty, some rows too."""
import pytest

from test_gpu_attention import DTYPES, Problem

pytestmark = pytest.mark.gpu


@DTYPES
@pytest.mark.parametrize("dim", [17, 32, 72, 80, 96, 100, 128])
@pytest.mark.parametrize("layout", ["heads first", "odd"])
@pytest.mark.parametrize("queries,keys", [(1, 3000), (5, 17000), (40, 5000)], ids=["4 parts", "16 parts", "two blocks"])
def test_parts_of_every_size(dtype, dim, layout, queries, keys):
    for window, lengths in (((None, 0), None), ((300, 0), None), ((None, 0), ([queries, queries - 1], [3, keys - 1500]))):
        Problem(2, queries, keys, 4, 2, dim, dtype, window=window, lengths=lengths, layout=layout).check()
