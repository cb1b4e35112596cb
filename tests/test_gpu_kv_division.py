"""SNEPPX_kv_attention where a row lies in as many shares as it may: 256, of which one
is kept for a row that begins and ends within shares."""
import pytest

from test_gpu_kv_attention import test_division_of_rows as check_division

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "int8"])
@pytest.mark.parametrize("lengths", [
    [254 * 128],                     # 254 shares of a step
    [253 * 128 + 1],
    [255 * 128],                     # 128 of two steps
    [1] * 64 + [762 * 128],          # 255 shares of three steps, the first begun by other rows
    [1] * 65 + [762 * 128 - 5],
    [1] * 66 + [761 * 128 + 1, 300],
], ids=lambda x: f"{len(x)}x{max(x)}")
def test_rows_in_the_most_shares(lib, lengths, dtype):
    check_division(lib, lengths, 1, 16, dtype)
