"""Rows of any alignment past what one launch's second grid dimension holds: 65535 tiles of 128 rows."""
import pytest

import fenix_b200 as fx
from test_i8_gpu import run_linear

pytestmark = pytest.mark.gpu

ROWS = 65535 * 128


@pytest.mark.parametrize("rows,launches", [(ROWS, 1), (ROWS + 1, 2), (ROWS + 70, 2), (ROWS + 128 * 5 + 3, 2)])
@pytest.mark.parametrize("mode", ["row", "tensor"])
def test_rows_of_two_launches(cuda_torch, rows, launches, mode):
    """The second launch's rows, their scales and their results begin where the first one's end; its few tiles may be shared by clusters."""
    if cuda_torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of free device memory")
    for n, k, yt in ((3, 17, "bf16"), (2, 300, "f32") if launches == 2 else (1, 5, "f32")):
        before = fx.kernel_launches()
        run_linear(cuda_torch, rows, n, k, yt, mode, bias=True, xs=k + 1 - k % 2, ws=k)
        assert fx.kernel_launches() - before == launches
        cuda_torch.cuda.empty_cache()
