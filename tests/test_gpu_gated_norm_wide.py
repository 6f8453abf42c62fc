"""gated_add_rms_norm on many rows of the widths whose backward keeps some values outside the registers."""
import pytest

from test_gpu_gated_norm import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("gate", ["none", "channel", "sequence", "token"])
@pytest.mark.parametrize("width", [4100, 8192])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_many_wide_rows(gpu, dtype, width, gate):
    shape = (3, 301, width)  # more rows than walkers, and than one of them takes of a gate
    check(gpu, dtype, shape, {"none": None, "channel": (width,), "sequence": (3, 1, width), "token": shape}[gate], width == 8192, 0.5)
    check(gpu, dtype, shape, {"none": None, "channel": (width,), "sequence": (3, 1, width), "token": shape}[gate], width != 8192, 0.5, w32=True)
