"""CPU checks of the largest fp8 products: what no launch can hold is refused before anything is launched, by the
size query too (pointers are never dereferenced)."""
import pytest
import torch

from ada_mla import capi
from test_operators_boundary_cpu import FAKE, _caller, _ext

MOST_BLOCKS = 2 ** 30 - 64  # blocks of 128 inputs over all rows: four threads quantise one, 2^32 - 1 make a grid


@pytest.mark.parametrize("rows,inputs", [(2 ** 26, 2048), (2 ** 26 - 3, 2032), (2 ** 23, 2 ** 14), (2 ** 20 - 1, 2 ** 17 + 16)])
def test_blocks_of_x_past_a_grid(rows, inputs):
    blocks = -(-inputs // 128)
    assert rows * blocks > MOST_BLOCKS
    size = capi.load().mla_linear_fp8_workspace_size
    assert size(rows, inputs, 16) == 0
    for t in ("fp16", "bf16"):
        call = _caller("mla_quantize_fp8_" + t, "x q s rows k stride stream",
                       dict(x=FAKE, q=FAKE, s=FAKE, rows=rows, k=inputs, stride=0, stream=None))
        assert call() == capi.STATUS_INVALID_VALUE
        names = "x w ws out space bytes rows k n xstride wstride stream"
        call = _caller("mla_linear_fp8_" + t, names, dict.fromkeys(names.split(), FAKE) | dict(
            bytes=1 << 62, rows=rows, k=inputs, n=16, xstride=0, wstride=inputs, stream=None))
        assert call() == capi.STATUS_INVALID_VALUE
    m, f8 = _ext(), torch.float8_e4m3fn
    x = torch.zeros(1, inputs, dtype=torch.float16).expand(rows, inputs)
    with pytest.raises(RuntimeError, match="too many rows"):
        m.mla_quantize_fp8(x)
    with pytest.raises(RuntimeError, match="too many rows"):
        m.mla_linear_fp8(x, torch.zeros(16, inputs, dtype=f8), torch.zeros(1, blocks))


def test_the_most_blocks():
    size = capi.load().mla_linear_fp8_workspace_size
    assert size(2 ** 26 - 4, 2048, 16) >= (2 ** 26 - 4) * 2048  # 2^30 - 64 blocks
    assert size(2 ** 26 - 3, 2048, 16) == 0


@pytest.mark.parametrize("rows,inputs,outputs", [(2 ** 26, 64, 256), (2 ** 26, 16, 511), (2 ** 26 - 7, 128, 500), (2 ** 20, 16, 2 ** 15),
                                                 (1, 2 ** 22, 2 ** 26), (33, 16, 2 ** 26), (65, 4096, 2 ** 26)])
def test_sizes_within_the_limits_stay(rows, inputs, outputs):
    assert capi.load().mla_linear_fp8_workspace_size(rows, inputs, outputs) >= rows * inputs
