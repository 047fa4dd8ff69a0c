"""Which form the plan of the fp8 products takes: that the sizes tested on the GPU reach every form, with a last block
that the inputs fill and one that they do not, whole and split."""
import ctypes

import pytest

from ada_mla import capi
from linear_sizes import OWN, TILES

TAIL = {False, True}


@pytest.mark.parametrize("form", TILES)
def test_sizes_reach_their_form(form):
    outputs, rows, split = form
    for size in TILES[form]:
        got = capi.linear_fp8_plan(*size, quantized=True)
        assert (got[0], got[1], got[2] > 1) == form, (size, got)
        assert got[3] == 1 + split, size
        m, k, n = size
        assert m % 64 and n % 16, size  # neither fills its tiles
    assert {k % 128 != 0 for _, k, _ in TILES[form]} == TAIL
    if split:  # inputs that the splits do not share evenly, for either end
        uneven = {(k % 128 != 0, -(-k // 128) % capi.linear_fp8_plan(m, k, n, quantized=True)[2] != 0) for m, k, n in TILES[form]}
        assert (True, True) in uneven and (False, True) in uneven


@pytest.mark.parametrize("outputs", OWN)
def test_sizes_that_quantise_themselves(outputs):
    for size in OWN[outputs]:
        assert capi.linear_fp8_plan(*size) == (outputs, 16, 1, 1), size
    assert {k % 128 != 0 for _, k, _ in OWN[outputs]} == TAIL


@pytest.mark.parametrize("rows,inputs,outputs", [(16, 2048, 576), (16, 2048, 129280), (8, 4096, 4096), (1, 512, 65536), (16, 256, 32768),
                                                 (8, 1536, 24576), (4, 7168, 16384), (1, 32768, 2048), (1, 32768, 16384), (1, 16384, 129280)])
def test_rows_quantised_once(rows, inputs, outputs):
    # where the workgroups' own quantisation, round after round, takes longer than a launch for it
    product = capi.linear_fp8_plan(rows, inputs, outputs, quantized=True)
    assert capi.linear_fp8_plan(rows, inputs, outputs) == (*product[:3], product[3] + 1)


@pytest.mark.parametrize("rows,inputs,outputs,tiles", [(1, 32768, 70, (16, 16)), (1, 32768, 576, (16, 16)), (16, 32768, 2500, (16, 16)),
                                                       (20, 10240, 70, (16, 32)), (40, 7168, 576, (16, 64)), (64, 7168, 70, (16, 64))])
def test_few_workgroups_stream_faster(rows, inputs, outputs, tiles):
    # a step of the few-row kernel on few CUs is up to half of what it is on all of them: no split tiles for these
    assert capi.linear_fp8_plan(rows, inputs, outputs, quantized=True) == (*tiles, 1, 1)


@pytest.mark.parametrize("rows,inputs,outputs", [(1, 5120, 576), (16, 1280, 4096), (8, 1024, 24576), (1, 7168, 16384), (1, 24576, 576),
                                                 (2, 8192, 4096)])
def test_rows_quantised_by_every_workgroup(rows, inputs, outputs):
    assert capi.linear_fp8_plan(rows, inputs, outputs) == (16 if outputs <= 4096 else 32, 16, 1, 1)


def test_every_form_is_listed():
    # forms met over a grid of sizes are those listed
    met, step = set(), [16 * 2 ** i + 16 * (i % 2) for i in range(3, 11)]
    for k in step:
        for n in (16, 100, 576, 2000, 4096, 4999, 8192, 16000):
            for m in (1, 16, 17, 33, 64, 65, 100, 200, 333, 500, 1000, 2000, 4000, 8192):
                outputs, rows, splits, launches = capi.linear_fp8_plan(m, k, n, quantized=True)
                met.add((outputs, rows, splits > 1))
                assert launches == 1 + (splits > 1)
                own = capi.linear_fp8_plan(m, k, n)
                assert own[3] in (1, 2 + (splits > 1)) and (own[3] > 1 or own[1:3] == (16, 1))
    assert met <= set(TILES)


def test_plan_argument_errors():
    plan = capi.load().mla_linear_fp8_plan
    out = [ctypes.c_int() for _ in range(4)]
    at = [ctypes.byref(v) for v in out]
    assert plan(3, 256, 100, 0, *at) == capi.STATUS_SUCCESS
    for bad in ((0, 256, 100), (3, 24, 100), (3, 256, 0), (2 ** 26 + 1, 256, 100)):
        assert plan(*bad, 1, *at) == capi.STATUS_INVALID_VALUE
    for i in range(4):
        assert plan(3, 256, 100, 0, *at[:i], None, *at[i + 1:]) == capi.STATUS_INVALID_VALUE


def test_rows_in_several_launches():
    assert capi.linear_fp8_plan(2 ** 26, 64, 256) == (16, 64, 1, 3)  # quantised, then 2^20 row tiles x 16 x 256 threads: two grids
    assert capi.linear_fp8_plan(2 ** 26 - 64, 64, 256, quantized=True)[3] == 1
