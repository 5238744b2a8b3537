"""Which kernel an FP8 product takes (lm_fp8_plan_*, host only): every kernel is taken by some sizes, and one launch's
tiles are bounded."""
import dataclasses

import pytest

import litemind_amd as lm
from litemind_amd import workload as wl

F32, BF16 = lm.DT_F32, lm.DT_BF16


def tile(p):
    return p.tile_rows, p.tile_features


@pytest.mark.parametrize("rows,n,k,dtype,want,shared", [
    (1, 2048, 10944, F32, (16, 16), False), (48, 256, 8192, BF16, (16, 16), False),
    (65, 4100, 656, F32, (32, 128), False), (33, 1290, 4112, F32, (32, 128), True),
    (400, 5130, 656, F32, (64, 128), False), (300, 2056, 6016, F32, (64, 128), True),
    (3000, 1290, 656, F32, (128, 128), False), (4100, 130, 6016, F32, (128, 128), True),
    (3000, 5130, 6016, F32, (128, 256), False),
    (65, 4100, 656, BF16, (32, 128), False), (33, 1290, 4112, BF16, (32, 128), True),
    (400, 5130, 1424, BF16, (64, 128), False), (1300, 130, 6016, BF16, (64, 128), True),
    (3000, 1290, 656, BF16, (128, 128), False), (1000, 2056, 6016, BF16, (128, 128), True),
    (1930, 2056, 8208, BF16, (128, 256), False), (1000, 8200, 656, BF16, (256, 256), False)])
def test_gemm(rows, n, k, dtype, want, shared):
    p = lm.fp8_plan_gemm(rows, n, k, dtype)
    assert tile(p) == want and (p.shares > 1) == shared
    assert p.fp32_sums == (dtype == F32 or want == (16, 16))
    assert p.tiles == -(-rows // want[0]) * -(-n // want[1])


@pytest.mark.parametrize("groups,rows,n,k,dtype,want", [
    (64, 6, 2048, 1408, F32, (16, 16)), (4, 1040, 130, 1424, F32, (32, 128)), (6, 4800, 130, 656, F32, (64, 128)),
    (20, 8000, 130, 656, F32, (128, 128)), (16, 1600, 2056, 4112, F32, (128, 256)), (4, 1040, 130, 1424, BF16, (32, 128)),
    (6, 4800, 130, 656, BF16, (64, 128)), (20, 8000, 130, 656, BF16, (128, 128)), (16, 1600, 2056, 4112, BF16, (128, 256)),
    (160, 41600, 130, 144, BF16, (256, 256))])
def test_grouped_gemm(groups, rows, n, k, dtype, want):
    p = lm.fp8_plan_gemm(rows, n, k, dtype, groups=groups)
    assert tile(p) == want and p.shares == 1
    assert p.tiles == (rows // want[0] + groups if rows >= groups else rows) * -(-n // want[1])


@pytest.mark.parametrize("groups,rows,inter,k,kernel,rows_of_tile", [
    (1, 1, 144, 144, 0, 32), (8, 2080, 144, 656, 1, 32), (6, 4800, 144, 656, 2, 64), (20, 8000, 144, 656, 3, 128)])
def test_swiglu(groups, rows, inter, k, kernel, rows_of_tile):
    p = lm.fp8_plan_swiglu(groups, rows, inter, k)
    assert p.kernel == kernel and tile(p) == (rows_of_tile, 128) and p.fp32_sums == 1 and p.shares == 1


def test_layers():
    """V2-Lite's layers: what the shared experts' tiles lie beside, and which tiles take the FP8 matrix cores."""
    config = wl.V2_LITE.moe_config(num_layers=1)
    for tokens, beside, gate_up, down in ((1, 1, (0, 1), (16, 16)), (2, 1, (1, 1), (32, 128)), (128, 1, (1, 1), (32, 128)),
                                          (129, 0, (1, 1), (32, 128)), (512, 0, (3, 0), (64, 128)),
                                          (1024, 0, (3, 0), (128, 128)), (2048, 0, (4, 0), (256, 256))):
        p = lm.fp8_plan_layer(config, tokens)
        assert p.beside == beside and (p.gate_up.kernel, p.gate_up.fp32_sums) == gate_up and tile(p.down) == down, tokens
        assert (p.other_gate_up.tiles > 0) == (p.other_down.tiles > 0) == (not beside)
    p = lm.fp8_plan_layer(config, 512, dense=True)
    assert p.beside == 0 and p.gate_up.tiles == p.down.tiles == 0 and p.other_gate_up.tiles > 0 and p.other_down.shares > 1


def test_tiles_that_a_launch_has_room_for():
    """Where the tiles of the least cost are more than 2^22, larger ones are taken."""
    for dtype, room in ((F32, (128, 256)), (BF16, (256, 256))):
        p = lm.fp8_plan_gemm(512, 2 ** 20, 16, dtype, groups=512)
        assert p.tile_rows >= 32 and p.tile_features == room[1] and p.tiles <= 2 ** 22
        with pytest.raises(lm.LmError) as e:
            lm.fp8_plan_gemm(512, 2 ** 24, 16, dtype, groups=512)
        assert e.value.status == -1 and "tiles" in str(e.value)
    # a layer of 512 experts: no tokens that the path takes are too many
    d = dataclasses.replace(wl.V2_LITE, hidden=2 ** 20, inter=16, experts=512, top_k=16, n_shared=0)
    for tokens in (1, 100, 1000, 2000, 4095):
        assert lm.fp8_plan_layer(d.moe_config(num_layers=1), tokens).down.tiles <= 2 ** 22


@pytest.mark.parametrize("call", [
    lambda: lm.fp8_plan_gemm(0, 16, 16), lambda: lm.fp8_plan_gemm(1, 16, 24), lambda: lm.fp8_plan_gemm(2 ** 28, 16, 16),
    lambda: lm.fp8_plan_gemm(1, 0, 16), lambda: lm.fp8_plan_gemm(1, 16, 16, dtype=lm.DT_F64),
    lambda: lm.fp8_plan_gemm(1, 16, 16, groups=513), lambda: lm.fp8_plan_gemm(1, 16, 16, groups=-1),
    lambda: lm.fp8_plan_swiglu(0, 1, 16, 16), lambda: lm.fp8_plan_swiglu(1, 1, 24, 16),
    lambda: lm.fp8_plan_swiglu(1, 2 ** 28, 16, 16), lambda: lm.fp8_plan_swiglu(1, 0, 16, 16),
    lambda: lm.fp8_plan_layer(wl.V2_LITE.moe_config(), 0), lambda: lm.fp8_plan_layer(wl.V2_LITE.moe_config(), 2 ** 32 // 8448),
    lambda: lm.fp8_plan_layer(dataclasses.replace(wl.V2_LITE, inter=136).moe_config(), 1),
    lambda: lm.fp8_plan_layer(dataclasses.replace(wl.V2_LITE, dense_inter=0).moe_config(), 1, dense=True)])
def test_refusals(call):
    with pytest.raises(lm.LmError) as e:
        call()
    assert e.value.status == -1
