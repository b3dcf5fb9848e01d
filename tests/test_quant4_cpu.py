"""Weights in 4 bits where no GPU is needed: what is refused, and the plain forms that the GPU tests use."""
from __future__ import annotations

import pytest
import torch

import helpers
import quant4_util as Q


def _w(shape=(32, 128), group=64, pair=False):
    from moe_b200.ops import quant

    G, N, K = (1, *shape) if len(shape) == 2 else shape
    strips = G * (2 * -(-(N // 2) // 16) if pair else -(-N // 16))
    return quant.Weight4(torch.full((strips * -(-K // 64) * 512,), 0x88, dtype=torch.uint8),
                         torch.zeros(strips * -(-K // group) * 16, dtype=torch.bfloat16), shape, group, pair)


@pytest.mark.parametrize("change", ["codes short", "scales short", "codes dtype", "scales dtype", "strided", "group", "shape", "empty", "odd pair"])
def test_a_weight_of_the_wrong_parts_is_refused(change):
    from moe_b200.ops import core, quant

    codes, scales, shape, group, pair = torch.zeros(2 * 2 * 512, dtype=torch.uint8), torch.zeros(2 * 2 * 16, dtype=torch.bfloat16), (32, 128), 64, False
    quant.Weight4(codes, scales, shape, group, pair)
    if change == "codes short":
        codes = codes[:-1]
    elif change == "scales short":
        scales = scales[:-16]
    elif change == "codes dtype":
        codes = codes.to(torch.int8)
    elif change == "scales dtype":
        scales = scales.float()
    elif change == "strided":
        codes = torch.zeros(2 * 2 * 512, 2, dtype=torch.uint8)[:, 0]
    elif change == "group":
        group = 48
    elif change == "shape":
        shape = (1, 1, 32, 128)
    elif change == "empty":
        shape = (0, 128)
    else:
        shape, pair = (31, 128), True
    with pytest.raises(core.KernelError):
        quant.Weight4(codes, scales, shape, group, pair)


def test_sizes_that_the_kernels_do_not_count_are_refused():
    from moe_b200.ops import core, quant

    empty = torch.zeros(0, dtype=torch.uint8), torch.zeros(0, dtype=torch.bfloat16)
    for shape in ((1 << 31, 8), (8, (1 << 30) + 1), (1 << 31, 8, 8)):
        with pytest.raises(core.KernelError, match="sizes"):
            quant.Weight4(*empty, shape)


def test_no_cpu_path():
    from moe_b200.ops import core, quant

    w, pair, x = _w(), _w((2, 32, 128), pair=True), torch.zeros(3, 128, dtype=torch.bfloat16)
    with pytest.raises(core.KernelError):
        quant.quantize(torch.zeros(16, 64))
    with pytest.raises(core.KernelError):
        quant.dequantize(w)
    with pytest.raises(core.KernelError):
        quant.gemm4(x, w, torch.zeros(3, 32))
    with pytest.raises(core.KernelError):
        quant.experts4(x, torch.zeros(3, 1, dtype=torch.int32), torch.zeros(3, 1), pair, _w((2, 128, 16)), torch.zeros(3, 128))


def test_what_a_model_may_hold_in_4_bits(model_dirs):
    import moe_b200

    d = model_dirs.get("A", "bfloat16", seed=1, std=0.02)
    for kw in (dict(weights="int8"), dict(weights="int4", weight_group=48), dict(weights="int4", dtype="float32")):
        with pytest.raises(ValueError):
            moe_b200.load_model(d, device="cpu", **kw)
    with pytest.raises(ValueError):
        moe_b200.random_model(helpers.CONFIG_A, weights="fp4", device="cpu")


def test_a_weight_says_what_it_is():
    w = _w((3, 32, 70), 32, pair=True)
    assert (w.G, w.N, w.K) == (3, 32, 70) and w.nbytes == 3 * 2 * (2 * 512 + 3 * 32) and w.dtype == "int4" and "pair" in repr(w)
    assert not bool(Q.values_by_place(w).any())


def test_plain_values_are_bfloat16_and_near():
    torch.manual_seed(0)
    w = torch.randn(40, 96, dtype=torch.float64)
    v = Q.plain_values(w, 32)
    assert torch.equal(v, v.to(torch.bfloat16).double())
    step = w.reshape(40, 3, 32).abs().amax(-1, keepdim=True) / 7 * (1 + 2.0 ** -5)
    assert bool(((w - v).reshape(40, 3, 32).abs() <= step / 2 + 1e-12).all())
