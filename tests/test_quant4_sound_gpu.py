"""Weights held in 4 bits on the GPU: what a layer's 32-bit outputs keep, weights written right in front of a product, sizes that no tile divides, models that
hold everything they say they hold."""
from __future__ import annotations

import pytest
import torch

import quant4_util as Q
from test_quant4_gpu import BF, DEV, fine, quant, status, weight  # noqa: F401  (quant: a fixture)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ a layer of experts
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("T", [1, 5, 8])
def test_what_lies_between_a_layers_products_keeps_32_bits(quant, T, group):
    """One element of x and one of each row of the down projections are not zero, so that every output is one product: what lies between the two
    products shows as it is.  The gate's function is off by 2^-22 of itself and a few roundings (of 2^-24), the product's terms are added cut (2^-23 each), the
    scale, the token's weight and the gate of the shared expert round once each: 2^-20 covers them twice over.  Two bfloat16 terms would leave 2^-17."""
    H, E, size, shared = 264, 3, 200, 136
    torch.manual_seed(T * group)
    gu, GU = weight(quant, (E, 2 * size, H), group, pair=True)
    sgu, SGU = weight(quant, (2 * shared, H), group, pair=True, seed=1)

    def sparse(shape):
        w = torch.zeros(*shape, device=DEV)
        n = torch.arange(shape[-2], device=DEV)
        w[..., n, n % shape[-1]] = torch.randn(*shape[:-1], device=DEV)
        w4 = quant.quantize(w.to(BF), group)
        return w4, quant.dequantize(w4).double()

    (d, D), (sd, SD) = sparse((E, H, size)), sparse((H, shared))
    x = torch.zeros(T, H, dtype=BF, device=DEV)
    x[:, 77] = torch.randn(T, device=DEV).to(BF) * 30
    idx = torch.randint(0, E, (T, 1), dtype=torch.int32, device=DEV)
    w, gate = torch.rand(T, 1, device=DEV) + 0.5, torch.rand(T, device=DEV) + 0.5
    none = torch.full_like(idx, -1)

    def plain(GU, D, f):
        a = Q.gated("silu", *(x.double() @ GU.transpose(-1, -2)).chunk(2, dim=-1))           # (one product an element: exact)
        n = torch.arange(H, device=DEV)
        return f.double() * D[..., n, n % D.shape[-1]] * a[..., n % D.shape[-1]]

    for what in ("routed", "shared"):
        st, out = status(), torch.full((T, H), float("nan"), device=DEV)
        if what == "routed":
            assert quant.experts4(x, idx, w, gu, d, out, status=st)
            y = torch.stack([plain(GU[e], D[e], w[t])[t] for t, e in enumerate(idx[:, 0].tolist())])
        else:
            assert quant.experts4(x, none, w, gu, d, out, shared_gate_up=sgu, shared_down=sd, shared_gate=gate, status=st)
            y = plain(SGU[0], SD, gate.unsqueeze(1))
        fine(st)
        far = (out.double() - y).abs()
        assert bool((far <= 2.0 ** -20 * y.abs() + 1e-37).all()), f"{what}: {float((far / y.abs().clamp_min(1e-37)).max()):.3g} of an output"


# ------------------------------------------------------------------------------------------------ waits
@pytest.mark.parametrize("per", [3, 12])
@pytest.mark.parametrize("pair", [False, True])
def test_a_wait_of_streamed_groups_that_runs_out(quant, pair, per):
    """Groups of few rows, one and two tiles of rows at a time: every team of every block gives up on several runs of units, and as a whole."""
    from moe_b200.ops import core

    torch.manual_seed(per)
    groups, K, N = 9, 328, 640
    off = torch.arange(0, groups * per + 1, per, dtype=torch.int32, device=DEV)
    w4, W = weight(quant, (groups, N, K), pair=pair)
    st, x, out = status(), torch.randn(groups * per, K, device=DEV).to(BF), torch.empty(groups * per, N // 2 if pair else N, device=DEV)
    run = lambda: quant.gemm4(x, w4, out, swiglu=pair, group_offsets=off, status=st)  # noqa: E731
    L = quant.lib()
    L.moe_q4_set_wait_test(1, 2000)
    try:
        run()
        torch.cuda.synchronize()
    finally:
        L.moe_q4_set_wait_test(0, 0)
    assert int(st[0]) & 8, "the wait that ran out was not reported"
    with pytest.raises(core.KernelError, match="4-bit weights"):
        core.check_status(st)
    run()
    fine(st)
    for g in range(groups):
        Q.check_product(out[g * per:(g + 1) * per], x[g * per:(g + 1) * per], W[g], swiglu=pair)
