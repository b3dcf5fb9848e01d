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


# ------------------------------------------------------------------------------------------------ weights written right in front of a product
FORMS = {  # rows, N, K, pair, groups
    "block a strip": (3, 2048, 1024, False, 0), "streamed": (4, 16384, 512, True, 0), "streamed groups": (40, 512, 512, False, 8),
    "tensor core": (200, 2048, 1024, False, 0), "tensor core, splits": (40, 1024, 2048, False, 0), "wide groups": (400, 512, 512, True, 8), "layer": (4, 256, 512, True, 6)}


def _form(quant, form):
    """(the weights' stored tensors, their shapes, a call of Weight4's of them)"""
    M, N, K, pair, groups = FORMS[form]
    torch.manual_seed(len(form))
    x = torch.randn(M, K, device=DEV).to(BF)
    if form == "layer":
        shapes = [((groups, 2 * N, K), True), ((groups, K, N), False), ((4 * N, K), True), ((K, 2 * N), False)]
        idx = torch.rand(M, groups, device=DEV).topk(2, dim=1).indices.to(torch.int32).contiguous()
        w, gate = torch.rand(M, 2, device=DEV), torch.rand(M, device=DEV)

        def call(gu, d, sgu, sd):
            out = torch.empty(M, K, device=DEV)
            assert quant.experts4(x, idx, w, gu, d, out, shared_gate_up=sgu, shared_down=sd, shared_gate=gate)
            return out
    else:
        shapes = [((groups, N, K) if groups else (N, K), pair)]
        off = torch.arange(0, M + 1, M // groups, dtype=torch.int32, device=DEV) if groups else None
        call = lambda w4: quant.gemm4(x, w4, torch.empty(M, N // 2 if pair else N, device=DEV), swiglu=pair, group_offsets=off)  # noqa: E731
    return shapes, call


@pytest.mark.parametrize("form", list(FORMS))
def test_a_product_right_behind_the_kernels_that_wrote_its_weight(quant, form):
    """Other codes and scales into the same tensors by torch's kernels, the scales last, and a product of a new Weight4 of them in the next launch."""
    shapes, call = _form(quant, form)
    sets = []
    for seed in (1, 2):
        made = [quant.quantize((torch.randn(*s, device=DEV) * s[-1] ** -0.5).to(BF), 64, pair=p) for s, p in shapes]
        torch.cuda.synchronize()
        sets.append((made, call(*made)))
    assert not torch.equal(sets[0][1], sets[1][1])
    room = [(torch.empty_like(w.codes), torch.empty_like(w.scales)) for w in sets[0][0]]
    for _ in range(60):
        for made, want in sets:
            for (codes, scales), w in zip(room, made):
                codes.copy_(w.codes), scales.copy_(w.scales)
            got = call(*[quant.Weight4(c, s, w.shape, 64, pair=w.pair) for (c, s), w in zip(room, made)])
            assert torch.equal(got, want)


@pytest.mark.parametrize("form", list(FORMS))
def test_a_product_right_behind_the_quantiser_whatever_its_form(quant, form):
    shapes, call = _form(quant, form)
    ws = [(torch.randn(*s, device=DEV) * s[-1] ** -0.5).to(BF) for s, _ in shapes]
    want = call(*[quant.quantize(w, pair=p) for w, (_, p) in zip(ws, shapes)])
    for _ in range(60):
        assert torch.equal(call(*[quant.quantize(w, pair=p) for w, (_, p) in zip(ws, shapes)]), want)


@pytest.mark.parametrize("form", list(FORMS))
def test_a_weight_is_read_early_only_where_nothing_in_front_can_have_written_it(quant, form, monkeypatch):
    """The first product on a stream waits for what is in front of it, whatever other streams have done; a captured one leaves no trace; behind settle all read
    early."""
    shapes, call = _form(quant, form)
    made = [quant.quantize((torch.randn(*s, device=DEV) * s[-1] ** -0.5).to(BF), 64, pair=p) for s, p in shapes]
    early, real = [], quant.lib()

    class Spy:
        def __getattr__(self, name):
            fn = getattr(real, name)
            if not name.startswith(("moe_gemm_q4", "moe_experts_q4")):
                return fn

            def launch(*args):
                code = fn(*args)
                if code != -1:
                    early.append(bool(args[-3]))
                return code
            return launch

    monkeypatch.setattr(quant, "_lib", Spy())
    call(*made), call(*made)
    assert early == [False, True]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(*made), call(*made)
    torch.cuda.synchronize()
    assert early[2:] == [False, True]
    again = [quant.Weight4(w.codes, w.scales, w.shape, 64, pair=w.pair) for w in made]
    with torch.cuda.stream(side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            call(*again), call(*again)
        call(*again)
    torch.cuda.synchronize()
    assert early[4:] == [False, False, False]
    for w in again[:-1]:
        w.settle()
    torch.cuda.current_stream().synchronize()
    call(*again)
    again[-1].settle()
    call(*again)
    assert early[7:] == [False, True]
    torch.cuda.synchronize()


def test_a_models_weights_are_settled(quant):
    import helpers
    import moe_b200

    model = moe_b200.random_model(helpers.CONFIG_A, seed=1, weights="int4")
    held = [w for b in model.blocks for p in b.parts() for w in vars(p).values() if isinstance(w, quant.Weight4)]
    assert held and all(w.read_on is None for w in held)
