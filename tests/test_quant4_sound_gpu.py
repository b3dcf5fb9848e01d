"""Weights held in 4 bits on the GPU: what a layer's 32-bit outputs keep, weights written right in front of a product, sizes that no tile divides, models that
hold everything they say they hold."""
from __future__ import annotations

import pytest
import torch

import gpu_util as G
import quant4_util as Q
from test_quant4_gpu import BF, DEV, _designs as designs, fine, quant, status, weight  # noqa: F401  (quant: a fixture)

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


# ------------------------------------------------------------------------------------------------ sizes that no tile divides, stacks of any size
@pytest.mark.parametrize("rows", [[1, 0, 1], [40, 0, 17], [200, 150, 3]])
@pytest.mark.parametrize("K,pitch", [(7999, 8000), (7999, 7999), (6000, 6001), (131, 131), (136, 139)])
def test_groups_of_rows_that_are_no_whole_units(quant, K, pitch, rows):
    torch.manual_seed(K + rows[0])
    off, M = torch.tensor([0, *rows], dtype=torch.int32, device=DEV).cumsum(0).to(torch.int32), sum(rows)
    x = torch.randn(M, pitch, device=DEV).to(BF)[:, :K]
    for pair in (False, True):
        w4, W = weight(quant, (3, 48, K), 32 if K == 131 else 128, pair=pair)
        st, out = status(), torch.full((M, 24 if pair else 48), float("nan"), device=DEV)
        quant.gemm4(x, w4, out, swiglu=pair, group_offsets=off, any_rows=True, status=st)
        fine(st)
        for g in range(3):
            a, b = int(off[g]), int(off[g + 1])
            if a < b:
                Q.check_product(out[a:b], x[a:b], W[g], swiglu=pair)


@pytest.mark.parametrize("M", [1, 24, 25, 300])
@pytest.mark.parametrize("K,pitch,at", [(131, 131, 0), (128, 137, 5), (1001, 1008, 0), (64, 64, 1)])
def test_dense_rows_that_are_no_whole_units(quant, M, K, pitch, at):
    torch.manual_seed(M + K)
    x = torch.randn(M * pitch + at, device=DEV).to(BF)[at:].view(M, pitch)[:, :K]
    w4, W = weight(quant, (77, K))
    st, bias = status(), torch.randn(77, device=DEV)
    out = quant.gemm4(x, w4, torch.empty(M, 77, device=DEV), bias=bias, any_rows=True, status=st)
    fine(st)
    Q.check_product(out, x, W[0], bias=bias)


@pytest.mark.parametrize("M", [700, 60000])
def test_a_stack_of_more_groups_than_a_launch_takes(quant, M):
    """In several launches; rows in front of the first group and behind the last stay as they were."""
    G_, N, K = 2500, 24, 72
    torch.manual_seed(M)
    w4, W = weight(quant, (G_, N, K), 32)
    off = torch.cat([torch.tensor([3]), torch.randint(3, M - 2, (G_ - 1,)).sort().values, torch.tensor([M - 2])])
    x, st = torch.randn(M, K, device=DEV).to(BF), status()
    out = quant.gemm4(x, w4, torch.full((M, N), 7.0, device=DEV), group_offsets=off.to(torch.int32).to(DEV), status=st)
    fine(st)
    assert bool((out[:3] == 7).all()) and bool((out[M - 2:] == 7).all())
    group = torch.bucketize(torch.arange(3, M - 2), off[1:], right=True).to(DEV)
    xs = x[3:M - 2].double()
    y, mag = torch.empty(M - 5, N, dtype=torch.float64, device=DEV), torch.empty(M - 5, N, dtype=torch.float64, device=DEV)
    for a in range(0, M - 5, 4096):
        w = W[group[a:a + 4096]]
        y[a:a + 4096], mag[a:a + 4096] = torch.einsum("mk,mnk->mn", xs[a:a + 4096], w), torch.einsum("mk,mnk->mn", xs[a:a + 4096].abs(), w.abs())
    bound = (K / 16 + 80) * 2.0 ** -23 * mag + 2.0 ** -23 * y.abs()
    assert bool(((out[3:M - 2].double() - y).abs() <= bound).all())


def test_a_model_whose_experts_no_tile_divides(quant):
    """Rows between the experts' products of 5,503 elements: too long for the products of few rows, no whole units for the tensor cores."""
    import helpers
    import moe_b200

    config = {**helpers.CONFIG_A, "moe_intermediate_size": 5503, "num_hidden_layers": 2}
    held, same = [moe_b200.random_model(config, seed=3, weights="int4") for _ in range(2)]
    rows = []
    for b in same.blocks:                 # the same numbers in bfloat16
        for p in b.parts():
            for name, w in list(vars(p).items()):
                if isinstance(w, quant.Weight4):
                    setattr(p, name, quant.dequantize(w))
            if hasattr(p, "whole_in_4_bits"):
                p.whole_in_4_bits = False
    for model in (held, same):
        engine = moe_b200.Engine(model, max_tokens=512)
        slots = [engine.new_sequence() for _ in range(2)]
        got = [engine.step(slots, [list(range(20)), list(range(5, 40))], [[19], [34]]).float().clone()]
        got.append(engine.step(slots, [[3], [4]], [[0], [0]]).float().clone())
        model.rt.check()
        rows.append(torch.stack(got))
    far = float((rows[0] - rows[1]).abs().max() / rows[1].abs().max())
    assert far < G.TOL_CUT_BF16, far


# ------------------------------------------------------------------------------------------------ models
def parts_of(model):
    """Every part of every block, those inside others too."""
    found = []

    def add(p):
        found.append(p)
        for _, sub in getattr(p, "subs", []):
            add(sub)

    for b in model.blocks:
        for p in b.parts():
            add(p)
    return found


def held_by(part, quant):
    return {n: w for n, w in vars(part).items() if isinstance(w, quant.Weight4)}


def logits_of(model, prompts, steps=3):
    import moe_b200

    vocab = model.spec.vocab_size
    engine = moe_b200.Engine(model, max_tokens=4096)
    slots = [engine.new_sequence() for _ in prompts]
    got = [engine.step(slots, prompts, [[len(p) - 1] for p in prompts]).float().clone()]
    for i in range(steps):
        got.append(engine.step(slots, [[(7 * i + j) % vocab] for j in range(len(slots))], [[0]] * len(slots)).float().clone())
    model.rt.check()
    return torch.cat(got)




@pytest.mark.parametrize("which", range(len(designs())), ids=[n for n, _ in designs()])
def test_a_model_of_32_bit_weights_is_held_in_4_bits(quant, which, monkeypatch):
    """Quantised from the 32-bit values; against the same model whose matrices are the 4-bit ones' values in bfloat16."""
    import moe_b200
    from moe_b200.parts.base import Part

    _, config = designs()[which]
    held = moe_b200.random_model(config, seed=6, stored_dtype="float32", weights="int4")
    assert any(held_by(p, quant) for p in parts_of(held))
    with monkeypatch.context() as m:
        m.setattr(Part, "hold", lambda self, rt, w, pair=False: quant.dequantize(quant.quantize(w.contiguous(), 64, pair=pair)))
        same = moe_b200.random_model(config, seed=6, stored_dtype="float32")
    gen = torch.Generator().manual_seed(which)
    prompts = [torch.randint(0, held.spec.vocab_size, (n,), generator=gen).tolist() for n in (9, 1, 30)]
    a, b = logits_of(held, prompts), logits_of(same, prompts)
    far = float((a - b).abs().max() / b.abs().max())
    assert far < G.TOL_CUT_BF16, far


@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_a_folder_of_another_float_type_is_held_in_4_bits(quant, dtype, tmp_path, model_dirs):
    """Every matrix is what the quantiser makes of the stored numbers."""
    import moe_b200
    from moe_b200.weights.safetensors_io import write_safetensors
    from moe_b200.weights.store import SafetensorsStore

    d = model_dirs.get("A", "float32", seed=2, std=0.02)
    if dtype == "float16":
        import shutil

        store = SafetensorsStore(d)
        tensors = {n: store.raw(n).to(torch.float16) for n in store.names()}
        d16 = tmp_path / "half"
        d16.mkdir()
        shutil.copy(f"{d}/config.json", d16 / "config.json")
        write_safetensors(str(d16 / "model.safetensors"), tensors)
        d = str(d16)
    store = SafetensorsStore(d)
    model = moe_b200.load_model(d, weights="int4")
    for i, b in enumerate(model.blocks):
        assert {"wqkv", "wo"} <= set(held_by(b.mixer, quant)) and {"w_gu", "w_down", "ws_gu", "ws_down"} <= set(held_by(b.ffn, quant))
        stored = store.raw(f"model.layers.{i}.self_attn.o_proj.weight").float()
        assert torch.equal(quant.dequantize(b.mixer.wo).double().cpu(), Q.plain_values(stored, 64))


def all_designs():
    import importlib

    import helpers

    found = [("qwen " + n, c) for n, c in helpers.CONFIGS.items()]
    for u in ("supevik", "fogapel", "zosipel", "divadra", "ditazen", "kulanex"):
        m = importlib.import_module(u + "_util")
        found += [(f"{u} {n}", m.config_dict(n)) for n in ("mix", "lean", "ones", "wide", "odd") if n in m.CONFIGS]
    return found


# What a part keeps in 16 bits: routers, the narrow products behind a decay's logits (``w1_3``: as three copies), a latent's products a head
IN_16_BITS = {"w_router", "w_router3", "w1_3", "w_low1", "w_low2", "w_qc", "w_cv"}


@pytest.mark.parametrize("which", range(len(all_designs())), ids=[n for n, _ in all_designs()])
def test_the_matrices_of_a_model_are_held_in_4_bits(quant, which, monkeypatch):
    """All that the parts multiply by, and prompts so long that routers, norms and branches take their forms of many tokens, against the same model whose
    matrices are the 4-bit ones' values in bfloat16."""
    import moe_b200
    from moe_b200.parts.base import Part

    _, config = all_designs()[which]
    held = moe_b200.random_model(config, seed=8, weights="int4")
    for p in parts_of(held):
        assert p.category not in ("mixer", "ffn") or hasattr(p, "subs") or held_by(p, quant), p.kind
        left = {n for n, w in vars(p).items() if isinstance(w, torch.Tensor) and w.dtype == BF and w.dim() > 1}
        assert left <= IN_16_BITS, (p.kind, left)
    with monkeypatch.context() as m:
        m.setattr(Part, "hold", lambda self, rt, w, pair=False: quant.dequantize(quant.quantize(w.contiguous(), 64, pair=pair)))
        same = moe_b200.random_model(config, seed=8)
    gen = torch.Generator().manual_seed(which)
    prompts = [torch.randint(0, held.spec.vocab_size, (n,), generator=gen).tolist() for n in (9, 290, 1)]
    a, b = logits_of(held, prompts), logits_of(same, prompts)
    far = float((a - b).abs().max() / b.abs().max())
    assert far < G.TOL_CUT_BF16, far


@pytest.mark.parametrize("which", range(len(all_designs())), ids=[n for n, _ in all_designs()])
def test_the_bytes_of_a_step_are_those_that_are_held(quant, which):
    """Elements in 4 bits at theirs, all others at 16; so many tokens that every expert is read, and one."""
    import moe_b200
    from moe_b200 import cli

    _, config = all_designs()[which]
    group = (32, 64, 128)[which % 3]
    model = moe_b200.random_model(config, seed=8, weights="int4", weight_group=group)
    each = 0.5 + 2 / group
    for p in parts_of(model):
        if hasattr(p, "subs"):
            continue
        held = held_by(p, quant)
        full = p.step_elements(1 << 20)
        # (up to seven rows of zeros a matrix are held beside the model's own, and differential attention lays some rows out twice: what a step counts are the model's)
        in4 = min(full, sum(w.G * w.N * w.K for w in held.values()))
        room = 2 * sum(7 * w.K for w in held.values())
        assert abs(p.step_bytes(1 << 20, model.rt) - ((full - in4) * 2 + in4 * each)) <= room, p.kind
        if p.kind == "routed_experts":
            experts = p.w_gu.N * p.w_gu.K * p.E + p.w_down.N * p.w_down.K * p.E
            want = (full - in4) * 2 + (in4 - experts) * each + experts * each * p.k / p.E
            assert abs(p.step_bytes(1, model.rt) - want) <= 1e-9 * want
    rest, _ = cli.step_bytes(model, [10])
    blocks = sum(p.step_bytes(1, model.rt) for e in model.spec.schedule for p in model.blocks[e.layer].parts())
    assert rest > blocks > 0


@pytest.mark.parametrize("change", [dict(hidden_size=6400, num_experts=300), dict(num_experts=1100), dict(num_experts=300, num_experts_per_tok=20)])
def test_a_layer_that_its_kernels_do_not_take_is_routed_once(quant, change, monkeypatch):
    """Too wide, too many experts, or too many picks for the layer of few tokens: the products take it one by one, from the picks of one router."""
    import helpers
    import moe_b200
    from moe_b200.ops import core

    config = {**helpers.CONFIG_A, **change}
    model = moe_b200.random_model(config, seed=4, weights="int4")
    ffn = model.blocks[0].ffn
    tokens = 8
    assert not quant.takes_experts(tokens, ffn.k, ffn.w_gu) and quant.takes_experts(1, 2, quant.quantize(torch.ones(4, 32, 64, device=DEV), pair=True))
    x = torch.randn(tokens, model.spec.hidden_size, device=DEV)

    class H:
        act, f32, split = x.to(BF), x, None

    calls, rt = [], model.rt
    for name in ("router", "route_dispatch", "router_topk"):
        real = getattr(core, name)
        monkeypatch.setattr(core, name, lambda *a, _real=real, _name=name, **kw: (calls.append(_name), _real(*a, **kw))[1])
    out = ffn.forward(rt, H, type("B", (), dict(seq_of_token=None))())
    rt.check()
    assert len(calls) == 1, calls
    topk_idx, topk_w, sg = ffn.route(rt, H, type("B", (), dict(seq_of_token=None))())
    GU, D = [quant.dequantize(w).double() for w in (ffn.w_gu, ffn.w_down)]
    SGU, SD = [quant.dequantize(w).double() for w in (ffn.ws_gu, ffn.ws_down)]
    # (between the two products bfloat16 rows: 2^-8 of each term)
    mag, want = torch.zeros_like(out, dtype=torch.float64), torch.zeros_like(out, dtype=torch.float64)
    for t in range(tokens):
        pairs = [(GU[e], D[e], float(f)) for e, f in zip(topk_idx[t].tolist(), topk_w[t].tolist())] + [(SGU, SD, 1.0 if sg is None else float(sg[t]))]
        for gu, d, f in pairs:
            a = Q.gated("silu", *(gu @ H.act[t].double()).chunk(2))
            want[t] += f * (d @ a)
            mag[t] += f * (d.abs() @ a.abs())
    assert bool(((out.double() - want).abs() <= 2.0 ** -7 * mag + 1e-30).all())


# ------------------------------------------------------------------------------------------------ the gate's function
@pytest.mark.parametrize("M,groups", [(4, 0), (20, 0), (64, 0), (300, 0), (200, 4), (1200, 4)])
def test_gates_far_from_zero(quant, M, groups):
    """Every form at gates down to -100 and up to 100 whose sums are exact (one element of x is not zero), so that only silu(g) u is off.  Few rows: an exponential of 2 ulp
    and three roundings, below 2^-20 of it; the divisor is infinite from -88.73 on, and the zero that is left off by 88.73 e^-88.73 = 2.6e-37 < 2^-121 at most.  The tensor
    cores' epilogue: an exponential of 2 + 1.2 |g| ulp, a quotient of 2, two roundings, (5 + 1.2 |g|) 2^-23; zero from a divisor of 2^126 on, 88 2^-126 < 2^-119."""
    K, half = 64, 512
    gen = torch.Generator(device=DEV)
    gen.manual_seed(M)
    G_ = max(groups, 1)
    w = torch.zeros(G_, 2 * half, K, device=DEV)
    w[:, :half, 9] = torch.linspace(-7, 7, half, device=DEV).round()              # whole numbers up to 7: held as they are
    w[:, half:, 9] = torch.randint(1, 8, (G_, half), device=DEV, generator=gen).float()
    w[:, :, 20] = 7                       # (the scale of every group of 64 is 1; x is zero there)
    shape = w.shape if groups else w.shape[1:]
    w4 = quant.quantize(w.reshape(shape), pair=True)
    assert torch.equal(quant.dequantize(w4).float().reshape(w.shape), w)
    x = torch.zeros(M, K, dtype=BF, device=DEV)
    x[:, 9] = torch.linspace(0.01, 14.3, M, device=DEV).to(BF)
    off = torch.arange(0, M + 1, M // groups, dtype=torch.int32, device=DEV) if groups else None
    st, out = status(), torch.empty(M, half, device=DEV)
    quant.gemm4(x, w4, out, swiglu=True, group_offsets=off, status=st)
    fine(st)
    each = w.double().repeat_interleave(M // G_, dim=0) if groups else w.double().expand(M, -1, -1)
    g, u = [x[:, 9].double().unsqueeze(1) * each[:, h * half:(h + 1) * half, 9] for h in (0, 1)]
    y = g * torch.sigmoid(g) * u
    assert float(g.min()) < -99 and float(g.max()) > 99
    few = M <= quant.FEW_ROWS
    far = (out.double() - y).abs()
    room = 2.0 ** -20 * y.abs() + u.abs() * 2.0 ** -121 if few else (5 + 1.2 * g.abs()) * 2.0 ** -23 * y.abs() + u.abs() * 2.0 ** -119
    assert bool((far <= room).all()), float((far / room).max())


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_folder_with_a_weight_that_is_no_number_is_refused_in_a_line(quant, bad, tmp_path, model_dirs, capsys):
    import shutil

    import moe_b200
    from moe_b200 import cli
    from moe_b200.ops import core
    from moe_b200.weights.safetensors_io import write_safetensors
    from moe_b200.weights.store import SafetensorsStore

    d = model_dirs.get("A", "bfloat16", seed=2, std=0.02)
    store = SafetensorsStore(d)
    tensors = {n: store.raw(n).clone() for n in store.names()}
    tensors["model.layers.1.self_attn.o_proj.weight"][3, 5] = bad
    shutil.copy(f"{d}/config.json", tmp_path / "config.json")
    write_safetensors(str(tmp_path / "model.safetensors"), tensors)
    with pytest.raises(core.KernelError, match="not finite"):
        moe_b200.load_model(str(tmp_path), weights="int4")
    with pytest.raises(SystemExit):
        cli.main(["run", str(tmp_path), "--ids", "5", "-n", "1", "--weights", "int4"])
    assert "not finite" in capsys.readouterr().err


def test_a_status_without_room_for_what_is_reported_is_refused(quant):
    from moe_b200.ops import core

    (w4, _), (pair, _), (down, _) = weight(quant, (32, 64)), weight(quant, (2, 32, 64), pair=True), weight(quant, (2, 64, 16))
    x, idx, w = torch.zeros(2, 64, dtype=BF, device=DEV), torch.zeros(2, 1, dtype=torch.int32, device=DEV), torch.ones(2, 1, device=DEV)
    for n in (0, 1):
        small = torch.zeros(n, dtype=torch.int32, device=DEV)
        for call in (lambda: quant.quantize(torch.ones(32, 64, device=DEV), status=small), lambda: quant.gemm4(x, w4, torch.empty(2, 32, device=DEV), status=small),
                     lambda: quant.experts4(x, idx, w, pair, down, torch.empty(2, 64, device=DEV), status=small)):
            with pytest.raises(core.KernelError, match="status"):
                call()


@pytest.mark.parametrize("H", [64, 100, 133])
def test_a_gather_index_outside_its_tensor_is_reported_whatever_the_width(quant, H):
    """Rows of no whole 16-byte units too: the other rows are what they are, and the context lives on."""
    from moe_b200.ops import core
    from moe_b200.ops.linear import grouped_swiglu_linear
    from moe_b200.parts.base import Runtime

    torch.manual_seed(H)
    rt = Runtime(DEV, BF, 64)
    w4, W = weight(quant, (3, 48, H), pair=True)
    a = torch.randn(7, H, device=DEV).to(BF)
    rows = torch.tensor([3, 0, 6, 6, 1, 2, 5, 4, 0], dtype=torch.int32, device=DEV)
    off = torch.tensor([0, 4, 4, 9], dtype=torch.int32, device=DEV)
    for bad in (None, -1, 7, 1 << 30):
        at = rows.clone()
        if bad is not None:
            at[5] = bad
        out = grouped_swiglu_linear(rt, a, w4, off, at, 9)
        if bad is None:
            rt.check()
        else:
            with pytest.raises(core.KernelError, match="gather"):
                rt.check()
        for g, (lo, hi) in enumerate(((0, 4), (4, 4), (4, 9))):
            keep = [i for i in range(lo, hi) if bad is None or i != 5]
            if keep:
                Q.check_product(out[keep], a[rows[keep].long()], W[g], swiglu=True)


def test_the_command_line_times_a_model_with_4_bit_weights(model_dirs, capsys):
    from moe_b200 import cli

    d = model_dirs.get("D", "bfloat16", seed=1, std=0.02)
    said = []
    for more in ([], ["--weights", "int4", "--weight-group", "128"]):
        assert cli.main(["bench", d, "--tokens", "4", "--prompt-len", "9", "--batch", "3", *more]) == 0
        said.append(capsys.readouterr().out)
    assert all("roofline" in s and "tok/s" in s for s in said)
    read = [s.split("roofline ")[1].split(" weights")[0] for s in said]
    assert read[0] != read[1], read
