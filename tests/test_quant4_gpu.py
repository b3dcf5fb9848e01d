"""Weights held in 4 bits on the GPU: the quantiser, dense and grouped products at the sizes where their forms meet, a layer of experts of few tokens,
streams and graphs, waits that run out, and models that hold their matrices so."""
from __future__ import annotations

import ctypes

import pytest
import torch

import gpu_util as G
import helpers
import quant4_util as Q

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


@pytest.fixture(scope="module")
def quant():
    from moe_b200.ops import quant

    quant.lib()
    return quant


def status():
    from moe_b200.ops import core

    return core.new_status(DEV)


def fine(st):
    torch.cuda.synchronize()
    assert int(st[0]) == 0, st.tolist()


def weight(quant, shape, group=64, pair=False, std=None, seed=0):
    """(Weight4, its values in float64 [G, N, K])"""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    w = torch.randn(*shape, device=DEV, generator=gen) * (std or shape[-1] ** -0.5)
    w4 = quant.quantize(w.to(BF), group, pair=pair)
    v = quant.dequantize(w4).double()
    return w4, v if v.dim() == 3 else v.unsqueeze(0)


# ------------------------------------------------------------------------------------------------ quantiser
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("shape,pair", [((1, 1), False), ((16, 64), False), ((33, 130), False), ((3, 50, 333), False), ((2, 34, 96), True), ((62, 1000), True),
                                        ((32, 128), False), ((3, 48, 384), False), ((2, 64, 1152), True)])
def test_values_are_the_plain_ones(quant, shape, pair, dtype, group):
    torch.manual_seed(shape[-1] + group)
    kinds = {
        "normal": lambda: torch.randn(*shape, device=DEV) * 0.02,
        # quotients that are half a step, and maxima whose seventh is a border of five bits
        "ties": lambda: torch.randint(-255, 256, shape, device=DEV).float() * 2.0 ** -7,
        "halves": lambda: torch.randint(-15, 16, shape, device=DEV).float() / 2,
        "tiny": lambda: torch.randn(*shape, device=DEV) * 1e-37,
        "huge": lambda: torch.randn(*shape, device=DEV).clamp(-3, 3) * 1e38,
        "zeros": lambda: torch.randn(*shape, device=DEV) * (torch.rand(*shape, device=DEV) < 0.01),
    }
    for name, make in kinds.items():
        w = make().to(dtype)
        st = status()
        w4 = quant.quantize(w, group, pair=pair, status=st)
        got = quant.dequantize(w4)
        fine(st)
        assert torch.equal(got.double(), Q.plain_values(w, group)), name
        assert torch.equal(Q.values_by_place(w4).reshape(shape), got.double().cpu()), name


def test_what_is_no_number_is_reported_and_stays_in_its_group(quant):
    from moe_b200.ops import core

    w = torch.randn(20, 128, device=DEV)
    w[3, 5], w[18, 70] = float("inf"), float("nan")
    st = status()
    v = quant.dequantize(quant.quantize(w, 64, status=st))
    with pytest.raises(core.KernelError, match="not finite"):
        core.check_status(st)
    bad = torch.zeros_like(v, dtype=torch.bool)
    bad[3, :64], bad[18, 64:] = True, True
    assert torch.equal(v.isnan(), bad)
    clean = torch.where(bad, 0.0, w)
    assert torch.equal(v[~bad].double(), Q.plain_values(clean, 64)[~bad])


@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_weights_that_begin_anywhere(quant, dtype):
    room = torch.randn(3 * 48 * 128 + 1, device=DEV).to(dtype)
    for at in (0, 1):
        w = room[at:at + 3 * 48 * 128].view(3, 48, 128)
        back = torch.full((3 * 48 * 128 + 2,), 7.0, dtype=BF, device=DEV)
        got = quant.dequantize(quant.quantize(w), back[at:at + 3 * 48 * 128].view(3, 48, 128))
        assert torch.equal(got.double(), Q.plain_values(w, 64))
        assert bool((back[:at] == 7).all()) and bool((back[at + 3 * 48 * 128:] == 7).all())


def test_more_matrices_than_a_grid_has_blocks(quant):
    w = torch.randn(66000, 2, 8, device=DEV)
    assert torch.equal(quant.dequantize(quant.quantize(w, 32, pair=True)).double(), Q.plain_values(w, 32))


# ------------------------------------------------------------------------------------------------ dense products
@pytest.mark.parametrize("K", [1, 5, 64, 70, 200, 1411, 2048])
@pytest.mark.parametrize("M", [1, 3, 8, 9, 16, 17, 20, 24])
def test_few_rows(quant, M, K):
    torch.manual_seed(M * K)
    for i, (N, group, dtype) in enumerate([(1, 64, torch.float32), (50, 32, BF), (257, 128, torch.float32)]):
        w4, W = weight(quant, (N, K), group, seed=i)
        x, st = torch.randn(M, K, device=DEV).to(BF), status()
        bias = torch.randn(N, device=DEV) if i else None
        out = quant.gemm4(x, w4, torch.full((M, N), float("nan"), dtype=dtype, device=DEV), bias=bias, status=st)
        fine(st)
        Q.check_product(out, x, W[0], bias=bias)


@pytest.mark.parametrize("M", [17, 31, 64, 65, 113, 128, 200, 256, 257, 300, 515])
def test_more_rows(quant, M):
    torch.manual_seed(M)
    for i, (N, K, group, dtype) in enumerate([(100, 72, 32, torch.float32), (300, 1416, 64, BF), (2048, 640, 128, torch.float32), (131, 333, 64, BF)]):
        w4, W = weight(quant, (N, K), group, seed=i)
        x, st = torch.randn(M, K, device=DEV).to(BF), status()
        bias = torch.randn(N, device=DEV) if i % 2 else None
        out = quant.gemm4(x, w4, torch.full((M, N), float("nan"), dtype=dtype, device=DEV), bias=bias, status=st)
        fine(st)
        Q.check_product(out, x, W[0], bias=bias)


@pytest.mark.parametrize("M", [1, 8, 11, 23, 40, 130, 300])
@pytest.mark.parametrize("act,param", [("silu", 0.0), ("gelu_tanh", 0.0), ("clamped_sigmoid", 1.5)])
def test_gated_pairs(quant, M, act, param):
    torch.manual_seed(M)
    for i, (I, K, group, dtype) in enumerate([(1, 64, 64, BF), (43, 200, 32, torch.float32), (200, 1000, 128, BF)]):
        w4, W = weight(quant, (2 * I, K), group, pair=True, seed=i)
        x, st = torch.randn(M, K, device=DEV).to(BF), status()
        out = quant.gemm4(x, w4, torch.full((M, I), float("nan"), dtype=dtype, device=DEV), swiglu=True, act=act, act_param=param, status=st)
        fine(st)
        Q.check_product(out, x, W[0], swiglu=True, act=act, param=param)


@pytest.mark.parametrize("M", [5, 50])
@pytest.mark.parametrize("act", ["relu2", "gelu"])
def test_activations_of_an_ungated_product(quant, M, act):
    torch.manual_seed(M)
    w4, W = weight(quant, (90, 264))
    x, st = torch.randn(M, 264, device=DEV).to(BF), status()
    out = quant.gemm4(x, w4, torch.empty(M, 90, dtype=BF, device=DEV), act=act, status=st)
    fine(st)
    Q.check_product(out, x, W[0], act=act)


@pytest.mark.parametrize("M,N,K", [(1, 20000, 200), (7, 20000, 264), (12, 20000, 136), (16, 40000, 72), (8, 19000, 7040), (17, 7200, 1000), (24, 20000, 333),
                                   (19, 7200, 5000)])
def test_so_many_features_that_the_weights_are_streamed(quant, M, N, K):
    torch.manual_seed(K)
    for pair in (False, True):
        w4, W = weight(quant, (N, K), 32 if K == 72 else 64, pair=pair)
        x, st = torch.randn(M, K, device=DEV).to(BF), status()
        out = quant.gemm4(x, w4, torch.empty(M, N // 2 if pair else N, device=DEV), swiglu=pair, status=st)
        fine(st)
        Q.check_product(out, x, W[0], swiglu=pair)


@pytest.mark.parametrize("M", [4, 90])
def test_columns_of_wider_matrices(quant, M):
    """Pitches of x and out that are no row's length, also such that no wide load is aligned; what lies beside stays as it was."""
    torch.manual_seed(M)
    for K, pitch, at in ((128, 136, 8), (96, 101, 3), (64, 200, 120)):
        w4, W = weight(quant, (77, K))
        wide, st = torch.randn(M, pitch, device=DEV).to(BF), status()
        x = wide[:, at:at + K] if at + K <= pitch else wide[:, pitch - K:]
        big = torch.full((M, 90), 7.0, device=DEV)
        quant.gemm4(x, w4, big[:, 5:82], status=st)
        fine(st)
        Q.check_product(big[:, 5:82], x, W[0])
        assert bool((big[:, :5] == 7).all()) and bool((big[:, 82:] == 7).all())


def test_no_rows(quant):
    w4, _ = weight(quant, (20, 64))
    assert quant.gemm4(torch.empty(0, 64, dtype=BF, device=DEV), w4, torch.empty(0, 20, device=DEV)).shape == (0, 20)


def test_a_row_that_is_no_number_keeps_to_itself(quant):
    for M in (6, 70):
        w4, W = weight(quant, (100, 192))
        x = torch.randn(M, 192, device=DEV).to(BF)
        x[2], x[4, 7] = float("nan"), float("inf")
        out = quant.gemm4(x, w4, torch.empty(M, 100, device=DEV), status=status())
        rest = [i for i in range(M) if i not in (2, 4)]
        assert bool(out[2].isnan().all()) and not bool(out[4].isfinite().all())
        Q.check_product(out[rest], x[rest], W[0])


def test_a_product_right_behind_the_quantiser_of_its_weight(quant):
    """Products ask for their weights before they wait for what is in front of them: the quantiser lets them in when all is written."""
    torch.manual_seed(2)
    ws = [torch.randn(2048, 1024, device=DEV).to(BF) * 2.0 ** -5 for _ in range(4)]
    for M in (1, 40):
        x, outs = torch.randn(M, 1024, device=DEV).to(BF), [torch.empty(M, 2048, device=DEV) for _ in ws]
        for _ in range(20):
            for w, out in zip(ws, outs):
                quant.gemm4(x, quant.quantize(w), out)
        for w, out in zip(ws, outs):
            Q.check_product(out, x, quant.dequantize(quant.quantize(w)))


# ------------------------------------------------------------------------------------------------ grouped products
@pytest.mark.parametrize("rows", [[0, 3, 0, 0, 8, 9, 1, 0], [0] * 8, [17, 0, 16, 33, 1, 0, 8, 25], [17, 0, 40, 16, 1, 0, 100, 33], [300, 0, 1, 0, 0, 257, 64, 5], [0, 0, 0, 0, 0, 0, 0, 1]])
@pytest.mark.parametrize("pair", [False, True])
def test_groups(quant, rows, pair):
    """Groups with and without rows, rows in front of the first group and behind the last: those stay as they were."""
    torch.manual_seed(sum(rows))
    for N, K, group, before in ((70, 136, 64, 0), (48, 1000, 32, 5)):
        w4, W = weight(quant, (len(rows), N, K), group, pair=pair)
        off = [before]
        for r in rows:
            off.append(off[-1] + r)
        M = off[-1] + 3
        x, st = torch.randn(M, K, device=DEV).to(BF), status()
        out = torch.full((M, N // 2 if pair else N), 7.0, device=DEV)
        quant.gemm4(x, w4, out, swiglu=pair, group_offsets=torch.tensor(off, dtype=torch.int32, device=DEV), status=st)
        fine(st)
        for g, r in enumerate(rows):
            if r:
                Q.check_product(out[off[g]:off[g + 1]], x[off[g]:off[g + 1]], W[g], swiglu=pair)
        assert bool((out[:before] == 7).all()) and bool((out[off[-1]:] == 7).all())


def test_offsets_out_of_range_touch_nothing_else(quant):
    w4, W = weight(quant, (4, 40, 64))
    for M in (20, 200):
        x, guard = torch.randn(M, 64, device=DEV).to(BF), torch.full((M + 64, 40), 7.0, device=DEV)
        quant.gemm4(x, w4, guard[32:32 + M], group_offsets=torch.tensor([-5, 3, 2, M + 9, M + 90], dtype=torch.int32, device=DEV), status=status())
        torch.cuda.synchronize()
        assert bool((guard[:32] == 7).all()) and bool((guard[32 + M:] == 7).all())


@pytest.mark.parametrize("rows", [[40, 0, 17, 64, 1, 33, 128, 20], [129, 70, 128, 0, 90, 200, 100, 99], [150, 90, 200, 128, 110, 90, 140, 130]])
@pytest.mark.parametrize("N,dtype", [(512, torch.float32), (300, BF), (72, BF), (511, torch.float32)])
def test_groups_of_many_rows(quant, rows, N, dtype):
    """Either tile of the tensor-core form, whole and not, rows of the output in whole units and not; with a bias and an activation."""
    torch.manual_seed(N + len(rows))
    off = [0]
    for r in rows:
        off.append(off[-1] + r)
    M, K, offsets = off[-1], 328, torch.tensor(off, dtype=torch.int32, device=DEV)
    x, bias = torch.randn(M, K, device=DEV).to(BF), torch.randn(N, device=DEV)
    w4, W = weight(quant, (len(rows), N, K))
    pair4, P = weight(quant, (len(rows), 2 * N, K), 32, pair=True, seed=1)
    for odd in (0, 3):
        big = torch.full((M, N + 8 + odd), 7.0, dtype=dtype, device=DEV)
        out = big[:, odd:N + odd]
        for kw in (dict(bias=bias), dict(bias=bias, act="relu2"), dict(swiglu=True)):
            st = status()
            quant.gemm4(x, pair4 if "swiglu" in kw else w4, out, group_offsets=offsets, status=st, **kw)
            fine(st)
            for g, r in enumerate(rows):
                if r:
                    Q.check_product(out[off[g]:off[g + 1]], x[off[g]:off[g + 1]], P[g] if "swiglu" in kw else W[g], **kw)
            assert bool((big[:, :odd] == 7).all()) and bool((big[:, N + odd:] == 7).all())


def test_offsets_that_go_up_and_down_touch_nothing_else(quant):
    w4, W = weight(quant, (6, 40, 64))
    for M in (90, 700):
        x, guard = torch.randn(M, 64, device=DEV).to(BF), torch.full((M + 64, 40), 7.0, device=DEV)
        quant.gemm4(x, w4, guard[32:32 + M], group_offsets=torch.tensor([0, M, 0, M, 0, M, 1], dtype=torch.int32, device=DEV), status=status())
        torch.cuda.synchronize()
        assert bool((guard[:32] == 7).all()) and bool((guard[32 + M:] == 7).all())


@pytest.mark.parametrize("pitch", [0, 3, 8004])
def test_one_row_whatever_its_pitch(quant, pitch):
    """torch may say anything of the pitch of a single row."""
    (stack, W), off = weight(quant, (2, 24, 8000)), torch.tensor([0, 0, 1], dtype=torch.int32, device=DEV)
    row = torch.randn(8000, device=DEV).to(BF)
    x, room = row.as_strided((1, 8000), (pitch, 1)), torch.empty(24, device=DEV)
    quant.gemm4(x, stack, room.as_strided((1, 24), (pitch, 1)), group_offsets=off)
    Q.check_product(room.view(1, 24), row.view(1, -1), W[1])


@pytest.mark.parametrize("G_,M", [(1, 40), (1000, 900), (300, 6000)])
def test_one_group_and_very_many(quant, G_, M):
    torch.manual_seed(M)
    w4, W = weight(quant, (G_, 24, 72), 32)
    cuts = torch.randint(0, M + 1, (G_ - 1,)).sort().values.tolist()
    off = [0, *cuts, M]
    x, st = torch.randn(M, 72, device=DEV).to(BF), status()
    out = quant.gemm4(x, w4, torch.empty(M, 24, device=DEV), group_offsets=torch.tensor(off, dtype=torch.int32, device=DEV), status=st)
    fine(st)
    group = torch.bucketize(torch.arange(M), torch.tensor(off[1:]), right=True).to(DEV)
    y = torch.einsum("mk,mnk->mn", x.double(), W[group])
    bound = (72 / 16 + 80) * 2.0 ** -23 * torch.einsum("mk,mnk->mn", x.double().abs(), W[group].abs()) + 2.0 ** -23 * y.abs()
    assert bool(((out.double() - y).abs() <= bound).all())


# ------------------------------------------------------------------------------------------------ a layer of experts
def plain_layer(x, idx, w, GU, D, shared=None, gate=None):
    """Float64 (values, magnitudes of what was added up)."""
    x = x.double()
    T, H = x.shape
    y, size = torch.zeros(T, H, dtype=torch.float64, device=x.device), torch.zeros(T, H, dtype=torch.float64, device=x.device)

    def one(t, gu, d, f):
        half = gu.shape[0] // 2
        g, u = gu[:half] @ x[t], gu[half:] @ x[t]
        a = g * torch.sigmoid(g) * u
        K = x.shape[1]
        # what the 32-bit sums of the first product leave in a, as in check_product, and the two terms' rounding
        dg, du = [(K / 16 + 80) * 2.0 ** -23 * (m.abs() @ x[t].abs()) for m in (gu[:half], gu[half:])]
        da = 1.13 * dg * (u.abs() + du) + ((g * torch.sigmoid(g)).abs() + 1.13 * dg) * du + (2.0 ** -20 + 2.0 ** -16) * a.abs()
        y[t] += f * (d @ a)
        size[t] += abs(f) * (d.abs() @ ((d.shape[1] / 16 + 80) * 2.0 ** -23 * a.abs() + da))

    for t in range(T):
        for j in range(idx.shape[1]):
            e = int(idx[t, j])
            if 0 <= e < GU.shape[0]:
                one(t, GU[e], D[e], float(w[t, j]))
        if shared is not None:
            one(t, shared[0], shared[1], 1.0 if gate is None else float(gate[t]))
    return y, size + 64 * 2.0 ** -23 * y.abs()


def check_layer(got, y, size):
    off = size + Q.out_step(y, got.dtype) * 1.01
    far = (got.double() - y).abs()
    assert bool((far <= off).all()), f"off by {float((far / off).max()):.2f} of what rounding allows"


LAYERS = [  # T, H, E, top, size, shared, gate, group
    (1, 64, 1, 1, 16, 0, False, 32), (1, 2048, 60, 4, 200, 96, True, 64), (3, 264, 6, 2, 56, 88, True, 32), (5, 136, 300, 5, 40, 72, False, 128),
    (8, 72, 16, 2, 193, 57, True, 64), (8, 1000, 9, 8, 33, 0, False, 128), (7, 100, 1024, 16, 31, 500, True, 32), (4, 70, 5, 3, 64, 33, True, 64),
    (2, 333, 8, 2, 128, 64, True, 32), (8, 512, 2, 2, 704, 1408, True, 64)]


@pytest.mark.parametrize("case", LAYERS)
@pytest.mark.parametrize("dtype", [torch.float32, BF])
def test_a_layer_of_experts(quant, case, dtype):
    T, H, E, top, size, shared, gated, group = case
    torch.manual_seed(T * H)
    gu, GU = weight(quant, (E, 2 * size, H), group, pair=True)
    d, D = weight(quant, (E, H, size), group, seed=1)
    more, plain = {}, {}
    if shared:
        (sgu, SGU), (sd, SD) = weight(quant, (2 * shared, H), group, pair=True, seed=2), weight(quant, (H, shared), group, seed=3)
        more, plain = dict(shared_gate_up=sgu, shared_down=sd), dict(shared=(SGU[0], SD[0]))
        if gated:
            more["shared_gate"] = plain["gate"] = torch.rand(T, device=DEV)
    x, st = torch.randn(T, H, device=DEV).to(BF), status()
    w, idx = torch.rand(T, E, device=DEV).topk(min(top, E), dim=1)
    idx = idx.to(torch.int32).contiguous()
    big = torch.full((T, H + 3), 7.0, dtype=dtype, device=DEV)
    assert quant.experts4(x, idx, w.contiguous(), gu, d, big[:, :H], status=st, **more)
    fine(st)
    check_layer(big[:, :H], *plain_layer(x, idx, w, GU, D, **plain))
    assert bool((big[:, H:] == 7).all())


def test_picks_that_are_none_twice_the_same_or_no_experts(quant):
    T, H, E, top, size, shared = 6, 136, 7, 3, 50, 40
    torch.manual_seed(3)
    (gu, GU), (d, D) = weight(quant, (E, 2 * size, H), pair=True), weight(quant, (E, H, size), seed=1)
    (sgu, SGU), (sd, SD) = weight(quant, (2 * shared, H), pair=True, seed=2), weight(quant, (H, shared), seed=3)
    x, gate = torch.randn(T, H, device=DEV).to(BF), torch.rand(T, device=DEV)
    gate[5] = 0.0
    idx = torch.tensor([[0, 6, 3], [-1, -1, -1], [2, 2, 2], [4, -1, 4], [-1, 5, 1], [-1, -1, -1]], dtype=torch.int32, device=DEV)
    w = torch.rand(T, top, device=DEV)
    for with_shared in (True, False):
        more = dict(shared_gate_up=sgu, shared_down=sd, shared_gate=gate) if with_shared else {}
        st, out = status(), torch.full((T, H), float("nan"), device=DEV)
        assert quant.experts4(x, idx, w, gu, d, out, status=st, **more)
        fine(st)
        check_layer(out, *plain_layer(x, idx, w, GU, D, **(dict(shared=(SGU[0], SD[0]), gate=gate) if with_shared else {})))
        assert not bool(out[5].any())
    # every pick none, and no shared expert: zeros
    st, out = status(), torch.full((T, H), float("nan"), device=DEV)
    assert quant.experts4(x, torch.full_like(idx, -1), w, gu, d, out, status=st)
    fine(st)
    assert not bool(out.any())
    # an index outside the experts is reported and taken for none
    from moe_b200.ops import core

    idx[0, 1], idx[4, 0] = 7, -2
    assert quant.experts4(x, idx, w, gu, d, out, status=st)
    with pytest.raises(core.KernelError, match="expert"):
        core.check_status(st)
    check_layer(out, *plain_layer(x, idx, w, GU, D))


def test_a_token_that_is_no_number_keeps_to_itself(quant):
    T, H, E, size = 5, 128, 4, 48
    torch.manual_seed(4)
    (gu, GU), (d, D) = weight(quant, (E, 2 * size, H), pair=True), weight(quant, (E, H, size), seed=1)
    x = torch.randn(T, H, device=DEV).to(BF)
    x[1], x[3, 9] = float("nan"), float("inf")
    idx = torch.tensor([[0, 1], [0, 2], [1, 3], [2, 0], [3, 2]], dtype=torch.int32, device=DEV)
    w, out = torch.rand(T, 2, device=DEV), torch.empty(T, H, device=DEV)
    assert quant.experts4(x, idx, w, gu, d, out)
    rest = [0, 2, 4]
    assert bool(out[1].isnan().all()) and bool(out[3].isnan().any())
    y, size_ = plain_layer(x[rest], idx[rest], w[rest], GU, D)
    check_layer(out[rest], y, size_)


def test_an_expert_that_is_no_number_stays_with_the_tokens_that_picked_it(quant):
    T, H, E, size = 4, 128, 5, 80
    torch.manual_seed(6)
    for where in ("gate", "down"):
        wu, wd = torch.randn(E, 2 * size, H, device=DEV) * H ** -0.5, torch.randn(E, H, size, device=DEV) * size ** -0.5
        (wu if where == "gate" else wd)[2, 3, 5] = float("nan")
        gu, d = quant.quantize(wu.to(BF), pair=True), quant.quantize(wd.to(BF))
        x = torch.randn(T, H, device=DEV).to(BF)
        idx = torch.tensor([[0, 1], [2, 0], [3, 1], [4, 3]], dtype=torch.int32, device=DEV)
        w, out = torch.rand(T, 2, device=DEV), torch.empty(T, H, device=DEV)
        assert quant.experts4(x, idx, w, gu, d, out)
        rest = [0, 2, 3]
        assert bool(out[1, 3].isnan())
        y, size_ = plain_layer(x[rest], idx[rest], w[rest], quant.dequantize(gu).double().nan_to_num(), quant.dequantize(d).double().nan_to_num())
        check_layer(out[rest], y, size_)


def test_what_a_layer_does_not_take(quant):
    from moe_b200.ops import core

    (gu, _), (d, _) = weight(quant, (4, 32, 64), pair=True), weight(quant, (4, 64, 16))
    idx, w = torch.zeros(9, 2, dtype=torch.int32, device=DEV), torch.zeros(9, 2, device=DEV)
    out = torch.full((9, 64), 7.0, device=DEV)
    assert not quant.experts4(torch.zeros(9, 64, dtype=BF, device=DEV), idx, w, gu, d, out)
    assert not quant.experts4(torch.zeros(8, 64, dtype=BF, device=DEV), idx[:1].repeat(8, 9), w[:1].repeat(8, 9), gu, d, out[:8])
    assert bool((out == 7).all())
    x = torch.zeros(2, 64, dtype=BF, device=DEV)
    ok = dict(topk_idx=idx[:2], topk_w=w[:2], gate_up=gu, down=d, out=out[:2])
    for bad in (dict(topk_idx=idx[:3]), dict(topk_idx=idx[:2].long()), dict(topk_w=w[:2].double()), dict(gate_up=d), dict(down=gu), dict(out=out[:3]),
                dict(shared_gate=w[:2, 0].contiguous()), dict(shared_down=weight(quant, (64, 16))[0]), dict(down=weight(quant, (4, 64, 16), 32)[0]),
                dict(status=torch.zeros(4, dtype=torch.int32)), dict(topk_idx=idx[:2, :0], topk_w=w[:2, :0])):
        with pytest.raises(core.KernelError):
            quant.experts4(x, **{**ok, **bad})


def test_rows_that_shared_memory_does_not_hold(quant):
    """A layer so wide is left to the products one by one; a stack so long goes to the tensor core, or is refused where its rows are no whole units."""
    from moe_b200.ops import core

    (gu, _), (d, _) = weight(quant, (2, 32, 8000), 128, pair=True), weight(quant, (2, 8000, 16), 128)
    idx, w = torch.zeros(2, 1, dtype=torch.int32, device=DEV), torch.ones(2, 1, device=DEV)
    x, out = torch.randn(2, 8000, device=DEV).to(BF), torch.full((2, 8000), 7.0, device=DEV)
    assert not quant.experts4(x, idx, w, gu, d, out) and bool((out == 7).all())
    off = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    stack, W = weight(quant, (2, 24, 8000))
    out = quant.gemm4(x, stack, torch.empty(2, 24, device=DEV), group_offsets=off)
    for g in range(2):
        Q.check_product(out[g:g + 1], x[g:g + 1], W[g])
    odd, _ = weight(quant, (2, 24, 7999))
    with pytest.raises(core.KernelError):
        quant.gemm4(x[:, :7999], odd, torch.empty(2, 24, device=DEV), group_offsets=off)


def test_refusals(quant):
    from moe_b200.ops import core

    (w, _), (pair, _), (stack, _) = weight(quant, (32, 64)), weight(quant, (32, 64), pair=True), weight(quant, (3, 32, 64))
    x, out, off = torch.zeros(5, 64, dtype=BF, device=DEV), torch.zeros(5, 32, device=DEV), torch.zeros(4, dtype=torch.int32, device=DEV)
    for args, kw in (((x.float(), w, out), {}), ((x.half(), w, out), {}), ((x[:, :63], w, out), {}), ((x, w, out[:4]), {}), ((x, w, out[:, :31]), {}),
                     ((x, w, out.double()), {}), ((x, pair, out[:, :16]), {}), ((x, w, out), dict(swiglu=True)), ((x, w, out), dict(bias=out[0, :31])),
                     ((x, w, out), dict(bias=out[0].to(BF))), ((x, pair, out[:, :16]), dict(swiglu=True, bias=out[0, :16])), ((x, w, out), dict(act="tanh")),
                     ((x, pair, out[:, :16]), dict(swiglu=True, act="relu2")), ((x, stack, out), {}), ((x, stack, out), dict(group_offsets=off[:3])),
                     ((x, stack, out), dict(group_offsets=off.long())), ((x.t().contiguous().t(), w, out), {}), ((x[0], w, out), {}),
                     ((x, w, out[:1].expand(5, 32)), {}), ((x.cpu(), w, out), {}), ((x, w, out.cpu()), {})):
        with pytest.raises(core.KernelError):
            quant.gemm4(*args, **kw)
    for bad in (dict(w=torch.zeros(32, 64, dtype=torch.float16, device=DEV)), dict(w=torch.zeros(32, 128, device=DEV)[:, ::2]), dict(w=out[0]),
                dict(w=out[:0]), dict(w=out, group=16), dict(w=out[:3].contiguous(), pair=True)):
        with pytest.raises(core.KernelError):
            quant.quantize(**bad)
    with pytest.raises(core.KernelError):
        quant.dequantize(w, torch.empty(32, 63, dtype=BF, device=DEV))


# ------------------------------------------------------------------------------------------------ streams, graphs, waits
def _run_together(quant, T, st):
    """Quantise, project, route through a layer's experts, and the same rows grouped: what a layer does with such weights."""
    H, E, size, shared, top = 256, 6, 48, 80, 2
    torch.manual_seed(0)
    proj = quant.quantize(torch.randn(H, H, device=DEV).to(BF) * H ** -0.5, 64, status=st)
    (gu, GU), (d, D) = weight(quant, (E, 2 * size, H), pair=True), weight(quant, (E, H, size), seed=1)
    (sgu, SGU), (sd, SD) = weight(quant, (2 * shared, H), pair=True, seed=2), weight(quant, (H, shared), seed=3)
    x = torch.randn(T, H, device=DEV).to(BF)
    idx = torch.rand(T, E, device=DEV).topk(top, dim=1).indices.to(torch.int32).contiguous()
    w, gate = torch.rand(T, top, device=DEV), torch.rand(T, device=DEV)
    order = idx.reshape(-1).long().argsort(stable=True)
    off = torch.cat([torch.zeros(1, device=DEV), torch.bincount(idx.reshape(-1), minlength=E).cumsum(0)]).to(torch.int32)

    def step():
        h = quant.gemm4(x, proj, torch.empty(T, H, dtype=BF, device=DEV), status=st)
        whole = torch.empty(T, H, device=DEV)
        taken = quant.experts4(h, idx, w, gu, d, whole, shared_gate_up=sgu, shared_down=sd, shared_gate=gate, status=st)
        a = quant.gemm4(h[order // top], gu, torch.empty(T * top, size, dtype=BF, device=DEV), swiglu=True, group_offsets=off, status=st)
        y = quant.gemm4(a, d, torch.empty(T * top, H, device=DEV), group_offsets=off, status=st)
        s = quant.gemm4(quant.gemm4(h, sgu, torch.empty(T, shared, dtype=BF, device=DEV), swiglu=True, status=st), sd,
                        torch.empty(T, H, device=DEV), status=st)
        grouped = torch.zeros(T, H, device=DEV).index_add_(0, order // top, y * w.reshape(-1)[order].unsqueeze(1)) + gate.unsqueeze(1) * s
        return h, whole if taken else None, grouped

    return x, proj, step, (idx, w, GU, D, (SGU[0], SD[0]), gate)


@pytest.mark.parametrize("T", [1, 8, 60])
def test_the_operators_together(quant, T):
    st = status()
    x, proj, step, (idx, w, GU, D, shared, gate) = _run_together(quant, T, st)
    h, whole, grouped = step()
    fine(st)
    Q.check_product(h, x, quant.dequantize(proj))
    y, size = plain_layer(h, idx, w, GU, D, shared, gate)
    assert (whole is not None) == (T <= 8)
    if whole is not None:
        check_layer(whole, y, size)
    # the products one by one round what lies between the two to bfloat16: 2^-8 of each term
    half = GU.shape[1] // 2
    _, terms = plain_layer(h, idx, w.abs(), GU, D.abs(), (shared[0], shared[1].abs()), gate)
    hd = h.double()
    mag = torch.zeros_like(y)
    for t in range(T):
        for e, f in [(int(e), float(f)) for e, f in zip(idx[t], w[t])]:
            g, u = GU[e, :half] @ hd[t], GU[e, half:] @ hd[t]
            mag[t] += f * (D[e].abs() @ (g * torch.sigmoid(g) * u).abs())
        s = shared[0].shape[0] // 2
        g, u = shared[0][:s] @ hd[t], shared[0][s:] @ hd[t]
        mag[t] += float(gate[t]) * (shared[1].abs() @ (g * torch.sigmoid(g) * u).abs())
    assert bool(((grouped.double() - y).abs() <= size + 2.0 ** -8 * mag + 2.0 ** -21 * mag).all())


def test_two_streams_at_once_and_replays(quant):
    """The same results from two streams that run beside one another, from a captured graph and from its replays on other inputs."""
    st = status()
    runs = [_run_together(quant, T, st) for T in (4, 40)]
    want = [[t.clone() if t is not None else None for t in run[2]()] for run in runs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in runs]
    for _ in range(5):
        got = []
        for s, run in zip(streams, runs):
            with torch.cuda.stream(s):
                got.append(run[2]())
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            for u, v in zip(a, b):
                assert (u is None and v is None) or torch.equal(u, v)
    graphs = []
    for s, run in zip(streams, runs):
        with torch.cuda.stream(s):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                out = run[2]()
        graphs.append((g, out))
    torch.cuda.synchronize()
    for again in range(3):
        for s, (g, _), run in zip(streams, graphs, runs):
            with torch.cuda.stream(s):
                run[0].mul_(-1.0 if again else 1.0)
                g.replay()
        torch.cuda.synchronize()
        for (g, out), run in zip(graphs, runs):
            for u, v in zip(out, run[2]()):
                assert (u is None and v is None) or torch.equal(u, v)
    fine(st)


@pytest.mark.parametrize("form,fault", [("tensor core", 1), ("tensor core", 2), ("tensor core", 3), ("splits", 1), ("splits", 3), ("stream", 1), ("layer", 1)])
def test_a_wait_that_runs_out_is_reported_and_leaves_the_gpu_in_order(quant, form, fault, monkeypatch):
    from moe_b200.ops import core

    if form == "tensor core":                   # (in a split tile nobody waits for the products but who issues them)
        monkeypatch.setattr(quant, "_splits", lambda *a: 1)

    torch.manual_seed(1)
    T, N, K = {"tensor core": (300, 700, 640), "splits": (40, 256, 1024), "stream": (3, 20000, 256), "layer": (4, 256, 256)}[form]
    st, x = status(), torch.randn(T, K, device=DEV).to(BF)
    if form == "layer":
        (gu, GU), (d, D) = weight(quant, (5, 96, K), pair=True), weight(quant, (5, K, 48), seed=1)
        idx = torch.tensor([[0, 1], [2, 3], [4, 0], [1, 2]], dtype=torch.int32, device=DEV)
        w, out = torch.rand(T, 2, device=DEV), torch.empty(T, K, device=DEV)
        run = lambda: quant.experts4(x, idx, w, gu, d, out, status=st)  # noqa: E731
        check = lambda: check_layer(out, *plain_layer(x, idx, w, GU, D))  # noqa: E731
    else:
        w4, W = weight(quant, (N, K))
        out = torch.empty(T, N, device=DEV)
        run = lambda: quant.gemm4(x, w4, out, status=st)  # noqa: E731
        check = lambda: Q.check_product(out, x, W[0])  # noqa: E731
    L = quant.lib()
    L.moe_q4_set_wait_test(fault, 2000)
    try:
        run()
        torch.cuda.synchronize()
    finally:
        L.moe_q4_set_wait_test(0, 0)
    assert int(st[0]) & 8, "the wait that ran out was not reported"
    with pytest.raises(core.KernelError, match="4-bit weights"):
        core.check_status(st)
    for _ in range(3):
        run()
    fine(st)
    check()


@pytest.mark.parametrize("fault", [1, 2, 3])
def test_a_wait_of_groups_that_runs_out(quant, fault):
    from moe_b200.ops import core

    torch.manual_seed(2)
    rows, K, N = [40, 90, 0, 128, 60], 640, 300
    off = torch.tensor([0, 40, 130, 130, 258, 318], dtype=torch.int32, device=DEV)
    w4, W = weight(quant, (5, N, K))
    st, x, out = status(), torch.randn(318, K, device=DEV).to(BF), torch.empty(318, N, device=DEV)
    L = quant.lib()
    L.moe_q4_set_wait_test(fault, 2000)
    try:
        quant.gemm4(x, w4, out, group_offsets=off, status=st)
        torch.cuda.synchronize()
    finally:
        L.moe_q4_set_wait_test(0, 0)
    assert int(st[0]) & 8, "the wait that ran out was not reported"
    with pytest.raises(core.KernelError, match="4-bit weights"):
        core.check_status(st)
    quant.gemm4(x, w4, out, group_offsets=off, status=st)
    fine(st)
    at = 0
    for g, r in enumerate(rows):
        if r:
            Q.check_product(out[at:at + r], x[at:at + r], W[g])
        at += r


# ------------------------------------------------------------------------------------------------ models
def _designs():
    import ditazen_util
    import divadra_util
    import fogapel_util
    import kulanex_util
    import supevik_util
    import zosipel_util

    found = [("qwen " + n, helpers.CONFIGS[n]) for n in ("A", "B", "D", "E")]
    for u in (supevik_util, fogapel_util, zosipel_util, divadra_util, ditazen_util, kulanex_util):
        n = sorted(u.CONFIGS)[0]
        found.append((u.__name__[:-5], u.config_dict(n)))
    return found


@pytest.mark.parametrize("which", range(10))
def test_a_model_with_its_matrices_in_4_bits(quant, which, monkeypatch):
    """Prompts and single tokens, against the same model whose matrices are the 4-bit ones' values in bfloat16: the same numbers, other kernels."""
    import moe_b200
    from moe_b200.ops.quant import Weight4
    from moe_b200.parts.base import Part

    name, config = _designs()[which]
    std = 0.02
    held = moe_b200.random_model(config, seed=5, std=std, weights="int4", weight_group=(32, 64, 128)[which % 3])
    kept = [w for b in held.blocks for p in b.parts() for w in vars(p).values() if isinstance(w, Weight4)]
    assert kept or which >= 4, "nothing is held in 4 bits"
    group = held.rt.weight_group

    def values(self, rt, w, pair=False):
        if w.dtype != BF:
            return w
        return quant.dequantize(quant.quantize(w.contiguous(), group, pair=pair))

    with monkeypatch.context() as m:
        m.setattr(Part, "hold", values)
        same = moe_b200.random_model(config, seed=5, std=std)
    vocab = held.spec.vocab_size
    gen = torch.Generator().manual_seed(which)
    prompts = [torch.randint(0, vocab, (n,), generator=gen).tolist() for n in (9, 1, 30)]
    rows = []
    for model in (held, same):
        engine = moe_b200.Engine(model, max_tokens=2048)
        slots = [engine.new_sequence() for _ in prompts]
        got = [engine.step(slots, prompts, [[len(p) - 1] for p in prompts]).float().clone()]
        for i in range(3):
            got.append(engine.step(slots, [[(7 * i + j) % vocab] for j in range(3)], [[0]] * 3).float().clone())
        model.rt.check()
        rows.append(torch.stack(got))
    far = float((rows[0] - rows[1]).abs().max() / rows[1].abs().max())
    assert far < G.TOL_CUT_BF16, far


def test_the_command_line_generates_with_4_bit_weights(model_dirs, capsys):
    from moe_b200 import cli

    d = model_dirs.get("D", "bfloat16", seed=1, std=0.02)
    cli.main(["run", d, "--ids", "5,17,3", "-n", "6", "--weights", "int4", "--weight-group", "32", "--no-stream"])
    assert capsys.readouterr().out.strip()
    with pytest.raises(SystemExit):
        cli.main(["run", d, "--ids", "5", "-n", "1", "--weights", "int3"])
