"""Products over weights held in 4 bits, as cases that can be timed and compared.

A weight W [G, N, K] in 4 bits is a pair of tensors.  ``group`` neighbouring k of a row share a scale s of five
significant bits, and an element is q s with a whole number q from -7 to 7, which bfloat16 holds exactly.

  codes   uint8 [G, ceil(N / 16), ceil(K / 64), 8, 4, 4, 2, 2]: the byte at [.., strip, block, r, t, j, h, p] holds k = 64 block +
          16 j + 4 t + 2 p + h of rows 16 strip + r (low four bits) and 16 strip + r + 8 (high four bits), each as q + 8
  scales  bfloat16 [G, ceil(N / 16), ceil(K / group), 8, 2]: rows r and r + 8 of a strip beside one another

Rows beyond N have scale 0, elements beyond K have q = 0.  A pair (gate rows and up rows, N / 2 each) fills whole strips of 16 rows with
either half: 2 ceil(N / 2 / 16) strips.

Operators (``op``)
  quantize  the values that a bfloat16 matrix keeps in 4 bits: s = max |w| / 7 rounded to five bits, q = w / s rounded, q s
  gemm      y = x W^T (+ bias), or with ``swiglu`` silu(x Wg^T) * (x Wu^T) where W's rows are Wg's and then Wu's
  grouped   the same where rows [offsets[g], offsets[g + 1]) of x meet W[g]: routed experts
  experts   a whole layer of routed experts for a few tokens: each token's ``top`` experts by their weights, and the shared
            expert by its gate
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BF, F4, F8 = torch.bfloat16, torch.float32, torch.float64


def _gemm(M, N, K, group=64, swiglu=False, bias=False, out="float32", **more):
    return dict(more, op="gemm", M=M, N=N, K=K, group=group, swiglu=swiglu, bias=bias, out=out)


def _grouped(tokens, top, G, N, K, group=64, swiglu=False, out="bfloat16", **more):
    return dict(more, op="grouped", tokens=tokens, top=top, G=G, N=N, K=K, group=group, swiglu=swiglu, out=out)


def _experts(T, H, E, top, size, shared, group=64, out="bfloat16", **more):
    return dict(more, op="experts", T=T, H=H, E=E, top=top, size=size, shared=shared, group=group, out=out)


def _quantize(N, K, group=64, **more):
    return dict(more, op="quantize", N=N, K=K, group=group)


def listed():
    return [
        # loading: the fused gate and up rows of a shared expert
        _quantize(11264, 2048, name="quantize-shared"),
        # loading: one routed expert's down projection of a small model, sizes that are no whole tiles
        _quantize(1000, 700, 32, name="quantize-odd"),
        # one user waits for the next token: the attention's output projection, where latency counts
        _gemm(1, 2048, 2048, name="output-1"),
        # the benchmark's headline batch: queries, keys and values with their bias
        _gemm(8, 6144, 2048, bias=True, name="qkv-8"),
        # a wide model's shared expert, sixteen sequences: the stream of weights counts
        _gemm(16, 20480, 3584, 128, swiglu=True, out="bfloat16", name="shared-wide-16"),
        # a few short questions that arrive together
        _gemm(113, 2048, 5632, out="bfloat16", name="down-113"),
        # a prompt through the shared expert's gate and up rows
        _gemm(2048, 5632, 2048, swiglu=True, out="bfloat16", name="shared-2048"),
        # a busy server's step: every expert is read, a few rows each
        _grouped(64, 4, 60, 2048, 1408, name="routed-down-64"),
        # a prompt through all experts' gate and up rows
        _grouped(2048, 4, 60, 1408, 2048, swiglu=True, name="routed-2048"),
        # a whole layer of experts for one token and for the headline batch
        _experts(1, 2048, 60, 4, 1408, 5632, name="layer-1"),
        _experts(8, 2048, 60, 4, 1408, 5632, name="layer-8"),
        # a small model without a shared expert, three sequences
        _experts(3, 1024, 32, 2, 704, 0, 32, name="layer-small-3"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _size(rng, low, high):
    """Mostly whole units of 8, now and then any number."""
    n = _log(rng, low, high)
    return n if rng.random() < 0.2 else max(8, n // 8 * 8)


def draw(rng):
    group = rng.choice([32, 64, 64, 128])
    op = rng.choice(["quantize", "gemm", "gemm", "gemm", "grouped", "grouped", "experts", "experts"])
    if op == "quantize":
        return _quantize(_size(rng, 16, 11264), _size(rng, 40, 2048), group)
    if op == "gemm":
        swiglu = rng.random() < 0.4
        rows = rng.choice(["few", "some", "many"])
        M = {"few": _log(rng, 1, 16), "some": _log(rng, 17, 256), "many": _log(rng, 257, 4096)}[rows]
        N, K = _size(rng, 100, 6144), _size(rng, 100, 5632)
        while 2 * M * N * K * (2 if swiglu else 1) > 4.7e10:
            M = M * 3 // 4
        if M > 64:                       # prompts come in rows of whole 16-byte units
            K = max(8, K // 8 * 8)
        return _gemm(M, N, K, group, swiglu=swiglu, bias=not swiglu and rng.random() < 0.5,
                     out="bfloat16" if swiglu or M > 64 else rng.choice(["float32", "bfloat16"]))
    if op == "grouped":
        G, top = rng.choice([(60, 4), (32, 2), (64, 8), (16, 2)])
        N, K, swiglu = _size(rng, 100, 2048), max(8, _log(rng, 100, 2048) // 8 * 8), rng.random() < 0.5
        tokens = _log(rng, 5, 2048)
        while 2 * tokens * top * N * K * (2 if swiglu else 1) > 9e10:
            tokens = tokens * 3 // 4
        return _grouped(tokens, top, G, N, K, group, swiglu=swiglu)
    E, top = rng.choice([(60, 4), (32, 2), (64, 8), (16, 2)])
    H, size = max(64, _log(rng, 64, 2048) // 8 * 8), _size(rng, 32, 1408)
    return _experts(rng.randint(1, 8 if top < 8 else 4), H, E, top, size, rng.choice([0, _size(rng, 32, 5632)]), group)


def _weight(G, N, K, group, gen, pair=False):
    """A weight as it lies in 4 bits, drawn where it lies: q as a normal distribution cut at its group's maximum leaves them,
    scales that keep a row's squares at a sum of about one."""
    half = N // 2 if pair else N
    S, B, Q = -(-half // 16) * (2 if pair else 1), -(-K // 64), -(-K // group)
    codes = torch.empty(G, S, B, 8, 4, 4, 2, 2, dtype=torch.uint8, device=DEV)
    k = (torch.arange(4, device=DEV).view(4, 1, 1, 1) * 4 + torch.arange(4, device=DEV).view(1, 4, 1, 1) * 16
         + torch.arange(2, device=DEV).view(1, 1, 2, 1) + torch.arange(2, device=DEV).view(1, 1, 1, 2) * 2)
    k = torch.arange(B, device=DEV).view(B, 1, 1, 1, 1, 1) * 64 + k
    for g in range(G):
        q = (torch.randn((2,) + codes.shape[1:], device=DEV, generator=gen) * 2.9).round_().clamp_(-7, 7) + 8
        q = torch.where(k < K, q, 8.0).to(torch.uint8)
        codes[g] = q[0] | (q[1] << 4)
    s = (1.0 / (2.8 * math.sqrt(K))) * (1 + 0.15 * torch.randn(G, S, Q, 8, 2, device=DEV, generator=gen)).clamp_(0.5, 2.0)
    m, e = torch.frexp(s)
    row = (torch.arange(S, device=DEV) % -(-half // 16) * 16).view(S, 1, 1, 1) + torch.arange(8, device=DEV).view(8, 1) + 8 * torch.arange(2, device=DEV)
    return codes, (torch.ldexp((m * 32).round(), e - 5) * (row < half)).to(BF)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)

    def rnd(*shape):
        return torch.randn(*shape, device=DEV, generator=gen)

    s = {"case": case, "status": torch.zeros(4, dtype=torch.int32, device=DEV)}
    op, group = case["op"], case["group"]
    if op == "quantize":
        s["w"] = (rnd(case["N"], case["K"]) * 0.02 * (1 + 0.3 * rnd(case["N"], 1).abs())).to(BF)
    elif op == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        s["x"] = rnd(M, K).to(BF)
        s["codes"], s["scales"] = _weight(1, N * (2 if case["swiglu"] else 1), K, group, gen, case["swiglu"])
        s["bias"] = rnd(N) if case["bias"] else None
    elif op == "grouped":
        G, top, K = case["G"], case["top"], case["K"]
        s["x"] = rnd(case["tokens"] * top, K).to(BF)
        s["codes"], s["scales"] = _weight(G, case["N"] * (2 if case["swiglu"] else 1), K, group, gen, case["swiglu"])
        picks = (torch.rand(case["tokens"], G, device=DEV, generator=gen)).topk(top, dim=1).indices
        rows = torch.bincount(picks.reshape(-1), minlength=G)
        s["offsets"] = torch.cat([rows.new_zeros(1), rows.cumsum(0)]).to(torch.int32)
        s["most"] = int(rows.max())
    else:
        T, H, E, top, size, shared = (case[n] for n in ("T", "H", "E", "top", "size", "shared"))
        s["x"] = rnd(T, H).to(BF)
        w, idx = (rnd(T, E) * 1.5).softmax(1).topk(top, dim=1)
        s["idx"], s["w"] = idx.to(torch.int32).contiguous(), w.contiguous()
        s["gu"], s["down"] = _weight(E, 2 * size, H, group, gen, True), _weight(E, H, size, group, gen)
        s["sgu"] = s["sdown"] = s["gate"] = None
        if shared:
            s["sgu"], s["sdown"] = _weight(1, 2 * shared, H, group, gen, True), _weight(1, H, shared, group, gen)
            s["gate"] = torch.sigmoid(rnd(T))
    return s


# ---------------------------------------------------------------------------------------------- plain forms
def _values(codes, scales, N, K, group, pair=False):
    """[G, N, K] float32 from the stored bytes."""
    G, S, B = codes.shape[:3]
    if pair:
        return _values(codes.view(2 * G, S // 2, *codes.shape[2:]), scales.view(2 * G, S // 2, *scales.shape[2:]), N // 2, K, group).view(G, N, K)
    q = torch.stack([codes & 15, codes >> 4], dim=3)                          # [G, S, B, 2, 8, 4 t, 4 j, 2 h, 2 p]
    q = q.permute(0, 1, 3, 4, 2, 6, 5, 8, 7).reshape(G, S * 16, B * 64)[:, :N, :K].float() - 8
    s = scales.float().permute(0, 1, 4, 3, 2).reshape(G, S * 16, -1)[:, :N]
    return q * s.repeat_interleave(group, dim=2)[:, :, :K]


def _silu_mul(y):
    g, u = y.chunk(2, dim=-1)
    return g / (1 + torch.exp(-g)) * u


def _plain(s):
    case = s["case"]
    op, group = case["op"], case["group"]
    if op == "quantize":
        N, K = case["N"], case["K"]
        w = s["w"].double()
        w = torch.cat([w, w.new_zeros(N, -K % group)], dim=1).view(N, -1, group)
        m, e = torch.frexp(w.abs().amax(dim=2, keepdim=True) / 7)
        sc = torch.ldexp((m * 32).round(), e - 5)
        q = torch.where(sc > 0, (w / sc).round(), 0.0)
        return (q * sc).view(N, -1)[:, :K].to(BF)
    out = getattr(torch, case["out"])
    if op == "gemm":
        W = _values(s["codes"], s["scales"], case["N"] * (2 if case["swiglu"] else 1), case["K"], group, case["swiglu"])[0]
        y = s["x"].float() @ W.t()
        y = _silu_mul(y) if case["swiglu"] else y if s["bias"] is None else y + s["bias"]
        return y.to(out)
    if op == "grouped":
        W = _values(s["codes"], s["scales"], case["N"] * (2 if case["swiglu"] else 1), case["K"], group, case["swiglu"])
        off, P = s["offsets"].long(), s["x"].shape[0]
        row = torch.arange(P, device=DEV)
        g = torch.searchsorted(off[1:].contiguous(), row, right=True)
        x = torch.zeros(case["G"], s["most"], case["K"], device=DEV)
        x[g, row - off[g]] = s["x"].float()
        y = (x @ W.transpose(1, 2))[g, row - off[g]]
        return (_silu_mul(y) if case["swiglu"] else y).to(out)
    T, H, top, size, shared = (case[n] for n in ("T", "H", "top", "size", "shared"))
    e = s["idx"].reshape(-1).long()
    x = s["x"].float()
    gu = _values(s["gu"][0][e], s["gu"][1][e], 2 * size, H, group, True)
    act = _silu_mul((gu @ x.repeat_interleave(top, dim=0).unsqueeze(2)).squeeze(2))
    down = _values(s["down"][0][e], s["down"][1][e], H, size, group)
    y = (down @ act.unsqueeze(2)).view(T, top, H)
    y = (y * s["w"].unsqueeze(2)).sum(dim=1)
    if shared:
        a = _silu_mul(x @ _values(*s["sgu"], 2 * shared, H, group, True)[0].t())
        y = y + s["gate"].unsqueeze(1) * (a @ _values(*s["sdown"], H, shared, group)[0].t())
    return y.to(out)


# ------------------------------------------------------------------------------------ the framework's operators
def _own(s):
    from moe_b200.ops import quant

    case = s["case"]
    op, group = case["op"], case["group"]
    if op == "quantize":
        return quant.dequantize(quant.quantize(s["w"], group, status=s["status"]))
    out = getattr(torch, case["out"])
    if op == "experts":
        T, H, E, size, shared = (case[n] for n in ("T", "H", "E", "size", "shared"))
        y = torch.empty(T, H, dtype=out, device=DEV)
        more = {}
        if shared:
            more = dict(shared_gate_up=quant.Weight4(*s["sgu"], (2 * shared, H), group, pair=True),
                        shared_down=quant.Weight4(*s["sdown"], (H, shared), group), shared_gate=s["gate"])
        quant.experts4(s["x"], s["idx"], s["w"], quant.Weight4(*s["gu"], (E, 2 * size, H), group, pair=True),
                       quant.Weight4(*s["down"], (E, H, size), group), y, status=s["status"], **more)
        return y
    rows = case["N"] * (2 if case["swiglu"] else 1)
    shape = (rows, case["K"]) if op == "gemm" else (case["G"], rows, case["K"])
    y = torch.empty(s["x"].shape[0], case["N"], dtype=out, device=DEV)
    quant.gemm4(s["x"], quant.Weight4(s["codes"], s["scales"], shape, group, pair=case["swiglu"]), y, swiglu=case["swiglu"], bias=s.get("bias"),
                group_offsets=s.get("offsets"), status=s["status"])
    return y


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------- in 64 bits
def _element(codes, scales, N, K, group, pair=False):
    """[N, K] float64 of one weight [strips, blocks, ..], each element fetched by its own place."""
    flat, sc = codes.reshape(-1), scales.double().reshape(-1)
    n, k = torch.arange(N, device=DEV).unsqueeze(1), torch.arange(K, device=DEV).unsqueeze(0)
    c, r, strip = k % 64, n % 16, n // 16
    if pair:
        r, strip = n % (N // 2) % 16, n % (N // 2) // 16 + n // (N // 2) * (codes.shape[0] // 2)
    byte = (strip * codes.shape[1] + k // 64) * 512 + (r % 8) * 64 + (c % 16 // 4) * 16 + (c // 16) * 4 + (c % 2) * 2 + c % 4 // 2
    q = torch.bitwise_right_shift(flat[byte].to(torch.int32), (r // 8 * 4).to(torch.int32)).bitwise_and_(15).double() - 8
    return q * sc[((strip * scales.shape[1] + k // group) * 8 + r % 8) * 2 + r // 8]


def _swiglu8(x, W):
    half = W.shape[0] // 2
    a, b = x @ W[:half].t(), x @ W[half:].t()
    return a * torch.sigmoid(a) * b


def exact(case, seed):
    s = prepare(case, seed)
    op, group = case["op"], case["group"]
    if op == "quantize":
        N, K = case["N"], case["K"]
        w, out = s["w"].double(), torch.empty(N, K, dtype=F8, device=DEV)
        for k in range(0, K, group):
            piece = w[:, k:k + group]
            top = piece.abs().max(dim=1, keepdim=True).values / 7
            unit = torch.exp2(torch.floor(torch.log2(top.clamp_min(1e-300))) - 4)      # the fifth significant bit
            unit = torch.where(top / unit >= 32, unit * 2, torch.where(top / unit < 16, unit / 2, unit))
            step = torch.round(top / unit) * unit
            out[:, k:k + group] = torch.where(step > 0, torch.round(piece / step.clamp_min(1e-300)) * step, 0.0)
        return out
    if op == "gemm":
        W = _element(s["codes"][0], s["scales"][0], case["N"] * (2 if case["swiglu"] else 1), case["K"], group, case["swiglu"])
        x = s["x"].double()
        return _swiglu8(x, W) if case["swiglu"] else x @ W.t() + (0 if s["bias"] is None else s["bias"].double())
    if op == "grouped":
        x, off = s["x"].double(), s["offsets"].tolist()
        out = torch.zeros(x.shape[0], case["N"], dtype=F8, device=DEV)
        for g in range(case["G"]):
            if off[g] < off[g + 1]:
                W = _element(s["codes"][g], s["scales"][g], case["N"] * (2 if case["swiglu"] else 1), case["K"], group, case["swiglu"])
                rows = x[off[g]:off[g + 1]]
                out[off[g]:off[g + 1]] = _swiglu8(rows, W) if case["swiglu"] else rows @ W.t()
        return out
    x, T, H, size, shared = s["x"].double(), case["T"], case["H"], case["size"], case["shared"]
    out = torch.zeros(T, H, dtype=F8, device=DEV)
    for t in range(T):
        for j, e in enumerate(s["idx"][t].tolist()):
            a = _swiglu8(x[t:t + 1], _element(s["gu"][0][e], s["gu"][1][e], 2 * size, H, group, True))
            out[t] += s["w"][t, j].double() * (a @ _element(s["down"][0][e], s["down"][1][e], H, size, group).t())[0]
    if shared:
        a = _swiglu8(x, _element(s["sgu"][0][0], s["sgu"][1][0], 2 * shared, H, group, True))
        out += s["gate"].double().unsqueeze(1) * (a @ _element(s["sdown"][0][0], s["sdown"][1][0], H, shared, group).t())
    return out


def work(case):
    per = 0.5 + 2 / case["group"]                       # bytes of an element in 4 bits
    if case["op"] == "quantize":
        n = case["N"] * case["K"]
        return {"bytes": n * (2 + 2 * per + 2), "flops": 4 * n}
    size = 2 if case["out"] == "bfloat16" else 4
    if case["op"] == "gemm":
        M, K, rows = case["M"], case["K"], case["N"] * (2 if case["swiglu"] else 1)
        return {"bytes": rows * K * per + 2 * M * K + size * M * case["N"], "flops": 2 * M * rows * K}
    if case["op"] == "grouped":
        G, K, rows = case["G"], case["K"], case["N"] * (2 if case["swiglu"] else 1)
        P, read = case["tokens"] * case["top"], G * (1 - (1 - case["top"] / G) ** case["tokens"])
        return {"bytes": read * rows * K * per + 2 * P * K + size * P * case["N"], "flops": 2 * P * rows * K}
    T, H, E, top = case["T"], case["H"], case["E"], case["top"]
    read = E * (1 - (1 - top / E) ** T)
    return {"bytes": 3 * H * (read * case["size"] + case["shared"]) * per + T * H * (2 + size),
            "flops": 6 * T * H * (top * case["size"] + case["shared"])}
