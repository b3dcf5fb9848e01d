"""Python face of the kernel library ``q4``: weights held in 4 bits and the products over them.

A ``Weight4`` stands for a matrix [N, K] or a stack of them [G, N, K].  ``group`` (32, 64 or 128) neighbouring elements of a
row share a scale s = max |w| / 7 rounded to five significant bits; an element is q s with q = w / s rounded, a whole number from -7 to 7.  q s
has at most eight significant bits, so it is a bfloat16: a product over a ``Weight4`` is the product over ``dequantize`` of it, but for the
order of the 32-bit sums (and silu's exponential, quicker for many rows: 2 + 1.2 |g| ulp).  0.5 + 2 / group bytes an element.

    w4 = quantize(w, group=64)                 # w: float32 or bfloat16, on the device
    gemm4(x, w4, out, bias=b)                  # out = x w^T (+ b); x bfloat16 [M, K], any M
    gemm4(x, pair4, out, swiglu=True)          # out = silu(x gate^T) * (x up^T); pair4 = quantize(cat([gate, up]), pair=True)
    gemm4(xs, stack4, out, group_offsets=o)    # rows [o[g], o[g + 1]) of xs meet stack4[g]
    experts4(x, idx, w, gate_up4, down4, out)  # a layer of routed experts for up to 8 tokens, in two launches

Everything launches on the current stream of the current device, and a tensor on another device is refused.  The functions may be
called while a CUDA graph is captured.
"""
from __future__ import annotations

import functools
import os
from ctypes import c_float, c_int, c_longlong, c_uint, c_void_p
from typing import Optional, Tuple

import torch

from . import build, core, tc

GROUPS = (32, 64, 128)
SIZE_MAX = 1 << 30
EXPERTS_TOKENS = 8            # tokens that ``experts4`` takes
FEW_ROWS = 24                 # rows up to which a product streams its weights through registers
GROUP_FEW_ROWS = 14           # the same of groups, on average
GROUPS_A_LAUNCH = 1024        # groups that one launch of a grouped product takes

_U8, _BF16, _F32 = torch.uint8, torch.bfloat16, torch.float32
_lib = None


def lib():
    global _lib
    if _lib is None:
        L = build.load("q4")
        P, I, F, LL = c_void_p, c_int, c_float, c_longlong
        for name, args in (("moe_q4_quantize", [P, I, I, I, I, I, I, P, P, P, P]),
                           ("moe_q4_dequantize", [P, P, I, I, I, I, I, P, P]),
                           ("moe_gemm_q4", [P, I, I, P, P, I, I, I, I, I, P, I, I, P, P, I, F, I, P, P]),
                           ("moe_gemm_q4_tc", [P, I, I, P, P, I, I, I, I, I, P, I, I, P, P, I, F, I, I, P, P]),
                           ("moe_experts_q4", [P, I, I, I, P, P, I, I, I, P, P, P, P, I, P, P, P, P, P, I, P, LL, P, I, I, I, P, P])):
            fn = getattr(L, name)
            fn.argtypes, fn.restype = args, c_int
        L.moe_q4_holds_rows.argtypes, L.moe_q4_holds_rows.restype = [I, I, I], c_int
        L.moe_q4_set_wait_test.argtypes, L.moe_q4_set_wait_test.restype = [I, c_uint], None
        L.moe_q4_set_pdl.argtypes, L.moe_q4_set_pdl.restype = [I], None
        if os.environ.get("MOE_B200_PDL", "1") == "0":      # programmatic dependent launch off
            L.moe_q4_set_pdl(0)
        _lib = L
    return _lib


class Weight4:
    """A matrix ``shape`` = (N, K), or a stack (G, N, K), in 4 bits.

    ``codes``: uint8 [G, strips, ceil(K / 64), 8, 4, 4, 2, 2] (any shape of that many elements): strips of 16 rows; the byte at
    [.., strip, block, r, t, j, h, p] holds k = 64 block + 16 j + 4 t + 2 p + h of rows r (low four bits) and r + 8 (high four bits) of the
    strip, each as q + 8.  ``scales``: bfloat16 [G, strips, ceil(K / group), 8, 2], rows r and r + 8 beside one another, each of at most five
    significant bits.  Rows beyond N have scale 0, elements beyond K q = 0.  With ``pair`` the rows are a gated feed-forward's, N / 2 of
    the gate and N / 2 of up, and either half fills whole strips; a pair is what products with ``swiglu`` take.

    Products read a weight before the kernel in front of them on their stream has ended, as soon as that cannot be the one that wrote it: from a
    weight's second product on a stream on, or on any stream behind ``settle``.  So ``codes`` and ``scales`` may be written (on the product's stream, or ordered
    before it) right until the weight's first product, and not after it: who writes other ones into the same tensors makes another ``Weight4`` of them."""

    __slots__ = ("codes", "scales", "shape", "group", "pair", "G", "N", "K", "place", "pointers", "read_on")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape: Tuple[int, ...], group: int = 64, pair: bool = False):
        if len(shape) == 2:
            G = 1
            N, K = shape
        elif len(shape) == 3:
            G, N, K = shape
        else:
            raise core.KernelError(f"Weight4: the shape is (N, K) or (G, N, K), not {tuple(shape)}")
        if not (0 < G <= SIZE_MAX and 0 < N <= SIZE_MAX and 0 < K <= SIZE_MAX):
            raise core.KernelError(f"Weight4: sizes from 1 to 2^30, not {tuple(shape)}")
        if group not in GROUPS:
            raise core.KernelError(f"Weight4: the group is one of {GROUPS}, not {group}")
        if pair and N % 2:
            raise core.KernelError("Weight4: a pair has as many gate rows as up rows")
        strips = G * _strips(N, pair)
        nc, ns = strips * ((K + 63) // 64) * 512, strips * ((K + group - 1) // group) * 16
        pc, ps, place = codes.data_ptr(), scales.data_ptr(), codes.get_device()
        if (codes.dtype is not _U8 or scales.dtype is not _BF16 or codes.numel() != nc or scales.numel() != ns or not codes.is_contiguous()
                or not scales.is_contiguous() or (pc | ps) & 15 or scales.get_device() != place):
            raise core.KernelError(f"Weight4: codes and scales of {tuple(shape)} in groups of {group} are contiguous uint8 and bfloat16 tensors "
                                   f"of {nc} and {ns} elements on one device")
        self.codes, self.scales, self.shape, self.group, self.pair = codes, scales, tuple(shape), group, bool(pair)
        self.G, self.N, self.K, self.place, self.pointers = G, N, K, place, (pc, ps)
        self.read_on = ()             # the streams that have had a product of this weight; None: all may be taken to

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def dtype(self) -> str:
        """(No ``torch.dtype``: whoever asks whether a weight is bfloat16 is told no.)"""
        return "int4"

    def __reduce__(self):
        """(A copy, or what is stored and read back, has tensors of its own: their addresses, and what has read them.)"""
        return Weight4, (self.codes, self.scales, self.shape, self.group, self.pair)

    def _parts(self, groups: int):
        """(so many neighbouring matrices of a stack, the first one's number)"""
        codes, scales = self.codes.view(self.G, -1), self.scales.view(self.G, -1)
        for g in range(0, self.G, groups):
            part = Weight4(codes[g:g + groups], scales[g:g + groups], (min(groups, self.G - g), self.N, self.K), self.group, self.pair)
            part.read_on = self.read_on
            yield part, g

    def settle(self) -> None:
        """Waits until the device has done what it was given, the writing of this weight with it."""
        if self.place >= 0:
            torch.cuda.synchronize(self.device)
        self.read_on = None

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + 2 * self.scales.numel()

    def __repr__(self):
        return f"Weight4({'x'.join(map(str, self.shape))}, groups of {self.group}{', pair' if self.pair else ''})"


def _strips(N: int, pair: bool) -> int:
    return (N // 2 + 15) // 16 * 2 if pair else (N + 15) // 16


def _here(place: int, what: str):
    """A kernel launches on the current device's current stream: its tensors have to lie there."""
    if place < 0:
        raise core.KernelError(f"{what}: expected CUDA tensors; there is no CPU path")
    if core._raw_device is not None and place != core._raw_device():
        raise core.KernelError(f"{what}: tensors on cuda:{place}, but the current device is cuda:{core._raw_device()}")


def _on(t: Optional[torch.Tensor], place: int, name: str, dtype, numel: Optional[int] = None):
    if t is None:
        return None
    if t.dtype is not dtype or t.get_device() != place or not t.is_contiguous() or (numel is not None and t.numel() != numel):
        raise core.KernelError(f"{name}: expected a contiguous {dtype} tensor{'' if numel is None else f' of {numel} elements'} on cuda:{place}, got "
                               f"{t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _status(t: torch.Tensor, place: int):
    """(Faults and, beside them, where the first wait ran out.)"""
    if t.numel() < 2:
        raise core.KernelError("status: expected what core.new_status makes")
    return _on(t, place, "status", torch.int32)


def _matrix(t: torch.Tensor, place: int, name: str, wide: bool):
    """(rows, columns, row pitch) of a matrix with dense rows, bfloat16 or (``wide``) float32."""
    dtype = t.dtype
    if (dtype is not _BF16 and not (wide and dtype is _F32)) or t.get_device() != place or t.dim() != 2:
        raise core.KernelError(f"{name}: expected a matrix of bfloat16{' or float32' if wide else ''} on cuda:{place}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    rows, columns = t.shape
    pitch, step = t.stride()
    if rows <= 1:                 # (whatever torch says of the pitch)
        pitch = columns
    if (step != 1 and columns > 1) or pitch < columns or pitch > 0x7fffffff or rows >= 1 << 28:
        raise core.KernelError(f"{name}: expected less than 2^28 dense rows that do not overlap, less than 2^31 elements apart, got strides {t.stride()} of "
                               f"{tuple(t.shape)}")
    return rows, columns, pitch


def _have_read(stream: int, *weights: Weight4):
    """(Not what is captured: a graph's launches say nothing of the stream that it was captured on.)"""
    if _capturing():
        return
    for w in weights:
        read_on = w.read_on
        if read_on is not None and stream not in read_on:
            w.read_on = read_on + (stream,)


_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", torch.cuda.is_current_stream_capturing)


def quantize(w: torch.Tensor, group: int = 64, *, pair: bool = False, status=None) -> Weight4:
    """The matrix or stack ``w`` (float32 or bfloat16, contiguous) in 4 bits.  A group that holds an infinity or a NaN is marked so that
    products over it are NaN, and reported through ``status``."""
    core._chk(w, "w")
    core._dt(w)
    _here(w.get_device(), "quantize")
    if w.dim() not in (2, 3) or not w.numel() or max(w.shape) > SIZE_MAX:
        raise core.KernelError(f"quantize: a matrix or a stack of matrices of sizes from 1 to 2^30, not {tuple(w.shape)}")
    if group not in GROUPS:
        raise core.KernelError(f"quantize: the group is one of {GROUPS}, not {group}")
    G, N, K = (1, *w.shape) if w.dim() == 2 else w.shape
    if pair and N % 2:
        raise core.KernelError("quantize: a pair has as many gate rows as up rows")
    strips = _strips(N, pair)
    device = w.device                     # (a tensor of one dimension takes two thirds of the host time of one of eight)
    codes = torch.empty(G * strips * -(-K // 64) * 512, dtype=torch.uint8, device=device)
    scales = torch.empty(G * strips * -(-K // group) * 16, dtype=torch.bfloat16, device=device)
    core._ok((_lib or lib()).moe_q4_quantize(w.data_ptr(), core._dt(w), G, N, K, group, pair, codes.data_ptr(), scales.data_ptr(),
                                             None if status is None else _status(status, w.get_device()), core._stream()), "quantize")
    return Weight4(codes, scales, w.shape, group, pair)


def dequantize(w: Weight4, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The values that ``w`` stands for, exactly, as bfloat16 of ``w.shape``."""
    _here(w.place, "dequantize")
    if out is None:
        out = torch.empty(w.shape, dtype=torch.bfloat16, device=w.device)
    elif tuple(out.shape) != w.shape:
        raise core.KernelError(f"dequantize: out is {tuple(out.shape)}, the weight {w.shape}")
    core._ok((_lib or lib()).moe_q4_dequantize(*w.pointers, w.G, w.N, w.K, w.group, w.pair, _on(out, w.place, "out", torch.bfloat16), core._stream()),
             "dequantize")
    return out


def gemm4(x: torch.Tensor, w: Weight4, out: torch.Tensor, *, swiglu: bool = False, bias: Optional[torch.Tensor] = None,
          group_offsets: Optional[torch.Tensor] = None, act: str = "silu", act_param: float = 0.0, any_rows: bool = False, status=None) -> torch.Tensor:
    """out = x w^T (+ bias), or act(x gate^T) * (x up^T) with ``swiglu`` and a pair; ``act``: as in ``tc.gemm_tc``.

    x: bfloat16 [M, K], dense rows of any pitch, of magnitudes below 2^119 (few rows meet the codes before the scale); out: float32 or bfloat16 [M, N] (a pair:
    [M, N / 2]), dense rows of any pitch.
    A stack needs ``group_offsets`` (int32 [G + 1], ascending): rows [offsets[g], offsets[g + 1]) of x meet w[g]; rows that no group
    has are left as they were.

    The tensor cores take rows of x in whole 16-byte units (K and the pitch multiples of 8, an aligned first row).  Of others, ``any_rows`` copies those that
    only they take, or take at once; without it a dense product of many such rows reads the weight once for every 24 of them, and groups with K beyond 5,500
    or so are refused."""
    place = x.get_device()
    _here(place, "gemm4")
    M, K, ldx = _matrix(x, place, "x", False)
    rows, N, ldo = _matrix(out, place, "out", True)
    if w.place != place or K != w.K or rows != M or N != (w.N // 2 if swiglu else w.N):
        raise core.KernelError(f"gemm4: shapes x{tuple(x.shape)} w{w.shape} out{tuple(out.shape)}, on {x.device} and {w.device}")
    if swiglu != w.pair:
        raise core.KernelError("gemm4: a pair is multiplied with swiglu, another weight without")
    if swiglu:
        if bias is not None or act not in core.GLU_ACTS:
            raise core.KernelError("gemm4: a gated product takes no bias and an activation of core.GLU_ACTS")
        code = core.GLU_ACTS[act]
    else:
        if act != "silu" and act not in core.PLAIN_ACTS:
            raise core.KernelError("gemm4: the activation of an ungated product is one of core.PLAIN_ACTS")
        code = core.PLAIN_ACTS.get(act, 0)
    if group_offsets is None and w.G != 1:
        raise core.KernelError("gemm4: a stack needs group_offsets")
    pb = None if bias is None else _on(bias, place, "bias", _F32, N)
    po = None if group_offsets is None else _on(group_offsets, place, "group_offsets", torch.int32, w.G + 1)
    st = None if status is None else _status(status, place)
    if not M:
        return out
    if w.G > GROUPS_A_LAUNCH:
        for part, g in w._parts(GROUPS_A_LAUNCH):
            gemm4(x, part, out, swiglu=swiglu, bias=bias, group_offsets=group_offsets[g:g + part.G + 1], act=act, act_param=act_param, any_rows=any_rows, status=status)
        return out
    L, stream, read_on = _lib or lib(), core._stream(), w.read_on
    early = read_on is None or stream in read_on
    pc, ps = w.pointers
    # Few rows stream the weights through registers, more go to the tensor core, whose tiles cost the same for 16 rows as for 100.  (us, this way / the
    # other: 17 rows of 6,144 x 2,048 7.3 / 10.2, 24 8.4 / 10.3, 32 in passes of 24 16 / 10.5; of 2,048 x 5,632 10.2 / 11.5, 12.0 / 11.5; of a pair
    # 11,264 x 2,048 9.8 / 15.3, 10.2 / 15.4; of 40,960 x 2,048 20.9 / 38.2, 21.4 / 38.2.  60 experts of a pair 2,816 x 2,048 at 14 rows an expert 79 / 98, at 16 93 / 99; of 2,048 x 1,408 50 / 51, 57 / 51.)
    few = M <= (FEW_ROWS if po is None else GROUP_FEW_ROWS * w.G)
    if any_rows and (K % 8 or ldx % 8 or x.data_ptr() % 16) and not (few and (po is None or _holds_rows(K, w.group, False))):
        few, ldx = False, (K + 7) // 8 * 8           # (as many blocks and groups of k as before: the weight's elements there are zeros)
        whole = torch.zeros(M, ldx, dtype=_BF16, device=x.device)
        whole[:, :K] = x
        x, K = whole, ldx
    done = -1
    for form in (few, not few):            # (what one does not take, -1, the other may)
        if form:
            done = L.moe_gemm_q4(x.data_ptr(), ldx, M, pc, ps, w.G, w.N, K, w.group, w.pair, out.data_ptr(), out.dtype is _BF16, ldo, pb, po,
                                 code, act_param, early, st, stream)
        else:
            done = L.moe_gemm_q4_tc(x.data_ptr(), ldx, M, pc, ps, w.G, w.N, K, w.group, w.pair, out.data_ptr(), out.dtype is _BF16, ldo, pb,
                                    po, code, act_param, 1 if po is not None else _splits(M, N, w, place), early, st, stream)
        if done != -1:
            core._ok(done, "gemm4")
            if not early:
                _have_read(stream, w)
            return out
    raise core.KernelError("gemm4: a stack of K beyond 5,500 or so with rows that are no whole 16-byte units (any_rows copies them)")


def _splits(M: int, N: int, w: Weight4, place: int) -> int:
    """K splits of a tensor-core product whose tiles (128 features, 64 of a pair, and up to 256 rows) leave SMs without work: four or two where a cluster
    of that size finds room for every tile at once, 4 blocks of 64 k and more each.  (us, none / 2 / 3 / 4 / 8: 113 rows of 2,048 x 5,632, 16 tiles, 34.8 /
    20.8 / - / 13.0 / 20.5; 32 rows of 6,144 x 2,048, 48 tiles, 13.4 / 10.4 / 16.6 / 14.8 / 26.2: clusters of three or eight leave SMs of a GPC unused,
    and what does not fit at once takes a second round.)"""
    tiles, sms, blocks = -(-M // 256) * -(-N // (64 if w.pair else 128)), tc.num_sms(place), -(-w.K // 64)
    for splits in (4, 2):
        if tiles * splits <= sms * 9 // 10 and blocks >= 4 * splits:
            return splits
    return 1


@functools.lru_cache(maxsize=None)
def _holds_rows(K: int, group: int, layer: bool) -> bool:
    """Whether shared memory holds what groups of few rows (``layer``: a layer of experts) need of rows so long."""
    return bool((_lib or lib()).moe_q4_holds_rows(K, group, layer))


def takes_experts(tokens: int, top_k: int, gate_up: Weight4) -> bool:
    """Whether ``experts4`` takes so many tokens and picks through these experts."""
    return tokens <= EXPERTS_TOKENS and gate_up.G <= GROUPS_A_LAUNCH and tokens * top_k <= 128 and _holds_rows(gate_up.K, gate_up.group, True)


def experts4(x: torch.Tensor, topk_idx: torch.Tensor, topk_w: torch.Tensor, gate_up: Weight4, down: Weight4, out: torch.Tensor, *,
             shared_gate_up: Optional[Weight4] = None, shared_down: Optional[Weight4] = None, shared_gate: Optional[torch.Tensor] = None,
             status=None) -> bool:
    """A layer of routed experts for up to 8 tokens, in two launches:

        out_t = sum_j w_tj down_e(silu(gate_e x_t) * (up_e x_t)) + gate_t shared(x_t),   e = idx_tj

    x: bfloat16 [T, H]; topk_idx int32 and topk_w float32 [T, k]; gate_up: a pair's stack [E, 2 I, H], down: [E, H, I]; the shared expert's two
    likewise without the stack, shared_gate float32 [T] (None: 1); out: float32 or bfloat16 [T, H].  An index of -1 is no pick
    (all of a row's: zeros but for the shared expert), any other outside [0, E) is reported through ``status`` and taken for none.  False, with
    nothing launched, for what ``takes_experts`` says no to: more tokens, more than 1,024 experts or 128 picks, or rows that shared memory does not hold (H beyond
    6,000 or so)."""
    place = x.get_device()
    _here(place, "experts4")
    T, H, ldx = _matrix(x, place, "x", False)
    rows, columns, ldo = _matrix(out, place, "out", True)
    E, size, k = gate_up.G, gate_up.N // 2, topk_idx.shape[-1] if topk_idx.dim() == 2 else 0
    if (not gate_up.pair or down.pair or gate_up.K != H or down.G != E or down.N != H or down.K != size or rows != T or columns != H
            or topk_idx.shape != (T, k) or topk_w.shape != (T, k) or gate_up.place != place or down.place != place or not k):
        raise core.KernelError(f"experts4: shapes x{tuple(x.shape)} gate_up{gate_up.shape} down{down.shape} picks{tuple(topk_idx.shape)} "
                               f"weights{tuple(topk_w.shape)} out{tuple(out.shape)}")
    group, shared, s = gate_up.group, 0, (None, None, None, None)
    if (shared_gate_up is None) != (shared_down is None) or (shared_gate is not None and shared_down is None):
        raise core.KernelError("experts4: the shared expert is a pair and its down projection, its gate goes with them")
    if shared_gate_up is not None:
        shared, s = shared_gate_up.N // 2, shared_gate_up.pointers + shared_down.pointers
        if (not shared_gate_up.pair or shared_down.pair or shared_gate_up.shape != (2 * shared, H) or shared_down.shape != (H, shared)
                or shared_gate_up.place != place or shared_down.place != place):
            raise core.KernelError(f"experts4: shapes of the shared expert {shared_gate_up.shape} {shared_down.shape}, on {x.device}")
        if shared_gate_up.group != group or shared_down.group != group:
            group = -1
    if down.group != group:
        raise core.KernelError("experts4: the weights of a layer have one group size")
    pi, pw = _on(topk_idx, place, "topk_idx", torch.int32), _on(topk_w, place, "topk_w", torch.float32)
    pg, ps = _on(shared_gate, place, "shared_gate", torch.float32, T), None if status is None else _status(status, place)
    if not takes_experts(T, k, gate_up):
        return False
    if not T:
        return True
    L, stream = _lib or lib(), core._stream()
    weights = (gate_up, down) if shared_gate_up is None else (gate_up, down, shared_gate_up, shared_down)
    early = True
    for w in weights:
        early = early and (w.read_on is None or stream in w.read_on)
    slots = min(T * k, E)
    scratch = torch.empty((slots * -(-size // 64) + -(-shared // 64)) * 3072, dtype=torch.uint8, device=x.device)
    code = L.moe_experts_q4(x.data_ptr(), ldx, T, H, pi, pw, k, E, size, *gate_up.pointers, *down.pointers, shared, *s, pg, group, scratch.data_ptr(),
                            scratch.numel(), out.data_ptr(), out.dtype is _BF16, ldo, early, ps, stream)
    core._ok(code, "experts4")
    if not early:
        _have_read(stream, *weights)
    core.launches += 1            # (two kernels)
    return True
