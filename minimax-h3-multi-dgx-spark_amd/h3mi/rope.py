"""q/k RMSNorm + split-half rotary embedding, in place, and rotary positions of any
layout from the positions themselves (HIP, gfx950).

rms_rope_split_half_ stands in for comfy-kitchen's ck.rms_rope_split_half_ / rms_rope_split_half as
the reference calls them on the attention's q and k
(comfyui_nodes/minimax-h3-sp/minimax_sp/sp_forward.py:279-296): q, k
[1, s, heads, dim] views of the qkv projection, rope_freqs from
rope_rotation_table (:548) with rot_dim = rope_freqs.shape[-3] * 2.  Each
(token, head) row becomes the eager F.rms_norm of the row followed by the
split-half rotation: the pair (y[i], y[i + rot/2]) times the token's 2 x 2
table entry i, in fp32, rounded to bf16.

rotary_ and rotary have no counterpart in the reference, whose tables come from the host
program: they take the tokens' positions, as kv_extend_ gives them, and the pairs'
frequencies (rotary_frequencies), turn split halves or interleaved pairs of all or a
part of each head, and turn back.
"""
import ctypes
import math

import torch
from torch.autograd import forward_ad

from ._lib import RSQRT_HW, RSQRT_RN, RopeRowsC, _fast, check, lib, ptr, same_gpu, stream_of, wrote

_MODES = {"hw": RSQRT_HW, "rn": RSQRT_RN}


def _rows(t, name):
    if t.dtype != torch.bfloat16 or not t.is_cuda:
        raise ValueError(f"{name} must be a bfloat16 GPU tensor")
    if t.dim() == 4:
        if t.shape[0] != 1:
            raise ValueError(f"{name}: batch dimension must be 1")
        t = t[0]
    if t.dim() != 3:
        raise ValueError(f"{name} must be [1, s, heads, dim] or [s, heads, dim]")
    S, H, D = t.shape
    if t.stride(2) != 1 or (H > 1 and t.stride(1) != D):
        raise ValueError(f"{name}: heads must be contiguous (strides [*, dim, 1])")
    return t, S, H, D, t.stride(0) if S > 1 else H * D


def rms_rope_split_half_(q, k, rope_freqs, qw, kw, epsilon=1e-6, rot_dim=None, rsqrt="hw", rstd_out=None):
    """In place on q and k; returns (q, k).  rope_freqs: [..., s, rot/2, 2, 2]
    bf16 (leading singleton dimensions allowed), or None with rot_dim 0."""
    if rsqrt == "hw" and rstd_out is None:
        r = _fast.rms_rope_(q, k, rope_freqs, qw, kw, epsilon, rot_dim)
        if r is not None:
            return r
    q3, S, H, D, ldq = _rows(q, "q")
    k3, Sk, Hk, Dk, ldk = _rows(k, "k")
    if (Sk, Hk, Dk) != (S, H, D):
        raise ValueError("q and k must have the same [s, heads, dim]")
    if rot_dim is None:
        rot_dim = 0 if rope_freqs is None else rope_freqs.shape[-3] * 2
    tab = None
    if rot_dim:
        if rope_freqs is None or rope_freqs.dtype != torch.bfloat16 or not rope_freqs.is_cuda:
            raise ValueError("rope_freqs must be a bfloat16 GPU tensor")
        if tuple(rope_freqs.shape[-4:]) != (S, rot_dim // 2, 2, 2) or any(d != 1 for d in rope_freqs.shape[:-4]):
            raise ValueError(f"rope_freqs must be [.., {S}, {rot_dim // 2}, 2, 2]")
        tab = rope_freqs.contiguous()
    for w, name in ((qw, "qw"), (kw, "kw")):
        if w.dtype != torch.bfloat16 or not w.is_cuda or w.numel() != D or not w.is_contiguous():
            raise ValueError(f"{name} must be a contiguous bfloat16 GPU tensor of {D} elements")
    if rstd_out is not None and (rstd_out.dtype != torch.float32 or rstd_out.numel() != S * 2 * H
                                 or not rstd_out.is_contiguous()):
        raise ValueError("rstd_out must be contiguous float32 with s * 2 * heads elements")
    same_gpu(q3, k=k3, rope_freqs=tab, qw=qw, kw=kw, rstd_out=rstd_out)
    check(lib.h3mi_rms_rope_split_half_bf16(ptr(q3), ptr(k3), ptr(tab) if tab is not None else None, ptr(qw), ptr(kw),
                                            S, H, D, ldq, ldk, rot_dim, float(epsilon), _MODES[rsqrt],
                                            ptr(rstd_out) if rstd_out is not None else None, stream_of(q3)))
    wrote(q, k, rstd_out)
    return q, k


def rms_rope_split_half(q, k, rope_freqs, qw, kw, epsilon=1e-6, rot_dim=None, rsqrt="hw"):
    """Out-of-place form (the reference's in_training branch): returns new (q, k)."""
    qo = q.contiguous().clone()
    ko = k.contiguous().clone()
    return rms_rope_split_half_(qo, ko, rope_freqs, qw, kw, epsilon, rot_dim, rsqrt)


def rotary_frequencies(rot_dim, base=10000.0, scaling=None, factor=1.0, window=8192, device="cuda"):
    """(freqs fp64 [rot_dim / 2], amplitude) for rotary_ and rotary: base ** (-2 i / rot_dim) radians a token, and 1.

    scaling, for contexts of `factor` (>= 1) times the `window` tokens that the frequencies were made for:
      "linear"  positions count for 1 / factor: all frequencies are divided by it
      "ntk"     the base grows by factor ** (rot_dim / (rot_dim - 2)): the slowest pair is divided by factor, the fastest stays
      "yarn"    pairs that turn once in the window or less are divided by factor, those that turn 32 times and more stay; in between
                the share that stays falls evenly with a pair's index, from the last whole index of 32 turns or more to the first
                of one or less.  The amplitude is 1 + 0.1 ln factor.  (Amplitude and both bounds: Peng et al., 2023.  Their share
                falls evenly with the number of turns; by the index is how checkpoints with such configurations are run.)"""
    rot_dim, base, factor = int(rot_dim), float(base), float(factor)
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError("rot_dim must be even and at least 2")
    if not (base > 1.0 and math.isfinite(base)) or not (factor >= 1.0 and math.isfinite(factor)) or not 0 < window < math.inf:
        raise ValueError("base must be above 1, factor at least 1 and window above 0, all of them finite")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError("scaling must be None, 'linear', 'ntk' or 'yarn'")
    if scaling == "ntk" and rot_dim > 2:
        base *= factor ** (rot_dim / (rot_dim - 2))
    i = torch.arange(rot_dim // 2, dtype=torch.float64)
    f, amplitude = base ** (-2.0 * i / rot_dim), 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn" and factor > 1.0:
        def at(turns):  # the pair, as a real number, that turns so often in the window
            return rot_dim * math.log(window / (2 * math.pi * turns)) / (2 * math.log(base))
        lo, hi = math.floor(at(32.0)), math.ceil(at(1.0))  # lo < hi: a pair of 32 turns is before one of a single turn
        keep = 1 - ((i - lo) / (hi - lo)).clamp(0, 1)
        f, amplitude = f * (keep + (1 - keep) / factor), 1 + 0.1 * math.log(factor)
    return f.to(device), amplitude


def _turned(x, positions, dim, name):
    """(rows, heads, token stride, sequence stride) of [n, rows, heads, dim]."""
    if x.dtype != torch.bfloat16 or x.dim() != 4:
        raise ValueError(f"{name} must be bfloat16 [n, rows, heads, dim]")
    if tuple(x.shape[:2]) != tuple(positions.shape) or x.shape[3] != dim:
        raise ValueError(f"{name} must be [{positions.shape[0]}, {positions.shape[1]}, heads, {dim}]")
    n, rows, h, d = x.shape
    if x.numel() and (x.stride(3) != 1 or (h > 1 and x.stride(2) != d)):
        raise ValueError(f"{name}: heads must be contiguous (strides [*, *, dim, 1])")
    if torch.is_grad_enabled() and x.requires_grad:
        raise RuntimeError("rotary records no gradient: call it under torch.no_grad() (a gradient is turned by rotary with inverse=True)")
    if forward_ad.unpack_dual(x).tangent is not None:
        raise RuntimeError("rotary has no forward-mode gradient: call it with the primal tensors")
    return h, x.stride(1) if rows > 1 else h * d, x.stride(0) if n > 1 else rows * h * d


def _rotary(q, k, positions, freqs, interleaved, inverse, amplitude, in_place):
    if positions.dim() != 2 or positions.dtype != torch.int32 or not positions.is_contiguous():
        raise ValueError("positions must be contiguous int32 [n, rows]")
    if freqs.dim() != 1 or freqs.dtype != torch.float64 or not freqs.is_contiguous():
        raise ValueError("freqs must be contiguous float64 [rot / 2]")
    if q.dim() != 4:
        raise ValueError("q must be bfloat16 [n, rows, heads, dim]")
    (n, rows), dim, outs, sides = positions.shape, q.shape[3], [], []
    for x, name in ((q, "q"), (k, "k")):
        if x is None:
            outs.append(None), sides.append(None)
            continue
        h, ld, bs = _turned(x, positions, dim, name)
        same_gpu(positions, **{name: x, "freqs": freqs})
        out = x if in_place else torch.empty(x.shape, dtype=torch.bfloat16, device=x.device)
        outs.append(out)
        sides.append(RopeRowsC(x.data_ptr(), out.data_ptr(), h, ld, bs, *((ld, bs) if in_place else (h * dim, rows * h * dim))))
    if positions.numel() and any(x is not None and x.shape[2] == 0 for x in (q, k)):
        raise ValueError("q and k must have heads")
    with torch.cuda.device(positions.device):
        check(lib.h3mi_rope_bf16(ctypes.byref(sides[0]), None if k is None else ctypes.byref(sides[1]), ptr(positions), ptr(freqs), n, rows,
                                 dim, 2 * freqs.numel(), int(bool(interleaved)), int(bool(inverse)), float(amplitude), stream_of(positions)))
    if in_place:
        wrote(q, k)
    return tuple(outs)


def rotary_(q, k, positions, freqs, interleaved=False, inverse=False, amplitude=1.0):
    """Rotary positions, in place on q and k (k may be None); returns (q, k).

    q, k bf16 [n, rows, heads, dim], each with its own number of heads, views of a projection's output serve; positions int32
    [n, rows], freqs fp64 [rot / 2] radians a token (rotary_frequencies).  The first rot elements of each head are turned, pairs
    (i, i + rot / 2) or, interleaved, (2 i, 2 i + 1): by position times frequency, formed in 64 bits, and scaled by amplitude.
    inverse turns back, with the same amplitude: the transpose, which a gradient goes through.  Rows at a position below 0,
    and the elements from rot on, are left as they are."""
    done = _fast.rotary(q, k, positions, freqs, interleaved, inverse, amplitude, True)
    return done if done is not None else _rotary(q, k, positions, freqs, interleaved, inverse, amplitude, True)


def rotary(q, k, positions, freqs, interleaved=False, inverse=False, amplitude=1.0):
    """rotary_ into new tensors; returns them."""
    done = _fast.rotary(q, k, positions, freqs, interleaved, inverse, amplitude, False)
    return done if done is not None else _rotary(q, k, positions, freqs, interleaved, inverse, amplitude, False)
