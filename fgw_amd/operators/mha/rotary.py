"""Rotary positions of query and key heads (no reference counterpart: the reference's operator
takes Q and K as they are).

A pair (a, b) of a row at position p becomes

  a' = s (a cos t - b sin t),   b' = s (b cos t + a sin t),   t = p w_i,

for the pairs of the first `dim` dims of each head, (i, i + dim / 2) or, interleaved,
(2 i, 2 i + 1), with w_i = base ** (-2 i / dim), scaled for long contexts as Rotary says; s is 1
but for "yarn". Frequencies are kept as 64-bit fractions of a turn, so that positions of any size
(int32 or int64, negative ones too) keep all their digits; products and sums are fp32, each result
is rounded once to the rows' type.

apply_rotary rotates rows on their own, and is differentiable; mha_paged_append (paged_extend.py)
rotates on the way into the paged cache.
"""
from __future__ import annotations

import math

import torch

from fgw_amd import _lib

_kv = _lib.load_kv_module()

SCALINGS = {  # kind -> (required, optional with their values)
    "linear": (("factor",), {}),
    "base": (("factor",), {}),
    "yarn": (("factor", "original"), {"beta_fast": 32.0, "beta_slow": 1.0, "attention": None}),
    "bands": (("factor", "original"), {"low": 1.0, "high": 4.0}),
}


def _scaling(scaling):
    if scaling is None:
        return None, {}
    options = dict(scaling)
    kind = options.pop("kind", None)
    if kind not in SCALINGS:
        raise ValueError(f"scaling kind must be one of {', '.join(SCALINGS)}")
    required, optional = SCALINGS[kind]
    unknown = set(options) - set(required) - set(optional)
    if unknown or any(name not in options for name in required):
        raise ValueError(f"{kind} scaling takes {', '.join(required)}"
                         + (f" and optionally {', '.join(optional)}" if optional else ""))
    options = {**optional, **options}
    for name, value in options.items():
        if value is not None and not (math.isfinite(value) and value > 0):
            raise ValueError(f"scaling {name} must be positive and finite")
    return kind, options


def rotary_frequencies(dim, base=10000.0, scaling=None):
    """(w_0 .. w_(dim/2 - 1) in radians a position, s), in 64 bits.

    scaling None, or a dict of kind and its values; L = original context, f = factor:
      linear  w / f
      base    base * f ** (dim / (dim - 2)) for base (dim > 2)
      yarn    w / f for the slow pairs, w for the fast ones, and a ramp over the pair's index i
              from low = floor(d(beta_fast)) to high = ceil(d(beta_slow)), d(n) = dim ln(L / (2 pi
              n)) / (2 ln base), the index that makes n turns in L; s = attention, or
              0.1 ln f + 1 (1 for f <= 1)
      bands   by n = L w / (2 pi), the turns in L: w / f up to n = low, w from n = high on, and
              between them (1 - r) w / f + r w with r = (n - low) / (high - low)
    """
    if dim <= 0 or dim % 16:
        raise ValueError("rotated dims must be a positive multiple of 16")
    if not (math.isfinite(base) and base > 1.0):
        raise ValueError("the base must be finite and above 1")
    kind, o = _scaling(scaling)
    if kind == "base":
        base = base * o["factor"] ** (dim / (dim - 2))
    freqs = [base ** (-2.0 * i / dim) for i in range(dim // 2)]
    if kind == "linear":
        return [w / o["factor"] for w in freqs], 1.0
    if kind == "bands":
        if o["high"] <= o["low"]:
            raise ValueError("scaling high must be above low")
        out = []
        for w in freqs:
            r = (o["original"] * w / (2 * math.pi) - o["low"]) / (o["high"] - o["low"])
            r = min(max(r, 0.0), 1.0)
            out.append((1 - r) * w / o["factor"] + r * w)
        return out, 1.0
    if kind == "yarn":
        def index(turns):
            return dim * math.log(o["original"] / (2 * math.pi * turns)) / (2 * math.log(base))
        low = max(math.floor(index(o["beta_fast"])), 0)
        high = min(math.ceil(index(o["beta_slow"])), dim - 1)
        out = []
        for i, w in enumerate(freqs):
            slow = min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
            out.append(w / o["factor"] * slow + w * (1 - slow))
        scale = o["attention"]
        if scale is None:
            scale = 0.1 * math.log(o["factor"]) + 1.0 if o["factor"] > 1.0 else 1.0
        return out, scale
    return freqs, 1.0


class Rotary:
    """The frequencies of a model's rotary positions on one GPU, built once and kept.

    dim: rotated dims of a head (a multiple of 16, at most the head dim); interleaved: pairs
    (2 i, 2 i + 1) instead of (i, i + dim / 2); base and scaling as in rotary_frequencies.
    turns [dim / 2] int64 holds w_i / (2 pi) in units of 2^-64, modulo a turn.
    """

    def __init__(self, dim, *, base=10000.0, interleaved=False, scaling=None, device=None):
        freqs, self.scale = rotary_frequencies(dim, base, scaling)
        self.dim = dim
        self.interleaved = bool(interleaved)
        whole = 1 << 64
        turns = [round(w / (2 * math.pi) * whole) % whole for w in freqs]
        turns = [t - whole if t >= whole // 2 else t for t in turns]  # the same 64 bits, as int64
        self.turns = torch.tensor(turns, dtype=torch.int64, device="cuda" if device is None else device)


class _Rotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, rotary, inverse):
        ctx.save_for_backward(positions)
        ctx.save_for_forward(positions)
        ctx.rotary, ctx.inverse = rotary, inverse
        return _rotate(x, positions, rotary, inverse, None)

    @staticmethod
    def backward(ctx, grad):
        # The map is s times a rotation: its transpose is the same with the angle reversed.
        positions, = ctx.saved_tensors
        return apply_rotary(_aligned(grad), positions, ctx.rotary, inverse=not ctx.inverse), None, None, None

    @staticmethod
    def jvp(ctx, tangent, *_):
        positions, = ctx.saved_tensors
        return apply_rotary(_aligned(tangent), positions, ctx.rotary, inverse=ctx.inverse)


def _aligned(x):
    """x as rows that the kernel takes: gradients and tangents come with any strides."""
    if (x.stride(-1) != 1 or x.data_ptr() % 16
            or any(n % (16 // x.element_size()) for n in x.stride()[:-1])):
        return x.clone(memory_format=torch.contiguous_format)
    return x


def _rotate(x, positions, rotary, inverse, out):
    return _kv.rotate(x, positions, rotary.turns, rotary.dim, rotary.interleaved, rotary.scale, inverse,
                      out)


def apply_rotary(x, positions, rotary, *, inverse=False, out=None):
    """Rows x [T, H, D] (FP16, BF16 or FP32) rotated to positions [T] (int32 or int64).

    x may have any strides that are multiples of 16 bytes, its last dim contiguous. inverse turns
    the other way: the transpose of the forward, so its gradient. Returns a new contiguous tensor,
    or out ([T, H, D], x itself for in place, else memory apart from x and positions). Differentiable
    in x, twice too, and in forward mode; out is for calls that record no gradient, and requires none.
    A backward pass can be captured into a HIP graph like any of torch's, while no eager graph of the
    same leaves lives.
    """
    if not isinstance(rotary, Rotary):
        raise TypeError("rotary must be a Rotary")
    if isinstance(x, torch.Tensor) and (x.requires_grad and torch.is_grad_enabled() or _kv.has_tangent(x)):
        if out is not None:
            raise ValueError("out cannot be given where a gradient is recorded")
        return _Rotate.apply(x, positions, rotary, bool(inverse))
    return _rotate(x, positions, rotary, bool(inverse), out)
