"""Frequencies of rotary positions (the plan that :func:`b200fp8.ops.rotary` takes).

Pair i of the ``rotary_dim / 2`` pairs turns by ``w_i = theta ** (-2 i / rotary_dim)`` radians
per position.  For contexts longer than a model was trained on the frequencies are stretched:

  {"kind": "linear", "factor": s}   w_i / s
  {"kind": "ntk", "factor": s}      theta * s ** (rotary_dim / (rotary_dim - 2)) as theta
  {"kind": "yarn", "factor": s, "original_length": n, "fast": 32, "slow": 1, "magnitude": None}
      pairs that turn more than ``fast`` times in ``n`` positions keep w_i, those that turn less
      than ``slow`` times get w_i / s, with a ramp linear in i between (its ends rounded outwards to
      whole i, and cut off at 0 and rotary_dim - 1: it may end behind the last pair); rotated
      elements are multiplied by ``magnitude`` (None: 0.1 ln s + 1)  [Peng et al., "YaRN", 2023]
"""
from __future__ import annotations

import math
from decimal import Context, Decimal, localcontext
from typing import List, Optional, Tuple

import torch


# Frequencies are computed in whole multiples of 2^-192, which _DIGITS decimal digits hold.
_BITS, _DIGITS = 192, 70
_TWO_PI = Decimal("6.2831853071795864769252867665590057683943387987502116419498891846156328125724")
with localcontext(Context(prec=_DIGITS)):
    _TURNS = int((1 << _BITS) / _TWO_PI)  # of a radian


def _exact(rotary_dim: int, theta: float, scaling: Optional[dict]) -> Tuple[List[int], float]:
    half = rotary_dim // 2
    opts = dict(scaling or {"kind": "none"})
    kind = opts.pop("kind", None)
    known = {"none": (), "linear": ("factor",), "ntk": ("factor",),
             "yarn": ("factor", "original_length", "fast", "slow", "magnitude")}
    if kind not in known:
        raise ValueError(f"unknown scaling kind {kind!r}")
    if set(opts) - set(known[kind]):
        raise ValueError(f"scaling {kind!r} has no {sorted(set(opts) - set(known[kind]))}")
    factor = float(opts.get("factor", 1.0))
    if kind != "none" and "factor" not in opts or not factor > 0 or not math.isfinite(factor):
        raise ValueError("scaling needs a factor > 0")
    with localcontext(Context(prec=_DIGITS)):
        log_theta = Decimal(float(theta)).ln()
        if kind == "ntk":
            log_theta += Decimal(factor).ln() * half / (half - 1)
        step = int((-log_theta / half).exp() * (1 << _BITS))
    w = [1 << _BITS]
    while len(w) < half:  # half <= 128 products, each cut off by less than 2^-192
        w.append(w[-1] * step >> _BITS)
    num, den = factor.as_integer_ratio()
    if kind == "linear":
        return [x * den // num for x in w], 1.0
    if kind != "yarn":
        return w, 1.0
    length = opts.get("original_length")
    fast, slow = float(opts.get("fast", 32.0)), float(opts.get("slow", 1.0))
    if not length or not length > 0 or not fast > 0 or not slow > 0:
        raise ValueError("yarn needs original_length, fast and slow > 0")

    def at(turns):  # the pair that turns so often in the original length
        return half * math.log(length / (turns * 2 * math.pi)) / math.log(theta)

    lo, hi = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), rotary_dim - 1)
    span = max(hi - lo, 1)
    ramp = [min(max(i - lo, 0), span) for i in range(half)]  # of the span
    magnitude = opts.get("magnitude")
    if magnitude is None:
        magnitude = 0.1 * math.log(factor) + 1.0
    return [(x * (span - r) + x * den // num * r) // span for x, r in zip(w, ramp)], float(magnitude)


def frequencies(rotary_dim: int, theta: float, scaling: Optional[dict] = None):
    """(w_i in radians per position as a list of floats, magnitude of the rotated elements)."""
    w, magnitude = _exact(rotary_dim, theta, scaling)
    return [x / (1 << _BITS) for x in w], magnitude


class RotaryPlan:
    """Frequencies of one head geometry on one device, made once.

    ``layout`` "half" pairs elements (i, i + rotary_dim / 2), "interleaved" (2 i, 2 i + 1);
    ``rotary_dim`` (None: head_dim) elements of a head turn, the rest passes through.  The
    frequencies are held in 64-bit fixed point as turns per position (2^64 = one turn), rounded
    once from their exact values: an angle is off by 2^-65 of a turn a position, 2^-34 of a turn
    at position 2^31."""

    def __init__(self, head_dim: int, *, rotary_dim: Optional[int] = None, theta: float = 1e4,
                 layout: str = "half", scaling: Optional[dict] = None, device="cuda"):
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if head_dim % 8 or not 8 <= head_dim <= 256:
            raise ValueError("head_dim must be a multiple of 8 up to 256")
        if rotary_dim % 8 or not 8 <= rotary_dim <= head_dim:
            raise ValueError("rotary_dim must be a multiple of 8 up to head_dim")
        if layout not in ("half", "interleaved"):
            raise ValueError("layout must be 'half' or 'interleaved'")
        if not theta > 1 or not math.isfinite(theta):
            raise ValueError("theta must be > 1")
        self.head_dim, self.rotary_dim, self.theta = head_dim, rotary_dim, float(theta)
        self.interleaved = layout == "interleaved"
        w, self.magnitude = _exact(rotary_dim, float(theta), scaling)
        self.radians = [x / (1 << _BITS) for x in w]
        # w / (2 pi) at twice the bits, rounded to 64
        cut = 2 * _BITS - 64
        fixed = [(x * _TURNS + (1 << cut - 1) >> cut) % (1 << 64) for x in w]
        self.freqs = torch.tensor([f - (1 << 64) if f >= 1 << 63 else f for f in fixed],
                                  dtype=torch.int64, device=device)
        self.known_calls = {}  # of ops.rotary
