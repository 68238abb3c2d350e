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
from typing import Optional

import torch


def frequencies(rotary_dim: int, theta: float, scaling: Optional[dict] = None):
    """(w_i in radians per position as a list of floats, magnitude of the rotated elements)."""
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
    if kind == "ntk":
        theta = theta * factor ** (half / (half - 1))
    w = [theta ** (-i / half) for i in range(half)]
    if kind == "linear":
        return [x / factor for x in w], 1.0
    if kind != "yarn":
        return w, 1.0
    length = opts.get("original_length")
    fast, slow = float(opts.get("fast", 32.0)), float(opts.get("slow", 1.0))
    if not length or not length > 0 or not fast > 0 or not slow > 0:
        raise ValueError("yarn needs original_length, fast and slow > 0")

    def at(turns):  # the pair that turns so often in the original length
        return half * math.log(length / (turns * 2 * math.pi)) / math.log(theta)

    lo, hi = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), rotary_dim - 1)
    ramp = [min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0) for i in range(half)]
    magnitude = opts.get("magnitude")
    if magnitude is None:
        magnitude = 0.1 * math.log(factor) + 1.0
    return [x * (1 - r) + x / factor * r for x, r in zip(w, ramp)], float(magnitude)


class RotaryPlan:
    """Frequencies of one head geometry on one device, made once.

    ``layout`` "half" pairs elements (i, i + rotary_dim / 2), "interleaved" (2 i, 2 i + 1);
    ``rotary_dim`` (None: head_dim) elements of a head turn, the rest passes through.  The
    frequencies are held in 64-bit fixed point as turns per position (2^64 = one turn), so
    that angles stay exact at positions in the millions."""

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
        self.radians, self.magnitude = frequencies(rotary_dim, float(theta), scaling)
        fixed = [round(w / (2 * math.pi) * 2.0 ** 64) % (1 << 64) for w in self.radians]
        self.freqs = torch.tensor([f - (1 << 64) if f >= 1 << 63 else f for f in fixed],
                                  dtype=torch.int64, device=device)
        self.known_calls = {}  # of ops.rotary
