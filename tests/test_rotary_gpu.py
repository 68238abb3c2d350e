"""b2f_rotary against the 64-bit oracle.

Tolerance of an element: half a step of the output type (eps / 2 of the value), and for the f32
work in front of it 2^-20 of the pair's magnitude: the angle is off by 2^-25 of a turn at most
(its 32-bit fraction rounded to f32), 2^-22.3 in radians; sincospi, two products and a sum are
good for 2^-22 each; the norm adds rsqrt, a sum of head_dim squares and three products (2^-21)."""
from __future__ import annotations

import pytest
import torch

from helpers import gen, randn
from oracle import serving

pytestmark = pytest.mark.gpu

F32, BF16, F16, E4M3 = torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn


def _mods():
    from b200fp8 import ops, rotary
    return ops, rotary


def _pair_size(y, rot, interleaved, head_dim):
    """Magnitude of every element's pair."""
    z = y.unflatten(-1, (-1, head_dim)).clone()
    r = z[..., :rot]
    two = r.unflatten(-1, (-1, 2)) if interleaved else r.unflatten(-1, (2, -1)).transpose(-1, -2)
    size = two.norm(dim=-1, keepdim=True).expand_as(two)
    z[..., :rot] = (size if interleaved else size.transpose(-1, -2)).flatten(-2)
    return z.abs().flatten(1)


def _check(got, want, rot, interleaved, head_dim, out_scale=1.0):
    half = torch.finfo(got.dtype).eps / 2
    tiny = {F32: 2.0 ** -126, BF16: 2.0 ** -126, F16: 2.0 ** -25, E4M3: 2.0 ** -10}[got.dtype]
    value = got.cpu().double() * out_scale
    if got.dtype == E4M3:  # saturates: at 448 / 128 = 3.5 here, which normal values do pass
        want = want.clamp(-448 * out_scale, 448 * out_scale)
    bound = want.abs() * half + _pair_size(want, rot, interleaved, head_dim) * 2.0 ** -20 + \
        tiny * out_scale
    assert bool(((value - want).abs() <= bound).all()), float((value - want).abs().max())


@pytest.mark.parametrize("rows,heads,kv,dim,rot,inter,src,dst,norm,bits", [
    (1, 1, 1, 64, 64, False, BF16, BF16, False, 32),
    (1, 32, 8, 128, 128, False, E4M3, BF16, True, 32),
    (7, 3, 1, 96, 48, False, F32, F32, False, 64),
    (5, 5, 5, 8, 8, True, F16, F16, False, 32),
    (33, 16, 4, 256, 64, False, BF16, E4M3, True, 64),
    (301, 12, 12, 64, 32, True, F16, F32, True, 32),
    (2, 2, 0, 104, 40, True, F32, BF16, False, 32),
    (3000, 7, 1, 128, 128, True, BF16, F16, False, 64),
    (9, 4, 2, 256, 256, True, E4M3, E4M3, True, 32),
    (17, 9, 3, 40, 24, False, F32, E4M3, False, 32),
])
def test_against_64_bits(rows, heads, kv, dim, rot, inter, src, dst, norm, bits):
    ops, rotary = _mods()
    g = gen(rows * 31 + dim)
    plan = rotary.RotaryPlan(dim, rotary_dim=rot, theta=1e6, device="cuda",
                             layout="interleaved" if inter else "half")
    ins = 1 / 64 if src == E4M3 else 1.0
    outs = 1 / 128 if dst == E4M3 else 1.0
    q = (randn((rows, heads * dim), g) / (ins if src == E4M3 else 1)).to(src)
    k = (randn((rows, kv * dim), g) / (ins if src == E4M3 else 1)).to(src) if kv else None
    pos = torch.randint(0, 300000, (rows,), generator=g).to(torch.int32 if bits == 32 else
                                                            torch.int64)
    wq = randn((dim,), g, 0.1) if norm else None
    wk = randn((dim,), g, 0.1) if norm and kv else None
    got = ops.rotary(q.cuda(), None if k is None else k.cuda(), pos.cuda(), plan, heads=heads,
                     kv_heads=kv, in_scale=ins, out_dtype=dst, out_scale=outs,
                     q_weight=None if wq is None else wq.cuda(),
                     k_weight=None if wk is None else wk.cuda())
    assert (got[1] is None) == (kv == 0)
    for x, w, y in ((q, wq, got[0]), (k, wk, got[1])):
        if x is not None:
            want = serving.rotary(x, pos, plan.radians, head_dim=dim, interleaved=inter,
                                  in_scale=ins, weight=w)
            _check(y, want, rot, inter, dim, outs)


@pytest.mark.parametrize("scaling", [
    {"kind": "linear", "factor": 4.0}, {"kind": "ntk", "factor": 4.0},
    {"kind": "yarn", "factor": 16.0, "original_length": 8192},
    {"kind": "yarn", "factor": 2.0, "original_length": 4096, "fast": 16, "slow": 2,
     "magnitude": 1.0}])
def test_stretched_frequencies_at_far_positions(scaling):
    """Positions up to 2^31 - 1 (and negative ones): the angle of 64-bit fixed point holds."""
    ops, rotary = _mods()
    plan = rotary.RotaryPlan(128, theta=1e6, scaling=scaling, device="cuda")
    pos = torch.tensor([0, 1, 131071, 1 << 20, (1 << 31) - 1, -1, -(1 << 20)])
    q = randn((7, 256), gen(5))
    got, _ = ops.rotary(q.cuda(), None, pos.cuda(), plan, heads=2)
    want = serving.rotary(q, pos, plan.radians, head_dim=128, magnitude=plan.magnitude)
    # the oracle's own angle (a 53-bit product) is off by 2^31 2^-53 = 2^-22 radians at the most
    _check(got, want, 128, False, 128)


@pytest.mark.parametrize("inter", [False, True])
def test_inverse_turns_back_and_is_the_transpose(inter):
    ops, rotary = _mods()
    g = gen(8)
    plan = rotary.RotaryPlan(64, rotary_dim=48, theta=1e4, device="cuda",
                             layout="interleaved" if inter else "half",
                             scaling={"kind": "yarn", "factor": 4.0, "original_length": 1024})
    x, y = randn((50, 128), g), randn((50, 128), g)
    pos = torch.randint(0, 5000, (50,), generator=g).cuda()
    fx, _ = ops.rotary(x.cuda(), None, pos, plan, heads=2)
    by, _ = ops.rotary(y.cuda(), None, pos, plan, heads=2, inverse=True)
    a, b = (fx.cpu().double() * y.double()).sum(1), (x.double() * by.cpu().double()).sum(1)
    size = (x.double().norm(dim=1) * y.double().norm(dim=1)) * plan.magnitude
    assert bool(((a - b).abs() <= size * 2.0 ** -19).all())
    back, _ = ops.rotary(fx, None, pos, plan, heads=2, inverse=True)
    want = x.double().unflatten(-1, (2, 64)).clone()
    want[..., :48] *= plan.magnitude ** 2
    assert bool(((back.cpu().double() - want.flatten(1)).abs() <= 2.0 ** -18 * 8).all())


def test_strided_heads_in_place_and_other_stream():
    """Heads of a q | gate projection, k in place of itself, on a stream of its own."""
    ops, rotary = _mods()
    g = gen(9)
    rows, d = 20, 128
    proj = randn((rows, 4 * 2 * d + 16), g).to(BF16)
    k = randn((rows, 2 * d), g).to(BF16)
    pos = torch.arange(rows, dtype=torch.int32) + 77
    plan = rotary.RotaryPlan(d, theta=1e6, device="cuda")
    pc, kc, posc = proj.cuda(), k.cuda(), pos.cuda()
    before = pc.clone()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        q, same = ops.rotary(pc[:, 8:], kc, posc, plan, heads=4, kv_heads=2, q_head_stride=2 * d,
                             k_out=kc)
    s.synchronize()
    assert same.data_ptr() == kc.data_ptr() and torch.equal(pc, before)
    src = proj[:, 8:8 + 8 * d].unflatten(1, (4, 2, d))[:, :, 0].flatten(1)
    _check(q, serving.rotary(src, pos, plan.radians, head_dim=d), d, False, d)
    _check(kc, serving.rotary(k, pos, plan.radians, head_dim=d), d, False, d)


def test_captured_replay_reads_new_positions():
    ops, rotary = _mods()
    plan = rotary.RotaryPlan(64, device="cuda")
    q = randn((6, 128), gen(3)).cuda()
    pos = torch.arange(6, device="cuda", dtype=torch.int32)
    out = torch.empty_like(q)
    ops.rotary(q, None, pos, plan, heads=2, q_out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.rotary(q, None, pos, plan, heads=2, q_out=out)
    pos += 1000
    graph.replay()
    want = serving.rotary(q.cpu(), pos.cpu(), plan.radians, head_dim=64)
    torch.cuda.synchronize()
    _check(out, want, 64, False, 64)


def test_nan_and_infinity_stay_in_their_pair():
    ops, rotary = _mods()
    plan = rotary.RotaryPlan(64, device="cuda")
    q = torch.ones((1, 64))
    q[0, 3], q[0, 10] = float("nan"), float("inf")
    got, _ = ops.rotary(q.cuda(), None, torch.tensor([9], device="cuda"), plan, heads=1)
    bad = (~torch.isfinite(got[0])).nonzero().flatten().tolist()
    assert bad == [3, 10, 35, 42]


@pytest.mark.parametrize("inter", [False, True])
def test_positions_beyond_32_bits(inter):
    """Angles of positions up to 2^40, by the exact frequencies: off by 2^-65 of a turn a position,
    2^-25 of a turn at 2^40, as much as the rounding of the fraction that the tolerance counts."""
    from decimal import Decimal, localcontext
    ops, rotary = _mods()
    g = gen(11)
    plan = rotary.RotaryPlan(64, theta=1e4, device="cuda", layout="interleaved" if inter else "half")
    pos = torch.tensor([1, 1 << 33, -(1 << 36) + 5, (1 << 40) - 1, 987654321987])
    q = randn((5, 64), g)
    got, _ = ops.rotary(q.cuda(), None, pos.cuda(), plan, heads=1)
    with localcontext() as c:
        c.prec = 60
        two_pi = Decimal("6.2831853071795864769252867665590057683943387987502116419498892")
        rest = [[float((p * Decimal(10000) ** (Decimal(-i) / 32)).remainder_near(two_pi))
                 for i in range(32)] for p in pos.tolist()]
    for row, angles in enumerate(rest):
        want = serving.rotary(q[row:row + 1], torch.ones(1), angles, head_dim=64, interleaved=inter)
        _check(got[row:row + 1], want, 64, inter, 64)
