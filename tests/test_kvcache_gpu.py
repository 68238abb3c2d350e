"""The 4-bit paged cache: writing, reading, attention and page bookkeeping against the 64-bit
oracle.

Codes and scales have to be the oracle's, bit for bit: a quotient of 16-bit values is never so
near a border that f32 takes it to the other side.

Attention, element by element: P is rounded to f16 (2^-11 of itself, and 2^-25 * 2^-7 of the
row's largest for the smallest ones), so the sum of p |v| / sum of p, the mass, bounds that part
at 2^-11; scores are f32 sums of exact products, off by 2^-21 of the largest sum of |q k|, which
moves every p by as much; the output is rounded by half a step."""
from __future__ import annotations

import pytest
import torch

from helpers import gen, randn
from oracle import serving

pytestmark = pytest.mark.gpu

F32, BF16, F16, E4M3 = torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn


def _cache(**kw):
    from b200fp8.kvcache import Fp4Cache
    return Fp4Cache(**kw)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _filled(lens, news, *, kv, d, page, g, ks=0.25, vs=0.25, dtype=BF16, layers=1, garbage=False):
    """A cache whose sequences hold random tokens, written in two parts (the last `news` apart)."""
    width = max(1, max(-(-n // page) for n in lens))
    pages = sum(-(-n // page) for n in lens) + 3
    c = _cache(layers=layers, pages=pages, page_size=page, kv_heads=kv, head_dim=d,
               max_seqs=len(lens), max_pages=width, k_scale=ks, v_scale=vs)
    if garbage:  # unused places hold NaN scales
        c.storage.fill_(0xff)
    # pages strewn over the pool
    order = torch.randperm(pages, generator=g).int()
    at = 0
    for b, n in enumerate(lens):
        m = -(-n // page)
        c.table[b, :m] = order[at:at + m].cuda()
        c.refs[order[at:at + m].long().cuda()] = 1
        at += m
    c.lens.copy_(_ints(lens))
    total = sum(lens)
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    k, v = randn((total, kv * d), g).to(dtype), randn((total, kv * d), g).to(dtype)
    if total:
        c.write(k.cuda(), v.cuda(), starts=_ints(starts), layer=layers - 1)
    return c, k, v, starts


def _oracle_kv(c, b, length, layer=0):
    return serving.cached(c.storage[layer].cpu(), c.table[b].cpu(), length, c.page_size,
                          c.head_dim, c.k_scale, c.v_scale)


def _check_attention(c, q, out, lens, starts, heads, *, layer=0, causal=True, q_scale=1.0,
                     sm_scale=None, gate=None, out_scale=1.0, lse=None, rows=None):
    d = c.head_dim
    half = torch.finfo(out.dtype).eps / 2
    tiny = {BF16: 0.0, F16: 2.0 ** -25, E4M3: 2.0 ** -10}[out.dtype]
    for b in range(len(starts) - 1):
        row = b if rows is None else rows[b]
        lo, hi = starts[b], starts[b + 1]
        if lo == hi:
            continue
        k, v = _oracle_kv(c, row, lens[row], layer)
        if lens[row] == 0:
            k = v = torch.zeros((0, c.kv_heads, d), dtype=torch.float64)
        want, l, mass, size = serving.attention(
            q[lo:hi].double().unflatten(-1, (heads, d)) * q_scale, k, v, causal=causal,
            sm_scale=sm_scale, gate=None if gate is None else gate[lo:hi].unflatten(-1, (heads, d)))
        got = out[lo:hi].cpu().double().unflatten(-1, (heads, d)) * out_scale
        if out.dtype == E4M3:  # saturates: at 448 / 256 = 1.75 here, which some values pass
            want = want.clamp(-448 * out_scale, 448 * out_scale)
        bound = mass * (2.0 ** -11 + 2.0 ** -16 + size * 2.0 ** -20) + want.abs() * half + \
            tiny * out_scale
        bad = (got - want).abs() > bound
        assert not bool(bad.any()), (b, float((got - want).abs().max()), float(bound.max()))
        if lse is not None:
            have = lse[lo:hi].cpu().double()
            assert torch.equal(torch.isinf(have), torch.isinf(l))
            fine = ~torch.isinf(l)
            assert bool(((have - l)[fine].abs() <= 2.0 ** -20 * (1 + size + l[fine].abs())).all())


@pytest.mark.parametrize("dtype", [BF16, F16, F32, E4M3])
@pytest.mark.parametrize("d,page,kv", [(64, 16, 1), (128, 32, 3), (256, 64, 2)])
def test_written_codes_and_read_values_are_the_oracles(dtype, d, page, kv):
    g = gen(d + page)
    lens = [1, page, page + 1, 3 * page - 1]
    scale = 0.25 if dtype != F32 else 0.3
    ins = 1 / 64 if dtype == E4M3 else 1.0
    width = 3
    c = _cache(layers=2, pages=12, page_size=page, kv_heads=kv, head_dim=d, max_seqs=4,
               max_pages=width, k_scale=scale, v_scale=2 * scale)
    c.extend(_ints(lens))
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    k = randn((starts[-1], kv * d), g)
    k[0, :16] = 0.0
    k[1, :16] *= 1e-6   # its scale rounds to 0
    k[2, :16] *= 1e6    # saturates
    k[3, 16:32] = torch.arange(16) * 0.25  # values on the borders between codes
    v = randn((starts[-1], kv * d), g) * 3
    k, v = (k / ins).to(dtype), (v / ins).to(dtype)
    if dtype == E4M3:
        k, v = k.float().nan_to_num(448).to(dtype), v.float().nan_to_num(448).to(dtype)
    other = c.storage[0].clone()
    c.write(k.cuda(), v.cuda(), starts=_ints(starts), layer=1, k_in_scale=ins, v_in_scale=ins)
    rk, rv = c.read(starts[-1], starts=_ints(starts), layer=1, dtype=F32)
    torch.cuda.synchronize()
    assert torch.equal(c.storage[0], other)
    f32 = lambda s: float(torch.tensor(s, dtype=F32))  # noqa: E731
    for x, read, s in ((k, rk, f32(scale)), (v, rv, f32(2 * scale))):
        x = (x.float() * ins).unflatten(-1, (kv, d))
        code, s8, value = serving.pack(x, s)
        # scale * k_scale is rounded to f32 once before the code multiplies it
        assert torch.allclose(read.cpu().unflatten(-1, (kv, d)).double(), value, atol=0,
                              rtol=0 if dtype != F32 else 2.0 ** -23)
    for b in range(4):
        kk, _ = _oracle_kv(c, b, lens[b], 1)
        assert torch.allclose(kk.flatten(1), rk[starts[b]:starts[b + 1]].cpu().double(), rtol=2e-7)
    for half in (BF16, F16):
        hk, hv = c.read(starts[-1], starts=_ints(starts), layer=1, dtype=half)
        assert torch.equal(hk, rk.to(half)) and torch.equal(hv, rv.to(half))


def test_nan_and_infinity_on_writing():
    c = _cache(layers=1, pages=1, page_size=16, kv_heads=1, head_dim=64, max_seqs=1, max_pages=1)
    c.extend(_ints([1]))
    k = torch.ones((1, 64))
    k[0, 5], k[0, 20], k[0, 40] = float("nan"), float("inf"), -float("inf")
    c.write(k.cuda(), k.cuda())
    rk, _ = c.read(1, dtype=F32)
    rk = rk.cpu()[0]
    assert bool(torch.isnan(rk[:16]).all()) and bool(torch.isfinite(rk[16:]).all())
    assert float(rk[20]) == 448 * 6 and float(rk[40]) == -448 * 6


def test_rows_behind_the_last_sequence_and_partial_batches():
    """Packed rows outside of the sequences stay as they are; rows names table rows out of order."""
    g = gen(4)
    lens = [20, 7, 40]
    c, _, _, _ = _filled(lens, None, kv=2, d=64, page=16, g=g)
    starts, rows = _ints([2, 5, 6]), [2, 0]
    k, v = randn((9, 128), g).to(BF16), randn((9, 128), g).to(BF16)
    c.write(k.cuda(), v.cuda(), rows=_ints(rows), starts=starts)
    rk = torch.full((9, 128), 7.0, dtype=BF16, device="cuda")
    rv = rk.clone()
    c.read(9, rows=_ints(rows), starts=starts, k=rk, v=rv)
    q = randn((9, 256), g).to(BF16)
    out = torch.full((9, 256), 5.0, dtype=BF16, device="cuda")
    lse = torch.full((9, 4), 3.0, device="cuda")
    c.attention(q.cuda(), heads=4, rows=_ints(rows), starts=starts, out=out, lse=lse)
    torch.cuda.synchronize()
    for i in (0, 1, 6, 7, 8):
        assert bool((rk[i] == 7).all()) and bool((out[i] == 5).all()) and bool((lse[i] == 3).all())
    _, _, want = serving.pack(k[2:6].unflatten(-1, (2, 64)), 0.25)
    assert torch.equal(rk[2:6].cpu().double().unflatten(-1, (2, 64)), want)
    _check_attention(c, q, out, lens, [2, 5, 6], 4, lse=lse, rows=rows)
    from b200fp8 import device_status
    assert device_status() == 0


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("heads,kv", [(1, 1), (8, 2), (16, 1), (5, 1), (40, 2)])
def test_one_token_steps(d, page, heads, kv):
    g = gen(d * page + heads)
    lens = [1, 15, 16, 17, 31, 33, 64, 127, 128, 129, 300, 0]
    c, _, _, _ = _filled(lens, None, kv=kv, d=d, page=page, g=g, garbage=True)
    q = randn((len(lens), heads * d), g).to(BF16)
    out, lse = c.attention(q.cuda(), heads=heads, return_lse=True)
    torch.cuda.synchronize()
    assert bool((out[-1] == 0).all())
    _check_attention(c, q, out, lens, list(range(len(lens) + 1)), heads, lse=lse)


@pytest.mark.parametrize("q_dtype,out_dtype", [(BF16, F16), (F16, BF16), (E4M3, E4M3)])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_several_new_tokens(q_dtype, out_dtype, d, causal):
    """Chunks of new tokens of different lengths, more of them than are cached among them (the
    first ones see nothing), with gate and every type."""
    g = gen(d + causal)
    lens, news = [70, 3, 200, 33, 0, 129], [5, 3, 37, 1, 0, 129]
    c, _, _, _ = _filled(lens, None, kv=2, d=d, page=16, g=g, garbage=True)
    heads = 6
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    qs = 1 / 64 if q_dtype == E4M3 else 1.0
    q = (randn((starts[-1], heads * d), g) / qs).clamp(-440, 440).to(q_dtype)
    gate = (randn((starts[-1], heads * d), g) * 64).clamp(-440, 440).to(E4M3)
    outs = 1 / 256 if out_dtype == E4M3 else 1.0
    out, lse = c.attention(q.cuda(), heads=heads, starts=_ints(starts), causal=causal, q_scale=qs,
                           gate=gate.cuda(), gate_scale=1 / 64, out_dtype=out_dtype,
                           ctx_scale=outs, return_lse=True)
    torch.cuda.synchronize()
    _check_attention(c, q, out, lens, starts, heads, causal=causal, q_scale=qs,
                     gate=gate.float() / 64, out_scale=outs, lse=lse)


def test_more_new_tokens_than_cached():
    """A sequence with fewer cached than new tokens: its first tokens see no key."""
    g = gen(77)
    lens = [4, 50]
    c, _, _, _ = _filled(lens, None, kv=1, d=128, page=16, g=g)
    starts = [0, 30, 40]
    q = randn((40, 2 * 128), g).to(BF16)
    out, lse = c.attention(q.cuda(), heads=2, starts=_ints(starts), return_lse=True)
    torch.cuda.synchronize()
    assert bool((out[:26] == 0).all()) and bool(torch.isinf(lse[:26]).all())
    _check_attention(c, q, out, lens, starts, 2, lse=lse)


def test_long_sequences_are_split_and_joined_the_same_every_time():
    g = gen(12)
    lens = [9000, 40, 3000]
    c, _, _, _ = _filled(lens, None, kv=1, d=128, page=64, g=g)
    q = (randn((3, 4 * 128), g) * 3).to(BF16)
    first, l0 = c.attention(q.cuda(), heads=4, return_lse=True)
    for _ in range(3):
        again, l1 = c.attention(q.cuda(), heads=4, return_lse=True)
        assert torch.equal(first, again) and torch.equal(l0, l1)
    _check_attention(c, q, first, lens, [0, 1, 2, 3], 4, lse=l0)


def test_a_late_large_score_moves_the_maximum():
    """Scores that grow along the sequence by far more than the slack of the running maximum."""
    g = gen(2)
    n, d = 600, 64
    c = _cache(layers=1, pages=40, page_size=16, kv_heads=1, head_dim=d, max_seqs=1, max_pages=40,
               k_scale=1 / 16)
    c.extend(_ints([n]))
    k = randn((n, d), g) * 0.05 + torch.linspace(-4, 4, n)[:, None]
    v = randn((n, d), g)
    c.write(k.to(BF16).cuda(), v.to(BF16).cuda())
    for sign in (1.0, -1.0):
        q = torch.full((1, d), sign).to(BF16)
        out, lse = c.attention(q.cuda(), heads=1, sm_scale=1.0, return_lse=True)
        torch.cuda.synchronize()
        _check_attention(c, q, out, [n], [0, 1], 1, sm_scale=1.0, lse=lse)


@pytest.mark.parametrize("scale", [1e-30, 1e30])
def test_queries_of_any_size(scale):
    """bf16 queries outside the range of f16 lose nothing (sm_scale brings the scores back)."""
    g = gen(6)
    c, _, _, _ = _filled([100], None, kv=1, d=128, page=32, g=g)
    q = (randn((1, 128), g) * scale).to(BF16)
    out = c.attention(q.cuda(), heads=1, sm_scale=1.0 / scale)
    torch.cuda.synchronize()
    _check_attention(c, q, out, [100], [0, 1], 1, sm_scale=1.0 / scale)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_nan_reaches_only_those_who_see_it(d):
    """A NaN in a late token's key or value leaves earlier tokens of the chunk alone, and one in
    another sequence too."""
    for which in ("k", "v"):
        g = gen(d)
        lens = [50, 50]
        c, k, v, starts = _filled(lens, None, kv=1, d=d, page=16, g=g)
        k, v = k.clone(), v.clone()
        (k if which == "k" else v)[45, 3] = float("nan")
        c.write(k.cuda(), v.cuda(), starts=_ints(starts))
        q = randn((20, 2 * d), g).to(BF16)
        out = c.attention(q.cuda(), heads=2, starts=_ints([0, 10, 20]))
        torch.cuda.synchronize()
        clean = torch.isfinite(out).all(1).cpu()
        assert clean.tolist() == [True] * 5 + [False] * 5 + [True] * 10
        assert bool(torch.isnan(out[5:10, :16]).all())
        ok = [i for i in range(20) if clean[i]]
        for b, lo, hi in ((0, 0, 5), (1, 10, 20)):
            kk, vv = _oracle_kv(c, b, 50)
            seen = 45 if b == 0 else 50
            want, _, mass, size = serving.attention(
                q[lo:hi].double().unflatten(-1, (2, d)), kk[:seen], vv[:seen])
            got = out[lo:hi].cpu().double().unflatten(-1, (2, d))
            bound = mass * (2.0 ** -11 + 2.0 ** -16 + size * 2.0 ** -20) + want.abs() * 2.0 ** -8
            assert bool(((got - want).abs() <= bound).all())
        assert len(ok) == 15


def test_bad_lists_are_left_out_and_recorded():
    """Pages and rows out of range lead nowhere: their keys are not attended, their tokens not
    written, and the status word says so."""
    from b200fp8 import device_status
    g = gen(21)
    lens = [64, 40]
    c, _, _, _ = _filled(lens, None, kv=1, d=64, page=16, g=g)
    good = c.table.clone()
    assert device_status(reset=True) == 0
    c.table[0, 1], c.table[0, 2] = c.pages + 5, -1
    q = randn((2, 64), g).to(BF16)
    out = c.attention(q.cuda(), heads=1)
    torch.cuda.synchronize()
    assert device_status(reset=True) == 5
    k, v = serving.cached(c.storage[0].cpu(), good[0].cpu(), 64, 16, 64, 0.25, 0.25)
    keep = [i for i in range(64) if i // 16 not in (1, 2)]
    want, _, mass, size = serving.attention(q[:1].double().unflatten(-1, (1, 64)), k[keep], v[keep])
    err = (out[0].cpu().double() - want.flatten()).abs()
    bound = mass.flatten() * (2.0 ** -11 + 2.0 ** -16 + size * 2.0 ** -20) + want.flatten().abs() * 2.0 ** -8
    assert bool((err <= bound).all())
    before = c.storage.clone()
    x = randn((2, 64), g).to(BF16).cuda()
    c.write(x, x, rows=_ints([7, -3]))
    rk, _ = c.read(2, rows=_ints([7, -3]))
    assert torch.equal(c.storage, before) and bool((rk == 0).all())
    out = c.attention(q.cuda(), heads=1, rows=_ints([9, 1]))
    assert bool((out[0] == 0).all()) and bool((out[1] != 0).any())
    assert device_status(reset=True) == 5
    c.lens[1] = 10000  # more than the table row holds: cut off at what it holds, pages -1 left out
    c.attention(q.cuda(), heads=1)
    c.lens[1] = -4
    out = c.attention(q.cuda(), heads=1)
    assert bool((out[1] == 0).all())
    c.lens[1] = 40
    out = c.attention(q.cuda(), heads=1, starts=_ints([0, 5, 2]))  # not ascending, too far
    torch.cuda.synchronize()
    assert device_status(reset=True) == 5


def test_two_streams_and_two_graphs_do_not_share_work():
    """Two calls at once, and two captured graphs replayed at once, on one cache."""
    g = gen(31)
    lens = [2000, 1500, 7]
    c, _, _, _ = _filled(lens, None, kv=2, d=128, page=32, g=g)
    qs = [(randn((3, 8 * 128), g)).to(BF16).cuda() for _ in range(2)]
    want = [c.attention(q, heads=8) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [torch.empty_like(q) for q in qs]
    for _ in range(5):
        for s, q, o in zip(streams, qs, outs):
            with torch.cuda.stream(s):
                c.attention(q, heads=8, out=o)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    graphs = []
    for q, o in zip(qs, outs):
        o.zero_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            c.attention(q, heads=8, out=o)
        graphs.append(graph)
    for _ in range(5):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_strided_queries_and_outputs():
    g = gen(41)
    lens = [77, 12]
    c, _, _, _ = _filled(lens, None, kv=1, d=64, page=16, g=g)
    wide = randn((2, 3 * 64 + 16), g).to(BF16)
    gate = randn((2, 3 * 80), g).to(BF16)
    hold = torch.full((2, 3 * 64 + 32), 9.0, dtype=F16, device="cuda")
    c.attention(wide.cuda()[:, 16:], heads=3, gate=gate.cuda(), gate_head_stride=80,
                out=hold[:, 16:16 + 192])
    torch.cuda.synchronize()
    assert bool((hold[:, :16] == 9).all()) and bool((hold[:, 208:] == 9).all())
    gg = gate.float().unflatten(-1, (3, 80))[..., :64].flatten(1)
    _check_attention(c, wide[:, 16:], hold[:, 16:208], lens, [0, 1, 2], 3, gate=gg)


# ------------------------------------------------------------------------------------ pages

def _same(c, o):
    assert c.lens.tolist() == o.lens
    assert c.refs.tolist() == o.refs
    assert c.table.tolist() == o.table


@pytest.mark.parametrize("seed", range(4))
def test_page_bookkeeping_follows_the_oracle(seed):
    """Random runs of extend, fork, free and compact, refused calls among them; the tokens of
    every row stay what they were."""
    from b200fp8 import device_status
    import random
    rng = random.Random(seed)
    page = rng.choice([16, 32, 64])
    rows, cols, pages = 12, 6, 30
    c = _cache(layers=2, pages=pages, page_size=page, kv_heads=1, head_dim=64, max_seqs=rows,
               max_pages=cols)
    c.storage.copy_(torch.randint(0, 256, c.storage.shape, generator=gen(seed)).to(torch.uint8))
    o = serving.Pages(pages, rows, cols, page)
    store = c.storage.cpu().clone()
    device_status(reset=True)
    for step in range(40):
        what = rng.choice(["extend", "extend", "fork", "free", "compact"])
        bad = False
        if what == "extend":
            n = rng.randint(1, 4)
            who = [rng.randrange(rows) for _ in range(n)] if rng.random() < .2 else rng.sample(range(rows), n)
            counts = [rng.randint(0, 3 * page) for _ in who]
            bad = not o.extend(who, counts)
            c.extend(_ints(counts), rows=_ints(who))
        elif what == "fork":
            full = [r for r in range(rows) if o.lens[r]] or [0]
            empty = [r for r in range(rows) if not o.lens[r]]
            n = min(len(empty), rng.randint(1, 3))
            if not n:
                continue
            src = [rng.choice(full) for _ in range(n)]
            dst = rng.sample(empty, n)
            if rng.random() < .15:
                dst[0] = rng.randrange(-1, rows + 1)
            bad = not o.fork(src, dst)
            c.fork(_ints(src), _ints(dst))
        elif what == "free":
            who = rng.sample(range(rows), rng.randint(1, 3))
            o.free(who)
            c.free(_ints(who + who[:1]))
        else:
            o.compact()
            c.compact()
        for a, b in o.copies:
            store[:, b] = store[:, a]
        o.copies.clear()
        torch.cuda.synchronize()
        assert (device_status(reset=True) != 0) == bad, (what, step)
        _same(c, o)
        assert torch.equal(c.storage.cpu(), store)
    assert c.free_pages() == sum(r == 0 for r in o.refs)


def test_large_pool_and_many_rows():
    """More pages than one round of the scan covers, 1024 rows in one call."""
    rows, page = 1024, 16
    c = _cache(layers=1, pages=40000, page_size=page, kv_heads=1, head_dim=64, max_seqs=rows,
               max_pages=40)
    o = serving.Pages(40000, rows, 40, page)
    counts = [(i * 37) % 500 for i in range(rows)]
    o.extend(list(range(rows)), counts)
    c.extend(_ints(counts))
    who = list(range(0, rows, 3))
    o.free(who)
    c.free(_ints(who))
    o.compact()
    c.compact()
    again = [500] * len(who)
    o.extend(who, again)
    c.extend(_ints(again), rows=_ints(who))
    torch.cuda.synchronize()
    _same(c, o)
    c.free()
    assert c.free_pages() == 40000 and int(c.lens.sum()) == 0


def test_too_few_pages_change_nothing():
    from b200fp8 import device_status
    c = _cache(layers=1, pages=5, page_size=16, kv_heads=1, head_dim=64, max_seqs=3, max_pages=9)
    device_status(reset=True)
    c.extend(_ints([40, 17, 0]))
    state = [t.clone() for t in (c.table, c.lens, c.refs)]
    c.extend(_ints([0, 0, 1]))
    assert device_status(reset=True) == 6
    c.fork(_ints([0]), _ints([2]))
    assert device_status(reset=True) == 6
    assert all(torch.equal(a, b) for a, b in zip(state, (c.table, c.lens, c.refs)))


def test_copy_pages():
    c = _cache(layers=3, pages=700, page_size=16, kv_heads=2, head_dim=64, max_seqs=1, max_pages=1)
    c.storage.copy_(torch.randint(0, 256, c.storage.shape, generator=gen(1)).to(torch.uint8))
    want = c.storage.clone()
    src, dst = list(range(0, 600, 2)), list(range(1, 601, 2))
    want[:, dst] = want[:, src]
    c.copy_pages(src, dst)
    torch.cuda.synchronize()
    assert torch.equal(c.storage, want)
    from b200fp8 import B2FError
    for bad in (([1, 2], [3, 3]), ([1, 2], [2, 5]), ([1], [700]), ([-1], [0])):
        with pytest.raises(B2FError):
            c.copy_pages(*bad)


def test_a_served_sequence():
    """The operators as they are used: a prompt, forked samples that grow apart, a freed one,
    packing, and steps of a captured graph; every step's context against the oracle."""
    from b200fp8 import device_status, ops, rotary
    g = gen(100)
    kv, heads, d, page = 2, 8, 128, 16
    c = _cache(layers=1, pages=64, page_size=page, kv_heads=kv, head_dim=d, max_seqs=6,
               max_pages=12, k_scale=1 / 8, v_scale=1 / 8)
    plan = rotary.RotaryPlan(d, theta=1e6, device="cuda")
    device_status(reset=True)
    lens = [0] * 6

    def step(rows, news):
        starts = [0]
        for n in news:
            starts.append(starts[-1] + n)
        for r, n in zip(rows, news):
            lens[r] += n
        pos = torch.tensor([lens[r] - n + i for r, n in zip(rows, news) for i in range(n)],
                           dtype=torch.int32)
        q, k, v = (randn((starts[-1], h * d), g).to(BF16).cuda() for h in (heads, kv, kv))
        c.extend(_ints(news), rows=_ints(rows))
        q, k = ops.rotary(q, k, pos.cuda(), plan, heads=heads, kv_heads=kv)
        c.write(k, v, rows=_ints(rows), starts=_ints(starts))
        out, lse = c.attention(q, heads=heads, rows=_ints(rows), starts=_ints(starts),
                               return_lse=True)
        torch.cuda.synchronize()
        _check_attention(c, q.cpu(), out, lens, starts, heads, lse=lse, rows=rows)

    step([0, 3], [37, 20])
    c.fork(_ints([0, 0, 3]), _ints([1, 2, 5]))
    for r, s in ((1, 0), (2, 0), (5, 3)):
        lens[r] = lens[s]
    step([0, 1, 2, 3, 5], [1] * 5)
    step([5, 2, 0], [2, 1, 17])
    c.free(_ints([0]))
    lens[0] = 0
    c.compact()
    step([1, 2, 3, 5], [1] * 4)
    assert int((c.refs > 0).nonzero().max()) < 64 - c.free_pages() + 4
    assert device_status() == 0


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("heads,kv,page", [(4, 1, 16), (8, 2, 64), (14, 2, 32)])
def test_chunks_of_prompts(d, heads, kv, page):
    """Chunks with enough rows for the tensor-core tiles: rows that end inside a tile, in one or
    both tiles, sequences cut among CTAs, prefixes of all lengths, an empty sequence, a chunk that
    is the whole sequence, every page size."""
    g = gen(d + heads)
    lens = [700, 130, 61, 0, 257, 1000, 128]
    news = [90, 130, 61, 0, 33, 150, 1]
    c, _, _, _ = _filled(lens, None, kv=kv, d=d, page=page, g=g, garbage=True)
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    q = randn((starts[-1], heads * d), g).to(BF16)
    out, lse = c.attention(q.cuda(), heads=heads, starts=_ints(starts), return_lse=True)
    again, _ = c.attention(q.cuda(), heads=heads, starts=_ints(starts), return_lse=True)
    torch.cuda.synchronize()
    assert torch.equal(out, again)
    _check_attention(c, q, out, lens, starts, heads, lse=lse)


@pytest.mark.parametrize("scale", [0.3, 1.0, 2.0 ** -64, 2.0 ** 64, 0.9999999, 1.0000001])
def test_codes_are_those_of_the_f32_quotient(scale):
    """Values within a few units of the last place of every border between two codes, and on it, for
    groups of all scales (subnormal and saturated ones among them), zeros of both signs, values so
    small that their quotients underflow.  The rule is the f32 quotient's, in numpy's division."""
    import numpy as np
    rng = np.random.default_rng(7)
    n, d, f = 512, 128, np.float32
    scale = float(f(scale))
    s8 = torch.arange(1, 0x7f, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    want_s = s8[rng.integers(0, len(s8), (n, d // 16, 1))].astype(f)
    s = (want_s * f(scale)).astype(f)
    border = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], f)[rng.integers(0, 7, (n, d // 16, 16))]
    x = (border * s).astype(f)
    x = (x.view(np.int32) + rng.integers(-3, 4, x.shape, dtype=np.int32)).view(f)
    tiny = rng.random(x.shape) < 0.1
    x = np.where(tiny, rng.choice(np.array([0.0, 1e-45, 1e-30, 1e-38], f), x.shape), x).astype(f)
    x[..., 0:1] = 6 * want_s * f(scale)  # fixes the scale of the group
    x[: n // 8, :, 1:2] = 1e4 * want_s[: n // 8] * f(scale)  # another one, saturated for many
    x = (x * np.where(rng.random(x.shape) < 0.5, f(-1), f(1))).astype(f)
    top = np.abs(x).max(-1, keepdims=True)
    got_s8 = torch.from_numpy((top / f(f(6) * f(scale))).astype(f)).clamp(max=448).to(torch.float8_e4m3fn)
    div = (got_s8.float().numpy() * f(scale)).astype(f)
    with np.errstate(divide="ignore", invalid="ignore", under="ignore"):
        q = np.where(div > 0, (x / div).astype(f), f(0))
    steps = (np.abs(q)[..., None] > np.array([0.25, 1.25, 2.5, 5.0], f)).sum(-1) + \
        (np.abs(q)[..., None] >= np.array([0.75, 1.75, 3.5], f)).sum(-1)
    codes = steps + 8 * np.signbit(q)
    c = _cache(layers=1, pages=n // 16, page_size=16, kv_heads=1, head_dim=d, max_seqs=1,
               max_pages=n // 16, k_scale=scale, v_scale=scale)
    c.extend(_ints([n]))
    flat = torch.from_numpy(x).flatten(1).cuda()
    c.write(flat, flat)
    torch.cuda.synchronize()
    pages = c.table[0].long().cpu()
    block = c.storage[0].cpu()[pages, 0]
    for at in (0, 16 * d * 9 // 16):
        packed = block[:, at:at + 16 * d // 2].reshape(n, d // 2)
        got = torch.stack([packed & 15, packed >> 4], -1).flatten(1).numpy()
        scales = block[:, at + 16 * d // 2:at + 16 * d * 9 // 16].reshape(n, d // 16)
        assert torch.equal(scales, got_s8.view(torch.uint8)[..., 0])
        assert (got == codes.reshape(n, d)).all()


@pytest.mark.parametrize("q_dtype,out_dtype", [(F16, BF16), (E4M3, E4M3)])
@pytest.mark.parametrize("causal", [True, False])
def test_chunks_with_gate_types_and_uniform_lengths(q_dtype, out_dtype, causal):
    g = gen(5 + causal)
    lens, n, heads, d = [300, 50, 40], 48, 8, 128
    c, _, _, _ = _filled(lens, None, kv=2, d=d, page=16, g=g, garbage=True)
    qs = 1 / 64 if q_dtype == E4M3 else 1.0
    q = (randn((3 * n, heads * d), g) / qs).clamp(-440, 440).to(q_dtype)
    gate = (randn((3 * n, heads * d), g) * 64).clamp(-440, 440).to(E4M3)
    outs = 1 / 256 if out_dtype == E4M3 else 1.0
    out, lse = c.attention(q.cuda(), heads=heads, causal=causal, q_scale=qs, gate=gate.cuda(),
                           gate_scale=1 / 64, out_dtype=out_dtype, ctx_scale=outs, return_lse=True)
    torch.cuda.synchronize()
    _check_attention(c, q, out, lens, [0, n, 2 * n, 3 * n], heads, causal=causal, q_scale=qs,
                     gate=gate.float() / 64, out_scale=outs, lse=lse)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("which", ["k", "v"])
def test_nan_in_a_chunk_reaches_only_those_who_see_it(d, which):
    g = gen(d + 1)
    lens = [200, 200]
    c, k, v, starts = _filled(lens, None, kv=1, d=d, page=16, g=g)
    k, v = k.clone(), v.clone()
    (k if which == "k" else v)[150, 3] = float("nan")
    c.write(k.cuda(), v.cuda(), starts=_ints(starts))
    q = randn((200, 2 * d), g).to(BF16)
    out = c.attention(q.cuda(), heads=2, starts=_ints([0, 100, 200]))
    torch.cuda.synchronize()
    clean = torch.isfinite(out).all(1).cpu().tolist()
    assert clean == [True] * 50 + [False] * 50 + [True] * 100
    assert bool(torch.isnan(out[50:100, :16]).all())
    for b, lo, hi, seen in ((0, 0, 50, 150), (1, 100, 200, 200)):
        kk, vv = _oracle_kv(c, b, 200)
        want, _, mass, size = serving.attention(q[lo:hi].double().unflatten(-1, (2, d)),
                                                kk[:seen], vv[:seen])
        got = out[lo:hi].cpu().double().unflatten(-1, (2, d))
        bound = mass * (2.0 ** -11 + 2.0 ** -16 + size * 2.0 ** -20) + want.abs() * 2.0 ** -8
        assert bool(((got - want).abs() <= bound).all())


def test_bad_pages_in_a_chunk_are_left_out():
    from b200fp8 import device_status
    g = gen(22)
    c, _, _, _ = _filled([300], None, kv=1, d=128, page=16, g=g)
    good = c.table.clone()
    device_status(reset=True)
    c.table[0, 3], c.table[0, 9] = c.pages, -1
    q = randn((100, 128), g).to(BF16)
    out = c.attention(q.cuda(), heads=1)
    torch.cuda.synchronize()
    assert device_status(reset=True) == 5
    k, v = serving.cached(c.storage[0].cpu(), good[0].cpu(), 300, 16, 128, 0.25, 0.25)
    hidden = [i for i in range(300) if i // 16 in (3, 9)]
    for i in (0, 57, 99):
        keep = [j for j in range(201 + i) if j not in hidden]
        want, _, mass, size = serving.attention(q[i:i + 1].double().unflatten(-1, (1, 128)),
                                                k[keep], v[keep])
        err = (out[i].cpu().double() - want.flatten()).abs()
        bound = mass.flatten() * (2.0 ** -11 + 2.0 ** -16 + size * 2.0 ** -20) + want.flatten().abs() * 2.0 ** -8
        assert bool((err <= bound).all())


def test_late_large_scores_in_a_chunk_move_the_maximum():
    g = gen(3)
    n, d = 500, 128
    c = _cache(layers=1, pages=40, page_size=16, kv_heads=1, head_dim=d, max_seqs=1, max_pages=40,
               k_scale=1 / 16)
    c.extend(_ints([n]))
    k = randn((n, d), g) * 0.05 + torch.linspace(-4, 4, n)[:, None]
    c.write(k.to(BF16).cuda(), randn((n, d), g).to(BF16).cuda())
    q = torch.cat([torch.full((64, d), 0.5), torch.full((64, d), -0.5)]).to(BF16)
    out, lse = c.attention(q.cuda(), heads=1, sm_scale=1.0, return_lse=True)
    torch.cuda.synchronize()
    _check_attention(c, q, out, [n], [0, 128], 1, sm_scale=1.0, lse=lse)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 100])
def test_bad_pages_of_all_kinds_in_a_long_sequence(d, n):
    """Pages that are not there, of every number that says so, in one in four of the steps: their keys
    are left out by every row, those of the steps next to them are not."""
    from b200fp8 import device_status
    g = gen(d + n)
    length = 2500
    c, _, _, _ = _filled([length], None, kv=1, d=d, page=16, g=g)
    good = c.table.clone()
    device_status(reset=True)
    hidden = set()
    for i, bad in zip(range(3, length // 16, 32), (c.pages, -1, -2 ** 31, 2 ** 31 - 1, -7)):
        c.table[0, i] = bad
        hidden.update(range(16 * i, 16 * i + 16))
    q = randn((n, 2 * d), g).to(BF16)
    out = c.attention(q.cuda(), heads=2)
    torch.cuda.synchronize()
    assert device_status(reset=True) == 5
    k, v = serving.cached(c.storage[0].cpu(), good[0].cpu(), length, 16, d, 0.25, 0.25)
    for i in {0, n // 2, n - 1}:
        keep = [j for j in range(length - n + 1 + i) if j not in hidden]
        want, _, mass, size = serving.attention(q[i:i + 1].double().unflatten(-1, (2, d)),
                                                k[keep], v[keep])
        err = (out[i].cpu().double() - want.flatten()).abs()
        bound = (mass * (2.0 ** -11 + 2.0 ** -16 + size * 2.0 ** -20) + want.abs() * 2.0 ** -8).flatten()
        assert bool((err <= bound).all())


@pytest.mark.parametrize("n", [3, 100])
def test_queries_and_scales_too_small_for_a_product(n):
    """Queries and a key scale whose product underflows: all scores are 0, and rows average the
    values that they see, no others."""
    g = gen(n)
    d, length = 128, 170
    c = _cache(layers=1, pages=16, page_size=16, kv_heads=1, head_dim=d, max_seqs=1, max_pages=16,
               k_scale=2.0 ** -64, v_scale=0.25)
    c.extend(_ints([length]))
    k = (randn((length, d), g) * 2.0 ** -64).to(BF16)
    c.write(k.cuda(), randn((length, d), g).to(BF16).cuda())
    q = (randn((n, 2 * d), g) * 2.0 ** -124).to(BF16)
    out, lse = c.attention(q.cuda(), heads=2, return_lse=True)
    torch.cuda.synchronize()
    _, v = serving.cached(c.storage[0].cpu(), c.table[0].cpu(), length, 16, d, 2.0 ** -64, 0.25)
    v = v.reshape(length, d)
    for i in range(n):
        seen = v[:length - n + 1 + i]
        # P is one value for all keys, exact in f16: the roundings are those of the sums and of the output
        bound = seen.abs().mean(0) * 2.0 ** -15 + seen.mean(0).abs() * 2.0 ** -8
        for h in range(2):
            err = (out[i, h * d:(h + 1) * d].cpu().double() - seen.mean(0)).abs()
            assert bool((err <= bound).all())
        want = torch.log(torch.tensor(float(len(seen)), dtype=torch.float64))
        assert bool(((lse[i].cpu().double() - want).abs() < 2.0 ** -18).all())


@pytest.mark.parametrize("d", [64, 128, 256])
def test_pages_layers_and_lists_with_strides_of_their_own(d):
    """Pages 2 GB apart (byte offsets that pass 32 bits), layers between them, a table inside a wider
    one, length and count lists inside longer ones; every call on it, both forms of the attention."""
    from b200fp8 import device_status
    from b200fp8.kvcache import Fp4Cache
    g = gen(d)
    kv, page, heads = 2, 16, 8
    block = page * d * 9 // 8
    far, mid = 2 ** 31 + 4096, 2 ** 20
    base = torch.empty(5 * far, dtype=torch.uint8, device="cuda")
    storage = base.as_strided((2, 5, kv, block), (mid, far, block, 1))
    storage.fill_(0xff)
    table = torch.full((4, 9), 77, dtype=torch.int32, device="cuda")
    lens = torch.full((6,), 99, dtype=torch.int32, device="cuda")
    refs = torch.full((8,), 55, dtype=torch.int32, device="cuda")
    table[1:4, 2:5], lens[2:5], refs[1:6] = -1, 0, 0
    device_status(reset=True)
    c = Fp4Cache.from_buffers(storage, table[1:4, 2:5], lens[2:5], refs[1:6], page_size=page,
                              head_dim=d, k_scale=0.25, v_scale=0.25)
    c.extend(_ints([10, 40]))          # page 0; pages 1, 2, 3
    k, v = (randn((50, kv * d), g).to(BF16) for _ in range(2))
    for layer in range(2):
        c.write(k.cuda(), v.cuda(), starts=_ints([0, 10, 50]), layer=layer)
    c.free(_ints([0]))                 # page 0
    c.fork(_ints([1]), _ints([2]))     # its last page into page 0
    q = randn((40, heads * d), g).to(BF16)
    for row in (1, 2):
        for n in (1, 40):
            out, lse = c.attention(q[:n].cuda(), heads=heads, rows=_ints([row]), layer=1,
                                   return_lse=True)
            torch.cuda.synchronize()
            _check_attention(c, q[:n], out, [0, 40, 40], [0, n], heads, layer=1, lse=lse, rows=[row])
    c.free(_ints([1]))                 # page 3; its other pages are row 2's too
    assert c.table[2].tolist() == [1, 2, 0] and refs[1:6].tolist() == [1, 1, 1, 0, 0]
    kept = [t.clone() for t in c.read(40, rows=_ints([2]), layer=1)]
    c.extend(_ints([16]), rows=_ints([0]))   # page 3
    c.free(_ints([2]))
    c.compact()                        # page 3 to page 0
    assert c.table[0, 0].item() == 0 and refs[1:6].tolist() == [1, 0, 0, 0, 0]
    c.copy_pages([0], [4])
    torch.cuda.synchronize()
    assert torch.equal(storage[:, 0], storage[:, 4])
    rk, rv = serving.cached(storage[1].cpu(), torch.tensor([1, 2]), 32, page, d, 0.25, 0.25)
    assert torch.equal(kept[0][:32].cpu().double(), rk.flatten(1).to(BF16).double())
    assert torch.equal(kept[1][:32].cpu().double(), rv.flatten(1).to(BF16).double())
    assert device_status(reset=True) == 0
    assert (table[0] == 77).all() and (table[:, :2] == 77).all() and (table[:, 5:] == 77).all()
    assert lens[:2].tolist() == [99, 99] and lens[5].item() == 99
    assert refs[0].item() == 55 and refs[6:].tolist() == [55, 55]


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("blank,long", [(53, 1), (160, 30)])
def test_rows_that_see_nothing_beside_sequences_that_are_cut(d, blank, long):
    """Sequences with many new tokens and no cached ones in front of long ones, which are cut among
    the CTAs that fill the first ones' rows with zeros: every row is written, the same every time,
    in both forms of the attention."""
    g = gen(d + blank)
    heads, page = 4, 16
    lens = [0] * 8 + [1900, 700, 2301] * 4
    news = [blank] * 8 + [long] * 12
    c, _, _, _ = _filled(lens, None, kv=1, d=d, page=page, g=g)
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    q = randn((starts[-1], heads * d), g).to(BF16)
    first = None
    for _ in range(8):
        out = torch.full((starts[-1], heads * d), float("nan"), dtype=BF16, device="cuda")
        lse = torch.full((starts[-1], heads), float("nan"), device="cuda")
        c.attention(q.cuda(), heads=heads, starts=_ints(starts), out=out, lse=lse)
        torch.cuda.synchronize()
        if first is None:
            first = out, lse
        assert torch.equal(out, first[0]) and torch.equal(lse, first[1])
    assert bool((out[:8 * blank] == 0).all()) and bool((lse[:8 * blank] == -float("inf")).all())
    _check_attention(c, q, out, lens, starts, heads, lse=lse)


def _cut_wrongly(seqs, which):
    """starts that leave the batch at one end, the tokens of the batch, and those of the sequence
    that is cut wrongly; the others have two tokens each."""
    tokens = 2 * seqs + 3
    starts = [2 * i for i in range(seqs + 1)]
    if which == "end":
        starts[-1] = tokens + 10
        return starts, tokens, range(2 * seqs - 2, tokens)
    starts[0] = -4
    return starts, tokens, range(0, 2)


@pytest.mark.parametrize("seqs", [1, 2, 31, 32, 33])
@pytest.mark.parametrize("which", ["start", "end"])
def test_sequences_cut_outside_of_the_batch_are_not_written(seqs, which):
    """However many sequences a call has, one whose tokens are not all in the batch is left out of
    it and recorded; the others are written and read."""
    from b200fp8 import device_status
    from b200fp8.kvcache import Fp4Cache
    g = gen(seqs)
    c, _, _, _ = _filled([40] * seqs, None, kv=1, d=64, page=16, g=g)
    starts, tokens, bad = _cut_wrongly(seqs, which)
    k, v = randn((tokens, 64), g).to(BF16), randn((tokens, 64), g).to(BF16)
    ref = Fp4Cache.from_buffers(c.storage.clone(), c.table, c.lens, c.refs, page_size=16,
                                head_dim=64, k_scale=0.25, v_scale=0.25)
    good = [b for b in range(seqs) if starts[b] >= 0 and starts[b + 1] <= tokens]
    if good:
        ref.write(k[2 * good[0]:2 * good[-1] + 2].cuda(), v[2 * good[0]:2 * good[-1] + 2].cuda(),
                  rows=_ints(good))
    assert device_status(reset=True) == 0
    c.write(k.cuda(), v.cuda(), starts=_ints(starts))
    assert device_status(reset=True) == 5
    assert torch.equal(c.storage, ref.storage)
    rk, rv = (torch.full((tokens, 64), 7.0, dtype=BF16, device="cuda") for _ in range(2))
    c.read(tokens, starts=_ints(starts), k=rk, v=rv)
    assert device_status(reset=True) == 5
    for x, r in ((k, rk), (v, rv)):
        r = r.cpu()
        for t in range(tokens):
            if t in bad:
                assert bool((r[t] == 0).all())
            elif t >= 2 * seqs:
                assert bool((r[t] == 7).all())
            else:
                assert torch.equal(r[t].double(), serving.pack(x[t], 0.25)[2])


@pytest.mark.parametrize("seqs", [2, 33])
@pytest.mark.parametrize("which", ["start", "end"])
def test_sequences_cut_outside_of_the_batch_are_not_attended(seqs, which):
    from b200fp8 import device_status
    g = gen(seqs + 1)
    lens = [40] * seqs
    c, _, _, _ = _filled(lens, None, kv=1, d=64, page=16, g=g)
    starts, tokens, bad = _cut_wrongly(seqs, which)
    q = randn((tokens, 128), g).to(BF16)
    out = torch.full((tokens, 128), 5.0, dtype=BF16, device="cuda")
    assert device_status(reset=True) == 0
    c.attention(q.cuda(), heads=2, starts=_ints(starts), out=out)
    assert device_status(reset=True) == 5
    for t in [*bad, *range(2 * seqs, tokens)]:
        assert bool((out[t] == 5).all())
    good = [b for b in range(seqs) if starts[b] >= 0 and starts[b + 1] <= tokens]
    _check_attention(c, q, out, lens, [2 * b for b in good] + [2 * good[-1] + 2], 2, rows=good)


@pytest.mark.parametrize("seqs", [31, 32, 33, 64, 1025])
@pytest.mark.parametrize("each", [None, 1])
def test_writing_and_reading_many_sequences(seqs, each):
    """Packed tokens find their sequences, empty ones among them, however many there are."""
    from b200fp8 import device_status
    g = gen(seqs)
    lens = [(i * 7) % 5 if each is None else each for i in range(seqs)]
    device_status(reset=True)
    c, k, v, starts = _filled(lens, None, kv=2, d=64, page=16, g=g)
    rk, rv = c.read(starts[-1], starts=_ints(starts))
    for x, r in ((k, rk), (v, rv)):
        want = serving.pack(x.unflatten(-1, (2, 64)), 0.25)[2].flatten(1)
        assert torch.equal(r.cpu().double(), want)
    if each is not None:  # without starts, and a table row at a time from the other end
        back = list(range(seqs - 1, -1, -1))
        c.write(v.cuda(), k.cuda(), rows=_ints(back))
        bk, bv = c.read(seqs)
        assert torch.equal(bk.flip(0), rv) and torch.equal(bv.flip(0), rk)
    assert device_status() == 0


@pytest.mark.parametrize("d,seqs,new,starts", [
    (64, 170, 1, False), (64, 170, 1, True), (128, 600, 1, False), (128, 600, 1, True),
    (256, 600, 1, True), (64, 600, 14, True), (128, 170, 26, True), (256, 390, 13, False)])
@pytest.mark.parametrize("empty", [False, True])
def test_attention_of_many_sequences(d, seqs, new, starts, empty):
    """More sequences than a CTA has threads, single tokens and chunks of 100 rows and more, with
    and without sequences that hold nothing (more of them than there are CTAs, with `empty`)."""
    g = gen(d + seqs + new)
    heads, page = 8, 16
    lens = [0 if (i % 8 != 5 if empty else i % 9 == 4) else 1 + (i * 29) % 70 for i in range(seqs)]
    lens[seqs // 2] = 900
    c, _, _, _ = _filled(lens, None, kv=1, d=d, page=page, g=g, garbage=True)
    news = [new] * seqs
    if starts and new > 1:
        news = [0 if i % 11 == 3 else new for i in range(seqs)]
    at = [0]
    for n in news:
        at.append(at[-1] + n)
    q = randn((at[-1], heads * d), g).to(BF16)
    out = torch.full((at[-1], heads * d), float("nan"), dtype=BF16, device="cuda")
    lse = torch.full((at[-1], heads), float("nan"), device="cuda")
    c.attention(q.cuda(), heads=heads, starts=_ints(at) if starts else None, out=out, lse=lse)
    _check_attention(c, q, out, lens, at, heads, lse=lse)


@pytest.mark.parametrize("d,seqs,kv,group,new", [
    (64, 170, 1, 4, 1), (64, 1500, 1, 2, 1), (128, 600, 2, 4, 1), (128, 200, 1, 16, 5),
    (256, 600, 1, 2, 1), (256, 170, 1, 8, 3), (64, 3, 2, 8, 11)])
def test_many_sequences_in_a_short_table(d, seqs, kv, group, new):
    """Tables so short that items are not cut: more items than CTAs, several row tiles a sequence,
    sequences without keys, fewer keys than new tokens."""
    g = gen(d + seqs)
    most = 112 if d == 256 else 240
    lens = [0 if i % 6 == 5 else 1 + (i * 53) % most for i in range(seqs)]
    c, _, _, _ = _filled(lens, None, kv=kv, d=d, page=16, g=g, garbage=True)
    heads = kv * group
    for starts in (None, [i * new for i in range(seqs + 1)]):
        q = randn((seqs * new, heads * d), g).to(BF16)
        out = torch.full((seqs * new, heads * d), float("nan"), dtype=BF16, device="cuda")
        lse = torch.full((seqs * new, heads), float("nan"), device="cuda")
        c.attention(q.cuda(), heads=heads, starts=None if starts is None else _ints(starts), out=out,
                    lse=lse)
        _check_attention(c, q, out, lens, [i * new for i in range(seqs + 1)], heads, lse=lse)


def test_first_calls_inside_a_capture():
    """A graph may be captured before any call has run eagerly: the same as the eager calls."""
    import subprocess
    import sys
    code = """
import sys, torch
sys.path[:0] = [%r, %r]
from b200fp8 import device_status, kvcache, ops, rotary
ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
torch.manual_seed(3)
make = lambda: kvcache.Fp4Cache(layers=1, pages=400, page_size=16, kv_heads=1, head_dim=64,
                                max_seqs=4, max_pages=90, k_scale=0.25, v_scale=0.25)
plan = rotary.RotaryPlan(64, device="cuda")
counts, src, dst, back = ints([1100, 700, 0, 0]), ints([0]), ints([2]), ints([1])
k, v, q = (torch.randn(1800, h * 64, device="cuda").bfloat16() for h in (1, 1, 4))
starts, pos = ints([0, 1100, 1800]), torch.arange(1800, device="cuda", dtype=torch.int32)

def calls(c):
    c.extend(counts)
    qr, kr = ops.rotary(q, k, pos, plan, heads=4, kv_heads=1)
    c.write(kr, v, rows=ints_01, starts=starts)
    c.fork(src, dst)
    c.free(back)
    c.compact()
    one = c.attention(qr[:1], heads=4, rows=dst)
    many = c.attention(qr[:300], heads=4, rows=src)
    return (one, many, *c.read(1100, rows=dst))

ints_01 = ints([0, 1])
a, b = make(), make()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = calls(a)
graph.replay()
want = calls(b)
torch.cuda.synchronize()
assert all(torch.equal(x, y) for x, y in zip(got, want))
assert torch.equal(a.table, b.table) and torch.equal(a.refs, b.refs) and torch.equal(a.lens, b.lens)
assert device_status() == 0 and a.lens.tolist() == [1100, 0, 1100, 0]
print("same")
"""
    import pathlib
    root = pathlib.Path(__file__).resolve().parents[1]
    run = subprocess.run([sys.executable, "-c", code % (str(root / "airi-summer-kernel-evo_b200"),
                                                        str(root))],
                         capture_output=True, text=True, timeout=300)
    assert run.stdout.strip() == "same", run.stderr[-2000:]
