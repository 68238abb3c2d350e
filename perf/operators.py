"""The serving-cache operators of this repository, as they are timed and compared.

Four operators carry a decoder block from prompts to single tokens:

  rotary     rotary positions of q and k at explicit positions (half or interleaved pairs, part
             of the head, stretched frequencies for long contexts), with the head norm in front
  write      keys and values quantised to 4 bits into the pages of a cache, and read back
  attention  attention of new tokens over that cache
  pages      forking, freeing and compacting the sequences of the cache

``own`` false: elementary torch operations in 32 bits.  ``own`` true: this repository's kernels.

A cache page holds, for each kv head, [K codes | K scales | V codes | V scales]: codes are e2m1
(two to a byte, the even element in the low nibble), and every 16 consecutive elements of a head
share one e4m3 scale; value = code * scale * k_scale (v_scale).
"""
import math
import os
import random
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_DEV = "cuda"
_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32,
       "e4m3": torch.float8_e4m3fn}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4, "e4m3": 1}


def _package():
    path = os.path.join(_ROOT, "airi-summer-kernel-evo_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from b200fp8 import kvcache, ops, rotary
    return ops, rotary, kvcache


# ------------------------------------------------------------------------------------ cases

def listed():
    return [
        # one decoding step of 8 sequences far into their contexts: the gated block's q and k
        # (e4m3 from its projection) normalised and rotated; latency is what counts
        dict(name="rotary_step", op="rotary", tokens=8, heads=32, kv_heads=8, head_dim=128,
             rotary_dim=128, layout="half", theta=1e6, scaling="none", far=200000,
             src="e4m3", dst="bf16", norm=True),
        # a prompt of odd length through a head that is rotated in part (64 of 256)
        dict(name="rotary_prompt_partial", op="rotary", tokens=4099, heads=16, kv_heads=4,
             head_dim=256, rotary_dim=64, layout="half", theta=1e7, scaling="none", far=4099,
             src="bf16", dst="bf16", norm=False),
        # interleaved pairs with stretched frequencies, a batch of prompts in f32
        dict(name="rotary_prompt_stretched", op="rotary", tokens=8192, heads=32, kv_heads=8,
             head_dim=128, rotary_dim=128, layout="interleaved", theta=1e6, scaling="yarn",
             far=131072, src="f32", dst="f32", norm=False),
        # one token of each of 24 sequences into the cache
        dict(name="write_step", op="write", seqs=24, length=2047, new=1, kv_heads=8, head_dim=128,
             page=16, src="bf16", mix=1),
        # four prompts, 2048 tokens the longest, into the cache
        dict(name="write_prompt", op="write", seqs=4, length=2048, new=2048, kv_heads=8,
             head_dim=128, page=64, src="bf16", mix=2),
        # one user, a short context: the smallest call of a serving loop
        dict(name="attend_short", op="attention", seqs=1, length=197, new=1, heads=32, kv_heads=8,
             head_dim=128, page=16, src="bf16", dst="bf16", mix=3, gate=False, lse=False),
        # a batch of 64 conversations of all lengths
        dict(name="attend_batch", op="attention", seqs=64, length=8191, new=1, heads=32,
             kv_heads=8, head_dim=128, page=16, src="bf16", dst="bf16", mix=4, gate=False,
             lse=False),
        # two very long contexts: the work of a sequence has to be split
        dict(name="attend_long", op="attention", seqs=2, length=131072, new=1, heads=32,
             kv_heads=8, head_dim=128, page=64, src="bf16", dst="f16", mix=0, gate=False,
             lse=True),
        # the gated block with head_dim 256: e4m3 queries and gate, e4m3 context
        dict(name="attend_gated_256", op="attention", seqs=16, length=4000, new=1, heads=16,
             kv_heads=4, head_dim=256, page=32, src="e4m3", dst="e4m3", mix=5, gate=True,
             lse=False),
        # chunks of prompts of different lengths behind cached prefixes
        dict(name="attend_chunk", op="attention", seqs=3, length=8192, new=512, heads=32,
             kv_heads=8, head_dim=128, page=64, src="bf16", dst="bf16", mix=6, gate=False,
             lse=False),
        # eight samples of each of 8 prompts, replaced every step of a search
        dict(name="fork_samples", op="fork", layers=4, pages=4096, seqs=8, copies=8, length=1500,
             kv_heads=8, head_dim=128, page=16, mix=7),
        # a pool with a third of its pages in use, packed to its front
        dict(name="compact_pool", op="compact", layers=4, pages=6000, seqs=40, copies=0,
             length=1600, kv_heads=8, head_dim=128, page=16, mix=8),
    ]


_MOST = {"rotary": 8192 * 40 * 128 * 8, "write": 2048 * 4 * 8 * 128 * 2,
         "keys": 2 * 131072 * 8 * 128, "pairs": 512 * 8192 * 32 * 128 * 2}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "write", "attention", "attention", "fork", "compact"])
    kv = rng.choice([1, 2, 4, 8])
    if op == "rotary":
        dim = rng.choice([64, 96, 128, 256])
        rot = rng.choice([dim, dim, dim // 2, dim // 4])
        src = rng.choice(["bf16", "f16", "f32", "e4m3"])
        dst = "bf16" if src == "e4m3" else src
        heads = kv * rng.choice([1, 2, 4, 7])
        per = (heads + kv) * dim * (_SIZE[src] + _SIZE[dst])
        return dict(op="rotary", tokens=_log(rng, 1, min(8192, max(2, _MOST["rotary"] // per))),
                    heads=heads, kv_heads=kv, head_dim=dim, rotary_dim=rot,
                    layout=rng.choice(["half", "interleaved"]), theta=rng.choice([1e4, 1e6, 1e7]),
                    scaling=rng.choice(["none", "linear", "ntk", "yarn"]),
                    far=_log(rng, 100, 1000000), src=src, dst=dst, norm=rng.random() < 0.3)
    dim = rng.choice([64, 128, 128, 256])
    page = rng.choice([16, 32, 64])
    mix = rng.randrange(1 << 20)
    if op == "write":
        seqs = _log(rng, 1, 64)
        most = max(1, _MOST["write"] // (seqs * kv * dim * 2))
        new = 1 if rng.random() < 0.3 else _log(rng, 1, min(2048, most))
        return dict(op="write", seqs=seqs, length=new + _log(rng, 1, 3000), new=new, kv_heads=kv,
                    head_dim=dim, page=page, src=rng.choice(["bf16", "f16", "f32"]), mix=mix)
    if op == "attention":
        group = rng.choice([1, 2, 4, 5, 8, 16])
        seqs = _log(rng, 1, 64)
        new = rng.choice([1, 1, 1, 2, 3, 4, _log(rng, 5, 300)])
        most = min(131072, _MOST["keys"] // (seqs * kv * dim),
                   _MOST["pairs"] // (seqs * new * kv * group * dim))
        length = _log(rng, 1, max(2, most))
        return dict(op="attention", seqs=seqs, length=length, new=min(new, length),
                    heads=kv * group, kv_heads=kv, head_dim=dim, page=page,
                    src=rng.choice(["bf16", "f16", "e4m3"]), dst=rng.choice(["bf16", "f16"]),
                    mix=mix, gate=rng.random() < 0.3, lse=rng.random() < 0.3)
    seqs = _log(rng, 2, 32)
    copies = rng.choice([1, 2, 4, 8]) if op == "fork" else 0
    length = _log(rng, page, 3000 if page < 64 else 6000)
    need = seqs * (-(-length // page) + copies)
    return dict(op=op, layers=rng.choice([1, 2, 4]), pages=need * rng.choice([2, 3]) + 8,
                seqs=seqs, copies=copies, length=length, kv_heads=kv, head_dim=dim, page=page,
                mix=mix)


def _lengths(case):
    """Cached tokens and new tokens of every sequence, by the case alone: the first sequence is
    the longest; with a mix the others differ, and one of four or more is empty."""
    rng, n, top, new = random.Random(case["mix"]), case["seqs"], case["length"], case.get("new", 0)
    lens = [top] + [top if not case["mix"] else rng.randint(max(1, top // 16), top)
                    for _ in range(n - 1)]
    news = [new] * n
    if new > 1 and case["mix"]:
        news = [new] + [rng.randint(1, new) for _ in range(n - 1)]
    if case["op"] == "attention" and case["mix"] and n >= 4 and new == 1:
        lens[n // 2] = 0
    if case["op"] == "write" and new == top:
        lens = list(news)
    if case["op"] in ("fork", "compact"):
        return lens, news
    return [max(a, b) if a else 0 for a, b in zip(lens, news)], news


def _block_bytes(case):
    return case["page"] * case["head_dim"] * 9 // 8


def work(case):
    op = case["op"]
    if op == "rotary":
        n = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["head_dim"]
        turned = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["rotary_dim"]
        return {"bytes": n * (_SIZE[case["src"]] + _SIZE[case["dst"]]) + 4 * case["tokens"],
                "flops": 3 * turned + (4 * n if case["norm"] else 0)}
    lens, news = _lengths(case)
    if op == "write":
        n = sum(news) * case["kv_heads"] * case["head_dim"] * 2
        # read the 16- or 32-bit values, write the codes; read the codes, write 16-bit values
        return {"bytes": n * (_SIZE[case["src"]] + 9 / 16 + 9 / 16 + 2), "flops": 4 * n}
    if op == "attention":
        d, hq = case["head_dim"], case["heads"]
        tokens = sum(news)
        pairs = sum(sum(max(0, n - k + i + 1) for i in range(k)) for n, k in zip(lens, news))
        io = tokens * hq * (d * (_SIZE[case["src"]] + _SIZE[case["dst"]]
                                 + (1 if case["gate"] else 0)) + (4 if case["lse"] else 0))
        return {"bytes": sum(lens) * case["kv_heads"] * d * 9 / 8 + io, "flops": 4 * pairs * hq * d}
    page = case["layers"] * case["kv_heads"] * _block_bytes(case)
    per = [-(-n // case["page"]) for n in lens]
    if op == "fork":
        part = sum(1 for n in lens if n % case["page"]) * case["copies"]
        return {"bytes": 2 * part * page + 8 * case["copies"] * sum(per) + 8 * case["pages"],
                "flops": 0}
    # the pages of a random pool that lie behind the last one in use after packing
    live = sum(per)
    return {"bytes": 2 * live * (1 - live / case["pages"]) * page + 8 * live + 8 * case["pages"],
            "flops": 0}


# ------------------------------------------------------------------------------------ inputs

_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _pack(x, scale):
    """[..., D] values -> (codes uint8 [..., D/2], scales uint8 [..., D/16]) as the cache holds
    them: the scale is the group's largest magnitude / 6, the code the nearest e2m1 value."""
    g = x.float().unflatten(-1, (-1, 16))
    top = g.abs().amax(-1, keepdim=True)
    six = torch.tensor(6.0, device=x.device) * scale
    s8 = (top / six).clamp(max=448.0).to(torch.float8_e4m3fn)
    s = s8.float() * torch.tensor(scale, device=x.device)
    y = torch.where(s > 0, g / s, torch.zeros_like(g))
    a = y.abs()
    code = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int()
            + (a > 2.5).int() + (a >= 3.5).int() + (a > 5.0).int())
    code = (code + 8 * (torch.signbit(y)).int()).flatten(-2)
    packed = (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8)
    return packed, s8.view(torch.uint8).squeeze(-1)


def _unpack(codes, scales, scale):
    """The values that codes [..., D/2] and scales [..., D/16] stand for, f32 [..., D]."""
    one = torch.tensor(_E2M1 + [-v for v in _E2M1], device=codes.device)
    byte = torch.arange(256, device=codes.device)
    pair = torch.stack([one[byte & 15], one[byte >> 4]], -1)
    v = pair[codes.int()].flatten(-2).unflatten(-1, (-1, 16))
    s = scales.view(torch.float8_e4m3fn).float() * scale
    return (v * s.unsqueeze(-1)).flatten(-2)


def _parts(pages, case):
    """The four parts of page blocks [..., block bytes]: codes and scales of K and of V."""
    p, d = case["page"], case["head_dim"]
    kc, ks, vc, vs = pages.split([p * d // 2, p * d // 16, p * d // 2, p * d // 16], -1)
    return (kc.unflatten(-1, (p, d // 2)), ks.unflatten(-1, (p, d // 16)),
            vc.unflatten(-1, (p, d // 2)), vs.unflatten(-1, (p, d // 16)))


def _normal(shape, g, dtype, spread=1.0):
    return (torch.randn(shape, generator=g, device=_DEV) * spread).to(_DT[dtype])


def _pool(case, g, layers, pages, lens, room):
    """A cache with its pages strewn over the pool: storage, table, lengths, use counts."""
    p, d, h = case["page"], case["head_dim"], case["kv_heads"]
    per = [-(-n // p) for n in room]
    width = max(1, max(per))
    order = torch.randperm(pages, generator=g, device=_DEV).int()
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=_DEV)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    refs = torch.zeros(pages, dtype=torch.int32, device=_DEV)
    refs[order[:at].long()] = 1
    storage = torch.empty((layers, pages, h, _block_bytes(case)), dtype=torch.uint8, device=_DEV)
    for layer in storage:
        # keys and values with the unequal channels that projections have
        gain = torch.exp(0.5 * torch.randn((h, 1, d), generator=g, device=_DEV))
        parts = _parts(layer, case)
        for i in (0, 2):
            for at in range(0, pages, 4096):
                n = min(4096, pages - at)
                x = torch.randn((n, h, p, d), generator=g, device=_DEV) * gain
                codes, scales = _pack(x, 0.25)
                parts[i][at:at + n], parts[i + 1][at:at + n] = codes, scales
    return dict(storage=storage, table=table, refs=refs,
                lens=torch.tensor(lens, dtype=torch.int32, device=_DEV))


def _frequencies(case):
    """Radians per position of every pair (64 bits) and the factor on the rotated part."""
    half = case["rotary_dim"] // 2
    i = torch.arange(half, dtype=torch.float64, device=_DEV)
    theta, stretch = case["theta"], 8.0
    if case["scaling"] == "ntk":
        theta = theta * stretch ** (half / max(half - 1, 1))
    w = theta ** (-i / half)
    if case["scaling"] == "linear":
        return w / stretch, 1.0
    if case["scaling"] != "yarn":
        return w, 1.0
    # pairs that turn often in the trained length keep their frequency, slow ones are stretched
    at = lambda turns: half * math.log(16384 / (turns * 2 * math.pi)) / math.log(theta)  # noqa: E731
    lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), half - 1)
    ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
    return w * (1 - ramp) + w / stretch * ramp, 0.1 * math.log(stretch) + 1.0


def _scaling_argument(case):
    return {"none": None, "linear": {"kind": "linear", "factor": 8.0},
            "ntk": {"kind": "ntk", "factor": 8.0},
            "yarn": {"kind": "yarn", "factor": 8.0, "original_length": 16384}}[case["scaling"]]


def prepare(case, seed):
    g = torch.Generator(device=_DEV).manual_seed(seed)
    op = case["op"]
    if op == "rotary":
        t, d = case["tokens"], case["head_dim"]
        spread = 40.0 if case["src"] == "e4m3" else 1.0
        st = dict(case=case, q=_normal((t, case["heads"] * d), g, case["src"], spread),
                  k=_normal((t, case["kv_heads"] * d), g, case["src"], spread),
                  positions=torch.randint(0, case["far"], (t,), generator=g, device=_DEV).int(),
                  wq=None, wk=None)
        if case["norm"]:
            st["wq"] = _normal((d,), g, "f32", 0.1)
            st["wk"] = _normal((d,), g, "f32", 0.1)
        if own:
            ops, rotary, _ = _package()
            st["ops"] = ops
            st["plan"] = rotary.RotaryPlan(d, rotary_dim=case["rotary_dim"], theta=case["theta"],
                                           layout=case["layout"], scaling=_scaling_argument(case),
                                           device=_DEV)
        return st
    lens, news = _lengths(case)
    layers = case.get("layers", 1)
    spare = sum(-(-n // case["page"]) for n in lens)
    st = dict(case=case, **_pool(case, g, layers, case.get("pages", spare + spare // 8 + 1),
                                 lens, lens))
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    t, d = starts[-1], case["head_dim"]
    if op in ("write", "attention"):
        st["starts"] = None
        if max(news) > 1:
            st["starts"] = torch.tensor(starts, dtype=torch.int32, device=_DEV)
        st["most"] = max(news)
    if op == "write":
        st["k"] = _normal((t, case["kv_heads"] * d), g, case["src"])
        st["v"] = _normal((t, case["kv_heads"] * d), g, case["src"])
    if op == "attention":
        spread = 40.0 if case["src"] == "e4m3" else 1.0
        st["q"] = _normal((t, case["heads"] * d), g, case["src"], spread)
        st["gate"] = _normal((t, case["heads"] * d), g, "e4m3", 60.0) if case["gate"] else None
    if op == "fork":
        n, c = case["seqs"], case["copies"]
        width = st["table"].shape[1]
        more = torch.full((n * c, width), -1, dtype=torch.int32, device=_DEV)
        st["table"] = torch.cat([st["table"], more])
        st["lens"] = torch.cat([st["lens"], st["lens"].new_zeros(n * c)])
        st["src"] = torch.arange(n, device=_DEV, dtype=torch.int32).repeat_interleave(c)
        st["dst"] = torch.arange(n, n + n * c, device=_DEV, dtype=torch.int32)
    if op == "compact":
        st["strewn"] = (st["table"].clone(), st["refs"].clone())
    if own:
        _, _, kvcache = _package()
        st["cache"] = kvcache.Fp4Cache.from_buffers(
            st["storage"], st["table"], st["lens"], st["refs"], page_size=case["page"],
            head_dim=d, k_scale=0.25, v_scale=0.25)
    return st


# ------------------------------------------------------------------------------------ one pass

def run(st):
    case = st["case"]
    op = case["op"]
    if own:
        if op == "rotary":
            q, k = st["ops"].rotary(
                st["q"], st["k"], st["positions"], st["plan"], heads=case["heads"],
                kv_heads=case["kv_heads"], in_scale=_in_scale(case), q_weight=st["wq"],
                k_weight=st["wk"], out_dtype=_DT[case["dst"]])
            return {"q": q, "k": k}
        cache = st["cache"]
        if op == "write":
            cache.write(st["k"], st["v"], starts=st["starts"])
            k, v = cache.read(st["k"].shape[0], starts=st["starts"], dtype=torch.bfloat16)
            return {"k": k, "v": v}
        if op == "attention":
            got = cache.attention(
                st["q"], heads=case["heads"], starts=st["starts"], q_scale=_in_scale(case),
                gate=st["gate"], gate_scale=1 / 64, out_dtype=_DT[case["dst"]],
                ctx_scale=_ctx_scale(case), return_lse=case["lse"])
            return {"out": got[0], "lse": got[1]} if case["lse"] else {"out": got}
        if op == "fork":
            cache.free(st["dst"])
            cache.fork(st["src"], st["dst"])
        else:
            # every pass packs the same strewn pool
            st["table"].copy_(st["strewn"][0])
            st["refs"].copy_(st["strewn"][1])
            cache.compact()
        return {"storage": st["storage"], "table": st["table"], "lens": st["lens"],
                "refs": st["refs"]}
    if op == "rotary":
        w, factor = _frequencies(case)
        angle = st["positions"].double()[:, None] * w
        cos, sin = (angle.cos() * factor).float()[:, None], (angle.sin() * factor).float()[:, None]
        return {"q": _rotate(st["q"], st["wq"], cos, sin, case),
                "k": _rotate(st["k"], st["wk"], cos, sin, case)}
    if op == "write":
        return _write(st)
    if op == "attention":
        return _attend(st)
    if op == "fork":
        return _fork(st)
    return _compact(st)


def _in_scale(case):
    return 1 / 64 if case["src"] == "e4m3" else 1.0


def _ctx_scale(case):
    return 1 / 256 if case["dst"] == "e4m3" else 1.0


def _rotate(x, weight, cos, sin, case):
    d, rot = case["head_dim"], case["rotary_dim"]
    x = x.float().unflatten(-1, (-1, d)) * _in_scale(case)
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * (1.0 + weight)
    y, rest = x[..., :rot], x[..., rot:]
    if case["layout"] == "half":
        a, b = y[..., :rot // 2], y[..., rot // 2:]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = y[..., 0::2], y[..., 1::2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([y, rest], -1).flatten(-2).to(_DT[case["dst"]])


def _owners(st):
    """Sequence and place in its new tokens of every packed token; new tokens of each sequence."""
    b, t = st["lens"].shape[0], (st["k"] if "k" in st else st["q"]).shape[0]
    if st["starts"] is None:
        n = torch.full((b,), t // b, device=_DEV, dtype=torch.int32)
        first = torch.arange(b, device=_DEV, dtype=torch.int32) * (t // b)
    else:
        n, first = st["starts"].diff(), st["starts"][:-1]
    seq = torch.repeat_interleave(torch.arange(b, device=_DEV), n.long(), output_size=t)
    return seq, torch.arange(t, device=_DEV) - first[seq].long(), n


def _write(st):
    case = st["case"]
    seq, i, n = _owners(st)
    pos = st["lens"][seq].long() - n[seq].long() + i
    page = st["table"][seq, pos // case["page"]].long()
    slot = pos % case["page"]
    kc, ks, vc, vs = _parts(st["storage"][0], case)
    out = {}
    for name, codes, scales in (("k", kc, ks), ("v", vc, vs)):
        x = st[name].unflatten(-1, (-1, case["head_dim"]))
        c, s = _pack(x, 0.25)
        codes[page, :, slot] = c
        scales[page, :, slot] = s
        out[name] = _unpack(codes[page, :, slot], scales[page, :, slot], 0.25).flatten(-2).to(
            torch.bfloat16)
    return out


def _attend(st):
    case = st["case"]
    d, hk, hq = case["head_dim"], case["kv_heads"], case["heads"]
    group, b, most = hq // hk, st["lens"].shape[0], st["most"]
    seq, i, n = _owners(st)
    pages = st["storage"][0][st["table"].clamp(min=0).long()]  # [B, pages, H, bytes]
    kc, ks, vc, vs = _parts(pages, case)
    flat = lambda x: x.transpose(2, 3).flatten(1, 2).transpose(1, 2)  # noqa: E731  [B, H, L, D]
    k = flat(_unpack(kc, ks, 0.25))
    v = flat(_unpack(vc, vs, 0.25))
    q = torch.zeros((b, most, hk, group, d), device=_DEV)
    q[seq, i] = st["q"].float().unflatten(-1, (hk, group, d)) * _in_scale(case)
    s = q.permute(0, 2, 1, 3, 4).flatten(2, 3) @ k.transpose(-1, -2) * (1.0 / math.sqrt(d))
    last = st["lens"].long()[:, None] - n.long()[:, None] + torch.arange(most, device=_DEV)
    key = torch.arange(k.shape[2], device=_DEV)
    seen = key <= last.repeat_interleave(group, 1)[:, :, None]  # [B, rows, L]
    s = s.masked_fill(~seen[:, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    ref = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(s - ref)
    total = p.sum(-1, keepdim=True)
    o = torch.where(total > 0, p @ v / total, torch.zeros((), device=_DEV))
    lse = (ref + torch.log(total)).squeeze(-1)
    back = lambda x: x.unflatten(2, (most, group)).transpose(1, 2)[seq, i]  # noqa: E731
    o, lse = back(o).flatten(1), back(lse).flatten(1)
    if case["gate"]:
        o = o * torch.sigmoid(st["gate"].float() / 64)
    if case["dst"] == "e4m3":
        o = (o / _ctx_scale(case)).clamp(-448, 448)
    out = {"out": o.to(_DT[case["dst"]])}
    if case["lse"]:
        out["lse"] = lse
    return out


def _drop(st, rows):
    """Lets go of the pages of `rows`."""
    pages = st["table"][rows]
    st["refs"].scatter_add_(0, pages.clamp(min=0).long().flatten(), -(pages >= 0).int().flatten())
    st["table"][rows] = -1
    st["lens"][rows] = 0


def _fork(st):
    case = st["case"]
    src, dst = st["src"].long(), st["dst"].long()
    _drop(st, dst)
    n = st["lens"][src]
    full, part = n // case["page"], n % case["page"] > 0
    unused = torch.argsort((st["refs"] > 0).int(), stable=True)  # free pages first, ascending
    fresh = unused[part.cumsum(0).clamp(min=1) - 1]
    theirs = st["table"][src]
    col = torch.arange(theirs.shape[1], device=_DEV)
    shared = col < full[:, None]
    tail = part[:, None] & (col == full[:, None])
    none = torch.full_like(theirs, -1)
    st["table"][dst] = torch.where(shared, theirs,
                                   torch.where(tail, fresh.int()[:, None], none))
    st["lens"][dst] = n
    mine = st["table"][dst]
    st["refs"].scatter_add_(0, mine.clamp(min=0).long().flatten(), (mine >= 0).int().flatten())
    last = theirs.gather(1, ((n.long() - 1) // case["page"])[:, None])[:, 0].long()
    to = torch.where(part, fresh, last)  # a full last page is shared: copied onto itself
    st["storage"][:, to] = st["storage"][:, last]
    return {"storage": st["storage"], "table": st["table"], "lens": st["lens"],
            "refs": st["refs"]}


def _compact(st):
    st["table"].copy_(st["strewn"][0])
    st["refs"].copy_(st["strewn"][1])
    refs = st["refs"]
    at = torch.arange(refs.shape[0], device=_DEV)
    used = refs > 0
    front = at < used.sum()
    moved = used & ~front
    holes = torch.argsort((~(~used & front)).int(), stable=True)
    to = torch.where(moved, holes[moved.cumsum(0).clamp(min=1) - 1], at)
    src = moved.nonzero()[:, 0]
    st["storage"][:, to[src]] = st["storage"][:, src]
    table = st["table"]
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()].int(), table))
    refs.copy_(torch.zeros_like(refs).scatter_add_(0, to, refs))
    return {"storage": st["storage"], "table": st["table"], "lens": st["lens"], "refs": refs}


# ------------------------------------------------------------------------------------ 64 bits

def exact(case, seed):
    global own
    op = case["op"]
    if op in ("fork", "compact"):
        return None  # whole numbers and bytes only
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    d = case["head_dim"]
    if op == "rotary":
        w, factor = _frequencies(case)
        turn = torch.polar(torch.full_like(w, factor).expand(case["tokens"], -1).contiguous(),
                           st["positions"].double()[:, None] * w)[:, None]
        got = {}
        for name in ("q", "k"):
            x = st[name].double().reshape(case["tokens"], -1, d) * _in_scale(case)
            if case["norm"]:
                rms = (x.pow(2).sum(-1, keepdim=True) / d + 1e-6).sqrt()
                x = x / rms * (1 + st["w" + name].double())
            rot = x[..., :case["rotary_dim"]]
            two = (rot.unflatten(-1, (2, -1)).transpose(-1, -2) if case["layout"] == "half"
                   else rot.unflatten(-1, (-1, 2)))
            z = torch.view_as_real(torch.view_as_complex(two.contiguous()) * turn)
            z = z.transpose(-1, -2) if case["layout"] == "half" else z
            y = x.clone()
            y[..., :case["rotary_dim"]] = z.reshape(rot.shape)
            got[name] = y.reshape(case["tokens"], -1)
        return got
    lens, news = _lengths(case)
    if op == "write":
        grid = torch.tensor([-v for v in _E2M1[:0:-1]] + _E2M1, dtype=torch.float64, device=_DEV)
        even = torch.tensor([1, 0, 1, 0, 1, 0, 1, 0, 1, 0, 1, 0, 1, 0, 1], device=_DEV)
        got = {}
        for name in ("k", "v"):
            x = st[name].double().reshape(-1, 16)
            s = (x.abs().amax(1, keepdim=True) / 6 / 0.25).clamp(max=448).float().to(
                torch.float8_e4m3fn).double() * 0.25
            y = torch.where(s > 0, x / s, torch.zeros_like(x)).clamp(-6, 6)
            hi = torch.searchsorted(grid, y).clamp(max=14)
            lo = (hi - 1).clamp(min=0)
            up, down = grid[hi] - y, y - grid[lo]
            # nearest value, a tie to the one with an even code
            pick = torch.where((up < down) | ((up == down) & (even[hi] == 0)), hi, lo)
            got[name] = (grid[pick] * s).reshape(st[name].shape)
        return got
    hk, hq = case["kv_heads"], case["heads"]
    out = torch.zeros((sum(news), hq, d), dtype=torch.float64, device=_DEV)
    lse = torch.full((sum(news), hq), -math.inf, dtype=torch.float64, device=_DEV)
    q = st["q"].double().reshape(-1, hq, d) * _in_scale(case)
    one = torch.tensor(_E2M1 + [-v for v in _E2M1], dtype=torch.float64, device=_DEV)
    first = 0
    for b, (n, k) in enumerate(zip(lens, news)):
        used = st["table"][b, :-(-n // case["page"])].long() if n else None
        for h in range(hk if n else 0):
            kv = []
            block = st["storage"][0, used, h].contiguous()
            parts = _parts(block, case)
            for codes, scales in (parts[:2], parts[2:]):
                x = torch.stack([one[(codes & 15).long()], one[(codes >> 4).long()]], -1)
                x = x.reshape(-1, d // 16, 16)
                s = scales.contiguous().view(torch.float8_e4m3fn).double().reshape(-1, d // 16, 1)
                kv.append((x * s * 0.25).reshape(-1, d)[:n])
            heads = slice(h * hq // hk, (h + 1) * hq // hk)
            s = torch.einsum("thd,ld->thl", q[first:first + k, heads], kv[0]) / math.sqrt(d)
            at = torch.arange(n - k, n, device=_DEV)
            s = s.masked_fill(torch.arange(n, device=_DEV) > at[:, None, None], -math.inf)
            total = torch.logsumexp(s, -1)
            lse[first:first + k, heads] = total
            p = torch.exp(s - total[..., None])
            out[first:first + k, heads] = torch.einsum("thl,ld->thd", p, kv[1])
        first += k
    out = out.reshape(sum(news), hq * d)
    if case["gate"]:
        out = out / (1 + torch.exp(-st["gate"].double() / 64))
    out = out / _ctx_scale(case)
    got = {"out": out}
    if case["lse"]:
        got["lse"] = lse.reshape(sum(news), hq)
    return got
