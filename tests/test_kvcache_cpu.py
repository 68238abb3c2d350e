"""CPU-side checks of the serving operators: struct mirrors, refusals of the C entries before any
launch, the frequency plan, and the oracle against itself."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from oracle import serving
from test_abi_cpu import _struct_fields


def _lib():
    from b200fp8 import _lib
    return _lib


@pytest.mark.parametrize("struct,cls", [
    ("b2f_rotary_args", "RotaryArgs"), ("b2f_kv4_cache", "Kv4Cache"),
    ("b2f_kv4_batch", "Kv4Batch"), ("b2f_kv4_write_args", "Kv4WriteArgs"),
    ("b2f_kv4_read_args", "Kv4ReadArgs"), ("b2f_kv4_attn_args", "Kv4AttnArgs"),
    ("b2f_kv4_pool", "Kv4Pool")])
def test_structs_mirror_the_header(struct, cls):
    assert [f[0] for f in getattr(_lib(), cls)._fields_] == _struct_fields(struct)


def _refuses(fn, a, match, **fields):
    """fn(a) with the fields set is refused with a message, and nothing is launched."""
    L = _lib()
    old = {}
    for path, value in fields.items():
        at = a
        *parents, name = path.split("__")
        for p in parents:
            at = getattr(at, p)
        old[path] = (at, name, getattr(at, name))
        setattr(at, name, value)
    assert fn(ctypes.byref(a), None) == L.B2F_ERR_ARG, fields
    assert match in L.lib().b2f_last_error().decode(), L.lib().b2f_last_error()
    for at, name, value in old.values():
        setattr(at, name, value)


def test_rotary_refusals():
    L = _lib()
    lib = L.lib()
    a = L.RotaryArgs()
    lib.b2f_rotary_args_init(ctypes.byref(a))
    assert a.in_scale == a.out_scale == a.magnitude == 1.0 and a.position_bits == 32
    a.rows, a.q_heads, a.k_heads, a.head_dim, a.rotary_dim = 4, 2, 1, 128, 128
    a.q = a.k = a.q_out = a.k_out = a.positions = a.freqs = 4096
    a.q_ld, a.k_ld, a.q_out_ld, a.k_out_ld = 256, 128, 256, 128
    a.q_head_stride = a.k_head_stride = 128
    f = lib.b2f_rotary
    assert f(None, None) == L.B2F_ERR_ARG
    _refuses(f, a, "empty", rows=0)
    _refuses(f, a, "empty", q_heads=0, k_heads=0)
    _refuses(f, a, "head_dim", head_dim=12)
    _refuses(f, a, "head_dim", head_dim=264)
    _refuses(f, a, "rotary_dim", rotary_dim=136)
    _refuses(f, a, "rotary_dim", rotary_dim=4)
    _refuses(f, a, "dtype", in_dtype=4)
    _refuses(f, a, "int32 or int64", position_bits=16)
    _refuses(f, a, "null", freqs=None)
    _refuses(f, a, "null tensor", k=None)
    _refuses(f, a, "misaligned", positions=4098)
    _refuses(f, a, "pitch", q_ld=248)
    _refuses(f, a, "stride", q_head_stride=132)
    _refuses(f, a, "aligned", q=4100)
    _refuses(f, a, "aligned", k_ld=130)
    _refuses(f, a, "out_scale", out_scale=0.0)
    _refuses(f, a, "e4m3 output", out_scale=0.5)
    _refuses(f, a, "go together", q_weight=4096)
    _refuses(f, a, "weights must be", q_weight=4104, k_weight=4096)
    _refuses(f, a, "inverse", q_weight=4096, k_weight=4096, inverse=1)


def _cache(L, a):
    c = a.cache
    c.storage, c.table, c.lens = 4096, 4096, 4096
    c.pages, c.kv_heads, c.head_dim, c.page_size = 8, 2, 128, 16
    c.page_stride = 2 * 16 * 128 * 9 // 8
    c.table_rows, c.table_cols, c.table_ld = 4, 4, 4
    a.batch.seqs, a.batch.tokens = 4, 8


_BAD_CACHES = [
    ("null cache", dict(cache__storage=None)), ("null cache", dict(cache__lens=None)),
    ("head_dim", dict(cache__head_dim=96)), ("page_size", dict(cache__page_size=8)),
    ("empty cache", dict(cache__pages=0)), ("table shape", dict(cache__table_ld=3)),
    ("2^30", dict(cache__table_cols=1 << 28, cache__table_ld=1 << 28)),
    ("page_stride", dict(cache__page_stride=4592)), ("aligned", dict(cache__storage=4104)),
    ("scale", dict(cache__k_scale=0.0)), ("scale", dict(cache__v_scale=math.inf)),
    ("scale", dict(cache__v_scale=math.nan)), ("empty batch", dict(batch__tokens=0)),
    ("multiple of seqs", dict(batch__tokens=9)),
    ("more sequences", dict(batch__seqs=8)), ("misaligned", dict(batch__rows=4097)),
]


@pytest.mark.parametrize("name", ["write", "read", "attn"])
def test_cache_refusals(name):
    L = _lib()
    lib = L.lib()
    cls = {"write": L.Kv4WriteArgs, "read": L.Kv4ReadArgs, "attn": L.Kv4AttnArgs}[name]
    a = cls()
    getattr(lib, f"b2f_kv4_{name}_args_init")(ctypes.byref(a))
    assert a.cache.k_scale == 1.0 and a.cache.v_scale == 1.0
    f = getattr(lib, "b2f_kv4_attention" if name == "attn" else f"b2f_kv4_{name}")
    assert f(None, None) == L.B2F_ERR_ARG
    _cache(L, a)
    if name == "attn":
        a.heads, a.q, a.out, a.q_ld, a.out_ld = 8, 4096, 4096, 1024, 1024
    else:
        a.k = a.v = 4096
        a.k_ld = a.v_ld = 256
    for match, fields in _BAD_CACHES:
        _refuses(f, a, match, **fields)
    if name != "attn":
        _refuses(f, a, "null tensor", k=None)
        _refuses(f, a, "pitch", v_ld=248)
        _refuses(f, a, "aligned", k=4100)
        _refuses(f, a, "", dtype=7)
        if name == "read":
            _refuses(f, a, "f32, bf16 or f16", dtype=L.DTYPE_E4M3)
        return
    _refuses(f, a, "multiple of kv_heads", heads=7)
    _refuses(f, a, "null tensor", q=None)
    _refuses(f, a, "bf16, f16 or e4m3", q_dtype=L.DTYPE_F32)
    _refuses(f, a, "bf16, f16 or e4m3", out_dtype=L.DTYPE_F32)
    _refuses(f, a, "aligned", q_ld=1020)
    _refuses(f, a, "aligned", out=4100)
    _refuses(f, a, "gate must", gate=4096, gate_dtype=L.DTYPE_F32)
    _refuses(f, a, "gate row pitch", gate=4096, gate_ld=1000, gate_head_stride=128)
    _refuses(f, a, "ctx_scale", ctx_scale=0.0)
    _refuses(f, a, "q_scale", q_scale=-1.0)
    _refuses(f, a, "e4m3 output", ctx_scale=0.5)
    _refuses(f, a, "misaligned lse", lse=4097)
    if not torch.cuda.is_available():
        assert lib.b2f_kv4_attention_workspace_bytes(ctypes.byref(a)) == -1


def test_pool_refusals():
    L = _lib()
    lib = L.lib()
    p = L.Kv4Pool()
    p.storage = p.table = p.lens = p.refs = 4096
    p.layers, p.pages, p.page_size, p.page_bytes = 2, 8, 16, 4608
    p.page_stride, p.layer_stride = 4608, 8 * 4608
    p.table_rows, p.table_cols, p.table_ld = 4, 4, 4
    ints = (ctypes.c_int * 2)(0, 1)
    calls = [lambda q, s: lib.b2f_kv4_extend(q, None, 4096, 2, s),
             lambda q, s: lib.b2f_kv4_fork(q, 4096, 4096, 2, 4096, 1 << 20, s),
             lambda q, s: lib.b2f_kv4_free(q, 4096, 2, s),
             lambda q, s: lib.b2f_kv4_compact(q, 4096, 1 << 20, s),
             lambda q, s: lib.b2f_kv4_copy_pages(q, ints, ints, 2, s)]
    for f in calls:
        for match, fields in [("null pool", dict(refs=None)), ("page_size", dict(page_size=48)),
                              ("empty pool", dict(pages=0)), ("2^20", dict(pages=1 << 21)),
                              ("table shape", dict(table_rows=0)),
                              ("page_bytes", dict(page_bytes=4600)),
                              ("page_bytes", dict(page_stride=4592)),
                              ("layer_stride", dict(layer_stride=8)),
                              ("aligned", dict(storage=4104)), ("misaligned", dict(lens=4098))]:
            _refuses(f, p, match, **fields)
    for f, match in [(lambda q, s: lib.b2f_kv4_extend(q, None, 4096, 5, s), "more rows"),
                     (lambda q, s: lib.b2f_kv4_extend(q, 4096, 4096, 1025, s), "1024"),
                     (lambda q, s: lib.b2f_kv4_extend(q, None, None, 2, s), "null rows"),
                     (lambda q, s: lib.b2f_kv4_fork(q, None, 4096, 2, 4096, 64, s), "null rows"),
                     (lambda q, s: lib.b2f_kv4_fork(q, 4096, 4096, 2, 4096, 8, s), "workspace"),
                     (lambda q, s: lib.b2f_kv4_free(q, 4096, 0, s), "1 to 1024"),
                     (lambda q, s: lib.b2f_kv4_compact(q, 4096, 16, s), "workspace"),
                     (lambda q, s: lib.b2f_kv4_copy_pages(q, ints, None, 2, s), "empty list"),
                     (lambda q, s: lib.b2f_kv4_copy_pages(q, ints, (ctypes.c_int * 2)(3, 8), 2, s),
                      "out of range"),
                     (lambda q, s: lib.b2f_kv4_copy_pages(q, ints, (ctypes.c_int * 2)(3, 3), 2, s),
                      "twice"),
                     (lambda q, s: lib.b2f_kv4_copy_pages(q, ints, (ctypes.c_int * 2)(1, 3), 2, s),
                      "both read and written")]:
        _refuses(f, p, match)


def test_python_refusals():
    from b200fp8 import ops, rotary
    from b200fp8.kvcache import Fp4Cache
    with pytest.raises(ValueError, match="page_size"):
        Fp4Cache(layers=1, pages=1, page_size=8, kv_heads=1, head_dim=64, max_seqs=1, max_pages=1,
                 device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        Fp4Cache(layers=1, pages=1, page_size=16, kv_heads=1, head_dim=64, max_seqs=1, max_pages=1,
                 device="cpu")
    storage = torch.zeros((1, 2, 1, 1152), dtype=torch.uint8)
    lists = [torch.zeros((1, 2), dtype=torch.int32), torch.zeros(1, dtype=torch.int32),
             torch.zeros(2, dtype=torch.int32)]
    with pytest.raises(ValueError, match="storage"):
        Fp4Cache.from_buffers(storage[..., ::2], *lists, page_size=16, head_dim=64)
    with pytest.raises(TypeError, match="int32"):
        Fp4Cache.from_buffers(storage, lists[0].long(), *lists[1:], page_size=16, head_dim=64)
    with pytest.raises(ValueError, match="refs"):
        Fp4Cache.from_buffers(storage, lists[0], lists[1], lists[2][:1], page_size=16, head_dim=64)
    plan = rotary.RotaryPlan(64, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        ops.rotary(torch.zeros((1, 64)), None, torch.zeros(1, dtype=torch.int32), plan, heads=1)
    for kw in (dict(head_dim=60), dict(head_dim=264), dict(head_dim=64, rotary_dim=72),
               dict(head_dim=64, rotary_dim=20), dict(head_dim=64, layout="pairs"),
               dict(head_dim=64, theta=0.5), dict(head_dim=64, scaling={"kind": "linear"}),
               dict(head_dim=64, scaling={"kind": "cubic", "factor": 2.0}),
               dict(head_dim=64, scaling={"kind": "yarn", "factor": 2.0}),
               dict(head_dim=64, scaling={"kind": "ntk", "factor": -1.0}),
               dict(head_dim=64, scaling={"kind": "ntk", "factor": 2.0, "fast": 3})):
        with pytest.raises(ValueError):
            rotary.RotaryPlan(kw.pop("head_dim"), device="cpu", **kw)


def test_frequencies():
    from b200fp8.rotary import RotaryPlan, frequencies
    w, m = frequencies(64, 1e4)
    assert m == 1.0 and w[0] == 1.0 and abs(w[16] - 1e-2) < 1e-12
    lin, _ = frequencies(64, 1e4, {"kind": "linear", "factor": 4.0})
    assert all(abs(a / 4 - b) < 1e-15 for a, b in zip(w, lin))
    ntk, _ = frequencies(64, 1e4, {"kind": "ntk", "factor": 4.0})
    assert ntk[0] == 1.0 and abs(ntk[-1] - w[-1] / 4) < 1e-12  # the slowest pair is stretched fully
    y, m = frequencies(64, 1e4, {"kind": "yarn", "factor": 4.0, "original_length": 4096})
    assert abs(m - (0.1 * math.log(4) + 1)) < 1e-12
    assert y[0] == w[0] and abs(y[-1] - w[-1] / 4) < 1e-15
    assert all(b / 4 - 1e-15 <= a <= b + 1e-15 for a, b in zip(y, w))
    plan = RotaryPlan(64, theta=1e4, device="cpu")
    turns = [(int(f) % (1 << 64)) / 2.0 ** 64 for f in plan.freqs]
    assert all(abs(t - x / (2 * math.pi)) < 1e-16 for t, x in zip(turns, w))


@pytest.mark.parametrize("length,factor,lo,hi,last", [
    (131072, 4.0, 45, 70, 0.46), (1048576, 8.0, 59, 84, 0.86)])
def test_a_ramp_of_frequencies_may_end_behind_the_last_pair(length, factor, lo, hi, last):
    """Trained lengths in which every pair turns more than once: none is stretched fully.  Pair i
    of 64 at base 1e4 turns length * 1e4^(-i / 64) / (2 pi) times; the ramp runs from the last
    whole i with 32 turns or more (lo) to the first with one or fewer (hi), which is no pair here."""
    from b200fp8.rotary import frequencies
    turns = lambda i: length * 1e4 ** (-i / 64) / (2 * math.pi)  # noqa: E731
    assert turns(lo) >= 32 > turns(lo + 1) and turns(hi - 1) > 1 >= turns(hi) and turns(63) > 1
    y, _ = frequencies(128, 1e4, {"kind": "yarn", "factor": factor, "original_length": length})
    for i in range(64):
        part = max(0, i - lo) / (hi - lo)  # of the way from w to w / factor
        want = 1e4 ** (-i / 64) * (1 - part + part / factor)
        assert abs(y[i] - want) <= 1e-14 * want, i
    assert abs(y[63] * 1e4 ** (63 / 64) - last) < 0.005


def _pi():
    """pi as a fraction, good to 2^-300: Machin's formula."""
    from fractions import Fraction
    one = 1 << 320

    def arctan_of_inverse(x):
        total, term, k = 0, one // x, 0
        while term:
            total += (-1) ** k * (term // (2 * k + 1))
            term //= x * x
            k += 1
        return total
    return Fraction(4 * (4 * arctan_of_inverse(5) - arctan_of_inverse(239)), one)


@pytest.mark.parametrize("rotary_dim,theta,scaling", [
    (64, 1e4, None), (16, 1e7, None), (128, 1e6, None), (64, 1e4, {"kind": "linear", "factor": 8.0}),
    (16, 1e4, {"kind": "ntk", "factor": 8.0})])
def test_frequencies_are_rounded_once(rotary_dim, theta, scaling):
    """The words of the plan are within half a unit of the exact frequencies, in turns: in whole
    numbers, the power of a word that has no root in it lies between those of its neighbours."""
    from fractions import Fraction
    from b200fp8.rotary import RotaryPlan
    half, pi = rotary_dim // 2, _pi()
    kind, factor = (scaling or {}).get("kind"), int((scaling or {}).get("factor", 1))
    plan = RotaryPlan(rotary_dim, theta=theta, scaling=scaling, device="cpu")
    for i, word in enumerate(plan.freqs.tolist()):
        # w = theta^(-i / half), / factor, or with theta * factor^(half / (half - 1)) as theta
        n = half * (half - 1) if kind == "ntk" else half
        power = Fraction(1, int(theta) ** (i * n // half))
        if kind == "linear":
            power /= factor ** n
        if kind == "ntk":
            power /= factor ** (i * half)
        near = Fraction(10000001, 10000000)  # a little more than a half, for the digits of pi
        low, high = (((word % (1 << 64)) * 2 + s) * pi / (1 << 64) for s in (-near, near))
        assert low ** n <= power <= high ** n, i


def test_oracle_pack_round_trip():
    """Values on the grid survive; a tie goes to the even code; the page layout is the header's."""
    x = torch.tensor([0.0, 0.5, -0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, 0.25, 0.75, 1.25, 1.75, 2.5,
                      3.5, 5.0])
    code, s8, value = serving.pack(x, 1.0)
    assert int(s8[0]) == 0x38  # e4m3 of 1
    assert value.tolist() == [0.0, 0.5, -0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, 0.0, 1.0, 1.0, 2.0,
                              2.0, 4.0, 4.0]
    assert int(code[2]) == 9
    block = torch.zeros(16 * 64 * 9 // 8, dtype=torch.uint8)
    block[1], block[512] = 0x72, 0x40  # element 2 of token 0: code 2, element 3: code 7; scale 2
    k, v = serving.unpack_block(block, 16, 64, 0.5, 1.0)
    assert k[0, :4].tolist() == [0.0, 0.0, 1.0, 6.0] and float(v.abs().sum()) == 0.0


def test_calls_in_the_documents_name_the_arguments_as_the_methods_do():
    """A positional argument of a method that an example or sentence calls stands where the method
    has the parameter of that name."""
    import ast
    import inspect
    import pathlib
    import re
    from b200fp8 import kvcache
    root = pathlib.Path(__file__).resolve().parents[1]
    texts = [kvcache.__doc__, (root / "INTEGRATION.md").read_text()]
    seen = set()
    for call in re.findall(r"cache\.(?:extend|write|read|fork|free|attention)\([^`\n]*?\)",
                           "\n".join(texts)):
        node = ast.parse(call, mode="eval").body
        method = getattr(kvcache.Fp4Cache, node.func.attr)
        names = list(inspect.signature(method).parameters)[1:]
        for arg, name in zip(node.args, names):
            assert isinstance(arg, ast.Name) and arg.id == name, call
        assert {k.arg for k in node.keywords} <= set(names), call
        seen.add(node.func.attr)
    assert {"extend", "write", "attention"} <= seen


def test_page_numbers_beyond_an_int_name_no_page(monkeypatch):
    """copy_pages hands numbers of any size on as numbers out of range, not as their low 32 bits."""
    from b200fp8.kvcache import Fp4Cache
    c = Fp4Cache.__new__(Fp4Cache)
    c.pages, c._pool = 8, _lib().Kv4Pool()
    given = []
    monkeypatch.setattr(Fp4Cache, "_run", lambda self, fn, pool, src, dst, n: given.append(
        (list(src), list(dst))))
    c.copy_pages([2 ** 32 + 1, 3, -2 ** 32, 8], [2 ** 64 + 2, 2 ** 31 + 4, 5, 7])
    (src, dst), = given
    assert src[1] == 3 and dst[2:] == [5, 7]
    assert all(not 0 <= p < 8 for p in (src[0], src[2], src[3], dst[0], dst[1]))


def test_scales_of_scores_have_to_be_finite():
    """A NaN as sm_scale is not "no sm_scale", and a product of scales beyond f32 is not a number."""
    L = _lib()
    a = L.Kv4AttnArgs()
    L.lib().b2f_kv4_attn_args_init(ctypes.byref(a))
    _cache(L, a)
    a.heads, a.q, a.out, a.q_ld, a.out_ld = 8, 4096, 4096, 1024, 1024
    f = L.lib().b2f_kv4_attention
    for bad in (math.nan, math.inf, -math.inf):
        _refuses(f, a, "sm_scale must be finite", sm_scale=bad)
    _refuses(f, a, "passes f32", sm_scale=1e30, q_scale=1e30)
    _refuses(f, a, "passes f32", q_scale=3e38, cache__k_scale=2.0 ** 64)


def test_a_weight_belongs_to_its_own_heads():
    """A k_weight in a call without k does not normalise q, nor the other way round."""
    L = _lib()
    a = L.RotaryArgs()
    L.lib().b2f_rotary_args_init(ctypes.byref(a))
    a.rows, a.q_heads, a.head_dim, a.rotary_dim = 4, 2, 128, 128
    a.q = a.k = a.q_out = a.k_out = a.positions = a.freqs = 4096
    a.q_ld = a.k_ld = a.q_out_ld = a.k_out_ld = 256
    a.q_head_stride = a.k_head_stride = 128
    f = L.lib().b2f_rotary
    # inverse: a call that takes the weight is refused for another reason, and nothing is launched
    _refuses(f, a, "go together", k_weight=4096, inverse=1)
    _refuses(f, a, "go together", q_heads=0, k_heads=2, q_weight=4096, inverse=1)
    _refuses(f, a, "inverse", q_weight=4096, inverse=1)
    _refuses(f, a, "inverse", q_weight=4096, k_weight=4096, inverse=1)


def test_rows_beyond_an_int_are_refused():
    """2^32 + 1 rows of 8 elements fit on the GPU, but not in the C entry's int: one row there."""
    from b200fp8 import ops, rotary
    plan = rotary.RotaryPlan(8, device="cpu")
    for rows in (1 << 31, (1 << 32) + 1):
        q = torch.zeros((1, 8), dtype=torch.float8_e4m3fn).expand(rows, 8)
        with pytest.raises(ValueError, match="rows"):
            ops.rotary(q, None, torch.zeros(1, dtype=torch.int32).expand(rows), plan, heads=1,
                       q_out=q)


def test_a_step_runs_on_the_device_of_its_tensors(monkeypatch):
    """QwenBlock.step launches where its tensors are, whatever the current device, and refuses a
    block, cache and input that are not on one device (devices by fakes: nothing is launched)."""
    from types import SimpleNamespace
    from b200fp8 import blocks
    blk = blocks.QwenBlock.__new__(blocks.QwenBlock)
    blk.h, blk.hk, blk.dh, blk.rot, blk.hidden, blk.eps, blk.ns = 2, 1, 64, 64, 128, 1e-6, 1.0
    now = [0]

    class On:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.old, now[0] = now[0], self.index

        def __exit__(self, *_):
            now[0] = self.old

    class Launched(Exception):
        pass

    def launch(*_, **__):
        raise Launched(now[0])

    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "device", On)
    monkeypatch.setattr(blocks.ops, "norm_quant", launch)
    tensor = lambda i: SimpleNamespace(dim=lambda: 2, shape=(1, 128), get_device=lambda: i)  # noqa: E731
    plan = SimpleNamespace(head_dim=64, rotary_dim=64, interleaved=False)
    for hidden, block, cache in ((1, 1, 1), (0, 0, 0), (0, 1, 1), (1, 0, 1), (1, 1, 0)):
        blk.in_norm = tensor(block)
        kv = SimpleNamespace(kv_heads=1, head_dim=64, device=torch.device("cuda", cache), _index=cache)
        call = lambda: blk.step(tensor(hidden), kv, plan, positions=None)  # noqa: E731
        if hidden == block == cache:
            with pytest.raises(Launched, match=str(hidden)):
                call()
        else:
            with pytest.raises(ValueError, match="one device"):
                call()
    assert now == [0]
