"""CPU checks of the entry points over the 8-bit pool: every refusal happens before the GPU is touched."""
from __future__ import annotations

import pytest

from test_paged import _at, _err
from test_paged import attn_args as attn16
from test_paged import store_args as store16


def _with_scales(a, after, scales):
    """The f16 call's arguments with two more pointers behind the pools."""
    keys = list(a)
    i = keys.index(after) + 1
    return {**{k: a[k] for k in keys[:i]}, **scales, **{k: a[k] for k in keys[i:]}}


SCALES = dict(ks8=_at(0x8000000), vs8=_at(0x8100000))


def store_args(**kw):
    names = ("qo qodt qos q qs k ks v vs dt qn kn ndt eps kp vp nb block pos slots start T nh nkv d rope n_rot theta stream").split()
    a = _with_scales(dict(zip(names, store16())), "vp", SCALES)
    a.update(kw)
    return list(a.values())


def attn_args(**kw):
    names = ("out odt os q qdt qs kp vp nb block table w stride lens cu n T max_new max_len nh nkv d gate gs ws wsb stream").split()
    a = _with_scales(dict(zip(names, attn16())), "vp", SCALES)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,msg", [
    ({"d": 96}, "head_dim"), ({"nkv": 0}, "n_kv_heads"), ({"nh": 40, "qs": 5120, "qos": 5120}, "16 query heads"),
    ({"block": 32}, "block"), ({"block": 0}, "block"), ({"k": None}, "null"), ({"v": None}, "null"), ({"q": None}, "null"),
    ({"kp": None}, "null"), ({"vp": None}, "null"), ({"ks8": None}, "null"), ({"vs8": None}, "null"), ({"qn": None}, "together"),
    ({"dt": 3}, "dtype"), ({"qodt": 9}, "dtype"), ({"ndt": 2}, "norm_dtype"), ({"eps": float("nan")}, "eps"),
    ({"rope": 4}, "rope"), ({"rope": 3, "n_rot": 12}, "n_rot"), ({"theta": 0.0}, "theta"), ({"ks": 252}, "strides"),
    ({"qos": 1000}, "strides"), ({"ks": 258}, "aligned"), ({"k": _at(0x3000008)}, "aligned"), ({"kp": _at(0x6000008)}, "aligned"),
    ({"ks8": _at(0x8000008)}, "aligned"), ({"vs8": _at(0x8100004)}, "aligned"), ({"nb": 1 << 25}, "31 bits"),
    ({"slots": None}, "without slots"), ({"slots": None, "pos": None, "start": 252}, "without slots"), ({"T": 1 << 29}, "too many"),
])
def test_store_refusals(hiplib, kw, msg):
    assert hiplib.yhip_qk_norm_rope_kv8_store(*store_args(**kw)) == -22 and msg in _err(hiplib)


def test_store_of_nothing(hiplib):
    assert hiplib.yhip_qk_norm_rope_kv8_store(*store_args(T=0)) == 0
    assert hiplib.yhip_qk_norm_rope_kv8_store(*store_args(T=0, qo=None, q=None, k=None, v=None, pos=None, slots=None)) == 0


# (the pools take 0x10000 bytes each: 4 blocks of 64 positions, 2 heads of 128; their scales 0x200)
@pytest.mark.parametrize("kw", [
    {"qo": _at(0x6000000 + 0xfff0)}, {"qo": _at(0x7000000 - 4096)}, {"qo": _at(0x8000000 + 0x1f0)}, {"qo": _at(0x8100000 - 10224)},
    {"qo": _at(0x5000000)}, {"qo": _at(0x5200000)}, {"qo": _at(0x5300000 - 10224)}, {"vp": _at(0x6000000 + 0xfff0)},
    {"kp": _at(0x2000000)}, {"kp": _at(0x3000000 - 0xfff0)}, {"vp": _at(0x4000000)}, {"kp": _at(0x5000000)},
    {"ks8": _at(0x6000000)}, {"vs8": _at(0x8000000 + 0x1f0)}, {"ks8": _at(0x7000000 - 0x1f0)}, {"vs8": _at(0x3000000)},
    {"ks8": _at(0x2000000)}, {"ks8": _at(0x5200000)}, {"vs8": _at(0x5300000)}, {"vs8": _at(0x5100000 - 0x1f0)},
    {"ks8": _at(0x4000000), "qo": None, "q": None},
])
def test_store_overlaps(hiplib, kw):
    assert hiplib.yhip_qk_norm_rope_kv8_store(*store_args(**kw)) == -22 and "overlap" in _err(hiplib)


@pytest.mark.parametrize("kw,msg", [
    ({"out": None}, "null"), ({"q": None}, "null"), ({"kp": None}, "null"), ({"vp": None}, "null"), ({"ks8": None}, "null"),
    ({"vs8": None}, "null"), ({"table": None}, "null"), ({"lens": None}, "null"), ({"cu": None}, "null"), ({"odt": 3}, "dtype"),
    ({"qdt": 4}, "dtype"), ({"block": 16}, "block"), ({"block": 192}, "block"), ({"d": 80}, "head_dim"), ({"nkv": 0}, "n_kv_heads"),
    ({"nh": 34, "os": 4352, "qs": 4352}, "16 query heads"), ({"w": 0}, "max_blocks"), ({"stride": 3}, "max_blocks"),
    ({"max_len": 0}, "max_len"), ({"max_len": 257}, "max_len"), ({"n": 65536}, "n_seq"), ({"n": 65535, "nkv": 129, "nh": 129, "qs": 16512, "os": 16512}, "too many sequences"), ({"nb": 1 << 31}, "too many blocks"),
    ({"w": 1 << 22, "stride": 1 << 22, "max_len": 1 << 27, "T": 1 << 20, "max_new": 1 << 20, "q": _at(1 << 40)}, "in chunks"),
    ({"max_new": 6}, "max_new"), ({"qs": 1000}, "stride"), ({"os": 1028}, "stride"), ({"gate": _at(0x8800000), "gs": 1000}, "gate_stride"),
    ({"q": _at(0x2000008)}, "aligned"), ({"out": _at(0x1000004)}, "aligned"), ({"kp": _at(0x6000008)}, "aligned"),
    ({"ks8": _at(0x8000008)}, "aligned"), ({"vs8": _at(0x8100001)}, "aligned"), ({"out": _at(0x2000000)}, "overlaps"),
])
def test_attn_refusals(hiplib, kw, msg):
    assert hiplib.yhip_paged_attn8(*attn_args(**kw)) == -22 and msg in _err(hiplib)


def test_attn_of_nothing(hiplib):
    null = dict(out=None, q=None, kp=None, vp=None, ks8=None, vs8=None, table=None, lens=None)
    for kw in ({"T": 0, "max_new": 0}, {"n": 0}, {"max_new": 0}, {"T": 0, "max_new": 0, **null}, {"n": 0, **null}):
        assert hiplib.yhip_paged_attn8(*attn_args(**kw)) == 0


def test_attn_of_too_much_in_all(hiplib):
    """Each sequence fits a call, all of them do not."""
    big = dict(n=65535, T=65535, max_new=1, max_len=0x7fffffff, w=32768, stride=32768, block=65536, q=_at(1 << 40))
    assert hiplib.yhip_paged_attn8(*attn_args(**big)) == -22 and "in chunks" in _err(hiplib)


@pytest.mark.parametrize("kw", [
    {"out": _at(0x6000000 + 0xfff0)}, {"out": _at(0x7000000 - 4096)}, {"out": _at(0x8000000)}, {"out": _at(0x8100000 - 4096)},
    {"out": _at(0x5000000)}, {"out": _at(0x5100000 - 4096)}, {"out": _at(0x5200000 - 10224)}, {"vs8": _at(0x1000000 + 10224)},
    {"ws": _at(0x1000000 + 10224)}, {"ws": _at(0x2000000 - 16)}, {"ws": _at(0x6000000 + 0xfff0)}, {"ws": _at(0x7000000)},
    {"ws": _at(0x8000000 + 0x1f0)}, {"ws": _at(0x8100000)}, {"ws": _at(0x5000020)}, {"ws": _at(0x5100000)}, {"ws": _at(0x5200000)},
    {"gate": _at(0x9000000), "gs": 1024, "ws": _at(0x9000000 + 5 * 4096 - 16)},
])
def test_attn_overlaps(hiplib, kw):
    kw = dict(w=64, stride=64, max_len=4096, wsb=1 << 30, **{"ws": _at(1 << 40), **kw})
    assert hiplib.yhip_paged_attn8(*attn_args(**kw)) == -22 and "overlaps" in _err(hiplib)


@pytest.mark.parametrize("kw", [{}, {"max_new": 5}, {"d": 64, "os": 512, "qs": 512}])
def test_attn_workspace_of_calls_that_need_one(hiplib, kw):
    kw = dict(w=64, stride=64, max_len=4096, **kw)
    a = dict(zip(("T", "n", "max_new", "max_len", "nh", "nkv", "d"), (5, 3, kw.get("max_new", 2), 4096, 8, 2, kw.get("d", 128))))
    need = hiplib.yhip_paged_attn8_workspace(*a.values())
    assert need > 0
    for ws, n in ((None, need), (_at(1 << 40), need - 1), (_at(1 << 40), 0), (_at((1 << 40) + 8), need)):
        assert hiplib.yhip_paged_attn8(*attn_args(**kw, ws=ws, wsb=n)) == -28 and "workspace" in _err(hiplib)


def test_a_workspace_for_more_serves_less(hiplib):
    """Every bound lowered on its own or with the others: never more bytes."""
    need = hiplib.yhip_paged_attn8_workspace
    for d in (64, 128, 256):
        for nh, nkv in ((14, 2), (28, 4), (32, 8), (16, 16)):
            for T, n, mn, ml in ((4096, 64, 512, 32768), (600, 3, 500, 700), (64, 64, 1, 131072), (40, 10, 4, 1500), (2048, 1, 2048, 4096)):
                most = need(T, n, mn, ml, nh, nkv, d)
                for t2 in (T, T // 2, n):
                    for n2 in (n, (n + 1) // 2, 1):
                        for mn2 in (mn, max(1, mn // 3), 1):
                            for ml2 in (ml, ml // 2 + 1, 300, 1):
                                if mn2 <= t2:
                                    assert need(t2, n2, mn2, min(ml2, ml), nh, nkv, d) <= most, (d, nh, nkv, T, n, mn, ml, t2, n2, mn2, ml2)


def from_args(**kw):
    a = dict(k8=_at(0x1000000), v8=_at(0x2000000), ks=_at(0x3000000), vs=_at(0x3100000), n8=4, kc=_at(0x4000000), vc=_at(0x5000000),
             n16=5, dst=_at(0x6000000), src=_at(0x6100000), n=3, block=64, nkv=2, d=128, stream=None)
    a.update(kw)
    return list(a.values())


def to_args(**kw):
    a = dict(kc=_at(0x4000000), vc=_at(0x5000000), n16=5, k8=_at(0x1000000), v8=_at(0x2000000), ks=_at(0x3000000), vs=_at(0x3100000),
             n8=4, dst=_at(0x6000000), src=_at(0x6100000), n=3, block=64, nkv=2, d=128, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,msg", [
    ({"block": 96}, "power of two"), ({"block": 32}, "power of two"), ({"d": 96}, "head_dim"), ({"nkv": 0}, "n_kv_heads"),
    *[({k: None}, "null") for k in ("k8", "v8", "ks", "vs", "kc", "vc", "dst", "src")],
    *[({k: _at(0x9000008)}, "aligned") for k in ("k8", "v8", "ks", "vs", "kc", "vc")],
    ({"n8": 1 << 31}, "too many"), ({"n16": 1 << 31}, "too many"), ({"n": 1 << 31}, "too many"), ({"n": 1 << 30}, "too many"),
    ({"n": 1 << 20, "block": 65536}, "too many"), ({"n": 1 << 23}, "too many"), ({"n": 1 << 22, "block": 128}, "too many"),
])
def test_pages_refusals(hiplib, kw, msg):
    assert hiplib.yhip_kv8_from_pages(*from_args(**kw)) == -22 and msg in _err(hiplib)
    assert hiplib.yhip_kv8_to_pages(*to_args(**kw)) == -22 and msg in _err(hiplib)


# (8-bit pools of 0x10000 bytes with scales of 0x200, f16 pools of 0x28000)
@pytest.mark.parametrize("f,args,kw", [
    *[("yhip_kv8_from_pages", from_args, kw) for kw in (
        {"v8": _at(0x1000000 + 0xfff0)}, {"ks": _at(0x2000000)}, {"vs": _at(0x3000000 + 0x1f0)}, {"k8": _at(0x4000000 + 0x27ff0)},
        {"vs": _at(0x5000000 - 0x1f0)}, {"dst": _at(0x1000000)}, {"src": _at(0x3100000 + 0x1fc)})],
    *[("yhip_kv8_to_pages", to_args, kw) for kw in (
        {"vc": _at(0x4000000 + 0x27ff0)}, {"kc": _at(0x1000000 + 0xfff0)}, {"vc": _at(0x3100000 - 0x27ff0)}, {"dst": _at(0x5000000)},
        {"src": _at(0x4000000 + 0x27ffc)})],
])
def test_pages_overlaps(hiplib, f, args, kw):
    assert getattr(hiplib, f)(*args(**kw)) == -22 and "overlaps" in _err(hiplib)


def test_pages_of_nothing(hiplib):
    none = {k: None for k in ("k8", "v8", "ks", "vs", "kc", "vc", "dst", "src")}
    for kw in ({}, none):
        assert hiplib.yhip_kv8_from_pages(*from_args(n=0, **kw)) == 0 and hiplib.yhip_kv8_to_pages(*to_args(n=0, **kw)) == 0


def test_python_refusals():
    torch = pytest.importorskip("torch")
    from yllm_amd import YhipError
    from yllm_amd import paged as PG

    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    kv = PG.PagedKV8.empty(4, 2, 128, device="cpu")
    assert (kv.n_blocks, kv.n_kv, kv.block, kv.head_dim) == (4, 2, 64, 128)
    assert not kv.k.view(torch.uint8).any() and kv.v.shape == (4, 2, 1, 128, 64) and kv.k_scale.shape == kv.v_scale.shape == (4, 2, 64)
    half = PG.PagedKV.empty(4, 2, 128, device="cpu")
    q, k = torch.zeros(5, 1024), torch.zeros(5, 256)
    A, S = PG.paged_attn8, PG.qk_norm_rope_kv8_store
    wrong = [PG.PagedKV8(kv.v, kv.v, kv.k_scale, kv.v_scale), PG.PagedKV8(kv.k, kv.k, kv.k_scale, kv.v_scale),
             PG.PagedKV8(kv.k, kv.v, kv.k_scale[:3], kv.v_scale), PG.PagedKV8(kv.k, kv.v, kv.k_scale, kv.v_scale.view(torch.uint8)),
             PG.PagedKV8(kv.k.view(torch.uint8), kv.v, kv.k_scale, kv.v_scale), half]
    bad = [lambda: PG.PagedKV8.empty(4, 2, 128, block=48, device="cpu"),
           lambda: PG.PagedKV8.empty(1, 1, 64, block=1 << 17, device="cpu"),
           *[lambda c=c: A(q, c, i(3, 4), i(3), i(4), 8, 2) for c in wrong],
           *[lambda c=c: S(c, q, k, k, 8, 2, 1e6, positions=i(5), slots=i(5)) for c in wrong],
           *[lambda c=c: PG.kv8_from_pages(c, half, i(3), i(3)) for c in wrong],
           *[lambda c=c: PG.kv8_to_pages(half, c, i(3), i(3)) for c in wrong],
           lambda: PG.paged_attn(q, kv, i(3, 4), i(3), i(4), 8, 2),                          # an 8-bit pool for an f16 one
           lambda: PG.qk_norm_rope_kv_store(kv, q, k, k, 8, 2, 1e6, positions=i(5), slots=i(5)),
           lambda: S(kv, q, k, k, 8, 2, 1e6, positions=i(5), slots=i(5)),                    # on the CPU
           lambda: S(kv, q, k, k, 8, 2, 1e6, slots=i(5)), lambda: S(kv, q, k, k.half(), 8, 2, 1e6, pos_start=0),
           lambda: S(kv, q[:4], k, k, 8, 2, 1e6), lambda: S(kv, q, k, k[:, :200], 8, 2, 1e6),
           lambda: A(q, kv, i(3, 4), i(3), i(4), 8, 2), lambda: A(q, kv, i(3, 4), i(3), i(3), 8, 2),
           lambda: A(q[:, :512], kv, i(3, 4), i(3), i(4), 8, 2), lambda: A(q, kv, i(3, 4), i(3).long(), i(4), 8, 2),
           lambda: A(q, kv, i(3, 4), i(3), i(4), 8, 2, gate=torch.zeros(5, 1024).half()),
           lambda: PG.kv8_from_pages(kv, half, i(3), i(3)),                                  # on the CPU
           lambda: PG.kv8_to_pages(half, kv, i(3), i(4)), lambda: PG.kv8_to_pages(half, kv, i(3).long(), i(3)),
           lambda: PG.kv8_from_pages(kv, PG.PagedKV.empty(4, 2, 128, block=128, device="cpu"), i(3), i(3)),
           lambda: PG.kv8_from_pages(kv, PG.PagedKV.empty(4, 1, 128, device="cpu"), i(3), i(3))]
    for f in bad:
        with pytest.raises(YhipError):
            f()


# ---- yhip_call: the same entry points by number, their arguments as words ------------------------------

def _calls():
    from test_paged import plan_args

    from yllm_amd._lib import CALLS

    args = (plan_args, store16, attn16, store_args, attn_args, from_args, to_args)
    return dict(zip(CALLS, args))


def test_call_numbers_are_those_of_the_header():
    import re
    from pathlib import Path

    from yllm_amd._lib import CALLS

    text = (Path(__file__).resolve().parent.parent / "include" / "yllm_hip.h").read_text()
    numbers = {n.lower(): int(v) for n, v in re.findall(r"#define YHIP_CALL_(\w+) (\d+)u", text)}
    assert numbers == {n[5:]: i for i, n in enumerate(CALLS)}


@pytest.mark.parametrize("name", ["yhip_paged_plan", "yhip_qk_norm_rope_kv_store", "yhip_paged_attn", "yhip_qk_norm_rope_kv8_store",
                                  "yhip_paged_attn8", "yhip_kv8_from_pages", "yhip_kv8_to_pages"])
def test_calls_by_number_answer_as_the_entry_points_do(hiplib, name):
    """Every argument in turn as 0, as 1 and as a large value: calls that are refused are refused with the same words (those
    that would launch are left out: there is nothing at these addresses)."""
    from yllm_amd import YhipError
    from yllm_amd._lib import SIGNATURES, fast

    base = [getattr(a, "value", a) for a in _calls()[name]()]
    direct, types = getattr(hiplib, name), SIGNATURES[name][1]
    floats = {i for i, t in enumerate(types) if t.__name__ == "c_float"}
    assert len(base) == len(types)
    # (a base that is refused last of all: its written tensors overlap)
    same = {"yhip_paged_plan": (11, 12), "yhip_qk_norm_rope_kv_store": (15, 14), "yhip_paged_attn": (0, 6),
            "yhip_qk_norm_rope_kv8_store": (15, 14), "yhip_paged_attn8": (0, 6), "yhip_kv8_from_pages": (1, 0), "yhip_kv8_to_pages": (1, 0)}[name]
    base[same[0]] = base[same[1]]
    assert direct(*base) == -22
    said = 0
    for i in range(len(base) - 1):
        if i in same:
            continue                                              # (without the overlap it would launch)
        for v in (0, 1, 0x7ffffff0, base[i]):
            a = list(base)
            a[i] = float(v) if i in floats and v is not None else v
            rc = direct(*a)
            if rc == 0:
                continue
            msg = _err(hiplib)
            assert fast(name)(*a) == rc and _err(hiplib) == msg, (i, v)
            said += 1
    assert said > len(base)
    with pytest.raises(YhipError):
        fast(name)(*base[:-1])                                    # too few
    i = next(k for k, t in enumerate(types) if t.__name__ in ("c_uint", "c_uint32"))
    a = list(base)
    a[i] = (1 << 32) + 1
    assert fast(name)(*a) == -22 and "does not fit" in _err(hiplib)
    for bad in (-1, 1 << 64, "x"):
        a[i] = bad
        with pytest.raises(YhipError):
            fast(name)(*a)


def test_calls_that_are_none(hiplib):
    words = bytes(8 * 40)
    assert hiplib.yhip_call(7, words, 16) == -22 and "no call" in _err(hiplib)
    assert hiplib.yhip_call(0, words, 15) == -22 and "words" in _err(hiplib)
    assert hiplib.yhip_call(0, None, 16) == -22 and "words" in _err(hiplib)


@pytest.mark.parametrize("name", ["yhip_paged_plan", "yhip_qk_norm_rope_kv_store", "yhip_paged_attn", "yhip_qk_norm_rope_kv8_store",
                                  "yhip_paged_attn8", "yhip_kv8_from_pages", "yhip_kv8_to_pages"])
def test_only_a_pointer_may_be_none(hiplib, name):
    """None for a number is refused wherever it stands, as the entry point's own binding refuses it; for a pointer it is null."""
    import ctypes

    from yllm_amd import YhipError
    from yllm_amd._lib import SIGNATURES, fast

    base = [getattr(a, "value", a) for a in _calls()[name]()]
    direct, types = getattr(hiplib, name), SIGNATURES[name][1]
    # (block or head_dim 0 is refused before anything would launch)
    k = next(k for k in range(len(base)) if base[k] == 64 and direct(*base[:k], 0, *base[k + 1:]) == -22)
    nothing = list(base)
    nothing[k] = 0
    for i, t in enumerate(types):
        for a in (list(base), list(nothing)):
            a[i] = None
            if t is ctypes.c_void_p:
                if a[k] == 0:
                    assert fast(name)(*a) == direct(*a) == -22
                continue
            with pytest.raises(ctypes.ArgumentError):
                direct(*a)
            with pytest.raises(YhipError, match=f"argument {i} .*None") as e:
                fast(name)(*a)
            assert e.value.code == -22


@pytest.mark.parametrize("eight", [False, True])
def test_attention_without_a_number(hiplib, monkeypatch, eight):
    """A max_new of None is refused with a workspace as without one (max_len alone may be None)."""
    torch = pytest.importorskip("torch")
    from yllm_amd import YhipError
    from yllm_amd import paged as PG

    monkeypatch.setattr(PG, "elsewhere", lambda *a: None)           # (as if these tensors were on the current GPU)
    monkeypatch.setattr(PG, "_stream", lambda: 0)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    cache = (PG.PagedKV8 if eight else PG.PagedKV).empty(4, 2, 128, device="cpu")
    f = PG.paged_attn8 if eight else PG.paged_attn
    with pytest.raises(YhipError, match="None"):
        f(torch.zeros(5, 1024), cache, i(3, 4), i(3), i(4), 8, None, 256, workspace=torch.zeros(1 << 20, dtype=torch.uint8))


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("start", [0, -1, -(1 << 31), 1 << 32])
def test_a_start_that_slots_make_unused(hiplib, monkeypatch, eight, start):
    """With slots a row's place and position are its own: pos_start may hold any number (-1 for "none", say).  The call gets as
    far as its last check, that q_out overlaps k."""
    torch = pytest.importorskip("torch")
    from yllm_amd import YhipError
    from yllm_amd import paged as PG

    monkeypatch.setattr(PG, "elsewhere", lambda *a: None)           # (as if these tensors were on the current GPU)
    monkeypatch.setattr(PG, "_stream", lambda: 0)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    cache = (PG.PagedKV8 if eight else PG.PagedKV).empty(4, 2, 128, device="cpu")
    f = PG.qk_norm_rope_kv8_store if eight else PG.qk_norm_rope_kv_store
    row = torch.zeros(5, 1024)
    args = (torch.zeros(5, 1024), row[:, 512:768], torch.zeros(5, 256), 8, 2, 1e6)
    with pytest.raises(YhipError, match="q_out overlaps"):
        f(cache, *args, positions=i(5), slots=i(5), pos_start=start, q_out=row)
    for wrong in (None, "0", 1.5):
        with pytest.raises(YhipError):
            f(cache, *args, positions=i(5), slots=i(5), pos_start=wrong, q_out=row)
    if start < 0:
        with pytest.raises(YhipError, match="range"):
            f(cache, *args, pos_start=start, q_out=row)


def test_a_waves_share_of_the_lds_holds_all_that_is_put_into_it(tmp_path):
    """The few-row kernel's shares (csrc/paged_decode8_lds.hpp, compiled for the host): each holds a wave's rows [16][D + 4] with
    16 maxima, 16 sums and a flag, and the first one before that the queries as f16 [1 or 2 parts][16][D + 8], whatever lies
    behind it; a multiple of 16 bytes."""
    import subprocess
    from pathlib import Path

    csrc = Path(__file__).resolve().parent.parent / "yllm_amd" / "csrc"
    src, exe = tmp_path / "lds.cpp", tmp_path / "lds"
    sizes = [(d, prec) for d in (64, 128, 256) for prec in ("false", "true")]
    src.write_text('#include "paged_decode8_lds.hpp"\n#include <stdio.h>\nint main() {\n'
                   + "".join(f'printf("%d\\n", yhip::kDecode8Lds<{d}, {p}>);\n' for d, p in sizes) + "}\n")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", f"-I{csrc}", str(src), "-o", str(exe)], check=True)
    got = [4 * int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    for (d, prec), have in zip(sizes, got, strict=True):
        rows, queries = 4 * (16 * (d + 4) + 16 + 16 + 1), 2 * (2 if prec == "true" else 1) * 16 * (d + 8)
        assert have >= max(rows, queries) and have % 16 == 0, (d, prec, have, rows, queries)
