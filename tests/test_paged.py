"""CPU checks of the paged entry points: every refusal happens before the GPU is touched."""
from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

import pytest

P = ctypes.c_void_p(0x100000)  # never dereferenced: validation fails first
Q = ctypes.c_void_p(0x40000000)


def _at(x):
    return ctypes.c_void_p(x)


def _err(lib):
    return lib.yhip_last_error().decode()


def plan_args(**kw):
    a = dict(table=_at(0x10000), w=4, stride=4, ctx=_at(0x20000), new=_at(0x30000), free=_at(0x40000), cap=10,
             n_free=_at(0x50000), n_seq=3, n_tok=9, block=64, cu=_at(0x60000), lens=_at(0x70000), slots=_at(0x80000),
             pos=_at(0x90000), counts=_at(0xa0000), stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,msg", [
    ({"block": 32}, "power of two"), ({"block": 96}, "power of two"), ({"block": 1 << 17}, "power of two"),
    ({"n_seq": 8193}, "n_seq"), ({"n_tok": 1 << 31}, "31 bits"), ({"w": 0}, "max_blocks"), ({"w": 5}, "table_stride"),
    ({"table": None}, "null"), ({"ctx": None}, "null"), ({"new": None}, "null"), ({"n_free": None}, "null"),
    ({"free": None}, "null"), ({"cu": None}, "null"), ({"lens": None}, "null"), ({"slots": None}, "null"),
    ({"pos": None}, "null"), ({"counts": None}, "null"),
    ({"lens": _at(0x20000)}, "overlaps an input"), ({"counts": _at(0x50000)}, "overlaps an input"),
    ({"counts": _at(0x50000 - 12)}, "overlaps an input"), ({"slots": _at(0x90000 - 4)}, "two outputs"),
    ({"table": _at(0x40000 - 40)}, "overlaps an input"),
])
def test_plan_refusals(hiplib, kw, msg):
    assert hiplib.yhip_paged_plan(*plan_args(**kw)) == -22 and msg in _err(hiplib)


def store_args(**kw):
    a = dict(qo=_at(0x1000000), qodt=1, qos=1024, q=_at(0x2000000), qs=1024, k=_at(0x3000000), ks=256,
             v=_at(0x4000000), vs=256, dt=1, qn=_at(0x5000000), kn=_at(0x5100000), ndt=1, eps=1e-6, kp=_at(0x6000000),
             vp=_at(0x7000000), nb=4, block=64, pos=_at(0x5200000), slots=_at(0x5300000), start=0, T=5, nh=8, nkv=2,
             d=128, rope=2, n_rot=0, theta=1e6, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,msg", [
    ({"d": 96}, "head_dim"), ({"nkv": 0}, "n_kv_heads"), ({"nh": 1}, "n_kv_heads"), ({"nh": 40, "qs": 5120, "qos": 5120}, "16 query heads"),
    ({"block": 32}, "block"), ({"block": 0}, "block"), ({"k": None}, "null"), ({"v": None}, "null"), ({"q": None}, "null"),
    ({"kp": None}, "null"), ({"vp": None}, "null"), ({"qn": None}, "together"), ({"kn": None}, "together"),
    ({"dt": 3}, "dtype"), ({"qodt": 9}, "dtype"), ({"ndt": 2}, "norm_dtype"), ({"eps": -1.0}, "eps"),
    ({"eps": float("nan")}, "eps"), ({"rope": 4}, "rope"), ({"rope": 3, "n_rot": 0}, "n_rot"), ({"rope": 3, "n_rot": 12}, "n_rot"),
    ({"rope": 3, "n_rot": 136}, "n_rot"), ({"theta": 0.0}, "theta"), ({"ks": 252}, "strides"), ({"vs": 128}, "strides"),
    ({"qs": 1000}, "strides"), ({"qos": 1000}, "strides"), ({"ks": 258}, "aligned"), ({"k": _at(0x3000008)}, "aligned"),
    ({"qn": _at(0x5000004)}, "aligned"), ({"kp": _at(0x6000008)}, "aligned"), ({"nb": 1 << 25}, "31 bits"),
    ({"slots": None}, "without slots"), ({"slots": None, "pos": None, "start": 252}, "without slots"),
    ({"T": 1 << 29}, "too many"), ({"qo": _at(0x2000000 + 64)}, "overlaps"), ({"qo": _at(0x2000000), "qodt": 0}, "overlaps"),
    ({"qo": _at(0x3000000)}, "overlaps"), ({"qo": _at(0x4000000 - 512)}, "overlaps"),
])
def test_store_refusals(hiplib, kw, msg):
    assert hiplib.yhip_qk_norm_rope_kv_store(*store_args(**kw)) == -22 and msg in _err(hiplib)


def test_store_of_nothing(hiplib):
    assert hiplib.yhip_qk_norm_rope_kv_store(*store_args(T=0)) == 0
    assert hiplib.yhip_qk_norm_rope_kv_store(*store_args(T=0, qo=None, q=None, k=None, v=None, pos=None, slots=None)) == 0


def test_positions_past_31_bits(hiplib):
    """Rows with slots and no positions count from pos_start."""
    assert hiplib.yhip_qk_norm_rope_kv_store(*store_args(pos=None, start=0x7ffffffc)) == -22 and "31 bits" in _err(hiplib)
    assert hiplib.yhip_qk_norm_rope_kv_store(*store_args(pos=None, start=0xffffffff)) == -22 and "31 bits" in _err(hiplib)


def test_attn_of_too_much_in_all(hiplib):
    """Each sequence fits a call, all of them do not."""
    big = dict(n=65535, T=65535, max_new=1, max_len=0x7fffffff, w=32768, stride=32768, block=65536, q=_at(1 << 40))
    assert hiplib.yhip_paged_attn(*attn_args(**big)) == -22 and "in chunks" in _err(hiplib)


def attn_args(**kw):
    a = dict(out=_at(0x1000000), odt=1, os=1024, q=_at(0x2000000), qdt=1, qs=1024, kp=_at(0x6000000), vp=_at(0x7000000),
             nb=4, block=64, table=_at(0x5000000), w=4, stride=4, lens=_at(0x5100000), cu=_at(0x5200000), n=3, T=5,
             max_new=2, max_len=200, nh=8, nkv=2, d=128, gate=None, gs=0, ws=None, wsb=0, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,msg", [
    ({"out": None}, "null"), ({"q": None}, "null"), ({"kp": None}, "null"), ({"vp": None}, "null"), ({"table": None}, "null"),
    ({"lens": None}, "null"), ({"cu": None}, "null"), ({"odt": 3}, "dtype"), ({"qdt": 4}, "dtype"), ({"block": 16}, "block"),
    ({"block": 192}, "block"), ({"d": 80}, "head_dim"), ({"nkv": 0}, "n_kv_heads"), ({"nh": 34, "os": 4352, "qs": 4352}, "16 query heads"),
    ({"w": 0}, "max_blocks"), ({"stride": 3}, "max_blocks"), ({"max_len": 0}, "max_len"), ({"max_len": 257}, "max_len"),
    ({"n": 65536}, "n_seq"), ({"nb": 1 << 31}, "too many blocks"), ({"w": 1 << 22, "stride": 1 << 22, "max_len": 1 << 27, "T": 1 << 20, "max_new": 1 << 20, "q": _at(1 << 40)}, "in chunks"), ({"max_new": 6}, "max_new"), ({"qs": 1000}, "stride"), ({"os": 1028}, "stride"),
    ({"gate": _at(0x8000000), "gs": 1000}, "gate_stride"), ({"q": _at(0x2000008)}, "aligned"), ({"out": _at(0x1000004)}, "aligned"),
    ({"kp": _at(0x6000008)}, "aligned"), ({"out": _at(0x2000000)}, "overlaps"), ({"gate": _at(0x1000000 + 4096), "gs": 1024}, "overlaps"),
])
def test_attn_refusals(hiplib, kw, msg):
    assert hiplib.yhip_paged_attn(*attn_args(**kw)) == -22 and msg in _err(hiplib)


def test_attn_of_nothing(hiplib):
    null = dict(out=None, q=None, kp=None, vp=None, table=None, lens=None)
    for kw in ({"T": 0, "max_new": 0}, {"n": 0}, {"max_new": 0}, {"T": 0, "max_new": 0, **null}, {"n": 0, **null}):
        assert hiplib.yhip_paged_attn(*attn_args(**kw)) == 0


def test_attn_workspace_is_checked(hiplib):
    need = hiplib.yhip_paged_attn_workspace(5, 3, 2, 200, 8, 2, 128)
    if need:
        assert hiplib.yhip_paged_attn(*attn_args(ws=P, wsb=need - 1)) == -28 and "workspace" in _err(hiplib)
        assert hiplib.yhip_paged_attn(*attn_args(ws=_at(0x100008), wsb=need)) == -28


def test_python_refusals():
    torch = pytest.importorskip("torch")
    from yllm_amd import YhipError
    from yllm_amd import paged as PG

    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    kv = PG.PagedKV.empty(4, 2, 128, device="cpu")
    assert (kv.n_blocks, kv.n_kv, kv.block, kv.head_dim) == (4, 2, 64, 128)
    flat = PG.PagedKV(kv.k, kv.k.clone())  # V in rows, as K
    bad = [lambda: PG.PagedKV.empty(4, 2, 128, block=48, device="cpu"),
           lambda: PG.PagedKV.empty(1, 1, 64, block=1 << 17, device="cpu"),
           lambda: PG.paged_attn(torch.zeros(5, 1024), flat, i(3, 4), i(3), i(4), 8, 2),
           lambda: PG.qk_norm_rope_kv_store(flat, None, torch.zeros(5, 256), torch.zeros(5, 256), 8, 2, 1e6),
           lambda: PG.paged_plan(i(3, 4), i(3), i(3), i(9), i(1), 64, 9),                   # on the CPU
           lambda: PG.paged_plan(i(3, 4).t(), i(4), i(4), i(9), i(1), 64, 9),
           lambda: PG.paged_plan(i(3, 4).long(), i(3), i(3), i(9), i(1), 64, 9),
           lambda: PG.paged_plan(i(3, 4), i(2), i(3), i(9), i(1), 64, 9),
           lambda: PG.paged_plan(i(3, 4), i(3), i(3), i(9), i(2), 64, 9)]
    q, k = torch.zeros(5, 1024), torch.zeros(5, 256)
    S = PG.qk_norm_rope_kv_store
    bad += [lambda: S(kv, q, k, k, 8, 2, 1e6, positions=i(5), slots=i(5)),                   # on the CPU
            lambda: S(kv, q, k, k, 8, 2, 1e6, slots=i(5)), lambda: S(kv, q, k, k.half(), 8, 2, 1e6, pos_start=0),
            lambda: S(kv, q[:4], k, k, 8, 2, 1e6), lambda: S(kv, q, k, k[:, :200], 8, 2, 1e6),
            lambda: S(kv, q, k, k, 8, 2, 1e6, positions=i(4), slots=i(5)),
            lambda: S(kv, q, k, k, 8, 2, 1e6, q_norm=torch.ones(64), k_norm=torch.ones(128)),
            lambda: S(kv, q, k, k, 8, 2, 1e6, q_norm=torch.ones(128).half(), k_norm=torch.ones(128))]
    A = PG.paged_attn
    bad += [lambda: A(q, kv, i(3, 4), i(3), i(4), 8, 2), lambda: A(q, kv, i(3, 4), i(3), i(3), 8, 2),
            lambda: A(q[:, :512], kv, i(3, 4), i(3), i(4), 8, 2), lambda: A(q, kv, i(3, 4), i(3).long(), i(4), 8, 2),
            lambda: A(q, kv, i(3, 4), i(3), i(4), 8, 2, out=torch.zeros(4, 1024)),
            lambda: A(q, kv, i(3, 4), i(3), i(4), 8, 2, gate=torch.zeros(5, 1024).half())]
    for f in bad:
        with pytest.raises(YhipError):
            f()


def test_chunks_of_a_line_of_any_length(tmp_path):
    """The line's cuts (csrc/paged_chunks.hpp, compiled for the host): equal chunks, one per workgroup at most, that cover
    it, also where a sum comes near 2^32."""
    csrc = Path(__file__).resolve().parent.parent / "yllm_amd" / "csrc"
    src, exe = tmp_path / "chunks.cpp", tmp_path / "chunks"
    src.write_text('#include "paged_chunks.hpp"\n#include <stdio.h>\n#include <inttypes.h>\nint main() {\n'
                   'uint64_t t; uint32_t w, m;\nwhile (scanf("%" SCNu64 " %" SCNu32 " %" SCNu32, &t, &w, &m) == 3) {\n'
                   'const auto c = yhip::paged_chunks(t, w, m);\nprintf("%u %u\\n", c.units, c.n); } }\n')
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", f"-I{csrc}", str(src), "-o", str(exe)], check=True)
    near = [(1 << b) + k for b in (31, 32, 33) for k in (-(1 << 24), -(1 << 23), -(1 << 23) - 512, -(1 << 22), -513, -511, -1, 0, 1, 511)]
    cases = [(t, w, m) for t in [0, 1, 9, 100, 4096, 10 ** 6, (1 << 38) - 1, *near] for w in (8, 256, 512, 520) for m in (2, 4, 26, 3344)]
    run = subprocess.run([str(exe)], input="".join(f"{t} {w} {m}\n" for t, w, m in cases), capture_output=True, text=True, check=True)
    got = [tuple(map(int, line.split())) for line in run.stdout.splitlines()]
    assert len(got) == len(cases)
    for (t, w, m), (units, n) in zip(cases, got):
        want = max(min(-(-t // w), 0x7fffffff), m)
        assert (units, n) == (want, -(-t // want)), (t, w, m)


# (addresses of attn_args and store_args: the pools take 0x20000 bytes each)
@pytest.mark.parametrize("kw", [
    {"out": _at(0x6000000 + 0x1fff0)}, {"out": _at(0x7000000 - 4096)}, {"out": _at(0x5000000)}, {"out": _at(0x5100000 - 4096)},
    {"out": _at(0x5200000 - 10224)}, {"kp": _at(0x1000000 - 0x1fff0)}, {"vp": _at(0x1000000 + 10224)},
    {"ws": _at(0x1000000 + 10224)}, {"ws": _at(0x2000000 - 16)}, {"ws": _at(0x6000000 + 0x1fff0)}, {"ws": _at(0x7000000)},
    {"ws": _at(0x5000020)}, {"ws": _at(0x5100000)}, {"ws": _at(0x5200000)}, {"gate": _at(0x9000000), "gs": 1024, "ws": _at(0x9000000 + 5 * 4096 - 16)},
])
def test_attn_overlaps(hiplib, kw):
    """What the call writes (the rows, the workspace) is neither what it reads nor each other."""
    kw = dict(w=64, stride=64, max_len=4096, wsb=1 << 30, **{"ws": _at(1 << 40), **kw})
    assert hiplib.yhip_paged_attn(*attn_args(**kw)) == -22 and "overlaps" in _err(hiplib)


@pytest.mark.parametrize("kw", [
    {"qo": _at(0x6000000 + 0x1fff0)}, {"qo": _at(0x7000000 - 4096)}, {"qo": _at(0x5000000)}, {"qo": _at(0x5100000 - 4096)},
    {"qo": _at(0x5200000)}, {"qo": _at(0x5300000 - 10224)}, {"vp": _at(0x6000000 + 0x1fff0)}, {"kp": _at(0x2000000)},
    {"kp": _at(0x3000000 - 0x1fff0)}, {"vp": _at(0x4000000)}, {"vp": _at(0x3000000)}, {"kp": _at(0x5000000)}, {"kp": _at(0x5100000)},
    {"vp": _at(0x5200000)}, {"vp": _at(0x5300000)}, {"kp": _at(0x4000000), "qo": None, "q": None},
])
def test_store_overlaps(hiplib, kw):
    """What the call writes (the queries, the pools) is neither what it reads (q_out may be q) nor each other."""
    assert hiplib.yhip_qk_norm_rope_kv_store(*store_args(**kw)) == -22 and "overlap" in _err(hiplib)


@pytest.mark.parametrize("kw", [{}, {"max_new": 5}, {"d": 64, "os": 512, "qs": 512}])
def test_attn_workspace_of_calls_that_need_one(hiplib, kw):
    kw = dict(w=64, stride=64, max_len=4096, **kw)
    a = dict(zip(("T", "n", "max_new", "max_len", "nh", "nkv", "d"), (5, 3, kw.get("max_new", 2), 4096, 8, 2, kw.get("d", 128))))
    need = hiplib.yhip_paged_attn_workspace(*a.values())
    assert need > 0
    for ws, n in ((None, need), (_at(1 << 40), need - 1), (_at(1 << 40), 0), (_at((1 << 40) + 8), need)):
        assert hiplib.yhip_paged_attn(*attn_args(**kw, ws=ws, wsb=n)) == -28 and "workspace" in _err(hiplib)
