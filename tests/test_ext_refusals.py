"""What the int4 and log-probability ops refuse: every check of a descriptor runs on the CPU, over the dispatch layer
compiled for the host, and again on the built library on the GPU, where nothing of a refused call is launched."""
import ctypes as C
import os
import subprocess

import pytest

from plow_amd import abi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NH = 12
INVAL, UNSUP, OK = abi.E_INVAL, abi.E_UNSUPPORTED, 0


def product(t=(0, 1, 2, 3), i=(4, 64, 128, 32), **kw):
    return abi.inst(abi.OP_X_GEMM_W4, t=list(t), i=list(i), **kw)


def glu(t=(0, 1, 2, 3, None, 5, 6), i=(4, 64, 128, 32, 0, 1), **kw):
    return abi.inst(abi.OP_X_GEMM_GLU_W4, t=list(t), i=list(i), **kw)


def slots(op, t=(0, 1, 2, 3, 4), i=(8, 64, 128, 4, 2, 1, 16, 32)):
    return abi.inst(op, t=list(t), i=list(i))


def grouped(op, t, i):
    return abi.inst(op, t=list(t), i=list(i), slots=8)


def logprob(t=(0, 1, 2, 3, 4, 5, 6), i=(2, 100, 1, 5), f=()):
    return abi.inst(abi.OP_X_LOGPROB, t=list(t), i=list(i), f=f)


G48, D49, G85, D86 = 48, 49, 85, 86
T85, I85 = (0, 1, 2, 3, 4, 5), (64, 128, 4, 16, 0, 1, 32, 0)
T86, I86 = (0, 1, 2, 3, 4, None, 6, 7), (128, 64, 4, 16, 0, 0, 32, 0)


def repl(seq, at, v):
    s = list(seq)
    s += [0] * (at + 1 - len(s))
    s[at] = v
    return tuple(s)


# (name, descriptor, expected code, handle shifted off its alignment: (slot, bytes) or None)
CASES = [
    ("product", product(), OK, None),
    ("product f32", product(i=(4, 64, 128, 64 | abi.W4_SCALE_F16, 136, 70, 1)), OK, None),
    ("product zero points", product(t=(0, 1, 2, 3, 4)), OK, None),
    ("product no out", product(t=(None, 1, 2, 3)), INVAL, None),
    ("product no x", product(t=(0, None, 2, 3)), INVAL, None),
    ("product no W", product(t=(0, 1, None, 3)), INVAL, None),
    ("product no S", product(t=(0, 1, 2, None)), INVAL, None),
    ("product extra operand", product(t=(0, 1, 2, 3, 4, 5)), INVAL, None),
    ("product M 0", product(i=(0, 64, 128, 32)), INVAL, None),
    ("product N 0", product(i=(4, 0, 128, 32)), INVAL, None),
    ("product K 0", product(i=(4, 64, 0, 32)), INVAL, None),
    ("product K not groups", product(i=(4, 64, 96, 64)), INVAL, None),
    ("product group 16", product(i=(4, 64, 128, 16)), INVAL, None),
    ("product group 0", product(i=(4, 64, 128, 0)), INVAL, None),
    ("product group flags", product(i=(4, 64, 128, 32 | 0x20000)), INVAL, None),
    ("product x pitch short", product(i=(4, 64, 128, 32, 120)), INVAL, None),
    ("product x pitch odd", product(i=(4, 64, 128, 32, 132)), INVAL, None),
    ("product out pitch short", product(i=(4, 64, 128, 32, 0, 63)), INVAL, None),
    ("product out type", product(i=(4, 64, 128, 32, 0, 0, 2)), INVAL, None),
    ("product x misaligned", product(), INVAL, (1, 2)),
    ("product W misaligned", product(), INVAL, (2, 8)),
    ("product S misaligned", product(), INVAL, (3, 1)),
    ("product S at an odd element", product(), OK, (3, 2)),
    ("product out misaligned", product(i=(4, 64, 128, 32, 0, 0, 1)), INVAL, (0, 2)),
    ("product N huge", product(i=(4, (1 << 28) + 1, 128, 32)), INVAL, None),
    ("product M huge", product(i=(65535 * 128 + 1, 64, 128, 32)), INVAL, None),
    ("product K huge", product(i=(4, 64, (1 << 24) + 128, 128)), INVAL, None),
    ("glu", glu(), OK, None),
    ("glu zero points", glu(t=(0, 1, 2, 3, 4, 5, 6, 7)), OK, None),
    ("glu one zero point", glu(t=(0, 1, 2, 3, 4, 5, 6)), INVAL, None),
    ("glu no up", glu(t=(0, 1, 2, 3, None, None, 6)), INVAL, None),
    ("glu no up scale", glu(t=(0, 1, 2, 3, None, 5)), INVAL, None),
    ("glu activation", glu(i=(4, 64, 128, 32, 0, 5)), INVAL, None),
    ("glu out pitch", glu(i=(4, 64, 128, 32, 0, 1, 60)), INVAL, None),
    ("glu up misaligned", glu(), INVAL, (5, 8)),
    ("48", slots(G48), OK, None),
    ("48 ztab", slots(G48, t=(0, 1, 2, 3, 4, 5)), OK, None),
    ("48 no table", slots(G48, t=(0, 1, None, 3, 4)), INVAL, None),
    ("48 no scales", slots(G48, t=(0, 1, 2, 3)), INVAL, None),
    ("48 no slots", slots(G48, i=(0, 64, 128, 4, 2, 1, 16, 32)), INVAL, None),
    ("48 part of a row", slots(G48, i=(8, 64, 128, 4, 3, 1, 16, 32)), INVAL, None),
    ("48 one shared row", slots(G48, i=(7, 64, 128, 4, 0, 1, 16, 32)), OK, None),
    ("48 no experts", slots(G48, i=(8, 64, 128, 0, 2, 1, 16, 32)), INVAL, None),
    ("48 too many experts", slots(G48, i=(8, 64, 128, 1057, 2, 1, 16, 32)), INVAL, None),
    ("48 too many slots", slots(G48, i=((1 << 20) + 1, 64, 128, 4, 2, 1, 16, 32)), INVAL, None),
    ("48 group", slots(G48, i=(8, 64, 128, 4, 2, 1, 16, 48)), INVAL, None),
    ("48 K", slots(G48, i=(8, 64, 100, 4, 2, 1, 16, 32)), INVAL, None),
    ("48 activation", slots(G48, i=(8, 64, 128, 4, 2, 7, 16, 32)), INVAL, None),
    ("48 x misaligned", slots(G48), INVAL, (1, 8)),
    ("48 another encoding", slots(G48, i=(8, 128, 128, 4, 2, 1, 17, 32)), INVAL, None),
    ("49", slots(D49, i=(8, 128, 64, 4, 0, 0, 16, 32)), OK, None),
    ("49 no part", slots(D49, t=(None, 1, 2, 3, 4), i=(8, 128, 64, 4, 0, 0, 16, 32)), INVAL, None),
    ("85", grouped(G85, T85, I85), OK, None),
    ("85 ztab", grouped(G85, (0, 1, 2, 3, 4, 5, 6), I85), OK, None),
    ("85 arm", grouped(G85, T85, repl(I85, 7, 8)), UNSUP, None),
    ("85 no row_token", grouped(G85, repl(T85, 5, None), I85), INVAL, None),
    ("85 no stab", grouped(G85, repl(T85, 3, None), I85), INVAL, None),
    ("85 no experts", grouped(G85, T85, repl(I85, 2, 0)), INVAL, None),
    ("85 too many experts", grouped(G85, T85, repl(I85, 2, 65536)), INVAL, None),
    ("85 group", grouped(G85, T85, repl(I85, 6, 33)), INVAL, None),
    ("86", grouped(D86, T86, I86), OK, None),
    ("86 fused combine", grouped(D86, T86, repl(I86, 5, 2)), INVAL, None),
    ("86 no gate", grouped(D86, repl(T86, 7, None), I86), INVAL, None),
    ("86 arm", grouped(D86, T86, repl(I86, 7, 2)), UNSUP, None),
    ("logprob", logprob(), OK, None),
    ("logprob scale", logprob(f=(0.5,)), OK, None),
    ("logprob mask", logprob(t=(0, 1, 2, 3, 4, 5, 6, 7)), OK, None),
    ("logprob no logits", logprob(t=(0, None, 2, 3)), INVAL, None),
    ("logprob T 0", logprob(i=(0, 100, 1, 5)), INVAL, None),
    ("logprob T huge", logprob(i=(1 << 24, 100, 1, 5)), INVAL, None),
    ("logprob V 0", logprob(i=(2, 0, 1, 5)), INVAL, None),
    ("logprob V huge", logprob(i=(2, 1 << 31, 1, 5)), INVAL, None),
    ("logprob tokens without ids", logprob(t=(0, 1, None, 3)), INVAL, None),
    ("logprob tokens without out", logprob(t=(None, 1, 2, 3)), INVAL, None),
    ("logprob alternatives", logprob(i=(2, 100, 1, 65)), INVAL, None),
    ("logprob alternatives without out", logprob(t=(0, 1, 2, 3)), INVAL, None),
    ("logprob nothing asked", logprob(t=(0, 1, 2), i=(2, 100, 0, 0)), INVAL, None),
    ("logprob pitch", logprob(i=(2, 100, 1, 5, 99)), INVAL, None),
    ("logprob flags", logprob(i=(2, 100, 1, 5, 0, 2)), INVAL, None),
    ("logprob i7", logprob(i=(2, 100, 1, 5, 0, 0, 0, 1)), INVAL, None),
    ("logprob mask pitch", logprob(t=(0, 1, 2, 3, 4, 5, 6, 7), i=(2, 100, 1, 5, 0, 0, 3)), INVAL, None),
    ("logprob scale negative", logprob(f=(-1.0,)), INVAL, None),
    ("logprob scale infinite", logprob(f=(float("inf"),)), INVAL, None),
    ("logprob scale NaN", logprob(f=(float("nan"),)), INVAL, None),
    ("logprob logits misaligned", logprob(i=(2, 100, 1, 5, 0, 1)), INVAL, (1, 2)),
    ("logprob ids misaligned", logprob(), INVAL, (2, 2)),
]


def table(base, shift):
    t = (C.c_void_p * NH)()
    for n in range(NH):
        t[n] = base + n * (1 << 16)
    if shift:
        t[shift[0]] += shift[1]
    return t


@pytest.fixture(scope="module")
def host_lib(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("host") / "api_host.so")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-w",
                           "-Wl,-z,lazy", "-x", "c++", os.path.join(ROOT, "plow_amd", "csrc", "api.hip"),
                           os.path.join(ROOT, "tests", "api_host_stub.cpp"), "-o", out])
    lib = C.CDLL(out, mode=os.RTLD_LAZY)
    lib.plow_moe_create.argtypes = [C.POINTER(C.c_void_p), C.c_int]
    lib.plow_moe_destroy.argtypes = [C.c_void_p]
    lib.plow_moe_check.argtypes = [C.c_void_p, C.POINTER(abi.PlowDevInst), C.POINTER(C.c_void_p)]
    lib.plow_moe_last_error.argtypes, lib.plow_moe_last_error.restype = [C.c_void_p], C.c_char_p
    for name in ("plow_moe_pf", "plow_moe_dec"):
        getattr(lib, name).argtypes = [C.c_void_p, C.POINTER(abi.PlowDevInst), C.c_uint32, C.POINTER(C.c_void_p), C.c_uint32, C.c_void_p]
    return lib


@pytest.fixture(scope="module")
def host_ctx(host_lib):
    h = C.c_void_p()
    assert host_lib.plow_moe_create(C.byref(h), 0) == 0
    yield h
    host_lib.plow_moe_destroy(h)


@pytest.mark.parametrize("case", CASES, ids=lambda c: c[0])
def test_checks_on_the_host(host_lib, host_ctx, case):
    name, inst, code, shift = case
    got = host_lib.plow_moe_check(host_ctx, C.byref(inst), table(1 << 32, shift))
    text = host_lib.plow_moe_last_error(host_ctx).decode()
    assert got == code, (name, got, text)
    assert bool(text) == bool(code), text


def test_segments_on_the_host(host_lib, host_ctx):
    """A segment whose GLU and DOWN disagree over the zero points or the encoding is refused before any launch."""
    base = table(1 << 32, None)
    bad = [[slots(G48, t=(0, 1, 2, 3, 4, 5)), slots(D49, t=(6, 0, 2, 3, 4), i=(8, 128, 64, 4, 0, 0, 16, 32))],
           [slots(G48), slots(D49, t=(6, 0, 2, 3, 4), i=(8, 128, 64, 4, 0, 0, 2, 32))],
           [grouped(G85, (0, 1, 2, 3, 4, 5, 8), I85), grouped(D86, (6, 0, 2, 3, 4, None, 9, 7), I86)]]
    for pair in bad:
        arr = abi.inst_array(pair)
        assert host_lib.plow_moe_dec(host_ctx, arr, 2, base, 4, None) == INVAL
        assert b"segment" in host_lib.plow_moe_last_error(host_ctx)


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    """The built library gives the same answers, and a refused op of a run keeps the whole run from starting."""
    import torch

    from plow_amd.lib import Moe, MoeError
    moe = Moe(0)
    buf = torch.full((NH << 16,), 5, dtype=torch.uint8, device="cuda")
    for name, inst, code, shift in CASES:
        assert moe.check(inst, table(buf.data_ptr(), shift)) == code, (name, moe.last_error())
        if code:
            with pytest.raises(MoeError):
                moe.exec(inst, table(buf.data_ptr(), shift))
            with pytest.raises(MoeError):
                moe.exec_many([product(), inst], table(buf.data_ptr(), shift))
    torch.cuda.synchronize()
    assert (buf == 5).all(), "a refused run wrote something"
    moe.close()
