"""Limits of the log-probability op and segments of mixed encodings: refused by the descriptor checks, on the CPU over the
dispatch layer compiled for the host."""
import ctypes as C

import pytest

from plow_amd import abi
from test_ext_refusals import D49, G48, INVAL, OK, host_ctx, host_lib, logprob, slots, table  # noqa: F401

# (name, descriptor, expected code)
CASES = [
    # a wave steps through a row's given tokens 64 at a time in 32 bits
    ("given tokens at the limit", logprob(i=(2, 100, 0x7FFFFFFF, 5)), OK),
    ("given tokens past the limit", logprob(i=(2, 100, 0x80000000, 5)), INVAL),
    ("given tokens that wrap", logprob(i=(2, 100, 0xFFFFFFFF, 5)), INVAL),
    # a factor so small that logits further apart than the largest f32 would count
    ("smallest scale", logprob(f=(1e-30,)), OK),
    ("largest scale", logprob(f=(1e30,)), OK),
    ("scale below", logprob(f=(9e-31,)), INVAL),
    ("scale subnormal", logprob(f=(1e-42,)), INVAL),
    ("scale above", logprob(f=(1.1e30,)), INVAL),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: c[0])
def test_limits_on_the_host(host_lib, host_ctx, case):  # noqa: F811
    name, inst, code = case
    got = host_lib.plow_moe_check(host_ctx, C.byref(inst), table(1 << 32, None))
    assert got == code, (name, got, host_lib.plow_moe_last_error(host_ctx).decode())


@pytest.mark.parametrize("glu_enc,down_enc", [(2, 16), (1, 16), (0, 16), (16, 2), (16, 1), (16, 0)])
def test_segments_of_mixed_encodings_on_the_host(host_lib, host_ctx, glu_enc, down_enc):  # noqa: F811
    """GLU and DOWN of one weight table are both int4 or neither: an int4 DOWN behind another GLU is refused like the
    reverse. (An op that no library serves ends the run, so that a pair let through is not launched.)"""
    def enc(at):
        return 32 if at == 16 else 0
    run = [slots(G48, i=(8, 128, 128, 4, 2, 1, glu_enc, enc(glu_enc))),
           slots(D49, t=(6, 0, 2, 3, 4), i=(8, 128, 128, 4, 0, 0, down_enc, enc(down_enc))), abi.inst(0x7FFF, t=[], i=[])]
    assert host_lib.plow_moe_dec(host_ctx, abi.inst_array(run), 3, table(1 << 32, None), 4, None) == INVAL
    assert b"segment" in host_lib.plow_moe_last_error(host_ctx)
