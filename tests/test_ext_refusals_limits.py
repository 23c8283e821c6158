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
