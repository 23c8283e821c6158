"""Log probabilities of tokens on the GPU against 64-bit references: widths from one token to a vocabulary, pitches and
alignments, ties, masks that leave nothing, infinities and NaN in allowed and forbidden places, temperatures."""
import math

import pytest
import torch

import ext_cases as ec
from plow_amd import abi

pytestmark = pytest.mark.gpu
NAMES = ("logprob", "entropy", "lse", "alt_ids", "alt_logprob")


@pytest.fixture(scope="module")
def moe():
    from plow_amd.lib import Moe
    m = Moe(0)
    yield m
    m.close()


def call(moe, x, V, ids, A, scale=1.0, mask=None, offset=0, stream=None, noalloc=False):
    """x [T][pitch] on the CPU; offset: elements by which the logits start off their allocation."""
    T, pitch = x.shape
    flat = torch.zeros(T * pitch + offset, dtype=x.dtype)
    flat[offset:] = x.flatten()
    flat = flat.cuda()
    lg = flat[offset:]
    n = ids.shape[1]
    o = {"logprob": torch.full((T + 1, n), 7.0), "entropy": torch.full((T + 1,), 7.0), "lse": torch.full((T + 1,), 7.0),
         "alt_ids": torch.full((T + 1, A), 7, dtype=torch.int32), "alt_logprob": torch.full((T + 1, A), 7.0)}
    o = {k: v.cuda() for k, v in o.items()}
    tensors = [o["logprob"], lg, ids.cuda(), o["entropy"], o["alt_ids"], o["alt_logprob"], o["lse"], None if mask is None else mask.cuda()]
    inst = abi.inst(abi.OP_X_LOGPROB, t=[0 if n else None, 1, 2 if n else None, 3, 4 if A else None, 5 if A else None, 6,
                                         None if mask is None else 7],
                    i=[T, V, n, A, pitch, abi.LOGPROB_F32 if x.dtype == torch.float32 else 0, 0 if mask is None else mask.shape[1]],
                    f=[scale])
    torch.cuda.synchronize()
    if noalloc:
        import ctypes as C
        err = C.create_string_buffer(256)
        assert moe.lib.plow_moe_exec_noalloc(C.byref(inst), ec.table_of(tensors), None, err, 256) == 0, err.value
    else:
        moe.exec(inst, ec.table_of(tensors), stream)
    torch.cuda.synchronize()
    got = {k: v.cpu() for k, v in o.items()}
    for k, v in got.items():
        assert v[T:].numel() == 0 or (v[T:] == 7).all(), f"{k}: written past the last row"
    return {k: v[:T] for k, v in got.items()}


def check(got, want, scale=1.0, top=50.0, V=1):
    """Bound of an f32 log probability: d = c (x - m) rounds twice (2 * 2^-24 of its size); Z is a sum of positive terms,
    each exp off by its argument's rounding and a few units, added in chains of V / 64 at most before trees: its
    logarithm is off by (V / 64 + 16) * 2^-24 at most. 4 * covers the entropy, whose terms are weighted by d."""
    assert torch.equal(got["alt_ids"], want["alt_ids"])
    for k in ("logprob", "entropy", "lse", "alt_logprob"):
        a, b = got[k].double(), want[k]
        assert torch.equal(torch.isnan(a), torch.isnan(b)), k
        inf = torch.isinf(b)
        assert torch.equal(a[inf], b[inf]), k
        ok = ~torch.isnan(b) & ~inf
        assert not torch.isinf(a[ok]).any(), k
        tol = ec.EPS_F32 * (4 * (V / 64 + 16) + 4 * b[ok].abs() + 4 * top * scale)
        d = (a[ok] - b[ok]).abs()
        assert (d <= tol).all(), (k, d.max().item(), tol.min().item())


def logits(T, pitch, V, dtype, seed, peaked=True):
    g = ec.gen(seed)
    x = torch.randn(T, pitch, generator=g) * 2.5
    if peaked:
        x[:, : max(1, V // 300)] += torch.rand(T, 1, generator=g) * 9
    x[:, V:] = 1000.0 if pitch > V else 0.0     # what lies between the rows must not count
    return x.to(dtype)


SHAPES = [(1, 1, 1), (1, 2, 2), (3, 5, 8), (1, 63, 3), (2, 64, 5), (5, 65, 20), (4, 255, 64), (3, 1000, 7), (1, 4096, 20), (2, 4097, 64),
          (1, 50257, 20), (17, 32000, 5), (300, 777, 4), (1, 151937, 64), (3, 130001, 0), (700, 2049, 1)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,V,A", SHAPES)
def test_logprob(moe, T, V, A, dtype):
    print(f"[case] logprob T={T} V={V} A={A} {dtype}", flush=True)
    for extra, offset, n, scale in ((0, 0, 1, 1.0), (3, 1, 3, 0.7)):
        x = logits(T, V + extra, V, dtype, V + T)
        ids = torch.randint(0, V, (T, n), generator=ec.gen(1), dtype=torch.int32)
        check(call(moe, x, V, ids, A, scale, offset=offset), ec.logprob64(x, V, ids, A, scale), scale, V=V)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [33, 1000, 32000, 100003])
def test_ties_go_to_the_lowest_id(moe, V, dtype):
    g = ec.gen(V)
    T, A = 5, 40
    x = torch.randint(-3, 4, (T, V), generator=g).float()
    x[1] = 2.0                                    # all equal
    x[2] = torch.where(torch.rand(V, generator=g) < 0.5, 0.0, -0.0)   # both zeros are one value
    x[3] = -5.0
    x[3, V // 2:] = torch.arange(V - V // 2).float() / 64             # rising
    x[4] = -torch.arange(V).float() / 64                              # falling
    x = x.to(dtype)
    ids = torch.zeros(T, 1, dtype=torch.int32)
    check(call(moe, x, V, ids, A), ec.logprob64(x, V, ids, A), top=2000.0, V=V)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [31, 64, 2000, 70001])
def test_masks(moe, V, dtype):
    """A bit mask, among others one that leaves nothing and one that leaves the last token; infinities, NaN and the
    type's lowest value where the mask forbids."""
    T, A, words = 7, 10, (V + 31) // 32 + 1
    g = ec.gen(V)
    x = logits(T, V, V, dtype, V)
    mask = torch.randint(-2 ** 31, 2 ** 31, (T, words), generator=g, dtype=torch.int64).to(torch.int32)
    mask[0] = 0
    mask[1] = 0
    mask[1, (V - 1) // 32] = -2 ** 31 if (V - 1) % 32 == 31 else 1 << ((V - 1) % 32)
    mask[2] = -1
    mask[3, 0] = ~(1 << 3)
    x[3, 3] = math.nan
    mask[4, 0] = ~(1 << 5)
    x[4, 5] = math.inf
    mask[5, 0] = ~(1 << 6)
    x[5, 6] = torch.finfo(dtype).min
    ids = torch.stack([torch.full((T,), V - 1), torch.arange(T)], 1).to(torch.int32)
    check(call(moe, x, V, ids, A, 1.3, mask), ec.logprob64(x, V, ids, A, 1.3, mask), 1.3, V=V)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [9, 500, 40000])
def test_minus_infinity_nan_and_extremes(moe, V, dtype):
    T, A = 8, 6
    x = logits(T, V, V, dtype, V + 1)
    x[0] = -math.inf                              # nothing left
    x[1, : V - 2] = -math.inf                     # two tokens left
    x[2, 4] = math.nan
    x[3, 1] = math.inf
    x[4, 0], x[4, 3] = math.inf, math.nan
    x[5] = torch.finfo(dtype).min                 # uniform at the lowest value
    x[6, :] = torch.finfo(dtype).min
    x[6, V // 2] = 3.0
    x[7, 2] = -math.nan
    ids = torch.tensor([[0, V - 1]] * T, dtype=torch.int32)
    ids[6, 0] = V // 2
    ids[6, 1] = V // 2
    got, want = call(moe, x, V, ids, A), ec.logprob64(x, V, ids, A)
    # beside a finite maximum the lowest value has probability 0 and a log probability of its own size, or -inf
    for r in (6,):
        far = got["alt_logprob"][r, 1:]
        assert (far < -1e38).all()
        got["alt_logprob"][r, 1:] = want["alt_logprob"][r, 1:].float() * 0
        want["alt_logprob"][r, 1:] = 0
    got["lse"][5], want["lse"][5] = got["lse"][5] / torch.finfo(dtype).max, want["lse"][5] / torch.finfo(dtype).max
    check(got, want, V=V)


def test_given_tokens(moe):
    """A token id that asks for nothing, ids past the vocabulary, the same id twice, many ids of one row."""
    T, V = 3, 1000
    x = logits(T, V, V, torch.float32, 3)
    ids = torch.randint(0, V, (T, 600), generator=ec.gen(2), dtype=torch.int32)
    ids[:, 0], ids[:, 1], ids[:, 2], ids[:, 3], ids[:, 4] = -1, V, 2 ** 31 - 1, 17, 17
    ids[1, 5] = -2
    check(call(moe, x, V, ids, 0), ec.logprob64(x, V, ids, 0), V=V)


def test_only_some_outputs(moe):
    T, V, A = 4, 5000, 8
    x = logits(T, V, V, torch.float32, 4)
    want = ec.logprob64(x, V, torch.zeros(T, 0, dtype=torch.int32), A)
    xd, ent = x.cuda(), torch.zeros(T, device="cuda")
    moe.exec(abi.inst(abi.OP_X_LOGPROB, t=[None, 0, None, 1], i=[T, V, 0, 0, 0, 1]), ec.table_of([xd, ent]))
    ids = torch.zeros(T, A, dtype=torch.int32, device="cuda")
    moe.exec(abi.inst(abi.OP_X_LOGPROB, t=[None, 0, None, None, 1], i=[T, V, 0, A, 0, 1]), ec.table_of([xd, ids]))
    alt = torch.zeros(T, A, device="cuda")
    moe.exec(abi.inst(abi.OP_X_LOGPROB, t=[None, 0, None, None, None, 1], i=[T, V, 0, A, 0, 1]), ec.table_of([xd, alt]))
    torch.cuda.synchronize()
    assert (ent.cpu().double() - want["entropy"]).abs().max() < 1e-5
    assert torch.equal(ids.cpu(), want["alt_ids"])
    assert (alt.cpu().double() - want["alt_logprob"]).abs().max() < 1e-5


def test_probability_near_one(moe):
    """A token that holds almost everything: its log probability and the entropy keep their digits."""
    V = 30000
    x = torch.zeros(2, V)
    x[0, 77], x[1, V - 1] = 40.0, 25.0
    ids = torch.tensor([[77], [V - 1]], dtype=torch.int32)
    got, want = call(moe, x, V, ids, 3), ec.logprob64(x, V, ids, 3)
    assert torch.equal(got["alt_ids"], want["alt_ids"])
    # -ln Z with Z = 1 + eps: an f32 Z resolves 2^-24
    assert (got["logprob"].double() - want["logprob"]).abs().max() <= 4 * ec.EPS_F32
    assert (got["entropy"].double() - want["entropy"]).abs().max() <= 64 * ec.EPS_F32


def test_noalloc_and_other_stream(moe):
    for T, V in ((1, 100003), (9, 4000)):
        x = logits(T, V, V, torch.bfloat16, 8)
        ids = torch.randint(0, V, (T, 2), generator=ec.gen(1), dtype=torch.int32)
        want = ec.logprob64(x, V, ids, 20)
        check(call(moe, x, V, ids, 20, noalloc=True), want, V=V)
        s = torch.cuda.Stream()
        check(call(moe, x, V, ids, 20, stream=s.cuda_stream), want, V=V)
