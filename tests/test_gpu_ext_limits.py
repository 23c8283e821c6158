"""Int4 products, int4 experts and log probabilities where a call's sizes or addresses are unusual: tensors past 4 GiB,
very many rows, very long rows, scales and zero points at odd addresses, one expert for every slot, a token that lists
an expert twice, extreme temperatures, the entry point without a context, graphs of two contexts replayed side by side."""
import ctypes as C

import pytest
import torch

import ext_cases as ec
from ext_cases import EPS_F32, HALF_BF16
from plow_amd import abi

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def moe():
    from plow_amd.lib import Moe
    m = Moe(0)
    yield m
    m.close()


def gen(seed):
    return ec.gen(seed, "cuda")


def weights(g, N, K, G, zero=True):
    W = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8, device="cuda")
    S = ((torch.rand(N, K // G, generator=g, device="cuda") + 0.5) * 0.006).to(torch.bfloat16)
    return W, S, torch.randint(0, 16, (N, K // G), generator=g, dtype=torch.uint8, device="cuda") if zero else None


def close(got, x, W, S, Z):
    want = x.double() @ ec.dequant64(W, S, Z).T.contiguous()
    err = (got.double() - want).abs()
    bound = ec.abs_bound(x, W, S, Z)
    assert (err <= bound + EPS_F32 * want.abs()).all(), (err / bound).max()
    assert err.norm() <= 1e-6 * want.norm(), err.norm() / want.norm()


@pytest.fixture(scope="module")
def large():
    """Weights of 4.5 GB."""
    yield weights(gen(1), 1100003, 8192, 128)
    torch.cuda.empty_cache()


@pytest.mark.parametrize("M", [1, 8, 24, 40, 130])
def test_weights_past_32_bits(moe, large, M):
    W, S, Z = large
    N, K = W.shape[0], 2 * W.shape[1]
    assert W.numel() > 1 << 32
    print(f"[case] large M={M}", flush=True)
    x = torch.randn(M, K, generator=gen(M), device="cuda").to(torch.bfloat16)
    o = torch.full((M, N), 7.0, device="cuda")
    moe.exec(abi.inst(abi.OP_X_GEMM_W4, t=[0, 1, 2, 3, 4], i=[M, N, K, 128, 0, 0, 1]), ec.table_of([o, x, W, S, Z]))
    for at in (slice(0, 70), slice(1 << 20, (1 << 20) + 300), slice(N - 300, N)):
        close(o[:, at], x, W[at], S[at], Z[at])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logits_past_32_bits(moe, dtype):
    T, V = (9001, 120001) if dtype == torch.float32 else (18001, 120001)
    print(f"[case] logits {T} x {V} {dtype}", flush=True)
    x = torch.zeros(T, V, dtype=dtype, device="cuda")
    rows = [0, 5, T // 2, T - 2, T - 1]
    for r in rows:
        x[r] = (torch.randn(V, generator=gen(r), device="cuda") * 3).to(dtype)
    ids = torch.randint(0, V, (T, 1), generator=gen(3), device="cuda", dtype=torch.int32)
    lp, ent, lse = (torch.full((T, 1), 7.0, device="cuda") for _ in range(3))
    aid, alp = torch.zeros(T, 5, dtype=torch.int32, device="cuda"), torch.zeros(T, 5, device="cuda")
    moe.exec(abi.inst(abi.OP_X_LOGPROB, t=[0, 1, 2, 3, 4, 5, 6], i=[T, V, 1, 5, 0, abi.LOGPROB_F32 if dtype == torch.float32 else 0]),
             ec.table_of([lp, x, ids, ent, aid, alp, lse]))
    torch.cuda.synchronize()
    want = ec.logprob64(x[rows].cpu(), V, ids[rows].cpu(), 5)
    assert torch.equal(aid[rows].cpu(), want["alt_ids"])
    # Z is off by (V / 64 + 16) roundings at most, d by two of its size (below 30)
    tol = EPS_F32 * (4 * (V / 64 + 16) + 4 * 30)
    for got, k in ((lp, "logprob"), (ent[:, 0], "entropy"), (lse[:, 0], "lse"), (alp, "alt_logprob")):
        assert (got[rows].cpu().double() - want[k]).abs().max() <= tol, k
    flat = [r for r in (1, 6, T - 3) if r not in rows]
    assert (lp[flat].cpu().double() + torch.log(torch.tensor(float(V), dtype=torch.float64))).abs().max() <= tol
    assert torch.equal(aid[flat].cpu(), torch.arange(5, dtype=torch.int32).expand(len(flat), 5))


def test_very_many_rows(moe):
    """More rows than a grid has tiles of 16 for, and of a tensor of fewer than 64 groups."""
    M = 1100003
    for N, K, G in ((64, 64, 32), (31, 32, 32)):
        print(f"[case] rows {M} x {N} x {K}", flush=True)
        w = weights(gen(N), N, K, G)
        x = torch.randn(M, K, generator=gen(5), device="cuda").to(torch.bfloat16)
        o = torch.full((M + 1, N), 7.0, device="cuda")
        moe.exec(abi.inst(abi.OP_X_GEMM_W4, t=[0, 1, 2, 3, 4], i=[M, N, K, G, 0, 0, 1]), ec.table_of([o, x, *w]))
        close(o[:M], x, *w)
        assert (o[M] == 7).all()


@pytest.mark.parametrize("M", [1, 2, 40])
def test_very_long_rows(moe, M):
    """The longest rows: 2^24 columns."""
    N, K, G = 5, 1 << 24, 128
    print(f"[case] long M={M}", flush=True)
    w = weights(gen(7), N, K, G)
    x = (torch.randn(M, K, generator=gen(8), device="cuda")).to(torch.bfloat16)
    o = torch.zeros(M, N, device="cuda")
    moe.exec(abi.inst(abi.OP_X_GEMM_W4, t=[0, 1, 2, 3, 4], i=[M, N, K, G, 0, 0, 1]), ec.table_of([o, x, *w]))
    want, norm = torch.zeros(M, N, dtype=torch.float64, device="cuda"), torch.zeros(M, N, dtype=torch.float64, device="cuda")
    for k in range(0, K, 1 << 20):
        d = ec.dequant64(w[0][:, k // 2:(k + (1 << 20)) // 2], *(t[:, k // G:(k + (1 << 20)) // G] for t in w[1:]))
        xs = x[:, k:k + (1 << 20)].double()
        want += xs @ d.T.contiguous()
        norm += xs.square() @ d.square().T.contiguous()
    # terms of random signs: a partial sum is about sqrt(norm) in size at most, and each of its K / G additions, of sums
    # of 128 products inside 62 / 7.5 times the terms' size, rounds by half a step of it (in the worst order all of them
    # one after the other; rounding errors of random signs add up to the square root of their number)
    tol = 8 * 62 / 7.5 * EPS_F32 * (K / G) ** 0.5 * norm.sqrt()
    assert ((o.double() - want).abs() <= tol).all(), ((o.double() - want).abs() / tol).max()


@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("M,N,K", [(1, 130, 2048), (9, 130, 2176), (24, 65500, 512), (70, 260, 1152), (200, 2050, 384), (96, 7168, 256)])
def test_scales_at_odd_addresses(moe, M, N, K, G):
    """Scales one element and zero points one byte off any larger alignment."""
    print(f"[case] odd addresses M={M} N={N} K={K} G={G}", flush=True)
    W, S, Z = weights(gen(M), N, K, G)
    s1, z1 = torch.zeros(S.numel() + 1, dtype=S.dtype, device="cuda"), torch.zeros(Z.numel() + 1, dtype=Z.dtype, device="cuda")
    s1[1:], z1[1:] = S.flatten(), Z.flatten()
    x = torch.randn(M, K, generator=gen(2), device="cuda").to(torch.bfloat16)
    o = torch.zeros(M, N, device="cuda")
    moe.exec(abi.inst(abi.OP_X_GEMM_W4, t=[0, 1, 2, 3, 4], i=[M, N, K, G, 0, 0, 1]), ec.table_of([o, x, W, s1[1:], z1[1:]]))
    close(o, x, W, S, Z)


def experts(E, H, I, G, seed):
    g = gen(seed)
    sets = [[weights(g, n, k, G) for _ in range(E)] for n, k in ((I, H), (I, H), (H, I))]
    tabs = [torch.tensor([[sets[m][e][c].data_ptr() for m in range(3)] for e in range(E)], dtype=torch.int64).cuda() for c in range(3)]
    return sets, tabs


def routed(E, H, I, G, eid, run, seed=1):
    """GLU and DOWN of slots with the experts eid [T][k] through run(insts, tensors); every slot checked."""
    T, k = eid.shape
    sets, tabs = experts(E, H, I, G, seed)
    gate = torch.rand(T, k, generator=gen(4), device="cuda") + 0.1
    tab = torch.stack([eid.cuda(), gate.view(torch.int32)], 2).reshape(T * k, 2).contiguous()
    x = torch.randn(T, H, generator=gen(5), device="cuda").to(torch.bfloat16)
    fu = torch.full((T * k + 1, I), 3.0, dtype=torch.bfloat16, device="cuda")
    part = torch.full((T * k + 1, H), 3.0, device="cuda")
    run([abi.inst(abi.OP_MOE_GROUP_GLU_FP8_BLK, t=[0, 1, 2, 3, 4, 5], i=[T * k, I, H, E, k, abi.ACT_SILU, abi.ENC_INT4G, G]),
         abi.inst(abi.OP_MOE_GROUP_DOWN_FP8_BLK, t=[6, 0, 2, 3, 4, 5], i=[T * k, H, I, E, 0, 0, abi.ENC_INT4G, G])], [fu, x, tab, *tabs, part])
    torch.cuda.synchronize()
    assert (fu[-1] == 3).all() and (part[-1] == 3).all()
    for e in eid.unique().tolist():
        s = (eid.view(-1) == e).nonzero()[:, 0].cuda()
        d = [ec.dequant64(*m[e]).T.contiguous() for m in sets]
        xr = x[s // k].double()
        want = ec.act64(xr @ d[0], xr @ d[1], abi.ACT_SILU)
        assert (fu[s].double() - want).norm() <= 0.65 * HALF_BF16 * want.norm(), e
        want = fu[s].double() @ d[2] * gate.view(-1)[s].double()[:, None]
        assert (part[s].double() - want).norm() <= 1e-6 * want.norm(), e


@pytest.mark.parametrize("T,E,k", [(4, 6, 3), (40, 6, 3), (300, 3, 2), (900, 40, 1)])
def test_one_expert_for_every_slot_and_twice_in_a_token(moe, T, E, k):
    print(f"[case] one expert T={T} E={E} k={k}", flush=True)
    run = lambda insts, t: moe.exec_many(insts, ec.table_of(t))
    routed(E, 256, 192, 64, torch.full((T, k), E - 1, dtype=torch.int32), run)
    eid = torch.randint(0, E, (T, k), generator=ec.gen(T), dtype=torch.int32)
    eid[:, -1] = eid[:, 0]
    routed(E, 384, 128, 32, eid, run)


@pytest.mark.parametrize("stated", [150, 600, 1 << 20, 0xFFFFFFFF])
def test_gathered_rows_whatever_count_is_stated(moe, stated):
    """The row count that a grouped op may state chooses a form and a grid; a wrong one costs time, not rows."""
    print(f"[case] gathered, stated {stated}", flush=True)
    T, E, k, H, I, G = 200, 5, 3, 256, 192, 64
    sets, tabs = experts(E, H, I, G, 3)
    eid = torch.randint(0, E, (T, k), generator=ec.gen(1), dtype=torch.int32)
    eid[: T // 2, 0] = 3
    gate = torch.rand(T, k, generator=ec.gen(2)) + 0.1
    tab = torch.stack([eid, gate.view(torch.int32)], 2).reshape(T * k, 2).contiguous().cuda()
    x = torch.randn(T, H, generator=gen(5), device="cuda").to(torch.bfloat16)
    R = abi.max_rows(T, k, E)
    fu, part = torch.zeros(R, I, dtype=torch.bfloat16, device="cuda"), torch.full((T * k + 1, H), 3.0, device="cuda")
    maps = [torch.zeros(n, dtype=torch.int32, device="cuda") for n in (3 * E + 1, R, R, R)]
    tensors = ec.table_of([fu, x, tab, *tabs, part, *maps])
    for d in (abi.inst(abi.OP_MOE_ALIGN_PF, t=[7, 2, 8, 9, 10], i=[T, E, k]),
              abi.inst(abi.OP_MOE_GROUP_GLU_PF, t=[0, 1, 3, 4, 7, 8, 5], i=[I, H, E, abi.ENC_INT4G, 0, abi.ACT_SILU, G, abi.ARM_A16], slots=stated),
              abi.inst(abi.OP_MOE_GROUP_DOWN_PF, t=[6, 0, 3, 4, 7, 5, 9, 10], i=[H, I, E, abi.ENC_INT4G, 0, 0, G, abi.ARM_A16], slots=stated)):
        moe.exec(d, tensors)
    torch.cuda.synchronize()
    assert (part[-1] == 3).all()
    for e in range(E):
        s = (eid.view(-1) == e).nonzero()[:, 0]
        d = [ec.dequant64(*m[e]).T.contiguous() for m in sets]
        xr = x[(s // k).cuda()].double()
        # the intermediate rounds to bf16: half a step of each value, spread evenly, 0.58 of it in the mean square
        want = ec.act64(xr @ d[0], xr @ d[1], abi.ACT_SILU) @ d[2] * gate.view(-1)[s].cuda().double()[:, None]
        assert (part[s.cuda()].double() - want).norm() <= 0.65 * HALF_BF16 * want.norm(), e


@pytest.mark.parametrize("T", [2, 50, 400])
def test_experts_without_a_context(moe, T):
    fn = moe.lib.plow_moe_exec_noalloc

    def run(insts, t):
        err, tab = C.create_string_buffer(256), ec.table_of(t)
        for d in insts:
            assert fn(C.byref(d), tab, None, err, 256) == 0, err.value
    routed(8, 256, 160, 32, torch.randint(0, 8, (T, 4), generator=ec.gen(T), dtype=torch.int32), run)


@pytest.mark.parametrize("scale", [1e30, 1e-30, 50.0])
def test_extreme_temperatures(moe, scale):
    T, V, A = 3, 5000, 7
    g = ec.gen(6)
    x = torch.randn(T, V, generator=g)
    x[1, 17] = 30.0
    ids = torch.randint(0, V, (T, 2), generator=g, dtype=torch.int32)
    ids[1, 0] = 17
    want = ec.logprob64(x, V, ids, A, scale)
    lp, ent, lse = torch.zeros(T, 2, device="cuda"), torch.zeros(T, device="cuda"), torch.zeros(T, device="cuda")
    aid, alp = torch.zeros(T, A, dtype=torch.int32, device="cuda"), torch.zeros(T, A, device="cuda")
    moe.exec(abi.inst(abi.OP_X_LOGPROB, t=[0, 1, 2, 3, 4, 5, 6], i=[T, V, 2, A, 0, abi.LOGPROB_F32], f=[scale]),
             ec.table_of([lp, x.cuda(), ids.cuda(), ent, aid, alp, lse]))
    torch.cuda.synchronize()
    assert torch.equal(aid.cpu(), want["alt_ids"])
    for got, k in ((lp, "logprob"), (ent, "entropy"), (lse, "lse"), (alp, "alt_logprob")):
        got = got.cpu().double()
        assert torch.isfinite(got).all(), k
        # c itself rounds to f32, c (x - m) twice more; Z is off by (V / 64 + 16) roundings; the entropy weights d by e^d
        tol = EPS_F32 * (4 * (V / 64 + 16) + 4 * want[k].abs()) + (4 * EPS_F32 * 30 * min(scale, 50.0) if k == "entropy" else 0)
        assert ((got - want[k]).abs() <= tol).all(), (k, (got - want[k]).abs().max())


def test_graphs_of_two_contexts_side_by_side():
    """Split products and split rows of logits captured from a context each, replayed on two streams at once."""
    from plow_amd.lib import Moe
    jobs = []
    for n, (M, N, K) in enumerate([(16, 7168, 2048), (100, 1000, 4096)]):
        m, w = Moe(0), weights(gen(n), N, K, 64)
        x = torch.randn(M, K, generator=gen(n + 9), device="cuda").to(torch.bfloat16)
        o, lse = torch.zeros(M, N, device="cuda"), torch.zeros(M, device="cuda")
        aid = torch.zeros(M, 9, dtype=torch.int32, device="cuda")
        insts = [abi.inst(abi.OP_X_GEMM_W4, t=[0, 1, 2, 3, 4], i=[M, N, K, 64, 0, 0, 1]),
                 abi.inst(abi.OP_X_LOGPROB, t=[None, 0, None, None, 5, None, 6], i=[M, N, 0, 9, 0, abi.LOGPROB_F32])]
        tab = ec.table_of([o, x, *w, aid, lse])
        m.exec_many(insts, tab)
        torch.cuda.synchronize()
        want = [t.clone() for t in (o, aid, lse)]
        st, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.stream(st):
            g.capture_begin()
            m.exec_many(insts, tab, st.cuda_stream)
            g.capture_end()
        jobs.append((m, g, st, (o, aid, lse), want, (x, w, insts, tab)))
    torch.cuda.synchronize()
    for _ in range(4):
        for _, _, _, out, _, _ in jobs:
            for t in out:
                t.zero_()
        torch.cuda.synchronize()
        for _ in range(10):
            for _, g, st, _, _, _ in jobs:
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        for _, _, _, out, want, _ in jobs:
            for a, b in zip(out, want):
                assert torch.equal(a, b)
    for j in jobs:
        j[0].close()
