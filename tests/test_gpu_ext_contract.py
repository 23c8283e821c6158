"""What the int4 and log-probability ops promise beyond their formulas: finite log probabilities wherever the value is
representable, the same bits on every call whatever staging the context holds, a kernel form that follows the call's
rows."""
import ctypes as C

import numpy as np
import pytest
import torch

import ext_cases as ec
from plow_amd import abi

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def moe():
    from plow_amd.lib import Moe
    m = Moe(0)
    yield m
    m.close()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [50, 20000])
@pytest.mark.parametrize("scale", [0.25, 0.49, 1e-30])
def test_logits_further_apart_than_a_type_reaches(moe, V, dtype, scale):
    """Largest minus smallest logit is past the largest f32, the log probability c (x - m) - ln Z is not."""
    print(f"[case] far apart V={V} {dtype} c={scale}", flush=True)
    T, A, top = 3, 7, torch.finfo(dtype).max
    x = torch.randn(T, V, generator=ec.gen(V))
    x[:, 5] = top
    x[0, 9] = -top
    x[1, V - 1] = -top * 0.99
    x[2, 6:] = -top
    x[2, 20] = 0.0
    x = x.to(dtype)
    ids = torch.tensor([[9, 5], [V - 1, 0], [6, 20]], dtype=torch.int32)
    c = float(np.float32(scale))
    want = ec.logprob64(x, V, ids, A, c)
    lp, ent, lse = torch.zeros(T, 2, device="cuda"), torch.zeros(T, device="cuda"), torch.zeros(T, device="cuda")
    aid, alp = torch.zeros(T, A, dtype=torch.int32, device="cuda"), torch.zeros(T, A, device="cuda")
    moe.exec(abi.inst(abi.OP_X_LOGPROB, t=[0, 1, 2, 3, 4, 5, 6], i=[T, V, 2, A, 0, abi.LOGPROB_F32 if dtype == torch.float32 else 0], f=[scale]),
             ec.table_of([lp, x.cuda(), ids.cuda(), ent, aid, alp, lse]))
    torch.cuda.synchronize()
    assert torch.equal(aid.cpu(), want["alt_ids"])
    # x - m, c times it and ln Z taken off: a rounding each; every other token's e^d is 0, so that ln Z and the entropy
    # are 0, and c m of the log of the sum rounds once
    for got, k in ((lp, "logprob"), (ent, "entropy"), (lse, "lse"), (alp, "alt_logprob")):
        got = got.cpu().double()
        assert torch.isfinite(got).all(), (k, got)
        assert ((got - want[k]).abs() <= 3 * ec.EPS_F32 * want[k].abs()).all(), (k, got, want[k])


@pytest.mark.parametrize("M,N,K,glu", [(300, 14336, 8192, False), (1000, 2100, 14336, True), (700, 4096, 14336, False), (90, 7168, 7168, False)])
def test_same_bits_whatever_staging_the_context_holds(M, N, K, glu):
    """A larger staging block does not cut a dense call differently."""
    from plow_amd.lib import Moe
    print(f"[case] staging M={M} N={N} K={K} glu={glu}", flush=True)
    moe, g = Moe(0), ec.gen(M)
    a, b = (tuple(t.cuda() for t in ec.weights(g, (), N, K, 128, True, "bf16")) for _ in range(2))
    x = torch.randn(M, K, generator=g).to(torch.bfloat16).cuda()
    outs = []
    for grow in (0, 1):
        if grow:
            moe.reserve_staging(1 << 14, 1 << 15)            # 285 MB
        o = torch.zeros(M, N, dtype=torch.bfloat16 if glu else torch.float32, device="cuda")
        inst = (abi.inst(abi.OP_X_GEMM_GLU_W4, t=[0, 1, 2, 3, 4, 5, 6, 7], i=[M, N, K, 128, 0, abi.ACT_SILU]) if glu else
                abi.inst(abi.OP_X_GEMM_W4, t=[0, 1, 2, 3, 4], i=[M, N, K, 128, 0, 0, 1]))
        moe.exec(inst, ec.table_of([o, x, *a, *b]))
        torch.cuda.synchronize()
        outs.append(o.cpu())
    assert torch.equal(outs[0], outs[1]), (outs[0].float() - outs[1].float()).abs().max()
    moe.close()


def experts(E, H, I, G, seed):
    g = ec.gen(seed)
    sets = [tuple(t.cuda() for t in ec.weights(g, (E,), n, k, G, True, "bf16", 0.02)) for n, k in ((I, H), (I, H), (H, I))]
    return sets, [torch.tensor([[s[c][e].data_ptr() for s in sets] for e in range(E)], dtype=torch.int64).cuda() for c in range(3)]


@pytest.mark.parametrize("E,slots,tiles", [(4, 48, True), (8, 64, True), (16, 64, True), (32, 64, True), (8, 16, False), (64, 48, False)])
def test_slots_that_share_experts_run_as_tiles(moe, E, slots, tiles):
    """Slot-major experts of a few slots each stream their expert by themselves only while few slots share one: with more
    of them the rows run as the tiles of a larger batch do, bit for bit."""
    print(f"[case] shared experts E={E} slots={slots}", flush=True)
    H, I, G, k = 2048, 512, 64, 2
    sets, tabs = experts(E, H, I, G, 4)
    T = slots // k
    eid = torch.rand(T, E, generator=ec.gen(E)).topk(k, dim=1).indices.to(torch.int32)
    x = torch.randn(33, H, generator=ec.gen(6)).to(torch.bfloat16).cuda()
    got = []
    for rows in (T, 33):                                     # 66 slots always run as tiles; the rows behind T are padding
        e2 = torch.full((rows, k), -1, dtype=torch.int32)
        e2[:T] = eid
        gate = torch.full((rows, k), 0.75)
        tab = torch.stack([e2, gate.view(torch.int32)], 2).reshape(rows * k, 2).contiguous().cuda()
        fu, part = torch.zeros(rows * k, I, dtype=torch.bfloat16, device="cuda"), torch.zeros(rows * k, H, device="cuda")
        moe.exec_many([abi.inst(abi.OP_MOE_GROUP_GLU_FP8_BLK, t=[0, 1, 2, 3, 4, 5], i=[rows * k, I, H, E, k, abi.ACT_SILU, abi.ENC_INT4G, G]),
                       abi.inst(abi.OP_MOE_GROUP_DOWN_FP8_BLK, t=[6, 0, 2, 3, 4, 5], i=[rows * k, H, I, E, 0, 0, abi.ENC_INT4G, G])],
                      ec.table_of([fu, x, tab, *tabs, part]))
        torch.cuda.synchronize()
        got.append((fu[:slots].cpu(), part[:slots].cpu()))
    assert (torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])) == tiles
    assert (got[0][1].double() - got[1][1].double()).norm() <= 2.0 ** -8 * got[1][1].double().norm()


@pytest.mark.parametrize("form", ["one by one", "one by one, captured", "segment"])
@pytest.mark.parametrize("T,E,k", [(333, 4, 2), (700, 3, 1), (30, 8, 2), (3, 8, 2), (97, 8, 2), (96, 8, 2)])
def test_gathered_experts_without_a_stated_count(moe, T, E, k, form):
    """Ops 85 / 86 whose caller states no row count: the form is chosen on the device from the routing meta and the bytes
    are those of the run that states the count (24 rows of an expert on average lie on one side, more on the other)."""
    print(f"[case] unstated T={T} E={E} k={k} {form}", flush=True)
    H, I, G = 2176, 1152, 64
    sets, tabs = experts(E, H, I, G, 3)
    eid = torch.rand(T, E, generator=ec.gen(T)).topk(k, dim=1).indices.to(torch.int32)
    gate = torch.rand(T, k, generator=ec.gen(2)) + 0.1
    tab = torch.stack([eid, gate.view(torch.int32)], 2).reshape(T * k, 2).contiguous().cuda()
    x = torch.randn(T, H, generator=ec.gen(5)).to(torch.bfloat16).cuda()
    R = abi.max_rows(T, k, E)
    maps = [torch.zeros(n, dtype=torch.int32, device="cuda") for n in (3 * E + 1, R, R, R)]
    fu, part = torch.zeros(R, I, dtype=torch.bfloat16, device="cuda"), torch.zeros(T * k + 1, H, device="cuda")
    tensors = ec.table_of([fu, x, tab, *tabs, part, *maps])

    def ops(n):
        return [abi.inst(abi.OP_MOE_GROUP_GLU_PF, t=[0, 1, 3, 4, 7, 8, 5], i=[I, H, E, abi.ENC_INT4G, 0, abi.ACT_SILU, G, abi.ARM_A16], slots=n),
                abi.inst(abi.OP_MOE_GROUP_DOWN_PF, t=[6, 0, 3, 4, 7, 5, 9, 10], i=[H, I, E, abi.ENC_INT4G, 0, 0, G, abi.ARM_A16], slots=n)]
    moe.exec(abi.inst(abi.OP_MOE_ALIGN_PF, t=[7, 2, 8, 9, 10], i=[T, E, k]), tensors)
    got = []
    for n in (T * k, 0):
        fu.fill_(3.0), part.fill_(3.0)
        run = ops(n)
        torch.cuda.synchronize()
        if n or form == "one by one":
            for d in run:
                moe.exec(d, tensors)
        elif form == "segment":
            moe.pf(run, tensors, T)
        else:
            side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
            with torch.cuda.stream(side):
                graph.capture_begin()
                for d in run:
                    moe.exec(d, tensors, side.cuda_stream)
                graph.capture_end()
            for _ in range(3):
                fu.fill_(3.0), part.fill_(3.0)
                graph.replay()
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        got.append((fu.cpu(), part.cpu()))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    assert (got[1][1][-1] == 3).all()


def test_gathered_experts_without_a_context_choose_nothing_on_the_device(moe):
    """plow_moe_exec_noalloc has one workspace for all calls on a GPU: ops 85 / 86 use nothing of it, so that calls on
    several streams may overlap, each with the bytes of the form for few rows."""
    E, k, H, I, G = 4, 2, 2176, 1152, 64
    sets, tabs = experts(E, H, I, G, 9)
    jobs = []
    for T in (6, 300, 500, 9):
        eid = torch.rand(T, E, generator=ec.gen(T)).topk(k, dim=1).indices.to(torch.int32)
        tab = torch.stack([eid, torch.full((T, k), 0.5).view(torch.int32)], 2).reshape(T * k, 2).contiguous().cuda()
        x = torch.randn(T, H, generator=ec.gen(5)).to(torch.bfloat16).cuda()
        R = abi.max_rows(T, k, E)
        maps = [torch.zeros(n, dtype=torch.int32, device="cuda") for n in (3 * E + 1, R, R, R)]
        fu, part = torch.zeros(R, I, dtype=torch.bfloat16, device="cuda"), torch.zeros(T * k, H, device="cuda")
        keep = [fu, x, tab, *tabs, part, *maps]
        tensors = ec.table_of(keep)
        pair = [abi.inst(abi.OP_MOE_GROUP_GLU_PF, t=[0, 1, 3, 4, 7, 8, 5], i=[I, H, E, abi.ENC_INT4G, 0, abi.ACT_SILU, G, abi.ARM_A16]),
                abi.inst(abi.OP_MOE_GROUP_DOWN_PF, t=[6, 0, 3, 4, 7, 5, 9, 10], i=[H, I, E, abi.ENC_INT4G, 0, 0, G, abi.ARM_A16])]
        moe.exec(abi.inst(abi.OP_MOE_ALIGN_PF, t=[7, 2, 8, 9, 10], i=[T, E, k]), tensors)
        assert moe.dec(pair, tensors, T) == 0                # the decode segment: the form for few rows, whatever the count
        torch.cuda.synchronize()
        want = (fu.clone(), part.clone())
        fu.zero_(), part.zero_()
        jobs.append((pair, tensors, keep, want, torch.cuda.Stream()))
    torch.cuda.synchronize()
    err = C.create_string_buffer(256)
    for _ in range(5):
        for pair, tensors, _, _, st in jobs:
            for d in pair:
                assert moe.lib.plow_moe_exec_noalloc(C.byref(d), tensors, st.cuda_stream, err, 256) == 0, err.value
    torch.cuda.synchronize()
    for _, _, keep, want, _ in jobs:
        assert torch.equal(keep[0], want[0]) and torch.equal(keep[6], want[1])
