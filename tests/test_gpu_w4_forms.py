"""The int4 products at sizes where their many-row kernels come into play: tiles of 16 to 128 rows, one or two sets of
channels a wave, with and without a split of K, for each group size with and without zero points, K ending inside a
step and N inside a tile. References in 64 bits."""
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


def gpu(s):
    return tuple(None if t is None else t.cuda() for t in s)


PRODUCTS = [(24, 4100, 2176), (24, 65500, 512), (33, 24000, 384), (200, 4100, 640), (36, 33000, 640), (48, 17000, 2176),
            (120, 33000, 384), (400, 3000, 4096), (96, 7168, 2048)]


@pytest.mark.parametrize("zero", [False, True])
@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_product_forms(moe, M, N, K, G, zero):
    K -= G % 128                                     # not a multiple of the kernels' steps
    print(f"[case] product M={M} N={N} K={K} G={G} zero={zero}", flush=True)
    g = ec.gen(M + N + G)
    w = gpu(ec.weights(g, (), N, K, G, zero, "f16" if zero else "bf16"))
    x = torch.randn(M, K, generator=g).to(torch.bfloat16).cuda()
    o = torch.full((M + 1, N), 7.0, device="cuda")
    inst = abi.inst(abi.OP_X_GEMM_W4, t=[0, 1, 2, 3, 4 if zero else None],
                    i=[M, N, K, ec.group_field(G, "f16" if zero else "bf16"), 0, 0, 1])
    moe.exec(inst, ec.table_of([o, x, *w]))
    want = x.double() @ ec.dequant64(*w).T.contiguous()
    assert (o[M] == 7).all(), "written outside the output"
    err = (o[:M].double() - want).abs()
    bound = ec.abs_bound(x, *w)
    assert (err <= bound + EPS_F32 * want.abs()).all(), (err / bound).max()
    assert err.norm() <= 1e-6 * want.norm(), err.norm() / want.norm()


GLUS = [(36, 17000, 640), (20, 17000, 384), (36, 4100, 4096), (250, 4100, 384), (250, 1000, 4096), (200, 4100, 640), (30, 9000, 640), (500, 4100, 640)]


@pytest.mark.parametrize("zero", [False, True])
@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("M,N,K", GLUS)
def test_glu_forms(moe, M, N, K, G, zero):
    K -= G % 128
    print(f"[case] glu M={M} N={N} K={K} G={G} zero={zero}", flush=True)
    g = ec.gen(M + N + G)
    a, b = (gpu(ec.weights(g, (), N, K, G, zero, "bf16", 0.02)) for _ in range(2))
    x = torch.randn(M, K, generator=g).to(torch.bfloat16).cuda()
    o = torch.full((M + 1, N), 7.0, dtype=torch.bfloat16, device="cuda")
    z = zero or None
    inst = abi.inst(abi.OP_X_GEMM_GLU_W4, t=[0, 1, 2, 3, z and 4, 5, 6, z and 7], i=[M, N, K, G, 0, abi.ACT_SILU])
    moe.exec(inst, ec.table_of([o, x, *a, *b]))
    gt, up = x.double() @ ec.dequant64(*a).T.contiguous(), x.double() @ ec.dequant64(*b).T.contiguous()
    want = ec.act64(gt, up, abi.ACT_SILU)
    assert (o[M] == 7).all(), "written outside the output"
    got = o[:M].double()
    # the activation's slope is below 1.2 and its size below |g| + 1; its own few roundings in f32, half a step of the result
    eg, eu = ec.abs_bound(x, *a), ec.abs_bound(x, *b)
    tol = 1.2 * eg * (up.abs() + 1 + eu) + 1.2 * eu * (gt.abs() + 1) + 2.0 ** -19 * (want.abs() + 1e-6)
    assert ((got - want).abs() <= tol + HALF_BF16 * (want.abs() + tol)).all()
    assert (got - want).norm() <= 0.65 * HALF_BF16 * want.norm()


@pytest.mark.parametrize("zero", [False, True])
@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("T,E,k,H,I", [(40, 4, 2, 2176, 1100), (90, 4, 2, 640, 1408), (70, 2, 1, 384, 640), (260, 3, 2, 384, 640), (20, 40, 8, 1408, 640)])
def test_experts_many_rows(moe, T, E, k, H, I, G, zero):
    """Slot-major experts whose average rows call for tiles of 16, 32 and 64 rows, one expert taking more of them."""
    I -= I % G
    H -= H % G
    print(f"[case] experts T={T} E={E} k={k} H={H} I={I} G={G} zero={zero}", flush=True)
    g = ec.gen(T + E + G)
    sets = [gpu(ec.weights(g, (E,), n, kk, G, zero, "bf16", 0.02)) for n, kk in ((I, H), (I, H), (H, I))]
    tabs = [None if sets[0][c] is None else torch.tensor([[s[c][e].data_ptr() for s in sets] for e in range(E)], dtype=torch.int64).cuda()
            for c in range(3)]
    score = torch.rand(T, E, generator=g)
    score[: T // 3, 0] += 1.0
    eid = score.topk(k, dim=1).indices.to(torch.int32)
    eid[T // 2, 0] = -1                               # a slot that no expert serves
    gate = torch.rand(T, k, generator=g) + 0.1
    tab = torch.stack([eid, gate.view(torch.int32)], 2).reshape(T * k, 2).contiguous().cuda()
    x = torch.randn(T, H, generator=g).to(torch.bfloat16).cuda()
    fu = torch.full((T * k + 1, I), 3.0, dtype=torch.bfloat16, device="cuda")
    part = torch.full((T * k + 1, H), 3.0, device="cuda")
    z = 5 if zero else None
    insts = [abi.inst(abi.OP_MOE_GROUP_GLU_FP8_BLK, t=[0, 1, 2, 3, 4, z], i=[T * k, I, H, E, k, abi.ACT_SILU, abi.ENC_INT4G, G]),
             abi.inst(abi.OP_MOE_GROUP_DOWN_FP8_BLK, t=[6, 0, 2, 3, 4, z], i=[T * k, H, I, E, 0, 0, abi.ENC_INT4G, G])]
    moe.exec_many(insts, ec.table_of([fu, x, tab, *tabs, part]))
    torch.cuda.synchronize()
    assert (fu[-1] == 3).all() and (part[-1] == 3).all()
    e_of, slot = eid.view(-1), torch.arange(T * k)
    assert (part[:-1].cpu()[e_of < 0] == 0).all() and (fu[:-1].cpu()[e_of < 0] == 3).all()
    for e in range(E):
        s = slot[e_of == e].cuda()
        if not len(s):
            continue
        d = [ec.dequant64(*(None if t is None else t[e] for t in m)).T.contiguous() for m in sets]
        xr = x[s // k].double()
        want = ec.act64(xr @ d[0], xr @ d[1], abi.ACT_SILU)
        assert (fu[s].double() - want).norm() <= 0.65 * HALF_BF16 * want.norm(), e
        want = fu[s].double() @ d[2] * gate.view(-1)[s.cpu()].cuda().double()[:, None]
        assert (part[s].double() - want).norm() <= 1e-6 * want.norm(), e
