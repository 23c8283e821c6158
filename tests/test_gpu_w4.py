"""Products with 4-bit integer weights and group scales on the GPU against 64-bit references: the dense ops over row
counts, odd widths, groups, zero points, scale types, pitches and output types; GLU activations; routed experts slot by
slot (with padded slots and experts that are not resident) and on gathered rows."""
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


def dev(t):
    return None if t is None else t.cuda()


def run(moe, insts, tensors):
    keep = [dev(t) if t is not None and not t.is_cuda else t for t in tensors]
    moe.exec_many(insts, ec.table_of(keep))
    torch.cuda.synchronize()
    return keep


def product(moe, M, N, K, G, zero, scale, out, ldx=0, ldo=0, seed=0):
    g = ec.gen(seed + M * 7 + N)
    W, S, Z = ec.weights(g, (), N, K, G, zero, scale)
    px, po = ldx or K, ldo or N
    x = torch.randn(M, px, generator=g).to(torch.bfloat16)
    dt = torch.float32 if out == "f32" else torch.bfloat16
    o = torch.full((M + 1, po), 7.0, dtype=dt, device="cuda")
    inst = abi.inst(abi.OP_X_GEMM_W4, t=[0, 1, 2, 3, 4 if zero else None],
                    i=[M, N, K, ec.group_field(G, scale), ldx, ldo, 1 if out == "f32" else 0])
    run(moe, [inst], [o, x, W, S, Z])
    got = o.cpu().double()
    assert (got[M] == 7.0).all() and (got[:, N:] == 7.0).all(), "written outside the output"
    want = x[:, :K].double() @ ec.dequant64(W, S, Z).T
    err = (got[:M, :N] - want).abs()
    bound = ec.abs_bound(x[:, :K], W, S, Z)
    half = HALF_BF16 if out == "bf16" else EPS_F32
    assert (err <= (bound + half * (want.abs() + bound))).all(), (err / bound).max()
    rel = (err.norm() / want.norm()).item()
    # roundings to bf16 are spread evenly over half a step: 0.58 of it in the mean square; f32 sums of a few thousand
    # terms with random signs lie within a few 2^-24 of the terms' norm, the offset of 16 costs a factor of 7
    assert rel <= (0.6 * HALF_BF16 if out == "bf16" else 1e-6), rel
    return rel


SHAPES = [(1, 1, 32, 32), (1, 17, 64, 32), (1, 130, 256, 128), (2, 63, 96, 32), (3, 64, 1408, 128), (4, 257, 192, 64),
          (5, 16, 320, 64), (8, 100, 2816, 128), (15, 33, 4096, 32), (16, 128, 512, 64), (17, 129, 1024, 128), (31, 48, 224, 32),
          (33, 255, 384, 128), (48, 65, 1152, 64), (64, 320, 768, 32), (65, 31, 640, 128), (127, 144, 2048, 64),
          (128, 512, 256, 32), (130, 129, 1408, 128), (257, 260, 448, 64), (513, 96, 160, 32)]


@pytest.mark.parametrize("zero", [False, True])
@pytest.mark.parametrize("M,N,K,G", SHAPES)
def test_product(moe, M, N, K, G, zero):
    print(f"[case] product M={M} N={N} K={K} G={G} zero={zero}", flush=True)
    scale = "f16" if (M + N) % 2 else "bf16"
    for out in ("bf16", "f32"):
        product(moe, M, N, K, G, zero, scale, out)


@pytest.mark.parametrize("M", [1, 4, 16, 40, 200])
def test_product_pitches(moe, M):
    print(f"[case] pitches M={M}", flush=True)
    product(moe, M, 77, 384, 64, True, "bf16", "f32", ldx=392, ldo=80)
    product(moe, M, 77, 384, 128, False, "f16", "bf16", ldx=1024, ldo=1001)


@pytest.mark.parametrize("M", [1, 3, 16, 100])
def test_product_wide_and_long(moe, M):
    """A head-like width and long rows."""
    print(f"[case] wide M={M}", flush=True)
    product(moe, M, 20011, 512, 64, False, "bf16", "f32")
    product(moe, M, 192, 14336, 128, True, "bf16", "f32")
    product(moe, M, 640, 7168, 32, False, "f16", "bf16")


def test_rows_are_independent(moe):
    """A row with an infinity or NaN spoils its own outputs only; signed zeros and the largest codes stay exact."""
    g = ec.gen(5)
    for M in (1, 5, 40, 130):
        N, K, G = 70, 256, 64
        W, S, Z = ec.weights(g, (), N, K, G, False, "bf16")
        x = torch.randn(M + 2, K, generator=g).to(torch.bfloat16)
        x[M // 2, 7] = float("inf")
        x[M // 2 + 1, 9] = float("nan")
        o = torch.zeros(M + 2, N, device="cuda")
        run(moe, [abi.inst(abi.OP_X_GEMM_W4, t=[0, 1, 2, 3], i=[M + 2, N, K, G, 0, 0, 1])], [o, x, W, S])
        got = o.cpu().double()
        bad = torch.zeros(M + 2, dtype=torch.bool)
        bad[M // 2] = bad[M // 2 + 1] = True
        assert not torch.isfinite(got[bad]).any()
        want = x[~bad].double() @ ec.dequant64(W, S, Z).T
        assert (got[~bad] - want).norm() <= 1e-6 * want.norm()


def test_product_exact_integers(moe):
    """Small integer activations and power-of-two scales: every sum is exact, so the output is equal."""
    g = ec.gen(9)
    for M in (1, 2, 7, 16, 33, 129):
        for G in (32, 64, 128):
            N, K = 150, 512
            W, S, Z = ec.weights(g, (), N, K, G, True, "bf16")
            S = torch.pow(2.0, torch.randint(-3, 3, S.shape, generator=g).float()).to(torch.bfloat16)
            x = torch.randint(-8, 9, (M, K), generator=g).to(torch.bfloat16)
            o = torch.zeros(M, N, device="cuda")
            run(moe, [abi.inst(abi.OP_X_GEMM_W4, t=[0, 1, 2, 3, 4], i=[M, N, K, G, 0, 0, 1])], [o, x, W, S, Z])
            assert torch.equal(o.cpu().double(), x.double() @ ec.dequant64(W, S, Z).T), (M, G)


GLU_SHAPES = [(1, 33, 64, 32), (1, 512, 2048, 128), (2, 100, 256, 64), (4, 65, 384, 128), (9, 130, 320, 32), (16, 96, 1408, 128),
              (30, 257, 192, 64), (61, 80, 512, 128), (64, 64, 96, 32), (90, 144, 768, 64), (300, 130, 256, 32)]


@pytest.mark.parametrize("M,N,K,G", GLU_SHAPES)
def test_glu(moe, M, N, K, G):
    print(f"[case] glu M={M} N={N} K={K} G={G}", flush=True)
    g = ec.gen(M + N)
    zero, scale = M % 2 == 0, "f16" if N % 2 else "bf16"
    a, b = ec.weights(g, (), N, K, G, zero, scale, 0.02), ec.weights(g, (), N, K, G, zero, scale, 0.02)
    x = torch.randn(M, K, generator=g).to(torch.bfloat16)
    o = torch.full((M + 1, N + 3), 7.0, dtype=torch.bfloat16, device="cuda")
    z = zero or None
    inst = abi.inst(abi.OP_X_GEMM_GLU_W4, t=[0, 1, 2, 3, z and 4, 5, 6, z and 7],
                    i=[M, N, K, ec.group_field(G, scale), 0, abi.ACT_SILU, N + 3])
    run(moe, [inst], [o, x, *a, *b])
    got = o.cpu().double()
    assert (got[M] == 7).all() and (got[:, N:] == 7).all()
    gt, up = x.double() @ ec.dequant64(*a).T, x.double() @ ec.dequant64(*b).T
    check_glu(got[:M, :N], gt, up, ec.abs_bound(x, *a[:2], a[2]), ec.abs_bound(x, *b[:2], b[2]))


def check_glu(got, gt, up, eg, eu, act=1, f0=0.0, f1=0.0):
    """The activation's slope is below 1.2 and its size below |g| + 1; expf, the division and the products round a few
    times in f32; half a bf16 step on the result."""
    want = ec.act64(gt, up, act, f0, f1)
    tol = 1.2 * eg * (up.abs() + 1 + eu) + eu * (gt.abs() + 1) * 1.2
    tol = tol + 2.0 ** -19 * (want.abs() + 1e-6)
    assert ((got - want).abs() <= tol + HALF_BF16 * (want.abs() + tol)).all()
    # roundings spread over half a step, except where an activation clamps: many outputs are then the same value with
    # the same rounding (limit 1.25: silu(1.25) * 1.25 = 1.21453 lies 0.46 of a step of 2^-7 off its bf16 neighbour)
    assert (got - want).norm() <= (1.0 if act >= 2 else 0.65) * HALF_BF16 * want.norm()


@pytest.mark.parametrize("M", [1, 12, 80])
@pytest.mark.parametrize("act,f0,f1", [(0, 0.0, 0.0), (2, 1.5, 2.0), (2, 1.5, 0.0), (3, 1.702, 2.0), (4, 0.0, 1.25)])
def test_glu_activations(moe, M, act, f0, f1):
    g = ec.gen(act + M)
    N, K, G = 96, 256, 32
    a, b = ec.weights(g, (), N, K, G, False, "bf16", 0.03), ec.weights(g, (), N, K, G, False, "bf16", 0.03)
    x = torch.randn(M, K, generator=g).to(torch.bfloat16)
    o = torch.zeros(M, N, dtype=torch.bfloat16, device="cuda")
    run(moe, [abi.inst(abi.OP_X_GEMM_GLU_W4, t=[0, 1, 2, 3, None, 5, 6], i=[M, N, K, G, 0, act], f=[f0, f1])], [o, x, *a, *b])
    gt, up = x.double() @ ec.dequant64(*a).T, x.double() @ ec.dequant64(*b).T
    check_glu(o.cpu().double(), gt, up, ec.abs_bound(x, *a), ec.abs_bound(x, *b), act, f0, f1)


# ---- routed experts --------------------------------------------------------------------------------

def expert_set(E, H, I, G, zero, scale, seed, std=0.02):
    g = ec.gen(seed)
    sets = [ec.weights(g, (E,), n, k, G, zero, scale, std) for n, k in ((I, H), (I, H), (H, I))]
    d = [tuple(dev(t) for t in s) for s in sets]

    def ptr(col):
        if d[0][col] is None:
            return None
        return torch.tensor([[s[col][e].data_ptr() for s in d] for e in range(E)], dtype=torch.int64)
    return sets, d, [ptr(0), ptr(1), ptr(2)]


def routing(T, E, k, seed, idle=0.0, hot=False):
    g = ec.gen(seed)
    score = torch.rand(T, E, generator=g)
    if hot:
        score[:, E // 2] += 1.0
    eid = score.topk(k, dim=1).indices.to(torch.int32)
    if idle:
        eid[torch.rand(T, k, generator=g) < idle] = -1
    gate = torch.rand(T, k, generator=g) + 0.1
    return eid, gate, torch.stack([eid, gate.view(torch.int32)], 2).reshape(T * k, 2).contiguous()


def check_slots(sets, x, eid, gate, fu, part, G, act, absent=()):
    """fu and part slot by slot; part against the fu that was written (a bf16 tensor of its own)."""
    T, k = eid.shape
    deq = [[None] * eid.max().add(1).clamp(min=1).item() for _ in range(3)]
    e2 = n2 = fe2 = fn2 = 0.0
    for s in range(T * k):
        e = int(eid.view(-1)[s])
        if e < 0 or e in absent:
            assert (part[s] == 0).all(), f"slot {s} is not served: its row must be zero"
            continue
        for j in range(3):
            if deq[j][e] is None:
                deq[j][e] = ec.dequant64(*(None if t is None else t[e] for t in sets[j]))
        xr = x[s // k].double()
        want_fu = ec.act64(deq[0][e] @ xr, deq[1][e] @ xr, act)
        err = fu[s] - want_fu
        fe2, fn2 = fe2 + float(err @ err), fn2 + float(want_fu @ want_fu)
        assert (err.abs() <= 1.1 * HALF_BF16 * want_fu.abs() + 1e-4 * want_fu.abs().max()).all(), s
        want = (deq[2][e] @ fu[s]) * float(gate.view(-1)[s])
        d = part[s] - want
        e2, n2 = e2 + float(d @ d), n2 + float(want @ want)
    if fn2:
        assert fe2 ** 0.5 <= 0.65 * HALF_BF16 * fn2 ** 0.5, (fe2 / fn2) ** 0.5
        assert e2 ** 0.5 <= 1e-6 * n2 ** 0.5, (e2 / n2) ** 0.5


SLOT_CASES = [  # T, E, k, H, I, G, zero, idle, hot
    (1, 4, 1, 128, 32, 32, False, 0.0, False), (1, 16, 4, 256, 160, 32, True, 0.0, False), (2, 8, 2, 320, 96, 32, False, 0.5, False),
    (3, 5, 5, 512, 192, 64, True, 0.2, False), (7, 32, 8, 256, 128, 128, False, 0.0, False), (16, 12, 3, 1408, 64, 64, True, 0.1, True),
    (40, 6, 2, 256, 224, 32, False, 0.1, True), (90, 3, 2, 384, 128, 128, True, 0.05, False), (200, 4, 2, 128, 256, 64, False, 0.0, True),
    (5, 1056, 8, 128, 32, 32, False, 0.0, False), (4, 3, 2, 128, 128, 128, False, 1.0, False)]


@pytest.mark.parametrize("case", SLOT_CASES, ids=str)
def test_experts_slot_major(moe, case):
    T, E, k, H, I, G, zero, idle, hot = case
    print(f"[case] slots {case}", flush=True)
    scale = "f16" if I % 64 else "bf16"
    sets, d, (wt, st, zt) = expert_set(E, H, I, G, zero, scale, T + E)
    eid, gate, tab = routing(T, E, k, T, idle, hot)
    x = torch.randn(T, H, generator=ec.gen(3)).to(torch.bfloat16)
    fu = torch.full((T * k + 1, I), 3.0, dtype=torch.bfloat16, device="cuda")
    part = torch.full((T * k + 1, H), 3.0, device="cuda")
    f = ec.group_field(G, scale)
    z = 5 if zero else None
    insts = [abi.inst(abi.OP_MOE_GROUP_GLU_FP8_BLK, t=[0, 1, 2, 3, 4, z], i=[T * k, I, H, E, k, abi.ACT_SILU, abi.ENC_INT4G, f]),
             abi.inst(abi.OP_MOE_GROUP_DOWN_FP8_BLK, t=[6, 0, 2, 3, 4, z], i=[T * k, H, I, E, 0, 0, abi.ENC_INT4G, f])]
    run(moe, insts, [fu, x, tab, wt, st, zt, part])
    fc, pc = fu.cpu().double(), part.cpu().double()
    assert (fc[-1] == 3).all() and (pc[-1] == 3).all()
    check_slots(sets, x, eid, gate, fc, pc, G, 1)


def test_experts_not_resident(moe):
    """An expert whose pointers are null is skipped: its slots' rows of the down product are zero."""
    T, E, k, H, I, G = 6, 8, 3, 128, 64, 32
    for col in (0, 1, 2):
        sets, d, tabs = expert_set(E, H, I, G, True, "bf16", 1)
        eid, gate, tab = routing(T, E, k, 2)
        absent = {int(eid[0, 0]), int(eid[3, 1])}
        for e in absent:
            tabs[col][e] = 0
        x = torch.randn(T, H, generator=ec.gen(3)).to(torch.bfloat16)
        fu = torch.zeros(T * k, I, dtype=torch.bfloat16, device="cuda")
        part = torch.full((T * k, H), 3.0, device="cuda")
        insts = [abi.inst(abi.OP_MOE_GROUP_GLU_FP8_BLK, t=[0, 1, 2, 3, 4, 5], i=[T * k, I, H, E, k, 1, abi.ENC_INT4G, G]),
                 abi.inst(abi.OP_MOE_GROUP_DOWN_FP8_BLK, t=[6, 0, 2, 3, 4, 5], i=[T * k, H, I, E, 0, 0, abi.ENC_INT4G, G])]
        run(moe, insts, [fu, x, tab, *tabs, part])
        check_slots(sets, x, eid, gate, fu.cpu().double(), part.cpu().double(), G, 1, absent)


GATHER_CASES = [  # T, E, k, H, I, G, zero, hot
    (1, 8, 2, 128, 64, 32, False, False), (9, 16, 4, 256, 160, 32, True, False), (50, 8, 2, 384, 128, 64, False, True),
    (130, 4, 2, 256, 192, 64, True, False), (300, 5, 3, 1408, 128, 128, False, True), (700, 2, 1, 128, 288, 32, True, False)]


@pytest.mark.parametrize("stated", [True, False])
@pytest.mark.parametrize("case", GATHER_CASES, ids=str)
def test_experts_gathered(moe, case, stated):
    """Ops 84, 85, 86 at the int4 encoding, with the row count stated or left to the op itself."""
    T, E, k, H, I, G, zero, hot = case
    print(f"[case] gathered {case} stated={stated}", flush=True)
    sets, d, (wt, st, zt) = expert_set(E, H, I, G, zero, "bf16", T + E)
    eid, gate, tab = routing(T, E, k, T, 0.0, hot)
    x = torch.randn(T, H, generator=ec.gen(3)).to(torch.bfloat16)
    R = abi.max_rows(T, k, E)
    fu = torch.full((R, I), 3.0, dtype=torch.bfloat16, device="cuda")
    part = torch.full((T * k + 1, H), 3.0, device="cuda")
    maps = [torch.zeros(n, dtype=torch.int32, device="cuda") for n in (3 * E + 1, R, R, R)]
    n = T * k if stated else 0
    z = 5 if zero else None
    insts = [abi.inst(abi.OP_MOE_ALIGN_PF, t=[7, 2, 8, 9, 10], i=[T, E, k]),
             abi.inst(abi.OP_MOE_GROUP_GLU_PF, t=[0, 1, 3, 4, 7, 8, z], i=[I, H, E, abi.ENC_INT4G, 0, 1, G, abi.ARM_A16], slots=n),
             abi.inst(abi.OP_MOE_GROUP_DOWN_PF, t=[6, 0, 3, 4, 7, z, 9, 10], i=[H, I, E, abi.ENC_INT4G, 0, 0, G, abi.ARM_A16], slots=n)]
    keep = [t.cuda() if t is not None else None for t in (x, tab, wt, st, zt)]
    tensors = [fu, *keep, part, *maps]
    for inst in insts:   # one at a time: no align op of the same run states the count
        moe.exec(inst, ec.table_of(tensors))
    torch.cuda.synchronize()
    rp = maps[2].cpu()
    rows = torch.zeros(T * k, dtype=torch.long)
    live = (rp >= 0).nonzero()[:, 0]
    used = int(maps[0].cpu()[3 * E]) * abi.MPF_BM
    live = live[live < used]
    rows[rp[live].long()] = live
    fc, pc = fu.cpu().double(), part.cpu().double()
    assert (pc[-1] == 3).all()
    check_slots(sets, x, eid, gate, fc[rows], pc, G, 1)


def test_same_bits_on_every_call(moe):
    """Sums have a fixed order: the same call gives the same bits."""
    g = ec.gen(1)
    for M, N, K in ((1, 300, 4096), (16, 300, 4096), (70, 200, 2048)):
        W, S, Z = (dev(t) for t in ec.weights(g, (), N, K, 64, True, "bf16"))
        x = torch.randn(M, K, generator=g).to(torch.bfloat16).cuda()
        outs = []
        for _ in range(3):
            o = torch.zeros(M, N, device="cuda")
            run(moe, [abi.inst(abi.OP_X_GEMM_W4, t=[0, 1, 2, 3, 4], i=[M, N, K, 64, 0, 0, 1])], [o, x, W, S, Z])
            outs.append(o.cpu())
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_noalloc_entry_point(moe):
    """The entry point without a context serves the ops too (no K split there: equal to rounding)."""
    import ctypes as C
    g = ec.gen(2)
    fn = moe.lib.plow_moe_exec_noalloc
    for M in (1, 16, 100):
        N, K, G = 200, 2048, 64
        W, S, Z = (dev(t) for t in ec.weights(g, (), N, K, G, True, "bf16"))
        x = torch.randn(M, K, generator=g).to(torch.bfloat16).cuda()
        a, b = torch.zeros(M, N, device="cuda"), torch.zeros(M, N, device="cuda")
        for o, call in ((a, "ctx"), (b, "none")):
            inst = abi.inst(abi.OP_X_GEMM_W4, t=[0, 1, 2, 3, 4], i=[M, N, K, G, 0, 0, 1])
            tab = ec.table_of([o, x, W, S, Z])
            if call == "ctx":
                moe.exec(inst, tab)
            else:
                err = C.create_string_buffer(256)
                assert fn(C.byref(inst), tab, None, err, 256) == 0, err.value
            torch.cuda.synchronize()
        assert (a - b).norm() <= 2e-6 * a.norm()
