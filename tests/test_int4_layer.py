"""Int4 group-scaled weights and log probabilities as they are used: the oracle's restatement against 64-bit torch and
torch's own quantizer round trip (CPU); whole layers and heads against the oracle, a layer and the head behind it in one
run, eager, captured and replayed, on several streams and contexts (GPU)."""
import ctypes as C
import math
import threading

import numpy as np
import pytest
import torch

import ext_cases as ec
import oracle_lib as ol
from plow_amd import abi, layer, synth


def host_op(oracle, inst, tensors, threads=3):
    assert oracle.plow_oracle_exec(C.byref(inst), ec.table_of(tensors), threads) == 0


# ---- the oracle and the quantizer, on the CPU -----------------------------------------------------

@pytest.mark.parametrize("group,zero,f16", [(32, False, False), (64, True, False), (128, True, True), (32, False, True)])
def test_quantizer_round_trip(group, zero, f16):
    """Every weight comes back within half a step of its group's scale (and the scale's own rounding)."""
    w = torch.randn(24, 512, generator=ec.gen(group)) * 0.05
    w[3, :group] = 0
    w[4] = w[4].abs() + 0.1            # a group on one side of zero keeps its zero point in range
    q, s, z = synth.quant_int4_group(w, group, zero, f16)
    assert q.shape == (24, 256) and s.shape == (24, 512 // group) and (z is not None) == zero
    back = ec.dequant64(q, s, z)
    step = s.double().repeat_interleave(group, 1)
    # rounding the scale moves the ends of the range by up to 15 * 2^-9 of a step, rounding the zero point by half a step
    assert ((back - w.double()).abs() <= step * (1.06 if zero else 0.55) + 1e-12).all()
    assert (back[3, :group] == 0).all()


@pytest.mark.parametrize("M,N,K,G,zero,scale", [(1, 5, 64, 32, False, "bf16"), (3, 17, 256, 64, True, "f16"), (2, 9, 384, 128, True, "bf16")])
def test_oracle_products_against_torch(oracle, M, N, K, G, zero, scale):
    g = ec.gen(M + N)
    a, b = ec.weights(g, (), N, K, G, zero, scale, 0.03), ec.weights(g, (), N, K, G, zero, scale, 0.03)
    x = torch.randn(M, K + 8, generator=g).to(torch.bfloat16)
    f32 = torch.zeros(M, N + 2)
    host_op(oracle, abi.inst(abi.OP_X_GEMM_W4, t=[0, 1, 2, 3, 4 if zero else None],
                             i=[M, N, K, ec.group_field(G, scale), K + 8, N + 2, 1]), [f32, x, *a])
    gt, up = (x[:, :K].double() @ ec.dequant64(*w).T for w in (a, b))
    assert ((f32[:, :N].double() - gt).abs() <= ec.EPS_F32 * gt.abs() + 1e-12).all() and (f32[:, N:] == 0).all()
    out = torch.zeros(M, N, dtype=torch.bfloat16)
    host_op(oracle, abi.inst(abi.OP_X_GEMM_GLU_W4, t=[0, 1, 2, 3, 4 if zero else None, 5, 6, 7 if zero else None],
                             i=[M, N, K, ec.group_field(G, scale), K + 8, 1]), [out, x, *a, *b])
    want = ec.silu64(gt) * up
    assert ((out.double() - want).abs() <= 1.01 * ec.HALF_BF16 * want.abs() + 1e-7).all()


def test_oracle_logprob_against_torch(oracle):
    T, V, A = 5, 300, 7
    x = torch.randn(T, V, generator=ec.gen(1)) * 3
    x[1] = -math.inf
    x[2, 7], x[3, 9] = math.nan, math.inf
    x[4, 10:50] = 2.5
    ids = torch.randint(0, V, (T, 3), generator=ec.gen(2), dtype=torch.int32)
    ids[0, 0], ids[4, 1] = -1, V + 3
    mask = torch.randint(-2 ** 31, 2 ** 31, (T, 10), generator=ec.gen(3), dtype=torch.int64).to(torch.int32)
    for m in (None, mask):
        for dt in (torch.float32, torch.bfloat16):
            xs = x.to(dt)
            o = {"logprob": torch.zeros(T, 3), "entropy": torch.zeros(T), "lse": torch.zeros(T),
                 "alt_ids": torch.zeros(T, A, dtype=torch.int32), "alt_logprob": torch.zeros(T, A)}
            host_op(oracle, abi.inst(abi.OP_X_LOGPROB, t=[0, 1, 2, 3, 4, 5, 6, None if m is None else 7],
                                     i=[T, V, 3, A, 0, 1 if dt == torch.float32 else 0], f=[1.25]),
                    [o["logprob"], xs, ids, o["entropy"], o["alt_ids"], o["alt_logprob"], o["lse"], m])
            want = ec.logprob64(xs, V, ids, A, 1.25, m)
            assert torch.equal(o["alt_ids"], want["alt_ids"])
            for k in ("logprob", "entropy", "lse", "alt_logprob"):
                assert torch.allclose(o[k].double(), want[k], rtol=2 ** -23, atol=1e-6, equal_nan=True), k


def test_plans_of_int4_layers_and_heads():
    """The emitter's wiring: zero-point table and group field on the expert ops, int4 dense shared expert, head chain."""
    cfg = layer.MoeConfig("p", H=256, E=8, I=128, k=2, T=4, enc="int4g", arm="a16dec", group=64, zero_points=True,
                          scale_f16=True, n_shared=2, shared_mode="dense", emit_align=False)
    p = layer.plan_layer(cfg)
    ops = [d.op for d in p.insts]
    assert ops == [180, 83, 48, 49, abi.OP_X_GEMM_GLU_W4, abi.OP_X_GEMM_W4, 87]
    glu, down = p.insts[2], p.insts[3]
    assert glu.i[6] == down.i[6] == abi.ENC_INT4G and glu.i[7] == down.i[7] == 64 | abi.W4_SCALE_F16
    assert glu.t[5] == down.t[5] == p.slots["ztab"] and p.specs["Ws_down"].shape == (256, 128)
    assert p.specs["Ws_up_scale"].dtype == "f16" and p.specs["Ws_up_zero"].shape == (256, 4)
    p = layer.plan_layer(layer.MoeConfig("p", H=256, E=8, I=128, k=2, T=4, enc="int4g", arm="a16"))
    glu, down = p.insts[p.index("glu")], p.insts[p.index("down")]
    assert (glu.op, glu.i[3], glu.i[6], glu.i[7], glu.t[6]) == (85, 16, 128, 0, abi.TENSOR_NONE)
    assert (down.op, down.i[3], down.i[6], down.t[5]) == (86, 16, 128, abi.TENSOR_NONE)
    h = layer.plan_head(layer.HeadConfig("h", T=3, H=256, V=1000, enc="int4g", n_alt=5, masked=True))
    assert [d.op for d in h.insts] == [1, abi.OP_X_GEMM_W4, abi.OP_X_LOGPROB] and h.insts[1].i[6] == 1
    assert layer.plan_head(layer.HeadConfig("h", T=3, H=256, V=1000)).insts[1].op == 180
    assert layer.config("c7", 4).arm == "a16dec" and layer.config("c7", 64).arm == "a16"


# ---- layers and heads on the GPU ------------------------------------------------------------------

@pytest.fixture(scope="module")
def moe():
    from plow_amd.lib import Moe
    m = Moe(0)
    yield m
    m.close()


LAYERS = [  # T, arm, group, zero, f16, shared
    (1, "a16dec", 32, False, False, "fold"), (1, "a16", 128, True, False, "dense"), (7, "a16dec", 64, True, True, "dense"),
    (24, "a16", 32, False, True, "fold"), (60, "a16dec", 128, False, False, None), (150, "a16", 64, True, False, "dense"),
    (400, "a16", 128, False, False, "fold")]


@pytest.mark.gpu
@pytest.mark.parametrize("T,arm,group,zero,f16,shared", LAYERS)
def test_layer_against_the_oracle(moe, oracle, T, arm, group, zero, f16, shared):
    from gpu_harness import assert_output_close, assert_routing_equal, both
    print(f"[case] int4 layer T={T} {arm} g{group} zero={zero} f16={f16} {shared}", flush=True)
    cfg = layer.MoeConfig("int4", H=512, E=12, I=256, k=3, T=T, scoring="sigmoid", norm_topk=True, bias=True, enc="int4g",
                          arm=arm, group=group, zero_points=zero, scale_f16=f16, n_shared=2 if shared == "dense" else 1 if shared else 0,
                          shared_mode=shared, residual=T % 2 == 0)
    plan, dev, host = both(moe, oracle, cfg, seed=T)
    assert_routing_equal(plan, dev, host)
    assert_output_close(dev.np("out"), host.np("out"))
    # the products are f32 sums rounded once: far closer than the layer tolerance
    a, b = ol.bf2f(dev.np("out")).astype(np.float64), ol.bf2f(host.np("out")).astype(np.float64)
    assert np.linalg.norm(a - b) <= 2.0 ** -8 * np.linalg.norm(b)


HEADS = [(1, 1003, "int4g", False, 20, False), (5, 4096, "bf16", False, 3, True), (33, 777, "int4g", True, 64, True), (70, 5000, "int4g", False, 0, False)]


@pytest.mark.gpu
@pytest.mark.parametrize("T,V,enc,zero,A,masked", HEADS)
def test_head_against_the_oracle(moe, oracle, T, V, enc, zero, A, masked):
    print(f"[case] head T={T} V={V} {enc} A={A} masked={masked}", flush=True)
    cfg = layer.HeadConfig("head", T=T, H=512, V=V, enc=enc, group=64, zero_points=zero, n_given=2, n_alt=A, masked=masked, scale=0.8)
    plan = layer.plan_head(cfg)
    dev = synth.bind_head(plan, "cuda", seed=T)
    host = synth.to_host(dev)
    moe.exec_many(plan.insts, dev.table())
    torch.cuda.synchronize()
    # the log probabilities from the logits the device made: the norm's row differs by bf16 steps between the two
    host.t["logits"] = dev.t["logits"].cpu()
    host._table = None
    inst = plan.insts[plan.index("logprob")]
    assert oracle.plow_oracle_exec(C.byref(inst), host.table(), 4) == 0
    for name in ("logprob", "entropy", "lse", "alt_logprob"):
        if name in plan.specs:
            assert torch.allclose(dev.t[name].cpu(), host.t[name], rtol=1e-6, atol=2e-5), name
    if A:
        assert torch.equal(dev.t["alt_tokens"].cpu(), host.t["alt_tokens"])
    want = dev.t["xn"].cpu().double() @ (ec.dequant64(host.t["Wh"], host.t["Wh_scale"], host.t.get("Wh_zero")) if enc == "int4g"
                                         else host.t["Wh"].double()).T
    assert (dev.t["logits"].cpu().double() - want).norm() <= 2e-6 * want.norm()


def layer_and_head(T, arm="a16dec", V=2003, seed=1):
    """One run: an int4 layer with a dense int4 shared expert, and the head behind its output."""
    lc = layer.MoeConfig("l", H=512, E=12, I=256, k=3, T=T, scoring="sigmoid", norm_topk=True, bias=True, enc="int4g", arm=arm,
                         group=64, zero_points=True, n_shared=2, shared_mode="dense", residual=True)
    hc = layer.HeadConfig("h", T=T, H=512, V=V, enc="int4g", group=64, n_alt=8, masked=False)
    lp, hp = layer.plan_layer(lc), layer.plan_head(hc)
    lb, hb = synth.bind(lp, "cuda", seed=seed), synth.bind_head(hp, "cuda", seed=seed)
    hb.t["x"] = lb.t["out"]
    base = len(lp.slots)
    tab = (C.c_void_p * (base + len(hp.slots)))()
    for b, off in ((lb, 0), (hb, base)):
        for n, v in enumerate(b.table()):
            tab[off + n] = v
    insts = list(lp.insts)
    for d in hp.insts:
        d = abi.PlowDevInst.from_buffer_copy(d)
        for j in range(8):
            if d.t[j] != abi.TENSOR_NONE:
                d.t[j] += base
        insts.append(d)
    return lb, hb, abi.inst_array(insts), tab


OUT = ("logprob", "entropy", "lse", "alt_tokens", "alt_logprob")


@pytest.mark.gpu
@pytest.mark.parametrize("T,arm", [(1, "a16dec"), (6, "a16dec"), (40, "a16"), (200, "a16")])
def test_layer_and_head_in_one_run_captured_and_replayed(moe, T, arm):
    """Two graphs of two batches over one context, replayed in turn with eager runs and other work in between: every
    replay equals the eager result bit for bit, and the run equals its ops one at a time."""
    print(f"[case] layer + head T={T} {arm}", flush=True)
    runs = [layer_and_head(T, arm, seed=s) for s in (1, 2)]
    st = torch.cuda.current_stream().cuda_stream
    graphs = []
    for lb, hb, insts, tab in runs:
        moe.exec_many(insts, tab, st)
        torch.cuda.synchronize()
        whole = {n: hb.t[n].clone() for n in OUT}
        for d in insts:
            moe.exec(d, tab, st)
        torch.cuda.synchronize()
        for n in OUT:
            assert torch.equal(whole[n], hb.t[n]), n
        side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.stream(side):
            g.capture_begin()
            moe.exec_many(insts, tab, side.cuda_stream)
            g.capture_end()
        torch.cuda.synchronize()
        graphs.append(g)
    for n in range(3):
        for (lb, hb, insts, tab), g in zip(runs, graphs):
            lb.t["x"].copy_(synth.randn_bf16(tuple(lb.t["x"].shape), 1.0, "cuda", 900 + n))
            moe.exec_many(insts, tab, st)
            torch.cuda.synchronize()
            want = {k: hb.t[k].clone() for k in OUT}
            for k in OUT:
                hb.t[k].zero_()
            torch.randn(1 << 16, device="cuda").sum()
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            for k in OUT:
                assert torch.equal(hb.t[k], want[k]), (n, k)
            assert torch.isfinite(want["logprob"]).all() and (want["alt_tokens"] >= 0).all()


@pytest.mark.gpu
def test_contexts_on_streams_of_their_own():
    """Two contexts driven from two threads on two streams at once give what each gives alone."""
    from plow_amd.lib import Moe
    moes = [Moe(0), Moe(0)]
    runs = [layer_and_head(5, "a16dec", seed=3), layer_and_head(48, "a16", seed=4)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    want = []
    for m, (lb, hb, insts, tab) in zip(moes, runs):
        m.exec_many(insts, tab)
        torch.cuda.synchronize()
        want.append({k: hb.t[k].clone() for k in OUT})
        for k in OUT:
            hb.t[k].zero_()
    torch.cuda.synchronize()

    def work(i):
        for _ in range(20):
            moes[i].exec_many(runs[i][2], runs[i][3], streams[i].cuda_stream)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(2):
        for k in OUT:
            assert torch.equal(runs[i][1].t[k], want[i][k]), (i, k)
    for m in moes:
        m.close()


@pytest.mark.gpu
def test_segment_entry_points(moe):
    """The prefill and decode segment entry points take int4 pairs."""
    for arm, fn in (("a16dec", moe.dec), ("a16", moe.pf)):
        cfg = layer.MoeConfig("s", H=256, E=8, I=128, k=2, T=9, enc="int4g", arm=arm, group=32, zero_points=True)
        plan = layer.plan_layer(cfg)
        a, b = synth.bind(plan, "cuda", seed=5), synth.bind(plan, "cuda", seed=5)
        moe.exec_many(plan.insts, a.table())
        assert fn(plan.insts, b.table(), cfg.T) == 0
        torch.cuda.synchronize()
        assert torch.equal(a.t["out"], b.t["out"]) and bool((a.t["out"] != 0).any())
