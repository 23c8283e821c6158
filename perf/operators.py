"""The operators of models whose weights are 4-bit integers with group scales, and of the answer's log
probabilities, as measurable cases: what each one's inputs are, its plain form in elementary torch
operations, the framework's call, and its definition in 64 bits.

Weights: ``W`` u8 [N][K / 2], low nibble = even k; ``S`` bf16 or f16 [N][K / G], one scale for G neighbouring
k of a row; ``Z`` u8 [N][K / G] with values 0..15, or none (8 everywhere). The weight is (q - z) * s.

  product   out[m][n] = sum_k x[m][k] * w[n][k], bf16 or f32
  glu       out[m][n] = bf16(silu(sum_k x wg) * sum_k x wu)
  experts   the routed experts of one layer on given routing tables: GLU, down, gated sum over a token's
            slots, either slot by slot (decode) or on rows gathered by expert (prefill)
  logprob   per row of logits: log probabilities of given tokens, entropy, log of the sum of exponentials and
            the most likely tokens with their log probabilities; a bit mask may forbid tokens
"""
import math

import torch

own = False

GROUP_F16 = 0x10000          # field of the descriptors: group size, this bit: the scales are f16
UNUSED = -1                  # routing slot of a padded row / token id that asks for nothing (0xFFFFFFFF)


# ---- cases -----------------------------------------------------------------------------------------

def _product(name, M, N, K, G, zero=False, scale="bf16", out="bf16"):
    return {"name": name, "op": "product", "M": M, "N": N, "K": K, "G": G, "zero": zero, "scale": scale, "out": out}


def _glu(name, M, N, K, G, zero=False, scale="bf16"):
    return {"name": name, "op": "glu", "M": M, "N": N, "K": K, "G": G, "zero": zero, "scale": scale}


def _experts(name, T, H, I, E, k, G, form, zero=False, scale="bf16", pad=0):
    return {"name": name, "op": "experts", "T": T, "H": H, "I": I, "E": E, "k": k, "G": G, "form": form, "zero": zero,
            "scale": scale, "pad": pad}


def _logprob(name, T, V, n, A, dtype, mask=False, scale=1.0, extra=0):
    return {"name": name, "op": "logprob", "T": T, "V": V, "n": n, "A": A, "dtype": dtype, "mask": mask, "scale": scale,
            "extra": extra}


def listed():
    return [
        # one token through the down projection of the small layer's shared expert: latency counts
        _product("product-1-small", 1, 2048, 2816, 128),
        # a decode batch through a narrow projection, groups of 32 with zero points
        _product("product-16-g32-zero", 16, 7168, 2048, 32, zero=True),
        # the head of a model at one token: every row of an odd-sized vocabulary, f32 logits
        _product("product-1-head", 1, 120001, 4096, 64, scale="f16", out="f32"),
        # a prompt of 2048 tokens through one projection
        _product("product-2048", 2048, 4096, 7168, 128),
        # gate and up of the shared expert at one token
        _glu("glu-1-g32", 1, 2048, 7168, 32),
        # the same op of the small layer for an odd batch, with zero points
        _glu("glu-61-zero", 61, 2816, 2048, 128, zero=True),
        # one token through eight of 384 experts
        _experts("experts-1", 1, 7168, 2048, 384, 8, 32, "slots"),
        # a decode batch of 64 rows, the last three of them padding
        _experts("experts-64-pad", 64, 4096, 1536, 128, 8, 128, "slots", zero=True, pad=3),
        # a prompt through the small layer's experts
        _experts("experts-512-gathered", 512, 2048, 1408, 64, 6, 128, "gathered"),
        # one sampled token: its log probability and twenty alternatives
        _logprob("logprob-1", 1, 120001, 1, 20, "f32"),
        # a decode batch under a grammar's mask, with a temperature
        _logprob("logprob-64-mask", 64, 32000, 1, 5, "bf16", mask=True, scale=1.25),
        # scoring a prompt of 2048 tokens
        _logprob("logprob-2048", 2048, 120001, 1, 0, "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["product", "glu", "experts", "logprob"])
    G = rng.choice([32, 64, 128])
    zero, scale = rng.random() < 0.5, rng.choice(["bf16", "f16"])
    if op in ("product", "glu"):
        while True:
            M, K = _log(rng, 1, 2048), G * max(1, _log(rng, 256, 7168) // G)
            N = _log(rng, 64, 120001) if op == "product" else _log(rng, 64, 4096)
            if M * N * K <= 2048 * 4096 * 7168 // 2 and N * K <= 120001 * 4096 and M * N <= 64 << 20:
                break
        if op == "glu":
            c = _glu("", M, N, K, G, zero, scale)
        else:
            c = _product("", M, N, K, G, zero, scale, rng.choice(["bf16", "f32"]))
    elif op == "experts":
        while True:
            T, E, k = _log(rng, 1, 512), _log(rng, 8, 256), rng.randint(1, 8)
            H, I = 128 * max(1, _log(rng, 512, 7168) // 128), G * max(1, _log(rng, 256, 2048) // G)
            if E * H * I <= 128 * 4096 * 1536 and T * E * H * I <= 512 * 64 * 2048 * 1408:
                break
        form = rng.choice(["slots", "gathered"])
        c = _experts("", T, H, I, E, k, G, form, zero, scale, rng.randint(0, T // 4) if form == "slots" else 0)
    else:
        while True:
            T, V = _log(rng, 1, 2048), _log(rng, 1000, 150000)
            A = rng.choice([0, 0, 1, 5, 20, rng.randint(2, 64)])
            if T * V <= (48 << 20 if A else 2048 * 120001):
                break
        c = _logprob("", T, V, rng.choice([0, 1, 1, rng.randint(2, 5)]), A, rng.choice(["f32", "bf16"]), rng.random() < 0.4,
                     rng.choice([1.0, round(rng.uniform(0.5, 2.0), 3)]), rng.choice([0, 0, rng.randint(1, 64)]))
    c.pop("name")
    return c


# ---- inputs ----------------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _nibbles(g, shape):
    """Random bytes of two nibbles each, more of them near the middle than at the ends (quantized weights)."""
    a = torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.uint8)
    b = torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.uint8)
    return (a & b) + (((a ^ b) & 0xEE) >> 1)


def _weights(g, c, lead, N, K):
    s = (torch.rand(*lead, N, K // c["G"], generator=g, device="cuda") + 0.5) * 0.006
    z = torch.randint(5, 12, (*lead, N, K // c["G"]), generator=g, device="cuda", dtype=torch.uint8) if c["zero"] else None
    return {"W": _nibbles(g, (*lead, N, K // 2)), "S": s.to(torch.bfloat16 if c["scale"] == "bf16" else torch.float16), "Z": z}


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda").to(torch.bfloat16)


def _pointers(*tensors):
    """[E][3] table of the experts' parts of three tensors."""
    rows = [[t.data_ptr() + e * t[0].numel() * t.element_size() for t in tensors] for e in range(tensors[0].shape[0])]
    return torch.tensor(rows, dtype=torch.int64, device="cuda")


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = {"case": c}
    if c["op"] in ("product", "glu"):
        s["x"] = _randn(g, c["M"], c["K"])
        s["w"] = _weights(g, c, (), c["N"], c["K"])
        if c["op"] == "glu":
            s["w2"] = _weights(g, c, (), c["N"], c["K"])
        s["out"] = torch.zeros(c["M"], c["N"], device="cuda",
                               dtype=torch.float32 if c.get("out") == "f32" else torch.bfloat16)
    elif c["op"] == "experts":
        T, H, I, E, k = c["T"], c["H"], c["I"], c["E"], c["k"]
        s["x"] = _randn(g, T, H)
        s["gate"], s["up"], s["down"] = (_weights(g, c, (E,), n, kk) for n, kk in ((I, H), (I, H), (H, I)))
        eid = torch.rand(T, E, generator=g, device="cuda").topk(k, dim=1).indices.to(torch.int32)
        if c["pad"]:
            eid[T - c["pad"]:] = UNUSED
        gates = torch.rand(T, k, generator=g, device="cuda") + 0.1
        gates /= gates.sum(1, keepdim=True)
        s["table"] = torch.stack([eid, gates.view(torch.int32)], dim=2).reshape(T * k, 2).contiguous()
        ws = (s["gate"], s["up"], s["down"])
        s["wtab"], s["stab"] = _pointers(*(w["W"] for w in ws)), _pointers(*(w["S"] for w in ws))
        s["ztab"] = _pointers(*(w["Z"] for w in ws)) if c["zero"] else None
        rows = T * k if c["form"] == "slots" else T * k + 63 * E
        s["fu"] = torch.zeros(rows, I, device="cuda", dtype=torch.bfloat16)
        s["part"] = torch.zeros(T * k, H, device="cuda")
        s["out"] = torch.zeros(T, H, device="cuda", dtype=torch.bfloat16)
        if c["form"] == "gathered":
            s["meta"] = torch.zeros(3 * E + 1, device="cuda", dtype=torch.int32)
            s["row_token"], s["row_partidx"] = (torch.zeros(rows, device="cuda", dtype=torch.int32) for _ in range(2))
            s["row_gate"] = torch.zeros(rows, device="cuda")
    else:
        T, V, n, A = c["T"], c["V"], c["n"], c["A"]
        # a heavy head and a long tail, as a model's logits have
        x = torch.randn(T, V + c["extra"], generator=g, device="cuda") * 2.5
        x[:, : max(1, V // 500)] += torch.rand(T, 1, generator=g, device="cuda") * 8
        s["logits"] = x.to(torch.bfloat16 if c["dtype"] == "bf16" else torch.float32)
        s["ids"] = torch.randint(0, V, (T, n), generator=g, device="cuda", dtype=torch.int32)
        s["mask"] = None
        if c["mask"]:
            words = (V + 31) // 32
            s["mask"] = torch.randint(-2 ** 31, 2 ** 31, (T, words), generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
            s["mask"][T // 2] = 0 if T > 4 else -1          # a row that allows nothing
        f32 = {"device": "cuda", "dtype": torch.float32}
        s["logprob"], s["entropy"], s["lse"] = torch.zeros(T, n, **f32), torch.zeros(T, **f32), torch.zeros(T, **f32)
        s["alt_ids"], s["alt_logprob"] = torch.zeros(T, A, device="cuda", dtype=torch.int32), torch.zeros(T, A, **f32)
    return s


# ---- one pass --------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state)
    if op == "product":
        return _round(state["x"].float() @ _plain_weight(state["w"]).T, state["out"].dtype)
    if op == "glu":
        x = state["x"].float()
        return _round(_silu(x @ _plain_weight(state["w"]).T) * (x @ _plain_weight(state["w2"]).T), torch.bfloat16)
    return _plain_experts(state) if op == "experts" else _plain_logprob(state)


def _round(v, dtype):
    return v.to(dtype)


def _silu(v):
    return v / (1.0 + torch.exp(-v))


def _plain_weight(w, pick=None):
    """(q - z) * s in 32 bits of all rows, or of the experts `pick`."""
    W, S, Z = ((None if t is None else t if pick is None else t[pick]) for t in (w["W"], w["S"], w["Z"]))
    G = 2 * W.shape[-1] // S.shape[-1]
    q = torch.stack([W & 15, W >> 4], dim=-1).reshape(*S.shape, G).float()
    q = (q - (8.0 if Z is None else Z.float().unsqueeze(-1))) * S.float().unsqueeze(-1)
    return q.reshape(*W.shape[:-1], 2 * W.shape[-1])


def _plain_experts(s):
    c = s["case"]
    T, H, I, E, k = c["T"], c["H"], c["I"], c["E"], c["k"]
    eid = s["table"][:, 0].long()
    gates = s["table"][:, 1].contiguous().view(torch.float32)
    live = (eid >= 0).unsqueeze(1)
    at = eid.clamp(min=0)
    tok = torch.arange(T * k, device="cuda") // k
    x = s["x"].float()
    if T * k <= E // 2:   # a few slots: each slot's own expert
        rows = x[tok].unsqueeze(2)
        g = (_plain_weight(s["gate"], at) @ rows).squeeze(2)
        u = (_plain_weight(s["up"], at) @ rows).squeeze(2)
        fu = torch.where(live, _silu(g) * u, 0.0).to(torch.bfloat16)
        y = (_plain_weight(s["down"], at) @ fu.float().unsqueeze(2)).squeeze(2)
    else:                 # many: every expert's product with every token, and the slots' rows of it
        g = (x @ _plain_weight(s["gate"]).reshape(E * I, H).T).reshape(T, E, I)[tok, at]
        u = (x @ _plain_weight(s["up"]).reshape(E * I, H).T).reshape(T, E, I)[tok, at]
        fu = torch.where(live, _silu(g) * u, 0.0).to(torch.bfloat16)
        f = torch.zeros(E, T, I, device="cuda")
        f.index_put_((at, tok), fu.float() * live, accumulate=True)
        y = torch.bmm(f, _plain_weight(s["down"]).transpose(1, 2))[at, tok]
    part = torch.where(live, y * gates.unsqueeze(1), 0.0)
    out = part.reshape(T, k, H).sum(1).to(torch.bfloat16)
    return {"fu": fu, "out": out} if c["form"] == "slots" else {"out": out}


def _allowed(s, V):
    bit = torch.arange(V, device="cuda")
    return ((s["mask"][:, bit // 32] >> (bit % 32)) & 1).bool()


def _plain_logprob(s):
    c = s["case"]
    T, V, A = c["T"], c["V"], c["A"]
    x = s["logits"][:, :V].float()
    if s["mask"] is not None:
        x = torch.where(_allowed(s, V), x, -math.inf)
    m = x.amax(1, keepdim=True)
    base = torch.where(m == -math.inf, 0.0, m)
    d = (x - base) * c["scale"]
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    logz = torch.log(total)
    entropy = torch.where(total > 0, logz - torch.where(e > 0, e * d, 0.0).sum(1, keepdim=True) / total, 0.0)
    # an entry of -inf has no probability, in a row without any other as well
    logp = torch.where(d == -math.inf, -math.inf, d - logz)
    top, ids = (v[:, :A] for v in torch.sort(x, dim=1, descending=True, stable=True)) if A else (x[:, :0], s["alt_ids"][:, :0])
    return {"logprob": logp.gather(1, s["ids"].long()), "entropy": entropy[:, 0], "lse": (base * c["scale"] + logz)[:, 0],
            "alt_ids": torch.where(top == -math.inf, UNUSED, ids).to(torch.int32),
            "alt_logprob": logp.gather(1, ids.long())}


# ---- the framework's calls -------------------------------------------------------------------------

_moe = None


def _calls(s):
    """The descriptors and the handle table of one pass: what a program builds once for its buffers."""
    global _moe
    import ctypes

    from plow_amd import abi
    from plow_amd.lib import Moe
    if _moe is None:
        _moe = Moe(torch.cuda.current_device())
    c, tensors, insts = s["case"], [], []

    def h(t):
        if t is None:
            return None
        tensors.append(t)
        return len(tensors) - 1

    def group():
        return c["G"] | (abi.W4_SCALE_F16 if c["scale"] == "f16" else 0)

    if c["op"] == "product":
        w = s["w"]
        insts.append(abi.inst(abi.OP_X_GEMM_W4, t=[h(s["out"]), h(s["x"]), h(w["W"]), h(w["S"]), h(w["Z"])],
                              i=[c["M"], c["N"], c["K"], group(), 0, 0, 1 if c["out"] == "f32" else 0]))
    elif c["op"] == "glu":
        a, b = s["w"], s["w2"]
        insts.append(abi.inst(abi.OP_X_GEMM_GLU_W4, t=[h(s["out"]), h(s["x"]), h(a["W"]), h(a["S"]), h(a["Z"]),
                                                       h(b["W"]), h(b["S"]), h(b["Z"])],
                              i=[c["M"], c["N"], c["K"], group(), 0, abi.ACT_SILU, 0]))
    elif c["op"] == "experts":
        T, H, I, E, k = c["T"], c["H"], c["I"], c["E"], c["k"]
        out, x, fu, part, table = (h(s[n]) for n in ("out", "x", "fu", "part", "table"))
        wt, st, zt = h(s["wtab"]), h(s["stab"]), h(s["ztab"])
        if c["form"] == "slots":
            insts.append(abi.inst(abi.OP_MOE_GROUP_GLU_FP8_BLK, t=[fu, x, table, wt, st, zt],
                                  i=[T * k, I, H, E, k, abi.ACT_SILU, abi.ENC_INT4G, group()]))
            insts.append(abi.inst(abi.OP_MOE_GROUP_DOWN_FP8_BLK, t=[part, fu, table, wt, st, zt],
                                  i=[T * k, H, I, E, 0, 0, abi.ENC_INT4G, group()]))
        else:
            meta, rt, rp, rg = (h(s[n]) for n in ("meta", "row_token", "row_partidx", "row_gate"))
            insts.append(abi.inst(abi.OP_MOE_ALIGN_PF, t=[meta, table, rt, rp, rg], i=[T, E, k]))
            insts.append(abi.inst(abi.OP_MOE_GROUP_GLU_PF, t=[fu, x, wt, st, meta, rt, zt],
                                  i=[I, H, E, abi.ENC_INT4G, 0, abi.ACT_SILU, group(), abi.ARM_A16], slots=T * k))
            insts.append(abi.inst(abi.OP_MOE_GROUP_DOWN_PF, t=[part, fu, wt, st, meta, zt, rp, rg],
                                  i=[H, I, E, abi.ENC_INT4G, 0, 0, group(), abi.ARM_A16], slots=T * k))
        insts.append(abi.inst(abi.OP_MOE_COMBINE_PF, t=[out, None, None, part], i=[H, k, T]))
    else:
        T, V, n, A = c["T"], c["V"], c["n"], c["A"]
        alt = A > 0
        insts.append(abi.inst(abi.OP_X_LOGPROB,
                              t=[h(s["logprob"]) if n else None, h(s["logits"]), h(s["ids"]) if n else None, h(s["entropy"]),
                                 h(s["alt_ids"]) if alt else None, h(s["alt_logprob"]) if alt else None, h(s["lse"]),
                                 h(s["mask"])],
                              i=[T, V, n, A, V + c["extra"], abi.LOGPROB_F32 if c["dtype"] == "f32" else 0], f=[c["scale"]]))
    table = (ctypes.c_void_p * len(tensors))(*(t.data_ptr() for t in tensors))
    return abi.inst_array(insts), table


def _own(s):
    if "calls" not in s:
        s["calls"] = _calls(s)
    insts, table = s["calls"]
    _moe.exec_many(insts, table, torch.cuda.current_stream().cuda_stream)
    op = s["case"]["op"]
    if op in ("product", "glu"):
        return s["out"]
    if op == "experts":
        return {n: s[n] for n in (("fu", "out") if s["case"]["form"] == "slots" else ("out",))}
    return {n: s[n] for n in ("logprob", "entropy", "lse", "alt_ids", "alt_logprob")}


# ---- what a pass cannot do without -----------------------------------------------------------------

def _weight_bytes(c, N, K):
    return N * K / 2 + N * (K // c["G"]) * (3 if c["zero"] else 2)


def work(case):
    c = case
    if c["op"] in ("product", "glu"):
        M, N, K = c["M"], c["N"], c["K"]
        mats = 2 if c["op"] == "glu" else 1
        return {"bytes": mats * _weight_bytes(c, N, K) + 2 * M * K + M * N * (4 if c.get("out") == "f32" else 2),
                "flops": 2 * mats * M * N * K}
    if c["op"] == "experts":
        T, H, I, E, k = c["T"] - c["pad"], c["H"], c["I"], c["E"], c["k"]
        hit = E * (1 - (1 - k / E) ** T)   # experts with a row, on average
        fu = 2 * T * k * I if c["form"] == "slots" else 0   # (an output there)
        return {"bytes": hit * (2 * _weight_bytes(c, I, H) + _weight_bytes(c, H, I)) + 4 * T * H + fu + 8 * T * k,
                "flops": 6 * T * k * H * I}
    T, V = c["T"], c["V"]
    return {"bytes": T * V * (4 if c["dtype"] == "f32" else 2) + (T * ((V + 31) // 32) * 4 if c["mask"] else 0) +
            T * (8 * c["n"] + 8 * c["A"] + 8), "flops": 6 * T * V}


# ---- the definitions in 64 bits --------------------------------------------------------------------

def _exact_rows(w, x, lead=None):
    """x [M][K] times the weight's rows: groups of k one after the other, nibbles picked apart by arithmetic."""
    W, S, Z = ((None if t is None else t if lead is None else t[lead]) for t in (w["W"], w["S"], w["Z"]))
    N, K = W.shape[0], 2 * W.shape[1]
    G = K // S.shape[1]
    y = torch.zeros(x.shape[0], N, dtype=torch.float64, device=x.device)
    step = max(1, (1 << 27) // N // G) * G
    for k0 in range(0, K, step):
        k1 = min(K, k0 + step)
        b = W[:, k0 // 2:k1 // 2].long()
        q = torch.empty(N, k1 - k0, dtype=torch.float64, device=x.device)
        q[:, 0::2], q[:, 1::2] = (b % 16).double(), (b // 16).double()
        q -= 8 if Z is None else Z[:, k0 // G:k1 // G].double().repeat_interleave(G, dim=1)
        q *= S[:, k0 // G:k1 // G].double().repeat_interleave(G, dim=1)
        y += x[:, k0:k1].double() @ q.T
    return y


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "product":
        return _exact_rows(s["w"], s["x"])
    if c["op"] == "glu":
        g = _exact_rows(s["w"], s["x"])
        return g * torch.sigmoid(g) * _exact_rows(s["w2"], s["x"])
    if c["op"] == "experts":
        T, H, I, k = c["T"], c["H"], c["I"], c["k"]
        tab = s["table"].cpu()
        eid, gates = tab[:, 0], tab[:, 1].contiguous().view(torch.float32).double()
        fu = torch.zeros(T * k, I, dtype=torch.float64, device="cuda")
        out = torch.zeros(T, H, dtype=torch.float64, device="cuda")
        for e in sorted(set(eid.tolist()) - {UNUSED}):
            slots = (eid == e).nonzero()[:, 0]
            tok = (slots // k).cuda()
            g = _exact_rows(s["gate"], s["x"][tok], e)
            f = (g * torch.sigmoid(g) * _exact_rows(s["up"], s["x"][tok], e))
            fu[slots.cuda()] = f
            f = f.to(torch.bfloat16)   # the intermediate is a bf16 tensor of its own
            out.index_add_(0, tok, _exact_rows(s["down"], f, e) * gates[slots].cuda().unsqueeze(1))
        return {"fu": fu, "out": out} if c["form"] == "slots" else {"out": out}
    T, V, A = c["T"], c["V"], c["A"]
    got = {"logprob": [], "entropy": [], "lse": [], "alt_logprob": []}
    for r0 in range(0, T, 64):   # a few rows at a time
        x = s["logits"][r0:r0 + 64, :V].double() * c["scale"]
        if s["mask"] is not None:
            words = s["mask"][r0:r0 + 64].cpu().numpy().astype("<i4").view("uint8")
            bits = torch.from_numpy(__import__("numpy").unpackbits(words, axis=1, bitorder="little")[:, :V]).bool().cuda()
            x = x.masked_fill(~bits, -math.inf)
        none = (x == -math.inf).all(1)
        lse = torch.logsumexp(x, 1)
        logp = torch.where(x == -math.inf, x, x - lse.unsqueeze(1))
        p = torch.exp(logp)
        got["logprob"].append(logp.gather(1, s["ids"][r0:r0 + 64].long()))
        got["entropy"].append(torch.where(none, 0.0, -torch.special.xlogy(p, p).sum(1)))
        got["lse"].append(lse)
        got["alt_logprob"].append(logp.topk(A, dim=1).values)
    return {**{n: torch.cat(v) for n, v in got.items()}, "alt_ids": None}
