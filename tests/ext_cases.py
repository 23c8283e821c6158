"""Inputs, 64-bit references and descriptors of the int4 group-scale products and the log-probability op, for the
GPU tests and (refusals) the CPU ones."""
import ctypes as C
import math

import torch

from plow_amd import abi

EPS_F32 = 2.0 ** -24
HALF_BF16 = torch.finfo(torch.bfloat16).eps / 2      # 2^-8: half a step relative to the value


def gen(seed, device="cpu"):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    return g


def weights(g, lead, N, K, G, zero, scale, std=0.006):
    """(W, S, Z): packed nibbles, scales, zero points (None: 8)."""
    W = torch.randint(0, 256, (*lead, N, K // 2), generator=g, dtype=torch.uint8)
    S = ((torch.rand(*lead, N, K // G, generator=g) + 0.5) * std).to(torch.float16 if scale == "f16" else torch.bfloat16)
    Z = torch.randint(0, 16, (*lead, N, K // G), generator=g, dtype=torch.uint8) if zero else None
    return W, S, Z


def dequant64(W, S, Z):
    G = 2 * W.shape[-1] // S.shape[-1]
    q = torch.stack([W & 15, W >> 4], -1).flatten(-2).double()
    z = torch.full_like(q, 8.0) if Z is None else Z.double().repeat_interleave(G, -1)
    return (q - z) * S.double().repeat_interleave(G, -1)


def abs_bound(x, W, S, Z):
    """Bound of |computed - exact| of one f32 sum: the kernels add q + 16 and take 16 + z off again, both at most 31
    in size, so at most 2 * 31 * s * |x| per k passes through the sum; a sum of n terms in any order is off by at
    most n * 2^-24 of the sum of their sizes, and the group sums are scaled and added on top (K / G roundings more;
    n = 2 K covers both)."""
    G = 2 * W.shape[-1] // S.shape[-1]
    K = 2 * W.shape[-1]
    s = S.double().abs().repeat_interleave(G, -1)
    return 2 * K * EPS_F32 * 62.0 * (x.double().abs() @ s.T)


def group_field(G, scale):
    return G | (abi.W4_SCALE_F16 if scale == "f16" else 0)


def table_of(tensors):
    t = (C.c_void_p * max(1, len(tensors)))()
    for n, a in enumerate(tensors):
        t[n] = None if a is None else a.data_ptr()
    return t


def silu64(v):
    return v * torch.sigmoid(v)


def act64(g, u, act, f0=0.0, f1=0.0):
    if act == 0:
        return 0.5 * g * (1 + torch.tanh(0.7978845608028654 * (g + 0.044715 * g ** 3))) * u
    if act == 1:
        return silu64(g) * u
    if act == 2:
        return f0 * torch.tanh(g / f0) * torch.sigmoid(g) * (f1 * torch.tanh(u / f1) if f1 > 0 else u)
    if act == 3:
        g, u = g.clamp(max=f1), u.clamp(-f1, f1)
        return g * torch.sigmoid(f0 * g) * (u + 1)
    return silu64(g.clamp(max=f1)) * u.clamp(-f1, f1)


def logprob64(x, V, ids, A, scale=1.0, mask=None):
    """x [T][>= V] -> dict of f64 results (alternatives by stable order of the values as stored)."""
    x = x[:, :V].double()
    if mask is not None:
        bit = torch.arange(V)
        ok = ((mask[:, bit // 32].long() >> (bit % 32)) & 1).bool()
        x = torch.where(ok, x, -math.inf)
    T = x.shape[0]
    bad = torch.isnan(x).any(1) | (x == math.inf).any(1)
    # relative to the maximum: beside values of 1e38 even 64 bits lose the logarithm of the sum
    m = x.max(1, keepdim=True).values
    y = (x - torch.where(torch.isinf(m), 0.0, m)) * scale
    logz = torch.logsumexp(y, 1, keepdim=True)
    lse = (torch.where(torch.isinf(m), 0.0, m) * scale + logz)[:, 0]
    lse[bad] = math.nan
    logp = torch.where(x == -math.inf, -math.inf, y - logz)
    p = logp.exp()
    ent = -(torch.special.xlogy(p, p)).sum(1)
    ent[(x == -math.inf).all(1)] = 0.0
    logp[bad] = math.nan
    ent[bad] = math.nan
    key = torch.nan_to_num(x, nan=math.inf, posinf=1e300, neginf=-math.inf)
    order = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :A]
    top = x.gather(1, order)
    alt_ids, alt = order.to(torch.int32), logp.gather(1, order)
    alt_ids[top == -math.inf] = -1
    if A > V:
        alt_ids = torch.cat([alt_ids, torch.full((T, A - V), -1, dtype=torch.int32)], 1)
        alt = torch.cat([alt, torch.where(bad, math.nan, -math.inf)[:, None].expand(T, A - V).double()], 1)
    lp = torch.zeros(ids.shape, dtype=torch.float64)
    if ids.numel():
        i = ids.long() & 0xFFFFFFFF
        lp = logp.gather(1, i.clamp(max=V - 1))
        lp[i >= V] = math.nan
        lp[i == 0xFFFFFFFF] = 0.0
    return {"logprob": lp, "entropy": ent, "lse": lse, "alt_ids": alt_ids, "alt_logprob": alt}
