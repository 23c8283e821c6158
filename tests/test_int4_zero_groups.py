"""Groups of int4 weights that are all zero, and groups so small that a 16-bit scale hardly holds them: the quantizer on
the CPU, the products on the GPU."""
import pytest
import torch

import ext_cases as ec
from plow_amd import abi, synth


@pytest.mark.parametrize("zero", [False, True])
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("size", [1e-9, 3e-8, 3e-7, 6e-7, 2e-6, 1e-4, 1.0, 1e5])
def test_quantizer_at_the_ends_of_the_scales_range(size, f16, zero):
    """Codes are real codes and every weight comes back within half a step, also where the scale is subnormal; a scale
    of normal size moves the ends of the range by its own rounding as well (7.5 or 15 steps times 2^-8 at most)."""
    w = torch.randn(16, 256, generator=ec.gen(3)) * size
    w[2, :64] = 0
    q, s, z = synth.quant_int4_group(w, 64, zero, f16)
    assert torch.isfinite(s.float()).all() and (s.float() >= 0).all()
    back = ec.dequant64(q, s, z)
    step = s.double().repeat_interleave(64, 1)
    assert torch.isfinite(back).all()
    assert ((back - w.double()).abs() <= step * (1.06 if zero else 0.55)).all(), ((back - w.double()).abs() / step).max()
    assert (back[2, :64] == 0).all() and (s[2, 0] == 0), "a group of zeros needs no scale"
    # no step is coarser than the group needs, but for the scale type's own step (f16: 2^-24)
    need = w.view(16, 4, 64).double()
    need = (need.amax(2).clamp(min=0) - need.amin(2).clamp(max=0)) / 15 if zero else need.abs().amax(2) / 7
    assert (s.double() <= need * (1 + 2.0 ** -8) + (2.0 ** -24 if f16 else 0.0)).all()


def test_quantizer_refuses_what_no_scale_holds():
    w = torch.zeros(2, 64)
    w[1, 5] = 7 * 66000.0
    synth.quant_int4_group(w, 32)                       # (bf16 reaches further)
    with pytest.raises(ValueError):
        synth.quant_int4_group(w, 32, scale_f16=True)
    for bad in (float("inf"), float("nan")):
        w[1, 5] = bad
        for zero in (False, True):
            with pytest.raises(ValueError):
                synth.quant_int4_group(w, 32, zero)


@pytest.mark.gpu
@pytest.mark.parametrize("zero", [False, True])
@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("M", [1, 5, 24, 40, 130])
def test_rows_of_zeros_give_zeros(M, G, zero):
    """Quantized rows without a weight in them: their outputs are exactly 0 in every kernel form."""
    from plow_amd.lib import Moe
    print(f"[case] zero rows M={M} G={G} zero={zero}", flush=True)
    moe = Moe(0)
    N, K = 260, 1024
    w = torch.randn(N, K, generator=ec.gen(G)) * 0.02
    w[::3] = 0
    q, s, z = synth.quant_int4_group(w, G, zero)
    x = torch.randn(M, K, generator=ec.gen(M)).to(torch.bfloat16)
    o = torch.full((M, N), 7.0, device="cuda")
    keep = [o, x.cuda(), q.cuda(), s.cuda(), None if z is None else z.cuda()]
    moe.exec(abi.inst(abi.OP_X_GEMM_W4, t=[0, 1, 2, 3, 4 if zero else None], i=[M, N, K, G, 0, 0, 1]), ec.table_of(keep))
    torch.cuda.synchronize()
    got = o.cpu()
    assert (got[:, ::3] == 0).all(), got[:, ::3].abs().max()
    want = x.double() @ ec.dequant64(q, s, z).T
    assert ((got.double() - want).abs() <= ec.abs_bound(x, q, s, z) + ec.EPS_F32 * want.abs()).all()
    moe.close()


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 5, 24, 40, 130])
def test_codes_at_the_zero_point_with_a_large_scale(M):
    """Foreign weights may give a group of zeros any scale: what the sum of 16 + q leaves behind is then scaled up and
    stays within the bound that the contract states."""
    from plow_amd.lib import Moe
    moe = Moe(0)
    N, K, G = 130, 512, 64
    g = ec.gen(M)
    q, s, z = ec.weights(g, (), N, K, G, True, "bf16")
    s[:, 2], z[:, 2] = 64.0, 11
    q[:, G: G + G // 2] = 0xBB
    x = torch.randn(M, K, generator=g).to(torch.bfloat16)
    o = torch.zeros(M, N, device="cuda")
    moe.exec(abi.inst(abi.OP_X_GEMM_W4, t=[0, 1, 2, 3, 4], i=[M, N, K, G, 0, 0, 1]),
             ec.table_of([o, x.cuda(), q.cuda(), s.cuda(), z.cuda()]))
    torch.cuda.synchronize()
    want = x.double() @ ec.dequant64(q, s, z).T
    assert ((o.cpu().double() - want).abs() <= ec.abs_bound(x, q, s, z) + ec.EPS_F32 * want.abs()).all()
    moe.close()
