"""The 4-bit linear under tensor scales whose product leaves F32's normal range, as two operands of ordinary F32 values can bring
them.  The bound is that of the linear elsewhere (products summed in F32, an instruction's terms off by up to 2^-22 of the sum of
magnitudes; three roundings for the scales and the result), plus a step of 2^-149 where results themselves are that small."""
import numpy as np
import pytest

import fp4_reference as ref

pytestmark = pytest.mark.gpu


def _operand(be, ops, rows, k, seed, scale):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((rows, k), device="cuda", generator=g) * scale
    return be.fp4_quantize(x, ops.NVFP4, be.fp4_tensor_scale(x))


def _values(q):
    return ref.values(q.codes.cpu().numpy(), q.scales.cpu().numpy(), q.format, q.rows, q.k, q.tensor_scale.item())


@pytest.mark.parametrize("m", [3, 130, 3000])           # the last one on pairs of SMs
@pytest.mark.parametrize("scale_a,scale_b", [(1e-18, 1e-18), (1e-10, 1e-27), (1e-27, 1e-10), (3e-21, 1e-17), (1e18, 1e18), (1e15, 1e22), (1e-20, 1e20), (1e20, 1e-20)])
def test_values(gpu, m, scale_a, scale_b):
    import torch
    be, ops = gpu
    n, k = 4000, 320
    a, b = _operand(be, ops, m, k, 1, scale_a), _operand(be, ops, n, k, 2, scale_b)
    got = be.fp4_linear(a, b, dtype=torch.float32).double().cpu().numpy()
    va, vb = _values(a), _values(b)
    want, mass = va @ vb.T, np.abs(va) @ np.abs(vb).T
    bound = (k // 64 + 2) * 2.0 ** -22 * mass + 4 * 2.0 ** -24 * np.abs(want) + 2.0 ** -149
    largest = float(np.finfo(np.float32).max)       # rounding to F32 makes what lies past it infinite
    finite, infinite = np.abs(want) + bound <= largest, np.abs(want) - bound > largest
    assert (np.abs(got - want) <= bound)[finite].all(), float((np.abs(got - want) / bound)[finite].max())
    assert finite.mean() > 0.5 and (got[infinite] == np.sign(want[infinite]) * np.inf).all()


@pytest.mark.parametrize("m", [2, 200, 5000])
def test_large_sums_of_small_products(gpu, m):
    """Every element is the largest of its format: sums of k 2688^2 under scales whose product is 2^-152, exact in F32."""
    import torch
    be, ops = gpu
    n, k, g = 5000, 4096, 2.0 ** -76
    scale = torch.tensor([g], device="cuda")
    a = be.fp4_quantize(torch.full((m, k), 2688.0 * g, device="cuda"), ops.NVFP4, scale)
    b = be.fp4_quantize(torch.full((n, k), 2688.0 * g, device="cuda"), ops.NVFP4, scale)
    got = be.fp4_linear(a, b, torch.zeros(n, device="cuda"), dtype=torch.float32)
    want = k * 2688.0 ** 2 * g * g
    assert abs(want) > 1.2e-38 and ((got.double() - want).abs() <= (k // 64 + 2) * 2.0 ** -22 * want).all()


@pytest.mark.parametrize("m", [4, 180, 5000])
def test_large_scales(gpu, m):
    """Scales whose product overflows: rows of zeros give zeros (and the bias), small rows finite values, large ones infinities."""
    import torch
    be, ops = gpu
    n, k = 5000, 256
    x, w = torch.zeros((m, k), device="cuda"), torch.zeros((n, k), device="cuda")
    x[1, 7], x[2] = 4.0e18, 1.0e24                 # the smallest values that these scales hold, and large ones
    w[:] = 3.0e18
    w[0], w[1] = 0.0, 2.0e23
    scale = torch.tensor([4.0e20], device="cuda")
    a, b = be.fp4_quantize(x, ops.NVFP4, scale), be.fp4_quantize(w, ops.NVFP4, scale)
    bias = torch.full((n,), 1.5, device="cuda")
    va, vb = _values(a), _values(b)
    want = torch.from_numpy(va @ vb.T).cuda() + 1.5
    got = be.fp4_linear(a, b, bias, dtype=torch.float32)
    assert not torch.isnan(got).any()
    huge = want.abs() > 3.4e38
    assert huge.any() and (want[1] > 1e36).any() and torch.equal(torch.isinf(got), huge)
    assert ((got.double() - want).abs()[~huge] <= 2.0 ** -18 * want.abs()[~huge]).all()
    assert (got[0] == 1.5).all() and (got[:, 0] == 1.5).all()


def test_scales_of_zero(gpu):
    import torch
    be, ops = gpu
    a, b = _operand(be, ops, 5, 64, 1, 1.0), _operand(be, ops, 40, 64, 2, 1.0)
    for ga, gb in ((0.0, 3.0e38), (3.0e38, 0.0), (0.0, 0.0)):
        a.tensor_scale, b.tensor_scale = torch.tensor([ga], device="cuda"), torch.tensor([gb], device="cuda")
        assert (be.fp4_linear(a, b, dtype=torch.float32) == 0).all()
