"""SiLU and GELU-tanh of the channels-last GroupNorm and the 4-bit linear, at arguments that are known exactly: a product of zeros
plus an F32 bias, and a group without variance, both give the bias itself.

With w the sigmoid's argument (y for SiLU, 2 sqrt(2 / pi) (y + 0.044715 y^3) for GELU-tanh) the value is y sigmoid(w).  Bounds
relative to the VALUE (a bound relative to the argument would hide any error of a large negative one):
  F32 results   the exponential is off by at most 2 ulp = 2^-22, its product with y, the sum 1 + e and the quotient by half a step
                (2^-24) each: below 2^-21.  GELU-tanh's w takes four more roundings or rounded constants, 2^-22 |w| altogether, and
                an error of the exponent is a relative error of the exponential.  An exponential below 2^-126 lies in steps of
                2^-149 and may be off by two of them, 2^-148, times |y| < 128 (|w| < 104 where it is not 0, and |y| <= |w|):
                2^-141, and half a step for the product: below 2^-140 absolute.
  bf16 results  rounded once, 2^-8; before that |w| is off by 2^-23 (SiLU: constant and product) or 2^-22 |w|, the exponential,
                the shared reciprocal and six operations add at most 2^-20.  A sigmoid below 2^-126 may count as zero: |y| 2^-126 is
                below 2^-119 there, GELU-tanh's y being smaller than SiLU's.
Arguments below -2^60 and infinities: the sigmoid is 0, so y sigmoid(w) is -0, and for -infinity it is infinity times 0, a NaN, as
the framework's other activations give."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

SILU, GELU_TANH = 0, 2


def _arguments():
    rng = np.random.default_rng(4)
    magnitudes = np.concatenate([np.logspace(-38, 38, 700), rng.uniform(0.0, 12.0, 900), rng.uniform(0.0, 130.0, 900),
                                 [0.0, 1.0, 5.0, 43.0, 44.0, 63.0, 64.0, 87.0, 88.0, 89.0, 103.0, 104.0, 3.4e38, np.inf]])
    y = np.concatenate([magnitudes, -magnitudes, [np.nan]]).astype(np.float32)
    rng.shuffle(y)                      # neighbours of every kind: two values share a reciprocal
    return y[:len(y) // 256 * 256]


def _want(y, kind):
    """(value, |w|) in 64 bits; e^-|w| keeps the quotient finite."""
    y = y.astype(np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        w = y if kind == SILU else 2.0 * np.sqrt(2.0 / np.pi) * (y + 0.044715 * y ** 3)
        e = np.exp(-np.abs(w))
        value = np.where(w < 0, y * e, y) / (1.0 + e)
    return value, np.abs(w)


def _check(got, y, kind):
    import torch
    want, w = _want(y, kind)
    value = got.double().cpu().numpy().reshape(-1, len(y))
    assert (np.isnan(value) == np.isnan(want)).all()
    infinite = np.isinf(want)
    with np.errstate(invalid="ignore"):
        if got.dtype == torch.float32:
            bound = (2.0 ** -21 + (0.0 if kind == SILU else 2.0 ** -22) * np.minimum(w, 200.0)) * np.abs(want) + 2.0 ** -140
        else:
            before = (2.0 ** -20 + 2.0 ** -22 * np.minimum(w, 200.0)) * np.abs(want)
            bound = before + 2.0 ** -8 * (np.abs(want) + before) + 2.0 ** -119
            infinite = infinite | (np.abs(want) > 3.38e38)      # past bf16's largest value
        over = (np.abs(value - want) > bound) & ~np.isnan(want) & ~infinite
    assert (value[:, np.isinf(want)] == want[np.isinf(want)]).all()
    assert not over.any(), f"{over.any(axis=0).sum()} of {len(y)} arguments, y = {y[over.any(axis=0)][:8]}, got {value[0][over.any(axis=0)][:8]}, want {want[over.any(axis=0)][:8]}"


@pytest.mark.parametrize("kind", [SILU, GELU_TANH])
@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("m", [1, 40, 9000])        # the last one on pairs of SMs
@pytest.mark.parametrize("cut", [0, 3])             # a width off the 16-byte boundaries too
def test_linear(gpu, kind, out, m, cut):
    import torch
    be, ops = gpu
    y = _arguments()
    y = y[:len(y) - cut]
    a = be.fp4_quantize(torch.zeros((m, 64), device="cuda"), ops.MXFP4)
    w = be.fp4_quantize(torch.zeros((len(y), 64), device="cuda"), ops.MXFP4)
    _check(be.fp4_linear(a, w, torch.from_numpy(y).cuda(), kind, dtype={"bf16": torch.bfloat16, "f32": torch.float32}[out]), y, kind)


@pytest.mark.parametrize("kind", [SILU, GELU_TANH])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("spatial,cut", [(3, 0), (40, 0), (600, 0), (9000, 0), (5, 1), (700, 1), (700, 2), (700, 4)])
def test_group_norm(gpu, kind, dtype, spatial, cut):
    """A constant map has no variance: what is left is the bias.  cut: widths that take shorter vectors."""
    import torch
    be, ops = gpu
    y = _arguments()
    y = y[:len(y) - cut]
    c = len(y)
    x = torch.full((1, spatial, c), 2.0, device="cuda", dtype={"bf16": torch.bfloat16, "f32": torch.float32}[dtype])
    groups = max(g for g in range(1, 33) if c % g == 0)
    _check(be.group_norm_channels_last(x, groups, None, torch.from_numpy(y).cuda(), 1e-6, activation=kind), y, kind)
