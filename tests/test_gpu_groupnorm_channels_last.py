"""Channels-last GroupNorm (+ activation) on the GPU against 64 bits.

Bound.  With z = (x - mean) / std * gamma: the difference, the product with rsqrt(var) * gamma (itself two roundings) and
the final multiply-add are half an F32 step each, the F32 mean is half a step of |mean|, and the variance comes from F32
sums of at most 32 terms next to an anchor of the data's own size, each relative 32 * 2^-24 of a second moment that is at
most a few times the variance: below 128 * 2^-24 |z| altogether.  The mean comes from F32 sums too, and where x lies next to
it nothing scales its error down: a run of n <= 32 terms d = x - K adds to within n 2^-24 sum |d| (one rounding for each
difference, n - 1 for partial sums that are no larger than sum |d|), so the mean is off by at most 32 * 2^-24 times the mean
|d|.  In units of the group's standard deviation mean |x - mean| <= 1, and the anchors, n_r elements weighing on one of
them, have mean |K - mean| <= sqrt(sum n_r (K_r - mean)^2 / N) <= sqrt(32): 32 (1 + sqrt(32)) < 214 steps of gamma.  That
term falls away for small integers, whose sums are exact (|d| <= 16, s2 <= 32 * 256 < 2^24); test_exact_sums asks for the
bound without it.  Activations have slopes below 1.2 and are evaluated to
2^-20 of their argument; the result is rounded once."""
import numpy as np
import pytest

import fp4_reference as ref

pytestmark = pytest.mark.gpu


def _make(shape, dtype, seed, affine=True, offset=0.5):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = shape[-1]
    x = torch.randn(shape, device="cuda", generator=g) * (0.5 + torch.rand((c,), device="cuda", generator=g)) + offset * torch.randn((c,), device="cuda", generator=g)
    w = torch.randn((c,), device="cuda", generator=g) * 0.2 + 1 if affine else None
    b = torch.randn((c,), device="cuda", generator=g) * 0.3 if affine else None
    return x.to(dtype), w, b


def _check(got, x, groups, w, b, eps, kind, exact_sums=False):
    import torch
    v = x.double().flatten(1, -2).unflatten(2, (groups, -1))
    var, mean = torch.var_mean(v, dim=(1, 3), correction=0, keepdim=True)
    inv = 1.0 / torch.sqrt(var + eps)
    gamma = 1.0 if w is None else w.double()
    z = ((v - mean) * inv).flatten(2) * gamma
    y = z + (0.0 if b is None else b.double())
    offset = (mean * inv).expand_as(v).flatten(2).abs() * (1.0 if w is None else gamma.abs())
    bound = 2.0 ** -24 * (128 * z.abs() + 2 * offset + 2 * y.abs())
    if not exact_sums:
        bound = bound + 2.0 ** -24 * 214 * (1.0 if w is None else gamma.abs())
    if kind is not None:
        bound = 1.2 * bound + 2.0 ** -20 * y.abs()
    want = torch.from_numpy(ref.activation(y.cpu().numpy(), kind)).cuda()
    half = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -24
    error = (got.double().reshape(want.shape) - want).abs()
    over = error > bound + half * (want.abs() + bound) + 1e-30
    assert not over.any(), f"{int(over.sum())} of {over.numel()}, worst {float((error / (bound + half * want.abs() + 1e-30)).max()):.3g} times the bound"


SHAPES = [
    # (shape, groups)
    ((1, 1, 1), 1), ((2, 1, 64), 32), ((1, 2, 8), 8), ((3, 7, 3), 3), ((2, 33, 6), 2), ((1, 1, 320), 32), ((1, 5, 24), 4),
    ((1, 256, 512), 32), ((2, 16, 16, 128), 32), ((3, 1035, 320), 32), ((1, 3, 20, 30, 96), 8), ((2, 500, 36), 12), ((1, 700, 7), 1),
    ((1, 4000, 50), 5), ((5, 64, 64), 1), ((2, 9, 2560), 32), ((1, 40, 4096), 2), ((1, 33, 4112), 16), ((1, 17, 2050), 2),
    # rows that are no whole vectors, folded, with and without a rest
    ((1, 200003, 1), 1), ((1, 60001, 3), 1), ((1, 60001, 3), 3), ((1, 50001, 10), 1), ((1, 50000, 10), 5), ((1, 33333, 30), 10),
    ((2, 40000, 5), 1), ((2, 40001, 5), 5), ((3, 20001, 12), 4), ((1, 9001, 100), 25), ((1, 5003, 402), 6), ((1, 3001, 2001), 3),
    ((1, 60000, 64), 8), ((1, 30000, 100), 4), ((4, 3000, 40), 8), ((1, 24960, 128), 32), ((300, 5, 16), 4),
]


# maps of a few MB, which L2 keeps between the passes: full and ragged last rows, slabs of several groups and of one, several entries
MIDDLE = [
    ((1, 4097, 512), 32), ((1, 24960, 512), 32), ((1, 26624, 256), 16), ((1, 26625, 256), 16), ((2, 1100, 320), 32), ((1, 9216, 320), 32),
    ((1, 1500, 2048), 16), ((1, 12000, 32), 1), ((3, 6000, 128), 8), ((1, 5001, 96), 2), ((1, 9999, 192), 6), ((2, 5300, 64), 1),
    # groups of an even number of channels that is no multiple of a vector's, small to large
    ((3, 1035, 320), 32), ((8, 1035, 320), 32), ((2, 4099, 320), 32), ((2, 1030, 640), 32), ((1, 30001, 96), 16), ((1, 50001, 30), 15), ((1, 40001, 24), 4),
]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_shapes(gpu, dtype, shape, groups):
    import torch
    be, ops = gpu
    x, w, b = _make(shape, {"bf16": torch.bfloat16, "f32": torch.float32}[dtype], sum(shape))
    _check(be.group_norm_channels_last(x, groups, w, b, 1e-6), x, groups, w, b, 1e-6, None)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("shape,groups", SHAPES + MIDDLE)
def test_exact_sums(gpu, dtype, shape, groups):
    """Integers up to 8: every sum is exact, so one element missing or counted twice shows in the mean."""
    import torch
    be, ops = gpu
    g = torch.Generator(device="cuda").manual_seed(sum(shape))
    x = torch.randint(-8, 9, shape, device="cuda", generator=g).to({"bf16": torch.bfloat16, "f32": torch.float32}[dtype])
    _, w, b = _make(shape[-1:], torch.float32, 1)
    _check(be.group_norm_channels_last(x, groups, w, b, 1e-6), x, groups, w, b, 1e-6, None, exact_sums=True)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kind", [None, 0, 2, 4])
@pytest.mark.parametrize("shape,groups", MIDDLE)
def test_middle_shapes(gpu, dtype, kind, shape, groups):
    import torch
    be, ops = gpu
    x, w, b = _make(shape, {"bf16": torch.bfloat16, "f32": torch.float32}[dtype], sum(shape))
    out = be.group_norm_channels_last(x, groups, w, b, 1e-6, activation=kind)
    _check(out, x, groups, w, b, 1e-6, kind)
    again = be.group_norm_channels_last(x, groups, w, b, 1e-6, activation=kind, out=x)   # in place, and the same bits
    assert again.data_ptr() == x.data_ptr() and torch.equal(again, out)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kind", [None, 0, 1, 2, 3, 4])
@pytest.mark.parametrize("shape,groups", [((2, 100, 96), 8), ((1, 8200, 256), 32), ((1, 41, 21), 7)])
@pytest.mark.parametrize("affine", [True, False])
def test_activations(gpu, dtype, kind, shape, groups, affine):
    import torch
    be, ops = gpu
    x, w, b = _make(shape, {"bf16": torch.bfloat16, "f32": torch.float32}[dtype], 5, affine)
    _check(be.group_norm_channels_last(x, groups, w, b, 1e-5, activation=kind), x, groups, w, b, 1e-5, kind)
    if affine:   # parameters in bf16 are used as stored
        w, b = w.bfloat16(), b.bfloat16()
        _check(be.group_norm_channels_last(x, groups, w, b, 1e-5, activation=kind), x, groups, w, b, 1e-5, kind)


@pytest.mark.parametrize("offset", [40.0, 1000.0])
@pytest.mark.parametrize("shape", [(2, 300, 64), (1, 20000, 64)])
def test_large_common_offset(gpu, offset, shape):
    import torch
    be, ops = gpu
    x, w, b = _make(shape, torch.float32, 3, offset=0.1)
    x = x + offset
    _check(be.group_norm_channels_last(x, 8, w, b, 1e-6), x, 8, w, b, 1e-6, None)


def test_matches_the_channels_first_operator(gpu):
    """The permuted vrb_group_norm: same statistics to F32 rounding, so bf16 results differ by at most one rounding."""
    import torch
    be, ops = gpu
    x, w, b = _make((2, 9, 10, 128), torch.bfloat16, 1)
    got = be.group_norm_channels_last(x, 32, w, b, 1e-6)
    first = be.group_norm(x.permute(0, 3, 1, 2).contiguous(), 32, w.bfloat16(), b.bfloat16(), 1e-6).permute(0, 2, 3, 1)
    wb = be.group_norm_channels_last(x, 32, w.bfloat16(), b.bfloat16(), 1e-6)
    step = 2.0 ** -7 * first.float().abs()
    assert ((wb.float() - first.float()).abs() <= step + 1e-6).all()
    assert got.shape == x.shape


def test_constant_groups_and_bad_values(gpu):
    """A group without variance gives the bias; an infinity or a NaN spoils its own group only."""
    import torch
    be, ops = gpu
    for shape in ((2, 50, 64), (1, 40000, 64)):
        x, w, b = _make(shape, torch.float32, 4)
        x[..., :8] = 3.0
        clean = be.group_norm_channels_last(x, 8, w, b, 1e-6)
        assert torch.equal(clean[..., :8], b[:8].expand_as(clean[..., :8]))
        x[0, 7, 20] = float("nan")
        x[0, 30, 41] = float("inf")
        y = be.group_norm_channels_last(x, 8, w, b, 1e-6)
        bad = torch.zeros_like(y, dtype=torch.bool)
        bad[0, :, 16:24] = True
        bad[0, :, 40:48] = True
        assert torch.equal(y[~bad], clean[~bad])
        assert torch.isnan(y[0, :, 16:24]).all() and torch.isnan(y[0, :, 40:48]).all()


def test_unaligned_and_in_place(gpu):
    import torch
    be, ops = gpu
    for dtype in (torch.bfloat16, torch.float32):
        x, w, b = _make((2, 333, 64), dtype, 6)
        want = be.group_norm_channels_last(x, 8, w, b, 1e-6)
        shifted = torch.empty(x.numel() + 1, device="cuda", dtype=dtype)[1:].view(x.shape)
        shifted.copy_(x)
        _check(be.group_norm_channels_last(shifted, 8, w, b, 1e-6), x, 8, w, b, 1e-6, None)
        y = x.clone()
        assert torch.equal(be.group_norm_channels_last(y, 8, w, b, 1e-6, out=y), want)
        big = torch.randn((1, 50000, 64), device="cuda").to(dtype)
        want = be.group_norm_channels_last(big, 8, w, b, 1e-6)
        assert torch.equal(be.group_norm_channels_last(big, 8, w, b, 1e-6, out=big), want)


def test_repeats_captures_and_streams(gpu):
    """Bit-identical repeats; two graphs with scratch of their own, replayed at once on two streams."""
    import torch
    be, ops = gpu
    shapes = [(1, 300, 128), (2, 30000, 64), (1, 260, 512)]
    data = [_make(s, torch.bfloat16, i) for i, s in enumerate(shapes)]

    def step(i, x=None):
        return be.group_norm_channels_last(data[i][0] if x is None else x, 32, data[i][1], data[i][2], 1e-6, activation=ops.SILU)
    want = [step(i) for i in range(3)]
    for _ in range(3):
        assert all(torch.equal(step(i), want[i]) for i in range(3))
    torch.cuda.synchronize()
    graphs, outs, statics = [], [], []
    for i in range(3):
        static = torch.zeros_like(data[i][0])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(i, static))
        graphs.append(graph)
        statics.append(static)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for i in range(3):
        statics[i].copy_(data[i][0])
    torch.cuda.synchronize()
    for _ in range(5):
        for i in range(3):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(outs[i], want[i]) for i in range(3))


def test_middle_maps_bad_values_and_alignment(gpu):
    """An infinity or a NaN spoils its own group only; a map off the 16-byte boundaries takes another way to the same bound."""
    import torch
    be, ops = gpu
    for dtype in (torch.bfloat16, torch.float32):
        x, w, b = _make((1, 4100, 512), dtype, 8)
        clean = be.group_norm_channels_last(x, 32, w, b, 1e-6, activation=ops.SILU)
        shifted = torch.empty(x.numel() + 1, device="cuda", dtype=dtype)[1:].view(x.shape)
        shifted.copy_(x)
        _check(be.group_norm_channels_last(shifted, 32, w, b, 1e-6, activation=ops.SILU), x, 32, w, b, 1e-6, ops.SILU)
        x[0, 4099, 33] = float("nan")
        x[0, 5, 500] = float("inf")
        y = be.group_norm_channels_last(x, 32, w, b, 1e-6, activation=ops.SILU)
        bad = torch.zeros_like(y, dtype=torch.bool)
        bad[0, :, 32:48] = True
        bad[0, :, 496:512] = True
        assert torch.equal(y[~bad], clean[~bad]) and torch.isnan(y[bad]).all()


def test_middle_maps_together(gpu):
    """Clusters that each want a whole SM, from four streams at once, eager and replayed."""
    import torch
    be, ops = gpu
    shapes = [((1, 4096, 512), 32), ((4, 4096, 128), 8), ((1, 16000, 512), 32), ((8, 1035, 320), 8)]
    data = [_make(s, torch.bfloat16, 20 + i) for i, (s, _) in enumerate(shapes)]
    want = [be.group_norm_channels_last(x, g, w, b, 1e-6) for (x, w, b), (_, g) in zip(data, shapes)]
    graphs, outs = [], []
    for (x, w, b), (_, g) in zip(data, shapes):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(be.group_norm_channels_last(x, g, w, b, 1e-6))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in shapes]
    torch.cuda.synchronize()
    eager = []
    for _ in range(10):
        for i, ((x, w, b), (_, g)) in enumerate(zip(data, shapes)):
            with torch.cuda.stream(streams[i]):
                eager.append((i, be.group_norm_channels_last(x, g, w, b, 1e-6)))
                graphs[i].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i, y in eager) and all(torch.equal(y, z) for y, z in zip(outs, want))


def test_first_call_of_a_process_is_captured(gpu):
    """No call of the library before the capture: room for clusters and shared memory are asked for while capturing."""
    import os
    import subprocess
    import sys
    code = """
import torch
from vrhino_b200 import ops
be = ops.B200Backend()
x = torch.randn((1, 5000, 512), device="cuda").bfloat16()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = be.group_norm_channels_last(x, 32, None, None, 1e-6, activation=0)
graph.replay()
torch.cuda.synchronize()
assert torch.equal(y, be.group_norm_channels_last(x, 32, None, None, 1e-6, activation=0))
print("captured")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=root, timeout=120)
    assert done.returncode == 0 and "captured" in done.stdout, done.stderr[-2000:]


def test_past_32_bit_offsets(gpu):
    import torch
    be, ops = gpu
    s, c = (1 << 31) // 64 + 777, 64
    x = torch.randn((1, s, c), device="cuda", dtype=torch.bfloat16)
    y = be.group_norm_channels_last(x, 8, None, None, 1e-6, activation=ops.SILU)
    v = x[0].view(s, 8, 8)
    mean = v.sum(dim=(0, 2), dtype=torch.float64) / (s * 8)
    second = sum(part.double().square().sum(dim=(0, 2)) for part in v.split(1 << 22)) / (s * 8)
    inv = 1.0 / torch.sqrt(second - mean ** 2 + 1e-6)
    for rows in (slice(0, 5), slice(s - 5, s), slice(s // 2, s // 2 + 5)):
        z = (v[rows].double() - mean[:, None]) * inv[:, None]
        want = (z / (1.0 + torch.exp(-z))).flatten(1)
        assert ((y[0, rows].double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5).all()


def test_leaves_what_lies_behind_and_refuses(gpu):
    import torch
    be, ops = gpu
    x, w, b = _make((1, 50, 64), torch.bfloat16, 1)
    buffer = torch.full((3, 50, 64), 7.0, device="cuda", dtype=torch.bfloat16)
    be.group_norm_channels_last(x, 8, w, b, 1e-6, out=buffer[1:2])
    assert (buffer[0] == 7.0).all() and (buffer[2] == 7.0).all()
    assert be.group_norm_channels_last(x[:, :0], 8, w, b, 1e-6).shape == (1, 0, 64)
    for bad in (lambda: be.group_norm_channels_last(x, 7, w, b, 1e-6), lambda: be.group_norm_channels_last(x, 0, w, b, 1e-6),
                lambda: be.group_norm_channels_last(x[0, 0], 8, w, b, 1e-6)):
        with pytest.raises(ops.VrbError, match="shape/groups mismatch"):
            bad()
    with pytest.raises(ops.VrbError, match="weight mismatch"):
        be.group_norm_channels_last(x, 8, w[:8].contiguous(), b, 1e-6)
    with pytest.raises(ops.VrbError, match="unknown activation"):
        be.group_norm_channels_last(x, 8, w, b, 1e-6, activation=9)
    with pytest.raises(ops.VrbError, match="contiguous"):
        be.group_norm_channels_last(x.transpose(1, 2), 10, None, None, 1e-6)
