"""Channels-last GroupNorm of many groups: past 64 the statistics are finished by a kernel of their own, which the normalise
pass then reads; slabs of the on-chip forms hold up to 128 groups.  Bounds: test_gpu_groupnorm_channels_last.py."""
import pytest

from kernel_names import kernel_names
from test_gpu_groupnorm_channels_last import _check, _make

pytestmark = pytest.mark.gpu

# (shape, groups): read twice, with sums finished apart
PASSES = [
    ((1, 60000, 130), 65), ((2, 30000, 96), 96), ((1, 40000, 128), 128), ((3, 9001, 640), 320), ((1, 20000, 320), 320),
    ((1, 5000, 4096), 4096), ((2, 3001, 2560), 1280), ((1, 3000, 5001), 1667), ((5, 801, 2310), 770), ((1, 40001, 131), 131),
    ((160, 900, 264), 88), ((1, 2999, 4098), 4098),
]
# on the chip, slabs of many groups, of a number of them that only divides as a whole, and one past the most
ON_CHIP = [
    ((2, 30, 97), 97), ((1, 40, 127), 127), ((1, 40, 131), 131), ((1, 12, 904), 113), ((1, 900, 904), 113), ((2, 1100, 640), 320), ((3, 5, 4096), 4096),
    ((1, 1, 300), 100), ((1, 2, 256), 256), ((1, 4000, 512), 128), ((2, 64, 1024), 512), ((1, 700, 5000), 2500),
]


def _dtype(name):
    import torch
    return {"bf16": torch.bfloat16, "f32": torch.float32}[name]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("shape,groups", PASSES + ON_CHIP)
def test_shapes(gpu, dtype, shape, groups):
    import torch
    be, ops = gpu
    x, w, b = _make(shape, _dtype(dtype), sum(shape))
    got = be.group_norm_channels_last(x, groups, w, b, 1e-6)
    _check(got, x, groups, w, b, 1e-6, None)
    for kind in (ops.SILU, ops.GELU_TANH):
        out = be.group_norm_channels_last(x, groups, w, b, 1e-6, activation=kind)
        _check(out, x, groups, w, b, 1e-6, kind)
    assert torch.equal(be.group_norm_channels_last(x, groups, w, b, 1e-6, activation=ops.GELU_TANH, out=x), out)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("shape,groups", PASSES + ON_CHIP)
def test_exact_sums(gpu, dtype, shape, groups):
    """Integers up to 8: every sum is exact, so one element missing or counted twice shows in the mean."""
    import torch
    be, ops = gpu
    x = torch.randint(-8, 9, shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(sum(shape))).to(_dtype(dtype))
    _, w, b = _make(shape[-1:], torch.float32, 1)
    _check(be.group_norm_channels_last(x, groups, w, b, 1e-6), x, groups, w, b, 1e-6, None, exact_sums=True)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("shape,groups", PASSES)
def test_kernels(gpu, dtype, shape, groups):
    """The shapes above do run the three kernels."""
    be, ops = gpu
    x, w, b = _make(shape, _dtype(dtype), 1)
    names = kernel_names(lambda: be.group_norm_channels_last(x, groups, w, b, 1e-6))
    assert len(names) == 3 and sum("gcl_finalize" in n for n in names) == 1, names


def test_bad_values_and_graphs(gpu):
    """An infinity or a NaN spoils its own group only; two graphs side by side, each with sums and statistics of its own."""
    import torch
    be, ops = gpu
    data = [(_make((2, 20001, 320), torch.bfloat16, 1), 160), (_make((1, 9000, 1024), torch.float32, 2), 512)]
    want, graphs, outs = [], [], []
    for (x, w, b), groups in data:
        clean = be.group_norm_channels_last(x, groups, w, b, 1e-6, activation=ops.SILU)
        x[0, 77, 5], x[-1, 8000, -1] = float("inf"), float("nan")
        y = be.group_norm_channels_last(x, groups, w, b, 1e-6, activation=ops.SILU)
        bad = torch.zeros_like(y, dtype=torch.bool)
        bad[0, :, 4:6], bad[-1, :, -2:] = True, True
        assert torch.equal(y[~bad], clean[~bad]) and torch.isnan(y[bad]).all()
        want.append(torch.nan_to_num(y.float()))
    torch.cuda.synchronize()
    for (x, w, b), groups in data:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(be.group_norm_channels_last(x, groups, w, b, 1e-6, activation=ops.SILU))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in data]
    for _ in range(6):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(torch.nan_to_num(y.float()), z) for y, z in zip(outs, want))
