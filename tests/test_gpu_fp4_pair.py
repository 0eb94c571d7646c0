"""The 4-bit linear's kernel on pairs of SMs, which takes the large products: several stages, ring turns, ragged ends, all
epilogues.  Every shape is checked to reach that kernel, so that another choice of kernels cannot drop the coverage unseen.

Bound, as for the linear elsewhere: an instruction sums 64 products and adds them to the accumulator, a term of it off by up to
2^-23 of the sum of magnitudes, so |error| <= (ceil(k / 64) + 2) 2^-22 sum |a b|, then half a step each for the scales, the bias
and the result, two roundings for the scales' product and its own.  Activations: slope below 1.2, evaluated to 2^-20 of their
argument (test_gpu_gated_activations.py holds them to their value)."""
import numpy as np
import pytest

import fp4_reference as ref
from kernel_names import kernel_names

pytestmark = pytest.mark.gpu

HALF = {"bf16": 2.0 ** -8, "f32": 2.0 ** -24}
# stages of 256 elements of k in a ring of 5, steps of 64; tiles of 256 x 256
SHAPES = [
    (4100, 1000, 4099),    # four stages, the last one ragged; no row of the result on a 16-byte boundary
    (4100, 2600, 4104),    # two turns of the ring and a stage of one step
    (4609, 300, 4360),     # two stages, the second of 44 elements
    (9000, 64, 2000),      # one step
    (2049, 1344, 8200),    # a last stage of one whole step, tiles of one row
]


def _dtype(name):
    import torch
    return {"bf16": torch.bfloat16, "f32": torch.float32}[name]


def _data(rows, k, seed, scale=1.0):
    import torch
    return torch.randn((rows, k), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)) * scale


def _packed(be, ops, x, fmt):
    return be.fp4_quantize(x, fmt, be.fp4_tensor_scale(x) if fmt == ops.NVFP4 else None)


def _values(q):
    import torch
    v = ref.values(q.codes.cpu().numpy(), q.scales.cpu().numpy(), q.format, q.rows, q.k, None if q.tensor_scale is None else q.tensor_scale.item())
    return torch.from_numpy(v).cuda()


def _reached(be, a, b, *args, **kwargs):
    names = kernel_names(lambda: be.fp4_linear(a, b, *args, **kwargs))
    assert len(names) == 1 and "fp4_linear_pair_kernel" in names[0], names


def _activation(y, kind):
    import torch
    if kind == 0:
        return y / (1.0 + torch.exp(-y))
    if kind == 1:
        return 0.5 * y * torch.special.erfc(-y / 2.0 ** 0.5)
    if kind == 2:
        return 0.5 * y * (1.0 + torch.tanh((2.0 / np.pi) ** 0.5 * (y + 0.044715 * y ** 3)))
    return torch.tanh(y) if kind == 3 else y.clamp(min=0.0)


def _check(got, a, b, bias=None, kind=None):
    import torch
    va, vb = _values(a), _values(b)
    acc, mass = va @ vb.t(), va.abs() @ vb.abs().t()
    y = acc if bias is None else acc + bias.double()
    bound = (-(-a.k // 64) + 2) * 2.0 ** -22 * mass + 3 * 2.0 ** -24 * acc.abs() + 2.0 ** -24 * y.abs()
    want = y
    if kind is not None:
        want = _activation(y, kind)
        bound = 1.2 * bound + 2.0 ** -20 * y.abs() + 1e-30
    half = HALF["bf16" if got.dtype == torch.bfloat16 else "f32"]
    over = (got.double() - want).abs() > bound + half * (want.abs() + bound) + 1e-40
    assert not over.any(), f"{int(over.sum())} of {over.numel()}, first at {over.nonzero()[0].tolist()}"


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_shapes(gpu, fmt, out, m, k, n):
    be, ops = gpu
    a, b = _packed(be, ops, _data(m, k, 1, 2.0), fmt), _packed(be, ops, _data(n, k, 2, 0.05), fmt)
    _reached(be, a, b, dtype=_dtype(out))
    _check(be.fp4_linear(a, b, dtype=_dtype(out)), a, b)


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_exact_products(gpu, fmt, m, k, n):
    """Elements of the format itself under a scale of 1: products are multiples of 1/4 and sums stay below 2^17, so all of them are
    exact in F32 and one product missing or counted twice shows."""
    import torch
    be, ops = gpu
    g = torch.Generator(device="cuda").manual_seed(m + k)
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device="cuda")
    x, w = (table[torch.randint(0, 8, (rows, k), device="cuda", generator=g)] * (1 - 2 * torch.randint(0, 2, (rows, k), device="cuda", generator=g)) for rows in (m, n))
    x[:, ::16], w[:, ::16] = 6.0, -6.0       # every block's largest magnitude, so that every scale is 1
    a, b = be.fp4_quantize(x, fmt), be.fp4_quantize(w, fmt)
    assert torch.equal(be.fp4_dequantize(a, torch.float32), x)
    _reached(be, a, b, dtype=torch.float32)
    assert torch.equal(be.fp4_linear(a, b, dtype=torch.float32).double(), x.double() @ w.double().t())


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("kind", [None, 0, 1, 2, 3, 4])
@pytest.mark.parametrize("n", [4099, 4104])
def test_bias_and_activation(gpu, fmt, out, kind, n):
    import torch
    be, ops = gpu
    m, k = 4100, 600
    a, b = _packed(be, ops, _data(m, k, 3, 2.0), fmt), _packed(be, ops, _data(n, k, 4, 0.1), fmt)
    for dtype in (torch.bfloat16, torch.float32):
        bias = _data(1, n, 9)[0].to(dtype)
        _reached(be, a, b, bias, kind, dtype=_dtype(out))
        _check(be.fp4_linear(a, b, bias, kind, dtype=_dtype(out)), a, b, bias, kind)
    if kind is not None:
        _check(be.fp4_linear(a, b, None, kind, dtype=_dtype(out)), a, b, None, kind)


@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("n", [2503, 2504])
def test_result_anywhere(gpu, out, n):
    """A result off the 16-byte boundaries has the bits of one on them, and what lies around it stays as it was."""
    import torch
    be, ops = gpu
    m, k = 2500, 1000
    a, b = _packed(be, ops, _data(m, k, 5), 0), _packed(be, ops, _data(n, k, 6), 0)
    bias = _data(1, n, 7)[0]
    _reached(be, a, b, bias, ops.GELU_TANH, dtype=_dtype(out))
    want = be.fp4_linear(a, b, bias, ops.GELU_TANH, dtype=_dtype(out))
    for shift in (0, 1, 3, 4):
        buffer = torch.full((m * n + 600,), 7.0, device="cuda", dtype=_dtype(out))
        got = be.fp4_linear(a, b, bias, ops.GELU_TANH, dtype=_dtype(out), out=buffer[shift:shift + m * n].view(m, n))
        assert torch.equal(got, want)
        assert (buffer[:shift] == 7.0).all() and (buffer[shift + m * n:] == 7.0).all()


@pytest.mark.parametrize("fmt", [0, 1])
def test_bad_rows_stay_apart(gpu, fmt):
    import torch
    be, ops = gpu
    m, k, n = 4100, 600, 4099
    x, w = _data(m, k, 1), _data(n, k, 2)
    x[m - 1, 577], x[300, 3], w[4097, 300] = float("nan"), float("inf"), float("-inf")
    x[1], w[7] = 0.0, 0.0
    scale = torch.tensor([0.01], device="cuda") if fmt == ops.NVFP4 else None
    a, b = be.fp4_quantize(x, fmt, scale), be.fp4_quantize(w, fmt, scale)
    _reached(be, a, b, dtype=torch.float32)
    y = be.fp4_linear(a, b, dtype=torch.float32)
    bad = torch.zeros((m, n), dtype=torch.bool, device="cuda")
    bad[m - 1], bad[300], bad[:, 4097] = True, True, True
    assert torch.equal(torch.isnan(y), bad)
    assert (y[1][~bad[1]] == 0).all() and (y[:, 7][~bad[:, 7]] == 0).all()


def test_repeats_streams_and_graphs(gpu):
    """Bit-identical repeats, two shapes at once on two streams, eager and replayed, beside split products."""
    import torch
    be, ops = gpu
    jobs = []
    for i, (m, k, n, reaches) in enumerate([(4100, 2600, 4104, True), (2500, 1000, 2503, True), (30, 2048, 3000, False)]):
        a, b = _packed(be, ops, _data(m, k, i), 0), _packed(be, ops, _data(n, k, i + 9), 0)
        if reaches:
            _reached(be, a, b)
        jobs.append((a, b))
    want = [be.fp4_linear(a, b) for a, b in jobs]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for a, b in jobs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(be.fp4_linear(a, b))
        graphs.append(graph)
    streams, got = [torch.cuda.Stream() for _ in jobs], []
    for _ in range(8):
        for i, (a, b) in enumerate(jobs):
            with torch.cuda.stream(streams[i]):
                got.append((i, be.fp4_linear(a, b)))
                graphs[i].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i, y in got) and all(torch.equal(x, y) for x, y in zip(outs, want))


def test_chain_at_size(gpu):
    """A feed-forward at size: normalised rows packed, up with GELU, packed, down into the accumulation, residual epilogue; the bias
    in the product's own epilogue has the bits of the chain's."""
    import torch
    be, ops = gpu
    rows, c, inner = 9000, 1536, 4096
    x = _data(rows, c, 1).bfloat16().view(2, rows // 2, c)
    up, down = _packed(be, ops, _data(inner, c, 2, 0.03), 0), _packed(be, ops, _data(c, inner, 3, 0.03), 0)
    bias_up, bias_down = _data(1, inner, 4, 0.1)[0].bfloat16(), _data(1, c, 5, 0.1)[0].bfloat16()
    h = be.group_norm_channels_last(x, 32, None, None, 1e-6, activation=ops.SILU)
    q = be.fp4_quantize(h, 0, be.fp4_tensor_scale(h))
    _reached(be, q, up, bias_up, ops.GELU_TANH)
    mid = be.fp4_linear(q, up, bias_up, ops.GELU_TANH)
    _check(mid.view(rows, inner), q, up, bias_up, ops.GELU_TANH)
    p = be.fp4_quantize(mid, 0, be.fp4_tensor_scale(mid))
    _reached(be, p, down, dtype=torch.float32)
    acc = be.fp4_linear(p, down, dtype=torch.float32)
    _check(acc.view(rows, c), p, down)
    fused = be.fp4_linear(p, down, bias_down)
    assert torch.equal(fused, ops.linear_output(be, acc, bias_down))
    got = ops.linear_output_gated_residual(be, ops.Policy(), x, acc, bias_down, None)
    assert torch.equal(got, ops.fused_gated_residual(be, ops.Policy(), x, ops.linear_output(be, acc, bias_down), None))
