"""The 4-bit operators on the GPU against their 64-bit forms (fp4_reference.py).

Packing and the tensor scale are exact: every rounding is that of a real quotient, so codes and scale bytes have to be
equal.  Unpacking is two F32 operations, restated here in F32.  The linear accumulates in F32: an instruction sums 64
products and adds them to the accumulator, and a term of it may be off by an F32 step (2^-23, truncation) of the sum of
magnitudes, so |error| <= (ceil(k / 64) + 2) * 2^-22 * sum |a b| before bias and activation; alpha, the bias add and the
result's rounding add half a step each."""
import numpy as np
import pytest

import fp4_reference as ref

pytestmark = pytest.mark.gpu

F32_HALF, BF16_HALF = 2.0 ** -24, 2.0 ** -8


def _np(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def _data(rows, k, dtype, seed, scale=1.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn((rows, k), device="cuda", generator=g) * scale).to(dtype)


def _dtype(name):
    import torch
    return {"bf16": torch.bfloat16, "f32": torch.float32}[name]


def _check_pack(q, x, fmt, g=None):
    codes, scales = ref.quantize(_np(x), fmt, None if g is None else float(g))
    assert np.array_equal(q.scales.cpu().numpy(), scales)
    assert np.array_equal(q.codes.cpu().numpy(), codes)


# ------------------------------------------------------------------------------------------- packing --
@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 16), (2, 15), (3, 33), (5, 31), (128, 64), (129, 65), (37, 1000), (257, 999), (31, 1536), (2, 8200),
                                    (300, 5), (200, 17), (130, 48), (400, 63)])
def test_pack_is_exact(gpu, fmt, dtype, rows, k):
    be, ops = gpu
    buffer = _data(1, rows * k + 3, _dtype(dtype), rows * 7 + k, 3.0)[0]
    for shift in (0, 1, 3):   # on and off a 16-byte boundary
        x = buffer[shift:shift + rows * k].view(rows, k)
        g = be.fp4_tensor_scale(x) if fmt == ops.NVFP4 else None
        _check_pack(be.fp4_quantize(x, fmt, g), x, fmt, g)


@pytest.mark.parametrize("g", [1.0, 0.37, 3.0e-5, 1.1e20, 2.0 ** -110, 3.0e38, 1.0e-42])
def test_pack_at_rounding_borders(gpu, g):
    """Values on the borders of e2m1 and e4m3, an F32 step below and above, under tensor scales with full mantissas and
    outside the range of the F32 form."""
    import torch
    be, ops = gpu
    gf = np.float32(g)
    rows = []
    rng = np.random.default_rng(5)
    borders = (ref.E2M1[1:] + ref.E2M1[:-1]) / 2
    with np.errstate(over="ignore"):
        for code in list(range(1, 127, 3)) + [126]:
            s = ref.E4M3[code]
            for step in (-1, 0, 1):
                top = np.float32(6.0 * float(gf) * s)
                v = np.concatenate([borders, borders, [0.0]]) * s * float(gf)
                v = v.astype(np.float32)
                v = np.where(v > 0, (v.view(np.int32) + step).clip(0).view(np.float32), v) if step else v
                rows.append(np.concatenate([[top], v]) * rng.choice([-1, 1], 16))
                edge = np.float32(6.0 * float(gf) * (s + ref.E4M3[code - 1]) / 2)   # a border of the scale itself
                edge = (np.array([edge]).view(np.int32) + step).clip(0).view(np.float32)[0]
                rows.append(np.concatenate([[edge], rng.uniform(-1, 1, 15) * edge]))
    x = np.array(rows, np.float32)
    x = x[np.isfinite(x).all(axis=1)]
    t = torch.from_numpy(x).cuda()
    scale = torch.tensor([gf], device="cuda")
    _check_pack(be.fp4_quantize(t, ops.NVFP4, scale), t, ref.NVFP4, gf)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("g", [1.0, 0.125, 1.0 / 3.0, 0.7, 3.0 / 2688.0, 1.875 / 2688.0, 1.9453125 / 2688.0, 1.7890625 / 2688.0])
def test_pack_values_of_few_bits(gpu, dtype, g):
    """Values of three to eight significant bits under tensor scales that put them on or within an F32 step of the borders:
    exact ties, and blocks in which every value is next to one."""
    import torch
    be, ops = gpu
    rng = np.random.default_rng(11)
    bits = rng.integers(2, 8, (256, 1))
    x = np.round(rng.uniform(-1, 1, (256, 256)) * 2.0 ** bits) / 2.0 ** bits * 2.0 ** rng.integers(-6, 3, (256, 1))
    x[:, ::16] = rng.choice([1.0, 1.5, 1.75, 1.25, 1.125, 1.875], (256, 16)) * 2.0 ** rng.integers(-3, 4, (256, 16))
    t = torch.from_numpy(x).cuda().to(_dtype(dtype))
    scale = torch.tensor([g], device="cuda", dtype=torch.float32)
    _check_pack(be.fp4_quantize(t, ops.NVFP4, scale), t, ref.NVFP4, np.float32(g))
    _check_pack(be.fp4_quantize(t, ops.MXFP4), t, ref.MXFP4)


@pytest.mark.parametrize("fmt", [0, 1])
def test_pack_special_values(gpu, fmt):
    """Zeros, infinities, NaN, subnormals and the largest values, each in a block of its own and mixed."""
    import torch
    be, ops = gpu
    inf, nan, big, tiny = float("inf"), float("nan"), 3.4028234e38, 1e-45
    x = torch.randn(12, 96, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    x[0] = 0.0
    x[1, :32] = -0.0
    x[2, 5], x[3, 40], x[4, 95] = inf, -inf, nan
    x[5, 0], x[5, 33] = big, -big
    x[6] = tiny
    x[7, :32] = tiny * 1000
    x[8] = torch.linspace(-1.2e-38, 1.2e-38, 96, device="cuda")
    x[9, 0], x[9, 1] = inf, nan
    for dtype in (torch.float32, torch.bfloat16):
        y = x.to(dtype)
        for g in ([None] if fmt else [None, 1.0, 1e-30, 2e38, 0.0, inf, nan]):
            scale = None if g is None else torch.tensor([g], device="cuda")
            _check_pack(be.fp4_quantize(y, fmt, scale), y, fmt, None if scale is None else np.float32(g))


def test_tensor_scale(gpu):
    import torch
    be, ops = gpu
    for dtype in (torch.float32, torch.bfloat16):
        for n in (1, 7, 8, 9, 1000, 1 << 20, (1 << 20) + 3):
            buffer = _data(1, n + 3, dtype, n)[0]
            for x in (buffer[:n], buffer[3:]):   # the second starts off a 16-byte boundary
                want = np.float32(float(x.float().abs().max()) / 2688.0)
                assert be.fp4_tensor_scale(x).item() == want
            # the largest magnitude at either end
            for at in (0, n - 1):
                y = buffer[:n].clone()
                y[at] = -1000.0
                assert be.fp4_tensor_scale(y).item() == np.float32(1000.0 / 2688.0)
    assert be.fp4_tensor_scale(torch.zeros(100, device="cuda")).item() == 0.0
    x = torch.ones(5000, device="cuda")
    x[4321] = float("-inf")
    assert be.fp4_tensor_scale(x).item() == float("inf")
    x[17] = float("nan")
    assert np.isnan(be.fp4_tensor_scale(x).item())


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 33), (129, 64), (200, 999), (7, 1536), (77, 5), (1001, 17), (300, 63), (40, 65), (9, 2051)])
def test_unpack_is_exact(gpu, fmt, dtype, rows, k):
    """All codes and scale bytes at random (NaN scales among them)."""
    import torch
    be, ops = gpu
    rng = np.random.default_rng(rows + k)
    codes = rng.integers(0, 256, (rows, ref.row_bytes(k)), dtype=np.uint8)
    scales = rng.integers(0, 128 if fmt == 0 else 256, ref.scale_bytes(fmt, rows, k)).astype(np.uint8)
    g = np.float32(0.0123) if fmt == 0 else None
    q = ops.Fp4Tensor(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), None if g is None else torch.tensor([g], device="cuda"), fmt, (rows, k))
    e, s = ref.parts(codes, scales, fmt, rows, k)
    with np.errstate(over="ignore", invalid="ignore"):
        want = (e * s).astype(np.float32) * (g if g is not None else np.float32(1.0))
    want = torch.from_numpy(want).to(_dtype(dtype))
    for shift in (0, 1, 3):   # the result on and off a 16-byte boundary, and what lies around it
        buffer = torch.full((rows * k + 16,), 7.0, device="cuda", dtype=_dtype(dtype))
        got = be.fp4_dequantize(q, _dtype(dtype), out=buffer[shift:shift + rows * k].view(rows, k)).cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got, 0.0), torch.nan_to_num(want, 0.0))
        assert (buffer[:shift] == 7.0).all() and (buffer[shift + rows * k:] == 7.0).all()


def test_pack_and_unpack_past_32_bit_offsets(gpu):
    """2^31 + elements: rows at the far end equal the same rows packed alone."""
    import torch
    be, ops = gpu
    rows, k = 33 * 1024 + 5, 65536 + 32
    x = torch.randn((rows, k), device="cuda", dtype=torch.bfloat16)
    q = be.fp4_quantize(x, ops.MXFP4)
    last = be.fp4_quantize(x[-5:].contiguous(), ops.MXFP4)
    assert torch.equal(q.codes[-5:], last.codes)
    back = be.fp4_dequantize(q)
    assert torch.equal(back[-5:], be.fp4_dequantize(last))
    assert torch.equal(back[:3], be.fp4_dequantize(be.fp4_quantize(x[:3].contiguous(), ops.MXFP4)))


# -------------------------------------------------------------------------------------------- linear --
def _packed(be, ops, rows, k, fmt, seed, scale=1.0):
    import torch
    x = _data(rows, k, torch.float32, seed, scale)
    return be.fp4_quantize(x, fmt, be.fp4_tensor_scale(x) if fmt == ops.NVFP4 else None)


def _reference(a, b, bias, kind):
    """(values, bound of the error before the result's rounding) in 64 bits"""
    va = ref.values(a.codes.cpu().numpy(), a.scales.cpu().numpy(), a.format, a.rows, a.k, None if a.tensor_scale is None else a.tensor_scale.item())
    vb = ref.values(b.codes.cpu().numpy(), b.scales.cpu().numpy(), b.format, b.rows, b.k, None if b.tensor_scale is None else b.tensor_scale.item())
    acc, mass = va @ vb.T, np.abs(va) @ np.abs(vb).T
    y = acc + (0.0 if bias is None else _np(bias))
    bound = (-(-a.k // 64) + 2) * 2.0 ** -22 * mass + 3 * F32_HALF * np.abs(acc) + F32_HALF * np.abs(y)
    out = ref.activation(y, kind)
    if kind is not None:   # every activation's slope is below 1.2; evaluating it adds less than 2^-20 of its argument
        bound = 1.2 * bound + 2.0 ** -20 * np.abs(y) + 1e-30
    return out, bound


def _check_linear(got, a, b, bias, kind):
    import torch
    want, bound = _reference(a, b, bias, kind)
    half = BF16_HALF if got.dtype == torch.bfloat16 else F32_HALF
    error = np.abs(_np(got).reshape(want.shape) - want)
    over = error > bound + half * (np.abs(want) + bound) + 1e-40
    assert not over.any(), f"{over.sum()} of {over.size}, worst {np.max(error / (bound + half * np.abs(want) + 1e-300)):.3g} times the bound"


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("m,k,n", [
    (1, 1, 1), (1, 16, 8), (2, 1536, 264), (5, 33, 7), (16, 4096, 128), (17, 520, 130), (40, 64, 333), (64, 2048, 1024), (100, 256, 96),
    (128, 64, 128), (128, 256, 256), (129, 320, 129), (255, 1000, 257), (300, 288, 1003), (513, 1024, 512), (1000, 500, 640),
])
def test_linear(gpu, fmt, out, m, k, n):
    be, ops = gpu
    a, b = _packed(be, ops, m, k, fmt, m + k, 2.0), _packed(be, ops, n, k, fmt, n + k + 1, 0.05)
    _check_linear(be.fp4_linear(a, b, dtype=_dtype(out)), a, b, None, None)


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("kind", [None, 0, 1, 2, 3, 4])
@pytest.mark.parametrize("m,n", [(3, 200), (150, 264), (300, 131)])
def test_linear_bias_and_activation(gpu, fmt, out, kind, m, n):
    import torch
    be, ops = gpu
    a, b = _packed(be, ops, m, 384, fmt, 3, 2.0), _packed(be, ops, n, 384, fmt, 4, 0.1)
    for dtype in (torch.bfloat16, torch.float32):
        bias = _data(1, n, dtype, 9)[0]
        _check_linear(be.fp4_linear(a, b, bias, kind, dtype=_dtype(out)), a, b, bias, kind)


@pytest.mark.parametrize("m,k,n", [(2, 512, 256), (200, 512, 300), (700, 512, 600)])
def test_linear_many_tiles_and_long_k(gpu, m, k, n):
    """A long k (more stages than buffers) and many tiles per CTA, on rows whose products are exact in F32."""
    import torch
    be, ops = gpu
    k *= 40
    a, b = _packed(be, ops, m, k, ops.MXFP4, 1), _packed(be, ops, n, k, ops.MXFP4, 2)
    _check_linear(be.fp4_linear(a, b, dtype=torch.float32), a, b, None, None)
    a, b = _packed(be, ops, m * 8, 64, ops.NVFP4, 1), _packed(be, ops, n * 16, 64, ops.NVFP4, 2)
    _check_linear(be.fp4_linear(a, b, dtype=torch.float32), a, b, None, None)


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("m", [3, 160, 600])
def test_linear_keeps_bad_rows_to_themselves(gpu, fmt, m):
    """A NaN or an infinity in one row of either operand reaches that row or column of the result and nothing else; rows of
    zeros give zeros."""
    import torch
    be, ops = gpu
    x, w = _data(m, 200, torch.float32, 1), _data(140, 200, torch.float32, 2)
    x[m - 1, 77], w[5, 3] = float("nan"), float("inf")
    x[1] = 0.0
    scale = torch.tensor([0.01], device="cuda") if fmt == ops.NVFP4 else None
    y = be.fp4_linear(be.fp4_quantize(x, fmt, scale), be.fp4_quantize(w, fmt, scale), dtype=torch.float32)
    bad = torch.zeros((m, 140), dtype=torch.bool, device="cuda")
    bad[m - 1], bad[:, 5] = True, True
    assert torch.equal(torch.isnan(y), bad)
    assert (y[1][~bad[1]] == 0).all()


@pytest.mark.parametrize("m,n", [(2, 96), (130, 200), (515, 264)])
def test_linear_leaves_what_lies_behind(gpu, m, n):
    import torch
    be, ops = gpu
    a, b = _packed(be, ops, m, 320, 0, 1), _packed(be, ops, n, 320, 0, 2)
    for dtype in (torch.bfloat16, torch.float32):
        buffer = torch.full((m + 300, n), 7.0, device="cuda", dtype=dtype)
        be.fp4_linear(a, b, dtype=dtype, out=buffer[:m])
        assert (buffer[m:] == 7.0).all()
        assert torch.equal(buffer[:m], be.fp4_linear(a, b, dtype=dtype))
    x = _data(m, 77, torch.bfloat16, 5)
    codes = torch.full((m + 4, ref.row_bytes(77)), 9, device="cuda", dtype=torch.uint8)
    scales = torch.full((ref.scale_bytes(0, m, 77) + 512,), 9, device="cuda", dtype=torch.uint8)
    q = ops.Fp4Tensor(codes[:m], scales[:-512], None, 0, (m, 77))
    be.fp4_quantize(x, 0, None, out=q)
    assert (codes[m:] == 9).all() and (scales[-512:] == 9).all()
    _check_pack(q, x, 0)


def test_linear_unaligned_result(gpu):
    import torch
    be, ops = gpu
    a, b = _packed(be, ops, 150, 128, 0, 1), _packed(be, ops, 136, 128, 0, 2)
    want = be.fp4_linear(a, b)
    shifted = torch.empty(150 * 136 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(150, 136)
    assert torch.equal(be.fp4_linear(a, b, out=shifted), want)


def test_linear_past_32_bit_offsets(gpu):
    import torch
    be, ops = gpu
    m, n, k = 70_000, 31_000, 32
    a, b = _packed(be, ops, m, k, 1, 1), _packed(be, ops, n, k, 1, 2)
    y = be.fp4_linear(a, b)
    va, vb = be.fp4_dequantize(a, torch.float32), be.fp4_dequantize(b, torch.float32)
    for rows in (slice(0, 3), slice(m - 3, m), slice(69_272, 69_275)):
        want = (va[rows].double() @ vb.double().t())
        assert torch.allclose(y[rows].double(), want, rtol=2.0 ** -8, atol=1e-4)


def test_runs_repeat_bit_for_bit(gpu):
    import torch
    be, ops = gpu
    for m, k, n in ((2, 4096, 512), (90, 2048, 300), (700, 1536, 900)):
        a, b = _packed(be, ops, m, k, 0, 1), _packed(be, ops, n, k, 0, 2)
        first = be.fp4_linear(a, b, dtype=torch.float32)
        for _ in range(5):
            assert torch.equal(be.fp4_linear(a, b, dtype=torch.float32), first)


@pytest.mark.parametrize("m", [2, 200])
def test_captured_and_replayed(gpu, m):
    """Quantise + linear captured into two graphs that live side by side, replayed on new inputs on a side stream."""
    import torch
    be, ops = gpu
    w = _packed(be, ops, 264, 640, 0, 4, 0.1)
    bias = _data(1, 264, torch.bfloat16, 2)[0]
    scale = torch.tensor([0.002], device="cuda")
    inputs = [_data(m, 640, torch.bfloat16, s) for s in (1, 2)]

    def step(x):
        return be.fp4_linear(be.fp4_quantize(x, 0, scale), w, bias, ops.GELU_TANH)
    want = [step(x) for x in inputs]
    torch.cuda.synchronize()
    graphs, statics, outs = [], [], []
    for _ in range(2):
        static = torch.zeros_like(inputs[0])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(static))
        graphs.append(graph)
        statics.append(static)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for order in ((0, 1), (1, 0)):
            for i in (0, 1):
                statics[i].copy_(inputs[order[i]])
            for i in (0, 1):
                graphs[i].replay()
            side.synchronize()
            for i in (0, 1):
                assert torch.equal(outs[i], want[order[i]])


def test_first_calls_of_a_process_are_captured(gpu):
    """No call of the library before the capture: attributes, occupancy and the encoder are looked up while capturing."""
    import subprocess
    import sys
    code = """
import torch
from vrhino_b200 import ops
be = ops.B200Backend()
x = {m: torch.randn((m, 640), device="cuda").bfloat16() for m in (2, 40, 700)}
h = {s: torch.randn((1, s, 64), device="cuda").bfloat16() for s in (50, 60000)}
w = torch.randn((900, 640), device="cuda")
torch.cuda.synchronize()
def run():
    q = be.fp4_quantize(w, 0, be.fp4_tensor_scale(w))
    y = [be.fp4_linear(be.fp4_quantize(x[m], 0, q.tensor_scale), q) for m in x]
    return y + [be.group_norm_channels_last(h[s], 8, None, None, 1e-6, activation=0) for s in h] + [be.fp4_dequantize(q)]
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    captured = run()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(captured, run()))
print("captured")
"""
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=root, timeout=120)
    assert done.returncode == 0 and "captured" in done.stdout, done.stderr[-2000:]


def test_many_clusters_on_many_streams(gpu):
    """Clusters along k of several shapes, more at once than the SMs hold, from eight streams: allocations of tensor memory must
    not wait for each other."""
    import torch
    be, ops = gpu
    jobs = [(_packed(be, ops, m, k, 0, m), _packed(be, ops, n, k, 0, m + 1)) for m, k, n in
            ((1, 512, 4096), (2, 8192, 512), (16, 4096, 1024), (30, 2048, 3000), (64, 8192, 640), (100, 4096, 900), (300, 512, 300), (600, 1024, 2000))]
    want = [be.fp4_linear(a, b) for a, b in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    got = []
    for _ in range(30):
        for i, (a, b) in enumerate(jobs):
            with torch.cuda.stream(streams[i]):
                got.append(be.fp4_linear(a, b))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i % len(jobs)]) for i, y in enumerate(got))


def test_two_streams_at_once(gpu):
    import torch
    be, ops = gpu
    jobs = [(_packed(be, ops, m, 1024, 0, m), _packed(be, ops, 700, 1024, 0, m + 1)) for m in (2, 300, 90, 1000)]
    want = [be.fp4_linear(a, b) for a, b in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = []
    for _ in range(10):
        for (a, b), s in zip(jobs, streams):
            with torch.cuda.stream(s):
                got.append(be.fp4_linear(a, b))
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % len(jobs)])


def test_no_wait_ran_out(gpu):
    import ctypes
    from vrhino_b200 import _lib
    failures = ctypes.c_int(-1)
    _lib.call("vrb_async_wait_failures", ctypes.byref(failures))
    assert failures.value == 0


# ----------------------------------------------------------------------------------- used together --
@pytest.mark.parametrize("fmt", [0, 1])
def test_group_norm_into_linear_into_residual(gpu, fmt):
    """A VAE attention block's projection as it would run: channels-last GroupNorm + SiLU, packed rows, the 4-bit linear into
    the F32 accumulation, and the framework's own epilogue with the residual update."""
    import torch
    be, ops = gpu
    x = _data(2 * 144, 256, torch.bfloat16, 1).view(2, 144, 256)
    w = _packed(be, ops, 256, 256, fmt, 2, 0.06)
    bias = _data(1, 256, torch.bfloat16, 3)[0]
    h = be.group_norm_channels_last(x, 32, None, None, 1e-6, activation=ops.SILU)
    q = be.fp4_quantize(h, fmt, be.fp4_tensor_scale(h) if fmt == ops.NVFP4 else None)
    acc = be.fp4_linear(q, w, dtype=torch.float32)
    assert acc.shape == (2, 144, 256)
    got = ops.linear_output_gated_residual(be, ops.Policy(), x, acc, bias, None)
    want, bound = _reference(q, w, None, None)
    assert (np.abs(_np(acc).reshape(want.shape) - want) <= bound).all()
    chain = ops.fused_gated_residual(be, ops.Policy(), x, ops.linear_output(be, acc, bias), None)
    assert torch.equal(got, chain)
    fused = be.fp4_linear(q, w, bias)     # bias in the product's own epilogue
    _check_linear(fused, q, w, bias, None)
    assert torch.equal(fused, ops.linear_output(be, acc, bias))


# ------------------------------------------------------------------------------------------ refusals --
def test_refusals(gpu):
    import torch
    be, ops = gpu
    a, b = _packed(be, ops, 4, 64, 0, 1), _packed(be, ops, 8, 64, 0, 2)
    c = _packed(be, ops, 8, 96, 0, 2)
    d = _packed(be, ops, 8, 64, 1, 2)
    for x, w in ((a, c), (a, d)):
        with pytest.raises(ops.VrbError, match="differ in format or width"):
            be.fp4_linear(x, w)
    with pytest.raises(ops.VrbError, match="linear bias mismatch"):
        be.fp4_linear(a, b, torch.zeros(7, device="cuda"))
    with pytest.raises(ops.VrbError, match="do not match the shape"):
        be.fp4_linear(a, ops.Fp4Tensor(b.codes, b.scales[:-1], b.tensor_scale, 0, b.shape))
    with pytest.raises(ops.VrbError, match="do not match the shape"):
        be.fp4_dequantize(ops.Fp4Tensor(a.codes, a.scales, a.tensor_scale, 0, (4, 65)))
    with pytest.raises(ops.VrbError, match="one F32"):
        be.fp4_quantize(torch.zeros(4, 64, device="cuda"), 0, torch.zeros(2, device="cuda"))
    with pytest.raises(ops.VrbError, match="one F32"):
        be.fp4_quantize(torch.zeros(4, 64, device="cuda"), 0, torch.zeros(1))
    with pytest.raises(ops.VrbError, match="must be positive"):
        be.fp4_quantize(torch.zeros(0, 64, device="cuda"))
    with pytest.raises(ops.VrbError, match="no tensor scale"):
        be.fp4_quantize(torch.zeros(4, 64, device="cuda"), 1, torch.ones(1, device="cuda"))
    with pytest.raises(ops.VrbError, match="unknown 4-bit format"):
        be.fp4_quantize(torch.zeros(4, 64, device="cuda"), 7)
    with pytest.raises(ops.VrbError, match="output buffer"):
        be.fp4_linear(a, b, out=torch.zeros(4, 8, device="cuda"))
    with pytest.raises(ops.VrbError, match="unknown activation"):
        be.fp4_linear(a, b, activation=9)
