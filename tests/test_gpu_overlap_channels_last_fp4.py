"""Channels-last GroupNorm and the 4-bit operators with overlapped launches off and on: the same bits, back to back too, where every
call reads what the one before it wrote."""
import pytest

pytestmark = pytest.mark.gpu


def test_overlap_on_and_off_agree(gpu):
    import torch
    from vrhino_b200 import _lib
    be, ops = gpu
    lib = _lib.load()
    g = torch.Generator(device="cuda").manual_seed(1)

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, device="cuda", generator=g) * scale).bfloat16()

    def chain(x, weights, groups):
        y = x
        for w in weights:
            h = be.group_norm_channels_last(y, groups, None, None, 1e-6, activation=ops.SILU)
            q = be.fp4_quantize(h, w.format, be.fp4_tensor_scale(h) if w.format == ops.NVFP4 else None)
            y = be.fp4_linear(q, w)
        return y, be.fp4_dequantize(q)

    def packed(n, k, fmt):
        w = normal(n, k, scale=0.05)
        return be.fp4_quantize(w, fmt, be.fp4_tensor_scale(w) if fmt == ops.NVFP4 else None)
    # maps for registers, for shared memory, for two passes with and without a kernel that finishes the sums; few rows and many
    jobs = [(normal(1, 64, 256), [packed(256, 256, 0)] * 3, 32), (normal(1, 4096, 512), [packed(512, 512, 1)] * 3, 32),
            (normal(3, 9000, 640), [packed(640, 640, 0)] * 2, 32), (normal(1, 40000, 320), [packed(320, 320, 1)] * 2, 160)]
    previous = lib.vrb_set_launch_overlap(0)
    try:
        plain = [chain(*job) for job in jobs]
        torch.cuda.synchronize()
        assert lib.vrb_set_launch_overlap(1) == 0
        for _ in range(3):
            overlapped = [chain(*job) for job in jobs]
        torch.cuda.synchronize()
    finally:
        lib.vrb_set_launch_overlap(previous)
    for (y, v), (z, u) in zip(plain, overlapped):
        assert torch.equal(y, z) and torch.equal(v, u) and torch.isfinite(y.float()).all()
