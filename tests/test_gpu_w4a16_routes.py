"""Every kernel that the 4-bit linear's plan chooses from, over enough steps of columns that its stages in
LDS come round (two to four of them), in each group size it has an instance for, against the 64-bit
product. Each row states the route it tests, and the plan is held to it: sizes that a later rule sends
elsewhere fail here instead of testing another kernel.

Tolerance as in tests/test_gpu_w4a16.py: the output's rounding, eps / 2 |y|, and the fp32 sums: terms of
size |x| (31 + 24) s, 32 + 4 roundings inside a group's chain and one for each group, wave, slice (up to
16 of these two) and the bias after it.
"""
import pytest
import torch

from specdec_nanovllm_amd import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def weights(w, s):
    """The 4-bit weight in 64 bits, and 55 times its scales."""
    n, half = w.shape
    codes = torch.stack((w & 15, w >> 4), -1).view(n, 2 * half).double() - 8
    scales = s.double().repeat_interleave(2 * half // s.shape[1], 1)
    return codes * scales, 55 * scales


def check(got, x, w, s, b):
    eps = float(torch.finfo(x.dtype).eps)
    wx, sx = weights(w, s)
    want = x.double() @ wx.T.contiguous() + b.double()
    size = x.double().abs() @ sx.T.contiguous() + b.double().abs()
    tol = eps / 2 * want.abs() + (36 + 4 * s.shape[1] + 16) * 2**-24 * size + 1e-7
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), f"off by {off.max().item():.3g} in {int((off > tol).sum())} outputs"


# (rows, columns of the output, K, group): (tile rows, tile columns, K slices); tile rows 0: the kernel for few
# rows, with the weight rows of its tiles and its waves
FEW = [
    ((1, 4100, 1312, 32), (0, 16, 4)), ((1, 16391, 1312, 32), (0, 32, 4)), ((2, 19456, 832, 64), (0, 32, 4)),
    ((1, 19456, 2560, 128), (0, 32, 4)), ((3, 16391, 1312, 32), (0, 32, 4)), ((5, 19456, 1344, 64), (0, 32, 4)),
    ((8, 16391, 1152, 128), (0, 32, 4)), ((8, 19456, 2560, 128), (0, 32, 4)), ((7, 16391, 800, 32), (0, 32, 4)),
    ((1, 151936, 256, 64), (0, 32, 4)), ((5, 151936, 288, 32), (0, 32, 4)), ((8, 151936, 384, 128), (0, 32, 4)),
    ((9, 4100, 1312, 32), (0, 16, 4)), ((16, 9001, 1600, 64), (0, 16, 4)), ((16, 2560, 9728, 128), (0, 16, 6)),
    ((20, 4096, 1024, 128), (0, 16, 2)), ((32, 3000, 2016, 32), (0, 16, 2)), ((32, 3000, 1984, 64), (0, 16, 2))]
SOME = [
    ((16, 19456, 1312, 32), (32, 128, 3)), ((20, 33000, 1312, 32), (32, 128, 1)), ((20, 33000, 832, 64), (32, 128, 1)),
    ((32, 33000, 1152, 128), (32, 128, 1)), ((17, 16391, 3328, 64), (32, 128, 3)), ((32, 9001, 1312, 32), (32, 64, 3)),
    ((20, 9001, 3328, 64), (32, 64, 3)), ((20, 2570, 9728, 128), (32, 64, 12)), ((33, 16391, 1312, 32), (64, 128, 3)),
    ((40, 19456, 832, 64), (64, 128, 3)), ((64, 33000, 1152, 128), (64, 128, 1)), ((64, 33000, 1312, 32), (64, 128, 1)),
    ((56, 33000, 832, 64), (64, 128, 1)), ((56, 19456, 2560, 128), (64, 128, 3)), ((40, 9001, 1312, 32), (64, 64, 1)),
    ((56, 2570, 9728, 64), (64, 64, 6)), ((64, 2570, 4160, 32), (64, 64, 6)), ((56, 2570, 9728, 128), (64, 64, 6))]
MANY = [
    ((130, 9001, 1312, 32), (64, 64, 1)), ((300, 2570, 1280, 128), (64, 64, 1)), ((100, 1300, 9728, 64), (64, 64, 6)),
    # eight waves that take turns: one slice of five steps and more, half a step of columns at the end
    ((100, 16391, 1312, 32), (128, 128, 1)), ((66, 19456, 832, 64), (128, 128, 1)), ((100, 24500, 768, 128), (128, 128, 1)),
    ((129, 16391, 832, 64), (128, 192, 1)), ((130, 19456, 1280, 128), (128, 192, 1)),
    ((257, 16391, 832, 64), (128, 256, 1)), ((300, 19456, 1280, 128), (128, 256, 1)),
    # and in K slices
    ((200, 2570, 9728, 32), (128, 128, 6)), ((500, 2570, 9728, 64), (128, 128, 3)), ((200, 2570, 9728, 128), (128, 128, 6)),
    ((777, 1300, 9728, 64), (128, 192, 5)), ((777, 1300, 9728, 128), (128, 192, 5)),
    ((777, 2570, 9728, 128), (128, 256, 3)), ((300, 4100, 9728, 64), (128, 256, 5))]


@pytest.mark.parametrize("sizes,route", FEW + SOME + MANY, ids=lambda t: "x".join(map(str, t)))
@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_routes(sizes, route, kind):
    """Activations in strided rows with NaN beside them, outputs in strided rows whose neighbours
    stay, the slices' workspace and none (one slice)."""
    m, n, k, group = sizes
    lib = _lib.load()
    if torch.cuda.get_device_properties(0).multi_processor_count == 256:
        plan = lib.sd_w4a16_plan(m, n, k, group)
        assert (plan >> 20, plan >> 8 & 0xfff, plan & 0xff) == route
    g = torch.Generator(device=DEV).manual_seed(m + n + k)
    w = torch.randint(0, 256, (n, k // 2), generator=g, device=DEV, dtype=torch.uint8)
    s = ((torch.rand((n, k // group), generator=g, device=DEV) + 0.2) * 0.02).to(kind)
    b = torch.randn((n,), generator=g, device=DEV).to(kind)
    wide = torch.full((m, k + 16), float("nan"), device=DEV, dtype=kind)
    x = wide[:, 8:k + 8].copy_(torch.randn((m, k), generator=g, device=DEV))
    out = torch.full((m, n + 3), 7.0, device=DEV, dtype=kind)
    y = ops.w4a16_linear(x, w, s, b, out=out[:, 1:n + 1])
    check(y, x, w, s, b)
    assert bool((out[:, 0] == 7).all()) and bool((out[:, n + 1:] == 7).all())
    whole = ops.w4a16_linear(x, w, s, b)  # aligned rows of its own
    assert torch.equal(whole, y)
    if lib.sd_w4a16_workspace_size(m, n, k, group):
        y = torch.full((m, n), float("nan"), device=DEV, dtype=kind)
        _lib.check(lib.sd_w4a16_linear(x.data_ptr(), x.stride(0), w.data_ptr(), k // 2, s.data_ptr(),
                                       _lib.dtype_code(kind), group, b.data_ptr(), y.data_ptr(), n, m, n, k,
                                       _lib.dtype_code(kind), None, 0, _lib.stream_ptr(x.device)))
        check(y, x, w, s, b)
