"""Products with weights in 4 bits: zero points of any byte, and each kernel with each epilogue."""
import pytest
import torch

from gpu_util import announce
from oracle import drafts as ref
from test_gpu_w4 import rounding, tolerance, weight

pytestmark = pytest.mark.gpu


def K():
    from energonai_amd import kernel
    return kernel


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,Kd,N,group", [(1, 264, 40, 32), (20, 264, 40, 64), (40, 2304, 2001, 128), (90, 1024, 300, 64), (257, 264, 16401, 32)])
def test_zero_points_of_any_byte(rows, Kd, N, group, dtype):
    """Zero points are what they say, 16 and 255 among them."""
    codes, scales, z = weight(N, Kd, group, dtype, True, rows)
    g = torch.Generator().manual_seed(3)
    z = torch.randint(0, 256, z.shape, generator=g, dtype=torch.uint8)
    z[0, 0], z[N // 2, -1], z[-1, 0] = 16, 255, 15
    x = torch.randn(rows, Kd, generator=g).to(dtype)
    announce("w4 zero points", rows, Kd, N, group, dtype)
    w = K().w4_weight(codes.cuda(), scales.cuda(), z.cuda(), group_size=group)
    c = torch.stack((codes & 15, codes >> 4), -1).view(N, Kd).double()
    s, zero = (t.double().repeat_interleave(group, 1)[:, :Kd] for t in (scales, z))
    values, size = (c - zero) * s, x.double().abs() @ (s.abs() * (c + zero)).t()
    want = x.double() @ values.t()
    rounded = x.double().abs() @ values.abs().t() if rows > 64 else None
    got = K().linear_w4(x.cuda(), w).cpu().double()
    off = (got - want).abs() - tolerance(want, size, dtype, Kd, None, rounded)
    assert float(off.max()) <= 0, float(off.max())


def check(rows, Kd, N, group, zeros, dtype, bias, act, runs):
    from energonai_amd import _lib
    assert (_lib.fn.en_linear_w4_workspace_bytes(rows, N, Kd) > 0) == runs, "another form of the kernel than the case is for"
    codes, scales, z = weight(N, Kd, group, dtype, zeros, rows + N)
    g = torch.Generator().manual_seed(rows)
    x, b = torch.randn(rows, Kd, generator=g).to(dtype), torch.randn(N, generator=g).to(dtype) if bias else None
    w = K().w4_weight(codes.cuda(), scales.cuda(), None if z is None else z.cuda(), group_size=group)
    want, size = ref.w4_linear(x, codes, scales, z, group, b, act)
    got = K().linear_w4(x.cuda(), w, bias=None if b is None else b.cuda(), activation=act).cpu().double()
    off = (got - want).abs() - tolerance(want, size, dtype, Kd, act, rounding(rows, x, codes, scales, z, group))
    assert float(off.max()) <= 0, float(off.max())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows", [17, 20, 33, 40, 48, 49, 64])
def test_some_rows_of_wide_weights(rows, group, dtype):
    """Two, three and four tiles of rows against four tiles of W a workgroup, whose last one is ragged, with the channels in one run and in four."""
    announce("w4 some rows, wide", rows, group, dtype)
    check(rows, 2304, 2001, group, rows % 2 == 0, dtype, False, None, True)
    check(rows, 264, 14408 + 9, group, rows % 2 == 1, dtype, False, None, False)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act", [None, "relu", "gelu_tanh", "gelu"])
@pytest.mark.parametrize("rows,Kd,N,group,runs", [
    (7, 136, 8201, 64, False), (12, 136, 8201, 32, False),                      # four tiles of W a workgroup
    (40, 2304, 2001, 128, True), (20, 2304, 2001, 32, True), (64, 2304, 2001, 64, True),       # ... their sums joined
    (40, 264, 14417, 64, False),
    (90, 4096, 700, 64, True),                                                  # tiles of 128 x 128, joined
    (300, 264, 2001, 128, False),
    (257, 264, 16401, 32, False),                                               # tiles of 256 x 256
])
def test_epilogue_of_each_form(rows, Kd, N, group, runs, act, dtype):
    announce("w4 epilogue of each form", rows, Kd, N, group, act, dtype)
    check(rows, Kd, N, group, True, dtype, True, act, runs)
