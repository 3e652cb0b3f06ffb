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
