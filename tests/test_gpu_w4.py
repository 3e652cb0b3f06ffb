"""Products with weights in 4 bits against a plain restatement in 64 bits."""
import pytest
import torch

from gpu_util import announce
from oracle import drafts as ref

pytestmark = pytest.mark.gpu


def K():
    from energonai_amd import kernel
    return kernel


def weight(N, Kd, group, dtype, zeros, seed):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (N, Kd // 2), generator=g, dtype=torch.uint8)
    scales = ((0.5 + torch.rand(N, -(-Kd // group), generator=g)) * (1 - 2 * torch.randint(0, 2, (N, 1), generator=g)) / 4 / Kd ** 0.5).to(dtype)
    z = torch.randint(0, 16, scales.shape, generator=g, dtype=torch.uint8) if zeros else None
    return codes, scales, z


MANY = 64            # rows up to which no weight is rounded


def tolerance(want, size, dtype, Kd, act, rounded=None):
    """Half a step of the result, and fp32 sums: at most 128 products of a group and their sums of x, the groups' sums one after another, over
    the waves and the bias, each half of 2^-23 of sum |scale| (code + zero) |x|.  GELU's slope is below 1.13, and its fp32 functions are good to 2^-19.
    ``rounded``: sum |weight| |x| of products with weights that are rounded to the activations' type, half a step of each (all
    scales here are above 2^-10 and weights whole multiples of them, so that none is among fp16's subnormal numbers)."""
    off = size * (2 * 128 + Kd // 32 + 32) * 2 ** -24
    if rounded is not None:
        off = off + torch.finfo(dtype).eps / 2 * rounded
    slope, own = (1.13, want.abs() * 2 ** -19 + 2 ** -21) if act in ("gelu", "gelu_tanh") else (1.0, 0.0)
    return torch.finfo(dtype).eps / 2 * want.abs() + slope * off + own + (2 ** -25 if dtype == torch.float16 else 1e-40)


def rounding(rows, x, codes, scales, z, group):
    return x.double().abs() @ ref.w4_values(codes, scales, z, group)[0].abs().t() if rows > MANY else None


CASES = [
    # rows, din, dout, group
    (1, 8, 1, 32), (1, 768, 2304, 64), (1, 136, 17, 128), (2, 32, 16, 32), (7, 200, 33, 64), (16, 128, 48, 128), (17, 1000, 65, 32), (31, 2048, 64, 64),
    (33, 512, 100, 128), (48, 384, 31, 64), (64, 1024, 272, 128), (65, 264, 128, 32), (100, 640, 50, 64), (130, 1536, 144, 128), (257, 520, 300, 32),
    (400, 256, 96, 64), (1, 8192, 32, 128), (5, 16384, 16, 128), (3, 64, 5000, 64), (2, 200, 9001, 32), (16, 264, 8200, 128), (20, 2304, 2000, 64),
    (48, 2200, 1111, 32), (64, 3200, 1500, 128), (90, 4096, 700, 64), (300, 1160, 1000, 128), (1100, 136, 8230, 64), (520, 264, 16500, 32), (257, 1000, 16400, 128),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("rows,Kd,N,group", CASES)
def test_product(rows, Kd, N, group, zeros, dtype):
    announce("w4", rows, Kd, N, group, zeros, dtype)
    codes, scales, z = weight(N, Kd, group, dtype, zeros, rows + N)
    x = torch.randn(rows, Kd, generator=torch.Generator().manual_seed(rows)).to(dtype)
    w = K().w4_weight(codes.cuda(), scales.cuda(), None if z is None else z.cuda(), group_size=group)
    want, size = ref.w4_linear(x, codes, scales, z, group)
    got = K().linear_w4(x.cuda(), w).cpu()
    assert got.shape == (rows, N)
    off = (got.double() - want).abs() - tolerance(want, size, dtype, Kd, None, rounding(rows, x, codes, scales, z, group))
    assert float(off.max()) <= 0, float(off.max())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act", [None, "none", "relu", "gelu_tanh", "gelu"])
@pytest.mark.parametrize("rows", [1, 20, 90, 200])
def test_bias_and_activation(rows, act, dtype):
    N, Kd, group = 77, 320, 64
    codes, scales, z = weight(N, Kd, group, dtype, True, 5)
    g = torch.Generator().manual_seed(6)
    x, bias = torch.randn(1, rows, Kd, generator=g).to(dtype), torch.randn(N, generator=g).to(dtype)
    w = K().w4_weight(codes.cuda(), scales.cuda(), z.cuda(), group_size=group)
    announce("w4 epilogue", rows, act, dtype)
    want, size = ref.w4_linear(x[0], codes, scales, z, group, bias, act)
    got = K().linear_w4(x.cuda(), w, bias=bias.cuda(), activation=act).cpu()
    assert got.shape == (1, rows, N)
    off = (got[0].double() - want).abs() - tolerance(want, size, dtype, Kd, act, rounding(rows, x[0], codes, scales, z, group))
    assert float(off.max()) <= 0, float(off.max())


def test_rows_keep_to_themselves():
    """A row that is not a number, or infinite, behind and before others; what lies behind a row's end; strides and addresses; no rows."""
    N, Kd, group, dtype = 40, 200, 64, torch.float16
    codes, scales, z = weight(N, Kd, group, dtype, True, 8)
    w = K().w4_weight(codes.cuda(), scales.cuda(), z.cuda(), group_size=group)
    for rows in (3, 40, 150, 300):
        wide = torch.full((rows, Kd + 16), float("nan"), dtype=dtype, device="cuda")
        x = wide[:, 8:8 + Kd]
        x.copy_(torch.randn(rows, Kd, generator=torch.Generator().manual_seed(9)))
        announce("w4 rows", rows)
        want = K().linear_w4(x.contiguous(), w)
        assert want.isfinite().all()
        assert torch.equal(K().linear_w4(x, w), want)                      # rows 16 channels apart, NaN between them
        odd = torch.full((rows, Kd + 3), float("nan"), dtype=dtype, device="cuda")[:, 1:1 + Kd]
        odd.copy_(x)
        assert torch.equal(K().linear_w4(odd, w), want)
        assert torch.equal(K().linear_w4(x.t().contiguous().t(), w), want)
        x[1] = float("nan")
        x[2, 7] = float("inf")
        got = K().linear_w4(x, w)
        assert torch.equal(got[0], want[0]) and torch.equal(got[3:], want[3:]) and got[1].isnan().all() and not got[2].isfinite().any()
    assert K().linear_w4(torch.empty(0, Kd, dtype=dtype, device="cuda"), w).shape == (0, N)
    assert K().linear_w4(torch.empty(2, 0, Kd, dtype=dtype, device="cuda"), w).shape == (2, 0, N)
    assert K().linear_w4(torch.zeros(Kd, dtype=dtype, device="cuda"), w).shape == (N,)


def test_results_do_not_change_from_call_to_call():
    codes, scales, z = weight(300, 4096, 128, torch.bfloat16, False, 2)
    w = K().w4_weight(codes.cuda(), scales.cuda(), group_size=128)
    for rows in (1, 30, 200):
        x = torch.randn(rows, 4096, device="cuda", dtype=torch.bfloat16)
        announce("w4 repeated", rows)
        first = K().linear_w4(x, w)
        for _ in range(5):
            assert torch.equal(K().linear_w4(x, w), first)


def test_codes_past_4_gib():
    """Codes whose offsets pass 32 bits: a weight of equal rows, whose products are equal too.  (Scales are above 2^-14 here, and so is what is
    rounded.)"""
    N, Kd, dtype = 4112, 1 << 21, torch.float16
    codes, scales, z = weight(16, Kd, 128, dtype, False, 4)
    w = K().w4_weight(codes.cuda().repeat(N // 16, 1), scales.cuda().repeat(N // 16, 1), group_size=128)
    assert w.codes.numel() > 1 << 32
    x = torch.randn(130, Kd, generator=torch.Generator().manual_seed(2)).to(dtype)
    want, size = ref.w4_linear(x[:1], codes, scales, z, 128)
    for rows in (1, 20, 130):
        announce("codes past 4 GiB", rows)
        got = K().linear_w4(x[:rows].cuda(), w).cpu()
        assert torch.equal(got.view(rows, -1, 16), got[:, :16].view(rows, 1, 16).expand(-1, N // 16, -1))
        rounded = x[:1].double().abs() @ ref.w4_values(codes, scales, z, 128)[0].abs().t() if rows > MANY else None
        assert ((got[:1, :16].double() - want).abs() <= tolerance(want, size, dtype, Kd, None, rounded)).all()


def test_rows_far_apart():
    """Rows of a view of any stride, among them those farther apart than the kernels take."""
    N, Kd, dtype = 40, 64, torch.bfloat16
    codes, scales, z = weight(N, Kd, 32, dtype, True, 8)
    w = K().w4_weight(codes.cuda(), scales.cuda(), z.cuda(), group_size=32)
    for rows, apart in ((3, 1 << 21), (3, (1 << 21) + 8), (300, 1 << 21), (2, 1 << 24), (5, 0)):
        x = torch.zeros(rows * apart + Kd, dtype=dtype, device="cuda").as_strided((rows, Kd), (apart, 1))
        x.copy_(torch.randn(1 if apart == 0 else rows, Kd, generator=torch.Generator().manual_seed(9)).to(dtype)) if apart else x[0].copy_(torch.randn(Kd).to(dtype))
        announce("w4 rows far apart", rows, apart)
        assert torch.equal(K().linear_w4(x, w), K().linear_w4(x.contiguous(), w))


@pytest.mark.parametrize("zero_points", [False, True])
def test_quantized_weight(zero_points):
    announce("w4 quantize", zero_points)
    dense = torch.randn(50, 264, generator=torch.Generator().manual_seed(1)).half()
    codes, scales, zeros = K().w4_codes(dense, 64, zero_points)
    w = K().w4_quantize(dense.cuda(), 64, zero_points)
    x = torch.eye(264, dtype=torch.float16)
    back = K().linear_w4(x.cuda(), w).cpu()
    want, _ = ref.w4_values(codes, scales, zeros, 64)
    # the host's and the device's rounding may differ where a value lies between two codes
    assert ((back.t().double() - want).abs() <= 1.01 * scales.double().repeat_interleave(64, 1)[:, :264] + 2 ** -11 * want.abs()).all()
    assert ((back.t().double() - dense.double()).abs() <= 1.52 * scales.double().repeat_interleave(64, 1)[:, :264]).all()


def test_refusals():
    codes, scales, z = (None if t is None else t.cuda() for t in weight(40, 200, 64, torch.float16, True, 8))
    k = K()
    for args in ((codes.int(), scales), (codes[:, :99].contiguous(), scales), (codes, scales[:, :3].contiguous()), (codes, scales.float()), (codes, scales, z.int()),
                 (codes, scales, z[:5].contiguous()), (codes.cpu(), scales), (codes.t(), scales)):
        with pytest.raises(RuntimeError):
            k.w4_weight(*args, group_size=64)
    for group in (16, 48, 256):
        with pytest.raises(RuntimeError):
            k.w4_weight(codes, scales, group_size=group)
    w = k.w4_weight(codes, scales, z, group_size=64)
    x = torch.zeros(3, 200, dtype=torch.float16, device="cuda")
    for args, kw in (((x.bfloat16(), w), {}), ((x[:, :192], w), {}), ((x.cpu(), w), {}), ((x, tuple(w)), {}), ((x, w), dict(activation="tanh")), ((x, w), dict(bias=x[0])),
                     ((x, w), dict(bias=torch.zeros(40, device="cuda"))), ((x, w._replace(in_features=264)), {}), ((x, w._replace(scales=scales)), {})):
        with pytest.raises(RuntimeError):
            k.linear_w4(*args, **kw)
