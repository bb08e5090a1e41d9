"""Products of a few tokens with 4-bit weights against the definition in 64 bits.

Bound.  With u = 2^-24, the products (16 + q) x (q x for FP32 tokens) are exact in FP32 or rounded once, and a lane adds the
32 columns of one group, in the worst case with one rounding of at most u times (31 or 15) sum|x| per column and one each
for the offset's sum and product: 36 u (o + 15 + o + z) sum|x|, o = 16 (0), below 36 * 62 u (36 * 30 u) sum|x| times |s|.
The matrix-core form adds whole groups of up to 128 columns, in the worst case one rounding per column: 132 in the place of
36.  FP32 tokens (four and more) go there as three parts each, of one sign, which add up to them: 3 * 128 exact products with
q - z, of magnitude 15 at most, so 388 in the place of 36 and 15 in the place of 30.  Adding the groups is off by u (N / 32 + 16) sum |s| (q - z) |x|, then the result is rounded once."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def half(t):
    return torch.finfo(t).eps / 2


def make(M, N, group, dtype, zeros, seed, ldq_extra=0, ldg_extra=0):
    """Random weights in strided buffers whose padding must not matter."""
    g = torch.Generator().manual_seed(seed)
    groups = -(-N // group)
    ldq = -(-((N + 1) // 2) // 4) * 4 + ldq_extra
    q = torch.randint(0, 256, (max(M, 1), max(ldq, 4)), generator=g, dtype=torch.uint8).cuda()   # a random half byte behind an odd row's end
    s = torch.full((max(M, 1), groups + ldg_extra), float("nan"))
    s[:, :groups] = torch.randn(max(M, 1), groups, generator=g) * 0.05
    z = torch.full((max(M, 1), groups + ldg_extra), 255, dtype=torch.uint8)
    z[:, :groups] = torch.randint(0, 16, (max(M, 1), groups), generator=g, dtype=torch.uint8)
    return q, s.to(dtype).cuda(), z.cuda() if zeros else None


def dense(q, s, z, M, N, group):
    low, high = (q & 15).double(), (q >> 4).double()
    w = torch.stack((low, high), 2).view(q.shape[0], -1)[:M, :N]
    groups = -(-N // group)
    zz = (z[:M, :groups].double() if z is not None else torch.full((M, groups), 8.0, dtype=torch.float64, device=q.device))
    zz = zz.repeat_interleave(group, 1)[:, :N]
    ss = s[:M, :groups].double().repeat_interleave(group, 1)[:, :N]
    return w - zz, ss


def check(blas, batch, M, N, group, dtype, zeros, seed, alpha=1.0, beta=0.0, ldq_extra=0, ldg_extra=0, pad=0, offset=0.0):
    q, s, z = make(M, N, group, dtype, zeros, seed, ldq_extra, ldg_extra)
    g = torch.Generator().manual_seed(seed + 1)
    xb = torch.full((batch, N + pad), float("nan"), dtype=dtype)
    xb[:, :N] = (torch.randn(batch, N, generator=g) + offset).to(dtype)
    x = xb.cuda()[:, :N]
    yb = torch.full((batch, M + pad), float("nan"), dtype=dtype)
    if beta != 0:
        yb[:, :M] = torch.randn(batch, M, generator=g).to(dtype)
    yb = yb.cuda()
    y0 = yb.clone().double()[:, :M]
    blas.w4_gemv(batch, M, N, group, alpha, q, s, z, x, beta, yb[:, :M])
    w, ss = dense(q, s, z, M, N, group)
    x64 = x.double()
    ref = alpha * (x64 @ (w * ss).t().contiguous())
    worst = (132 * 62 if dtype != F32 else 388 * 15 if batch >= 4 else 36 * 30) * (x64.abs() @ ss.abs().t().contiguous()) + (N / 32 + 16) * (x64.abs() @ (w * ss).abs().t().contiguous())
    if beta != 0:
        ref = ref + beta * y0
    tol = half(dtype) * ref.abs() + U * (abs(alpha) * worst + 3 * ref.abs() + (abs(beta) * y0.abs() if beta != 0 else 0))
    tol = tol + (2.0 ** -25 if dtype == F16 else 0)
    got = yb[:, :M].double()
    assert torch.all((got - ref).abs() <= tol), float(((got - ref).abs() / tol).max())
    if pad:
        assert torch.all(torch.isnan(yb[:, M:]))
    return yb[:, :M].clone()


# (M, N): one row, one column, odd ones, rows ending inside a group, a byte and a dword, several panels of x
SIZES = [(1, 1), (1, 64), (3, 2), (5, 31), (16, 33), (17, 100), (31, 255), (64, 1000), (130, 2047), (33, 2049), (1000, 4096), (257, 4101), (20, 40000),
         (2, 70001)]


@pytest.mark.parametrize("M,N", SIZES)
@pytest.mark.parametrize("dtype,zeros,group", [(F32, False, 32), (F32, True, 128), (F16, False, 64), (F16, True, 32), (BF16, False, 128), (BF16, True, 64),
                                               (BF16, False, 32)])
def test_single_token(blas, M, N, dtype, zeros, group):
    check(blas, 1, M, N, group, dtype, zeros, M + N, pad=(M + N) % 3)


@pytest.mark.parametrize("batch,M", [(1, 4149), (2, 5001), (1, 9001), (2, 12300), (1, 16500), (3, 4200), (4, 8200), (16, 12500), (17, 4111)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_many_rows(blas, batch, M, dtype):
    """Several rows to a wave and several turns to a workgroup, the last of them cut."""
    check(blas, batch, M, 321, 64, dtype, True, M)


@pytest.mark.parametrize("batch", [2, 3, 4, 5, 7, 8, 13, 16, 17, 33])
@pytest.mark.parametrize("dtype,zeros,group", [(F32, True, 64), (F16, True, 128), (F16, False, 32), (BF16, True, 32), (BF16, False, 64), (BF16, False, 128)])
def test_several_tokens(blas, batch, dtype, zeros, group):
    for M, N in ((1, 130), (45, 1000), (100, 2309), (18, 9001)):
        check(blas, batch, M, N, group, dtype, zeros, batch + M, pad=batch % 3)


@pytest.mark.parametrize("batch", [1, 3, 9])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_strides_and_scaling(blas, batch, dtype):
    check(blas, batch, 77, 1023, 64, dtype, True, 5, alpha=-0.75, beta=0.5, ldq_extra=12, ldg_extra=3, pad=5)
    check(blas, batch, 40, 513, 128, dtype, False, 6, alpha=2.0, beta=1.0, ldq_extra=4, ldg_extra=1)
    check(blas, batch, 40, 600, 32, dtype, False, 7, alpha=0.0, beta=1.0)


@pytest.mark.parametrize("batch", [1, 6])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_tokens_with_a_large_mean(blas, batch, dtype):
    """The offset of the nibbles must not cost accuracy where x has one sign."""
    check(blas, batch, 50, 3000, 128, dtype, False, 8, offset=8.0)
    check(blas, batch, 50, 3000, 64, dtype, True, 9, offset=-8.0)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_a_token_gets_the_same_bits_in_any_place(blas, dtype):
    """Within one kernel form, a token's product does not depend on its neighbours."""
    q, s, z = make(200, 3001, 64, dtype, True, 3)
    for batch in (4, 16):
        x = torch.randn(batch, 3001, device="cuda").to(dtype)
        y = torch.empty(batch, 200, dtype=dtype, device="cuda")
        blas.w4_gemv(batch, 200, 3001, 64, 1.0, q, s, z, x, 0.0, y)
        r = torch.empty_like(y)
        blas.w4_gemv(batch, 200, 3001, 64, 1.0, q, s, z, x.flip(0).contiguous(), 0.0, r)
        assert torch.equal(r.flip(0), y)


def test_empty_products(blas):
    q, s, z = make(5, 64, 32, BF16, False, 1)
    x, y = torch.randn(2, 64, device="cuda").to(BF16), torch.full((2, 5), 3.0, dtype=BF16, device="cuda")
    blas.w4_gemv(0, 5, 64, 32, 1.0, q, s, None, x[:0], 0.0, y[:0])
    assert torch.all(y == 3)
    blas.w4_gemv(2, 5, 0, 32, 1.0, q[:, :0], s[:, :0], None, x[:, :0], 0.5, y)     # no columns: y = beta * y
    assert torch.all(y == 1.5)
    blas.w4_gemv(2, 5, 0, 32, 1.0, q[:, :0], s[:, :0], None, x[:, :0], 0.0, y)
    assert torch.all(y == 0)


@pytest.mark.parametrize("batch", [1, 5])
def test_infinite_and_missing_numbers_stay_in_their_token(blas, batch):
    q, s, _ = make(40, 300, 64, BF16, False, 11)
    x = torch.randn(batch + 1, 300, device="cuda").to(BF16)
    x[-1, 7], x[-1, 200] = float("nan"), float("inf")
    y = torch.empty(batch + 1, 40, dtype=BF16, device="cuda")
    blas.w4_gemv(batch + 1, 40, 300, 64, 1.0, q, s, None, x, 0.0, y)
    assert torch.all(torch.isnan(y[-1])) and torch.all(torch.isfinite(y[:-1]))


@pytest.mark.parametrize("batch", [1, 2, 3, 4, 7])
def test_missing_numbers_of_fp32_tokens(blas, batch):
    """Every infinity and NaN, also one whose upper bits alone are an infinity's, stays in its token and reaches all of it."""
    q, s, _ = make(40, 300, 64, F32, False, 12)
    for bits in (0x7F800000, 0x7F800001, 0x7FC00000, -0x7FFFFF):   # the last: a NaN of negative sign
        x = torch.randn(batch + 1, 300, device="cuda")
        x.view(torch.int32)[-1, 7] = bits
        y = torch.empty(batch + 1, 40, device="cuda")
        blas.w4_gemv(batch + 1, 40, 300, 64, 1.0, q, s, None, x, 0.0, y)
        assert not torch.any(torch.isfinite(y[-1])) and torch.all(torch.isfinite(y[:-1]))


@pytest.mark.parametrize("batch", [1, 3, 4, 16])
@pytest.mark.parametrize("exponent", [-130, -118, -105, 60, 121])
def test_range_of_fp32_tokens(blas, batch, exponent):
    """Values far below one lose at most what is under 2^-133 each, large ones nothing, up to a factor of 64 below the largest."""
    M, N, group = 48, 700, 64
    q, _, _ = make(M, N, group, F32, False, 13)
    s = torch.rand(M, -(-N // group), device="cuda") * 0.02 + 0.01   # below 0.03: sums of 700 stay below 2^127
    g = torch.Generator().manual_seed(14)
    x = (torch.rand(batch, N, generator=g) * 2 - 1).mul(2.0 ** exponent).cuda()
    y = torch.empty(batch, M, device="cuda")
    blas.w4_gemv(batch, M, N, group, 1.0, q, s, None, x, 0.0, y)
    w, ss = dense(q, s, None, M, N, group)
    ref = x.double() @ (w * ss).t().contiguous()
    worst = (388 * 15 if batch >= 4 else 36 * 30) * (x.double().abs() @ ss.abs().t().contiguous()) + (N / 32 + 16) * (x.double().abs() @ (w * ss).abs().t().contiguous())
    tiny = (2.0 ** -133 * 15 + 2.0 ** -148 * 4) * N * 0.03 + 2.0 ** -148 * N   # and results that are subnormal themselves
    assert torch.all((y.double() - ref).abs() <= U * (worst + 3 * ref.abs()) + tiny)


def test_packed_by_the_host_function(blas):
    """The product with a packed matrix is the product with what the packing stands for."""
    M, N, group = 96, 1100, 64
    W = torch.randn(M, N) / 33
    groups = -(-N // group)
    q, s, z = torch.zeros(M, 560, dtype=torch.uint8), torch.zeros(M, groups, dtype=BF16), torch.zeros(M, groups, dtype=torch.uint8)
    for zeros in (None, z):
        blas.w4_quantize(M, N, group, W, q, s, zeros)
        x = torch.randn(1, N).to(BF16)
        y = torch.empty(1, M, dtype=BF16, device="cuda")
        blas.w4_gemv(1, M, N, group, 1.0, q.cuda(), s.cuda(), None if zeros is None else zeros.cuda(), x.cuda(), 0.0, y)
        # every weight is within a step (|w| <= 5 / 33, scale below (10 / 33) / 7) of its own
        full = x.double() @ W.double().t()
        assert torch.all((y.cpu().double() - full).abs() <= (10 / 33 / 7) * x.double().abs().sum() + 0.01)
        w, ss = dense(q, s, zeros, M, N, group)
        ref = x.double() @ (w * ss).t()
        assert torch.all((y.cpu().double() - ref).abs() <= half(BF16) * ref.abs() + U * 36 * 62 * (x.double().abs() @ ss.abs().t()) + 64 * U * (x.double().abs() @ (w * ss).abs().t()))


def test_rows_beyond_4_gib(blas):
    """Weights whose rows start beyond 2^32 bytes."""
    M, N, stride = 1100, 256, 1 << 22
    buf = torch.zeros(M * stride, dtype=torch.uint8, device="cuda")
    q = buf.view(M, stride)[:, : N // 2]
    q.copy_(torch.randint(0, 256, (M, N // 2), dtype=torch.uint8))
    s = torch.rand(M, 2, device="cuda").to(BF16)
    for batch in (1, 8):
        x = torch.randn(batch, N, device="cuda").to(BF16)
        y, near = torch.empty(batch, M, dtype=BF16, device="cuda"), torch.empty(batch, M, dtype=BF16, device="cuda")
        blas.w4_gemv(batch, M, N, 128, 1.0, q, s, None, x, 0.0, y)
        blas.w4_gemv(batch, M, N, 128, 1.0, q.contiguous(), s, None, x, 0.0, near)
        assert torch.equal(y, near)


def test_refusals(blas):
    q, s, _ = make(8, 64, 32, F16, False, 1)
    x, y = torch.randn(1, 64, device="cuda").half(), torch.empty(1, 8, device="cuda").half()
    for args in ((1, 8, 64, 16, 1.0, q, s, None, x, 0.0, y), (1, 8, 64, 32, 1.0, q, s.float(), None, x, 0.0, y),
                 (1, 8, 64, 32, 1.0, q[:, 1:], s, None, x, 0.0, y), (1, 8, 64, 32, 1.0, q, s, None, x.cpu(), 0.0, y),
                 (1, 9, 64, 32, 1.0, q, s, None, x, 0.0, y), (1, 8, 64, 32, 1.0, q, s, None, x, 0.0, y.t()),
                 (1, 8, 64, 32, 1.0, q, s[:, :1], None, x, 0.0, y)):
        with pytest.raises(blas.HpcdnnError):
            blas.w4_gemv(*args)
