"""Every kernel form of the 4-bit products where its pipelines run: several rows or row tiles to a wave together with many
columns, so that each wave loads ahead over steps, scale segments, panels of x and rows; exact results where the arithmetic
leaves no rounding but the last; numbers below the smallest normal one.

Bounds as in test_w4_gpu.py, with u = 2^-24: 16-bit tokens 36 (one and two tokens) or 132 (matrix cores) roundings of at most
62 u |s| |x| in a group, FP32 tokens 36 of 30 u or 388 of 15 u; u (N / 32 + 16) of sum |s| |q - z| |x| where groups are added."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def half(t):
    return torch.finfo(t).eps / 2


def weights(M, N, group, dtype, zeros, seed):
    """Packed weights on the GPU: q bytes, scales, zero points or None."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    groups = -(-N // group)
    q = torch.randint(0, 256, (M, -(-((N + 1) // 2) // 4) * 4), generator=g, device="cuda", dtype=torch.uint8)
    s = (torch.randn(M, groups, generator=g, device="cuda") * 0.05).to(dtype)
    z = torch.randint(0, 16, (M, groups), generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    return q, s, z


def rows64(q, s, z, rows, N, group):
    """q - z and s of the given rows, a value per column, in 64 bits."""
    q = q[rows]
    w = torch.stack((q & 15, q >> 4), 2).view(len(rows), -1)[:, :N].double()
    zero = 8.0 if z is None else z[rows].double().repeat_interleave(group, 1)[:, :N]
    return w - zero, s[rows].double().repeat_interleave(group, 1)[:, :N]


def matrix_cores(batch, dtype):
    return batch >= (4 if dtype == F32 else 3)


def check_rows(blas, batch, M, N, group, dtype, packed, x):
    """The product with all M rows; some of them against 64 bits, the first and the last among them."""
    q, s, z = packed
    y = torch.full((batch, M), float("nan"), dtype=dtype, device="cuda")
    blas.w4_gemv(batch, M, N, group, 1.0, q, s, z, x, 0.0, y)
    some = torch.arange(0, M, 257, device="cuda")
    rows = torch.unique(torch.cat((torch.arange(min(M, 18), device="cuda"), some, torch.arange(max(0, M - 34), M, device="cuda"))))
    w, ss = rows64(q, s, z, rows, N, group)
    x64 = x.double()
    ref = x64 @ (w * ss).t().contiguous()
    chain = 388 * 15 if matrix_cores(batch, dtype) else 36 * 30
    if dtype != F32:
        chain = (132 if matrix_cores(batch, dtype) else 36) * 62
    worst = chain * (x64.abs() @ ss.abs().t().contiguous()) + (N / 32 + 16) * (x64.abs() @ (w * ss).abs().t().contiguous())
    tol = half(dtype) * ref.abs() + U * (worst + 3 * ref.abs()) + (2.0 ** -25 if dtype == F16 else 0)
    got = y[:, rows].double()
    assert torch.all((got - ref).abs() <= tol), (batch, group, z is not None, float(((got - ref).abs() / tol).max()))
    assert not torch.any(torch.isnan(y))


@pytest.mark.parametrize("M", [4200, 8200, 12500, 16500])
@pytest.mark.parametrize("N", [9001, 20000])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_many_rows_and_columns(blas, M, N, dtype):
    """Two to four rows or row tiles to a wave, of many pieces and units, in every group size, with zero points and without."""
    g = torch.Generator(device="cuda").manual_seed(M + N)
    x = torch.randn(17, N, generator=g, device="cuda").to(dtype)
    for group in (32, 64, 128):
        for zeros in (False, True):
            packed = weights(M, N, group, dtype, zeros, M + group)
            for batch in (1, 2, 3, 7, 16, 17):
                check_rows(blas, batch, M, N, group, dtype, packed, x[:batch])


@pytest.mark.parametrize("dtype,batch,N", [(F32, 1, 40001), (F32, 2, 19000), (F32, 3, 13001), (F16, 1, 76001), (F16, 2, 40000), (BF16, 2, 37001)])
@pytest.mark.parametrize("M", [600, 9000, 16500])
def test_several_panels_and_rows(blas, dtype, batch, N, M):
    """More columns than LDS holds of x, with one, two and four rows to a wave."""
    x = torch.randn(batch, N, device="cuda").to(dtype)
    for group, zeros in ((32, True), (128, False)):
        check_rows(blas, batch, M, N, group, dtype, weights(M, N, group, dtype, zeros, N), x)


@pytest.mark.parametrize("batch", [1, 2, 3, 5, 16, 17])
@pytest.mark.parametrize("M", [48, 4200, 8200, 12500, 16500])
@pytest.mark.parametrize("dtype,group,zeros", [(F32, 32, True), (F32, 64, False), (F32, 128, True), (F16, 32, False), (F16, 128, True), (BF16, 64, True),
                                               (BF16, 128, False)])
def test_one_column_at_a_time(blas, batch, M, dtype, group, zeros):
    """Tokens with a single value, in every column in turn where M is small, and scales that are powers of two.  16-bit tokens: every step but
    the last rounding is exact.  FP32 tokens, whose values fill their 24 bits: on the matrix cores the three parts of
    (q - z) x are added with one rounding that counts, whichever its direction (2 u); else q x and its difference with z x are
    rounded once each."""
    N = 1200 if M == 48 else 20001
    columns = torch.arange(0, N, 1 if M == 48 else 257)
    g = torch.Generator().manual_seed(M + batch)
    q, _, z = weights(M, N, group, dtype, zeros, 5 * M + group)
    groups = -(-N // group)
    s = torch.exp2(torch.randint(-6, 3, (M, groups), generator=g).float()).to(dtype).cuda()
    values = 1 + torch.randint(1, 1 << 23, (len(columns),), generator=g).double() * 2.0 ** -23 if dtype == F32 else torch.rand(len(columns), generator=g).double() + 1
    values = (values * torch.where(torch.rand(len(columns), generator=g) < 0.5, -1, 1)).to(dtype).cuda()
    for first in range(0, len(columns), 64 * batch):
        cols, val = columns[first:first + 64 * batch].cuda(), values[first:first + 64 * batch]
        calls = -(-len(cols) // batch)
        x = torch.zeros(calls * batch, N, dtype=dtype, device="cuda")
        x[torch.arange(len(cols), device="cuda"), cols] = val
        y = torch.empty(calls * batch, M, dtype=dtype, device="cuda")
        for c in range(calls):
            blas.w4_gemv(batch, M, N, group, 1.0, q, s, z, x[c * batch:(c + 1) * batch], 0.0, y[c * batch:(c + 1) * batch])
        nibble = torch.where(cols % 2 == 0, q[:, cols // 2] & 15, q[:, cols // 2] >> 4).double()
        zero = z[:, cols // group].double() if zeros else 8.0
        scale = s[:, cols // group].double()
        ref = ((nibble - zero) * scale * val.double()).t()
        if dtype != F32:
            tol = half(dtype) * ref.abs()
        elif matrix_cores(batch, dtype):
            tol = 2 * U * ref.abs()
        else:
            tol = U * (ref.abs() + (nibble * scale * val.double()).abs().t() * (1 + U))
        bad = (y[:len(cols)].double() - ref).abs() > tol
        assert not torch.any(bad), (int(cols[torch.nonzero(bad)[0, 0]]), int(torch.nonzero(bad)[0, 1]))


@pytest.mark.parametrize("batch", [4, 13, 16, 17])
@pytest.mark.parametrize("M,N", [(48, 1200), (70, 9001), (8200, 4100), (12500, 4100), (16500, 20001)])
def test_lower_bits_of_fp32_tokens(blas, batch, M, N):
    """Columns in pairs of equal weight, the second with the first's upper 16 bits and the other sign: what is left is the lower
    bits' product.  Upper parts are multiples of 2^-7 below 2, so their sums of a group are exact and vanish, and every rounding is of what the
    lower parts add up to, |x_lower| < 2^-7: 388 (2 u of each, whatever the direction) per group and one per group and wave."""
    group = 64
    q, s, z = weights(M, N, group, F32, True, N)
    q = (q & 15) * 17                                          # both columns of a byte
    s = s.abs()
    g = torch.Generator(device="cuda").manual_seed(batch)
    x = torch.rand(batch, N + N % 2, generator=g, device="cuda") + 1
    x[:, 1::2] = -(x[:, 0::2].contiguous().view(torch.int32) & -65536).view(F32)
    x = x[:, :N].contiguous()
    if N % 2:
        x[:, -1] = 0                                           # a column without a partner
    y = torch.empty(batch, M, device="cuda")
    blas.w4_gemv(batch, M, N, group, 1.0, q, s, z, x, 0.0, y)
    rows = torch.arange(0, M, max(1, M // 100), device="cuda")
    w, ss = rows64(q, s, z, rows, N, group)
    x64 = x.double()
    ref = x64 @ (w * ss).t().contiguous()
    lower = (x64[:, 0:N - 1:2] + x64[:, 1:N:2]).abs()
    size = lower @ (w * ss)[:, 0:N - 1:2].abs().t().contiguous()
    tol = U * (2 * 388 + N / 32 + 16) * size
    assert torch.all((y[:, rows].double() - ref).abs() <= tol)
    assert float((2.0 ** -16 * (x64[:, 0:N - 1:2].abs() @ (w * ss)[:, 0:N - 1:2].abs().t().contiguous()) / tol).min()) > 0.1   # the bound sees the last part


@pytest.mark.parametrize("batch", [1, 2, 3, 8, 16, 17])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("M,N", [(48, 700), (4200, 2100), (16500, 300)])
def test_subnormal_fp16_tokens(blas, batch, zeros, M, N):
    """FP16 values below 2^-14, down to the smallest, count in full."""
    group = 64
    q, s, z = weights(M, N, group, F16, zeros, 17)
    s = s * 20
    g = torch.Generator(device="cuda").manual_seed(batch)
    for top in (2, 30, 1024):                                   # values of at most that many times 2^-24
        x = (torch.randint(-top + 1, top, (batch, N), generator=g, device="cuda").float() * 2.0 ** -24).half()
        check_rows(blas, batch, M, N, group, F16, (q, s, z), x)


@pytest.mark.parametrize("batch", [1, 2, 3, 8, 16, 17])
@pytest.mark.parametrize("zeros", [False, True])
def test_subnormal_bf16_tokens(blas, batch, zeros):
    """BF16 values below 2^-126 count in full too: they and their products with q are whole multiples of 2^-133, which FP32
    sums hold exactly."""
    M, N, group = 200, 700, 64
    q, _, z = weights(M, N, group, BF16, zeros, 18)
    s = torch.full((M, -(-N // group)), 2.0 ** 100, dtype=BF16, device="cuda")
    k = torch.randint(-127, 128, (batch, N), device="cuda")
    x = torch.where(k < 0, -32768 - k, k).to(torch.int16).view(BF16)
    assert torch.equal(x.double(), k.double() * 2.0 ** -133)
    y = torch.empty(batch, M, dtype=BF16, device="cuda")
    blas.w4_gemv(batch, M, N, group, 1.0, q, s, z, x, 0.0, y)
    w, ss = rows64(q, s, z, torch.arange(M, device="cuda"), N, group)
    ref = x.double() @ (w * ss).t().contiguous()
    assert torch.all((y.double() - ref).abs() <= (half(BF16) + 2 * U) * ref.abs())
