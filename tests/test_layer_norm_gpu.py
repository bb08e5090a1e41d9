"""Layer normalisation and its gradient against the definition in 64 bits.

Bounds, with u = 2^-24 and H = half a step of the stored type relative to the value.  A sum of n terms whose longest
chain of additions is k is off by at most k u times the sum of the magnitudes; a lane adds at most 16 values, a wave 6
and the waves of a row 5 more partial sums, so k = 32 covers a row's sums.  The mean is then off by 32 u mean|x|, which y
sees times rstd |w|; the variance by 64 u of itself, rstd by half of that and a few roundings (40 u)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
# (rows, cols): one token and many, a single column, widths around one and two vectors per lane, around a whole
# workgroup, the widest row, and odd ones whose rows start on any address
SIZES = [(1, 1), (3, 2), (1, 8192), (5, 63), (7, 255), (2, 256), (9, 257), (6, 511), (4, 513), (130, 1000), (33, 1023), (3, 1025), (300, 130),
         (2, 4095), (2, 4097), (3, 6144), (2, 8191), (2, 8200), (1, 16383), (2, 16384), (1025, 96)]


def half(t):
    return torch.finfo(t).eps / 2


def rows_of(rows, cols, dtype, seed, pad=0, offset=0.0):
    """A strided rows x cols tensor inside a larger buffer, and the buffer."""
    g = torch.Generator().manual_seed(seed)
    buf = torch.full((rows, cols + pad), float("nan"), dtype=dtype)
    buf[:, :cols] = (torch.randn(rows, cols, generator=g) * 2 + offset).to(dtype)
    buf = buf.cuda()
    return buf[:, :cols], buf


def forward64(x, w, b, eps):
    x = x.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    xh = (x - mean) * rstd
    w = torch.ones_like(x[0]) if w is None else w.double()
    b = torch.zeros_like(x[0]) if b is None else b.double()
    return mean[:, 0], rstd[:, 0], xh, xh * w + b, w, b


def check_forward(blas, rows, cols, dtype, wtype, seed, pad=0, offset=0.0, params=True, eps=1e-5):
    x, _ = rows_of(rows, cols, dtype, seed, pad, offset)
    g = torch.Generator().manual_seed(seed + 1)
    w = (1 + 0.3 * torch.randn(cols, generator=g)).to(wtype).cuda() if params else None
    b = torch.randn(cols, generator=g).to(wtype).cuda() if params else None
    y, ybuf = rows_of(rows, cols, dtype, seed + 2, pad)
    mean, rstd = torch.full((rows,), float("nan"), device="cuda"), torch.full((rows,), float("nan"), device="cuda")
    blas.layer_norm(rows, cols, x, w, b, eps, y, mean, rstd)
    m, r, xh, ref, w64, b64 = forward64(x, w, b, eps)
    spread = x.double().abs().mean(1)
    assert torch.all((mean.double() - m).abs() <= 33 * U * spread)
    # a mean that is off by d adds d^2 to the variance: beside rounding, relative to var + eps
    drift = (33 * U * spread * r) ** 2
    assert torch.all((rstd.double() - r).abs() <= (40 * U + drift) * r)
    tol = half(dtype) * ref.abs() + U * ((40 * spread * r)[:, None] * w64.abs() + 50 * (xh * w64).abs() + 2 * b64.abs()) + drift[:, None] * (xh * w64).abs()
    tol = tol + (2.0 ** -25 if dtype == F16 else 0)       # half a step of the smallest FP16 numbers
    assert torch.all((y.double() - ref).abs() <= tol)
    if pad:
        assert torch.all(torch.isnan(ybuf[:, cols:]))
    return x, w, b, mean, rstd


@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("dtype,wtype", [(F32, F32), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)])
def test_forward(blas, rows, cols, dtype, wtype):
    check_forward(blas, rows, cols, dtype, wtype, rows * 7 + cols, pad=(rows + cols) % 3)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_forward_without_parameters_or_statistics(blas, dtype):
    check_forward(blas, 5, 321, dtype, F32, 3, pad=2, params=False)
    x, _ = rows_of(4, 100, dtype, 9)
    a, b = torch.empty_like(x), torch.empty_like(x)
    mean, rstd = torch.empty(4, device="cuda"), torch.empty(4, device="cuda")
    blas.layer_norm(4, 100, x, None, None, 1e-5, a, mean, rstd)
    blas.layer_norm(4, 100, x, None, None, 1e-5, b)
    assert torch.equal(a, b)


def test_forward_of_rows_with_a_large_mean(blas):
    # a mean 500 times the spread: sums of squares would lose the variance
    check_forward(blas, 6, 1000, F32, F32, 5, offset=1000.0)
    check_forward(blas, 3, 5000, F32, F32, 6, offset=-1000.0)


@pytest.mark.parametrize("cols", [64, 1000, 5000])
def test_rows_that_are_constant_or_hold_infinities(blas, cols):
    x = torch.randn(4, cols, device="cuda")
    x[0] = 3.25                    # variance 0: y = b
    x[1, cols // 2] = float("inf")
    x[2, 0] = float("nan")
    b = torch.randn(cols, device="cuda")
    y = torch.empty_like(x)
    blas.layer_norm(4, cols, x, None, b, 1e-5, y)
    assert torch.equal(y[0], b)
    assert torch.all(torch.isnan(y[1])) and torch.all(torch.isnan(y[2]))
    assert torch.all(torch.isfinite(y[3]))       # the other rows are not touched by it


def check_grad(blas, rows, cols, dtype, wtype, seed, pad=0, weight=True, ws_fill=float("nan")):
    x, _ = rows_of(rows, cols, dtype, seed, pad, offset=0.5)
    dy, _ = rows_of(rows, cols, dtype, seed + 1, (pad + 1) % 3)
    g = torch.Generator().manual_seed(seed + 2)
    w = (1 + 0.3 * torch.randn(cols, generator=g)).to(wtype).cuda() if weight else None
    mean = x.float().mean(1)
    rstd = 1 / torch.sqrt(x.float().var(1, unbiased=False) + 1e-5)
    dx, dxbuf = rows_of(rows, cols, dtype, seed + 3, pad)
    dw, db = torch.full((cols,), float("nan"), dtype=wtype, device="cuda"), torch.full((cols,), float("nan"), dtype=wtype, device="cuda")
    ws = torch.full((blas.layer_norm_grad_workspace_bytes(rows, cols) // 4,), ws_fill, device="cuda")
    blas.layer_norm_grad(rows, cols, dy, x, w, mean, rstd, dx, dw, db, ws)

    r64, dy64 = rstd.double()[:, None], dy.double()
    xh = (x.double() - mean.double()[:, None]) * r64
    gw = dy64 * (w.double() if weight else 1.0)
    a, c = gw.mean(1, keepdim=True), (gw * xh).mean(1, keepdim=True)
    ref = r64 * (gw - a - xh * c)
    sa, sc = gw.abs().mean(1, keepdim=True), (gw * xh).abs().mean(1, keepdim=True)
    tol = half(dtype) * ref.abs() + U * r64 * (36 * sa + 40 * sc * xh.abs() + 6 * gw.abs()) + (2.0 ** -25 if dtype == F16 else 0)
    assert torch.all((dx.double() - ref).abs() <= tol)
    # a column is added along a team's rows, over the teams of a workgroup (at most 16) and over the workgroups (at most 256,
    # in 32 runs of 8): at most rows + 16 additions that change a sum, beyond 256 rows rows / 256 + 16 + 8 + 32; the wave's
    # own sums and the roundings of xh: 8 more.  Both are below
    k = min(rows, rows / 256 + 128) + 16
    for got, terms in ((dw, dy64 * xh), (db, dy64)):
        want = terms.sum(0)
        assert torch.all((got.double() - want).abs() <= half(wtype) * want.abs() + k * U * terms.abs().sum(0) + (2.0 ** -25 if wtype == F16 else 0))
    if pad:
        assert torch.all(torch.isnan(dxbuf[:, cols:]))
    return dx, dw, db, (dy, x, w, mean, rstd, ws)


@pytest.mark.parametrize("rows,cols", SIZES + [(4099, 72), (2500, 1001)])
@pytest.mark.parametrize("dtype,wtype", [(F32, F32), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)])
def test_gradient(blas, rows, cols, dtype, wtype):
    check_grad(blas, rows, cols, dtype, wtype, rows * 11 + cols, pad=(rows + cols) % 3)


@pytest.mark.parametrize("rows,cols", [(300, 8200), (259, 8195), (513, 5002), (40, 16384), (2050, 4203), (2333, 2306), (2100, 4800)])
@pytest.mark.parametrize("dtype,wtype", [(F32, F32), (F16, F16), (BF16, F32)])
def test_gradient_of_wide_rows(blas, rows, cols, dtype, wtype):
    """One row to a workgroup at a time, more rows than workgroups and fewer; nine waves to a row and many rows."""
    check_grad(blas, rows, cols, dtype, wtype, rows + cols, pad=(rows + cols) % 3)


@pytest.mark.parametrize("rows,cols", [(300, 130), (40, 3000)])
def test_gradient_parts_are_the_same_alone(blas, rows, cols):
    dx, dw, db, (dy, x, w, mean, rstd, ws) = check_grad(blas, rows, cols, BF16, F32, 77)
    one = torch.empty_like(x)
    blas.layer_norm_grad(rows, cols, dy, x, w, mean, rstd, one, None, None)       # no workspace needed
    assert torch.equal(one, dx)
    p, q = torch.empty_like(dw), torch.empty_like(db)
    blas.layer_norm_grad(rows, cols, dy, x, w, mean, rstd, None, p, None, ws)
    blas.layer_norm_grad(rows, cols, dy, x, w, mean, rstd, None, None, q, ws)
    assert torch.equal(p, dw) and torch.equal(q, db)
    again = check_grad(blas, rows, cols, BF16, F32, 77, ws_fill=1e30)             # nothing depends on the workspace's contents
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw) and torch.equal(again[2], db)


def test_gradient_without_weight_or_rows(blas):
    check_grad(blas, 17, 500, F32, F32, 5, weight=False)
    z = torch.empty(0, 12, device="cuda")
    dw, db = torch.full((12,), 7.0, device="cuda"), torch.full((12,), 7.0, device="cuda")
    e = torch.empty(0, device="cuda")
    blas.layer_norm_grad(0, 12, z, z, None, e, e, z, dw, db)
    assert torch.all(dw == 0) and torch.all(db == 0)


@pytest.mark.parametrize("rows,cols", [(5, 24), (3, 700)])
def test_gradient_against_differences(blas, rows, cols):
    """Central differences of the kernel's own forward pass in FP32, L = sum c y.  A step h adds h^2 / 6 of the third
    derivative and the rounding of y (a few u of |y| per element, over 2 h) to the quotient."""
    g = torch.Generator().manual_seed(cols)
    x, c = torch.randn(rows, cols, generator=g).cuda(), torch.randn(rows, cols, generator=g).cuda()
    w, b = (1 + 0.1 * torch.randn(cols, generator=g)).cuda(), torch.randn(cols, generator=g).cuda()
    y, mean, rstd = torch.empty_like(x), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    ws = torch.empty(blas.layer_norm_grad_workspace_bytes(rows, cols), dtype=torch.uint8, device="cuda")
    blas.layer_norm(rows, cols, x, w, b, 1e-5, y, mean, rstd)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    blas.layer_norm_grad(rows, cols, c, x, w, mean, rstd, dx, dw, db, ws)

    def loss(x, w, b):
        blas.layer_norm(rows, cols, x, w, b, 1e-5, y)
        return float((c.double() * y.double()).sum())

    h = 2.0 ** -6
    noise = 8 * U * float((c.abs() * (y.abs() + 3)).double().sum()) / h
    for t, grad in ((x, dx), (w, dw), (b, db)):
        flat, gf = t.view(-1), grad.view(-1)
        for i in range(0, flat.numel(), max(1, flat.numel() // 7)):
            old = flat[i].clone()
            flat[i] = old + h
            up = loss(x, w, b)
            flat[i] = old - h
            down = loss(x, w, b)
            flat[i] = old
            # third derivative of xh along one coordinate: below 30 rstd^3 |c| here (all of order one)
            third = h * h * 5 * float((c.abs() * w.abs()).max()) * float(rstd.max()) ** 3
            assert abs((up - down) / (2 * h) - float(gf[i])) <= noise + third


def test_rows_beyond_4_gib(blas):
    """Rows whose offset passes 2^31 elements and 2^32 bytes."""
    cols, stride = 300, 1 << 21
    rows = (1 << 31) // stride + 3
    buf = torch.zeros(rows * stride, dtype=BF16, device="cuda")
    x = buf.view(rows, stride)[:, :cols]
    x.copy_(torch.randn(rows, cols, device="cuda"))
    y = torch.empty(rows, cols, dtype=BF16, device="cuda")
    blas.layer_norm(rows, cols, x, None, None, 1e-5, y)
    near = torch.empty_like(y)
    blas.layer_norm(rows, cols, x.contiguous(), None, None, 1e-5, near)
    assert torch.equal(y, near)
