"""The layer operators as they are used together: a feed-forward block with experts, forward and backward, its products by
the library's SGEMM; a decode step of norms and 4-bit products; all of it captured into a graph and on a stream of its own."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

EPS = 1e-5


class Block:
    """y[t] = sum_j w[t][j] * (LN(x[t]) @ W[expert j of t]), every buffer allocated once."""

    def __init__(self, blas, tokens, topk, experts, cols, seed):
        g = torch.Generator().manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g).cuda()
        self.blas, self.sizes = blas, (tokens, topk, experts, cols)
        self.x, self.dy = r(tokens, cols) * 2 + 0.5, r(tokens, cols)
        self.w, self.b = 1 + 0.1 * r(cols), 0.1 * r(cols)
        self.W = r(experts, cols, cols) / cols ** 0.5
        self.Wt = self.W.transpose(1, 2).contiguous()
        top = torch.topk(torch.randn(tokens, experts, generator=g), topk, dim=1)
        self.ids = top.indices.to(torch.int32).cuda()
        self.ids[-2:] = -1                                             # padding
        self.weights = torch.softmax(top.values, 1).cuda().contiguous()
        n = tokens * topk
        e = lambda *s, dtype=torch.float32: torch.empty(*s, dtype=dtype, device="cuda")
        self.h, self.mean, self.rstd, self.y, self.dh, self.dx = e(tokens, cols), e(tokens), e(tokens), e(tokens, cols), e(tokens, cols), e(tokens, cols)
        self.hs, self.ys, self.dys, self.dhs = (torch.zeros(n, cols, device="cuda") for _ in range(4))
        self.offsets, self.pos, self.order = e(experts + 1, dtype=torch.int32), e(tokens, topk, dtype=torch.int32), e(n, dtype=torch.int32)
        self.dweights, self.dw, self.db, self.dW = e(tokens, topk), e(cols), e(cols), torch.zeros_like(self.W)
        self.ws = e(max(blas.layer_norm_grad_workspace_bytes(tokens, cols), blas.expert_sort_workspace_bytes(tokens, topk, experts), 16), dtype=torch.uint8)

    def route(self):
        T, k, E, C = self.sizes
        self.blas.layer_norm(T, C, self.x, self.w, self.b, EPS, self.h, self.mean, self.rstd)
        self.blas.expert_sort(T, k, E, self.ids, self.offsets, self.pos, self.order, self.ws)
        self.blas.expert_gather(T, k, T * k, C, self.h, self.pos, self.hs)

    def products(self, rows):
        _, _, E, C = self.sizes
        for e in range(E):
            a, b = rows[e], rows[e + 1]
            self.blas.sgemm(b - a, C, C, self.hs[a:b], self.W[e], self.ys[a:b], 1.0, 0.0)

    def combine(self):
        T, k, E, C = self.sizes
        self.blas.expert_combine(T, k, T * k, C, self.ys, self.pos, self.weights, self.y)

    def backward(self, rows):
        T, k, E, C = self.sizes
        blas = self.blas
        blas.expert_combine_grad(T, k, T * k, C, self.dy, self.ys, self.pos, self.weights, self.dys, self.dweights)
        for e in range(E):
            a, b = rows[e], rows[e + 1]
            blas.sgemm_tn(C, C, b - a, self.hs[a:b], self.dys[a:b], self.dW[e], 1.0, 0.0)
            blas.sgemm(b - a, C, C, self.dys[a:b], self.Wt[e], self.dhs[a:b], 1.0, 0.0)
        blas.expert_combine(T, k, T * k, C, self.dhs, self.pos, None, self.dh)
        blas.layer_norm_grad(T, C, self.dh, self.x, self.w, self.mean, self.rstd, self.dx, self.dw, self.db, self.ws)

    def step(self, rows):
        self.route()
        self.products(rows)
        self.combine()
        self.backward(rows)

    def outputs(self):
        return [t.clone() for t in (self.y, self.dx, self.dw, self.db, self.dW, self.dweights, self.offsets, self.pos)]


def reference(b):
    """The block in float64 on the CPU, gradients by automatic differentiation."""
    leaf = lambda t: t.double().cpu().clone().requires_grad_()
    x, w, bias, W, weights = leaf(b.x), leaf(b.w), leaf(b.b), leaf(b.W), leaf(b.weights)
    mean = x.mean(1, keepdim=True)
    h = (x - mean) / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + EPS) * w + bias
    y = torch.zeros_like(x)
    ids = b.ids.cpu()
    for e in range(b.sizes[2]):
        t, j = torch.nonzero(ids == e, as_tuple=True)
        y = y.index_add(0, t, (h[t] @ W[e]) * weights[t, j][:, None])
    y.backward(b.dy.double().cpu())
    return [y.detach(), x.grad, w.grad, bias.grad, W.grad, weights.grad]


@pytest.mark.parametrize("tokens,topk,experts,cols", [(37, 2, 5, 96), (200, 3, 8, 257), (1500, 4, 16, 128)])
def test_expert_block_forward_and_backward(blas, tokens, topk, experts, cols):
    """Relative to the size of the whole result, a stage adds at most (longest sum of a matrix product or column: about
    sqrt(its terms) + 50) u, u = 2^-24; the six stages one after the other, a gradient of the norm tripling what comes
    in (it subtracts two means): 6 * 3 * (sqrt(tokens * topk) + sqrt(cols) + 50) u."""
    b = Block(blas, tokens, topk, experts, cols, cols)
    b.route()
    rows = b.offsets.tolist()
    b.step(rows)
    tol = 18 * ((tokens * topk) ** 0.5 + cols ** 0.5 + 50) * 2.0 ** -24
    for got, want in zip(b.outputs()[:6], reference(b)):
        assert float((got.double().cpu() - want).norm()) <= tol * float(want.norm())
    assert torch.all(b.y[-2:] == 0) and torch.all(b.dweights[-2:] == 0)


def test_expert_block_captured_and_replayed(blas):
    b = Block(blas, 300, 2, 6, 160, 3)
    b.route()
    rows = b.offsets.tolist()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        b.step(rows)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            b.step(rows)
    torch.cuda.synchronize()
    for replay in range(4):
        # other tokens and weights; the choices move within each expert's share, so that the products' sizes stay
        perm = torch.randperm(298).cuda()
        b.ids[:298] = b.ids[:298][perm].clone()
        b.x.mul_(-0.75).add_(0.1 * replay)
        b.w.add_(0.01)
        b.weights.mul_(0.9)
        b.ws.fill_(0x5A)
        for t in (b.y, b.dx, b.dw, b.db, b.dweights):
            t.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = b.outputs()
        b.step(rows)
        torch.cuda.synchronize()
        for i, (g, e) in enumerate(zip(got, b.outputs())):
            assert torch.equal(g, e), (replay, i)


def test_large_sort_and_norm_gradient_captured(blas):
    """The forms with a workspace: several workgroups that read each other's counts, partial sums of many rows."""
    T, k, E, C = 9000, 4, 100, 520
    ids = torch.randint(-1, E, (T, k), dtype=torch.int32).cuda()
    x, dy = torch.randn(T, C, device="cuda").half(), torch.randn(T, C, device="cuda").half()
    w = torch.rand(C, device="cuda")
    o, pos, order = (torch.empty(n, dtype=torch.int32, device="cuda") for n in (E + 1, T * k, T * k))
    y, dx, dw, db = torch.empty_like(x), torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
    mean, rstd = torch.empty(T, device="cuda"), torch.empty(T, device="cuda")
    ws = torch.empty(max(blas.layer_norm_grad_workspace_bytes(T, C), blas.expert_sort_workspace_bytes(T, k, E)), dtype=torch.uint8, device="cuda")

    def step():
        blas.layer_norm(T, C, x, w, None, EPS, y, mean, rstd)
        blas.expert_sort(T, k, E, ids, o, pos, order, ws)
        blas.layer_norm_grad(T, C, dy, x, w, mean, rstd, dx, dw, db, ws)

    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            step()
    for replay in range(4):
        ids.copy_(torch.randint(-1, E, (T, k), dtype=torch.int32))
        x.copy_(torch.randn(T, C))
        order.fill_(-9)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (y, o, pos, order, dx, dw, db)]
        order.fill_(-9)
        step()
        torch.cuda.synchronize()
        for g, e in zip(got, (y, o, pos, order, dx, dw, db)):
            assert torch.equal(g, e), replay


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch", [1, 2, 6])
def test_decode_step(blas, dtype, batch):
    """Norm, 4-bit projection up, 4-bit projection down added to the residual, on a stream of its own and captured.  In 64
    bits from the packed weights; each stage rounds to the type once: half a step H of the normalised row (of size about 1)
    and of the hidden row go through the next product as noise, bounded by H times the sum of magnitudes."""
    C, F, group = 320, 712, 64
    g = torch.Generator().manual_seed(batch)
    mats = []
    for M, N in ((F, C), (C, F)):
        W = torch.randn(M, N, generator=g) / N ** 0.5
        q = torch.zeros(M, -(-N // 8) * 4, dtype=torch.uint8)
        s, z = torch.zeros(M, -(-N // group), dtype=dtype), torch.zeros(M, -(-N // group), dtype=torch.uint8)
        blas.w4_quantize(M, N, group, W, q, s, z)
        both = torch.stack((q & 15, q >> 4), 2).view(M, -1)[:, :N].double()
        full = (both - z.double().repeat_interleave(group, 1)[:, :N]) * s.double().repeat_interleave(group, 1)[:, :N]
        mats.append((q.cuda(), s.cuda(), z.cuda(), full))
    x = torch.randn(batch, C, generator=g).to(dtype).cuda()
    w = torch.rand(C, generator=g).to(dtype).cuda()
    h, u, y = torch.empty_like(x), torch.empty(batch, F, dtype=dtype, device="cuda"), torch.empty_like(x)

    def step():
        y.copy_(x)
        blas.layer_norm(batch, C, x, w, None, EPS, h)
        blas.w4_gemv(batch, F, C, group, 1.0, *mats[0][:3], h, 0.0, u)
        blas.w4_gemv(batch, C, F, group, 1.0, *mats[1][:3], u, 1.0, y)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    eager = y.clone()
    x64 = x.double().cpu()
    m = x64.mean(1, keepdim=True)
    h64 = (x64 - m) / torch.sqrt(((x64 - m) ** 2).mean(1, keepdim=True) + EPS) * w.double().cpu()
    u64 = h64 @ mats[0][3].t()
    y64 = x64 + u64 @ mats[1][3].t()
    H = torch.finfo(dtype).eps / 2 + 60 * 2.0 ** -24     # rounding, and the FP32 sums of a stage
    up, down = mats[0][3].abs(), mats[1][3].abs()
    u_off = 1.01 * H * (h64.abs() @ up.t()) + H * (u64.abs() + 8 * (h64.abs() @ up.t()))
    y_off = u_off @ down.t() + H * (y64.abs() + 8 * (u64.abs() @ down.t()))
    assert torch.all((eager.double().cpu() - y64).abs() <= y_off)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            step()
    for replay in range(3):
        x.mul_(-0.5)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone()
        step()
        torch.cuda.synchronize()
        assert torch.equal(got, y), replay


def test_two_streams_at_once(blas):
    """Calls on two streams share nothing but read-only inputs."""
    T, C = 700, 1000
    x, dy, w = torch.randn(T, C, device="cuda"), torch.randn(T, C, device="cuda"), torch.rand(C, device="cuda")
    mean, rstd = x.mean(1), 1 / x.std(1)

    def make():
        return (torch.empty_like(x), torch.empty_like(w), torch.empty_like(w),
                torch.empty(blas.layer_norm_grad_workspace_bytes(T, C), dtype=torch.uint8, device="cuda"))

    want = make()
    blas.layer_norm_grad(T, C, dy, x, w, mean, rstd, *want[:3], want[3])
    torch.cuda.synchronize()
    streams, sets = [torch.cuda.Stream() for _ in range(2)], [make() for _ in range(2)]
    for _ in range(5):
        for st, b in zip(streams, sets):
            with torch.cuda.stream(st):
                blas.layer_norm_grad(T, C, dy, x, w, mean, rstd, *b[:3], b[3])
    torch.cuda.synchronize()
    for b in sets:
        for got, ref in zip(b[:3], want[:3]):
            assert torch.equal(got, ref)


def test_nothing_is_allocated(blas):
    b = Block(blas, 64, 2, 4, 64, 1)
    b.route()
    rows = b.offsets.tolist()
    views = b.step(rows)  # noqa: F841
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    b.step(rows)
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() == before
    assert np.isfinite(b.y.cpu().numpy()).all()
