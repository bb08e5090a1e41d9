"""The layer operators at the ends of what their documentation allows: the most choices, more tokens than a launch has teams for,
very wide rows, calls without rows or columns, first calls inside a capture, a workspace shared by two graphs, rows that hold
infinities and NaN."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def half(t):
    return torch.finfo(t).eps / 2


def test_sort_of_two_billion_choices(blas):
    """Slots up to 2^31: every slot at the place that names it, places of an expert in slot order."""
    tokens, topk, experts = 34636833, 62, 5                      # 2^31 - 2 slots
    n = tokens * topk
    assert n == 2 ** 31 - 2
    e = lambda k: torch.empty(k, dtype=torch.int32, device="cuda")  # noqa: E731
    ids, pos, order, offsets = e(n).view(tokens, topk), e(n).view(tokens, topk), e(n), e(experts + 1)
    flat, step = ids.view(-1), 1 << 28
    for a in range(0, n, step):
        s = torch.arange(a, min(n, a + step), device="cuda")
        flat[a:a + step] = ((s * 2654435761 >> 13) % (experts + 1) - 1).to(torch.int32)   # -1: nowhere
    order.fill_(-9)
    ws = torch.empty(blas.expert_sort_workspace_bytes(tokens, topk, experts), dtype=torch.uint8, device="cuda")
    blas.expert_sort(tokens, topk, experts, ids, offsets, pos, order, ws)
    counts = torch.zeros(experts, dtype=torch.int64, device="cuda")
    for a in range(0, n, step):
        part = flat[a:a + step]
        for k in range(experts):
            counts[k] += (part == k).sum()
    want = torch.cat((torch.zeros(1, dtype=torch.int64, device="cuda"), counts.cumsum(0)))
    assert torch.equal(offsets.long(), want)
    sent = int(want[-1])
    for a in range(0, n, step):
        place, b = pos.view(-1)[a:a + step], min(n, a + step)
        inside = place >= 0
        assert torch.equal(inside, flat[a:b] >= 0)
        slots = torch.arange(a, b, device="cuda", dtype=torch.int32)
        assert torch.equal(order[place[inside].long()], slots[inside])
        del slots, inside
    for k in range(experts):                                      # slots grow within an expert
        first, last = int(want[k]), int(want[k + 1])
        for a in range(first, last, step):
            part = order[a:min(last, a + step + 1)]
            assert torch.all(part[1:] > part[:-1])
            assert torch.all(flat[part[:: 997].long()] == k)
    assert torch.all(order[sent:] == -9)


@pytest.mark.parametrize("topk", [1, 2])
@pytest.mark.parametrize("dtype,cols", [(F32, 9), (BF16, 6), (F16, 11), (BF16, 5)])
def test_more_tokens_than_teams(blas, topk, dtype, cols):
    """A launch has 2^22 teams of a wave (with one choice, of four tokens each): the tokens beyond are taken in a further turn."""
    tokens = (1 << 22) * (4 if topk == 1 else 1) + 1237
    n = tokens * topk
    g = torch.Generator(device="cuda").manual_seed(cols)
    pos = torch.randperm(n, generator=g, device="cuda").to(torch.int32).view(tokens, topk)
    pos[torch.rand(tokens, topk, generator=g, device="cuda") < 0.05] = -1
    sent, p = pos >= 0, pos.clamp(min=0).long()
    x = torch.randn(tokens, cols, generator=g, device="cuda").to(dtype)
    out = torch.full((n, cols), 7.0, dtype=dtype, device="cuda")
    blas.expert_gather(tokens, topk, n, cols, x, pos, out)
    want = torch.full_like(out, 7.0)
    for j in range(topk):
        want[p[sent[:, j], j]] = x[sent[:, j]]
    assert torch.equal(out, want)
    w = torch.rand(tokens, topk, generator=g, device="cuda")
    y = torch.empty_like(x)
    blas.expert_combine(tokens, topk, n, cols, out, pos, w, y)
    terms = torch.where(sent[..., None], out[p].double() * w.double()[..., None], 0.0)
    tiny = 2.0 ** -25 if dtype == F16 else 0
    assert torch.all((y.double() - terms.sum(1)).abs() <= half(dtype) * terms.sum(1).abs() + (topk + 1) * U * terms.abs().sum(1) + tiny)
    dxs, dw = torch.full_like(out, 7.0), torch.empty_like(w)
    blas.expert_combine_grad(tokens, topk, n, cols, x, out, pos, w, dxs, dw)
    dot = torch.where(sent[..., None], out[p].double() * x.double()[:, None, :], 0.0)
    assert torch.all((dw.double() - dot.sum(2)).abs() <= 25 * U * dot.abs().sum(2)) and torch.all(dw[~sent] == 0)
    full = x.double()[:, None, :] * w.double()[..., None]
    assert torch.all(((dxs[p].double() - full).abs() <= (half(dtype) + U) * full.abs() + tiny)[sent])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("cols", [1 << 20, 999999])
def test_very_wide_expert_rows(blas, dtype, cols):
    tokens, topk, n = 3, 2, 7
    pos = torch.tensor([[6, 0], [-1, 3], [5, 1]], dtype=torch.int32, device="cuda")
    x = torch.randn(tokens, cols, device="cuda").to(dtype)
    xs = torch.full((n, cols), 3.0, dtype=dtype, device="cuda")
    blas.expert_gather(tokens, topk, n, cols, x, pos, xs)
    for row, t in ((6, 0), (0, 0), (3, 1), (5, 2), (1, 2)):
        assert torch.equal(xs[row], x[t])
    assert torch.all(xs[2] == 3) and torch.all(xs[4] == 3)
    y = torch.empty_like(x)
    blas.expert_combine(tokens, topk, n, cols, xs, pos, None, y)
    assert torch.equal(y[0], (2 * x[0].float()).to(dtype)) and torch.equal(y[1], x[1])
    dw = torch.empty(tokens, topk, device="cuda")
    blas.expert_combine_grad(tokens, topk, n, cols, x, xs, pos, None, None, dw)
    want = (x.double() ** 2).sum(1)
    # cols / 256 additions to a thread, lanes and waves: see test_experts_gpu.py
    assert torch.all((dw[0].double() - want[0]).abs() <= (cols / 256 + 24) * U * want[0])
    assert float(dw[1, 0]) == 0


def test_calls_without_rows_or_columns(blas):
    pos = torch.tensor([[0, 1], [-1, 2]], dtype=torch.int32, device="cuda")
    none, dw = torch.empty(2, 0, device="cuda"), torch.full((2, 2), 5.0, device="cuda")
    blas.expert_combine_grad(2, 2, 3, 0, none, torch.empty(3, 0, device="cuda"), pos, None, None, dw)
    assert torch.all(dw == 0)
    dy, dw = torch.randn(2, 30, device="cuda"), torch.full((2, 2), 5.0, device="cuda")
    empty = torch.empty(0, 30, device="cuda")
    blas.expert_combine_grad(2, 2, 0, 30, dy, empty, pos, None, empty.clone(), dw)
    assert torch.all(dw == 0)
    y = torch.full((2, 30), 5.0, device="cuda")
    blas.expert_combine(2, 2, 0, 30, empty, pos, None, y)
    assert torch.all(y == 0)
    blas.expert_gather(2, 2, 0, 30, dy, pos, empty)
    blas.expert_gather(0, 2, 2, 30, dy[:0], pos[:0], y)
    blas.layer_norm(0, 30, empty, None, None, 1e-5, empty.clone())
    blas.layer_norm(2, 0, none, None, None, 1e-5, none.clone())
    torch.cuda.synchronize()
    assert torch.all(y == 0)


@pytest.mark.parametrize("dtype,batch,N", [(F32, 1, 30000), (F16, 2, 30000), (BF16, 1, 60000)])
def test_a_first_call_inside_a_capture(blas, dtype, batch, N):
    """Also of the forms that take more than 64 KiB of LDS, which a kernel has to be allowed once."""
    M, group = 3000, 128
    g = torch.Generator(device="cuda").manual_seed(N)
    q = torch.randint(0, 256, (M, N // 2), generator=g, dtype=torch.uint8, device="cuda")
    s = torch.rand(M, -(-N // group), generator=g, device="cuda").to(dtype)
    x = torch.randn(batch, N, generator=g, device="cuda").to(dtype)
    y = torch.zeros(batch, M, dtype=dtype, device="cuda")
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            blas.w4_gemv(batch, M, N, group, 1.0, q, s, None, x, 0.0, y)
    for replay in range(3):
        x.mul_(-0.5)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = torch.empty_like(y)
        blas.w4_gemv(batch, M, N, group, 1.0, q, s, None, x, 0.0, want)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and float(y.float().abs().max()) > 0, replay


def test_two_graphs_share_a_workspace(blas):
    """Replayed in turn on one stream: nothing in the workspace outlives a call."""
    T, k, E, C = 6000, 2, 31, 520
    x, dy, w = torch.randn(T, C, device="cuda"), torch.randn(T, C, device="cuda"), torch.rand(C, device="cuda")
    mean, rstd = x.mean(1), 1 / x.std(1)
    ids = torch.randint(-1, E, (T, k), dtype=torch.int32, device="cuda")
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
    offsets, pos = torch.empty(E + 1, dtype=torch.int32, device="cuda"), torch.empty_like(ids)
    ws = torch.empty(max(blas.layer_norm_grad_workspace_bytes(T, C), blas.expert_sort_workspace_bytes(T, k, E)), dtype=torch.uint8, device="cuda")
    calls = (lambda: blas.layer_norm_grad(T, C, dy, x, w, mean, rstd, dx, dw, db, ws), lambda: blas.expert_sort(T, k, E, ids, offsets, pos, None, ws))
    for call in calls:
        call()
    torch.cuda.synchronize()
    want = [t.clone() for t in (dx, dw, db, offsets, pos)]
    graphs, side = [torch.cuda.CUDAGraph() for _ in calls], torch.cuda.Stream()
    with torch.cuda.stream(side):
        for graph, call in zip(graphs, calls):
            with torch.cuda.graph(graph, stream=side):
                call()
        for order in ((0, 1), (1, 0), (0, 0, 1, 1), (1, 0, 1)):
            for t in (dx, dw, db, offsets, pos):
                t.fill_(-7)
            for i in order:
                graphs[i].replay()
            side.synchronize()
            for got, ref in zip((dx, dw, db, offsets, pos), want):
                assert torch.equal(got, ref), order


@pytest.mark.parametrize("rows,cols", [(40, 300), (700, 1001), (300, 4096), (30, 12000)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_gradient_rows_with_infinities_and_nan_stay_alone(blas, rows, cols, dtype):
    """dx of the other rows has the same bits as without them; dw and db have NaN where the formula has it."""
    g = torch.Generator(device="cuda").manual_seed(cols)
    x, dy = (torch.randn(rows, cols, generator=g, device="cuda").to(dtype) for _ in range(2))
    w = torch.rand(cols, generator=g, device="cuda")
    mean, rstd = x.float().mean(1), 1 / x.float().std(1)
    ws = torch.empty(blas.layer_norm_grad_workspace_bytes(rows, cols), dtype=torch.uint8, device="cuda")
    out = lambda: (torch.empty_like(x), torch.empty_like(w), torch.empty_like(w))  # noqa: E731
    clean, bad = out(), out()
    blas.layer_norm_grad(rows, cols, dy, x, w, mean, rstd, *clean, ws)
    x[rows // 2, cols // 3], x[rows - 1, cols - 1], dy[3, 5] = float("inf"), float("nan"), float("-inf")
    mean[9] = float("nan")
    blas.layer_norm_grad(rows, cols, dy, x, w, mean, rstd, *bad, ws)
    hit = torch.zeros(rows, dtype=torch.bool, device="cuda")
    hit[[3, 9, rows // 2, rows - 1]] = True
    assert torch.equal(bad[0][~hit], clean[0][~hit])
    assert not torch.any(torch.isfinite(bad[0][hit][:, 7]))
    assert torch.all(torch.isnan(bad[1]))                        # row 9's xh is NaN in every column
    db_ok = torch.arange(cols, device="cuda") != 5
    assert torch.equal(bad[2][db_ok], clean[2][db_ok]) and float(bad[2][5]) == float("-inf")
