"""Tokens sorted by expert and back: places, offsets and copied rows exactly, sums against 64 bits.

A sum over topk choices is added in order: off by (topk + 1) u of the magnitudes (u = 2^-24).  A dot product is added over a
thread's columns (cols / 256, in vectors of at most 8), 6 lanes' steps and 4 waves: k = cols / 256 + 24 roundings."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def half(t):
    return torch.finfo(t).eps / 2


def choices(tokens, topk, experts, seed, dropped=0.1):
    g = torch.Generator().manual_seed(seed)
    ids = (torch.randn(tokens, topk, generator=g).abs() * experts / 2).to(torch.int32)     # few far out: sent nowhere
    ids[torch.rand(tokens, topk, generator=g) < dropped] = -1
    if tokens > 3:
        ids[3] = ids[3, 0]                                                                  # the same expert twice
    return ids


def sort_by_hand(ids, experts):
    flat = ids.reshape(-1).tolist()
    where = [[] for _ in range(experts)]
    for slot, e in enumerate(flat):
        if 0 <= e < experts:
            where[e].append(slot)
    order, offsets = [], [0]
    for w in where:
        order += w
        offsets.append(len(order))
    pos = [-1] * len(flat)
    for place, slot in enumerate(order):
        pos[slot] = place
    return offsets, torch.tensor(pos, dtype=torch.int32).view(ids.shape), order


def sort(blas, ids, experts, ws_fill=0x7F, strided=0):
    tokens, topk = ids.shape
    buf = torch.full((tokens, topk + strided), 1, dtype=torch.int32)
    buf[:, :topk] = ids
    dev = buf.cuda()[:, :topk]
    offsets = torch.full((experts + 1,), -9, dtype=torch.int32, device="cuda")
    pos = torch.full((tokens, topk), -9, dtype=torch.int32, device="cuda")
    order = torch.full((tokens * topk,), -9, dtype=torch.int32, device="cuda")
    ws = torch.full((max(blas.expert_sort_workspace_bytes(tokens, topk, experts), 16),), ws_fill, dtype=torch.uint8, device="cuda")
    blas.expert_sort(tokens, topk, experts, dev, offsets, pos, order, ws)
    return offsets, pos, order, dev, ws


@pytest.mark.parametrize("tokens,topk,experts", [(1, 1, 1), (1, 8, 512), (5, 3, 7), (64, 1, 2), (63, 5, 64), (100, 2, 511), (1024, 4, 128), (1365, 3, 33),
                                                 (1366, 3, 33), (4097, 1, 8), (3000, 8, 256), (40000, 2, 8), (9001, 7, 512), (262145, 5, 60)])
def test_sort(blas, tokens, topk, experts):
    ids = choices(tokens, topk, experts, tokens + topk)
    offsets, pos, order, dev, ws = sort(blas, ids, experts, strided=tokens % 3)
    ro, rp, rorder = sort_by_hand(ids, experts)
    assert offsets.tolist() == ro
    assert torch.equal(pos.cpu(), rp)
    assert order[: len(rorder)].tolist() == rorder
    assert torch.all(order[len(rorder):] == -9)            # behind the last place nothing is written
    # without the list of choices: the same places
    p2, o2 = torch.empty_like(pos), torch.empty_like(offsets)
    blas.expert_sort(tokens, topk, experts, dev, o2, p2, None, ws)
    assert torch.equal(p2, pos) and torch.equal(o2, offsets)


@pytest.mark.parametrize("tokens", [0, 6, 5000])
def test_sort_of_nothing(blas, tokens):
    ids = torch.full((tokens, 2), -1, dtype=torch.int32)
    offsets, pos, order, _, _ = sort(blas, ids, 9)
    assert torch.all(offsets == 0) and torch.all(pos == -1) and torch.all(order == -9)


def test_sort_of_one_expert(blas):
    ids = torch.full((7000, 2), 4, dtype=torch.int32)
    offsets, pos, order, _, _ = sort(blas, ids, 5)
    assert offsets.tolist() == [0, 0, 0, 0, 0, 14000] and torch.equal(pos.view(-1).cpu(), torch.arange(14000, dtype=torch.int32))


def rows(n, cols, dtype, seed, pad=0):
    g = torch.Generator().manual_seed(seed)
    buf = torch.full((n, cols + pad), float("nan"), dtype=dtype)
    buf[:, :cols] = torch.randn(n, cols, generator=g).to(dtype)
    buf = buf.cuda()
    return buf[:, :cols], buf


SIZES = [(1, 1, 1, 1), (3, 2, 4, 8), (7, 8, 16, 1001), (50, 3, 9, 2048), (20, 4, 8, 2050), (33, 2, 64, 4096), (5, 6, 8, 16385), (300, 5, 6, 40), (9, 64, 70, 96),
         (6, 1, 3, 2050), (7, 1, 4, 1001), (61, 1, 5, 200), (33, 1, 4, 3), (1030, 1, 9, 4100)]


@pytest.mark.parametrize("tokens,topk,experts,cols", SIZES)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_gather(blas, tokens, topk, experts, cols, dtype):
    ids = choices(tokens, topk, experts, cols)
    offsets, pos, order, _, _ = sort(blas, ids, experts)
    x, _ = rows(tokens, cols, dtype, 1, pad=tokens % 3)
    n = int(offsets[-1])
    out, buf = rows(tokens * topk, cols, dtype, 2, pad=topk % 3)
    before = buf.clone()
    blas.expert_gather(tokens, topk, tokens * topk, cols, x, pos, out)
    assert torch.equal(out[:n], x[order[:n].long() // topk])
    assert torch.equal(out[n:], before[n:, :cols]) and torch.all(torch.isnan(buf[:, cols:]))
    # a buffer with fewer rows than there are choices: the rest is dropped
    few = n // 2
    short, sbuf = rows(max(few + 2, 1), cols, dtype, 3)
    keep = sbuf.clone()
    blas.expert_gather(tokens, topk, few, cols, x, pos, short)
    assert torch.equal(short[:few], x[order[:few].long() // topk]) and torch.equal(short[few:], keep[few:])


# beside those: a token's choices in one workgroup of the gradient, and in two
@pytest.mark.parametrize("tokens,topk,experts,cols", SIZES + [(5000, 5, 20, 1030), (3000, 5, 20, 2051)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("weighted", [True, False])
def test_combine_and_gradient(blas, tokens, topk, experts, cols, dtype, weighted):
    ids = choices(tokens, topk, experts, cols + 1, dropped=0.3)
    offsets, pos, order, _, _ = sort(blas, ids, experts)
    n = int(offsets[-1])
    xs, xbuf = rows(tokens * topk, cols, dtype, 4, pad=topk % 2)
    xbuf[n:] = float("nan")                                   # places that no choice has are not read
    g = torch.Generator().manual_seed(cols)
    w = torch.rand(tokens, topk, generator=g).cuda() if weighted else None
    y, ybuf = rows(tokens, cols, dtype, 5, pad=tokens % 3)
    blas.expert_combine(tokens, topk, tokens * topk, cols, xs, pos, w, y)
    sent = (pos >= 0)
    p = pos.clamp(min=0).long()
    w64 = w.double() if weighted else torch.ones(tokens, topk, dtype=torch.float64, device="cuda")
    terms = torch.where(sent[..., None], xs.double()[p] * w64[..., None], 0.0)
    ref = terms.sum(1)
    tiny = 2.0 ** -25 if dtype == F16 else 0
    assert torch.all((y.double() - ref).abs() <= half(dtype) * ref.abs() + (topk + 1) * U * terms.abs().sum(1) + tiny)
    assert torch.all(torch.isnan(ybuf[:, cols:]))
    assert torch.all(y[~sent.any(1)] == 0)

    dy, _ = rows(tokens, cols, dtype, 6, pad=1)
    dxs, dbuf = rows(tokens * topk, cols, dtype, 7, pad=2)
    before = dbuf.clone()
    dw = torch.full((tokens, topk), float("nan"), device="cuda")
    blas.expert_combine_grad(tokens, topk, tokens * topk, cols, dy, xs, pos, w, dxs, dw)
    want = torch.zeros(tokens * topk, cols, dtype=torch.float64, device="cuda")
    want[pos[sent].long()] = (dy.double()[:, None, :] * w64[..., None])[sent]
    assert torch.all((dxs[:n].double() - want[:n]).abs() <= (half(dtype) + U) * want[:n].abs() + tiny)
    assert torch.equal(dxs[n:], before[n:, :cols]) and torch.all(torch.isnan(dbuf[:, cols:]))
    prod = torch.where(sent[..., None], xs.double()[p] * dy.double()[:, None, :], 0.0)
    assert torch.all((dw.double() - prod.sum(2)).abs() <= (cols / 256 + 24) * U * prod.abs().sum(2))
    assert torch.all(dw[~sent] == 0)
    # either output alone
    d2, w2 = dxs.clone(), torch.empty_like(dw)
    blas.expert_combine_grad(tokens, topk, tokens * topk, cols, dy, xs, pos, w, d2, None)
    blas.expert_combine_grad(tokens, topk, tokens * topk, cols, dy, xs, pos, w, None, w2)
    assert torch.equal(d2[:n], dxs[:n]) and torch.equal(w2, dw)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_places_out_of_range_are_skipped(blas, dtype):
    tokens, topk, cols, n = 6, 3, 130, 10
    pos = torch.tensor([[0, -1, 9], [10, 2, 3], [-2147483648, 2147483647, 4], [5, 6, 7], [-5, 10, 11], [8, 1, -1]], dtype=torch.int32).cuda()
    x, _ = rows(tokens, cols, dtype, 1)
    out, _ = rows(n, cols, dtype, 2)
    blas.expert_gather(tokens, topk, n, cols, x, pos, out)
    for t in range(tokens):
        for j in range(topk):
            p = int(pos[t, j])
            if 0 <= p < n:
                assert torch.equal(out[p], x[t])
    w = torch.rand(tokens, topk).cuda()
    y = torch.empty_like(x)
    blas.expert_combine(tokens, topk, n, cols, out, pos, w, y)
    ok = ((pos >= 0) & (pos < n)).float()
    ref = x.double() * (w * ok).sum(1).double()[:, None]
    assert torch.all((y.double() - ref).abs() <= (half(dtype) + 6 * U) * ref.abs())
    dw = torch.empty(tokens, topk, device="cuda")
    dxs = torch.full((n + 4, cols), 7.0, dtype=dtype, device="cuda")
    blas.expert_combine_grad(tokens, topk, n, cols, x, out, pos, w, dxs[:n], dw)
    assert torch.all(dw[ok == 0] == 0) and torch.all(dw[ok == 1] > 0) and torch.all(dxs[n:] == 7)
    blas.expert_combine(tokens, topk, 0, cols, out[:0], pos, w, y)
    assert torch.all(y == 0)


def test_gradients_against_differences(blas):
    """combine is linear in the rows and in the weights: a difference over any step is the gradient up to rounding."""
    tokens, topk, experts, cols = 6, 3, 4, 37
    ids = choices(tokens, topk, experts, 3)
    offsets, pos, _, _, _ = sort(blas, ids, experts)
    xs, _ = rows(tokens * topk, cols, F32, 1)
    xs = xs.contiguous()
    w, c = torch.rand(tokens, topk).cuda(), torch.randn(tokens, cols).cuda()
    dxs, dw = torch.zeros_like(xs), torch.empty_like(w)
    blas.expert_combine_grad(tokens, topk, tokens * topk, cols, c, xs, pos, w, dxs, dw)
    y = torch.empty(tokens, cols, device="cuda")

    def loss():
        blas.expert_combine(tokens, topk, tokens * topk, cols, xs, pos, w, y)
        return float((c.double() * y.double()).sum())

    scale = float((c.abs().double() * 3 * 4).sum())
    for t, grad in ((xs, dxs), (w, dw)):
        flat, gf = t.view(-1), grad.view(-1)
        for i in range(0, flat.numel(), max(1, flat.numel() // 19)):
            old = flat[i].clone()
            flat[i] = old + 0.5
            up = loss()
            flat[i] = old - 0.5
            down = loss()
            flat[i] = old
            assert abs(up - down - float(gf[i])) <= 8 * U * scale
    # gather and its gradient: <gather(x), s> = <x, combine(s)> with unit weights
    x, _ = rows(tokens, cols, F32, 9)
    x = x.contiguous()
    out = torch.zeros_like(xs)
    blas.expert_gather(tokens, topk, tokens * topk, cols, x, pos, out)
    n = int(offsets[-1])
    blas.expert_combine(tokens, topk, tokens * topk, cols, xs, pos, None, y)
    left, right = (out[:n].double() * xs[:n].double()).sum(), (x.double() * y.double()).sum()
    assert abs(float(left - right)) <= 8 * U * float((out[:n].abs().double() * xs[:n].abs().double()).sum())


def test_rows_beyond_4_gib(blas):
    cols, stride = 200, 1 << 21
    n = (1 << 31) // stride + 4
    buf = torch.zeros(n * stride, dtype=BF16, device="cuda")
    xs = buf.view(n, stride)[:, :cols]
    pos = torch.tensor([[n - 1, 0], [n - 2, 1]], dtype=torch.int32).cuda()
    x = torch.randn(2, cols, device="cuda").to(BF16)
    blas.expert_gather(2, 2, n, cols, x, pos, xs)
    assert torch.equal(xs[n - 1], x[0]) and torch.equal(xs[n - 2], x[1]) and torch.equal(xs[0], x[0])
    y = torch.empty_like(x)
    blas.expert_combine(2, 2, n, cols, xs, pos, None, y)
    assert torch.equal(y, (2 * x.float()).to(BF16))
    dw = torch.empty(2, 2, device="cuda")
    blas.expert_combine_grad(2, 2, n, cols, x, xs, pos, None, None, dw)
    want = (x.double() ** 2).sum(1)[:, None].expand(2, 2)
    assert torch.all((dw.double() - want).abs() <= 32 * U * want)
