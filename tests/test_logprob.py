"""ops.label_log_probs: CPU path, refusals, and the HIP kernels against the definition in 64 bits.

Tolerances.  A row's sums are chains of at most L = C / 256 + 32 additions of terms that carry about
4 half-ulps each, so s and t have a relative error of at most (L + 4) 2^-24 (t relative to its terms'
size, at most (1 + log C) s).  log p adds the rounding of x − m and of the final difference."""
import math

import numpy as np
import pytest
import torch

from tensorflowdistributedlearning_amd import ops
from tensorflowdistributedlearning_amd.ops.logprob import ref_label_log_probs, MAX_TOP_K

INF = float("inf")


def tol_rows(C):
    return (C / 256 + 40) * 2.0 ** -24 * (1 + math.log(C))


def make(N, C, dtype, seed=0, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(N, C, generator=g) * scale).to(dtype)
    y = torch.randint(0, C, (N,), generator=g)
    return x, y


def exact_grad(x, y, ti, g, h, gt, ignore=-100):
    """Gradient of sum(g log p_y + h H + gt log p_ti) from its formula, 64 bits."""
    lp = torch.log_softmax(x.double(), -1)
    p = lp.exp()
    lp0 = torch.where(p > 0, lp, 0.0)
    H = -(p * lp0).sum(-1)
    valid = (y != ignore).double()
    g = g.double() * valid
    d = -p * (g[:, None] + h.double()[:, None] * (lp0 + H[:, None]))
    d.scatter_add_(1, y.clamp(0, x.shape[1] - 1)[:, None], g[:, None])
    if ti is not None:
        d -= p * gt.double().sum(1, keepdim=True)
        d.scatter_add_(1, ti, gt.double())
    return d


def check_grad(dx, want, x, g, h, gt):
    C = x.shape[1]
    lp = torch.log_softmax(x.double(), -1)
    p = lp.exp()
    lp0 = torch.where(p > 0, lp, 0.0)
    size = g.abs().double() + h.abs().double() * (1 + math.log(C)) * 2
    if gt is not None:
        size = size + gt.abs().double().sum(1)
    # p from three rounded floats: relative 4 tol; h (log p + H) grows with |log p|
    tol = p * (size[:, None] + h.abs().double()[:, None] * lp0.abs()) * \
        (4 * tol_rows(C) + 2.0 ** -22 * (1 + lp0.abs()))
    tol += 2.0 ** -22 * want.abs() + 1e-37
    if dx.dtype == torch.bfloat16:
        tol += want.abs() * torch.finfo(torch.bfloat16).eps / 2 * (1 + 2.0 ** -8) + 1e-38
    err = (dx.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


# ------------------------------------------------------------------------------------------ CPU
def test_cpu_matches_torch_and_gradient_differences():
    x, y = make(5, 9, torch.float32)
    r = ops.label_log_probs(x, y, top_k=4)
    lp = torch.log_softmax(x, -1)
    assert torch.allclose(r.log_prob, lp[range(5), y], atol=1e-6)
    assert torch.allclose(r.entropy, -(lp.exp() * lp).sum(-1), atol=1e-6)
    assert torch.equal(r.top_index, torch.sort(x, 1, descending=True).indices[:, :4])
    xd = x.double().requires_grad_(True)

    def f(t):
        o = ref_label_log_probs(t, y, 3, dtype=torch.float64)
        return o.log_prob, o.entropy, o.top_log_prob
    assert torch.autograd.gradcheck(f, (xd,))
    g, h, gt = torch.randn(5), torch.randn(5), torch.randn(5, 3)
    o = f(xd)
    got, = torch.autograd.grad(o, xd, [g.double(), h.double(), gt.double()])
    ti = torch.sort(x, 1, descending=True).indices[:, :3]
    assert torch.allclose(got, exact_grad(x, y, ti, g, h, gt), atol=1e-12)


def test_cpu_special_rows():
    x = torch.zeros(6, 4)
    x[0] = -INF
    x[1, 1] = float("nan")
    x[2, 3] = INF
    x[3, :3] = -INF
    x[5] = torch.finfo(torch.float32).min
    y = torch.tensor([2, 1, 1, 0, -100, 9])
    x.requires_grad_(True)
    r = ops.label_log_probs(x, y, top_k=2)
    assert r.log_prob[0] == -INF and r.entropy[0] == 0 and r.top_index[0].tolist() == [0, 1]
    assert r.log_prob[1].isnan() and r.log_prob[2].isnan() and r.top_index[1].tolist() == [0, 1]
    assert r.log_prob[3] == -INF and r.entropy[3] == 0 and r.top_index[3].tolist() == [3, 0]
    assert r.log_prob[4] == 0 and r.log_prob[5].isnan()
    assert math.isclose(float(r.entropy[5].detach()), math.log(4), rel_tol=1e-6)
    d, = torch.autograd.grad(r.entropy[0] + r.log_prob[4], x)
    assert bool((d[[0, 3, 4, 5]] == 0).all())  # (rows 1 and 2: 0 times NaN)


def test_refusals():
    x, y = make(4, 10, torch.float32)
    with pytest.raises(ValueError):
        ops.label_log_probs(x, y, top_k=11)
    with pytest.raises(ValueError):
        ops.label_log_probs(torch.zeros(2, 100), None, top_k=MAX_TOP_K + 1)
    with pytest.raises(ValueError):
        ops.label_log_probs(x, y[:3])
    with pytest.raises(TypeError):
        ops.label_log_probs(x, y.float())
    with pytest.raises(TypeError):
        ops.label_log_probs(x.half(), y)
    with pytest.raises(ValueError):
        ops.label_log_probs(torch.zeros(3, 0), None)


def test_empty_batch_and_leading_dimensions():
    r = ops.label_log_probs(torch.zeros(0, 5), torch.zeros(0, dtype=torch.long), top_k=2)
    assert r.log_prob.shape == (0,) and r.top_index.shape == (0, 2)
    x, y = make(12, 7, torch.float32)
    a = ops.label_log_probs(x.view(2, 3, 2, 7), y.view(2, 3, 2), top_k=3)
    b = ops.label_log_probs(x, y, top_k=3)
    assert a.log_prob.shape == (2, 3, 2) and a.top_index.shape == (2, 3, 2, 3)
    assert torch.equal(a.top_log_prob.view(12, 3), b.top_log_prob)


# ------------------------------------------------------------------------------------------ GPU
SIZES = [(1, 1), (3, 1), (5, 2), (70, 7), (1, 8), (33, 9), (65, 16), (1000, 21), (9, 33), (7, 64),
         (5, 65), (19, 127), (6, 129), (3, 256), (4, 300), (129, 1000), (3, 1024), (2, 1025),
         (3, 2047), (2, 2048), (3, 2049), (1, 4096), (2, 8191), (2, 8193), (700, 2500),
         (1, 20001), (3, 50021), (520, 32769), (1, 131072), (1, 131071)]


def check_forward(r, x, y, k, ignore=-100):
    C = x.shape[1]
    xd = x.double()
    lp = torch.log_softmax(xd, -1)
    p = lp.exp()
    ent = -(p * torch.where(p > 0, lp, 0.0)).sum(-1)
    tol = tol_rows(C)
    if y is not None:
        want = torch.where(y == ignore, 0.0, lp.gather(1, y.clamp(0, C - 1)[:, None])[:, 0])
        assert bool(((r.log_prob.double() - want).abs() <= tol + 2.0 ** -22 * want.abs()).all())
    assert bool(((r.entropy.double() - ent).abs() <= 2 * tol).all())
    if k:
        order = torch.sort(x.float() + 0.0, dim=1, descending=True, stable=True).indices[:, :k]
        assert torch.equal(r.top_index, order)
        want = lp.gather(1, order)
        assert bool(((r.top_log_prob.double() - want).abs() <= tol + 2.0 ** -22 * want.abs()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,C", SIZES)
def test_gpu_forward_backward(gpu, N, C, dtype):
    x, y = make(N, C, dtype, seed=N * 7 + C)
    if N > 2:
        y[N // 2] = -100
    x, y = x.to(gpu), y.to(gpu)
    for k in sorted({0, min(C, 1), min(C, 5), min(C, 32)}):
        check_forward(ops.label_log_probs(x, y, top_k=k), x, y, k)
    k = min(C, 3)
    g, h, gt = (torch.randn(*s, device=gpu) for s in ((N,), (N,), (N, k)))
    xg = x.clone().requires_grad_(True)
    r = ops.label_log_probs(xg, y, top_k=k)
    dx, = torch.autograd.grad([r.log_prob, r.entropy, r.top_log_prob], xg, [g, h, gt],
                              retain_graph=True)
    check_grad(dx, exact_grad(x, y, r.top_index, g, h, gt), x, g, h, gt)
    dx, = torch.autograd.grad([r.log_prob], xg, [g])  # one output alone
    check_grad(dx, exact_grad(x, y, None, g, h * 0, None), x, g, h * 0, None)


@pytest.mark.gpu
@pytest.mark.parametrize("C", [5, 21, 100, 1000, 3000, 40000])
def test_gpu_ties_take_the_lowest_index(gpu, C):
    k = min(C, 32)
    g = torch.Generator().manual_seed(C)
    rows = [torch.zeros(C), torch.full((C,), -2.5), torch.randint(0, 3, (C,), generator=g).float(),
            torch.arange(C).float().neg() / 64, torch.arange(C).float() / 64,
            (torch.arange(C) % 2048 < 8).float(), torch.zeros(C)]
    rows[-1][1::2] = -0.0
    x = torch.stack(rows).to(gpu)
    for dt in (torch.float32, torch.bfloat16):
        xt = x.to(dt)
        check_forward(ops.label_log_probs(xt, None, top_k=k), xt, None, k)


@pytest.mark.gpu
def test_gpu_candidates_overflow(gpu):
    """Ascending blocks that put more candidates above the bound than the list holds: the k-pass
    branch."""
    C = 1 << 20
    x = torch.zeros(600, C, device=gpu, dtype=torch.bfloat16)  # one workgroup per row
    lane = torch.arange(C, device=gpu) // 8 % 1024
    x[0] = torch.where(lane < 16 * 8, torch.arange(C, device=gpu) / C + 1, 0.0).to(torch.bfloat16)
    x[599] = torch.where(lane == 3, 1.0, 0.0).to(torch.bfloat16)
    r = ops.label_log_probs(x[[0, 599]].repeat(300, 1), None, top_k=32)
    for i in (0, 1):
        order = torch.sort(x[[0, 599][i]].float(), descending=True, stable=True).indices[:32]
        assert torch.equal(r.top_index[i], order) and torch.equal(r.top_index[598 + i], order)


@pytest.mark.gpu
@pytest.mark.parametrize("C", [3, 21, 500, 1999, 2500, 70000])
def test_gpu_special_rows(gpu, C):
    k = min(C, 4)
    lowest = torch.finfo(torch.bfloat16).min
    x = torch.randn(10, C)
    x[0] = -INF                                  # nothing left
    x[1, C // 2] = float("nan")
    x[2, C - 1] = INF
    x[3] = -INF
    x[3, C - 2] = 1.5                            # one class left
    x[4, ::2] = lowest                           # the type's lowest value as a mask
    x[5] = lowest
    x[6] += 1e4                                  # far offset
    x[7, ::3] = -INF
    x[8] = 3e38
    x[9, 0] = -3e38
    y = torch.tensor([1, 0, 0, C - 2, 1, 2, -100, 1, C, -7])
    for dt in (torch.bfloat16, torch.float32):
        xt = x.to(dt).to(gpu).requires_grad_(True)
        r = ops.label_log_probs(xt, y.to(gpu), top_k=k)
        want = ref_label_log_probs(xt.detach().cpu(), y, k, dtype=torch.float64)
        for got, w in ((r.log_prob, want.log_prob), (r.entropy, want.entropy),
                       (r.top_log_prob, want.top_log_prob)):
            got, w = got.detach().cpu().double(), w.double()
            assert torch.equal(got.isnan(), w.isnan()) and torch.equal(got.isinf(), w.isinf())
            ok = w.isfinite()
            assert bool(((got - w).abs()[ok] <= 2 * tol_rows(C) + 2.0 ** -22 * w.abs()[ok]).all())
        assert torch.equal(r.top_index.cpu(), want.top_index)
        dx, = torch.autograd.grad(r.entropy.sum() + r.log_prob[:8].nan_to_num().sum(), xt)
        assert bool((dx[0] == 0).all()) and bool(dx[1].isnan().all()) and bool(dx[2].isnan().all())
        assert bool(dx[3:8].isfinite().all()) and bool((dx[7, ::3][2:] == 0).all())
        # a gradient through a label out of range is NaN, and only there
        dx, = torch.autograd.grad(
            [ops.label_log_probs(xt, y.to(gpu)).log_prob], xt, [torch.ones(10, device=gpu)])
        assert bool(dx[8:].isnan().all()) and bool(dx[4:8].isfinite().all())


@pytest.mark.gpu
@pytest.mark.parametrize("C", [19, 1000, 5000])
def test_gpu_strides_orders_and_types(gpu, C):
    wide = torch.randn(37, C + 13, device=gpu, dtype=torch.bfloat16)
    y = torch.randint(0, C, (37,), device=gpu, dtype=torch.int32)
    views = [wide[:, 5:5 + C], wide[::2, :C], wide[:, :C].t().contiguous().t(), wide[:1, :C].expand(37, C)]
    for v in views:
        yy = y[: v.shape[0]]
        a, b = (ops.label_log_probs(t, yy, top_k=4) for t in (v, v.contiguous()))
        assert all(torch.equal(p, q) for p, q in zip(a, b))
        leaf = v.detach().requires_grad_(True)  # keeps the strides
        d, = torch.autograd.grad(ops.label_log_probs(leaf, yy).log_prob.sum(), leaf)
        c = v.contiguous().detach().requires_grad_(True)
        w, = torch.autograd.grad(ops.label_log_probs(c, yy).log_prob.sum(), c)
        assert torch.equal(d, w)
    # a gradient that arrives expanded (a sum) or strided
    x = wide[:, :C].contiguous().requires_grad_(True)
    r = ops.label_log_probs(x, y)
    a, = torch.autograd.grad(r.log_prob, x, torch.ones(1, device=gpu).expand(37), retain_graph=True)
    b, = torch.autograd.grad(r.log_prob, x, torch.ones(74, device=gpu)[::2])
    assert torch.equal(a, b)


@pytest.mark.gpu
def test_gpu_repeatable_and_rows_untouched_by_neighbours(gpu):
    x, y = make(300, 9000, torch.bfloat16)
    x, y = x.to(gpu), y.to(gpu)
    a = ops.label_log_probs(x, y, top_k=8)
    b = ops.label_log_probs(x, y, top_k=8)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    x2 = x.clone()
    x2[1::2] = float("nan")
    c = ops.label_log_probs(x2, y, top_k=8)
    assert all(torch.equal(p[::2], q[::2]) for p, q in zip(a, c))


@pytest.mark.gpu
def test_gpu_graph_replays_and_side_stream(gpu):
    x, y = make(4, 40000, torch.bfloat16)
    x, y = x.to(gpu), y.to(gpu)
    xs = x.clone().requires_grad_(True)
    ones = torch.ones(4, device=gpu)

    def step():
        r = ops.label_log_probs(xs, y, top_k=5)
        d, = torch.autograd.grad([r.log_prob, r.entropy], xs, [ones, ones])
        return tuple(t.detach() for t in (*r, d))  # no eager graph of xs lives into the capture
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
        side = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(p, q) for p, q in zip(side, step()))
    graphs = []
    for _ in range(2):  # two graphs: no workspace of one is the other's
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for i in range(4):
        with torch.no_grad():
            xs.copy_(torch.randn_like(x) * (i + 1))
        for g, _ in graphs:
            g.replay()
        want = step()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(p, q) for p, q in zip(out, want))


@pytest.mark.gpu
@pytest.mark.parametrize("N,C", [(70000, 65537), (4300000, 1001)])
def test_gpu_offsets_past_32_bits(gpu, N, C):
    """More than 2^32 logits: rows at both ends equal the same rows alone."""
    x = torch.zeros(N, C, device=gpu, dtype=torch.bfloat16)
    for a in (0, N - 50):
        x[a:a + 50] = torch.randn(50, C, device=gpu).to(torch.bfloat16)
    y = torch.arange(N, device=gpu) * 7 % C
    x.requires_grad_(True)
    r = ops.label_log_probs(x, y, top_k=3)
    d, = torch.autograd.grad(r.log_prob, x, torch.ones(N, device=gpu))
    for a in (0, N - 50):
        part = x.detach()[a:a + 50].clone().requires_grad_(True)
        q = ops.label_log_probs(part, y[a:a + 50], top_k=3)
        e, = torch.autograd.grad(q.log_prob, part, torch.ones(50, device=gpu))
        # (few rows are split over workgroups: another order of additions)
        assert torch.allclose(r.log_prob[a:a + 50], q.log_prob, rtol=0, atol=2 * tol_rows(C))
        assert torch.equal(r.top_index[a:a + 50], q.top_index)
        assert torch.allclose(d[a:a + 50].float(), e.float(), rtol=2.0 ** -7, atol=1e-6)


def test_refuses_rows_past_the_kernels_counters():
    """Shapes only (stride 0): nothing of that size is read."""
    x = torch.zeros(1).expand(1, 2 ** 31 - 100)
    for f in (lambda: ops.label_log_probs(x, torch.zeros(1, dtype=torch.long)),
              lambda: ops.confidence_penalty_cross_entropy(x, torch.zeros(1, dtype=torch.long))):
        with pytest.raises(ValueError, match="classes"):
            f()


@pytest.mark.gpu
def test_gpu_longest_row(gpu):
    """Equal logits: s = C exactly (C = 32767 * 2^16), so log p = -log C to one rounding of each of
    log s and its difference, H = log C, and the gradient is 1 - 1/C at the label, -1/C elsewhere."""
    C = 2 ** 31 - 2 ** 16
    x = torch.zeros(1, C, device=gpu, dtype=torch.bfloat16, requires_grad=True)
    r = ops.label_log_probs(x, torch.tensor([C - 1], device=gpu), top_k=3)
    want = float(np.log(float(C)))
    for got in (-r.log_prob, r.entropy, -r.top_log_prob[:, 2]):
        assert abs(float(got.detach()) - want) <= want * 2.0 ** -22
    assert r.top_index.tolist() == [[0, 1, 2]]
    d, = torch.autograd.grad(r.log_prob, x)
    assert float(d[0, C - 1]) == 1.0
    lo, hi = float(d[0, :C - 1].min()), float(d[0, :C - 1].max())
    assert lo == hi and abs(lo * C + 1) <= 2.0 ** -8 + 2.0 ** -17  # bf16; exp of a log to 2^-22 x 22


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("C", [5, 300, 2500])
def test_gradient_of_labels_out_of_range(C, device):
    """NaN in the whole row where a gradient arrives at such a label's log-probability, none where
    it is zero or another output's; ignored and empty rows have none."""
    x = torch.randn(6, C, generator=torch.Generator().manual_seed(C))
    x[5] = -INF
    y = torch.tensor([1, C, -7, -100, 2 ** 40, C + 3], device=device)
    x = x.to(device).requires_grad_(True)
    bad = torch.tensor([False, True, True, False, True, False])

    def grad(f, *g):
        return torch.autograd.grad(f(), x, *g)[0].cpu()
    d = grad(lambda: ops.label_log_probs(x, y).log_prob.sum())
    assert torch.equal(d.isnan().all(1), bad) and torch.equal(d.isnan().any(1), bad)
    assert bool((d[[3, 5]] == 0).all()) and bool((d[0] != 0).any())
    for k in (0, 2):
        d = grad(lambda: ops.label_log_probs(x, y, top_k=k).log_prob,
                 torch.tensor([1.0, 0, 0, 1, -2, 0], device=device))
        assert d.isnan().all(1).tolist() == [False] * 4 + [True, False] and bool(d[:4].isfinite().all())
        assert bool((d[1:4] == 0).all())
    assert bool(grad(lambda: ops.label_log_probs(x, y, top_k=2).entropy.sum()).isfinite().all())
    loss = ops.confidence_penalty_cross_entropy(x, y, 0.1)
    assert bool(loss.isnan())
    d = grad(lambda: loss)
    assert torch.equal(d.isnan().all(1), bad) and torch.equal(d.isnan().any(1), bad)
