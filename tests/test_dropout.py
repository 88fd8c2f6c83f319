"""ops.dropout: generator, mask statistics, CPU path, refusals, and the HIP kernel against the
CPU's mask and 64-bit products.  A kept value is x times a float scale: two roundings to 24 bits
(the scale's and the product's), then one to the type."""
import pytest
import torch

from tensorflowdistributedlearning_amd import ops
from tensorflowdistributedlearning_amd.ops.dropout import ref_dropout_keep, ref_philox4x32


def key_of(seed, call, device="cpu"):
    return torch.tensor([seed, call], dtype=torch.int64, device=device)


def words(*hexes):
    return [torch.tensor(int(h, 16)) for h in hexes]


@pytest.mark.parametrize("ctr,key,rounds,want", [
    (["0"] * 4, ["0"] * 2, 7, "5f6fb709 0d893f64 4f121f81 4f730a48"),
    (["0"] * 4, ["0"] * 2, 10, "6627e8d5 e169c58d bc57ac4c 9b00dbd8"),
    (["ffffffff"] * 4, ["ffffffff"] * 2, 10, "408f276d 41c83b0e a20bc7c6 6d5451fd"),
    (["243f6a88", "85a308d3", "13198a2e", "03707344"], ["a4093822", "299f31d0"], 10,
     "d16cfe09 94fdcceb 5001e420 24126ea1"),
])
def test_philox_published_answers(ctr, key, rounds, want):
    out = ref_philox4x32(words(*ctr), words(*key), rounds)
    assert " ".join("%08x" % int(v) for v in out) == want


def test_mask_statistics():
    n = 1 << 20
    for p in (0.1, 0.5, 0.9):
        a, b = (ref_dropout_keep(n, p, key_of(11, c)) for c in (0, 1))
        sd = (p * (1 - p) / n) ** 0.5
        for m in (a, b):
            assert abs(float(m.float().mean()) - (1 - p)) < 5 * sd + 2.0 ** -17
        both = float((a & b).float().mean())  # two calls are independent
        assert abs(both - (1 - p) ** 2) < 5 * ((1 - p) ** 2 / n) ** 0.5 + 2.0 ** -15


def test_cpu_forward_backward_and_second_derivative():
    x = torch.randn(7, 13, requires_grad=True)
    k = key_of(5, 2)
    y = ops.dropout(x, 0.25, k)
    keep = ref_dropout_keep(91, 0.25, k).view(7, 13)
    assert torch.equal(y == 0, ~keep) and torch.allclose(y[keep], x[keep] / 0.75)
    g = torch.randn(7, 13, requires_grad=True)
    d, = torch.autograd.grad(y, x, g, create_graph=True)
    assert torch.equal(d, ops.dropout(g, 0.25, k))
    dd, = torch.autograd.grad(d.sum(), g)  # linear: the same mask again
    assert torch.equal(dd, ops.dropout(torch.ones(7, 13), 0.25, k))
    eps = 2.0 ** -6
    num = (ops.dropout(x.detach() + eps, 0.25, k) - ops.dropout(x.detach() - eps, 0.25, k)) / (2 * eps)
    assert torch.allclose(dd, num, atol=1e-4)


def test_edges_and_refusals():
    x = torch.randn(9)
    k = key_of(1, 0)
    assert ops.dropout(x, 0.0, k) is x
    assert bool((ops.dropout(x, 1.0, k) == 0).all())
    assert ops.dropout(torch.zeros(0, 4), 0.5, k).shape == (0, 4)
    bad = torch.full((64,), float("nan"))
    y = ops.dropout(bad, 0.5, k)
    assert bool((y[~ref_dropout_keep(64, 0.5, k)] == 0).all())  # a dropped NaN is 0
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError):
            ops.dropout(x, p, k)
    with pytest.raises(TypeError):
        ops.dropout(x.half(), 0.5, k)
    with pytest.raises(ValueError):
        ops.dropout(x, 0.5, k.int())
    with pytest.raises(ValueError):
        ops.dropout(x, 0.5, torch.zeros(3, dtype=torch.int64))
    xr = x.clone().requires_grad_(True)
    y = ops.dropout(xr, 0.5, k)
    k[1] += 1
    with pytest.raises(RuntimeError):  # another mask than the forward's would be wrong
        y.sum().backward()


def test_key_stream_cpu():
    s = ops.DropoutKeys(42, "cpu", first=7)
    a, b = s.next(), s.next()
    assert a.tolist() == [42, 7] and b.tolist() == [42, 8]


# ------------------------------------------------------------------------------------------ GPU
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (3, 5), (33, 67), (256, 2048),
                                   (2, 5, 7, 24), (1, 1, 1), (1000003,)])
@pytest.mark.parametrize("p", [1e-4, 0.1, 0.5, 0.93, 1.0])
def test_gpu_matches_definition(gpu, shape, dtype, p):
    g = torch.Generator().manual_seed(len(shape) * 100 + shape[0])
    x = torch.randn(*shape, generator=g).to(dtype)
    dy = torch.randn(*shape, generator=g).to(dtype)
    key = key_of(-(0x3B67AE85 << 32) + 17, (3 << 34) + 99)
    keep = ref_dropout_keep(x.numel(), p, key).view(shape)
    cut = round(65536 * p)
    xg = x.to(gpu).requires_grad_(True)
    y = ops.dropout(xg, p, key.to(gpu))
    d, = torch.autograd.grad(y, xg, dy.to(gpu))
    for got, src in ((y, x), (d, dy)):
        want = torch.where(keep, src.double() * (65536 / max(65536 - cut, 1)), 0.0)
        tol = want.abs() * 2.0 ** -23
        if dtype == torch.bfloat16:
            tol += want.abs() * torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -22)
        assert got.dtype == dtype and got.shape == shape
        assert bool(((got.detach().cpu().double() - want).abs() <= tol).all())


@pytest.mark.gpu
def test_gpu_views_alignment_and_strides(gpu):
    k = key_of(3, 4, gpu)
    base = torch.randn(4099, device=gpu)
    for dt in (torch.bfloat16, torch.float32):
        b = base.to(dt)
        for off in (1, 3, 4):
            assert torch.equal(ops.dropout(b[off:], 0.3, k), ops.dropout(b[off:].clone(), 0.3, k))
    m = torch.randn(64, 48, device=gpu)
    assert torch.equal(ops.dropout(m.t(), 0.3, k), ops.dropout(m.t().contiguous(), 0.3, k))
    x = m.clone().requires_grad_(True)
    d, = torch.autograd.grad(ops.dropout(x, 0.3, k).sum(), x)  # an expanded gradient
    assert torch.equal(d, ops.dropout(torch.ones_like(m), 0.3, k))
    with pytest.raises(ValueError):
        ops.dropout(m, 0.3, key_of(3, 4))  # key on another device


@pytest.mark.gpu
def test_gpu_large_index(gpu):
    """More than 2^32 bytes and a tail: the last elements against the CPU's mask."""
    n = (1 << 31) + 11
    x = torch.ones(n, device=gpu, dtype=torch.bfloat16)
    key = key_of(8, 1)
    y = ops.dropout(x, 0.5, key.to(gpu))
    first = n // 8 * 8 - 64
    blk = torch.arange(first // 8, (n + 7) // 8)
    w = ref_philox4x32((blk & 0xFFFFFFFF, blk >> 32, key[1].expand(blk.shape), torch.zeros_like(blk)),
                       (key[0], torch.tensor(0)))
    bits = torch.stack([h for c in w for h in (c & 0xFFFF, c >> 16)], 1).reshape(-1)[: n - first]
    assert torch.equal(y[first:].cpu() != 0, bits >= 32768)


@pytest.mark.gpu
def test_gpu_graph_draws_new_masks(gpu):
    keys = ops.DropoutKeys(9, gpu)
    x = torch.ones(5000, device=gpu, requires_grad=True)

    def step():
        k = keys.next()
        y = ops.dropout(x, 0.5, k)
        d, = torch.autograd.grad(y.sum(), x)
        return k, y.detach(), d  # no eager graph of x lives into the capture
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
        with pytest.raises(RuntimeError):
            ops.DropoutKeys(1, gpu)
    calls, masks = [], []
    for _ in range(4):
        g.replay()
        eager = step()  # eager draws in between take numbers of their own
        torch.cuda.synchronize()
        calls += [int(out[0][1]), int(eager[0][1])]
        assert torch.equal(out[1], ops.dropout(x, 0.5, out[0].clone())) and torch.equal(out[1], out[2])
        masks.append(out[1].detach().clone())
    assert calls == list(range(1, 9))
    assert not any(torch.equal(masks[0], m) for m in masks[1:])


def test_probabilities_that_round_to_one_are_refused():
    """p < 1 within half a step (2^-17) of 1 would drop everything; p = 1 does so by name."""
    from tensorflowdistributedlearning_amd.models.layers import Dropout
    x, k = torch.ones(70000), key_of(1, 0)
    for p in (0.999995, 1 - 2.0 ** -17, 1 - 2.0 ** -53):
        with pytest.raises(ValueError):
            ops.dropout(x, p, k)
        with pytest.raises(ValueError):
            Dropout(p)
    p = 1 - 2.0 ** -16
    y = ops.dropout(x, p, k)
    keep = ref_dropout_keep(70000, p, k)
    assert torch.equal(y, keep * 65536.0) and torch.equal(Dropout(p, seed=1)(x), y)
    assert bool((ops.dropout(x, 1.0, k) == 0).all())
    assert ops.dropout(x, 2.0 ** -18, k) is x  # rounds to 0: nothing is dropped


def test_model_refuses_a_dropout_that_rounds_to_one(tmp_path):
    from tensorflowdistributedlearning_amd.model import Model
    with pytest.raises(ValueError):
        Model(str(tmp_path / "m"), "none", n_gpus=1, n_fold=2, arch="resnet18", image_size=32, num_classes=4,
              synthetic=True, device="cpu", save_best=0, export_format="none", dropout=0.999995)
