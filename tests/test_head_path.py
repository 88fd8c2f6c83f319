"""The classification head's operators as the models use them: dropout before the classifier,
the entropy-regularised loss, 8-bit linear layers in inference, ranked predictions."""
import copy
import time

import numpy as np
import pytest
import torch

from tensorflowdistributedlearning_amd import models, ops
from tensorflowdistributedlearning_amd.engine.trainer import Trainer
from tensorflowdistributedlearning_amd.models.layers import Dropout, Linear
from tensorflowdistributedlearning_amd.ops.dropout import ref_dropout_keep
from tensorflowdistributedlearning_amd.ops.logprob import ref_label_log_probs


# ------------------------------------------------------------------------------------------ loss
def ref_loss(x, y, w, ignore=-100):
    lp = torch.log_softmax(x.double(), -1)
    counts = y != ignore
    h = -(lp.exp() * lp).sum(-1)
    per = lp.gather(-1, y.clamp_min(0).unsqueeze(-1)).squeeze(-1) + w * h
    return -per[counts].sum() / counts.sum().clamp_min(1)


@pytest.mark.parametrize("w", [0.0, 0.1, -0.2])
def test_confidence_penalty_loss_and_gradient(w):
    x = torch.randn(6, 10, dtype=torch.float32, requires_grad=True)
    y = torch.tensor([1, 2, -100, 0, 9, -100])
    loss = ops.confidence_penalty_cross_entropy(x, y, w)
    xd = x.detach().double().requires_grad_(True)
    want = ref_loss(xd, y, w)
    assert abs(float(loss.detach()) - float(want)) < 1e-5
    g, = torch.autograd.grad(loss, x)
    gd, = torch.autograd.grad(want, xd)
    assert torch.allclose(g.double(), gd, atol=1e-6)
    none = ops.confidence_penalty_cross_entropy(x, torch.full((6,), -100), w)
    assert float(none.detach()) == 0.0
    if w == 0.0:  # equals the framework's cross-entropy where every row counts
        a = ops.confidence_penalty_cross_entropy(x, y.clamp_min(0))
        assert torch.allclose(a, ops.softmax_cross_entropy(x, y.clamp_min(0)), atol=1e-6)


# ------------------------------------------------------------------------------------------ layers
def test_dropout_layer():
    with pytest.raises(ValueError):
        Dropout(1.0)
    d = Dropout(0.5, seed=3)
    x = torch.ones(64, 32)
    a, b = d(x), d(x)
    assert torch.equal(a != 0, ref_dropout_keep(2048, 0.5, torch.tensor([3, 0])).view(64, 32))
    assert not torch.equal(a, b)
    assert torch.equal(Dropout(0.5, seed=3)(x), a)
    d.eval()
    assert d(x) is x
    e = copy.deepcopy(d).train()
    assert torch.equal(e(x) != 0, ref_dropout_keep(2048, 0.5, torch.tensor([3, 2])).view(64, 32))


@pytest.mark.parametrize("arch", ["resnet18", "xception41"])
def test_models_take_dropout(arch):
    torch.manual_seed(0)
    m = models.build(arch, num_classes=7, dropout=0.5)
    assert isinstance(m.drop, Dropout) and not any("drop" in k for k in m.state_dict())
    assert models.build(arch, num_classes=7).drop is None
    x = torch.randn(2, 64, 64, 3)
    m.eval()
    with torch.no_grad():
        assert torch.equal(m(x), m(x))


def test_training_step_with_dropout_and_entropy_term():
    torch.manual_seed(1)
    m = models.resnet18(num_classes=5, dropout=0.3)
    tr = Trainer(m, lambda o, y: ops.confidence_penalty_cross_entropy(o, y, 0.1), "cpu", "sgd",
                 dict(lr=0.01))
    x, y = torch.randn(4, 32, 32, 3), torch.tensor([0, 1, 2, 3])
    for _ in range(2):
        loss, out = tr.train_step(x, y)
        assert bool(torch.isfinite(loss)) and out.shape == (4, 5)
    assert int(m.drop.__dict__["_keys"].state[1]) == 2  # one draw per step
    assert all(bool(torch.isfinite(p.grad).all()) for p in m.parameters())


# ------------------------------------------------------------------------------------------ int8
def int8_bound(x, w, b):
    """How far 8-bit rows and weights can put a linear layer off: half a step on each side."""
    sx = x.abs().amax(1, keepdim=True) / 127
    sw = w.abs().amax(1) / 127
    k = x.shape[1]
    return (sx / 2) * w.abs().sum(1) + (sw / 2) * x.abs().sum(1, keepdim=True) + k * sx * sw / 4


def test_enable_int8_linear():
    torch.manual_seed(2)
    m = torch.nn.Sequential(Linear(96, 11))
    x = torch.randn(5, 96)
    with torch.no_grad():
        full = m.eval()(x)
        assert models.enable_int8(m) == 1
        y = m(x)
        w, b = m[0].conv.weight.view(11, 96), m[0].conv.bias
        assert not torch.equal(y, full)
        assert bool(((y - full).abs() <= int8_bound(x, w, b) * 1.001 + 1e-6).all())
        m[0].conv.weight.mul_(2)
        from tensorflowdistributedlearning_amd.models import params
        params.bump_version()  # as the optimizers and state-dict loads do: laid out again
        assert bool(((m(x) - 2 * y + b).abs() < 1e-4).all())
    assert torch.equal(m(x).detach(), m.train()(x).detach())  # autograd / training: full precision


def test_enable_int8_pointwise_and_export_keep_results():
    torch.manual_seed(3)
    m = models.resnet50(num_classes=6).eval()
    x = torch.randn(2, 64, 64, 3)
    with torch.no_grad():
        full = m(x)
        n = models.enable_int8(m, pointwise=True)
        assert n == 1 + 2 * 16 + 1  # head, conv1 / conv3 of 16 blocks, the stride-1 shortcut
        y = m(x)
    cos = torch.nn.functional.cosine_similarity(y.view(1, -1), full.view(1, -1))
    assert not torch.equal(y, full) and float(cos) > 0.98
    from tensorflowdistributedlearning_amd.engine.serving import export_mode
    with torch.no_grad(), export_mode("portable"):
        assert torch.allclose(m(x), full, atol=1e-3)


# ------------------------------------------------------------------------------------------ Model
def test_model_options_and_ranked_classes(tmp_path):
    from tensorflowdistributedlearning_amd.model import Model
    kw = dict(n_gpus=1, n_fold=2, arch="resnet18", image_size=32, num_classes=4, synthetic=True,
              device="cpu", save_best=0, export_format="none", max_folds=1)
    for bad in (dict(dropout=1.0), dict(arch="deeplab_ref", dropout=0.1),
                dict(arch="deeplab_ref", int8=True)):
        with pytest.raises(ValueError):
            Model(str(tmp_path / "bad"), "none", **{**kw, **bad})
    m = Model(str(tmp_path / "m"), "none", dropout=0.2, entropy_weight=0.05, int8=True, **kw)
    assert m.config()["dropout"] == 0.2
    m.train(16, None, batch_size=4, steps=2)
    p = m.predict_classes(6, 4)
    labels = np.array([0, 1, 2, 3, 0, 1])
    r = m.rank_classes(6, 4, top_k=9, labels=labels)
    assert r["classes"].shape == (6, 4)  # no more alternatives than classes
    order = np.argsort(-p, axis=1, kind="stable")
    assert np.array_equal(r["classes"], order)
    assert np.allclose(r["log_probs"], np.log(np.take_along_axis(p, order, 1)), atol=1e-5)
    assert np.allclose(r["label_log_probs"], np.log(p[np.arange(6), labels]), atol=1e-5)
    assert np.allclose(r["entropy"], -(p * np.log(p)).sum(1), atol=1e-5)
    with pytest.raises(ValueError):
        m.rank_classes(6, 4, top_k=33)


def test_resumed_run_draws_the_same_masks(tmp_path):
    from tensorflowdistributedlearning_amd.model import Model
    kw = dict(n_gpus=1, n_fold=4, arch="resnet18", image_size=32, num_classes=10, synthetic=True,
              device="cpu", save_best=0, export_format="none", max_folds=1, dropout=0.5, lr=0.05,
              lr_schedule="step", lr_decay_steps=3, lr_decay_rate=0.5, save_checkpoints_steps=2)
    whole = Model(str(tmp_path / "a"), "none", **kw).train(64, None, batch_size=8, steps=4)[0]
    Model(str(tmp_path / "b"), "none", **kw).train(64, None, batch_size=8, steps=2)
    rest = Model(str(tmp_path / "b"), "none", **kw).train(64, None, batch_size=8, steps=4)[0]
    np.testing.assert_allclose(rest["train_loss"], whole["train_loss"][2:], rtol=1e-4, atol=1e-5)
    m = Model(str(tmp_path / "b"), "none", **kw)
    for k in (0, -1):
        with pytest.raises(ValueError, match="top_k"):
            m.rank_classes(4, 4, top_k=k)


def test_int8_linear_follows_its_parameter():
    torch.manual_seed(8)
    m = Linear(40, 6).eval()
    models.enable_int8(m)
    x = torch.randn(3, 40)
    with torch.inference_mode():
        a = m(x)
    blocks = m.__dict__["_int8_w"][2].blocks
    with torch.no_grad():
        m.conv.weight.mul_(-1)
        b = m(x)
        assert m.__dict__["_int8_w"][2].blocks is blocks  # written in place
        m.conv.weight = torch.nn.Parameter(-m.conv.weight.detach())  # version 0 like the first one
        c = m(x)
    bias = m.conv.bias.detach()
    assert torch.allclose(b - bias, bias - a, atol=1e-6) and torch.equal(c, a)


# ------------------------------------------------------------------------------------------ GPU
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,C", [(1, 5), (7, 1000), (4096, 21), (4097, 21), (30000, 3), (65, 9000)])
def test_gpu_confidence_penalty_loss(gpu, N, C, dtype):
    """Loss and gradient against 64 bits.  The rows' values are within tests/test_logprob.py's bound
    (below 2^-14 for these sizes), their mean is taken in 64 bits; a gradient entry
    is a difference of terms of the size (|g| + |h| (1 + log C)) p."""
    gen = torch.Generator().manual_seed(N + C)
    x = (torch.randn(N, C, generator=gen) * 2).to(dtype)
    y = torch.randint(0, C, (N,), generator=gen)
    y[::5] = -100 if N > 1 else y[0]
    for w in (0.0, 0.3):
        xg = x.to(gpu).requires_grad_(True)
        loss = ops.confidence_penalty_cross_entropy(xg, y.to(gpu), w)
        g, = torch.autograd.grad(loss, xg, torch.tensor(1.7, device=gpu))
        xd = x.double().requires_grad_(True)
        want = ref_loss(xd, y, w)
        gd, = torch.autograd.grad(want, xd, torch.tensor(1.7, dtype=torch.float64))
        assert abs(float(loss.detach()) - float(want.detach())) < 2.0 ** -13
        n = int((y != -100).sum())
        tol = 1.7 / n * (1 + w * (1 + np.log(C))) * 2.0 ** -14 + gd.abs() * 2.0 ** -20
        if dtype == torch.bfloat16:
            tol = tol + gd.abs() * torch.finfo(dtype).eps / 2
        assert bool(((g.double().cpu() - gd).abs() <= tol).all())
        assert bool((g[y == -100] == 0).all())
    none = ops.confidence_penalty_cross_entropy(xg, torch.full((N,), -100, device=gpu), 0.3)
    g, = torch.autograd.grad(none, xg)
    assert float(none.detach()) == 0.0 and bool((g == 0).all())


@pytest.mark.gpu
def test_gpu_loss_graph_of_many_rows(gpu):
    """Replayed with eager work in between: nothing in the graph clears memory."""
    x = torch.randn(3, 101, 101, 21, device=gpu, dtype=torch.bfloat16)
    y = torch.randint(0, 21, (3, 101, 101), device=gpu)
    xs = x.clone().requires_grad_(True)

    def step():
        loss = ops.confidence_penalty_cross_entropy(xs, y, 0.1)
        g, = torch.autograd.grad(loss, xs)
        return loss.detach(), g
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            xs.copy_(torch.randn_like(x) * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


@pytest.mark.gpu
def test_gpu_autograd_refusals(gpu):
    """Second derivatives, inputs changed in between, and a capture over a live eager graph."""
    x = torch.randn(4, 50, device=gpu, requires_grad=True)
    y = torch.arange(4, device=gpu)
    for f in (lambda: ops.label_log_probs(x, y).log_prob.sum(),
              lambda: ops.confidence_penalty_cross_entropy(x, y, 0.1)):
        g, = torch.autograd.grad(f(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(g.sum() + x.sum(), x)  # also where another path reaches x
        assert torch.equal(g.detach(), torch.autograd.grad(f(), x)[0])
    z = x.detach().clone().requires_grad_(True)
    out = ops.label_log_probs(z * 1, y).entropy.sum()
    out.backward()  # through a non-leaf
    assert bool(z.grad.isfinite().all())
    v = x.detach().clone().requires_grad_(True)
    r = ops.label_log_probs(v, y)
    with torch.no_grad():
        v.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        r.log_prob.sum().backward()
    live = ops.dropout(x, 0.5, torch.zeros(2, dtype=torch.int64, device=gpu)) + \
        ops.label_log_probs(x, y).entropy[:, None]  # an eager graph of x on this stream
    key = torch.zeros(2, dtype=torch.int64, device=gpu)
    for f in (lambda: ops.label_log_probs(x, y), lambda: ops.dropout(x, 0.5, key),
              lambda: ops.confidence_penalty_cross_entropy(x, y)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            torch.zeros(1, device=gpu)
            with pytest.raises(RuntimeError, match="eager graph of this input is still alive"):
                f()
    del live


@pytest.mark.gpu
def test_gpu_empty_and_one_dimensional_inputs(gpu):
    y0 = torch.zeros(0, dtype=torch.long, device=gpu)
    x0 = torch.zeros(0, 40, device=gpu, requires_grad=True)
    r = ops.label_log_probs(x0, y0, top_k=3)
    assert r.log_prob.shape == (0,) and r.top_index.shape == (0, 3)
    g, = torch.autograd.grad(r.log_prob.sum(), x0)
    assert g.shape == (0, 40)
    assert float(ops.confidence_penalty_cross_entropy(x0, y0).detach()) == 0.0
    v = torch.randn(40, device=gpu)
    one = ops.label_log_probs(v, torch.tensor(3, device=gpu), top_k=2)
    assert one.log_prob.shape == () and one.top_index.shape == (2,)
    assert torch.equal(one.top_log_prob, ops.label_log_probs(v[None], None, top_k=2).top_log_prob[0])
    w = ops.Int8Weight(torch.ones(6, 40, dtype=torch.int8, device=gpu), torch.ones(6, device=gpu))
    assert ops.int8_linear(v, w).shape == (6,)
    assert torch.equal(ops.int8_linear(v, w, residual=torch.ones(6, device=gpu)), ops.int8_linear(v, w) + 1)
    assert ops.int8_linear(torch.zeros(0, 3, 40, device=gpu), w).shape == (0, 3, 6)
    assert ops.quantize_rows(torch.zeros(0, 40, device=gpu)).scale.shape == (0,)
    key = torch.zeros(2, dtype=torch.int64, device=gpu)
    assert ops.dropout(torch.zeros(0, 3, device=gpu), 0.5, key).shape == (0, 3)


@pytest.mark.gpu
def test_gpu_int8_weight_follows_statistics_and_refuses_capture(gpu):
    from tensorflowdistributedlearning_amd.models.layers import ConvBN
    torch.manual_seed(6)
    m = ConvBN(64, 48, 1, 1, 0, relu=True).to(gpu).eval()
    seq = torch.nn.Sequential(m)
    assert models.enable_int8(seq, pointwise=True) == 1
    x = torch.randn(2, 5, 5, 64, device=gpu, dtype=torch.bfloat16)
    with torch.no_grad():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            torch.zeros(1, device=gpu)
            with pytest.raises(RuntimeError, match="before capturing"):
                m(x)
        a = m(x)
        m.train()
        m.bn.running_var.mul_(4)
        m.eval()
        b = m(x)
    assert torch.allclose(b.float() * 2, a.float(), atol=0.02, rtol=0.02)


@pytest.mark.gpu
def test_gpu_head_training_step_and_graph(gpu):
    """Dropout → linear → entropy-regularised loss through the Trainer, eager and captured."""
    torch.manual_seed(4)
    m = models.resnet18(num_classes=37, dropout=0.4)
    tr = Trainer(m, lambda o, y: ops.confidence_penalty_cross_entropy(o, y, 0.1), gpu, "sgd",
                 dict(lr=1e-3))
    x = torch.randn(8, 64, 64, 8, device=gpu, dtype=torch.bfloat16)
    x[..., 3:] = 0
    y = torch.randint(0, 37, (8,), device=gpu)
    y[3] = -100
    loss, out = tr.train_step(x, y)
    want = ref_loss(out.float().cpu(), y.cpu(), 0.1)
    assert abs(float(loss) - float(want)) < 1e-4 * max(1.0, abs(float(want)))
    tr.capture(x, y, warmup=1)
    state = m.drop.__dict__["_keys"].state
    first = int(state[1])
    losses = []
    for i in range(3):
        loss, out = tr.replay()
        torch.cuda.synchronize()
        want = ref_loss(out.float().cpu(), y.cpu(), 0.1)
        assert abs(float(loss) - float(want)) < 1e-4 * max(1.0, abs(float(want)))
        assert int(state[1]) == first + i + 1  # every replay draws its own mask
        losses.append(float(loss))
    tr.release_graph()
    assert len(set(losses)) == 3


@pytest.mark.gpu
@pytest.mark.parametrize("pointwise", [False, True])
def test_gpu_int8_serving_path(gpu, pointwise):
    """Folded ResNet → 8-bit layers → log-probabilities and alternatives, against the same network
    on the CPU path (same 8-bit rule, fp32 elsewhere), and replayed from a graph."""
    torch.manual_seed(5)
    m = models.resnet50(num_classes=101).eval()
    with torch.no_grad():  # distinct logits
        m.fc.conv.weight.mul_(20)
    g = copy.deepcopy(m).to(gpu)
    for net in (m, g):
        models.enable_int8(net, pointwise=pointwise)
    x = torch.randn(4, 64, 64, 3)
    with torch.no_grad():
        a = m(x)
        xg = x.to(gpu, torch.bfloat16)
        b = g(xg)
        cos = torch.nn.functional.cosine_similarity(a.flatten(), b.float().cpu().flatten(), dim=0)
        assert float(cos) > 0.99
        r = ops.label_log_probs(b, torch.arange(4, device=gpu), top_k=5)
        w = ref_label_log_probs(b.cpu(), torch.arange(4), 5, dtype=torch.float64)
        assert torch.equal(r.top_index.cpu(), w.top_index)
        assert torch.allclose(r.log_prob.cpu().double(), w.log_prob, atol=1e-5)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            g(xg)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.label_log_probs(g(xg), None, top_k=5)
        for i in range(3):
            xg.copy_(torch.randn_like(xg))
            graph.replay()
            want = ops.label_log_probs(g(xg), None, top_k=5)
            torch.cuda.synchronize()
            assert torch.equal(out.top_index, want.top_index)
            assert torch.equal(out.top_log_prob, want.top_log_prob)


@pytest.mark.gpu
def test_gpu_capture_refusal_sees_through_reshapes(gpu):
    """Logits of more than two dimensions reach the kernels as a view of the leaf."""
    x = torch.randn(2, 3, 50, device=gpu, requires_grad=True)
    t = torch.randn(3, 50, 4, device=gpu, requires_grad=True)
    y = torch.zeros(2, 3, dtype=torch.long, device=gpu)
    z = torch.zeros(3, 4, dtype=torch.long, device=gpu)
    live = x.sum() + t.sum()
    for f in (lambda: ops.label_log_probs(x, y), lambda: ops.confidence_penalty_cross_entropy(x, y),
              lambda: ops.label_log_probs(t.transpose(1, 2), z)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            torch.zeros(1, device=gpu)
            with pytest.raises(RuntimeError, match="eager graph of this input is still alive"):
                f()
    del live
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):  # without one it is captured
        g, = torch.autograd.grad(ops.label_log_probs(x, y).log_prob.sum(), x)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        want, = torch.autograd.grad(ops.label_log_probs(x, y).log_prob.sum(), x)
        assert torch.equal(g, want)


@pytest.mark.gpu
def test_gpu_int8_graph_follows_the_weights(gpu):
    """A captured forward reads the 8-bit weights of the last eager call, on whichever stream."""
    from tensorflowdistributedlearning_amd.models import params
    torch.manual_seed(7)
    m = Linear(256, 48).to(gpu).eval()
    models.enable_int8(m)
    x = torch.randn(5, 256, device=gpu, dtype=torch.bfloat16)
    with torch.no_grad():
        m(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m(x)
        for i in range(3):
            m.conv.weight.mul_(-1.5)
            params.bump_version()
            torch.cuda.synchronize()
            with torch.cuda.stream(torch.cuda.Stream()):
                want = m(x)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)


def _refolded(m, i):
    """New statistics, affine parameters and weights, as a training phase leaves them."""
    m.train()
    with torch.no_grad():
        m.bn.running_mean.add_(0.5 + i)
        m.bn.running_var.mul_(2.0)
        m.bn.beta.add_(0.25)
        m.conv.weight.mul_(-1.5)
    m.eval()


def test_int8_pointwise_refresh_is_in_place():
    """Weight, scales and folded bias keep their storage over a refold: a graph reads all three."""
    from tensorflowdistributedlearning_amd.models.layers import ConvBN
    torch.manual_seed(9)
    m = ConvBN(24, 10, 1, 1, 0, relu=True).eval()
    assert models.enable_int8(torch.nn.Sequential(m), pointwise=True) == 1
    x = torch.randn(2, 3, 3, 24)
    with torch.no_grad():
        m(x)
        w, b = m.folded_int8(x.dtype, x.device)
        where = [t.data_ptr() for t in (w.blocks, w.scale, b)]
        for i in range(2):
            _refolded(m, i)
            y = m(x)
            w2, b2 = m.folded_int8(x.dtype, x.device)
            assert [t.data_ptr() for t in (w2.blocks, w2.scale, b2)] == where
            wf, bf = m.folded_params(x.dtype, x.device)
            assert torch.equal(b2, bf)
            fresh = ops.int8_linear(x, ops.Int8Weight.quantize(wf.view(10, 24)), bias=bf, relu=True)
            assert torch.equal(y, fresh)


@pytest.mark.gpu
def test_gpu_int8_pointwise_graph_follows_the_fold(gpu):
    """A captured 8-bit ConvBN reads weight, scales and bias of the last eager call."""
    from tensorflowdistributedlearning_amd.models.layers import ConvBN
    torch.manual_seed(10)
    m = ConvBN(64, 48, 1, 1, 0, relu=True).to(gpu).eval()
    models.enable_int8(torch.nn.Sequential(m), pointwise=True)
    x = torch.randn(2, 5, 5, 64, device=gpu, dtype=torch.bfloat16)
    with torch.no_grad():
        old = m(x).clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m(x)
        for i in range(3):
            _refolded(m, i)
            want = m(x)
            torch.full((64, 48), 1e9, device=gpu)  # storage that was released has other contents
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want) and not torch.equal(out, old)


def test_int8_weight_is_made_once_by_two_threads(monkeypatch):
    """Two threads that both find the 8-bit form out of date get the same one: a graph captured with
    either's follows later refreshes."""
    import threading
    from tensorflowdistributedlearning_amd.models import layers
    from tensorflowdistributedlearning_amd.models.layers import ConvBN
    calls, quantize = [], ops.Int8Weight.quantize

    def slow(w):
        calls.append(1)
        time.sleep(0.2)
        return quantize(w)
    monkeypatch.setattr(layers.Int8Weight, "quantize", staticmethod(slow))
    lin, bn = Linear(40, 6).eval(), ConvBN(40, 6, 1, 1, 0).eval()
    models.enable_int8(torch.nn.Sequential(lin, bn), pointwise=True)
    for m, x in ((lin, torch.randn(3, 40)), (bn, torch.randn(1, 3, 1, 40))):
        calls.clear()
        seen = []
        real = layers.int8_linear
        monkeypatch.setattr(layers, "int8_linear", lambda a, w, **k: (seen.append(w), real(a, w, **k))[1])

        def work():
            with torch.no_grad():
                m(x)
        ts = [threading.Thread(target=work) for _ in range(2)]
        for t in ts:
            t.start()
        for t in ts:
            t.join()
        monkeypatch.setattr(layers, "int8_linear", real)
        assert len(calls) == 1 and len(seen) == 2 and seen[0] is seen[1]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["linear", "pointwise"])
def test_gpu_int8_refresh_waits_for_earlier_products(gpu, kind):
    """A product, and a replay, that another stream has queued but not run read the weights of
    their call, not those of a refresh issued after them."""
    from tensorflowdistributedlearning_amd.models import params
    from tensorflowdistributedlearning_amd.models.layers import ConvBN
    torch.manual_seed(11)
    m = (Linear(1024, 512) if kind == "linear" else ConvBN(1024, 512, 1, 1, 0)).to(gpu).eval()
    assert models.enable_int8(torch.nn.Sequential(m), pointwise=True) == 1
    x = torch.randn(300, 1024, device=gpu, dtype=torch.bfloat16)
    if kind == "pointwise":
        x = x.view(3, 10, 10, 1024)
    with torch.no_grad():
        want = m(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m(x)
        for replay in (False, True):
            torch.cuda.synchronize()
            a = torch.cuda.Stream()
            with torch.cuda.stream(a):
                torch.cuda._sleep(20_000_000)  # the refresh below is issued before this ends
                if replay:
                    graph.replay()
                else:
                    got = m(x)
            m.conv.weight.mul_(-1.5)
            params.bump_version()
            new = m(x)
            torch.cuda.synchronize()
            assert torch.equal(out if replay else got, want) and not torch.equal(new, want)
            want = new


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("reentrant", [False, True])
def test_dropout_layer_under_recomputation(reentrant, device):
    """Activation recomputation calls the layer again in the backward pass: without a key it would
    draw another mask than the forward's (refused); with one it is a function of its arguments."""
    from torch.utils.checkpoint import checkpoint
    d = Dropout(0.5, seed=4)
    x = torch.ones(64, 32, device=device, requires_grad=True)
    y = checkpoint(lambda t: d(t * 2) ** 2, x, use_reentrant=reentrant)
    with pytest.raises(RuntimeError, match="draws a new mask"):
        y.sum().backward()
    d.eval()
    checkpoint(lambda t: d(t * 2) ** 2, x, use_reentrant=reentrant).sum().backward()  # no mask
    d.train()
    x.grad = None
    key = d.next_key(device)
    y = checkpoint(lambda t, k: d(t * 2, key=k) ** 2, x, key, use_reentrant=reentrant)
    y.sum().backward()
    keep = ref_dropout_keep(2048, 0.5, key.cpu()).view(64, 32)
    # y = (2 · 2 x)² = 16 where kept, its derivative 2 · 4 x · 4 = 32: exact in fp32
    assert torch.equal(y.detach().cpu(), keep * 16.0) and torch.equal(x.grad.cpu(), keep * 32.0)
    assert torch.equal(d.eval()(x, key=key), x)


def test_dropout_stream_outlives_start_at_and_other_devices():
    """A captured step advances the stream's state at every replay: the state stays where it is for
    as long as the layer lives."""
    d, x, y = Dropout(0.5, seed=3), torch.ones(64), torch.ones(64, device="meta")
    d(x)
    state = d.__dict__["_keys"].state
    d.start_at(7)
    assert torch.equal(d(x) != 0, ref_dropout_keep(64, 0.5, torch.tensor([3, 7])))
    assert d.__dict__["_keys"].state is state and int(state[1]) == 8
    d(y)  # another device in between: neither stream starts again
    assert torch.equal(d(x) != 0, ref_dropout_keep(64, 0.5, torch.tensor([3, 8])))
    assert d.__dict__["_keys"].state is state
    early = Dropout(0.5, seed=3)
    early.start_at(8)
    assert torch.equal(early(x) != 0, ref_dropout_keep(64, 0.5, torch.tensor([3, 8])))


def test_dropout_stream_made_under_inference_mode():
    d, x = Dropout(0.5, seed=3), torch.ones(64, requires_grad=True)
    with torch.inference_mode():
        d(x)
    d(x).sum().backward()
    assert torch.equal(x.grad != 0, ref_dropout_keep(64, 0.5, torch.tensor([3, 1])))


@pytest.mark.gpu
def test_gpu_dropout_start_at_reaches_a_captured_step(gpu):
    d = Dropout(0.5, seed=5)
    x = torch.ones(5000, device=gpu)
    d(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = d(x)
    for first in (20, 3):
        d.start_at(first)
        for i in range(3):
            torch.full((2,), -1, dtype=torch.int64, device=gpu)  # storage that was released
            graph.replay()
            keep = ref_dropout_keep(5000, 0.5, torch.tensor([5, first + i]))
            assert torch.equal(out.cpu() != 0, keep)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_forward_mode_derivatives_are_not_dropped(device):
    """A tangent comes out (the log-probabilities and the loss on the CPU) or the call is refused."""
    import torch.autograd.forward_ad as fw
    x, v = torch.randn(4, 50, device=device), torch.randn(4, 50, device=device)
    y, key = torch.arange(4, device=device), torch.zeros(2, dtype=torch.int64, device=device)
    w = ops.Int8Weight.quantize(torch.randn(50, 50, device=device))
    b = torch.ones(50, device=device)
    with fw.dual_level():
        d, db = fw.make_dual(x, v), fw.make_dual(b, b)
        calls = {"log_probs": lambda: ops.label_log_probs(d, y).log_prob,
                 "loss": lambda: ops.confidence_penalty_cross_entropy(d, y, 0.1),
                 "dropout": lambda: ops.dropout(d, 0.5, key), "rows": lambda: ops.quantize_rows(d),
                 "x": lambda: ops.int8_linear(d, w), "bias": lambda: ops.int8_linear(x, w, db),
                 "residual": lambda: ops.int8_linear(x, w, None, d)}
        for name, f in calls.items():
            if device == "cpu" and name in ("log_probs", "loss"):
                t = fw.unpack_dual(f()).tangent
                xg = x.clone().requires_grad_(True)
                o = (ops.label_log_probs(xg, y).log_prob if name == "log_probs" else
                     ops.confidence_penalty_cross_entropy(xg, y, 0.1))
                want = (torch.autograd.grad(o.sum(), xg)[0] * v).sum()
                assert abs(float(t.sum()) - float(want)) < 1e-4
            else:
                with pytest.raises(RuntimeError):
                    f()
        # a backward pass over tangents (forward over reverse)
        if device != "cpu":
            xg = x.clone().requires_grad_(True)
            for o in (ops.label_log_probs(xg, y).log_prob, ops.label_log_probs(xg, None, 2).top_log_prob,
                      ops.dropout(xg, 0.5, key), ops.confidence_penalty_cross_entropy(xg, y, 0.1)):
                one = torch.ones_like(o)
                with pytest.raises(RuntimeError, match="forward-mode"):
                    torch.autograd.grad(o, xg, fw.make_dual(one, one))
        assert torch.equal(ops.int8_linear(x, w, b), ops.int8_linear(fw.unpack_dual(d).primal, w, b))
    ops.dropout(x, 0.5, key)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("arch", ["xception41", "deeplab", "resnet18"])
def test_enable_int8_counts_the_layers_it_turns(arch, device, monkeypatch):
    from tensorflowdistributedlearning_amd.models import layers
    torch.manual_seed(12)
    if arch == "deeplab":  # five of its ConvBNs write into a slice of a concatenation
        m, x = models.DeepLabResNet(model_name="m", input_shape=(101, 101)), torch.randn(1, 101, 101, 2)
    else:
        m, x = models.build(arch, num_classes=6), torch.randn(1, 64, 64, 3)
    m = m.to(device).eval()
    if device == "cuda":
        x = torch.nn.functional.pad(x, (0, 8 - x.shape[-1])).to(device, torch.bfloat16)
    real, used = layers.int8_linear, set()
    monkeypatch.setattr(layers, "int8_linear", lambda a, w, **k: (used.add(w), real(a, w, **k))[1])
    with torch.no_grad():
        full = m(x)
        assert models.enable_int8(m, pointwise=True) > 0 and not used
        y = m(x)
        assert len(used) == models.enable_int8(m, pointwise=True)
    cos = torch.nn.functional.cosine_similarity(y.float().flatten(), full.float().flatten(), dim=0)
    assert not torch.equal(y, full) and float(cos) > 0.98
