"""ops.int8_linear / quantize_rows: CPU path, refusals, and the HIP kernels against the definition in
64 bits.

The quantised values are exact (compared as integers).  An output is the exact integer sum, rounded
to 24 bits, times two rounded scales (their product rounded), plus bias and residual: each of the
at most 7 roundings is 2^-24 of the largest partial result, then one rounding to the type."""
import pytest
import torch

from tensorflowdistributedlearning_amd import ops
from tensorflowdistributedlearning_amd.ops.int8 import (from_blocks, ref_quantize_rows, to_blocks,
                                                        MAX_K)


def make(M, K, N, dtype, seed=0, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(M, K, generator=g) * torch.exp(torch.randn(M, 1, generator=g))).to(dtype)
    wq = torch.randint(-127, 128, (N, K), generator=g).to(torch.int8)
    ws = torch.rand(N, generator=g) / 127 + 1e-4
    bias = torch.randn(N, generator=g)
    res = torch.randn(M, N, generator=g).to(dtype)
    return tuple(t.to(device) for t in (x, wq, ws, bias, res))


def exact(x, wq, ws, bias, res, relu):
    """(y, size of the largest partial result) in 64 bits."""
    xd = x.double().cpu()
    top = xd.abs().amax(1).clamp_min(2.0 ** -40)
    q = torch.round(127 * xd / top[:, None])
    y = (q @ wq.double().cpu().t()) * (top / 127)[:, None] * ws.double().cpu()
    size = y.abs()
    for t in (bias, res):
        if t is not None:
            y = y + t.double().cpu()
            size = size + t.double().cpu().abs()
    return (y.clamp_min(0) if relu else y), size


def check(y, x, wq, ws, bias=None, res=None, relu=False):
    want, size = exact(x, wq, ws, bias, res, relu)
    assert y.dtype == x.dtype and y.shape == want.shape
    tol = 7 * 2.0 ** -24 * size
    if x.dtype == torch.bfloat16:
        tol += (want.abs() + tol) * torch.finfo(torch.bfloat16).eps / 2
    err = (y.double().cpu() - want).abs()
    assert bool((err <= tol).all()), float((err / tol.clamp_min(1e-300)).max())


# ------------------------------------------------------------------------------------------ CPU
def test_block_order_round_trip():
    for r, k in ((1, 1), (16, 64), (17, 130), (50, 1000)):
        q = torch.randint(-127, 128, (r, k)).to(torch.int8)
        p = to_blocks(q)
        assert p.shape[0] % 16 == 0 and p.shape[1] % 128 == 0
        assert torch.equal(from_blocks(p, r, k), q)
    q = torch.arange(16 * 64).remainder(127).to(torch.int8).view(16, 64)
    assert int(to_blocks(q).view(-1)[(1 * 16 + 3) * 16 + 5]) == int(q[3, 16 + 5])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_cpu_linear(dtype):
    x, wq, ws, bias, res = make(9, 33, 11, dtype)
    w = ops.Int8Weight(wq, ws)
    check(ops.int8_linear(x, w), x, wq, ws)
    check(ops.int8_linear(x, w, bias, res, True), x, wq, ws, bias, res, True)
    y = ops.int8_linear(x.view(3, 3, 33), w, bias)
    assert torch.equal(y.view(9, 11), ops.int8_linear(ops.quantize_rows(x), w, bias))


def test_cpu_quantisation_error_and_weights():
    x = torch.randn(5, 200)
    r = ops.quantize_rows(x)
    step = x.abs().amax(1, keepdim=True) / 127
    assert bool(((r.dequantize() - x).abs() <= step / 2 * (1 + 2.0 ** -16)).all())
    w = torch.randn(7, 200)
    iw = ops.Int8Weight.quantize(w)
    assert bool(((iw.dequantize() - w).abs() <= w.abs().amax(1, keepdim=True) / 254 * (1 + 2.0 ** -16)).all())


def test_refusals():
    x, wq, ws, bias, res = make(4, 20, 6, torch.float32)
    w = ops.Int8Weight(wq, ws)
    bad = [lambda: ops.int8_linear(x[:, :19], w), lambda: ops.int8_linear(x, w, bias[:5]),
           lambda: ops.int8_linear(x, w, bias.double()), lambda: ops.int8_linear(x, w, None, res[:3]),
           lambda: ops.int8_linear(x, w, None, res.bfloat16()), lambda: ops.Int8Weight(wq, ws[:3]),
           lambda: ops.Int8Weight(wq.int(), ws), lambda: ops.Int8Weight(wq[0], ws),
           lambda: ops.quantize_rows(torch.zeros(2, 0)), lambda: ops.quantize_rows(torch.tensor(1.0)),
           lambda: ops.Int8Weight(torch.zeros(1, MAX_K + 1, dtype=torch.int8), torch.ones(1))]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    for f in (lambda: ops.int8_linear(x.half(), w), lambda: ops.int8_linear(x, wq)):
        with pytest.raises(TypeError):
            f()
    with pytest.raises(RuntimeError):
        ops.int8_linear(x.clone().requires_grad_(True), w)
    with torch.no_grad():
        ops.int8_linear(x.clone().requires_grad_(True), w)


def test_cpu_special_rows():
    x, wq, ws, bias, _ = make(6, 20, 6, torch.float32)
    x[0] = 0
    x[1, 3] = float("nan")
    x[2, 4] = float("inf")
    x[3] = 1e-30
    x[4] = 3e38
    y = ops.int8_linear(x, ops.Int8Weight(wq, ws), bias, relu=False)
    assert torch.equal(y[0], bias) and bool(y[1:3].isnan().all()) and bool(y[[3, 5]].isfinite().all())
    assert ops.int8_linear(x[:0], ops.Int8Weight(wq, ws)).shape == (0, 6)


# ------------------------------------------------------------------------------------------ GPU
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 2048), (3, 17), (16, 64), (17, 65), (33, 1999), (5, 2049),
                                 (40, 4096), (7, 4100), (18, 8192), (3, 20001), (1000, 256), (2, 131071)])
def test_gpu_quantize_rows(gpu, M, K, dtype):
    x = make(M, K, 1, dtype, seed=M + K)[0]
    if M > 2:
        x[1] = 0
    # ties: halves of the maximum, and steps of a maximum whose scale is a power of two
    x[0, : K // 2] = (torch.randint(-254, 255, (K // 2,)) / 2 ** 9).to(dtype)
    x[0, -1] = 254 / 2 ** 9
    if M > 2:
        x[2, ::2] = x[2].abs().max() / 2
    r = ops.quantize_rows(x.to(gpu))
    q, s = ref_quantize_rows(x)
    assert torch.equal(from_blocks(r.blocks, M, K).cpu(), q)
    assert torch.equal(r.scale.cpu(), s)
    full = from_blocks(r.blocks, *r.blocks.shape).cpu()  # the padding is zero
    assert int(full[M:].abs().sum()) == 0 and int(full[:, K:].abs().sum()) == 0


@pytest.mark.gpu
def test_gpu_quantize_extremes_and_views(gpu):
    for dt in (torch.bfloat16, torch.float32):
        x = torch.randn(40, 300).to(dt)
        x[0] = torch.finfo(dt).max
        x[1, ::2] = torch.finfo(dt).max
        x[2] *= 1e-20
        x[3] = torch.finfo(dt).tiny / 4
        x[4, 299] = float("nan")
        x[5, 0] = -float("inf")
        x[6] *= 1e30
        x[7] = 2.0 ** -40
        q, s = ref_quantize_rows(x)
        r = ops.quantize_rows(x.to(gpu))
        assert torch.equal(from_blocks(r.blocks, 40, 300).cpu(), q)
        assert torch.equal(r.scale.cpu().nan_to_num(-1), s.nan_to_num(-1))
        xg = x.to(gpu)
        for v in (xg[:, 3:203], xg[::3], xg.t(), xg[5:6].expand(9, 300), xg[:, 1:2]):
            a, b = ops.quantize_rows(v), ops.quantize_rows(v.clone(memory_format=torch.contiguous_format))
            assert torch.equal(a.blocks, b.blocks)
            assert torch.equal(a.scale.nan_to_num(-1), b.scale.nan_to_num(-1))


SHAPES = [(1, 1, 1), (1, 2048, 1000), (2, 64, 16), (4, 100, 33), (5, 8192, 257), (15, 333, 70),
          (16, 128, 128), (17, 1000, 1003), (31, 65, 4), (33, 64, 65), (64, 512, 1000), (65, 2048, 96),
          (127, 129, 127), (128, 128, 256), (129, 640, 129), (300, 1999, 301), (513, 256, 1024),
          (1000, 64, 64), (2049, 1999, 1003), (4000, 130, 17), (1, 131071, 3), (260, 20000, 40), (16, 4096, 50), (16, 4100, 50),
          (7, 9000, 20), (48, 5000, 100), (40, 2000, 33), (900, 1100, 3000), (4700, 1100, 2600)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_gpu_linear(gpu, M, K, N, dtype):
    x, wq, ws, bias, res = make(M, K, N, dtype, seed=M + K + N, device=gpu)
    w = ops.Int8Weight(wq, ws)
    assert torch.equal(w.dequantize(), wq.float() * ws[:, None])
    check(ops.int8_linear(x, w), x, wq, ws)
    check(ops.int8_linear(x, w, bias, res, True), x, wq, ws, bias, res, True)
    a = ops.int8_linear(ops.quantize_rows(x), w, bias)
    assert torch.equal(a, ops.int8_linear(x, w, bias))


@pytest.mark.gpu
def test_gpu_extreme_sums(gpu):
    """Every product 127 · 127 at the longest K: the 32-bit sum does not wrap."""
    K = MAX_K
    x = torch.ones(3, K, device=gpu)
    wq = torch.full((5, K), 127, dtype=torch.int8, device=gpu)
    wq[1] = -128
    ws = torch.full((5,), 2.0 ** -20, device=gpu)
    y = ops.int8_linear(x, ops.Int8Weight(wq, ws))
    check(y, x, wq, ws)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 9, 40, 300])
def test_gpu_special_rows_layouts_and_neighbours(gpu, M):
    x, wq, ws, bias, res = make(M, 300, 130, torch.bfloat16, device=gpu)
    w = ops.Int8Weight(wq, ws)
    want = ops.int8_linear(x, w, bias, res, True)
    for t in (x.t().contiguous().t(), torch.cat([x, x], 1)[:, 300:]):
        assert torch.equal(ops.int8_linear(t, w, bias, res, True), want)
    r2 = torch.cat([res, res], 1)[:, :130]  # a strided residual
    assert torch.equal(ops.int8_linear(x, w, bias, r2, True), want)
    x[M // 2, 7] = float("nan")
    y = ops.int8_linear(x, w, bias, res, True)
    keep = torch.arange(M, device=gpu) != M // 2
    assert bool(y[M // 2].isnan().all()) and torch.equal(y[keep], want[keep])
    # storage behind the output is left as it was
    buf = torch.full((M * 130 + 64,), 7.0, device=gpu, dtype=torch.bfloat16)
    rows = ops.quantize_rows(x)
    from tensorflowdistributedlearning_amd.ops.common import ext
    ext().int8_gemm(rows.blocks, rows.scale, w.blocks, w.scale, 300, bias, res, True,
                    buf[: M * 130].view(M, 130))
    assert bool((buf[M * 130:] == 7).all()) and torch.equal(buf[: M * 130].view(M, 130)[keep], want[keep])


@pytest.mark.gpu
def test_gpu_devices_and_entry_checks(gpu):
    x, wq, ws, bias, res = make(4, 64, 6, torch.bfloat16)
    w = ops.Int8Weight(wq.to(gpu), ws.to(gpu))
    for f in (lambda: ops.int8_linear(x, w), lambda: ops.int8_linear(x.to(gpu), w, bias),
              lambda: ops.Int8Weight(wq.to(gpu), ws)):
        with pytest.raises(ValueError):
            f()
    from tensorflowdistributedlearning_amd.ops.common import ext
    rows = ops.quantize_rows(x.to(gpu))
    y = torch.empty(4, 6, device=gpu, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):  # another K than the blocks'
        ext().int8_gemm(rows.blocks, rows.scale, w.blocks, w.scale, 300, None, None, False, y)
    with pytest.raises(RuntimeError):  # more rows than were quantised
        ext().int8_gemm(rows.blocks, rows.scale, w.blocks, w.scale, 64, None, None, False,
                        torch.empty(40, 6, device=gpu, dtype=torch.bfloat16))


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 8, 50, 700])
def test_gpu_graph_replays_and_side_stream(gpu, M):
    x, wq, ws, bias, _ = make(M, 1000, 260, torch.bfloat16, device=gpu)
    w = ops.Int8Weight(wq, ws)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = ops.int8_linear(x, w, bias)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(side, ops.int8_linear(x, w, bias))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops.int8_linear(x, w, bias)
        graphs.append((g, out))
    for i in range(3):
        x.copy_(torch.randn_like(x) * (i + 1))
        for g, _ in graphs:
            g.replay()
        want = ops.int8_linear(x, w, bias)
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for _, out in graphs)


@pytest.mark.gpu
def test_gpu_outputs_past_32_bit_offsets(gpu):
    """More than 2^32 outputs: the last rows equal a small product of the same rows."""
    M, K, N = 70000, 65, 65537
    x, wq, ws, bias, _ = make(M, K, 1, torch.bfloat16, device=gpu)
    g = torch.Generator(device=gpu).manual_seed(1)
    wq = torch.randint(-127, 128, (N, K), generator=g, device=gpu, dtype=torch.int8)
    w = ops.Int8Weight(wq, torch.rand(N, generator=g, device=gpu))
    y = ops.int8_linear(x, w)
    for a in (0, M // 2, M - 40):
        assert torch.equal(y[a:a + 40], ops.int8_linear(x[a:a + 40].contiguous(), w))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,K", [(1535, 600), (1536, 600), (2559, 600), (2561, 600), (50, 512), (50, 513),
                                 (30, 4097), (2600, 5000), (21, 16385), (9, 33000)])
def test_gpu_quantize_row_groups(gpu, M, K, dtype):
    """Where the quantiser changes the rows of a workgroup and what it holds of a row; the padding
    rows of the last group are written too."""
    x = make(M, K, 1, dtype, seed=M + K)[0]
    x[M - 1, K // 2] = float("inf")
    r = ops.quantize_rows(x.to(gpu))
    q, s = ref_quantize_rows(x)
    assert torch.equal(from_blocks(r.blocks, M, K).cpu(), q)
    assert torch.equal(r.scale[:-1].cpu(), s[:-1]) and bool(r.scale[-1].isnan())
    full = from_blocks(r.blocks, *r.blocks.shape).cpu()
    assert int(full[M:].abs().sum()) == 0 and int(full[:, K:].abs().sum()) == 0
