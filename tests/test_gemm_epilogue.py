"""The dense GEMM with bias, activation and residual in its epilogue against 64-bit arithmetic."""

import math

import pytest
import torch
import torch.nn.functional as F

from helpers import assert_output_close, half_ulp
from neuropress_b200 import _cabi, kernels

DEV = "cuda"
ACTS = {None: lambda v: v, "none": lambda v: v, "relu": torch.relu, "silu": F.silu, "gelu": F.gelu,
        "gelu_tanh": lambda v: F.gelu(v, approximate="tanh")}

# Largest error next to the output's own rounding, relative to RMS(y): the accumulator takes K / 16 steps of at
# most 2^-23 of the running sum (K = 14336: 1.1e-4), the activation a few 2^-24 more and its slope (<= 1.13); the
# RMS after relu / silu / gelu is no less than half of that before it.
TOL = 5e-4


def make(m, n, k, dtype, seed, bias=True, residual=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g).to(dtype)
    w = (torch.randn(n, k, generator=g) * k ** -0.5 * 1.5).to(dtype)
    b = torch.randn(n, generator=g) * 0.5 if bias else None
    r = torch.randn(m, n, generator=g).to(dtype) if residual else None
    return x, w, b, r


def plain(x, w, b, act, r, dev="cpu"):
    """64-bit, on the CPU (or on the GPU for the sizes where that takes too long)."""
    y = x.to(dev).double() @ w.to(dev).double().T
    if b is not None:
        y = y + b.to(dev).double()
    y = ACTS[act](y)
    return y if r is None else y + r.to(dev).double()


def run(x, w, b, act, r):
    return kernels.gemm_epilogue(x.to(DEV), w.to(DEV), None if b is None else b.to(DEV), act,
                                 None if r is None else r.to(DEV))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("m", [1, 16, 33, 130, 300])
def test_activations(m, act, dtype):
    x, w, b, r = make(m, 520, 256, dtype, seed=m)
    for bias in (b, None):
        for res in (r, None):
            y = run(x, w, bias, act, res)
            assert y.dtype == dtype and y.shape == (m, 520)
            assert_output_close(y, plain(x, w, bias, act, res), dtype, tol=TOL)
    assert _cabi.gemm_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [
    (1, 1, 8), (1, 7, 16), (3, 33, 72), (1, 128, 64), (1, 4096, 4096), (2, 1000, 2056), (5, 129, 8192), (8, 300, 136),
    (9, 2048, 2048), (16, 14336, 1024), (17, 255, 520), (31, 777, 1000), (32, 1024, 8192), (48, 640, 4104),
    (64, 512, 2048), (65, 4099, 264), (97, 384, 14336), (128, 8192, 512), (129, 1023, 1024), (160, 2048, 2048),
    (192, 96, 8192), (201, 513, 4096), (255, 1024, 1032), (256, 640, 2048), (257, 1000, 256), (384, 2049, 512),
    (1000, 1000, 328), (2048, 512, 1024), (513, 4096, 4096)])
def test_shapes(shape):
    m, n, k = shape
    for dtype in (torch.bfloat16, torch.float16):
        x, w, b, r = make(m, n, k, dtype, seed=m + n + k)
        y = run(x, w, b, "silu", r)
        ref = plain(x, w, b, "silu", r, DEV if m * n * k > 1 << 28 else "cpu")
        assert_output_close(y, ref, dtype, tol=TOL)
        assert torch.equal(y, run(x, w, b, "silu", r))     # no sum depends on scheduling
    assert _cabi.gemm_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [
    (1, 9601, 264), (3, 19200, 136), (33, 9480, 4104), (100, 9601, 520), (128, 18944, 264), (150, 12801, 2056),
    (161, 9475, 1032), (176, 9600, 8192), (201, 12803, 4104), (208, 18432, 136), (256, 9481, 264), (256, 9216, 1096),
    (300, 8192, 520), (400, 8190, 2056), (416, 9344, 72), (30, 40000, 264), (33, 40001, 264), (201, 20000, 8200),
    (9000, 130, 264), (18689, 100, 72)])
def test_many_tiles(shape):
    """Two CTAs to an SM, CTA pairs and the sizes where the forms change over, with odd and even rows of outputs."""
    m, n, k = shape
    x, w, b, r = make(m, n, k, torch.bfloat16, seed=m + n + k)
    y = run(x, w, b, "gelu", r)
    assert_output_close(y, plain(x, w, b, "gelu", r, DEV), torch.bfloat16, tol=TOL)
    assert torch.equal(y, run(x, w, b, "gelu", r))
    x, w, b, r = make(m, n, k, torch.float16, seed=m + n + k, bias=False)
    assert_output_close(run(x, w, b, "none", r), plain(x, w, b, "none", r, DEV), torch.float16, tol=TOL)
    assert _cabi.gemm_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 40, 140, 400])
def test_plain_product_agrees_with_gemm(m):
    x, w, b, _ = make(m, 1024, 2048, torch.bfloat16, seed=m)
    y = run(x, w, b, None, None)
    z = kernels.gemm(x.to(DEV), w.to(DEV), b.to(DEV)).double().cpu()
    # either is rounded by half an ulp, so two results of the same sum may lie a whole one apart
    bound = 2 * half_ulp(z, torch.bfloat16) * (1 + 2.0 ** -7) + TOL * z.square().mean().sqrt()
    assert bool(((y.double().cpu() - z).abs() <= bound).all())


@pytest.mark.gpu
@pytest.mark.parametrize("m", [2, 20, 140, 300])
def test_bad_values_stay_in_their_row_and_column(m):
    x, w, b, r = make(m, 200, 256, torch.bfloat16, seed=m)
    good = run(x, w, b, "relu", r)
    x2, w2, r2 = x.clone(), w.clone(), r.clone()
    x2[1, 7] = math.nan
    w2[100, 3] = math.inf
    r2[0, 5] = -math.inf
    y = run(x2, w2, b, "relu", r2)
    keep = torch.ones(m, 200, dtype=torch.bool)
    keep[1] = False
    keep[:, 100] = False
    keep[0, 5] = False
    assert torch.equal(y.cpu()[keep], good.cpu()[keep])
    assert bool(torch.isnan(y[1]).all()) and float(y[0, 5]) == -math.inf
    x2 = torch.full_like(x, 200.0)                      # far out on both sides of the activations
    for act in ("silu", "gelu", "gelu_tanh", "relu"):
        assert_output_close(run(x2, w, b, act, None), plain(x2, w, b, act, None), torch.bfloat16, tol=TOL)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 16, 100, 300])
def test_unaligned_residual_and_output_in_place(m):
    """A residual that starts at an odd element, and at the C entry an output that is the residual."""
    x, w, b, r = make(m, 264, 512, torch.float16, seed=m)
    shifted = torch.empty(m * 264 + 1, dtype=torch.float16, device=DEV)[1:].view(m, 264)
    shifted.copy_(r)
    want = run(x, w, b, "gelu", r)
    xg, wg, bg = x.to(DEV), w.to(DEV), b.to(DEV)
    assert torch.equal(kernels.gemm_epilogue(xg, wg, bg, "gelu", shifted), want)
    lib = _cabi.load_library()
    for buf in (shifted, r.to(DEV)):
        rc = lib.npb_gemm_epilogue(xg.data_ptr(), wg.data_ptr(), bg.data_ptr(), 3, buf.data_ptr(), buf.data_ptr(), m, 264,
                                   512, 0, _cabi.stream_ptr())
        assert rc == 0 and torch.equal(buf, want)


@pytest.mark.gpu
def test_rows_behind_the_last_are_left_alone():
    x, w, b, r = (None if t is None else t.to(DEV) for t in make(5, 200, 512, torch.bfloat16, seed=1))
    out = torch.full((9, 200), 7.0, dtype=torch.bfloat16, device=DEV)
    lib = _cabi.load_library()
    rc = lib.npb_gemm_epilogue(x.data_ptr(), w.data_ptr(), b.data_ptr(), 2, r.data_ptr(), out[2:].data_ptr(), 5, 200, 512,
                               1, _cabi.stream_ptr())
    assert rc == 0
    assert torch.equal(out[2:7], kernels.gemm_epilogue(x, w, b, "silu", r))
    assert bool((out[:2] == 7).all()) and bool((out[7:] == 7).all())


@pytest.mark.gpu
def test_streams_and_graphs():
    """Calls in flight on two streams, and graphs captured from them, replayed side by side."""
    sets = [[t.to(DEV) for t in make(m, 1024, 4096, torch.bfloat16, seed=m)] for m in (4, 150)]
    want = [kernels.gemm_epilogue(*s[:3], "silu", s[3]) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(kernels.gemm_epilogue(*sets[i][:3], "silu", sets[i][3]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])
    graphs, outs = [], []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(kernels.gemm_epilogue(*s[:3], "silu", s[3]))
        graphs.append(graph)
    for _ in range(3):
        for i, graph in enumerate(graphs):
            with torch.cuda.stream(streams[i]):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    assert _cabi.gemm_device_status() == 0


@pytest.mark.gpu
def test_empty():
    w = torch.zeros(16, 64, dtype=torch.bfloat16, device=DEV)
    assert kernels.gemm_epilogue(w[:0], w, None, "gelu").shape == (0, 16)
    assert kernels.gemm_epilogue(w, w[:0], None, "gelu", w[:, :0].contiguous()).shape == (16, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 500])
def test_decoded_weight_takes_activation_and_residual(rows):
    import oracle
    from synthetic import make_activations, make_vq_layer

    d = make_vq_layer(384, 512, num_centroids=4096, bits=12, seed=5, bias=True)
    x = make_activations(rows, 512, torch.bfloat16, seed=rows)
    r = make_activations(rows, 384, torch.bfloat16, seed=rows + 1)
    y = kernels.vq_dequant_gemm(x.to(DEV), d.packed.to(DEV), d.centroids.to(DEV), 12, 384, d.bias.to(DEV),
                                activation="gelu", residual=r.to(DEV))
    w = oracle.vq_decode(d.packed, d.centroids, 12, 384, 512, torch.bfloat16)
    assert_output_close(y, plain(x, w, d.bias, "gelu", r), torch.bfloat16, tol=TOL)


# ---- refusals: no GPU needed -------------------------------------------------------------
def test_wrapper_refuses():
    x, w, b, r = make(2, 8, 16, torch.bfloat16, seed=1)
    for a in ((x[0], w), (x, w[0]), (x, w[:, :8])):
        with pytest.raises(RuntimeError, match="expected x"):
            kernels.gemm_epilogue(*a)
    for a in ((x.half(), w), (x, w, b, None, r.half())):
        with pytest.raises(RuntimeError, match="same dtype"):
            kernels.gemm_epilogue(*a)
    with pytest.raises(RuntimeError, match="unknown activation"):
        kernels.gemm_epilogue(x, w, b, "swish")
    for bad in (r[:1], r[:, :4], r[0]):
        with pytest.raises(RuntimeError, match="residual must be"):
            kernels.gemm_epilogue(x, w, b, None, bad)
    with pytest.raises(RuntimeError, match="CUDA"):
        kernels.gemm_epilogue(x, w, b, "silu", r)


def test_c_entry_refuses():
    if not _cabi.library_available():
        pytest.skip("library not built")
    lib = _cabi.load_library()
    good = dict(x=4096, w=4096, bias=4096, act=1, res=4096, y=4096, M=2, N=8, K=16, dtype=1)

    def call(**change):
        return lib.npb_gemm_epilogue(*{**good, **change}.values(), None)

    for change in ({"act": -1}, {"act": 5}, {"x": None}, {"w": None}, {"y": None}, {"M": -1}, {"N": -1}, {"K": -8}):
        assert call(**change) == 1, change
    assert call(dtype=2) == 2 and call(M=1 << 31) == 2
    assert call(K=12) == 3 and call(K=0) == 3
    for change in ({"x": 4098}, {"w": 4104}, {"y": 4097}, {"res": 4097}, {"bias": 4098}):
        assert call(**change) == 4, change
    assert call(M=0, x=None) == 0
