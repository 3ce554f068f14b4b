"""The mixture-of-experts layer over 4-bit experts against a plain 64-bit implementation."""

import ctypes
import math

import pytest
import torch

from helpers import half_ulp
from neuropress_b200 import _cabi, kernels

DEV = "cuda"

def assert_close(y, ref, dtype):
    """|y - ref| <= half an ulp of the output + 2^-12 sum |D| |h| + 2e-4 RMS(row).  Between the two kernels h has
    11 significant bits, an error of at most 2^-12 of each value, whatever the terms are.  The rest is fp32: a
    row's product is formed as sum (magic + q) x - (magic + z) sum x, so against codes of spread 4.6 the roundings
    (2^-24, about ten in a row) count 1040 / 4.6 = 226 times in fp16, 4e-5 of the RMS in the mean, and the
    largest of some 1e5 outputs lies within five times that."""
    ref, spread = ref
    y = y.detach().cpu().double()
    assert y.shape == ref.shape and bool(torch.isfinite(y).all())
    rms = ref.square().mean(-1, keepdim=True).sqrt()
    beyond = (y - ref).abs() - half_ulp(ref, dtype) - 2.0 ** -12 * spread - 2e-4 * rms
    assert float(beyond.max()) <= 0, (float(beyond.max()), float(rms.max()))


class Experts:
    def __init__(self, e, h, i, g, asym, seed):
        gen = torch.Generator().manual_seed(seed)
        self.e, self.h, self.i, self.g = e, h, i, g

        def weight(rows, cols):
            codes = torch.randint(0, 256, (e, rows, cols // 2), generator=gen, dtype=torch.uint8)
            scale = ((torch.rand(e, rows, cols // g, generator=gen) + 0.5) * (0.2 * cols ** -0.5)).half()
            zero = (torch.rand(e, rows, cols // g, generator=gen) * 2 + 7).half() if asym else None
            return codes, scale, zero

        self.gate, self.up, self.down = weight(i, h), weight(i, h), weight(h, i)
        self.gen = gen

    def on(self, device):
        return tuple(tuple(None if t is None else t.to(device) for t in w) for w in (self.gate, self.up, self.down))

    def inputs(self, t, dtype, logit_dtype=torch.float32):
        return (torch.randn(t, self.h, generator=self.gen).to(dtype),
                (torch.randn(t, self.e, generator=self.gen) * 1.5).to(logit_dtype))


def dense(weight, e, g):
    codes, scale, zero = weight
    q = torch.empty(codes.shape[1], codes.shape[2] * 2, dtype=torch.float64)
    q[:, 0::2], q[:, 1::2] = (codes[e] & 15).double(), (codes[e] >> 4).double()
    z = 8.0 if zero is None else zero[e].double().repeat_interleave(g, 1)
    return (q - z) * scale[e].double().repeat_interleave(g, 1)


def plain(ex, x, logits, top_k, renorm):
    """The layer in 64 bits, and sum_e w_e sum_i |D_e[j, i]| |h_e[i]|."""
    l = logits.double()
    order = torch.sort(l, dim=-1, descending=True, stable=True).indices[:, :top_k]
    y, spread = torch.zeros(2, *x.shape, dtype=torch.float64)
    for t in range(x.shape[0]):
        if bool(torch.isnan(l[t]).any() | (l[t] == math.inf).any()):
            y[t] = math.nan
            continue
        if bool((l[t] == -math.inf).all()):
            continue
        p = torch.softmax(l[t], -1)
        total = p[order[t]].sum() if renorm else 1.0
        for e in order[t].tolist():
            if l[t, e] == -math.inf:
                continue
            xd = x[t].double()
            h = torch.nn.functional.silu(dense(ex.gate, e, ex.g) @ xd) * (dense(ex.up, e, ex.g) @ xd)
            y[t] += p[e] / total * (dense(ex.down, e, ex.g) @ h)
            spread[t] += p[e] / total * (dense(ex.down, e, ex.g).abs() @ h.abs())
    return y, spread


def run(ex, x, logits, top_k, renorm=True):
    return kernels.q_moe(x.to(DEV), logits.to(DEV), *ex.on(DEV), top_k, ex.g, renormalize=renorm)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("asym", [False, True])
@pytest.mark.parametrize("t,e,k,h,i,g", [
    (1, 8, 2, 256, 128, 32), (2, 5, 3, 96, 160, 32), (3, 64, 8, 512, 96, 32), (4, 1, 1, 1024, 64, 64),
    (5, 4, 4, 192, 384, 96), (8, 16, 2, 32, 32, 32), (17, 40, 6, 640, 256, 128), (32, 8, 2, 2048, 512, 64),
    (31, 3, 1, 352, 224, 32), (1, 512, 16, 64, 64, 32), (32, 100, 16, 128, 96, 32), (1, 4, 2, 4096, 1376, 32),
])
def test_matches_plain_implementation(t, e, k, h, i, g, asym, dtype):
    ex = Experts(e, h, i, g, asym, seed=t * 7 + e)
    x, logits = ex.inputs(t, dtype)
    for renorm in (True, False):
        y = run(ex, x, logits, k, renorm)
        assert y.dtype == dtype
        assert_close(y, plain(ex, x, logits, k, renorm), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("asym", [False, True])
@pytest.mark.parametrize("t", [1, 2, 3, 4, 20])
@pytest.mark.parametrize("h,i,g", [(1024, 512, 64), (512, 1024, 64), (1024, 2048, 128), (2048, 2048, 256)])
def test_groups_of_a_power_of_two(t, h, i, g, asym):
    """Groups wider than a block in rows of whole 16-byte pieces, for every number of tokens to a product."""
    ex = Experts(3, h, i, g, asym, seed=h + i + t)
    x, logits = ex.inputs(t, torch.float16)
    assert_close(run(ex, x, logits, 2), plain(ex, x, logits, 2, True), torch.float16)


@pytest.mark.gpu
@pytest.mark.parametrize("asym", [False, True])
@pytest.mark.parametrize("t,e,k,h,i,g", [
    (32, 2, 1, 16384, 64, 32), (7, 2, 2, 64, 16384, 32), (8, 2, 1, 16352, 224, 224), (1, 3, 2, 16352, 32, 32),
    (32, 2, 1, 4096, 16352, 32), (3, 2, 1, 8192, 2080, 32), (32, 1, 1, 16384, 2048, 2048),
])
def test_widest(t, e, k, h, i, g, asym):
    """The ends of the range, where tokens and rings compete for shared memory and units get smaller."""
    ex = Experts(e, h, i, g, asym, seed=h + i)
    x, logits = ex.inputs(t, torch.bfloat16)
    if h * i > 1 << 24:                              # some tokens of the largest, each of them on its own
        y = run(ex, x, logits, k)
        some = torch.tensor([0, t - 1])
        assert_close(y[some], plain(ex, x[some], logits[some], k, True), torch.bfloat16)
    else:
        assert_close(run(ex, x, logits, k), plain(ex, x, logits, k, True), torch.bfloat16)
    assert _cabi.gemm_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("t", [33, 70])
def test_more_tokens_than_a_call_takes(t):
    ex = Experts(6, 128, 96, 32, False, seed=t)
    x, logits = ex.inputs(t, torch.bfloat16)
    assert_close(run(ex, x, logits, 2), plain(ex, x, logits, 2, True), torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("logit_dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_ties_go_to_the_lowest_expert(logit_dtype):
    ex = Experts(40, 64, 64, 32, False, seed=3)
    x, logits = ex.inputs(9, torch.float16, logit_dtype)
    logits[0] = 0.25                                   # every expert ties
    logits[1:5] = (logits[1:5] * 2).round() / 2        # a few values
    logits[5, 33:] = 9.0
    logits[6] = torch.where(torch.arange(40) % 2 == 0, 0.0, -0.0).to(logit_dtype)   # +0 and -0 are equal
    logits[7] = torch.finfo(logit_dtype).min           # the type's lowest value is a value like any other
    assert_close(run(ex, x, logits, 5), plain(ex, x, logits, 5, True), torch.float16)


@pytest.mark.gpu
@pytest.mark.parametrize("e", [3, 33, 200])
def test_masked_and_broken_rows(e):
    ex = Experts(e, 96, 64, 32, True, seed=e)
    x, logits = ex.inputs(12, torch.bfloat16)
    logits[0] = -math.inf                               # padding: no expert left
    logits[1, 1:] = -math.inf                           # one expert left, three asked for
    logits[2, :-2] = -math.inf
    logits[3, e // 2] = math.nan
    logits[4] = math.nan
    logits[5, 0] = math.inf
    logits[6] = -math.inf
    logits[6, e - 1] = math.nan
    logits[7] = -math.inf
    logits[7, 1] = math.inf
    for renorm in (True, False):
        y = run(ex, x, logits, 3, renorm).cpu()
        ref, spread = plain(ex, x, logits, 3, renorm)
        assert bool((y[0] == 0).all())
        broken = torch.isnan(ref).all(-1)
        assert broken.sum() == 5
        assert bool(torch.isnan(y[broken]).all())
        assert_close(y[~broken], (ref[~broken], spread[~broken]), torch.bfloat16)


@pytest.mark.gpu
def test_all_tokens_on_one_expert_and_one_on_its_own():
    ex = Experts(8, 512, 192, 64, False, seed=11)
    x, logits = ex.inputs(32, torch.bfloat16)
    logits[:, 5] = 20.0
    logits[30, 5], logits[30, 0] = -20.0, 20.0
    assert_close(run(ex, x, logits, 1), plain(ex, x, logits, 1, True), torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_bad_token_leaves_the_others_alone(bad):
    ex = Experts(4, 256, 128, 32, False, seed=12)
    x, logits = ex.inputs(8, torch.float16)
    good = run(ex, x, logits, 2)
    x2 = x.clone()
    x2[3, 100] = bad
    y = run(ex, x2, logits, 2)
    keep = torch.arange(8) != 3
    assert torch.equal(y[keep], good[keep]) and not bool(torch.isfinite(y[3]).all())


@pytest.mark.gpu
def test_same_bits_every_time():
    ex = Experts(6, 384, 160, 32, False, seed=13)
    x, logits = ex.inputs(11, torch.bfloat16)
    first = run(ex, x, logits, 2)
    for _ in range(5):
        assert torch.equal(run(ex, x, logits, 2), first)


@pytest.mark.gpu
def test_no_tokens():
    ex = Experts(4, 64, 64, 32, False, seed=1)
    x, logits = ex.inputs(0, torch.bfloat16)
    assert run(ex, x, logits, 2).shape == (0, 64)


@pytest.mark.gpu
def test_streams_and_graphs_that_share_nothing():
    """Two calls in flight on two streams, and two captured graphs replayed in turn and side by side."""
    ex = Experts(8, 1024, 512, 32, False, seed=21)
    w = ex.on(DEV)
    sets = [tuple(a.to(DEV) for a in ex.inputs(8, torch.bfloat16)) for _ in range(2)]
    want = [kernels.q_moe(*s, *w, 2, 32) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(kernels.q_moe(*sets[i], *w, 2, 32))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])
    graphs, outs = [], []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            first = kernels.q_moe(*s, *w, 2, 32)
            outs.append(kernels.q_moe(first, s[1], *w, 2, 32))
        graphs.append(graph)
    second = [kernels.q_moe(want[i], sets[i][1], *w, 2, 32) for i in range(2)]
    for _ in range(3):
        for i, graph in enumerate(graphs):
            with torch.cuda.stream(streams[i]):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, second))


# ---- refusals: no GPU needed -------------------------------------------------------------
def test_wrapper_refuses():
    ex = Experts(4, 64, 96, 32, False, seed=1)
    x, l = ex.inputs(2, torch.bfloat16)
    w = (ex.gate, ex.up, ex.down)
    with pytest.raises(RuntimeError, match="expected x"):
        kernels.q_moe(x[0], l, *w, 2, 32)
    with pytest.raises(RuntimeError, match="expected x"):
        kernels.q_moe(x, l[:1], *w, 2, 32)
    with pytest.raises(RuntimeError, match="float16 or bfloat16"):
        kernels.q_moe(x.float(), l, *w, 2, 32)
    for k in (0, 5, 17):
        with pytest.raises(RuntimeError, match="top_k"):
            kernels.q_moe(x, l, *w, k, 32)
    for g in (0, 16, 48, 64):       # 64 divides H, not I
        with pytest.raises(RuntimeError, match="group_size"):
            kernels.q_moe(x, l, *w, 2, g)
    with pytest.raises(RuntimeError, match="codes of gate"):
        kernels.q_moe(x, l[:, :3], *w, 2, 32)
    with pytest.raises(RuntimeError, match="codes of down"):
        kernels.q_moe(x, l, ex.gate, ex.up, ex.up, 2, 32)
    with pytest.raises(RuntimeError, match="zero_point of up"):
        kernels.q_moe(x, l, ex.gate, (ex.up[0], ex.up[1][:, :-1], None), ex.down, 2, 32)
    with pytest.raises(RuntimeError, match="both have zero points"):
        kernels.q_moe(x, l, ex.gate, (ex.up[0], ex.up[1], ex.up[1]), ex.down, 2, 32)
    with pytest.raises(RuntimeError, match="uint8"):
        kernels.q_moe(x, l, (ex.gate[0].int(), ex.gate[1], None), ex.up, ex.down, 2, 32)
    with pytest.raises(RuntimeError, match="CUDA"):
        kernels.q_moe(x, l, *w, 2, 32)


def test_c_entry_refuses():
    if not _cabi.library_available():
        pytest.skip("library not built")
    lib = _cabi.load_library()

    def weight(codes=4096, scale=4096, zp=None, nbits=4, g=32):
        s = _cabi.QWeightStruct()
        s.codes, s.scale, s.zero_point, s.nbits, s.group_size = codes, scale, zp, nbits, g
        return s

    good = dict(x=4096, dtype=1, logits=4096, ldt=2, T=2, E=4, H=64, I=96, gate=weight(), up=weight(), down=weight(),
                k=2, renorm=1, ws=4096, ws_bytes=lib.npb_q_moe_workspace_bytes(2, 2, 96), y=4096)

    def call(**change):
        a = {**good, **change}
        for name in ("gate", "up", "down"):
            a[name] = None if a[name] is None else ctypes.byref(a[name])
        return lib.npb_q_moe(*a.values(), None)

    for change in ({"T": -1}, {"E": 0}, {"H": 0}, {"I": 0}, {"k": 0}, {"k": 5}, {"gate": None}, {"down": None},
                   {"x": None}, {"logits": None}, {"ws": None}, {"y": None}, {"up": weight(codes=None)}):
        assert call(**change) == 1, change
    for change in ({"dtype": 2}, {"ldt": 3}, {"T": 33}, {"E": 513}, {"k": 17, "E": 100}, {"gate": weight(nbits=8)},
                   {"down": weight(g=16)}, {"gate": weight(zp=4096)}, {"gate": weight(g=64)},
                   {"H": 16416}, {"I": 16416}):
        assert call(**change) == 2, change
    assert call(H=72) == 3 and call(I=100) == 3 and call(gate=weight(g=96)) == 3
    assert call(gate=weight(scale=4104)) == 4 and call(down=weight(zp=4104)) == 4
    assert call(x=4098) == 4 and call(ws=4104) == 4 and call(gate=weight(codes=4104)) == 4 and call(y=4097) == 4
    assert call(ws_bytes=good["ws_bytes"] - 1) == 6
    assert call(T=0, x=None) == 0
    assert lib.npb_q_moe_workspace_bytes(2, 2, 96) > 2 * 2 * 96 * 2
    assert lib.npb_q_moe_workspace_bytes(33, 2, 96) == 0 and lib.npb_q_moe_workspace_bytes(2, 2, 97) == 0
