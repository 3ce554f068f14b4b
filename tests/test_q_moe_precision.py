"""How exact the mixture-of-experts layer is: tokens with one large channel, a bound on the rounding of h that stays tight
at every width, and weights of mixed forms, against a plain 64-bit implementation."""

import ctypes

import pytest
import torch

from helpers import half_ulp
from neuropress_b200 import _cabi, kernels
from test_q_moe import Experts, dense

DEV = "cuda"


def layer(x, logits, weights, groups, top_k, h_as=None):
    """The layer in 64 bits (renormalised weights) and sqrt(sum_e w_e^2 sum_i D_e[j, i]^2 h_e[i]^2); h_as rounds h to a
    type.  weights: (gate, up, down); groups: their group sizes."""
    y, square = torch.zeros(2, *x.shape, dtype=torch.float64)
    for t in range(x.shape[0]):
        order = torch.sort(logits[t].double(), descending=True, stable=True).indices[:top_k]
        p = torch.softmax(logits[t].double()[order], 0)
        for w, e in zip(p, order.tolist()):
            gate, up = (dense(weights[k], e, groups[k]) @ x[t].double() for k in range(2))
            h = w * torch.nn.functional.silu(gate) * up
            if h_as is not None:
                h = h.to(h_as).double()
            d = dense(weights[2], e, groups[2])
            y[t] += d @ h
            square[t] += d.square() @ h.square()
    return y, square.sqrt()


def excess(y, ref, spread, dtype, sums=5e-4):
    """How far the worst output is beyond half a step of its type + 3 * 2^-11 sqrt(sum D^2 h^2) + sums * RMS(row).

    h has 11 significant bits between the kernels: each value is off by at most 2^-11 of the power of two below it, evenly
    spread, a standard deviation of at most 2^-11 / sqrt(3) of the value and of 0.74 times that over all mantissas
    (E 1/m^2 over a logarithmic mantissa is 0.54).  Independent errors add in squares, so the second term is 5.2 of the
    first and 7 of the second deviation of their sum.  The third term: a block of 32 is summed as C + sum (1024 + q) x', C
    about 4100 of x's deviation (half of the x' are divided by 16), in eight steps that each lose up to 2^-23 of the sum so
    far, about 1e-3 in all, against the block's own 26 (codes of spread 4.6): 4e-5.  Three products in a row: 7e-5 of the
    RMS, of which the default of 5e-4 is seven times."""
    y = y.detach().cpu().double()
    assert y.shape == ref.shape and bool(torch.isfinite(y).all())
    rms = ref.square().mean(-1, keepdim=True).sqrt()
    return float(((y - ref).abs() - half_ulp(ref, dtype) - 3 * 2.0 ** -11 * spread - sums * rms).max())


def run(x, logits, weights, groups, top_k):
    """Through the C entry, which takes a group size for down of its own."""
    lib = _cabi.load_library()
    dev = [tuple(None if a is None else a.to(DEV).contiguous() for a in w) for w in weights]
    structs = [_cabi.q_struct(*w, 4, g) for w, g in zip(dev, groups)]
    x, logits = x.to(DEV), logits.to(DEV)
    t, h = x.shape
    i = weights[0][0].shape[1]
    size = lib.npb_q_moe_workspace_bytes(t, top_k, i)
    ws = torch.empty(size, dtype=torch.uint8, device=DEV)
    y = torch.empty_like(x)
    rc = lib.npb_q_moe(x.data_ptr(), _cabi.dtype_code(x.dtype), logits.data_ptr(), _cabi.dtype_code(logits.dtype), t,
                       logits.shape[1], h, i, *(ctypes.byref(s) for s in structs), top_k, 1, ws.data_ptr(), size,
                       y.data_ptr(), _cabi.stream_ptr())
    assert rc == 0
    torch.cuda.synchronize()
    return y


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("t", [1, 3, 9])
def test_one_large_channel_without_weight(t, dtype):
    """A channel 2^14 times the others whose weights are all zero: the others still count in full."""
    ex = Experts(3, 512, 256, 32, False, seed=t)
    x, logits = ex.inputs(t, dtype)
    x[:, 64:96] = 0
    x[:, 70] = 2.0 ** 14
    for codes, _, _ in (ex.gate, ex.up):
        codes[:, :, 32:48] = 0x88          # columns 64 to 95: q = 8, weight zero
    weights, groups = (ex.gate, ex.up, ex.down), (32, 32, 32)
    assert excess(run(x, logits, weights, groups, 2), *layer(x, logits, weights, groups, 2), dtype) <= 0


@pytest.mark.gpu
@pytest.mark.parametrize("asym", [False, True])
@pytest.mark.parametrize("large", [30.0, 1000.0])
@pytest.mark.parametrize("t", [2, 4, 12])
def test_one_large_channel(t, large, asym):
    """One channel far above the others, with weights like any other.  Its block is summed from C = 1032 times it, and each
    of eight steps loses up to 2^-23 of that: 5e-4 in the mean, where the weights have 4.6, so 1.1e-4 of the RMS for each of
    gate and up.  With the 7e-5 of all blocks 1.7e-4, of which 1.2e-3 is seven times."""
    ex = Experts(4, 1024, 192, 32, asym, seed=int(large) + t)
    x, logits = ex.inputs(t, torch.float16)
    x[:, 322] = large
    x[t // 2, 322] = -large
    weights, groups = (ex.gate, ex.up, ex.down), (32, 32, 32)
    y = run(x, logits, weights, groups, 2)
    assert excess(y, *layer(x, logits, weights, groups, 2), torch.float16, sums=1.2e-3) <= 0


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("t", [2, 4, 10])
def test_a_token_with_an_infinity_is_nan_throughout(t, dtype, bad):
    """Its other channels may be beyond fp16 (bf16 rows); the other tokens are as without it."""
    ex = Experts(3, 256, 128, 32, True, seed=t)
    x, logits = ex.inputs(t, dtype)
    weights, groups = (ex.gate, ex.up, ex.down), (32, 32, 32)
    good = run(x, logits, weights, groups, 2)
    x[1, 77] = bad
    x[1, 78] = torch.finfo(dtype).max
    y = run(x, logits, weights, groups, 2)
    assert bool(torch.isnan(y[1]).all())
    keep = torch.arange(t) != 1
    assert torch.equal(y[keep], good[keep])


@pytest.mark.gpu
@pytest.mark.parametrize("asym", [False, True])
@pytest.mark.parametrize("t,e,k,h,i,g", [
    (1, 2, 2, 64, 16384, 32), (3, 2, 1, 128, 8192, 128), (7, 3, 2, 256, 4096, 32), (32, 2, 1, 96, 2048, 32),
    (4, 4, 2, 2048, 512, 64), (20, 8, 2, 512, 352, 32),
])
def test_rounding_of_h_at_every_width(t, e, k, h, i, g, asym):
    ex = Experts(e, h, i, g if h % g == 0 else 32, asym, seed=h + i + t)
    groups = (ex.g,) * 3
    x, logits = ex.inputs(t, torch.float16)
    weights = (ex.gate, ex.up, ex.down)
    assert excess(run(x, logits, weights, groups, k), *layer(x, logits, weights, groups, k), torch.float16) <= 0


# group sizes of gate / up and of down (rows of whole 16-byte pieces of groups or not, one block to a group or more), and
# which of the two have zero points
@pytest.mark.gpu
@pytest.mark.parametrize("t", [2, 4, 13])
@pytest.mark.parametrize("asym_up,asym_down", [(False, True), (True, False), (True, True), (False, False)])
@pytest.mark.parametrize("g_up,g_down", [(32, 64), (64, 32), (96, 32), (32, 96), (128, 96), (96, 128), (256, 512)])
def test_mixed_forms(g_up, g_down, asym_up, asym_down, t):
    h, i = (768, 1536) if 96 in (g_up, g_down) else (1024, 2048)
    up = Experts(3, h, i, g_up, asym_up, seed=g_up + t)
    down = Experts(3, h, i, g_down, asym_down, seed=g_down + t)
    x, logits = up.inputs(t, torch.float16)
    weights, groups = (up.gate, up.up, down.down), (g_up, g_up, g_down)
    assert excess(run(x, logits, weights, groups, 2), *layer(x, logits, weights, groups, 2), torch.float16) <= 0


@pytest.mark.gpu
def test_wrapper_takes_zero_points_in_one_place_only():
    for asym_up in (False, True):
        a, b = (Experts(4, 256, 128, 32, s, seed=5) for s in (asym_up, not asym_up))
        x, logits = a.inputs(6, torch.float16)
        weights = (a.gate, a.up, b.down)
        on = [tuple(None if v is None else v.to(DEV) for v in w) for w in weights]
        y = kernels.q_moe(x.to(DEV), logits.to(DEV), *on, 2, 32)
        assert excess(y, *layer(x, logits, weights, (32, 32, 32), 2), torch.float16) <= 0


# ---- on the CPU -----------------------------------------------------------------------------
@pytest.mark.parametrize("i", [256, 4096])
def test_the_bound_sees_a_loss_of_three_bits_of_h(i):
    ex = Experts(2, 64, i, 32, False, seed=i)
    x, logits = ex.inputs(6, torch.float16)
    weights, groups = (ex.gate, ex.up, ex.down), (32, 32, 32)
    ref, spread = layer(x, logits, weights, groups, 2)
    as_stored = layer(x, logits, weights, groups, 2, torch.float16)[0].half()
    assert excess(as_stored, ref, spread, torch.float16) <= 0
    eight_bits = layer(x, logits, weights, groups, 2, torch.bfloat16)[0].half()
    assert excess(eight_bits, ref, spread, torch.float16) > 0
