"""How exact the mixture-of-experts layer is: tokens with one large channel, against a plain 64-bit implementation."""

import ctypes

import pytest
import torch

from helpers import half_ulp
from neuropress_b200 import _cabi
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
