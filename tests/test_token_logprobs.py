"""Token log probabilities, entropy and top alternatives against a plain 64-bit implementation."""

import math

import pytest
import torch

from neuropress_b200 import _cabi, kernels

DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
IGNORED = -100


def plain(logits, targets, n):
    """fp64 on the CPU; the definitions of masked rows and of rows with NaN / +inf spelled out."""
    l = logits.detach().cpu().double()
    t = targets.cpu()
    r, v = l.shape
    # the maximum comes off first: next to -3e38 even 64 bits cannot hold the logarithm of the sum
    d = l - l.amax(-1, keepdim=True)
    logp = d - torch.log(d.exp().sum(-1, keepdim=True))
    nothing = (l == -math.inf).all(-1)
    logp[nothing] = -math.inf
    broken = torch.isnan(l).any(-1) | (l == math.inf).any(-1)
    logp[broken] = math.nan
    p = logp.exp()
    entropy = -torch.where(p > 0, p * logp, 0.0).sum(-1)
    entropy[nothing], entropy[broken] = 0.0, math.nan
    known = (t >= 0) & (t < v)
    given = logp.gather(1, torch.where(known, t, 0)[:, None])[:, 0]
    given = torch.where(known, given, 0.0)
    order = torch.where(torch.isnan(l), -math.inf, l)
    # NaN after -inf: stable sort of the values, then of "is NaN"
    ids = torch.sort(order, dim=-1, descending=True, stable=True).indices
    nan_last = torch.sort(torch.isnan(l).gather(1, ids).int(), dim=-1, stable=True).indices
    ids = ids.gather(1, nan_last)[:, :n]
    return given, entropy, logp.gather(1, ids), ids


def check(logits, targets, n):
    got = kernels.token_logprobs(logits, targets, top_n=n)
    want = plain(logits, targets, n)
    r, v = logits.shape
    assert [tuple(g.shape) for g in got] == [(r,), (r,), (r, n), (r, n)]
    assert [g.dtype for g in got] == [torch.float32] * 3 + [torch.int64]
    assert torch.equal(got[3].cpu(), want[3])
    # fp32 chain of a sum: a tile of 32 terms, the thread's tiles, 21 merges, a few roundings per term
    # (e^d, d and its scaling: |d| <= ~ln V + |log p| matters); relative to 1 + the values at hand
    steps = 96 + v / 8192
    for g, w in zip(got[:3], want[:3]):
        g = g.cpu().double()
        assert torch.equal(torch.isnan(g), torch.isnan(w))
        inf = torch.isinf(w)
        assert torch.equal(torch.isinf(g), inf) and torch.equal(g[inf], w[inf])
        fine = ~inf & ~torch.isnan(w)
        bound = 2.0 ** -24 * steps * (1 + math.log(v) + w[fine].abs())
        assert bool(((g[fine] - w[fine]).abs() <= bound).all()), float(((g[fine] - w[fine]).abs() - bound).max())


def make(r, v, dtype, seed, scale=2.5):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(r, v, generator=g) * scale).to(dtype)
    targets = torch.randint(0, v, (r,), generator=g)
    return logits.to(DEV), targets.to(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,n", [((1, 1), 1), ((1, 7), 7), ((3, 33), 20), ((2, 255), 32), ((5, 1000), 5),
                                     ((4, 4097), 20), ((1, 32000), 32), ((33, 16384), 1), ((7, 50001), 8),
                                     ((700, 301), 3), ((600, 5003), 20), ((2, 140001), 20), ((4, 9000), 0)])
def test_matches_plain_implementation(shape, n, dtype):
    logits, targets = make(*shape, dtype, seed=shape[1] + n)
    check(logits, targets, n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset", [0, 1, 3, 7])
def test_strided_rows_and_odd_starts(offset, dtype):
    logits, targets = make(6, 9000, dtype, seed=offset)
    view = logits[:, offset:8200 + offset]
    check(view, targets % 8200, 9)
    flat = logits.reshape(-1)[offset:offset + 5 * 8111].view(5, 8111)
    check(flat, targets[:5] % 8111, 20)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [40, 3001, 33003])
def test_masked_and_degenerate_rows(v, dtype):
    logits, targets = make(14, v, dtype, seed=v)
    lowest = torch.finfo(dtype).min
    logits[0] = -math.inf                            # nothing left
    logits[1] = 1.5                                  # constant: every id ties
    logits[2, 5:] = -math.inf                        # five tokens left, the top list runs into the mask
    logits[3, : v - 2] = -math.inf
    logits[4] = lowest                               # masked with the type's lowest value
    logits[5, 3:] = lowest
    logits[6] = torch.arange(v, device=DEV).float().to(dtype)           # ascending
    logits[7] = -torch.arange(v, device=DEV).float().to(dtype)
    logits[8, v // 2] = math.nan
    logits[9, v // 3] = math.inf
    logits[10] = math.nan
    logits[11] = (torch.arange(v, device=DEV) % 3).to(dtype)            # massive ties
    logits[12, ::2] = -math.inf
    logits[12, 1::4] = lowest
    logits[13] = -math.inf
    logits[13, v // 2] = lowest
    targets[2] = v - 1                               # a masked token is asked for
    for n in (0, 1, 20, 32):
        check(logits, targets, n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [3001, 6150])
def test_masked_rows_among_many(v, dtype):
    """The form for many rows, whose sums treat masked elements apart."""
    logits, targets = make(10, v, dtype, seed=v)
    lowest = torch.finfo(dtype).min
    logits[0] = -math.inf
    logits[1, ::2] = -math.inf
    logits[2, 5:] = -math.inf
    logits[3, : v - 2] = -math.inf
    logits[4, 1::3] = lowest
    logits[5, v // 2] = math.nan
    logits[6, v // 3] = math.inf
    logits[7, v // 2:] = -math.inf
    logits[8, : v // 2] = lowest
    targets[2] = v - 1
    many, t = logits.repeat(60, 1), targets.repeat(60)
    check(many[290:310], t[290:310], 20)             # few rows
    whole = kernels.token_logprobs(many, t, top_n=20)
    few = kernels.token_logprobs(logits, targets, top_n=20)
    ref = plain(logits, targets, 20)
    for w, f in zip(whole, few):
        # a row is split by how its start is aligned, the same way for every eighth copy of ten rows of 2 or 4 bytes
        # an element (80 V elements are whole vectors): those have the same bits
        w = w.view(60, *f.shape).nan_to_num(7.0)
        assert torch.equal(w[8:], w[:52])
    check(many, t, 20)
    assert torch.equal(whole[3][:10].cpu(), ref[3]) and torch.equal(few[3].cpu(), ref[3])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_large_values_on_one_thread_and_large_offsets(dtype):
    """Large values that all fall to one thread's share, and a common offset far from zero."""
    logits, targets = make(3, 65536 * 2, dtype, seed=4)
    period = 256 * (16 // logits.element_size())
    logits[0, 5::period] = 50 + torch.arange(logits[0, 5::period].numel(), device=DEV).to(dtype) / 8
    logits[1] += 10000 if dtype != torch.float16 else 2000
    big = logits.repeat(300, 1)[:, :period * 40]     # one CTA per row
    check(logits, targets, 32)
    sample = torch.tensor([0, 1, 2, 897], device=DEV)
    t = targets.repeat(300) % big.shape[1]
    whole = kernels.token_logprobs(big, t, top_n=20)
    part = plain(big[sample], t[sample], 20)
    assert torch.equal(whole[3][sample].cpu(), part[3])


@pytest.mark.gpu
def test_targets_outside_the_vocabulary():
    logits, _ = make(8, 5000, torch.bfloat16, seed=1)
    targets = torch.tensor([0, 4999, 5000, -1, IGNORED, 2 ** 40, -2 ** 62, 17], device=DEV)
    check(logits, targets, 4)


@pytest.mark.gpu
def test_no_rows():
    out = kernels.token_logprobs(torch.empty(0, 100, device=DEV), torch.empty(0, dtype=torch.int64, device=DEV), 3)
    assert [tuple(o.shape) for o in out] == [(0,), (0,), (0, 3), (0, 3)]


@pytest.mark.gpu
def test_same_bits_every_time_on_another_stream_and_in_a_graph():
    logits, targets = make(40, 30011, torch.bfloat16, seed=8)
    first = kernels.token_logprobs(logits, targets, top_n=20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = kernels.token_logprobs(logits, targets, top_n=20)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = kernels.token_logprobs(logits, targets, top_n=20)
    other, _ = make(40, 30011, torch.bfloat16, seed=9)
    logits.copy_(other)
    graph.replay()
    fresh = kernels.token_logprobs(logits, targets, top_n=20)
    assert all(torch.equal(a, b) for a, b in zip(held, fresh))


# ---- refusals: no GPU needed -------------------------------------------------------------
def test_wrapper_refuses():
    l, t = torch.zeros(2, 10), torch.zeros(2, dtype=torch.int64)
    for args in ((l[0], t), (l, t[:1]), (l, t[:, None])):
        with pytest.raises(RuntimeError, match="expected logits"):
            kernels.token_logprobs(*args)
    with pytest.raises(RuntimeError, match="int64"):
        kernels.token_logprobs(l, t.int())
    for n in (-1, 11, 33):
        with pytest.raises(RuntimeError, match="top_n"):
            kernels.token_logprobs(l, t, n)
    with pytest.raises(RuntimeError, match="top_n"):
        kernels.token_logprobs(l[:, :0], t)
    with pytest.raises(RuntimeError, match="contiguous"):
        kernels.token_logprobs(torch.zeros(10, 2).T, t)
    with pytest.raises(RuntimeError, match="overlap"):
        kernels.token_logprobs(torch.zeros(1, 10).expand(2, 10), t)
    with pytest.raises(RuntimeError, match="CUDA"):
        kernels.token_logprobs(l, t)


def test_c_entry_refuses():
    if not _cabi.library_available():
        pytest.skip("library not built")
    lib = _cabi.load_library()
    good = dict(logits=4096, ld=100, R=2, V=100, dtype=1, targets=4096, top_n=2, lp=4096, ent=4096, top=4096, ids=4096)

    def call(**change):
        return lib.npb_token_logprobs(*{**good, **change}.values(), None)

    for change in ({"R": -1}, {"V": 0}, {"top_n": -1}, {"ld": 99}, {"logits": None}, {"targets": None}, {"lp": None},
                   {"ent": None}, {"top": None}, {"ids": None}):
        assert call(**change) == 1, change
    for change in ({"top_n": 33}, {"top_n": 101}, {"dtype": 3}, {"R": 1 << 27}, {"V": 1 << 30, "ld": 1 << 30}):
        assert call(**change) == 2, change
    assert call(logits=4097) == 4 and call(logits=4098, dtype=2) == 4
    assert call(R=0, logits=None) == 0
