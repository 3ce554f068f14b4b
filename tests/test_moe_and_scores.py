"""The modules over the new kernels, and the kernels together as a decoder uses them."""

import math

import pytest
import torch
import torch.nn.functional as F
from torch import nn

from helpers import assert_output_close, half_ulp
from neuropress_b200 import kernels
from neuropress_b200.nn import NPLinear, NPMoE, NPRMSNorm, TokenScores, score_tokens
from synthetic import make_q_layer

DEV = "cuda"


def q_linear(n, k, seed, gs=32, asym=False, bias=False):
    d = make_q_layer(n, k, group_size=gs, asym=asym, seed=seed, bias=bias)
    return NPLinear(d.codes, d.scale, n, k, gs, 4, "asym" if asym else "sym", "auto", bias=d.bias, zero_point=d.zero_point)


def dense(m):
    """The linear's weight in 64 bits."""
    q = torch.empty(m.out_features, m.in_features, dtype=torch.float64)
    codes = m.u8_blob.cpu()
    q[:, 0::2], q[:, 1::2] = (codes & 15).double(), (codes >> 4).double()
    wide = lambda t: t.cpu().double().view(m.out_features, -1).repeat_interleave(m.group_size, 1)  # noqa: E731
    return (q - (8.0 if m.zero_point is None else wide(m.zero_point))) * wide(m.scale)


class Expert(nn.Module):
    def __init__(self, h, i, seed, names=("gate_proj", "up_proj", "down_proj"), **kw):
        super().__init__()
        for k, (name, n, width) in enumerate(zip(names, (i, i, h), (h, h, i))):
            setattr(self, name, q_linear(n, width, seed * 3 + k, **kw))


def moe_reference(experts, x, logits, top_k, renorm):
    y = torch.zeros(x.shape, dtype=torch.float64)
    spread = torch.zeros_like(y)
    for t in range(x.shape[0]):
        p = torch.softmax(logits[t].double(), -1)
        top = torch.sort(p, descending=True, stable=True).indices[:top_k]
        w = p[top] / (p[top].sum() if renorm else 1.0)
        for weight, e in zip(w, top.tolist()):
            g, u, d = (dense(m) for m in experts[e])
            h = F.silu(g @ x[t].double()) * (u @ x[t].double())
            y[t] += weight * (d @ h)
            spread[t] += weight * (d.abs() @ h.abs())
    return y, spread


def assert_moe_close(y, ref, dtype):
    ref, spread = ref   # 11 significant bits of h between the kernels, then fp32 (see test_q_moe.assert_close)
    y = y.detach().cpu().double()
    rms = ref.square().mean(-1, keepdim=True).sqrt()
    assert float(((y - ref).abs() - half_ulp(ref, dtype) - 2.0 ** -12 * spread - 2e-4 * rms).max()) <= 0


@pytest.mark.gpu
@pytest.mark.parametrize("asym,gs", [(False, 32), (True, 64)])
@pytest.mark.parametrize("shape", [(1,), (7,), (2, 3), (40,)])
def test_module_matches_its_experts(shape, asym, gs):
    h, i, e = 256, 192, 6
    experts = [Expert(h, i, s, gs=gs, asym=asym) for s in range(e)]
    g = torch.Generator().manual_seed(sum(shape))
    router = nn.Linear(h, e, bias=False)
    with torch.no_grad():
        router.weight.copy_(torch.randn(e, h, generator=g) * h ** -0.5 * 2)
    moe = NPMoE.from_experts(router.to(torch.bfloat16), experts, 2).to(DEV)
    x = torch.randn(*shape, h, generator=g).to(torch.bfloat16)
    y = moe(x.to(DEV))
    assert y.shape == x.shape and y.dtype == torch.bfloat16
    x2 = x.reshape(-1, h)
    logits = moe.router(x2.to(DEV)).detach().cpu()
    triples = [(m.gate_proj, m.up_proj, m.down_proj) for m in experts]
    assert_moe_close(y.reshape(-1, h), moe_reference(triples, x2, logits, 2, True), torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,chunk", [(5, 1024), (50, 16), (33, 32)])
def test_scores_of_a_lowered_head(rows, chunk):
    h, v = 512, 1000
    head = q_linear(v, h, seed=3).to(DEV)
    g = torch.Generator().manual_seed(rows)
    hidden = torch.randn(1, rows, h, generator=g).to(torch.bfloat16).to(DEV)
    targets = torch.randint(0, 990, (1, rows), generator=g)
    targets[0, 2] = -100
    got = score_tokens(head, hidden, targets.to(DEV), top_n=4, rows_per_chunk=chunk, vocab_size=990)
    assert isinstance(got, TokenScores) and got.logprob.shape == (1, rows) and got.top_ids.shape == (1, rows, 4)
    # the head's bands round differently at other row counts: the reference reads the logits chunk by chunk too
    logits = torch.cat([head(hidden[0, r:r + chunk]) for r in range(0, rows, chunk)])[:, :990].double().cpu()
    logp = torch.log_softmax(logits, -1)
    want = torch.where(targets[0] >= 0, logp.gather(1, targets[0].clamp_min(0)[:, None])[:, 0], 0.0)
    assert float((got.logprob[0].double().cpu() - want).abs().max()) <= 2.0 ** -24 * 200 * 16
    assert torch.equal(got.top_ids[0].cpu(), torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :4])
    entropy = torch.special.entr(logp.exp()).sum(-1)
    assert float((got.entropy[0].double().cpu() - entropy).abs().max()) <= 2.0 ** -24 * 200 * 16


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 6, 45])
def test_a_decoder_block_and_its_scores(rows):
    """Norm -> experts -> residual; norm -> dense MLP with bias + gelu and bias + residual in the epilogues; norm ->
    lm_head -> scores: each step against 64 bits from the step before it, then all of it captured and replayed."""
    h, i, e, v = 256, 128, 5, 700
    g = torch.Generator().manual_seed(rows)
    rnd = lambda *s, scale=1.0: (torch.randn(*s, generator=g) * scale).to(torch.bfloat16)  # noqa: E731
    experts = [Expert(h, i, s, names=("w1", "w3", "w2")) for s in range(e)]
    router = nn.Linear(h, e, bias=False).to(torch.bfloat16)
    with torch.no_grad():
        router.weight.copy_(rnd(e, h, scale=h ** -0.5 * 2))
    moe = NPMoE.from_experts(router, experts, 2, renormalize=False).to(DEV)
    norm = NPRMSNorm((torch.rand(h, generator=g) + 0.5).to(torch.bfloat16), 1e-5).to(DEV)
    w1, w2 = rnd(4 * h, h, scale=h ** -0.5).to(DEV), rnd(h, 4 * h, scale=h ** -0.5 / 2).to(DEV)
    b1, b2 = torch.randn(4 * h, generator=g).to(DEV), torch.randn(h, generator=g).to(DEV)
    head = q_linear(v, h, seed=9).to(DEV)
    x = rnd(rows, h).to(DEV)
    targets = torch.randint(0, v, (rows,), generator=g).to(DEV)

    def run():
        a = norm(x)
        m = moe(a)
        x1 = x + m
        b = norm(x1)
        f = kernels.gemm_epilogue(b, w1, b1, "gelu")
        x2 = kernels.gemm_epilogue(f, w2, b2, residual=x1)
        return a, m, x1, b, f, x2, score_tokens(head, norm(x2), targets, top_n=3)

    a, m, x1, b, f, x2, scores = run()
    triples = [(t.w1, t.w3, t.w2) for t in experts]
    assert_moe_close(m, moe_reference(triples, a.cpu(), moe.router(a).detach().cpu(), 2, False), torch.bfloat16)
    d = lambda t: t.double().cpu()  # noqa: E731
    assert_output_close(f, F.gelu(d(b) @ d(w1).T + d(b1)), torch.bfloat16, tol=5e-4)
    assert_output_close(x2, d(f) @ d(w2).T + d(b2) + d(x1), torch.bfloat16, tol=5e-4)
    logits = d(head(norm(x2)))
    logp = torch.log_softmax(logits, -1).gather(1, targets.cpu()[:, None])[:, 0]
    assert float((d(scores.logprob) - logp).abs().max()) <= 2.0 ** -24 * 200 * (1 + float(logp.abs().max()))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        again = run()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(again[:6], (a, m, x1, b, f, x2)))
    assert all(torch.equal(p, q) for p, q in zip(again[6], scores))


# ---- on the CPU ---------------------------------------------------------------------------
def test_from_experts_stacks_the_wire_format():
    experts = [Expert(64, 96, s, asym=True) for s in range(3)]
    moe = NPMoE.from_experts(nn.Linear(64, 3), experts, 2)
    assert (moe.num_experts, moe.hidden_size, moe.intermediate_size, moe.group_size) == (3, 64, 96, 32)
    assert torch.equal(moe.up_codes[1], experts[1].up_proj.u8_blob)
    assert torch.equal(moe.down_scale.view(3, -1)[2], experts[2].down_proj.scale)
    assert torch.equal(moe.gate_zero_point.view(3, -1)[0], experts[0].gate_proj.zero_point)
    again = NPMoE.from_experts(nn.Linear(64, 3), [Expert(64, 96, s + 7, asym=True) for s in range(3)], 2)
    again.load_state_dict(moe.state_dict())
    assert all(torch.equal(p, q) for p, q in zip(again.buffers(), moe.buffers()))
    pairs = NPMoE.from_experts(nn.Linear(64, 3), [(x.gate_proj, x.up_proj, x.down_proj) for x in experts], 1)
    assert torch.equal(pairs.gate_codes, moe.gate_codes)


def test_from_experts_refuses():
    router = nn.Linear(64, 2)
    good = [Expert(64, 96, s) for s in range(2)]
    with pytest.raises(ValueError, match="at least one"):
        NPMoE.from_experts(router, [], 1)
    with pytest.raises(ValueError, match="three NPLinear"):
        NPMoE.from_experts(router, [good[0], nn.Linear(4, 4)], 1)
    for other in (Expert(64, 96, 5, bias=True), Expert(64, 96, 5, gs=16)):
        with pytest.raises(ValueError, match="without bias"):
            NPMoE.from_experts(router, [good[0], other], 1)
    for other in (Expert(64, 128, 5), Expert(64, 96, 5, asym=True)):
        with pytest.raises(ValueError, match="agree"):
            NPMoE.from_experts(router, [good[0], other], 1)
    for k in (0, 3):
        with pytest.raises(ValueError, match="top_k"):
            NPMoE.from_experts(router, good, k)
    with pytest.raises(ValueError, match="group_size"):
        NPMoE.from_experts(router, [Expert(64, 96, 1, gs=16)], 1)
    moe = NPMoE.from_experts(router, good, 1)
    with pytest.raises(RuntimeError, match="float16 or bfloat16"):
        moe(torch.zeros(2, 64))
    with pytest.raises(RuntimeError, match="CUDA"):
        moe.to(torch.float16)(torch.zeros(2, 64, dtype=torch.float16))


def test_score_tokens_refuses_and_takes_nothing():
    head = nn.Linear(8, 20)
    with pytest.raises(RuntimeError, match="expected hidden"):
        score_tokens(head, torch.zeros(3, 8), torch.zeros(4, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="rows_per_chunk"):
        score_tokens(head, torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64), rows_per_chunk=0)
    with pytest.raises(RuntimeError, match="CUDA"):
        score_tokens(head, torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64))
    none = score_tokens(head, torch.zeros(2, 0, 8), torch.zeros(2, 0, dtype=torch.int64), top_n=3)
    assert none.logprob.shape == (2, 0) and none.top_ids.shape == (2, 0, 3) and math.prod(none.entropy.shape) == 0
