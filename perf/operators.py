"""Cases and plain forms of the operators next to the quantized linears.

Three operators are measured, each as a user's program calls it:

``gemm``      dense product with bias, activation and residual add in its epilogue:
              ``y = T(act(x W^T + b) + r)``.
``moe``       a mixture-of-experts layer for a few tokens over 4-bit group-affine experts:
              softmax routing, gate / up products, ``silu(gate) * up``, down product, weighted sum.
``logprobs``  log probabilities of given tokens with entropy and the top alternatives.

With ``own`` false ``run`` computes them with elementary torch operations in 32 bits, rounded once
at the end; with ``own`` true it calls ``neuropress_b200.kernels``.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one token through a square projection with the residual add behind it: latency and the weight's stream
        {"name": "gemm_1x4096x4096", "op": "gemm", "m": 1, "n": 4096, "k": 4096, "dtype": "bf16", "bias": False,
         "act": "none", "residual": True},
        # a small decode batch through the first product of an MLP, bias and gelu
        {"name": "gemm_16x14336x4096", "op": "gemm", "m": 16, "n": 14336, "k": 4096, "dtype": "bf16", "bias": True,
         "act": "gelu", "residual": False},
        # a ragged batch of short prompts through a down projection: odd rows, long K, few tiles
        {"name": "gemm_201x4096x14336", "op": "gemm", "m": 201, "n": 4096, "k": 14336, "dtype": "fp16", "bias": True,
         "act": "none", "residual": True},
        # a prefill of 4096 rows through the widest projection
        {"name": "gemm_4096x28672x8192", "op": "gemm", "m": 4096, "n": 28672, "k": 8192, "dtype": "bf16",
         "bias": False, "act": "silu", "residual": False},
        # one token, 8 of 64 experts
        {"name": "moe_1_e64_k8", "op": "moe", "t": 1, "e": 64, "top_k": 8, "h": 2048, "i": 1024, "g": 32,
         "asym": False, "dtype": "bf16", "renorm": True},
        # four tokens, 2 of 8 large experts, zero points
        {"name": "moe_4_e8_k2", "op": "moe", "t": 4, "e": 8, "top_k": 2, "h": 4096, "i": 14336, "g": 64,
         "asym": True, "dtype": "fp16", "renorm": True},
        # 32 tokens, 8 of 64: most experts are read, about four tokens each; ragged widths
        {"name": "moe_32_e64_k8", "op": "moe", "t": 32, "e": 64, "top_k": 8, "h": 4096, "i": 1376, "g": 32,
         "asym": False, "dtype": "bf16", "renorm": False},
        # the token just sampled: one row
        {"name": "logprobs_1x32000", "op": "logprobs", "r": 1, "v": 32000, "pad": 0, "top_n": 5, "dtype": "bf16"},
        # a decode batch with alternatives, vocabulary padded to a wider row
        {"name": "logprobs_33x128000", "op": "logprobs", "r": 33, "v": 128000, "pad": 256, "top_n": 20,
         "dtype": "bf16"},
        # rows of odd length, fp32 logits: no row after the first starts on a 16-byte boundary
        {"name": "logprobs_300x50001", "op": "logprobs", "r": 300, "v": 50001, "pad": 0, "top_n": 8, "dtype": "fp32"},
        # the perplexity of a long text
        {"name": "logprobs_4096x128000", "op": "logprobs", "r": 4096, "v": 128000, "pad": 0, "top_n": 0,
         "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["gemm", "moe", "logprobs"])
    if op == "gemm":
        m = _log_int(rng, 1, 4096)
        n = _log_int(rng, 256, 16384)
        k = 8 * _log_int(rng, 32, 1792)
        return {"op": op, "m": m, "n": n, "k": k, "dtype": rng.choice(["bf16", "fp16"]), "bias": rng.random() < 0.5,
                "act": rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]), "residual": rng.random() < 0.5}
    if op == "moe":
        g = rng.choice([32, 64, 128])
        e = _log_int(rng, 4, 64)
        return {"op": op, "t": _log_int(rng, 1, 32), "e": e, "top_k": rng.randint(1, min(8, e)),
                "h": g * _log_int(rng, 512 // g, 4096 // g), "i": g * _log_int(rng, 256 // g, 1376 // g), "g": g,
                "asym": rng.random() < 0.5, "dtype": rng.choice(["bf16", "fp16"]), "renorm": rng.random() < 0.5}
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    v = _log_int(rng, 1000, 160000)
    r = _log_int(rng, 1, max(2, min(4096, 4096 * 128000 // (v * (2 if dtype == "fp32" else 1)))))
    return {"op": op, "r": r, "v": v, "pad": rng.choice([0, 0, 7, 64]), "top_n": rng.randint(0, 20), "dtype": dtype}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)

    if case["op"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        return {"case": case, "x": normal(m, k, dtype=dt), "w": normal(n, k, scale=k ** -0.5, dtype=dt),
                "bias": normal(n, scale=0.5) if case["bias"] else None,
                "residual": normal(m, n, dtype=dt) if case["residual"] else None}
    if case["op"] == "moe":
        t, e, h, i, g = case["t"], case["e"], case["h"], case["i"], case["g"]

        def weight(rows, cols):
            codes = torch.randint(0, 256, (e, rows, cols // 2), generator=gen, device="cuda", dtype=torch.uint8)
            # codes have a standard deviation of 4.6: products of unit inputs come out near unit size
            scale = (torch.rand(e, rows, cols // g, generator=gen, device="cuda") + 0.5) * (0.2 * cols ** -0.5)
            zero = torch.rand(e, rows, cols // g, generator=gen, device="cuda") * 2 + 7 if case["asym"] else None
            return codes, scale.half(), None if zero is None else zero.half()

        return {"case": case, "x": normal(t, h, dtype=dt), "logits": normal(t, e, scale=1.5),
                "gate": weight(i, h), "up": weight(i, h), "down": weight(h, i)}
    r, v = case["r"], case["v"]
    rows = normal(r, v + case["pad"], scale=2.5, dtype=dt)
    # the few tokens a trained model finds likely, and a masked part of the vocabulary
    likely = torch.randint(0, v, (r, 8), generator=gen, device="cuda")
    rows.scatter_add_(1, likely, normal(r, 8, scale=4.0).abs().to(dt) + 6)
    rows[:, v - v // 100:v] = -math.inf
    targets = torch.randint(0, v - v // 100, (r,), generator=gen, device="cuda")
    targets[torch.rand(r, generator=gen, device="cuda") < 0.05] = -100
    return {"case": case, "logits": rows[:, :v], "targets": targets}


def run(state):
    case = state["case"]
    if own:
        return _own(case, state)
    if case["op"] == "gemm":
        return _plain_gemm(case, state)
    if case["op"] == "moe":
        return _plain_moe(case, state)
    return _plain_logprobs(case, state)


def _own(case, state):
    from neuropress_b200 import kernels

    if case["op"] == "gemm":
        return kernels.gemm_epilogue(state["x"], state["w"], state["bias"], activation=case["act"],
                                     residual=state["residual"])
    if case["op"] == "moe":
        return kernels.q_moe(state["x"], state["logits"], state["gate"], state["up"], state["down"], case["top_k"],
                             case["g"], renormalize=case["renorm"])
    out = kernels.token_logprobs(state["logits"], state["targets"], top_n=case["top_n"])
    return {"logprob": out[0], "entropy": out[1], "top_logprobs": out[2], "top_ids": out[3]}


def _plain_gemm(case, state):
    y = state["x"].float() @ state["w"].float().T
    if state["bias"] is not None:
        y = y + state["bias"]
    act = case["act"]
    if act == "relu":
        y = y.clamp_min(0)
    elif act == "silu":
        y = y / (1 + torch.exp(-y))
    elif act == "gelu":
        y = 0.5 * y * torch.erfc(y * -(0.5 ** 0.5))
    elif act == "gelu_tanh":
        y = 0.5 * y * (1 + torch.tanh((2 / math.pi) ** 0.5 * (y + 0.044715 * y * y * y)))
    if state["residual"] is not None:
        y = y + state["residual"].float()
    return y.to(state["x"].dtype)


def _first_largest(values, n):
    """Indices of the n largest along the last axis, equal values by ascending index."""
    bits = (values.float() + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)  # a larger float has a larger whole number
    index = torch.arange(values.shape[-1], device=values.device)
    return torch.topk(order * 2 ** 20 + (2 ** 20 - 1 - index), n, dim=-1).indices


def _chosen_weights(weight, ids, g):
    """The experts' [t, k, rows, cols] weights in 32 bits: (q - z) * s."""
    codes, scale, zero = weight
    codes = codes[ids]
    q = torch.stack((codes & 15, codes >> 4), dim=-1).float()
    q = q.reshape(*codes.shape[:-1], codes.shape[-1] * 2 // g, g)
    z = 8.0 if zero is None else zero[ids].float()[..., None]
    return ((q - z) * scale[ids].float()[..., None]).flatten(-2)


def _plain_moe(case, state):
    x, logits = state["x"].float(), state["logits"].float()
    ids = _first_largest(logits, case["top_k"])
    p = torch.exp(logits - logits.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    p = p.gather(1, ids)
    if case["renorm"]:
        p = p / p.sum(-1, keepdim=True)
    gate = (_chosen_weights(state["gate"], ids, case["g"]) @ x[:, None, :, None])[..., 0]
    up = (_chosen_weights(state["up"], ids, case["g"]) @ x[:, None, :, None])[..., 0]
    h = gate / (1 + torch.exp(-gate)) * up
    out = (_chosen_weights(state["down"], ids, case["g"]) @ h[..., None])[..., 0]
    return (out * p[..., None]).sum(1).to(state["x"].dtype)


def _plain_logprobs(case, state):
    logits, targets, n = state["logits"].float(), state["targets"], case["top_n"]
    d = logits - logits.amax(-1, keepdim=True)
    p = torch.exp(d)
    total = p.sum(-1)
    lse = torch.log(total)
    entropy = lse - torch.where(p > 0, p * d, 0.0).sum(-1) / total
    known = (targets >= 0) & (targets < case["v"])
    chosen = d.gather(1, torch.where(known, targets, 0)[:, None])[:, 0] - lse
    ids = _first_largest(state["logits"], n)
    return {"logprob": torch.where(known, chosen, 0.0), "entropy": entropy,
            "top_logprobs": d.gather(1, ids) - lse[:, None], "top_ids": ids}


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        moved = size * (m * k + n * k + m * n * (2 if case["residual"] else 1)) + (4 * n if case["bias"] else 0)
        return {"bytes": moved, "flops": 2 * m * n * k}
    if case["op"] == "moe":
        t, e, k, h, i = case["t"], case["e"], case["top_k"], case["h"], case["i"]
        read = e * (1 - (1 - k / e) ** t)  # experts that t tokens choose, on average
        per_expert = 3 * h * i * (0.5 + (4 if case["asym"] else 2) / case["g"])
        return {"bytes": int(read * per_expert + 2 * size * t * h + 4 * t * e), "flops": 6 * t * k * h * i}
    r, v = case["r"], case["v"]
    return {"bytes": r * v * size + r * (16 + 12 * case["top_n"]), "flops": 5 * r * v}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "gemm":
        y = torch.nn.functional.linear(s["x"].double(), s["w"].double(),
                                       None if s["bias"] is None else s["bias"].double())
        if case["act"] == "relu":
            y = torch.relu(y)
        elif case["act"] == "silu":
            y = torch.nn.functional.silu(y)
        elif case["act"] != "none":
            y = torch.nn.functional.gelu(y, approximate="tanh" if case["act"] == "gelu_tanh" else "none")
        return y if s["residual"] is None else y + s["residual"].double()
    if case["op"] == "moe":
        probs = torch.softmax(s["logits"].double(), -1)
        order = torch.sort(s["logits"].double(), dim=-1, descending=True, stable=True).indices[:, :case["top_k"]]
        share = torch.zeros_like(probs).scatter(1, order, probs.gather(1, order))
        if case["renorm"]:
            share = share / share.sum(-1, keepdim=True)
        y = torch.zeros(s["x"].shape, dtype=torch.float64, device="cuda")

        def dense(weight, e):
            codes, scale, zero = (None if w is None else w[e] for w in weight)
            q = torch.empty(codes.shape[0], codes.shape[1] * 2, dtype=torch.float64, device="cuda")
            q[:, 0::2], q[:, 1::2] = (codes % 16).double(), (codes // 16).double()
            wide = scale.double().repeat_interleave(case["g"], 1)
            return (q - (8 if zero is None else zero.double().repeat_interleave(case["g"], 1))) * wide

        for e in range(case["e"]):
            h = torch.nn.functional.silu(s["x"].double() @ dense(s["gate"], e).T) * (s["x"].double()
                                                                                 @ dense(s["up"], e).T)
            y += share[:, e:e + 1] * (h @ dense(s["down"], e).T)
        return y
    logp = torch.log_softmax(s["logits"].double(), -1)
    entropy = torch.special.entr(torch.exp(logp)).sum(-1)
    known = s["targets"] >= 0
    given = logp[torch.arange(case["r"], device="cuda"), s["targets"].clamp_min(0)]
    top = torch.sort(logp, dim=-1, descending=True, stable=True)
    n = case["top_n"]
    return {"logprob": torch.where(known, given, 0.0), "entropy": entropy, "top_logprobs": top.values[:, :n].clone(),
            "top_ids": top.indices[:, :n].clone()}
