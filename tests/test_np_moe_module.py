"""NPMoE as a module of a model: casts, moves and the limits of its kernel."""

import pytest
import torch
from torch import nn

from neuropress_b200.nn import NPMoE
from test_moe_and_scores import Expert

DEV = "cuda"


def make(asym=True):
    router = nn.Linear(64, 3, bias=False)
    with torch.no_grad():
        router.weight.copy_(torch.randn(3, 64, generator=torch.Generator().manual_seed(1)) / 8)
    return NPMoE.from_experts(router, [Expert(64, 96, s, asym=asym) for s in range(3)], 2)


@pytest.mark.parametrize("asym", [False, True])
@pytest.mark.parametrize("cast", [lambda m: m.to(torch.bfloat16), lambda m: m.half(), lambda m: m.float(),
                                  lambda m: m.double(), lambda m: m.bfloat16().float(),
                                  lambda m: m.to("cpu", torch.bfloat16)])
def test_a_cast_leaves_the_packed_weights(cast, asym):
    moe = make(asym)
    before = {k: v.clone() for k, v in moe.state_dict().items()}
    assert cast(moe) is moe
    for name, b in moe.named_buffers():
        assert b.dtype == before[name].dtype and torch.equal(b, before[name]), name
    assert moe.router.weight.dtype == cast(nn.Linear(2, 2)).weight.dtype


def test_a_cast_inside_a_model_and_an_empty_move():
    model = nn.Sequential(make(), nn.Linear(64, 4)).to(torch.bfloat16)
    assert model[0].gate_scale.dtype == torch.float16 and model[1].weight.dtype == torch.bfloat16
    meta = make().to("meta")
    assert meta.up_scale.device.type == "meta" and meta.up_scale.dtype == torch.float16
    assert meta.to_empty(device="cpu").up_scale.shape == make().up_scale.shape


@pytest.mark.gpu
def test_moved_and_cast_in_one_step_it_runs():
    want = make()
    want.router.to(torch.bfloat16)
    want.to(DEV)
    got = make().to(DEV, torch.bfloat16)
    x = torch.randn(5, 64, generator=torch.Generator().manual_seed(2)).to(DEV, torch.bfloat16)
    assert torch.equal(got(x), want(x))
    assert got.gate_scale.is_cuda and got.gate_scale.dtype == torch.float16


def test_the_kernels_limits_are_checked_when_it_is_built():
    def weight(e, rows, cols):
        codes = torch.zeros(1, 1, 1, dtype=torch.uint8).expand(e, rows, cols // 2)
        return codes, torch.zeros(1), None

    def build(e, h, i, top_k):
        return NPMoE(nn.Identity(), weight(e, i, h), weight(e, i, h), weight(e, h, i), top_k, 32)

    assert build(32, 32, 32, 16).top_k == 16
    with pytest.raises(ValueError, match="top_k"):
        build(32, 32, 32, 17)
    with pytest.raises(ValueError, match="at most 512 experts"):
        build(513, 32, 32, 2)
    for h, i in ((16416, 32), (32, 16416)):
        with pytest.raises(ValueError, match="at most 16384"):
            build(1, h, i, 1)
