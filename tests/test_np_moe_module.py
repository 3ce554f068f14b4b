"""NPMoE as a module of a model: casts and moves."""

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
