"""The experts' block on MXFP4 weights has no backward pass: a gradient asked of it is an error."""

from __future__ import annotations

import pytest
import torch

import mmfp4
from gpu_helpers import DEV, announce

pytestmark = pytest.mark.gpu


def operands(T):
    g = torch.Generator(DEV).manual_seed(T)
    rnd = lambda *s: torch.randn(s, generator=g, device=DEV)                # noqa: E731
    gu, dn = mmfp4.mxfp4_quantize(rnd(8, 128, 96) * 0.05), mmfp4.mxfp4_quantize(rnd(8, 96, 64) * 0.05)
    return rnd(T, 96).bfloat16(), rnd(96, 8).bfloat16() * 0.1, (*gu, *dn)


@pytest.mark.parametrize("T", [3, 200])
@pytest.mark.parametrize("which", ["tokens", "router", "both"])
def test_gradients_are_an_error(T, which):
    """A layer's residual or another loss would carry a backward pass past the experts."""
    announce(f"moe_mlp_mxfp4 gradient {T} {which}")
    x, gate, w = operands(T)
    x.requires_grad_(which != "router")
    gate.requires_grad_(which != "tokens")
    probs, ids = mmfp4.moe_route(x @ gate, 2)
    y = mmfp4.moe_mlp_mxfp4(x, *w, ids, probs)
    with torch.no_grad():
        want = mmfp4.moe_mlp_mxfp4(x, *w, ids, probs)
    assert not want.requires_grad and torch.equal(y.detach(), want)
    with pytest.raises(RuntimeError, match="moe_mlp_mxfp4"):
        (x + y).float().sum().backward()
    with pytest.raises(RuntimeError, match="moe_mlp_mxfp4"):
        y = mmfp4.moe_mlp_mxfp4(x, *w, ids, probs)
        torch.autograd.grad(probs.sum() + y.sum(), gate if which != "tokens" else x)
    # without the experts' part the rest trains
    y = mmfp4.moe_mlp_mxfp4(x.detach(), *w, ids, probs.detach())
    assert torch.equal(y, want) and not y.requires_grad
    (x + y + (x @ gate).sum()).float().sum().backward()


def test_inputs_are_checked_before():
    announce("moe_mlp_mxfp4 refusals with gradients")
    x, gate, w = operands(5)
    probs, ids = mmfp4.moe_route(x @ gate.requires_grad_(True), 2)
    with pytest.raises(ValueError):
        mmfp4.moe_mlp_mxfp4(x, *w, ids[:3], probs)
    with pytest.raises(TypeError):
        mmfp4.moe_mlp_mxfp4(x, *w, ids.float(), probs)
    with pytest.raises(RuntimeError, match="GPU"):
        mmfp4.moe_mlp_mxfp4(x, *w, ids, probs.cpu())


def test_captured():
    announce("moe_mlp_mxfp4 captured with gradients enabled")
    x, gate, w = operands(40)
    gate.requires_grad_(True)

    def step():
        probs, ids = mmfp4.moe_route(x @ gate, 2)
        return mmfp4.moe_mlp_mxfp4(x, *w, ids, probs)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(3):
        x.copy_(operands(40 + i)[0][:40])
        graph.replay()
        with torch.no_grad():
            want = step()
        torch.cuda.synchronize()
        assert torch.equal(held.detach(), want)
