"""BidirectionalMamba with fused_block: the same block with its norm,
projections and MLP in this package's kernels."""

import importlib.util
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu


def _pair(cuda, **kw):
    from selectssm_b200 import BidirectionalMamba
    blocks = []
    for fused in (False, True):
        torch.manual_seed(0)
        blocks.append(BidirectionalMamba(64, hidden_features=16, expansion_factor=2.0, mlp_layer=True, fused_block=fused,
                                         **kw).to(cuda))
    for a, b in zip(blocks[0].parameters(), blocks[1].parameters()):
        assert torch.equal(a, b)
    return blocks


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-4), (torch.bfloat16, 3e-2)])
@pytest.mark.parametrize("kw", [{"norm_type": "group"}, {"norm_type": "rms", "activation": "gelu"},
                                {"norm_type": "layer", "concatenate_fwd_rev": False, "activation": "relu"},
                                {"norm_type": "none", "complement": True, "tie_in_proj": True, "tie_gate": True}])
def test_fused_block_equals_unfused(cuda, dtype, tol, kw):
    """Without dropout both compute the same block (the framework's parity
    tolerances: 1e-4 of the largest value in fp32; bf16 rounds intermediate
    results in different places)."""
    plain, fused = _pair(cuda, **kw)
    x = torch.randn(2, 96, 64, device=cuda).to(dtype)
    dy = torch.randn(2, 96, 64, device=cuda).to(dtype)
    outs = []
    for m in (plain, fused):
        xi = x.clone().requires_grad_()
        y = m(xi)
        y.backward(dy)
        outs.append([y.detach(), xi.grad, *[p.grad for p in m.parameters()]])
    if kw.get("activation") == "relu" and dtype == torch.bfloat16:
        # a value that bf16 rounds to either side of relu's kink has either slope,
        # so only the outputs are comparable (the gradients are, in fp32)
        outs = [o[:1] for o in outs]
    for a, b in zip(*outs):
        assert float((a.float() - b.float()).abs().max()) <= tol * float(a.float().abs().max())


def test_dropout_follows_the_given_rng(cuda):
    _, m = _pair(cuda, norm_type="group", mlp_dropout_rate=0.3)
    x = torch.randn(2, 50, 64, device=cuda)
    a, b = m(x, train=True, dropout_rng=(1, 2)), m(x, train=True, dropout_rng=(1, 2))
    assert torch.equal(a, b)
    rng = torch.tensor([1, 2], dtype=torch.int64, device=cuda)
    assert torch.equal(a, m(x, train=True, dropout_rng=rng))
    assert not torch.equal(a, m(x, train=True, dropout_rng=(1, 4)))
    assert torch.equal(m(x), m(x, dropout_rng=(5, 5)))      # no dropout outside training
    torch.manual_seed(3)
    c = m(x, train=True)
    torch.manual_seed(3)
    assert torch.equal(c, m(x, train=True))
    assert not torch.equal(c, m(x, train=True))


def test_example_learns(cuda, monkeypatch):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "train_block.py")
    spec = importlib.util.spec_from_file_location("train_block", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    monkeypatch.setattr(sys, "argv", ["train_block.py", "--steps", "60", "--length", "128", "--width", "64"])
    first, last = example.main()
    assert first > 1.0 and last < 0.8 * first  # chance is log 4


def test_a_captured_step_needs_a_device_rng(cuda):
    """Seeds drawn on the host would be frozen into the graph with their mask."""
    _, m = _pair(cuda, norm_type="group", mlp_dropout_rate=0.3)
    x = torch.randn(2, 50, 64, device=cuda)
    rng = torch.tensor([1, 2], dtype=torch.int64, device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.no_grad(), torch.cuda.stream(side):
        m(x, train=True)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="dropout_rng"):
            m(x, train=True)
        y = m(x, train=True, dropout_rng=rng)
        m(x)  # nothing is drawn
    outs = []
    for offset in (2, 4):
        rng[1] = offset
        graph.replay()
        torch.cuda.synchronize()
        outs.append(y.clone())
        with torch.no_grad():
            assert torch.equal(y, m(x, train=True, dropout_rng=(1, offset)))
    assert not torch.equal(*outs)
