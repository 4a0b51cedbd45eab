"""The local-attention example, end to end: it trains every weight and its cached steps agree with one pass."""

import importlib.util
import os

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("window_attention_example",
                                                  os.path.join(ROOT, "examples", "window_attention.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_training_and_generation(example):
    first, last, _, apart = example.run(steps=40, n=96, B=8, n_new=24, log=None)
    assert last < 0.75 * first
    # two bfloat16 results of one formula, through a projection and a layer norm: each logit is a sum of 64 terms
    # of order 1/8 x 1 with relative differences of about 2^-8
    assert apart < 16 * 2.0 ** -8


def test_every_weight_gets_a_gradient(example):
    torch.manual_seed(1)
    model = example.Model().cuda()
    with torch.no_grad():
        for m in (model.source, model.transport, model.answer):
            m.pos_weight.normal_(std=0.3)
    tokens, source = example.batch(4, 70, torch.Generator().manual_seed(1), "cuda")
    model(tokens, source).square().mean().backward()
    for name, p in model.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all(), name
        assert float(p.grad.abs().max()) > 0, name
