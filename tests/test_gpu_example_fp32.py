"""The example's decoder trained in fp32: its attention and head as plain products, which
head sizes that the attention kernel has not take by themselves."""
import copy
import importlib.util
from pathlib import Path

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


@pytest.fixture
def example():
    path = Path(__file__).resolve().parent.parent / "examples" / "generate.py"
    spec = importlib.util.spec_from_file_location("generate_example_fp32", path)
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    return ex


def never(*args, **kw):
    raise AssertionError("a bf16 operator was called")


@pytest.mark.parametrize("rotary", [False, True])
def test_fp32(dev, example, monkeypatch, rotary):
    torch.manual_seed(0)
    model = example.Decoder(layers=2, rotary=rotary, fp32=True).to(dev)
    data = example.patterns(3, 41, torch.Generator().manual_seed(2)).to(dev)
    monkeypatch.setattr(example, "packed_attention", never)
    monkeypatch.setattr(example, "linear_cross_entropy", never)
    twin = copy.deepcopy(model)  # (a forward pass moves its layers' error feedback on)
    loss = model.loss(data[:, :-1], data[:, 1:])
    want = F.cross_entropy(twin(data[:, :-1]).flatten(0, 1), data[:, 1:].flatten())
    assert torch.equal(loss.detach(), want.detach())
    got = torch.autograd.grad(loss, list(model.parameters()))
    ref = torch.autograd.grad(want, list(twin.parameters()))
    assert all(torch.equal(a, b) for a, b in zip(got, ref))


def test_fp32_attention(dev, example):
    """Against the formula: values whose products and sums fp32 has exactly, but for
    the softmax: 2^-20 of a weight."""
    torch.manual_seed(0)
    layer = example.Layer(64, 4, 64, True)
    qkv = (torch.randint(-8, 9, (2, 9, 3 * 64)) / 4.0).to(dev)
    got = layer.attend(qkv, None, None).double().cpu()
    q, k, v = qkv.double().cpu().reshape(2, 9, 3, 4, 16).permute(2, 0, 3, 1, 4)
    s = (q @ k.transpose(-2, -1) / 4.0).masked_fill(torch.ones(9, 9).triu(1).bool(), -torch.inf)
    p = torch.softmax(s, -1)
    want = (p @ v).transpose(1, 2).reshape(2, 9, 64)
    tol = (2.0**-20 * p @ v.abs() * 4).transpose(1, 2).reshape(2, 9, 64)
    assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("heads", [2, 8])
def test_other_head_sizes_train(dev, example, heads):
    """d 256: heads of 128 by the kernel, of 32 as they were."""
    torch.manual_seed(0)
    model = example.Decoder(layers=1, heads=heads).to(dev)
    losses = example.train(model, 2, seq=32, batch=2)
    assert all(torch.isfinite(torch.tensor(losses)))
    assert all(p.grad is not None and p.grad.any() for p in model.parameters())
