"""What examples/generate.py refuses before anything reaches the GPU (no GPU
needed: the model's tables and the page lists stay on the CPU)."""
import importlib.util
from pathlib import Path

import pytest
import torch


@pytest.fixture
def server(monkeypatch):
    path = Path(__file__).resolve().parent.parent / "examples" / "generate.py"
    spec = importlib.util.spec_from_file_location("generate_example_cpu", path)
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    monkeypatch.setattr(ex.K, "fused_dual_quantize_fp8", lambda w, block: (w, w, w, w))
    return ex.Server(ex.Decoder(layers=1, positions=32))


@pytest.mark.parametrize("tokens,match", [
    ([[1] * 33], "32 positions"), ([[1, 256]], "tokens must lie"), ([[-1]], "tokens must lie")])
def test_indices_that_a_table_does_not_have(server, tokens, match):
    seq = server.cache.open()
    with pytest.raises(ValueError, match=match):
        server.step([seq], tokens)
    assert server.cache.length(seq) == 0 and server.cache.free_pages == 256


def test_a_sequence_that_grows_past_the_positions(server):
    seq = server.cache.open()
    server.cache.extend([seq], [32])
    with pytest.raises(ValueError, match="32 positions"):
        server.step([seq], [[5]])
    assert server.cache.length(seq) == 32
    with pytest.raises(ValueError, match="32 positions"):
        server.generate([[1] * 33], 1)
    assert server.cache.free_pages == 254  # (what the refused prompt opened is closed)
    with pytest.raises(ValueError, match="32 positions"):
        server.model(torch.zeros(1, 33, dtype=torch.long))


def test_nothing_to_generate(server):
    assert server.generate([[1], [2, 3]], 0) == [[], []]
    with pytest.raises(ValueError, match="a prompt"):
        server.generate([[1], []], 4)
