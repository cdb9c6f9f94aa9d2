"""Attention within packed sequences: how many sequences and heads a call takes."""
import pytest
import torch

from tcfp_amd import attention as A

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def test_sequences_times_heads(dev):
    """As many as a launch's grid takes, and a ValueError past that."""
    at = torch.full((65536,), 4, dtype=torch.int32, device=dev)
    at[0] = 0
    for heads, kv in ((256, 256), (256, 32)):
        q = torch.randn(4, heads, 64, device=dev).to(BF16).requires_grad_()
        k, v = (torch.randn(4, kv, 64, device=dev).to(BF16).requires_grad_() for _ in range(2))
        o = A.packed_attention(q, k, v, at, max_len=4)
        got = (o, *torch.autograd.grad(o, (q, k, v), torch.ones_like(o)))
        o = A.packed_attention(q, k, v, at[:2], max_len=4)
        want = (o, *torch.autograd.grad(o, (q, k, v), torch.ones_like(o)))
        for a, b in zip(got, want):
            torch.testing.assert_close(a, b, rtol=3 * 2.0**-8, atol=1e-4 * float(b.detach().abs().max()))
    for heads, kv in ((257, 257), (512, 8), (65535, 1)):
        q = torch.zeros(4, heads, 64, dtype=BF16, device=dev)
        k = torch.zeros(4, kv, 64, dtype=BF16, device=dev)
        with pytest.raises(ValueError, match="sequences"):
            A.packed_attention(q, k, k, at, max_len=4)
        with pytest.raises(ValueError, match="sequences"):
            A.packed_attention(q.requires_grad_(), k, k, at, max_len=4)
