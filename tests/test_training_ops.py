"""The training operators' host side: frequencies, refusals, workspaces (no GPU
needed)."""
import ctypes
import math

import pytest
import torch

from tcfp_amd import _hip, attention, loss, rotary
from test_lds_copy_waits import _code_objects, short_waits


def status(name, *args):
    lib = _hip.load_library()
    rc = getattr(lib, name)(*args)
    return lib.tcfp_status_string(rc).decode() if rc else "ok"


BUF = ctypes.create_string_buffer(4096)
PTR = (ctypes.addressof(BUF) + 255) // 256 * 256  # never read: the calls are refused


# ---------------------------------------------------------------- frequencies


def test_frequencies():
    f = rotary.rotary_frequencies(8, base=16.0)
    assert f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([1.0, 0.5, 0.25, 0.125], dtype=torch.float64), rtol=1e-15)
    assert torch.equal(rotary.rotary_frequencies(8, base=16.0, factor=4.0), f / 4)
    # a trained length of 64: 10.2, 5.1, 2.5 and 1.27 turns
    got = rotary.rotary_frequencies(8, base=16.0, factor=4.0, trained_length=64, slow_turns=2.0,
                                    fast_turns=6.0)
    turns = 64 * f / (2 * math.pi)
    keep = ((turns - 2) / 4).clamp(0, 1)
    assert float(keep[0]) == 1.0 and 0 < float(keep[1]) < 1 and float(keep[3]) == 0.0
    assert torch.allclose(got, f * (keep + (1 - keep) / 4), rtol=1e-15)


@pytest.mark.parametrize("kw", [
    dict(dim=7), dict(dim=0), dict(dim=8, base=0.0), dict(dim=8, base=math.inf),
    dict(dim=8, factor=0.5), dict(dim=8, factor=math.nan), dict(dim=8, trained_length=0),
    dict(dim=8, trained_length=9, slow_turns=3.0, fast_turns=3.0)])
def test_frequencies_refused(kw):
    with pytest.raises(ValueError):
        rotary.rotary_frequencies(**kw)


# ------------------------------------------------------------------- refusals


def test_no_cpu_path():
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    at = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="only on the GPU"):
        attention.packed_attention(x, x, x, at, max_len=4)
    with pytest.raises(RuntimeError, match="only on the GPU"):
        attention.packed_attention_forward(x, x, x, at, max_len=4)
    with pytest.raises(RuntimeError, match="only on the GPU"):
        rotary.rotary_embedding(x, None, torch.arange(4), rotary.rotary_frequencies(64))
    h, t = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int64)
    for f in (loss.linear_cross_entropy, loss.linear_cross_entropy_forward):
        with pytest.raises(RuntimeError, match="only on the GPU"):
            f(h, h, t)
    with pytest.raises(RuntimeError, match="only on the GPU"):
        loss.linear_cross_entropy_backward(torch.ones(()), h, h, t, torch.zeros(4))


def rotary_call(**kw):
    a = dict(qt=64, qh=64, heads=1, kt=64, kh=64, kheads=0, dtype=1, tokens=2, dim=64, rot=64)
    a.update(kw)
    return status("tcfp_rotary", PTR, a["qt"], a["qh"], a["heads"], PTR, a["kt"], a["kh"], a["kheads"],
                  a["dtype"], a["tokens"], a["dim"], PTR, PTR, a["rot"], 0, 1.0, 0, PTR, PTR, None)


def test_rotary_refused():
    shape = status("tcfp_scale_bf16", PTR, 7, PTR, 0, PTR, None)
    assert shape != "ok"
    for kw in (dict(rot=0), dict(rot=3), dict(rot=66), dict(dim=1), dict(dim=70000), dict(tokens=-1),
               dict(heads=-1), dict(heads=65536), dict(kheads=70000), dict(dim=8192, rot=4098)):
        assert rotary_call(**kw) == shape, kw
    assert "dtype" in rotary_call(dtype=7).lower()
    assert rotary_call(tokens=0) == "ok" and rotary_call(heads=0) == "ok"


def packed_call(**kw):
    a = dict(q=PTR, token=128, head=64, batch=1, tokens=4, keys=4, heads=2, kv=1, dim=64, longest=4,
             scale=0.125, window=0)
    a.update(kw)
    return status("tcfp_packed_attention", a["q"], a["token"], a["head"], PTR, 64, 64, PTR, 64, 64, PTR,
                  PTR, a["batch"], a["tokens"], a["keys"], a["heads"], a["kv"], a["dim"], a["longest"],
                  a["scale"], 1, a["window"], PTR, None, None, None)


def test_packed_attention_refused():
    shape = status("tcfp_scale_bf16", PTR, 7, PTR, 0, PTR, None)
    for kw in (dict(dim=32), dict(dim=96), dict(heads=3, kv=2), dict(heads=0), dict(kv=0), dict(batch=0),
               dict(batch=70000), dict(tokens=-1), dict(keys=-1), dict(tokens=(1 << 29) + 1),
               dict(longest=-1), dict(window=-1), dict(scale=math.inf), dict(scale=math.nan),
               dict(token=-64), dict(token=1 << 24),
               dict(batch=65535, heads=65535)):
        assert packed_call(**kw) == shape, kw
    for kw in (dict(q=PTR + 2), dict(token=130), dict(head=65)):
        assert "align" in packed_call(**kw).lower(), kw
    assert packed_call(tokens=0) == "ok"


def loss_call(**kw):
    a = dict(h=PTR, ldh=64, ldw=64, tokens=4, vocab=10, dim=64, total=PTR, count=PTR, ws=PTR, nb=1 << 30)
    a.update(kw)
    return status("tcfp_linear_cross_entropy", a["h"], a["ldh"], PTR, a["ldw"], PTR, -100, a["tokens"],
                  a["vocab"], a["dim"], PTR, PTR, 1, a["total"], a["count"], a["ws"], a["nb"], None)


def test_cross_entropy_refused():
    shape = status("tcfp_scale_bf16", PTR, 7, PTR, 0, PTR, None)
    for kw in (dict(dim=60), dict(dim=0), dict(vocab=0), dict(tokens=-1), dict(ldh=56), dict(ldw=8),
               dict(ldh=1 << 23), dict(ldw=1 << 24), dict(total=None), dict(count=None)):
        assert loss_call(**kw) == shape, kw
    for kw in (dict(h=PTR + 8), dict(ldh=68), dict(ldw=100)):
        assert "align" in loss_call(**kw).lower(), kw
    for kw in (dict(ws=None), dict(nb=16), dict(ws=PTR + 8)):
        assert "workspace" in loss_call(**kw).lower(), kw


# ------------------------------------------------------------------ workspaces


def test_workspaces():
    lib = _hip.load_library()
    back, train = (lib.tcfp_linear_cross_entropy_backward_workspace_bytes,
                   lib.tcfp_linear_cross_entropy_train_workspace_bytes)
    for f in (back, train):
        assert f(0, 100, 64, 1, 1) == f(-1, 100, 64, 1, 1) == f(4, 0, 64, 1, 1) == 0
        # what is not wanted takes nothing
        assert f(1000, 50001, 1056, 0, 1) <= f(1000, 50001, 1056, 1, 1)
    # the logits' gradients of a run stay within 256 MiB (or are a run of 256 classes), of
    # a whole pass within 1 GiB
    for tokens in (1, 100, 8192, 100000, 400000):
        for vocab in (256, 50001, 1 << 20, 5 << 20):
            # (and 256 bytes, of which one float holds what all gradients are divided by)
            assert back(tokens, vocab, 64, 0, 0) <= max(256 << 20, 512 * tokens) + 256
            assert train(tokens, vocab, 64, 0, 0) <= (1 << 30) + (1 << 28)  # (parts, sums)
    packed = lib.tcfp_packed_attention_backward_workspace_bytes
    assert packed(100, 100, 0, 100, 4, 2, 64) == packed(100, 100, 1, 100, 4, 3, 64) == 0
    # delta; with many tiles of keys no parts beside it
    assert packed(1 << 20, 1 << 20, 64, 1 << 14, 8, 8, 128) == (1 << 20) * 8 * 4
    one = packed(4096, 4096, 1, 4096, 8, 1, 128)
    assert one > 4096 * 8 * 4 and (one - 4096 * 8 * 4) % (2 * 4096 * 128 * 4) == 0
    for bound in (1 << 30, 2**62):
        assert packed(4096, 4096, 1, bound, 8, 1, 128) == one


@pytest.mark.parametrize("kernel", ["product_kernel", "packed_forward_kernel"])
def test_copies_into_lds_keep_their_wait_states(kernel, tmp_path):
    text = next(t for t in _code_objects(tmp_path) if kernel in t)
    copies, short = short_waits(text)
    assert copies > 0
    assert not short, (len(short), copies, short[:3])
