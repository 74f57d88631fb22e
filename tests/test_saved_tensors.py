"""What saved-tensor hooks hand to the backwards (CPU, no kernel is launched): other
strides are made contiguous, other sizes, types and devices refused before a pointer
reaches the library."""
import ctypes

import pytest
import torch

import femtochat_amd as F
from femtochat_amd import _lib, answer_loss, kernels

B, T, H, HKV, D, V = 2, 5, 4, 2, 16, 7


class Ctx:
    """The context of a node: what its forward set, and the tensors it saved as
    `swap` returns them."""
    def __init__(self, wanted=1):
        self.needs_input_grad = (True,) * wanted + (False,) * (9 - wanted)

    def save_for_backward(self, *tensors):
        self.saved = tensors

    def mark_non_differentiable(self, *_):
        pass

    @property
    def saved_tensors(self):
        return tuple(self.swap(i, t) for i, t in enumerate(self.saved))


@pytest.fixture
def calls(monkeypatch):
    """The library's calls, recorded as (entry, arguments), and CPU tensors let through."""
    seen = []
    monkeypatch.setattr(kernels, "_call", lambda device, entry, *args: seen.append((entry.__name__, args)))
    monkeypatch.setattr(answer_loss, "_call", lambda device, entry, *args: seen.append((entry.__name__, args)))
    monkeypatch.setattr(kernels, "_check_common", lambda A, Q, *_: (Q.device,) + tuple(Q.shape))
    monkeypatch.setattr(answer_loss, "_desc", lambda *a, **k: _lib.AnswerDesc(V, 2, T, 0, -1, 1, 0, 0, 0))
    return seen


def _attention(swap):
    ctx = Ctx(3)
    Q, K, W = (torch.randn(B, T, h, D).bfloat16() for h in (H, HKV, HKV))
    pos = torch.arange(T, dtype=torch.int32).repeat(B, 1)
    F.AttentionFunction.forward(ctx, Q, K, W, (-1, 0), None, pos, 5.0, torch.ones(H), torch.full((B, T), 2, dtype=torch.int32))
    ctx.swap = swap
    return ctx, lambda: F.AttentionFunction.backward(ctx, torch.zeros(B, T, H, D, dtype=torch.bfloat16))


def _policy(swap):
    ctx = Ctx()
    o = torch.zeros(2, T)
    F.PolicyLossFunction.forward(ctx, torch.randn(2, T, V), torch.zeros(2, T, dtype=torch.int64), o, o, None, (0.2, 0.2), 0.0, -1, "none")
    ctx.swap = swap
    return ctx, lambda: F.PolicyLossFunction.backward(ctx, torch.ones(2, T))


def _preference(swap):
    ctx = Ctx()
    F.PreferenceLossFunction.forward(ctx, torch.randn(2, T, V), torch.zeros(2, T, dtype=torch.int64), torch.zeros(2), 0.1, 0.0, -1, "none")
    ctx.swap = swap
    return ctx, lambda: F.PreferenceLossFunction.backward(ctx, torch.ones(1), None)


NODES = {"attention": _attention, "policy": _policy, "preference": _preference}


def _values(at, like):
    """The memory at an address, read as the kernels read a tensor like `like`."""
    n = like.numel() * like.element_size()
    raw = torch.frombuffer(bytearray((ctypes.c_char * n).from_address(at)), dtype=like.dtype)
    return raw.view(like.shape)


@pytest.mark.parametrize("node", NODES)
def test_other_strides(calls, node, monkeypatch):
    """Every saved tensor comes back transposed in memory; the call gets contiguous values."""
    read = []
    first = 3 if node == "attention" else 2  # of the call's arguments that are saved tensors (Q K V O l m positions; logits, tokens)
    count = 7 if node == "attention" else 2

    def call(device, entry, *args):
        if entry.__name__.endswith("bwd"):
            read.extend(_values(args[first + i], ctx.saved[i]).equal(ctx.saved[i]) for i in range(count))

    ctx, backward = NODES[node](lambda i, t: t if t.dim() < 2 else t.transpose(1, -1).contiguous().transpose(1, -1))
    for t in ctx.saved:  # what the stubbed forward left unwritten
        if t.dtype.is_floating_point:
            t.copy_(torch.arange(t.numel()).view(t.shape) % 113)
    monkeypatch.setattr(kernels, "_call", call)
    monkeypatch.setattr(answer_loss, "_call", call)
    backward()
    assert len(read) == count and all(read)


@pytest.mark.parametrize("node", NODES)
@pytest.mark.parametrize("what", ["device", "size", "dtype"])
def test_other_tensors(calls, node, what):
    """Each saved tensor in turn comes back on another device, shorter, or in another type."""
    def spoil(t):
        if what == "device":
            return t.to("meta")
        if what == "size":
            return t[:-1]
        return t.to(torch.float64)

    ctx, _ = NODES[node](None)
    for which, t in enumerate(ctx.saved):
        if t is None:
            continue
        ctx, backward = NODES[node](lambda i, x: spoil(x) if i == which else x)
        del calls[:]
        with pytest.raises((ValueError, TypeError), match="saved"):
            backward()
        assert not calls, (node, which)
