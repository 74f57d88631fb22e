"""Verification of drafted tokens on the MI355X: which of them the target model
keeps, and its next token, from given random numbers.

It follows the model's pass over a run or a tree of drafted tokens
(``femtochat_amd.cache``).  Node 0 is the last token of the text, the nodes after it are
drafted; ``logits`` (B, N, V) holds at node i the model's logits behind it, p their
softmax at ``temperature``::

    draws       node i was drawn from q, the softmax of draft_logits (B, N - 1, V) at i - 1:
                accepted if u[i] q(x) < p(x); the first refusal ends the run, and the
                next token is drawn from max(p - q, 0), or where that leaves nothing
                (less than 2^-40) from p
    candidates  no draft_logits: a node's children (a run's next node) are tried in
                order: accepted if u[i] (1 - what those before it have of p) < p(x); the
                next token is drawn from p without those tried

Either way the text is distributed as the model's own samples are.  A token outside the
vocabulary counts as no node: the run ends before it.  The next token of
a draw is the first whose cumulative weight is above u[0] of the whole.  At temperature 0
the largest logit (the first of several) is accepted and drawn.  The reference has no
counterpart.
"""
from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import Optional, Tuple

import torch

from . import _lib
from .kernels import _call, _check_tensor, _check_workspace, _dtype_code, _ptr
from .loss import _INDEX

__all__ = ["verify_drafts", "verify_drafts_", "verify_drafts_workspace_bytes"]

_LOGITS = (torch.float32, torch.bfloat16)
_I32 = (torch.int32,)


@lru_cache(maxsize=256)
def _plan(B, N, V, dtype, index, tree, draft, temperature):
    """(descriptor, its workspace bytes) of a call."""
    d = _lib.VerifyDesc(B, N, V, dtype, index, tree, draft, temperature)
    n = ctypes.c_size_t(0)
    _lib.check(_lib.lib().fc_verify_workspace_bytes(ctypes.byref(d), ctypes.byref(n)))
    return d, n.value


def _checked(logits, tokens, uniforms, draft_logits, parents, counts, temperature):
    if not isinstance(logits, torch.Tensor) or logits.dim() != 3:
        raise ValueError("logits must be a (B, N, V) tensor")
    device = logits.device
    if device.type != "cuda":
        raise ValueError("the MI355X verification needs tensors on a HIP device (torch 'cuda'); there is no CPU path")
    B, N, V = logits.shape
    _check_tensor("logits", logits, (B, N, V), _LOGITS, device)
    _check_tensor("tokens", tokens, (B, N), tuple(_INDEX), device)
    if uniforms is not None or temperature != 0:
        _check_tensor("uniforms", uniforms, (B, N), (torch.float32,), device)
    if draft_logits is not None:
        if parents is not None:
            raise ValueError("draft_logits go with a run of drafted tokens; a tree's nodes are candidates")
        _check_tensor("draft_logits", draft_logits, (B, N - 1, V), (logits.dtype,), device)
    tree = 0
    if parents is not None:
        tree = 2 if isinstance(parents, torch.Tensor) and parents.dim() == 2 else 1
        _check_tensor("parents", parents, (B, N) if tree == 2 else (N,), _I32, device)
    if counts is not None:
        _check_tensor("counts", counts, (B,), _I32, device)
    d, nbytes = _plan(B, N, V, _dtype_code(logits.dtype), _INDEX[tokens.dtype], tree, int(draft_logits is not None), float(temperature))
    return device, d, nbytes


def verify_drafts_workspace_bytes(logits, tokens, uniforms, *, draft_logits=None, parents=None, counts=None,
                                  temperature: float = 1.0) -> int:
    """Bytes of the caller-owned workspace that a call with these arguments accepts (0 when it needs none)."""
    n = _checked(logits, tokens, uniforms, draft_logits, parents, counts, temperature)[2]
    return n + 256 if n > 0 else 0


def verify_drafts_(path: torch.Tensor, kept: torch.Tensor, token: torch.Tensor, logits: torch.Tensor, tokens: torch.Tensor,
                   uniforms: Optional[torch.Tensor], *, draft_logits: Optional[torch.Tensor] = None,
                   parents: Optional[torch.Tensor] = None, counts: Optional[torch.Tensor] = None,
                   temperature: float = 1.0, workspace: Optional[torch.Tensor] = None) -> None:
    """``verify_drafts`` into the caller's path (B, N), kept (B,) and token (B,), int32."""
    checked = _checked(logits, tokens, uniforms, draft_logits, parents, counts, temperature)
    B, N = tokens.shape
    _check_tensor("path", path, (B, N), _I32, checked[0])
    _check_tensor("kept", kept, (B,), _I32, checked[0])
    _check_tensor("token", token, (B,), _I32, checked[0])
    _verify(checked, path, kept, token, logits, tokens, uniforms, draft_logits, parents, counts, workspace)


def _verify(checked, path, kept, token, logits, tokens, uniforms, draft_logits, parents, counts, workspace) -> None:
    device, d, nbytes = checked
    at = None
    if nbytes > 0:
        if workspace is None:  # freed to this stream's pool on return, so later work on the stream comes after the kernels
            workspace = torch.empty(nbytes + 256, dtype=torch.uint8, device=device)
        else:
            _check_workspace(workspace, nbytes + 256, device)
        at = (workspace.data_ptr() + 255) & ~255
    _call(device, _lib.lib().fc_verify_drafts, ctypes.byref(d), logits.data_ptr(), _ptr(draft_logits), tokens.data_ptr(),
          _ptr(uniforms), _ptr(parents), _ptr(counts), path.data_ptr(), kept.data_ptr(), token.data_ptr(),
          at, nbytes)


def verify_drafts(logits: torch.Tensor, tokens: torch.Tensor, uniforms: Optional[torch.Tensor], *,
                  draft_logits: Optional[torch.Tensor] = None, parents: Optional[torch.Tensor] = None,
                  counts: Optional[torch.Tensor] = None, temperature: float = 1.0,
                  workspace: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(path, kept, token): the accepted nodes (B, N) from node 0 on, with -1 behind them, their
    number (B,), and the next token (B,), all int32 (module documentation).

    logits and draft_logits are float32 or bfloat16, ``tokens`` (B, N) int32 or int64 the nodes'
    tokens (node 0's is not read), ``uniforms`` (B, N) float32 in [0, 1) a random number per node,
    node 0's for the next token (None at temperature 0).  ``parents``, (N,) or (B, N) int32, and
    ``counts`` (B,) are those of ``cached_attention``; without parents the nodes are a run.
    A row with a NaN or +infinity, or without a finite logit, accepts nothing and has the next
    token -1; a sequence of no nodes (counts 0) keeps none."""
    if not isinstance(tokens, torch.Tensor) or tokens.dim() != 2:
        raise ValueError("tokens must be a (B, N) tensor")
    checked = _checked(logits, tokens, uniforms, draft_logits, parents, counts, temperature)
    device = checked[0]
    path = torch.empty_like(tokens, dtype=torch.int32)
    kept, token = torch.empty(2, tokens.shape[0], dtype=torch.int32, device=device).unbind(0)
    _verify(checked, path, kept, token, logits, tokens, uniforms, draft_logits, parents, counts, workspace)
    return path, kept, token
