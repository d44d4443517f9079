"""Trainable GDN-2 (mirrors the reference module gdn2_pipeline.py).

``gdn2_pallas_forward_trainable(q,k,v,w,b,g,scale,h0=None)`` returns
``(out, h_final)`` and is differentiable w.r.t. q, k, v, w, b, g and h0;
``scale`` is not (the reference's custom_vjp with nondiff_argnums=(6,),
gdn2_pipeline.py:59-61, 143-159).  In PyTorch the custom VJP is a
``torch.autograd.Function``; its backward returns the reference's cotangents
(dq, dk, dv, dw, db, dg, dh0) (gdn2_pipeline.py:137).

By default the forward keeps its per-chunk state in the workspace so the
backward skips the forward recompute; ``recompute=True`` instead saves only
the inputs, exactly like the reference (gdn2_pipeline.py:64-67).
"""
from __future__ import annotations

import contextlib
import threading

import torch

from . import gdn2_bwd as _bwd
from . import gdn2_fwd as _fwd
from .gdn2_checkpoint import Gdn2Checkpoint, gdn2_checkpoint_pack, gdn2_checkpoint_unpack

_FINAL_CLIP = 1e4  # gdn2_pipeline.py:34


def _gdn2_core_fwd(q, k, v, w, b, g, scale, h0, keep_residuals=True):
    """Forward rule: returns ((out, h_final), residuals) (gdn2_pipeline.py:64-67)."""
    if _fwd._head_dim(q) in _fwd._STAGE_D:   # stage kernels; the backward recomputes
        o, h_final = _fwd.gdn2_pallas_forward(q, k, v, w, b, g, scale, h0)
        return (o, h_final), (q, k, v, w, b, g, h0, None)
    p = _fwd._Prepared(q, k, v, w, b, g, scale, h0)
    o, h_final, ws = _fwd._run_forward(p, save_residuals=keep_residuals)
    residuals = (q, k, v, w, b, g, h0, ws if keep_residuals else None)
    return (o, h_final), residuals


def _gdn2_core_bwd(scale, residuals, cotangents):
    """Backward rule: returns (dq, dk, dv, dw, db, dg, dh0) (gdn2_pipeline.py:70-137)."""
    q, k, v, w, b, g, h0 = residuals[:7]
    ws = residuals[7] if len(residuals) > 7 else None
    do, dh_final = cotangents
    return _bwd.gdn2_backward(q, k, v, w, b, g, scale, h0, do, dh_final, workspace=ws)


class _Gdn2Core(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, w, b, g, h0, scale, recompute):
        (o, h_final), res = _gdn2_core_fwd(q, k, v, w, b, g, scale, h0,
                                           keep_residuals=not recompute)
        ctx.scale = scale
        ctx.ws = res[7]
        ctx.save_for_backward(q, k, v, w, b, g, h0)
        return o, h_final

    @staticmethod
    def backward(ctx, do, dh_final):
        q, k, v, w, b, g, h0 = ctx.saved_tensors
        if do is None:
            do = torch.zeros(q.shape, dtype=torch.float32, device=q.device)
        grads = _gdn2_core_bwd(ctx.scale, (q, k, v, w, b, g, h0, ctx.ws), (do, dh_final))
        ctx.ws = None
        dq, dk, dv, dw, db, dg, dh0 = grads
        return dq, dk, dv, dw, db, dg, dh0, None, None


# What a call of gdn2_fwd / gdn2_bwd reads from the module.
_SETTINGS = ("BT", "BC", "CLIP", "EXACT_BT", "PAIR64", "MASKED_TAIL", "GATES")
_settings_lock = threading.Lock()   # backward passes of several devices have a thread each


def _settings():
    return {n: getattr(_fwd, n) for n in _SETTINGS}


@contextlib.contextmanager
def _with_settings(saved):
    """gdn2_fwd's settings as ``saved``, for one call."""
    with _settings_lock:
        now = _settings()
        vars(_fwd).update(saved)
        try:
            yield
        finally:
            vars(_fwd).update(now)


class _Gdn2CoreInt8(torch.autograd.Function):
    """_Gdn2Core that keeps q, k, v, w, b in 8 bits and recomputes the forward
    from the restored values in the backward, under the forward's settings: the
    kept w, b and g are what GATES said they are then."""

    @staticmethod
    def forward(ctx, q, k, v, w, b, g, h0, scale):
        ctx.settings = _settings()
        o, h_final = _fwd.gdn2_pallas_forward(q, k, v, w, b, g, scale, h0)
        kept = gdn2_checkpoint_pack(q, k, v, w, b)
        ctx.scale, ctx.shapes, ctx.dtypes, ctx.on_host = scale, kept.shapes, kept.dtypes, kept.on_host
        ctx.at = [at for at, _, _ in kept.buffers]
        ctx.save_for_backward(g, h0, *(t for _, *pair in kept.buffers for t in pair))
        return o, h_final

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do, dh_final):
        g, h0, *kept = ctx.saved_tensors
        if do is None:
            do = torch.zeros(g.shape, dtype=torch.float32, device=g.device)
        q, k, v, w, b = gdn2_checkpoint_unpack(
            Gdn2Checkpoint(list(zip(ctx.at, kept[::2], kept[1::2])), ctx.shapes, ctx.dtypes,
                           ctx.on_host))
        with _with_settings(ctx.settings):
            grads = _bwd.gdn2_backward(q, k, v, w, b, g, ctx.scale, h0, do, dh_final)
        return *grads, None


def gdn2_pallas_forward_trainable(q, k, v, w, b, g, scale, h0=None, recompute=False,
                                  checkpoint=None):
    """Trainable Gated DeltaNet-2 forward with the fused backward.

    Args: q, k, v, w, b, g (batch, seq_len, heads, d_head) CUDA tensors;
    scale a Python float; h0 (batch, heads, d_head, d_head), zero if None.
    Returns out (batch, seq_len, heads, d_head) and h_final
    (batch, heads, d_head, d_head), both float32.

    checkpoint="int8" keeps q, k, v, w, b in 8 bits (gdn2_checkpoint_pack) and
    g, h0 as they are, and recomputes the forward: the gradients are those at
    the restored inputs, the outputs those of the inputs.  ``recompute`` makes no
    difference then.  The backward runs under the settings of gdn2_fwd (BT, CLIP,
    GATES and the others) that its forward had.
    """
    if checkpoint not in (None, "int8"):
        raise _fwd.Gdn2ShapeError(f"checkpoint={checkpoint!r}: None or 'int8'")
    B, T, H, D = q.shape
    if h0 is None:
        h0 = torch.zeros((B, H, D, D), dtype=torch.float32, device=q.device)
    if checkpoint == "int8":
        return _Gdn2CoreInt8.apply(q, k, v, w, b, g, h0, float(scale))
    return _Gdn2Core.apply(q, k, v, w, b, g, h0, float(scale), bool(recompute))
