"""The layer operators around ``chunk_kda`` in a Kimi-Linear block (fla/layers/kda.py:147-165, 191, 306) and around ``selective_scan``
in a state space block:

* ``short_conv`` -- the short causal depthwise convolution (+ SiLU) applied to the q / k / v projections; call surface of
  flash-linear-attention's ``causal_conv1d`` (fla/modules/convolution.py) for the arguments a KDA layer uses;
* ``rms_norm_gated`` -- the gated RMS norm applied to the attention output, ``rmsnorm(x) * weight * act(g)``; call
  surface of ``rms_norm_gated`` (fla/modules/fused_norm_gate.py:846-869) without residual / bias;
* ``short_conv_update`` -- one token of the convolution for each sequence of a batch, against a pool of windows;
* ``add_rms_norm`` -- the residual's addition and the RMS norm before a block; ``add_rms_norm_fp8`` the same with an 8-bit
  output and its scales.

``short_conv``, ``rms_norm_gated`` and ``add_rms_norm`` are differentiable (streaming sm_100a kernels, autograd and launches in
the host extension, csrc/host/host_layer_ops.cpp and host_ssm.cpp). No Triton, no fallback."""
from __future__ import annotations

import torch

from .. import _native
from ..utils import get_varlen_tables


@torch.compiler.disable
def short_conv(x, weight, bias=None, initial_state=None, output_final_state=False, activation="silu", cu_seqlens=None,
               cu_seqlens_cpu=None):
    """Causal depthwise convolution over time, then SiLU (``activation`` ``"silu"``/``"swish"``) or nothing (``None``).

    x: ``[B, T, D]`` bf16 (``B == 1`` with ``cu_seqlens``); weight: ``[D, W]``, ``W <= 4`` (a ``[D, 1, W]`` conv1d weight
    is accepted), tap ``W - 1`` multiplies the current token; bias: ``[D]`` or None; initial_state: ``[N, D, W]`` -- the
    last ``W`` inputs of a previous call, newest last -- or None; with ``output_final_state`` the same record for this
    call is returned. Returns ``(y, final_state)``. Gradients flow to x, weight and bias."""
    assert activation in (None, "silu", "swish"), "activation must be None, 'silu' or 'swish'."
    tab = None if cu_seqlens is None else get_varlen_tables(cu_seqlens, cu_seqlens_cpu).native
    return _native.host().short_conv(x, weight, bias, initial_state, output_final_state, activation is not None, tab)


@torch.compiler.disable
def rms_norm_gated(x, g, weight, activation="sigmoid", eps=1e-6):
    """``x * rsqrt(mean(x^2, -1) + eps) * weight * act(g)`` with ``act`` = ``"sigmoid"`` (what the KDA layer uses) or
    ``"swish"``/``"silu"`` (``g * sigmoid(g)``). x, g: ``[..., D]`` bf16, D in {128, 256, 512, 1024}; weight ``[D]``.
    Gradients flow to x, g and weight."""
    assert activation in ("sigmoid", "swish", "silu"), "activation must be 'sigmoid', 'swish' or 'silu'."
    return _native.host().rms_norm_gated(x, g, weight, activation != "sigmoid", eps)


def short_conv_update(x, weight, cache, cache_indices=None, bias=None, activation="silu", out=None):
    """One token of ``short_conv`` for each of ``N`` sequences, as a decode step.

    x: ``[N, D]`` or ``[N, 1, D]`` bf16, D a multiple of 8; weight: ``[D, W]`` (or ``[D, 1, W]``), ``W <= 4``; cache:
    ``[pool, D, W]`` fp32, contiguous: the last ``W`` inputs of each slot, newest last (what ``short_conv`` returns as its final
    state); each used window takes in its token, in place. cache_indices: ``[N]`` int32 slots, negative = skip the sequence (zero
    output, no access to the pool), or None for slot = sequence; a slot may be named once in a call. A slot past the pool is skipped
    too and reported by ``check_status``. Returns ``y`` shaped like x (``out`` if given). No gradients, and tangents are refused;
    autograd knows that cache and out were written to."""
    assert activation in (None, "silu", "swish"), "activation must be None, 'silu' or 'swish'."
    return _native.host().short_conv_update(x, weight, cache, cache_indices, bias, activation is not None, out)


@torch.compiler.disable
def add_rms_norm(x, weight, residual=None, eps=1e-6):
    """``v = x + residual`` and ``y = v * rsqrt(mean(v^2, -1) + eps) * weight``; returns ``(y, v)``.

    x: ``[..., D]`` bf16 or fp32, D a multiple of 8 up to 16384; weight: ``[D]``; residual: the stream that the block adds to, of the
    shape of x, in fp32 or in the type of x, or None (then ``v`` is x itself). ``v`` has the residual's type, to which the sum is
    rounded once before it is normalised; ``y`` has the type of x. Gradients flow to x, residual and weight from both results, the
    same from run to run; they cannot be differentiated again."""
    y, v = _native.host().add_rms_norm(x, weight, residual, eps)
    return y, x if v is None else v


def add_rms_norm_fp8(x, weight, residual=None, eps=1e-6, group_size=None):
    """``add_rms_norm`` with ``y`` in 8 bits for a projection in e4m3; returns ``(q, scale, v)`` with ``q * scale = y`` up to the
    rounding of q.

    ``scale`` is fp32, ``max(amax / 448, 2^-126)`` over each row (``group_size`` None: ``[...]``) or over each ``group_size``
    (32, 64, 128 or 256) neighbouring columns (``[..., D / group_size]``); ``q`` is ``torch.float8_e4m3fn``. A row that holds a
    NaN is NaN in all of q and scale; one that holds an infinity is NaN where its scale covers the infinity, and zero in other groups (all else
    is divided by an infinite norm). Other arguments as for ``add_rms_norm``. No gradients, and tangents are refused."""
    q, scale, v = _native.host().add_rms_norm_fp8(x, weight, residual, eps, 0 if group_size is None else group_size)
    return q, scale, x if v is None else v
