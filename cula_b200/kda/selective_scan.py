"""The selective state space recurrence: ``selective_scan`` over whole sequences, with gradients, and ``selective_scan_update`` for one
token of each sequence against a pool of states. Hand-written sm_100a kernels (csrc/kda_selective_scan_fwd.cu, _bwd.cu,
kda_selective_step.cu); checks, autograd and launches in the host extension (csrc/host/host_ssm.cpp). No Triton, no fallback."""
from __future__ import annotations

import torch

from .. import _native
from ..utils import get_varlen_tables


@torch.compiler.disable
def selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=False, initial_state=None, output_final_state=False,
                   cu_seqlens=None, cu_seqlens_cpu=None):
    """Per channel ``d`` and state ``n``, with ``step = softplus(dt + dt_bias)`` (or ``dt + dt_bias``)::

        h_t = exp(step_t * A[d, n]) * h_{t-1} + step_t * x_t * B_t[n]
        y_t = (sum_n C_t[n] * h_t[n] + D * x_t) * silu(z_t)

    x, dt, z: ``[B, T, D]`` bf16 or fp32 (``B == 1`` with ``cu_seqlens``); A: ``[D, S]``, ``S <= 64``; B, C: ``[B, T, S]``, or
    ``[B, T, G, S]`` for groups of ``D / G`` channels (a multiple of 8); D, dt_bias: ``[D]`` or None; z None: no gate. Activations
    have one type; views of a projection's output are read in place. initial_state: ``[N, D, S]`` fp32 or None for zeros, one per
    sequence; with ``output_final_state`` the states after the last tokens are returned, of a sequence without tokens the one before.
    Rows of a packed batch past its last token have zero outputs and gradients. States and sums are fp32; errors of states and of
    parameters' gradients relative to 64 bits are about 1e-6 (those of a plain fp32 program 0.5e-6 to 2e-6).

    Returns ``(y, final_state)``, y in the type of x. Gradients flow from both to every tensor argument, are the same from run to
    run and cannot be differentiated again. A forward call that gradients will be asked of keeps, in fp32, the states before every
    eighth token (``4 * S / 8`` bytes per token and channel, S rounded up to 8, 16, 32 or 64, for 64 tokens at a time: short sequences
    pay for 64) and with a gate y before it (4 bytes); the backward pass takes shares of dB and dC for every 128, 64, 32 or 16
    channels (``8 * S`` bytes per token and group each) while it runs."""
    tab = None if cu_seqlens is None else get_varlen_tables(cu_seqlens, cu_seqlens_cpu).native
    return _native.host().selective_scan(x, dt, A, B, C, D, z, dt_bias, dt_softplus, initial_state, output_final_state, tab)


def selective_scan_update(x, dt, A, B, C, state, state_indices=None, D=None, z=None, dt_bias=None, dt_softplus=False, out=None):
    """One token of ``selective_scan`` for each of ``N`` sequences, as a decode step.

    x, dt, z: ``[N, D]`` (or ``[N, 1, D]``); B, C: ``[N, S]`` or ``[N, G, S]`` (with x's token axis, if it has one); state:
    ``[pool, D, S]`` fp32, contiguous, updated in place. state_indices: ``[N]`` int32 slots, negative = skip the sequence (zero output,
    no access to the pool), or None for slot = sequence; a slot may be named once in a call. A slot past the pool is skipped too and
    reported by ``check_status``. Returns ``y`` shaped like x (``out`` if given). No gradients, and tangents are refused; autograd knows
    that state and out were written to."""
    return _native.host().selective_scan_update(x, dt, A, B, C, state, state_indices, D, z, dt_bias, dt_softplus, out)
