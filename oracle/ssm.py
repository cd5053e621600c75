"""CPU oracle for the operators of a selective state space block -- TEST INFRASTRUCTURE, NOT PRODUCT CODE (only tests/ import it).
The definitions, token by token, in the type of the inputs (the tests pass 64 bits); differentiable by autograd."""
import torch
import torch.nn.functional as F


def _per_channel(m, D):
    """[..., G, S] to [..., D, S]"""
    return m.repeat_interleave(D // m.shape[-2], -2)


def selective_scan_ref(x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=False, initial_state=None, cu_seqlens=None):
    """Returns (y [B, T, D], final states [N, D, S])."""
    n, T, ch = x.shape
    B, C = (m.unsqueeze(2) if m.dim() == 3 else m for m in (B, C))
    step = dt if dt_bias is None else dt + dt_bias
    if dt_softplus:
        step = F.softplus(step, threshold=1e9)
    bounds = [(b, 0, T) for b in range(n)] if cu_seqlens is None else \
        [(0, int(cu_seqlens[i]), int(cu_seqlens[i + 1])) for i in range(len(cu_seqlens) - 1)]
    rows = [[None] * T for _ in range(n)]
    finals = []
    for i, (b, first, last) in enumerate(bounds):
        h = x.new_zeros(ch, A.shape[1]) if initial_state is None else initial_state[i]
        for t in range(first, last):
            h = torch.exp(step[b, t, :, None] * A) * h + (step[b, t] * x[b, t])[:, None] * _per_channel(B[b, t], ch)
            y = (h * _per_channel(C[b, t], ch)).sum(-1)
            if D is not None:
                y = y + D * x[b, t]
            rows[b][t] = y if z is None else y * F.silu(z[b, t])
        finals.append(h)
    zero = x.new_zeros(ch)                                                     # rows past the packed tokens
    y = torch.stack([torch.stack([zero if r is None else r for r in row]) if row else x.new_zeros(0, ch) for row in rows]) if n else x.new_zeros(0, T, ch)
    return y, torch.stack(finals) if finals else x.new_zeros(0, ch, A.shape[1])


def selective_scan_update_ref(x, dt, A, B, C, state, state_indices=None, D=None, z=None, dt_bias=None, dt_softplus=False):
    """Returns (y [N, D], the pool after the step)."""
    pool, y = state.clone(), torch.zeros_like(x)
    for n in range(x.shape[0]):
        slot = n if state_indices is None else int(state_indices[n])
        if 0 <= slot < pool.shape[0]:
            part = lambda m: None if m is None else m[n][None, None]  # noqa: E731, B023
            o, h = selective_scan_ref(part(x), part(dt), A, part(B), part(C), D, part(z), dt_bias, dt_softplus, pool[slot][None])
            y[n], pool[slot] = o[0, 0], h[0]
    return y, pool


def short_conv_update_ref(x, weight, cache, cache_indices=None, bias=None, activation="silu"):
    """Returns (y [N, D], the pool after the step)."""
    pool, y = cache.clone(), torch.zeros_like(x)
    for n in range(x.shape[0]):
        slot = n if cache_indices is None else int(cache_indices[n])
        if 0 <= slot < pool.shape[0]:
            pool[slot] = torch.cat([pool[slot][:, 1:], x[n][:, None]], 1)
            pre = (pool[slot] * weight).sum(-1) + (0 if bias is None else bias)
            y[n] = F.silu(pre) if activation else pre
    return y, pool


def add_rms_norm_ref(x, weight, residual=None, eps=1e-6, stream=None):
    """Returns (y, v). ``stream``: the type that the sum is rounded to (its derivative is taken as one), or None for no rounding."""
    v = x if residual is None else x + residual
    if stream is not None and residual is not None:
        v = v + (v.detach().to(torch.float32).to(stream).to(v.dtype) - v.detach())
    return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + eps) * weight, v


def quantize_e4m3_ref(y, group_size=None):
    """Returns (q as numbers, scale) with one scale per row, or per group of neighbouring columns."""
    size = group_size or y.shape[-1]
    g = y.reshape(*y.shape[:-1], -1, size)
    scale = (g.abs().amax(-1) / 448.0).clamp(min=2.0 ** -126)
    q = (g / scale[..., None]).to(torch.float32).clamp(-448, 448).to(torch.float8_e4m3fn).to(y.dtype).reshape(y.shape)
    return q, scale if group_size else scale[..., 0]
