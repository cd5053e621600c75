"""The operators of a selective state space block, as timed cases, and their plain forms.

  scan        ``selective_scan``: the recurrence h_t = exp(dt_t A) h_{t-1} + dt_t x_t B_t, y_t = C_t h_t + D x_t over whole
              prompts, gated by silu(z); without gradients, or with every gradient (``train``)
  scan_step   ``selective_scan_update``: one token of each of ``rows`` sequences against a pool of states
  conv_step   ``short_conv_update``: one token of each of ``rows`` sequences against a pool of convolution windows
  norm        ``add_rms_norm``: the residual's addition and the RMS norm before the block, without gradients or with (``train``)
  norm8       ``add_rms_norm_fp8``: the same with an 8-bit output and its scales, per row (``group`` 0) or per group of columns

A case is a dict of plain values. ``dtype`` is the type of the activations (``"bf16"`` or ``"fp32"``), ``res`` that of the
residual stream (``"none"``: there is none). ``run`` computes the plain form where ``own`` is false, and calls the framework
where it is true.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
E4M3_MAX = 448.0
SCALE_MIN = 2.0 ** -126
EPS = 1e-5
MOST_SCAN = 4 * 2048 * 4096 * 16        # tokens x channels x states of the largest scan
MOST_NORM = 16384 * 4096                # elements of the largest norm
MOST_STEP = 256 * 4096 * 16             # sequences x channels x states of the largest step


def listed():
    return [
        # the next turn of a chat: a handful of tokens continued from a state; latency
        dict(name="scan_turn", kind="scan", B=1, T=37, N=0, D=2048, S=16, G=1, dtype="bf16", gate=True, states=True, train=False),
        # three long documents packed into one call: few chains, each thousands of tokens long
        dict(name="scan_long", kind="scan", B=1, T=16384, N=3, D=2048, S=16, G=1, dtype="bf16", gate=True, states=True, train=False),
        # fine-tuning of a small layer in 32 bits: odd lengths, an odd number of states, two groups of B and C, every gradient
        dict(name="scan_train_small", kind="scan", B=2, T=333, N=0, D=528, S=12, G=2, dtype="fp32", gate=True, states=True, train=True),
        # pre-training: the largest step
        dict(name="scan_train", kind="scan", B=4, T=2048, N=0, D=4096, S=16, G=1, dtype="bf16", gate=True, states=False, train=True),
        # interactive generation: one sequence, one token
        dict(name="scan_step_one", kind="scan_step", rows=1, D=4096, S=16, G=1, dtype="bf16", gate=True, indexed=False),
        # a serving step at a full batch, its states anywhere in the pool
        dict(name="scan_step_full", kind="scan_step", rows=256, D=4096, S=16, G=1, dtype="bf16", gate=True, indexed=True),
        # the convolution before those two: an odd number of live sequences, one of them padding, and the full batch
        dict(name="conv_step_odd", kind="conv_step", rows=33, D=4096, W=4, bias=True, act=True, indexed=True),
        dict(name="conv_step_full", kind="conv_step", rows=256, D=12288, W=4, bias=True, act=True, indexed=True),
        # the norm of a small model in training, its residual stream in 32 bits, and that of the largest step
        dict(name="norm_train_small", kind="norm", rows=333, D=520, dtype="bf16", res="fp32", train=True),
        dict(name="norm_train", kind="norm", rows=8192, D=4096, dtype="bf16", res="bf16", train=True),
        # the norm before an 8-bit projection: a serving step with one scale per 128 columns, a long prompt with one per row
        dict(name="norm8_step", kind="norm8", rows=33, D=4096, dtype="bf16", res="bf16", group=128),
        dict(name="norm8_prompt", kind="norm8", rows=16384, D=4096, dtype="bf16", res="fp32", group=0),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["scan", "scan", "scan", "scan_step", "conv_step", "norm", "norm8"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if kind in ("norm", "norm8"):
        unit = rng.choice([8, 128])
        D = unit * _spread(rng, 64 // unit or 1, 8192 // unit)
        rows = _spread(rng, 1, min(16384, MOST_NORM // D))
        if kind == "norm8":
            return dict(kind=kind, rows=rows, D=D, dtype=dtype, res=rng.choice(["bf16", "fp32", "none"]) if dtype == "bf16" else "fp32",
                        group=rng.choice([0, 128]) if D % 128 == 0 else 0)
        return dict(kind=kind, rows=rows, D=D, dtype=dtype, res=rng.choice(["bf16", "fp32", "none"]) if dtype == "bf16" else "fp32",
                    train=rng.random() < 0.6)
    if kind == "conv_step":
        return dict(kind=kind, rows=_spread(rng, 1, 256), D=8 * _spread(rng, 8, 1536), W=rng.choice([4, 4, 3, 2]),
                    bias=rng.random() < 0.5, act=rng.random() < 0.8, indexed=rng.random() < 0.7)
    S = rng.choice([16, 16, 16, 8, 32, _spread(rng, 1, 64)])
    G = rng.choice([1, 1, 1, 2, 4])
    D = 8 * G * _spread(rng, 8, 512 // G)
    if kind == "scan_step":
        return dict(kind=kind, rows=_spread(rng, 1, min(256, MOST_STEP // (D * S))), D=D, S=S, G=G, dtype=dtype,
                    gate=rng.random() < 0.7, indexed=rng.random() < 0.7)
    N = _spread(rng, 2, 64) if rng.random() < 0.35 else 0
    most = MOST_SCAN // (D * max(8, S))
    if N:
        B, T = 1, _spread(rng, 4 * N, min(16384, most))
    else:
        B = _spread(rng, 1, 8)
        T = _spread(rng, 1, min(8192, most // B))
    return dict(kind=kind, B=B, T=T, N=N, D=D, S=S, G=G, dtype=dtype, gate=rng.random() < 0.7, states=rng.random() < 0.6,
                train=rng.random() < 0.5)


def _lengths(total, n, gen):
    """The bounds of n uneven lengths (each at least 1) that add up to total."""
    w = (0.8 * torch.randn(n, generator=gen, device=gen.device)).exp().double().cpu()
    cuts = (torch.cumsum(w, 0) / w.sum() * (total - n)).floor().long() + torch.arange(1, n + 1)
    cuts[-1] = total
    return torch.cat([torch.zeros(1, dtype=torch.int64), cuts]).to(torch.int32)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))

    def rn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32).to(dtype)

    def uni(lo, hi, *shape):
        return lo + (hi - lo) * torch.rand(*shape, generator=gen, device=dev)

    s, kind, D = dict(case), case["kind"], case["D"]
    if kind in ("norm", "norm8"):
        dt, R = DTYPES[case["dtype"]], case["rows"]
        s.update(x=rn(R, D, dtype=dt), w=1.0 + 0.1 * rn(D), r=None if case["res"] == "none" else (4.0 * rn(R, D)).to(DTYPES[case["res"]]))
        if case.get("train"):
            s.update(dy=rn(R, D, dtype=dt), dr=None if s["r"] is None else rn(R, D, dtype=s["r"].dtype))
            for t in (s["x"], s["w"], s["r"]):
                if t is not None:
                    t.requires_grad_(True)
        return s

    def slots(rows):
        if not case["indexed"]:
            return rows, None
        pool = rows + rows // 4 + 1
        idx = torch.randperm(pool, generator=gen, device=dev)[:rows].to(torch.int32)
        if rows >= 8:
            idx[rows // 3] = -1                                     # a padded place in the batch
        return pool, idx

    if kind == "conv_step":
        pool, s["idx"] = slots(case["rows"])
        s.update(x=rn(case["rows"], D, dtype=torch.bfloat16), w=0.3 * rn(D, case["W"]), b=0.1 * rn(D) if case["bias"] else None,
                 pool=rn(pool, D, case["W"]).to(torch.bfloat16).float())
        return s
    S, G, dt = case["S"], case["G"], DTYPES[case["dtype"]]
    # rates and steps as a trained layer has them: channels that forget within a token to ones that remember thousands
    A = -torch.arange(1, S + 1, device=dev, dtype=torch.float32) * (0.1 * rn(D, S)).exp()
    step = uni(math.log(1e-3), math.log(1e-1), D).exp()
    bias = step + torch.log(-torch.expm1(-step))                    # softplus(bias) = step
    s.update(A=A, bias=bias, skip=1.0 + 0.1 * rn(D))
    if kind == "scan_step":
        R = case["rows"]
        pool, s["idx"] = slots(R)
        s.update(x=rn(R, D, dtype=dt), dt=(0.5 * rn(R, D)).to(dt), Bm=rn(R, G, S, dtype=dt), Cm=rn(R, G, S, dtype=dt),
                 z=rn(R, D, dtype=dt) if case["gate"] else None, pool=0.5 * rn(pool, D, S))
        return s
    B, T, n = case["B"], case["T"], case["N"] or case["B"]
    s.update(x=rn(B, T, D, dtype=dt), dt=(0.5 * rn(B, T, D)).to(dt), Bm=rn(B, T, G, S, dtype=dt), Cm=rn(B, T, G, S, dtype=dt),
             z=rn(B, T, D, dtype=dt) if case["gate"] else None, h0=0.5 * rn(n, D, S) if case["states"] else None, cu=None, cu_cpu=None)
    if case["N"]:
        s["cu_cpu"] = _lengths(T, case["N"], gen)
        s["cu"] = s["cu_cpu"].to(dev)
    if case["train"]:
        s["leaves"] = [t for t in (s["x"], s["dt"], A, s["Bm"], s["Cm"], s["skip"], s["z"], bias, s["h0"]) if t is not None]
        for t in s["leaves"]:
            t.requires_grad_(True)
        s["dy"] = rn(B, T, D, dtype=dt)
        s["dh"] = 0.1 * rn(n, D, S) if case["states"] else None
    return s


# ---------------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------------
def _recur(a, b):
    """h[:, t] = a[:, t] h[:, t-1] + b[:, t] for all t, by doubling the span that each place has taken in."""
    k, T = 1, a.shape[1]
    while k < T:
        b = torch.cat([b[:, :k], b[:, k:] + a[:, k:] * b[:, :-k]], 1)
        a = torch.cat([a[:, :k], a[:, k:] * a[:, :-k]], 1)
        k *= 2
    return b


def _softplus(v):
    return v.clamp(min=0) + torch.log1p(torch.exp(-v.abs()))


def _per_channel(m, D):
    """[..., G, S] to [..., G, 1, S]-like over the channels: [..., D, S] without a copy where G is 1."""
    G = m.shape[-2]
    return m if G == 1 else m.repeat_interleave(D // G, -2)


def _scan_plain(s):
    D, G, S = s["D"], s["G"], s["S"]
    x, raw, Bm, Cm = s["x"].float(), s["dt"].float() + s["bias"], s["Bm"].float(), s["Cm"].float()
    A, skip = s["A"], s["skip"]
    dt = _softplus(raw)
    n_batch, T = x.shape[:2]
    if s["cu"] is None:
        first, last, seq = slice(0, 1), slice(T - 1, T), None
    else:
        first, last, seq = s["cu"][:-1].long(), s["cu"][1:].long() - 1, s["N"]
    Bd, Cd = _per_channel(Bm, D), _per_channel(Cm, D)
    a = torch.exp(dt[..., None] * A)                                # [B, T, D, S]
    b = (dt * x)[..., None] * Bd
    a_in = a.clone()
    if s["h0"] is not None:                                         # the state before the first token of each sequence
        b[:, first] += a[:, first] * (s["h0"][:, None] if seq is None else s["h0"][None])
    a_in[:, first] = 0
    h = _recur(a_in, b)
    del b
    y = (h * Cd).sum(-1) + skip * x
    out = y
    if s["z"] is not None:
        z = s["z"].float()
        sig = torch.sigmoid(z)
        out = y * z * sig
    fin = h[:, last]
    fin = fin[:, 0] if seq is None else fin[0]
    res = [out.to(s["x"].dtype)] + ([fin.contiguous()] if s["states"] else [])
    if not s["train"]:
        return res
    # the gradients: g_t = dL/dh_t = dy_t C_t + a_{t+1} g_{t+1}
    dout = s["dy"].float()
    dy = dout
    dz = None
    if s["z"] is not None:
        dy = dout * z * sig
        dz = dout * y * sig * (1 + z * (1 - sig))
    g = dy[..., None] * Cd
    if s["dh"] is not None:
        g[:, last] += s["dh"][:, None] if seq is None else s["dh"][None]
    a_next = torch.cat([a_in[:, 1:], torch.zeros_like(a_in[:, :1])], 1)          # zero where the next token begins a sequence
    g = _recur(a_next.flip(1), g.flip(1)).flip(1)
    del a_next, a_in
    per_group = lambda m: m.reshape(n_batch, T, G, D // G, S).sum(3)  # noqa: E731
    dC = per_group(dy[..., None] * h)
    dB = per_group((dt * x)[..., None] * g)
    gB = (g * Bd).sum(-1)
    prev = torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], 1)
    prev[:, first] = 0 if s["h0"] is None else (s["h0"][:, None] if seq is None else s["h0"][None])
    del h
    ga = g * a                                                       # gradient of the state before the token
    w = ga * prev                                                    # and of dt A
    ddt = x * gB + (w * A).sum(-1)
    ddt = ddt * torch.sigmoid(raw)
    dA = (w * dt[..., None]).sum((0, 1))
    grads = [dt * gB + skip * dy, ddt, dA, dB, dC, (dy * x).sum((0, 1))]
    like = [s["x"], s["dt"], A, s["Bm"], s["Cm"], skip]
    if dz is not None:
        grads.append(dz)
        like.append(s["z"])
    grads.append(ddt.sum((0, 1)))
    like.append(s["bias"])
    if s["h0"] is not None:
        gh = ga[:, first]
        grads.append((gh[:, 0] if seq is None else gh[0]).contiguous())
        like.append(s["h0"])
    return res + [g_.to(t.dtype) for g_, t in zip(grads, like)]


def _step_plain(s):
    x, dt = s["x"].float(), _softplus(s["dt"].float() + s["bias"])
    idx = torch.arange(s["rows"], device=x.device) if s["idx"] is None else s["idx"].long()
    live = (idx >= 0)[:, None]
    old = s["pool"][idx.clamp(min=0)]
    Bd, Cd = _per_channel(s["Bm"].float(), s["D"]), _per_channel(s["Cm"].float(), s["D"])
    h = torch.exp(dt[..., None] * s["A"]) * old + (dt * x)[..., None] * Bd
    y = (h * Cd).sum(-1) + s["skip"] * x
    if s["z"] is not None:
        z = s["z"].float()
        y = y * z * torch.sigmoid(z)
    s["pool"][idx[live[:, 0]]] = h[live[:, 0]]
    return [torch.where(live, y, torch.zeros_like(y)).to(s["x"].dtype), s["pool"]]


def _conv_plain(s):
    idx = torch.arange(s["rows"], device=s["x"].device) if s["idx"] is None else s["idx"].long()
    live = (idx >= 0)[:, None]
    win = torch.cat([s["pool"][idx.clamp(min=0)][..., 1:], s["x"].float()[..., None]], -1)
    y = (win * s["w"]).sum(-1)
    if s["b"] is not None:
        y = y + s["b"]
    if s["act"]:
        y = y * torch.sigmoid(y)
    s["pool"][idx[live[:, 0]]] = win[live[:, 0]]
    return [torch.where(live, y, torch.zeros_like(y)).to(s["x"].dtype), s["pool"]]


def _norm_plain(s):
    x, w, r = s["x"].detach(), s["w"].detach(), None if s["r"] is None else s["r"].detach()
    new = x if r is None else (x.float() + r.float()).to(r.dtype)   # the stream as it is kept; the norm is of that
    v = new.float()
    rstd = torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS)
    y = v * rstd * w
    tail = [] if r is None else [new]
    if s["kind"] == "norm8":
        groups = y.reshape(s["rows"], -1, s["group"] or s["D"])
        scale = (groups.abs().amax(-1) / E4M3_MAX).clamp(min=SCALE_MIN)
        q = (groups / scale[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).reshape(y.shape)
        return [q, scale if s["group"] else scale[:, 0]] + tail
    out = [y.to(x.dtype)] + tail
    if not s["train"]:
        return out
    n, dy = v * rstd, s["dy"].float()
    dn = dy * w
    dv = rstd * (dn - n * (dn * n).mean(-1, keepdim=True))
    dw = (dy * n).sum(0)
    if r is None:
        return out + [dv.to(x.dtype), dw]
    dv = dv + s["dr"].float()
    return out + [dv.to(x.dtype), dw, dv.to(r.dtype)]


# ---------------------------------------------------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------------------------------------------------
def _scan_own(s):
    from cula_b200.kda import selective_scan

    def call():
        return selective_scan(s["x"], s["dt"], s["A"], s["Bm"], s["Cm"], D=s["skip"], z=s["z"], dt_bias=s["bias"], dt_softplus=True,
                              initial_state=s["h0"], output_final_state=s["states"], cu_seqlens=s["cu"], cu_seqlens_cpu=s["cu_cpu"])

    if not s["train"]:
        with torch.no_grad():
            y, fin = call()
        return [y] + ([fin] if s["states"] else [])
    y, fin = call()
    outs, ups = ([y, fin], [s["dy"], s["dh"]]) if s["states"] else ([y], [s["dy"]])
    return [*(t.detach() for t in outs), *torch.autograd.grad(outs, s["leaves"], ups)]


def _step_own(s):
    from cula_b200.kda import selective_scan_update
    y = selective_scan_update(s["x"], s["dt"], s["A"], s["Bm"], s["Cm"], s["pool"], state_indices=s["idx"], D=s["skip"], z=s["z"],
                              dt_bias=s["bias"], dt_softplus=True)
    return [y, s["pool"]]


def _conv_own(s):
    from cula_b200.kda import short_conv_update
    y = short_conv_update(s["x"], s["w"], s["pool"], cache_indices=s["idx"], bias=s["b"], activation="silu" if s["act"] else None)
    return [y, s["pool"]]


def _norm_own(s):
    from cula_b200.kda import add_rms_norm, add_rms_norm_fp8
    if s["kind"] == "norm8":
        q, scale, new = add_rms_norm_fp8(s["x"], s["w"], residual=s["r"], eps=EPS, group_size=s["group"] or None)
        return [q, scale] + ([] if s["r"] is None else [new])
    if not s["train"]:
        with torch.no_grad():
            y, new = add_rms_norm(s["x"], s["w"], residual=s["r"], eps=EPS)
        return [y] + ([] if s["r"] is None else [new])
    y, new = add_rms_norm(s["x"], s["w"], residual=s["r"], eps=EPS)
    if s["r"] is None:
        return [y.detach(), *torch.autograd.grad([y], [s["x"], s["w"]], [s["dy"]])]
    return [y.detach(), new.detach(), *torch.autograd.grad([y, new], [s["x"], s["w"], s["r"]], [s["dy"], s["dr"]])]


def run(state):
    s, kind = state, state["kind"]
    if own:
        return {"scan": _scan_own, "scan_step": _step_own, "conv_step": _conv_own, "norm": _norm_own, "norm8": _norm_own}[kind](s)
    with torch.no_grad():
        return {"scan": _scan_plain, "scan_step": _step_plain, "conv_step": _conv_plain, "norm": _norm_plain, "norm8": _norm_plain}[kind](s)


# ---------------------------------------------------------------------------------------------------------------------
# 64 bits, token by token; gradients by differentiating that
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    f = lambda t: None if t is None else t.detach().double()  # noqa: E731
    if kind == "conv_step":
        x, w, b, pool = f(s["x"]), f(s["w"]), f(s["b"]), f(s["pool"])
        y = torch.zeros_like(x)
        for i, slot in enumerate(range(case["rows"]) if s["idx"] is None else s["idx"].tolist()):
            if slot >= 0:
                pool[slot] = torch.cat([pool[slot][:, 1:], x[i][:, None]], 1)
                y[i] = torch.einsum("dw,dw->d", pool[slot], w) + (0 if b is None else b)
        return [torch.nn.functional.silu(y) if case["act"] else y, pool]
    if kind in ("norm", "norm8"):
        leaf = lambda t: None if t is None else f(t).requires_grad_(bool(case.get("train")))  # noqa: E731
        x, w, r = leaf(s["x"]), leaf(s["w"]), leaf(s["r"])
        total = x if r is None else x + r
        if r is not None:                                            # kept in the stream's type; the rounding has derivative one
            total = total + (total.detach().float().to(s["r"].dtype).double() - total.detach())
        y = total / torch.sqrt(torch.mean(total * total, -1, keepdim=True) + EPS) * w
        tail = [] if r is None else [total]
        if kind == "norm8":
            size = case["group"] or case["D"]
            most = torch.stack([p.abs().max(-1).values for p in y.split(size, -1)], -1)
            scale = torch.clamp(most / E4M3_MAX, min=SCALE_MIN)
            q = (y / scale.repeat_interleave(size, -1)).float().to(torch.float8_e4m3fn).double()
            return [q, scale if case["group"] else scale[:, 0]] + tail
        if not case["train"]:
            return [y] + tail
        outs, ups, leaves = [y] + tail, [f(s["dy"])] + ([] if r is None else [f(s["dr"])]), [x, w] + ([] if r is None else [r])
        return [t.detach() for t in outs] + list(torch.autograd.grad(outs, leaves, ups))
    train = bool(case.get("train"))
    names = ["x", "dt", "A", "Bm", "Cm", "skip"] + (["z"] if s["z"] is not None else []) + ["bias"]
    if kind == "scan" and s["h0"] is not None:
        names.append("h0")
    v = {k: f(s[k]).requires_grad_(train) for k in names}
    D, G = case["D"], case["G"]
    delta = torch.nn.functional.softplus(v["dt"] + v["bias"])

    def advance(h, row):                                             # one token of some sequences; row indexes the flat inputs
        step, x = row(delta), row(v["x"])
        wide = lambda m: m.unsqueeze(-2).expand(*m.shape[:-1], D // G, m.shape[-1]).flatten(-3, -2)  # noqa: E731
        h = torch.exp(step.unsqueeze(-1) * v["A"]) * h + (step * x).unsqueeze(-1) * wide(row(v["Bm"]))
        y = torch.einsum("...ds,...ds->...d", h, wide(row(v["Cm"]))) + v["skip"] * x
        return h, y if "z" not in v else y * torch.nn.functional.silu(row(v["z"]))

    if kind == "scan_step":
        pool = f(s["pool"])
        idx = list(range(case["rows"])) if s["idx"] is None else s["idx"].tolist()
        y = torch.zeros_like(v["x"])
        for i, slot in enumerate(idx):
            if slot >= 0:
                pool[slot], y[i] = advance(pool[slot], lambda m: m[i])  # noqa: B023
        return [y, pool]
    with torch.set_grad_enabled(train):
        if s["cu"] is None:
            h = v["h0"] if "h0" in v else torch.zeros(case["B"], D, case["S"], dtype=torch.float64, device=s["x"].device)
            rows = []
            # by bands of tokens taken apart once: an index into the whole input for each token would make its gradient quadratic
            parts = {k: m.unbind(1) for k, m in (("d", delta), *((k, v[k]) for k in ("x", "Bm", "Cm", "z") if k in v))}
            key = {id(delta): "d", **{id(v[k]): k for k in ("x", "Bm", "Cm", "z") if k in v}}
            for t in range(case["T"]):
                h, y = advance(h, lambda m: parts[key[id(m)]][t])  # noqa: B023
                rows.append(y)
            y, fin = torch.stack(rows, 1), h
        else:
            parts = {k: m[0].unbind(0) for k, m in (("d", delta), *((k, v[k]) for k in ("x", "Bm", "Cm", "z") if k in v))}
            key = {id(delta): "d", **{id(v[k]): k for k in ("x", "Bm", "Cm", "z") if k in v}}
            rows, fins, cu = [], [], s["cu_cpu"].tolist()
            for n in range(case["N"]):
                h = v["h0"][n] if "h0" in v else torch.zeros(D, case["S"], dtype=torch.float64, device=s["x"].device)
                for t in range(cu[n], cu[n + 1]):
                    h, y = advance(h, lambda m: parts[key[id(m)]][t])  # noqa: B023
                    rows.append(y)
                fins.append(h)
            y, fin = torch.stack(rows)[None], torch.stack(fins)
        outs = [y] + ([fin] if case["states"] else [])
        if not train:
            return outs
        grads = torch.autograd.grad(outs, [v[k] for k in names], [f(s["dy"])] + ([f(s["dh"])] if case["states"] else []))
    return [t.detach() for t in outs] + list(grads)


def work(case):
    kind, D = case["kind"], case["D"]
    if kind == "conv_step":
        live = case["rows"]
        return dict(bytes=live * D * (2 + 2 + 8 * case["W"]) + D * 4 * (case["W"] + 1), flops=live * D * (2 * case["W"] + 5))
    e = 2 if case["dtype"] == "bf16" else 4
    if kind in ("norm", "norm8"):
        n = case["rows"] * D
        r = {"none": 0, "bf16": 2, "fp32": 4}[case["res"]]
        if kind == "norm8":
            return dict(bytes=n * (e + 2 * r + 1) + case["rows"] * 4 * (D // case["group"] if case["group"] else 1) + 4 * D, flops=7 * n)
        fwd = n * (2 * e + 2 * r) + 4 * D
        # a training step reads the stream and the upstream gradients again and writes the gradients
        return dict(bytes=fwd + (n * ((r or e) + e + r + e + r) + 4 * D if case["train"] else 0), flops=n * (18 if case["train"] else 5))
    S, G = case["S"], case["G"]
    rows = case["rows"] if kind == "scan_step" else case["B"] * case["T"]
    acts = rows * (D * e * (2 + bool(case["gate"])) + 2 * G * S * e)           # x, dt, z, B, C
    if kind == "scan_step":
        return dict(bytes=acts + rows * D * e + rows * D * S * 8 + D * 4 * (S + 2), flops=rows * D * (7 * S + 20))
    state = (case["N"] or case["B"]) * D * S * 4 if case["states"] else 0
    fwd_bytes, fwd_flops = acts + rows * D * e + 2 * state + D * 4 * (S + 2), rows * D * (7 * S + 20)
    if not case["train"]:
        return dict(bytes=fwd_bytes, flops=fwd_flops)
    # a training step reads its inputs and the upstream gradient again and writes every gradient
    return dict(bytes=fwd_bytes + acts + rows * D * e + acts + 3 * state + 2 * D * 4 * (S + 2), flops=fwd_flops + rows * D * (20 * S + 40))
