"""The selective scan and its single-token step: the oracle against a direct sum and finite differences (CPU), refusals (CPU), and the
CUDA operators against the oracle in 64 bits (GPU): values, states and every gradient.

Tolerances, fixed before the first run: an output in bf16 is rounded once, at most 2^-8 of its value, so its error in norm is at most 2^-8
plus that of the fp32 arithmetic; that one is at most 2^-22 (the exponential's error) per step on the way from an input to an output, at
most T + 64 steps, and cancellation between terms of random sign makes it at most four times larger relative to the result."""
import pytest
import torch
import torch.nn.functional as F

from oracle.naive_kda import err_ratio
from oracle.ssm import selective_scan_ref, selective_scan_update_ref


def tol(dtype, T):
    return (2.0 ** -8 if dtype == torch.bfloat16 else 0.0) + 4 * (T + 64) * 2.0 ** -22


def make(B, T, D, S, G=1, dtype=torch.bfloat16, gate=True, skip=True, bias=True, h0=0, seed=0, four_dims=None):
    """Inputs on the CPU, activations rounded to their type. Steps from 1e-3 to 1e-1, rates as at a layer's start."""
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    bc = (B, T, G, S) if (G > 1 if four_dims is None else four_dims) else (B, T, S)
    step = torch.exp(-6.9 + 4.6 * torch.rand(D, generator=gen))
    return dict(x=rn(B, T, D).to(dtype), dt=(0.5 * rn(B, T, D)).to(dtype), A=-torch.arange(1, S + 1.0) * (0.1 * rn(D, S)).exp(),
                B=rn(*bc).to(dtype), C=rn(*bc).to(dtype), D=1 + 0.1 * rn(D) if skip else None, z=rn(B, T, D).to(dtype) if gate else None,
                dt_bias=torch.log(torch.expm1(step)) if bias else None, dt_softplus=bias, initial_state=0.5 * rn(h0, D, S) if h0 else None)


def in64(a, grad=False):
    return {k: v.double().requires_grad_(grad) if torch.is_tensor(v) else v for k, v in a.items()}


def on_gpu(a, grad=False):
    return {k: v.cuda().requires_grad_(grad) if torch.is_tensor(v) else v for k, v in a.items()}


# ------------------------------------------------------------------ CPU ------------------------------------------------------------------
def test_oracle_is_the_sum_over_past_tokens():
    a = in64(make(1, 9, 8, 3, h0=1, dtype=torch.float32))
    y, fin = selective_scan_ref(**a)
    step = F.softplus(a["dt"] + a["dt_bias"])[0]
    total = torch.cumsum(step, 0)
    for t in range(9):
        h = torch.exp(total[t][:, None] * a["A"]) * a["initial_state"][0]
        for s in range(t + 1):
            h = h + torch.exp((total[t] - total[s])[:, None] * a["A"]) * (step[s] * a["x"][0, s])[:, None] * a["B"][0, s]
        ref = ((h * a["C"][0, t]).sum(-1) + a["D"] * a["x"][0, t]) * F.silu(a["z"][0, t])
        assert (y[0, t] - ref).abs().max() < 1e-12
    assert (fin[0] - h).abs().max() < 1e-12


def test_oracle_gradients_against_differences():
    a = in64(make(1, 6, 8, 2, h0=2, dtype=torch.float32), grad=True)
    names = [k for k, v in a.items() if torch.is_tensor(v)]
    cu = torch.tensor([0, 4, 6])
    assert torch.autograd.gradcheck(lambda *v: selective_scan_ref(**{**a, **dict(zip(names, v))}, cu_seqlens=cu), [a[k] for k in names])


def test_refusals():
    from cula_b200.kda import selective_scan, selective_scan_update
    a = make(2, 5, 16, 4)

    def bad(error, match, **change):
        with pytest.raises(error, match=match):
            selective_scan(**{**a, **change})

    bad(AssertionError, r"\[B, T, D\]", x=a["x"][0])
    bad(AssertionError, "bfloat16 or float32", x=a["x"].half())
    bad(AssertionError, "shape of x", dt=a["dt"][:, :4])
    bad(AssertionError, "shape of x", z=a["z"][:, :4])
    bad(AssertionError, "type of x", dt=a["dt"].float())
    bad(AssertionError, "type of x", B=a["B"].float())
    bad(AssertionError, r"A must be \[D, S\]", A=a["A"][:8])
    bad(AssertionError, "1 to 64", A=torch.zeros(16, 65), B=torch.zeros(2, 5, 65).bfloat16(), C=torch.zeros(2, 5, 65).bfloat16())
    bad(AssertionError, "1 to 64", A=torch.zeros(16, 0), B=torch.zeros(2, 5, 0).bfloat16(), C=torch.zeros(2, 5, 0).bfloat16())
    bad(AssertionError, "state size of A", B=a["B"][..., :3], C=a["C"][..., :3])
    bad(AssertionError, "tokens of x", B=a["B"][:, :4], C=a["C"][:, :4])
    bad(AssertionError, "B and C must be", B=a["B"][:, :, None])
    bad(AssertionError, "multiple of 8", B=a["B"][:, :, None].expand(2, 5, 4, 4), C=a["C"][:, :, None].expand(2, 5, 4, 4))
    bad(AssertionError, "multiple of 8", B=a["B"][:, :, None].expand(2, 5, 3, 4), C=a["C"][:, :, None].expand(2, 5, 3, 4))
    bad(AssertionError, r"D must be \[D\]", D=torch.ones(8))
    bad(AssertionError, r"dt_bias must be \[D\]", dt_bias=torch.ones(8))
    bad(ValueError, "initial_state must be", initial_state=torch.zeros(1, 16, 4))
    bad(AssertionError, "float32", initial_state=torch.zeros(2, 16, 4).bfloat16())
    bad(ValueError, "on the device of x", A=a["A"].to("meta"))
    bad(ValueError, "on the device of x", z=a["z"].to("meta"))
    bad(ValueError, "on the device of x", initial_state=torch.zeros(2, 16, 4, device="meta"))
    bad(ValueError, "batch size is expected to be 1", cu_seqlens=torch.tensor([0, 5], dtype=torch.int32))
    one = {k: v[:1] if torch.is_tensor(v) and v.dim() == 3 else v for k, v in a.items()}
    with pytest.raises(ValueError, match="past the 5 tokens"):
        selective_scan(**{**one, "cu_seqlens": torch.tensor([0, 3, 6], dtype=torch.int32)})
    with pytest.raises(ValueError, match="initial_state must be"):
        selective_scan(**{**one, "cu_seqlens": torch.tensor([0, 3, 5], dtype=torch.int32), "initial_state": torch.zeros(1, 16, 4)})
    with pytest.raises(ValueError, match="non-decreasing"):
        selective_scan(**{**one, "cu_seqlens": torch.tensor([0, 4, 3], dtype=torch.int32)})
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            selective_scan(**a)

    s = dict(x=a["x"][:, 0], dt=a["dt"][:, 0], A=a["A"], B=a["B"][:, 0], C=a["C"][:, 0], state=torch.zeros(2, 16, 4))

    def bad_step(error, match, **change):
        with pytest.raises(error, match=match):
            selective_scan_update(**{**s, **change})

    bad_step(AssertionError, r"\[N, D\]", x=a["x"])
    bad_step(ValueError, "state must be", state=torch.zeros(2, 16, 5))
    bad_step(AssertionError, "contiguous float32", state=torch.zeros(2, 16, 4).bfloat16())
    bad_step(AssertionError, "contiguous float32", state=torch.zeros(2, 4, 16).transpose(1, 2))
    bad_step(ValueError, "holds 1 states for 2", state=torch.zeros(1, 16, 4))
    bad_step(ValueError, "one int32 slot", state_indices=torch.zeros(3, dtype=torch.int32))
    bad_step(ValueError, "one int32 slot", state_indices=torch.zeros(2))
    bad_step(ValueError, "on the device of x", state_indices=torch.zeros(2, dtype=torch.int32, device="meta"))
    bad_step(ValueError, "on the device of x", state=torch.zeros(2, 16, 4, device="meta"))
    bad_step(ValueError, "out must be", out=torch.zeros(2, 16))
    bad_step(AssertionError, "shape of x", dt=a["dt"][:, 0, :8])
    bad_step(AssertionError, "B and C must be", B=a["B"])
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            selective_scan_update(**s)


def test_c_entries_refuse_what_they_cannot_do():
    """No null structure, no sizes that contradict each other: an error code before anything is launched."""
    import ctypes

    from cula_b200 import _native
    lib = _native.lib()
    for name in ("selective_scan_fwd", "selective_scan_bwd", "selective_step", "conv_step", "add_rms_norm_fwd", "add_rms_norm_bwd"):
        call = getattr(lib, "cula_kda_" + name)
        assert call(None, None) == -1
        zeros = ctypes.create_string_buffer(1024)                   # every size zero, every pointer null
        assert call(ctypes.byref(zeros), None) in (0, -1)
    assert lib.cula_kda_selective_scan_tiles(64, 1, 65) == -1 and lib.cula_kda_selective_scan_tiles(200, 1, 16) == 4
    assert lib.cula_kda_selective_scan_state_floats(200, 1, 16) == 4 * 1024 and lib.cula_kda_selective_scan_state_floats(0, 1, 16) == -1
    assert lib.cula_kda_add_rms_norm_shares(128, 0) == 0


def chunks_of(T, lens):
    return [-(-n // 64) for n in ([T] if lens is None else lens)]


CUT = [(None, 1500, 40, 16), ([700, 0, 1000, 30, 129], 1900, 24, 12)]


@pytest.mark.parametrize("backward", [False, True])
def test_few_channels_and_long_sequences_are_cut(backward):
    """What the GPU test of cut sequences stands on; and many short sequences of many channels are not."""
    from cula_b200 import _native
    plan, tiles = _native.host().selective_scan_segments, _native.lib().cula_kda_selective_scan_tiles
    for lens, T, D, S in CUT:
        chunks = chunks_of(T, lens)
        assert 0 < plan(len(chunks), sum(chunks), max(chunks), tiles(D, 1, S), lens is not None, backward) < max(chunks)
    assert plan(64, 64 * 4, 4, tiles(4096, 1, 16), False, backward) == 0 and plan(1, 1, 1, 1, False, backward) == 0


# ------------------------------------------------------------------ GPU ------------------------------------------------------------------
def check_all(a, cu=None, want_final=True, seed=9, names=None):
    """Outputs and every gradient of a call against the oracle's."""
    from cula_b200.kda import selective_scan
    gen = torch.Generator().manual_seed(seed)
    r, d = in64(a, True), on_gpu(a, True)
    y_ref, f_ref = selective_scan_ref(**r, cu_seqlens=cu)
    dy, df = torch.randn(*y_ref.shape, generator=gen).to(a["x"].dtype), 0.1 * torch.randn(*f_ref.shape, generator=gen)
    y, fin = selective_scan(**d, output_final_state=want_final, cu_seqlens=None if cu is None else cu.cuda())
    with torch.no_grad():
        y_plain, fin_plain = selective_scan(**d, output_final_state=want_final, cu_seqlens=None if cu is None else cu.cuda())
    leaves = [k for k, v in a.items() if torch.is_tensor(v)]
    if want_final:
        ref = torch.autograd.grad([y_ref, f_ref], [r[k] for k in leaves], [dy.double(), df.double()])
        got = torch.autograd.grad([y, fin], [d[k] for k in leaves], [dy.cuda(), df.cuda()])
    else:
        ref = torch.autograd.grad([y_ref], [r[k] for k in leaves], [dy.double()], allow_unused=True)
        got = torch.autograd.grad([y], [d[k] for k in leaves], [dy.cuda()])
    torch.cuda.synchronize()
    T = a["x"].shape[1]
    assert y.dtype == a["x"].dtype and torch.equal(y, y_plain)
    errors = {"y": err_ratio(y_ref.detach(), y.detach().double().cpu()) / tol(y.dtype, T)}
    if want_final:
        assert fin.dtype == torch.float32 and torch.equal(fin, fin_plain)
        errors["fin"] = err_ratio(f_ref.detach(), fin.detach().double().cpu()) / tol(fin.dtype, T)
    for k, g, g_ref in zip(leaves, got, ref):
        assert g.dtype == a[k].dtype and g.shape == a[k].shape
        errors[k] = err_ratio(g_ref, g.double().cpu()) / tol(g.dtype, T)
    assert all(e < 1 for e in errors.values()), errors


CASES = [
    # B, T, D, S, G, dtype, gate, skip, bias, states
    (1, 1, 8, 1, 1, "bf16", True, True, True, True),
    (2, 7, 24, 3, 1, "fp32", False, True, True, True),
    (1, 64, 64, 16, 1, "bf16", True, False, True, False),
    (3, 65, 72, 16, 1, "fp32", True, True, True, True),
    (2, 130, 128, 12, 2, "bf16", True, True, False, True),
    (1, 33, 264, 8, 1, "fp32", True, True, True, False),
    (2, 40, 48, 17, 3, "bf16", True, True, True, True),
    (1, 100, 40, 32, 1, "fp32", False, False, False, True),
    (1, 50, 24, 33, 1, "bf16", True, True, True, True),
    (2, 31, 16, 64, 2, "fp32", True, True, True, True),
    (1, 9, 520, 4, 5, "fp32", True, True, True, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,D,S,G,dtype,gate,skip,bias,states", CASES)
def test_scan_matches_oracle(B, T, D, S, G, dtype, gate, skip, bias, states):
    dtype = torch.bfloat16 if dtype == "bf16" else torch.float32
    a = make(B, T, D, S, G, dtype, gate, skip, bias, B if states else 0, seed=T)
    if not bias:                                                    # steps as they are: positive, small
        a["dt"] = (0.05 * a["dt"].float().abs()).to(dtype)
    check_all(a, want_final=states)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,S,dtype,tail", [([1, 63, 64, 65, 7], 16, "bf16", 0), ([5, 0, 130, 0], 12, "fp32", 9), ([0, 3], 40, "fp32", 1),
                                               ([8, 8, 8], 5, "bf16", 0)])
def test_scan_of_packed_sequences(lens, S, dtype, tail):
    dtype = torch.bfloat16 if dtype == "bf16" else torch.float32
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    check_all(make(1, int(cu[-1]) + tail, 72, S, 1, dtype, h0=len(lens), seed=S), cu=cu)


@pytest.mark.gpu
def test_rows_past_the_packed_tokens_are_zero():
    from cula_b200.kda import selective_scan
    a = make(1, 20, 16, 4, h0=2)
    for k in ("x", "dt", "B", "C", "z"):
        a[k][:, 13:] = float("nan")
    d = on_gpu(a, True)
    y, fin = selective_scan(**d, output_final_state=True, cu_seqlens=torch.tensor([0, 6, 13], dtype=torch.int32, device="cuda"))
    grads = torch.autograd.grad([y, fin], [d[k] for k in ("x", "dt", "B", "C", "z", "A")], [torch.ones_like(y), torch.ones_like(fin)])
    assert (y[:, 13:] == 0).all() and y.isfinite().all() and fin.isfinite().all()
    for g in grads[:5]:
        assert (g[:, 13:] == 0).all() and g.isfinite().all()
    assert grads[5].isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("lens,T,D,S", [(None, 1500, 40, 16), ([700, 0, 1000, 30, 129], 1900, 24, 12)])
def test_sequences_cut_into_segments(lens, T, D, S):
    """Few channels and long sequences: the planner cuts them, forward and backward."""
    cu = None if lens is None else torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    check_all(make(1, T, D, S, 1, torch.float32, h0=1 if lens is None else len(lens), seed=T), cu=cu)


@pytest.mark.gpu
def test_errors_do_not_add_up_over_a_memory():
    """Fast and slow channels in 32 bits. The exponential's mean error, at most 2^-26 where states remember up to 56 tokens, adds up to 8.4e-7;
    three roundings per token, at most 2^-24 and independent, to 3^0.5 (2 x 56)^0.5 2^-25 in root mean square, there and back (5.5e-7): 1e-6
    for both in quadrature, a quarter more for the spread between channels."""
    from cula_b200.kda import selective_scan
    a = make(2, 200, 64, 32, 1, torch.float32, h0=2, seed=21)
    gen = torch.Generator().manual_seed(22)
    dy, df = torch.randn(2, 200, 64, generator=gen), 0.1 * torch.randn(2, 64, 32, generator=gen)
    leaves = [k for k, v in a.items() if torch.is_tensor(v)]
    r, d = in64(a, True), on_gpu(a, True)
    ref, got = selective_scan_ref(**r), selective_scan(**d, output_final_state=True)
    g_ref = torch.autograd.grad(ref, [r[k] for k in leaves], [dy.double(), df.double()])
    g_got = torch.autograd.grad(got, [d[k] for k in leaves], [dy.cuda(), df.cuda()])
    errors = {k: err_ratio(u.detach(), v.detach().double().cpu()) for k, u, v in zip(["y", "fin"] + leaves, [*ref, *g_ref], [*got, *g_got])}
    assert all(e < 1.25e-6 for e in errors.values()), errors


@pytest.mark.gpu
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_bad_value_stays_in_its_channel(value):
    """NaN or infinity in one live token of x: its channel from that token on, and no other channel, sequence or earlier token."""
    from cula_b200.kda import selective_scan
    a = on_gpu(make(2, 40, 72, 16, 1, torch.float32, h0=2, seed=31))
    clean = selective_scan(**a, output_final_state=True)
    a["x"][1, 21, 5] = value
    y, fin = selective_scan(**a, output_final_state=True)
    hit = torch.zeros(2, 40, 72, dtype=torch.bool, device="cuda")
    hit[1, 21:, 5] = True
    assert torch.equal(y[~hit], clean[0][~hit]) and not y[hit].isfinite().any()
    assert torch.equal(fin[0], clean[1][0]) and torch.equal(fin[1, torch.arange(72) != 5], clean[1][1, torch.arange(72) != 5])
    assert not fin[1, 5].isfinite().any()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [13, 16, 75])
def test_states_that_forget_at_once(T):
    """Rates of minus infinity: such a state holds its token alone. The last tile of tokens is whole or not."""
    from cula_b200.kda import selective_scan
    a = make(2, T, 24, 6, 1, torch.float32, h0=2, seed=T)
    a["A"][::2, 1::2] = float("-inf")
    gen = torch.Generator().manual_seed(23)
    dy, df = torch.randn(2, T, 24, generator=gen), torch.randn(2, 24, 6, generator=gen)
    leaves = ["x", "A", "B", "C", "D", "z", "initial_state"]         # of dt, autograd's derivative of the oracle is 0 times infinity
    r, d = in64(a, True), on_gpu(a, True)
    ref, got = selective_scan_ref(**r), selective_scan(**d, output_final_state=True)
    assert got[1].isfinite().all()
    g_ref = torch.autograd.grad(ref, [r[k] for k in leaves], [dy.double(), df.double()])
    g_got = torch.autograd.grad(got, [d[k] for k in leaves + ["dt"]], [dy.cuda(), df.cuda()])
    for k, u, v in zip(["y", "fin"] + leaves, [*ref, *g_ref], [*got, *g_got]):
        assert err_ratio(u.detach(), v.detach().double().cpu()) < tol(torch.float32, T), k
    assert g_got[-1].isfinite().all()


@pytest.mark.gpu
def test_no_tokens():
    from cula_b200.kda import selective_scan
    a = on_gpu(make(2, 0, 16, 4, h0=2))
    y, fin = selective_scan(**a, output_final_state=True)
    assert y.shape == (2, 0, 16) and torch.equal(fin, a["initial_state"])
    a = on_gpu(make(1, 5, 16, 4))
    y, fin = selective_scan(**a, output_final_state=True, cu_seqlens=torch.tensor([0, 0, 0], dtype=torch.int32, device="cuda"))
    assert (y == 0).all() and fin.shape == (2, 16, 4) and (fin == 0).all()
    y, fin = selective_scan(**a, output_final_state=True, cu_seqlens=torch.tensor([0], dtype=torch.int32, device="cuda"))
    assert (y == 0).all() and fin.shape == (0, 16, 4)


@pytest.mark.gpu
@pytest.mark.parametrize("T,cu,n", [(0, None, 2), (5, [0, 0, 0], 2), (5, [0], 0)])
def test_gradients_of_no_tokens(T, cu, n):
    """They are zeros, and the one of the first states is that of the last."""
    from cula_b200.kda import selective_scan
    a = on_gpu(make(2 if cu is None else 1, T, 16, 4, h0=2), grad=True)
    a["initial_state"] = torch.randn(n, 16, 4, device="cuda", requires_grad=True)
    y, fin = selective_scan(**a, output_final_state=True, cu_seqlens=None if cu is None else torch.tensor(cu, dtype=torch.int32, device="cuda"))
    assert torch.equal(fin, a["initial_state"]) and (y == 0).all()
    dfin = torch.randn_like(fin)
    names = [k for k, v in a.items() if torch.is_tensor(v)]
    for k, g in zip(names, torch.autograd.grad([y, fin], [a[k] for k in names], [torch.ones_like(y), dfin])):
        assert g.shape == a[k].shape and g.dtype == a[k].dtype
        assert torch.equal(g, dfin if k == "initial_state" else torch.zeros_like(a[k])), k


@pytest.mark.gpu
def test_gradients_are_not_differentiated_again():
    from cula_b200.kda import selective_scan
    a = on_gpu(make(1, 9, 16, 4, dtype=torch.float32), grad=True)
    plain = torch.autograd.grad(selective_scan(**a)[0].square().sum(), [a["x"], a["A"]])
    gx, gA = torch.autograd.grad(selective_scan(**a)[0].square().sum(), [a["x"], a["A"]], create_graph=True)
    assert torch.equal(gx, plain[0]) and torch.equal(gA, plain[1])
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        torch.autograd.grad(gx.sum(), a["x"])
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        torch.autograd.grad((gA * a["A"]).sum(), a["A"])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_views_are_read_in_place_or_copied(dtype):
    """Parts of wider rows, broadcast rows, misaligned views: the same values as contiguous tensors, gradients in the views' shape."""
    from cula_b200.kda import selective_scan
    gen = torch.Generator().manual_seed(3)
    rn = lambda *s: torch.randn(*s, generator=gen).to(dtype).cuda()  # noqa: E731
    B, T, D, S = 2, 37, 32, 8
    A, h0 = -torch.rand(D, S, generator=gen).cuda() - 0.1, torch.randn(B, D, S, generator=gen).cuda()
    wide, bc, flat = rn(B, T, 3 * D), rn(B, T, 2 * S + 3), rn(B * T * D + 1)
    for x, dt, z, Bm, Cm in [(wide[..., :D], wide[..., D:2 * D], wide[..., 2 * D:], bc[..., :S], bc[..., S:2 * S]),
                             (flat[1:].view(B, T, D), wide[:1, :, :D].expand(B, T, D), wide[:, :1, :D].expand(B, T, D), bc[..., 1:S + 1], bc[:, :1, :S].expand(B, T, S)),
                             (wide.transpose(0, 1)[:B, :B, :D].transpose(0, 1), *(wide[:, :B, :D],) * 2, *(bc[:, :B, :S],) * 2)]:
        leaves = [t.detach().requires_grad_(True) for t in (x, dt, z, Bm, Cm)]
        twins = [t.detach().clone(memory_format=torch.contiguous_format).requires_grad_(True) for t in (x, dt, z, Bm, Cm)]
        outs = []
        for v in (leaves, twins):
            y, fin = selective_scan(v[0], v[1], A, v[3], v[4], z=v[2], dt_softplus=True, initial_state=h0[:v[0].shape[0]], output_final_state=True)
            outs.append([y, fin, *torch.autograd.grad([y, fin], v, [torch.ones_like(y), torch.ones_like(fin)])])
        for p, q in zip(*outs):
            assert p.shape == q.shape and torch.equal(p, q)


@pytest.mark.gpu
def test_gradients_are_the_same_from_run_to_run_and_agree_with_differences():
    from cula_b200.kda import selective_scan
    a = make(2, 90, 136, 16, 1, torch.float32, h0=2, seed=4)
    leaves = [k for k, v in a.items() if torch.is_tensor(v)]
    gen = torch.Generator().manual_seed(5)
    dy, df = torch.randn(2, 90, 136, generator=gen).cuda(), torch.randn(2, 136, 16, generator=gen).cuda()

    def grads():
        d = on_gpu(a, True)
        y, fin = selective_scan(**d, output_final_state=True)
        return torch.autograd.grad([y, fin], [d[k] for k in leaves], [dy, df])

    first = grads()
    for g, h in zip(first, grads()):
        assert torch.equal(g, h)
    d = on_gpu(a)

    def loss(change):
        y, fin = selective_scan(**{**d, **change}, output_final_state=True)
        return ((y * dy).double().sum() + (fin * df).double().sum()).item()

    for k, g in zip(leaves, first):
        way = torch.randn(a[k].shape, generator=gen).cuda()
        eps = 1e-2 * a[k].abs().mean().item()                       # the third-order term is eps^2 of the value, rounding 2^-22 / eps
        diff = (loss({k: d[k] + eps * way}) - loss({k: d[k] - eps * way})) / (2 * eps)
        assert abs(diff - (g.double() * way).sum().item()) < 2e-2 * (g.double().norm() * way.norm() / way.numel() ** 0.5).item(), k


@pytest.mark.gpu
def test_parameters_in_16_bits_and_one_tensor_in_several_places():
    """bf16 parameters get bf16 gradients; x passed as dt and z too gets the sum of theirs."""
    from cula_b200.kda import selective_scan
    a = make(2, 40, 24, 6, h0=0, seed=8)
    a = {**a, "dt": None, "z": None, **{k: a[k].bfloat16() for k in ("A", "D", "dt_bias")}}
    r, d = in64(a, True), on_gpu(a, True)
    y_ref, _ = selective_scan_ref(**{**r, "dt": r["x"], "z": r["x"]})
    y, _ = selective_scan(**{**d, "dt": d["x"], "z": d["x"]})
    names = ["x", "A", "B", "C", "D", "dt_bias"]
    got, ref = torch.autograd.grad(y.float().sum(), [d[k] for k in names]), torch.autograd.grad(y_ref.sum(), [r[k] for k in names])
    assert err_ratio(y_ref.detach(), y.detach().double().cpu()) < tol(torch.bfloat16, 40)
    for k, g, h in zip(names, got, ref):
        # three gradients of x are rounded one by one and their sum twice more
        assert g.dtype == torch.bfloat16 and err_ratio(h, g.double().cpu()) < (5 if k == "x" else 1) * tol(torch.bfloat16, 40), k


@pytest.mark.gpu
def test_only_one_result_is_differentiated():
    from cula_b200.kda import selective_scan
    a = make(1, 30, 16, 4, 1, torch.float32, h0=1)
    r, d = in64(a, True), on_gpu(a, True)
    y_ref, f_ref = selective_scan_ref(**r)
    y, fin = selective_scan(**d, output_final_state=True)
    for out, out_ref in ((y, y_ref), (fin, f_ref)):
        names = ["x", "dt", "A", "B", "initial_state"]
        got = torch.autograd.grad(out.sum(), [d[k] for k in names], retain_graph=True)
        ref = torch.autograd.grad(out_ref.sum(), [r[k] for k in names], retain_graph=True)
        for g, h in zip(got, ref):
            assert err_ratio(h, g.double().cpu()) < tol(torch.float32, 30)
    with torch.no_grad():
        assert not selective_scan(**d)[0].requires_grad and selective_scan(**d)[1] is None


@pytest.mark.gpu
@pytest.mark.parametrize("cut", [1, 64, 77])
def test_a_prompt_in_two_calls(cut):
    from cula_b200.kda import selective_scan
    a = make(2, 150, 64, 16, h0=2, seed=6)
    d = on_gpu(a)
    part = lambda lo, hi, **kw: {k: v[:, lo:hi] if k in ("x", "dt", "B", "C", "z") else v for k, v in {**d, **kw}.items()}  # noqa: E731
    y, fin = selective_scan(**d, output_final_state=True)
    y1, mid = selective_scan(**part(0, cut), output_final_state=True)
    y2, end = selective_scan(**part(cut, 150, initial_state=mid), output_final_state=True)
    # Not bit for bit: a sequence may be cut into segments, whose states are joined with one exponential of the sum of their steps in the
    # place of a product of exponentials. Both are within 2^-22 per step of the definition (tol without the output's rounding), so they are
    # within twice that of each other; outputs may then fall on either side of a rounding border, half a step of 2^-8 away.
    assert err_ratio(fin.cpu(), end.cpu()) < 2 * tol(torch.float32, 150)
    assert err_ratio(y.double().cpu(), torch.cat([y1, y2], 1).double().cpu()) < 2.0 ** -8 + 2 * tol(torch.float32, 150)


@pytest.mark.gpu
def test_forward_and_backward_in_a_cuda_graph_on_another_stream():
    from cula_b200.kda import selective_scan
    a = make(1, 700, 32, 16, h0=1, seed=7)                          # cut into segments: every kernel is in it
    d = on_gpu(a, True)
    leaves = [v for v in d.values() if torch.is_tensor(v)]
    dy = torch.randn(1, 700, 32, device="cuda").bfloat16()

    def step():
        y, fin = selective_scan(**d, output_final_state=True)
        return [y, fin, *torch.autograd.grad([y, fin], leaves, [dy, torch.ones_like(fin)])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = [t.clone() for t in step()]
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    with torch.no_grad():
        d["x"].mul_(2.0)
    graph.replay()
    torch.cuda.synchronize()
    doubled = [t.clone() for t in static]
    for t, u in zip(doubled, step()):
        assert torch.equal(t, u)
    with torch.no_grad():
        d["x"].mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    for t, u in zip(static, eager):
        assert torch.equal(t, u)


@pytest.mark.gpu
def test_rows_past_32_bits():
    """More than 2^31 elements per tensor: the last tokens, forward and backward, against a call on them alone."""
    from cula_b200.kda import selective_scan
    D, S, tail = 1024, 16, 300
    T = 2 ** 31 // D + 128 + tail
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty(1, T, D, device="cuda", dtype=torch.bfloat16).fill_(0.5)
    x[:, -tail - 200:] = torch.randn(1, tail + 200, D, device="cuda", generator=gen).bfloat16()
    dt = torch.full((1, 1, D), -1.0, device="cuda", dtype=torch.bfloat16).expand(1, T, D)
    bc = torch.randn(1, 1, S, device="cuda", generator=gen).bfloat16().expand(1, T, S)
    A = -torch.rand(D, S, device="cuda", generator=gen) - 0.05
    x.requires_grad_(True)
    y, fin = selective_scan(x, dt, A, bc, bc, dt_softplus=True, output_final_state=True)
    with torch.no_grad():
        _, h = selective_scan(x[:, :-tail], dt[:, :-tail], A, bc[:, :-tail], bc[:, :-tail], dt_softplus=True, output_final_state=True)
    part = x.detach()[:, -tail:].clone().requires_grad_(True)
    y2, fin2 = selective_scan(part, dt[:, -tail:], A, bc[:, -tail:], bc[:, -tail:], dt_softplus=True, initial_state=h, output_final_state=True)
    assert err_ratio(y2.detach().double().cpu(), y.detach()[:, -tail:].double().cpu()) < tol(torch.bfloat16, tail)
    assert err_ratio(fin2.detach().double().cpu(), fin.detach().double().cpu()) < 2 * tol(torch.float32, tail)
    dy2 = torch.randn(y2.shape, device="cuda", generator=gen).bfloat16()
    dy = torch.zeros_like(y)
    dy[:, -tail:] = dy2
    del y2, h
    g, = torch.autograd.grad(y, x, dy)
    g2, = torch.autograd.grad(selective_scan(part, dt[:, -tail:], A, bc[:, -tail:], bc[:, -tail:], dt_softplus=True)[0], part, dy2)
    assert err_ratio(g2.double().cpu(), g[:, -tail:].double().cpu()) < 2 * tol(torch.bfloat16, tail)
    del x, y, dy, g
    torch.cuda.empty_cache()


# ------------------------------------------------------------------ one token ------------------------------------------------------------------
@pytest.mark.gpu
def test_step_in_a_pool_past_32_bits():
    from cula_b200.kda import selective_scan_update
    D, S = 4096, 64
    slots = 2 ** 31 // (D * S) + 3
    pool = torch.empty(slots, D, S, device="cuda")
    small = torch.randn(2, D, S, device="cuda")
    pool[0], pool[slots - 1] = small[0], small[1]
    a = on_gpu({k: v[:, 0] if k in ("x", "dt", "B", "C", "z") else v for k, v in make(2, 1, D, S, seed=3).items()})
    del a["initial_state"]
    y = selective_scan_update(**a, state=pool, state_indices=torch.tensor([0, slots - 1], dtype=torch.int32, device="cuda"))
    assert torch.equal(y, selective_scan_update(**a, state=small)) and torch.equal(pool[0], small[0]) and torch.equal(pool[slots - 1], small[1])
    del pool
    torch.cuda.empty_cache()


@pytest.mark.gpu
def test_steps_in_a_cuda_graph():
    from cula_b200.kda import selective_scan_update
    a = on_gpu({k: v[:, 0] if k in ("x", "dt", "B", "C", "z") else v for k, v in make(40, 1, 256, 16, seed=5).items()})
    del a["initial_state"]
    start = torch.randn(50, 256, 16, device="cuda")
    idx = torch.randperm(50, device="cuda")[:40].to(torch.int32)
    pool, eager = start.clone(), start.clone()
    y0 = selective_scan_update(**a, state=eager, state_indices=idx)
    y1 = selective_scan_update(**a, state=eager, state_indices=idx)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = selective_scan_update(**a, state=pool, state_indices=idx)
    pool.copy_(start)
    for ref in (y0, y1):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ref)
    assert torch.equal(pool, eager)


@pytest.mark.gpu
@pytest.mark.parametrize("N,D,S,G,dtype,gate,indexed", [(1, 8, 1, 1, "bf16", True, False), (3, 40, 16, 1, "fp32", True, True), (5, 264, 12, 1, "bf16", False, True),
                                                        (2, 48, 5, 3, "fp32", True, False), (4, 64, 33, 2, "bf16", True, True), (2, 16, 64, 1, "fp32", True, True),
                                                        (600, 136, 16, 1, "bf16", True, True)])
def test_step_matches_oracle(N, D, S, G, dtype, gate, indexed):
    from cula_b200.kda import check_status, selective_scan_update
    dtype = torch.bfloat16 if dtype == "bf16" else torch.float32
    a = {k: v[:, 0] if k in ("x", "dt", "B", "C", "z") and v is not None else v for k, v in make(N, 1, D, S, G, dtype, gate, seed=N).items()}
    del a["initial_state"]
    gen = torch.Generator().manual_seed(8)
    pool = torch.randn(N + 3, D, S, generator=gen)
    idx = torch.randperm(N + 3, generator=gen)[:N].to(torch.int32) if indexed else None
    if indexed and N > 2:
        idx[1] = -1
    y_ref, pool_ref = selective_scan_update_ref(**in64(a), state=pool.double(), state_indices=idx)
    state = pool.cuda()
    y = selective_scan_update(**on_gpu(a), state=state, state_indices=None if idx is None else idx.cuda())
    torch.cuda.synchronize()
    check_status(torch.device("cuda", 0))
    assert err_ratio(y_ref, y.double().cpu()) < tol(dtype, 1) and err_ratio(pool_ref, state.double().cpu()) < tol(torch.float32, 1)
    touched = torch.zeros(N + 3, dtype=torch.bool)
    touched[(torch.arange(N) if idx is None else idx[idx >= 0]).long()] = True
    assert torch.equal(state.cpu()[~touched], pool[~touched])


@pytest.mark.gpu
def test_step_without_softplus_and_with_parameters_in_16_bits():
    from cula_b200.kda import selective_scan_update
    a = {k: v[:, 0] if k in ("x", "dt", "B", "C", "z") else v for k, v in make(5, 1, 72, 16, 1, torch.float32, seed=6).items()}
    del a["initial_state"]
    a.update(dt_softplus=False, dt=0.05 * a["dt"].abs(), dt_bias=0.01 * torch.rand(72, generator=torch.Generator().manual_seed(1)))
    for k in ("A", "D", "dt_bias"):
        a[k] = a[k].bfloat16()
    pool = torch.randn(5, 72, 16, generator=torch.Generator().manual_seed(2))
    y_ref, pool_ref = selective_scan_update_ref(**in64(a), state=pool.double())
    state = pool.cuda()
    y = selective_scan_update(**on_gpu(a), state=state)
    assert err_ratio(y_ref, y.double().cpu()) < tol(torch.float32, 1) and err_ratio(pool_ref, state.double().cpu()) < tol(torch.float32, 1)


@pytest.mark.gpu
def test_step_with_a_token_axis_views_and_out():
    from cula_b200.kda import selective_scan_update
    a = on_gpu(make(4, 1, 32, 8, seed=1, four_dims=True))
    wide = torch.cat([a["x"], a["dt"], a["z"]], -1)
    pool = torch.randn(4, 32, 8, device="cuda")
    p1, p2 = pool.clone(), pool.clone()
    y1 = selective_scan_update(a["x"], a["dt"], a["A"], a["B"], a["C"], p1, D=a["D"], z=a["z"], dt_bias=a["dt_bias"], dt_softplus=True)
    out = torch.empty(4, 32, device="cuda", dtype=torch.bfloat16)
    y2 = selective_scan_update(wide[:, 0, :32], wide[:, 0, 32:64], a["A"], a["B"][:, 0, 0], a["C"][:, 0, 0], p2, D=a["D"], z=wide[:, 0, 64:],
                               dt_bias=a["dt_bias"], dt_softplus=True, out=out, state_indices=torch.arange(4, device="cuda"))
    assert y1.shape == (4, 1, 32) and y2 is not None and out.data_ptr() == y2.data_ptr()
    assert torch.equal(y1[:, 0], y2) and torch.equal(p1, p2)


@pytest.mark.gpu
def test_step_slot_past_the_pool_is_reported():
    from cula_b200.kda import check_status, selective_scan_update
    a = on_gpu(make(2, 1, 16, 4))
    pool = torch.randn(3, 16, 4, device="cuda")
    before = pool.clone()
    y = selective_scan_update(a["x"], a["dt"], a["A"], a["B"], a["C"], pool, state_indices=torch.tensor([3, 1], dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert (y[0] == 0).all() and torch.equal(pool[[0, 2]], before[[0, 2]]) and not torch.equal(pool[1], before[1])
    with pytest.raises(RuntimeError, match="past the end of the pool"):
        check_status(torch.device("cuda", 0))
    check_status(torch.device("cuda", 0))


@pytest.mark.gpu
def test_step_slots_past_32_bits_name_no_other_slot():
    from cula_b200.kda import check_status, selective_scan_update
    a = on_gpu(make(3, 1, 16, 4))
    pool = torch.randn(3, 16, 4, device="cuda")
    before = pool.clone()
    y = selective_scan_update(a["x"], a["dt"], a["A"], a["B"], a["C"], pool, state_indices=torch.tensor([2 ** 32, 2, 2 - 2 ** 32], device="cuda"))
    torch.cuda.synchronize()
    assert (y[[0, 2]] == 0).all() and torch.equal(pool[:2], before[:2])
    want = before[2:].clone()
    selective_scan_update(a["x"][1:2], a["dt"][1:2], a["A"], a["B"][1:2], a["C"][1:2], want)
    assert torch.equal(pool[2:], want)
    with pytest.raises(RuntimeError, match="past the end of the pool"):
        check_status(torch.device("cuda", 0))


@pytest.mark.gpu
def test_prompt_then_steps_equal_the_whole_sequence():
    from cula_b200.kda import selective_scan, selective_scan_update
    a = on_gpu(make(2, 80, 64, 16, 1, torch.float32, seed=2))
    y, fin = selective_scan(**a, output_final_state=True)
    first = {k: v[:, :70] if k in ("x", "dt", "B", "C", "z") else v for k, v in a.items()}
    _, state = selective_scan(**first, output_final_state=True)
    for t in range(70, 80):
        o = selective_scan_update(a["x"][:, t], a["dt"][:, t], a["A"], a["B"][:, t], a["C"][:, t], state, D=a["D"], z=a["z"][:, t], dt_bias=a["dt_bias"],
                                  dt_softplus=True)
        assert err_ratio(y[:, t].cpu(), o.cpu()) < tol(torch.float32, 80)
    assert err_ratio(fin.cpu(), state.cpu()) < tol(torch.float32, 80)
