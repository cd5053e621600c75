"""The C entries of a state space block's operators: what they refuse, and that members which a call does not use may hold anything. On
the CPU an accepted call ends with the runtime's error (there is no device, so that nothing is launched), which is above zero."""
import pytest
import torch

from oracle.naive_kda import err_ratio
from oracle.ssm import selective_scan_ref
from tests.block_c import GARBAGE, ConvStepArgs, NormArgs, ScanArgs, StepArgs, call

EINVAL, EALIGN = -1, -2
AT = 0x10000                                                         # aligned; never read, since nothing is launched without a device
cpu_only = pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are made up: only without a device")


def scan(**change):
    """A scan of two sequences of 70 tokens, 16 channels, 4 states, without anything optional."""
    a = dict(x=AT, dt=AT, Bm=AT, Cm=AT, A=AT, y=AT, x_row=16, dt_row=16, b_row=4, c_row=4, x_seq=16 * 70, dt_seq=16 * 70, b_seq=4 * 70, c_seq=4 * 70,
             rows=140, T=70, D=16, S=4, G=1, n_seqs=2, num_chunks=4, states=AT, dy=AT, dx=AT, ddt=AT, dBm=AT, dCm=AT, dA=AT, part_bc=AT, part_A=AT,
             cta_rows=1, vec_bc=1)
    return ScanArgs(**{**a, **change})


def packed(**change):
    return scan(**{**dict(cu_seqlens=AT, chunk_offsets=AT, seq_order=AT, total_tokens=140, x_seq=0, dt_seq=0, b_seq=0, c_seq=0), **change})


def norm(**change):
    a = dict(x=AT, w=AT, y=AT, v=AT, rstd=AT, dy=AT, dx=AT, part_w=AT, dw=AT, R=3, x_row=64, D=64, eps=1e-6)
    return NormArgs(**{**a, **change})


@cpu_only
@pytest.mark.parametrize("entry", ["selective_scan_fwd", "selective_scan_bwd"])
def test_members_that_a_scan_does_not_use_may_hold_anything(entry):
    assert call(entry, scan()) > 0 and call(entry, packed()) > 0
    for members in ("seg_state seg_dt", "z_row z_seq y_pre dz", "part_skip part_bias", "chunk_indices", "chunk_offsets seq_order", "total_tokens"):
        assert call(entry, scan(**{m: GARBAGE for m in members.split()})) > 0, members
    for members in ("chunk_indices", "x_seq dt_seq z_seq b_seq c_seq", "T", "seg_state seg_dt"):
        assert call(entry, packed(**{m: GARBAGE for m in members.split()})) > 0, members
    assert call(entry, packed(seg_chunks=1, seg_state=AT, seg_dt=AT, seq_order=None)) > 0
    # what a call does use is looked at as before
    assert call(entry, scan(seg_chunks=1, seg_state=GARBAGE, seg_dt=AT)) == EALIGN and call(entry, scan(seg_chunks=1)) == EINVAL
    assert call(entry, scan(x_seq=3)) == EALIGN and call(entry, scan(z=AT, z_row=3, y_pre=AT, dz=AT)) == EALIGN
    assert call(entry, scan(z=AT, z_row=16, z_seq=1120, y_pre=GARBAGE, dz=AT)) == EALIGN
    assert call(entry, packed(chunk_offsets=None)) == EINVAL and call(entry, packed(seq_order=None)) == EINVAL
    if entry.endswith("bwd"):
        assert call(entry, scan(dz=GARBAGE, z=AT, z_row=16, z_seq=1120, y_pre=AT)) == EALIGN
        assert call(entry, scan(dskip=AT)) == EINVAL and call(entry, scan(dskip=AT, part_skip=GARBAGE)) == EALIGN
        assert call(entry, scan(skip=AT + 4, dt_bias=AT + 4)) > 0    # read one by one, as in the forward pass


@cpu_only
def test_members_that_a_norm_does_not_use_may_hold_anything():
    for entry, members in (("add_rms_norm_fwd", "r r_out r_row scale v dy dr_out dx dr part_w dw"), ("add_rms_norm_bwd", "dr_out dr r r_out r_row x y scale")):
        assert call(entry, norm(**{m: GARBAGE for m in members.split()})) > 0
    assert call("add_rms_norm_fwd", norm(res=1, r=GARBAGE, r_out=AT, r_row=64)) == EALIGN
    assert call("add_rms_norm_bwd", norm(res=1, dr_out=GARBAGE)) == EALIGN


@cpu_only
def test_sizes_at_which_counts_would_pass_32_bits_are_refused():
    most = 2 ** 30
    for entry in ("selective_scan_fwd", "selective_scan_bwd"):
        seg = dict(seg_state=AT, seg_dt=AT)
        assert call(entry, scan(seg_chunks=2 ** 24, **seg)) > 0      # one segment each; 2^26 chunks of 64 tokens are 0 in 32 bits
        for chunks in (2 ** 24 + 1, 2 ** 25, 2 ** 26, 2 ** 31 - 1):
            assert call(entry, scan(seg_chunks=chunks, **seg)) == EINVAL and call(entry, packed(seg_chunks=chunks, **seg)) == EINVAL
        assert call(entry, scan(T=most + 1, n_seqs=1, rows=most + 1, num_chunks=2 ** 24 + 1)) == EINVAL
        assert call(entry, packed(total_tokens=most + 1, rows=most + 1)) == EINVAL
        assert call(entry, scan(D=2 ** 24 + 8, x_row=2 ** 24 + 8, dt_row=2 ** 24 + 8)) == EINVAL
    step = dict(x=AT, dt=AT, Bm=AT, Cm=AT, A=AT, state=AT, y=AT, indices=AT, status=AT, D=16, S=4, G=1, pool=1, x_row=16, dt_row=16, b_row=4, c_row=4)
    conv = dict(x=AT, w=AT, cache=AT, y=AT, indices=AT, status=AT, D=16, W=4, pool=1, x_row=16)
    for entry, args, kind in (("selective_step", step, StepArgs), ("conv_step", conv, ConvStepArgs)):
        assert call(entry, kind(**args, rows=most)) > 0
        for rows in (most + 1, 2 ** 31 - 1):                         # rows ahead of the last one are numbered too
            assert call(entry, kind(**args, rows=rows)) == EINVAL
        assert call(entry, kind(**{**args, "D": 2 ** 24 + 8}, rows=1)) == EINVAL


def test_kept_states_that_an_int_cannot_count_are_refused():
    from cula_b200 import _native
    floats = _native.lib().cula_kda_selective_scan_state_floats
    assert floats(2 ** 23, 2 ** 20, 16) == 2 ** 30                   # a tile of 1024 per group
    for D, G in ((2 ** 24, 2 ** 21), (2 ** 24, 2 ** 22)):
        assert floats(D, G, 16) == EINVAL


@pytest.mark.gpu
def test_workspaces_that_a_scan_does_not_use_are_not_written():
    """y before the gate is kept with the states only, and shares of dskip and dbias are written where these gradients are asked for."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    rn = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    T, D, S = 20, 16, 4
    x, dt, z, dy, Bm, Cm, A = rn(T, D), rn(T, D).abs(), rn(T, D), rn(T, D), rn(T, S), rn(T, S), -rn(D, S).abs()
    out = {k: torch.empty(T, D, device="cuda") for k in ("y", "dx", "ddt", "dz")}
    bc = {k: torch.empty(T, S, device="cuda") for k in ("dBm", "dCm")}
    spare = torch.full((T, D), 7.0, device="cuda")
    own = dict(states=torch.empty(8 * 1024, device="cuda"), y_pre=torch.empty(T, D, device="cuda"), dA=torch.empty(D, S, device="cuda"),
               part_bc=torch.empty(T * 16, device="cuda"), part_A=torch.empty(D * 8, device="cuda"))
    at = lambda ts: {k: t.data_ptr() for k, t in ts.items()}  # noqa: E731
    base = dict(x=x.data_ptr(), dt=dt.data_ptr(), z=z.data_ptr(), Bm=Bm.data_ptr(), Cm=Cm.data_ptr(), A=A.data_ptr(), x_row=D, dt_row=D, z_row=D, b_row=S, c_row=S,
                rows=T, T=T, D=D, S=S, G=1, n_seqs=1, num_chunks=1, fp32=1, cta_rows=1, dy=dy.data_ptr(), **at(out), **at(bc))
    stream = torch.cuda.current_stream().cuda_stream
    assert call("selective_scan_fwd", ScanArgs(**base, y_pre=spare.data_ptr()), stream) == 0
    assert call("selective_scan_fwd", ScanArgs(**base, **at({k: own[k] for k in ("states", "y_pre")})), stream) == 0
    assert call("selective_scan_bwd", ScanArgs(**base, **at(own), part_skip=spare.data_ptr(), part_bias=spare.data_ptr()), stream) == 0
    torch.cuda.synchronize()
    assert (spare == 7.0).all() and own["dA"].isfinite().all()


def scan_through_c(a, cu, dy, dhT, seg_chunks, cta_rows):
    """Forward and backward of one scan with segments and CTA rows as asked for; everything that is written is NaN before."""
    from cula_b200 import _native
    from cula_b200.utils import VarlenTables
    lib, d = _native.lib(), {k: v.cuda().contiguous() if torch.is_tensor(v) else v for k, v in a.items()}
    (n, T, D), (G, S), dtype = a["x"].shape, a["B"].shape[2:], a["x"].dtype
    SP = next(p for p in (8, 16, 32, 64) if p >= S)
    tab = None if cu is None else VarlenTables(cu.cuda())
    n_seqs, chunks = (n, n * -(-T // 64)) if cu is None else (tab.n_seqs, tab.num_chunks)
    slots = 0 if not seg_chunks else n_seqs * -(-(-(-T // 64)) // seg_chunks) if cu is None else chunks // seg_chunks + n_seqs
    tiles = lib.cula_kda_selective_scan_tiles(D, G, S)
    nan = lambda *s, t=torch.float32: torch.full(s, float("nan"), device="cuda", dtype=t)  # noqa: E731
    out = dict(y=nan(n, T, D, t=dtype), hT=nan(n_seqs, D, S), dx=nan(n, T, D, t=dtype), ddt=nan(n, T, D, t=dtype), dz=nan(n, T, D, t=dtype),
               dBm=nan(n, T, G, S, t=dtype), dCm=nan(n, T, G, S, t=dtype), dA=nan(D, S), dskip=nan(D), dbias=nan(D), dh0=nan(n_seqs, D, S))
    work = dict(states=nan(chunks * 8, lib.cula_kda_selective_scan_state_floats(D, G, S)), y_pre=nan(n, T, D), part_bc=nan(tiles, n * T, G, 2, SP),
                part_A=nan(cta_rows, D, SP), part_skip=nan(cta_rows, D), part_bias=nan(cta_rows, D), seg_state=nan(max(1, slots), D, SP), seg_dt=nan(max(1, slots), D))
    up = dict(dy=dy.cuda(), dhT=dhT.cuda())
    ins = dict(x=d["x"], dt=d["dt"], z=d["z"], Bm=d["B"], Cm=d["C"], A=d["A"], skip=d["D"], dt_bias=d["dt_bias"], h0=d["initial_state"])
    tables = {} if cu is None else {k: getattr(tab, k).contiguous() for k in ("cu_seqlens", "chunk_offsets", "seq_order")}
    args = ScanArgs(**{k: t.data_ptr() for k, t in {**out, **work, **up, **ins, **tables}.items()}, x_row=D, dt_row=D, z_row=D, b_row=G * S, c_row=G * S,
                    x_seq=T * D, dt_seq=T * D, z_seq=T * D, b_seq=T * G * S, c_seq=T * G * S, rows=n * T, T=T, D=D, S=S, G=G, n_seqs=n_seqs, num_chunks=chunks,
                    total_tokens=0 if cu is None else tab.total_tokens, seg_chunks=seg_chunks, cta_rows=cta_rows, softplus=1, fp32=dtype == torch.float32,
                    vec_bc=S % 4 == 0)
    stream = torch.cuda.current_stream().cuda_stream
    assert call("selective_scan_fwd", args, stream) == 0 and call("selective_scan_bwd", args, stream) == 0
    torch.cuda.synchronize()
    return {k: t.cpu() for k, t in out.items()}, slots


@pytest.mark.gpu
@pytest.mark.parametrize("lens,D,S,dtype,seg_chunks,cta_rows", [
    ([70, 0, 130, 5, 0, 200, 64], 272, 5, "bf16", 0, 1), ([70, 0, 130, 5, 0, 200, 64], 272, 5, "fp32", 1, 2),
    ([70, 0, 130, 5, 0, 200, 64], 144, 16, "fp32", 0, 2), ([70, 0, 130, 5, 0, 200, 64], 144, 16, "bf16", 1, 1), (None, 144, 16, "bf16", 2, 3),
    ([70, 0, 130, 5, 0, 200, 64], 80, 32, "bf16", 0, 1), ([70, 0, 130, 5, 0, 200, 64], 80, 32, "fp32", 2, 2), (None, 80, 32, "fp32", 0, 2),
    ([70, 0, 130, 5, 0, 200, 64], 48, 64, "fp32", 0, 2), ([70, 0, 130, 5, 0, 200, 64], 48, 64, "bf16", 1, 2), (None, 48, 64, "fp32", 1, 1)])
def test_ctas_that_walk_several_sequences_or_segments(lens, D, S, dtype, seg_chunks, cta_rows):
    """Two groups of two channel tiles (the second not whole), every gradient: what a CTA hands on from one item to the next, sums over items,
    empty sequences between, segments of every state width. Tolerances as for whole calls (test_selective_scan.py)."""
    from tests.test_selective_scan import in64, make, tol
    dtype = torch.bfloat16 if dtype == "bf16" else torch.float32
    cu = None if lens is None else torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    n, T = (5, 150) if cu is None else (1, int(cu[-1]))
    N = n if cu is None else len(lens)
    a = make(n, T, D, S, 2, dtype, h0=N, seed=S + seg_chunks)
    gen = torch.Generator().manual_seed(3)
    dy, dh = torch.randn(n, T, D, generator=gen).to(dtype), 0.1 * torch.randn(N, D, S, generator=gen)
    got, slots = scan_through_c(a, cu, dy, dh, seg_chunks, cta_rows)
    items = slots if seg_chunks else N
    assert items >= 5 and items > cta_rows                          # the loop over items is entered again
    if seg_chunks:
        assert max(-(-(-(-k // 64)) // seg_chunks) for k in ([T] if lens is None else lens)) >= 2
    r = in64(a, True)
    y, fin = selective_scan_ref(**r, cu_seqlens=cu)
    leaves = dict(dx="x", ddt="dt", dz="z", dBm="B", dCm="C", dA="A", dskip="D", dbias="dt_bias", dh0="initial_state")
    ref = dict(zip(leaves, torch.autograd.grad([y, fin], [r[k] for k in leaves.values()], [dy.double(), dh.double()])), y=y.detach(), hT=fin.detach())
    errors = {k: err_ratio(ref[k], got[k]) / tol(got[k].dtype, T) for k in ref}
    assert all(e < 1 for e in errors.values()), errors
