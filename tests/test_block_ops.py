"""The operators around the selective scan: the residual RMS norm (and its 8-bit output), the short convolution for single tokens, and a
whole state space block of them, against the oracle in 64 bits.

Tolerances, fixed before the first run. One rounding to bf16 is at most 2^-8 of the value (the 4e-3 below), one to e4m3 at most 2^-4 where
it is normal; fp32 arithmetic of a norm has at most about 30 roundings of 2^-24 on the way, and the reciprocal square root 2^-22: 4e-6."""
import pytest
import torch

from oracle.layer_ops import short_conv_ref
from oracle.naive_kda import err_ratio
from oracle.ssm import add_rms_norm_ref, quantize_e4m3_ref, selective_scan_ref, short_conv_update_ref

TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
BF16, FP32 = 2.0 ** -8 + 4e-6, 4e-6


def test_conv_step_oracle_continues_the_convolution():
    gen = torch.Generator().manual_seed(0)
    x, w, b = (torch.randn(*s, generator=gen, dtype=torch.float64) for s in ((2, 9, 8), (8, 4), (8,)))
    y, _ = short_conv_ref(x, w, b)
    _, cache = short_conv_ref(x[:, :6], w, b)
    for t in range(6, 9):
        o, cache = short_conv_update_ref(x[:, t], w, cache.double(), bias=b)
        assert err_ratio(y[:, t], o) < 1e-12


def test_norm_oracle_gradients_against_differences():
    gen = torch.Generator().manual_seed(1)
    x, r = (torch.randn(3, 8, generator=gen, dtype=torch.float64, requires_grad=True) for _ in range(2))
    w = torch.randn(8, generator=gen, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda x, w, r: add_rms_norm_ref(x, w, r), (x, w, r))


def test_refusals():
    from cula_b200.kda import add_rms_norm, add_rms_norm_fp8, short_conv_update
    x, w = torch.zeros(2, 16).bfloat16(), torch.ones(16)
    for call in (add_rms_norm, add_rms_norm_fp8):
        for error, match, args in [(AssertionError, "bfloat16 or float32", (x.half(), w)), (AssertionError, "multiple of 8", (x[:, :12], w[:12])),
                                   (AssertionError, "multiple of 8", (torch.zeros(1, 16392).bfloat16(), torch.ones(16392))),
                                   (AssertionError, "weight must be", (x, w[:8])), (AssertionError, "shape of x", (x, w, x[:1])),
                                   (AssertionError, "in float32 or in the type", (x.float(), w, x)), (AssertionError, "in float32 or in the type", (x, w, x.half())),
                                   (ValueError, "on the device of x", (x, w.to("meta"))), (ValueError, "on the device of x", (x, w, x.to("meta")))]:
            with pytest.raises(error, match=match):
                call(*args)
        if not torch.cuda.is_available():
            with pytest.raises(RuntimeError, match="no CPU fallback"):
                call(x, w)
    with pytest.raises(AssertionError, match="group_size"):
        add_rms_norm_fp8(x, w, group_size=16)
    with pytest.raises(AssertionError, match="multiple of group_size"):
        add_rms_norm_fp8(x, w, group_size=32)
    cw, cache = torch.zeros(16, 4), torch.zeros(2, 16, 4)
    for error, match, args in [(AssertionError, "bfloat16", (x.float(), cw, cache)), (AssertionError, r"\[N, D\]", (torch.zeros(2, 2, 16).bfloat16(), cw, cache)),
                               (AssertionError, "W <= 4", (x, torch.zeros(16, 5), cache)), (AssertionError, "multiple of 8", (x[:, :12], cw[:12], cache)),
                               (ValueError, "cache must be", (x, cw, cache[:, :8])), (AssertionError, "contiguous float32", (x, cw, cache.bfloat16())),
                               (AssertionError, "contiguous float32", (x, cw, torch.zeros(2, 4, 16).transpose(1, 2))),
                               (ValueError, "aligned", (x, cw, torch.zeros(2 * 16 * 4 + 1)[1:].view(2, 16, 4))),
                               (ValueError, "holds 1 states", (x, cw, cache[:1])), (ValueError, "on the device of x", (x, cw.to("meta"), cache)),
                               (ValueError, "on the device of x", (x, cw, cache.to("meta"))),
                               (ValueError, "one int32 slot", (x, cw, cache, torch.zeros(1, dtype=torch.int32))),
                               (AssertionError, "bias must be", (x, cw, cache, None, torch.zeros(8)))]:
        with pytest.raises(error, match=match):
            short_conv_update(*args)
    with pytest.raises(AssertionError, match="activation"):
        short_conv_update(x, cw, cache, activation="relu")
    with pytest.raises(ValueError, match="out must be"):
        short_conv_update(x, cw, cache, out=torch.zeros(2, 16))
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            short_conv_update(x, cw, cache)


def test_tangents_are_refused_not_dropped():
    """The operators without gradients have no forward derivatives either."""
    import torch.autograd.forward_ad as fw

    from cula_b200.kda import add_rms_norm_fp8, selective_scan_update, short_conv_update
    x, A, bc, one = torch.ones(2, 16).bfloat16(), -torch.ones(16, 4), torch.ones(2, 4).bfloat16(), torch.ones(16)
    calls = [(selective_scan_update, dict(x=x, dt=x, A=A, B=bc, C=bc, state=torch.zeros(2, 16, 4), D=one, z=x, dt_bias=one)),
             (short_conv_update, dict(x=x, weight=torch.ones(16, 4), cache=torch.zeros(2, 16, 4), bias=one)),
             (add_rms_norm_fp8, dict(x=x, weight=one, residual=x))]
    for call, args in calls:
        for name in args:
            with fw.dual_level(), pytest.raises(RuntimeError, match="no forward derivative"):
                call(**{**args, name: fw.make_dual(args[name], torch.ones_like(args[name]))})


# ------------------------------------------------ residual RMS norm ------------------------------------------------
NORMS = [(1, 8, "bf16", "bf16"), (5, 64, "fp32", "fp32"), (3, 264, "bf16", "fp32"), (33, 520, "bf16", "none"), (7, 1000, "fp32", "none"), (333, 1024, "bf16", "bf16"),
         (2, 1032, "bf16", "bf16"), (400, 2056, "bf16", "fp32"), (5, 4096, "bf16", "bf16"), (310, 4096, "fp32", "fp32"), (9, 4104, "bf16", "none"), (6, 8192, "fp32", "fp32"),
         (3, 16384, "bf16", "fp32"), (2, 12288, "fp32", "none"),
         (35, 128, "bf16", "bf16"), (40, 72, "fp32", "fp32"), (33, 136, "bf16", "none"), (9, 512, "bf16", "fp32"), (11, 768, "fp32", "fp32"), (400, 2560, "bf16", "bf16"),
         (5, 2568, "fp32", "none"), (301, 5120, "bf16", "fp32"), (4, 6144, "bf16", "none"), (300, 8192, "bf16", "bf16"), (301, 8200, "bf16", "bf16")]


def norm_inputs(R, D, dtype, res, seed=0):
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    return rn(R, D).to(TYPES[dtype]), 1 + 0.1 * rn(D), None if res == "none" else (3 * rn(R, D)).to(TYPES[res])


@pytest.mark.gpu
@pytest.mark.parametrize("R,D,dtype,res", NORMS)
def test_norm_matches_oracle(R, D, dtype, res):
    from cula_b200.kda import add_rms_norm
    x, w, r = norm_inputs(R, D, dtype, res)
    ref = [t.double().requires_grad_(True) for t in (x, w, r) if t is not None]
    y_ref, v_ref = add_rms_norm_ref(*ref, eps=1e-5, stream=None if r is None else r.dtype)
    dev = [t.cuda().requires_grad_(True) for t in (x, w, r) if t is not None]
    y, v = add_rms_norm(*dev, eps=1e-5)
    gen = torch.Generator().manual_seed(5)
    dy, dv = torch.randn(R, D, generator=gen).to(x.dtype), torch.randn(R, D, generator=gen).to(x.dtype if r is None else r.dtype)
    got = torch.autograd.grad([y, v], dev, [dy.cuda(), dv.cuda()])
    want = torch.autograd.grad([y_ref, v_ref], ref, [dy.double(), dv.double()])
    torch.cuda.synchronize()
    bound = {torch.bfloat16: BF16, torch.float32: FP32}
    assert y.dtype == x.dtype and err_ratio(y_ref.detach(), y.detach().double().cpu()) < bound[y.dtype]
    if r is not None:
        assert torch.equal(v.cpu(), (x.float() + r.float()).to(r.dtype))
    else:
        assert v is dev[0]
    for g, h, t in zip(got, want, (x, w, r)):
        # without a residual stream the gradient of x is the sum of two that were rounded apart
        assert g.dtype == t.dtype and err_ratio(h, g.double().cpu()) < (2 if r is None else 1) * bound[t.dtype]
    for g, h in zip(got, torch.autograd.grad(add_rms_norm(*dev, eps=1e-5), dev, [dy.cuda(), dv.cuda()])):
        assert torch.equal(g, h)
    with torch.no_grad():
        assert torch.equal(add_rms_norm(*dev, eps=1e-5)[0], y)


@pytest.mark.gpu
def test_norm_with_one_gradient_only_and_views():
    from cula_b200.kda import add_rms_norm
    x, w, r = norm_inputs(40, 96, "bf16", "fp32")
    ref = [t.double().requires_grad_(True) for t in (x, w, r)]
    dev = [t.cuda().requires_grad_(True) for t in (x, w, r)]
    outs, outs_ref = add_rms_norm(*dev), add_rms_norm_ref(*ref, stream=r.dtype)
    for o, o_ref in zip(outs, outs_ref):
        got = torch.autograd.grad(o.float().square().sum(), dev, retain_graph=True, allow_unused=True)
        want = torch.autograd.grad(o_ref.square().sum(), ref, retain_graph=True, allow_unused=True)
        for g, h in zip(got, want):
            if h is not None:
                assert err_ratio(h, g.double().cpu()) < 3 * BF16       # the upstream gradient is rounded too
    # a part of wider rows, a misaligned view, a shape of three dimensions
    wide = torch.randn(40, 200, device="cuda").bfloat16()
    flat = torch.randn(40 * 96 + 1, device="cuda").bfloat16()
    for v in (wide[:, 8:104], wide[:, 3:99], flat[1:].view(40, 96), wide[:, :96].unflatten(0, (4, 10)), wide[:, :96].unflatten(0, (4, 10)).transpose(0, 1)):
        y, s = add_rms_norm(v, dev[1], dev[2].view(v.shape))
        y2, s2 = add_rms_norm(v.clone(memory_format=torch.contiguous_format), dev[1], dev[2].view(v.shape))
        assert y.shape == v.shape and torch.equal(y, y2) and torch.equal(s, s2)
    assert add_rms_norm(wide[:0, :96], dev[1], dev[2][:0])[0].shape == (0, 96)


@pytest.mark.gpu
def test_norm_gradients_of_no_rows_and_not_differentiated_again():
    from cula_b200.kda import add_rms_norm
    x, w, r = (t.cuda().requires_grad_(True) for t in norm_inputs(5, 96, "bf16", "fp32"))
    y, v = add_rms_norm(x[:0], w, r[:0])
    for leaf, g in zip((x, w, r), torch.autograd.grad([y.sum(), v.sum()], [x, w, r])):
        assert g.dtype == leaf.dtype and torch.equal(g, torch.zeros_like(leaf))
    y, v = add_rms_norm(x, w, r)
    gx, gw = torch.autograd.grad(y.float().square().sum(), [x, w], create_graph=True)
    for g in (gx, gw):
        with pytest.raises(RuntimeError, match="cannot be differentiated again"):
            torch.autograd.grad(g.sum(), x)


@pytest.mark.gpu
@pytest.mark.parametrize("R,D,dtype,res,group", [(*n, g) for n in NORMS for g in (None, 32, 128, 256) if g is None or n[1] % g == 0])
def test_norm_in_8_bits(R, D, dtype, res, group):
    from cula_b200.kda import add_rms_norm_fp8
    x, w, r = norm_inputs(R, D, dtype, res, seed=2)
    y_ref, v_ref = add_rms_norm_ref(x.double(), w.double(), None if r is None else r.double(), eps=1e-5, stream=None if r is None else r.dtype)
    q_ref, s_ref = quantize_e4m3_ref(y_ref, group)
    q, s, v = add_rms_norm_fp8(x.cuda(), w.cuda(), None if r is None else r.cuda(), eps=1e-5, group_size=group)
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape and s.shape == s_ref.shape and torch.equal(v.cpu().double(), v_ref)
    assert err_ratio(s_ref, s.double().cpu()) < FP32
    # every value within half a step of e4m3 (relative 2^-4, absolute 2^-10 below its normal range), and hardly one beside the nearest
    size = group or D
    back = q.float().cpu().double().unflatten(-1, (-1, size)) * s.cpu().double().reshape(R, -1, 1)
    err, lim = (back.flatten(-2) - y_ref).abs(), 2.0 ** -4 * y_ref.abs() + (2.0 ** -10 * s_ref.reshape(R, -1, 1)).expand(R, -1, size).flatten(-2)
    assert (err <= lim * 1.0001).all()
    assert (q.float().cpu().double() != q_ref).double().mean() < 1e-3


@pytest.mark.gpu
@pytest.mark.parametrize("D", [128, 4096])
def test_norm_in_8_bits_of_zeros_infinities_and_nan(D):
    from cula_b200.kda import add_rms_norm_fp8
    x = torch.randn(5, D, device="cuda").bfloat16()
    x[0] = 0
    x[1, 3] = float("nan")
    x[2, 5] = float("inf")
    x[3] = 1e-30
    w = torch.ones(D, device="cuda")
    for group in (None, 128):
        q, s, _ = add_rms_norm_fp8(x, w, group_size=group)
        q, s = q.float(), s.reshape(5, -1)
        assert (q[0] == 0).all() and (s[0] == 2.0 ** -126).all()
        assert q[1].isnan().all() and s[1].isnan().all()
        assert q[2, 5].isnan() and (s[2].isnan() if group is None else s[2, :1].isnan()).all()
        assert q[3].isfinite().all() and q[4].isfinite().all() and s[3:].isfinite().all()


@pytest.mark.gpu
def test_norm_past_32_bits_and_in_a_cuda_graph_on_another_stream():
    from cula_b200.kda import add_rms_norm, add_rms_norm_fp8
    D = 8192
    R = 2 ** 31 // D + 3
    x = torch.empty(R, D, device="cuda", dtype=torch.bfloat16).fill_(1.0)
    x[-2:] = torch.randn(2, D, device="cuda").bfloat16()
    w = torch.ones(D, device="cuda", requires_grad=True)
    y, _ = add_rms_norm(x, w, x)
    y2, _ = add_rms_norm(x[-2:], w, x[-2:])
    assert torch.equal(y[-2:], y2)
    q, s, _ = add_rms_norm_fp8(x, w, x, group_size=128)
    q2, s2, _ = add_rms_norm_fp8(x[-2:], w, x[-2:], group_size=128)
    assert torch.equal(q[-2:].float(), q2.float()) and torch.equal(s[-2:], s2)
    dy = torch.zeros_like(y)
    dy[-2:] = 1.0
    g, = torch.autograd.grad(y, w, dy)
    g2, = torch.autograd.grad(y2, w, dy[-2:])
    assert err_ratio(g2.double().cpu(), g.double().cpu()) < FP32
    del x, y, q, s, dy
    torch.cuda.empty_cache()
    x, r = torch.randn(70, 264, device="cuda").bfloat16().requires_grad_(True), torch.randn(70, 264, device="cuda", requires_grad=True)
    w = torch.rand(264, device="cuda", requires_grad=True)

    def step():
        y, v = add_rms_norm(x, w, r)
        return [y.detach(), v.detach(), *torch.autograd.grad([y, v], [x, w, r], [torch.ones_like(y), torch.ones_like(v)])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = [t.clone() for t in step()]
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    graph.replay()
    torch.cuda.synchronize()
    for t, u in zip(static, eager):
        assert torch.equal(t, u)


@pytest.mark.gpu
def test_capture_beside_a_living_eager_graph_is_refused():
    """The engine would end the process; the operators' backward passes say what is wrong instead, and the capture works afterwards."""
    from cula_b200.kda import add_rms_norm, selective_scan
    x = torch.randn(1, 40, 64, device="cuda").bfloat16().requires_grad_(True)
    w, A = torch.rand(64, device="cuda", requires_grad=True), -torch.rand(64, 8, device="cuda") - 0.1
    bc = torch.randn(1, 40, 8, device="cuda").bfloat16()
    for call in (lambda: add_rms_norm(x, w)[0], lambda: selective_scan(x, x, A, bc, bc, dt_softplus=True)[0]):
        def step(call=call):
            y = call()
            return torch.autograd.grad(y, x, torch.ones_like(y))[0]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = step().clone()
        side.synchronize()
        alive = call()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="earlier graph of the same leaves"):
            with torch.cuda.graph(graph):
                step()
        torch.cuda.synchronize()
        del alive, graph
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            static = step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(static, eager)


# More rows than the blocks hold at once (148 SMs): blocks of 512, 256 and 128 threads walk several rows, or several groups of narrow rows, the last
# of them not whole. Every row is compared.
LOOPS = [(1500, 4096, "bf16", "none"), (1501, 4096, "bf16", "fp32"), (1300, 8192, "bf16", "bf16"), (1201, 8192, "bf16", "fp32"), (700, 12288, "bf16", "fp32"),
         (40003, 64, "bf16", "fp32"), (20009, 128, "bf16", "bf16"), (6001, 520, "fp32", "fp32"), (3001, 2560, "bf16", "none")]


@pytest.mark.gpu
@pytest.mark.parametrize("R,D,dtype,res", LOOPS)
def test_norm_of_more_rows_than_blocks(R, D, dtype, res):
    test_norm_matches_oracle(R, D, dtype, res)


@pytest.mark.gpu
@pytest.mark.parametrize("R,D,dtype,res,group", [(*n, g) for n in LOOPS for g in (None, 64) if g is None or n[1] % g == 0])
def test_norm_in_8_bits_of_more_rows_than_blocks(R, D, dtype, res, group):
    test_norm_in_8_bits(R, D, dtype, res, group)


@pytest.mark.gpu
def test_norm_and_conv_step_with_parameters_in_16_bits():
    """The same results as with the parameters' values in 32 bits, and gradients in 16."""
    from cula_b200.kda import add_rms_norm, add_rms_norm_fp8, short_conv_update
    gen = torch.Generator().manual_seed(12)
    x, r = torch.randn(20, 264, generator=gen).bfloat16().cuda(), torch.randn(20, 264, generator=gen).cuda()
    w16 = (1 + 0.1 * torch.randn(264, generator=gen)).bfloat16().cuda().requires_grad_(True)
    w32 = w16.detach().float().requires_grad_(True)
    (y, v), (y2, v2) = add_rms_norm(x, w16, r), add_rms_norm(x, w32, r)
    g, g2 = torch.autograd.grad(y, w16, torch.ones_like(y))[0], torch.autograd.grad(y2, w32, torch.ones_like(y))[0]
    assert torch.equal(y, y2) and torch.equal(v, v2) and g.dtype == torch.bfloat16 and torch.equal(g, g2.bfloat16())
    for a, b in zip(add_rms_norm_fp8(x, w16, r), add_rms_norm_fp8(x, w32, r)):
        assert torch.equal(a.float(), b.float())
    cw, b = torch.randn(264, 4, generator=gen).bfloat16().cuda(), torch.randn(264, generator=gen).bfloat16().cuda()
    pools = [torch.randn(20, 264, 4, generator=gen).cuda()] * 2
    pools = [p.clone() for p in pools]
    assert torch.equal(short_conv_update(x, cw, pools[0], bias=b), short_conv_update(x, cw.float(), pools[1], bias=b.float())) and torch.equal(*pools)


# ------------------------------------------------ short convolution, single tokens ------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("N,D,W", [(256, 12288, 4), (255, 12288, 3), (131, 8200, 2)])
def test_conv_step_of_more_rows_than_blocks(N, D, W):
    """Blocks walk five rows or more each; skipped sequences among the first, middle and last of them."""
    from cula_b200.kda import check_status, short_conv_update
    gen = torch.Generator().manual_seed(N)
    rn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    x, w, b, pool = rn(N, D).bfloat16(), 0.5 * rn(D, W), 0.1 * rn(D), rn(N + 2, D, W)
    idx = torch.randperm(N + 2, generator=gen)[:N].to(torch.int32)
    idx[[0, 7, N // 2, N // 2 + 1, N - 1]] = -1
    y_ref, pool_ref = short_conv_update_ref(x.double(), w.double(), pool.double(), idx, b.double())
    cache = pool.cuda()
    y = short_conv_update(x.cuda(), w.cuda(), cache, idx.cuda(), b.cuda())
    torch.cuda.synchronize()
    check_status(torch.device("cuda", 0))
    assert torch.equal(cache.cpu().double(), pool_ref) and (y.cpu()[idx < 0] == 0).all()
    assert err_ratio(y_ref, y.double().cpu()) < BF16


@pytest.mark.gpu
def test_conv_step_in_a_pool_past_32_bits():
    from cula_b200.kda import short_conv_update
    D = 12288
    slots = 2 ** 31 // (D * 4) + 3
    pool = torch.empty(slots, D, 4, device="cuda")
    small = torch.randn(2, D, 4, device="cuda")
    pool[0], pool[slots - 1] = small[0], small[1]
    x, w = torch.randn(2, D, device="cuda").bfloat16(), torch.randn(D, 4, device="cuda")
    y = short_conv_update(x, w, pool, torch.tensor([0, slots - 1], dtype=torch.int32, device="cuda"))
    assert torch.equal(y, short_conv_update(x, w, small)) and torch.equal(pool[0], small[0]) and torch.equal(pool[slots - 1], small[1])
    del pool
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("N,D,W,bias,act,indexed", [(1, 8, 4, True, "silu", False), (3, 264, 3, False, "silu", True), (33, 1032, 4, True, None, True),
                                                    (5, 520, 2, True, "swish", True), (2, 16, 1, False, "silu", False), (700, 512, 4, True, "silu", True)])
def test_conv_step_matches_oracle(N, D, W, bias, act, indexed):
    from cula_b200.kda import check_status, short_conv_update
    gen = torch.Generator().manual_seed(N)
    rn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    x, w, b, pool = rn(N, D).bfloat16(), 0.5 * rn(D, W), 0.1 * rn(D) if bias else None, rn(N + 2, D, W)
    idx = torch.randperm(N + 2, generator=gen)[:N].to(torch.int32) if indexed else None
    if indexed:
        idx[N // 2] = -1
    y_ref, pool_ref = short_conv_update_ref(x.double(), w.double(), pool.double(), idx, None if b is None else b.double(), act)
    cache = pool.cuda()
    y = short_conv_update(x.cuda(), w.cuda()[:, None], cache, None if idx is None else idx.cuda(), None if b is None else b.cuda(), act)
    torch.cuda.synchronize()
    check_status(torch.device("cuda", 0))
    assert torch.equal(cache.cpu().double(), pool_ref)
    assert N == 1 or (y[N // 2] == 0).all() or not indexed
    assert err_ratio(y_ref, y.double().cpu()) < BF16


@pytest.mark.gpu
def test_conv_step_continues_a_prompt_bit_for_bit():
    from cula_b200.kda import check_status, short_conv, short_conv_update
    gen = torch.Generator().manual_seed(2)
    x, w, b = torch.randn(3, 20, 64, generator=gen).bfloat16().cuda(), torch.randn(64, 4, generator=gen).cuda(), torch.randn(64, generator=gen).cuda()
    y, end = short_conv(x, w, b, output_final_state=True)
    _, cache = short_conv(x[:, :15].contiguous(), w, b, output_final_state=True)
    for t in range(15, 20):
        o = short_conv_update(x[:, t:t + 1], w, cache, bias=b)
        assert o.shape == (3, 1, 64) and (o[:, 0].float() - y[:, t].float()).abs().max() <= 2.0 ** -7 * y[:, t].float().abs().max()
    assert torch.equal(cache, end)
    # a slot past the pool
    before = cache.clone()
    o = short_conv_update(x[:, 0], w, cache, torch.tensor([-1, 7, 2], dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert (o[:2] == 0).all() and torch.equal(cache[:2], before[:2]) and not torch.equal(cache[2], before[2])
    with pytest.raises(RuntimeError, match="past the end of the pool"):
        check_status(torch.device("cuda", 0))


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["state", "out"])
def test_what_a_step_changes_in_place_is_not_taken_for_unchanged(which):
    """A graph that has kept a pool, or the place of an output, for its backward pass says so when a step has written to it since."""
    from cula_b200.kda import selective_scan_update, short_conv_update
    x, A, bc = torch.ones(2, 16, device="cuda").bfloat16(), -torch.ones(16, 4, device="cuda"), torch.ones(2, 4, device="cuda").bfloat16()
    for step in (lambda pool, out: selective_scan_update(x, x, A, bc, bc, pool, out=out), lambda pool, out: short_conv_update(x, -A, pool, out=out)):
        pool, out = (torch.ones(2, 16, 4, device="cuda", requires_grad=True) * 2), (torch.ones(2, 16, device="cuda").bfloat16().requires_grad_(True) * 2)
        loss = (pool if which == "state" else out).square().sum()
        step(pool.detach() if which == "out" else pool, out if which == "out" else None)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    with torch.inference_mode():
        pool = torch.ones(2, 16, 4, device="cuda")
    step(pool, None)                                                 # has no version: nothing to tell, nothing refused
    torch.cuda.synchronize()


# ------------------------------------------------ a whole block ------------------------------------------------
def block(p, x, res, ops):
    """norm -> input projection -> convolution -> projections to step, B and C -> scan, gated -> output projection; returns (out, stream)."""
    h, res = ops["norm"](x, p["nw"], res)
    u, z = (h @ p["w_in"].to(h.dtype)).chunk(2, -1)
    u = ops["conv"](u, p["cw"], p["cb"])
    dt, B, C = (u @ p["w_x"].to(h.dtype)).split([p["R"], p["S"], p["S"]], -1)
    y = ops["scan"](u, dt @ p["w_dt"].to(h.dtype), -torch.exp(p["A_log"]), B, C, p["D"], z, p["dt_bias"])
    return y @ p["w_out"].to(h.dtype), res


def block_params(gen, M=64, D=128, S=16, R=8):
    rn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    step = torch.exp(-6.9 + 4.6 * torch.rand(D, generator=gen))
    return dict(nw=1 + 0.1 * rn(M), w_in=rn(M, 2 * D) / 8, cw=0.3 * rn(D, 4), cb=0.1 * rn(D), w_x=rn(D, R + 2 * S) / 11, w_dt=rn(R, D) / 3,
                A_log=torch.log(torch.arange(1, S + 1.0)).repeat(D, 1), D=torch.ones(D), dt_bias=torch.log(torch.expm1(step)), w_out=rn(D, M) / 11, R=R, S=S)


@pytest.mark.gpu
def test_a_block_trains_and_decodes():
    """Forward and every gradient of a block against the oracle's composition in 64 bits, then the prompt's last tokens as single steps."""
    from cula_b200.kda import add_rms_norm, selective_scan, selective_scan_update, short_conv, short_conv_update
    gen = torch.Generator().manual_seed(11)
    p = block_params(gen)
    x, res = torch.randn(2, 90, 64, generator=gen).bfloat16(), torch.randn(2, 90, 64, generator=gen)
    kept = {}

    def conv(u, w, b, state=None):
        y, kept["conv"] = short_conv(u, w, b, output_final_state=True)
        return y

    def scan(u, dt, A, B, C, D, z, bias):
        y, kept["scan"] = selective_scan(u, dt, A, B, C, D=D, z=z, dt_bias=bias, dt_softplus=True, output_final_state=True)
        return y

    whole = dict(norm=add_rms_norm, conv=conv, scan=scan)
    ref = dict(norm=add_rms_norm_ref, conv=lambda u, w, b: short_conv_ref(u, w, b)[0],
               scan=lambda u, dt, A, B, C, D, z, bias: selective_scan_ref(u, dt, A, B, C, D, z, bias, True)[0])
    names = [k for k, v in p.items() if torch.is_tensor(v)]
    d = {k: v.cuda().requires_grad_(True) if torch.is_tensor(v) else v for k, v in p.items()}
    r = {k: v.double().requires_grad_(True) if torch.is_tensor(v) else v for k, v in p.items()}
    out, stream = block(d, x.cuda(), res.cuda(), whole)
    out_ref, stream_ref = block(r, x.double(), res.double(), ref)
    # six roundings to bf16 on the way (and as many of the weights), each at most 2^-8 and independent: sqrt(12) of them, doubled for products
    bound = 2 * 12 ** 0.5 * 2.0 ** -8
    assert err_ratio(out_ref.detach(), out.detach().double().cpu()) < bound and err_ratio(stream_ref, stream.double().cpu()) < 1e-6
    up = torch.randn(2, 90, 64, generator=gen).bfloat16()
    got = torch.autograd.grad(out, [d[k] for k in names], up.cuda())
    want = torch.autograd.grad(out_ref, [r[k] for k in names], up.double())
    for k, g, h in zip(names, got, want):
        assert err_ratio(h, g.double().cpu()) < 2 * bound, k             # the way there and back

    with torch.no_grad():
        x, res = x.cuda(), res.cuda()
        full, _ = block(d, x, res, whole)
        block(d, x[:, :80], res[:, :80], whole)
        windows, states = kept["conv"], kept["scan"]
        step = dict(norm=add_rms_norm, conv=lambda u, w, b: short_conv_update(u, w, windows, bias=b),
                    scan=lambda u, dt, A, B, C, D, z, bias: selective_scan_update(u, dt, A, B, C, states, D=D, z=z, dt_bias=bias, dt_softplus=True))
        for t in range(80, 90):
            o, _ = block(d, x[:, t], res[:, t], step)
            assert err_ratio(full[:, t].double().cpu(), o.double().cpu()) < bound
    torch.cuda.synchronize()
