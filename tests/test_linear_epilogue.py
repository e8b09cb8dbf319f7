"""mc_sm100_linear_epilogue against the formula in 64 bits.  The bound on each element is the oracle's (accumulation,
activation, one rounding), derived beside it."""
import numpy as np
import pytest

import oracle_np as onp

ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


# ---- CPU: the formula, refusals --------------------------------------------------------------------------------------
def test_formula_known_answers():
    one = np.ones((1, 1))
    for act, want in (("none", -2.0), ("relu", 0.0), ("silu", -2.0 / (1 + np.exp(2.0))), ("gelu", -2.0 * 0.022750131948179),
                      ("gelu_tanh", -0.045402305912)):
        y, e = onp.linear_epilogue_f64(one, -2.0 * one, act=act)
        assert abs(y[0, 0] - want) < 1e-9 and e[0, 0] > 0
    y, _ = onp.linear_epilogue_f64([[1.0], [3.0]], [[2.0]], scale=[1.0, 0.5], bias=[1.0, 1.0], residual=[[10.0]], act="relu", gated=True)
    assert y[0, 0] == 3.0 * 4.0 + 10.0


def test_refusals(pkg):
    call = pkg.launch_linear_epilogue
    ok = dict(stream=16)
    for bad in ((None, 16, 16, 1, 8, 8), (16, None, 16, 1, 8, 8), (16, 16, None, 1, 8, 8), (16, 16, 16, 0, 8, 8), (16, 16, 16, 1, 0, 8),
                (16, 16, 16, 1, 8, 0), (17, 16, 16, 1, 8, 8), (16, 17, 16, 1, 8, 8), (16, 16, 17, 1, 8, 8)):
        w, x, y, M, N, K = bad
        with pytest.raises(pkg.McError) as e:
            call(w, None, x, y, M, N, K, **ok)
        assert e.value.status == pkg.MC_E_INVALID_ARGUMENT and "invalid args" in e.value.message
    for M, N, K in ((2 ** 30 + 1, 8, 8), (1, 2 ** 30 + 1, 8), (1, 8, 2 ** 30 + 8)):
        with pytest.raises(pkg.McError) as e:
            call(16, None, 16, 16, M, N, K, **ok)
        assert e.value.status == pkg.MC_E_INVALID_ARGUMENT
    for kw in (dict(gated=True, N=7), dict(x_stride=7), dict(y_stride=7), dict(residual=32, residual_stride=7), dict(bias=33), dict(residual=33)):
        kw = dict(kw)
        N = kw.pop("N", 8)
        with pytest.raises(pkg.McError) as e:
            call(16, None, 16, 48, 2, N, 8, **kw, **ok)
        assert e.value.status == pkg.MC_E_INVALID_ARGUMENT, kw
    with pytest.raises(pkg.McError) as e:                          # scales of e4m3 weights are fp32
        call(16, 18, 16, 16, 1, 8, 8, **ok)
    assert e.value.status == pkg.MC_E_INVALID_ARGUMENT
    with pytest.raises(pkg.McError) as e:                          # in place needs one stride
        call(16, None, 16, 48, 2, 8, 8, residual=48, residual_stride=8, y_stride=16, **ok)
    assert "one buffer" in e.value.message
    # the struct itself: size, activation, gate, reserved word
    lib, good = pkg.lib(), [88, 1, 8, 8, 0, 0, 0, 0, 0, 0, 16, 0, 16, 16, 0, 0]
    for field, value in ((0, 84), (4, 5), (5, 2), (9, 1)):
        bad = list(good)
        bad[field] = value
        assert lib.mc_sm100_linear_epilogue(pkg.LINEAR_CALL.pack(*bad), None, 0) == pkg.MC_E_INVALID_ARGUMENT
        assert "invalid call struct" in pkg.last_error()
    assert lib.mc_sm100_linear_epilogue(None, None, 0) == pkg.MC_E_INVALID_ARGUMENT
    with pytest.raises(KeyError):
        call(16, None, 16, 16, 1, 8, 8, activation="swish", **ok)


def test_tile_plan(pkg):
    """Host logic: every choice is a plan the kernel has, slices are never empty, big calls take the widest tile whole."""
    for wb in (1, 2):
        assert pkg.debug_tile_plan(wb, 8192, 11520, 2304) == (2, 256, 1)
        assert pkg.debug_tile_plan(wb, 128, 2304, 5760, 148)[2] > 1
        for M in (65, 129, 500, 4000, 1 << 20):
            for N in (1, 63, 2304, 122753):
                for K in (8, 64, 65, 2304, 30000):
                    cg, bn, s = pkg.debug_tile_plan(wb, M, N, K)
                    assert (cg, bn) in ((1, 64), (1, 128), (2, 128), (2, 256)) and s in (1, 2, 4) and s <= -(-K // 64) and bn // s >= (32 if cg == 2 else 16) and cg * s <= 8
        assert pkg.debug_tile_plan(wb, 300, 300, 300, 1)[0] in (1, 2)


def test_plans_that_the_tiled_kernel_does_not_have_are_refused(pkg):
    """The hook takes the plans of the rule; anything else leaves what was set."""
    for plan in ((1, 64, 3), (1, 128, 3), (2, 128, 3), (1, 64, 0), (1, 64, 8), (2, 256, 8), (1, 64, 256), (1, 256, 1), (2, 64, 1), (3, 128, 1), (1, 0, 1),
                 (1, 64 + 65536, 1), (257, 64, 1)):
        with pytest.raises(pkg.McError) as e:
            pkg.debug_set_tile_plan(*plan)
        assert e.value.status == pkg.MC_E_INVALID_ARGUMENT and "no plan" in e.value.message, plan
    for plan in PLANS:
        pkg.debug_set_tile_plan(*plan)
    pkg.debug_set_tile_plan()


def test_tensors_of_other_widths_are_refused(pkg):
    """The binding decides between bf16 and e4m3 by the scales: codes without them, and anything else that is not as wide as what it
    stands for, is refused before the call (nothing is launched: the tensors are the host's)."""
    import torch
    t = lambda dtype, *s: torch.zeros(s, dtype=dtype)  # noqa: E731
    bf, u8, f32, f64 = torch.bfloat16, torch.uint8, torch.float32, torch.float64
    ok = dict(w=t(bf, 8, 16), scale=None, x=t(bf, 1, 16), y=t(bf, 1, 8))
    for bad in (dict(w=t(u8, 8, 16)), dict(w=t(f32, 8, 16)), dict(scale=t(f32, 8)), dict(w=t(u8, 8, 16), scale=t(bf, 8)), dict(w=t(u8, 8, 16), scale=t(f64, 8)),
                dict(x=t(f32, 1, 16)), dict(x=t(u8, 1, 16)), dict(y=t(f32, 1, 8)), dict(y=t(u8, 1, 8)), dict(bias=t(f32, 8)), dict(residual=t(f32, 1, 8))):
        with pytest.raises(pkg.McError) as e:
            pkg.launch_linear_epilogue(**{**ok, **bad}, M=1, N=8, K=16, stream=16)
        assert e.value.status == pkg.MC_E_INVALID_ARGUMENT and "launch_linear_epilogue: " in e.value.message, list(bad)


# ---- GPU -------------------------------------------------------------------------------------------------------------
def _make(M, N, K, e4m3, bias, residual, gated, seed):
    n_out = N // 2 if gated else N
    w = onp.seeded_bf16(seed, (N, K), 0.02 if K > 64 else 0.3)
    q, sc = onp.make_fp8_weight(w) if e4m3 else (None, None)
    x = onp.seeded_bf16(seed + 1, (M, K), 1.0)
    b = onp.seeded_bf16(seed + 2, (N,), 0.5) if bias else None
    r = onp.seeded_bf16(seed + 3, (M, n_out), 1.0) if residual else None
    return w, q, sc, x, b, r


def _wide(a, pad, fill=0x7FC0):
    """Rows of `a` in a wider, poisoned matrix."""
    out = np.full((a.shape[0], a.shape[1] + pad), fill, np.uint16)
    out[:, :a.shape[1]] = a
    return out


def _run(pkg, M, N, K, e4m3=False, bias=False, residual=False, act="none", gated=False, x_pad=0, y_pad=0, r_pad=0, in_place=False,
         offset=0, seed=1, pdl=False):
    import gpu_util as g
    import torch
    w, q, sc, x, b, r = _make(M, N, K, e4m3, bias, residual or in_place, gated, seed)
    n_out = N // 2 if gated else N
    if in_place:
        r_pad = y_pad

    def put(a):
        """`offset` elements behind an aligned address"""
        t = torch.zeros(a.size + offset, dtype=torch.uint8 if a.dtype == np.uint8 else torch.int16, device="cuda")
        t[offset:] = g.dev(a).reshape(-1)
        return t[offset:]
    dx, dw = put(_wide(x, x_pad)), put(q if e4m3 else w)
    dy = g.dev(_wide(r, y_pad)) if in_place else g.empty_u16(M, n_out + y_pad)
    dr = dy if in_place else (g.dev(_wide(r, r_pad)) if residual else None)
    pkg.launch_linear_epilogue(dw, g.dev(sc) if e4m3 else None, dx, dy, M, N, K, bias=g.dev(b) if bias else None, residual=dr,
                               activation=act, gated=gated, x_stride=K + x_pad, y_stride=n_out + y_pad, residual_stride=n_out + r_pad, pdl=pdl)
    g.sync()
    got = g.host_u16(dy).reshape(M, n_out + y_pad)
    assert np.all(got[:, n_out:] == 0x7FC0), "columns between the rows were written"
    f = onp.bf16_to_f32
    want, bound = onp.linear_epilogue_f64(onp.e4m3_to_f32(q) if e4m3 else f(w), f(x), sc, f(b) if bias else None,
                                          f(r) if r is not None else None, act, gated)
    d = np.abs(f(got[:, :n_out]).astype(np.float64) - want)
    assert np.all(d <= bound), (float(np.max(d / bound)), np.argwhere(~(d <= bound))[:4].tolist())
    return got


SHAPES = [(1, 1, 1), (1, 2, 7), (2, 31, 16), (3, 130, 24), (5, 96, 72), (1, 2304, 2304), (1, 257, 5760), (4, 514, 256), (7, 65, 777), (8, 1000, 512),
          (16, 3456, 256), (17, 258, 1040), (33, 300, 2304), (64, 128, 64), (65, 128, 64), (100, 66, 96), (127, 384, 320), (128, 256, 128),
          (129, 514, 136), (200, 1026, 1040), (255, 30, 48), (256, 512, 512), (301, 770, 2304), (513, 258, 72), (1030, 130, 80),
          (70, 1, 64), (2000, 2, 16), (17, 1, 16), (33, 7, 32), (20, 1411, 3600), (24, 5720, 720), (12, 2310, 1600)]


PLANS = [(1, 64, 1), (1, 64, 2), (1, 64, 4), (1, 128, 1), (1, 128, 2), (1, 128, 4), (2, 128, 1), (2, 128, 2), (2, 128, 4), (2, 256, 1), (2, 256, 2), (2, 256, 4)]


@pytest.mark.gpu
@pytest.mark.parametrize("plan", PLANS)
def test_tile_plans(pkg, plan):
    """Every way of cutting a call of more than 64 rows, at sizes around its tiles, and many more tiles than SMs."""
    pkg.debug_set_tile_plan(*plan)
    try:
        for e4m3 in (False, True):
            _run(pkg, 128, 64, 64, e4m3, seed=1)
            assert pkg.debug_take_error() == 0
            _run(pkg, 128, 256, 512, e4m3, seed=2)
            _run(pkg, 65, 30, 1040, e4m3, bias=True, residual=True, act="silu", seed=3)
            _run(pkg, 300, 514, 656, e4m3, bias=True, residual=True, act="gelu", gated=True, seed=4)
            _run(pkg, 300, 515, 656, e4m3, bias=True, residual=True, act="relu", seed=5)
            _run(pkg, 257, 520, 80, e4m3, bias=True, residual=True, y_pad=3, r_pad=1, x_pad=8, seed=6)
            _run(pkg, 2600, 2000, 192, e4m3, bias=True, in_place=True, seed=7)
            _run(pkg, 2600, 2002, 192, e4m3, act="silu", gated=True, in_place=True, y_pad=3, seed=8)
            assert pkg.debug_take_error() == 0
    finally:
        pkg.debug_set_tile_plan()


@pytest.mark.gpu
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_shapes(pkg, shape, e4m3):
    M, N, K = shape
    _run(pkg, M, N, K, e4m3, seed=sum(shape))
    _run(pkg, M, N, K, e4m3, bias=True, residual=True, act="silu", seed=sum(shape) + 7)
    if N % 2 == 0:
        _run(pkg, M, N, K, e4m3, bias=True, residual=True, act="silu", gated=True, seed=sum(shape) + 14)


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M", [1, 6, 20, 140])
def test_activations(pkg, M, act, gated):
    for e4m3 in (False, True):
        _run(pkg, M, 196, 208, e4m3, bias=True, act=act, gated=gated, seed=M)
        _run(pkg, M, 196, 208, e4m3, residual=True, act=act, gated=gated, seed=M + 5)
        if M == 20:
            _run(pkg, 40, 196, 1200, e4m3, bias=True, residual=True, act=act, gated=gated, seed=M + 6)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 3, 12, 70, 300])
def test_strides_in_place_and_alignment(pkg, M):
    for e4m3 in (False, True):
        _run(pkg, M, 132, 80, e4m3, bias=True, residual=True, x_pad=8, y_pad=4, r_pad=2, seed=M)
        _run(pkg, M, 132, 80, e4m3, residual=True, x_pad=3, y_pad=5, r_pad=1, seed=M + 1)     # rows of x not 16-byte aligned
        _run(pkg, M, 131, 80, e4m3, bias=True, in_place=True, seed=M + 2)
        _run(pkg, M, 132, 96, e4m3, act="gelu", gated=True, in_place=True, y_pad=7, seed=M + 3)
        _run(pkg, M, 132, 80, e4m3, bias=True, residual=True, offset=1, seed=M + 4)           # w and x at odd addresses
        _run(pkg, M, 132, 80, e4m3, bias=True, residual=True, seed=M + 5, pdl=True)


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("y_at,r_at", [(1, 1), (1, 0), (0, 1), (3, 2)])
def test_output_and_residual_at_any_address(pkg, y_at, r_at, gated):
    """y and the residual begin anywhere in an allocation, rows even and odd numbers of elements apart: what stands around y stays."""
    import gpu_util as g
    import torch
    for M, N, y_pad, r_pad in ((70, 74, 0, 0), (1, 66, 0, 0), (33, 130, 1, 0), (200, 262, 0, 1), (131, 140, 3, 2)):
        w, _, _, x, b, r = _make(M, N, 80, False, True, True, gated, M + y_at)
        n_out = N // 2 if gated else N
        ly, lr = n_out + y_pad, n_out + r_pad
        y = torch.full((y_at + M * ly + 8,), 0x7FC0, dtype=torch.int16, device="cuda")
        res = torch.zeros(r_at + M * lr, dtype=torch.int16, device="cuda")
        res[r_at:] = g.dev(_wide(r, r_pad)).reshape(-1)
        pkg.launch_linear_epilogue(g.dev(w), None, g.dev(x), y[y_at:], M, N, 80, bias=g.dev(b), residual=res[r_at:], activation="gelu_tanh", gated=gated,
                                   y_stride=ly, residual_stride=lr)
        g.sync()
        flat = g.host_u16(y).reshape(-1)
        got = flat[y_at:y_at + M * ly].reshape(M, ly)
        assert np.all(flat[:y_at] == 0x7FC0) and np.all(flat[y_at + M * ly:] == 0x7FC0) and np.all(got[:, n_out:] == 0x7FC0)
        f = onp.bf16_to_f32
        want, bound = onp.linear_epilogue_f64(f(w), f(x), None, f(b), f(r), "gelu_tanh", gated)
        d = np.abs(f(got[:, :n_out]).astype(np.float64) - want)
        assert np.all(d <= bound), (M, N, float(np.max(d / bound)))


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 9, 64, 200])
def test_a_row_that_is_not_finite_stays_alone(pkg, M):
    import gpu_util as g
    for e4m3 in (False, True):
        w, q, sc, x, _, _ = _make(M, 160, 192, e4m3, False, False, False, M)
        args = (g.dev(q if e4m3 else w), g.dev(sc) if e4m3 else None)
        bad = x.copy()
        bad[M // 2, 5] = 0x7FC0                                                              # NaN
        if M > 8:
            bad[2, 7] = 0x7F80                                                               # +infinity
        ys = []
        for v in (x, bad):
            y = g.empty_u16(M, 160)
            pkg.launch_linear_epilogue(*args, g.dev(v), y, M, 160, 192, activation="relu")
            g.sync()
            ys.append(g.host_u16(y))
        f = [onp.bf16_to_f32(y) for y in ys]
        assert np.all(np.isnan(f[1][M // 2])), "max(NaN, 0) is NaN"
        keep = [m for m in range(M) if m != M // 2 and not (M > 8 and m == 2)]
        assert np.array_equal(ys[0][keep], ys[1][keep])
        if M > 8:
            assert np.all((f[1][2] == 0) | (f[1][2] == np.inf) | np.isnan(f[1][2]))


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 5, 40, 130])
def test_codes_that_are_not_numbers_count_as_480(pkg, M):
    """e4m3 codes 0x7F / 0xFF follow the library's decoder."""
    import gpu_util as g
    N, K = 96, 64
    q = np.full((N, K), 0x38, np.uint8)                            # 1.0
    q[5, 3], q[6, 4] = 0x7F, 0xFF
    x = np.full((M, K), 0x3F80, np.uint16)
    sc, y = np.ones(N, np.float32), g.empty_u16(M, N)
    pkg.launch_linear_epilogue(g.dev(q), g.dev(sc), g.dev(x), y, M, N, K)
    g.sync()
    want = np.full((M, N), 64.0)
    want[:, 5], want[:, 6] = 63.0 + 480.0, 63.0 - 480.0
    got = onp.bf16_to_f32(g.host_u16(y))
    assert np.all(np.abs(got - want) <= 2.0 ** -8 * np.abs(want))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 5760, 2304), (40, 5760, 2304), (700, 1280, 2304)])
def test_same_bits_every_time(pkg, shape):
    a = _run(pkg, *shape, bias=True, residual=True, act="gelu_tanh", seed=3)
    for _ in range(3):
        assert np.array_equal(a, _run(pkg, *shape, bias=True, residual=True, act="gelu_tanh", seed=3))


@pytest.mark.gpu
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("shape", [(2500, 2304, 5760, False), (3001, 11520, 2304, True), (33, 122753, 2304, False), (1, 122753, 2304, False),
                                   (9000, 200, 4096, False), (600, 3456, 2304, False), (150, 11520, 2304, True)])
def test_large(pkg, shape, e4m3):
    """Sizes of real work, the reference product in 64 bits on the GPU."""
    import torch
    M, N, K, gated = shape
    g = torch.Generator(device="cuda")
    g.manual_seed(M + N)
    n_out = N // 2 if gated else N
    w = (torch.randn(N, K, generator=g, device="cuda") * 0.02).bfloat16()
    x, r = torch.randn(M, K, generator=g, device="cuda").bfloat16(), torch.randn(M, n_out, generator=g, device="cuda").bfloat16()
    b = (torch.randn(N, generator=g, device="cuda") * 0.5).bfloat16()
    sc = None
    if e4m3:
        sc = w.float().abs().amax(1) / 448.0
        w = (w.float() / sc[:, None]).to(torch.float8_e4m3fn)
    y = torch.full((M, n_out), float("nan"), dtype=torch.bfloat16, device="cuda")
    pkg.launch_linear_epilogue(w.view(torch.uint8) if e4m3 else w, sc, x, y, M, N, K, bias=b, residual=r, activation="silu" if gated else "none", gated=gated)
    rows = torch.randperm(M, generator=g, device="cuda")[:256]
    wd = w.double() * sc.double()[:, None] if e4m3 else w.double()
    z = x[rows].double() @ wd.T + b.double()
    ez = 2.0 ** -23 * ((K + 3) * (x[rows].double().abs() @ wd.abs().T + b.double().abs()))
    if gated:
        a, u = z[:, 0::2] * torch.sigmoid(z[:, 0::2]), z[:, 1::2]
        ea = 1.13 * ez[:, 0::2] + 2.0 ** -16 * a.abs()
        z, ez = a * u, ea * u.abs() + a.abs() * ez[:, 1::2] + ea * ez[:, 1::2]
    z = z + r[rows].double()
    ez = ez + 2.0 ** -22 * z.abs()
    bound = ez + 2.0 ** -8 * (z.abs() + ez)
    assert bool(((y[rows].double() - z).abs() <= bound).all())
    assert bool(torch.isfinite(y).all())
    # typical error, far below the worst case: one rounding of a random value is off by 2^-9 / sqrt(3) of it on average
    rel = float((y[rows].double() - z).norm() / z.norm())
    assert rel <= 2.0 ** -8, rel


@pytest.mark.gpu
def test_streams_and_graph(pkg):
    """Two calls at once on two streams, and both captured into one graph and replayed with other inputs."""
    import torch
    M, N, K = 200, 640, 512
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    w = [(torch.randn(N, K, generator=g, device="cuda") * 0.05).bfloat16() for _ in range(2)]
    x = [torch.randn(m, K, generator=g, device="cuda").bfloat16() for m in (M, 3)]
    y = [torch.empty(m, N, dtype=torch.bfloat16, device="cuda") for m in (M, 3)]
    ref = [torch.empty_like(t) for t in y]
    for i in range(2):
        pkg.launch_linear_epilogue(w[i], None, x[i], ref[i], x[i].shape[0], N, K, activation="silu")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()

    def both():
        side.wait_stream(torch.cuda.current_stream())
        pkg.launch_linear_epilogue(w[0], None, x[0], y[0], M, N, K, activation="silu")
        with torch.cuda.stream(side):
            pkg.launch_linear_epilogue(w[1], None, x[1], y[1], 3, N, K, activation="silu")
        torch.cuda.current_stream().wait_stream(side)
    both()
    torch.cuda.synchronize()
    assert torch.equal(y[0], ref[0]) and torch.equal(y[1], ref[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    for t in x:
        t.neg_()
    for i in range(2):
        pkg.launch_linear_epilogue(w[i], None, x[i], ref[i], x[i].shape[0], N, K, activation="silu")
        y[i].zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y[0], ref[0]) and torch.equal(y[1], ref[1])


@pytest.mark.gpu
@pytest.mark.parametrize("M", [3, 70])
def test_rows_more_than_2_32_elements_apart(pkg, M):
    """Strides whose last row starts beyond 32-bit element numbers; what lies between the rows stays as it was."""
    import torch
    N, K = 72, 96
    far = (2 ** 32 // (M - 1) // 8 + 3) * 8
    g = torch.Generator(device="cuda")
    g.manual_seed(M)
    w, x, r = ((torch.randn(*s, generator=g, device="cuda") * 0.5).bfloat16() for s in ((N, K), (M, K), (M, N)))
    buf = torch.zeros((M - 1) * far + max(N, K), dtype=torch.bfloat16, device="cuda")
    rows = torch.as_strided(buf, (M, max(N, K)), (far, 1))
    rows[:, :K] = x
    near, y = torch.empty(M, N, dtype=torch.bfloat16, device="cuda"), torch.empty(M, N, dtype=torch.bfloat16, device="cuda")
    pkg.launch_linear_epilogue(w, None, x, near, M, N, K, residual=r, activation="silu")
    pkg.launch_linear_epilogue(w, None, buf, y, M, N, K, residual=r, activation="silu", x_stride=far)
    assert torch.equal(near, y)
    rows[:, :N] = r
    pkg.launch_linear_epilogue(w, None, x, buf, M, N, K, residual=buf, activation="silu", y_stride=far, residual_stride=far)
    assert torch.equal(near, rows[:, :N])
    rows[:, :] = 0
    assert int(torch.count_nonzero(buf)) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 20, 200])
def test_waits_for_the_kernel_before(pkg, M):
    """Weights, activation, bias and residual written by the kernel just before, without pdl: plain stream order."""
    import torch
    N, K = 1200, 1600
    g = torch.Generator(device="cuda")
    g.manual_seed(M)
    src = [(torch.randn(*s, generator=g, device="cuda") * 0.1).bfloat16() for s in ((N, K), (M, K), (N,), (M, N))]
    want = torch.empty(M, N, dtype=torch.bfloat16, device="cuda")
    pkg.launch_linear_epilogue(src[0], None, src[1], want, M, N, K, bias=src[2], residual=src[3])
    dst = [torch.zeros_like(t) for t in src]
    y = torch.empty_like(want)
    big = torch.zeros(1 << 26, device="cuda")
    for _ in range(5):
        for t in dst:
            t.zero_()
        y.zero_()
        torch.cuda.synchronize()
        big.add_(1.0)                                              # the copies queue up behind it
        for d, t in zip(dst, src):
            d.copy_(t)
        pkg.launch_linear_epilogue(dst[0], None, dst[1], y, M, N, K, bias=dst[2], residual=dst[3])
        pkg.launch_linear_epilogue(dst[0], None, dst[1], y, M, N, K, bias=dst[2], residual=dst[3])
        assert torch.equal(y, want)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 12, 40, 300])
def test_waits_for_both_streams_it_joins(pkg, M):
    """x comes from this stream's short kernel, the residual from another stream's long one, joined by an event; eager and replayed."""
    import torch
    N, K, L = 512, 256, 8192
    g = torch.Generator(device="cuda")
    g.manual_seed(M)
    w1, w2 = [(torch.randn(*s, generator=g, device="cuda") * 0.05).bfloat16() for s in ((K, 64), (N, K))]
    wl = (torch.randn(L, 2048, generator=g, device="cuda") * 0.02).bfloat16()
    x0 = torch.randn(M, 64, generator=g, device="cuda").bfloat16()
    xl = torch.randn(1024, 2048, generator=g, device="cuda").bfloat16()
    x1, long, y = [torch.full(s, float("nan"), dtype=torch.bfloat16, device="cuda") for s in ((M, K), (1024, L), (M, N))]
    side = torch.cuda.Stream()

    def run(apart):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side if apart else torch.cuda.current_stream()):
            for _ in range(3):
                pkg.launch_linear_epilogue(wl, None, xl, long, 1024, L, 2048)
        pkg.launch_linear_epilogue(w1, None, x0, x1, M, K, 64, activation="silu")
        torch.cuda.current_stream().wait_stream(side)
        # the last rows that the long kernel writes
        pkg.launch_linear_epilogue(w2, None, x1, y, M, N, K, residual=long[1024 - M:, L - N:], residual_stride=L)
    run(False)
    torch.cuda.synchronize()
    want = y.clone()
    assert torch.isfinite(want.float()).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(True)
    for replay in (False, True, True):
        for t in (x1, long, y):
            t.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay() if replay else run(True)
        torch.cuda.synchronize()
        assert torch.equal(y, want), replay


@pytest.mark.gpu
def test_several_threads(pkg):
    """Four host threads, each with its own stream, shapes and types; every call gives the bits it gives alone."""
    import threading
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    jobs = []
    for M, N, K, e4m3 in ((1, 700, 512, False), (9, 700, 512, True), (40, 1500, 2048, False), (300, 640, 512, True)):
        w = torch.randint(0, 0x70, (N, K), dtype=torch.uint8, generator=g, device="cuda") if e4m3 else torch.randn(N, K, generator=g, device="cuda").bfloat16()
        sc = torch.rand(N, generator=g, device="cuda") if e4m3 else None
        x = torch.randn(M, K, generator=g, device="cuda").bfloat16()
        ys = [torch.empty(M, N, dtype=torch.bfloat16, device="cuda") for _ in range(25)]
        pkg.launch_linear_epilogue(w, sc, x, ys[0], M, N, K, activation="gelu")
        jobs.append((M, N, K, w, sc, x, ys, ys[0].clone(), torch.cuda.Stream()))
    torch.cuda.synchronize()
    errors = []

    def work(M, N, K, w, sc, x, ys, _, stream):
        try:
            with torch.cuda.stream(stream):
                for y in ys:
                    pkg.launch_linear_epilogue(w, sc, x, y, M, N, K, activation="gelu")
        except Exception as e:      # reported by the main thread
            errors.append(e)
    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors
    for j in jobs:
        assert all(torch.equal(y, j[7]) for y in j[6])


@pytest.mark.gpu
@pytest.mark.parametrize("act", ACTS)
def test_activations_over_every_bf16(pkg, act):
    """z runs through every bf16 value: the activation's own error, tails, infinities and NaN included."""
    import gpu_util as g
    bits = np.arange(65536, dtype=np.uint16)
    x = np.zeros((65536, 8), np.uint16)
    x[:, 0] = bits
    w = np.zeros((8, 8), np.uint16)
    w[:, 0] = 0x3F80                                            # 1.0
    y = g.empty_u16(65536, 8)
    pkg.launch_linear_epilogue(g.dev(w), None, g.dev(x), y, 65536, 8, 8, activation=act)
    g.sync()
    z = onp.bf16_to_f32(bits).astype(np.float64)
    got = onp.bf16_to_f32(g.host_u16(y).reshape(65536, 8)).astype(np.float64)
    assert np.array_equal(got, np.repeat(got[:, :1], 8, axis=1), equal_nan=True)
    ok = np.isfinite(z)
    with np.errstate(over="ignore"):
        want, bound = onp.linear_epilogue_f64(np.ones((1, 1)), z[ok][:, None], act=act)
    d = np.abs(got[ok, 0] - want[:, 0])
    assert np.all(d <= bound[:, 0]), (act, z[ok][np.argmax(d / bound[:, 0])], float(np.max(d / bound[:, 0])))
    assert np.isnan(got[np.isnan(z), 0]).all()
    assert got[np.isposinf(z), 0][0] == np.inf


@pytest.mark.gpu
def test_one_row_that_needs_48_kb_is_a_process_s_first_call():
    """The activation alone fits the 48 KB that a launch may take unasked, with the kernel's static shared memory it does not."""
    import subprocess
    import sys
    code = ("import sys; sys.path[:0] = %r\nimport importlib, test_linear_epilogue as t\npkg = importlib.import_module('minicpm5-5080fast_b200')\n"
            "for K, e4m3 in ((24560, False), (12272, True)):\n    for gated in (False, True):\n        t._run(pkg, 1, 8, K, e4m3, gated=gated)") % [p for p in sys.path if p]
    p = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert p.returncode == 0, p.stderr[-2000:]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(4096, 11520, 2304, True, False), (2048, 2304, 5760, False, True), (301, 2304, 2304, False, False), (33, 122753, 2304, False, False)])
def test_same_bits_between_other_calls(pkg, shape):
    """Calls one behind the other without a wait, another call's inputs between them: every output of the first inputs has the same bits."""
    import torch
    M, N, K, gated, e4m3 = shape
    g = torch.Generator(device="cuda")
    g.manual_seed(M)
    n_out = N // 2 if gated else N
    w = torch.randint(0, 0x70, (N, K), dtype=torch.uint8, generator=g, device="cuda") if e4m3 else (torch.randn(N, K, generator=g, device="cuda") * 0.02).bfloat16()
    sc = torch.rand(N, generator=g, device="cuda") * 1e-3 if e4m3 else None
    xs = [torch.randn(M, K, generator=g, device="cuda").bfloat16() for _ in range(2)]
    ys = [torch.full((M, n_out), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(9)]
    for i, y in enumerate(ys):
        pkg.launch_linear_epilogue(w, sc, xs[1 if i % 3 == 1 else 0], y, M, N, K, activation="silu" if gated else "none", gated=gated)
    torch.cuda.synchronize()
    for i, y in enumerate(ys):
        assert torch.equal(y, ys[1 if i % 3 == 1 else 0]), i
    assert bool(torch.isfinite(ys[0]).all()) and not torch.equal(ys[0], ys[1])


def _long_k(pkg, M, K, e4m3):
    """One feature, zeros but for some places around every cut of K: sums of small whole numbers, exact in every order."""
    import gpu_util as g
    import torch
    r = np.random.default_rng(M)
    cuts = np.arange(9, dtype=np.int64) * (K // 8)
    at = np.unique(np.clip(np.concatenate([cuts - 65, cuts - 64, cuts - 1, cuts, cuts + 63, cuts + 64, r.integers(0, K, 40)]), 0, K - 1))
    wv, xv = r.integers(1, 3, at.size), r.integers(-2, 3, (M, at.size))
    w = torch.zeros(K, dtype=torch.uint8 if e4m3 else torch.bfloat16, device="cuda")
    w[g.dev(at)] = g.dev(np.where(wv == 2, 0x40, 0x38).astype(np.uint8)) if e4m3 else g.dev(wv.astype(np.float32)).bfloat16()
    x = torch.zeros((M, K), dtype=torch.bfloat16, device="cuda")
    for m in range(M):
        x[m, g.dev(at)] = g.dev(xv[m].astype(np.float32)).bfloat16()
    sc = torch.ones(1, device="cuda") if e4m3 else None
    y = torch.full((M, 1), float("nan"), dtype=torch.bfloat16, device="cuda")
    begin, end = torch.cuda.Event(True), torch.cuda.Event(True)
    begin.record()
    pkg.launch_linear_epilogue(w, sc, x, y, M, 1, K)
    end.record()
    torch.cuda.synchronize()
    assert pkg.debug_take_error() == 0, "a wait ran out"
    want = xv @ wv
    assert np.abs(want).max() <= 256                                # whole numbers that bf16 holds
    assert y[:, 0].float().tolist() == want.tolist()
    return begin.elapsed_time(end)


@pytest.mark.gpu
@pytest.mark.parametrize("e4m3", [False, True])
def test_the_longest_sums(pkg, e4m3):
    """K = 2^30: a CTA's slice takes longer than the limit of a single wait."""
    for M in (1, 2):
        assert _long_k(pkg, M, 2 ** 30, e4m3) > 200.0


@pytest.mark.gpu
@pytest.mark.parametrize("plan", [(1, 64, 1), (2, 128, 1), (1, 128, 2), (2, 256, 2)])
@pytest.mark.parametrize("e4m3", [False, True])
def test_the_longest_sums_of_a_tile(pkg, plan, e4m3):
    pkg.debug_set_tile_plan(*plan)
    try:
        assert _long_k(pkg, 1, 2 ** 28 * plan[2], e4m3) > 200.0
    finally:
        pkg.debug_set_tile_plan()


# The activation of one row stands in shared memory where 200 KB hold it with the biases and residuals of a CTA's outputs: 102400 bf16
# or, behind e4m3 weights, 51200 are exactly 200 KB.
@pytest.mark.gpu
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("N", [1, 8, 15, 66, 300])
@pytest.mark.parametrize("around", [-32, -16, 0, 16])
def test_one_row_with_the_longest_activations(pkg, N, around, e4m3):
    K = (51200 if e4m3 else 102400) + around
    _run(pkg, 1, N, K, e4m3, seed=N)
    _run(pkg, 1, N, K, e4m3, bias=True, residual=True, act="silu", seed=N + 1)
    if N % 2 == 0:
        _run(pkg, 1, N, K, e4m3, bias=True, residual=True, act="gelu", gated=True, seed=N + 2)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2304, 11520), (500, 30000), (5000, 9216)])
def test_one_row_with_long_activations(pkg, shape):
    for e4m3 in (False, True):
        _run(pkg, 1, *shape, e4m3, bias=True, residual=True, act="relu", seed=3)
        _run(pkg, 1, *shape, e4m3, bias=True, in_place=True, act="silu", gated=True, seed=4)


@pytest.mark.gpu
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("shape", [(40, 10000, 3584), (64, 5000, 5312), (48, 9600, 4112), (33, 5632, 2816)])
def test_three_and_six_slices_of_many_rows(pkg, shape, e4m3):
    """33 to 64 rows, K cut in three (74 to 90 row tiles) or six (38 to 44): the rings that stand beside the larger exchange."""
    _run(pkg, *shape, e4m3, bias=True, residual=True, act="silu", seed=shape[0])
    _run(pkg, *shape, e4m3, bias=True, residual=True, act="gelu", gated=True, seed=shape[0] + 1)
    assert pkg.debug_take_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("act,want", [("none", -np.inf), ("relu", 0.0), ("gelu", np.nan), ("gelu_tanh", np.nan), ("silu", np.nan)])
def test_activations_of_minus_infinity(pkg, act, want):
    """z is -infinity through the bias of every third feature: each kernel gives what the formula's own operations give; its neighbours
    stay finite."""
    import gpu_util as g
    for M, N, K in ((1, 96, 64), (6, 96, 64), (40, 96, 2048), (140, 96, 64), (9, 96, 63)):
        for e4m3 in (False, True):
            w, q, sc, x, b, _ = _make(M, N, K, e4m3, True, False, False, M)
            b = b.copy()
            b[::3] = 0xFF80
            y = g.empty_u16(M, N)
            pkg.launch_linear_epilogue(g.dev(q if e4m3 else w), g.dev(sc) if e4m3 else None, g.dev(x), y, M, N, K, bias=g.dev(b), activation=act)
            g.sync()
            got = onp.bf16_to_f32(g.host_u16(y))
            assert np.array_equal(got[:, ::3], np.full_like(got[:, ::3], want), equal_nan=True), (M, e4m3)
            assert np.isfinite(np.delete(got, np.s_[::3], axis=1)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 40, 12272), (8, 40, 12288), (5, 33, 12272), (9, 40, 5872), (16, 40, 5888), (16, 33, 5872)])
def test_few_rows_around_the_longest_staged_activation(pkg, shape):
    """e4m3, up to 16 rows: the whole activation stands in shared memory up to K = 12280 (from nine rows on 5880)."""
    _run(pkg, *shape, True, bias=True, residual=True, act="silu", seed=shape[0])


def _captured_first():
    """A process's first calls, recorded into a graph and replayed: what a call asks of its kernel once happens under capture."""
    import importlib
    import gpu_util as g
    import torch
    pkg = importlib.import_module("minicpm5-5080fast_b200")
    f, jobs = onp.bf16_to_f32, []
    for M, N, K, e4m3 in ((1, 40, 512, False), (1, 40, 24560, False), (1, 40, 512, True), (5, 40, 512, True), (20, 40, 2048, False), (40, 136, 2048, True),
                          (130, 136, 512, False), (130, 136, 512, True), (3, 40, 77, False)):
        w, q, sc, x, b, r = _make(M, N, K, e4m3, True, True, False, M)
        dev = [g.dev(q if e4m3 else w), g.dev(sc) if e4m3 else None, g.dev(x), g.empty_u16(M, N), g.dev(b), g.dev(r)]
        jobs.append((M, N, K, dev, onp.linear_epilogue_f64(onp.e4m3_to_f32(q) if e4m3 else f(w), f(x), sc, f(b), f(r), "silu")))
    V = 107000
    counts, seen = torch.full((64, V), 9, dtype=torch.int32, device="cuda"), torch.full((64, (V + 31) // 32), -1, dtype=torch.int32, device="cuda")
    tokens = np.random.default_rng(1).integers(0, V, (64, 9)).astype(np.int32)
    d_tokens, d_offsets = g.dev(tokens.reshape(-1)), g.dev(np.arange(65, dtype=np.uint32) * 9)
    lg, out = onp.seeded_bf16(3, (64, V), 2.0), g.empty_u16(64, V)
    cfg = np.zeros((64, 8), np.uint32)
    cfg[:, :3] = np.float32([1.5, 0.5, 0.25]).view(np.uint32)
    cfg[:, 3], cfg[:, 4] = np.arange(64), 0xFFFFFFFF
    d_lg, d_cfg = g.dev(lg), g.dev(cfg)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for M, N, K, (w, sc, x, y, b, r), _ in jobs:
            pkg.launch_linear_epilogue(w, sc, x, y, M, N, K, bias=b, residual=r, activation="silu")
        pkg.token_history(counts, seen, d_tokens, 64, V, offsets=d_offsets, rebuild=True)
        pkg.logits_process(d_lg, out, 64, V, V, V, d_cfg, pkg.logits_tables(V, counts=counts, seen=seen))
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for M, N, K, dev, (want, bound) in jobs:
        assert np.all(np.abs(f(g.host_u16(dev[3])) - want) <= bound), (M, N, K)
    c, s = np.zeros((64, V), np.int32), np.zeros((64, V), bool)
    onp.token_history(c, s, [(i, tokens[i].tolist(), 0) for i in range(64)], True)
    assert np.array_equal(counts.cpu().numpy(), c) and np.array_equal(seen.cpu().numpy().view(np.uint32), onp.pack_bits(s))
    assert np.array_equal(g.host_u16(out), np.stack([onp.logits_process_f32(lg[i], (1.5, 0.5, 0.25), c[i], s[i], None, [], []) for i in range(64)]))


@pytest.mark.gpu
def test_a_process_s_first_calls_are_captured():
    import subprocess
    import sys
    code = "import sys; sys.path[:0] = %r\nimport test_linear_epilogue as t\nt._captured_first()" % [p for p in sys.path if p]
    p = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert p.returncode == 0, p.stderr[-2000:]
