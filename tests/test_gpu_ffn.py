"""gemm_bias_act_residual, gated_gemm and their backward passes against 64 bits, and what a program does with them."""
import pytest
import torch

import ffn_reference as R

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def rnd(*shape, seed, scale=1.0, dtype=BF):
    """A tensor between poisoned bands (256 bytes on either side keep a fresh allocation's alignment)."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    n = 1
    for d in shape:
        n *= d
    buf = torch.full((n + 256,), float("nan"), device="cuda", dtype=dtype)
    v = buf[128:128 + n].view(*shape)
    v.copy_(torch.randn(shape, device="cuda", generator=g) * scale)
    return v


def ints(*shape, seed, lo=-2, hi=3):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randint(lo, hi, shape, device="cuda", generator=g).to(BF)


@pytest.fixture(params=[(0, 0), (1, 0), (2, 0), (3, 0), (4, 1), (4, 2), (4, 8)],
                ids=["chosen", "512x256", "256x256", "128x128", "cluster1", "cluster2", "cluster8"])
def tile(request, tcab_lib):
    """Every kernel whatever the size: the tile shapes of the persistent one, and the one with a tile per cluster."""
    import tcacomp_b200 as T
    T.tune("ffn", 0, request.param[0], 0, request.param[1])
    yield request.param
    T.tune("ffn")


# rows from one token on, extents that end inside boxes, blocks and tiles, one K block and many
SIZES = [(1, 8, 8), (1, 256, 128), (7, 64, 264), (16, 512, 40), (33, 200, 136), (128, 64, 256), (129, 1000, 520),
         (250, 72, 1032), (300, 648, 392), (515, 136, 776)]


@pytest.mark.parametrize("m,k,n", SIZES)
def test_forward_against_64_bits(tile, cuda, m, k, n):
    import tcacomp_b200 as T
    a, b = rnd(m, k, seed=1), rnd(k, n, seed=2, scale=k ** -0.5)
    bias, res = rnd(n, seed=3, scale=0.3, dtype=torch.float32), rnd(m, n, seed=4, scale=2.0)
    for act, use_bias, use_res, save in (("gelu", 1, 1, 1), ("silu", 1, 0, 0), ("none", 0, 1, 0), ("relu", 0, 0, 1), ("gelu_tanh", 1, 1, 0)):
        z, e = R.project(a, b, bias if use_bias else None)
        want = R.act(z, act)
        bound = R.SLOPE * e + R.ACT_ERR * (1 + want.abs())
        if use_res:
            want = want + res.double()
            bound = bound + R.H32 * want.abs()
        pre = torch.full((m, n), 5.0, device="cuda", dtype=BF) if save else None
        c = T.gemm_bias_act_residual(a, b, bias if use_bias else None, res if use_res else None, act, preact=pre)
        R.check(c, want, bound + R.H16 * (want.abs() + bound), f"c ({act})")
        if save:
            R.check(pre, z, e + R.H16 * (z.abs() + e), f"preact ({act})")
    assert T.device_status() == 0


@pytest.mark.parametrize("m,k,n", SIZES)
def test_gated_forward_against_64_bits(tile, cuda, m, k, n):
    import tcacomp_b200 as T
    x, wg, wu = rnd(m, k, seed=1), rnd(k, n, seed=2, scale=k ** -0.5), rnd(k, n, seed=3, scale=k ** -0.5)
    bg, bu = rnd(n, seed=4, scale=0.3, dtype=torch.float32), rnd(n, seed=5, scale=0.3, dtype=torch.float32)
    for act, use_bias, save in (("silu", 0, 1), ("gelu", 1, 0), ("gelu_tanh", 1, 1), ("sigmoid", 0, 0), ("relu", 0, 1)):
        g, eg = R.project(x, wg, bg if use_bias else None)
        u, eu = R.project(x, wu, bu if use_bias else None)
        f = R.act(g, act)
        ef = R.SLOPE * eg + R.ACT_ERR * (1 + f.abs())
        want = f * u
        bound = u.abs() * ef + f.abs() * eu + ef * eu + R.H32 * want.abs()
        gate, up = (torch.full((m, n), 5.0, device="cuda", dtype=BF) for _ in range(2))
        h = T.gated_gemm(x, wg, wu, bg if use_bias else None, bu if use_bias else None, act,
                         **({"gate": gate, "up": up} if save else {}))
        R.check(h, want, bound + R.H16 * (want.abs() + bound), f"h ({act})")
        if save:
            R.check(gate, g, eg + R.H16 * (g.abs() + eg), f"gate ({act})")
            R.check(up, u, eu + R.H16 * (u.abs() + eu), f"up ({act})")
    assert T.device_status() == 0


def check_contraction(got, left, right, left_err, what):
    """got = left @ right, the left operand known to `left_err` per element besides its rounding to bf16: elementwise with
    absolute values, and in norm (|E R|_F <= |E|_F |R|_2), where roundings do not add up as if they had one sign."""
    want = left @ right
    s = left.abs() @ right.abs()
    acc = (left.shape[1] + 2) * 2.0 ** -23 * s
    bound = R.H16 * s + left_err @ right.abs() + acc
    R.check(got, want, bound + R.H16 * (want.abs() + bound), what)
    norm = (R.H16 * float(torch.linalg.norm(left)) + float(torch.linalg.norm(left_err))) * R.spectral(right) + float(torch.linalg.norm(acc))
    R.check_norm(got, want, norm + R.H16 * (float(torch.linalg.norm(want)) + norm), what)


@pytest.mark.parametrize("m,k,n", SIZES)
def test_backward_against_64_bits(tile, cuda, m, k, n):
    import tcacomp_b200 as T
    a, b, dc, z = rnd(m, k, seed=1), rnd(k, n, seed=2, scale=k ** -0.5), rnd(m, n, seed=3, scale=0.05), rnd(m, n, seed=4, scale=1.5)
    z[0, :4] = torch.tensor([0.0, -30.0, 30.0, -0.0], device="cuda")
    for act in ("none", "relu", "silu", "gelu", "gelu_tanh"):
        got = T.gemm_bias_act_backward(dc, a, b, None if act == "none" else z, act)
        dz = dc.double() * (R.slope(z.double(), act) if act != "none" else 1.0)
        err = torch.zeros_like(dz) if act in ("none", "relu") else R.ACT_ERR * (1 + z.double().abs()) * dc.double().abs()
        check_contraction(got["da"], dz, b.double().t(), err, f"da ({act})")
        check_contraction(got["db"].t(), dz.t(), a.double(), err.t(), f"db ({act})")
        R.check(got["dbias"], dz.sum(0), err.sum(0) + (64 + m / 8) * R.H32 * dz.abs().sum(0), f"dbias ({act})")
    assert T.device_status() == 0


@pytest.mark.parametrize("m,k,n", SIZES)
def test_gated_backward_against_64_bits(tile, cuda, m, k, n):
    import tcacomp_b200 as T
    x, wg, wu = rnd(m, k, seed=1), rnd(k, n, seed=2, scale=k ** -0.5), rnd(k, n, seed=3, scale=k ** -0.5)
    dh, gate, up = rnd(m, n, seed=4, scale=0.05), rnd(m, n, seed=5, scale=1.5), rnd(m, n, seed=6)
    for act in ("silu", "gelu", "gelu_tanh", "sigmoid", "relu"):
        got = T.gated_gemm_backward(dh, x, wg, wu, gate, up, act, want=("dx", "dw_gate", "dw_up", "dbias_gate", "dbias_up"))
        d, g, u = dh.double(), gate.double(), up.double()
        dgate, dup = d * u * R.slope(g, act), d * R.act(g, act)
        e1 = R.ACT_ERR * (1 + g.abs()) * (d * u).abs() + 2 * R.H32 * dgate.abs()
        e2 = R.ACT_ERR * (1 + R.act(g, act).abs()) * d.abs() + R.H32 * dup.abs()
        check_contraction(got["dx"], torch.cat([dgate, dup], 1), torch.cat([wg, wu], 1).double().t(), torch.cat([e1, e2], 1), f"dx ({act})")
        check_contraction(got["dw_gate"].t(), dgate.t(), x.double(), e1.t(), f"dw_gate ({act})")
        check_contraction(got["dw_up"].t(), dup.t(), x.double(), e2.t(), f"dw_up ({act})")
        chain = (64 + m / 8) * R.H32
        R.check(got["dbias_gate"], dgate.sum(0), e1.sum(0) + chain * dgate.abs().sum(0), f"dbias_gate ({act})")
        R.check(got["dbias_up"], dup.sum(0), e2.sum(0) + chain * dup.abs().sum(0), f"dbias_up ({act})")
    assert T.device_status() == 0


# small integers: every product and sum is exact in fp32, so the results are the exact ones rounded to bf16
EXACT = [(1, 64, 64), (5, 1032, 264), (64, 2056, 520), (128, 4096, 256), (257, 520, 1288), (640, 328, 712), (1000, 1000, 1096), (1537, 264, 2312)]


@pytest.mark.parametrize("m,k,n", EXACT)
def test_exact_on_small_integers(tile, cuda, m, k, n):
    import tcacomp_b200 as T
    a, b, b2 = ints(m, k, seed=1), ints(k, n, seed=2), ints(k, n, seed=3)
    res, dc = ints(m, n, seed=4, lo=-9, hi=10), ints(m, n, seed=5)
    z, z2 = a.double() @ b.double(), a.double() @ b2.double()
    pre = torch.empty((m, n), device="cuda", dtype=BF)
    c = T.gemm_bias_act_residual(a, b, None, res, "relu", preact=pre)
    assert torch.equal(c, (z.clamp(min=0) + res.double()).float().to(BF)) and torch.equal(pre, z.float().to(BF))
    gate, up = torch.empty_like(pre), torch.empty_like(pre)
    h = T.gated_gemm(a, b, b2, act="relu", gate=gate, up=up)
    # the product of two integers below 2^12 is exact in fp32
    assert torch.equal(gate, z.float().to(BF)) and torch.equal(up, z2.float().to(BF))
    assert torch.equal(h, (z.clamp(min=0) * z2).float().to(BF))
    got = T.gemm_bias_act_backward(dc, a, b, pre, "relu")
    dz = dc.double() * (pre.double() > 0)
    assert torch.equal(got["da"], (dz @ b.double().t()).float().to(BF))
    assert torch.equal(got["db"], (a.double().t() @ dz).float().to(BF))
    assert torch.equal(got["dbias"].double(), dz.sum(0))
    got = T.gated_gemm_backward(dc, a, b, b2, ints(m, n, seed=6), ints(m, n, seed=7), "relu")
    g, u = ints(m, n, seed=6).double(), ints(m, n, seed=7).double()
    dg, du = dc.double() * u * (g > 0), dc.double() * g.clamp(min=0)
    assert torch.equal(got["dx"], (dg @ b.double().t() + du @ b2.double().t()).float().to(BF))
    assert torch.equal(got["dw_gate"], (a.double().t() @ dg).float().to(BF))
    assert torch.equal(got["dw_up"], (a.double().t() @ du).float().to(BF))
    assert T.device_status() == 0


def test_gradients_against_differences(tcab_lib, cuda):
    """Along random directions the 64-bit forward's central difference is what the kernels' gradients say."""
    import tcacomp_b200 as T
    m, k, n = 48, 96, 160
    x, wg, wu = rnd(m, k, seed=1), rnd(k, n, seed=2, scale=k ** -0.5), rnd(k, n, seed=3, scale=k ** -0.5)
    bg, bu, dh = rnd(n, seed=4, dtype=torch.float32), rnd(n, seed=5, dtype=torch.float32), rnd(m, n, seed=6)
    at = [t.double() for t in (x, wg, wu, bg, bu)]

    def gated(x_, g_, u_, bg_, bu_):
        return ((R.act(x_ @ g_ + bg_, "gelu") * (x_ @ u_ + bu_)) * dh.double()).sum()

    def plain(x_, b_, bias_):
        return (R.act(x_ @ b_ + bias_, "silu") * dh.double()).sum()

    def differences(f, at, grads, forward_rounding):
        for i, grad in enumerate(grads):
            d = torch.randn(at[i].shape, device="cuda", dtype=torch.float64)
            ends = [f(*[p + s * 1e-5 * d if j == i else p for j, p in enumerate(at)]) for s in (1, -1)]
            want, got = (ends[0] - ends[1]) / 2e-5, (grad.double() * d).sum()
            # three roundings to bf16 reach a gradient: the kept projections, the operand, the result; the directions'
            # signs are random, so the elementwise bound is far from reached
            bound = forward_rounding * R.H16 * (grad.double().abs() * d.abs()).sum() + 1e-6 * (1 + want.abs())
            assert (got - want).abs() <= bound, (i, float(got), float(want), float(bound))

    gate, up = torch.empty((m, n), device="cuda", dtype=BF), torch.empty((m, n), device="cuda", dtype=BF)
    T.gated_gemm(x, wg, wu, bg, bu, "gelu", gate=gate, up=up)
    got = T.gated_gemm_backward(dh, x, wg, wu, gate, up, "gelu", want=("dx", "dw_gate", "dw_up", "dbias_gate", "dbias_up"))
    differences(gated, at, [got[name] for name in ("dx", "dw_gate", "dw_up", "dbias_gate", "dbias_up")], 4)
    z = torch.empty((m, n), device="cuda", dtype=BF)
    T.gemm_bias_act_residual(x, wg, bg, None, "silu", preact=z)
    got = T.gemm_bias_act_backward(dh, x, wg, z, "silu")
    differences(plain, [at[0], at[1], at[3]], [got["da"], got["db"], got["dbias"]], 4)


def test_activation_values_and_slopes(tile, cuda):
    """Over the whole range of arguments: an empty contraction stores act(bias), one row's dbias is the slope in fp32."""
    import tcacomp_b200 as T
    grid = torch.cat([torch.linspace(-40, 40, 3997, device="cuda"), torch.logspace(-30, 38, 200, device="cuda"),
                      -torch.logspace(-30, 38, 200, device="cuda"), torch.tensor([0.0, -0.0, float("nan")], device="cuda")])
    n = grid.numel()
    assert n % 8 == 0
    none = torch.empty((1, 0), device="cuda", dtype=BF)
    for act in ("relu", "silu", "gelu", "gelu_tanh"):
        want = R.act(grid.double(), act)
        got = T.gemm_bias_act_residual(none, torch.empty((0, n), device="cuda", dtype=BF), grid, act=act)[0]
        bound = R.ACT_ERR * (1 + want.abs())
        # values below fp32's smallest normal number may be flushed to zero
        R.check(got, want, bound + R.H16 * (want.abs() + bound) + 2.0 ** -126, f"{act}")
        z = grid.to(BF)
        wslope = R.slope(z.double(), act)
        if act == "relu":
            wslope[torch.isnan(z)] = 0  # a comparison with NaN is false
        a, b = torch.zeros((1, 8), device="cuda", dtype=BF), torch.zeros((8, n), device="cuda", dtype=BF)
        got = T.gemm_bias_act_backward(torch.ones((1, n), device="cuda", dtype=BF), a, b, z.view(1, n), act, want=("dbias",))["dbias"]
        # beyond 1e3 every slope here is 0 or 1 to the last bit (the reference's own formula overflows there)
        far = z.double().abs() > 1e3
        wslope = torch.where(far, (z > 0).double(), wslope)
        R.check(got, wslope, R.ACT_ERR * (1 + z.double().abs().clamp(max=40)), f"slope of {act}")


def test_two_threads_on_their_own_streams(tcab_lib, cuda):
    """Host threads that call at the same time, each on a stream of its own: the results are those of calls alone."""
    import threading

    import tcacomp_b200 as T
    sets = [(rnd(200, 256, seed=40 + i), rnd(256, 520, seed=50 + i), rnd(200, 520, seed=60 + i)) for i in range(2)]
    want = [(T.gemm_bias_act_residual(a, b, None, dc, "silu"), T.gemm_bias_act_backward(dc, a, b, dc, "silu")) for a, b, dc in sets]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        a, b, dc = sets[i]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                c = T.gemm_bias_act_residual(a, b, None, dc, "silu")
                g = T.gemm_bias_act_backward(dc, a, b, dc, "silu")
            torch.cuda.current_stream().synchronize()
        if not torch.equal(c, want[i][0]) or any(not torch.equal(g[k], want[i][1][k]) for k in g):
            bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad and T.device_status() == 0


def test_empty_extents(tcab_lib, cuda):
    import tcacomp_b200 as T
    bias = torch.linspace(-1, 1, 16, device="cuda")
    a, b, res = torch.empty((3, 0), device="cuda", dtype=BF), torch.empty((0, 16), device="cuda", dtype=BF), ints(3, 16, seed=1)
    c = T.gemm_bias_act_residual(a, b, bias, res, "relu")  # an empty contraction: act(bias) + residual
    assert torch.equal(c, (bias.clamp(min=0)[None] + res.float()).to(BF))
    h = T.gated_gemm(a, b, b, bias, bias, "relu")
    assert torch.equal(h, (bias.clamp(min=0) * bias)[None].expand(3, 16).to(BF))
    none = torch.empty((0, 32), device="cuda", dtype=BF)
    w = ints(32, 16, seed=2)
    assert T.gemm_bias_act_residual(none, w, act="gelu").shape == (0, 16)
    out = {"da": torch.empty((0, 32), device="cuda", dtype=BF), "db": torch.full((32, 16), 7.0, device="cuda", dtype=BF),
           "dbias": torch.full((16,), 7.0, device="cuda")}
    zero = torch.empty((0, 16), device="cuda", dtype=BF)
    got = T.gemm_bias_act_backward(zero, none, w, zero, "gelu", out=out)  # no rows: the sums over them are zero
    assert not got["db"].any() and not got["dbias"].any()
    got = T.gated_gemm_backward(zero, none, w, w, zero, zero, "silu", want=("dx", "dw_gate", "dw_up", "dbias_gate", "dbias_up"))
    assert not got["dw_gate"].any() and not got["dw_up"].any() and not got["dbias_gate"].any() and not got["dbias_up"].any()
    wide, x = torch.empty((32, 0), device="cuda", dtype=BF), ints(5, 32, seed=3)
    got = T.gemm_bias_act_backward(torch.empty((5, 0), device="cuda", dtype=BF), x, wide, act="none", want=("da", "db"))
    assert got["da"].shape == (5, 32) and not got["da"].any() and got["db"].shape == (32, 0)
    assert T.device_status() == 0


def test_rows_with_special_values_stay_their_own(tcab_lib, cuda):
    import tcacomp_b200 as T
    for m in (5, 300):
        a, b = rnd(m, 128, seed=1), rnd(128, 264, seed=2)
        clean = T.gemm_bias_act_residual(a, b, act="gelu")
        bad = a.clone()
        bad[3, 7], bad[1, 0] = float("nan"), float("inf")
        got = T.gemm_bias_act_residual(bad, b, act="gelu")
        assert torch.isnan(got[3].float()).all() and not torch.isfinite(got[1].float()).all()
        keep = [i for i in range(m) if i not in (1, 3)]
        assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("m", [3, 200])
def test_outputs_in_canaries_and_residual_in_place(tcab_lib, cuda, m):
    import tcacomp_b200 as T
    k, n = 136, 392
    a, b, res, dc = rnd(m, k, seed=1), rnd(k, n, seed=2), rnd(m, n, seed=3), rnd(m, n, seed=4)

    def canary(*shape, dtype=BF):
        size = 1
        for d in shape:
            size *= d
        buf = torch.full((size + 256,), 3.0, device="cuda", dtype=dtype)
        return buf, buf[128:128 + size].view(*shape)

    def intact(buf):
        assert (buf[:128] == 3).all() and (buf[-128:] == 3).all()

    want = T.gemm_bias_act_residual(a, b, None, res, "silu")
    (cb, c), (zb, z) = canary(m, n), canary(m, n)
    T.gemm_bias_act_residual(a, b, None, res, "silu", out=c, preact=z)
    intact(cb), intact(zb)
    assert torch.equal(c, want)
    r2 = res.clone()
    assert T.gemm_bias_act_residual(a, b, None, r2, "silu", out=r2) is r2 and torch.equal(r2, want)
    bufs = {"da": canary(m, k), "db": canary(k, n), "dbias": canary(n, dtype=torch.float32)}
    got = T.gemm_bias_act_backward(dc, a, b, z, "silu", out={name: v for name, (_, v) in bufs.items()})
    ref = T.gemm_bias_act_backward(dc, a, b, z, "silu")
    for name, (buf, v) in bufs.items():
        intact(buf)
        assert torch.equal(got[name], ref[name])
    only = T.gemm_bias_act_backward(dc, a, b, z, "silu", want=("dbias",))
    assert list(only) == ["dbias"] and torch.equal(only["dbias"], ref["dbias"])


def block_forward(T, p, x):
    """A feed-forward sublayer: norm, gated projections, output projection with the residual stream added."""
    y, mean, rstd = T.layernorm_rows_stats(x, p["gamma"], p["beta"])
    gate, up = torch.empty((x.shape[0], p["w_up"].shape[1]), device=x.device, dtype=BF), None
    up = torch.empty_like(gate)
    h = T.gated_gemm(y, p["w_gate"], p["w_up"], act="silu", gate=gate, up=up)
    out = T.gemm_bias_act_residual(h, p["w_down"], p["b_down"], x, "none")
    return out, (y, mean, rstd, gate, up, h)


def block_backward(T, p, x, kept, dout):
    y, mean, rstd, gate, up, h = kept
    down = T.gemm_bias_act_backward(dout, h, p["w_down"], act="none")
    mid = T.gated_gemm_backward(down["da"], y, p["w_gate"], p["w_up"], gate, up, "silu")
    dx, dgamma, dbeta = T.layernorm_rows_backward(mid["dx"], x, p["gamma"], mean, rstd)
    return {"dx_branch": dx, "dgamma": dgamma, "dbeta": dbeta, "dw_gate": mid["dw_gate"], "dw_up": mid["dw_up"],
            "dw_down": down["db"], "db_down": down["dbias"]}


def block_params(d, f):
    return {"gamma": rnd(d, seed=11, scale=0.2).add_(1), "beta": rnd(d, seed=12, scale=0.1), "w_gate": rnd(d, f, seed=13, scale=d ** -0.5),
            "w_up": rnd(d, f, seed=14, scale=d ** -0.5), "w_down": rnd(f, d, seed=15, scale=f ** -0.5),
            "b_down": rnd(d, seed=16, scale=0.1, dtype=torch.float32)}


@pytest.mark.parametrize("m,d,f", [(1, 256, 712), (77, 264, 520), (400, 512, 1096)])
def test_a_sublayer_forward_and_backward(tcab_lib, cuda, m, d, f):
    """The operators as a training step calls them, against 64 bits with bf16 roundings at the same places. What is left
    then are fp32 sums and values that a rounding tie lets fall the other way, one step in a small share of the elements:
    less than half a step over the whole of each result."""
    import tcacomp_b200 as T
    p, x, dout = block_params(d, f), rnd(m, d, seed=17, scale=2.0), rnd(m, d, seed=18, scale=0.1)
    out, kept = block_forward(T, p, x)
    got = block_backward(T, p, x, kept, dout)
    q = lambda t: t.float().to(BF).double()  # noqa: E731
    P = {name: t.double() for name, t in p.items()}
    wy, mean, rstd = R.layernorm(x, p["gamma"], p["beta"], 1e-5)[:3]
    y = q(wy)
    g, u = y @ P["w_gate"], y @ P["w_up"]
    h = q(R.act(g, "silu") * u)
    want = q(h @ P["w_down"] + P["b_down"] + x.double())
    g, u = q(g), q(u)
    dh = q(dout.double() @ P["w_down"].t())
    dg, du = q(dh * u * R.slope(g, "silu")), q(dh * R.act(g, "silu"))
    dy = q(dg @ P["w_gate"].t() + du @ P["w_up"].t())
    dx, dgamma, dbeta = R.layernorm_grads(dy, x, p["gamma"], mean, rstd)[:3]
    ref = {"dx_branch": q(dx), "dgamma": dgamma, "dbeta": dbeta, "dw_gate": q(y.t() @ dg), "dw_up": q(y.t() @ du),
           "dw_down": q(h.t() @ dout.double()), "db_down": dout.double().sum(0)}
    R.check_norm(out, want, R.H16 * float(torch.linalg.norm(want)), "out")
    for name, w in ref.items():
        R.check_norm(got[name], w, R.H16 * float(torch.linalg.norm(w)), name)


def test_a_training_step_captured_and_replayed(tcab_lib, cuda):
    """Two captured sublayer steps replayed at once on two streams beside eager ones on a third, whose stream is given."""
    import tcacomp_b200 as T
    p = block_params(256, 520)
    xs, douts = [rnd(300, 256, seed=20 + i) for i in range(3)], [rnd(300, 256, seed=30 + i) for i in range(3)]
    want = []
    for x, dout in zip(xs, douts):
        out, kept = block_forward(T, p, x)
        want.append((out, block_backward(T, p, x, kept, dout)))
    graphs, res = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, kept = block_forward(T, p, xs[i])
            res.append((out, block_backward(T, p, xs[i], kept, douts[i])))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        with torch.cuda.stream(streams[2]):
            out, kept = block_forward(T, p, xs[2])
        eager = T.gemm_bias_act_backward(douts[2], kept[5], p["w_down"], act="none", stream=streams[2])
    torch.cuda.synchronize()
    for (out, grads), (o, g) in zip(res, want):
        assert torch.equal(out, o) and all(torch.equal(grads[name], g[name]) for name in g)
    assert torch.equal(out, want[1][0]) and torch.equal(eager["db"], want[2][1]["dw_down"])
    assert T.device_status() == 0


def test_a_captured_fork_and_join(tcab_lib, cuda):
    """A capture whose calls wait for events of another stream: both branches of a sublayer and what joins them."""
    import tcacomp_b200 as T
    p = block_params(256, 520)
    x, y = rnd(130, 256, seed=50), rnd(130, 256, seed=51)
    want = T.gemm_bias_act_residual(block_forward(T, p, x)[0], p["w_gate"], None, block_forward(T, p, y)[1][3], "none")
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            gate = block_forward(T, p, y)[1][3]
        out = block_forward(T, p, x)[0]
        main.wait_stream(side)
        got = T.gemm_bias_act_residual(out, p["w_gate"], None, gate, "none")
    for _ in range(5):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_offsets_past_32_bits(tcab_lib, cuda):
    """Tensors of 4.29e9 elements, 8.6 GB each: the last row, some in the middle, the last columns."""
    import tcacomp_b200 as T
    m, k, n = 65528, 16, 65536
    a, b, bias = rnd(m, k, seed=1), rnd(k, n, seed=2), torch.randn(n, device="cuda")
    c, z = torch.empty(m, n, device="cuda", dtype=BF), torch.empty(m, n, device="cuda", dtype=BF)
    T.gemm_bias_act_residual(a, b, bias, None, "silu", out=c, preact=z)
    rows = [0, 1, 16384, 32767, 32768, 49999, m - 2, m - 1]
    want, e = R.project(a[rows], b, bias)
    R.check(z[rows], want, e + R.H16 * (want.abs() + e), "preact")
    want = R.act(want, "silu")
    bound = R.SLOPE * e + R.ACT_ERR * (1 + want.abs())
    R.check(c[rows], want, bound + R.H16 * (want.abs() + bound), "c")
    # dz = z silu'(z), with z in dc's place too: rounded once, then contracted over the 65536 columns
    got = T.gemm_bias_act_backward(z, a, b, z, "silu", want=("da",))["da"]
    zr = z[rows].double()
    dz = zr * R.slope(zr, "silu")
    e_dz = zr.abs() * R.ACT_ERR * (1 + R.act(zr, "silu").abs()) + R.H32 * dz.abs()
    e_dz = e_dz + R.H16 * (dz.abs() + e_dz)
    want, size = dz @ b.double().t(), (dz.abs() + e_dz) @ b.double().abs().t()
    bound = e_dz @ b.double().abs().t() + (n + 2) * 2.0 ** -23 * size
    R.check(got[rows], want, bound + R.H16 * (want.abs() + bound), "da")
    del c, z
    torch.cuda.empty_cache()


def test_a_stream_of_another_device(tcab_lib, cuda):
    import types

    import tcacomp_b200 as T
    other = types.SimpleNamespace(device_index=1, cuda_stream=0)
    a = rnd(8, 16, seed=1)
    for call in (lambda: T.gemm_bias_act_residual(a, rnd(16, 8, seed=2), act="none", stream=other),
                 lambda: T.gated_gemm(a, rnd(16, 8, seed=2), rnd(16, 8, seed=3), stream=other),
                 lambda: T.layernorm_rows_stats(a, a[0], a[1], stream=other)):
        with pytest.raises(ValueError, match="stream is on cuda:1"):
            call()
