"""layernorm_rows_stats and layernorm_rows_backward against 64 bits, and what a training program does with them."""
import pytest
import torch

import ffn_reference as R

pytestmark = pytest.mark.gpu

BF, F = torch.bfloat16, torch.float32


def make(shape, dtype, seed=0, shift=0):
    """x, gamma, beta, dy; shift: elements by which every tensor's start leaves its 16-byte alignment."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def t(*s, scale=1.0, add=0.0):
        n = 1
        for d in s:
            n *= d
        buf = torch.full((n + 64,), float("nan"), device="cuda", dtype=dtype)  # poisoned around the operand
        v = buf[8 + shift:8 + shift + n].view(*s)
        v.copy_(torch.randn(s, device="cuda", generator=g) * scale + add)
        return v

    cols = shape[-1]
    x = t(*shape, scale=2.0, add=0.5)
    x[..., ::7] *= 5
    return x, t(cols, scale=0.3, add=1.0), t(cols, scale=0.2), t(*shape, scale=0.1)


# rows of every kernel: one vector and less, short rows in a warp, a CTA per row, more than one CTA's registers; whole
# vectors and not; few rows and many
SHAPES = [((1, 1), 0), ((3, 5), 0), ((1, 8), 0), ((33, 64), 0), ((257, 96), 0), ((1000, 200), 0), ((70, 129), 0),
          ((5, 1001), 0), ((129, 1024), 0), ((9, 1024), 1), ((40, 1280), 0), ((301, 2048), 0), ((4, 4096), 0), ((1, 8192), 0),
          ((170, 8200), 0), ((13, 12288), 0), ((21, 16384), 0), ((6, 16400), 0), ((7, 20001), 0), ((200, 33000), 0),
          ((2, 3, 5, 72), 0), ((640,), 0)]


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("shape,shift", SHAPES)
def test_statistics_and_gradients_against_64_bits(tcab_lib, cuda, shape, shift, dtype):
    import tcacomp_b200 as T
    x, gamma, beta, dy = make(shape, dtype, seed=len(shape) + shape[-1], shift=shift)
    y, mean, rstd = T.layernorm_rows_stats(x, gamma, beta, 1e-5)
    assert torch.equal(y, T.layernorm_rows(x, gamma, beta, 1e-5)), "the rows are those of layernorm_rows"
    assert mean.shape == (x.shape[:-1] or (1,)) and mean.dtype == F and rstd.dtype == F
    wy, wm, wr, ey, em, er = R.layernorm(x, gamma, beta, 1e-5)
    h = R.half_step(dtype)
    R.check(y, wy, ey + h * (wy.abs() + ey), "y")
    R.check(mean.view(wm.shape), wm, em + R.H32 * wm.abs(), "mean")
    R.check(rstd.view(wr.shape), wr, er, "rstd")
    dx, dgamma, dbeta = T.layernorm_rows_backward(dy, x, gamma, mean, rstd)
    wx, wg, wb, ex, eg, eb = R.layernorm_grads(dy, x, gamma, mean.view(wm.shape), rstd.view(wr.shape))
    R.check(dx, wx, ex + h * (wx.abs() + ex), "dx")
    R.check(dgamma, wg, eg, "dgamma")
    R.check(dbeta, wb, eb, "dbeta")
    again = T.layernorm_rows_backward(dy, x, gamma, mean, rstd)
    assert all(torch.equal(p, q) for p, q in zip((dx, dgamma, dbeta), again)), "the same call gives the same bits"


@pytest.mark.parametrize("shape", [(37, 72), (11, 4096), (5, 1003)])
def test_gradients_against_differences(tcab_lib, cuda, shape):
    """Along random directions the 64-bit forward's central difference is what the kernel's gradients say."""
    import tcacomp_b200 as T
    x, gamma, beta, dy = make(shape, F, seed=3)
    _, mean, rstd = T.layernorm_rows_stats(x, gamma, beta, 1e-5)
    dx, dgamma, dbeta = T.layernorm_rows_backward(dy, x, gamma, mean, rstd)
    _, _, _, _, e_mean, e_rstd = R.layernorm(x, gamma, beta, 1e-5)
    _, _, _, ex, eg, eb = R.layernorm_grads(dy, x, gamma, mean, rstd)

    def loss(x_, g_, b_):
        mu = x_.mean(-1, keepdim=True)
        r = ((x_ - mu).square().mean(-1, keepdim=True) + 1e-5).rsqrt()
        return (((x_ - mu) * r * g_ + b_) * dy.double()).sum()

    at = [x.double(), gamma.double(), beta.double()]
    for i, (grad, err) in enumerate(zip((dx, dgamma, dbeta), (ex, eg, eb))):
        d = torch.randn(at[i].shape, device="cuda", dtype=torch.float64)
        step = 1e-5
        ends = []
        for sign in (1, -1):
            moved = list(at)
            moved[i] = at[i] + sign * step * d
            ends.append(loss(*moved))
        want = (ends[0] - ends[1]) / (2 * step)
        got = (grad.double() * d).sum()
        # the kernel's own error, that of the statistics it was given (a relative 2^-24-sized change of mean and rstd
        # moves every term of the gradient by as much), and the difference quotient's (third derivative * step^2)
        rel = float((e_rstd / rstd.double()).max() + (e_mean * rstd.double()).max())
        bound = (err * d.abs()).sum() + 8 * rel * (grad.double().abs() * d.abs()).sum() + \
            rel * (dy.double().abs().sum() * d.abs().max()) + 1e-7 * (1 + want.abs())
        assert (got - want).abs() <= bound, (i, float(got), float(want), float(bound))


def test_rows_and_columns_with_special_values(tcab_lib, cuda):
    """A NaN or an infinity stays in its row of dx, and in its column of dgamma and dbeta only as the sums say."""
    import tcacomp_b200 as T
    x, gamma, beta, dy = make((64, 512), BF, seed=9)
    x[5, 17] = float("inf")
    x[9, 100] = float("nan")
    x[20] = 0.75  # no spread at all: rstd = 1 / sqrt(eps)
    y, mean, rstd = T.layernorm_rows_stats(x, gamma, beta, 1e-5)
    dx, dgamma, dbeta = T.layernorm_rows_backward(dy, x, gamma, mean, rstd)
    bad = torch.zeros(64, dtype=torch.bool, device="cuda")
    bad[5] = bad[9] = True
    assert torch.isfinite(dx[~bad].float()).all() and not torch.isfinite(dx[bad].float()).all(-1).any()
    assert torch.isnan(dgamma).all() and torch.isfinite(dbeta).all()
    assert float(mean[20]) == 0.75
    want = (torch.tensor(1e-5, dtype=torch.float32).double()).rsqrt()
    assert abs(float(rstd[20]) - float(want)) <= 4 * R.H32 * float(want)


def test_no_rows(tcab_lib, cuda):
    import tcacomp_b200 as T
    x, gamma, beta, _ = make((1, 128), F)
    e = x[:0]
    y, mean, rstd = T.layernorm_rows_stats(e, gamma, beta)
    assert y.shape == (0, 128) and mean.shape == (0,)
    dgamma, dbeta = torch.full((128,), 7.0, device="cuda"), torch.full((128,), 7.0, device="cuda")
    dx, dgamma, dbeta = T.layernorm_rows_backward(e, e, gamma, mean, rstd, dgamma=dgamma, dbeta=dbeta)
    assert dx.shape == (0, 128) and not dgamma.any() and not dbeta.any()


@pytest.mark.parametrize("cols", [200, 4096, 20008])
def test_in_place_and_outputs_in_canaries(tcab_lib, cuda, cols):
    """dx over dy, dx over x, y over x; nothing outside the outputs is written."""
    import tcacomp_b200 as T
    x, gamma, beta, dy = make((50, cols), BF, seed=4)
    y, mean, rstd = T.layernorm_rows_stats(x, gamma, beta)
    want = T.layernorm_rows_backward(dy, x, gamma, mean, rstd)
    d2 = dy.clone()
    got = T.layernorm_rows_backward(d2, x, gamma, mean, rstd, dx=d2)
    assert got[0] is d2 and all(torch.equal(p, q) for p, q in zip(want, got))
    x2 = x.clone()
    got = T.layernorm_rows_backward(dy, x2, gamma, mean, rstd, dx=x2)
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    x3 = x.clone()
    T.layernorm_rows_stats(x3, gamma, beta, out=x3)
    assert torch.equal(x3, y)
    buf = torch.full((50 * cols + 512,), 3.0, device="cuda", dtype=BF)
    sums = torch.full((2, cols + 64), 3.0, device="cuda")
    out = buf[256:256 + 50 * cols].view(50, cols)
    T.layernorm_rows_backward(dy, x, gamma, mean, rstd, dx=out, dgamma=sums[0, 32:32 + cols], dbeta=sums[1, 32:32 + cols])
    assert torch.equal(out, want[0]) and torch.equal(sums[0, 32:32 + cols], want[1])
    assert (buf[:256] == 3).all() and (buf[-256:] == 3).all() and (sums[:, :32] == 3).all() and (sums[:, -32:] == 3).all()


def test_captured_and_replayed_beside_another_stream(tcab_lib, cuda):
    """Two captured passes replayed at once and an eager one on a third stream: each has a workspace of its own."""
    import tcacomp_b200 as T
    sets = [make((300, 1024), BF, seed=s) for s in range(3)]
    stats = [T.layernorm_rows_stats(x, g, b)[1:] for x, g, b, _ in sets]
    want = [T.layernorm_rows_backward(dy, x, g, *st) for (x, g, b, dy), st in zip(sets, stats)]
    graphs, outs = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        x, g, b, dy = sets[i]
        with torch.cuda.graph(graph):
            outs.append(T.layernorm_rows_backward(dy, x, g, *stats[i]))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        x, g, b, dy = sets[2]
        eager = T.layernorm_rows_backward(dy, x, g, *stats[2], stream=streams[2])
    torch.cuda.synchronize()
    for got, w in zip(outs + [eager], want):
        assert all(torch.equal(p, q) for p, q in zip(got, w))


@pytest.mark.parametrize("rows,cols", [(1048568, 4096), (65528, 65536)])
def test_offsets_past_32_bits(tcab_lib, cuda, rows, cols):
    """Tensors of 4.29e9 elements: rows at both ends and in the middle, dx written over dy."""
    import tcacomp_b200 as T
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    x = torch.randn(rows, cols, device="cuda", generator=g, dtype=BF)
    gamma = torch.randn(cols, device="cuda", generator=g, dtype=BF)
    dy, mean, rstd = T.layernorm_rows_stats(x, gamma, gamma, 1e-5)
    pick = [0, 1, rows // 4, rows // 2 - 1, rows // 2, rows - 2, rows - 1]
    wy, wm, wr, ey, em, er = R.layernorm(x[pick], gamma, gamma, 1e-5)
    few = dy[pick].clone()
    R.check(few, wy, ey + R.H16 * (wy.abs() + ey), "y")
    R.check(mean[pick], wm, em + R.H32 * wm.abs(), "mean")
    R.check(rstd[pick], wr, er, "rstd")
    dx, dgamma, dbeta = T.layernorm_rows_backward(dy, x, gamma, mean, rstd, dx=dy)
    wx, _, _, ex, _, _ = R.layernorm_grads(few, x[pick], gamma, mean[pick], rstd[pick])
    R.check(dx[pick], wx, ex + R.H16 * (wx.abs() + ex), "dx")
    assert torch.isfinite(dgamma).all() and torch.isfinite(dbeta).all()
    del x, dx, dy
    torch.cuda.empty_cache()
