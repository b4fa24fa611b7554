"""What the feed-forward operators refuse, before any launch and without a device."""
import ctypes as C

import pytest
import torch


def T_(shape, dtype=1, data=0x100000):
    from tcacomp_b200 import _lib
    t = _lib.Tensor()
    t.data, t.dtype, t.rank = data, dtype, len(shape)
    for i, d in enumerate(shape):
        t.dims[i] = d
    return t


class Space:
    """Fake operands, none of which overlaps another."""

    def __init__(self):
        self.at = 0x1000000

    def __call__(self, *shape, dtype=1, shift=0):
        self.at += 0x1000000
        return T_(shape, dtype, self.at + shift)


def ref(t):
    return None if t is None else C.byref(t)


def message(lib):
    return lib.tcab_last_error().decode()


def call(lib, name, args):
    return getattr(lib, name)(*[ref(a) if a is None or hasattr(a, "rank") else a for a in args])


def test_layernorm_forms(tcab_lib):
    from tcacomp_b200 import _lib
    L, S = tcab_lib, Space()

    def stats(**kw):
        a = dict(x=S(4, 64), gamma=S(64), beta=S(64), y=S(4, 64), mean=S(4, dtype=0), rstd=S(4, dtype=0))
        a.update(kw)
        return call(L, "tcab_layernorm_rows_stats", [a["x"], a["gamma"], a["beta"], C.c_float(1e-5), a["y"], a["mean"], a["rstd"], None])

    assert stats(x=None) == _lib.ERR_INVALID_ARG
    assert stats(x=S(4, 0), y=S(4, 0)) == _lib.ERR_SHAPE and "positive" in message(L)
    assert stats(x=S(4, 64, dtype=2)) == _lib.ERR_DTYPE
    assert stats(y=S(4, 65)) == _lib.ERR_SHAPE
    assert stats(y=S(4, 64, dtype=0)) == _lib.ERR_DTYPE
    assert stats(gamma=S(63)) == _lib.ERR_SHAPE and "gamma" in message(L)
    assert stats(mean=S(5, dtype=0)) == _lib.ERR_SHAPE and "mean" in message(L)
    assert stats(rstd=S(4)) == _lib.ERR_DTYPE
    assert stats(mean=S(4, dtype=0, shift=2)) == _lib.ERR_ALIGNMENT
    m = S(4, dtype=0)
    assert stats(mean=m, rstd=m) == _lib.ERR_INVALID_ARG and "overlaps" in message(L)
    x = S(4, 64)
    assert stats(x=x, y=T_((4, 64), 1, x.data + 64)) == _lib.ERR_INVALID_ARG  # shifted over x
    if not torch.cuda.is_available():
        assert stats(x=x, y=x) == _lib.ERR_CUDA  # over x itself is allowed: refused for the missing device only

    def back(**kw):
        a = dict(dy=S(4, 64), x=S(4, 64), gamma=S(64), mean=S(4, dtype=0), rstd=S(4, dtype=0), dx=S(4, 64), dgamma=S(64, dtype=0),
                 dbeta=S(64, dtype=0))
        a.update(kw)
        return call(L, "tcab_layernorm_rows_backward", [a[n] for n in ("dy", "x", "gamma", "mean", "rstd", "dx", "dgamma", "dbeta")] + [None, 0, None])

    assert back(dy=S(4, 63)) == _lib.ERR_SHAPE
    assert back(dgamma=S(64)) == _lib.ERR_DTYPE
    assert back(dbeta=S(65, dtype=0)) == _lib.ERR_SHAPE
    assert back(dx=None) == _lib.ERR_INVALID_ARG
    g = S(64, dtype=0)
    assert back(dgamma=g, dbeta=g) == _lib.ERR_INVALID_ARG and "overlaps" in message(L)
    x = S(4, 64)
    assert back(x=x, dx=T_((4, 64), 1, x.data + 2)) == _lib.ERR_INVALID_ARG


def test_contraction_forms(tcab_lib):
    from tcacomp_b200 import _lib
    L, S = tcab_lib, Space()

    def fwd(act=3, **kw):
        a = dict(a=S(5, 64), b=S(64, 40), bias=S(40, dtype=0), residual=S(5, 40), preact=None, c=S(5, 40))
        a.update(kw)
        return call(L, "tcab_gemm_bias_act_residual", [a["a"], a["b"], a["bias"], a["residual"], act, a["preact"], a["c"], None])

    assert fwd(a=S(5, 64, dtype=0)) == _lib.ERR_DTYPE
    assert fwd(b=S(72, 40)) == _lib.ERR_SHAPE and "dim k" in message(L)
    assert fwd(a=S(5, 60), b=S(60, 40)) == _lib.ERR_ALIGNMENT and "multiples of 8" in message(L)
    assert fwd(b=S(64, 36), c=S(5, 36), bias=None, residual=None) == _lib.ERR_ALIGNMENT
    assert fwd(a=S(5, 64, shift=8)) == _lib.ERR_ALIGNMENT
    assert fwd(c=S(5, 48)) == _lib.ERR_SHAPE
    assert fwd(residual=S(1, 40)) == _lib.ERR_SHAPE and "residual" in message(L)
    assert fwd(bias=S(40)) == _lib.ERR_DTYPE
    assert fwd(bias=S(5, 40, dtype=0)) == _lib.ERR_SHAPE
    assert fwd(preact=S(5, 40, dtype=0)) == _lib.ERR_DTYPE
    assert fwd(act=5) == _lib.ERR_INVALID_ARG and fwd(act=-1) == _lib.ERR_INVALID_ARG and "activation" in message(L)
    r = S(5, 40)
    assert fwd(residual=r, preact=r) == _lib.ERR_INVALID_ARG  # only c may be the residual
    assert fwd(c=r, preact=r) == _lib.ERR_INVALID_ARG
    a = S(5, 40)
    assert fwd(a=a, b=S(40, 40), c=a) == _lib.ERR_INVALID_ARG and "overlaps" in message(L)

    def back(act=3, **kw):
        a = dict(dc=S(5, 40), a=S(5, 64), b=S(64, 40), preact=S(5, 40), da=S(5, 64), db=S(64, 40), dbias=S(40, dtype=0))
        a.update(kw)
        return call(L, "tcab_gemm_bias_act_backward", [a["dc"], a["a"], a["b"], a["preact"], act, a["da"], a["db"], a["dbias"], None, 0, None])

    assert back(preact=None) == _lib.ERR_INVALID_ARG and "preact" in message(L)
    assert back(dc=S(5, 48)) == _lib.ERR_SHAPE
    assert back(da=S(5, 40)) == _lib.ERR_SHAPE
    assert back(db=S(64, 40, dtype=0)) == _lib.ERR_DTYPE
    assert back(dbias=S(40)) == _lib.ERR_DTYPE
    assert back(act=5) == _lib.ERR_INVALID_ARG
    d = S(5, 40)
    assert back(dc=d, da=T_((5, 64), 1, d.data)) == _lib.ERR_INVALID_ARG


def test_gated_forms(tcab_lib):
    from tcacomp_b200 import _lib
    L, S = tcab_lib, Space()

    def fwd(act=2, **kw):
        a = dict(x=S(5, 64), w_gate=S(64, 40), w_up=S(64, 40), bg=S(40, dtype=0), bu=S(40, dtype=0), gate=S(5, 40), up=S(5, 40), h=S(5, 40))
        a.update(kw)
        return call(L, "tcab_gated_gemm", [a["x"], a["w_gate"], a["w_up"], a["bg"], a["bu"], act, a["gate"], a["up"], a["h"], None])

    assert fwd(w_up=S(64, 48)) == _lib.ERR_SHAPE
    assert fwd(bg=None) == _lib.ERR_INVALID_ARG and "both or neither" in message(L)
    assert fwd(up=None) == _lib.ERR_INVALID_ARG
    assert fwd(act=0) == _lib.ERR_INVALID_ARG and fwd(act=6) == _lib.ERR_INVALID_ARG
    h = S(5, 40)
    assert fwd(h=h, gate=h) == _lib.ERR_INVALID_ARG

    def back(act=2, **kw):
        a = dict(dh=S(5, 40), x=S(5, 64), w_gate=S(64, 40), w_up=S(64, 40), gate=S(5, 40), up=S(5, 40), dx=S(5, 64), dw_gate=S(64, 40),
                 dw_up=S(64, 40), dbg=None, dbu=None)
        a.update(kw)
        return call(L, "tcab_gated_gemm_backward", [a[n] for n in ("dh", "x", "w_gate", "w_up", "gate", "up")] + [act] +
                    [a[n] for n in ("dx", "dw_gate", "dw_up", "dbg", "dbu")] + [None, 0, None])

    assert back(dw_up=None) == _lib.ERR_INVALID_ARG and "both or neither" in message(L)
    assert back(dbg=S(40, dtype=0)) == _lib.ERR_INVALID_ARG
    assert back(gate=None) == _lib.ERR_INVALID_ARG
    assert back(act=0) == _lib.ERR_INVALID_ARG
    w = S(64, 40)
    assert back(w_gate=w, dw_gate=w) == _lib.ERR_INVALID_ARG


def test_without_a_device_and_python_arguments(tcab_lib):
    import tcacomp_b200 as T
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    g = torch.zeros(64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        T.layernorm_rows_stats(x, g, g)
    with pytest.raises(ValueError, match="CUDA"):
        T.gemm_bias_act_residual(x, torch.zeros(64, 8, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="unknown activation 'tanh'"):
        T.gemm_bias_act_residual(x, x, act="tanh")
    with pytest.raises(ValueError, match="unknown activation 'sigmoid'"):
        T.gemm_bias_act_backward(x, x, x, act="sigmoid")
    with pytest.raises(ValueError, match="unknown activation 'none'"):
        T.gated_gemm(x, x, x, act="none")
    with pytest.raises(ValueError, match="unknown activation"):
        T.gated_gemm_backward(x, x, x, x, x, x, act="swish")
    if torch.cuda.is_available():
        return
    from tcacomp_b200 import _lib
    S = Space()
    assert call(tcab_lib, "tcab_gated_gemm", [S(5, 64), S(64, 40), S(64, 40), None, None, 2, None, None, S(5, 40), None]) == _lib.ERR_CUDA
    assert call(tcab_lib, "tcab_gemm_bias_act_residual", [S(5, 64), S(64, 40), None, None, 0, None, S(5, 40), None]) == _lib.ERR_CUDA


def test_workspace_apart_from_the_tensors(tcab_lib):
    """A workspace that begins or ends inside a tensor of the call is refused; one that only touches it gets further."""
    from tcacomp_b200 import _lib
    L, S = tcab_lib, Space()
    dc, a, b, z, da, db = S(5, 40), S(5, 64), S(64, 40), S(5, 40), S(5, 64), S(64, 40)
    x, g, mean, rstd, dx = S(4, 64), S(64), S(4, dtype=0), S(4, dtype=0), S(4, 64)
    dg, dbt = S(64, dtype=0), S(64, dtype=0)
    h, gate, up, w1, w2, dw1, dw2 = S(5, 40), S(5, 40), S(5, 40), S(64, 40), S(64, 40), S(64, 40), S(64, 40)

    def gemm(ws, n):
        return call(L, "tcab_gemm_bias_act_backward", [dc, a, b, z, 3, da, db, None, ws, n, None])

    def norm(ws, n):
        return call(L, "tcab_layernorm_rows_backward", [dx, x, g, mean, rstd, dx, dg, dbt, ws, n, None])

    def gated(ws, n):
        return call(L, "tcab_gated_gemm_backward", [h, a, w1, w2, gate, up, 2, da, dw1, dw2, None, None, ws, n, None])

    for fn, tensors in ((gemm, {"dc": dc, "a": a, "preact": z, "db": db}), (norm, {"x": x, "rstd": rstd, "dgamma": dg}),
                        (gated, {"dh": h, "up": up, "w_up": w2, "dx": da, "dw_up": dw2})):
        for name, t in tensors.items():
            size = 4 * t.dims[0] if t.rank == 1 else 2 * t.dims[0] * t.dims[1]
            for ws in (t.data, t.data - 4080, t.data + size - 16):
                assert fn(ws, 4096) == _lib.ERR_INVALID_ARG and f"workspace overlaps {name}" in message(L), (name, ws - t.data)
            for ws in (t.data - 4096, t.data + size):
                fn(ws, 16)
                assert "workspace overlaps" not in message(L)


def test_extents_of_31_bits(tcab_lib):
    """With an empty contraction an extent may pass 31 bits without a tensor passing 2^32 elements."""
    from tcacomp_b200 import _lib
    L = tcab_lib
    far = 1 << 40
    n = (1 << 31) + 8
    a, b, c = T_((1, 0), 1, 0), T_((0, n), 1, 0), T_((1, n), 1, far)
    assert call(L, "tcab_gemm_bias_act_residual", [a, b, None, None, 0, None, c, None]) == _lib.ERR_TOO_LARGE and "2^31" in message(L)
    assert call(L, "tcab_gated_gemm", [a, b, b, None, None, 2, None, None, c, None]) == _lib.ERR_TOO_LARGE
    x, y, g, st = T_((1, n), 1, far), T_((1, n), 1, 2 * far), T_((n,), 1, 3 * far), T_((1,), 0, 4 * far)
    assert call(L, "tcab_layernorm_rows_stats", [x, g, T_((n,), 1, 5 * far), 1e-5, y, st, T_((1,), 0, 6 * far), None]) == _lib.ERR_TOO_LARGE


def test_outputs_asked_for_by_name(tcab_lib):
    import tcacomp_b200 as T
    x = torch.zeros(8, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="unknown output 'dx'"):
        T.gemm_bias_act_backward(x, x, x, x, "silu", want=("da", "dx"))
    with pytest.raises(ValueError, match="unknown output 'da'"):
        T.gated_gemm_backward(x, x, x, x, x, x, "silu", out={"da": x})
    for stream in (None, torch.cuda.ExternalStream(0) if torch.cuda.is_available() else None):
        with pytest.raises(ValueError, match="CUDA"):
            T.gated_gemm_backward(x, x, x, x, x, x, "silu", stream=stream)
    with pytest.raises(TypeError, match="x must be a torch.Tensor"):
        T.layernorm_rows_stats(None, x, x)
