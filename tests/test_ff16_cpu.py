"""The 16-bit feed-forward operators on the CPU: the torch statement of each
against the float64 oracle, the oracle's gradients against differences, the
refusals of the Python entry points, and the C ABI's argument checks (which
return before any launch)."""

from __future__ import annotations

import pytest
import torch
import torch.nn as nn

import diffucore_amd as D
from diffucore_amd import _ff16, _lib
from oracle import ff16 as O

ACTS = sorted(_ff16.ACTIVATIONS)


def _rand(*shape, seed=0, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def _within(got, want, bound, what):
    assert got.shape == want.shape, what
    off = (got.double() - want).abs() - bound
    assert bool((off <= 0).all()), f"{what}: off by {float(off.max()):.3g} past its bound"


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
def test_linear_act_on_cpu_tensors(act, dt):
    x, w, b = _rand(2, 3, 20, dtype=dt), _rand(7, 20, seed=1, dtype=dt, std=0.3), _rand(7, seed=2, dtype=dt)
    res, dy = _rand(2, 3, 7, seed=3, dtype=dt), _rand(2, 3, 7, seed=4, dtype=dt)
    leaves = [t.requires_grad_(True) for t in (x, w, b, res)]
    y = D.linear_act(x, w, b, act=act, residual=res)
    assert y.dtype == dt and y.shape == (2, 3, 7)
    want = O.linear(x.detach().double().view(6, 20), w.detach().double(), b.detach().double(), act,
                    res.detach().double().view(6, 7), dt, dy.double().view(6, 7))
    _within(y.detach().view(6, 7), *want["y"], "y")
    for name, g in zip(("dx", "dw", "db", "dres"), torch.autograd.grad(y, leaves, dy)):
        value, bound = want[name]
        _within(g.reshape(value.shape), value, bound + O.U[dt] * value.abs() * 4 + 1e-6, name)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("fused", [True, False])
def test_gated_linear_on_cpu_tensors(act, fused):
    x, wv, wg = _rand(5, 12), _rand(6, 12, seed=1), _rand(6, 12, seed=2)
    bv, bg = _rand(6, seed=3), _rand(6, seed=4)
    if fused:
        y = D.gated_linear(x, torch.cat([wv, wg]), torch.cat([bv, bg]), act=act)
    else:
        y = D.gated_linear(x, wv, bv, gate_weight=wg, gate_bias=bg, act=act)
    want = O.gated(*(t.double() for t in (x, wv, wg, bv, bg)), act, torch.float32)["y"]
    _within(y, *want, "y")


@pytest.mark.parametrize("affine", [True, False])
def test_layer_norm_on_cpu_tensors(affine):
    x = _rand(4, 33, dtype=torch.bfloat16)
    w, b = (_rand(33, seed=1), _rand(33, seed=2)) if affine else (None, None)
    want = O.layer_norm(x.double(), w.double() if affine else None, b.double() if affine else None, 1e-5,
                        torch.bfloat16)["y"]
    _within(D.layer_norm(x, w, b), *want, "y")


def _difference(f, x, v, h=1e-5):
    return float((f(x + h * v) - f(x - h * v)) / (2 * h))


@pytest.mark.parametrize("act", ACTS)
def test_oracle_gradients_against_differences(act):
    """Directional central differences of the float64 forwards: the error is
    h^2 / 6 times a third derivative plus 2^-53 / h, below 1e-7 of values of order 10."""
    x, w, b, dy = (_rand(*s, seed=i, dtype=torch.float64) for i, s in enumerate([(4, 6), (5, 6), (5,), (4, 5)]))
    wg, bg = _rand(5, 6, seed=7, dtype=torch.float64), _rand(5, seed=8, dtype=torch.float64)
    dt = torch.float32
    got = O.linear(x, w, b, act, None, dt, dy)
    for name, t, f in (("dx", x, lambda t: (O.linear(t, w, b, act, None, dt)["y"][0] * dy).sum()),
                       ("dw", w, lambda t: (O.linear(x, t, b, act, None, dt)["y"][0] * dy).sum()),
                       ("db", b, lambda t: (O.linear(x, w, t, act, None, dt)["y"][0] * dy).sum())):
        v = _rand(*t.shape, seed=9, dtype=torch.float64)
        assert abs(float((got[name][0] * v).sum()) - _difference(f, t, v)) < 1e-6, name
    got = O.gated(x, w, wg, b, bg, act, dt, dy)
    for name, i in (("dx", 0), ("dw", 1), ("dwg", 2), ("db", 3), ("dbg", 4)):
        args = [x, w, wg, b, bg]

        def f(t, i=i):
            return (O.gated(*args[:i], t, *args[i + 1:], act, dt)["y"][0] * dy).sum()
        v = _rand(*args[i].shape, seed=9, dtype=torch.float64)
        assert abs(float((got[name][0] * v).sum()) - _difference(f, args[i], v)) < 1e-6, name


def test_oracle_layer_norm_gradients_against_differences():
    x, w, b, dy = (_rand(*s, seed=i, dtype=torch.float64) for i, s in enumerate([(3, 9), (9,), (9,), (3, 9)]))
    got = O.layer_norm(x, w, b, 1e-5, torch.float32, dy)
    for name, i in (("dx", 0), ("dw", 1), ("db", 2)):
        args = [x, w, b]

        def f(t, i=i):
            return (O.layer_norm(*args[:i], t, *args[i + 1:], 1e-5, torch.float32)["y"][0] * dy).sum()
        v = _rand(*args[i].shape, seed=9, dtype=torch.float64)
        assert abs(float((got[name][0] * v).sum()) - _difference(f, args[i], v)) < 1e-6, name


def test_geglu_ff_matches_the_module():
    proj, out = nn.Linear(16, 48), nn.Linear(24, 16)
    x = _rand(2, 5, 16)
    v, g = proj(x).chunk(2, dim=-1)
    ref = out(v * torch.nn.functional.gelu(g)) + x
    assert torch.allclose(D.geglu_ff(x, proj, out, residual=x), ref, atol=1e-5)


def test_empty_inputs():
    w, b = _rand(6, 8), _rand(6)
    assert D.linear_act(_rand(0, 8), w, b, act="silu").shape == (0, 6)
    assert D.gated_linear(_rand(2, 0, 8), w, b).shape == (2, 0, 3)
    assert D.layer_norm(_rand(0, 8)).shape == (0, 8)
    assert D.linear_act(_rand(3, 8), _rand(0, 8)).shape == (3, 0)


@pytest.mark.parametrize("call, error, match", [
    (lambda x, w, b: D.linear_act(x, w, b, act="relu6"), ValueError, "act must be one of"),
    (lambda x, w, b: D.gated_linear(x, w, b, act="geglu"), ValueError, "act must be one of"),
    (lambda x, w, b: D.linear_act(x.double(), w.double()), TypeError, "x is"),
    (lambda x, w, b: D.gated_linear(x.double(), w.double()), TypeError, "x is"),
    (lambda x, w, b: D.linear_act(x.int(), w.int()), TypeError, "x is"),
    (lambda x, w, b: D.linear_act(x, w.t(), b), ValueError, "weight is"),
    (lambda x, w, b: D.linear_act(x, w[0], b), ValueError, "1-dimensional"),
    (lambda x, w, b: D.linear_act(x, w, b[:3]), ValueError, "bias is"),
    (lambda x, w, b: D.linear_act(x, w.double(), b), TypeError, "weight is"),
    (lambda x, w, b: D.linear_act(x, w, b.int()), TypeError, "bias is"),
    (lambda x, w, b: D.linear_act(x, w, b, residual=torch.zeros(6)), ValueError, "residual is"),
    (lambda x, w, b: D.linear_act(x, w, b, residual=torch.zeros(4, 6, dtype=torch.float64)), TypeError, "residual"),
    (lambda x, w, b: D.linear_act(x, w.to("meta"), b), ValueError, "weight is on"),
    (lambda x, w, b: D.linear_act(x.to("meta"), w.to("meta")), RuntimeError, "GPU and CPU"),
    (lambda x, w, b: D.linear_act(torch.zeros(4, 0), torch.zeros(6, 0)), ValueError, "empty"),
    (lambda x, w, b: D.linear_act(torch.tensor(1.0), w), ValueError, "at least one dim"),
    (lambda x, w, b: D.gated_linear(x, w[:5], b[:5]), ValueError, "value and gate halves"),
    (lambda x, w, b: D.gated_linear(x, w, b, gate_bias=b), ValueError, "gate_bias goes with"),
    (lambda x, w, b: D.gated_linear(x, w, b, gate_weight=w[:4]), ValueError, "gate_weight is"),
    (lambda x, w, b: D.gated_linear(x.half(), w.half(), b, gate_weight=w.half(), gate_bias=b.half()), TypeError,
     "gate_bias"),
    (lambda x, w, b: D.layer_norm(x, b), ValueError, "weight is"),
    (lambda x, w, b: D.layer_norm(x, x[0], x[0].half()), TypeError, "weight is"),
    (lambda x, w, b: D.layer_norm(x.double()), TypeError, "x is"),
    (lambda x, w, b: D.layer_norm(torch.zeros(4, 0)), ValueError, "empty"),
])
def test_refusals(call, error, match):
    x, w, b = _rand(4, 8), _rand(6, 8, seed=1), _rand(6, seed=2)
    with pytest.raises(error, match=match):
        call(x, w, b)


# ---------------------------------------------------------------- C ABI argument checks

P = 1 << 20   # a 16-byte aligned address that no check may read


def _rc(name, *args):
    so = _lib.lib()
    if so is None:
        pytest.skip("library not built")
    rc = getattr(so, name)(*args)
    return rc, so.dc_last_error().decode()


def _linear(x=P, ldx=64, w=P, ldw=64, bias=None, bdt=-1, res=None, ldr=0, act=0, out=P, ldo=32, z=None, dt=1, M=4,
            N=32, K=64, ws=None, n=0):
    return _rc("dc_linear16", x, ldx, w, ldw, bias, bdt, res, ldr, act, out, ldo, z, dt, M, N, K, ws, n, None)


def _gated(x=P, ldx=64, wv=P, wg=P, ldw=64, bv=None, bg=None, bdt=-1, act=1, out=P, ldo=32, zv=None, zg=None,
           dt=0, M=4, N=32, K=64, ws=None, n=0):
    return _rc("dc_gated16", x, ldx, wv, ldw, wg, ldw, bv, bg, bdt, act, out, ldo, zv, zg, dt, M, N, K, ws, n, None)


def _lbwd(dy=P, ldy=32, x=P, ldx=64, w=P, ldw=64, z=P, act=1, dx=P, lddx=64, dw=P, lddw=64, db=P, ddt=0, dt=1,
          M=4, N=32, K=64, ws=P, n=1 << 30):
    return _rc("dc_linear16_bwd", dy, ldy, x, ldx, w, ldw, z, act, dx, lddx, dw, lddw, db, ddt, dt, M, N, K, ws, n,
               None)


def _gbwd(dy=P, ldy=32, x=P, ldx=64, w=P, ldw=64, wg=P, zv=P, zg=P, act=1, dx=P, lddx=64, dw=P, dwg=P, lddw=64,
          db=P, dbg=P, ddt=0, dt=1, M=4, N=32, K=64, ws=P, n=1 << 30):
    return _rc("dc_gated16_bwd", dy, ldy, x, ldx, w, ldw, wg, ldw, zv, zg, act, dx, lddx, dw, dwg, lddw, db, dbg,
               ddt, dt, M, N, K, ws, n, None)


def _norm(x=P, ldx=8, xdt=0, w=None, b=None, wdt=-1, y=P, ldy=8, stats=None, M=4, D_=8):
    return _rc("dc_layer_norm", x, ldx, xdt, w, b, wdt, 1e-5, y, ldy, stats, M, D_, None)


@pytest.mark.parametrize("call, kw, code, match", [
    (_linear, dict(M=-1), 1, "bad M/N/K"), (_linear, dict(M=1 << 30), 1, "too large"),
    (_linear, dict(N=1 << 29), 1, "too large"), (_linear, dict(K=1 << 22, ldx=1 << 22), 1, "too large"),
    (_linear, dict(dt=2), 1, "dtype"), (_linear, dict(act=3), 1, "act"), (_linear, dict(K=0), 1, "bad M/N/K"),
    (_linear, dict(x=None), 1, "null"), (_linear, dict(out=None), 1, "null"),
    (_linear, dict(bias=P, bdt=3), 1, "bias_dtype"), (_linear, dict(bias=P, bdt=0, dt=1), 1, "bias_dtype"),
    (_linear, dict(ldo=31), 1, "stride"),
    (_linear, dict(res=P, ldr=8), 1, "stride"), 
    (_linear, dict(ldx=63), 1, "stride"), (_linear, dict(ldw=56), 1, "stride"),
    (_linear, dict(M=40, K=60, ldx=60, ldw=60), 4, "needs"), (_linear, dict(M=40, ldx=68), 4, "needs"),
    (_linear, dict(M=40, x=P + 8), 4, "needs"), (_linear, dict(M=40, x=P + 8, ws=P + 8, n=1 << 20), 4, "aligned"),
    (_linear, dict(M=0, x=None), 0, ""), (_linear, dict(N=0), 0, ""),
    (_gated, dict(wg=None), 1, "null"), (_gated, dict(act=3), 1, "act"), (_gated, dict(zv=P), 1, "together"),
    (_gated, dict(bg=P, bdt=-1), 1, "bias_dtype"), (_gated, dict(M=40, wg=P + 2), 4, "needs"),
    (_gated, dict(M=0), 0, ""), (_gated, dict(K=0), 1, "bad M/N/K"), (_gated, dict(dt=2), 1, "dtype"),
    (_lbwd, dict(z=None), 1, "null"), (_lbwd, dict(dy=None), 1, "null"), (_lbwd, dict(ldy=31), 1, "stride"),
    (_lbwd, dict(lddx=60), 1, "stride"), (_lbwd, dict(lddw=60), 1, "stride"),
    (_lbwd, dict(ddt=3), 1, "db_dtype"), (_lbwd, dict(n=64), 4, "needs"), (_lbwd, dict(ws=P + 8), 4, "aligned"),
    (_lbwd, dict(K=0), 1, "bad M/N/K"), (_lbwd, dict(dt=2), 1, "dtype"), (_lbwd, dict(act=9), 1, "act"),
    (_lbwd, dict(dx=None, dw=None, db=None, ws=None, n=0), 0, ""),
    (_lbwd, dict(M=0, dw=None, db=None, dy=None), 0, ""),
    (_gbwd, dict(zg=None), 1, "null"), (_gbwd, dict(wg=None), 1, "null"), 
    (_gbwd, dict(lddw=60, dwg=None), 1, "stride"), (_gbwd, dict(ddt=-1, dbg=None), 1, "db_dtype"),
    (_gbwd, dict(ws=None), 4, "needs"), (_gbwd, dict(dt=3), 1, "dtype"),
    (_gbwd, dict(dx=None, dw=None, dwg=None, db=None, dbg=None, ws=None, n=0), 0, ""),
    (_norm, dict(M=-1), 1, "M must be"), (_norm, dict(D_=0), 1, "D 1"), (_norm, dict(D_=(1 << 24) + 1), 1, "2\\^24"),
    (_norm, dict(xdt=3), 1, "x_dtype"), (_norm, dict(w=P, wdt=3), 1, "w_dtype"), (_norm, dict(y=None), 1, "null"),
    (_norm, dict(ldx=7), 1, "stride"), (_norm, dict(M=0, x=None), 0, ""),
])
def test_c_abi_refusals(call, kw, code, match):
    rc, msg = call(**kw)
    assert rc == code
    if code:
        import re
        assert re.search(match, msg), msg


def test_c_abi_layer_norm_bwd():
    rc, msg = _rc("dc_layer_norm_bwd", P, 8, P, 8, 0, None, 0, P, None, 8, P, P, 4, 8, None, 0, None)
    assert rc == 4 and "workspace" in msg
    rc, msg = _rc("dc_layer_norm_bwd", P, 7, P, 8, 0, None, 0, P, P, 8, None, None, 4, 8, None, 0, None)
    assert rc == 1 and "stride" in msg
    rc, msg = _rc("dc_layer_norm_bwd", P, 8, P, 8, 0, None, 0, None, P, 8, None, None, 4, 8, None, 0, None)
    assert rc == 1 and "null" in msg
    assert _rc("dc_layer_norm_bwd", P, 8, P, 8, 0, None, 0, P, None, 8, None, None, 4, 8, None, 0, None)[0] == 0


def test_workspace_queries_cover_padded_operands():
    """An operand that has to be copied adds its padded size; aligned ones of a
    shape that is not split add nothing."""
    so = _lib.lib()
    if so is None:
        pytest.skip("library not built")
    M, N, K = 4096, 4096, 2048
    assert so.dc_saved16_bytes(5, 7) == 105 and so.dc_saved16_bytes(0, 7) == 0
    q = so.dc_linear16_workspace_bytes
    assert q(P, K, P, K, M, N, K) == 0
    assert q(P + 2, K, P, K, M, N, K) == 2 * M * K
    assert q(P, K + 1, P + 2, K, M, N, K) == 2 * (M + N) * K
    assert q(P, K - 1, P, K - 1, M, N, K - 1) == 2 * (M + N) * K
    g = so.dc_gated16_workspace_bytes
    assert g(P, K, P, K, P + 2, K, M, N, K) == 2 * N * K
    b = so.dc_linear16_bwd_workspace_bytes
    assert b(P, N, P, K, P, K, 0, 1, M, N, K) == 0
    assert b(P, N, P, K, P, K, 1, 1, M, N, K) == 2 * M * N   # dz
    assert q(P, 0, P, 0, 0, N, K) == 0 and b(P, 0, P, 0, P, 0, 0, 15, M, N, 0) == 0
