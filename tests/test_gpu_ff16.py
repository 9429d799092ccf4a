"""The 16-bit feed-forward operators on the GPU against float64, element by
element within the oracle's derived bounds (``oracle/ff16.py``): sizes from one
row to many, odd and ragged widths, strides and alignments, both weight
layouts, every gradient; then what calls share - streams, captured graphs,
repeated and concurrent use - and a sublayer made of all three."""

from __future__ import annotations

import pytest
import torch
import torch.nn as nn

import diffucore_amd as D
from diffucore_amd import _ff16
from oracle import ff16 as O

pytestmark = pytest.mark.gpu
ACTS = sorted(_ff16.ACTIVATIONS)
DTYPES = [torch.bfloat16, torch.float16]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rand(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def _within(got, want, what):
    value, bound = want
    assert got.numel() == value.numel(), what
    got = got.detach().double().reshape(value.shape)
    off = (got - value).abs() - bound
    assert bool((off <= 0).all()), f"{what}: {int((off > 0).sum())} past the bound, worst by {float(off.max()):.3g}"


def _check_linear(M, K, N, dt, act, bias=True, res=False, seed=0, bias_dt=None, x=None, w=None, dy=None, r=None):
    print(f"[ff16] linear {M} x {K} -> {N} {dt} {act} bias={bias} res={res}", flush=True)
    g = _gen(seed)
    x = _rand(g, M, K, dtype=dt) if x is None else x
    w = _rand(g, N, K, dtype=dt, std=K ** -0.5) if w is None else w
    b = _rand(g, N, dtype=bias_dt or dt, std=0.3) if bias else None
    r = (_rand(g, M, N, dtype=dt) if r is None else r) if res else None
    dy = _rand(g, M, N, dtype=dt) if dy is None else dy
    f = lambda t: None if t is None else t.double()   # noqa: E731
    want = O.linear(f(x), f(w), f(b), act, f(r), dt, f(dy), bias_dt)
    with torch.no_grad():
        _within(D.linear_act(x, w, b, act=act, residual=r), want["y"], "y")
    named = [("dx", x), ("dw", w), ("db", b), ("dres", r)]
    leaves = [t.detach().requires_grad_(True) if t is not None else None for _, t in named]
    y = D.linear_act(leaves[0], leaves[1], leaves[2], act=act, residual=leaves[3])
    _within(y, want["y"], "y (training)")
    live = [(n, t) for (n, _), t in zip(named, leaves) if t is not None]
    for (n, t), grad in zip(live, torch.autograd.grad(y, [t for _, t in live], dy)):
        assert grad.dtype == t.dtype and grad.shape == t.shape
        _within(grad, want[n], n)


def _check_gated(M, K, N, dt, act, bias=True, fused=True, seed=0, bias_dt=None, x=None):
    print(f"[ff16] gated {M} x {K} -> {N} {dt} {act} bias={bias} fused={fused}", flush=True)
    g = _gen(seed)
    x = _rand(g, M, K, dtype=dt) if x is None else x
    w = _rand(g, 2 * N, K, dtype=dt, std=K ** -0.5)
    b = _rand(g, 2 * N, dtype=bias_dt or dt, std=0.3) if bias else None
    dy = _rand(g, M, N, dtype=dt)
    wd, bd = w.double(), [None, None] if b is None else b.double().chunk(2)
    want = O.gated(x.double(), wd[:N], wd[N:], bd[0], bd[1], act, dt, dy.double(), bias_dt)
    leaf = lambda t: None if t is None else t.detach().clone().requires_grad_(True)   # noqa: E731
    x = x.detach().requires_grad_(True)
    if fused:
        w, b = leaf(w), leaf(b)
        call = lambda: D.gated_linear(x, w, b, act=act)   # noqa: E731
        live = [("dx", x), ("dw", w), ("db", b)]
    else:
        wv, wg = leaf(w[:N]), leaf(w[N:])
        bv, bg = (None, None) if b is None else (leaf(b[:N]), leaf(b[N:]))
        call = lambda: D.gated_linear(x, wv, bv, gate_weight=wg, gate_bias=bg, act=act)   # noqa: E731
        live = [("dx", x), ("dw", wv), ("db", bv), ("dwg", wg), ("dbg", bg)]
    with torch.no_grad():
        _within(call(), want["y"], "y")
    y = call()
    _within(y, want["y"], "y (training)")
    live = [(n, t) for n, t in live if t is not None]
    for (n, t), grad in zip(live, torch.autograd.grad(y, [t for _, t in live], dy)):
        assert grad.dtype == t.dtype and grad.shape == t.shape
        if fused and n in ("dw", "db"):
            _within(grad[:N], want[n], n)
            _within(grad[N:], want[n + "g"], n + "g")
        else:
            _within(grad, want[n], n)


def _check_norm(M, D_, dt, wt=None, affine=(True, True), seed=0, x=None, offset=0.5, dy=None):
    print(f"[ff16] layer_norm {M} x {D_} {dt} w {wt} {affine}", flush=True)
    g = _gen(seed)
    x = (_rand(g, M, D_) + _rand(g, M, 1, std=offset)).to(dt) if x is None else x
    wt = wt or dt
    w = (1 + _rand(g, D_, std=0.3)).to(wt) if affine[0] else None
    b = _rand(g, D_, dtype=wt, std=0.3) if affine[1] else None
    dy = _rand(g, M, D_, dtype=dt) if dy is None else dy
    f = lambda t: None if t is None else t.double()   # noqa: E731
    want = O.layer_norm(f(x), f(w), f(b), 1e-5, dt, f(dy), wt)
    _within(D.layer_norm(x, w, b, 1e-5), want["y"], "y")
    live = [(n, t.detach().requires_grad_(True)) for n, t in (("dx", x), ("dw", w), ("db", b)) if t is not None]
    got = dict(live)
    y = D.layer_norm(got["dx"], got.get("dw"), got.get("db"), 1e-5)
    _within(y, want["y"], "y (training)")
    for (n, t), grad in zip(live, torch.autograd.grad(y, [t for _, t in live], dy)):
        assert grad.dtype == t.dtype and grad.shape == t.shape
        _within(grad, want[n], n)


# ---------------------------------------------------------------- sizes

@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M", [1, 2, 7, 16, 17, 33, 64, 65, 154, 300, 1030])
def test_linear_rows(gpu, M, dt):
    _check_linear(M, 320, 640, dt, "silu", res=True, seed=M)


@pytest.mark.parametrize("K, N", [(8, 8), (1, 1), (3, 5), (16, 1), (40, 72), (63, 65), (64, 64), (127, 257), (128, 136),
                                  (200, 1000), (1155, 577), (2560, 640), (4096, 48), (24, 4000)])
@pytest.mark.parametrize("M", [1, 19, 260])
def test_linear_widths(gpu, M, K, N):
    _check_linear(M, K, N, DTYPES[(M + K) % 2], ACTS[(K + N) % len(ACTS)], res=(K + M) % 2 == 0, seed=K + N)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias, res", [(False, False), (True, False), (False, True)])
def test_linear_activations(gpu, act, bias, res, dt):
    _check_linear(130, 96, 264, dt, act, bias, res)
    _check_linear(3, 96, 264, dt, act, bias, res)


@pytest.mark.parametrize("M, K, N", [(2048, 1280, 1280), (515, 2048, 2600), (4096, 640, 640), (100, 5120, 1280),
                                     (9000, 72, 328), (40, 8192, 264)])
@pytest.mark.parametrize("dt", DTYPES)
def test_linear_large(gpu, M, K, N, dt):
    _check_linear(M, K, N, dt, "gelu_tanh", res=True)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M", [3, 130])
def test_gated_activations(gpu, act, M):
    _check_gated(M, 96, 136, DTYPES[M % 2], act)
    _check_gated(M, 1024, 136, DTYPES[1 - M % 2], act, bias=False, fused=False)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("M", [1, 5, 16, 17, 40, 128, 333, 1100])
def test_gated_rows(gpu, M, fused, dt):
    _check_gated(M, 320, 272, dt, "gelu", fused=fused, seed=M)


@pytest.mark.parametrize("K, N", [(8, 8), (1, 1), (5, 3), (16, 2), (40, 72), (63, 65), (64, 32), (127, 257),
                                  (1000, 2731), (2560, 640), (24, 2000)])
@pytest.mark.parametrize("M", [1, 19, 260])
def test_gated_widths(gpu, M, K, N):
    act = ACTS[(K + N) % len(ACTS)]
    _check_gated(M, K, N, DTYPES[(M + K) % 2], act, bias=(K + M) % 3 != 0, fused=(K + N + M) % 2 == 0, seed=K + N)


@pytest.mark.parametrize("M, K, N", [(2048, 640, 2560), (515, 1280, 1300), (4100, 320, 1280)])
@pytest.mark.parametrize("dt", DTYPES)
def test_gated_large(gpu, M, K, N, dt):
    _check_gated(M, K, N, dt, "gelu")


@pytest.mark.parametrize("D_", [1, 2, 7, 8, 9, 63, 64, 65, 320, 333, 384, 385, 640, 768, 1280, 1536, 1537, 2048, 2731,
                                3079, 5120, 6144, 6145, 12288, 12289, 16384, 20001])
@pytest.mark.parametrize("M", [1, 37])
def test_norm_widths(gpu, M, D_):
    _check_norm(M, D_, DTYPES[D_ % 2], seed=D_)
    _check_norm(M, D_, torch.float32, seed=D_)


@pytest.mark.parametrize("dt", [*DTYPES, torch.float32])
@pytest.mark.parametrize("wt", [*DTYPES, torch.float32])
def test_norm_types(gpu, dt, wt):
    _check_norm(50, 328, dt, wt)
    _check_norm(5, 13000, dt, wt)


@pytest.mark.parametrize("affine", [(False, False), (True, False), (False, True)])
def test_norm_without_parameters(gpu, affine):
    _check_norm(21, 640, torch.bfloat16, affine=affine)
    _check_norm(3, 13001, torch.float32, affine=affine)


@pytest.mark.parametrize("M, D_", [(4999, 640), (33000, 24), (700, 5000), (600, 13312)])
def test_norm_many_rows(gpu, M, D_):
    _check_norm(M, D_, torch.bfloat16, torch.float32)


def test_norm_of_an_offset_stream(gpu):
    """Means a thousand deviations out: the squared deviations are taken from
    the mean, so nothing cancels (float32; the bound carries the mean's error)."""
    _check_norm(64, 640, torch.float32, offset=1000.0)


# ---------------------------------------------------------------- strides and alignment

def _strided(g, M, W, dt, how):
    if how == "pad8":
        return _rand(g, M, W + 8, dtype=dt)[:, :W]
    if how == "odd":
        return _rand(g, M, W + 5, dtype=dt)[:, :W]
    if how == "offset":
        return _rand(g, M, W + 16, dtype=dt)[:, 3:3 + W]
    if how == "transposed":
        return _rand(g, W, M, dtype=dt).t()
    if how == "rows2":
        return _rand(g, 2 * M, W, dtype=dt)[::2]
    if how == "flip":
        return _rand(g, M, W, dtype=dt).flip(0)
    assert how == "expand"
    return _rand(g, 1, W, dtype=dt).expand(M, W)


HOW = ["pad8", "odd", "offset", "transposed", "rows2", "expand"]


@pytest.mark.parametrize("how", HOW)
@pytest.mark.parametrize("M", [1, 5, 140])
def test_strides(gpu, M, how):
    g = _gen(5)
    dt = torch.bfloat16
    _check_linear(M, 96, 72, dt, "gelu", res=True, x=_strided(g, M, 96, dt, how), r=_strided(g, M, 72, dt, how),
                  dy=_strided(g, M, 72, dt, how))
    _check_linear(M, 96, 72, dt, "none", x=_strided(g, M, 96, dt, how), w=_strided(g, 72, 96, dt, how),
                  dy=_strided(g, M, 72, dt, how))
    _check_gated(M, 96, 40, dt, "silu", x=_strided(g, M, 96, dt, how))
    _check_norm(M, 96, dt, x=_strided(g, M, 96, dt, how), dy=_strided(g, M, 96, dt, how))


def test_leading_dims_and_parameter_strides(gpu):
    g = _gen(6)
    x = _rand(g, 2, 3, 5, 64, dtype=torch.float16)
    w = _rand(g, 48, 64, dtype=torch.float16, std=0.1)
    b = _rand(g, 96, dtype=torch.float16)[::2]
    y = D.linear_act(x.transpose(0, 1), w, b, act="gelu")
    ref = D.linear_act(x.transpose(0, 1).contiguous(), w, b.contiguous(), act="gelu")
    assert y.shape == (3, 2, 5, 48) and torch.equal(y, ref)
    p = _rand(g, 128)[::2]
    assert torch.equal(D.layer_norm(x, p, p), D.layer_norm(x, p.contiguous(), p.contiguous()))
    v = _rand(g, 64, dtype=torch.float16)
    assert D.linear_act(v, w).shape == (48,) and D.layer_norm(v).shape == (64,)


@pytest.mark.parametrize("act", ["none", "gelu"])
def test_float32_bias(gpu, act):
    _check_linear(70, 64, 72, torch.bfloat16, act, bias_dt=torch.float32)
    _check_gated(70, 64, 72, torch.float16, "silu", bias_dt=torch.float32, fused=True)
    _check_gated(2, 64, 72, torch.float16, "silu", bias_dt=torch.float32, fused=False)


# ---------------------------------------------------------------- values

@pytest.mark.parametrize("M", [2, 80])
def test_infinities_and_nan_stay_in_their_rows(gpu, M):
    g = _gen(7)
    dt = torch.bfloat16
    x = _rand(g, M, 128, dtype=dt)
    w = _rand(g, 64, 128, dtype=dt, std=0.1)
    clean = {"linear": D.linear_act(x, w, act="gelu"), "gated": D.gated_linear(x, w), "norm": D.layer_norm(x)}
    bad = x.clone()
    bad[1, 3] = float("nan")
    got = {"linear": D.linear_act(bad, w, act="gelu"), "gated": D.gated_linear(bad, w), "norm": D.layer_norm(bad)}
    for name in clean:
        assert got[name][1].isnan().all(), name
        keep = [i for i in range(M) if i != 1]
        assert torch.equal(got[name][keep], clean[name][keep]), name
    bad[1, 3] = float("inf")
    y = D.linear_act(bad, w)
    assert torch.equal(y[1].float(), torch.where(w[:, 3] > 0, float("inf"), float("-inf")).float())


@pytest.mark.parametrize("F_, K", [(40, 72), (70, 200), (127, 65), (300, 264)])
@pytest.mark.parametrize("half", [0, 1])
def test_infinite_weights_reach_their_column_only(gpu, half, F_, K):
    """An infinite weight in a half's last row, where the product's sum over
    that half ends inside a stage of 64: dx's column is infinite with the sign
    of its dz, never NaN, and the others stay as they are without it."""
    g = _gen(12)
    dt = torch.bfloat16
    x = _rand(g, 70, K, dtype=dt).requires_grad_(True)
    w = _rand(g, 2 * F_, K, dtype=dt, std=0.1)
    dy = _rand(g, 70, F_, dtype=dt)
    clean, = torch.autograd.grad(D.gated_linear(x, w, act="silu"), [x], dy)
    y = D.gated_linear(x, w, act="silu")
    v, gate = (t[:, -1] for t in (x.detach().double() @ w.double().T).chunk(2, dim=1))
    a, slope = O.act(gate, "silu")
    dz = dy[:, -1].double() * (v * slope if half else a)
    w.data[(1 + half) * F_ - 1, 1] = float("inf")   # after the forward: its pre-activations stay finite
    got, = torch.autograd.grad(y, [x], dy)
    keep = [c for c in range(K) if c != 1]
    assert torch.equal(got[:, keep], clean[:, keep])
    assert torch.equal(got[:, 1].double(), torch.sign(dz) * float("inf"))


@pytest.mark.parametrize("act", [a for a in ACTS if a != "none"])
def test_far_out_pre_activations(gpu, act):
    """Values where x s (1 - s) or x phi(x) would turn into inf * 0: slopes
    are 0 or 1 there, and products past fp16's range end as inf, never NaN."""
    for dt, big in ((torch.bfloat16, 1e30), (torch.float16, 6e4)):
        x = torch.tensor([[big], [-big], [100.0], [-100.0], [0.0]], device="cuda", dtype=dt).requires_grad_(True)
        w = torch.ones(8, 1, device="cuda", dtype=dt).requires_grad_(True)
        y = D.linear_act(x, w, act=act)
        assert torch.equal(y[:, 0].float(), torch.relu(x.detach().float())[:, 0])
        dx, = torch.autograd.grad(y, [x], torch.ones_like(y))
        assert dx[:, 0].tolist() == [8.0, 0.0, 8.0, 0.0, 4.0]
    x = torch.full((3, 16), 200.0, device="cuda", dtype=torch.float16).requires_grad_(True)
    w = torch.full((4, 16), 100.0, device="cuda", dtype=torch.float16)   # value 320000: past fp16
    wg = torch.full((4, 16), -1.0, device="cuda", dtype=torch.float16)   # gate -3200: act and slope 0
    y = D.gated_linear(x, w, gate_weight=wg, act=act)
    dx, = torch.autograd.grad(y, [x], torch.ones_like(y))
    assert bool((y == 0).all()) and bool((dx == 0).all())


def test_empty_calls(gpu):
    w = torch.randn(6, 8, device="cuda", dtype=torch.float16).requires_grad_(True)
    b = torch.randn(6, device="cuda", dtype=torch.float16).requires_grad_(True)
    x = torch.zeros(0, 8, device="cuda", dtype=torch.float16).requires_grad_(True)
    r = torch.zeros(0, 6, device="cuda", dtype=torch.float16).requires_grad_(True)
    for y, leaves in ((D.linear_act(x, w, b, act="silu", residual=r), [x, w, b, r]),
                      (D.gated_linear(x, w, b), [x, w, b]),
                      (D.layer_norm(x, w[0], b[:1].expand(8)), [x, w, b])):
        assert y.shape[0] == 0
        for t, grad in zip(leaves, torch.autograd.grad(y, leaves, torch.zeros_like(y))):
            assert grad.shape == t.shape and not bool(grad.any())
    assert D.linear_act(torch.zeros(3, 8, device="cuda", dtype=torch.float16), w[:0]).shape == (3, 0)


def test_gpu_refusals(gpu):
    x, w = torch.zeros(4, 8, device="cuda"), torch.zeros(6, 8, device="cuda")
    with pytest.raises(TypeError, match="fp16 or bf16"):
        D.linear_act(x, w)
    with pytest.raises(TypeError, match="fp16 or bf16"):
        D.gated_linear(x, w)
    with pytest.raises(ValueError, match="weight is on"):
        D.linear_act(x.half(), w.half().cpu())
    with pytest.raises(ValueError, match="bias is on"):
        D.layer_norm(x, bias=torch.zeros(8))


# ---------------------------------------------------------------- random shapes

def random_call(seed):
    """One call of random sizes (over their logarithm, every third one a
    multiple of 64), types, layout and strides, checked in full."""
    import random
    rng = random.Random(seed)
    size = lambda lo, hi: int(2.0 ** rng.uniform(lo, hi))   # noqa: E731
    wide = lambda lo, hi: size(lo, hi) if rng.random() < 2 / 3 else -(-size(lo, hi) // 64) * 64   # noqa: E731
    dt = rng.choice(DTYPES)
    kind = rng.choice(["linear", "gated", "norm"])
    M = size(0, 11.5)
    if kind == "norm":
        dt = rng.choice([*DTYPES, torch.float32])
        return _check_norm(M, wide(0, 14), dt, rng.choice([None, torch.float32]), seed=seed)
    K, N = wide(0, 11.5), wide(0, 11.5)
    g = _gen(seed)
    pad = rng.choice([0, 0, 8, 3])
    x = _rand(g, M, K + pad, dtype=dt)[:, :K]
    bias_dt = rng.choice([None, torch.float32])
    if kind == "linear":
        return _check_linear(M, K, N, dt, rng.choice(ACTS), rng.random() < 0.7, rng.random() < 0.5, seed, bias_dt, x=x)
    return _check_gated(M, K, N, dt, rng.choice(ACTS), rng.random() < 0.7, rng.random() < 0.5, seed, bias_dt, x=x)


@pytest.mark.parametrize("seed", range(60))
def test_random_calls(gpu, seed):
    random_call(seed)


# ---------------------------------------------------------------- past 32 bits

def test_layer_norm_past_32_bits(gpu):
    """2.2e9 elements: the last rows equal a call on them alone."""
    M, D_ = 270000, 8192
    x = torch.empty(M, D_, device="cuda", dtype=torch.bfloat16)
    x[:64].normal_()
    x[-64:].normal_()
    x[64:-64] = x[0]
    w = torch.randn(D_, device="cuda")
    y = D.layer_norm(x, w)
    for rows in (slice(0, 64), slice(M - 64, M)):
        assert torch.equal(y[rows], D.layer_norm(x[rows], w))
    t = x.requires_grad_(True)
    dx, = torch.autograd.grad(D.layer_norm(t, w), [t], y)
    tail = x[-64:].detach().requires_grad_(True)
    want, = torch.autograd.grad(D.layer_norm(tail, w), [tail], y[-64:])
    assert torch.equal(dx[-64:], want)


def test_products_past_32_bits(gpu):
    """An input of 2.4e9 elements and, the other way round, an output of as
    many: their last rows equal calls on those rows alone (each output is summed
    in the same order on every tile, so the bits agree)."""
    M, K, N = 300000, 8192, 64
    g = _gen(13)
    x = torch.empty(M, K, device="cuda", dtype=torch.bfloat16)
    x[-512:] = _rand(g, 512, K, dtype=torch.bfloat16)
    x[:-512] = x[-1]
    w = _rand(g, N, K, dtype=torch.bfloat16, std=0.02)
    y = D.linear_act(x, w, act="gelu")
    f = lambda t: t.double()   # noqa: E731
    want = O.linear(f(x[-512:]), f(w), None, "gelu", None, torch.bfloat16)
    _within(y[-512:], want["y"], "y")
    t = x.requires_grad_(True)
    dy = torch.zeros(M, N, device="cuda", dtype=torch.bfloat16)
    dy[-512:] = _rand(g, 512, N, dtype=torch.bfloat16)
    lw = w.detach().requires_grad_(True)
    dx, dw = torch.autograd.grad(D.linear_act(t, lw, act="gelu"), [t, lw], dy)
    want = O.linear(f(x[-512:].detach()), f(w), None, "gelu", None, torch.bfloat16, f(dy[-512:]))
    _within(dx[-512:], want["dx"], "dx")
    assert not bool(dx[:-512].any())
    _within(dw, want["dw"], "dw")   # the other rows' gradients are 0
    del dx, t, x
    wide = _rand(g, K, N, dtype=torch.bfloat16, std=0.1)
    h = y.detach()
    out = D.gated_linear(h, wide, gate_weight=wide)
    want = O.gated(f(h[-512:]), f(wide), f(wide), None, None, "gelu", torch.bfloat16)
    _within(out[-512:], want["y"], "gated y")


def test_huge_row_strides(gpu):
    """Rows 2^22 elements and more apart (32-bit offsets within a tile would not
    reach them) are copied first."""
    g = _gen(14)
    big = torch.empty(40, (1 << 22) + 8, device="cuda", dtype=torch.float16)
    big[:, :64] = _rand(g, 40, 64, dtype=torch.float16)
    x = big[:, :64]
    w = _rand(g, 72, 64, dtype=torch.float16, std=0.1)
    assert torch.equal(D.linear_act(x, w, act="silu"), D.linear_act(x.contiguous(), w, act="silu"))
    a, b = (t.detach().requires_grad_(True) for t in (x, x.contiguous()))
    dy = _rand(g, 40, 72, dtype=torch.float16)
    lw = w.requires_grad_(True)
    for p, q in zip(torch.autograd.grad(D.linear_act(a, lw), [a, lw], dy),
                    torch.autograd.grad(D.linear_act(b, lw), [b, lw], dy)):
        assert torch.equal(p, q)
    assert torch.equal(D.layer_norm(x), D.layer_norm(x.contiguous()))


# ---------------------------------------------------------------- how calls are used

def test_partial_gradients(gpu):
    """Each gradient alone equals its part of all of them."""
    g = _gen(8)
    dt = torch.bfloat16
    t = {"x": _rand(g, 90, 72, dtype=dt), "w": _rand(g, 136, 72, dtype=dt, std=0.1), "b": _rand(g, 136, dtype=dt),
         "r": _rand(g, 90, 136, dtype=dt)}
    n = {"x": _rand(g, 90, 72, dtype=dt), "w": _rand(g, 72, dtype=dt), "b": _rand(g, 72, dtype=dt)}
    s = {"x": t["x"], "w": t["w"], "b": t["b"], "wg": t["w"] * 0.5, "bg": t["b"] * 0.5}
    calls = [(t, lambda x, w, b, r: D.linear_act(x, w, b, act="silu", residual=r)),
             (t, lambda x, w, b, r: D.linear_act(x, w, b, residual=r)),
             ({k: t[k] for k in "xwb"}, lambda x, w, b: D.gated_linear(x, w, b)),
             (s, lambda x, w, b, wg, bg: D.gated_linear(x, w, b, gate_weight=wg, gate_bias=bg)),
             (n, lambda x, w, b: D.layer_norm(x, w, b))]
    for tensors, call in calls:
        leaves = {k: v.detach().requires_grad_(True) for k, v in tensors.items()}
        y = call(**leaves)
        dy = torch.randn_like(y)
        full = torch.autograd.grad(y, list(leaves.values()), dy, retain_graph=True)
        again = torch.autograd.grad(y, list(leaves.values()), dy)
        for a, c in zip(full, again):
            assert torch.equal(a, c)
        for (k, v), want in zip(tensors.items(), full):
            one = {q: u.detach().requires_grad_(q == k) for q, u in tensors.items()}
            got, = torch.autograd.grad(call(**one), [one[k]], dy)
            assert torch.equal(got, want), k


def test_weight_used_twice_accumulates(gpu):
    g = _gen(9)
    x = _rand(g, 33, 64, dtype=torch.bfloat16)
    w = _rand(g, 64, 64, dtype=torch.bfloat16, std=0.1).requires_grad_(True)
    h = D.linear_act(x, w, act="silu")
    y = D.linear_act(h, w, residual=h)
    y.float().sum().backward()
    xd, wd = x.double(), w.detach().double().requires_grad_(True)
    hd = torch.nn.functional.silu(xd @ wd.T)
    (hd @ wd.T + hd).sum().backward()
    rel = float((w.grad.double() - wd.grad).norm() / wd.grad.norm())
    assert rel < 3 * 2.0 ** -8   # three roundings of half a step each on the way (h, dz, dw)


def test_saved_tensors_are_version_checked(gpu):
    w = torch.randn(64, 64, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
    x = torch.randn(8, 64, device="cuda", dtype=torch.bfloat16)
    y = D.linear_act(x, w, act="gelu")
    x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_non_default_stream(gpu):
    g = _gen(10)
    x, w = _rand(g, 700, 640, dtype=torch.float16), _rand(g, 1280, 640, dtype=torch.float16, std=0.04)
    refs = D.linear_act(x, w, act="gelu"), D.gated_linear(x, w), D.layer_norm(x)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            outs.append((D.linear_act(x, w, act="gelu"), D.gated_linear(x, w), D.layer_norm(x)))
    torch.cuda.synchronize()
    for out in outs:
        for a, b in zip(out, refs):
            assert torch.equal(a, b)


@pytest.mark.parametrize("M, K, N", [(1, 512, 264), (24, 4096, 264), (300, 320, 640)])
def test_graph_replays(gpu, M, K, N):
    """Forward and backward of a sublayer captured once, replayed on new
    inputs with eager work between: every replay equals the eager result."""
    g = _gen(11)
    dt = torch.bfloat16
    x, dy = _rand(g, M, K, dtype=dt), _rand(g, M, K, dtype=dt)
    p = {"nw": _rand(g, K, dtype=dt), "nb": _rand(g, K, dtype=dt), "w1": _rand(g, 2 * N, K, dtype=dt, std=K ** -0.5),
         "b1": _rand(g, 2 * N, dtype=dt), "w2": _rand(g, K, N, dtype=dt, std=N ** -0.5), "b2": _rand(g, K, dtype=dt)}

    def step(x, dy):
        leaves = [t.detach().requires_grad_(True) for t in (x, *p.values())]
        lx, nw, nb, w1, b1, w2, b2 = leaves
        y = D.linear_act(D.gated_linear(D.layer_norm(lx, nw, nb), w1, b1), w2, b2, residual=lx)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    sx, sdy = x.clone(), dy.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(sx, sdy)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(sx, sdy)
    for i in range(4):
        nx, ndy = _rand(g, M, K, dtype=dt), _rand(g, M, K, dtype=dt)
        want = step(nx, ndy)
        sx.copy_(nx)
        sdy.copy_(ndy)
        graph.replay()
        torch.cuda.synchronize()
        for j, (a, b) in enumerate(zip(captured, want)):
            assert torch.equal(a, b), f"replay {i}, tensor {j}"


@pytest.mark.parametrize("M", [1, 2, 154, 1024])
def test_sublayer(gpu, M):
    """``x + out(GEGLU(proj)(LN(x)))`` as it is used, with every gradient,
    against float64. Each of the three operators rounds its outputs (and its
    gated middle's gradient) to 16 bits: relative L2 below 6 half steps."""
    torch.manual_seed(M)
    dt = torch.bfloat16
    norm, proj, out = nn.LayerNorm(320), nn.Linear(320, 2 * 1280), nn.Linear(1280, 320)
    mods = [m.to("cuda", dt) for m in (norm, proj, out)]
    x = torch.randn(2, M, 320, device="cuda", dtype=dt).requires_grad_(True)
    params = [p for m in mods for p in m.parameters()]
    y = D.geglu_ff(D.layer_norm(x, norm.weight, norm.bias, norm.eps), proj, out, residual=x)
    dy = torch.randn_like(y)
    got = torch.autograd.grad(y, [x, *params], dy)
    xd = x.detach().double().requires_grad_(True)
    pd = [p.detach().double().requires_grad_(True) for p in params]
    v, g = torch.nn.functional.linear(torch.nn.functional.layer_norm(xd, (320,), pd[0], pd[1], norm.eps), pd[2],
                                      pd[3]).chunk(2, -1)
    yd = torch.nn.functional.linear(v * torch.nn.functional.gelu(g), pd[4], pd[5]) + xd
    want = torch.autograd.grad(yd, [xd, *pd], dy.double())
    for i, (a, b) in enumerate([(y, yd), *zip(got, want)]):
        rel = float((a.detach().double() - b.detach()).norm() / b.detach().norm())
        assert rel < 6 * 2.0 ** -8, (i, rel)


@pytest.mark.parametrize("level", [0, 2])
def test_unet_block_trains_as_eager(gpu, level):
    """The UNet block on these operators (``unet_block.to_fused16``) against the
    eager fp16 block: output and every gradient. Both round at every op, the
    eager one at more of them (norm, projection, gelu, product, sum: 5 to our
    3), so the two differ by at most the sum of both, taken as 16 half steps in
    relative L2 (a chain of three sublayers)."""
    import copy

    import unet_block as UB
    lv = UB.LEVELS[level]
    blk = UB.build(lv, gpu)
    fused = UB.to_fused16(copy.deepcopy(blk))
    x, ctx = UB.inputs(lv, gpu)
    dy = torch.randn_like(x)
    got = []
    for b in (blk, fused):
        t = x.detach().requires_grad_(True)
        y = b(t, ctx)
        got.append((y.detach(), *torch.autograd.grad(y, [t, *b.parameters()], dy)))
    names = ["y", "dx"] + [n for n, _ in blk.named_parameters()]
    for n, a, b in zip(names, *got):
        rel = float((a.double() - b.double()).norm() / a.double().norm())
        assert rel < 16 * 2.0 ** -11, (n, rel)
    with torch.no_grad():
        assert torch.equal(fused(x, ctx), got[1][0])
