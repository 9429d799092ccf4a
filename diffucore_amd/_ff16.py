"""The feed-forward sublayer in 16 bits, trainable: layer norm, a linear layer
with its bias, activation and residual in one kernel, and the gated (GEGLU /
SwiGLU) projection, each with its backward pass on this package's gfx950
kernels (``dc_layer_norm``, ``dc_linear16``, ``dc_gated16`` and their
gradients in the C ABI).

They are the 16-bit companions of ``ln_mod_quantize``, ``Int8Linear`` and
``int8_geglu_ff``: for the layers a W8A8 model keeps in fp16 / bf16, and for
training (LoRAs, fine-tuning), which the int8 path does not do. The reference
runs torch's own ops there (``unet.py:148-183``).

All of them take tensors of any leading shape and any strides, enqueue on
torch's current stream of the tensors' device, and are differentiable once.
Sums, statistics and gradients are accumulated in float32 and rounded once; for
the backward pass of an activation its input is kept in float32, and the
gradient at it is rounded to 16 bits as the operand of the products that follow.
CPU tensors run the same formulas in torch ops; GPU tensors always run the
HIP kernels, and raise where the library is missing.
"""

from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from . import _lib

ACTIVATIONS = {"none": 0, "gelu": 1, "gelu_tanh": 2, "silu": 4, "quick_gelu": 5}
_HALF = (torch.float16, torch.bfloat16)
_FLOAT = (torch.float16, torch.bfloat16, torch.float32)
_FWD, _GATED, _DX, _DX2, _DW, _DW2 = range(6)


def _act(z: torch.Tensor, act: str) -> torch.Tensor:
    if act == "none":
        return z
    if act == "silu":
        return F.silu(z)
    if act == "quick_gelu":
        return z * torch.sigmoid(1.702 * z)
    return F.gelu(z, approximate="tanh" if act == "gelu_tanh" else "none")


# ─── argument checks ─────────────────────────────────────────────────────────

def _check_act(what: str, act: str, gated: bool = False) -> int:
    if act not in ACTIVATIONS or (gated and act == "none"):
        allowed = sorted(a for a in ACTIVATIONS if not (gated and a == "none"))
        raise ValueError(f"{what}: act must be one of {allowed}, got {act!r}")
    return ACTIVATIONS[act]


def _check_input(what: str, x: torch.Tensor) -> None:
    if x.dim() < 1:
        raise ValueError(f"{what}: x needs at least one dim")
    if x.shape[-1] == 0:
        raise ValueError(f"{what}: the last dim of x is empty")


def _check_like(what: str, name: str, t: torch.Tensor, x: torch.Tensor, shape: tuple, dtypes: tuple) -> None:
    if t.device != x.device:
        raise ValueError(f"{what}: {name} is on {t.device}, x on {x.device}")
    if tuple(t.shape) != shape:
        raise ValueError(f"{what}: {name} is {tuple(t.shape)}, expected {shape}")
    if t.dtype not in dtypes:
        raise TypeError(f"{what}: {name} is {t.dtype}, expected {' or '.join(str(d) for d in dtypes)}")


def _check_product(what: str, x: torch.Tensor, weight: torch.Tensor) -> None:
    _check_input(what, x)
    if weight.dim() != 2:
        raise ValueError(f"{what}: weight is {weight.dim()}-dimensional, expected [out, in]")
    _check_like(what, "weight", weight, x, (weight.shape[0], x.shape[-1]), (x.dtype,))
    if x.is_cuda and x.dtype not in _HALF:
        raise TypeError(f"{what}: the kernels take fp16 or bf16 tensors, got {x.dtype}")
    if not (x.is_cuda or _host(x)):
        raise RuntimeError(f"{what}: diffucore_amd runs on GPU and CPU tensors (got a {x.device} tensor)")


def _host(t: torch.Tensor) -> bool:
    return t.device.type == "cpu"


def _needs_grad(*ts) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


# ─── operands ────────────────────────────────────────────────────────────────

def _flat(t: torch.Tensor) -> torch.Tensor:
    """``t`` as rows over its last dim, unit stride along it, rows that do not
    overlap (any row stride and alignment). A single row's stride is its
    length, whatever the tensor calls it."""
    t = t.reshape(-1, t.shape[-1]) if t.dim() != 2 else t
    if (t.stride(1) != 1 and t.shape[1] != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        t = t.contiguous()
    if t.shape[0] == 1 or t.shape[1] == 1:
        t = t.contiguous().view(t.shape)
        if t.stride(0) != t.shape[1] or t.stride(1) != 1:
            t = t.as_strided(t.shape, (t.shape[1], 1))
    return t


def _operand(t: torch.Tensor) -> torch.Tensor:
    """``t [R, W]`` as an operand of the products: 16-byte aligned rows, zeros
    up to a width that is a multiple of 8 (a copy where ``t`` has none)."""
    t = _flat(t)
    w = t.shape[1]
    if w % 8:
        return F.pad(t, (0, -w % 8))
    if t.data_ptr() % 16 or (t.stride(0) % 8 and t.shape[0] > 1):
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _ptr(t):
    return None if t is None else t.data_ptr()


def _code(t) -> int:
    return _lib.NONE if t is None else _lib.dtype_code(t.dtype)


def _contig(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _scratch(nbytes: int, device):
    return torch.empty(nbytes, device=device, dtype=torch.uint8) if nbytes else None


def _workspace(so, op: int, M: int, N: int, K: int, device):
    n = so.dc_linear16_workspace_bytes(op, M, N, K)
    return _scratch(n, device), n


# ─── layer norm ──────────────────────────────────────────────────────────────

def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dim, in
    ``x``'s dtype (fp16, bf16 or float32; ``weight`` and ``bias`` of one dtype,
    ``x``'s or another of the three, such as float32 master weights). The
    statistics are float32, from deviations to the mean. One pass over the
    rows; the backward pass is one more and the sum of its partial weight
    gradients."""
    what = "layer_norm"
    _check_input(what, x)
    if x.dtype not in _FLOAT:
        raise TypeError(f"{what}: x is {x.dtype}, expected fp16, bf16 or float32")
    D = x.shape[-1]
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            _check_like(what, name, t, x, (D,), _FLOAT)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"{what}: weight is {weight.dtype}, bias {bias.dtype}")
    if _host(x):
        y = F.layer_norm(x.float(), (D,), None if weight is None else weight.float(), None, eps)
        return (y if bias is None else y + bias.float()).to(x.dtype)
    if not x.is_cuda:
        raise RuntimeError(f"{what}: diffucore_amd runs on GPU and CPU tensors (got a {x.device} tensor)")
    if _needs_grad(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, eps)
    return _norm_forward(x, weight, bias, eps, False)[0]


def _norm_forward(x, weight, bias, eps, keep: bool):
    so = _lib.require()
    x2 = _flat(x)
    M, D = x2.shape
    weight, bias = _contig(weight), _contig(bias)
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    stats = torch.empty((2, M), device=x.device, dtype=torch.float32) if keep else None
    with _lib.device_ctx(x.device):
        rc = so.dc_layer_norm(x2.data_ptr(), x2.stride(0), _code(x2), _ptr(weight), _ptr(bias),
                              _code(weight if weight is not None else bias), eps, y.data_ptr(), D, _ptr(stats), M, D,
                              _lib.stream_ptr(x.device))
    _lib.check(rc, "dc_layer_norm")
    return y, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = _norm_forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.param_dtype = weight.dtype if weight is not None else bias.dtype if bias is not None else None
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        want_x, want_w, want_b, _ = ctx.needs_input_grad
        so = _lib.require()
        x2, dy2, dev = _flat(x), _flat(dy), x.device
        M, D = x2.shape
        weight = _contig(weight)
        dx = torch.empty(x.shape, device=dev, dtype=x.dtype) if want_x else None
        dw = torch.empty(D, device=dev, dtype=ctx.param_dtype) if want_w else None
        db = torch.empty(D, device=dev, dtype=ctx.param_dtype) if want_b else None
        with _lib.device_ctx(dev):
            need = so.dc_layer_norm_bwd_workspace_bytes(M, D, _code(x)) if want_w or want_b else 0
            ws = _scratch(need, dev)
            code = _lib.NONE if ctx.param_dtype is None else _lib.dtype_code(ctx.param_dtype)
            rc = so.dc_layer_norm_bwd(dy2.data_ptr(), dy2.stride(0), x2.data_ptr(), x2.stride(0), _code(x),
                                      _ptr(weight), code, stats.data_ptr(), _ptr(dx), D, _ptr(dw), _ptr(db), M, D,
                                      _ptr(ws), need, _lib.stream_ptr(dev))
        _lib.check(rc, "dc_layer_norm_bwd")
        return dx, dw, db, None


# ─── linear with bias, activation and residual ───────────────────────────────

def linear_act(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, act: str = "none",
               residual: torch.Tensor | None = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual``, rounded once, in one kernel:
    ``x [..., K]``, ``weight [N, K]`` of one dtype (fp16 or bf16), ``bias [N]``
    of that dtype or float32, ``residual [..., N]`` of ``x``'s dtype. ``act`` is
    one of :data:`ACTIVATIONS` (``"gelu"`` the erf form, ``"quick_gelu"``
    ``z * sigmoid(1.702 z)``). Any sizes; widths that are not multiples of 8
    or rows that are not 16-byte aligned cost a padded copy of the operand."""
    what = "linear_act"
    code = _check_act(what, act)
    _check_product(what, x, weight)
    N = weight.shape[0]
    if bias is not None:
        _check_like(what, "bias", bias, x, (N,), (x.dtype, torch.float32))
    if residual is not None:
        _check_like(what, "residual", residual, x, (*x.shape[:-1], N), (x.dtype,))
    if _host(x):
        y = _act(F.linear(x.float(), weight.float(), None if bias is None else bias.float()), act)
        return (y if residual is None else y + residual.float()).to(x.dtype)
    if _needs_grad(x, weight, bias, residual):
        return _LinearAct.apply(x, weight, bias, residual, code)
    return _linear_forward(x, weight, bias, residual, code, False)[0]


def _linear_forward(x, weight, bias, residual, act: int, keep: bool):
    so = _lib.require()
    dev, dt = x.device, _lib.dtype_code(x.dtype)
    x2, w2 = _operand(x), _operand(weight)
    (M, K), N = x2.shape, w2.shape[0]
    out = torch.empty((*x.shape[:-1], N), device=dev, dtype=x.dtype)
    if M == 0 or N == 0:
        return out, None
    bias = _contig(bias)
    r2 = None if residual is None else _flat(residual)
    z = torch.empty((M, N), device=dev, dtype=torch.float32) if keep else None
    with _lib.device_ctx(dev):
        ws, need = _workspace(so, _FWD, M, N, K, dev)
        rc = so.dc_linear16(x2.data_ptr(), x2.stride(0), w2.data_ptr(), w2.stride(0), _ptr(bias), _code(bias),
                            _ptr(r2), 0 if r2 is None else r2.stride(0), act, out.data_ptr(), N, _ptr(z), N, dt, M, N,
                            K, _ptr(ws), need, _lib.stream_ptr(dev))
    _lib.check(rc, "dc_linear16")
    return out, z


def _dx(so, dz, w, dz2, w2, M: int, N: int, x: torch.Tensor) -> torch.Tensor:
    """``dz @ w (+ dz2 @ w2)`` in ``x``'s shape; ``dz`` and ``w`` are operands."""
    dev, K = x.device, x.shape[-1]
    dx = torch.empty(x.shape, device=dev, dtype=x.dtype)
    ws, need = _workspace(so, _DX if dz2 is None else _DX2, M, N, K, dev)
    rc = so.dc_linear16_dx(dz.data_ptr(), dz.stride(0), w.data_ptr(), w.stride(0), _ptr(dz2), _ptr(w2),
                           0 if w2 is None else w2.stride(0), dx.data_ptr(), K, _lib.dtype_code(x.dtype), M, N, K,
                           _ptr(ws), need, _lib.stream_ptr(dev))
    _lib.check(rc, "dc_linear16_dx")
    return dx


def _dw(so, dz, x2, dz2, dw, dw2, M: int, N: int, K: int) -> None:
    """``dw = dz.T @ x2`` (and ``dw2`` of ``dz2``); ``dz`` and ``x2`` are operands."""
    dev = dz.device
    ws, need = _workspace(so, _DW if dz2 is None else _DW2, M, N, K, dev)
    rc = so.dc_linear16_dw(dz.data_ptr(), dz.stride(0), x2.data_ptr(), x2.stride(0), _ptr(dz2), dw.data_ptr(), K,
                           _ptr(dw2), _lib.dtype_code(dz.dtype), M, N, K, _ptr(ws), need, _lib.stream_ptr(dev))
    _lib.check(rc, "dc_linear16_dw")


class _LinearAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        keep = act != 0 and any(ctx.needs_input_grad[:3])
        y, z = _linear_forward(x, weight, bias, residual, act, keep)
        ctx.save_for_backward(x, weight, z)
        ctx.act, ctx.bias_dtype = act, None if bias is None else bias.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        want_x, want_w, want_b, want_r, _ = ctx.needs_input_grad
        dx = dw = db = None
        if want_x or want_w or want_b:
            so, dev, dt = _lib.require(), x.device, _lib.dtype_code(x.dtype)
            N, K = weight.shape
            M = x.numel() // K
            if M == 0 or N == 0:
                return (torch.zeros_like(x) if want_x else None, torch.zeros_like(weight) if want_w else None,
                        torch.zeros(N, device=dev, dtype=ctx.bias_dtype) if want_b else None,
                        dy if want_r else None, None)
            dy2 = _flat(dy)
            with _lib.device_ctx(dev):
                db = torch.empty(N, device=dev, dtype=ctx.bias_dtype) if want_b else None
                pad = -(-N // 64) * 64
                dz = torch.empty((M, pad), device=dev, dtype=x.dtype) if ctx.act else None
                if dz is not None or want_b:
                    need = so.dc_act16_bwd_workspace_bytes(M, N, 0) if want_b else 0
                    ws = _scratch(need, dev)
                    rc = so.dc_act16_bwd(dy2.data_ptr(), dy2.stride(0), _ptr(z), N, ctx.act, _ptr(dz), pad, _ptr(db),
                                         _code(db), dt, M, N, _ptr(ws), need, _lib.stream_ptr(dev))
                    _lib.check(rc, "dc_act16_bwd")
                if dz is None and (want_x or want_w):
                    dz = _operand(dy2)
                if want_x:
                    dx = _dx(so, dz, _operand(weight), None, None, M, N, x)
                if want_w:
                    dw = torch.empty((N, K), device=dev, dtype=x.dtype)
                    _dw(so, dz, _operand(x), None, dw, None, M, N, K)
        return dx, dw, db, dy if want_r else None, None


# ─── gated projection ────────────────────────────────────────────────────────

def gated_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
                 gate_weight: torch.Tensor | None = None, gate_bias: torch.Tensor | None = None,
                 act: str = "gelu") -> torch.Tensor:
    """``(x @ Wv.T + bv) * act(x @ Wg.T + bg)``, both projections, the
    activation and the product in one kernel, rounded once. ``weight [2F, K]``
    holds the value rows and then the gate rows (the GEGLU projection's layout,
    as :func:`geglu_quantize` takes it), or, with ``gate_weight [F, K]``, the
    value rows alone (``weight [F, K]``); the biases likewise. ``act`` is one of
    :data:`ACTIVATIONS` except ``"none"``. Types as in :func:`linear_act`."""
    what = "gated_linear"
    code = _check_act(what, act, gated=True)
    _check_product(what, x, weight)
    N = weight.shape[0]
    if gate_weight is not None:
        _check_like(what, "gate_weight", gate_weight, x, tuple(weight.shape), (x.dtype,))
    elif gate_bias is not None:
        raise ValueError(f"{what}: gate_bias goes with gate_weight (bias holds both halves)")
    elif N % 2:
        raise ValueError(f"{what}: weight has {N} rows, expected value and gate halves")
    bias_types = (x.dtype, torch.float32)
    for name, t in (("bias", bias), ("gate_bias", gate_bias)):
        if t is not None:
            _check_like(what, name, t, x, (N,), bias_types)
    if bias is not None and gate_bias is not None and bias.dtype != gate_bias.dtype:
        raise TypeError(f"{what}: bias is {bias.dtype}, gate_bias {gate_bias.dtype}")
    if _host(x):
        xf = x.float()
        if gate_weight is None:
            v, g = F.linear(xf, weight.float(), None if bias is None else bias.float()).chunk(2, dim=-1)
        else:
            v = F.linear(xf, weight.float(), None if bias is None else bias.float())
            g = F.linear(xf, gate_weight.float(), None if gate_bias is None else gate_bias.float())
        return (v * _act(g, act)).to(x.dtype)
    if _needs_grad(x, weight, bias, gate_weight, gate_bias):
        return _GatedLinear.apply(x, weight, bias, gate_weight, gate_bias, code)
    return _gated_forward(x, weight, bias, gate_weight, gate_bias, code, False)[0]


def _halves(weight, gate_weight):
    """Value and gate weights ``[F, K]`` as operands, of one stacked weight or two."""
    w = _operand(weight)
    if gate_weight is not None:
        return w, _operand(gate_weight)
    f = w.shape[0] // 2
    return w[:f], w[f:]


def _gated_forward(x, weight, bias, gate_weight, gate_bias, act: int, keep: bool):
    so = _lib.require()
    dev = x.device
    x2 = _operand(x)
    wv, wg = _halves(weight, gate_weight)
    (M, K), N = x2.shape, wv.shape[0]
    out = torch.empty((*x.shape[:-1], N), device=dev, dtype=x.dtype)
    if M == 0 or N == 0:
        return out, None
    bias, gate_bias = _contig(bias), _contig(gate_bias)
    bv, bg = _ptr(bias), _ptr(gate_bias)
    if gate_weight is None and bias is not None:
        bg = bv + N * bias.element_size()
    z = torch.empty((2, M, N), device=dev, dtype=torch.float32) if keep else None
    zv = _ptr(z)
    with _lib.device_ctx(dev):
        ws, need = _workspace(so, _GATED, M, N, K, dev)
        rc = so.dc_gated16(x2.data_ptr(), x2.stride(0), wv.data_ptr(), wv.stride(0), wg.data_ptr(), wg.stride(0), bv,
                           bg, _code(bias if bias is not None else gate_bias), act, out.data_ptr(), N, zv,
                           None if z is None else zv + M * N * 4, N, _lib.dtype_code(x.dtype), M, N, K, _ptr(ws), need,
                           _lib.stream_ptr(dev))
    _lib.check(rc, "dc_gated16")
    return out, z


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, gate_weight, gate_bias, act):
        y, z = _gated_forward(x, weight, bias, gate_weight, gate_bias, act, True)
        ctx.save_for_backward(x, weight, gate_weight, z)
        ctx.act, ctx.bias_dtype = act, bias.dtype if bias is not None else None if gate_bias is None else gate_bias.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, gate_weight, z = ctx.saved_tensors
        want_x, want_w, want_b, want_wg, want_bg, _ = ctx.needs_input_grad
        so, dev, K = _lib.require(), x.device, x.shape[-1]
        fused = gate_weight is None
        N = weight.shape[0] // 2 if fused else weight.shape[0]
        M = x.numel() // K

        def empty(want, *shape, dtype=x.dtype):
            return torch.empty(shape, device=dev, dtype=dtype) if want else None

        rows = 2 * N if fused else N
        dw, dwg = empty(want_w, rows, K), empty(want_wg, N, K)
        db, dbg = empty(want_b, rows, dtype=ctx.bias_dtype), empty(want_bg, N, dtype=ctx.bias_dtype)
        if M == 0 or N == 0:
            for t in (dw, dwg, db, dbg):
                if t is not None:
                    t.zero_()
            return torch.zeros_like(x) if want_x else None, dw, db, dwg, dbg, None
        dy2, pad = _flat(dy), -(-N // 64) * 64
        dz = torch.empty((2, M, pad), device=dev, dtype=x.dtype)
        with _lib.device_ctx(dev):
            sums = want_b or want_bg
            need = so.dc_act16_bwd_workspace_bytes(M, N, 1) if sums else 0
            ws = _scratch(need, dev)
            dbv, dbg_p = _ptr(db), _ptr(dbg)
            if fused and want_b:
                dbg_p = dbv + N * db.element_size()
            zv, dzv = z.data_ptr(), dz.data_ptr()
            rc = so.dc_gated16_bwd(dy2.data_ptr(), dy2.stride(0), zv, zv + M * N * 4, N, ctx.act, dzv,
                                   dzv + M * pad * 2, pad, dbv, dbg_p,
                                   _lib.dtype_code(ctx.bias_dtype) if sums else _lib.NONE, _lib.dtype_code(x.dtype),
                                   M, N, _ptr(ws), need, _lib.stream_ptr(dev))
            _lib.check(rc, "dc_gated16_bwd")
            dx = None
            if want_x:
                wv, wg = _halves(weight, gate_weight)
                dx = _dx(so, dz[0], wv, dz[1], wg, M, N, x)
            if want_w or want_wg:
                x2 = _operand(x)
                if fused:
                    _dw(so, dz[0], x2, dz[1], dw[:N], dw[N:], M, N, K)
                elif want_w and want_wg:
                    _dw(so, dz[0], x2, dz[1], dw, dwg, M, N, K)
                else:
                    _dw(so, dz[0] if want_w else dz[1], x2, None, dw if want_w else dwg, None, M, N, K)
        return dx, dw, db, dwg, dbg, None


def geglu_ff(x: torch.Tensor, proj: nn.Linear, out: nn.Linear, residual: torch.Tensor | None = None,
             act: str = "gelu") -> torch.Tensor:
    """The UNet feed-forward ``out(GEGLU(proj)(x)) + residual``
    (``unet.py:148-165``) on 16-bit ``nn.Linear`` layers, as
    :func:`int8_geglu_ff` runs it on W8A8 ones: :func:`gated_linear` on
    ``proj``'s stacked value and gate rows, then :func:`linear_act`."""
    h = gated_linear(x, proj.weight, proj.bias, act=act)
    return linear_act(h, out.weight, out.bias, residual=residual)
