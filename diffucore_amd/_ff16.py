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
They can be captured into a HIP graph after one call of the same shapes; a
backward pass is captured as torch's own are: no eager autograd graph of the
same leaves may be alive then (detach the leaves, or drop its outputs first).
Sums, statistics and gradients are accumulated in float32 and rounded once; for
the backward pass of an activation its input is kept in 24 bits, and the
gradient at it is rounded to 16 bits as the operand of the products that follow.
CPU tensors run the same formulas in torch ops; GPU tensors always run the
HIP kernels, and raise where the library is missing.
"""

from __future__ import annotations

import functools

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from . import _lib

ACTIVATIONS = {"none": 0, "gelu": 1, "gelu_tanh": 2, "silu": 4, "quick_gelu": 5}
_HALF = (torch.float16, torch.bfloat16)
_FLOAT = (torch.float16, torch.bfloat16, torch.float32)
_WANT_DX, _WANT_DW, _WANT_DW2, _WANT_DB = 1, 2, 4, 8   # DC_WANT_*


def _act(z: torch.Tensor, act: str) -> torch.Tensor:
    if act == "none":
        return z
    if act == "silu":
        return F.silu(z)
    if act == "quick_gelu":
        return z * torch.sigmoid(1.702 * z)
    return F.gelu(z, approximate="tanh" if act == "gelu_tanh" else "none")


# ─── argument checks ─────────────────────────────────────────────────────────

def _check_act(what: str, act: str) -> int:
    if act not in ACTIVATIONS:
        raise ValueError(f"{what}: act must be one of {sorted(ACTIVATIONS)}, got {act!r}")
    return ACTIVATIONS[act]


def _check_input(what: str, x: torch.Tensor) -> None:
    if x.dim() < 1:
        raise ValueError(f"{what}: x needs at least one dim")
    if x.shape[-1] == 0:
        raise ValueError(f"{what}: the last dim of x is empty")


def _check_like(what: str, name: str, t: torch.Tensor, x: torch.Tensor, shape: tuple, dtypes: tuple) -> None:
    if t.shape == shape and t.dtype in dtypes and t.device == x.device:
        return
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
    if x.is_cuda:
        if x.dtype not in _HALF:
            raise TypeError(f"{what}: the kernels take fp16 or bf16 tensors, got {x.dtype}")
    elif x.dtype not in _FLOAT:
        raise TypeError(f"{what}: x is {x.dtype}, expected fp16, bf16 or float32")
    elif not _host(x):
        raise RuntimeError(f"{what}: diffucore_amd runs on GPU and CPU tensors (got a {x.device} tensor)")


def _host(t: torch.Tensor) -> bool:
    return t.device.type == "cpu"


def _needs_grad(*ts) -> bool:
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


# ─── operands ────────────────────────────────────────────────────────────────

def _flat(t: torch.Tensor) -> torch.Tensor:
    """``t`` as rows over its last dim, unit stride along it, rows that do not
    overlap (any row stride and alignment). A single row's stride is its
    length, whatever the tensor calls it."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    rows, width = t.shape
    step, unit = t.stride()
    if unit == 1 and (step == width or (step > width and rows != 1)):
        return t
    if (unit != 1 and width != 1) or (rows != 1 and step < width):
        t = t.contiguous()
    return t.as_strided((rows, width), (width if rows == 1 else t.stride(0), 1))


def _ptr(t):
    return None if t is None else t.data_ptr()


_CODES = {None: _lib.NONE, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}


def _code(t) -> int:
    return _CODES[None if t is None else t.dtype]


def _contig(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _scratch(nbytes: int, device):
    return torch.empty(nbytes, device=device, dtype=torch.uint8) if nbytes else None


@functools.lru_cache(maxsize=1024)
def _scratch_bytes(query: str, device_index: int, *args) -> int:
    """A workspace query on the current device (``device_index``), with each
    pointer given as its offset in 16 bytes: a plain number per shape, the most
    recent 1024 kept."""
    return int(getattr(_lib.require(), query)(*args))


def _at(t: torch.Tensor) -> int:
    """``t``'s address as the workspace queries see it: its alignment."""
    return 16 + t.data_ptr() % 16


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
    if not x.is_cuda and _host(x):
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
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    stats = torch.empty((2, M), device=x.device, dtype=torch.float32) if keep else None
    with _lib.device_ctx(x.device):
        rc = so.dc_layer_norm(x2.data_ptr(), x2.stride(0), _code(x2), _ptr(weight), _ptr(bias),
                              _code(weight if weight is not None else bias), eps, y.data_ptr(), D, _ptr(stats), M, D,
                              _lib.stream_ptr(x.device))
    if rc:
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
        dx = torch.empty_like(x, memory_format=torch.contiguous_format) if want_x else None
        dw = torch.empty(D, device=dev, dtype=ctx.param_dtype) if want_w else None
        db = torch.empty(D, device=dev, dtype=ctx.param_dtype) if want_b else None
        with _lib.device_ctx(dev):
            need = 0
            if want_w or want_b:
                need = _scratch_bytes("dc_layer_norm_bwd_workspace_bytes", dev.index, M, D, _code(x))
            ws = _scratch(need, dev)
            rc = so.dc_layer_norm_bwd(dy2.data_ptr(), dy2.stride(0), x2.data_ptr(), x2.stride(0), _code(x),
                                      _ptr(weight), _CODES[ctx.param_dtype], stats.data_ptr(), _ptr(dx), D, _ptr(dw),
                                      _ptr(db), M, D, _ptr(ws), need, _lib.stream_ptr(dev))
        if rc:
            _lib.check(rc, "dc_layer_norm_bwd")
        return dx, dw, db, None


# ─── linear with bias, activation and residual ───────────────────────────────

def linear_act(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, act: str = "none",
               residual: torch.Tensor | None = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual``, rounded once, in one kernel:
    ``x [..., K]``, ``weight [N, K]`` of one dtype (fp16 or bf16), ``bias [N]``
    of that dtype or float32, ``residual [..., N]`` of ``x``'s dtype. ``act`` is
    one of :data:`ACTIVATIONS` (``"gelu"`` the erf form, ``"quick_gelu"``
    ``z * sigmoid(1.702 z)``). Any sizes; an operand whose width or row stride
    is not a multiple of 8, or that is not 16-byte aligned, costs a padded copy."""
    what = "linear_act"
    code = _check_act(what, act)
    _check_product(what, x, weight)
    N = weight.shape[0]
    if bias is not None:
        _check_like(what, "bias", bias, x, (N,), (x.dtype, torch.float32))
    if residual is not None:
        _check_like(what, "residual", residual, x, (*x.shape[:-1], N), (x.dtype,))
    if not x.is_cuda:
        y = _act(F.linear(x.float(), weight.float(), None if bias is None else bias.float()), act)
        return (y if residual is None else y + residual.float()).to(x.dtype)
    if _needs_grad(x, weight, bias, residual):
        return _LinearAct.apply(x, weight, bias, residual, code)
    return _linear_forward(x, weight, bias, residual, code, False)[0]


def _linear_forward(x, weight, bias, residual, act: int, keep: bool):
    so = _lib.require()
    dev, dt = x.device, _CODES[x.dtype]
    x2, w2 = _flat(x), _flat(weight)
    (M, K), N = x2.shape, w2.shape[0]
    out = torch.empty((*x.shape[:-1], N), device=dev, dtype=x.dtype)
    if M == 0 or N == 0:
        return out, None
    bias = _contig(bias)
    r2 = None if residual is None else _flat(residual)
    z = torch.empty(3 * M * N, device=dev, dtype=torch.uint8) if keep else None   # dc_saved16_bytes
    ldx, ldw = x2.stride(0), w2.stride(0)
    with _lib.device_ctx(dev):
        need = _scratch_bytes("dc_linear16_workspace_bytes", dev.index, _at(x2), ldx, _at(w2), ldw, M, N, K)
        ws = _scratch(need, dev)
        rc = so.dc_linear16(x2.data_ptr(), ldx, w2.data_ptr(), ldw, _ptr(bias), _code(bias), _ptr(r2),
                            0 if r2 is None else r2.stride(0), act, out.data_ptr(), N, _ptr(z), dt, M, N, K,
                            _ptr(ws), need, _lib.stream_ptr(dev))
    if rc:
        _lib.check(rc, "dc_linear16")
    return out, z


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
        dres = dy if want_r else None
        if not (want_x or want_w or want_b):
            return None, None, None, dres, None
        so, dev, dt = _lib.require(), x.device, x.dtype
        N, K = weight.shape
        dx = torch.empty_like(x, memory_format=torch.contiguous_format) if want_x else None
        dw = torch.empty((N, K), device=dev, dtype=dt) if want_w else None
        db = torch.empty(N, device=dev, dtype=ctx.bias_dtype) if want_b else None
        M = x.numel() // K
        if M == 0 or N == 0:
            return (*(t if t is None else t.zero_() for t in (dx, dw, db)), dres, None)
        dy2, x2, w2 = _flat(dy), _flat(x), _flat(weight)
        ldy, ldx, ldw = dy2.stride(0), x2.stride(0), w2.stride(0)
        want = want_x * _WANT_DX + want_w * _WANT_DW + want_b * _WANT_DB
        with _lib.device_ctx(dev):
            need = _scratch_bytes("dc_linear16_bwd_workspace_bytes", dev.index, _at(dy2), ldy, _at(x2), ldx, _at(w2),
                                  ldw, ctx.act, want, M, N, K)
            ws = _scratch(need, dev)
            rc = so.dc_linear16_bwd(dy2.data_ptr(), ldy, x2.data_ptr(), ldx, w2.data_ptr(), ldw, _ptr(z), ctx.act,
                                    _ptr(dx), K, _ptr(dw), K, _ptr(db), _code(db), _CODES[dt], M, N, K,
                                    _ptr(ws), need, _lib.stream_ptr(dev))
        if rc:
            _lib.check(rc, "dc_linear16_bwd")
        return dx, dw, db, dres, None


# ─── gated projection ────────────────────────────────────────────────────────

def gated_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
                 gate_weight: torch.Tensor | None = None, gate_bias: torch.Tensor | None = None,
                 act: str = "gelu") -> torch.Tensor:
    """``(x @ Wv.T + bv) * act(x @ Wg.T + bg)``, both projections, the
    activation and the product in one kernel, rounded once. ``weight [2F, K]``
    holds the value rows and then the gate rows (the GEGLU projection's layout,
    as :func:`geglu_quantize` takes it), or, with ``gate_weight [F, K]``, the
    value rows alone (``weight [F, K]``); the biases likewise. ``act`` is one of
    :data:`ACTIVATIONS` (``"none"``: the plain product). Types as in :func:`linear_act`."""
    what = "gated_linear"
    code = _check_act(what, act)
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
    if not x.is_cuda:
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
    """Value and gate weights ``[F, K]``, of one stacked weight or two."""
    w = _flat(weight)
    if gate_weight is not None:
        return w, _flat(gate_weight)
    f = w.shape[0] // 2
    return w[:f], w[f:]


def _gated_forward(x, weight, bias, gate_weight, gate_bias, act: int, keep: bool):
    so = _lib.require()
    dev = x.device
    x2 = _flat(x)
    wv, wg = _halves(weight, gate_weight)
    (M, K), N = x2.shape, wv.shape[0]
    out = torch.empty((*x.shape[:-1], N), device=dev, dtype=x.dtype)
    if M == 0 or N == 0:
        return out, None
    bias, gate_bias = _contig(bias), _contig(gate_bias)
    bv, bg = _ptr(bias), _ptr(gate_bias)
    if gate_weight is None and bias is not None:
        bg = bv + N * bias.element_size()
    half = -(-3 * M * N // 16) * 16   # dc_saved16_bytes, the next one aligned
    z = torch.empty(2 * half, device=dev, dtype=torch.uint8) if keep else None
    zv = _ptr(z)
    ldx, ldv, ldg = x2.stride(0), wv.stride(0), wg.stride(0)
    with _lib.device_ctx(dev):
        need = _scratch_bytes("dc_gated16_workspace_bytes", dev.index, _at(x2), ldx, _at(wv), ldv, _at(wg), ldg, M, N,
                              K)
        ws = _scratch(need, dev)
        rc = so.dc_gated16(x2.data_ptr(), ldx, wv.data_ptr(), ldv, wg.data_ptr(), ldg, bv, bg,
                           _code(bias if bias is not None else gate_bias), act, out.data_ptr(), N, zv,
                           None if z is None else zv + half, _CODES[x.dtype], M, N, K, _ptr(ws), need,
                           _lib.stream_ptr(dev))
    if rc:
        _lib.check(rc, "dc_gated16")
    return out, z


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, gate_weight, gate_bias, act):
        y, z = _gated_forward(x, weight, bias, gate_weight, gate_bias, act, True)
        ctx.save_for_backward(x, weight, gate_weight, z)
        either = bias if bias is not None else gate_bias
        ctx.act, ctx.bias_dtype = act, None if either is None else either.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, gate_weight, z = ctx.saved_tensors
        want_x, want_w, want_b, want_wg, want_bg, _ = ctx.needs_input_grad
        so, dev, dt, K = _lib.require(), x.device, x.dtype, x.shape[-1]
        fused = gate_weight is None
        rows = weight.shape[0]
        N = rows // 2 if fused else rows
        dx = torch.empty_like(x, memory_format=torch.contiguous_format) if want_x else None
        dw = torch.empty((rows, K), device=dev, dtype=dt) if want_w else None
        dwg = torch.empty((N, K), device=dev, dtype=dt) if want_wg else None
        db = torch.empty(rows, device=dev, dtype=ctx.bias_dtype) if want_b else None
        dbg = torch.empty(N, device=dev, dtype=ctx.bias_dtype) if want_bg else None
        M = x.numel() // K
        if M == 0 or N == 0:
            return (*(t if t is None else t.zero_() for t in (dx, dw, db, dwg, dbg)), None)
        dy2, x2 = _flat(dy), _flat(x)
        wv, wg = _halves(weight, gate_weight)
        ldy, ldx, ldv, ldg = dy2.stride(0), x2.stride(0), wv.stride(0), wg.stride(0)
        dwv_p, dwg_p, dbv_p, dbg_p = _ptr(dw), _ptr(dwg), _ptr(db), _ptr(dbg)
        if fused and want_w:
            dwg_p = dwv_p + N * K * dw.element_size()
        if fused and want_b:
            dbg_p = dbv_p + N * db.element_size()
        want = (want_x * _WANT_DX + want_w * _WANT_DW + (want_w if fused else want_wg) * _WANT_DW2
                + (want_b or want_bg) * _WANT_DB)
        zv = z.data_ptr()
        with _lib.device_ctx(dev):
            need = _scratch_bytes("dc_gated16_bwd_workspace_bytes", dev.index, _at(dy2), ldy, _at(x2), ldx, _at(wv),
                                  ldv, _at(wg), ldg, want, M, N, K)
            ws = _scratch(need, dev)
            rc = so.dc_gated16_bwd(dy2.data_ptr(), ldy, x2.data_ptr(), ldx, wv.data_ptr(), ldv, wg.data_ptr(), ldg, zv,
                                   zv + z.numel() // 2, ctx.act, _ptr(dx), K, dwv_p, dwg_p, K, dbv_p, dbg_p,
                                   _CODES[ctx.bias_dtype],
                                   _CODES[dt], M, N, K, _ptr(ws), need, _lib.stream_ptr(dev))
        if rc:
            _lib.check(rc, "dc_gated16_bwd")
        return dx, dw, db, dwg, dbg, None


def geglu_ff(x: torch.Tensor, proj: nn.Linear, out: nn.Linear, residual: torch.Tensor | None = None,
             act: str = "gelu") -> torch.Tensor:
    """The UNet feed-forward ``out(GEGLU(proj)(x)) + residual``
    (``unet.py:148-165``) on 16-bit ``nn.Linear`` layers, as
    :func:`int8_geglu_ff` runs it on W8A8 ones: :func:`gated_linear` on
    ``proj``'s stacked value and gate rows, then :func:`linear_act`."""
    h = gated_linear(x, proj.weight, proj.bias, act=act)
    return linear_act(h, out.weight, out.bias, residual=residual)
