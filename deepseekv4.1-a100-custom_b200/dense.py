"""Dense feed-forward operators around the MoE path: the residual stream with its norm (`add_rms_norm`, `add_rms_norm_quant`), a projection with
bias, activation and residual in its epilogue (`linear_act`, `linear_act_q8`), the gated projection (`gated_linear`), and the block they form
(`DenseFFN`).  All are kernels of the library (include/b200_moe.h, "dense feed-forward operators") launched on the current stream of the
tensors' device; nothing synchronises.  Scratch and outputs come from torch's allocator per call, so calls on several streams, and captured
CUDA graphs, share no memory.

`add_rms_norm`, `linear_act` and `gated_linear` are differentiable in reverse mode, once: gradients of a create_graph backward raise when they are
differentiated again, and inputs with a forward-mode tangent are refused.  The FP8 forms are for serving and refuse inputs that require a gradient.
A captured backward pass needs what torch asks of any: capture it on the stream that ran the warm-up, and drop eager graphs of the same leaves first."""
from __future__ import annotations

import ctypes
import importlib.util
import os

import torch

from . import _lib as L

_PAIR = {torch.bfloat16: 0, torch.float16: 1}
_ACT = L.ACTIVATIONS

# ------------------------------------------------------------------ marshalling
# The small calls of a decode step are bound by the host, so nothing here builds objects that a call does not need: addresses go to ctypes as
# plain integers, the stream is read without a Stream object, contiguous tensors without a view, and the device is switched only when it is not
# the current one (a norm or a projection of few strided rows: 13 us, calls in a row; plain calls do not come here, they take csrc/fastcall.cpp's 4.4 to 6.4).
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice
_functions: dict = {}


_fast = None  # csrc/fastcall.cpp, bound on the first call


def _bind():
    """The extension with the short way for plain calls; it answers None to what is not plain."""
    global _fast
    path = os.path.join(L.HERE, "csrc", "_fastcall.so")
    if not os.path.exists(path):
        raise RuntimeError(f"{path} is missing: build it with `python -c 'import __graft_entry__ as g; g.build()'`")
    spec = importlib.util.spec_from_file_location("_fastcall", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    lib = L.lib()
    mod.bind({n: ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in (
        "b200_add_rms_norm", "b200_add_rms_norm_bwd_workspace_bytes", "b200_add_rms_norm_bwd", "b200_linear_act", "b200_linear_act_bwd_workspace_bytes", "b200_linear_act_bwd",
        "b200_gated_linear", "b200_gated_linear_bwd", "b200_dense_product", "b200_align_rows", "b200_linear_act_q8", "b200_linear_act_q8_workspace_bytes", "b200_error_string")})
    _fast = mod
    return mod


def _call(name: str, index: int, *args) -> None:
    fn = _functions.get(name)
    if fn is None:
        fn = _functions[name] = getattr(L.lib(), name)
    if index == _current_device():
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        L.check(rc, name)


def _size(name: str, index: int, *args) -> int:
    """A *_workspace_bytes function, which sizes for the current device."""
    fn = getattr(L.lib(), name)
    if index == _current_device():
        return fn(*args)
    with torch.cuda.device(index):
        return fn(*args)


def _device(a, b=None, c=None, d=None, e=None, f=None) -> int:
    """Index of the device that all tensors are on."""
    index = a.get_device()
    if (index < 0 or b is not None and b.get_device() != index or c is not None and c.get_device() != index or d is not None and d.get_device() != index
            or e is not None and e.get_device() != index or f is not None and f.get_device() != index):
        L.require_cuda(a, b, c, d, e, f)  # says what is wrong
    return index


def _ptr(t) -> int | None:
    return None if t is None else t.data_ptr()


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[..., D] as rows [R, D] with a unit inner stride and rows that do not overlap (a copy only where the strides do not allow a view)."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    if t.is_contiguous():
        return t
    if t.shape[1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        t = t.contiguous()
    return t


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _mat(t: torch.Tensor | None, cols: int):
    """(tensor to keep alive, address, row stride) of [..., cols] read as rows."""
    if t is None:
        return None, None, 0
    if not t.is_contiguous():
        t = _rows(t)
        return t, t.data_ptr(), _ld(t)
    return t, t.data_ptr(), cols


def _pitch(n: int) -> int:
    return (n + 7) // 8 * 8


def _fetchable(t: torch.Tensor, ld: int) -> bool:
    """Rows as the tensor-core kernels fetch them: 16-byte aligned base, a stride that is a multiple of 8 elements."""
    return not (t.data_ptr() & 15 or ld & 7)


def _aligned(x: torch.Tensor, w: torch.Tensor | None, K: int):
    """Copies of the rows x [R, K] and w [N, K] (w may be None) that the kernels can fetch, both in one launch: (scratch, rows of x, row stride)."""
    ld = _pitch(K)
    rx, rw = x.shape[0], 0 if w is None else w.shape[0]
    buf = torch.empty(rx + rw, ld, device=x.device, dtype=x.dtype)
    p = buf.data_ptr()
    _call("b200_align_rows", x.get_device(), x.data_ptr(), _ld(x), p, rx, _ptr(w), 0 if w is None else _ld(w), p + 2 * rx * ld, rw, K, ld)
    return buf, rx, ld


def _tma_rows(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """One matrix as fetchable rows: (rows, row stride)."""
    t = _rows(t)
    r, d = t.shape
    ld = t.stride(0) if r > 1 else _pitch(d)
    if _fetchable(t, ld):
        return t, ld
    buf, _, ld = _aligned(t, None, d)
    return buf[:, :d], ld


def _operands(x: torch.Tensor, w: torch.Tensor, K: int):
    """x [..., K] and w [N, K] as rows for the tensor-core kernels: (x, address, stride, w, address, stride); the tensors are kept for their memory."""
    if not K & 7 and x.is_contiguous() and w.is_contiguous():
        xp, wp = x.data_ptr(), w.data_ptr()
        if not (xp | wp) & 15:
            return x, xp, K, w, wp, K
    x, w = _rows(x), _rows(w)
    x_ld, w_ld = x.stride(0) if x.shape[0] > 1 else _pitch(K), w.stride(0) if w.shape[0] > 1 else _pitch(K)
    okx, okw = _fetchable(x, x_ld), _fetchable(w, w_ld)
    if okx and okw:
        return x, x.data_ptr(), x_ld, w, w.data_ptr(), w_ld
    if okx:
        w, _, w_ld = _aligned(w, None, K)
    elif okw:
        x, _, x_ld = _aligned(x, None, K)
    else:
        buf, rx, x_ld = _aligned(x, w, K)
        w_ld = x_ld
        x, w = buf[:rx], buf[rx:]
    return x, x.data_ptr(), x_ld, w, w.data_ptr(), w_ld


_grad_enabled = torch.is_grad_enabled


def _wants_grad(a, b=None, c=None, d=None) -> bool:
    return _grad_enabled() and (a.requires_grad or b is not None and b.requires_grad or c is not None and c.requires_grad or d is not None and d.requires_grad)


def _no_tangents(*ts) -> None:
    """Inputs that carry a forward-mode tangent are refused: the result would have none, which torch takes for a derivative of zero."""
    if (_fast or _bind()).tangents(ts):
        raise NotImplementedError("the dense operators have no forward-mode derivatives")


def _product(a, a_ld, a_mn, b, b_ld, b_mn, M, N, K, shape=None) -> torch.Tensor:
    out = torch.empty(shape or (M, N), device=a.device, dtype=a.dtype)
    _call("b200_dense_product", a.get_device(), a.data_ptr(), a_ld, a_mn, b.data_ptr(), b_ld, b_mn, _PAIR[a.dtype], M, N, K, out.data_ptr(), N)
    return out


def _once(out, inputs, incoming):
    """Gradients of a backward pass that records its graph (create_graph): csrc/fastcall.cpp's `once` stands guard over a second differentiation.  `inputs`: for
    each gradient the positions, among the function's tensor inputs, of those that it depends on."""
    return (_fast or _bind()).once(out, inputs, incoming)


def _scratch(nbytes: int, device) -> torch.Tensor | None:
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _restored(t: torch.Tensor, shape, dtype, device) -> torch.Tensor:
    """A tensor as `ctx.saved_tensors` returns it.  A saved-tensor hook (`torch.autograd.graph.save_on_cpu`) may hand back other strides and another address
    than were saved, so a backward pass takes both from here; other values' sizes, type or device it may not hand back."""
    if t.shape != shape or t.dtype is not dtype or t.device != device:
        raise RuntimeError(f"a saved-tensor hook returned {t.dtype} {tuple(t.shape)} on {t.device} for {dtype} {tuple(shape)} on {device}")
    return t


# ------------------------------------------------------------------ residual addition + rms norm
def _norm_args(x, residual, weight, eps):
    index, dt, D = _device(x, residual, weight), x.dtype, x.shape[-1]
    assert dt in L.DTYPES, f"x must be bfloat16, float16 or float32, got {dt}"
    assert 1 <= D <= 16384, f"width {D} is outside 1..16384"
    assert residual is None or (residual.dtype is dt and residual.shape == x.shape), "residual must have the type and shape of x"
    assert weight is None or (weight.shape == (D,) and (weight.dtype is dt or weight.dtype is torch.float32)), "weight must be [D], in x's type or float32"
    assert eps >= 0.0, "eps must not be negative"
    return index, D


def _norm_forward(index, D, x, residual, weight, eps, y, s, q8, sf):
    x, xp, x_ld = _mat(x, D)
    residual, rp, r_ld = _mat(residual, D)
    w_f32 = 0
    if weight is not None:
        w_f32 = weight.dtype is torch.float32
        weight = weight.contiguous()
    _call("b200_add_rms_norm", index, xp, x_ld, rp, r_ld, _ptr(weight), w_f32, L.DTYPES[x.dtype], x.numel() // D, D, eps, _ptr(y), _ptr(s), _ptr(q8), _ptr(sf))


class _AddRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        x2, r2 = _rows(x), _rows(residual) if residual is not None else None
        y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
        s = torch.empty_like(y) if residual is not None else None
        wc = weight.contiguous() if weight is not None else None
        _norm_forward(x.get_device(), x.shape[-1], x2, r2, wc, eps, y, s, None, None)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x2, r2, wc)
        ctx.eps, ctx.shape, ctx.rows, ctx.w_dtype, ctx.has_residual = eps, x.shape, x2.shape, wc.dtype if wc is not None else None, residual is not None
        return (y, s) if residual is not None else y

    @staticmethod
    def backward(ctx, gy, gs=None):
        if not _grad_enabled():
            return _AddRmsNorm.gradients(ctx, gy, gs)
        with torch.no_grad():
            dx, dr, dw, _ = _AddRmsNorm.gradients(ctx, gy, gs)
        if gy is not None:
            of_s = [0] + [1] * ctx.has_residual
            every = of_s + [len(of_s)] * (ctx.w_dtype is not None)
            dx, dr, dw = _once([dx, dr, dw], [every, every, of_s], [gy, gs])
        return dx, dr, dw, None

    @staticmethod
    def gradients(ctx, gy, gs=None):
        x, r, w = ctx.saved_tensors
        need_x, need_r, need_w, _ = ctx.needs_input_grad
        if gy is None:  # the normed output was not used
            return gs if need_x else None, gs if need_r else None, torch.zeros_like(w) if need_w else None, None
        dev = gy.device
        x = _rows(_restored(x, ctx.rows, gy.dtype, dev))
        r = _rows(_restored(r, ctx.rows, gy.dtype, dev)) if r is not None else None
        w = _restored(w, (ctx.rows[1],), ctx.w_dtype, dev).contiguous() if w is not None else None
        gy = gy.contiguous()
        gs = gs.contiguous() if gs is not None else None
        rows, D = x.shape
        ds = torch.empty(ctx.shape, device=dev, dtype=x.dtype)
        dw = torch.empty_like(w) if need_w else None
        nb = _size("b200_add_rms_norm_bwd_workspace_bytes", dev.index, rows, D) if need_w else 0
        ws = _scratch(nb, dev)
        _call("b200_add_rms_norm_bwd", dev.index, x.data_ptr(), _ld(x), _ptr(r), 0 if r is None else _ld(r), _ptr(w), w is not None and w.dtype is torch.float32, L.DTYPES[x.dtype],
              rows, D, ctx.eps, gy.data_ptr(), _ptr(gs), ds.data_ptr(), _ptr(dw), _ptr(ws), nb)
        return ds if need_x else None, ds if need_r else None, dw, None


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor | None = None, weight: torch.Tensor | None = None, eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """x, residual [..., D] bf16 | fp16 | fp32 -> (y, s): s = x + residual (x itself without a residual), y = s / sqrt(mean(s^2) + eps) * weight.
    The norm is taken of the unrounded fp32 sum.  weight [D] in x's type or fp32, or None for ones.  Differentiable."""
    plain = (_fast or _bind()).norm(x, residual, weight, eps, False, True)
    if plain is not None:
        return plain
    _no_tangents(x, residual, weight)
    index, D = _norm_args(x, residual, weight, eps)
    if _wants_grad(x, residual, weight):
        out = _AddRmsNorm.apply(x, residual, weight, float(eps))
        return out if residual is not None else (out, x)
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    s = torch.empty_like(y) if residual is not None else None
    _norm_forward(index, D, x, residual, weight, float(eps), y, s, None, None)
    return y, (x if s is None else s)


def add_rms_norm_quant(x: torch.Tensor, residual: torch.Tensor | None = None, weight: torch.Tensor | None = None, eps: float = 1e-6, want_y: bool = False):
    """The same norm with y in 8 bits -> (q8, sf, s[, y]): q8 uint8 e4m3 codes [rows, D], sf uint8 E8M0 [rows, D/32], rows = all leading
    dimensions together (what `cukern.mx_grouped` and `linear_act_q8` take); q8 * 2^(sf - 127) is y quantised per 32 from its fp32 value.  want_y:
    y in x's type too.  D % 32 == 0.  No gradient."""
    plain = (_fast or _bind()).norm(x, residual, weight, eps, True, want_y)
    if plain is not None:
        return plain
    _no_tangents(x, residual, weight)
    index, D = _norm_args(x, residual, weight, eps)
    assert D % 32 == 0, f"width {D} is not a multiple of 32"
    assert not _wants_grad(x, residual, weight), "add_rms_norm_quant has no gradient: use add_rms_norm, or detach its inputs"
    dev, rows = x.device, x.numel() // D
    q8 = torch.empty(rows, D, device=dev, dtype=torch.uint8)
    sf = torch.empty(rows, D // 32, device=dev, dtype=torch.uint8)
    s = torch.empty(x.shape, device=dev, dtype=x.dtype) if residual is not None else None
    y = torch.empty(x.shape, device=dev, dtype=x.dtype) if want_y else None
    _norm_forward(index, D, x, residual, weight, float(eps), y, s, q8, sf)
    if s is None:
        s = x
    return (q8, sf, s, y) if want_y else (q8, sf, s)


# ------------------------------------------------------------------ projection with bias, activation, residual
def _linear_forward(index, dt, ops, M, N, K, bias, act, residual, out, z, z_ld):
    _, xp, x_ld, _, wp, w_ld = ops
    bp, rp, r_ld = None, None, 0
    if bias is not None:
        bias = bias.contiguous()
        bp = bias.data_ptr()
    if residual is not None:
        residual, rp, r_ld = _mat(residual, N)
    _call("b200_linear_act", index, xp, x_ld, wp, w_ld, _PAIR[dt], M, N, K, bp, act, rp, r_ld, out.data_ptr(), N, _ptr(z), z_ld)


class _LinearAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, act, residual):
        N, K = w.shape
        ops = _operands(x, w, K)
        M = x.numel() // K
        out = torch.empty((*x.shape[:-1], N), device=x.device, dtype=x.dtype)
        z_ld = _pitch(N)
        z = torch.empty(M, z_ld, device=x.device, dtype=torch.float32) if act else None
        _linear_forward(x.get_device(), x.dtype, ops, M, N, K, bias, act, residual, out, z, z_ld)
        ctx.save_for_backward(ops[0], ops[3], z)
        ctx.dims, ctx.saved_shapes, ctx.act, ctx.x_shape = (M, N, K), (ops[0].shape, ops[3].shape), act, x.shape
        ctx.has_bias = bias is not None
        return out

    @staticmethod
    def backward(ctx, gy):
        if not _grad_enabled():
            return _LinearAct.gradients(ctx, gy)
        with torch.no_grad():
            dx, dw, db, _, dr = _LinearAct.gradients(ctx, gy)
        curved = ctx.act > 1  # without an activation, and with relu but for its corner, the slope does not depend on z
        of_z = [0, 1] + [2] * ctx.has_bias if curved else []
        return *_once([dx, dw, db], [of_z if curved else [1], of_z if curved else [0], of_z], [gy]), None, dr

    @staticmethod
    def gradients(ctx, gy):
        x, w, z = ctx.saved_tensors
        need_x, need_w, need_b, _, need_r = ctx.needs_input_grad
        (M, N, K), dev, dt = ctx.dims, gy.device, gy.dtype
        x, x_ld = _tma_rows(_restored(x, ctx.saved_shapes[0], dt, dev))
        w, w_ld = _tma_rows(_restored(w, ctx.saved_shapes[1], dt, dev))
        z = _restored(z, (M, _pitch(N)), torch.float32, dev).contiguous() if z is not None else None
        g2 = _rows(gy)
        dx = dw = db = None
        if need_b:
            db = torch.empty(N, device=dev, dtype=dt)
        dz, dz_ld = g2, _ld(g2)
        if (need_x or need_w) and (ctx.act or N % 8):
            dz_ld = _pitch(N)
            dz = torch.empty(M, dz_ld, device=dev, dtype=dt)
        if dz is not g2 or need_b:
            nb = L.lib().b200_linear_act_bwd_workspace_bytes(M, N) if need_b else 0
            ws = _scratch(nb, dev)
            _call("b200_linear_act_bwd", dev.index, g2.data_ptr(), _ld(g2), _ptr(z), _pitch(N), ctx.act, _PAIR[dt], M, N, dz.data_ptr() if dz is not g2 else None, dz_ld,
                  _ptr(db), _ptr(ws), nb)
        if (need_x or need_w) and dz is g2:
            dz, dz_ld = _tma_rows(g2)
        if need_x:
            dx = _product(dz, dz_ld, 0, w, w_ld, 1, M, K, N, ctx.x_shape)
        if need_w:
            dw = _product(dz, dz_ld, 1, x, x_ld, 1, N, K, M) if M else torch.zeros(N, K, device=dev, dtype=dt)
        return dx, dw, db, None, gy if need_r else None


def _assert_counts(M: int, N: int, K: int) -> None:
    """The library counts rows and columns in 32 bits, a tile's overhang included; ctypes would cut a larger number without a word."""
    assert M <= 1 << 30 and N <= 1 << 30 and K <= 1 << 30, f"rows, N and K are 2^30 at most, got {M}, {N}, {K}"


def _act_code(act) -> int:
    code = L.ACTIVATIONS.get(act)
    assert code is not None, f"act must be one of {sorted(a for a in L.ACTIVATIONS if a)} or None, got {act!r}"
    return code


def linear_act(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None, act: str | None = None, residual: torch.Tensor | None = None) -> torch.Tensor:
    """act(x w^T + bias) + residual: x [..., K], w [N, K], bias [N], residual [..., N], all bf16 or all fp16; act None, "relu", "silu", "gelu"
    (z Phi(z)) or "gelu_tanh".  fp32 accumulation, one rounding at the end.  Any K, N and number of rows up to 2^30; rows of x or w that do not start on
    16 bytes (a K that is no multiple of 8, an odd slice) are copied first.  Differentiable in x, w, bias and residual; with an activation a call
    that needs a gradient also keeps the pre-activation (N fp32 values per row)."""
    out = (_fast or _bind()).linear(x, w, bias, _ACT.get(act, -1), residual)
    if out is not None:
        return out
    _no_tangents(x, w, bias, residual)
    index, code, dt = _device(x, w, bias, residual), _act_code(act), x.dtype
    assert dt in _PAIR and w.dtype is dt and w.dim() == 2, "x and w must be both bfloat16 or both float16, w [N, K]"
    (N, K), xs = w.shape, x.shape
    assert xs and xs[-1] == K and K >= 1 and N >= 1, f"x {tuple(xs)} does not fit w {tuple(w.shape)}"
    _assert_counts(x.numel() // K, N, K)
    shape = (*xs[:-1], N)
    assert bias is None or (bias.dtype is dt and bias.shape == (N,)), "bias must be [N] in x's type"
    assert residual is None or (residual.dtype is dt and residual.shape == shape), "residual must have the type and shape of the result"
    if _wants_grad(x, w, bias, residual):
        return _LinearAct.apply(x, w, bias, code, residual)
    out = torch.empty(shape, device=x.device, dtype=dt)
    _linear_forward(index, dt, _operands(x, w, K), x.numel() // K, N, K, bias, code, residual, out, None, 0)
    return out


def linear_act_q8(x8: torch.Tensor, xsf: torch.Tensor, w8: torch.Tensor, s8: torch.Tensor, bias: torch.Tensor | None = None, act: str | None = None,
                  residual: torch.Tensor | None = None) -> torch.Tensor:
    """The projection on FP8 operands: x8 uint8 e4m3 [rows, K] + xsf uint8 E8M0 [rows, K/32] (`add_rms_norm_quant`, `cukern.mx_quantize_rows`), w8
    uint8 e4m3 [N, K] in natural k order (`w8.unpermute_k` of a W8's bytes) + s8 uint8 E8M0 [ceil(N/32), K/32].  bias [N], residual [rows, N] and
    the result bf16; products and sums in fp32.  K % 128 == 0.  No gradient."""
    out = (_fast or _bind()).q8(x8, xsf, w8, s8, bias, _ACT.get(act, -1), residual)
    if out is not None:
        return out
    _no_tangents(bias, residual)
    index, code, u8 = _device(x8, xsf, w8, s8, bias, residual), _act_code(act), torch.uint8
    assert x8.dtype is u8 and xsf.dtype is u8 and w8.dtype is u8 and s8.dtype is u8, "x8, xsf, w8 and s8 are uint8"
    assert x8.dim() == 2 and w8.dim() == 2 and xsf.dim() == 2 and s8.dim() == 2, "x8, xsf, w8 and s8 are matrices"
    (M, K), N = x8.shape, w8.shape[0]
    assert K % 128 == 0 and K > 0 and w8.shape[1] == K and N >= 1, f"x8 {tuple(x8.shape)} / w8 {tuple(w8.shape)}: the widths must be equal and a multiple of 128"
    _assert_counts(M, N, K)
    s_rows, s_cols = s8.shape
    assert s_cols < 1 << 31, f"s8 has {s_cols} columns"
    assert xsf.shape == (M, K // 32) and s_rows == (N + 31) // 32 and s_cols >= K // 32, "one scale per 32 k: xsf [rows, K/32], s8 [ceil(N/32), K/32]"
    assert bias is None or (bias.dtype is torch.bfloat16 and bias.shape == (N,)), "bias must be bfloat16 [N]"
    assert residual is None or (residual.dtype is torch.bfloat16 and residual.shape == (M, N)), "residual must be bfloat16 [rows, N]"
    assert not _wants_grad(x8, bias, residual), "linear_act_q8 has no gradient"
    x8, xsf, w8, s8 = x8.contiguous(), xsf.contiguous(), w8.contiguous(), s8.contiguous()
    residual, rp, r_ld = _mat(residual, N)
    if bias is not None:
        bias = bias.contiguous()
    out = torch.empty(M, N, device=x8.device, dtype=torch.bfloat16)
    nb = L.lib().b200_linear_act_q8_workspace_bytes(M, N, K)  # none for decode-sized calls
    ws = _scratch(nb, x8.device)
    _call("b200_linear_act_q8", index, x8.data_ptr(), xsf.data_ptr(), w8.data_ptr(), s8.data_ptr(), s_cols, M, N, K, _ptr(bias), code, rp, r_ld, out.data_ptr(), N, _ptr(ws),
          nb)
    return out


# ------------------------------------------------------------------ gated projection
def _gated_forward(index, dt, ops, M, inter, K, act, limit, out, gu, gu_ld):
    _, xp, x_ld, _, wp, w_ld = ops
    _call("b200_gated_linear", index, xp, x_ld, wp, w_ld, _PAIR[dt], M, inter, K, act, limit, out.data_ptr(), inter, _ptr(gu), gu_ld)


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w13, act, limit):
        n2, K = w13.shape
        inter = n2 // 2
        ops = _operands(x, w13, K)
        M = x.numel() // K
        out = torch.empty((*x.shape[:-1], inter), device=x.device, dtype=x.dtype)
        gu_ld = _pitch(n2)
        gu = torch.empty(M, gu_ld, device=x.device, dtype=torch.float32)
        _gated_forward(x.get_device(), x.dtype, ops, M, inter, K, act, limit, out, gu, gu_ld)
        ctx.save_for_backward(ops[0], ops[3], gu)
        ctx.dims, ctx.saved_shapes, ctx.act, ctx.limit, ctx.x_shape = (M, n2, K), (ops[0].shape, ops[3].shape), act, limit, x.shape
        return out

    @staticmethod
    def backward(ctx, gy):
        if not _grad_enabled():
            return _GatedLinear.gradients(ctx, gy)
        with torch.no_grad():
            dx, dw, _, _ = _GatedLinear.gradients(ctx, gy)
        return *_once([dx, dw], [[0, 1], [0, 1]], [gy]), None, None

    @staticmethod
    def gradients(ctx, gy):
        x, w, gu = ctx.saved_tensors
        need_x, need_w = ctx.needs_input_grad[:2]
        (M, n2, K), dev, dt = ctx.dims, gy.device, gy.dtype
        gu_ld = _pitch(n2)
        x, x_ld = _tma_rows(_restored(x, ctx.saved_shapes[0], dt, dev))
        w, w_ld = _tma_rows(_restored(w, ctx.saved_shapes[1], dt, dev))
        gu = _restored(gu, (M, gu_ld), torch.float32, dev).contiguous()
        g2 = _rows(gy)
        dx = dw = None
        dgu = torch.empty(M, gu_ld, device=dev, dtype=dt)
        _call("b200_gated_linear_bwd", dev.index, g2.data_ptr(), _ld(g2), gu.data_ptr(), gu_ld, ctx.act, ctx.limit, _PAIR[dt], M, n2 // 2, dgu.data_ptr(), gu_ld)
        if need_x:
            dx = _product(dgu, gu_ld, 0, w, w_ld, 1, M, K, n2, ctx.x_shape)
        if need_w:
            dw = _product(dgu, gu_ld, 1, x, x_ld, 1, n2, K, M) if M else torch.zeros(n2, K, device=dev, dtype=dt)
        return dx, dw, None, None


def gated_linear(x: torch.Tensor, w13: torch.Tensor, act: str | None = "silu", limit: float = 0.0) -> torch.Tensor:
    """act(min(g, limit)) * min(max(u, -limit), limit) with [g | u] = x w13^T, both projections and the product in one kernel: x [..., K], w13
    [2 * inter, K] (gate rows, then up rows: the layout of the expert weights), both bf16 or both fp16 -> [..., inter].  limit 0: no clamps.
    Differentiable in x and w13; a call that needs a gradient also keeps g and u (2 * inter fp32 values per row)."""
    out = (_fast or _bind()).gated(x, w13, _ACT.get(act, -1), limit)
    if out is not None:
        return out
    _no_tangents(x, w13)
    index, code, dt = _device(x, w13), _act_code(act), x.dtype
    assert dt in _PAIR and w13.dtype is dt and w13.dim() == 2, "x and w13 must be both bfloat16 or both float16, w13 [2 * inter, K]"
    (n2, K), xs = w13.shape, x.shape
    assert n2 >= 2 and n2 % 2 == 0 and K >= 1 and xs and xs[-1] == K, f"x {tuple(xs)} does not fit w13 {tuple(w13.shape)}"
    assert limit >= 0.0, "limit must not be negative"
    _assert_counts(x.numel() // K, n2, K)
    if _wants_grad(x, w13):
        return _GatedLinear.apply(x, w13, code, float(limit))
    out = torch.empty((*xs[:-1], n2 // 2), device=x.device, dtype=dt)
    _gated_forward(index, dt, _operands(x, w13, K), x.numel() // K, n2 // 2, K, code, float(limit), out, None, 0)
    return out


# ------------------------------------------------------------------ the block
class DenseFFN:
    """A non-expert feed-forward block on the residual stream: s = x + residual; h = gated_linear(norm(s), w13); returns h w2^T + s, the stream
    behind the block.

    w13 [2 * inter, D] and w2 [D, inter]: bf16 or fp16 tensors (trainable: every step is differentiable), or `W8` containers with E8M0 scales (D and
    inter multiples of 128, serving only): the normed rows and the gated product then stay in 8 bits between the steps, and with a limit the
    clamps take a NaN for the limit, as the expert kernels' do (in 16 bits it stays one).  A natural-k-order copy of the W8 bytes is made once here, as MoELayer
    does for the shared expert."""

    def __init__(self, norm_weight: torch.Tensor | None, w13, w2, *, eps: float = 1e-6, act: str = "silu", limit: float = 0.0):
        from .w8 import W8, unpermute_k
        self.norm_weight, self.eps, self.act, self.limit = norm_weight, eps, act, limit
        self.w13, self.w2 = w13, w2
        self.inter, self.dim = w13.shape[0] // 2, w13.shape[1]
        assert tuple(w2.shape) == (self.dim, self.inter) and w13.shape[0] == 2 * self.inter, f"w13 {tuple(w13.shape)} does not fit w2 {tuple(w2.shape)}"
        _act_code(act)
        assert limit >= 0.0, "limit must not be negative"
        self._nat = None
        if isinstance(w13, W8) or isinstance(w2, W8):
            assert isinstance(w13, W8) and isinstance(w2, W8) and w13.s8.dtype == torch.uint8 and w2.s8.dtype == torch.uint8, "w13 and w2: two W8 with E8M0 scales"
            assert self.dim % 128 == 0 and self.inter % 128 == 0 and act == "silu", "the FP8 block needs widths that are multiples of 128 and act 'silu'"
            self._nat = (unpermute_k(w13.w8), unpermute_k(w2.w8))

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
        """x, residual [..., D] -> [..., D]."""
        if self._nat is None:
            y, s = add_rms_norm(x, residual, self.norm_weight, self.eps)
            return linear_act(gated_linear(y, self.w13, self.act, self.limit), self.w2, residual=s)
        from . import cukern
        assert x.dtype == torch.bfloat16, "the FP8 block takes bfloat16 activations"
        q8, sf, s = add_rms_norm_quant(x, residual, self.norm_weight, self.eps)
        T = q8.shape[0]
        if T == 0:
            return s
        tpw = 128 if T > 64 else 32
        rows = 128
        while rows > 32 and (T + tpw - 1) // tpw * (self.inter // rows) < 148:
            rows //= 2
        h8, hsf = cukern.mx_grouped(self._nat[0], self.w13.s8, q8, sf, None, None, None, None, None, T, epilogue="swiglu_q8", limit=self.limit, tokens_per_work=tpw,
                                    rows_per_tile=rows)
        return linear_act_q8(h8, hsf, self._nat[1], self.w2.s8, residual=s.reshape(T, self.dim)).view(x.shape)

    __call__ = forward
