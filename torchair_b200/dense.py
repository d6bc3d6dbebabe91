"""torch.ops.npu.* operators of the layer's dense 16-bit parts: shared experts, projections and their training.

    npu_gated_ffn(x, weight1, weight2)     y = (act(x weight1[:, :I]) * (x weight1[:, I:])) weight2 (+ biases, + residual)
    npu_linear_act(x, weight)              y = act(x weight + bias) + residual
    npu_checkpoint_quant / _dequant        activations kept in int8, one fp32 scale per row and 64 values
    npu_checkpoint_weight_grad             x^T grad of a linear layer whose x was kept so

Weights are [in, out] like the grouped operators' [E, K, N]; a transposed view of an [out, in] parameter is used as it is.
The gate half of weight1 comes first (activate_left of npu_dequant_swiglu_quant).  bf16 and fp16; products and epilogues are
fp32, rounded once per result.  The first two are differentiable: the values before the activation are kept for the backward
pass in the input's type, or, with checkpoint_int8, together with x in 8 bits.  The backward pass then differentiates at the
kept values.  As everywhere in this package "CUDA" implementations launch on the current stream, "Meta" ones carry the shape
rules, there is no CPU implementation, and argument combinations that are not built raise.
"""
from __future__ import annotations

import contextlib

import torch

from . import _lib
from .ops import _npu, _ptr, _st, _workspace

_ACT = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
KEEP_BLOCK = 64        # values of a row that share a scale in an 8-bit checkpoint

_FFN = ("(Tensor x, Tensor weight1, Tensor weight2, *, Tensor? bias1=None, Tensor? bias2=None, Tensor? residual=None, "
        "str activation=\"silu\", bool checkpoint_int8=False) -> ")
_LINEAR = ("(Tensor x, Tensor weight, *, Tensor? bias=None, Tensor? residual=None, str activation=\"none\", "
           "bool checkpoint_int8=False) -> ")
_npu.define("npu_gated_ffn" + _FFN + "Tensor")
_npu.define("npu_gated_ffn_keep" + _FFN + "(Tensor, Tensor, Tensor, Tensor, Tensor)")
_npu.define("npu_gated_ffn_backward(Tensor grad, Tensor x, Tensor x_scale, Tensor weight1, Tensor weight2, Tensor kept, Tensor kept_scale, "
            "str activation, bool[] output_mask) -> (Tensor, Tensor, Tensor, Tensor, Tensor)")
_npu.define("npu_linear_act" + _LINEAR + "Tensor")
_npu.define("npu_linear_act_keep" + _LINEAR + "(Tensor, Tensor, Tensor, Tensor, Tensor)")
_npu.define("npu_linear_act_backward(Tensor grad, Tensor x, Tensor x_scale, Tensor weight, Tensor kept, Tensor kept_scale, "
            "str activation, bool[] output_mask) -> (Tensor, Tensor, Tensor)")
_npu.define("npu_checkpoint_quant(Tensor x) -> (Tensor, Tensor)")
_npu.define("npu_checkpoint_dequant(Tensor q, Tensor scale, *, int output_dtype=15) -> Tensor")
_npu.define("npu_checkpoint_weight_grad(Tensor q, Tensor scale, Tensor grad) -> Tensor")

OP_NAMES = ["npu_gated_ffn", "npu_gated_ffn_keep", "npu_gated_ffn_backward", "npu_linear_act", "npu_linear_act_keep",
            "npu_linear_act_backward", "npu_checkpoint_quant", "npu_checkpoint_dequant", "npu_checkpoint_weight_grad"]


# --------------------------------------------------------------------------------------------------
# helpers
# --------------------------------------------------------------------------------------------------
def _up(v: int, step: int) -> int:
    return -(-v // step) * step


def _on(t: torch.Tensor):
    """Context in which t's device is the current one (launches and their streams belong to the current device)."""
    return contextlib.nullcontext() if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _same(op: str, x: torch.Tensor, **others):
    for name, t in others.items():
        if t is None:
            continue
        if t.dtype != x.dtype:
            raise RuntimeError(f"{op}: `{name}` is {t.dtype}, x is {x.dtype}; all 16-bit tensors of a call have one dtype")
        if t.device != x.device:
            raise RuntimeError(f"{op}: `{name}` is on {t.device}, x is on {x.device}")


def _act_code(op: str, activation: str) -> int:
    if activation not in _ACT:
        raise RuntimeError(f"{op}: activation {activation!r} (one of {', '.join(_ACT)})")
    return _ACT[activation]


def _check16(op: str, x: torch.Tensor):
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise NotImplementedError(f"{op}: x must be bf16 or fp16, got {x.dtype}")


def _copy_2d(src: torch.Tensor, dst: torch.Tensor):
    """dst = src inside src's shape, zero elsewhere (2-D, 16-bit, any strides)."""
    _lib.call("tab_copy_2d", _ptr(src), src.stride(0), src.stride(1), src.shape[0], src.shape[1], _ptr(dst), dst.stride(0), dst.stride(1),
              dst.shape[0], dst.shape[1], _stream(src))


def _rows(t: torch.Tensor, cols: int) -> torch.Tensor:
    """t [m, n] as an operand contiguous along its rows with `cols` >= n columns (a multiple of 8): itself where its memory allows
    that, else a zero-padded copy."""
    if t.shape[1] == cols and t.stride(1) == 1 and t.data_ptr() % 16 == 0:
        if t.shape[0] <= 1:
            return t.as_strided(t.shape, (cols, 1))
        if t.stride(0) % 8 == 0 and t.stride(0) >= cols:
            return t
    out = torch.empty((t.shape[0], cols), dtype=t.dtype, device=t.device)
    _copy_2d(t, out)
    return out


def _matrix(t: torch.Tensor, rows: int, cols: int) -> torch.Tensor:
    """Like _rows for a weight [r, c], which may also be contiguous along its columns."""
    if t.shape == (rows, cols) and t.data_ptr() % 16 == 0:
        if t.stride(1) == 1 and t.stride(0) % 8 == 0 and t.stride(0) >= cols:
            return t
        if t.stride(0) == 1 and t.stride(1) % 8 == 0 and t.stride(1) >= rows:
            return t
    if t.stride(0) == 1 and t.stride(1) != 1:          # keep the order that the weight (and so its gradient) has
        out = torch.empty((cols, rows), dtype=t.dtype, device=t.device).t()
    else:
        out = torch.empty((rows, cols), dtype=t.dtype, device=t.device)
    _copy_2d(t, out)
    return out


def _halves(t: torch.Tensor, rows: int, half: int) -> torch.Tensor:
    """weight1 [H, 2 I] with either half padded to `half` columns, when I is not a multiple of 8."""
    inner = t.shape[1] // 2
    if inner == half:
        return _matrix(t, rows, 2 * half)
    if t.stride(0) == 1 and t.stride(1) != 1:
        out = torch.empty((2 * half, rows), dtype=t.dtype, device=t.device).t()
    else:
        out = torch.empty((rows, 2 * half), dtype=t.dtype, device=t.device)
    _copy_2d(t[:, :inner], out[:, :half])
    _copy_2d(t[:, inner:], out[:, half:])
    return out


def _vector(t, n: int):
    """A bias of n (padded) values, 16-byte aligned, or None."""
    if t is None or (t.shape[0] == n and t.stride(0) == 1 and t.data_ptr() % 16 == 0):
        return t
    return _rows(t.unsqueeze(0), n)[0]


def _as_b(t: torch.Tensor):
    """(ld, mn) of a 2-D operand [index of the product, contraction] that came from _rows or _matrix, or of its transpose."""
    return (t.stride(0), 0) if t.stride(1) == 1 else (t.stride(1), 1)


_ws_sizes = {}


def _ws_bytes(name: str, *dims: int) -> int:
    """Workspace sizes depend on the sizes and the number of SMs only; asking once per shape saves a foreign call."""
    key = (name, torch.cuda.current_device()) + dims
    size = _ws_sizes.get(key)
    if size is None:
        if len(_ws_sizes) > 4096:
            _ws_sizes.clear()
        size = _ws_sizes[key] = _lib.workspace_bytes(name, *dims)
    return size


def _matmul(a: torch.Tensor, b: torch.Tensor, *, bias=None, residual=None, act: int = 0, kept=None, kept_scale=None, out=None) -> torch.Tensor:
    """act(a b^T + bias) + residual for a [m, k], b [n, k] (either contiguous along either index); n a multiple of 8."""
    m, k = a.shape
    n = b.shape[0]
    if out is None:
        out = torch.empty((m, n), dtype=a.dtype, device=a.device)
    lda, a_mn = _as_b(a)
    ldb, b_mn = _as_b(b)
    nbytes = _ws_bytes("tab_dense_matmul_workspace_bytes", m, n, k)
    ws = _workspace(nbytes, a.device) if nbytes else None
    q = kept if kept_scale is not None else None
    _lib.call("tab_dense_matmul", a.data_ptr(), lda, a_mn, b.data_ptr(), ldb, b_mn, _st(a.dtype, "dense matmul"), m, n, k, _ptr(bias),
              _ptr(residual), act, None if q is not None else _ptr(kept), _ptr(q), _ptr(kept_scale), 0 if kept is None else kept.shape[1],
              out.data_ptr(), _ptr(ws), nbytes, _stream(a))
    return out


def _weight_grad(x: torch.Tensor, dz: torch.Tensor, like: torch.Tensor) -> torch.Tensor:
    """x^T dz [k, n], in the memory order of the weight `like`; x [m, k], dz [m, n] with rows contiguous."""
    if x.shape[0] == 0:
        return torch.zeros((x.shape[1], dz.shape[1]), dtype=x.dtype, device=x.device)
    if like.stride(0) == 1 and like.stride(1) != 1:
        return _matmul(dz.t(), x.t()).t()
    return _matmul(x.t(), dz.t())


def _act_grad(grad: torch.Tensor, act: int, kept, kept_scale, want_dz: bool, want_sums: bool):
    """(grad act'(kept), column sums of it), either of them None when not wanted (without an activation dz is grad itself)."""
    m, n = grad.shape
    dz = torch.empty((m, n), dtype=grad.dtype, device=grad.device) if want_dz and act else None
    sums = out = None
    if want_sums:
        splits = _ws_bytes("tab_act_grad_splits", m, n)
        sums = torch.empty((splits, n), dtype=torch.float32, device=grad.device)
        out = torch.empty((n,), dtype=grad.dtype, device=grad.device)
    if dz is not None or sums is not None:
        q = kept if kept_scale is not None else None
        _lib.call("tab_act_grad", grad.data_ptr(), grad.stride(0), _st(grad.dtype, "act grad"), m, n, act, None if q is not None else _ptr(kept),
                  _ptr(q), _ptr(kept_scale), 0 if kept is None else kept.shape[1], _ptr(dz), _ptr(sums), _stream(grad))
    if sums is not None:
        _lib.call("tab_column_sums", sums.data_ptr(), sums.shape[0], n, out.data_ptr(), _st(grad.dtype, "column sums"), _stream(grad))
    return (dz if act else grad), out


def _quant(x: torch.Tensor):
    """x [m, n] (rows contiguous) -> int8 [m, n], fp32 [m, ceil(n / 64)]."""
    m, n = x.shape
    q = torch.empty((m, n), dtype=torch.int8, device=x.device)
    scale = torch.empty((m, _up(n, KEEP_BLOCK) // KEEP_BLOCK), dtype=torch.float32, device=x.device)
    _lib.call("tab_checkpoint_quant", x.data_ptr(), _st(x.dtype, "npu_checkpoint_quant"), x.stride(0), m, n, q.data_ptr(), n,
              scale.data_ptr(), scale.shape[1], _stream(x))
    return q, scale


def _dequant(q: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype, cols: int = None) -> torch.Tensor:
    """int8 [m, n] with its scales -> dtype [m, cols], cols >= n zero-padded."""
    m, n = q.shape
    cols = n if cols is None else cols
    y = torch.empty((m, cols), dtype=dtype, device=q.device)
    _lib.call("tab_checkpoint_dequant", q.data_ptr(), q.stride(0), scale.data_ptr(), scale.stride(0), m, n, y.data_ptr(),
              _st(dtype, "npu_checkpoint_dequant"), cols, cols, _stream(q))
    return y


def _cut(t: torch.Tensor, shape) -> torch.Tensor:
    """The unpadded corner of a padded result, contiguous in the same order."""
    if tuple(t.shape) == tuple(shape):
        return t
    if t.dim() == 1:
        return _cut(t.unsqueeze(0), (1, shape[0]))[0]
    if t.stride(0) == 1 and t.stride(1) != 1:
        return _cut(t.t(), (shape[1], shape[0])).t()
    out = torch.empty(shape, dtype=t.dtype, device=t.device)
    _copy_2d(t[:shape[0], :shape[1]], out)
    return out


def _cut_halves(t: torch.Tensor, rows: int, inner: int) -> torch.Tensor:
    """[rows8, 2 I8] (or [2 I8]) -> [rows, 2 I] (or [2 I])"""
    if t.dim() == 1:
        return _cut_halves(t.unsqueeze(0), 1, inner)[0]
    half = t.shape[1] // 2
    if t.shape[0] == rows and half == inner:
        return t
    if t.stride(0) == 1 and t.stride(1) != 1:
        out = torch.empty((2 * inner, rows), dtype=t.dtype, device=t.device).t()
    else:
        out = torch.empty((rows, 2 * inner), dtype=t.dtype, device=t.device)
    _copy_2d(t[:rows, :inner], out[:, :inner])
    _copy_2d(t[:rows, half:half + inner], out[:, inner:])
    return out


def _empty(like: torch.Tensor, dtype=None) -> torch.Tensor:
    return torch.empty((0,), dtype=dtype or like.dtype, device=like.device)


# --------------------------------------------------------------------------------------------------
# npu_gated_ffn
# --------------------------------------------------------------------------------------------------
def _ffn_check(op, x, weight1, weight2, bias1, bias2, residual, activation):
    _check16(op, x)
    if x.dim() < 1 or weight1.dim() != 2 or weight2.dim() != 2:
        raise RuntimeError(f"{op}: x must be [..., H], weight1 [H, 2 I] and weight2 [I, H]")
    h = x.shape[-1]
    inner = weight2.shape[0]
    if h == 0 or inner == 0 or weight1.shape[0] != h or weight1.shape[1] != 2 * inner or weight2.shape[1] != h:
        raise RuntimeError(f"{op}: x {tuple(x.shape)}, weight1 {tuple(weight1.shape)} and weight2 {tuple(weight2.shape)} do not fit "
                           "[..., H], [H, 2 I] and [I, H]")
    if bias1 is not None and bias1.shape != (2 * inner,) or bias2 is not None and bias2.shape != (h,):
        raise RuntimeError(f"{op}: bias1 must be [2 I] = [{2 * inner}] and bias2 [H] = [{h}]")
    if residual is not None and residual.shape != x.shape:
        raise RuntimeError(f"{op}: residual must have the shape of x, got {tuple(residual.shape)}")
    _same(op, x, weight1=weight1, weight2=weight2, bias1=bias1, bias2=bias2, residual=residual)
    return _act_code(op, activation), h, inner


def _ffn_meta(x, weight1, weight2, *, bias1=None, bias2=None, residual=None, activation="silu", checkpoint_int8=False):
    _ffn_check("npu_gated_ffn", x, weight1, weight2, bias1, bias2, residual, activation)
    return torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _kept_meta(x, m, width, n_scales, checkpoint_int8):
    dev = x.device
    if checkpoint_int8:
        h = x.shape[-1]
        return (torch.empty((m, width), dtype=torch.int8, device=dev), torch.empty((m, n_scales), dtype=torch.float32, device=dev),
                torch.empty((m, h), dtype=torch.int8, device=dev),
                torch.empty((m, _up(h, KEEP_BLOCK) // KEEP_BLOCK), dtype=torch.float32, device=dev))
    return (torch.empty((m, width), dtype=x.dtype, device=dev), torch.empty((0,), dtype=torch.float32, device=dev),
            torch.empty((0,), dtype=torch.int8, device=dev), torch.empty((0,), dtype=torch.float32, device=dev))


def _ffn_keep_meta(x, weight1, weight2, *, bias1=None, bias2=None, residual=None, activation="silu", checkpoint_int8=False):
    _ffn_check("npu_gated_ffn", x, weight1, weight2, bias1, bias2, residual, activation)
    m = x.numel() // x.shape[-1]
    width = 2 * _up(weight2.shape[0], KEEP_BLOCK if checkpoint_int8 else 8)
    return (torch.empty(x.shape, dtype=x.dtype, device=x.device),) + _kept_meta(x, m, width, width // KEEP_BLOCK, checkpoint_int8)


def _ffn_forward(op, x, weight1, weight2, bias1, bias2, residual, activation, keep, checkpoint_int8):
    act, h, inner = _ffn_check(op, x, weight1, weight2, bias1, bias2, residual, activation)
    shape = x.shape
    x = x.reshape(-1, h)
    m = x.shape[0]
    h8, inner8 = _up(h, 8), _up(inner, 8)
    kept = kept_scale = x_q = x_scale = None
    with _on(x):
        if keep:
            if checkpoint_int8:
                xr = x if x.stride(1) == 1 else x.contiguous()
                x_q, x_scale = _quant(xr)
                kept = torch.empty((m, 2 * _up(inner, KEEP_BLOCK)), dtype=torch.int8, device=x.device)
                kept_scale = torch.empty((m, kept.shape[1] // KEEP_BLOCK), dtype=torch.float32, device=x.device)
            else:
                kept = torch.empty((m, 2 * inner8), dtype=x.dtype, device=x.device)
        y = torch.empty((m, h8), dtype=x.dtype, device=x.device)
        if m:
            xp = _rows(x, h8)
            w1, w2 = _halves(weight1, h8, inner8), _matrix(weight2, inner8, h8)
            if bias1 is not None:
                bias1 = _vector(bias1, 2 * inner8) if inner == inner8 else _halves(bias1.unsqueeze(0), 1, inner8)[0]
            bias2 = _vector(bias2, h8)
            if residual is not None:
                residual = _contiguous_rows(residual.reshape(m, h), h8)
            ld1, mn1 = _as_b(w1.t())
            ld2, mn2 = _as_b(w2.t())
            nbytes = _ws_bytes("tab_gated_ffn_workspace_bytes", m, h8, inner8)
            ws = _workspace(nbytes, x.device)
            q = kept if checkpoint_int8 else None
            _lib.call("tab_gated_ffn", xp.data_ptr(), xp.stride(0), w1.data_ptr(), ld1, mn1, w2.data_ptr(), ld2, mn2, _st(x.dtype, op), m, h8, inner8,
                      _ptr(bias1), _ptr(bias2), _ptr(residual), act, None if q is not None else _ptr(kept), _ptr(q), _ptr(kept_scale),
                      0 if kept is None else kept.shape[1], y.data_ptr(), ws.data_ptr(), nbytes, _stream(x))
        y = _cut(y, (m, h)).view(shape)
    return y, kept, kept_scale, x_q, x_scale


def _contiguous_rows(t: torch.Tensor, cols: int) -> torch.Tensor:
    """t [m, n] as [m, cols] without gaps between rows, 16-byte aligned."""
    if t.shape[1] == cols and t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t
    out = torch.empty((t.shape[0], cols), dtype=t.dtype, device=t.device)
    _copy_2d(t, out)
    return out


def _ffn_cuda(x, weight1, weight2, *, bias1=None, bias2=None, residual=None, activation="silu", checkpoint_int8=False):
    return _ffn_forward("npu_gated_ffn", x, weight1, weight2, bias1, bias2, residual, activation, False, False)[0]


def _ffn_keep_cuda(x, weight1, weight2, *, bias1=None, bias2=None, residual=None, activation="silu", checkpoint_int8=False):
    y, kept, kept_scale, x_q, x_scale = _ffn_forward("npu_gated_ffn", x, weight1, weight2, bias1, bias2, residual, activation, True, checkpoint_int8)
    if not checkpoint_int8:
        kept_scale, x_q, x_scale = _empty(x, torch.float32), _empty(x, torch.int8), _empty(x, torch.float32)
    return y, kept, kept_scale, x_q, x_scale


def _ffn_backward_meta(grad, x, x_scale, weight1, weight2, kept, kept_scale, activation, output_mask):
    _act_code("npu_gated_ffn_backward", activation)
    shapes = (grad.shape, weight1.shape, weight2.shape, (weight1.shape[1],), (weight2.shape[1],))
    return tuple(torch.empty(s if want else (0,), dtype=grad.dtype, device=grad.device) for s, want in zip(shapes, output_mask))


def _ffn_backward_cuda(grad, x, x_scale, weight1, weight2, kept, kept_scale, activation, output_mask):
    op = "npu_gated_ffn_backward"
    act, (inner, h) = _act_code(op, activation), weight2.shape
    want_x, want_w1, want_w2, want_b1, want_b2 = output_mask
    shape = grad.shape
    dtype = grad.dtype
    grad, x = grad.reshape(-1, h), x.reshape(-1, h)
    _same(op, grad, weight1=weight1, weight2=weight2)
    m = grad.shape[0]
    h8, inner8 = _up(h, 8), _up(inner, 8)
    int8 = kept.dtype == torch.int8
    dx = dw1 = dw2 = db1 = db2 = None
    with _on(grad):
        if m == 0:
            return tuple(torch.zeros(s if want else (0,), dtype=dtype, device=grad.device) for s, want in
                         zip((shape, weight1.shape, weight2.shape, (2 * inner,), (h,)), output_mask))
        dy = _rows(grad, h8)
        if want_x or want_w1 or want_w2 or want_b1:
            w2 = _matrix(weight2, inner8, h8)
            dz = torch.empty((m, 2 * inner8), dtype=dtype, device=grad.device)
            hidden = torch.empty((m, inner8), dtype=dtype, device=grad.device)
            ld2, mn2 = _as_b(w2)
            nbytes = _ws_bytes("tab_dense_matmul_workspace_bytes", m, inner8, h8)
            ws = _workspace(nbytes, grad.device) if nbytes else None
            _lib.call("tab_gated_matmul_grad", dy.data_ptr(), dy.stride(0), w2.data_ptr(), ld2, mn2, _st(dtype, op), m, inner8, h8, act,
                      None if int8 else kept.data_ptr(), kept.data_ptr() if int8 else None, kept_scale.data_ptr() if int8 else None,
                      kept.shape[1], dz.data_ptr(), hidden.data_ptr(), _ptr(ws), nbytes, _stream(grad))
        if want_w2:
            dw2 = _cut(_weight_grad(hidden, dy, weight2), (inner, h))
        if want_x:
            dx = _cut(_matmul(dz, _halves(weight1, h8, inner8)), (m, h)).view(shape)
        if want_w1:
            xp = _dequant(x, x_scale, dtype, h8) if x.dtype == torch.int8 else _rows(x, h8)
            dw1 = _cut_halves(_weight_grad(xp, dz, weight1), h, inner)
        if want_b1:
            db1 = _cut_halves(_act_grad(dz, 0, None, None, False, True)[1], 1, inner)
        if want_b2:
            db2 = _cut(_act_grad(dy, 0, None, None, False, True)[1], (h,))
    none = _empty(grad)
    return tuple(none if t is None else t for t in (dx, dw1, dw2, db1, db2))


class _GatedFfn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight1, weight2, bias1, bias2, residual, activation, checkpoint_int8):
        with torch._C._AutoDispatchBelowAutograd():
            y, kept, kept_scale, x_q, x_scale = torch.ops.npu.npu_gated_ffn_keep.default(
                x, weight1, weight2, bias1=bias1, bias2=bias2, residual=residual, activation=activation, checkpoint_int8=checkpoint_int8)
        ctx.save_for_backward(x_q if checkpoint_int8 else x, x_scale, weight1, weight2, kept, kept_scale)
        ctx.activation = activation
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        need = ctx.needs_input_grad
        mask = [need[0], need[1], need[2], need[3], need[4]]
        out = torch.ops.npu.npu_gated_ffn_backward.default(grad, *ctx.saved_tensors, ctx.activation, mask)
        return tuple(t if want else None for t, want in zip(out, mask)) + (grad if need[5] else None, None, None)


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _ffn_autograd(x, weight1, weight2, *, bias1=None, bias2=None, residual=None, activation="silu", checkpoint_int8=False):
    if _wants_grad(x, weight1, weight2, bias1, bias2, residual):
        return _GatedFfn.apply(x, weight1, weight2, bias1, bias2, residual, activation, checkpoint_int8)
    with torch._C._AutoDispatchBelowAutograd():
        return torch.ops.npu.npu_gated_ffn.default(x, weight1, weight2, bias1=bias1, bias2=bias2, residual=residual, activation=activation)


# --------------------------------------------------------------------------------------------------
# npu_linear_act
# --------------------------------------------------------------------------------------------------
def _linear_check(op, x, weight, bias, residual, activation):
    _check16(op, x)
    if x.dim() < 1 or weight.dim() != 2 or weight.shape[0] != x.shape[-1] or 0 in weight.shape:
        raise RuntimeError(f"{op}: x {tuple(x.shape)} and weight {tuple(weight.shape)} do not fit [..., K] and [K, N]")
    n = weight.shape[1]
    if bias is not None and bias.shape != (n,):
        raise RuntimeError(f"{op}: bias must be [N] = [{n}]")
    out_shape = x.shape[:-1] + (n,)
    if residual is not None and residual.shape != out_shape:
        raise RuntimeError(f"{op}: residual must be {tuple(out_shape)}, got {tuple(residual.shape)}")
    _same(op, x, weight=weight, bias=bias, residual=residual)
    return _act_code(op, activation), out_shape


def _linear_meta(x, weight, *, bias=None, residual=None, activation="none", checkpoint_int8=False):
    _, shape = _linear_check("npu_linear_act", x, weight, bias, residual, activation)
    return torch.empty(shape, dtype=x.dtype, device=x.device)


def _linear_keep_meta(x, weight, *, bias=None, residual=None, activation="none", checkpoint_int8=False):
    act, shape = _linear_check("npu_linear_act", x, weight, bias, residual, activation)
    m = x.numel() // x.shape[-1]
    y = torch.empty(shape, dtype=x.dtype, device=x.device)
    width = _up(weight.shape[1], KEEP_BLOCK if checkpoint_int8 else 8) if act else 0
    return (y,) + _kept_meta(x, m, width, width // KEEP_BLOCK, checkpoint_int8)


def _linear_forward(op, x, weight, bias, residual, activation, keep, checkpoint_int8):
    act, out_shape = _linear_check(op, x, weight, bias, residual, activation)
    k, n = weight.shape
    x = x.reshape(-1, k)
    m = x.shape[0]
    k8, n8 = _up(k, 8), _up(n, 8)
    kept = kept_scale = x_q = x_scale = None
    with _on(x):
        if keep:
            if checkpoint_int8:
                x_q, x_scale = _quant(x if x.stride(1) == 1 else x.contiguous())
            # without an activation the backward pass does not need its argument
            width = 0 if not act else _up(n, KEEP_BLOCK) if checkpoint_int8 else n8
            kept = torch.empty((m, width), dtype=torch.int8 if checkpoint_int8 else x.dtype, device=x.device)
            if checkpoint_int8:
                kept_scale = torch.empty((m, width // KEEP_BLOCK), dtype=torch.float32, device=x.device)
        y = torch.empty((m, n8), dtype=x.dtype, device=x.device)
        if m:
            if residual is not None:
                residual = _contiguous_rows(residual.reshape(m, n), n8)
            _matmul(_rows(x, k8), _matrix(weight, k8, n8).t(), bias=_vector(bias, n8), residual=residual, act=act,
                    kept=kept if act else None, kept_scale=kept_scale if act else None, out=y)
        y = _cut(y, (m, n)).view(out_shape)
    return y, kept, kept_scale, x_q, x_scale


def _linear_cuda(x, weight, *, bias=None, residual=None, activation="none", checkpoint_int8=False):
    return _linear_forward("npu_linear_act", x, weight, bias, residual, activation, False, False)[0]


def _linear_keep_cuda(x, weight, *, bias=None, residual=None, activation="none", checkpoint_int8=False):
    y, kept, kept_scale, x_q, x_scale = _linear_forward("npu_linear_act", x, weight, bias, residual, activation, True, checkpoint_int8)
    if not checkpoint_int8:
        kept_scale, x_q, x_scale = _empty(x, torch.float32), _empty(x, torch.int8), _empty(x, torch.float32)
    return y, kept, kept_scale, x_q, x_scale


def _linear_backward_meta(grad, x, x_scale, weight, kept, kept_scale, activation, output_mask):
    _act_code("npu_linear_act_backward", activation)
    shapes = (grad.shape[:-1] + (weight.shape[0],), weight.shape, (weight.shape[1],))
    return tuple(torch.empty(s if want else (0,), dtype=grad.dtype, device=grad.device) for s, want in zip(shapes, output_mask))


def _linear_backward_cuda(grad, x, x_scale, weight, kept, kept_scale, activation, output_mask):
    op = "npu_linear_act_backward"
    act, (k, n) = _act_code(op, activation), weight.shape
    want_x, want_w, want_b = output_mask
    x_shape = grad.shape[:-1] + (k,)
    dtype = grad.dtype
    grad, x = grad.reshape(-1, n), x.reshape(-1, k)
    _same(op, grad, weight=weight)
    m = grad.shape[0]
    k8, n8 = _up(k, 8), _up(n, 8)
    int8 = kept.dtype == torch.int8
    dx = dw = db = None
    with _on(grad):
        if m == 0:
            return tuple(torch.zeros(s if want else (0,), dtype=dtype, device=grad.device) for s, want in
                         zip((x_shape, weight.shape, (n,)), output_mask))
        dz, db = _act_grad(_rows(grad, n8), act, kept if act else None, kept_scale if act and int8 else None, want_x or want_w, want_b)
        if want_x:
            dx = _cut(_matmul(dz, _matrix(weight, k8, n8)), (m, k)).view(x_shape)
        if want_w:
            xp = _dequant(x, x_scale, dtype, k8) if x.dtype == torch.int8 else _rows(x, k8)
            dw = _cut(_weight_grad(xp, dz, weight), (k, n))
        if want_b:
            db = _cut(db, (n,))
    none = _empty(grad)
    return tuple(none if t is None else t for t in (dx, dw, db))


class _LinearAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation, checkpoint_int8):
        with torch._C._AutoDispatchBelowAutograd():
            y, kept, kept_scale, x_q, x_scale = torch.ops.npu.npu_linear_act_keep.default(
                x, weight, bias=bias, residual=residual, activation=activation, checkpoint_int8=checkpoint_int8)
        ctx.save_for_backward(x_q if checkpoint_int8 else x, x_scale, weight, kept, kept_scale)
        ctx.activation = activation
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        need = ctx.needs_input_grad
        mask = [need[0], need[1], need[2]]
        out = torch.ops.npu.npu_linear_act_backward.default(grad, *ctx.saved_tensors, ctx.activation, mask)
        return tuple(t if want else None for t, want in zip(out, mask)) + (grad if need[3] else None, None, None)


def _linear_autograd(x, weight, *, bias=None, residual=None, activation="none", checkpoint_int8=False):
    if _wants_grad(x, weight, bias, residual):
        return _LinearAct.apply(x, weight, bias, residual, activation, checkpoint_int8)
    with torch._C._AutoDispatchBelowAutograd():
        return torch.ops.npu.npu_linear_act.default(x, weight, bias=bias, residual=residual, activation=activation)


# --------------------------------------------------------------------------------------------------
# npu_checkpoint_quant, npu_checkpoint_dequant, npu_checkpoint_weight_grad
# --------------------------------------------------------------------------------------------------
def _ck_quant_meta(x):
    if x.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise NotImplementedError(f"npu_checkpoint_quant: x must be bf16, fp16 or fp32, got {x.dtype}")
    if x.dim() < 1:
        raise RuntimeError("npu_checkpoint_quant: x must have at least one dimension")
    return (torch.empty(x.shape, dtype=torch.int8, device=x.device),
            torch.empty(x.shape[:-1] + (_up(x.shape[-1], KEEP_BLOCK) // KEEP_BLOCK,), dtype=torch.float32, device=x.device))


def _ck_quant_cuda(x):
    q, scale = _ck_quant_meta(x)
    cols = x.shape[-1]
    if x.numel() == 0:
        return q, scale
    rows = x.numel() // cols
    if x.dim() != 2 or x.stride(1) != 1:
        x = x.contiguous().view(rows, cols)
    with _on(x):
        _lib.call("tab_checkpoint_quant", x.data_ptr(), _st(x.dtype, "npu_checkpoint_quant"), x.stride(0), rows, cols, q.data_ptr(), cols,
                  scale.data_ptr(), scale.shape[-1], _stream(x))
    return q, scale


def _ck_check(op, q, scale):
    if q.dtype != torch.int8 or scale.dtype != torch.float32:
        raise RuntimeError(f"{op}: q must be int8 and scale fp32, got {q.dtype} and {scale.dtype}")
    if q.dim() < 1 or scale.shape != q.shape[:-1] + (_up(q.shape[-1], KEEP_BLOCK) // KEEP_BLOCK,):
        raise RuntimeError(f"{op}: scale {tuple(scale.shape)} does not hold one value per row and {KEEP_BLOCK} values of q {tuple(q.shape)}")
    if q.device != scale.device:
        raise RuntimeError(f"{op}: q is on {q.device}, scale is on {scale.device}")


def _ck_dequant_meta(q, scale, *, output_dtype=15):
    _ck_check("npu_checkpoint_dequant", q, scale)
    dtype = {5: torch.float16, 6: torch.float32, 15: torch.bfloat16}.get(output_dtype)
    if dtype is None:
        raise NotImplementedError(f"npu_checkpoint_dequant: output_dtype={output_dtype} (5 fp16, 6 fp32 or 15 bf16)")
    return torch.empty(q.shape, dtype=dtype, device=q.device)


def _ck_dequant_cuda(q, scale, *, output_dtype=15):
    y = _ck_dequant_meta(q, scale, output_dtype=output_dtype)
    if y.numel() == 0:
        return y
    cols = q.shape[-1]
    q, scale = q.contiguous(), scale.contiguous()
    with _on(q):
        _lib.call("tab_checkpoint_dequant", q.data_ptr(), cols, scale.data_ptr(), scale.shape[-1], q.numel() // cols, cols, y.data_ptr(),
                  output_dtype, cols, cols, _stream(q))
    return y


def _ck_weight_grad_meta(q, scale, grad):
    op = "npu_checkpoint_weight_grad"
    _ck_check(op, q, scale)
    _check16(op, grad)
    if grad.dim() != q.dim() or grad.shape[:-1] != q.shape[:-1] or grad.shape[-1] == 0 or q.shape[-1] == 0:
        raise RuntimeError(f"{op}: q {tuple(q.shape)} and grad {tuple(grad.shape)} must be [..., K] and [..., N] of the same rows")
    if grad.device != q.device:
        raise RuntimeError(f"{op}: grad is on {grad.device}, q is on {q.device}")
    return torch.empty((q.shape[-1], grad.shape[-1]), dtype=grad.dtype, device=grad.device)


def _ck_weight_grad_cuda(q, scale, grad):
    out = _ck_weight_grad_meta(q, scale, grad)
    k, n = out.shape
    if q.numel() == 0:
        return out.zero_()
    q, scale, grad = q.contiguous().view(-1, k), scale.contiguous().view(-1, scale.shape[-1]), grad.reshape(-1, n)
    with _on(grad):
        x = _dequant(q, scale, grad.dtype, _up(k, 8))
        return _cut(_weight_grad(x, _rows(grad, _up(n, 8)), out), (k, n))


for _name, _meta, _cuda in (
        ("npu_gated_ffn", _ffn_meta, _ffn_cuda),
        ("npu_gated_ffn_keep", _ffn_keep_meta, _ffn_keep_cuda),
        ("npu_gated_ffn_backward", _ffn_backward_meta, _ffn_backward_cuda),
        ("npu_linear_act", _linear_meta, _linear_cuda),
        ("npu_linear_act_keep", _linear_keep_meta, _linear_keep_cuda),
        ("npu_linear_act_backward", _linear_backward_meta, _linear_backward_cuda),
        ("npu_checkpoint_quant", _ck_quant_meta, _ck_quant_cuda),
        ("npu_checkpoint_dequant", _ck_dequant_meta, _ck_dequant_cuda),
        ("npu_checkpoint_weight_grad", _ck_weight_grad_meta, _ck_weight_grad_cuda)):
    _npu.impl(_name, _meta, "Meta")
    _npu.impl(_name, _cuda, "CUDA")
for _name, _fn in (("npu_gated_ffn", _ffn_autograd), ("npu_linear_act", _linear_autograd)):
    _npu.impl(_name, _fn, "AutogradCUDA")

