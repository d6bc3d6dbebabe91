"""torch.ops.npu.* operators of the layer's dense 16-bit parts: shared experts, projections and their training.

    npu_gated_ffn(x, weight1, weight2)     y = (act(x weight1[:, :I]) * (x weight1[:, I:])) weight2 (+ biases, + residual)
    npu_linear_act(x, weight)              y = act(x weight + bias) + residual
    npu_checkpoint_quant / _dequant        activations kept in int8, one fp32 scale per row and 64 values
    npu_checkpoint_weight_grad             x^T grad of a linear layer whose x was kept so
                                           (x = q scale is rounded to grad's type first: it has to lie in its range, beyond 65504
                                           it is infinite in fp16 and below 2^-25 zero)

Weights are [in, out] like the grouped operators' [E, K, N]; a transposed view of an [out, in] parameter is used as it is.
The gate half of weight1 comes first (activate_left of npu_dequant_swiglu_quant).  bf16 and fp16; products and epilogues are
fp32.  A layer's result is rounded once; a block's hidden rows are rounded to 16 bits before the second product, as its operand, and so
are the derivatives that the gradient products take.  The first two are differentiable: the values before the activation are kept for the backward
pass in the input's type, or, with checkpoint_int8, together with x in 8 bits.  The backward pass then differentiates at the
kept values.  The *_keep and *_backward forms are what the gradients are made of; they and the checkpoint operators are not
differentiable themselves: a gradient through them raises when it is asked for.  Forward-mode differentiation raises everywhere.

As everywhere in this package the CUDA implementations launch on the current stream, the "Meta" ones (here) carry the shape
rules, there is no CPU implementation, and argument combinations that are not built raise.  The CUDA and autograd sides are C++
(csrc/torch_dense.cpp, libtorchair_b200_torch.so): at decode sizes a Python host path would take several times the kernel.
"""
from __future__ import annotations

import os

import torch

from . import _lib
from .ops import _npu

_ACT = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
KEEP_BLOCK = 64        # values of a row that share a scale in an 8-bit checkpoint

_FFN = ("(Tensor x, Tensor weight1, Tensor weight2, *, Tensor? bias1=None, Tensor? bias2=None, Tensor? residual=None, "
        "str activation=\"silu\", bool checkpoint_int8=False) -> ")
_LINEAR = ("(Tensor x, Tensor weight, *, Tensor? bias=None, Tensor? residual=None, str activation=\"none\", "
           "bool checkpoint_int8=False) -> ")
_npu.define("npu_gated_ffn" + _FFN + "Tensor")
_npu.define("npu_gated_ffn_keep" + _FFN + "(Tensor, Tensor, Tensor, Tensor, Tensor)")
_npu.define("npu_gated_ffn_backward(Tensor grad, Tensor x, Tensor x_scale, Tensor weight1, Tensor weight2, Tensor kept, Tensor kept_scale, "
            "str activation, bool[5] output_mask) -> (Tensor, Tensor, Tensor, Tensor, Tensor)")
_npu.define("npu_linear_act" + _LINEAR + "Tensor")
_npu.define("npu_linear_act_keep" + _LINEAR + "(Tensor, Tensor, Tensor, Tensor, Tensor)")
_npu.define("npu_linear_act_backward(Tensor grad, Tensor x, Tensor x_scale, Tensor weight, Tensor kept, Tensor kept_scale, "
            "str activation, bool[3] output_mask) -> (Tensor, Tensor, Tensor)")
_npu.define("npu_checkpoint_quant(Tensor x) -> (Tensor, Tensor)")
_npu.define("npu_checkpoint_dequant(Tensor q, Tensor scale, *, int output_dtype=15) -> Tensor")
_npu.define("npu_checkpoint_weight_grad(Tensor q, Tensor scale, Tensor grad) -> Tensor")

OP_NAMES = ["npu_gated_ffn", "npu_gated_ffn_keep", "npu_gated_ffn_backward", "npu_linear_act", "npu_linear_act_keep",
            "npu_linear_act_backward", "npu_checkpoint_quant", "npu_checkpoint_dequant", "npu_checkpoint_weight_grad"]


def _up(v: int, step: int) -> int:
    return -(-v // step) * step


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


# --------------------------------------------------------------------------------------------------
# shape rules
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


def _grad_meta(grad, shape, want):
    """An empty gradient: of a weight in the order in memory that the weight has, of anything else contiguous."""
    if not want:
        shape = (0,)
    elif isinstance(shape, torch.Tensor):
        if shape.stride(0) == 1 and shape.stride(1) != 1:
            return torch.empty(shape.shape[::-1], dtype=grad.dtype, device=grad.device).t()
        shape = shape.shape
    return torch.empty(shape, dtype=grad.dtype, device=grad.device)


def _ffn_backward_meta(grad, x, x_scale, weight1, weight2, kept, kept_scale, activation, output_mask):
    _act_code("npu_gated_ffn_backward", activation)
    shapes = (grad.shape, weight1, weight2, (weight1.shape[1],), (weight2.shape[1],))
    return tuple(_grad_meta(grad, s, want) for s, want in zip(shapes, output_mask))


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


def _linear_backward_meta(grad, x, x_scale, weight, kept, kept_scale, activation, output_mask):
    _act_code("npu_linear_act_backward", activation)
    shapes = (grad.shape[:-1] + (weight.shape[0],), weight, (weight.shape[1],))
    return tuple(_grad_meta(grad, s, want) for s, want in zip(shapes, output_mask))


def _ck_quant_meta(x):
    if x.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise NotImplementedError(f"npu_checkpoint_quant: x must be bf16, fp16 or fp32, got {x.dtype}")
    if x.dim() < 1:
        raise RuntimeError("npu_checkpoint_quant: x must have at least one dimension")
    return (torch.empty(x.shape, dtype=torch.int8, device=x.device),
            torch.empty(x.shape[:-1] + (_up(x.shape[-1], KEEP_BLOCK) // KEEP_BLOCK,), dtype=torch.float32, device=x.device))


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


def _ck_weight_grad_meta(q, scale, grad):
    op = "npu_checkpoint_weight_grad"
    _ck_check(op, q, scale)
    _check16(op, grad)
    if grad.dim() != q.dim() or grad.shape[:-1] != q.shape[:-1] or grad.shape[-1] == 0 or q.shape[-1] == 0:
        raise RuntimeError(f"{op}: q {tuple(q.shape)} and grad {tuple(grad.shape)} must be [..., K] and [..., N] of the same rows")
    if grad.device != q.device:
        raise RuntimeError(f"{op}: grad is on {grad.device}, q is on {q.device}")
    return torch.empty((q.shape[-1], grad.shape[-1]), dtype=grad.dtype, device=grad.device)


for _name, _meta in (
        ("npu_gated_ffn", _ffn_meta), ("npu_gated_ffn_keep", _ffn_keep_meta), ("npu_gated_ffn_backward", _ffn_backward_meta),
        ("npu_linear_act", _linear_meta), ("npu_linear_act_keep", _linear_keep_meta), ("npu_linear_act_backward", _linear_backward_meta),
        ("npu_checkpoint_quant", _ck_quant_meta), ("npu_checkpoint_dequant", _ck_dequant_meta),
        ("npu_checkpoint_weight_grad", _ck_weight_grad_meta)):
    _npu.impl(_name, _meta, "Meta")

if os.path.exists(_lib.TORCH_LIB_PATH):
    if os.path.exists(_lib.TORCH_LIB_PATH + ".torch"):       # written by _build.py
        with open(_lib.TORCH_LIB_PATH + ".torch") as _f:
            _built = _f.read()
        if not _built.startswith(torch.__version__ + " "):
            raise RuntimeError(f"{_lib.TORCH_LIB_PATH} was built against torch {_built}, installed is {torch.__version__}: build it "
                               "again with `python torchair_b200/_build.py`")
    torch.ops.load_library(_lib.TORCH_LIB_PATH)
else:
    def _missing(*args, **kwargs):
        raise RuntimeError(f"{_lib.TORCH_LIB_PATH} is missing: build it with `python -m torchair_b200._build`; torchair_b200 has no "
                           "fallback implementation")

    for _name in OP_NAMES:
        _npu.impl(_name, _missing, "CUDA")
