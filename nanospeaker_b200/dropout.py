"""Dropout whose mask is a function of the element's index and a state on the device, made again in the
backward and never stored: out = residual + dropout(x) in one pass.

The state `rng` is an int64 CUDA tensor (seed, call). An element's random word is one of the four of
Philox4x32-10 at counter (index // 4, call) under the key seed, so two calls with the same state drop the
same elements, and states that differ in either value are independent; the caller counts `call` up
(`rng[1] += 1`, on the device: also inside a captured graph, whose replays then differ). Kernel:
csrc/dropout.cu.
"""
from typing import Optional, Tuple

import torch

from . import kernels as K
from .moe_kernel import native_ok, refuse_forward_mode

DROPOUT_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


@torch.library.custom_op("moe_b200::dropout_add", mutates_args=())
def _dropout_add(x: torch.Tensor, residual: Optional[torch.Tensor], p: float,
                 rng: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(out, the state it was made with: rng may have moved on by the time of the backward)."""
    used = torch.empty_like(rng)
    with torch.cuda.device(x.device):
        return K.dropout(x, residual, p, rng, used), used


@_dropout_add.register_fake
def _(x, residual, p, rng):
    return torch.empty(x.shape, dtype=x.dtype, device=x.device), torch.empty_like(rng)


@torch.library.custom_op("moe_b200::dropout_bwd", mutates_args=())
def _dropout_bwd(grad: torch.Tensor, p: float, used: torch.Tensor) -> torch.Tensor:
    with torch.cuda.device(grad.device):
        return K.dropout(grad, None, p, used)


@_dropout_bwd.register_fake
def _(grad, p, used):
    return torch.empty(grad.shape, dtype=grad.dtype, device=grad.device)


def _setup(ctx, inputs, output):
    ctx.p = inputs[2]
    ctx.save_for_backward(output[1])
    ctx.mark_non_differentiable(output[1])


def _backward(ctx, grad, _):
    dx = _dropout_bwd(grad, ctx.p, ctx.saved_tensors[0]) if ctx.needs_input_grad[0] else None
    return dx, grad if ctx.needs_input_grad[1] else None, None, None


_dropout_add.register_autograd(_backward, setup_context=_setup)


def _bwd_setup(ctx, inputs, output):
    ctx.p = inputs[1]
    ctx.save_for_backward(inputs[2])


def _bwd_backward(ctx, grad):
    return _dropout_bwd(grad, ctx.p, ctx.saved_tensors[0]), None, None


_dropout_bwd.register_autograd(_bwd_backward, setup_context=_bwd_setup)   # (linear: the same mask again)


def dropout_add(x: torch.Tensor, residual: Optional[torch.Tensor], p: float,
                rng: torch.Tensor) -> torch.Tensor:
    """residual + x / (1 - p) where an element's random word is at least p * 2^32, residual alone where
    not; differentiable in x and residual.

    x         bf16, fp16 or fp32, any shape; elements are numbered in row-major order
    residual  the same shape and dtype, or None
    p         0 <= p < 1, in units of 2^-32
    rng       int64 [2] on x's device: (seed, call)

    A dropped element adds nothing even where it is infinite or NaN."""
    if native_ok(x):
        out = K.shim().dropout_add(x, residual, p, rng)
        if out is not None:
            return out
    refuse_forward_mode("dropout_add", x, residual)
    if x.dtype not in DROPOUT_DTYPES:
        raise ValueError(f"dropout computes in bf16, fp16 or fp32, got {x.dtype}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"the residual {tuple(residual.shape)} {residual.dtype} has to be as x, "
                         f"{tuple(x.shape)} {x.dtype}")
    if not 0 <= p < 1:
        raise ValueError(f"p ({p}) has to be in [0, 1)")
    if rng.dtype != torch.int64 or tuple(rng.shape) != (2,):
        raise ValueError(f"rng is int64 [2], (seed, call); got {rng.dtype} {tuple(rng.shape)}")
    if not x.is_cuda or rng.device != x.device or (residual is not None and residual.device != x.device):
        raise ValueError(f"dropout_add takes tensors of one CUDA device, got {x.device} and {rng.device}")
    return _dropout_add(x, residual, float(p), rng.contiguous())[0]
