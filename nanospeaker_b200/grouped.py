"""Products grouped by expert over ragged runs, for any widths: what the block's fused GEMMs
(`moe_kernel.moe_experts`, expert width 128, bf16, runs padded to 128 rows) do not cover.

  y[r] = x[r] @ w[g]  for the rows r of run g,  offsets[g] <= r < offsets[g + 1]

and its two gradients, dx[r] = dy[r] @ w[g]^T and dw[g] = sum over run g of x[r]^T dy[r]. Runs lie back to
back, have any length (also none) and are known on the device only; nothing synchronises. Kernels:
csrc/grouped.cu.
"""
import torch

from . import kernels as K
from .moe_kernel import native_ok, refuse_forward_mode

MAX_GROUPS = 1024
MAX_WIDTH = 2 ** 31 - 257
GROUPED_DTYPES = (torch.bfloat16, torch.float16)


def _check(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor) -> None:
    if x.dim() != 2 or w.dim() != 3 or offsets.dim() != 1:
        raise ValueError(f"grouped_mm takes x [R, K], w [G, K, N] and offsets [G + 1], got "
                         f"{tuple(x.shape)}, {tuple(w.shape)} and {tuple(offsets.shape)}")
    if x.shape[1] != w.shape[1] or offsets.numel() != w.shape[0] + 1:
        raise ValueError(f"x {tuple(x.shape)}, w {tuple(w.shape)} and {offsets.numel()} offsets do not "
                         "fit together")
    if x.dtype not in GROUPED_DTYPES or w.dtype != x.dtype:
        raise ValueError(f"grouped_mm computes in bf16 or fp16, x and w alike; got {x.dtype} and "
                         f"{w.dtype}")
    if offsets.dtype != torch.int32:
        raise ValueError(f"offsets are int32, got {offsets.dtype}")
    if not (8 <= w.shape[1] <= MAX_WIDTH and 8 <= w.shape[2] <= MAX_WIDTH) or w.shape[1] % 8 or w.shape[2] % 8:
        raise ValueError(f"the widths of w {tuple(w.shape)} have to be multiples of 8, below 2^31 - 256")
    if not 1 <= w.shape[0] <= MAX_GROUPS:
        raise ValueError(f"{w.shape[0]} groups: 1 to {MAX_GROUPS} are covered")
    if not (x.is_cuda and x.device == w.device == offsets.device):
        raise ValueError(f"grouped_mm takes tensors of one CUDA device, got {x.device}, {w.device} and "
                         f"{offsets.device}")


@torch.library.custom_op("moe_b200::grouped_mm", mutates_args=())
def _grouped_mm(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    with torch.cuda.device(x.device):
        return K.grouped_mm(x, w, offsets.contiguous())


@_grouped_mm.register_fake
def _(x, w, offsets):
    return x.new_empty((x.shape[0], w.shape[2]))


@torch.library.custom_op("moe_b200::grouped_wgrad", mutates_args=())
def _grouped_wgrad(a: torch.Tensor, b: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    with torch.cuda.device(a.device):
        return K.grouped_wgrad(a, b, offsets.contiguous())


@_grouped_wgrad.register_fake
def _(a, b, offsets):
    return a.new_empty((offsets.numel() - 1, a.shape[1], b.shape[1]))


def _setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs)


def _gradients(x, w, offsets, dy, want_x, want_w):
    """(dx, dw), each None unless wanted; dw lies as w does."""
    dy = dy.to(x.dtype)
    dx = _grouped_mm(dy, w.transpose(1, 2), offsets) if want_x else None
    if not want_w:
        return dx, None
    if w.stride(1) == 1 and w.stride(2) != 1:
        return dx, _grouped_wgrad(dy, x, offsets).transpose(1, 2)
    return dx, _grouped_wgrad(x, dy, offsets)


def _backward(ctx, dy):
    return (*_gradients(*ctx.saved_tensors, dy, *ctx.needs_input_grad[:2]), None)


_grouped_mm.register_autograd(_backward, setup_context=_setup)


def grouped_mm(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """Rows offsets[g] .. offsets[g + 1] of x times w[g], for every group g; differentiable in x and w.

    x        [R, K], bf16 or fp16, rows sorted by group
    w        [G, K, N] of x's dtype, K and N multiples of 8, up to 1024 groups; also as a transposed view
             of a [G, N, K] tensor, read in place (its gradient then lies the same way)
    offsets  int32 [G + 1] on the device, not decreasing, within [0, R]

    Returns [R, N]. Rows of no run (before offsets[0], from offsets[G] on) give zeros and take zero
    gradients. Offsets that decrease or leave [0, R] are taken into range and reported by
    `kernels.check_status`. Sums are fp32, rounded once; both directions are bitwise reproducible. The
    gradients cannot be differentiated again."""
    if native_ok(x):
        y = K.shim().grouped_mm(x, w, offsets, MAX_GROUPS)
        if y is not None:
            return y
    refuse_forward_mode("grouped_mm", x, w)
    _check(x, w, offsets)
    return _grouped_mm(x, w, offsets)
