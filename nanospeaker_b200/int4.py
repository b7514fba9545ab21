"""Weights in 4 bits with group scales, for batches that generate: few rows, so that the weights' bytes are
the time. W[k, n] = (level[k, n] - 8) * scale[k // group, n] with levels 0 .. 15.

  quantize_int4(w)     a weight (or a stack of them) rounded to an Int4Weight, once
  int4_mm(x, weight)   x @ W
  int4_experts(...)    the block's routed and shared GLU experts; beside `fused_moe_forward`, whose
                       weights are 16-bit

Inference only: there are no gradients. Kernels: csrc/int4.cu.
"""
from typing import Optional

import torch

from . import kernels as K
from .moe_kernel import _act_id, native_ok, refuse_forward_mode

INT4_DTYPES = (torch.bfloat16, torch.float16)
GROUPS = (32, 64, 128)      # inputs that share a scale
MAX_WIDTH = 2 ** 31 - 257
BLOCK, CHUNK, STRIP = 64, 8, 16   # inputs of a block, blocks of a chunk, outputs of a strip


class Int4Weight:
    """A matrix [K, N] (x @ W), or a stack [G, K, N] of them, in 4 bits, laid out as the kernels read it
    (include/moe_b200.h).

    shape     (K, N) or (G, K, N)
    group     inputs that share a scale: 32, 64 or 128 (the last group of a matrix may be short)
    dtype     of the scales, bf16 or fp16: that of the activations
    data      uint8 [G, bytes of a matrix] (G = 1 for a matrix), contiguous, on 16 bytes"""

    def __init__(self, data: torch.Tensor, shape, group: int, dtype: torch.dtype):
        shape = tuple(shape)
        if dtype not in INT4_DTYPES:
            raise ValueError(f"scales are bf16 or fp16, got {dtype}")
        _check_group(group)
        if len(shape) not in (2, 3):
            raise ValueError(f"a weight is [K, N] or [G, K, N], got {shape}")
        _check_widths(*shape[-2:])
        want = (shape[0] if len(shape) == 3 else 1, _matrix_bytes(*shape[-2:], group))
        if data.dtype != torch.uint8 or tuple(data.shape) != want or not data.is_contiguous():
            raise ValueError(f"a weight {shape} in groups of {group} is {want} bytes in one piece, got "
                             f"{data.dtype} {tuple(data.shape)}")
        if data.device.type != "meta" and data.data_ptr() % 16:
            raise ValueError("packed weights have to start on 16 bytes")
        self.data, self.shape, self.group, self.dtype = data, shape, group, dtype

    device = property(lambda self: self.data.device)

    def to(self, device) -> "Int4Weight":
        return Int4Weight(self.data.to(device), self.shape, self.group, self.dtype)

    @classmethod
    def from_levels(cls, levels: torch.Tensor, scales: torch.Tensor, group: int) -> "Int4Weight":
        """From uint8 levels [..., K, N] (0 .. 15, the value is level - 8) and scales
        [..., ceil(K / group), N]."""
        if levels.dtype != torch.uint8 or levels.dim() not in (2, 3):
            raise ValueError(f"levels are uint8 [K, N] or [G, K, N], got {levels.dtype} "
                             f"{tuple(levels.shape)}")
        if scales.dtype not in INT4_DTYPES:
            raise ValueError(f"scales are bf16 or fp16, got {scales.dtype}")
        _check_group(group)
        k, n = levels.shape[-2:]
        _check_widths(k, n)
        if bool((levels > 15).any()):
            raise ValueError("levels are 0 .. 15")
        if tuple(scales.shape) != (*levels.shape[:-2], -(-k // group), n):
            raise ValueError(f"levels {tuple(levels.shape)} in groups of {group} do not take scales "
                             f"{tuple(scales.shape)}")
        q = levels.reshape(-1, k, n)
        g, kb, ns = q.shape[0], -(-k // BLOCK), -(-n // STRIP)
        kg = -(-kb * BLOCK // group)
        if (kb * BLOCK, ns * STRIP) != (k, n):
            padded = q.new_full((g, kb * BLOCK, ns * STRIP), 8)
            padded[:, :k, :n] = q
            q = padded
        # input 64 kb + 32 half + 8 t + 4 j + 2 hi + b, output 16 ns + 8 i + lane row: bit 4 (2 hi + i) + 16 b
        # of word 2 half + j of lane 4 row + t
        q = q.view(g, kb, 2, 4, 2, 2, 2, ns, 2, 8)
        words = torch.zeros((), dtype=torch.int32, device=q.device)
        for hi in range(2):
            for b in range(2):
                for i in range(2):
                    part = q[:, :, :, :, :, hi, b, :, i].to(torch.int32)
                    words = words | (part << (4 * (2 * hi + i) + 16 * b))
        # [g, kb, half, t, j, ns, row] -> [g, kb, ns, row, t, half, j]
        words = words.permute(0, 1, 5, 6, 3, 2, 4).reshape(g, kb, ns, 512 // 4)
        s = scales.new_zeros((g, kg, ns * STRIP))
        s[:, :scales.shape[-2], :n] = scales.reshape(g, -1, n)
        s = s.view(g, kg, ns, 2, 8).transpose(3, 4).reshape(g, kg, ns, STRIP)
        # chunk by chunk, strip by strip: the levels of its blocks, its scales
        pieces = []
        for blocks, groups in _chunks(kb, kg, group):
            w = words[:, blocks].transpose(1, 2).reshape(g, ns, -1).view(torch.uint8)
            c = s[:, groups].transpose(1, 2).reshape(g, ns, -1).view(torch.uint8)
            pieces.append(torch.cat([w, c], 2).view(g, -1))
        return cls(torch.cat(pieces, 1) if len(pieces) > 1 else pieces[0], levels.shape, group,
                   scales.dtype)

    def to_levels(self):
        """(levels, scales) as from_levels takes them."""
        k, n = self.shape[-2:]
        g, kb, ns = self.data.shape[0], -(-k // BLOCK), -(-n // STRIP)
        kg = -(-kb * BLOCK // self.group)
        words, scales, at = [], [], 0
        for blocks, groups in _chunks(kb, kg, self.group):
            nb, ng = blocks.stop - blocks.start, groups.stop - groups.start
            size = nb * 512 + ng * 32
            piece = self.data[:, at:at + ns * size].view(g, ns, size)
            at += ns * size
            words.append(piece[:, :, :nb * 512].contiguous().view(torch.int32).view(g, ns, nb, 8, 4, 2, 2))
            scales.append(piece[:, :, nb * 512:].contiguous().view(self.dtype).view(g, ns, ng, 8, 2))
        words, s = torch.cat(words, 2), torch.cat(scales, 2)     # words: row, t, half, j
        one = torch.arange(2, device=self.device)
        bit = 8 * one[:, None, None] + 16 * one[None, :, None] + 4 * one[None, None, :]
        q = (words[..., None, None, None] >> bit.to(torch.int32)) & 15   # hi, b, i
        q = q.permute(0, 2, 5, 4, 6, 7, 8, 1, 9, 3).reshape(g, kb * BLOCK, ns * STRIP)[:, :k, :n]
        s = s.permute(0, 2, 1, 4, 3).reshape(g, kg, ns * STRIP)[:, :-(-k // self.group), :n]
        return (q.to(torch.uint8).reshape(self.shape),
                s.reshape(*self.shape[:-2], *s.shape[-2:]).contiguous())

    def dequantize(self) -> torch.Tensor:
        """The weight in fp32."""
        q, s = self.to_levels()
        k = q.shape[-2]
        return (q.float() - 8) * s.float().repeat_interleave(self.group, -2)[..., :k, :]


def _chunks(kb: int, kg: int, group: int):
    """(blocks, scale groups) of every chunk, as slices."""
    each = CHUNK * BLOCK // group
    for c in range(-(-kb // CHUNK)):
        yield (slice(c * CHUNK, min(kb, (c + 1) * CHUNK)), slice(c * each, min(kg, (c + 1) * each)))


def _check_group(group: int) -> None:
    if group not in GROUPS:
        raise ValueError(f"scale groups of {group} inputs: {GROUPS} are covered")


def _check_widths(k: int, n: int) -> None:
    if not (8 <= k <= MAX_WIDTH and 1 <= n <= MAX_WIDTH) or k % 8:
        raise ValueError(f"a weight of {k} inputs and {n} outputs: inputs have to be a multiple of 8, both below "
                         "2^31 - 256")


def _matrix_bytes(k: int, n: int, group: int) -> int:
    """moe_b200_int4_bytes."""
    kb = -(-k // BLOCK)
    return -(-n // STRIP) * (kb * 512 + -(-kb * BLOCK // group) * 32)


def quantize_int4(w: torch.Tensor, group: int = 64, dtype: Optional[torch.dtype] = None) -> Int4Weight:
    """w [K, N] or [G, K, N] rounded to 4 bits: a group's scale is its largest magnitude / 7, in `dtype`
    (default: w's, bf16 for fp32), its levels the nearest ones. Weights that are not finite, or too large for the scales, raise."""
    dtype = dtype or (w.dtype if w.dtype in INT4_DTYPES else torch.bfloat16)
    if w.dim() not in (2, 3):
        raise ValueError(f"a weight is [K, N] or [G, K, N], got {tuple(w.shape)}")
    if dtype not in INT4_DTYPES:
        raise ValueError(f"scales are bf16 or fp16, got {dtype}")
    _check_group(group)
    w = w.detach().float()
    if not bool(torch.isfinite(w).all()):
        raise ValueError("a weight with infinities or NaN cannot be held in 4 bits")
    k, n = w.shape[-2:]
    groups = -(-k // group)
    padded = torch.nn.functional.pad(w, (0, 0, 0, groups * group - k))
    blocks = padded.view(*w.shape[:-2], groups, group, n)
    scales = (blocks.abs().amax(-2) / 7).to(dtype)
    if not bool(torch.isfinite(scales).all()):
        raise ValueError(f"weights too large for scales in {dtype}")
    s = scales.float().unsqueeze(-2)
    levels = torch.where(s > 0, blocks / s, 0.0).round().clamp(-8, 7) + 8
    levels = levels.to(torch.uint8).view(*w.shape[:-2], groups * group, n)[..., :k, :].contiguous()
    return Int4Weight.from_levels(levels, scales, group)


def _check_types(x: torch.Tensor, *weights: Int4Weight) -> None:
    for w in weights:
        if not isinstance(w, Int4Weight):
            raise TypeError(f"expected an Int4Weight (quantize_int4 makes one), got {type(w).__name__}")
        if w.dtype != x.dtype:
            raise ValueError(f"activations in {x.dtype} with scales in {w.dtype}: they have to be alike")


def _check_call(x: torch.Tensor, tensors, weights) -> None:
    if not x.is_cuda or any(t.device != x.device for t in (*tensors, *weights)):
        raise ValueError("4-bit products take tensors of one CUDA device, got "
                         f"{[str(t.device) for t in (x, *tensors, *weights)]}")
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, *tensors)):
        raise RuntimeError("products with 4-bit weights have no gradients: call them under "
                           "torch.no_grad()")


@torch.library.custom_op("moe_b200::int4_mm", mutates_args=())
def _int4_mm(x: torch.Tensor, data: torch.Tensor, group: int, n_dim: int) -> torch.Tensor:
    with torch.cuda.device(x.device):
        return K.int4_mm(x, data, group, n_dim)


@_int4_mm.register_fake
def _(x, data, group, n_dim):
    return x.new_empty((x.shape[0], n_dim))


def int4_mm(x: torch.Tensor, weight: Int4Weight) -> torch.Tensor:
    """x [..., K] times a weight [K, N] held in 4 bits -> [..., N], in x's dtype (that of the scales).

    Made for few rows: up to 32 read the weight once, more read and convert it once per 32 (65535 * 32 rows at
    most). Past some 50 rows a 16-bit weight is the faster one (4096 x 4096, us of this / of a 16-bit product: 1 row
    7.7 / 14.8, 16 8.8 / 11.6, 64 13.3 / 11.4, 256 45 / 12, 4096 590 / 90); `dequantize` makes it, 0.6 ms. fp32 sums,
    rounded once; bitwise reproducible."""
    if type(weight) is Int4Weight and native_ok(x):
        out = K.shim().int4_mm(x, weight.data, weight.dtype, weight.shape, weight.group)
        if out is not None:
            return out
    refuse_forward_mode("int4_mm", x)
    _check_types(x, weight)
    if len(weight.shape) != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[0]:
        raise ValueError(f"int4_mm takes x [..., K] and one matrix [K, N], got {tuple(x.shape)} and "
                         f"{weight.shape}")
    _check_call(x, (), (weight,))
    out = _int4_mm(x.reshape(-1, x.shape[-1]), weight.data, weight.group, weight.shape[1])
    return out.view(*x.shape[:-1], weight.shape[1])


@torch.library.custom_op("moe_b200::int4_experts", mutates_args=())
def _int4_experts(x: torch.Tensor, topk_w: torch.Tensor, topk_idx: torch.Tensor, w_in: torch.Tensor,
                  w_out: torch.Tensor, shared_in: Optional[torch.Tensor],
                  shared_out: Optional[torch.Tensor], d_hidden: int, group: int, act: int) -> torch.Tensor:
    with torch.cuda.device(x.device):
        return K.int4_experts(x, topk_w.contiguous(), topk_idx.contiguous(), w_in, w_out, shared_in,
                              shared_out, d_hidden, group, act)


@_int4_experts.register_fake
def _(x, topk_w, topk_idx, w_in, w_out, shared_in, shared_out, d_hidden, group, act):
    return x.new_empty(x.shape)


def int4_experts(x: torch.Tensor, topk_w: torch.Tensor, topk_idx: torch.Tensor, w_in: Int4Weight,
                 w_out: Int4Weight, activation: str = "silu", shared_in: Optional[Int4Weight] = None,
                 shared_out: Optional[Int4Weight] = None) -> torch.Tensor:
    """out[t] = sum_j topk_w[t, j] * expert topk_idx[t, j] of x[t], plus every shared expert of x[t]; an
    expert is (act(gate) * up) @ w_out[e] with [gate | up] = x @ w_in[e].

    x         [T, D] bf16 or fp16
    topk_w    [T, k] in x's dtype, topk_idx [T, k] int64: what TopKRouter returns
    w_in      Int4Weight [E, D, 2H], w_out [E, H, D], H a multiple of 16, one scale group size for all
    shared_*  the same for the always-on experts, [S, D, 2H] and [S, H, D]

    No dispatch comes before it and nothing synchronises: made for batches that generate. (Of 32 experts of 1024 x
    768, four a token: 64 tokens 30 us, 1024 244, 8192 1800; sorting the pairs for `grouped_mm` with 16-bit weights,
    the rest in torch, takes 296, 309 and 858, so from some 1500 tokens that is the faster way.) Up to 65535 experts,
    the shared ones counted once per 8 to 32 tokens. An id outside
    [0, E) adds nothing and is reported by `kernels.check_status`. fp32 sums; the GLU's result keeps
    fp32's range and 16 bits or more; one rounding to x's dtype at the end; bitwise reproducible."""
    act = _act_id(activation)
    if native_ok(x):
        plain = _experts_fit(w_in, w_out, shared_in, shared_out)
        if plain is not None:
            out = K.shim().int4_experts(x, topk_w, topk_idx, *plain, act)
            if out is not None:
                return out
    refuse_forward_mode("int4_experts", x, topk_w)
    shared = () if shared_in is None and shared_out is None else (shared_in, shared_out)
    weights = (w_in, w_out, *shared)
    _check_types(x, *weights)
    if x.dim() != 2 or topk_idx.dim() != 2 or topk_w.shape != topk_idx.shape or \
            topk_idx.shape[0] != x.shape[0] or not 1 <= topk_idx.shape[1] < 2 ** 31:
        raise ValueError(f"int4_experts takes x [T, D] with topk_w and topk_idx [T, k], got "
                         f"{tuple(x.shape)}, {tuple(topk_w.shape)} and {tuple(topk_idx.shape)}")
    if topk_w.dtype != x.dtype or topk_idx.dtype != torch.int64:
        raise ValueError(f"topk_w has x's dtype and topk_idx is int64, got {topk_w.dtype} and "
                         f"{topk_idx.dtype}")
    d = x.shape[1]
    h = w_out.shape[1] if len(w_out.shape) == 3 else 0
    for pair in (weights[:2], weights[2:]):
        if pair and not (len(pair[0].shape) == len(pair[1].shape) == 3
                         and pair[0].shape == (pair[1].shape[0], d, 2 * h)
                         and pair[1].shape == (pair[0].shape[0], h, d)):
            raise ValueError(f"expert weights {pair[0].shape} and {pair[1].shape} do not fit "
                             f"d_model {d} and d_hidden {h}")
    if h % 16:
        raise ValueError(f"experts of width {h}: a multiple of 16 is covered")
    if len({w.group for w in weights}) > 1:
        raise ValueError("the experts' weights have scale groups of different sizes")
    _check_call(x, (topk_w, topk_idx), weights)
    sh = [w.data for w in shared] or [None] * 2
    return _int4_experts(x, topk_w, topk_idx, w_in.data, w_out.data, *sh, h, w_in.group, act)


def _experts_fit(w_in, w_out, shared_in, shared_out):
    """The arguments of the native call for expert weights that fit one another, else None (the caller
    then finds out what is wrong with them)."""
    if type(w_in) is not Int4Weight or type(w_out) is not Int4Weight:
        return None
    (e, d, h2), (e2, h, d2) = (w.shape if len(w.shape) == 3 else (0, 0, 0) for w in (w_in, w_out))
    if (h < 16 or h % 16 or h2 != 2 * h or e2 != e or d2 != d or w_in.group != w_out.group
            or w_in.dtype != w_out.dtype):
        return None
    if shared_in is None and shared_out is None:
        sh = (None, None)
    else:
        if type(shared_in) is not Int4Weight or type(shared_out) is not Int4Weight:
            return None
        s = shared_in.shape[0]
        if (shared_in.shape != (s, d, h2) or shared_out.shape != (s, h, d)
                or not shared_in.group == shared_out.group == w_in.group
                or not shared_in.dtype == shared_out.dtype == w_in.dtype):
            return None
        sh = (shared_in.data, shared_out.data)
    return (w_in.data, w_out.data, *sh, w_in.dtype, d, h, w_in.group)
