"""4-bit microscaled weights (OCP MXFP4) beside the lossless coders: ``convert_all_linear(model, algo="mxfp4")``.

A quarter of BF16's bytes (4.25 bits a value) for a rounding of every weight: blocks of 32 values along a row share a power of
two, each value is one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives.  :class:`MXFP4Weight` stands where a
:class:`HuffmanWeight` does: as the weight of ``F.linear`` or of a :class:`CompressedLinear`.  Products take BF16 activations as
they are (nothing but the weight is quantised), sum in 32 bits and round once; the gradient with respect to the input flows
through the frozen weight.  :func:`gated_mxfp4` is the first half of a gated feed-forward block in one kernel.

The reference has no counterpart.
"""
from __future__ import annotations

from typing import Callable, Optional, Tuple

import torch
import torch.nn.functional as F
from torch import Tensor, nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import ops, transfer

__all__ = ["MXFP4Weight", "linear_mxfp4", "gated_mxfp4", "GatedMXFP4", "GatedMLP"]

BLOCK = 32
ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2}
_TYPES = (torch.bfloat16, torch.float16, torch.float32)


class MXFP4Weight(nn.Module):
    """A ``[M, K]`` weight of 4-bit floats with a scale byte for every 32 (``K`` a multiple of 32).

    Buffers, padded with zeros to tiles of 16 rows and groups of 128 columns: ``codes`` u8 ``[ceil(M/16), ceil(K/128), 16, 4, 16]`` and
    ``scales`` u8 ``[ceil(M/16), ceil(K/128), 16, 4]``, in the order that the kernels read (``include/bf16_huffman_b200.h``);
    :meth:`from_packed` and :meth:`packed` translate from and to the plain order that checkpoints have.
    """

    algo = "mxfp4"

    def __init__(self, codes: Tensor, scales: Tensor, out_features: int, in_features: int):
        super().__init__()
        tiles, groups = _padded(out_features, in_features)
        for name, t, shape in (("codes", codes, (tiles, groups, 16, 4, 16)), ("scales", scales, (tiles, groups, 16, 4))):
            if t.dtype != torch.uint8 or tuple(t.shape) != shape:
                raise ValueError(f"{name} of a {out_features} x {in_features} weight must be u8 {shape}, not {t.dtype} {tuple(t.shape)}")
        # as register_buffer and nn.Module's attributes leave them, in a quarter of the time
        self._buffers.update(codes=codes, scales=scales)
        self.__dict__.update(out_features=int(out_features), in_features=int(in_features))

    @property
    def shape(self) -> Tuple[int, int]:
        return (self.out_features, self.in_features)

    def nbytes(self) -> int:
        return sum(b.nelement() * b.element_size() for b in self.buffers())

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        if func is not F.linear:
            return NotImplemented
        return linear_mxfp4(*args, **(kwargs or {}))

    def rows(self, lo: int, hi: int) -> "MXFP4Weight":
        """Rows ``lo`` to ``hi`` as a weight of their own."""
        codes, scales = self.packed()
        return type(self).from_packed(codes[lo:hi], scales[lo:hi])

    def get_weight(self) -> Tensor:
        """Dense BF16 ``[M, K]``: exactly the values that the products use."""
        b = self.__dict__["_buffers"]
        if not b["codes"].is_cuda:
            raise AssertionError("the dense matrix of a 4-bit weight is made on a CUDA device")
        return ops.dense_mxfp4(b["codes"], b["scales"], self.out_features, self.in_features)

    # -- making one ---------------------------------------------------------------------------
    @classmethod
    def compress(cls, a: Tensor, to_cpu: bool = True) -> "MXFP4Weight":
        """``a`` (BF16, FP16 or FP32) rounded to the format: the scale of a block is ``2^(floor(log2 max|v|) - 2)``, values go to
        the nearest code (ties to even) and saturate at 6 scales.  A block with an infinity or a NaN becomes NaN."""
        if a.dim() != 2 or a.dtype not in _TYPES:
            raise ValueError(f"want a matrix of BF16, FP16 or FP32, got {a.dtype} {tuple(a.shape)}")
        a = a.detach()
        if not a.is_cuda and not torch.cuda.is_available():
            raise RuntimeError("bf16_huffman_infer_b200 needs a CUDA device: there is no CPU implementation")
        if not a.is_cuda:
            a = a.to(torch.device("cuda", torch.cuda.current_device()))
        a = a.contiguous()
        if a.data_ptr() % 16:
            a = a.clone()
        tiles, groups = _padded(*a.shape)
        codes, scales = _empty(tiles, groups, a.device)
        ops.mxfp4_quantize(a, codes, scales)
        if to_cpu:
            codes, scales = transfer.download(codes), transfer.download(scales)
        return cls(codes, scales, *a.shape)

    @classmethod
    def from_packed(cls, codes: Tensor, scales: Tensor) -> "MXFP4Weight":
        """From the plain order: ``codes`` u8 ``[M, K/2]`` (the even element in the low half of a byte) and ``scales`` u8 ``[M, K/32]``
        (E8M0; also as ``torch.float8_e8m0fnu``), on their device.  A block with values beyond BF16's range (scale bytes 253 and 254:
        4 or 6 times 2^126, 2 and more times 2^127) becomes NaN, as one with an infinity does in :meth:`compress`; without them it is kept
        under the scale byte 252."""
        if scales.dtype == torch.float8_e8m0fnu:
            scales = scales.view(torch.uint8)
        if codes.dim() != 2 or codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or codes.size(1) % 16 \
                or tuple(scales.shape) != (codes.size(0), codes.size(1) // 16):
            raise ValueError(f"want codes u8 [M, K/2] and scales u8 [M, K/32], got {codes.dtype} {tuple(codes.shape)}, "
                             f"{scales.dtype} {tuple(scales.shape)}")
        M, K = codes.size(0), 2 * codes.size(1)
        tiles, groups = _padded(M, K)
        if codes.is_cuda:
            c, s = _empty(tiles, groups, codes.device)
            codes = codes.contiguous()
            ops.mxfp4_from_packed(codes.clone() if codes.data_ptr() % 4 else codes, scales.contiguous(), c, s)
            return cls(c, s, M, K)
        codes, scales = _within_range(codes.view(M, -1, 16), scales)
        s = F.pad(scales, (0, groups * 4 - K // 32, 0, tiles * 16 - M))
        # a NaN block holds zero codes
        c = codes.masked_fill((scales == 255)[..., None], 0).view(M, -1)
        c = F.pad(c, (0, groups * 64 - K // 2, 0, tiles * 16 - M)).view(tiles, 16, groups, 4, 4, 4)     # tile, row, group, block, quarter, byte
        low, high = c & 15, c >> 4
        byte = [low[..., 0] | low[..., 1] << 4, low[..., 2] | low[..., 3] << 4, high[..., 0] | high[..., 1] << 4, high[..., 2] | high[..., 3] << 4]
        c = torch.stack(byte, -1).permute(0, 2, 1, 4, 3, 5).reshape(tiles, groups, 16, 4, 16)
        return cls(c, s.view(tiles, 16, groups, 4).transpose(1, 2).contiguous(), M, K)

    def packed(self) -> Tuple[Tensor, Tensor]:
        """``(codes u8 [M, K/2], scales u8 [M, K/32])`` in the plain order; the inverse of :meth:`from_packed` (scale bytes 253 and 254 aside)."""
        M, K = self.shape
        tiles, groups = self.codes.shape[:2]
        c = self.codes.view(tiles, groups, 16, 4, 4, 4).permute(0, 2, 1, 4, 3, 5).reshape(tiles * 16, groups * 16, 4)
        low, high = c & 15, c >> 4
        byte = [low[..., 0] | low[..., 2] << 4, high[..., 0] | high[..., 2] << 4, low[..., 1] | low[..., 3] << 4, high[..., 1] | high[..., 3] << 4]
        c = torch.stack(byte, -1).view(tiles * 16, groups * 64)[:M, :K // 2].contiguous()
        return c, self.scales.transpose(1, 2).reshape(tiles * 16, groups * 4)[:M, :K // 32].contiguous()


def _within_range(codes: Tensor, scales: Tensor) -> Tuple[Tensor, Tensor]:
    """Blocks ``[M, blocks, 16]`` without the scale bytes 253 and 254: the same values under 252, or NaN where there is none."""
    up = torch.where((scales == 253) | (scales == 254), scales.int() - 252, 0)[..., None]
    if not bool(up.any()):
        return codes, scales
    # of 0, 0.5, 1, 1.5, 2, 3, 4, 6 the codes of once, twice and four times the value; 8: beyond the range
    table = torch.tensor([[0, 1, 2, 3, 4, 5, 6, 7], [0, 2, 4, 5, 6, 7, 8, 8], [0, 4, 6, 7, 8, 8, 8, 8]], dtype=torch.uint8, device=codes.device)
    low, high = table[up, (codes & 7).int()], table[up, (codes >> 4 & 7).int()]
    beyond = ((low | high) & 8 != 0).any(-1)
    scales = torch.where(up[..., 0] > 0, 252, scales).masked_fill(beyond, 255)
    return codes & 0x88 | low & 7 | (high & 7) << 4, scales.to(torch.uint8)


def _padded(M: int, K: int) -> Tuple[int, int]:
    """Tiles of rows and groups of columns of a weight."""
    if M < 1 or K < BLOCK or K % BLOCK:
        raise ValueError(f"an MXFP4 weight needs at least one row and a multiple of {BLOCK} columns, not {M} x {K}")
    return (M + 15) // 16, (K + 127) // 128


def _empty(tiles: int, groups: int, device: torch.device) -> Tuple[Tensor, Tensor]:
    return (torch.empty(tiles, groups, 16, 4, 16, dtype=torch.uint8, device=device),
            torch.empty(tiles, groups, 16, 4, dtype=torch.uint8, device=device))


_is_grad_enabled, _interpreter = torch.is_grad_enabled, torch._C._functorch.peek_interpreter_stack


def _recorded(x: Tensor, bias: Optional[Tensor]) -> bool:
    """Whether a call on these tensors is to be recorded for a backward pass."""
    return _is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad))


def _transformed() -> bool:
    """Whether a tangent, a batch dimension or a gradient of torch.func may ride on a tensor."""
    return forward_ad._current_level >= 0 or _interpreter() is not None


def _plain(x: Tensor) -> Tensor:
    """``x`` as the kernels read it: rows one after another from a 16-byte boundary."""
    if not x.is_contiguous():
        x = x.contiguous()
    return x.clone() if x.data_ptr() % 16 else x


def _under_autocast(input: Tensor, bias: Optional[Tensor]) -> Tuple[Tensor, Optional[Tensor]]:
    """Input and bias as ``torch.autocast`` to BF16 hands them to ``F.linear``; as they are without it."""
    if torch.is_autocast_enabled("cuda") and torch.get_autocast_dtype("cuda") is torch.bfloat16:
        input, bias = (t.to(torch.bfloat16) if t is not None and t.is_cuda and t.dtype in _TYPES else t for t in (input, bias))
    return input, bias


def _check(input: Tensor, weight: "MXFP4Weight", bias: Optional[Tensor]) -> None:
    """What the operators do not see for themselves."""
    if not input.is_cuda or input.dtype is not torch.bfloat16:
        raise AssertionError(f"products on 4-bit weights take BF16 tensors on a CUDA device, not {input.dtype} on {input.device}")
    if input.dim() < 1 or input.size(-1) != weight.in_features:
        raise RuntimeError(f"input of shape {tuple(input.shape)} does not fit a weight of {weight.in_features} columns")
    if bias is not None and (bias.dtype is not torch.bfloat16 or bias.shape != (weight.out_features,) or bias.device != input.device):
        raise RuntimeError(f"bias must be a BF16 vector of {weight.out_features} values on {input.device}")


def _product(x: Tensor, weight: "MXFP4Weight", bias: Optional[Tensor]) -> Tensor:
    b = weight.__dict__["_buffers"]
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    return ops.forward_mxfp4(_plain(x), b["codes"], b["scales"], weight.out_features, bias)


def _rows_of_eight(dy: Tensor) -> Tensor:
    """Rows of a gradient as the kernels read them: a multiple of 8 values apart."""
    dy = dy.flatten(0, -2) if dy.dim() > 1 else dy[None]
    if dy.size(1) % 8 == 0:
        return _plain(dy)
    out = dy.new_empty(dy.size(0), (dy.size(1) + 7) // 8 * 8)
    out[:, :dy.size(1)] = dy
    return out


class _Held:
    """Hands a weight through an autograd function, which would otherwise ask its ``__torch_function__`` about the call."""

    __slots__ = ("weight",)

    def __init__(self, weight: "MXFP4Weight"):
        self.weight = weight


def _linear_backward(ctx, dy: Tensor):
    dx = db = None
    if ctx.needs_input_grad[0]:
        dx = _LinearGradient.apply(dy, ctx.held) if _recorded(dy, None) or _transformed() else _input_gradient(dy, ctx.held.weight)
    if ctx.needs_input_grad[2]:
        db = dy.sum(tuple(range(dy.dim() - 1)), dtype=torch.float32).to(dy.dtype) if dy.dim() > 1 else dy
    return dx, None, db


class _Linear(torch.autograd.Function):
    """The product where only backward passes are asked of it: the form with a separate ``setup_context`` binds its arguments by signature
    in every call, which takes longer than the product of a small layer."""

    @staticmethod
    def forward(ctx, x, held, bias):
        ctx.held = held
        return _product(x, held.weight, bias)

    backward = staticmethod(_linear_backward)


class _LinearTransformed(torch.autograd.Function):
    """The same under the transformations of torch.func and forward-mode derivatives."""

    @staticmethod
    def forward(x, held, bias):
        return _product(x, held.weight, bias)

    @staticmethod
    def setup_context(ctx, inputs, output):
        ctx.held, ctx.shape = inputs[1], output.shape

    backward = staticmethod(_linear_backward)

    @staticmethod
    def jvp(ctx, dx, _, db):
        if dx is None:
            return db.expand(ctx.shape)
        return linear_mxfp4(dx, ctx.held.weight, db)

    @staticmethod
    def vmap(info, in_dims, x, held, bias):
        return _batched(info, in_dims, x, bias, lambda x, bias: linear_mxfp4(x, held.weight, bias))


def _input_gradient(dy: Tensor, weight: "MXFP4Weight") -> Tensor:
    b = weight.__dict__["_buffers"]
    dx = ops.mxfp4_linear_grad(_rows_of_eight(dy), b["codes"], b["scales"], weight.out_features, weight.in_features)
    return dx if dy.dim() == 2 else dx.view(*dy.shape[:-1], weight.in_features)


class _LinearGradient(torch.autograd.Function):
    """dx = dy W, itself linear in dy."""

    @staticmethod
    def forward(dy, held):
        return _input_gradient(dy, held.weight)

    @staticmethod
    def setup_context(ctx, inputs, output):
        ctx.held = inputs[1]

    @staticmethod
    def backward(ctx, ddx):
        return linear_mxfp4(ddx, ctx.held.weight), None

    @staticmethod
    def jvp(ctx, ddy, _):
        return _LinearGradient.apply(ddy, ctx.held)

    @staticmethod
    def vmap(info, in_dims, dy, held):
        return _LinearGradient.apply(dy.movedim(in_dims[0], 0), held), 0


def _batched(info, in_dims, x: Tensor, bias: Optional[Tensor], call: Callable) -> Tuple[Tensor, int]:
    """``call`` over a batch dimension of ``x``; a bias with one of its own is handed on item by item."""
    if in_dims[2] is None:
        return call(x.movedim(in_dims[0], 0), bias), 0
    bias = bias.movedim(in_dims[2], 0)
    x = x.expand(info.batch_size, *x.shape) if in_dims[0] is None else x.movedim(in_dims[0], 0)
    return torch.stack([call(a, b) for a, b in zip(x.unbind(0), bias.unbind(0))]), 0


def linear_mxfp4(input: Tensor, weight: MXFP4Weight, bias: Optional[Tensor] = None) -> Tensor:
    """``F.linear`` on a 4-bit weight: ``input`` BF16 ``[..., K]``, any number of rows; the bias (BF16, a value for each output) is part
    of the 32-bit sum.  Differentiable with respect to the input and the bias, also by forward-mode derivatives and under the
    transformations of ``torch.func``.  Under ``torch.autocast`` to BF16, FP32 and FP16 inputs and biases are cast; other types are
    refused."""
    if input.dtype is not torch.bfloat16 or (bias is not None and bias.dtype is not torch.bfloat16):
        input, bias = _under_autocast(input, bias)
    _check(input, weight, bias)
    if _transformed():
        return _LinearTransformed.apply(input, _Held(weight), bias)
    if _recorded(input, bias):
        return _Linear.apply(input, _Held(weight), bias)
    return _product(input, weight, bias)


class _Gated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, held, bias, activation):
        weight = held.weight
        ctx.held, ctx.activation = held, activation
        inter = weight.out_features // 2
        pre = torch.empty(*x.shape[:-1], 2 * inter, dtype=torch.float32, device=x.device)
        h = _gated(x, weight, bias, activation, pre)
        ctx.save_for_backward(pre)
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        pre, = ctx.saved_tensors
        w = ctx.held.weight
        b = w.__dict__["_buffers"]
        dpre = ops.mxfp4_gated_grad(pre, dh.contiguous(), ctx.activation)
        dx = db = None
        if ctx.needs_input_grad[0]:
            dx = ops.mxfp4_linear_grad(dpre, b["codes"], b["scales"], w.out_features, w.in_features).view(*dh.shape[:-1], w.in_features)
        if ctx.needs_input_grad[2]:
            db = dpre[:, :w.out_features].sum(0, dtype=torch.float32).to(dh.dtype)
        return dx, None, db, None


def _gated(x: Tensor, weight: MXFP4Weight, bias: Optional[Tensor], activation: int, pre: Optional[Tensor]) -> Tensor:
    b = weight.__dict__["_buffers"]
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    return ops.gated_mxfp4(_plain(x), b["codes"], b["scales"], weight.out_features, bias, activation, pre)


def gated_mxfp4(input: Tensor, weight: MXFP4Weight, bias: Optional[Tensor] = None, activation: str = "silu") -> Tensor:
    """``act(x G^T + b_g) * (x U^T + b_u)`` for the stacked weight ``[G; U]`` (gate rows first) and bias ``[b_g; b_u]``: BF16 ``[..., M/2]``
    from BF16 ``[..., K]`` in one kernel, the projections kept in 32 bits.  ``activation``: ``"silu"``, ``"gelu"`` or
    ``"gelu_tanh"``.  Differentiable once with respect to the input and the bias, by backward passes alone (forward-mode derivatives
    and the transformations of ``torch.func`` are refused); a call that may be differentiated keeps the projections (8 bytes a
    gated value) for the backward pass.  There the projections' gradients are rounded to BF16, the operand of the product that makes the
    input's, and that one once more: its error is 1.4 times that of one rounding (0.0023 against 0.0017 of its norm).  ``torch.autocast``
    as in :func:`linear_mxfp4`."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, not {activation!r}")
    if weight.out_features % 2:
        raise RuntimeError(f"a stacked weight has an even number of rows, not {weight.out_features}")
    if input.dtype is not torch.bfloat16 or (bias is not None and bias.dtype is not torch.bfloat16):
        input, bias = _under_autocast(input, bias)
    _check(input, weight, bias)
    if _recorded(input, bias) or _transformed():
        return _Gated.apply(input, _Held(weight), bias, ACTIVATIONS[activation])
    return _gated(input, weight, bias, ACTIVATIONS[activation], None)


class GatedMXFP4(nn.Module):
    """The gate and up projection of a feed-forward block with the activation and the product: :func:`gated_mxfp4` on its weight."""

    def __init__(self, weight: MXFP4Weight, bias: Optional[Tensor], activation: str):
        super().__init__()
        if activation not in ACTIVATIONS or weight.out_features % 2:
            raise ValueError(f"no gated pair: {weight.shape}, {activation!r}")
        self.weight = weight
        self.bias = bias
        self.activation = activation

    def forward(self, input: Tensor) -> Tensor:
        return gated_mxfp4(input, self.weight, self.bias, self.activation)


class GatedMLP(nn.Module):
    """``down_proj(act(gate_proj(x)) * up_proj(x))`` with the two first projections stacked."""

    def __init__(self, gate_up: GatedMXFP4, down_proj: nn.Module):
        super().__init__()
        self.gate_up = gate_up
        self.down_proj = down_proj

    def forward(self, x: Tensor) -> Tensor:
        return self.down_proj(self.gate_up(x))
