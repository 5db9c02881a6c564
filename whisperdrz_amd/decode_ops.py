"""Fused small operations of the decode step, backed by the gfx950 kernels in libwdrz_attn.so.

* :func:`add_layernorm_` — ``x += delta; return ln(x)``: the residual add closing a sub-layer
  and the LayerNorm opening the next (reference ``src/whisperdrz/model.py:420-433``, the final
  ``ln`` at ``model.py:609-613``), one launch instead of two.
* :func:`ln_linear` — the same add and LayerNorm inside the Linear that takes the result, for the
  one to four rows of a small step.
* :func:`masked_argmax` — ``decode_batch``'s greedy sampling tail (``decoding.py:1729-1761``):
  additive -65504 mask, repetition penalty, argmax, one launch instead of six.
* :func:`token_logprobs` — log probabilities of given tokens, entropy and top alternatives of each row, one pass.
* :func:`linear_gelu` — the MLP's ``Linear(n_state, 4 n_state)`` + ``GELU`` (``model.py:388-391``,
  applied at ``model.py:434``): GEMM, bias, rounding and exact GELU in one launch.
* :func:`linear4` — the same with 4-bit weights and group scales (:class:`QuantLinear4`).

There is no fallback: CPU tensors, fp32 LayerNorm inputs and a missing library raise.
"""
from __future__ import annotations

import functools
from typing import NamedTuple, Optional

import torch
import torch.nn as nn

from . import _lib
from .attention import (_check_cuda, _counted_workspace, _current_device, _dtype_code, _raise, _raw_stream, _stream_handle)

__all__ = ["QuantLinear4", "TokenLogprobs", "token_logprobs", "add_layernorm_", "layer_norm", "linear4", "linear4_partials", "linear_gelu", "ln_linear",
           "masked_argmax"]

_LN16 = {torch.bfloat16: _lib.WDRZ_BF16, torch.float16: _lib.WDRZ_F16}


def _rows(t: torch.Tensor, name: str) -> torch.Tensor:
    r = t.reshape(-1, t.shape[-1])
    if r.stride(-1) != 1 or r.data_ptr() != t.data_ptr():
        raise ValueError(f"{name} must have contiguous rows")
    return r


def add_layernorm_(x: torch.Tensor, delta: Optional[torch.Tensor], ln: nn.LayerNorm) -> torch.Tensor:
    """In place ``x += delta`` (when ``delta`` is given), then returns ``ln(x)`` (fp32 statistics)."""
    _check_cuda("x", x, x.device)
    if x.dtype not in _LN16:
        raise TypeError(f"x: dtype {x.dtype} is not supported (bfloat16, float16)")
    xr = _rows(x, "x")
    dr = None
    if delta is not None:
        _check_cuda("delta", delta, x.device)
        if delta.dtype != x.dtype or delta.shape != x.shape:
            raise ValueError("delta must match x in shape and dtype")
        dr = delta.reshape(xr.shape) if delta.is_contiguous() else delta.contiguous().reshape(xr.shape)
    w = ln.weight.detach()
    b = ln.bias.detach()
    if w.dtype != x.dtype:
        raise TypeError("the LayerNorm parameters must have the activations' dtype")
    y = torch.empty_like(xr)
    rc = _lib.load().wdrz_add_layernorm(
        _LN16[x.dtype], xr.data_ptr(), xr.stride(0), dr.data_ptr() if dr is not None else None,
        dr.stride(0) if dr is not None else 0, w.data_ptr(), b.data_ptr(), y.data_ptr(), y.stride(0),
        xr.shape[0], xr.shape[1], float(ln.eps), _stream_handle(),
    )
    if rc != _lib.WDRZ_OK:
        _raise(rc, "add_layernorm_")
    return y.view(x.shape)


def layer_norm(x: torch.Tensor, ln: nn.LayerNorm) -> torch.Tensor:
    return add_layernorm_(x, None, ln)


def masked_argmax(logits: torch.Tensor, blocked: Optional[torch.Tensor] = None,
                  penalty: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Greedy token per row of ``logits [rows, V]`` under the bool ``blocked`` mask (additive
    -65504) and the bool ``penalty`` mask (repetition penalty 1.2), as decode_batch computes it."""
    _check_cuda("logits", logits, logits.device)
    if logits.dim() == 3:
        logits = logits[:, -1, :]
    if logits.stride(-1) != 1:
        logits = logits.contiguous()
    rows, V = (int(v) for v in logits.shape)
    out = torch.empty(rows, dtype=torch.long, device=logits.device)
    masks = []
    for name, m in (("blocked", blocked), ("penalty", penalty)):
        if m is None:
            masks.append((None, 0))
            continue
        _check_cuda(name, m, logits.device)
        if m.dtype != torch.bool or m.shape[-1] < V or m.dim() != 2 or m.stride(-1) != 1:
            raise ValueError(f"{name} must be a bool [rows, >= V] tensor with contiguous rows")
        masks.append((m, m.stride(0)))
    rc = _lib.load().wdrz_masked_argmax(
        _dtype_code(logits, "logits"), logits.data_ptr(), logits.stride(0),
        masks[0][0].data_ptr() if masks[0][0] is not None else None, masks[0][1],
        masks[1][0].data_ptr() if masks[1][0] is not None else None, masks[1][1],
        out.data_ptr(), rows, V, _stream_handle(),
    )
    if rc != _lib.WDRZ_OK:
        _raise(rc, "masked_argmax")
    return out


class TokenLogprobs(NamedTuple):
    """``logprobs`` and ``entropy`` fp32 ``[...]``, ``top_logprobs`` fp32 and ``top_ids`` int64 ``[..., top]``."""

    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: torch.Tensor
    top_ids: torch.Tensor


@functools.lru_cache(maxsize=1024)
def _logprobs_workspace_size(rows: int, V: int, top: int) -> int:
    return int(_lib.load().wdrz_token_logprobs_workspace_size(rows, V, top))


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0,
                   blocked: Optional[torch.Tensor] = None) -> TokenLogprobs:
    """What ``logits`` ``[..., V]`` say about ``tokens`` ``[...]`` (int64): ``log_softmax(logits)`` at each token, the
    distribution's entropy in nats, and the ``top`` (0 .. 32) likeliest tokens, of equal ones the lower index first.
    bf16, fp16 or fp32 logits of up to 2^20 tokens; sums and results in fp32 or more. Inference only.

    ``blocked`` (bool ``[rows, >= V]``, as :func:`masked_argmax` takes it) are tokens that cannot be chosen: they count
    as -inf. A token out of range has NaN. A row that has nothing left has log probabilities of -inf, entropy 0
    and no alternatives; one with NaN or +inf among its tokens is NaN. Alternatives that do not exist have id -1.
    """
    if not (isinstance(logits, torch.Tensor) and logits.is_cuda):
        _check_cuda("logits", logits, logits.device if isinstance(logits, torch.Tensor) else None)
    device = logits.device
    dt = _dtype_code(logits, "logits")
    if logits.dim() < 1 or logits.shape[-1] == 0:
        raise ValueError("logits must be [..., V] with tokens")
    _check_cuda("tokens", tokens, device)
    shape, V = logits.shape[:-1], logits.shape[-1]
    if tokens.shape != shape or tokens.dtype is not torch.int64:
        raise ValueError(f"tokens must be int64 {tuple(shape)}, got {tokens.dtype} {tuple(tokens.shape)}")
    x = logits if logits.dim() == 2 else logits.reshape(-1, V)
    if x.stride(1) != 1 and V > 1 or x.stride(0) < 0:
        x = x.contiguous()
    rows = x.shape[0]
    if not tokens.is_contiguous():
        tokens = tokens.contiguous()
    mask, m_stride = None, 0
    if blocked is not None:
        _check_cuda("blocked", blocked, device)
        if blocked.dtype is not torch.bool or blocked.dim() != 2 or blocked.shape[0] != rows or blocked.shape[1] < V \
                or blocked.stride(1) != 1:
            raise ValueError(f"blocked must be a bool [{rows}, >= {V}] tensor with contiguous rows")
        mask, m_stride = blocked.data_ptr(), blocked.stride(0)
    index = device.index
    if index != _current_device():  # launches go to the current device
        with torch.cuda.device(index):
            return token_logprobs(logits, tokens, top, blocked)
    logprobs = torch.empty(*(shape or ((),)), dtype=torch.float32, device=device)
    entropy = torch.empty_like(logprobs)
    top_logprobs = logprobs.new_empty(*shape, max(top, 0))
    top_ids = tokens.new_empty(*shape, max(top, 0))
    lib, nbytes = _lib.load(), _logprobs_workspace_size(rows, V, max(top, 0))
    workspace = _counted_workspace(device, nbytes) if nbytes else None
    rc = lib.wdrz_token_logprobs(
        dt, x.data_ptr(), x.stride(0), mask, m_stride, tokens.data_ptr(), logprobs.data_ptr(), entropy.data_ptr(),
        top_logprobs.data_ptr(), top_ids.data_ptr(), rows, V, top, None if workspace is None else workspace.data_ptr(),
        0 if workspace is None else workspace.numel(), _raw_stream(index))
    if rc != _lib.WDRZ_OK:
        _raise(rc, "token_logprobs")
    return TokenLogprobs(logprobs, entropy, top_logprobs, top_ids)


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], gelu: bool = False) -> torch.Tensor:
    """``x @ weight.T + bias`` (``gelu``: then the exact GELU) for 16-bit ``x [..., K]``, rounded
    like torch's 16-bit modules: the Linear's output to the storage type, then the GELU's."""
    _check_cuda("x", x, x.device)
    if x.dtype not in _LN16:
        raise TypeError(f"x: dtype {x.dtype} is not supported (bfloat16, float16)")
    xr = _rows(x, "x")
    w = weight.detach()
    b = bias.detach() if bias is not None else None
    if w.dtype != x.dtype or (b is not None and b.dtype != x.dtype):
        raise TypeError("the Linear's parameters must have the activations' dtype")
    if w.stride(-1) != 1 or w.shape[1] != xr.shape[1]:
        raise ValueError("weight must be [N, K] with contiguous rows and K = x.shape[-1]")
    if b is not None and not b.is_contiguous():
        b = b.contiguous()
    N = int(w.shape[0])
    y = torch.empty(xr.shape[0], N, dtype=x.dtype, device=x.device)
    rc = _lib.load().wdrz_linear(
        _LN16[x.dtype], xr.data_ptr(), xr.stride(0), w.data_ptr(), w.stride(0),
        b.data_ptr() if b is not None else None, y.data_ptr(), y.stride(0),
        xr.shape[0], N, xr.shape[1], 1 if gelu else 0, _stream_handle(),
    )
    if rc != _lib.WDRZ_OK:
        _raise(rc, "linear")
    return y.view(*x.shape[:-1], N)


def linear_gelu(x: torch.Tensor, lin: nn.Linear, gelu: bool = True) -> torch.Tensor:
    """``GELU(lin(x))`` (``gelu=False``: ``lin(x)``) for 16-bit ``x [..., K]``, rounded like the
    reference's two modules: the Linear's output to the storage type, then the GELU's."""
    return linear(x, lin.weight, lin.bias, gelu)


def linear_partials(x: torch.Tensor, lin: nn.Linear, n_split: int = 4) -> torch.Tensor:
    """fp32 split-K partial products of ``lin`` (no bias) for 16-bit ``x [..., K]``: a tensor
    ``[n_split, rows, N]`` whose sum over the first dimension is ``x @ lin.weight.T``; its
    consumer (``add_layernorm_partials_``) adds the bias and rounds like the Linear's output."""
    _check_cuda("x", x, x.device)
    if x.dtype not in _LN16:
        raise TypeError(f"x: dtype {x.dtype} is not supported (bfloat16, float16)")
    xr = _rows(x, "x")
    w = lin.weight.detach()
    if w.dtype != x.dtype:
        raise TypeError("the Linear's parameters must have the activations' dtype")
    if w.stride(-1) != 1 or w.shape[1] != xr.shape[1]:
        raise ValueError("weight must be [N, K] with contiguous rows and K = x.shape[-1]")
    N = int(w.shape[0])
    part = torch.empty(n_split, xr.shape[0], N, dtype=torch.float32, device=x.device)
    rc = _lib.load().wdrz_linear_partials(
        _LN16[x.dtype], xr.data_ptr(), xr.stride(0), w.data_ptr(), w.stride(0), part.data_ptr(),
        xr.shape[0], N, xr.shape[1], n_split, _stream_handle(),
    )
    if rc != _lib.WDRZ_OK:
        _raise(rc, "linear_partials")
    return part


def add_layernorm_partials_(x: torch.Tensor, partials: torch.Tensor, lin: nn.Linear,
                            ln: nn.LayerNorm) -> torch.Tensor:
    """In place ``x += lin(h)`` where ``partials = linear_partials(h, lin)`` (the sum of the
    partials plus ``lin.bias``, rounded to ``x``'s type like the Linear's output), then returns
    ``ln(x)`` as ``add_layernorm_`` does."""
    _check_cuda("x", x, x.device)
    if x.dtype not in _LN16:
        raise TypeError(f"x: dtype {x.dtype} is not supported (bfloat16, float16)")
    xr = _rows(x, "x")
    n_split = int(partials.shape[0])
    if partials.dtype != torch.float32 or tuple(partials.shape[1:]) != tuple(xr.shape) or not partials.is_contiguous():
        raise ValueError("partials must be contiguous fp32 [n_split, rows, n] matching x")
    if lin.bias is None:
        raise ValueError("the Linear must have a bias")
    db = lin.bias.detach()
    w = ln.weight.detach()
    b = ln.bias.detach()
    if w.dtype != x.dtype or db.dtype != x.dtype:
        raise TypeError("the LayerNorm and Linear parameters must have the activations' dtype")
    y = torch.empty_like(xr)
    rc = _lib.load().wdrz_add_layernorm_partials(
        _LN16[x.dtype], xr.data_ptr(), xr.stride(0), partials.data_ptr(), n_split, db.data_ptr(),
        w.data_ptr(), b.data_ptr(), y.data_ptr(), y.stride(0), xr.shape[0], xr.shape[1], float(ln.eps),
        _stream_handle(),
    )
    if rc != _lib.WDRZ_OK:
        _raise(rc, "add_layernorm_partials_")
    return y.view(x.shape)


def _check_linear4_sizes(lin: "QuantLinear4", packed: torch.Tensor, scales: torch.Tensor, bias: Optional[torch.Tensor]) -> None:
    """The kernels read all of a layer's buffers: they have to be as large as its features say."""
    N, K = lin.out_features, lin.in_features
    tiles = -(-N // 16)
    if packed.shape != (tiles, -(-K // 128), 1024) or scales.shape != (tiles, K // lin.group, 16) \
            or not (packed.is_contiguous() and scales.is_contiguous()):
        raise ValueError(f"packed {tuple(packed.shape)} and scales {tuple(scales.shape)} must be contiguous "
                         f"{(tiles, -(-K // 128), 1024)} and {(tiles, K // lin.group, 16)}")
    if bias is not None and (bias.shape != (N,) or not bias.is_contiguous()):
        raise ValueError(f"bias {tuple(bias.shape)} must be contiguous [{N}]")


class QuantLinear4(nn.Module):
    """A Linear with 4-bit weights: ``weight[n, k] = codes[n, k] * scales[n, k // group]``, codes whole
    numbers -7..7 and scales of the activations' 16-bit type, packed once for :func:`linear4`.

    ``from_linear`` rounds a 16-bit Linear, ``from_codes`` takes codes and scales from elsewhere. ``group`` is
    32, 64 or 128 and divides the inputs. Inference only: the weights are buffers without gradients, contiguous,
    ``packed`` uint8 ``[ceil(N / 16), ceil(K / 128), 1024]``, ``scales`` ``[ceil(N / 16), K / group, 16]``, ``bias`` ``[N]``."""

    GROUPS = (32, 64, 128)

    def __init__(self, in_features: int, out_features: int, group: int, packed: torch.Tensor, scales: torch.Tensor,
                 bias: Optional[torch.Tensor]):
        super().__init__()
        if group not in self.GROUPS or in_features <= 0 or out_features <= 0 or in_features % group:
            raise NotImplementedError(f"group {group} must be one of {self.GROUPS} and divide the {in_features} inputs "
                                      f"of {out_features} outputs")
        if packed.dtype is not torch.uint8 or scales.dtype not in _LN16 or (bias is not None and bias.dtype != scales.dtype):
            raise TypeError("packed must be uint8, scales and bias share a 16-bit dtype (bfloat16, float16)")
        if scales.device != packed.device or (bias is not None and bias.device != packed.device):
            raise ValueError("packed, scales and bias must be on one device")
        self.in_features, self.out_features, self.group = in_features, out_features, group
        _check_linear4_sizes(self, packed, scales, bias)
        self.register_buffer("packed", packed)
        self.register_buffer("scales", scales)
        self.register_buffer("bias", bias)

    @classmethod
    def from_codes(cls, codes: torch.Tensor, scales: torch.Tensor, bias: Optional[torch.Tensor] = None) -> "QuantLinear4":
        """``codes`` ``[N, K]`` whole numbers -7..7, ``scales`` ``[N, K / group]`` (bf16 or fp16), ``bias`` ``[N]``."""
        if codes.dim() != 2 or scales.dim() != 2 or scales.shape[0] != codes.shape[0] or codes.shape[0] == 0 \
                or scales.shape[1] == 0 or codes.shape[1] % scales.shape[1]:
            raise ValueError(f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} must be [N, K] and [N, K / group]")
        N, K = (int(n) for n in codes.shape)
        group = K // int(scales.shape[1])
        if group not in cls.GROUPS:
            raise NotImplementedError(f"group {group} is not one of {cls.GROUPS}")
        if scales.dtype not in _LN16 or (bias is not None and (bias.dtype != scales.dtype or tuple(bias.shape) != (N,))):
            raise TypeError("scales and bias must share a 16-bit dtype (bfloat16, float16), bias [N]")
        if codes.is_floating_point() or codes.is_complex() or codes.dtype == torch.bool:
            raise TypeError(f"codes: dtype {codes.dtype} is not a whole type")
        codes = codes.detach()
        if bool(((codes < -7) | (codes > 7)).any()):
            raise ValueError("codes must lie in -7..7")
        tiles, chunks = -(-N // 16), -(-K // 128)
        nib = codes.abs().to(torch.uint8) | ((codes < 0).to(torch.uint8) << 3)
        full = torch.zeros(tiles * 16, chunks * 128, dtype=torch.uint8, device=codes.device)
        full[:N, :K] = nib
        # [tile, n, chunk, s, g, half, i] -> [tile, chunk, g, n, s, i], the halves in one byte
        full = full.view(tiles, 16, chunks, 4, 4, 2, 4).permute(0, 2, 4, 1, 3, 6, 5)
        packed = (full[..., 0] | (full[..., 1] << 4)).reshape(tiles, chunks, 1024).contiguous()
        s = torch.zeros(tiles * 16, K // group, dtype=scales.dtype, device=scales.device)
        s[:N] = scales.detach()
        s = s.view(tiles, 16, K // group).transpose(1, 2).contiguous()
        return cls(K, N, group, packed, s, None if bias is None else bias.detach().contiguous())

    @classmethod
    def from_weight(cls, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, group: int = 64) -> "QuantLinear4":
        """Rounds ``weight`` ``[N, K]``: a group's scale is its largest magnitude / 7 (in the weight's type),
        its codes the nearest whole numbers."""
        if weight.dim() != 2 or weight.dtype not in _LN16:
            raise TypeError("weight must be 2-D, bfloat16 or float16")
        N, K = (int(n) for n in weight.shape)
        if group not in cls.GROUPS or K % group:
            raise NotImplementedError(f"group {group} must be one of {cls.GROUPS} and divide the {K} inputs")
        w = weight.detach().float().view(N, K // group, group)
        scales = (w.abs().amax(-1) / 7).to(weight.dtype)
        s = scales.float()
        codes = torch.where(s[..., None] > 0, w / s[..., None], torch.zeros_like(w)).round_().clamp_(-7, 7)
        return cls.from_codes(codes.view(N, K).to(torch.int8), scales, bias)

    @classmethod
    def from_linear(cls, lin: nn.Linear, group: int = 64) -> "QuantLinear4":
        return cls.from_weight(lin.weight, lin.bias, group)

    def dequantize(self) -> torch.Tensor:
        """The fp32 weight ``[N, K]`` that the codes and scales stand for."""
        tiles, chunks, _ = self.packed.shape
        p = self.packed.view(tiles, chunks, 4, 16, 4, 4)
        nib = torch.stack([p & 15, p >> 4], -1).permute(0, 3, 1, 4, 2, 6, 5).reshape(tiles * 16, chunks * 128)
        codes = (nib & 7).float() * (1 - 2 * (nib >> 3).float())
        s = self.scales.transpose(1, 2).reshape(tiles * 16, -1).float().repeat_interleave(self.group, 1)
        return codes[: self.out_features, : self.in_features] * s[: self.out_features]

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return linear4(x, self)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, group={self.group}, bias={self.bias is not None}"


class QuantLinear4Rows(QuantLinear4):
    """``features`` output features of another layer from ``first`` on, whole tiles of 16: views of that layer's
    buffers, taken at every use. It has none of its own, so ``to``, ``load_state_dict`` and copies leave the weights
    in one place."""

    def __init__(self, whole: QuantLinear4, first: int, features: int, bias: bool = True):
        nn.Module.__init__(self)
        if first % 16 or features % 16 or features <= 0 or not 0 <= first <= whole.out_features - features:
            raise ValueError(f"features {first} .. {first + features - 1} are not whole tiles of the layer's {whole.out_features}")
        self.in_features, self.out_features, self.group = whole.in_features, features, whole.group
        self._whole, self._first, self._bias = (whole,), first, bias  # the tuple keeps it from being a submodule

    @property
    def packed(self) -> torch.Tensor:
        return self._whole[0].packed[self._first // 16:(self._first + self.out_features) // 16]

    @property
    def scales(self) -> torch.Tensor:
        return self._whole[0].scales[self._first // 16:(self._first + self.out_features) // 16]

    @property
    def bias(self) -> Optional[torch.Tensor]:
        b = self._whole[0].bias
        return b[self._first:self._first + self.out_features] if self._bias and b is not None else None


def _linear4_operands(x: torch.Tensor, lin: QuantLinear4):
    """The checked rows ``[M, K]`` of ``x`` and the layer's packed weights, scales and bias."""
    dtype = x.dtype
    if dtype not in _LN16:
        raise TypeError(f"x: dtype {dtype} is not supported (bfloat16, float16)")
    # nn.Module's attribute lookup costs 0.15 us a name
    own = lin._buffers or {"packed": lin.packed, "scales": lin.scales, "bias": lin.bias}
    packed, scales, bias = own["packed"], own["scales"], own["bias"]
    _check_cuda("x", x, packed.device)
    if scales.dtype != dtype or scales.device != x.device or (
            bias is not None and (bias.dtype != dtype or bias.device != x.device)):
        raise TypeError("the Linear's scales and bias must have the activations' dtype and device")
    # buffers can be replaced after the construction; their counts take 0.5 us a call, their shapes 0.7
    tiles = (lin.out_features + 15) // 16
    if packed.numel() != tiles * ((lin.in_features + 127) // 128) * 1024 or packed.dtype is not torch.uint8 \
            or scales.numel() != tiles * 16 * (lin.in_features // lin.group) or not packed.is_contiguous() \
            or not scales.is_contiguous() or (bias is not None and (bias.numel() != lin.out_features or not bias.is_contiguous())):
        _check_linear4_sizes(lin, packed, scales, bias)
        raise TypeError("the Linear's packed weights must be uint8")
    if x.dim() == 0 or x.shape[-1] != lin.in_features:
        raise ValueError(f"x must have {lin.in_features} features, got {tuple(x.shape)}")
    return x if x.dim() == 2 and x.stride(1) == 1 else _rows(x, "x"), packed, scales, bias


def linear4(x: torch.Tensor, lin: QuantLinear4, gelu: bool = False) -> torch.Tensor:
    """``lin(x)`` (``gelu``: then the exact GELU) for 16-bit ``x [..., K]``: fp32 accumulation, bias and
    activation, one rounding."""
    xr, packed, scales, bias = _linear4_operands(x, lin)
    index = x.device.index
    if index != _current_device():  # launches go to the current device
        with torch.cuda.device(index):
            return linear4(x, lin, gelu)
    M, K, N = xr.shape[0], lin.in_features, lin.out_features
    y = x.new_empty((*x.shape[:-1], N))
    rc = _lib.load().wdrz_linear4(
        _LN16[x.dtype], xr.data_ptr(), xr.stride(0) if M > 1 else K, packed.data_ptr(), scales.data_ptr(),
        None if bias is None else bias.data_ptr(), y.data_ptr(), N, M, N, K, lin.group, 1 if gelu else 0, _raw_stream(index))
    if rc != _lib.WDRZ_OK:
        _raise(rc, "linear4")
    return y


def linear4_partials(x: torch.Tensor, lin: QuantLinear4, n_split: int = 4) -> torch.Tensor:
    """:func:`linear_partials` of a Linear with 4-bit weights: fp32 ``[n_split, rows, N]`` whose sum over the
    first dimension is ``x @ weight.T`` (no bias), for :func:`add_layernorm_partials_`."""
    xr, packed, scales, _ = _linear4_operands(x, lin)
    index = x.device.index
    if index != _current_device():  # launches go to the current device
        with torch.cuda.device(index):
            return linear4_partials(x, lin, n_split)
    M, K, N = xr.shape[0], lin.in_features, lin.out_features
    part = torch.empty(n_split, M, N, dtype=torch.float32, device=x.device)
    rc = _lib.load().wdrz_linear4_partials(
        _LN16[x.dtype], xr.data_ptr(), xr.stride(0) if M > 1 else K, packed.data_ptr(), scales.data_ptr(),
        part.data_ptr(), M, N, K, lin.group, n_split, _raw_stream(index))
    if rc != _lib.WDRZ_OK:
        _raise(rc, "linear4_partials")
    return part


LN_LINEAR_ROWS = 4  # rows ln_linear takes (every workgroup repeats their LayerNorm)
LN_LINEAR_MAX_K = 1536


def ln_linear(x: torch.Tensor, partials: torch.Tensor, lin: nn.Linear, ln: nn.LayerNorm, weight: torch.Tensor,
              bias: Optional[torch.Tensor], gelu: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """``linear(add_layernorm_partials_(x, partials, lin, ln), weight, bias, gelu)`` in one launch,
    for up to LN_LINEAR_ROWS rows of at most LN_LINEAR_MAX_K. ``x`` is left as it is: returns the
    new residual and the Linear's output."""
    _check_cuda("x", x, x.device)
    if x.dtype not in _LN16:
        raise TypeError(f"x: dtype {x.dtype} is not supported (bfloat16, float16)")
    xr = _rows(x, "x")
    M, K = (int(v) for v in xr.shape)
    if lin.bias is None:
        raise ValueError("the Linear must have a bias")
    w, b = weight.detach(), bias.detach() if bias is not None else None
    lw, lb, db = ln.weight.detach(), ln.bias.detach(), lin.bias.detach()
    for name, t in (("partials", partials), ("weight", w), ("bias", b), ("ln.weight", lw), ("ln.bias", lb),
                    ("lin.bias", db)):
        if t is not None:
            _check_cuda(name, t, x.device)
    if any(p is not None and p.dtype != x.dtype for p in (w, b, lw, lb, db)):
        raise TypeError("the LayerNorm and Linear parameters must have the activations' dtype")
    if w.stride(-1) != 1 or w.shape[1] != K or tuple(lw.shape) != (K,) or tuple(db.shape) != (K,):
        raise ValueError("weight must be [N, K] with contiguous rows and K = x.shape[-1] = the LayerNorm's width")
    if partials.dtype != torch.float32 or tuple(partials.shape[1:]) != (M, K) or not partials.is_contiguous():
        raise ValueError("partials must be contiguous fp32 [n_split, rows, n] matching x")
    if b is not None and not b.is_contiguous():
        b = b.contiguous()
    N = int(w.shape[0])
    x_new = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    y = torch.empty(M, N, dtype=x.dtype, device=x.device)
    rc = _lib.load().wdrz_ln_linear(
        _LN16[x.dtype], xr.data_ptr(), xr.stride(0), partials.data_ptr(), int(partials.shape[0]), db.data_ptr(),
        x_new.data_ptr(), K, lw.data_ptr(), lb.data_ptr(), float(ln.eps), w.data_ptr(), w.stride(0),
        b.data_ptr() if b is not None else None, y.data_ptr(), N, M, N, K, 1 if gelu else 0, _stream_handle(),
    )
    if rc != _lib.WDRZ_OK:
        _raise(rc, "ln_linear")
    return x_new, y.view(*x.shape[:-1], N)


def step_begin(tokens: torch.Tensor, positions: torch.Tensor, emb: torch.Tensor, pos_emb: torch.Tensor,
               ln: nn.LayerNorm, slots: Optional[torch.Tensor], lens: torch.Tensor):
    """A cached step's prologue in one launch: ``x = emb[tokens] + pos_emb[positions]``, ``ln(x)``,
    the int32 slot map (None without ``slots``) and ``lens[:, slots]`` (``lens[:, :B]`` without).

    ``tokens`` / ``positions`` int64 ``[B, sq]`` (any strides), 16-bit tables ``[n_vocab, n]`` /
    ``[n_ctx, n]``, ``slots`` int64 ``[B]``, ``lens`` int32 ``[n_layers, n_slots]`` contiguous. An id out
    of range reads nothing and gives a NaN row (a slot: length -1, NaN from the attention); WDRZ_DEBUG=1
    refuses it."""
    for name, t in (("emb", emb), ("pos_emb", pos_emb), ("tokens", tokens), ("positions", positions), ("lens", lens),
                    ("ln.weight", ln.weight), ("ln.bias", ln.bias)):
        _check_cuda(name, t, emb.device)
    if emb.dtype not in _LN16:
        raise TypeError(f"emb: dtype {emb.dtype} is not supported (bfloat16, float16)")
    B, sq = (int(v) for v in tokens.shape)
    n = int(emb.shape[1])
    e, p, lw, lb = emb.detach(), pos_emb.detach(), ln.weight.detach(), ln.bias.detach()
    if any(t.dtype != e.dtype for t in (p, lw, lb)):
        raise TypeError("the tables and the LayerNorm must share a dtype")
    if tuple(positions.shape) != (B, sq) or p.shape[1] != n or tuple(lw.shape) != (n,) or e.stride(-1) != 1 \
            or p.stride(-1) != 1 or not lens.is_contiguous():
        raise ValueError("shapes or strides of the step's inputs do not match")
    if tokens.dtype != torch.int64 or positions.dtype != torch.int64 or lens.dtype != torch.int32:
        raise TypeError("tokens and positions must be int64, lens int32")
    slots32 = None
    if slots is not None:
        _check_cuda("slots", slots, e.device)
        if slots.dtype != torch.int64 or tuple(slots.shape) != (B,):
            raise ValueError(f"slots must be int64 [{B}]")
        slots = slots.contiguous()
        slots32 = torch.empty(B, dtype=torch.int32, device=e.device)
    elif B > lens.shape[1]:
        raise ValueError(f"{B} rows exceed the {lens.shape[1]} slots")
    if _lib.debug_mode():  # host copies of the ids: debugging runs only, not graph capture
        from .debug import check_step_metadata

        check_step_metadata(tokens.cpu().numpy(), positions.cpu().numpy(),
                            slots.cpu().numpy() if slots is not None else None, e.shape[0], p.shape[0], lens.shape[1])
    x = torch.empty(B, sq, n, dtype=e.dtype, device=e.device)
    h = torch.empty_like(x)
    seqlens = torch.empty(lens.shape[0], B, dtype=torch.int32, device=e.device)
    i64x2 = _lib.ctypes.c_int64 * 2
    rc = _lib.load().wdrz_step_begin(
        _LN16[e.dtype], tokens.data_ptr(), i64x2(*tokens.stride()), positions.data_ptr(), i64x2(*positions.stride()),
        e.data_ptr(), e.stride(0), e.shape[0], p.data_ptr(), p.stride(0), p.shape[0], lw.data_ptr(), lb.data_ptr(),
        float(ln.eps), x.data_ptr(), h.data_ptr(), slots.data_ptr() if slots is not None else None,
        slots32.data_ptr() if slots is not None else None, lens.data_ptr(), seqlens.data_ptr(), B, sq, n,
        lens.shape[0], lens.shape[1], _stream_handle(),
    )
    if rc != _lib.WDRZ_OK:
        _raise(rc, "step_begin")
    return x, h, slots32, seqlens


def step_end_(lens: torch.Tensor, seqlens: torch.Tensor, slots: Optional[torch.Tensor], sq: int) -> None:
    """``lens[:, slots] += sq`` (``lens[:, :B]`` without ``slots``) from the lengths ``seqlens`` that
    ``step_begin`` gathered."""
    _check_cuda("lens", lens, lens.device)
    _check_cuda("seqlens", seqlens, lens.device)
    if lens.dtype != torch.int32 or seqlens.dtype != torch.int32:
        raise TypeError("lens and seqlens must be int32")
    if lens.dim() != 2 or seqlens.dim() != 2 or seqlens.shape[0] != lens.shape[0] or not lens.is_contiguous() \
            or not seqlens.is_contiguous():
        raise ValueError("lens and seqlens must be contiguous [n_layers, n_slots] and [n_layers, B]")
    if slots is not None:
        _check_cuda("slots", slots, lens.device)
        if slots.dtype != torch.int64 or tuple(slots.shape) != (seqlens.shape[1],):
            raise ValueError(f"slots must be int64 [{seqlens.shape[1]}]")
        slots = slots.contiguous()
    elif seqlens.shape[1] > lens.shape[1]:
        raise ValueError(f"{seqlens.shape[1]} rows exceed the {lens.shape[1]} slots")
    rc = _lib.load().wdrz_step_end(lens.data_ptr(), seqlens.data_ptr(), slots.data_ptr() if slots is not None else None,
                                   seqlens.shape[1], sq, lens.shape[0], lens.shape[1], _stream_handle())
    if rc != _lib.WDRZ_OK:
        _raise(rc, "step_end_")
