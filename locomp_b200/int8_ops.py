"""The int8 path of a decoder layer: tokens quantised to int8 with a scale each, products of int8 tokens and int8 weights, and
the norms around a block.

  quantize_tokens(x, weight=None)     x, or its RMS norm, as int8 tokens
  silu_mul_tokens(gate, up)           SiLU(gate) * up as int8 tokens
  int8_matmul(x, x_scales, w, w_scales)
  Int8Linear(w, scales)               a layer that takes float activations or int8 tokens
  residual_norms(hidden, delta, ...)  the norm after a block, its gate and residual scale, and the norm before the next block

The reference has none of these: its int8 matvec (examples/38_quantized_matmul.py:94-134) and its norms
(examples/34_fused_residual_norm.py:18-60, examples/54_smollm2_inference.py:40-73) keep float activations.  Weights are those of
`quantize(w, K, bits=8)`: int8 [N, K] with one scale per output channel.
"""
from __future__ import annotations

from contextlib import contextmanager
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _lib
from .decode_ops import _finish, _same
from .ops import _float_kind, _same_device
from .tensor import KIND_TO_CODE, KIND_TO_TORCH, Operand, _require_cuda, current_stream_ptr, resolve


@dataclass
class QuantizedTokens:
    """Rows of int8 values that stand for q * scale: `q` int8 [..., n], `scales` float32 [...].  Rows of q that this package
    makes start on 16 bytes, so that the product's kernel can read them by TMA (n % 16 != 0: q is a view of wider rows)."""
    q: torch.Tensor
    scales: torch.Tensor

    @property
    def shape(self) -> Tuple[int, ...]:
        return tuple(self.q.shape)


@contextmanager
def _on(device: int, stream):
    """Work on a device and on `stream` (None: the device's current one): what is allocated in here belongs to that stream."""
    if isinstance(stream, torch.cuda.Stream) and stream.device.index != device:          # (its context would launch on its own device)
        raise ValueError(f"the operands live on cuda:{device}, the stream on {stream.device}")
    with torch.cuda.device(device):
        if stream is None:
            yield
            return
        if not isinstance(stream, torch.cuda.Stream):
            stream = torch.cuda.ExternalStream(int(stream), device=device)
        with torch.cuda.stream(stream):
            yield


def _resolve_rows(arg, name: str, bf16: bool = False) -> Tuple[Operand, int]:
    """An operand whose rows may be further apart than they are long (torch tensors only), and how far."""
    if isinstance(arg, torch.Tensor) and arg.is_cuda and arg.dim() > 0 and arg.numel() and not arg.is_contiguous():
        ld = _lib.calls.row_stride(arg)
        if ld is not None:
            one_row = resolve(arg[(0,) * (arg.dim() - 1)].reshape(-1), name, bf16)      # (checks the type)
            return Operand(arg.data_ptr(), one_row.kind, tuple(arg.shape), arg.numel(), arg.device.index, arg), ld
    op = resolve(arg, name, bf16)
    return op, op.shape[-1] if op.shape else 0


def _rows_of(op: Operand, name: str) -> Tuple[int, int]:
    if not op.shape:
        raise ValueError(f"{name} must be [n] or [rows, n]")
    n = op.shape[-1]
    return (op.size // n if n else 0), n


def _pair(out):
    """The tensors of the tokens that a call is given to write."""
    if out is None:
        return None
    if not isinstance(out, QuantizedTokens):
        raise TypeError(f"out must be QuantizedTokens, got {type(out)}")
    return out.q, out.scales


def _empty_tokens(shape, device) -> QuantizedTokens:
    n = shape[-1]
    wide = torch.empty(tuple(shape[:-1]) + ((n + 15) // 16 * 16,), dtype=torch.int8, device=device)
    return QuantizedTokens(wide[..., :n], torch.empty(tuple(shape[:-1]), dtype=torch.float32, device=device))


def _tokens_out(out: Optional[QuantizedTokens], shape, dev: int) -> Tuple[QuantizedTokens, int, int, int]:
    """The tokens a call writes, the addresses of q and scales, and how far apart the rows of q are."""
    rows, n = 1, shape[-1]
    for size in shape[:-1]:
        rows *= size
    if rows and not n:
        raise ValueError("rows of no values have no scale")
    given = _pair(out)
    if given is None:
        out = _empty_tokens(shape, torch.device("cuda", dev))
        given = _pair(out)
    qo, ld = _resolve_rows(given[0], "out.q")
    so = resolve(given[1], "out.scales")
    if qo.kind != "i8" or qo.size != rows * n or (rows and qo.shape[-1] != n):
        raise ValueError(f"out.q must hold {rows} int8 rows of {n}")
    if so.kind != "f32" or so.size != rows:
        raise ValueError(f"out.scales must hold {rows} float32 values")
    if qo.host is not None or so.host is not None:
        raise TypeError("out must live on the device")
    if qo.device != dev or so.device != dev:
        raise ValueError("all operands must live on one device")
    return out, qo.ptr, so.ptr, ld


# ------------------------------------------------------------------------------------------ rows
def quantize_tokens(x, weight=None, eps: float = 1e-5, *, out: Optional[QuantizedTokens] = None, stream=None,
                    bf16: bool = False) -> QuantizedTokens:
    """x ([n], [rows, n] or [..., n]; rows may be further apart than n) as int8 tokens: scale = max|v| / 127 over a row, q = rint(v / scale),
    with v = x or, where `weight` is given, rms_norm(x, weight, eps).  A row of zeros has scale 1; a row that holds an infinity or a NaN
    has scale NaN (and q 0), and so do all products with it.  Without `weight`: the values and scales of quantize(x, n, bits=8), but for
    such rows and for scales that would be below 2**-126."""
    if stream is None and not bf16 and isinstance(x, torch.Tensor):
        res = _lib.calls.quantize_tokens(x, weight, eps, _pair(out))
        if res is not NotImplemented:
            return QuantizedTokens(*res) if out is None else out
    xo, ldx = _resolve_rows(x, "x", bf16)
    rows, n = _rows_of(xo, "x")
    wo = None if weight is None else resolve(weight, "weight", bf16)
    if wo is not None and wo.size != n:
        raise ValueError(f"weight must hold n = {n} values, got {wo.size}")
    _, dev = _same(xo) if wo is None else _same(xo, wo)
    code = _float_kind(xo, "x")
    _require_cuda()
    with _on(dev, stream):
        t, q_ptr, s_ptr, ldq = _tokens_out(out, xo.shape, dev)
        _lib.check(_lib.lib().lcq_quantize_tokens(xo.ptr, ldx, wo.ptr if wo else None, q_ptr, ldq, s_ptr, rows, n, float(eps), code,
                                                  current_stream_ptr()))
    return t


def silu_mul_tokens(gate, up, *, out: Optional[QuantizedTokens] = None, stream=None, bf16: bool = False) -> QuantizedTokens:
    """gate * sigmoid(gate) * up as int8 tokens (see quantize_tokens).  gate and up: [n] or [rows, n]; they may be the halves
    gu[:, :n] and gu[:, n:] of what a fused projection gave."""
    if stream is None and not bf16 and isinstance(gate, torch.Tensor):
        res = _lib.calls.silu_mul_tokens(gate, up, _pair(out))
        if res is not NotImplemented:
            return QuantizedTokens(*res) if out is None else out
    (go, ldg), (uo, ldu) = _resolve_rows(gate, "gate", bf16), _resolve_rows(up, "up", bf16)
    if go.shape != uo.shape:
        raise ValueError(f"gate and up must have one shape, got {go.shape} and {uo.shape}")
    rows, n = _rows_of(go, "gate")
    _, dev = _same(go, uo)
    code = _float_kind(go, "gate")
    _require_cuda()
    with _on(dev, stream):
        t, q_ptr, s_ptr, ldq = _tokens_out(out, go.shape, dev)
        _lib.check(_lib.lib().lcq_silu_mul_tokens(go.ptr, ldg, uo.ptr, ldu, q_ptr, ldq, s_ptr, rows, n, code, current_stream_ptr()))
    return t


def residual_norms(hidden, delta, weight=None, eps: float = 1e-5, *, post_weight=None, gate=None, scale: float = 1.0, hidden_out=None,
                   out=None, quantized: bool = False, stream=None, bf16: bool = False):
    """What stands between two blocks, in one pass over the rows:

        y = delta                       or rms_norm(delta, post_weight, eps)       the norm after the block
        y = y * gate                    where a gate is given
        hidden += scale * y             in place, or into `hidden_out`
        out = rms_norm(hidden, weight, eps)                                        the norm before the next block

    residual_rms_norm is the case without post_weight, gate and scale.  hidden, delta: [n] or [rows, n].  gate: [n], one value a channel,
    or [g, n] with rows % g == 0, each row for rows / g consecutive rows of hidden (a sequence's tokens; g = rows: its own for each).
    Arithmetic is float32; hidden is rounded to its type as it is stored, and the second norm reads it so.  All operands share hidden's type; delta
    may be float32 beside it, as a product leaves it with out_dtype="f32", and is then rounded only as it is added.
    quantized=True: out is QuantizedTokens (see quantize_tokens).  weight=None: no norm follows, and the result is the new hidden."""
    if stream is None and not bf16 and isinstance(hidden, torch.Tensor):
        o = (out.q, out.scales) if isinstance(out, QuantizedTokens) else out
        res = _lib.calls.residual_norms(hidden, delta, weight, eps, post_weight, gate, scale, hidden_out, o, quantized)
        if res is not NotImplemented:
            if out is not None:
                return out
            return QuantizedTokens(*res) if quantized else res
    ho, do = resolve(hidden, "hidden", bf16), resolve(delta, "delta", bf16)
    rows, n = _rows_of(ho, "hidden")
    if do.size != ho.size or not do.shape or do.shape[-1] != n:
        raise ValueError("delta must match hidden")
    parts = {name: resolve(v, name, bf16) for name, v in (("weight", weight), ("post_weight", post_weight), ("gate", gate)) if v is not None}
    for name in ("weight", "post_weight"):
        if name in parts and parts[name].size != n:
            raise ValueError(f"{name} must hold n = {n} values, got {parts[name].size}")
    gate_rows = 0
    if gate is not None:
        gate_rows = parts["gate"].size // n if n else 0
        if not parts["gate"].shape or parts["gate"].shape[-1] != n or (rows and (gate_rows == 0 or rows % gate_rows)):
            raise ValueError(f"gate must be [n] or [g, n] with {rows} rows a multiple of g, got shape {parts['gate'].shape}")
    if weight is None and (quantized or out is not None):
        raise ValueError("without weight there is no norm to write to out or to quantise")
    if hidden_out is None:
        if ho.host is not None:
            raise TypeError("hidden is updated in place and must be a device tensor")
        hno, new_hidden = ho, hidden
    else:
        hno, new_hidden = resolve(hidden_out, "hidden_out", bf16), hidden_out
        if hno.host is not None:
            raise TypeError("hidden_out must be a device tensor")
        if hno.size != ho.size:
            raise ValueError(f"hidden_out must hold {ho.size} values, got {hno.size}")
    kind, dev = _same(ho, hno, *parts.values())
    if do.kind not in (kind, "f32"):
        raise TypeError(f"delta must be {kind} as hidden is, or f32, got {do.kind}")
    _same_device(ho, do)
    code = _float_kind(ho, "hidden")
    _require_cuda()
    with _on(dev, stream):
        oo, res, out_ptr, ldo, scales = None, new_hidden, None, n, None
        if quantized:
            res, out_ptr, scales, ldo = _tokens_out(out, ho.shape, dev)
        elif weight is not None:
            res = torch.empty(ho.shape, dtype=KIND_TO_TORCH[kind], device=torch.device("cuda", dev)) if out is None else out
            oo = resolve(res, "out", bf16)
            if oo.size != ho.size:
                raise ValueError(f"out must hold {ho.size} values, got {oo.size}")
            _same(ho, oo)
            out_ptr = oo.ptr
        ptr = {name: op.ptr for name, op in parts.items()}
        _lib.check(_lib.lib().lcq_residual_norms_delta(ho.ptr, do.ptr, KIND_TO_CODE[do.kind], ptr.get("post_weight"), ptr.get("gate"), gate_rows,
                                                       float(scale), ptr.get("weight"), hno.ptr, out_ptr, ldo, scales, rows, n, float(eps), code,
                                                       current_stream_ptr()))
        return res if oo is None else _finish(oo, res)


# ------------------------------------------------------------------------------------------ the product
def int8_matmul(x, x_scales, w, w_scales, *, out=None, out_dtype: Optional[str] = None, stream=None,
                workspace_buf: Optional[torch.Tensor] = None):
    """out[m, n] = (sum_k x[m, k] * w[n, k]) * x_scales[m] * w_scales[n]: an exact integer sum, scaled in float32 and rounded once.

    x: int8 [K] or [M, K]; x_scales: float32, M values; w: int8 [N, K]; w_scales: N values (f32 / f16 / bf16).  x may have more dimensions, as
    quantize_tokens gives them for a batch of sequences: [..., K] with x_scales of the shape [...].  Rows of x and w may be
    further apart than K; those that do not start on 16 bytes (K % 16 != 0 in contiguous storage) cost a copy.
    Returns a torch CUDA tensor [N], [M, N] or [..., N] of out_dtype ("f32", "f16", "bf16"; default "f16") or `out`.  K is at most 131071.
    Scratch is needed for such copies only: workspace_buf, or memory that the call takes from torch's allocator on its stream; under CUDA-graph capture
    that is the graph's own, so that no two graphs share it."""
    if isinstance(x, torch.Tensor) and stream is None:
        res = _lib.calls.int8_matmul(x, x_scales, w, w_scales, out, -1 if out_dtype is None else KIND_TO_CODE.get(out_dtype, -2), workspace_buf)
        if res is not NotImplemented:
            return res
    (xo, ldx), (wo, ldw) = _resolve_rows(x, "x"), _resolve_rows(w, "w")
    xso, wso = resolve(x_scales, "x_scales"), resolve(w_scales, "w_scales")
    for op, name in ((xo, "x"), (wo, "w")):
        if op.kind != "i8":
            raise TypeError(f"{name} must be int8, got {op.kind}")
    if not xo.shape or (len(xo.shape) > 2 and xso.shape != xo.shape[:-1]):
        raise ValueError(f"x must be [K] or [M, K], or [..., K] with x_scales of [...], got shapes {xo.shape} and {xso.shape}")
    if len(wo.shape) != 2:
        raise ValueError(f"w must be [N, K], got shape {wo.shape}")
    M, K, N = 1, xo.shape[-1], wo.shape[0]
    for size in xo.shape[:-1]:
        M *= size
    if wo.shape[1] != K:
        raise ValueError(f"x has K={K} but the weights hold K={wo.shape[1]}")
    if xso.kind != "f32" or xso.size != M:
        raise ValueError(f"x_scales must hold M = {M} float32 values, got {xso.size} of {xso.kind}")
    if wso.size != N:
        raise ValueError(f"w_scales must hold N = {N} values, got {wso.size}")
    sk = _float_kind(wso, "w_scales")
    if out_dtype is not None and out_dtype not in KIND_TO_CODE:
        raise ValueError(f"out_dtype must be one of f32/f16/bf16, got {out_dtype}")
    dev = _same_device(xo, xso, wo, wso)
    _require_cuda()
    L = _lib.lib()
    with _on(dev, stream):
        res = torch.empty(xo.shape[:-1] + (N,), dtype=KIND_TO_TORCH[out_dtype or "f16"], device=torch.device("cuda", dev)) if out is None else out
        oo = resolve(res, "out")
        if oo.size != M * N:
            raise ValueError(f"out must hold M*N = {M * N} values, got {oo.size}")
        if out_dtype is not None and oo.kind != out_dtype:
            raise TypeError(f"out is {oo.kind} but out_dtype={out_dtype}")
        ok = _float_kind(oo, "out")
        if oo.device != dev:
            raise ValueError("all operands must live on one device")
        sp = current_stream_ptr()
        need = L.lcq_int8_matmul_workspace_bytes(M, N, K, _on_16(xo, M, ldx), _on_16(wo, N, ldw))
        if need == (1 << 64) - 1:
            _lib.check(L.lcq_int8_matmul(xo.ptr, ldx, xso.ptr, wo.ptr, ldw, wso.ptr, oo.ptr, M, N, K, sk, ok, None, 0, sp))    # raises

        def launch(ws):
            _lib.check(L.lcq_int8_matmul(xo.ptr, ldx, xso.ptr, wo.ptr, ldw, wso.ptr, oo.ptr, M, N, K, sk, ok,
                                         ws.data_ptr() if ws is not None else None, ws.numel() * ws.element_size() if ws is not None else 0, sp))
        if need == 0:
            launch(None)
        elif workspace_buf is not None:
            if workspace_buf.numel() * workspace_buf.element_size() < need or workspace_buf.device.index != dev or not workspace_buf.is_contiguous():
                raise ValueError(f"workspace_buf must hold {need} bytes on cuda:{dev}")
            launch(workspace_buf)
        else:
            launch(torch.empty(need, dtype=torch.uint8, device=torch.device("cuda", dev)))
        if oo.host is not None:
            return _finish(oo, res)
    return res


def _on_16(op: Operand, rows: int, ld: int) -> bool:
    return rows == 0 or (op.ptr % 16 == 0 and (rows == 1 or ld % 16 == 0))


def int8_matmul_workspace_bytes(M: int, N: int, K: int, x_on_16: bool = True, w_on_16: bool = True) -> int:
    """Scratch bytes int8_matmul needs for this problem (0 if none).  x_on_16, w_on_16: whether rows of x and of w start on 16 bytes, as those
    of QuantizedTokens and Int8Linear do; any other are copied into the scratch first (x whole, w at most 48 MiB at a time)."""
    n = _lib.lib().lcq_int8_matmul_workspace_bytes(M, N, K, x_on_16, w_on_16)
    if n == (1 << 64) - 1:
        raise ValueError("no kernel covers this problem")
    return int(n)


class Int8Linear:
    """y = x @ (w * scales)^T in int8: w int8 [N, K] and one scale for each of its rows, as quantize(weights, K, bits=8) makes them.

    linear(x): x is QuantizedTokens, or float activations, which are quantised first; linear(x, weight): their RMS norm with that
    weight is.  x: [K], [M, K] or [..., K].  The result has the type of the activations (tokens: float16), or out_dtype, or is written to `out`."""

    def __init__(self, w: torch.Tensor, scales: torch.Tensor):
        if not (w.is_cuda and scales.is_cuda):
            raise ValueError("Int8Linear keeps its weights on a CUDA device")
        if w.dtype != torch.int8 or w.dim() != 2:
            raise TypeError(f"w must be int8 [N, K], got {w.dtype} with {w.dim()} dimensions")
        if scales.numel() != w.shape[0]:
            raise ValueError(f"scales must hold N = {w.shape[0]} values, got {scales.numel()}")
        self.out_features, self.in_features = w.shape
        if w.stride(1) != 1 or w.stride(0) < self.in_features or w.stride(0) % 16 or w.data_ptr() % 16:      # rows on 16 bytes, for TMA
            wide = torch.zeros(self.out_features, (self.in_features + 15) // 16 * 16, dtype=torch.int8, device=w.device)
            wide[:, :self.in_features] = w
            w = wide[:, :self.in_features]
        self.w, self.scales = w, scales.contiguous()

    @property
    def weight_bytes(self) -> int:
        return self.w.numel() + self.scales.numel() * self.scales.element_size()

    def __call__(self, x, weight=None, eps: float = 1e-5, *, out=None, out_dtype: Optional[str] = None, stream=None,
                 workspace_buf: Optional[torch.Tensor] = None):
        if not isinstance(x, QuantizedTokens):
            if out is None and out_dtype is None:
                out_dtype = resolve(x, "x").kind if not isinstance(x, torch.Tensor) else \
                    {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16"}.get(x.dtype)
            x = quantize_tokens(x, weight, eps, stream=stream)
        elif weight is not None:
            raise ValueError("tokens that are quantised already cannot be normalised")
        return int8_matmul(x.q, x.scales, self.w, self.scales, out=out, out_dtype=out_dtype, stream=stream, workspace_buf=workspace_buf)
