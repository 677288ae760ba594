"""Sequence operators on the HIP library: one layer of a selective state-space sequence model and the reading of its answers.

    y, state = causal_conv(x, weight, bias, state=..., lengths=...)            tae_causal_conv
    y, state = selective_scan(x, dt, A, B, C, D=..., z=..., ...)               tae_selective_scan
    residual, normed = norm_residual(residual, block, gate=..., ...)           tae_norm_residual
    q, scale = quantize_int8(weight); y = int8_linear(x, q, scale, bias)       tae_quantize_int8, tae_int8_linear
    logp, entropy, ids, top_logp = token_logprobs(logits, tokens, top=8)       tae_token_logprobs

They stand beside ``Channel_AE_HIP`` as the recurrent and convolution stacks, the power norm, the precisions and ``count_errors`` do
inside it, and follow its manner: all arithmetic runs in libturboae_hip.so on tensors of a ROCm device (no CPU fallback), a call enqueues
work on the current stream of its tensors' device and never synchronises, and wrong shapes, types, devices or layouts raise ``ValueError``
before anything is launched.  The path is inference: a tensor that requires a gradient is refused (call under ``torch.no_grad()``),
and so is one with a forward-mode tangent.  No reference counterpart.

Activations are float32, float16 or bfloat16, (batch, len, channels) with adjacent channels - a slice of a wider tensor is taken as it is,
without a copy; parameters and states named float32 are float32.  Sums, norms, softmax statistics and states are kept in 32 bits or more
and each result is rounded once.  ``lengths`` (int32, one for each sequence) marks padding: positions at or behind it are not read, their
outputs are zero, and the state is the one after the last position in front of them.  Sizes, rows of all leading dimensions together among
them, are below 2^31.  ``int8_linear`` and ``token_logprobs`` take any number of leading dimensions: rows that one distance leads through are
taken as they lie; other inputs of three and more dimensions are copied first, as ``reshape`` does it, and a matrix whose last elements are
apart is refused.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import _lib

_DTYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}                   # TAE_DTYPE_*
_ACT = {"linear": 1, "tanh": 2, "sigmoid": 5, "silu": 6}                           # TAE_ACT_*

__all__ = ["causal_conv", "selective_scan", "norm_residual", "quantize_int8", "int8_linear", "token_logprobs"]


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


class _Call:
    """The checks that every tensor of a call goes through, against the first of them; a call of a single token costs little more."""

    __slots__ = ("name", "device", "dtype", "grad", "new")

    def __init__(self, name: str, first: torch.Tensor):
        if not isinstance(first, torch.Tensor) or not first.is_cuda:
            raise _lib.TurboAEError(f"{name}: needs tensors on a ROCm GPU device (no CPU fallback)")
        if first.dtype not in _DTYPE:
            raise ValueError(f"{name}: float32, float16 or bfloat16 wanted, got {first.dtype}")
        self.name, self.device, self.dtype, self.grad, self.new = name, first.device, first.dtype, torch.is_grad_enabled(), first.new_empty
        if getattr(forward_ad, "_current_level", 0) >= 0:                          # inside a dual_level, the only place for tangents
            self.__class__ = _CallAmongTangents

    def too_large(self, *sizes: int) -> None:
        raise ValueError(f"{self.name}: sizes must be below 2^31, got {sizes}")

    def tensor(self, t: Optional[torch.Tensor], what: str, shape: Tuple[int, ...], dtype: torch.dtype, dense: bool = False) -> Optional[int]:
        """Address of a tensor after its checks (None for None): shape, type, device, adjacent last elements; dense: contiguous."""
        if t is None:
            return None
        if t.shape != shape or t.dtype is not dtype or t.device != self.device:
            raise ValueError(f"{self.name}: {what} must be {dtype} of shape {tuple(shape)} on {self.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
        if not t.is_contiguous():
            if dense:
                raise ValueError(f"{self.name}: {what} must be contiguous")
            if shape[-1] > 1 and t.stride(-1) != 1:
                raise ValueError(f"{self.name}: adjacent elements of {what}'s last dimension must be adjacent in memory")
        if self.grad and t.requires_grad:
            raise ValueError(f"{self.name}: {what} requires a gradient, but this path is inference only (call it under torch.no_grad())")
        return t.data_ptr()

    def out(self, t: Optional[torch.Tensor], what: str, shape: Tuple[int, ...], dtype: torch.dtype) -> torch.Tensor:
        """A given output after its checks, or a new one."""
        if t is None:
            return self.new(shape, dtype=dtype)
        self.tensor(t, what, shape, dtype, dense=True)
        return t

    def workspace(self, args: ctypes.Structure, size) -> Optional[torch.Tensor]:
        # Freed after the call: the caching allocator hands it out again to later work of the same stream only
        n = size(ctypes.byref(args))
        if n == 0:
            return None
        w = self.new(n, dtype=torch.uint8)
        args.workspace, args.workspace_bytes = w.data_ptr(), n
        return w

    def run(self, entry, *args) -> None:
        index = self.device.index
        if torch.cuda.current_device() == index:
            rc = entry(*args, _raw_stream(index))
        else:
            with torch.cuda.device(index):
                rc = entry(*args, _raw_stream(index))
        if rc:
            _lib.check(rc)


class _CallAmongTangents(_Call):
    """The same where tensors may have forward-mode tangents, which torch.no_grad() does not turn off."""

    __slots__ = ()

    def tensor(self, t, what, shape, dtype, dense=False):
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError(f"{self.name}: {what} has a forward-mode tangent, but this path is inference only (call it with unpack_dual's primal)")
        return super().tensor(t, what, shape, dtype, dense)


_MOST = 0x7FFFFFFF                               # the library's sizes have 32 bits, and ctypes would cut larger ones to them


def _sequence(c: _Call, what: str, t: torch.Tensor) -> Tuple[int, int, int]:
    if t.dim() != 3 or t.numel() == 0:
        raise ValueError(f"{c.name}: {what} must have shape (batch, len, channels), none of them 0, got {tuple(t.shape)}")
    shape = t.shape
    if max(shape) > _MOST:
        c.too_large(*shape)
    return shape


def _strides(t: Optional[torch.Tensor]) -> Tuple[int, int]:
    """Distances between sequences and between positions; a tensor of another shape is refused by its own check."""
    return t.stride()[:2] if t is not None and t.dim() == 3 else (0, 0)


def _in_place_or_apart(name: str, out: torch.Tensor, same: Optional[torch.Tensor], *others: Optional[torch.Tensor]) -> None:
    """An output may be `same` itself, element for element; one that overlaps an input in any other way is refused."""
    b, n = out.data_ptr(), _extent(out)
    for t in (same, *others):
        if t is None or not t.is_cuda or t is same and t.data_ptr() == b and t.dtype is out.dtype and t.shape == out.shape and t.stride() == out.stride():
            continue
        a = t.data_ptr()
        if a < b + n and b < a + _extent(t):
            raise ValueError(f"{name}: an output overlaps an input without being the one that it may replace")


def _extent(t: torch.Tensor) -> int:
    """Bytes from a tensor's first element to behind its last."""
    return (sum((s - 1) * d for s, d in zip(t.shape, t.stride())) + 1) * t.element_size() if t.numel() else 0


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, state: Optional[torch.Tensor] = None,
                lengths: Optional[torch.Tensor] = None, act: str = "silu", state_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Short causal convolution of each channel: ``y[t] = act(bias + sum_k weight[:, k] * x[t - taps + 1 + k])``.

    x (batch, len, channels); weight (channels, taps) and bias (channels) float32, 1 to 8 taps; act "silu" or "linear".  ``state``
    (batch, taps - 1, channels) of x's type: the last inputs of an earlier call, oldest first (None: zeros).  Returns (y, the state after
    this call); with one position this is the single-token step.  ``state_out`` receives the state and may be ``state`` itself."""
    c = _Call("causal_conv", x)
    B, L, E = _sequence(c, "x", x)
    if weight.dim() != 2:
        raise ValueError(f"causal_conv: weight must have shape (channels, taps), got {tuple(weight.shape)}")
    K = weight.shape[1]
    if not 1 <= K <= 8 or act not in ("linear", "silu"):
        raise ValueError(f"causal_conv: 1 to 8 taps and act 'linear' or 'silu' wanted, got {K} and {act!r}")
    f32 = torch.float32
    y = c.new((B, L, E), dtype=c.dtype)
    if state_out is not None and K > 1:
        _in_place_or_apart(c.name, state_out, state, x, weight, bias, lengths)
    given, state_out = state_out, c.out(state_out, "state_out", (B, K - 1, E), c.dtype)
    args = _lib.TaeConvArgs(ctypes.sizeof(_lib.TaeConvArgs), _DTYPE[c.dtype], B, L, E, K, _ACT[act], 0, x.stride(0), x.stride(1),
                            c.tensor(x, "x", (B, L, E), c.dtype), c.tensor(weight, "weight", (E, K), f32, True), c.tensor(bias, "bias", (E,), f32, True),
                            c.tensor(state, "state", (B, K - 1, E), c.dtype, True) if K > 1 else None,
                            c.tensor(lengths, "lengths", (B,), torch.int32, True), y.data_ptr(), state_out.data_ptr() if K > 1 else None)
    c.run(_lib.load().tae_causal_conv, ctypes.byref(args))
    if given is not None:                        # autograd sees it as after any operation in place
        increment_version(given)
    return y, state_out


def selective_scan(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, D: Optional[torch.Tensor] = None,
                   z: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None, softplus: bool = True, state: Optional[torch.Tensor] = None,
                   lengths: Optional[torch.Tensor] = None, state_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Selective state-space scan.  Per channel e and state n, with ``d = softplus(dt + dt_bias)`` (``dt + dt_bias`` with softplus=False):

        h[t] = exp(d[t] A[e, n]) h[t-1] + d[t] B[t, n] x[t, e]
        y[t, e] = (sum_n C[t, n] h[t] + D[e] x[t, e]) * z[t, e] * sigmoid(z[t, e])

    x, dt, z (batch, len, channels) and B, C (batch, len, states) of one type, up to 64 states; A (channels, states), D, dt_bias
    (channels) and ``state`` (batch, channels, states; None: zeros) float32.  Returns (y, the state after the last position); with one
    position this is the single-token step.  ``state_out`` receives the state and may be ``state`` itself."""
    c = _Call("selective_scan", x)
    b, L, E = _sequence(c, "x", x)
    if A.dim() != 2 or not 1 <= A.shape[1] <= 64:
        raise ValueError(f"selective_scan: A must have shape (channels, states) with 1 to 64 states, got {tuple(A.shape)}")
    N = A.shape[1]
    f32 = torch.float32
    y = c.new((b, L, E), dtype=c.dtype)
    if state_out is not None:
        _in_place_or_apart(c.name, state_out, state, x, dt, A, B, C, D, z, dt_bias, lengths)
    given, state_out = state_out, c.out(state_out, "state_out", (b, E, N), f32)
    args = _lib.TaeScanArgs(ctypes.sizeof(_lib.TaeScanArgs), _DTYPE[c.dtype], b, L, E, N, 1 if softplus else 0, 0,
                            *_strides(x), *_strides(dt), *_strides(B), *_strides(C), *_strides(z),
                            c.tensor(x, "x", (b, L, E), c.dtype), c.tensor(dt, "dt", (b, L, E), c.dtype), c.tensor(A, "A", (E, N), f32, True),
                            c.tensor(B, "B", (b, L, N), c.dtype), c.tensor(C, "C", (b, L, N), c.dtype), c.tensor(D, "D", (E,), f32, True),
                            c.tensor(z, "z", (b, L, E), c.dtype), c.tensor(dt_bias, "dt_bias", (E,), f32, True),
                            c.tensor(state, "state", (b, E, N), f32, True), c.tensor(lengths, "lengths", (b,), torch.int32, True),
                            y.data_ptr(), state_out.data_ptr(), None, 0)
    lib = _lib.load()
    w = c.workspace(args, lib.tae_selective_scan_workspace)  # noqa: F841
    c.run(lib.tae_selective_scan, ctypes.byref(args))
    if given is not None:                        # autograd sees it as after any operation in place
        increment_version(given)
    return y, state_out


def norm_residual(residual: torch.Tensor, block: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None,
                  post_weight: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None, pre_weight: Optional[torch.Tensor] = None,
                  pre_bias: Optional[torch.Tensor] = None, center: bool = False, gate_act: str = "sigmoid", alpha: float = 1.0, eps: float = 1e-5,
                  residual_out: Optional[torch.Tensor] = None, dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """The norms around a block with its gate and residual scale, each row read once:

        p = norm(block) * post_weight + post_bias        (without post_weight: block)
        r = residual + alpha * scale * gate_act(gate) * p
        normed = norm(r) * pre_weight + pre_bias         (of r before its rounding; without pre_weight: None)

    ``norm(v) = (v - mean) / sqrt(mean((v - mean)^2) + eps)``, mean 0 unless center.  residual, block (batch, len, dim); gate of that
    shape or (batch, 1, dim), one for each sequence; gate_act "linear", "tanh", "sigmoid" or "silu"; the residual has the block's type or
    float32; scale, weights and biases (dim) float32.  Without a block r is the residual, and ``dtype`` names normed's type (None: the
    residual's); with one it has the block's.  Returns (r, normed); ``residual_out`` receives r and may be ``residual`` itself."""
    c = _Call("norm_residual", residual if block is None else block)
    B, L, D = _sequence(c, "residual", residual)
    f32 = torch.float32
    if block is None and dtype is not None:
        if dtype not in _DTYPE:
            raise ValueError(f"norm_residual: dtype must be float32, float16 or bfloat16, got {dtype}")
        c.dtype = dtype
    elif dtype is not None and dtype is not c.dtype:
        raise ValueError(f"norm_residual: with a block normed has its type, {c.dtype}, got dtype {dtype}")
    if residual.dtype not in (c.dtype, f32):
        raise ValueError(f"norm_residual: the residual has the block's type or float32, got {residual.dtype} beside {c.dtype}")
    if gate_act not in _ACT:
        raise ValueError(f"norm_residual: gate_act must be one of {sorted(_ACT)}, got {gate_act!r}")
    if block is None and pre_weight is None:
        raise ValueError("norm_residual: nothing to do without a block and without pre_weight")
    ga = 0, 0
    if gate is not None:
        per_token = tuple(gate.shape) == (B, L, D)
        c.tensor(gate, "gate", (B, L, D) if per_token else (B, 1, D), c.dtype)
        ga = gate.stride(0), gate.stride(1) if per_token else 0
    out = residual_out
    if out is None:
        out = residual if block is None else c.new((B, L, D), dtype=residual.dtype)
    else:
        c.tensor(out, "residual_out", (B, L, D), residual.dtype)
        (inner, n), (outer, m) = sorted(((out.stride(1), L), (out.stride(0), B))) if B > 1 and L > 1 else ((out.stride(1), L), (out.stride(0), B))
        if (n > 1 and inner < D) or (m > 1 and outer < (n - 1) * inner + D):
            raise ValueError("norm_residual: rows of residual_out overlap")
        _in_place_or_apart(c.name, out, residual, block, gate, scale, post_weight, post_bias, pre_weight, pre_bias)
    write = block is not None or (residual_out is not None and residual_out is not residual)
    normed = c.new((B, L, D), dtype=c.dtype) if pre_weight is not None else None
    vectors = [c.tensor(v, what, (D,), f32, True) for v, what in ((scale, "scale"), (post_weight, "post_weight"), (post_bias, "post_bias"),
                                                                  (pre_weight, "pre_weight"), (pre_bias, "pre_bias"))]
    args = _lib.TaeNormArgs(ctypes.sizeof(_lib.TaeNormArgs), _DTYPE[c.dtype], _DTYPE[residual.dtype], B, L, D, 1 if center else 0, _ACT[gate_act], eps, alpha,
                            *_strides(residual), *_strides(block), *ga, *_strides(out), c.tensor(residual, "residual", (B, L, D), residual.dtype),
                            c.tensor(block, "block", (B, L, D), c.dtype), None if gate is None else gate.data_ptr(), *vectors,
                            out.data_ptr() if write else None, None if normed is None else normed.data_ptr())
    c.run(_lib.load().tae_norm_residual, ctypes.byref(args))
    if write and residual_out is not None:
        increment_version(residual_out)
    return out, normed


def quantize_int8(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows in 8-bit whole numbers with a scale each: ``scale = max|x| / 127``, ``q = round(127 x / max|x|)``, halves to even (a row of
    zeros: 0).  x (rows, columns).  Returns (q int8, scale float32); q's rows start on 64-byte boundaries, zero-filled behind the columns,
    as ``int8_linear`` wants its weights.  A row with an infinity or NaN gets the scale NaN."""
    c = _Call("quantize_int8", x)
    if x.dim() != 2 or 0 in x.shape:
        raise ValueError(f"quantize_int8: x must have shape (rows, columns), none of them 0, got {tuple(x.shape)}")
    R, K = x.shape
    if max(R, K) > _MOST:
        c.too_large(R, K)
    address = c.tensor(x, "x", (R, K), c.dtype)
    step = -(-K // 64) * 64
    q = c.new((R, step), dtype=torch.int8)
    scale = c.new(R, dtype=torch.float32)
    c.run(_lib.load().tae_quantize_int8, _DTYPE[c.dtype], address, x.stride(0), R, K, q.data_ptr(), step, scale.data_ptr())
    return q[:, :K], scale


def int8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``y = (q(x) @ weight.T) * scale(x) * weight_scale + bias`` with the rows of x quantised as ``quantize_int8`` does it, inside the call;
    products are summed exactly, in 32-bit whole numbers.  x (..., inputs); weight (outputs, inputs) int8 without -128, rows on 16-byte
    boundaries (``quantize_int8`` lays them so); weight_scale and bias (outputs) float32; at most 131072 inputs."""
    c = _Call("int8_linear", x)
    if x.dim() < 1 or 0 in x.shape or weight.dim() != 2 or 0 in weight.shape:
        raise ValueError(f"int8_linear: x (..., inputs) and weight (outputs, inputs) wanted, none of them 0, got {tuple(x.shape)} and {tuple(weight.shape)}")
    N, K = weight.shape
    M = x.numel() // x.shape[-1]
    if M > _MOST or N > _MOST:
        c.too_large(M, N)
    rows = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    if K > 131072:
        raise ValueError(f"int8_linear: at most 131072 inputs, got {K}")
    c.tensor(rows, "x", (M, K), c.dtype)
    address = c.tensor(weight, "weight", (N, K), torch.int8)
    step = weight.stride(0) if N > 1 else -(-K // 16) * 16
    if address % 16 or step % 16 or step < K:
        raise ValueError("int8_linear: weight rows must start on 16-byte boundaries (quantize_int8 lays them so)")
    if weight.storage_offset() + (N - 1) * step + -(-K // 16) * 16 > weight.untyped_storage().nbytes():
        raise ValueError("int8_linear: the last weight row must reach to its next 16-byte boundary (quantize_int8 lays them so)")
    f32 = torch.float32
    y = c.new((*x.shape[:-1], N), dtype=c.dtype)
    args = _lib.TaeInt8Args(ctypes.sizeof(_lib.TaeInt8Args), _DTYPE[c.dtype], M, K, N, 0, rows.stride(0), step, rows.data_ptr(), address,
                            c.tensor(weight_scale, "weight_scale", (N,), f32, True), c.tensor(bias, "bias", (N,), f32, True), y.data_ptr(), None, 0)
    lib = _lib.load()
    w = c.workspace(args, lib.tae_int8_linear_workspace)  # noqa: F841
    c.run(lib.tae_int8_linear, ctypes.byref(args))
    return y


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor], Optional[torch.Tensor]]:
    """Log probability of each row's given token, the row's entropy (nats), and its ``top`` (0 to 32) most probable tokens.

    logits (..., vocab), at most 2^21; tokens (...) int32 or int64.  Returns (logp, entropy, ids, top_logp): float32 (...), float32 (...),
    int64 and float32 (..., top), the last two None with top=0; equal logits come in ascending order of their ids.  A logit of -inf is a
    token that cannot occur; in a row of nothing else every log probability is -inf and the entropy 0.  A row with +inf or NaN has none:
    NaN, ids -1.  A negative token marks a row without one (log probability 0, as for padding), one at or above vocab gives NaN."""
    c = _Call("token_logprobs", logits)
    if logits.dim() < 1 or 0 in logits.shape or tuple(tokens.shape) != tuple(logits.shape[:-1]) or tokens.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"token_logprobs: logits (..., vocab), none of them 0, and int32 or int64 tokens (...) wanted, got {tuple(logits.shape)} and {tokens.dtype} {tuple(tokens.shape)}")
    V = logits.shape[-1]
    if not 0 <= top <= min(32, V) or V > 1 << 21:
        raise ValueError(f"token_logprobs: top must be in 0..32 and at most vocab, vocab at most 2^21, got {top} of {V}")
    R = logits.numel() // V
    if R > _MOST:
        c.too_large(R)
    flat = logits if logits.dim() == 2 else logits.reshape(-1, V)
    shape = tuple(tokens.shape)
    logp = c.new(shape, dtype=torch.float32)
    entropy = c.new(shape, dtype=torch.float32)
    ids = c.new((*shape, top), dtype=torch.int64) if top else None
    top_logp = c.new((*shape, top), dtype=torch.float32) if top else None
    args = _lib.TaeLogprobsArgs(ctypes.sizeof(_lib.TaeLogprobsArgs), _DTYPE[c.dtype], 8 if tokens.dtype == torch.int64 else 4, R, V, top, flat.stride(0),
                                c.tensor(flat, "logits", (R, V), c.dtype), c.tensor(tokens, "tokens", shape, tokens.dtype, True), logp.data_ptr(), entropy.data_ptr(),
                                ids.data_ptr() if top else None, top_logp.data_ptr() if top else None, None, 0)
    lib = _lib.load()
    w = c.workspace(args, lib.tae_token_logprobs_workspace)  # noqa: F841
    c.run(lib.tae_token_logprobs, ctypes.byref(args))
    return logp, entropy, ids, top_logp
