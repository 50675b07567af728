"""Norm and rotation of queries and keys, the step between a decoder layer's projections and
its attention call, as one pass over both tensors (csrc/fa_rope.hip), with its backward.

No counterpart in the reference, which starts at the attention call. Names, checks and the
choice of a backend follow :mod:`.attention`: inputs the gfx950 kernels do not serve run the
same formulas in PyTorch under ``backend="auto"`` and raise under ``backend="triton"``.
"""

from __future__ import annotations

import math
from numbers import Real

import torch

from . import _lib, _native, _ops
from .attention import (_REASON_LIBRARY, _SUPPORTED_ARCH, _SUPPORTED_DTYPES, Backend, _device_arch,
                        _forward_ad_active, _warn_library_once)


def _check_backend(backend: str) -> None:
    if backend not in ("auto", "triton", "torch"):
        raise ValueError("backend must be one of: 'auto', 'triton', 'torch'")


def _binding(backend: str):
    """The C++ binding, which serves the call or finds that Python has to look; None where the
    call does not go there (torch.compile cannot trace into it)."""
    if (backend == "auto" or backend == "triton") and not torch.compiler.is_dynamo_compiling():
        return _native.module()
    return None


def _check_tensor(name: str, t, ndim: int, shape: str) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.ndim != ndim:
        raise ValueError(f"{name} must have shape {shape}; got {tuple(t.shape)}")


def _gpu_reason(t: torch.Tensor) -> str | None:
    """Why no gfx950 kernel can run on ``t``'s device, or None."""
    if t.device.type != "cuda":
        return "the Triton kernel requires a CUDA tensor"
    arch = _device_arch(t.device)
    if not arch.startswith(_SUPPORTED_ARCH):
        return ("the tuned kernel requires an AMD Instinct MI355X (gfx950) GPU; "
                f"found {arch or 'an unknown device'}")
    ok, why = _lib.available()
    return None if ok else f"{_REASON_LIBRARY}: {why}"


def _falls_back(backend: str, reason: str | None) -> bool:
    """Whether a call runs in PyTorch: ``reason`` says why no kernel serves it (None: one
    does). ``backend="triton"`` raises instead."""
    if backend == "torch":
        return True
    if reason is None:
        return False
    if backend == "triton":
        raise RuntimeError(f"Triton backend is unavailable: {reason}")
    if _REASON_LIBRARY in reason:
        _warn_library_once(reason)
    return True


def _validate(query, key, cos, sin, query_weight, key_weight, eps, positions, interleaved) -> None:
    shape = "(batch, heads, sequence, head_dim)"
    for name, t in (("query", query), ("key", key)):
        _check_tensor(name, t, 4, shape)
        if 0 in t.shape:
            raise ValueError(f"{name} dimensions must all be greater than zero")
        if not t.is_floating_point():
            raise ValueError(f"{name} must be a floating-point tensor; got {t.dtype}")
    if query.device != key.device:
        raise ValueError("query and key must be on the same device")
    if query.dtype != key.dtype:
        raise ValueError("query and key must have the same dtype")
    B, _, N, D = query.shape
    if (key.shape[0], key.shape[2], key.shape[3]) != (B, N, D):
        raise ValueError("query and key batch, sequence and head dimensions must match")
    for name, t in (("cos", cos), ("sin", sin)):
        _check_tensor(name, t, 2, "(positions, rotated values / 2)")
        if t.dtype != torch.float32 or t.device != query.device:
            raise ValueError(f"{name} must be float32 on the query's device")
    if cos.shape != sin.shape:
        raise ValueError("cos and sin must have the same shape")
    if 0 in cos.shape or 2 * cos.shape[1] > D:
        raise ValueError(
            f"cos and sin must have between 1 and head_dim / 2 = {D // 2} columns and at least "
            f"one row; got {tuple(cos.shape)}")
    if (query_weight is None) != (key_weight is None):
        raise ValueError("query_weight and key_weight must both be given or both be None")
    for name, w in (("query_weight", query_weight), ("key_weight", key_weight)):
        if w is None:
            continue
        _check_tensor(name, w, 1, "(head_dim,)")
        if w.shape[0] != D or w.device != query.device:
            raise ValueError(f"{name} must have head_dim = {D} values on the query's device")
        if w.dtype not in (query.dtype, torch.float32) or w.dtype != query_weight.dtype:
            raise ValueError("the norm weights must both have the query's dtype or both float32")
    if not isinstance(eps, Real) or not math.isfinite(float(eps)) or eps < 0:
        raise ValueError("eps must be a finite real number that is not negative")
    if not isinstance(interleaved, bool):
        raise TypeError("interleaved must be a bool")
    if positions is None:
        if N > cos.shape[0]:
            raise ValueError(f"cos and sin have {cos.shape[0]} rows for {N} tokens")
    else:
        if not isinstance(positions, torch.Tensor):
            raise TypeError("positions must be a torch.Tensor")
        if tuple(positions.shape) not in ((N,), (B, N)):
            raise ValueError(
                f"positions must have shape ({N},) or ({B}, {N}); got {tuple(positions.shape)}")
        if positions.dtype not in (torch.int32, torch.int64) or positions.device != query.device:
            raise ValueError("positions must be int32 or int64 on the query's device")


def _kernel_reason(query, key, cos, sin, eps) -> str | None:
    if query.device.type != "cuda":
        return _gpu_reason(query)
    if query.dtype not in _SUPPORTED_DTYPES:
        return "the kernel currently supports float16 and bfloat16"
    if query.shape[3] > 128 or query.shape[3] % 8:
        return "head_dim must be a multiple of 8 of at most 128"
    if cos.shape[1] % 8:
        return "the number of rotated values must be a multiple of 16"
    if max(query.shape[1], key.shape[1]) >= 1 << 15 or query.shape[0] * query.shape[2] >= 1 << 31:
        return "too many heads or tokens for one launch"
    if eps > torch.finfo(torch.float32).max:
        return f"eps {eps!r} is outside float32"
    if _forward_ad_active() or (torch.is_grad_enabled() and (cos.requires_grad or sin.requires_grad)):
        return "the kernel has no derivative in cos and sin and no forward-mode derivative"
    return _gpu_reason(query)


def _torch_rope(x, w, cos, sin, eps, positions, interleaved):
    """The formulas in PyTorch, in float32 (float64 for a float64 input)."""
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    y = x.to(wide)
    if positions is None:
        c, s = cos[:x.shape[2]], sin[:x.shape[2]]
    else:
        known = (positions >= 0) & (positions < cos.shape[0])
        at = torch.where(known, positions, 0).long()
        # [N, R/2] or [B, 1, N, R/2]; a token outside the tables is NaN, and by the product so
        # are its gradients (the tables' are not: where keeps them apart)
        known = known[..., None]
        c, s = (torch.where(known, t[at], math.nan) for t in (cos, sin))
        if positions.ndim == 2:
            known, c, s = known[:, None], c[:, None], s[:, None]
        y = y * torch.where(known, 1.0, math.nan).to(wide)
    if w is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * w.to(wide)
    c, s, half = c.to(wide), s.to(wide), cos.shape[1]
    turned, rest = y[..., :2 * half], y[..., 2 * half:]
    if interleaved:
        a, b = turned[..., ::2], turned[..., 1::2]
        z = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        z = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((z, rest), -1).to(x.dtype)


class _QkNormRope(torch.autograd.Function):
    """The kernels' autograd bridge. Saves the inputs only where a norm's gradient needs them."""

    @staticmethod
    def forward(ctx, query, key, query_weight, key_weight, cos, sin, positions, eps, interleaved):
        norm = query_weight is not None
        ctx.save_for_backward(query if norm else None, key if norm else None, query_weight,
                              key_weight, cos, sin, positions)
        ctx.eps, ctx.interleaved = eps, interleaved
        return _ops.qk_norm_rope(query, key, cos, sin, query_weight, key_weight, eps, positions,
                                 interleaved)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_query, grad_key):
        query, key, query_weight, key_weight, cos, sin, positions = ctx.saved_tensors
        grads = _ops.qk_norm_rope_bwd(
            grad_query, grad_key, query, key, cos, sin, query_weight, key_weight, ctx.eps,
            positions, ctx.interleaved, weights=ctx.needs_input_grad[2:4])
        return (*grads, None, None, None, None, None)


def qk_norm_rope(
    query: torch.Tensor,
    key: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    *,
    query_weight: torch.Tensor | None = None,
    key_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    positions: torch.Tensor | None = None,
    interleaved: bool = False,
    backend: Backend = "auto",
) -> tuple[torch.Tensor, torch.Tensor]:
    """RMS-normalise each head's queries and keys and rotate them by their positions.

    query [B, Hq, N, D] and key [B, Hkv, N, D] may be strided (views of projections). Each row
    x becomes ``y = x / sqrt(mean(x^2) + eps) * weight`` (``y = x`` without weights, which are
    given for both or for neither: [D], of the inputs' dtype or float32), and its first R
    values are rotated in pairs by its token's R / 2 angles: the values i and i + R / 2, or with
    ``interleaved`` 2 i and 2 i + 1. ``cos`` and ``sin`` [P, R / 2] hold the angles' cosines and
    sines in float32 for P positions; ``positions`` [N] or [B, N] (int32 or int64) names each
    token's row, by default 0 .. N - 1. A token whose position is not in [0, P) gets NaN, in its
    gradients too.

    Returns contiguous (query, key), computed in float32 and rounded once, differentiable in
    query, key and the weights. The gfx950 kernels serve float16 and bfloat16 with head_dim a
    multiple of 8 up to 128 and R a multiple of 16; a weight's gradient is a float32 sum in a
    fixed order.

    A call that records gradients raises while it is captured into a graph if a result of an
    earlier call with the same leaf tensors is alive on the default stream, since a backward
    captured with it would draw that stream into the capture: drop or detach the result first,
    and capture a forward alone under ``torch.no_grad()``.
    """
    native = _binding(backend)
    if native is not None and not _forward_ad_active():
        out = native.qk_norm_rope(query, key, cos, sin, query_weight, key_weight, eps, positions,
                                  interleaved)
        if out is not None:
            return out
    _check_backend(backend)
    _validate(query, key, cos, sin, query_weight, key_weight, eps, positions, interleaved)
    eps = float(eps)
    if _falls_back(backend, None if backend == "torch" else _kernel_reason(
            query, key, cos, sin, eps)):
        return tuple(_torch_rope(x, w, cos, sin, eps, positions, interleaved).contiguous()
                     for x, w in ((query, query_weight), (key, key_weight)))
    weights = () if query_weight is None else (query_weight, key_weight)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (query, key, *weights)):
        if native is not None:
            native.refuse_mixed_capture([query, key, *weights])
        return _QkNormRope.apply(query, key, query_weight, key_weight, cos, sin, positions,
                                 eps, interleaved)
    return _ops.qk_norm_rope(query, key, cos, sin, query_weight, key_weight, eps, positions,
                             interleaved)
