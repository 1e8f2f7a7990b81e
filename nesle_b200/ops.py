"""Policy-learning operators on the GPU (include/nesle_ops.h): what a recurrent
actor-critic on the batched core computes beside the env step.

* ``int8_linear`` / ``quantize_rows`` / ``Int8Weight`` -- product of 8-bit
  integers with a scale for each token and channel.  RAM observations are bytes
  already and go in as they are.
* ``delta_step`` / ``delta_scan`` -- the gated delta rule, a memory of fixed
  size for every env and head: one token in place (rollout), and a whole
  rollout with its gradients (update).
* ``orthogonalize`` -- Newton-Schulz orthogonalisation of matrix updates, for
  the ``Muon`` optimiser (nesle_b200.muon).

Calls go on the caller's current torch stream, return before the work is done,
and never synchronise the host.  Argument errors raise ValueError, CUDA errors
RuntimeError.  There is no CPU fallback: tensors must be on a CUDA device.  They
are read as they lie in memory: a lazily negated view (``Tensor.is_neg``) is to be
resolved first.
No counterpart in the reference.
"""
from __future__ import annotations

import ctypes
import functools

import torch
from torch.autograd import forward_ad

from . import _lib

__all__ = ["Int8Weight", "delta_scan", "delta_step", "int8_linear", "orthogonalize", "quantize_rows", "stalls"]

_DTYPE = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_stream = torch._C._cuda_getCurrentRawStream
# What a kernel writes in place has changed for autograd too: a gradient that saved the old values is then refused.
_written = torch.autograd.graph.increment_version


def _require(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


def _on(x: torch.Tensor, index: int, name: str) -> None:
    if not isinstance(x, torch.Tensor) or x.get_device() != index:
        raise ValueError(f"{name} must be a tensor on cuda:{index}")


def _cuda_device(x, name: str) -> int:
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    return x.get_device()


def _no_grad_path(name: str, *tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{name} has no gradient; call it under torch.no_grad() or on detached tensors")
    if forward_ad._current_level >= 0:  # within a dual_level()
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError(f"{name} has no forward-mode derivative; call it on primal tensors")


def _call(name: str, args: bytes, *rest: int) -> None:
    lib = _lib.load()
    rc = getattr(lib, name)(args, *rest)
    if rc:
        _lib.check(rc, lib)


def stalls(device: int = 0) -> int:
    """Times that a kernel gave up on an internal wait (0 unless something is broken); synchronises."""
    n = ctypes.c_uint32()
    _lib.check(_lib.load().nesle_ops_stalls(device, ctypes.byref(n)))
    return n.value


# ------------------------------------------------------------------ 8-bit product

def _rows(x: torch.Tensor) -> tuple[torch.Tensor, int]:
    """(..., cols) as (rows, cols) with unit column stride and rows that do not overlap, and the rows' distance; copies
    only where the layout has to change.  Where a stride carries no meaning (one row, or none) it is the row length."""
    if x.dim() != 2:
        x = x.reshape(x.shape[:-1].numel(), x.shape[-1])  # not -1, which says nothing where there are no columns
    rows, cols = x.shape
    ld, unit = x.stride()
    if (unit != 1 and cols > 1) or (ld < cols and rows > 1):
        x, ld = x.contiguous(), cols
    return x, ld if rows > 1 else max(cols, 1)


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Symmetric 8-bit quantisation of the last dimension: ``(q, scale)`` with ``q = round(x / scale)`` (half to even)
    clamped to [-127, 127], ``scale = max|x| / 127`` in fp32, of shapes ``x.shape`` and ``x.shape[:-1]``.  A zero row has
    scale 0.  A NaN or an infinity in a row becomes the row's scale.  ``q``'s rows lie a multiple of 16 bytes apart, as
    :func:`int8_linear` reads them best."""
    dev = _cuda_device(x, "x")
    dtype = _DTYPE.get(x.dtype)
    _require(dtype is not None, "x must be float32, bfloat16 or float16")
    _require(x.dim() >= 1, "x needs at least one dimension")
    _no_grad_path("quantize_rows", x)
    shape = x.shape
    cols = shape[-1]
    if cols == 0:
        return x.new_empty(shape, dtype=torch.int8), x.new_zeros(shape[:-1], dtype=torch.float32)
    x, ld = _rows(x)
    rows = x.shape[0]
    ld_q = -(-cols // 16) * 16
    q = torch.empty((rows, ld_q), dtype=torch.int8, device=x.device)
    scale = torch.empty(shape[:-1], dtype=torch.float32, device=x.device)
    lib = _lib.load()
    rc = lib.nesle_quantize_rows(x.data_ptr(), dtype, rows, cols, ld, q.data_ptr(), ld_q, scale.data_ptr(), dev, _stream(dev))
    if rc:
        _lib.check(rc, lib)
    if ld_q != cols:
        q = q[:, :cols]
    return (q if len(shape) == 2 else q.unflatten(0, shape[:-1]) if len(shape) > 2 else q[0]), scale


class Int8Weight:
    """A weight matrix ``(n, k)`` in 8 bits with a scale for each channel, laid out once for :func:`int8_linear`: rows
    padded with zeros to a multiple of 16 bytes, and the same matrix + 128 as unsigned bytes for unsigned tokens.  A copy,
    without gradients."""

    def __init__(self, q: torch.Tensor, scale: torch.Tensor):
        dev = _cuda_device(q, "q")
        _require(q.dtype == torch.int8 and q.dim() == 2, "q must be a 2-D int8 tensor")
        _on(scale, dev, "scale")
        _require(scale.dtype == torch.float32 and scale.shape == q.shape[:1], "scale must be float32 of shape (n,)")
        self.n, self.k = q.shape
        self.ld = max(16, -(-self.k // 16) * 16)
        if self.ld == self.k:
            self.q = q.detach().clone(memory_format=torch.contiguous_format)
        else:
            self.q = torch.nn.functional.pad(q.detach(), (0, self.ld - self.k))
        self.biased = self.q.view(torch.uint8) ^ 128  # two's complement: flipping the top bit adds 128
        self.scale = scale.detach().clone(memory_format=torch.contiguous_format)
        self.device = q.device
        self._index = dev

    @classmethod
    def from_float(cls, weight: torch.Tensor) -> "Int8Weight":
        """Quantises a floating ``(n, k)`` matrix, each channel by its own largest magnitude."""
        return cls(*quantize_rows(weight.detach()))

    @property
    def shape(self) -> tuple[int, int]:
        return self.n, self.k


def int8_linear(x: torch.Tensor, weight: Int8Weight, x_scale: torch.Tensor | float | None = None,
                bias: torch.Tensor | None = None, *, relu: bool = False, out_dtype: torch.dtype = torch.bfloat16,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """``act(x_scale * weight.scale * (x @ weight.q.T) + bias)`` with the integer product exact in 32 bits, for which k
    is at most 33,025 with uint8 tokens and 131,071 with others.

    ``x`` is ``(..., k)``: uint8 (RAM bytes) or int8 with ``x_scale`` a number or a float32 tensor ``x.shape[:-1]``; or
    floating, which is quantised per token first (:func:`quantize_rows`; ``x_scale`` stays None).  ``bias`` is float32
    ``(n,)``.  The result is ``(..., n)`` in ``out_dtype`` (bfloat16, float16 or float32), or written to ``out``, which may
    lie on the memory of ``x``, ``x_scale`` and ``bias``."""
    dev = _cuda_device(x, "x")
    _require(isinstance(weight, Int8Weight) and weight._index == dev, f"weight must be an Int8Weight on cuda:{dev}")
    n, k = weight.n, weight.k
    shape = x.shape
    _require(len(shape) >= 1 and shape[-1] == k, f"x must have {k} columns, has shape {tuple(shape)}")
    _no_grad_path("int8_linear", x, bias, x_scale if isinstance(x_scale, torch.Tensor) else None, out)
    if x.dtype in _DTYPE:
        _require(x_scale is None, "x_scale is computed where x is floating")
        x, x_scale = quantize_rows(x)
    unsigned = x.dtype == torch.uint8
    _require(unsigned or x.dtype == torch.int8, "x must be uint8, int8 or floating")
    shape = shape[:-1]
    x, ld_x = _rows(x)
    m = x.shape[0]
    scale_ptr, scale_value, bias_ptr = 0, 0.0, 0
    if isinstance(x_scale, torch.Tensor):
        _on(x_scale, dev, "x_scale")
        _require(x_scale.dtype == torch.float32 and x_scale.shape == shape, f"x_scale must be float32 of shape {tuple(shape)}")
        x_scale = x_scale.contiguous()
        scale_ptr = x_scale.data_ptr()
    else:
        _require(x_scale is not None, "x_scale is needed where x is integer")
        scale_value = float(x_scale)
    if bias is not None:
        _on(bias, dev, "bias")
        _require(bias.dtype == torch.float32 and bias.shape == (n,), f"bias must be float32 of shape ({n},)")
        bias = bias.detach().contiguous()
        bias_ptr = bias.data_ptr()
    fresh = out is None
    if fresh:
        _require(out_dtype in _DTYPE, "out_dtype must be float32, bfloat16 or float16")
        out = torch.empty((*shape, n), dtype=out_dtype, device=x.device)
        ld_y = max(n, 1)
    else:
        _on(out, dev, "out")
        _require(out.dtype in _DTYPE and out.shape == (*shape, n), f"out must be floating of shape {(*shape, n)}")
        _require(out.dim() == 2 or out.is_contiguous(), "out of other than two dimensions must be contiguous")
        ld_y = out.stride(0) if out.dim() == 2 and m > 1 else max(n, 1)
        _require(out.dim() != 2 or out.stride(1) == 1 or n <= 1, "out must have unit column stride")
        _require(ld_y >= n, "out's rows must not overlap")
    x_ptr = x.data_ptr()
    # many rows that do not lie on 16 bytes are laid out again in scratch memory (as much as nesle_int8_workspace says)
    need = m * (-(-k // 16) * 16) if m > 64 and (x_ptr % 16 or ld_x % 16) else 0
    scratch = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
    lib = _lib.load()
    rc = lib.nesle_int8_linear(
        _lib.INT8_ARGS.pack(x_ptr, unsigned, ld_x, scale_ptr, scale_value, weight.q.data_ptr(), weight.biased.data_ptr(),
                            weight.ld, weight.scale.data_ptr(), bias_ptr, out.data_ptr(), _DTYPE[out.dtype], ld_y, m, k, n,
                            relu, scratch.data_ptr() if need else 0, need, dev), _stream(dev))
    if rc:
        if rc != _lib.NESLE_ERR_OVERLAP or fresh:
            _lib.check(rc, lib)
        # tiles still read the memory when others write it: the results go there last
        y = int8_linear(x, weight, x_scale.flatten() if scale_ptr else x_scale, bias, relu=relu, out_dtype=out.dtype)
        out.copy_(y.view(out.shape))
    elif not fresh:
        _written(out)
    return out


# ------------------------------------------------------------------ Newton-Schulz

def orthogonalize(update: torch.Tensor, *, steps: int = 5, eps: float = 1e-7,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """Orthogonalises each matrix of ``update`` (``(..., rows, cols)``, float32, bfloat16 or float16, any strides):
    divided by its Frobenius norm plus ``eps``, then ``steps`` Newton-Schulz rounds X <- aX + (bA + cA^2)X with
    A = X X^T on the smaller side and (a, b, c) = (3.4445, -4.7750, 2.0315).  Singular values end between about 0.7 and
    1.2, singular vectors stay.  The result is bfloat16 of the same shape, or written to ``out`` (contiguous bfloat16).
    Products carry 22 bits of both operands; a zero matrix stays zero, a NaN or an infinity makes its matrix NaN."""
    dev = _cuda_device(update, "update")
    _require(update.dtype in _DTYPE, "update must be float32, bfloat16 or float16")
    _require(update.dim() >= 2, "update must have at least two dimensions")
    _require(1 <= steps < 1 << 31 and int(steps) == steps, "steps must be a whole number, at least 1")
    _no_grad_path("orthogonalize", update, out)
    rows, cols = update.shape[-2:]
    fresh = out is None
    if fresh:
        out = torch.empty(update.shape, dtype=torch.bfloat16, device=update.device)
    else:
        _on(out, dev, "out")
        _require(out.dtype == torch.bfloat16 and out.shape == update.shape and out.is_contiguous(),
                 f"out must be contiguous bfloat16 of shape {tuple(update.shape)}")
    x = update if update.dim() == 3 else update.reshape(-1, rows, cols) if out.numel() else update.new_empty((0, rows, cols))

    def args(scratch=0, size=0):
        return _lib.ORTH_ARGS.pack(x.data_ptr(), _DTYPE[x.dtype], *x.stride(), *x.shape, int(steps), eps, out.data_ptr(), scratch,
                                   size, dev)

    need = _lib.load().nesle_orth_workspace(args())
    scratch = torch.empty(need, dtype=torch.uint8, device=x.device)
    _call("nesle_orthogonalize", args(scratch.data_ptr(), need), _stream(dev))
    if not fresh:
        _written(out)
    return out


# ------------------------------------------------------------------ gated delta rule

def _delta_inputs(q, k, v, g, beta, reset, lead: str) -> int:
    """Checks what delta_step and delta_scan share; ``lead`` names the dimensions before the head size."""
    dev = _cuda_device(q, "q")
    shape, dtype = q.shape, q.dtype
    dims = len(lead) + 1
    _require(dtype in _DTYPE, "q must be float32, bfloat16 or float16")
    _require(len(shape) == dims, f"q must have shape ({', '.join(lead)}, dk)")
    heads = shape[:-1]
    for name, x in (("k", k), ("v", v), ("g", g), ("beta", beta)):
        _on(x, dev, name)
    if k.shape != shape or k.dtype != dtype:
        raise ValueError(f"k must be {dtype} of shape {tuple(shape)}")
    if v.dim() != dims or v.shape[:-1] != heads or v.dtype != dtype:
        raise ValueError(f"v must be {dtype} of shape {tuple(heads)} + (dv,)")
    if g.dtype != torch.float32 or g.shape != heads:
        raise ValueError(f"g must be float32 of shape {tuple(heads)}")
    if beta.dtype != torch.float32 or beta.shape != heads:
        raise ValueError(f"beta must be float32 of shape {tuple(heads)}")
    _require(1 <= shape[-1] <= 128 and 1 <= v.shape[-1] <= 128, "head sizes must be 1 to 128")
    if reset is not None:
        _on(reset, dev, "reset")
        if reset.dtype not in (torch.bool, torch.uint8) or reset.shape != shape[:-2]:
            raise ValueError(f"reset must be bool or uint8 of shape {tuple(shape[:-2])}")
    return dev


def _unit(x: torch.Tensor) -> torch.Tensor:
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def delta_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
               state: torch.Tensor, reset: torch.Tensor | None = None, *, scale: float | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """One token of the gated delta rule for every env and head; ``state`` is updated in place:

        S0 = 0 where reset else exp(g) S;  u = beta (v - S0^T k);  S = S0 + k u^T;  o = scale S^T q

    ``q, k``: (n, h, dk), ``v``: (n, h, dv), float32, bfloat16 or float16; ``g, beta``: (n, h) float32; ``state``:
    (n, h, dk, dv) float32 with contiguous matrices; ``reset``: (n,) bool or uint8.  ``scale`` is dk ** -0.5 unless
    given.  Returns ``o`` (n, h, dv) in q's type, or writes it to ``out`` (contiguous; it may lie on the memory of the
    inputs, but ``state`` must share none with them).  Without gradients: for a sequence with gradients see
    :func:`delta_scan`."""
    dev = _delta_inputs(q, k, v, g, beta, reset, "nh")
    _no_grad_path("delta_step", q, k, v, g, beta, state, out)
    n, h, dk = q.shape
    dv = v.shape[-1]
    _on(state, dev, "state")
    if state.dtype != torch.float32 or state.shape != (n, h, dk, dv):
        raise ValueError(f"state must be float32 of shape {(n, h, dk, dv)}")
    s_n, s_h, s_k, s_v = state.stride()
    _require((s_v == 1 or dv == 1) and (s_k == dv or dk == 1), "state's matrices must be contiguous")
    inner, outer = (s_n * (n - 1), s_h) if h > 1 and (n <= 1 or s_n <= s_h) else (s_h * (h - 1), s_n)
    _require((n <= 1 or s_n >= dk * dv) and (h <= 1 or s_h >= dk * dv) and (n * h <= 1 or outer >= inner + dk * dv),
             "state's matrices must not overlap")
    fresh = out is None
    if fresh:
        out = torch.empty((n, h, dv), dtype=q.dtype, device=q.device)
    else:
        _on(out, dev, "out")
        _require(out.dtype == q.dtype and out.shape == (n, h, dv) and out.is_contiguous(),
                 f"out must be contiguous {q.dtype} of shape {(n, h, dv)}")
    q, k, v = _unit(q), _unit(k), _unit(v)
    reset_ptr, reset_n = (0, 0) if reset is None else (reset.data_ptr(), reset.stride(0))
    lib = _lib.load()
    rc = lib.nesle_delta_step(
        _lib.DELTA_STEP_ARGS.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), *q.stride()[:2], *k.stride()[:2], *v.stride()[:2],
                                  _DTYPE[q.dtype], g.data_ptr(), beta.data_ptr(), *g.stride(), *beta.stride(), reset_ptr,
                                  reset_n, state.data_ptr(), s_n, s_h, out.data_ptr(), n, h, dk, dv,
                                  dk ** -0.5 if scale is None else scale, dev), _stream(dev))
    if rc:
        if rc != _lib.NESLE_ERR_OVERLAP or fresh:
            _lib.check(rc, lib)
        # a head's other warps still read q and k when one writes its columns: the results go there last
        out.copy_(delta_step(q, k, v, g, beta, state, reset, scale=scale))
    else:
        _written(state if fresh else (state, out))
    return out


def _scan_args(q, k, v, g, beta, reset, state, scale, dev, *rest: int) -> bytes:
    """``rest``: o, final_state, errors, checkpoints, d_o, d_final, dq, d_k, d_v, dg, dbeta, dstate as far as given."""
    reset_ptr, reset_t, reset_n = (0, 0, 0) if reset is None else (reset.data_ptr(), *reset.stride())
    return _lib.DELTA_ARGS.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), *q.stride()[:3], *k.stride()[:3], *v.stride()[:3],
                                _DTYPE[q.dtype], g.data_ptr(), beta.data_ptr(), *g.stride(), *beta.stride(), reset_ptr,
                                reset_t, reset_n, 0 if state is None else state.data_ptr(), *q.shape, v.shape[-1], scale,
                                *rest, *(0,) * (12 - len(rest)), dev)


@functools.lru_cache(maxsize=256)
def _scan_sizes(t: int, n: int, h: int, dk: int, dv: int) -> tuple[int, int]:
    """Floats of the errors and the states that a scan keeps for its gradients."""
    sizes = _lib.DELTA_ARGS.pack(*(0,) * 25, t, n, h, dk, dv, 0.0, *(0,) * 12, 0)
    lib = _lib.load()
    return lib.nesle_delta_error_floats(sizes), lib.nesle_delta_checkpoint_floats(sizes)


@functools.lru_cache(maxsize=256)
def _scan_split(t: int, n: int, h: int, dk: int, dv: int, dev: int, dtype: int = _lib.BF16) -> int:
    """Floats of the workspace with which a scan cuts its sequences into segments; 0 where it does not."""
    sizes = _lib.DELTA_ARGS.pack(*(0,) * 12, dtype, *(0,) * 12, t, n, h, dk, dv, 0.0, *(0,) * 12, dev)
    return _lib.load().nesle_delta_split_floats(sizes)


class _DeltaScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, beta, state, reset, scale, grad, dev):
        (t, n, h, dk), dv, device = q.shape, v.shape[-1], q.device
        o = torch.empty((t, n, h, dv), dtype=q.dtype, device=device)
        final = torch.empty((n, h, dk, dv), dtype=torch.float32, device=device)
        kept = (0, 0)
        if grad:
            sizes = _scan_sizes(t, n, h, dk, dv)
            errors = torch.empty(sizes[0], dtype=torch.float32, device=device)
            checkpoints = torch.empty(sizes[1], dtype=torch.float32, device=device)
            kept = errors.data_ptr(), checkpoints.data_ptr()
            ctx.save_for_backward(q, k, v, g, beta, reset, errors, checkpoints)
            ctx.scale, ctx.has_state, ctx.dev = scale, state is not None, dev
            ctx.set_materialize_grads(False)
        split = _scan_split(t, n, h, dk, dv, dev, _DTYPE[q.dtype])
        ends = torch.empty(split, dtype=torch.float32, device=device) if split else None
        _call("nesle_delta_scan_split",
              _scan_args(q, k, v, g, beta, reset, state, scale, dev, o.data_ptr(), final.data_ptr(), *kept),
              ends.data_ptr() if split else 0, _stream(dev))
        return o, final

    @staticmethod
    def backward(ctx, d_o, d_final):
        if torch.is_grad_enabled():  # create_graph=True
            raise RuntimeError("delta_scan has first derivatives only")
        q, k, v, g, beta, reset, errors, checkpoints = ctx.saved_tensors
        dev, device, (t, n, h, dk) = ctx.dev, q.device, q.shape
        d_o = torch.zeros_like(v, memory_format=torch.contiguous_format) if d_o is None else d_o.contiguous()
        if d_final is not None:
            d_final = d_final.contiguous()
        dq, dk_, dv_ = (torch.empty(x.shape, dtype=x.dtype, device=device) for x in (q, k, v))
        dg, dbeta = (torch.empty(x.shape, dtype=torch.float32, device=device) for x in (g, beta))
        dstate = None
        if ctx.has_state and ctx.needs_input_grad[5]:
            dstate = torch.empty((n, h, dk, v.shape[-1]), dtype=torch.float32, device=device)
        if t == 0:
            if dstate is not None:
                dstate = torch.zeros_like(dstate) if d_final is None else d_final.clone()
        else:
            _call("nesle_delta_scan_backward",
                  _scan_args(q, k, v, g, beta, reset, None, ctx.scale, dev, 0, 0, errors.data_ptr(), checkpoints.data_ptr(),
                             d_o.data_ptr(), 0 if d_final is None else d_final.data_ptr(), dq.data_ptr(), dk_.data_ptr(),
                             dv_.data_ptr(), dg.data_ptr(), dbeta.data_ptr(), 0 if dstate is None else dstate.data_ptr()),
                  _stream(dev))
        return dq, dk_, dv_, dg, dbeta, dstate, None, None, None, None


def delta_scan(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
               state: torch.Tensor | None = None, reset: torch.Tensor | None = None, *,
               scale: float | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The gated delta rule over t tokens, time first as rollouts are stored: ``(o, final_state)``, both differentiable
    in all floating inputs.  It is :func:`delta_step` token by token (up to rounding).

    ``q, k``: (t, n, h, dk), ``v``: (t, n, h, dv), one of float32, bfloat16 and float16, any strides (rows copied unless
    the last is 1); ``g, beta``: (t, n, h) float32; ``state``: (n, h, dk, dv) float32 before the first token, or None for
    zeros; ``reset``: (t, n) bool or uint8, True where a token starts an episode: nothing before it, not even a NaN,
    reaches it, and no gradient passes.  A NaN or an infinity in a token reaches no earlier one (in the gradients it may
    spoil all tokens of its episode).  States and sums are fp32 throughout; products take them as sums of bfloat16, whose
    largest number, 3.39e38, is the largest that counts as finite.  With gradients a call keeps one state for
    every 16 tokens until its backward pass."""
    dev = _delta_inputs(q, k, v, g, beta, reset, "tnh")
    t, n, h, dk = q.shape
    if state is not None:
        _on(state, dev, "state")
        if state.dtype != torch.float32 or state.shape != (n, h, dk, v.shape[-1]):
            raise ValueError(f"state must be float32 of shape {(n, h, dk, v.shape[-1])}")
        state = state.contiguous()
    grad = torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (q, k, v, g, beta, state))
    return _DeltaScan.apply(_unit(q), _unit(k), _unit(v), g, beta, state, reset, dk ** -0.5 if scale is None else float(scale),
                            grad, dev)
