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
RuntimeError.  There is no CPU fallback: tensors must be on a CUDA device.
No counterpart in the reference.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib

__all__ = ["Int8Weight", "delta_scan", "delta_step", "int8_linear", "orthogonalize", "quantize_rows", "stalls"]

_DTYPE = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def _require(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


def _on(x: torch.Tensor, device: torch.device, name: str) -> None:
    _require(isinstance(x, torch.Tensor) and x.device == device, f"{name} must be a tensor on {device}")


def _cuda_device(x, name: str) -> torch.device:
    _require(isinstance(x, torch.Tensor) and x.is_cuda, f"{name} must be a CUDA tensor")
    return x.device


def _stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


def _no_grad_path(name: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError(f"{name} has no gradient; call it under torch.no_grad() or on detached tensors")


def stalls(device: int = 0) -> int:
    """Times that a kernel gave up on an internal wait (0 unless something is broken); synchronises."""
    n = ctypes.c_uint32()
    _lib.check(_lib.load().nesle_ops_stalls(device, ctypes.byref(n)))
    return n.value


# ------------------------------------------------------------------ 8-bit product

def _rows(x: torch.Tensor) -> torch.Tensor:
    """(..., cols) as (rows, cols) with unit column stride; copies only where the layout has to change."""
    x = x.reshape(-1, x.shape[-1]) if x.dim() != 2 else x
    return x if x.stride(1) == 1 or x.shape[1] <= 1 else x.contiguous()


def _ld(x: torch.Tensor) -> int:
    """Row stride of a 2-D tensor; where a stride carries no meaning (one row, or none) the row length."""
    return x.stride(0) if x.shape[0] > 1 else max(x.shape[1], 1)


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Symmetric 8-bit quantisation of the last dimension: ``(q, scale)`` with ``q = round(x / scale)`` (half to even)
    in [-127, 127], ``scale = max|x| / 127`` in fp32, of shapes ``x.shape`` and ``x.shape[:-1]``.  A zero row has scale
    0.  A NaN or an infinity in a row becomes the row's scale.  ``q``'s rows lie a multiple of 16 bytes apart, as
    :func:`int8_linear` reads them best."""
    dev = _cuda_device(x, "x")
    _require(x.dtype in _DTYPE, "x must be float32, bfloat16 or float16")
    _require(x.dim() >= 1, "x needs at least one dimension")
    _no_grad_path("quantize_rows", x)
    shape, x = x.shape, x if x.dim() > 1 else x[None]
    cols = shape[-1]
    if cols == 0:
        return x.new_empty(shape, dtype=torch.int8), x.new_zeros(shape[:-1], dtype=torch.float32)
    x2 = _rows(x)
    if x2.stride(0) < cols and x2.shape[0] > 1:  # rows that overlap or repeat (an expanded tensor)
        x2 = x2.contiguous()
    ld = -(-cols // 16) * 16
    q = torch.empty((x2.shape[0], ld), dtype=torch.int8, device=dev)[:, :cols]
    scale = torch.empty(x2.shape[0], dtype=torch.float32, device=dev)
    _lib.check(_lib.load().nesle_quantize_rows(x2.data_ptr(), _DTYPE[x2.dtype], x2.shape[0], cols, _ld(x2), q.data_ptr(),
                                               ld, scale.data_ptr(), dev.index, _stream(dev)))
    return (q if len(shape) == 2 else q.unflatten(0, shape[:-1]) if len(shape) > 2 else q[0]), scale.view(shape[:-1])


class Int8Weight:
    """A weight matrix ``(n, k)`` in 8 bits with a scale for each channel, laid out once for :func:`int8_linear`: rows
    padded with zeros to a multiple of 16 bytes, and the same matrix + 128 as unsigned bytes for unsigned tokens."""

    def __init__(self, q: torch.Tensor, scale: torch.Tensor):
        dev = _cuda_device(q, "q")
        _require(q.dtype == torch.int8 and q.dim() == 2, "q must be a 2-D int8 tensor")
        _on(scale, dev, "scale")
        _require(scale.dtype == torch.float32 and scale.shape == q.shape[:1], "scale must be float32 of shape (n,)")
        self.n, self.k = q.shape
        self.ld = max(16, -(-self.k // 16) * 16)
        self.q = torch.zeros((self.n, self.ld), dtype=torch.int8, device=dev)
        self.q[:, :self.k] = q
        self.biased = self.q.view(torch.uint8) ^ 128  # two's complement: flipping the top bit adds 128
        self.scale = scale.detach().contiguous().clone()
        self.device = dev

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
    """``act(x_scale * weight.scale * (x @ weight.q.T) + bias)`` with the integer product exact in 32 bits.

    ``x`` is ``(..., k)``: uint8 (RAM bytes) or int8 with ``x_scale`` a number or a float32 tensor ``x.shape[:-1]``; or
    floating, which is quantised per token first (:func:`quantize_rows`; ``x_scale`` stays None).  ``bias`` is float32
    ``(n,)``.  The result is ``(..., n)`` in ``out_dtype`` (bfloat16, float16 or float32), or written to ``out``."""
    dev = _cuda_device(x, "x")
    _require(isinstance(weight, Int8Weight) and weight.device == dev, f"weight must be an Int8Weight on {dev}")
    _require(x.dim() >= 1 and x.shape[-1] == weight.k, f"x must have {weight.k} columns, has shape {tuple(x.shape)}")
    _no_grad_path("int8_linear", x, bias)
    if x.dtype in _DTYPE:
        _require(x_scale is None, "x_scale is computed where x is floating")
        x, x_scale = quantize_rows(x)
    _require(x.dtype in (torch.uint8, torch.int8), "x must be uint8, int8 or floating")
    shape = x.shape[:-1]
    x2 = _rows(x if x.dim() > 1 else x[None])
    if x2.stride(0) < x2.shape[1] and x2.shape[0] > 1:
        x2 = x2.contiguous()
    m, k = x2.shape
    a = _lib.Int8Args()
    if isinstance(x_scale, torch.Tensor):
        _on(x_scale, dev, "x_scale")
        _require(x_scale.dtype == torch.float32 and x_scale.shape == shape, f"x_scale must be float32 of shape {tuple(shape)}")
        x_scale = x_scale.contiguous()
        a.x_scale = x_scale.data_ptr()
    else:
        _require(x_scale is not None, "x_scale is needed where x is integer")
        a.x_scale_value = float(x_scale)
    if bias is not None:
        _on(bias, dev, "bias")
        _require(bias.dtype == torch.float32 and bias.shape == (weight.n,), f"bias must be float32 of shape ({weight.n},)")
        bias = bias.detach().contiguous()
        a.bias = bias.data_ptr()
    if out is None:
        _require(out_dtype in _DTYPE, "out_dtype must be float32, bfloat16 or float16")
        out = torch.empty((*shape, weight.n), dtype=out_dtype, device=dev)
    else:
        _on(out, dev, "out")
        _require(out.dtype in _DTYPE and out.shape == (*shape, weight.n), f"out must be floating of shape {(*shape, weight.n)}")
        _require(out.dim() < 3 or out.is_contiguous(), "out of more than two dimensions must be contiguous")
    y = out.view(-1, weight.n) if out.dim() != 2 else out
    _require(y.stride(1) == 1 or y.shape[1] <= 1, "out must have unit column stride")
    _require(y.shape[0] <= 1 or y.stride(0) >= weight.n, "out's rows must not overlap")
    a.x, a.x_unsigned, a.ld_x = x2.data_ptr(), x2.dtype == torch.uint8, _ld(x2)
    a.w, a.w_biased, a.ld_w, a.w_scale = weight.q.data_ptr(), weight.biased.data_ptr(), weight.ld, weight.scale.data_ptr()
    a.y, a.y_dtype, a.ld_y = y.data_ptr(), _DTYPE[y.dtype], _ld(y)
    a.m, a.k, a.n, a.relu, a.device = m, k, weight.n, relu, dev.index
    lib = _lib.load()
    need = lib.nesle_int8_workspace(ctypes.byref(a))
    if need:
        scratch = torch.empty(need, dtype=torch.uint8, device=dev)
        a.workspace, a.workspace_bytes = scratch.data_ptr(), need
    _lib.check(lib.nesle_int8_linear(ctypes.byref(a), _stream(dev)))
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
    _no_grad_path("orthogonalize", update)
    rows, cols = update.shape[-2:]
    if out is None:
        out = torch.empty(update.shape, dtype=torch.bfloat16, device=dev)
    else:
        _on(out, dev, "out")
        _require(out.dtype == torch.bfloat16 and out.shape == update.shape and out.is_contiguous(),
                 f"out must be contiguous bfloat16 of shape {tuple(update.shape)}")
    x = update if update.dim() == 3 else update.reshape(-1, rows, cols) if out.numel() else update.new_empty((0, rows, cols))
    a = _lib.OrthArgs(x.data_ptr(), _DTYPE[x.dtype], *x.stride(), *x.shape, steps, eps, out.data_ptr(), None, 0, dev.index)
    lib = _lib.load()
    need = lib.nesle_orth_workspace(ctypes.byref(a))
    if need:
        scratch = torch.empty(need, dtype=torch.uint8, device=dev)
        a.workspace, a.workspace_bytes = scratch.data_ptr(), need
    _lib.check(lib.nesle_orthogonalize(ctypes.byref(a), _stream(dev)))
    return out


# ------------------------------------------------------------------ gated delta rule

def _delta_inputs(q, k, v, g, beta, reset, lead: str):
    """Checks what delta_step and delta_scan share; ``lead`` names the dimensions before the head size."""
    dev = _cuda_device(q, "q")
    dims = len(lead) + 1
    _require(q.dtype in _DTYPE, "q must be float32, bfloat16 or float16")
    _require(q.dim() == dims, f"q must have shape ({', '.join(lead)}, dk)")
    for name, x in (("k", k), ("v", v), ("g", g), ("beta", beta)):
        _on(x, dev, name)
    _require(k.shape == q.shape and k.dtype == q.dtype, f"k must be {q.dtype} of shape {tuple(q.shape)}")
    _require(v.dim() == dims and v.shape[:-1] == q.shape[:-1] and v.dtype == q.dtype,
             f"v must be {q.dtype} of shape {tuple(q.shape[:-1])} + (dv,)")
    for name, x in (("g", g), ("beta", beta)):
        _require(x.dtype == torch.float32 and x.shape == q.shape[:-1], f"{name} must be float32 of shape {tuple(q.shape[:-1])}")
    _require(1 <= q.shape[-1] <= 128 and 1 <= v.shape[-1] <= 128, "head sizes must be 1 to 128")
    if reset is not None:
        _on(reset, dev, "reset")
        _require(reset.dtype in (torch.bool, torch.uint8) and reset.shape == q.shape[:-2],
                 f"reset must be bool or uint8 of shape {tuple(q.shape[:-2])}")
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
    given.  Returns ``o`` (n, h, dv) in q's type, or writes it to ``out`` (contiguous).  Without gradients: for a
    sequence with gradients see :func:`delta_scan`."""
    dev = _delta_inputs(q, k, v, g, beta, reset, "nh")
    _no_grad_path("delta_step", q, k, v, g, beta, state)
    n, h, dk = q.shape
    dv = v.shape[-1]
    _on(state, dev, "state")
    _require(state.dtype == torch.float32 and state.shape == (n, h, dk, dv), f"state must be float32 of shape {(n, h, dk, dv)}")
    _require((state.stride(3) == 1 or dv == 1) and (state.stride(2) == dv or dk == 1), "state's matrices must be contiguous")
    _require((n <= 1 or state.stride(0) >= dk * dv) and (h <= 1 or state.stride(1) >= dk * dv), "state's matrices must not overlap")
    if out is None:
        out = torch.empty((n, h, dv), dtype=q.dtype, device=dev)
    else:
        _on(out, dev, "out")
        _require(out.dtype == q.dtype and out.shape == (n, h, dv) and out.is_contiguous(),
                 f"out must be contiguous {q.dtype} of shape {(n, h, dv)}")
    q, k, v = _unit(q), _unit(k), _unit(v)
    a = _lib.DeltaStepArgs(q.data_ptr(), k.data_ptr(), v.data_ptr(), q.stride(0), q.stride(1), k.stride(0), k.stride(1),
                           v.stride(0), v.stride(1), _DTYPE[q.dtype], g.data_ptr(), beta.data_ptr(), g.stride(0), g.stride(1),
                           beta.stride(0), beta.stride(1), None if reset is None else reset.data_ptr(),
                           0 if reset is None else reset.stride(0), state.data_ptr(), state.stride(0), state.stride(1),
                           out.data_ptr(), n, h, dk, dv, dk ** -0.5 if scale is None else scale, dev.index)
    _lib.check(_lib.load().nesle_delta_step(ctypes.byref(a), _stream(dev)))
    return out


def _scan_args(q, k, v, g, beta, reset, state, scale, dev):
    t, n, h, dk = q.shape
    return _lib.DeltaArgs(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), q_t=q.stride(0), q_n=q.stride(1), q_h=q.stride(2),
                          k_t=k.stride(0), k_n=k.stride(1), k_h=k.stride(2), v_t=v.stride(0), v_n=v.stride(1),
                          v_h=v.stride(2), dtype=_DTYPE[q.dtype], g=g.data_ptr(), beta=beta.data_ptr(), g_t=g.stride(0),
                          g_n=g.stride(1), g_h=g.stride(2), beta_t=beta.stride(0), beta_n=beta.stride(1),
                          beta_h=beta.stride(2), reset=None if reset is None else reset.data_ptr(),
                          reset_t=0 if reset is None else reset.stride(0), reset_n=0 if reset is None else reset.stride(1),
                          state=None if state is None else state.data_ptr(), t=t, n=n, h=h, dk=dk, dv=v.shape[-1],
                          scale=scale, device=dev.index)


class _DeltaScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, beta, state, reset, scale, grad):
        dev, (t, n, h, dk), dv = q.device, q.shape, v.shape[-1]
        o = torch.empty((t, n, h, dv), dtype=q.dtype, device=dev)
        final = torch.empty((n, h, dk, dv), dtype=torch.float32, device=dev)
        a = _scan_args(q, k, v, g, beta, reset, state, scale, dev)
        a.o, a.final_state = o.data_ptr(), final.data_ptr()
        lib = _lib.load()
        if grad:
            errors = torch.empty(lib.nesle_delta_error_floats(ctypes.byref(a)), dtype=torch.float32, device=dev)
            checkpoints = torch.empty(lib.nesle_delta_checkpoint_floats(ctypes.byref(a)), dtype=torch.float32, device=dev)
            a.errors, a.checkpoints = errors.data_ptr(), checkpoints.data_ptr()
            ctx.save_for_backward(q, k, v, g, beta, reset, errors, checkpoints)
            ctx.scale, ctx.has_state = scale, state is not None
            ctx.set_materialize_grads(False)
        _lib.check(lib.nesle_delta_scan(ctypes.byref(a), _stream(dev)))
        return o, final

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_o, d_final):
        q, k, v, g, beta, reset, errors, checkpoints = ctx.saved_tensors
        dev, (t, n, h, dk) = q.device, q.shape
        d_o = torch.zeros_like(v, memory_format=torch.contiguous_format) if d_o is None else d_o.contiguous()
        if d_final is not None:
            d_final = d_final.contiguous()
        dq, dk_, dv_ = (torch.empty(x.shape, dtype=x.dtype, device=dev) for x in (q, k, v))
        dg, dbeta = (torch.empty(x.shape, dtype=torch.float32, device=dev) for x in (g, beta))
        dstate = None
        if ctx.has_state and ctx.needs_input_grad[5]:
            dstate = torch.empty((n, h, dk, v.shape[-1]), dtype=torch.float32, device=dev)
        if t == 0:
            if dstate is not None:
                dstate = torch.zeros_like(dstate) if d_final is None else d_final.clone()
            return dq, dk_, dv_, dg, dbeta, dstate, None, None, None
        a = _scan_args(q, k, v, g, beta, reset, None, ctx.scale, dev)
        a.errors, a.checkpoints, a.d_o = errors.data_ptr(), checkpoints.data_ptr(), d_o.data_ptr()
        a.d_final = None if d_final is None else d_final.data_ptr()
        a.dq, a.d_k, a.d_v, a.dg, a.dbeta = (x.data_ptr() for x in (dq, dk_, dv_, dg, dbeta))
        a.dstate = None if dstate is None else dstate.data_ptr()
        _lib.check(_lib.load().nesle_delta_scan_backward(ctypes.byref(a), _stream(dev)))
        return dq, dk_, dv_, dg, dbeta, dstate, None, None, None


def delta_scan(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
               state: torch.Tensor | None = None, reset: torch.Tensor | None = None, *,
               scale: float | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The gated delta rule over t tokens, time first as rollouts are stored: ``(o, final_state)``, both differentiable
    in all floating inputs.  It is :func:`delta_step` token by token (up to rounding).

    ``q, k``: (t, n, h, dk), ``v``: (t, n, h, dv), one of float32, bfloat16 and float16, any strides (rows copied unless
    the last is 1); ``g, beta``: (t, n, h) float32; ``state``: (n, h, dk, dv) float32 before the first token, or None for
    zeros; ``reset``: (t, n) bool or uint8, True where a token starts an episode: nothing before it, not even a NaN,
    reaches it, and no gradient passes.  States and sums are fp32 throughout.  With gradients a call keeps one state for
    every 16 tokens until its backward pass."""
    dev = _delta_inputs(q, k, v, g, beta, reset, "tnh")
    t, n, h, dk = q.shape
    if state is not None:
        _on(state, dev, "state")
        _require(state.dtype == torch.float32 and state.shape == (n, h, dk, v.shape[-1]),
                 f"state must be float32 of shape {(n, h, dk, v.shape[-1])}")
        state = state.contiguous()
    grad = torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (q, k, v, g, beta, state))
    return _DeltaScan.apply(_unit(q), _unit(k), _unit(v), g, beta, state, reset, dk ** -0.5 if scale is None else float(scale),
                            grad)
