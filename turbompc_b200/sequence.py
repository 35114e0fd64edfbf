"""Sequence operators of a learned policy around the MPC solve, over the CUDA
C ABI: linear attention with a decay per head (whole sequences, with its
gradient, and single tokens), the residual addition with its root-mean-square
norm, and the gated linear layer.

All are CUDA kernels on the current stream, for float32 and bfloat16 tensors
on one device; sums, states and statistics are held in float32 and rounded
once when a result is stored.  There is no CPU fallback.  ``linear_attention``,
``add_rms_norm`` and ``gated_linear`` are differentiable (once).
"""
from __future__ import annotations

import struct
from typing import Optional, Tuple

import torch

from . import _ffi

ACTIVATIONS = {"silu": _ffi.ACT_SILU, "gelu": _ffi.ACT_GELU}
MAX_HEAD_DIM = 128

_SUFFIX = {torch.float32: "f32", torch.bfloat16: "bf16"}
_ENTRIES = {}  # (entry point, dtype) -> (ctypes function, its name)
# TmpcSeqView and TmpcLinAttnDims as packed bytes: a single token's launch is
# shorter than the building of a few ctypes structures.
_VIEW = struct.Struct("Pqqq").pack
_DIMS = struct.Struct("6i").pack


def _suffix(dtype: torch.dtype) -> str:
    s = _SUFFIX.get(dtype)
    if s is None:
        raise TypeError(f"sequence operators support float32/bfloat16, got {dtype}")
    return s


def _check(t: torch.Tensor, name: str, dtype: torch.dtype, device: torch.device) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.dtype != dtype:
        raise TypeError(f"{name} has dtype {t.dtype}, expected {dtype}")
    if not t.is_cuda:
        raise ValueError(f"{name}: turbompc_b200 kernels need CUDA tensors (no CPU fallback)")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """The kernels take any stride but the last axis's."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _p(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else (t.data_ptr() or None)


def _view(t: torch.Tensor) -> bytes:
    st = t.stride()
    if len(st) == 3:  # (B, heads, dim): one token
        return _VIEW(t.data_ptr(), st[0], 0, st[1])
    return _VIEW(t.data_ptr(), st[0], st[1], st[2])


def _empty(shape, dtype, device) -> torch.Tensor:
    return torch.empty(shape, dtype=dtype, device=device)


def _workspace(nbytes: int, device) -> Optional[torch.Tensor]:
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes > 0 else None


def _call(entry: str, dtype: torch.dtype, device: torch.device, *args) -> None:
    """One C call on the device's current stream."""
    found = _ENTRIES.get((entry, dtype))
    if found is None:
        name = f"{entry}_{_suffix(dtype)}"
        found = _ENTRIES[entry, dtype] = (getattr(_ffi.load(), name), name)
    fn, name = found
    index = device.index
    stream = torch._C._cuda_getCurrentRawStream(index)
    if torch._C._cuda_getDevice() == index:
        code = fn(*args, stream)
    else:
        with torch.cuda.device(index):
            code = fn(*args, stream)
    if code:
        raise _ffi.TmpcError(name, code)


def _grad_needed(*tensors) -> bool:
    if not torch.is_grad_enabled():
        return False
    for t in tensors:
        if t is not None and t.requires_grad:
            return True
    return False


# ---------------------------------------------------------------------------
# Linear attention
# ---------------------------------------------------------------------------
def _attention_dims(q, k, v, log_decay, axes: Tuple[str, ...]):
    """(B, T, H, G, dk, dv) of checked arguments."""
    try:
        sq, sk, sv = q.shape, k.shape, v.shape
        dtype, device = q.dtype, q.device
        if (len(sq) == len(sk) == len(sv) == len(axes) and dtype in _SUFFIX and k.dtype == dtype and v.dtype == dtype
                and q.is_cuda and k.device == device and v.device == device
                and log_decay.dtype == torch.float32 and log_decay.device == device):
            H, G, dk, dv = sq[-2], sk[-2], sq[-1], sv[-1]
            if (sk[-1] == dk and sv[-2] == G and sk[0] == sq[0] == sv[0] and sk[1:-2] == sq[1:-2] == sv[1:-2]
                    and log_decay.shape == (H,) and G > 0 and H > 0 and H % G == 0
                    and 1 <= dk <= MAX_HEAD_DIM and 1 <= dv <= MAX_HEAD_DIM):
                return sq[0], (sq[1] if len(axes) == 4 else 1), H, G, dk, dv
    except AttributeError:
        pass
    # something is wrong: say what
    if not isinstance(q, torch.Tensor):
        raise TypeError(f"q must be a tensor, got {type(q).__name__}")
    _suffix(q.dtype)
    for name, t in (("q", q), ("k", k), ("v", v)):
        _check(t, name, q.dtype, q.device)
        if t.dim() != len(axes):
            raise ValueError(f"{name} must be ({', '.join(axes)}), got shape {tuple(t.shape)}")
    if k.shape[:-1] != v.shape[:-1] or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != q.shape[-1]:
        raise ValueError(f"shapes of q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not fit")
    H, G, dk, dv = q.shape[-2], k.shape[-2], q.shape[-1], v.shape[-1]
    if G < 1 or H < 1 or H % G:
        raise ValueError(f"{H} query heads do not divide into {G} key / value heads")
    if not (1 <= dk <= MAX_HEAD_DIM and 1 <= dv <= MAX_HEAD_DIM):
        raise ValueError(f"head sizes {dk}, {dv} must be within 1..{MAX_HEAD_DIM}")
    _check(log_decay, "log_decay", torch.float32, q.device)
    raise ValueError(f"log_decay has shape {tuple(log_decay.shape)}, expected ({H},)")


def _check_state(t, name: str, want, device, contiguous: bool = False) -> None:
    _check(t, name, torch.float32, device)
    if t.shape != want:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {want}")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _attention_forward(dims, q, k, v, log_decay, lengths, initial, scale, want_state):
    B, T, H, _, dk, dv = dims
    dtype, device = q.dtype, q.device
    o = _empty((B, T, H, dv), dtype, device)
    state = _empty((B, H, dk, dv), torch.float32, device) if want_state else None
    packed = _DIMS(*dims)
    need = _ffi.load().tmpc_linear_attention_workspace_bytes(packed)
    ws = _workspace(need, device)
    _call("tmpc_linear_attention", dtype, device, packed, _view(q), _view(k), _view(v), _view(o), _p(log_decay),
          _p(lengths), _p(initial), _p(state), scale, _p(ws), need)
    return o, state


class _LinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, initial, lengths, scale, dims, want_state):
        ctx.set_materialize_grads(False)
        ctx.dims, ctx.scale = dims, scale
        ctx.save_for_backward(q, k, v, log_decay, initial, lengths)
        return _attention_forward(dims, q, k, v, log_decay, lengths, initial, scale, want_state)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do, dstate):
        q, k, v, log_decay, initial, lengths = ctx.saved_tensors
        dims, dtype, dev = ctx.dims, q.dtype, q.device
        if do is None:
            do = torch.zeros((dims[0], dims[1], dims[2], dims[5]), dtype=dtype, device=dev)
        do = _rows(do)
        dstate = None if dstate is None else dstate.contiguous()
        dq, dk, dv = _empty(q.shape, dtype, dev), _empty(k.shape, dtype, dev), _empty(v.shape, dtype, dev)
        dlog = torch.empty_like(log_decay) if ctx.needs_input_grad[3] else None
        dinit = torch.empty_like(initial) if ctx.needs_input_grad[4] else None
        packed = _DIMS(*dims)
        need = _ffi.load().tmpc_linear_attention_backward_workspace_bytes(packed)
        ws = _workspace(need, dev)
        _call("tmpc_linear_attention_backward", dtype, dev, packed, _view(q), _view(k), _view(v), _view(do), _view(dq),
              _view(dk), _view(dv), _p(log_decay), _p(lengths), _p(initial), _p(dstate), _p(dlog), _p(dinit), ctx.scale,
              _p(ws), need)
        return dq, dk, dv, dlog, dinit, None, None, None, None


def linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, *,
                     scale: Optional[float] = None, initial_state: Optional[torch.Tensor] = None,
                     lengths: Optional[torch.Tensor] = None, return_state: bool = False):
    """Causal linear attention with a decay per head over whole sequences:

        S_t = exp(log_decay_h) S_{t-1} + k_t v_t^T,    o_t = scale S_t^T q_t

    q (B, T, H, dk), k (B, T, G, dk), v (B, T, G, dv), float32 or bfloat16,
    any strides; G divides H and query head h reads key / value head
    h // (H // G).  log_decay (H,) float32, meant to be <= 0 (-inf: no memory).
    ``scale`` defaults to dk ** -0.5.  ``initial_state`` (B, H, dk, dv) float32
    is S before the first token (default zero).  ``lengths`` (B,) int32: tokens
    at and past a sequence's length give zero outputs and zero gradients and
    leave the state alone.  Returns o (B, T, H, dv), or (o, state) with the
    float32 state after the last token, which ``linear_attention_step`` and a
    later call's ``initial_state`` continue from.  Products are taken over
    chunks of tokens in bfloat16, so a NaN or infinity in a valid token may
    also reach the earlier outputs of its chunk.

    Differentiable with respect to q, k, v, log_decay and initial_state.
    """
    dims = _attention_dims(q, k, v, log_decay, ("B", "T", "H", "D"))
    B, _, H, _, dk, dv = dims
    scale = dk ** -0.5 if scale is None else float(scale)
    if initial_state is not None:
        _check_state(initial_state, "initial_state", (B, H, dk, dv), q.device)
        initial_state = initial_state.contiguous()
    if lengths is not None:
        _check(lengths, "lengths", torch.int32, q.device)
        if lengths.shape != (B,):
            raise ValueError(f"lengths has shape {tuple(lengths.shape)}, expected ({B},)")
        lengths = lengths.contiguous()
    q, k, v, log_decay = _rows(q), _rows(k), _rows(v), log_decay.contiguous()
    if _grad_needed(q, k, v, log_decay, initial_state):
        o, state = _LinearAttention.apply(q, k, v, log_decay, initial_state, lengths, scale, dims, bool(return_state))
    else:
        o, state = _attention_forward(dims, q, k, v, log_decay, lengths, initial_state, scale, bool(return_state))
    return (o, state) if return_state else o


def linear_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                          state: torch.Tensor, *, scale: Optional[float] = None,
                          state_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token of ``linear_attention`` for every sequence: q (B, H, dk),
    k (B, G, dk), v (B, G, dv); ``state`` (B, H, dk, dv) float32, contiguous,
    is updated in place, or left alone and the new state written to
    ``state_out``.  Returns o (B, H, dv).  Not differentiable: a call that
    needs gradients is refused (use ``linear_attention`` with T = 1)."""
    dims = _attention_dims(q, k, v, log_decay, ("B", "H", "D"))
    B, _, H, _, dk, dv = dims
    dtype, device = q.dtype, q.device
    out_state = state if state_out is None else state_out
    _check_state(state, "state", (B, H, dk, dv), device, contiguous=True)
    if state_out is not None:
        _check_state(out_state, "state_out", (B, H, dk, dv), device, contiguous=True)
    if _grad_needed(q, k, v, log_decay, state, out_state):
        raise RuntimeError("linear_attention_step has no gradient; call it under torch.no_grad(), or use "
                           "linear_attention with T = 1")
    scale = dk ** -0.5 if scale is None else float(scale)
    q, k, v, log_decay = _rows(q), _rows(k), _rows(v), log_decay.contiguous()
    o = _empty((B, H, dv), dtype, device)
    _call("tmpc_linear_attention_step", dtype, device, _DIMS(*dims), _view(q), _view(k), _view(v), _view(o),
          _p(log_decay), _p(state), _p(out_state), scale)
    return o


# ---------------------------------------------------------------------------
# Residual addition and root-mean-square norm
# ---------------------------------------------------------------------------
def _norm_forward(x, residual, weight, eps, want_inv):
    shape, dtype, device = x.shape, x.dtype, x.device
    d = shape[-1]
    x2 = _rows(x if len(shape) == 2 else x.reshape(-1, d))
    y = _empty(shape, dtype, device)
    r2 = s = None
    if residual is not None:
        r2 = _rows(residual if len(shape) == 2 else residual.reshape(-1, d))
        s = _empty(shape, dtype, device)
    rows = x2.shape[0]
    inv = _empty((rows,), torch.float32, device) if want_inv else None
    _call("tmpc_add_rms_norm", dtype, device, rows, d, _p(x2), x2.stride(0), _p(r2), 0 if r2 is None else r2.stride(0),
          _p(weight), eps, _p(y), _p(s), _p(inv))
    return y, s, inv


class _AddRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        ctx.set_materialize_grads(False)
        y, s, inv = _norm_forward(x, residual, weight, eps, True)
        ctx.save_for_backward(x.contiguous() if s is None else s, weight, inv)
        ctx.shape, ctx.has_residual = x.shape, residual is not None
        return y, s

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, ds):
        t, weight, inv = ctx.saved_tensors
        d, rows = t.shape[-1], inv.shape[0]
        if dy is None:
            dy = torch.zeros(ctx.shape, dtype=t.dtype, device=t.device)
        dy = dy.contiguous()
        ds = None if ds is None else ds.contiguous()
        dx, dw = _empty(ctx.shape, t.dtype, t.device), torch.empty_like(weight)
        need = _ffi.load().tmpc_add_rms_norm_workspace_bytes(rows, d)
        ws = _workspace(need, t.device)
        _call("tmpc_add_rms_norm_backward", t.dtype, t.device, rows, d, _p(dy), _p(ds), _p(t), _p(weight), _p(inv),
              _p(dx), _p(dw), _p(ws), need)
        return dx, (dx if ctx.has_residual else None), dw, None


def add_rms_norm(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor,
                 eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """t = x + residual, y = t (mean(t^2) + eps)^(-1/2) weight over the last
    axis (1..16384 elements); returns (y, t).  With ``residual`` None, t = x.
    The norm is taken of t before t is rounded to the tensors' type.
    Differentiable with respect to x, residual and weight."""
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"x must be a tensor, got {type(x).__name__}")
    dtype, device, shape = x.dtype, x.device, x.shape
    _suffix(dtype)
    _check(x, "x", dtype, device)
    if len(shape) < 1 or not 1 <= shape[-1] <= 16384:
        raise ValueError(f"x must have 1..16384 elements on its last axis, got shape {tuple(shape)}")
    if residual is not None:
        _check(residual, "residual", dtype, device)
        if residual.shape != shape:
            raise ValueError(f"residual has shape {tuple(residual.shape)}, expected {tuple(shape)}")
    _check(weight, "weight", dtype, device)
    if weight.shape != shape[-1:]:
        raise ValueError(f"weight has shape {tuple(weight.shape)}, expected ({shape[-1]},)")
    weight = weight.contiguous()
    if _grad_needed(x, residual, weight):
        y, s = _AddRmsNorm.apply(x, residual, weight, float(eps))
    else:
        y, s, _ = _norm_forward(x, residual, weight, float(eps), False)
    return y, (x if s is None else s)


# ---------------------------------------------------------------------------
# Gated linear layer
# ---------------------------------------------------------------------------
def _aligned(t: torch.Tensor) -> torch.Tensor:
    """Contiguous, and at an address the tensor-core kernels' copies can read."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _gated_forward(x2, w_gate, w_up, act):
    rows, d, f = x2.shape[0], x2.shape[1], w_gate.shape[0]
    dtype, device = x2.dtype, x2.device
    h = _empty((rows, f), dtype, device)
    need = _ffi.load().tmpc_gated_linear_workspace_bytes(rows, d, f, x2.element_size())
    ws = _workspace(need, device)
    _call("tmpc_gated_linear", dtype, device, rows, d, f, _p(x2), _p(w_gate), _p(w_up), act, _p(h), _p(ws), need)
    return h


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x2, w_gate, w_up, act):
        ctx.save_for_backward(x2, w_gate, w_up)
        ctx.act = act
        return _gated_forward(x2, w_gate, w_up, act)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        x2, w_gate, w_up = ctx.saved_tensors
        rows, d, f = x2.shape[0], x2.shape[1], w_gate.shape[0]
        dh = dh.contiguous()
        dx = torch.empty_like(x2) if ctx.needs_input_grad[0] else None
        want_w = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        dwg, dwu = (torch.empty_like(w_gate), torch.empty_like(w_up)) if want_w else (None, None)
        need = _ffi.load().tmpc_gated_linear_backward_workspace_bytes(rows, d, f, x2.element_size())
        ws = _workspace(need, x2.device)
        _call("tmpc_gated_linear_backward", x2.dtype, x2.device, rows, d, f, _p(x2), _p(w_gate), _p(w_up), ctx.act,
              _p(dh), _p(dx), _p(dwg), _p(dwu), _p(ws), need)
        return dx, dwg, dwu, None


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, activation: str = "silu") -> torch.Tensor:
    """h = act(x w_gate^T) * (x w_up^T): both projections, the activation and
    the product of a gated feed-forward block.  x (..., d), w_gate and w_up
    (f, d); ``activation`` "silu" or "gelu" (the exact, erf form).  Returns h (..., f).
    Differentiable with respect to x, w_gate and w_up; the projections are
    recomputed in the backward pass, not kept."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"x must be a tensor, got {type(x).__name__}")
    _suffix(x.dtype)
    _check(x, "x", x.dtype, x.device)
    for name, w in (("w_gate", w_gate), ("w_up", w_up)):
        _check(w, name, x.dtype, x.device)
        if w.dim() != 2:
            raise ValueError(f"{name} must be (f, d), got shape {tuple(w.shape)}")
    if x.dim() < 1 or x.shape[-1] < 1 or w_gate.shape[0] < 1 or w_gate.shape != w_up.shape or \
            w_gate.shape[1] != x.shape[-1]:
        raise ValueError(f"shapes of x {tuple(x.shape)}, w_gate {tuple(w_gate.shape)} and w_up {tuple(w_up.shape)} "
                         "do not fit")
    act = ACTIVATIONS[activation]
    x2 = _aligned(x if x.dim() == 2 else x.reshape(-1, x.shape[-1]))
    w_gate, w_up = _aligned(w_gate), _aligned(w_up)
    if _grad_needed(x2, w_gate, w_up):
        h = _GatedLinear.apply(x2, w_gate, w_up, act)
    else:
        h = _gated_forward(x2, w_gate, w_up, act)
    return h if x.dim() == 2 else h.reshape(*x.shape[:-1], w_gate.shape[0])
