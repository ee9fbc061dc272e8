"""Operators of the training step around the memory layer, over the C ABI.

``layer_norm`` / ``layer_norm_backward`` cover the LayerNorm of the model's
blocks with the residual add before it (memory_pool_model/model.py:87,96,124),
``linear_cross_entropy`` / ``linear_cross_entropy_backward`` the integer-label
cross entropy of the tied logits (model.py:125 under the trainer's loss)
without the ``[tokens, vocab]`` logits, ``orthogonalize`` an update for the
Dense kernels (the value table has its row-wise Adagrad in ``sparse``).  Like
``MemoryLayer.backward`` they are explicit functions, not autograd nodes.

Activations are float32, float16 or bfloat16 CUDA tensors and results have
their type; parameters of the norm, losses and statistics are float32.  Input
rows may be strided (a slice of a wider tensor); other layouts are copied.
The kernels run on the tensors' device, on ``stream`` or that device's
current stream.  With ``check=True`` a call waits for its kernels and raises
where they recorded a failure.

The usual calls -- contiguous tensors of the current device, its current
stream, no check -- go through an extension module (``csrc/fast_calls.cpp``)
that answers None to all others; those, and every error, take the general way
over ctypes here.
"""

from __future__ import annotations

import ctypes as C
import functools
from typing import Dict, Optional, Sequence, Tuple

import torch

from . import _lib as L
from .memory import _DTYPES, _workspace

def _usable(module):
    """The extension module if it was built for this torch (another's layouts differ), else None."""
    return module if getattr(module, "torch_version", None) == torch.__version__ else None


try:
    from . import _fast
except ImportError:          # not built for this interpreter: every call takes the general way
    _fast = None
_fast = _usable(_fast)


def _on_tensor_device(fn):
    """Runs ``fn`` (first argument: a CUDA tensor) with that tensor's device
    current and its ``stream`` keyword as the current stream, so that kernels
    launch and temporaries are allocated there."""
    @functools.wraps(fn)
    def wrapped(first, *args, stream: Optional[torch.cuda.Stream] = None, **kw):
        if not isinstance(first, torch.Tensor) or not first.is_cuda:
            raise TypeError(f"{fn.__name__[1:]}: the first argument must be a CUDA tensor (no CPU path)")
        if stream is None and first.get_device() == torch._C._cuda_getDevice():
            return fn(first, *args, **kw)
        if stream is None:
            with torch.cuda.device(first.device):
                return fn(first, *args, **kw)
        if stream.device != first.device:
            raise ValueError("stream belongs to another device than the tensors")
        with torch.cuda.stream(stream):
            return fn(first, *args, **kw)
    return wrapped


def _stream(t: torch.Tensor) -> int:
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def _call(entry: str, *args) -> None:
    # ctypes takes a structure by reference where the signature has a pointer
    status = getattr(L.lib(), entry)(*args)
    if status:
        raise L.MemlayerError(status, entry)


def _like(t: torch.Tensor, name: str, like: torch.Tensor) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor (no CPU path)")
    if t.device != like.device or t.dtype != like.dtype:
        raise TypeError(f"{name} must have the device and type of the first tensor")
    if t.shape != like.shape:
        raise ValueError(f"{name} must have shape {tuple(like.shape)}")
    return t


def _rows(t: torch.Tensor, d: int) -> Tuple[torch.Tensor, int]:
    """``t`` with rows of ``d`` entries that a stride apart describes, and that stride."""
    if t.is_contiguous():
        return t, d
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= d:
        return t, t.stride(0)
    return t.contiguous(), d


def _vector(t: torch.Tensor, name: str, n: int, like: torch.Tensor) -> torch.Tensor:
    """A float32 vector of ``n`` entries on the device of ``like``."""
    if not isinstance(t, torch.Tensor) or t.device != like.device:
        raise TypeError(f"{name} must be a CUDA tensor on the device of the first tensor")
    if t.numel() != n:
        raise ValueError(f"{name} must have {n} entries")
    if t.dtype is not torch.float32:
        t = t.to(torch.float32)
    return t if t.is_contiguous() else t.contiguous()


def _dtype(t: torch.Tensor) -> int:
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise TypeError(f"{t.dtype} is not supported (float32, float16 or bfloat16)") from None


def _check_status(ws: torch.Tensor, stream: int) -> None:
    code = C.c_int32(0)
    _call("memlayer_train_status", ws.data_ptr(), code, stream)
    if code.value:
        raise L.DeviceError(f"device status {code.value}: {L.DEVICE_ERRORS.get(code.value, 'unknown')}")


def layer_norm(x: torch.Tensor, scale: torch.Tensor, bias: torch.Tensor, *,
               residual: Optional[torch.Tensor] = None, eps: float = 1e-6,
               stream: Optional[torch.cuda.Stream] = None):
    """LayerNorm over the last dimension of ``x [..., d]`` (flax's epsilon by
    default): ``y = (x - mean) / sqrt(var + eps) * scale + bias``.  With
    ``residual`` the norm reads ``x + residual`` (rounded to the type of
    ``x``) and ``(y, x + residual)`` is returned, the second being what
    ``layer_norm_backward`` takes as its input."""
    if _fast is not None and stream is None:
        out = _fast.layer_norm(x, scale, bias, residual, eps)
        if out is not None:
            return out
    return _layer_norm(x, scale, bias, residual, eps, stream=stream)


@_on_tensor_device
def _layer_norm(x, scale, bias, residual, eps):
    code = _dtype(x)
    if x.dim() == 0:
        raise ValueError("x must have at least one dimension")
    d = x.shape[-1]
    xr, ldx = _rows(x, d)
    sc, bi = _vector(scale, "scale", d, x), _vector(bias, "bias", d, x)
    y = torch.empty_like(xr, memory_format=torch.contiguous_format)
    cfg = L.MemlayerNormConfig(x.numel() // d if d else 0, d, code, eps)
    if residual is None:
        a = L.MemlayerNormArgs(xr.data_ptr(), ldx, None, 0, sc.data_ptr(), bi.data_ptr(), y.data_ptr(), None)
        _call("memlayer_layer_norm", cfg, a, _stream(x))
        return y
    rr, ldr = _rows(_like(residual, "residual", x), d)
    total = torch.empty_like(y)
    a = L.MemlayerNormArgs(xr.data_ptr(), ldx, rr.data_ptr(), ldr, sc.data_ptr(), bi.data_ptr(), y.data_ptr(),
                           total.data_ptr())
    _call("memlayer_layer_norm", cfg, a, _stream(x))
    return y, total


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, scale: torch.Tensor, *,
                        dresidual: Optional[torch.Tensor] = None, eps: float = 1e-6, check: bool = False,
                        stream: Optional[torch.cuda.Stream] = None,
                        ) -> Tuple[torch.Tensor, Dict[str, torch.Tensor]]:
    """Gradients of ``sum(dy * layer_norm(x, scale, bias))``: ``(dx, {"scale",
    "bias"})``.  ``x`` is the forward's normalised input (its sum when it had
    a residual; ``dx`` is then the gradient of both summands).  ``dresidual``,
    the gradient that reaches ``x`` beside the norm, is added to ``dx``."""
    if _fast is not None and stream is None and not check:
        out = _fast.layer_norm_backward(dy, x, scale, dresidual, eps)
        if out is not None:
            return out[0], {"scale": out[1], "bias": out[2]}
    return _layer_norm_backward(dy, x, scale, dresidual, eps, check, stream=stream)


@_on_tensor_device
def _layer_norm_backward(dy, x, scale, dresidual, eps, check):
    code = _dtype(dy)
    if dy.dim() == 0:
        raise ValueError("dy must have at least one dimension")
    d = dy.shape[-1]
    g, ldg = _rows(dy, d)
    xr, ldx = _rows(_like(x, "x", dy), d)
    rr, ldr = (None, 0) if dresidual is None else _rows(_like(dresidual, "dresidual", dy), d)
    sc = _vector(scale, "scale", d, dy)
    dx = torch.empty_like(g, memory_format=torch.contiguous_format)
    ds, db = sc.new_empty(d), sc.new_empty(d)
    cfg = L.MemlayerNormConfig(dy.numel() // d if d else 0, d, code, eps)
    nb = C.c_size_t()
    _call("memlayer_layer_norm_backward_workspace_size", cfg, nb)
    ws = _workspace(nb.value, dy.device)
    a = L.MemlayerNormGrads(g.data_ptr(), ldg, xr.data_ptr(), ldx, None if rr is None else rr.data_ptr(), ldr,
                            sc.data_ptr(), dx.data_ptr(), ds.data_ptr(), db.data_ptr())
    s = _stream(dy)
    _call("memlayer_layer_norm_backward", cfg, a, ws.data_ptr(), nb.value, s)
    if check:
        _check_status(ws, s)
    return dx, {"scale": ds, "bias": db}


def _targets(targets: torch.Tensor, ignore_index: int) -> torch.Tensor:
    """``targets`` as int32; an id that 32 bits cannot hold stays out of range and is not the ignored one."""
    t = targets.dtype
    if t is torch.int32:
        return targets
    if t in (torch.uint8, torch.int8, torch.int16, torch.uint16):
        # as they are: compared in their own type with 32-bit limits, every id would be out of range
        return targets.to(torch.int32)
    if t not in (torch.int64, torch.uint32):
        raise ValueError(f"targets must be integers of at most 32 bits or int64, not {t}")
    targets = targets.to(torch.int64)
    bad = -1 if ignore_index != -1 else -2
    return torch.where((targets >= -2 ** 31) & (targets < 2 ** 31), targets, bad).to(torch.int32)


def _loss_args(h, weight, targets, ignore_index):
    code = _dtype(h)
    if not isinstance(weight, torch.Tensor) or weight.device != h.device or weight.dtype != h.dtype:
        raise TypeError("weight must be a CUDA tensor with the device and type of h")
    if h.dim() == 0 or weight.dim() != 2 or weight.shape[1] != h.shape[-1]:
        raise ValueError("h must be [..., d] and weight [vocab, d]")
    if not isinstance(targets, torch.Tensor) or targets.device != h.device:
        raise TypeError("targets must be a tensor on the device of h")
    if targets.shape != h.shape[:-1]:
        raise ValueError(f"targets must have shape {tuple(h.shape[:-1])}")
    if not -2 ** 31 <= ignore_index < 2 ** 31:
        raise ValueError("ignore_index must fit 32 bits")
    V, d = weight.shape
    targets = _targets(targets, ignore_index)
    t = targets.contiguous()
    hr, ldh = _rows(h, d)
    wr, ldw = _rows(weight, d)
    cfg = L.MemlayerLossConfig(t.numel(), d, V, code, ignore_index)
    return cfg, hr, ldh, wr, ldw, t


def _loss_workspace(cfg, backward: int, device):
    nb = C.c_size_t()
    _call("memlayer_cross_entropy_workspace_size", cfg, backward, nb)
    return _workspace(nb.value, device), nb.value


def linear_cross_entropy(h: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *, ignore_index: int = -100,
                         check: bool = False, stream: Optional[torch.cuda.Stream] = None,
                         ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Softmax cross entropy of the logits ``h @ weight.T`` against integer
    ``targets``, without storing them: ``(loss, lse)``, float32 of the shape
    of ``targets`` (any integer type but uint64), ``lse`` being log sum exp of
    the logits.  A token whose target is ``ignore_index`` has loss 0; any
    other target outside the vocabulary gives NaN, and raises with
    ``check=True``."""
    if _fast is not None and stream is None and not check:
        out = _fast.linear_cross_entropy(h, weight, targets, ignore_index)
        if out is not None:
            return out
    return _linear_cross_entropy(h, weight, targets, ignore_index, check, stream=stream)


@_on_tensor_device
def _linear_cross_entropy(h, weight, targets, ignore_index, check):
    cfg, hr, ldh, wr, ldw, t = _loss_args(h, weight, targets, ignore_index)
    loss = torch.empty(t.shape, dtype=torch.float32, device=h.device)
    lse = torch.empty_like(loss)
    ws, nb = _loss_workspace(cfg, 0, h.device)
    a = L.MemlayerLossArgs(hr.data_ptr(), ldh, wr.data_ptr(), ldw, t.data_ptr(), loss.data_ptr(), lse.data_ptr())
    s = _stream(h)
    _call("memlayer_cross_entropy", cfg, a, ws.data_ptr(), nb, s)
    if check:
        _check_status(ws, s)
    return loss, lse


def linear_cross_entropy_backward(h: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, lse: torch.Tensor,
                                  dloss: torch.Tensor, *, dlse: Optional[torch.Tensor] = None,
                                  ignore_index: int = -100, check: bool = False,
                                  stream: Optional[torch.cuda.Stream] = None,
                                  ) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(dh, dweight)`` of ``sum(dloss * loss) + sum(dlse * lse)`` for the
    forward on the same ``h``, ``weight`` and ``targets`` that gave ``lse``
    (a mean over n tokens: ``dloss`` filled with 1 / n).  ``dloss`` is not
    read at ignored tokens, and ``h`` may hold anything there unless ``dlse``
    gives them a gradient.  Above 128 tokens of a 16-bit type the logits'
    gradient is rounded once to that type before it is multiplied with
    ``weight`` and ``h``."""
    if _fast is not None and stream is None and not check:
        out = _fast.linear_cross_entropy_backward(h, weight, targets, lse, dloss, dlse, ignore_index)
        if out is not None:
            return out
    return _linear_cross_entropy_backward(h, weight, targets, lse, dloss, dlse, ignore_index, check, stream=stream)


@_on_tensor_device
def _linear_cross_entropy_backward(h, weight, targets, lse, dloss, dlse, ignore_index, check):
    cfg, hr, ldh, wr, ldw, t = _loss_args(h, weight, targets, ignore_index)
    n = t.numel()
    ls, dl = _vector(lse, "lse", n, h), _vector(dloss, "dloss", n, h)
    de = None if dlse is None else _vector(dlse, "dlse", n, h)
    dh = torch.empty_like(hr, memory_format=torch.contiguous_format)
    dw = torch.empty_like(wr, memory_format=torch.contiguous_format)
    ws, nb = _loss_workspace(cfg, 1, h.device)
    a = L.MemlayerLossArgs(hr.data_ptr(), ldh, wr.data_ptr(), ldw, t.data_ptr(), None, None)
    g = L.MemlayerLossGrads(ls.data_ptr(), dl.data_ptr(), None if de is None else de.data_ptr(), dh.data_ptr(),
                            dw.data_ptr())
    s = _stream(h)
    _call("memlayer_cross_entropy_backward", cfg, a, g, ws.data_ptr(), nb, s)
    if check:
        _check_status(ws, s)
    return dh, dw


def orthogonalize(update: torch.Tensor, *, steps: int = 5,
                  coefficients: Sequence[float] = (3.4445, -4.7750, 2.0315), eps: float = 1e-7,
                  check: bool = False, stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """Newton-Schulz orthogonalisation of the matrices ``update [..., m, n]``
    (gradients or momenta of Dense kernels): ``X = U / (|U|_F + eps)``, then
    ``steps`` times ``X <- (a I + b X X^T + c (X X^T)^2) X``, which brings
    every singular value near 1.  Returns a tensor like ``update``; the caller
    scales and subtracts it.  Products run on 22-bit operands whatever the
    type; coefficients whose iteration would leave their range are refused."""
    if _fast is not None and stream is None and not check:
        out = _fast.orthogonalize(update, steps, *coefficients, eps)
        if out is not None:
            return out
    return _orthogonalize(update, steps, coefficients, eps, check, stream=stream)


@_on_tensor_device
def _orthogonalize(update, steps, coefficients, eps, check):
    code = _dtype(update)
    if update.dim() < 2:
        raise ValueError("update must be [..., m, n]")
    a, b, c = coefficients
    m, n = update.shape[-2:]
    u = update.contiguous()
    out = torch.empty_like(u)
    cfg = L.MemlayerOrthConfig(u.numel() // (m * n) if m * n else 0, m, n, code, steps, a, b, c, eps)
    nb = C.c_size_t()
    _call("memlayer_orthogonalize_workspace_size", cfg, nb)
    ws = _workspace(nb.value, u.device)
    s = _stream(u)
    _call("memlayer_orthogonalize", cfg, u.data_ptr(), out.data_ptr(), ws.data_ptr(), nb.value, s)
    if check:
        _check_status(ws, s)
    return out
