"""Operators on policy logits and legal-move lists, on torch CUDA tensors.

For programs that score or tune a policy next to the engine: log-probabilities
over the legal moves with their backward pass, a clipped policy loss with a KL
term and a preference loss over lines of moves. They read what
``B200Network.evaluate_priors`` reads -- a row of policy logits for each
position (from ``evaluate_device`` or a trainer's own network) and the legal
moves as a CSR list of policy indices -- and the losses return their gradient
with respect to the logits in the same pass, for ``logits.backward(grad)``.

Each function is one call of the C ABI (``include/mfb200.h``, which defines the
formulas and the treatment of empty, masked and malformed rows) on the logits'
device and its current stream; nothing is synchronised or kept, and the calls
can be captured into a CUDA graph. Wrong shapes, types or devices raise
``ValueError``, errors of the library ``RuntimeError``. There is no CPU path.

Common arguments: ``logits`` [batch, classes] float32, bfloat16 or float16,
unit stride along a row; ``move_offsets`` int32 [batch + 1] and ``move_index``
int16 [moves]; ``played`` int32 [batch], the played move's place in its
position's list or -1; ``softmax_temp``. Gradients have the logits' type, or
that of ``grad_logits`` where the caller gives the tensor to write (which may be
other columns of the logits' own buffer).
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from ._lib import lib

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class _Rows(ctypes.Structure):
    _fields_ = [("logits", ctypes.c_void_p), ("logits_stride", ctypes.c_int64),
                ("logits_type", ctypes.c_int32), ("batch", ctypes.c_int32),
                ("classes", ctypes.c_int32), ("move_offsets", ctypes.c_void_p),
                ("move_index", ctypes.c_void_p), ("num_moves", ctypes.c_int64),
                ("played", ctypes.c_void_p), ("softmax_temp", ctypes.c_double)]


class _ClipConfig(ctypes.Structure):
    _fields_ = [("clip_low", ctypes.c_double), ("clip_high", ctypes.c_double),
                ("kl_coef", ctypes.c_float), ("entropy_coef", ctypes.c_float),
                ("scale", ctypes.c_float)]


class _PreferenceConfig(ctypes.Structure):
    _fields_ = [("beta", ctypes.c_float), ("label_smoothing", ctypes.c_float),
                ("scale", ctypes.c_float)]


class MoveLogprobs(NamedTuple):
    moves: torch.Tensor             # [moves] log-probability of each listed move
    played: Optional[torch.Tensor]  # [batch] of the played move (None without `played`)
    entropy: torch.Tensor           # [batch]


class ClippedPolicyLoss(NamedTuple):
    total: torch.Tensor                  # [] sum of `loss`
    loss: torch.Tensor                   # [batch]
    logp: torch.Tensor                   # [batch] of the played move
    kl: Optional[torch.Tensor]           # [batch] (None without reference logits)
    entropy: torch.Tensor                # [batch]
    grad_logits: Optional[torch.Tensor]  # [batch, classes] (None with grad=False)


class PreferenceLoss(NamedTuple):
    total: torch.Tensor                  # [] sum of `loss`
    loss: torch.Tensor                   # [pairs]
    margin: torch.Tensor                 # [pairs]
    line_logp: torch.Tensor              # [2 * pairs]
    logp: torch.Tensor                   # [batch] of the played move
    row_grad: torch.Tensor               # [batch] gradient of the total with respect to logp
    grad_logits: Optional[torch.Tensor]  # [batch, classes] (None with grad=False)


_vp, _int, _i64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64
_native = None


def _lib():
    global _native
    if _native is None:
        L = lib()
        L.mfb200_policy_last_error.restype = ctypes.c_char_p
        L.mfb200_policy_last_error.argtypes = []
        rows = ctypes.POINTER(_Rows)
        L.mfb200_move_logprobs.restype = _int
        L.mfb200_move_logprobs.argtypes = [rows, _vp, _vp, _vp, _vp]
        L.mfb200_move_logprobs_backward.restype = _int
        L.mfb200_move_logprobs_backward.argtypes = [rows, _vp, _vp, _vp, _vp, _i64, _int, _vp]
        L.mfb200_clipped_policy_loss.restype = _int
        L.mfb200_clipped_policy_loss.argtypes = [
            rows, ctypes.POINTER(_ClipConfig), _vp, _vp, _vp, _vp, _i64, _int, _vp, _vp, _vp, _vp,
            _vp, _vp, _i64, _int, _vp]
        L.mfb200_preference_loss.restype = _int
        L.mfb200_preference_loss.argtypes = [
            rows, ctypes.POINTER(_PreferenceConfig), _vp, _int, _vp, _vp, _vp, _vp, _vp, _vp, _vp,
            _vp, _vp, _vp, _i64, _int, _vp]
        _native = L
    return _native


def _vector(t, name, dtype, size, device):
    """Pointer of a contiguous 1-D tensor of the given type and size (None: any)."""
    try:
        if (t.dtype is dtype and t.get_device() == device and t.is_contiguous() and t.dim() == 1
                and (size is None or t.numel() == size)):
            return t.data_ptr()
    except AttributeError:
        pass
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.dim() != 1:
        raise ValueError(f"{name} must be a 1-D {dtype} tensor")
    if t.get_device() != device:
        raise ValueError(f"{name} is on {t.device}, the logits on cuda:{device}")
    if size is not None and t.numel() != size:
        raise ValueError(f"{name} has {t.numel()} entries, expected {size}")
    raise ValueError(f"{name} must be contiguous")


def _matrix(t, name, shape, device):
    """(pointer, row stride, type) of a [batch, classes] tensor."""
    kind = TYPES.get(t.dtype) if isinstance(t, torch.Tensor) else None
    if kind is None or t.dim() != 2:
        raise ValueError(f"{name} must be a 2-D float32, bfloat16 or float16 tensor")
    if t.shape != shape:
        raise ValueError(f"{name} is {tuple(t.shape)}, expected {tuple(shape)}")
    if t.get_device() != device:
        raise ValueError(f"{name} is on {t.device}, the logits on cuda:{device}")
    rows, cols = shape
    stride, unit = t.stride()
    if unit != 1 and cols > 1:
        raise ValueError(f"{name} must have unit stride along a row")
    return t.data_ptr(), stride if rows > 1 else cols, kind


def _rows(logits, move_offsets, move_index, played, softmax_temp):
    """The C struct, the logits' shape and the device's index."""
    kind = TYPES.get(logits.dtype) if isinstance(logits, torch.Tensor) else None
    if kind is None or logits.dim() != 2:
        raise ValueError("logits must be a 2-D float32, bfloat16 or float16 tensor")
    device = logits.get_device()
    if device < 0:
        raise ValueError("logits must be a CUDA tensor: there is no CPU path")
    shape = logits.shape
    batch, classes = shape
    stride, unit = logits.stride()
    if unit != 1 and classes > 1:
        raise ValueError("logits must have unit stride along a row")
    off = _vector(move_offsets, "move_offsets", torch.int32, batch + 1, device)
    index = _vector(move_index, "move_index", torch.int16, None, device)
    at = None if played is None else _vector(played, "played", torch.int32, batch, device)
    return _Rows(logits.data_ptr(), stride if batch > 1 else classes, kind, batch, classes, off,
                 index, move_index.numel(), at, softmax_temp), shape, device


def _gradient(logits, shape, grad, grad_logits, device):
    """(tensor, pointer, row stride, type) of the gradient to write."""
    if grad_logits is None:
        if not grad:
            return None, None, 0, 0
        grad_logits = torch.empty_like(logits)  # contiguous for rows that are padded
        return grad_logits, grad_logits.data_ptr(), shape[1], TYPES[grad_logits.dtype]
    return (grad_logits, *_matrix(grad_logits, "grad_logits", shape, device))


def _call(fn, device, *args):
    """The library call on the logits' device and its current stream."""
    if device == torch.cuda.current_device():
        rc = fn(*args, _stream_of(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _stream_of(device))
    if rc != 0:
        raise RuntimeError(_native.mfb200_policy_last_error().decode())


# torch.cuda.current_stream builds a Stream object (3 us); its raw handle takes 0.1 us
_stream_of = getattr(torch._C, "_cuda_getCurrentRawStream",
                     lambda device: torch.cuda.current_stream(device).cuda_stream)


def move_logprobs(logits, move_offsets, move_index, played=None, *,
                  softmax_temp: float = 1.0) -> MoveLogprobs:
    """Log-probabilities of the legal moves, of the played moves and the
    entropy of each position (``mfb200_move_logprobs``). Entries of ``moves`` that
    no position's list holds (a longer ``move_index``, a malformed list) are not set."""
    L = _lib()
    rows, shape, device = _rows(logits, move_offsets, move_index, played, softmax_temp)
    f = torch.float32
    moves = torch.empty_like(move_index, dtype=f)
    at = None if played is None else torch.empty_like(played, dtype=f)
    entropy = logits.new_empty(shape[0], dtype=f) if at is None else torch.empty_like(at)
    _call(L.mfb200_move_logprobs, device, rows, moves.data_ptr(),
          None if at is None else at.data_ptr(), entropy.data_ptr())
    return MoveLogprobs(moves, at, entropy)


def move_logprobs_backward(logits, move_offsets, move_index, played=None, *, grad_moves=None,
                           grad_played=None, grad_entropy=None, softmax_temp: float = 1.0,
                           grad_logits=None) -> torch.Tensor:
    """Gradient of the logits from the float32 gradients of move_logprobs'
    outputs, each optional (``mfb200_move_logprobs_backward``). With
    ``grad_moves = -target`` this is the gradient of the cross-entropy to a
    distribution over the legal moves, such as the search's visit counts."""
    L = _lib()
    rows, shape, device = _rows(logits, move_offsets, move_index, played, softmax_temp)
    f = torch.float32
    gm = None if grad_moves is None else _vector(grad_moves, "grad_moves", f, move_index.numel(), device)
    gp = None if grad_played is None else _vector(grad_played, "grad_played", f, shape[0], device)
    gh = None if grad_entropy is None else _vector(grad_entropy, "grad_entropy", f, shape[0], device)
    if gp is not None and played is None:
        raise ValueError("grad_played needs played")
    grad, ptr, stride, kind = _gradient(logits, shape, True, grad_logits, device)
    _call(L.mfb200_move_logprobs_backward, device, rows, gm, gp, gh, ptr, stride, kind)
    return grad


def clipped_policy_loss(logits, move_offsets, move_index, played, old_logp, advantage, *,
                        ref_logits=None, weight=None, clip_low: float = 0.2,
                        clip_high: float = 0.2, kl_coef: float = 0.0, entropy_coef: float = 0.0,
                        scale: Optional[float] = None, softmax_temp: float = 1.0,
                        grad: bool = True, grad_logits=None) -> ClippedPolicyLoss:
    """Clipped policy loss with a KL term against ``ref_logits`` and its
    gradient (``mfb200_clipped_policy_loss``). ``old_logp``, ``advantage`` and
    ``weight`` are float32 [batch]; ``scale`` defaults to 1 / batch."""
    L = _lib()
    rows, shape, device = _rows(logits, move_offsets, move_index, played, softmax_temp)
    if played is None:
        raise ValueError("played must be a 1-D torch.int32 tensor")
    n, f = shape[0], torch.float32
    old = _vector(old_logp, "old_logp", f, n, device)
    adv = _vector(advantage, "advantage", f, n, device)
    w = None if weight is None else _vector(weight, "weight", f, n, device)
    ref, ref_stride, ref_kind = ((None, 0, 0) if ref_logits is None
                                 else _matrix(ref_logits, "ref_logits", shape, device))
    g, ptr, stride, kind = _gradient(logits, shape, grad, grad_logits, device)
    cfg = _ClipConfig(clip_low, clip_high, kl_coef, entropy_coef,
                      scale if scale is not None else 1.0 / max(n, 1))
    total = old_logp.new_empty(())
    loss, logp, entropy = (torch.empty_like(old_logp), torch.empty_like(old_logp),
                           torch.empty_like(old_logp))
    kl = None if ref is None else torch.empty_like(old_logp)
    _call(L.mfb200_clipped_policy_loss, device, rows, cfg, old, adv, w, ref, ref_stride, ref_kind,
          loss.data_ptr(), logp.data_ptr(), None if kl is None else kl.data_ptr(),
          entropy.data_ptr(), total.data_ptr(), ptr, stride, kind)
    return ClippedPolicyLoss(total, loss, logp, kl, entropy, g)


def preference_loss(logits, move_offsets, move_index, played, line_offsets, ref_logp, *,
                    beta: float = 0.1, label_smoothing: float = 0.0, weight=None,
                    scale: Optional[float] = None, softmax_temp: float = 1.0, grad: bool = True,
                    grad_logits=None) -> PreferenceLoss:
    """Preference loss over pairs of lines and its gradient
    (``mfb200_preference_loss``). ``line_offsets`` int32 [2 * pairs + 1] into
    the positions: line 2i is the preferred, 2i + 1 the rejected one of pair i.
    ``ref_logp`` float32 [batch] is the reference policy's log-probability of
    each played move, ``weight`` float32 [pairs]; ``scale`` defaults to 1 / pairs."""
    L = _lib()
    rows, shape, device = _rows(logits, move_offsets, move_index, played, softmax_temp)
    if played is None:
        raise ValueError("played must be a 1-D torch.int32 tensor")
    n, f = shape[0], torch.float32
    lines = _vector(line_offsets, "line_offsets", torch.int32, None, device)
    if line_offsets.numel() % 2 != 1:
        raise ValueError("line_offsets must have 2 * pairs + 1 entries")
    pairs = line_offsets.numel() // 2
    ref = _vector(ref_logp, "ref_logp", f, n, device)
    w = None if weight is None else _vector(weight, "weight", f, pairs, device)
    g, ptr, stride, kind = _gradient(logits, shape, grad, grad_logits, device)
    cfg = _PreferenceConfig(beta, label_smoothing, scale if scale is not None else 1.0 / max(pairs, 1))
    total = ref_logp.new_empty(())
    logp, rest, row_grad = (torch.empty_like(ref_logp), torch.empty_like(ref_logp),
                            torch.empty_like(ref_logp))
    loss = ref_logp.new_empty(pairs)
    margin = torch.empty_like(loss)
    line_logp = ref_logp.new_empty(2 * pairs)
    _call(L.mfb200_preference_loss, device, rows, cfg, lines, pairs, ref, w, logp.data_ptr(),
          rest.data_ptr(), row_grad.data_ptr(), line_logp.data_ptr(), margin.data_ptr(), loss.data_ptr(),
          total.data_ptr(), ptr, stride, kind)
    return PreferenceLoss(total, loss, margin, line_logp, logp, row_grad, g)
