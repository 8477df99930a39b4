"""Distillation from a teacher's top logits (noise_distill): the loss of each row and its gradient.

With s = softcap tanh(z / softcap) / temperature (softcap 0: z / temperature), p the softmax of a row's teacher
logits / temperature over its entries and lse = logsumexp(s):
  loss = temperature^2 sum_k p_k (log p_k - s[id_k] + lse)
The fixed model's head has softcap 15 (utils/model.py:204). No call is recorded by autograd; calls run on the
current stream of their tensors' device and keep nothing between calls.
"""
from __future__ import annotations

import torch

from . import _lib
from .attention import DTYPE_CODES, _meta, _pointer, checked, device_index, launch

MAX_ENTRIES = 1024


def _row_stride(t: torch.Tensor):
    """Row stride of a matrix whose columns are contiguous and whose rows do not overlap, else None."""
    rows, cols = t.shape
    if (t.stride(1) != 1 and cols != 1) or (t.stride(0) < cols and rows != 1):
        return None
    return t.stride(0) if rows > 1 else cols


def _matrix(t: torch.Tensor, stride):
    """t, or a contiguous copy where its layout cannot be taken, and its row stride."""
    return (t, stride) if stride is not None else (t.clone(memory_format=torch.contiguous_format), t.shape[1])


def _check(name, logits, ids, teacher, temperature, softcap, dloss, lse, fused):
    if logits.dim() != 2 or ids.dim() != 2 or teacher.shape != ids.shape or len(ids) != len(logits):
        raise ValueError(f'{name}: logits [N, V], ids and teacher [N, K] expected, got {tuple(logits.shape)}, '
                         f'{tuple(ids.shape)} and {tuple(teacher.shape)}')
    if logits.dtype not in DTYPE_CODES or teacher.dtype not in DTYPE_CODES:
        raise ValueError(f'{name}: logits and teacher must be fp32, bf16 or fp16, got {logits.dtype} and {teacher.dtype}')
    if ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f'{name}: ids must be int32 or int64, got {ids.dtype}')
    N, V = logits.shape
    if not 1 <= ids.shape[1] <= MAX_ENTRIES or V < 1 or V > 1 << 30:
        raise ValueError(f'{name}: 1 to {MAX_ENTRIES} entries a row and 1 to 2^30 logits, got {ids.shape[1]} and {V}')
    if not 0 < temperature < float('inf') or not 0 <= softcap < float('inf'):
        raise ValueError(f'{name}: temperature must be positive and softcap not negative, got {temperature} and {softcap}')
    for t, what, dtype in ((dloss, 'dloss', torch.float32), (lse, 'lse', torch.float64)):
        if t is not None and (t.shape != (N,) or t.dtype != dtype):
            raise ValueError(f'{name}: {what} must be {dtype} [{N}], got {t.dtype} {tuple(t.shape)}')
    if fused:
        limit = int(_lib.load().noise_distill_max_vocab(DTYPE_CODES[logits.dtype], int(softcap > 0)))
        if V > limit:
            raise ValueError(f'{name}: loss and gradient in one pass take at most {limit} logits a row of {logits.dtype}, '
                             f'got {V}; use distill_loss and distill_backward')
    return ((DTYPE_CODES[logits.dtype], DTYPE_CODES[teacher.dtype], ids.dtype == torch.int64, V, ids.shape[1]),
            _row_stride(logits), _row_stride(ids), _row_stride(teacher))


def _call(name, logits, ids, teacher, temperature, softcap, dloss=None, lse=None, want_loss=True, want_grad=False):
    temperature, softcap = float(temperature), float(softcap)
    key = (name, _meta(logits), _meta(ids), _meta(teacher), temperature, softcap, _meta(dloss), _meta(lse))
    head, ld, ids_ld, teacher_ld = checked(
        key, lambda: _check(name, logits, ids, teacher, temperature, softcap, dloss, lse, want_loss and want_grad))
    N, V = logits.shape
    device = device_index(name, logits, ids, teacher, dloss, lse)
    where = logits.device
    loss = torch.empty(N, dtype=torch.float32, device=where) if want_loss else None
    out_lse = torch.empty(N, dtype=torch.float64, device=where) if want_loss and not want_grad else None
    grad = torch.empty(N, V, dtype=logits.dtype, device=where) if want_grad else None
    if N:
        (logits, ld), (ids, ids_ld) = _matrix(logits, ld), _matrix(ids, ids_ld)
        teacher, teacher_ld = _matrix(teacher, teacher_ld)
        dloss = None if dloss is None else dloss.contiguous()
        lse = None if lse is None else lse.contiguous()
        a = _lib.DISTILL.pack(*head, temperature, softcap, N, ld, ids_ld, teacher_ld, V, logits.data_ptr(),
                              ids.data_ptr(), teacher.data_ptr(), _pointer(dloss), _pointer(lse), _pointer(loss),
                              _pointer(out_lse), _pointer(grad))
        launch('noise_distill', device, a)
    return loss, out_lse, grad


def distill_loss(logits: torch.Tensor, ids: torch.Tensor, teacher: torch.Tensor, *, temperature: float = 1.0,
                 softcap: float = 0.0):
    """Losses of logits [N, V] against the teacher's entries: ids [N, K] (int32 or int64, K up to 1,024) and their
    logits teacher [N, K]. An id outside [0, V) marks an absent entry, equal ids add up, and a row without an entry
    above -inf has loss 0. Returns (loss fp32 [N], lse fp64 [N]); lse is what distill_backward needs, in 64 bits because
    all of a row's gradient shares its error."""
    return _call('distill_loss', logits, ids, teacher, temperature, softcap)[:2]


def distill_backward(dloss: torch.Tensor, logits: torch.Tensor, ids: torch.Tensor, teacher: torch.Tensor,
                     lse: torch.Tensor, *, temperature: float = 1.0, softcap: float = 0.0) -> torch.Tensor:
    """Gradient [N, V] of sum_n dloss[n] loss[n] with respect to the logits, from distill_loss's inputs and lse."""
    if dloss is None or lse is None:
        raise ValueError('distill_backward: dloss and lse are required')
    return _call('distill_backward', logits, ids, teacher, temperature, softcap, dloss, lse, False, True)[2]


def distill_loss_grad(logits: torch.Tensor, ids: torch.Tensor, teacher: torch.Tensor, *, temperature: float = 1.0,
                      softcap: float = 0.0, dloss: torch.Tensor | None = None):
    """Losses and the gradient of sum_n dloss[n] loss[n] (dloss None: of their sum) in one pass that reads the logits
    once. Returns (loss fp32 [N], grad [N, V] of the logits' type)."""
    loss, _, grad = _call('distill_loss_grad', logits, ids, teacher, temperature, softcap, dloss, None, True, True)
    return loss, grad
