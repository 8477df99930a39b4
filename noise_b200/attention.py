"""Attention operators for any lengths, head counts and layouts, with their gradients.

  qk_norm_rope, qk_norm_rope_backward          -> noise_qk_norm_rope (queries and keys in one launch)
  window_attention, window_attention_backward  -> noise_window_attention, noise_window_attention_backward
  window_attention_token                       -> noise_window_token (one new token per sequence over a cache)

The fixed model's own attention (utils/model.py:17-31, 81-97) is order 'rotate_norm', its layer's window and
sinks 0. Tensors are [B, T, heads, D] with D contiguous; views of a packed projection or a cache are taken
as they are, and a layout the kernels cannot address (a misaligned or broadcast one) is copied first. No
call is recorded by autograd: gradients come from the backward calls. Calls run on the current stream of
their tensors' device and keep nothing between calls, so they can be captured into graphs.
"""
from __future__ import annotations

import torch

from . import _lib

DTYPE_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ORDERS = {'rotate_norm': 0, 'norm_rotate': 1}
NORM_EPS = torch.finfo(torch.float32).eps


def device_index(name: str, *tensors) -> int:
    """The one CUDA device of the tensors (None entries are skipped)."""
    index = tensors[0].get_device()
    for t in tensors:
        if t is not None and (t.get_device() != index or index < 0):
            raise ValueError(f'{name}: every tensor must be on one CUDA device, got {t.device} and {tensors[0].device}')
    return index


def launch(name: str, device: int, *args) -> None:
    """One library call on the device's current stream (the last argument of every entry point)."""
    if device != torch.cuda.current_device():
        with torch.cuda.device(device):
            return launch(name, device, *args)
    # the raw handle of torch.cuda.current_stream(device), without building a Stream object
    _lib.call(name, *args, torch._C._cuda_getCurrentRawStream(device))


def _pointer(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


# What the checks of a call gave, by the call's shapes, strides, types and options: a repeated call skips them.
_CHECKED: dict = {}


def checked(key, make):
    found = _CHECKED.get(key)
    if found is None:
        if len(_CHECKED) >= 4096:
            _CHECKED.clear()
        found = _CHECKED[key] = make()
    return found


def _meta(t: torch.Tensor | None):
    return None if t is None else (t.shape, t.stride(), t.dtype)


def _steps(t: torch.Tensor, broadcast: bool):
    """Element strides {batch, token, head} if the kernels can step through t, else None: D contiguous, strides of whole
    16 bytes, no dimension broadcast (unless allowed). A dimension of one element is never stepped along. The
    address must be 16-byte aligned besides."""
    sb, st, sh, sd = t.stride()
    B, T, H, D = t.shape
    if B == 1:
        sb = 0
    if T == 1:
        st = 0
    if H == 1:
        sh = 0
    if (sd != 1 and D != 1) or (sb | st | sh) * t.element_size() & 15:
        return None
    if not broadcast and ((B > 1 and not sb) or (T > 1 and not st) or (H > 1 and not sh)):
        return None
    return sb, st, sh


def _rows(t: torch.Tensor, steps, broadcast: bool = False):
    """t, or a contiguous copy where its layout (steps None) or its address cannot be taken, and its steps."""
    if steps is None or t.data_ptr() & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        steps = _steps(t, broadcast)
    return t, steps


def _like(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t, memory_format=torch.contiguous_format)


# ------------------------------------------------------------------------------------------------
# norms of queries and keys with the rotation
# ------------------------------------------------------------------------------------------------
def _qk_check(q, k, rope, positions, q_weight, k_weight, order):
    """Refuses what noise_qk_norm_rope does not take; (B, T, H, Hk, D, positions' batch stride)."""
    name = 'qk_norm_rope'
    if q.dim() != 4 or k.dim() != 4 or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError(f'{name}: q [B, T, H, D] and k [B, T, Hk, D] expected, got {tuple(q.shape)} and {tuple(k.shape)}')
    if q.dtype not in DTYPE_CODES or k.dtype != q.dtype:
        raise ValueError(f'{name}: q and k must share fp32, bf16 or fp16, got {q.dtype} and {k.dtype}')
    B, T, H, D = q.shape
    Hk = k.shape[2]
    if D % 16 or not 16 <= D <= 256 or not H or not Hk:
        raise ValueError(f'{name}: D must be a multiple of 16 up to 256 and heads at least 1, got {tuple(q.shape)}')
    if order not in ORDERS:
        raise ValueError(f'{name}: order must be one of {sorted(ORDERS)}, got {order!r}')
    if rope.dim() != 2 or rope.shape[1] != D or not len(rope) or rope.dtype != torch.float32 or not rope.is_contiguous():
        raise ValueError(f'{name}: rope must be a contiguous fp32 [positions, {D}] table of cos | sin, got '
                         f'{rope.dtype} {tuple(rope.shape)}')
    stride = 0
    if positions is None:
        if T > len(rope):
            raise ValueError(f'{name}: {T} tokens but a table of {len(rope)} positions')
    else:
        if positions.dtype != torch.int32 or positions.shape not in ((T,), (B, T)) or \
                (T > 1 and positions.stride(-1) != 1):
            raise ValueError(f'{name}: positions must be int32 [T] or [B, T] with contiguous rows, got {positions.dtype} '
                             f'{tuple(positions.shape)}')
        if positions.dim() == 2 and B > 1:
            stride = positions.stride(0)
    for w in (q_weight, k_weight):
        if w is not None and (w.dtype != torch.float32 or w.shape != (D,) or not w.is_contiguous()):
            raise ValueError(f'{name}: weights must be contiguous fp32 [{D}], got {w.dtype} {tuple(w.shape)}')
    return B, T, H, Hk, D, stride


def _qk_plan(q, k, rope, positions, q_weight, k_weight, order, eps, dq=None, dk=None):
    """(leading fields of NoiseQkNorm, table rows, positions' stride, steps of q, of k, of contiguous results, of dq and
    dk, workspace bytes)."""
    eps = float(eps)
    key = ('qk', q.shape, q.stride(), q.dtype, k.shape, k.stride(), k.dtype, rope.shape, rope.stride(), rope.dtype,
           _meta(positions), _meta(q_weight), _meta(k_weight), order, eps, _meta(dq), _meta(dk))

    def make():
        B, T, H, Hk, D, stride = _qk_check(q, k, rope, positions, q_weight, k_weight, order)
        head = (DTYPE_CODES[q.dtype], ORDERS[order], B, T, H, Hk, D, eps)
        grad_steps, need = (None, None), 0
        if dq is not None:
            if dq.shape != q.shape or dk.shape != k.shape or dq.dtype != q.dtype or dk.dtype != q.dtype:
                raise ValueError('qk_norm_rope_backward: dq and dk must have the shapes and type of q and k')
            grad_steps = _steps(dq, True), _steps(dk, True)
            if q_weight is not None or k_weight is not None:
                need = int(_lib.load().noise_qk_norm_workspace_bytes(D))
        return (head, len(rope), stride, _steps(q, True), _steps(k, True),
                (T * H * D, H * D, D, T * Hk * D, Hk * D, D), *grad_steps, need)

    plan = checked(key, make)
    if rope.data_ptr() & 15:
        raise ValueError('qk_norm_rope: rope must be 16-byte aligned')
    return plan


_NO_STEPS = (0, 0, 0, 0, 0, 0)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, rope: torch.Tensor, *, positions: torch.Tensor | None = None,
                 q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
                 order: str = 'rotate_norm', eps: float = NORM_EPS, out=None):
    """Per-head RMS norms of q [B, T, H, D] and k [B, T, Hk, D] and their rotation, one launch for both.

    order 'rotate_norm' (utils/model.py:86-88): norm(R x); 'norm_rotate': R norm(x). rope is a table like
    Weights.rope: fp32 [positions, D], cos | sin; positions int32 [T] or [B, T] picks its rows (default: token
    t row t), and a position outside the table gives NaN rows. q_weight, k_weight: fp32 [D] weights of the
    norms. out: (q_out, k_out) to write to, of any addressable layout (a cache's rows, or q and k themselves); one that
    overlaps anything else the call reads, the other or itself is refused. Returns (q_out, k_out)."""
    head, table, stride, qs, ks, out_steps, *_ = _qk_plan(q, k, rope, positions, q_weight, k_weight, order, eps)
    if out is None:
        q_out, k_out = _like(q), _like(k)
    else:
        q_out, k_out = out
        q_step, k_step = (_steps(t, False) if t.dim() == 4 else None for t in out)
        if q_out.shape != q.shape or k_out.shape != k.shape or q_out.dtype != q.dtype or k_out.dtype != q.dtype or \
                q_step is None or k_step is None or (q_out.data_ptr() | k_out.data_ptr()) & 15:
            raise ValueError('qk_norm_rope: out must have the shapes and type of q and k, 16-byte aligned rows')
        out_steps = q_step + k_step
    device = device_index('qk_norm_rope', q, k, rope, positions, q_weight, k_weight, q_out, k_out)
    (q, qs), (k, ks) = _rows(q, qs, True), _rows(k, ks, True)
    a = _lib.QK_NORM.pack(*head, rope.data_ptr(), table, _pointer(positions), stride, _pointer(q_weight),
                          _pointer(k_weight), q.data_ptr(), k.data_ptr(), 0, 0, q_out.data_ptr(), k_out.data_ptr(), *qs, *ks,
                          *_NO_STEPS, *out_steps, 0, 0)
    if out is not None and _lib.load().noise_qk_norm_overlap(a, 0):
        raise ValueError('qk_norm_rope: out overlaps an input other than in place, or itself')
    launch('noise_qk_norm_rope', device, a, 0, None, 0)
    return q_out, k_out


def qk_norm_rope_backward(dq: torch.Tensor, dk: torch.Tensor, q: torch.Tensor, k: torch.Tensor, rope: torch.Tensor, *,
                          positions: torch.Tensor | None = None, q_weight: torch.Tensor | None = None,
                          k_weight: torch.Tensor | None = None, order: str = 'rotate_norm', eps: float = NORM_EPS):
    """Gradients of qk_norm_rope: dq, dk are those of its results, q, k and the rest its inputs. Returns the
    gradients of (q, k, q_weight, k_weight); a weight that was not given has None. The weights' sums run in a
    fixed order."""
    head, table, stride, qs, ks, out_steps, dqs, dks, need = _qk_plan(q, k, rope, positions, q_weight, k_weight, order, eps,
                                                                      dq, dk)
    device = device_index('qk_norm_rope_backward', q, k, dq, dk, rope, positions, q_weight, k_weight)
    (q, qs), (k, ks) = _rows(q, qs, True), _rows(k, ks, True)
    (dq, dqs), (dk, dks) = _rows(dq, dqs, True), _rows(dk, dks, True)
    gq, gk = _like(q), _like(k)
    gwq = None if q_weight is None else torch.empty_like(q_weight)
    gwk = None if k_weight is None else torch.empty_like(k_weight)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    a = _lib.QK_NORM.pack(*head, rope.data_ptr(), table, _pointer(positions), stride, _pointer(q_weight),
                          _pointer(k_weight), q.data_ptr(), k.data_ptr(), dq.data_ptr(), dk.data_ptr(), gq.data_ptr(),
                          gk.data_ptr(), *qs, *ks, *dqs, *dks, *out_steps, _pointer(gwq), _pointer(gwk))
    launch('noise_qk_norm_rope', device, a, 1, _pointer(ws), need)
    return gq, gk, gwq, gwk


# ------------------------------------------------------------------------------------------------
# sliding-window attention with sinks
# ------------------------------------------------------------------------------------------------
class _Status:
    """The device status word of a call with bounded waits: the caller's, unread, or one of this call's own
    that is checked before it returns (which waits for the GPU)."""

    def __init__(self, name: str, status: torch.Tensor | None):
        if status is not None and (status.dtype != torch.int32 or status.numel() < 1):
            raise ValueError(f'{name}: status must be an int32 word')
        self.name, self.word, self.own = name, status, status is None

    def pointer(self, device: int) -> int:
        if self.own:
            if torch.cuda.is_current_stream_capturing():
                raise ValueError(f'{self.name}: a captured call needs the caller\'s status word')
            self.word = torch.zeros(1, dtype=torch.int32, device=device)
        elif self.word.get_device() != device:
            raise ValueError(f'{self.name}: status is on {self.word.device}, the tensors on cuda:{device}')
        return self.word.data_ptr()

    def finish(self):
        if self.own:
            code = int(self.word.item())
            if code:
                raise _lib.NoiseError(f'{self.name}: device status {_lib.STATUS_NAMES.get(code, code)}')


def _window_check(name, q, k, v, window, sinks, lengths, offset, scale, token):
    """Refuses what the kernels do not take; the leading fields of NoiseWindow up to `scale`."""
    if q.dim() != (3 if token else 4) or k.dim() != 4 or v.shape != k.shape or q.shape[0] != k.shape[0] or \
            q.shape[-1] != k.shape[3]:
        raise ValueError(f'{name}: q {"[B, H, D]" if token else "[B, Tq, H, D]"} and k, v [B, Tk, Hk, D] expected, got '
                         f'{tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}')
    if q.dtype not in (torch.bfloat16, torch.float16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f'{name}: q, k and v must share bf16 or fp16, got {q.dtype}, {k.dtype} and {v.dtype}')
    B, Tk, Hk, D = k.shape
    H, Tq = q.shape[-2], 1 if token else q.shape[1]
    if D % 8 or not 8 <= D <= 128:
        raise ValueError(f'{name}: D must be a multiple of 8 up to 128, got {D}')
    if not Hk or not H or H % Hk:
        raise ValueError(f'{name}: {H} query heads do not share {Hk} key heads evenly')
    if Tk < 1 or Tq > Tk or Tk > 1 << 30:
        raise ValueError(f'{name}: {Tq} queries need 1 to 2^30 keys, at least as many, got {Tk}')
    if B > 65535 or H > 65535:
        raise ValueError(f'{name}: at most 65,535 sequences and heads a call')
    window, sinks = Tk if window is None else min(window, Tk), min(sinks, Tk)
    if window < 0 or sinks < 0:
        raise ValueError(f'{name}: window and sinks cannot be negative, got {window} and {sinks}')
    scale = D ** -0.5 if scale is None else scale
    if not 2.0 ** -100 <= scale <= 2.0 ** 100:
        raise ValueError(f'{name}: scale must lie in [2^-100, 2^100], got {scale}')
    if lengths is not None and (lengths.dtype != torch.int32 or lengths.shape != (B,) or
                                (B > 1 and lengths.stride(0) != 1)):
        raise ValueError(f'{name}: lengths must be contiguous int32 [{B}], got {lengths.dtype} {tuple(lengths.shape)}')
    if offset is None:
        offset = Tk - Tq
    elif not 0 <= offset <= Tk - Tq:
        raise ValueError(f'{name}: offset must lie in [0, {Tk - Tq}], got {offset}')
    return DTYPE_CODES[q.dtype], B, Tq, Tk, H, Hk, D, offset, window, sinks, scale


def _window_plan(name, q, k, v, window, sinks, lengths, offset, scale, token, dout=None, out=None, lse=None):
    """(leading fields of NoiseWindow, steps of q, k, v, of dout)."""
    window, offset = (n if n is None else int(n) for n in (window, offset))
    sinks, scale = int(sinks), scale if scale is None else float(scale)
    key = (name, q.shape, q.stride(), q.dtype, k.shape, k.stride(), k.dtype, v.shape, v.stride(), v.dtype, _meta(lengths),
           window, sinks, offset, scale, _meta(dout), _meta(out), _meta(lse))

    def make():
        head = _window_check(name, q, k, v, window, sinks, lengths, offset, scale, token)
        if dout is not None:
            if q.dtype != torch.bfloat16:
                raise ValueError(f'{name}: bf16 only, got {q.dtype}')
            if dout.shape != q.shape or out.shape != q.shape or dout.dtype != q.dtype or out.dtype != q.dtype:
                raise ValueError(f'{name}: dout and out must have the shape and type of q')
            if lse.shape != (head[1], head[4], head[2]) or lse.dtype != torch.float32:
                raise ValueError(f'{name}: lse must be fp32 [B, H, Tq], got {lse.dtype} {tuple(lse.shape)}')
        return (head, _steps(q.unsqueeze(1) if token else q, False), _steps(k, False), _steps(v, False),
                None if dout is None else _steps(dout, False))

    return checked(key, make)


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int | None, sinks: int = 0, *,
                     lengths: torch.Tensor | None = None, offset: int | None = None, scale: float | None = None,
                     status: torch.Tensor | None = None):
    """Causal attention where the query at position p sees keys p - window .. p (utils/model.py:21-25) and the
    first `sinks` keys; window None: every earlier key. q [B, Tq, H, D], k and v [B, Tk, Hk, D] of bf16 or fp16,
    H a multiple of Hk, D a multiple of 8 up to 128; query row i is at position offset + i (default offset
    Tk - Tq: the queries are the last ones). lengths: int32 [B] on the device; tokens of sequence b from lengths[b] on
    are padding, whose keys and values are not used and whose query rows give zeros. Keys and values behind the last
    query (the free rows of a cache) are not used either. A key or value of another token must be finite: it reaches the
    128-query tiles of the queries that see it.
    status: an int32 word that a device wait which ran out sets; without one the call waits for the
    GPU and checks its own. Returns (out [B, Tq, H, D], lse fp32 [B, H, Tq])."""
    name = 'window_attention'
    head, qs, ks, vs, _ = _window_plan(name, q, k, v, window, sinks, lengths, offset, scale, False)
    st = _Status(name, status)
    device = device_index(name, q, k, v, lengths)
    out = _like(q)
    lse = torch.empty((head[1], head[4], head[2]), dtype=torch.float32, device=q.device)
    if not out.numel():
        return out, lse
    (q, qs), (k, ks), (v, vs) = _rows(q, qs), _rows(k, ks), _rows(v, vs)
    a = _lib.WINDOW.pack(*head, _pointer(lengths), q.data_ptr(), k.data_ptr(), v.data_ptr(), *qs, *ks, *vs,
                         out.data_ptr(), lse.data_ptr())
    launch('noise_window_attention', device, a, st.pointer(device))
    st.finish()
    return out, lse


def window_attention_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                              lse: torch.Tensor, window: int | None, sinks: int = 0, *,
                              lengths: torch.Tensor | None = None, offset: int | None = None,
                              scale: float | None = None, status: torch.Tensor | None = None):
    """Gradients of window_attention (bf16): dout is out's, and out, lse are what it returned for the same
    arguments. Padding rows get zeros. Sums run in a fixed order. Returns (dq, dk, dv)."""
    name = 'window_attention_backward'
    head, qs, ks, vs, gs = _window_plan(name, q, k, v, window, sinks, lengths, offset, scale, False, dout, out, lse)
    st = _Status(name, status)
    device = device_index(name, q, k, v, dout, out, lse, lengths)
    if not q.numel():
        return torch.empty_like(q), torch.zeros_like(k), torch.zeros_like(v)
    dq, dk, dv = _like(q), _like(k), _like(v)
    (q, qs), (k, ks), (v, vs), (dout, gs) = _rows(q, qs), _rows(k, ks), _rows(v, vs), _rows(dout, gs)
    out, lse = out.contiguous(), lse.contiguous()
    if out.data_ptr() & 15:
        out = out.clone()
    a = _lib.WINDOW.pack(*head, _pointer(lengths), q.data_ptr(), k.data_ptr(), v.data_ptr(), *qs, *ks, *vs,
                         out.data_ptr(), lse.data_ptr())
    need = _lib.load().noise_window_backward_workspace_bytes(a)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device)
    launch('noise_window_attention_backward', device, a, dout.data_ptr(), _lib.STEPS.pack(*gs), dq.data_ptr(),
           dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), need, st.pointer(device))
    st.finish()
    return dq, dk, dv


def window_attention_token(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor,
                           window: int | None, sinks: int = 0, *, scale: float | None = None, with_lse: bool = False):
    """The newest token of each sequence over a cache: q [B, H, D], k and v [B, Tk, Hk, D], lengths int32 [B]. The
    query of sequence b is at position lengths[b] - 1, its own key and value included in the cache, and sees what
    window_attention would show it; only those keys are read. lengths[b] = 0 gives zeros (lse -inf). Returns out [B, H, D],
    with with_lse (out, lse fp32 [B, H])."""
    name = 'window_attention_token'
    if lengths is None:
        raise ValueError(f'{name}: lengths are required')
    head, qs, ks, vs, _ = _window_plan(name, q, k, v, window, sinks, lengths, None, scale, True)
    device = device_index(name, q, k, v, lengths)
    out = _like(q)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device) if with_lse else None
    if not out.numel():
        return (out, lse) if with_lse else out
    if qs is None or q.data_ptr() & 15:
        q, qs = q.clone(memory_format=torch.contiguous_format), (q.shape[1] * q.shape[2], 0, q.shape[2])
    (k, ks), (v, vs) = _rows(k, ks), _rows(v, vs)
    a = _lib.WINDOW.pack(*head, lengths.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), *qs, *ks, *vs,
                         out.data_ptr(), _pointer(lse))
    launch('noise_window_token', device, a)
    return (out, lse) if with_lse else out
