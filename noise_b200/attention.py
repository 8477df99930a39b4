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


def check_cuda(name: str, *tensors) -> torch.device:
    """The one CUDA device of the tensors (None entries are skipped)."""
    dev = tensors[0].device
    for t in tensors:
        if t is not None and (t.device != dev or t.device.type != 'cuda'):
            raise ValueError(f'{name}: every tensor must be on one CUDA device, got {t.device} and {dev}')
    return dev


def launch(name: str, dev: torch.device, *args) -> None:
    """One library call on dev's current stream (the last argument of every entry point)."""
    if dev.index == torch.cuda.current_device():
        _lib.call(name, *args, torch.cuda.current_stream(dev).cuda_stream)
    else:
        with torch.cuda.device(dev):
            _lib.call(name, *args, torch.cuda.current_stream(dev).cuda_stream)


def _addressable(t: torch.Tensor, broadcast: bool = False) -> bool:
    """16-byte rows that the kernels can step through: D contiguous, aligned pointer and strides."""
    unit = 16 // t.element_size()
    if t.stride(-1) != 1 and t.shape[-1] != 1:
        return False
    if t.data_ptr() % 16:
        return False
    for n, s in zip(t.shape[:-1], t.stride()[:-1]):
        if n > 1 and (s % unit or s < 0 or (s == 0 and not broadcast)):
            return False
    return True


def _rows(t: torch.Tensor, broadcast: bool = False) -> torch.Tensor:
    return t if _addressable(t, broadcast) else t.clone(memory_format=torch.contiguous_format)


def _strides(t: torch.Tensor):
    """Element strides {batch, token, head}; a dimension of one element is never stepped along."""
    return _lib.Strides3(*(s if n > 1 else 0 for n, s in zip(t.shape[:3], t.stride()[:3])))


# ------------------------------------------------------------------------------------------------
# norms of queries and keys with the rotation
# ------------------------------------------------------------------------------------------------
def _qk_args(q, k, rope, positions, q_weight, k_weight, order, eps) -> _lib.NoiseQkNorm:
    name = 'qk_norm_rope'
    if q.dim() != 4 or k.dim() != 4 or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError(f'{name}: q [B, T, H, D] and k [B, T, Hk, D] expected, got {tuple(q.shape)} and {tuple(k.shape)}')
    if q.dtype not in DTYPE_CODES or k.dtype != q.dtype:
        raise ValueError(f'{name}: q and k must share fp32, bf16 or fp16, got {q.dtype} and {k.dtype}')
    B, T, H, D = q.shape
    if D % 16 or not 16 <= D <= 256 or not H or not k.shape[2]:
        raise ValueError(f'{name}: D must be a multiple of 16 up to 256 and heads at least 1, got {tuple(q.shape)}')
    if order not in ORDERS:
        raise ValueError(f'{name}: order must be one of {sorted(ORDERS)}, got {order!r}')
    if rope.dim() != 2 or rope.shape[1] != D or not len(rope) or rope.dtype != torch.float32 or not rope.is_contiguous() \
            or rope.data_ptr() % 16:
        raise ValueError(f'{name}: rope must be a contiguous fp32 [positions, {D}] table of cos | sin, got '
                         f'{rope.dtype} {tuple(rope.shape)}')
    a = _lib.NoiseQkNorm()
    if positions is None:
        if T > len(rope):
            raise ValueError(f'{name}: {T} tokens but a table of {len(rope)} positions')
    else:
        if positions.dtype != torch.int32 or positions.shape not in ((T,), (B, T)) or \
                (T > 1 and positions.stride(-1) != 1):
            raise ValueError(f'{name}: positions must be int32 [T] or [B, T] with contiguous rows, got {positions.dtype} '
                             f'{tuple(positions.shape)}')
        a.positions = positions.data_ptr()
        a.positions_stride = positions.stride(0) if positions.dim() == 2 and B > 1 else 0
    for w, field in ((q_weight, 'wq'), (k_weight, 'wk')):
        if w is not None:
            if w.dtype != torch.float32 or w.shape != (D,) or not w.is_contiguous():
                raise ValueError(f'{name}: weights must be contiguous fp32 [{D}], got {w.dtype} {tuple(w.shape)}')
            setattr(a, field, w.data_ptr())
    a.dtype, a.order, a.B, a.T, a.H, a.Hk, a.D = DTYPE_CODES[q.dtype], ORDERS[order], B, T, H, k.shape[2], D
    a.eps = eps
    a.rope, a.table = rope.data_ptr(), len(rope)
    return a


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, rope: torch.Tensor, *, positions: torch.Tensor | None = None,
                 q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
                 order: str = 'rotate_norm', eps: float = NORM_EPS, out=None):
    """Per-head RMS norms of q [B, T, H, D] and k [B, T, Hk, D] and their rotation, one launch for both.

    order 'rotate_norm' (utils/model.py:86-88): norm(R x); 'norm_rotate': R norm(x). rope is a table like
    Weights.rope: fp32 [positions, D], cos | sin; positions int32 [T] or [B, T] picks its rows (default: token
    t row t), and a position outside the table gives NaN rows. q_weight, k_weight: fp32 [D] weights of the
    norms. out: (q_out, k_out) to write to, of any addressable layout (a cache's rows, or q and k themselves).
    Returns (q_out, k_out)."""
    a = _qk_args(q, k, rope, positions, q_weight, k_weight, order, eps)
    if out is None:
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    else:
        q_out, k_out = out
        for o, x in ((q_out, q), (k_out, k)):
            if o.shape != x.shape or o.dtype != x.dtype or not _addressable(o):
                raise ValueError('qk_norm_rope: out must have the shapes and type of q and k, 16-byte aligned rows')
    dev = check_cuda('qk_norm_rope', q, k, rope, positions, q_weight, k_weight, q_out, k_out)
    q, k = _rows(q, True), _rows(k, True)
    a.q, a.k, a.q_out, a.k_out = q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr()
    a.q_stride, a.k_stride, a.q_out_stride, a.k_out_stride = _strides(q), _strides(k), _strides(q_out), _strides(k_out)
    launch('noise_qk_norm_rope', dev, _lib.byref(a), 0, None, 0)
    return q_out, k_out


def qk_norm_rope_backward(dq: torch.Tensor, dk: torch.Tensor, q: torch.Tensor, k: torch.Tensor, rope: torch.Tensor, *,
                          positions: torch.Tensor | None = None, q_weight: torch.Tensor | None = None,
                          k_weight: torch.Tensor | None = None, order: str = 'rotate_norm', eps: float = NORM_EPS):
    """Gradients of qk_norm_rope: dq, dk are those of its results, q, k and the rest its inputs. Returns the
    gradients of (q, k, q_weight, k_weight); a weight that was not given has None. The weights' sums run in a
    fixed order."""
    a = _qk_args(q, k, rope, positions, q_weight, k_weight, order, eps)
    for g, x in ((dq, q), (dk, k)):
        if g.shape != x.shape or g.dtype != x.dtype:
            raise ValueError('qk_norm_rope_backward: dq and dk must have the shapes and type of q and k')
    dev = check_cuda('qk_norm_rope_backward', q, k, dq, dk, rope, positions, q_weight, k_weight)
    q, k, dq, dk = _rows(q, True), _rows(k, True), _rows(dq, True), _rows(dk, True)
    gq, gk = (torch.empty(x.shape, dtype=x.dtype, device=dev) for x in (q, k))
    gwq, gwk = (None if w is None else torch.empty_like(w) for w in (q_weight, k_weight))
    a.q, a.k, a.dq, a.dk = q.data_ptr(), k.data_ptr(), dq.data_ptr(), dk.data_ptr()
    a.q_out, a.k_out = gq.data_ptr(), gk.data_ptr()
    a.q_stride, a.k_stride, a.dq_stride, a.dk_stride = _strides(q), _strides(k), _strides(dq), _strides(dk)
    a.q_out_stride, a.k_out_stride = _strides(gq), _strides(gk)
    ws, need = None, 0
    if gwq is not None or gwk is not None:
        need = int(_lib.load().noise_qk_norm_workspace_bytes(q.shape[3]))
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        a.dwq, a.dwk = (None if g is None else g.data_ptr() for g in (gwq, gwk))
    launch('noise_qk_norm_rope', dev, _lib.byref(a), 1, None if ws is None else ws.data_ptr(), need)
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

    def pointer(self, dev) -> int:
        if self.own:
            if torch.cuda.is_current_stream_capturing():
                raise ValueError(f'{self.name}: a captured call needs the caller\'s status word')
            self.word = torch.zeros(1, dtype=torch.int32, device=dev)
        elif self.word.device != dev:
            raise ValueError(f'{self.name}: status is on {self.word.device}, the tensors on {dev}')
        return self.word.data_ptr()

    def finish(self):
        if self.own:
            code = int(self.word.item())
            if code:
                raise _lib.NoiseError(f'{self.name}: device status {_lib.STATUS_NAMES.get(code, code)}')


def _window_args(name, q, k, v, window, sinks, lengths, scale, token) -> _lib.NoiseWindow:
    dims = 3 if token else 4
    if q.dim() != dims or k.dim() != 4 or v.shape != k.shape or q.shape[0] != k.shape[0] or q.shape[-1] != k.shape[-1]:
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
    window = Tk if window is None else int(window)
    if window < 0 or sinks < 0:
        raise ValueError(f'{name}: window and sinks cannot be negative, got {window} and {sinks}')
    scale = D ** -0.5 if scale is None else float(scale)
    if not 0 < scale < float('inf'):
        raise ValueError(f'{name}: scale must be positive, got {scale}')
    a = _lib.NoiseWindow()
    if lengths is not None:
        if lengths.dtype != torch.int32 or lengths.shape != (B,) or (B > 1 and lengths.stride(0) != 1):
            raise ValueError(f'{name}: lengths must be contiguous int32 [{B}], got {lengths.dtype} {tuple(lengths.shape)}')
        a.lengths = lengths.data_ptr()
    a.dtype, a.B, a.Tq, a.Tk, a.H, a.Hk, a.D = DTYPE_CODES[q.dtype], B, Tq, Tk, H, Hk, D
    a.offset, a.window, a.sinks, a.scale = Tk - Tq, min(window, Tk), min(int(sinks), Tk), scale
    return a


def _offset(name, a, offset):
    if offset is not None:
        if not 0 <= offset <= a.Tk - a.Tq:
            raise ValueError(f'{name}: offset must lie in [0, {a.Tk - a.Tq}], got {offset}')
        a.offset = int(offset)


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int | None, sinks: int = 0, *,
                     lengths: torch.Tensor | None = None, offset: int | None = None, scale: float | None = None,
                     status: torch.Tensor | None = None):
    """Causal attention where the query at position p sees keys p - window .. p (utils/model.py:21-25) and the
    first `sinks` keys; window None: every earlier key. q [B, Tq, H, D], k and v [B, Tk, Hk, D] of bf16 or fp16,
    H a multiple of Hk, D a multiple of 8 up to 128; query row i is at position offset + i (default offset
    Tk - Tq: the queries are the last ones). lengths: int32 [B] on the device; tokens of sequence b from lengths[b] on
    are padding, whose keys and values are not used and whose query rows give zeros. A key or value of a
    token that is not padding must be finite: it reaches the 128-query tiles of the queries that see it.
    status: an int32 word that a device wait which ran out sets; without one the call waits for the
    GPU and checks its own. Returns (out [B, Tq, H, D], lse fp32 [B, H, Tq])."""
    name = 'window_attention'
    a = _window_args(name, q, k, v, window, sinks, lengths, scale, False)
    _offset(name, a, offset)
    st = _Status(name, status)
    dev = check_cuda(name, q, k, v, lengths)
    out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    lse = torch.empty(a.B, a.H, a.Tq, dtype=torch.float32, device=dev)
    if not out.numel():
        return out, lse
    q, k, v = _rows(q), _rows(k), _rows(v)
    a.q, a.k, a.v, a.out, a.lse = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr()
    a.q_stride, a.k_stride, a.v_stride = _strides(q), _strides(k), _strides(v)
    launch('noise_window_attention', dev, _lib.byref(a), st.pointer(dev))
    st.finish()
    return out, lse


def window_attention_token(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor,
                           window: int | None, sinks: int = 0, *, scale: float | None = None) -> torch.Tensor:
    """The newest token of each sequence over a cache: q [B, H, D], k and v [B, Tk, Hk, D], lengths int32 [B]. The
    query of sequence b is at position lengths[b] - 1, its own key and value included in the cache, and sees what
    window_attention would show it; only those keys are read. lengths[b] = 0 gives zeros. Returns out [B, H, D]."""
    name = 'window_attention_token'
    if lengths is None:
        raise ValueError(f'{name}: lengths are required')
    a = _window_args(name, q, k, v, window, sinks, lengths, scale, True)
    dev = check_cuda(name, q, k, v, lengths)
    out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    if not out.numel():
        return out
    if not _addressable(q):
        q = q.clone(memory_format=torch.contiguous_format)
    k, v = _rows(k), _rows(v)
    a.q, a.k, a.v, a.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    a.q_stride = _lib.Strides3(q.stride(0) if a.B > 1 else 0, 0, q.stride(1) if a.H > 1 else 0)
    a.k_stride, a.v_stride = _strides(k), _strides(v)
    launch('noise_window_token', dev, _lib.byref(a))
    return out
