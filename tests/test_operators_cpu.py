"""What the attention operators and the distillation loss refuse, and their argument blocks, without a GPU: the
Python checks run before any device is asked for, and the C entries answer with a status before any CUDA call."""
import ctypes
import shutil
import struct
import subprocess

import pytest
import torch

from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]
BF = torch.bfloat16


def z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


ROPE = torch.zeros(16, 64)


@pytest.mark.parametrize('args,kw,match', [
    ((z(2, 3, 4, 64), z(2, 3, 2, 32), ROPE), {}, 'expected'),
    ((z(2, 3, 4, 64), z(2, 4, 2, 64), ROPE), {}, 'expected'),
    ((z(3, 4, 64), z(3, 2, 64), ROPE), {}, 'expected'),
    ((z(2, 3, 4, 64), z(2, 3, 2, 64, dtype=torch.float16), ROPE), {}, 'share'),
    ((z(2, 3, 4, 64, dtype=torch.float64), z(2, 3, 2, 64, dtype=torch.float64), ROPE), {}, 'share'),
    ((z(2, 3, 4, 40), z(2, 3, 2, 40), torch.zeros(16, 40)), {}, 'multiple of 16'),
    ((z(2, 3, 4, 272), z(2, 3, 2, 272), torch.zeros(16, 272)), {}, 'multiple of 16'),
    ((z(2, 3, 0, 64), z(2, 3, 2, 64), ROPE), {}, 'heads at least 1'),
    ((z(2, 3, 4, 64), z(2, 3, 2, 64), ROPE.double()), {}, 'table'),
    ((z(2, 3, 4, 64), z(2, 3, 2, 64), torch.zeros(16, 32)), {}, 'table'),
    ((z(2, 3, 4, 64), z(2, 3, 2, 64), torch.zeros(64, 16).t()), {}, 'table'),
    ((z(2, 17, 4, 64), z(2, 17, 2, 64), ROPE), {}, '17 tokens but a table of 16'),
    ((z(2, 3, 4, 64), z(2, 3, 2, 64), ROPE), dict(order='norm'), 'order'),
    ((z(2, 3, 4, 64), z(2, 3, 2, 64), ROPE), dict(positions=torch.zeros(2, 3, dtype=torch.int64)), 'positions'),
    ((z(2, 3, 4, 64), z(2, 3, 2, 64), ROPE), dict(positions=torch.zeros(2, dtype=torch.int32)), 'positions'),
    ((z(2, 3, 4, 64), z(2, 3, 2, 64), ROPE), dict(q_weight=z(64)), 'weights'),
    ((z(2, 3, 4, 64), z(2, 3, 2, 64), ROPE), dict(k_weight=torch.zeros(32)), 'weights'),
    ((z(2, 3, 4, 64), z(2, 3, 2, 64), ROPE), dict(out=(z(2, 3, 4, 64), z(2, 3, 3, 64))), 'out must'),
    ((z(2, 3, 4, 64), z(2, 3, 2, 64), ROPE), dict(out=(z(2, 3, 4, 64), z(2, 3, 1, 64).expand(2, 3, 2, 64))), 'out must'),
    ((z(2, 3, 4, 64), z(2, 3, 2, 64), ROPE), {}, 'one CUDA device'),
])
def test_qk_norm_rope_refuses(args, kw, match):
    from noise_b200.attention import qk_norm_rope
    with pytest.raises(ValueError, match=match):
        qk_norm_rope(*args, **kw)


def test_qk_norm_rope_backward_refuses():
    from noise_b200.attention import qk_norm_rope_backward
    q, k = z(2, 3, 4, 64), z(2, 3, 2, 64)
    with pytest.raises(ValueError, match='dq and dk'):
        qk_norm_rope_backward(q, q, q, k, ROPE)
    with pytest.raises(ValueError, match='dq and dk'):
        qk_norm_rope_backward(q.float(), k, q, k, ROPE)


ONE = torch.ones(2, dtype=torch.int32)


@pytest.mark.parametrize('args,kw,match', [
    ((z(2, 5, 4, 64), z(2, 5, 2, 64), z(2, 5, 2, 32), 3), {}, 'expected'),
    ((z(2, 5, 4, 64), z(1, 5, 2, 64), z(1, 5, 2, 64), 3), {}, 'expected'),
    ((z(2, 5, 4, 64), z(2, 5, 3, 64), z(2, 5, 3, 64), 3), {}, 'evenly'),
    ((z(2, 5, 4, 64), z(2, 5, 0, 64), z(2, 5, 0, 64), 3), {}, 'evenly'),
    ((z(2, 6, 4, 64), z(2, 5, 2, 64), z(2, 5, 2, 64), 3), {}, 'at least as many'),
    ((z(2, 0, 4, 64), z(2, 0, 2, 64), z(2, 0, 2, 64), 3), {}, 'at least as many'),
    ((z(2, 5, 4, 136), z(2, 5, 2, 136), z(2, 5, 2, 136), 3), {}, 'multiple of 8'),
    ((z(2, 5, 4, 60), z(2, 5, 2, 60), z(2, 5, 2, 60), 3), {}, 'multiple of 8'),
    ((z(2, 5, 4, 64).float(), z(2, 5, 2, 64).float(), z(2, 5, 2, 64).float(), 3), {}, 'bf16 or fp16'),
    ((z(2, 5, 4, 64), z(2, 5, 2, 64), z(2, 5, 2, 64).half(), 3), {}, 'bf16 or fp16'),
    ((z(2, 5, 4, 64), z(2, 5, 2, 64), z(2, 5, 2, 64), -1), {}, 'negative'),
    ((z(2, 5, 4, 64), z(2, 5, 2, 64), z(2, 5, 2, 64), 3, -2), {}, 'negative'),
    ((z(2, 5, 4, 64), z(2, 5, 2, 64), z(2, 5, 2, 64), 3), dict(scale=0.0), 'scale'),
    ((z(2, 5, 4, 64), z(2, 5, 2, 64), z(2, 5, 2, 64), 3), dict(scale=float('nan')), 'scale'),
    ((z(2, 5, 4, 64), z(2, 5, 2, 64), z(2, 5, 2, 64), 3), dict(scale=2.0 ** -101), 'scale'),
    ((z(2, 5, 4, 64), z(2, 5, 2, 64), z(2, 5, 2, 64), 3), dict(scale=2.0 ** 101), 'scale'),
    ((z(2, 5, 4, 64), z(2, 5, 2, 64), z(2, 5, 2, 64), 3), dict(offset=1), 'offset'),
    ((z(2, 5, 4, 64), z(2, 5, 2, 64), z(2, 5, 2, 64), 3), dict(lengths=ONE.long()), 'lengths'),
    ((z(2, 5, 4, 64), z(2, 5, 2, 64), z(2, 5, 2, 64), 3), dict(lengths=torch.ones(3, dtype=torch.int32)), 'lengths'),
    ((z(2, 5, 4, 64), z(2, 5, 2, 64), z(2, 5, 2, 64), 3), dict(status=torch.zeros(1)), 'status'),
    ((z(2, 5, 4, 64), z(2, 5, 2, 64), z(2, 5, 2, 64), 3), {}, 'one CUDA device'),
])
def test_window_attention_refuses(args, kw, match):
    from noise_b200.attention import window_attention, window_attention_backward
    with pytest.raises(ValueError, match=match):
        window_attention(*args, **kw)
    q, k, v, *rest = args
    with pytest.raises(ValueError, match=match):
        window_attention_backward(q, q, k, v, q, torch.zeros(2, 4, q.shape[1]), *rest, **kw)


def test_window_attention_backward_refuses():
    from noise_b200.attention import window_attention_backward
    q, k, lse = z(2, 5, 4, 64), z(2, 5, 2, 64), torch.zeros(2, 4, 5)
    h = [t.half() for t in (q, q, k, k, q)]
    with pytest.raises(ValueError, match='bf16 only'):
        window_attention_backward(*h, lse, 3)
    with pytest.raises(ValueError, match='dout and out'):
        window_attention_backward(z(2, 5, 4, 32), q, k, k, q, lse, 3)
    with pytest.raises(ValueError, match='lse must'):
        window_attention_backward(q, q, k, k, q, lse[:, :2], 3)


def test_window_attention_token_refuses():
    from noise_b200.attention import window_attention_token
    q, k = z(2, 4, 64), z(2, 5, 2, 64)
    with pytest.raises(ValueError, match='lengths are required'):
        window_attention_token(q, k, k, None, 3)
    with pytest.raises(ValueError, match='expected'):
        window_attention_token(q[:, None], k, k, ONE, 3)
    with pytest.raises(ValueError, match='lengths must'):
        window_attention_token(q, k, k, ONE[:1], 3)
    with pytest.raises(ValueError, match='one CUDA device'):
        window_attention_token(q, k, k, ONE, 3)


LOGITS, IDS, TEACHER = torch.zeros(3, 10), torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, 4)


@pytest.mark.parametrize('args,kw,match', [
    ((LOGITS[0], IDS, TEACHER), {}, 'expected'),
    ((LOGITS, IDS[:2], TEACHER[:2]), {}, 'expected'),
    ((LOGITS, IDS, TEACHER[:, :3]), {}, 'expected'),
    ((LOGITS.double(), IDS, TEACHER), {}, 'fp32, bf16 or fp16'),
    ((LOGITS, IDS, TEACHER.long()), {}, 'fp32, bf16 or fp16'),
    ((LOGITS, IDS.short(), TEACHER), {}, 'int32 or int64'),
    ((LOGITS, IDS[:, :0], TEACHER[:, :0]), {}, 'entries'),
    ((LOGITS, torch.zeros(3, 1025, dtype=torch.int32), torch.zeros(3, 1025)), {}, 'entries'),
    ((LOGITS[:, :0], IDS, TEACHER), {}, 'entries'),
    ((LOGITS, IDS, TEACHER), dict(temperature=0.0), 'temperature'),
    ((LOGITS, IDS, TEACHER), dict(temperature=float('nan')), 'temperature'),
    ((LOGITS, IDS, TEACHER), dict(softcap=-1.0), 'softcap'),
    ((LOGITS, IDS, TEACHER), {}, 'one CUDA device'),
])
def test_distill_refuses(args, kw, match):
    from noise_b200.distill import distill_backward, distill_loss, distill_loss_grad
    for call in (lambda: distill_loss(*args, **kw), lambda: distill_loss_grad(*args, **kw),
                 lambda: distill_backward(torch.zeros(3), *args, torch.zeros(3, dtype=torch.float64), **kw)):
        with pytest.raises(ValueError, match=match):
            call()


def test_distill_refuses_wrong_row_vectors_and_rows_too_long():
    from noise_b200 import _lib
    from noise_b200.distill import distill_backward, distill_loss_grad
    lse = torch.zeros(3, dtype=torch.float64)
    with pytest.raises(ValueError, match='required'):
        distill_backward(None, LOGITS, IDS, TEACHER, lse)
    with pytest.raises(ValueError, match='dloss must'):
        distill_backward(torch.zeros(2), LOGITS, IDS, TEACHER, lse)
    with pytest.raises(ValueError, match='lse must'):
        distill_backward(torch.zeros(3), LOGITS, IDS, TEACHER, lse.float())
    limit = _lib.load().noise_distill_max_vocab(0, 0)
    assert limit > 131072 and _lib.load().noise_distill_max_vocab(1, 1) > 131072
    with pytest.raises(ValueError, match='at most'):
        distill_loss_grad(torch.zeros(1, 1).expand(1, limit + 1), IDS[:1], TEACHER[:1])


# ------------------------------------------------------------------------------------------------
# the C entries: statuses that come before any CUDA call (0 ok, 1 bad argument, 4 workspace, 5 unsupported)
# ------------------------------------------------------------------------------------------------
P = 1 << 20  # a 16-byte aligned address that no call here reads


def window(lib_struct, **kw):
    f = dict(dtype=1, B=2, Tq=5, Tk=5, H=4, Hk=2, D=64, offset=0, window=3, sinks=0, scale=0.125, lengths=0, q=P, k=P, v=P,
             qs=(5 * 256, 256, 64), ks=(5 * 128, 128, 64), vs=(5 * 128, 128, 64), out=P, lse=P)
    f.update(kw)
    return lib_struct.pack(*(f[n] for n in ('dtype', 'B', 'Tq', 'Tk', 'H', 'Hk', 'D', 'offset', 'window', 'sinks', 'scale',
                                            'lengths', 'q', 'k', 'v')), *f['qs'], *f['ks'], *f['vs'], f['out'], f['lse'])


@pytest.mark.parametrize('kw,code', [
    (dict(dtype=0), 5), (dict(D=60), 5), (dict(D=136), 5), (dict(H=3), 1), (dict(Tq=6), 1), (dict(offset=1), 1),
    (dict(offset=-1), 1), (dict(window=-1), 1), (dict(sinks=-1), 1), (dict(scale=0.0), 1), (dict(q=P + 2), 1), (dict(k=0), 1),
    (dict(qs=(5 * 256, 256, 60)), 1), (dict(ks=(5 * 128, 0, 64)), 1), (dict(vs=(5 * 128, -128, 64)), 1), (dict(out=P + 8), 1),
    (dict(lse=0), 1), (dict(B=70000), 5), (dict(Tq=0), 1), (dict(B=-1), 1), (dict(B=0), 0),
])
def test_window_entries_refuse(kw, code):
    from noise_b200 import _lib
    lib = _lib.load()
    a = window(_lib.WINDOW, **kw)
    assert lib.noise_window_attention(a, P, None) == code
    steps = _lib.STEPS.pack(5 * 256, 256, 64)
    assert lib.noise_window_attention_backward(a, P, steps, P, P, P, None, 0, P, None) == code
    if 'Tq' not in kw and 'offset' not in kw and 'lse' not in kw and 'qs' not in kw:
        assert lib.noise_window_token(window(_lib.WINDOW, lengths=P, **kw), None) == code


def test_window_backward_entry_refuses():
    from noise_b200 import _lib
    lib = _lib.load()
    a, steps = window(_lib.WINDOW), _lib.STEPS.pack(5 * 256, 256, 64)
    need = lib.noise_window_backward_workspace_bytes(a)
    assert need > 0 and lib.noise_window_backward_workspace_bytes(window(_lib.WINDOW, H=3)) == -1
    back = lib.noise_window_attention_backward
    assert back(a, P, steps, P, P, P, P, need - 1, P, None) == 4
    assert back(a, P, steps, P, P, P, None, need, P, None) == 4
    assert back(a, P + 2, steps, P, P, P, P, need, P, None) == 1
    assert back(a, P, steps, P + 8, P, P, P, need, P, None) == 1
    assert back(a, P, steps, P, P, P, P, need, None, None) == 1
    assert back(window(_lib.WINDOW, dtype=2), P, steps, P, P, P, P, need, P, None) == 5
    assert lib.noise_window_attention(a, None, None) == 1
    assert lib.noise_window_token(a, None) == 1  # lengths are required


def qk(lib_struct, **kw):
    f = dict(dtype=1, order=0, B=2, T=3, H=4, Hk=2, D=64, eps=1e-6, rope=P, table=16, positions=0, pos_stride=0, wq=0, wk=0,
             q=P, k=P, dq=P, dk=P, qo=P, ko=P, qs=(768, 256, 64), dwq=0, dwk=0)
    f.update(kw)
    return lib_struct.pack(*(f[n] for n in ('dtype', 'order', 'B', 'T', 'H', 'Hk', 'D', 'eps', 'rope', 'table', 'positions',
                                            'pos_stride', 'wq', 'wk', 'q', 'k', 'dq', 'dk', 'qo', 'ko')),
                           *f['qs'], *([768, 256, 64] * 5), f['dwq'], f['dwk'])


@pytest.mark.parametrize('kw,back,code', [
    (dict(D=40), 0, 5), (dict(D=272), 0, 5), (dict(dtype=3), 0, 5), (dict(rope=0), 0, 1), (dict(rope=P + 4), 0, 1),
    (dict(table=0), 0, 1), (dict(H=0), 0, 1), (dict(q=P + 2), 0, 1), (dict(qs=(768, 256, 60)), 0, 1), (dict(ko=0), 0, 1),
    (dict(dq=0), 1, 1), (dict(wq=P), 1, 1), (dict(dwk=P), 1, 1), (dict(wq=P, dwq=P), 1, 4), (dict(B=0), 0, 0),
])
def test_qk_norm_entry_refuses(kw, back, code):
    from noise_b200 import _lib
    assert _lib.load().noise_qk_norm_rope(qk(_lib.QK_NORM, **kw), back, None, 0, None) == code


def distill(lib_struct, **kw):
    f = dict(dtype=0, tdtype=0, ids64=0, V=10, K=4, tau=1.0, cap=0.0, N=3, ld=10, ids_ld=4, t_ld=4, g_ld=10, z=P, ids=P, t=P,
             dloss=0, lse_in=0, loss=P, lse=0, grad=0)
    f.update(kw)
    return lib_struct.pack(*f.values())


@pytest.mark.parametrize('kw,code', [
    (dict(V=0), 1), (dict(K=0), 1), (dict(K=1025, ids_ld=1025, t_ld=1025), 5), (dict(tau=0.0), 1), (dict(cap=-1.0), 1),
    (dict(ld=9), 1), (dict(ids_ld=3), 1), (dict(z=0), 1), (dict(loss=0), 1), (dict(dtype=4), 5), (dict(tdtype=7), 5),
    (dict(lse_in=P), 1), (dict(grad=P + 4 * 1000, g_ld=9), 1), (dict(grad=P + 40), 1), (dict(N=0), 0),
    (dict(V=1 << 20, ld=1 << 20, g_ld=1 << 20, grad=P << 12), 5),
])
def test_distill_entry_refuses(kw, code):
    from noise_b200 import _lib
    assert _lib.load().noise_distill(distill(_lib.DISTILL, **kw), None) == code


@pytest.mark.skipif(shutil.which('gcc') is None, reason='no C compiler')
def test_argument_blocks_follow_the_header(tmp_path):
    """Every packed block has its struct's size, and its fields their offsets."""
    from noise_b200 import _lib
    blocks = {
        'NoiseQkNorm': (_lib.QK_NORM, 'dtype order B T H Hk D eps rope table positions positions_stride wq wk q k dq dk q_out '
                                      'k_out q_stride k_stride dq_stride dk_stride q_out_stride k_out_stride dwq dwk'),
        'NoiseWindow': (_lib.WINDOW, 'dtype B Tq Tk H Hk D offset window sinks scale lengths q k v q_stride k_stride v_stride '
                                     'out lse'),
        'NoiseDistill': (_lib.DISTILL, 'dtype teacher_dtype ids_int64 V K temperature softcap N ld ids_ld teacher_ld grad_ld '
                                       'logits ids teacher dloss lse_in loss lse grad'),
    }
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "noise_b200.h"', 'int main(void) {']
    for name, (_, fields) in blocks.items():
        lines.append(f'printf("%zu", sizeof({name}));')
        lines += [f'printf(" %zu", offsetof({name}, {f}));' for f in fields.split()] + ['printf("\\n");']
    src = tmp_path / 'offsets.c'
    src.write_text('\n'.join(lines + ['return 0; }']))
    subprocess.run(['gcc', f'-I{ROOT / "include"}', str(src), '-o', str(tmp_path / 'offsets')], check=True)
    rows = subprocess.run([str(tmp_path / 'offsets')], check=True, capture_output=True, text=True).stdout.split('\n')
    for (name, (block, fields)), row in zip(blocks.items(), rows):
        want = [int(x) for x in row.split()]
        assert block.size == want[0], name
        # offsets from the format: one step per field, arrays of three strides as one
        at, got = 0, []
        codes = [c for c in _expand(block.format)]
        widths = [3 if f.endswith('stride') and f != 'positions_stride' else 1 for f in fields.split()]
        i = 0
        for w in widths:
            size = struct.calcsize(codes[i])
            at = (at + size - 1) // size * size
            got.append(at)
            for _ in range(w):
                at += size
                i += 1
        assert got == want[1:] and i == len(codes), name


def _expand(fmt):
    n = ''
    for ch in fmt.replace(' ', ''):
        if ch.isdigit():
            n += ch
        else:
            yield from ch * int(n or 1)
            n = ''


def test_exact_local_is_off_in_the_recipe():
    from noise_b200.dust import recipe
    assert recipe(1.0).exact_local is False and ctypes.sizeof(ctypes.c_void_p) == 8
