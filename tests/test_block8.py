"""The C entries of rope and the block-scaled paged cache refuse what they cannot run before any device
work: no GPU needed."""
import ctypes
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import superl8_amd as sl8
from superl8_amd import _lib

ROOT = Path(__file__).resolve().parent.parent


def rope(**c):
    a = dict(q=16, k=16, dtype=0, qb=0, qh=0, q_s=0, kb=0, kh=0, k_s=0, pos=16, pos64=0, pos_axis=4, pos_b=0, table=16, rows=8,
             sections=None, axes=1, inter=0, inv=0, qo=16, ko=16, B=1, Hq=1, Hkv=1, S=4, D=64, R=64)
    return _lib.load().sl8_rope(*(a | c).values(), None)


def append(**c):
    a = dict(k=16, v=16, q=None, dtype=0, kt=0, kh=0, vt=0, vh=0, qt=0, qh=0, pos=None, pos64=0, table=None, rows=0,
             sections=None, axes=1, inter=0, rot=0, cu=None, lens=16, bt=16, kc=16, ksc=16, vc=16, vsc=16,
             qo=None, T=2, B=2, Hq=0, Hkv=1, D=64, R=0, nb=4, bs=16, maxb=2)
    return _lib.load().sl8_kv_append_block8(*(a | c).values(), None)


def attn(**c):
    a = dict(q=16, dtype=0, rot=0, mul=1.0, k=16, ks=16, v=16, vs=16, cu=None, lens=16, bt=16, out=16, T=2,
             B=2, Hq=2, Hkv=1, D=64, nb=400, bs=16, maxb=200, window=-1,
             ws=16, ws_bytes=1 << 40)
    return _lib.load().sl8_attn_paged_block8(*(a | c).values(), None)


@pytest.mark.parametrize("call,change,word", [
    (rope, dict(dtype=7), b"float"), (rope, dict(D=63), b"head dim"), (rope, dict(D=514), b"head dim"),
    (rope, dict(R=66), b"rotary dim"), (rope, dict(R=3), b"rotary dim"), (rope, dict(R=0), b"rotary dim"),
    (rope, dict(axes=5), b"axes"), (rope, dict(axes=0), b"axes"), (rope, dict(rows=0), b"positions"),
    (rope, dict(axes=2), b"sections"), (rope, dict(axes=2, sections=(ctypes.c_int32 * 2)(16, 15)), b"add up"),
    (rope, dict(table=None), b"null"), (rope, dict(q=None), b"null"), (rope, dict(ko=None), b"null"),
    (rope, dict(table=20), b"aligned"), (rope, dict(S=1 << 31), b"too large"), (rope, dict(B=-1), b"shape"),
    (append, dict(dtype=2), b"float16"), (append, dict(D=96), b"head dim"), (append, dict(bs=24), b"block_size"),
    (append, dict(bs=144), b"block_size"), (append, dict(bs=0), b"block_size"), (append, dict(T=3), b"one row"),
    (append, dict(q=16, qo=16, Hq=1), b"positions"), (append, dict(pos=16, table=16, rows=4, R=40), b"16"),
    (append, dict(lens=None), b"null"), (append, dict(bt=None), b"null"), (append, dict(ksc=None), b"null"),
    (append, dict(k=24), b"aligned"), (append, dict(kc=20), b"aligned"), (append, dict(T=1 << 28, B=1), b"large"),
    (append, dict(kt=4), b"aligned"), (append, dict(vh=12), b"aligned"),
    (append, dict(q=16, qo=16, Hq=1, pos=16, table=16, rows=4, R=32, qt=4), b"aligned"),
    (attn, dict(dtype=2), b"float16"), (attn, dict(D=32), b"head dim"), (attn, dict(bs=8), b"block_size"),
    (attn, dict(Hq=3, Hkv=2), b"divisible"), (attn, dict(T=3), b"one row"), (attn, dict(q=None), b"null"),
    (attn, dict(lens=None), b"null"), (attn, dict(vs=None), b"null"), (attn, dict(q=24), b"aligned"),
    (attn, dict(k=8), b"aligned"), (attn, dict(maxb=1 << 31), b"large"), (attn, dict(maxb=1 << 26), b"large"),
    (rope, dict(S=(1 << 31) - 1), b"too large"), (append, dict(T=(1 << 28) - 1, B=1, cu=16), b"too large"),
    (append, dict(T=1 << 23, B=1 << 23), b"too large"),
    (attn, dict(T=(1 << 24) - 1, B=(1 << 24) - 1, Hq=1), b"too large"),
    (attn, dict(ws=None), b"workspace"), (attn, dict(ws_bytes=100), b"workspace"), (attn, dict(ws=24), b"workspace"),
])
def test_refused(call, change, word):
    assert call(**change) == -1
    assert word in _lib.load().sl8_last_error()


@pytest.mark.parametrize("call,change", [(rope, dict(B=0)), (rope, dict(S=0)), (append, dict(T=0, B=0)),
                                         (attn, dict(T=0, B=0)), (attn, dict(Hq=0))])
def test_nothing_to_do(call, change):
    assert call(**change) == 0


@pytest.mark.parametrize("T,B,Hq,Hkv,D", [(100, 1, 8, 2, 0), (100, 1, 8, 2, 96), (100, 1, 8, 2, -64), (100, 1, 8, 3, 64),
                                          (100, 1, 2, 4, 64), (0, 1, 8, 2, 64), (100, 0, 8, 2, 64), (100, 1, 0, 2, 64),
                                          (100, 1, 8, 0, 64), (-1, 1, 8, 2, 64), (1 << 28, 1, 8, 2, 64)])
def test_workspace_of_refused_sizes(T, B, Hq, Hkv, D):
    """A C caller asks before the call that refuses: nothing to reserve, and the process goes on."""
    code = f"from superl8_amd import _lib; assert _lib.load().sl8_attn_paged_block8_workspace({T}, {B}, {Hq}, " \
           f"{Hkv}, {D}, 1 << 20) == 0"
    assert subprocess.run([sys.executable, "-c", code], cwd=ROOT).returncode == 0
    assert _lib.load().sl8_attn_paged_block8_workspace(100, 1, 8, 2, 64, 1 << 20) > 0


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 2, 3, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        sl8.rope(x, x, torch.zeros(3, dtype=torch.int32), torch.zeros(4, 64))
    c, s = torch.zeros(2, 2, 16, 64, dtype=torch.int8), torch.ones(2, 2)
    bt, n = torch.zeros(3, 1, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        sl8.quantize_kv_append_block8(x[0].transpose(0, 1), x[0].transpose(0, 1), c, s, c, s, bt, n)
    with pytest.raises(RuntimeError, match="CUDA"):
        sl8.attn_paged_block8(x[0].transpose(0, 1), c, s, c, s, bt, n)


def test_rotation_needs_a_power_of_two():
    with pytest.raises(ValueError, match="power-of-two"):
        sl8.quantize_kv_append_block8(torch.zeros(1, 1, 96), *[None] * 5, None, None, rotate=True)


def test_table_on_the_cpu():
    t = sl8.rope_table(50, 8, sections=(1, 3), device="cpu").double()
    f = torch.tensor([1.0, 1.0, 10000.0 ** (-1 / 3), 10000.0 ** (-2 / 3)], dtype=torch.float64)
    a = torch.arange(50, dtype=torch.float64)[:, None] * f
    assert torch.allclose(t, torch.cat([a.cos(), a.sin()], 1), rtol=0, atol=2.0 ** -24)
