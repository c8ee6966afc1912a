"""The block-scaled paged int8 cache: append (with the position rotation on the way) and attention
against plain 64-bit forms, their bounds, what they leave alone, and a run of them together."""
import math

import pytest
import torch

import superl8_amd as sl8
from superl8_amd import _C, _lib
from tests.test_rope_gpu import check as check_rope
from tests.test_rope_gpu import turned

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
DEV = "cuda"
LOG2E = math.log2(math.e)


def hadamard(d):
    h = torch.ones(1, 1, dtype=torch.float64)
    while h.shape[0] < d:
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
    return (h / math.sqrt(d)).to(DEV)


def i32(x):
    return torch.tensor(x, device=DEV, dtype=torch.int32)


class Cache:
    """A shuffled pool of random codes with the blocks of sequences of up to `cap` tokens each."""

    def __init__(self, cap, Hkv, D, bs, spare=2, scale=3.5 / 127):
        need = [-(-n // bs) for n in cap]
        nb = sum(need) + spare
        order = torch.randperm(nb, device=DEV).int()
        self.table = torch.full((len(cap), max(need + [1])), -1, device=DEV, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.k, self.v = (torch.randint(-127, 128, (nb, Hkv, bs, D), device=DEV, dtype=torch.int8)
                          for _ in range(2))
        self.ks, self.vs = ((torch.rand(nb, Hkv, device=DEV) + 0.5) * scale for _ in range(2))
        self.bs = bs

    def args(self):
        return self.k, self.ks, self.v, self.vs, self.table

    def copy(self):
        c = object.__new__(Cache)
        c.__dict__ = {n: t.clone() if torch.is_tensor(t) else t for n, t in self.__dict__.items()}
        return c

    def rows(self, b, h, n):
        """K and V of the first n tokens of sequence b, head h, in 64 bits, and V's scales."""
        pages = self.table[b, :-(-n // self.bs)].long()
        k, v = ((c[pages, h].double() * s[pages, h].double()[:, None, None]).flatten(0, 1)[:n]
                for c, s in ((self.k, self.ks), (self.v, self.vs)))
        return k, v, self.vs[pages, h].double().repeat_interleave(self.bs)[:n]


def offsets(new):
    return i32([sum(new[:i]) for i in range(len(new) + 1)])


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
def append_and_check(c, new, total, k, v, q=None, pos=None, table=None, sections=None, interleaved=False,
                     rotate=False, cu=True):
    """Appends and checks every code and scale of the pool. Codes of new rows stand within half a step
    of the value, plus: 2^-22 of the pair's products (rope) and D log2(D) sums of 2^-24 of the row's
    2-norm (rotation), 127 * 2^-22 for the scale's and the quotient's roundings."""
    was = c.copy()
    T, Hkv, D = k.shape
    bs = c.bs
    got = sl8.quantize_kv_append_block8(k, v, *c.args(), i32(total), cu_lens=offsets(new) if cu else None,
                                        q=q, positions=pos, table=table, sections=sections,
                                        interleaved=interleaved, rotate=rotate)
    kk, err = k.double(), torch.zeros(T, Hkv, 1, device=DEV, dtype=torch.float64)
    if pos is not None:
        p = (pos if sections else pos[None])[:, None]  # [A, 1, T]
        if q is not None:
            check_rope(got.transpose(0, 1)[None], *turned(q.transpose(0, 1)[None], p, table, sections,
                                                         interleaved, False))
        kk, size = (x[0].transpose(0, 1) for x in turned(k.transpose(0, 1)[None], p, table, sections,
                                                         interleaved, False))
        err = size.amax(-1, keepdim=True) * 3 * 2.0 ** -24
        if rotate:
            err = err * math.sqrt(D)
    if rotate:
        err = err + kk.norm(dim=-1, keepdim=True) * (math.log2(D) + 1) * 2.0 ** -24
        kk = kk @ hadamard(D)
    written = torch.zeros(c.k.shape[0], bs, device=DEV, dtype=torch.bool)
    held = torch.zeros_like(written)
    touched = torch.zeros(c.k.shape[0], device=DEV, dtype=torch.bool)
    for x, e, code, scale, code0, scale0 in ((kk, err, c.k, c.ks, was.k, was.ks),
                                             (v.double(), 0 * err, c.v, c.vs, was.v, was.vs)):
        t = 0
        for b, n in enumerate(new):
            at = total[b] - n
            t_end = t + n
            while t < t_end:
                page, off = int(c.table[b, at // bs]), at % bs
                m = min(bs - off, t_end - t)
                rows, tol = x[t:t + m].transpose(0, 1), e[t:t + m].transpose(0, 1)  # [Hkv, m, D]
                least = torch.full((Hkv,), 2.0 ** -60, device=DEV, dtype=torch.float64)
                if off:
                    least = torch.maximum(least, scale0[page].double())
                want = torch.maximum(rows.abs().amax((1, 2)) / 127, least)
                s = scale[page].double()
                assert bool(((s - want).abs() <= want * 2.0 ** -22 + tol.amax((1, 2)) / 127).all())
                s = s[:, None, None]
                lim = s * (0.5 + 127 * 2.0 ** -22) + tol
                assert bool(((code[page][:, off:off + m].double() * s - rows).abs() <= lim).all())
                ratio = (scale0[page] / scale[page])[:, None, None]
                again = torch.round(code0[page][:, :off].float() * ratio).to(torch.int8)
                assert torch.equal(code[page][:, :off], again)
                written[page, off:off + m] = held[page, :off] = touched[page] = True
                at, t = at + m, t + m
        same = ~(written | held)[:, None, :, None].expand(code.shape)
        assert torch.equal(code[same], code0[same]) and torch.equal(scale[~touched], scale0[~touched])
    return got


def news(T, Hq, Hkv, D, dtype, size=1.0):
    x = (torch.randn(T, Hq + 2 * Hkv, D, device=DEV) * size).to(dtype)
    return x.split([Hq, Hkv, Hkv], 1)


@pytest.mark.parametrize("D,bs", [(64, 16), (64, 128), (128, 16), (128, 48), (128, 128), (256, 16), (256, 112)])
@pytest.mark.parametrize("rotate", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_append_ragged(D, bs, rotate, dtype):
    new, old = [1, 3 * bs + 5, bs, 2, 17, bs - 1], [0, 5, bs, bs - 1, bs + 3, 1]
    total = [a + b for a, b in zip(new, old)]
    c = Cache(total, 2, D, bs)
    q, k, v = news(sum(new), 6, 2, D, dtype, 2.0)
    sections = (D // 8, D // 4, D // 8)
    pos = torch.randint(0, 300, (3, sum(new)), device=DEV)
    append_and_check(c, new, total, k, v, q, pos, sl8.rope_table(300, D), sections, rotate=rotate)


@pytest.mark.parametrize("R,interleaved,sections", [(32, False, None), (48, True, (5, 19)), (96, False, (7, 41)),
                                                    (16, True, None), (128, True, (1, 2, 3, 58))])
def test_append_partial_rotation(R, interleaved, sections):
    new, total = [4, 9, 30], [20, 9, 61]
    c = Cache(total, 3, 128, 32)
    q, k, v = news(43, 3, 3, 128, F16)
    pos = torch.randint(0, 99, (len(sections), 43) if sections else (43,), device=DEV, dtype=torch.int32)
    append_and_check(c, new, total, k, v, q, pos, sl8.rope_table(99, R), sections, interleaved, True)


@pytest.mark.parametrize("B", [1, 3, 70, 200])
def test_append_one_each(B):
    """The decode step, with and without cu_lens, sequences starting blocks among them."""
    total = [1 + (i * 7) % 50 for i in range(B)]
    c = Cache(total, 2, 64, 16)
    _, k, v = news(B, 0, 2, 64, F16)
    d = c.copy()
    append_and_check(c, [1] * B, total, k, v, rotate=True, cu=False)
    append_and_check(d, [1] * B, total, k, v, rotate=True)
    assert torch.equal(c.k, d.k) and torch.equal(c.vs, d.vs)


def test_append_many_sequences_some_without_tokens():
    new = [(i * 5) % 4 for i in range(150)]
    total = [n + (i * 3) % 40 for i, n in enumerate(new)]
    c = Cache([max(1, t) for t in total], 1, 64, 32)
    _, k, v = news(sum(new), 0, 1, 64, BF16)
    append_and_check(c, new, total, k, v)


def test_scales_grow_and_stay():
    """Large rows requantise the block, small ones leave it; zeros take the least scale and a block of
    zeros takes the next rows' scale."""
    c = Cache([40], 1, 64, 16)
    z = torch.zeros(1, 1, 64, device=DEV, dtype=F16)
    append_and_check(c, [1], [17], z, z)
    page = int(c.table[0, 1])
    assert float(c.ks[page, 0]) == 2.0 ** -60 and not c.k[page, 0, 0].any()
    for i, size in enumerate((1e-4, 1.0, 0.01, 1000.0, 1.0)):
        _, k, v = news(1, 0, 1, 64, F16, size)
        append_and_check(c, [1], [18 + i], k, v)
    _, k, v = news(2, 0, 1, 64, BF16, 1e-30)  # below the least scale: codes of zero
    append_and_check(c, [2], [34], k, v)
    assert float(c.ks[int(c.table[0, 2]), 0]) == 2.0 ** -60
    _, k, v = news(3, 0, 1, 64, BF16, 1e36)
    append_and_check(c, [3], [37], k, v, rotate=True)


def test_append_is_idempotent_and_in_views():
    """The same step again changes nothing; rows of misaligned or transposed tensors are the same."""
    new, total = [5, 20], [12, 43]
    c = Cache(total, 2, 64, 16)
    x = torch.randn(25, 4, 64, device=DEV).to(F16)
    append_and_check(c, new, total, x[:, :2], x[:, 2:])
    d = c.copy()
    append_and_check(c, new, total, x[:, :2], x[:, 2:])
    assert torch.equal(c.k, d.k) and torch.equal(c.ks, d.ks) and torch.equal(c.v, d.v)
    odd = torch.empty(25 * 4 * 64 + 3, device=DEV, dtype=F16)[3:].view(25, 4, 64).copy_(x)
    append_and_check(c, new, total, odd[:, :2], odd[:, 2:])
    by_head = x.transpose(0, 1).contiguous().transpose(0, 1)
    append_and_check(c, new, total, by_head[:, :2], by_head[:, 2:].transpose(1, 2).contiguous().transpose(1, 2))
    assert torch.equal(c.k, d.k) and torch.equal(c.vs, d.vs)


def test_append_skips_what_is_not_there():
    """Block ids outside the pool, more tokens than the table holds, lengths below the new tokens,
    offsets past the rows: nothing else is written; rows past the last offset only have Q turned."""
    c = Cache([40, 40, 40], 1, 64, 16, spare=4)
    c.table[0, 1], c.table[1, 1] = -1, c.k.shape[0]
    was = c.copy()
    q, k, v = news(30, 1, 1, 64, F16)
    pos = torch.arange(30, device=DEV)
    out = sl8.quantize_kv_append_block8(k, v, *c.args(), i32([20, 20, 3]), cu_lens=i32([0, 10, 20, 29]), q=q,
                                        positions=pos, table=sl8.rope_table(40, 64))
    check_rope(out.transpose(0, 1)[None], *turned(q.transpose(0, 1)[None], pos[None, None],
                                                  sl8.rope_table(40, 64), None, False, False))
    first = [int(c.table[0, 0]), int(c.table[1, 0])]
    for x, y in ((c.k, was.k), (c.v, was.v), (c.ks, was.ks), (c.vs, was.vs)):
        other = [i for i in range(x.shape[0]) if i not in first]
        assert torch.equal(x[other], y[other]) and not torch.equal(x[first], y[first])
    d = c.copy()
    big = i32([0, 10 ** 6, 2 * 10 ** 6, 2 ** 31 - 1])  # past the rows
    sl8.quantize_kv_append_block8(k, v, *c.args(), i32([-5, 2 ** 31 - 1, -2 ** 31]), cu_lens=big)
    assert torch.equal(c.k, d.k) and torch.equal(c.ks, d.ks)
    sl8.quantize_kv_append_block8(k[:3], v[:3], c.k, c.ks, c.v, c.vs, c.table[:, :0], i32([5, 6, 7]))
    none = torch.zeros(0, 1, 16, 64, device=DEV, dtype=torch.int8)
    sl8.quantize_kv_append_block8(k[:3], v[:3], none, torch.zeros(0, 1, device=DEV), none,
                                  torch.zeros(0, 1, device=DEV), c.table, i32([5, 6, 7]))
    assert torch.equal(c.k, d.k) and torch.equal(c.ks, d.ks)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def coded_queries(T, Hq, D, dtype, rotate, size=0.02):
    """Queries whose int8 codes are no matter of rounding: whole steps with one of 127 per row (in the
    rotated frame with `rotate`, where 16 bits leave them within a quarter of a step: 127 steps in a
    row of norm sqrt(D) * 40 are off by 2^-9 * 127 at most in bf16 once sums are over)."""
    q = (torch.randn(T, Hq, D, device=DEV, dtype=torch.float64) * 30).round().clamp(-120, 120)
    q[..., 3] = 127
    q = q * 2.0 ** round(math.log2(size))
    if rotate:
        q = q @ hadamard(D)
    return q.to(dtype)


def plain_attn(c, q, new, total, rotate, scale, window):
    """The operator in 64 bits; sum p |v| per element and max p vs per row, for the tolerance."""
    x = q.double()
    if rotate:
        x = x @ hadamard(q.shape[-1])
    qs = x.abs().amax(-1, keepdim=True) / 127
    qs = torch.where(qs == 0, 1.0, qs)
    x = torch.round(x / qs) * qs
    out, size, top = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x[..., :1])
    Hkv = c.k.shape[1]
    G = q.shape[1] // Hkv
    t = 0
    for b, (m, n) in enumerate(zip(new, total)):
        for h in range(Hkv if m else 0):
            k, v, vs = c.rows(b, h, n)
            for j in range(h * G, h * G + G):
                w = x[t:t + m, j] @ k.T * scale
                i = torch.arange(n - m, n, device=DEV)[:, None]
                key = torch.arange(n, device=DEV)
                seen = key <= i
                if window >= 0:
                    seen = seen & (key > i - window)
                p = torch.softmax(w.masked_fill(~seen, -math.inf), -1).nan_to_num(0.0)
                out[t:t + m, j], size[t:t + m, j] = p @ v, p @ v.abs()
                top[t:t + m, j] = (p * vs).amax(-1, keepdim=True)
        t += m
    return out, size, top


def attn_and_check(c, q, new, total, rotate=False, scale=None, window=-1, cu=True):
    """Tolerance: p rounded to 16 bits (2^-11), exp2 and its argument in 32 (logits of up to 2^7 in base
    2 by 4 roundings: 2^-15), the sums of N keys in 32 (N * 2^-24), each relative to sum p |v|; weights
    below the 16-bit normals (2^-25 of the largest, 127 codes, N keys); the output's rounding."""
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    got = sl8.attn_paged_block8(q, *c.args(), i32(total), cu_lens=offsets(new) if cu else None, scale=scale,
                                rotate=rotate, window_left=window)
    want, size, top = plain_attn(c, q, new, total, rotate, scale, window)
    N, eps = max(total), torch.finfo(q.dtype).eps / 2
    lim = size * (2.0 ** -11 + 2.0 ** -15 + N * 2.0 ** -24) + N * 127 * 2.0 ** -25 * top + \
        eps * (1 + 2.0 ** -8) * want.abs() + 2.0 ** -25
    err = (got.double() - want).abs()
    assert got.dtype == q.dtype and got.shape == q.shape
    assert bool((err <= lim).all()), (float((err - lim).max()), float(err.max()))
    return got


def attn_and_check_small_weights(c, q, new, total, window=-1, scale=None):
    """attn_and_check with what the 16-bit weights keep: the largest contribution's weight is 2^8 at least, half a
    step of the subnormal ones 2^-25, so a weight is off by 2^-33 of that contribution's beside its 2^-11."""
    got = attn_and_check(c, q, new, total, window=window, scale=scale)
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    want, size, top = plain_attn(c, q, new, total, False, scale, window)
    N, eps = max(total), torch.finfo(q.dtype).eps / 2
    lim = size * (2.0 ** -11 + 2.0 ** -15 + N * 2.0 ** -24) + N * 127 * 2.0 ** -33 * top + \
        eps * (1 + 2.0 ** -8) * want.abs() + 2.0 ** -25
    err = (got.double() - want).abs()
    assert bool((err <= lim).all()), (float((err - lim).max()), float(err.max()))


def split_tiles(T, B, Hq, Hkv, D, keys):
    """Tiles of 64 keys above which a sequence's keys are split over workgroups, from the size of the
    workspace (which holds ROWS rows for every workgroup that is resident at once); no workspace, no split."""
    ws = _lib.load().sl8_attn_paged_block8_workspace(T, B, Hq, Hkv, D, keys)
    assert ws > 0
    G = Hq // Hkv
    rows = -(-T * G // B)
    ROWS = 16 if rows <= 16 else 32 if rows <= 32 and D < 256 else 64 if rows <= 64 else 128
    pairs = Hkv * (T * G // ROWS + B)
    slots = (ws - 32 * pairs - 16) // (ROWS * (D + 2) * 4)
    if ROWS <= 32:
        return 16
    return 128 * (12 * slots + 32 * min(Hkv * max(B, T * G // ROWS), slots)) // (D * slots)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bs", [16, 48, 128])
@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (8, 2), (8, 1), (6, 2)])
def test_decode(D, bs, Hq, Hkv):
    total = [1, 2, 15, 16, 17, 63, 64, 65, 130, 777]
    c = Cache(total, Hkv, D, bs)
    for dtype, rotate in ((F16, False), (BF16, True)):
        attn_and_check(c, coded_queries(10, Hq, D, dtype, rotate), [1] * 10, total, rotate, cu=False)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Hq,new", [(2, 1), (8, 1), (6, 2), (8, 4), (2, 16), (32, 1)])
def test_fp16_weights_in_two_parts(D, Hq, new):
    """Up to 16 rows of a sequence and KV head in fp16: no 2^-11 of sum p |v|, which one 16-bit weight alone
    would add. The parts leave 2^-22 of a weight and 2^-33 of the largest."""
    total = [new, new + 1, 17, 40, 130, 777, 3000]
    c = Cache(total, 2, D, 16)
    q = coded_queries(new * 7, Hq, D, F16, False)
    got = sl8.attn_paged_block8(q, *c.args(), i32(total), cu_lens=offsets([new] * 7), rotate=False)
    want, size, top = plain_attn(c, q, [new] * 7, total, False, D ** -0.5, -1)
    N = max(total)
    lim = size * (2.0 ** -22 + 2.0 ** -15 + N * 2.0 ** -24) + N * 127 * 2.0 ** -33 * top + \
        2.0 ** -11 * (1 + 2.0 ** -8) * want.abs() + 2.0 ** -25
    assert bool(((got.double() - want).abs() <= lim).all())


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("new", [2, 5, 8, 16])
@pytest.mark.parametrize("G", [1, 3, 8])
def test_drafts(D, new, G):
    total = [new, new + 1, 100, 333, 1030]
    c = Cache(total, 2, D, 32)
    attn_and_check(c, coded_queries(new * 5, 2 * G, D, F16, False), [new] * 5, total)


@pytest.mark.parametrize("D,Hq,Hkv,bs", [(64, 4, 1, 64), (128, 8, 2, 16), (128, 5, 5, 32), (256, 4, 2, 16),
                                         (256, 2, 1, 128)])
@pytest.mark.parametrize("window", [-1, 0, 1, 100])
def test_ragged_prompts(D, Hq, Hkv, bs, window):
    new = [1, 200, 0, 37, 129, 64, 3]
    total = [500, 200, 90, 1000, 130, 64, 700]
    c = Cache(total, Hkv, D, bs)
    q = coded_queries(sum(new), Hq, D, BF16, True)
    out = attn_and_check(c, q, new, total, True, window=window)
    if window == 0:
        assert not out.any()


def test_many_sequences():
    new = [1 + (i % 3 == 0) * (i % 7) for i in range(150)]
    total = [n + (i * 37) % 400 for i, n in enumerate(new)]
    c = Cache(total, 2, 64, 16)
    attn_and_check(c, coded_queries(sum(new), 8, 64, F16, False), new, total)


@pytest.mark.parametrize("B,new", [(100, 1), (70, 3), (130, 20)])
@pytest.mark.parametrize("cu", [True, False])
def test_many_sequences_one_long(B, new, cu):
    """More sequences than a wave holds, and keys split over workgroups for the long ones."""
    if not cu and new > 1:
        return
    total = [new + (i * 31) % 90 for i in range(B)]
    total[B // 2], total[B - 1] = 3333, 1500
    c = Cache(total, 1, 128, 16)
    attn_and_check(c, coded_queries(B * new, 4, 128, F16, False), [new] * B, total, cu=cu)


@pytest.mark.parametrize("B", [63, 65, 700, 5000])
def test_many_sequences_some_without_rows(B):
    """Sequences of 0 to 3 new tokens found by their offsets, the first and the last ones empty."""
    new = [0, 0] + [(i * 7) % 4 for i in range(B - 4)] + [0, 0]
    total = [n + (i * 5) % 21 for i, n in enumerate(new)]
    c = Cache(total, 1, 64, 16)
    q, k, v = news(sum(new), 1, 1, 64, F16)
    append_and_check(c, new, total, k, v)
    for Hq in (2, 80)[:1 if B > 100 else 2]:  # a unit or several of a token
        attn_and_check(c, coded_queries(sum(new), Hq, 64, F16, False), new, total)


@pytest.mark.parametrize("new", [1, 2, 7])
@pytest.mark.parametrize("Hq,D", [(17, 128), (33, 64), (65, 128), (130, 64), (200, 256), (300, 128)])
@pytest.mark.parametrize("cu", [True, False])
def test_wide_groups(new, Hq, D, cu):
    """All query heads on one KV head: groups that end inside a unit or span several."""
    if not cu and new > 1:
        return
    total = [30 + new, 1500, new]
    c = Cache(total, 1, D, 32)
    attn_and_check(c, coded_queries(3 * new, Hq, D, F16, False), [new] * 3, total, cu=cu)


@pytest.mark.parametrize("new", [1, 4, 300])
def test_long_contexts(new):
    total = [40000, 9, 20001] if new < 100 else [20001]
    new = [min(new, n) for n in total]
    c = Cache(total, 1, 128, 64)
    attn_and_check(c, coded_queries(sum(new), 4, 128, F16, False, 0.06), new, total)


def test_peaked_and_flat_softmax_and_scale():
    total = [600, 350]
    c = Cache(total, 2, 128, 16)
    for new in ([1, 1], [3, 2], [200, 150]):
        for scale in (0.0, 1e-3, 0.3, -0.1):  # logits of up to 2^7 in base 2 stay in the tolerance
            attn_and_check(c, coded_queries(sum(new), 4, 128, F16, False, 0.02), new, total, scale=scale)


@pytest.mark.parametrize("new", [1, 4, 200])
def test_scales_of_blocks_far_apart(new):
    """Blocks of V a millionfold apart, blocks of the least scale, and keys whose weight lies in a
    block of small values: the largest contribution sets the reference, not the largest weight."""
    total = [400, 400]
    c = Cache(total, 1, 128, 16)
    c.vs[::3] *= 1e-6
    c.vs[1::5] = 2.0 ** -60
    c.k[1::5] = 0
    c.vs[2::7] *= 1e4
    q = coded_queries(2 * new, 4, 128, BF16, False, 0.06)
    attn_and_check(c, q, [new] * 2, total)
    c.vs[:] = 2.0 ** -60  # nothing but least scales: weights as usual, an output of nearly nothing
    assert float(sl8.attn_paged_block8(q, *c.args(), i32(total), cu_lens=offsets([new] * 2),
                                       rotate=False).abs().max()) <= 127 * 2.0 ** -60 * (1 + 2.0 ** -7)


@pytest.mark.parametrize("new", [1, 3, 90])
def test_scales_of_zero(new):
    """Blocks of zeros whose scales say 0: V adds nothing and its keys keep their weights."""
    total = [150, 200]
    c = Cache(total, 1, 64, 16)
    for scale in (c.ks, c.vs):
        scale[::4] = 0
    q = coded_queries(2 * new, 4, 64, F16, False)
    attn_and_check(c, q, [new] * 2, total)
    c.ks[:], c.vs[:] = 0, 0
    # no weight times 127 codes of 2^-60
    assert not sl8.attn_paged_block8(q, *c.args(), i32(total), cu_lens=offsets([new] * 2), rotate=False).any()


@pytest.mark.parametrize("new", [1, 3, 90])
def test_unread_places(new):
    """Codes and scales of unused blocks, slots behind the last token, table entries past the context
    and rows behind the last sequence hold anything."""
    total = [100, 201, 90]
    c = Cache(total, 2, 128, 32)
    q = coded_queries(3 * new + 7, 8, 128, F16, False)
    cu = offsets([new] * 3)
    lens = i32(total)
    want = sl8.attn_paged_block8(q, *c.args(), lens, cu_lens=cu, rotate=False)
    used = torch.zeros(c.k.shape[0], dtype=torch.bool, device=DEV)
    for b, n in enumerate(total):
        pages = c.table[b, :-(-n // 32)].long()
        used[pages] = True
        c.k[pages[-1], :, n % 32 or 32:] = 127
        c.v[pages[-1], :, n % 32 or 32:] = -127
        c.table[b, -(-n // 32):] = 2 ** 31 - 1
    c.ks[~used], c.vs[~used] = math.nan, math.inf
    got = sl8.attn_paged_block8(q, *c.args(), lens, cu_lens=cu, rotate=False)
    assert torch.equal(got, want) and not got[3 * new:].any() and bool(got[:3 * new].isfinite().all())


@pytest.mark.parametrize("B,new,n", [(2, 1, 90), (3, 3, 150), (2, 90, 201), (100, 1, 40), (3, 1, 3000), (70, 5, 2500),
                                     (2, 100, 5000)])
def test_rows_of_no_sequence(B, new, n):
    """Offsets that start behind row 0 and end in front of the last, as a part of a batch has them: the rows of no
    sequence append nothing and are zeros in whole and in split calls, whatever the memory held."""
    total = [n - 3 * (i % 9) for i in range(B)]
    front, back, rows = 6, 5, B * new
    c = Cache(total, 1, 64, 16)
    q, k, v = news(front + rows + back, 4, 1, 64, F16)
    part = slice(front, front + rows)
    cu, lens = offsets([new] * B), i32(total)
    d = c.copy()
    sl8.quantize_kv_append_block8(k, v, *c.args(), lens, cu_lens=cu + front, rotate=False)
    sl8.quantize_kv_append_block8(k[part], v[part], *d.args(), lens, cu_lens=cu, rotate=False)
    assert torch.equal(c.k, d.k) and torch.equal(c.v, d.v) and torch.equal(c.ks, d.ks) and torch.equal(c.vs, d.vs)
    q = q.contiguous()
    want = sl8.attn_paged_block8(q[part], *c.args(), lens, cu_lens=cu, rotate=False)
    torch.full_like(q, math.nan)  # (its memory is the output's next)
    got = sl8.attn_paged_block8(q, *c.args(), lens, cu_lens=cu + front, rotate=False)
    assert not got[:front].any() and not got[front + rows:].any()
    # (the mean rows of a sequence may choose another kernel: both within 2^-10 of sum p |v| and half a step)
    assert float((got[part].double() - want.double()).abs().max()) <= 2.0 ** -9 * 127 * 1.5 * 3.5 / 127
    none = sl8.attn_paged_block8(q, *c.args()[:4], c.table[:0], i32([]), cu_lens=i32([front]))
    assert not none.any()


@pytest.mark.parametrize("new", [1, 3, 90])
def test_attention_skips_what_is_not_there(new):
    """A block id outside the pool hides its keys; contexts beyond the table end with it; negative ones
    give zeros; offsets out of order fault nothing."""
    total = [160, 160]
    c = Cache(total, 1, 64, 16)
    q = coded_queries(2 * new, 2, 64, F16, False)
    hide = c.copy()
    hide.table[0, 3], hide.table[1, 0] = -7, hide.k.shape[0]
    got = sl8.attn_paged_block8(q, *hide.args(), i32(total), cu_lens=offsets([new] * 2), rotate=False)
    # the same with the hidden keys' weights driven to nothing: K zeroed apart, a logit far below
    x = q.double()
    for b in range(2):
        k, v, _ = c.rows(b, 0, 160)
        gone = torch.zeros(160, dtype=torch.bool, device=DEV)
        gone[slice(48, 64) if b == 0 else slice(0, 16)] = True
        i = torch.arange(160 - new, 160, device=DEV)[:, None]
        bad = (torch.arange(160, device=DEV) > i) | gone
        for h in range(2):
            p = torch.softmax((x[b * new:(b + 1) * new, h] @ k.T / 8).masked_fill(bad, -math.inf), -1)
            err = (got[b * new:(b + 1) * new, h].double() - p @ v).abs()
            # as attn_and_check, with |v| up to 127 * 1.5 steps
            assert float(err.max()) <= (2.0 ** -10 + 2.0 ** -14) * 127 * 1.5 * 3.5 / 127
    hide.table[:] = -1
    assert not sl8.attn_paged_block8(q, *hide.args(), i32(total), cu_lens=offsets([new] * 2),
                                     rotate=False).any()
    long = sl8.attn_paged_block8(q, *c.args(), i32([160 + new, 2 ** 31 - 1]), cu_lens=offsets([new] * 2),
                                 rotate=False)
    assert bool(long.isfinite().all())
    assert not sl8.attn_paged_block8(q, *c.args(), i32([0, -2 ** 31]), cu_lens=offsets([new] * 2),
                                     rotate=False).any()
    for cu in ([5, 3, 1], [0, 2 ** 31 - 1, -4], [-9, -9, 2 ** 31 - 1]):  # out of order: no fault
        sl8.attn_paged_block8(q, *c.args(), i32(total), cu_lens=i32(cu), rotate=False)
    torch.cuda.synchronize()


@pytest.mark.parametrize("new", [1, 3, 90])
def test_blocks_that_left_the_window(new):
    """Blocks in front of every row's window may be anyone's: their codes and scales are not used."""
    total, bs, window = [300, 170], 16, 20
    c = Cache(total, 2, 64, bs)
    q = coded_queries(2 * new, 4, 64, F16, False)
    run = lambda: sl8.attn_paged_block8(q, *c.args(), i32(total), cu_lens=offsets([new] * 2), rotate=False,
                                        window_left=window)
    want = run()
    for bad in (math.nan, math.inf):
        for b, n in enumerate(total):
            gone = c.table[b, :(n - new - window + 1) // bs].long()
            c.k[gone], c.v[gone], c.ks[gone], c.vs[gone] = 127, -127, bad, bad
        assert bool(want.isfinite().all()) and torch.equal(run(), want)


@pytest.mark.parametrize("D,window", [(64, 3001), (128, 1500), (128, 3001), (256, 1500), (256, 3001)])
@pytest.mark.parametrize("B,new", [(3, 1), (3, 5), (3, 12), (2, 20), (2, 150), (70, 1), (70, 5)])
@pytest.mark.parametrize("Hq,Hkv", [(4, 1), (2, 2)])
def test_window_over_split_keys(D, window, B, new, Hq, Hkv):
    """Windows that begin and end inside the keys of a split, with splits that some rows of a unit do not see."""
    total = [9000, 5003, 2600][:B] + [new + (i * 31) % 90 for i in range(B - 3)]
    T, bs = B * new, 16
    assert window // 64 > split_tiles(T, B, Hq, Hkv, D, -(-9000 // bs) * bs)
    c = Cache(total, Hkv, D, bs)
    attn_and_check_small_weights(c, coded_queries(T, Hq, D, F16, False), [new] * B, total, window)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 5, 30, 200])
@pytest.mark.parametrize("step", [10.0, 20.0, 24.5])
def test_small_weights(D, new, step):
    """The key of the largest weight has a value of zero; 40000 of 2^-step to 2^-(1.16 step) of it make the output."""
    N = 40000
    c = Cache([N], 1, D, 64)
    c.k[:], c.v[:], c.ks[:], c.vs[:] = 0, c.v.abs().clamp(min=1), 1 / 127, 1
    c.k[..., 0].random_(-20, 1)
    first = int(c.table[0, 0])
    c.k[first, 0, 0, 0], c.v[first, 0, 0] = 127, 0
    q = torch.zeros(new, 4, D, device=DEV, dtype=F16)
    q[..., 0] = 1
    attn_and_check_small_weights(c, q, [new], [N], scale=step / LOG2E)


@pytest.mark.parametrize("new", [1, 40, 1024])
def test_long_tail_of_small_weights(new):
    """One key of weight 1 whose value is zero, 2^17 of weight 2^-26.2, which make the output. They stand
    2^8 above where the 16-bit weights put the largest at least, 2^-18.2: half a step there is 2^-25,
    2^-6.8 of the weight, and all of them are rounded alike."""
    N, step = 1 << 17, 26.2
    c = Cache([N], 1, 64, 128)
    c.k[:], c.v[:], c.ks[:], c.vs[:] = 0, 127, 1 / 127, 1
    first = int(c.table[0, 0])
    c.k[first, 0, 0, 0], c.v[first, 0, 0] = 127, 0
    q = torch.zeros(new, 64, 64, device=DEV, dtype=F16)
    q[..., 0] = 1
    got = sl8.attn_paged_block8(q, *c.args(), i32([N]), cu_lens=offsets([new]), scale=step / LOG2E, rotate=False)
    tail = (torch.arange(N - new, N, device=DEV, dtype=torch.float64) * 2.0 ** -step)[:, None, None]
    want = 127 * tail / (1 + tail)
    assert float(((got.double() - want) / want).abs().max()) <= 2.0 ** -6


def test_empty_calls():
    c = Cache([20], 2, 64, 16)
    q = torch.zeros(0, 4, 64, device=DEV, dtype=F16)
    assert sl8.attn_paged_block8(q, *c.args()[:4], c.table[:0], i32([]).int()).shape == q.shape
    q = torch.ones(3, 4, 64, device=DEV, dtype=F16)
    out = sl8.attn_paged_block8(q, *c.args()[:4], c.table[:0], i32([]), cu_lens=i32([0]))
    assert not out.any()
    out = sl8.attn_paged_block8(q, *c.args(), i32([20]), cu_lens=i32([0, 0]))
    assert not out.any()
    assert sl8.attn_paged_block8(q[:, :0], *c.args(), i32([20]), cu_lens=i32([0, 3])).shape == (3, 0, 64)
    zero = sl8.attn_paged_block8(torch.zeros_like(q), *c.args(), i32([20]), cu_lens=i32([0, 3]), rotate=True)
    k, v, _ = c.rows(0, 1, 20)  # a query of zeros: the plain mean
    # weights of 20 equal keys: 2^-11 of sum p |v|, and the output's half step
    assert float((zero[2, 3].double() - v.mean(0)).abs().max()) <= 2.0 ** -10 * float(v.abs().max())


def test_offsets_past_32_bits():
    """A pool of more than 2^32 bytes whose last blocks hold the sequences."""
    D, bs, Hkv = 256, 128, 8
    nb = (1 << 32) // (D * bs * Hkv) + 40
    c = object.__new__(Cache)
    c.k, c.v = (torch.empty(nb, Hkv, bs, D, device=DEV, dtype=torch.int8) for _ in range(2))
    c.ks, c.vs = (torch.ones(nb, Hkv, device=DEV) for _ in range(2))
    c.bs = bs
    c.table = torch.arange(nb - 1, nb - 13, -1, device=DEV).int().view(2, 6)
    new, total = [300, 5], [700, 5]
    c.k[-12:].random_(-127, 128)
    c.v[-12:].random_(-127, 128)
    c.ks[-12:] = c.vs[-12:] = 3.5 / 127
    k, v = (torch.randn(305, Hkv, D, device=DEV).to(F16) for _ in range(2))
    pages = c.table.long()
    sl8.quantize_kv_append_block8(k, v, *c.args(), i32(total), cu_lens=offsets(new), rotate=False)
    kk, vv, _ = c.rows(0, 7, 700)
    # half a step of the scale each
    assert float((kk[400:] - k[:300, 7].double()).abs().max()) <= 0.51 * float(c.ks[pages].max())
    assert float((vv[400:] - v[:300, 7].double()).abs().max()) <= 0.51 * float(c.vs[pages].max())
    attn_and_check(c, coded_queries(305, 16, D, F16, False), new, total)
    attn_and_check(c, coded_queries(2, 16, D, F16, False), [1, 1], total, cu=False)


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("rotate", [False, True])
@pytest.mark.parametrize("D,bs,dtype", [(64, 32, F16), (128, 16, BF16)])
def test_serving_run(rotate, D, bs, dtype):
    """Prompts in two chunks, then decode steps and a step of drafted tokens: each token's output stands
    within the int8 cache's error of full-precision attention of all tokens so far."""
    from tests.tolerances import cos_sim, rel_l1

    Hq, Hkv, B = 8, 2, 3
    steps = [[40, 100, 7], [33, 1, 64], [1, 1, 1], [1, 1, 1], [4, 4, 4], [1, 1, 1]]
    cap = [sum(s[b] for s in steps) for b in range(B)]
    c = Cache(cap, Hkv, D, bs)
    table = sl8.rope_table(400, D)
    seen = [[] for _ in range(B)]
    outs, refs, done = [], [], [0] * B
    for new in steps:
        T = sum(new)
        q, k, v = news(T, Hq, Hkv, D, dtype)
        done = [a + b for a, b in zip(done, new)]
        pos = torch.cat([torch.arange(n - m, n, device=DEV) for m, n in zip(new, done)])
        q1 = sl8.quantize_kv_append_block8(k, v, *c.args(), i32(done), cu_lens=offsets(new), q=q, positions=pos,
                                           table=table, rotate=rotate)
        outs.append(sl8.attn_paged_block8(q1, *c.args(), i32(done), cu_lens=offsets(new), rotate=rotate))
        qr, kr = (turned(x.transpose(0, 1)[None], pos[None, None], table, None, False, False)[0][0].transpose(0, 1)
                  for x in (q, k))
        t = 0
        for b, m in enumerate(new):
            seen[b].append((kr[t:t + m], v[t:t + m].double()))
            kk, vv = (torch.cat([s[i] for s in seen[b]]) for i in (0, 1))
            n = kk.shape[0]
            mask = torch.arange(n, device=DEV) > torch.arange(n - m, n, device=DEV)[:, None]
            ref = torch.empty(m, Hq, D, device=DEV, dtype=torch.float64)
            for h in range(Hq):
                w = qr[t:t + m, h] @ kk[:, h // 4].T / math.sqrt(D)
                ref[:, h] = torch.softmax(w.masked_fill(mask, -math.inf), -1) @ vv[:, h // 4]
            refs.append(ref)
            t += m
    out, ref = torch.cat(outs), torch.cat(refs)
    # int8 rows of one scale per block: the bars of the int8 cache (tests of the per-token one)
    assert cos_sim(out, ref) >= 0.998 and rel_l1(out, ref) <= 0.05


def test_prompt_as_prefill():
    """A prompt's rows, rotated by `rope` and attended by attn_int8_fwd, agree with the cache's way."""
    from tests.tolerances import assert_int8_quality

    S, Hq, Hkv, D = 200, 8, 2, 128
    q, k, v = news(S, Hq, Hkv, D, F16)
    pos, table = torch.arange(S, device=DEV), sl8.rope_table(S, D)
    q4, k4 = (x.transpose(0, 1)[None] for x in (q, k))
    qr, kr = sl8.rope(q4, k4, pos, table)
    want = sl8.attn_int8_fwd(qr, kr, v.transpose(0, 1)[None].contiguous(), causal=True)
    c = Cache([S], Hkv, D, 16)
    q1 = sl8.quantize_kv_append_block8(k, v, *c.args(), i32([S]), cu_lens=i32([0, S]), q=q, positions=pos,
                                       table=table)
    assert torch.equal(q1.transpose(0, 1)[None], qr)
    got = sl8.attn_paged_block8(q1, *c.args(), i32([S]), cu_lens=i32([0, S]))
    assert_int8_quality(got.transpose(0, 1)[None], want, min_cos=0.998, max_rel_l1=0.05)


def test_decode_agrees_with_the_cache_of_token_scales():
    """One scale per block said once per token: the per-token cache's decode gives the same rows."""
    total = [333, 64, 5]
    c = Cache(total, 2, 128, 16)
    q = coded_queries(3, 8, 128, F16, False)
    got = attn_and_check(c, q, [1] * 3, total, cu=False)
    per_token = [s[:, :, None].expand(-1, -1, 16).contiguous() for s in (c.ks, c.vs)]
    table = c.table.clamp(min=0)
    want = sl8.attn_paged_decode_cached(q[:, :, None], c.k, per_token[0], c.v, per_token[1], table,
                                        i32(total), 16, rotate=False)[:, :, 0]
    # both within 2^-11 of sum p |v| (|v| <= 127 * 1.5 steps) and half an fp16 step each
    assert float((got.double() - want.double()).abs().max()) <= 2.0 ** -9 * 127 * 1.5 * 3.5 / 127


@pytest.mark.parametrize("new", [1, 3, 70])
def test_streams_and_repeats(new):
    """The same bits on another stream and again, two calls at once on two streams, and results that do
    not depend on where the blocks lie."""
    total = [900, 1300, 70]
    c = Cache(total, 2, 128, 16)
    q = coded_queries(3 * new, 8, 128, F16, False)
    cu, lens = offsets([new] * 3), i32(total)
    want = sl8.attn_paged_block8(q, *c.args(), lens, cu_lens=cu, rotate=False)
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in sides * 3:
        with torch.cuda.stream(s):
            got.append(sl8.attn_paged_block8(q, *c.args(), lens, cu_lens=cu, rotate=False))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    order = torch.randperm(c.k.shape[0], device=DEV)
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device=DEV)
    moved = sl8.attn_paged_block8(q, c.k[order], c.ks[order], c.v[order], c.vs[order],
                                  place[c.table.long().clamp(min=0)].int(), lens, cu_lens=cu, rotate=False)
    assert torch.equal(moved, want)


def test_step_in_a_graph():
    """A decode step captured once, replayed with new tokens, lengths and contexts; eager work between."""
    total = torch.tensor([100, 37, 640])
    c = Cache([200, 200, 800], 2, 128, 16)
    table = sl8.rope_table(1000, 128)
    q, k, v = (x.contiguous() for x in news(3, 8, 2, 128, F16))
    lens, pos = total.to(DEV).int(), total.to(DEV) - 1

    def step(c):
        q1 = sl8.quantize_kv_append_block8(k, v, *c.args(), lens, q=q, positions=pos, table=table)
        return sl8.attn_paged_block8(q1, *c.args(), lens)

    d = c.copy()
    step(c.copy())  # warm
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(c)
    for i in range(5):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, device=DEV))
        lens.add_(i * 7 % 5 + 1)
        pos.copy_(lens - 1)
        g.replay()
        torch.cuda.synchronize()
        want = step(d)
        assert torch.equal(out, want) and torch.equal(c.k, d.k) and torch.equal(c.vs, d.vs)


def test_two_graphs():
    """Two captured calls of different sizes replayed by turns: no memory between them is shared."""
    total = [1500, 800]
    c = Cache(total, 2, 128, 16)
    lens = i32(total)
    calls = [(coded_queries(2, 8, 128, F16, False), None), (coded_queries(140, 8, 128, F16, False), i32([0, 100, 140]))]
    want = [sl8.attn_paged_block8(q, *c.args(), lens, cu_lens=cu, rotate=False) for q, cu in calls]
    graphs, outs = [], []
    for q, cu in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(sl8.attn_paged_block8(q, *c.args(), lens, cu_lens=cu, rotate=False))
        graphs.append(g)
    for _ in range(3):
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_refusals():
    c = Cache([40, 40], 2, 64, 16)
    q, k, v = (x.contiguous() for x in news(2, 4, 2, 64, F16))
    lens, cu = i32([30, 30]), i32([0, 1, 2])
    pos, table = torch.zeros(2, device=DEV, dtype=torch.int32), torch.ones(5, 64, device=DEV)
    base = dict(k_cache=c.k, k_scale=c.ks, v_cache=c.v, v_scale=c.vs, block_table=c.table, context_lens=lens,
                cu_lens=cu)
    shared = [
        dict(k_cache=c.k.float()), dict(v_cache=c.v[:-1]), dict(k_cache=c.k[:, :1], v_cache=c.v[:, :1]),
        dict(k_cache=c.k[..., :32], v_cache=c.v[..., :32]), dict(k_cache=c.k[:, :, :8], v_cache=c.v[:, :, :8]),
        dict(k_scale=c.ks.double()), dict(v_scale=c.vs[:, :1]), dict(k_scale=c.ks[:, :, None].expand(-1, -1, 16)),
        dict(block_table=c.table.long()), dict(block_table=c.table[:1]), dict(context_lens=lens.long()),
        dict(context_lens=lens[None]), dict(cu_lens=cu.long()), dict(cu_lens=cu[:2]), dict(block_table=c.table.cpu()),
        dict(k_cache=c.k.transpose(0, 1).contiguous().transpose(0, 1)),
    ]
    for change in shared + [dict(q=q.float()), dict(q=q[0]), dict(q=q[:, :3]), dict(cu_lens=None, q=q[:1]),
                            dict(q=q.transpose(0, 1).contiguous().transpose(0, 1))]:
        with pytest.raises(RuntimeError, match="fni8"):
            _C.attn_paged_block8(**dict(q=q, q_mul=1.0, rotate=False) | base | change)
    turn = dict(q=q, positions=pos, table=table)
    for change in shared + [dict(k_new=k.float()), dict(v_new=v.to(BF16)), dict(k_new=k[:1]), dict(k_new=k[0]),
                            dict(q=q), dict(positions=pos), dict(turn, q=q.to(BF16)), dict(turn, q=q[:1]),
                            dict(turn, table=table[:, :40]), dict(turn, positions=pos[:1]),
                            dict(turn, sections=(32,)), dict(turn, positions=pos.float())]:
        with pytest.raises(RuntimeError, match="fni8"):
            _C.kv_append_block8(**dict(k_new=k, v_new=v) | base | change)
    for D, bs in ((96, 16), (32, 16), (64, 24), (64, 144)):
        bad = torch.zeros(4, 2, bs, D, device=DEV, dtype=torch.int8)
        sc = torch.ones(4, 2, device=DEV)
        x = torch.zeros(2, 2, D, device=DEV, dtype=F16)
        for call in (lambda: _C.attn_paged_block8(x, 1.0, False, bad, sc, bad, sc, c.table, lens),
                     lambda: _C.kv_append_block8(x, x, bad, sc, bad, sc, c.table, lens)):
            with pytest.raises(RuntimeError, match="fni8"):
                call()
