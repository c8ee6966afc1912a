"""Attention of drafted trees over the block-scaled paged cache, its rows' logarithms, and the keys' gathered
softmax weights, against plain 64-bit forms."""
import math

import pytest
import torch

import superl8_amd as sl8
from superl8_amd import _C
from tests.test_block8_gpu import BF16, DEV, F16, Cache, coded_queries, hadamard, i32, news, offsets

pytestmark = pytest.mark.gpu


def masks(new, words, some=0.5, rng=None):
    """Random masks, with no regard to trees: rows that see none of the new tokens, not themselves, later ones."""
    g = rng or torch.Generator().manual_seed(7)
    bits = [torch.rand(n, min(n, 64 * words), generator=g) < some for n in new]
    for b in bits:
        b[0] = False
        b[-1] = True
    return bits


def packed(bits, words):
    rows = []
    for b in bits:
        for r in b.tolist():
            x = sum(1 << j for j, on in enumerate(r) if on)
            w = [x >> (64 * k) & (1 << 64) - 1 for k in range(words)]
            rows.append([y - (1 << 64) if y >> 63 else y for y in w])
    return torch.tensor(rows, device=DEV, dtype=torch.int64).reshape(len(rows), words)


def plain(c, q, new, total, rotate, scale, window, bits=None):
    """The attention in 64 bits: out, sum p |v|, the largest p vs, ln of the sums, and the scores' softmax weights
    by key [B][Hkv, total] with the lse that it gives."""
    x = q.double()
    if rotate:
        x = x @ hadamard(q.shape[-1])
    qs = x.abs().amax(-1, keepdim=True) / 127
    qs = torch.where(qs == 0, 1.0, qs)
    x = torch.round(x / qs) * qs
    out, size, top = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x[..., :1])
    lse = torch.full(x.shape[:2], -math.inf, device=DEV, dtype=torch.float64)
    Hkv = c.k.shape[1]
    G = q.shape[1] // Hkv
    sums = [torch.zeros(Hkv, n, device=DEV, dtype=torch.float64) for n in total]
    t = 0
    for b, (m, n) in enumerate(zip(new, total)):
        old = n - m
        key = torch.arange(n, device=DEV)
        if bits is None:
            i = torch.arange(old, n, device=DEV)[:, None]
            seen = key <= i
            if window >= 0:
                seen = seen & (key > i - window)
        else:
            near = torch.zeros(m, m, dtype=torch.bool, device=DEV)
            near[:, :bits[b].shape[1]] = bits[b].to(DEV)
            far = torch.ones(m, old, dtype=torch.bool, device=DEV)
            if window >= 0:
                room = (window - near.sum(1)).clamp(min=0)
                far = far & (key[:old] >= old - room[:, None])
            seen = torch.cat([far, near], 1)
        for h in range(Hkv if m else 0):
            k, v, vs = c.rows(b, h, n)
            for j in range(h * G, h * G + G):
                w = (x[t:t + m, j] @ k.T * scale).masked_fill(~seen, -math.inf)
                p = torch.softmax(w, -1).nan_to_num(0.0)
                out[t:t + m, j], size[t:t + m, j] = p @ v, p @ v.abs()
                top[t:t + m, j] = (p * vs).amax(-1, keepdim=True)
                lse[t:t + m, j] = torch.logsumexp(w, -1)
                sums[b][h] += p.sum(0)
        t += m
    return out, size, top, lse, sums


def tree_and_check(c, q, new, total, bits, words=1, rotate=False, window=-1, cu=True):
    """Tolerances: the output's as for causal rows (weights in 16 bits 2^-11, exp2 and its argument 2^-15, N sums
    2^-24 each, weights below the 16-bit normals 2^-25 of the largest, the output's rounding); the logarithm's by
    what shifts a sum: scores of up to 2^7 in base 2 by 4 roundings (2^-15), N additions, its own rounding."""
    scale = q.shape[-1] ** -0.5
    got, lse = sl8.attn_paged_block8(q, *c.args(), i32(total), cu_lens=offsets(new) if cu else None, rotate=rotate,
                                     window_left=window, tree_mask=None if bits is None else packed(bits, words),
                                     return_lse=True)
    want, size, top, ln, _ = plain(c, q, new, total, rotate, scale, window, bits)
    N, eps = max(total), torch.finfo(q.dtype).eps / 2
    lim = size * (2.0 ** -11 + 2.0 ** -15 + N * 2.0 ** -24) + N * 127 * 2.0 ** -25 * top + \
        eps * (1 + 2.0 ** -8) * want.abs() + 2.0 ** -25
    assert got.dtype == q.dtype and got.shape == q.shape
    assert bool(((got.double() - want).abs() <= lim).all()), float(((got.double() - want).abs() - lim).max())
    assert lse.dtype == torch.float32 and lse.shape == q.shape[:2]
    none = ln == -math.inf
    assert torch.equal(lse == -math.inf, none)
    off = torch.where(none, 0.0, (lse.double() - ln).abs())
    assert bool((off <= 2.0 ** -15 + N * 2.0 ** -24 + 2.0 ** -22 * torch.where(none, 0.0, ln.abs())).all()), float(off.max())
    return got, lse


@pytest.mark.parametrize("D,Hq,Hkv,bs", [(64, 4, 1, 16), (64, 8, 8, 64), (128, 8, 2, 16), (128, 6, 2, 48),
                                         (128, 16, 2, 128), (256, 4, 4, 16), (256, 8, 1, 32)])
@pytest.mark.parametrize("most,words", [(3, 1), (17, 1), (64, 1), (65, 2), (130, 3), (256, 4), (70, 1)])
def test_tree(D, Hq, Hkv, bs, most, words):
    new = [most, max(1, most // 2), 1]
    total = [most + 211, most // 2 + 64, 1 + 130]
    c = Cache(total, Hkv, D, bs)
    q = coded_queries(sum(new), Hq, D, F16 if D != 128 else BF16, bs == 16)
    tree_and_check(c, q, new, total, masks(new, words), words, rotate=bs == 16)


@pytest.mark.parametrize("old", [0, 1, 15, 63, 64, 65, 1000])
@pytest.mark.parametrize("n", [1, 2, 40, 100])
def test_where_the_tree_begins(old, n):
    """Trees behind contexts of every phase of a tile, and with nothing in front."""
    c = Cache([old + n, n], 2, 64, 16)
    q = coded_queries(2 * n, 4, 64, F16, False)
    tree_and_check(c, q, [n, n], [old + n, n], masks([n, n], 2), 2)


@pytest.mark.parametrize("window", [0, 1, 5, 40, 130, 100000])
@pytest.mark.parametrize("D,G", [(64, 1), (128, 4), (256, 8)])
def test_window(window, D, G):
    new, total = [70, 9, 33], [70 + 500, 9 + 3, 33 + 64]
    c = Cache(total, 2, D, 32)
    q = coded_queries(sum(new), 2 * G, D, BF16, False)
    tree_and_check(c, q, new, total, masks(new, 2, 0.2), 2, window=window)


@pytest.mark.parametrize("B,n,old", [(1, 26, 5000), (2, 60, 9000), (70, 5, 300), (3, 130, 3000)])
def test_split_keys(B, n, old):
    total = [n + max(1, old // (1 + i)) for i in range(B)]
    c = Cache(total, 2, 128, 16)
    q = coded_queries(B * n, 8, 128, F16, True)
    tree_and_check(c, q, [n] * B, total, masks([n] * B, 3), 3, rotate=True)


@pytest.mark.parametrize("new", [[1, 1, 1], [7, 0, 20], [150, 3, 90]])
@pytest.mark.parametrize("window", [-1, 50])
def test_chain_is_causal(new, window):
    """Masks of chains, which with a window mark its last tokens only (what is marked is seen), give what causal rows
    give, each within its tolerance; lse without a mask."""
    total = [n + o for n, o in zip(new, (300, 40, 77))]
    c = Cache(total, 2, 128, 32)
    q = coded_queries(sum(new), 8, 128, F16, False)
    tree_and_check(c, q, new, total, None, window=window)
    chains = [torch.ones(n, n, dtype=torch.bool).tril().triu(1 - window if window >= 0 else -n) for n in new]
    got, lse = tree_and_check(c, q, new, total, chains, 3, window=window)
    same, ln = sl8.attn_paged_block8(q, *c.args(), i32(total), cu_lens=offsets(new), rotate=False, window_left=window,
                                     return_lse=True)
    assert torch.equal(same, sl8.attn_paged_block8(q, *c.args(), i32(total), cu_lens=offsets(new), rotate=False,
                                                   window_left=window))
    assert float((lse - ln).abs().nan_to_num(0.0).max()) <= 2.0 ** -14 + 2 * 500 * 2.0 ** -24 + 2.0 ** -18


def test_one_row_a_sequence_without_offsets():
    total = [90, 3, 1]
    c = Cache(total, 2, 64, 16)
    q = coded_queries(3, 4, 64, F16, False)
    bits = [torch.ones(1, 1, dtype=torch.bool), torch.zeros(1, 1, dtype=torch.bool), torch.zeros(1, 1, dtype=torch.bool)]
    got, lse = tree_and_check(c, q, [1] * 3, total, bits, cu=False)
    assert bool((got[2] == 0).all()) and bool((lse[2] == -math.inf).all())
    one = sl8.attn_paged_block8(q, *c.args(), i32(total), rotate=False, tree_mask=packed(bits, 1)[:, 0])
    assert torch.equal(one, got)


def test_rows_of_no_sequence_and_short_contexts():
    """Padding rows in front and behind: zeros and -inf, whatever their masks; contexts shorter than the new tokens
    and below 0 are answered without a fault; blocks outside the pool are not there."""
    c = Cache([60, 50], 2, 128, 16)
    q = coded_queries(40, 4, 128, F16, False)
    cu = i32([5, 15, 30])
    mask = torch.full((40, 2), -1, device=DEV, dtype=torch.int64)
    out, lse = sl8.attn_paged_block8(q, *c.args(), i32([60, 50]), cu_lens=cu, rotate=False, tree_mask=mask, return_lse=True)
    rest = torch.ones(40, dtype=torch.bool, device=DEV)
    rest[5:30] = False
    assert bool((out[rest] == 0).all()) and bool((lse[rest] == -math.inf).all())
    assert bool(torch.isfinite(lse[~rest]).all())
    for lens in ([4, 2], [-7, 0], [2 ** 31 - 1, 60]):
        out, lse = sl8.attn_paged_block8(q, *c.args(), i32(lens), cu_lens=cu, rotate=False, tree_mask=mask, return_lse=True)
        assert bool(torch.isfinite(out).all()) and not bool(torch.isnan(lse).any())
    c.table[0, 1] = 10 ** 6
    got, _ = sl8.attn_paged_block8(q, *c.args(), i32([60, 50]), cu_lens=cu, rotate=False, tree_mask=mask, return_lse=True)
    assert bool(torch.isfinite(got).all())
    out, lse = sl8.attn_paged_block8(q[:0], *c.args(), i32([60, 50]), cu_lens=i32([0, 0, 0]), rotate=False,
                                     tree_mask=mask[:0], return_lse=True)
    assert out.shape == (0, 4, 128) and lse.shape == (0, 4)


def test_masks_from_parents():
    parents = [-1, 0, 0, 1, 2, 2, 3, -1, 0, 1, 2, 3, 4]  # a tree of 7, then one of 6
    got = sl8.tree_mask(torch.tensor(parents, device=DEV), i32([0, 7, 13]), words=2)
    for t, (first, n) in enumerate([(0, 7)] * 7 + [(7, 6)] * 6):
        want, at = 0, t - first
        while at >= 0:
            want |= 1 << at
            at = parents[first + at]
        assert got[t].tolist() == [want, 0]
    n = 200  # a chain over words
    got = sl8.tree_mask(torch.arange(-1, n - 1, device=DEV, dtype=torch.int32), words=4)
    assert torch.equal(got, packed([torch.ones(n, n, dtype=torch.bool).tril()], 4))
    assert sl8.tree_mask(torch.tensor([5, -3, 1])).tolist() == [[1], [2], [6]]  # (a parent that is not there: none)


# ---------------------------------------------------------------------------
# the keys' weights
# ---------------------------------------------------------------------------
def weights_and_check(c, q, new, total, rotate=False, window=-1, decay=1.0, cu=True, strided=False):
    """Tolerance, relative: scores of up to 2^7 in base 2 by 4 roundings and the lse's product (2^-15), exp2, R
    additions (R * 2^-24), and the rounding of the fading; what 32 bits have no normal number for is nothing."""
    B, Hkv, cap = len(new), c.k.shape[1], c.table.shape[1] * c.bs
    scale = q.shape[-1] ** -0.5
    _, _, _, lse, sums = plain(c, q, new, total, rotate, scale, window)
    lse32 = lse.float()
    # what the rounded lse makes of the sums: relative 2^-24 of |lse|
    weights = torch.rand(B, Hkv, cap + 3, device=DEV)
    if strided:
        weights = torch.rand(Hkv, B, cap + 8, device=DEV).transpose(0, 1)[..., 5:]
    was = weights.clone()
    sl8.attn_weights_block8(q, lse32, c.k, c.ks, c.table, i32(total), weights, cu_lens=offsets(new) if cu else None,
                            rotate=rotate, window_left=window, decay=decay)
    R = max(new) * q.shape[1] // Hkv
    big = float(lse[lse.isfinite()].abs().max()) if bool(lse.isfinite().any()) else 0.0
    for b, (m, n) in enumerate(zip(new, total)):
        old = was[b, :, :n].double() * decay
        old[:, n - m:] = 0
        want = old + sums[b]
        lim = sums[b] * (2.0 ** -15 + R * 2.0 ** -24 + big * 2.0 ** -23) + want * 2.0 ** -22 + 2.0 ** -120
        err = (weights[b, :, :n].double() - want).abs()
        assert bool((err <= lim).all()), (b, float((err - lim).max()), float(err.max()))
        assert torch.equal(weights[b, :, n:], was[b, :, n:])
    return weights


@pytest.mark.parametrize("D,Hq,Hkv,bs", [(64, 4, 4, 16), (64, 8, 1, 48), (128, 8, 2, 16), (128, 6, 2, 128),
                                         (256, 8, 2, 32)])
@pytest.mark.parametrize("new", [[1, 1, 1], [5, 1, 0], [40, 7, 33], [300, 2, 129]])
@pytest.mark.parametrize("decay,window", [(1.0, -1), (0.9, 37)])
def test_weights(D, Hq, Hkv, bs, new, decay, window):
    total = [n + o for n, o in zip(new, (200, 63, 1))]
    c = Cache(total, Hkv, D, bs)
    q = coded_queries(sum(new), Hq, D, F16 if D == 128 else BF16, bs == 16)
    weights_and_check(c, q, new, total, rotate=bs == 16, window=window, decay=decay, strided=bs == 16)


@pytest.mark.parametrize("B", [1, 63, 65, 200])
def test_weights_of_many_sequences(B):
    total = [1 + 37 * i % 301 for i in range(B)]
    c = Cache(total, 2, 64, 16)
    q = coded_queries(B, 4, 64, F16, False)
    weights_and_check(c, q, [1] * B, total, cu=False)


@pytest.mark.parametrize("new", [1, 33, 1100])
def test_weights_of_long_contexts(new):
    c = Cache([new + 3000], 2, 128, 32)
    q = coded_queries(new, 8, 128, BF16, False)
    weights_and_check(c, q, [new], [new + 3000], window=2000 if new == 33 else -1)


@pytest.mark.parametrize("new", [1, 40, 700])
def test_unread_places(new):
    """Scales and codes that no key has do not matter: NaN in blocks of no sequence (the pool's first among them), old
    codes behind a context's end, table entries past it."""
    total = [new + 37, new + 5]
    c = Cache(total, 2, 64, 16)
    used = {x for b, n in enumerate(total) for x in c.table[b, :-(-n // 16)].tolist()}
    if 0 in used:  # the pool's first block is nobody's
        spare = next(i for i in range(c.k.shape[0]) if i not in used)
        c.table[c.table == 0] = spare
        for t in (c.k, c.ks, c.v, c.vs):
            t[spare] = t[0]
        used = (used - {0}) | {spare}
    free = [i for i in range(c.k.shape[0]) if i not in used]
    c.ks[free] = math.nan
    c.table[1, -1] = 0
    q = coded_queries(2 * new, 4, 64, F16, False)
    w = weights_and_check(c, q, [new, new], total, window=20 if new == 40 else -1)
    assert bool(torch.isfinite(w).all())
    c.table[0, 0] = -1  # keys that are not there
    lse = torch.zeros(2 * new, 4, device=DEV)
    sl8.attn_weights_block8(q, lse, c.k, c.ks, c.table, i32(total), w, cu_lens=offsets([new, new]), rotate=False)
    assert bool(torch.isfinite(w).all())


def test_weights_sum_to_the_rows():
    """With the lse of the attention itself each row's weights add up to 1."""
    new, total = [70, 1], [400, 90]
    c = Cache(total, 2, 128, 16)
    q, _, _ = (x.contiguous() for x in news(71, 8, 2, 128, F16))
    _, lse = sl8.attn_paged_block8(q, *c.args(), i32(total), cu_lens=offsets(new), return_lse=True)
    w = torch.zeros(2, 2, c.table.shape[1] * 16, device=DEV)
    sl8.attn_weights_block8(q, lse, c.k, c.ks, c.table, i32(total), w, cu_lens=offsets(new))
    got = w.double().sum(-1)
    # (a code next to a half may differ between the two: 2^-10 of a row, one in a thousand rows)
    want = torch.tensor([[280.0], [4.0]], device=DEV, dtype=torch.float64)
    assert bool(((got - want).abs() <= want * 2.0 ** -10).all())


def test_weights_leave_alone_what_is_not_there():
    """Rows of lse -inf, blocks outside the pool, contexts of 0 and below, rows of no sequence."""
    c = Cache([50, 40, 30], 2, 64, 16)
    q = coded_queries(6, 4, 64, F16, False)
    w = torch.rand(3, 2, c.table.shape[1] * 16, device=DEV)
    was = w.clone()
    lse = torch.full((6, 4), -math.inf, device=DEV)
    sl8.attn_weights_block8(q, lse, c.k, c.ks, c.table, i32([50, 0, -3]), w, cu_lens=i32([1, 3, 4, 5]), rotate=False)
    assert torch.equal(w[0, :, :48], was[0, :, :48]) and bool((w[0, :, 48:50] == 0).all())
    assert torch.equal(w[0, :, 50:], was[0, :, 50:]) and torch.equal(w[1:], was[1:])
    c.table[0, 1] = -1
    w2 = was.clone()
    sl8.attn_weights_block8(q, torch.zeros_like(lse), c.k, c.ks, c.table, i32([50, 40, 30]), w2,
                            cu_lens=i32([0, 2, 4, 6]), rotate=False)
    assert torch.equal(w2[0, :, 16:32], was[0, :, 16:32]) and not torch.equal(w2[0, :, :16], was[0, :, :16])
    sl8.attn_weights_block8(q[:0], lse[:0], c.k, c.ks, c.table, i32([50, 40, 30]), w2, cu_lens=i32([0] * 4), decay=0.5)
    sl8.attn_weights_block8(q[:0], lse[:0], c.k, c.ks, c.table[:0], i32([]), w2[:0], cu_lens=i32([0]))


def test_streams_and_repeats():
    """The same bits again, on other streams and two at once; where the blocks lie does not matter."""
    new, total = [30, 90], [900, 1200]
    c = Cache(total, 2, 128, 16)
    q = coded_queries(120, 8, 128, F16, False)
    bits = masks(new, 2)
    mask, cu, lens = packed(bits, 2), offsets(new), i32(total)

    def run():
        out, lse = sl8.attn_paged_block8(q, *c.args(), lens, cu_lens=cu, rotate=False, tree_mask=mask, return_lse=True)
        w = torch.ones(2, 2, c.table.shape[1] * 16, device=DEV)
        sl8.attn_weights_block8(q, lse, c.k, c.ks, c.table, lens, w, cu_lens=cu, rotate=False, decay=0.5)
        return out, lse, w

    want = run()
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(2)] * 2:
        with torch.cuda.stream(s):
            got.append(run())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


def test_in_a_graph():
    """Captured once, replayed with other queries, masks and lengths; eager work between."""
    total = torch.tensor([300, 120])
    c = Cache([400, 400], 2, 128, 16)
    q = coded_queries(40, 8, 128, F16, False)
    mask = packed(masks([25, 15], 1), 1)
    cu, lens = i32([0, 25, 40]), total.to(DEV).int()
    w = torch.rand(2, 2, c.table.shape[1] * 16, device=DEV)

    def step(w):
        out, lse = sl8.attn_paged_block8(q, *c.args(), lens, cu_lens=cu, tree_mask=mask, return_lse=True)
        sl8.attn_weights_block8(q, lse, c.k, c.ks, c.table, lens, w, cu_lens=cu, decay=0.5)
        return out, lse

    step(w.clone())
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step(w)
    for i in range(4):
        q.copy_(torch.randn(q.shape, device=DEV))
        mask.copy_(packed(masks([25, 15], 1, 0.3 + 0.1 * i), 1))
        lens.add_(i)
        w2 = w.clone()
        g.replay()
        torch.cuda.synchronize()
        want = step(w2)
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(w, w2)


def test_refusals():
    c = Cache([40, 40], 2, 64, 16)
    q = torch.zeros(2, 4, 64, device=DEV, dtype=F16)
    mask, lens, cu = torch.ones(2, 1, device=DEV, dtype=torch.int64), i32([30, 30]), i32([0, 1, 2])
    base = dict(q=q, q_mul=1.0, rotate=False, k_cache=c.k, k_scale=c.ks, v_cache=c.v, v_scale=c.vs,
                block_table=c.table, context_lens=lens, cu_lens=cu, tree_mask=mask)
    for change in [dict(tree_mask=mask.int()), dict(tree_mask=mask[:1]), dict(tree_mask=mask.expand(2, 5)),
                   dict(tree_mask=mask[:, :0]), dict(tree_mask=mask[None]), dict(tree_mask=mask.cpu()),
                   dict(q=q.float()), dict(cu_lens=cu[:2])]:
        with pytest.raises(RuntimeError, match="fni8"):
            _C.attn_paged_block8(**base | change)
    w, lse = torch.ones(2, 2, c.table.shape[1] * 16, device=DEV), torch.zeros(2, 4, device=DEV)
    base = dict(q=q, q_mul=1.0, rotate=False, lse=lse, k_cache=c.k, k_scale=c.ks, block_table=c.table,
                context_lens=lens, weights=w, cu_lens=cu)
    for change in [dict(lse=lse.double()), dict(lse=lse[:1]), dict(lse=lse[:, :2]), dict(lse=lse.cpu()),
                   dict(weights=w.double()), dict(weights=w[:1]), dict(weights=w[:, :1]), dict(weights=w[..., :-1]),
                   dict(weights=w[:1].expand(2, -1, -1)), dict(weights=w[:, :1].expand(-1, 2, -1)),
                   dict(weights=w.transpose(1, 2).contiguous().transpose(1, 2)), dict(weights=w.cpu()),
                   dict(decay=math.inf), dict(decay=math.nan), dict(q=q.float()), dict(q=q[:, :3]),
                   dict(k_cache=c.k.float()), dict(context_lens=lens.long()), dict(cu_lens=None, q=q[:1], lse=lse[:1])]:
        with pytest.raises(RuntimeError, match="fni8"):
            _C.attn_weights_block8(**base | change)
    for bad in (torch.zeros(3), torch.zeros(2, 2, dtype=torch.int32)):
        with pytest.raises(ValueError, match="parents"):
            sl8.tree_mask(bad)
    with pytest.raises(ValueError, match="words"):
        sl8.tree_mask(torch.zeros(2, dtype=torch.int32), words=5)


@pytest.mark.parametrize("window", [-1, 30])
@pytest.mark.parametrize("n", [1, 5, 64, 90])
def test_bits_of_tokens_that_are_not_there(n, window):
    """They count for nothing, for a window either."""
    c = Cache([n + 200, n], 2, 128, 16)
    q = coded_queries(2 * n, 8, 128, F16, False)
    bits = masks([n, n], 3)
    clean = packed(bits, 3)
    stray = clean.clone()
    for w in range(3):
        there = max(0, min(64, n - 64 * w))
        stray[:, w] |= 0 if there == 64 else -1 << there
    args = dict(cu_lens=offsets([n, n]), rotate=False, window_left=window, return_lse=True)
    want = sl8.attn_paged_block8(q, *c.args(), i32([n + 200, n]), tree_mask=clean, **args)
    got = sl8.attn_paged_block8(q, *c.args(), i32([n + 200, n]), tree_mask=stray, **args)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("new,old,Hkv,window", [([130], [3000], 1, -1), ([300, 20], [40, 5000], 2, -1), ([600], [0], 1, -1),
                                                ([260], [1500], 1, 100), ([140, 0, 140], [700, 9, 80], 1, -1)])
def test_weights_of_rows_in_parts(new, old, Hkv, window):
    """Few items of many rows: behind long and short contexts, where parts end inside a token's heads or hold none."""
    total = [n + o for n, o in zip(new, old)]
    c = Cache(total, Hkv, 64, 16)
    q = coded_queries(sum(new), 10 * Hkv, 64, F16, False)
    weights_and_check(c, q, new, total, window=window, decay=0.5)


# ---------------------------------------------------------------------------
# each row's weights alone
# ---------------------------------------------------------------------------
def row_sums(c, q, lens, rotate, window=-1, lse=None):
    """What each row's weights add up to, heads apart (as many query heads as KV heads, a row a sequence)."""
    B, H, _ = q.shape
    if lse is None:
        _, lse = sl8.attn_paged_block8(q, *c.args(), lens, rotate=rotate, window_left=window, return_lse=True)
    w = torch.zeros(B, H, c.table.shape[1] * c.bs, device=DEV)
    sl8.attn_weights_block8(q, lse, c.k, c.ks, c.table, lens, w, rotate=rotate, window_left=window, decay=0.0)
    return w.double().sum(-1), lse


def sums_are_one(sums, lse, N):
    """The same codes and exact products on both sides; each score rounds 4 times at up to 2^7 in base 2 (2^-15, and
    again in the sum that lse is of), exp2 on both sides and N additions (N * 2^-24 each), lse itself and its
    product 2^-23 of its size."""
    lim = 2 * 2.0 ** -15 + 2 * N * 2.0 ** -24 + lse.double().abs() * 2.0 ** -22
    off = (sums - 1).abs()
    assert bool((off <= lim).all()), (float(off.max()), int((off > lim).sum()))


@pytest.mark.parametrize("rotate", [True, False])
@pytest.mark.parametrize("D,H", [(64, 32), (128, 16), (256, 8)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_weights_of_each_row_sum_to_one(D, H, dtype, rotate):
    """Single tokens of a thousand sequences on shared blocks: the codes of every row are those that its lse is of."""
    c = Cache([90, 33], H, D, 16)
    B = 1024
    c.table = c.table[torch.arange(B, device=DEV) % 2].contiguous()
    lens = torch.where(torch.arange(B, device=DEV) % 2 == 0, 90, 33).int()
    q = torch.randn(B, H, D, device=DEV).to(dtype)
    sums_are_one(*row_sums(c, q, lens, rotate), 90)


@pytest.mark.parametrize("D,G,n,window", [(64, 4, 300, -1), (128, 1, 700, -1), (128, 8, 260, 70), (256, 2, 300, -1),
                                          (256, 1, 40, -1)])
def test_weights_of_a_prompt_sum_to_one(D, G, n, window):
    """A prompt's rows in tiles, then each alone behind what it sees."""
    H, total = 8, n + 50
    c = Cache([total], H // G, D, 16)
    q = torch.randn(n, H, D, device=DEV).to(F16)
    _, lse = sl8.attn_paged_block8(q, *c.args(), i32([total]), cu_lens=offsets([n]), window_left=window, return_lse=True)
    d = c.copy()  # the KV head of each query head, as one of its own
    for name in ("k", "ks", "v", "vs"):
        setattr(d, name, getattr(c, name).repeat_interleave(G, 1).contiguous())
    d.table = c.table.expand(n, -1).contiguous()
    lens = torch.arange(total - n + 1, total + 1, device=DEV, dtype=torch.int32)
    sums_are_one(*row_sums(d, q, lens, True, window, lse), total)


@pytest.mark.parametrize("cu", [False, True])
@pytest.mark.parametrize("decay,window", [(0.9, -1), (1.0, 100)])
def test_weights_of_more_items_than_are_resident(decay, window, cu):
    """Single tokens, a wave an item: each wave takes several, and with a window skips some."""
    total = [1 + 1500 + 401 * i % 700 for i in range(130)]
    c = Cache(total, 8, 64, 32)
    q = coded_queries(130, 8, 64, F16, False)
    weights_and_check(c, q, [1] * 130, total, window=window, decay=decay, cu=cu)


@pytest.mark.parametrize("decay,window", [(0.9, -1), (1.0, 100)])
@pytest.mark.parametrize("n", [44, 70])
def test_weights_of_more_shared_items_than_are_resident(n, decay, window):
    """The same with four waves an item, sequences without new rows and with few among the others."""
    new = [(n, n - 3, 2 * n, n, 0, n, 1)[i % 7] for i in range(70)]
    total = [m + 300 + 401 * i % 700 for i, m in enumerate(new)]
    c = Cache(total, 8, 64, 32)
    q = coded_queries(sum(new), 8, 64, F16, False)
    weights_and_check(c, q, new, total, window=window, decay=decay)


@pytest.mark.parametrize("new,old", [([1200] + [1] * 66, 100), ([1] * 40 + [300] + [1] * 200, 60)])
def test_weights_of_a_prompt_beside_single_tokens(new, old):
    """On average many rows a sequence (four waves an item), and few (one)."""
    total = [n + old + 37 * i % 900 for i, n in enumerate(new)]
    c = Cache(total, 2, 128, 16)
    q = coded_queries(sum(new), 8, 128, F16, False)
    weights_and_check(c, q, new, total, decay=0.5)
