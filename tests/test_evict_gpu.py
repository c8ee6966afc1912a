"""Eviction from the block-scaled paged cache: what stays, where it goes, what is left alone; and a run of the
operators together."""
import math

import pytest
import torch

import superl8_amd as sl8
from superl8_amd import _C
from tests.test_block8_gpu import DEV, F16, Cache, i32, news, offsets
from tests.test_tree_gpu import packed

pytestmark = pytest.mark.gpu


class Room(Cache):
    """A pool for sequences of `cap` tokens, with blocks for `budget` of each beside theirs."""

    def __init__(self, cap, budget, Hkv, D, bs):
        super().__init__(cap, Hkv, D, bs, spare=sum(-(-min(n, budget) // bs) for n in cap) + 2)
        free = sorted(set(range(self.k.shape[0])) - {x for r in self.table.tolist() for x in r})
        need = [-(-min(n, budget) // bs) for n in cap]
        self.to = torch.full((len(cap), max(1, -(-min(budget, self.table.shape[1] * bs) // bs))), -1, device=DEV,
                             dtype=torch.int32)
        for b, n in enumerate(need):
            self.to[b, :n] = i32([free.pop() for _ in range(n)])


def kept_of(w, n, budget, sinks, recent):
    """The indexes that stay of n weights (a list), from the definition."""
    if n <= budget:
        return list(range(n))
    between = sorted(range(sinks, n - recent), key=lambda i: (-w[i], i))[:budget - sinks - recent]
    return list(range(sinks)) + sorted(between) + list(range(n - recent, n))


def evict_and_check(c, lens, weights, budget, sinks=0, recent=0):
    """Every index, weight, code and scale, equal: a scale is a maximum, a quotient and a product of an integer
    below 128 round once each, and the product's half steps are those of the quotient's rounding."""
    was, old = c.copy(), weights.clone()
    new_lens, kept = sl8.kv_evict_block8(*c.args(), i32(lens), weights, c.to, budget=budget, sinks=sinks, recent=recent)
    bs, Hkv = c.bs, c.k.shape[1]
    k, ks, v, vs = (t.clone() for t in (was.k, was.ks, was.v, was.vs))
    assert new_lens.tolist() == [max(0, min(n, budget)) for n in lens]
    for b, n in enumerate(lens):
        for h in range(Hkv):
            keep = kept_of(old[b, h, :max(n, 0)].tolist(), max(n, 0), budget, sinks, recent)
            m = len(keep)
            assert kept[b, h].tolist() == keep + [-1] * (budget - m), (b, h)
            at = torch.tensor(keep, device=DEV, dtype=torch.long)
            old[b, h, :m] = old[b, h, at] + 0.0  # (-0 comes back as 0)
            page = was.table[b].long()[at // bs]
            for codes, scales, c0, s0 in ((k, ks, was.k, was.ks), (v, vs, was.v, was.vs)):
                rows, sc = c0[page, h, at % bs].float(), s0[page, h]
                for i in range(0, m, bs):
                    to, s = int(c.to[b, i // bs]), sc[i:i + bs]
                    top = s.max().clamp_min(2.0 ** -60)
                    scales[to, h] = top
                    codes[to, h, :len(s)] = torch.round(rows[i:i + bs] * (s / top)[:, None]).to(torch.int8)
    assert torch.equal(weights, old)
    for name, got, want in (("k_scale", c.ks, ks), ("v_scale", c.vs, vs), ("k", c.k, k), ("v", c.v, v)):
        assert torch.equal(got, want), name
    return new_lens, kept


def weights_for(c, extra=0):
    return torch.rand(c.table.shape[0], c.k.shape[1], c.table.shape[1] * c.bs + extra, device=DEV).log().neg()


@pytest.mark.parametrize("D,Hkv,bs", [(64, 1, 16), (64, 3, 128), (128, 2, 16), (128, 2, 48), (256, 2, 32), (256, 1, 112)])
@pytest.mark.parametrize("budget,sinks,recent", [(1, 0, 0), (1, 0, 1), (40, 4, 9), (64, 0, 0), (100, 100, 0),
                                                 (97, 0, 97), (97, 1, 95), (1000, 3, 5)])
def test_evict(D, Hkv, bs, budget, sinks, recent):
    lens = [211, 97, 1, 0, 160]
    c = Room(lens, budget, Hkv, D, bs)
    evict_and_check(c, lens, weights_for(c, 3), budget, sinks, recent)


@pytest.mark.parametrize("n,budget", [(4096, 1000), (4097, 4096), (5000, 3), (16384, 5001), (20000, 19999),
                                      (32768, 2048), (33000, 700), (40000, 39990)])
def test_lengths(n, budget):
    """From lengths held in registers to those that are read again."""
    lens = [n, n // 3]
    c = Room([n, n // 3], budget, 1, 64, 64)
    evict_and_check(c, lens, weights_for(c), budget, min(5, budget), min(100, budget // 2 - 1) if budget > 100 else 0)


@pytest.mark.parametrize("n", [300, 5000, 34000])
@pytest.mark.parametrize("values", [[0.0], [1.0, 1.0, 2.0], [0.0, -0.0, 1e-38, -1e-38], [-3.0, 5.0, math.inf, -math.inf],
                                    [1e-45, 3e38, 1.0]])
def test_ties_and_odd_values(n, values):
    """Equal weights: the lowest indexes stay; zeros of both signs, subnormal, negative and infinite ones."""
    c = Room([n], n // 2, 2, 64, 32)
    w = torch.tensor(values, device=DEV)[torch.randint(0, len(values), (1, 2, c.table.shape[1] * 32), device=DEV)]
    evict_and_check(c, [n], w, n // 2, 2, 7)


def test_weights_that_differ_in_a_bit():
    """Weights next to each other in 32 bits, where bins have to be told apart to the last."""
    n = 3000
    c = Room([n], 1234, 1, 64, 16)
    bits = (torch.randperm(c.table.shape[1] * 16, device=DEV) // 3 + 0x3F800000).to(torch.int32)
    evict_and_check(c, [n], bits.view(torch.float32).reshape(1, 1, -1).contiguous(), 1234)


def test_nan_weights_fault_nothing():
    """No meaning, but indexes in their ranges, ascending, as many as the budget."""
    n = 2000
    c = Room([n], 700, 1, 64, 16)
    w = weights_for(c)
    w[0, 0, ::3] = math.nan
    lens, kept = sl8.kv_evict_block8(*c.args(), i32([n]), w, c.to, budget=700)
    assert lens.tolist() == [700] and bool((kept[0, 0].diff() > 0).all())
    assert int(kept.min()) >= 0 and int(kept.max()) < n


def test_scales_far_apart_and_equal():
    """Rows from blocks of scales far apart lose what their block's largest hides; of equal scales none."""
    n = 600
    c = Room([n], 300, 2, 128, 16)
    c.ks *= 2.0 ** torch.randint(-20, 20, c.ks.shape, device=DEV).float()
    c.ks[c.table[0, 3]] = 0
    c.vs[:] = 0.03
    evict_and_check(c, [n], weights_for(c), 300, 20, 20)
    # in a second round of the same budget nothing changes
    c.table, c.to = c.to, c.table
    d = c.copy()
    new, kept = sl8.kv_evict_block8(*c.args(), i32([300]), weights_for(c), c.to, budget=300)
    assert kept[0, 0].tolist() == list(range(300))
    a, b = c.table[0].long(), c.to[0].long()
    m = 300 // 16 * 16
    assert torch.equal(c.k[a].transpose(1, 2).flatten(0, 1)[:m], c.k[b].transpose(1, 2).flatten(0, 1)[:m])
    assert torch.equal(c.ks[a][:18], c.ks[b][:18]) and torch.equal(d.k[a], c.k[a])


def test_what_is_not_there():
    """Source blocks outside the pool arrive as zeros; destinations outside it are not written; lengths past
    the table end there; nothing is evicted from empty batches."""
    c = Room([200, 100], 50, 1, 64, 16)
    c.table[0, 2], c.table[1, 0] = -1, 10 ** 6
    d, w = c.copy(), weights_for(c)
    lens, kept = sl8.kv_evict_block8(*c.args(), i32([200, 100]), w, c.to, budget=50)
    for b in range(2):
        for i, j in enumerate(kept[b, 0].tolist()):
            if j // 16 == (2, 0)[b]:
                assert bool((c.k[c.to[b, i // 16].long(), 0, i % 16] == 0).all())
    bad = d.copy()
    bad.to = torch.full_like(d.to, 10 ** 6)
    bad.to[1] = -5
    sl8.kv_evict_block8(*bad.args(), i32([200, 100]), weights_for(bad), bad.to, budget=50)
    assert torch.equal(bad.k, d.k) and torch.equal(bad.vs, d.vs)
    cap = d.table.shape[1] * 16
    lens, _ = sl8.kv_evict_block8(*d.args(), i32([2 ** 31 - 1, -9]), weights_for(d), d.to, budget=50)
    assert lens.tolist() == [50, 0] and cap > 50
    lens, kept = sl8.kv_evict_block8(*d.args()[:4], d.table[:0], i32([]), w[:0], d.to[:0], budget=5)
    assert lens.shape == (0,) and kept.shape == (0, 1, 5)


def test_streams_graphs_and_strides():
    lens = [900, 333]
    c = Room(lens, 128, 2, 128, 16)
    w = torch.rand(2, 2, c.table.shape[1] * 16 + 40, device=DEV).transpose(0, 1)[..., 7:]
    d, e = c.copy(), c.copy()
    w0 = w.clone()
    want = evict_and_check(d, lens, w0, 128, 3, 11)
    n = i32(lens)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    w1 = w.clone()
    with torch.cuda.stream(s):
        got = sl8.kv_evict_block8(*e.args(), n, w1, e.to, budget=128, sinks=3, recent=11)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(w1, w0) and torch.equal(e.k, d.k)
    g = torch.cuda.CUDAGraph()
    w2 = w.clone()
    with torch.cuda.graph(g):
        out = sl8.kv_evict_block8(*c.args(), n, w2, c.to, budget=128, sinks=3, recent=11)
    for i in range(4):
        w2.copy_(torch.rand(w2.shape, device=DEV))
        n.sub_(i)
        w3 = w2.clone()
        g.replay()
        torch.cuda.synchronize()
        want = sl8.kv_evict_block8(*d.args(), n, w3, d.to, budget=128, sinks=3, recent=11)
        assert all(torch.equal(a, b) for a, b in zip(out, want)) and torch.equal(w2, w3)
        assert torch.equal(c.k[c.to.long()], d.k[d.to.long()]) and torch.equal(c.vs, d.vs)


def test_refusals():
    c = Room([90, 40], 32, 2, 64, 16)
    w, lens = weights_for(c), i32([90, 40])
    base = dict(k_cache=c.k, k_scale=c.ks, v_cache=c.v, v_scale=c.vs, block_table=c.table, context_lens=lens,
                weights=w, new_table=c.to, budget=32)
    for change in [dict(budget=0), dict(budget=-1), dict(sinks=-1), dict(recent=-1), dict(sinks=20, recent=13),
                   dict(new_table=c.to[:, :1]), dict(new_table=c.to.long()), dict(new_table=c.to[:1]),
                   dict(new_table=c.to[0]), dict(new_table=c.to.cpu()), dict(weights=w.half()), dict(weights=w[..., :50]),
                   dict(weights=w[:1].expand(2, -1, -1)), dict(k_cache=c.k.float()), dict(v_cache=c.v[:-1]),
                   dict(k_scale=c.ks[:, :1]), dict(block_table=c.table.long()), dict(context_lens=lens[:1]),
                   dict(k_cache=c.k[0])]:
        with pytest.raises(RuntimeError, match="fni8"):
            _C.kv_evict_block8(**base | change)


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("rotate", [False, True])
def test_drafting_run(rotate):
    """A layer as a server runs it: int8 projections of Q, K and V, a tree of drafts appended and checked, the
    accepted path appended over them, its weights gathered, the cache cut to its budget, a single token. Each step's
    attention stands within the int8 cache's error of full-precision attention over what the cache should hold."""
    from tests.tolerances import cos_sim, rel_l1

    Hq, Hkv, D, bs, B, E = 8, 2, 64, 16, 2, 256
    budget, keep = 64, 8
    old = [90, 120]
    parents = [-1, 0, 0, 1, 1, 2, 4]
    path = [0, 1, 4, 6]
    c = Room([200, 200], budget, Hkv, D, bs)
    wq = torch.randint(-127, 128, ((Hq + 2 * Hkv) * D, E), device=DEV, dtype=torch.int8)
    ws = torch.full(((Hq + 2 * Hkv) * D,), 1 / (72 * math.sqrt(E)), device=DEV)
    table = sl8.rope_table(400, D)
    held = [[[] for _ in range(B)] for _ in range(2)]  # keys and values, turned, as they should be

    def project(T):
        x = torch.randn(T, E, device=DEV, dtype=F16)
        y = sl8.linear_w8a8(x, wq, ws)
        xi, xs = sl8.quantize_i8_rowwise(x)
        full = (xi.double() @ wq.double().T * xs.double()[:, None] * ws.double()).view(T, Hq + 2 * Hkv, D)
        q, k, v = y.view(T, Hq + 2 * Hkv, D).split([Hq, Hkv, Hkv], 1)
        return q, k, v, full.split([Hq, Hkv, Hkv], 1)

    def turned(x, pos):
        cs = table[pos].double()[:, None]
        co, si = cs[..., :D // 2], cs[..., D // 2:]
        a, b = x[..., :D // 2], x[..., D // 2:]
        return torch.cat([a * co - b * si, b * co + a * si], -1)

    def ref(q, rows, b, seen=None):
        k, v = (torch.cat(h[b]) for h in held)
        out = torch.empty(len(rows), Hq, D, device=DEV, dtype=torch.float64)
        for h in range(Hq):
            w = q[rows, h] @ k[:, h // 4].T / math.sqrt(D)
            if seen is not None:
                w = w.masked_fill(~seen, -math.inf)
            out[:, h] = torch.softmax(w, -1) @ v[:, h // 4]
        return out

    def near(got, want):
        assert cos_sim(got, want) >= 0.998 and rel_l1(got, want) <= 0.05

    # the prompts
    q, k, v, f = project(sum(old))
    pos = torch.cat([torch.arange(n, device=DEV) for n in old])
    weights = torch.empty(B, Hkv, c.table.shape[1] * bs, device=DEV)
    cu, lens = offsets(old), i32(old)
    q1 = sl8.quantize_kv_append_block8(k, v, *c.args(), lens, cu_lens=cu, q=q, positions=pos, table=table, rotate=rotate)
    _, lse = sl8.attn_paged_block8(q1, *c.args(), lens, cu_lens=cu, rotate=rotate, return_lse=True)
    sl8.attn_weights_block8(q1, lse, c.k, c.ks, c.table, lens, weights, cu_lens=cu, rotate=rotate)
    for b, n in enumerate(old):
        assert abs(float(weights[b, :, :n].sum()) / (Hq * n) - 1) < 2e-3  # a row's weights are 1 in all
    for b, (t0, t1) in enumerate(((0, old[0]), (old[0], sum(old)))):
        held[0][b].append(turned(f[1], pos)[t0:t1])
        held[1][b].append(f[2][t0:t1])

    # a tree of drafts
    n = len(parents)
    mask = sl8.tree_mask(i32(parents * B), offsets([n] * B))
    bits = packed([torch.tensor([[bool(int(mask[i, 0]) >> j & 1) for j in range(n)] for i in range(n)])] * B, 1)
    assert torch.equal(mask, bits)
    depth = [bin(int(mask[i, 0])).count("1") - 1 for i in range(n)]
    q, k, v, f = project(B * n)
    pos = torch.tensor([o + d for o in old for d in depth], device=DEV)
    lens, cu = i32([o + n for o in old]), offsets([n] * B)
    q1 = sl8.quantize_kv_append_block8(k, v, *c.args(), lens, cu_lens=cu, q=q, positions=pos, table=table, rotate=rotate)
    out, lse = sl8.attn_paged_block8(q1, *c.args(), lens, cu_lens=cu, rotate=rotate, tree_mask=mask, return_lse=True)
    fq, fk = turned(f[0], pos), turned(f[1], pos)
    wants = []
    for b in range(B):
        rows = torch.arange(b * n, b * n + n, device=DEV)
        held[0][b].append(fk[rows])
        held[1][b].append(f[2][rows])
        see = torch.tensor([[bool(int(mask[i, 0]) >> j & 1) for j in range(n)] for i in range(n)], device=DEV)
        wants.append(ref(fq, rows, b, torch.cat([torch.ones(n, old[b], dtype=torch.bool, device=DEV), see], 1)))
        held[0][b][-1], held[1][b][-1] = fk[rows[path]], f[2][rows[path]]
    near(out, torch.cat(wants))

    # the accepted path over the drafts, and its weights
    at = torch.tensor([b * n + i for b in range(B) for i in path], device=DEV)
    m = len(path)
    lens, cu = i32([o + m for o in old]), offsets([m] * B)
    sl8.quantize_kv_append_block8(k[at], v[at], *c.args(), lens, cu_lens=cu, q=q[at], positions=pos[at], table=table,
                                  rotate=rotate)
    before = weights.clone()
    sl8.attn_weights_block8(q1[at], lse[at], c.k, c.ks, c.table, lens, weights, cu_lens=cu, rotate=rotate)
    for b, o in enumerate(old):
        got = float(weights[b, :, :o + m].sum() - before[b, :, :o].sum())
        assert abs(got / (Hq * m) - 1) < 0.02  # (the cache's codes were rounded again under some of them)

    # down to the budget, then a token
    lens, kept = sl8.kv_evict_block8(*c.args(), lens, weights, c.to, budget=budget, sinks=2, recent=keep)
    assert lens.tolist() == [budget] * B
    c.table = torch.cat([c.to, c.table[:, -1:]], 1).contiguous()  # (a block more for what comes)
    for b in range(B):
        for x in (0, 1):
            rows = torch.cat(held[x][b])
            held[x][b] = [torch.stack([rows[kept[b, h].long(), h] for h in range(Hkv)], 1)]
    q, k, v, f = project(B)
    pos = torch.tensor([o + m for o in old], device=DEV)
    lens = lens + 1
    q1 = sl8.quantize_kv_append_block8(k, v, *c.args(), lens, q=q, positions=pos, table=table, rotate=rotate)
    out = sl8.attn_paged_block8(q1, *c.args(), lens, rotate=rotate)
    fq, fk = turned(f[0], pos), turned(f[1], pos)
    wants = []
    for b in range(B):
        held[0][b].append(fk[b:b + 1])
        held[1][b].append(f[2][b:b + 1])
        wants.append(ref(fq, [b], b))
    near(out, torch.cat(wants))
