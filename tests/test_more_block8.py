"""The C entries of the int8 linear, of drafted trees, gathered weights and eviction refuse what they cannot run before
any device work: no GPU needed. And the masks of trees, which torch makes on any device."""
import pytest
import torch

import superl8_amd as sl8
from superl8_amd import _lib


def tree(**c):
    a = dict(q=16, dtype=0, rot=0, mul=1.0, k=16, ks=16, v=16, vs=16, cu=None, lens=16, bt=16, mask=16, words=1, out=16,
             lse=16, T=2, B=2, Hq=2, Hkv=1, D=64, nb=400, bs=16, maxb=200, window=-1, ws=16, ws_bytes=1 << 40)
    return _lib.load().sl8_attn_paged_block8_tree(*(a | c).values(), None)


def weights(**c):
    a = dict(q=16, dtype=0, rot=0, mul=1.0, lse=16, k=16, ks=16, cu=None, lens=16, bt=16, w=16, wb=400, wh=200, decay=1.0,
             T=2, B=2, Hq=2, Hkv=1, D=64, nb=400, bs=16, maxb=4, window=-1, ws=16, ws_bytes=1 << 40)
    return _lib.load().sl8_attn_weights_block8(*(a | c).values(), None)


def evict(**c):
    a = dict(k=16, ks=16, v=16, vs=16, lens=16, bt=16, w=16, wb=400, wh=200, to=16, new=16, kept=16, B=2, Hkv=1, D=64,
             nb=400, bs=16, maxb=4, to_maxb=2, budget=32, sinks=0, recent=0)
    return _lib.load().sl8_kv_evict_block8(*(a | c).values(), None)


def linear(**c):
    a = dict(x=16, xdt=0, w=16, ws=16, bias=None, bdt=0, out=16, odt=0, M=2, N=8, K=64, work=16, bytes=1 << 40)
    return _lib.load().sl8_linear_w8a8(*(a | c).values(), None)


@pytest.mark.parametrize("call,change,word", [
    (tree, dict(words=0), b"words"), (tree, dict(words=5), b"words"), (tree, dict(mask=20), b"aligned"),
    (tree, dict(lse=18), b"aligned"), (tree, dict(dtype=2), b"float16"), (tree, dict(D=32), b"head dim"),
    (tree, dict(Hq=3, Hkv=2), b"divisible"), (tree, dict(T=3), b"one row"), (tree, dict(q=None), b"null"),
    (tree, dict(ws=None), b"workspace"), (tree, dict(ws_bytes=100), b"workspace"), (tree, dict(maxb=1 << 26), b"large"),
    (weights, dict(dtype=2), b"float16"), (weights, dict(D=80), b"head dim"), (weights, dict(bs=24), b"block_size"),
    (weights, dict(Hq=3, Hkv=2), b"divisible"), (weights, dict(Hq=0), b"divisible"), (weights, dict(T=3), b"one row"),
    (weights, dict(lse=None), b"null"), (weights, dict(w=None), b"null"), (weights, dict(ks=None), b"null"),
    (weights, dict(nb=0), b"blocks"), (weights, dict(k=24), b"aligned"), (weights, dict(ws=None), b"workspace"),
    (weights, dict(ws_bytes=100), b"workspace"), (weights, dict(T=1 << 23, B=1 << 23, maxb=1 << 25), b"large"),
    (weights, dict(T=1 << 28, B=1 << 28), b"large"),
    (evict, dict(budget=0), b"budget"), (evict, dict(budget=-4), b"budget"), (evict, dict(sinks=-1), b"budget"),
    (evict, dict(sinks=20, recent=13), b"budget"), (evict, dict(recent=33), b"budget"), (evict, dict(to_maxb=1), b"new_table"),
    (evict, dict(budget=64, to_maxb=3), b"new_table"), (evict, dict(budget=1 << 30), b"large"), (evict, dict(D=96), b"head dim"),
    (evict, dict(bs=8), b"block_size"), (evict, dict(kept=None), b"null"), (evict, dict(vs=None), b"null"),
    (evict, dict(to=None), b"null"), (evict, dict(v=8), b"aligned"), (evict, dict(B=1 << 23), b"large"),
    (linear, dict(xdt=5), b"float16"), (linear, dict(odt=5), b"out_dtype"), (linear, dict(bias=16, bdt=7), b"bias"),
    (linear, dict(K=12), b"multiple of 4"), (linear, dict(K=66), b"multiple of 4"), (linear, dict(K=1 << 17), b"multiple of 4"),
    (linear, dict(M=-1), b"large"), (linear, dict(N=1 << 24), b"large"), (linear, dict(x=None), b"null"),
    (linear, dict(w=20), b"aligned"), (linear, dict(w=18, K=68), b"aligned"), (linear, dict(x=24), b"aligned"),
    (linear, dict(work=None), b"workspace"), (linear, dict(bytes=10), b"workspace"), (linear, dict(work=24), b"workspace"),
])
def test_refused(call, change, word):
    lib = _lib.load()
    assert call(**change) == -1
    assert word in lib.sl8_last_error() and b"fni8" in lib.sl8_last_error()


def test_nothing_to_do():
    assert tree(T=0, B=2, cu=16) == 0 and tree(T=0, B=0) == 0
    assert weights(T=0, B=0) == 0 and weights(maxb=0) == 0 and evict(B=0) == 0
    assert linear(M=0) == 0 and linear(N=0) == 0


def test_workspaces():
    lib = _lib.load()
    assert lib.sl8_attn_weights_block8_workspace(10, 2, 8, 4, 128, 400) >= 80 * 128
    for bad in ((0, 2, 8, 4, 128, 400), (10, 0, 8, 4, 128, 400), (10, 2, 0, 4, 128, 400), (10, 2, 8, 0, 128, 400),
                (10, 2, 8, 3, 128, 400), (10, 2, 8, 4, 0, 400), (-1, 2, 8, 4, 64, 400), (1 << 40, 2, 8, 4, 64, 400),
                (10, 2, 8, 4, 64, 1 << 40), (10, 1 << 20, 8, 4, 64, 1 << 25)):
        assert lib.sl8_attn_weights_block8_workspace(*bad) == 0
    assert lib.sl8_linear_w8a8_workspace(17, 100, 100) >= 32 * 128
    for bad in ((0, 8, 64), (8, 0, 64), (8, 8, 8), (1 << 40, 8, 64), (8, 8, 1 << 20)):
        assert lib.sl8_linear_w8a8_workspace(*bad) == 0
    for bad in ((0, 1, 2, 1, 64, 100), (2, 2, 3, 2, 64, 100), (2, 2, 2, 1, 96, 100)):
        assert lib.sl8_attn_paged_block8_tree_workspace(*bad) == 0


def test_cpu_tensors_raise():
    x, w = torch.zeros(2, 64, dtype=torch.float16), torch.zeros(4, 64, dtype=torch.int8)
    with pytest.raises(RuntimeError, match="CUDA"):
        sl8.linear_w8a8(x, w, torch.ones(4))
    c, s, t = torch.zeros(4, 1, 16, 64, dtype=torch.int8), torch.ones(4, 1), torch.zeros(2, 2, dtype=torch.int32)
    n, wt = torch.ones(2, dtype=torch.int32), torch.zeros(2, 1, 32)
    with pytest.raises(RuntimeError, match="CUDA"):
        sl8.kv_evict_block8(c, s, c, s, t, n, wt, t, budget=16)
    q = torch.zeros(2, 1, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        sl8.attn_weights_block8(q, torch.zeros(2, 1), c, s, t, n, wt)


def test_masks_of_random_trees():
    g = torch.Generator().manual_seed(3)
    for n, words in ((1, 1), (30, 1), (64, 1), (65, 2), (250, 4), (90, 1)):
        new = [n, max(1, n // 3)]
        parents, want = [], []
        for m in new:
            above = []
            for i in range(m):
                p = int(torch.randint(-1, i, (1,), generator=g)) if i else -1
                above.append(1 << i | (above[p] if p >= 0 else 0))
                parents.append(p)
            want += [a & (1 << 64 * words) - 1 for a in above]
        cu = torch.tensor([0, n, sum(new)], dtype=torch.int32)
        got = sl8.tree_mask(torch.tensor(parents), cu, words=words)
        assert got.shape == (sum(new), words) and got.dtype == torch.int64
        for r, a in zip(got.tolist(), want):
            assert sum((x & (1 << 64) - 1) << (64 * k) for k, x in enumerate(r)) == a
    assert sl8.tree_mask(torch.zeros(0, dtype=torch.int32)).shape == (0, 1)


@pytest.mark.parametrize("n,words", [(65, 1), (100, 1), (128, 1), (129, 1), (200, 2), (300, 4), (700, 4)])
def test_masks_of_paths_longer_than_their_words(n, words):
    """A token behind the last bit still has the bits of all above it: chains, chains whose parents stand behind
    their children, and one beside a sequence of its own."""
    full = (1 << 64 * words) - 1
    whole = lambda r: sum((x & (1 << 64) - 1) << (64 * k) for k, x in enumerate(r))
    down = sl8.tree_mask(torch.arange(-1, n - 1), words=words)
    assert [whole(r) for r in down.tolist()] == [(1 << i + 1) - 1 & full for i in range(n)]
    up = sl8.tree_mask(torch.arange(1, n + 1), words=words)  # (the last one's parent is not there)
    assert [whole(r) for r in up.tolist()] == [(1 << n) - (1 << i) & full for i in range(n)]
    two = sl8.tree_mask(torch.cat([torch.arange(-1, 2), torch.arange(-1, n - 1)]).int(),
                        torch.tensor([0, 3, 3 + n], dtype=torch.int32), words=words)
    assert [whole(r) for r in two.tolist()] == [(1 << i + 1) - 1 & full for i in [*range(3), *range(n)]]


@pytest.mark.parametrize("lens,new", [(4096, 4096), (4096, 4100), (4100, 4096)])
def test_lengths_are_not_written_where_they_are_read(lens, new):
    """Heads of a sequence read its length while another one's workgroup writes the new one."""
    assert evict(lens=lens, new=new) == -1
    assert b"new_lens" in _lib.load().sl8_last_error()


@pytest.mark.parametrize("change", [dict(T=1 << 27, B=1, Hq=1, D=256, cu=16), dict(T=1 << 24, B=2, Hq=8, Hkv=8, D=256, cu=16),
                                    dict(T=1 << 27, B=1, Hq=2, D=128, cu=16), dict(T=(1 << 27) + 1, B=1, Hq=4, Hkv=4, D=64, cu=16)])
def test_rows_that_a_launch_cannot_hold(change):
    """The pass over the rows has a workgroup of 256 threads for 2048 elements, and a launch below 2^32 threads."""
    assert weights(**change) == -1
    assert b"large" in _lib.load().sl8_last_error()
    c = dict(Hkv=1) | change
    assert _lib.load().sl8_attn_weights_block8_workspace(c["T"], c["B"], c["Hq"], c["Hkv"], c["D"], 64) == 0
