"""`rope` against the turned pairs in 64 bits: every layout, type, axis count and stride form, the
inverse as the gradient, and the refusals.

Tolerance: x cos - x' sin in fp32 rounds two products and a sum (an fma saves one), each by 2^-24 of
at most |x cos| + |x' sin|, then once to the output's type (half a step, eps / 2 of the value, or
half of the least subnormal)."""
import pytest
import torch

import superl8_amd as sl8
from superl8_amd import _C

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def turned(x, pos, table, sections, interleaved, inverse):
    """Plain 64-bit form on x [B,H,S,D], pos [A,B,S]; also |x cos| + |x' sin| of every element."""
    x, table = x.double(), table.double()
    half = table.shape[1] // 2
    out, size = x.clone(), torch.zeros_like(x)
    pair = 0
    for axis, n in enumerate(sections or (half,)):
        for p in range(pair, pair + n):
            at = pos[axis].long().clamp(0, table.shape[0] - 1)
            c, s = table[at, p][:, None], table[at, half + p][:, None]
            s = -s if inverse else s
            i, j = (2 * p, 2 * p + 1) if interleaved else (p, p + half)
            out[..., i] = x[..., i] * c - x[..., j] * s
            out[..., j] = x[..., j] * c + x[..., i] * s
            size[..., i] = (x[..., i] * c).abs() + (x[..., j] * s).abs()
            size[..., j] = (x[..., j] * c).abs() + (x[..., i] * s).abs()
        pair += n
    return out, size


def check(got, want, size):
    info = torch.finfo(got.dtype)
    lim = 3 * 2.0 ** -24 * size + info.eps / 2 * (1 + 2.0 ** -10) * want.abs() + info.tiny * info.eps / 2
    err = (got.double() - want).abs()
    assert bool((err <= lim).all()), float((err - lim).max())


def inputs(B, Hq, Hkv, S, D, R, axes, dtype, rows=700, pos_dtype=torch.int64, fused=True):
    x = torch.randn(B, S, Hq + 2 * Hkv, D, device="cuda").to(dtype)
    q, k = x[:, :, :Hq].transpose(1, 2), x[:, :, Hq:Hq + Hkv].transpose(1, 2)
    if not fused:
        q, k = q.contiguous(), k.contiguous()
    pos = torch.randint(0, rows, (axes, B, S), device="cuda").to(pos_dtype)
    return q, k, pos, torch.randn(rows, R, device="cuda").clamp_(-1, 1)


CASES = [  # B, Hq, Hkv, S, D, R, sections, dtype, interleaved
    (1, 1, 1, 1, 64, 64, None, F16, False),
    (3, 8, 2, 5, 128, 128, None, BF16, False),
    (2, 32, 8, 17, 128, 128, (16, 24, 24), F16, False),
    (2, 5, 1, 33, 128, 64, (3, 29), BF16, False),
    (2, 16, 16, 49, 80, 80, (20, 20), F16, False),
    (1, 16, 16, 21, 72, 72, (18, 18), BF16, False),
    (2, 4, 4, 7, 72, 36, None, F16, True),
    (2, 4, 2, 9, 80, 40, None, F32, False),
    (1, 3, 1, 130, 256, 256, (1, 2, 3, 122), F32, False),
    (2, 6, 3, 11, 128, 96, (5, 7, 36), F16, True),
    (1, 7, 7, 4, 34, 6, (1, 2), F32, True),
    (1, 2, 1, 3, 2, 2, None, F16, False),
    (1, 300, 40, 2, 64, 32, None, F16, False),
    (1, 2, 2, 3, 512, 512, None, BF16, True),
]


@pytest.mark.parametrize("B,Hq,Hkv,S,D,R,sections,dtype,interleaved", CASES)
@pytest.mark.parametrize("inverse", [False, True])
def test_rope(B, Hq, Hkv, S, D, R, sections, dtype, interleaved, inverse):
    axes = len(sections) if sections else 1
    q, k, pos, table = inputs(B, Hq, Hkv, S, D, R, axes, dtype)
    q0, k0 = q.clone(), k.clone()
    got = sl8.rope(q, k, pos if sections else pos[0], table, sections=sections,
                   interleaved=interleaved, inverse=inverse)
    for x, x0, y in zip((q, k), (q0, k0), got):
        assert y.is_contiguous() and y.dtype == dtype and y.shape == x.shape
        check(y, *turned(x0, pos, table, sections, interleaved, inverse))
        assert torch.equal(x, x0)


@pytest.mark.parametrize("pos_dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("sections", [None, (30, 34)])
def test_positions_shared_by_the_batch_and_outside_the_table(pos_dtype, sections):
    axes = len(sections) if sections else 1
    q, k, pos, table = inputs(3, 4, 2, 13, 128, 128, axes, F16, pos_dtype=pos_dtype)
    pos[:, 0, 0], pos[:, 0, 1], pos[:, 0, 2] = -1, 700, 2 ** 31 - 1
    if pos_dtype == torch.int64:
        pos[:, 0, 3], pos[:, 0, 4] = 2 ** 40, -(2 ** 40)
    shared = pos[:, 0].contiguous()
    got = sl8.rope(q, k, shared if sections else shared[0], table, sections=sections)
    full = pos[:, :1].expand(axes, 3, 13)
    for x, y in zip((q, k), got):
        check(y, *turned(x, full, table, sections, False, False))


def test_views_and_no_k():
    q, k, pos, table = inputs(2, 8, 4, 10, 64, 64, 1, BF16)
    want, size = turned(q, pos, table, None, False, False)
    for view in (q, q.contiguous(), q.transpose(2, 3).contiguous().transpose(2, 3)):
        y, none = sl8.rope(view, None, pos[0], table)
        assert none is None
        check(y, want, size)
    odd = torch.randn(2 * 8 * 10 * 64 + 1, device="cuda").to(BF16)[1:].view(2, 8, 10, 64)  # 2-byte aligned
    check(sl8.rope(odd, odd, pos[0], table)[1], *turned(odd, pos, table, None, False, False))
    one = q[:1, :1, :1].expand(2, 8, 10, 64)  # broadcast
    check(sl8.rope(one, None, pos[0], table)[0], *turned(one, pos, table, None, False, False))
    wide = torch.randn(table.shape[0], 65, device="cuda")[:, 1:]  # a table in a view
    check(sl8.rope(q, None, pos[0], wide)[0], *turned(q, pos, wide, None, False, False))


@pytest.mark.parametrize("B,S,H", [(0, 4, 2), (2, 0, 2), (2, 4, 0)])
def test_empty(B, S, H):
    x = torch.zeros(B, H, S, 64, device="cuda", dtype=F16)
    y, z = sl8.rope(x, x, torch.zeros(S, device="cuda", dtype=torch.int32), torch.ones(3, 64, device="cuda"))
    assert y.shape == z.shape == x.shape


@pytest.mark.parametrize("interleaved", [False, True])
def test_inverse_is_the_gradient(interleaved):
    """Against autograd through the 64-bit form and against differences of the kernel itself."""
    q, k, pos, _ = inputs(2, 4, 2, 9, 80, 80, 2, F32, fused=False)
    table = sl8.rope_table(700, 80, sections=(20, 20))
    g = torch.randn_like(q)
    got, _ = sl8.rope(g, None, pos, table, sections=(20, 20), interleaved=interleaved, inverse=True)
    x = q.double().requires_grad_()
    turned(x, pos, table, (20, 20), interleaved, False)[0].backward(g.double())
    lim = turned(g, pos, table, (20, 20), interleaved, True)[1] * 2.0 ** -22
    assert bool(((got.double() - x.grad).abs() <= lim).all())
    d = torch.randn_like(q)
    hi, _ = sl8.rope(q + d, None, pos, table, sections=(20, 20), interleaved=interleaved)
    lo, _ = sl8.rope(q - d, None, pos, table, sections=(20, 20), interleaved=interleaved)
    num = ((hi.double() - lo.double()) / 2 * g.double()).sum()
    # the map is linear: only fp32 roundings of 5760 products of size ~1 stand between the two
    assert abs(float(num - (got.double() * d.double()).sum())) <= q.numel() * 2.0 ** -20


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("sections,interleaved,inverse", [(None, False, False), ((9, 23), True, False),
                                                          ((16, 8, 8), False, True)])
def test_autograd(dtype, sections, interleaved, inverse):
    """What requires a gradient gets the turn back of the outputs' gradients, whichever of them there are."""
    q, k, pos, table = inputs(2, 4, 2, 9, 80, 64, len(sections or (0,)), dtype)
    pos = pos if sections else pos[0]
    how = dict(sections=sections, interleaved=interleaved)
    gq, gk = torch.randn_like(q), torch.randn_like(k)
    wq, wk = sl8.rope(gq, gk, pos, table, **how, inverse=not inverse)
    run = lambda q, k: sl8.rope(q, k, pos, table, **how, inverse=inverse)
    plain = run(q, k)
    assert not any(t.requires_grad for t in plain)
    lq, lk = q.clone().requires_grad_(), k.clone().requires_grad_()
    yq, yk = run(lq, lk)
    assert torch.equal(yq, plain[0]) and torch.equal(yk, plain[1])
    torch.autograd.backward((yq, yk), (gq, gk))
    assert torch.equal(lq.grad, wq) and torch.equal(lk.grad, wk)
    x = q.double().requires_grad_()
    p = pos if sections else pos[None]
    turned(x, p, table, sections, interleaved, inverse)[0].backward(gq.double())
    check(lq.grad, x.grad, turned(gq, p, table, sections, interleaved, not inverse)[1])
    # one of the outputs, one of the inputs, no k, nothing
    assert torch.equal(torch.autograd.grad(run(lq, lk)[1], lk, gk)[0], wk)
    assert torch.equal(torch.autograd.grad(run(lq, lk)[0], lq, gq)[0], wq)
    assert torch.autograd.grad(run(lq, lk)[0], lk, gq, allow_unused=True)[0] is None
    assert torch.equal(torch.autograd.grad(run(q, lk), lk, (gq, gk))[0], wk)
    assert torch.equal(torch.autograd.grad(run(lq, k), lq, (gq, gk))[0], wq)
    assert torch.equal(torch.autograd.grad(run(lq, None)[0], lq, gq)[0], wq)
    with torch.no_grad():
        assert not run(lq, lk)[0].requires_grad
    # views of one leaf, a broadcast gradient
    both = torch.cat([q, k], 1).requires_grad_()
    one = torch.ones((), device="cuda", dtype=dtype)
    d, = torch.autograd.grad(run(both[:, :4], both[:, 4:]), both, (one.expand(q.shape), one.expand(k.shape)))
    dq, dk = sl8.rope(torch.ones_like(q), torch.ones_like(k), pos, table, **how, inverse=not inverse)
    assert torch.equal(d, torch.cat([dq, dk], 1))
    # the gradient's own gradient: the turn again
    v = gq.clone().requires_grad_()
    d, = torch.autograd.grad(run(lq, None)[0], lq, v, create_graph=True)
    assert torch.equal(torch.autograd.grad(d, v, q)[0], plain[0])


def test_captured_gradient():
    """A captured backward is refused beside a living eager graph of the same leaves, and the explicit call is not."""
    q, _, pos, table = inputs(2, 4, 2, 9, 64, 64, 1, F32)
    leaf, g = q.clone().requires_grad_(), torch.randn_like(q)
    alive = sl8.rope(leaf, None, pos[0], table)[0]  # noqa: F841
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            torch.autograd.grad(sl8.rope(leaf, None, pos[0], table)[0], leaf, g)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):  # (what needs no backward is captured as ever)
        y, _ = sl8.rope(leaf, None, pos[0], table)
        with torch.no_grad():
            d, _ = sl8.rope(g, None, pos[0], table, inverse=True)
    want, = torch.autograd.grad(alive, leaf, g)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, alive) and torch.equal(d, want)


def test_rope_table_far_positions():
    """Angles of far positions from 64 bits, rounded once."""
    t = sl8.rope_table(200001, 64, base=500000.0)
    a = 200000.0 * 500000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)
    want = torch.cat([a.cos(), a.sin()])
    # 2^-25 of the rounding, and 2e5 rad times the 2^-53 of power and product
    assert float((t[200000].cpu().double() - want).abs().max()) <= 2.0 ** -24
    with pytest.raises(ValueError):
        sl8.rope_table(10, 63)
    with pytest.raises(ValueError):
        sl8.rope_table(10, 64, sections=(16, 15))


def test_other_stream_and_graph():
    q, k, pos, table = inputs(2, 8, 2, 6, 128, 128, 1, F16)
    want = sl8.rope(q, k, pos[0], table)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = sl8.rope(q, k, pos[0], table)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    qs, g = torch.zeros_like(q), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = sl8.rope(qs, k, pos[0], table)
    for i in range(3):
        qs.copy_(q * (i + 1))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], sl8.rope(qs, k, pos[0], table)[0])


def test_refusals():
    q, k, pos, table = inputs(2, 4, 2, 6, 64, 64, 1, F16)
    p = pos[0]
    bad = [
        dict(q=q.to(torch.int8)), dict(k=k.float()), dict(k=k[:1]), dict(k=k[..., :32]), dict(q=q[0]),
        dict(positions=p.float()), dict(positions=p[:, :5]), dict(positions=p[:1, :1]),
        dict(positions=pos, sections=None), dict(sections=(32,)), dict(sections=(31, 2), positions=pos),
        dict(positions=pos, sections=(0, 32)), dict(positions=pos.expand(5, 2, 6), sections=(1, 1, 1, 1, 28)),
        dict(table=table.double()), dict(table=table[:, :63]), dict(table=table[:0]), dict(table=table[0]),
        dict(table=torch.ones(9, 66, device="cuda")), dict(table=table.cpu()), dict(positions=p.cpu()),
    ]
    for change in bad:
        args = dict(q=q, k=k, positions=p, table=table, sections=None) | change
        with pytest.raises(RuntimeError, match="fni8"):
            _C.rope(**args)
