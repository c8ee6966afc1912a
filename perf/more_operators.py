"""Performance cases of four operators of a serving step: the projections of int8 weights, the attention
that checks a tree of drafted tokens, and a cache that is kept within a budget.

  linear   `linear_w8a8`: x @ w^T of int8 weights with a scale per output channel, x quantised with a
           scale per token, bias added, rounded once
  tree     `attn_paged_block8(tree_mask=)`: attention of drafted tokens, each of which sees its
           sequence's context and the drafted tokens that its mask names; with the sums' logarithms
  weights  `attn_weights_block8`: each cached key's softmax weights of a step's rows added to what it
           had before
  evict    `kv_evict_block8`: the tokens of the largest weights of each head (and the first and last
           ones) moved into other blocks of the cache

`listed()` holds workloads of serving; `draw` samples the ranges that they stand for. A case is a
dict of plain values. With `own` false `run` computes the operators' plain forms in elementary torch
operations, with `own` true it calls this package.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
FLOOR = 2.0 ** -60  # the least scale of a block


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _linear(M, N, K, dtype="fp16", out="", bias=False):
    return dict(kind="linear", M=M, N=N, K=K, dtype=dtype, out=out or dtype, bias=bias)


def _tree(B, new, old, Hq, Hkv, D, block, dtype="fp16", rotate=True, window=-1, lse=False):
    """B sequences of about `old` tokens (see _lens), each with a tree of up to `new` drafted ones."""
    return dict(kind="tree", B=B, new=new, old=old, Hq=Hq, Hkv=Hkv, D=D, block=block, dtype=dtype,
                rotate=rotate, window=window, lse=lse)


def _weights(B, new, old, Hq, Hkv, D, block, dtype="fp16", rotate=True, window=-1, decay=1.0):
    return dict(kind="weights", B=B, new=new, old=old, Hq=Hq, Hkv=Hkv, D=D, block=block, dtype=dtype,
                rotate=rotate, window=window, decay=decay)


def _evict(B, old, budget, sinks, recent, Hkv, D, block):
    return dict(kind="evict", B=B, new=1, old=old, budget=budget, sinks=sinks, recent=recent, Hkv=Hkv, D=D,
                block=block, dtype="fp16")


def listed() -> list[dict]:
    return [
        # one token through a square projection: the smallest product, where latency counts
        dict(name="linear_one", **_linear(1, 4096, 4096)),
        # 16 tokens of a decode step through a wide up-projection: the weights' bytes
        dict(name="linear_step_bf16", **_linear(16, 17408, 5120, "bf16")),
        # a few hundred tokens, odd sizes, a bias, fp32 out (the logits of a small head)
        dict(name="linear_odd_bias", **_linear(333, 5003, 2052, "bf16", "fp32", True)),
        # a long prompt through the wide projection: the most arithmetic
        dict(name="linear_prompt", **_linear(4096, 17408, 5120)),
        # 26 drafted tokens of one conversation: the smallest tree
        dict(name="tree_one", **_tree(1, 26, 776, 32, 8, 128, 16)),
        # 60 drafted tokens of each of 16 sequences of mixed lengths
        dict(name="tree_batch_bf16", **_tree(16, 60, 8191, 32, 8, 128, 32, "bf16", lse=True)),
        # wide trees of odd sizes, wide heads, a sliding window, keys that are not rotated
        dict(name="tree_wide_window", **_tree(4, 129, 5003, 16, 2, 256, 64, rotate=False, window=2048)),
        # the keys' weights of a decode step of 32 sequences: the bytes of K
        dict(name="weights_step", **_weights(32, 1, 8191, 32, 8, 128, 16)),
        # those of the last rows of prompts of mixed odd lengths, fading, 64-wide heads, a window
        dict(name="weights_ragged_bf16", **_weights(6, 33, 3001, 16, 4, 64, 32, "bf16", False, 1000, 0.9)),
        # those of all rows of a prompt behind a cached prefix: the arithmetic
        dict(name="weights_prompt", **_weights(1, 2048, 2048, 32, 8, 128, 64)),
        # a few conversations that ran over their budget by a little: the smallest eviction
        dict(name="evict_step", **_evict(4, 1100, 1024, 4, 64, 8, 128, 16)),
        # long contexts cut down to an eighth
        dict(name="evict_long", **_evict(8, 32768, 4096, 16, 256, 8, 128, 32)),
    ]


def _log(rng: random.Random, lo: float, hi: float) -> int:
    return max(int(lo), min(int(hi), round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi)))))))


def _heads(rng: random.Random) -> tuple[int, int]:
    hkv = rng.choice([1, 2, 4, 8])
    return hkv * rng.choice([1, 2, 4, 8] if hkv < 8 else [1, 2, 4]), hkv


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["linear", "tree", "weights", "evict"])
    dtype = rng.choice(["fp16", "bf16"])
    if kind == "linear":
        N, K = _log(rng, 16, 17408), 4 * _log(rng, 16, 2048)
        if rng.random() < 0.5:  # what models have
            N, K = max(16, N // 64 * 64), max(64, K // 64 * 64)
        M = _log(rng, 1, min(8192, 360000000000 // (N * K)))
        return _linear(M, N, K, dtype, rng.choice([dtype, dtype, "fp32"]), rng.random() < 0.3)
    hq, hkv = _heads(rng)
    D, block = rng.choice([64, 128, 128, 256]), rng.choice([16, 32, 64, 128])
    window = -1 if rng.random() < 0.75 else _log(rng, 64, 3000)
    rotate = rng.random() < 0.7
    if kind == "evict":
        B = _log(rng, 1, 64)
        old = _log(rng, 40, min(60000, (1 << 28) // (B * hkv * D)))
        budget = _log(rng, 16, old * 1.1)
        recent = rng.randint(0, budget // 2)
        return _evict(B, old, budget, rng.randint(0, min(16, budget - recent)), recent, hkv, D, block)
    B = _log(rng, 1, 64)
    if kind == "tree":
        new = _log(rng, 2, 200)
        most = min((1 << 28) // (B * hkv * D), 250000000 // (B * hq * new))
        return _tree(B, new, _log(rng, 30, max(60, min(65000, most))), hq, hkv, D, block, dtype, rotate, window,
                     rng.random() < 0.5)
    new = 1 if rng.random() < 0.4 else _log(rng, 2, 2000)
    B = max(1, min(B, 3000 // new))
    most = min((1 << 28) // (B * hkv * D), 250000000 // (B * hq * new))
    return _weights(B, new, _log(rng, 30, max(60, min(65000, most))), hq, hkv, D, block, dtype, rotate, window,
                    rng.choice([1.0, 1.0, 0.95]))


def _lens(c) -> tuple[list[int], list[int]]:
    """New tokens and lengths before them of each sequence: from new / 2 to new, and spread evenly (in the
    logarithm) over a factor of 8 (those of an eviction: of 1.5)."""
    B = c["B"]
    new = [max(1, c["new"] - i * c["new"] // (2 * B)) for i in range(B)]
    over = 1.5 if c["kind"] == "evict" else 8
    old = [max(1, round(c["old"] * over ** -(i / max(1, B - 1)))) for i in range(B)]
    random.Random(B).shuffle(old)
    if c["kind"] == "evict":
        old = [n - 1 for n in old]
    return new, old


def _words(c) -> int:
    return -(-c["new"] // 64)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _codes(g, *shape):
    """int8 codes of normal values in groups whose largest is 3.5 deviations."""
    out = torch.empty(*shape, device=DEV, dtype=torch.int8)
    for part in out.flatten().split(1 << 27):
        part.copy_((torch.randn(part.shape, device=DEV, generator=g, dtype=torch.float16) * 36)
                   .round_().clamp_(-127, 127))
    return out


def _i32(x) -> torch.Tensor:
    return torch.tensor(x, device=DEV, dtype=torch.int32)


def _tables(order: torch.Tensor, blocks: list[int]) -> torch.Tensor:
    """A table of each sequence's blocks, in the order given; rows end with the first block."""
    most, at, rows = max(blocks), 0, []
    for n in blocks:
        rows.append(torch.cat([order[at:at + n], order[:1].expand(most - n)]))
        at += n
    return torch.stack(rows).contiguous()


def _parents(n: int, rng: random.Random) -> list[int]:
    """A tree of n drafted tokens, parents first: levels of about a tenth, at least two, of the nodes."""
    width = max(2, n // 10)
    return [-1] + [rng.randrange(max(0, i - 2 * width), i) for i in range(1, n)]


def _masks(new: list[int], words: int, seed: int) -> torch.Tensor:
    """int64 [T, words]: bit j of a row: the sequence's drafted token j is it or stands above it."""
    rng, out = random.Random(seed), []
    for n in new:
        bits = []
        for i, p in enumerate(_parents(n, rng)):
            bits.append(1 << i | (bits[p] if p >= 0 else 0))
        for b in bits:
            w = [b >> (64 * k) & (1 << 64) - 1 for k in range(words)]
            out.append([x - (1 << 64) if x >> 63 else x for x in w])
    return torch.tensor(out, device=DEV, dtype=torch.int64)


def _hadamard(d: int) -> torch.Tensor:
    h = torch.ones(1, 1, device=DEV, dtype=torch.float64)
    while h.shape[0] < d:
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
    return h / math.sqrt(d)


def prepare(case: dict, seed: int) -> dict:
    c, g, dt = case, _gen(seed), DTYPES[case["dtype"]]
    if c["kind"] == "linear":
        x = torch.randn(c["M"], c["K"], device=DEV, generator=g)
        x[:, torch.randint(0, c["K"], (max(1, c["K"] // 200),), device=DEV, generator=g)] *= 6
        s = {"case": c, "x": x.to(dt), "w": _codes(g, c["N"], c["K"]), "bias": None,
             "ws": (torch.rand(c["N"], device=DEV, generator=g) + 0.5) / (36 * math.sqrt(c["K"]))}
        if c["bias"]:
            s["bias"] = torch.randn(c["N"], device=DEV, generator=g).to(dt)
        return s
    new, old = _lens(c)
    total, bs, Hkv, D = [a + b for a, b in zip(new, old)], c["block"], c["Hkv"], c["D"]
    blocks = [-(-n // bs) for n in total]
    # an eviction's destination: the pool's first blocks
    to = [-(-min(n, c["budget"]) // bs) for n in total] if c["kind"] == "evict" else [0]
    nd = sum(to)
    order = torch.randperm(sum(blocks) + 3, device=DEV, generator=g).to(torch.int32) + nd
    s = {"case": c, "cache": _codes(g, 2, nd + order.shape[0], Hkv, bs, D), "blocks": _tables(order, blocks),
         "lens": _i32(total), "cu": _i32([sum(new[:i]) for i in range(len(new) + 1)]),
         "hadamard": _hadamard(D)}
    s["scale"] = (torch.rand(s["cache"].shape[:3], device=DEV, generator=g) * 0.4 + 0.8) * (3.5 / 127)
    if c["kind"] == "evict":
        s["to"] = _tables(torch.randperm(nd, device=DEV, generator=g).to(torch.int32), to)
        s["weights"] = torch.rand(c["B"], Hkv, max(blocks) * bs, device=DEV, generator=g).log_().neg_()
        s["values"] = torch.empty(2, nd, Hkv, bs, D, device=DEV, dtype=dt)
        return s
    s["q"] = (torch.randn(sum(new), c["Hq"], D, device=DEV, generator=g) * 2).to(dt)
    if c["kind"] == "tree":
        s["mask"] = _masks(new, _words(c), seed)
        return s
    # the logarithms of the rows' sums, as the attention of the same step gives them
    s["weights"] = torch.rand(c["B"], Hkv, max(blocks) * bs, device=DEV, generator=g)
    w, b, i = _scores(s, _seen_causal(s))
    s["lse"] = _by_rows(s, torch.logsumexp(w, -1, keepdim=True), b, i)[..., 0].contiguous()
    return s


# ---------------------------------------------------------------------------
# the plain forms, in 32 bits
# ---------------------------------------------------------------------------
def _plain_linear(s):
    x = s["x"].float()
    xs = x.abs().amax(-1, keepdim=True) * torch.tensor(1 / 127, device=DEV)
    xs = torch.where(xs == 0, 1.0, xs)
    codes = torch.round(x / xs).clamp(-127, 127)
    y = (codes @ s["w"].float().T) * xs * s["ws"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(DTYPES[s["case"]["out"]])


def _tokens(s):
    """Sequence and place in its new tokens of every token, and the length before them."""
    cu = s["cu"].long()
    t = torch.arange(s["q"].shape[0], device=cu.device)
    b = torch.searchsorted(cu, t, right=True) - 1
    return b, t - cu[b], s["lens"].long() - (cu[1:] - cu[:-1])


def _padded(s, t):
    """Rows of all tokens [T, ...] by sequence, [B, new, ...]; those past a sequence's last are others'."""
    at = s["cu"].long()[:-1, None] + torch.arange(s["case"]["new"], device=DEV)
    return t[at.clamp(max=t.shape[0] - 1)]


def _by_heads(s, t):
    """[T, Hq, n] -> [B, Hkv, G * new, n]."""
    c = s["case"]
    t = _padded(s, t).unflatten(2, (c["Hkv"], -1))
    return t.permute(0, 2, 3, 1, 4).flatten(2, 3)


def _by_rows(s, t, b, i):
    """Back: [B, Hkv, G * new, n] -> [T, Hq, n]."""
    return t.unflatten(2, (-1, s["case"]["new"])).permute(0, 3, 1, 2, 4).flatten(2, 3)[b, i]


def _seen_causal(s):
    """[B, 1, G * new, keys]: what each row sees of its sequence's tokens."""
    c = s["case"]
    _, _, before = _tokens(s)
    n = torch.arange(s["blocks"].shape[1] * c["block"], device=DEV)
    last = (before[:, None] + torch.arange(c["new"], device=DEV)).repeat(1, c["Hq"] // c["Hkv"])[:, None, :, None]
    seen = (n <= last) & (n < s["lens"].long()[:, None, None, None])
    return seen & (n > last - c["window"]) if c["window"] >= 0 else seen


def _seen_tree(s):
    """The same of a tree: the tokens before the new ones, of which the window keeps as many as the marked
    ones leave of it, and the marked ones."""
    c = s["case"]
    _, _, before = _tokens(s)
    mask = _padded(s, s["mask"])
    bits = (mask[..., None] >> torch.arange(64, device=DEV) & 1).bool().flatten(2)  # [B, new, 64 words]
    n = torch.arange(s["blocks"].shape[1] * c["block"], device=DEV)
    at = n - before[:, None]  # [B, keys]: place among the new tokens
    near = bits.gather(2, at.clamp(0, bits.shape[2] - 1)[:, None].expand(-1, c["new"], -1))
    near &= ((at >= 0) & (at < bits.shape[2]) & (n < s["lens"].long()[:, None]))[:, None]
    far = (at < 0)[:, None].expand_as(near)
    if c["window"] >= 0:
        room = (c["window"] - bits.sum(-1)).clamp(min=0)
        far = far & (at[:, None] >= -room[..., None])
    return (near | far).repeat(1, c["Hq"] // c["Hkv"], 1)[:, None]


def _side(s, j):
    """Codes of every sequence's blocks [B, Hkv, keys, D] and their scales [B, Hkv, keys]."""
    t = s["blocks"].long()
    x = s["cache"][j][t].transpose(1, 2).flatten(2, 3).float()
    return x, s["scale"][j][t].transpose(1, 2).repeat_interleave(s["case"]["block"], 2)


def _scores(s, seen):
    """Scores (natural logarithm) of every row and key, -inf where it does not see it."""
    c = s["case"]
    # the query rows in int8, one scale each (in 64 bits, as a quotient next to a half takes one code or the next)
    x = s["q"].double()
    if c["rotate"]:
        x = x @ s["hadamard"]
    qs = x.abs().amax(-1, keepdim=True).float() * torch.tensor(1 / 127, device=DEV)
    qs = torch.where(qs == 0, 1.0, qs)
    x = torch.round((x / qs).float()).clamp(-127, 127)
    b, i, _ = _tokens(s)
    k, ks = _side(s, 0)
    w = _by_heads(s, x) @ k.transpose(2, 3).contiguous()
    del k
    w *= _by_heads(s, qs) * (1 / math.sqrt(c["D"]))
    w *= ks[:, :, None]
    return w.masked_fill_(~seen, -math.inf), b, i


def _plain_tree(s):
    w, b, i = _scores(s, _seen_tree(s))
    top = w.amax(-1, keepdim=True).clamp_min(-1e30)
    w -= top
    w.exp_()
    total = w.sum(-1, keepdim=True)
    v, vs = _side(s, 1)
    w *= vs[:, :, None]
    out = (w @ v) / torch.where(total == 0, 1.0, total)
    out = _by_rows(s, out, b, i).to(s["q"].dtype)
    return (out, _by_rows(s, top + total.log(), b, i)[..., 0]) if s["case"]["lse"] else out


def _plain_weights(s):
    c = s["case"]
    w, _, _ = _scores(s, _seen_causal(s))
    lse = _by_heads(s, s["lse"][..., None])
    w -= torch.where(lse == -math.inf, math.inf, lse)
    w.exp_()
    _, _, before = _tokens(s)
    new = s["lens"].long() - before
    mine = torch.arange(c["new"], device=DEV) < new[:, None]  # rows past a sequence's last are others'
    w *= mine.repeat(1, c["Hq"] // c["Hkv"])[:, None, :, None]
    n = torch.arange(w.shape[-1], device=DEV)
    was = torch.where(n < before[:, None, None], s["weights"] * c["decay"], 0)
    here = n < s["lens"].long()[:, None, None]
    s["weights"].copy_(torch.where(here, was + w.sum(2), s["weights"]))
    return s["weights"]


def _plain_evict(s):
    c, bs, D = s["case"], s["case"]["block"], s["case"]["D"]
    B, Hkv, S = s["weights"].shape
    lens, budget = s["lens"].long(), c["budget"]
    n = torch.arange(S, device=DEV)
    rank = s["weights"].masked_fill((n < c["sinks"]) | (n >= lens[:, None, None] - c["recent"]), math.inf)
    rank = rank.masked_fill(n >= lens[:, None, None], -math.inf)
    order = torch.sort(rank, dim=-1, descending=True, stable=True)[1][..., :budget]  # ties: the lowest first
    new = lens.clamp(max=budget)
    i = torch.arange(order.shape[-1], device=DEV)
    live = (i < new[:, None, None]).expand(order.shape)
    kept = torch.sort(torch.where(live, order, S), -1)[0]
    at = torch.where(live, kept, 0)
    s["weights"][..., :at.shape[-1]] = torch.where(live, s["weights"].gather(-1, at),
                                                   s["weights"][..., :at.shape[-1]])
    b, h = (torch.arange(k, device=DEV).view(v) for k, v in ((B, (B, 1, 1)), (Hkv, (1, Hkv, 1))))
    page, off = s["blocks"].long()[b, at // bs], at % bs
    codes, scale = s["cache"][:, page, h, off], s["scale"][:, page, h]
    blocks = -(-at.shape[-1] // bs)
    pad = torch.nn.functional.pad(torch.where(live, scale, 0), (0, blocks * bs - at.shape[-1]))
    fresh = pad.unflatten(-1, (blocks, bs)).amax(-1).clamp_min(FLOOR)  # [2, B, Hkv, blocks]
    codes = torch.round(codes * (scale / fresh[..., i // bs])[..., None]).to(torch.int8)
    bb, hh, ii = live.nonzero(as_tuple=True)
    to = s["to"].long()[bb, ii // bs]
    s["cache"][:, to, hh, ii % bs] = codes[:, bb, hh, ii]
    s["scale"][:, to, hh] = fresh[:, bb, hh, ii // bs]
    kept = torch.where(live, kept, -1).to(torch.int32)
    return new.to(torch.int32), torch.nn.functional.pad(kept, (0, budget - kept.shape[-1]), value=-1)


def run(state: dict):
    s, c = state, state["case"]
    if own:
        import superl8_amd as sl8
    if c["kind"] == "linear":
        if not own:
            return _plain_linear(s)
        return sl8.linear_w8a8(s["x"], s["w"], s["ws"], bias=s["bias"], out_dtype=DTYPES[c["out"]])
    if c["kind"] == "tree":
        if not own:
            return _plain_tree(s)
        return sl8.attn_paged_block8(s["q"], s["cache"][0], s["scale"][0], s["cache"][1], s["scale"][1],
                                     s["blocks"], s["lens"], cu_lens=s["cu"], rotate=c["rotate"],
                                     window_left=c["window"], tree_mask=s["mask"], return_lse=c["lse"])
    if c["kind"] == "weights":
        if not own:
            return _plain_weights(s)
        sl8.attn_weights_block8(s["q"], s["lse"], s["cache"][0], s["scale"][0], s["blocks"], s["lens"],
                                s["weights"], cu_lens=s["cu"], rotate=c["rotate"], window_left=c["window"],
                                decay=c["decay"])
        return s["weights"]
    if own:
        lens, kept = sl8.kv_evict_block8(s["cache"][0], s["scale"][0], s["cache"][1], s["scale"][1], s["blocks"],
                                         s["lens"], s["weights"], s["to"], budget=c["budget"], sinks=c["sinks"],
                                         recent=c["recent"])
    else:
        lens, kept = _plain_evict(s)
    # what the blocks that were written now stand for
    nd = s["values"].shape[1]
    torch.mul(s["cache"][:, :nd], s["scale"][:, :nd, :, None, None], out=s["values"])
    return lens, kept, s["weights"], s["values"], s["scale"][:, :nd]


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case: dict) -> dict:
    c = case
    if c["kind"] == "linear":
        M, N, K = c["M"], c["N"], c["K"]
        size = 4 if c["out"] == "fp32" else 2
        return {"bytes": 2 * M * K + N * K + 4 * N + 2 * N * c["bias"] + size * M * N,
                "flops": 2 * M * N * K}
    new, old = _lens(c)
    T, bs, Hkv, D = sum(new), c["block"], c["Hkv"], c["D"]
    total = [a + b for a, b in zip(new, old)]
    if c["kind"] == "evict":
        kept = [min(n, c["budget"]) for n in total]
        blocks = sum(-(-n // bs) for n in kept)
        # the weights read, the kept ones and their places written; the kept rows read and written; the
        # blocks' codes as the values that they stand for, and their scales
        return {"bytes": Hkv * (4 * sum(total) + 8 * sum(kept) + 4 * D * sum(kept) + blocks * 2 * (bs * D * 3 + 8)),
                "flops": 2 * 2 * Hkv * D * sum(kept)}
    keys = pairs = 0
    for n, o in zip(new, old):
        first = max(0, o - c["window"] + 1) if c["window"] >= 0 else 0
        keys += o + n - first
        if c["kind"] == "tree":
            pairs += n * (o - first + 1 + round(math.log2(n)))
        else:
            pairs += sum(min(o + i + 1, c["window"]) if c["window"] >= 0 else o + i + 1 for i in range(n))
    if c["kind"] == "tree":
        return {"bytes": keys * Hkv * 2 * D + 2 * Hkv * 4 * (keys // bs) + 4 * T * c["Hq"] * D + 8 * T * _words(c)
                + 4 * T * c["Hq"] * c["lse"], "flops": 4 * pairs * c["Hq"] * D}
    # with no fading the weights of keys that no row sees stay as they are
    held = sum(total) if c["decay"] != 1 else keys
    return {"bytes": keys * Hkv * D + Hkv * 4 * (keys // bs) + T * c["Hq"] * (2 * D + 4) + 8 * Hkv * held,
            "flops": 2 * pairs * c["Hq"] * D}


# ---------------------------------------------------------------------------
# the same outputs in 64 bits, from the definitions
# ---------------------------------------------------------------------------
def _exact_codes(x):
    """Rows as int8 codes and their scales; scales and quotients are fp32 numbers by definition."""
    step = x.abs().amax(-1, keepdim=True).float() * torch.tensor(1 / 127, device=DEV)
    step = torch.where(step == 0, 1.0, step).double()
    return torch.round((x / step).float()).clamp(-127, 127).double(), step


def _exact_linear(c, seed):
    s = prepare(c, seed)
    out = []
    for x in s["x"].split(1024):
        codes, step = _exact_codes(x.double())
        y = torch.cat([codes @ w.double().T for w in s["w"].split(8192)], 1) * step * s["ws"].double()
        out.append(y if s["bias"] is None else y + s["bias"].double())
    return torch.cat(out)


def _exact_rows(s, t, b, h):
    """Keys, values (64 bits) and rows of sequence b and KV head h: what each row's scores are."""
    c = s["case"]
    new, old = _lens(c)
    n, G = old[b] + new[b], c["Hq"] // c["Hkv"]
    pages = s["blocks"][b, :-(-n // c["block"])].long()
    k, v = ((s["cache"][j, pages, h].double() * s["scale"][j, pages, h].double()[:, None, None])
            .flatten(0, 1)[:n] for j in (0, 1))
    q = s["q"][t:t + new[b], h * G:(h + 1) * G].double()
    if c["rotate"]:
        q = q @ _hadamard(c["D"])
    codes, step = _exact_codes(q)
    return k, v, (codes * step).transpose(0, 1) / math.sqrt(c["D"])  # [G, new, D]


def _exact_tree(c, seed):
    s = prepare(c, seed)
    new, old = _lens(c)
    G = c["Hq"] // c["Hkv"]
    out = torch.zeros(s["q"].shape, device=DEV, dtype=torch.float64)
    lse = torch.zeros(s["q"].shape[:2], device=DEV, dtype=torch.float64)
    t = 0
    for b in range(c["B"]):
        n = old[b] + new[b]
        ok = torch.zeros(new[b], n, dtype=torch.bool)
        for i, words in enumerate(s["mask"][t:t + new[b]].tolist()):
            marked = [j for j in range(new[b]) if words[j // 64] >> (j % 64) & 1]
            first = max(0, old[b] - max(0, c["window"] - len(marked))) if c["window"] >= 0 else 0
            ok[i, first:old[b]] = True
            ok[i, [old[b] + j for j in marked]] = True
        ok = ok.to(DEV)
        for h in range(c["Hkv"]):
            k, v, q = _exact_rows(s, t, b, h)
            for g in range(G):
                w = (q[g] @ k.T).masked_fill(~ok, -math.inf)
                out[t:t + new[b], h * G + g] = torch.softmax(w, -1) @ v
                lse[t:t + new[b], h * G + g] = torch.logsumexp(w, -1)
        t += new[b]
    return (out, lse) if c["lse"] else out


def _exact_weights(c, seed):
    s = prepare(c, seed)
    new, old = _lens(c)
    out, t, G = s["weights"].double(), 0, c["Hq"] // c["Hkv"]
    for b in range(c["B"]):
        n = old[b] + new[b]
        i = torch.arange(old[b], n, device=DEV)[:, None]
        j = torch.arange(n, device=DEV)
        hide = j > i
        if c["window"] >= 0:
            hide |= j <= i - c["window"]
        for h in range(c["Hkv"]):
            k, _, q = _exact_rows(s, t, b, h)
            row = out[b, h, :n]
            row[:old[b]] *= c["decay"]
            row[old[b]:] = 0
            for g in range(G):
                w = (q[g] @ k.T).masked_fill(hide, -math.inf)
                row += (w - s["lse"][t:t + new[b], h * G + g].double()[:, None]).exp().sum(0)
        t += new[b]
    return out


def _exact_evict(c, seed):
    s = prepare(c, seed)
    _, old = _lens(c)
    bs, S = c["block"], s["weights"].shape[-1]
    nd = s["values"].shape[1]
    codes, scale = s["cache"][:, :nd].double(), s["scale"][:, :nd].double()
    weights = s["weights"].double()
    kept = torch.full((c["B"], c["Hkv"], c["budget"]), -1, device=DEV, dtype=torch.int32)
    lens = []
    for b in range(c["B"]):
        n = old[b] + 1
        m = min(n, c["budget"])
        lens.append(m)
        first = min(c["sinks"], n)
        last = max(first, n - c["recent"])
        for h in range(c["Hkv"]):
            keep = torch.arange(n, device=DEV)
            if n > m:
                between = torch.argsort(-s["weights"][b, h, first:last], stable=True)[:m - first - (n - last)]
                keep = torch.cat([keep[:first], first + between.sort()[0], keep[last:]])
            kept[b, h, :m] = keep.to(torch.int32)
            weights[b, h, :m] = s["weights"][b, h, keep].double()
            pages = s["blocks"][b, keep // bs].long()
            for x in (0, 1):
                was = s["scale"][x, pages, h].double()
                rows = s["cache"][x, pages, h, keep % bs].double()
                for blk, (r, w) in enumerate(zip(rows.split(bs), was.split(bs))):
                    to = w.max().clamp_min(FLOOR)
                    page = s["to"][b, blk].long()
                    scale[x, page, h] = to
                    codes[x, page, h, :r.shape[0]] = torch.round(r * (w / to)[:, None])
    return _i32(lens), kept, weights, codes * scale[..., None, None], scale


def exact(case: dict, seed: int):
    # (an eviction's blocks are gone through one by one)
    if case["kind"] == "evict" and case["B"] * case["Hkv"] * case["budget"] / case["block"] > 20000:
        return None
    return {"linear": _exact_linear, "tree": _exact_tree, "weights": _exact_weights,
            "evict": _exact_evict}[case["kind"]](case, seed)
