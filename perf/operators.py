"""Performance cases of three operators that a model served from a block-scaled paged cache uses.

  rope     `rope`: rotary positions of one to four axes on Q and K, or their gradient (`inverse`)
  append   `quantize_kv_append_block8`: a step's K/V, rotated by position on the way, into a paged
           int8 cache that holds one scale per block of tokens and head; the rotated Q comes back
  attn     `attn_paged_block8`: attention of one to thousands of new tokens per sequence over
           that cache

`listed()` holds workloads of serving and training; `draw` samples the ranges that they stand
for. A case is a dict of plain values. With `own` false `run` computes the operators' plain forms
in elementary torch operations, with `own` true it calls this package.
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
def _text(sections) -> str:
    """Pairs per axis as a plain value: "16,24,24"; one axis: nothing."""
    return ",".join(map(str, sections))


def _sections(c) -> list[int]:
    return [int(x) for x in c["sections"].split(",")] if c["sections"] else []


def _rope(B, Hq, Hkv, S, D, R=0, sections=(), dtype="fp16", interleaved=False, inverse=False):
    return dict(kind="rope", B=B, Hq=Hq, Hkv=Hkv, S=S, D=D, R=R or D, sections=_text(sections),
                dtype=dtype, interleaved=interleaved, inverse=inverse)


def _append(B, new, old, Hq, Hkv, D, block, R=0, sections=(), dtype="fp16", interleaved=False,
            rotate=True):
    """B sequences that hold about `old` tokens get about `new` each (see _lens)."""
    return dict(kind="append", B=B, new=new, old=old, Hq=Hq, Hkv=Hkv, D=D, block=block, R=R or D,
                sections=_text(sections), dtype=dtype, interleaved=interleaved, rotate=rotate)


def _attn(B, new, old, Hq, Hkv, D, block, dtype="fp16", rotate=True, window=-1, spread=True):
    return dict(kind="attn", B=B, new=new, old=old, Hq=Hq, Hkv=Hkv, D=D, block=block, dtype=dtype,
                rotate=rotate, window=window, spread=spread)


def listed() -> list[dict]:
    return [
        # one new token of each of 64 sequences: launches and latency count
        dict(name="rope_step", **_rope(64, 32, 8, 1, 128)),
        # a video prompt: positions in time, height and width, Q and K views of one projection
        dict(name="rope_video_bf16", **_rope(1, 32, 8, 6121, 128, sections=(16, 24, 24),
                                             dtype="bf16")),
        # a vision tower of 80-wide heads in training: the gradient through positions in two axes
        dict(name="rope_vision_grad", **_rope(4, 16, 16, 4096, 80, sections=(20, 20),
                                              dtype="fp32", inverse=True)),
        # a decode step of 32 sequences: the smallest append
        dict(name="append_step", **_append(32, 1, 40, 32, 8, 128, 16)),
        # five drafted tokens of 16 sequences, rotary positions on a part of wide heads
        dict(name="append_draft_d256", **_append(16, 5, 70, 16, 2, 256, 32, R=64, interleaved=True,
                                                 rotate=False)),
        # four prompts of mixed lengths with positions in three axes, bf16
        dict(name="append_prompts_bf16", **_append(4, 2500, 20, 32, 8, 128, 64,
                                                   sections=(16, 24, 24), dtype="bf16")),
        # one token of one short conversation: the smallest attention
        dict(name="attn_one", **_attn(1, 1, 776, 32, 8, 128, 16)),
        # serving: one token of each of 32 sequences of mixed lengths
        dict(name="attn_step_mixed", **_attn(32, 1, 8191, 32, 8, 128, 16)),
        # long contexts of one length: the largest stream of bytes
        dict(name="attn_step_32k_bf16", **_attn(16, 1, 32767, 32, 8, 128, 64, dtype="bf16",
                                                spread=False)),
        # a pending token and four drafted ones per sequence, eight query heads to a KV head
        dict(name="attn_draft_bf16", **_attn(16, 5, 16379, 64, 8, 128, 32, dtype="bf16")),
        # a chunk of a long prompt behind its cached prefix: the most arithmetic
        dict(name="attn_chunk_16k", **_attn(1, 2048, 14336, 32, 8, 128, 16)),
        # chunks of mixed odd lengths, 64-wide heads, a sliding window
        dict(name="attn_ragged_window", **_attn(6, 1301, 5003, 16, 4, 64, 32, rotate=False,
                                                window=1024)),
    ]


def _log(rng: random.Random, lo: float, hi: float) -> int:
    return max(int(lo), min(int(hi), round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _heads(rng: random.Random) -> tuple[int, int]:
    hkv = rng.choice([1, 2, 4, 8])
    return hkv * rng.choice([1, 2, 4, 8] if hkv < 8 else [1, 2, 4]), hkv


def _axes(rng: random.Random, R: int) -> list[int]:
    """One axis, or R / 2 pairs shared out among two to four."""
    n = rng.choice([1, 1, 2, 3, 4])
    cuts = sorted(rng.sample(range(1, R // 2), n - 1))
    return [b - a for a, b in zip([0] + cuts, cuts + [R // 2])] if n > 1 else []


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["rope", "append", "attn", "attn"])
    hq, hkv = _heads(rng)
    dtype = rng.choice(["fp16", "bf16"])
    if kind == "rope":
        D = rng.choice([64, 72, 80, 128, 128, 256])
        R = rng.choice([D, D, D // 2])
        if rng.random() < 0.25:
            dtype = "fp32"
        B = _log(rng, 1, 64)
        S = _log(rng, 1, max(1, 20000000 // (B * (hq + hkv) * D)))
        return _rope(B, hq, hkv, S, D, R, _axes(rng, R), dtype, interleaved=rng.random() < 0.3,
                     inverse=rng.random() < 0.3)
    D, block = rng.choice([64, 128, 128, 256]), rng.choice([16, 32, 64, 128])
    if kind == "append":
        B = _log(rng, 1, 128)
        new = _log(rng, 1, max(1, 30000000 // (B * (hq + 2 * hkv) * D)))
        R = rng.choice([D, D, D // 2])
        return _append(B, new, _log(rng, 1, 300), hq, hkv, D, block, R, _axes(rng, R), dtype,
                       interleaved=rng.random() < 0.3, rotate=rng.random() < 0.7)
    spread = rng.random() < 0.8
    rotate = rng.random() < 0.7
    if rng.random() < 0.6:  # a step of one to 16 tokens a sequence
        B = _log(rng, 1, 64)
        most = (1 << 28) // (B * hkv * D)
        return _attn(B, rng.choice([1, 1, _log(rng, 2, 16)]), _log(rng, 60, min(65000, most)), hq,
                     hkv, D, block, dtype, rotate, -1 if rng.random() < 0.8 else 1000, spread)
    B, new = _log(rng, 1, 6), _log(rng, 17, 1500)
    most = 120000000000 // (4 * B * hq * D * new)
    return _attn(B, new, _log(rng, 1, max(2, min(30000, most))), hq, hkv, D, block, dtype, rotate,
                 -1 if rng.random() < 0.7 else _log(rng, 64, 2000), spread)


def _lens(c) -> tuple[list[int], list[int]]:
    """New tokens and lengths before them of each sequence. Up to 16 new tokens: the same of each;
    more: odd lengths from new / 2 to new. Old lengths: spread evenly (in the logarithm) over a
    factor of 16, or the same."""
    B = c["B"]
    new = [c["new"]] * B
    if c["new"] > 16 and B > 1:
        new = [max(1, round(c["new"] * 2 ** -(i / (B - 1)))) | 1 for i in range(B)]
    if c["kind"] == "attn" and c["spread"]:
        old = [max(1, round(c["old"] * 16 ** -(i / max(1, B - 1)))) for i in range(B)]
    else:
        old = [c["old"]] * B
        if c["kind"] == "append":  # starting at different places of a block, some of them at its first
            old = [max(0, c["old"] - 5 * i) for i in range(B)]
    random.Random(c["B"]).shuffle(old)
    return new, old


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _table(n: int, pairs: int, axes: list[int]) -> torch.Tensor:
    """cos | sin of position * 10000^(-pair / pairs), from 64 bits; with two axes (images) the
    frequencies start again at each."""
    i = torch.arange(pairs, device=DEV, dtype=torch.float64)
    i = i / pairs if len(axes) != 2 else torch.cat([i[:a] / a for a in axes])
    a = torch.arange(n, device=DEV, dtype=torch.float64)[:, None] * 10000.0 ** -i
    return torch.cat([a.cos(), a.sin()], 1).float()


def _codes(g, *shape):
    """int8 codes of normal values in blocks whose largest is 3.5 deviations."""
    out = torch.empty(*shape, device=DEV, dtype=torch.int8)
    for part in out.flatten().split(1 << 27):
        part.copy_((torch.randn(part.shape, device=DEV, generator=g, dtype=torch.float16) * 36)
                   .round_().clamp_(-127, 127))
    return out


def _pool(c, g, total: list[int]):
    """A pool of blocks in shuffled order, a few more than the sequences take, with their table."""
    bs = c["block"]
    most = max(-(-n // bs) for n in total)
    used = sum(-(-n // bs) for n in total)
    nb = used + 3
    order = torch.randperm(nb, device=DEV, generator=g).to(torch.int32)
    rows, at = [], 0
    for n in total:
        k = -(-n // bs)
        rows.append(torch.cat([order[at:at + k], order.new_zeros(most - k)]))
        at += k
    cache = _codes(g, 2, nb, c["Hkv"], bs, c["D"])
    scale = (torch.rand(2, nb, c["Hkv"], device=DEV, generator=g) * 0.4 + 0.8) * (3.5 / 127)
    return cache, scale, torch.stack(rows)


def _offsets(new: list[int]) -> torch.Tensor:
    return torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], device=DEV, dtype=torch.int32)


def _hadamard(d: int, dtype=torch.float32) -> torch.Tensor:
    h = torch.ones(1, 1, device=DEV, dtype=torch.float64)
    while h.shape[0] < d:
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
    return (h / math.sqrt(d)).to(dtype)


def prepare(case: dict, seed: int) -> dict:
    c, g, dt = case, _gen(seed), DTYPES[case["dtype"]]
    if c["kind"] == "rope":
        B, Hq, Hkv, S, D = (c[x] for x in ("B", "Hq", "Hkv", "S", "D"))
        # what a fused projection gives: Q and K are views of its rows (a gradient comes as such)
        x = torch.randn(B, S, Hq + 2 * Hkv, D, device=DEV, generator=g).to(dt)
        q, k = x[:, :, :Hq].transpose(1, 2), x[:, :, Hq:Hq + Hkv].transpose(1, 2)
        n = 8192 if S > 1 else 32768
        axes = len(_sections(c))
        shape = (axes, B, S) if axes else (B, S)
        pos = torch.randint(0, n, shape, device=DEV, generator=g)
        return {"case": c, "q": q, "k": k, "pos": pos, "table": _table(n, c["R"] // 2, _sections(c))}
    new, old = _lens(c)
    total = [a + b for a, b in zip(new, old)]
    cache, scale, blocks = _pool(c, g, total)
    s = {"case": c, "cache": cache, "scale": scale, "blocks": blocks,
         "lens": torch.tensor(total, device=DEV, dtype=torch.int32), "cu": _offsets(new),
         "hadamard": _hadamard(c["D"])}
    T = sum(new)
    if c["kind"] == "attn":
        s["q"] = (torch.randn(T, c["Hq"], c["D"], device=DEV, generator=g) * 2).to(dt)
        return s
    x = torch.randn(T, c["Hq"] + 2 * c["Hkv"], c["D"], device=DEV, generator=g)
    x[:, c["Hq"]:] *= 0.5 + 1.5 * torch.rand(T, 1, 1, device=DEV, generator=g)
    s["q"], s["k"], s["v"] = x.to(dt).split([c["Hq"], c["Hkv"], c["Hkv"]], 1)
    axes = len(_sections(c))
    s["pos"] = torch.randint(0, 8192, (axes, T) if axes else (T,), device=DEV, generator=g)
    s["table"] = _table(8192, c["R"] // 2, _sections(c))
    s["values"] = torch.empty(cache.shape, device=DEV, dtype=dt)
    return s


# ---------------------------------------------------------------------------
# the plain forms, in 32 bits
# ---------------------------------------------------------------------------
def _angles(table, pos, sections):
    """cos and sin of each position and pair: [..., pairs]."""
    half = table.shape[1] // 2
    if not sections:
        row = table[pos.long()]
        return row[..., :half], row[..., half:]
    axis = torch.repeat_interleave(torch.arange(len(sections), device=table.device),
                                   torch.tensor(sections, device=table.device), output_size=half)
    at = pos.long()[axis].movedim(0, -1)
    i = torch.arange(half, device=table.device)
    return table[at, i], table[at, half + i]


def _turn(x, cos, sin, interleaved):
    """The pairs of x's first 2 * pairs elements turned by their angles; the rest as they are."""
    half = cos.shape[-1]
    y, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = y[..., 0::2], y[..., 1::2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = y[..., :half], y[..., half:]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([y, rest], -1)


def _plain_rope(s):
    c = s["case"]
    cos, sin = (t.unsqueeze(1) for t in _angles(s["table"], s["pos"], _sections(c)))
    if c["inverse"]:
        sin = -sin
    return tuple(_turn(x.float(), cos, sin, c["interleaved"]).to(x.dtype) for x in (s["q"], s["k"]))


def _tokens(s):
    """Sequence and place in its new tokens of every token, and the length before them."""
    cu = s["cu"].long()
    t = torch.arange(s["q"].shape[0], device=cu.device)
    b = torch.searchsorted(cu, t, right=True) - 1
    return b, t - cu[b], s["lens"].long() - (cu[1:] - cu[:-1])


def _plain_append(s):
    c = s["case"]
    cache, scale, bs = s["cache"], s["scale"], c["block"]
    cos, sin = (t.unsqueeze(1) for t in _angles(s["table"], s["pos"], _sections(c)))
    q, k = (_turn(x.float(), cos, sin, c["interleaved"]) for x in (s["q"], s["k"]))
    if c["rotate"]:
        k = k @ s["hadamard"]
    x = torch.stack([k, s["v"].float()])  # [2, T, Hkv, D]
    b, i, before = _tokens(s)
    slot = before[b] + i
    page, off = s["blocks"][b, slot // bs].long(), slot % bs
    # slots that a block keeps: those before the first new token of its sequence
    keep = torch.zeros(cache.shape[1], device=DEV, dtype=torch.long)
    first = s["blocks"].gather(1, (before // bs)[:, None])[:, 0].long()
    keep[first] = before % bs
    touched = torch.zeros(cache.shape[1], device=DEV, dtype=torch.bool)
    touched[page] = True
    amax = torch.zeros_like(scale).index_reduce_(1, page, x.abs().amax(-1), "amax")
    kept = torch.where((keep > 0)[:, None], scale, 0)
    fresh = torch.maximum(kept, amax * torch.tensor(1 / 127, device=DEV)).clamp_min(FLOOR)
    new = torch.where(touched[:, None], fresh, scale)
    held = (torch.arange(bs, device=DEV) < keep[:, None])[:, None, :, None] & touched[:, None, None, None]
    again = torch.round(cache * (scale / new)[..., None, None]).to(torch.int8)
    cache.copy_(torch.where(held, again, cache))
    scale.copy_(new)
    codes = torch.round(x / new[:, page][..., None]).clamp(-127, 127).to(torch.int8)
    cache[:, page, :, off] = codes.permute(1, 0, 2, 3)
    return q.to(s["q"].dtype)


def _plain_attn(s):
    c, q = s["case"], s["q"]
    B, Hq, Hkv, D, M = c["B"], c["Hq"], c["Hkv"], c["D"], c["new"] | (c["new"] > 16)
    G = Hq // Hkv
    x = q.float()
    if c["rotate"]:
        x = x @ s["hadamard"]
    # the query rows in int8, one scale each
    qs = x.abs().amax(-1, keepdim=True) * torch.tensor(1 / 127, device=DEV)
    qs = torch.where(qs == 0, 1.0, qs)
    x = torch.round(x / qs).clamp(-127, 127)
    b, i, before = _tokens(s)
    cu, lens = s["cu"].long(), s["lens"].long()
    at = cu[:-1, None] + torch.arange(M, device=DEV)
    at = at.clamp(max=q.shape[0] - 1)  # rows past a sequence's last are computed and not taken

    def rows(t):  # [T, Hq, n] -> [B, Hkv, G * M, n]
        return t[at].reshape(B, M, Hkv, G, -1).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * M, -1)

    def keys(j):  # codes of every sequence's blocks, [B, Hkv, N, D] and their scales [B, Hkv, N]
        t = s["blocks"].long()
        x = s["cache"][j][t].transpose(1, 2).flatten(2, 3).float()
        return x, s["scale"][j][t].transpose(1, 2).repeat_interleave(c["block"], 2)

    k, ks = keys(0)
    w = rows(x) @ k.transpose(2, 3).contiguous()
    del k
    w *= rows(qs) * (1 / math.sqrt(D))
    w *= ks[:, :, None]
    n = torch.arange(w.shape[-1], device=DEV)
    last = (before[:, None] + torch.arange(M, device=DEV)).repeat(1, G)[:, None, :, None]
    seen = (n <= last) & (n < lens[:, None, None, None])
    if c["window"] >= 0:
        seen &= n > last - c["window"]
    w.masked_fill_(~seen, -math.inf)
    w -= w.amax(-1, keepdim=True).clamp_min(-1e30)
    w.exp_()
    total = w.sum(-1, keepdim=True)
    v, vs = keys(1)
    w *= vs[:, :, None]
    out = (w @ v) / torch.where(total == 0, 1.0, total)
    out = out.reshape(B, Hkv, G, M, D).permute(0, 3, 1, 2, 4).reshape(B, M, Hq, D)
    return out[b, i].to(q.dtype)


def run(state: dict):
    s, c = state, state["case"]
    if c["kind"] == "rope":
        if not own:
            return _plain_rope(s)
        import superl8_amd as sl8
        return sl8.rope(s["q"], s["k"], s["pos"], s["table"], sections=_sections(c) or None,
                        interleaved=c["interleaved"], inverse=c["inverse"])
    if c["kind"] == "append":
        if own:
            import superl8_amd as sl8
            q = sl8.quantize_kv_append_block8(
                s["k"], s["v"], s["cache"][0], s["scale"][0], s["cache"][1], s["scale"][1],
                s["blocks"], s["lens"], cu_lens=s["cu"], q=s["q"], positions=s["pos"],
                table=s["table"], sections=_sections(c) or None, interleaved=c["interleaved"],
                rotate=c["rotate"])
        else:
            q = _plain_append(s)
        # what the cache now stands for
        torch.mul(s["cache"], s["scale"][..., None, None], out=s["values"])
        return q, s["values"], s["scale"]
    if not own:
        return _plain_attn(s)
    import superl8_amd as sl8
    return sl8.attn_paged_block8(s["q"], s["cache"][0], s["scale"][0], s["cache"][1], s["scale"][1],
                                 s["blocks"], s["lens"], cu_lens=s["cu"], rotate=c["rotate"],
                                 window_left=c["window"])


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case: dict) -> dict:
    c, size = case, 4 if case["dtype"] == "fp32" else 2
    D, axes = c["D"], max(1, len(_sections(c))) if "sections" in c else 0
    if c["kind"] == "rope":
        T = c["B"] * c["S"]
        n = T * (c["Hq"] + c["Hkv"])
        return {"bytes": 2 * size * n * D + 8 * axes * T + 4 * T * c["R"], "flops": 3 * n * c["R"]}
    new, old = _lens(c)
    T, bs, Hkv = sum(new), c["block"], c["Hkv"]
    total = [a + b for a, b in zip(new, old)]
    if c["kind"] == "append":
        blocks = sum(-(-n // bs) for n in total) + 3
        # Q in and out, K and V in, positions and their angles; the blocks' codes as the values
        # that they stand for, read once and written once, and their scales
        elems = 2 * T * Hkv * D
        rot = 2 * T * Hkv * D * int(math.log2(D)) if c["rotate"] else 0
        return {"bytes": 2 * (2 * T * c["Hq"] * D + elems) + 8 * axes * T + 4 * T * c["R"]
                + 2 * blocks * Hkv * (bs * D * 3 + 8),
                "flops": 3 * T * (c["Hq"] + Hkv) * c["R"] + 4 * elems + rot}
    keys = pairs = 0
    for n, o in zip(new, old):
        first = max(0, o - c["window"] + 1) if c["window"] >= 0 else 0
        keys += o + n - first
        pairs += sum(min(o + i + 1, c["window"]) if c["window"] >= 0 else o + i + 1 for i in range(n))
    return {"bytes": keys * Hkv * 2 * D + 2 * Hkv * 4 * (keys // bs) + 4 * T * c["Hq"] * D,
            "flops": 4 * pairs * c["Hq"] * D}


# ---------------------------------------------------------------------------
# the same outputs in 64 bits, from the definitions
# ---------------------------------------------------------------------------
def _exact_turn(c, x, pos, table):
    """x [tokens, heads, D] with pair p of its first R elements turned by the angle of its axis."""
    R, out = c["R"], x.double().clone()
    sections = _sections(c) or [R // 2]
    pos = pos if c["sections"] else pos[None]
    p = 0
    for axis, n in enumerate(sections):
        for pair in range(p, p + n):
            i, j = (2 * pair, 2 * pair + 1) if c["interleaved"] else (pair, pair + R // 2)
            co = table[pos[axis].long(), pair].double()[:, None]
            si = table[pos[axis].long(), pair + R // 2].double()[:, None]
            if c.get("inverse"):
                si = -si
            out[..., i] = co * x[..., i].double() - si * x[..., j].double()
            out[..., j] = si * x[..., i].double() + co * x[..., j].double()
        p += n
    return out


def _exact_rope(c, seed):
    s = prepare(c, seed)
    B, S, D = c["B"], c["S"], c["D"]
    pos = s["pos"].flatten(-2)
    return tuple(_exact_turn(c, x.transpose(1, 2).reshape(B * S, -1, D), pos, s["table"])
                 .reshape(B, S, -1, D).transpose(1, 2) for x in (s["q"], s["k"]))


def _exact_append(c, seed):
    s = prepare(c, seed)
    new, old = _lens(c)
    bs = c["block"]
    q, k = (_exact_turn(c, s[x], s["pos"], s["table"]) for x in ("q", "k"))
    if c["rotate"]:
        k = k @ _hadamard(c["D"], torch.float64)
    codes, scale = s["cache"].double(), s["scale"].double()
    for j, x in enumerate((k, s["v"].double())):
        t = 0
        for b in range(c["B"]):
            at, end = old[b], old[b] + new[b]
            while at < end:
                page, off = int(s["blocks"][b, at // bs]), at % bs
                n = min(bs - off, end - at)
                rows = x[t:t + n].transpose(0, 1)  # [Hkv, n, D]
                was = scale[j, page].clone()
                to = (rows.abs().amax((1, 2)) / 127).clamp_min(FLOOR)
                if off:
                    to = torch.maximum(to, was)
                    codes[j, page, :, :off] = torch.round(codes[j, page, :, :off] * (was / to)[:, None, None])
                codes[j, page, :, off:off + n] = torch.round(rows / to[:, None, None])
                scale[j, page] = to
                at, t = at + n, t + n
    return q, codes * scale[..., None, None], scale


def _exact_attn(c, seed):
    s = prepare(c, seed)
    new, old = _lens(c)
    G, D, bs = c["Hq"] // c["Hkv"], c["D"], c["block"]
    q = s["q"].double()
    if c["rotate"]:
        q = q @ _hadamard(D, torch.float64)
    step = q.abs().amax(-1, keepdim=True) / 127
    q = torch.round(q / step) * step
    out = torch.zeros_like(q)
    t = 0
    for b in range(c["B"]):
        n = old[b] + new[b]
        pages = s["blocks"][b, :-(-n // bs)].long()
        i = torch.arange(old[b], n, device=DEV).repeat(G)[:, None]
        for h in range(c["Hkv"]):
            k, v = ((s["cache"][j, pages, h].double() * s["scale"][j, pages, h].double()[:, None, None])
                    .flatten(0, 1)[:n] for j in (0, 1))
            rows = q[t:t + new[b], h * G:(h + 1) * G].transpose(0, 1).reshape(-1, D)
            res = torch.empty_like(rows)
            for r in range(0, rows.shape[0], 2048):
                part = slice(r, r + 2048)
                w = rows[part] @ k.T / math.sqrt(D)
                j = torch.arange(n, device=DEV)
                w.masked_fill_(j > i[part], -math.inf)
                if c["window"] >= 0:
                    w.masked_fill_(j <= i[part] - c["window"], -math.inf)
                res[part] = torch.softmax(w, -1) @ v
            out[t:t + new[b], h * G:(h + 1) * G] = res.reshape(G, new[b], D).transpose(0, 1)
        t += new[b]
    return out


def exact(case: dict, seed: int):
    return {"rope": _exact_rope, "append": _exact_append, "attn": _exact_attn}[case["kind"]](case, seed)
