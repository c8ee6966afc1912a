"""Public operators of the hot path, drop-in for superl8/ops.py of the reference.

Same names, keyword arguments, routing and error behaviour as the reference
wrappers (reference superl8/ops.py:70-175 attn_int8_fwd, :230-267
attn_int8_decode, :531-584 quantize_kv_cache, :671-727 attn_decode_cached,
:730-849 quantize_kv_write_paged / attn_paged_decode_cached,
:975-991 quantize_i8_rowwise, :1254-1347 linear_q4k / linear_q5k / linear_q6k / _linear_kquant),
dispatching to the gfx950 kernels through `_C`.
"""
from __future__ import annotations

import math

import torch

from . import _C
from .quant.core import LOG2E
from .quant.rotation import hadamard_dim

# Decode-shape M cap for the k-quant linear (reference ops.py:1289).
_KQUANT_DECODE_MAX_M = 16


def attn_int8_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, causal: bool = False,
                  scale: float | None = None, int8_pv: bool = False, rotate: bool = False,
                  window_left: int = -1, per_warp_quant: bool = True,
                  internal_accuracy_gate: bool = True) -> torch.Tensor:
    """INT8-QK^T FlashAttention-2 prefill (MFMA), fp16/bf16 PV; ``int8_pv`` = full W8A8.

    q, k, v: fp16/bf16 [B, H, S, D]. Q/K are quantised per row (K smoothed) in
    the prologue; causal attention is bottom-right aligned; ``window_left>=0``
    adds a left window (fp16-PV path only). With ``internal_accuracy_gate``,
    a Q row whose max/median magnitude ratio exceeds 12 sends the whole call
    to full-precision attention (reference ops.py:115-147).
    """
    from . import quant

    if internal_accuracy_gate:
        fired, qk = quant.quantize_qk_gated(q, k, softmax_scale=scale, rotate=rotate,
                                            defer=False if int8_pv else "host")
    elif int8_pv and window_left < 0 and not rotate and quant.core.fused_ok(q, k, v):
        # one prologue for Q, K and V
        s = (1.0 / math.sqrt(q.shape[-1])) if scale is None else scale
        q_i8, q_scale, k_i8, k_scale, _k_mean, v_i8, v_scale = _C.quantize_qkv_fused(
            q, k, v, s * quant.LOG2E)
        return _C.attn_w8a8_fwd(q_i8, q_scale, k_i8, k_scale, v_i8, v_scale.squeeze(-2), causal,
                                causal_diag=k.shape[-2] - q.shape[-2] if causal else 0,
                                per_warp_quant=per_warp_quant)
    else:
        fired, qk = False, quant.quantize_qk(q, k, softmax_scale=scale, rotate=rotate)
    if isinstance(fired, tuple):
        # gate decided on the device: the prologue sets its flag in pinned host
        # memory too, the attention is launched behind it (it exits at once if
        # the gate fired), and the host waits only for the prologue -- not for
        # the attention, so the next call's prologue is queued while this
        # attention runs (a plain .item() after the launch would wait for the
        # attention and leave the GPU idle during the next enqueue)
        flag, flag_host, flag_ready = fired
        q_i8, q_scale, k_i8, k_scale, _k_mean = qk
        refused = None
        try:
            out = _C.attn_int8_fwd(q_i8, q_scale.squeeze(-1).contiguous(), k_i8,
                                   k_scale.squeeze(-1).contiguous(), v.contiguous(), causal,
                                   window_left, gate_flag=flag)
        except RuntimeError as e:  # a V that only full precision takes: the gate decides first
            refused = e
        finally:
            flag_ready.synchronize()  # before flag_host is read, or let go
        if int(flag_host[0]) == 0:
            if refused is not None:
                raise refused
            return out
        fired = True
    if fired:
        import torch.nn.functional as F

        s = (1.0 / math.sqrt(q.shape[-1])) if scale is None else scale
        attn_mask = None
        if causal and q.shape[-2] != k.shape[-2]:
            m, n = q.shape[-2], k.shape[-2]
            attn_mask = torch.ones(m, n, device=q.device, dtype=torch.bool).tril(n - m)
        if window_left >= 0:
            m, n = q.shape[-2], k.shape[-2]
            i = torch.arange(m, device=q.device)[:, None] + (n - m)
            j = torch.arange(n, device=q.device)[None, :]
            attn_mask = (j <= i) & (j > i - window_left)
        return F.scaled_dot_product_attention(
            q, k, v.to(q.dtype) if v.dtype != q.dtype else v, attn_mask=attn_mask,
            is_causal=causal and attn_mask is None, scale=s,
            enable_gqa=q.shape[1] != k.shape[1]).to(v.dtype)

    q_i8, q_scale, k_i8, k_scale, _k_mean = qk
    q_scale = q_scale.squeeze(-1).contiguous()
    k_scale = k_scale.squeeze(-1).contiguous()
    if int8_pv:
        if window_left >= 0:
            raise ValueError("window_left is only supported on the fp16-PV path (int8_pv=False)")
        v_i8, v_scale = quant.quantize_v_perchannel(v)
        return _C.attn_w8a8_fwd(q_i8, q_scale, k_i8, k_scale, v_i8,
                                v_scale.squeeze(-2).contiguous(), causal,
                                causal_diag=k.shape[-2] - q.shape[-2] if causal else 0,
                                per_warp_quant=per_warp_quant)
    return _C.attn_int8_fwd(q_i8, q_scale, k_i8, k_scale, v.contiguous(), causal, window_left)


def attn_int8_decode(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
                     scale: float | None = None, rotate: bool = False,
                     num_splits: int | None = None) -> torch.Tensor:
    """Split-KV decode: q fp16 [B, Hq, 1, D] against k, v fp16 [B, Hkv, N, D]."""
    from .quant import quantize_qk

    if q.shape[-2] != 1:
        raise AssertionError(f"decode expects M=1, got M={q.shape[-2]}")
    q_i8, q_scale, k_i8, k_scale, _k_mean = quantize_qk(q, k, softmax_scale=scale, rotate=rotate)
    q_scale = q_scale.reshape(q.shape[0], q.shape[1], 1).contiguous()
    k_scale = k_scale.squeeze(-1).contiguous()
    ns = -1 if num_splits is None else int(num_splits)
    return _C.attn_int8_decode(q_i8, q_scale, k_i8, k_scale, v.contiguous(), ns)


def quantize_kv_cache(k: torch.Tensor, v: torch.Tensor, *, rotate: bool = False,
                      v_quant: str = "per_channel"):
    """Quantise a K/V cache once for persistent int8 storage (reference ops.py:531-584):
    K smoothed (+ optional Hadamard rotation) then per-row int8; V per-channel int8
    (v_scale [B,Hkv,D]) or, with v_quant="per_token", per-key int8 (v_scale [B,Hkv,N]).
    Returns (k_i8, k_scale [B,Hkv,N], v_i8, v_scale)."""
    from .quant import quantize_int8_rowwise, quantize_v_perchannel, quantize_v_rowwise, smooth_k

    if v_quant not in ("per_channel", "per_token"):
        raise ValueError(f"v_quant must be 'per_channel' or 'per_token', got {v_quant!r}")
    if rotate:
        hadamard_dim(k.shape[-1])
    if v_quant == "per_channel" and k.shape == v.shape and _C.prologue_ok(k, v):
        _, _, k_i8, k_scale, _, v_i8, v_scale = _C.quantize_qkv_fused(None, k, v, rotate=rotate)
        return k_i8, k_scale, v_i8, v_scale.squeeze(-2)
    k_s, _k_mean = smooth_k(k)
    if rotate:
        from .quant.rotation import rotate_last

        k_s = rotate_last(k_s)
    k_i8, k_scale = quantize_int8_rowwise(k_s)
    if v_quant == "per_channel":
        v_i8, v_scale = quantize_v_perchannel(v)
        v_scale = v_scale.squeeze(-2)
    else:
        v_i8, v_scale = quantize_v_rowwise(v)
        v_scale = v_scale.squeeze(-1)
    return k_i8.contiguous(), k_scale.squeeze(-1).contiguous(), v_i8.contiguous(), v_scale.contiguous()


def attn_decode_cached(q: torch.Tensor, k_i8: torch.Tensor, k_scale: torch.Tensor,
                       v_i8: torch.Tensor, v_scale: torch.Tensor, *, scale: float | None = None,
                       rotate: bool = False, num_splits: int | None = None) -> torch.Tensor:
    """Decode (M=1) against a pre-quantised int8 K/V cache from quantize_kv_cache
    (reference ops.py:671-727): only q is quantised per call. q fp16 [B,Hq,1,D] ->
    fp16 [B,Hq,1,D]; `rotate` must match the flag the cache was built with."""
    from .quant import LOG2E
    from .quant.rotation import rotate_last

    if q.shape[-2] != 1:
        raise AssertionError(f"decode expects M=1, got M={q.shape[-2]}")
    if v_scale.shape[-1] == k_i8.shape[2]:
        raise RuntimeError(
            "attn_decode_cached received a per-token V scale [B,H,N]; the contiguous int8-V "
            "decode kernel (attn_int8_decode_kv8) supports per-channel V scales [B,H,D] only")
    softmax_scale = (1.0 / (q.shape[-1] ** 0.5)) if scale is None else scale
    ns = -1 if num_splits is None else int(num_splits)
    q = q.contiguous()
    if _C.q16_ok(q):
        return _C.attn_int8_decode_kv8_q16(q, softmax_scale * LOG2E, rotate, k_i8.contiguous(),
                                           k_scale.contiguous(), v_i8.contiguous(),
                                           v_scale.contiguous(), ns)
    if rotate:
        q = rotate_last(q)
    q_shape = q.shape
    q_i8, q_scale = quantize_i8_rowwise(q.reshape(-1, q_shape[-1]).contiguous())
    q_i8 = q_i8.reshape(q_shape)
    q_scale = (q_scale.float() * (softmax_scale * LOG2E)).reshape(q_shape[0], q_shape[1], 1).contiguous()
    return _C.attn_int8_decode_kv8(q_i8.contiguous(), q_scale, k_i8.contiguous(),
                                   k_scale.contiguous(), v_i8.contiguous(), v_scale.contiguous(), ns)


def quantize_kv_write_paged(k_new: torch.Tensor, v_new: torch.Tensor, k_cache: torch.Tensor,
                            k_scale: torch.Tensor, v_cache: torch.Tensor, v_scale: torch.Tensor,
                            slot_mapping: torch.Tensor, *, rotate: bool = True) -> None:
    """Quantise-on-write of one new token per sequence into the paged int8 KV pool,
    in place (reference ops.py:730-775): per-token scales for K and V; `rotate`
    applies the Hadamard rotation to K (the smoothing usable one token at a time)."""
    if rotate:
        hadamard_dim(k_new.shape[-1])
    _C.kv_write_paged(k_new.contiguous(), v_new.contiguous(), slot_mapping.contiguous(),
                      k_cache, k_scale, v_cache, v_scale, rotate=rotate)


def attn_paged_decode_cached(q: torch.Tensor, k_cache: torch.Tensor, k_scale: torch.Tensor,
                             v_cache: torch.Tensor, v_scale: torch.Tensor,
                             block_table: torch.Tensor, context_lens: torch.Tensor,
                             block_size: int, *, max_context_len: int | None = None,
                             scale: float | None = None, rotate: bool = True,
                             num_splits: int | None = None) -> torch.Tensor:
    """Decode (M=1) against a paged int8 KV cache (reference ops.py:778-849): one
    launch for a batch of mixed-length sequences. `rotate` must match the flag the
    cache was written with; max_context_len defaults to max(context_lens) (a host sync)."""
    from .quant import LOG2E
    from .quant.rotation import rotate_last

    if q.shape[-2] != 1:
        raise AssertionError(f"paged decode expects M=1, got M={q.shape[-2]}")
    if max_context_len is None:
        max_context_len = int(context_lens.max().item())
    softmax_scale = (1.0 / (q.shape[-1] ** 0.5)) if scale is None else scale
    q = q.contiguous()
    if num_splits is None and _C.q16_ok(q):
        out = _C.attn_paged_decode_q16(q, softmax_scale * LOG2E, rotate, k_cache.contiguous(),
                                       k_scale.contiguous(), v_cache.contiguous(),
                                       v_scale.contiguous(), block_table.contiguous(),
                                       context_lens.contiguous(), int(block_size),
                                       int(max_context_len))
        if out is not None:
            return out
    if rotate:
        q = rotate_last(q)
    q_shape = q.shape
    q_i8, q_scale = quantize_i8_rowwise(q.reshape(-1, q_shape[-1]).contiguous())
    q_i8 = q_i8.reshape(q_shape)
    q_scale = (q_scale.float() * (softmax_scale * LOG2E)).reshape(q_shape[0], q_shape[1], 1).contiguous()
    ns = -1 if num_splits is None else int(num_splits)
    return _C.attn_paged_decode(q_i8.contiguous(), q_scale, k_cache.contiguous(),
                                k_scale.contiguous(), v_cache.contiguous(), v_scale.contiguous(),
                                block_table.contiguous(), context_lens.contiguous(),
                                int(block_size), int(max_context_len), ns)


def attn_paged_decode_k8v3(q: torch.Tensor, k_cache: torch.Tensor, k_scale: torch.Tensor,
                           v_packed: torch.Tensor, v_norm: torch.Tensor, v_codebook: torch.Tensor,
                           block_table: torch.Tensor, context_lens: torch.Tensor,
                           block_size: int, *, max_context_len: int | None = None,
                           scale: float | None = None, rotate: bool = True,
                           num_splits: int | None = None) -> torch.Tensor:
    """Decode (M=1) against a paged K8V3 store (reference ops.py:852-915): int8 K
    (rotated when `rotate`, per-token fp32 scale) and 3-bit Lloyd-Max V (packed
    codes int32 [num_blocks,Hkv,bs,3D/32], norms fp32 [num_blocks,Hkv,bs,D/128],
    codebook fp32 [8]) read inside one paged split-KV launch; D 128 or 256.
    Returns fp16 [B,Hq,1,D]."""
    from .quant import LOG2E
    from .quant.rotation import rotate_last

    if q.shape[-2] != 1:
        raise AssertionError(f"paged decode expects M=1, got M={q.shape[-2]}")
    if max_context_len is None:
        max_context_len = int(context_lens.max().item())
    softmax_scale = (1.0 / (q.shape[-1] ** 0.5)) if scale is None else scale
    q = q.contiguous()
    if num_splits is None and _C.q16_ok(q):
        out = _C.attn_paged_decode_k8v3_q16(q, softmax_scale * LOG2E, rotate, k_cache.contiguous(),
                                            k_scale.contiguous(), v_packed.contiguous(),
                                            v_norm.contiguous(), v_codebook.contiguous(),
                                            block_table.contiguous(), context_lens.contiguous(),
                                            int(block_size), int(max_context_len))
        if out is not None:
            return out
    if rotate:
        q = rotate_last(q)
    q_shape = q.shape
    q_i8, q_scale = quantize_i8_rowwise(q.reshape(-1, q_shape[-1]).contiguous())
    q_i8 = q_i8.reshape(q_shape)
    q_scale = (q_scale.float() * (softmax_scale * LOG2E)).reshape(q_shape[0], q_shape[1], 1).contiguous()
    ns = -1 if num_splits is None else int(num_splits)
    return _C.attn_paged_decode_k8v3(q_i8.contiguous(), q_scale, k_cache.contiguous(),
                                     k_scale.contiguous(), v_packed.contiguous(),
                                     v_norm.contiguous(), v_codebook.contiguous(),
                                     block_table.contiguous(), context_lens.contiguous(),
                                     int(block_size), int(max_context_len), ns)


def quantize_kv_write_paged_k8v3(k_new: torch.Tensor, v_new: torch.Tensor,
                                 k_cache: torch.Tensor, k_scale: torch.Tensor,
                                 v_packed: torch.Tensor, v_norm: torch.Tensor,
                                 slot_mapping: torch.Tensor, *, rotate: bool = True,
                                 codebook: torch.Tensor | None = None) -> torch.Tensor:
    """Write one new token per (batch, KV head) into a paged K8V3 store, in place:
    K rotated (when `rotate`) and quantised per row to int8; V quantised to 3-bit
    Lloyd-Max codes over 128-channel blocks (`codebook`, default the fixed
    Gaussian one) and packed. k_new, v_new fp16 [B,Hkv,D]; slot_mapping int32 [B]
    (flat slot = block * block_size + offset). Returns the codebook used, the
    `v_codebook` argument of attn_paged_decode_k8v3. (The reference store is
    written the same way by its serving code, reference
    tests/test_k8v3_paged_decode.py:32-83.)"""
    from .quant.lloydmax import pack_indices_lowbit, quantize_lloydmax
    from .quant.rotation import rotate_last

    B, Hkv, D = k_new.shape
    bs = k_cache.shape[2]
    if rotate:
        k_new = rotate_last(k_new)
    k_i8, k_sc = quantize_i8_rowwise(k_new.reshape(-1, D).contiguous())
    codes, norms, cb = quantize_lloydmax(v_new, bits=3, block_size=128, codebook=codebook)
    packed = pack_indices_lowbit(codes, 3)
    slots = slot_mapping.long()
    rows = ((slots // bs)[:, None] * Hkv + torch.arange(Hkv, device=slots.device)) * bs + \
        (slots % bs)[:, None]
    rows = rows.reshape(-1)
    k_cache.view(-1, D)[rows] = k_i8
    k_scale.view(-1)[rows] = k_sc
    v_packed.view(-1, v_packed.shape[-1])[rows] = packed.reshape(-1, packed.shape[-1])
    v_norm.view(-1, v_norm.shape[-1])[rows] = norms.reshape(-1, norms.shape[-1])
    return cb


def rope_table(max_positions: int, rotary_dim: int, *, base: float = 10000.0, sections=None,
               device="cuda") -> torch.Tensor:
    """The table of `rope`: fp32 [max_positions, rotary_dim], cos of the rotary_dim / 2 pairs, then
    sin, of position * base^(-pair / pairs), from 64 bits. With sections (pairs per axis) the
    frequencies start again at each axis, as positions in images have it; leave them out for one
    axis and for axes that share one row of frequencies (video)."""
    if rotary_dim < 2 or rotary_dim % 2 or max_positions < 1:
        raise ValueError(f"rope_table needs an even rotary dim and at least one position, got "
                         f"{rotary_dim} and {max_positions}")
    half = rotary_dim // 2
    if sections is not None and (min(sections, default=0) < 1 or sum(sections) != half):
        raise ValueError(f"sections must be positive and add up to {half}, got {list(sections)}")
    f = torch.cat([torch.arange(n, dtype=torch.float64) / n for n in (sections or (half,))])
    pos = torch.arange(max_positions, dtype=torch.float64, device=device)
    angle = pos[:, None] * (float(base) ** -f).to(pos.device)
    return torch.cat([angle.cos(), angle.sin()], 1).float()


class _Rope(torch.autograd.Function):
    """`rope` where a gradient is wanted: that of q and k is the turn back of that of q' and k'."""

    @staticmethod
    def forward(ctx, q, k, positions, table, sections, interleaved, inverse):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions, table)
        ctx.how = dict(sections=sections, interleaved=interleaved, inverse=not inverse)
        return _C.rope(q, k, positions, table, sections, interleaved, inverse)

    @staticmethod
    def backward(ctx, dq, dk):
        if torch.cuda.is_current_stream_capturing():
            # (a leaf's node of an eager graph that lives waits on its own stream, which is none of
            # the capture: that ends the process)
            raise RuntimeError("fni8 rope: its backward cannot be captured; capture "
                               "rope(dq, dk, ..., inverse=True) under no_grad instead")
        dq, dk = (d if need else None for d, need in zip((dq, dk), ctx.needs_input_grad))
        if dq is not None:
            dq, dk = rope(dq, dk, *ctx.saved_tensors, **ctx.how)
        elif dk is not None:
            dk, _ = rope(dk, None, *ctx.saved_tensors, **ctx.how)
        return dq, dk, None, None, None, None, None


def rope(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, table: torch.Tensor, *,
         sections=None, interleaved: bool = False, inverse: bool = False):
    """Rotary positions of q [B,Hq,S,D] and k [B,Hkv,S,D] (or None) in one launch, fp16/bf16/fp32:
    contiguous (q', k'), ready for attn_int8_fwd. Views of a fused projection are read in place.

    Pair p of the first R elements turns by the angle of table[position, p] (fp32 [P, R]: cos, then
    sin; see rope_table); (p, p + R/2) is a pair, or (2p, 2p+1) with `interleaved`. positions
    int32/int64 [S] or [B,S]; with `sections` (up to 4 counts of consecutive pairs, in order)
    [A,S] or [A,B,S], an axis for each. Positions outside the table count as its nearest end.
    `inverse` turns back, which is the gradient of q and k from that of q' and k': autograd records
    it for q and k that require one (not for the table), except that the backward cannot be captured
    into a graph: there call rope(dq, dk, ..., inverse=True)."""
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return _Rope.apply(q, k, positions, table, None if sections is None else tuple(sections),
                           interleaved, inverse)
    return _C.rope(q, k, positions, table, sections, interleaved, inverse)


def quantize_kv_append_block8(k_new: torch.Tensor, v_new: torch.Tensor, k_cache: torch.Tensor,
                              k_scale: torch.Tensor, v_cache: torch.Tensor, v_scale: torch.Tensor,
                              block_table: torch.Tensor, context_lens: torch.Tensor, *,
                              cu_lens: torch.Tensor | None = None, q: torch.Tensor | None = None,
                              positions: torch.Tensor | None = None,
                              table: torch.Tensor | None = None, sections=None,
                              interleaved: bool = False,
                              rotate: bool = True) -> torch.Tensor | None:
    """Append a step's new tokens to a paged int8 cache with one scale per block and head, in place,
    K (and q) turned by position on the way; returns the turned q [T,Hq,D] (None without q).

    k_new, v_new [T,Hkv,D] and q [T,Hq,D] fp16/bf16 (views of a fused projection are read in place);
    k_cache, v_cache int8 [num_blocks,Hkv,block_size,D] (D 64/128/256, block_size a multiple of 16,
    16..128); k_scale, v_scale fp32 [num_blocks,Hkv]. cu_lens int32 [B+1]: sequence b's new tokens
    are rows cu_lens[b]..cu_lens[b+1]-1 (None: one each); context_lens int32 [B]: its length with
    them; block_table int32 [B,max_blocks]. positions int32/int64 [T] (with `sections` [A,T]) and
    table as in `rope` (rotary dim a multiple of 16); without them K is taken as turned already.
    `rotate` as in quantize_kv_write_paged. A block that new tokens enter is requantised where its
    scale grows; sequences of one call must not write into the same block. Values must be finite."""
    if rotate:
        hadamard_dim(k_new.shape[-1])
    return _C.kv_append_block8(k_new, v_new, k_cache, k_scale, v_cache, v_scale,
                               block_table.contiguous(), context_lens.contiguous(),
                               None if cu_lens is None else cu_lens.contiguous(), q, positions,
                               table, sections, interleaved, rotate)


def attn_paged_block8(q: torch.Tensor, k_cache: torch.Tensor, k_scale: torch.Tensor,
                      v_cache: torch.Tensor, v_scale: torch.Tensor, block_table: torch.Tensor,
                      context_lens: torch.Tensor, *, cu_lens: torch.Tensor | None = None,
                      scale: float | None = None, rotate: bool = True,
                      window_left: int = -1, tree_mask: torch.Tensor | None = None,
                      return_lse: bool = False):
    """Attention over a paged int8 cache with one scale per block and head, written by
    quantize_kv_append_block8 (the same `rotate`): one to thousands of new tokens per sequence,
    mixed in one call, nothing read on the host.

    q [T,Hq,D] fp16/bf16 -> [T,Hq,D] of its dtype: sequence b's rows are cu_lens[b]..cu_lens[b+1]-1
    (None: row b), the last of its context_lens[b] tokens, which the cache holds already. Each sees
    the keys up to itself and, with window_left >= 0, only the last window_left of them; a row
    that sees none and rows of no sequence (a padded batch, offsets of a part of one) are zeros.

    tree_mask int64 [T] or [T,1..4] (see tree_mask): drafted tokens in a tree. A row sees its
    sequence's tokens in front of the new ones, and of those the j-th where bit j of its mask is set
    (bits stand for the first 64 to 256; itself too only if marked; bits of tokens that are not there
    count for nothing); a window counts the marked ones first and takes what is left of it in front.
    return_lse: (out, lse fp32 [T,Hq]), the logarithm of each row's sum of e^score, -inf where it sees
    nothing. With either, rows are rotated in 64 bits, as attn_weights_block8 does: a code next to a
    half may then be the next one to that of a call with neither."""
    softmax_scale = (1.0 / (q.shape[-1] ** 0.5)) if scale is None else scale
    q = q.contiguous()
    if q.data_ptr() % 16:
        q = q.clone()
    return _C.attn_paged_block8(q, softmax_scale * LOG2E, rotate, k_cache, k_scale, v_cache, v_scale,
                                block_table.contiguous(), context_lens.contiguous(),
                                None if cu_lens is None else cu_lens.contiguous(), window_left,
                                tree_mask, return_lse)


def tree_mask(parents: torch.Tensor, cu_lens: torch.Tensor | None = None, *, words: int = 1) -> torch.Tensor:
    """The masks of drafted tokens from their parents, for attn_paged_block8: int64 [T, words] with the
    bits of a token and of all above it. parents int32/int64 [T]: the parent's place among its
    sequence's new tokens (in front of or behind it), -1 for those that follow the context; cu_lens as
    there (None: one sequence of all rows). Tokens past a sequence's 64 * words-th have no bits."""
    if parents.dim() != 1 or parents.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"tree_mask needs parents int32 or int64 [T], got {parents.dtype} {list(parents.shape)}")
    if not 1 <= words <= _C._TREE_MAX_WORDS:
        raise ValueError(f"words must be 1..{_C._TREE_MAX_WORDS}, got {words}")
    T = parents.shape[0]
    t = torch.arange(T, device=parents.device)
    first, end = torch.zeros_like(t), torch.full_like(t, T)
    if cu_lens is not None:
        cu = cu_lens.long().contiguous()
        b = (torch.searchsorted(cu, t, right=True) - 1).clamp(0, max(cu.shape[0] - 2, 0))
        first, end = cu[b], cu[(b + 1).clamp(max=cu.shape[0] - 1)]
    place = t - first
    bit = torch.where((place >= 0) & (place < 64 * words), torch.ones_like(t) << (place % 64), 0)
    mask = torch.where(place[:, None] // 64 == torch.arange(words, device=t.device), bit[:, None], 0)
    up = torch.where(parents >= 0, first + parents.long(), T)
    # (a row T behind the others: no token, no bits, its own parent)
    up = torch.cat([torch.where((up >= first) & (up < end), up, T), up.new_full((1,), T)])
    mask = torch.cat([mask, mask.new_zeros(1, words)])
    # the masks of twice as many levels, each time; a path may be as long as the list, whatever has bits
    for _ in range(max(T - 1, 1).bit_length()):
        mask = mask | mask[up]
        up = up[up]
    return mask[:T]


def attn_weights_block8(q: torch.Tensor, lse: torch.Tensor, k_cache: torch.Tensor, k_scale: torch.Tensor,
                        block_table: torch.Tensor, context_lens: torch.Tensor, weights: torch.Tensor, *,
                        cu_lens: torch.Tensor | None = None, scale: float | None = None,
                        rotate: bool = True, window_left: int = -1, decay: float = 1.0) -> None:
    """Add up by cached key what softmax weights a step's rows gave it, in place: what kv_evict_block8
    decides by. weights fp32 [B,Hkv,tokens] (a table's max_blocks * block_size at least; dense rows) of
    sequence b, KV head h and token j becomes decay * weights plus the sum over its new rows, and over
    the heads of the group, of e^(score - lse); a new token's own starts from 0, so reused rows need no
    clearing, and entries behind the context are left alone.

    q [T,Hq,D], k_cache, k_scale, block_table, context_lens, cu_lens, scale, rotate and window_left as in
    attn_paged_block8, whose lse [T,Hq] (return_lse) this takes; rows are causal (drafted trees: the
    accepted rows with their lse, once they are appended). Rows of lse -inf add nothing."""
    softmax_scale = (1.0 / (q.shape[-1] ** 0.5)) if scale is None else scale
    q = q.contiguous()
    if q.data_ptr() % 16:
        q = q.clone()
    _C.attn_weights_block8(q, softmax_scale * LOG2E, rotate, lse.contiguous(), k_cache, k_scale,
                           block_table.contiguous(), context_lens.contiguous(), weights,
                           None if cu_lens is None else cu_lens.contiguous(), window_left, decay)


def kv_evict_block8(k_cache: torch.Tensor, k_scale: torch.Tensor, v_cache: torch.Tensor,
                    v_scale: torch.Tensor, block_table: torch.Tensor, context_lens: torch.Tensor,
                    weights: torch.Tensor, new_table: torch.Tensor, *, budget: int, sinks: int = 0,
                    recent: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """Cut sequences of a block-scaled paged cache down to `budget` tokens a KV head: the first
    `sinks`, the last `recent` and, between them, those of the largest weights (attn_weights_block8;
    ties to the lowest index, no NaN); heads keep different ones. Shorter sequences keep all.

    The kept tokens move in order into the blocks of new_table int32 [B,blocks], which no row of
    block_table in the call and no two of new_table may hold: from then on that is the sequence's table
    (the old blocks are only read: shared prefixes stay whole). A block takes the largest scale of those its rows come
    from; rows of others are rounded again, rows of the same are copied. weights [B,Hkv,tokens] of the
    kept tokens move to the front, in place. Returns (lengths int32 [B], kept int32 [B,Hkv,budget]: the
    tokens' old places, -1 behind the last). Nothing is read on the host."""
    return _C.kv_evict_block8(k_cache, k_scale, v_cache, v_scale, block_table.contiguous(),
                              context_lens.contiguous(), weights, new_table.contiguous(), budget, sinks,
                              recent)


def quantize_kv_cache_3bit(k: torch.Tensor, v: torch.Tensor, *, rotate: bool = True,
                           fit: bool = True, block_size: int = 128) -> dict:
    """3-bit Lloyd-Max storage codec of a whole K/V cache (reference ops.py:590-655):
    K smoothed (+ rotated), both packed with a codebook fitted to the
    unit-normalised blocks (`fit`) or the fixed Gaussian one."""
    from .quant import smooth_k
    from .quant.lloydmax import (lloyd_max_fit, lloydmax_bits_levels, pack_indices_lowbit,
                                 quantize_lloydmax)
    from .quant.rotation import rotate_last

    k_s, k_mean = smooth_k(k)
    if rotate:
        k_s = rotate_last(k_s)

    def enc(x):
        cb = None
        if fit:
            xb = x.float().reshape(*x.shape[:-1], x.shape[-1] // block_size, block_size)
            norm = torch.sqrt((xb * xb).sum(-1, keepdim=True))
            cb = lloyd_max_fit(xb / torch.where(norm == 0, torch.ones_like(norm), norm),
                               lloydmax_bits_levels(3))
        codes, norm, codebook = quantize_lloydmax(x, bits=3, block_size=block_size, codebook=cb)
        return pack_indices_lowbit(codes, 3).contiguous(), norm.contiguous(), codebook

    k_packed, k_norm, k_cb = enc(k_s)
    v_packed, v_norm, v_cb = enc(v)
    return {"k_packed": k_packed, "k_norm": k_norm, "k_codebook": k_cb, "v_packed": v_packed,
            "v_norm": v_norm, "v_codebook": v_cb, "k_mean": k_mean, "rotate": rotate,
            "block_size": block_size, "bits": 3}


def dequantize_kv_cache_3bit(packed: dict, d: int):
    """Inverse of quantize_kv_cache_3bit -> (k, v) fp16, K still smoothed and
    rotated (reference ops.py:658-668)."""
    from .quant.lloydmax import dequantize_lloydmax, unpack_indices_lowbit

    bs = packed["block_size"]
    k = dequantize_lloydmax(unpack_indices_lowbit(packed["k_packed"], 3, d), packed["k_norm"],
                            packed["k_codebook"], block_size=bs)
    v = dequantize_lloydmax(unpack_indices_lowbit(packed["v_packed"], 3, d), packed["v_norm"],
                            packed["v_codebook"], block_size=bs)
    return k.half(), v.half()


def quantize_i8_rowwise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Fused per-row symmetric int8: x[M,K] -> (q int8 [M,K], scale fp32 [M])."""
    return _C.quantize_i8_rowwise(x)


def linear_q4k(x: torch.Tensor, w_bytes: torch.Tensor, *, bias: torch.Tensor | None = None,
               out_dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """GGUF Q4_K linear on native 144-byte super-blocks: x [..., K] -> [..., N]."""
    return _linear_kquant(x, w_bytes, bias, out_dtype, _C.gemm_q4k,
                          getattr(_C, "gemm_decode_q4k", None), 4)


def linear_q5k(x: torch.Tensor, w_bytes: torch.Tensor, *, bias: torch.Tensor | None = None,
               out_dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """GGUF Q5_K linear on native 176-byte super-blocks (reference ops.py:1328-1336)."""
    return _linear_kquant(x, w_bytes, bias, out_dtype, _C.gemm_q5k,
                          getattr(_C, "gemm_decode_q5k", None), 5)


def linear_q6k(x: torch.Tensor, w_bytes: torch.Tensor, *, bias: torch.Tensor | None = None,
               out_dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """GGUF Q6_K linear on native 210-byte super-blocks (reference ops.py:1339-1347)."""
    return _linear_kquant(x, w_bytes, bias, out_dtype, _C.gemm_q6k,
                          getattr(_C, "gemm_decode_q6k", None))


def linear_w8a8(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, *,
                bias: torch.Tensor | None = None,
                out_dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """Linear layer of int8 weights: x [..., K] fp16/bf16/fp32, each row quantised as by
    quantize_i8_rowwise; w int8 [N,K] with w_scale fp32 [N] (a scale per output channel: the
    per_row_i8 QTensor) -> [..., N] of out_dtype. K a multiple of 4, at least 16. The integer sums are
    exact; scales and bias are applied in fp32 and the result is rounded once. A row of x that holds
    NaN or infinity gives no finite output; the other rows are as without it."""
    if x.dim() == 2:
        return _C.linear_w8a8(x.contiguous(), w.contiguous(), w_scale.contiguous(), bias, out_dtype)
    *lead, K = x.shape
    y = _C.linear_w8a8(x.reshape(-1, K).contiguous(), w.contiguous(), w_scale.contiguous(), bias, out_dtype)
    return y.reshape(*lead, y.shape[-1])


_FUSED_KQUANT_OPS = {"q4_k": linear_q4k, "q5_k": linear_q5k, "q6_k": linear_q6k}


def linear(x: torch.Tensor, qt, *, bias: torch.Tensor | None = None,
           out_dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """Scheme-dispatched linear over a ``superl8_amd.format.QTensor`` (reference
    ops.py:2088-2150, the ``gguf_kquant`` arm): native Q4_K / Q5_K / Q6_K bytes run
    on the fused kernels, ``per_row_i8`` weights that are not rotated on linear_w8a8; any other
    scheme or type tag raises ValueError."""
    if qt.scheme == "gguf_kquant":
        op = _FUSED_KQUANT_OPS.get(qt.codebook)
        if op is not None:
            return op(x, qt.data, bias=bias, out_dtype=out_dtype)
        raise ValueError(f"superl8.linear: gguf_kquant type {qt.codebook!r} has no fused kernel")
    if qt.scheme == "per_row_i8":
        if qt.rotated:
            raise ValueError("superl8.linear: rotated per_row_i8 weights have no product here")
        return linear_w8a8(x, qt.data, qt.scale, bias=bias, out_dtype=out_dtype)
    raise ValueError(f"superl8.linear: unsupported weight scheme {qt.scheme!r}")


def _linear_kquant(x, w_bytes, bias, out_dtype, tile_op, decode_op, fmt=None):
    *lead, K = x.shape
    x2 = x.reshape(-1, K).contiguous()
    w_bytes = w_bytes.contiguous()
    M = x2.shape[0]
    if M > _KQUANT_DECODE_MAX_M and fmt is not None and _C.linear_kq_ok(x2):  # one call
        y = _C.linear_kq(fmt, x2, w_bytes, out_dtype)
    else:
        x_i8, x_scale = quantize_i8_rowwise(x2)
        if decode_op is not None and x2.is_cuda and 0 < M <= _KQUANT_DECODE_MAX_M:
            y = decode_op(x_i8, x_scale, w_bytes, out_dtype)
        else:
            y = tile_op(x_i8, x_scale, w_bytes, out_dtype)
    if bias is not None:
        if bias.dim() and bias.dtype in (torch.float16, torch.bfloat16, torch.float32):
            y = (y + bias).to(y.dtype)  # added in fp32 and rounded once, whatever the two types
        else:
            y = (y.float() + bias.float()).to(y.dtype)
    return y.reshape(*lead, y.shape[-1])
