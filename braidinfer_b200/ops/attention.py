"""Paged cascade attention over chunk lists, and the fused QKV epilogue.

KV layout (per layer): ``[P, 2, Hkv, page, D]`` — the reference's HND pool
(``braidinfer/engine/page_manager.py:39-42``) with one K and one V slab per
(page, head).  A flat *slot* is ``page * page_size + offset``.

Attention metadata describes, for every sequence of a batch, an ordered list
of KV *segments*: cached chunks (system, contexts, retained outputs) followed
by the sequence's private pages.  Segment ``s`` holds ``seg_len[s]`` keys that
start at slot ``seg_offset[s]`` of its first page (pages listed in
``page_ids[seg_page_indptr[s]:seg_page_indptr[s+1]]``), whose first key sits at
global position ``seg_pos0[s]`` in the current composition and was rotated
when cached at ``seg_pos0[s] - seg_delta[s]``.

Masking rule: key ``j`` of segment ``s`` is visible to a query at position
``p`` iff ``seg_pos0[s] + j <= p``.  This gives causal attention inside the
private segment and inside a chunk's own prefill, and full visibility of every
earlier chunk — the cascade of ``braidinfer/layers/cascade_attention.py:50-231``
without its per-page Python loop.

With ``window`` W > 0 it must also hold that ``p - (seg_pos0[s] + j) < W`` or
``seg_pos0[s] + j < sinks``: the last W positions (the query's own among them)
and the first ``sinks`` positions of the composition.  A query that sees no key
gets zeros.  Slots that no query of a sequence sees may hold anything, NaN
included.  On CUDA, with a window or a 4-bit cache, a NaN in a query or in a key
that it sees makes its row NaN; one in a V row of a bf16 cache, or with many
queries of either, may also reach those queries of the sequence that do not see
it (weight 0 times NaN).

The cache may also be a 4-bit one (``kv4.KV4Layer``): same pages, slots and plan.

Queries are stored *unrotated*; the kernel rotates them by ``p - seg_delta[s]``
per segment (differential RoPE on the query side, O(|Q|) per chunk instead of
re-rotating O(|K|) cached keys).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Union

import torch

from ._ext import ext
from .kv4 import KV4Layer, kv4_pack_ref, kv4_unpack_ref
from .norm import rms_norm_ref
from .rope import apply_rope_ref


@dataclass
class AttnMeta:
    """Per-forward attention plan (device tensors, int32)."""

    qo_indptr: torch.Tensor       # [B+1]
    positions: torch.Tensor       # [T]
    seg_indptr: torch.Tensor      # [B+1]
    seg_page_indptr: torch.Tensor  # [S+1]
    seg_offset: torch.Tensor      # [S]
    seg_len: torch.Tensor         # [S]
    seg_pos0: torch.Tensor        # [S]
    seg_delta: torch.Tensor       # [S]
    page_ids: torch.Tensor        # [NP]
    num_seqs: int
    max_q_len: int
    max_kv_len: int
    decode: bool = False          # every sequence has exactly one query token
    num_splits: int = 1           # split-KV factor of the decode kernel
    # host copies (CPU reference path and planning)
    host: Optional[dict] = None
    # shared-prefix decode: the group's tokens [grp_qo_indptr[0], grp_qo_indptr[1])
    # attend once to segments [grp_seg_indptr[0], grp_seg_indptr[1]) (split into
    # shared_splits key ranges); seq_nsh flags the member sequences, whose own
    # segment lists leave those segments out
    grp_qo_indptr: Optional[torch.Tensor] = None
    grp_seg_indptr: Optional[torch.Tensor] = None
    seq_nsh: Optional[torch.Tensor] = None
    shared_splits: int = 0
    grp_max_q: int = 0


def qkv_prepare(qkv: torch.Tensor, positions: torch.Tensor, slot_mapping: torch.Tensor,
                kv_layer: Union[torch.Tensor, KV4Layer], num_q_heads: int, num_kv_heads: int, head_dim: int,
                cos: torch.Tensor, sin: torch.Tensor, q_norm: Optional[torch.Tensor] = None,
                k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6, use_rope: bool = True) -> torch.Tensor:
    """Split ``qkv[T, (Hq+2Hkv)*D]``; per-head q/k RMSNorm (Qwen3); RoPE on k;
    append k/v to the paged cache at ``slot_mapping``; return unrotated q ``[T, Hq, D]``.

    Replaces the reference's per-token ``.item()`` append loop
    (``braidinfer/kernels/kv_cache_utils.py:9-78``) with one kernel.

    Into a :class:`KV4Layer` the norm, RoPE and codes are computed in fp32 from
    the bf16 input (no rounding in between), and without a ``q_norm`` the
    returned q is a view of ``qkv``.  The slots of one call must differ, unless
    what they hold is never read (padding); on CUDA a slot outside the cache is
    skipped.
    """
    T = qkv.shape[0]
    if isinstance(kv_layer, KV4Layer):
        return _qkv_prepare_kv4(qkv, positions, slot_mapping, kv_layer, num_q_heads, num_kv_heads, head_dim, cos, sin,
                                q_norm, k_norm, eps, use_rope)
    if qkv.is_cuda:
        q = torch.empty(T, num_q_heads, head_dim, dtype=qkv.dtype, device=qkv.device)
        ext().qkv_prepare(q, qkv, positions, slot_mapping, kv_layer, q_norm, k_norm, float(eps), cos, sin,
                          num_q_heads, num_kv_heads, head_dim, bool(use_rope))
        return q
    qs, ks = num_q_heads * head_dim, num_kv_heads * head_dim
    q = qkv[:, :qs].reshape(T, num_q_heads, head_dim)
    k = qkv[:, qs:qs + ks].reshape(T, num_kv_heads, head_dim)
    v = qkv[:, qs + ks:qs + 2 * ks].reshape(T, num_kv_heads, head_dim)
    if q_norm is not None:
        q = rms_norm_ref(q, q_norm, eps)
        k = rms_norm_ref(k, k_norm, eps)
    if use_rope:
        k = apply_rope_ref(k, positions, cos, sin).to(qkv.dtype)
    P, _, Hkv, page, D = kv_layer.shape
    slots = slot_mapping.long()
    pg, off = slots // page, slots % page
    kv_layer[pg, 0, :, off, :] = k.to(kv_layer.dtype)
    kv_layer[pg, 1, :, off, :] = v.to(kv_layer.dtype)
    return q.contiguous()


def _qkv_prepare_kv4(qkv, positions, slot_mapping, kv_layer, num_q_heads, num_kv_heads, head_dim, cos, sin, q_norm,
                     k_norm, eps, use_rope):
    codes, scales = kv_layer
    if qkv.is_cuda:
        return ext().qkv_prepare_kv4(qkv, positions, slot_mapping, codes, scales, q_norm, k_norm, float(eps), cos, sin,
                                     num_q_heads, num_kv_heads, head_dim, bool(use_rope))
    qs = num_q_heads * head_dim
    view = qkv[:, :qs].unflatten(1, (num_q_heads, head_dim))

    def norm(x, w):
        return x if w is None else x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w.float()

    kv = qkv[:, qs:].float().unflatten(1, (2, num_kv_heads, head_dim))
    k = norm(kv[:, 0], k_norm)
    if use_rope:
        k = apply_rope_ref(k, positions, cos, sin)
    c, sc = kv4_pack_ref(torch.stack([k, kv[:, 1]], 1))
    slots, ps = slot_mapping.long(), kv_layer.page_size
    codes[slots // ps, :, :, slots % ps] = c
    scales[slots // ps, :, :, slots % ps] = sc
    return view if q_norm is None else norm(view.float(), q_norm).to(qkv.dtype)


def qkv_gemm(x: torch.Tensor, w_qkv: torch.Tensor, bias: Optional[torch.Tensor], rms_eps: Optional[float],
             positions: torch.Tensor, slot_mapping: torch.Tensor, kv_layer: Union[torch.Tensor, KV4Layer], num_q_heads: int,
             num_kv_heads: int, head_dim: int, cos: torch.Tensor, sin: torch.Tensor,
             q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6,
             use_rope: bool = True, rs_vec: Optional[torch.Tensor] = None,
             sp: Optional[torch.Tensor] = None) -> torch.Tensor:
    """QKV projection (fused input RMSNorm when ``rms_eps`` is set, norm weight
    folded into ``w_qkv``) with the q/k-norm, RoPE(k) and paged KV append done
    in the GEMM epilogue on CUDA.  Returns unrotated q ``[T, Hq, D]``.
    ``rs_vec``/``sp``: precomputed ``1/rms`` and sequence-parallel parameters
    (CUDA tensor-parallel prefill).  Into a :class:`KV4Layer` the projection and
    ``qkv_prepare`` are two launches; ``rs_vec``/``sp`` are refused there."""
    T = x.shape[0]
    if isinstance(kv_layer, KV4Layer):
        if rs_vec is not None or sp is not None:
            raise ValueError("qkv_gemm: a 4-bit cache takes no precomputed 1/rms and no sequence-parallel parameters")
        from .linear import linear

        return qkv_prepare(linear(x, w_qkv, bias, rms_eps=rms_eps), positions, slot_mapping, kv_layer, num_q_heads,
                           num_kv_heads, head_dim, cos, sin, q_norm, k_norm, eps, use_rope)
    if x.is_cuda:
        q = torch.empty(T, num_q_heads, head_dim, dtype=x.dtype, device=x.device)
        ext().gemm_qkv(q, x, w_qkv, bias, -1.0 if rms_eps is None else float(rms_eps), positions, slot_mapping,
                       kv_layer, q_norm, k_norm, float(eps), cos, sin, num_q_heads, num_kv_heads, head_dim,
                       bool(use_rope), rs_vec, sp)
        return q
    from .linear import linear

    qkv = linear(x, w_qkv, bias, rms_eps=rms_eps)
    return qkv_prepare(qkv, positions, slot_mapping, kv_layer, num_q_heads, num_kv_heads, head_dim, cos, sin,
                       q_norm, k_norm, eps, use_rope)


def attention_ref(q: torch.Tensor, kv_layer: Union[torch.Tensor, KV4Layer], meta: AttnMeta, cos: torch.Tensor,
                  sin: torch.Tensor, scale: float, use_rope: bool = True, window: int = 0,
                  sinks: int = 0) -> torch.Tensor:
    """fp32 restatement of the cascade kernels (one softmax over all segments)."""
    h = meta.host
    T, Hq, D = q.shape
    q4 = isinstance(kv_layer, KV4Layer)
    _, _, Hkv, page, _ = kv_layer.codes.shape if q4 else kv_layer.shape
    G = Hq // Hkv
    out = torch.zeros(T, Hq, D, dtype=torch.float32)
    qo, segp = h["qo_indptr"], h["seg_indptr"]
    for b in range(meta.num_seqs):
        t0, t1 = int(qo[b]), int(qo[b + 1])
        if t1 == t0:
            continue
        pos = h["positions"][t0:t1].long()
        scores, values = [], []
        segs = list(range(int(segp[b]), int(segp[b + 1])))
        if meta.seq_nsh is not None and int(h["seq_nsh"][b]):
            # a shared-prefix group member: its shared segments are listed once for the group
            segs = list(range(int(h["grp_seg_indptr"][0]), int(h["grp_seg_indptr"][1]))) + segs
        for s in segs:
            n = int(h["seg_len"][s])
            if n == 0:
                continue
            p0, p1 = int(h["seg_page_indptr"][s]), int(h["seg_page_indptr"][s + 1])
            pages = h["page_ids"][p0:p1].long()
            slot = int(h["seg_offset"][s]) + torch.arange(n)
            pg = pages[slot // page]
            off = slot % page
            if q4:
                kv = kv4_unpack_ref(kv_layer.codes[pg, :, :, off], kv_layer.scales[pg, :, :, off])
                k, v = kv[:, 0], kv[:, 1]
            else:
                k = kv_layer[pg, 0, :, off, :].float()  # [n, Hkv, D]
                v = kv_layer[pg, 1, :, off, :].float()
            qq = q[t0:t1].float()
            if use_rope:
                qq = apply_rope_ref(qq, pos - int(h["seg_delta"][s]), cos, sin)
            kk = k.repeat_interleave(G, dim=1)  # [n, Hq, D]
            sc = torch.einsum("thd,nhd->htn", qq, kk) * scale
            kpos = int(h["seg_pos0"][s]) + torch.arange(n)
            mask = kpos[None, :] > pos[:, None]  # [t, n]
            if window > 0:
                mask = mask | ((pos[:, None] - kpos[None, :] >= window) & (kpos[None, :] >= sinks))
            sc = sc.masked_fill(mask[None], float("-inf"))
            scores.append(sc)
            values.append(v.repeat_interleave(G, dim=1))
        if not scores:
            continue
        sc = torch.cat(scores, dim=-1)
        vv = torch.cat(values, dim=0)
        p = torch.softmax(sc, dim=-1)
        p = torch.nan_to_num(p, nan=0.0)
        out[t0:t1] = torch.einsum("htn,nhd->thd", p, vv)
    return out.to(q.dtype).reshape(T, Hq * D)


def attention(q: torch.Tensor, kv_layer: Union[torch.Tensor, KV4Layer], meta: AttnMeta, cos: torch.Tensor,
              sin: torch.Tensor, scale: float, use_rope: bool = True, workspace: Optional[dict] = None,
              window: int = 0, sinks: int = 0) -> torch.Tensor:
    """Attention of ``q [T, Hq, D]`` over the plan's segments -> ``[T, Hq * D]``
    (the masking rule, ``window`` and ``sinks``: module text; ``window`` 0 is no
    window, and ``sinks`` without one changes nothing).

    A :class:`KV4Layer` or a window takes its own kernels
    (``csrc/attention_rows.cu``): decode or not follows from the rows,
    ``meta.num_splits`` is not used, and a plan with a shared-prefix group is
    refused.  Calls of few rows a sequence split keys inside the kernel without a
    workspace.  With many rows a sequence and head_dim 128 the call may allocate
    partial results and, of a 4-bit cache, the plan's pages as bf16 (at most
    ``ext().attn_kv4_workspace_limit()`` bytes; a plan that would need more takes
    the kernel without); queries and such pages are then rounded to bf16."""
    window, sinks = int(window), int(sinks)
    if window < 0 or sinks < 0 or window >= 1 << 30 or sinks >= 1 << 30:
        raise ValueError(f"attention: window and sinks must be in [0, 2**30), got {window} and {sinks}")
    q4 = isinstance(kv_layer, KV4Layer)
    if (q4 or window > 0) and meta.seq_nsh is not None:
        raise ValueError("attention: a shared-prefix plan takes neither a 4-bit cache nor a window")
    if q.is_cuda:
        if q4 or window > 0:
            kv, scales = kv_layer if q4 else (kv_layer, None)
            return ext().attention_rows(None, q, kv, scales, meta.qo_indptr, meta.positions, meta.seg_indptr,
                                        meta.seg_page_indptr, meta.seg_offset, meta.seg_len, meta.seg_pos0,
                                        meta.seg_delta, meta.page_ids, cos, sin, float(scale), bool(use_rope),
                                        int(meta.num_seqs), int(meta.max_q_len), int(meta.max_kv_len), window, sinks)
        T, Hq, D = q.shape
        out = torch.empty(T, Hq * D, dtype=q.dtype, device=q.device)
        ws = workspace or {}
        ext().attention(out, q, kv_layer, meta.qo_indptr, meta.positions, meta.seg_indptr,
                        meta.seg_page_indptr, meta.seg_offset, meta.seg_len, meta.seg_pos0, meta.seg_delta,
                        meta.page_ids, cos, sin, float(scale), bool(use_rope), int(meta.num_seqs),
                        int(meta.max_q_len), int(meta.max_kv_len), bool(meta.decode), int(meta.num_splits),
                        ws.get("partial_o"), ws.get("partial_lse"), meta.grp_qo_indptr, meta.grp_seg_indptr,
                        meta.seq_nsh, int(meta.shared_splits), int(meta.grp_max_q))
        return out
    return attention_ref(q, kv_layer, meta, cos, sin, scale, use_rope, window, sinks)
