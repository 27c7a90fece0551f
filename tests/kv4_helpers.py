"""Plans, 64-bit definitions and error bounds for the 4-bit cache and windowed attention tests."""
import math

import torch

from braidinfer_b200 import ops


def make_plan(seqs, ps, pages, device, seed=0, qpos_shift=0):
    """seqs: [(queries, [(keys, offset, delta)])] -> (meta, tokens).  The queries are the last positions of their
    sequence, moved by ``qpos_shift``; pages are handed out in random order."""
    g = torch.Generator().manual_seed(seed)
    free = torch.randperm(pages, generator=g).tolist()
    qo, segi, spi, off, ln, p0, dl, pids, pos = [0], [0], [0], [], [], [], [], [], []
    most = 0
    for nq, segs in seqs:
        p = 0
        for n, o, d in segs:
            pids += [free.pop() for _ in range(-(-(o + n) // ps))]
            spi.append(len(pids))
            off.append(o)
            ln.append(n)
            p0.append(p)
            dl.append(d)
            p += n
        pos += [max(0, p - nq + i + qpos_shift) for i in range(nq)]
        qo.append(qo[-1] + nq)
        segi.append(len(ln))
        most = max(most, p)
    host = {k: torch.tensor(v, dtype=torch.int32) for k, v in dict(
        qo_indptr=qo, positions=pos, seg_indptr=segi, seg_page_indptr=spi, seg_offset=off, seg_len=ln, seg_pos0=p0,
        seg_delta=dl, page_ids=pids).items()}
    most_q = max(n for n, _ in seqs)
    meta = ops.AttnMeta(num_seqs=len(seqs), max_q_len=most_q, max_kv_len=max(1, most), decode=most_q == 1, host=host,
                        **{k: v.to(device) for k, v in host.items()})
    return meta, qo[-1]


def rand_layer4(pages, hkv, ps, d, seed=0, device="cpu"):
    """A 4-bit layer of random values (some K channels larger) and its content in fp64 [P, 2, Hkv, page, D]."""
    g = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn(pages, 2, hkv, ps, d, generator=g, device=device)
    x[:, 0] *= 1 + 3 * (torch.arange(d, device=device) % 17 == 3)
    codes, scales = ops.kv4_pack_ref(x)
    return ops.KV4Layer(codes, scales)


def unpack64(layer):
    """Values of a layer in fp64, from the words' definition."""
    codes, scales = layer
    d = codes.shape[-1] * 2
    w = codes.contiguous().view(torch.int32).long()
    sc = scales.double()
    out = torch.empty(*codes.shape[:-1], d, dtype=torch.float64, device=codes.device)
    for i in range(d // 16):
        for h in range(2):
            for j in range(8):
                e = 8 * i + h * d // 2 + j
                out[..., e] = ((w[..., 2 * i + h] >> (4 * j)) & 15) * sc[..., e // 64, 0] + sc[..., e // 64, 1]
    return out


def rotate64(x, pos, cos, sin):
    h = x.shape[-1] // 2
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    a, b = x[..., :h], x[..., h:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def code8(layer):
    """What code 8 of each element's group stands for, 8 s + z in fp64 [P, 2, Hkv, page, D]: a 4-bit V enters the product
    with the rounded P as its distance from it, sum_n p_n (8 s_n + z_n) is added from unrounded p."""
    sc = layer.scales.double()
    return (8 * sc[..., 0] + sc[..., 1]).repeat_interleave(64, -1)


def dense64(q, kv, meta, cos, sin, scale, window=0, sinks=0, use_rope=True, base=None):
    """(out, A, B): the definition in fp64 over values kv [P, 2, Hkv, page, D]; A = sum_n w_n (|v_n| + |v_n - base_n|)
    and B = sum_n w_n |v_n| scale sum_d |q_d k_nd|, bounds of what errors of P (which multiplies v - base) and of q are
    multiplied by."""
    dev = kv.device
    h = {k: v.tolist() for k, v in meta.host.items()}
    T, hq, d = q.shape
    hkv, ps = kv.shape[2], kv.shape[3]
    out = torch.zeros(T, hq, d, dtype=torch.float64, device=dev)
    A, B = torch.zeros_like(out), torch.zeros_like(out)
    for b in range(meta.num_seqs):
        t0, t1 = h["qo_indptr"][b], h["qo_indptr"][b + 1]
        pos = torch.tensor(h["positions"][t0:t1], device=dev)
        sc, ab, vs, us = [], [], [], []
        for s in range(h["seg_indptr"][b], h["seg_indptr"][b + 1]):
            n = h["seg_len"][s]
            if n == 0 or t1 == t0:
                continue
            slot = h["seg_offset"][s] + torch.arange(n, device=dev)
            pg = torch.tensor(h["page_ids"], device=dev)[h["seg_page_indptr"][s] + slot // ps]
            k, v = (kv[pg, i, :, slot % ps].double() for i in (0, 1))
            qq = q[t0:t1].double().to(dev)
            if use_rope:
                at = (pos - h["seg_delta"][s]).clamp(0, cos.shape[0] - 1)
                qq = rotate64(qq, at, cos.to(dev), sin.to(dev))
            kk = k.repeat_interleave(hq // hkv, 1)
            x = torch.einsum("thd,nhd->htn", qq, kk) * scale
            kp = h["seg_pos0"][s] + torch.arange(n, device=dev)
            gap = pos[:, None] - kp[None]
            ok = gap >= 0
            if window:
                ok &= (gap < window) | (kp < sinks)[None]
            sc.append(x.masked_fill(~ok[None], -math.inf))
            ab.append(torch.einsum("thd,nhd->htn", qq.abs(), kk.abs()) * abs(scale))
            vs.append(v.repeat_interleave(hq // hkv, 1))
            us.append((v.abs() + (v - base[pg, 1, :, slot % ps]).abs() if base is not None else v.abs())
                      .repeat_interleave(hq // hkv, 1))
        if not sc:
            continue
        x, ab, v, u = torch.cat(sc, -1), torch.cat(ab, -1), torch.cat(vs, 0), torch.cat(us, 0)
        seen = x > -math.inf
        w = torch.nan_to_num(torch.softmax(x, -1), nan=0.0)
        # values that nobody sees (they may be NaN) take no part
        some = seen.any(1).any(0)[:, None, None]
        v, u = torch.where(some, v, torch.zeros_like(v)), torch.where(some, u, torch.zeros_like(u))
        ab = torch.where(seen, ab, torch.zeros_like(ab))
        out[t0:t1] = torch.einsum("htn,nhd->thd", w, v)
        A[t0:t1] = torch.einsum("htn,nhd->thd", w, u)
        B[t0:t1] = torch.einsum("htn,nhd->thd", w * ab, v.abs())
    return out.reshape(T, -1), A.reshape(T, -1), B.reshape(T, -1)


def tolerance(out, A, B, q_eps, p_eps, kv_eps=0.0):
    """Elementwise bound: a relative error e of the rounded queries moves scores by at most e sum |q k| scale, so a
    weight by twice that (its own and the normaliser's, first order; 10% for the rest); P rounds by p_eps; K and V by
    kv_eps; the output by 2^-8 (bf16).  2^-15 A covers ex2.approx and fp32 sums over the tests' lengths."""
    return 1.1 * ((2 * (q_eps + kv_eps)) * B + (p_eps + kv_eps + 2 ** -15) * A) + 2 ** -8 * out.abs() + 1e-30


# what each kernel rounds: (queries, P, K and V)
ROWS4 = (2 ** -11, 2 ** -11, 0.0)   # fp16 queries and P, exact codes
ROWS16 = (2 ** -16, 2 ** -8, 0.0)   # queries as two bf16 terms, bf16 P
TC16 = (2 ** -8, 2 ** -8, 0.0)      # long prompts: bf16 queries and P ...
TC4 = (2 ** -8, 2 ** -8, 2 ** -8)   # ... and a 4-bit cache read into bf16


def check(got, ref, eps, what=""):
    out, A, B = ref
    tol = tolerance(out, A, B, *eps)
    err = (got.double().to(out.device) - out).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (what, int(bad.sum()), float((err / tol).nan_to_num(nan=9e9).max()),
                           bad.nonzero()[:3].tolist())
