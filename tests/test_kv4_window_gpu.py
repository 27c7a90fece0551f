"""The 4-bit cache kernels and windowed attention on a GPU against their definitions in 64 bits."""
import pytest
import torch
from kv4_helpers import ROWS4, ROWS16, TC4, TC16, check, code8, dense64, make_plan, rand_layer4, rotate64, tolerance, unpack64

from braidinfer_b200 import ops

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _tables(d, n=4096):
    return ops.build_cos_sin(d, 1e4, n, device=DEV)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _pool(bits, pages, hkv, ps, d, seed=0):
    """(cache argument, its values fp64, rounding of the kernels that read it)"""
    if bits == 4:
        layer = rand_layer4(pages, hkv, ps, d, seed, DEV)
        return layer, unpack64(layer)
    kv = torch.randn(pages, 2, hkv, ps, d, device=DEV, generator=_gen(seed)).bfloat16()
    return kv, kv.double()


def _run(q, cache, meta, d, window=0, sinks=0, rope=True, scale=None):
    cos, sin = _tables(d)
    return ops.attention(q, cache, meta, cos, sin, scale or d ** -0.5, rope, window=window, sinks=sinks)


def _against_definition(bits, d, G, hkv, ps, seqs, window, sinks, rope=True, pages=256, seed=0):
    meta, T = make_plan(seqs, ps, pages, DEV, seed)
    cache, kv = _pool(bits, pages, hkv, ps, d, seed)
    q = torch.randn(T, hkv * G, d, device=DEV, generator=_gen(seed + 1)).bfloat16()
    got = _run(q, cache, meta, d, window, sinks, rope)
    torch.cuda.synchronize()
    cos, sin = _tables(d)
    if d == 128 and meta.max_q_len > 1 and T * G >= 512:  # the long-prompt kernel
        check(got, dense64(q, kv, meta, cos, sin, d ** -0.5, window, sinks, rope), TC4 if bits == 4 else TC16)
    else:
        base = code8(cache) if bits == 4 else None
        check(got, dense64(q, kv, meta, cos, sin, d ** -0.5, window, sinks, rope, base), ROWS4 if bits == 4 else ROWS16)


# ------------------------------------------------------------ append, read
@pytest.mark.parametrize("d,hq,hkv", [(64, 4, 1), (128, 8, 2), (128, 12, 12)])
@pytest.mark.parametrize("T", [1, 7, 300])
@pytest.mark.parametrize("norm", [False, True])
def test_append_and_read(d, hq, hkv, T, norm):
    ps, P = 16, 32
    g = _gen(T)
    wide = (torch.randn(T, (hq + 2 * hkv) * d + 64, device=DEV, generator=g) * 3).bfloat16()
    qkv = wide[:, :(hq + 2 * hkv) * d]  # rows of a wider matrix
    slots = torch.randperm(P * ps, device=DEV, generator=g)[:T].int()
    pos = torch.randint(0, 4096, (T,), device=DEV, generator=g).int()
    cos, sin = _tables(d)
    qn = (1 + torch.rand(d, device=DEV, generator=g)).bfloat16() if norm else None
    kn = (50 * torch.randn(d, device=DEV, generator=g)).bfloat16() if norm else None
    cache = ops.KV4Cache(2, P, hkv, ps, d, device=DEV)
    cache.codes.fill_(0x5A)
    q = ops.qkv_prepare(qkv, pos, slots, cache[1], hq, hkv, d, cos, sin, qn, kn, 1e-6)
    got = ops.kv4_read(cache[1], slots).double()
    x = qkv.double().view(T, -1, d)
    qx, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    if norm:
        qx, k = (a / (a.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double() for a, w in ((qx, qn), (k, kn)))
    ref = torch.stack([rotate64(k, pos.long(), cos, sin), v], 1)
    assert ((q.double() - qx).abs() <= (2 ** -8 + 2 ** -20) * qx.abs()).all()
    a, b = (getattr(ref.unflatten(-1, (-1, 64)), f)(-1)[..., None].expand(T, 2, hkv, d // 64, 64).flatten(-2)
            for f in ("amin", "amax"))
    step, fp32 = (b - a) / 15, 2 ** -18 * (a.abs() + b.abs())  # fp32 norm and rotation of a row
    # half a step (s rounds by 2^-8), s and z rounded at the ends of the range, the read rounded
    tol = step * (0.5 + 2 ** -8) + 2 ** -8 * (a.abs() + b.abs()) + 2 ** -8 * (ref.abs() + step) + fp32
    assert ((got - ref).abs() <= tol).all()
    # and the codes are those of the CPU form except where fp32 sums put an element on the other side of a border
    cpu = ops.KV4Cache(1, P, hkv, ps, d)[0]
    ops.qkv_prepare(qkv.cpu(), pos.cpu(), slots.cpu(), cpu, hq, hkv, d, cos.cpu(), sin.cpu(),
                    None if qn is None else qn.cpu(), None if kn is None else kn.cpu(), 1e-6)
    s = slots.long()
    mine = unpack64(cache[1])[s // ps, :, :, s % ps]
    other = unpack64(cpu).to(DEV)[s // ps, :, :, s % ps]
    assert (mine != other).double().mean() <= 1e-2 and ((mine - other).abs() <= 1.1 * step + 2 ** -7 * (a.abs() + b.abs())).all()
    # nothing else was written
    touched = torch.zeros(P * ps, dtype=torch.bool, device=DEV)
    touched[s] = True
    rest = cache.codes[1].movedim(3, 1).reshape(P * ps, -1)[~touched]
    assert (rest == 0x5A).all() and (cache.codes[0] == 0x5A).all() and (cache.scales[0] == 0).all()


def test_append_skips_slots_outside_and_marks_broken_groups():
    d, hq, hkv, ps, P = 128, 2, 1, 16, 2
    qkv = torch.randn(5, 4 * d, device=DEV).bfloat16()
    qkv[1, 2 * d + 3] = float("nan")   # K of token 1, first half: its rotary partner breaks the second group too
    qkv[2, 3 * d + 100] = float("inf")  # V of token 2, second group
    qkv[3, 3 * d:] = 2.0
    cos, sin = _tables(d)
    layer = ops.KV4Cache(1, P, hkv, ps, d, device=DEV)[0]
    slots = torch.tensor([-1, 3, 4, 5, P * ps], device=DEV, dtype=torch.int32)
    pos = torch.tensor([0, 1, 2, 3, 4], device=DEV, dtype=torch.int32)
    ops.qkv_prepare(qkv, pos, slots, layer, hq, hkv, d, cos, sin)
    got = ops.kv4_read(layer, slots).float()
    assert (got[0] == 0).all() and (got[4] == 0).all()
    assert got[1, 0].isnan().all() and got[1, 1].isfinite().all()
    assert got[2, 1, 0, 64:].isnan().all() and got[2, 1, 0, :64].isfinite().all() and got[2, 0].isfinite().all()
    assert (got[3, 1] == 2).all()
    flat = layer.codes.movedim(3, 1).reshape(P * ps, -1)
    flat = torch.cat([flat[:3], flat[6:]])
    assert (flat == 0).all()


# --------------------------------------------------------------- attention
DECODE = [(1, [(37, 0, 5), (100, 3, -7), (9, 0, 0)]), (1, [(1, 0, 0)]), (1, [(300, 0, 0)]), (0, [(5, 0, 0)]),
          (1, [(64, 0, 2), (0, 0, 0), (64, 0, 0), (130, 0, 0)]), (1, [(16, 0, 0)]), (1, [(17, 15, 0)])]


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("d,G,hkv", [(64, 8, 2), (64, 1, 3), (128, 4, 2), (128, 2, 1), (128, 12, 1), (128, 40, 1)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (50, 3), (4000, 1)])
def test_decode(bits, d, G, hkv, window, sinks):
    if bits == 16 and window == 0:
        window = 1 << 29  # every earlier key, through the windowed kernels
    _against_definition(bits, d, G, hkv, 16, DECODE, window, sinks)


PROMPT = [(50, [(40, 0, 3), (70, 5, -11), (50, 0, 0)]), (1, [(1, 0, 0)]), (200, [(200, 0, 0)]), (0, [(8, 0, 0)]),
          (17, [(128, 0, 0), (33, 0, 0)]), (3, [(3, 0, 0)])]


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("d,G,hkv", [(64, 8, 2), (64, 1, 3), (128, 4, 2), (128, 1, 1)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (30, 0), (64, 16)])
@pytest.mark.parametrize("ps", [16, 48])
def test_several_queries(bits, d, G, hkv, window, sinks, ps):
    if bits == 16 and window == 0:
        window = 1 << 29
    _against_definition(bits, d, G, hkv, ps, PROMPT, window, sinks, seed=ps)


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("d", [64, 128])
def test_long_contexts_split_over_a_cluster(bits, d):
    seqs = [(1, [(3000, 7, 0), (2000, 0, 1)]), (1, [(129, 0, 0)]), (1, [(4096, 0, 0)])]
    _against_definition(bits, d, 4, 1, 256, seqs, 0 if bits == 4 else 3500, 0 if bits == 4 else 7, pages=64)


LONG = {
    "prompts": [(700, [(700, 0, 0)]), (0, [(3, 0, 0)]), (1500, [(1500, 0, 0)]), (1, [(1, 0, 0)])],
    "queries over chunks": [(300, [(1000, 0, 9), (0, 0, 0), (2000, 37, -3), (450, 0, 0)]), (290, [(290, 0, 0)])],
}


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("name", list(LONG))
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (100, 5), (700, 130), (1024, 0), (5000, 1)])
@pytest.mark.parametrize("ps,G,hkv", [(16, 4, 1), (256, 8, 2), (48, 4, 2)])
def test_long_prompts(bits, name, window, sinks, ps, G, hkv):
    """128-key tiles cut by windows, sinks, segments and pages; few row tiles, so keys are split too."""
    if bits == 16 and window == 0:
        window = 1 << 29
    _against_definition(bits, 128, G, hkv, ps, LONG[name], window, sinks, pages=-(-5200 // ps) + 12, seed=window)


@pytest.mark.parametrize("bits", [4, 16])
def test_without_rope_and_gpt2_heads(bits):
    _against_definition(bits, 64, 1, 12, 256, [(1, [(500, 0, 0)]), (1, [(3, 0, 0)])], 100, 0, rope=False, pages=16)


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("d", [64, 128])
def test_many_segments(bits, d):
    """More segments than the kernel keeps in shared memory, each with its own RoPE delta."""
    seqs = [(1, [(5 + j % 3, j % 16, j % 7) for j in range(90)]), (3, [(7, 0, -(j % 3)) for j in range(70)] + [(3, 0, 0)]),
            (1, [(0, 0, 0)] * 80 + [(4, 0, 0)])]
    _against_definition(bits, d, 4, 2, 16, seqs, 300, 9, pages=400)


@pytest.mark.parametrize("bits", [4, 16])
def test_negative_scale_and_zero_queries(bits):
    d = 128
    meta, T = make_plan([(1, [(200, 0, 0)]), (1, [(33, 0, 0)])], 16, 64, DEV)
    cache, kv = _pool(bits, 64, 2, 16, d)
    q = torch.randn(T, 8, d, device=DEV, generator=_gen(3)).bfloat16()
    q[1, 3:6] = 0
    cos, sin = _tables(d)
    got = _run(q, cache, meta, d, 100, 2, scale=-0.07)
    ref = dense64(q, kv, meta, cos, sin, -0.07, 100, 2, base=code8(cache) if bits == 4 else None)
    check(got, ref, ROWS4 if bits == 4 else ROWS16)


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("nq", [1, 6])
def test_rows_that_see_nothing_are_zero(bits, nq):
    d = 128
    meta, T = make_plan([(nq, [(40, 0, 0)]), (nq, [(0, 0, 0)]), (nq, [])], 16, 64, DEV)
    meta.positions[0] = 1000
    cache, _ = _pool(bits, 64, 2, 16, d)
    q = torch.randn(T, 8, d, device=DEV).bfloat16()
    out = _run(q, cache, meta, d, window=30).view(T, 8, d)
    assert (out[0] == 0).all() and (out[nq:] == 0).all()
    assert nq == 1 or (out[1:nq] != 0).any(-1).all()


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("nq", [1, 5, 300])
def test_slots_that_nobody_sees_may_hold_anything(bits, d, nq):
    """NaN and infinities in slots before, behind and between what the queries see."""
    ps = 16
    seqs = [(nq, [(30, 3, 0), (100, 5, 0), (16 + nq, 0, 0)]), (nq, [(nq, 0, 0)])]
    window, sinks = 40, 6
    meta, T = make_plan(seqs, ps, 64, DEV)
    cache, kv = _pool(bits, 64, 2, ps, d)
    q = torch.randn(T, 8, d, device=DEV, generator=_gen(2)).bfloat16()
    clean = _run(q, cache, meta, d, window, sinks)
    seen = torch.zeros(64, ps, dtype=torch.bool)
    h = meta.host
    for b in range(2):
        pos = h["positions"][h["qo_indptr"][b]:h["qo_indptr"][b + 1]]
        for s in range(int(h["seg_indptr"][b]), int(h["seg_indptr"][b + 1])):
            for j in range(int(h["seg_len"][s])):
                kp, slot = int(h["seg_pos0"][s]) + j, int(h["seg_offset"][s]) + j
                gap = pos - kp
                if ((gap >= 0) & ((gap < window) | (kp < sinks))).any():
                    seen[int(h["page_ids"][int(h["seg_page_indptr"][s]) + slot // ps]), slot % ps] = True
    bad = (~seen).to(DEV)[:, None, None, :, None].expand(64, 2, 2, ps, 1)
    if bits == 4:
        dirty = ops.KV4Layer(torch.where(bad, torch.full_like(cache.codes, 255), cache.codes),
                             torch.where(bad[..., None], torch.full_like(cache.scales, float("nan")), cache.scales))
    else:
        dirty = torch.where(bad, torch.full_like(cache, float("nan")), cache)
    assert torch.equal(_run(q, dirty, meta, d, window, sinks), clean) and clean.isfinite().all()


def test_large_scores_and_scales():
    """Scores that climb by far more than 2^8 along the keys, V steps that grow by 2^20: running maxima and the V scale move."""
    d, hkv, ps = 128, 1, 16
    meta, T = make_plan([(1, [(600, 0, 0)]), (4, [(300, 0, 0)])], ps, 64, DEV)
    layer, _ = _pool(4, 64, hkv, ps, d)
    ramp = torch.ones(64, ps, device=DEV)
    h = meta.host
    for s in range(2):
        for j in range(int(h["seg_len"][s])):
            ramp[int(h["page_ids"][int(h["seg_page_indptr"][s]) + j // ps]), j % ps] = j
    layer.scales[:, 0] = (layer.scales[:, 0].float() * (0.1 + ramp / 40)[:, None, :, None, None]).bfloat16()
    layer.scales[:, 1] = (layer.scales[:, 1].float() * torch.exp2(ramp / 15 - 20).clamp(max=2 ** 20)[:, None, :, None, None]).bfloat16()
    kv = unpack64(layer)
    q = torch.randn(T, 4, d, device=DEV, generator=_gen(3)).bfloat16()
    cos, sin = _tables(d)
    got = _run(q, layer, meta, d, rope=False)
    ref = dense64(q, kv, meta, cos, sin, d ** -0.5, use_rope=False, base=code8(layer))
    # P s is held in fp16 against the largest step (or offset) the warp has met: below 2^-14 of it a rounding is 2^-25 of
    # it, times a code of at most 8 from the middle, for each of at most 600 keys; weights sum to at least 1 (their
    # largest is), and 600 terms of up to A are summed in fp32
    out, A, B = ref
    tol = tolerance(out, A, B, *ROWS4) + 600 * 2 ** -24 * A + 600 * 2 ** -22 * layer.scales[:, 1].double().abs().amax()
    assert ((got.double() - out).abs() <= tol).all()


def test_a_cache_past_32_bit_offsets():
    d, hkv, ps = 128, 8, 256
    pages = (5 << 30) // (2 * hkv * ps * 64)  # 5 GiB of codes
    codes = torch.empty(pages, 2, hkv, ps, d // 2, dtype=torch.uint8, device=DEV)
    scales = torch.empty(pages, 2, hkv, ps, d // 64, 2, dtype=torch.bfloat16, device=DEV)
    small = rand_layer4(4, hkv, ps, d, 0, DEV)
    codes[-4:], scales[-4:] = small.codes, small.scales
    meta, T = make_plan([(1, [(700, 3, 0)])], ps, 4, DEV)
    q = torch.randn(T, 32, d, device=DEV, generator=_gen(4)).bfloat16()
    ref = _run(q, small, meta, d)
    slots = torch.tensor([5, 3 * ps + 255], device=DEV, dtype=torch.int32)
    read = ops.kv4_read(small, slots)
    meta.page_ids += pages - 4
    far = ops.KV4Layer(codes, scales)
    assert torch.equal(_run(q, far, meta, d), ref)
    assert torch.equal(ops.kv4_read(far, slots + (pages - 4) * ps), read)
    qkv = torch.randn(2, 48 * d, device=DEV, generator=_gen(5)).bfloat16()
    cos, sin = _tables(d)
    pos = torch.tensor([1, 2], device=DEV, dtype=torch.int32)
    for layer, s in ((small, slots), (far, slots + (pages - 4) * ps)):
        ops.qkv_prepare(qkv, pos, s, layer, 32, hkv, d, cos, sin)
    assert torch.equal(codes[-4:], small.codes) and torch.equal(scales[-4:], small.scales)


# ------------------------------------------------- streams, graphs, devices
@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("nq", [1, 9, 256])
def test_streams_and_graphs(bits, nq):
    """Two calls at once on two streams, and two captured graphs replayed together, give what one call gives."""
    d, hkv, ps = 128, 2, 16
    plans = [make_plan([(nq, [(2000 + 300 * i, 0, 0)]), (1, [(77, 0, 0)])], ps, 256, DEV, seed=i) for i in range(2)]
    cache, _ = _pool(bits, 256, hkv, ps, d)
    qs = [torch.randn(nq + 1, 8, d, device=DEV, generator=_gen(i)).bfloat16() for i in range(2)]
    call = [lambda i=i: _run(qs[i], cache, plans[i][0], d, window=900, sinks=2) for i in range(2)]
    alone = [c().clone() for c in call]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i].append(call[i]())
    torch.cuda.synchronize()
    assert all(torch.equal(o, alone[i]) for i in range(2) for o in outs[i])
    cos, sin = _tables(d)
    graphs, held = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(ops.attention(qs[i], cache, plans[i][0], cos, sin, d ** -0.5, window=900, sinks=2))
        graphs.append(g)
    for _ in range(10):
        for o in held:
            o.zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, a) for o, a in zip(held, alone))


def test_append_then_attend_in_one_graph():
    """The operators as a decode step uses them: append this step's tokens in 4 bits, then attend through a window, over
    what a prompt left in the cache; eager and replayed with new inputs, against the definition over what the cache holds."""
    d, hq, hkv, ps, P = 128, 8, 2, 16, 64
    cos, sin = _tables(d)
    cache = ops.KV4Cache(1, P, hkv, ps, d, device=DEV)[0]
    lens = [100, 33]
    meta, _ = make_plan([(1, [(n + 1, 0, 0)]) for n in lens], ps, P, DEV)
    spi = meta.host["seg_page_indptr"].tolist()
    slot = lambda b, j: int(meta.host["page_ids"][spi[b] + j // ps]) * ps + j % ps  # noqa: E731
    width = (hq + 2 * hkv) * d
    for b, n in enumerate(lens):  # the prompts
        s = torch.tensor([slot(b, j) for j in range(n)], device=DEV, dtype=torch.int32)
        ops.qkv_prepare(torch.randn(n, width, device=DEV, generator=_gen(b)).bfloat16(),
                        torch.arange(n, device=DEV, dtype=torch.int32), s, cache, hq, hkv, d, cos, sin)
    new = torch.tensor([slot(b, n) for b, n in enumerate(lens)], device=DEV, dtype=torch.int32)
    qkv = torch.randn(2, width, device=DEV, generator=_gen(7)).bfloat16()

    def step():
        q = ops.qkv_prepare(qkv, meta.positions, new, cache, hq, hkv, d, cos, sin)
        return q, ops.attention(q, cache, meta, cos, sin, d ** -0.5, window=50, sinks=4)

    q, out = step()
    check(out, dense64(q, unpack64(cache), meta, cos, sin, d ** -0.5, 50, 4, base=code8(cache)), ROWS4)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        q, out = step()
    qkv.copy_(torch.randn(2, width, device=DEV, generator=_gen(8)))
    g.replay()
    torch.cuda.synchronize()
    check(out, dense64(q, unpack64(cache), meta, cos, sin, d ** -0.5, 50, 4, base=code8(cache)), ROWS4)


def test_tokens_behind_the_last_sequence_are_left_alone():
    d = 128
    meta, T = make_plan([(1, [(40, 0, 0)])], 16, 8, DEV)
    meta.positions = torch.cat([meta.positions, meta.positions.new_zeros(3)])
    layer = rand_layer4(8, 2, 16, d, 0, DEV)
    q = torch.randn(T + 3, 8, d, device=DEV).bfloat16()
    out = torch.full((T + 3, 8 * d), 7.0, device=DEV, dtype=torch.bfloat16)
    from braidinfer_b200.ops._ext import ext
    cos, sin = _tables(d)
    ext().attention_rows(out, q, *layer, meta.qo_indptr, meta.positions, meta.seg_indptr, meta.seg_page_indptr,
                         meta.seg_offset, meta.seg_len, meta.seg_pos0, meta.seg_delta, meta.page_ids, cos, sin, 0.1,
                         True, 1, 1, 40, 0, 0)
    assert (out[T:] == 7).all() and (out[:T] != 7).any()


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("nq", [1, 5])
def test_page_ids_outside_the_pool_stay_inside_it(bits, nq):
    """The kernel reads the first or the last page instead; the other sequence's rows are what they were."""
    d = 128
    meta, T = make_plan([(nq, [(100, 0, 0)]), (nq, [(60, 0, 0)])], 16, 64, DEV)
    cache, _ = _pool(bits, 64, 2, 16, d)
    q = torch.randn(T, 8, d, device=DEV, generator=_gen(1)).bfloat16()
    good = _run(q, cache, meta, d, 200, 1)
    meta.page_ids[1], meta.page_ids[2] = -7, 64
    bad = _run(q, cache, meta, d, 200, 1)
    assert torch.equal(bad[nq:], good[nq:]) and bad.isfinite().all()


def test_refusals():
    d = 128
    meta, T = make_plan([(1, [(40, 0, 0)])], 16, 8, DEV)
    layer = rand_layer4(8, 2, 16, d, 0, DEV)
    q = torch.randn(T, 8, d, device=DEV).bfloat16()
    cos, sin = _tables(d)
    bad = [
        (q.float(), layer, meta, cos), (q[..., :64].contiguous(), layer, meta, cos), (q[:, :7].contiguous(), layer, meta, cos),
        (q, ops.KV4Layer(layer.codes.cpu(), layer.scales), meta, cos),
        (q, ops.KV4Layer(layer.codes, layer.scales.float()), meta, cos),
        (q, ops.KV4Layer(layer.codes[:4], layer.scales), meta, cos),
        (q, ops.KV4Layer(layer.codes[:, :, :, ::2], layer.scales[:, :, :, ::2]), meta, cos),
        (q, layer, meta, cos.half()), (q, layer, meta, cos[:, :32].contiguous()),
    ]
    for qq, ly, m, c in bad:
        with pytest.raises(RuntimeError):
            ops.attention(qq, ly, m, c, sin if c.shape == sin.shape else c, 0.1)
    meta.positions = meta.positions.long()
    with pytest.raises(RuntimeError, match="positions"):
        ops.attention(q, layer, meta, cos, sin, 0.1)
    qkv = torch.randn(2, 12 * d, device=DEV).bfloat16()
    i = torch.zeros(2, device=DEV, dtype=torch.int32)
    for args in ((qkv.float(), i, i, layer), (qkv[:, :-8], i, i, layer), (qkv, i.long(), i, layer), (qkv, i, i[:1], layer)):
        with pytest.raises(RuntimeError):
            ops.qkv_prepare(*args, 8, 2, d, cos, sin)
    with pytest.raises(RuntimeError):
        ops.kv4_read(layer, i.long())
    with pytest.raises(RuntimeError):
        ops.attention(q, torch.zeros(8, 2, 2, 24, d, device=DEV, dtype=torch.bfloat16), meta, cos, sin, 0.1, window=5)


# ------------------------------------------------------------------ engine
@pytest.mark.parametrize("extra", [dict(kv_cache_dtype="int4"), dict(sliding_window=24, attention_sinks=3),
                                   dict(kv_cache_dtype="int4", sliding_window=24)])
def test_engine_graphs_match_eager(extra, tmp_path):
    """Decode and short-prefill graphs give the tokens of eager steps, with either cache and a window, and a second
    engine beside the first."""
    from braidinfer_b200 import LLM, SamplingParams
    from braidinfer_b200.utils.synthetic import make_checkpoint
    ck = make_checkpoint(str(tmp_path), "tiny-llama", seed=0)
    prompts = [list(range(3, 70)), list(range(7, 30)), [5]]
    sp = SamplingParams(temperature=0, max_tokens=20, ignore_eos=True)
    got = []
    for eager in (True, False):
        llm = LLM(ck, num_kvcache_blocks=64, kvcache_block_size=16, max_graph_batch=4, enforce_eager=eager, **extra)
        got.append([o["token_ids"] for o in llm.generate(prompts, sp)])
        llm.exit()
    assert got[0] == got[1]


def test_checked_build_records_bad_slots_and_pages():
    """The bounds-checked build records a slot and a page id outside the 4-bit cache, whose accesses are skipped or held
    inside in every build."""
    try:
        from braidinfer_b200 import _C_checked as C
    except ImportError:
        pytest.skip("bounds-checked build not present")
    from braidinfer_b200.ops import _ext
    _ext.ext()
    saved, d = _ext._C, 128
    _ext._C = _ext._Counted(C)
    try:
        C.bounds_check_status()
        layer = rand_layer4(8, 2, 16, d, 0, DEV)
        cos, sin = _tables(d)
        pos = torch.zeros(2, device=DEV, dtype=torch.int32)
        qkv = torch.randn(2, 12 * d, device=DEV).bfloat16()
        ops.qkv_prepare(qkv, pos, torch.tensor([3, 128], device=DEV, dtype=torch.int32), layer, 8, 2, d, cos, sin)
        v = int(C.bounds_check_status())
        assert (v >> 48, v & 0xFFFFFFFFFFFF) == (1, 128)
        meta, T = make_plan([(1, [(40, 0, 0)])], 16, 8, DEV)
        q = torch.randn(T, 8, d, device=DEV).bfloat16()
        _run(q, layer, meta, d)
        assert int(C.bounds_check_status()) == 0
        meta.page_ids[1] = 9
        _run(q, layer, meta, d)
        v = int(C.bounds_check_status())
        assert (v >> 48, v & 0xFFFFFFFFFFFF) == (4, 9)
    finally:
        torch.cuda.synchronize()
        _ext._C = saved
