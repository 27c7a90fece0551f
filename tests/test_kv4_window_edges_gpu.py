"""4-bit and windowed attention on a GPU where launches, splits, values and batches end."""
import pytest
import torch
from kv4_helpers import ROWS4, ROWS16, TC4, TC16, check, code8, dense64, make_plan, rand_layer4, tolerance, unpack64

from braidinfer_b200 import ops
from braidinfer_b200.ops._ext import ext

pytestmark = pytest.mark.gpu

DEV = "cuda"
PLAN = ("qo_indptr", "positions", "seg_indptr", "seg_page_indptr", "seg_offset", "seg_len", "seg_pos0", "seg_delta",
        "page_ids")


@pytest.fixture
def tcgen05():
    """Calls of several queries with head_dim 128 take the tcgen05 kernel, whatever their size."""
    ext().attn_select_prefill_tc(1)
    yield
    ext().attn_select_prefill_tc(-1)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _tables(d, n=8192):
    return ops.build_cos_sin(d, 1e4, n, device=DEV)


def _pool(bits, pages, hkv, ps, d, seed=0):
    """(cache argument, its values fp64)"""
    if bits == 4:
        layer = rand_layer4(pages, hkv, ps, d, seed, DEV)
        return layer, unpack64(layer)
    kv = torch.randn(pages, 2, hkv, ps, d, device=DEV, generator=_gen(seed)).bfloat16()
    return kv, kv.double()


def _queries(T, hq, d, seed=1):
    return torch.randn(T, hq, d, device=DEV, generator=_gen(seed)).bfloat16()


# ---------------------------------------------------- launches and key splits
@pytest.mark.parametrize("bits", [4, 16])
def test_key_splits_without_keys_and_a_plan_written_just_before(bits, tcgen05):
    """Most key splits of the short sequences have no keys; the plan, the counters that join the splits and the memory of
    the output are written by the kernels right before the call, and two plans take turns."""
    d, G, ps, pages = 128, 4, 16, 600
    seqs = [(150, [(4000, 0, 0)]), (1, [(1, 0, 0)]), (3, [(140, 2, 0)]), (0, [(9, 0, 0)]), (20, [(20, 0, 0)])]
    plans = [make_plan(seqs, ps, pages, DEV, seed=i, qpos_shift=-7 * i)[0] for i in range(2)]
    cache, kv = _pool(bits, pages, 1, ps, d)
    T = 174
    q = _queries(T, G, d)
    cos, sin = _tables(d)
    window = 0 if bits == 4 else 1 << 29
    call = lambda meta: ops.attention(q, cache, meta, cos, sin, d ** -0.5, window=window)  # noqa: E731
    alone = []
    for meta in plans:
        torch.cuda.synchronize()
        alone.append(call(meta).clone())
        check(alone[-1], dense64(q, kv, meta, cos, sin, d ** -0.5, window), TC4 if bits == 4 else TC16)
    live = make_plan(seqs, ps, pages, DEV, seed=0)[0]
    outs = []
    for i in range(40):
        held = torch.full((T, G * d), float("nan"), device=DEV, dtype=torch.bfloat16)
        del held  # the call's output takes its place
        for f in PLAN:
            getattr(live, f).copy_(getattr(plans[i % 2], f))
        outs.append(call(live).clone())
    assert all(torch.equal(o, alone[i % 2]) for i, o in enumerate(outs))


@pytest.mark.parametrize("bits", [4, 16])
def test_a_call_without_any_visible_key_waits_for_what_came_before(bits, tcgen05):
    """No CTA has a key to load, so none waits for one: the zeros still come after what was written there before."""
    d, ps = 128, 16
    meta, T = make_plan([(256, [(0, 0, 0)])], ps, 16, DEV)
    cache, _ = _pool(bits, 16, 1, ps, d)
    q = _queries(T, 4, d)
    cos, sin = _tables(d)
    for _ in range(20):
        held = torch.empty(T, 4 * d, device=DEV, dtype=torch.bfloat16)
        held.fill_(7)
        del held
        out = ops.attention(q, cache, meta, cos, sin, d ** -0.5, window=300)
        after = out + 0
        assert (out == 0).all() and (after == 0).all()


# --------------------------------------------------------- tiles of the ring
@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("nq", [1, 4])
def test_every_number_of_tiles(bits, d, nq):
    """0 to 9 tiles of 64 or 128 keys in a CTA: fewer than the ring holds, as many, and more, so that the producer ends at
    every stage and phase.  Many sequences in one call, so that keys are not split."""
    hkv, G, ps = 2, 4, 16
    lens = [n for k in range(10) for n in (64 * k, 64 * k + 1)]
    seqs = [(nq, [(max(n, 1), 0, 0)]) for n in lens] * 12
    pages = sum(-(-max(n, 1) // ps) for n in lens) * 12
    meta, T = make_plan(seqs, ps, pages, DEV, qpos_shift=0)
    cache, kv = _pool(bits, pages, hkv, ps, d)
    q = _queries(T, hkv * G, d)
    cos, sin = _tables(d)
    window = 0 if bits == 4 else 1 << 29
    # of d 128 and several queries a sequence, the row kernel whatever the size of the batch
    ext().attn_select_prefill_tc(0)
    try:
        got = ops.attention(q, cache, meta, cos, sin, d ** -0.5, window=window)
    finally:
        ext().attn_select_prefill_tc(-1)
    ref = dense64(q, kv, meta, cos, sin, d ** -0.5, window, base=code8(cache) if bits == 4 else None)
    check(got, ref, ROWS4 if bits == 4 else ROWS16)


# ------------------------------------------------------------------ refusals
def test_head_counts_that_leave_nothing_are_refused():
    d, P, ps = 128, 4, 16
    empty = ops.KV4Layer(torch.zeros(P, 2, 0, ps, d // 2, dtype=torch.uint8, device=DEV),
                         torch.zeros(P, 2, 0, ps, d // 64, 2, dtype=torch.bfloat16, device=DEV))
    full = rand_layer4(P, 2, ps, d, 0, DEV)
    i = torch.zeros(3, dtype=torch.int32, device=DEV)
    cos, sin = _tables(d)
    qkv = torch.zeros(3, 2 * d, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="KV heads"):
        ops.kv4_read(empty, i)
    with pytest.raises(RuntimeError, match="KV heads"):
        ops.qkv_prepare(qkv, i, i, empty, 2, 0, d, cos, sin)
    with pytest.raises(RuntimeError, match="layout"):  # -2 + 2 * 2 heads are as wide as qkv
        ops.qkv_prepare(qkv, i, i, full, -2, 2, d, cos, sin)
    meta, T = make_plan([(1, [(20, 0, 0)])], ps, P, DEV)
    with pytest.raises(RuntimeError, match="head layout"):
        ops.attention(torch.zeros(T, 0, d, dtype=torch.bfloat16, device=DEV), full, meta, cos, sin, 0.1)
    with pytest.raises(RuntimeError, match="KV heads"):
        ops.attention(_queries(T, 4, d), empty, meta, cos, sin, 0.1)
    # no query heads to append with, and no tokens, are calls like any other
    assert ops.qkv_prepare(torch.zeros(1, 4 * d, dtype=torch.bfloat16, device=DEV), i[:1], i[:1], full, 0, 2, d, cos,
                           sin).shape == (1, 0, d)
    assert ops.kv4_read(full, i[:0]).shape == (0, 2, 2, d)


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("nq", [1, 300])
def test_tables_and_outputs_that_are_not_aligned_are_refused(bits, nq):
    """Contiguous tables one element into their storage: the kernels read them 16 bytes at a time."""
    d, ps, P = 128, 16, 64
    meta, T = make_plan([(nq, [(400, 0, 0)])], ps, P, DEV)
    cache, _ = _pool(bits, P, 2, ps, d)
    q = _queries(T, 8, d)
    cos, sin = _tables(d, 512)
    off = torch.empty(cos.numel() + 1, device=DEV)[1:].view_as(cos)
    off.copy_(cos)
    assert off.is_contiguous()
    for c, s in ((off, sin), (cos, off)):
        with pytest.raises(RuntimeError, match="aligned"):
            ops.attention(q, cache, meta, c, s, 0.1, window=100)
        if bits == 4:
            i = torch.zeros(1, dtype=torch.int32, device=DEV)
            with pytest.raises(RuntimeError, match="aligned"):
                ops.qkv_prepare(torch.zeros(1, 12 * d, dtype=torch.bfloat16, device=DEV), i, i, cache, 8, 2, d, c, s)
    out = torch.empty(T * 8 * d + 1, dtype=torch.bfloat16, device=DEV)[1:].view(T, 8 * d)
    kv, scales = cache if bits == 4 else (cache, None)
    with pytest.raises(RuntimeError, match="aligned"):
        ext().attention_rows(out, q, kv, scales, *(getattr(meta, f) for f in PLAN), cos, sin, 0.1, True, 1, nq, 400, 100, 0)
    # a table that starts at a later row is aligned
    got = ops.attention(q, cache, meta, cos[1:], sin[1:], 0.1, window=100)
    assert torch.equal(got, ops.attention(q, cache, meta, cos[1:].clone(), sin[1:].clone(), 0.1, window=100))


# ------------------------------------------------------------ scales and NaN
@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("rope", [False, True])
@pytest.mark.parametrize("scale", [-0.07, -1.5, 1e-30, 0.0])
def test_any_scale_in_the_tcgen05_kernel(bits, rope, scale, tcgen05):
    """Masked scores, maxima and edge tiles under a negative scale; a scale of 0 weighs every visible key alike."""
    d, G, hkv, ps, pages = 128, 4, 2, 16, 200
    seqs = [(300, [(700, 3, 0), (300, 0, 0)]), (40, [(40, 0, 0)]), (1, [(900, 0, 2)])]
    meta, T = make_plan(seqs, ps, pages, DEV)
    cache, kv = _pool(bits, pages, hkv, ps, d)
    q = _queries(T, hkv * G, d)
    cos, sin = _tables(d)
    got = ops.attention(q, cache, meta, cos, sin, scale, rope, window=500, sinks=3)
    ref = dense64(q, kv, meta, cos, sin, scale, 500, 3, rope)
    check(got, ref, TC4 if bits == 4 else TC16)


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("nq", [1, 6, 300])
def test_a_visible_nan_reaches_its_rows_and_no_other(bits, d, nq):
    """A NaN query, or a NaN in a key that a row sees, makes the row NaN, also where no other key of it is a number or
    where the other keys are other warps' and CTAs'; the other rows are what they were."""
    ps, hkv, G = 16, 2, 4
    lens = [1, 17, 33, 129, 3001]
    seqs = [(min(nq, n), [(n, 0, 0)]) for n in lens]
    pages = sum(-(-n // ps) for n in lens)
    meta, T = make_plan(seqs, ps, pages, DEV)
    cache, kv = _pool(bits, pages, hkv, ps, d)
    q = _queries(T, hkv * G, d)
    cos, sin = _tables(d)
    window = 0 if bits == 4 else 1 << 29
    run = lambda q, c: ops.attention(q, c, meta, cos, sin, d ** -0.5, window=window).view(T, hkv * G, d)  # noqa: E731
    clean = run(q, cache)
    assert clean.isfinite().all()
    h = meta.host
    first = [int(i) for i in h["qo_indptr"]]
    qn = q.clone()  # head 3 of each sequence's last token
    last = [i - 1 for i in first[1:]]
    qn[last, 3, 5] = float("nan")
    out = run(qn, cache)
    assert out[last, 3].isnan().all()
    out[last, 3] = clean[last, 3]
    assert torch.equal(out, clean)
    for b, n in enumerate(lens):  # the last key of one sequence after the other: only the last token sees it
        page, slot = int(h["page_ids"][int(h["seg_page_indptr"][b]) + (n - 1) // ps]), (n - 1) % ps
        if bits == 4:
            bad = ops.KV4Layer(cache.codes, cache.scales.clone())
            bad.scales[page, 0, 1, slot] = float("nan")
        else:
            bad = cache.clone()
            bad[page, 0, 1, slot, 7] = float("nan")
        out = run(q, bad)
        assert out[last[b], G:].isnan().all(), n
        out[last[b], G:] = clean[last[b], G:]
        assert torch.equal(out, clean), n


# --------------------------------------------- the ends of the 4-bit V range
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("nq", [1, 4])
@pytest.mark.parametrize("value", [0.0, -1000.0, 2.0 ** 30, -2.0 ** 45])
def test_constant_v_groups(d, nq, value):
    """Groups of one value have step 0: nothing moves the scale of P, and the offsets alone are summed, over scores that
    rise by nearly 2^8 without moving the maximum."""
    ps, hkv, G, n = 16, 1, 8 // nq if nq < 8 else 1, 3000
    pages = -(-n // ps) + 1
    meta, T = make_plan([(nq, [(n, 0, 0)])], ps, pages, DEV)
    layer = ops.KV4Cache(1, pages, hkv, ps, d, device=DEV)[0]
    h = meta.host
    kp = torch.zeros(pages, ps, device=DEV)
    for j in range(n):
        kp[int(h["page_ids"][j // ps]), j % ps] = j
    # K constant along D: score k d / d = k, in base 2 from 0 to 7.8 after the first 256 keys
    layer.scales[:, 0, :, :, :, 1] = torch.where(kp >= 256, 5.4, 0.0)[:, None, :, None].bfloat16()
    layer.scales[:, 1, :, :, :, 1] = value
    q = torch.ones(T, hkv * G, d, device=DEV, dtype=torch.bfloat16)
    cos, sin = _tables(d)
    got = ops.attention(q, layer, meta, cos, sin, 1.0 / d, use_rope=False)
    assert ((got.double() - value).abs() <= (2 ** -8 + 2 ** -15) * abs(value)).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("nq", [1, 4])
@pytest.mark.parametrize("exponent", [-45, 60, 110])
def test_v_steps_far_from_one(d, nq, exponent):
    ps, hkv, G, pages = 16, 2, 4, 64
    seqs = [(nq, [(300, 0, 0)]), (nq, [(40, 3, 0)])]
    meta, T = make_plan(seqs, ps, pages, DEV)
    layer = rand_layer4(pages, hkv, ps, d, 0, DEV)
    layer.scales[:, 1] *= 2.0 ** exponent
    q = _queries(T, hkv * G, d)
    cos, sin = _tables(d)
    got = ops.attention(q, layer, meta, cos, sin, d ** -0.5)
    check(got, dense64(q, unpack64(layer), meta, cos, sin, d ** -0.5, base=code8(layer)), ROWS4)


# -------------------------------------------------------- choice of the kernel
def _peak(call):
    """(what the call gives, bytes that it held beyond that at its peak)"""
    call()
    torch.cuda.synchronize()
    base = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = call()
    torch.cuda.synchronize()
    return out, torch.cuda.max_memory_allocated() - base - out.numel() * out.element_size()


@pytest.mark.parametrize("nq,n", [(2, 64), (3, 40)])
def test_many_sequences_of_few_queries_take_no_workspace(nq, n):
    """Rows of a sequence choose the kernel, not those of the batch: the pages are not read into bf16 for a few queries."""
    d, G, hkv, ps, keys = 128, 4, 2, 16, 1000
    pages = n * -(-keys // ps)
    meta, T = make_plan([(nq, [(keys, 0, 0)])] * n, ps, pages, DEV)
    cache, kv = _pool(4, pages, hkv, ps, d)
    q = _queries(T, hkv * G, d)
    cos, sin = _tables(d)
    out, held = _peak(lambda: ops.attention(q, cache, meta, cos, sin, d ** -0.5))
    check(out, dense64(q, kv, meta, cos, sin, d ** -0.5, base=code8(cache)), ROWS4)
    assert held <= 1 << 20 < pages * ps * hkv * 512


def test_a_shared_chunk_that_many_sequences_list_stays_within_the_workspace_limit():
    """160 sequences of 32 queries over one cached chunk of 8192 tokens: its pages, listed 160 times, would take 5.5 GB."""
    d, G, hkv, ps, nq, n, chunk = 128, 4, 8, 256, 32, 160, 8192
    one, _ = make_plan([(nq, [(chunk, 0, 3), (nq, 0, 0)])], ps, 40, DEV)
    layer = rand_layer4(40, hkv, ps, d, 0, DEV)
    cat = lambda f, step: torch.cat([getattr(one, f)[:-1] + i * step for i in range(n)] + [getattr(one, f)[-1:] + (n - 1) * step])  # noqa: E731
    many = ops.AttnMeta(num_seqs=n, max_q_len=nq, max_kv_len=one.max_kv_len, qo_indptr=cat("qo_indptr", nq),
                        seg_indptr=cat("seg_indptr", 2), seg_page_indptr=cat("seg_page_indptr", one.page_ids.numel()),
                        **{f: getattr(one, f).repeat(n) for f in ("positions", "seg_offset", "seg_len", "seg_pos0",
                                                                  "seg_delta", "page_ids")})
    limit = ext().attn_kv4_workspace_limit()
    assert many.page_ids.numel() * ps * hkv * 512 > limit
    q = _queries(nq, hkv * G, d)
    cos, sin = _tables(d, 9000)
    alone = ops.attention(q, layer, one, cos, sin, d ** -0.5)
    check(alone, dense64(q, unpack64(layer), one, cos, sin, d ** -0.5, base=code8(layer)), TC4)
    out, held = _peak(lambda: ops.attention(q.repeat(n, 1, 1), layer, many, cos, sin, d ** -0.5))
    assert held <= limit + (1 << 28)
    out = out.view(n, nq, -1)
    assert all(torch.equal(out[i], out[0]) for i in range(n))
    check(out[0], dense64(q, unpack64(layer), one, cos, sin, d ** -0.5, base=code8(layer)), TC4)


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("G,hkv", [(4, 2), (1, 8), (16, 1)])
def test_both_kernels_over_a_ragged_batch(bits, G, hkv):
    """The kernel that is chosen and the one that is not, over one long prompt among short ones."""
    d, ps = 128, 16
    seqs = [(400, [(300, 2, 1), (400, 0, 0)])] + [(1 + i % 5, [(60 + 37 * i, 0, 0)]) for i in range(12)]
    pages = 400
    meta, T = make_plan(seqs, ps, pages, DEV)
    cache, kv = _pool(bits, pages, hkv, ps, d)
    q = _queries(T, hkv * G, d)
    cos, sin = _tables(d)
    window = 0 if bits == 4 else 250
    ref = dense64(q, kv, meta, cos, sin, d ** -0.5, window, 2)
    outs = {}
    try:
        for mode in (0, 1, -1):
            ext().attn_select_prefill_tc(mode)
            outs[mode] = ops.attention(q, cache, meta, cos, sin, d ** -0.5, window=window, sinks=2)
            check(outs[mode], ref, TC4 if bits == 4 else TC16)
    finally:
        ext().attn_select_prefill_tc(-1)
    assert torch.equal(outs[-1], outs[0]) or torch.equal(outs[-1], outs[1])


def test_the_pool_leaves_room_for_the_workspace(tmp_path, monkeypatch):
    from braidinfer_b200 import LLM
    from braidinfer_b200.utils.synthetic import make_checkpoint
    ck = make_checkpoint(str(tmp_path), "tiny-qwen3", seed=0, head_dim=128)
    kw = dict(num_kvcache_blocks=32, kvcache_block_size=16, max_graph_batch=2)
    llm = LLM(ck, **kw)
    assert llm.model_runner.attention_workspace_bytes() == 0
    llm.exit()
    llm = LLM(ck, kv_cache_dtype="int4", **kw)
    mr = llm.model_runner
    limit = ext().attn_kv4_workspace_limit()
    # the pages of one sequence and the padding one in the prefill graphs; of 256 sequences in eager steps, the limit
    graph = (-(-mr.config.max_model_len // 16) + 17) * 16 * 2 * 512
    assert mr.attention_workspace_bytes() == min(limit, 256 * graph) + graph
    mr.config.num_kvcache_blocks = -1
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda *a: (120 << 30, 180 << 30))
    pages = mr.auto_num_pages()
    reserved = mr.attention_workspace_bytes()
    monkeypatch.setattr(mr, "attention_workspace_bytes", lambda: 0)
    assert abs((mr.auto_num_pages() - pages) * mr.kv_bytes_per_page() - reserved) <= mr.kv_bytes_per_page()
    llm.exit()


# ------------------------------------------------------------------- append
def test_append_gives_the_scales_of_the_cpu_form():
    """Ranges whose fifteenth lies on or next to a border between two bf16 numbers: 15 t with t of 9 bits."""
    d, ps, P = 64, 16, 16
    t = torch.arange(257, 512, 2)
    r = 15 * t
    top = (r // 32 * 32).float()
    x = torch.zeros(t.numel(), 3 * d)
    x[:, 2 * d], x[:, 2 * d + 1] = top, top - r.float()  # largest and least of V, both of at most 8 bits
    assert torch.equal(x.bfloat16().float(), x)
    slots = torch.arange(t.numel(), dtype=torch.int32)
    cos, sin = _tables(d)
    held = []
    for dev in ("cpu", DEV):
        layer = ops.KV4Cache(1, P, 1, ps, d, device=dev)[0]
        ops.qkv_prepare(x.bfloat16().to(dev), slots.to(dev), slots.to(dev), layer, 1, 1, d, cos.to(dev), sin.to(dev))
        held.append(layer)
    assert torch.equal(held[0].scales[:, 1], held[1].scales[:, 1].cpu())
    assert torch.equal(held[0].codes[:, 1], held[1].codes[:, 1].cpu())


@pytest.mark.multigpu
@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("nq", [1, 30, 300])
def test_tensors_on_another_device_than_the_current_one(bits, nq):
    if torch.cuda.device_count() < 2:
        pytest.skip("needs 2 GPUs")
    d, ps, hkv, G, pages = 128, 16, 2, 4, 64
    outs = []
    for dev in ("cuda:0", "cuda:1"):
        meta, T = make_plan([(nq, [(700, 0, 0)])], ps, pages, dev)
        cache = rand_layer4(pages, hkv, ps, d, 0, "cpu")
        cache = ops.KV4Layer(*(t.to(dev) for t in cache)) if bits == 4 else unpack64(cache).bfloat16().to(dev)
        q = torch.randn(T, hkv * G, d, generator=torch.Generator().manual_seed(1)).bfloat16().to(dev)
        cos, sin = ops.build_cos_sin(d, 1e4, 1024, device="cpu")
        out = ops.attention(q, cache, meta, cos.to(dev), sin.to(dev), d ** -0.5, window=600)
        assert out.device == torch.device(dev)
        outs.append(out.cpu())
        assert torch.cuda.current_device() == 0
    assert torch.equal(*outs)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("count", [3, 64])
@pytest.mark.parametrize("climb", [40, -6])
def test_decode_with_scores_and_v_steps_that_move(d, count, climb):
    """Decode rows whose scores climb by far more than 2^8 along the keys while V's steps climb by 2^40 or fall by 2^6:
    maxima and the power of two of P move, in the instances for few (3 sequences) and for many CTAs."""
    ps, hkv, G, pages = 16, 8, 1, 64 * 40
    lens = [600 - 7 * i for i in range(count)]
    meta, T = make_plan([(1, [(n, 0, 0)]) for n in lens], ps, pages, DEV)
    layer = rand_layer4(pages, hkv, ps, d, 0, DEV)
    part = torch.zeros(pages * ps, device=DEV)  # of every slot, how far along its sequence it lies
    h = meta.host
    largest = torch.zeros(T, hkv * G, d, dtype=torch.float64, device=DEV)
    places = []
    for b, n in enumerate(lens):
        j = torch.arange(n, device=DEV)
        at = h["page_ids"].to(DEV).long()[int(h["seg_page_indptr"][b]) + j // ps] * ps + j % ps
        part[at] = j / n
        places.append(at)
    part = part.view(pages, 1, ps, 1, 1)
    layer.scales[:, 0] = (layer.scales[:, 0].float() * (0.1 + 4 * part)).bfloat16()
    layer.scales[:, 1] = (layer.scales[:, 1].float() * torch.exp2(climb * (part - int(climb > 0)))).bfloat16()
    q = _queries(T, hkv * G, d)
    cos, sin = _tables(d)
    got = ops.attention(q, layer, meta, cos, sin, d ** -0.5, use_rope=False)
    out, A, B = dense64(q, unpack64(layer), meta, cos, sin, d ** -0.5, use_rope=False, base=code8(layer))
    # P s is held in fp16 against the largest step that the warp has met: below 2^-14 of it a rounding is 2^-25 of it,
    # times a code of at most 8 from the middle, for each key; the weights sum to at least 1, and as many terms of up to A
    # are summed in fp32
    for b, at in enumerate(places):
        step = layer.scales[at // ps, 1, :, at % ps][..., 0].double()  # [n, Hkv, D/64]
        largest[b] = step.amax(0).amax(-1)[:, None].expand(hkv, d)
    tol = tolerance(out, A, B, *ROWS4) + 600 * 2 ** -24 * A + 600 * 2 ** -22 * largest.view(T, -1)
    assert ((got.double() - out).abs() <= tol).all()
    # the bound says something: it is far below the outputs
    assert (tol.norm(dim=-1) <= 0.1 * out.norm(dim=-1)).all()


# -------------------------------------------------------------------- engine
@pytest.mark.parametrize("extra", [dict(kv_cache_dtype="int4"), dict(sliding_window=100, attention_sinks=3),
                                   dict(kv_cache_dtype="int4", sliding_window=100)])
@pytest.mark.parametrize("n", [33, 190, 250])
def test_engine_prefill_graphs_with_head_dim_128(extra, n, tmp_path, tcgen05):
    """A prompt through a captured prefill, padded in tokens, segments and pages, beside a padding sequence, on the tcgen05
    kernel and its workspace inside the graph: the K and V that it leaves are those of an eager step.  Layer 1's follow
    from the attention of layer 0."""
    from braidinfer_b200 import LLM, SamplingParams
    from braidinfer_b200.utils.synthetic import make_checkpoint
    ck = make_checkpoint(str(tmp_path), "tiny-qwen3", seed=0, head_dim=128)
    prompts = [[(7 * i + 13 * j) % 1000 + 3 for j in range(n)] for i in range(3)]
    held = []
    for eager in (True, False):
        llm = LLM(ck, num_kvcache_blocks=200, kvcache_block_size=16, max_graph_batch=2, enforce_eager=eager, **extra)
        for p in prompts:  # each on pages of its own; the graph is captured by the first and replayed by the others
            llm.generate([p], SamplingParams(temperature=0, max_tokens=1, ignore_eos=True))
        assert eager or llm.model_runner.prefill_graphs
        whole = llm.page_manager.kv_cache
        if isinstance(whole, ops.KV4Cache):
            held.append([unpack64(whole[i]) for i in range(2)])
        else:
            held.append([whole[i].double() for i in range(2)])
        llm.exit()
    scratch = 199
    for layer, (a, b) in enumerate(zip(*held)):
        a, b = (x[:scratch].movedim(3, 1).flatten(0, 1).flatten(1) for x in (a, b))  # a row per slot
        used = a.norm(dim=-1) > 0
        assert used.sum() >= 3 * n and torch.equal(used, b.norm(dim=-1) > 0)
        # bf16 hidden states differ by a few roundings of 2^-9, 2^-7 in all; in 4 bits such a shift puts 1 in 40 elements
        # on another code, a step (a fifteenth of the range, a third of the rms) off: 0.06 of the norm
        far = (a - b).norm(dim=-1)[used] / a.norm(dim=-1)[used]
        assert far.max() <= (2 ** -2 if "kv_cache_dtype" in extra else 2 ** -5), (layer, float(far.max()))


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("d,nq", [(64, 5), (128, 5), (128, 300)])
def test_queries_within_wider_rows(bits, d, nq):
    """Queries as the append returns them without a q norm, columns of the QKV rows, in every kernel."""
    hkv, G, ps, pages = 2, 4, 16, 64
    meta, T = make_plan([(nq, [(300, 1, 0), (nq, 0, 0)]), (1, [(33, 0, 0)])], ps, pages, DEV)
    cache, _ = _pool(bits, pages, hkv, ps, d)
    wide = torch.randn(T, (G + 2) * hkv * d + 8, device=DEV, generator=_gen(2)).bfloat16()
    q = wide[:, 8:8 + G * hkv * d].unflatten(1, (G * hkv, d))
    assert not q.is_contiguous()
    cos, sin = _tables(d)
    run = lambda q: ops.attention(q, cache, meta, cos, sin, d ** -0.5, window=250, sinks=2)  # noqa: E731
    assert torch.equal(run(q), run(q.contiguous()))
