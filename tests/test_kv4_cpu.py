"""The 4-bit cache and windowed attention on CPU: format, append, read-back, masks, refusals and the engine."""
import pytest
import torch
from kv4_helpers import dense64, make_plan, rand_layer4, unpack64
from safetensors.torch import load_file

from braidinfer_b200 import LLM, ChunkedLLM, ChunkType, SamplingParams, ops
from braidinfer_b200.config import Config
from braidinfer_b200.errors import ConfigurationError
from braidinfer_b200.utils import oracle
from braidinfer_b200.utils.synthetic import hf_config, make_checkpoint


@pytest.mark.parametrize("d", [64, 128])
def test_pack_is_within_half_a_step(d):
    g = torch.Generator().manual_seed(d)
    x = torch.randn(5, 3, d, generator=g) * torch.exp(2 * torch.randn(5, 3, 1, generator=g)) + torch.randn(5, 3, 1, generator=g)
    codes, scales = ops.kv4_pack_ref(x)
    assert codes.shape == (5, 3, d // 2) and codes.dtype == torch.uint8 and scales.shape == (5, 3, d // 64, 2)
    back = unpack64(ops.KV4Layer(codes, scales))
    grp = x.double().unflatten(-1, (-1, 64))
    a, b, s = grp.amin(-1), grp.amax(-1), scales[..., 0].double()
    bound = s / 2 + 2 ** -8 * (a.abs() + b.abs()) + 1e-6 * (b - a)
    assert ((back.unflatten(-1, (-1, 64)) - grp).abs() <= bound[..., None]).all()
    assert torch.equal(ops.kv4_unpack_ref(codes, scales).double(), back.float().double())


def test_pack_of_flat_and_broken_groups():
    x = torch.zeros(6, 128)
    x[1] = 3.5
    x[2, 70] = float("nan")
    x[3, 1] = float("inf")
    x[4, 5], x[4, 6] = 3e38, -3e38
    x[5, :64] = torch.arange(64.0)
    back = ops.kv4_unpack_ref(*ops.kv4_pack_ref(x))
    assert (back[0] == 0).all() and (back[1] == 3.5).all()
    assert back[2, 64:].isnan().all() and (back[2, :64] == 0).all()  # the group alone
    assert back[3, :64].isnan().all() and back[4, :64].isnan().all()
    assert (back[5, :64] - x[5, :64]).abs().max() <= 63 / 30 + 0.25


@pytest.mark.parametrize("d,norm,rope", [(64, False, True), (128, True, True), (128, True, False)])
def test_append_and_read(d, norm, rope):
    g = torch.Generator().manual_seed(3)
    T, hq, hkv, ps, P = 9, 6, 2, 16, 3
    qkv = torch.randn(T, (hq + 2 * hkv) * d, generator=g)
    slots = torch.randperm(P * ps, generator=g)[:T].int()
    pos = torch.randint(0, 50, (T,), generator=g).int()
    cos, sin = ops.build_cos_sin(d, 1e4, 64)
    w = (1 + torch.rand(d, generator=g)) if norm else None
    cache = ops.KV4Cache(2, P, hkv, ps, d)
    before = cache[0].codes.clone()
    q = ops.qkv_prepare(qkv, pos, slots, cache[1], hq, hkv, d, cos, sin, w, w, 1e-6, rope)
    assert q.shape == (T, hq, d) and torch.equal(cache[0].codes, before)
    if not norm:
        assert torch.equal(q, qkv[:, :hq * d].view(T, hq, d))
    x = qkv.double().view(T, -1, d)
    k, v = x[:, hq:hq + hkv], x[:, hq + hkv:]
    if norm:
        k = k / (k.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
    if rope:
        from kv4_helpers import rotate64
        k = rotate64(k, pos.long(), cos, sin)
    got = ops.kv4_read(cache[1], slots).double()
    ref = torch.stack([k, v], 1)
    a, b = (getattr(ref.unflatten(-1, (-1, 64)), f)(-1) for f in ("amin", "amax"))
    step = ((b - a) / 15)[..., None].expand(*a.shape, 64).flatten(-2)
    far = 2 ** -8 * (a.abs() + b.abs())[..., None].expand(*a.shape, 64).flatten(-2)
    # half a step (s itself may round up by 2^-8), the ends' rounding, the read's rounding
    assert ((got - ref).abs() <= step * (0.5 + 2 ** -8) + far + 2 ** -8 * ref.abs() + 2 ** -8 * step + 1e-5).all()
    outside = ops.kv4_read(cache[1], torch.tensor([-1, P * ps], dtype=torch.int32))
    assert (outside == 0).all()


@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (7, 0), (7, 3), (40, 1), (1000, 2)])
@pytest.mark.parametrize("bits", [4, 16])
def test_attention_ref_against_dense(window, sinks, bits):
    d, hkv, ps, P = 64, 2, 16, 32
    seqs = [(1, [(1, 0, 0)]), (5, [(20, 3, 4), (0, 0, 0), (33, 0, -2), (5, 0, 0)]), (0, [(4, 0, 0)]), (3, [(50, 0, 0)])]
    meta, T = make_plan(seqs, ps, P, "cpu")
    layer = rand_layer4(P, hkv, ps, d)
    kv = unpack64(layer)
    q = torch.randn(T, 4, d, generator=torch.Generator().manual_seed(1))
    cos, sin = ops.build_cos_sin(d, 1e4, 128)
    got = ops.attention(q, layer if bits == 4 else kv.float(), meta, cos, sin, d ** -0.5, window=window, sinks=sinks)
    out, A, B = dense64(q, kv, meta, cos, sin, d ** -0.5, window, sinks)
    # fp32 throughout: 64-term dot products and softmax sums of at most 58 keys, each term off by 2^-24
    assert ((got.double() - out).abs() <= 200 * 2 ** -24 * (A + B) + 1e-12).all()


def test_rows_that_see_nothing_are_zero():
    d = 64
    meta, T = make_plan([(2, [(8, 0, 0)])], 16, 4, "cpu")
    meta.positions[:] = meta.host["positions"][:] = torch.tensor([100, 3], dtype=torch.int32)
    layer = rand_layer4(4, 1, 16, d)
    q = torch.randn(T, 2, d)
    cos, sin = ops.build_cos_sin(d, 1e4, 128)
    out = ops.attention(q, layer, meta, cos, sin, 0.1, window=5)
    assert (out[0] == 0).all() and (out[1] != 0).any()


def test_refusals():
    d = 64
    layer = rand_layer4(4, 1, 16, d)
    meta, T = make_plan([(1, [(8, 0, 0)])], 16, 4, "cpu")
    q = torch.randn(T, 2, d)
    cos, sin = ops.build_cos_sin(d, 1e4, 128)
    for w, s in ((-1, 0), (0, -1), (1 << 30, 0), (5, 1 << 30)):
        with pytest.raises(ValueError, match="window and sinks"):
            ops.attention(q, layer, meta, cos, sin, 0.1, window=w, sinks=s)
    meta.seq_nsh = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="shared-prefix"):
        ops.attention(q, layer, meta, cos, sin, 0.1)
    with pytest.raises(ValueError, match="one-dimensional"):
        ops.kv4_read(layer, torch.zeros(1, 1, dtype=torch.int32))
    with pytest.raises(ValueError, match="head_dim"):
        ops.KV4Cache(1, 2, 1, 16, 96)
    with pytest.raises(ValueError, match="sequence-parallel"):
        ops.qkv_gemm(q.view(1, -1), q, None, None, None, None, layer, 2, 1, d, cos, sin, rs_vec=q)


# ------------------------------------------------------------------ engine
KW = dict(num_kvcache_blocks=64, kvcache_block_size=16, device="cpu", dtype="float32")


@pytest.fixture(scope="module")
def ckpt(tmp_path_factory):
    d = make_checkpoint(str(tmp_path_factory.mktemp("kv4")), "tiny-llama", seed=0, dtype=torch.float32)
    return d, hf_config("tiny-llama"), load_file(d + "/model.safetensors")


@pytest.mark.parametrize("window,sinks", [(20, 0), (9, 4)])
def test_engine_window_matches_the_oracle(ckpt, window, sinks):
    d, cfg, sd = ckpt
    llm = LLM(d, sliding_window=window, attention_sinks=sinks, **KW)
    llm.model_runner.capture_logits = []
    prompt = list(range(5, 60))
    out = llm.generate(prompt, SamplingParams(temperature=0, max_tokens=6, ignore_eos=True))[0]
    ids = prompt + out["token_ids"]
    n = len(ids)
    i, j = torch.arange(n)[:, None], torch.arange(n)[None]
    mask = (j <= i) & ((i - j < window) | (j < sinks))
    ref = oracle.forward(cfg, sd, ids, list(range(n)), mask)
    for k, lg in enumerate(llm.model_runner.capture_logits):
        assert (lg[0] - ref[len(prompt) - 1 + k]).abs().max() < 1e-4


def test_engine_int4_cache_holds_what_the_format_says(ckpt):
    """The first layer's K and V do not depend on the cache: in 4 bits they are the full-precision engine's to within
    the format's bound (half a step, the rounding of the group's ends)."""
    d, _, _ = ckpt
    prompt = list(range(5, 60))
    held = []
    for extra in ({}, dict(kv_cache_dtype="int4")):
        llm = LLM(d, **KW, **extra)
        pages = list(llm.page_manager.free_pages)
        llm.generate(prompt, SamplingParams(temperature=0, max_tokens=1, ignore_eos=True))
        held.append((llm.page_manager, pages))
    (full, p0), (int4, p1) = held
    assert isinstance(int4.kv_cache, ops.KV4Cache) and p0 == p1
    assert int4.bytes_per_page * 64 == full.bytes_per_page * (36 / 256) * 64  # fp32 rows of 64 elements: 256 bytes
    n = len(prompt)
    slots = torch.arange(n)
    pg, off = torch.tensor(p0)[slots // 16], slots % 16
    x = full.kv_cache[0][pg, :, :, off].double().unflatten(-1, (-1, 64))
    y = unpack64(int4.kv_cache[0])[pg, :, :, off].unflatten(-1, (-1, 64))
    least, most, s = x.amin(-1), x.amax(-1), int4.kv_cache[0].scales[pg, :, :, off][..., 0].double()
    bound = s / 2 + 2 ** -8 * (least.abs() + most.abs()) + 1e-5
    assert ((x - y).abs() <= bound[..., None]).all() and (x != y).any()


def test_engine_int4_chunks_and_persistence(ckpt, tmp_path):
    from braidinfer_b200.persistence import load_chunks, save_chunks

    d, _, _ = ckpt
    g = torch.Generator().manual_seed(0)
    toks = [torch.randint(0, 1024, (n,), generator=g).tolist() for n in (21, 40, 9)]
    kinds = [ChunkType.SYSTEM_PROMPT, ChunkType.CONTEXT, ChunkType.QUERY]
    sp = dict(temperature=0, max_tokens=5, ignore_eos=True)

    def build(**kw):
        cl = ChunkedLLM(d, kv_cache_dtype="int4", **KW, **kw)
        return cl, [cl.register_chunk(f"c{i}", k, token_ids=toks[i]) for i, k in enumerate(kinds)]

    a, ids = build()
    first = a.generate_from_chunks(ids[0], ids[2], [ids[1]], sp)["token_ids"]
    save_chunks(a, str(tmp_path))
    b = ChunkedLLM(d, kv_cache_dtype="int4", **KW)
    load_chunks(b, str(tmp_path))
    assert b.registry.peek(ids[1]).kv_cache_allocated
    assert b.generate_from_chunks(ids[0], ids[2], [ids[1]], sp)["token_ids"] == first
    with pytest.raises(ValueError, match="different model"):
        load_chunks(ChunkedLLM(d, **KW), str(tmp_path))


def test_config_refusals(ckpt):
    d, _, _ = ckpt
    for bad in (dict(kv_cache_dtype="int3"), dict(sliding_window=0), dict(sliding_window=-4),
                dict(sliding_window=8, attention_sinks=-1), dict(attention_sinks=4),
                dict(kv_cache_dtype="int4", tensor_parallel_size=2)):
        with pytest.raises(ConfigurationError):
            Config(d, **bad)
    with pytest.raises(ConfigurationError, match="head_dim"):
        Config(d, kv_cache_dtype="int4", hf_config=dict(hf_config("tiny-llama"), head_dim=32))
