"""The 8-bit cache and truncated sampling as the sampler uses them: forward passes that fill and read the cache,
generate(cache=, kv_dtype=, top_k=, top_p=, min_p=) step by step, the stepper."""
import numpy as np
import pytest

from oracle import kv8 as okv
from oracle import sampler as osamp
from oracle import sampling as osm
from oracle.bf16 import ulp_distance
from oracle.model import LLaDAConfig as OCfg
from oracle.model import init_weights
from tests.test_block_cache_gpu import build, max_rel

MASK_ID = 511

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def small():
    ocfg = OCfg(d_model=256, n_layers=3, n_heads=2, mlp_hidden=512, vocab_size=512)
    return ocfg, init_weights(ocfg, seed=33, std=0.05, head_scale=4.0)


def image_rows(kv, ocfg, n, L):
    """The bf16 image cache as [layers, n, L, 3, heads, 128]."""
    return kv.view(torch.bfloat16).view(ocfg.n_layers, n, L, 3, ocfg.n_heads, 128)


def case(seed, n=3, L=200):
    g = np.random.Generator(np.random.PCG64(seed))
    ids = torch.from_numpy(g.integers(0, 511, size=(n, L), dtype=np.int64)).cuda()
    km = np.ones((n, L), dtype=np.int64)
    km[n - 1, :70] = 0
    return g, ids, km, torch.from_numpy(km).cuda()


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
@pytest.mark.parametrize("packed", [True, False])
def test_filled_cache_holds_the_forwards_keys_and_values(lib, small, packed, dtype):
    ocfg, W = small
    model = build(ocfg, W, packed)
    n, L = 3, 200
    g, ids, km, am = case(1)
    rows = torch.arange(n * L, dtype=torch.int32, device="cuda")
    plain = model.forward_rows(ids, am, rows)
    kv, kv8 = model.kv_cache(n, L), model.kv_cache(n, L, dtype)
    image = model.forward_rows(ids, am, rows, kv_cache=kv)
    assert torch.equal(plain, model.forward_rows(ids, am, rows, kv_cache=kv8)) and torch.equal(plain, image)
    im = image_rows(kv, ocfg, n, L).double().cpu().numpy()
    for layer in range(ocfg.n_layers):
        k, v = (t.double().cpu().numpy() for t in kv8.read(layer))
        assert np.array_equal(k, okv.held(im[layer, :, :, 1], dtype, km)) and np.array_equal(v, okv.held(im[layer, :, :, 2], dtype, km))


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
@pytest.mark.parametrize("bs,bl", [(100, 36), (64, 64), (130, 70), (0, 200), (199, 1)])
def test_block_step_equals_the_image_step_on_the_held_values(lib, small, dtype, bs, bl):
    """The values a cache holds are exact in bf16: an image cache given them must lead to the same logits, up to the order
    of float32 sums (the forward's bf16 bound).  Writing the block back leaves the logits as they are."""
    ocfg, W = small
    model = build(ocfg, W)
    n, L = 3, 200
    g, ids, km, am = case(2)
    kv, a, b = model.kv_cache(n, L), model.kv_cache(n, L, dtype), model.kv_cache(n, L, dtype)
    for c in (kv, a, b):
        model.forward_rows(ids, am, None, kv_cache=c)
    im = image_rows(kv, ocfg, n, L)
    for layer in range(ocfg.n_layers):
        im[layer, :, :, 1], im[layer, :, :, 2] = a.read(layer)
    blk = torch.from_numpy(g.integers(0, 511, size=(n, bl), dtype=np.int64)).cuda()
    want = model.forward_block(blk, am, L, bs, kv, update_cache=False).float().cpu().numpy()
    before = a.data.clone()
    got = model.forward_block(blk, am, L, bs, a, update_cache=False)
    assert torch.equal(a.data, before)
    again = model.forward_block(blk, am, L, bs, b, update_cache=True)
    assert torch.equal(got, again) and not torch.equal(a.data, b.data)
    assert max_rel(got.float().cpu().numpy(), want) <= 2e-2
    # layer 0's fresh rows depend on the block's tokens alone: the written cache is known exactly
    kvu = model.kv_cache(n, L)
    model.forward_rows(ids, am, None, kv_cache=kvu)
    model.forward_block(blk, am, L, bs, kvu, update_cache=True)
    fresh = image_rows(kvu, ocfg, n, L)[0, :, bs:bs + bl].double().cpu().numpy()
    for i, t in enumerate(b.read(0)):
        old = a.read(0)[i].double().cpu().numpy()
        assert np.array_equal(t.double().cpu().numpy(), okv.updated(old, fresh[:, :, 1 + i], bs, dtype, km))


def test_mismatched_cache_is_refused(lib, small):
    ocfg, W = small
    model = build(ocfg, W)
    ids = torch.zeros((2, 32), dtype=torch.long, device="cuda")
    for bad in (model.kv_cache(1, 32, "e4m3"), model.kv_cache(2, 33, "e4m3")):
        with pytest.raises(ValueError):
            model.forward_rows(ids, None, None, kv_cache=bad)
        with pytest.raises(ValueError):
            model.forward_block(ids[:, :4], None, 32, 0, bad)
    with pytest.raises(AssertionError):
        model.forward_block(ids[:, :4], None, 32, 30, model.kv_cache(2, 32, "e4m3"))
    with pytest.raises(NotImplementedError):
        model.kv_cache(2, 32, "fp6")


@pytest.mark.parametrize("cache", ["dual", "prefix"])
@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
def test_single_step_blocks_equal_uncached(lib, small, cache, dtype):
    from llada_amd import generate
    ocfg, W = small
    model = build(ocfg, W)
    prompt = torch.from_numpy(np.random.Generator(np.random.PCG64(8)).integers(0, MASK_ID, size=(2, 9), dtype=np.int64))
    a = generate(model, prompt, steps=4, gen_length=32, block_length=8, mask_id=MASK_ID)
    assert torch.equal(a, generate(model, prompt, steps=4, gen_length=32, block_length=8, mask_id=MASK_ID, cache=cache, kv_dtype=dtype))


@pytest.mark.parametrize("cache,dtype", [(None, None), ("dual", None), ("dual", "e4m3"), ("prefix", "int8"), ("dual", "int8"), ("prefix", "e4m3")])
@pytest.mark.parametrize("cfg_scale", [0.0, 1.0])
def test_cached_sampled_generation_step_by_step(lib, small, cache, dtype, cfg_scale):
    """The operators together.  Every step of generate() with a cache, a temperature and a truncation: the forward calls it
    makes, made again on a second cache, give the logits (the kernels are deterministic); the oracle's draw on them names
    the candidates exactly and their softmax the confidences; the transfers are a valid top-k of those."""
    from llada_amd import generate
    ocfg, W = small
    model = build(ocfg, W)
    g = np.random.Generator(np.random.PCG64(9))
    B, P, G, bl, steps = 2, 40, 64, 32, 8
    L, V, spb = P + G, ocfg.vocab_size, 4
    prompt = g.integers(0, MASK_ID, size=(B, P), dtype=np.int64)
    am = np.ones((B, P), dtype=np.int64)
    am[1, :9] = 0
    us = [g.random((B, L)) for _ in range(steps)]
    draws, trace = iter(us), []
    T, top_k, top_p, min_p = 0.8, 60, 0.9, 0.02
    out = generate(model, torch.from_numpy(prompt), torch.from_numpy(am), steps=steps, gen_length=G, block_length=bl, temperature=T,
                   cfg_scale=cfg_scale, mask_id=MASK_ID, cache=cache, kv_dtype=dtype, top_k=top_k, top_p=top_p, min_p=min_p,
                   uniform_fn=lambda shape: torch.from_numpy(next(draws)),
                   step_callback=lambda b, s, x, x0, c: trace.append([b, s] + [t.cpu().numpy().copy() for t in (x, x0, c)]))
    assert len(trace) == steps
    nb = 2 * B if cfg_scale else B
    kv = model.kv_cache(nb, L, dtype) if cache else None
    mask = torch.from_numpy(np.concatenate([am, np.ones((B, G), np.int64)], 1)).cuda()
    mask = torch.cat([mask, mask]) if cfg_scale else mask
    x_in = np.full((B, L), MASK_ID, dtype=np.int64)
    x_in[:, :P] = prompt
    is_prompt = x_in != MASK_ID
    for step, (block, i, x_after, x0, conf) in enumerate(trace):
        bs, be = P + block * bl, P + (block + 1) * bl
        xt = torch.from_numpy(np.concatenate([x_in, np.where(is_prompt, MASK_ID, x_in)]) if cfg_scale else x_in).cuda()
        ce = be if cache == "dual" else L
        if kv is not None and i > 0:
            crows = None
            if cache == "prefix":
                crows = (torch.arange(nb, dtype=torch.int32, device="cuda")[:, None] * (ce - bs) + torch.arange(bl, dtype=torch.int32, device="cuda")).reshape(-1).contiguous()
            lg = model.forward_block(xt[:, bs:ce], mask, L, bs, kv, update_cache=False, logit_rows=crows)
        else:
            rows = (torch.arange(nb, dtype=torch.int32, device="cuda")[:, None] * L + torch.arange(bs, be, dtype=torch.int32, device="cuda")).reshape(-1).contiguous()
            lg = model.forward_rows(xt, mask, rows, kv_cache=kv)
        if cfg_scale:
            c, un = lg[:B * bl], lg[B * bl:]
            lg = un + (c - un) * (cfg_scale + 1)
        lg = lg.float().cpu().numpy().reshape(B, bl, V)
        for b in range(B):
            for j in range(L):
                if x_in[b, j] != MASK_ID or not bs <= j < be:
                    assert conf[b, j] == -np.inf and x0[b, j] == x_in[b, j]
                    continue
                t, _, _ = osm.sample(lg[b, j - bs], us[step][b, j], temperature=T, top_k=top_k, top_p=top_p, min_p=min_p)
                assert x0[b, j] == t
                want = osm.confidence(lg[b, j - bs], t, "low_confidence")
                assert ulp_distance(np.float32(conf[b, j]), np.float32(want)) <= 1
        changed = x_after != x_in
        assert np.array_equal(x_after[changed], x0[changed])
        k = osamp.get_num_transfer_tokens(x_in[:, bs:be] == MASK_ID, spb - i)[:, 0]
        for b in range(B):
            assert changed[b].sum() == k[b] and osamp.is_valid_topk(conf[b], changed[b], k[b])
        x_in = x_after
    assert np.array_equal(out.cpu().numpy(), x_in) and not (x_in == MASK_ID).any()


def test_stepper_and_the_librarys_uniforms(lib, small):
    """generate() with the library's own uniforms is reproducible, differs between seeds, and the stepper repeats it."""
    from llada_amd import generate
    from llada_amd.stepper import GenerationStepper
    ocfg, W = small
    model = build(ocfg, W)
    prompt = torch.from_numpy(np.random.Generator(np.random.PCG64(4)).integers(0, MASK_ID, size=(2, 8), dtype=np.int64)).cuda()
    kw = dict(temperature=1.2, top_p=0.95, top_k=100)
    a = generate(model, prompt, steps=8, gen_length=16, block_length=8, mask_id=MASK_ID, seed=5, **kw)
    assert torch.equal(a, generate(model, prompt, steps=8, gen_length=16, block_length=8, mask_id=MASK_ID, seed=5, **kw))
    assert not torch.equal(a, generate(model, prompt, steps=8, gen_length=16, block_length=8, mask_id=MASK_ID, seed=6, **kw))
    one = generate(model, prompt[1:], steps=8, gen_length=16, block_length=8, mask_id=MASK_ID, seed=5, row_offset=1, **kw)
    assert one.shape == (1, 24)
    st = GenerationStepper(model, prompt, gen_length=16, block_length=8, mask_id=MASK_ID, seed=5, **kw)
    for _ in range(8):
        st.step(2)
    assert torch.equal(st.x, a)


def test_truncation_off_leaves_the_gumbel_max(lib, small):
    """top_k 0, top_p 1, min_p 0 are the reference's sampler, bit for bit; temperature 0 ignores a truncation."""
    from llada_amd import generate
    ocfg, W = small
    model = build(ocfg, W)
    prompt = torch.from_numpy(np.random.Generator(np.random.PCG64(4)).integers(0, MASK_ID, size=(2, 8), dtype=np.int64))
    kw = dict(steps=8, gen_length=16, block_length=8, mask_id=MASK_ID, seed=2)
    assert torch.equal(generate(model, prompt, temperature=0.7, **kw), generate(model, prompt, temperature=0.7, top_k=0, top_p=1.0, min_p=0.0, **kw))
    assert torch.equal(generate(model, prompt, temperature=0., **kw), generate(model, prompt, temperature=0., top_k=3, top_p=0.5, **kw))
    assert torch.equal(generate(model, prompt, temperature=0., **kw), generate(model, prompt, temperature=0.9, top_k=1, **kw))


def test_refusals(lib, small):
    from llada_amd import generate
    ocfg, W = small
    model = build(ocfg, W)
    prompt = torch.zeros((1, 4), dtype=torch.long)
    kw = dict(steps=4, gen_length=4, block_length=4, mask_id=MASK_ID)
    for bad in (dict(kv_dtype="e4m3"), dict(kv_dtype="fp4", cache="dual"), dict(temperature=1.0, top_k=5, noise_fn=lambda s: torch.rand(s))):
        with pytest.raises(NotImplementedError):
            generate(model, prompt, **kw, **bad)
    for bad in (dict(temperature=1.0, top_p=-0.5), dict(temperature=1.0, min_p=1.5), dict(temperature=-1.0, top_k=4)):
        with pytest.raises(AssertionError):
            generate(model, prompt, **kw, **bad)
