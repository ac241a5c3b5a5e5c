"""Truncated sampling on an MI355X against the float64 restatement (oracle/sampling.py): tokens exactly, probabilities to
float32 rounding (2^-24) plus the float64 sums' noise."""
import ctypes as C

import numpy as np
import pytest

from oracle import rng as orng
from oracle import sampling as osm

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(params=["whole", "half"])
def lib(lib, request):
    """Every test of this file with both kinds of workgroup."""
    lib.llada_sample_rows_force(1 if request.param == "whole" else 2)
    yield lib
    lib.llada_sample_rows_force(0)


def bf16(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).cuda().to(torch.bfloat16)


def check(lg, u, probs=True, **kw):
    from llada_amd import sample_tokens
    tok, pr = sample_tokens(lg, uniforms=torch.from_numpy(u).cuda(), return_probs=True, **kw)
    rows = lg.float().cpu().numpy()
    per = {k: (v.float().cpu().numpy().astype(np.float64) if isinstance(v, torch.Tensor) else None) for k, v in kw.items()}
    tok, pr = tok.cpu().numpy(), pr.double().cpu().numpy()
    for r in range(rows.shape[0]):
        p = {k: (v if per[k] is None else (int(per[k][r]) if k == "top_k" else float(per[k][r]))) for k, v in kw.items()}
        t, q, n = osm.sample(rows[r], u[r], **p)
        assert tok[r] == t, (r, tok[r], t, p, u[r], n)
        assert abs(pr[r] - q) <= 2.0 ** -23 * q + 1e-30, (r, pr[r], q)
    return tok


def logits(seed, n, V, scale=2.2):
    g = np.random.Generator(np.random.PCG64(seed))
    x = g.standard_normal((n, V)).astype(np.float32) * scale
    x += np.where(g.random((n, V)) < 200.0 / V, 4 + 4 * g.random((n, V)), 0).astype(np.float32)
    return bf16(x)


def uniforms(seed, n):
    u = np.random.Generator(np.random.PCG64(seed + 500)).random(n)
    u[0] = 0.0
    if n > 2:
        u[1], u[2] = 1.0 - 2.0 ** -53, 1e-9
    return u


@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 40, 513, 4096, 50257, 126464, 131072])
@pytest.mark.parametrize("kw", [dict(), dict(temperature=0.0), dict(temperature=0.3, top_k=5), dict(temperature=1.7, top_p=0.9),
                                dict(temperature=0.8, min_p=0.05), dict(top_k=50, top_p=0.8, min_p=0.01), dict(top_k=1), dict(top_p=1e-9),
                                dict(min_p=1.0), dict(temperature=1e6, top_p=0.999, top_k=10 ** 9), dict(temperature=1e-6)])
def test_tokens_match_the_sorted_definition(lib, V, kw):
    n = 6
    if V == 131072:
        n = 3
    check(logits(V, n, V), uniforms(V, n), **kw)


@pytest.mark.parametrize("V", [50, 1000, 126464])
def test_ties_go_to_the_lowest_index(lib, V):
    """Few distinct values: groups of thousands of equal entries, cut in their middle."""
    g = np.random.Generator(np.random.PCG64(V))
    x = bf16(g.integers(0, 4, size=(8, V)).astype(np.float32))
    for kw in (dict(), dict(top_k=V // 3), dict(top_p=0.37), dict(top_k=V // 5, top_p=0.9), dict(min_p=0.2), dict(temperature=0.0)):
        check(x, uniforms(V, 8), **kw)
    same = bf16(np.full((3, V), 1.5))
    tok = check(same, np.array([0.0, 0.5, 1.0 - 2.0 ** -53]))
    assert tok[0] == 0 and tok[1] == V // 2 and tok[2] == V - 1
    check(same, np.array([0.0, 0.5, 1.0 - 2.0 ** -53]), top_k=V // 2 + 1)


def test_rows_with_infinities_nan_and_odd_values(lib):
    V = 3000
    g = np.random.Generator(np.random.PCG64(1))
    x = g.standard_normal((14, V)).astype(np.float32) * 3
    x[0, 5:2000] = -np.inf                     # most of the row masked
    x[1, :] = -np.inf                          # all of it
    x[2, :] = -np.inf
    x[2, 77] = -3.0
    x[3, [4, 9]] = np.nan
    x[4, [100, 200, 300]] = np.inf
    x[5] *= 1e4                                # beyond 2^9
    x[6] *= 1e-25                              # below 2^-55
    x[7, ::2] = 0.0
    x[7, 1::4] = -0.0                          # equal to +0
    x[8] = np.where(g.random(V) < 0.5, 3.0e38, -3.0e38)
    x[9] = np.nan
    x[10, ::3] = 1e-30                         # zeros, tiny and ordinary values in one row
    x[10, 1::3] = 0.0
    x[10, 2::3] = -1e-30
    x[11, 17] = 600.0
    x[12] = -np.abs(x[12]) * 1e3               # negative only, beyond the range
    x[13, :] = np.where(np.arange(V) % 2 == 0, np.inf, -np.inf)
    xb = bf16(x)
    for s in range(4):
        u = np.random.Generator(np.random.PCG64(s)).random(14)
        for kw in (dict(), dict(temperature=0.0), dict(top_k=7), dict(top_p=0.6, temperature=2.0), dict(min_p=0.1), dict(top_k=1000, top_p=0.9, min_p=0.001),
                   dict(temperature=1e4, min_p=0.999), dict(temperature=1e20, min_p=1.0)):
            check(xb, u, **kw)


def test_random_bit_patterns(lib):
    """Every bf16 pattern at once: the whole key space is occupied."""
    g = np.random.Generator(np.random.PCG64(9))
    bits = torch.from_numpy(g.integers(0, 65536, size=(4, 70000)).astype(np.int32)).to(torch.int16).cuda().view(torch.bfloat16)
    for kw in (dict(temperature=1e30), dict(temperature=1e30, top_k=30000), dict(temperature=1e30, top_p=0.5), dict()):
        check(bits, uniforms(3, 4), **kw)


@pytest.mark.parametrize("V,stride,shift", [(1000, 1003, 0), (999, 999, 1), (1001, 1016, 3), (126464, 126464, 4), (5, 9, 7)])
def test_strides_and_alignment(lib, V, stride, shift):
    n = 5
    buf = torch.full((n * stride + 16,), 50.0, dtype=torch.bfloat16, device="cuda")     # what lies between the rows must not be drawn
    view = buf[shift:shift + n * stride].view(n, stride)[:, :V]
    view.copy_(logits(V + shift, n, V))
    check(view, uniforms(V, n), top_p=0.9)
    check(view, uniforms(V + 1, n))


def test_parameters_per_row(lib):
    n, V = 8, 2000
    t = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 0.25, 1.0, 1.0])
    k = torch.tensor([0, 3, 0, 100, 1, 0, 50, 0])
    p = torch.tensor([1.0, 1.0, 0.5, 0.75, 1.0, 0.875, 1.0, 0.25])
    q = torch.tensor([0.0, 0.0, 0.0, 0.0, 0.5, 0.0, 0.125, 0.0])
    check(logits(2, n, V), uniforms(4, n), temperature=t.cuda(), top_k=k.cuda(), top_p=p.cuda(), min_p=q.cuda())
    check(logits(3, n, V), uniforms(5, n), temperature=0.75, top_k=k.cuda(), top_p=0.75, min_p=0.0)


def test_guidance_matches_combining_first(lib):
    from llada_amd import sample_tokens
    for V, cut in ((126464, 126464), (777, 777), (1000, 995)):
        a, b = logits(V, 6, V)[:, :cut], logits(V + 1, 6, V)[:, :cut]
        scale = 1.5
        both = b + (a - b) * (scale + 1)
        u = torch.from_numpy(uniforms(V, 6)).cuda()
        got = sample_tokens(a, 0.9, top_p=0.95, uniforms=u, uncond_logits=b, cfg_scale=scale)
        assert torch.equal(got, sample_tokens(both, 0.9, top_p=0.95, uniforms=u))


def test_shapes_streams_and_the_librarys_uniforms(lib):
    from llada_amd import sample_tokens
    x = logits(6, 6, 333)
    u = torch.from_numpy(uniforms(6, 6)).cuda()
    flat = sample_tokens(x, uniforms=u)
    assert torch.equal(sample_tokens(x.view(2, 3, 333), uniforms=u.view(2, 3)), flat.view(2, 3))
    assert sample_tokens(x[0], uniforms=u[0]).shape == () and sample_tokens(x[:0]).shape == (0,)
    assert torch.equal(sample_tokens(x[2].expand(4, 333), uniforms=u[2].expand(4)), flat[2].expand(4))
    a = sample_tokens(x, seed=5, step=3, row_offset=2)
    want = np.array([_philox_uniform(5, 3, 2 + r, 0) for r in range(6)])
    assert torch.equal(a, sample_tokens(x, uniforms=torch.from_numpy(want).cuda()))
    for bad in (lambda: sample_tokens(x.float()), lambda: sample_tokens(x, uniforms=u[:3]), lambda: sample_tokens(x, top_k=torch.ones(5)),
                lambda: sample_tokens(x, uncond_logits=x[:3])):
        with pytest.raises(ValueError):
            bad()
    for bad in (dict(top_p=0.0), dict(top_k=-1), dict(min_p=2.0), dict(temperature=-1.0)):
        with pytest.raises(AssertionError):
            sample_tokens(x, **bad)


def _philox_uniform(seed, step, row, col):
    o = orng.philox4x32(0, col, row, step, seed & 0xFFFFFFFF, (seed >> 32) ^ 4)
    return (float(int(o[0]) >> 5) * 67108864.0 + float(int(o[1]) >> 6)) / 9007199254740992.0


@pytest.mark.parametrize("rule", ["low_confidence", "high_confidence", "low_entropy", "high_entropy", "random"])
@pytest.mark.parametrize("flags", [0, 1, 2, 3])
def test_epilogue(lib, rule, flags):
    """llada_remask_scores_sampled: the drawn token at every active position, the rule's confidence (bf16, within one
    step of float64: one rounding of the value, float32 noise at a border), the defaults everywhere else."""
    from llada_amd import _lib
    from oracle.bf16 import ulp_distance
    B, L, V, mask_id, eos, eot, be = 2, 6, 4000, 3999, 17, 29, 5
    g = np.random.Generator(np.random.PCG64(flags + 1))
    lg = logits(11, B * L, V)
    lg[:, eos] += 6
    lg[:, eot] += 6
    x = torch.full((B, L), mask_id, dtype=torch.long, device="cuda")
    x[0, 1], x[1, 0] = 5, 6
    u = torch.from_numpy(g.random((B, L))).cuda()
    rs = torch.from_numpy(g.random((B, L)).astype(np.float32)).cuda()
    x0, conf = torch.empty_like(x), torch.empty((B, L), dtype=torch.float32, device="cuda")
    sp = _lib.Sampling(0.9, 0.9, 0.0, 40, None, None, None, None, u.data_ptr())
    a = _lib.RemaskArgs(lg.data_ptr(), None, 0.0, None, B * L, V, x.data_ptr(), B, L, be, mask_id, _lib.REMASK[rule], flags, eos, eot,
                        0.0, None, rs.data_ptr(), 0, 0, 0, x0.data_ptr(), conf.data_ptr(), None, 0)
    _lib.check(lib.llada_remask_scores_sampled(C.byref(a), C.byref(sp), _lib.stream_ptr()))
    torch.cuda.synchronize()
    rows = lg.float().cpu().numpy()
    for b in range(B):
        for c in range(L):
            got, cf = int(x0[b, c]), float(conf[b, c])
            if int(x[b, c]) != mask_id or c >= be:
                assert got == int(x[b, c]) and cf == -np.inf
                continue
            row = rows[b * L + c].copy()
            if flags & 1:
                row[eos] = -np.inf
            t, _, _ = osm.sample(row, float(u[b, c]), temperature=0.9, top_k=40, top_p=0.9)
            assert got == t
            if rule == "random":
                assert cf == float(rs[b, c])
                continue
            want = osm.confidence(row, t, rule, eot if flags & 2 else -1)
            if "entropy" in rule:      # the reference rounds log p, p, each product and the sum to bf16: 3 * 2^-8 a term, 2^-8 the sum
                assert abs(cf - want) <= 4 * 2.0 ** -8 * abs(want), (cf, want)
            else:
                assert ulp_distance(np.float32(cf), np.float32(want)) <= 1 or abs(cf - want) <= 2.0 ** -8 * max(want, 2.0 ** -7), (cf, want)


def test_replayed_graph(lib):
    from llada_amd import sample_tokens
    x, u = logits(70, 40, 8000), torch.from_numpy(uniforms(70, 40)).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        sample_tokens(x, 0.8, top_p=0.9, uniforms=u)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            tok = sample_tokens(x, 0.8, top_p=0.9, uniforms=u)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(4):
        x.copy_(logits(71 + i, 40, 8000))
        u.copy_(torch.from_numpy(uniforms(71 + i, 40)))
        g.replay()
        want = sample_tokens(x, 0.8, top_p=0.9, uniforms=u)
        torch.cuda.synchronize()
        assert torch.equal(tok, want)


def test_offsets_past_32_bits(lib):
    """More than 2^31 logits: the last rows' tokens are those of a call on them alone."""
    from llada_amd import sample_tokens
    n, V = 17100, 126464
    x = torch.zeros((n, V), dtype=torch.bfloat16, device="cuda")
    assert x.numel() > 2 ** 31
    x[-5:] = logits(90, 5, V)
    x[7] = x[-1]
    u = torch.rand(n, dtype=torch.float64, device="cuda")
    tok = sample_tokens(x, 0.9, top_p=0.95, uniforms=u)
    assert torch.equal(tok[-5:], sample_tokens(x[-5:].clone(), 0.9, top_p=0.95, uniforms=u[-5:]))
    keep = int(np.ceil(0.95 * V))                       # a row of zeros: the u-th of its first 95 %, in index order
    assert torch.equal(tok[100:-5], (u[100:-5] * keep).to(torch.int64))


def test_uniforms_outside_their_range_stay_inside_the_row(lib):
    from llada_amd import sample_tokens
    x = logits(91, 6, 700)
    u = torch.tensor([-1.0, 1.0, 2.0, float("nan"), float("inf"), -float("inf")], dtype=torch.float64, device="cuda")
    for kw in (dict(), dict(top_k=5), dict(top_p=0.5), dict(min_p=0.3), dict(temperature=0.0)):
        t = sample_tokens(x, uniforms=u, **kw)
        assert ((t >= 0) & (t < 700)).all()


def test_parameter_arrays_outside_their_ranges_act_like_the_nearest_end(lib):
    from llada_amd import sample_tokens
    x, u = logits(92, 4, 900), torch.from_numpy(uniforms(92, 4)).cuda()
    base = sample_tokens(x, uniforms=u)
    dev = dict(device="cuda")
    assert torch.equal(base, sample_tokens(x, uniforms=u, top_p=torch.tensor([1.5, 2.0, float("nan"), 1.0], **dev)))
    assert torch.equal(base, sample_tokens(x, uniforms=u, top_k=torch.tensor([0, -5, -1, 2 ** 31 - 1], **dev)))
    assert torch.equal(base, sample_tokens(x, uniforms=u, min_p=torch.tensor([0.0, -1.0, float("nan"), -0.5], **dev)))
    first = x.float().argmax(dim=1)
    for k in (dict(top_p=torch.full((4,), -0.5, **dev)), dict(min_p=torch.full((4,), 7.0, **dev)), dict(temperature=torch.tensor([0.0, -1.0, float("nan"), 0.0], **dev))):
        assert torch.equal(first, sample_tokens(x, uniforms=u, **k))


def test_top_k_past_32_bits_keeps_the_row(lib):
    from llada_amd import sample_tokens
    x, u = logits(90, 6, 1000), torch.from_numpy(uniforms(90, 6)).cuda()
    want = sample_tokens(x, uniforms=u)
    assert torch.equal(sample_tokens(x, top_k=2 ** 32 + 1, uniforms=u), want)
    assert torch.equal(sample_tokens(x, top_k=torch.full((6,), 2 ** 32 + 1, device="cuda"), uniforms=u), want)
    with pytest.raises(AssertionError):
        sample_tokens(x, top_k=5 - 2 ** 32, uniforms=u)


@pytest.mark.parametrize("n,V", [(259, 126464), (1029, 9000)])
def test_the_rule_picks_a_kind_that_gives_the_same(lib, n, V):
    from llada_amd import sample_tokens
    x, u = logits(95, n, V), uniforms(95, n)
    forced = [t.clone() for t in sample_tokens(x, 0.9, 40, 0.9, 0.01, uniforms=torch.from_numpy(u).cuda(), return_probs=True)]
    lib.llada_sample_rows_force(0)
    for k in (n, n - 5):
        tok, pr = sample_tokens(x[:k], 0.9, 40, 0.9, 0.01, uniforms=torch.from_numpy(u[:k]).cuda(), return_probs=True)
        assert torch.equal(tok, forced[0][:k]) and torch.equal(pr, forced[1][:k])
    check(x[:12], u[:12], temperature=0.9, top_k=40, top_p=0.9, min_p=0.01)


def test_ties_and_the_last_entry_of_a_long_row(lib):
    # the drawn entry in each chunk of the row, among few equal ones and among very many
    V = 131072
    places = list(range(0, V, 4099)) + [V - 1]
    x = torch.full((len(places), V), -3.0)
    for r, at in enumerate(places):
        x[r, at] = 8.0
    from llada_amd import sample_tokens
    tok = sample_tokens(x.cuda().to(torch.bfloat16), top_k=1)
    assert tok.tolist() == places
    flat = torch.full((len(places), V), 0.5).cuda().to(torch.bfloat16)
    u = (np.array(places) + 0.5) / V
    assert sample_tokens(flat, uniforms=torch.from_numpy(u).cuda()).tolist() == places


@pytest.mark.parametrize("V", [65528, 65529, 65530, 65536, 65543])
@pytest.mark.parametrize("shift", [0, 5])
def test_around_the_length_that_half_a_row_holds(lib, V, shift):
    from llada_amd import sample_tokens
    n = 4
    flat = torch.full((n * (V + 8) + 8,), 9.0).cuda().to(torch.bfloat16)      # what stands between the rows would win
    x = flat.as_strided((n, V), (V + 8, 1), shift)
    x.copy_(logits(V, n, V))
    x[1, V - 1] = 30.0
    u = uniforms(V, n)
    tok = check(x, u, top_p=0.97)
    assert tok[1] == V - 1
    un = flat.clone().as_strided((n, V), (V + 8, 1), shift)
    un.copy_(logits(V + 1, n, V))
    both = sample_tokens(x, 0.8, top_k=30, uniforms=torch.from_numpy(u).cuda(), uncond_logits=un, cfg_scale=1.5)
    d = ((x.float() - un.float()).to(torch.bfloat16).float() * 2.5).to(torch.bfloat16)
    first = (un.float() + d.float()).to(torch.bfloat16)
    assert torch.equal(both, sample_tokens(first, 0.8, top_k=30, uniforms=torch.from_numpy(u).cuda()))


@pytest.mark.parametrize("dtype", ["int8", "uint8", "int16", "int32", "float16"])
def test_top_k_arrays_of_narrow_types(lib, dtype):
    from llada_amd import sample_tokens
    x, u = logits(93, 4, 900), torch.from_numpy(uniforms(93, 4)).cuda()
    k = torch.tensor([0, 1, 100, 127], device="cuda")
    assert torch.equal(sample_tokens(x, top_k=k.to(getattr(torch, dtype)), uniforms=u), sample_tokens(x, top_k=k, uniforms=u))


def test_temperature_arrays_past_the_range(lib):
    """An infinite temperature acts like 1e30: equal weights for all finite entries, none but the largest past min_p = 1."""
    from llada_amd import sample_tokens
    x, u = logits(94, 4, 900), torch.from_numpy(uniforms(94, 4)).cuda()
    t = torch.tensor([float("inf"), 3e38, 1e30, float("inf")], device="cuda")
    for kw in (dict(min_p=1.0), dict(min_p=0.5), dict(top_k=5), dict(top_p=0.5), dict()):
        assert torch.equal(sample_tokens(x, t, uniforms=u, **kw), sample_tokens(x, 1e30, uniforms=u, **kw)), kw
    assert torch.equal(sample_tokens(x, t, min_p=1.0, uniforms=u), x.float().argmax(dim=1))


def test_more_rows_than_one_launch_takes(lib):
    """2^32 threads are a launch's limit; the library's uniforms, given ones and parameter arrays keep their rows."""
    from llada_amd import sample_tokens
    n, V = 2 ** 22 + 5, 8
    x = torch.randn((n, V), device="cuda").to(torch.bfloat16)
    t = torch.linspace(0.2, 2.0, n, device="cuda")
    k = (torch.arange(n, device="cuda") % 9).to(torch.int32)
    u = torch.rand(n, dtype=torch.float64, device="cuda")
    p, q = torch.full((n,), 0.9, device="cuda"), torch.full((n,), 0.01, device="cuda")
    tok, pr = sample_tokens(x, t, k, p, q, seed=3, row_offset=7, return_probs=True)
    given = sample_tokens(x, t, k, uniforms=u)
    for a, b in ((0, 9), (2 ** 21 - 4, 2 ** 21 + 4), (2 ** 22 - 4, n)):
        w, v = sample_tokens(x[a:b], t[a:b], k[a:b], p[a:b], q[a:b], seed=3, row_offset=7 + a, return_probs=True)
        assert torch.equal(tok[a:b], w) and torch.equal(pr[a:b], v)
        assert torch.equal(given[a:b], sample_tokens(x[a:b], t[a:b], k[a:b], uniforms=u[a:b]))
    with pytest.raises(ValueError, match="32 bits"):
        sample_tokens(x[:1, :1].expand(2 ** 32 + 2, 1))
