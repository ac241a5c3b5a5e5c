"""The remasking epilogue with truncated draws (llada_remask_scores_sampled) against llada_remask_scores and the float64
restatement: every remasking rule and flag, rows a forward has broken, the framework's own vocabulary."""
import ctypes as C

import numpy as np
import pytest

from oracle import sampling as osm
from oracle.bf16 import ulp_distance

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

RULES = ["low_confidence", "high_confidence", "low_entropy", "high_entropy", "random"]
VOCAB, EOS, EOT, MASK = 126464, 126081, 126348, 126336


@pytest.fixture(params=["whole", "half"])
def kind(lib, request):
    lib.llada_sample_rows_force(1 if request.param == "whole" else 2)
    yield lib
    lib.llada_sample_rows_force(0)


def logits(seed, n, V, scale=2.2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((n, V), generator=g, device="cuda") * scale
    likely = torch.rand((n, V), generator=g, device="cuda") * (V / 200.0)
    return (x + torch.where(likely < 1, 4 + 4 * likely, torch.zeros_like(x))).to(torch.bfloat16)


def epilogue(lib, lg, x, be, mask_id, rule, flags, eos, eot, u=None, rs=None, un=None, cfg=0.0, row_pos=None, T=0.9, top_k=0, top_p=1.0,
             min_p=0.0, arrays=(None,) * 4, plain=False):
    """(candidates, confidences) of llada_remask_scores_sampled, or of llada_remask_scores at temperature 0 (`plain`)."""
    from llada_amd import _lib
    B, L = x.shape
    x0, conf = torch.full_like(x, -7), torch.full((B, L), 9.0, dtype=torch.float32, device="cuda")
    ws = torch.empty(lib.llada_rows_workspace_bytes(lg.shape[0]), dtype=torch.uint8, device="cuda") if plain else None
    a = _lib.RemaskArgs(lg.data_ptr(), _lib.ptr(un), cfg, _lib.ptr(row_pos), lg.shape[0], lg.shape[1], x.data_ptr(), B, L, be, mask_id,
                        _lib.REMASK[rule], flags, eos, eot, 0.0, None, _lib.ptr(rs), 0, 0, 0, x0.data_ptr(), conf.data_ptr(), _lib.ptr(ws),
                        0 if ws is None else ws.numel())
    if plain:
        _lib.check(lib.llada_remask_scores(C.byref(a), _lib.stream_ptr()))
    else:
        sp = _lib.Sampling(T, top_p, min_p, top_k, *(_lib.ptr(t) for t in arrays), _lib.ptr(u))
        _lib.check(lib.llada_remask_scores_sampled(C.byref(a), C.byref(sp), _lib.stream_ptr()))
    torch.cuda.synchronize()
    return x0.cpu().numpy(), conf.cpu().numpy()


def close(cf, want, rule, f32=False):
    """Low confidence: one rounding to bf16, float32 noise at its border (one step), or to float32 (2^-24).  High confidence: p
    rounded, then 1 - p: 2^-8 together (2^-23).  Entropies: log p, p, each product and the sum rounded to bf16, 2^-8 each, and what
    float32 flushes."""
    if np.isnan(want) or np.isnan(cf):
        return bool(np.isnan(want) and np.isnan(cf))
    if "entropy" in rule:
        return abs(cf - want) <= 4 * 2.0 ** -8 * abs(want) + 1e-30
    if rule == "high_confidence":
        return abs(cf - want) <= (2.0 ** -23 if f32 else 2.0 ** -8 + 2.0 ** -15)
    return abs(cf - want) <= 2.0 ** -23 * want if f32 else ulp_distance(np.float32(cf), np.float32(want)) <= 1


def check_rows(lg, x, be, mask_id, rule, flags, eos, eot, u, got, rows=None, pos=None, params=None, broken=()):
    """Every (or the listed) logits row's candidate and confidence against the float64 restatement, the defaults elsewhere."""
    x0, conf = got
    B, L = x.shape
    xs = x.cpu().numpy()
    seen = np.zeros((B, L), bool)
    for r in range(lg.shape[0]):
        b, c = divmod(r if pos is None else int(pos[r]), L)
        if xs[b, c] != mask_id or c >= be:
            continue
        seen[b, c] = True
        if rows is not None and r not in rows:
            continue
        row = lg[r].float().cpu().numpy()
        if flags & 1:
            row[eos] = -np.inf
        t, _, _ = osm.sample(row, float(u[b, c]), **params(b))
        assert x0[b, c] == t, (r, x0[b, c], t)
        if rule == "random":
            continue
        if flags & 2 and params(b)["temperature"] == 0:     # there EOS leaves the softmax too (generate.py:100-101)
            row[eos] = -np.inf
        want = np.nan if r in broken else osm.confidence(row, t, rule, eot if flags & 2 else -1)
        assert close(float(conf[b, c]), want, rule, bool(flags & 4)), (r, float(conf[b, c]), want)
    assert (x0[~seen] == xs[~seen]).all() and (conf[~seen] == -np.inf).all()


@pytest.mark.parametrize("rule,flags", [(r, f) for r in RULES for f in (0, 1, 2, 3, 4, 6) if not ("entropy" in r and f & 3)])
def test_temperature_zero_is_the_plain_epilogue(kind, rule, flags):
    """The arg-max through the sampled form (as a scalar and as a row's own temperature) gives llada_remask_scores' candidates
    and confidences, EOS or EOT in the lead included.  (The entropy rules: where no entry is -inf; there the plain form's
    0 * log 0 is NaN.)  Float32 forms differ by the sums' rounding: 2^-15; bf16 ones by one step."""
    V, L, eos, eot = 4000, 16, 17, 29
    lg = logits(flags + 3, L, V)
    lg[1, eos], lg[2, eot], lg[3, eos] = 60.0, 61.0, 62.0
    lg[3, eot] = 61.5
    lg[4, eos] = lg[4].max()
    lg[5, 33] = 250.0
    x = torch.full((1, L), 3999, dtype=torch.long, device="cuda")
    rs = torch.rand((1, L), device="cuda")
    want = epilogue(kind, lg, x, L, 3999, rule, flags, eos, eot, rs=rs, plain=True)
    for k in (dict(T=0.0), dict(arrays=(torch.zeros(1, device="cuda"), None, None, None))):
        got = epilogue(kind, lg, x, L, 3999, rule, flags, eos, eot, rs=rs, **k)
        assert (got[0] == want[0]).all()
        for a, w in zip(got[1][0].astype(np.float64), want[1][0].astype(np.float64)):
            if rule == "random":
                assert a == w
            elif flags & 4 and "entropy" not in rule:
                assert abs(a - w) <= 2.0 ** -15 * max(w, 1 - w) + 1e-30, (a, w)
            else:       # an entropy: three roundings a term and one of the sum, each at most a step apart
                assert abs(a - w) <= 4 * 2.0 ** -7 * abs(w) + 1e-30 if "entropy" in rule else close(a, w, rule), (a, w)


@pytest.mark.parametrize("rule", RULES)
@pytest.mark.parametrize("T", [0.0, 0.9])
def test_rows_that_a_forward_broke(kind, rule, T):
    """A softmax over a NaN, an infinity or nothing at all is NaN: so is the confidence, which the transfer then ranks
    first, as after llada_remask_scores; the candidate is still the definition's.  A NaN in the entry that the softmax
    does not see changes nothing."""
    V, L, eos, eot = 2000, 9, 17, 29
    lg = logits(5, L, V)
    lg[1, 700] = float("nan")
    lg[2] = -float("inf")
    lg[3] = float("nan")
    lg[4, [5, 1999]] = float("inf")
    lg[5, eot] = float("nan")
    lg[6] = -float("inf")
    lg[6, eot] = 1.0
    lg[7, 3:] = -float("inf")
    lg[8, 1999] = -float("nan")
    x = torch.full((1, L), 1999, dtype=torch.long, device="cuda")
    u = torch.rand((1, L), dtype=torch.float64, device="cuda")
    rs = torch.rand((1, L), device="cuda")
    got = epilogue(kind, lg, x, L, 1999, rule, 2, eos, eot, u=u, rs=rs, T=T)
    check_rows(lg, x, L, 1999, rule, 2, eos, eot, u, got, params=lambda b: dict(temperature=T), broken=(1, 2, 3, 4, 6, 8))
    if rule == "random":
        assert (got[1] == rs.cpu().numpy()).all()
    elif T == 0.0 and "entropy" not in rule:
        want = epilogue(kind, lg, x, L, 1999, rule, 2, eos, eot, rs=rs, plain=True)
        assert (got[0] == want[0]).all() and (np.isnan(got[1]) == np.isnan(want[1])).all()


@pytest.mark.parametrize("rule", RULES[:4])
@pytest.mark.parametrize("lead", [100.0, 900.0, 5000.0])
def test_an_unseen_entry_far_above_the_rest(kind, rule, lead):
    """EOT can be drawn although the confidence's softmax does not see it; that softmax has a maximum of its own."""
    V, L, eos, eot = 3000, 6, 17, 29
    lg = logits(8, L, V)
    lg[:, eot] = lead
    lg[3:, 40] = lead                                       # an equal entry that is seen
    x = torch.full((1, L), 2999, dtype=torch.long, device="cuda")
    u = torch.tensor([[0.1, 0.5, 0.999, 0.1, 0.6, 0.999]], dtype=torch.float64, device="cuda")
    for T in (1e4, 1.0):
        got = epilogue(kind, lg, x, L, 2999, rule, 2, eos, eot, u=u, T=T)
        check_rows(lg, x, L, 2999, rule, 2, eos, eot, u, got, params=lambda b: dict(temperature=T))


def full_rows(seed, n):
    """Rows of the framework's vocabulary, some with what the second half's bookkeeping has to get right."""
    lg = logits(seed, n, VOCAB)
    lg[0, EOS] = 40.0                                       # EOS leads: taken out of the draw, or drawn
    lg[1, EOT] = 40.0
    lg[2, 100000] = 40.0                                    # a single entry of the second half
    lg[3, 70000:126400:7] = 30.0                            # equal entries of the second half
    lg[4, 3:126400:5] = 30.0                                # of both halves
    lg[5, -1] = 40.0
    lg[6, EOS - 1], lg[6, EOS + 1] = 40.0, 40.0             # the neighbours of the entry that is taken out
    lg[7, ::2], lg[7, 1::2] = 0.0, -0.0
    lg[8] = -float("inf")
    lg[8, [9, EOS, 126000]] = 2.0
    lg[9, 65536 + 5] = 1e-30                                # magnitudes without a bin of their own
    lg[10, EOS - 3] = 300.0
    lg[11, 40] = -1e4
    lg[11, EOS] = 20.0
    return lg


@pytest.mark.parametrize("rule,flags", [("low_confidence", 0), ("low_confidence", 1), ("high_confidence", 3), ("low_entropy", 3), ("high_entropy", 2),
                                        ("low_confidence", 7), ("random", 1)])
def test_the_frameworks_vocabulary(kind, rule, flags):
    lg = full_rows(1, 24)
    x = torch.full((2, 12), MASK, dtype=torch.long, device="cuda")
    g = np.random.Generator(np.random.PCG64(flags))
    u = torch.from_numpy(g.random((2, 12))).cuda()
    rs = torch.rand((2, 12), device="cuda")
    for kw in (dict(temperature=0.9, top_p=0.95), dict(temperature=1.3), dict(temperature=0.7, top_k=30, min_p=0.02)):
        got = epilogue(kind, lg, x, 12, MASK, rule, flags, EOS, EOT, u=u, rs=rs, T=kw["temperature"], top_k=kw.get("top_k", 0), top_p=kw.get("top_p", 1.0),
                       min_p=kw.get("min_p", 0.0))
        check_rows(lg, x, 12, MASK, rule, flags, EOS, EOT, u, got, params=lambda b: kw)
        if rule == "random":
            assert (got[1] == rs.cpu().numpy()).all()


@pytest.mark.parametrize("rule,flags", [("low_confidence", 1), ("low_entropy", 3)])
def test_more_rows_than_units_at_given_positions(lib, rule, flags):
    """528 rows in a shuffled order of positions, with no kind forced: the form that keeps half a row and streams the rest."""
    n, L, be = 528, 40, 33
    lg = full_rows(2, n)
    x = torch.full((16, L), MASK, dtype=torch.long, device="cuda")
    g = np.random.Generator(np.random.PCG64(3))
    pos = np.concatenate([b * L + np.arange(33) for b in range(16)])
    g.shuffle(pos)
    x.view(-1)[torch.from_numpy(pos[20:30]).cuda()] = 5     # rows whose position has been decided
    u = torch.from_numpy(g.random((16, L))).cuda()
    got = epilogue(lib, lg, x, be, MASK, rule, flags, EOS, EOT, u=u, row_pos=torch.from_numpy(pos.astype(np.int32)).cuda(), top_p=0.97)
    check_rows(lg, x, be, MASK, rule, flags, EOS, EOT, u, got, rows=set(range(12)) | set(range(30, n, 13)), pos=pos,
               params=lambda b: dict(temperature=0.9, top_p=0.97))


def test_guided_rows_of_the_frameworks_vocabulary(lib):
    lg, un = logits(21, 16, VOCAB), logits(22, 16, VOCAB)
    lg[0, EOS], lg[1, 100000], lg[2, EOS - 1] = 40.0, 40.0, 300.0
    both = un + (lg - un) * 2.5                             # (bf16 after each operation)
    x = torch.full((2, 8), MASK, dtype=torch.long, device="cuda")
    u = torch.rand((2, 8), dtype=torch.float64, device="cuda")
    for rule, flags in (("low_confidence", 1), ("low_entropy", 2), ("high_confidence", 3)):
        got = epilogue(lib, lg, x, 8, MASK, rule, flags, EOS, EOT, u=u, un=un, cfg=1.5, top_p=0.9)
        check_rows(both, x, 8, MASK, rule, flags, EOS, EOT, u, got, params=lambda b: dict(temperature=0.9, top_p=0.9))


def test_parameters_of_each_sequence(kind):
    V, B, L = 5000, 4, 5
    lg = logits(31, B * L, V)
    t = torch.tensor([0.0, 0.5, 1.0, 2.0], device="cuda")
    k = torch.tensor([0, 7, 0, 300], dtype=torch.int32, device="cuda")
    p = torch.tensor([1.0, 1.0, 0.5, 0.875], device="cuda")
    q = torch.tensor([0.0, 0.125, 0.0, 0.0], device="cuda")
    x = torch.full((B, L), V - 1, dtype=torch.long, device="cuda")
    u = torch.rand((B, L), dtype=torch.float64, device="cuda")
    got = epilogue(kind, lg, x, L, V - 1, "low_confidence", 0, 17, 29, u=u, arrays=(t, k, p, q))
    check_rows(lg, x, L, V - 1, "low_confidence", 0, 17, 29, u, got,
               params=lambda b: dict(temperature=float(t[b]), top_k=int(k[b]), top_p=float(p[b]), min_p=float(q[b])))


@pytest.mark.parametrize("rule", RULES)
def test_a_row_of_nan_under_gumbel_noise(lib, rule):
    """llada_remask_scores with a temperature on rows where no score compares: token 0, and NaN for its confidence."""
    from llada_amd import _lib
    V, L = 4096, 6
    lg = logits(41, L, V)
    lg[1] = float("nan")
    lg[4] = -float("nan")
    x = torch.full((1, L), V - 1, dtype=torch.long, device="cuda")
    rs = torch.rand((1, L), device="cuda")
    for scratch in (True, False):
        x0, conf = torch.full_like(x, -7), torch.full((1, L), 9.0, device="cuda")
        ws = torch.empty(lib.llada_rows_workspace_bytes(L), dtype=torch.uint8, device="cuda")
        a = _lib.RemaskArgs(lg.data_ptr(), None, 0.0, None, L, V, x.data_ptr(), 1, L, L, V - 1, _lib.REMASK[rule], 0, 17, 29, 0.8, None, rs.data_ptr(),
                            3, 0, 0, x0.data_ptr(), conf.data_ptr(), ws.data_ptr() if scratch else None, ws.numel() if scratch else 0)
        _lib.check(lib.llada_remask_scores(C.byref(a), _lib.stream_ptr()))
        assert (x0[0, [1, 4]] == 0).all() and ((x0 >= 0) & (x0 < V)).all()
        if rule == "random":
            assert torch.equal(conf, rs)
        else:
            assert torch.isnan(conf[0, [1, 4]]).all() and torch.isfinite(conf[0, [0, 2, 3, 5]]).all()
