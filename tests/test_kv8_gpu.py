"""The 8-bit key/value cache and the attention over it on an MI355X, against float64 restatements (oracle/kv8.py).

Written values are exact (power-of-two scales: the only rounding is the code's own), so the cache is compared bit for
bit.  Attention: the probabilities are rounded to bf16 once (2^-8 relative: half a step) before they are summed with the
values, the result once more; scores carry the float32 error of 128 products, at most 130 * 2^-24 of |q| |k|, and the
exponential's argument a rounding of its own size, below 2^-19 for scores up to 32 in the log2 domain.  A relative error e
of the scores' exponent moves numerator and denominator by e each, hence
    |out - exact| <= 2^-8 (spread + |exact|) + 2 e spread + 2^-20 spread,   spread = sum p |v| / sum p."""
import numpy as np
import pytest

from oracle import kv8 as okv

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def rows(seed, n, L, H, poison=None):
    """bf16 [Q | K | V] rows with uneven key channels; poison: positions whose keys and values hold NaN / inf."""
    g = np.random.Generator(np.random.PCG64(seed))
    x = g.standard_normal((n, L, 3, H, 128)).astype(np.float32)
    x[:, :, 1] *= np.exp(0.7 * g.standard_normal((H, 128))).astype(np.float32)
    if poison is not None:
        for b, t, val in poison:
            x[b, t, 1:] = val
    return torch.from_numpy(x.reshape(n, L, 3 * H * 128)).cuda().to(torch.bfloat16)


def split(x, H):
    n, L, _ = x.shape
    y = x.double().cpu().numpy().reshape(n, L, 3, H, 128)
    return y[:, :, 0], y[:, :, 1], y[:, :, 2]


def values(cache, layer=0):
    return [t.double().cpu().numpy() for t in cache.read(layer)]


def make(n, L, H, dtype, layers=1):
    from llada_amd import KVCache8
    return KVCache8(n, L, H, n_layers=layers, dtype=dtype, device="cuda")


def left_mask(n, L, seed=0):
    g = np.random.Generator(np.random.PCG64(seed + 91))
    m = np.ones((n, L), dtype=np.uint8)
    for b in range(n):
        m[b, :int(g.integers(0, max(1, L // 2 + 1)))] = 0
    return m


def same(a, b):
    return np.array_equal(a, b, equal_nan=True)


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
@pytest.mark.parametrize("n,L,H,masked", [(1, 1, 1, False), (2, 63, 2, True), (1, 64, 3, False), (2, 65, 2, False), (3, 200, 5, True)])
def test_fill_is_exact(lib, n, L, H, masked, dtype):
    x = rows(L + H, n, L, H)
    m = left_mask(n, L) if masked else None
    c = make(n, L, H, dtype)
    c.fill(0, x, None if m is None else torch.from_numpy(m).cuda())
    _, k, v = split(x, H)
    gk, gv = values(c)
    assert same(gk, okv.held(k, dtype, m)) and same(gv, okv.held(v, dtype, m))


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
def test_fill_values_of_every_size(lib, dtype):
    """Scale borders (largest magnitude at the code's range times a power of two and one step past it), subnormal codes,
    zeros, infinities, NaN, the smallest and largest bf16 values."""
    L, H = 64 * 6, 2
    x = rows(5, 1, L, H).float().reshape(1, L, 3, H, 128)
    x[0, 0:64] *= 2.0 ** -9
    x[0, 7, 1, 0, 3], x[0, 7, 2, 0, 3] = 448.0, 127.0
    x[0, 64:128] = 0.0
    x[0, 70, 1, 1, 0] = 450.0
    x[0, 71, 2, 1, 0] = 127.5
    x[0, 128:192] *= 1e-30
    x[0, 192:256] *= 2.0 ** 100
    x[0, 200, 1, 0, 5] = float("inf")
    x[0, 201, 2, 0, 5] = float("-inf")
    x[0, 202, 1, 1, 9] = float("nan")
    x[0, 203, 2, 1, 9] = float("nan")
    x[0, 256:320] *= 2.0 ** -100
    x[0, 330, 1, 0, :] = -0.0
    xb = x.reshape(1, L, -1).to(torch.bfloat16)
    c = make(1, L, H, dtype)
    c.fill(0, xb)
    _, k, v = split(xb, H)
    gk, gv = values(c)
    assert same(gk, okv.held(k, dtype)) and same(gv, okv.held(v, dtype))


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
@pytest.mark.parametrize("L,start,length", [(200, 0, 200), (200, 70, 1), (200, 64, 64), (200, 60, 10), (200, 137, 63), (200, 199, 1),
                                            (65, 0, 64), (300, 10, 250)])
def test_update_requantises_the_touched_blocks(lib, L, start, length, dtype):
    n, H = 2, 3
    m = left_mask(n, L, 7)
    mt = torch.from_numpy(m).cuda()
    x, y = rows(1, n, L, H), rows(2, n, length, H) * 3
    c = make(n, L, H, dtype, layers=3)
    c.fill(1, x, mt)
    c.update(1, y, start, mt)
    _, k, v = split(x, H)
    _, yk, yv = split(y, H)
    gk, gv = values(c, 1)
    assert same(gk, okv.updated(okv.held(k, dtype, m), yk, start, dtype, m))
    assert same(gv, okv.updated(okv.held(v, dtype, m), yv, start, dtype, m))
    for other in (0, 2):                       # the neighbouring layers stay what they were: zeros
        for t in values(c, other):
            assert not t.any()


def test_update_of_a_fresh_cache(lib):
    """A block of a new cache that is written in part holds zeros elsewhere."""
    c = make(1, 100, 2, "e4m3")
    y = rows(3, 1, 7, 2)
    c.update(0, y, 61)
    _, yk, _ = split(y, 2)
    want = okv.updated(np.zeros((1, 100, 2, 128)), yk, 61, "e4m3")
    assert same(values(c)[0], want)


def test_strided_and_flat_rows(lib):
    n, L, H = 2, 70, 2
    x = rows(4, n, L, H)
    want = None
    wide = torch.zeros((n, L, 3 * H * 128 + 64), dtype=torch.bfloat16, device="cuda")
    wide[..., :3 * H * 128] = x
    odd = torch.zeros((n, L, 3 * H * 128 + 3), dtype=torch.bfloat16, device="cuda")
    odd[..., :3 * H * 128] = x
    bigger = torch.zeros((n, L + 9, 3 * H * 128), dtype=torch.bfloat16, device="cuda")
    bigger[:, 4:4 + L] = x
    shifted = torch.zeros(x.numel() + 1, dtype=torch.bfloat16, device="cuda")[1:].view(x.shape)
    shifted.copy_(x)
    for form in (x, x.reshape(n * L, -1), wide, odd, bigger[:, 4:4 + L], shifted, x.transpose(0, 1).contiguous().transpose(0, 1)):
        c = make(n, L, H, "int8")
        c.fill(0, form)
        got = values(c)
        out = c.attend(0, form[:, 5:15] if form.dim() == 3 else x[:, 5:15]).float().cpu().numpy()
        want = want or (got, out)
        assert same(got[0], want[0][0]) and same(got[1], want[0][1]) and same(out, want[1])


def check_attend(c, x, H, n_q, dtype, m, fresh, start, fresh_rows=None):
    n, L, d = x.shape[0], x.shape[1], H * 128
    y = rows(77 + n_q, n, n_q, H) if fresh_rows is None else fresh_rows
    mt = None if m is None else torch.from_numpy(m).cuda()
    c.fill(0, x, mt)
    out = c.attend(0, y, mt, block=y if fresh else None, block_start=start if fresh else 0)
    assert out.shape == (n, n_q, d) and out.dtype == torch.bfloat16
    _, k, v = split(x, H)
    k, v = okv.held(k, dtype, m), okv.held(v, dtype, m)
    q, yk, yv = split(y, H)
    if fresh:
        k[:, start:start + n_q], v[:, start:start + n_q] = yk, yv
    want, spread = okv.attend(q, k, v, m)
    got = out.double().cpu().numpy().reshape(n, n_q, H, 128)
    keep = np.ones((n, L), bool) if m is None else m.astype(bool)
    kn = np.sqrt((np.where(keep[:, :, None, None], k, 0.0) ** 2).sum(-1)).max() if keep.any() else 0.0
    e = 130 * 2.0 ** -24 * np.sqrt((q ** 2).sum(-1)).max() * kn / np.sqrt(128) + 2.0 ** -19
    tol = 2.0 ** -8 * (spread + np.abs(want)) + (2 * e + 2.0 ** -20) * spread
    assert np.isfinite(got).all()
    worst = np.max(np.abs(got - want) - tol)
    assert worst <= 0, f"beyond the bound by {worst:.3g} (largest bound {tol.max():.3g})"
    return out


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
@pytest.mark.parametrize("n,L,H,n_q,start,fresh", [
    (1, 1, 1, 1, 0, False), (1, 1, 1, 1, 0, True), (2, 64, 2, 1, 63, True), (1, 65, 3, 31, 10, True), (2, 200, 2, 32, 60, True),
    (1, 384, 2, 33, 320, True), (3, 130, 1, 64, 64, True), (1, 257, 2, 65, 0, True), (2, 300, 2, 129, 171, True), (1, 200, 2, 200, 0, True),
    (1, 1030, 1, 32, 512, True), (2, 1030, 1, 200, 830, True), (1, 2100, 2, 3, 0, False), (1, 700, 5, 300, 0, False)])
@pytest.mark.parametrize("masked", [False, True])
def test_attend(lib, n, L, H, n_q, start, fresh, masked, dtype):
    m = left_mask(n, L, n_q) if masked else None
    check_attend(make(n, L, H, dtype), rows(L, n, L, H), H, n_q, dtype, m, fresh, start)


@pytest.mark.parametrize("n_q", [1, 40, 100])
def test_rows_a_mask_leaves_empty_and_poisoned_padding(lib, n_q):
    """One sequence without any unmasked token gives zeros; NaN and infinities under masked tokens, cached or fresh, reach
    nothing."""
    n, L, H, start = 3, 200, 2, 90
    m = np.ones((n, L), dtype=np.uint8)
    m[0] = 0
    m[1, :70] = 0
    m[1, 90] = 0
    m[2, 150:] = 0
    bad = [(1, 3, float("nan")), (1, 64, float("inf")), (2, 199, float("-inf")), (0, 5, float("nan"))]
    x = rows(8, n, L, H, bad)
    y = rows(9, n, n_q, H)
    y.view(n, n_q, 3, H, 128)[1, 0, 1:] = float("nan")
    y.view(n, n_q, 3, H, 128)[0, 0, 1:] = float("inf")
    c = make(n, L, H, "e4m3")
    out = check_attend(c, x, H, n_q, "e4m3", m, True, start, y)
    assert not out[0].any()


def test_cached_nan_under_a_later_mask(lib):
    """A NaN that the cache holds (written unmasked) does not reach the result of a call that masks its token; a call that
    attends it gives NaN."""
    n, L, H = 1, 130, 1
    x = rows(12, n, L, H, [(0, 77, float("nan"))])
    c = make(n, L, H, "e4m3")
    c.fill(0, x)
    m = torch.ones((n, L), dtype=torch.uint8, device="cuda")
    m[0, 77] = 0
    y = rows(13, n, 4, H)
    assert torch.isfinite(c.attend(0, y, m)).all()
    assert torch.isnan(c.attend(0, y)).all()


def test_one_hot_and_uniform(lib):
    """A query that matches one key only returns that key's value; equal scores return the mean."""
    L, H = 300, 2
    x = torch.zeros((1, L, 3, H, 128), dtype=torch.bfloat16, device="cuda")
    g = np.random.Generator(np.random.PCG64(5))
    x[0, :, 2] = torch.from_numpy(g.integers(-8, 9, size=(L, H, 128)).astype(np.float32)).cuda().to(torch.bfloat16)
    x[0, :, 1, :, 0] = -100.0
    x[0, 217, 1, :, 0] = 100.0
    c = make(1, L, H, "int8")
    c.fill(0, x.view(1, L, -1))
    q = torch.zeros((1, 3, 3, H, 128), dtype=torch.bfloat16, device="cuda")
    q[0, 1, 0, :, 0] = 64.0
    out = c.attend(0, q.view(1, 3, -1)).view(3, H, 128)
    assert torch.equal(out[1], x[0, 217, 2])
    mean = x[0, :, 2].double().mean(0)
    assert ((out[0].double() - mean).abs() <= 2.0 ** -8 * mean.abs() + 1e-6).all()       # p = 1 exactly: only the output rounds


def test_masks_of_every_type(lib):
    n, L, H = 2, 90, 1
    m = left_mask(n, L, 3)
    x, y = rows(14, n, L, H), rows(15, n, 5, H)
    ref = None
    for t in (torch.from_numpy(m).cuda(), torch.from_numpy(m).cuda().bool(), torch.from_numpy(m).cuda().long() * 7,
              torch.from_numpy(m).cuda().float(), torch.from_numpy(np.ascontiguousarray(m.T)).cuda().T):
        c = make(n, L, H, "e4m3")
        c.fill(0, x, t)
        out = c.attend(0, y, t)
        ref = out if ref is None else ref
        assert torch.equal(out, ref)


def test_key_splits_and_neighbours(lib):
    """The same rows with and without the key splits' scratch agree to rounding, and a query's result does not depend on the
    other sequences of the call."""
    n, L, H, n_q = 2, 3000, 2, 32
    x, y = rows(20, n, L, H), rows(21, n, n_q, H)
    c = make(n, L, H, "e4m3")
    c.fill(0, x)
    assert lib.llada_attn_kv8_workspace_bytes(n, n_q, L, H) > 0
    a = c.attend(0, y)
    c._ws_bytes[n_q] = 0
    b = c.attend(0, y)
    assert (a.float() - b.float()).abs().max() <= 2.0 ** -6 * a.float().abs().max()
    one = make(1, L, H, "e4m3")
    one.fill(0, x[1:])
    one._ws_bytes[n_q] = 0
    assert torch.equal(one.attend(0, y[1:]), b[1:])


def test_outputs_past_the_rows_stay(lib):
    n, L, H, n_q = 1, 100, 2, 5
    c = make(n, L, H, "e4m3")
    c.fill(0, rows(22, n, L, H))
    buf = torch.full((n * n_q + 4, H * 128), 7.0, dtype=torch.bfloat16, device="cuda")
    out = buf[:n * n_q].view(n, n_q, H * 128)
    y = rows(23, n, n_q, H)
    assert torch.equal(c.attend(0, y, out=out), c.attend(0, y))
    assert (buf[n * n_q:] == 7.0).all()
    with pytest.raises(ValueError):
        c.attend(0, y, out=buf)


def test_refusals(lib):
    from llada_amd import KVCache8
    c = make(2, 100, 2, "e4m3")
    x = rows(24, 2, 100, 2)
    for call in (lambda: c.fill(0, x[:1]), lambda: c.fill(0, x.float()), lambda: c.fill(0, x[..., :700]), lambda: c.update(0, x, 1),
                 lambda: c.update(0, x[:, :5], -1), lambda: c.update(0, x[:, :5].reshape(10, -1), 0), lambda: c.fill(0, x, torch.ones(2, 99, device="cuda")),
                 lambda: c.fill(0, x, torch.ones(2, 100)), lambda: c.attend(0, x[:, :5], block=x[:, :5], block_start=96),
                 lambda: c.attend(0, x[:, :0]), lambda: c.attend(0, x[0, :5]), lambda: c.fill(0, x.cpu())):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(IndexError):
        c.fill(1, x)
    with pytest.raises(IndexError):
        c.read(-1)
    with pytest.raises(NotImplementedError):
        KVCache8(1, 1, 1, dtype="bf16")


def test_captured_step_on_a_side_stream(lib):
    """update + attend captured once and replayed with new inputs, eager calls on the same cache in between, against eager
    results each time."""
    n, L, H, n_q, start = 2, 700, 2, 32, 300
    c, e = make(n, L, H, "int8"), make(n, L, H, "int8")
    x = rows(30, n, L, H)
    c.fill(0, x)
    e.fill(0, x)
    buf = rows(31, n, n_q, H)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.attend(0, buf, block=buf, block_start=start)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = c.attend(0, buf, block=buf, block_start=start)
            c.update(0, buf, start)
            after = c.read(0)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(4):
        buf.copy_(rows(40 + i, n, n_q, H))
        g.replay()
        want = e.attend(0, buf, block=buf, block_start=start)
        e.update(0, buf, start)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(after[0], e.read(0)[0]) and torch.equal(after[1], e.read(0)[1])
        torch.cuda.synchronize()


@pytest.mark.parametrize("nq", [1, 2, 4])
@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("n_q,start,fresh", [(20, 100, True), (75, 300, True), (150, 0, True), (260, 140, True), (33, 0, False)])
def test_every_way_to_deal_the_work(lib, nq, splits, n_q, start, fresh):
    """Query groups and key splits forced: the bound holds whatever the plan (fresh tiles in one split, in several, in none)."""
    n, L, H = 2, 400, 2
    try:
        lib.llada_attn_kv8_force(nq, splits)
        check_attend(make(n, L, H, "e4m3"), rows(L + nq, n, L, H), H, n_q, "e4m3", left_mask(n, L, n_q), fresh, start)
    finally:
        lib.llada_attn_kv8_force(0, 0)


@pytest.mark.parametrize("n_q,b_len,start", [(1, 200, 37), (20, 330, 64), (40, 130, 270), (140, 1, 399), (140, 400, 0), (5, 64, 128)])
@pytest.mark.parametrize("masked", [False, True])
def test_block_of_another_length_than_the_queries(lib, n_q, b_len, start, masked):
    """Fresh rows for more or fewer tokens than there are queries: several fresh tiles for few queries, one row for many."""
    n, L, H, dtype = 2, 400, 2, "e4m3"
    m = left_mask(n, L, b_len) if masked else None
    if masked:
        m[1, start:start + b_len:3] = 0
    mt = None if m is None else torch.from_numpy(m).cuda()
    x, y, f = rows(50, n, L, H), rows(51, n, n_q, H), rows(52, n, b_len, H)
    c = make(n, L, H, dtype)
    c.fill(0, x, mt)
    out = c.attend(0, y, mt, block=f, block_start=start)
    _, k, v = split(x, H)
    k, v = okv.held(k, dtype, m), okv.held(v, dtype, m)
    q = split(y, H)[0]
    _, k[:, start:start + b_len], v[:, start:start + b_len] = split(f, H)
    want, spread = okv.attend(q, k, v, m)
    got = out.double().cpu().numpy().reshape(n, n_q, H, 128)
    e = 130 * 2.0 ** -24 * np.sqrt((q ** 2).sum(-1)).max() * np.sqrt((k ** 2).sum(-1)).max() / np.sqrt(128) + 2.0 ** -19
    assert (np.abs(got - want) <= 2.0 ** -8 * (spread + np.abs(want)) + (2 * e + 2.0 ** -20) * spread).all()


def test_offsets_past_32_bits(lib):
    """A cache of more than 4 GiB: the last sequence's results and values equal those of a cache of that sequence alone."""
    n, L, H, n_q = 5, 131072, 32, 3
    new, q = rows(60, n, 130, H), rows(61, n, n_q, H)
    big, one = make(n, L, H, "e4m3"), make(1, L, H, "e4m3")
    assert big.layer_bytes > 2 ** 32
    try:
        lib.llada_attn_kv8_force(1, 1)
        for c, sel in ((big, slice(None)), (one, slice(n - 1, n))):
            c.update(0, new[sel], L - 130)
            c.update(0, new[sel, :64], 64)
        a, b = big.attend(0, q, block=new, block_start=L - 200), one.attend(0, q[n - 1:], block=new[n - 1:], block_start=L - 200)
    finally:
        lib.llada_attn_kv8_force(0, 0)
    assert torch.equal(a[n - 1:], b) and b.abs().max() > 0
    kb, ko = big.read(0)[0], one.read(0)[0]
    assert torch.equal(kb[n - 1], ko[0]) and ko[0, -100:].abs().max() > 0
    assert torch.equal(kb[0, 64:128], okv_held_like(new[0, :64], H))


def okv_held_like(rows_, H):
    k = rows_.double().cpu().numpy().reshape(1, 64, 3, H, 128)[:, :, 1]
    return torch.from_numpy(okv.held(k, "e4m3")[0]).cuda().to(torch.bfloat16)


def test_two_streams_at_once(lib):
    """Calls on two caches from two streams, key splits' scratch in use, give what they give one after the other."""
    L, H, n_q = 4096, 32, 16
    cs = [make(1, L, H, "e4m3") for _ in range(2)]
    qs = [rows(70 + i, 1, n_q, H) for i in range(2)]
    for i, c in enumerate(cs):
        c.fill(0, rows(72 + i, 1, L, H))
    want = [c.attend(0, q) for c, q in zip(cs, qs)]
    assert lib.llada_attn_kv8_workspace_bytes(1, n_q, L, H) > 0
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(cs[i].attend(0, qs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for t in got[i]:
            assert torch.equal(t, want[i])


@pytest.mark.parametrize("n,L,n_q", [(2, 200, 40), (1, 4200, 16), (2, 300, 150)])
def test_output_in_the_queries_memory_but_not_in_the_blocks(lib, n, L, n_q):
    from llada_amd import KVCache8
    H = 4
    cache = KVCache8(n, L, H)
    cache.fill(0, torch.randn(n, L, 3 * H * 128, device="cuda").to(torch.bfloat16))
    q = torch.randn(n, n_q, H * 128, device="cuda").to(torch.bfloat16)
    want = cache.attend(0, q)
    got = cache.attend(0, q, out=q)
    assert got.data_ptr() == q.data_ptr() and torch.equal(got, want)
    block = torch.randn(n, n_q, 3 * H * 128, device="cuda").to(torch.bfloat16)
    inside = block.view(-1)[: n * n_q * H * 128].view(n, n_q, H * 128)
    with pytest.raises(ValueError, match="overlaps"):
        cache.attend(0, block, block=block, out=inside)


def scaled_blocks(seed, n, L, H, exponents):
    """Rows whose 64-token blocks of values are N(0, 1) * 2^exponents[block % len], within bf16's finite range."""
    x = rows(seed, n, L, H).double().view(n, L, 3, H, 128)
    x[:, :, 1] *= 0.5
    e = torch.tensor([exponents[(t // 64) % len(exponents)] for t in range(L)], dtype=torch.float64, device="cuda")
    x[:, :, 2] = (x[:, :, 2] * 2.0 ** e[None, :, None, None]).clamp(-2.0 ** 127, 2.0 ** 127)
    return x.view(n, L, -1).to(torch.bfloat16)


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
@pytest.mark.parametrize("nq,splits,n_q", [(0, 0, 5), (1, 3, 20), (2, 1, 70), (4, 1, 140)])
@pytest.mark.parametrize("exponents", [(0, -100), (0, -108), (-110, 0), (-120, 0, 0), (0, -126, -118), (-100,), (-110, -104), (60, -60, 0), (80, 0),
                                       (0, 126), (126, 0), (126,), (126, -120, 0), (70, 126, 10)])
def test_value_blocks_of_every_size(lib, exponents, nq, splits, n_q, dtype):
    """The weights of a block's keys do not depend on the size of its values.  Beside check_attend's bound: what the exponential
    and the matrix unit may flush, for each of the L keys 2^-117 of the largest value."""
    n, L, H = 2, 330, 2
    x, y = scaled_blocks(L + n_q, n, L, H, exponents), rows(77 + n_q, n, n_q, H)
    c = make(n, L, H, dtype)
    c.fill(0, x)
    try:
        lib.llada_attn_kv8_force(nq, splits)
        got = c.attend(0, y).double().cpu().numpy().reshape(n, n_q, H, 128)
    finally:
        lib.llada_attn_kv8_force(0, 0)
    _, k, v = split(x, H)
    k, v, q = okv.held(k, dtype), okv.held(v, dtype), split(y, H)[0]
    want, spread = okv.attend(q, k, v)
    e = 130 * 2.0 ** -24 * np.sqrt((q ** 2).sum(-1)).max() * np.sqrt((k ** 2).sum(-1)).max() / np.sqrt(128) + 2.0 ** -19
    tol = 2.0 ** -8 * (spread + np.abs(want)) + (2 * e + 2.0 ** -20) * spread + L * 2.0 ** -117 * np.abs(v).max()
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) / tol)


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
def test_fill_at_the_top_of_bf16(lib, dtype):
    """Codes that would stand for 2^128 become the next lower one: every held value is finite, infinities included."""
    L, H = 64 * 5, 2
    x = rows(6, 1, L, H).float().reshape(1, L, 3, H, 128)
    top = torch.finfo(torch.bfloat16).max
    x[0, :256] *= 2.0 ** 124
    x[0, 3, 1, 0, 5], x[0, 4, 2, 1, 9] = top, -top
    x[0, 64:128, 1:] = top
    x[0, 130, 1:, :, 0], x[0, 131, 1:, :, 1], x[0, 132, 1:, :, 2] = top, float("inf"), float("-inf")
    x[0, 133, 1:, 1, 3] = float("nan")
    x[0, 200, 1:, :, 0] = 1.75 * 2.0 ** 127           # e4m3: the largest magnitude that fits 448 * 2^119
    x[0, 260, 1:, 0, 0], x[0, 261, 1:, 0, 1] = 127 * 2.0 ** 121, float("inf")     # likewise int8, 127 * 2^121
    xb = x.reshape(1, L, -1).to(torch.bfloat16)
    c = make(1, L, H, dtype)
    c.fill(0, xb)
    _, k, v = split(xb, H)
    for got, w in zip(values(c), (k, v)):
        want = okv.held(w, dtype)
        assert same(got, want) and not np.isinf(got).any()
    c.update(0, xb[:, 3:4], 70)                       # requantised beside what the block holds
    for got, w in zip(values(c), (k, v)):
        assert same(got, okv.updated(okv.held(w, dtype), w[:, 3:4], 70, dtype)) and not np.isinf(got).any()


def test_output_that_only_partly_covers_the_queries_is_refused(lib):
    """Without a block too: an output in the storage of [Q | K | V] rows, one shifted against q, one over its last rows."""
    n, L, H, n_q = 2, 100, 2, 6
    d = H * 128
    c = make(n, L, H, "e4m3")
    c.fill(0, rows(90, n, L, H))
    y = rows(91, n, n_q, H)
    want = c.attend(0, y)
    flat = torch.zeros((n * n_q + 4) * d, dtype=torch.bfloat16, device="cuda")
    q = flat[d:d + n * n_q * d].view(n, n_q, d)
    q.copy_(y[..., :d])
    for bad_q, bad in ((y, y.view(-1)[:n * n_q * d]), (q, flat[:n * n_q * d]), (q, flat[2 * d:2 * d + n * n_q * d]), (q, flat[d + 8:d + 8 + n * n_q * d])):
        with pytest.raises(ValueError, match="overlaps q"):
            c.attend(0, bad_q, out=bad.view(n, n_q, d))
    with pytest.raises(ValueError, match="overlaps the cache"):
        c.attend(0, q, out=c.data.view(-1)[4096:4096 + 2 * n * n_q * d].view(torch.bfloat16).view(n, n_q, d))
    after = flat[(n * n_q + 1) * d:(n * n_q + 1) * d + d]
    assert torch.equal(c.attend(0, q, out=q), want) and not after.any()
    one = make(1, L, H, "e4m3")                             # a single row may stand in its own [Q | K | V] row
    one.fill(0, rows(92, 1, L, H))
    z = rows(93, 1, 1, H)
    want = one.attend(0, z)
    assert torch.equal(one.attend(0, z, out=z[..., :d]), want)


@pytest.mark.parametrize("L", [64 * 30, 64 * 46])
def test_scratch_covers_a_block_cut_at_both_ends(lib, L):
    """Two tiles more than the cache has: the scratch asked for holds the splits that the call then plans."""
    n, H, n_q, start = 1, 2, 65, 1
    x, y = rows(95, n, L, H), rows(96, n, n_q, H)
    c = make(n, L, H, "e4m3")
    c.fill(0, x)
    a = c.attend(0, y, block=y, block_start=start)
    c._ws_bytes[n_q] *= 2
    assert torch.equal(c.attend(0, y, block=y, block_start=start), a)        # more scratch changes nothing: the same splits
    check_attend(c, x, H, n_q, "e4m3", None, True, start, y)


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
@pytest.mark.parametrize("nq,splits,n_q,fresh", [(0, 0, 5, False), (1, 3, 20, True), (2, 1, 70, False), (4, 1, 140, True)])
@pytest.mark.parametrize("exponents", [(20,), (25,), (30,), (40,), (70, 0), (0, 45, 100), (110,)])
def test_key_blocks_of_every_size(lib, exponents, nq, splits, n_q, fresh, dtype):
    """Scores past what the exponential's argument resolves: the softmax is one-hot, and its one value comes back (the largest
    probability is 1 up to a common factor: bf16 roundings of it and of the result).  Queries whose two largest scores float32
    sums could confuse (130 * 2^-24 of |q| |k| each) are left out."""
    n, L, H, start = 2, 330, 2, 100
    x, y = rows(97, n, L, H).double().view(n, L, 3, H, 128), rows(98, n, n_q, H)
    e = torch.tensor([exponents[(t // 64) % len(exponents)] for t in range(L)], dtype=torch.float64, device="cuda")
    x[:, :, 1] *= 2.0 ** e[None, :, None, None]
    x = x.view(n, L, -1).to(torch.bfloat16)
    f = rows(99, n, 90, H)
    if fresh:
        f.view(n, 90, 3, H, 128)[:, :, 1] *= 2.0 ** max(exponents)
    c = make(n, L, H, dtype)
    c.fill(0, x)
    try:
        lib.llada_attn_kv8_force(nq, splits)
        got = c.attend(0, y, block=f if fresh else None, block_start=start if fresh else 0).double().cpu().numpy().reshape(n, n_q, H, 128)
    finally:
        lib.llada_attn_kv8_force(0, 0)
    _, k, v = split(x, H)
    k, v, q = okv.held(k, dtype), okv.held(v, dtype), split(y, H)[0]
    if fresh:
        _, k[:, start:start + 90], v[:, start:start + 90] = split(f, H)
    assert np.isfinite(got).all()
    score = np.einsum("bqhd,bkhd->bhqk", q, k) / np.sqrt(128)
    top = np.sort(score, axis=3)[..., -2:]
    size = np.sqrt((q ** 2).sum(-1)).transpose(0, 2, 1)[..., None] * np.sqrt((k ** 2).sum(-1)).transpose(0, 2, 1)[:, :, None, :] / np.sqrt(128)
    clear = top[..., 1] - top[..., 0] > 2 * 130 * 2.0 ** -24 * size.max(axis=3) + 40
    at = score.argmax(axis=3)
    assert clear.mean() > 0.9
    for b in range(n):
        for h in range(H):
            rows_ = np.nonzero(clear[b, h])[0]
            want = v[b, at[b, h, rows_], h]
            assert (np.abs(got[b, rows_, h] - want) <= 2.0 ** -7 * np.abs(want) + 1e-12).all()


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
def test_tiny_keys_under_a_mask(lib, dtype):
    """Scores that vanish (key scales down to 2^-126 take the scores' multiplier below the normal numbers): equal weights for the
    unmasked keys, none for the others."""
    n, L, H, n_q = 2, 200, 2, 9
    m = left_mask(n, L, 5)
    m[1, 100:] = 0
    for e in (-100, -126):
        x = rows(100, n, L, H).double().view(n, L, 3, H, 128)
        x[:, :, 1] *= 2.0 ** e
        check_attend(make(n, L, H, dtype), x.view(n, L, -1).to(torch.bfloat16), H, n_q, dtype, m, False, 0)
