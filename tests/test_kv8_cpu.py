"""The 8-bit cache without a GPU: sizes, refusals (all decided before any launch), and the oracle on known values."""
import ctypes as C

import numpy as np
import pytest

from oracle import kv8 as okv

P16 = C.c_void_p(256)        # never dereferenced: every call below is refused first


def write(lib, **k):
    a = dict(qkv=P16, stride=768, mask=None, cache=P16, type=0, n_seq=1, L=64, H=2, start=0, len=64)
    a.update(k)
    return lib.llada_kv8_write(a["qkv"], a["stride"], a["mask"], a["cache"], a["type"], a["n_seq"], a["L"], a["H"], a["start"], a["len"], None)


def attend(lib, **k):
    a = dict(q=P16, stride=768, n_q=4, cache=P16, type=0, mask=None, out=P16, n_seq=1, L=64, H=2, block=None, b_stride=0, b_start=0,
             b_len=0, ws=None, ws_bytes=0)
    a.update(k)
    return lib.llada_attn_kv8(a["q"], a["stride"], a["n_q"], a["cache"], a["type"], a["mask"], a["out"], a["n_seq"], a["L"], a["H"],
                              a["block"], a["b_stride"], a["b_start"], a["b_len"], a["ws"], a["ws_bytes"], None)


def test_layer_bytes(lib):
    # scales: 8 bytes a (sequence, head, block), rounded up to 256; tiles: 16 KiB each
    assert lib.llada_kv8_layer_bytes(1, 64, 1) == 256 + 16384
    assert lib.llada_kv8_layer_bytes(1, 65, 1) == 256 + 2 * 16384
    assert lib.llada_kv8_layer_bytes(3, 1000, 32) == 3 * 32 * 16 * 8 + 3 * 32 * 16 * 16384
    # past 32 bits
    assert lib.llada_kv8_layer_bytes(64, 131072, 32) == 64 * 32 * 2048 * (8 + 16384)
    assert lib.llada_kv8_layer_bytes(0, 64, 1) == 0 and lib.llada_kv8_layer_bytes(1, 0, 1) == 0


@pytest.mark.parametrize("bad", [dict(qkv=None), dict(cache=None), dict(n_seq=0), dict(L=0), dict(H=0), dict(start=-1), dict(len=0),
                                 dict(start=1), dict(len=65), dict(start=2 ** 31 - 1, len=2 ** 31 - 1), dict(stride=760), dict(stride=772),
                                 dict(qkv=C.c_void_p(264)), dict(cache=C.c_void_p(128))])
def test_write_refuses(lib, bad):
    from llada_amd import _lib
    assert write(lib, **bad) == _lib.ERR_INVALID and lib.llada_last_error()


@pytest.mark.parametrize("bad", [dict(q=None), dict(cache=None), dict(out=None), dict(n_q=0), dict(stride=248), dict(stride=260),
                                 dict(q=C.c_void_p(264)), dict(out=C.c_void_p(264)), dict(ws=C.c_void_p(8)),
                                 dict(block=P16, b_stride=768, b_start=61, b_len=4), dict(block=P16, b_stride=768, b_start=-1, b_len=4),
                                 dict(block=P16, b_stride=768, b_start=0, b_len=0), dict(block=P16, b_stride=760, b_start=0, b_len=4),
                                 dict(block=C.c_void_p(264), b_stride=768, b_start=0, b_len=4),
                                 dict(block=P16, b_stride=768, b_start=2 ** 31 - 2, b_len=2 ** 31 - 2)])
def test_attend_refuses(lib, bad):
    from llada_amd import _lib
    assert attend(lib, **bad) == _lib.ERR_INVALID and lib.llada_last_error()


def test_unknown_type_and_read_refusals(lib):
    from llada_amd import _lib
    assert write(lib, type=2) == _lib.ERR_UNSUPPORTED
    assert attend(lib, type=-1) == _lib.ERR_UNSUPPORTED
    assert lib.llada_kv8_read(P16, 7, P16, P16, 1, 64, 1, None) == _lib.ERR_UNSUPPORTED
    assert lib.llada_kv8_read(None, 0, P16, P16, 1, 64, 1, None) == _lib.ERR_INVALID
    assert lib.llada_kv8_read(P16, 0, P16, C.c_void_p(8), 1, 64, 1, None) == _lib.ERR_INVALID
    with pytest.raises(NotImplementedError):
        from llada_amd import KVCache8
        KVCache8(1, 64, 2, dtype="fp4", device="cpu")
    with pytest.raises(ValueError):
        KVCache8(1, 0, 2, device="cpu")


def test_workspace_covers_what_a_call_uses(lib):
    """None where the queries fill the chip; otherwise whole splits of (row, head) partial results."""
    assert lib.llada_attn_kv8_workspace_bytes(64, 32, 4096, 32) == 0
    need = lib.llada_attn_kv8_workspace_bytes(1, 32, 4096, 32)
    assert need > 0 and need % (32 * 32 * (128 * 4 + 8)) == 0
    assert lib.llada_attn_kv8_workspace_bytes(1, 0, 64, 1) == 0


@pytest.mark.parametrize("dtype,top", [("e4m3", 448.0), ("int8", 127.0)])
def test_oracle_scale_borders(dtype, top):
    """The scale doubles exactly where the largest magnitude passes the code's range."""
    def one(amax):
        x = np.zeros((1, 64, 1, 128))
        x[0, 3, 0, 5] = amax
        return okv.held(x, dtype)[0, 3, 0, 5]
    assert one(top) == top and one(2 * top) == 2 * top and one(top * 2.0 ** -9) == top * 2.0 ** -9
    above = np.float64(top) * (1 + 2.0 ** -7)
    assert abs(one(above) - above) <= above * (2.0 ** -4 if dtype == "e4m3" else 2.0 ** -7)
    assert one(0.0) == 0.0


def test_oracle_matches_torch_float8_cast():
    torch = pytest.importorskip("torch")
    g = np.random.Generator(np.random.PCG64(3))
    x = torch.from_numpy(g.standard_normal((1, 128, 2, 128)).astype(np.float32)).to(torch.bfloat16).float().numpy()
    x[0, :, 1] *= 2.0 ** -12 * np.where(g.random((128, 128)) < 0.5, 1, 2.0 ** 9)
    got = okv.held(x, "e4m3")
    for t in (0, 64):
        for h in (0, 1):
            part = x[0, t:t + 64, h].astype(np.float64)
            k = np.ceil(np.log2(np.abs(part).max() / 448.0))
            want = torch.from_numpy((part / 2.0 ** k).astype(np.float32)).to(torch.float8_e4m3fn).float().numpy().astype(np.float64) * 2.0 ** k
            assert np.array_equal(got[0, t:t + 64, h], want)


def test_a_cache_needs_a_gpu():
    from llada_amd import KVCache8
    with pytest.raises(ValueError, match="GPU memory"):
        KVCache8(1, 64, 2, device="cpu")


@pytest.mark.parametrize("dtype,exponent,code", [("e4m3", 120, 240.0), ("int8", 122, 63.0)])
def test_oracle_at_the_top_of_bf16(dtype, exponent, code):
    """A code that would stand for 2^128 is the next lower one, for the largest finite value and for an infinity beside it."""
    x = np.zeros((1, 64, 1, 128))
    x[0, 0, 0, :3] = 255 * 2.0 ** 120, np.inf, -np.inf
    assert np.array_equal(okv.held(x, dtype)[0, 0, 0, :3], np.array([1, 1, -1]) * code * 2.0 ** exponent)
    x[0, 0, 0, 0] = okv.TOP[dtype] * 2.0 ** (exponent - 1)
    assert okv.held(x, dtype)[0, 0, 0, 0] == x[0, 0, 0, 0]


def test_which_outputs_race_with_the_queries():
    torch = pytest.importorskip("torch")
    from llada_amd.kv_cache import _output_races
    d, rows = 256, 12
    flat = torch.zeros(60 * d, dtype=torch.bfloat16)
    q, wide = flat[d:d + rows * d].view(2, 6, d), flat[:rows * 3 * d].view(2, 6, 3 * d)
    at = lambda i: flat[i:i + rows * d].view(2, 6, d)
    assert not _output_races(q, q, d) and not _output_races(at((rows + 1) * d), q, d) and not _output_races(torch.zeros_like(q), q, d)
    assert _output_races(at(0), q, d) and _output_races(at(d + 8), q, d) and _output_races(at(rows * d), q, d)
    assert _output_races(at(0), wide, 3 * d) and _output_races(at(3 * d), wide, 3 * d) and not _output_races(at((3 * rows - 2) * d + 0), wide[..., :d], 3 * d)
    assert not _output_races(wide[:1, :1, :d], wide[:1, :1], 3 * d) and _output_races(wide[:1, :2, :d], wide[:1, :2], 3 * d)


def test_sizes_past_the_library_are_refused(lib):
    """Sizes that 32 bits do not hold would wrap on their way into the library; launches end at 2^32 threads."""
    from llada_amd import KVCache8, _lib
    for sizes in ((2 ** 31, 64, 2), (1, 2 ** 32 + 64, 2), (1, 64, 2 ** 32 + 2)):
        with pytest.raises(ValueError, match="32 bits"):
            KVCache8(*sizes, device="cpu")
    many = dict(n_seq=2 ** 23, H=2, stride=768)
    assert write(lib, **many) == _lib.ERR_UNSUPPORTED
    assert attend(lib, **many) == _lib.ERR_UNSUPPORTED
    assert lib.llada_kv8_read(P16, 0, P16, P16, 2 ** 23, 64, 2, None) == _lib.ERR_UNSUPPORTED
