"""Truncated sampling without a GPU: the oracle on rows worked out by hand, and refusals."""
import ctypes as C

import numpy as np
import pytest

from oracle import sampling as osm

P16 = C.c_void_p(256)


def test_oracle_by_hand():
    l = np.log(np.array([1.0, 4.0, 2.0, 1.0]))       # order 1, 2, 0, 3; masses 4, 6, 7, 8 (of 8)
    assert [osm.sample(l, u)[0] for u in (0.0, 0.49, 0.51, 0.74, 0.76, 0.88, 0.999)] == [1, 1, 2, 2, 0, 3, 3]
    assert osm.sample(l, 0.99, top_k=2)[:1] == (2,) and abs(osm.sample(l, 0.99, top_k=2)[1] - 1 / 3) < 1e-15
    assert osm.sample(l, 0.99, top_p=0.5)[2] in (1, 2)
    assert osm.sample(l, 0.99, top_p=0.7)[2] == 2 and osm.sample(l, 0.99, top_p=0.8)[2] == 3
    assert osm.sample(l, 0.99, min_p=0.4)[2] == 2 and osm.sample(l, 0.99, min_p=1.0)[2] == 1
    assert osm.sample(l, 0.99, temperature=0.0)[0] == 1
    assert osm.sample(np.full(5, -np.inf), 0.3) == (0, 0.0, 0)
    assert osm.sample([np.nan, 1.0, np.inf, np.inf], 0.6)[0] == 3


def call(lib, sampling=True, **k):
    from llada_amd import _lib
    s = dict(temperature=1.0, top_p=1.0, min_p=0.0, top_k=0)
    a = dict(logits=P16, un=None, stride=64, n=2, V=64, tokens=P16)
    for key, v in k.items():
        (s if key in s else a)[key] = v
    sp = _lib.Sampling(s["temperature"], s["top_p"], s["min_p"], s["top_k"], None, None, None, None, None)
    return lib.llada_sample_rows(a["logits"], a["un"], a["stride"], 0.0, a["n"], a["V"], C.byref(sp) if sampling else None, 0, 0, 0, a["tokens"],
                                 None, None)


@pytest.mark.parametrize("bad", [dict(logits=None), dict(tokens=None), dict(n=0), dict(V=0), dict(stride=63), dict(temperature=-0.1),
                                 dict(temperature=float("nan")), dict(temperature=float("inf")), dict(top_k=-1), dict(top_p=0.0),
                                 dict(top_p=1.01), dict(top_p=float("nan")), dict(min_p=-0.1), dict(min_p=1.5), dict(min_p=float("nan")),
                                 dict(sampling=False), dict(logits=C.c_void_p(257)), dict(un=C.c_void_p(258))])
def test_refusals(lib, bad):
    from llada_amd import _lib
    assert call(lib, **bad) == _lib.ERR_INVALID and lib.llada_last_error()


def test_vocabulary_limit(lib):
    from llada_amd import _lib
    assert call(lib, V=131073, stride=131080) == _lib.ERR_UNSUPPORTED
    assert call(lib, V=131072, stride=131073) == _lib.ERR_UNSUPPORTED      # rows off the 16-byte grid hold seven fewer


def test_epilogue_refusals(lib):
    from llada_amd import _lib
    sp = _lib.Sampling(1.0, 1.0, 0.0, 0, None, None, None, None, None)
    assert lib.llada_remask_scores_sampled(None, C.byref(sp), None) == _lib.ERR_INVALID
    a = _lib.RemaskArgs()
    assert lib.llada_remask_scores_sampled(C.byref(a), C.byref(sp), None) == _lib.ERR_INVALID
    a = _lib.RemaskArgs(256, None, 0.0, None, 4, 64, 256, 2, 2, 2, 3, 0, 0, 0, 0, 1.0, None, None, 0, 0, 0, 256, 256, None, 0)
    assert lib.llada_remask_scores_sampled(C.byref(a), None, None) == _lib.ERR_INVALID
    a.vocab = 63
    assert lib.llada_remask_scores_sampled(C.byref(a), C.byref(sp), None) == _lib.ERR_UNSUPPORTED
    a.vocab, a.remasking = 64, 9
    assert lib.llada_remask_scores_sampled(C.byref(a), C.byref(sp), None) == _lib.ERR_UNSUPPORTED
    a.remasking, a.n_rows = 0, 3
    assert lib.llada_remask_scores_sampled(C.byref(a), C.byref(sp), None) == _lib.ERR_INVALID


def test_python_refusals():
    torch = pytest.importorskip("torch")
    from llada_amd import sample_tokens
    with pytest.raises(ValueError):
        sample_tokens(torch.zeros(2, 8, dtype=torch.bfloat16))              # no GPU tensor


@pytest.mark.parametrize("bad", [dict(top_k=-1), dict(top_p=0.0), dict(top_p=1.5), dict(top_p=float("nan")), dict(min_p=-0.5), dict(min_p=1.5)])
def test_scalars_out_of_range_are_refused_even_when_unused(bad):
    from llada_amd.sampling import truncates
    ok = dict(top_k=0, top_p=1.0, min_p=0.0)
    assert not truncates(0.7, **ok) and truncates(0.7, 5, 1.0, 0.0) and not truncates(0, 5, 0.5, 0.1)
    with pytest.raises(AssertionError):
        truncates(0, **{**ok, **bad})


@pytest.mark.parametrize("dtype", ["int8", "uint8", "int16", "int32", "int64", "bool", "float16", "bfloat16", "float32", "float64"])
def test_top_k_arrays_of_every_type(dtype):
    """Wide enough for the library's limit whatever the tensor's own type holds."""
    torch = pytest.importorskip("torch")
    from llada_amd.sampling import _top_k
    given = [0, 1, 1, 0] if dtype == "bool" else [0, 1, 100, 127] if dtype == "uint8" else [0, 1, 100, -3]
    got = _top_k(torch.tensor(given, dtype=getattr(torch, dtype))).to(torch.int32)
    assert got.tolist() == [max(g, -1) for g in given]
    if dtype in ("int64", "float32", "float64"):
        big = _top_k(torch.tensor([2 ** 40, -2 ** 40], dtype=getattr(torch, dtype))).to(torch.int32)
        assert big.tolist() == [2 ** 31 - 1, -1]


def test_epilogue_row_limit(lib):
    """One launch ends at 2^32 threads: as many rows of 1024 lanes."""
    from llada_amd import _lib
    sp = _lib.Sampling(1.0, 1.0, 0.0, 0, None, None, None, None, None)
    a = _lib.RemaskArgs(256, None, 0.0, None, 2 ** 22, 64, 256, 2 ** 11, 2 ** 11, 2, 3, 0, 0, 0, 0, 1.0, None, None, 0, 0, 0, 256, 256, None, 0)
    assert lib.llada_remask_scores_sampled(C.byref(a), C.byref(sp), None) == _lib.ERR_UNSUPPORTED
