"""Truncated sampling: temperature, top-k, top-p and min-p from one given uniform per row.

The reference's temperature (generate.py:8-19) is a Gumbel-max over the whole vocabulary and offers no truncation; this
is the operator behind ``generate(top_k=, top_p=, min_p=)``, for callers that sample rows of logits themselves."""
import ctypes as C

import torch

from . import _lib


def truncates(temperature, top_k, top_p, min_p):
    """Whether these scalars draw from a truncated distribution (temperature 0 is the arg-max whatever they are)."""
    assert top_k >= 0 and 0.0 < top_p <= 1.0 and 0.0 <= min_p <= 1.0, f"top_k={top_k}, top_p={top_p}, min_p={min_p}"
    return temperature != 0 and (top_k > 0 or top_p < 1.0 or min_p > 0.0)


TOP_K_MAX = 2 ** 31 - 1


def _top_k(k):
    """A top_k for the library's 32 bits: any larger one keeps the whole row as well (a negative one is refused there)."""
    if isinstance(k, torch.Tensor):        # (in a type that holds the limits: an int16 tensor's own does not)
        return k.to(torch.float64 if k.is_floating_point() else torch.int64).clamp(-1, TOP_K_MAX)
    return max(-1, min(int(k), TOP_K_MAX))


def scalar_sampling(temperature, top_k, top_p, min_p, uniforms=None):
    """The C parameters for one value of each; ``uniforms``: float64 tensor, or None for the library's own stream."""
    return _lib.Sampling(float(temperature), float(top_p), float(min_p), _top_k(top_k), None, None, None, None, _lib.ptr(uniforms))


def sample_tokens(logits, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, *, uniforms=None, uncond_logits=None, cfg_scale=0.0,
                  seed=0, step=0, row_offset=0, return_probs=False):
    """One token id per row of ``logits`` [..., vocab] (bf16, vocab up to 131072, or 131065 where the rows do not start at
    16-byte boundaries), int64 [...].

    With a row's entries ordered by (logit descending, index ascending) and w_i = exp((l_i - max) / temperature) in
    float64: top-k keeps the first ``top_k`` (0: all), top-p the shortest prefix of those with at least ``top_p`` of
    their mass, min-p the entries with w_i >= ``min_p``; what all three keep (at least one entry) is sampled: the token is
    the first whose running mass exceeds u times the kept total.  temperature 0 gives the arg-max.  ``temperature``,
    ``top_k``, ``top_p`` and ``min_p`` may each be a tensor with one value per row (held in float32 and int32).

    ``uniforms`` [...] float64 in [0, 1); without it u comes from the library's Philox stream, counters (row, step) with
    the rows numbered from ``row_offset``.  ``uncond_logits`` (same shape): combined with ``cfg_scale`` first, as
    generate.py:89-90 does.  ``return_probs``: also the tokens' probabilities among the kept entries (float32).

    Entries of -inf cost nothing; a row with a finite magnitude of 256 or more (a vocabulary masked with -1e4, say) takes about
    ten times as long as others."""
    if logits.dtype != torch.bfloat16 or not logits.is_cuda or logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError("logits: a bfloat16 GPU tensor [..., vocab] is wanted")
    lib, dev = _lib.load(), logits.device
    lead, vocab = logits.shape[:-1], logits.shape[-1]
    rows = logits if logits.dim() == 2 else logits.reshape(-1, vocab)
    n = rows.shape[0]
    if n > TOP_K_MAX:
        raise ValueError(f"{n} rows: they are counted in 32 bits")
    if rows.stride(1) != 1 and vocab > 1 or (n > 1 and rows.stride(0) < vocab):
        rows = rows.contiguous()
    stride = rows.stride(0) if n > 1 else vocab
    un = None
    if uncond_logits is not None:
        if uncond_logits.shape != logits.shape or uncond_logits.dtype != torch.bfloat16 or uncond_logits.device != dev:
            raise ValueError("uncond_logits: the shape, type and device of logits are wanted")
        un = uncond_logits.reshape(-1, vocab)
        if un.stride() != rows.stride() or (un.data_ptr() - rows.data_ptr()) % 16:
            rows, un, stride = rows.clone(memory_format=torch.contiguous_format), un.clone(memory_format=torch.contiguous_format), vocab
    arrays, keep = [None] * 4, []
    scalars = [temperature, _top_k(top_k), top_p, min_p]
    for i, (v, dtype, off) in enumerate(zip(scalars, (torch.float32, torch.int32, torch.float32, torch.float32), (1.0, 0, 1.0, 0.0))):
        if isinstance(v, torch.Tensor):
            if v.dim() and v.shape != lead:
                raise ValueError(f"a sampling parameter has shape {list(v.shape)}, the rows {list(lead)}")
            keep.append(v.to(device=dev, dtype=dtype).expand(lead).reshape(-1).contiguous())
            arrays[i], scalars[i] = keep[-1].data_ptr(), off
    t, k, p, q = scalars
    u = None
    if uniforms is not None:
        if uniforms.shape != lead or uniforms.device != dev:
            raise ValueError(f"uniforms: shape {list(lead)} on {dev} is wanted")
        u = uniforms if uniforms.dtype == torch.float64 and uniforms.is_contiguous() else uniforms.to(torch.float64).contiguous()
    with _lib.on_device(dev):
        tokens = torch.empty(lead, dtype=torch.int64, device=dev)
        probs = torch.empty(lead, dtype=torch.float32, device=dev) if return_probs else None
        if n:
            s = _lib.Sampling(float(t), float(p), float(q), k, *arrays, _lib.ptr(u))
            _lib.check(lib.llada_sample_rows(rows.data_ptr(), _lib.ptr(un), stride, float(cfg_scale), n, vocab, C.byref(s), seed, step,
                                             row_offset, tokens.data_ptr(), _lib.ptr(probs), _lib.stream_ptr(dev.index)))
    return (tokens, probs) if return_probs else tokens
