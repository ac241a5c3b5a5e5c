"""The operators of a block-cached, sampling denoise step, as they are measured.

Three operators, each in its plain form (elementary torch operations) and, where ``own`` is true, as the
calls a user makes of the framework:

``fill`` / ``update``  keys and values [n_seq, len, 3 d] (bf16 [Q | K | V] rows) written into a cache that holds them
    in 8 bits, one power-of-two scale for each 64-token block and head, for keys and for values; returned as the
    values the cache stands for.  scale = 2^k, k the smallest integer with amax <= 448 * 2^k (e4m3) or
    127 * 2^k (int8); amax over the block's unmasked tokens; code = round-to-nearest-even(x * 2^-k); a masked token
    is stored as zero.  An update takes the block's other tokens as the cache holds them.
``attend``  attention of n_q queries a sequence over such a cache, without a causal mask, the rows
    block_start .. block_start + len - 1 taken from fresh bf16 rows instead: softmax(q k^T / sqrt(128)) v.
``sample``  one token a row of logits from the distribution truncated by top-k, then top-p, then min-p, at a temperature,
    by inversion of given uniforms: entries ordered by (logit descending, index ascending), the token at which the
    running mass of the kept entries first exceeds u times their total.
"""
import math

import torch

own = False

HD = 128          # head dimension
TB = 64           # tokens of a scale block
VOCAB = 126464    # the framework's default configuration


def listed():
    return [
        # writing the cache: one short prompt's layer, a batch of long sequences, the left-padded batch of a harness,
        # a block of odd length in the middle of odd sequences
        {"name": "fill 1x384", "op": "fill", "n_seq": 1, "len": 384, "heads": 32, "dtype": "e4m3", "pad": 0},
        {"name": "fill 16x4096", "op": "fill", "n_seq": 16, "len": 4096, "heads": 32, "dtype": "e4m3", "pad": 0},
        {"name": "update 8x1150 int8", "op": "update", "n_seq": 8, "len": 1150, "heads": 32, "dtype": "int8", "pad": 1, "start": 509, "n_new": 37},
        # cached denoise steps: one prompt (latency), the benchmark's eight, a padded batch with a wide block, many long
        # sequences (bandwidth), everything right of a cached prefix (arithmetic), single queries over an odd length
        {"name": "attend 1x384 q32", "op": "attend", "n_seq": 1, "len": 384, "heads": 32, "dtype": "e4m3", "pad": 0, "start": 192, "n_q": 32, "fresh": True},
        {"name": "attend 8x384 q32", "op": "attend", "n_seq": 8, "len": 384, "heads": 32, "dtype": "e4m3", "pad": 0, "start": 160, "n_q": 32, "fresh": True},
        {"name": "attend 8x1150 q64 int8", "op": "attend", "n_seq": 8, "len": 1150, "heads": 32, "dtype": "int8", "pad": 1, "start": 515, "n_q": 64, "fresh": True},
        {"name": "attend 32x4096 q32", "op": "attend", "n_seq": 32, "len": 4096, "heads": 32, "dtype": "e4m3", "pad": 0, "start": 2048, "n_q": 32, "fresh": True},
        {"name": "attend 8x769 q321", "op": "attend", "n_seq": 8, "len": 769, "heads": 32, "dtype": "e4m3", "pad": 0, "start": 448, "n_q": 321, "fresh": True},
        {"name": "attend 5x2049 q1 int8", "op": "attend", "n_seq": 5, "len": 2049, "heads": 32, "dtype": "int8", "pad": 1, "start": 0, "n_q": 1, "fresh": False},
        # candidates of a step: one prompt's block, eight prompts' under guidance, a large batch
        {"name": "sample 32", "op": "sample", "rows": 32, "vocab": VOCAB, "temperature": 0.7, "top_k": 50, "top_p": 0.95, "min_p": 0.0, "cfg": 0.0},
        {"name": "sample 256 guided", "op": "sample", "rows": 256, "vocab": VOCAB, "temperature": 1.0, "top_k": 0, "top_p": 0.9, "min_p": 0.0, "cfg": 1.5},
        {"name": "sample 2048", "op": "sample", "rows": 2048, "vocab": VOCAB, "temperature": 0.8, "top_k": 0, "top_p": 1.0, "min_p": 0.02, "cfg": 0.0},
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["fill", "update", "attend", "attend", "attend", "sample", "sample"])
    if op == "sample":
        return {"op": op, "rows": _spread(rng, 1, 1500), "vocab": rng.choice([VOCAB, VOCAB, _spread(rng, 40, VOCAB)]),
                "temperature": round(rng.uniform(0.2, 1.8), 3), "top_k": rng.choice([0, 1, 20, 200, 5000]),
                "top_p": rng.choice([1.0, 0.5, 0.9, 0.99]), "min_p": rng.choice([0.0, 0.0, 0.05, 0.3]), "cfg": rng.choice([0.0, 0.0, 2.0])}
    heads, length, n_seq = rng.choice([2, 5, 16, 32]), _spread(rng, 1, 4096), _spread(rng, 1, 16)
    case = {"op": op, "n_seq": n_seq, "len": length, "heads": heads, "dtype": rng.choice(["e4m3", "int8"]), "pad": rng.choice([0, 1])}
    if op == "update":
        case["start"] = rng.randrange(length)
        case["n_new"] = _spread(rng, 1, length - case["start"])
    if op == "attend":
        case["n_q"] = _spread(rng, 1, min(length, 500))
        case["start"] = rng.randrange(length - case["n_q"] + 1)
        case["fresh"] = rng.choice([True, True, False])
    return case


def work(case):
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        return {"bytes": rows * vocab * (4 if case["cfg"] else 2) + rows * 20, "flops": 0}
    n, d = case["n_seq"], case["heads"] * HD
    all_tokens = n * case["len"]
    blocks = n * case["heads"] * -(-case["len"] // TB) * 2
    if case["op"] == "fill":      # rows read, codes and scales written, values returned
        return {"bytes": all_tokens * d * (4 + 2 + 4) + blocks * 4, "flops": 0}
    if case["op"] == "update":    # fresh rows read, the touched blocks' codes read and written, the whole layer returned
        first, last = case["start"] // TB, (case["start"] + case["n_new"] - 1) // TB
        touched = n * (min(case["len"], (last + 1) * TB) - first * TB)
        return {"bytes": n * case["n_new"] * d * 4 + touched * d * 4 + all_tokens * d * (2 + 4), "flops": 0}
    fresh = case["n_q"] if case["fresh"] else 0
    keys = n * (case["len"] - fresh)
    return {"bytes": keys * d * 2 + blocks * 4 + n * fresh * d * 4 + n * case["n_q"] * d * 4,
            "flops": 4 * n * case["n_q"] * case["len"] * d}


# ---- inputs ---------------------------------------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 13)


def _rows(g, n_seq, length, heads):
    """[Q | K | V] rows as a projection leaves them: some channels of the keys much larger than the rest."""
    d = heads * HD
    x = torch.randn((n_seq, length, 3 * d), generator=g, device="cuda", dtype=torch.bfloat16)
    channel = torch.ones(3 * d, device="cuda")
    channel[d:2 * d] = torch.exp(0.7 * torch.randn(d, generator=g, device="cuda"))
    channel[2 * d:] = 0.5
    return x.mul_(channel.to(torch.bfloat16))


def _mask(case):
    """Left padding: sequence i starts with some masked tokens (at least one token stays)."""
    if not case["pad"]:
        return None
    n, length = case["n_seq"], case["len"]
    gap = (torch.arange(n, device="cuda") * max(1, length // (2 * n))) % max(1, length)
    return (torch.arange(length, device="cuda")[None, :] >= gap[:, None]).to(torch.uint8)


def _inputs(case, seed):
    g = _generator(seed)
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        s = {"logits": torch.randn((rows, vocab), generator=g, device="cuda", dtype=torch.bfloat16).mul_(2.2)}
        likely = torch.rand((rows, vocab), generator=g, device="cuda") * (vocab / 200.0)   # a head of likely tokens over the bulk
        s["logits"] += torch.where(likely < 1.0, 4.0 + 4.0 * likely ** 2, torch.zeros_like(likely)).to(torch.bfloat16)
        del likely
        s["uncond"] = None
        if case["cfg"]:
            s["uncond"] = (s["logits"] + 0.5 * torch.randn((rows, vocab), generator=g, device="cuda", dtype=torch.bfloat16))
        s["u"] = torch.rand(rows, generator=g, device="cuda", dtype=torch.float64)
        return s
    s = {"rows": _rows(g, case["n_seq"], case["len"], case["heads"]), "mask": _mask(case)}
    if case["op"] == "update":
        s["new"] = _rows(g, case["n_seq"], case["n_new"], case["heads"])
    if case["op"] == "attend":
        s["new"] = _rows(g, case["n_seq"], case["n_q"], case["heads"])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["op"] in ("update", "attend"):      # the cache that earlier steps left
        rows = s.pop("rows")
        if own:
            from llada_amd import KVCache8
            s["cache"] = KVCache8(case["n_seq"], case["len"], case["heads"], dtype=case["dtype"], device="cuda")
            s["cache"].fill(0, rows, s["mask"])
        else:
            s["held"] = [_quantised(x, s["mask"], case["dtype"]) for x in _kv(rows, case["heads"])]
    elif own and case["op"] == "fill":
        from llada_amd import KVCache8
        s["cache"] = KVCache8(case["n_seq"], case["len"], case["heads"], dtype=case["dtype"], device="cuda")
    return s


# ---- plain forms ----------------------------------------------------------------------------------------------


def _kv(rows, heads):
    n, length, _ = rows.shape
    x = rows.view(n, length, 3, heads, HD)
    return x[:, :, 1], x[:, :, 2]


def _quantised(x, mask, dtype):
    """x [n, length, heads, HD] -> (codes [n, blocks, TB, heads, HD], scales [n, blocks, 1, heads, 1])."""
    n, length, heads, _ = x.shape
    blocks = -(-length // TB)
    x = x.float()
    if mask is not None:
        x = torch.where(mask.bool()[:, :, None, None], x, torch.zeros((), device=x.device))
    x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, blocks * TB - length)).view(n, blocks, TB, heads, HD)
    m, e = torch.frexp(x.abs().amax(dim=(2, 4), keepdim=True))        # amax = m * 2^e, 0.5 <= m < 1
    if dtype == "e4m3":                                               # 448 = 0.875 * 2^9
        k = e - 9 + (m > 0.875)
    else:                                                             # 127 = 0.9921875 * 2^7
        k = e - 7 + (m > 0.9921875)
    k = torch.where(m == 0, torch.zeros_like(k), k.clamp(min=-126))
    scale = ((k + 127) << 23).to(torch.int32).view(torch.float32)     # 2^k, exactly
    y = x / scale
    codes = y.to(torch.float8_e4m3fn) if dtype == "e4m3" else torch.round(y).to(torch.int8)
    return codes, scale


def _values(held, length):
    codes, scale = held
    n, blocks, _, heads, _ = codes.shape
    return (codes.float() * scale).view(n, blocks * TB, heads, HD)[:, :length]


def _plain_attend(s):
    case = s["case"]
    n, length, heads, n_q, start = case["n_seq"], case["len"], case["heads"], case["n_q"], case["start"]
    k, v = (_values(h, length) for h in s["held"])
    if case["fresh"]:
        fk, fv = _kv(s["new"], heads)
        k[:, start:start + n_q], v[:, start:start + n_q] = fk.float(), fv.float()
    if s["mask"] is not None:
        v = torch.where(s["mask"].bool()[:, :, None, None], v, torch.zeros((), device=v.device))
    q = s["new"].view(n, n_q, 3, heads, HD)[:, :, 0].float()
    k, v, q = (x.transpose(1, 2).contiguous() for x in (k, v, q))
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) / math.sqrt(HD)
    if s["mask"] is not None:
        score = score.masked_fill(~s["mask"].bool()[:, None, None, :], -math.inf)
    top = score.amax(dim=3, keepdim=True)
    p = torch.exp(score - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(dim=3, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    return torch.matmul(p, v).transpose(1, 2).reshape(n, n_q, heads * HD).to(torch.bfloat16)


def _plain_sample(s):
    case, logits = s["case"], s["logits"]
    if case["cfg"]:                                     # as the sampler combines: every operation rounded to bf16
        logits = s["uncond"] + (logits - s["uncond"]) * (case["cfg"] + 1.0)
    ordered, index = torch.sort(logits.float(), dim=1, descending=True, stable=True)
    w = ordered.double()
    w = torch.exp((w - w[:, :1]) / case["temperature"])
    mass = torch.cumsum(w, dim=1)
    vocab = w.shape[1]
    kept = torch.full((w.shape[0], 1), min(case["top_k"] or vocab, vocab), device=w.device)
    if case["top_p"] < 1.0:
        enough = case["top_p"] * mass.gather(1, kept - 1)
        kept = torch.minimum(kept, (mass < enough).sum(dim=1, keepdim=True) + 1)
    if case["min_p"] > 0.0:
        kept = torch.minimum(kept, (w >= case["min_p"]).sum(dim=1, keepdim=True))
    total = mass.gather(1, kept - 1)
    at = torch.minimum((mass <= s["u"][:, None] * total).sum(dim=1, keepdim=True), kept - 1)
    return {"token": index.gather(1, at)[:, 0], "prob": (w.gather(1, at) / total)[:, 0].float()}


def run(s):
    case = s["case"]
    if case["op"] == "sample":
        if own:
            from llada_amd import sample_tokens
            token, prob = sample_tokens(s["logits"], case["temperature"], top_k=case["top_k"], top_p=case["top_p"], min_p=case["min_p"],
                                        uniforms=s["u"], uncond_logits=s["uncond"], cfg_scale=case["cfg"], return_probs=True)
            return {"token": token, "prob": prob}
        return _plain_sample(s)
    if case["op"] == "attend":
        if own:
            return s["cache"].attend(0, s["new"], s["mask"], block=s["new"] if case["fresh"] else None, block_start=case["start"])
        return _plain_attend(s)
    if own:
        if case["op"] == "fill":
            s["cache"].fill(0, s["rows"], s["mask"])
        else:
            s["cache"].update(0, s["new"], case["start"], s["mask"])
        k, v = s["cache"].read(0)
        return {"k": k, "v": v}
    length, heads = case["len"], case["heads"]
    if case["op"] == "fill":
        held = [_quantised(x, s["mask"], case["dtype"]) for x in _kv(s["rows"], heads)]
    else:
        held = []
        begin, end = case["start"] // TB, -(-(case["start"] + case["n_new"]) // TB)
        for old, new in zip(s["held"], _kv(s["new"], heads)):
            x = _values(old, length)[:, begin * TB:end * TB]
            x[:, case["start"] - begin * TB:case["start"] - begin * TB + case["n_new"]] = new.float()
            part = None if s["mask"] is None else s["mask"][:, begin * TB:end * TB]
            codes, scale = _quantised(x, part, case["dtype"])
            old[0].view(torch.uint8)[:, begin:end] = codes.view(torch.uint8)
            old[1][:, begin:end] = scale
            held.append(old)
    return {name: _values(h, length).to(torch.bfloat16) for name, h in zip("kv", held)}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------


def _power_of_two(k):
    return ((k.long() + 1023) << 52).view(torch.float64)


def _held_exactly(x, mask, dtype):
    """The values a cache stands for, [n, length, heads, HD] in 64 bits, from the definition."""
    top, low = (448.0, 2.0 ** -9) if dtype == "e4m3" else (127.0, 1.0)
    out = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    for t in range(0, x.shape[1], TB):
        part = x[:, t:t + TB].double()
        if mask is not None:
            part = part * mask[:, t:t + TB, None, None].double()
        amax = part.abs().amax(dim=(1, 3), keepdim=True)
        m, e = torch.frexp(torch.where(amax > 0, amax, torch.full_like(amax, top)) / top)
        unit = _power_of_two((e - (m == 0.5).int()).clamp(min=-126))      # the smallest power with amax <= top * unit
        y = part / unit
        if dtype == "e4m3":      # three bits after the leading one; below 2^-6 steps of 2^-9
            step = _power_of_two((torch.frexp(y.abs().clamp(min=low))[1] - 1).clamp(min=-6) - 3)
        else:
            step = torch.ones_like(y)
        out[:, t:t + TB] = torch.round(y / step) * step * unit
    return out


def _exact_attend(case, s):
    n, length, heads, n_q, start = case["n_seq"], case["len"], case["heads"], case["n_q"], case["start"]
    out = torch.zeros((n, n_q, heads, HD), dtype=torch.float64, device="cuda")
    for i in range(n):
        mask = None if s["mask"] is None else s["mask"][i:i + 1]
        k, v = (_held_exactly(x[i:i + 1], mask, case["dtype"])[0] for x in _kv(s["rows"], heads))
        if case["fresh"]:
            fk, fv = _kv(s["new"][i:i + 1], heads)
            k[start:start + n_q], v[start:start + n_q] = fk[0].double(), fv[0].double()
        keep = slice(None) if mask is None else mask[0].bool()
        q = s["new"][i].view(n_q, 3, heads, HD)[:, 0].double()
        k, v = k[keep], v[keep]
        for h in range(heads):
            out[i, :, h] = torch.softmax(q[:, h] @ k[:, h].T * HD ** -0.5, dim=1) @ v[:, h]
    return out.reshape(n, n_q, heads * HD)


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "attend":
        return _exact_attend(case, s)
    if case["op"] == "sample":
        tokens, probs = [], []
        for r in range(case["rows"]):
            l = s["logits"][r]
            if case["cfg"]:
                l = s["uncond"][r] + (l - s["uncond"][r]) * (case["cfg"] + 1.0)
            l = l.double()
            values, index = torch.sort(l, descending=True, stable=True)
            p = torch.softmax(values / case["temperature"], dim=0)
            if case["top_k"]:
                p = p[:case["top_k"]] / p[:case["top_k"]].sum()
            ratio = p / p[0]
            if case["top_p"] < 1.0:
                p = p[:int((torch.cumsum(p, 0) < case["top_p"]).sum()) + 1]
            p = p[ratio[:len(p)] >= case["min_p"]]
            p = p / p.sum()
            at = min(int((torch.cumsum(p, 0) <= s["u"][r]).sum()), len(p) - 1)
            tokens.append(index[at])
            probs.append(p[at])
        return {"token": torch.stack(tokens), "prob": torch.stack(probs)}
    held = [_held_exactly(x, s["mask"], case["dtype"]) for x in _kv(s["rows"], case["heads"])]
    if case["op"] == "update":
        a = case["start"] // TB * TB
        b = min(case["len"], -(-(case["start"] + case["n_new"]) // TB) * TB)
        for x, new in zip(held, _kv(s["new"], case["heads"])):
            x[:, case["start"]:case["start"] + case["n_new"]] = new.double()
            x[:, a:b] = _held_exactly(x[:, a:b], None if s["mask"] is None else s["mask"][:, a:b], case["dtype"])
    return {"k": held[0], "v": held[1]}
