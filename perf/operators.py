"""Timed cases of the operators that serve a model from packed block formats, and their plain forms.

Three operators, as a program that answers with a quantised model calls them:

* ``linear``     y = x W^T + b with W held as packed E2M1 codes and group scales (MXFP4 or NVFP4);
* ``cache``      new K and V rows are quantised into the pages of an MX cache and read back;
* ``attention``  a chunk of new tokens (or one) attends to what the paged MX cache holds.

``listed()`` gives the fixed cases, ``draw(rng)`` more of the same ranges, ``prepare`` what a program has in hand before
the call, ``run`` one pass, ``work`` what a pass cannot do without and ``exact`` the result in 64 bits.

The cache is four tensors, ``[pages, kv_heads, page, ...]``: codes of K, scales of K, codes of V, scales of V.  A sequence's
tokens lie in the pages that its row of the page table names; entries behind its last page are -1.  ``lens`` counts the
tokens of a sequence with the new ones; ``starts`` (ragged batches) says where each sequence's new rows begin.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


# ------------------------------------------------------------------------------------------------------- the cases
def _linear(name, rows, n_in, n_out, fmt, dtype, bias=False):
    return {"name": name, "kind": "linear", "rows": rows, "n_in": n_in, "n_out": n_out, "format": fmt, "dtype": dtype, "bias": bias}


def _cache(name, seqs, new, context, kv_heads, head_dim, elem, dtype, page=16, ragged=False):
    return {"name": name, "kind": "cache", "seqs": seqs, "new": new, "context": context, "kv_heads": kv_heads,
            "head_dim": head_dim, "elem": elem, "dtype": dtype, "page": page, "ragged": ragged}


def _attention(name, seqs, new, context, heads, kv_heads, head_dim, elem, dtype, page=16, ragged=False, window=0, sinks=0):
    return {"name": name, "kind": "attention", "seqs": seqs, "new": new, "context": context, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "elem": elem, "dtype": dtype, "page": page, "ragged": ragged, "window": window, "sinks": sinks}


def listed():
    return [
        # the attention projection of the GPT-2-shaped block for one token: latency
        _linear("linear_one_small", 1, 768, 2304, "mxfp4", "fp32", bias=True),
        # one token through a wide projection: the weights' bytes
        _linear("linear_one_wide", 1, 8192, 28672, "nvfp4", "bf16"),
        # the vocabulary head of that block for three tokens, an odd number of outputs
        _linear("linear_head_odd", 3, 768, 50257, "mxfp4", "fp32"),
        # a batch of sequences that answer together, not a multiple of a tile
        _linear("linear_batch", 37, 4096, 11008, "nvfp4", "fp16", bias=True),
        # a prompt
        _linear("linear_prompt", 1024, 4096, 4096, "mxfp4", "fp32"),
        # one new token for each of 32 sequences of the GPT-2-shaped block
        _cache("cache_token", 32, 1, 1024, 12, 64, "e4m3", "fp32"),
        # prompts of different lengths written into 4-bit pages
        _cache("cache_prompts", 7, 4096, 4096, 8, 128, "e2m1", "bf16", page=64, ragged=True),
        # a few sequences, one token each, in the GPT-2 shape: latency
        _attention("attention_token_small", 4, 1, 1024, 12, 12, 64, "e4m3", "fp32"),
        # one token for each of 16 long contexts of different lengths, grouped heads: the cache's bytes
        _attention("attention_token_long", 16, 1, 32768, 32, 8, 128, "e4m3", "bf16", page=64),
        # one token over a sliding window with a few sinks, 4-bit pages
        _attention("attention_token_window", 96, 1, 8192, 24, 8, 96, "e2m1", "fp16", page=32, window=1024, sinks=4),
        # a chunk of a prompt over the pages before it: the largest
        _attention("attention_chunk", 2, 1024, 8192, 32, 8, 128, "e4m3", "bf16", page=64),
        # chunks of different lengths (some a single token) in one batch
        _attention("attention_chunk_ragged", 6, 300, 2000, 12, 12, 64, "e4m3", "fp32", page=16, ragged=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return w["bytes"] / 6.5e12 + w["flops"] / 1.6e15


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(["linear", "linear", "cache", "attention", "attention", "attention"])
        dtype = rng.choice(["fp32", "bf16", "fp16"])
        if kind == "linear":
            rows = _log_int(rng, 1, 64) if rng.random() < 0.8 else _log_int(rng, 64, 1500)
            case = _linear("", rows, 32 * _log_int(rng, 2, 300), _log_int(rng, 16, 33000), rng.choice(["mxfp4", "nvfp4"]), dtype,
                           rng.random() < 0.5)
        else:
            page, elem = rng.choice([16, 32, 64, 128]), rng.choice(["e4m3", "e2m1"])
            head_dim, kv_heads = rng.choice([32, 64, 64, 96, 128, 128, 192, 256]), rng.choice([1, 2, 3, 4, 8, 12])
            ragged = rng.random() < 0.5
            if kind == "cache":
                new = _log_int(rng, 1, 5000)
                case = _cache("", _log_int(rng, 1, 64), new, max(new, _log_int(rng, 1, 9000)), kv_heads, head_dim, elem, dtype, page, ragged)
                rows = sum(_lengths(case)[0])
                if rows * kv_heads * head_dim > 1 << 25:
                    continue
            else:
                new = 1 if rng.random() < 0.5 else _log_int(rng, 2, 1200)
                context = max(new, _log_int(rng, 1, 20000))
                window = rng.choice([0, 0, 0, _log_int(rng, 16, 4096)])
                case = _attention("", _log_int(rng, 1, 64), new, context, kv_heads * rng.choice([1, 1, 2, 3, 4, 8]), kv_heads, head_dim,
                                  elem, dtype, page, ragged, window, rng.choice([0, 4, 17]) if window else 0)
                # the plain form holds every score and the whole cache in 32 bits
                if case["seqs"] * case["heads"] * new * context > 1 << 29 or case["seqs"] * kv_heads * context * head_dim > 1 << 29:
                    continue
        if _cost(case) <= most:
            del case["name"]
            return case


def _lengths(case):
    """Tokens that are new, and tokens in all, of each sequence: spread over what the case allows, the first at its most."""
    b = case["seqs"]
    share = [1.0 if i == 0 else ((5 * i + 3) % b + 1) / b for i in range(b)]
    new = [max(1, int(case["new"] * share[-1 - i])) for i in range(b)] if case["ragged"] else [case["new"]] * b
    return new, [max(n, int(case["context"] * s)) for n, s in zip(new, share)]


# ------------------------------------------------------------------------------------------------------- the inputs
def _round_to(v, elem):
    """``v`` rounded to nearest even in E4M3 (largest 448) or E2M1 (largest 6), with saturation."""
    low, man, top = (-6, 3, 448.0) if elem == "e4m3" else (0, 1, 6.0)
    a = v.abs()
    quantum = torch.exp2((torch.frexp(a)[1] - 1).clamp(min=low).float() - man)
    return torch.where(v < 0, -1.0, 1.0) * (torch.round(a / quantum) * quantum).clamp(max=top)


_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _encode(r, elem):
    """Packed codes of values that the format holds."""
    if elem == "e4m3":
        return r.to(torch.float8_e4m3fn).view(torch.uint8)
    n = torch.bucketize(r.abs(), torch.tensor(_E2M1, device=r.device))
    n = (n + 8 * (torch.signbit(r)).long()).to(torch.uint8)
    return n[..., 0::2] | (n[..., 1::2] << 4)


def _decode(codes, elem):
    """The values that packed codes stand for, in 32 bits."""
    if elem == "e4m3":
        return codes.view(torch.float8_e4m3fn).float()
    one = torch.tensor(_E2M1 + tuple(-x for x in _E2M1), device=codes.device)
    both = torch.stack([one.repeat(16), one.repeat_interleave(16)], dim=1)
    return both[codes.long()].flatten(-2)


def _power(scales):
    return torch.exp2(scales.float() - 127.0)


def _mx(x, elem):
    """Codes and scale bytes of ``x`` in blocks of 32 along its last dimension."""
    blocks = x.float().unflatten(-1, (-1, 32))
    amax = blocks.abs().amax(-1)
    e = (torch.frexp(amax)[1] - 1 - (8 if elem == "e4m3" else 2)).clamp(-127, 127)
    e = torch.where(amax == 0, -127, e)
    r = _round_to(blocks * torch.exp2(-e.float())[..., None], elem)
    return _encode(r.flatten(-2), elem), (e + 127).to(torch.uint8)


def _nvfp4(x):
    """Codes, E4M3 scale bytes and the tensor scale of ``x``, blocks of 16 along its last dimension."""
    glob = x.abs().amax() / (448.0 * 6.0)
    blocks = x.unflatten(-1, (-1, 16))
    s = _round_to(blocks.abs().amax(-1) / (6.0 * glob), "e4m3")
    r = _round_to(torch.where(s[..., None] == 0, 0.0, blocks / (s * glob).clamp(min=1e-38)[..., None]), "e2m1")
    return _encode(r.flatten(-2), "e2m1"), s.to(torch.float8_e4m3fn).view(torch.uint8), glob.reshape(1)


def _activations(shape, gen):
    """Normal values with a few channels some ten times larger, as activations have them."""
    x = torch.randn(shape, device=DEV, generator=gen)
    return x * torch.where(torch.rand(shape[-1], device=DEV, generator=gen) < 0.02, 12.0, 1.0)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    state = {"case": case}
    if case["kind"] == "linear":
        n, k = case["n_out"], case["n_in"]
        w = torch.randn(n, k, device=DEV, generator=gen) * 0.02
        if case["format"] == "mxfp4":
            state["codes"], state["scales"] = _mx(w, "e2m1")
        else:
            state["codes"], state["scales"], state["global"] = _nvfp4(w)
        state["x"] = _activations((case["rows"], k), gen).to(dtype)
        state["bias"] = (0.1 * torch.randn(n, device=DEV, generator=gen)).to(dtype) if case["bias"] else None
        return state
    new, lens = _lengths(case)
    b, h, d, page, elem = case["seqs"], case["kv_heads"], case["head_dim"], case["page"], case["elem"]
    counts = [-(-x // page) for x in lens]
    width, total = max(counts), sum(counts) + 3
    # the pages of a sequence lie anywhere in the cache
    order = torch.randperm(total, device=DEV, generator=gen).to(torch.int32)
    ends = torch.tensor(counts, device=DEV).cumsum(0)
    at = torch.arange(width, device=DEV)
    left = torch.tensor(counts, device=DEV)[:, None]
    state["pages"] = torch.where(at < left, order[(ends[:, None] - left + at).clamp(max=total - 1)], -1).to(torch.int32)
    state["lens"] = torch.tensor(lens, device=DEV, dtype=torch.int32)
    state["starts"] = torch.tensor([0] + new, device=DEV).cumsum(0).to(torch.int32) if case["ragged"] else None
    lead = (sum(new),) if case["ragged"] else (b, case["new"])
    if case["kind"] == "cache":
        width_b = d if elem == "e4m3" else d // 2
        zeros = [torch.zeros(total, h, page, x, device=DEV, dtype=torch.uint8) for x in (width_b, d // 32)]
        state["cache"] = (zeros[0], zeros[1], zeros[0].clone(), zeros[1].clone())
        state["k"] = _activations(lead + (h, d), gen).to(dtype)
        state["v"] = torch.randn(lead + (h, d), device=DEV, generator=gen).to(dtype)
    else:
        k = _mx(_activations((total, h, page, d), gen), elem)
        v = _mx(torch.randn(total, h, page, d, device=DEV, generator=gen), elem)
        state["cache"] = (*k, *v)
        state["q"] = torch.randn(lead + (case["heads"], d), device=DEV, generator=gen).to(dtype)
    return state


# ------------------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if own:
        import mptorch_b200.quant as quant

        if case["kind"] == "linear":
            if case["format"] == "mxfp4":
                return quant.mx_linear(state["x"], state["codes"], state["scales"], state["bias"])
            return quant.nvfp4_linear(state["x"], state["codes"], state["scales"], state["global"], state["bias"])
        cache, pages, lens, starts = (state[x] for x in ("cache", "pages", "lens", "starts"))
        if case["kind"] == "cache":
            quant.mx_cache_write(state["k"], state["v"], cache, pages, lens, starts)
            new = state["k"].shape[0] if case["ragged"] else case["new"]
            return quant.mx_cache_read(cache, pages, lens, new, starts, dtype=state["k"].dtype)
        return quant.mx_attention(state["q"], cache, pages, lens, starts, window=case["window"], sinks=case["sinks"])
    return {"linear": _plain_linear, "cache": _plain_cache, "attention": _plain_attention}[case["kind"]](state)


def _plain_linear(state):
    x, scales = state["x"], state["scales"]
    if state["case"]["format"] == "mxfp4":
        s, group = _power(scales), 32
    else:
        s, group = scales.view(torch.float8_e4m3fn).float() * state["global"], 16
    w = (_decode(state["codes"], "e2m1").unflatten(-1, (-1, group)) * s[..., None]).flatten(-2)
    y = torch.matmul(x.float(), w.t())
    return (y if state["bias"] is None else y + state["bias"].float()).to(x.dtype)


def _rows(state, shape):
    """For each new row (sequence, place in the sequence), as tensors of the rows' leading shape."""
    starts, lens = state["starts"], state["lens"].long()
    if starts is None:
        b, n = shape[:2]
        seq = torch.arange(b, device=DEV)[:, None].expand(b, n)
        return seq, lens[:, None] - n + torch.arange(n, device=DEV)
    row = torch.arange(shape[0], device=DEV)
    seq = torch.bucketize(row, starts[1:].long(), right=True)
    return seq, lens[seq] - starts.long()[seq + 1] + row


def _plain_cache(state):
    case, k, v = state["case"], state["k"], state["v"]
    seq, pos = _rows(state, k.shape)
    page = state["pages"].long()[seq, pos // case["page"]]
    cache, off, back = state["cache"], pos % case["page"], []
    for x, codes, scales in ((k, cache[0], cache[1]), (v, cache[2], cache[3])):
        c, s = _mx(x, case["elem"])
        codes[page, :, off], scales[page, :, off] = c, s
        y = _decode(codes[page, :, off], case["elem"]).unflatten(-1, (-1, 32)) * _power(scales[page, :, off])[..., None]
        back.append(y.flatten(-2).to(x.dtype))
    return tuple(back)


def _plain_attention(state):
    case, q, starts = state["case"], state["q"], state["starts"]
    h, d, g = case["kv_heads"], case["head_dim"], case["heads"] // case["kv_heads"]
    pages, lens = state["pages"].long().clamp(min=0), state["lens"].long()
    k, v = (((_decode(c[pages], case["elem"]).unflatten(-1, (-1, 32)) * _power(s[pages])[..., None]).flatten(-2))
            .transpose(1, 2).flatten(2, 3) for c, s in (state["cache"][:2], state["cache"][2:]))      # [seqs, kv_heads, tokens, d]
    if starts is None:
        n, qs = torch.full_like(lens, q.shape[1]), q
        most = q.shape[1]
    else:
        n, most = starts[1:].long() - starts[:-1].long(), case["new"]
        at = (starts[:-1].long()[:, None] + torch.arange(most, device=DEV)).clamp(max=q.shape[0] - 1)
        qs = q[at]
    qs = qs.float().unflatten(2, (h, g)).permute(0, 2, 1, 3, 4).flatten(2, 3)                           # [seqs, kv_heads, new * g, d]
    s = torch.matmul(qs, k.transpose(-1, -2)) * (1.0 / math.sqrt(d))
    p = (lens - n)[:, None] + torch.arange(most, device=DEV)
    t = torch.arange(k.shape[2], device=DEV)
    seen = t <= p[..., None]
    if case["window"]:
        seen &= (t > p[..., None] - case["window"]) | (t < case["sinks"])
    seen = seen.repeat_interleave(g, dim=1)[:, None]
    s = s.masked_fill_(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    s = s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    o = torch.matmul(s, v) / s.sum(-1, keepdim=True).clamp(min=1e-30)
    o = o.unflatten(2, (most, g)).permute(0, 2, 1, 3, 4).flatten(2, 3).to(q.dtype)
    if starts is None:
        return o
    row = torch.arange(q.shape[0], device=DEV)
    seq = torch.bucketize(row, starts[1:].long(), right=True)
    return o[seq, row - starts.long()[seq]]


# ------------------------------------------------------------------------------------------------------- its work
def work(case):
    size = SIZE[case["dtype"]]
    if case["kind"] == "linear":
        m, n, k = case["rows"], case["n_out"], case["n_in"]
        weights = n * k // 2 + n * k // (32 if case["format"] == "mxfp4" else 16)
        return {"bytes": weights + size * (m * k + m * n + (n if case["bias"] else 0)), "flops": 2 * m * n * k}
    new, lens = _lengths(case)
    h, d = case["kv_heads"], case["head_dim"]
    row = (d if case["elem"] == "e4m3" else d // 2) + d // 32
    if case["kind"] == "cache":
        return {"bytes": 2 * sum(new) * h * (2 * d * size + row), "flops": 2 * sum(new) * h * d * 4}
    window, sinks = case["window"], case["sinks"]
    tokens = pairs = 0
    for n, length in zip(new, lens):
        for p in range(length - n, length):
            low = max(0, p - window + 1) if window else 0
            pairs += p + 1 - low + min(sinks, low)
        low = max(0, length - n - window + 1) if window else 0
        tokens += length - low + min(sinks, low)
    return {"bytes": 2 * tokens * h * row + 2 * sum(new) * case["heads"] * d * size + 4 * len(lens) * (1 + max(lens) // case["page"]),
            "flops": 4 * pairs * case["heads"] * d}


# ------------------------------------------------------------------------------------------------------- in 64 bits
def _value(codes, exp_bits, man_bits):
    """Values of float codes from their fields, in 64 bits (no infinities)."""
    c = codes.to(torch.int64)
    sign = 1.0 - 2.0 * ((c >> (exp_bits + man_bits)) & 1).double()
    e, m = (c >> man_bits) & ((1 << exp_bits) - 1), c & ((1 << man_bits) - 1)
    bias = (1 << (exp_bits - 1)) - 1
    return sign * torch.where(e > 0, m + (1 << man_bits), m).double() * torch.exp2((e.clamp(min=1) - bias - man_bits).double())


def _elements(codes, elem):
    if elem == "e4m3":
        return _value(codes, 4, 3)
    return torch.stack([_value(codes & 15, 2, 1), _value(codes >> 4, 2, 1)], dim=-1).flatten(-2)


def _held(codes, scales, elem):
    return _elements(codes, elem) * torch.exp2(scales.double() - 127).repeat_interleave(32, dim=-1)


def _nearest(x, elem):
    """What an MX block format holds of ``x``, in 64 bits: the nearest of all its values, the even one at a tie."""
    most, top = (8, 448.0) if elem == "e4m3" else (2, 6.0)
    bits = 8 if elem == "e4m3" else 4
    codes = torch.arange(1 << (bits - 1), device=x.device, dtype=torch.uint8)
    values = _value(codes, 4, 3) if elem == "e4m3" else _value(codes, 2, 1)
    values = values[values <= top]
    blocks = x.double().unflatten(-1, (-1, 32))
    amax = blocks.abs().amax(-1, keepdim=True)
    s = torch.where(amax > 0, torch.exp2((torch.frexp(amax)[1] - 1 - most).double()), 1.0)
    a = (blocks / s).abs().clamp(max=top)
    hi = torch.bucketize(a, values).clamp(max=len(values) - 1)
    lo = (hi - 1).clamp(min=0)
    below, above = a - values[lo], values[hi] - a
    take = torch.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)
    return (torch.sign(blocks) * values[take] * s).flatten(-2)


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "linear":
        x, out = state["x"].double(), []
        for i in range(0, case["n_out"], 4096):
            w, s = _elements(state["codes"][i:i + 4096], "e2m1"), state["scales"][i:i + 4096]
            if case["format"] == "mxfp4":
                w = w * torch.exp2(s.double() - 127).repeat_interleave(32, dim=-1)
            else:
                w = w * _value(s, 4, 3).repeat_interleave(16, dim=-1) * state["global"].double()
            out.append(x @ w.t())
        y = torch.cat(out, dim=1)
        return y if state["bias"] is None else y + state["bias"].double()
    if case["kind"] == "cache":
        return _nearest(state["k"], case["elem"]), _nearest(state["v"], case["elem"])
    new, lens = _lengths(case)
    q, group, out, at = state["q"], case["heads"] // case["kv_heads"], [], 0
    for b, (n, length) in enumerate(zip(new, lens)):
        pages = state["pages"][b, :-(-length // case["page"])].long()
        rows = q[at:at + n] if case["ragged"] else q[b]
        at += n
        where = torch.arange(length - n, length, device=DEV)[:, None]
        t = torch.arange(length, device=DEV)[None]
        hidden = t > where
        if case["window"]:
            hidden = hidden | ((where - t >= case["window"]) & (t >= case["sinks"]))
        heads = []
        for h in range(case["kv_heads"]):
            k, v = (_held(state["cache"][i][pages, h], state["cache"][i + 1][pages, h], case["elem"]).flatten(0, 1)[:length] for i in (0, 2))
            for j in range(h * group, (h + 1) * group):
                s = (rows[:, j].double() @ k.t()) / math.sqrt(case["head_dim"])
                heads.append(torch.softmax(s.masked_fill(hidden, -math.inf), dim=-1) @ v)
        out.append(torch.stack(heads, dim=1))
    return torch.cat(out) if case["ragged"] else torch.stack(out)
