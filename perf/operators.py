"""The exact path around the compressed cache, as timed cases.

A case is one pass through one operator:

* ``rotary``  ``apply_norm_rotary``: queries and keys normed per head and rotated;
* ``pages``   ``build_page_step``: block tables and slots of one scheduler step;
* ``packed``  ``compute_packed_attention``: a step's own tokens, several documents
              back to back, masked, capped or biased scores;
* ``paged``   ``compute_paged_attention``: one new token per sequence over a paged
              exact cache.

``own`` chooses between the plain torch form and the package's operators.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CAP = 50.0

_BASE = dict(dtype="bf16", q_heads=32, kv_heads=8, head_dim=128)


def _case(name, kind, **kw):
    c = dict(_BASE, kind=kind, **kw)
    if name:
        c["name"] = name
    return c


def _rotary(name, tokens, **kw):
    return _case(name, "rotary", **dict(dict(tokens=tokens, rotary_dim=128, interleaved=False, scaling="none",
                                             norm=True, far=32768), **kw))


def _pages(name, requests, **kw):
    return _case(name, "pages", **dict(dict(requests=requests, prompts=0, longest=16384, block=16), **kw))


def _packed(name, docs, longest, **kw):
    return _case(name, "packed", **dict(dict(docs=docs, longest=longest, even=False, causal=True, prefix=0, window=0,
                                             cap=0.0, alibi=False), **kw))


def _paged(name, seqs, longest, **kw):
    return _case(name, "paged", **dict(dict(seqs=seqs, longest=longest, even=False, block=16, window=0, cap=0.0,
                                            alibi=False), **kw))


def listed():
    return [
        # one decode step of 64 sequences: all latency
        _rotary("rotary_step", 64),
        # a long prompt's queries and keys, normed and rotated
        _rotary("rotary_prompt", 16384),
        # far positions of a context extended 32 times; neighbouring pairs, half of the head, no norm
        _rotary("rotary_far", 4001, dtype="fp16", q_heads=28, kv_heads=4, rotary_dim=64, interleaved=True,
                scaling="yarn", norm=False, far=1 << 20),
        # a pure decode step of 256 requests
        _pages("pages_decode", 256),
        # a step of 1000 requests, 50 of them prompts
        _pages("pages_mixed", 1000, prompts=50, longest=4096),
        # three short prompts: all latency
        _packed("packed_short", 3, 77),
        # one long prompt, scores capped
        _packed("packed_long", 1, 16384, even=True, cap=CAP),
        # many prompts of all lengths, scores biased by distance
        _packed("packed_docs", 40, 4096, alibi=True),
        # prompts whose first part is seen from everywhere
        _packed("packed_prefix", 8, 4096, dtype="fp16", q_heads=28, kv_heads=4, prefix=500),
        # one user's long chat: a step has one row per head to spread over the card
        _paged("paged_one", 1, 65408, even=True, dtype="fp16", q_heads=28, kv_heads=4),
        # a full batch of long contexts
        _paged("paged_long", 32, 32768, even=True),
        # a serving batch of all lengths, scores capped
        _paged("paged_ragged", 256, 4096, cap=CAP),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(("rotary", "pages", "packed", "packed", "paged", "paged"))
    kw = {}
    kw["q_heads"], kw["kv_heads"] = rng.choice(((32, 8), (28, 4), (8, 8)))
    kw["dtype"] = rng.choice(("bf16", "bf16", "fp16"))
    if kind == "pages":
        n = _log(rng, 1, 1000)
        return _pages("", n, prompts=rng.randint(0, min(n, 60)), longest=_log(rng, 64, 16384 if n <= 256 else 4096),
                      block=rng.choice((16, 16, 32, 64)))
    kw["head_dim"] = d = rng.choice((64, 128, 128, 128, 256))
    if kind == "rotary":
        kw["dtype"] = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        size = (2 if kw["dtype"] == "fp32" else 1) * d // 64 * (kw["q_heads"] + kw["kv_heads"])
        return _rotary("", _log(rng, 1, 16384 * 80 // max(80, size)), rotary_dim=rng.choice((d, d, d // 2)),
                       interleaved=rng.random() < 0.4, scaling=rng.choice(("none", "none", "linear", "ntk", "yarn")),
                       norm=rng.random() < 0.6, far=_log(rng, 2048, 1 << 20), **kw)
    kw["cap"] = rng.choice((0.0, 0.0, CAP))
    kw["alibi"] = rng.random() < 0.25
    if kind == "packed":
        docs = _log(rng, 1, 60)
        most = int(math.sqrt(16384.0 ** 2 * 32 * 128 / (docs * kw["q_heads"] * d)))
        longest = _log(rng, 16, min(16384, 65536 // docs, most))
        extra = rng.choice(("", "", "", "prefix", "window", "full"))
        if extra == "prefix":
            kw["prefix"] = _log(rng, 1, max(1, longest // 2))
        if extra == "window":
            kw["window"] = _log(rng, 16, 4096)
        return _packed("", docs, longest, causal=extra != "full", **kw)
    seqs = _log(rng, 1, 256)
    longest = _log(rng, 16, min(65408, (1 << 30) // (seqs * kw["kv_heads"] * d)))
    if rng.random() < 0.2:
        kw["window"] = _log(rng, 16, 4096)
    return _paged("", seqs, longest, even=rng.random() < 0.3, block=rng.choice((16, 16, 32, 64)), **kw)


# ----------------------------------------------------------------- inputs ---

def _generator(seed, stream):
    return torch.Generator(device="cuda").manual_seed(1013 * int(seed) + stream)


def _shuffled(values, seed, stream):
    order = torch.randperm(len(values), generator=torch.Generator().manual_seed(1013 * int(seed) + stream))
    return [values[i] for i in order.tolist()]


def _lengths(n, lo, hi):
    """n whole numbers of [lo, hi], spread over their logarithm: the same for all inputs of a case."""
    u = torch.rand(n, generator=torch.Generator().manual_seed(41), dtype=torch.float64)
    x = torch.exp(math.log(lo) + u * (math.log(hi + 1) - math.log(lo))).floor()
    return [min(hi, max(lo, int(v))) for v in x]


def _shape_lengths(case):
    """The tokens of the documents or sequences: the longest is always among them."""
    n = case["docs"] if case["kind"] == "packed" else case["seqs"]
    if case["even"]:
        return [case["longest"]] * n
    return [case["longest"]] + _lengths(n - 1, max(1, case["longest"] // 16), case["longest"])


def _slopes(case):
    """Slopes of the distance bias, a geometric row over the heads; None without a bias."""
    if not case["alibi"]:
        return None
    n = case["q_heads"]
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / n) for h in range(n)], dtype=torch.float32, device="cuda")


def _prefixes(case, lens):
    if not case["prefix"]:
        return None
    return [min(n, case["prefix"] + 3 * i) for i, n in enumerate(lens)]


def _projection(case, tokens, seed):
    """A layer's packed projection [tokens, (Hq + 2 Hkv) D] and its three views."""
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    x = torch.empty(tokens, hq + 2 * hkv, d, dtype=DTYPES[case["dtype"]], device="cuda")
    g = _generator(seed, 2)
    for i in range(0, tokens, 4096):
        m = min(tokens, i + 4096) - i
        x[i:i + m] = torch.randn(m, hq + 2 * hkv, d, generator=g, device="cuda").to(x.dtype)
    x[:, :hq] *= 2
    return x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]


def _prepare_rotary(case, seed):
    q, k, _ = _projection(case, case["tokens"], seed)
    g = _generator(seed, 3)
    d = case["head_dim"]
    state = dict(q=q, k=k, positions=torch.randint(0, case["far"], (case["tokens"],), generator=g, device="cuda"))
    for name in ("q_weight", "k_weight"):
        w = 1 + 0.2 * torch.randn(d, generator=g, device="cuda")
        state[name] = w.to(q.dtype) if case["norm"] else None
    if own:
        from smaq_amd.rotary import RotaryPositions
        state["rotary"] = RotaryPositions(case["rotary_dim"], base=10000.0, interleaved=case["interleaved"],
                                          scaling=case["scaling"], factor=32.0, original_length=4096, device="cuda")
    else:
        state["freqs"], state["gain"] = _plain_frequencies(case)
    return state


def _prepare_pages(case, seed):
    n, bs = case["requests"], case["block"]
    ctx = _shuffled(_lengths(n, 1, case["longest"]), seed, 1)
    new = [1] * n
    fresh = _lengths(case["prompts"], 16, case["longest"])
    for i, tokens in zip(_shuffled(range(n), seed, 5), fresh):
        ctx[i], new[i] = (0 if i % 2 else ctx[i] // 2), tokens
    width = -(-2 * case["longest"] // bs)
    held = [-(-c // bs) for c in ctx]
    taken = sum(-(-(c + m) // bs) - h for c, m, h in zip(ctx, new, held))
    blocks = sum(held) + taken + 64
    perm = torch.randperm(blocks, generator=_generator(seed, 6), device="cuda").to(torch.int32)
    table = torch.zeros(n, width, dtype=torch.int32, device="cuda")
    cols = torch.arange(width, device="cuda")
    h = torch.tensor(held, device="cuda")
    first = torch.cumsum(h, 0) - h
    mine = cols[None, :] < h[:, None]
    table[mine] = perm[(first[:, None] + cols[None, :])[mine]]
    return dict(context=torch.tensor(ctx, dtype=torch.int32, device="cuda"),
                new=torch.tensor(new, dtype=torch.int32, device="cuda"), table=table, free=perm[sum(held):].clone(),
                block=bs, tokens=sum(new))


def _prepare_packed(case, seed):
    lens = _shuffled(_shape_lengths(case), seed, 1)
    q, k, v = _projection(case, sum(lens), seed)
    prefix = _prefixes(case, lens)
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    return dict(q=q, k=k, v=v, lens=lens, starts=torch.tensor(starts, dtype=torch.int32, device="cuda"),
                causal=case["causal"], window=case["window"], cap=case["cap"],
                slopes=_slopes(case), prefix=prefix, scale=1.0 / math.sqrt(case["head_dim"]),
                prefix_lens=None if prefix is None else torch.tensor(prefix, dtype=torch.int32, device="cuda"))


def _prepare_paged(case, seed):
    lens = _shuffled(_shape_lengths(case), seed, 1)
    bs, hkv, d = case["block"], case["kv_heads"], case["head_dim"]
    held = [-(-n // bs) for n in lens]
    blocks = sum(held)
    cache = torch.empty(2, blocks, bs, hkv, d, dtype=DTYPES[case["dtype"]], device="cuda")
    flat, g = cache.view(-1, d), _generator(seed, 2)
    for i in range(0, flat.shape[0], 1 << 21):
        m = min(flat.shape[0], i + (1 << 21)) - i
        flat[i:i + m] = torch.randn(m, d, generator=g, device="cuda").to(cache.dtype)
    perm = torch.randperm(blocks, generator=_generator(seed, 6), device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), max(held), dtype=torch.int32, device="cuda")
    o = 0
    for b, h in enumerate(held):
        table[b, :h] = perm[o:o + h]
        o += h
    q = 2 * torch.randn(len(lens), case["q_heads"], d, generator=_generator(seed, 3), device="cuda")
    return dict(q=q.to(cache.dtype), cache=cache, table=table, lens=lens, longest=max(lens),
                seq_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), window=case["window"], cap=case["cap"],
                slopes=_slopes(case), scale=1.0 / math.sqrt(d))


def prepare(case, seed):
    kind = case["kind"]
    state = {"rotary": _prepare_rotary, "pages": _prepare_pages, "packed": _prepare_packed,
             "paged": _prepare_paged}[kind](case, seed)
    return dict(state, kind=kind, interleaved=case.get("interleaved", False))


# ------------------------------------------------------------------ plain ---

def _plain_frequencies(case):
    """(angle per position of each pair, gain of sine and cosine), in 64 bits."""
    r, factor, length = case["rotary_dim"], 32.0, 4096
    base = 10000.0 * factor ** (r / (r - 2)) if case["scaling"] == "ntk" else 10000.0
    i = torch.arange(r // 2, dtype=torch.float64, device="cuda")
    f = base ** (-2 * i / r)
    if case["scaling"] == "linear":
        return f / factor, 1.0
    if case["scaling"] != "yarn":
        return f, 1.0
    def pair(turns):
        return r * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base))
    lo, hi = max(0, math.floor(pair(32.0))), min(r - 1, math.ceil(pair(1.0)))
    slow = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
    return f * (1 - slow) + f / factor * slow, 0.1 * math.log(factor) + 1.0


def _plain_rotary(s):
    angle = s["positions"].double()[:, None] * s["freqs"]
    cos, sin = (angle.cos() * s["gain"]).float()[:, None], (angle.sin() * s["gain"]).float()[:, None]
    r = 2 * s["freqs"].shape[0]
    outs = []
    for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
        y = x.float()
        if w is not None:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * w.float()
        a, b = (y[..., 0:r:2], y[..., 1:r:2]) if s["interleaved"] else (y[..., :r // 2], y[..., r // 2:r])
        c, d = a * cos - b * sin, a * sin + b * cos
        turned = torch.stack((c, d), -1).flatten(-2) if s["interleaved"] else torch.cat((c, d), -1)
        outs.append(torch.cat((turned, y[..., r:]), -1).to(x.dtype))
    return tuple(outs)


def _plain_pages(s):
    ctx, new, table, free, bs, tokens = s["context"].long(), s["new"].long(), s["table"], s["free"], s["block"], s["tokens"]
    held = (ctx + bs - 1) // bs
    taken = (ctx + new + bs - 1) // bs - held
    ends = torch.cumsum(taken, 0)
    j = torch.arange(table.shape[1], device=table.device)[None, :] - held[:, None]
    fresh = (j >= 0) & (j < taken[:, None])
    src = ((ends - taken)[:, None] + j).clamp(0, free.shape[0] - 1)
    table.copy_(torch.where(fresh, free[src], table))
    starts = torch.zeros(ctx.shape[0] + 1, dtype=torch.int64, device=table.device)
    starts[1:] = torch.cumsum(new, 0)
    i = torch.arange(tokens, device=table.device)
    b = torch.searchsorted(starts, i, right=True) - 1
    p = ctx[b] + i - starts[b]
    slots = table[b, p // bs].long() * bs + p % bs
    return (table, slots, p, starts.to(torch.int32), (ctx + new).to(torch.int32),
            torch.stack((ends[-1], torch.zeros_like(ends[-1]))).to(torch.int32))


def _plain_scores(raw, i, j, s, slopes):
    """Scores of products ``raw`` [heads, queries, keys] of positions i and j."""
    x = raw * s["scale"]
    if s["cap"]:
        x = s["cap"] * torch.tanh(x / s["cap"])
    if slopes is not None:
        x = x - slopes[:, None, None] * (i[:, None] - j[None, :]).abs().to(x.dtype)
    return x


def _plain_weights(x):
    w = torch.exp(x - x.amax(-1, keepdim=True))
    return w / w.sum(-1, keepdim=True)


def _plain_packed(s):
    q, k, v = s["q"], s["k"], s["v"]
    hq, g = q.shape[1], q.shape[1] // k.shape[1]
    out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    t = 0
    for doc, n in enumerate(s["lens"]):
        i = torch.arange(n, device=q.device)
        seen = torch.ones(n, n, dtype=torch.bool, device=q.device)
        if s["causal"]:
            seen = i[None, :] <= i[:, None]
        if s["window"]:
            seen = seen & (i[None, :] > i[:, None] - s["window"])
        if s["prefix"] is not None:
            seen = seen | (i[None, :] < s["prefix"][doc])
        step = max(g, min(hq, (1 << 29) // (n * n) // g * g))
        for h in range(0, hq, step):
            m = min(hq, h + step) - h
            qh = q[t:t + n, h:h + m].float().transpose(0, 1).reshape(m // g, g * n, -1)
            kh = k[t:t + n, h // g:(h + m) // g].float().permute(1, 2, 0).contiguous()
            vh = v[t:t + n, h // g:(h + m) // g].float().transpose(0, 1).contiguous()
            raw = torch.matmul(qh, kh).view(m, n, n)
            x = _plain_scores(raw, i, i, s, None if s["slopes"] is None else s["slopes"][h:h + m])
            w = _plain_weights(x.masked_fill(~seen, float("-inf")))
            o = torch.matmul(w.view(m // g, g * n, n), vh)
            out[t:t + n, h:h + m] = o.view(m, n, -1).transpose(0, 1).to(out.dtype)
        t += n
    return out


def _plain_paged(s):
    q, cache, bs = s["q"], s["cache"], s["cache"].shape[2]
    hkv, d = cache.shape[3:]
    g = q.shape[1] // hkv
    out = torch.empty_like(q)
    for b, n in enumerate(s["lens"]):
        lo = max(0, n - s["window"]) if s["window"] else 0
        pages = s["table"][b, lo // bs:-(-n // bs)].long()
        k, v = (c[pages].reshape(-1, hkv, d)[lo % bs:n - lo // bs * bs].float() for c in cache)
        raw = torch.matmul(q[b].float().view(hkv, g, d), k.permute(1, 2, 0).contiguous()).view(hkv * g, 1, n - lo)
        j = torch.arange(lo, n, device=q.device)
        w = _plain_weights(_plain_scores(raw, j[-1:], j, s, s["slopes"]))
        o = torch.matmul(w.view(hkv, g, n - lo), v.transpose(0, 1).contiguous())
        out[b] = o.view(hkv * g, d).to(out.dtype)
    return out


# -------------------------------------------------------------------- own ---

def _own_rotary(s):
    from smaq_amd.rotary import apply_norm_rotary
    return apply_norm_rotary(s["q"], s["k"], s["positions"], s["rotary"], q_weight=s["q_weight"],
                             k_weight=s["k_weight"], eps=1e-6)


def _own_pages(s):
    from smaq_amd.paging import build_page_step
    step = build_page_step(s["context"], s["new"], s["table"], s["free"], s["block"], s["tokens"])
    return s["table"], step.slot_mapping, step.positions, step.query_start_loc, step.seq_lens, step.status


def _own_packed(s):
    from smaq_amd.exact_attention import compute_packed_attention
    return compute_packed_attention(s["q"], s["k"], s["v"], s["starts"], scale=s["scale"], causal=s["causal"],
                                    prefix_lens=s["prefix_lens"], window=s["window"], score_cap=s["cap"],
                                    alibi_slopes=s["slopes"])


def _own_paged(s):
    from smaq_amd.exact_attention import compute_paged_attention
    return compute_paged_attention(s["q"], s["cache"][0], s["cache"][1], s["table"], s["seq_lens"], s["longest"],
                                   scale=s["scale"], window=s["window"], score_cap=s["cap"],
                                   alibi_slopes=s["slopes"])


def run(state):
    forms = ({"rotary": _own_rotary, "pages": _own_pages, "packed": _own_packed, "paged": _own_paged} if own else
             {"rotary": _plain_rotary, "pages": _plain_pages, "packed": _plain_packed, "paged": _plain_paged})
    return forms[state["kind"]](state)


# ------------------------------------------------------------------- work ---

def _pairs(case, lens):
    """Visible (query, key) pairs of one head."""
    prefix, total = _prefixes(case, lens) or [0] * len(lens), 0
    for n, p in zip(lens, prefix):
        if not case["causal"]:
            total += n * n
            continue
        w = min(case["window"] or n, n)
        # p keys seen from all rows, and of the others those of the last w at or before the row
        total += p * n
        m = n - p
        w = min(w, m)
        total += w * (w + 1) // 2 + (m - w) * w
    return total


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    if case["kind"] == "rotary":
        n = case["tokens"] * (hq + hkv) * d
        return {"bytes": 2 * n * size + 8 * case["tokens"], "flops": 8 * n}
    if case["kind"] == "pages":
        tokens = case["requests"] + sum(_lengths(case["prompts"], 16, case["longest"]))
        fresh = tokens // case["block"] + case["requests"] // 2
        return {"bytes": 16 * tokens + 8 * fresh + 16 * case["requests"], "flops": 0}
    lens = _shape_lengths(case)
    if case["kind"] == "packed":
        return {"bytes": 2 * sum(lens) * (hq + hkv) * d * size, "flops": 4 * d * hq * _pairs(case, lens)}
    seen = sum(min(n, case["window"] or n) for n in lens)
    return {"bytes": 2 * seen * hkv * d * size + 2 * len(lens) * hq * d * size, "flops": 4 * d * hq * seen}


# ------------------------------------------------------------------ exact ---

def _exact_rotary(s):
    r = 2 * s["freqs"].shape[0]
    pairs = torch.arange(r // 2, device="cuda")
    first, second = (2 * pairs, 2 * pairs + 1) if s["interleaved"] else (pairs, pairs + r // 2)
    z = torch.polar(torch.full((), s["gain"], dtype=torch.float64, device="cuda"),
                    s["positions"].double()[:, None, None] * s["freqs"])
    outs = []
    for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
        y = x.double()
        if w is not None:
            y = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / y.shape[-1] + 1e-6) * w.double()
        turned = torch.complex(y[..., first], y[..., second]) * z
        y = y.clone()
        y[..., first], y[..., second] = turned.real, turned.imag
        outs.append(y)
    return tuple(outs)


def _exact_rows(q, k, v, i, j, seen, s, slope):
    """One head in 64 bits: queries q [n, D] at positions i over keys at j; seen [n, m] or None."""
    x = (q.double() @ k.double().T.contiguous()).mul_(s["scale"])
    if s["cap"]:
        x.div_(s["cap"]).tanh_().mul_(s["cap"])
    if slope is not None:
        x.sub_((i[:, None] - j[None, :]).abs().double().mul_(slope.double()))
    if seen is not None:
        x.masked_fill_(~seen, float("-inf"))
    return torch.softmax(x, -1) @ v.double()


def _exact_packed(s):
    q, k, v = s["q"], s["k"], s["v"]
    g = q.shape[1] // k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    t = 0
    for doc, n in enumerate(s["lens"]):
        j = torch.arange(n, device="cuda")
        for r in range(0, n, 8192):
            i = j[r:r + 8192]
            gap = i[:, None] - j[None, :]
            seen = gap >= 0 if s["causal"] else torch.ones_like(gap, dtype=torch.bool)
            if s["window"]:
                seen &= gap < s["window"]
            if s["prefix"] is not None:
                seen |= (j < s["prefix"][doc])[None, :]
            for h in range(q.shape[1]):
                out[t + r:t + r + len(i), h] = _exact_rows(q[t + r:t + r + len(i), h], k[t:t + n, h // g],
                                                           v[t:t + n, h // g], i, j, seen, s,
                                                           None if s["slopes"] is None else s["slopes"][h])
        t += n
    return out


def _exact_paged(s):
    q, bs = s["q"], s["cache"].shape[2]
    g = q.shape[1] // s["cache"].shape[3]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lens"]):
        j = torch.arange(max(0, n - s["window"]) if s["window"] else 0, n, device="cuda")
        page, offset = s["table"][b].long()[j // bs], j % bs
        for h in range(0, q.shape[1], g):
            k, v = s["cache"][0][page, offset, h // g], s["cache"][1][page, offset, h // g]
            for x in range(h, h + g):
                out[b, x] = _exact_rows(q[b, x:x + 1], k, v, j[-1:], j, None, s,
                                        None if s["slopes"] is None else s["slopes"][x])[0]
    return out


def exact(case, seed):
    if case["kind"] == "pages":
        return None
    state = prepare(case, seed)
    if case["kind"] == "rotary":
        state["freqs"], state["gain"] = _plain_frequencies(case)
        return _exact_rotary(state)
    return _exact_packed(state) if case["kind"] == "packed" else _exact_paged(state)
