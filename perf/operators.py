"""Measured cases of the serving operators: the paged key/value cache's append with rotary
positions, the attention that reads the cache, and the sampler on the device.

`run` computes an operator either in its plain form (elementary torch operations, `own` false)
or by the framework's entry points in `dpuf_b200.serving` (`own` true), on the same state.

The cache holds pages `[n_pages, n_kv, page, dim]` for keys and for values; `page_table[s, j]` is
the page of sequence s's positions `[j * page, (j + 1) * page)`, or -1 where none is held.

rope_append: token t of sequence `seq[t]` stands at `pos[t]`.  The first `rot` dimensions of each
head of q and k are turned by the angles whose cosines and sines are row `pos[t]` of the tables
(pairs (i, i + rot/2), or (2i, 2i + 1) where interleaved); k and v are stored at `pos[t]` in the
cache's type and the turned q is returned.

paged_attention: sequence s has new tokens `q_start[s] .. q_start[s+1]`, the last of its
`kv_len[s]` positions.  The token at position p sees positions j <= p (all of them where not
causal), and with a window w only j > p - w:  out = sum_j softmax_j(scale * q . k_j) v_j; a token
that sees nothing gets zeros.

sample: weights w_i = exp((l_i - max l) / temperature); of the entries ordered by (logit down,
index up) the first top_k are kept, of these the shortest prefix that holds top_p of their weight,
of these the ones with w_i >= min_p; id is the first kept index (in index order) whose running
weight exceeds u times the kept weight, prob its share of it.  temperature 0 takes the first
maximum.
"""
import math
import random

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    rope = {"op": "rope_append", "hq": 32, "hkv": 8, "dim": 128, "rot": 128, "page": 16, "shape_seed": 1}
    attn = {"op": "paged_attention", "hq": 32, "hkv": 8, "dim": 128, "page": 16, "window": 0, "causal": True,
            "shape_seed": 2}
    pick = {"op": "sample", "vocab": 151936, "spread": 3.0}
    return [
        # a decode step of the batched serving configuration: 64 sequences, one token each, the engine's
        # fp32 activations into an fp16 cache
        {**rope, "name": "rope_decode64", "seqs": 64, "tokens": 64, "pos_max": 2304, "type": "f32", "kv": "f16",
         "interleaved": False, "scaling": "none", "factor": 1.0},
        # prompts of a few requests at once; half of each head turned, interleaved pairs
        {**rope, "name": "rope_prompts", "seqs": 4, "tokens": 8191, "pos_max": 8192, "type": "bf16", "kv": "bf16",
         "rot": 64, "interleaved": True, "scaling": "linear", "factor": 4.0},
        # a large chunk late in a long context, angles stretched by wavelength
        {**rope, "name": "rope_long", "seqs": 1, "tokens": 16384, "pos_max": 131072, "type": "f16", "kv": "f16",
         "page": 64, "interleaved": False, "scaling": "yarn", "factor": 4.0},
        # batch-1 decode at a short context: the call's latency
        {**attn, "name": "attn_one_short", "seqs": 1, "q_min": 1, "q_max": 1, "kv_min": 168, "kv_max": 168,
         "type": "f16", "kv": "f16"},
        # a decode step of the batched serving configuration
        {**attn, "name": "attn_decode64", "seqs": 64, "q_min": 1, "q_max": 1, "kv_min": 2049, "kv_max": 2304,
         "type": "f16", "kv": "f16"},
        # one sequence far into a long context: few rows, a long axis
        {**attn, "name": "attn_one_long", "seqs": 1, "q_min": 1, "q_max": 1, "kv_min": 131071, "kv_max": 131071,
         "page": 64, "type": "bf16", "kv": "bf16"},
        # prefill of the serving configuration's prompts
        {**attn, "name": "attn_prompts", "seqs": 4, "q_min": 2048, "q_max": 2048, "kv_min": 2048, "kv_max": 2048,
         "type": "f16", "kv": "f16"},
        # a chunk of a long prompt over what the earlier chunks stored
        {**attn, "name": "attn_chunk", "seqs": 1, "q_min": 512, "q_max": 512, "kv_min": 33280, "kv_max": 33280,
         "page": 32, "type": "bf16", "kv": "bf16"},
        # a mixed batch of decode tokens and short odd chunks with a sliding window, fp32 activations over an
        # fp16 cache; some slots have no new token
        {**attn, "name": "attn_mixed", "seqs": 23, "q_min": 0, "q_max": 37, "kv_min": 37, "kv_max": 1777, "hq": 12,
         "hkv": 4, "dim": 64, "window": 511, "type": "f32", "kv": "f16"},
        # one sequence's next token with the usual filters: the call's latency
        {**pick, "name": "sample_one", "rows": 1, "type": "f32", "top_k": 50, "top_p": 0.95, "min_p": 0.0},
        # the serving batch's next tokens, nucleus and min-p, no top-k
        {**pick, "name": "sample_batch64", "rows": 64, "type": "f32", "top_k": 0, "top_p": 0.9, "min_p": 0.02},
        # many rows of flat logits in 16 bits (many equal values), a large top-k
        {**pick, "name": "sample_flat", "rows": 256, "type": "bf16", "top_k": 5000, "top_p": 0.98, "min_p": 0.0,
         "spread": 1.0},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(["rope_append", "paged_attention", "paged_attention", "sample"])
    seed = rng.randrange(1 << 30)
    if op == "sample":
        vocab = _log_int(rng, 1000, 262144)
        rows = _log_int(rng, 1, min(256, 256 * 151936 // vocab))
        return {"op": op, "vocab": vocab, "rows": rows, "type": rng.choice(["f32", "f16", "bf16"]),
                "spread": rng.choice([1.0, 2.0, 3.0, 5.0]), "top_k": rng.choice([0, 0, 1, _log_int(rng, 2, 10000)]),
                "top_p": rng.choice([1.0, 0.5, 0.9, 0.95, 0.99]), "min_p": rng.choice([0.0, 0.0, 0.01, 0.1])}
    hq, hkv = rng.choice([(32, 8), (16, 8), (8, 8), (12, 4), (6, 2), (28, 4), (16, 1), (3, 3)])
    dim = rng.choice([64, 64, 80, 96, 128, 128, 128])
    page = rng.choice([8, 16, 16, 32, 64, 128])
    both = {"op": op, "hq": hq, "hkv": hkv, "dim": dim, "page": page, "shape_seed": seed}
    if op == "rope_append":
        tokens = _log_int(rng, 1, 16384)
        seqs = _log_int(rng, 1, min(64, tokens))
        pos_max = max(_log_int(rng, 256, 131072), 2 * (-(-tokens // seqs)))
        kind = rng.choice([("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
        return {**both, "tokens": tokens, "seqs": seqs, "pos_max": pos_max, "type": kind[0], "kv": kind[1],
                "rot": rng.choice([dim, dim, dim // 2, dim // 4]), "interleaved": rng.random() < 0.5,
                "scaling": rng.choice(["none", "linear", "yarn"]), "factor": rng.choice([2.0, 4.0, 8.0])}
    # fp32 activations: decode steps and short chunks; 16 bits: up to whole prompts
    kind = rng.choice([("f16", "f16"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"),
                       ("f32", "f32")])
    q_max = 1 if rng.random() < 0.4 else _log_int(rng, 1, 64 if kind[0] == "f32" else 2048)
    kv_max = max(q_max, _log_int(rng, 16, 131072))
    stored = 2304 * 64 * 8 * 128 * 2 // (_BYTES[kind[1]] * hkv * dim)  # the serving batch's cache bytes
    scores = 4 * 32 * 2048 * 2048 // (q_max * hq)  # the prompts' scores
    kv_max = max(q_max, min(kv_max, stored, scores))
    most = max(1, min(64, stored // kv_max, scores // kv_max))
    seqs = _log_int(rng, 1, most)
    window = rng.choice([0, 0, 0, _log_int(rng, 1, kv_max)])
    q_min = rng.choice([0, q_max]) if seqs > 1 else q_max
    return {**both, "seqs": seqs, "q_min": q_min, "q_max": q_max, "kv_min": rng.choice([q_max, kv_max]),
            "kv_max": kv_max, "window": window, "causal": window > 0 or rng.random() < 0.8, "type": kind[0],
            "kv": kind[1]}


def _lengths(case):
    """New tokens and stored positions of each sequence, of the case alone; the first has the most of both."""
    rng = random.Random(case["shape_seed"])
    q = [case["q_max"]] + [rng.randint(case["q_min"], case["q_max"]) for _ in range(case["seqs"] - 1)]
    kv = [case["kv_max"]] + [rng.randint(max(case["kv_min"], n), case["kv_max"]) for n in q[1:]]
    return q, kv


def _spans(case):
    """First position and number of new tokens of each sequence of a rope_append case."""
    rng = random.Random(case["shape_seed"])
    n, total = case["seqs"], case["tokens"]
    count = [total // n + (1 if i < total % n else 0) for i in range(n)]
    return [(case["pos_max"] - c if i == 0 else rng.randint(0, case["pos_max"] - c), c) for i, c in enumerate(count)]


def _frequencies(case):
    """Turn per position of each pair, and the factor on cosine and sine, in 64 bits."""
    rot, base, factor = case["rot"], 1e6, case["factor"]
    freq = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if case["scaling"] == "linear":
        return freq / factor, 1.0
    if case["scaling"] == "yarn":  # fast pairs as they are, slow ones stretched, a ramp between
        orig = case["pos_max"] / factor
        turns = orig * freq / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        return freq * keep + freq / factor * (1 - keep), 0.1 * math.log(factor) + 1.0
    return freq, 1.0


def _page_table(spans, width, page, pages, device):
    """Table of `width` entries a sequence; `spans`: first and end position that each one holds."""
    table = torch.full((len(spans), width), -1, dtype=torch.int32)
    at = 0
    for s, (low, high) in enumerate(spans):
        if high > low:
            a, b = low // page, -(-high // page)
            table[s, a:b] = pages[at:at + b - a]
            at += b - a
    return table.to(device)


def _held(spans, page):
    return sum(-(-high // page) - low // page for low, high in spans if high > low)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    s = {"case": case}
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # a head's logits: a bulk of normal values and a few that stand out
        logits = torch.randn(rows, vocab, generator=g, device=dev) * case["spread"]
        top = torch.randint(0, vocab, (rows, 12), generator=g, device=dev)
        logits.scatter_add_(1, top, torch.rand(rows, 12, generator=g, device=dev) * 4 * case["spread"])
        s["logits"] = logits.to(_TYPES[case["type"]])
        s["u"] = torch.rand(rows, generator=g, device=dev)
        s["temperature"] = 0.5 + torch.rand(rows, generator=g, device=dev)
        if rows > 4:
            s["temperature"][3] = 0.0  # a greedy request among the others
        s["top_k"] = torch.full((rows,), case["top_k"], dtype=torch.int32, device=dev)
        s["top_p"] = torch.full((rows,), case["top_p"], device=dev)
        s["min_p"] = torch.full((rows,), case["min_p"], device=dev)
        return s
    hq, hkv, dim, page = case["hq"], case["hkv"], case["dim"], case["page"]
    if case["op"] == "rope_append":
        runs = _spans(case)
        spans = [(first, first + n) for first, n in runs]
        width = -(-case["pos_max"] // page)
    else:
        q_len, kv_len = _lengths(case)
        w = case["window"]
        # pages that lie before every window have been given back
        spans = [(max(0, b - a - w + 1) if w else 0, b) for a, b in zip(q_len, kv_len)]
        width = -(-case["kv_max"] // page)
    n_pages = _held(spans, page) + 3
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    s["page_table"] = _page_table(spans, width, page, order, dev)
    kv_type, x_type = _TYPES[case["kv"]], _TYPES[case["type"]]

    def normal(*shape, scale=1.0, dtype=x_type):
        return (torch.randn(*shape, generator=g, device=dev, dtype=torch.float32) * scale).to(dtype)

    s["k_pages"] = normal(n_pages, hkv, page, dim, dtype=kv_type)
    s["v_pages"] = normal(n_pages, hkv, page, dim, dtype=kv_type)
    if case["op"] == "rope_append":
        # one projection's output, q, k and v side by side
        qkv = normal(case["tokens"], (hq + 2 * hkv) * dim)
        s["q"], s["k"], s["v"] = (x.unflatten(1, (-1, dim)) for x in qkv.split([hq * dim, hkv * dim, hkv * dim], 1))
        freq, gain = _frequencies(case)
        angle = torch.arange(case["pos_max"], dtype=torch.float64, device=dev)[:, None] * freq.to(dev)
        s["cos"], s["sin"] = (gain * angle.cos()).float(), (gain * angle.sin()).float()
        s["seq"] = torch.cat([torch.full((n,), i, dtype=torch.int32) for i, (_, n) in enumerate(runs)]).to(dev)
        s["pos"] = torch.cat([torch.arange(a, a + n, dtype=torch.int32) for a, n in runs]).to(dev)
    else:
        s["q"] = normal(sum(q_len), hq, dim, scale=2.5)  # scores of real heads: some positions stand out
        start = [0]
        for n in q_len:
            start.append(start[-1] + n)
        s["q_start"] = torch.tensor(start, dtype=torch.int32, device=dev)
        s["kv_len"] = torch.tensor(kv_len, dtype=torch.int32, device=dev)
    if own:  # the handle that a program keeps for its cache
        from dpuf_b200 import serving

        s["cache"] = serving.PagedCache(s["k_pages"], s["v_pages"])
    return s


def run(state):
    op = state["case"]["op"]
    if own:
        return _RUN_OWN[op](state)
    return _RUN_PLAIN[op](state)


def _own_rope(s):
    from dpuf_b200 import serving

    q = serving.rope_append(s["cache"], s["page_table"], s["q"], s["k"], s["v"], s["cos"], s["sin"], s["seq"],
                            s["pos"], interleaved=s["case"]["interleaved"])
    return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _own_attention(s):
    from dpuf_b200 import serving

    c = s["case"]
    return {"out": serving.paged_attention(s["cache"], s["page_table"], s["q"], s["q_start"], s["kv_len"], c["q_max"],
                                           causal=c["causal"], window=c["window"])}


def _own_sample(s):
    from dpuf_b200 import serving

    ids, probs = serving.sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    return {"ids": ids, "probs": probs}


def _turn(x, cos, sin, rot, interleaved):
    y = x.float().clone()
    if interleaved:
        a, b = y[..., 0:rot:2].clone(), y[..., 1:rot:2].clone()
        y[..., 0:rot:2] = a * cos - b * sin
        y[..., 1:rot:2] = b * cos + a * sin
    else:
        a, b = y[..., : rot // 2].clone(), y[..., rot // 2 : rot].clone()
        y[..., : rot // 2] = a * cos - b * sin
        y[..., rot // 2 : rot] = b * cos + a * sin
    return y


def _plain_rope(s):
    c = s["case"]
    pos, seq = s["pos"].long(), s["seq"].long()
    cos, sin = s["cos"][pos][:, None, :], s["sin"][pos][:, None, :]
    q = _turn(s["q"], cos, sin, c["rot"], c["interleaved"]).to(s["q"].dtype)
    k = _turn(s["k"], cos, sin, c["rot"], c["interleaved"]).to(s["k_pages"].dtype)
    page = s["page_table"][seq, pos // c["page"]].long()
    s["k_pages"][page, :, pos % c["page"]] = k
    s["v_pages"][page, :, pos % c["page"]] = s["v"].to(s["v_pages"].dtype)
    return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _plain_attention(s):
    c = s["case"]
    n, hq, hkv, dim, q_max = c["seqs"], c["hq"], c["hkv"], c["dim"], c["q_max"]
    table = s["page_table"].long()
    start, kv_len = s["q_start"].long(), s["kv_len"].long()
    q_len = start[1:] - start[:-1]
    dev = table.device
    k, v = (p[table.clamp(min=0)].float().transpose(1, 2).reshape(n, hkv, -1, dim) for p in (s["k_pages"], s["v_pages"]))
    t = torch.arange(q_max, device=dev)
    row = (start[:-1, None] + t).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][row].float().unflatten(2, (hkv, hq // hkv)).permute(0, 2, 3, 1, 4).reshape(n, hkv, -1, dim)
    score = torch.matmul(q, k.transpose(2, 3)) * (dim ** -0.5)
    j = torch.arange(k.shape[2], device=dev)
    at = (kv_len - q_len)[:, None] + t  # position of each new token
    last = at if c["causal"] else (kv_len - 1)[:, None].expand(-1, q_max)
    sees = (j <= last[:, :, None]) & (j < kv_len[:, None, None])
    if c["window"]:
        sees &= j > at[:, :, None] - c["window"]
    score = score.unflatten(2, (hq // hkv, q_max)).masked_fill_(~sees[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = score.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = weight.sum(-1, keepdim=True)
    held = (j < kv_len[:, None]) & (table >= 0).repeat_interleave(c["page"], 1)
    v = v.masked_fill(~held[:, None, :, None], 0.0)
    o = torch.matmul(weight.flatten(2, 3), v).unflatten(2, (hq // hkv, q_max))
    o = (o / total.masked_fill(total == 0, 1.0)).permute(0, 3, 1, 2, 4).reshape(n, q_max, hq, dim)
    token = torch.arange(s["q"].shape[0], device=dev)
    seq = torch.searchsorted(start[1:], token, right=True)
    return {"out": o[seq, token - start[seq]].to(s["q"].dtype)}


def _plain_sample(s):
    # weights in 32 bits; their sums in 64, as the framework's sampler on the host has them: the rounding
    # of a running sum over the vocabulary would otherwise decide the id
    logits = s["logits"].float()
    rows, vocab = logits.shape
    heat = s["temperature"][:, None]
    hot = heat > 0
    top = logits.amax(1, keepdim=True)
    weight = torch.exp((logits - top) * (1.0 / torch.where(hot, heat, torch.ones_like(heat))))
    order = torch.sort(logits, dim=1, descending=True, stable=True).indices
    sorted_weight = weight.gather(1, order).double()
    rank = torch.arange(vocab, device=logits.device)
    limit = torch.where(s["top_k"] > 0, s["top_k"], vocab)[:, None]
    sorted_weight = sorted_weight.masked_fill(rank >= limit, 0.0)
    running = sorted_weight.cumsum(1)
    before = running - sorted_weight
    share = s["top_p"][:, None].double()
    keep = (rank < limit) & ((share >= 1) | (before < share * running[:, -1:]) | (rank == 0))
    keep &= sorted_weight >= s["min_p"][:, None].clamp(max=1.0).double()
    kept = torch.zeros_like(keep).scatter_(1, order, keep)
    mass = weight.double() * kept
    cdf = mass.cumsum(1)
    total = cdf[:, -1:]
    ids = (cdf > s["u"][:, None].double() * total).int().argmax(1)
    probs = mass.gather(1, ids[:, None]) / total
    first = (logits == top).int().argmax(1)
    ids = torch.where(hot[:, 0], ids, first).to(torch.int32)
    return {"ids": ids, "probs": torch.where(hot, probs, torch.ones_like(probs))[:, 0].float()}


_RUN_OWN = {"rope_append": _own_rope, "paged_attention": _own_attention, "sample": _own_sample}
_RUN_PLAIN = {"rope_append": _plain_rope, "paged_attention": _plain_attention, "sample": _plain_sample}


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * _BYTES[case["type"]] + case["rows"] * 28, "flops": 4 * n}
    hq, hkv, dim = case["hq"], case["hkv"], case["dim"]
    x, kv = _BYTES[case["type"]], _BYTES[case["kv"]]
    if case["op"] == "rope_append":
        t = case["tokens"]
        # in: q, k, v, a row of each table; out: q, k, v
        moved = t * ((2 * hq + 2 * hkv) * dim * x + 2 * hkv * dim * kv + case["rot"] * 4 + 8)
        return {"bytes": moved, "flops": 3 * t * (hq + hkv) * case["rot"]}
    pairs, seen = 0, 0
    for a, b in zip(*_lengths(case)):
        w = case["window"] or b
        if not a:
            continue
        if case["causal"]:
            low = max(0, b - a - w + 1)
            full = max(0, b - max(b - a, w - 1))  # tokens whose window is whole
            rest = a - full
            pairs += full * min(w, b) + rest * (b - a + 1) + rest * (rest - 1) // 2
        else:
            low = 0
            pairs += a * b
        seen += b - low
    tokens = sum(_lengths(case)[0])
    return {"bytes": 2 * seen * hkv * dim * kv + 2 * tokens * hq * dim * x, "flops": 4 * pairs * hq * dim}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s)
    if case["op"] == "rope_append":
        return _exact_rope(s)
    return _exact_attention(s)


def _exact_rope(s):
    c = s["case"]
    freq, gain = _frequencies(c)
    half = c["rot"] // 2
    angle = s["pos"].double()[:, None, None] * freq.to(s["pos"].device)
    spin = gain * torch.polar(torch.ones_like(angle), angle)

    def turn(x):  # each pair as a complex number
        x = x.double()
        z = x[..., : c["rot"]]
        z = z.unflatten(-1, (half, 2)) if c["interleaved"] else z.unflatten(-1, (2, half)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * spin)
        z = z if c["interleaved"] else z.transpose(-1, -2)
        return torch.cat([z.flatten(-2), x[..., c["rot"] :]], -1)

    pages = {"k_pages": s["k_pages"].double(), "v_pages": s["v_pages"].double()}
    new = {"k_pages": turn(s["k"]), "v_pages": s["v"].double()}
    for i in range(c["seqs"]):
        mine = (s["seq"] == i).nonzero()[:, 0]
        at = s["pos"][mine].long()
        page, slot = s["page_table"][i].long()[at // c["page"]], at % c["page"]
        for name in pages:
            pages[name][page, :, slot] = new[name][mine]
    return {"q": turn(s["q"]), **pages}


def _exact_attention(s):
    c = s["case"]
    hq, hkv, dim, page = c["hq"], c["hkv"], c["dim"], c["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    first = 0
    for i, (a, b) in enumerate(zip(*_lengths(c))):
        low = max(0, b - a - c["window"] + 1) // page * page if c["window"] else 0
        ids = s["page_table"][i, low // page : -(-b // page)].long()
        at = torch.arange(b - a, b, device=out.device)[:, None]
        j = torch.arange(low, b, device=out.device)
        hide = torch.zeros(a, b - low, dtype=torch.bool, device=out.device)
        if c["causal"]:
            hide |= j > at
        if c["window"]:
            hide |= j <= at - c["window"]
        for h in range(hkv if a else 0):
            k, v = (p[ids, h].reshape(-1, dim)[: b - low].double() for p in (s["k_pages"], s["v_pages"]))
            for g in range(h * hq // hkv, (h + 1) * hq // hkv):
                score = (s["q"][first : first + a, g].double() @ k.T / math.sqrt(dim)).masked_fill(hide, -math.inf)
                out[first : first + a, g] = torch.softmax(score, 1).nan_to_num(0.0) @ v
        first += a
    return {"out": out}


def _exact_sample(s):
    probs = []
    for r in range(s["case"]["rows"]):
        heat = s["temperature"][r].double()
        if heat <= 0:
            probs.append(torch.ones((), dtype=torch.float64, device=heat.device))
            continue
        row, order = torch.sort(s["logits"][r].double(), descending=True, stable=True)
        k = int(s["top_k"][r]) or row.numel()
        row, order = row[:k], order[:k]
        mass = torch.exp((row - row[0]) / heat)
        if s["top_p"][r] < 1:
            cdf = mass.cumsum(0)
            n = int(torch.searchsorted(cdf, s["top_p"][r].double() * cdf[-1])) + 1
            mass, order = mass[:n], order[:n]
        n = max(1, int((mass >= s["min_p"][r].double()).sum()))
        mass, order = mass[:n], order[:n]
        back = torch.sort(order).indices
        cdf = mass[back].cumsum(0)
        at = torch.searchsorted(cdf, s["u"][r].double() * cdf[-1], right=True).clamp(max=n - 1)
        probs.append(mass[back][at] / cdf[-1])
    # the id follows from comparisons of computed sums and has no 64-bit value of its own
    return {"ids": None, "probs": torch.stack(probs)}
