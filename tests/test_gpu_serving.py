"""Serving operators on the GPU against plain implementations in 64 bits.

The bounds follow from the arithmetic: u(T) is the unit roundoff of type T (half an ulp of 1).
rope_append rounds two products and a sum in fp32, then once to the output's type.  For
paged_attention see `attention_bound`.  Sampling is compared by id, except where the uniform falls
within a running sum's own error of a boundary."""
import math

import numpy as np
import pytest
import torch

from dpuf_b200 import serving

pytestmark = pytest.mark.gpu

U = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.float16, torch.bfloat16)}  # 2^-24, 2^-11, 2^-8
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
INT = torch.int32


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def table_for(lens, page, g, spare=2, width=None):
    """A table whose pages are a random permutation; entries beyond a sequence's length are -1."""
    need = [-(-n // page) for n in lens]
    width = width or max(max(need), 1)
    order = torch.randperm(sum(need) + spare, generator=g, device="cuda").to(INT)
    t = torch.full((len(lens), width), -1, dtype=INT, device="cuda")
    at = 0
    for s, n in enumerate(need):
        t[s, :n] = order[at:at + n]
        at += n
    return t, sum(need) + spare


# ---------------------------------------------------------------- rope_append
def turn64(x, cos, sin, rot, interleaved):
    """The turned x in 64 bits, and |a c| + |b s| of each element."""
    y = x.double().clone()
    size = torch.zeros_like(y)
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    p, q = x[..., a].double(), x[..., b].double()
    c, s = cos.double()[:, None], sin.double()[:, None]
    y[..., a], y[..., b] = p * c - q * s, q * c + p * s
    size[..., a], size[..., b] = (p * c).abs() + (q * s).abs(), (q * c).abs() + (p * s).abs()
    return y, size


def assert_turned(got, want, size, dtype):
    err = (got.double() - want).abs()
    # products and sum: 3 roundings of at most |a c| + |b s|; the store: one of the value (or of a subnormal)
    bound = 3 * U[F32] * size * 1.001 + U[dtype] * want.abs() * 1.01 + (2.0 ** -25 if dtype == F16 else 1e-40)
    assert bool((err <= bound).all()), float((err - bound).max())


@pytest.mark.parametrize("types", [(F32, F16, None), (F32, F32, None), (F16, F16, None), (BF16, BF16, None),
                                   (F32, F16, F16), (F32, BF16, BF16), (BF16, F32, F32)], ids=str)
@pytest.mark.parametrize("shape", [(1, 4, 2, 64, 64), (37, 6, 2, 128, 64), (129, 5, 1, 80, 80), (33, 3, 3, 72, 72),
                                   (70, 9, 3, 64, 10), (5, 8, 8, 256, 256)], ids=str)
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_append(types, shape, interleaved):
    dtype, kv_dtype, out_dtype = types
    n, hq, hkv, hd, rot = shape
    g = gen(n + rot)
    page, seqs = 16, 3
    lens = [200, 150, 260]
    table, n_pages = table_for(lens, page, g)
    cache = serving.PagedCache(normal(g, n_pages, hkv, page, hd, dtype=kv_dtype),
                               normal(g, n_pages, hkv, page, hd, dtype=kv_dtype))
    before = cache.k_pages.clone(), cache.v_pages.clone()
    # distinct places, in no order
    places = torch.cat([torch.stack([torch.full((m,), s), torch.arange(m)], 1) for s, m in enumerate(lens)])
    pick = places[torch.randperm(len(places), generator=torch.Generator().manual_seed(n))[:n]].to(INT).cuda()
    seq, pos = pick[:, 0].contiguous(), pick[:, 1].contiguous()
    cos, sin = serving.rope_table(260, rot, 1e4)
    qkv = normal(g, n, hq + 2 * hkv, hd, dtype=dtype)
    q, k, v = qkv.split([hq, hkv, hkv], 1)
    out = None if out_dtype is None else torch.empty(n, hq, hd, dtype=out_dtype, device="cuda")
    got = serving.rope_append(cache, table, q, k, v, cos, sin, seq, pos, interleaved, out)
    assert got.dtype == (out_dtype or dtype) and (out is None or got is out)
    c, s = cos[pos.long()], sin[pos.long()]
    assert_turned(got, *turn64(q, c, s, rot, interleaved), got.dtype)
    pages, rows = table[seq.long(), pos.long() // page].long(), pos.long() % page
    assert_turned(cache.k_pages[pages, :, rows], *turn64(k, c, s, rot, interleaved), kv_dtype)
    assert torch.equal(cache.v_pages[pages, :, rows], v.to(kv_dtype))
    before[0][pages, :, rows] = cache.k_pages[pages, :, rows]
    before[1][pages, :, rows] = cache.v_pages[pages, :, rows]
    assert torch.equal(before[0], cache.k_pages) and torch.equal(before[1], cache.v_pages)  # nothing else moved


def test_rope_append_unaligned_and_in_place():
    """Rows that start off 16-byte boundaries go element by element; q may be turned in place."""
    g = gen(3)
    n, hq, hkv, hd = 19, 4, 2, 64
    cache = serving.PagedCache.empty(4, hkv, 16, hd, F16)
    table = torch.tensor([[2, 0]], dtype=INT, device="cuda")
    cos, sin = serving.rope_table(32, hd)
    flat = normal(g, n, (hq + 2 * hkv) * hd + 3, dtype=F16)
    q, k, v = (x.unflatten(1, (-1, hd)) for x in flat[:, 1:-2].split([hq * hd, hkv * hd, hkv * hd], 1))
    pos = torch.arange(n, dtype=INT, device="cuda")
    seq = torch.zeros_like(pos)
    a = serving.rope_append(cache, table, q, k, v, cos, sin, seq, pos)
    ka = cache.k_pages[[2] * 16 + [0] * (n - 16), :, [i % 16 for i in range(n)]].clone()
    b = q.contiguous()
    serving.rope_append(cache, table, b, k.contiguous(), v.contiguous(), cos, sin, seq, pos, out=b)
    kb = cache.k_pages[[2] * 16 + [0] * (n - 16), :, [i % 16 for i in range(n)]]
    assert torch.equal(a, b) and torch.equal(ka, kb)  # the kernels do the same arithmetic


@pytest.mark.parametrize("hd,rot", [(128, 128), (128, 36), (80, 20), (256, 250), (8, 8)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_append_in_place(hd, rot, interleaved):
    """q turned in place equals q turned into a new tensor, with partners in other threads' runs too."""
    g = gen(rot)
    n, hq, hkv = 700, 6, 2
    cache = serving.PagedCache.empty(50, hkv, 16, hd, F16)
    table = torch.arange(50, dtype=INT, device="cuda")[None]
    cos, sin = serving.rope_table(800, rot)
    q, k, v = (normal(g, n, h, hd, dtype=F16) for h in (hq, hkv, hkv))
    pos = torch.arange(n, dtype=INT, device="cuda")
    want = serving.rope_append(cache, table, q, k, v, cos, sin, torch.zeros_like(pos), pos, interleaved)
    for _ in range(5):
        mine = q.clone()
        serving.rope_append(cache, table, mine, k, v, cos, sin, torch.zeros_like(pos), pos, interleaved, out=mine)
        assert torch.equal(mine, want)


@pytest.mark.parametrize("rot", [64, 10])  # both kernels
def test_rope_append_out_of_range(rot):
    """Padding, positions without a table row, sequences, entries and pages that are none."""
    g = gen(5)
    hq, hkv, hd, page = 4, 2, 64, 16
    cache = serving.PagedCache(normal(g, 3, hkv, page, hd, dtype=F16), normal(g, 3, hkv, page, hd, dtype=F16))
    before = cache.k_pages.clone(), cache.v_pages.clone()
    table = torch.tensor([[-1, 1, 3]], dtype=INT, device="cuda")
    cos, sin = serving.rope_table(60, rot)
    #                    padding, no row, no page, no such page, beyond the table, no such sequence (twice), held
    pos = torch.tensor([-1, 60, 5, 40, 50, 20, 20, 20], dtype=INT, device="cuda")
    seq = torch.tensor([0, 0, 0, 0, 0, 1, -1, 0], dtype=INT, device="cuda")
    q, k, v = (normal(g, 8, h, hd, dtype=F16) for h in (hq, hkv, hkv))
    out = serving.rope_append(cache, table, q, k, v, cos, sin, seq, pos)
    assert bool((out[0] == 0).all()) and bool(out[1].isnan().all()) and bool(out[2:].isfinite().all())
    assert torch.equal(cache.v_pages[1, :, 4], v[7])
    before[0][1, :, 4], before[1][1, :, 4] = cache.k_pages[1, :, 4], cache.v_pages[1, :, 4]
    assert torch.equal(before[0], cache.k_pages) and torch.equal(before[1], cache.v_pages)


# ---------------------------------------------------------------- paged_attention
def attention64(cache, table, q, q_start, kv_len, scale, causal, window):
    """Plain attention in 64 bits, sequence by sequence, and a bound on the error of each output."""
    page, hkv = cache.page_size, cache.n_kv
    n, hq, hd = q.shape
    out = torch.zeros(n, hq, hd, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(out)
    for s in range(len(kv_len)):
        first, end, total = q_start[s], q_start[s + 1], kv_len[s]
        if first == end or total == 0:
            continue
        p = torch.arange(total - (end - first), total, device="cuda")[:, None]
        low = max(0, total - (end - first) - window + 1) if window else 0  # no token of it sees less
        at = torch.arange(low, total, device="cuda")
        sees = at[None] <= p if causal else torch.ones(end - first, total - low, dtype=torch.bool, device="cuda")
        if window:
            sees = sees & (at[None] > p - window)
        pages, rows = table[s, at // page].long(), at % page
        k = cache.k_pages[pages, :, rows].double().repeat_interleave(hq // hkv, 1)
        v = cache.v_pages[pages, :, rows].double().repeat_interleave(hq // hkv, 1)
        x = q[first:end].double()
        score = (torch.einsum("thd,jhd->htj", x, k) * scale).masked_fill(~sees, -math.inf)
        w = torch.softmax(score, 2).nan_to_num(0.0)  # (a token that sees nothing)
        out[first:end] = torch.einsum("htj,jhd->thd", w, v)
        bound[first:end] = attention_bound(x, k, v, w, sees, scale, cache.dtype if q.dtype != F32 else F32, q.dtype)
    return out, bound


def attention_bound(x, k, v, w, sees, scale, p_type, out_type):
    """A score is a sum of head_dim fp32 products scaled by one more: off by e <= (head_dim + 3) u32 scale
    sum |q k|, and up to 2^-22 of |q||k| where q is split into two or three terms.  A weight is then off
    by the factor exp(2 e), by ex2's 2^-22 and by its rounding to the product's type; the two sums over n keys
    and the rescalings add n u32 each way.  The output is off by that much of sum w |v|, and by its own
    rounding."""
    hd = k.shape[2]
    n = sees.sum(1)[None]
    size_qk = torch.einsum("thd,jhd->htj", x.abs(), k.abs()).masked_fill(~sees, 0.0).amax(2)
    e = ((hd + 3) * U[F32] + 2.0 ** -22) * abs(scale) * size_qk
    rel = torch.expm1(2 * e) + 2.0 ** -20 + 2 * (n + 64) * U[F32] + (2 * U[p_type] if p_type != F32 else 0)
    rel = rel.transpose(0, 1)[:, :, None]
    size = torch.einsum("htj,jhd->thd", w, v.abs())
    return rel * size + U[out_type] * 1.01 * (size * (1 + rel)) + 2.0 ** -24


def run_attention(types, heads, hd, page, q_lens, kv_lens, causal=True, window=0, seed=0, junk=math.nan, scale=None,
                  out=None, repeats=0):
    dtype, kv_dtype = types
    hq, hkv = heads
    g = gen(seed + hd + page)
    lens = [max(0, n) for n in kv_lens]
    table, n_pages = table_for(lens, page, g)
    k, v = (normal(g, n_pages, hkv, page, hd, dtype=kv_dtype) for _ in range(2))
    # whatever stands beyond a sequence's length, in its last page and in spare pages, is never used
    used = torch.zeros(n_pages, page, dtype=torch.bool, device="cuda")
    for s, n in enumerate(lens):
        at = torch.arange(n, device="cuda")
        used[table[s, at // page].long(), at % page] = True
        if window:  # pages that lie before every window may have been given back
            gone = max(0, n - q_lens[s] - window + 1) // page
            table[s, :gone] = -1
    for x in (k, v):
        x.masked_fill_(~used[:, None, :, None], junk)
    cache = serving.PagedCache(k, v)
    q = normal(g, sum(q_lens), hq, hd, dtype=dtype, scale=2.0)
    start = [0]
    for n in q_lens:
        start.append(start[-1] + n)
    q_start = torch.tensor(start, dtype=INT, device="cuda")
    kv_len = torch.tensor(kv_lens, dtype=INT, device="cuda")
    got = serving.paged_attention(cache, table, q, q_start, kv_len, max(max(q_lens), 1), scale, causal, window, out)
    want, bound = attention64(cache, table, q, start, lens, hd ** -0.5 if scale is None else scale, causal, window)
    for _ in range(repeats):
        assert torch.equal(got, serving.paged_attention(cache, table, q, q_start, kv_len, max(max(q_lens), 1), scale,
                                                        causal, window))
    serving.attention_check()
    assert got.shape == q.shape and got.dtype == (dtype if out is None else out.dtype)
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), (float((err - bound).max()), float(err.max()))
    return got


TYPES = [(F16, F16), (BF16, BF16), (F32, F32), (F32, F16), (F32, BF16)]


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("heads", [(4, 2), (8, 1), (3, 3), (32, 8), (28, 4), (24, 1)], ids=str)
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_single_tokens(types, heads, hd):
    run_attention(types, heads, hd, 16, [1] * 7, [1, 2, 15, 16, 17, 129, 700])


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("hd", [8, 40, 72, 80, 96, 136, 192, 256])
def test_attention_head_sizes(types, hd):
    run_attention(types, (6, 2), hd, 8, [1, 5, 70], [65, 5, 203])


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256, 1024])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_pages(types, page, causal):
    run_attention(types, (4, 2), 64, page, [1, 33, 130, 7], [300, 33, 391, 1100], causal)


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("q_lens", [[2, 3], [4, 8, 1], [17], [128], [129, 1], [31, 0, 65]], ids=str)
def test_attention_chunks(types, q_lens):
    for extra in (0, 1, 100, 517):
        run_attention(types, (8, 2), 128, 16, q_lens, [n + extra for n in q_lens], seed=extra)


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("window", [1, 2, 63, 128, 400])
def test_attention_window(types, window):
    run_attention(types, (8, 2), 64, 16, [1, 1, 90, 200, 0], [1, 900, 500, 200, 77], window=window)


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("q_len,hd", [(1, 64), (1, 128), (6, 64), (200, 128)])
def test_attention_places_before_the_window(types, q_len, hd):
    """Positions in held pages that lie before every window may hold anything."""
    g = gen(31)
    dtype, kv_dtype = types
    table, n_pages = table_for([700], 64, g)
    k, v = (normal(g, n_pages, 2, 64, hd, dtype=kv_dtype) for _ in range(2))
    at = torch.arange(700 - q_len - 99, device="cuda")  # the first token sees 100 positions
    k[table[0, at // 64].long(), :, at % 64] = math.nan
    v[table[0, at // 64].long(), :, at % 64] = math.inf
    cache = serving.PagedCache(k, v)
    q = normal(g, q_len, 4, hd, dtype=dtype)
    got = serving.paged_attention(cache, table, q, torch.tensor([0, q_len], dtype=INT, device="cuda"),
                                  torch.tensor([700], dtype=INT, device="cuda"), q_len, window=100)
    want, bound = attention64(cache, table, q, [0, q_len], [700], hd ** -0.5, True, 100)
    assert bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("q_lens", [[1, 1, 0, 1], [5, 3, 0, 200]], ids=str)
def test_attention_empty_rows(types, q_lens):
    """Sequences without positions, tokens before the first position, sequences without tokens."""
    got = run_attention(types, (4, 2), 64, 16, q_lens, [0, 2, 40, 150])
    assert bool((got[: q_lens[0]] == 0).all())
    got = run_attention(types, (4, 2), 64, 16, q_lens, [0, 2, 40, 150], causal=False)
    assert bool((got[: q_lens[0]] == 0).all())
    got = run_attention(types, (4, 2), 64, 16, q_lens, [0, 2, 40, 150], window=3)
    assert bool((got[: q_lens[0]] == 0).all())


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("q_len", [1, 6, 200])
@pytest.mark.parametrize("before", [102, 9102])  # positions before the new tokens: one part, several
def test_attention_values_that_are_not_finite(types, hd, q_len, before):
    """A NaN or infinite query gives NaN in its own row alone; a NaN key in every row that sees it, also where it is
    all that the row sees of a block of keys (position 63 of a window of 40 that begins there)."""
    g = gen(hd + q_len)
    dtype, kv_dtype = types
    total, hq, hkv = before + q_len, 8, 2
    table, n_pages = table_for([total], 16, g)
    k, v = (normal(g, n_pages, hkv, 16, hd, dtype=kv_dtype) for _ in range(2))
    cache = serving.PagedCache(k, v)
    q = normal(g, q_len, hq, hd, dtype=dtype)
    start, kv = torch.tensor([0, q_len], dtype=INT, device="cuda"), torch.tensor([total], dtype=INT, device="cuda")
    want, bound = attention64(cache, table, q, [0, q_len], [total], hd ** -0.5, True, 0)
    token = q_len // 2
    for value, dim in ((math.nan, 0), (math.inf, hd - 1), (-math.inf, 5)):
        bad = q.clone()
        bad[token, 3, dim] = value  # (of the 100 keys and more that it sees, some have a score of +infinity)
        got = serving.paged_attention(cache, table, bad, start, kv, q_len)
        assert bool(got[token, 3].isnan().all()), value
        got[token, 3] = want[token, 3].to(got.dtype)
        assert bool(((got.double() - want).abs() <= bound).all()), value
    for at, window in ((0, 0), (before - 39, 40)):
        held = k[table[0, at // 16].long(), 1, at % 16].clone()
        k[table[0, at // 16].long(), 1, at % 16] = math.nan
        got = serving.paged_attention(cache, table, q, start, kv, q_len, window=window)
        k[table[0, at // 16].long(), 1, at % 16] = held
        sees = at - before + window if window else q_len  # tokens t < sees: at > before + t - window
        assert bool(got[:sees, 4:].isnan().all()), window


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("junk", [math.inf, -math.inf, 6e4])
def test_attention_unused_places(types, junk):
    run_attention(types, (8, 2), 64, 32, [1, 77, 1], [45, 201, 3], junk=junk)


@pytest.mark.parametrize("types", [(F16, F16), (BF16, BF16), (F32, F32), (F32, F16)], ids=str)
@pytest.mark.parametrize("q_len", [1, 6, 300])
def test_attention_long_axis(types, q_len):
    """Few rows over a long axis (joined parts) give what many short runs would."""
    run_attention(types, (8, 2), 64, 64, [q_len], [20011])


@pytest.mark.parametrize("q_lens", [[1] * 300, [2, 0, 1] * 100], ids=["ones", "mixed"])
def test_attention_many_sequences(q_lens):
    rng = np.random.RandomState(3)
    run_attention((F16, F16), (4, 1), 64, 16, q_lens, [int(n) + rng.randint(0, 90) for n in q_lens])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,q_lens", [((8, 2), [8]), ((8, 2), [40, 8]), ((8, 2), [64, 5, 32, 9]), ((3, 3), [17]),
                                          ((3, 3), [130, 17, 256]), ((6, 2), [100, 6, 6])], ids=str)
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_many_items_a_cta(dtype, heads, q_lens, hd):
    """Far more items than CTAs: a CTA runs through items of one tile and of two, whole and in parts, in
    every order, and does so again."""
    rng = np.random.RandomState(hd)
    q = [q_lens[i % len(q_lens)] for i in range(500)]
    kv = [n + rng.randint(0, 150) for n in q]
    run_attention((dtype, dtype), heads, hd, 16, q, kv, repeats=30)


@pytest.mark.parametrize("heads,q_lens", [((8, 2), [40, 9]), ((8, 2), [64, 128, 31]), ((3, 3), [256, 127]), ((16, 1), [16, 5])],
                         ids=str)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("wide", [False, True])
def test_attention_results_by_way_of_the_queries_buffer(heads, q_lens, hd, wide):
    """Partial tiles, and all tiles of fp32 results, pass through the shared memory that the queries of the item
    after next arrive in: many items a CTA, queries by TMA (the group divides 128)."""
    rng = np.random.RandomState(hd)
    q = [q_lens[i % len(q_lens)] for i in range(400)]
    kv = [n + rng.randint(0, 20) for n in q]
    out = torch.empty(sum(q), heads[0], hd, dtype=F32, device="cuda") if wide else None
    got = run_attention((F16, F16), heads, hd, 16, q, kv, out=out, repeats=0 if wide else 20)
    if wide:  # rounded once more it is the narrow result
        assert torch.equal(got.half(), run_attention((F16, F16), heads, hd, 16, q, kv, repeats=20))


@pytest.mark.parametrize("heads,seqs,q_len,kv_len", [((3, 3), 49, 216, 216), ((3, 3), 58, 216, 300), ((4, 2), 20, 70, 900),
                                                      ((4, 1), 37, 100, 1100), ((2, 2), 41, 257, 777), ((8, 2), 1, 333, 2500)])
def test_attention_cuts_at_item_ends(heads, seqs, q_len, kv_len):
    """Items from a few key blocks to some forty, so that the cuts between CTAs fall at every distance from
    an item's ends: moved there, or left where they are with several in one item."""
    run_attention((F16, F16), heads, 64, 32, [q_len] * seqs, [kv_len - 3 * i % q_len for i in range(seqs)], repeats=3)


@pytest.mark.parametrize("types", TYPES, ids=str)
def test_attention_scale_and_out(types):
    out = torch.empty(9, 4, 64, dtype=F32, device="cuda")
    run_attention(types, (4, 2), 64, 16, [1, 8], [50, 60], scale=0.31, out=out)
    run_attention(types, (4, 2), 64, 16, [9], [60], scale=0.0)
    run_attention(types, (4, 2), 64, 16, [3, 150], [60, 170], scale=-0.2)


@pytest.mark.parametrize("types", [(F32, F16), (F32, BF16), (F32, F32)], ids=str)
@pytest.mark.parametrize("size", [1e-6, 1e6])
def test_attention_range_of_q(types, size):
    """fp32 queries outside the range of the cache's type, with a scale that makes up for it."""
    g = gen(9)
    cache = serving.PagedCache(normal(g, 3, 2, 16, 64, dtype=types[1]), normal(g, 3, 2, 16, 64, dtype=types[1]))
    table = torch.tensor([[0, 2, 1]], dtype=INT, device="cuda")
    q = normal(g, 2, 4, 64, scale=size)
    start, kv = torch.tensor([0, 2], dtype=INT, device="cuda"), torch.tensor([40], dtype=INT, device="cuda")
    got = serving.paged_attention(cache, table, q, start, kv, 2, scale=0.125 / size)
    want, bound = attention64(cache, table, q, [0, 2], [40], 0.125 / size, True, 0)
    assert bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("types", [(F16, F16), (F32, F32)], ids=str)
@pytest.mark.parametrize("q_len", [1, 200])
def test_attention_strides(types, q_len):
    """q as a slice of a fused projection, a cache whose keys and values lie in one tensor token by token."""
    g = gen(11)
    dtype, kv_dtype = types
    hq, hkv, hd, page, n_pages = 8, 2, 64, 16, 20
    pool = normal(g, n_pages, page, 2, hkv, hd, dtype=kv_dtype)
    cache = serving.PagedCache(pool[:, :, 0].transpose(1, 2), pool[:, :, 1].transpose(1, 2))
    wide = torch.randperm(n_pages, generator=g, device="cuda").to(INT)[:14].expand(2, 14).contiguous()
    table = wide[:1, :14]
    q = normal(g, q_len, hq + 2 * hkv, hd, dtype=dtype)[:, 2 : 2 + hq]
    start = torch.tensor([0, q_len], dtype=INT, device="cuda")
    got = serving.paged_attention(cache, table, q, start, torch.tensor([211], dtype=INT, device="cuda"), q_len)
    want, bound = attention64(cache, table, q, [0, q_len], [211], hd ** -0.5, True, 0)
    assert bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("q_len", [1, 150])
def test_attention_offsets_past_32_bits(q_len):
    """Pages whose element offsets do not fit 32 bits."""
    hkv, page, hd = 8, 64, 128
    n_pages = (1 << 32) // (hkv * page * hd) + 40
    k = torch.zeros(n_pages, hkv, page, hd, dtype=F16, device="cuda")
    v = torch.zeros_like(k)
    cache = serving.PagedCache(k, v)
    g = gen(12)
    table = torch.tensor([[n_pages - 1, 3, n_pages - 7, n_pages // 2 + 1]], dtype=INT, device="cuda")
    kk, vv = (normal(g, 200, hkv, hd, dtype=F16) for _ in range(2))
    cos, sin = serving.rope_table(256, hd)
    pos = torch.arange(200, dtype=INT, device="cuda")
    q = normal(g, 200, 16, hd, dtype=F16)
    q = serving.rope_append(cache, table, q, kk, vv, cos, sin, torch.zeros_like(pos), pos)[200 - q_len:]
    assert torch.equal(v[n_pages - 7, :, 5], vv[133])
    got = serving.paged_attention(cache, table, q, torch.tensor([0, q_len], dtype=INT, device="cuda"),
                                  torch.tensor([200], dtype=INT, device="cuda"), q_len)
    want, bound = attention64(cache, table, q, [0, q_len], [200], hd ** -0.5, True, 0)
    assert bool(((got.double() - want).abs() <= bound).all())


def attention_inputs(q_len=1, seqs=5, dtype=F16):
    g = gen(21)
    lens = [300 + 211 * s for s in range(seqs)]
    table, n_pages = table_for(lens, 16, g)
    cache = serving.PagedCache(normal(g, n_pages, 2, 16, 64, dtype=dtype), normal(g, n_pages, 2, 16, 64, dtype=dtype))
    q = normal(g, q_len * seqs, 8, 64, dtype=dtype)
    start = torch.arange(0, q_len * seqs + 1, q_len, dtype=INT, device="cuda")
    return cache, table, q, start, torch.tensor(lens, dtype=INT, device="cuda"), q_len


@pytest.mark.parametrize("q_len", [1, 100])
def test_attention_repeats_bit_for_bit(q_len):
    args = attention_inputs(q_len)
    first = serving.paged_attention(*args)
    for _ in range(20):
        assert torch.equal(first, serving.paged_attention(*args))


@pytest.mark.parametrize("q_len", [1, 100])
def test_attention_on_streams_and_in_a_graph(q_len):
    args = attention_inputs(q_len)
    want = serving.paged_attention(*args)
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    torch.cuda.synchronize()
    for _ in range(5):
        for s in streams:  # several calls in flight, each stream with a workspace of its own
            with torch.cuda.stream(s):
                got.append(serving.paged_attention(*args))
    torch.cuda.synchronize()
    assert all(torch.equal(want, x) for x in got)
    out = torch.zeros_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(streams[0]):
        with torch.cuda.graph(graph, stream=streams[0]):
            serving.paged_attention(*args, out=out)
        graph.replay()
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(want, out)


@pytest.mark.parametrize("q_len", [1, 100])
def test_attention_graph_keeps_off_its_streams_workspace(q_len):
    """A graph's calls share nothing with later calls on the stream that it was captured on."""
    args = attention_inputs(q_len)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        want = serving.paged_attention(*args)
        out = torch.zeros_like(want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            serving.paged_attention(*args, out=out)
    held = [w[0] for key, w in serving._workspaces.items() if key[1] == s.cuda_stream]
    torch.cuda.synchronize()
    assert len(held) == 1
    held[0][256:5000] = 255  # as another call in flight may have them: the counters
    graph.replay()  # (once: a second call would find the first one's parts of the same inputs)
    torch.cuda.synchronize()
    held[0][256:5000] = 0
    assert torch.equal(want, out)


@pytest.mark.parametrize("q_len", [1, 100])
@pytest.mark.parametrize("given", [False, True])
def test_attention_graphs_of_one_stream_on_two(q_len, given):
    """Graphs captured one after the other on one stream, replayed on two at once while the first is in use too."""
    home, others = torch.cuda.Stream(), [torch.cuda.Stream() for _ in range(2)]
    sets = [attention_inputs(q_len, seqs) for seqs in (5, 9, 14)]
    want = [serving.paged_attention(*args) for args in sets]
    torch.cuda.synchronize()
    outs, graphs, spaces = [torch.zeros_like(w) for w in want], [], []
    for args, out in zip(sets[:2], outs):
        spaces.append(serving.attention_workspace() if given else None)
        graphs.append(torch.cuda.CUDAGraph())
        torch.cuda.synchronize()
        with torch.cuda.graph(graphs[-1], stream=home):
            for _ in range(3):
                serving.paged_attention(*args, out=out, workspace=spaces[-1])
    for _ in range(20):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for _ in range(5):
            for g, s in zip(graphs, others):
                with torch.cuda.stream(s):
                    g.replay()
            with torch.cuda.stream(home):
                serving.paged_attention(*sets[2], out=outs[2])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, outs))
    for ws in spaces:
        if ws is not None:
            serving.attention_check(workspace=ws)


@pytest.mark.parametrize("q_len", [1, 100])
def test_attention_workspace_after_a_wait_gave_up(q_len):
    """The error word set and the counters left anywhere, as a kernel that gave up leaves them: the check says so
    once and makes the workspace ready for use."""
    args = attention_inputs(q_len)
    want = serving.paged_attention(*args)
    ws = serving.attention_workspace()
    for _ in range(2):
        assert torch.equal(want, serving.paged_attention(*args, workspace=ws))
        serving.attention_check(workspace=ws)
        ws[:1] = 1
        ws[256:5000:4] = 3
        with pytest.raises(RuntimeError, match="gave up"):
            serving.attention_check(workspace=ws)
        serving.attention_check(workspace=ws)
    for error, bad in ((TypeError, ws.view(torch.int32)), (ValueError, ws[:-1]), (ValueError, ws.cpu()),
                       (ValueError, torch.zeros(ws.numel() + 1, dtype=torch.uint8, device="cuda")[1:]),
                       (ValueError, ws[None]), (ValueError, torch.zeros(2 * ws.numel(), dtype=torch.uint8, device="cuda")[::2])):
        with pytest.raises(error):
            serving.paged_attention(*args, workspace=bad)
        with pytest.raises(error):
            serving.attention_check(workspace=bad)


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("q_len", [1, 6, 100])
@pytest.mark.parametrize("hd", [64, 72, 136])
def test_attention_rows_of_no_sequence(types, q_len, hd):
    """Tokens before the first sequence's and after the last one's, as a padded batch has them, get zeros."""
    g = gen(hd)
    lens = [q_len + 90 * s for s in range(4)]
    table, n_pages = table_for(lens, 16, g)
    cache = serving.PagedCache(*(normal(g, n_pages, 3, 16, hd, dtype=types[1]) for _ in range(2)))
    n = q_len * len(lens)
    start = torch.arange(0, n + 1, q_len, dtype=INT, device="cuda")
    kv = torch.tensor(lens, dtype=INT, device="cuda")
    for before, after in ((0, 1), (3, 0), (2, 700)):
        q = normal(g, before + n + after, 6, hd, dtype=types[0])
        want = serving.paged_attention(cache, table, q[before : before + n], start, kv, q_len)
        for out_type in {types[0], F32}:
            out = torch.full_like(q, 7.0, dtype=out_type)
            serving.paged_attention(cache, table, q, start + before, kv, q_len, out=out)
            assert bool((out[:before] == 0).all()) and bool((out[before + n :] == 0).all())
            assert torch.equal(out[before : before + n].to(types[0]), want)
    nobody = torch.zeros(5, dtype=INT, device="cuda")  # all of them
    out = torch.full_like(q, 7.0)
    serving.paged_attention(cache, table, q, nobody, kv, q_len, out=out)
    assert bool((out == 0).all())


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("max_q", [1, 5, 100000])
def test_attention_max_q_that_is_not_the_longest(types, hd, max_q):
    """max_q chooses the kernel; sequences with more tokens than it says are computed all the same."""
    g = gen(hd + max_q)
    q_lens, lens = [1, 40, 7, 150], [30, 61, 7, 400]
    table, n_pages = table_for(lens, 16, g)
    cache = serving.PagedCache(*(normal(g, n_pages, 2, 16, hd, dtype=types[1]) for _ in range(2)))
    start = [0, 1, 41, 48, 198]
    q = normal(g, 198, 4, hd, dtype=types[0])
    for window in (0, 33):
        out = torch.full_like(q, math.nan)
        serving.paged_attention(cache, table, q, torch.tensor(start, dtype=INT, device="cuda"),
                                torch.tensor(lens, dtype=INT, device="cuda"), max_q, window=window, out=out)
        want, bound = attention64(cache, table, q, start, lens, hd ** -0.5, True, window)
        assert bool(((out.double() - want).abs() <= bound).all())


def test_attention_lengths_that_do_not_fit():
    """Lengths and starts are read on the device: ones beyond the table or the tokens are cut off."""
    cache, table, q, start, kv, _ = attention_inputs()
    held = table.shape[1] * 16
    want = serving.paged_attention(cache, table, q, start, kv.clamp(max=held), 1)
    kv2 = kv.clone()
    kv2[-1] = held + 5
    got = serving.paged_attention(cache, table, q, start, kv2, 1)
    assert torch.equal(got[:-1], want[:-1]) and bool(got.isfinite().all())
    start2 = start.clone()
    start2[-1] = 1000
    serving.paged_attention(cache, table, q, start2, kv, 1)
    kv2[0] = -3
    assert bool((serving.paged_attention(cache, table, q, start, kv2, 1)[0] == 0).all())


@pytest.mark.parametrize("seqs,width", [(0, 4), (0, 0), (3, 0), (3, 4)])
def test_a_batch_without_tokens(seqs, width):
    cache = serving.PagedCache.empty(4, 2, 16, 64)
    table = torch.zeros(seqs, width, dtype=INT, device="cuda")
    q, k = torch.zeros(0, 4, 64, dtype=F16, device="cuda"), torch.zeros(0, 2, 64, dtype=F16, device="cuda")
    cos, sin = serving.rope_table(8, 64)
    none = torch.zeros(0, dtype=INT, device="cuda")
    assert serving.rope_append(cache, table, q, k, k, cos, sin, none, none).shape == (0, 4, 64)
    start, kv = torch.zeros(seqs + 1, dtype=INT, device="cuda"), torch.zeros(seqs, dtype=INT, device="cuda")
    assert serving.paged_attention(cache, table, q, start, kv, 1).shape == (0, 4, 64)
    ids, probs = serving.sample(torch.zeros(0, 100, device="cuda"), torch.zeros(0, device="cuda"))
    assert ids.shape == probs.shape == (0,)


def test_attention_refusals():
    cache, table, q, start, kv, n = attention_inputs()
    ok = (cache, table, q, start, kv, n)

    def bad(error, at, value, **more):
        args = list(ok)
        args[at] = value
        with pytest.raises(error):
            serving.paged_attention(*args, **more)

    bad(TypeError, 1, table.long())
    bad(ValueError, 1, table[:, ::2])
    bad(ValueError, 1, table.cpu())
    bad(ValueError, 2, q[:, :, :32])
    bad(TypeError, 2, q.bfloat16())
    bad(ValueError, 2, q[:, :3])
    bad(ValueError, 2, q.transpose(1, 2).contiguous().transpose(1, 2))
    bad(TypeError, 3, start.long())
    bad(ValueError, 3, start[:-1].contiguous())
    bad(ValueError, 4, kv[:-1].contiguous())
    bad(ValueError, 5, 0)
    bad(ValueError, 5, n, window=-1)
    bad(ValueError, 5, n, window=4, causal=False)
    bad(ValueError, 5, n, scale=math.nan)
    bad(ValueError, 5, n, out=torch.empty(1, 2, device="cuda"))
    bad(TypeError, 5, n, out=torch.empty_like(q, dtype=BF16))


def test_rope_and_sample_refusals():
    cache = serving.PagedCache.empty(4, 2, 16, 64)
    table = torch.zeros(1, 2, dtype=INT, device="cuda")
    q, k = torch.zeros(1, 4, 64, dtype=F16, device="cuda"), torch.zeros(1, 2, 64, dtype=F16, device="cuda")
    cos, sin = serving.rope_table(8, 64)
    z = torch.zeros(1, dtype=INT, device="cuda")
    ok = [cache, table, q, k, k, cos, sin, z, z]
    for error, at, value in ((ValueError, 2, q[:, :, :32]), (ValueError, 3, q), (TypeError, 4, k.float()),
                             (TypeError, 5, cos.half()), (ValueError, 6, sin[:4].contiguous()), (TypeError, 7, z.long()),
                             (ValueError, 8, z.cpu()), (ValueError, 5, cos.repeat(1, 2))):
        args = list(ok)
        args[at] = value
        with pytest.raises(error):
            serving.rope_append(*args)
    x, u = torch.zeros(2, 8, device="cuda"), torch.zeros(2, device="cuda")
    for error, args in ((TypeError, (x.double(), u)), (TypeError, (x, None)), (TypeError, (x, u.double())),
                        (ValueError, (x, u[:1])), (ValueError, (x[0], u)), (ValueError, (x.t().contiguous().t(), u)),
                        (TypeError, (x, u, None, u)), (ValueError, (x.cpu(), u)),
                        (ValueError, (torch.zeros(2, (1 << 20) + 1, device="cuda"), u))):
        with pytest.raises(error):
            serving.sample(*args)
    with pytest.raises(ValueError):
        serving.PagedCache.empty(4, 2, 24, 64)
    with pytest.raises(ValueError):
        serving.PagedCache.empty(4, 2, 16, 60)


# ---------------------------------------------------------------- sample
def kept64(row, temp, k, p, m):
    """Indices kept (index order) and their weights, in 64 bits."""
    row = row.astype(np.float64)
    row = np.where(np.isnan(row), -np.inf, row)
    order = np.lexsort((np.arange(row.size), -row))
    top = row[order[0]]
    with np.errstate(invalid="ignore"):
        w = np.where(row == top, 1.0, np.exp((row - top) / temp))
    order = order[: k if k >= 1 else row.size]
    if p < 1:
        run = np.cumsum(w[order])
        n = int(np.searchsorted(run, p * run[-1])) + 1
        order = order[: max(1, n)]
    order = order[w[order] >= min(m, 1.0)]
    keep = np.sort(order)
    return keep, w[keep]


def check_rows(logits, u, temp=None, k=None, p=None, m=None):
    rows = logits.shape[0]
    dev = lambda x, t: None if x is None else torch.tensor(x, dtype=t, device="cuda")  # noqa: E731
    ids, probs = serving.sample(logits, dev(u, F32), dev(temp, F32), dev(k, INT), dev(p, F32), dev(m, F32))
    again = serving.sample(logits, dev(u, F32), dev(temp, F32), dev(k, INT), dev(p, F32), dev(m, F32))
    assert torch.equal(ids, again[0]) and torch.equal(probs, again[1])
    host = logits.float().cpu().numpy()
    ids, probs = ids.cpu().numpy(), probs.cpu().numpy().astype(np.float64)
    f32 = lambda x: float(np.float32(x))  # noqa: E731
    for r in range(rows):
        t = 1.0 if temp is None else f32(temp[r])
        if t <= 0:
            assert ids[r] == int(np.argmax(host[r])) and probs[r] == 1.0
            continue
        keep, w = kept64(host[r], t, 0 if k is None else k[r], 1.0 if p is None else f32(p[r]),
                         0.0 if m is None else f32(m[r]))
        total = w.sum()
        at = int(np.searchsorted(keep, ids[r]))
        # weights are off by (l - m) / T rounded twice, |x| <= 44 ln 2 + 1, and by expf's 2 ulp
        eps = (32 * 2 ** -23 + 2.0 ** -22) * total
        high = np.cumsum(w)
        target = f32(u[r]) * total
        if at < keep.size and keep[at] == ids[r]:
            assert high[at] - w[at] - eps <= target <= high[at] + eps, (r, ids[r])
            assert abs(probs[r] - w[at] / total) <= 2e-5 * w[at] / total + 1e-12
        else:  # only an entry whose place at the threshold hangs on the sums' error
            full = kept64(host[r], t, 0, 1.0, 0.0)[1].sum()
            assert p is not None or m is not None, (r, ids[r])
            loose = kept64(host[r], t, 0 if k is None else k[r], 1.0 if p is None else f32(p[r]) + eps / full,
                           0.0 if m is None else f32(m[r]) * (1 - 1e-5))[0]
            assert ids[r] in loose, (r, ids[r])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [1, 2, 7, 511, 4096, 4097, 32000, 151936, 262147])
def test_sample_filters(dtype, vocab):
    rng = np.random.RandomState(vocab)
    rows = 24
    logits = (torch.from_numpy(rng.standard_normal((rows, vocab)).astype(np.float32)) * 3).to(dtype).cuda()
    u = rng.random_sample(rows).astype(np.float32)
    temp = rng.choice([0.0, 0.3, 0.7, 1.0, 1.7, 8.0], rows).astype(np.float32)
    k = rng.choice([0, 1, 2, 50, 1000, 10 ** 6], rows).astype(np.int32)
    p = rng.choice([1.0, 0.0, 0.1, 0.5, 0.9, 0.99, 2.0], rows).astype(np.float32)
    m = rng.choice([0.0, 0.0, 0.01, 0.2, 1.0, 3.0], rows).astype(np.float32)
    check_rows(logits, u)
    check_rows(logits, u, temp)
    check_rows(logits, u, temp, k)
    check_rows(logits, u, temp, None, p)
    check_rows(logits, u, None, None, None, m)
    check_rows(logits, u, temp, k, p, m)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [300, 20000])
def test_sample_ties_go_to_the_lowest_index(dtype, vocab):
    """Few distinct values: the kept part of a class of equal entries is its lowest indices."""
    rng = np.random.RandomState(5)
    row = torch.from_numpy(rng.randint(0, 4, vocab).astype(np.float32))
    rows = 128
    u = (np.arange(rows) + 0.5).astype(np.float32) / rows
    logits = row.to(dtype).cuda().expand(rows, vocab).contiguous()
    for k in (1, 2, vocab // 8, vocab // 2, vocab - 1):
        check_rows(logits, u, None, [k] * rows)
    for p in (0.03, 0.31, 0.77):
        check_rows(logits, u, None, None, [p] * rows)
    check_rows(logits, u, None, [vocab // 3] * rows, [0.6] * rows)
    # the whole row equal: u = i / rows picks along the first k
    same = torch.zeros(rows, vocab, dtype=dtype, device="cuda")
    ids, probs = serving.sample(same, torch.tensor(u, device="cuda"), None,
                                torch.full((rows,), 64, dtype=INT, device="cuda"))
    assert ids.tolist() == [int(x * 64) for x in u] and bool((probs == 1 / 64).all())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("spread", [0.01, 0.3, 1.0, 2.0])
def test_sample_large_nuclei(dtype, spread):
    """Flat rows: a nucleus of much of the vocabulary, which no CTA can be handed."""
    rng = np.random.RandomState(int(100 * spread))
    for vocab in (3001, 90000, 151936):
        logits = (torch.from_numpy(rng.standard_normal((8, vocab)).astype(np.float32)) * spread).to(dtype).cuda()
        u = rng.random_sample(8).astype(np.float32)
        temp = rng.choice([0.5, 1.0, 1.5], 8).astype(np.float32)
        for p in (0.5, 0.9, 0.99, 0.9999):
            check_rows(logits, u, temp, None, [p] * 8)
        check_rows(logits, u, temp, [vocab // 2] * 8, [0.97] * 8)
        check_rows(logits, u, temp, None, [0.97] * 8, [0.05] * 8)


def test_sample_rows_beyond_shared_memory():
    """The longest rows do not fit the cluster's shared memory: what does not is read again."""
    rng = np.random.RandomState(4)
    logits = (torch.from_numpy(rng.standard_normal((3, 1 << 20)).astype(np.float32)) * 2).cuda()
    u = rng.random_sample(3).astype(np.float32)
    check_rows(logits, u)
    check_rows(logits, u, None, [40] * 3, [0.9] * 3)
    check_rows(logits, u, None, None, [0.95] * 3)
    check_rows(logits[:, 1:], u, None, [100000] * 3, [0.99] * 3)


def test_sample_unusual_values():
    inf, nan = math.inf, math.nan
    rows = [[-inf] * 5, [nan] * 5, [-inf, 2, -inf, -inf, 1], [nan, 1, nan, 0.5, -inf], [inf, 3, inf, -inf, nan],
            [-3e38, 3e38, 0, 0, 0], [1e-38, 0.0, -0.0, -1e-38, -1e9], [-1e9] * 5]
    logits = torch.tensor(rows, device="cuda")
    n = len(rows)
    for u in (0.0, 0.49, 0.9999999):
        ids, probs = serving.sample(logits, torch.full((n,), u, device="cuda"))
        ids, probs = ids.tolist(), probs.tolist()
        assert ids[0] == ids[1] == -1 and probs[0] == probs[1] == 0
        assert ids[2] in (1, 4) and ids[3] in (1, 3) and ids[4] == (0 if u < 0.5 else 2) and probs[4] == 0.5
        assert ids[5] == 1 and probs[5] == 1.0
        assert ids[6] == int(u * 4) and ids[7] == int(u * 5)
    one = torch.full((n,), 1.0, device="cuda")
    assert serving.sample(logits, one)[0].tolist()[4:] == [2, 1, 3, 4]  # u = 1 is taken for the last kept
    k = torch.ones(n, dtype=INT, device="cuda")
    assert serving.sample(logits, one, None, k)[0].tolist() == [-1, -1, 1, 1, 0, 1, 0, 0]
    greedy = torch.zeros(n, device="cuda")
    assert serving.sample(logits, one, greedy)[0].tolist() == [-1, -1, 1, 1, 0, 1, 0, 0]
    assert serving.sample(logits, one, greedy - 1)[0].tolist() == [-1, -1, 1, 1, 0, 1, 0, 0]
    hot, cold = torch.full((n,), inf, device="cuda"), torch.full((n,), 1e-45, device="cuda")
    assert serving.sample(logits, one, cold)[0].tolist() == [-1, -1, 1, 1, 2, 1, 0, 4]
    assert serving.sample(logits, greedy, hot)[0].tolist()[2:4] == [1, 1]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_sample_steps_without_a_finite_factor(dtype):
    """Infinite maxima, and temperatures whose reciprocal times the histogram's steps is beyond fp32."""
    rng = np.random.RandomState(12)
    logits = torch.from_numpy(rng.standard_normal((8, 40000)).astype(np.float32))
    endless = logits.to(dtype)
    endless[:, 17::97] = math.inf
    endless[:, 5::89] = math.nan
    u = rng.random_sample(8).astype(np.float32)
    for k, p in ((None, None), ([3] * 8, None), ([700] * 8, [0.9] * 8), ([20000] * 8, [0.5] * 8), (None, [0.9] * 8)):
        check_rows(endless.cuda(), u, None, k, p)
        if dtype != F16:  # (fp16 has no such values)
            check_rows((logits * 1e-37).to(dtype).cuda(), u, [1e-37] * 8, k, p)


def test_sample_masked_logits():
    """Rows whose entries are masked with the type's lowest value, or -1e9 as the engine's early exit leaves them."""
    rng = np.random.RandomState(8)
    for dtype, low in ((F32, -1e9), (F32, float(torch.finfo(F32).min)), (F16, float(torch.finfo(F16).min)),
                       (BF16, float(torch.finfo(BF16).min))):
        logits = torch.from_numpy(rng.standard_normal((16, 50000)).astype(np.float32)).to(dtype)
        logits[:, 1000:] = low
        logits[3] = low
        u = rng.random_sample(16).astype(np.float32)
        for k, p in ((None, None), ([40] * 16, None), (None, [0.8] * 16), ([3000] * 16, [0.8] * 16)):
            check_rows(logits.cuda(), u, None, k, p)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [3000, 20000, 151936])  # 1, 8 and 16 CTAs a row
def test_sample_flat_rows_with_min_p(dtype, vocab):
    """Equal and nearly equal logits, and very high temperatures: the histogram's steps are then so narrow that
    -ln(min_p) of them are more than an integer counts.  top_p ends half an entry's weight from the next (the
    fp32 weights' error adds up to 2^-24 vocab < 0.01 of one)."""
    rows, k = 6, vocab // 3
    rng = np.random.RandomState(vocab)
    u = rng.random_sample(rows).astype(np.float32)
    share = lambda p, n: [(math.floor(p * n) + 0.5) / n] * rows  # noqa: E731
    near = torch.from_numpy(rng.randint(0, 3, (rows, vocab)).astype(np.float32)) * 2.0 ** -20
    same = torch.zeros(rows, vocab)
    spread = torch.from_numpy(rng.standard_normal((rows, vocab)).astype(np.float32))
    for logits, temp in ((same, None), (same - 1e4, None), (near, None), (near + 1, None), (spread, 1e7), (spread, 1e30)):
        logits, temp = logits.to(dtype).cuda(), None if temp is None else [temp] * rows
        for m in (1e-30, 0.05) if temp else (1e-30, 0.05, 0.2, 1.0):  # (hot weights may round to 1)
            check_rows(logits, u, temp, None, share(0.9, vocab), [m] * rows)
        check_rows(logits, u, temp, [k] * rows, None, [0.05] * rows)
        check_rows(logits, u, temp, [k] * rows, share(0.7, k), [0.05] * rows)
        check_rows(logits, u, temp, None, None, [0.05] * rows)


def test_sample_strided_rows():
    rng = np.random.RandomState(9)
    wide = torch.from_numpy(rng.standard_normal((6, 5003)).astype(np.float32)).half().cuda()
    u = rng.random_sample(6).astype(np.float32)
    check_rows(wide[:, 1:-2], u, None, [20] * 6, [0.9] * 6)
    check_rows(wide[::2, 3:], u[:3], None, None, [0.9] * 3)
    check_rows(wide[:1].expand(6, 5003), u)


def test_sample_follows_the_weights():
    """Frequencies over many uniforms: 2^16 evenly spread u reproduce each share to within 1 / 2^16 per entry."""
    row = torch.tensor([0.0, 1.0, 2.0, -1.0, 0.5], device="cuda")
    n = 1 << 16
    u = (torch.arange(n, device="cuda", dtype=torch.float32) + 0.5) / n
    ids, probs = serving.sample(row.expand(n, 5), u)
    share = torch.softmax(row.double(), 0)
    count = torch.bincount(ids.long(), minlength=5).double() / n
    assert bool(((count - share).abs() <= 1.0 / n + 1e-6).all())
    assert bool(((probs.double() - share[ids.long()]).abs() <= 1e-6).all())


def test_serving_on_another_stream():
    g = gen(2)
    s = torch.cuda.Stream()
    logits, u = normal(g, 4, 1000), torch.rand(4, generator=g, device="cuda")
    want = serving.sample(logits, u)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        got = serving.sample(logits, u)
    s.synchronize()
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
