"""GPU: the serving-step operators at the ends of their ranges: temperatures
and offsets of logits, long rows of small probabilities, drafts that are not
finite, cache layouts and batches beyond one pass of a search.

Tolerances come from the arithmetic, as in test_gpu_serving.py.
"""
from __future__ import annotations

import math

import pytest

from test_gpu_serving import (BF16, F16, F32, TYPES, U, Batch, check_logprobs, dt, gen, i32, i64, randn, u_of,
                              ws)  # noqa: F401 (ws is a fixture)

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# log probabilities
# ---------------------------------------------------------------------------
def logprobs_held_to_64_bits(ctx, bh, ws, logits, k, scale):
    import torch

    rows, vocab = logits.shape
    tokens = torch.randint(0, vocab, (rows, 2), generator=gen(vocab), device="cuda", dtype=torch.int32)
    r = bh.token_logprobs(ctx, ws, logits, tokens, k, scale)

    def out_of_range(got, ids):
        """A log probability below what fp32 holds is -inf in it; here the 64-bit value takes its place."""
        u = logits.double() * scale
        exact = u.gather(1, ids.long()) - u.amax(1, keepdim=True)
        below = (got == -math.inf) & exact.isfinite() & (exact < torch.finfo(torch.float32).min)
        return torch.where(below, exact, got.double())

    check_logprobs(logits, tokens, r._replace(logprob=out_of_range(r.logprob, tokens),
                                              top_logprob=out_of_range(r.top_logprob, r.top_ids)), k, scale)
    assert ctx.status() == 0


@pytest.mark.parametrize("type_", [F32, F16, BF16])
@pytest.mark.parametrize("rows,vocab", [(3, 32768), (700, 4096)])
@pytest.mark.parametrize("scale", [0.01, 20.0, 100.0, 1e4, 1e6])
def test_logprobs_of_any_temperature(ctx, bh, ws, type_, rows, vocab, scale):
    """Products of maximum and scale that fp32 does not hold to a part of a nat."""
    logprobs_held_to_64_bits(ctx, bh, ws, randn(gen(vocab), rows, vocab, dtype=type_, scale=4.0), 8, scale)


@pytest.mark.parametrize("type_,offset", [(F32, 1e3), (F32, -1e3), (F32, 1e5), (F32, -1e9), (F32, 1e30), (F16, 2e4), (F16, -5e4),
                                          (BF16, 1e3), (BF16, -1e9), (BF16, 1e30)])
@pytest.mark.parametrize("rows", [2, 700])
def test_logprobs_of_logits_with_a_common_offset(ctx, bh, ws, type_, offset, rows):
    x = randn(gen(9), rows, 8192, scale=3.0)
    logprobs_held_to_64_bits(ctx, bh, ws, (x + offset).to(dt(type_)), 8, 1.0)
    x[:] = offset  # all equal
    logprobs_held_to_64_bits(ctx, bh, ws, x.to(dt(type_)), 8, 1.0)


def masked_rows(type_, rows, vocab, fill, every):
    """Rows at odd alignments, their values but every `every`-th replaced."""
    import torch

    x = randn(gen(vocab + every), rows, vocab + 1, dtype=type_, scale=3.0)[:, 1:]
    x[:, torch.arange(vocab, device="cuda") % every != every // 2] = fill
    return x


@pytest.mark.parametrize("type_", [BF16, F16, F32])
@pytest.mark.parametrize("fill", ["-inf", "lowest"])
@pytest.mark.parametrize("scale", [11.0, 25.0, 100.0, 1e4, 1e6])
def test_logprobs_of_masked_rows_at_low_temperatures(ctx, bh, ws, type_, fill, scale):
    import torch

    low = -math.inf if fill == "-inf" else torch.finfo(dt(type_)).min
    for rows, every in ((3, 5), (3, 50257), (600, 7)):
        logprobs_held_to_64_bits(ctx, bh, ws, masked_rows(type_, rows, 50257, low, every), 4, scale)
    logprobs_held_to_64_bits(ctx, bh, ws, randn(gen(3), 5, 50258, dtype=type_, scale=3.0)[:, 1:], 4, scale)  # nothing masked


@pytest.mark.parametrize("type_", [F16, BF16, F32])
@pytest.mark.parametrize("scale", [1e-2, 1e-3, 1e-4, 1e-6, 1e-30])
def test_logprobs_of_masked_rows_at_high_temperatures(ctx, bh, ws, type_, scale):
    """What is -inf has no probability, however flat the others' distribution is."""
    for rows, every in ((3, 5), (600, 7)):
        logprobs_held_to_64_bits(ctx, bh, ws, masked_rows(type_, rows, 20011, -math.inf, every), 4, scale)


@pytest.mark.parametrize("type_", [F32, F16, BF16])
def test_logprobs_of_the_largest_scales(ctx, bh, ws, type_):
    """Scales whose product with log2(e) passes fp32: the likeliest tokens share the row."""
    import torch

    x = randn(gen(4), 2, 5000, dtype=type_)
    x[:, 77] = x[:, 4001] = 9.0
    x[1, 300] = -math.inf
    r = bh.token_logprobs(ctx, ws, x, torch.tensor([[77, 5], [4001, 300]], dtype=torch.int32, device="cuda"), 2, 3e38)
    near = 16 * 2.0**-24
    assert (r.logprob[:, 0] + math.log(2)).abs().max() <= near and (r.logprob[:, 1] == -math.inf).all()
    assert (r.entropy - math.log(2)).abs().max() <= near
    assert r.top_ids.tolist() == [[77, 4001]] * 2 and (r.top_logprob + math.log(2)).abs().max() <= near
    assert ctx.status() == 0


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("act,cache_t", TYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("n_new,dim", [(33, 128), (64, 128), (64, 64), (40, 256)])
def test_attention_of_many_drafts_that_are_not_finite(ctx, bh, ws, act, cache_t, bad, n_new, dim):
    """Two drafts of three with one bad value of V each, over several tiles: a row
    has it where it sees the draft, and all else as if that value were zero."""
    import torch

    b = Batch(bh, 21, [70, 3], [n_new, 9], 8, 2, dim, act, cache_t, 16)
    lame = [(s, j, (5 * j) % 8) for s in range(2) for j in range(b.new[s]) if j % 3 != 1]
    at = [(*b.slots(s)[b.ctx[s] + j], c) for s, j, c in lame]

    def put(x):
        for blk, o, c in at:
            b.cache.v[blk, o, :, c] = x

    put(0.0)
    clean, lse0 = b.run(ctx, bh, ws, mask=b.mask(), return_lse=True)
    b.check(clean, lse0, True)
    for _ in range(3):
        put(bad)
        out, lse = b.run(ctx, bh, ws, mask=b.mask(), return_lse=True)
        put(0.0)
        hit = torch.zeros_like(out, dtype=torch.bool)
        for s, j, c in lame:
            for i in range(b.new[s]):
                if b.mask_h[b.start[s] + i] >> j & 1:
                    hit[b.start[s] + i, :, c] = True
        assert not out[hit].isfinite().any()
        b.check(torch.where(hit, clean, out), lse, True)
    assert ctx.status() == 0


@pytest.mark.parametrize("act,cache_t", [(F16, F16), (F32, F16), (BF16, BF16)])
@pytest.mark.parametrize("n_new,dim", [(1, 128), (4, 64), (8, 128), (64, 128), (64, 64), (2, 256)])
def test_attention_keeps_the_mass_of_small_probabilities(ctx, bh, ws, act, cache_t, n_new, dim):
    """One position has nearly all of the probability, 16000 others 2^-26 to
    2^-27.5 of it each, and values 2^10 times as large."""
    import torch

    n = 16000
    b = Batch(bh, 12, [n], [n_new], 4, 1, dim, act, cache_t, 16)
    g = gen(13)
    k, v = b.cache.k, b.cache.v
    k.zero_()
    # the score is k[0] + k[1]: the second part finer than the first one's rounding
    k[..., 0] = -math.log(2) * (26.1 + 1.3 * torch.rand(k.shape[:3], generator=g, device="cuda"))
    k[..., 1] = torch.rand(k.shape[:3], generator=g, device="cuda") * 0.03
    v[:] = (512 + 512 * torch.rand(v.shape, generator=g, device="cuda")).to(v.dtype)
    blk, o = b.slots(0)[5]
    k[blk, o], v[blk, o] = 0, 0
    b.q = torch.zeros_like(b.q)
    b.q[..., :2] = 1
    out = b.run(ctx, bh, ws, mask=b.mask(), scale=1.0)
    at = b.slots(0)
    i, j = torch.tensor([x for x, _ in at], device="cuda"), torch.tensor([y for _, y in at], device="cuda")
    keys, vals = k[i, j, 0].double(), v[i, j, 0].double()
    e = torch.exp(keys[:, 0] + keys[:, 1])
    for t in range(n_new):
        see = torch.ones(n + n_new, dtype=torch.bool, device="cuda")
        see[n:] = torch.tensor([bool(b.mask_h[t] >> x & 1) for x in range(n_new)], device="cuda")
        p = e * see
        want = (p @ vals) / p.sum()
        # the exponents' and sums' roundings; p's to 16 bits: a relative one, and where they are
        # subnormal (parts of f16, the largest 2^7, of fp32 rows 2^12 at least) half of 2^-24 each, signs at random
        near = want * (2 * 64 * U + 4 * math.sqrt(n) * U + u_of(act) * 2)
        if cache_t == F16:
            near = near + 4 * math.sqrt(n) * 2.0**-25 * 2.0 ** (-12 if act == F32 else -7) * 1024
        assert ((out[t].double() - want).abs() <= near).all(), (t, float(((out[t].double() - want).abs() / near).max()))
    assert ctx.status() == 0


# ---------------------------------------------------------------------------
# streams
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("as_handle", [False, True])
def test_outputs_on_another_stream_are_not_memory_that_the_current_one_still_writes(ctx, bh, ws, as_handle):
    import torch

    b = Batch(bh, 30, [40, 90], [2, 3], 4, 2, 64, BF16, BF16, 16)
    logits, tokens = randn(gen(31), 6, 5000), i32([1, 2, 3, 4, 5, 6])
    tables, free, lens, new = i32([[0, 1, -1], [2, 3, -1]]), i32([7, 8, 9]), i32([20, 31]), i32([2, 3])
    qkv, rope, pos, slot = randn(gen(32), 5, 8 * 64, dtype=BF16), bh.rope_table(99, 64), i32([1, 2, 3, 4, 5]), i64([1, 2, 3, 4, 5])
    calls = [lambda **kw: bh.kv_plan(ctx, lens, new, free, tables, 16, 5, **kw),
             lambda **kw: (bh.qk_norm_rope_append(ctx, qkv, 4, b.cache, rope, pos, slot, **kw),),
             lambda **kw: b.run(ctx, bh, ws, return_lse=True, **kw),
             lambda **kw: bh.token_logprobs(ctx, ws, logits, tokens, 3, **kw)]
    side = torch.cuda.Stream()
    for call in calls:
        want = [t.clone() for t in call()]
        torch.cuda.synchronize()
        old = [torch.empty_like(t) for t in want]
        torch.cuda._sleep(20_000_000)  # about 10 ms, before the current stream writes the blocks that it frees
        for t in old:
            t.fill_(7)
        del old, t
        got = call(stream=side.cuda_stream if as_handle else side)
        side.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))
    assert ctx.status() == 0


# ---------------------------------------------------------------------------
# many query rows: cache layouts, head sizes, long caches, many sequences
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("act", [F16, BF16])
@pytest.mark.parametrize("new_lens", [[9, 30, 1], [64, 20, 40]])  # up to 128 rows of a head, and more
@pytest.mark.parametrize("layout", ["token", "head", "padded"])
@pytest.mark.parametrize("dim,block", [(128, 8), (128, 16), (64, 64), (64, 24), (72, 16), (80, 32), (96, 128), (104, 256), (120, 512), (8, 16),
                                       (40, 8), (56, 48)])
def test_attention_of_many_rows_over_cache_layouts(ctx, bh, ws, act, new_lens, layout, dim, block):
    """Boxes of every size by tensor copies, heads that they reach beyond, and
    values behind the heads that are not numbers."""
    import torch

    b = Batch(bh, dim + block, [700, 129, 1500], new_lens, 8, 2, dim, act, act, block, layout)
    if layout == "padded":
        for t in (b.cache.k, b.cache.v):
            flat = torch.as_strided(t, (t.shape[0] * block * 3 * (dim + 16) - t.storage_offset(),), (1,), t.storage_offset())
            keep = t.clone()
            flat.fill_(math.nan)
            t.copy_(keep)
    out, lse = b.run(ctx, bh, ws, mask=b.mask(), return_lse=True)
    b.check(out, lse, True)
    assert ctx.status() == 0


@pytest.mark.parametrize("n_new", [8, 40])  # 32 and 160 rows of a head
def test_attention_of_many_rows_beyond_32_bit_offsets(ctx, bh, ws, n_new):
    import torch

    block, heads, dim = 64, 8, 128
    n_blocks = (1 << 31) // (block * heads * dim) + 40
    k, v = (torch.empty((n_blocks, block, heads, dim), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    small = Batch(bh, 40, [100, 700], [n_new, 3], 32, heads, dim, BF16, BF16, block)
    used = small.cache.k.shape[0]
    k[-used:], v[-used:] = small.cache.k, small.cache.v
    want = small.run(ctx, bh, ws, mask=small.mask())
    small.check(want, None, True)
    small.cache, small.tables = bh.PagedKV(k, v), torch.where(small.tables >= 0, small.tables + (n_blocks - used), -1)
    assert torch.equal(small.run(ctx, bh, ws, mask=small.mask()), want)
    assert ctx.status() == 0


@pytest.mark.parametrize("act,cache_t", TYPES)
@pytest.mark.parametrize("n_seq", [353, 900])  # more than any kernel has threads
@pytest.mark.parametrize("group", [1, 16])
def test_attention_of_many_sequences(ctx, bh, ws, act, cache_t, n_seq, group):
    new = [(7 * i) % 4 for i in range(n_seq)]
    new[3], new[-1] = 9, 5
    b = Batch(bh, n_seq, [(i * 37) % 150 if i % 11 else 600 for i in range(n_seq)], new, group, 1, 64, act, cache_t, 16)
    out, lse = b.run(ctx, bh, ws, mask=b.mask(), return_lse=True)
    b.check(out, lse, True)
    assert ctx.status() == 0


@pytest.mark.parametrize("act,cache_t", TYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("new_lens", [[1, 2], [30, 9], [64, 3]])
def test_attention_of_history_that_is_not_finite(ctx, bh, ws, act, cache_t, bad, new_lens):
    """A value of V shows in that value of the output and in no other, a key in
    its sequence's rows of its KV head and in no others."""
    import torch

    b = Batch(bh, 50, [400, 90], new_lens, 8, 2, 128, act, cache_t, 16)
    at = [b.slots(0)[17], b.slots(0)[333]]
    for (blk, o), c in zip(at, (5, 100)):
        b.cache.v[blk, o, 1, c] = 0
    clean, lse0 = b.run(ctx, bh, ws, mask=b.mask(), return_lse=True)
    b.check(clean, lse0, True)
    for (blk, o), c in zip(at, (5, 100)):
        b.cache.v[blk, o, 1, c] = bad
    out, lse = b.run(ctx, bh, ws, mask=b.mask(), return_lse=True)
    n = new_lens[0]
    assert not out[:n, 4:, [5, 100]].isfinite().any()
    out[:n, 4:, [5, 100]] = clean[:n, 4:, [5, 100]]
    assert torch.equal(out, clean) and torch.equal(lse, lse0)
    for (blk, o), c in zip(at, (5, 100)):
        b.cache.v[blk, o, 1, c] = 0
    b.cache.k[at[0][0], at[0][1], 1, 64] = bad
    out, lse = b.run(ctx, bh, ws, mask=b.mask(), return_lse=True)
    out[:n, 4:], lse[:n, 4:] = clean[:n, 4:], lse0[:n, 4:]
    assert torch.equal(out, clean) and torch.equal(lse, lse0)
    assert ctx.status() == 0
