"""The ops of a ragged batch (paged append, paged and packed attention, batched
sampling) against their formulas in 64 bits, at the sizes and masks where they
can go wrong, and together as a serving step runs them.

Tolerances. Attention rounds its weights to FP16 before the value product and
sums the rounded ones: each weight is off by at most 2^-11 of itself (half a
step), which moves a weighted mean by at most 2^-11 (max|v| + |o|) <= 2^-10
max|v|. A score of FP32 products and sums is off by at most (d + 2) 2^-24 B, B
the largest sum of |q||k|/sqrt(d) of a row, which moves a weight by that factor
and a mean by twice it times max|v|; exponentials and the joins of partial sums
add less than 2^-16 max|v|. The output is rounded once: 2^-11 |o|. The append
is held to the engine's own ops bit for bit, and to its formula within two
roundings of FP16 sums. Tokens are equal.
"""
import ctypes

import numpy as np
import pytest

import metal_infer as mi

pytestmark = pytest.mark.gpu

F16, F32, U32 = mi.DType.F16, mi.DType.F32, mi.DType.U32


def up(ctx, array, shape=None):
    a = np.ascontiguousarray(array)
    shape = list(shape or a.shape)
    if a.size == 0:
        kind = {np.dtype(np.float16): F16, np.dtype(np.float32): F32}.get(a.dtype, U32)
        return ctx.empty(shape, kind)
    if a.dtype == np.float16:
        return ctx.tensor_f16_bits(a.view(np.uint16), shape)
    if a.dtype == np.float32:
        t = ctx.empty(shape, F32)
        t.write(a)
        return t
    return ctx.tensor_u32(a.astype(np.uint32), shape)


def down(t):
    if t.dtype() == F16:
        return t.f16_bits().view(np.float16)
    return t.numpy()


def normal(rng, *shape):
    return rng.standard_normal(shape).astype(np.float16)


def paged(rng, lengths, page, spare=3, width=None):
    """A table of shuffled pages for `lengths`, unused places naming a page
    that does not exist; returns it with the number of pages."""
    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + spare
    order = rng.permutation(pages)
    table = np.full((len(lengths), width or max(1, max(counts, default=1))), 0xFFFFFFF0, np.uint32)
    at = 0
    for s, c in enumerate(counts):
        table[s, :c] = order[at:at + c]
        at += c
    return table, pages


def rows_of(table, s, n, page):
    p = np.arange(n)
    return table[s, p // page].astype(np.int64) * page + p % page


def attention64(q, k, v, visible):
    """One head: q [t, d], k / v [u, d]; row i sees keys [0, visible[i])."""
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    d = q.shape[1]
    out = np.zeros((q.shape[0], d))
    tol = np.zeros((q.shape[0], d))
    for i, n in enumerate(visible):
        if n <= 0:
            continue
        s = k[:n] @ q[i] / np.sqrt(d)
        w = np.exp(s - s.max())
        out[i] = (w / w.sum()) @ v[:n]
        big = np.abs(v[:n]).max()
        b = (np.abs(k[:n]) @ np.abs(q[i])).max() / np.sqrt(d)
        tol[i] = big * (2.0 ** -10 + 2.0 ** -16 + 2 * (d + 2) * 2.0 ** -24 * b) + 2.0 ** -11 * np.abs(out[i])
        tol[i] += 2.0 ** -25  # half a step of a subnormal
    return out, tol


def check(got, want, tol, what=""):
    got = got.astype(np.float64)
    assert got.shape == want.shape
    assert np.all(np.isfinite(got)), what
    over = np.abs(got - want) - tol
    assert over.max(initial=-1) <= 0, (what, float(np.abs(got - want).max()), float(over.max()))


def one(ctx, call):
    b = ctx.begin_batch()
    call(b)
    b.finish()


# ---- paged attention ----------------------------------------------------------------


def run_paged(ctx, q, kc, vc, lengths, table):
    out = up(ctx, np.full(q.shape, 7, np.float16))
    tensors = [up(ctx, x) for x in (q, kc, vc, np.asarray(lengths, np.uint32), table)]
    one(ctx, lambda b: b.paged_attention(*tensors, out))
    return down(out)


def check_paged(q, kc, vc, lengths, table, page, got):
    qh, kvh = q.shape[1], kc.shape[2]
    flat_k, flat_v = kc.reshape(-1, kvh, kc.shape[3]), vc.reshape(-1, kvh, kc.shape[3])
    for s, n in enumerate(lengths):
        r = rows_of(table, s, n, page)
        for h in range(qh):
            g = h // (qh // kvh)
            want, tol = attention64(q[s, h:h + 1], flat_k[r, g], flat_v[r, g], [n])
            check(got[s, h:h + 1], want, tol, (s, n, h))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("qh,kvh,page,lengths", [
    (2, 2, 16, [1]),
    (16, 8, 16, [0, 1, 15, 16, 17, 63, 64, 65, 0, 200]),
    (8, 1, 1, [5, 130, 64]),
    (32, 8, 64, [1000, 3, 257]),
    (7, 1, 24, [100, 24, 23, 25]),
    (20, 1, 7, [70, 129]),
    (34, 2, 48, [97, 1]),
    (4, 4, 300, [299, 301, 1]),
    (12, 2, 32, [40] * 150),
])
def test_paged_attention_matches_its_formula(ctx, hd, qh, kvh, page, lengths):
    rng = np.random.default_rng(hd + qh + page)
    table, pages = paged(rng, lengths, page)
    q, kc, vc = normal(rng, len(lengths), qh, hd), normal(rng, pages, page, kvh, hd), normal(rng, pages, page, kvh, hd)
    check_paged(q, kc, vc, lengths, table, page, run_paged(ctx, q, kc, vc, lengths, table))


def test_paged_attention_long_split_and_joined(ctx):
    rng = np.random.default_rng(5)
    lengths, page = [40001, 3, 9000], 16
    table, pages = paged(rng, lengths, page)
    q, kc, vc = normal(rng, 3, 4, 128), normal(rng, pages, page, 1, 128), normal(rng, pages, page, 1, 128)
    got = run_paged(ctx, q, kc, vc, lengths, table)
    check_paged(q, kc, vc, lengths, table, page, got)
    # the split does not depend on timing
    for _ in range(3):
        np.testing.assert_array_equal(got.view(np.uint16), run_paged(ctx, q, kc, vc, lengths, table).view(np.uint16))


def test_paged_attention_large_scores_and_equal_values(ctx):
    rng = np.random.default_rng(6)
    lengths, page, hd = [333, 77], 16, 128
    table, pages = paged(rng, lengths, page)
    q, kc = normal(rng, 2, 4, hd) * np.float16(8), normal(rng, pages, page, 2, hd) * np.float16(8)
    vc = normal(rng, pages, page, 2, hd)
    check_paged(q, kc, vc, lengths, table, page, run_paged(ctx, q, kc, vc, lengths, table))
    # a constant value row comes back as itself whatever the weights are
    vc[:] = np.float16(1.5)
    assert np.all(run_paged(ctx, q, kc, vc, lengths, table) == np.float16(1.5))


@pytest.mark.parametrize("stale", [np.nan, np.inf, -np.inf])
def test_paged_attention_ignores_stale_rows(ctx, stale):
    # everything that no sequence holds is not a number: rows behind a length
    # inside its last page, unused pages, and pages of longer tables
    rng = np.random.default_rng(7)
    lengths, page, hd = [70, 1, 0, 31], 32, 128
    table, pages = paged(rng, lengths, page, width=6)
    q = normal(rng, 4, 8, hd)
    kc, vc = (np.full((pages, page, 2, hd), stale, np.float16) for _ in range(2))
    for s, n in enumerate(lengths):
        r = rows_of(table, s, n, page)
        for c in (kc, vc):
            c.reshape(-1, 2, hd)[r] = normal(rng, n, 2, hd)
    got = run_paged(ctx, q, kc, vc, lengths, table)
    check_paged(q, kc, vc, lengths, table, page, got)
    assert np.all(got[2] == 0)


def test_paged_attention_shared_pages_and_contiguous_cache(ctx):
    # two requests with a common prefix name the same pages; a contiguous
    # cache viewed as pages gives what the engine's flash decode gives
    rng = np.random.default_rng(8)
    page, hd, n = 16, 128, 160
    kc, vc, q = normal(rng, 10, page, 8, hd), normal(rng, 10, page, 8, hd), normal(rng, 2, 16, hd)
    table = np.stack([np.arange(10), np.arange(10)]).astype(np.uint32)
    got = run_paged(ctx, q, kc, vc, [n, 100], table)
    check_paged(q, kc, vc, [n, 100], table, page, got)
    flat = ctx.attention(up(ctx, q[:1]), up(ctx, kc.reshape(n, 8, hd)), up(ctx, vc.reshape(n, 8, hd)),
                         mi.AttentionConfig(16, 8, hd, 1, n - 1), mi.AttentionKind.FLASH_DECODE)
    assert np.abs(down(flat).astype(float) - got[:1]).max() <= 2.0 ** -9 * np.abs(vc).max()


def test_paged_attention_reports_bad_pages_and_lengths(ctx):
    rng = np.random.default_rng(9)
    page, hd = 16, 64
    kc, vc, q = normal(rng, 4, page, 1, hd), normal(rng, 4, page, 1, hd), normal(rng, 2, 2, hd)
    good = np.array([[0, 1], [2, 3]], np.uint32)
    bad = np.array([[0, 1], [2, 4]], np.uint32)
    with pytest.raises(mi.CoreError) as e:
        run_paged(ctx, q, kc, vc, [20, 20], bad)
    assert e.value.status == mi.ERR_INVALID_ARGUMENT and "page" in e.value.message
    with pytest.raises(mi.CoreError) as e:
        run_paged(ctx, q, kc, vc, [20, 33], good)
    assert e.value.status == mi.ERR_INVALID_ARGUMENT and "length" in e.value.message
    # the context stays usable, and a place the length does not reach may hold anything
    check_paged(q, kc, vc, [20, 16], bad, page, run_paged(ctx, q, kc, vc, [20, 16], bad))


# ---- packed attention -----------------------------------------------------------------


def run_packed(ctx, q, k, v, qs, ks, causal, fill=7):
    out = up(ctx, np.full(q.shape, fill, np.float16))
    tensors = [up(ctx, x) for x in (q, k, v, np.asarray(qs, np.uint32), np.asarray(ks, np.uint32))]
    one(ctx, lambda b: b.packed_attention(*tensors, causal, out))
    return down(out)


def check_packed(q, k, v, qs, ks, causal, got, heads=None):
    qh, kvh = q.shape[1], k.shape[1]
    for s in range(len(qs) - 1):
        n, m = qs[s + 1] - qs[s], ks[s + 1] - ks[s]
        visible = [m - (n - 1 - i) if causal else m for i in range(n)]
        for h in heads if heads is not None else range(qh):
            g = h // (qh // kvh)
            want, tol = attention64(q[qs[s]:qs[s + 1], h], k[ks[s]:ks[s + 1], g], v[ks[s]:ks[s + 1], g], visible)
            check(got[qs[s]:qs[s + 1], h], want, tol, (s, h))


def starts(lengths, first=0):
    return np.concatenate([[first], first + np.cumsum(lengths)]).astype(np.int64)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("qh,kvh,queries,keys", [
    (2, 2, [1], [1]),
    (16, 8, [5, 1, 0, 64, 17], [5, 1, 0, 64, 17]),
    (8, 1, [33, 127, 128, 129], [33, 127, 128, 129]),
    (7, 1, [19, 37], [219, 37]),
    (32, 8, [1, 1, 40], [300, 1, 290]),
    (6, 2, [50, 9, 3], [20, 0, 3]),       # fewer keys than queries: empty rows
    (20, 1, [30], [70]),
    (4, 4, [300], [300]),
])
def test_packed_attention_matches_its_formula(ctx, hd, causal, qh, kvh, queries, keys):
    rng = np.random.default_rng(hd + qh + len(queries))
    qs, ks = starts(queries), starts(keys)
    q, k, v = normal(rng, qs[-1], qh, hd), normal(rng, ks[-1], kvh, hd), normal(rng, ks[-1], kvh, hd)
    check_packed(q, k, v, qs, ks, causal, run_packed(ctx, q, k, v, qs, ks, causal))


@pytest.mark.parametrize("hd,qh,kvh,queries,prefix", [(128, 4, 1, [1500, 700], 0), (64, 5, 1, [300, 260], 1111),
                                                      (128, 2, 2, [1025], 0)])
def test_packed_attention_long(ctx, hd, qh, kvh, queries, prefix):
    rng = np.random.default_rng(11)
    qs, ks = starts(queries), starts([n + prefix for n in queries])
    q, k, v = normal(rng, qs[-1], qh, hd), normal(rng, ks[-1], kvh, hd), normal(rng, ks[-1], kvh, hd)
    got = run_packed(ctx, q, k, v, qs, ks, True)
    check_packed(q, k, v, qs, ks, True, got, heads=[0, qh - 1])
    np.testing.assert_array_equal(got.view(np.uint16), run_packed(ctx, q, k, v, qs, ks, True).view(np.uint16))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("hd,qh,kvh,queries,keys", [
    (128, 8, 2, [7], [5000]), (64, 8, 2, [7], [5000]), (128, 4, 1, [1, 3], [9000, 100]),
    (128, 6, 2, [40, 0, 5], [4100, 0, 2000]), (64, 7, 1, [90, 5], [40, 4500]), (128, 16, 8, [64], [2549])])
def test_packed_attention_few_queries_over_many_keys(ctx, hd, qh, kvh, queries, keys, causal):
    # work that is split along its keys and joined
    rng = np.random.default_rng(17)
    qs, ks = starts(queries), starts(keys)
    q, k, v = normal(rng, qs[-1], qh, hd), normal(rng, ks[-1], kvh, hd), normal(rng, ks[-1], kvh, hd)
    got = run_packed(ctx, q, k, v, qs, ks, causal)
    check_packed(q, k, v, qs, ks, causal, got)
    np.testing.assert_array_equal(got.view(np.uint16), run_packed(ctx, q, k, v, qs, ks, causal).view(np.uint16))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("hd,qh,kvh,queries,prefix", [
    (64, 32, 4, [700, 500], 3000), (128, 24, 8, [1100, 1000], 4200), (128, 32, 4, [1210], 2700)])
def test_packed_attention_waves_with_little_in_the_last(ctx, hd, qh, kvh, queries, prefix, causal):
    # whole waves of work, and the rest split along its keys
    rng = np.random.default_rng(20)
    qs, ks = starts(queries), starts([n + prefix for n in queries])
    q, k, v = normal(rng, qs[-1], qh, hd), normal(rng, ks[-1], kvh, hd), normal(rng, ks[-1], kvh, hd)
    got = run_packed(ctx, q, k, v, qs, ks, causal)
    check_packed(q, k, v, qs, ks, causal, got, heads=[0, qh - 1])
    np.testing.assert_array_equal(got.view(np.uint16), run_packed(ctx, q, k, v, qs, ks, causal).view(np.uint16))


@pytest.mark.parametrize("stale", [np.nan, np.inf])
def test_packed_attention_split_ignores_masked_values(ctx, stale):
    rng = np.random.default_rng(18)
    qs, ks = starts([20, 6]), starts([3000, 40])
    q, k, v = normal(rng, 26, 4, 128), normal(rng, 3300, 2, 128), normal(rng, 3300, 2, 128)
    k[3040:], v[3040:] = stale, stale
    v[2990:3000] = stale   # seen by the last ten queries of the first sequence alone
    got = run_packed(ctx, q, k, v, qs, ks, True)
    clean = np.where(np.isfinite(v), v, 0)
    check_packed(q[:10], k, clean, [0, 10], [0, 2990], True, got[:10])
    check_packed(q[20:], k[3000:3040], clean[3000:3040], [0, 6], [0, 40], True, got[20:])
    assert not np.any(np.isfinite(got[10:20]))


@pytest.mark.parametrize("hidden", [0.0, np.inf])
def test_packed_attention_split_with_scores_of_minus_infinity(ctx, hidden):
    # keys of weight 0 that the rows see: they leave the others' result alone
    # where their values are finite, and 0 * inf is NaN, in any part
    rng = np.random.default_rng(19)
    q, k, v = normal(rng, 9, 2, 128), normal(rng, 4000, 1, 128), normal(rng, 4000, 1, 128)
    q[:, :, 0] = 1
    k[:2000, :, 0] = -np.inf
    v[7] += hidden
    got = run_packed(ctx, q, k, v, [0, 9], [0, 4000], True)
    if hidden:
        assert np.all(np.isnan(got))
    else:
        check_packed(q, k[2000:], v[2000:], [0, 9], [0, 2000], True, got)


def test_packed_attention_large_scores(ctx):
    rng = np.random.default_rng(12)
    qs = ks = starts([150, 260])
    q, k, v = (normal(rng, 410, 4, 128) * np.float16(8), normal(rng, 410, 2, 128) * np.float16(8),
               normal(rng, 410, 2, 128))
    # a row whose largest score comes last, and one whose first does
    k[140] = q[145, 0] * np.float16(0.5)
    k[0] = q[149, 3] * np.float16(0.5)
    check_packed(q, k, v, qs, ks, True, run_packed(ctx, q, k, v, qs, ks, True))
    # equal values: a mean of equal values under weights each off by at most
    # 2^-11 is off by that much, then rounded: one FP16 step of 0.75 (2^-11)
    v[:] = np.float16(-0.75)
    got = run_packed(ctx, q, k, v, qs, ks, True).astype(np.float64)
    assert np.abs(got + 0.75).max() <= 0.75 * 2.0 ** -11 + 2.0 ** -12


def test_packed_attention_leaves_other_rows(ctx):
    # rows before the first start and behind the last stay as they were
    rng = np.random.default_rng(13)
    qs, ks = starts([30, 50], 7), starts([30, 90], 11)
    q, k, v = normal(rng, 140, 4, 128), normal(rng, 200, 2, 128), normal(rng, 200, 2, 128)
    got = run_packed(ctx, q, k, v, qs, ks, True)
    check_packed(q, k, v, qs, ks, True, got)
    assert np.all(got[:7] == 7) and np.all(got[87:] == 7)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("stale", [np.nan, np.inf, -np.inf])
def test_packed_attention_ignores_masked_values(ctx, stale, hd):
    # keys and values of other sequences, of padding and behind a causal row
    # may hold anything
    rng = np.random.default_rng(14)
    qs, ks = starts([40, 33, 150]), starts([40, 33, 150])
    q, k, v = normal(rng, 260, 4, hd), normal(rng, 260, 2, hd), normal(rng, 260, 2, hd)
    k[223:], v[223:], q[223:] = stale, stale, stale
    clean_k, clean_v = k.copy(), v.copy()
    k[50:73], v[50:73] = stale, stale    # from row 10 of the middle sequence
    v[200:223] = stale                   # from row 127 of the last one
    k[210:223] = stale
    got = run_packed(ctx, q, k, v, qs, ks, True)
    want = run_packed(ctx, q, clean_k, clean_v, qs, ks, True)
    keep = np.r_[0:50, 73:200]
    check_packed(q[:223], np.where(np.isfinite(k), k, 0)[:223], np.where(np.isfinite(v), v, 0)[:223],
                 [0, 40], [0, 40], True, got)
    assert np.all(np.isfinite(got[keep]))
    assert np.abs(got[keep].astype(float) - want[keep]).max() <= 2.0 ** -9 * np.abs(clean_v[:223]).max()
    assert not np.any(np.isfinite(got[50:73])) and not np.any(np.isfinite(got[210:223]))


def test_packed_attention_reports_bad_starts(ctx):
    rng = np.random.default_rng(15)
    q, k, v = normal(rng, 20, 2, 64), normal(rng, 20, 2, 64), normal(rng, 20, 2, 64)
    for qs, ks in (([0, 10, 21], [0, 10, 20]), ([0, 10, 20], [0, 10, 21]), ([0, 12, 9], [0, 10, 20]),
                   ([0, 10, 20], [12, 10, 20])):
        with pytest.raises(mi.CoreError) as e:
            run_packed(ctx, q, k, v, qs, ks, True)
        assert e.value.status == mi.ERR_INVALID_ARGUMENT and "starts" in e.value.message
    check_packed(q, k, v, [0, 10, 20], [0, 10, 20], True, run_packed(ctx, q, k, v, [0, 10, 20], [0, 10, 20], True))


@pytest.mark.parametrize("queries,keys", [([40] * 50, [40] * 50), ([9, 5], [5000, 20])])
def test_packed_attention_reports_bad_starts_in_every_order_of_work(ctx, queries, keys):
    # work in a planned order, and work that is split along its keys
    rng = np.random.default_rng(21)
    qs, ks = starts(queries), starts(keys)
    q, k, v = normal(rng, qs[-1], 16, 64), normal(rng, ks[-1], 8, 64), normal(rng, ks[-1], 8, 64)
    for bad_q, bad_k in ((qs + (np.arange(len(qs)) == len(qs) - 1), ks), (qs, ks[::-1].copy()),
                         (qs, np.where(np.arange(len(ks)) == 1, ks[-1] + 1, ks))):
        with pytest.raises(mi.CoreError) as e:
            run_packed(ctx, q, k, v, bad_q, bad_k, True)
        assert e.value.status == mi.ERR_INVALID_ARGUMENT and "starts" in e.value.message
    check_packed(q, k, v, qs, ks, True, run_packed(ctx, q, k, v, qs, ks, True), heads=[0, 15])


def test_packed_attention_agrees_with_the_prefill_op(ctx):
    rng = np.random.default_rng(16)
    q, k, v = normal(rng, 100, 16, 128), normal(rng, 100, 8, 128), normal(rng, 100, 8, 128)
    got = run_packed(ctx, q, k, v, [0, 100], [0, 100], True)
    flat = ctx.attention(up(ctx, q), up(ctx, k), up(ctx, v), mi.AttentionConfig(16, 8, 128, 1, 0),
                         mi.AttentionKind.FLASH_PREFILL)
    assert np.abs(down(flat).astype(float) - got).max() <= 2.0 ** -9 * np.abs(v).max()


# ---- paged append -----------------------------------------------------------------------


def run_append(ctx, q, k, v, qw, kw, st, lengths, table, kc, vc, theta=1e6, eps=1e-6, in_place=False):
    t = [None if x is None else up(ctx, x)
         for x in (q, k, v, qw, kw, np.asarray(st, np.uint32), np.asarray(lengths, np.uint32), table, kc, vc)]
    q_out = None if q is None else t[0] if in_place else up(ctx, np.full(q.shape, 7, np.float16))
    one(ctx, lambda b: b.paged_append(*t, q_out, theta, eps))
    return None if q is None else down(q_out), down(t[8]), down(t[9])


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("qh,kvh,page,new,old", [
    (2, 1, 16, [1], [0]),
    (16, 8, 16, [1, 1, 1], [15, 16, 400]),
    (7, 1, 24, [30, 1, 0, 50], [5, 0, 9, 47]),
    (32, 8, 64, [700, 3], [0, 100000]),
])
def test_paged_append_has_the_bits_of_the_contiguous_ops(ctx, hd, norm, qh, kvh, page, new, old):
    rng = np.random.default_rng(qh + hd)
    total, lengths = sum(new), [a + b for a, b in zip(new, old)]
    st = starts(new)
    q, k, v = normal(rng, total, qh, hd), normal(rng, total, kvh, hd), normal(rng, total, kvh, hd)
    qw, kw = (normal(rng, hd), normal(rng, hd)) if norm else (None, None)
    spans = [(o // page, -(-n // page)) for o, n in zip(old, lengths)]
    pages = sum(b - a for a, b in spans) + 2
    table = np.full((len(new), max(b for _, b in spans)), 0xFFFFFFF0, np.uint32)
    order, at = rng.permutation(pages), 0
    for s, (a, b) in enumerate(spans):
        table[s, a:b] = order[at:at + b - a]
        at += b - a
    kc, vc = normal(rng, pages, page, kvh, hd), normal(rng, pages, page, kvh, hd)
    got_q, got_k, got_v = run_append(ctx, q, k, v, qw, kw, st, lengths, table, kc, vc)
    want_k, want_v = kc.reshape(-1, kvh, hd).copy(), vc.reshape(-1, kvh, hd).copy()
    want_q = np.empty_like(q)
    for s, n in enumerate(new):
        if n == 0:
            continue
        a, b = st[s], st[s + 1]
        if norm:
            flat = ctx.empty([old[s] + n, kvh, hd], F16)
            box = {}
            one(ctx, lambda bt: box.update(q=bt.qk_norm_rope_cache(
                up(ctx, q[a:b]), up(ctx, k[a:b]), up(ctx, qw), up(ctx, kw), flat,
                mi.QkNormRopeCacheConfig(old[s], 1e6, 1e-6))))
            want_q[a:b] = down(box["q"])
            rotated = down(flat)[old[s]:]
        else:
            want_q[a:b] = down(ctx.rope(up(ctx, q[a:b]), old[s], 1e6))
            rotated = down(ctx.rope(up(ctx, k[a:b]), old[s], 1e6))
        p = old[s] + np.arange(n)
        r = table[s, p // page].astype(np.int64) * page + p % page
        want_k[r], want_v[r] = rotated, v[a:b]
    for got, want in ((got_q, want_q), (got_k, want_k), (got_v, want_v)):
        np.testing.assert_array_equal(got.view(np.uint16).ravel(), want.view(np.uint16).ravel())
    # in place, and without queries
    again = run_append(ctx, q, k, v, qw, kw, st, lengths, table, kc, vc, in_place=True)
    np.testing.assert_array_equal(again[0].view(np.uint16), want_q.view(np.uint16))
    alone = run_append(ctx, None, k, v, None, kw, st, lengths, table, kc, vc)
    np.testing.assert_array_equal(alone[1].view(np.uint16), got_k.view(np.uint16))


def test_paged_append_matches_its_formula(ctx):
    # y = half(rot(x * rsqrt(mean x^2 + eps) * w)): FP32 sums of 128 terms and
    # four products (2^-20 of the magnitude), one FP16 rounding
    rng = np.random.default_rng(21)
    hd, n, old = 128, 9, 131000
    k, v, kw = normal(rng, n, 2, hd), normal(rng, n, 2, hd), normal(rng, hd)
    page = 128
    table = np.zeros((1, (old + n + page - 1) // page), np.uint32)
    table[0, old // page:] = np.arange(table.shape[1] - old // page)
    kc = np.zeros((3, page, 2, hd), np.float16)
    _, got, _ = run_append(ctx, None, k, v, None, kw, [0, n], [old + n], table, kc, kc.copy())
    pos = old + np.arange(n)
    rows = got.reshape(-1, 2, hd)[table[0, pos // page].astype(int) * page + pos % page].astype(np.float64)
    x = k.astype(np.float64)
    x = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + 1e-6) * kw.astype(np.float64)
    freq = np.array([np.float32(1e6 ** float(np.float32(-i) / np.float32(hd))) for i in range(0, hd, 2)])
    angle = (pos.astype(np.float32)[:, None] * freq).astype(np.float64)[:, None]
    a, b = x[..., :64], x[..., 64:]
    want = np.concatenate([a * np.cos(angle) - b * np.sin(angle), a * np.sin(angle) + b * np.cos(angle)], -1)
    size = np.concatenate([np.abs(a) + np.abs(b)] * 2, -1)
    check(rows, want, 2.0 ** -11 * np.abs(want) + 2.0 ** -20 * size + 2.0 ** -25)


def test_paged_append_leaves_other_slots_and_padding(ctx):
    rng = np.random.default_rng(22)
    hd, page = 64, 16
    k, v, q = normal(rng, 9, 2, hd), normal(rng, 9, 2, hd), normal(rng, 9, 4, hd)
    kc, vc = normal(rng, 5, page, 2, hd), normal(rng, 5, page, 2, hd)
    table = np.array([[3, 1], [4, 0]], np.uint32)
    got_q, got_k, got_v = run_append(ctx, q, k, v, None, None, [2, 4, 7], [17, 3], table, kc, vc)
    written = {3 * 16 + 15, 1 * 16 + 0, 4 * 16 + 0, 4 * 16 + 1, 4 * 16 + 2}
    for r in range(5 * page):
        same = np.array_equal(got_v.reshape(-1, 2, hd)[r].view(np.uint16), vc.reshape(-1, 2, hd)[r].view(np.uint16))
        assert same == (r not in written)
        if r not in written:
            np.testing.assert_array_equal(got_k.reshape(-1, 2, hd)[r].view(np.uint16),
                                          kc.reshape(-1, 2, hd)[r].view(np.uint16))
    assert np.all(got_q[:2] == 7) and np.all(got_q[7:] == 7) and not np.any(got_q[2:7] == 7)


def test_paged_append_reports_bad_arguments(ctx):
    rng = np.random.default_rng(23)
    hd, page = 64, 16
    k, v = normal(rng, 6, 1, hd), normal(rng, 6, 1, hd)
    kc, vc = normal(rng, 3, page, 1, hd), normal(rng, 3, page, 1, hd)
    table = np.array([[0, 1], [2, 3]], np.uint32)
    for st, lengths, t, word in (([0, 3, 7], [3, 3], table, "starts"), ([0, 4, 3], [4, 3], table, "starts"),
                                 ([0, 3, 6], [2, 3], table, "length"), ([0, 3, 6], [3, 33], table, "length"),
                                 ([0, 3, 6], [3, 19], table, "page")):
        with pytest.raises(mi.CoreError) as e:
            run_append(ctx, None, k, v, None, None, st, lengths, t, kc, vc)
        assert e.value.status == mi.ERR_INVALID_ARGUMENT and word in e.value.message, (st, lengths)
    _, _, got = run_append(ctx, None, k, v, None, None, [0, 3, 6], [3, 3], table, kc, vc)
    np.testing.assert_array_equal(got[0, :3], v[:3])


# ---- sampling -------------------------------------------------------------------------------


def sample64(bits, temperature, top_k, top_p, min_p, uniform):
    """The definition, one row: FP16 bits, extended precision."""
    bits = bits.astype(np.int64)
    index = np.nonzero((bits & 0x7C00) != 0x7C00)[0]
    if index.size == 0:
        return 0xFFFFFFFF
    b = bits[index]
    key = np.where(b & 0x8000, 0xFFFF - b, b | 0x8000)
    order = index[np.lexsort((index, -key))]
    if temperature == 0:
        return int(order[0])
    if top_k:
        order = order[:top_k]
    v = bits[order].astype(np.uint16).view(np.float16).astype(np.longdouble)
    w = np.exp((v - v[0]) / np.longdouble(np.float32(temperature)))
    before = np.cumsum(w) - w
    keep = (before < np.longdouble(np.float32(top_p)) * w.sum()) | (np.float32(top_p) >= 1)
    keep &= w >= np.longdouble(np.float32(min_p))
    keep[0] = True
    w = w[keep]
    ends = np.cumsum(w)
    at = np.searchsorted(ends, np.longdouble(np.float32(uniform)) * ends[-1], "right")
    return int(order[keep][min(at, w.size - 1)])


def run_sample(ctx, bits, options):
    rows = bits.shape[0]
    t, k, p, m, u = (np.array([o[i] for o in options]) for i in range(5))
    out = up(ctx, np.zeros(rows, np.uint32))
    tensors = [ctx.tensor_f16_bits(bits.ravel(), list(bits.shape)), up(ctx, t.astype(np.float32)),
               up(ctx, k.astype(np.uint32)), up(ctx, p.astype(np.float32)), up(ctx, m.astype(np.float32)),
               up(ctx, u.astype(np.float32))]
    one(ctx, lambda b: b.sample(*tensors, out))
    return out.to_u32_vec()


OPTIONS = [(1.0, 0, 1.0, 0.0), (0.7, 20, 0.95, 0.0), (0.0, 0, 1.0, 0.0), (1.3, 0, 0.8, 0.05), (0.6, 1, 1.0, 0.0),
           (1.0, 5, 0.0, 0.0), (2.0, 0, 1.0, 1.0), (0.05, 3, 0.5, 0.2), (30.0, 0, 0.999, 0.0), (1e-30, 0, 1.0, 0.0),
           (1.0, 4000000000, 1.0, 0.0), (1e30, 0, 0.3, 0.0)]
UNIFORMS = [0.0, 0.25, 0.5, 0.730001, float(np.float32(1) - np.float32(2) ** -24)]


def logits_of(kind, rng, n):
    if kind == "normal":
        x = (rng.standard_normal(n) * 2.5).astype(np.float16)
    elif kind == "equal":
        x = np.full(n, 1.25, np.float16)
    elif kind == "two values":
        x = rng.choice(np.array([0.5, -3.0], np.float16), n)
    elif kind == "zeros of both signs":
        x = rng.choice(np.array([0.0, -0.0], np.float16), n)
    elif kind == "lowest":
        x = np.full(n, -65504, np.float16)
        x[n // 2] = 3
    elif kind == "masked":
        x = (rng.standard_normal(n) * 2).astype(np.float16)
        x[rng.random(n) < 0.7] = -np.inf
        x[rng.random(n) < 0.05] = np.nan
        x[rng.random(n) < 0.05] = np.inf
    elif kind == "all bits":
        x = rng.integers(0, 65536, n).astype(np.uint16).view(np.float16)
    else:
        x = np.full(n, -np.inf, np.float16)
        x[::2] = np.nan
    return x.view(np.uint16)


@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 63, 1001, 32000])
@pytest.mark.parametrize("kind", ["normal", "equal", "two values", "zeros of both signs", "lowest", "masked",
                                  "all bits", "none finite"])
def test_sample_matches_its_definition(ctx, kind, n):
    rng = np.random.default_rng(n)
    options = [o + (u,) for o in OPTIONS for u in UNIFORMS]
    bits = np.stack([logits_of(kind, rng, n) for _ in options])
    want = np.array([sample64(b, *o) for b, o in zip(bits, options)], np.uint32)
    # as many rows as share the GPU among one, two, four or eight CTAs to a row
    for rows in (60, 20, 7, 120):
        pick = (np.arange(rows) * 7) % 60
        got = run_sample(ctx, bits[pick], [options[i] for i in pick])
        np.testing.assert_array_equal(got, want[pick])


@pytest.mark.parametrize("n,kind", [(151936, "normal"), (151937, "equal"), (262144, "two values"), (524224, "normal"),
                                    (524224, "equal")])
def test_sample_large_vocabularies(ctx, n, kind):
    rng = np.random.default_rng(3)
    options = [OPTIONS[0] + (0.37,), OPTIONS[1] + (0.9,), OPTIONS[3] + (0.999,), OPTIONS[2] + (0.1,),
               OPTIONS[8] + (UNIFORMS[-1],)]
    bits = np.stack([logits_of(kind, rng, n) for _ in options])
    np.testing.assert_array_equal(run_sample(ctx, bits, options),
                                  np.array([sample64(b, *o) for b, o in zip(bits, options)], np.uint32))


def test_sample_follows_its_distribution(ctx):
    # 8 candidates with known probabilities, uniforms on an even grid: the
    # counts are the probabilities to within one
    x = np.log(np.array([1, 2, 3, 4, 5, 6, 7, 8], np.float64)).astype(np.float16)
    rows = 4096
    got = run_sample(ctx, np.tile(x.view(np.uint16), (rows, 1)),
                     [(1.0, 0, 1.0, 0.0, (i + 0.5) / rows) for i in range(rows)])
    p = np.exp(x.astype(np.float64))
    assert np.abs(np.bincount(got, minlength=8) - rows * p / p.sum()).max() <= 1


@pytest.mark.parametrize("bad", [(-0.1, 0, 1.0, 0.0, 0.5), (float("nan"), 0, 1.0, 0.0, 0.5),
                                 (float("inf"), 0, 1.0, 0.0, 0.5), (1.0, 0, 1.1, 0.0, 0.5), (1.0, 0, -0.1, 0.0, 0.5),
                                 (1.0, 0, 1.0, float("nan"), 0.5), (1.0, 0, 1.0, 0.0, 1.0), (1.0, 0, 1.0, 0.0, -0.1)])
def test_sample_reports_bad_options(ctx, bad):
    rng = np.random.default_rng(4)
    bits = np.stack([logits_of("normal", rng, 100) for _ in range(2)])
    good = (1.0, 0, 1.0, 0.0, 0.5)
    with pytest.raises(mi.ModelError) as e:
        run_sample(ctx, bits, [good, bad])
    assert e.value.status == mi.ERR_CONFIG
    np.testing.assert_array_equal(run_sample(ctx, bits, [good, good]), [sample64(b, *good) for b in bits])


# ---- together, and how they may be called ------------------------------------------------------


class Serving:
    """One layer's step over a batch: prompts, then single tokens, through the
    ops; and the same on contiguous tensors in 64 bits."""

    def __init__(self, ctx, rng, prompts, qh=8, kvh=2, hd=64, page=16, vocab=500):
        self.ctx, self.rng, self.qh, self.kvh, self.hd, self.page = ctx, rng, qh, kvh, hd, page
        self.lengths = np.zeros(len(prompts), np.int64)
        self.prompts = prompts
        width = 8
        self.table = rng.permutation(len(prompts) * width).reshape(len(prompts), width).astype(np.uint32)
        shape = [len(prompts) * width, page, kvh, hd]
        self.kc, self.vc = up(ctx, np.full(shape, np.nan, np.float16)), up(ctx, np.full(shape, np.nan, np.float16))
        self.head = normal(rng, vocab, qh * hd)
        self.keys = [np.zeros((0, kvh, hd), np.float16) for _ in prompts]
        self.values = [np.zeros((0, kvh, hd), np.float16) for _ in prompts]

    def step(self, counts):
        ctx, hd = self.ctx, self.hd
        total, st = sum(counts), starts(counts)
        q, k, v = (normal(self.rng, total, h, hd) for h in (self.qh, self.kvh, self.kvh))
        first, self.lengths = self.lengths, self.lengths + counts
        tq, tk, tv, ts, tl, tt = (up(ctx, x) for x in (q, k, v, st.astype(np.uint32), self.lengths, self.table))
        out, rotated = up(ctx, np.zeros_like(q)), up(ctx, np.zeros_like(q))
        single = all(c == 1 for c in counts)
        b = ctx.begin_batch()
        b.paged_append(tq, tk, tv, None, None, ts, tl, tt, self.kc, self.vc, rotated, 1e4)
        if single:
            b.paged_attention(rotated, self.kc, self.vc, tl, tt, out)
        else:  # a first chunk: its keys are the prompt's
            kr = b.rope(tk, 0, 1e4) if len(counts) == 1 else up(ctx, np.concatenate(
                [down(ctx.rope(up(ctx, k[st[i]:st[i + 1]]), int(first[i]), 1e4)) for i in range(len(counts))]))
            b.packed_attention(rotated, kr, tv, ts, ts, True, out)
        last = [int(e) - 1 for e in st[1:]]
        b.finish()
        got, rq = down(out), down(rotated)
        for i in range(len(counts)):
            a, e = st[i], st[i + 1]
            kr = down(ctx.rope(up(ctx, k[a:e]), int(first[i]), 1e4))
            self.keys[i] = np.concatenate([self.keys[i], kr])
            self.values[i] = np.concatenate([self.values[i], v[a:e]])
            n = len(self.keys[i])
            for h in range(self.qh):
                g = h // (self.qh // self.kvh)
                want, tol = attention64(rq[a:e, h], self.keys[i][:, g], self.values[i][:, g],
                                        [n - (e - a) + j + 1 for j in range(e - a)])
                check(got[a:e, h], want, tol, (i, h))
        hidden = up(ctx, got[last].reshape(len(counts), -1))
        b = ctx.begin_batch()
        logits = b.matmul(hidden, up(ctx, self.head))
        b.finish()
        options = [(0.1 + i, 10, 0.9, 0.0, 0.3) for i in range(len(counts))]
        tokens = run_sample(ctx, logits.f16_bits(), options)
        np.testing.assert_array_equal(tokens, [sample64(x, *o) for x, o in zip(logits.f16_bits(), options)])


def test_a_serving_loop(ctx):
    s = Serving(ctx, np.random.default_rng(31), [20, 1, 47])
    s.step([20, 1, 47])
    for _ in range(3):
        s.step([1, 1, 1])


def test_zero_sequences_and_zero_tokens(ctx):
    e = lambda *shape: ctx.empty(list(shape), F16)  # noqa: E731
    u = lambda *shape: ctx.empty(list(shape), U32)  # noqa: E731
    f = lambda *shape: ctx.empty(list(shape), F32)  # noqa: E731
    b = ctx.begin_batch()
    b.paged_attention(e(0, 4, 64), e(3, 16, 2, 64), e(3, 16, 2, 64), u(0), u(0, 2), e(0, 4, 64))
    b.paged_append(e(0, 4, 64), e(0, 2, 64), e(0, 2, 64), None, None, u(2), u(1), u(1, 2), e(3, 16, 2, 64),
                   e(3, 16, 2, 64), e(0, 4, 64), 1e4)
    b.packed_attention(e(0, 4, 64), e(0, 2, 64), e(0, 2, 64), u(1), u(1), True, e(0, 4, 64))
    b.sample(e(0, 100), f(0), u(0), f(0), f(0), f(0), u(0))
    # queries without any key, and sequences without a page
    out = up(ctx, np.full((3, 4, 64), 7, np.float16))
    b.packed_attention(e(3, 4, 64), e(0, 2, 64), e(0, 2, 64), ctx.tensor_u32([0, 3], [2]), u(2), True, out)
    out2 = up(ctx, np.full((2, 4, 64), 7, np.float16))
    b.paged_attention(e(2, 4, 64), e(0, 16, 2, 64), e(0, 16, 2, 64), u(2), u(2, 0), out2)
    b.finish()
    assert np.all(down(out) == 0) and np.all(down(out2) == 0)


def test_profiling_names_the_ops(ctx):
    rng = np.random.default_rng(33)
    ctx.set_kernel_profiling(True)
    try:
        run_paged(ctx, normal(rng, 1, 2, 64), normal(rng, 1, 16, 1, 64), normal(rng, 1, 16, 1, 64), [3],
                  np.zeros((1, 1), np.uint32))
        names = [n for n, _ in ctx.take_kernel_profiles()]
    finally:
        ctx.set_kernel_profiling(False)
    assert "paged_attention" in names


class Graph:
    """Capture of a context's stream, and replays."""

    def __init__(self):
        self.rt = ctypes.CDLL("libcudart.so.12")
        self.exec = ctypes.c_void_p()

    def call(self, name, *args):
        status = getattr(self.rt, name)(*args)
        assert status == 0, (name, status)

    def capture(self, ctx, call):
        stream, graph = ctypes.c_void_p(ctx.stream()), ctypes.c_void_p()
        b = ctx.begin_batch()
        self.call("cudaStreamBeginCapture", stream, ctypes.c_int(2))  # relaxed
        try:
            call(b)
        finally:
            status = self.rt.cudaStreamEndCapture(stream, ctypes.byref(graph))
        assert status == 0
        b.finish()
        self.call("cudaGraphInstantiate", ctypes.byref(self.exec), graph, ctypes.c_ulonglong(0))
        self.call("cudaGraphDestroy", graph)
        return self

    def replay(self, stream):
        self.call("cudaGraphLaunch", self.exec, ctypes.c_void_p(stream))

    def close(self):
        self.call("cudaGraphExecDestroy", self.exec)


def test_captured_steps_replay_with_new_lengths_and_beside_each_other(ctx):
    rng = np.random.default_rng(34)
    other = mi.MetalContext(0)
    page, hd, width = 16, 128, 300
    cases = []
    for seed, lengths in ((1, [4000, 50]), (2, [37, 4500])):
        r = np.random.default_rng(seed)
        table = r.permutation(2 * width).reshape(2, width).astype(np.uint32)
        q, kc, vc = normal(r, 2, 8, hd), normal(r, 2 * width, page, 2, hd), normal(r, 2 * width, page, 2, hd)
        out = up(ctx, np.zeros_like(q))
        tensors = [up(ctx, x) for x in (q, kc, vc, np.array(lengths, np.uint32), table)]
        cases.append((q, kc, vc, lengths, table, tensors, out))
    run_paged(ctx, *cases[0][:5])  # attributes are set outside of a capture
    graphs = [Graph().capture(ctx, lambda b: b.paged_attention(*c[5], c[6])) for c in cases]
    ctx.synchronize()
    for _ in range(5):  # two graphs on two streams at once
        graphs[0].replay(ctx.stream())
        graphs[1].replay(other.stream())
    ctx.synchronize()
    other.synchronize()
    for q, kc, vc, lengths, table, _, out in cases:
        check_paged(q, kc, vc, lengths, table, page, down(out))
    # the step goes on: other lengths at the same addresses
    q, kc, vc, _, table, tensors, out = cases[0]
    tensors[3].write(np.array([0, 3999], np.uint32))
    graphs[0].replay(ctx.stream())
    ctx.synchronize()
    check_paged(q, kc, vc, [0, 3999], table, page, down(out))
    for g in graphs:
        g.close()
    del rng


def test_refusals(ctx):
    e = lambda *shape: ctx.empty(list(shape), F16)  # noqa: E731
    u = lambda *shape: ctx.empty(list(shape), U32)  # noqa: E731
    f = lambda *shape: ctx.empty(list(shape), F32)  # noqa: E731

    def refused(status, word, call):
        b = ctx.begin_batch()
        with pytest.raises(mi.CoreError) as err:
            call(b)
        b.finish()
        assert err.value.status == status and word in err.value.message, err.value.message

    cache, lengths, table = e(3, 16, 2, 64), u(2), u(2, 2)
    paged_args = dict(q=e(2, 4, 64), k=cache, v=e(3, 16, 2, 64), n=lengths, t=table, o=e(2, 4, 64))

    def paged_with(**kw):
        a = dict(paged_args, **kw)
        return lambda b: b.paged_attention(a["q"], a["k"], a["v"], a["n"], a["t"], a["o"])

    refused(mi.ERR_SHAPE, "head_dim", paged_with(q=e(2, 4, 96), k=e(3, 16, 2, 96), v=e(3, 16, 2, 96), o=e(2, 4, 96)))
    refused(mi.ERR_SHAPE, "divisible", paged_with(q=e(2, 3, 64), o=e(2, 3, 64)))
    refused(mi.ERR_SHAPE, "mismatch", paged_with(v=e(3, 16, 1, 64)))
    refused(mi.ERR_SHAPE, "rank 4", paged_with(k=e(48, 2, 64)))
    refused(mi.ERR_SHAPE, "queries", paged_with(q=e(3, 4, 64), o=e(3, 4, 64)))
    refused(mi.ERR_SHAPE, "rows", paged_with(t=u(3, 2)))
    refused(mi.ERR_SHAPE, "page size", paged_with(k=e(3, 0, 2, 64), v=e(3, 0, 2, 64)))
    refused(mi.ERR_DTYPE, "lengths", paged_with(n=f(2)))
    refused(mi.ERR_DTYPE, "query", paged_with(q=f(2, 4, 64)))
    refused(mi.ERR_INVALID_ARGUMENT, "overlaps", paged_with(o=paged_args["q"]))
    other = mi.MetalContext(0)
    refused(mi.ERR_INVALID_ARGUMENT, "another context", paged_with(n=other.empty([2], U32)))
    whole = e(2 * 4 * 64 + 8)
    odd = ctx.tensor_from_device(whole.data_ptr() + 2, [2, 4, 64], F16)
    refused(mi.ERR_INVALID_ARGUMENT, "boundary", paged_with(q=odd))

    packed = dict(q=e(5, 4, 64), k=e(6, 2, 64), v=e(6, 2, 64), qs=u(3), ks=u(3), o=e(5, 4, 64))

    def packed_with(**kw):
        a = dict(packed, **kw)
        return lambda b: b.packed_attention(a["q"], a["k"], a["v"], a["qs"], a["ks"], True, a["o"])

    refused(mi.ERR_SHAPE, "key starts", packed_with(ks=u(2)))
    refused(mi.ERR_SHAPE, "sequences + 1", packed_with(qs=u(0), ks=u(0)))
    refused(mi.ERR_SHAPE, "differ", packed_with(q=e(5, 4, 128), o=e(5, 4, 128)))
    refused(mi.ERR_SHAPE, "mismatch", packed_with(v=e(5, 2, 64)))
    refused(mi.ERR_INVALID_ARGUMENT, "overlaps", packed_with(o=packed["q"]))

    append = dict(q=e(5, 4, 64), k=e(5, 2, 64), v=e(5, 2, 64), qw=None, kw=None, s=u(3), n=u(2), t=u(2, 2), kc=cache,
                  vc=e(3, 16, 2, 64), o=e(5, 4, 64), theta=1e4)

    def append_with(**kw):
        a = dict(append, **kw)
        return lambda b: b.paged_append(*[a[x] for x in ("q", "k", "v", "qw", "kw", "s", "n", "t", "kc", "vc", "o")],
                                        a["theta"])

    refused(mi.ERR_SHAPE, "starts", append_with(s=u(2)))
    refused(mi.ERR_SHAPE, "incompatible", append_with(kc=e(3, 16, 1, 64), vc=e(3, 16, 1, 64)))
    refused(mi.ERR_INVALID_ARGUMENT, "go together", append_with(o=None))
    refused(mi.ERR_INVALID_ARGUMENT, "goes with", append_with(kw=e(64)))
    refused(mi.ERR_SHAPE, "key weight", append_with(kw=e(32), qw=e(64)))
    refused(mi.ERR_SHAPE, "tokens", append_with(q=e(4, 4, 64), o=e(4, 4, 64)))
    refused(mi.ERR_INVALID_ARGUMENT, "theta", append_with(theta=0.0))
    refused(mi.ERR_INVALID_ARGUMENT, "overlaps", append_with(vc=cache))

    sample = dict(x=e(2, 50), t=f(2), k=u(2), p=f(2), m=f(2), u=f(2), o=u(2))

    def sample_with(**kw):
        a = dict(sample, **kw)
        return lambda b: b.sample(*[a[x] for x in ("x", "t", "k", "p", "m", "u", "o")])

    refused(mi.ERR_SHAPE, "rank 2", sample_with(x=e(100)))
    refused(mi.ERR_SHAPE, "per-row", sample_with(p=f(3)))
    refused(mi.ERR_DTYPE, "top_k", sample_with(k=f(2)))
    refused(mi.ERR_SHAPE, "logits a row", sample_with(x=e(2, 0)))
    few = e(64)  # shapes are refused before anything is read
    huge = ctx.tensor_from_device(few.data_ptr(), [2, 2 ** 22 + 1], F16)
    refused(mi.ERR_SHAPE, "logits a row", sample_with(x=huge, o=u(2)))
    refused(mi.ERR_INVALID_ARGUMENT, "NULL", lambda b: mi._check(mi.lib().mi_batch_sample(b._h, *[None] * 7)))


def test_offsets_beyond_32_bits(ctx):
    # caches of more than 2^32 values: the pages at their end
    rng = np.random.default_rng(41)
    page, kvh, hd, n = 16, 8, 128, 77
    pages = 2 ** 32 // (page * kvh * hd) + 8
    kc, vc = ctx.empty([pages, page, kvh, hd], F16), ctx.empty([pages, page, kvh, hd], F16)
    table = (pages - 1 - np.arange(5)[None]).astype(np.uint32)
    q, k, v = normal(rng, n, 16, hd), normal(rng, n, kvh, hd), normal(rng, n, kvh, hd)
    out = up(ctx, np.zeros((1, 16, hd), np.float16))
    small = [ctx.empty([8, page, kvh, hd], F16) for _ in range(2)]
    low = (7 - np.arange(5)[None]).astype(np.uint32)
    results = []
    for a, b, t in ((kc, vc, table), (*small, low)):
        rotated = up(ctx, np.zeros_like(q))
        tt, tl, ts = up(ctx, t), up(ctx, np.array([n], np.uint32)), up(ctx, np.array([0, n], np.uint32))
        one(ctx, lambda bt: bt.paged_append(up(ctx, q), up(ctx, k), up(ctx, v), None, None, ts, tl, tt, a, b, rotated, 1e6))
        one(ctx, lambda bt: bt.paged_attention(up(ctx, down(rotated)[-1:]), a, b, tl, tt, out))
        results.append(down(out).view(np.uint16).copy())
    np.testing.assert_array_equal(results[0], results[1])
    assert np.any(results[0])


@pytest.mark.parametrize("hd", [64, 128])
def test_large_groups(ctx, hd):
    # more query heads to a KV head than a row tile or a product has places
    rng = np.random.default_rng(42)
    lengths = [37, 90]
    table, pages = paged(rng, lengths, 16)
    q, kc, vc = normal(rng, 2, 200, hd), normal(rng, pages, 16, 1, hd), normal(rng, pages, 16, 1, hd)
    check_paged(q, kc, vc, lengths, table, 16, run_paged(ctx, q, kc, vc, lengths, table))
    qs, ks = starts([5, 3]), starts([5, 103])
    q, k, v = normal(rng, 8, 200, hd), normal(rng, 108, 1, hd), normal(rng, 108, 1, hd)
    check_packed(q, k, v, qs, ks, True, run_packed(ctx, q, k, v, qs, ks, True))


def test_many_sequences(ctx):
    # more sequences than a block has threads, prompts of every small length
    rng = np.random.default_rng(43)
    lengths = [i % 7 for i in range(1500)]
    table, pages = paged(rng, lengths, 4)
    q, kc, vc = normal(rng, 1500, 2, 64), normal(rng, pages, 4, 1, 64), normal(rng, pages, 4, 1, 64)
    check_paged(q, kc, vc, lengths, table, 4, run_paged(ctx, q, kc, vc, lengths, table))
    qs = ks = starts(lengths)
    q, k, v = normal(rng, qs[-1], 2, 64), normal(rng, qs[-1], 1, 64), normal(rng, qs[-1], 1, 64)
    check_packed(q, k, v, qs, ks, True, run_packed(ctx, q, k, v, qs, ks, True))
    kc, vc = np.zeros((pages, 4, 1, 64), np.float16), np.zeros((pages, 4, 1, 64), np.float16)
    _, _, got = run_append(ctx, None, k, v, None, None, qs, lengths, table, kc, vc)
    for s in range(0, 1500, 97):
        np.testing.assert_array_equal(got.reshape(-1, 1, 64)[rows_of(table, s, lengths[s], 4)], v[qs[s]:qs[s + 1]])


@pytest.mark.parametrize("n", [1000003, 2 ** 22])
@pytest.mark.parametrize("kind", ["normal", "equal", "lowest"])
def test_sample_counts_beyond_16_bits(ctx, kind, n):
    rng = np.random.default_rng(44)
    options = [OPTIONS[0] + (0.37,), OPTIONS[8] + (UNIFORMS[-1],), (1.0, n // 2, 0.9, 0.0, 0.99)]
    bits = np.stack([logits_of(kind, rng, n) for _ in options])
    want = np.array([sample64(b, *o) for b, o in zip(bits, options)], np.uint32)
    np.testing.assert_array_equal(run_sample(ctx, bits, options), want)
    # as many rows as make a CTA take a whole one
    many = run_sample(ctx, np.tile(bits, (8, 1)), options * 8) if n < 2 ** 22 else np.tile(want, 8)
    np.testing.assert_array_equal(many, np.tile(want, 8))


def test_a_captured_step_of_all_ops(ctx):
    rng = np.random.default_rng(45)
    page, hd, qh, kvh, width = 16, 128, 8, 2, 20
    prompts = [150, 3, 90]
    st = starts(prompts)
    table = rng.permutation(3 * width).reshape(3, width).astype(np.uint32)
    q, k, v = (normal(rng, st[-1], h, hd) for h in (qh, kvh, kvh))
    logits = normal(rng, 40, 3000)
    kc, vc = ctx.empty([3 * width, page, kvh, hd], F16), ctx.empty([3 * width, page, kvh, hd], F16)
    t = {n: up(ctx, x) for n, x in dict(
        q=q, k=k, v=v, st=st.astype(np.uint32), n=np.array(prompts, np.uint32), table=table, last=q[st[1:] - 1],
        logits=logits, temp=np.full(40, 0.8, np.float32), top_k=np.full(40, 50, np.uint32),
        top_p=np.full(40, 0.9, np.float32), min_p=np.zeros(40, np.float32),
        u=rng.random(40).astype(np.float32)).items()}
    rotated, packed_out, paged_out, tokens = (up(ctx, np.zeros_like(q)), up(ctx, np.zeros_like(q)),
                                              up(ctx, np.zeros((3, qh, hd), np.float16)), ctx.empty([40], U32))

    def step(b):
        b.paged_append(t["q"], t["k"], t["v"], None, None, t["st"], t["n"], t["table"], kc, vc, rotated, 1e6)
        b.packed_attention(t["q"], t["k"], t["v"], t["st"], t["st"], True, packed_out)
        b.paged_attention(t["last"], kc, vc, t["n"], t["table"], paged_out)
        b.sample(t["logits"], t["temp"], t["top_k"], t["top_p"], t["min_p"], t["u"], tokens)

    outs = (rotated, packed_out, paged_out, tokens)
    one(ctx, step)
    eager = [down(o).copy() for o in outs]
    graph = Graph().capture(ctx, step)
    for _ in range(3):
        for o in outs:
            o.write(np.zeros_like(down(o)))
        graph.replay(ctx.stream())
        ctx.synchronize()
        for o, e in zip(outs, eager):
            np.testing.assert_array_equal(down(o).view(np.uint16), e.view(np.uint16))
    graph.close()
    check_packed(q, k, v, st, st, True, eager[1])
