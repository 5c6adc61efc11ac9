"""The ops of a ragged batch where their numbers, their order and their errors
are easily wrong: many keys of small weight, several open batches, kernels that
only large batches reach, first calls inside a capture.

Tolerances of attention. A weight is held in FP16 over a base at which the
row's largest is 2^7 or more: it is off by at most 2^-11 of itself or 2^-32 of
the largest, which is at most the sum, so a mean over n keys moves by at most
2 (2^-11 + n 2^-32) max|v|. The tensor cores cut a product off at 2^-25 of the
accumulator's power of two and the sum of 16 at 2^-23: (2^-25 + 2^-27) max|v| a
key, for the 8,240 keys at most that one accumulator takes. The weights of as
many are summed in FP32, every other one in one sum: 4,120 2^-24; adding up what
several accumulators took is off by 2^-24 for each. Exponentials and joins add
less than 2^-16, and the rounded output 2^-11.
"""
import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest

import metal_infer as mi
from test_batched_ops_gpu import (OPTIONS, UNIFORMS, Graph, attention64, check, check_packed, down, logits_of, normal, paged, rows_of,
                                  run_packed, run_paged, run_sample, sample64, starts, up)

pytestmark = pytest.mark.gpu


# ---- weights far below a row's largest --------------------------------------------


def small_weights(hd, exponent, n):
    """A query, a first key of weight 1 and n - 1 others of about 2^-exponent;
    the sum of the others' weights."""
    q, first = np.zeros(hd, np.float16), np.zeros(hd, np.float16)
    q[3] = 8
    first[3] = exponent * np.log(2) * np.sqrt(hd) / 8
    score = 8 * float(first[3]) / np.sqrt(hd)
    return q, first, (n - 1) * np.exp(-score)


def mean_bound(n):
    """Of a mean over n keys whose values are at most 1."""
    taken = min(n, 8240)
    return (2 * (2.0 ** -11 + n * 2.0 ** -32) + taken * (2.0 ** -25 + 2.0 ** -27) + (taken / 2 + 2 * n / 1024) * 2.0 ** -24
            + 2.0 ** -16 + 2.0 ** -11)


@pytest.mark.parametrize("other", [1, -1])
@pytest.mark.parametrize("exponent", [25.05, 24.5])
@pytest.mark.parametrize("hd,queries", [(64, 37888), (128, 37888), (64, 7), (128, 7)])
def test_packed_attention_sums_weights_far_below_the_largest(ctx, hd, queries, exponent, other):
    # a thread that sees all keys, and parts joined
    n = 131072
    q, first, rest = small_weights(hd, exponent, n)
    k, v = np.zeros((n, 1, hd), np.float16), np.full((n, 1, hd), other, np.float16)
    k[0, 0], v[0] = first, 1
    got = run_packed(ctx, np.tile(q, (queries, 1, 1)), k, v, [0, queries], [0, n], False).astype(np.float64)
    want = (1 + other * rest) / (1 + rest)
    assert np.abs(got - want).max() <= mean_bound(n), (got.min(), got.max(), want)


@pytest.mark.parametrize("hd,queries", [(64, 7), (128, 200)])
def test_packed_attention_sums_small_weights_in_rows_done_again(ctx, hd, queries):
    # the last key's value is not a number, and the last query alone sees it: the
    # rows before it meet it in the products and are computed a second time
    n = 131072
    q, first, rest = small_weights(hd, 25.05, n)
    k, v = np.zeros((n, 1, hd), np.float16), np.full((n, 1, hd), -1, np.float16)
    k[0, 0], v[0], v[n - 1] = first, 1, np.nan
    got = run_packed(ctx, np.tile(q, (queries, 1, 1)), k, v, [0, queries], [0, n], True).astype(np.float64)
    seen = rest / (n - 1) * (n - 1 - np.arange(queries - 1, 0, -1))
    want = ((1 - seen) / (1 + seen))[:, None]
    assert np.abs(got[:-1, 0] - want).max() <= mean_bound(n)
    assert np.all(np.isnan(got[-1]))


@pytest.mark.parametrize("hd,qh,kvh,queries,keys,causal", [
    (128, 16, 8, [2400, 2300], [20000, 9500], True),     # in a planned order
    (64, 16, 8, [2400, 2300], [20000, 9500], False),
    (128, 4, 1, [70, 300], [100, 66000], True),          # split, its parts as long
    (64, 8, 8, [1480], [25000], True),                   # one sequence
])
def test_packed_attention_rows_longer_than_an_accumulator_takes(ctx, hd, qh, kvh, queries, keys, causal):
    # scores that grow along the keys, so that what was put aside is weighed
    # down again and again; NaN behind the last sequence
    rng = np.random.default_rng(51)
    qs, ks = starts(queries), starts(keys)
    q, k, v = normal(rng, qs[-1], qh, hd) * np.float16(3), normal(rng, ks[-1] + 60, kvh, hd), normal(rng, ks[-1] + 60, kvh, hd)
    for s, n in enumerate(keys):
        k[ks[s]:ks[s + 1]] *= np.linspace(0.2, 1, n).astype(np.float16)[:, None, None]
    k[ks[-1]:], v[ks[-1]:] = np.nan, np.nan
    got = run_packed(ctx, q, k, v, qs, ks, causal)
    assert np.all(np.isfinite(got))
    for s, (n, m) in enumerate(zip(queries, keys)):
        for i in {0, 1, n // 2, n - 2, n - 1}:
            for h in (0, qh - 1):
                row, g = qs[s] + i, h // (qh // kvh)
                seen = m - (n - 1 - i) if causal else m
                want, tol = attention64(q[row:row + 1, h], k[ks[s]:ks[s + 1], g], v[ks[s]:ks[s + 1], g], [seen])
                big = np.abs(v[ks[s]:ks[s] + seen, g].astype(float)).max()
                check(got[row:row + 1, h], want, tol + big * mean_bound(seen), (s, i, h))
    np.testing.assert_array_equal(got.view(np.uint16), run_packed(ctx, q, k, v, qs, ks, causal).view(np.uint16))


@pytest.mark.parametrize("other", [1, -1])
@pytest.mark.parametrize("exponent", [25.05, 24.5])
@pytest.mark.parametrize("hd,qh", [(64, 1), (128, 1), (128, 12)])
def test_paged_attention_sums_weights_far_below_the_largest(ctx, hd, qh, exponent, other):
    # as many long sequences as leave a warp a quarter of one, all of the same pages
    n, page, sequences = 262144, 256, 296
    q, first, rest = small_weights(hd, exponent, n)
    k, v = np.zeros((n // page, page, 1, hd), np.float16), np.full((n // page, page, 1, hd), other, np.float16)
    k[0, 0, 0], v[0, 0] = first, 1
    table = np.tile(np.arange(n // page, dtype=np.uint32), (sequences, 1))
    got = run_paged(ctx, np.tile(q, (sequences, qh, 1)), k, v, [n] * sequences, table).astype(np.float64)
    want = (1 + other * rest) / (1 + rest)
    assert np.abs(got - want).max() <= mean_bound(n), (got.min(), got.max(), want)


@pytest.mark.parametrize("hd,qh,page", [(64, 3, 16), (64, 20, 24), (128, 3, 24), (128, 20, 16)])
def test_paged_attention_parts_longer_than_an_accumulator_takes(ctx, hd, qh, page):
    # scores that grow along the keys, so that what was put aside is weighed
    # down again and again; units that lie in one block, in two and in between
    rng = np.random.default_rng(52)
    n, sequences = 40000, 300
    lengths = [n - 7 * s for s in range(sequences)]
    table, pages = paged(rng, [n], page)
    table = np.tile(table, (sequences, 1))
    q = normal(rng, sequences, qh, hd) * np.float16(3)
    kc, vc = np.full((pages, page, 1, hd), np.nan, np.float16), np.full((pages, page, 1, hd), np.nan, np.float16)
    rows = rows_of(table, 0, n, page)
    kc.reshape(-1, hd)[rows] = normal(rng, n, hd) * np.linspace(0.2, 1, n).astype(np.float16)[:, None]
    vc.reshape(-1, hd)[rows] = normal(rng, n, hd)
    got = run_paged(ctx, q, kc, vc, lengths, table)
    assert np.all(np.isfinite(got))
    k, v = kc.reshape(-1, hd)[rows], vc.reshape(-1, hd)[rows]
    big = np.abs(v.astype(float)).max()
    for s in (0, 1, 77, 148, 149, 298, 299):
        for h in (0, qh - 1):
            want, tol = attention64(q[s, h:h + 1], k, v, [lengths[s]])
            check(got[s, h:h + 1], want, tol + big * mean_bound(n), (s, h))
    np.testing.assert_array_equal(got.view(np.uint16), run_paged(ctx, q, kc, vc, lengths, table).view(np.uint16))


@pytest.mark.parametrize("hd,n,sequences", [(64, 50, 2), (128, 3000, 2), (64, 30000, 300)])
def test_attention_over_scores_of_minus_infinity(ctx, hd, n, sequences):
    # keys of weight 0 in front leave the others' result alone; nothing but such
    # keys is 0 / 0, in one piece, in joined pieces and in what was put aside
    rng = np.random.default_rng(53)
    q, k, v = normal(rng, sequences, 2, hd), normal(rng, n, 1, hd), normal(rng, n, 1, hd)
    q[:, :, 0] = 1
    k[:n - 7, :, 0] = -np.inf
    page = 10
    table = np.tile(np.arange(n // page, dtype=np.uint32), (sequences, 1))
    lengths = [n if s % 2 == 0 else n - 7 for s in range(sequences)]
    got = run_paged(ctx, q, k.reshape(-1, page, 1, hd), v.reshape(-1, page, 1, hd), lengths, table)
    assert np.all(np.isnan(got[1::2]))
    for s in (0, sequences - 2):
        for h in (0, 1):
            check(got[s, h:h + 1], *attention64(q[s, h:h + 1], k[n - 7:, 0], v[n - 7:, 0], [7]), (s, h))
    for keys in (n, n - 7):
        got = run_packed(ctx, q[:2], k, v, [0, 2], [0, keys], False)
        if keys == n:
            check_packed(q[:2], k[n - 7:], v[n - 7:], [0, 2], [0, 7], False, got)
        else:
            assert np.all(np.isnan(got))


# ---- which batch answers for what a kernel refused ---------------------------------------


class Decode:
    """A small paged attention whose lengths may be bad."""

    def __init__(self, ctx, lengths=(20, 9)):
        rng = np.random.default_rng(61)
        self.q, self.kc, self.vc = normal(rng, 2, 2, 64), normal(rng, 4, 16, 1, 64), normal(rng, 4, 16, 1, 64)
        self.table, self.want = np.array([[0, 1], [2, 3]], np.uint32), None
        self.tensors = [up(ctx, x) for x in (self.q, self.kc, self.vc, np.array(lengths, np.uint32), self.table)]
        self.out = up(ctx, np.zeros_like(self.q))

    def __call__(self, b):
        b.paged_attention(*self.tensors, self.out)


def sample_call(ctx, uniform):
    rng = np.random.default_rng(62)
    one_of = lambda x: up(ctx, np.full(2, x, np.float32))  # noqa: E731
    t = [up(ctx, normal(rng, 2, 100)), one_of(1), up(ctx, np.zeros(2, np.uint32)), one_of(1), one_of(0), one_of(uniform),
         up(ctx, np.zeros(2, np.uint32))]
    return lambda b: b.sample(*t)


def committed(ctx, *calls):
    b = ctx.begin_batch()
    for call in calls:
        call(b)
    return b.commit()


def refused(status, word, call):
    with pytest.raises(mi.CoreError) as e:
        call()
    assert e.value.status == status and word in e.value.message, e.value.message


@pytest.mark.parametrize("first_waited", ["first", "last"])
def test_each_of_several_open_batches_answers_for_itself(ctx, first_waited):
    good, bad = Decode(ctx), Decode(ctx, (20, 33))
    batches = [(committed(ctx, good), None), (committed(ctx, bad), (mi.ERR_INVALID_ARGUMENT, "length")),
               (committed(ctx, good), None), (committed(ctx, sample_call(ctx, 1.0)), (mi.ERR_CONFIG, "sampling")),
               (committed(ctx, bad, good), (mi.ERR_INVALID_ARGUMENT, "length")), (committed(ctx, good), None)]
    ctx.synchronize()
    for p, wrong in batches if first_waited == "first" else batches[::-1]:
        if wrong:
            refused(*wrong, p.wait)
        else:
            p.wait()
    assert ctx.kernel_status() == 0


def test_the_context_answers_for_what_no_batch_does(ctx):
    # a committed batch keeps its answer; an abandoned one leaves it to the context
    p = committed(ctx, Decode(ctx, (20, 33)))
    assert ctx.kernel_status() == 0
    refused(mi.ERR_INVALID_ARGUMENT, "length", p.wait)
    b = ctx.begin_batch()
    sample_call(ctx, -1.0)(b)
    del b
    refused(mi.ERR_CONFIG, "sampling", ctx.kernel_status)
    assert ctx.kernel_status() == 0
    committed(ctx, Decode(ctx)).wait()


def test_a_replayed_refusal_comes_with_the_next_commit():
    ctx = mi.MetalContext(0)
    step, good = Decode(ctx), Decode(ctx)
    graph = Graph().capture(ctx, step)
    before = committed(ctx, good)
    step.tensors[3].write(np.array([20, 33], np.uint32))
    graph.replay(ctx.stream())
    after = committed(ctx, good)
    ctx.synchronize()
    before.wait()
    refused(mi.ERR_INVALID_ARGUMENT, "length", after.wait)
    graph.replay(ctx.stream())
    refused(mi.ERR_INVALID_ARGUMENT, "length", ctx.kernel_status)
    step.tensors[3].write(np.array([20, 9], np.uint32))
    graph.replay(ctx.stream())
    assert ctx.kernel_status() == 0
    graph.close()


def test_many_open_batches(ctx):
    # more than the context keeps words for at first
    bad, good = Decode(ctx, (40, 9)), Decode(ctx)
    pending = [committed(ctx, bad if i % 3 == 0 else good) for i in range(150)]
    for i, p in enumerate(pending):
        if i % 3 == 0:
            refused(mi.ERR_INVALID_ARGUMENT, "length", p.wait)
        else:
            p.wait()


def test_a_commit_beside_a_capture_of_another_context(ctx):
    # a capture that forbids the thread to allocate goes on beside another
    # context's batch and its commit
    other, rt = mi.MetalContext(0), ctypes.CDLL("libcudart.so.12")
    step, beside = Decode(ctx), Decode(other, (20, 33))
    b = other.begin_batch()
    beside(b)
    stream, graph = ctypes.c_void_p(ctx.stream()), ctypes.c_void_p()
    mine = ctx.begin_batch()
    ctx.synchronize()
    assert rt.cudaStreamBeginCapture(stream, ctypes.c_int(0)) == 0  # global
    try:
        step(mine)
        p = b.commit()
    finally:
        status = rt.cudaStreamEndCapture(stream, ctypes.byref(graph))
    assert status == 0 and rt.cudaGraphDestroy(graph) == 0
    refused(mi.ERR_INVALID_ARGUMENT, "length", p.wait)
    mine.finish()


# ---- together, without the host -------------------------------------------------------------


@pytest.mark.parametrize("norm", [True, False])
def test_prompts_in_chunks_and_then_single_tokens(ctx, norm):
    # each prompt's rotated keys and its values are appended twice: to the pages
    # that decoding reads, and, as pages of one row, end to end for the attention
    # of the prompt's chunks. One batch a step, nothing goes through the host.
    rng = np.random.default_rng(91)
    qh, kvh, hd, page, chunks = 8, 2, 64, 16, [[40, 7, 120], [33, 0, 81], [5, 90, 1]]
    totals = np.sum(chunks, 0)
    room = starts(totals + 3)  # of the packed rows of a prompt
    width = int((totals.max() + 3 + page - 1) // page)
    table = up(ctx, rng.permutation(3 * width).reshape(3, width).astype(np.uint32))
    rows = np.full((3, totals.max() + 3), 0xFFFFFFF0, np.uint32)
    for s in range(3):
        rows[s, :totals[s] + 3] = room[s] + np.arange(totals[s] + 3)
    rows = up(ctx, rows)
    kc, vc = (up(ctx, np.full((3 * width, page, kvh, hd), np.nan, np.float16)) for _ in range(2))
    kp, vp = (up(ctx, np.full((int(room[-1]), 1, kvh, hd), np.nan, np.float16)) for _ in range(2))
    weights = [up(ctx, normal(rng, hd)) if norm else None for _ in range(2)]
    keys, values, old = [np.zeros((0, kvh, hd), np.float16)] * 3, [np.zeros((0, kvh, hd), np.float16)] * 3, np.zeros(3, int)

    def rotated(x, weight, first):
        # the engine's contiguous ops, one sequence at a time
        if not norm:
            return down(ctx.rope(up(ctx, x), first, 1e4))
        flat, other = ctx.empty([first + len(x), x.shape[1], hd], mi.DType.F16), up(ctx, x)
        b = ctx.begin_batch()
        b.qk_norm_rope_cache(other, up(ctx, x), weight, weight, flat, mi.QkNormRopeCacheConfig(first, 1e4, 1e-6))
        b.finish()
        return down(flat)[first:]

    for counts in chunks + [[1, 1, 1]] * 3:
        single, st = counts == [1, 1, 1], starts(counts)
        q, k, v = (normal(rng, st[-1], h, hd) for h in (qh, kvh, kvh))
        lengths = old + counts
        tq, tk, tv, ts, tl = (up(ctx, x) for x in (q, k, v, st.astype(np.uint32), lengths.astype(np.uint32)))
        turned, out = up(ctx, np.zeros_like(q)), up(ctx, np.zeros_like(q))
        b = ctx.begin_batch()
        b.paged_append(tq, tk, tv, *weights, ts, tl, table, kc, vc, turned, 1e4)
        if single:
            b.paged_attention(turned, kc, vc, tl, table, out)
        else:
            # the prompts so far, packed end to end: one call for each, as their
            # rows have gaps between them
            b.paged_append(None, tk, tv, None, weights[1], ts, tl, rows, kp, vp, None, 1e4)
            flat_k, flat_v = kp.reshape([int(room[-1]), kvh, hd]), vp.reshape([int(room[-1]), kvh, hd])
            for s in range(3):
                b.packed_attention(turned, flat_k, flat_v, up(ctx, st[s:s + 2].astype(np.uint32)),
                                   up(ctx, np.array([room[s], room[s] + lengths[s]], np.uint32)), True, out)
        b.finish()
        got, rq = down(out), down(turned)
        for s, n in enumerate(counts):
            if n == 0:
                continue
            a, e = st[s], st[s + 1]
            np.testing.assert_array_equal(rq[a:e].view(np.uint16), rotated(q[a:e], weights[0], int(old[s])).view(np.uint16))
            keys[s] = np.concatenate([keys[s], rotated(k[a:e], weights[1], int(old[s]))])
            values[s] = np.concatenate([values[s], v[a:e]])
            for h in range(qh):
                g = h // (qh // kvh)
                want, tol = attention64(rq[a:e, h], keys[s][:, g], values[s][:, g],
                                        [lengths[s] - n + i + 1 for i in range(n)])
                check(got[a:e, h], want, tol, (counts, s, h))
        old = lengths


# ---- refusals -------------------------------------------------------------------------------


def test_paged_append_refuses_rotated_queries_over_a_tensor_that_it_reads(ctx):
    e = lambda *shape: ctx.empty(list(shape), mi.DType.F16)  # noqa: E731
    u = lambda *shape: ctx.empty(list(shape), mi.DType.U32)  # noqa: E731
    # every input at the output's address in turn: only the queries themselves may be there
    named = dict(query=e(3, 2, 64), key=e(3, 2, 64), value=e(3, 2, 64), query_weight=e(64), key_weight=e(64), starts=u(3),
                 lengths=u(2), table=u(2, 2), key_cache=e(3, 16, 2, 64), value_cache=e(3, 16, 2, 64))
    for name, t in named.items():
        whole = ctx.empty([2 * int(np.prod(t.shape())) + 400], mi.DType.U32)
        kind = t.dtype()
        over = ctx.tensor_from_device(whole.data_ptr(), t.shape(), kind)
        out = ctx.tensor_from_device(whole.data_ptr(), [3, 2, 64], mi.DType.F16)
        args = dict(named, **{name: over})
        b = ctx.begin_batch()
        if name == "query":
            b.paged_append(*args.values(), out, 1e4)
        else:
            with pytest.raises(mi.CoreError) as err:
                b.paged_append(*args.values(), out, 1e4)
            assert err.value.status == mi.ERR_INVALID_ARGUMENT and "overlaps" in err.value.message, name
        b.finish()


# ---- first calls inside a capture --------------------------------------------------------------


FIRST_CALLS = '''
import ctypes, sys
import numpy as np
import metal_infer as mi
from test_batched_ops_gpu import Graph, down, normal, starts, up
class Capture(Graph):
    def call(self, name, *args):
        if name == "cudaStreamBeginCapture":
            args = (args[0], ctypes.c_int(int(sys.argv[1])))
        super().call(name, *args)
ctx = mi.MetalContext(0)
rng = np.random.default_rng(71)
u32 = lambda x: up(ctx, np.asarray(x, np.uint32))
full = lambda *shape: up(ctx, np.zeros(shape, np.float16))
f16 = lambda *shape: up(ctx, normal(rng, *shape))
calls = {}
for hd in (64, 128):
    q, out = f16(3, 4, hd), full(3, 4, hd)
    calls["append", hd] = ("paged_append", [q, f16(3, 2, hd), f16(3, 2, hd), f16(hd), f16(hd), u32([0, 3]), u32([5]), u32([[0]]),
                                            full(1, 16, 2, hd), full(1, 16, 2, hd), out, 1e4], out)
    for page in (16, 24):
        out = full(3, 4, hd)
        calls["paged", hd, page] = ("paged_attention", [q, f16(3 * 48 // page, page, 2, hd), f16(3 * 48 // page, page, 2, hd),
                                                        u32([40, 0, 17]), u32(np.arange(3 * 48 // page).reshape(3, -1)), out], out)
    for name, qh, queries, keys in (("own", 4, [30], [30]), ("planned", 64, [50] * 20, [50] * 20), ("split", 4, [9], [5000]),
                                    ("long", 1, [37888], [9000]), ("long split", 4, [9], [90000])):
        out = full(sum(queries), qh, hd)
        kvh = 8 if qh == 64 else 1
        calls[name, hd] = ("packed_attention", [f16(sum(queries), qh, hd), f16(sum(keys), kvh, hd), f16(sum(keys), kvh, hd),
                                                u32(starts(queries)), u32(starts(keys)), False, out], out)
for rows in (3, 20, 40, 90):
    f = lambda x: up(ctx, np.full(rows, x, np.float32))
    out = u32([0] * rows)
    calls["sample", rows] = ("sample", [f16(rows, 999), f(0.8), u32([50] * rows), f(0.9), f(0), f(0.3), out], out)
ctx.synchronize()
graphs = {k: Capture().capture(ctx, lambda b: getattr(b, op)(*args)) for k, (op, args, _) in calls.items()}
got = {}
for k, g in graphs.items():
    g.replay(ctx.stream())
    got[k] = down(calls[k][2]).copy()
assert ctx.kernel_status() == 0
for k, (op, args, out) in calls.items():
    out.write(np.zeros_like(got[k]))
    b = ctx.begin_batch()
    getattr(b, op)(*args)
    b.finish()
    assert np.any(got[k]) and np.array_equal(got[k].view(np.uint8), down(out).view(np.uint8)), k
print("same:", len(calls))
'''


@pytest.mark.parametrize("mode", [0, 1, 2])  # global, of the thread, relaxed
def test_first_calls_inside_a_capture(mode):
    # a process that has called none of the ops: captured, replayed, and then called
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    path = os.pathsep.join(os.path.join(root, d) for d in ("tests", "metal-infer-rs_b200", "oracle"))
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS, str(mode)], env=dict(os.environ, PYTHONPATH=path), capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0 and "same:" in r.stdout, (r.stdout[-2000:], r.stderr[-2000:])


# ---- kernels that large batches reach -------------------------------------------------------------


@pytest.mark.parametrize("n", [49153, 151936, 200003, 524224])
@pytest.mark.parametrize("kind", ["normal", "equal", "two values", "masked", "lowest"])
def test_sample_large_vocabularies_in_large_batches(ctx, kind, n):
    # one CTA to a row (90 rows) and two (50): rows of several segments, after each
    # of which counts near 2^16 move to a list; an odd n leaves rows unaligned
    rng = np.random.default_rng(81)
    options = [OPTIONS[0] + (0.37,), OPTIONS[1] + (0.9,), OPTIONS[2] + (0.1,), OPTIONS[3] + (0.999,),
               OPTIONS[8] + (UNIFORMS[-1],), (1.0, n // 2, 0.9, 0.0, 0.99), (1.3, n - 1, 1.0, 0.0, 0.73)]
    bits = np.stack([logits_of(kind, rng, n) for _ in options])
    want = np.array([sample64(b, *o) for b, o in zip(bits, options)], np.uint32)
    for rows in (90, 50, 25, 7):
        pick = np.arange(rows) % len(options)
        np.testing.assert_array_equal(run_sample(ctx, bits[pick], [options[i] for i in pick]), want[pick])


@pytest.mark.parametrize("kind", ["normal", "equal", "two values"])
def test_sample_the_largest_vocabulary_in_large_batches(ctx, kind):
    # 86 segments to a CTA's row, and a count that moves to the list with most of them
    n, rng = 2 ** 22, np.random.default_rng(83)
    options = [OPTIONS[0] + (0.37,), (1.0, n // 2, 0.9, 0.0, 0.99)]
    bits = np.stack([logits_of(kind, rng, n) for _ in options])
    want = np.array([sample64(b, *o) for b, o in zip(bits, options)], np.uint32)
    for rows in (80, 44):
        pick = np.arange(rows) % 2
        np.testing.assert_array_equal(run_sample(ctx, bits[pick], [options[i] for i in pick]), want[pick])


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("queries,keys", [
    ([700, 0, 333, 1200, 1, 81, 160, 80, 900], [700, 0, 333, 1200, 1, 81, 160, 80, 900]),
    ([500, 640, 77, 300, 900, 129], [530, 700, 70, 0, 1000, 2129])])
def test_packed_attention_ragged_prompts_in_a_planned_order(ctx, hd, queries, keys, causal):
    # more than two items to an SM and no long prefix: the order from long to
    # short; sequences without queries or keys, last tiles of every size, and NaN
    # behind the last sequence
    rng = np.random.default_rng(82)
    qs, ks = starts(queries, 3), starts(keys, 5)
    q, k, v = normal(rng, qs[-1] + 9, 32, hd), normal(rng, ks[-1] + 200, 8, hd), normal(rng, ks[-1] + 200, 8, hd)
    q[qs[-1]:], k[ks[-1]:], v[ks[-1]:] = np.nan, np.nan, np.nan
    k[:5], v[:5] = np.inf, np.nan
    got = run_packed(ctx, q, k, v, qs, ks, causal)
    check_packed(q, k, v, qs, ks, causal, got, heads=[0, 31])
    assert np.all(np.isfinite(got[:qs[-1]])) and np.all(got[:3] == 7) and np.all(got[qs[-1]:] == 7)
    np.testing.assert_array_equal(got.view(np.uint16), run_packed(ctx, q, k, v, qs, ks, causal).view(np.uint16))
