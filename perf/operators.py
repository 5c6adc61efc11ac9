"""The operators of a batched serving step, as cases to be timed and compared.

Four operators that every step of a loop over several requests runs: the append
of rotated keys and values to a paged cache, attention of one new token per
request over its pages, attention over packed prompts, and sampling from given
random numbers. ``run`` computes them in plain torch operations, or, with
``own``, calls the engine's batch ops (metal_infer).
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

# (query heads, KV heads) of grouped-query models from small to large, and
# ratios that do not divide a tile
HEADS = [(16, 8), (32, 8), (64, 8), (8, 8), (28, 4), (12, 2), (7, 1), (40, 8)]
VOCABULARIES = [151936, 128256, 50257, 32000]
THETA = 1e6
EPSILON = 1e-6


def listed():
    return [
        # the decode step of a small batch appends one token a request
        dict(name="append_decode", op="append", sequences=16, low=1, high=1, offset=2000, qh=16, kvh=8, hd=128,
             page=16, norm=True),
        # prompts of different lengths enter the cache in one call
        dict(name="append_prompts", op="append", sequences=12, low=3, high=1500, offset=0, qh=32, kvh=8, hd=128,
             page=64, norm=True),
        # one user, a short conversation: the latency of a single call
        dict(name="decode_one", op="decode", sequences=1, low=900, high=900, qh=16, kvh=8, hd=128, page=16),
        # an ordinary serving batch: every length from a few tokens to thousands
        dict(name="decode_ragged", op="decode", sequences=64, low=1, high=8192, qh=32, kvh=8, hd=128, page=16),
        # many short chats of a model with narrow heads and much sharing
        dict(name="decode_many", op="decode", sequences=256, low=100, high=1500, qh=64, kvh=8, hd=64, page=64),
        # a few very long documents: the split over the length
        dict(name="decode_long", op="decode", sequences=3, low=70000, high=131072, qh=32, kvh=8, hd=128, page=128),
        # short questions arriving together
        dict(name="packed_short", op="packed", sequences=16, low=1, high=200, prefix=0, qh=16, kvh=8, hd=128),
        # prompts of mixed lengths in one call
        dict(name="packed_ragged", op="packed", sequences=10, low=20, high=2500, prefix=0, qh=32, kvh=8, hd=128),
        # one long prompt
        dict(name="packed_long", op="packed", sequences=1, low=8192, high=8192, prefix=0, qh=32, kvh=8, hd=128),
        # the last chunk of prompts whose beginning was computed before
        dict(name="packed_chunk", op="packed", sequences=3, low=200, high=700, prefix=4000, qh=64, kvh=8, hd=64),
        # sampling for one request
        dict(name="sample_one", op="sample", rows=1, vocabulary=151936),
        # sampling for a serving batch, options of their own for each request
        dict(name="sample_batch", op="sample", rows=96, vocabulary=151936),
    ]


def _spread(rng, low, high):
    """An integer in [low, high], even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "packed", "packed", "sample"])
    if op == "sample":
        return dict(op=op, rows=_spread(rng, 1, 96), vocabulary=rng.choice(VOCABULARIES + [rng.randint(1000, 151936)]))
    qh, kvh = rng.choice(HEADS)
    case = dict(op=op, qh=qh, kvh=kvh, hd=rng.choice([64, 128]))
    if op == "append":
        high = _spread(rng, 1, 1500)
        case.update(sequences=_spread(rng, 1, max(1, min(128, 8000 // high))), low=rng.randint(1, high), high=high,
                    offset=rng.choice([0, _spread(rng, 1, 200000)]), page=rng.choice([8, 16, 32, 64, 48]),
                    norm=rng.random() < 0.5)
    elif op == "decode":
        high = _spread(rng, 1, 131072)
        most = max(1, min(256, 3 * 131072 * 8 * 128 // (high * kvh * case["hd"])))
        case.update(sequences=_spread(rng, 1, most), low=rng.randint(1, high), high=high,
                    page=rng.choice([16, 32, 64, 128, 24]))
    else:
        high = _spread(rng, 1, 8192 if qh <= 32 else 4096)
        total = 8192 if qh <= 32 else 4096
        prefix = rng.choice([0, 0, _spread(rng, 1, 4000)])
        if prefix:
            high = min(high, 700)
        case.update(sequences=_spread(rng, 1, max(1, min(64, total // (high + prefix)))), low=rng.randint(1, high),
                    high=high, prefix=prefix)
    return case


def _lengths(case):
    """The case's lengths: `high` once, the others even over the logarithm."""
    rng = random.Random("%s %s %s" % (case["sequences"], case["low"], case["high"]))
    return [case["high"]] + [_spread(rng, case["low"], case["high"]) for _ in range(case["sequences"] - 1)]


def _key_lengths(case):
    """Keys of each packed sequence: its own and a prefix computed before."""
    rng = random.Random("%s %s" % (case["sequences"], case["prefix"]))
    return [n + (rng.randint(case["prefix"] // 2, case["prefix"]) if case["prefix"] else 0) for n in _lengths(case)]


def _starts(lengths):
    return [sum(lengths[:i]) for i in range(len(lengths) + 1)]


def _pages(case, first, last, generator):
    """A page table [sequences, pages of the longest] for the positions
    [first, last) of each sequence, in shuffled physical pages; places outside
    of the positions name page 0. Returns it with the number of pages."""
    page = case["page"]
    spans = [(a // page, -(-b // page)) for a, b in zip(first, last)]
    count = sum(b - a for a, b in spans)
    order = torch.randperm(count, generator=generator).tolist()
    table, at = torch.zeros(len(spans), max(b for _, b in spans), dtype=torch.int32), 0
    for s, (a, b) in enumerate(spans):
        table[s, a:b] = torch.tensor(order[at:at + b - a], dtype=torch.int32)
        at += b - a
    return table, count


def _logits(rows, vocabulary, generator):
    """Logits as a head gives them: a wide bulk and a few likely tokens."""
    x = torch.randn(rows, vocabulary, generator=generator, device="cuda") * 2.2
    top = torch.randint(0, vocabulary, (rows, 24), generator=generator, device="cuda")
    return x.scatter_add_(1, top, torch.rand(rows, 24, generator=generator, device="cuda") * 12).half()


def prepare(case, seed):
    engine = _engine() if own else None  # its stream is the inputs' too
    host = torch.Generator().manual_seed(seed)
    device = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=device, device="cuda", dtype=torch.float16)

    def words(values):
        return torch.as_tensor(values, dtype=torch.int32).cuda()

    state = dict(case=case, op=case["op"])
    if case["op"] == "sample":
        rows = case["rows"]

        def pick(values):
            return torch.tensor(values)[torch.randint(0, len(values), (rows,), generator=host)].cuda()

        state.update(logits=_logits(rows, case["vocabulary"], device),
                     temperature=pick([0.6, 0.7, 1.0, 1.0, 1.3, 0.0]), top_p=pick([1.0, 0.95, 0.8]),
                     min_p=pick([0.0, 0.0, 0.05]), top_k=pick([0, 0, 20, 50]).int(),
                     uniform=torch.rand(rows, generator=host).cuda(),
                     tokens=torch.zeros(rows, dtype=torch.int32, device="cuda"))
    else:
        qh, kvh, hd, lengths = case["qh"], case["kvh"], case["hd"], _lengths(case)
        total = sum(lengths)
        if case["op"] == "packed":
            keys = _key_lengths(case)
            state.update(query=normal(total, qh, hd), key=normal(sum(keys), kvh, hd), value=normal(sum(keys), kvh, hd),
                         query_starts=words(_starts(lengths)), key_starts=words(_starts(keys)),
                         out=torch.zeros(total, qh, hd, dtype=torch.float16, device="cuda"))
        elif case["op"] == "decode":
            table, count = _pages(case, [0] * len(lengths), lengths, host)
            state.update(query=normal(len(lengths), qh, hd), key_cache=normal(count, case["page"], kvh, hd),
                         value_cache=normal(count, case["page"], kvh, hd), lengths=words(lengths), table=table.cuda(),
                         out=torch.zeros(len(lengths), qh, hd, dtype=torch.float16, device="cuda"))
        else:
            # positions before the offset belong to earlier steps: their pages
            # are not touched, so the cache holds only those that are
            first = [case["offset"] + 7 * s for s in range(len(lengths))] if case["offset"] else [0] * len(lengths)
            last = [a + n for a, n in zip(first, lengths)]
            table, count = _pages(case, first, last, host)
            state.update(query=normal(total, qh, hd), key=normal(total, kvh, hd), value=normal(total, kvh, hd),
                         query_weight=(1 + 0.1 * normal(hd)) if case["norm"] else None,
                         key_weight=(1 + 0.1 * normal(hd)) if case["norm"] else None,
                         starts=words(_starts(lengths)), lengths=words(last), table=table.cuda(),
                         key_cache=normal(count, case["page"], kvh, hd),
                         value_cache=normal(count, case["page"], kvh, hd),
                         query_out=torch.zeros(total, qh, hd, dtype=torch.float16, device="cuda"))
    if own:
        # what a program over the engine holds: its context, an open batch and
        # tensor handles over its device memory
        mi, context, *_ = state["engine"] = engine
        context.kernel_status()  # raises what the kernels of earlier passes refused
        kinds = {torch.float16: mi.DType.F16, torch.float32: mi.DType.F32, torch.int32: mi.DType.U32}
        state["handles"] = {k: context.tensor_from_device(t.data_ptr(), list(t.shape), kinds[t.dtype])
                            for k, t in state.items() if isinstance(t, torch.Tensor)}
    return state


_engines = {}  # by device


def _engine():
    """The engine on torch's current device, with its stream made torch's current
    one: what torch and the engine do then follows one another without a wait.
    (A caller that leaves it for another stream orders the two itself.)"""
    device = torch.cuda.current_device()
    if device not in _engines:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                        "metal-infer-rs_b200"))
        import metal_infer as mi
        context = mi.MetalContext(device)
        _engines[device] = (mi, context, context.begin_batch(), torch.cuda.ExternalStream(context.stream(), device))
    stream = _engines[device][3]
    if torch.cuda.current_stream() != stream:
        stream.wait_stream(torch.cuda.current_stream())
        torch.cuda.set_stream(stream)
    return _engines[device]


def run(state):
    return _run_own(state) if own else PLAIN[state["op"]](state)


def _run_own(state):
    case, h, batch = state["case"], state["handles"], state["engine"][2]
    if state["op"] == "sample":
        batch.sample(h["logits"], h["temperature"], h["top_k"], h["top_p"], h["min_p"], h["uniform"], h["tokens"])
        return state["tokens"]
    if state["op"] == "append":
        batch.paged_append(h["query"], h["key"], h["value"], h.get("query_weight"), h.get("key_weight"), h["starts"],
                           h["lengths"], h["table"], h["key_cache"], h["value_cache"], h["query_out"], THETA, EPSILON)
        return {k: state[k] for k in ("query_out", "key_cache", "value_cache")}
    if state["op"] == "decode":
        batch.paged_attention(h["query"], h["key_cache"], h["value_cache"], h["lengths"], h["table"], h["out"])
    else:
        batch.packed_attention(h["query"], h["key"], h["value"], h["query_starts"], h["key_starts"], True, h["out"])
    return state["out"]


# ---- plain forms ------------------------------------------------------------


def _softmax_products(scores, seen, value, equation):
    """Softmax over the last axis where `seen`, times the values; rows that
    see nothing are zero."""
    scores = scores.masked_fill(~seen, -math.inf)
    most = scores.amax(-1, keepdim=True)
    weights = (scores - most.masked_fill(most == -math.inf, 0.0)).exp()
    total = weights.sum(-1, keepdim=True)
    return torch.einsum(equation, weights / total.masked_fill(total == 0.0, 1.0), value)


def plain_decode(state):
    case = state["case"]
    count, qh, hd = state["query"].shape
    kvh = case["kvh"]
    table = state["table"].long()
    key = state["key_cache"][table].reshape(count, -1, kvh, hd).float()
    value = state["value_cache"][table].reshape(count, -1, kvh, hd).float()
    seen = torch.arange(key.shape[1], device="cuda")[None] < state["lengths"][:, None]
    value = value.masked_fill(~seen[:, :, None, None], 0.0)
    query = state["query"].float().reshape(count, kvh, qh // kvh, hd)
    scores = torch.einsum("skgd,sukd->skgu", query, key) * hd ** -0.5
    out = _softmax_products(scores, seen[:, None, None], value, "skgu,sukd->skgd")
    return out.reshape(count, qh, hd).half()


def plain_packed(state):
    total, qh, hd = state["query"].shape
    units, kvh, _ = state["key"].shape
    query_starts, key_starts = state["query_starts"], state["key_starts"]
    row = torch.arange(total, device="cuda", dtype=torch.int32)
    column = torch.arange(units, device="cuda", dtype=torch.int32)
    row_of = torch.bucketize(row, query_starts[1:], right=True)
    column_of = torch.bucketize(column, key_starts[1:], right=True)
    # counted from the ends of both: the last query sees the last key
    before = (query_starts[1:][row_of] - row)[:, None] <= (key_starts[1:][column_of] - column)[None]
    seen = (row_of[:, None] == column_of[None]) & before
    query = state["query"].float().reshape(total, kvh, qh // kvh, hd)
    scores = torch.einsum("tkgd,ukd->kgtu", query, state["key"].float()) * hd ** -0.5
    out = _softmax_products(scores, seen, state["value"].float(), "kgtu,ukd->tkgd")
    return out.reshape(total, qh, hd).half()


def _rotated(x, weight, position):
    """Per-head RMSNorm (with a weight) and rotation of the half pairs, in 32
    bits. Frequencies and angles are 32-bit values by the operator's
    definition; their cosines and sines are taken in 64."""
    hd = x.shape[-1]
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPSILON) * weight.float()
    exponent = -torch.arange(0, hd, 2, device="cuda", dtype=torch.float32) / hd
    frequency = torch.pow(torch.tensor(THETA, dtype=torch.float64, device="cuda"), exponent.double()).float()
    angle = (position.float()[:, None] * frequency).double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x[..., :hd // 2], x[..., hd // 2:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1).half()


def plain_append(state):
    starts, lengths = state["starts"].long(), state["lengths"].long()
    token = torch.arange(state["key"].shape[0], device="cuda")
    sequence = torch.bucketize(token, starts[1:], right=True)
    position = lengths[sequence] - starts[1:][sequence] + token
    page = state["case"]["page"]
    where = (state["table"].long()[sequence, position // page], position % page)
    state["key_cache"][where] = _rotated(state["key"], state["key_weight"], position)
    state["value_cache"][where] = state["value"]
    state["query_out"].copy_(_rotated(state["query"], state["query_weight"], position))
    return {k: state[k] for k in ("query_out", "key_cache", "value_cache")}


def _order(logits):
    """FP16 values as integers of the same order (-0 below +0)."""
    bits = logits.view(torch.int16).int()
    return torch.where(bits < 0, -(bits & 0x7FFF) - 1, bits)


def plain_sample(state):
    logits = state["logits"]
    order, index = torch.sort(_order(logits), dim=1, descending=True, stable=True)
    value = logits.gather(1, index).double()
    rank = torch.arange(value.shape[1], device="cuda")[None]
    temperature = state["temperature"].double()[:, None]
    weight = ((value - value[:, :1]) / temperature.masked_fill(temperature == 0.0, 1.0)).exp()
    top_k = state["top_k"][:, None]
    weight = weight.masked_fill((top_k > 0) & (rank >= top_k), 0.0)
    before = weight.cumsum(1) - weight
    top_p = state["top_p"].double()[:, None]
    kept = (top_p >= 1.0) | (before < top_p * weight.sum(1, keepdim=True))
    kept &= weight >= state["min_p"].double()[:, None]
    kept[:, 0] = True
    weight = weight * kept
    summed = weight.cumsum(1)
    place = (summed <= state["uniform"].double()[:, None] * summed[:, -1:]).sum(1)
    place = torch.minimum(place, (weight > 0.0).sum(1) - 1)
    place = place.masked_fill(state["temperature"] == 0.0, 0)
    return index.gather(1, place[:, None])[:, 0].int()


PLAIN = dict(append=plain_append, decode=plain_decode, packed=plain_packed, sample=plain_sample)


# ---- what a pass cannot do without ------------------------------------------


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocabulary"]
        return dict(bytes=2 * n + 24 * case["rows"], flops=2 * n)
    qh, kvh, hd, lengths = case["qh"], case["kvh"], case["hd"], _lengths(case)
    total = sum(lengths)
    if case["op"] == "append":
        return dict(bytes=2 * total * (qh + 2 * kvh) * hd * 2, flops=6 * total * (qh + kvh) * hd)
    if case["op"] == "decode":
        pages = sum(-(-n // case["page"]) for n in lengths)
        return dict(bytes=4 * total * kvh * hd + 4 * len(lengths) * qh * hd + 4 * pages, flops=4 * total * qh * hd)
    keys = _key_lengths(case)
    pairs = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(lengths, keys))
    return dict(bytes=4 * total * qh * hd + 4 * sum(keys) * kvh * hd, flops=4 * pairs * qh * hd)


# ---- the definitions in 64 bits ----------------------------------------------


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = kept
    return EXACT[case["op"]](case, state)


def _exact_rows(query, key, value, offset):
    """Attention of one sequence in 64 bits: query [t, qh, hd] at positions
    offset, offset + 1, ... over key / value [u, kvh, hd]."""
    t, qh, hd = query.shape
    u, kvh, _ = key.shape
    out = torch.zeros(t, qh, hd, dtype=torch.float64, device="cuda")
    for head in range(qh):
        k, v = key[:, head * kvh // qh].double(), value[:, head * kvh // qh].double()
        for a in range(0, t, 2048):
            s = query[a:a + 2048, head].double() @ k.T / math.sqrt(hd)
            places = torch.arange(a, min(t, a + 2048), device="cuda")[:, None] + offset
            s = torch.where(torch.arange(u, device="cuda")[None] <= places, s, -math.inf)
            out[a:a + 2048, head] = torch.softmax(s, -1) @ v
    return out


def exact_decode(case, state):
    out = []
    for s, n in enumerate(_lengths(case)):
        pages = state["table"][s, :-(-n // case["page"])].long()
        key, value = (state[c][pages].flatten(0, 1)[:n] for c in ("key_cache", "value_cache"))
        out.append(_exact_rows(state["query"][s:s + 1], key, value, n - 1))
    return torch.cat(out)


def exact_packed(case, state):
    out, at, from_ = [], 0, 0
    for n, m in zip(_lengths(case), _key_lengths(case)):
        out.append(_exact_rows(state["query"][at:at + n], state["key"][from_:from_ + m],
                               state["value"][from_:from_ + m], m - n))
        at, from_ = at + n, from_ + m
    return torch.cat(out)


def exact_append(case, state):
    hd = case["hd"]
    frequency = np.array([np.float32(THETA ** float(np.float32(-i) / np.float32(hd))) for i in range(0, hd, 2)])

    def turned(x, weight, positions):
        x = x.double()
        if weight is not None:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / hd + EPSILON) * weight.double()
        angle = torch.from_numpy((positions.astype(np.float32)[:, None] * frequency).astype(np.float64)).cuda()
        z = torch.complex(x[..., :hd // 2].contiguous(), x[..., hd // 2:].contiguous())
        z = z * torch.polar(torch.ones_like(angle), angle)[:, None]
        return torch.cat([z.real, z.imag], -1)

    caches = {c: state[c].double() for c in ("key_cache", "value_cache")}
    query, at = [], 0
    for s, n in enumerate(_lengths(case)):
        first = int(state["lengths"][s]) - n
        positions = np.arange(first, first + n)
        slots = (state["table"][s].long()[torch.from_numpy(positions // case["page"]).cuda()],
                 torch.from_numpy(positions % case["page"]).cuda())
        caches["key_cache"][slots] = turned(state["key"][at:at + n], state["key_weight"], positions)
        caches["value_cache"][slots] = state["value"][at:at + n].double()
        query.append(turned(state["query"][at:at + n], state["query_weight"], positions))
        at += n
    return dict(query_out=torch.cat(query), **caches)


def exact_sample(case, state):
    tokens = []
    rows = {k: state[k].cpu().numpy() for k in ("logits", "temperature", "top_k", "top_p", "min_p", "uniform")}
    for r in range(case["rows"]):
        bits = rows["logits"][r].view(np.uint16).astype(np.int64)
        key = np.where(bits & 0x8000, 0xFFFF - bits, bits | 0x8000)
        order = np.lexsort((np.arange(key.size), -key))
        if rows["top_k"][r]:
            order = order[:rows["top_k"][r]]
        if rows["temperature"][r] == 0:
            tokens.append(int(order[0]))
            continue
        v = rows["logits"][r][order].astype(np.longdouble)
        w = np.exp((v - v[0]) / np.longdouble(rows["temperature"][r]))
        ends = np.cumsum(w)
        keep = max(1, int(np.sum(w >= rows["min_p"][r])))
        if rows["top_p"][r] < 1:
            keep = min(keep, int(np.searchsorted(ends, np.longdouble(rows["top_p"][r]) * ends[-1], "left")) + 1)
        ends = ends[:keep]
        place = int(np.searchsorted(ends, np.longdouble(rows["uniform"][r]) * ends[-1], "right"))
        tokens.append(int(order[min(place, keep - 1)]))
    return torch.tensor(tokens, dtype=torch.int32)


EXACT = dict(append=exact_append, decode=exact_decode, packed=exact_packed, sample=exact_sample)
