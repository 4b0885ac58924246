"""A decoder's operators: the cache (written, read back, shared between executors), attention that reads it, sampling of tokens.
Against plain implementations in 64 bits; what holds whole numbers has to be the same."""
import ctypes
import math

import numpy as np
import pytest

from kyanite_b200 import _lib
from kyanite_b200.executor import CudaExecutor, KnError, KvCache, plan_describe
from kyanite_b200.graph import BATCH, DType, Graph, OpKind, shape
from kyanite_b200.optimizer import optimize_graph

I8, F16, F32, I32 = DType.I8, DType.F16, DType.F32, DType.I32


# ------------------------------------------------------------------------------------------------ plain forms


def quantise(x):
    """(q, scale) of rows: scale = max|x| * (1/127) and q = round(x / scale), in f32 as IEEE has them"""
    x = x.astype(np.float32)
    scale = (np.abs(x).max(-1, keepdims=True) * (np.float32(1) / np.float32(127))).astype(np.float32)
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.where(scale > 0, np.clip(np.rint(x / scale), -127, 127), 0)
    return q, scale


class PlainCache:
    """[2][sequences][heads][capacity][dim], as the numbers that it stands for"""

    def __init__(self, sequences, heads, capacity, dim, dtype):
        self.dtype, self.capacity = dtype, capacity
        self.held = np.zeros((2, sequences, heads, capacity, dim), np.float32)

    def write(self, keys, values, start, count=None):
        for part, x in enumerate((keys, values)):
            if self.dtype == I8:
                q, scale = quantise(x)
                with np.errstate(invalid="ignore"):
                    x = q.astype(np.float32) * scale
            else:
                with np.errstate(over="ignore"):
                    x = x.astype(np.float16).astype(np.float32)
            for s in range(x.shape[0]):
                for t in range(x.shape[1] if count is None else min(count[s], x.shape[1])):
                    if 0 <= start[s] + t < self.capacity:
                        self.held[part, s, :, start[s] + t] = x[s, t]


def plain_attention(q, held, start, count=None, scale=None, softcap=0.0, window=0, slopes=None, prefix=None, prefix_length=0):
    """(result, largest |value| that a row sees, largest sum of |scale q k|) in 64 bits"""
    n, tokens, heads, dim = q.shape
    start = [int(x) for x in start]
    group = heads // held.shape[2]
    scale = float(np.float32(1 / math.sqrt(dim) if scale is None else scale))
    out, size, sums = np.zeros(q.shape), np.zeros(q.shape[:3]), np.zeros(q.shape[:3])
    for s in range(n):
        for t in range(tokens):
            if start[s] + t < 0 or (count is not None and t >= count[s]):
                continue
            shared = 0 if prefix is None else min(max(prefix_length, 0), prefix.shape[3])
            p = shared + start[s] + t
            end = min(p + 1, shared + held.shape[3])
            first = max(0, p - window + 1) if window else 0
            if first >= end:
                continue
            for h in range(heads):
                both = held[:, s, h // group, :end - shared] if shared < end else held[:, s, h // group, :0]
                if prefix is not None:
                    both = np.concatenate([prefix[:, 0, h // group, :min(shared, end)], both], 1)
                k, v = both[:, first:end].astype(np.float64)
                x = scale * (k @ q[s, t, h].astype(np.float64))
                if softcap:
                    x = softcap * np.tanh(x / softcap)
                if slopes is not None:
                    x = x - float(slopes[h]) * (p - np.arange(first, end))
                e = np.exp(x - x.max())
                out[s, t, h] = (e[:, None] * v).sum(0) / e.sum()
                size[s, t, h], sums[s, t, h] = np.abs(v).max(), abs(scale) * (np.abs(k) @ np.abs(q[s, t, h].astype(np.float64))).max()
    return out, size, sums


def attention_tolerance(dtype, size, sums, keys):
    """Per row.  Scores are off by at most (2^-22, of q in two halves of 11 bits, + 2^-21, of sums of up to 256 products that are
    themselves sums of 16, and of cap, slope and exponent) of sum |q k|; a relative error of the weights twice that, of which
    the result has as much of the largest value.  Weights: 2^-11 of each in f16, 2^-22 in two halves (f32); sums of weights
    and results: a step of 2^-24 for each 16 keys.  The result's own rounding: 2^-11 (f16), 2^-24."""
    score = 2 * sums * (2.0 ** -22 + 2.0 ** -21) + 2.0 ** -20
    weights = 2.0 ** -11 if dtype == F16 else 2.0 ** -22
    return size * (score + weights + (keys / 16 + 16) * 2.0 ** -24 + (2.0 ** -11 if dtype == F16 else 2.0 ** -24)) + 1e-30


def plain_sample(logits, uniform, temperature=None, top_k=None, top_p=None, min_p=None):
    """Weights in whole steps of 2^-44, as whole numbers without limit"""
    out = []
    for r, row in enumerate(logits.astype(np.float64)):
        row = np.where(np.isnan(row), -np.inf, row)
        most, t = row.max(), 1.0 if temperature is None else float(temperature[r])
        if most == -np.inf or not t > 0:
            out.append(-1 if most == -np.inf else int(np.argmax(row)))
            continue
        with np.errstate(invalid="ignore"):
            z = np.where(row == most, 0.0, (row - most) / t)
        weight = [int(w) for w in np.rint(np.exp(z) * 2.0 ** 44)]
        order = [int(i) for i in np.argsort(-row, kind="stable")]
        if top_k is not None and top_k[r] > 0:
            order = order[:top_k[r]]
        if top_p is not None and not top_p[r] >= 1:
            goal, mass, kept = float(top_p[r]) * float(sum(weight[i] for i in order)), 0, []
            for i in order:
                kept.append(i)
                mass += weight[i]
                if mass >= goal:
                    break
            order = kept
        if min_p is not None:
            order = order[:1] + [i for i in order[1:] if weight[i] >= float(min_p[r]) * 2.0 ** 44]
        goal, mass, token = float(uniform[r]) * float(sum(weight[i] for i in order)), 0, -1
        for i in sorted(order):
            mass += weight[i]
            token = i
            if mass > goal:
                break
        out.append(token)
    return np.array(out, np.int32)


# ------------------------------------------------------------------------------------------------ graphs, host only


def attention_graph(sequences=2, tokens=1, heads=4, kv_heads=2, dim=64, capacity=40, dtype=F16, storage=I8, count=False, slopes=False, prefix=0, **more):
    g = Graph()
    cache = g.cache(sequences, kv_heads, capacity, dim, storage)
    q = g.input((sequences, tokens, heads, dim), dtype)
    start = g.input((sequences,), I32)
    n = g.input((sequences,), I32) if count else None
    slope = g.input((heads,)) if slopes else None
    if prefix:
        more.update(prefix=g.cache(1, kv_heads, prefix, dim, storage), prefix_length=g.input((1,), I32))
    g.output(g.cache_attention(q, cache, start, n, slopes=slope, **more))
    return g


def test_builder_refuses():
    g = Graph()
    cache, other = g.cache(2, 3, 10, 64), g.cache(2, 3, 10, 64)
    assert cache != other and g[cache].dtype == I8
    k = g.input((2, 5, 3, 64), F16)
    start = g.input((2,), I32)
    for bad in (lambda: g.cache(2, 0, 10, 64), lambda: g.cache(2, 3, 0, 64), lambda: g.cache(2, 3, 10, 257), lambda: g.cache(2, 3, 10, 64, F32),
                lambda: g.output(cache), lambda: g.view(cache, (2 * 2 * 3 * 10 * 64,)), lambda: g.slice(cache, 3, (0, 1)), lambda: g.add(cache, cache),
                lambda: g.cache_write(k, k, k, start), lambda: g.cache_write(cache, k, g.input((2, 5, 3, 32), F16), start),
                lambda: g.cache_write(cache, k, g.input((2, 5, 3, 64)), start), lambda: g.cache_write(cache, k, k, g.input((2,))),
                lambda: g.cache_write(cache, k, k, g.input((3,), I32)), lambda: g.cache_write(cache, k, k, start, g.input((1,), I32)),
                lambda: g.cache_write(cache, k, k, start, k), lambda: g.cache_read(cache, I8), lambda: g.cache_read(k),
                lambda: g.cache_attention(k, k, start), lambda: g.cache_attention(g.input((2, 5, 4, 64), F16), cache, start),
                lambda: g.cache_attention(g.input((2, 5, 3, 32), F16), cache, start), lambda: g.cache_attention(k, cache, k),
                lambda: g.cache_attention(k, cache, start, softcap=-1.0), lambda: g.cache_attention(k, cache, start, window=-1),
                lambda: g.cache_attention(k, cache, start, scale=math.inf), lambda: g.cache_attention(k, cache, start, slopes=g.input((2,))),
                lambda: g.cache_attention(k, cache, start, prefix=other), lambda: g.cache_attention(k, cache, start, prefix=other, prefix_length=g.input((1,), I32)),
                lambda: g.cache_attention(k, cache, start, prefix=g.cache(1, 3, 8, 64, F16), prefix_length=g.input((1,), I32)),
                lambda: g.sample(k, start), lambda: g.sample(g.input((2, 7), I32), g.input((2,))), lambda: g.sample(g.input((2, 7)), start),
                lambda: g.sample(g.input((2, 7)), g.input((3,))), lambda: g.sample(g.input((2, 7)), g.input((2,)), top_k=g.input((2,))),
                lambda: g.sample(g.input((2, (1 << 19) + 1)), g.input((2,)))):
        with pytest.raises(ValueError):
            bad()


def test_a_written_cache_has_no_other_user():
    g = Graph()
    cache, read = g.cache(2, 3, 10, 64), g.cache(2, 3, 10, 64)
    k, start = g.input((2, 5, 3, 64), F16), g.input((2,), I32)
    written = g.cache_write(cache, k, k, start)
    assert g.cache_write(cache, k, k, start) == written          # the same value
    again = g.cache_write(written, k, k, start, start)           # a second write behind the first
    g.output(g.cache_read(again))
    for bad in (lambda: g.cache_read(cache), lambda: g.cache_attention(k, written, start), lambda: g.cache_write(cache, k, k, start, start)):
        with pytest.raises(ValueError):
            bad()
    g.cache_read(read)
    with pytest.raises(ValueError):
        g.cache_write(read, k, k, start)
    assert "cachewrite" in plan_describe(g, 1)


def test_plan_of_a_decoder_step():
    """Writes are planned whether or not an output depends on them, before what reads what they return, and keep the caches' order."""
    g = Graph()
    one, two = g.cache(BATCH, 2, 100, 64), g.cache(BATCH, 2, 100, 64, F16)
    x, start = g.input(shape(BATCH, 1, 2, 64)), g.input(shape(BATCH), I32)
    g.cache_write(two, x, x, start)
    y = g.cache_attention(x, g.cache_write(one, x, x, start), start)
    g.output(g.sample(g.view(y, shape(BATCH, 128)), g.input(shape(BATCH))))
    for graph in (g, optimize_graph(g)):
        text = plan_describe(graph, 3)
        steps = [line.split()[2] for line in text.splitlines() if line.startswith("step")]
        assert sorted(steps) == ["CacheAttention", "CacheWrite", "CacheWrite", "Sample"]
        assert steps.index("CacheWrite") < steps.index("CacheAttention") < steps.index("Sample")
        assert [tuple(d.eval(3) for d in graph[c].shape) for c in graph.caches] == [(2, 3, 2, 100, 64)] * 2
        assert [graph[c].dtype for c in graph.caches] == [I8, F16]
    outer = Graph()
    args = [outer.input(g[v].shape, g[v].dtype) for v in g.inputs]
    first, second = outer.call(g, args), outer.call(g, args)
    assert len(outer.caches) == 4 and first != second
    assert plan_describe(outer, 2).count("CacheWrite") == 4


def test_blobs_are_checked():
    lib = _lib.load()

    def status(blob):
        out = ctypes.c_void_p()
        r = lib.kn_graph_from_blob(blob, len(blob), ctypes.byref(out))
        if r == 0:
            lib.kn_graph_destroy(out)
        return r

    g = attention_graph(count=True, slopes=True, prefix=5, softcap=20.0, window=7)
    good = g.to_bytes()
    assert status(good) == 0
    for cut in range(16, len(good), 7):
        assert status(good[:cut]) == 2
    at = good.rindex(np.float32(20.0).tobytes())
    assert status(good[:at] + np.float32(math.nan).tobytes() + good[at + 4:]) == 2
    assert status(good[:at] + np.float32(-1.0).tobytes() + good[at + 4:]) == 2
    # the attention's operands are seven numbers in front of scale and softcap: query, cache, start, count, slopes, prefix, its length
    def with_operand(k, v):
        p = at - 4 - 4 * 7 + 4 * k
        return good[:p] + np.uint32(v).tobytes() + good[p + 4:]
    query, cache = g.inputs[0].index, g.caches[0].index
    assert status(with_operand(1, cache)) == 0
    for k, v in ((0, cache), (1, query), (2, cache), (3, cache), (5, query), (6, 0xFFFFFFFF), (5, 0xFFFFFFFF), (0, 10 ** 6), (0, 0xFFFFFFFF)):
        assert status(with_operand(k, v)) == 2, (k, v)
    # shapes are checked when the batch is known
    q = Graph()
    c = q.cache(BATCH, 2, 10, 64)
    x = q.input((4, 1, 2, 64))
    with pytest.raises(ValueError):
        q.cache_attention(x, c, q.input(shape(BATCH), I32))
    w = Graph()
    c = w.cache(2, 2, 10, 64)
    k, start = w.input((2, 3, 2, 64)), w.input((2,), I32)
    w.output(w.cache_read(w.cache_write(c, k, k, start)))
    blob = w.to_bytes()
    size = np.array([2], "<u8").tobytes()
    at = blob.index(size, 20 + 4)                                 # the cache's first axis: not 2 parts
    with pytest.raises(KnError):
        plan_describe(blob[:at] + np.array([3], "<u8").tobytes() + blob[at + 8:], 1)


def test_optional_operands_keep_their_places():
    for flags in range(16):
        g = Graph()
        logits, uniform = g.input((3, 9)), g.input((3,))
        given = [g.input((3,), I32 if i == 1 else F32) if flags >> i & 1 else None for i in range(4)]
        g.output(g.sample(logits, uniform, *given))
        assert g[g.outputs[0]].present == tuple(v is not None for v in given)
        assert plan_describe(g, 1).count("r:") == 2 + bin(flags).count("1")


# ------------------------------------------------------------------------------------------------ on the GPU: the cache


def numbers(seed, *dims, dtype=F16):
    x = np.random.default_rng(seed).standard_normal(dims) * np.exp(0.5 * np.random.default_rng(seed + 1).standard_normal(dims[-1:]))
    return x.astype(dtype.np)


def filled(sequences, heads, capacity, dim, storage, seed, lengths=None):
    """(KvCache, PlainCache) that hold the same `lengths` positions"""
    cache, plain = KvCache(0, sequences, heads, capacity, dim, storage), PlainCache(sequences, heads, capacity, dim, storage)
    g = Graph()
    c = g.cache(sequences, heads, capacity, dim, storage)
    k, v = (g.input((sequences, capacity, heads, dim), F16) for _ in range(2))
    g.cache_write(c, k, v, g.constant((sequences,), np.zeros(sequences), I32), g.input((sequences,), I32))
    with CudaExecutor(0, g, 1) as ex:
        ex.set_cache(0, cache)
        keys, values = (numbers(seed + i, sequences, capacity, heads, dim) for i in range(2))
        n = np.full(sequences, capacity, np.int32) if lengths is None else np.array(lengths, np.int32)
        ex.evaluate([keys, values, n])
    plain.write(keys, values, np.zeros(sequences, int), n)
    return cache, plain


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [1, 20, 64, 80, 100, 128, 192, 200, 256])
@pytest.mark.parametrize("storage, dtype, out", [(I8, F16, F32), (I8, F32, F16), (F16, F32, F32), (F16, F16, F16)])
def test_cache_write_and_read(dim, storage, dtype, out):
    sequences, heads, capacity, tokens = 5, 3, 37, 9
    cache, plain = KvCache(0, sequences, heads, capacity, dim, storage), PlainCache(sequences, heads, capacity, dim, storage)
    g = Graph()
    c = g.cache(sequences, heads, capacity, dim, storage)
    k, v = (g.input((sequences, tokens, heads, dim), dtype) for _ in range(2))
    g.output(g.cache_read(g.cache_write(c, k, v, g.input((sequences,), I32), g.input((sequences,), I32)), out))
    with CudaExecutor(0, g, 1) as ex:
        ex.set_cache(0, cache)
        # in front of the cache, over its end, far outside, nothing, more than there are; then once more over part of it
        for seed, start, count in ((1, [0, -4, 33, 10, 20], [9, 9, 9, 0, 100]), (2, [5, 2 ** 31 - 1, -2 ** 31, 36, 22], [3, 9, 9, 9, -1])):
            keys, values = numbers(seed, sequences, tokens, heads, dim, dtype=dtype), numbers(seed + 50, sequences, tokens, heads, dim, dtype=dtype)
            keys[0, 0] = 0
            got = ex.evaluate([keys, values, np.array(start, np.int32), np.array(count, np.int32)])[0]
            plain.write(keys, values, start, count)
            assert np.array_equal(got, plain.held.astype(out.np))


@pytest.mark.gpu
@pytest.mark.parametrize("storage", [I8, F16])
def test_cache_write_takes_any_strides(storage):
    """Keys as a slice of a wider matrix with the heads in front, values as one row for all tokens"""
    sequences, heads, capacity, tokens, dim = 2, 3, 20, 7, 40
    g = Graph()
    c = g.cache(sequences, heads, capacity, dim, storage)
    wide = g.input((sequences, heads, tokens, 2 * dim + 1))
    k = g.permute(g.slice(wide, 3, (1, dim + 1)), [0, 2, 1, 3])
    row = g.input((sequences, 1, heads, dim))
    v = g.flip(g.broadcast(row, (sequences, tokens, heads, dim)), 3)
    start = g.input((sequences, 2), I32)
    g.output(g.cache_read(g.cache_write(c, k, v, g.index(start, 1, 1)), F32))
    a, b, s = numbers(3, sequences, heads, tokens, 2 * dim + 1, dtype=F32), numbers(4, sequences, 1, heads, dim, dtype=F32), np.array([[9, 2], [9, 13]], np.int32)
    plain = PlainCache(sequences, heads, capacity, dim, storage)
    with CudaExecutor(0, g, 1) as ex:
        ex.set_cache(0, KvCache(0, sequences, heads, capacity, dim, storage))
        got = ex.evaluate([a, b, s])[0]
    plain.write(a[..., 1:dim + 1].transpose(0, 2, 1, 3), np.broadcast_to(b[..., ::-1], (sequences, tokens, heads, dim)), s[:, 1])
    assert np.array_equal(got, plain.held)


@pytest.mark.gpu
def test_cache_of_numbers_at_the_ends():
    """Rows next to nothing, of the largest numbers, and with infinities or NaN, which read back as NaN throughout"""
    g = Graph()
    c = g.cache(1, 1, 6, 64)
    k = g.input((1, 6, 1, 64))
    g.output(g.cache_read(g.cache_write(c, k, k, g.input((1,), I32)), F32))
    x = numbers(5, 1, 6, 1, 64, dtype=F32)
    x[0, 1] *= np.float32(1e-44)
    x[0, 2] = x[0, 2] / np.abs(x[0, 2]).max() * np.float32(3.4e38)
    x[0, 3, 0, 7], x[0, 4, 0, 9] = np.inf, np.nan
    x[0, 5] = 0
    with CudaExecutor(0, g, 1) as ex:
        ex.set_cache(0, KvCache(0, 1, 1, 6, 64))
        got = ex.evaluate([x, np.zeros(1, np.int32)])[0]
    q, scale = quantise(x[0, :, 0])
    for part in got[:, 0, 0]:
        for t in (0, 1, 2, 5):
            assert np.array_equal(part[t], (q[t] * scale[t]).astype(np.float32)), t
        assert np.isnan(part[3]).all() and np.isnan(part[4]).all()


# ------------------------------------------------------------------------------------------------ on the GPU: attention


def attend(ex_graph, caches, inputs):
    with CudaExecutor(0, ex_graph, 1) as ex:
        for i, c in enumerate(caches):
            ex.set_cache(i, c)
        first = ex.evaluate(inputs)[0]
        for _ in range(2):                       # nothing is left behind from one launch to the next
            assert np.array_equal(ex.evaluate(inputs)[0], first, equal_nan=True)
    return first


def check_attention(sequences, tokens, heads, kv_heads, dim, capacity, start, dtype=F16, storage=I8, count=None, slopes=False, prefix=0, prefix_length=None, seed=1, **more):
    start = np.array(start, np.int32)
    cache, plain = filled(sequences, kv_heads, capacity, dim, storage, seed)
    caches, held_prefix = [cache], None
    q = (1.5 * numbers(seed + 9, sequences, tokens, heads, dim, dtype=F32)).astype(dtype.np)
    g = attention_graph(sequences, tokens, heads, kv_heads, dim, capacity, dtype, storage, count is not None, slopes, prefix, **more)
    inputs, plain_more = [q, start], dict(more)
    if count is not None:
        inputs.append(np.array(count, np.int32))
    if slopes:
        plain_more["slopes"] = (0.5 ** np.arange(1, heads + 1)).astype(np.float32)
        inputs.append(plain_more["slopes"])
    if prefix:
        shared, held_prefix = filled(1, kv_heads, prefix, dim, storage, seed + 20)
        caches.append(shared)
        prefix_length = prefix if prefix_length is None else prefix_length
        plain_more.update(prefix=held_prefix.held, prefix_length=prefix_length)
        inputs.append(np.array([prefix_length], np.int32))
    got = attend(g, caches, inputs).astype(np.float64)
    want, size, sums = plain_attention(q, plain.held, start, count, **plain_more)
    off = np.abs(got - want).max(-1)
    allowed = attention_tolerance(dtype, size, sums, capacity + prefix)
    assert np.isfinite(got).all()
    assert (off <= allowed).all(), (float((off / allowed).max()), np.argwhere(off > allowed)[:5])
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, storage", [(F16, I8), (F16, F16), (F32, I8), (F32, F16)])
@pytest.mark.parametrize("dim", [1, 24, 64, 80, 128, 192, 256])
def test_attention_types_and_dims(dtype, storage, dim):
    check_attention(3, 1, 4, 2, dim, 150, [149, 0, 70], dtype, storage)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("heads, kv_heads, tokens", [(1, 1, 1), (8, 8, 1), (8, 1, 1), (9, 1, 1), (14, 2, 1), (32, 2, 1), (20, 1, 3), (6, 2, 17), (4, 4, 40), (5, 5, 130)])
def test_attention_rows(dtype, heads, kv_heads, tokens):
    check_attention(2, tokens, heads, kv_heads, 64, 200, [200 - tokens, 3], dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("storage", [I8, F16])
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 127, 128, 129, 1000, 4099])
def test_attention_lengths(storage, length):
    check_attention(2, 1, 4, 2, 128, length, [length - 1, length // 2], F16, storage)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("more", [dict(softcap=5.0), dict(window=1), dict(window=17), dict(window=1000), dict(slopes=True), dict(scale=0.0), dict(scale=-0.4),
                                  dict(softcap=30.0, window=40, slopes=True)], ids=str)
def test_attention_scores(dtype, more):
    check_attention(3, 3, 6, 2, 64, 120, [117, 20, 0], dtype, **more)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("prefix, length, own, tokens, more", [
    (100, None, [49, 0, 20], 1, {}), (100, 33, [49, 0, 20], 2, {}), (100, 0, [49, 0, 20], 1, {}), (1, None, [49, 0, 20], 1, {}), (700, 513, [40, 1, 2], 5, {}),
    (100, None, [49, 0, 20], 2, dict(window=30)), (100, None, [49, 3, 20], 1, dict(window=1, slopes=True)), (64, 10 ** 6, [49, 0, 20], 1, dict(softcap=9.0)),
    (64, -5, [49, 0, 20], 1, {})])
def test_attention_with_a_shared_prefix(dtype, prefix, length, own, tokens, more):
    check_attention(3, tokens, 8, 2, 64, 60, own, dtype, prefix=prefix, prefix_length=length, **more)


def plan_says(text, **sizes):
    return text in plan_describe(attention_graph(**sizes), 1)


def test_which_rows_are_taken_128_at_a_time():
    assert plan_says(", 128 rows at a time", tokens=32, heads=4, kv_heads=2)
    assert not plan_says("rows at a time", tokens=31, heads=4, kv_heads=2)
    for no in (dict(dtype=F32), dict(storage=F16), dict(dim=136)):
        assert not plan_says("rows at a time", tokens=100, heads=4, kv_heads=2, **no)
    # of a prefix: 64 rows of all sequences, and 2^20 positions read by 16 rows at a time
    assert plan_says("the prefix 128 rows at a time", sequences=32, prefix=2 ** 14)
    assert not plan_says("rows at a time", sequences=31, prefix=2 ** 15) and not plan_says("rows at a time", sequences=32, prefix=2 ** 14 - 1)
    assert plan_says("the prefix 128 rows at a time", sequences=32, tokens=9, prefix=2 ** 13) and not plan_says("rows at a time", sequences=32, tokens=8, prefix=2 ** 13)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [20, 64, 100, 128])
@pytest.mark.parametrize("sequences, heads, kv_heads, tokens, capacity, start", [
    (2, 4, 2, 32, 40, [8, 0]), (1, 1, 1, 128, 128, [0]), (1, 1, 1, 129, 200, [60]), (2, 8, 2, 70, 700, [600, 33]), (1, 2, 1, 300, 2100, [1790]), (3, 7, 1, 40, 64, [24, 0, 11])])
def test_attention_of_many_rows(dim, sequences, heads, kv_heads, tokens, capacity, start):
    assert plan_says(", 128 rows at a time", sequences=sequences, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, capacity=capacity)
    check_attention(sequences, tokens, heads, kv_heads, dim, capacity, start)


@pytest.mark.gpu
@pytest.mark.parametrize("more", [dict(softcap=5.0), dict(window=1), dict(window=70), dict(slopes=True), dict(softcap=30.0, window=200, slopes=True), dict(prefix=90, prefix_length=77),
                                  dict(prefix=500, window=130), dict(prefix=64, softcap=20.0, slopes=True), dict(prefix=300, prefix_length=0), dict(scale=-0.3)], ids=str)
def test_attention_scores_of_many_rows(more):
    check_attention(2, 80, 4, 2, 64, 450, [370, 9], **more)


@pytest.mark.gpu
def test_attention_of_padded_many_rows():
    got = check_attention(6, 70, 4, 2, 64, 100, [5, -30, 60, -90, 2 ** 31 - 1, -2 ** 31], count=[40, 70, 70, 70, 70, 70])
    assert (got[0, 40:] == 0).all() and (got[1, :30] == 0).all() and (got[3] == 0).all() and (got[5] == 0).all()
    got = check_attention(2, 66, 4, 2, 64, 100, [150, 33], window=20)
    assert (got[0] == 0).all() and (got[1] != 0).any(-1).all()
    check_attention(3, 64, 2, 1, 128, 64, [0, 0, 0], count=[0, -3, 100])


@pytest.mark.gpu
@pytest.mark.parametrize("what", [np.inf, np.nan])
def test_hidden_positions_of_many_rows_may_hold_anything(what):
    heads, dim, capacity, tokens = 2, 64, 200, 64
    cache, plain = filled(1, heads, capacity, dim, I8, 1)
    g = Graph()
    c = g.cache(1, heads, capacity, dim, I8)
    k, start = g.input((1, 1, heads, dim)), g.input((1,), I32)
    g.cache_write(c, k, k, start)
    bad = np.full((1, 1, heads, dim), what, np.float32)
    with CudaExecutor(0, g, 1) as ex:
        ex.set_cache(0, cache)
        for at in (170, 199, 20, 163):       # behind the end, in front of the window, the last new token
            ex.evaluate([bad, np.array([at], np.int32)])
    q = numbers(9, 1, tokens, heads, dim)
    got = attend(attention_graph(1, tokens, heads, heads, dim, capacity, F16, I8, window=60), [cache], [q, np.array([100], np.int32)]).astype(np.float64)
    want, size, sums = plain_attention(q[:, :63], plain.held, [100], window=60)
    assert (np.abs(got[:, :63] - want).max(-1) <= attention_tolerance(F16, size, sums, capacity)).all()
    assert np.isnan(got[:, 63]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("sequences, heads, kv_heads, dim, tokens, prefix, length, more", [
    (40, 8, 2, 128, 1, 1000, None, {}), (70, 4, 4, 64, 1, 256, 100, {}), (9, 8, 1, 100, 2, 300, 0, {}), (33, 4, 1, 128, 1, 4000, 3999, dict(window=300)),
    (16, 16, 2, 64, 3, 700, 650, dict(slopes=True, softcap=15.0)), (70, 8, 1, 64, 1, 512, 512, {})])
def test_prefix_of_all_sequences_at_once(sequences, heads, kv_heads, dim, tokens, prefix, length, more):
    start = [(7 * s) % (60 - tokens) for s in range(sequences)]
    start[1], start[2] = -1, -9                                     # sequences that see nothing (of their own, or at all)
    check_attention(sequences, tokens, heads, kv_heads, dim, 60, start, prefix=prefix, prefix_length=length, count=[tokens] * (sequences - 1) + [0], **more)


@pytest.mark.gpu
@pytest.mark.parametrize("sequences, heads, kv_heads, dim, tokens, prefix, length, more", [
    (40, 8, 2, 128, 1, 13200, 1000, {}), (70, 4, 4, 64, 1, 3800, 100, {}), (70, 4, 4, 64, 1, 3800, None, {}), (9, 8, 1, 100, 2, 117000, 0, {}),
    (33, 4, 1, 128, 1, 32000, 3999, dict(window=300)), (16, 16, 2, 64, 3, 17000, 650, dict(slopes=True, softcap=15.0)), (70, 8, 1, 64, 1, 15000, 512, {})])
def test_long_prefix_of_all_sequences_at_once(sequences, heads, kv_heads, dim, tokens, prefix, length, more):
    sizes = dict(sequences=sequences, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, capacity=60, prefix=prefix)
    assert plan_says("the prefix 128 rows at a time", **sizes)
    start = [(7 * s) % (60 - tokens) for s in range(sequences)]
    start[1], start[2] = -1, -9
    check_attention(sequences, tokens, heads, kv_heads, dim, 60, start, prefix=prefix, prefix_length=length, count=[tokens] * (sequences - 1) + [0], **more)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, F32])
def test_attention_of_padded_and_empty_rows(dtype):
    """Padded tokens, sequences in front of position 0 (partly), beyond the capacity (what is there is seen), far outside"""
    got = check_attention(6, 4, 4, 2, 64, 30, [5, -2, 28, -9, 2 ** 31 - 1, -2 ** 31], dtype, count=[2, 4, 4, 4, 4, 4])
    assert (got[0, 2:] == 0).all() and (got[1, :2] == 0).all() and (got[3] == 0).all() and (got[5] == 0).all()
    assert (got[0, :2] != 0).any(-1).all() and (got[1, 2:] != 0).any(-1).all()
    got = check_attention(2, 2, 4, 2, 64, 30, [100, 29], dtype, window=20)      # a window behind the capacity: nothing is left in it
    assert (got[0] == 0).all() and (got[1] != 0).any(-1).all()
    check_attention(3, 2, 2, 2, 64, 10, [4, 5, 6], dtype, count=[0, -3, 100])


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [[3000, 1, 17, 900, 128, 64, 2047], [1] * 300, [40] * 37 + [2500]], ids=str)
def test_attention_of_ragged_batches(lengths):
    check_attention(len(lengths), 1, 4, 1, 64, max(lengths), [n - 1 for n in lengths], F16)
    check_attention(len(lengths), 1, 4, 1, 64, max(lengths), [n - 1 for n in lengths], F32, F16)


@pytest.mark.gpu
@pytest.mark.parametrize("storage", [I8, F16])
@pytest.mark.parametrize("what", [np.inf, np.nan])
def test_hidden_positions_may_hold_anything(storage, what):
    """Behind a sequence's end, in front of a window, and among the new tokens themselves"""
    sequences, heads, dim, capacity, tokens = 2, 2, 64, 50, 3
    cache, plain = filled(sequences, heads, capacity, dim, storage, 1)
    g = Graph()
    c = g.cache(sequences, heads, capacity, dim, storage)
    k, start = g.input((sequences, 1, heads, dim)), g.input((sequences,), I32)
    g.cache_write(c, k, k, start)
    bad = np.full((sequences, 1, heads, dim), what, np.float32)
    with CudaExecutor(0, g, 1) as ex:
        ex.set_cache(0, cache)
        for at in ([40, 24], [41, 25], [3, 1], [39, 23]):       # behind the end, in front of the window, the last new token
            ex.evaluate([bad, np.array(at, np.int32)])
    g = attention_graph(sequences, tokens, heads, heads, dim, capacity, F16, storage, window=20)
    q = numbers(9, sequences, tokens, heads, dim)
    got = attend(g, [cache], [q, np.array([37, 21], np.int32)]).astype(np.float64)
    want, size, sums = plain_attention(q[:, :2], plain.held, [37, 21], window=20)
    assert (np.abs(got[:, :2] - want).max(-1) <= attention_tolerance(F16, size, sums, capacity)).all()
    assert np.isnan(got[:, 2]).all()


@pytest.mark.gpu
def test_attention_of_large_and_small_queries():
    """f32 queries past f16's range and below it keep their bits"""
    for size in (1e6, 1e-6):
        cache, plain = filled(1, 1, 60, 64, I8, 3)
        q = numbers(4, 1, 1, 2, 64, dtype=F32) * np.float32(size)
        got = attend(attention_graph(1, 1, 2, 1, 64, 60, F32, scale=0.1 / size), [cache], [q, np.array([59], np.int32)]).astype(np.float64)
        want, most, sums = plain_attention(q, plain.held, [59], scale=0.1 / size)
        assert (np.abs(got - want).max(-1) <= attention_tolerance(F32, most, sums, 60)).all()


@pytest.mark.gpu
def test_one_hot_attention_copies_values():
    """A key that outweighs all others: its value, to the last bit of an i8 cache's value in f32"""
    cache = KvCache(0, 1, 1, 300, 64)
    g = Graph()
    c = g.cache(1, 1, 300, 64)
    k, v = (g.input((1, 300, 1, 64)) for _ in range(2))
    g.cache_write(c, k, v, g.constant((1,), [0], I32))
    keys, values = np.zeros((1, 300, 1, 64), np.float32), numbers(8, 1, 300, 1, 64, dtype=F32)
    for t in range(300):
        keys[0, t, 0, t % 64] = 1 + t // 64
    with CudaExecutor(0, g, 1) as ex:
        ex.set_cache(0, cache)
        ex.evaluate([keys, values])
    q = np.zeros((1, 1, 64, 64), np.float32)
    q[0, 0, np.arange(64), np.arange(64)] = 1000
    got = attend(attention_graph(1, 1, 64, 1, 64, 300, F32), [cache], [q, np.array([299], np.int32)])
    whole, scale = quantise(values[0, :, 0])
    last = [max(t for t in range(300) if t % 64 == d) for d in range(64)]
    np.testing.assert_allclose(got[0, 0], (whole * scale)[last], rtol=2.0 ** -22)


@pytest.mark.gpu
@pytest.mark.parametrize("storage, dtype", [(I8, F16), (F16, F32)])
def test_positions_far_into_a_large_cache(storage, dtype):
    """Behind 4 GB of a cache: what is written there is what is read there, with a penalty on distance"""
    sequences, heads, dim, capacity, tokens, window = 2, 2, 256, 2_200_000, 3, 40
    cache = KvCache(0, sequences, heads, capacity, dim, storage)
    assert cache.nbytes > 4 << 30
    g = Graph()
    c = g.cache(sequences, heads, capacity, dim, storage)
    k, v = (g.input((sequences, 50, heads, dim)) for _ in range(2))
    g.cache_write(c, k, v, g.input((sequences,), I32))
    keys, values = (numbers(i, sequences, 50, heads, dim, dtype=F32) for i in (1, 2))
    base = capacity - 50
    with CudaExecutor(0, g, 1) as ex:
        ex.set_cache(0, cache)
        ex.evaluate([keys, values, np.array([base, base], np.int32)])
    near = PlainCache(sequences, heads, 50, dim, storage)
    near.write(keys, values, [0, 0])
    for many in (tokens, 40):
        q = numbers(9, sequences, many, 2 * heads, dim, dtype=dtype)
        slopes = np.array([0.5, 0.25, 0.1, 0.01], np.float32)
        got = attend(attention_graph(sequences, many, 2 * heads, heads, dim, capacity, dtype, storage, slopes=True, window=window), [cache],
                     [q, np.array([base + 50 - many, base + 45 - many], np.int32), slopes]).astype(np.float64)
        # (what lies in front is 0: keys whose scores are their distance alone, values of nothing)
        held = np.concatenate([np.zeros_like(near.held), near.held], 3)
        want, size, sums = plain_attention(q, held, [100 - many, 95 - many], slopes=slopes, window=window)
        assert (np.abs(got - want).max(-1) <= attention_tolerance(dtype, size, sums, window)).all()


@pytest.mark.gpu
def test_no_sequences():
    g = Graph()
    c = g.cache(BATCH, 2, 30, 64)
    x, start = g.input(shape(BATCH, 3, 2, 64), F16), g.input(shape(BATCH), I32)
    y = g.cache_attention(x, g.cache_write(c, x, x, start), start)
    g.output(y)
    g.output(g.sample(g.view(g.value_cast(y, F32), shape(BATCH, 3 * 2 * 64)), g.input(shape(BATCH))))
    with CudaExecutor(0, g, 0) as ex:
        out = ex.evaluate([np.zeros((0, 3, 2, 64), np.float16), np.zeros(0, np.int32), np.zeros(0, np.float32)])
    assert out[0].shape == (0, 3, 2, 64) and out[1].shape == (0,)


# ------------------------------------------------------------------------------------------------ on the GPU: attention, what nothing above asks for


def held_after(cache, plain, writes):
    """Writes rows (part, sequence, head, position, channel -> number) into both, position by position; their other numbers stay"""
    _, sequences, heads, capacity, dim = plain.held.shape
    g = Graph()
    c = g.cache(sequences, heads, capacity, dim, plain.dtype)
    k, v = (g.input((sequences, 1, heads, dim)) for _ in range(2))
    g.cache_write(c, k, v, g.input((sequences,), I32), g.input((sequences,), I32))
    with CudaExecutor(0, g, 1) as ex:
        ex.set_cache(0, cache)
        for (part, s, h, t, d), x in writes.items():
            row = plain.held[:, :, :, t][:, :, None].copy()             # [2][sequences][1][heads][dim]
            row[part, s, 0, h, d] = x
            start, count = np.full(sequences, t, np.int32), (np.arange(sequences) == s).astype(np.int32)
            ex.evaluate([row[0], row[1], start, count])
            plain.write(row[0], row[1], start, count)


def check_rows(got, q, plain, start, dtype, **more):
    """Rows with infinities or NaN are those of the definition, number by number; the others within their tolerance, as if the
    infinities, which are not in them, were 0"""
    with np.errstate(invalid="ignore"):
        want = plain_attention(q, plain.held, start, **more)[0]
    finite = np.where(np.isfinite(plain.held), plain.held, 0)
    _, size, sums = plain_attention(np.where(np.isfinite(q), q, 0), finite, start, **more)
    allowed = attention_tolerance(dtype, size, sums, plain.capacity)[..., None]
    got, there = got.astype(np.float64), np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), np.argwhere(np.isnan(got) != np.isnan(want))[:5]
    assert np.array_equal(got[np.isinf(want)], want[np.isinf(want)])
    assert (np.abs(np.where(there, got, 0) - np.where(there, want, 0)) <= allowed).all()


CAPPED = [dict(), dict(softcap=5.0), dict(softcap=30.0, window=50)]


@pytest.mark.gpu
@pytest.mark.parametrize("more", CAPPED, ids=str)
@pytest.mark.parametrize("what", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("dtype, storage, tokens, heads, dim", [(F16, I8, 1, 4, 64), (F16, I8, 5, 4, 128), (F16, F16, 3, 4, 64), (F32, I8, 3, 4, 64), (F32, F16, 3, 2, 128), (F16, I8, 40, 4, 64),
                                                                (F16, I8, 130, 2, 128)])
def test_rows_of_an_8_bit_cache_and_queries_that_hold_no_numbers(dtype, storage, tokens, heads, dim, what, more):
    """NaN stays NaN, with a cap and without: a query's, and a written row's (its scale is NaN) for whoever sees it"""
    capacity, start = 240, [240 - tokens, 30]
    cache, plain = filled(2, 2, capacity, dim, storage, 1)
    q = numbers(9, 2, tokens, heads, dim, dtype=dtype)
    q[1, tokens // 2, 1, 7] = what if storage == F16 and np.isnan(what) else np.nan
    if storage == I8:
        held_after(cache, plain, {(0, 0, 0, 200, 5): what, (0, 1, 1, 31, 0): what, (1, 1, 0, 20, 3): what})
    got = attend(attention_graph(2, tokens, heads, 2, dim, capacity, dtype, storage, **more), [cache], [q, np.array(start, np.int32)])
    check_rows(got, q, plain, start, dtype, **more)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, tokens, heads, dim", [(F16, 1, 2, 64), (F16, 1, 8, 128), (F16, 7, 8, 64), (F16, 3, 4, 192), (F16, 5, 8, 256), (F32, 1, 4, 64), (F32, 6, 4, 128), (F32, 2, 4, 256)])
def test_infinite_values_of_a_16_bit_cache(dtype, tokens, heads, dim):
    """Whoever sees an infinite value has it, whatever tile it is in; both of them, or a NaN, are a NaN"""
    capacity, start = 300, [300 - tokens, 100]
    cache, plain = filled(2, 2, capacity, dim, F16, 1)
    held_after(cache, plain, {(1, 0, 0, 5, 0): np.inf, (1, 0, 0, 64, 1): -np.inf, (1, 0, 0, 299, 2): np.inf, (1, 0, 1, 130, 3): np.inf, (1, 0, 1, 131, 3): -np.inf,
                              (1, 0, 1, 200, 9): np.nan, (1, 1, 0, 100, 4): 1e6, (1, 1, 0, 17, dim - 1): -1e6, (1, 1, 1, 250, 6): np.inf, (1, 1, 1, 101, 8): np.inf})
    q = numbers(9, 2, tokens, heads, dim, dtype=dtype)
    # (the last: scores some hundred apart, weights that f32 does not hold)
    for more in (dict(), dict(window=150), dict(slopes=np.full(heads, 0.02, np.float32)), dict(scale=480 / dim)):
        g = attention_graph(2, tokens, heads, 2, dim, capacity, dtype, F16, **{k: v if k != "slopes" else True for k, v in more.items()})
        got = attend(g, [cache], [q, np.array(start, np.int32)] + ([more["slopes"]] if "slopes" in more else []))
        check_rows(got, q, plain, start, dtype, **more)


@pytest.mark.gpu
@pytest.mark.parametrize("more", [dict(), dict(softcap=5.0)], ids=str)
@pytest.mark.parametrize("dtype, tokens, heads, dim", [(F16, 1, 4, 64), (F16, 7, 8, 128), (F32, 1, 4, 64), (F32, 6, 4, 128), (F32, 2, 4, 256)])
def test_infinite_keys_of_a_16_bit_cache(dtype, tokens, heads, dim, more):
    """A score of minus infinity weighs nothing; one of infinity leaves no number; under a cap both are the cap"""
    capacity, start = 300, [300 - tokens, 100]
    for at, x in ((5, np.inf), (64, -np.inf), (299, np.inf), (130, -1e6)):
        cache, plain = filled(2, 2, capacity, dim, F16, 1)
        held_after(cache, plain, {(0, 0, 0, at, 2): x, (0, 1, 1, at // 3, 5): x})
        q = numbers(9, 2, tokens, heads, dim, dtype=dtype)
        got = attend(attention_graph(2, tokens, heads, 2, dim, capacity, dtype, F16, **more), [cache], [q, np.array(start, np.int32)])
        check_rows(got, q, plain, start, dtype, **more)


@pytest.mark.gpu
@pytest.mark.parametrize("prefix", [0, 70])
@pytest.mark.parametrize("dtype, tokens, heads", [(F16, 1, 4), (F16, 9, 4), (F32, 2, 4), (F16, 40, 4), (F16, 70, 2)])
def test_penalties_far_behind_the_capacity(dtype, tokens, heads, prefix):
    """Positions that f32, or a difference in 32 bits, do not hold: only how much further one key is than another decides"""
    for start in ([2 ** 24 + 1, 2 ** 24 - 40], [2 ** 25 + 3, 2 ** 30 + 5], [2 ** 31 - 1, 2 ** 31 - tokens], [100, 99]):
        check_attention(2, tokens, heads, 2, 64, 100, start, dtype, slopes=True, prefix=prefix)


@pytest.mark.gpu
@pytest.mark.parametrize("sequences, prefix, length", [(70, 17000, 500), (32, 2 ** 15, 64)])
def test_penalties_far_behind_the_capacity_with_a_long_prefix(sequences, prefix, length):
    assert plan_says("the prefix 128 rows at a time", sequences=sequences, heads=8, kv_heads=2, dim=64, capacity=40, prefix=prefix)
    start = [(2 ** 24 + 1, 2 ** 31 - 1, 39, 5, 2 ** 25 + 3)[i % 5] for i in range(sequences)]
    check_attention(sequences, 1, 8, 2, 64, 40, start, slopes=True, prefix=prefix, prefix_length=length)


@pytest.mark.gpu
@pytest.mark.parametrize("storage", [I8, F16])
@pytest.mark.parametrize("sequences, tokens, heads, kv_heads, dim", [(40, 1, 8, 2, 64), (40, 1, 4, 4, 128), (9, 5, 8, 2, 256)])
def test_weights_keep_more_bits_than_results(storage, sequences, tokens, heads, kv_heads, dim):
    """Few keys whose values nearly cancel: of weights of 11 bits (2^-12 of each) the small results would be far off"""
    check_weights(sequences, tokens, heads, kv_heads, dim, storage)


def check_weights(sequences, tokens, heads, kv_heads, dim, storage):
    capacity = tokens + 6
    start = [s % 6 for s in range(sequences)]
    cache, plain = filled(sequences, kv_heads, capacity, dim, storage, 1)
    q = numbers(9, sequences, tokens, heads, dim)
    got = attend(attention_graph(sequences, tokens, heads, kv_heads, dim, capacity, F16, storage, scale=0.3 / dim ** 0.5), [cache], [q, np.array(start, np.int32)]).astype(np.float64)
    want, size, sums = plain_attention(q, plain.held, start, scale=0.3 / dim ** 0.5)
    # the tolerance of results whose weights have 22 bits, and the result's own rounding, of which a number next to nothing has the least step
    allowed = attention_tolerance(F32, size, sums, capacity)[..., None] + np.abs(want) * 2.0 ** -11 + 2.0 ** -25
    assert (np.abs(got - want) <= allowed).all(), float((np.abs(got - want) / allowed).max())


@pytest.mark.gpu
@pytest.mark.parametrize("sequences, tokens, heads, kv_heads, dim", [(3, 64, 2, 2, 64), (2, 40, 8, 2, 128), (2, 150, 2, 2, 100)])
def test_weights_of_many_rows_keep_more_bits_than_results(sequences, tokens, heads, kv_heads, dim):
    assert plan_says(", 128 rows at a time", sequences=sequences, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, capacity=tokens + 6)
    check_weights(sequences, tokens, heads, kv_heads, dim, I8)


@pytest.mark.gpu
def test_results_do_not_depend_on_how_many_sequences_there_are():
    """A prefix that 31 sequences read by 16 rows at a time, and 32 of them by 128: the same sequence has the same result but for a rounding"""
    got, want = [], None
    for n in (31, 32):
        sizes = dict(heads=4, kv_heads=2, dim=64, capacity=40, prefix=2 ** 14)
        assert plan_says("the prefix 128 rows at a time", sequences=n, **sizes) == (n == 32)
        (cache, plain), (shared, held) = filled(n, 2, 40, 64, I8, 1), filled(1, 2, 2 ** 14, 64, I8, 30)
        q = np.repeat(numbers(9, 1, 1, 4, 64), n, 0)
        x = attend(attention_graph(sequences=n, **sizes), [cache, shared], [q, np.full(n, -1, np.int32), np.array([5], np.int32)])
        assert (x == 0).all()                                       # (in front of position 0: sees nothing)
        k = np.repeat(numbers(50, 1, 1, 2, 64), n, 0)
        g = Graph()
        c = g.cache(n, 2, 40, 64)
        a, at = g.input((n, 1, 2, 64), F16), g.input((n,), I32)
        g.cache_write(c, a, a, at)
        with CudaExecutor(0, g, 1) as ex:
            ex.set_cache(0, cache)
            ex.evaluate([k, np.zeros(n, np.int32)])
        plain.write(k, k, [0] * n)
        x = attend(attention_graph(sequences=n, scale=0.04, **sizes), [cache, shared], [q, np.zeros(n, np.int32), np.array([5], np.int32)]).astype(np.float64)
        assert (x == x[:1]).all()
        got.append(x[0])
        want, size, sums = plain_attention(q[:1], plain.held[:, :1], [0], scale=0.04, prefix=held.held, prefix_length=5)
        allowed = attention_tolerance(F32, size, sums, 6)[..., None] + np.abs(want) * 2.0 ** -11 + 2.0 ** -25
        assert (np.abs(x[:1] - want) <= allowed).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, storage, sequences, tokens, heads, kv_heads, dim", [
    (F16, I8, 3, 1, 4, 2, 64), (F16, I8, 2, 5, 8, 2, 128), (F16, F16, 2, 2, 4, 2, 80), (F32, I8, 3, 1, 4, 2, 64), (F32, F16, 2, 4, 6, 2, 100), (F16, I8, 2, 33, 4, 2, 64), (F16, I8, 2, 70, 2, 1, 100),
    (F16, I8, 1, 129, 3, 3, 128)])
def test_attention_takes_queries_of_any_strides(dtype, storage, sequences, tokens, heads, kv_heads, dim):
    """Heads in front of tokens, the middle of wider rows (on and off 16 bytes), one row for all tokens, channels backwards, every other token"""
    capacity = 2 * tokens + 30
    cache, plain = filled(sequences, kv_heads, capacity, dim, storage, 1)
    start = [tokens + 25 - i for i in range(sequences)]
    for form in ("turned", "inside 8", "inside 1", "one", "backwards", "every other"):
        dims = {"turned": (sequences, heads, tokens, dim), "inside 8": (sequences, tokens, heads, dim + 16), "inside 1": (sequences, tokens, heads, dim + 3),
                "one": (sequences, 1, heads, dim), "every other": (sequences, 2 * tokens, heads, dim)}.get(form, (sequences, tokens, heads, dim))
        x = numbers(9, *dims, dtype=dtype)
        g = Graph()
        c = g.cache(sequences, kv_heads, capacity, dim, storage)
        a = g.input(dims, dtype)
        view, q = {"turned": lambda: (g.permute(a, [0, 2, 1, 3]), x.transpose(0, 2, 1, 3)), "inside 8": lambda: (g.slice(a, 3, (8, dim + 8)), x[..., 8:dim + 8]),
                   "inside 1": lambda: (g.slice(a, 3, (1, dim + 1)), x[..., 1:dim + 1]),
                   "one": lambda: (g.broadcast(a, (sequences, tokens, heads, dim)), np.broadcast_to(x, (sequences, tokens, heads, dim))),
                   "backwards": lambda: (g.flip(a, 3), x[..., ::-1]), "every other": lambda: (g.slice(a, 1, (0, 2 * tokens, 2)), x[:, ::2])}[form]()
        g.output(g.cache_attention(view, c, g.input((sequences,), I32)))
        assert "copy" not in plan_describe(g, 1)                        # read where it lies
        got = attend(g, [cache], [x, np.array(start, np.int32)]).astype(np.float64)
        want, size, sums = plain_attention(q, plain.held, start)
        assert (np.abs(got - want).max(-1) <= attention_tolerance(dtype, size, sums, capacity)).all(), form


@pytest.mark.gpu
def test_many_rows_far_into_a_large_cache():
    """Behind 4 GB of a cache, 128 rows at a time"""
    heads, dim, capacity, tokens, window = 2, 128, 17_000_000, 64, 40
    sizes = dict(sequences=1, tokens=tokens, heads=heads, kv_heads=heads, dim=dim, capacity=capacity)
    assert plan_says(", 128 rows at a time", **sizes)
    cache = KvCache(0, 1, heads, capacity, dim)
    assert cache.nbytes > 2 * (4 << 30)
    g = Graph()
    c = g.cache(1, heads, capacity, dim)
    k, v = (g.input((1, 120, heads, dim)) for _ in range(2))
    g.cache_write(c, k, v, g.input((1,), I32))
    keys, values, base = numbers(1, 1, 120, heads, dim, dtype=F32), numbers(2, 1, 120, heads, dim, dtype=F32), capacity - 120
    with CudaExecutor(0, g, 1) as ex:
        ex.set_cache(0, cache)
        ex.evaluate([keys, values, np.array([base], np.int32)])
    near = PlainCache(1, heads, 120, dim, I8)
    near.write(keys, values, [0])
    q, slopes = numbers(9, 1, tokens, heads, dim), np.array([0.3, 0.01], np.float32)
    got = attend(attention_graph(slopes=True, window=window, **sizes), [cache], [q, np.array([base + 56], np.int32), slopes]).astype(np.float64)
    want, size, sums = plain_attention(q, near.held, [56], slopes=slopes, window=window)
    assert (np.abs(got - want).max(-1) <= attention_tolerance(F16, size, sums, window)).all()


def test_short_prefixes_are_read_by_few_rows():
    """The sizes of test_prefix_of_all_sequences_at_once: 16 rows at a time"""
    for sequences, heads, kv_heads, dim, tokens, prefix in ((40, 8, 2, 128, 1, 1000), (70, 4, 4, 64, 1, 256), (9, 8, 1, 100, 2, 300), (33, 4, 1, 128, 1, 4000), (16, 16, 2, 64, 3, 700), (70, 8, 1, 64, 1, 512)):
        assert not plan_says("rows at a time", sequences=sequences, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, capacity=60, prefix=prefix)


# ------------------------------------------------------------------------------------------------ on the GPU: sampling


def sample(logits, uniform, **given):
    g = Graph()
    names = ("temperature", "top_k", "top_p", "min_p")
    x = g.input(logits.shape, DType.of(logits.dtype))
    u = g.input(uniform.shape)
    inputs = {n: g.input(given[n].shape, I32 if n == "top_k" else F32) for n in names if n in given}
    g.output(g.sample(x, u, **inputs))
    with CudaExecutor(0, g, 1) as ex:
        return ex.evaluate([logits, uniform] + [given[n] for n in inputs])[0]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("rows, vocab", [(1, 1), (3, 2), (40, 31), (5, 1000), (64, 4097), (3, 32000), (2, 150001)])
def test_sample(dtype, rows, vocab):
    rng = np.random.default_rng(vocab)
    logits = (3 * rng.standard_normal((rows, vocab))).astype(dtype.np)
    logits[rng.random((rows, vocab)) < 0.1] = -np.inf
    uniform = rng.random(rows, dtype=np.float32)
    given = {"temperature": rng.uniform(0.3, 3, rows).astype(np.float32), "top_k": rng.integers(-1, 2 * min(vocab, 100), rows).astype(np.int32),
             "top_p": rng.uniform(0.2, 1.1, rows).astype(np.float32), "min_p": rng.uniform(0, 0.1, rows).astype(np.float32)}
    for names in ([], ["temperature"], ["top_k"], ["top_p"], ["min_p"], list(given), ["temperature", "top_k", "top_p"], ["top_p", "min_p"]):
        some = {n: given[n] for n in names}
        assert np.array_equal(sample(logits, uniform, **some), plain_sample(logits, uniform, **some)), names


@pytest.mark.gpu
def test_sample_among_equals():
    """Equal logits: the lowest indexes are kept; shares that fall on a border to the last bit"""
    vocab = 5000
    logits = np.zeros((64, vocab), np.float32)
    logits[:, ::3] = np.float32(-0.0)
    uniform = (np.arange(64) / 64).astype(np.float32)
    for given in (dict(), dict(top_k=np.full(64, 1000, np.int32)), dict(top_p=np.full(64, 0.5, np.float32)), dict(top_p=np.full(64, 0.25, np.float32), top_k=np.full(64, 4, np.int32)),
                  dict(top_p=np.zeros(64, np.float32)), dict(min_p=np.ones(64, np.float32)), dict(min_p=np.full(64, 2, np.float32))):
        got = sample(logits, uniform, **given)
        assert np.array_equal(got, plain_sample(logits, uniform, **given)), given
    assert np.array_equal(sample(logits, uniform), np.arange(64) * vocab // 64)
    logits[:, 7] = logits[:, 4321] = 1                                   # two that are likeliest
    greedy = dict(temperature=np.zeros(64, np.float32))
    assert (sample(logits, uniform, **greedy) == 7).all()
    assert set(sample(logits, uniform, top_k=np.full(64, 2, np.int32))) == {7, 4321}
    assert set(sample(logits, uniform, top_k=np.full(64, 1, np.int32))) == {7}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("spread", [1e-6, 1e-3, 0.05])
def test_sample_of_logits_close_together(dtype, spread):
    """Thousands of tokens between which a cut falls, of few different logits or of many"""
    rng = np.random.default_rng(7)
    rows, vocab = 12, 20011
    logits = (5 + spread * rng.standard_normal((rows, vocab))).astype(dtype.np)
    uniform = rng.random(rows, dtype=np.float32)
    for given in (dict(top_k=rng.integers(1, vocab, rows).astype(np.int32)), dict(top_p=rng.uniform(0.05, 0.95, rows).astype(np.float32)),
                  dict(top_k=rng.integers(2000, vocab, rows).astype(np.int32), top_p=rng.uniform(0.05, 0.95, rows).astype(np.float32), min_p=np.full(rows, 0.9, np.float32))):
        assert np.array_equal(sample(logits, uniform, **given), plain_sample(logits, uniform, **given)), given


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, rows, vocab", [(F32, 2, 1 << 19), (F16, 2, 1 << 19), (F32, 1, 8 * 46080 + 1), (F16, 333, 2048), (F32, 700, 5)])
def test_sample_of_the_largest_vocabularies_and_many_rows(dtype, rows, vocab):
    rng = np.random.default_rng(vocab)
    logits = (4 * rng.standard_normal((rows, vocab))).astype(dtype.np)
    uniform = rng.random(rows, dtype=np.float32)
    given = dict(temperature=rng.uniform(0.5, 2, rows).astype(np.float32), top_p=rng.uniform(0.3, 1.1, rows).astype(np.float32))
    assert np.array_equal(sample(logits, uniform, **given), plain_sample(logits, uniform, **given))


@pytest.mark.gpu
def test_sample_without_weights():
    """Rows of nothing but -infinity or NaN; infinities share all of the weight; temperatures from far below to far above 1"""
    vocab = 777
    logits = np.zeros((8, vocab), np.float32)
    logits[0] = -np.inf
    logits[1] = np.nan
    logits[2] = np.nan
    logits[2, 70] = -3
    logits[3, [5, 600]] = np.inf
    logits[4] = np.finfo(np.float32).min
    logits[5] = -np.inf
    logits[5, -1] = np.finfo(np.float32).min
    logits[6, 1] = np.finfo(np.float32).max
    logits[7] = np.arange(vocab)
    for t in (0.0, 1e-30, 1.0, 1e30, np.inf, -1.0, np.nan):
        for u in (0.0, 0.75, float(np.nextafter(np.float32(1), np.float32(0)))):
            given = dict(temperature=np.full(8, t, np.float32), top_p=np.full(8, 0.999, np.float32))
            got = sample(logits, np.full(8, u, np.float32), **given)
            assert np.array_equal(got[[0, 1, 2, 5]], [-1, -1, 70, vocab - 1])
            assert got[3] == (600 if t > 0 and u > 0.5 else 5)
            if not math.isinf(t):
                assert np.array_equal(got, plain_sample(logits, np.full(8, u, np.float32), **given)), (t, u)


def sample_sideways(logits, uniform, **given):
    """The same of logits whose rows do not lie together: the kernel that reads a row again and again"""
    g = Graph()
    names = ("temperature", "top_k", "top_p", "min_p")
    x, u = g.input(logits.shape[::-1], DType.of(logits.dtype)), g.input(uniform.shape)
    inputs = {n: g.input(given[n].shape, I32 if n == "top_k" else F32) for n in names if n in given}
    g.output(g.sample(g.permute(x, [1, 0]), u, **inputs))
    with CudaExecutor(0, g, 1) as ex:
        return ex.evaluate([np.ascontiguousarray(logits.T), uniform] + [given[n] for n in inputs])[0]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("rule", [dict(), dict(top_k=50), dict(min_p=0.01), dict(top_p=1.0), dict(top_p=0.9), dict(top_k=3, min_p=1e-6)], ids=str)
def test_sample_at_low_temperatures(dtype, rule):
    """From where a logit's step is far above the temperature to where it is far below: logits of size 1 to 60000, some of them next to
    the highest, forbidden tokens among them, an odd vocabulary"""
    rng = np.random.default_rng(3)
    vocab, sizes = 1001, (1, 20, 100, 1000, 60000)
    logits = np.stack([np.float32(a) * (1 - rng.random(vocab, dtype=np.float32)) for a in sizes + tuple(-a for a in sizes)]).astype(dtype.np)
    logits[:, rng.random(vocab) < 0.1] = -np.inf
    logits[:, 500], logits[:, 77] = logits.max(-1), np.nan
    for i in range(1, 30):                                               # down from the highest in steps
        logits[:, 500 + 7 * i] = np.nextafter(logits[:, 500 + 7 * (i - 1)], np.array(-np.inf, dtype.np))
    rows = len(logits)
    given = {k: np.full(rows, v, np.int32 if k == "top_k" else np.float32) for k, v in rule.items()}
    for t in (1e-45, 1e-30, 1e-8, 1e-7, 1e-6, 3e-6, 1e-5, 1e-4, 1e-3, 0.03):
        given["temperature"] = np.full(rows, t, np.float32)
        for u in (0.0, 0.25, 0.6, float(np.nextafter(np.float32(1), np.float32(0)))):
            uniform = np.full(rows, u, np.float32)
            want = plain_sample(logits, uniform, **given)
            assert np.array_equal(sample(logits, uniform, **given), want), (t, u)
            assert np.array_equal(sample_sideways(logits, uniform, **given), want), (t, u)


@pytest.mark.gpu
@pytest.mark.parametrize("draw", [sample, sample_sideways])
def test_sample_by_numbers_out_of_range(draw):
    """As the documentation has them, the same by both kernels; forbidden tokens in front, between and behind are not drawn"""
    logits = np.full((7, 301), -np.inf, np.float32)
    logits[:, [9, 40, 41, 200, 250]] = [1, 2, 2, np.nan, 0.5]
    uniform = np.array([1, 2, np.inf, -0.5, -np.inf, np.nan, 0], np.float32)
    assert draw(logits, uniform).tolist() == [250] * 3 + [9] * 4
    assert draw(logits, uniform, top_k=np.full(7, 2, np.int32)).tolist() == [41] * 3 + [40] * 4
    for name in ("temperature", "top_p", "min_p"):
        assert draw(logits, uniform, **{name: np.full(7, np.nan, np.float32)}).tolist() == [40] * 7, name
    assert draw(logits, uniform, min_p=np.full(7, 1.5, np.float32)).tolist() == [40] * 7
    assert draw(logits, uniform, min_p=np.full(7, -1, np.float32)).tolist() == [250] * 3 + [9] * 4


@pytest.mark.gpu
def test_tokens_that_weigh_nothing_are_not_drawn():
    """As many tokens as a cluster holds, two steps below the highest, at a temperature that leaves e^-59 of its weight to each: together 2^-66 of it"""
    logits = np.full((2, 8 * 46080), np.float32(20), np.float32)
    step = np.float32(20) - np.nextafter(np.float32(20), np.float32(0))
    logits[:, 1:] -= 2 * step
    given = dict(temperature=np.full(2, step * np.float32(1.49 / 44), np.float32))
    uniform = np.full(2, np.nextafter(np.float32(1), np.float32(0)), np.float32)
    assert sample(logits, uniform, **given).tolist() == [0, 0]
    assert sample(logits[:, :1 << 14], uniform, **given).tolist() == [0, 0]


@pytest.mark.gpu
def test_sample_reads_any_strides():
    """Logits of the last of several tokens, read in place, and a matrix that lies on its side"""
    rng = np.random.default_rng(2)
    x = rng.standard_normal((3, 5, 701)).astype(np.float32)
    g = Graph()
    a = g.input((3, 5, 701))
    u = g.input((3,))
    g.output(g.sample(g.index(a, 1, 4), u))
    g.output(g.sample(g.permute(g.index(a, 0, 1), [1, 0]), g.broadcast(g.index(u, 0, 2), (701,))))
    uniform = np.array([0.1, 0.5, 0.9], np.float32)
    with CudaExecutor(0, g, 1) as ex:
        one, two = ex.evaluate([x, uniform])
    assert np.array_equal(one, plain_sample(x[:, 4], uniform))
    assert np.array_equal(two, plain_sample(x[1].T, np.full(701, 0.9, np.float32)))


# ------------------------------------------------------------------------------------------------ on the GPU: handles


@pytest.mark.gpu
@pytest.mark.parametrize("use_cuda_graph", [True, False])
def test_caches_that_take_turns(use_cuda_graph):
    """Three caches attached in turn, with one, two and three passes of either kind before the next: steps launched one by one, captured, and
    replayed all read the cache that is attached, with inputs that change from pass to pass"""
    held = [filled(2, 2, 40, 64, I8, seed) for seed in (1, 2, 3)]
    with CudaExecutor(0, attention_graph(), 1, use_cuda_graph=use_cuda_graph) as ex:
        for turn in range(9):
            cache, plain = held[turn % 3]
            ex.set_cache(0, cache)
            for i in range(1 + turn // 3):
                q, start = numbers(20 * turn + i, 2, 1, 4, 64), np.array([39 - turn, 5 + i], np.int32)
                if turn % 2:
                    got = ex.evaluate([q, start])[0]
                else:
                    ex.host_inputs[0][...], ex.host_inputs[1][...] = q, start
                    ex.upload_inputs()
                    ex.run_async()
                    ex.download_outputs()
                    ex.synchronize()
                    got = ex.host_outputs[0].copy()
                want, size, sums = plain_attention(q, plain.held, start)
                assert (np.abs(got.astype(np.float64) - want).max(-1) <= attention_tolerance(F16, size, sums, 40)).all(), (turn, i)


@pytest.mark.gpu
def test_timing_steps_leaves_caches_as_they_are():
    """A write whose keys are computed, in memory that a later step uses again: timing it by itself does not write that into the cache"""
    sequences, heads, dim, capacity = 2, 2, 64, 40
    cache, plain = filled(sequences, heads, capacity, dim, I8, 1)
    g = Graph()
    c = g.cache(sequences, heads, capacity, dim)
    x, start = g.input((sequences, 1, heads, dim), F32), g.input((sequences,), I32)
    k = g.softmax(x, 3)
    written = g.cache_write(c, k, k, start)
    g.output(g.cache_read(written, F32))
    g.output(g.softmax(g.softmax(g.softmax(x, 2), 1), 0))
    a, at = numbers(5, sequences, 1, heads, dim, dtype=F32), np.array([7, 39], np.int32)
    with CudaExecutor(0, g, 1) as ex:
        ex.set_cache(0, cache)
        first = ex.evaluate([a, at])[0].copy()
        for again in range(2):
            ex.evaluate([a, np.array([8, 50], np.int32)])           # (position 8 is the second evaluation's)
            now = ex.evaluate([2 * a, np.array([9, 50], np.int32)])[0].copy()
            for i in list(range(ex.step_count()[0]))[::-1] * 2:
                assert ex.time_step(i, 3) > 0
            reader = Graph()
            reader.output(reader.cache_read(reader.cache(sequences, heads, capacity, dim), F32))
            with CudaExecutor(0, reader, 1) as other:
                other.set_cache(0, cache)
                assert np.array_equal(other.evaluate([])[0], now)
        assert np.array_equal(first[..., 10:, :], now[..., 10:, :]) and np.array_equal(first[..., :8, :], now[..., :8, :])


@pytest.mark.gpu
def test_copies_are_waited_for_by_a_kernel_that_has_given_up():
    """The self-test's second part: behind a wait that ran out a copy is waited for, and has come; with the caches' executors usable afterwards"""
    lib = _lib.load()
    cache, plain = filled(2, 2, 40, 64, I8, 1)
    q, start = numbers(9, 2, 1, 4, 64), np.array([39, 5], np.int32)
    with CudaExecutor(0, attention_graph(), 1) as ex:
        ex.set_cache(0, cache)
        first = ex.evaluate([q, start])[0]
        for _ in range(3):
            assert lib.kn_executor_selftest_wait_expiry(ex._ptr, 200) == 7
            assert b"(code 99)" in lib.kn_last_error()              # 100: a copy that did not come, or was not waited for
            assert np.array_equal(ex.evaluate([q, start])[0], first)


@pytest.mark.gpu
def test_cache_handles_are_checked():
    g = attention_graph()
    inputs = [numbers(1, 2, 1, 4, 64), np.zeros(2, np.int32)]
    with CudaExecutor(0, g, 1) as ex:
        assert ex.cache_count == 1
        for call in (lambda: ex.evaluate(inputs), ex.run_async, lambda: ex.time_step(0), lambda: ex.evaluate_begin(inputs)):
            with pytest.raises(KnError, match="no cache"):
                call()
        good = KvCache(0, 2, 2, 40, 64)
        assert good.nbytes == 2 * 2 * 2 * 48 * (64 + 4)        # (positions in sixteens, a scale each)
        for sizes in ((1, 2, 40, 64), (2, 1, 40, 64), (2, 2, 41, 64), (2, 2, 40, 63), (2, 2, 40, 64, F16)):
            with pytest.raises(KnError):
                ex.set_cache(0, KvCache(0, *sizes))
        for index in (-1, 1):
            with pytest.raises(KnError):
                ex.set_cache(index, good)
        ex.set_cache(0, good)
        assert (ex.evaluate(inputs)[0] == 0).all()               # zeros until something is written
        good.close()                                             # the executor keeps what it has attached
        assert (ex.evaluate(inputs)[0] == 0).all()
        with pytest.raises(ValueError):
            ex.set_cache(0, good)
        ex.set_cache(0, None)
        with pytest.raises(KnError, match="no cache"):
            ex.evaluate(inputs)
    two = attention_graph(sequences=1, prefix=40)
    with CudaExecutor(0, two, 1) as ex:
        one = KvCache(0, 1, 2, 40, 64)
        ex.set_cache(0, one)
        with pytest.raises(KnError, match="same cache"):
            ex.set_cache(1, one)
    for sizes in ((0, 2, 40, 64), (2, 2, 40, 257), (2, 2, 40, 64, F32)):
        with pytest.raises((KnError, ValueError)):
            KvCache(0, *sizes)
    with pytest.raises(Exception):
        KvCache(99, 2, 2, 40, 64)


@pytest.mark.gpu
def test_executors_share_a_cache_in_the_order_of_their_calls():
    """Written by one executor, read by another, on streams of their own, without a wait by the host in between; a third, with the
    list of steps launched one by one, goes on; then another cache takes the place of the first."""
    sequences, heads, capacity, dim, tokens = 3, 2, 512, 64, 500
    g = Graph()
    c = g.cache(sequences, heads, capacity, dim)
    k, v = (g.input((sequences, tokens, heads, dim), F16) for _ in range(2))
    g.cache_write(c, k, v, g.input((sequences,), I32))
    reader = attention_graph(sequences, 1, 4, heads, dim, capacity)
    q, at = numbers(3, sequences, 1, 4, dim), np.array([480, 7, 300], np.int32)
    caches = [KvCache(0, sequences, heads, capacity, dim) for _ in range(2)]
    with CudaExecutor(0, g, 1) as writer, CudaExecutor(0, reader, 1) as a, CudaExecutor(0, reader, 1, use_cuda_graph=False) as b:
        for round_, cache in enumerate(caches):
            for ex in (writer, a, b):
                ex.set_cache(0, cache)
            plain = PlainCache(sequences, heads, capacity, dim, I8)
            for seed in range(2):
                keys, values = numbers(10 * round_ + seed, sequences, tokens, heads, dim), numbers(10 * round_ + seed + 5, sequences, tokens, heads, dim)
                plain.write(keys, values, [0] * 3)
                for to, x in zip(writer.host_inputs, (keys, values, np.zeros(3, np.int32))):
                    to[...] = x
                for ex in (a, b):
                    ex.host_inputs[0][...], ex.host_inputs[1][...] = q, at
                    ex.upload_inputs()
                    ex.synchronize()
                writer.upload_inputs()
                for _ in range(20):
                    writer.run_async()
                a.run_async()
                b.run_async()
                want, size, sums = plain_attention(q, plain.held, at)
                for ex in (a, b):
                    ex.download_outputs()
                    ex.synchronize()
                    assert (np.abs(ex.host_outputs[0] - want).max(-1) <= attention_tolerance(F16, size, sums, capacity)).all()
        writer.run_async()
    with CudaExecutor(0, reader, 1) as late:                     # the one that had the cache last is gone
        late.set_cache(0, caches[1])
        assert np.isfinite(late.evaluate([q, at])[0]).all()
