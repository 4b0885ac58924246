"""Performance cases of the operators that answer with a decoder: a cache of keys and values that is quantised as it is
written, attention that reads it, and sampling of tokens.

A case is one graph around one operator, at one set of sizes:

    op "cache"      keys and values of new tokens are written behind the earlier ones of every sequence, and the cache is read back
    op "attention"  one to many new tokens of every sequence attend to what the cache holds of it (and of a prefix that all share)
    op "sample"     one token for every row of logits

Where `own` is false the operators are computed in their plain form: elementary torch operations in 32 bits (in 64 where a
border between tokens hangs on it), rounded once.  Where it is true they are steps of an executor: inputs are in the executor's
device buffers, where the steps before would have left them, and a pass is one `run_async`.
"""
import functools
import math

import numpy as np
import torch

own = False
DEVICE = "cuda"
TYPES = {"f16": torch.float16, "f32": torch.float32}

# ------------------------------------------------------------------------------------------------ the cases


def _cache(seqs, heads, dim, capacity, tokens, earlier, storage="i8", dtype="f16"):
    """`tokens`: new ones of the longest sequence; `earlier`: those that the fullest sequence holds before them."""
    return {"op": "cache", "seqs": seqs, "kv_heads": heads, "dim": dim, "capacity": capacity, "tokens": tokens, "earlier": earlier,
            "storage": storage, "dtype": dtype}


def _attention(seqs, heads, kv_heads, dim, length, tokens=1, storage="i8", dtype="f16", ragged=True, cap=0.0, window=0, slopes=False, prefix=0):
    """`length`: positions of the longest sequence behind the shared prefix, its new tokens among them."""
    return {"op": "attention", "seqs": seqs, "heads": heads, "kv_heads": kv_heads, "dim": dim, "length": length, "tokens": tokens,
            "storage": storage, "dtype": dtype, "ragged": ragged, "cap": cap, "window": window, "slopes": slopes, "prefix": prefix}


def _sample(rows, vocab, dtype="f32", rule="mixed"):
    return {"op": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "rule": rule}


def listed():
    return [
        # the smallest call: one conversation, one new token, a short history; every head has keys of its own
        {"name": "attend_s1_l333", **_attention(1, 32, 32, 128, 333)},
        # a server's batch of conversations of middling length, four query heads to a pair of keys and values
        {"name": "attend_s16_l2048", **_attention(16, 32, 8, 128, 2048)},
        # the same server with its memory full
        {"name": "attend_s64_l8192", **_attention(64, 32, 8, 128, 8192)},
        # one reader of a very long document
        {"name": "attend_s1_l131072", **_attention(1, 32, 8, 128, 131072, ragged=False)},
        # a network in f32 with narrow heads, half storage and a penalty on distance
        {"name": "attend_f32_d64", **_attention(24, 12, 12, 64, 1500, storage="f16", dtype="f32", slopes=True)},
        # capped scores over a window of the latest positions, wide heads, guessed tokens checked five at a time
        {"name": "attend_cap_window", **_attention(8, 16, 8, 256, 8000, tokens=5, cap=50.0, window=4096)},
        # many answers to one long prompt
        {"name": "attend_prefix_4096", **_attention(64, 32, 8, 128, 300, prefix=4096)},
        # the next piece of a long prompt, behind what is in the cache already
        {"name": "attend_chunk_512", **_attention(2, 32, 8, 128, 4608, tokens=512, ragged=False)},
        # one token behind each of many histories; then the cache is handed on
        {"name": "cache_s32_t1", **_cache(32, 8, 128, 1024, 1, 1000)},
        # prompts of ragged length into an empty cache, in f32
        {"name": "cache_s7_t1500", **_cache(7, 32, 128, 1536, 1500, 0, dtype="f32")},
        # one answer, the configured decoder's vocabulary
        {"name": "sample_r1_v32000", **_sample(1, 32000)},
        # a large batch over a large vocabulary, the heaviest draw: every token may be taken
        {"name": "sample_r200_v128256", **_sample(200, 128256, dtype="f16", rule="plain")},
    ]


def _spread(rng, low, high):
    """A whole number from low to high, spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    most = _cost(_attention(64, 32, 8, 128, 8192))
    while True:
        op = rng.choice(["attention", "attention", "attention", "cache", "sample"])
        if op == "sample":
            case = _sample(_spread(rng, 1, 256), _spread(rng, 500, 200000), rng.choice(["f32", "f16"]),
                           rng.choice(["mixed", "mixed", "plain", "greedy", "narrow"]))
        elif op == "cache":
            capacity = _spread(rng, 16, 4096)
            tokens = rng.choice([1, _spread(rng, 1, capacity)])
            case = _cache(_spread(rng, 1, 64), rng.choice([1, 4, 8, 12, 32]), rng.choice([64, 80, 96, 128, 256]), capacity, tokens,
                          rng.randrange(0, capacity - tokens + 1), rng.choice(["i8", "i8", "f16"]), rng.choice(["f16", "f32"]))
        else:
            kv = rng.choice([1, 2, 4, 8, 12, 32])
            group = rng.choice([1, 1, 2, 4, 7, 8])
            tokens = rng.choice([1, 1, 1, _spread(rng, 2, 8), _spread(rng, 8, 300)])
            case = _attention(_spread(rng, 1, 128), kv * group, kv, rng.choice([64, 80, 96, 128, 128, 256]),
                              tokens + _spread(rng, 1, 50000), tokens, rng.choice(["i8", "i8", "f16"]), rng.choice(["f16", "f16", "f32"]),
                              rng.random() < 0.7, rng.choice([0.0, 0.0, 30.0]), rng.choice([0, 0, _spread(rng, 16, 4096)]),
                              rng.random() < 0.25, rng.choice([0, 0, 0, _spread(rng, 16, 8192)]))
        if _cost(case) <= most:
            return case


def _cost(case):
    """About what a pass of the plain form moves through memory, in bytes."""
    if case["op"] == "sample":
        return 100.0 * case["rows"] * case["vocab"]
    if case["op"] == "cache":
        return 30.0 * case["seqs"] * case["kv_heads"] * case["capacity"] * case["dim"]
    held = case["seqs"] * (case["length"] + case["prefix"])
    return held * (18.0 * case["kv_heads"] * case["dim"] + 24.0 * case["heads"] * case["tokens"])


# ------------------------------------------------------------------------------------------------ inputs


def _lengths(count, longest, ragged, least=1):
    """Lengths of `count` sequences: the first has the longest, the others are spread down to a quarter of it."""
    if not ragged:
        return [longest] * count
    return [max(least, int(round(longest * (1 - 0.75 * ((i * 0.6180339887498949) % 1.0))))) for i in range(count)]


def _plan(case):
    """(positions that each sequence holds before the new tokens, its new tokens)"""
    if case["op"] == "cache":
        held = _lengths(case["seqs"], case["earlier"], True, 0)
        new = _lengths(case["seqs"], case["tokens"], True)
    else:
        total = _lengths(case["seqs"], case["length"], case["ragged"], case["tokens"])
        new = [case["tokens"]] * case["seqs"]
        held = [n - case["tokens"] for n in total]
    return held, new


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed) * 7919 + 17)


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEVICE)


def _channels(gen, heads, dim):
    """How large a head's channels are: a few of them stand out, as in trained keys."""
    size = torch.exp(0.4 * _normal(gen, heads, dim))
    return size * torch.where(torch.rand(heads, dim, generator=gen, device=DEVICE) < 0.03, 4.0, 1.0)


def _keys_and_values(gen, case, seqs, length, sizes):
    """[2][seqs][length][kv_heads][dim]: keys and values as projections leave them"""
    x = _normal(gen, 2, seqs, length, case["kv_heads"], case["dim"])
    x[0].mul_(sizes[0])
    x[1].mul_(sizes[1])
    return x.to(TYPES[case["dtype"]])


def _quantised(x):
    """(whole numbers from -127 to 127, their scales): the values of a position of a head share one"""
    x = x.float()
    scale = x.abs().amax(-1, keepdim=True) / 127.0
    q = torch.where(scale > 0, torch.round(x / scale), torch.zeros_like(x))
    return q.to(torch.int8), scale


PIECE = 256  # positions that a prompt is written in at a time


def _held(gen, case, sizes, seqs, length, capacity, cache, valid):
    """Fills a cache with `length` positions of every sequence of which the first valid[s] count: into `cache`, a handle of the
    framework, or into arrays [2][seqs][kv_heads][capacity][dim] that are returned with their scales."""
    shape = (2, seqs, case["kv_heads"], capacity, case["dim"])
    i8 = case["storage"] == "i8"
    arrays = scales = None
    if cache is None:
        arrays = torch.zeros(shape, dtype=torch.int8 if i8 else torch.float16, device=DEVICE)
        scales = torch.zeros(*shape[:4], 1, device=DEVICE) if i8 else None
    for at in range(0, length, PIECE):
        x = _keys_and_values(gen, case, seqs, min(PIECE, length - at), sizes)
        count = (valid - at).clamp(0, x.shape[2]).to(torch.int32)
        if cache is not None:
            padded = torch.zeros(2, seqs, PIECE, *x.shape[3:], dtype=x.dtype, device=DEVICE)
            padded[:, :, :x.shape[2]] = x
            writer = _writer(seqs, case["kv_heads"], case["dim"], capacity, PIECE, case["storage"], case["dtype"])
            writer.executor.set_cache(0, cache)
            writer(padded[0], padded[1], torch.full_like(count, at), count)
            torch.cuda.synchronize()
            continue
        keep = torch.arange(x.shape[2], device=DEVICE)[None, :] < count[:, None]
        x = torch.where(keep[None, :, :, None, None], x, torch.zeros_like(x)).transpose(2, 3)
        if i8:
            q, s = _quantised(x)
            arrays[:, :, :, at:at + x.shape[3]] = q
            scales[:, :, :, at:at + x.shape[3]] = s
        else:
            arrays[:, :, :, at:at + x.shape[3]] = x.to(torch.float16)
    return arrays, scales


def _inputs(case, seed, cache=None, prefix=None):
    gen = _generator(seed)
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # a few tokens that fit, many that do not, and some that are forbidden
        logits = 2.0 * _normal(gen, rows, vocab) + 6.0 * (torch.rand(rows, vocab, generator=gen, device=DEVICE) < 40.0 / vocab)
        logits = torch.where(torch.rand(rows, vocab, generator=gen, device=DEVICE) < 0.01, -math.inf, logits).to(TYPES[case["dtype"]])
        uniform = torch.rand(rows, generator=gen, device=DEVICE)
        kind = torch.randint(0, 6, (rows,), generator=gen, device=DEVICE)
        temperature, top_k = torch.full((rows,), 1.0, device=DEVICE), torch.zeros(rows, dtype=torch.int32, device=DEVICE)
        top_p, min_p = torch.ones(rows, device=DEVICE), torch.zeros(rows, device=DEVICE)
        if case["rule"] == "greedy":
            temperature.zero_()
        elif case["rule"] == "narrow":
            temperature.fill_(0.7), top_k.fill_(50), top_p.fill_(0.9)
        elif case["rule"] == "mixed":
            temperature = 0.6 + 0.6 * torch.rand(rows, generator=gen, device=DEVICE)
            top_k = torch.where(kind < 2, 40, 0).to(torch.int32)
            top_p = torch.where((kind > 0) & (kind < 4), 0.95, 1.0)
            min_p = torch.where(kind > 3, 0.02, 0.0)
        return {"logits": logits, "uniform": uniform, "temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p}
    held, new = (torch.tensor(v, dtype=torch.int32, device=DEVICE) for v in _plan(case))
    sizes = _channels(gen, case["kv_heads"], case["dim"]), _channels(gen, case["kv_heads"], case["dim"])
    out = {"start": held}
    if case["op"] == "cache":
        out["held"], out["held_scales"] = _held(gen, case, sizes, case["seqs"], int(max(_plan(case)[0])), case["capacity"], cache, held)
        x = _keys_and_values(gen, case, case["seqs"], case["tokens"], sizes)
        out.update(keys=x[0], values=x[1], count=new)
        return out
    out["held"], out["held_scales"] = _held(gen, case, sizes, case["seqs"], case["length"], case["length"], cache, held + new)
    if case["prefix"]:
        whole = torch.full((1,), case["prefix"], dtype=torch.int32, device=DEVICE)
        out["prefix"], out["prefix_scales"] = _held(gen, case, sizes, 1, case["prefix"], case["prefix"], prefix, whole)
        out["prefix_length"] = whole
    q = _normal(gen, case["seqs"], case["tokens"], case["heads"], case["dim"]) * 1.2
    # (scores that spread as those of trained heads do, whatever the channels' sizes)
    group = case["heads"] // case["kv_heads"]
    q = (q / sizes[0].square().mean(-1).sqrt().repeat_interleave(group, 0)[None, None, :, None]).to(TYPES[case["dtype"]])
    out["q"] = q
    if case["slopes"]:
        out["slopes"] = torch.exp2(-8.0 * (1 + torch.arange(case["heads"], device=DEVICE, dtype=torch.float32)) / case["heads"])
    return out


# ------------------------------------------------------------------------------------------------ the framework's calls


class _DeviceArray:
    """An executor's device buffer as torch sees it; a tensor made of it keeps the executor, whose memory it is."""

    def __init__(self, executor, is_output, index):
        self.executor = executor
        array = (executor.host_outputs if is_output else executor.host_inputs)[index]
        pointer, _ = executor.device_buffer(is_output, index)
        self.__cuda_array_interface__ = {"shape": array.shape, "typestr": array.dtype.str, "data": (pointer, False), "version": 3}


class _Program:
    """An executor whose inputs and outputs stay on the GPU."""

    def __init__(self, graph):
        from kyanite_b200.executor import CudaExecutor
        self.executor = CudaExecutor(0, graph, 1)
        arrays = lambda is_output, n: [torch.as_tensor(_DeviceArray(self.executor, is_output, i), device=DEVICE) for i in range(n)]  # noqa: E731
        self.inputs = arrays(False, len(self.executor.host_inputs))
        self.outputs = arrays(True, len(self.executor.host_outputs))

    def load(self, *tensors):
        for to, x in zip(self.inputs, tensors, strict=True):
            to.copy_(x)
        torch.cuda.synchronize()

    def __call__(self, *tensors):
        self.load(*tensors)
        self.executor.run_async()


def _dtype(name):
    from kyanite_b200.graph import DType
    return {"f16": DType.F16, "f32": DType.F32, "i8": DType.I8, "i32": DType.I32}[name]


@functools.lru_cache(maxsize=2)
def _writer(seqs, kv_heads, dim, capacity, tokens, storage, dtype):
    """A program that writes pieces of prompts into a cache."""
    from kyanite_b200.graph import Graph
    g = Graph()
    cache = g.cache(seqs, kv_heads, capacity, dim, _dtype(storage))
    k, v = (g.input((seqs, tokens, kv_heads, dim), _dtype(dtype)) for _ in range(2))
    start, count = (g.input((seqs,), _dtype("i32")) for _ in range(2))
    g.cache_write(cache, k, v, start, count)
    return _Program(g)


def _handle(case, seqs, capacity):
    from kyanite_b200.executor import KvCache
    return KvCache(0, seqs, case["kv_heads"], capacity, case["dim"], _dtype(case["storage"]))


def _program(case, caches):
    from kyanite_b200.graph import Graph
    g = Graph()
    if case["op"] == "sample":
        logits = g.input((case["rows"], case["vocab"]), _dtype(case["dtype"]))
        uniform, temperature = (g.input((case["rows"],)) for _ in range(2))
        top_k = g.input((case["rows"],), _dtype("i32"))
        top_p, min_p = (g.input((case["rows"],)) for _ in range(2))
        g.output(g.sample(logits, uniform, temperature, top_k, top_p, min_p))
        return _Program(g)
    capacity = case["capacity"] if case["op"] == "cache" else case["length"]
    cache = g.cache(case["seqs"], case["kv_heads"], capacity, case["dim"], _dtype(case["storage"]))
    prefix = g.cache(1, case["kv_heads"], case["prefix"], case["dim"], _dtype(case["storage"])) if case.get("prefix") else None
    if case["op"] == "cache":
        k, v = (g.input((case["seqs"], case["tokens"], case["kv_heads"], case["dim"]), _dtype(case["dtype"])) for _ in range(2))
        start, count = (g.input((case["seqs"],), _dtype("i32")) for _ in range(2))
        g.output(g.cache_read(g.cache_write(cache, k, v, start, count), _dtype("f16")))
    else:
        q = g.input((case["seqs"], case["tokens"], case["heads"], case["dim"]), _dtype(case["dtype"]))
        start = g.input((case["seqs"],), _dtype("i32"))
        slopes = g.input((case["heads"],)) if case["slopes"] else None
        length = g.input((1,), _dtype("i32")) if prefix is not None else None
        g.output(g.cache_attention(q, cache, start, softcap=case["cap"], window=case["window"], slopes=slopes, prefix=prefix, prefix_length=length))
    program = _Program(g)
    for i, c in enumerate(caches):
        program.executor.set_cache(i, c)
    return program


def prepare(case, seed):
    if not own:
        return {"case": case, **_inputs(case, seed)}
    if case["op"] == "sample":
        program = _program(case, [])
        x = _inputs(case, seed)
        program.load(x["logits"], x["uniform"], x["temperature"], x["top_k"], x["top_p"], x["min_p"])
        return {"program": program}
    caches = [_handle(case, case["seqs"], case["capacity"] if case["op"] == "cache" else case["length"])]
    if case.get("prefix"):
        caches.append(_handle(case, 1, case["prefix"]))
    x = _inputs(case, seed, *caches)
    program = _program(case, caches)
    names = ("keys", "values", "start", "count") if case["op"] == "cache" else ("q", "start", "slopes", "prefix_length")
    program.load(*(x[n] for n in names if n in x))
    return {"program": program, "caches": caches}


def run(state):
    if "program" in state:
        state["program"].executor.run_async()
        return state["program"].outputs
    case = state["case"]
    return [{"cache": _plain_cache, "attention": _plain_attention, "sample": _plain_sample}[case["op"]](case, state)]


# ------------------------------------------------------------------------------------------------ the plain forms


def _values(held, scales):
    return held.float() * scales if scales is not None else held.float()


def _plain_cache(case, x):
    """[2][seqs][kv_heads][capacity][dim] in f16: what the cache holds once the new tokens are written"""
    at = torch.arange(case["capacity"], device=DEVICE)[None, :] - x["start"][:, None]   # the new token that belongs there
    fresh = ((at >= 0) & (at < x["count"][:, None]))[None, :, None, :, None]
    new = torch.stack([x["keys"], x["values"]]).transpose(2, 3)
    index = at.clamp(0, case["tokens"] - 1).long()[None, :, None, :, None].expand(2, -1, new.shape[2], -1, new.shape[4])
    if x["held_scales"] is None:
        new = new.to(torch.float16)
        x["held"] = torch.where(fresh, torch.gather(new, 3, index), x["held"])
        return x["held"].clone()
    q, scale = _quantised(new)
    x["held"] = torch.where(fresh, torch.gather(q, 3, index), x["held"])
    x["held_scales"] = torch.where(fresh, torch.gather(scale, 3, index[..., :1]), x["held_scales"])
    return _values(x["held"], x["held_scales"]).to(torch.float16)


def _plain_attention(case, x):
    """[seqs][tokens][heads][dim]: softmax(scores) . values of every new token"""
    s, t, h, kv, d, p = (case[k] for k in ("seqs", "tokens", "heads", "kv_heads", "dim", "prefix"))
    held = _values(x["held"], x["held_scales"])                                        # [2][s][kv][length][d]
    if p:
        shared = _values(x["prefix"], x["prefix_scales"]).expand(2, s, kv, p, d)
        held = torch.cat([shared, held], 3)
    q = x["q"].float().view(s, t, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(s, kv, (h // kv) * t, d)
    scores = torch.matmul(q, held[0].transpose(-1, -2)) / math.sqrt(d)
    scores = scores.view(s, kv, h // kv, t, -1)
    if case["cap"]:
        scores = case["cap"] * torch.tanh(scores / case["cap"])
    key = torch.arange(held.shape[3], device=DEVICE)
    row = x["start"][:, None] + torch.arange(t, device=DEVICE)[None, :] + p
    distance = (row[:, :, None] - key[None, None, :])[:, None, None]                   # [s][1][1][t][keys]
    if case["slopes"]:
        scores = scores - x["slopes"].view(1, kv, h // kv, 1, 1) * distance
    seen = distance >= 0
    if case["window"]:
        seen = seen & (distance < case["window"])
    scores = scores.masked_fill(~seen, -math.inf)
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = torch.matmul(e.view(s, kv, (h // kv) * t, -1), held[1]) / e.sum(-1).view(s, kv, (h // kv) * t, 1)
    return out.view(s, kv, h // kv, t, d).permute(0, 3, 1, 2, 4).reshape(s, t, h, d).to(TYPES[case["dtype"]])


def _plain_sample(case, x):
    """[rows], whole numbers of 32 bits: tokens by falling logit, the lowest index first among equals; the first top_k of them; of these the fewest that
    have top_p of their mass; of these the ones that are at least min_p times as likely as the likeliest.  Drawn from what is left, in the
    order of the index: the first token behind which more than `uniform` of the mass lies.  Temperature 0: the likeliest."""
    logits = x["logits"].double()
    top, order = torch.sort(logits, dim=-1, descending=True, stable=True)
    t = x["temperature"].double()[:, None]
    weight = torch.exp((top - top[:, :1]) / torch.where(t > 0, t, torch.ones_like(t)))
    rank = torch.arange(logits.shape[1], device=DEVICE)[None, :]
    k = torch.where(x["top_k"] > 0, x["top_k"], logits.shape[1])[:, None]
    weight = torch.where(rank < k, weight, torch.zeros_like(weight))
    before = torch.cumsum(weight, -1) - weight
    keep = (before < x["top_p"].double()[:, None] * weight.sum(-1, keepdim=True)) | (x["top_p"][:, None] >= 1)
    keep &= (weight >= x["min_p"].double()[:, None])
    keep |= rank == 0
    weight = torch.where(keep, weight, torch.zeros_like(weight))
    mass = torch.cumsum(torch.zeros_like(weight).scatter_(-1, order, weight), -1)
    over = mass > x["uniform"].double()[:, None] * mass[:, -1:]
    token = torch.argmax(over.to(torch.uint8), -1)
    return torch.where(t[:, 0] > 0, token, order[:, 0]).to(torch.int32)


# ------------------------------------------------------------------------------------------------ from the definitions, in 64 bits


def exact(case, seed):
    x = _inputs(case, seed)
    return [{"cache": _exact_cache, "attention": _exact_attention, "sample": _exact_sample}[case["op"]](case, x)]


def _exact_values(held, scales):
    return held.double() if scales is None else held.double() * scales.double()


def _exact_cache(case, x):
    out = _exact_values(x["held"], x["held_scales"])
    for s, (start, count) in enumerate(zip(*_plan(case))):
        for part, new in enumerate((x["keys"], x["values"])):
            rows = new[s, :count].transpose(0, 1)                                      # [kv][count][d]
            if case["storage"] == "i8":
                scale = rows.float().abs().amax(-1, keepdim=True) / 127.0              # (the scale is a number of 32 bits)
                whole = torch.round(rows.float() / torch.where(scale > 0, scale, torch.ones_like(scale)))
                out[part, s, :, start:start + count] = whole.double() * scale.double()
            else:
                out[part, s, :, start:start + count] = rows.to(torch.float16).double()
    return out


def _exact_attention(case, x):
    group, d, p = case["heads"] // case["kv_heads"], case["dim"], case["prefix"]
    held, new = _plan(case)
    out = torch.zeros(case["seqs"], case["tokens"], case["heads"], d, dtype=torch.float64, device=DEVICE)
    shared = _exact_values(x["prefix"], x["prefix_scales"])[:, 0] if p else None
    for s in range(case["seqs"]):
        total = held[s] + new[s]
        scales = None if x["held_scales"] is None else x["held_scales"][:, s, :, :total]
        keys, values = _exact_values(x["held"][:, s, :, :total], scales)               # [kv][total][d]
        if p:
            keys, values = torch.cat([shared[0], keys], 1), torch.cat([shared[1], values], 1)
        for t in range(case["tokens"]) if case["tokens"] < 16 else [slice(0, case["tokens"])]:
            rows = torch.arange(case["tokens"], device=DEVICE)[t].reshape(-1)
            q = x["q"][s, rows].double().view(len(rows), case["kv_heads"], group, d)
            score = torch.einsum("tkgd,kcd->tkgc", q, keys) / math.sqrt(d)
            if case["cap"]:
                score = case["cap"] * torch.tanh(score / case["cap"])
            away = (p + held[s] + rows)[:, None, None, None] - torch.arange(keys.shape[1], device=DEVICE)
            if case["slopes"]:
                score = score - x["slopes"].double().view(1, case["kv_heads"], group, 1) * away
            hidden = (away < 0) | ((away >= case["window"]) if case["window"] else torch.zeros_like(away, dtype=torch.bool))
            share = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
            out[s, rows] = torch.einsum("tkgc,kcd->tkgd", share, values).reshape(len(rows), case["heads"], d)
    return out


def _exact_sample(case, x):
    logits, found = x["logits"].double().cpu().numpy(), []
    for r in range(case["rows"]):
        u, t, k, p, m = (float(x[n][r]) for n in ("uniform", "temperature", "top_k", "top_p", "min_p"))
        order = np.argsort(-logits[r], kind="stable")
        if t == 0:
            found.append(order[0])
            continue
        order = order[:int(k)] if k > 0 else order
        weight = np.exp((logits[r][order] - logits[r][order[0]]) / t).astype(np.longdouble)
        if p < 1:
            order = order[:1 + int(np.searchsorted(np.cumsum(weight)[:-1], p * weight.sum(), "left"))]
        weight = weight[:len(order)]
        left = (weight >= m) | (np.arange(len(order)) == 0)
        by_index = np.sort(order[left])
        mass = np.cumsum(weight[left][np.argsort(order[left])])
        found.append(by_index[min(int(np.searchsorted(mass, u * mass[-1], "right")), len(by_index) - 1)])
    return torch.tensor(np.array(found), dtype=torch.int32)


# ------------------------------------------------------------------------------------------------ what a pass needs


def work(case):
    if case["op"] == "sample":
        size = {"f16": 2, "f32": 4}[case["dtype"]]
        return {"bytes": float(case["rows"] * (case["vocab"] * size + 24)), "flops": 2.0 * case["rows"] * case["vocab"]}
    token = 2 * case["kv_heads"] * (case["dim"] * (1 if case["storage"] == "i8" else 2) + (4 if case["storage"] == "i8" else 0))
    size = {"f16": 2, "f32": 4}[case["dtype"]]
    held, new = _plan(case)
    if case["op"] == "cache":
        fresh = 2 * case["kv_heads"] * case["dim"] * size
        whole = case["seqs"] * case["capacity"]
        # new tokens in and into the cache, the cache out of memory and its values into it
        return {"bytes": float(sum(new) * (fresh + token) + whole * (token + 4 * case["kv_heads"] * case["dim"])),
                "flops": 2.0 * case["dim"] * case["kv_heads"] * (2 * sum(new) + whole)}
    window = case["window"] or 1 << 40
    p = case["prefix"]
    read = sum(min(h + n, window + n - 1) for h, n in zip(held, new))
    shared = min(p, max(0, max(window - 1 - h for h in held)))
    pairs = sum(min(p + h + t + 1, window) for h, n in zip(held, new) for t in range(n))
    ends = 2 * case["seqs"] * case["tokens"] * case["heads"] * case["dim"] * size
    return {"bytes": float((read + shared) * token + ends), "flops": 4.0 * case["heads"] * case["dim"] * pairs}
