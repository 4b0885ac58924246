"""A decoder that answers: prompts into caches, tokens one by one, against the same weights' `llama_decoder` evaluated whole."""
import numpy as np
import pytest

from kyanite_b200 import configs
from kyanite_b200.answering import Answerer
from kyanite_b200.executor import MATH_F32, plan_describe
from kyanite_b200.graph import DType

SMALL = dict(layers=2, d_model=128, heads=4, ffn=192, vocab=301)


@pytest.mark.parametrize("dtype", [DType.F16, DType.F32])
def test_plan(dtype):
    graph = configs.llama_answer(1, 64, dtype=dtype, **SMALL)
    text = plan_describe(graph, 3)
    steps = [line.split()[2] for line in text.splitlines() if line.startswith("step")]
    assert steps.count("CacheWrite") == steps.count("CacheAttention") == 2 and steps.count("Sample") == 1
    assert len(graph.caches) == 2
    # keys, values and queries are written and read where the projections left them
    assert not any("copy" in line for line in text.splitlines())


def test_answer_rows():
    assert configs.answer_rows(np.array([3, 1, 0], np.int32), 4).tolist() == [2, 4, 8]


def whole_logits(ids, dtype, oracle):
    """Logits behind each of the last tokens of `ids`, by the whole decoder on the CPU, in f32 (exact weights of `dtype`)"""
    graph, _ = configs.llama_decoder(seq=len(ids), dtype=dtype, **SMALL)
    return oracle(graph.to_bytes(), 1, [np.array([ids], np.int32)])[0][0]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, cache_dtype, limit", [
    # f32 throughout but for keys and values of 11 bits (f16): logits of size 0.2 from 256 values of a few products each
    (DType.F32, DType.F16, 4e-4),
    (DType.F32, DType.I8, 6e-3),
    (DType.F16, DType.I8, 8e-3)])
def test_answers_are_those_of_the_whole_decoder(dtype, cache_dtype, limit):
    """Greedy answers to prompts of ragged lengths, longer than a piece and shorter: each token is the likeliest one behind the prompt and the
    tokens so far, or (rounding) within `limit` of it; the logits that it was drawn from are the whole decoder's.  Rounding keys and
    values to 8 bits (1 / 254 of a row's largest, which is some 2.5 times its usual size) moves a context by that share of itself at most."""
    from oracle.cpu_eval import cpu_eval_graph
    prompts = [list(range(5, 5 + n)) for n in (1, 7, 8, 9, 20)]
    with Answerer(0, batch=5, capacity=64, piece=8, dtype=dtype, cache_dtype=cache_dtype, with_logits=True, math_mode=MATH_F32, **SMALL) as a:
        sequences = [list(x) for x in prompts]
        token = a.prompt(prompts, 0.0, temperature=0.0)
        seen = {}
        for step in range(6):
            for s in range(5):
                sequences[s].append(int(token[s]))
            token = a.step(token, 0.0, temperature=0.0)
            seen[step] = (token.copy(), a.last_outputs[1].astype(np.float64))
        assert a.held.tolist() == [len(x) + 6 for x in prompts]
        for s in range(5):
            logits = whole_logits(sequences[s], dtype, cpu_eval_graph).astype(np.float64)
            for step in range(6):
                want = logits[len(prompts[s]) + step]
                assert np.abs(seen[step][1][s] - want).max() <= limit
                assert want.max() - want[seen[step][0][s]] <= 2 * limit
                assert seen[step][0][s] == seen[step][1][s].argmax()


@pytest.mark.gpu
def test_answers_with_given_random_numbers():
    """The same random numbers, the same tokens, also after forgetting; prompts and calls that do not fit are refused"""
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, 301, n).tolist() for n in (11, 3, 30)]
    uniform = rng.random((8, 3), dtype=np.float32)
    sampling = dict(temperature=0.8, top_k=50, top_p=0.95)
    with Answerer(0, batch=3, capacity=64, piece=32, math_mode=MATH_F32, **SMALL) as a:
        first = a.answer(prompts, 8, uniform, **sampling)
        a.forget()
        assert np.array_equal(a.answer(prompts, 8, uniform, **sampling), first)
        assert (first >= 0).all() and (first < 301).all() and len({tuple(x) for x in first}) == 3
        with pytest.raises(ValueError):
            a.prompt([[1] * 60] * 3, 0.5)
        with pytest.raises(ValueError):
            a.prompt([[1], [2], []], 0.5)
        with pytest.raises(ValueError):
            a.prompt([[1]], 0.5)


@pytest.mark.gpu
def test_what_does_not_fit_leaves_the_answerer_as_it_was():
    """A prompt of several pieces, or an answer, that would pass the capacity is refused before its first piece goes in"""
    with Answerer(0, batch=2, capacity=20, piece=8, math_mode=MATH_F32, **SMALL) as a:
        with pytest.raises(ValueError, match="more than 20 positions"):
            a.prompt([[1] * 21, [2]], 0.5)
        assert a.held.tolist() == [0, 0]
        with pytest.raises(ValueError, match="more than 20 positions"):
            a.answer([[1] * 17, [2]], 5, 0.5)
        with pytest.raises(ValueError, match="one token"):
            a.answer([[1], [2]], 0, 0.5)
        assert a.held.tolist() == [0, 0]
        assert a.answer([[1] * 17, [2]], 4, 0.5).shape == (2, 4) and a.held.tolist() == [20, 4]
