"""Answers of a LLaMA-shaped decoder (`configs.llama_answer`): prompts of any lengths are taken in piece by piece into caches
that stay on the GPU, then every step draws one token for each sequence from what the caches hold.

    with Answerer(0, batch=16, capacity=2048, layers=32) as a:
        tokens = a.answer(prompts, 100, uniform)          # [16, 100]
"""
from __future__ import annotations

from typing import Sequence

import numpy as np

from . import configs
from .executor import CudaExecutor, KvCache
from .graph import DType

__all__ = ["Answerer"]


class Answerer:
    """`batch` sequences of up to `capacity` positions.  `piece`: tokens of a prompt that go in at a time.  Other arguments are
    `llama_answer`'s.  One executor takes in prompts and one makes a step; they share the caches, one per layer."""

    def __init__(self, device, batch: int, capacity: int, piece: int = 256, layers: int = 32, d_model: int = 4096, heads: int = 32,
                 cache_dtype: DType = DType.I8, math_mode=None, **more):
        self.batch, self.capacity, self.piece = int(batch), int(capacity), int(piece)
        build = lambda tokens: configs.llama_answer(tokens, capacity, layers=layers, d_model=d_model, heads=heads, cache_dtype=cache_dtype, **more)  # noqa: E731
        self.caches = [KvCache(device, batch, heads, capacity, d_model // heads, cache_dtype) for _ in range(layers)]
        self.prompt_executor = CudaExecutor(device, build(self.piece), batch, math_mode=math_mode)
        self.step_executor = CudaExecutor(device, build(1), batch, math_mode=math_mode)
        for ex in (self.prompt_executor, self.step_executor):
            for i, c in enumerate(self.caches):
                ex.set_cache(i, c)
        self.held = np.zeros(self.batch, np.int32)      # positions of each sequence that the caches hold
        self.last_outputs = None

    def _room(self, count):
        if (self.held + np.asarray(count) > self.capacity).any():
            raise ValueError(f"a sequence would have more than {self.capacity} positions")

    def _run(self, executor, ids, count, sampling):
        tokens = ids.shape[1]
        self._room(count)
        self.last_outputs = executor.evaluate([ids, self.held, count, configs.answer_rows(count, tokens), *sampling])
        self.held = self.held + count
        return self.last_outputs[0]

    def _sampling(self, uniform, temperature, top_k, top_p):
        full = lambda v, dtype: np.ascontiguousarray(np.broadcast_to(np.asarray(v, dtype), (self.batch,)))  # noqa: E731
        return full(uniform, np.float32), full(temperature, np.float32), full(top_k, np.int32), full(top_p, np.float32)

    def prompt(self, prompts: Sequence[Sequence[int]], uniform, temperature=1.0, top_k=0, top_p=1.0) -> np.ndarray:
        """Takes in a prompt for every sequence, behind what it holds already, and draws the token that follows each."""
        if len(prompts) != self.batch or min(len(x) for x in prompts) < 1:
            raise ValueError(f"expected {self.batch} prompts of one token and more")
        self._room([len(x) for x in prompts])       # (all of it fits, or none goes in)
        sampling, found = self._sampling(uniform, temperature, top_k, top_p), np.zeros(self.batch, np.int32)
        for at in range(0, max(len(x) for x in prompts), self.piece):
            count = np.array([min(max(len(x) - at, 0), self.piece) for x in prompts], np.int32)
            ids = np.zeros((self.batch, self.piece), np.int32)
            for row, x, n in zip(ids, prompts, count):
                row[:n] = x[at:at + n]
            drawn = self._run(self.prompt_executor, ids, count, sampling)
            ends = (count > 0) & (np.array([len(x) for x in prompts]) <= at + self.piece)
            found = np.where(ends, drawn, found)
        return found

    def step(self, tokens, uniform, temperature=1.0, top_k=0, top_p=1.0) -> np.ndarray:
        """Puts one token behind every sequence and draws the next."""
        ids = np.ascontiguousarray(np.asarray(tokens, np.int32).reshape(self.batch, 1))
        return self._run(self.step_executor, ids, np.ones(self.batch, np.int32), self._sampling(uniform, temperature, top_k, top_p))

    def answer(self, prompts: Sequence[Sequence[int]], tokens: int, uniform, **sampling) -> np.ndarray:
        """`tokens` tokens for every prompt, by random numbers `uniform` [tokens, batch] (or one for all)."""
        if tokens < 1:
            raise ValueError(f"expected one token and more, got {tokens}")
        if len(prompts) == self.batch:
            self._room([len(x) + tokens - 1 for x in prompts])
        uniform = np.broadcast_to(np.asarray(uniform, np.float32), (tokens, self.batch))
        out = [self.prompt(prompts, uniform[0], **sampling)]
        for u in uniform[1:]:
            out.append(self.step(out[-1], u, **sampling))
        return np.stack(out, 1)

    def forget(self):
        """Empties the caches: the next prompts begin new sequences."""
        self.held = np.zeros(self.batch, np.int32)

    def close(self):
        for x in (self.prompt_executor, self.step_executor, *self.caches):
            x.close()

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()
