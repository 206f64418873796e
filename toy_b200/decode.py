"""Decode with a KV cache over the session's weights: the host side of toy's
KV engine (lib/toy/llm/engine/llama_kv_engine.rb; SmolLM2KVStepResult.decode_step
:2350 takes one token at a position and returns the next token's logits,
decode_batch :2381 runs a prompt through it; enable_kv_q8! :359 keeps K and V
as Q8_0). The weights are those of a realised LlamaSeqEngine (after training,
or after load_gguf); every step is one graph replay on the GPU."""
from __future__ import annotations

import ctypes as C
from typing import Sequence

import numpy as np

from ._lib import check, lib


class KVDecoder:
    def __init__(self, engine, max_T: int, n_seq: int = 1, kv_q8: bool = False):
        self.eng = engine
        self.max_T, self.n_seq = max_T, n_seq
        self.vocab = engine.cfg.vocab
        check(lib().tb2_kv_realize(engine.sess, max_T, n_seq, 8 if kv_q8 else 0), "tb2_kv_realize")
        self._logits = np.empty((n_seq, self.vocab), np.float32)

    def reset(self) -> None:
        check(lib().tb2_kv_reset(self.eng.sess), "tb2_kv_reset")

    def decode_step(self, tokens: Sequence[int], positions: Sequence[int]) -> np.ndarray:
        """One token per sequence at its position; returns logits [n_seq, vocab]."""
        t = np.ascontiguousarray(np.asarray(tokens, np.int64).reshape(self.n_seq))
        p = np.ascontiguousarray(np.asarray(positions, np.int64).reshape(self.n_seq))
        check(lib().tb2_kv_decode(self.eng.sess, t.ctypes.data_as(C.POINTER(C.c_longlong)),
                                  p.ctypes.data_as(C.POINTER(C.c_longlong)), self.n_seq,
                                  self._logits.ctypes.data_as(C.POINTER(C.c_float))), "tb2_kv_decode")
        return self._logits.copy()

    def decode_batch(self, token_ids: np.ndarray, pos0: int = 0) -> np.ndarray:
        """Run [n_seq, n] prompt tokens through the cache from position pos0;
        returns the logits after every token, [n, n_seq, vocab]."""
        ids = np.asarray(token_ids, np.int64).reshape(self.n_seq, -1)
        return np.stack([self.decode_step(ids[:, i], np.full(self.n_seq, pos0 + i)) for i in range(ids.shape[1])])

    def generate(self, prompt: np.ndarray, n_new: int) -> np.ndarray:
        """Greedy continuation of [n_seq, n] prompts by n_new tokens each."""
        ids = np.asarray(prompt, np.int64).reshape(self.n_seq, -1)
        logits = self.decode_batch(ids)[-1]
        out = []
        pos = ids.shape[1]
        for _ in range(n_new):
            nxt = np.argmax(logits, axis=-1)
            out.append(nxt)
            logits = self.decode_step(nxt, np.full(self.n_seq, pos))
            pos += 1
        return np.stack(out, axis=1)

    def close(self) -> None:
        lib().tb2_kv_free(self.eng.sess)


_KV_TYPES = {"f32": 0, "f16": 1, "q8_0": 8, "bf16": 30}


class PagedKVDecoder:
    """Decode over a paged cache: up to n_seq sequences of unlike lengths share n_pages pages of page_size tokens
    (tb2_kv_*_paged). kv_type: "f32", "f16", "bf16" or "q8_0"."""

    def __init__(self, engine, max_T: int, n_seq: int, n_pages: int, page_size: int = 16, kv_type: str = "bf16"):
        if kv_type not in _KV_TYPES:
            raise ValueError(f"toy_b200: kv_type is one of {', '.join(_KV_TYPES)}, not {kv_type!r}")
        if max(max_T, n_seq, n_pages, page_size) >= 2**31:
            raise ValueError("toy_b200: max_T, n_seq, n_pages and page_size are below 2^31")
        self.eng = engine
        self.max_T, self.n_seq, self.n_pages, self.page_size = max_T, n_seq, n_pages, page_size
        self.vocab = engine.cfg.vocab
        check(lib().tb2_kv_realize_paged(engine.sess, max_T, n_seq, _KV_TYPES[kv_type], page_size, n_pages),
              "tb2_kv_realize_paged")
        self._logits = np.empty((n_seq, self.vocab), np.float32)

    def reset(self) -> None:
        check(lib().tb2_kv_reset(self.eng.sess), "tb2_kv_reset")

    def decode_step(self, tokens: Sequence[int]) -> np.ndarray:
        """tokens[b] appended to sequence b (-1: nothing); logits [n_seq, vocab] of the tokens after them. MemoryError
        when the pool has too few free pages: the step did nothing, and may be repeated after a release."""
        t = np.ascontiguousarray(np.asarray(tokens, np.int64).reshape(self.n_seq))
        rc = lib().tb2_kv_decode_paged(self.eng.sess, t.ctypes.data_as(C.POINTER(C.c_longlong)), self.n_seq,
                                       self._logits.ctypes.data_as(C.POINTER(C.c_float)))
        if rc == -5:
            raise MemoryError("toy_b200: no free pages for this decode step")
        check(rc, "tb2_kv_decode_paged")
        return self._logits.copy()

    def release(self, seqs: Sequence[int]) -> None:
        """Empty these sequences (0 .. n_seq - 1) and give their pages back."""
        at = np.asarray(seqs, np.int64).reshape(-1)
        if ((at < 0) | (at >= self.n_seq)).any():
            raise ValueError(f"toy_b200: sequences are 0 to {self.n_seq - 1}")
        d = np.zeros(self.n_seq, np.int32)
        d[at] = 1
        check(lib().tb2_kv_release(self.eng.sess, d.ctypes.data_as(C.POINTER(C.c_int)), self.n_seq), "tb2_kv_release")

    def state(self) -> tuple:
        """(lengths [n_seq], free pages)."""
        lens, free = np.zeros(self.n_seq, np.int32), C.c_int(0)
        check(lib().tb2_kv_paged_state(self.eng.sess, lens.ctypes.data_as(C.POINTER(C.c_int)), self.n_seq,
                                       C.byref(free)), "tb2_kv_paged_state")
        return lens, free.value

    def generate(self, prompts: Sequence[Sequence[int]], n_new: int) -> list:
        """Greedy continuations of prompts of any lengths (one per sequence, at least a token each) by n_new tokens. The
        sequences start empty, as KVDecoder.generate starts at position 0, and keep their prompt and continuation (but
        the last token) when it returns. ValueError or MemoryError, before anything is changed, where max_T or n_pages
        is too small for that."""
        feed = [list(map(int, p)) for p in prompts]
        if len(feed) != self.n_seq or any(not p for p in feed):
            raise ValueError("toy_b200: one prompt of a token or more per sequence")
        if any(t < 0 or t >= self.vocab for p in feed for t in p):
            raise ValueError(f"toy_b200: tokens are 0 to {self.vocab - 1}")
        if n_new < 1:
            return [[] for _ in feed]
        held = [len(p) + n_new - 1 for p in feed]
        if max(held) > self.max_T:
            raise ValueError(f"toy_b200: a prompt and {n_new} new tokens pass max_T ({self.max_T})")
        if sum(-(-h // self.page_size) for h in held) > self.n_pages:
            raise MemoryError(f"toy_b200: {self.n_pages} pages do not hold the prompts and {n_new} new tokens each")
        self.reset()
        out = [[] for _ in feed]
        at = [0] * self.n_seq
        while any(len(o) < n_new for o in out):
            toks = [feed[b][at[b]] if len(out[b]) < n_new else -1 for b in range(self.n_seq)]
            logits = self.decode_step(toks)
            for b in range(self.n_seq):
                if toks[b] < 0:
                    continue
                at[b] += 1
                if at[b] == len(feed[b]):
                    nxt = int(np.argmax(logits[b]))
                    out[b].append(nxt)
                    feed[b].append(nxt)
        return out

    def close(self) -> None:
        lib().tb2_kv_free(self.eng.sess)
