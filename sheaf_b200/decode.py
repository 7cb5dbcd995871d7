"""GPT decoding over key/value caches with the runtime's decoding operators.

`CachedDecoder` runs the model of sheaf_lowering.models (examples/nanoGPT/
model.shf) on a batch of sequences, one or several tokens per call: per layer
the keys and values go into the cache (`kv_cache_write`) and the attention
reads them there (`kv_cache_attention`), between the lowered programs of
`gpt_cached_programs`.  `beam_search` adds `beam_select` and `beam_reorder`.
"""
from __future__ import annotations

from typing import Dict, List, Optional, Sequence, Tuple

import numpy as np

from sheaf_lowering import generate as G
from sheaf_lowering import models as M

from .session import B200Error, B200Session, DeviceBuffer

MAX_TOKENS = 64  # tokens per slot and call (sb_kv_cache_attention)


class CachedDecoder:
    """`slots` sequences of up to `c.block_size` positions; `params` maps the
    names of `gpt_param_leaves` to host arrays (uploaded once) or device buffers;
    `dtype` is the caches' type: "f32", "bf16" or "int8"."""

    def __init__(self, session: B200Session, c: M.GPTConfig, params: Dict[str, object], slots: int,
                 dtype: str = "f32"):
        self.session, self.c, self.slots = session, c, slots
        self.params = {n: session.buffer(params[n]) if isinstance(params[n], np.ndarray) else params[n]
                       for n, _ in M.gpt_param_leaves(c)}
        self.caches = [session.kv_cache(slots, c.n_head, c.block_size, c.n_embd // c.n_head, dtype)
                       for _ in range(c.n_layer)]
        self._programs: Dict[int, List[tuple]] = {}

    def _load(self, tokens: int):
        if not 1 <= tokens <= MAX_TOKENS:
            raise B200Error(3, f"a call takes 1 to {MAX_TOKENS} tokens per slot, not {tokens}")
        if tokens not in self._programs:
            progs = G.gpt_cached_programs(self.c, self.slots, tokens)
            for p in progs.values():
                if not self.session.has_function(p.qualified):
                    self.session.load_stablehlo(p.text)
            # each program with its weights: start, one per layer but the last, logits
            last = self.c.n_layer - 1
            low = [progs["start"]] + [progs["layer"]] * last + [progs["logits"]]
            self._programs[tokens] = [(p.qualified, self._weights(p, i - 1, i)) for i, p in enumerate(low)]
        return self._programs[tokens]

    def _weights(self, low, done: int, nxt: int) -> List[DeviceBuffer]:
        """The weights among a program's arguments: those of layers `done` and `nxt`, and the shared ones."""
        names = (n.replace("done.", f"transformer.h.{done}.").replace("next.", f"transformer.h.{nxt}.")
                 for n in low.arg_names)
        return [self.params[n] for n in names if n in self.params]

    def forward(self, tokens, positions: Sequence[int], parents: Optional[np.ndarray] = None,
                logits: bool = True) -> Optional[DeviceBuffer]:
        """The tokens [slots, S] (host or device, f32 ids) at positions
        positions[n] + t into the caches; returns their logits [slots * S, V]
        (logits=False: None).  With `parents` [slots, S] they are a tree of
        drafted tokens after the positions before positions[n]: token t then
        stands at place positions[n] + its depth in the tree, and sees its
        ancestors alone.  A slot with a negative position is idle."""
        sess, N = self.session, self.slots
        S = tokens.shape[-1]
        if tuple(tokens.shape) != (N, S):
            raise B200Error(3, f"tokens are [{N}, S], not {tuple(tokens.shape)}")
        progs = self._load(S)
        pos = np.asarray(positions, np.int64)
        if pos.shape != (N,) or (pos + S > self.c.block_size).any():
            raise B200Error(3, f"positions are [{N}] and end within the {self.c.block_size} of the model")
        pos = np.maximum(pos, -1).astype(np.int32)
        depth = np.tile(np.arange(S, dtype=np.int32), (N, 1))
        tree = None
        if parents is not None:
            parents = np.asarray(parents, np.int32)
            if parents.shape != (N, S):
                raise B200Error(3, f"parents are [{N}, {S}]")
            for t in range(S):
                up = parents[:, t]
                has = (up >= 0) & (up < t)
                depth[:, t] = np.where(has, depth[np.arange(N), np.where(has, up, 0)] + 1, 0)
            tree = sess.buffer(parents)
        place = sess.buffer(np.maximum(pos[:, None] + depth, 0).astype(np.float32))
        at = sess.buffer(pos)
        token = sess.buffer(tokens.astype(np.float32)) if isinstance(tokens, np.ndarray) else tokens
        name, weights = progs[0]
        x, q, k, v = sess.call_device(name, weights + [token, place])
        y = sess.zeros(q.shape)
        for cache, (name, weights) in zip(self.caches, progs[1:]):
            sess.kv_cache_write(cache, at, k, v)
            sess.kv_cache_attention(cache, at, q, y, parents=tree)
            if cache is not self.caches[-1]:
                x, q, k, v = sess.call_device(name, weights + [x, y])
        return sess.call_device(name, weights + [x, y])[0] if logits else None

    def prompt(self, tokens: np.ndarray, chunk: int = MAX_TOKENS):
        """The tokens [slots, P] of a prompt into the caches, from position 0."""
        tokens = np.asarray(tokens, np.float32)
        for p in range(0, tokens.shape[1], chunk):
            self.forward(tokens[:, p:p + chunk], np.full(self.slots, p), logits=False)

    def beam_search(self, prompt: np.ndarray, beams: int, steps: int,
                    eos: int = -1) -> Tuple[np.ndarray, np.ndarray]:
        """The `beams` best continuations of each prompt [groups, P] (P >= 1) by
        `steps` tokens, found by beam search: (tokens [groups, beams, steps],
        scores [groups, beams]), best first.  groups * beams = slots.  The caches
        follow the beams on the device; the host reads the result alone."""
        sess, N, c = self.session, self.slots, self.c
        groups, P = prompt.shape
        if groups * beams != N or P < 1 or steps < 1 or P + steps - 1 > c.block_size:
            raise B200Error(3, f"{groups} prompts of {P} tokens and {beams} beams for {steps} steps do not fit "
                               f"{N} slots of {c.block_size} positions")
        tp = G.token_program(groups, beams)
        if not sess.has_function(tp.qualified):
            sess.load_stablehlo(tp.text)
        each = np.repeat(np.asarray(prompt, np.float32), beams, axis=0)
        self.prompt(each[:, :-1])
        first = np.full((groups, beams), -np.inf, np.float32)
        first[:, 0] = 0.0  # the beams of a group hold the same prefix: one of them counts
        scores = sess.buffer(first)
        finished = sess.zeros((groups, beams), "i32") if eos >= 0 else None
        token = sess.buffer(each[:, -1:])
        states = [b for cache in self.caches for b in cache.buffers()]
        history = []
        for i in range(steps):
            logits = self.forward(token, np.full(N, P - 1 + i))
            parents, chosen = (sess.zeros((groups, beams), "i32") for _ in range(2))
            sess.beam_select(logits, scores, scores, parents, chosen, finished=finished, out_finished=finished,
                             eos=eos)
            history.append((parents, chosen))
            if i + 1 < steps:
                live = sess.buffer(np.full(N, P + i, np.int32))
                sess.beam_reorder(states, parents, [2] * len(states), lengths=live)
                token = sess.call_device(tp.qualified, [chosen])[0]
        out = np.empty((groups, beams, steps), np.int32)
        row = np.tile(np.arange(beams), (groups, 1))
        for i in reversed(range(steps)):  # from the last selection back to the first
            parents, chosen = (b.to_host() for b in history[i])
            out[:, :, i] = np.take_along_axis(chosen, row, 1)
            row = np.take_along_axis(parents, row, 1)
        return out, scores.to_host()

    def release(self):
        for cache in self.caches:
            cache.release()
