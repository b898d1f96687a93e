"""Prefill and greedy decode of a ``workloads.LlamaModel`` on the device: the
prefill graph, then decode steps, each one pass of the decode-step graph at
pos = T + i over the same KV-cache states, with the token chosen on the
device between them (``corm_greedy_embed``: the first argmax of each
sequence's logits and its embedding row as the next input) — the loop the
reference's host runs between its LLM entries (the prefill entry, then a
decode entry per token, with LlmDequant / argmax / LlmEmbed on the host).

``PagedLlamaRunner`` serves sequences of any lengths instead: prompts, chunks of
them and single tokens of several sequences in one pass over a paged KV cache
(no counterpart in the reference, which runs one sequence at a time).
"""
from __future__ import annotations

import threading
from contextlib import contextmanager
from typing import Dict, Hashable, List, Optional, Sequence

import numpy as np
import torch

from . import ops
from ._lib import CORM_EINVAL, CormError
from .paged import PagedBatch, PagedCache, PagePool
from .simulator import GpuSimulator


class LlamaRunner:
    def __init__(self, model, device=None, fuse: bool = True):
        self.m = model
        self.pre = GpuSimulator(model.prefill_graph, device=device, fuse=fuse)
        self.dec = GpuSimulator(model.decode_graph, device=self.pre.device, fuse=fuse, share=self.pre)
        self.device = self.pre.device
        self.states = self.pre.states_to_device()
        self.out_pre = model.prefill_graph.output_tensors[0].onnx_name
        self.out_dec = model.decode_graph.output_tensors[0].onnx_name
        emb = np.rint(model.emb * 2.0 ** model.E["fr"]).astype(np.int32)
        self.table = torch.from_numpy(emb).to(self.device)
        self.h = torch.empty(model.B * model.D + 4, dtype=torch.int32, device=self.device)
        self.raw_pre = None

    def prefill(self, feeds=None) -> torch.Tensor:
        """The prefill pass (lean: only the logits kept); returns the int16
        logits [B][vocab] on the device."""
        feeds = self.m.prefill_feeds if feeds is None else feeds
        if self.raw_pre is None:
            g = self.m.prefill_graph
            self.raw_pre = {t.onnx_name: (np.asarray(feeds[t.onnx_name]).astype(np.int64).reshape(-1) if t.host
                                          else self.pre._to_raw(t, feeds[t.onnx_name])) for t in g.input_tensors}
        res, _ = self.pre.forward_raw(self.raw_pre, keep=[self.out_pre], states=self.states)
        return res[self.out_pre]

    def decode_step(self, logits: torch.Tensor, i: int, ids: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Decode step i (pos = T + i) after ``logits``: the next tokens'
        embedding rows, then one decode-step pass; returns its logits."""
        m = self.m
        ops.greedy_embed(logits, self.table, self.h, ids, batch=m.B, vocab=m.vocab, dim=m.D)
        res, _ = self.dec.forward_raw({"h_step": self.h, "pos": np.array([m.T + i])}, keep=[self.out_dec],
                                      states=self.states)
        return res[self.out_dec]

    def generate(self, steps: int) -> List[np.ndarray]:
        """Prefill then ``steps`` greedy steps; returns the token ids chosen
        before every step ([B] each)."""
        lg = self.prefill()
        ids = torch.empty((steps, self.m.B), dtype=torch.int32, device=self.device)
        for i in range(steps):
            lg = self.decode_step(lg, i, ids[i])
        self.last_logits = lg
        return [r for r in ids.cpu().numpy()]


class PagedLlamaRunner:
    """Passes of a ``workloads.LlamaModel`` over a paged KV cache of ``pages``
    pages of ``page`` rows (``bits`` 16 or 8) a layer.  A sequence is any hashable
    name; it comes into being with its first tokens and holds its pages until
    ``release``.  Every pass takes the unit's softmax, a prompt's and a single
    token's alike, so at 16 bits a token's words do not depend on how its sequence
    was cut into passes nor on what ran beside it (with 8 bits nor do they: a row's
    codes are its own).  Calls from several threads take turns, and passes on
    different streams follow one another on the device."""

    GRAPHS = 64  # graphs kept, the last used (one of 32 layers: 1.1 MB of the host's memory, 0.1 s to build)

    def __init__(self, model, pages: int, page: int = 64, bits: int = 16, device=None, fuse: bool = True):
        self.m, self.fuse = model, fuse
        self.device = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        self.caches = [PagedCache(pages, page, model.KV, model.HD, bits, device=self.device) for _ in range(model.L)]
        self.pool = PagePool(pages, page)
        self.length: Dict[Hashable, int] = {}
        emb = np.rint(model.emb * 2.0 ** model.E["fr"]).astype(np.int32)
        self.table = torch.from_numpy(emb).to(self.device)
        self._sims: Dict[tuple, GpuSimulator] = {}
        self._share: Optional[GpuSimulator] = None
        self._ws: Optional[torch.Tensor] = None
        self._lock = threading.RLock()
        # the last pass, and its stream
        self._done = torch.cuda.Event() if self.device.type == "cuda" else None
        self._stream: Optional[int] = None

    @contextmanager
    def _turn(self, *used: Optional[torch.Tensor]):
        """One call at a time, its device work behind the last call's: they share the
        pool, the pages, the weights and the simulators.  used: the caller's tensors,
        perhaps another stream's."""
        with self._lock:
            if self._done is None:
                yield
                return
            stream = torch.cuda.current_stream(self.device)
            stream.wait_event(self._done)
            if stream.cuda_stream != self._stream:  # a workspace stays with the stream that it was allocated on
                self._stream, self._ws = stream.cuda_stream, None
            for t in used:
                if t is not None and t.is_cuda:
                    t.record_stream(stream)
            try:
                yield
            finally:
                self._done.record(stream)

    def _sim(self, rows: int, head: bool) -> GpuSimulator:
        key = (rows, head)
        s = self._sims.pop(key, None)
        if s is None:
            g = self.m.head_graph(rows) if head else self.m.paged_graph(rows)
            s = GpuSimulator(g, device=self.device, fuse=self.fuse, share=self._share)
            self._share = self._share or s
            while len(self._sims) >= self.GRAPHS:
                del self._sims[next(iter(self._sims))]
        self._sims[key] = s  # (the last used last)
        return s

    def _run(self, sim: GpuSimulator, h: torch.Tensor) -> torch.Tensor:
        """A graph's output rows of the residual rows h, in the workspace of all."""
        out = sim._graph.output_tensors[0].onnx_name
        sim._ws = self._ws
        try:
            return sim.forward_raw({"h_step": h}, keep=[out])[0][out]
        finally:
            self._ws, sim._ws, sim.paged = sim._ws, None, None

    @staticmethod
    def _padded(rows: int) -> int:
        """The rows a pass is built for: graphs of few row counts serve all."""
        return rows if rows <= 16 else -(-rows // 64) * 64

    def _room(self, seqs: Sequence[Hashable], new: Sequence[int]) -> List[int]:
        """The positions of the sequences' next rows; an error where a pass over
        ``new`` rows of each cannot be made."""
        m = self.m
        at = [self.length.get(s, 0) for s in seqs]
        if len(set(seqs)) != len(seqs) or not seqs or min(new) < 1:
            raise CormError(CORM_EINVAL, "PagedLlamaRunner: distinct sequences with a token or more each expected")
        for s, a, n in zip(seqs, at, new):
            if a + n > m.C:
                raise CormError(CORM_EINVAL, f"PagedLlamaRunner: sequence {s!r}: {a + n} positions, the model has {m.C}")
        need = sum(max(-(-(a + n) // self.pool.page) - len(self.pool.held.get(s, [])), 0) for s, a, n in zip(seqs, at, new))
        if need > len(self.pool.free):
            raise MemoryError(f"PagedLlamaRunner: {need} pages wanted, {len(self.pool.free)} free (no sequence changed)")
        return at

    def _pass(self, seqs: Sequence[Hashable], new: Sequence[int], at: Sequence[int], h: torch.Tensor) -> torch.Tensor:
        """The layers over h (int32, the new rows packed; whole padded rows), the
        last row of every sequence through the head: its logits.  at: ``_room``'s."""
        m = self.m
        tables = [self.pool.extend(s, a + n) for s, a, n in zip(seqs, at, new)]
        batch = PagedBatch.of(tables, new, at, device=self.device)
        sim = self._sim(self._padded(batch.rows), False)
        sim.paged = (self.caches, batch)
        out = self._run(sim, h)
        B = len(seqs)
        last = torch.empty(B * m.D + 4, dtype=torch.int32, device=self.device)
        rows = out[:batch.rows * m.D].view(batch.rows, m.D)
        torch.index_select(rows, 0, batch.cu[1:] - 1, out=last[:B * m.D].view(B, m.D))
        logits = self._run(self._sim(B, True), last)
        self.length.update({s: a + n for s, a, n in zip(seqs, at, new)})
        return logits

    def _rows(self, rows: int) -> torch.Tensor:
        return torch.zeros(self._padded(rows) * self.m.D + 4, dtype=torch.int32, device=self.device)

    def append(self, seqs: Sequence[Hashable], ids: Sequence[Sequence[int]]) -> torch.Tensor:
        """One pass over new tokens of some sequences (prompts, chunks, single
        tokens together): int16 logits [len(seqs)][vocab] of their last ones."""
        tokens = [np.asarray(i, np.int64) for i in ids]
        if len(tokens) != len(seqs) or any(t.ndim != 1 for t in tokens):
            raise CormError(CORM_EINVAL, f"PagedLlamaRunner: a list of tokens for each of {len(seqs)} sequences expected, got "
                                         f"{[t.shape for t in tokens]}")
        new = [t.size for t in tokens]
        flat = np.concatenate(tokens) if new else np.zeros(0, np.int64)
        if flat.size and (flat.min() < 0 or flat.max() >= self.m.vocab):
            raise CormError(CORM_EINVAL, f"PagedLlamaRunner: token ids in [0, {self.m.vocab}) expected")
        with self._turn():
            at = self._room(seqs, new)
            h, n = self._rows(flat.size), flat.size * self.m.D
            torch.index_select(self.table, 0, torch.from_numpy(flat).to(self.device), out=h[:n].view(flat.size, self.m.D))
            return self._pass(seqs, new, at, h)

    def step(self, seqs: Sequence[Hashable], logits: torch.Tensor, ids: Optional[torch.Tensor] = None) -> torch.Tensor:
        """A greedy token for each of ``seqs`` after ``logits`` (their order),
        chosen on the device (int32 ``ids`` if given); its logits."""
        new = [1] * len(seqs)
        with self._turn(logits, ids):
            at = self._room(seqs, new)  # (before ids is written)
            h = self._rows(len(seqs))
            ops.greedy_embed(logits, self.table, h, ids, batch=len(seqs), vocab=self.m.vocab, dim=self.m.D)
            return self._pass(seqs, new, at, h)

    def generate(self, prompts: Dict[Hashable, Sequence[int]], steps: int) -> Dict[Hashable, List[int]]:
        """The prompts in one pass, then ``steps`` greedy tokens of each."""
        seqs = list(prompts)
        lg = self.append(seqs, [prompts[s] for s in seqs])
        ids = torch.empty((steps, len(seqs)), dtype=torch.int32, device=self.device)
        for i in range(steps):
            lg = self.step(seqs, lg, ids[i])
        self.last_logits = lg
        return dict(zip(seqs, ids.cpu().numpy().T.tolist()))

    def release(self, seq: Hashable) -> None:
        """Ends a sequence; its pages are free."""
        with self._lock:
            self.pool.release(seq)
            self.length.pop(seq, None)
