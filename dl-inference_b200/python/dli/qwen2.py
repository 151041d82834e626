"""Greedy generation over a Qwen2 graph exported by dli_export.qwen2.

Qwen2Runner drives one tensor-parallel rank: it binds the weights to the
engine once (Engine.set_constants), runs prefill through Engine.run, and
replays the decode step from a captured CUDA graph. Token ids and positions
stay on the device between steps: each decode step writes the argmax ids and
advances the positions inside the graph's static input buffers.

With `page_size` the KV cache is a pool of pages (16-bit, or 4-bit with
kv_dtype="fp4") instead of a row of `capacity` tokens per sequence: the runner
holds one set of sequences, opened with the rows they need (`open`, `extend`,
`close`; prefill and generate open theirs), and a page table per batch size that
stays at its address, so captured decode steps follow its contents.
"""
from __future__ import annotations

import contextlib
import json
from typing import Any

import torch

from . import PLUGIN_PATH, Engine, Graph
from .pages import PagePool


class Qwen2Runner:
    def __init__(self, shape: Any, weights: dict[str, torch.Tensor], capacity: int,
                 tp_size: int = 1, tp_rank: int = 0, communicator: int = 0,
                 plugin: str = PLUGIN_PATH, fused_glu: bool = True, fused_exchange: bool = True,
                 page_size: int = 0, num_pages: int = 0, kv_dtype: str | None = None):
        """`weights` come from dli_export.qwen2.transform_weights with the same
        `fused_glu` (the fused SwiGLU GEMM serves bfloat16/float16 weights).
        `fused_exchange`: tensor-parallel projections push their partial rows
        from the GEMM epilogue (linear_all_reduce_add_rms_norm nodes).
        `page_size`, `num_pages`, `kv_dtype`: a paged cache, where `capacity` is the
        most rows that one sequence may have."""
        from dli_export.qwen2 import build_graph, rotary_tables

        self.shape = shape
        self.capacity = capacity
        self.device = next(iter(weights.values())).device
        self.dtype = weights["layers.0.wqkv"].dtype
        self.engine = Engine()
        self.engine.load_library(plugin)
        if tp_size > 1:
            self.engine.set_communicator(communicator, tp_rank, tp_size)
        self.pool = PagePool(num_pages, page_size) if page_size else None
        # one page more than the pool's: warm-up steps write and read only that
        self.graph = Graph.from_json(json.dumps(build_graph(
            shape, capacity, tp_size, fused_glu=fused_glu, fused_exchange=fused_exchange, page_size=page_size,
            num_pages=num_pages + 1 if page_size else num_pages, kv_dtype=kv_dtype)))
        self.sequences: list[list[int]] = []  # pages of the open sequences
        self._tables: dict[int, torch.Tensor] = {}
        consts = dict(weights)
        if "rotary_cos" not in consts:
            cos, sin = rotary_tables(shape, capacity)
            consts["rotary_cos"], consts["rotary_sin"] = cos.to(self.device), sin.to(self.device)
        self.engine.set_constants(consts)
        self._graphs: dict[int, tuple] = {}

    # -- plain engine calls -------------------------------------------------------
    def forward(self, input_ids: torch.Tensor, positions: torch.Tensor, profile=None):
        """input_ids [B,S] int64, positions [B] int64 (cache row of the first token).
        Returns (logits of the last token, next ids). With tensor parallelism over a
        vocabulary that divides evenly, the logits are this rank's slice of the
        vocabulary (ids [rank*V/tp, (rank+1)*V/tp)); the next ids are global.
        `profile` (a dli.ProfileSession) times every node of the run. A paged cache
        needs as many open sequences as input_ids has, with pages for the new rows."""
        if self.pool is not None and len(self.sequences) != input_ids.shape[0]:
            raise ValueError(f"{len(self.sequences)} sequences are open, {input_ids.shape[0]} called for")
        return self._step(input_ids, positions, profile)

    def _step(self, input_ids, positions, profile=None):
        inputs = {"input_ids": input_ids, "positions": positions}
        if self.pool is not None:
            inputs["page_table"] = self.page_table(input_ids.shape[0])
        out = self.engine.run(self.graph, inputs, profile=profile)
        return out["logits"], out["next_ids"]

    # -- sequences of a paged cache -----------------------------------------------------
    def page_table(self, batch: int) -> torch.Tensor:
        """The device page table [batch, max_pages] of the open sequences; entries
        without a page are -1, which the kernels report and do not follow."""
        if batch not in self._tables:
            width = self.pool.pages_for(self.capacity)
            self._tables[batch] = torch.full((batch, width), -1, dtype=torch.int32, device=self.device)
        return self._tables[batch]

    def _write_table(self) -> None:
        table = self.page_table(len(self.sequences))
        rows = [p + [-1] * (table.shape[1] - len(p)) for p in self.sequences]
        table.copy_(torch.tensor(rows, dtype=torch.int32))

    def open(self, rows: list[int]) -> None:
        """Closes the open sequences and opens one per element, with pages for that
        many rows. Raises MemoryError when the pool has too few pages."""
        if self.pool is None:
            raise ValueError("open: the cache is not paged")
        if not rows or any(r < 0 or r > self.capacity for r in rows):
            raise ValueError("open: between 0 and capacity rows per sequence")
        self.close()
        sequences: list[list[int]] = [[] for _ in rows]
        self.pool.grow(sequences, rows)
        self.sequences = sequences
        self._write_table()

    def extend(self, rows: list[int]) -> None:
        """Gives the open sequences pages until they hold rows[i] rows each; what they
        have cached stays."""
        if self.pool is None or len(rows) != len(self.sequences):
            raise ValueError("extend: one row count per open sequence")
        if any(r < 0 or r > self.capacity for r in rows):
            raise ValueError("extend: between 0 and capacity rows per sequence")
        self.pool.grow(self.sequences, rows)
        self._write_table()

    def close(self) -> None:
        """Returns the open sequences' pages to the pool."""
        if self.sequences:
            self.page_table(len(self.sequences)).fill_(-1)
        for pages in self.sequences:
            self.pool.give_back(pages)
        self.sequences = []

    def cached_rows(self, layer: int, count: int):
        """(k, v), each [B, kv_heads, count, head_dim] of the model's dtype: the first
        `count` cached rows of every sequence in a layer."""
        k, v, _ = self.engine.kv_cache_entry(f"layer_{layer}")
        if self.pool is None:
            return k[:, :, :count], v[:, :, :count]
        if not self.sequences:
            raise ValueError("cached_rows: no open sequences")
        import dli_sm100

        return dli_sm100.paged_gather(k, v, self.page_table(len(self.sequences)), count, self.shape.head_dim, self.dtype)

    def check_device_error(self) -> None:
        """Raises RuntimeError when a kernel of this process reported an error
        through the device error word: a bounded wait that ran out (a
        tensor-parallel peer that never arrived, a tensor-core pipeline stall) or
        an out-of-range id or position. Such a kernel returns early, so the
        outputs of the run are not valid. Synchronises the current stream. After
        an exchange timeout every rank must reset its exchange buffer
        (dli_sm100_tp_exchange_reset) before the group runs again."""
        import dli_sm100

        dli_sm100.check_device_error()

    def reset(self) -> None:
        """Forgets cached sequences (rows are rewritten by position, so nothing to clear);
        the pages of a paged cache return to the pool."""
        self.engine.kv_cache_reset()
        self.close()

    # -- CUDA-graph decode ----------------------------------------------------------
    def profile_decode_step(self, batch: int, profile) -> None:
        """Captures one decode step with every node between CUDA-event markers,
        replays it once and leaves the session holding that replay's per-node
        device times (call profile.finalize() next). The step runs at the last
        cache row, like the warm-up of the decode graph, so live sequences are
        not disturbed. The markers make the step slower than the decode graph."""
        ids = torch.zeros(batch, 1, dtype=torch.int64, device=self.device)
        pos = torch.full((batch,), self.capacity - 1, dtype=torch.int64, device=self.device)
        with self._on_spare_page(batch):
            self._warm_up(ids, pos, 1)
            profile.reserve(len(self.graph.node_ops()))
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                self._step(ids, pos, profile=profile)
            g.replay()
        torch.cuda.synchronize(self.device)
        del g

    @contextlib.contextmanager
    def _on_spare_page(self, batch: int):
        """Points a paged cache's table at the page outside the pool, for steps whose
        rows nobody reads, and back when they are done or have failed. All sequences of
        such a step write the same row of that page with the same values."""
        if self.pool is None:
            yield
            return
        held = self.page_table(batch).clone()
        self.page_table(batch).fill_(self.pool.num_pages)
        try:
            yield
        finally:
            self.page_table(batch).copy_(held)

    def _warm_up(self, ids: torch.Tensor, pos: torch.Tensor, steps: int) -> None:
        stream = torch.cuda.Stream(self.device)
        stream.wait_stream(torch.cuda.current_stream(self.device))
        try:
            with torch.cuda.stream(stream):
                for _ in range(steps):
                    self._step(ids, pos)
        finally:
            torch.cuda.current_stream(self.device).wait_stream(stream)

    def _capture(self, batch: int):
        # Warm-up and capture write one cache row per sequence; the last row is only
        # read after a later step has rewritten it, so live sequences are not disturbed.
        ids = torch.zeros(batch, 1, dtype=torch.int64, device=self.device)
        pos = torch.full((batch,), self.capacity - 1, dtype=torch.int64, device=self.device)
        with self._on_spare_page(batch):
            self._warm_up(ids, pos, 2)  # the caching allocator and per-kernel attributes
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            logits, next_ids = self._step(ids, pos)
            ids.copy_(next_ids.view(batch, 1))
            pos.add_(1)
        self._graphs[batch] = (g, ids, pos, logits, next_ids)
        return self._graphs[batch]

    def decode_graph(self, batch: int):
        return self._graphs.get(batch) or self._capture(batch)

    def release_graphs(self) -> None:
        """Drops the captured decode graphs. A graph captured with tensor
        parallelism holds NCCL launches on the runner's communicator: release it
        before that communicator (or the process group) is destroyed."""
        torch.cuda.synchronize(self.device)
        self._graphs.clear()

    def prefill(self, prompt: torch.Tensor, start: torch.Tensor | None = None):
        """prompt [B,S] on the device; returns (logits of the last token, next ids)."""
        b, s = prompt.shape
        if self.pool is not None and start is None:
            self._hold(b, s)
        if start is None:
            start = torch.zeros(b, dtype=torch.int64, device=self.device)
        return self.forward(prompt, start)

    def _hold(self, batch: int, rows: int) -> None:
        """Pages for `rows` rows of each of `batch` sequences, opened if others are."""
        if len(self.sequences) != batch:
            self.open([rows] * batch)
        else:
            self.extend([rows] * batch)

    def generate(self, prompt: torch.Tensor, steps: int, use_graph: bool = True) -> torch.Tensor:
        """Greedy decoding: returns [B, steps] device ids (the first from prefill)."""
        b, s = prompt.shape
        if s + steps > self.capacity:
            raise ValueError("prompt + steps exceeds the KV-cache capacity")
        if self.pool is not None:
            self._hold(b, s + steps)
        out = torch.empty(b, steps, dtype=torch.int64, device=self.device)
        _, nxt = self.prefill(prompt)
        out[:, 0] = nxt
        if steps == 1:
            return out
        if use_graph:
            g, ids, pos, _, next_ids = self.decode_graph(b)
            ids.copy_(nxt.view(b, 1))
            pos.fill_(s)
            for t in range(1, steps):
                g.replay()
                out[:, t] = next_ids
        else:
            ids = nxt.view(b, 1)
            pos = torch.full((b,), s, dtype=torch.int64, device=self.device)
            for t in range(1, steps):
                _, nxt = self.forward(ids, pos)
                out[:, t] = nxt
                ids = nxt.view(b, 1)
                pos = pos + 1
        self.check_device_error()
        return out
