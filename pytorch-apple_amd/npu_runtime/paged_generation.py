"""Generation of many sequences at once over paged caches: chunked prompts, batched decoding, sampling.

Runs the step graph of ``irgen.qwen.build_paged_ir`` (any graph with its inputs and outputs). Each step packs the next
token of every decoding sequence and as much of the waiting prompts as its rows hold; sequences take their slot and
pages when they start and give them back when they end, so a batch of prompts may be larger than the graph's slots or
the pool. A second, smaller graph over the same pools, one row per slot, takes the steps that only decode.

The pools stay on the device and are updated in place; the tokens of a step are read back, since they decide what the
next step holds. A sequence's uniform numbers come from its own generator, seeded with (seed, its index among the
prompts), so its tokens do not depend on which others share its steps beyond the rounding of the model itself.
"""

from __future__ import annotations

from dataclasses import dataclass

import numpy as np
import torch

_TORCH = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
_BATCH = ("block_table", "q_start", "kv_len", "last_rows", "temperature", "top_k", "top_p", "min_p", "u")


@dataclass(frozen=True)
class SamplingParams:
    """``serving.sample``'s parameters: ``temperature`` 0 takes the likeliest token; ``top_k`` 0, ``top_p`` 1 and
    ``min_p`` 0 cut nothing."""
    temperature: float = 1.0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0
    seed: int = 0


@dataclass
class _Sequence:
    index: int
    tokens: list[int]        # prompt, then what was generated
    prompt_len: int
    params: SamplingParams
    rng: np.random.Generator
    slot: int = -1
    pages: list[int] | None = None
    cached: int = 0          # tokens whose keys and values are in the pages


def _shapes(ir: dict) -> dict:
    return {s["name"]: (tuple(s["shape"]), s["dtype"]) for s in ir["graph_inputs"]}


class PagedGenerator:
    """``step`` (and ``decode``, a graph of one row per slot, if given) run by ``DAGExecutor`` s on ``backend``, or by
    all-CPU plans with ``backend=None``. A ``decode`` of as many rows as ``step`` has nothing to save and is not run."""

    def __init__(self, step, step_ir: dict, decode=None, decode_ir: dict | None = None, backend=None):
        shapes = _shapes(step_ir)
        missing = [n for n in ("input_ids", *_BATCH) if n not in shapes]
        if missing:
            raise ValueError(f"not a paged step graph: it has no input {missing}")
        self.backend = backend
        self.pool_names = [n for n in shapes if n not in ("input_ids", *_BATCH)]
        self.shapes = shapes
        self.slots, self.table_pages = shapes["block_table"][0]
        if not self.pool_names:
            raise ValueError("not a paged step graph: it has no page pools")
        layouts = {n["attrs"].get("page_layout", "hnd") for ir in (step_ir, decode_ir) if ir is not None
                   for n in ir["nodes"] if n["op_type"] in ("serving.paged_append.default", "serving.paged_attention.default")}
        if len(layouts) != 1:
            raise ValueError(f"not graphs of one page_layout: {sorted(layouts)}")
        dims = shapes[self.pool_names[0]][0]
        self.pages, self.page_size = dims[0], dims[2 if layouts == {"hnd"} else 1]
        self.graphs = []   # (executor, rows, output names) of decode, if it is run, and step: no two of the same rows
        for dag, ir in ((decode, decode_ir), (step, step_ir)):
            if dag is None and ir is None:
                continue
            got = _shapes(ir)
            rows = got.pop("input_ids")[0][0]
            if got != {n: s for n, s in shapes.items() if n != "input_ids"}:
                raise ValueError("the decode graph's slots and pools are not the step graph's")
            if rows < self.slots:
                raise ValueError(f"a graph of {rows} rows for {self.slots} slots: every slot needs a row")
            self.graphs.append((dag, rows, [o["name"] for o in ir["graph_outputs"]]))
        if len(self.graphs) == 2 and self.graphs[0][1] == self.graphs[1][1]:
            del self.graphs[0]
        self._bufs: dict = {}
        self._written: dict = {}
        self._moved: dict = {}

    # -- buffers ---------------------------------------------------------------------------

    def _input(self, key, arr: np.ndarray):
        """The buffer of a graph input, written only where its contents changed."""
        if self.backend is None:
            return arr.copy()
        if key not in self._bufs:
            self._bufs[key] = self.backend.allocate_buffer(arr.copy())
        elif not np.array_equal(self._written[key], arr):
            self._bufs[key].write_from_numpy(arr)
        self._written[key] = arr.copy()
        return self._bufs[key]

    def _pools(self) -> dict:
        if "pools" not in self._bufs:
            zeros = {n: torch.zeros(self.shapes[n][0], dtype=_TORCH[self.shapes[n][1]]) for n in self.pool_names}
            if self.backend is not None:
                zeros = {n: self.backend.allocate_buffer(t) for n, t in zeros.items()}
            else:
                zeros = {n: t.view(torch.uint16).numpy() if t.dtype == torch.bfloat16 else t.numpy()
                         for n, t in zeros.items()}
            self._bufs["pools"] = zeros
        return self._bufs["pools"]

    # -- generation ------------------------------------------------------------------------

    def generate(self, prompts, max_tokens: int, sampling: SamplingParams | list[SamplingParams] | None = None,
                 eos_token_id: int | None = None) -> list[list[int]]:
        """Up to ``max_tokens`` tokens after each of ``prompts`` (lists of ids), without the EOS token."""
        sampling = SamplingParams() if sampling is None else sampling
        per = list(sampling) if isinstance(sampling, (list, tuple)) else [sampling] * len(prompts)
        if len(per) != len(prompts):
            raise ValueError(f"{len(per)} sampling parameters for {len(prompts)} prompts")
        if max_tokens < 1:
            raise ValueError(f"max_tokens must be at least 1, got {max_tokens}")
        most = min(self.table_pages, self.pages) * self.page_size
        waiting = []
        for i, (prompt, p) in enumerate(zip(prompts, per)):
            ids = [int(t) for t in prompt]
            if not ids or len(ids) + max_tokens - 1 > most:
                raise ValueError(f"prompt {i}: {len(ids)} tokens and {max_tokens} more, and a sequence holds 1 to {most}")
            waiting.append(_Sequence(i, ids, len(ids), p, np.random.default_rng([p.seed, i])))
        done: list[list[int] | None] = [None] * len(prompts)
        waiting.reverse()
        free_pages, free_slots = list(range(self.pages))[::-1], list(range(self.slots))[::-1]
        table = np.zeros((self.slots, self.table_pages), np.int32)
        par = {"temperature": np.zeros(self.slots, np.float32), "top_k": np.zeros(self.slots, np.int32),
               "top_p": np.ones(self.slots, np.float32), "min_p": np.zeros(self.slots, np.float32)}
        running: dict[int, _Sequence] = {}
        while waiting or running:
            while waiting and free_slots:   # in order: a sequence starts once its whole length has pages
                s = waiting[-1]
                need = -(-(s.prompt_len + max_tokens - 1) // self.page_size)
                if need > len(free_pages):
                    break
                waiting.pop()
                s.slot, s.pages = free_slots.pop(), [free_pages.pop() for _ in range(need)]
                table[s.slot, :need] = s.pages
                for name, v in par.items():
                    v[s.slot] = getattr(s.params, name)
                running[s.slot] = s
            for s in self._step(running, table, par):
                new = s.tokens[s.prompt_len:]
                ended = eos_token_id is not None and new[-1] == eos_token_id
                if ended or len(new) == max_tokens:
                    done[s.index] = new[:-1] if ended else new
                    del running[s.slot]
                    free_slots.append(s.slot)
                    free_pages += s.pages[::-1]
        return done

    def _step(self, running: dict[int, _Sequence], table: np.ndarray, par: dict) -> list[_Sequence]:
        """One step of the running sequences; those that got a token."""
        n = np.zeros(self.slots, np.int64)
        for slot, s in running.items():
            n[slot] = min(len(s.tokens) - s.cached, 1)   # every sequence a row, ...
        if any(len(s.tokens) - s.cached > 1 for s in running.values()):
            dag, rows, outputs = self.graphs[-1]
            for slot, s in sorted(running.items(), key=lambda kv: kv[1].index):   # ... then the prompts, first come
                n[slot] += min(len(s.tokens) - s.cached - n[slot], rows - n.sum())
        else:
            dag, rows, outputs = self.graphs[0]
        ids = np.zeros(rows, np.int64)
        start = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
        kv = np.zeros(self.slots, np.int32)
        last = np.zeros(self.slots, np.int64)
        u = np.zeros(self.slots, np.float32)
        drawn = []
        for slot, s in running.items():
            k = int(n[slot])
            ids[start[slot]:start[slot + 1]] = s.tokens[s.cached:s.cached + k]
            s.cached += k
            kv[slot], last[slot] = s.cached, start[slot + 1] - 1
            if s.cached == len(s.tokens):
                u[slot] = s.rng.random(dtype=np.float32)
                drawn.append(s)
        feed = {"input_ids": self._input(("input_ids", rows), ids)}
        for name, arr in (("block_table", table), ("q_start", start), ("kv_len", kv), ("last_rows", last), ("u", u),
                          *par.items()):
            feed[name] = self._input(name, arr)
        pools = self._pools()
        out = dag.execute({**feed, **pools})
        if self.backend is None:
            self._bufs["pools"] = dict(zip(self.pool_names, (out[o] for o in outputs[1:])))
        else:
            if rows not in self._moved:   # (pools that the graph of these rows does not update in place, always the same)
                self._moved[rows] = [(n, o) for n, o in zip(self.pool_names, outputs[1:])
                                     if isinstance(out[o], np.ndarray)   # (of a part of the graph that runs on the host)
                                     or out[o].native_handle.data_ptr() != pools[n].native_handle.data_ptr()]
            for n, o in self._moved[rows]:
                if isinstance(out[o], np.ndarray):
                    pools[n].write_from_numpy(out[o])
                else:
                    pools[n].native_handle.copy_(out[o].native_handle)
        tokens = out[outputs[0]]
        tokens = tokens.to_numpy() if hasattr(tokens, "to_numpy") else np.asarray(tokens)
        for s in drawn:
            s.tokens.append(int(tokens[s.slot]))
        return drawn
