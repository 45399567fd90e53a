"""Beam search on the batched pass: every beam a sequence of the engine, the prompt's pages shared by all beams of a search.

A step is one captured graph: the pass of up to 64 rows (:class:`BatchDecode`) with attention that reads the shared pages once for
all beams (:func:`prefix_attention`), the choice of the next beams over beams and vocabulary (:func:`beam_select`), the cached states
that follow them (:func:`beam_reorder`) and the rows of the next pass (:func:`beam_advance`).  The choice never visits the host: what
was chosen is written down and read back at the end.  Two graphs take turns, because the tables and the beams' scores of a step are
read while those of the next are written.

  python -m bloomery_b200.runtime.beam -m model.gguf --prompt "Once upon a time" --beams 4 --new 32
"""
from __future__ import annotations

import os
from dataclasses import dataclass
from typing import List, Optional, Sequence

import torch

from ..ops.beam import MAX_BEAMS, BeamScratch, beam_advance, beam_reorder, beam_select
from ..ops.prefix import PrefixPlan
from .batch_decode import BUCKETS, BatchDecode
from .kv import PAGE


@dataclass
class Hypothesis:
    tokens: List[int]               # without the prompt and without the end's id
    score: float                    # log-probability of the tokens, the end's included
    rank: float                     # score / length ** alpha
    finished: bool


class BeamSearch:
    """Searches of ``beams`` beams, ``groups`` prompts at a time, in slots ``first_slot`` and on of a :class:`DecodeEngine` with
    grouped-query attention.  ``eos``: the id that ends a sequence (-1: none does); candidates are ranked by score / length ** alpha.

    ``shared_attention``: whether the prompt's pages are read once for all beams (:func:`prefix_attention`, queries and probabilities
    of 11 bits) or by each beam, as in every other batched pass (22 bits or more).  None, the default, shares where there is
    something to share, and q8_0 caches in any case.  Device time of a layer's attention, shared / not, of 16 beams (32 heads over
    4 of 128) with 20, 400 and 2,000 positions of their own: nothing shared 12.7 / 8.0, 16.4 / 17.8, 29.3 / 25.2 us in f16 and 13.1 /
    8.8, 17.4 / 19.7, 33.2 / 49.2 in q8_0; behind 512 shared ones 13.5 / 19.0, 16.6 / 20.7, 29.5 / 27.9 in f16."""

    CHECK = 16                      # steps between looks at whether every beam has ended

    def __init__(self, engine, beams: int, groups: int = 1, eos: Optional[int] = None, alpha: float = 0.0, max_new: int = 512,
                 first_slot: int = 0, shared_attention: Optional[bool] = None):
        from .engine import DecodeEngine
        s = engine.spec
        if type(engine) is not DecodeEngine:             # their experts are elsewhere, or on several cards
            raise NotImplementedError("beam search runs on a whole model on one card; tiered and sharded engines keep their own passes")
        if s.mla:
            raise NotImplementedError("beam search runs on grouped-query attention")
        if not 1 <= beams <= MAX_BEAMS or groups < 1 or beams * groups > BUCKETS[-1]:
            raise ValueError(f"up to {BUCKETS[-1]} beams in all")
        if first_slot < 0 or first_slot + beams * groups > engine.n_slots:
            raise ValueError(f"{beams * groups} beams need as many slots of the engine")
        self.e, self.B, self.G, self.alpha, self.max_new = engine, beams, groups, float(alpha), max_new
        self.eos = s.eos_id if eos is None else eos
        R = self.R = beams * groups
        M = self.M = BatchDecode.bucket(R)
        dev = engine.device
        self.slots = list(range(first_slot, first_slot + R))
        self.bd = BatchDecode(engine, max_rows=M)
        self.shared_attention = shared_attention
        self.plan = None if shared_attention is False else \
            PrefixPlan([beams] * groups + [M - R] * (M > R), [0] * (groups + (M > R)), s.n_q, s.n_kv, s.head_dim, dev)
        self.scratch = BeamScratch(groups, beams, s.vocab, dev)
        i32 = dict(dtype=torch.int32, device=dev)
        self.slots_dev = torch.tensor(self.slots, **i32)
        self.parent, self.token = torch.zeros(R, **i32), torch.zeros(R, **i32)
        self.scores = [torch.zeros(groups, beams, device=dev) for _ in range(2)]
        self.done = [torch.zeros(groups, beams, **i32) for _ in range(2)]
        self.lengths = [torch.zeros(groups, beams, **i32) for _ in range(2)]
        self.held = torch.zeros(groups, **i32)
        self.hist, self.count = torch.zeros(max_new, 2, R, **i32), torch.zeros(1, **i32)
        self.tables = [engine.kv.table, torch.empty_like(engine.kv.table)]
        self.graphs: dict = {}                           # (step & 1, whether the attention is the shared one) -> graph

    # ---- one step -----------------------------------------------------------------------------------------------
    def _enqueue(self, par: int) -> None:
        e, kv, now, nxt = self.e, self.e.kv, par, par ^ 1
        kept, kv.table = kv.table, self.tables[now]
        try:
            self.bd.enqueue(self.M)
        finally:
            kv.table = kept
        beam_select(self.bd.logits[:self.R], self.scores[now], self.scratch, self.parent, self.token, self.scores[nxt],
                    done=self.done[now] if self.eos >= 0 else None, lengths=self.lengths[now], out_done=self.done[nxt],
                    out_lengths=self.lengths[nxt], eos=self.eos, alpha=self.alpha, fault=e.fault)
        beam_reorder(kv.k, kv.v, self.tables[now], self.tables[nxt], self.slots_dev, self.parent.view(self.G, self.B), self.held, e.fault)
        beam_advance(self.bd.tokens, self.bd.row_pos, self.bd.row_seq, self.held, self.hist, self.count, self.slots_dev, self.parent,
                     self.token, self.done[nxt], self.scores[nxt], self.G, self.B)

    def _step(self, i: int) -> None:
        """Step ``i`` on the current stream: the first two of either attention run as launches, the next two are captured."""
        par = i & 1
        key = par, self.bd.prefix is not None
        if key not in self.graphs and i >= 2 and self.e.use_graphs:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=self.bd._stream):
                self._enqueue(par)
            self.graphs[key] = g
        if key in self.graphs:
            self.graphs[key].replay()
        else:
            self._enqueue(par)

    # ---- a search -----------------------------------------------------------------------------------------------
    def search(self, prompts: Sequence[Sequence[int]], max_new: Optional[int] = None) -> List[List[Hypothesis]]:
        """The beams of every prompt, best first.  The slots of the search are empty before and after it."""
        e, kv, B, G = self.e, self.e.kv, self.B, self.G
        n_new = self.max_new if max_new is None else max_new
        if len(prompts) != G or any(len(p) < 1 for p in prompts):
            raise ValueError(f"{G} prompts of one id at least")
        if not 1 <= n_new <= self.max_new:
            raise ValueError(f"1 to {self.max_new} new ids")
        if max(len(p) for p in prompts) + n_new > e.slot_ctx:
            raise ValueError(f"a prompt and {n_new} new ids exceed the slot context of {e.slot_ctx}")
        try:
            return self._search([list(map(int, p)) for p in prompts], n_new)
        finally:
            with e._lock:
                # whoever gets these pages, and the table, next does so behind the steps
                torch.cuda.current_stream(e.device).wait_stream(self.bd._stream)
                kv.pinned.difference_update(self.slots)
                for slot in self.slots:
                    e.reset(slot)
                kv.dirty = True                          # the tables were rewritten on the card
                kv.sync_table()

    def _search(self, prompts: List[List[int]], n_new: int) -> List[List[Hypothesis]]:
        e, kv, bd, B, G, R = self.e, self.e.kv, self.bd, self.B, self.G, self.R
        shared = []
        for g, prompt in enumerate(prompts):
            own = self.slots[g * B:(g + 1) * B]
            with e._lock:
                kv.pinned.update(own)                    # from here on: a prompt's passes protect its own slot alone
                for slot in own:
                    e.reset(slot)
            n = len(prompt) - 1                          # the last id is the first pass's
            if n:
                e.prefill(own[0], prompt[:n])
            with e._lock:
                for slot in own[1:]:
                    kv.share_prefix(own[0], slot, n)
                for slot in own:
                    kv.ensure(slot, len(prompt) + n_new)     # pages behind the shared ones belong to a beam each
            shared.append(n // PAGE * PAGE if B > 1 else 0)
        # sequences that made room for the beams are copied out on this stream: the steps write their pages behind that
        bd._stream.wait_stream(torch.cuda.current_stream(e.device))
        with e._lock, torch.cuda.stream(bd._stream):
            share = self.shared_attention
            if share is None:
                share = e.kv_q8 or any(shared)
            bd.prefix = self.plan if share else None
            if share:
                self.plan.set_prefix(shared + [0] * (self.M > R))
            kv.sync_table()
            self.tables[0] = kv.table
            self.tables[1].copy_(kv.table)
            h = bd._params_np
            h[:2] = 0
            h[2] = -1
            for g, prompt in enumerate(prompts):
                h[1, g * B:(g + 1) * B] = len(prompt) - 1
                h[0, g * B], h[2, g * B] = prompt[-1], self.slots[g * B]
            bd.params.copy_(bd.params_host, non_blocking=True)
            first = torch.full((G, B), float("-inf"))
            first[:, 0] = 0.0
            self.scores[0].copy_(first)
            self.done[0].zero_()
            self.lengths[0].zero_()
            self.held.copy_(torch.tensor([len(p) for p in prompts], dtype=torch.int32))
            self.count.zero_()
            steps = 0
            for i in range(n_new):
                self._step(i)
                steps = i + 1
                if self.eos >= 0 and steps % self.CHECK == 0 and bool(self.done[steps & 1].all()):
                    break
            last = steps & 1
            hist = self.hist[:steps].cpu()
            scores, done, lengths = self.scores[last].cpu(), self.done[last].cpu(), self.lengths[last].cpu()
            status = int(bd.status)
        if status != 0:
            raise RuntimeError("a bounded wait inside the GEMM kernel ran out (status word set)")
        e.check_fault()
        return [[self._trace(hist, g, i, float(scores[g, i]), bool(done[g, i]), int(lengths[g, i])) for i in range(B)
                 if float(scores[g, i]) > float("-inf")] for g in range(G)]

    def _trace(self, hist: torch.Tensor, g: int, i: int, score: float, finished: bool, length: int) -> Hypothesis:
        tokens = []
        for step in range(hist.shape[0] - 1, -1, -1):
            at = g * self.B + i
            tokens.append(int(hist[step, 1, at]))
            i = int(hist[step, 0, at])
        tokens.reverse()
        tokens = tokens[:length]                         # a finished beam repeats the end's id
        if finished and tokens and tokens[-1] == self.eos:
            tokens.pop()
        return Hypothesis(tokens, score, score / max(1, length) ** self.alpha, finished)


def main(argv: Optional[Sequence[str]] = None) -> int:
    import argparse
    ap = argparse.ArgumentParser(description="beam search over a checkpoint, or over random weights of a tiny model")
    ap.add_argument("-m", "--model", help="a GGUF file or a safetensors folder; without one, random weights and ids")
    ap.add_argument("--prompt", default="Once upon a time")
    ap.add_argument("--beams", type=int, default=4)
    ap.add_argument("--new", type=int, default=32)
    ap.add_argument("--alpha", type=float, default=0.0)
    ap.add_argument("--separate", action="store_true", help="every beam reads the prompt's pages itself, with more bits of each probability")
    a = ap.parse_args(argv)
    from ..models.weights import Weights, open_model, synth_tensors
    from .engine import DecodeEngine
    tk = None
    if a.model:
        from ..serve.tokenizer import from_folder, from_gguf
        _, w, handle = open_model(a.model, "cuda:0")
        tk = from_folder(a.model, w.spec.vocab) if os.path.isdir(a.model) else from_gguf(handle, w.spec.vocab)
    else:
        from ..models.spec import tiny_qwen3moe
        spec = tiny_qwen3moe()
        w = Weights.from_items(spec, synth_tensors(spec, "cpu", seed=0), "cpu").to("cuda:0")
    ids = tk.encode(a.prompt) if tk is not None else [1 + b for b in a.prompt.encode()]
    eng = DecodeEngine(w, n_slots=a.beams, slot_ctx=(len(ids) + a.new + PAGE) // PAGE * PAGE)
    for h in BeamSearch(eng, a.beams, alpha=a.alpha, max_new=a.new, shared_attention=False if a.separate else None).search([ids])[0]:
        print(f"{h.rank:10.4f}  {tk.decode(h.tokens) if tk is not None else h.tokens}")
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
