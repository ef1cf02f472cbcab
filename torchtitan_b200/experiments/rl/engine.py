"""Paged-KV generation engine for the framework's own decoder models.

It runs the *training* model object (``Decoder`` with ``GQAttention`` blocks: llama3, qwen3 dense and
MoE, llama4) for inference: a packed prefill of all prompts in one pass (document-masked flash
attention), then batched single-token decode steps over a block-table KV cache with the paged decode
kernel and the top-p sampler. Because projections, norms, RoPE and the log-softmax are the same
kernels the trainer uses, the generator's per-token log-probabilities match the trainer's recomputed
ones to rounding, which is the property the reference obtains by registering its model inside vLLM
(torchtitan/experiments/rl/unified/models/vllm_wrapper.py:40-408, models/attention.py:20-225).

Samples of one prompt share the prompt's full KV blocks (reference-counted); only the partial tail
block is copied per sample. With ``cudagraph=True`` a decode step of a given batch size is captured
once in a CUDA graph and replayed (inputs live in static buffers), removing per-step launch overhead.

For long generations, ``split_decode=True`` decodes with attention split over the cache's length, and ``cache_budget``
bounds the tokens that a sequence keeps in the cache: attention weights are accumulated per cached token, and a sequence
that outgrows the budget by ``cache_slack`` is cut back to its most attended tokens (per layer and kv head). Positions go on
counting, up to the rows of the model's rotary table; the sequence's pages are its own, shared with the prompt's other samples
only until the first step cuts a prompt that outgrows the budget back. Both keep a sequence's result independent of the batch
it runs in. Penalties, biases and a grammar change what is drawn; the reported log-probabilities stay those of the model's own
logits, which is what the trainer recomputes.
"""

from __future__ import annotations

from collections.abc import Callable, Sequence
from dataclasses import dataclass

import torch

from torchtitan_b200 import ops
from torchtitan_b200.models.common.attention import AttentionMasks
from torchtitan_b200.ops import serving


class BlockAllocator:
    """Host-side free list with reference counts (blocks shared by samples of one prompt)."""

    def __init__(self, num_blocks: int):
        self.free = list(range(num_blocks - 1, -1, -1))
        self.refs = [0] * num_blocks

    def alloc(self) -> int:
        if not self.free:
            raise RuntimeError("KV cache exhausted: raise gpu_memory_limit or lower the batch / max_tokens")
        b = self.free.pop()
        self.refs[b] = 1
        return b

    def share(self, b: int) -> int:
        self.refs[b] += 1
        return b

    def release(self, b: int) -> None:
        self.refs[b] -= 1
        if self.refs[b] == 0:
            self.free.append(b)

    @property
    def available(self) -> int:
        return len(self.free)


class PagedKVCache:
    def __init__(self, *, n_layers: int, num_blocks: int, block_size: int, n_kv_heads: int, head_dim: int, dtype, device,
                 with_scores: bool = False):
        self.block_size, self.num_blocks = block_size, num_blocks
        shape = (num_blocks, block_size, n_kv_heads, head_dim)
        self.k = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(n_layers)]
        self.v = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(n_layers)]
        # accumulated attention weights, one per layer, block, kv head and slot
        self.scores = torch.zeros(n_layers, num_blocks, n_kv_heads, block_size, device=device) if with_scores else None
        self.alloc = BlockAllocator(num_blocks)

    def copy_block(self, src: int, dst: int) -> None:
        for k, v in zip(self.k, self.v):
            k[dst].copy_(k[src])
            v[dst].copy_(v[src])
        if self.scores is not None:
            self.scores[:, dst].copy_(self.scores[:, src])

    def clear_scores(self, blocks: list[int]) -> None:
        """Blocks that are handed out again start without weights."""
        if self.scores is not None and blocks:
            self.scores[:, torch.tensor(blocks, device=self.scores.device)] = 0.0

    @staticmethod
    def bytes_per_block(n_layers, block_size, n_kv_heads, head_dim, dtype, with_scores: bool = False) -> int:
        row = 2 * head_dim * torch.empty((), dtype=dtype).element_size() + (4 if with_scores else 0)
        return n_layers * block_size * n_kv_heads * row


@dataclass
class _Seq:
    prompt: int                 # index of the prompt this sample belongs to
    blocks: list[int]
    length: int                 # tokens whose KV is in the cache
    position: int               # tokens seen so far: the next token's position
    tokens: list[int]
    logprobs: list[float]
    done: bool = False
    hit_eos: bool = False


_OBSERVED = 16      # last tokens of a prompt whose attention weights are accumulated before decoding begins


class _LogitShaper:
    """What ``GenerationEngine.generate`` puts between a step's logits and the sampler."""

    def __init__(self, prompts, n_samples: int, max_tokens: int, repetition: float, presence: float, frequency: float,
                 logit_bias: dict[int, float] | None, grammar, device):
        self.device, self.grammar = device, grammar
        self.penalties = {"repetition_penalty": repetition, "presence_penalty": presence, "frequency_penalty": frequency}
        self.penalised = (repetition, presence, frequency) != (1.0, 0.0, 0.0)
        if self.penalised:
            rows = [p for p in prompts for _ in range(n_samples)]
            width = max(len(p) for p in rows) + max_tokens
            self.history = torch.tensor([list(p) + [-1] * (width - len(p)) for p in rows], dtype=torch.int32, device=device)
            self.prompt_lens = torch.tensor([len(p) for p in rows], dtype=torch.int32, device=device)
            self.lens = self.prompt_lens.clone()
        self.bias = None
        if logit_bias:
            self.bias = (torch.tensor(list(logit_bias), dtype=torch.int32, device=device).unsqueeze(0),
                         torch.tensor(list(logit_bias.values()), dtype=torch.float32, device=device).unsqueeze(0))
        self.top_id = max(logit_bias, default=-1) if logit_bias else -1
        if logit_bias and min(logit_bias) < 0:
            raise ValueError("logit_bias names a token below 0")

    def __call__(self, logits, seqs, active: list[int]):
        B, V = logits.shape
        if self.top_id >= V:
            raise ValueError(f"logit_bias names token {self.top_id} of a vocabulary of {V}")
        kw = {}
        if self.penalised:
            rows = torch.tensor(active, device=self.device)
            kw = {"tokens": self.history[rows], "lens": self.lens[rows], "prompt_lens": self.prompt_lens[rows], **self.penalties}
        if self.bias is not None:
            kw |= {"bias_ids": self.bias[0].expand(B, -1), "bias_values": self.bias[1].expand(B, -1)}
        if self.grammar is not None and (mask := self._mask(seqs, active, V)) is not None:
            kw["allowed"] = mask
        return serving.process_logits(logits, **kw) if kw else logits

    def _mask(self, seqs, active, V: int):
        words = -(-V // 32)
        rows = [self.grammar(si, list(seqs[si].tokens)) for si in active]
        if all(r is None for r in rows):
            return None
        bits = torch.full((len(rows), words * 32), True)
        for j, ids in enumerate(rows):
            if ids is None:
                continue
            if not len(ids) or min(ids) < 0 or max(ids) >= V:
                raise ValueError(f"the grammar of sequence {active[j]} allows no token, or one outside the vocabulary of {V}")
            bits[j] = False
            bits[j, torch.as_tensor(list(ids), dtype=torch.long)] = True
        w = (bits.view(len(rows), words, 32).long() << torch.arange(32)).sum(-1)
        return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32).to(self.device)

    def check(self, shaped, logprobs, active: list[int]) -> None:
        """Refuses a step in which the grammar and the biases left a sequence nothing: the sampler marks it with NaN."""
        if self.grammar is None and self.bias is None:
            return
        for j in logprobs.isnan().nonzero().flatten().tolist():
            if bool((shaped[j] == float("-inf")).all()):
                raise ValueError(f"the grammar and logit_bias leave sequence {active[j]} no token")

    def said(self, active: list[int], tokens) -> None:
        if self.penalised:
            rows = torch.tensor(active, device=self.device)
            self.history[rows, self.lens[rows].long()] = tokens.to(torch.int32)
            self.lens[rows] += 1


class GenerationEngine:
    def __init__(self, model, *, block_size: int = 16, num_blocks: int = 4096, max_batch: int = 512,
                 cudagraph: bool = False, eos_id: int | None = None, split_decode: bool = False,
                 cache_budget: int | None = None, cache_recent: int | None = None, cache_slack: int | None = None):
        if cache_budget is None and (cache_recent is not None or cache_slack is not None):
            raise ValueError("cache_recent and cache_slack go with cache_budget")
        if cache_budget is not None:
            # by default a quarter of the budget goes to the latest tokens, and an eviction makes room for an eighth
            cache_recent = cache_budget // 4 if cache_recent is None else cache_recent
            cache_slack = max(block_size, cache_budget // 8) if cache_slack is None else cache_slack
            if cache_budget < 1 or not 0 <= cache_recent <= cache_budget or cache_slack < 1:
                raise ValueError(f"cache_budget {cache_budget} >= 1, cache_recent {cache_recent} in [0, cache_budget] and "
                                 f"cache_slack {cache_slack} >= 1 are wanted")
        self.split_decode = split_decode or cache_budget is not None
        self.cache_budget, self.cache_recent, self.cache_slack = cache_budget, cache_recent, cache_slack
        self.evictions = 0
        self.model = model
        p = next(model.parameters())
        self.device, self.dtype = p.device, p.dtype
        att = next(iter(model.layers.values())).attention
        self.n_kv_heads, self.head_dim = att.n_kv_heads, att.head_dim
        self.cache = PagedKVCache(n_layers=len(model.layers), num_blocks=num_blocks, block_size=block_size,
                                  n_kv_heads=self.n_kv_heads, head_dim=self.head_dim, dtype=self.dtype, device=self.device,
                                  with_scores=cache_budget is not None)
        self.block_size, self.max_batch, self.eos_id = block_size, max_batch, eos_id
        self.cudagraph = cudagraph and self.device.type == "cuda"
        self._graphs: dict[tuple[int, int], tuple] = {}
        self.decode_steps = 0
        self.weight_half = 0   # which half of a double-buffered parameter arena the model currently reads

    def _check_position(self, position: int) -> None:
        """Rows of the rotary table are read by position, on the GPU without a check."""
        if position >= (rows := self.model.freqs_cis.shape[0]):
            raise ValueError(f"position {rows} is past the model's rotary table (max_seq_len {rows}): shorten the prompt or max_tokens")

    # ---- one pass over the blocks with cache reads/writes -----------------------------------------
    def _attention(self, att, x, positions, layer: int, meta):
        T = x.shape[1]
        q = att.wq(x).view(1, T, -1, att.head_dim)
        k = att.wk(x).view(1, T, -1, att.head_dim)
        v = att.wv(x).view(1, T, -1, att.head_dim)
        if att.q_norm is not None:
            q, k = att.q_norm(q), att.k_norm(k)
        if att.use_rope:
            table = self.model.freqs_cis
            q = ops.rope(q, table, positions, att.rope_layout)
            k = ops.rope(k, table, positions, att.rope_layout)
        serving.kv_cache_write(self.cache.k[layer], self.cache.v[layer], k[0], v[0], meta["slots"])
        scale = att.scaling if att.scaling is not None else att.head_dim**-0.5
        if meta["prefill"]:
            out = ops.attention(q, k, v, causal=True, scale=scale, doc_ids=meta["doc_ids"])
            # the prompt's weights so far: those of its last tokens' queries, the earliest first
            for rows, lens in meta.get("observe", ()):
                serving.paged_attention_split(q[0, rows], self.cache.k[layer], self.cache.v[layer], meta["block_tables"], lens, scale,
                                              scores=self.cache.scores[layer])
        elif self.split_decode:
            scores = self.cache.scores[layer] if self.cache.scores is not None else None
            out = serving.paged_attention_split(q[0], self.cache.k[layer], self.cache.v[layer], meta["block_tables"],
                                                meta["context_lens"], scale, scores=scores).unsqueeze(0)
        else:
            out = serving.paged_attention_decode(q[0], self.cache.k[layer], self.cache.v[layer], meta["block_tables"],
                                                 meta["context_lens"], scale).unsqueeze(0)
        return att.wo(out.reshape(1, T, -1))

    def _forward(self, tokens, positions, meta, last_index=None):
        m = self.model
        h = m.tok_embeddings(tokens)
        for li, layer in enumerate(m.layers.values()):
            h = h + self._attention(layer.attention, layer.attention_norm(h), positions, li, meta)
            ff = layer.moe if getattr(layer, "moe_enabled", False) else layer.feed_forward
            h = h + ff(layer.ffn_norm(h))
        if last_index is not None:
            h = h[:, last_index]
        return m.output(m.norm(h))[0]

    # ---- public ------------------------------------------------------------------------------------
    @torch.no_grad()
    def generate(self, prompts: list[list[int]], *, n_samples: int, max_tokens: int, temperature: float, top_p: float,
                 generator: torch.Generator | None = None, repetition_penalty: float = 1.0, presence_penalty: float = 0.0,
                 frequency_penalty: float = 0.0, logit_bias: dict[int, float] | None = None,
                 grammar: Callable[[int, list[int]], Sequence[int] | None] | None = None) -> list[_Seq]:
        """Returns ``len(prompts) * n_samples`` sequences, samples of one prompt adjacent.

        The penalties and ``logit_bias`` (token -> added to its logit) are those of ``serving.process_logits``.
        ``grammar(i, tokens)`` is asked before every token of sequence ``i`` with what it has generated: the token ids that
        may come next (at least one that ``logit_bias`` leaves), or None for any."""
        dev, bs = self.device, self.block_size
        shaper = _LogitShaper(prompts, n_samples, max_tokens, repetition_penalty, presence_penalty, frequency_penalty, logit_bias,
                              grammar, dev)
        prompt_blocks: list[list[int]] = []
        scratch: list[int] = []
        seqs: list[_Seq] = []
        was_training = self.model.training
        self.model.eval()
        try:
            # -- prefill: all prompts packed in one row -------------------------------------------------
            toks, pos, doc, slots, last = [], [], [], [], []
            for i, p in enumerate(prompts):
                self._check_position(len(p) - 1)
                nblk = (len(p) + bs - 1) // bs
                blks: list[int] = []
                prompt_blocks.append(blks)
                for _ in range(nblk):
                    blks.append(self.cache.alloc.alloc())
                toks += p
                pos += range(len(p))
                doc += [i] * len(p)
                slots += [blks[t // bs] * bs + t % bs for t in range(len(p))]
                last.append(len(toks) - 1)
            T = len(toks)
            pad = -T % 128 if dev.type == "cuda" else 0      # the flash kernel works on 128-token tiles
            if pad:
                scratch.append(self.cache.alloc.alloc())      # padded tokens write into a throw-away block
                toks += [0] * pad
                pos += [t % self.model.freqs_cis.shape[0] for t in range(pad)]
                doc += [len(prompts)] * pad
                slots += [scratch[0] * bs + (t % bs) for t in range(pad)]
            t_ = lambda x, dt: torch.tensor(x, dtype=dt, device=dev)  # noqa: E731
            if self.cache.scores is not None:
                self.cache.clear_scores([b for blks in prompt_blocks for b in blks])
            meta = {"prefill": True, "slots": t_(slots, torch.int32), "doc_ids": t_(doc, torch.int32).unsqueeze(0)}
            if self.cache.scores is not None:
                width = max(len(blks) for blks in prompt_blocks)
                meta["block_tables"] = t_([blks + [0] * (width - len(blks)) for blks in prompt_blocks], torch.int32)
                meta["observe"] = [(t_([at - min(back, len(p) - 1) for at, p in zip(last, prompts)], torch.long),
                                    t_([max(0, len(p) - back) for p in prompts], torch.int32))
                                   for back in reversed(range(min(_OBSERVED, max(len(p) for p in prompts))))]
            logits = self._forward(t_(toks, torch.long).unsqueeze(0), t_(pos, torch.int32).unsqueeze(0), meta,
                                   last_index=t_(last, torch.long))
            while scratch:
                self.cache.alloc.release(scratch.pop())

            # -- fork samples: share full prompt blocks, copy the partial tail ----------------------------
            for i, p in enumerate(prompts):
                # weights are a sequence's own: no shared blocks, but for those of a prompt that the first decode step cuts back
                # into every sample's own before anything is written
                full = len(p) // bs if self.cache.scores is None else len(prompt_blocks[i]) if self._outgrown(len(p)) else 0
                for s in range(n_samples):
                    blks = [self.cache.alloc.share(b) for b in prompt_blocks[i][:full]]
                    seqs.append(_Seq(prompt=i, blocks=blks, length=len(p), position=len(p), tokens=[], logprobs=[]))
                    for src in prompt_blocks[i][full:]:
                        blks.append(self.cache.alloc.alloc())
                        self.cache.copy_block(src, blks[-1])
                while prompt_blocks[i]:
                    self.cache.alloc.release(prompt_blocks[i].pop())
            first_logits = logits.repeat_interleave(n_samples, dim=0)

            # -- decode -------------------------------------------------------------------------------------
            active = list(range(len(seqs)))
            cur_logits = first_logits
            for step in range(max_tokens):
                u = torch.rand(len(active), device=dev, generator=generator) if generator is not None or dev.type != "cuda" \
                    else torch.rand(len(active), device=dev)
                shaped = shaper(cur_logits, seqs, active)
                tok, lp = serving.sample_top_p(shaped, temperature, top_p, u)
                if shaped is not cur_logits:
                    shaper.check(shaped, lp, active)
                    lp = ops.token_logprobs(cur_logits, tok)
                    shaper.said(active, tok)
                tok_l, lp_l = tok.tolist(), lp.tolist()
                nxt = []
                for j, si in enumerate(active):
                    s = seqs[si]
                    s.tokens.append(tok_l[j])
                    s.logprobs.append(lp_l[j])
                    if self.eos_id is not None and tok_l[j] == self.eos_id:
                        s.done = s.hit_eos = True
                    elif len(s.tokens) >= max_tokens:
                        s.done = True
                    else:
                        nxt.append((si, tok_l[j]))
                if not nxt:
                    break
                active = [si for si, _ in nxt]
                cur_logits = self._decode_step(seqs, active, [t for _, t in nxt])
            return seqs
        finally:
            for s in seqs:
                for b in s.blocks:
                    self.cache.alloc.release(b)
                s.blocks = []
            for blks in (*prompt_blocks, scratch):      # not empty where a step above raised before the samples took over
                for b in blks:
                    self.cache.alloc.release(b)
            if was_training:
                self.model.train()

    def _outgrown(self, length: int) -> bool:
        return self.cache_budget is not None and length >= self.cache_budget + self.cache_slack

    def _evict(self, seqs: list[_Seq]) -> None:
        """Cut the caches of ``seqs`` back to the budget, layer by layer, into new blocks; the old ones are released. As many
        sequences at a time as the free blocks hold: what they give back serves the next."""
        need = -(-self.cache_budget // self.block_size) if seqs else 0
        while seqs:
            group = max(1, self.cache.alloc.available // need)
            self._evict_group(seqs[:group], need)
            seqs = seqs[group:]

    def _evict_group(self, seqs: list[_Seq], need: int) -> None:
        dev = self.device
        new: list[list[int]] = []
        try:
            for _ in seqs:
                new.append([])
                for _ in range(need):
                    new[-1].append(self.cache.alloc.alloc())
            self.cache.clear_scores([b for blks in new for b in blks])
            width = max(len(s.blocks) for s in seqs)
            old_t = torch.tensor([s.blocks + [0] * (width - len(s.blocks)) for s in seqs], dtype=torch.int32, device=dev)
            lens = torch.tensor([s.length for s in seqs], dtype=torch.int32, device=dev)
            new_t = torch.tensor(new, dtype=torch.int32, device=dev)
            for k, v, scores in zip(self.cache.k, self.cache.v, self.cache.scores):
                serving.kv_cache_evict(k, v, scores, old_t, lens, new_t, self.cache_budget, self.cache_recent)
        except BaseException:
            for blks in new:
                for b in blks:
                    self.cache.alloc.release(b)
            raise
        for s, blks in zip(seqs, new):
            for b in s.blocks:
                self.cache.alloc.release(b)
            s.blocks, s.length = blks, self.cache_budget
        self.evictions += len(seqs)

    def _decode_step(self, seqs, active, last_tokens):
        dev, bs = self.device, self.block_size
        B = len(active)
        slots, ctx, pos, handed_out = [], [], [], []
        self._evict([seqs[si] for si in active if self._outgrown(seqs[si].length)])
        for si in active:
            s = seqs[si]
            self._check_position(s.position)
            if s.length % bs == 0 and s.length // bs >= len(s.blocks):
                s.blocks.append(self.cache.alloc.alloc())
                handed_out.append(s.blocks[-1])
            slots.append(s.blocks[s.length // bs] * bs + s.length % bs)
            s.length += 1
            ctx.append(s.length)
            pos.append(s.position)
            s.position += 1
        self.cache.clear_scores(handed_out)
        maxb = max(len(seqs[si].blocks) for si in active)
        maxb = -(-maxb // 8) * 8                        # few distinct table widths => few captured graphs
        bt = [seqs[si].blocks + [0] * (maxb - len(seqs[si].blocks)) for si in active]
        t_ = lambda x, dt: torch.tensor(x, dtype=dt, device=dev)  # noqa: E731
        tokens, positions = t_(last_tokens, torch.long).unsqueeze(0), t_(pos, torch.int32).unsqueeze(0)
        meta = {"prefill": False, "slots": t_(slots, torch.int32), "block_tables": t_(bt, torch.int32),
                "context_lens": t_(ctx, torch.int32)}
        self.decode_steps += 1
        if not self.cudagraph:
            return self._forward(tokens, positions, meta)
        key = (B, maxb, self.weight_half)     # captured graphs hold parameter addresses: one set per arena half
        if key not in self._graphs:
            static = {"tokens": tokens.clone(), "positions": positions.clone(),
                      "meta": {k: (v.clone() if torch.is_tensor(v) else v) for k, v in meta.items()}}
            if self.cache.scores is not None:
                static["meta"]["context_lens"].zero_()      # the warm-up passes must not add weights; the real lengths follow below
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())      # after the last write to what the warm-up passes read
            with torch.cuda.stream(s):
                for _ in range(2):                      # warm-up outside capture
                    self._forward(static["tokens"], static["positions"], static["meta"])
            torch.cuda.current_stream().wait_stream(s)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                out = self._forward(static["tokens"], static["positions"], static["meta"])
            self._graphs[key] = (g, static, out)
        g, static, out = self._graphs[key]
        static["tokens"].copy_(tokens)
        static["positions"].copy_(positions)
        for k, v in meta.items():
            if torch.is_tensor(v):
                static["meta"][k].copy_(v)
        g.replay()
        return out
