"""Generation-side ops: paged-KV decode attention, KV-cache writes and the token sampler.

PyTorch definitions (any device) and dispatch to the native kernels on CUDA. The cache layout is
``[num_blocks, block_size, n_kv_heads, head_dim]`` for keys and values; ``block_tables[b, i]`` is the
cache block holding tokens ``i*block_size ... (i+1)*block_size-1`` of sequence ``b``.

Reference counterpart: vLLM's paged attention and sampler as used by
torchtitan/experiments/rl/unified/models/attention.py:62-117 and actors/generator.py:251-260
(temperature, top-p, sampled-token log-probability from an fp32 log-softmax of the raw logits).

For long caches: attention split over the cache's length, eviction by accumulated attention weight, and penalties, biases
and grammar masks on the logits.
"""

from __future__ import annotations

import math

import torch

from . import native
from torchtitan_b200.tools.logging import logger, warn_once


def kv_cache_write(k_cache, v_cache, k, v, slots):
    """Scatter new keys/values ``[T, Hkv, D]`` into flat cache slots ``slots[T]`` (= block * block_size + offset)."""
    if k.is_cuda and native.has("tt_kv_write"):
        from .cuda_ops import kv_write

        return kv_write(k_cache, v_cache, k, v, slots)
    kc, vc = k_cache.view(-1, *k_cache.shape[2:]), v_cache.view(-1, *v_cache.shape[2:])
    kc.index_copy_(0, slots.long(), k.to(kc.dtype))
    vc.index_copy_(0, slots.long(), v.to(vc.dtype))


def paged_attention_decode(q, k_cache, v_cache, block_tables, context_lens, scale: float):
    """One query token per sequence: ``q [B, H, D]`` attends to the first ``context_lens[b]`` cached tokens
    of its sequence. Returns ``[B, H, D]``. GQA: query head h reads kv head ``h // (H / Hkv)``."""
    if q.is_cuda and native.has("tt_paged_decode") and q.dtype == torch.bfloat16 and q.shape[-1] == 128 and \
            (q.shape[1] // k_cache.shape[2]) in (1, 2, 4, 8):
        from .cuda_ops import paged_decode

        return paged_decode(q, k_cache, v_cache, block_tables, context_lens, scale)
    B, H, D = q.shape
    nb, bs, Hkv, _ = k_cache.shape
    max_ctx = block_tables.shape[1] * bs
    idx = (block_tables.long().unsqueeze(-1) * bs + torch.arange(bs, device=q.device)).view(B, max_ctx)
    k = k_cache.view(-1, Hkv, D)[idx]            # [B, ctx, Hkv, D]
    v = v_cache.view(-1, Hkv, D)[idx]
    rep = H // Hkv
    k = k.repeat_interleave(rep, dim=2).float()
    v = v.repeat_interleave(rep, dim=2).float()
    s = torch.einsum("bhd,bchd->bhc", q.float(), k) * scale
    dead = torch.arange(max_ctx, device=q.device).view(1, 1, -1) >= context_lens.view(B, 1, 1)
    s = s.masked_fill(dead, float("-inf"))
    p = torch.softmax(s, dim=-1)
    return torch.einsum("bhc,bchd->bhd", p, v).to(q.dtype)


_WHOLE = (torch.int32, torch.int64)


def _whole_numbers(t, name: str, rows: int, dims: int, device) -> None:
    """``t`` must hold whole numbers on ``device``, ``[rows]`` or ``[rows, any]``."""
    if not torch.is_tensor(t) or t.dtype not in _WHOLE:
        raise TypeError(f"{name} must be an int32 or int64 tensor")
    if t.dim() != dims or t.shape[0] != rows:
        raise ValueError(f"{name} must have shape {[rows, '*'][:dims]}, got {list(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other tensors are on {device}")


def _no_gradient(what: str, *tensors) -> None:
    for t in tensors:
        if t is not None and t.requires_grad:
            raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad() or on detached tensors")


def _check_cache(k_cache, v_cache, scores, block_tables, context_lens, batch: int) -> None:
    """What the ops over a paged cache have in common."""
    shape, dev = k_cache.shape, k_cache.device
    if len(shape) != 4 or v_cache.shape != shape:
        raise ValueError(f"caches must be [num_blocks, block_size, n_kv_heads, head_dim] and alike, got {list(k_cache.shape)} and {list(v_cache.shape)}")
    if v_cache.dtype != k_cache.dtype:
        raise TypeError(f"key and value cache differ in type: {k_cache.dtype}, {v_cache.dtype}")
    if v_cache.device != dev:
        raise ValueError(f"key cache on {dev}, value cache on {v_cache.device}")
    nb, bs, hkv, _ = shape
    if 0 in shape:
        raise ValueError(f"empty cache {list(shape)}")
    bt, cl = block_tables, context_lens
    if not (type(bt) is type(cl) is torch.Tensor and bt.dtype in _WHOLE and cl.dtype in _WHOLE and bt.device == cl.device == dev
            and bt.dim() == 2 and cl.shape == bt.shape[:1] == (batch,)):      # something may be wrong: say what
        _whole_numbers(bt, "block_tables", batch, 2, dev)
        _whole_numbers(cl, "context_lens", batch, 1, dev)
    if bt.shape[1] * bs >= 1 << 30:
        raise ValueError("block_tables hold 2^30 tokens or more")
    if scores is not None:
        if scores.dtype != torch.float32:
            raise TypeError(f"scores must be fp32, got {scores.dtype}")
        if tuple(scores.shape) != (nb, hkv, bs) or scores.device != dev or not scores.is_contiguous():
            raise ValueError(f"scores must be a contiguous [num_blocks, n_kv_heads, block_size] = {[nb, hkv, bs]} tensor on {dev}")
    if dev.type == "cpu" and batch:
        room = block_tables.shape[1] * bs
        if int(context_lens.min()) < 0 or int(context_lens.max()) > room:
            raise ValueError(f"context_lens must be in [0, {room}] (the tokens that block_tables has room for)")
        live = torch.arange(block_tables.shape[1]) < ((context_lens + bs - 1) // bs).unsqueeze(1)
        used = block_tables[live]
        if used.numel() and (int(used.min()) < 0 or int(used.max()) >= nb):
            raise ValueError(f"block_tables name pages outside [0, {nb})")


def paged_attention_split(q, k_cache, v_cache, block_tables, context_lens, scale: float, *, window: int | None = None,
                          sinks=None, scores=None, return_lse: bool = False):
    """One query token per sequence over a paged cache, the work split over the cache's length and joined.

    As :func:`paged_attention_decode` (``q [B, H, D]`` -> ``[B, H, D]``), for any number of query heads per kv head, with

    ``window``      only the last ``window`` cached tokens are attended to (the query is the last of them);
    ``sinks``       ``[H]`` logits that join the softmax's denominator only;
    ``scores``      fp32 ``[num_blocks, n_kv_heads, block_size]``: every token's attention weights, summed over the query
                    heads of its kv head, are added to its slot in place (what :func:`kv_cache_evict` goes by). A page that
                    several sequences share collects the weights of all of them, in no fixed order;
    ``return_lse``  also returns the log of the softmax's denominator, fp32 ``[B, H]``.

    A sequence without tokens gives zeros (and a denominator of the sink alone). What unused slots of the cache hold does not
    matter; a NaN or infinity in an attended value gives NaN. On CUDA a length or page number outside the table or the cache
    gives NaN for that sequence, in its scores too (no score is added for a page outside); on the CPU it raises. CUDA kernels:
    bf16 and fp16, head_dim 64, 128 and 256, caches with contiguous heads on 16-byte boundaries (other strides are free); on them
    a sequence's result depends, to the bit, neither on the others in the batch nor on the table's width. Other types and head
    dims take the definition below. The workspace is ``4 * B * H * (head_dim + 2)`` bytes per 512 tokens of the table's width (or window;
    256 times that at most), and with ``scores`` ``4 * B * H`` per token of it: give tables no wider than the longest sequence
    needs. No gradient.

    Reference counterpart: the attention of the generator, torchtitan/experiments/rl/unified/models/attention.py:62-117.
    """
    if torch.is_grad_enabled():
        _no_gradient("paged_attention_split", q, k_cache, v_cache, sinks)
    if q.dim() != 3:
        raise ValueError(f"q must be [batch, heads, head_dim], got {list(q.shape)}")
    B, H, D = q.shape
    _check_cache(k_cache, v_cache, scores, block_tables, context_lens, B)
    nb, bs, hkv, kd = k_cache.shape
    if q.dtype != k_cache.dtype or not q.is_floating_point():
        raise TypeError(f"q and the caches must be of one floating type, got {q.dtype} and {k_cache.dtype}")
    if q.device != k_cache.device:
        raise ValueError(f"q is on {q.device}, the caches are on {k_cache.device}")
    if D != kd or H % hkv:
        raise ValueError(f"{H} query heads of size {D} do not go with {hkv} kv heads of size {kd}")
    if window is not None and (not isinstance(window, int) or window < 1):
        raise ValueError(f"window must be a whole number of at least 1, got {window}")
    if sinks is not None and (tuple(sinks.shape) != (H,) or sinks.device != q.device):
        raise ValueError(f"sinks must be one value per query head [{H}] on {q.device}")
    if q.is_cuda:
        from . import cuda_ops

        if D in cuda_ops.PAGED_SPLIT_DIMS and q.dtype in (torch.bfloat16, torch.float16):
            return cuda_ops.paged_split(q, k_cache, v_cache, block_tables, context_lens, scale, window, sinks, scores, return_lse)
        warn_once(logger, f"paged_attention_split with {q.dtype}, head_dim {D} takes the PyTorch path")
    room = block_tables.shape[1] * bs
    span = room if window is None else min(room, window)
    lens = context_lens.long()
    start = (lens - span).clamp(min=0) if window is not None else torch.zeros_like(lens)
    pos = start.unsqueeze(1) + torch.arange(span, device=q.device)
    live = pos < lens.unsqueeze(1)                                             # [B, span]
    pos = pos.clamp(max=max(room - 1, 0))
    page = block_tables.long().gather(1, pos // bs).masked_fill(~live, 0) if room else pos
    off = pos % bs
    wrong = (page < 0) | (page >= nb)                                          # the CPU has refused these already
    page = page.masked_fill(wrong, 0)
    bad = wrong.any(1) | (lens < 0) | (lens > room)
    dead = ~live.view(B, span, 1, 1)
    acc = torch.float64 if q.dtype == torch.float64 else torch.float32
    k = k_cache[page, off].to(acc).masked_fill(dead, 0.0)                     # [B, span, Hkv, D]
    v = v_cache[page, off].to(acc).masked_fill(dead, 0.0)
    x = torch.einsum("bhgd,bnhd->bhgn", q.to(acc).view(B, hkv, H // hkv, D), k) * scale
    x = x.masked_fill(~live.view(B, 1, 1, span), -math.inf)
    if sinks is not None:
        x = torch.cat((x, sinks.to(acc).view(1, hkv, H // hkv, 1).expand(B, -1, -1, 1)), dim=-1)
    lse = torch.logsumexp(x, dim=-1, keepdim=True) if x.shape[-1] else x.new_full((B, hkv, H // hkv, 1), -math.inf)
    w = torch.exp(x[..., :span] - lse.masked_fill(lse == -math.inf, 0.0))     # nothing to attend to: zero weights
    w = w.masked_fill(bad.view(B, 1, 1, 1), math.nan)
    out = torch.einsum("bhgn,bnhd->bhgd", w, v).reshape(B, H, D).to(q.dtype)
    out, lse = out.masked_fill(bad.view(B, 1, 1), math.nan), lse.masked_fill(bad.view(B, 1, 1, 1), math.nan)
    live = live & ~wrong & (lens >= 0).unsqueeze(1) & (lens <= room).unsqueeze(1)
    if scores is not None:
        at = (page.unsqueeze(1) * hkv + torch.arange(hkv, device=q.device).view(1, hkv, 1)) * bs + off.unsqueeze(1)
        scores.view(-1).index_add_(0, at.reshape(-1), w.sum(2).masked_fill(~live.unsqueeze(1), 0.0).reshape(-1).float())
    return (out, lse.reshape(B, H).float()) if return_lse else out


def kv_cache_evict(k_cache, v_cache, scores, block_tables, context_lens, new_tables, keep: int, recent: int = 0):
    """Cut every sequence back to its ``keep`` most attended tokens, separately for each kv head.

    A sequence of at most ``keep`` tokens stays whole. Of a longer one the last ``recent`` tokens stay and, of those before,
    the ``keep - recent`` with the largest accumulated weight in ``scores`` (see :func:`paged_attention_split`; equal scores:
    the earlier token; NaN counts as the largest). What stays is copied in its order, keys, values and scores, to the first
    slots of the pages ``new_tables [B, >= ceil(keep / block_size)]``, slots behind it are left as they are. The old pages
    are only read: they may be shared, and the caller frees them. The new pages must be distinct pages that no sequence of
    the call uses (checked on the CPU; on CUDA an overlap leaves undefined contents in them).

    Returns ``(new_lens int32 [B], kept int32 [B, n_kv_heads, keep])``: the tokens now in slots 0, 1, ... and -1 behind them.
    On CUDA a length outside the table counts as 0, and rows whose page number lies outside the cache are not moved; rows of
    ``head_dim * itemsize`` bytes must be multiples of 16 on 16-byte boundaries. No gradient.

    No counterpart in the reference, whose generator keeps every token.
    """
    if torch.is_grad_enabled():
        _no_gradient("kv_cache_evict", k_cache, v_cache, scores)
    if scores is None:
        raise ValueError("kv_cache_evict goes by scores")
    B = block_tables.shape[0]
    _check_cache(k_cache, v_cache, scores, block_tables, context_lens, B)
    nb, bs, hkv, D = k_cache.shape
    if not isinstance(keep, int) or not isinstance(recent, int) or not 1 <= keep < 1 << 30 or not 0 <= recent <= keep:
        raise ValueError(f"keep must be a whole number in [1, 2^30) and recent one in [0, keep], got {keep} and {recent}")
    _whole_numbers(new_tables, "new_tables", B, 2, k_cache.device)
    room = block_tables.shape[1] * bs
    most = min(keep, room)
    if new_tables.shape[1] * bs < most:
        raise ValueError(f"new_tables have room for {new_tables.shape[1] * bs} of {most} kept tokens")
    if k_cache.is_cuda:
        from .cuda_ops import kv_evict

        return kv_evict(k_cache, v_cache, scores, block_tables, context_lens, new_tables, keep, recent)
    old, lens = block_tables.long(), context_lens.long()
    left = lens.clamp(max=keep)
    need = torch.arange(new_tables.shape[1]) < ((left + bs - 1) // bs).unsqueeze(1)
    fresh = new_tables.long()[need]
    if fresh.numel() and (int(fresh.min()) < 0 or int(fresh.max()) >= nb):
        raise ValueError(f"new_tables name pages outside [0, {nb})")
    in_use = old[torch.arange(old.shape[1]) < ((lens + bs - 1) // bs).unsqueeze(1)]
    if fresh.unique().numel() != fresh.numel() or bool(torch.isin(fresh, in_use).any()):
        raise ValueError("new_tables must name distinct pages that no sequence of the call uses")
    kept = torch.full((B, hkv, keep), -1, dtype=torch.int32)
    moves = []
    for b, n in enumerate(lens.tolist()):
        for h in range(hkv):
            idx = torch.arange(n)
            if n > keep:
                first = n - recent
                s = scores[old[b, : -(-n // bs)], h].reshape(-1)[:first]       # behind its pages a table may hold anything
                best = torch.sort(s, descending=True, stable=True).indices[: keep - recent]
                idx = torch.cat((best.sort().values, torch.arange(first, n)))
            j = torch.arange(idx.numel())
            kept[b, h, : idx.numel()] = idx.to(torch.int32)
            moves.append((old[b, idx // bs], idx % bs, new_tables[b].long()[j // bs], j % bs, torch.full_like(j, h)))
    if moves:
        sp, so, dp, do, h = (torch.cat(m) for m in zip(*moves))
        k_cache[dp, do, h], v_cache[dp, do, h], scores[dp, h, do] = k_cache[sp, so, h], v_cache[sp, so, h], scores[sp, h, so]
    return left.to(torch.int32), kept


LOGIT_BIASES_MAX = 1024
HISTORY_MAX = (1 << 20) - 1


def _setting(value, name: str, batch: int, device, positive: bool = False):
    if torch.is_tensor(value):
        if tuple(value.shape) != (batch,) or value.dtype != torch.float32 or value.device != device:
            raise ValueError(f"{name} must be a number or an fp32 tensor [{batch}] on {device}")
        bad = value.device.type == "cpu" and (not bool(torch.isfinite(value).all()) or (positive and bool((value <= 0).any())))
    else:
        bad = not math.isfinite(value) or (positive and value <= 0)
    if bad:
        raise ValueError(f"{name} must be finite{' and positive' if positive else ''}, got {value}")
    return value


def process_logits(logits, tokens=None, lens=None, prompt_lens=None, *, repetition_penalty=1.0, presence_penalty=0.0,
                   frequency_penalty=0.0, bias_ids=None, bias_values=None, allowed=None, out=None):
    """Penalties for repeated tokens, biases and grammar masks on ``logits [B, V]`` (fp32, bf16 or fp16), before
    :func:`sample_top_p`. In this order, in fp32, rounded once to the logits' type:

    * ``x / repetition_penalty`` where ``x > 0``, else ``x * repetition_penalty``, for tokens among the first ``lens[b]`` of
      ``tokens [B, L]`` (prompt and generated);
    * ``x - frequency_penalty * count - presence_penalty`` for tokens that occur ``count > 0`` times among those generated,
      i.e. from ``prompt_lens[b]`` on;
    * ``x + bias_values`` for ``bias_ids [B, N]`` (at most 1024 entries; entries of the same token add up in their order);
    * ``-inf`` where bit ``i % 32`` of ``allowed[b, i // 32]`` (int32) is 0.

    The penalties are numbers or fp32 tensors ``[B]``. ``lens`` / ``prompt_lens`` (whole numbers ``[B]``) default to ``L`` and
    0. Token and bias ids below 0 are padding; ids of ``V`` and above raise on the CPU and are skipped on CUDA. A row whose
    mask allows nothing is ``-inf`` throughout (:func:`sample_top_p` marks it by a log-probability of NaN). ``out`` may be
    ``logits`` itself. Returns the adjusted logits. No gradient.

    No counterpart in the reference, whose generator samples by temperature and top-p
    (torchtitan/experiments/rl/unified/actors/generator.py:251-260).
    """
    if torch.is_grad_enabled():
        _no_gradient("process_logits", logits, bias_values, out)
    if logits.dim() != 2:
        raise ValueError(f"logits must be [batch, vocabulary], got {list(logits.shape)}")
    if logits.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError(f"logits must be fp32, bf16 or fp16, got {logits.dtype}")
    (B, V), dev = logits.shape, logits.device
    rep = _setting(repetition_penalty, "repetition_penalty", B, dev, positive=True)
    pres = _setting(presence_penalty, "presence_penalty", B, dev)
    freq = _setting(frequency_penalty, "frequency_penalty", B, dev)
    if tokens is not None:
        _whole_numbers(tokens, "tokens", B, 2, dev)
        if tokens.shape[1] > HISTORY_MAX:
            raise ValueError(f"tokens are longer than {HISTORY_MAX}")
        for t, name in ((lens, "lens"), (prompt_lens, "prompt_lens")):
            if t is not None:
                _whole_numbers(t, name, B, 1, dev)
    elif lens is not None or prompt_lens is not None or any(torch.is_tensor(p) or p != d for p, d in ((rep, 1.0), (pres, 0.0), (freq, 0.0))):
        raise ValueError("penalties and lengths need tokens")
    if (bias_ids is None) != (bias_values is None):
        raise ValueError("bias_ids and bias_values go together")
    if bias_ids is not None:
        _whole_numbers(bias_ids, "bias_ids", B, 2, dev)
        if bias_values.dtype != torch.float32 or bias_values.shape != bias_ids.shape or bias_values.device != dev:
            raise ValueError(f"bias_values must be fp32 {list(bias_ids.shape)} on {dev}")
        if bias_ids.shape[1] > LOGIT_BIASES_MAX:
            raise ValueError(f"at most {LOGIT_BIASES_MAX} biases per row, got {bias_ids.shape[1]}")
    if allowed is not None:
        if allowed.dtype != torch.int32 or allowed.dim() != 2 or allowed.shape[0] != B or allowed.shape[1] * 32 < V or allowed.device != dev:
            raise ValueError(f"allowed must be int32 [{B}, at least {-(-V // 32)}] on {dev}")
    if out is not None:
        if out.shape != logits.shape or out.dtype != logits.dtype or out.device != dev or out.stride(-1) != 1:
            raise ValueError("out must be like logits, with contiguous rows")
        if B > 1 and out.stride(0) < V:
            raise ValueError("the rows of out overlap")
        same = out.data_ptr() == logits.data_ptr() and out.stride() == logits.stride()
        if not same and out.untyped_storage().data_ptr() == logits.untyped_storage().data_ptr():
            raise ValueError("out must be logits itself or a tensor of its own")
    if logits.is_cuda:
        from .cuda_ops import adjust_logits

        return adjust_logits(logits, tokens, lens, prompt_lens, rep, pres, freq, bias_ids, bias_values, allowed, out)
    x = logits.float()
    col = lambda p: p.view(B, 1) if torch.is_tensor(p) else p  # noqa: E731
    if tokens is not None:
        L = tokens.shape[1]
        at = torch.arange(L)
        live = (tokens >= 0) & (at < (lens if lens is not None else torch.full((B,), L)).unsqueeze(1))
        if bool((tokens.masked_fill(~live, 0) >= V).any()):
            raise ValueError(f"tokens outside the vocabulary of {V}")
        said = live & (at >= prompt_lens.unsqueeze(1)) if prompt_lens is not None else live
        ids = tokens.long().masked_fill(~live, 0)
        seen = torch.zeros(B, V, dtype=torch.int32).scatter_add_(1, ids, live.to(torch.int32)) > 0
        count = torch.zeros(B, V, dtype=torch.int32).scatter_add_(1, ids, said.to(torch.int32))
        x = torch.where(seen, torch.where(x > 0, x / col(rep), x * col(rep)), x)
        x = torch.where(count > 0, x - col(freq) * count - col(pres), x)
    if bias_ids is not None:
        ok = bias_ids >= 0
        if bool((bias_ids >= V).any()):
            raise ValueError(f"bias_ids outside the vocabulary of {V}")
        total = torch.zeros(B, V).scatter_add_(1, bias_ids.long().clamp(min=0), bias_values.masked_fill(~ok, 0.0))
        x = x + total
    if allowed is not None:
        i = torch.arange(V)
        x = x.masked_fill(((allowed[:, i // 32] >> (i % 32)) & 1) == 0, -math.inf)
    x = x.to(logits.dtype)
    return out.copy_(x) if out is not None else x


def sample_top_p(logits, temperature: float, top_p: float, uniforms):
    """Sample one token per row of ``logits [B, V]``.

    ``uniforms [B]`` in [0, 1) drives the draw by inverse CDF in vocabulary index order -- over the whole vocabulary
    when ``top_p >= 1`` (plain multinomial sampling), over the nucleus otherwise -- so a given (logits, uniform) pair
    yields the same token on every device up to rounding at CDF boundaries. The nucleus is the set of tokens at least as
    likely as the last token needed to reach a cumulative mass of ``top_p`` from the most likely down (ties at that
    probability are all kept).
    A row that allows nothing (``-inf`` throughout, see :func:`process_logits`) gives token 0 with a log-probability of NaN, and
    so does one with NaN or ``+inf`` in it unless it is greedy.
    ``temperature == 0`` is greedy (lowest index on ties). Returns (tokens int64 [B], log-probabilities fp32 [B]); the log-probability is taken from the
    fp32 log-softmax of the *unscaled* logits, which is what the trainer recomputes."""
    if logits.is_cuda and native.has("tt_sample") and (top_p >= 1.0 or temperature <= 0.0 or native.has("tt_sample_top_p")):
        from .cuda_ops import sample as native_sample

        return native_sample(logits, temperature, uniforms, top_p)
    lf = logits.float()
    logp_raw = torch.log_softmax(lf, dim=-1)
    if temperature <= 0.0:
        tok = lf.argmax(-1)
        return tok, logp_raw.gather(1, tok.view(-1, 1)).squeeze(1)
    probs = torch.softmax(lf / temperature, dim=-1)
    if top_p >= 1.0:
        cdf = probs.cumsum(-1)
        target = uniforms.float().view(-1, 1) * cdf[:, -1:]
        last = logits.shape[-1] - 1 - (probs > 0).flip(-1).float().argmax(-1)      # a token without mass is never drawn
        tok = torch.minimum((cdf <= target).sum(-1), last)
        return tok, logp_raw.gather(1, tok.view(-1, 1)).squeeze(1)
    keep = nucleus_mask(probs, top_p)
    cdf = (probs * keep).cumsum(-1)
    target = uniforms.float().view(-1, 1) * cdf[:, -1:]
    tok = (cdf <= target).sum(-1)
    # a nucleus that rounding extends to everything holds tokens without mass too: none of them is drawn
    last_kept = logits.shape[-1] - 1 - (keep & (probs > 0)).flip(-1).float().argmax(-1)
    tok = torch.minimum(tok, last_kept)
    return tok, logp_raw.gather(1, tok.view(-1, 1)).squeeze(1)


def nucleus_mask(probs, top_p: float):
    """Boolean [B, V]: tokens whose probability is >= that of the last token taken when accumulating ``top_p`` of mass
    from the most likely token down (the most likely token is always in)."""
    sp, _ = probs.sort(dim=-1, descending=True)
    taken = (sp.cumsum(-1) - sp) < top_p
    cut = torch.where(taken, sp, torch.full_like(sp, float("inf"))).amin(-1, keepdim=True)
    return probs >= cut
