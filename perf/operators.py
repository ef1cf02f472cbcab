"""What a decode step over a long paged KV cache costs: split attention, eviction by accumulated attention weight, and
the adjustment of logits (penalties, biases, grammar masks), each in a plain form and as this framework's own call.

``own`` selects the side: False computes the operators with elementary torch operations in 32 bits, True calls
``torchtitan_b200.ops.serving``.
"""

from __future__ import annotations

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------------- cases
def _attend(name, *, batch, tokens, heads, kv_heads, dim, page=16, ragged=False, window=0, sinks=False, scores=False,
            dtype="bf16"):
    return {"name": name, "op": "attend", "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": page, "ragged": ragged, "window": window, "sinks": sinks, "scores": scores, "dtype": dtype}


def _evict(name, *, batch, tokens, keep, recent, kv_heads, dim, page=16, ragged=False, dtype="bf16"):
    return {"name": name, "op": "evict", "batch": batch, "tokens": tokens, "keep": keep, "recent": recent, "kv_heads": kv_heads,
            "dim": dim, "page": page, "ragged": ragged, "dtype": dtype}


def _logits(name, *, batch, vocab, history, biases, mask, per_row, dtype="fp32"):
    return {"name": name, "op": "logits", "batch": batch, "vocab": vocab, "history": history, "biases": biases, "mask": mask,
            "per_row": per_row, "dtype": dtype}


def listed():
    return [
        # the first steps of a single chat: nothing but latency
        _attend("attend one short", batch=1, tokens=33, heads=32, kv_heads=8, dim=128),
        # one sequence at the end of a long document: 148 SMs have to share 8 kv heads
        _attend("attend one long", batch=1, tokens=131072, heads=32, kv_heads=8, dim=128),
        # a server's batch: requests of every age in one step, four kv heads, eight query heads each, weights accumulated
        _attend("attend ragged scored", batch=64, tokens=4096, heads=32, kv_heads=4, dim=128, ragged=True, scores=True),
        # rollouts of a policy update: many samples, two query heads to a kv head
        _attend("attend rollouts", batch=128, tokens=8192, heads=16, kv_heads=8, dim=128, ragged=True),
        # sliding-window layers with sink logits, half-size heads
        _attend("attend window sinks", batch=48, tokens=2500, heads=64, kv_heads=8, dim=64, page=32, ragged=True, window=128,
                sinks=True),
        # wide heads in half precision, sixteen query heads to a kv head, odd page size
        _attend("attend wide fp16", batch=6, tokens=5003, heads=64, kv_heads=4, dim=256, page=24, scores=True, dtype="fp16"),
        # one sequence that has outgrown its budget by a page or two
        _evict("evict one", batch=1, tokens=1056, keep=1024, recent=64, kv_heads=8, dim=128),
        # a batch of long rollouts cut back to a quarter
        _evict("evict ragged", batch=32, tokens=8192, keep=2048, recent=256, kv_heads=8, dim=128, ragged=True),
        # a long prompt compressed before the first token
        _evict("evict long prompt", batch=2, tokens=131072, keep=16384, recent=1024, kv_heads=4, dim=128, page=64),
        # one request with repetition penalties on bf16 logits
        _logits("logits one", batch=1, vocab=128256, history=200, biases=0, mask=False, per_row=False, dtype="bf16"),
        # a batch with everything on, each request with settings of its own
        _logits("logits batch", batch=256, vocab=151936, history=2048, biases=32, mask=True, per_row=True),
        # odd vocabulary, rows that do not start on vector boundaries, long histories
        _logits("logits odd long", batch=24, vocab=50021, history=32768, biases=300, mask=True, per_row=True, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    case = _drawn(rng)
    del case["name"]
    return case


def _drawn(rng):
    op = rng.choice(["attend", "attend", "evict", "logits"])
    if op == "attend":
        heads, kv = rng.choice([(32, 8), (16, 8), (32, 4), (64, 8), (64, 4), (40, 8), (16, 16), (7, 1), (20, 4), (16, 2), (128, 8)])
        dim = rng.choice([64, 128, 128, 256])
        batch = _log(rng, 1, 160)
        most = max(64, min(150000, (1 << 29) // (kv * dim * batch)))
        return _attend("", batch=batch, tokens=_log(rng, 1, most), heads=heads, kv_heads=kv, dim=dim,
                       page=rng.choice([8, 16, 16, 24, 32, 64, 128]), ragged=rng.random() < 0.7,
                       window=_log(rng, 16, 4096) if rng.random() < 0.25 else 0, sinks=rng.random() < 0.25,
                       scores=rng.random() < 0.3, dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if op == "evict":
        kv, dim = rng.choice([1, 2, 4, 8, 16]), rng.choice([64, 128, 128, 256])
        batch = _log(rng, 1, 64)
        tokens = _log(rng, 32, max(64, min(200000, (1 << 28) // (kv * dim * batch))))
        keep = max(1, int(tokens * rng.uniform(0.02, 0.98)))
        return _evict("", batch=batch, tokens=tokens, keep=keep, recent=int(keep * rng.choice([0.0, rng.random(), rng.random()])),
                      kv_heads=kv, dim=dim, page=rng.choice([8, 16, 16, 24, 32, 64, 128]), ragged=rng.random() < 0.6,
                      dtype=rng.choice(["bf16", "bf16", "fp16"]))
    batch = _log(rng, 1, 256)
    return _logits("", batch=batch, vocab=_log(rng, 1000, 150000), history=_log(rng, 1, min(40000, 1 + (1 << 22) // batch)),
                   biases=rng.choice([0, 1, 17, 300, 1000]), mask=rng.random() < 0.5, per_row=rng.random() < 0.5,
                   dtype=rng.choice(["fp32", "fp32", "bf16", "fp16"]))


# ------------------------------------------------------------------------------------------------------ inputs
def _lengths(case, gen):
    """Tokens of each sequence, on the host: all the same, or spread evenly up to the longest, in an order of the seed's."""
    B, n = case["batch"], case["tokens"]
    if not case["ragged"]:
        return [n] * B
    return [-(-n * (i + 1) // B) for i in torch.randperm(B, generator=gen).tolist()]


def _tables(lens, page, gen, extra=0):
    """Shuffled pages for every sequence (tables padded with page 0) and their number; ``extra`` pages more per sequence
    make a second table. The pages come in no order, as after hours of serving."""
    need = [-(-n // page) for n in lens]
    total = sum(need) + extra * len(lens)
    perm = torch.randperm(total, generator=gen).to(torch.int32)
    width = max(need)
    table = torch.zeros(len(lens), width, dtype=torch.int32)
    at = 0
    for b, w in enumerate(need):
        table[b, :w] = perm[at : at + w]
        at += w
    second = perm[at:].view(len(lens), extra) if extra else None
    return table, second, total


def prepare(case, seed):
    dev = torch.device("cuda")
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        t = torch.empty(*shape, dtype=dt, device=dev).normal_(generator=gen)
        return t if scale == 1.0 else t.mul_(scale)

    s = {"case": case}
    if case["op"] == "attend":
        lens = _lengths(case, host)
        table, _, pages = _tables(lens, case["page"], host)
        H, Hkv, D, P = case["heads"], case["kv_heads"], case["dim"], case["page"]
        s |= {"q": normal(case["batch"], H, D, scale=1.5), "k": normal(pages, P, Hkv, D), "v": normal(pages, P, Hkv, D),
              "tables": table.to(dev), "lens": torch.tensor(lens, dtype=torch.int32, device=dev), "scale": D**-0.5,
              "window": case["window"] or None,
              "sinks": torch.empty(H, device=dev).normal_(generator=gen) if case["sinks"] else None,
              "scores": torch.rand(pages, Hkv, P, generator=gen, device=dev) if case["scores"] else None}
    elif case["op"] == "evict":
        lens = _lengths(case, host)
        Hkv, D, P = case["kv_heads"], case["dim"], case["page"]
        table, second, pages = _tables(lens, P, host, extra=-(-min(case["keep"], max(lens)) // P))
        # accumulated weights: heavy-tailed, a tenth never looked at (equal values, so the order of ties counts)
        sc = torch.empty(pages, Hkv, P, device=dev).log_normal_(-4.0, 2.0, generator=gen)
        sc *= torch.rand(pages, Hkv, P, generator=gen, device=dev) > 0.1
        s |= {"k": normal(pages, P, Hkv, D), "v": normal(pages, P, Hkv, D), "scores": sc, "tables": table.to(dev),
              "new": second.to(dev), "lens": torch.tensor(lens, dtype=torch.int32, device=dev)}
    else:
        B, V, L = case["batch"], case["vocab"], case["history"]
        # what was said before follows a heavy-tailed distribution over the vocabulary; padding is -1
        u = torch.rand(B, L, generator=gen, device=dev)
        tokens = (V * u.pow(4)).to(torch.int32).clamp_(max=V - 1)
        lens = torch.randint(1, L + 1, (B,), generator=host)
        lens[B // 2] = L
        prompt = (lens * torch.rand(B, generator=host)).to(torch.int32)
        lens = lens.to(torch.int32).to(dev)
        tokens.masked_fill_(torch.arange(L, device=dev) >= lens.unsqueeze(1), -1)
        s |= {"logits": normal(B, V, scale=3.0), "tokens": tokens, "total": lens, "prompt": prompt.to(dev)}

        def setting(lo, hi):
            t = torch.rand(B, generator=host) * (hi - lo) + lo
            return t.to(dev) if case["per_row"] else float(t[0])

        s |= {"repetition": setting(1.0, 1.5), "presence": setting(0.0, 1.0), "frequency": setting(0.0, 0.5)}
        nb = case["biases"]
        ids = torch.randint(0, V, (B, nb), generator=host).to(torch.int32) if nb else None
        if nb > 2:  # the same token twice, and a shorter list padded with -1
            ids[:, 1] = ids[:, 0]
            ids[:, -1] = -1
        s |= {"bias_ids": ids.to(dev) if nb else None,
              "bias_values": torch.empty(B, nb, device=dev).normal_(0.0, 5.0, generator=gen) if nb else None}
        words = -(-V // 32)
        s["allowed"] = None
        if case["mask"]:  # grammars allow few tokens in some rows and most in others
            few = torch.randint(-(1 << 31), 1 << 31, (3, B, words), generator=gen, device=dev, dtype=torch.int64).to(torch.int32)
            s["allowed"] = torch.where((torch.arange(B, device=dev) % 2 == 0).view(B, 1), few[0] & few[1] & few[2], few[0] | few[1])
    return s


# -------------------------------------------------------------------------------------------------------- runs
def run(s):
    return {"attend": _run_attend, "evict": _run_evict, "logits": _run_logits}[s["case"]["op"]](s)


def _run_attend(s):
    if own:
        from torchtitan_b200.ops import serving

        out = serving.paged_attention_split(s["q"], s["k"], s["v"], s["tables"], s["lens"], s["scale"], window=s["window"],
                                            sinks=s["sinks"], scores=s["scores"])
        return {"out": out, "scores": s["scores"]}
    q, k, v, tables, lens, scores = s["q"], s["k"], s["v"], s["tables"], s["lens"].long(), s["scores"]
    B, H, D = q.shape
    P, Hkv = k.shape[1], k.shape[2]
    room = tables.shape[1] * P
    span = room if s["window"] is None else min(room, s["window"])
    first = torch.zeros_like(lens) if s["window"] is None else (lens - s["window"]).clamp(min=0)
    pos = first.unsqueeze(1) + torch.arange(span, device=q.device)
    live = pos < lens.unsqueeze(1)
    pos = pos.clamp(max=room - 1)
    page, off = tables.long().gather(1, pos // P), pos % P
    x = torch.einsum("bhgd,bnhd->bhgn", q.float().view(B, Hkv, H // Hkv, D), k[page, off].float()) * s["scale"]
    x = x.masked_fill(~live.view(B, 1, 1, span), float("-inf"))
    top = x.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        sink = s["sinks"].float().view(1, Hkv, H // Hkv, 1)
        top = torch.maximum(top, sink)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + torch.exp(sink - top)
    w = e / total
    out = torch.einsum("bhgn,bnhd->bhgd", w, v[page, off].float()).reshape(B, H, D).to(q.dtype)
    if scores is not None:
        at = (page.unsqueeze(1) * Hkv + torch.arange(Hkv, device=q.device).view(1, Hkv, 1)) * P + off.unsqueeze(1)
        scores.view(-1).scatter_add_(0, at.reshape(-1), w.sum(2).reshape(-1))
    return {"out": out, "scores": scores}


def _run_evict(s):
    keep, recent = s["case"]["keep"], s["case"]["recent"]
    if own:
        from torchtitan_b200.ops import serving

        lens, kept = serving.kv_cache_evict(s["k"], s["v"], s["scores"], s["tables"], s["lens"], s["new"], keep, recent)
        return {"lens": lens, "kept": kept, "k": s["k"], "v": s["v"], "scores": s["scores"]}
    k, v, scores, tables, new, lens = s["k"], s["v"], s["scores"], s["tables"].long(), s["new"].long(), s["lens"].long()
    B, P, Hkv = tables.shape[0], k.shape[1], k.shape[2]
    room = tables.shape[1] * P
    head = torch.arange(Hkv, device=k.device)
    pos = torch.arange(room, device=k.device)
    x = scores[tables].permute(0, 2, 1, 3).reshape(B, Hkv, room)
    age = lens.unsqueeze(1) - pos
    x = x.masked_fill((age <= recent).unsqueeze(1), float("inf")).masked_fill((age <= 0).unsqueeze(1), float("-inf"))
    most = min(keep, room)
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[..., :most]
    left = lens.clamp(max=keep)
    rank = torch.arange(most, device=k.device)
    valid = (rank < left.unsqueeze(1)).unsqueeze(1).expand(B, Hkv, most)
    order = order.masked_fill(~valid, room).sort(-1).values
    kept = torch.full((B, Hkv, keep), -1, dtype=torch.int32, device=k.device)
    kept[..., :most] = order.masked_fill(~valid, -1).to(torch.int32)
    src = torch.where(valid, order, order[..., :1])          # what is not there repeats the first row: the same values again
    dst = torch.where(valid, rank, 0)
    seq = torch.arange(B, device=k.device).view(B, 1, 1)
    sp, so, dp, do = tables[seq, src // P], src % P, new[seq, dst // P], dst % P
    h = head.view(1, Hkv, 1)
    k[dp, do, h] = k[sp, so, h]
    v[dp, do, h] = v[sp, so, h]
    scores[dp, h, do] = scores[sp, h, so]
    return {"lens": left.to(torch.int32), "kept": kept, "k": k, "v": v, "scores": scores}


def _run_logits(s):
    if own:
        from torchtitan_b200.ops import serving

        return serving.process_logits(s["logits"], s["tokens"], s["total"], s["prompt"], repetition_penalty=s["repetition"],
                                      presence_penalty=s["presence"], frequency_penalty=s["frequency"], bias_ids=s["bias_ids"],
                                      bias_values=s["bias_values"], allowed=s["allowed"])
    logits, tokens, V = s["logits"], s["tokens"], s["logits"].shape[1]
    B, L = tokens.shape

    def column(t):
        return t.view(B, 1) if torch.is_tensor(t) else t

    at = torch.arange(L, device=logits.device)
    live = (at < s["total"].unsqueeze(1)) & (tokens >= 0)
    said = live & (at >= s["prompt"].unsqueeze(1))
    ids = tokens.clamp(min=0).long()
    seen = torch.zeros(B, V, dtype=torch.int32, device=logits.device).scatter_add_(1, ids, live.to(torch.int32))
    count = torch.zeros(B, V, dtype=torch.int32, device=logits.device).scatter_add_(1, ids, said.to(torch.int32))
    x = logits.float()
    x = torch.where(seen > 0, torch.where(x > 0, x / column(s["repetition"]), x * column(s["repetition"])), x)
    x = x - column(s["frequency"]) * count - column(s["presence"]) * (count > 0)
    if s["bias_ids"] is not None:
        ok = s["bias_ids"] >= 0
        x = x + torch.zeros(B, V, device=x.device).scatter_add_(1, s["bias_ids"].clamp(min=0).long(), s["bias_values"] * ok)
    if s["allowed"] is not None:
        word = torch.arange(V, device=x.device)
        x = x.masked_fill(((s["allowed"][:, word // 32] >> (word % 32)) & 1) == 0, float("-inf"))
    return x.to(logits.dtype)


# -------------------------------------------------------------------------------------------------------- work
def work(case):
    """Bytes and operations that one pass cannot do without; lengths of ragged batches count with their mean."""
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "logits":
        B, V, nb = case["batch"], case["vocab"], case["biases"]
        return {"bytes": B * (2 * V * size + 4 * case["history"] / 2 + 8 * nb + (V / 8 if case["mask"] else 0)), "flops": B * V * 4}
    n = case["tokens"] * ((case["batch"] + 1) / (2 * case["batch"]) if case["ragged"] else 1.0)
    if case["op"] == "attend":
        n = min(n, case["window"]) if case["window"] else n
        rows = case["batch"] * n * case["kv_heads"]
        return {"bytes": rows * (2 * case["dim"] * size + (8 if case["scores"] else 0)) + 2 * case["batch"] * case["heads"] * case["dim"] * size,
                "flops": 4 * case["batch"] * n * case["heads"] * case["dim"]}
    rows = case["batch"] * case["kv_heads"]
    moved = min(n, case["keep"])
    return {"bytes": rows * (4 * n + moved * (2 * 2 * case["dim"] * size + 4 + 4)), "flops": rows * n}


# ------------------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "evict": _exact_evict, "logits": _exact_logits}[case["op"]](s)


def _exact_attend(s):
    """Sequence by sequence, softmax written out, in 64 bits."""
    q, k, v = s["q"].double(), s["k"], s["v"]
    B, H, D = q.shape
    P, Hkv = k.shape[1], k.shape[2]
    out = torch.zeros(B, H, D, dtype=torch.float64, device=q.device)
    scores = s["scores"].double() if s["scores"] is not None else None
    for b, n in enumerate(s["lens"].tolist()):
        lo = max(0, n - s["window"]) if s["window"] else 0
        pages = s["tables"][b, : -(-n // P)].long()
        keys = k[pages].reshape(-1, Hkv, D)[lo:n].double().transpose(0, 1)       # [Hkv, tokens, D]
        vals = v[pages].reshape(-1, Hkv, D)[lo:n].double().transpose(0, 1)
        x = torch.bmm(q[b].view(Hkv, H // Hkv, D), keys.transpose(1, 2)) * s["scale"]
        den = torch.logsumexp(x, -1, keepdim=True)
        if s["sinks"] is not None:
            den = torch.logaddexp(den, s["sinks"].double().view(Hkv, H // Hkv, 1))
        w = torch.exp(x - den)
        out[b] = torch.bmm(w, vals).reshape(H, D)
        if scores is not None:
            t = torch.arange(lo, n, device=q.device)
            scores[pages[t // P], :, t % P] += w.sum(1).t()
    return {"out": out, "scores": scores}


def _exact_evict(s):
    """Head by head: the tokens sorted by (score, earlier first), the best of them put back in order."""
    keep, recent = s["case"]["keep"], s["case"]["recent"]
    k, v, sc = s["k"], s["v"], s["scores"]
    P, Hkv = k.shape[1], k.shape[2]
    lens = s["lens"].tolist()
    moves = []
    for b, n in enumerate(lens):
        pages, to = s["tables"][b].long(), s["new"][b].long()
        for h in range(Hkv):
            old = max(0, n - recent)
            x = sc[pages, h].reshape(-1)[:old].double()
            best = torch.argsort(-x, stable=True)[: max(0, keep - (n - old))] if n > keep else torch.arange(old, device=x.device)
            idx = torch.cat((best.sort().values, torch.arange(old, n, device=x.device)))
            j = torch.arange(idx.numel(), device=x.device)
            moves.append((pages[idx // P], idx % P, to[j // P], j % P, torch.full_like(j, h)))
    sp, so, dp, do, h = (torch.cat(t) for t in zip(*moves))
    k[dp, do, h], v[dp, do, h], sc[dp, h, do] = k[sp, so, h], v[sp, so, h], sc[sp, h, so]
    return {"lens": None, "kept": None, "k": k, "v": v, "scores": sc.double()}


def _exact_logits(s):
    """Row by row, counts from a bincount, in 64 bits."""
    x = s["logits"].double()
    B, V = x.shape
    total, prompt = s["total"].tolist(), s["prompt"].tolist()

    def of(t, b):
        return float(t[b]) if torch.is_tensor(t) else t

    bit = torch.arange(V, device=x.device)
    for b in range(B):
        seen = torch.bincount(s["tokens"][b, : total[b]].long(), minlength=V) > 0
        count = torch.bincount(s["tokens"][b, prompt[b] : total[b]].long(), minlength=V).double()
        r = of(s["repetition"], b)
        x[b] = torch.where(seen, torch.where(x[b] > 0, x[b] / r, x[b] * r), x[b])
        x[b] -= of(s["frequency"], b) * count + of(s["presence"], b) * (count > 0).double()
        if s["bias_ids"] is not None:
            ids = s["bias_ids"][b].long()
            x[b].index_add_(0, ids[ids >= 0], s["bias_values"][b][ids >= 0].double())
        if s["allowed"] is not None:
            w = s["allowed"][b].long() & 0xFFFFFFFF
            x[b][(w[bit // 32] >> (bit % 32)) & 1 == 0] = float("-inf")
    return x
