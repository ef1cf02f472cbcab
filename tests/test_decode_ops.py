"""Decode-time ops over a paged KV cache: split attention, eviction by accumulated weight, logit adjustment.

Each against a plain definition in 64 bits, on the CPU and (``-m gpu``) on the kernels. Tolerances: a rounding to type t is
off by at most ``finfo(t).eps / 2`` relative to the value. Attention adds to that the fp32 arithmetic before it: a dot product
of D terms is off by at most ``D * 2^-23`` of the sum of its terms' sizes S (2^-23 instead of 2^-24: tensor cores may
truncate), an exponential's argument error carries over relative to the weight, the weights go into the second product with
at least 16 bits (2^-16), and a sum of n of them is off by at most ``n * 2^-23``, numerator and denominator each.
"""

import math

import pytest
import torch

from torchtitan_b200.ops import serving

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def make_cache(lens, *, hkv, dim, page, dtype, device, seed=0, packed=False, spare=3, table_dtype=torch.int32, width=0):
    """Caches whose unused slots hold NaN and infinities, tables of shuffled pages (padded with 0), lengths."""
    g = _gen(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    perm = torch.randperm(pages, generator=g)
    table = torch.zeros(len(lens), max(max(need, default=0), 1, width), dtype=table_dtype)
    shape = (pages, page, 2, hkv, dim) if packed else (2, pages, page, hkv, dim)
    kv = torch.full(shape, float("nan"))
    kv.view(-1)[::3] = float("inf")
    kv = kv.to(dtype)
    k, v = (kv[:, :, 0], kv[:, :, 1]) if packed else (kv[0], kv[1])
    at = 0
    for b, n in enumerate(lens):
        own = perm[at : at + need[b]]
        at += need[b]
        table[b, : need[b]] = own.to(table_dtype)
        t = torch.arange(n)
        k[own[t // page], t % page] = torch.randn(n, hkv, dim, generator=g).to(dtype)
        v[own[t // page], t % page] = torch.randn(n, hkv, dim, generator=g).to(dtype)
    free = perm[at:].to(table_dtype)
    if device != "cpu":
        kv = kv.to(device)
        k, v = (kv[:, :, 0], kv[:, :, 1]) if packed else (kv[0], kv[1])
    return k, v, table.to(device), torch.tensor(lens, dtype=table_dtype, device=device), free


def rows_of(cache, table, n):
    page = cache.shape[1]
    t = torch.arange(n, device=cache.device)
    return cache[table[t // page].long(), t % page]


def attention_oracle(q, k, v, table, lens, scale, window=None, sinks=None):
    """(out, lse, weights per sequence [Hkv, n], the sizes that errors are relative to), in 64 bits on the CPU."""
    q, k, v, table = q.cpu().double(), k.cpu(), v.cpu(), table.cpu()
    B, H, D = q.shape
    hkv = k.shape[2]
    out, lse = torch.zeros(B, H, D, dtype=torch.float64), torch.full((B, H), -math.inf, dtype=torch.float64)
    weights, size, dots = [], torch.zeros(B, H, D, dtype=torch.float64), torch.zeros(B, H, dtype=torch.float64)
    for b, n in enumerate(lens.tolist()):
        lo = max(0, n - window) if window else 0
        keys = rows_of(k, table[b], n)[lo:].double().repeat_interleave(H // hkv, 1).transpose(0, 1)   # [H, n, D]
        vals = rows_of(v, table[b], n)[lo:].double().repeat_interleave(H // hkv, 1).transpose(0, 1)
        x = torch.einsum("hd,hnd->hn", q[b], keys) * scale
        full = x if sinks is None else torch.cat((x, sinks.cpu().double().view(H, 1)), 1)
        if full.shape[1]:
            lse[b] = torch.logsumexp(full, 1)
        w = torch.exp(x - lse[b].nan_to_num(neginf=0.0).view(H, 1))
        out[b] = torch.einsum("hn,hnd->hd", w, vals)
        size[b] = torch.einsum("hn,hnd->hd", w, vals.abs())
        if n > lo:
            dots[b] = torch.einsum("hd,hnd->hn", q[b].abs(), keys.abs()).amax(1) * scale
        weights.append(torch.cat((torch.zeros(hkv, lo, dtype=torch.float64), w.view(hkv, H // hkv, n - lo).sum(1)), 1))
    return out, lse, weights, size, dots


def check_attention(got, oracle, n_max, dim, dtype, lse=None, scores=None, before=None, table=None):
    out, ref_lse, weights, size, dots = oracle
    arg = dim * 2**-23 * dots + 2**-20                          # error of an exponential's argument (natural log)
    rel = 2 * (arg + n_max * 2**-23) + 2**-16
    tol = (torch.finfo(dtype).eps / 2 if dtype != FP32 else 2**-23) * out.abs() * 1.01 + size * rel.unsqueeze(-1)
    err = (got.cpu().double() - out).abs()
    assert torch.isfinite(got).all()
    assert (err <= tol + 1e-30).all(), float((err / (tol + 1e-30)).max())
    if lse is not None:
        fine = torch.isfinite(ref_lse)
        assert torch.equal(lse.cpu()[~fine].double(), ref_lse[~fine])
        assert ((lse.cpu().double() - ref_lse).abs()[fine] <= (arg + n_max * 2**-23 + ref_lse.abs() * 2**-22)[fine]).all()
    if scores is not None:
        page = scores.shape[2]
        worst = float(rel.max())
        want = before.cpu().double().clone()
        hkv = scores.shape[1]
        bound = torch.zeros_like(want)
        for b, w in enumerate(weights):
            t = torch.arange(w.shape[1])
            pages = table.cpu()[b].long()[t // page]
            for h in range(hkv):
                want[pages, h, t % page] += w[h]
                bound[pages, h, t % page] += w[h] * worst
        assert ((scores.cpu().double() - want).abs() <= bound + want.abs() * 2**-23).all()


ATTENTION_CASES = [
    # lens, H, Hkv, D, page, dtype, options
    ([1], 8, 8, 128, 16, BF16, {}),
    ([0, 1, 15, 16, 17], 8, 2, 128, 16, BF16, {}),
    ([255, 256, 257, 64, 63], 16, 2, 64, 16, BF16, {"scores": True}),
    ([300, 5, 1029], 6, 2, 128, 7, FP16, {"scores": True, "sinks": True}),
    ([33, 700], 7, 1, 64, 1, BF16, {"packed": True}),
    ([513, 40], 40, 2, 128, 32, BF16, {"sinks": True, "scores": True}),
    ([100, 31], 64, 2, 64, 24, FP16, {"window": 32, "scores": True}),
    ([1000, 3, 0, 129], 16, 1, 256, 64, BF16, {"window": 130, "sinks": True, "scores": True}),
    ([700, 16, 5], 8, 4, 128, 8, FP16, {"window": 1, "scores": True}),
    ([90, 1], 4, 4, 256, 128, FP16, {"packed": True, "scores": True, "long": True}),
    ([2500, 17], 12, 4, 128, 16, BF16, {"window": 100000, "wide": 400, "scores": True}),
    ([50, 0, 19], 4, 2, 48, 16, FP32, {"scores": True, "sinks": True, "window": 20}),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("case", range(len(ATTENTION_CASES)))
def test_split_attention(case, device):
    lens, H, hkv, D, page, dtype, opt = ATTENTION_CASES[case]
    k, v, table, n, _ = make_cache(lens, hkv=hkv, dim=D, page=page, dtype=dtype, device=device, seed=case, packed=opt.get("packed", False),
                                   table_dtype=torch.int64 if opt.get("long") else torch.int32, width=opt.get("wide", 0))
    g = _gen(100 + case)
    q = (torch.randn(len(lens), 2, H, D, generator=g) * 2).to(dtype).to(device)[:, 1]           # rows with a stride of their own
    sinks = torch.randn(H, generator=g).to(device) if opt.get("sinks") else None
    scores = torch.rand(k.shape[0], hkv, page, generator=g).to(device) if opt.get("scores") else None
    before = scores.clone() if scores is not None else None
    out, lse = serving.paged_attention_split(q, k, v, table, n, D**-0.5, window=opt.get("window"), sinks=sinks, scores=scores,
                                             return_lse=True)
    assert out.dtype == dtype and lse.dtype == FP32
    oracle = attention_oracle(q, k, v, table, n, D**-0.5, opt.get("window"), sinks)
    check_attention(out, oracle, max(lens), D, dtype, lse, scores, before, table)
    for b, ln in enumerate(lens):
        if ln == 0:
            assert (out[b] == 0).all()
    again = serving.paged_attention_split(q, k, v, table, n, D**-0.5, window=opt.get("window"), sinks=sinks)
    assert torch.equal(out, again)                              # with and without weights and lse: the same bits


@pytest.mark.parametrize("device", DEVICES)
def test_split_attention_sinks_of_minus_infinity_and_shared_pages(device):
    k, v, table, n, _ = make_cache([40, 40], hkv=2, dim=64, page=16, dtype=BF16, device=device)
    table[1] = table[0]
    q = torch.randn(2, 4, 64, generator=_gen(1)).to(BF16).to(device)
    none = torch.full((4,), -math.inf, device=device)
    scores = torch.zeros(k.shape[0], 2, 16, device=device)
    out = serving.paged_attention_split(q, k, v, table, n, 0.125, sinks=none, scores=scores)
    assert torch.equal(out, serving.paged_attention_split(q, k, v, table, n, 0.125))
    # both sequences' weights: each sums to one per query head
    assert abs(float(scores.double().sum()) - 2 * 4) <= 8 * (40 * 2**-23 + 2**-14)


@pytest.mark.parametrize("device", DEVICES)
def test_split_attention_extreme_logits(device):
    """One token takes all the weight, at the start, the middle and the end, with logits of +-10^4."""
    D, n = 64, 600
    for at in (0, 257, n - 1):
        k, v, table, lens, _ = make_cache([n], hkv=1, dim=D, page=16, dtype=BF16, device=device)
        q = torch.full((1, 2, D), 100.0, device=device).to(BF16)
        k[table[0].long()] = -1.0
        k[table[0, at // 16].long(), at % 16] = 1.0
        out = serving.paged_attention_split(q, k, v, table, lens, 1.0)
        assert torch.equal(out, rows_of(v, table[0], n)[at].expand(1, 2, D))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_split_attention_many_small_weights(device, dtype):
    """One token far ahead of very many equal ones, which together hold half of the weight: each of their weights is far below
    what fp16 can hold next to the largest."""
    D, n = 64, 50000
    k, v, table, lens, _ = make_cache([n], hkv=1, dim=D, page=64, dtype=dtype, device=device)
    q = torch.zeros(1, 2, D, device=device, dtype=dtype)
    q[..., 0], q[:, 1, 1] = 1.0, 0.03125
    k[table[0].long()] = 0.0
    k[..., 0] = -10.8125                                                   # e^-10.8 = 1 / 49600
    k[..., 1] = 0.25
    k[table[0, 300].long(), 7] = 0.0
    v[table[0].long()] += 3.0                                              # a mean that errors of one sign would shift
    out, lse = serving.paged_attention_split(q, k, v, table, lens, 1.0, return_lse=True)
    check_attention(out, attention_oracle(q, k, v, table, lens, 1.0), n, D, dtype, lse)


@pytest.mark.parametrize("device", DEVICES)
def test_split_attention_sink_of_infinity_takes_everything(device):
    k, v, table, n, _ = make_cache([40, 1200], hkv=2, dim=64, page=16, dtype=BF16, device=device)
    q = torch.randn(2, 4, 64, generator=_gen(1)).to(BF16).to(device)
    sinks = torch.tensor([math.inf, 0.0, math.inf, -math.inf], device=device)
    scores = torch.zeros(k.shape[0], 2, 16, device=device)
    out, lse = serving.paged_attention_split(q, k, v, table, n, 0.125, sinks=sinks, scores=scores, return_lse=True)
    assert (out[:, ::2] == 0).all() and (lse[:, ::2] == math.inf).all() and torch.isfinite(scores).all()
    assert torch.equal(out[:, 3], serving.paged_attention_split(q, k, v, table, n, 0.125)[:, 3])


def test_split_attention_refusals():
    k, v, table, n, _ = make_cache([20, 3], hkv=2, dim=64, page=16, dtype=BF16, device="cpu")
    q = torch.randn(2, 4, 64).to(BF16)

    def call(**kw):
        a = {"q": q, "k_cache": k, "v_cache": v, "block_tables": table, "context_lens": n, "scale": 0.125} | kw
        return serving.paged_attention_split(**a)

    call()
    scores = torch.zeros(k.shape[0], 2, 16)
    for kw, err in [
        ({"q": q[0]}, ValueError), ({"q": q.float()}, TypeError), ({"q": q[:, :3]}, ValueError), ({"q": q[..., :32]}, ValueError),
        ({"q": q[:1]}, ValueError), ({"k_cache": k[0]}, ValueError), ({"v_cache": v[:, :8]}, ValueError), ({"v_cache": v.float()}, TypeError),
        ({"block_tables": table.float()}, TypeError), ({"block_tables": table[:1]}, ValueError), ({"context_lens": n.short()}, TypeError),
        ({"context_lens": n.view(2, 1)}, ValueError), ({"context_lens": n + 100}, ValueError), ({"context_lens": n - 4}, ValueError),
        ({"block_tables": table + 1000}, ValueError), ({"block_tables": table - 1000}, ValueError), ({"window": 0}, ValueError), ({"window": 2.5}, ValueError),
        ({"sinks": torch.zeros(3)}, ValueError), ({"scores": scores.double()}, TypeError), ({"scores": scores.transpose(1, 2)}, ValueError),
        ({"scores": scores[:1]}, ValueError), ({"q": q.clone().requires_grad_()}, RuntimeError), ({"k_cache": k[:0], "v_cache": v[:0]}, ValueError),
        ({"q": q.int(), "k_cache": k.int(), "v_cache": v.int()}, TypeError),
    ]:
        with pytest.raises(err):
            call(**kw)
    with torch.no_grad():
        call(q=q.clone().requires_grad_())
    assert serving.paged_attention_split(q[:0], k, v, table[:0], n[:0], 0.125).shape == (0, 4, 64)
    assert (serving.paged_attention_split(q, k, v, table[:, :0], n * 0, 0.125) == 0).all()


# ------------------------------------------------------------------------------------------------------- eviction
def evict_oracle(scores, table, lens, keep, recent):
    """Kept tokens of every (sequence, head): sorted in Python by (larger score first, lower index first)."""
    scores, table = scores.cpu(), table.cpu()
    page = scores.shape[2]
    kept = []
    for b, n in enumerate(lens.tolist()):
        for h in range(scores.shape[1]):
            s = [float(scores[int(table[b, t // page]), h, t % page]) for t in range(n)]
            old = list(range(n)) if n <= keep else sorted(range(n - recent), key=lambda t: (not math.isnan(s[t]), -s[t] if s[t] == s[t] else 0.0, t))
            idx = old if n <= keep else sorted(old[: keep - recent]) + list(range(n - recent, n))
            kept.append(idx + [-1] * (keep - len(idx)))
    return torch.tensor(kept, dtype=torch.int32).view(len(lens), -1, keep)


EVICT_CASES = [
    # lens, Hkv, D, page, dtype, keep, recent, distribution
    ([10], 1, 8, 4, BF16, 3, 1, "ties"),
    ([1, 5, 6, 7, 0], 2, 64, 16, BF16, 6, 0, "spread"),
    ([100, 99, 30], 3, 128, 7, FP16, 40, 40, "spread"),
    ([1500, 2049, 64], 2, 64, 16, BF16, 1024, 100, "zeros"),
    ([3000, 1200], 4, 16, 32, FP32, 1100, 1, "ties"),
    ([257, 513], 2, 64, 1, BF16, 256, 255, "special"),
    ([5000], 2, 64, 64, FP16, 1, 0, "special"),
    ([4097, 12], 1, 128, 128, BF16, 4096, 64, "equal"),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("case", range(len(EVICT_CASES)))
def test_evict(case, device):
    lens, hkv, D, page, dtype, keep, recent, kind = EVICT_CASES[case]
    width = -(-min(keep, max(lens)) // page)
    k, v, table, n, free = make_cache(lens, hkv=hkv, dim=D, page=page, dtype=dtype, device=device, seed=case, packed=case % 2 == 1,
                                      spare=width * len(lens) + 2)
    fresh = free[: width * len(lens)].view(len(lens), width).to(device)
    g = _gen(case)
    s = torch.empty(k.shape[0], hkv, page).log_normal_(-3.0, 2.0, generator=g)
    if kind == "zeros":
        s *= torch.rand(s.shape, generator=g) > 0.7
    elif kind == "ties":
        s = torch.randint(0, 3, s.shape, generator=g).float()
        s[::2] *= -1.0                                           # negative values and both zeros
    elif kind == "special":
        r = torch.randint(0, 12, s.shape, generator=g)
        s[r == 0], s[r == 1], s[r == 2], s[r == 3] = math.nan, math.inf, -math.inf, 1e-42
    elif kind == "equal":
        s.fill_(0.25)
    s = s.to(device)
    k0, v0, s0 = k.clone(), v.clone(), s.clone()
    new_lens, kept = serving.kv_cache_evict(k, v, s, table, n, fresh, keep, recent)
    want = evict_oracle(s0, table, n, keep, recent)
    assert new_lens.dtype == torch.int32 and new_lens.tolist() == [min(x, keep) for x in lens]
    assert kept.dtype == torch.int32 and torch.equal(kept.cpu(), want)
    # the caches: kept rows on the new pages, everything else as it was (bits, so that NaN compare)
    as_int = {2: torch.int16, 4: torch.int32}[k.element_size()]
    for cache, orig in ((k, k0), (v, v0)):
        exp = orig.clone()
        for b in range(len(lens)):
            for h in range(hkv):
                idx = want[b, h][want[b, h] >= 0].long().to(device)
                j = torch.arange(len(idx), device=device)
                exp[fresh[b].long()[j // page], j % page, h] = orig[table[b].long()[idx // page], idx % page, h]
        assert torch.equal(cache.contiguous().view(as_int), exp.contiguous().view(as_int))
    exp = s0.clone()
    for b in range(len(lens)):
        for h in range(hkv):
            idx = want[b, h][want[b, h] >= 0].long().to(device)
            j = torch.arange(len(idx), device=device)
            exp[fresh[b].long()[j // page], h, j % page] = s0[table[b].long()[idx // page], h, idx % page]
    assert torch.equal(s.view(torch.int32), exp.view(torch.int32))


def test_evict_refusals():
    k, v, table, n, free = make_cache([40, 20], hkv=2, dim=64, page=16, dtype=BF16, device="cpu", spare=8)
    s, fresh = torch.rand(k.shape[0], 2, 16), free[:4].view(2, 2)

    def call(**kw):
        a = {"k_cache": k.clone(), "v_cache": v.clone(), "scores": s.clone(), "block_tables": table, "context_lens": n, "new_tables": fresh,
             "keep": 32, "recent": 4} | kw
        return serving.kv_cache_evict(**a)

    call()
    for kw, err in [
        ({"keep": 0}, ValueError), ({"keep": 32.0}, ValueError), ({"recent": 33}, ValueError), ({"recent": -1}, ValueError), ({"keep": 33}, ValueError),
        ({"scores": None}, ValueError), ({"scores": s.half()}, TypeError), ({"new_tables": fresh.float()}, TypeError),
        ({"new_tables": fresh[:1]}, ValueError), ({"new_tables": fresh + 1000}, ValueError), ({"new_tables": table[:, :2]}, ValueError),
        ({"new_tables": fresh[:1].expand(2, 2)}, ValueError), ({"context_lens": n + 100}, ValueError), ({"v_cache": v[1:]}, ValueError),
        ({"k_cache": k.clone().requires_grad_()}, RuntimeError),
    ]:
        with pytest.raises(err):
            call(**kw)


# --------------------------------------------------------------------------------------------------------- logits
def logits_oracle(x, tokens, lens, prompts, rep, pres, freq, bias, allowed):
    """Row by row and token by token, in 64 bits; also the largest size that a step went through."""
    y, size = x.cpu().double(), x.cpu().double().abs()
    B, V = y.shape
    of = lambda p, b: float(p[b]) if torch.is_tensor(p) else float(p)  # noqa: E731
    for b in range(B):
        hist = [] if tokens is None else tokens[b, : int(lens[b])].tolist()
        out = hist[int(prompts[b]) :] if prompts is not None else hist
        for t in {t for t in hist if 0 <= t < V}:
            y[b, t] = y[b, t] / of(rep, b) if y[b, t] > 0 else y[b, t] * of(rep, b)
        size[b] = torch.maximum(size[b], y[b].abs())
        for t in {t for t in out if 0 <= t < V}:
            y[b, t] -= of(freq, b) * out.count(t)
            size[b, t] = max(float(size[b, t]), abs(float(y[b, t])), of(freq, b) * out.count(t))
            y[b, t] -= of(pres, b)
            size[b, t] = max(float(size[b, t]), abs(float(y[b, t])))
        if bias is not None:
            for t, w in zip(bias[0][b].tolist(), bias[1][b].double().tolist()):
                if 0 <= t < V:
                    size[b, t] = max(float(size[b, t]), 0.0) + abs(w)
                    y[b, t] += w
        if allowed is not None:
            for i in range(V):
                if not (int(allowed[b, i // 32]) >> (i % 32)) & 1:
                    y[b, i] = -math.inf
    return y, size


LOGIT_CASES = [
    # B, V, dtype, history, options
    (1, 1, FP32, 1, {}),
    (3, 31, BF16, 7, {"bias": 3}),
    (2, 33, FP16, 40, {"mask": True}),
    (4, 1000, FP32, 100, {"bias": 50, "mask": True, "rows": True}),
    (2, 4097, BF16, 900, {"bias": 1024, "mask": True, "rows": True, "long": True}),
    (2, 9001, FP32, 0, {"mask": True}),
    (3, 8192, FP32, None, {"bias": 5}),
    (2, 5003, FP16, 300, {"rows": True, "strided": True, "bias": 9, "mask": True}),
    (2, 20011, BF16, 5000, {"inplace": True, "mask": True}),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("case", range(len(LOGIT_CASES)))
def test_process_logits(case, device):
    B, V, dtype, L, opt = LOGIT_CASES[case]
    g = _gen(case)
    wide = torch.randn(B, V + 5, generator=g) * 4
    if V > 30:
        wide[:, 3], wide[:, 4], wide[:, 5] = math.inf, -math.inf, 0.0
    x = (wide[:, 2 : 2 + V] if opt.get("strided") else wide[:, :V].contiguous()).to(dtype)
    idt = torch.int64 if opt.get("long") else torch.int32
    tokens = lens = prompts = None
    if L is not None:
        tokens = (V * torch.rand(B, L, generator=g) ** 3).to(idt).clamp(max=V - 1)
        lens = torch.randint(0, L + 1, (B,), generator=g).to(idt)
        lens[-1] = L
        prompts = (lens * torch.rand(B, generator=g)).to(idt)
        tokens[:, ::7] = -1
    setting = lambda lo, hi: torch.rand(B, generator=g) * (hi - lo) + lo if opt.get("rows") else lo + 0.3 * (hi - lo)  # noqa: E731
    rep, pres, freq = (setting(0.5, 2.0), setting(-1.0, 1.0), setting(0.0, 0.7)) if L is not None else (1.0, 0.0, 0.0)
    bias = None
    if opt.get("bias"):
        ids = torch.randint(0, V, (B, opt["bias"]), generator=g).to(idt)
        ids[:, 1::4] = ids[:, 0:1]                               # the same token several times
        ids[:, 2::9] = -1
        bias = (ids, torch.randn(B, opt["bias"], generator=g) * 3)
    allowed = None
    if opt.get("mask"):
        allowed = torch.randint(-(2**31), 2**31, (B, -(-V // 32) + 1), generator=g).to(torch.int32)
        allowed[0] = 0                                           # a row that may say nothing
    d = lambda t: t.to(device) if torch.is_tensor(t) else t  # noqa: E731
    xd = x.clone().to(device) if not opt.get("strided") else wide.to(dtype).to(device)[:, 2 : 2 + V]
    keep = xd.clone()
    out = xd if opt.get("inplace") else None
    got = serving.process_logits(xd, d(tokens), d(lens), d(prompts), repetition_penalty=d(rep), presence_penalty=d(pres),
                                 frequency_penalty=d(freq), bias_ids=d(bias[0]) if bias else None, bias_values=d(bias[1]) if bias else None,
                                 allowed=d(allowed), out=out)
    assert got.dtype == dtype and (got is xd) == bool(opt.get("inplace"))
    if not opt.get("inplace"):
        assert torch.equal(xd.nan_to_num(), keep.nan_to_num())
    want, size = logits_oracle(x, tokens, lens, prompts, rep, pres, freq, bias, allowed)
    got = got.cpu().double()
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine], want[~fine])
    steps = 4 + (opt.get("bias") or 0)                           # fp32 roundings, each half a step of the largest size on the way
    tol = size * steps * 2**-24 + (torch.finfo(dtype).eps / 2 * want.abs() * 1.01 if dtype != FP32 else 0.0)
    assert ((got - want).abs()[fine] <= tol[fine]).all()
    same = fine & (want == x.double()) & (size == x.double().abs())
    assert torch.equal(got[same], x.double()[same])              # what nothing applies to keeps its bits


def test_process_logits_refusals():
    x, tok = torch.randn(2, 40), torch.randint(0, 40, (2, 5))
    ids, val = torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3)
    ok = torch.full((2, 2), -1, dtype=torch.int32)
    serving.process_logits(x, tok, bias_ids=ids, bias_values=val, allowed=ok)
    for args, kw, err in [
        ((x[0],), {}, ValueError), ((x.double(),), {}, TypeError), ((x, tok.float()), {}, TypeError), ((x, tok[:1]), {}, ValueError),
        ((x, tok, tok), {}, ValueError), ((x,), {"repetition_penalty": 1.2}, ValueError), ((x, None, torch.ones(2, dtype=torch.int32)), {}, ValueError),
        ((x, tok), {"repetition_penalty": 0.0}, ValueError), ((x, tok), {"repetition_penalty": math.nan}, ValueError),
        ((x, tok), {"repetition_penalty": torch.tensor([1.0, -1.0])}, ValueError), ((x, tok), {"presence_penalty": math.inf}, ValueError),
        ((x, tok), {"frequency_penalty": torch.zeros(3)}, ValueError), ((x, tok), {"presence_penalty": torch.zeros(2).double()}, ValueError),
        ((x,), {"bias_ids": ids}, ValueError), ((x,), {"bias_values": val}, ValueError), ((x,), {"bias_ids": ids, "bias_values": val[:, :2]}, ValueError),
        ((x,), {"bias_ids": ids + 40, "bias_values": val}, ValueError), ((x, tok + 40), {}, ValueError),
        ((x,), {"bias_ids": ids.expand(2, 3).repeat(1, 400), "bias_values": val.repeat(1, 400)}, ValueError),
        ((x,), {"allowed": ok[:, :1]}, ValueError), ((x,), {"allowed": ok.long()}, ValueError), ((x,), {"out": x.half()}, ValueError),
        ((x,), {"out": x[:1]}, ValueError), ((x.clone().requires_grad_(),), {}, RuntimeError),
    ]:
        with pytest.raises(err):
            serving.process_logits(*args, **kw)
    base = torch.randn(2, 80)
    with pytest.raises(ValueError):
        serving.process_logits(base[:, :40], out=base[:, 1:41])
    with pytest.raises(ValueError, match="overlap"):
        serving.process_logits(base[:1].expand(2, 80), out=base[:1].expand(2, 80))
    assert serving.process_logits(x[:0]).shape == (0, 40)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("top_p", [1.0, 0.9])
def test_sampler_never_draws_a_masked_token(device, top_p):
    """Draws at both ends of the distribution, with the first and last tokens masked."""
    V = 3001
    x = torch.randn(4, V, generator=_gen(5)).to(device)
    allowed = torch.zeros(4, -(-V // 32), dtype=torch.int32, device=device)
    allowed[:, 40], allowed[:, 2] = 1 << 5, 1 << 30                   # tokens 1285 and 94
    y = serving.process_logits(x, allowed=allowed)
    for u in (0.0, 0.5, 1.0 - 2**-24, 1.0):                           # 1.0: a target at the total, which rounding can produce
        tok, lp = serving.sample_top_p(y, 1.0, top_p, torch.full((4,), u, device=device))
        assert set(tok.tolist()) <= {94, 1285} and torch.isfinite(lp).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("temperature,top_p", [(0.0, 1.0), (1.0, 1.0), (0.7, 0.9)])
@pytest.mark.parametrize("V", [1, 33, 3001, 50021])
def test_sampler_of_rows_that_allow_nothing(V, temperature, top_p, dtype, device):
    """A row whose mask leaves nothing gives token 0 and a NaN log-probability, and its neighbours what they give alone."""
    x = torch.randn(5, V, generator=_gen(V)).to(dtype).to(device)
    allowed = torch.full((5, -(-V // 32)), -1, dtype=torch.int32, device=device)
    allowed[1], allowed[4] = 0, 0
    u = torch.tensor([0.0, 0.5, 0.9, 0.3, 1.0 - 2**-24], device=device)
    tok, lp = serving.sample_top_p(serving.process_logits(x, allowed=allowed), temperature, top_p, u)
    some = [0, 2, 3]
    want, want_lp = serving.sample_top_p(x[some], temperature, top_p, u[some])
    assert tok[[1, 4]].tolist() == [0, 0] and lp[[1, 4]].isnan().all()
    assert torch.equal(tok[some], want) and torch.equal(lp[some], want_lp)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("top_p", [1.0, 0.9])
def test_sampler_of_rows_without_a_distribution(top_p, device):
    """Drawing from logits with NaN or infinity in them: a token of the vocabulary, marked by its log-probability."""
    x = torch.randn(3, 2049, generator=_gen(2)).to(device)
    x[0, 700], x[1, 1500], x[2] = math.nan, math.inf, math.nan
    tok, lp = serving.sample_top_p(x, 1.0, top_p, torch.tensor([0.2, 0.5, 0.99], device=device))
    assert tok.tolist() == [0, 0, 0] and lp.isnan().all()


# ------------------------------------------------------------------------------------------ together, as a program uses them
@pytest.mark.parametrize("device", DEVICES)
def test_decode_steps_with_a_bounded_cache(device):
    """Thirty decode steps of three sequences: write, attend with weights, cut back, adjust logits, draw -- against lists of
    rows in 64 bits."""
    B, H, hkv, D, page, keep, recent, slack, V = 3, 4, 2, 64, 4, 12, 3, 4, 64
    g = _gen(3)
    pages = 64
    k = torch.full((pages, page, hkv, D), float("nan"), dtype=BF16, device=device)
    v, scores = torch.full_like(k, float("nan")), torch.zeros(pages, hkv, page, device=device)
    proj = torch.randn(H * D, V, generator=g).double() * 0.2
    free = torch.randperm(pages, generator=g).tolist()
    blocks, length = [[] for _ in range(B)], [0] * B
    history = torch.full((B, 40), -1, dtype=torch.int32)
    rows = [[[] for _ in range(hkv)] for _ in range(B)]               # oracle: (k, v, score, position) per head
    evictions = 0
    for step in range(30):
        over = [b for b in range(B) if length[b] >= keep + slack]
        if over:
            evictions += len(over)
            new = [[free.pop() for _ in range(-(-keep // page))] for _ in over]
            scores[torch.tensor(new).view(-1)] = 0.0
            wide = max(len(blocks[b]) for b in over)
            old = torch.tensor([blocks[b] + [0] * (wide - len(blocks[b])) for b in over], dtype=torch.int32, device=device)
            n = torch.tensor([length[b] for b in over], dtype=torch.int32, device=device)
            lens, kept = serving.kv_cache_evict(k, v, scores, old, n, torch.tensor(new, dtype=torch.int32, device=device), keep, recent)
            for i, b in enumerate(over):
                free = blocks[b] + free
                blocks[b], length[b] = new[i], int(lens[i])
                for h in range(hkv):
                    r = rows[b][h]
                    best = sorted(range(len(r) - recent), key=lambda t: (-r[t][2], t))[: keep - recent]
                    idx = sorted(best) + list(range(len(r) - recent, len(r)))
                    assert kept[i, h].tolist() == idx
                    rows[b][h] = [r[t] for t in idx]
        q, nk, nv = (torch.randn(B, m, D, generator=g).mul(1.5).to(BF16) for m in (H, hkv, hkv))
        slots = []
        for b in range(B):
            if length[b] % page == 0:
                blocks[b].append(free.pop())
                scores[blocks[b][-1]] = 0.0
            slots.append(blocks[b][-1] * page + length[b] % page)
            length[b] += 1
            for h in range(hkv):
                rows[b][h].append([nk[b, h].double(), nv[b, h].double(), 0.0, step])
        serving.kv_cache_write(k, v, nk.to(device), nv.to(device), torch.tensor(slots, dtype=torch.int32, device=device))
        wide = max(len(x) for x in blocks)
        table = torch.tensor([x + [0] * (wide - len(x)) for x in blocks], dtype=torch.int32, device=device)
        out = serving.paged_attention_split(q.to(device), k, v, table, torch.tensor(length, dtype=torch.int32, device=device), D**-0.5,
                                            scores=scores)
        want = torch.zeros(B, H, D, dtype=torch.float64)
        for b in range(B):
            for h in range(hkv):
                r = rows[b][h]
                keys, vals = torch.stack([x[0] for x in r]), torch.stack([x[1] for x in r])
                w = torch.softmax(q[b, h * 2 : h * 2 + 2].double() @ keys.t() * D**-0.5, -1)
                want[b, h * 2 : h * 2 + 2] = w @ vals
                for t, x in enumerate(w.sum(0).tolist()):
                    r[t][2] += x
        # rounding to bf16 on top of 2^-10 relative to the largest value that is summed (|v| < 8)
        assert ((out.cpu().double() - want).abs() <= want.abs() * 2**-8 * 1.01 + 8 * 2**-10).all()
        logits = (out.cpu().double().view(B, -1) @ proj).float()
        allowed = torch.randint(-(2**31), 2**31, (B, 2), generator=g).to(torch.int32)
        allowed[:, 0] |= 1
        n = torch.full((B,), step, dtype=torch.int32)
        y = serving.process_logits(logits.to(device), history.to(device), n.to(device), n.to(device) // 2, repetition_penalty=1.3,
                                   presence_penalty=0.4, frequency_penalty=0.2, bias_ids=torch.tensor([[3]] * B, device=device),
                                   bias_values=torch.full((B, 1), 0.5, device=device), allowed=allowed.to(device))
        ref, size = logits_oracle(logits, history, n, n // 2, 1.3, 0.4, 0.2, (torch.tensor([[3]] * B), torch.full((B, 1), 0.5)), allowed)
        fine = torch.isfinite(ref)
        assert torch.equal(torch.isfinite(y.cpu()), fine) and ((y.cpu().double() - ref).abs()[fine] <= (size * 6 * 2**-24)[fine]).all()
        tok, _ = serving.sample_top_p(y, 0.0, 1.0, torch.zeros(B, device=device))
        assert all((int(allowed[b, t // 32]) >> (t % 32)) & 1 for b, t in enumerate(tok.tolist()))
        history[:, step] = tok.cpu().to(torch.int32)
    assert evictions >= 6


@pytest.mark.parametrize("device", DEVICES)
def test_arguments_that_are_parts_of_larger_tensors(device):
    """Tables, lengths, histories, biases and masks as a server slices them from its buffers give what copies give."""
    g = _gen(9)
    k, v, table, n, free = make_cache([600, 33, 90], hkv=2, dim=64, page=8, dtype=FP16, device=device, spare=40)
    q = torch.randn(3, 4, 64, generator=g).to(FP16).to(device)
    sinks = torch.randn(4, generator=g).to(BF16).to(device)
    wide = torch.full((3, table.shape[1] + 7), -9, dtype=torch.int32, device=device)
    wide[:, 3 : 3 + table.shape[1]] = table
    part, every_other = wide[:, 3 : 3 + table.shape[1]], torch.stack((n, n * 0 - 1), 1)[:, 0]
    out = serving.paged_attention_split(q, k, v, table, n, 0.125, sinks=sinks.float(), window=500)
    assert torch.equal(out, serving.paged_attention_split(q, k, v, part, every_other, 0.125, sinks=sinks, window=500))
    fresh = free[:24].view(3, 8).to(device)
    fresh_wide = torch.full((3, 20), -1, dtype=torch.int32, device=device)
    fresh_wide[:, 1:9] = fresh
    s = torch.rand(k.shape[0], 2, 8, generator=g).to(device)
    results = []
    for tables, lens, new in ((table, n, fresh), (part, every_other, fresh_wide[:, 1:9])):
        kk, vv, ss = k.clone(), v.clone(), s.clone()
        new_lens, kept = serving.kv_cache_evict(kk, vv, ss, tables, lens, new, 60, 10)
        results.append((new_lens, kept, kk.view(torch.int16), vv.view(torch.int16), ss))
    assert all(torch.equal(a, b) for a, b in zip(*results))
    V, L, N = 777, 101, 13
    logits = torch.randn(3, V + 9, generator=g).to(device)
    tok = torch.randint(0, V, (3, 2 * L + 6), generator=g).to(device)
    ids, vals = torch.randint(0, V, (3, N + 4), generator=g).to(device), torch.randn(3, N + 4, generator=g).to(device)
    mask = torch.randint(-(2**31), 2**31, (3, 40), generator=g).to(torch.int32).to(device)
    rep, lens = torch.rand(3, 2, generator=g).to(device) + 0.5, torch.tensor([[100, 0], [0, 1], [57, 2]], device=device)
    parts = (logits[:, 5 : 5 + V], tok[:, 3 : 3 + L], lens[:, 0], lens[:, 1], ids[:, 1 : 1 + N], vals[:, 2 : 2 + N], mask[:, 7:32], rep[:, 1])

    def call(x, t, n, p, i, w, m, r):
        return serving.process_logits(x, t, n, p, repetition_penalty=r, frequency_penalty=0.3, bias_ids=i, bias_values=w, allowed=m)

    assert torch.equal(call(*parts), call(*(x.clone(memory_format=torch.contiguous_format) for x in parts)))
    stepped = tok[:, : 2 * L : 2]                                          # tokens that do not lie next to each other
    assert torch.equal(call(parts[0], stepped, *parts[2:]), call(parts[0], stepped.contiguous(), *parts[2:]))
    room = torch.zeros(3, V + 3, device=device)
    got = serving.process_logits(parts[0], parts[1], frequency_penalty=0.3, out=room[:, 1 : 1 + V])
    assert torch.equal(got, serving.process_logits(parts[0], parts[1], frequency_penalty=0.3)) and (room[:, 0] == 0).all() and (room[:, 1 + V :] == 0).all()


def _debug_model(dtype=FP32, device="cpu"):
    import dataclasses

    from torchtitan_b200.models.qwen3 import model_registry

    cfg = dataclasses.replace(model_registry("debugmodel").model, n_layers=2)
    cfg.rope = dataclasses.replace(cfg.rope, max_seq_len=512)
    torch.manual_seed(0)
    model = cfg.build().to(dtype=dtype, device=device)
    with torch.no_grad():
        model.init_weights(buffer_device=torch.device(device))
    return model


PROMPTS = [[1, 5, 9, 12, 7], [3, 4, 100, 200, 300, 17, 21, 9, 2, 8, 8, 41], [11]]


def _generate(engine, prompts=PROMPTS, n=2, new=40, temperature=0.0, **kw):
    free = engine.cache.alloc.available
    seqs = engine.generate(prompts, n_samples=n, max_tokens=new, temperature=temperature, top_p=1.0,
                           generator=torch.Generator(engine.device).manual_seed(1), **kw)
    assert engine.cache.alloc.available == free
    return [s.tokens for s in seqs], [s.logprobs for s in seqs]


def _engine(model, **kw):
    from torchtitan_b200.experiments.rl.engine import GenerationEngine

    return GenerationEngine(model, block_size=4, num_blocks=300, **kw)


def test_engine_split_decode_and_ample_budget_change_nothing():
    model = _debug_model()
    tokens, lps = _generate(_engine(model))
    for kw in ({"split_decode": True}, {"cache_budget": 64}):
        t, lp = _generate(_engine(model, **kw))
        assert t == tokens
        # the same fp32 sums in another order, through two layers: well within 2^-12 of a log-probability near 8
        assert (torch.tensor(lp) - torch.tensor(lps)).abs().max() < 2**-12


def test_engine_bounded_cache():
    model = _debug_model()
    kw = {"cache_budget": 16, "cache_recent": 4, "cache_slack": 6}
    e = _engine(model, **kw)
    seen = []
    step = e._forward

    def spy(tokens, positions, meta, last_index=None):
        if not meta["prefill"]:
            seen.append((meta["context_lens"].tolist(), positions[0].tolist()))
        return step(tokens, positions, meta, last_index)

    e._forward = spy
    tokens, _ = _generate(e, temperature=1.0)
    assert e.evictions >= 6 and max(max(n) for n, _ in seen) <= 16 + 6
    assert seen[-1][1] == [len(p) + 38 for p in PROMPTS for _ in range(2)]     # positions count on
    assert (e.cache.scores >= 0).all()
    # a sequence alone gives what it gives in a batch, greedily
    batch, _ = _generate(_engine(model, **kw))
    for i, p in enumerate(PROMPTS):
        alone, _ = _generate(_engine(model, **kw), prompts=[p], n=1)
        assert alone[0] == batch[2 * i] == batch[2 * i + 1]
    for blocks in (14, 7, 4):                                                   # too few to go on, to fork, to hold the prompts
        with pytest.raises(RuntimeError, match="exhausted"):
            _generate_all(_engine_of(model, blocks, **kw))


def _engine_of(model, blocks, **kw):
    from torchtitan_b200.experiments.rl.engine import GenerationEngine

    return GenerationEngine(model, block_size=4, num_blocks=blocks, **kw)


def _generate_all(engine):
    blocks = engine.cache.alloc.available
    try:
        engine.generate(PROMPTS[:2], n_samples=1, max_tokens=30, temperature=0.0, top_p=1.0)
    finally:
        assert engine.cache.alloc.available == blocks                          # nothing is lost when the blocks run out


def test_engine_penalties_bias_and_grammar():
    model = _debug_model()
    plain, _ = _generate(_engine(model), new=20)
    # a strong presence penalty: no token twice
    tokens, lps = _generate(_engine(model), new=20, presence_penalty=1000.0)
    assert all(len(set(t)) == 20 for t in tokens) and any(len(set(t)) < 20 for t in plain)
    from torchtitan_b200.experiments.rl.losses import compute_token_log_probs_packed

    # what is reported are the model's own log-probabilities
    ref = compute_token_log_probs_packed(model, [p for p in PROMPTS for _ in range(2)], tokens, "cpu")
    assert all(torch.allclose(torch.tensor(a), b, atol=2e-5) for a, b in zip(lps, ref))
    assert all(set(t) == {77} for t in _generate(_engine(model), new=5, logit_bias={77: 1e4, 3: -1e4})[0])
    rep, _ = _generate(_engine(model), new=20, repetition_penalty=1e6)
    assert all(t[0] not in t[1:] for t in rep)

    def grammar(i, said):
        return None if i == 0 else [2 * i, 2 * i + 1] if len(said) % 2 else range(40, 50)

    tokens, _ = _generate(_engine(model), new=12, grammar=grammar, temperature=1.0)
    for i, t in enumerate(tokens[1:], start=1):
        assert all(x in (2 * i, 2 * i + 1) if j % 2 else 40 <= x < 50 for j, x in enumerate(t))
    for bad in (lambda i, s: [], lambda i, s: [5000], lambda i, s: [-1]):
        with pytest.raises(ValueError, match="grammar"):
            _generate(_engine(model), new=3, grammar=bad)
    for bias in ({-1: 1.0}, {5000: 1.0}):
        with pytest.raises(ValueError, match="logit_bias"):
            _generate(_engine(model), new=3, logit_bias=bias)


def test_engine_and_generator_refuse():
    from torchtitan_b200.experiments.rl.generator import Generator

    model = _debug_model()
    for kw in ({"cache_recent": 3}, {"cache_slack": 3}, {"cache_budget": 0}, {"cache_budget": 4, "cache_recent": 5}, {"cache_budget": 4, "cache_slack": 0}):
        with pytest.raises(ValueError, match="cache_"):
            _engine(model, **kw)
    with pytest.raises(ValueError, match="batch_invariant_mode"):
        Generator(Generator.Config(cache_budget=64), model_spec=None, batch_invariant_mode=True)


@pytest.mark.gpu
@pytest.mark.parametrize("graphs", [False, True])
def test_engine_bounded_cache_on_the_gpu(graphs):
    """bf16 on the kernels, eager and captured: bounded, nothing lost, batch-independent, the same with and without graphs."""
    model = _debug_model(BF16, "cuda")
    kw = {"cache_budget": 16, "cache_recent": 4, "cache_slack": 6}
    e = _engine(model, cudagraph=graphs, **kw)
    tokens, lps = _generate(e)
    assert e.evictions >= 6 and bool((e.cache.scores >= 0).all())
    eager, eager_lps = _generate(_engine(model, **kw))
    assert tokens == eager and lps == eager_lps
    again, again_lps = _generate(e, presence_penalty=0.5, grammar=lambda i, s: range(100, 400))
    assert all(100 <= x < 400 for t in again for x in t)


def test_engine_captures_with_every_write_before_the_side_stream_waits(monkeypatch):
    """Capture under a budget on fakes of the streams: between the moment the side stream waits for the current one and the moment
    the current one waits for it, nothing is written on the current stream (the warm-up passes would not be ordered behind it),
    and the warm-up passes see no tokens, so that they add no weights."""
    from contextlib import contextmanager

    from torch.utils._python_dispatch import TorchDispatchMode

    at, writes, warm = {"stream": "current", "open": False}, [], []

    class Stream:
        def __init__(self, name="side"):
            self.name = name

        def wait_stream(self, other):
            at["open"] = self.name == "side"

    class Graph:
        def replay(self):
            at["replayed"] = True

    @contextmanager
    def on(stream):
        before, at["stream"] = at["stream"], stream.name
        yield
        at["stream"] = before

    @contextmanager
    def capture(graph):
        yield

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            if at["open"] and at["stream"] == "current" and func._schema.is_mutable:
                writes.append(str(func))
            return func(*args, **(kwargs or {}))

    monkeypatch.setattr(torch.cuda, "Stream", Stream)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: Stream("current"))
    monkeypatch.setattr(torch.cuda, "stream", on)
    monkeypatch.setattr(torch.cuda, "CUDAGraph", Graph)
    monkeypatch.setattr(torch.cuda, "graph", capture)
    e = _engine(_debug_model(), cache_budget=16, cache_recent=4, cache_slack=6)
    e.cudagraph = True
    forward = e._forward

    def spy(tokens, positions, meta, last_index=None):
        if at["open"]:
            warm.append((at["stream"], meta["context_lens"].tolist()))
        return forward(tokens, positions, meta, last_index)

    e._forward = spy
    with Watch():
        e.generate(PROMPTS, n_samples=1, max_tokens=3, temperature=0.0, top_p=1.0)
    assert at["replayed"] and not writes
    assert warm and all(stream == "side" and lens == [0] * len(PROMPTS) for stream, lens in warm)


@pytest.mark.gpu
def test_engine_captured_steps_add_the_weights_of_eager_ones():
    """Every captured step is the first of its batch size and width here: the accumulated weights have the bits of eager steps."""
    model = _debug_model(BF16, "cuda")
    kw = {"cache_budget": 16, "cache_recent": 4, "cache_slack": 6}
    for new in (2, 3, 8, 30):
        captured, eager = _engine(model, cudagraph=True, **kw), _engine(model, **kw)
        assert _generate(captured, new=new) == _generate(eager, new=new)
        assert captured.evictions == eager.evictions and torch.equal(captured.cache.scores, eager.cache.scores)


def test_whole_numbers_are_narrowed_to_values_outside():
    from torchtitan_b200.ops import cuda_ops

    far = torch.tensor([0, 7, -1, -9, 2**31 - 1, 2**31, 2**32, 2**32 + 7, -(2**32), -(2**63), 2**63 - 1])
    assert cuda_ops._i32(far).tolist() == [0, 7, -1, -1] + [2**31 - 1] * 4 + [-1, -1, 2**31 - 1]
    near = far[:4].to(torch.int32)
    assert cuda_ops._i32(near) is near


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("beyond", [-7, 1 << 30, -(1 << 31)])
def test_evict_does_not_look_at_table_entries_behind_a_sequence(beyond, device):
    """Behind a sequence's pages a table may hold anything, as for the attention."""
    k, v, table, n, free = make_cache([40, 9, 0], hkv=2, dim=64, page=16, dtype=BF16, device=device, spare=12)
    fresh = free[:6].view(3, 2).to(device)
    s = torch.rand(k.shape[0], 2, 16, generator=_gen(4)).to(device)
    results = []
    for fill in (0, beyond):
        wide = torch.full((3, 6), fill, dtype=torch.int32, device=device)
        for b, pages in enumerate((3, 1, 0)):
            wide[b, :pages] = table[b, :pages]
        kk, vv, ss = k.clone(), v.clone(), s.clone()
        lens, kept = serving.kv_cache_evict(kk, vv, ss, wide, n, fresh, 20, 4)
        results.append((lens, kept, kk.view(torch.int16), vv.view(torch.int16), ss))
    assert results[0][0].tolist() == [20, 9, 0] and all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("device", DEVICES)
def test_evict_refuses_a_keep_of_2_to_the_30(device):
    """Kept tokens are counted in 32 bits, in steps of thousands: 2^32 + 5 must not become 5, nor a loop pass 2^31 (an empty batch,
    as `kept` has `keep` columns)."""
    k, v, table, n, free = make_cache([40], hkv=2, dim=64, page=16, dtype=BF16, device=device, spare=8)
    s, fresh = torch.zeros(k.shape[0], 2, 16, device=device), free[:4].view(1, 4).to(device)
    for keep in (1 << 30, (1 << 31) - 1, 1 << 31, (1 << 32) + 5):
        with pytest.raises(ValueError, match="keep"):
            serving.kv_cache_evict(k, v, s, table[:0], n[:0], fresh[:0], keep)
    lens, kept = serving.kv_cache_evict(k, v, s, table[:0], n[:0], fresh[:0], (1 << 30) - 1)
    assert lens.shape == (0,) and kept.shape == (0, 2, (1 << 30) - 1)


@pytest.mark.parametrize("device", DEVICES)
def test_sampler_draws_no_masked_token_where_rounding_keeps_everything(device):
    """top_p next to 1: the mass of all tokens falls short of it by rounding, so that the nucleus takes the masked ones in."""
    x = torch.stack([torch.randn(3001, generator=_gen(seed)) for seed in range(200)]).to(device)
    x[:, 2000:] = -math.inf
    for u in (0.5, 1.0 - 2**-24, 1.0):
        tok, lp = serving.sample_top_p(x, 1.0, 1.0 - 2**-24, torch.full((200,), u, device=device))
        assert int(tok.max()) < 2000 and torch.isfinite(lp).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_engine_refuses_a_step_that_leaves_no_token(temperature, device):
    """A grammar whose only tokens a bias of -inf takes away, at the first token or a later one of one sequence."""
    model = _debug_model(BF16 if device == "cuda" else FP32, device)
    for at in (0, 2):
        with pytest.raises(ValueError, match="sequence 3"):
            _generate_then_count(_engine(model), temperature, grammar=lambda i, said, at=at: [5, 6] if i == 3 and len(said) == at else None,
                                 logit_bias={5: -math.inf, 6: -math.inf})
    tokens, _ = _generate(_engine(model), new=5, grammar=lambda i, said: [5, 6, 7], logit_bias={5: -math.inf, 6: -math.inf})
    assert all(set(t) == {7} for t in tokens)


def _generate_then_count(engine, temperature, **kw):
    free = engine.cache.alloc.available
    try:
        engine.generate(PROMPTS, n_samples=2, max_tokens=4, temperature=temperature, top_p=1.0, **kw)
    finally:
        assert engine.cache.alloc.available == free


LONG_PROMPT = [(7 * i) % 500 + 1 for i in range(90)]


@pytest.mark.parametrize("device", DEVICES)
def test_engine_bounded_cache_needs_no_copy_of_a_long_prompt_per_sample(device):
    """Prompts that outgrow the budget: the samples need their prompt's blocks once and the budget's each, and give what they
    give with blocks to spare. 90 + 5 tokens in blocks of 4: 23 + 2 blocks (and one for padding); a sample keeps 16 + 6 tokens."""
    model = _debug_model(BF16 if device == "cuda" else FP32, device)
    kw = {"cache_budget": 16, "cache_recent": 4, "cache_slack": 6}

    def run(num_blocks):
        e = _engine_of(model, num_blocks, **kw)
        return _generate(e, prompts=[LONG_PROMPT, LONG_PROMPT[:5]], n=6, new=12, temperature=1.0), e.evictions

    assert run(25 + 12 * 6 + 1) == run(600)


@pytest.mark.parametrize("device", DEVICES)
def test_engine_evicts_in_groups_that_the_free_blocks_allow(device):
    """Three samples grow to 6 blocks each and are cut back to 4 in the same step: with 4 blocks free one after the other, as the
    blocks that one gives back serve the next."""
    model = _debug_model(BF16 if device == "cuda" else FP32, device)
    kw = {"cache_budget": 16, "cache_recent": 4, "cache_slack": 6}

    def run(num_blocks):
        e = _engine_of(model, num_blocks, **kw)
        return _generate(e, prompts=[LONG_PROMPT[:22]], n=3, new=20, temperature=1.0), e.evictions

    # 22 tokens at the 1st, 7th, 13th and 19th of 19 steps: each cuts back to 16, and six more make 22 again
    assert run(3 * 6 + 4) == run(600) and run(600)[1] == 3 * 4
    with pytest.raises(RuntimeError, match="exhausted"):
        run(3 * 6 + 3)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("where", ["prefill", "fork", "decode", "evict"])
def test_engine_returns_every_block_when_a_step_fails(where, device, monkeypatch):
    """An exception anywhere in a run (as where memory runs out) leaves all blocks free."""
    e = _engine(_debug_model(BF16 if device == "cuda" else FP32, device), cache_budget=16, cache_recent=4, cache_slack=6)
    forward, evict, calls = e._forward, serving.kv_cache_evict, []

    class Failed(Exception):
        pass

    def fail_forward(tokens, positions, meta, last_index=None):
        if meta["prefill"] == (where == "prefill"):
            raise Failed
        return forward(tokens, positions, meta, last_index)

    def fail_evict(*args):
        calls.append(1)
        if len(calls) == 2:                        # the second layer's
            raise Failed
        return evict(*args)

    def fail_copy(src, dst):
        raise Failed

    if where in ("prefill", "decode"):
        e._forward = fail_forward
    elif where == "fork":
        e.cache.copy_block = fail_copy
    else:
        monkeypatch.setattr(serving, "kv_cache_evict", fail_evict)
    free = e.cache.alloc.available
    with pytest.raises(Failed):
        e.generate([LONG_PROMPT, LONG_PROMPT[:6]], n_samples=2, max_tokens=4, temperature=0.0, top_p=1.0)
    assert e.cache.alloc.available == free == e.cache.num_blocks and not any(e.cache.alloc.refs)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kw", [{}, {"cache_budget": 16, "cache_recent": 4, "cache_slack": 6}])
def test_engine_refuses_positions_past_the_rotary_table(kw, device):
    """A bounded cache never fills up, so the table of 512 positions is what ends a sequence: its rows are read by position."""
    model = _debug_model(BF16 if device == "cuda" else FP32, device)
    prompt = [(5 * i) % 300 + 1 for i in range(500)]
    e = _engine(model, **kw)
    tokens, _ = _generate(e, prompts=[prompt, prompt[:9]], n=1, new=13)       # positions 500 ... 511
    assert [len(t) for t in tokens] == [13, 13]
    for prompts, new in (([prompt[:9], prompt], 14), ([prompt + prompt[:13]], 1)):
        with pytest.raises(ValueError, match="position 512"):
            e.generate(prompts, n_samples=1, max_tokens=new, temperature=0.0, top_p=1.0)
        assert e.cache.alloc.available == e.cache.num_blocks


@pytest.mark.parametrize("device", DEVICES)
def test_engine_with_a_short_rotary_table(device):
    """A table shorter than the padding of a prefill on the GPU (up to 127 tokens)."""
    import dataclasses

    from torchtitan_b200.models.qwen3 import model_registry

    cfg = dataclasses.replace(model_registry("debugmodel").model, n_layers=2)
    seen = []
    for rows in (40, 512):
        cfg.rope = dataclasses.replace(cfg.rope, max_seq_len=rows)
        torch.manual_seed(0)
        model = cfg.build().to(dtype=BF16 if device == "cuda" else FP32, device=device)
        with torch.no_grad():
            model.init_weights(buffer_device=torch.device(device))
        e = _engine(model)
        forward, past = e._forward, []

        def spy(tokens, positions, meta, last_index=None, forward=forward, past=past):
            past.append(int(positions.max()))
            return forward(tokens, positions, meta, last_index)

        e._forward = spy
        seen.append(_generate(e, n=1, new=4))
        assert rows > 40 or max(past) < rows
    assert seen[0] == seen[1]
