"""What only the kernels of the decode-time ops can get wrong: captured graphs, streams, batch composition, large offsets,
pages and lengths outside the cache (answered by the kernels' own bounds checks)."""

import pytest
import torch

from test_decode_ops import BF16, FP16, attention_oracle, check_attention, make_cache, rows_of

from torchtitan_b200.ops import cuda_ops, serving

pytestmark = pytest.mark.gpu


def _attend(q, k, v, table, n, **kw):
    return serving.paged_attention_split(q, k, v, table, n, q.shape[-1] ** -0.5, **kw)


@pytest.mark.parametrize("D,H,hkv", [(64, 8, 1), (128, 32, 4), (128, 16, 16), (256, 48, 2)])
def test_a_sequence_gives_the_same_bits_in_every_batch(D, H, hkv):
    lens = [3000, 1, 700, 40, 1025, 9000]
    k, v, table, n, _ = make_cache(lens, hkv=hkv, dim=D, page=16, dtype=BF16, device="cuda")
    q = torch.randn(len(lens), H, D, device="cuda").to(BF16)
    out, lse = _attend(q, k, v, table, n, return_lse=True)
    for b in range(len(lens)):
        one, l1 = _attend(q[b : b + 1], k, v, table[b : b + 1], n[b : b + 1], return_lse=True)
        assert torch.equal(one[0], out[b]) and torch.equal(l1[0], lse[b])
    narrow = -(-40 // 16)                                          # a table of its own width
    assert torch.equal(_attend(q[3:4], k, v, table[3:4, :narrow].contiguous(), n[3:4])[0], out[3])


@pytest.mark.parametrize("lens", [[4096 * 16 + 13], [20000, 70000, 5], [128 * 256, 128 * 256 + 1, 128 * 256 - 1]])
def test_long_sequences(lens):
    k, v, table, n, _ = make_cache(lens, hkv=2, dim=64, page=64, dtype=BF16, device="cuda")
    q = (torch.randn(len(lens), 16, 64, device="cuda") * 2).to(BF16)
    scores = torch.zeros(k.shape[0], 2, 64, device="cuda")
    out, lse = _attend(q, k, v, table, n, scores=scores, return_lse=True)
    check_attention(out, attention_oracle(q, k, v, table, n, 0.125), max(lens), 64, BF16, lse, scores, torch.zeros_like(scores), table)


def test_offsets_past_32_bits():
    """A cache of 2^32 + elements: the sequence lies on its last pages."""
    page, hkv, D = 64, 8, 128
    pages = (1 << 32) // (page * hkv * D) + 40
    k = torch.zeros(pages, page, hkv, D, dtype=BF16, device="cuda")
    v = torch.zeros_like(k)
    last = torch.arange(pages - 32, pages, device="cuda", dtype=torch.int32)
    k[-40:].normal_()
    v[-40:].normal_()
    n = torch.tensor([32 * page - 5], dtype=torch.int32, device="cuda")
    q = torch.randn(1, 16, D, device="cuda").to(BF16)
    scores = torch.zeros(pages, hkv, page, device="cuda")
    table = last.view(1, -1)
    out = _attend(q, k, v, table, n, scores=scores)
    small = torch.arange(32, dtype=torch.int32, device="cuda").view(1, -1)
    s2 = torch.zeros(32, hkv, page, device="cuda")
    assert torch.equal(out, _attend(q, k[-32:].clone(), v[-32:].clone(), small, n, scores=s2))
    assert torch.equal(scores[-32:], s2)
    fresh = torch.arange(pages - 40, pages - 32, dtype=torch.int32, device="cuda").view(1, -1)
    lens, kept = serving.kv_cache_evict(k, v, scores, table, n, fresh, 8 * page, 7)
    for h in range(hkv):
        idx = kept[0, h].long()
        want = rows_of(k, last, 32 * page)[idx, h]
        assert torch.equal(rows_of(k, fresh[0], 8 * page)[:, h], want)
    del k, v


def test_captured_and_replayed():
    """One graph for attention with weights, eviction and logits; new lengths, tables and logits on every replay. Two graphs
    replayed in turn, an eager call between them."""
    lens = [300, 20, 0, 130]
    k, v, table, n, free = make_cache(lens, hkv=2, dim=128, page=16, dtype=BF16, device="cuda", spare=40, width=32)
    fresh = free[:16].view(4, 4).to("cuda")
    q = torch.randn(4, 8, 128, device="cuda").to(BF16)
    scores = torch.zeros(k.shape[0], 2, 16, device="cuda")
    x, tok = torch.randn(4, 5003, device="cuda"), torch.randint(0, 5003, (4, 50), device="cuda")
    tl = torch.tensor([50, 3, 0, 20], dtype=torch.int32, device="cuda")

    def step():
        out = _attend(q, k, v, table, n, scores=scores)
        lens, kept = serving.kv_cache_evict(k, v, scores, table, n, fresh, 64, 8)
        return out, lens, kept, serving.process_logits(x, tok, tl, repetition_penalty=1.2, frequency_penalty=0.1)

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step()
        graphs.append((g, res))
    for i, new in enumerate(([300, 20, 0, 130], [17, 0, 4, 1], [512, 500, 1, 16])):
        new = [min(a, c) for a, c in zip(new, [304, 32, 0, 144])]      # within what was written
        new = [min(a, b) for a, b in zip(new, lens)]
        n.copy_(torch.tensor(new, dtype=torch.int32))
        x.normal_()
        results = []
        for g, res in (graphs[i % 2], graphs[(i + 1) % 2], (None, None)):
            scores.zero_()
            if g is None:
                res = step()
            else:
                g.replay()
            results.append([t.clone() for t in (*res, scores)])
        for r in results[:2]:
            assert all(torch.equal(a, b) for a, b in zip(r, results[2]))


def test_other_streams():
    """Work on a side stream, with workspaces whose memory the main stream reuses at once."""
    k, v, table, n, _ = make_cache([5000, 100], hkv=2, dim=128, page=16, dtype=FP16, device="cuda")
    q = torch.randn(2, 8, 128, device="cuda").to(FP16)
    x, tok = torch.randn(8, 30011, device="cuda"), torch.randint(0, 30011, (8, 2000), device="cuda")
    want = _attend(q, k, v, table, n), serving.process_logits(x, tok, presence_penalty=0.5)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        with torch.cuda.stream(side):
            a, b = _attend(q, k, v, table.long(), n.long()), serving.process_logits(x, tok, presence_penalty=0.5)
        torch.empty(1 << 22, device="cuda").fill_(float("nan"))
        c = _attend(q, k, v, table, n)
        side.synchronize()
        assert torch.equal(a, want[0]) and torch.equal(b, want[1]) and torch.equal(c, want[0])


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (256, FP16), (48, torch.float32)])
def test_lengths_and_pages_outside_are_not_followed(dim, dtype):
    """The kernels (and the definition, where there is none) check what the host cannot see: NaN for that sequence, the others
    untouched by it."""
    k, v, table, n, free = make_cache([40, 64, 33, 50], hkv=2, dim=dim, page=16, dtype=dtype, device="cuda", spare=20)
    q = torch.randn(4, 4, dim, device="cuda").to(dtype)
    good = _attend(q, k, v, table, n)
    bad_t, bad_n = table.clone(), n.clone()
    bad_t[0, 1], bad_n[2], bad_n[3] = k.shape[0], 65, -1
    scores = torch.zeros(k.shape[0], 2, 16, device="cuda")
    out, lse = _attend(q, k, v, bad_t, bad_n, scores=scores, return_lse=True)
    assert out[[0, 2, 3]].isnan().all() and lse[[0, 2, 3]].isnan().all() and torch.equal(out[1], good[1])
    bad_t[0, 1] = -5
    assert _attend(q, k, v, bad_t, n)[0].isnan().all()
    # beyond the sequence, a table may hold anything
    wild = torch.full((4, 9), 1 << 30, dtype=torch.int32, device="cuda")
    wild[:, :4] = table
    for b, ln in enumerate([40, 64, 33, 50]):
        wild[b, -(-ln // 16) :] = -7
    got = _attend(q, k, v, wild, n)
    if dtype != torch.float32:
        assert torch.equal(got, good)
    else:   # library products sum in another order: 64 tokens and 48 dims of values below 8, each sum off by n * 2^-23 of its terms
        assert ((got - good).abs() <= 8 * (2 * 64 + 2 * 48 * 8) * 2**-23).all()
    k0, v0, scores = k.clone(), v.clone(), torch.rand(k.shape[0], 2, 16, device="cuda")
    fresh = free[:8].view(4, 2).to("cuda")
    fresh[1, 0] = 1 << 30
    lens, kept = serving.kv_cache_evict(k, v, scores, bad_t, bad_n, fresh, 32, 4)
    assert lens.tolist() == [32, 32, 0, 0] and (kept[2:] == -1).all()
    as_int = {2: torch.int16, 4: torch.int32}[k.element_size()]
    untouched = torch.ones(k.shape[0], dtype=torch.bool, device="cuda")
    untouched[fresh[0].long()], untouched[fresh[1, 1].long()] = False, False
    assert torch.equal(k[untouched].view(as_int), k0[untouched].view(as_int))
    assert torch.equal(v[untouched].view(as_int), v0[untouched].view(as_int))
    x = torch.randn(2, 100, device="cuda")
    tok = torch.tensor([[5, 100, -1, 1 << 30], [7, 7, 7, 7]], device="cuda")
    y = serving.process_logits(x, tok, torch.tensor([99, -3], device="cuda"), presence_penalty=2.0,
                               bias_ids=torch.tensor([[100, 3], [-9, 1 << 30]], device="cuda"), bias_values=torch.ones(2, 2, device="cuda"))
    want = x.clone()
    want[0, 5] -= 2.0
    want[0, 3] += 1.0
    assert torch.equal(y, want)


def test_layouts_the_kernels_refuse():
    k, v, table, n, free = make_cache([40], hkv=2, dim=64, page=16, dtype=BF16, device="cuda")
    q = torch.randn(1, 4, 64, device="cuda").to(BF16)
    off = torch.zeros(k.numel() + 8, dtype=BF16, device="cuda")[3:][: k.numel()].view(k.shape)
    for kk in (off, k.transpose(2, 3).contiguous().transpose(2, 3)):
        with pytest.raises(ValueError, match="16-byte"):
            _attend(q, kk, v, table, n)
    odd = torch.zeros(6, 16, 2, 12, dtype=BF16, device="cuda")
    with pytest.raises(ValueError, match="16 bytes"):
        serving.kv_cache_evict(odd, odd.clone(), torch.zeros(6, 2, 16, device="cuda"), table, n, free.view(1, -1).to("cuda"), 32)


def test_wide_batches_and_vocabularies():
    """More rows than an axis of a small grid, a vocabulary larger than a cluster holds at once."""
    B = 5000
    k, v, table, n, _ = make_cache([1 + i % 3 for i in range(50)], hkv=1, dim=64, page=4, dtype=BF16, device="cuda")
    q = torch.randn(50, 2, 64, device="cuda").to(BF16)
    want = _attend(q, k, v, table, n)
    got = _attend(q.repeat(B // 50, 1, 1), k, v, table.repeat(B // 50, 1), n.repeat(B // 50))
    assert torch.equal(got, want.repeat(B // 50, 1, 1))
    V = 1_000_003
    x = torch.randn(2, V, device="cuda")
    tok = torch.randint(0, V, (2, 3000), device="cuda")
    y = serving.process_logits(x, tok, frequency_penalty=0.5)
    count = torch.zeros(2, V, device="cuda").scatter_add_(1, tok, torch.ones(2, 3000, device="cuda"))
    assert torch.equal(y, x - 0.5 * count)


def test_queries_on_odd_addresses():
    k, v, table, n, _ = make_cache([70, 9], hkv=2, dim=64, page=16, dtype=BF16, device="cuda")
    wide = torch.randn(2, 4 * 65 + 1, device="cuda").to(BF16)
    q = wide[:, 1:].view(2, 4, 65)[..., :64]
    assert torch.equal(_attend(q, k, v, table, n), _attend(q.clone(), k, v, table, n))


@pytest.mark.parametrize("D", [64, 128, 256])
def test_a_wider_table_changes_no_bit(D):
    """The same sequences with tables of their own width and much wider ones: the join takes another form, the sums do not."""
    lens = [513, 1500, 16000, 7000, 0]
    k, v, table, n, _ = make_cache(lens, hkv=2, dim=D, page=16, dtype=BF16, device="cuda")
    q = torch.randn(len(lens), 6, D, device="cuda").to(BF16)
    sinks = torch.randn(6, device="cuda")
    wide = torch.zeros(len(lens), 9000, dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table
    for s in (None, sinks):
        a, b = _attend(q, k, v, table, n, sinks=s, return_lse=True), _attend(q, k, v, wide, n, sinks=s, return_lse=True)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def _evict_by_sort(scores, table, n, keep, recent):
    """Kept tokens from a stable descending sort; scores without NaN, all sequences longer than keep."""
    B, page, hkv = table.shape[0], scores.shape[2], scores.shape[1]
    x = scores[table.long()].permute(0, 2, 1, 3).reshape(B, hkv, -1)
    age = n.long().unsqueeze(1) - torch.arange(x.shape[-1], device="cuda")
    x = x.masked_fill((age <= recent).unsqueeze(1), float("inf")).masked_fill((age <= 0).unsqueeze(1), float("-inf"))
    return torch.sort(x, dim=-1, descending=True, stable=True).indices[..., :keep].sort(-1).values.to(torch.int32)


@pytest.mark.parametrize("B,hkv,n,keep,recent", [(40, 4, 60000, 1000, 100), (1, 2, 500000, 70000, 5000), (2, 3, 40001, 40000, 0), (200, 1, 300, 20, 3)])
def test_evict_long_and_many(B, hkv, n, keep, recent):
    """More keys to a block than its shared memory holds, clusters of several sizes, many rows."""
    page, D = 64, 8
    width, need = -(-n // page), -(-keep // page)
    perm = torch.randperm(B * (width + need), device="cuda").to(torch.int32)
    table, fresh = perm[: B * width].view(B, width), perm[B * width :].view(B, need)
    k = torch.randn(perm.numel(), page, hkv, D, device="cuda").to(BF16)
    v = torch.randn_like(k)
    scores = torch.empty(perm.numel(), hkv, page, device="cuda").log_normal_(-3, 2)
    scores *= torch.rand_like(scores) > 0.5
    lens = torch.full((B,), n, dtype=torch.int32, device="cuda")
    want = _evict_by_sort(scores, table, lens, keep, recent)
    new_lens, kept = serving.kv_cache_evict(k, v, scores, table, lens, fresh, keep, recent)
    assert torch.equal(kept, want) and (new_lens == keep).all()
    idx = want[-1, -1].long()
    for c in (k, v):
        assert torch.equal(rows_of(c, fresh[-1], keep)[:, -1], rows_of(c, table[-1], n)[idx, -1])


def test_very_long_history():
    V, L = 5000, 300_001
    x = torch.randn(2, V, device="cuda")
    tok = torch.randint(0, V, (2, L), device="cuda")
    tok[:, ::3] = 17
    y = serving.process_logits(x, tok, prompt_lens=torch.tensor([0, 100_000], device="cuda"), frequency_penalty=0.25)
    for b, p in enumerate((0, 100_000)):
        assert torch.equal(y[b], x[b] - 0.25 * torch.bincount(tok[b, p:], minlength=V))


@pytest.mark.parametrize("B", [31, 33, 300, 1025])
def test_batches_of_every_length(B):
    """Empty, short and many-chunk sequences mixed, batches on both sides of a warp's and a launch's number of sequences: each
    sequence as by itself."""
    g = torch.Generator().manual_seed(B)
    choice = torch.tensor([0, 0, 1, 17, 511, 512, 513, 1500, 2100])
    lens = choice[torch.randint(0, len(choice), (B,), generator=g)].tolist()
    lens[0], lens[-1] = 0, 0
    k, v, table, n, _ = make_cache(lens, hkv=1, dim=64, page=32, dtype=BF16, device="cuda", seed=B)
    q = torch.randn(B, 3, 64, device="cuda").to(BF16)
    scores = torch.zeros(k.shape[0], 1, 32, device="cuda")
    out, lse = _attend(q, k, v, table, n, scores=scores, return_lse=True)
    empty = torch.tensor([x == 0 for x in lens], device="cuda")
    assert (out[empty] == 0).all() and (lse[empty] == -float("inf")).all()
    alone = torch.zeros_like(scores)
    for b in sorted({0, 1, B // 2, B - 2, B - 1, *torch.randint(0, B, (20,), generator=g).tolist()}):
        one, l1 = _attend(q[b : b + 1], k, v, table[b : b + 1], n[b : b + 1], scores=alone, return_lse=True)
        assert torch.equal(one[0], out[b]) and torch.equal(l1[0], lse[b])
        pages = table[b, : -(-lens[b] // 32)].long()
        assert torch.equal(alone[pages], scores[pages])


@pytest.mark.parametrize("B,hkv,D,page,dtype", [(1, 1, 8, 1, BF16), (3, 2, 512, 16, FP16), (1, 8, 128, 16, torch.float32), (150, 2, 64, 7, BF16),
                                                (2, 3, 24, 32, torch.float32), (40, 2, 128, 16, BF16)])
@pytest.mark.parametrize("n,keep,recent", [(40, 39, 5), (700, 200, 0), (1999, 1500, 1500), (8000, 600, 599)])
def test_evict_small_and_large_forms(B, hkv, D, page, dtype, n, keep, recent):
    """Caches around the sizes at which the selection and the move share a launch; rows of 16 bytes to 1 KB; lengths that differ."""
    g = torch.Generator(device="cuda").manual_seed(n)
    lens = (n - torch.randint(0, n - keep, (B,), generator=g, device="cuda")).to(torch.int32)        # all longer than keep
    lens[0] = n
    width, need = -(-n // page), -(-keep // page)
    perm = torch.randperm(B * (width + need), generator=g, device="cuda").to(torch.int32)
    table, fresh = perm[: B * width].view(B, width), perm[B * width :].view(B, need)
    k = torch.randn(perm.numel(), page, hkv, D, generator=g, device="cuda").to(dtype)
    v = torch.randn(perm.numel(), page, hkv, D, generator=g, device="cuda").to(dtype)
    scores = torch.rand(perm.numel(), hkv, page, generator=g, device="cuda").mul_(8).floor_()          # many ties
    want = _evict_by_sort(scores, table, lens, keep, recent)
    k0, v0, s0 = k.clone(), v.clone(), scores.clone()
    new_lens, kept = serving.kv_cache_evict(k, v, scores, table, lens, fresh, keep, recent)
    assert torch.equal(kept, want) and (new_lens == keep).all()
    j, seq, h = torch.arange(keep, device="cuda"), torch.arange(B, device="cuda").view(B, 1, 1), torch.arange(hkv, device="cuda").view(1, hkv, 1)
    sp, so, dp, do = table[seq, want // page].long(), want.long() % page, fresh[seq, (j // page).view(1, 1, -1)].long(), (j % page).view(1, 1, -1)
    k0[dp, do, h], v0[dp, do, h], s0[dp, h, do] = k0[sp, so, h], v0[sp, so, h], s0[sp, h, so]
    assert torch.equal(k, k0) and torch.equal(v, v0) and torch.equal(scores, s0)


def _past_32_bits(t, at, value):
    t = t.long().clone()
    t[at] = value
    return t


@pytest.mark.parametrize("value", [2**32, 2**32 + 1, 2**31, -(2**63), -(2**32), 2**63 - 1])
def test_whole_numbers_past_32_bits_are_outside(value):
    """int64 tables, lengths and ids are checked by their value, not by their lower half (which names real pages and tokens)."""
    k, v, table, n, free = make_cache([40, 64, 33], hkv=2, dim=64, page=16, dtype=BF16, device="cuda", spare=20)
    q = torch.randn(3, 4, 64, device="cuda").to(BF16)
    good = _attend(q, k, v, table, n)
    for bad_t, bad_n in ((_past_32_bits(table, (0, 1), value), n.long()), (table.long(), _past_32_bits(n, 0, value))):
        scores = torch.zeros(k.shape[0], 2, 16, device="cuda")
        out, lse = _attend(q, k, v, bad_t, bad_n, scores=scores, return_lse=True)
        assert out[0].isnan().all() and lse[0].isnan().all() and torch.equal(out[1:], good[1:])
        others = torch.ones(k.shape[0], dtype=torch.bool, device="cuda")
        others[table[0, :3].long()] = False
        assert torch.isfinite(scores[others]).all()
    fresh = free[:6].view(3, 2).to("cuda")
    scores = torch.rand(k.shape[0], 2, 16, device="cuda")
    k0 = k.clone()
    lens, kept = serving.kv_cache_evict(k, v, scores, table, _past_32_bits(n, 0, value), fresh, 32, 4)
    assert lens.tolist() == [0, 32, 32] and (kept[0] == -1).all()
    assert torch.equal(k[fresh[0].long()].view(torch.int16), k0[fresh[0].long()].view(torch.int16))
    k1 = k.clone()
    serving.kv_cache_evict(k, v, scores, table, n, _past_32_bits(fresh, (0, 0), value), 32, 4)
    moved = torch.zeros(k.shape[0], dtype=torch.bool, device="cuda")
    moved[fresh.view(-1)[1:].long()] = True
    assert torch.equal(k[~moved].view(torch.int16), k1[~moved].view(torch.int16))
    x = torch.randn(2, 100, device="cuda")
    tok = torch.tensor([[5, value, 6], [7, 7, value]], device="cuda")
    far = torch.tensor([3, value], device="cuda")
    y = serving.process_logits(x, tok, far, presence_penalty=2.0, bias_ids=torch.tensor([[value, 3], [4, value]], device="cuda"),
                               bias_values=torch.ones(2, 2, device="cuda"))
    want = x.clone()
    want[0, [5, 6]] -= 2.0
    want[1, 7] -= 2.0 if value > 0 else 0.0                                # a length above the list's is the list's, one below 0 is 0
    want[0, 3] += 1.0
    want[1, 4] += 1.0
    assert torch.equal(y, want)
    y = serving.process_logits(x, tok, prompt_lens=far * 0 + value, frequency_penalty=0.5)
    want = x.clone()
    if value < 0:
        want[0, [5, 6]] -= 0.5
        want[1, 7] -= 1.0
    assert torch.equal(y, want)


@pytest.mark.parametrize("past", [-1, 0, 1, 70_000])
def test_where_chunks_begin_to_grow(past):
    """Sequences around the length from which chunks are longer than the least, with a short one beside them. A term passes at
    most chunk + 4 + 256 additions (its chunk's, the groups', the join's), so errors are bounded by that many, not by the tokens:
    a chunk left out of a sum would show."""
    least, most = cuda_ops._split_rule()
    n = least * most + past
    k, v, table, lens, _ = make_cache([n, 700], hkv=2, dim=64, page=64, dtype=FP16, device="cuda", seed=past)
    for b, m in enumerate((n, 700)):
        v[table[b, : -(-m // 64)].long()] += 3.0                  # what is missing does not average out
    q = torch.randn(2, 4, 64, device="cuda").to(FP16)
    scores = torch.zeros(k.shape[0], 2, 64, device="cuda")
    out, lse = _attend(q, k, v, table, lens, scores=scores, return_lse=True)
    oracle = attention_oracle(q, k, v, table, lens, 0.125)
    check_attention(out, oracle, 2 * least + 4 + most, 64, FP16, lse, scores, torch.zeros_like(scores), table)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_join_of_more_chunks_than_one_pass_holds(D):
    """137 chunks: with 256 dims more than 32 warps fetch at once."""
    n = 70_000
    k, v, table, lens, _ = make_cache([n, 33], hkv=1, dim=D, page=128, dtype=FP16, device="cuda", seed=D)
    for b, m in enumerate((n, 33)):
        v[table[b, : -(-m // 128)].long()] += 3.0
    q = torch.randn(2, 2, D, device="cuda").to(FP16)
    scores = torch.zeros(k.shape[0], 1, 128, device="cuda")
    out, lse = _attend(q, k, v, table, lens, scores=scores, return_lse=True)
    check_attention(out, attention_oracle(q, k, v, table, lens, D**-0.5), 512 + 4 + 256, D, FP16, lse, scores, torch.zeros_like(scores), table)


@pytest.mark.parametrize("sinks", [False, True])
@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, BF16), (256, FP16)])
def test_join_by_warps(D, dtype, sinks):
    """Enough heads for a warp to join each, up to 32 chunks: the bits of every sequence by itself, which a block joins -- of its
    weights too, which show a last bit of the denominator that the output's rounding hides."""
    lens = [16_384, 0, 1, 600, 5000, 1024, 1025, 12_345] + [1100 + 7 * i for i in range(12)]
    H, hkv = 64, 4
    assert len(lens) * H >= 1184
    k, v, table, n, _ = make_cache(lens, hkv=hkv, dim=D, page=32, dtype=dtype, device="cuda", seed=D)
    for seed in range(10):
        torch.manual_seed(seed)
        q = torch.randn(len(lens), H, D, device="cuda").to(dtype)
        sink = torch.randn(H, device="cuda") if sinks else None
        scores, alone = torch.zeros(k.shape[0], hkv, 32, device="cuda"), torch.zeros(k.shape[0], hkv, 32, device="cuda")
        out, lse = _attend(q, k, v, table, n, sinks=sink, scores=scores, return_lse=True)
        for b in range(len(lens)):
            one, l1 = _attend(q[b : b + 1], k, v, table[b : b + 1], n[b : b + 1], sinks=sink, scores=alone, return_lse=True)
            assert torch.equal(one[0], out[b]) and torch.equal(l1[0], lse[b])
        assert torch.equal(scores, alone)
    short = [3, 5, 6]
    oracle = attention_oracle(q[short], k, v, table[short], n[short], D**-0.5, sinks=sink)
    check_attention(out[short], oracle, 512 + 4 + 256, D, dtype, lse[short])


@pytest.mark.parametrize("G,D", [(72, 64), (130, 128), (65, 64)])
def test_many_query_heads_to_a_kv_head(G, D):
    """Weights are summed 64 query heads at a time."""
    lens = [1500, 3, 0, 64]
    k, v, table, n, _ = make_cache(lens, hkv=2, dim=D, page=16, dtype=BF16, device="cuda", seed=G)
    q = torch.randn(len(lens), 2 * G, D, device="cuda").to(BF16)
    scores = torch.rand(k.shape[0], 2, 16, device="cuda")
    before = scores.clone()
    out, lse = _attend(q, k, v, table, n, scores=scores, return_lse=True)
    check_attention(out, attention_oracle(q, k, v, table, n, D**-0.5), max(lens), D, BF16, lse, scores, before, table)
