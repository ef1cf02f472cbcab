// Eviction from a paged KV cache by accumulated attention weight.
//
// For every (sequence, kv head) with n cached tokens: n <= keep keeps all of them; otherwise the last `recent` tokens stay
// and, of the n - recent before them, the keep - recent with the largest score, ties going to the lowest index. What stays
// is copied, in its order, to the first slots of new pages: the old pages are only read, so they may be shared.
//
// Selection: the score's bits, mapped so that unsigned order is score order, lie in some range [lo, hi] of keys. A histogram
// of 2048 equal parts of that range says which part the last kept key is in; that part is the next range, until the range is
// one key or all of it is kept (at most three rounds of 11 bits each; usually two, since the first splits the occupied part
// of the scale rather than the 32 bits). Of the keys in the last range the first in index order are taken. A cluster of CTAs
// shares one (sequence, kv head): each holds its part of the keys in shared memory and reads the others' histograms there.
//
// What bounds it: the move reads and writes every kept row once and is memory-bound (32 sequences up to 8192, 8 kv heads, keep
// 2048: 545 MB, 98 us, 0.85 of the measured copy rate; 86 us where only the latest tokens stay, without a selection); the selection reads 4 bytes a
// token and is a chain of some ten meetings: 23 of the 48 us of 2 x 131072 tokens with 4 kv heads, whose 64 blocks do not fill
// the GPU. Clusters of 16 would, but did not fit next to each other: 92 us where clusters of 8 took 57.
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <type_traits>

namespace cg = cooperative_groups;

namespace {

struct Args {
  char *k, *v;
  float* scores;             // [pages, Hkv, page]
  const int *tables, *lens, *fresh;
  int *new_lens, *kept;      // [B], [B, Hkv, keep]
  long long k_page, k_tok, k_head, v_page, v_tok, v_head;   // bytes
  long long table_row, fresh_row;
  int B, Hkv, page, width, fresh_width, pages, row_bytes, keep, recent, page_shift;
  int held;                  // keys of a CTA that its shared memory holds, a multiple of four
  bool fours;                // every four tokens of a page lie on a 16-byte boundary of the scores
};

// Larger key = kept earlier. NaN counts as the largest value, both zeros are one value.
__device__ __forceinline__ uint32_t key_of(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t b = __float_as_uint(v + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

constexpr uint32_t kZero = 0x80000000u;       // key_of(0)

__device__ __forceinline__ int length_of(const Args& a, int b) {
  const int n = a.lens[b];
  return n < 0 || n > a.width * a.page ? 0 : n;
}

__device__ __forceinline__ uint32_t key_at(const Args& a, int b, int h, int t) {
  const int p = a.tables[b * a.table_row + t / a.page];
  if (p < 0 || p >= a.pages) return 0u;
  return key_of(a.scores[(static_cast<long long>(p) * a.Hkv + h) * a.page + t % a.page]);
}

constexpr int kBins = 2048;
constexpr int kMostParts = 8;
constexpr int kAhead = 4;
constexpr int kMostHeld = 48 * 1024;      // keys

// Exclusive sum over the block's threads; total: the sum of all.
template <int WARPS>
__device__ __forceinline__ int block_scan(int v, int* s_warp, int& total) {
  static_assert(WARPS <= 32, "one warp sum per lane");
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += up;
  }
  if (lane == 31) s_warp[warp] = inc;
  __syncthreads();
  const int mine = lane < WARPS ? s_warp[lane] : 0;
  int w = mine;
#pragma unroll
  for (int o = 1; o < WARPS; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += up;
  }
  total = __shfl_sync(0xffffffffu, w, WARPS - 1);
  const int before = __shfl_sync(0xffffffffu, w - mine, warp);
  __syncthreads();
  return before + inc - v;
}

// Writes the kept indices of kv head h of sequence b in order. `parts` CTAs of a cluster cut the tokens into equal parts (one CTA
// alone needs none), `part` is this one.
template <int kThreads>
__device__ __forceinline__ void select_rows(const Args& a, int b, int h, int parts, int part) {
  constexpr int kWarps = kThreads / 32, kEach = kBins / kThreads;      // bins of a thread
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int n = length_of(a, b), left = min(n, a.keep);
  int* kept = a.kept + (static_cast<long long>(b) * a.Hkv + h) * a.keep;
  if (h == 0 && part == 0 && tid == 0) a.new_lens[b] = left;
  for (int j = left + part * kThreads + tid; j < a.keep; j += parts * kThreads) kept[j] = -1;
  if (n <= a.keep) {                       // the same for the whole cluster
    for (int j = part * kThreads + tid; j < n; j += parts * kThreads) kept[j] = j;
    return;
  }
  const int old = n - a.recent;
  for (int j = part * kThreads + tid; j < a.recent; j += parts * kThreads) kept[a.keep - a.recent + j] = old + j;
  int want = a.keep - a.recent;            // of the first `old` tokens
  if (want == 0) return;

  extern __shared__ __align__(16) uint32_t keys[];
  __shared__ __align__(16) int hist[2][kBins];
  __shared__ uint32_t s_lo, s_hi, s_pos;
  __shared__ int s_warp[kWarps], s_want, s_bin, s_in_bin;
  __shared__ int s_above, s_equal, s_positive;
  const int per = ((old + parts - 1) / parts + 3) / 4 * 4, t0 = min(old, part * per), count = min(old, t0 + per) - t0;
  const bool all_held = count <= a.held;
  auto key = [&](int i) { return all_held || i < a.held ? keys[i] : key_at(a, b, h, t0 + i); };

  if (tid == 0) { s_lo = s_pos = 0xffffffffu; s_hi = 0; s_positive = 0; }
  for (int i = tid; i < 2 * kBins; i += kThreads) hist[0][i] = 0;
  __syncthreads();
  // the lowest and highest key, and apart from them those above zero: often many tokens were never looked at, and a range that
  // reaches down to their zero would have few of its parts where the others are
  uint32_t lo = 0xffffffffu, hi = 0, pos = 0xffffffffu;
  int positive = 0;
  auto see = [&](uint32_t k) {
    lo = min(lo, k);
    hi = max(hi, k);
    if (k > kZero) { pos = min(pos, k); ++positive; }
  };
  // several loads on their way at a time, pages first; four tokens of a page with each where pages allow it
  if (a.fours) {
    for (int i0 = 4 * tid; i0 < count; i0 += 4 * kAhead * kThreads) {
      int page[kAhead], slot[kAhead];
      float4 s[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int i = i0 + 4 * u * kThreads, t = t0 + i, at = a.page_shift >= 0 ? t >> a.page_shift : t / a.page;
        slot[u] = t - at * a.page;
        page[u] = i < count ? a.tables[b * a.table_row + at] : -1;
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (page[u] >= 0 && page[u] < a.pages)
          s[u] = *reinterpret_cast<const float4*>(a.scores + (static_cast<long long>(page[u]) * a.Hkv + h) * a.page + slot[u]);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int i = i0 + 4 * u * kThreads;
        if (i >= count) continue;
        uint4 k = make_uint4(0, 0, 0, 0);
        if (page[u] >= 0 && page[u] < a.pages) k = make_uint4(key_of(s[u].x), key_of(s[u].y), key_of(s[u].z), key_of(s[u].w));
        if (i < a.held) *reinterpret_cast<uint4*>(keys + i) = k;         // held is a multiple of four
        see(k.x);
        if (i + 1 < count) see(k.y);
        if (i + 2 < count) see(k.z);
        if (i + 3 < count) see(k.w);
      }
    }
  } else {
    for (int i0 = tid; i0 < count; i0 += kAhead * kThreads) {
      int page[kAhead], slot[kAhead];
      uint32_t k[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int i = i0 + u * kThreads, t = t0 + i, at = a.page_shift >= 0 ? t >> a.page_shift : t / a.page;
        slot[u] = t - at * a.page;
        page[u] = i < count ? a.tables[b * a.table_row + at] : -1;
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const bool ok = page[u] >= 0 && page[u] < a.pages;
        const float s = ok ? a.scores[(static_cast<long long>(page[u]) * a.Hkv + h) * a.page + slot[u]] : 0.f;
        k[u] = ok ? key_of(s) : 0u;
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int i = i0 + u * kThreads;
        if (i >= count) continue;
        if (i < a.held) keys[i] = k[u];
        see(k[u]);
      }
    }
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  pos = __reduce_min_sync(0xffffffffu, pos);
  positive = __reduce_add_sync(0xffffffffu, positive);
  if (lane == 0) {
    atomicMin(&s_lo, lo);
    atomicMax(&s_hi, hi);
    atomicMin(&s_pos, pos);
    atomicAdd(&s_positive, positive);
  }
  auto meet = [&]() { if (parts > 1) cluster.sync(); else __syncthreads(); };
  meet();
  lo = pos = 0xffffffffu, hi = 0, positive = 0;
#pragma unroll
  for (int p = 0; p < kMostParts; ++p)
    if (p < parts) {
      lo = min(lo, *cluster.map_shared_rank(&s_lo, p));
      hi = max(hi, *cluster.map_shared_rank(&s_hi, p));
      pos = min(pos, *cluster.map_shared_rank(&s_pos, p));
      positive += *cluster.map_shared_rank(&s_positive, p);
    }
  if (positive >= want) {
    lo = pos;
  } else {
    want -= positive;
    hi = kZero;
  }
  // invariant: `want` of the keys in [lo, hi] are kept, and all above hi
  for (int round = 0; lo < hi; ++round) {
    int* mine = hist[round & 1];
    const int shift = max(0, 21 - __clz(hi - lo));
    // the lowest key (tokens that were never looked at, often) is counted apart: its bin would make the threads wait in line
    int lowest = 0;
    auto count_key = [&](uint32_t k) {
      if (k > lo && k <= hi) atomicAdd(&mine[(k - lo) >> shift], 1);
      lowest += k == lo;
    };
    if (all_held) {
      for (int i = 4 * tid; i < count; i += 4 * kThreads) {
        const uint4 k = *reinterpret_cast<const uint4*>(keys + i);
        count_key(k.x);
        if (i + 1 < count) count_key(k.y);
        if (i + 2 < count) count_key(k.z);
        if (i + 3 < count) count_key(k.w);
      }
    } else {
      for (int i = tid; i < count; i += kThreads) count_key(key(i));
    }
    lowest = __reduce_add_sync(0xffffffffu, lowest);
    if (lane == 0 && lowest) atomicAdd(&mine[0], lowest);
    meet();
    // bins from the top, kEach to a thread; all parts' loads at once
    using Bins = std::conditional_t<kEach == 4, int4, int2>;
    union { Bins v; int n[kEach]; } of[kMostParts];
    int c[kEach];
#pragma unroll
    for (int p = 0; p < kMostParts; ++p) {
      of[p].v = Bins{};
      if (p < parts)
        of[p].v = *reinterpret_cast<const Bins*>((parts > 1 ? cluster.map_shared_rank(mine, p) : mine) + kBins - kEach * (tid + 1));
    }
    int sum = 0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      c[e] = 0;
#pragma unroll
      for (int p = 0; p < kMostParts; ++p) c[e] += of[p].n[kEach - 1 - e];
      sum += c[e];
    }
    int total;
    int above = block_scan<kWarps>(sum, s_warp, total);
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      if (above < want && above + c[e] >= want) {
        s_bin = kBins - 1 - kEach * tid - e;
        s_want = want - above;
        s_in_bin = c[e];
      }
      above += c[e];
    }
    // the next round's histogram: the others were done with it when they came to this round's meeting
    for (int i = tid; i < kBins; i += kThreads) hist[(round + 1) & 1][i] = 0;
    __syncthreads();
    lo += static_cast<uint32_t>(s_bin) << shift;
    hi = lo + min(hi - lo, (1u << shift) - 1);
    want = s_want;
    const bool all = s_in_bin == want;
    __syncthreads();
    if (all) break;
  }
  // kept: above hi, and the first `want` in [lo, hi]. A warp owns a run of consecutive tokens.
  const int run = (count + kWarps - 1) / kWarps, i0 = min(count, warp * run), i1 = min(count, i0 + run);
  int above = 0, equal = 0;
  for (int i = i0 + lane; i < i1; i += 32) {
    const uint32_t k = key(i);
    above += k > hi;
    equal += k >= lo && k <= hi;
  }
  above = __reduce_add_sync(0xffffffffu, above);
  equal = __reduce_add_sync(0xffffffffu, equal);
  int all_above, all_equal;
  int above_at = block_scan<kWarps>(lane == 0 ? above : 0, s_warp, all_above);
  int equal_at = block_scan<kWarps>(lane == 0 ? equal : 0, s_warp, all_equal);
  if (tid == 0) { s_above = all_above; s_equal = all_equal; }
  meet();
  for (int p = 0; p < part; ++p) {
    above_at += *cluster.map_shared_rank(&s_above, p);
    equal_at += *cluster.map_shared_rank(&s_equal, p);
  }
  above_at = __shfl_sync(0xffffffffu, above_at, 0);
  equal_at = __shfl_sync(0xffffffffu, equal_at, 0);
  const uint32_t below = (1u << lane) - 1;
  for (int i = i0; i < i1; i += 32) {
    const bool in = i + lane < i1;
    const uint32_t k = in ? key(i + lane) : 0;
    const uint32_t am = __ballot_sync(0xffffffffu, in && k > hi), em = __ballot_sync(0xffffffffu, in && k >= lo && k <= hi);
    const int rank = equal_at + __popc(em & below);              // among those in [lo, hi]
    const bool take = ((am >> lane) & 1) || (((em >> lane) & 1) && rank < want);
    if (take) kept[above_at + __popc(am & below) + min(rank, want)] = t0 + i + lane;
    above_at += __popc(am);
    equal_at += __popc(em);
  }
  if (parts > 1) cluster.sync();           // no CTA leaves while another may read its shared memory
}

// Cluster = (kv head, sequence).
template <int kThreads>
__global__ void __launch_bounds__(kThreads) select_kernel(const Args a) {
  asm volatile("griddepcontrol.launch_dependents;");
  const int parts = cg::this_cluster().num_blocks();
  select_rows<kThreads>(a, blockIdx.y, blockIdx.x / parts, parts, cg::this_cluster().block_rank());
}

// Moves piece c (16 bytes of key and of value) of the kept rows j[0..N), all loads before the stores; rows at `left` and behind
// are none. The first piece takes the scores along.
template <int N>
__device__ __forceinline__ void move_pieces(const Args& a, int b, int h, const int* kept, const int (&j)[N], int left, int c) {
  uint4 kv[N], vv[N];
  float s[N];
  long long dst_page[N];
#pragma unroll
  for (int u = 0; u < N; ++u) {
    dst_page[u] = -1;
    if (j[u] >= left) continue;
    const int t = kept[j[u]];
    const int sp = a.tables[b * a.table_row + t / a.page], dp = a.fresh[b * a.fresh_row + j[u] / a.page], so = t % a.page;
    if (sp < 0 || sp >= a.pages || dp < 0 || dp >= a.pages) continue;
    dst_page[u] = dp;
    kv[u] = __ldcs(reinterpret_cast<const uint4*>(a.k + sp * a.k_page + so * a.k_tok + h * a.k_head + c * 16));
    vv[u] = __ldcs(reinterpret_cast<const uint4*>(a.v + sp * a.v_page + so * a.v_tok + h * a.v_head + c * 16));
    if (c == 0) s[u] = a.scores[(static_cast<long long>(sp) * a.Hkv + h) * a.page + so];
  }
#pragma unroll
  for (int u = 0; u < N; ++u) {
    if (dst_page[u] < 0) continue;
    const int to = j[u] % a.page;
    __stcs(reinterpret_cast<uint4*>(a.k + dst_page[u] * a.k_page + to * a.k_tok + h * a.k_head + c * 16), kv[u]);
    __stcs(reinterpret_cast<uint4*>(a.v + dst_page[u] * a.v_page + to * a.v_tok + h * a.v_head + c * 16), vv[u]);
    if (c == 0) a.scores[(dst_page[u] * a.Hkv + h) * a.page + to] = s[u];
  }
}

// kRowsEach kept rows to a group of row_bytes / 16 threads. The rows pass once: they are marked first to leave the caches.
// 32 sequences up to 8192, 8 kv heads, keep 2048 (545 MB): 122 us with 4 rows and plain accesses, 117 with 4 marked, 118 with 2
// plain, 111 with 2 marked, 109 with blocks of 128 instead of 256 threads (the whole call, in a graph).
constexpr int kRowsEach = 2, kMoveThreads = 128;

__global__ void __launch_bounds__(kMoveThreads, 12) move_kernel(const Args a) {
  const int per = a.row_bytes / 16;
  const int b = blockIdx.y;
  asm volatile("griddepcontrol.wait;" ::: "memory");          // started early: the selection must be complete
  const int left = min(length_of(a, b), a.keep);
  const long long i = static_cast<long long>(blockIdx.x) * kMoveThreads + threadIdx.x;
  const int c = static_cast<int>(i % per);
  const long long r = i / per;
  const int h = static_cast<int>(r % a.Hkv);
  const long long j0 = r / a.Hkv * kRowsEach;
  if (j0 >= left) return;
  int j[kRowsEach];
#pragma unroll
  for (int u = 0; u < kRowsEach; ++u) j[u] = static_cast<int>(j0) + u;
  move_pieces(a, b, h, a.kept + (static_cast<long long>(b) * a.Hkv + h) * a.keep, j, left, c);
}

// Small caches in one launch, as launches are most of their time: cluster = (kv head, sequence), its first CTA selects, all move.
// 1056 tokens, 8 kv heads, keep 1024: 18 us a call against 20.4 with two launches (9.5 against 8.4 in a captured graph); with 512
// threads 10.1, with clusters of 4 14.6.
constexpr int kSmallRoom = 8192, kSmallBytes = 128 << 10;     // tokens of a table; kept keys and values to a CTA

template <int kThreads>
__global__ void __launch_bounds__(kThreads) small_kernel(const Args a) {
  cg::cluster_group cluster = cg::this_cluster();
  const int movers = cluster.num_blocks(), rank = cluster.block_rank(), b = blockIdx.y, h = blockIdx.x / movers;
  if (rank == 0) select_rows<kThreads>(a, b, h, 1, 0);
  if (movers > 1) cluster.sync(); else __syncthreads();
  const int left = min(length_of(a, b), a.keep), per = a.row_bytes / 16, rows = movers * kThreads / per;     // rows of a pass
  const int at = rank * kThreads + threadIdx.x, c = at % per;
  if (at / per >= rows) return;
  for (int j0 = at / per; j0 < left; j0 += 2 * rows) {
    const int j[2] = {j0, j0 + rows};
    move_pieces(a, b, h, a.kept + (static_cast<long long>(b) * a.Hkv + h) * a.keep, j, left, c);
  }
}

}  // namespace

extern "C" {

// v: the arguments as 64-bit words in the order of the names below; cache strides in bytes, table strides in elements.
int tt_kv_evict(const long long* v, cudaStream_t st) {
  enum { K, V, SCORES, TABLES, LENS, FRESH, NEW_LENS, KEPT, K_PAGE, K_TOK, K_HEAD, V_PAGE, V_TOK, V_HEAD, TABLE_ROW, FRESH_ROW, BATCH,
         KV_HEADS, PAGE, WIDTH, FRESH_WIDTH, PAGES, ROW_BYTES, KEEP, RECENT };
  auto at = [&](int i) { return reinterpret_cast<void*>(v[i]); };
  auto num = [&](int i) { return static_cast<int>(v[i]); };
  const int B = num(BATCH), Hkv = num(KV_HEADS), page = num(PAGE), width = num(WIDTH), fresh_width = num(FRESH_WIDTH), pages = num(PAGES),
            row_bytes = num(ROW_BYTES), keep = num(KEEP), recent = num(RECENT);
  if (B <= 0 || Hkv <= 0) return 0;
  if (B > 65535 || row_bytes % 16 || keep < 1 || recent < 0 || recent > keep) return -2;
  const long long room = static_cast<long long>(width) * page, most = room < keep ? room : keep;
  if (most > static_cast<long long>(fresh_width) * page) return -2;
  // CTAs of a (sequence, kv head): as many as give every SM one, but none with fewer than 2048 tokens
  int parts = 1;
  while (parts < kMostParts && static_cast<long long>(B) * Hkv * parts < 148 && room / (2 * parts) >= 2048) parts *= 2;
  const long long per = ((room + parts - 1) / parts + 3) / 4 * 4;
  const int held = static_cast<int>(per < kMostHeld ? per : kMostHeld);
  Args a{static_cast<char*>(at(K)), static_cast<char*>(at(V)), static_cast<float*>(at(SCORES)), static_cast<const int*>(at(TABLES)),
         static_cast<const int*>(at(LENS)), static_cast<const int*>(at(FRESH)), static_cast<int*>(at(NEW_LENS)),
         static_cast<int*>(at(KEPT)), v[K_PAGE], v[K_TOK], v[K_HEAD], v[V_PAGE], v[V_TOK], v[V_HEAD], v[TABLE_ROW], v[FRESH_ROW],
         B, Hkv, page, width, fresh_width, pages, row_bytes, keep, recent, page & (page - 1) ? -1 : __builtin_ctz(page), held,
         page % 4 == 0 && v[SCORES] % 16 == 0};
  int movers = 1;
  while (movers < 8 && static_cast<long long>(B) * Hkv * movers < 148) movers *= 2;
  const bool small = room <= kSmallRoom && most * row_bytes * 2 <= static_cast<long long>(kSmallBytes) * movers && row_bytes <= 16 * 512;
  // many rows: blocks of 512 threads, several to an SM; few: 1024 threads each
  const bool wide = static_cast<long long>(B) * Hkv * parts < 148;
  const auto select = wide ? select_kernel<1024> : select_kernel<512>;
  static std::atomic<uint64_t> ready{0};          // devices on which the kernels may take their shared memory
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return -4;
  if (!(ready.load(std::memory_order_relaxed) >> dev & 1)) {
    for (const auto f : {select_kernel<1024>, select_kernel<512>, small_kernel<1024>, small_kernel<512>})
      if (cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostHeld * 4) != cudaSuccess) return -4;
    ready.fetch_or(uint64_t{1} << dev);
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  if (small) {
    attr[0].val.clusterDim.x = movers;
    cfg.gridDim = dim3(Hkv * movers, B);
    cfg.blockDim = dim3(movers > 1 ? 1024 : 512);          // blocks alone on their SMs, or several to one
    cfg.dynamicSmemBytes = static_cast<size_t>((room + 3) / 4 * 4) * 4;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = movers > 1;
    a.held = static_cast<int>((room + 3) / 4 * 4);
    return cudaLaunchKernelEx(&cfg, movers > 1 ? small_kernel<1024> : small_kernel<512>, a) == cudaSuccess ? 0 : -4;
  }
  cfg.gridDim = dim3(Hkv * parts, B);
  cfg.blockDim = dim3(wide ? 1024 : 512);
  cfg.dynamicSmemBytes = static_cast<size_t>(held) * 4;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = parts > 1;                       // a block by itself is a cluster of one
  if (cudaLaunchKernelEx(&cfg, select, a) != cudaSuccess) return -4;
  cfg.numAttrs = 1;
  const long long threads = (most + kRowsEach - 1) / kRowsEach * Hkv * (row_bytes / 16);
  if (threads > 0) {
    // the move's CTAs come up while the selection runs and wait there for its end
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(static_cast<unsigned>((threads + kMoveThreads - 1) / kMoveThreads), B);
    cfg.blockDim = dim3(kMoveThreads);
    cfg.dynamicSmemBytes = 0;
    if (cudaLaunchKernelEx(&cfg, move_kernel, a) != cudaSuccess) return -4;
  }
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}

}  // extern "C"
