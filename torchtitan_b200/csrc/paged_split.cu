// Decode attention over a paged KV cache, split over the cache's length and joined.
//
// One query token per sequence. With x_j = scale * log2(e) * q.k_j over the live tokens j of a sequence, a chunk c of them
// gives m_c = max x_j, l_c = sum 2^(x_j - m_c) and o_c = sum 2^(x_j - m_c) v_j; the join takes M = max_c m_c (and the sink
// logit, where there is one) and
//     out = sum_c 2^(m_c - M) o_c / (sum_c 2^(m_c - M) l_c + 2^(sink - M)).
// Where chunks begin and end follows from the sequence's own length alone (chunk_len below), never from the batch or the
// number of SMs: a sequence's result has the same bits in every batch.
//
// The accumulated weights: per kv head, score_j += sum over its query heads of 2^(x_j - M_h) / l_h. The x_j are kept in a
// workspace between the two passes (4 bytes per token and head next to the 4*D of K and V).
//
// Rows without tokens give zeros. A page number outside the cache, or a length outside the table, gives NaN for that
// sequence and is never followed.
//
// What bounds it: K and V are read once, 4 * D bytes per token and kv head, against 4 * D operations per query head: memory,
// as long as the instructions per byte stay few. So the products go to the matrix units (eight query heads share every
// fragment of K and V; with plain multiplications the same case took 3.8 ms instead of 0.38), tokens are copied to shared
// memory by asynchronous 16-byte copies that run two steps ahead in every warp (24 KB a warp, 192 KB an SM on their way), and
// nothing but the meeting at a chunk's end makes warps wait for one another. A bulk copy per row took 20 cycles a row and
// stopped at 3.5 TB/s; copies with the address of every row looked up, at 3.6.
// Chunks of 512 tokens: with 256 the partial results and meetings cost 128 sequences up to 8192 (16/8 heads) 375 us against
// 353, with 1024 a ragged batch is left waiting for its last chunks (64 sequences up to 4096, 32/4 heads: 99 us against 81).
// Measured (several B200s, calls back to back): 128 sequences up to 8192 tokens, 16/8 heads of 128: 363 to 385 us, 5.6 to 6.0 TB/s,
// 0.86 to 0.91 of the measured copy rate; one of 131072, 32/8 heads: 99 to 103 us, 5.2 to 5.4 TB/s; 64 up to 4096, 32/4 heads, with
// scores: 72 us, 3.9 TB/s. With the products left out 32 of 8192 and one of 131072 take the same time.
// Not bound by memory: 256 dims with 16 query heads to a kv head (6 of 5003, fp16: 45 us in a graph, 19 us of bytes). One CTA of
// eight warps fills an SM, the busiest has 1024 tokens where the mean is 811, and a warp spends 32 % of its time on fixed
// latencies, 16 % on tokens, 11 % on meetings: the dependent products, exchange and transposes of every 16 tokens.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <type_traits>

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kMinChunk = 512;    // tokens
constexpr int kMaxChunks = 256;   // per sequence: bounds the workspace and the join's work
constexpr int kTile = 8;          // query heads of one kv head in a tile of columns
constexpr int kMaxBatch = 1024;   // sequences of one launch (their chunk counts are kept in shared memory)

struct Args {
  const void *q, *k, *v;
  const int *tables, *lens;
  void* out;
  float* lse;          // [B, H] or null
  const float* sinks;  // [H] or null
  float* scores;       // [pages, Hkv, page] or null
  float* ws_o;         // [B, chunks, H, D]
  float2* ws_ml;       // [B, chunks, H]
  float2* ws_tot;      // [B, H]: M and the denominator (with scores)
  float* ws_x;         // [B, Hkv, span, H / Hkv] (with scores)
  long long q_b, q_h, k_page, k_tok, k_head, v_page, v_tok, v_head, table_row;
  int B, H, Hkv, page, width, pages, window, span, chunks, page_shift;
  bool whole;                                   // every eight tokens of a step lie on one page
  float scale;
};

__host__ __device__ inline int chunk_len(int n) {
  const int c = ((n + kMaxChunks - 1) / kMaxChunks + 63) / 64 * 64;
  return c > kMinChunk ? c : kMinChunk;
}

// The tokens of sequence b that are read: [lo, n), of which those before `first` are masked. bad: the length is not one.
struct Range {
  int lo, first, n;
  bool bad;
};
__device__ __forceinline__ Range range_of(const Args& a, int b) {
  Range r;
  r.n = a.lens[b];
  r.bad = r.n < 0 || r.n > a.width * a.page;
  if (r.bad) r.n = 0;
  r.first = a.window > 0 ? max(0, r.n - a.window) : 0;
  r.lo = r.first & ~15;
  return r;
}

// ---- pieces of the matrix path
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool ok) {   // zeros where !ok (src is not read then)
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void wait_group() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ float ex2(float x) {      // 2^x, off by at most 2^-22 of it; results below 2^-126 are 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void ldm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <typename T> __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// (lower half, upper half) rounded to T
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t v);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v)); }
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }

// The end of a query head: sink, division, output of dims d and d + 1. top, sum, x: maximum, sum and weighted values over all
// of its tokens. Three kernels end in it, and a sequence must get the same bits from each: products and sums are rounded on
// their own here and in the joins' sums, not left to the compiler to contract in one kernel and not in another.
template <typename T, int D>
__device__ __forceinline__ void finish(const Args& a, int b, int h, int d, float top, float sum, float2 x) {
  const long long bh = static_cast<long long>(b) * a.H + h;
  if (a.sinks) {
    const float sink = __fmul_rn(a.sinks[h], kLog2e), all = fmaxf(top, sink), base = all == -INFINITY ? 0.f : all;
    const float f = exp2f(__fsub_rn(top, base));
    x.x = __fmul_rn(x.x, f);
    x.y = __fmul_rn(x.y, f);
    sum = __fadd_rn(__fmul_rn(sum, f), sink == all && all != -INFINITY ? 1.f : exp2f(__fsub_rn(sink, base)));
    top = all;
  }
  *reinterpret_cast<uint32_t*>(static_cast<T*>(a.out) + bh * D + d) = sum == 0.f ? 0u : pack2<T>(x.x / sum, x.y / sum);
  if (d == 0) {
    if (a.lse) a.lse[bh] = __fmul_rn(__fadd_rn(top, log2f(sum)), kLn2);
    if (a.ws_tot) a.ws_tot[bh] = make_float2(top, sum);
  }
}

constexpr int kGroups = 4;       // of warps: each takes every fourth step of a chunk
constexpr int kRows = 16;        // tokens of one step of a warp

// How D dims are shared: a warp takes at most 128 of them, so that its results stay in registers; with 256, two warps of a
// group take the same tokens, add up their halves of the logits through shared memory, and go on with half the dims each.
template <int D> struct Shape {
  static constexpr int kDims = D < 128 ? D : 128, kParts = D / kDims, kWarps = kGroups * kParts;
};

// A warp's stage: kRows rows of K, then of V. Rows lie 16 bytes more than their length apart, so that the eight rows of a
// matrix load touch different banks.
template <int D> struct Ring {
  static constexpr int kRowBytes = 2 * Shape<D>::kDims, kRowPitch = kRowBytes + 16, kStageBytes = 2 * kRows * kRowPitch;
  static constexpr int kStages = 3;
  static constexpr int kBytes = Shape<D>::kWarps * kStages * kStageBytes;
};
template <int D, int NT> struct Exchange {     // [group][2 turns][part][NT * 4 logits][lane]
  static constexpr int kBytes = Shape<D>::kParts > 1 ? kGroups * 2 * 2 * NT * 4 * 32 * 4 : 0;
};
template <int D, int NT> constexpr int smem_bytes() { return Ring<D>::kBytes + kGroups * kTile * NT * 8 + Exchange<D, NT>::kBytes; }

// One piece of work: chunk c of sequence b for a tile of NT * 8 query heads of kv head hk.
struct Item {
  int b, c, hk, tile, t0, t1, chunks;
  Range r;
};

// items are numbered ((sequence, chunk), kv head, tile), the last fastest: neighbours read the same tokens' heads, which lie
// next to each other in the cache. first[b]: chunks of the sequences before b. The warp looks for the last sequence that
// begins at or before bc, 32 candidates at a time (at most two rounds).
__device__ __forceinline__ void item_at(Item& it, const Args& a, const int* first, int bc, int hkt, int tiles) {
  const int lane = threadIdx.x % 32;
  it.hk = tiles == 1 ? hkt : hkt / tiles;
  it.tile = hkt - it.hk * tiles;
  int b = 0;
  if (a.B > 32) b = 32 * (__popc(__ballot_sync(0xffffffffu, lane * 32 < a.B && first[lane * 32] <= bc)) - 1);
  b += __popc(__ballot_sync(0xffffffffu, b + lane < a.B && first[b + lane] <= bc)) - 1;
  it.b = b;
  it.c = bc - first[b];
  it.chunks = first[b + 1] - first[b];
  it.r = range_of(a, b);
  const int len = chunk_len(it.r.n - it.r.lo);
  it.t0 = it.r.lo + it.c * len;
  it.t1 = min(it.r.n, it.t0 + len);
}

// Tokens as rows of the products' left operand, query heads as columns: S^T = K q^T and O^T += V^T P^T, eight query heads
// being one tile of columns, so that groups of up to 8 heads waste nothing. P is passed as its rounding to T plus the
// rounding of the remainder, which keeps 16 bits of it (P in T alone would add an error as large as the output's own
// rounding). A group of warps (one, or two with 256 dims)
// owns every fourth 16 tokens of a chunk; every warp has a ring of stages, and its loads run ahead across chunks.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(32 * Shape<D>::kWarps) split_kernel(const Args a) {
  using R = Ring<D>;
  constexpr int kExchange = Exchange<D, NT>::kBytes;
  constexpr float kLift = std::is_same_v<T, __half> ? 7.f : 0.f;
  constexpr int DW = Shape<D>::kDims, DP = Shape<D>::kParts, kWarps = Shape<D>::kWarps;
  extern __shared__ __align__(128) unsigned char smem[];
  float2* s_ml = reinterpret_cast<float2*>(smem + R::kBytes);                                // [group][NT * 8]
  float* s_x = reinterpret_cast<float*>(s_ml + kGroups * kTile * NT);                        // [group][2][part][NT * 4][lane]
  int* first = reinterpret_cast<int*>(reinterpret_cast<char*>(s_x) + kExchange);                // [B + 1]
  __shared__ int s_sum[kWarps], s_free[kWarps];
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, group = warp / DP, part = warp % DP;
  const int G = a.H / a.Hkv, tiles = (G + kTile * NT - 1) / (kTile * NT), hkts = a.Hkv * tiles;
  asm volatile("griddepcontrol.launch_dependents;");       // the join's CTAs may come up, and wait for this grid's end

  // how many chunks the sequences before each one have
  {
    constexpr int kThreads = 32 * kWarps;
    const int per = (a.B + kThreads - 1) / kThreads, b0 = min(a.B, tid * per), b1 = min(a.B, b0 + per);
    int sum = 0;
#pragma unroll 4
    for (int b = b0; b < b1; ++b) {
      const Range r = range_of(a, b);
      const int n = r.n - r.lo;
      first[b] = sum;
      sum += n > 0 ? (n + chunk_len(n) - 1) / chunk_len(n) : 0;
    }
    int inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    if (lane == 31) s_sum[warp] = inc;
    __syncthreads();
    int add = inc - sum;
    for (int w = 0; w < warp; ++w) add += s_sum[w];
    for (int b = b0; b < b1; ++b) first[b] += add;
    if (tid == kThreads - 1) first[a.B] = add + sum;
    __syncthreads();
  }
  const int items = first[a.B] * hkts;
  const uint32_t ring = smem_u32(smem) + warp * R::kStages * R::kStageBytes;
  const T* kc = static_cast<const T*>(a.k) + part * DW;
  const T* vc = static_cast<const T*>(a.v) + part * DW;

  // ---- the loads: `head` is the item being loaded, ht its next token, page its table entry for row lane % 16
  Item head = {};
  int hi = blockIdx.x, ht = 0, page = -1, slot = 0;
  int h_bc = hi / hkts, h_hkt = hi - h_bc * hkts;
  const int d_bc = gridDim.x / hkts, d_hkt = gridDim.x - d_bc * hkts;      // from one item of this CTA to its next
  const T *k_head = kc, *v_head = vc;             // of the item being loaded
  auto look_up = [&]() {                          // the table entry of the step at ht, ahead of its use
    const int t = ht + (lane & 15);
    const bool live = t >= head.r.first && t < head.t1;
    const int at = !live ? 0 : a.page_shift >= 0 ? t >> a.page_shift : t / a.page;
    slot = t - at * a.page;
    page = live ? a.tables[head.b * a.table_row + at] : -1;
    if (live && (page < 0 || page >= a.pages)) page = -2;         // named outside the cache
  };
  // q as the right operand: column = head, consecutive k in a register. The item that the warp computes next and its q are
  // fetched when the loads reach it, two steps before.
  Item it = {}, next = {};
  uint2 qn[NT][DW / 16];
  int next_i = -1, cur = -1;                      // numbers of the items in `next` and `it`
  const int cx = 2 * (lane & 3);                  // this thread's columns (heads): cx, cx + 1 of each tile
  auto fetch_q = [&]() {
    const int g0 = next.tile * kTile * NT, ng = min(kTile * NT, G - g0);
    const T* q = static_cast<const T*>(a.q) + next.b * a.q_b + (next.hk * G + g0) * a.q_h + part * DW + cx;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int g = nt * kTile + lane / 4;
#pragma unroll
      for (int kk = 0; kk < DW / 16; ++kk) {
        qn[nt][kk] = make_uint2(0, 0);
        if (g < ng) {
          const T* qp = q + g * a.q_h + kk * 16;
          qn[nt][kk].x = *reinterpret_cast<const uint32_t*>(qp);
          qn[nt][kk].y = *reinterpret_cast<const uint32_t*>(qp + 8);
        }
      }
    }
  };
  auto enter = [&]() {
    item_at(head, a, first, h_bc, h_hkt, tiles);
    ht = head.t0 + group * kRows;
    k_head = kc + head.hk * a.k_head;
    v_head = vc + head.hk * a.v_head;
    if (cur < 0 ? next_i < 0 : hi == cur + static_cast<int>(gridDim.x)) {
      next = head;
      next_i = hi;
      fetch_q();
    }
  };
  auto settle = [&]() {                           // the first step at or after (hi, ht) that this warp has
    while (hi < items && ht >= head.t1) {
      hi += gridDim.x;
      h_bc += d_bc;
      h_hkt += d_hkt;
      if (h_hkt >= hkts) {
        h_hkt -= hkts;
        ++h_bc;
      }
      if (hi < items) enter();
    }
    if (hi < items) look_up();
  };
  if (hi < items) {
    enter();
    settle();
  }
  // A lane copies 16 bytes of every (256 / DW)-th row, of keys and of values; one commit group, empty when nothing is left.
  constexpr int CH = DW / 8, RPI = 32 / CH;        // 16-byte pieces of a row, rows of one copy instruction
  const int ch = lane % CH, row0 = lane / CH;
  auto load = [&](int stage) {
    if (hi < items) {
      uint32_t dst = ring + stage * R::kStageBytes + row0 * R::kRowPitch + ch * 16;
      const int pa = __shfl_sync(0xffffffffu, page, 0), pb = __shfl_sync(0xffffffffu, page, 8);
      if (a.whole && ht >= head.r.first && ht + kRows <= head.t1 && pa >= 0 && pb >= 0) {
        // all sixteen tokens live, each eight of them on one page (its size is a multiple of 8, and so is ht)
        const int sa = __shfl_sync(0xffffffffu, slot, 0) + row0, sb = __shfl_sync(0xffffffffu, slot, 8) + row0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const T* ks = k_head + (h ? pb : pa) * a.k_page + (h ? sb : sa) * a.k_tok + ch * 8;
          const T* vs = v_head + (h ? pb : pa) * a.v_page + (h ? sb : sa) * a.v_tok + ch * 8;
#pragma unroll
          for (int i = 0; i < 8 / RPI; ++i) {
            const uint32_t at = dst + (h * 8 + i * RPI) * R::kRowPitch;
            copy16(at, ks);
            copy16(at + kRows * R::kRowPitch, vs);
            ks += RPI * a.k_tok;
            vs += RPI * a.v_tok;
          }
        }
      } else {
        // row by row: zeros for masked tokens, whatever the cache holds there, and for the key of a token on a bad page NaN,
        // which makes the sequence NaN
#pragma unroll 2
        for (int i = 0; i < kRows / RPI; ++i) {
          const int p = __shfl_sync(0xffffffffu, page, i * RPI + row0), s = __shfl_sync(0xffffffffu, slot, i * RPI + row0);
          const bool ok = p >= 0;
          const T* ks = ok ? k_head + p * a.k_page + s * a.k_tok + ch * 8 : kc;
          const T* vs = ok ? v_head + p * a.v_page + s * a.v_tok + ch * 8 : vc;
          if (p == -2)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst), "r"(0x7fff7fffu) : "memory");
          else
            copy16(dst, ks, ok);
          copy16(dst + kRows * R::kRowPitch, vs, ok);
          dst += RPI * R::kRowPitch;
        }
      }
      ht += kGroups * kRows;
      settle();
    }
    commit();
  };
#pragma unroll
  for (int s = 0; s < R::kStages - 1; ++s) load(s);
  int stage = 0;

  const float c2 = a.scale * kLog2e;
  int turn = 0;                                   // of the exchange's two buffers
  for (int i = blockIdx.x; i < items; i += gridDim.x) {
    cur = i;
    if (next_i != i) {                            // the loads passed it while an earlier item was computed
      const int bc = i / hkts;
      item_at(next, a, first, bc, i - bc * hkts, tiles);
      next_i = i;
      fetch_q();
    }
    it = next;
    const int hk = it.hk, g0 = it.tile * kTile * NT, ng = min(kTile * NT, G - g0);
    uint2 qf[NT][DW / 16];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int kk = 0; kk < DW / 16; ++kk) qf[nt][kk] = qn[nt][kk];
    float o[NT][DW / 16][4], m[NT][2], base[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      base[nt][0] = base[nt][1] = l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int dd = 0; dd < DW / 16; ++dd)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][dd][e] = 0.f;
    }
    for (int t = it.t0 + group * kRows; t < it.t1; t += kGroups * kRows) {
      load(stage == 0 ? R::kStages - 1 : stage - 1);
      wait_group<R::kStages - 1>();
      __syncwarp();
      const uint32_t ks = ring + stage * R::kStageBytes, vs = ks + kRows * R::kRowPitch;
      float s[NT][4], s2[NT][4];                  // two chains: a product waits for the one before it
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nt][e] = s2[nt][e] = 0.f;
      {
        const uint32_t at = ks + (lane & 15) * R::kRowPitch + (lane >> 4) * 16;
#pragma unroll
        for (int kk = 0; kk < DW / 16; ++kk) {
          uint32_t kf[4];
          ldm4(kf, at + kk * 32);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma<T>(kk & 1 ? s2[nt] : s[nt], kf, qf[nt][kk].x, qf[nt][kk].y);
          }
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nt][e] += s2[nt][e];
      if constexpr (DP == 2) {
        // the other half of the dims; a buffer is written again two steps later, past another meeting
        float* buf = s_x + ((group * 2 + turn) * 2) * NT * 4 * 32 + lane;
#pragma unroll
        for (int j = 0; j < NT * 4; ++j) buf[(part * NT * 4 + j) * 32] = s[j / 4][j % 4];
        asm volatile("bar.sync %0, 64;" ::"r"(1 + group) : "memory");
#pragma unroll
        for (int j = 0; j < NT * 4; ++j) s[j / 4][j % 4] += buf[((part ^ 1) * NT * 4 + j) * 32];
        turn ^= 1;
      }
      uint32_t hi_p[NT][2], lo_p[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nt][e] *= c2;
        if (t < it.r.first || t + kRows > it.t1) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int tt = t + lane / 4 + (e >> 1) * 8;
            if (tt < it.r.first || tt >= it.t1) s[nt][e] = -INFINITY;
          }
        }
        if (a.ws_x && part == 0) {
          float* xt = a.ws_x + ((static_cast<long long>(it.b) * a.Hkv + hk) * a.span + (t - it.r.lo)) * G + g0;
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            const int g = nt * kTile + cx, r = lane / 4 + (e >> 1) * 8;
            if (g >= ng || t + r < it.r.first || t + r >= it.t1) continue;
            if (G % 2 == 0) {
              *reinterpret_cast<float2*>(xt + r * G + g) = make_float2(s[nt][e], s[nt][e + 1]);
            } else {
              xt[r * G + g] = s[nt][e];
              if (g + 1 < ng) xt[r * G + g + 1] = s[nt][e + 1];
            }
          }
        }
        // The exponents' base is the largest logit so far, or one at most 8 below it (and for fp16 another 7 below): it is raised,
        // and what was summed is scaled, only when a logit is over 2^8 above it, which after the first step is rare. Weights
        // then go up to 2^15. bf16 loses nothing by that; fp16, whose steps end at 2^-24, keeps weights down to 2^-32 of the
        // largest that way, where a base at the largest itself would round what is below 2^-25 of it to nothing.
        const float big0 = fmaxf(s[nt][0], s[nt][2]), big1 = fmaxf(s[nt][1], s[nt][3]);
        if (__any_sync(0xffffffffu, big0 > m[nt][0] + 8.f || big1 > m[nt][1] + 8.f)) {
          float f[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float top = e ? big1 : big0;
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            top = fmaxf(top, m[nt][e]);
            f[e] = ex2(m[nt][e] - (top == -INFINITY ? 0.f : top));
            base[nt][e] = top == -INFINITY ? 0.f : top - kLift;
            m[nt][e] = top;
            l[nt][e] *= f[e];
          }
#pragma unroll
          for (int dd = 0; dd < DW / 16; ++dd)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[nt][dd][e] *= f[e & 1];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nt][e] = ex2(s[nt][e] - base[nt][e & 1]);
        l[nt][0] += s[nt][0] + s[nt][2];
        l[nt][1] += s[nt][1] + s[nt][3];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t top = pack2<T>(s[nt][2 * h], s[nt][2 * h + 1]);
          const float2 back = unpack2<T>(top);
          hi_p[nt][h] = transpose8(top);
          lo_p[nt][h] = transpose8(pack2<T>(s[nt][2 * h] - back.x, s[nt][2 * h + 1] - back.y));
        }
      }
      {
        const uint32_t at = vs + ((lane & 7) + ((lane >> 4) << 3)) * R::kRowPitch + ((lane >> 3) & 1) * 16;
#pragma unroll
        for (int dd = 0; dd < DW / 16; ++dd) {
          uint32_t vf[4];
          ldm4t(vf, at + dd * 32);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma<T>(o[nt][dd], vf, hi_p[nt][0], hi_p[nt][1]);
            mma<T>(o[nt][dd], vf, lo_p[nt][0], lo_p[nt][1]);
          }
        }
      }
      __syncwarp();                               // before the stage is filled again
      stage = stage + 1 == R::kStages ? 0 : stage + 1;
    }

    // ---- the four groups' results, in their order
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = l[nt][e];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        if (lane < 4 && part == 0) s_ml[group * kTile * NT + nt * kTile + cx + e] = make_float2(m[nt][e] - kLift, x);
      }
    const long long row = static_cast<long long>(it.b) * a.chunks * a.H + static_cast<long long>(it.c) * a.H + hk * G + g0;
    // a warp's results go through the stage of its ring that waits to be filled
    constexpr int kPitch = DW + 4;                // the rows of the four columns that a store writes lie in different banks
    static_assert(kTile * NT * kPitch * 4 <= R::kStageBytes, "results fit a stage");
    {
      const int idle = stage == 0 ? R::kStages - 1 : stage - 1;
      if (lane == 0) s_free[warp] = idle;
      float* mine = reinterpret_cast<float*>(smem + (warp * R::kStages + idle) * R::kStageBytes);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int dd = 0; dd < DW / 16; ++dd)
#pragma unroll
          for (int e = 0; e < 4; ++e) mine[(nt * kTile + cx + (e & 1)) * kPitch + dd * 16 + lane / 4 + (e >> 1) * 8] = o[nt][dd][e];
    }
    __syncthreads();
    // 128 threads to a part: sixteen to a head, two dims of every 32 to a thread
    const int mp = tid / 128, mh = tid % 128 / 16, d = tid % 16 * 2;
    const float* from[kGroups];
#pragma unroll
    for (int w = 0; w < kGroups; ++w)
      from[w] = reinterpret_cast<const float*>(smem + ((w * DP + mp) * R::kStages + s_free[w * DP + mp]) * R::kStageBytes);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int gg = nt * kTile + mh;
      if (gg >= ng) break;
      float top = -INFINITY, sum = 0.f, f[kGroups];
#pragma unroll
      for (int w = 0; w < kGroups; ++w) top = fmaxf(top, s_ml[w * kTile * NT + gg].x);
      const float from_top = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int w = 0; w < kGroups; ++w) {
        const float2 y = s_ml[w * kTile * NT + gg];
        f[w] = ex2(y.x - from_top);
        sum += y.y * f[w];            // NaN tokens leave m alone: 0 * NaN carries a sum of NaN on
      }
#pragma unroll
      for (int j = 0; j < DW / 32; ++j) {
        const int at = j * 32 + d, dim = mp * DW + at;
        float2 x = make_float2(0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kGroups; ++w) {
          const float2 y = *reinterpret_cast<const float2*>(from[w] + gg * kPitch + at);
          x.x += y.x * f[w];
          x.y += y.y * f[w];
        }
        if (it.chunks > 1) {
          if (dim == 0) a.ws_ml[row + gg] = make_float2(top, sum);
          *reinterpret_cast<float2*>(a.ws_o + (row + gg) * D + dim) = x;
        } else {
          finish<T, D>(a, it.b, hk * G + g0 + gg, dim, top, sum, x);
        }
      }
    }
    __syncthreads();
  }
  if (a.chunks <= 1) {                            // no join follows: sequences without tokens are answered here
    for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
      const Range r = range_of(a, b);
      if (r.n > 0) continue;
      for (int j = tid * 2; j < a.H * D; j += 64 * kWarps) finish<T, D>(a, b, j / D, j % D, -INFINITY, r.bad ? NAN : 0.f, make_float2(0.f, 0.f));
    }
  }
}

// CTA = (query head, sequence): a warp for every 32nd chunk, a lane for D / 32 dims; the warps' sums are added in their order.
// Where there are fewer than 32 chunks the block has fewer warps, one for each.
constexpr int kJoinWarps = 32;
static_assert(kMaxChunks <= 32 * kJoinWarps, "a chunk's maximum and sum to a thread");

template <int V> __device__ __forceinline__ void load_dims(float (&y)[V], const float* p) {
  if constexpr (V == 2) {
    const float2 u = *reinterpret_cast<const float2*>(p);
    y[0] = u.x, y[1] = u.y;
  } else {
#pragma unroll
    for (int v = 0; v < V; v += 4) {
      const float4 u = *reinterpret_cast<const float4*>(p + v);
      y[v] = u.x, y[v + 1] = u.y, y[v + 2] = u.z, y[v + 3] = u.w;
    }
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(32 * kJoinWarps) join_kernel(const Args a) {
  constexpr int V = D / 32, kAhead = V == 8 ? 4 : 8;
  const int warps = blockDim.x / 32;
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const Range r = range_of(a, b);
  const int span = r.n - r.lo, nc = span > 0 ? (span + chunk_len(span) - 1) / chunk_len(span) : 0;
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (nc == 1) return;                             // written by the split kernel
  __shared__ float s_f[kMaxChunks], s_top[kJoinWarps], s_sum[kJoinWarps];
  __shared__ __align__(16) float s_x[kJoinWarps][D];
  const float2* ml = a.ws_ml + static_cast<long long>(b) * a.chunks * a.H + h;
  const float* po = a.ws_o + (static_cast<long long>(b) * a.chunks * a.H + h) * D + lane * V;
  float y[kAhead][V];
  auto fetch = [&](int u0) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if ((u0 + u) * warps + warp < nc) load_dims<V>(y[u], po + static_cast<long long>((u0 + u) * warps + warp) * a.H * D);
  };
  fetch(0);                                        // on their way while the maximum is found
  const float2 mine = tid < nc ? ml[static_cast<long long>(tid) * a.H] : make_float2(-INFINITY, 0.f);
  float top = mine.x;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) s_top[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kMaxChunks / 32; ++w)
    if (w < warps) top = fmaxf(top, s_top[w]);
  const float f = ex2(mine.x - (top == -INFINITY ? 0.f : top));
  if (tid < nc) s_f[tid] = f;
  float sum = tid < nc ? __fmul_rn(mine.y, f) : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum = __fadd_rn(sum, __shfl_xor_sync(0xffffffffu, sum, o));
  if (lane == 0) s_sum[warp] = sum;
  __syncthreads();
  float x[V] = {};
  for (int u0 = 0; u0 * warps < nc; u0 += kAhead) {
    if (u0) fetch(u0);
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if ((u0 + u) * warps + warp < nc) {
        const float g = s_f[(u0 + u) * warps + warp];
#pragma unroll
        for (int v = 0; v < V; ++v) x[v] = __fadd_rn(x[v], __fmul_rn(y[u][v], g));
      }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) s_x[warp][lane * V + v] = x[v];
  __syncthreads();
  if (tid < D / 2) {
    sum = r.bad ? NAN : 0.f;
#pragma unroll
    for (int w = 0; w < kMaxChunks / 32; ++w)
      if (w < warps) sum = __fadd_rn(sum, s_sum[w]);
    float2 all = *reinterpret_cast<const float2*>(s_x[0] + 2 * tid);
#pragma unroll 8
    for (int w = 1; w < warps; ++w) {
      const float2 u = *reinterpret_cast<const float2*>(s_x[w] + 2 * tid);
      all.x = __fadd_rn(all.x, u.x);
      all.y = __fadd_rn(all.y, u.y);
    }
    finish<T, D>(a, b, h, 2 * tid, top, sum, all);
  }
}

// The same for tables of at most 32 chunks, with the same sums in the same order (a table's width must not change a bit): a
// warp per query head, a lane for each chunk's (maximum, sum) and for D / 32 dims.
constexpr int kFewThreads = 256;

template <typename T, int D>
__global__ void __launch_bounds__(kFewThreads) join_few_kernel(const Args a) {
  constexpr int V = D / 32, kAhead = 8;
  static_assert(kJoinWarps == 32, "a chunk to each of the other form's warps");
  const int lane = threadIdx.x % 32;
  const long long bh = static_cast<long long>(blockIdx.x) * (kFewThreads / 32) + threadIdx.x / 32;
  const int b = static_cast<int>(bh / a.H), h = static_cast<int>(bh % a.H);
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (b >= a.B) return;
  const Range r = range_of(a, b);
  const int span = r.n - r.lo, nc = span > 0 ? (span + chunk_len(span) - 1) / chunk_len(span) : 0;
  if (nc == 1) return;                             // written by the split kernel
  const float2* ml = a.ws_ml + static_cast<long long>(b) * a.chunks * a.H + h;
  const float* po = a.ws_o + (static_cast<long long>(b) * a.chunks * a.H + h) * D + lane * V;
  const float2 mine = lane < nc ? ml[static_cast<long long>(lane) * a.H] : make_float2(-INFINITY, 0.f);
  float top = mine.x;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float f = ex2(mine.x - (top == -INFINITY ? 0.f : top));
  float sum = lane < nc ? __fmul_rn(mine.y, f) : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum = __fadd_rn(sum, __shfl_xor_sync(0xffffffffu, sum, o));
  if (r.bad) sum = NAN;
  float all[V] = {};
  for (int c0 = 0; c0 < nc; c0 += kAhead) {
    float y[kAhead][V];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (c0 + u < nc) load_dims<V>(y[u], po + static_cast<long long>(c0 + u) * a.H * D);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const float g = __shfl_sync(0xffffffffu, f, (c0 + u) % 32);
      if (c0 + u < nc)
#pragma unroll
        for (int v = 0; v < V; ++v) all[v] = __fadd_rn(all[v], __fmul_rn(y[u][v], g));
    }
  }
#pragma unroll
  for (int v = 0; v < V; v += 2) finish<T, D>(a, b, h, lane * V + v, top, sum, make_float2(all[v], all[v + 1]));
}

// CTA = (chunk, kv head, sequence): a token's weights over the query heads of its kv head, added to its score. One addition
// per page slot and sequence for every 64 query heads of the kv head, in their order (the same thread adds them); atomic only
// because two sequences may share a page.
__global__ void __launch_bounds__(512) score_kernel(const Args a) {
  const int c = blockIdx.x, hk = blockIdx.y, b = blockIdx.z, G = a.H / a.Hkv, tid = threadIdx.x;
  const Range r = range_of(a, b);
  const int len = chunk_len(r.n - r.lo), t0 = r.lo + c * len, t1 = min(r.n, t0 + len);
  __shared__ float2 s_tot[64];                    // of 64 heads at a time: M and 1 / l, 0 where there is no weight
  const float* x = a.ws_x + (static_cast<long long>(b) * a.Hkv + hk) * a.span * G;
  asm volatile("griddepcontrol.wait;" ::: "memory");        // in every CTA: what follows on the stream relies on it
  if (t0 >= t1) return;
  for (int g0 = 0; g0 < G; g0 += 64) {
    const int ng = min(64, G - g0);
    __syncthreads();
    if (tid < ng) {
      const float2 y = a.ws_tot[static_cast<long long>(b) * a.H + hk * G + g0 + tid];
      s_tot[tid] = make_float2(y.x == -INFINITY ? 0.f : y.x, y.y == 0.f ? 0.f : 1.f / y.y);
    }
    __syncthreads();
    for (int t = t0 + tid; t < t1; t += blockDim.x) {
      const int at = a.page_shift >= 0 ? t >> a.page_shift : t / a.page;
      const int p = a.tables[b * a.table_row + at];
      if (t < r.first || p < 0 || p >= a.pages) continue;
      const float* xt = x + static_cast<long long>(t - r.lo) * G + g0;
      float w = 0.f;
      if (G % 4 == 0) {
#pragma unroll 2
        for (int g = 0; g < ng; g += 4) {
          const float4 y = *reinterpret_cast<const float4*>(xt + g);
          w += ex2(y.x - s_tot[g].x) * s_tot[g].y + ex2(y.y - s_tot[g + 1].x) * s_tot[g + 1].y +
               ex2(y.z - s_tot[g + 2].x) * s_tot[g + 2].y + ex2(y.w - s_tot[g + 3].x) * s_tot[g + 3].y;
        }
      } else {
        for (int g = 0; g < ng; ++g) w += ex2(xt[g] - s_tot[g].x) * s_tot[g].y;
      }
      atomicAdd(a.scores + (static_cast<long long>(p) * a.Hkv + hk) * a.page + (t - at * a.page), w);
    }
  }
}

constexpr int kMostSmem = 227 * 1024 - 1024;       // dynamic; the rest is for the static variables

int sm_count(int dev) {
  static std::atomic<int> known[64];
  int n = known[dev].load(std::memory_order_relaxed);
  if (!n) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) n = 148;
    known[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

template <typename T, int D, int NT>
int launch(const Args& a, int dev, cudaStream_t st) {
  const int G = a.H / a.Hkv, tiles = (G + kTile * NT - 1) / (kTile * NT);
  const int bytes = smem_bytes<D, NT>() + (a.B + 1) * 4;
  if (bytes > kMostSmem) return -2;
  static std::atomic<uint64_t> ready{0};        // devices on which the kernel may take its shared memory
  if (!(ready.load(std::memory_order_relaxed) >> dev & 1)) {
    if (cudaFuncSetAttribute(split_kernel<T, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem) != cudaSuccess) return -4;
    ready.fetch_or(uint64_t{1} << dev);
  }
  const long long most = static_cast<long long>(a.B) * a.chunks * a.Hkv * tiles;
  const int per_sm = 228 * 1024 / (bytes + 1024);
  const long long grid = static_cast<long long>(sm_count(dev)) * (per_sm > 0 ? per_sm : 1);
  split_kernel<T, D, NT><<<static_cast<unsigned>(most < 1 ? 1 : most < grid ? most : grid), 32 * Shape<D>::kWarps, bytes, st>>>(a);
  // these come up while the kernel before them runs, and wait for its end (griddepcontrol.wait) before they touch its results
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.H, a.B);
  cfg.blockDim = dim3(32 * (a.chunks >= kJoinWarps ? kJoinWarps : a.chunks > D / 64 ? a.chunks : D / 64));
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (a.chunks <= 1 && !a.scores) return cudaGetLastError() == cudaSuccess ? 0 : -4;
  // a warp per head wants at least a warp for every scheduler twice over; with fewer heads a block per head is faster (384
  // heads of 256 dims, 10 chunks: 50 us against 52 for the whole call; 2048 heads of 128, 8 chunks: 69 against 71)
  if (a.chunks > 32 || static_cast<long long>(a.H) * a.B < 1184) {
    if (a.chunks > 1 && cudaLaunchKernelEx(&cfg, join_kernel<T, D>, a) != cudaSuccess) return -4;
  } else if (a.chunks > 1) {
    cfg.gridDim = dim3(static_cast<unsigned>((static_cast<long long>(a.H) * a.B + kFewThreads / 32 - 1) / (kFewThreads / 32)));
    cfg.blockDim = dim3(kFewThreads);
    if (cudaLaunchKernelEx(&cfg, join_few_kernel<T, D>, a) != cudaSuccess) return -4;
  }
  if (a.scores && a.chunks > 0) {
    cfg.gridDim = dim3(a.chunks, a.Hkv, a.B);
    // few blocks: a thread for each of the usual 512 tokens (240 blocks: 45 us against 48 for the whole call; 2048 blocks: 71
    // against 69)
    cfg.blockDim = dim3(static_cast<long long>(a.chunks) * a.Hkv * a.B < 1184 ? 512 : 256);
    if (cudaLaunchKernelEx(&cfg, score_kernel, a) != cudaSuccess) return -4;
  }
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}

}  // namespace

extern "C" {

// The chunk rule's numbers, for the size of the workspaces: a sequence of at most n live tokens (its window + 15, where there
// is one) is cut into at most min(most, ceil(n / least)) chunks.
int tt_paged_split_least_chunk() { return kMinChunk; }
int tt_paged_split_most_chunks() { return kMaxChunks; }

// v: the arguments as 64-bit words -- addresses, whole numbers, strides in elements -- in the order of the names below. One
// block instead of some thirty arguments: a call from Python spends its time on those. dtype: 0 = bf16, 2 = fp16.
int tt_paged_split(const long long* v, float scale, cudaStream_t st) {
  enum { Q, K, V, TABLES, LENS, OUT, LSE, SINKS, SCORES, WS_O, WS_ML, WS_TOT, WS_X, Q_B, Q_H, K_PAGE, K_TOK, K_HEAD, V_PAGE, V_TOK,
         V_HEAD, TABLE_ROW, BATCH, HEADS, KV_HEADS, DIM, PAGE, WIDTH, PAGES, WINDOW, SPAN, CHUNKS, DTYPE };
  auto at = [&](int i) { return reinterpret_cast<void*>(v[i]); };
  auto num = [&](int i) { return static_cast<int>(v[i]); };
  const int B = num(BATCH), H = num(HEADS), Hkv = num(KV_HEADS), D = num(DIM), page = num(PAGE), dtype = num(DTYPE);
  if (B <= 0 || H <= 0) return 0;
  if (Hkv <= 0 || H % Hkv) return -12;
  if (B > kMaxBatch) return -2;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return -4;
  Args a = {};
  a.q = at(Q);
  a.k = at(K);
  a.v = at(V);
  a.tables = static_cast<const int*>(at(TABLES));
  a.lens = static_cast<const int*>(at(LENS));
  a.out = at(OUT);
  a.lse = static_cast<float*>(at(LSE));
  a.sinks = static_cast<const float*>(at(SINKS));
  a.scores = static_cast<float*>(at(SCORES));
  a.ws_o = static_cast<float*>(at(WS_O));
  a.ws_ml = static_cast<float2*>(at(WS_ML));
  a.ws_tot = static_cast<float2*>(at(WS_TOT));
  a.ws_x = static_cast<float*>(at(WS_X));
  a.q_b = v[Q_B];
  a.q_h = v[Q_H];
  a.k_page = v[K_PAGE];
  a.k_tok = v[K_TOK];
  a.k_head = v[K_HEAD];
  a.v_page = v[V_PAGE];
  a.v_tok = v[V_TOK];
  a.v_head = v[V_HEAD];
  a.table_row = v[TABLE_ROW];
  a.B = B;
  a.H = H;
  a.Hkv = Hkv;
  a.page = page;
  a.width = num(WIDTH);
  a.pages = num(PAGES);
  a.window = num(WINDOW);
  a.span = num(SPAN);
  a.chunks = num(CHUNKS);
  a.page_shift = page & (page - 1) ? -1 : __builtin_ctz(page);
  a.whole = page % 8 == 0;
  a.scale = scale;
#define PICK(T)                                   \
  switch (D) {                                    \
    case 64: return H / Hkv > kTile ? launch<T, 64, 2>(a, dev, st) : launch<T, 64, 1>(a, dev, st);     \
    case 128: return H / Hkv > kTile ? launch<T, 128, 2>(a, dev, st) : launch<T, 128, 1>(a, dev, st);  \
    case 256: return H / Hkv > kTile ? launch<T, 256, 2>(a, dev, st) : launch<T, 256, 1>(a, dev, st);  \
    default: return -10;                          \
  }
  if (dtype == 0) { PICK(__nv_bfloat16) }
  if (dtype == 2) { PICK(__half) }
#undef PICK
  return -11;
}

}  // extern "C"
