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
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kMinChunk = 256;    // tokens
constexpr int kMaxChunks = 128;   // per sequence: bounds the workspace and the join's work
constexpr int kTile = 8;          // query heads of one kv head that a CTA takes together

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
  int B, H, Hkv, page, width, pages, window, span, chunks;
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

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16(v); }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half(v); }

__device__ __forceinline__ int page_of(const Args& a, int b, int t) {
  const int p = a.tables[b * a.table_row + t / a.page];
  return p >= 0 && p < a.pages ? p : -1;
}

// CTA = (chunk, kv head and tile of its query heads, sequence). A warp takes every fourth token; a lane holds D / 32 dims.
template <typename T, int D>
__global__ void __launch_bounds__(128) split_kernel(const Args a) {
  constexpr int E = D / 32;
  const int c = blockIdx.x, tiles = gridDim.y / a.Hkv, hk = blockIdx.y / tiles, b = blockIdx.z;
  const int G = a.H / a.Hkv, g0 = (blockIdx.y % tiles) * kTile, ng = min(kTile, G - g0);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const Range r = range_of(a, b);
  const int len = chunk_len(r.n - r.lo), t0 = r.lo + c * len, t1 = min(r.n, t0 + len);
  if (t0 >= t1) return;
  __shared__ float s_o[4][kTile][D];
  __shared__ float2 s_ml[4][kTile];
  float qf[kTile][E], acc[kTile][E], m[kTile], l[kTile];
#pragma unroll
  for (int g = 0; g < kTile; ++g) {
    m[g] = -INFINITY;
    l[g] = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      acc[g][e] = 0.f;
      qf[g][e] = g < ng ? to_f(static_cast<const T*>(a.q)[b * a.q_b + (hk * G + g0 + g) * a.q_h + lane * E + e]) : 0.f;
    }
  }
  for (int t = t0 + warp; t < t1; t += 4) {
    if (t < r.first) continue;
    const int p = page_of(a, b, t);
    const T* kp = static_cast<const T*>(a.k) + max(p, 0) * a.k_page + (t % a.page) * a.k_tok + hk * a.k_head + lane * E;
    const T* vp = static_cast<const T*>(a.v) + max(p, 0) * a.v_page + (t % a.page) * a.v_tok + hk * a.v_head + lane * E;
    float kf[E], vf[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      kf[e] = to_f(kp[e]);
      vf[e] = to_f(vp[e]);
    }
#pragma unroll
    for (int g = 0; g < kTile; ++g) {
      float x = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) x += qf[g][e] * kf[e];
      for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
      x = p < 0 ? NAN : x * a.scale * kLog2e;
      if (a.ws_x && lane == 0 && g < ng)
        a.ws_x[((static_cast<long long>(b) * a.Hkv + hk) * a.span + (t - r.lo)) * G + g0 + g] = x;
      const float top = fmaxf(m[g], x);
      const float f = top == -INFINITY ? 0.f : exp2f(m[g] - top), w = x == -INFINITY ? 0.f : exp2f(x - top);
      m[g] = top;
      l[g] = l[g] * f + w;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[g][e] = acc[g][e] * f + w * vf[e];
    }
  }
#pragma unroll
  for (int g = 0; g < kTile; ++g) {
#pragma unroll
    for (int e = 0; e < E; ++e) s_o[warp][g][lane * E + e] = acc[g][e];
    if (lane == 0) s_ml[warp][g] = make_float2(m[g], l[g]);
  }
  __syncthreads();
  const long long row = (static_cast<long long>(b) * a.chunks + c) * a.H + hk * G + g0;
  for (int i = threadIdx.x; i < ng * D; i += 128) {
    const int g = i / D, d = i % D;
    float top = -INFINITY, sum = 0.f, o = 0.f;
    for (int w = 0; w < 4; ++w) top = fmaxf(top, s_ml[w][g].x);
    for (int w = 0; w < 4; ++w) {
      const float f = s_ml[w][g].x == -INFINITY ? 0.f : exp2f(s_ml[w][g].x - top);
      // a warp whose tokens all gave NaN has m = -inf but a NaN sum: the sum is taken whole
      sum += s_ml[w][g].x == -INFINITY ? s_ml[w][g].y : s_ml[w][g].y * f;
      o += s_ml[w][g].x == -INFINITY ? s_o[w][g][d] : s_o[w][g][d] * f;
    }
    a.ws_o[(row + g) * D + d] = o;
    if (d == 0) a.ws_ml[row + g] = make_float2(top, sum);
  }
}

// CTA = (query head, sequence).
template <typename T, int D>
__global__ void __launch_bounds__(128) join_kernel(const Args a) {
  const int h = blockIdx.x, b = blockIdx.y;
  const Range r = range_of(a, b);
  const int span = r.n - r.lo, nc = span > 0 ? (span + chunk_len(span) - 1) / chunk_len(span) : 0;
  const float2* ml = a.ws_ml + static_cast<long long>(b) * a.chunks * a.H + h;
  const float* po = a.ws_o + (static_cast<long long>(b) * a.chunks * a.H + h) * D;
  const float sink = a.sinks ? a.sinks[h] * kLog2e : -INFINITY;
  float top = sink;
  for (int c = 0; c < nc; ++c) top = fmaxf(top, ml[static_cast<long long>(c) * a.H].x);
  float sum = sink == -INFINITY ? 0.f : exp2f(sink - top);
  for (int c = 0; c < nc; ++c) {
    const float2 x = ml[static_cast<long long>(c) * a.H];
    sum += x.x == -INFINITY ? x.y : x.y * exp2f(x.x - top);
  }
  if (r.bad) sum = NAN;
  for (int d = threadIdx.x; d < D; d += 128) {
    float o = 0.f;
    for (int c = 0; c < nc; ++c) {
      const float mc = ml[static_cast<long long>(c) * a.H].x, x = po[static_cast<long long>(c) * a.H * D + d];
      o += mc == -INFINITY ? x : x * exp2f(mc - top);
    }
    static_cast<T*>(a.out)[(static_cast<long long>(b) * a.H + h) * D + d] = from_f<T>(sum == 0.f ? 0.f : o / sum);
  }
  if (threadIdx.x == 0) {
    if (a.lse) a.lse[static_cast<long long>(b) * a.H + h] = (top + log2f(sum)) * kLn2;
    if (a.ws_tot) a.ws_tot[static_cast<long long>(b) * a.H + h] = make_float2(top, sum);
  }
}

// CTA = (chunk, kv head, sequence): a token's weights over the query heads of its kv head, added to its score. One addition
// per page slot and sequence, atomic only because two sequences may share a page.
__global__ void __launch_bounds__(128) score_kernel(const Args a) {
  const int c = blockIdx.x, hk = blockIdx.y, b = blockIdx.z, G = a.H / a.Hkv;
  const Range r = range_of(a, b);
  const int len = chunk_len(r.n - r.lo), t0 = r.lo + c * len, t1 = min(r.n, t0 + len);
  const float2* tot = a.ws_tot + static_cast<long long>(b) * a.H + hk * G;
  for (int t = t0 + threadIdx.x; t < t1; t += 128) {
    const int p = page_of(a, b, t);
    if (t < r.first || p < 0) continue;
    const float* x = a.ws_x + ((static_cast<long long>(b) * a.Hkv + hk) * a.span + (t - r.lo)) * G;
    float w = 0.f;
    for (int g = 0; g < G; ++g) w += x[g] == -INFINITY ? 0.f : exp2f(x[g] - tot[g].x) / tot[g].y;
    atomicAdd(a.scores + (static_cast<long long>(p) * a.Hkv + hk) * a.page + t % a.page, w);
  }
}

template <typename T, int D>
int launch(const Args& a, cudaStream_t st) {
  const int G = a.H / a.Hkv, tiles = (G + kTile - 1) / kTile;
  if (a.chunks > 0) split_kernel<T, D><<<dim3(a.chunks, a.Hkv * tiles, a.B), 128, 0, st>>>(a);
  join_kernel<T, D><<<dim3(a.H, a.B), 128, 0, st>>>(a);
  if (a.scores && a.chunks > 0) score_kernel<<<dim3(a.chunks, a.Hkv, a.B), 128, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}

}  // namespace

extern "C" {

// Chunks that a sequence of at most `tokens` live tokens (its window, where there is one) can be cut into, and the tokens
// that are read for it: the sizes of the workspaces.
int tt_paged_split_chunks(int tokens, int window) {
  const int span = window > 0 && window + 15 < tokens ? window + 15 : tokens;
  const int c = (span + kMinChunk - 1) / kMinChunk;
  return c < kMaxChunks ? c : kMaxChunks;
}

// dtype: 0 = bf16, 2 = fp16. strides: q (sequence, head), k (page, token, head), v (page, token, head), table row.
int tt_paged_split(const void* q, const void* k, const void* v, const int* tables, const int* lens, void* out, float* lse,
                   const float* sinks, float* scores, float* ws_o, void* ws_ml, void* ws_tot, float* ws_x,
                   const long long* strides, int B, int H, int Hkv, int D, int page, int width, int pages, int window, int span,
                   int chunks, float scale, int dtype, cudaStream_t st) {
  if (B <= 0 || H <= 0) return 0;
  if (Hkv <= 0 || H % Hkv) return -12;
  if (B > 65535) return -2;
  Args a{q, k, v, tables, lens, out, lse, sinks, scores, ws_o, static_cast<float2*>(ws_ml), static_cast<float2*>(ws_tot), ws_x,
         strides[0], strides[1], strides[2], strides[3], strides[4], strides[5], strides[6], strides[7], strides[8],
         B, H, Hkv, page, width, pages, window, span, chunks, scale};
#define PICK(T)                                   \
  switch (D) {                                    \
    case 64: return launch<T, 64>(a, st);         \
    case 128: return launch<T, 128>(a, st);       \
    case 256: return launch<T, 256>(a, st);       \
    default: return -10;                          \
  }
  if (dtype == 0) { PICK(__nv_bfloat16) }
  if (dtype == 2) { PICK(__half) }
#undef PICK
  return -11;
}

}  // extern "C"
