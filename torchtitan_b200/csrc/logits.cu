// Adjustment of a step's logits: penalties for tokens that were said before, biases, grammar masks.
//
// Per row, with c_i = how often token i was generated and s_i = whether it occurs in the prompt or what was generated:
//     x_i -> x_i / r if x_i > 0 else x_i * r          where s_i
//     x_i -> x_i - f * c_i - p * [c_i > 0]
//     x_i -> x_i + bias_i
//     x_i -> -inf                                     where the mask's bit i is 0
// computed in fp32 in this order, each step rounded on its own (no contraction, so that the result does not depend on the
// compiler), and rounded once to the logits' type. Tokens outside [0, V) in the history and the biases are skipped.
//
// The history is a list of tokens. A CTA takes a part of a row's vocabulary and keeps a word per token of it in shared memory:
// bits 0..19 how often it was generated, bit 20 that it was in the prompt, bits 21..31 one plus its entry in the bias list.
// Every CTA of a row reads the whole history for that: it comes from L2, 16 bytes to a thread, and needs no waiting for other
// CTAs (sharing the reading among a cluster of eight, counting in the owner's shared memory, took longer at every length up
// to 32768: 24 rows of 50021 logits 34 us against 18, 256 rows of 151936 with 2048 tokens 104 us against 67). Then it
// streams its part, 16 bytes to a thread, which the L2 has fetched meanwhile.
//
// What bounds it: each logit is read and written once. 256 rows of 151936 fp32 logits with 2048 tokens of history, 32 biases and
// a mask: 63 us, 5.1 TB/s, 0.77 of the measured copy rate; with a mask and one token of history 52 us. Parts of 12288 logits, four blocks of 512
// threads to an SM: with 6144 more of the time goes to the histories (74 us against 67), with 20480 fewer blocks overlap. Where
// blocks are few and histories long (24 rows of 50021 bf16 logits, 32768 tokens: 16 us in a graph, 1 us of bytes) a block has its SM
// to itself, but still the registers and the two loads ahead of one that shares it: 27 % of a warp's time is waiting for tokens.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

namespace {

constexpr int kThreads = 512;
constexpr int kMostPart = 12288;     // logits of one CTA
constexpr int kMaxBias = 1024;
constexpr int kAhead = 2;             // 16-byte pieces of the history that a thread loads before it counts them
constexpr uint32_t kCount = (1u << 20) - 1, kPrompt = 1u << 20;

struct Args {
  const void* x;
  void* y;
  const void* tokens;                 // int32 or int64 [B, L] or null
  const int *lens, *prompts;          // [B] or null
  const float *rep_t, *pres_t, *freq_t;   // [B] or null
  const int* bias_ids;                // [B, nb] or null
  const float* bias_values;
  const int* allowed;                 // [B, words] or null
  long long x_row, y_row, tok_row, id_row, val_row, mask_row;
  int V, L, nb, tok64, part;
  float rep, pres, freq;
};

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16(v); }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half(v); }

struct Setting { float rep, pres, freq; };

__device__ __forceinline__ float adjust(float x, uint32_t w, const Setting& s, const float* s_sum) {
  const uint32_t count = w & kCount;
  if (count | (w & kPrompt)) x = x > 0.f ? __fdiv_rn(x, s.rep) : __fmul_rn(x, s.rep);
  if (count) x = __fsub_rn(__fsub_rn(x, __fmul_rn(s.freq, static_cast<float>(count))), s.pres);
  if (w >> 21) x = __fadd_rn(x, s_sum[(w >> 21) - 1]);
  return x;
}

// Calls f(token, index) for the row's first n tokens, 16 bytes of them to a thread where they lie on such boundaries.
template <typename I, typename F>
__device__ __forceinline__ void each_token(const I* tok, int n, F f) {
  constexpr int N = 16 / sizeof(I);
  const int head = min(n, static_cast<int>((16 - reinterpret_cast<uintptr_t>(tok) % 16) % 16 / sizeof(I)));
  const int vectors = (n - head) / N;
  for (int i = threadIdx.x; i < head; i += kThreads) f(tok[i], i);
  for (int v0 = threadIdx.x; v0 < vectors; v0 += kAhead * kThreads) {       // loads first: counting must not hold them up
    union { uint4 v; I t[N]; } r[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (v0 + u * kThreads < vectors) r[u].v = *reinterpret_cast<const uint4*>(tok + head + (v0 + u * kThreads) * N);
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (v0 + u * kThreads < vectors)
#pragma unroll
        for (int e = 0; e < N; ++e) f(r[u].t[e], head + (v0 + u * kThreads) * N + e);
  }
  for (int i = head + vectors * N + threadIdx.x; i < n; i += kThreads) f(tok[i], i);
}

// WORDS: there are penalties or biases; otherwise only the mask is applied.
template <typename T, bool WORDS>
__global__ void __launch_bounds__(kThreads, 4) adjust_kernel(const Args a) {
  constexpr int E = 16 / sizeof(T);
  const int b = blockIdx.y, tid = threadIdx.x;
  const int v0 = min(a.V, static_cast<int>(blockIdx.x) * a.part), v1 = min(a.V, v0 + a.part);
  const T* x = static_cast<const T*>(a.x) + b * a.x_row;
  T* y = static_cast<T*>(a.y) + b * a.y_row;
  // the first logit of the part on a 16-byte boundary of x; word i of the part lies at pad + i, so that the words of a
  // vector lie on such a boundary too
  const int head = static_cast<int>((16 - reinterpret_cast<uintptr_t>(x + v0) % 16) % 16 / sizeof(T)), pad = (E - head) % E;
  extern __shared__ __align__(16) uint32_t word[];                       // [part + 2 E]
  int* s_id = reinterpret_cast<int*>(word + a.part + 2 * E);             // [nb]
  float* s_val = reinterpret_cast<float*>(s_id + a.nb);                  // [nb]
  float* s_sum = s_val + a.nb;                                           // [nb]
  __shared__ uint32_t s_again[WORDS ? kMaxBias / 32 : 1];
  // the logits and their mask come into L2 while the history is counted
  if (tid < 2 && v1 - v0 >= 64) {
    const uintptr_t from = tid == 0 ? reinterpret_cast<uintptr_t>(x + v0) : reinterpret_cast<uintptr_t>(a.allowed + b * a.mask_row + v0 / 32);
    const uintptr_t to = tid == 0 ? reinterpret_cast<uintptr_t>(x + v1) : reinterpret_cast<uintptr_t>(a.allowed + b * a.mask_row + v1 / 32);
    const uint32_t size = static_cast<uint32_t>((to & ~uintptr_t{15}) - (from & ~uintptr_t{15}));
    if ((tid == 0 || a.allowed) && size > 0)
      asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(from & ~uintptr_t{15}), "r"(size) : "memory");
  }
  Setting set{1.f, 0.f, 0.f};
  if constexpr (WORDS) {
    set = {a.rep_t ? a.rep_t[b] : a.rep, a.pres_t ? a.pres_t[b] : a.pres, a.freq_t ? a.freq_t[b] : a.freq};
    for (int i = tid; i < (a.part + 2 * E) / 4; i += kThreads) reinterpret_cast<uint4*>(word)[i] = make_uint4(0, 0, 0, 0);
    if (tid < kMaxBias / 32) s_again[tid] = 0;
    for (int i = tid; i < a.nb; i += kThreads) {
      s_id[i] = a.bias_ids[b * a.id_row + i];
      s_val[i] = s_sum[i] = a.bias_values[b * a.val_row + i];
    }
    __syncthreads();
    // the first entry to come claims its token; another one of the same token marks the claiming entry
    bool again = false;
    for (int i = tid; i < a.nb; i += kThreads) {
      const int id = s_id[i];
      if (id < v0 || id >= v1) continue;
      uint32_t* w = &word[pad + id - v0];
      uint32_t old = *w;
      while (!(old >> 21)) {
        const uint32_t seen = atomicCAS(w, old, old | (static_cast<uint32_t>(i + 1) << 21));
        if (seen == old) break;
        old = seen;
      }
      if (const uint32_t by = old >> 21) {
        atomicOr(&s_again[(by - 1) / 32], 1u << ((by - 1) % 32));
        again = true;
      }
    }
    if (a.tokens) {
      const int n = min(a.L, a.lens ? max(a.lens[b], 0) : a.L), np = a.prompts ? a.prompts[b] : 0;
      const uint32_t size = v1 - v0;
      auto count = [&](long long t, int i) {
        const unsigned long long at = static_cast<unsigned long long>(t - v0);
        if (at >= size) return;
        if (i >= np) atomicAdd(&word[pad + at], 1u); else atomicOr(&word[pad + at], kPrompt);
      };
      auto count32 = [&](int t, int i) {
        const uint32_t at = static_cast<uint32_t>(t) - static_cast<uint32_t>(v0);    // below 0 wraps to 2^31 and more
        if (at >= size) return;
        if (i >= np) atomicAdd(&word[pad + at], 1u); else atomicOr(&word[pad + at], kPrompt);
      };
      if (a.tok64) each_token(static_cast<const long long*>(a.tokens) + b * a.tok_row, n, count);
      else each_token(static_cast<const int*>(a.tokens) + b * a.tok_row, n, count32);
    }
    if (__syncthreads_or(again)) {
      // some tokens have several entries: a warp per such token sums them in their order
      const int lane = tid % 32;
      int turn = 0;
      for (int g = 0; g < (a.nb + 31) / 32; ++g) {
        for (uint32_t todo = s_again[g]; todo; todo &= todo - 1) {
          if (turn++ % (kThreads / 32) != tid / 32) continue;
          const int i = g * 32 + __ffs(todo) - 1, id = s_id[i];
          float sum = 0.f;
          bool any = false;
          for (int j0 = 0; j0 < a.nb; j0 += 32) {
            const int j = j0 + lane;
            const int other = j < a.nb ? s_id[j] : -1;
            const float v = j < a.nb ? s_val[j] : 0.f;
            for (uint32_t same = __ballot_sync(0xffffffffu, other == id); same; same &= same - 1) {
              const float u = __shfl_sync(0xffffffffu, v, __ffs(same) - 1);
              sum = any ? __fadd_rn(sum, u) : u;
              any = true;
            }
          }
          if (lane == 0) s_sum[i] = sum;
        }
      }
      __syncthreads();
    }
  }
  const uint32_t* mask = a.allowed ? reinterpret_cast<const uint32_t*>(a.allowed) + b * a.mask_row : nullptr;
  auto one = [&](int i) {
    float f = to_f(x[i]);
    if constexpr (WORDS) f = adjust(f, word[pad + i - v0], set, s_sum);
    y[i] = mask && !((mask[i / 32] >> (i % 32)) & 1u) ? from_f<T>(-INFINITY) : (WORDS ? from_f<T>(f) : x[i]);
  };
  // vectors where x and y lie alike, single logits before and behind them (and everywhere otherwise: 256 rows of 151937 fp32 logits
  // out of padded rows into dense ones 96 us, into rows padded alike 60)
  const bool alike = reinterpret_cast<uintptr_t>(x) % 16 == reinterpret_cast<uintptr_t>(y) % 16;
  const int w0 = alike ? min(v1, v0 + head) : v1, w1 = w0 + (v1 - w0) / E * E;
  for (int i = v0 + tid; i < w0; i += kThreads) one(i);
  for (int i = w1 + tid; i < v1; i += kThreads) one(i);
#pragma unroll 2
  for (int i = w0 + tid * E; i < w1; i += kThreads * E) {
    union { uint4 v; T e[E]; } r;
    r.v = *reinterpret_cast<const uint4*>(x + i);
    if constexpr (WORDS) {
      uint32_t w[E], any = 0;
#pragma unroll
      for (int e = 0; e < E; e += 4) *reinterpret_cast<uint4*>(w + e) = *reinterpret_cast<const uint4*>(word + pad + i - v0 + e);
#pragma unroll
      for (int e = 0; e < E; ++e) any |= w[e];
      if (any) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (w[e]) r.e[e] = from_f<T>(adjust(to_f(r.e[e]), w[e], set, s_sum));
      }
    }
    if (mask) {
      uint32_t m = mask[i / 32] >> (i % 32);
      if (i % 32 > 32 - E) m |= mask[i / 32 + 1] << (32 - i % 32);       // the vector's bits reach into the next word
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (!((m >> e) & 1u)) r.e[e] = from_f<T>(-INFINITY);
    }
    *reinterpret_cast<uint4*>(y + i) = r.v;
  }
}

template <typename T>
int launch(Args a, int B, cudaStream_t st) {
  const bool words = a.tokens || a.nb;
  // parts of equal size, at most kMostPart logits and, where rows are few, as many as give every SM a CTA, down to 1024
  int parts = (a.V + kMostPart - 1) / kMostPart;
  if (static_cast<long long>(B) * parts < 148) parts = max(parts, min((147 + B) / B, a.V / 1024));
  a.part = ((a.V + parts - 1) / parts + 31) / 32 * 32;
  const dim3 grid((a.V + a.part - 1) / a.part, B);
  if (words) {
    const int bytes = (a.part + 2 * (16 / static_cast<int>(sizeof(T)))) * 4 + a.nb * 12;
    static std::atomic<uint64_t> ready{0};        // devices on which the kernel may take its shared memory
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return -4;
    if (!(ready.load(std::memory_order_relaxed) >> dev & 1)) {
      if (cudaFuncSetAttribute(adjust_kernel<T, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (kMostPart + 64) * 4 + kMaxBias * 12) != cudaSuccess)
        return -4;
      ready.fetch_or(uint64_t{1} << dev);
    }
    adjust_kernel<T, true><<<grid, kThreads, bytes, st>>>(a);
  } else {
    adjust_kernel<T, false><<<grid, kThreads, 0, st>>>(a);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}

}  // namespace

extern "C" {

// v: the arguments as 64-bit words in the order of the names below; strides in elements. dtype: 0 = bf16, 1 = fp32, 2 = fp16.
int tt_process_logits(const long long* v, float rep, float pres, float freq, cudaStream_t st) {
  enum { X, Y, TOKENS, LENS, PROMPTS, REP, PRES, FREQ, BIAS_IDS, BIAS_VALUES, ALLOWED, X_ROW, Y_ROW, TOK_ROW, ID_ROW, VAL_ROW, MASK_ROW,
         TOK64, ENTRIES, BATCH, VOCAB, LENGTH, DTYPE };
  auto at = [&](int i) { return reinterpret_cast<void*>(v[i]); };
  const int B = static_cast<int>(v[BATCH]), dtype = static_cast<int>(v[DTYPE]);
  if (B <= 0 || v[VOCAB] <= 0) return 0;
  if (v[ENTRIES] > kMaxBias || v[LENGTH] > static_cast<int>(kCount) || B > 65535 || v[VOCAB] >= 1 << 30) return -2;
  Args a = {};
  a.x = at(X);
  a.y = at(Y);
  a.tokens = at(TOKENS);
  a.lens = static_cast<const int*>(at(LENS));
  a.prompts = static_cast<const int*>(at(PROMPTS));
  a.rep_t = static_cast<const float*>(at(REP));
  a.pres_t = static_cast<const float*>(at(PRES));
  a.freq_t = static_cast<const float*>(at(FREQ));
  a.bias_ids = static_cast<const int*>(at(BIAS_IDS));
  a.bias_values = static_cast<const float*>(at(BIAS_VALUES));
  a.allowed = static_cast<const int*>(at(ALLOWED));
  a.x_row = v[X_ROW];
  a.y_row = v[Y_ROW];
  a.tok_row = v[TOK_ROW];
  a.id_row = v[ID_ROW];
  a.val_row = v[VAL_ROW];
  a.mask_row = v[MASK_ROW];
  a.V = static_cast<int>(v[VOCAB]);
  a.L = static_cast<int>(v[LENGTH]);
  a.nb = static_cast<int>(v[ENTRIES]);
  a.tok64 = static_cast<int>(v[TOK64]);
  a.rep = rep;
  a.pres = pres;
  a.freq = freq;
  if (dtype == 0) return launch<__nv_bfloat16>(a, B, st);
  if (dtype == 1) return launch<float>(a, B, st);
  if (dtype == 2) return launch<__half>(a, B, st);
  return -11;
}

}  // extern "C"
