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
// The history is a list of tokens. A cluster of CTAs covers the vocabulary (or a slab of it), each CTA one part, for which it
// keeps a word per token in shared memory: bits 0..19 how often it was generated, bit 20 that it was in the prompt, bits
// 21..31 one plus its entry in the bias list. The CTAs share the reading of the history and count in the word's owner, so a
// row's history is read once. Then every CTA streams its part, 16 bytes to a thread.
#include <cuda_bf16.h>
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 512;
constexpr int kCluster = 8;
constexpr int kMostPart = 12288;     // logits of one CTA
constexpr int kMaxBias = 1024;
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

// WORDS: there are penalties or biases (a cluster per slab of the vocabulary); otherwise only the mask is applied.
template <typename T, bool WORDS>
__global__ void __launch_bounds__(kThreads) adjust_kernel(const Args a) {
  constexpr int E = 16 / sizeof(T);
  const int b = blockIdx.y, tid = threadIdx.x;
  const int slab0 = blockIdx.x / kCluster * kCluster * a.part;                  // first logit of the cluster
  const int v0 = min(a.V, static_cast<int>(blockIdx.x) * a.part), v1 = min(a.V, v0 + a.part);
  const T* x = static_cast<const T*>(a.x) + b * a.x_row;
  T* y = static_cast<T*>(a.y) + b * a.y_row;
  // the first logit of the part on a 16-byte boundary of x; word i of the part lies at pad + i, so that the words of a
  // vector lie on such a boundary too
  const int head = static_cast<int>((16 - reinterpret_cast<uintptr_t>(x + v0) % 16) % 16 / sizeof(T)), pad = (E - head) % E;
  extern __shared__ __align__(16) uint32_t word[];
  __shared__ __align__(16) int s_id[WORDS ? kMaxBias : 4];
  __shared__ float s_val[WORDS ? kMaxBias : 1], s_sum[WORDS ? kMaxBias : 1];
  Setting set{1.f, 0.f, 0.f};
  if constexpr (WORDS) {
    cg::cluster_group cluster = cg::this_cluster();
    set = {a.rep_t ? a.rep_t[b] : a.rep, a.pres_t ? a.pres_t[b] : a.pres, a.freq_t ? a.freq_t[b] : a.freq};
    const int nb4 = (a.nb + 3) / 4 * 4;
    for (int i = tid; i < (a.part + 2 * E) / 4; i += kThreads) reinterpret_cast<uint4*>(word)[i] = make_uint4(0, 0, 0, 0);
    for (int i = tid; i < nb4; i += kThreads) {
      s_id[i] = i < a.nb ? a.bias_ids[b * a.id_row + i] : -1;
      s_val[i] = i < a.nb ? a.bias_values[b * a.val_row + i] : 0.f;
    }
    cluster.sync();
    if (a.tokens) {
      const int n = min(a.L, a.lens ? max(a.lens[b], 0) : a.L), np = a.prompts ? a.prompts[b] : 0;
      const int slab1 = min(static_cast<long long>(a.V), slab0 + static_cast<long long>(kCluster) * a.part);
      for (int i = cluster.block_rank() * kThreads + tid; i < n; i += kCluster * kThreads) {
        const long long t = a.tok64 ? static_cast<const long long*>(a.tokens)[b * a.tok_row + i]
                                    : static_cast<const int*>(a.tokens)[b * a.tok_row + i];
        if (t < slab0 || t >= slab1) continue;
        const int owner = static_cast<int>(t - slab0) / a.part, at = static_cast<int>(t - slab0) - owner * a.part;
        // the owner's padding follows from its part's address
        const int o_head = static_cast<int>((16 - reinterpret_cast<uintptr_t>(x + slab0 + owner * a.part) % 16) % 16 / sizeof(T));
        uint32_t* w = cluster.map_shared_rank(word, owner) + (E - o_head) % E + at;
        if (i < np) atomicOr(w, kPrompt); else atomicAdd(w, 1u);
      }
    }
    // an entry's token in this part: the first entry of a token sums them all, in their order
    for (int i = tid; i < a.nb; i += kThreads) {
      const int id = s_id[i];
      if (id < v0 || id >= v1) continue;
      float sum = 0.f;
      bool first = true;
      for (int j = 0; j < nb4; j += 4) {
        const int4 q = *reinterpret_cast<const int4*>(s_id + j);
        if (q.x == id) { first &= j >= i; sum = __fadd_rn(sum, s_val[j]); }
        if (q.y == id) { first &= j + 1 >= i; sum = __fadd_rn(sum, s_val[j + 1]); }
        if (q.z == id) { first &= j + 2 >= i; sum = __fadd_rn(sum, s_val[j + 2]); }
        if (q.w == id) { first &= j + 3 >= i; sum = __fadd_rn(sum, s_val[j + 3]); }
      }
      if (first) {
        s_sum[i] = sum;
        atomicOr(&word[pad + id - v0], static_cast<uint32_t>(i + 1) << 21);
      }
    }
    cluster.sync();
  }
  const uint32_t* mask = a.allowed ? reinterpret_cast<const uint32_t*>(a.allowed) + b * a.mask_row : nullptr;
  auto one = [&](int i) {
    float f = to_f(x[i]);
    if constexpr (WORDS) f = adjust(f, word[pad + i - v0], set, s_sum);
    y[i] = mask && !((mask[i / 32] >> (i % 32)) & 1u) ? from_f<T>(-INFINITY) : (WORDS ? from_f<T>(f) : x[i]);
  };
  // vectors where x and y lie alike, single logits before and behind them (and everywhere otherwise)
  const bool alike = reinterpret_cast<uintptr_t>(x) % 16 == reinterpret_cast<uintptr_t>(y) % 16;
  const int w0 = alike ? min(v1, v0 + head) : v1, w1 = w0 + (v1 - w0) / E * E;
  for (int i = v0 + tid; i < w0; i += kThreads) one(i);
  for (int i = w1 + tid; i < v1; i += kThreads) one(i);
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
      const uint32_t m = __funnelshift_r(mask[i / 32], mask[(i + E - 1) / 32], i % 32);
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
  // parts of equal size: a cluster (or several) per row, each CTA at most kMostPart logits and, where rows are few, as many
  // clusters as give every SM a CTA, down to 1024 logits each
  int slabs = (a.V + kCluster * kMostPart - 1) / (kCluster * kMostPart);
  while (static_cast<long long>(B) * slabs * kCluster < 148 && a.V / (slabs * kCluster) >= 2048) ++slabs;
  a.part = ((a.V + slabs * kCluster - 1) / (slabs * kCluster) + 31) / 32 * 32;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kCluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(slabs * kCluster, B);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  if (words) {
    cfg.dynamicSmemBytes = static_cast<size_t>(a.part + 2 * (16 / sizeof(T))) * 4;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaFuncSetAttribute(adjust_kernel<T, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (kMostPart + 64) * 4) != cudaSuccess) return -4;
    return cudaLaunchKernelEx(&cfg, adjust_kernel<T, true>, a) == cudaSuccess ? 0 : -4;
  }
  return cudaLaunchKernelEx(&cfg, adjust_kernel<T, false>, a) == cudaSuccess ? 0 : -4;
}

}  // namespace

extern "C" {

// dtype: 0 = bf16, 1 = fp32, 2 = fp16. strides (elements): x row, y row, tokens row, bias ids row, bias values row, mask row.
int tt_process_logits(const void* x, void* y, const void* tokens, int tok64, const int* lens, const int* prompts, const float* rep_t,
                      const float* pres_t, const float* freq_t, float rep, float pres, float freq, const int* bias_ids,
                      const float* bias_values, int nb, const int* allowed, const long long* strides, int B, int V, int L, int dtype,
                      cudaStream_t st) {
  if (B <= 0 || V <= 0) return 0;
  if (nb > kMaxBias || L > static_cast<int>(kCount) || B > 65535 || V >= 1 << 30) return -2;
  Args a{x, y, tokens, lens, prompts, rep_t, pres_t, freq_t, bias_ids, bias_values, allowed,
         strides[0], strides[1], strides[2], strides[3], strides[4], strides[5], V, L, nb, tok64, 0, rep, pres, freq};
  if (dtype == 0) return launch<__nv_bfloat16>(a, B, st);
  if (dtype == 1) return launch<float>(a, B, st);
  if (dtype == 2) return launch<__half>(a, B, st);
  return -11;
}

}  // extern "C"
