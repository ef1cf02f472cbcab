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
// The history is a list of tokens; a CTA counts those of its part of the vocabulary in shared memory: bits 0..19 count,
// bit 20 = seen, bits 21..31 = 1 + entry of the bias list.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace {

constexpr int kThreads = 256;
constexpr int kPart = 4096;          // logits of one CTA
constexpr int kMaxBias = 1024;
constexpr uint32_t kCount = (1u << 20) - 1, kSeen = 1u << 20;

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
  int V, L, nb, tok64;
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

template <typename T>
__global__ void __launch_bounds__(kThreads) adjust_kernel(const Args a) {
  const int b = blockIdx.y, tid = threadIdx.x, v0 = blockIdx.x * kPart, v1 = min(a.V, v0 + kPart);
  __shared__ uint32_t word[kPart];
  __shared__ int s_id[kMaxBias];
  __shared__ float s_val[kMaxBias], s_sum[kMaxBias];
  for (int i = tid; i < kPart; i += kThreads) word[i] = 0;
  for (int i = tid; i < a.nb; i += kThreads) {
    s_id[i] = a.bias_ids[b * a.id_row + i];
    s_val[i] = a.bias_values[b * a.val_row + i];
  }
  __syncthreads();
  if (a.tokens) {
    const int n = min(a.L, a.lens ? max(a.lens[b], 0) : a.L), np = a.prompts ? a.prompts[b] : 0;
    for (int i = tid; i < n; i += kThreads) {
      const long long t = a.tok64 ? static_cast<const long long*>(a.tokens)[b * a.tok_row + i]
                                  : static_cast<const int*>(a.tokens)[b * a.tok_row + i];
      if (t < v0 || t >= v1) continue;
      if (i >= np) atomicAdd(&word[t - v0], 1u);
      atomicOr(&word[t - v0], kSeen);
    }
  }
  // one sum per entry, over all entries of the same token in their order: the same value whichever entry is looked up
  for (int i = tid; i < a.nb; i += kThreads) {
    const int id = s_id[i];
    if (id < v0 || id >= v1) continue;
    float sum = 0.f;
    for (int j = 0; j < a.nb; ++j)
      if (s_id[j] == id) sum = __fadd_rn(sum, s_val[j]);
    s_sum[i] = sum;
  }
  __syncthreads();
  for (int i = tid; i < a.nb; i += kThreads) {
    const int id = s_id[i];
    if (id >= v0 && id < v1) atomicMax(&word[id - v0], (word[id - v0] & (kSeen | kCount)) | (static_cast<uint32_t>(i + 1) << 21));
  }
  __syncthreads();
  const float rep = a.rep_t ? a.rep_t[b] : a.rep, pres = a.pres_t ? a.pres_t[b] : a.pres, freq = a.freq_t ? a.freq_t[b] : a.freq;
  for (int i = v0 + tid; i < v1; i += kThreads) {
    float x = to_f(static_cast<const T*>(a.x)[b * a.x_row + i]);
    const uint32_t w = word[i - v0];
    if (w & kSeen) x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
    if (w & kCount) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, static_cast<float>(w & kCount))), pres);
    if (w >> 21) x = __fadd_rn(x, s_sum[(w >> 21) - 1]);
    if (a.allowed && !((static_cast<uint32_t>(a.allowed[b * a.mask_row + i / 32]) >> (i % 32)) & 1u)) x = -INFINITY;
    static_cast<T*>(a.y)[b * a.y_row + i] = from_f<T>(x);
  }
}

}  // namespace

extern "C" {

// dtype: 0 = bf16, 1 = fp32, 2 = fp16. strides (elements): x row, y row, tokens row, bias ids row, bias values row, mask row.
int tt_process_logits(const void* x, void* y, const void* tokens, int tok64, const int* lens, const int* prompts, const float* rep_t,
                      const float* pres_t, const float* freq_t, float rep, float pres, float freq, const int* bias_ids,
                      const float* bias_values, int nb, const int* allowed, const long long* strides, int B, int V, int L, int dtype,
                      cudaStream_t st) {
  if (B <= 0 || V <= 0) return 0;
  if (nb > kMaxBias || L > static_cast<int>(kCount) || B > 65535) return -2;
  Args a{x, y, tokens, lens, prompts, rep_t, pres_t, freq_t, bias_ids, bias_values, allowed,
         strides[0], strides[1], strides[2], strides[3], strides[4], strides[5], V, L, nb, tok64, rep, pres, freq};
  const dim3 grid((V + kPart - 1) / kPart, B);
  if (dtype == 0) adjust_kernel<__nv_bfloat16><<<grid, kThreads, 0, st>>>(a);
  else if (dtype == 1) adjust_kernel<float><<<grid, kThreads, 0, st>>>(a);
  else if (dtype == 2) adjust_kernel<__half><<<grid, kThreads, 0, st>>>(a);
  else return -11;
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}

}  // extern "C"
