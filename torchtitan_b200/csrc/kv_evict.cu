// Eviction from a paged KV cache by accumulated attention weight.
//
// For every (sequence, kv head) with n cached tokens: n <= keep keeps all of them; otherwise the last `recent` tokens stay
// and, of the n - recent before them, the keep - recent with the largest score, ties going to the lowest index. What stays
// is copied, in its order, to the first slots of new pages: the old pages are only read, so they may be shared.
//
// Selection: the score's bits, mapped so that unsigned order is score order, are cut 8 at a time from the top: a histogram
// of the digit among the tokens that match the digits found so far gives the next digit of the keep-th largest. Four passes
// find it exactly; what equals it is taken in index order until the count is full.
#include <cuda_runtime.h>
#include <stdint.h>

namespace {

struct Args {
  char *k, *v;
  float* scores;             // [pages, Hkv, page]
  const int *tables, *lens, *fresh;
  int *new_lens, *kept;      // [B], [B, Hkv, keep]
  long long k_page, k_tok, k_head, v_page, v_tok, v_head;   // bytes
  long long table_row, fresh_row;
  int B, Hkv, page, width, fresh_width, pages, row_bytes, keep, recent;
};

// Larger key = kept earlier. NaN counts as the largest value, both zeros are one value.
__device__ __forceinline__ uint32_t key_of(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t b = __float_as_uint(v + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

__device__ __forceinline__ int length_of(const Args& a, int b) {
  const int n = a.lens[b];
  return n < 0 || n > a.width * a.page ? 0 : n;
}

__device__ __forceinline__ uint32_t key_at(const Args& a, int b, int h, int t) {
  const int p = a.tables[b * a.table_row + t / a.page];
  if (p < 0 || p >= a.pages) return 0u;
  return key_of(a.scores[(static_cast<long long>(p) * a.Hkv + h) * a.page + t % a.page]);
}

constexpr int kThreads = 1024;

// CTA = (kv head, sequence): writes the kept indices in order.
__global__ void __launch_bounds__(kThreads) select_kernel(const Args a) {
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int n = length_of(a, b), left = min(n, a.keep);
  int* kept = a.kept + (static_cast<long long>(b) * a.Hkv + h) * a.keep;
  if (h == 0 && tid == 0) a.new_lens[b] = left;
  for (int j = left + tid; j < a.keep; j += kThreads) kept[j] = -1;
  if (n <= a.keep) {
    for (int j = tid; j < n; j += kThreads) kept[j] = j;
    return;
  }
  const int old = n - a.recent;
  int want = a.keep - a.recent;       // of the first `old` tokens
  __shared__ int hist[256];
  __shared__ uint32_t s_prefix;
  __shared__ int s_want, s_base, s_ties;
  __shared__ int s_warp[32], s_warp_t[32];
  uint32_t prefix = 0;
  if (want > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kThreads) hist[i] = 0;
      __syncthreads();
      for (int t = tid; t < old; t += kThreads) {
        const uint32_t key = key_at(a, b, h, t);
        if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(key >> shift) & 255], 1);
      }
      __syncthreads();
      if (tid == 0) {
        int d = 255, above = 0;
        while (d > 0 && above + hist[d] < want) above += hist[d--];
        s_want = want - above;
        s_prefix = prefix | (static_cast<uint32_t>(d) << shift);
      }
      __syncthreads();
      want = s_want;
      prefix = s_prefix;
      __syncthreads();
    }
  }
  // now `want` of the tokens that equal prefix are taken, lowest index first, and all above it
  if (tid == 0) { s_base = 0; s_ties = 0; }
  __syncthreads();
  for (int t0 = 0; t0 < n; t0 += kThreads) {
    const int t = t0 + tid;
    bool take = false, tie = false;
    if (t < n) {
      if (t >= old) take = true;
      else if (a.keep > a.recent) {
        const uint32_t key = key_at(a, b, h, t);
        take = key > prefix;
        tie = key == prefix;
      }
    }
    const uint32_t tie_mask = __ballot_sync(0xffffffffu, tie);
    if (lane == 0) s_warp_t[warp] = __popc(tie_mask);
    __syncthreads();
    int before = s_ties;
    for (int w = 0; w < warp; ++w) before += s_warp_t[w];
    if (tie && before + __popc(tie_mask & ((1u << lane) - 1)) < want) take = true;
    const uint32_t mask = __ballot_sync(0xffffffffu, take);
    if (lane == 0) s_warp[warp] = __popc(mask);
    __syncthreads();
    int at = s_base;
    for (int w = 0; w < warp; ++w) at += s_warp[w];
    if (take) kept[at + __popc(mask & ((1u << lane) - 1))] = t;
    __syncthreads();
    if (tid == 0)
      for (int w = 0; w < 32; ++w) { s_base += s_warp[w]; s_ties += s_warp_t[w]; }
    __syncthreads();
  }
}

// One thread per 16 bytes of a kept row; the first of a row's threads moves its score too.
__global__ void __launch_bounds__(256) move_kernel(const Args a) {
  const int per = a.row_bytes / 16;
  const int b = blockIdx.y;
  const int left = min(length_of(a, b), a.keep);
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  const int c = static_cast<int>(i % per);
  const long long r = i / per;
  const int h = static_cast<int>(r % a.Hkv);
  const long long j = r / a.Hkv;
  if (j >= left) return;
  const int t = a.kept[(static_cast<long long>(b) * a.Hkv + h) * a.keep + j];
  const int sp = a.tables[b * a.table_row + t / a.page], dp = a.fresh[b * a.fresh_row + j / a.page];
  if (sp < 0 || sp >= a.pages || dp < 0 || dp >= a.pages) return;
  const int so = t % a.page, to = static_cast<int>(j % a.page);
  *reinterpret_cast<uint4*>(a.k + dp * a.k_page + to * a.k_tok + h * a.k_head + c * 16) =
      *reinterpret_cast<const uint4*>(a.k + sp * a.k_page + so * a.k_tok + h * a.k_head + c * 16);
  *reinterpret_cast<uint4*>(a.v + dp * a.v_page + to * a.v_tok + h * a.v_head + c * 16) =
      *reinterpret_cast<const uint4*>(a.v + sp * a.v_page + so * a.v_tok + h * a.v_head + c * 16);
  if (c == 0)
    a.scores[(static_cast<long long>(dp) * a.Hkv + h) * a.page + to] = a.scores[(static_cast<long long>(sp) * a.Hkv + h) * a.page + so];
}

}  // namespace

extern "C" {

// strides in bytes: k (page, token, head), v (page, token, head), then in elements: table row, new table row.
int tt_kv_evict(void* k, void* v, float* scores, const int* tables, const int* lens, const int* fresh, int* new_lens, int* kept,
                const long long* strides, int B, int Hkv, int page, int width, int fresh_width, int pages, int row_bytes, int keep,
                int recent, cudaStream_t st) {
  if (B <= 0 || Hkv <= 0) return 0;
  if (B > 65535 || row_bytes % 16 || keep < 1 || recent < 0 || recent > keep) return -2;
  const long long room = static_cast<long long>(width) * page, most = room < keep ? room : keep;
  if (most > static_cast<long long>(fresh_width) * page) return -2;
  Args a{static_cast<char*>(k), static_cast<char*>(v), scores, tables, lens, fresh, new_lens, kept,
         strides[0], strides[1], strides[2], strides[3], strides[4], strides[5], strides[6], strides[7],
         B, Hkv, page, width, fresh_width, pages, row_bytes, keep, recent};
  select_kernel<<<dim3(Hkv, B), kThreads, 0, st>>>(a);
  const long long threads = most * Hkv * (row_bytes / 16);
  if (threads > 0) move_kernel<<<dim3(static_cast<unsigned>((threads + 255) / 256), B), 256, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}

}  // extern "C"
