// Which pages a sparse attention call reads: a bound on the scores of each page
// from its Key bounds, and the best of them (lf_int4_select).
//
// One CTA per (query token, KV head).  The bound is a dot product of whole
// numbers, so every page's score is exact and the choice is the same on every
// run.
#include "lf_int4.cuh"

namespace lf {

struct SelectParams {
  Int4Pool pool;
  const void* q;
  int64_t q_seq, q_head, q_tok;
  int q_len, group;
  const int8_t* bounds;
  int64_t bounds_page, bounds_head;
  const int32_t *lengths, *counts;
  int top, sink, recent;
  int32_t* picked;
  int32_t* status;
};

constexpr int kSelectThreads = 256;
constexpr int kMaxSelectPages = 32768;  // candidates whose scores fit in shared memory

template <typename T, int D>
__global__ void __launch_bounds__(kSelectThreads) int4_select_kernel(const __grid_constant__ SelectParams p) {
  extern __shared__ float score_s[];
  __shared__ int plus_s[D], minus_s[D];
  __shared__ float most_s[kSelectThreads / 32];
  const int h = blockIdx.x, i = blockIdx.y, b = blockIdx.z;
  const int slots = p.top + p.sink + p.recent;
  int32_t* picked = p.picked + ((static_cast<int64_t>(b) * p.q_len + i) * p.pool.kv_heads + h) * slots;
  const int n = min((int4_seen(p.lengths[b], p.counts != nullptr ? p.counts[b] : p.q_len, i) + kInt4Page - 1) / kInt4Page, p.pool.table_width);
  if (n <= slots) {
    for (int s = threadIdx.x; s < slots; s += kSelectThreads) picked[s] = s < n ? s : -1;
    return;
  }
  const T* q = static_cast<const T*>(p.q) + b * p.q_seq + static_cast<int64_t>(h) * p.group * p.q_head + i * p.q_tok;
  float most = 0.0f;
  for (int x = threadIdx.x; x < p.group * D; x += kSelectThreads) {
    const float v = fabsf(Scalar<T>::load(q + (x / D) * p.q_head + x % D));
    most = isfinite(v) ? fmaxf(most, v) : most;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
  if ((threadIdx.x & 31) == 0) most_s[threadIdx.x >> 5] = most;
  __syncthreads();
  for (int w = 0; w < kSelectThreads / 32; ++w) most = fmaxf(most, most_s[w]);
  const int f = exponent127(most);
  if (threadIdx.x < D) {
    int plus = 0, minus = 0;
    for (int j = 0; j < p.group; ++j) {
      const float v = Scalar<T>::load(q + j * p.q_head + threadIdx.x);
      const int c = isfinite(v) ? __float2int_rn(scalbnf(v, -f)) : 0;
      plus += max(c, 0);
      minus += min(c, 0);
    }
    plus_s[threadIdx.x] = plus;
    minus_s[threadIdx.x] = minus;
  }
  __syncthreads();
  const int first = p.sink, count = n - p.sink - p.recent;  // candidates: pages first .. first + count - 1
  for (int c = threadIdx.x; c < count; c += kSelectThreads) {
    const int id = int4_page_id(p.pool, b, first + c);
    float score = -INFINITY;
    if (id >= 0) {
      const int8_t* rec = p.bounds + id * p.bounds_page + h * p.bounds_head;
      int sum = 0;
      for (int d = 0; d < D; ++d) sum += rec[d] * plus_s[d] + rec[D + d] * minus_s[d];
      score = __int2float_rn(sum) * pow2(rec[2 * D]);
    } else if (p.status != nullptr) {
      atomicExch(p.status, LF_ERR_OUT_OF_RANGE);
    }
    score_s[c] = score;
  }
  __syncthreads();
  // A candidate's place: how many are better.  Then the chosen ones in order.
  for (int c = threadIdx.x; c < count; c += kSelectThreads) {
    const float mine = score_s[c];
    int better = 0;
    for (int o = 0; o < count; ++o) better += score_s[o] > mine || (score_s[o] == mine && o < c);
    if (better < p.top) {
      int place = 0;  // chosen candidates before this one
      for (int o = 0; o < c; ++o) {
        int r = 0;
        for (int x = 0; x < count; ++x) r += score_s[x] > score_s[o] || (score_s[x] == score_s[o] && x < o);
        place += r < p.top;
      }
      picked[p.sink + place] = first + c;
    }
  }
  for (int s = threadIdx.x; s < p.sink; s += kSelectThreads) picked[s] = s;
  for (int s = threadIdx.x; s < p.recent; s += kSelectThreads) picked[p.sink + p.top + s] = n - p.recent + s;
}

template <typename T>
static int launch_select(const SelectParams& p, int D, cudaStream_t stream) {
  const dim3 grid(p.pool.kv_heads, p.q_len, p.pool.batch);
  const int smem = p.pool.table_width * static_cast<int>(sizeof(float));
  const void* kern = D == 128 ? reinterpret_cast<const void*>(int4_select_kernel<T, 128>)
                              : reinterpret_cast<const void*>(int4_select_kernel<T, 64>);
  if (raise_smem_limit(kern, smem, false) != cudaSuccess) return launch_status("lf_int4_select");
  if (D == 128)
    int4_select_kernel<T, 128><<<grid, kSelectThreads, smem, stream>>>(p);
  else
    int4_select_kernel<T, 64><<<grid, kSelectThreads, smem, stream>>>(p);
  return launch_status("lf_int4_select");
}

}  // namespace lf

extern "C" int lf_int4_select(const lf_int4_pool* pool, int head_dim, const void* q, int q_dtype, int64_t q_seq_stride,
                              int64_t q_head_stride, int64_t q_tok_stride, int q_len, int n_q, const int8_t* bounds,
                              int64_t bounds_page_stride, int64_t bounds_head_stride, const int32_t* lengths,
                              const int32_t* counts, int top_pages, int sink_pages, int recent_pages, int32_t* picked, int32_t* status,
                              lf_stream_t stream) {
  lf::SelectParams p;
  const int bad = lf::check_int4_pool("lf_int4_select", pool, head_dim, p.pool);
  if (bad != LF_OK) return bad;
  LF_CHECK_ARG(q && bounds && lengths && picked, "lf_int4_select: null pointer");
  LF_CHECK_SUPPORTED(q_dtype == LF_F16 || q_dtype == LF_BF16, "lf_int4_select: query dtype %d (fp16 or bf16)", q_dtype);
  LF_CHECK_ARG(q_len > 0 && q_len <= 65535 && n_q > 0 && n_q % p.pool.kv_heads == 0,
               "lf_int4_select: q_len %d, %d query heads on %d KV heads", q_len, n_q, p.pool.kv_heads);
  LF_CHECK_SUPPORTED(n_q / p.pool.kv_heads <= 64, "lf_int4_select: %d query heads per KV head (64 at most)",
                     n_q / p.pool.kv_heads);
  LF_CHECK_ARG(top_pages >= 0 && sink_pages >= 0 && recent_pages >= 1 && top_pages <= (1 << 24) &&
                   sink_pages <= (1 << 24) && recent_pages <= (1 << 24),
               "lf_int4_select: top %d, sink %d, recent %d pages (recent at least 1)", top_pages, sink_pages, recent_pages);
  LF_CHECK_ARG(bounds_page_stride > 2 * head_dim && bounds_head_stride > 2 * head_dim,
               "lf_int4_select: bounds records overlap");
  LF_CHECK_SUPPORTED(p.pool.table_width <= lf::kMaxSelectPages, "lf_int4_select: %d pages per sequence (%d at most)",
                     p.pool.table_width, lf::kMaxSelectPages);
  p.q = q;
  p.q_seq = q_seq_stride;
  p.q_head = q_head_stride;
  p.q_tok = q_tok_stride;
  p.q_len = q_len;
  p.group = n_q / p.pool.kv_heads;
  p.bounds = bounds;
  p.bounds_page = bounds_page_stride;
  p.bounds_head = bounds_head_stride;
  p.lengths = lengths;
  p.counts = counts;
  p.top = top_pages;
  p.sink = sink_pages;
  p.recent = recent_pages;
  p.picked = picked;
  p.status = status;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return q_dtype == LF_F16 ? lf::launch_select<__half>(p, head_dim, s) : lf::launch_select<__nv_bfloat16>(p, head_dim, s);
}
