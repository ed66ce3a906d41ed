// Attention over the 4-bit paged cache (lf_int4_attend): dense over a
// sequence's pages, or over a list of picked ones.
//
// One CTA per (q-head, query token, sequence), one pass over its pages with a
// running maximum and sum: two threads per token form the scores of a page,
// one thread per channel sums the Values.
#include "lf_int4.cuh"

namespace lf {

struct AttendParams {
  Int4Pool pool;
  const void* q;
  int64_t q_seq, q_head, q_tok;
  int q_len, group;
  const int32_t *lengths, *counts;
  const int32_t* picked;
  int slots;
  float scale_log2;
  void* out;
  int64_t out_seq, out_head, out_tok;
  int32_t* status;
};

constexpr int kAttendThreads = 128;

template <typename T, int D>
__global__ void __launch_bounds__(kAttendThreads) int4_attend_kernel(const __grid_constant__ AttendParams p) {
  __shared__ float q_s[D], p_s[kInt4Page];
  const int head = blockIdx.x, i = blockIdx.y, b = blockIdx.z, h = head / p.group, tid = threadIdx.x;
  const int seen = int4_seen(p.lengths[b], p.counts != nullptr ? p.counts[b] : p.q_len, i);
  const T* q = static_cast<const T*>(p.q) + b * p.q_seq + head * p.q_head + i * p.q_tok;
  if (tid < D) q_s[tid] = Scalar<T>::load(q + tid) * p.scale_log2;
  __syncthreads();
  const int n = (seen + kInt4Page - 1) / kInt4Page;
  const int32_t* picked =
      p.picked == nullptr ? nullptr : p.picked + ((static_cast<int64_t>(b) * p.q_len + i) * p.pool.kv_heads + h) * p.slots;
  const int todo = picked == nullptr ? n : p.slots;
  float m = -1e30f, l = 0.0f, acc = 0.0f;
  for (int s = 0; s < todo; ++s) {
    const int page = picked == nullptr ? s : picked[s];
    if (page < 0 || page >= n) continue;
    const int id = int4_page_id(p.pool, b, page);
    if (id < 0) {
      if (tid == 0 && p.status != nullptr) atomicExch(p.status, LF_ERR_OUT_OF_RANGE);
      continue;
    }
    const uint32_t* rec = reinterpret_cast<const uint32_t*>(p.pool.words) + int4_record(p.pool, id, h);
    const int k = tid >> 1, half = tid & 1;
    float dot = 0.0f;
    for (int w = half * (D / 16); w < (half + 1) * (D / 16); ++w) {
      const int t = w / (D / 32), G = w % (D / 32);
      const uint32_t c = rec[k * (D / 8) + w], kp = rec[8 * D + k * (D / 32) + G];
      for (int x = 0; x < 8; ++x)
        dot += q_s[32 * G + 8 * t + x] * fmaf(static_cast<float>((c >> (4 * x)) & 15u), half_lo(kp), half_hi(kp));
    }
    dot += __shfl_xor_sync(0xffffffffu, dot, 1);
    if (page * kInt4Page + k >= seen) dot = -INFINITY;
    __syncthreads();
    if (half == 0) p_s[k] = dot;
    __syncthreads();
    float top = m;
    for (int x = 0; x < kInt4Page; ++x) top = fmaxf(top, p_s[x]);
    const float fix = exp2f(m - top);
    m = top;
    l *= fix;
    acc *= fix;
    const int w = (tid % D) >> 6, u = (tid >> 5) & 1, g = (tid & 31) >> 2, x = tid & 3, G = (tid % D) >> 5;
    for (int tok = 0; tok < min(kInt4Page, seen - page * kInt4Page); ++tok) {
      const float pr = exp2f(p_s[tok] - m);
      l += pr;
      const uint32_t c = rec[10 * D + (tok >> 3) * D + g * (D / 8) + ((tok & 7) >> 1) * (D / 32) + (tok & 1) * (D / 64) + w];
      const uint32_t vp = rec[18 * D + tok * (D / 32) + G];
      acc += pr * fmaf(static_cast<float>((c >> (4 * (4 * u + x))) & 15u), half_lo(vp), half_hi(vp));
    }
  }
  T* out = static_cast<T*>(p.out) + b * p.out_seq + head * p.out_head + i * p.out_tok;
  if (tid < D) Scalar<T>::store(out + tid, l == 0.0f ? 0.0f : acc / l);
}

template <typename T>
static int launch_attend(const AttendParams& p, int D, cudaStream_t stream) {
  const dim3 grid(p.group * p.pool.kv_heads, p.q_len, p.pool.batch);
  if (D == 128)
    int4_attend_kernel<T, 128><<<grid, kAttendThreads, 0, stream>>>(p);
  else
    int4_attend_kernel<T, 64><<<grid, kAttendThreads, 0, stream>>>(p);
  return launch_status("lf_int4_attend");
}

}  // namespace lf

extern "C" size_t lf_int4_workspace_bytes(int batch, int kv_heads, int n_q, int q_len, int head_dim) {
  if (batch <= 0 || kv_heads <= 0 || n_q <= 0 || q_len <= 0 || head_dim <= 0) return 0;
  return 16;
}

extern "C" int lf_int4_attend(const lf_int4_pool* pool, int head_dim, const void* q, int dtype, int64_t q_seq_stride,
                              int64_t q_head_stride, int64_t q_tok_stride, int q_len, int n_q, const int32_t* lengths,
                              const int32_t* counts, const int32_t* picked, int slots, float scaling, void* out, int64_t out_seq_stride,
                              int64_t out_head_stride, int64_t out_tok_stride, void* workspace, size_t workspace_bytes,
                              int32_t* status, lf_stream_t stream) {
  lf::AttendParams p;
  const int bad = lf::check_int4_pool("lf_int4_attend", pool, head_dim, p.pool);
  if (bad != LF_OK) return bad;
  LF_CHECK_ARG(q && lengths && out, "lf_int4_attend: null pointer");
  LF_CHECK_SUPPORTED(dtype == LF_F16 || dtype == LF_BF16, "lf_int4_attend: dtype %d (fp16 or bf16)", dtype);
  LF_CHECK_ARG(q_len > 0 && q_len <= 65535 && n_q > 0 && n_q % p.pool.kv_heads == 0,
               "lf_int4_attend: q_len %d, %d query heads on %d KV heads", q_len, n_q, p.pool.kv_heads);
  LF_CHECK_ARG(picked == nullptr || slots > 0, "lf_int4_attend: %d slots", slots);
  LF_CHECK_ARG(workspace && workspace_bytes >= lf_int4_workspace_bytes(p.pool.batch, p.pool.kv_heads, n_q, q_len, head_dim),
               "lf_int4_attend: workspace of %zu bytes is too small", workspace_bytes);
  p.q = q;
  p.q_seq = q_seq_stride;
  p.q_head = q_head_stride;
  p.q_tok = q_tok_stride;
  p.q_len = q_len;
  p.group = n_q / p.pool.kv_heads;
  p.lengths = lengths;
  p.counts = counts;
  p.picked = picked;
  p.slots = slots;
  p.scale_log2 = scaling * 1.4426950408889634f;
  p.out = out;
  p.out_seq = out_seq_stride;
  p.out_head = out_head_stride;
  p.out_tok = out_tok_stride;
  p.status = status;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return dtype == LF_F16 ? lf::launch_attend<__half>(p, head_dim, s) : lf::launch_attend<__nv_bfloat16>(p, head_dim, s);
}
