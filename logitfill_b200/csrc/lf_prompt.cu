// Attention of whole prompts over their own tokens (lf_prompt_attend).
#include <cmath>

#include "lf_common.cuh"

namespace lf {

struct PromptParams {
  const void *q, *k, *v;
  void* out;
  int64_t q_seq, q_head, q_tok, k_seq, k_head, k_tok, v_seq, v_head, v_tok, o_seq, o_head, o_tok;
  const int32_t *starts, *counts;
  int32_t* status;
  float scale_log2;
  int batch, tokens, n_q, n_kv, group;
};

// Rows of sequence b: its first, how many tokens it has, and how many out rows it covers.
struct PromptSpan { int64_t first; int tokens, rows; };
__device__ __forceinline__ PromptSpan prompt_span(const PromptParams& p, int b) {
  if (p.starts != nullptr) {
    const int first = min(max(p.starts[b], 0), p.tokens), last = min(max(p.starts[b + 1], first), p.tokens);
    return {first, last - first, last - first};
  }
  return {0, p.counts != nullptr ? min(max(p.counts[b], 0), p.tokens) : p.tokens, p.tokens};
}

// One row by one warp: q over the first n keys, in fp32; the lane keeps D / 32 channels.
template <typename T, int D>
__device__ __forceinline__ void prompt_row(const T* q, const T* k, int64_t k_tok, const T* v, int64_t v_tok, int n, float scale_log2, T* out) {
  constexpr int kOwn = D / 32, kAhead = 4;
  const int d = (threadIdx.x & 31) * kOwn;
  float qx[kOwn], acc[kOwn], top = -INFINITY, sum = 0.0f;
#pragma unroll
  for (int x = 0; x < kOwn; ++x) {
    qx[x] = Scalar<T>::load(q + d + x);
    acc[x] = 0.0f;
  }
  for (int j = 0; j < n; j += kAhead) {
    float s[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      s[u] = 0.0f;
      const T* row = k + min(j + u, n - 1) * k_tok + d;
#pragma unroll
      for (int x = 0; x < kOwn; ++x) s[u] = fmaf(qx[x], Scalar<T>::load(row + x), s[u]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int u = 0; u < kAhead; ++u) s[u] += __shfl_xor_sync(0xffffffffu, s[u], o);
    float now = top;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      s[u] *= scale_log2;
      if (j + u < n) now = fmaxf(now, s[u]);
    }
    const float base = now == -INFINITY ? 0.0f : now, fix = exp2f(top - base);
    sum *= fix;
#pragma unroll
    for (int x = 0; x < kOwn; ++x) acc[x] *= fix;
    top = now;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (j + u >= n) break;
      const float w = exp2f(s[u] - base);
      sum += w;
      const T* row = v + (j + u) * v_tok + d;
#pragma unroll
      for (int x = 0; x < kOwn; ++x) acc[x] = fmaf(w, Scalar<T>::load(row + x), acc[x]);
    }
  }
#pragma unroll
  for (int x = 0; x < kOwn; ++x) Scalar<T>::store(out + d + x, sum == 0.0f ? 0.0f : acc[x] / sum);
}

// A warp to a row; rows of sequence blockIdx.z and q-head blockIdx.y.
template <typename T, int D>
__global__ void __launch_bounds__(256) prompt_simple_kernel(const __grid_constant__ PromptParams p) {
  grid_dep_wait();
  const int h = blockIdx.y;
  for (int b = blockIdx.z; b < p.batch; b += gridDim.z) {
    const PromptSpan s = prompt_span(p, b);
    const T* k = static_cast<const T*>(p.k) + b * p.k_seq + s.first * p.k_tok + h / p.group * p.k_head;
    const T* v = static_cast<const T*>(p.v) + b * p.v_seq + s.first * p.v_tok + h / p.group * p.v_head;
    for (int64_t i = blockIdx.x * 8 + (threadIdx.x >> 5); i < s.rows; i += gridDim.x * 8)
      prompt_row<T, D>(static_cast<const T*>(p.q) + b * p.q_seq + (s.first + i) * p.q_tok + h * p.q_head, k, p.k_tok, v, p.v_tok,
                       i < s.tokens ? static_cast<int>(i) + 1 : 0, p.scale_log2,
                       static_cast<T*>(p.out) + b * p.o_seq + (s.first + i) * p.o_tok + h * p.o_head);
  }
}

template <typename T> static const void* prompt_kernel(int head_dim) {
  return head_dim == 128 ? reinterpret_cast<const void*>(prompt_simple_kernel<T, 128>) : reinterpret_cast<const void*>(prompt_simple_kernel<T, 64>);
}

}  // namespace lf

extern "C" int lf_prompt_attend(const lf_prompt* a, lf_stream_t stream) {
  using namespace lf;
  LF_CHECK_ARG(a != nullptr, "lf_prompt_attend: null arguments");
  LF_CHECK_SUPPORTED(a->dtype == LF_F16 || a->dtype == LF_BF16, "lf_prompt_attend: dtype %d (fp16 or bf16)", a->dtype);
  LF_CHECK_SUPPORTED(a->head_dim == 64 || a->head_dim == 128, "lf_prompt_attend: head_dim %d (64 or 128)", a->head_dim);
  LF_CHECK_ARG(a->batch >= 0 && a->tokens >= 0 && a->n_kv > 0 && a->n_q > 0 && a->n_q % a->n_kv == 0,
               "lf_prompt_attend: batch %d, %d tokens, %d query heads on %d KV heads", a->batch, a->tokens, a->n_q, a->n_kv);
  LF_CHECK_SUPPORTED(a->n_q / a->n_kv <= 128 && a->n_q <= 65535, "lf_prompt_attend: %d query heads on %d KV heads (128 to one at most)",
                     a->n_q, a->n_kv);
  LF_CHECK_ARG(std::isfinite(a->scaling * 1.4426950408889634f), "lf_prompt_attend: scaling is not a finite number");
  if (a->batch == 0 || a->tokens == 0) return LF_OK;
  LF_CHECK_ARG(a->q && a->k && a->v && a->out, "lf_prompt_attend: null pointer");
  PromptParams p;
  const uintptr_t at = reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v) |
                       reinterpret_cast<uintptr_t>(a->out);
  LF_CHECK_ARG(at % 16 == 0, "lf_prompt_attend: rows must be 16-byte aligned");
  p.q = a->q;
  p.k = a->k;
  p.v = a->v;
  p.out = a->out;
  const bool many = a->starts == nullptr && a->batch > 1;
  bool fits = true;
  auto stride = [&](int64_t s, bool used) -> int64_t {
    fits = fits && (!used || (s > 0 && s % 8 == 0));
    return used ? s : 0;
  };
  p.q_seq = stride(a->q_seq_stride, many);
  p.q_head = stride(a->q_head_stride, a->n_q > 1);
  p.q_tok = stride(a->q_tok_stride, a->tokens > 1);
  p.k_seq = stride(a->k_seq_stride, many);
  p.k_head = stride(a->k_head_stride, a->n_kv > 1);
  p.k_tok = stride(a->k_tok_stride, a->tokens > 1);
  p.v_seq = stride(a->v_seq_stride, many);
  p.v_head = stride(a->v_head_stride, a->n_kv > 1);
  p.v_tok = stride(a->v_tok_stride, a->tokens > 1);
  p.o_seq = stride(a->out_seq_stride, many);
  p.o_head = stride(a->out_head_stride, a->n_q > 1);
  p.o_tok = stride(a->out_tok_stride, a->tokens > 1);
  LF_CHECK_ARG(fits, "lf_prompt_attend: strides must be positive multiples of 8 elements");
  p.starts = a->starts;
  p.counts = a->starts == nullptr ? a->counts : nullptr;
  p.status = a->status;
  p.scale_log2 = a->scaling * 1.4426950408889634f;
  p.batch = a->batch;
  p.tokens = a->tokens;
  p.n_q = a->n_q;
  p.n_kv = a->n_kv;
  p.group = a->n_q / a->n_kv;
  const int64_t rows = (static_cast<int64_t>(a->tokens) + 7) / 8;
  void* args[] = {&p};
  const cudaError_t err = launch_programmatic(
      a->dtype == LF_F16 ? prompt_kernel<__half>(a->head_dim) : prompt_kernel<__nv_bfloat16>(a->head_dim),
      dim3(static_cast<unsigned>(rows < 65535 ? rows : 65535), a->n_q, a->batch < 65535 ? a->batch : 65535), dim3(256), 0,
      reinterpret_cast<cudaStream_t>(stream), args);
  if (err != cudaSuccess) {
    set_error("lf_prompt_attend: %s", cudaGetErrorString(err));
    return LF_ERR_LAUNCH;
  }
  return launch_status("lf_prompt_attend");
}
