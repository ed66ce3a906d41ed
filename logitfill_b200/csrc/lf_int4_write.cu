// Writing tokens into the 4-bit paged cache and reading them back.
//
// Quantiser, for the 32 channels x of one group of one token (fp32):
//   s = fp16(RN(RN(max x - min x) * RN(1/15))),  z = fp16(min x)
//   r = RN(1 / s), or 0 where s = 0
//   code = clamp(round_half_even(RN(RN(x - z) * r)), 0, 15)
//   stored value = RN(code * s + z)
// The codes are formed with the fp16 scale and minimum that the reader uses,
// so the minimum's rounding costs no accuracy; a group whose scale or minimum
// is not a finite fp16 number (a NaN, an infinity, a value past 65504) reads
// back as NaN.
#include "lf_int4.cuh"

namespace lf {

template <typename T> __device__ __forceinline__ void load8(const T* p, float (&x)[8]);
template <> __device__ __forceinline__ void load8<float>(const float* p, float (&x)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
template <> __device__ __forceinline__ void load8<__half>(const __half* p, float (&x)[8]) {
  const uint4 w = *reinterpret_cast<const uint4*>(p);
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = half_lo(v[i]);
    x[2 * i + 1] = half_hi(v[i]);
  }
}
template <> __device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, float (&x)[8]) {
  const uint4 w = *reinterpret_cast<const uint4*>(p);
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(v[i] << 16);
    x[2 * i + 1] = __uint_as_float(v[i] & 0xFFFF0000u);
  }
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&x)[8]);
template <> __device__ __forceinline__ void store8<float>(float* p, const float (&x)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
template <> __device__ __forceinline__ void store8<__half>(__half* p, const float (&x)[8]) {
  uint32_t v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    v[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(v[0], v[1], v[2], v[3]);
}
template <> __device__ __forceinline__ void store8<__nv_bfloat16>(__nv_bfloat16* p, const float (&x)[8]) {
  uint32_t v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    v[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(v[0], v[1], v[2], v[3]);
}

// Codes (eight nibbles) and the parameter word of a lane's eight channels; the
// four lanes of a group take its extremes together.
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], uint32_t& param) {
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = min_nan(lo, x[i]);
    hi = max_nan(hi, x[i]);
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  const uint16_t sb = float_to_half_bits(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f));
  const uint16_t zb = float_to_half_bits(lo);
  if ((sb & 0x7C00u) == 0x7C00u || (zb & 0x7C00u) == 0x7C00u) {
    param = 0x7FFF7FFFu;
    return 0;
  }
  param = sb | (static_cast<uint32_t>(zb) << 16);
  const float s = half_bits_to_float(sb), z = half_bits_to_float(zb);
  const float r = s > 0.0f ? __fdiv_rn(1.0f, s) : 0.0f;
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float c = fminf(fmaxf(__fmul_rn(__fsub_rn(x[i], z), r), 0.0f), 15.0f);
    w |= static_cast<uint32_t>(__float2int_rn(c)) << (4 * i);
  }
  return w;
}

struct WriteParams {
  Int4Pool pool;
  const void *key, *value;
  int64_t k_seq, k_head, k_tok, v_seq, v_head, v_tok;
  int tokens;
  const int32_t *start, *counts;
  int8_t* bounds;
  int64_t bounds_page, bounds_head;  // bytes
  int32_t* status;
};

constexpr int kWriteThreads = 128;

// Channel bounds of a complete page's Key, from its record: the extremes of
// the stored values over the tokens, rounded outwards to whole steps of 2^e.
// Every thread of the CTA calls it.
template <int D>
__device__ void write_bounds(const int32_t* rec, int8_t* out) {
  constexpr int kCols = D / 8, kParts = kWriteThreads / kCols, kTok = kInt4Page / kParts;
  __shared__ float up_s[kParts][D], low_s[kParts][D];
  __shared__ float most_s[kWriteThreads / 32];
  const int col = threadIdx.x % kCols, part = threadIdx.x / kCols;
  const int t = col / (D / 32), G = col % (D / 32);
  float up[8], low[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    up[i] = -INFINITY;
    low[i] = INFINITY;
  }
  for (int k = part * kTok; k < (part + 1) * kTok; ++k) {
    const uint32_t w = __ldcg(reinterpret_cast<const uint32_t*>(rec) + k * kCols + col);
    const uint32_t pw = __ldcg(reinterpret_cast<const uint32_t*>(rec) + 8 * D + k * (D / 32) + G);
    const float s = half_lo(pw), z = half_hi(pw);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v = __fmaf_rn(static_cast<float>((w >> (4 * i)) & 15u), s, z);
      v = isfinite(v) ? v : 0.0f;
      up[i] = fmaxf(up[i], v);
      low[i] = fminf(low[i], v);
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    up_s[part][32 * G + 8 * t + i] = up[i];
    low_s[part][32 * G + 8 * t + i] = low[i];
  }
  __syncthreads();
  const int d = threadIdx.x;
  float u = 0.0f, l = 0.0f, m = 0.0f;
  if (d < D) {
    u = up_s[0][d];
    l = low_s[0][d];
#pragma unroll
    for (int q = 1; q < kParts; ++q) {
      u = fmaxf(u, up_s[q][d]);
      l = fminf(l, low_s[q][d]);
    }
    m = fmaxf(fabsf(u), fabsf(l));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) most_s[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int q = 0; q < kWriteThreads / 32; ++q) m = fmaxf(m, most_s[q]);
  const int e = exponent127(m);
  const float inv = pow2(-e);
  if (d < D) {
    out[d] = static_cast<int8_t>(ceilf(u * inv));
    out[D + d] = static_cast<int8_t>(floorf(l * inv));
  }
  if (d == 0) out[2 * D] = static_cast<int8_t>(e);
}

template <typename T, int D>
__global__ void __launch_bounds__(kWriteThreads) int4_write_kernel(const __grid_constant__ WriteParams p) {
  constexpr int kLanes = D / 8, kRows = kWriteThreads / kLanes;
  const int b = blockIdx.z, h = blockIdx.y;
  const int start = p.start[b];
  const int count = p.counts != nullptr ? min(p.counts[b], p.tokens) : p.tokens;
  if (count <= 0) return;
  if (start < 0 || start > INT32_MAX - count) {
    if (threadIdx.x == 0 && p.status != nullptr) atomicExch(p.status, LF_ERR_OUT_OF_RANGE);
    return;
  }
  const int page = start / kInt4Page + blockIdx.x;
  const int first = max(start, page * kInt4Page), last = min(start + count, (page + 1) * kInt4Page);
  if (first >= last) return;
  const int id = int4_page_id(p.pool, b, page);
  if (id < 0) {
    if (threadIdx.x == 0 && p.status != nullptr) atomicExch(p.status, LF_ERR_OUT_OF_RANGE);
    return;
  }
  int32_t* rec = p.pool.words + int4_record(p.pool, id, h);
  const int l = threadIdx.x % kLanes, row = threadIdx.x / kLanes;
  const T* key = static_cast<const T*>(p.key) + b * p.k_seq + h * p.k_head + 8 * l;
  const T* value = static_cast<const T*>(p.value) + b * p.v_seq + h * p.v_head + 8 * l;
  const int G = l >> 2, t = l & 3, u = G & 1;
  for (int pos0 = first; pos0 < last; pos0 += kRows) {  // whole warps stay together for the shuffles
    const int pos = min(pos0 + row, last - 1);
    const bool mine = pos0 + row < last;
    const int64_t src = pos - start;
    float xk[8], xv[8];
    load8<T>(key + src * p.k_tok, xk);
    load8<T>(value + src * p.v_tok, xv);
    uint32_t kp, vp;
    const uint32_t kw = quantise8(xk, kp);
    const uint32_t vw = quantise8(xv, vp);
    // The lane's channels are 4 of chunk g = 2 t and 4 of g + 1; the lane of the
    // neighbouring group (u flipped) holds the other halves of both words.
    const uint32_t got = __shfl_xor_sync(0xffffffffu, u == 0 ? vw >> 16 : vw & 0xFFFFu, 4);
    const uint32_t vword = u == 0 ? (vw & 0xFFFFu) | (got << 16) : got | (vw & 0xFFFF0000u);
    if (mine) {
      const int k = pos - page * kInt4Page;
      rec[k * (D / 8) + t * (D / 32) + G] = static_cast<int32_t>(kw);
      const int blk = k >> 3, pair = (k & 7) >> 1, odd = k & 1;
      rec[10 * D + blk * D + (2 * t + u) * (D / 8) + pair * (D / 32) + odd * (D / 64) + (G >> 1)] =
          static_cast<int32_t>(vword);
      if (t == 0) {
        rec[8 * D + k * (D / 32) + G] = static_cast<int32_t>(kp);
        rec[18 * D + k * (D / 32) + G] = static_cast<int32_t>(vp);
      }
    }
  }
  if (p.bounds == nullptr || last != (page + 1) * kInt4Page) return;
  __syncthreads();  // the page is complete: this CTA's stores are visible to all its threads
  write_bounds<D>(rec, p.bounds + id * p.bounds_page + h * p.bounds_head);
}

struct ReadParams {
  Int4Pool pool;
  const int32_t *start, *counts;
  int tokens;
  void *out_k, *out_v;
  int32_t* status;
};

// out [batch][kv_heads][tokens][D]: token i is position start[b] + i, zero from
// counts[b] on.
template <typename T, int D>
__global__ void __launch_bounds__(kWriteThreads) int4_read_kernel(const __grid_constant__ ReadParams p) {
  constexpr int kLanes = D / 8, kRows = kWriteThreads / kLanes;
  const int b = blockIdx.z, h = blockIdx.y;
  const int start = p.start[b];
  const int count = p.counts != nullptr ? p.counts[b] : p.tokens;
  const int l = threadIdx.x % kLanes, row = threadIdx.x / kLanes;
  const int G = l >> 2, t = l & 3, u = G & 1, w = G >> 1;
  const int last = min((static_cast<int>(blockIdx.x) + 1) * kInt4Page, p.tokens);
  for (int i = blockIdx.x * kInt4Page + row; i < last; i += kRows) {
    float xk[8] = {}, xv[8] = {};
    const int64_t pos = static_cast<int64_t>(start) + i;
    if (i < count) {
      const int id = pos < 0 || pos > INT32_MAX ? -1 : int4_page_id(p.pool, b, static_cast<int>(pos / kInt4Page));
      if (id < 0) {
        if (p.status != nullptr) atomicExch(p.status, LF_ERR_OUT_OF_RANGE);
      } else {
        const uint32_t* rec = reinterpret_cast<const uint32_t*>(p.pool.words) + int4_record(p.pool, id, h);
        const int k = static_cast<int>(pos % kInt4Page);
        const uint32_t kw = rec[k * (D / 8) + t * (D / 32) + G];
        const uint32_t kp = rec[8 * D + k * (D / 32) + G], vp = rec[18 * D + k * (D / 32) + G];
        const uint32_t* vc = rec + 10 * D + (k >> 3) * D + 2 * t * (D / 8) + ((k & 7) >> 1) * (D / 32) + (k & 1) * (D / 64) + w;
        const uint32_t vw = ((vc[0] >> (16 * u)) & 0xFFFFu) | ((vc[D / 8] >> (16 * u)) << 16);
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          xk[n] = __fmaf_rn(static_cast<float>((kw >> (4 * n)) & 15u), half_lo(kp), half_hi(kp));
          xv[n] = __fmaf_rn(static_cast<float>((vw >> (4 * n)) & 15u), half_lo(vp), half_hi(vp));
        }
      }
    }
    const int64_t dst = ((static_cast<int64_t>(b) * p.pool.kv_heads + h) * p.tokens + i) * D + 8 * l;
    store8<T>(static_cast<T*>(p.out_k) + dst, xk);
    store8<T>(static_cast<T*>(p.out_v) + dst, xv);
  }
}

// One thread per channel bound.
__global__ void int4_read_bounds_kernel(const int8_t* bounds, int64_t page_stride, int64_t head_stride, int heads,
                                        int D, int64_t total, float* out) {
  const int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x;
  if (i >= total) return;
  const int c = static_cast<int>(i % (2 * D));
  const int64_t r = i / (2 * D);
  const int8_t* rec = bounds + r / heads * page_stride + r % heads * head_stride;
  out[i] = static_cast<float>(rec[c]) * pow2(rec[2 * D]);
}

template <template <typename, int> class Launch, typename P>
static int by_type(int dtype, int D, dim3 grid, const P& p, cudaStream_t stream) {
  switch (dtype * 2 + (D == 128)) {
    case LF_F32 * 2: return Launch<float, 64>::go(grid, p, stream);
    case LF_F32 * 2 + 1: return Launch<float, 128>::go(grid, p, stream);
    case LF_F16 * 2: return Launch<__half, 64>::go(grid, p, stream);
    case LF_F16 * 2 + 1: return Launch<__half, 128>::go(grid, p, stream);
    case LF_BF16 * 2: return Launch<__nv_bfloat16, 64>::go(grid, p, stream);
    default: return Launch<__nv_bfloat16, 128>::go(grid, p, stream);
  }
}
template <typename T, int D> struct WriteLaunch {
  static int go(dim3 grid, const WriteParams& p, cudaStream_t stream) {
    int4_write_kernel<T, D><<<grid, kWriteThreads, 0, stream>>>(p);
    return launch_status("lf_int4_write");
  }
};
template <typename T, int D> struct ReadLaunch {
  static int go(dim3 grid, const ReadParams& p, cudaStream_t stream) {
    int4_read_kernel<T, D><<<grid, kWriteThreads, 0, stream>>>(p);
    return launch_status("lf_int4_read");
  }
};

int check_int4_pool(const char* what, const lf_int4_pool* pool, int head_dim, Int4Pool& out) {
  LF_CHECK_ARG(pool && pool->pages && pool->table, "%s: null pool, pages or page table", what);
  LF_CHECK_SUPPORTED(head_dim == 64 || head_dim == 128, "%s: head_dim %d (64 or 128)", what, head_dim);
  LF_CHECK_ARG(pool->kv_heads > 0 && pool->batch > 0 && pool->n_pages > 0 && pool->table_width > 0,
               "%s: empty pool, batch or page table", what);
  LF_CHECK_SUPPORTED(pool->kv_heads <= 65535 && pool->batch <= 65535, "%s: %d KV heads, batch %d (65535 at most)", what,
                     pool->kv_heads, pool->batch);
  LF_CHECK_ARG((reinterpret_cast<uintptr_t>(pool->pages) & 15) == 0 && pool->page_stride % 4 == 0 &&
                   pool->head_stride % 4 == 0 && pool->head_stride >= 20 * head_dim &&
                   pool->page_stride >= 20 * head_dim && pool->table_stride >= pool->table_width,
               "%s: records must be 16-byte aligned and apart", what);
  LF_CHECK_SUPPORTED(pool->table_width <= INT32_MAX / kInt4Page, "%s: page table width %d", what, pool->table_width);
  out.words = pool->pages;
  out.page_stride = pool->page_stride;
  out.head_stride = pool->head_stride;
  out.table = pool->table;
  out.table_stride = pool->table_stride;
  out.table_width = pool->table_width;
  out.n_pages = pool->n_pages;
  out.kv_heads = pool->kv_heads;
  out.batch = pool->batch;
  return LF_OK;
}

}  // namespace lf

extern "C" int lf_int4_write(const lf_int4_pool* pool, int head_dim, const void* key, const void* value, int dtype,
                             int64_t k_seq_stride, int64_t k_head_stride, int64_t k_tok_stride, int64_t v_seq_stride,
                             int64_t v_head_stride, int64_t v_tok_stride, int tokens, const int32_t* start,
                             const int32_t* counts, int8_t* bounds, int64_t bounds_page_stride,
                             int64_t bounds_head_stride, int32_t* status, lf_stream_t stream) {
  lf::WriteParams p;
  const int bad = lf::check_int4_pool("lf_int4_write", pool, head_dim, p.pool);
  if (bad != LF_OK) return bad;
  LF_CHECK_ARG(key && value && start, "lf_int4_write: null pointer");
  LF_CHECK_ARG(dtype == LF_F32 || dtype == LF_F16 || dtype == LF_BF16, "lf_int4_write: dtype %d", dtype);
  LF_CHECK_ARG(tokens >= 0 && tokens <= (1 << 30), "lf_int4_write: %d tokens", tokens);
  const int64_t unit = dtype == LF_F32 ? 4 : 8;  // elements in 16 bytes
  LF_CHECK_ARG(((reinterpret_cast<uintptr_t>(key) | reinterpret_cast<uintptr_t>(value)) & 15) == 0 &&
                   (k_seq_stride | k_head_stride | k_tok_stride | v_seq_stride | v_head_stride | v_tok_stride) % unit == 0,
               "lf_int4_write: Key and Value rows must be 16-byte aligned");
  LF_CHECK_ARG(bounds == nullptr || (bounds_page_stride > 2 * head_dim && bounds_head_stride > 2 * head_dim),
               "lf_int4_write: bounds records overlap");
  if (tokens == 0) return LF_OK;
  p.key = key;
  p.value = value;
  p.k_seq = k_seq_stride;
  p.k_head = k_head_stride;
  p.k_tok = k_tok_stride;
  p.v_seq = v_seq_stride;
  p.v_head = v_head_stride;
  p.v_tok = v_tok_stride;
  p.tokens = tokens;
  p.start = start;
  p.counts = counts;
  p.bounds = bounds;
  p.bounds_page = bounds_page_stride;
  p.bounds_head = bounds_head_stride;
  p.status = status;
  // tokens that start anywhere in a page touch at most this many pages
  const dim3 grid((tokens + 2 * lf::kInt4Page - 2) / lf::kInt4Page, p.pool.kv_heads, p.pool.batch);
  return lf::by_type<lf::WriteLaunch>(dtype, head_dim, grid, p, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int lf_int4_read(const lf_int4_pool* pool, int head_dim, const int32_t* start, const int32_t* counts,
                            int tokens, void* out_k, void* out_v, int out_dtype, int32_t* status, lf_stream_t stream) {
  lf::ReadParams p;
  const int bad = lf::check_int4_pool("lf_int4_read", pool, head_dim, p.pool);
  if (bad != LF_OK) return bad;
  LF_CHECK_ARG(start && out_k && out_v, "lf_int4_read: null pointer");
  LF_CHECK_ARG(out_dtype == LF_F32 || out_dtype == LF_F16 || out_dtype == LF_BF16, "lf_int4_read: dtype %d", out_dtype);
  LF_CHECK_ARG(tokens >= 0 && tokens <= (1 << 30), "lf_int4_read: %d tokens", tokens);
  LF_CHECK_ARG(((reinterpret_cast<uintptr_t>(out_k) | reinterpret_cast<uintptr_t>(out_v)) & 15) == 0,
               "lf_int4_read: outputs must be 16-byte aligned");
  if (tokens == 0) return LF_OK;
  p.start = start;
  p.counts = counts;
  p.tokens = tokens;
  p.out_k = out_k;
  p.out_v = out_v;
  p.status = status;
  const dim3 grid((tokens + lf::kInt4Page - 1) / lf::kInt4Page, p.pool.kv_heads, p.pool.batch);
  return lf::by_type<lf::ReadLaunch>(out_dtype, head_dim, grid, p, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int lf_int4_read_bounds(const int8_t* bounds, int64_t page_stride, int64_t head_stride, int n_pages,
                                   int kv_heads, int head_dim, float* out, lf_stream_t stream) {
  LF_CHECK_ARG(bounds && out, "lf_int4_read_bounds: null pointer");
  LF_CHECK_SUPPORTED(head_dim == 64 || head_dim == 128, "lf_int4_read_bounds: head_dim %d (64 or 128)", head_dim);
  LF_CHECK_ARG(n_pages > 0 && kv_heads > 0 && page_stride > 2 * head_dim && head_stride > 2 * head_dim,
               "lf_int4_read_bounds: empty or overlapping records");
  const int64_t total = static_cast<int64_t>(n_pages) * kv_heads * 2 * head_dim;
  const int64_t blocks = (total + 255) / 256;
  LF_CHECK_SUPPORTED(blocks <= INT32_MAX, "lf_int4_read_bounds: %d pages", n_pages);
  lf::int4_read_bounds_kernel<<<static_cast<unsigned>(blocks), 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      bounds, page_stride, head_stride, kv_heads, head_dim, total, out);
  return lf::launch_status("lf_int4_read_bounds");
}
