// Writing tokens into the 4-bit paged cache and reading them back.
//
// Quantiser, for the 32 channels x of one group of one token (fp32):
//   s = fp16(RN(RN(max x - min x) * RN(1/15))),  z = fp16(min x)
//   r = RN(1 / s), or 0 where s = 0
//   code = clamp(round_half_even(RN(RN(x - z) * r)), 0, 15)
//   stored value = RN(code * s + z)
// The codes are formed with the fp16 scale and minimum that the reader uses,
// so the minimum's rounding costs no accuracy; a group whose scale or minimum
// is not a finite fp16 number (a NaN, an infinity, a range past 15 * 65504)
// reads back as NaN.
//
// Both directions move 4 D bytes of 16-bit Key and Value and 1.25 D of record per
// token and head, so HBM would bound them; what is left above that is arithmetic.
// It is kept small by extremes of packed pairs, two of them in one shuffle; three
// fp32 instructions (two of them on pairs) and one integer one per code; codes
// read back as subnormal halves.  The writer builds a page's record in shared
// memory and stores whole rows of it: the record's order puts a token's Value words
// 64 bytes apart, and stored one by one they would fill eight times as many sectors
// (66 us instead of 49).
//
// Measured for 16 sequences of 4096 bf16 tokens, 4 KV heads, D 128 (176 MB each
// way): write 46.3 us (3.8 TB/s), of which loads and stores alone 32.9, parameters
// 2.3, codes 5, bounds 6; the issue slots are 76 % busy.  Read 31.6 us (5.6 TB/s).
// One token of 16 sequences: 2 to 3 us each, the latency of three dependent loads.
#include <type_traits>

#include "lf_int4.cuh"

namespace lf {

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

// Smaller (larger) half of each pair, NaN where one is NaN.
template <typename T, bool kMax> __device__ __forceinline__ uint32_t pick2(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (std::is_same<T, __half>::value) {
    if constexpr (kMax)
      asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else
      asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  } else {
    if constexpr (kMax)
      asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else
      asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  }
  return r;
}
template <typename T> struct Chunk {  // eight 16-bit channels
  uint32_t w[4];
  __device__ __forceinline__ void load(const T* p) {
    const uint4 x = *reinterpret_cast<const uint4*>(p);
    w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
  }
  __device__ __forceinline__ void unpack(float (&x)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __half>::value) {
        x[2 * i] = half_lo(w[i]);
        x[2 * i + 1] = half_hi(w[i]);
      } else {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
      }
    }
  }
  __device__ __forceinline__ void extremes(float& lo, float& hi) const {
    const uint32_t a = pick2<T, false>(pick2<T, false>(w[0], w[1]), pick2<T, false>(w[2], w[3]));
    const uint32_t b = pick2<T, true>(pick2<T, true>(w[0], w[1]), pick2<T, true>(w[2], w[3])) ^ 0x80008000u;
    // (min, -max) in one word: one shuffle joins both over the group's four lanes
    uint32_t both = pick2<T, false>(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) both = pick2<T, false>(both, __shfl_xor_sync(0xffffffffu, both, o));
    if constexpr (std::is_same<T, __half>::value) {
      lo = half_lo(both);
      hi = -half_hi(both);
    } else {
      lo = __uint_as_float(both << 16);
      hi = -__uint_as_float(both & 0xFFFF0000u);
    }
  }
};
template <> struct Chunk<float> {
  float v[8];
  __device__ __forceinline__ void load(const float* p) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
  __device__ __forceinline__ void unpack(float (&x)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = v[i];
  }
  __device__ __forceinline__ void extremes(float& lo, float& hi) const {
    lo = hi = v[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
      lo = min_nan(lo, v[i]);
      hi = max_nan(hi, v[i]);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
  }
};

// A group's parameters from its extremes: the stored word, z and r / 16 (0 for a
// group that is not stored; negative where the largest channel's code would be 16:
// codes grow with x, so no other group needs the clamp to 15.  It takes a |min| of
// a thousand steps or more, whose fp16 rounding then shows in x - z).
struct GroupParams {
  uint32_t word;
  float z, r16;
};
__device__ __forceinline__ GroupParams group_params(float lo, float hi) {
  const uint16_t sb = float_to_half_bits(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f));
  const uint16_t zb = float_to_half_bits(lo);
  const bool bad = (sb & 0x7C00u) == 0x7C00u || (zb & 0x7C00u) == 0x7C00u;
  const float s = half_bits_to_float(sb);
  GroupParams g;
  g.word = bad ? 0x7FFF7FFFu : sb | (static_cast<uint32_t>(zb) << 16);
  g.z = half_bits_to_float(zb);
  // r / 16: a power of two less, so the product with it is the definition's over
  // 16 and its saturation to [0, 1] clamps the code to 0 .. 16 for free
  g.r16 = s > 0.0f && !bad ? __frcp_rn(s) * 0.0625f : 0.0f;
  if (__fmul_rn(__fsub_rn(hi, g.z), g.r16) >= 15.5f / 16.0f) g.r16 = -g.r16;
  return g;
}

// Codes (eight nibbles) of a lane's eight channels.  16 y + 1.5 * 2^23 rounds to a
// whole number, half to even, in the low bits of the sum; the magic numbers,
// shifted as the codes are, come off at the end.
template <typename T>
__device__ __forceinline__ uint32_t quantise8(const Chunk<T>& chunk, const GroupParams& g) {
  float x[8];
  chunk.unpack(x);
  const float r16 = fabsf(g.r16);
  uint32_t c[8];
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float2 d = __fadd2_rn(make_float2(x[i], x[i + 1]), make_float2(-g.z, -g.z));
    float2 y;
    asm("mul.rn.sat.f32 %0, %1, %2;" : "=f"(y.x) : "f"(d.x), "f"(r16));
    asm("mul.rn.sat.f32 %0, %1, %2;" : "=f"(y.y) : "f"(d.y), "f"(r16));
    const float2 m = __ffma2_rn(y, make_float2(16.0f, 16.0f), make_float2(12582912.0f, 12582912.0f));
    c[i] = __float_as_uint(m.x);
    c[i + 1] = __float_as_uint(m.y);
  }
  if (g.r16 < 0.0f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = min(c[i], kMagicBits + 15u);
  }
  uint32_t w = c[7];
#pragma unroll
  for (int i = 6; i >= 0; --i) w = w * 16u + c[i];
  return w - kMagicBits * 0x11111111u;
}

struct TokenParams {  // of a write (key, value: sources) or a read (destinations)
  Int4Pool pool;
  void *key, *value;
  int64_t k_seq, k_head, k_tok, v_seq, v_head, v_tok;
  int tokens;
  const int32_t *start, *counts;
  int8_t* bounds;
  int64_t bounds_page, bounds_head;  // bytes
  int32_t* status;
};

constexpr int kWriteThreads = 128;

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
  float r;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// The eight codes of a word times 2^-24, in the order n, n + 4, as floats: the
// halves of w & 0x000f000f are subnormal (16 times that in w & 0x00f000f0).
__device__ __forceinline__ void codes8(uint32_t w, float (&even)[4], float (&odd)[4]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t a = w & 0x000f000fu, b = w & 0x00f000f0u;
    even[2 * i] = half_lo(a);
    even[2 * i + 1] = half_hi(a);
    odd[2 * i] = half_lo(b);
    odd[2 * i + 1] = half_hi(b);
    w >>= 8;
  }
}
// RN(code * scale + min) of the eight channels of a word, in channel order.  The
// powers of two that the codes carry go into the scale, so every product is exact.
__device__ __forceinline__ void values8(uint32_t w, float s, float z, float (&v)[8]) {
  float even[4], odd[4];
  codes8(w, even, odd);
  const float s0 = s * 0x1p24f, s1 = s * 0x1p20f;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      v[2 * i + 4 * j] = __fmaf_rn(even[2 * i + j], s0, z);
      v[2 * i + 4 * j + 1] = __fmaf_rn(odd[2 * i + j], s1, z);
    }
}

// Channel bounds of a complete page's Key from its record in shared memory: the
// extremes of the stored values over the tokens, rounded outwards to whole steps
// of 2^e.  Every thread of the CTA calls it.
template <int D>
__device__ void write_bounds(const uint32_t* rec, int8_t* out) {
  constexpr int kCols = D / 8, kParts = kWriteThreads / kCols, kTok = kInt4Page / kParts;
  __shared__ float up_s[kParts][D + 4], low_s[kParts][D + 4];
  __shared__ float most_s[kWriteThreads / 32];
  const int col = threadIdx.x % kCols, part = threadIdx.x / kCols;
  const int t = col / (D / 32), G = col % (D / 32);
  float up[8], low[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    up[i] = -INFINITY;
    low[i] = INFINITY;
  }
#pragma unroll
  for (int i = 0; i < kTok; i += 2) {
    float v[2][8];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int k = part + (i + x) * kParts;
      uint32_t p = rec[8 * D + k * (D / 32) + G];
      if ((p & 0x7C00u) == 0x7C00u) p = 0;  // a group that holds no numbers counts as zeros
      values8(rec[k * kCols + col] & (p == 0 ? 0u : ~0u), half_lo(p), half_hi(p), v[x]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      up[i] = max3(up[i], v[0][i], v[1][i]);
      low[i] = min3(low[i], v[0][i], v[1][i]);
    }
  }
#pragma unroll
  for (int i = 0; i < 8; i += 4) {
    *reinterpret_cast<float4*>(&up_s[part][32 * G + 8 * t + i]) = make_float4(up[i], up[i + 1], up[i + 2], up[i + 3]);
    *reinterpret_cast<float4*>(&low_s[part][32 * G + 8 * t + i]) = make_float4(low[i], low[i + 1], low[i + 2], low[i + 3]);
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

// Word x (0 .. 20 D / 64 - 1) of token k in a record: Key codes, Key parameters,
// Value codes, Value parameters.
template <int D>
__device__ __forceinline__ int token_word(int k, int x) {
  constexpr int kC = D / 8, kP = D / 32;
  const int v = x >= kC + kP, y = x - v * (kC + kP);
  if (y >= kC) return v * 10 * D + 8 * D + k * kP + y - kC;
  if (v == 0) return k * kC + y;
  const int g = y / (D / 64), w = y % (D / 64);
  return 10 * D + (k >> 3) * D + g * kC + ((k & 7) >> 1) * kP + (k & 1) * (D / 64) + w;
}

// One CTA per (page, KV head), so that a page's bounds need no second launch; ten
// of them an SM hide each other's loads (eight and twelve measure the same).  Its tokens of the page, and the page's bounds once
// its last slot is written.
template <typename T, int D>
__global__ void __launch_bounds__(kWriteThreads, 10) int4_write_kernel(const __grid_constant__ TokenParams p) {
  constexpr int kLanes = D / 8, kRows = kWriteThreads / kLanes, kWords = 20 * D / kInt4Page;
  __shared__ __align__(16) uint32_t rec_s[20 * D];
  const int b = blockIdx.z, h = blockIdx.y, tid = threadIdx.x;
  grid_dep_wait();
  const int start = p.start[b];
  const int count = p.counts != nullptr ? min(p.counts[b], p.tokens) : p.tokens;
  if (count <= 0) return;
  if (start < 0 || start > INT32_MAX - count) {
    if (tid == 0 && p.status != nullptr) atomicExch(p.status, LF_ERR_OUT_OF_RANGE);
    return;
  }
  const int page = start / kInt4Page + blockIdx.x;
  const int64_t base = static_cast<int64_t>(page) * kInt4Page;
  if (base >= start + count) return;
  // slots of the page to write
  const int k0 = max(static_cast<int>(start - base), 0), k1 = static_cast<int>(min(start + count - base, int64_t{kInt4Page}));
  const int id = int4_page_id(p.pool, b, page);
  if (id < 0) {
    if (tid == 0 && p.status != nullptr) atomicExch(p.status, LF_ERR_OUT_OF_RANGE);
    return;
  }
  uint32_t* rec = reinterpret_cast<uint32_t*>(p.pool.words) + int4_record(p.pool, id, h);
  const bool whole = p.bounds != nullptr && k1 == kInt4Page;
  if (whole) {  // the slots written before, for the bounds
    for (int x = tid; x < k0 * (D / 8); x += kWriteThreads) rec_s[x] = __ldcg(rec + x);
    for (int x = tid; x < k0 * (D / 32); x += kWriteThreads) rec_s[8 * D + x] = __ldcg(rec + 8 * D + x);
  }

  // Row `row` of every kRows slots: the addresses step by constants.
  const int l = tid % kLanes, row = tid / kLanes;
  const int64_t from = base - start + row;  // source token of slot `row`
  const T* key = static_cast<const T*>(p.key) + b * p.k_seq + h * p.k_head + from * p.k_tok + 8 * l;
  const T* value = static_cast<const T*>(p.value) + b * p.v_seq + h * p.v_head + from * p.v_tok + 8 * l;
  const int64_t k_step = p.k_tok * kRows, v_step = p.v_tok * kRows;
  const int G = l >> 2, t = l & 3, u = G & 1;
  const bool odd = l & 1;
  uint32_t* kcode = rec_s + row * (D / 8) + t * (D / 32) + G;
  uint32_t* vcode = rec_s + 10 * D + (row >> 3) * D + (2 * t + u) * (D / 8) + ((row & 7) >> 1) * (D / 32) + (row & 1) * (D / 64) +
                    (G >> 1);
  uint32_t* param = rec_s + (odd ? 18 : 8) * D + row * (D / 32) + G;
#pragma unroll 2
  for (int it = 0; it < kInt4Page / kRows; ++it, key += k_step, value += v_step, kcode += kRows * (D / 8),
           vcode += kRows * (D / 8), param += kRows * (D / 32)) {
    const int k = it * kRows;
    if (k + kRows <= k0 || k >= k1) continue;  // whole warps stay together for the shuffles
    const bool live = k + row >= k0 && k + row < k1;
    Chunk<T> ck = {}, cv = {};
    if (live) {
      ck.load(key);
      cv.load(value);
    }
    // Even lanes form the Key group's parameters, odd ones the Value group's.
    float klo, khi, vlo, vhi;
    ck.extremes(klo, khi);
    cv.extremes(vlo, vhi);
    const GroupParams mine = group_params(odd ? vlo : klo, odd ? vhi : khi);
    GroupParams other;
    other.z = __shfl_xor_sync(0xffffffffu, mine.z, 1);
    other.r16 = __shfl_xor_sync(0xffffffffu, mine.r16, 1);
    const uint32_t kw = quantise8<T>(ck, odd ? other : mine);
    const uint32_t vw = quantise8<T>(cv, odd ? mine : other);
    // The lane's channels are 4 of chunk g = 2 t and 4 of g + 1; the lane of the
    // neighbouring group (u flipped) holds the other halves of both words.
    const uint32_t got = __shfl_xor_sync(0xffffffffu, u == 0 ? vw >> 16 : vw & 0xFFFFu, 4);
    if (live) {
      *kcode = kw;
      *vcode = u == 0 ? (vw & 0xFFFFu) | (got << 16) : got | (vw & 0xFFFF0000u);
      if (t < 2) *param = mine.word;
    }
  }
  __syncthreads();
  if (k1 - k0 == kInt4Page) {
#pragma unroll
    for (int x = tid; x < 5 * D; x += kWriteThreads)
      reinterpret_cast<uint4*>(rec)[x] = reinterpret_cast<const uint4*>(rec_s)[x];
  } else {
    for (int x = tid; x < (k1 - k0) * kWords; x += kWriteThreads) {
      const int at = token_word<D>(k0 + x / kWords, x % kWords);
      rec[at] = rec_s[at];
    }
  }
  if (whole) write_bounds<D>(rec_s, p.bounds + id * p.bounds_page + h * p.bounds_head);
}

// Token i is position start[b] + i, zero from counts[b] on.  One CTA per 64 tokens, which lie in two pages at most.
template <typename T, int D>
__global__ void __launch_bounds__(kWriteThreads) int4_read_kernel(const __grid_constant__ TokenParams p) {
  constexpr int kLanes = D / 8, kRows = kWriteThreads / kLanes;
  const int b = blockIdx.z, h = blockIdx.y;
  grid_dep_wait();
  const int start = p.start[b];
  const int count = p.counts != nullptr ? min(p.counts[b], p.tokens) : p.tokens;
  const int l = threadIdx.x % kLanes, row = threadIdx.x / kLanes;
  const int G = l >> 2, t = l & 3, u = G & 1, w = G >> 1;
  const int i0 = blockIdx.x * kInt4Page, last = min(i0 + kInt4Page, p.tokens);
  const int64_t pos0 = static_cast<int64_t>(start) + i0;
  const int k0 = static_cast<int>(pos0 & (kInt4Page - 1));  // slot of its page, rounded down
  auto record = [&](int x) -> const uint32_t* {  // of the first page, or of the one after
    const int64_t page = (pos0 - k0) / kInt4Page + x;  // negative for a position below 0
    const int id = page >= 0 && page < p.pool.table_width ? int4_page_id(p.pool, b, static_cast<int>(page)) : -1;
    return id < 0 ? nullptr : reinterpret_cast<const uint32_t*>(p.pool.words) + int4_record(p.pool, id, h);
  };
  const uint32_t *rec0 = record(0), *rec1 = record(1);
  T* key = static_cast<T*>(p.key) + b * p.k_seq + h * p.k_head + i0 * p.k_tok + 8 * l;
  T* value = static_cast<T*>(p.value) + b * p.v_seq + h * p.v_head + i0 * p.v_tok + 8 * l;
  constexpr int kAtOnce = 4;  // rows whose loads are in flight together (one: 38 us for the prompts above, four: 31.4)
  for (int r0 = row; r0 < last - i0; r0 += kAtOnce * kRows) {
    uint32_t kw[kAtOnce], kp[kAtOnce], vp[kAtOnce], v0[kAtOnce], v1[kAtOnce];
#pragma unroll
    for (int y = 0; y < kAtOnce; ++y) {
      const int i = r0 + y * kRows, k = k0 + i, s = k & (kInt4Page - 1);
      const uint32_t* rec = k < kInt4Page ? rec0 : rec1;
      const bool there = i < last - i0 && i0 + i < count;
      kw[y] = kp[y] = vp[y] = v0[y] = v1[y] = 0;
      if (there && rec != nullptr) {
        kw[y] = rec[s * (D / 8) + t * (D / 32) + G];
        kp[y] = rec[8 * D + s * (D / 32) + G];
        vp[y] = rec[18 * D + s * (D / 32) + G];
        const uint32_t* vc = rec + 10 * D + (s >> 3) * D + 2 * t * (D / 8) + ((s & 7) >> 1) * (D / 32) + (s & 1) * (D / 64) + w;
        v0[y] = vc[0];
        v1[y] = vc[D / 8];
      } else if (there && p.status != nullptr) {
        atomicExch(p.status, LF_ERR_OUT_OF_RANGE);
      }
    }
#pragma unroll
    for (int y = 0; y < kAtOnce; ++y) {
      const int i = r0 + y * kRows;
      float xk[8], xv[8];
      values8(kw[y], half_lo(kp[y]), half_hi(kp[y]), xk);
      values8(__byte_perm(v0[y], v1[y], u == 0 ? 0x5410 : 0x7632), half_lo(vp[y]), half_hi(vp[y]), xv);
      if (i < last - i0) {
        store8<T>(key + i * p.k_tok, xk);
        store8<T>(value + i * p.v_tok, xv);
      }
    }
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

template <typename P>
static int launch(const void* kern, const char* what, dim3 grid, P p, cudaStream_t stream) {
  void* args[] = {&p};
  const cudaError_t err = launch_programmatic(kern, grid, dim3(kWriteThreads), 0, stream, args);
  if (err != cudaSuccess) {
    set_error("%s: %s", what, cudaGetErrorString(err));
    return LF_ERR_LAUNCH;
  }
  return launch_status(what);
}
template <typename T> static const void* write_kernel(int D) {
  return D == 128 ? reinterpret_cast<const void*>(int4_write_kernel<T, 128>)
                  : reinterpret_cast<const void*>(int4_write_kernel<T, 64>);
}
template <typename T> static const void* read_kernel(int D) {
  return D == 128 ? reinterpret_cast<const void*>(int4_read_kernel<T, 128>)
                  : reinterpret_cast<const void*>(int4_read_kernel<T, 64>);
}

int check_int4_pool(const char* what, const lf_int4_pool& pool, int head_dim, Int4Pool& out) {
  LF_CHECK_ARG(pool.pages && pool.table, "%s: null pages or page table", what);
  LF_CHECK_SUPPORTED(head_dim == 64 || head_dim == 128, "%s: head_dim %d (64 or 128)", what, head_dim);
  LF_CHECK_ARG(pool.kv_heads > 0 && pool.batch > 0 && pool.n_pages > 0 && pool.table_width > 0,
               "%s: empty pool, batch or page table", what);
  LF_CHECK_SUPPORTED(pool.kv_heads <= 65535 && pool.batch <= 65535, "%s: %d KV heads, batch %d (65535 at most)", what,
                     pool.kv_heads, pool.batch);
  LF_CHECK_ARG((reinterpret_cast<uintptr_t>(pool.pages) & 15) == 0 && pool.page_stride % 4 == 0 &&
                   pool.head_stride % 4 == 0 && pool.head_stride >= 20 * head_dim &&
                   pool.page_stride >= 20 * head_dim && pool.table_stride >= pool.table_width,
               "%s: records must be 16-byte aligned and apart", what);
  LF_CHECK_SUPPORTED(pool.table_width <= INT32_MAX / kInt4Page, "%s: page table width %d", what, pool.table_width);
  out.words = pool.pages;
  out.page_stride = pool.page_stride;
  out.head_stride = pool.head_stride;
  out.table = pool.table;
  out.table_stride = pool.table_stride;
  out.table_width = pool.table_width;
  out.n_pages = pool.n_pages;
  out.kv_heads = pool.kv_heads;
  out.batch = pool.batch;
  return LF_OK;
}

// Checks shared by writes and reads.
static int check_tokens(const char* what, const lf_int4_tokens* a, TokenParams& p) {
  LF_CHECK_ARG(a != nullptr, "%s: null arguments", what);
  const int bad = check_int4_pool(what, a->pool, a->head_dim, p.pool);
  if (bad != LF_OK) return bad;
  LF_CHECK_ARG(a->tokens >= 0 && a->tokens <= (1 << 30), "%s: %d tokens", what, a->tokens);
  LF_CHECK_ARG(a->tokens == 0 || (a->key && a->value && a->start), "%s: null pointer", what);
  LF_CHECK_ARG(a->dtype == LF_F32 || a->dtype == LF_F16 || a->dtype == LF_BF16, "%s: dtype %d", what, a->dtype);
  const int64_t unit = a->dtype == LF_F32 ? 4 : 8;  // elements in 16 bytes
  LF_CHECK_ARG(((reinterpret_cast<uintptr_t>(a->key) | reinterpret_cast<uintptr_t>(a->value)) & 15) == 0 &&
                   (a->k_seq_stride | a->k_head_stride | a->k_tok_stride | a->v_seq_stride | a->v_head_stride |
                    a->v_tok_stride) % unit == 0,
               "%s: Key and Value rows must be 16-byte aligned", what);
  LF_CHECK_ARG(a->bounds == nullptr || (a->bounds_page_stride > 2 * a->head_dim && a->bounds_head_stride > 2 * a->head_dim),
               "%s: bounds records overlap", what);
  p.key = a->key;
  p.value = a->value;
  p.k_seq = a->k_seq_stride;
  p.k_head = a->k_head_stride;
  p.k_tok = a->k_tok_stride;
  p.v_seq = a->v_seq_stride;
  p.v_head = a->v_head_stride;
  p.v_tok = a->v_tok_stride;
  p.tokens = a->tokens;
  p.start = a->start;
  p.counts = a->counts;
  p.bounds = a->bounds;
  p.bounds_page = a->bounds_page_stride;
  p.bounds_head = a->bounds_head_stride;
  p.status = a->status;
  return LF_OK;
}

}  // namespace lf

extern "C" int lf_int4_write(const lf_int4_tokens* a, lf_stream_t stream) {
  lf::TokenParams p;
  const int bad = lf::check_tokens("lf_int4_write", a, p);
  if (bad != LF_OK || a->tokens == 0) return bad;
  // tokens that start anywhere in a page touch at most this many pages
  const dim3 grid((a->tokens + 2 * lf::kInt4Page - 2) / lf::kInt4Page, p.pool.kv_heads, p.pool.batch);
  const void* kern = a->dtype == LF_F32   ? lf::write_kernel<float>(a->head_dim)
                     : a->dtype == LF_F16 ? lf::write_kernel<__half>(a->head_dim)
                                          : lf::write_kernel<__nv_bfloat16>(a->head_dim);
  return lf::launch(kern, "lf_int4_write", grid, p, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int lf_int4_read(const lf_int4_tokens* a, lf_stream_t stream) {
  lf::TokenParams p;
  const int bad = lf::check_tokens("lf_int4_read", a, p);
  if (bad != LF_OK || a->tokens == 0) return bad;
  const dim3 grid((a->tokens + lf::kInt4Page - 1) / lf::kInt4Page, p.pool.kv_heads, p.pool.batch);
  const void* kern = a->dtype == LF_F32   ? lf::read_kernel<float>(a->head_dim)
                     : a->dtype == LF_F16 ? lf::read_kernel<__half>(a->head_dim)
                                          : lf::read_kernel<__nv_bfloat16>(a->head_dim);
  return lf::launch(kern, "lf_int4_read", grid, p, reinterpret_cast<cudaStream_t>(stream));
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
