// The 4-bit paged cache: record format and the pieces its kernels share.
//
// A page holds kInt4Page tokens.  The record of one (page, KV head) is 20 D
// int32 words (D = head_dim, 64 or 128):
//   [0, 8D)    Key codes: channel 32 G + 8 t + n of token k is nibble n of word
//              k * D/8 + t * D/32 + G
//   [8D, 10D)  Key parameters: word k * D/32 + G holds token k's scale (low
//              half) and minimum (high half), fp16, of channels 32 G .. 32 G + 31
//   [10D, 18D) Value codes: channel 64 w + 32 u + 4 g + n of token 8 b + 2 t + o
//              is nibble 4 u + n of word b * D + g * D/8 + t * D/32 + o * D/64 + w
//   [18D, 20D) Value parameters, as the Key's
// Both code orders are those of m16n8k16 fragments: lane 4 g + t of a warp that
// multiplies 8 or 16 tokens loads its codes as one 16-byte piece (8 bytes at D
// 64) and the warp's pieces lie side by side, so the loads are conflict-free in
// shared memory and whole sectors in HBM.
//
// A value is stored as code * scale + minimum, rounded once to fp32.
#pragma once

#include "lf_common.cuh"

namespace lf {

constexpr int kInt4Page = 64;    // tokens per page
constexpr int kInt4Group = 32;   // channels that share a scale and a minimum
constexpr int kBoundsMinExp = -40;

// A pool of records and the page table that orders it into sequences.
struct Int4Pool {
  int32_t* words;
  int64_t page_stride, head_stride;  // words
  const int32_t* table;              // [batch][table_width] page ids
  int64_t table_stride;
  int table_width, n_pages, kv_heads, batch;
};

// Pool page of logical page `page` of sequence b, or -1 where the table or the
// page id is out of range.
__device__ __forceinline__ int int4_page_id(const Int4Pool& p, int b, int page) {
  if (page < 0 || page >= p.table_width) return -1;
  const int id = p.table[b * p.table_stride + page];
  return id < p.n_pages ? id : -1;
}
__device__ __forceinline__ int64_t int4_record(const Int4Pool& p, int id, int h) {
  return id * p.page_stride + h * p.head_stride;
}

// Tokens that query token i of a sequence sees (count: its query tokens).
__device__ __forceinline__ int int4_seen(int length, int count, int i) {
  return i < count ? max(0, length - count + 1 + i) : 0;
}

__device__ __forceinline__ float half_lo(uint32_t w) { return half_bits_to_float(static_cast<uint16_t>(w)); }
__device__ __forceinline__ float half_hi(uint32_t w) { return half_bits_to_float(static_cast<uint16_t>(w >> 16)); }

// The smallest e >= kBoundsMinExp with most <= 127 * 2^e, for most >= 0 and finite.
__device__ __forceinline__ int exponent127(float most) {
  if (!(most > 0.0f)) return kBoundsMinExp;
  const uint32_t bits = __float_as_uint(most);
  const int exp = static_cast<int>(bits >> 23);
  if (exp == 0) {  // below the normal range: most < 2^-126
    int x;
    const float f = frexpf(most, &x);
    return max(f <= 127.0f / 128.0f ? x - 7 : x - 6, kBoundsMinExp);
  }
  // most = f * 2^x with x = exp - 126 and f in [1/2, 1); f <= 127/128 by its mantissa bits
  const int x = exp - 126;
  return max((bits & 0x7FFFFFu) <= 0x7E0000u ? x - 7 : x - 6, kBoundsMinExp);
}
// 2^e for e in [-126, 127].
__device__ __forceinline__ float pow2(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Checks the C ABI's pool and copies it for a kernel (lf_int4_write.cu).
int check_int4_pool(const char* what, const lf_int4_pool& pool, int head_dim, Int4Pool& out);
// lf_int4_select's checks alone, and the call itself for the queries times sign (1 or
// -1) (lf_int4_select.cu).
int check_int4_select(const lf_int4_query* a);
int int4_select_pages(const lf_int4_query* a, float sign, cudaStream_t stream);

}  // namespace lf
