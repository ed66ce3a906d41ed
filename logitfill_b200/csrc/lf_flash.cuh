// Tensor-core attention over 16-bit operands: what its kernels share on top of
// lf_tcgen05.cuh.  Tiles are 128 rows of 64-channel halves in the 128-byte swizzle: row
// r of a half is the 128 bytes at 128 r, its 16-byte chunk c at chunk c ^ (r % 8).
#pragma once

#include <cuda.h>

#include "lf_common.cuh"
#include "lf_tcgen05.cuh"

namespace lf {
namespace sm100 {

constexpr int kHalfBytes = 128 * 128;  // one half of a tile

// Shared-memory matrix descriptor in the 128-byte swizzle (the tile 1024-byte aligned).
// K-major operands: the next 8 rows 1024 bytes on (the leading offset is not used).
// MN-major operands: the next 8 k 1024 bytes on, the next 64 channels a half on.
__device__ __forceinline__ uint64_t swizzled_desc(uint32_t smem_addr) {
  uint64_t d = static_cast<uint64_t>((smem_addr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>(kHalfBytes >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}
// Instruction descriptor, kind::f16: A and B both fp16 or both bf16, fp32 accumulator.
__host__ __device__ constexpr uint32_t idesc_16(bool bf16, int M, int N, bool b_mn_major, bool negate_a) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((negate_a ? 1u : 0u) << 13) |
         ((b_mn_major ? 1u : 0u) << 16) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}
// D[tmem] (+)= A[smem] * B[smem]
__device__ __forceinline__ void mma_16_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem]
__device__ __forceinline__ void mma_16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 32 consecutive columns of this thread's lane; the registers hold them after a
// tmem_wait_ld and a tmem_settle of each.
__device__ __forceinline__ void tmem_ld_x32(uint32_t taddr, float* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, "
      "%22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
        "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]),
        "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]),
        "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
      : "r"(taddr));
}
// Keeps uses of 32 loaded registers behind the wait.
__device__ __forceinline__ void tmem_settle(float* r) {
  asm volatile("" : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]),
    "+f"(r[7]), "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]),
    "+f"(r[15]), "+f"(r[16]), "+f"(r[17]), "+f"(r[18]), "+f"(r[19]), "+f"(r[20]), "+f"(r[21]), "+f"(r[22]),
    "+f"(r[23]), "+f"(r[24]), "+f"(r[25]), "+f"(r[26]), "+f"(r[27]), "+f"(r[28]), "+f"(r[29]), "+f"(r[30]),
    "+f"(r[31]));
}
__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, "
      "%22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]));
}

// Two numbers rounded to T, the first in the low half.
template <typename T> __device__ __forceinline__ uint32_t pack_two(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack_two<__half>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <> __device__ __forceinline__ uint32_t pack_two<__nv_bfloat16>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// A box of a 4-D tensor map into shared memory, completing on bar.
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// Wait of a whole warp for a barrier's phase, with a limit: false once a wait of this CTA
// has given up (*stop), for all lanes alike.
constexpr uint64_t kTileWaitNs = 2000000000ull;
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* stop) {
  bool ok = mbar_try_wait(bar, parity);
  if (!ok) {
    const uint64_t t0 = globaltimer_ns();
    for (uint32_t n = 1; !ok; ++n) {
      ok = mbar_try_wait(bar, parity);
      if (!ok && (n & 63u) == 0u && (*stop != 0 || globaltimer_ns() - t0 > kTileWaitNs)) break;
    }
    if (!ok) *stop = 1;
  }
  return __all_sync(0xffffffffu, ok);
}

// The softmax of one 128 x 128 tile of scores, row by row (a thread to a row, TMEM lane =
// row).  Weights stand at 2^kLift for the running maximum.  It is moved only where a
// score passes it by 2^kSlack, so most tiles skip the rescaling of the output.
constexpr float kSlack = 8.0f;
template <typename T> constexpr float kLift = 0.0f;
// fp16 ends at steps of 2^-24: with the largest weight at 2^7, what is lost of a small
// weight is 2^-32 of it at most (and 2^(7 + 8) still fits).
template <> constexpr float kLift<__half> = 7.0f;

struct RowState {
  float top;  // running maximum times c, -inf before any score
  float sum;  // of the weights
};

// Scores of the row's 128 columns, of which the first `seen` are visible (masked: whether
// that is to be looked at), from s to weights in T at the same TMEM columns.  c > 0.
// Returns the factor that the output so far has to be multiplied by (1 mostly).
template <typename T>
__device__ __forceinline__ float soften(uint32_t tmem_s, float c, bool masked, int seen, RowState& st) {
  float s[128];
#pragma unroll
  for (int i = 0; i < 4; ++i) tmem_ld_x32(tmem_s + 32 * i, s + 32 * i);
  tmem_wait_ld();
#pragma unroll
  for (int i = 0; i < 4; ++i) tmem_settle(s + 32 * i);
  if (masked) {
#pragma unroll
    for (int i = 0; i < 128; ++i) s[i] = i < seen ? s[i] : -INFINITY;
  }
  float most[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) most[k] = fmaxf(s[k], s[k + 4]);
#pragma unroll
  for (int i = 8; i < 128; i += 8)
#pragma unroll
    for (int k = 0; k < 4; ++k) most[k] = fmaxf(fmaxf(most[k], s[i + k]), s[i + k + 4]);
  const float now = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * c;
  float fix = 1.0f;
  if (now > st.top + kSlack) {  // (the first score of a row always: top is -inf)
    fix = ex2(st.top - now);
    st.top = now;
    st.sum *= fix;
  }
  // The product of maximum and c is rounded once, and taken as it is everywhere: it
  // cancels in the quotient of output and sum.
  const float base = kLift<T> - (st.top == -INFINITY ? 0.0f : st.top);
  float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    uint32_t w[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const float2 x = __ffma2_rn(make_float2(s[64 * part + 2 * i], s[64 * part + 2 * i + 1]), make_float2(c, c), make_float2(base, base));
      const float2 e = make_float2(ex2(x.x), ex2(x.y));
      sum[i & 1] = __fadd2_rn(sum[i & 1], e);
      w[i] = pack_two<T>(e.x, e.y);
    }
    tmem_st_x32(tmem_s + 32 * part, w);
  }
  st.sum += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
  return fix;
}

// The output rows so far times their factors.
template <int D>
__device__ __forceinline__ void rescale(uint32_t tmem_o, float fix) {
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    float o[32];
    tmem_ld_x32(tmem_o + 32 * i, o);
    tmem_wait_ld();
    tmem_settle(o);
    uint32_t w[32];
#pragma unroll
    for (int k = 0; k < 32; ++k) w[k] = __float_as_uint(o[k] * fix);
    tmem_st_x32(tmem_o + 32 * i, w);
  }
}

}  // namespace sm100
}  // namespace lf
