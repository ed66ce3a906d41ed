// Tensor-core attention over 16-bit operands: what its kernels share on top of
// lf_tcgen05.cuh.  Tiles are 128 rows of 64-channel halves in the 128-byte swizzle: row
// r of a half is the 128 bytes at 128 r, its 16-byte chunk c at chunk c ^ (r % 8).
#pragma once

#include <cuda.h>

#include <type_traits>

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
// 16 columns, waited for.
__device__ __forceinline__ void tmem_ld_x16(uint32_t taddr, float* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]), "=f"(r[10]),
        "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]));
}
// A warpgroup's registers per thread from here on; the sum over the block may not pass what
// it was launched with, or the raise would wait
// for good (launched_with).
template <int N> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

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

// How the waits of a CTA end before their time, in its shared memory.
struct Waits {
  uint64_t moved;  // when a role was last seen at work that others wait for, however long it takes (globaltimer)
  int stop;        // one gave up
};
// Wait of a whole warp for a barrier's phase, with a limit: false once a wait of this CTA
// has given up, for all lanes alike.  The clock is read once in 1024 tries.  kMoves: the limit
// is on a time in which nothing moves; work that may take longer (prompt_row's) writes
// Waits::moved.  (The other kernel does without: looked at there too, it took 283 us for a
// chunk in place of 272.)
constexpr uint64_t kTileWaitNs = 2000000000ull;
template <bool kMoves>
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile Waits* waits, uint64_t limit_ns = kTileWaitNs) {
  bool ok = mbar_try_wait(bar, parity);
  uint64_t since = 0;
  for (uint32_t n = 1; !ok; ++n) {
    ok = mbar_try_wait(bar, parity);
    if ((n & 1023u) == 0u && !ok) {
      const uint64_t now = globaltimer_ns();
      if (since == 0) since = now;
      if (waits->stop != 0 || (now - since > limit_ns && (!kMoves || static_cast<int64_t>(now - waits->moved) > static_cast<int64_t>(limit_ns)))) {
        waits->stop = 1;
        break;
      }
    }
  }
  return __all_sync(0xffffffffu, ok);
}

// Products of one tile (128 rows), issued by one lane of the calling warp.
// Scores: queries times Keys, D channels of 128 rows each in shared memory (+=: to what is
// there).  `full`, if given, completes with them, and so with everything that this warp
// issued before.
template <int D>
__device__ __forceinline__ void issue_scores(uint32_t tmem_s, uint32_t queries, uint32_t keys, uint32_t idesc, bool add, uint64_t* full) {
  if (elect_one()) {
    const uint64_t a = swizzled_desc(queries), b = swizzled_desc(keys);
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      const uint32_t off = (k >> 2) * (kHalfBytes >> 4) + (k & 3) * 2;
      mma_16_ss(tmem_s, a + off, b + off, idesc, add || k > 0);
    }
    if (full != nullptr) mma_commit(full);
  }
  __syncwarp();
}
// Outputs: weights (in the scores' place, kTerms numbers each) times Values, keys 64 half +
// 32 part .. of both halves.  done: as full, or null.
template <int kTerms>
__device__ __forceinline__ void issue_outputs(uint32_t tmem_o, uint32_t tmem_p, uint32_t values, uint32_t idesc, int part, bool fresh, uint64_t* done) {
  if (elect_one()) {
    const uint64_t v = swizzled_desc(values);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = 4 * (i >> 1) + 2 * part + (i & 1);
#pragma unroll
      for (int x = 0; x < kTerms; ++x)
        mma_16_ts(tmem_o, tmem_p + 64 * x + 8 * k, v + k * (16 * 128 >> 4), idesc, !fresh || part + i + x > 0);
    }
    if (done != nullptr) mma_commit(done);
  }
  __syncwarp();
}
__device__ __forceinline__ void arrive_once(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// The softmax of one 128 x 128 tile of scores by 8 warps: two threads to a row (TMEM lane =
// row), 64 columns each.  One thread to a row has its 128 exponentials in a chain that
// the tensor core waits for: 3500 cycles a step of two tiles, against 2048 of its own;
// four warps to a scheduler also cover one another's latencies.  Weights stand at
// 2^kLift for the running maximum.  It is moved only where a score passes it by 2^kSlack,
// so most tiles skip the rescaling of the output.
constexpr float kSlack = 8.0f;
template <typename T> constexpr float kLift = 0.0f;
// fp16 ends at steps of 2^-24: with the largest weight at 2^7, what is lost of a small
// weight is 2^-32 of it at most (and 2^(7 + 8) still fits).
template <> constexpr float kLift<__half> = 7.0f;

struct RowState {
  float top;   // running maximum of the scores times c, -inf before any
  float sum;   // of the weights; NaN once a score was NaN or +inf
  bool large;  // a maximum was so large that the rounding of its product with c reaches the exponent
  __device__ __forceinline__ bool empty() const { return top == -INFINITY && sum == sum; }  // nothing above -inf was seen
};
__device__ __forceinline__ RowState no_scores() { return RowState{-INFINITY, 0.0f, false}; }
constexpr float kLargeTop = 1024.0f;  // 2^-14 of an exponent is lost from here on

__device__ __forceinline__ float max_nan2(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// What the two threads of a row tell one another: a number each, by way of shared memory
// and a barrier that all 8 warps of the tile arrive at.
struct Pair {
  float* mine;
  const float* other;
  uint64_t* met;
  uint32_t phase;
  template <typename Wait>
  __device__ __forceinline__ bool meet(Wait&& wait) {
    arrive_once(met);
    return wait(met, phase++ & 1);
  }
  // The next exchange may begin once the other thread has read this one's number: after
  // another meeting, or a barrier that it arrives at later.  (The next step's scores are
  // such a barrier, and the last step's outputs: both come behind the weights of all 8 warps,
  // which each hands over behind its read.)
  template <typename Wait>
  __device__ __forceinline__ bool exchange(float x, float& y, Wait&& wait) {
    *const_cast<volatile float*>(mine) = x;
    if (!meet(wait)) return false;
    y = *const_cast<const volatile float*>(other);
    return true;
  }
};

// This thread's 64 scores, of which the first `seen` are visible (masked: whether that is to
// be looked at).  Returns their largest (NaN where one is).
__device__ __forceinline__ float row_scores(uint32_t tmem_s, float (&s)[64], bool masked, int seen) {
#pragma unroll
  for (int i = 0; i < 2; ++i) tmem_ld_x32(tmem_s + 32 * i, s + 32 * i);
  tmem_wait_ld();
#pragma unroll
  for (int i = 0; i < 2; ++i) tmem_settle(s + 32 * i);
  if (masked) {
#pragma unroll
    for (int i = 0; i < 64; ++i) s[i] = i < seen ? s[i] : -INFINITY;
  }
  float most[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) most[k] = s[k];
#pragma unroll
  for (int i = 4; i < 60; i += 8)
#pragma unroll
    for (int k = 0; k < 4; ++k) most[k] = max3_nan(most[k], s[i + k], s[i + k + 4]);
#pragma unroll
  for (int k = 0; k < 4; ++k) most[k] = max_nan2(most[k], s[60 + k]);
  return max3_nan(max_nan2(most[0], most[1]), most[2], most[3]);
}

// The row's maximum moved by its tile's largest score (c > 0).  Returns the factor that
// the output so far has to be multiplied by (1 mostly).
__device__ __forceinline__ float move_top(float most, float c, RowState& st) {
  const float now = most * c;
  float fix = 1.0f;
  if (now > st.top + kSlack) {  // (the first score of a row always: top is -inf)
    fix = ex2(st.top - now);
    st.top = now;
    st.sum *= fix;
    st.large |= fabsf(now) >= kLargeTop && now < INFINITY;
  }
  if (!(now < INFINITY)) st.sum = NAN;  // a score that is NaN or +inf makes the row's result NaN
  return fix;
}
// 2^x for x >= -126 without the special function unit: x = n + r with |r| <= 1/2 (the
// nearest whole number by adding 1.5 * 2^23), 2^r by its minimax polynomial (relative
// error; found with Remez' algorithm), n added to the exponent.  Within 7.5e-5 (degree 3)
// and 2.7e-6 (degree 4): below a weight's own rounding to bf16 (2^-9) and fp16 (2^-12).
template <int kDegree>
__device__ __forceinline__ float2 exp2_poly(float2 x) {
  const float2 magic = make_float2(12582912.0f, 12582912.0f);
  x.x = fmaxf(x.x, -126.0f);
  x.y = fmaxf(x.y, -126.0f);
  const float2 n = __fadd2_rn(x, magic);
  const float2 whole = __fadd2_rn(n, make_float2(-12582912.0f, -12582912.0f));
  const float2 r = __ffma2_rn(whole, make_float2(-1.0f, -1.0f), x);
  auto step = [&](float2 y, float k) { return __ffma2_rn(y, r, make_float2(k, k)); };
  float2 y;
  if constexpr (kDegree == 3) {
    y = step(make_float2(0.05517166906f, 0.05517166906f), 0.2426111222f);
    y = step(step(y, 0.6932609855f), 0.9999280735f);
  } else {
    static_assert(kDegree == 4, "polynomials of degree 3 and 4");
    y = step(make_float2(0.009570101912f, 0.009570101912f), 0.05591786032f);
    y = step(step(step(y, 0.2402474483f), 0.6931218147f), 0.9999992614f);
  }
  return make_float2(__uint_as_float(__float_as_uint(y.x) + (__float_as_uint(n.x) << 23)),
                     __uint_as_float(__float_as_uint(y.y) + (__float_as_uint(n.y) << 23)));
}

// Weights of 32 scores, stored in T at 16 columns, and with kTerms 2 what T's rounding left
// of them 64 columns on.  kPoly of every 8 pairs go by the polynomial: the special function
// unit gives 16 results a cycle, as long as the tensor core takes for both products of them.
template <typename T, int kPoly, int kTerms>
__device__ __forceinline__ void row_weights(uint32_t tmem_p, const float* s, float c, RowState& st) {
  // The product of maximum and c is rounded once, and taken as it is everywhere: it cancels
  // in the quotient of output and sum.  (Rows of RowState::large are done again elsewhere.)
  const float base = kLift<T> - (st.top == -INFINITY ? 0.0f : st.top);
  float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
  for (int part = 0; part < kTerms; ++part) {  // (two terms: 8 columns at a time, for registers)
    uint32_t w[16 / kTerms], low[8];
#pragma unroll
    for (int i = 0; i < 16 / kTerms; ++i) {
      const int at = 16 * part / kTerms + i;
      const float2 x = __ffma2_rn(make_float2(s[2 * at], s[2 * at + 1]), make_float2(c, c), make_float2(base, base));
      const float2 e = at % 8 < kPoly ? exp2_poly<std::is_same<T, __half>::value ? 4 : 3>(x) : make_float2(ex2(x.x), ex2(x.y));
      sum[i & 1] = __fadd2_rn(sum[i & 1], e);
      w[i] = pack_two<T>(e.x, e.y);
      if constexpr (kTerms == 2) {
        const float2 r = __fadd2_rn(e, make_float2(-half_bits_to_float(w[i] & 0xFFFFu), -half_bits_to_float(w[i] >> 16)));
        low[i] = pack_two<T>(r.x, r.y);
      }
    }
    if constexpr (kTerms == 1) {
      tmem_st_x16(tmem_p, w);
    } else {
      tmem_st_x8(tmem_p + 8 * part, w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7]);
      tmem_st_x8(tmem_p + 64 + 8 * part, low[0], low[1], low[2], low[3], low[4], low[5], low[6], low[7]);
    }
  }
  st.sum += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
}

// kN columns of the output rows so far times their factors.
template <int kN>
__device__ __forceinline__ void rescale(uint32_t tmem_o, float fix) {
#pragma unroll
  for (int i = 0; i < kN / 16; ++i) {
    float o[16];
    tmem_ld_x16(tmem_o + 16 * i, o);
    uint32_t w[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) w[k] = __float_as_uint(o[k] * fix);
    tmem_st_x16(tmem_o + 16 * i, w);
  }
}

// A thread's part of a tile: columns 64 half .. of its row's scores to weights (which take
// the first 64 columns' place, two to a column), first 32 columns, then 32: the output
// product over these may begin when `early`, then `ready` has 8 warps' arrivals.
// fresh: the row's first tile.  (The output product before is done: it was issued before
// these scores, whose barrier the caller has seen.)
// wait(barrier, parity) is false once a limit ran out, and so is the result then.
// on_masked() is called on a masked tile before its first weights are handed over.
template <typename T, int D, int kPoly, int kTerms, typename Wait, typename Masked>
__device__ __forceinline__ bool soften_tile(uint32_t tmem_s, uint32_t tmem_o, int half, float c, bool masked, int seen, bool fresh,
                                            RowState& st, Pair& pair, uint64_t* early, uint64_t* ready, Wait&& wait, Masked&& on_masked) {
  float s[64], other;
  const float most = row_scores(tmem_s + 64 * half, s, masked, seen - 64 * half);
  if (!pair.exchange(most, other, wait)) return false;
  const float fix = move_top(max_nan2(most, other), c, st);
  if (masked && !on_masked()) return false;
  if (!fresh && __any_sync(0xffffffffu, fix != 1.0f)) rescale<D / 2>(tmem_o + D / 2 * half, fix);
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    if (masked)  // a masked score's weight is 0, not 2^-126
      row_weights<T, 0, kTerms>(tmem_s + 32 * half + 16 * part, s + 32 * part, c, st);
    else
      row_weights<T, kPoly, kTerms>(tmem_s + 32 * half + 16 * part, s + 32 * part, c, st);
    tmem_wait_st();
    tc_fence_before();
    arrive_once(part == 0 ? early : ready);
  }
  return true;
}

// The row's sum, of both its threads': called once the row's outputs are done, which keeps it
// behind the last step's exchange.  (The next exchange may follow at once.)
template <typename Wait>
__device__ __forceinline__ bool join_sums(RowState& st, Pair& pair, Wait&& wait) {
  float other;
  if (!pair.exchange(st.sum, other, wait)) return false;
  st.sum += other;
  return pair.meet(wait);
}

}  // namespace sm100
}  // namespace lf
