// Attention over the 4-bit paged cache for sequences that share their first pages
// (lf_int4_attend_prefix).
//
// Mathematics.  The shared tokens' part of a row's softmax (maximum, sum, accumulators)
// is the same sum whether the row's sequence holds the pages or another does.  So the
// queries of all sequences of a group are the rows of one product with the shared Keys,
// one with the shared Values, and what lf_int4_attend would have read for every sequence
// is read and unpacked once for 256 rows.  Three kernels:
//   plan     the groups' members, and the line of all Key tiles of all units (256 rows of a
//            KV head of a group), cut into equal ranges, one per CTA;
//   prefix   the shared pages: every (unit, range) leaves a record of maxima, sums and
//            accumulators;
//   suffix   lf_int4_attend's kernel from the shared pages' end on, whose last step adds
//            the unit's records (lf_int4_attend.cu).
//
// The product runs on tcgen05 with fp16 operands.  Codes become fp16 numbers code * s + z,
// rounded once (2^-11); the queries of a row are scaled by a power of two, so that bf16 and
// fp16 enter exactly.  With an fp16 output, whose own rounding is as fine, Keys and weights
// enter as sums of two fp16 numbers, in two products: error against 64 bits 0.00053 of the
// result with one number each (0.0002 is the output's rounding alone), 0.00031 with two for
// the Keys, 0.00028 with two for both.  Numbers that may pass the fp16 range (a scale of 2^11
// or a minimum of 2^15 at least), a NaN, a page that is not in the pool, or scores too
// large for the exponent are not done here: the group of sequences is marked, and its
// members read these pages themselves, in the suffix kernel, which can do that.
//
// Order of channels.  A word's nibbles n and n + 4 lie in one fp16 pair (w >> 4 n) &
// 0x000f000f.  For Key, a sum over channels has no order: Keys and queries both take the
// channels of a group of 8 as (0, 4), (1, 5), (2, 6), (3, 7).  For Value, the two are
// channels 32 apart; the accumulators' columns come in the codes' order, and the record is
// written in the channels'.
//
// Roles of the prefix kernel (28 warps, one CTA an SM): 16 softmax warps and one for the
// products, as in lf_prompt.cu; one copies pages (cp.async.bulk, Keys and Values apart, the
// ids of 32 pages at a time); 8 unpack them into swizzled fp16 tiles, K-major for Key and
// MN-major for Value, 16 bytes a store without bank conflicts; one looks for parameters out
// of range.
//
// What bounds it.  A chunk of 512 tokens behind 32768, 28 heads on 4, D 128, bf16: 281 us,
// 864 TFLOP/s, 51 % of the measured 1680 (replayed; 272 to 288 by the GPU; back to back 297).  A step takes 2.35 us
// with 256 rows (1.2 of products), 1.98 with 128 and 1.86 with 32: with one tile the chain of
// scores, softmax and outputs is not hidden, with two it is in part.  Unpacking is behind it:
// half of it left out took 2.27 and 1.97.  (fp16 outputs: 4.6 and 3.5; with each term of a Key
// unpacked in a pass of its own 5.4 and 4.1; D 64: 2.6 and 2.4, was 3.1 and 2.3.)  64 sequences
// behind 16384 tokens, 40 heads on 8: 76 us (under the profiler: plan 6, prefix 56, suffix and
// merge 27); 320 rows to a KV head fill a unit of 256 and a quarter of another.  The chunk
// took 424 us with four warps unpacking and three tiles in the ring, 342 with eight warps, 285
// with four tiles.
#include <cmath>
#include <type_traits>

#include "lf_flash.cuh"
#include "lf_int4.cuh"

namespace lf {

using namespace sm100;

struct PrefixParams {
  Int4Pool pool;
  const void* q;
  int64_t q_seq, q_head, q_tok;
  int q_len, heads;               // query heads of a KV head
  const int32_t *lengths, *counts, *group, *shared;
  int groups, grid, head_dim, fp16, always;
  float scale_log2;
  int32_t* status;
  PrefixPlan plan;
};

// -------------------------------------------------------------------- plan

constexpr int kMaxGroups = 4096;

// Whether the shared pages are read once, or by each sequence as lf_int4_attend does, is a
// matter of sizes.  In ns on a B200: a page costs lf_int4_attend's kernel about 2 for up to 8
// query columns and 2.9 for 16 (D 128; half at D 64), every time it is read; a Key tile of a
// unit costs 16 here, 23 with the two terms of fp16 (D 64: 11 and 16), and the two kernels
// more and the records 17000 (D 64: 12500).  Measured in us, that kernel / these three,
// replayed.  28 heads on 4, D 128, bf16, one token each: 8192 shared tokens, 16 sequences
// 25 / 30, 32 sequences 41 / 37; 32768 tokens, 4 sequences 28 / 37, 8: 41 / 39, 16: 69 / 41,
// 32: 127 / 54.  40 heads on 8: 8192 tokens, 8 sequences 25 / 28, 16: 41 / 29; 32768 tokens, 4
// sequences 41 / 48, 8: 69 / 48; fp16, 8: 75 / 69, 16: 140 / 72.  One sequence behind 32768
// tokens, 28 heads on 4, bf16: 8 query tokens 37 / 45, 16: 50 / 48, 32: 85 / 56, 128: 298 / 124.
__host__ __device__ __forceinline__ int64_t visit_ns(int64_t pages, int columns, int head_dim) {
  return pages * ((columns + 15) / 16) * (columns <= 8 ? 20 : 29) * head_dim / 1280;
}
__host__ __device__ __forceinline__ int tile_ns(int head_dim, bool fp16) { return head_dim == 128 ? (fp16 ? 23 : 16) : (fp16 ? 16 : 11); }
__host__ __device__ __forceinline__ int64_t fixed_ns(int head_dim) { return head_dim == 128 ? 17000 : 12500; }

// Shared pages of group g that its `count` members (one of them `any`) have.
__device__ __forceinline__ int group_pages(const PrefixParams& p, int g, int count, int any) {
  if (count == 0) return 0;
  // All pages of one member are its own: the complete ones (what a page's unwritten slots
  // hold may not be read here) are read in this way, its queries' own tokens among them.
  if (count == 1) return p.q_len * p.heads <= 16 ? 0 : min(max(p.lengths[any], 0) / kInt4Page, p.pool.table_width);
  return min(max(p.shared[g], 0), p.pool.table_width);
}
// What a group's shared pages take in the line, and what reading them once saves.
struct GroupCost { int tiles, steps, places; int64_t saved; };
__device__ __forceinline__ GroupCost group_cost(const PrefixParams& p, int pages, int count) {
  GroupCost c;
  const int rows = count * p.q_len * p.heads;
  c.tiles = pages > 0 ? (rows + kPrefixRows - 1) / kPrefixRows : 0;
  c.steps = (pages + 1) / 2;
  c.places = c.tiles * p.pool.kv_heads * (c.steps + kPrefixCost);
  c.saved = visit_ns(static_cast<int64_t>(pages) * count * p.pool.kv_heads, p.q_len * p.heads, p.head_dim) -
            static_cast<int64_t>(c.places) * tile_ns(p.head_dim, p.fp16);
  return c;
}

__global__ void __launch_bounds__(32) int4_prefix_plan_kernel(const __grid_constant__ PrefixParams p) {
  __shared__ int count_s[kMaxGroups], first_s[kMaxGroups], any_s[kMaxGroups];
  const int lane = threadIdx.x;
  grid_dep_trigger();  // the prefix kernel's CTAs may start: they wait for this one before they read
  grid_dep_wait();
  for (int g = lane; g < p.groups; g += 32) count_s[g] = 0;
  __syncwarp();
  // Each sequence's rank among its group's.
  for (int b0 = 0; b0 < p.pool.batch; b0 += 32) {
    const int b = b0 + lane;
    int g = b < p.pool.batch ? p.group[b] : -1;
    if (g >= p.groups) g = -1;
    if (g < 0) g = -1;
    const uint32_t same = __match_any_sync(0xffffffffu, g);
    const int before = __popc(same & ((1u << lane) - 1u));
    const int rank = g >= 0 ? count_s[g] + before : -1;
    __syncwarp();
    if (g >= 0 && before == 0) {
      count_s[g] += __popc(same);
      any_s[g] = b;
    }
    __syncwarp();
    if (b < p.pool.batch) p.plan.seqs[b] = PrefixSeq{g, rank};
  }
  // Whether it pays in all.
  int64_t saved = 0;
  for (int g = lane; g < p.groups; g += 32) {
    const int count = count_s[g], pages = group_pages(p, g, count, any_s[g]);
    saved += max(static_cast<int64_t>(0), group_cost(p, pages, count).saved);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) saved += __shfl_xor_sync(0xffffffffu, saved, o);
  const bool pays = p.always || saved > fixed_ns(p.head_dim);
  // The groups' places in the lists and in the line.
  int members = 0, units = 0, places = 0;
  for (int g0 = 0; g0 < p.groups; g0 += 32) {
    const int g = g0 + lane;
    const int count = g < p.groups ? count_s[g] : 0;
    int pages = pays && g < p.groups ? group_pages(p, g, count, any_s[g]) : 0;
    if (!p.always && group_cost(p, pages, count).saved <= 0) pages = 0;
    const GroupCost cost = group_cost(p, pages, count);
    const int tiles = cost.tiles, steps = cost.steps, n_units = tiles * p.pool.kv_heads, n_places = cost.places;
    int m = count, u = n_units, x = n_places;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, m, o), b = __shfl_up_sync(0xffffffffu, u, o), c = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) {
        m += a;
        u += b;
        x += c;
      }
    }
    if (g < p.groups) {
      first_s[g] = members + m - count;
      p.plan.groups[g] = PrefixGroup{pages, pages > 0, members + m - count, count, units + u - n_units, places + x - n_places, tiles, steps};
    }
    members += __shfl_sync(0xffffffffu, m, 31);
    units += __shfl_sync(0xffffffffu, u, 31);
    places += __shfl_sync(0xffffffffu, x, 31);
  }
  __syncwarp();
  for (int b = lane; b < p.pool.batch; b += 32) {
    const PrefixSeq s = p.plan.seqs[b];  // (this lane's own store)
    if (s.group >= 0) p.plan.members[first_s[s.group] + s.rank] = b;
  }
  if (lane == 0) {
    p.plan.head[0] = places;
    p.plan.head[1] = max(1, (places + p.grid - 1) / p.grid);
  }
}

// ------------------------------------------------------------ shared pages

template <int D> struct PrefixCfg {
  static constexpr int kTile = 128 * D * 2;        // bytes of 128 fp16 rows
  static constexpr int kSlots = D == 128 ? 4 : 8;  // Key and Value tiles
  static constexpr int kRaw = 40 * D;              // bytes of a page's Keys or Values: codes, then parameters
  static constexpr int kStages = D == 128 ? 3 : 8;  // two pages' Keys or Values, as they are in the pool
  static constexpr int kSmem = 2 * kTile + kSlots * kTile + kStages * 2 * kRaw + 3072;  // with what the roles share
  static constexpr int kO = 256;                   // TMEM columns: scores of both tiles, then outputs
};
constexpr int kPrefixThreads = 896;
// Registers a thread: 72 at launch, then split by what the warpgroups hold: 64 scores of a
// row, a few words and their parameters, counters.
constexpr int kPrefixLaunchRegs = 72, kRowRegs = 88, kUnpackRegs = 56, kOtherRegs = 32;
constexpr int kUnpackWarps = 8;
static_assert(512 * kRowRegs + 32 * kUnpackWarps * kUnpackRegs + 128 * kOtherRegs <= kPrefixThreads * kPrefixLaunchRegs,
              "more registers than the block has");
constexpr int kUnpackWarp = 16, kProductWarp = kUnpackWarp + kUnpackWarps, kCopyWarp = kProductWarp + 1, kCheckWarp = kProductWarp + 2;
constexpr float kNoScore = -3e38f;  // the maximum of a row that sees nothing: below any score

struct PrefixShared {
  uint64_t raw_full[8], raw_empty[8], kv_full[8], kv_empty[8], q_ready[2], s_full[2], p_early[2], p_ready[2], met[2], o_done[2], last;
  Waits waits;
  uint32_t tmem;
  alignas(128) float told[2][2][128];  // between the two threads of a row
};

// Steps of one unit that this CTA has.
struct Piece { int g, h, tile, first, n, unit; };
// The pieces of a CTA's range, in order; every lane of a warp calls it.
struct Walk {
  const PrefixPlan& plan;
  int kv_heads, groups, at, end, g0;
  PrefixGroup group;
  int g;
  __device__ __forceinline__ Walk(const PrefixPlan& plan, int kv_heads, int groups) : plan(plan), kv_heads(kv_heads), groups(groups), g0(0), g(-1) {
    const int per = plan.head[1];
    at = blockIdx.x * per;
    end = min(plan.head[0], at + per);
    group = PrefixGroup{};
  }
  __device__ __forceinline__ int group_end(const PrefixGroup& y) const {
    return y.places + y.tiles * kv_heads * (y.steps + kPrefixCost);
  }
  __device__ __forceinline__ bool next(Piece& piece) {
    while (at < end) {
      while (g < 0 || at >= group_end(group)) {
        const int x = g0 + (threadIdx.x & 31);
        const uint32_t any = __ballot_sync(0xffffffffu, x < groups && at < group_end(plan.groups[min(x, groups - 1)]));
        if (any != 0) {
          g = g0 + __ffs(any) - 1;
          group = plan.groups[g];
        } else {
          g0 += 32;
          if (g0 >= groups) return false;
        }
      }
      const int span = group.steps + kPrefixCost, x = (at - group.places) / span, start = group.start(x);
      const int first = max(at, start) - start, stop = min(end - start, group.steps);
      at = min(end, start + group.steps);
      if (first >= stop) continue;
      piece = Piece{g, x / group.tiles, x % group.tiles, first, stop - first, group.units + x};
      return true;
    }
    return false;
  }
};

// fp16 numbers that make up a Key, and a weight.
template <typename T> constexpr int kTerms = std::is_same<T, __half>::value ? 2 : 1;

__device__ __forceinline__ uint32_t hfma2_rn(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
__device__ __forceinline__ uint32_t hadd2_rn(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t hsub2_rn(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t hmul2_rn(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// A word's eight codes as fp16 pairs: codes (0, 4), (1, 5), (2, 6), (3, 7).
__device__ __forceinline__ void codes_of(uint32_t w, uint32_t (&c)[4]) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const uint32_t x = w >> (8 * k);
    const uint32_t even = (x & 0x000F000Fu) | 0x64006400u, odd = (x & 0x00F000F0u) | 0x64006400u;  // 1024 + code, 1024 + 16 code
    c[2 * k] = hsub2_rn(even, 0x64006400u);
    c[2 * k + 1] = hfma2_rn(odd, 0x2C002C00u, 0xD400D400u);  // / 16 - 64
  }
}
// code * s2 + z2, rounded once.
__device__ __forceinline__ uint4 unpack_word(uint32_t w, uint32_t s2, uint32_t z2) {
  uint32_t c[4];
  codes_of(w, c);
  return make_uint4(hfma2_rn(c[0], s2, z2), hfma2_rn(c[1], s2, z2), hfma2_rn(c[2], s2, z2), hfma2_rn(c[3], s2, z2));
}
// The same as the sum of two fp16 numbers.  x = RN(code s) and r = code s - x, exact by an
// fma; a = RN(x + z) and what it leaves out, exact by Knuth's two-sum; the second number is
// that and r, rounded.
__device__ __forceinline__ void unpack_word_exactly(uint32_t w, uint32_t s2, uint32_t z2, uint4& high, uint4& low) {
  uint32_t c[4], y[4], e[4];
  codes_of(w, c);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t x = hmul2_rn(c[k], s2), r = hfma2_rn(c[k], s2, x ^ 0x80008000u);
    y[k] = hadd2_rn(x, z2);
    const uint32_t b = hsub2_rn(y[k], x);
    e[k] = hadd2_rn(hadd2_rn(hsub2_rn(x, hsub2_rn(y[k], b)), hsub2_rn(z2, b)), r);
  }
  high = make_uint4(y[0], y[1], y[2], y[3]);
  low = make_uint4(e[0], e[1], e[2], e[3]);
}
// Non-zero in a sign's place where a scale is 2^11 at least, a minimum 2^15, or one is not finite.
__device__ __forceinline__ uint32_t wide_bits(uint32_t sz) { return (sz & 0x7FFF7FFFu) + 0x08001800u; }

template <int kN> __device__ __forceinline__ void words_of(const uint8_t* at, uint32_t (&w)[kN]) {
  if constexpr (kN == 4) {
    const uint4 x = *reinterpret_cast<const uint4*>(at);
    w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
  } else {
    const uint2 x = *reinterpret_cast<const uint2*>(at);
    w[0] = x.x; w[1] = x.y;
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kPrefixThreads, 1) int4_prefix_kernel(const __grid_constant__ PrefixParams p) {
  using C = PrefixCfg<D>;
  constexpr int kSlots = C::kSlots, kStages = C::kStages, kG = D / kInt4Group;
  constexpr int kLoads = kTerms<T> + 1;  // tiles of a step: the Key's terms, then Value
  extern __shared__ __align__(1024) uint8_t dynamic[];
  uint8_t* queries = dynamic;
  uint8_t* ring = queries + 2 * C::kTile;
  uint8_t* raw = ring + kSlots * C::kTile;
  PrefixShared& sh = *reinterpret_cast<PrefixShared*>(raw + kStages * 2 * C::kRaw);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  if (warp == kProductWarp) {
    tmem_alloc(&sh.tmem, 512);
    tmem_relinquish();
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&sh.kv_full[i], kUnpackWarps);
      mbar_init(&sh.kv_empty[i], 1);
    }
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&sh.raw_full[i], 1);
      mbar_init(&sh.raw_empty[i], kUnpackWarps + 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&sh.q_ready[t], 8);
      mbar_init(&sh.s_full[t], 1);
      mbar_init(&sh.p_early[t], 8);
      mbar_init(&sh.p_ready[t], 8);
      mbar_init(&sh.met[t], 8);
      mbar_init(&sh.o_done[t], 1);
    }
    mbar_init(&sh.last, 1);
    sh.waits.stop = 0;
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *const_cast<volatile uint32_t*>(&sh.tmem), 0);
  grid_dep_trigger();  // all CTAs of this grid run at once, so the suffix kernel's take nothing that one needs
  grid_dep_wait();

  auto wait = [&](uint64_t* bar, uint32_t parity) { return warp_wait<false>(bar, parity, &sh.waits); };
  const int per_member = p.q_len * p.heads;

  if (warp == kCopyWarp) {
    // ---------------------------------------------------------------- copies of pages
    fewer_registers<kOtherRegs>();
    Walk walk(p.plan, p.pool.kv_heads, p.groups);
    Piece piece;
    uint32_t n = 0;
    bool ok = true;
    while (ok && walk.next(piece)) {
      const int pages = walk.group.pages, leader = p.plan.members[walk.group.members];
      const int32_t* words = p.pool.words + piece.h * p.pool.head_stride;
      int ids = 0;
      for (int i = 0; i < piece.n; ++i) {
        const int page = 2 * (piece.first + i), two = page + 1 < pages ? 2 : 1;
        if ((i & 15) == 0) {  // the ids of 32 pages, one a lane
          ids = page + lane < pages ? int4_page_id(p.pool, leader, page + lane) : 0;
          if (ids < 0) {
            p.plan.groups[piece.g].live = 0;  // its members look for themselves
            ids = 0;
          }
        }
        const int id0 = __shfl_sync(0xffffffffu, ids, 2 * (i & 15)), id1 = __shfl_sync(0xffffffffu, ids, 2 * (i & 15) + 1);
        for (int value = 0; ok && value < 2; ++value, ++n) {
          const int stage = n % kStages;
          if (n >= kStages && !(ok = wait(&sh.raw_empty[stage], (n / kStages - 1) & 1))) break;
          if (elect_one()) {
            const int32_t* from = words + value * 10 * D;
            mbar_arrive_expect_tx(&sh.raw_full[stage], two * C::kRaw);
            bulk_g2s(raw + stage * 2 * C::kRaw, from + id0 * p.pool.page_stride, C::kRaw, &sh.raw_full[stage]);
            if (two == 2) bulk_g2s(raw + (2 * stage + 1) * C::kRaw, from + id1 * p.pool.page_stride, C::kRaw, &sh.raw_full[stage]);
          }
          __syncwarp();
        }
        if (!ok) break;
      }
    }
    for (int i = 0; i < kStages; ++i) {  // no copy outlives the CTA
      const uint32_t used = n / kStages + (static_cast<uint32_t>(i) < n % kStages ? 1 : 0);
      if (used != 0) mbar_wait_bounded(&sh.raw_full[i], (used - 1) & 1, kTileWaitNs);
    }
  } else if (warp >= kUnpackWarp && warp < kUnpackWarp + kUnpackWarps) {
    // ---------------------------------------------------------------- pages to fp16 tiles
    fewer_registers<kUnpackRegs>();
    Walk walk(p.plan, p.pool.kv_heads, p.groups);
    Piece piece;
    uint32_t n = 0;
    bool ok = true;
    const int w = warp - kUnpackWarp;
    while (ok && walk.next(piece)) {
      const int pages = walk.group.pages;
      for (int i = 0; ok && i < piece.n; ++i, ++n) {
        const int page = 2 * (piece.first + i);
#pragma unroll 1
        for (int value = 0; value < 2; ++value) {  // the Key's terms, then Value
          const uint32_t load = kLoads * n + (value ? kLoads - 1 : 0), slot = load % kSlots, unit = 2 * n + value, stage = unit % kStages;
          const uint32_t next = (load + 1) % kSlots;  // of a Key's second term
          if (!(ok = wait(&sh.raw_full[stage], (unit / kStages) & 1))) break;
          if (load >= kSlots && !(ok = wait(&sh.kv_empty[slot], (load / kSlots - 1) & 1))) break;
          if (kLoads == 3 && !value && load + 1 >= kSlots && !(ok = wait(&sh.kv_empty[next], ((load + 1) / kSlots - 1) & 1))) break;
          uint8_t *tile = ring + slot * C::kTile, *second = ring + next * C::kTile;
#pragma unroll
          for (int part = 0; part < 16 / kUnpackWarps; ++part) {
            // 8 tokens of a page at a time
            const int block = part * kUnpackWarps + w, half = block >> 3, b = block & 7;  // half: which page; b: its 8 tokens
            const uint8_t* rec = raw + (2 * stage + half) * C::kRaw;
            const bool there = page + half < pages;
            if (!value) {
              // Key: lane = (token, t), its kG words the groups' channels 8 t .. 8 t + 7.  Tokens x and
              // x + 4 in a quarter of the warp store to different banks.
              const int t = lane & 3, tok = 8 * b + ((lane >> 2) & 1) * 4 + (lane >> 3), row = half * 64 + tok;
              uint32_t code[kG], sz[kG];
              words_of<kG>(rec + (tok * (D / 8) + t * kG) * 4, code);
              words_of<kG>(rec + 32 * D + tok * kG * 4, sz);
#pragma unroll
              for (int G = 0; G < kG; ++G) {
                const uint32_t s2 = __byte_perm(sz[G], 0, 0x1010), z2 = __byte_perm(sz[G], 0, 0x3232);
                uint4 x = make_uint4(0, 0, 0, 0), y = x;
                if (there) {
                  if constexpr (kLoads == 2)
                    x = unpack_word(code[G], s2, z2);
                  else
                    unpack_word_exactly(code[G], s2, z2, x, y);
                }
                const int at = (G >> 1) * kHalfBytes + row * 128 + (((4 * (G & 1) + t) ^ (row & 7)) << 4);
                *reinterpret_cast<uint4*>(tile + at) = x;
                if constexpr (kLoads == 3) *reinterpret_cast<uint4*>(second + at) = y;
              }
            } else {
              // Value: lane = (g, t), its words [token 2 t + o][w]: channels 64 w + 32 u + 4 g + n.
              const int t = lane & 3, g = lane >> 2;
              uint32_t code[kG], sz[2][kG];
              words_of<kG>(rec + (b * D + g * (D / 8) + t * kG) * 4, code);
              words_of<kG>(rec + 32 * D + (8 * b + 2 * t) * kG * 4, sz[0]);
              words_of<kG>(rec + 32 * D + (8 * b + 2 * t + 1) * kG * 4, sz[1]);
#pragma unroll
              for (int o = 0; o < 2; ++o)
#pragma unroll
                for (int x = 0; x < kG / 2; ++x) {
                  const uint32_t a = sz[o][2 * x], c = sz[o][2 * x + 1];
                  const uint32_t s2 = __byte_perm(a, c, 0x5410), z2 = __byte_perm(a, c, 0x7632);
                  const int row = half * 64 + 8 * b + 2 * t + o;
                  const uint4 y = there ? unpack_word(code[o * (kG / 2) + x], s2, z2) : make_uint4(0, 0, 0, 0);
                  *reinterpret_cast<uint4*>(tile + x * kHalfBytes + row * 128 + ((g ^ (row & 7)) << 4)) = y;
                }
            }
          }
          fence_proxy_async_smem();
          arrive_once(&sh.kv_full[slot]);
          if (kLoads == 3 && !value) arrive_once(&sh.kv_full[next]);
          arrive_once(&sh.raw_empty[stage]);
        }
      }
    }
  } else if (warp == kCheckWarp) {
    // ---------------------------------------------------------------- parameters out of fp16's range
    fewer_registers<kOtherRegs>();
    Walk walk(p.plan, p.pool.kv_heads, p.groups);
    Piece piece;
    uint32_t n = 0;
    bool ok = true;
    while (ok && walk.next(piece)) {
      uint32_t wide = 0;
      for (int i = 0; ok && i < 2 * piece.n; ++i, ++n) {
        const int stage = n % kStages, two = 2 * (piece.first + i / 2) + 1 < walk.group.pages ? 2 : 1;
        if (!(ok = wait(&sh.raw_full[stage], (n / kStages) & 1))) break;
        for (int half = 0; half < two; ++half) {
          const uint4* at = reinterpret_cast<const uint4*>(raw + (2 * stage + half) * C::kRaw + 32 * D) + lane;
#pragma unroll
          for (int x = 0; x < D / 64; ++x) {
            const uint4 y = at[32 * x];
            wide |= wide_bits(y.x) | wide_bits(y.y) | wide_bits(y.z) | wide_bits(y.w);
          }
        }
        arrive_once(&sh.raw_empty[stage]);
      }
      if ((wide & 0x80008000u) != 0) p.plan.groups[piece.g].live = 0;
    }
  } else if (warp == kProductWarp) {
    // ---------------------------------------------------------------- products
    fewer_registers<kOtherRegs>();
    // As prompt attention's: scores of step s after the outputs of step s - 1, tile by tile.
    Walk walk(p.plan, p.pool.kv_heads, p.groups);
    Piece piece;
    const uint32_t idesc_s = idesc_16(false, 128, 128, false, false), idesc_o = idesc_16(false, 128, D, true, false);
    const uint32_t ring_a = smem_u32(ring);
    uint32_t step = 0, made[2] = {0, 0}, asked[2] = {0, 0};
    bool had[2] = {false, false}, fresh = false, ends = false, ok = true;
    auto output = [&](int t) -> bool {  // of the step before
      if (!had[t]) return true;
      const uint32_t load = kLoads * step - 1, slot = load % kSlots;
      if (!wait(&sh.kv_full[slot], (load / kSlots) & 1)) return false;
      for (int part = 0; part < 2; ++part) {
        if (!wait(part == 0 ? &sh.p_early[t] : &sh.p_ready[t], made[t] & 1)) return false;
        tc_fence_after();
        issue_outputs<kTerms<T>>(tmem + C::kO + t * D, tmem + 128 * t, ring_a + slot * C::kTile, idesc_o, part, fresh, ends && part == 1 ? &sh.o_done[t] : nullptr);
      }
      ++made[t];
      return true;
    };
    auto keys_there = [&]() -> bool {
      for (uint32_t load = kLoads * step; load < kLoads * step + kLoads - 1; ++load)
        if (!wait(&sh.kv_full[load % kSlots], (load / kSlots) & 1)) return false;
      return true;
    };
    auto scores = [&](int t) {
      tc_fence_after();
#pragma unroll
      for (int x = 0; x < kLoads - 1; ++x)
        issue_scores<D>(tmem + 128 * t, smem_u32(queries) + t * C::kTile, ring_a + (kLoads * step + x) % kSlots * C::kTile, idesc_s, x > 0,
                        x == kLoads - 2 ? &sh.s_full[t] : nullptr);
    };
    while (ok && walk.next(piece)) {
      const bool two = piece.tile * kPrefixRows + 128 < walk.group.count * per_member;
      for (int i = 0; i < piece.n; ++i, ++step) {
        if (i == 0) {  // (new queries are made only after the outputs of the piece before)
          if (step > 0 && !(ok = output(0) && output(1))) break;
          if (!(ok = keys_there() && wait(&sh.q_ready[0], asked[0]++ & 1))) break;
          scores(0);
          if (two && !(ok = wait(&sh.q_ready[1], asked[1]++ & 1))) break;
          if (two) scores(1);
        } else {
          if (!(ok = keys_there())) break;
          if (!(ok = output(0))) break;
          scores(0);
          if (!(ok = output(1))) break;
          if (two) scores(1);
        }
        had[0] = true;
        had[1] = two;
        fresh = i == 0;
        ends = i == piece.n - 1;
      }
    }
    if (ok && step > 0 && *const_cast<volatile int*>(&sh.waits.stop) == 0 && output(0)) output(1);  // the last step's
  } else if (warp < kUnpackWarp) {
    // ---------------------------------------------------------------- softmax, one tile a warpgroup
    more_registers<kRowRegs>();
    const int t = warp >> 3, half = (warp >> 2) & 1, r = (warp & 3) * 32 + lane;
    const uint32_t mine = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16), tm_s = mine + 128 * t, tm_o = mine + C::kO + t * D;
    Pair pair = {&sh.told[t][half][r], &sh.told[t][half ^ 1][r], &sh.met[t], 0};
    Walk walk(p.plan, p.pool.kv_heads, p.groups);
    Piece piece;
    uint32_t count = 0, pieces = 0, steps = 0;
    const bool frees = (warp & 7) == 0;
    bool ok = true;
    while (ok && walk.next(piece)) {
      const int row = piece.tile * kPrefixRows + t * 128 + r, rows = walk.group.count * per_member;
      const uint32_t before = steps;  // of the CTA
      steps += piece.n;
      if (piece.tile * kPrefixRows + t * 128 >= rows) continue;
      // ---- the row's query, as fp16 at a power of two: each thread half of its channels
      float c = 1e-36f;
      int vis = walk.group.pages * kInt4Page;
      {
        uint4 x[D / 16];
        float most = 0.0f, other;
        if (row < rows) {
          const int m = row / per_member, in = row - m * per_member, i = in / p.heads, b = p.plan.members[walk.group.members + m];
          const T* q = static_cast<const T*>(p.q) + b * p.q_seq + (piece.h * p.heads + in - i * p.heads) * p.q_head + i * p.q_tok + D / 2 * half;
          vis = min(vis, int4_seen(p.lengths[b], p.counts != nullptr ? p.counts[b] : p.q_len, i));
#pragma unroll
          for (int k = 0; k < D / 16; ++k) x[k] = *reinterpret_cast<const uint4*>(q + 8 * k);
        } else {
#pragma unroll
          for (int k = 0; k < D / 16; ++k) x[k] = make_uint4(0, 0, 0, 0);
        }
        auto number = [&](uint32_t v, bool high) {
          if constexpr (std::is_same<T, __half>::value) return high ? half_hi(v) : half_lo(v);
          return __uint_as_float(high ? v & 0xFFFF0000u : v << 16);
        };
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t v[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
#pragma unroll
          for (int y = 0; y < 4; ++y) most = fmaxf(most, fmaxf(fabsf(number(v[y], false)), fabsf(number(v[y], true))));
        }
        if (!(ok = pair.exchange(most, other, wait))) break;
        most = fmaxf(most, other);
        // 2^kq brings the largest magnitude to [2^13, 2^14), or as near as 2^126 does
        const int kq = most > 0.0f && most < INFINITY ? min(126, 13 - (static_cast<int>(__float_as_uint(most) >> 23) - 127)) : 0;
        const float up = p.scale_log2 < 0.0f ? -pow2(kq) : pow2(kq);
        c = fmaxf(pow2(-kq) * fabsf(p.scale_log2), 1e-36f);  // positive, so that a masked score's -inf stays one
        uint8_t* tile = queries + t * C::kTile + r * 128;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t v[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
          float f[8];
#pragma unroll
          for (int y = 0; y < 8; ++y) f[y] = number(v[y >> 1], y & 1) * up;
          const uint4 w = make_uint4(pack_two<__half>(f[0], f[4]), pack_two<__half>(f[1], f[5]), pack_two<__half>(f[2], f[6]),
                                     pack_two<__half>(f[3], f[7]));
          const int chunk = D / 16 * half + k;
          *reinterpret_cast<uint4*>(tile + (chunk >> 3) * kHalfBytes + (((chunk & 7) ^ (r & 7)) << 4)) = w;
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.q_ready[t]);
      const int vis_min = __reduce_min_sync(0xffffffffu, vis);
      // ---- its steps
      RowState st = no_scores();
      for (int i = 0; i < piece.n; ++i, ++count) {
        const int at = (piece.first + i) * 128;
        if (!(ok = wait(&sh.s_full[t], count & 1))) break;
        tc_fence_after();
        if (frees && (t == 1 || rows - piece.tile * kPrefixRows <= 128)) {
          // The step's last scores are done, and with them all products before: the Key tile
          // is free, and the Value tile of the step before.
          const uint32_t load = kLoads * (before + i);
#pragma unroll
          for (int x = 0; x < kLoads - 1; ++x) arrive_once(&sh.kv_empty[(load + x) % kSlots]);
          if (load > 0) arrive_once(&sh.kv_empty[(load - 1) % kSlots]);
        }
        if (!(ok = soften_tile<__half, D, 0, kTerms<T>>(tm_s, tm_o, half, c, at + 128 > vis_min, vis - at, i == 0, st, pair, &sh.p_early[t], &sh.p_ready[t],
                                          wait, [] { return true; })))
          break;
      }
      if (__any_sync(0xffffffffu, st.large && row < rows) && lane == 0) p.plan.groups[piece.g].live = 0;
      if (!ok || !(ok = wait(&sh.o_done[t], pieces++ & 1))) break;
      if (!(ok = join_sums(st, pair, wait))) break;
      tc_fence_after();
      // ---- its record
      float* rec = p.plan.records + (piece.unit + static_cast<int64_t>(blockIdx.x)) * prefix_record(D);
      const int in = t * 128 + r;
      float* acc = rec + 2 * kPrefixRows + static_cast<int64_t>(in) * D;
      if (row < rows && half == 0) {
        rec[in] = st.top == -INFINITY ? kNoScore : fmaxf(st.top, kNoScore);
        rec[kPrefixRows + in] = st.empty() ? 0.0f : st.sum;
      }
#pragma unroll
      for (int y = 0; y < D / 64; ++y) {
        const int x = D / 64 * half + y;
        float o[32];
        tmem_ld_x32(tm_o + 32 * x, o);
        tmem_wait_ld();
        tmem_settle(o);
        if (row < rows) {
          // column 64 w + 8 g + 2 n + u is channel 64 w + 32 u + 4 g + n
#pragma unroll
          for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int u = 0; u < 2; ++u)
              *reinterpret_cast<float4*>(acc + 64 * (x >> 1) + 32 * u + 4 * (4 * (x & 1) + g)) =
                  make_float4(o[8 * g + u], o[8 * g + 2 + u], o[8 * g + 4 + u], o[8 * g + 6 + u]);
        }
      }
      tc_fence_before();
    }
  } else {
    fewer_registers<kOtherRegs>();  // (of a warpgroup, all warps at once)
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kProductWarp) {
    tc_fence_after();
    if (sh.waits.stop != 0) {  // a wait gave up, of any role: products may be in flight, and end before their operands go
      if (elect_one()) mma_commit(&sh.last);
      __syncwarp();
      mbar_wait_bounded(&sh.last, 0, kTileWaitNs);
    }
    tmem_dealloc(tmem, 512);
  }
  if (threadIdx.x == 0 && sh.waits.stop != 0 && p.status != nullptr) atomicExch(p.status, LF_ERR_DEVICE_TIMEOUT);
}

// ------------------------------------------------------------------- host

// Bytes of the plan's lists.
static size_t plan_bytes(int batch, int groups) {
  return (16 + static_cast<size_t>(groups) * sizeof(PrefixGroup) + static_cast<size_t>(batch) * (sizeof(PrefixSeq) + 4) + 255) / 256 * 256;
}
// The fewest members of a group whose pages are read once (plan kernel: group_pages, group_cost).
// Where sizes decide, n members save something only where n visits of P pages take longer than
// the steps of one unit at least, of which there are more than P / 2:
// n A D / 1280 > tile_ns / 2, with visit_ns' factor A.  So records are few where queries are
// many: a row of records for each of 1024 sequences that might share would be 1 GB for 8 KV
// heads, D 128; by this rule it is 0.2.
static int64_t least_members(int64_t columns, int head_dim, bool fp16, bool always) {
  const int64_t least = columns <= 16 ? 2 : 1;
  if (always) return least;
  const int64_t a = (columns + 15) / 16 * (columns <= 8 ? 20 : 29), n = 640 * tile_ns(head_dim, fp16) / (a * head_dim) + 1;
  return n > least ? n : least;
}
// Records that there can be: one of each unit and CTA that meet, no more than units and CTAs.
static int64_t most_units(int64_t batch, int64_t kv_heads, int64_t columns, int64_t groups, int64_t least) {
  const int64_t most_groups = batch / least;  // that read pages once
  return most_groups == 0 ? 0 : (batch * columns / kPrefixRows + (groups < most_groups ? groups : most_groups)) * kv_heads;
}
static size_t prefix_bytes(int64_t batch, int64_t groups, int64_t units, int head_dim) {
  return plan_bytes(static_cast<int>(batch), static_cast<int>(groups)) +
         static_cast<size_t>(units + sm_count()) * prefix_record(head_dim) * 4;
}
// Units that a call may have; 0 where each sequence reads its pages itself, whatever the groups are.
static int64_t call_units(const lf_int4_prefix& a) {
  const lf_int4_query& q = a.query;
  if (a.groups <= 0 || a.groups > kMaxGroups || q.pool.kv_heads <= 0 || q.pool.batch <= 0 || q.q_len <= 0 || q.n_q < q.pool.kv_heads || q.head_dim <= 0)
    return 0;
  const int64_t columns = static_cast<int64_t>(q.q_len) * (q.n_q / q.pool.kv_heads);
  if (columns * q.pool.batch > (1 << 30)) return 0;  // (refused)
  const bool small =
      visit_ns(static_cast<int64_t>(q.pool.batch) * q.pool.kv_heads * q.pool.table_width, static_cast<int>(columns), q.head_dim) <= fixed_ns(q.head_dim);
  if (small && !a.always) return 0;
  return most_units(q.pool.batch, q.pool.kv_heads, columns, a.groups, least_members(columns, q.head_dim, q.dtype == LF_F16, a.always != 0));
}

template <typename T>
static const void* prefix_kernel_of(int head_dim) {
  return head_dim == 128 ? reinterpret_cast<const void*>(int4_prefix_kernel<T, 128>) : reinterpret_cast<const void*>(int4_prefix_kernel<T, 64>);
}

}  // namespace lf

extern "C" size_t lf_int4_prefix_workspace_bytes(int batch, int kv_heads, int n_q, int q_len, int head_dim, int groups) {
  if (batch <= 0 || kv_heads <= 0 || n_q < kv_heads || q_len <= 0 || head_dim <= 0 || groups < 0) return 0;
  const int64_t columns = static_cast<int64_t>(q_len) * (n_q / kv_heads);
  return lf::prefix_bytes(batch, groups, lf::most_units(batch, kv_heads, columns, groups, lf::least_members(columns, head_dim, false, true)), head_dim);
}

extern "C" size_t lf_int4_prefix_workspace_need(const lf_int4_prefix* a) {
  if (a == nullptr) return 0;
  const int64_t units = lf::call_units(*a);
  return units == 0 ? 0 : lf::prefix_bytes(a->query.pool.batch, a->groups, units, a->query.head_dim);
}

extern "C" int lf_int4_attend_prefix(const lf_int4_prefix* a, lf_stream_t stream) {
  using namespace lf;
  LF_CHECK_ARG(a != nullptr, "lf_int4_attend_prefix: null arguments");
  const lf_int4_query& q = a->query;
  LF_CHECK_ARG(q.picked == nullptr, "lf_int4_attend_prefix: pages were picked");
  const int bad = check_int4_attend(&q);
  if (bad != LF_OK) return bad;
  LF_CHECK_ARG(a->groups >= 0 && (a->groups == 0 || (a->group && a->shared)), "lf_int4_attend_prefix: null pointer");
  LF_CHECK_SUPPORTED(a->groups <= kMaxGroups, "lf_int4_attend_prefix: %d groups (%d at most)", a->groups, kMaxGroups);
  const int64_t units = call_units(*a);
  if (units == 0) return lf_int4_attend(&q, stream);
  PrefixParams p;
  const int ok = check_int4_pool("lf_int4_attend_prefix", q.pool, q.head_dim, p.pool);
  if (ok != LF_OK) return ok;
  p.q = q.q;
  p.q_seq = q.q_seq_stride;
  p.q_head = q.q_head_stride;
  p.q_tok = q.q_tok_stride;
  p.q_len = q.q_len;
  p.heads = q.n_q / p.pool.kv_heads;
  p.lengths = q.lengths;
  p.counts = q.counts;
  p.group = a->group;
  p.shared = a->shared;
  p.groups = a->groups;
  p.head_dim = q.head_dim;
  p.fp16 = q.dtype == LF_F16;
  p.always = a->always;
  p.scale_log2 = q.scaling * 1.4426950408889634f;
  p.status = q.status;
  const int sms = sm_count();
  const int64_t records = units + sms;
  const int64_t steps = (p.pool.table_width + 1) / 2 + kPrefixCost;
  LF_CHECK_SUPPORTED(records <= (1 << 30) / steps && static_cast<int64_t>(p.pool.batch) * p.q_len * p.heads <= (1 << 30),
                     "lf_int4_attend_prefix: %d sequences of %d pages are too many for one call", p.pool.batch, p.pool.table_width);
  LF_CHECK_ARG(a->workspace && (reinterpret_cast<uintptr_t>(a->workspace) & 15) == 0 &&
                   a->workspace_bytes >= prefix_bytes(p.pool.batch, p.groups, units, q.head_dim),
               "lf_int4_attend_prefix: workspace of %zu bytes is missing, misaligned or too small", a->workspace_bytes);
  uint8_t* at = static_cast<uint8_t*>(a->workspace);
  p.plan.head = reinterpret_cast<int*>(at);
  p.plan.groups = reinterpret_cast<PrefixGroup*>(at + 16);
  p.plan.seqs = reinterpret_cast<PrefixSeq*>(p.plan.groups + p.groups);
  p.plan.members = reinterpret_cast<int*>(p.plan.seqs + p.pool.batch);
  p.plan.records = reinterpret_cast<float*>(at + plan_bytes(p.pool.batch, p.groups));
  const int64_t most_steps = units * steps;
  p.grid = static_cast<int>(most_steps < sms ? most_steps : sms);

  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const void* kern = q.dtype == LF_F16 ? prefix_kernel_of<__half>(q.head_dim) : prefix_kernel_of<__nv_bfloat16>(q.head_dim);
  const int smem = q.head_dim == 128 ? PrefixCfg<128>::kSmem : PrefixCfg<64>::kSmem;
  cudaError_t err = raise_smem_limit(kern, smem, true);
  if (!launched_with(kern, kPrefixLaunchRegs)) {
    set_error("lf_int4_attend_prefix: the kernel was not built for %d registers a thread", kPrefixLaunchRegs);
    return LF_ERR_LAUNCH;
  }
  void* args[] = {&p};
  if (err == cudaSuccess)
    err = launch_programmatic(reinterpret_cast<const void*>(int4_prefix_plan_kernel), dim3(1), dim3(32), 0, s, args);
  if (err == cudaSuccess) err = launch_programmatic(kern, dim3(p.grid), dim3(kPrefixThreads), smem, s, args);
  if (err != cudaSuccess) {
    set_error("lf_int4_attend_prefix: %s", cudaGetErrorString(err));
    return LF_ERR_LAUNCH;
  }
  return int4_attend_suffix(&q, p.plan, s);
}
