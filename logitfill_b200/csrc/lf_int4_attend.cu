// Attention over the 4-bit paged cache (lf_int4_attend): dense over a
// sequence's pages, or over a list of picked ones.
//
// Mathematics.  A unit is one KV head of one sequence (of one query token in a
// sparse call) with up to 8 NT query columns (q-head, query token).  With codes
// c, scales s and minima z per token and group G of 32 channels,
//   score[k][col] = sum_G s_kG * (sum_{d in G} c_kd q_d) + sum_G z_kG * (sum_{d in G} q_d)
//   out[col][d]   = sum_k p_k (c_kd s_kG + z_kG)
// Keys: the tensor cores multiply the raw codes.  A nibble needs no conversion:
// in the fp16 pair w & 0x000f000f each half is the subnormal code * 2^-24, in
// w & 0x00f000f0 it is 16 code * 2^-24, and m16n8k16 takes subnormals exactly.
// The queries are scaled by a power of two per column (and 1/16 for the odd
// nibbles), so a bf16 or fp16 query enters exactly; products are summed in fp32.
// Values: code * s + z is rounded once to fp16 (one fma on the exact code), and
// so is p: each costs 2^-11 of a token's share p |value|, below a bf16 output's own
// rounding.  (Multiplying raw codes by p s instead would round a number that may
// be many times p |value|.)  For an fp16 output, whose rounding is as fine, p enters
// as the sum of two fp16 numbers, at two products a tile more per group: error
// against 64 bits 1.3 times the output rounding's instead of 1.6.  Small weights
// keep fewer bits: fp16 ends at steps of 2^-24.  So that a dominant token does not
// press the rest of its warp's tokens below that, the largest weight is put at 2^7
// and not at 1: what is lost of a weight is then 2^-32 of the warp's largest at most.
// A Value group that may pass the fp16 range stays out of the product and is added in
// fp32 at the end (add_apart).
//
// The work is one pass over the pages with a running maximum and sum.  The
// maximum is moved only when a score passes it by 2^8 (p <= 2^15 fits), so most
// tiles skip the rescaling.  It is kept in the units of the codes' products, whose sum
// starts from it: scores come out relative to it, and no rounding of a large product
// of score and scaling reaches the exponent.
//
// Split.  All pages of all units form one line, cut into equal ranges, one per
// CTA (the lengths are read on the device, so nothing is planned on the host).
// Before each unit's pages lie kUnitCost empty places, the cost of taking up
// another unit in pages: a CTA whose range goes on into the next unit gets that
// many fewer, and short ranges end at the units' ends.  Two warps share a page,
// 32 tokens each, and each warp copies its half pages through its own ring of
// cp.async stages: no barrier until the unit's end.  A unit that lies in one
// range is finished there; otherwise each CTA leaves a partial (maximum, sum,
// accumulator) and the last one to arrive (an atomic ticket) merges them in the
// order of the ranges, so results do not depend on timing.
//
// Measured at 8 sequences of 32k tokens, 28 heads on 4, D 128, bf16 (168 MB), replayed
// in a graph: 41.7 us, 4.0 TB/s, 62 % of a plain copy's rate.  Of it 3.5 us pass before
// the first page is there (lengths, table and pages are dependent loads), 4 after the
// last one (partial, ticket, merge).  The loop takes 26 to 33 (traced in an earlier form
// of it, of the same time); its copies alone end at 25, so instructions and their
// latencies bound it: some 650 a warp for its 32 tokens, a third of them the Values'
// dequantisation, issue slots 57 % busy with three warps a scheduler.
#include <cmath>
#include <type_traits>

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
  int rows, cols, col_tiles;  // sequences (or query tokens), query columns of a unit, column tiles
  float* partials;
  uint32_t* tickets;
  int32_t* status;
  int sms;  // of the device (for the launch)
  PrefixPlan prefix;  // of a call with shared pages
};

constexpr int kTile = 16;             // tokens of one tensor-core step
constexpr int kPart = kInt4Page / 2;  // tokens of a page that one warp takes
constexpr int kSubs = kPart / kTile;
constexpr float kLift = 7.0f;         // log2 of the weight that a running maximum stands for
constexpr float kSlack = 8.0f;        // log2 a score may pass the running maximum by
constexpr float kNoMax = -3e38f;      // below any score
constexpr int kMinPages = 4;          // places of a range at least: two pages for each pair of warps
// Empty places before a unit's pages: at 8 x 32k 16 cost 2 us more than 6, 40 2.4 (fitted
// before the merge had its present form, as merge_pages below; fewer than 6 not tried).
constexpr int kUnitCost = 6;

// CTAs of four warps, three an SM (168 registers a thread), or two with 16 columns
// at D 128 (255), which hide each other's start and merge; the stages are what 227
// KB of shared memory hold.  Compared at 8 x 32k tokens, 28 heads on 4, before
// the loop had its present form: one CTA of 12 warps 53.8 us (starts and merges lie
// bare), three of 4 warps 48.7 us; four CTAs with two stages 55.5 us (too few bytes in
// flight); 16 tokens a warp instead of 32 52.0 us (a page's fixed work twice as often).
template <int D, int NT> struct AttendCfg {
  static constexpr int kWarps = 4, kThreads = 32 * kWarps, kTeams = kWarps / 2;
  static constexpr int kCtas = D == 128 && NT == 2 ? 2 : 3;
  static constexpr int kStages = D == 64 ? 6 : kCtas == 2 ? 5 : 3;
  static constexpr int kCodes = kPart * D / 2, kPar = kPart * D / 8;  // bytes of a warp's part, Key or Value
  static constexpr int kStageBytes = 2 * (kCodes + kPar);
  static constexpr int kPad = D + 4;  // floats between the columns of a merge buffer
  static constexpr int kRing = kWarps * kStages * kStageBytes;
  static constexpr int kMerge = kWarps * 8 * NT * (kPad + 2) * 4;
  static constexpr int kRecord = 8 * NT * (D + 2);  // floats of a partial: maxima, sums, accumulators
  // 16 partials where that costs no CTA: 60 KB of ring would hold 14 (D 128)
  static constexpr int kRoom = NT == 1 && kMerge < 64 * kRecord ? 64 * kRecord : kMerge;
  static constexpr int kSmem = kRing > kRoom ? kRing : kRoom;
  static constexpr int kFit = kSmem / (4 * kRecord);  // partials that are merged at once
};

// fp16 numbers that make up a weight.
template <typename T> constexpr int kWeightTerms = std::is_same<T, __half>::value ? 2 : 1;

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same from zero.
__device__ __forceinline__ void mma16816_zero(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma1688_zero(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%7,%7,%7};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(b0), "f"(0.0f));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// c += a b on two fp32 numbers in one instruction.
__device__ __forceinline__ void fma2(float& c0, float& c1, float a0, float a1, float b0, float b1) {
  const float2 c = __ffma2_rn(make_float2(a0, a1), make_float2(b0, b1), make_float2(c0, c1));
  c0 = c.x;
  c1 = c.y;
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Codes n0 and n1 of a byte n0 + 16 n1 in both halves, as exact fp16 numbers, from
// x = 1024 + byte: 1024 + 16 n1 by its bits, brought back by one fma, and what it
// leaves of x.
__device__ __forceinline__ void two_codes(uint32_t x, uint32_t& even, uint32_t& odd) {
  const uint32_t high = x & 0xFFF0FFF0u;
  odd = hfma2(high, 0x2C002C00u, 0xD400D400u);  // / 16 - 64
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(even) : "r"(x), "r"(high));
}
__device__ __forceinline__ bool is_nan_param(uint32_t w) { return (w & 0x7C00u) == 0x7C00u || (w & 0x7C000000u) == 0x7C000000u; }
// Whether code * s + z may pass the fp16 range: only where s is 2^11 or |z| 2^15 at
// least (else it is 15 * 2^11 + 2^15 = 63488 at most).
__device__ __forceinline__ bool is_wide_param(uint32_t w) {
  return ((w & 0x7FFFu) >= 0x6800u || (w & 0x7FFF0000u) >= 0x78000000u) && !is_nan_param(w);
}
// Whether a Value group of token tok (seen by some column) stays out of the product.
__device__ __forceinline__ bool stays_apart(uint32_t w, int tok, int vis_min) {
  return is_wide_param(w) || (tok >= vis_min && is_nan_param(w));
}
// Larger magnitude of each half (a NaN gives way to a number).
__device__ __forceinline__ uint32_t max_abs2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a & 0x7FFF7FFFu), "r"(b & 0x7FFF7FFFu));
  return r;
}
// kWords (2 or 4) words of shared memory in one load.
template <int kWords>
__device__ __forceinline__ void load_words(const uint8_t* at, uint32_t (&w)[kWords]) {
  if constexpr (kWords == 4) {
    const uint4 x = *reinterpret_cast<const uint4*>(at);
    w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
  } else {
    const uint2 x = *reinterpret_cast<const uint2*>(at);
    w[0] = x.x; w[1] = x.y;
  }
}
// Weights of 16 tokens (pr, spent: rows g and g + 8 of the scores' fragments) as the
// product's B operand, columns by tokens, in kTerms fp16 numbers.
template <int kTerms>
__device__ __forceinline__ void weight_operand(float (&pr)[4], uint32_t (&b)[kTerms][2]) {
#pragma unroll
  for (int y = 0; y < kTerms; ++y)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint32_t w = pack_half2(pr[2 * k], pr[2 * k + 1]);
      b[y][k] = transpose8x8(w);
      if (y + 1 < kTerms) {
        pr[2 * k] -= half_lo(w);
        pr[2 * k + 1] -= half_hi(w);
      }
    }
}
// Values of channels 4 g + n of group G for a pair of tokens, from its code words
// ([token][w]), scales and minima.
template <int kG>
__device__ __forceinline__ void value_operand(const uint32_t (&words)[kG], int G, uint32_t s2, uint32_t z2, uint32_t (&v)[4]) {
  // bytes of the even and the odd token, as 1024 + byte
  const uint32_t y = __byte_perm(words[G >> 1], words[kG / 2 + (G >> 1)], (G & 1) ? 0x7362 : 0x5140);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    uint32_t even, odd;
    two_codes(__byte_perm(y, 0x64646464u, k == 0 ? 0x4140 : 0x4342), even, odd);
    v[2 * k] = hfma2(even, s2, z2);
    v[2 * k + 1] = hfma2(odd, s2, z2);
  }
}
// sums += Values (two pairs of tokens) times weights.
template <int D, int NT, int kTerms>
__device__ __forceinline__ void add_values(float (&acc)[NT][D / 16][4], int G, const uint32_t (&v)[2][4],
                                           const uint32_t (&pb)[NT][kTerms][2]) {
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int y = 0; y < kTerms; ++y) {
      mma16816(acc[nt][2 * G], v[0][0], v[0][1], v[1][0], v[1][1], pb[nt][y][0], pb[nt][y][1]);
      mma16816(acc[nt][2 * G + 1], v[0][2], v[0][3], v[1][2], v[1][3], pb[nt][y][0], pb[nt][y][1]);
    }
}

// Adds 1 and returns what was there.  What the CTA wrote before the barrier ahead
// of it is visible to whoever takes a later ticket.
__device__ __forceinline__ uint32_t take_ticket(uint32_t* ticket) {
  uint32_t n;
  asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(n) : "l"(ticket) : "memory");
  return n;
}
__device__ __forceinline__ void add_scaled(float4& v, float f, float4 y) {
  v.x = fmaf(f, y.x, v.x);
  v.y = fmaf(f, y.y, v.y);
  v.z = fmaf(f, y.z, v.z);
  v.w = fmaf(f, y.w, v.w);
}

// Tokens that row r (a sequence, or a query token of one) sees at most.
template <bool kSparse>
__device__ __forceinline__ int row_tokens(const AttendParams& p, int r) {
  const int b = kSparse ? r / p.q_len : r;
  const int length = p.lengths[b], count = p.counts != nullptr ? p.counts[b] : p.q_len;
  return int4_seen(length, count, kSparse ? r - b * p.q_len : max(0, min(count, p.q_len) - 1));
}
// Pages of a row that sees `tokens`, behind its shared ones, at least 1, so that an empty row is visited
// and zeroed.
template <bool kSparse>
__device__ __forceinline__ int row_pages(const AttendParams& p, int tokens, int shared) {
  const int n = tokens / kInt4Page + (tokens % kInt4Page != 0);
  return max(1, min(n, kSparse ? p.slots : p.pool.table_width) - shared);
}

// Shared pages of sequence b, which are not among its own here.
template <bool kPrefix>
__device__ __forceinline__ int shared_pages(const AttendParams& p, int b) {
  if constexpr (!kPrefix) return 0;
  const int g = p.prefix.seqs[b].group;
  return g >= 0 && p.prefix.groups[g].live != 0 ? p.prefix.groups[g].pages : 0;
}

// Where the records of a unit's first column are.
struct SharedRows {
  const PrefixGroup* group;  // null: no shared pages
  int row, h, per;
};
// Adds the shared pages' part of kItems rows (row[k] of the group, channels d[k] .. d[k] + 3)
// to their maxima, sums and accumulators.
template <int D, int kItems>
__device__ __forceinline__ void add_shared(const PrefixPlan& plan, const SharedRows& where, const int (&row)[kItems], const int (&d)[kItems],
                                           float (&top)[kItems], float (&sum)[kItems], float4 (&v)[kItems]) {
  constexpr int kAhead = kItems <= 2 ? 4 : 2;  // parts whose loads wait for memory together, of all items
  const PrefixGroup& g = *where.group;
  const float* rec[kItems];
  int n[kItems], most = 0;
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    const int x = where.h * g.tiles + row[k] / kPrefixRows, start = g.start(x), first = start / where.per;
    n[k] = (start + g.steps - 1) / where.per - first + 1;
    most = max(most, n[k]);
    rec[k] = plan.records + (g.units + x + first) * prefix_record(D) + row[k] % kPrefixRows;
  }
#pragma unroll 1
  for (int x0 = 0; x0 < most; x0 += kAhead) {
    float tops[kAhead][kItems], sums[kAhead][kItems];
    float4 parts[kAhead][kItems];
#pragma unroll
    for (int x = 0; x < kAhead; ++x)
#pragma unroll
      for (int k = 0; k < kItems; ++k) {
        tops[x][k] = kNoMax;
        sums[x][k] = 0.0f;
        parts[x][k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (x0 + x < n[k]) {
          const float* at = rec[k] + (x0 + x) * prefix_record(D);
          tops[x][k] = at[0];
          sums[x][k] = at[kPrefixRows];
          parts[x][k] = *reinterpret_cast<const float4*>(at + 2 * kPrefixRows + row[k] % kPrefixRows * static_cast<int64_t>(D - 1) + d[k]);
        }
      }
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      float now = top[k];
#pragma unroll
      for (int x = 0; x < kAhead; ++x) now = fmaxf(now, tops[x][k]);
      const float fix = ex2(top[k] - now);
      top[k] = now;
      sum[k] *= fix;
      v[k] = make_float4(v[k].x * fix, v[k].y * fix, v[k].z * fix, v[k].w * fix);
#pragma unroll
      for (int x = 0; x < kAhead; ++x) {
        const float f = ex2(tops[x][k] - now);
        sum[k] = fmaf(f, sums[x][k], sum[k]);
        add_scaled(v[k], f, parts[x][k]);
      }
    }
  }
}

// Places of a range below which the merge costs more than the range: with n pages
// a unit in ranges of r, r pages take 0.3 r us and the last to arrive another 0.1 us
// for each of n / r parts, least at r = sqrt(n / 3).
__device__ __forceinline__ int merge_pages(int total, int units) {
  return static_cast<int>(sqrtf(static_cast<float>(total / units) / 3.0f));
}

// A unit, as add_apart needs it.
struct Unit {
  int b, h, c0, i0, first, stop, length, count, seen_max, vis_min;
  const int32_t* listed;  // pages of a sparse unit
  int shared;             // pages before its first
};
// Value groups that stayed out of the products of a warp's pages, added in fp32 to its
// sums in the merge buffer: those that may pass the fp16 range (scaled to fit it, they
// would cost the small groups beside them their low bits), and NaN ones that only some
// columns see.  It goes through the warp's pages again, token by token, with scores of
// its own (top: the maxima that the sums are relative to, in log2).  Slow where there are
// many: 8 x 32k tokens, 28 heads on 4, D 128, 42 us without any, 88 with one in every 64
// tokens, 305 in every 4th, 940 in every one; a second product in the loop took 104 for
// that, but cost the calls without any 3 %, for its registers.
template <typename T, int D, int NT, bool kSparse>
__device__ __noinline__ void add_apart(const AttendParams& p, const Unit& u, const int* vis, float* sums, const float* top) {
  constexpr int kG = D / kInt4Group, kOwn = D / 32, kCol = 8 * NT, kPad = AttendCfg<D, NT>::kPad;
  const int part = (threadIdx.x >> 5) & 1, lane = threadIdx.x & 31;
  const int d = lane * kOwn, G = d / kInt4Group;  // the lane's channels: kOwn from d on
  float q[kCol][kOwn];
#pragma unroll
  for (int col = 0; col < kCol; ++col) {
    const int c = min(u.c0 + col, p.cols - 1), i = kSparse || p.q_len == 1 ? 0 : c / p.group;
    const T* from = static_cast<const T*>(p.q) + u.b * p.q_seq + (u.h * p.group + c - i * p.group) * p.q_head +
                    (u.i0 + i) * p.q_tok + d;
#pragma unroll
    for (int x = 0; x < kOwn; ++x) q[col][x] = Scalar<T>::load(from + x);
  }
#pragma unroll 1
  for (int place = u.first + (threadIdx.x >> 6); place < u.stop; place += AttendCfg<D, NT>::kTeams) {
    const int page = kSparse ? u.listed[place] : u.shared + place;
    if (page < 0 || page > (u.seen_max - 1) / kInt4Page) continue;  // (seen_max > 0: there was a group to add)
    const int id = int4_page_id(p.pool, u.b, page), base = page * kInt4Page + part * kPart;
    if (id < 0 || base >= u.seen_max) continue;
    const uint32_t* rec = reinterpret_cast<const uint32_t*>(p.pool.words) + int4_record(p.pool, id, u.h);
    bool apart = false;
    if (base + lane < u.seen_max) {
      uint32_t sz[kG];
      load_words<kG>(reinterpret_cast<const uint8_t*>(rec + 18 * D + (part * kPart + lane) * kG), sz);
#pragma unroll
      for (int x = 0; x < kG; ++x) apart |= stays_apart(sz[x], base + lane, u.vis_min);
    }
#pragma unroll 1
    for (uint32_t rest = __ballot_sync(0xffffffffu, apart); rest != 0; rest &= rest - 1) {
      const int tok = base + __ffs(rest) - 1, k = tok % kInt4Page;
      const uint32_t ksz = rec[8 * D + k * kG + G], vsz = rec[18 * D + k * kG + G];
      const uint32_t kc = rec[k * (D / 8) + d % 32 / 8 * kG + G] >> (4 * (d % 8));
      const uint32_t vc = rec[10 * D + (k >> 3) * D + d % 32 / 4 * (D / 8) + (k & 7) / 2 * kG + (k & 1) * (D / 64) + d / 64] >>
                          (16 * (G & 1) + 4 * (d % 4));
      float key[kOwn], value[kOwn], score[kCol];
#pragma unroll
      for (int x = 0; x < kOwn; ++x) {
        key[x] = fmaf(static_cast<float>(kc >> (4 * x) & 15u), half_lo(ksz), half_hi(ksz));
        value[x] = fmaf(static_cast<float>(vc >> (4 * x) & 15u), half_lo(vsz), half_hi(vsz));
      }
#pragma unroll
      for (int col = 0; col < kCol; ++col) {
        score[col] = 0.0f;
#pragma unroll
        for (int x = 0; x < kOwn; ++x) score[col] = fmaf(q[col][x], key[x], score[col]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) score[col] += __shfl_xor_sync(0xffffffffu, score[col], o);
      }
      if (stays_apart(vsz, tok, u.vis_min)) {
#pragma unroll
        for (int col = 0; col < kCol; ++col) {
          if (tok >= vis[col]) continue;
          const float w = ex2(fminf(fmaf(score[col], p.scale_log2, -top[col]), kSlack) + kLift);
#pragma unroll
          for (int x = 0; x < kOwn; ++x) sums[col * kPad + d + x] = fmaf(w, value[x], sums[col * kPad + d + x]);
        }
      }
    }
  }
}

template <typename T, int D, int NT, bool kSparse, bool kPrefix>
__global__ void __launch_bounds__(AttendCfg<D, NT>::kThreads, AttendCfg<D, NT>::kCtas)
    int4_attend_kernel(const __grid_constant__ AttendParams p) {
  using C = AttendCfg<D, NT>;
  constexpr int kG = D / kInt4Group, kCol = 8 * NT, kStages = C::kStages, kWarps = C::kWarps;
  constexpr int kCodes = C::kCodes, kPar = C::kPar;
  constexpr int kTerms = kWeightTerms<T>;
  extern __shared__ __align__(128) uint8_t smem[];  // 8 x 32k, from Python: 39.8 us; 42.2 at 112 past a multiple
  __shared__ int meta_s[kWarps][kStages];  // first token of each stage's part of a page, -1: nothing to do
  __shared__ int last_s;
  __shared__ Unit unit_s;
  __shared__ int vis_s[kWarps][kCol];  // tokens that each column sees
  __shared__ SharedRows rows_s;
  __shared__ int apart_s[kWarps];       // a Value group stayed out of the product
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int per_row = p.pool.kv_heads * p.col_tiles;
  grid_dep_wait();

  // The line of pages: its length, and the row where this CTA's range begins.
  auto places = [&](int r) {
    return r < p.rows ? (row_pages<kSparse>(p, row_tokens<kSparse>(p, r), shared_pages<kPrefix>(p, r)) + kUnitCost) * per_row : 0;
  };
  const int places0 = places(lane);
  int total = __reduce_add_sync(0xffffffffu, places0);
  for (int r0 = 32; r0 < p.rows; r0 += 32) total += __reduce_add_sync(0xffffffffu, places(r0 + lane));
  const int per = max(kMinPages, max(static_cast<int>((total + gridDim.x - 1) / gridDim.x), merge_pages(total, p.rows * per_row)));
  const int begin = blockIdx.x * per, end = min(total, begin + per);
  if (begin >= end) return;
  int row = 0, row_base = 0;
  for (int r0 = 0; r0 < p.rows; r0 += 32) {
    const int n = r0 == 0 ? places0 : places(r0 + lane);
    int upto = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, row_base + upto > begin);
    if (past != 0) {
      const int l = __ffs(past) - 1;
      row = r0 + l;
      row_base += __shfl_sync(0xffffffffu, upto - n, l);
      break;
    }
    row_base += __shfl_sync(0xffffffffu, upto, 31);
  }

  uint8_t* ring = smem + warp * kStages * C::kStageBytes;
  const uint32_t ring_a = smem_addr(ring) + lane * 16;
  const int team = warp >> 1, part = warp & 1;
  // Byte offsets in a record of this lane's pieces: Key codes (Value codes 40 D
  // later), and parameters, the first half of the lanes Key's, the others Value's.
  constexpr int kParLanes = kPar / 16;  // lanes' worth of a half page's Key parameters
  const int code_at = part * kCodes + lane * 16;
  int at = begin;
  while (at < end) {
    // ------------------------------------------------------------ one unit
    const int shared = shared_pages<kPrefix>(p, row);
    const int seen_max = row_tokens<kSparse>(p, row), n_pages = row_pages<kSparse>(p, seen_max, shared);
    const int in_row = at - row_base, unit_in_row = in_row / (n_pages + kUnitCost);
    const int unit_begin = row_base + unit_in_row * (n_pages + kUnitCost) + kUnitCost;  // its first page's place
    const int unit_end = unit_begin + n_pages;
    const int first = max(0, at - unit_begin), stop = min(end, unit_end) - unit_begin;
    const int h = unit_in_row / p.col_tiles, c0 = (unit_in_row - h * p.col_tiles) * kCol;
    at = unit_begin + stop;
    const int row_now = row;
    if (at - row_base == (n_pages + kUnitCost) * per_row) {
      row_base = at;
      ++row;
    }
    if (stop <= first) continue;
    const int b = kSparse ? row_now / p.q_len : row_now;
    const int i0 = kSparse ? row_now - b * p.q_len : 0;
    const int length = p.lengths[b], count = p.counts != nullptr ? p.counts[b] : p.q_len;
    if (tid == 0 && p.status != nullptr && (seen_max - 1) / kInt4Page >= p.pool.table_width)
      atomicExch(p.status, LF_ERR_OUT_OF_RANGE);

    // Query column c of the unit is query token i0 + c / group of q-head h * group + c % group.
    auto token_of = [&](int c) { return kSparse || p.q_len == 1 ? 0 : c / p.group; };
    uint4 qw[NT][kG];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int c = c0 + nt * 8 + g, i = token_of(c);
      const T* q = static_cast<const T*>(p.q) + b * p.q_seq + (h * p.group + c - i * p.group) * p.q_head + (i0 + i) * p.q_tok;
#pragma unroll
      for (int G = 0; G < kG; ++G)
        qw[nt][G] = c < p.cols ? *reinterpret_cast<const uint4*>(q + 32 * G + 8 * t) : make_uint4(0, 0, 0, 0);
    }

    // This warp's pages: first + team, then every kTeams-th.  Their ids, 32 at a
    // time, one per lane.
    const int mine_n = first + team < stop ? (stop - first - team + C::kTeams - 1) / C::kTeams : 0;
    const int32_t* listed =
        kSparse ? p.picked + (static_cast<int64_t>(row_now) * p.pool.kv_heads + h) * p.slots : nullptr;
    int ids = -1, logicals = -1;
    int issued = 0, into = 0;  // pages issued, the stage of the next
    const uint8_t* head_words = reinterpret_cast<const uint8_t*>(p.pool.words + h * p.pool.head_stride);
    auto issue = [&]() {
      if (issued < mine_n) {
        if ((issued & 31) == 0) {
          ids = logicals = -1;
          if (issued + lane < mine_n) {
            logicals = shared + first + team + (issued + lane) * C::kTeams;
            if constexpr (kSparse) logicals = listed[logicals];
            if (logicals >= 0 && seen_max > 0 && logicals <= (seen_max - 1) / kInt4Page) {
              ids = int4_page_id(p.pool, b, logicals);
              if (ids < 0 && p.status != nullptr) atomicExch(p.status, LF_ERR_OUT_OF_RANGE);
            }
          }
        }
        const int id = __shfl_sync(0xffffffffu, ids, issued & 31);
        const int logical = __shfl_sync(0xffffffffu, logicals, issued & 31);
        if (lane == 0) meta_s[warp][into] = id < 0 ? -1 : logical * kInt4Page + part * kPart;
        if (id >= 0) {
          const uint8_t* rec = head_words + id * p.pool.page_stride * 4;
          const uint32_t dst = ring_a + into * C::kStageBytes;
          const uint8_t* kc = rec + code_at;
#pragma unroll
          for (int x = 0; x < kCodes / 512; ++x) {
            cp_async16(dst + x * 512, kc + x * 512);
            cp_async16(dst + kCodes + x * 512, kc + 40 * D + x * 512);
          }
          if constexpr (kParLanes == 32) {
            cp_async16(dst + 2 * kCodes, rec + 32 * D + part * kPar + lane * 16);
            cp_async16(dst + 2 * kCodes + 512, rec + 72 * D + part * kPar + lane * 16);
          } else {
            const int v = lane / kParLanes;
            cp_async16(dst + 2 * kCodes, rec + 32 * D + v * 40 * D + part * kPar + (lane - v * kParLanes) * 16);
          }
        }
        ++issued;
        into = into + 1 == kStages ? 0 : into + 1;
      }
      cp_commit();
    };
#pragma unroll 1
    for (int s = 0; s < kStages - 1; ++s) issue();

    // Query fragments, sums and scales of this unit's columns.
    uint32_t qf[NT][2 * kG][2], qz[NT];
    float c2[NT][2];
    int vis_min = INT32_MAX;
    const float flip = p.scale_log2 < 0.0f ? -1.0f : 1.0f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float x[kG][8], most = 0.0f;
#pragma unroll
      for (int G = 0; G < kG; ++G) {
        const uint32_t v[4] = {qw[nt][G].x, qw[nt][G].y, qw[nt][G].z, qw[nt][G].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if constexpr (std::is_same<T, __half>::value) {
            x[G][2 * k] = half_lo(v[k]);
            x[G][2 * k + 1] = half_hi(v[k]);
          } else {
            x[G][2 * k] = __uint_as_float(v[k] << 16);
            x[G][2 * k + 1] = __uint_as_float(v[k] & 0xFFFF0000u);
          }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) most = fmaxf(most, fabsf(x[G][k]));
      }
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
      // 2^kq brings the column's largest magnitude to [2^13, 2^14) (below where the largest
      // is under 2^-114: 2^127 is the last power there is)
      const int kq = most > 0.0f && most < INFINITY
                         ? min(127, 13 - (static_cast<int>(__float_as_uint(most) >> 23) - 127))
                         : 0;
      const float up = pow2(kq) * flip;
      float sums[kG];
#pragma unroll
      for (int G = 0; G < kG; ++G) {
        sums[G] = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          x[G][k] *= up;
          sums[G] += x[G][k];
        }
        sums[G] += __shfl_xor_sync(0xffffffffu, sums[G], 1);
        sums[G] += __shfl_xor_sync(0xffffffffu, sums[G], 2);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          qf[nt][2 * G + k][0] = pack_half2(x[G][2 * k], x[G][2 * k + 4]);
          qf[nt][2 * G + k][1] = pack_half2(x[G][2 * k + 1] * 0.0625f, x[G][2 * k + 5] * 0.0625f);
        }
      }
      // The column's sum over group t's channels as two fp16 limbs (22 bits).
      float mine = 0.0f;
#pragma unroll
      for (int G = 0; G < kG; ++G) mine = t == G ? sums[G] : mine;
      mine *= 0x1p-10f;
      const float hi = __half2float(__float2half_rn(mine));
      qz[nt] = pack_half2(hi, mine - hi);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int kc = __shfl_sync(0xffffffffu, kq, (2 * t + k) * 4);
        // positive, so that a masked score's -inf stays one
        c2[nt][k] = fmaxf(pow2(10 - kc) * fabsf(p.scale_log2), 1e-36f);
        const int col = min(c0 + nt * 8 + 2 * t + k, p.cols - 1);
        const int vis = int4_seen(length, count, i0 + token_of(col));
        if (g == 0) vis_s[warp][nt * 8 + 2 * t + k] = vis;
        vis_min = min(vis_min, vis);
      }
    }
    vis_min = __reduce_min_sync(0xffffffffu, vis_min);

    if constexpr (kPrefix) {
      if (tid == 0) {
        rows_s.group = nullptr;
        if (shared > 0) {
          const PrefixSeq s = p.prefix.seqs[b];
          rows_s = SharedRows{p.prefix.groups + s.group, s.rank * p.cols + c0, h, p.prefix.head[1]};
        }
      }
    }
    if (tid == 0) unit_s = Unit{b, h, c0, i0, first, stop, length, count, seen_max, vis_min, listed, shared};
    if (lane == 0) apart_s[warp] = 0;
    float acc[NT][2 * kG][4], back[NT][2], l[NT][2];  // back: the running maxima, negated, times 2^-14
    bool fresh = true;  // before the first part
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        back[nt][k] = 0.0f;
        l[nt][k] = 0.0f;
      }
#pragma unroll
      for (int x = 0; x < 2 * kG; ++x)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[nt][x][k] = 0.0f;
    }

    // ------------------------------------------------------- its half pages
    int st = 0;
    for (int j = 0; j < mine_n; ++j) {
      cp_wait<kStages - 2>();
      __syncwarp();
      issue();
      const int base = meta_s[warp][st];
      uint8_t* stage = ring + st * C::kStageBytes;
      st = st + 1 == kStages ? 0 : st + 1;
      if (base < 0 || base >= seen_max) continue;
      const bool masked = base + kPart > vis_min;  // tokens here that not every column sees

      // Value parameters in pairs of tokens, as the fragments take them: in place
      // of (s, z) of tokens 2 x and 2 x + 1 a lane writes (s, s'), (z, z').
      {
        constexpr int kQ = kG / 2;  // groups of a lane: two lanes for each of the 16 pairs
        const int x = lane >> 1, q = lane & 1;
        uint32_t* par = reinterpret_cast<uint32_t*>(stage + 2 * kCodes + kPar);
        uint32_t e[kQ], o[kQ];
#pragma unroll
        for (int k = 0; k < kQ; ++k) {
          e[k] = par[2 * x * kG + q * kQ + k];
          o[k] = par[(2 * x + 1) * kG + q * kQ + k];
        }
        bool any_apart = false;
        const int tok = base + 2 * x;
        if (masked) {  // what an unwritten slot holds must not be read
#pragma unroll
          for (int k = 0; k < kQ; ++k) {
            if (tok >= seen_max) e[k] = 0;
            if (tok + 1 >= seen_max) o[k] = 0;
            any_apart |= (tok >= vis_min && is_nan_param(e[k])) || (tok + 1 >= vis_min && is_nan_param(o[k]));
          }
        }
        uint32_t s2[kQ], z2[kQ], most = 0;
#pragma unroll
        for (int k = 0; k < kQ; ++k) {
          s2[k] = __byte_perm(e[k], o[k], 0x5410);
          z2[k] = __byte_perm(e[k], o[k], 0x7632);
          most = max_abs2(most, hmul2(s2[k], 0x4C004C00u));  // 16 s
          most = max_abs2(most, z2[k]);
        }
        any_apart |= (most & 0x7FFFu) >= 0x7800u || (most & 0x7FFF0000u) >= 0x78000000u;  // 2^15: is_wide_param of one
        if (__any_sync(0xffffffffu, any_apart)) {
          if (lane == 0) apart_s[warp] = 1;
#pragma unroll
          for (int k = 0; k < kQ; ++k) {
            if (stays_apart(e[k], tok, vis_min)) e[k] = 0;
            if (stays_apart(o[k], tok + 1, vis_min)) o[k] = 0;
            s2[k] = __byte_perm(e[k], o[k], 0x5410);
            z2[k] = __byte_perm(e[k], o[k], 0x7632);
          }
        }
        __syncwarp();  // every lane has read its words
        if constexpr (kQ == 2)
          *reinterpret_cast<uint4*>(par + 4 * lane) = make_uint4(s2[0], z2[0], s2[1], z2[1]);
        else
          *reinterpret_cast<uint2*>(par + 2 * lane) = make_uint2(s2[0], z2[0]);
        __syncwarp();
      }

      // Scores of the part's tokens, 16 at a time (rows g and g + 8 of the fragment).
      float x[kSubs][NT][4];
#pragma unroll
      for (int sub = 0; sub < kSubs; ++sub) {
        const uint8_t* kcode = stage + sub * (kTile * D / 2);
        const uint8_t* kpar = stage + 2 * kCodes + sub * (kTile * D / 8);
        uint32_t kw[2][kG], ks[2][kG], kz[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          load_words<kG>(kcode + r * (4 * D) + lane * (4 * kG), kw[r]);
          load_words<kG>(kpar + (8 * r + g) * (4 * kG), ks[r]);
          kz[r] = t < kG ? *reinterpret_cast<const uint32_t*>(kpar + (8 * r + g) * (4 * kG) + t * 4) : 0u;
          kz[r] = __byte_perm(kz[r], 0, 0x3232);
        }
        float dot[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma1688_zero(x[sub][nt], kz[0], kz[1], qz[nt]);
#pragma unroll
          for (int k = 0; k < 4; ++k) dot[nt][k] = back[nt][k & 1];
        }
#pragma unroll
        for (int G = 0; G < kG; ++G) {
          const uint32_t a[2][2] = {{kw[0][G], kw[1][G]}, {kw[0][G] >> 8, kw[1][G] >> 8}};
          const float s0 = half_lo(ks[0][G]), s1 = half_lo(ks[1][G]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float d[4];
            mma16816_zero(d, a[0][0] & 0x000f000fu, a[0][1] & 0x000f000fu, a[0][0] & 0x00f000f0u, a[0][1] & 0x00f000f0u,
                          qf[nt][2 * G][0], qf[nt][2 * G][1]);
            mma16816(d, a[1][0] & 0x000f000fu, a[1][1] & 0x000f000fu, a[1][0] & 0x00f000f0u, a[1][1] & 0x00f000f0u,
                     qf[nt][2 * G + 1][0], qf[nt][2 * G + 1][1]);
            dot[nt][0] = fmaf(d[0], s0, dot[nt][0]);
            dot[nt][1] = fmaf(d[1], s0, dot[nt][1]);
            dot[nt][2] = fmaf(d[2], s1, dot[nt][2]);
            dot[nt][3] = fmaf(d[3], s1, dot[nt][3]);
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int k = 0; k < 4; k += 2) fma2(x[sub][nt][k], x[sub][nt][k + 1], dot[nt][k], dot[nt][k + 1], 16384.0f, 16384.0f);
      }
      if (masked) {
#pragma unroll
        for (int sub = 0; sub < kSubs; ++sub)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int tok = base + sub * kTile + 8 * r + g;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int k = 0; k < 2; ++k)
                if (tok >= vis_s[warp][nt * 8 + 2 * t + k]) x[sub][nt][2 * r + k] = -INFINITY;
          }
      }

      // The running maxima, moved where a score passes one by more than the slack, and set
      // by the first part (a column that sees nothing of it sees nothing of the later ones).
      bool move = fresh;
      float most[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          most[nt][k] = fmaxf(x[0][nt][k], x[0][nt][k + 2]);
#pragma unroll
          for (int sub = 1; sub < kSubs; ++sub) most[nt][k] = fmaxf(most[nt][k], fmaxf(x[sub][nt][k], x[sub][nt][k + 2]));
          move |= most[nt][k] * c2[nt][k] > kSlack;
        }
      if (__any_sync(0xffffffffu, move)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float fix[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float by = most[nt][k];
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) by = fmaxf(by, __shfl_xor_sync(0xffffffffu, by, o));
            if (!(by > (fresh ? -INFINITY : 0.0f))) by = 0.0f;
            fix[k] = fresh ? 1.0f : ex2(-by * c2[nt][k]);
            back[nt][k] -= by * 0x1p-14f;
            l[nt][k] *= fix[k];
#pragma unroll
            for (int sub = 0; sub < kSubs; ++sub) {
              x[sub][nt][k] -= by;
              x[sub][nt][k + 2] -= by;
            }
          }
#pragma unroll
          for (int y = 0; y < 2 * kG; ++y)
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[nt][y][k] *= fix[k & 1];
        }
        fresh = false;
      }

#pragma unroll
      for (int sub = 0; sub < kSubs; ++sub) {
        uint32_t pb[NT][kTerms][2];  // weights as the product's B operand: columns by tokens
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float pr[4];
#pragma unroll
          for (int k = 0; k < 4; k += 2) {
            float a0 = kLift, a1 = kLift;
            fma2(a0, a1, x[sub][nt][k], x[sub][nt][k + 1], c2[nt][0], c2[nt][1]);
            pr[k] = ex2(a0);
            pr[k + 1] = ex2(a1);
            const float2 sum = __fadd2_rn(make_float2(l[nt][0], l[nt][1]), make_float2(pr[k], pr[k + 1]));
            l[nt][0] = sum.x;
            l[nt][1] = sum.y;
          }
          weight_operand<kTerms>(pr, pb[nt]);
        }

        // Values: codes of 16 tokens, pairs (2t, 2t + 1) of each half, and their parameters.
        const uint8_t* vcode = stage + kCodes + sub * (kTile * D / 2);
        const uint8_t* vpair = stage + 2 * kCodes + kPar + sub * (kTile * D / 8);
        uint32_t vw[2][kG], sz[2][2 * kG];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          load_words<kG>(vcode + r * (4 * D) + lane * (4 * kG), vw[r]);
          load_words<kG>(vpair + (4 * r + t) * (8 * kG), *reinterpret_cast<uint32_t(*)[kG]>(&sz[r][0]));
          load_words<kG>(vpair + (4 * r + t) * (8 * kG) + 4 * kG, *reinterpret_cast<uint32_t(*)[kG]>(&sz[r][kG]));
        }
#pragma unroll
        for (int G = 0; G < kG; ++G) {
          uint32_t v[2][4];  // half, channel 4 g + n of the group
#pragma unroll
          for (int r = 0; r < 2; ++r) value_operand<kG>(vw[r], G, sz[r][2 * G], sz[r][2 * G + 1], v[r]);
          add_values<D>(acc, G, v, pb);
        }
      }
    }
    cp_wait<0>();
    __syncthreads();  // the rings are free: the merge buffer takes their place

    // ------------------------------------------ the warps' results, merged
    float* merge = reinterpret_cast<float*>(smem);
    float* top_w = merge + kWarps * kCol * C::kPad;
    float* sum_w = top_w + kWarps * kCol;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float sum = l[nt][k];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const int col = warp * kCol + nt * 8 + 2 * t + k;
        if (g == 0) {
          top_w[col] = sum == 0.0f ? kNoMax : fmaxf(-back[nt][k] * 16384.0f * c2[nt][k], kNoMax);
          sum_w[col] = sum;
        }
#pragma unroll
        for (int G = 0; G < kG; ++G)
          *reinterpret_cast<float4*>(merge + col * C::kPad + 32 * G + 4 * g) =
              make_float4(acc[nt][2 * G][k], acc[nt][2 * G][k + 2], acc[nt][2 * G + 1][k], acc[nt][2 * G + 1][k + 2]);
      }
    __syncwarp();
    if (apart_s[warp] != 0)
      add_apart<T, D, NT, kSparse>(p, unit_s, vis_s[warp], merge + warp * kCol * C::kPad, top_w + warp * kCol);
    __syncthreads();

    const bool whole = first == 0 && stop == n_pages;
    T* out = static_cast<T*>(p.out) + b * p.out_seq;
    auto store = [&](int col, int d, float4 v, float sum) {
      const int c = c0 + col, i = token_of(c);
      if (c >= p.cols) return;
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // a column that sees nothing
      T* o = out + (h * p.group + c - i * p.group) * p.out_head + (i0 + i) * p.out_tok + d;
      struct alignas(4 * sizeof(T)) Four { T x[4]; } f;
      Scalar<T>::store(f.x, v.x * inv);
      Scalar<T>::store(f.x + 1, v.y * inv);
      Scalar<T>::store(f.x + 2, v.z * inv);
      Scalar<T>::store(f.x + 3, v.w * inv);
      *reinterpret_cast<Four*>(o) = f;
    };
    // The partial of range x of this unit: the range that begins inside the unit
    // uses its CTA's first record, the unit's first range the second.
    const int first_cta = unit_begin / per, last_cta = (unit_end - 1) / per, parts = last_cta - first_cta + 1;
    auto record = [&](int x) { return p.partials + (2 * static_cast<int64_t>(x) + (x == first_cta)) * C::kRecord; };
    float* mine = record(blockIdx.x);
    constexpr int kItems = kCol * D / 4 / C::kThreads;  // (column, four channels) a thread merges
    // The thread's items with what the shared pages gave, stored.
    auto store_shared = [&](float (&top)[kItems], float (&sum)[kItems], float4 (&v)[kItems]) {
      int row[kItems], d[kItems];
#pragma unroll
      for (int it = 0; it < kItems; ++it) {
        const int item = tid + it * C::kThreads;
        row[it] = rows_s.row + min(item / (D / 4), p.cols - 1 - c0);
        d[it] = item % (D / 4) * 4;
      }
      if (rows_s.group != nullptr) add_shared<D>(p.prefix, rows_s, row, d, top, sum, v);
#pragma unroll
      for (int it = 0; it < kItems; ++it) store((tid + it * C::kThreads) / (D / 4), d[it], v[it], sum[it]);
    };
    float tops[kItems], sums[kItems];
    float4 all[kItems];
#pragma unroll
    for (int it = 0; it < kItems; ++it) {
      const int item = tid + it * C::kThreads, col = item / (D / 4), d = item % (D / 4) * 4;
      float top = top_w[col], sum = 0.0f;
#pragma unroll
      for (int w = 1; w < kWarps; ++w) top = fmaxf(top, top_w[w * kCol + col]);
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = ex2(top_w[w * kCol + col] - top);
        sum = fmaf(f, sum_w[w * kCol + col], sum);
        add_scaled(v, f, *reinterpret_cast<const float4*>(merge + (w * kCol + col) * C::kPad + d));
      }
      if (whole) {
        if constexpr (kPrefix) {
          tops[it] = top;
          sums[it] = sum;
          all[it] = v;
        } else {
          store(col, d, v, sum);
        }
      } else {
        *reinterpret_cast<float4*>(mine + 2 * kCol + col * D + d) = v;
        if (d == 0) {
          mine[col] = top;
          mine[kCol + col] = sum;
        }
      }
    }
    if constexpr (kPrefix) {
      if (whole) store_shared(tops, sums, all);
    }
    if (!whole) {
      __syncthreads();
      if (tid == 0) {
        uint32_t* ticket = p.tickets + static_cast<int64_t>(row_now) * per_row + unit_in_row;
        const uint32_t n = take_ticket(ticket) + 1;
        if (n == static_cast<uint32_t>(parts)) *ticket = 0;  // every range has arrived: ready for the next call
        last_s = n == static_cast<uint32_t>(parts);
      }
      __syncthreads();
      if (last_s) {
        // The parts, as many as shared memory holds, in one round of copies: 14 parts
        // take 4 us from the ticket to the end in two rounds through registers, 2.8 so.
        float top[kItems], sum[kItems];
        float4 v[kItems];
#pragma unroll
        for (int it = 0; it < kItems; ++it) {
          top[it] = kNoMax;
          sum[it] = 0.0f;
          v[it] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        for (int x0 = 0; x0 < parts; x0 += C::kFit) {
          const int n = min(C::kFit, parts - x0);
          for (int x = 0; x < n; ++x) {
            const float* rec = record(first_cta + x0 + x);
            for (int c = tid * 4; c < C::kRecord; c += C::kThreads * 4) cp_async16(smem_addr(merge + x * C::kRecord + c), rec + c);
          }
          cp_commit();
          cp_wait<0>();
          __syncthreads();
          float now[kItems];
#pragma unroll
          for (int it = 0; it < kItems; ++it) now[it] = top[it];
#pragma unroll 4
          for (int x = 0; x < n; ++x)
#pragma unroll
            for (int it = 0; it < kItems; ++it)
              now[it] = fmaxf(now[it], merge[x * C::kRecord + (tid + it * C::kThreads) / (D / 4)]);
#pragma unroll
          for (int it = 0; it < kItems; ++it) {
            const float fix = ex2(top[it] - now[it]);
            top[it] = now[it];
            sum[it] *= fix;
            v[it] = make_float4(v[it].x * fix, v[it].y * fix, v[it].z * fix, v[it].w * fix);
          }
#pragma unroll 4
          for (int x = 0; x < n; ++x)
#pragma unroll
            for (int it = 0; it < kItems; ++it) {
              const int item = tid + it * C::kThreads, col = item / (D / 4), d = item % (D / 4) * 4;
              const float* rec = merge + x * C::kRecord;
              const float f = ex2(rec[col] - now[it]);
              sum[it] = fmaf(f, rec[kCol + col], sum[it]);
              add_scaled(v[it], f, *reinterpret_cast<const float4*>(rec + 2 * kCol + col * D + d));
            }
          __syncthreads();
        }
        if constexpr (kPrefix) {
          store_shared(top, sum, v);
        } else {
#pragma unroll
          for (int it = 0; it < kItems; ++it) {
            const int item = tid + it * C::kThreads;
            store(item / (D / 4), item % (D / 4) * 4, v[it], sum[it]);
          }
        }
      }
    }
    __syncthreads();  // the merge buffer is free for the next unit's stages
  }
}

// The partials: two records per CTA of the largest grid.
static size_t partial_bytes(int sms) {
  using A = AttendCfg<128, 1>;
  using B = AttendCfg<128, 2>;
  using E = AttendCfg<64, 2>;
  constexpr int a = A::kCtas * A::kRecord, b = B::kCtas * B::kRecord, e = E::kCtas * E::kRecord;
  constexpr int most = a > b ? (a > e ? a : e) : (b > e ? b : e);
  return static_cast<size_t>(sms) * 2 * most * sizeof(float);
}

template <typename T, int D, int NT, bool kSparse, bool kPrefix = false>
static int launch_attend(AttendParams p, cudaStream_t stream) {
  using C = AttendCfg<D, NT>;
  const void* kern = reinterpret_cast<const void*>(int4_attend_kernel<T, D, NT, kSparse, kPrefix>);
  cudaError_t err = raise_smem_limit(kern, C::kSmem, true);
  if (err != cudaSuccess) {
    set_error("lf_int4_attend: %s", cudaGetErrorString(err));
    return LF_ERR_CUDA;
  }
  // No more CTAs than ranges there can be.
  const int64_t units = static_cast<int64_t>(p.rows) * p.pool.kv_heads * p.col_tiles;
  const int64_t pages = units * (kSparse ? p.slots : p.pool.table_width);
  const int64_t ranges = (pages + units * kUnitCost + kMinPages - 1) / kMinPages, slots = static_cast<int64_t>(p.sms) * C::kCtas;
  void* args[] = {&p};
  err = launch_programmatic(kern, dim3(static_cast<unsigned>(ranges < slots ? ranges : slots)), dim3(C::kThreads), C::kSmem,
                            stream, args);
  if (err != cudaSuccess) {
    set_error("lf_int4_attend: %s", cudaGetErrorString(err));
    return LF_ERR_LAUNCH;
  }
  return launch_status("lf_int4_attend");
}
// 16 columns a unit where a unit has more than 8: the codes are then unpacked once
// for both halves.  Measured at 8 x 16k tokens, D 128: 7 columns 27.9 us in tiles of
// 8, 35.7 in one of 16 (fewer warps fit); 16 columns 41.3 us in two tiles, 35.9 in one
// (now 26.4 and 34.8).  Four column tiles in one at D 64 do not pay: 25 columns of
// drafts 28.2 us, 25.2 in two tiles of 16.
template <typename T, int D>
static int launch_attend_by(const AttendParams& p, cudaStream_t stream) {
  if (p.prefix.head != nullptr)
    return p.cols <= 8 ? launch_attend<T, D, 1, false, true>(p, stream) : launch_attend<T, D, 2, false, true>(p, stream);
  if (p.cols <= 8)
    return p.picked ? launch_attend<T, D, 1, true>(p, stream) : launch_attend<T, D, 1, false>(p, stream);
  return p.picked ? launch_attend<T, D, 2, true>(p, stream) : launch_attend<T, D, 2, false>(p, stream);
}
static int tile_columns(int64_t cols) { return cols <= 8 ? 8 : 16; }

}  // namespace lf

extern "C" size_t lf_int4_workspace_clear_from(void) { return lf::partial_bytes(lf::sm_count()); }

extern "C" size_t lf_int4_workspace_bytes(int batch, int kv_heads, int n_q, int q_len, int head_dim) {
  if (batch <= 0 || kv_heads <= 0 || n_q < kv_heads || q_len <= 0 || head_dim <= 0) return 0;
  // one ticket per unit: the dense and the sparse call's units, whichever are more
  const int64_t group = n_q / kv_heads;
  const int64_t dense = (group * q_len + 15) / 16, sparse = (group + 15) / 16 * q_len;
  const int64_t units = static_cast<int64_t>(batch) * kv_heads * (dense > sparse ? dense : sparse);
  return lf::partial_bytes(lf::sm_count()) + (static_cast<size_t>(units) * 4 + 15) / 16 * 16;
}

namespace lf {

// Checks the arguments and fills p; launches nothing.
static int check_attend(const lf_int4_query* a, AttendParams& p) {
  LF_CHECK_ARG(a != nullptr, "lf_int4_attend: null arguments");
  const int bad = check_int4_pool("lf_int4_attend", a->pool, a->head_dim, p.pool);
  if (bad != LF_OK) return bad;
  LF_CHECK_ARG(a->q && a->lengths && a->out, "lf_int4_attend: null pointer");
  LF_CHECK_SUPPORTED(a->dtype == LF_F16 || a->dtype == LF_BF16, "lf_int4_attend: dtype %d (fp16 or bf16)", a->dtype);
  LF_CHECK_ARG(a->q_len > 0 && a->q_len <= 65535 && a->n_q > 0 && a->n_q % p.pool.kv_heads == 0,
               "lf_int4_attend: q_len %d, %d query heads on %d KV heads", a->q_len, a->n_q, p.pool.kv_heads);
  const bool sparse = a->picked != nullptr;
  LF_CHECK_ARG(!sparse || a->slots > 0, "lf_int4_attend: %d slots", a->slots);
  LF_CHECK_ARG(std::isfinite(a->scaling), "lf_int4_attend: scaling is not a finite number");
  LF_CHECK_ARG((reinterpret_cast<uintptr_t>(a->q) & 15) == 0 && (a->q_seq_stride | a->q_head_stride | a->q_tok_stride) % 8 == 0,
               "lf_int4_attend: query rows must be 16-byte aligned");
  LF_CHECK_ARG((reinterpret_cast<uintptr_t>(a->out) & 7) == 0 &&
                   (a->out_seq_stride | a->out_head_stride | a->out_tok_stride) % 4 == 0,
               "lf_int4_attend: output rows must be 8-byte aligned");
  const int64_t group = a->n_q / p.pool.kv_heads;
  const int64_t rows = sparse ? static_cast<int64_t>(p.pool.batch) * a->q_len : p.pool.batch;
  const int64_t cols = sparse ? group : group * a->q_len;
  const int64_t per_tile = tile_columns(cols), col_tiles = (cols + per_tile - 1) / per_tile;
  const int64_t pages = sparse ? a->slots : p.pool.table_width;
  LF_CHECK_SUPPORTED(rows * p.pool.kv_heads <= (1 << 30) / (pages + kUnitCost) / col_tiles && cols <= (1 << 30),
                     "lf_int4_attend: %d sequences of %lld pages are too many for one call", p.pool.batch,
                     static_cast<long long>(pages));
  p.sms = sm_count();
  if (p.sms <= 0) {
    set_error("lf_int4_attend: the current device's SMs cannot be counted");
    return LF_ERR_CUDA;
  }
  LF_CHECK_ARG(a->workspace && (reinterpret_cast<uintptr_t>(a->workspace) & 15) == 0 &&
                   a->workspace_bytes >= lf_int4_workspace_bytes(p.pool.batch, p.pool.kv_heads, a->n_q, a->q_len, a->head_dim),
               "lf_int4_attend: workspace of %zu bytes is missing, misaligned or too small", a->workspace_bytes);
  p.q = a->q;
  p.q_seq = a->q_seq_stride;
  p.q_head = a->q_head_stride;
  p.q_tok = a->q_tok_stride;
  p.q_len = a->q_len;
  p.group = static_cast<int>(group);
  p.rows = static_cast<int>(rows);
  p.cols = static_cast<int>(cols);
  p.col_tiles = static_cast<int>(col_tiles);
  p.lengths = a->lengths;
  p.counts = a->counts;
  p.picked = a->picked;
  p.slots = a->slots;
  p.scale_log2 = a->scaling * 1.4426950408889634f;
  p.out = a->out;
  p.out_seq = a->out_seq_stride;
  p.out_head = a->out_head_stride;
  p.out_tok = a->out_tok_stride;
  p.partials = static_cast<float*>(a->workspace);
  p.tickets = reinterpret_cast<uint32_t*>(static_cast<char*>(a->workspace) + partial_bytes(p.sms));
  p.status = a->status;
  p.prefix = PrefixPlan{};
  return LF_OK;
}

static int launch_attend(const lf_int4_query* a, const AttendParams& p, lf_stream_t stream) {
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (a->dtype == LF_F16) return a->head_dim == 128 ? launch_attend_by<__half, 128>(p, s) : launch_attend_by<__half, 64>(p, s);
  return a->head_dim == 128 ? launch_attend_by<__nv_bfloat16, 128>(p, s) : launch_attend_by<__nv_bfloat16, 64>(p, s);
}

int check_int4_attend(const lf_int4_query* a) {
  AttendParams p;
  return check_attend(a, p);
}

int int4_attend_suffix(const lf_int4_query* a, const PrefixPlan& plan, cudaStream_t stream) {
  AttendParams p;
  const int bad = check_attend(a, p);
  if (bad != LF_OK) return bad;
  p.prefix = plan;
  return launch_attend(a, p, reinterpret_cast<lf_stream_t>(stream));
}

}  // namespace lf

extern "C" int lf_int4_attend(const lf_int4_query* a, lf_stream_t stream) {
  lf::AttendParams p;
  const int bad = lf::check_attend(a, p);
  return bad != LF_OK ? bad : lf::launch_attend(a, p, stream);
}

extern "C" int lf_int4_attend_sparse(const lf_int4_query* a, lf_stream_t stream) {
  lf::AttendParams p;
  int bad = lf::check_int4_select(a);
  if (bad == LF_OK) bad = lf::check_attend(a, p);
  if (bad == LF_OK) bad = lf::int4_select_pages(a, a->scaling < 0.0f ? -1.0f : 1.0f, reinterpret_cast<cudaStream_t>(stream));
  return bad != LF_OK ? bad : lf::launch_attend(a, p, stream);
}
