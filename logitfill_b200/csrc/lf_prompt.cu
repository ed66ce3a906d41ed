// Attention of whole prompts over their own tokens (lf_prompt_attend).
//
// Mathematics.  Row (token i, q-head) of a sequence: scores s_j = scaling q . k_j for j <= i,
//   out = sum_j 2^(c s_j - m) v_j / sum_j 2^(c s_j - m),  c = log2(e),
// in one pass over the Keys with a running maximum m and sum (fp32).  Scores are fp32 sums
// of exact products; a weight is rounded once to the Value's type for its product (2^-9
// bf16, 2^-12 fp16: as fine as the output), the sums stay in fp32.
//
// Tiles.  The q-heads of a KV head are packed into the rows: a query tile is 128 / group
// tokens times group heads, 128 rows at most, so that short prompts and drafts fill it too
// and a Key tile is read once for the group.  A CTA takes items of two query tiles and
// goes through the Key tiles (128 tokens) that they see, from the diagonal back to the
// start.  20 warps: two threads to a row of scores (16 warps), one warp each for the
// products, the TMA copies and the plan.  Shared memory holds the queries (2 tiles) and a
// ring of Key and Value tiles in the 128-byte swizzle; tensor memory both tiles' scores
// (128 columns, whose place the weights take) and outputs (D columns).
//   products   per step: outputs of the step before (weights from tensor memory times
//              Values), then scores (queries times Keys, both from shared memory), tile by
//              tile: one tile's products run beside the other's softmax;
//   softmax    scores to weights, see lf_flash.cuh; the output is rescaled only where the
//              maximum moved by more than 2^8; at the end the row is stored.
// Where a Key tile is seen in part, weights of 0 would still spread a NaN or an infinity
// among the Values behind: those tiles are scanned (scan_value), and an item that has one
// is done row by row (prompt_row), as are rows whose scores are too large for fp32's
// exponent arithmetic.
//
// Order of work.  The plan deals items out by falling cost over all sequences, from
// alternating ends, without atomics: results do not depend on timing.
//
// What bounds it.  4 x 4096 tokens, 28 heads on 4, D 128, bf16: 450 us, 1068 TFLOP/s, 64 %
// of the measured 1680; one prompt of 8192: 414 us, 1163 TFLOP/s, 69 % (replayed in a
// graph, with pauses; 3 % more on some GPUs; back to back under the power cap 526 and 486).
// A step of both tiles takes some 3700 cycles, 2048 of them products (tensor cores 49 % busy
// over the launch of one prompt of 4096, issue slots 48 %): the exponentials, 2048 cycles of
// the special function unit without the polynomial, the other instructions of the softmax
// and the hand-overs between the roles overlap in part only.  (When 8192 tokens took 446 us,
// the loop without any softmax took 377, and with its products cut to a quarter as well 237:
// hand-overs alone were over half of a step.)
#include <atomic>
#include <cmath>
#include <type_traits>

#include "lf_common.cuh"
#include "lf_flash.cuh"

namespace lf {

struct PromptParams {
  const void *q, *k, *v;
  void* out;
  int64_t q_seq, q_head, q_tok, k_seq, k_head, k_tok, v_seq, v_head, v_tok, o_seq, o_head, o_tok;
  const int32_t *starts, *counts;
  int32_t* status;
  float scale_log2;
  int batch, tokens, n_kv, group;
  int wide_out;  // out rows are 32-byte aligned
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
// What waits for the row meanwhile learns from `moved` that it comes on: a warp has 16 rows of
// some 0.2 us a key, which is more than the waits' limit from some hundred thousand keys on.
template <typename T, int D>
__device__ __forceinline__ void prompt_row(const T* q, const T* k, int64_t k_tok, const T* v, int64_t v_tok, int n, float scale_log2, T* out,
                                           volatile uint64_t* moved) {
  constexpr int kOwn = D / 32, kAhead = 4;
  const int d = (threadIdx.x & 31) * kOwn;
  // positive, so that -inf stays one; the difference to the maximum before the product
  const float c = fmaxf(fabsf(scale_log2), 1e-36f), sign = scale_log2 < 0.0f ? -1.0f : 1.0f;
  float qx[kOwn], acc[kOwn], top = -INFINITY, sum = 0.0f;
#pragma unroll
  for (int x = 0; x < kOwn; ++x) {
    qx[x] = Scalar<T>::load(q + d + x);
    acc[x] = 0.0f;
  }
  for (int j = 0; j < n; j += kAhead) {
    if (j % 4096 == 0 && (threadIdx.x & 31) == 0) *moved = sm100::globaltimer_ns();
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
      s[u] *= sign;
      if (j + u < n) now = fmaxf(now, s[u]);
    }
    const float base = now == -INFINITY ? 0.0f : now, fix = exp2f((top - base) * c);
    sum *= fix;
#pragma unroll
    for (int x = 0; x < kOwn; ++x) acc[x] *= fix;
    top = now;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (j + u >= n) break;
      const float w = exp2f((s[u] - base) * c);
      sum += w;
      const T* row = v + (j + u) * v_tok + d;
#pragma unroll
      for (int x = 0; x < kOwn; ++x) acc[x] = fmaf(w, Scalar<T>::load(row + x), acc[x]);
    }
  }
#pragma unroll
  for (int x = 0; x < kOwn; ++x) Scalar<T>::store(out + d + x, sum == 0.0f ? 0.0f : acc[x] / sum);
}

using namespace sm100;

// Shared memory and barriers of a CTA.
template <int D> struct PromptCfg {
  static constexpr int kTile = 128 * D * 2;                      // bytes of 128 rows
  static constexpr int kSlots = D == 128 ? 5 : 8;                // Key and Value tiles in flight
  static constexpr int kSmem = 2 * kTile + kSlots * kTile + 3072;  // with what the roles share, and room to align
  static constexpr int kO = 256;                                 // TMEM columns: scores of both tiles, then outputs
};
constexpr int kPromptThreads = 640;
// Registers a thread: 96 at launch, then split between the softmax, whose 64 scores stay in
// registers, and the others.
constexpr int kLaunchRegs = 96, kSoftmaxRegs = 104, kOtherRegs = 64;
static_assert(512 * kSoftmaxRegs + 128 * kOtherRegs <= kPromptThreads * kLaunchRegs, "more registers than the block has");
// Of every 8 pairs of exponentials, those by the polynomial.  8192 tokens, 28 heads on 4,
// D 128: none 420 us, two 414, three 418.
constexpr int kPolyPairs = 2;
constexpr int kMmaWarp = 16, kLoadWarp = 17, kPlanWarp = 18;

// A piece of work: two query tiles of one KV head of one sequence.
struct PromptItem {
  int b, h;        // b < 0: no more
  int tok;         // first token of the first tile
  int tokens, rows;
  int first;       // row of the sequence's first token
  int n[2];        // Key tiles that each query tile sees
};

struct PromptShared {
  uint64_t kv_full[8], kv_empty[8], q_full, q_empty, s_full[2], p_early[2], p_ready[2], met[2], o_done[2], item_full[2], item_empty[2], last;
  PromptItem item[2];
  int bad[2];      // a Value that not all rows of a masked tile see is not finite
  Waits waits;
  uint32_t tmem;
  alignas(128) float told[2][2][128];  // between the two threads of a row
};

// 32 bytes of a row: one store where rows are 32-byte aligned (a whole sector by one lane).
template <typename T> __device__ __forceinline__ void store_row(T* at, const uint32_t (&w)[8], int wide) {
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
                 "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  } else {
    *reinterpret_cast<uint4*>(at) = make_uint4(w[0], w[1], w[2], w[3]);
    *reinterpret_cast<uint4*>(at + 8) = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

// A weight of 0 does not keep a NaN or an infinity out of a product.  So of a Value tile
// that some row sees in part, the 256 threads of a query tile zero the rows behind the
// sequence, and a number that is not finite is reported: it sends the item to prompt_row.
template <typename T, int D> __device__ __forceinline__ bool scan_value(uint8_t* tile, int live) {
  uint32_t seen = 0;
#pragma unroll
  for (int x = 0; x < D / 16; ++x) {
    const int i = (threadIdx.x & 255) + 256 * x;  // 16 bytes; 8 of them a row, 1024 a half
    uint4* at = reinterpret_cast<uint4*>(tile) + i;
    const uint4 y = *at;
    if (i % 1024 / 8 >= live) {  // (the other query tile's threads may have done it: then it is only read)
      if ((y.x | y.y | y.z | y.w) != 0) *at = make_uint4(0, 0, 0, 0);
    } else {
      // an exponent of all ones carries into the sign's place
      constexpr uint32_t kOne = std::is_same<T, __half>::value ? 0x04000400u : 0x00800080u;
      seen |= ((y.x & 0x7FFF7FFFu) + kOne) | ((y.y & 0x7FFF7FFFu) + kOne) | ((y.z & 0x7FFF7FFFu) + kOne) | ((y.w & 0x7FFF7FFFu) + kOne);
    }
  }
  fence_proxy_async_smem();
  return (seen & 0x80008000u) != 0;
}

// Whether some row of the query tile that begins at token t0 does not see all of Key tile j.
__device__ __forceinline__ bool tile_masked(int t0, int j) { return (j + 1) * 128 > t0 + 1; }

template <typename T, int D>
__global__ void __launch_bounds__(kPromptThreads, 1)
    prompt_kernel(const __grid_constant__ PromptParams p, const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                  const __grid_constant__ CUtensorMap v_map) {
  using C = PromptCfg<D>;
  constexpr bool kBf16 = !std::is_same<T, __half>::value;
  constexpr int kHalves = D / 64, kSlots = C::kSlots;
  extern __shared__ __align__(1024) uint8_t dynamic[];
  const uint32_t base = smem_u32(dynamic), ring = base + 2 * C::kTile;
  uint8_t* ring_ptr = dynamic + 2 * C::kTile;
  PromptShared& sh = *reinterpret_cast<PromptShared*>(ring_ptr + kSlots * C::kTile);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int per_tile = 128 / p.group;  // tokens of a query tile

  if (warp == kMmaWarp) {
    tmem_alloc(&sh.tmem, 512);
    tmem_relinquish();
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&sh.kv_full[i], 1);
      mbar_init(&sh.kv_empty[i], 1);
    }
    mbar_init(&sh.q_full, 1);
    mbar_init(&sh.q_empty, 1);
    mbar_init(&sh.last, 1);
    for (int t = 0; t < 2; ++t) {
      mbar_init(&sh.s_full[t], 1);
      mbar_init(&sh.p_early[t], 8);
      mbar_init(&sh.p_ready[t], 8);
      mbar_init(&sh.met[t], 8);
      mbar_init(&sh.o_done[t], 1);
      mbar_init(&sh.item_full[t], 1);
      mbar_init(&sh.item_empty[t], 18);
    }
    sh.waits.moved = 0;
    sh.waits.stop = 0;
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *const_cast<volatile uint32_t*>(&sh.tmem), 0);
  grid_dep_wait();

  auto wait = [&](uint64_t* bar, uint32_t parity) { return warp_wait<true>(bar, parity, &sh.waits); };
  // The next item (number n of this CTA), copied from the plan's slot.
  auto take = [&](uint32_t n, PromptItem& it) -> bool {
    if (!wait(&sh.item_full[n & 1], (n >> 1) & 1)) return false;
    it = sh.item[n & 1];
    return it.b >= 0;
  };
  auto give = [&](uint32_t n) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.item_empty[n & 1]);
  };

  if (warp == kPlanWarp) {
    // ---------------------------------------------------------------- plan
    fewer_registers<kOtherRegs>();
    // Items in the order of falling cost: by their number of tokens before, over all
    // sequences (a padded sequence's rows behind its tokens among them, which cost little);
    // a CTA takes them from alternating ends of rounds as wide as the grid.
    const int span = 2 * per_tile;
    auto pairs_of = [&](int b) { return (prompt_span(p, b).rows + span - 1) / span; };
    // Items of one KV head at level x or above, over all sequences (64 bits: starts may be anything).
    auto above = [&](int x) -> int64_t {
      int64_t n = 0;
      for (int b = lane; b < p.batch; b += 32) n += max(0, pairs_of(b) - x);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
      return n;
    };
    int most = 0;
    for (int b = lane; b < p.batch; b += 32) most = max(most, pairs_of(b));
    most = __reduce_max_sync(0xffffffffu, most);
    const int64_t total = above(0) * p.n_kv;
    // The level of the last item, the level's first item and the next one's, and how far into
    // the sequences its search went, with how many of the level it passed: items come in
    // order, so none is searched from the start again.  (65000 sequences of one token, 8 KV
    // heads: 1315 ms so, by the square of their number, and 11 this way.)
    int low = 0, b0 = 0, passed = 0;
    int64_t level_first = 0, level_end = 0;
    uint32_t n = 0;
    for (int64_t round = 0;; ++round, ++n) {
      if (n >= 2 && !wait(&sh.item_empty[n & 1], ((n >> 1) & 1) ^ 1)) break;
      const int64_t x = round * gridDim.x + ((round & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
      PromptItem it;
      it.b = -1;
      if (x < total) {
        if (x >= level_end) {
          int high = most - 1;  // the level: the largest with more than x items at or above it
          low = 0;
          while (low < high) {
            const int mid = (low + high + 1) >> 1;
            if (above(mid) * p.n_kv > x) low = mid; else high = mid - 1;
          }
          level_first = low + 1 < most ? above(low + 1) * p.n_kv : 0;
          level_end = low > 0 ? above(low) * p.n_kv : total;
          b0 = 0;
          passed = 0;
        }
        const int64_t y = x - level_first;
        const int rank = static_cast<int>(y / p.n_kv);  // among the level's sequences
        it.h = static_cast<int>(y - static_cast<int64_t>(rank) * p.n_kv);
        for (; b0 < p.batch; b0 += 32) {
          const uint32_t has = __ballot_sync(0xffffffffu, b0 + lane < p.batch && pairs_of(b0 + lane) > low);
          if (rank - passed < __popc(has)) {
            it.b = b0 + __fns(has, 0, rank - passed + 1);
            break;
          }
          passed += __popc(has);
        }
        const PromptSpan s = prompt_span(p, max(it.b, 0));
        it.first = static_cast<int>(s.first);
        it.tokens = s.tokens;
        it.rows = s.rows;
        it.tok = low * span;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int t0 = it.tok + t * per_tile;
          it.n[t] = t0 < s.tokens ? (min(t0 + per_tile, s.tokens) - 1) / 128 + 1 : 0;
        }
      }
      if (lane == 0) {
        sh.item[n & 1] = it;
        sh.bad[n & 1] = 0;
        mbar_arrive(&sh.item_full[n & 1]);
      }
      __syncwarp();
      if (it.b < 0) break;
    }
  } else if (warp == kLoadWarp) {
    // ---------------------------------------------------------------- copies
    fewer_registers<kOtherRegs>();
    uint32_t load = 0, n_q = 0;  // tiles and query pairs copied so far
    if (lane < 3) prefetch_map(lane == 0 ? &q_map : lane == 1 ? &k_map : &v_map);
    PromptItem it;
    bool ok = true;
    for (uint32_t n = 0; ok && take(n, it); ++n) {
      give(n);
      const int steps = max(it.n[0], it.n[1]);
      if (steps == 0) continue;
      if (n_q > 0 && !(ok = wait(&sh.q_empty, (n_q - 1) & 1))) break;
      ++n_q;
      if (elect_one()) {
        mbar_arrive_expect_tx(&sh.q_full, 2 * kHalves * per_tile * p.group * 128);
        for (int t = 0; t < 2; ++t)
          for (int c = 0; c < kHalves; ++c)
            tma_load_4d(base + t * C::kTile + c * kHalfBytes, &q_map, 64 * c, it.h * p.group, it.first + it.tok + t * per_tile,
                        p.starts != nullptr ? 0 : it.b, &sh.q_full);
      }
      __syncwarp();
      for (int i = 0; i < 2 * steps; ++i, ++load) {
        const int slot = load % kSlots, j = steps - 1 - (i >> 1);
        if (load >= kSlots && !(ok = wait(&sh.kv_empty[slot], (load / kSlots - 1) & 1))) break;
        if (elect_one()) {
          mbar_arrive_expect_tx(&sh.kv_full[slot], C::kTile);
          for (int c = 0; c < kHalves; ++c)
            tma_load_4d(ring + slot * C::kTile + c * kHalfBytes, (i & 1) ? &v_map : &k_map, 64 * c, it.first + 128 * j, it.h,
                        p.starts != nullptr ? 0 : it.b, &sh.kv_full[slot]);
        }
        __syncwarp();
      }
    }
    // No copy outlives the CTA (after a wait that gave up: as far as the limit goes).
    for (int i = 0; i < kSlots; ++i) {
      const uint32_t used = load / kSlots + (static_cast<uint32_t>(i) < load % kSlots ? 1 : 0);
      if (used != 0) mbar_wait_bounded(&sh.kv_full[i], (used - 1) & 1, kTileWaitNs);
    }
    if (n_q > 0) mbar_wait_bounded(&sh.q_full, (n_q - 1) & 1, kTileWaitNs);
  } else if (warp == kMmaWarp) {
    // ---------------------------------------------------------------- products
    fewer_registers<kOtherRegs>();
    // Step s of the CTA: scores of Key tile (load 2 s) for both query tiles, after the
    // output product of step s - 1 (Value tile, load 2 s - 1), tile by tile: while the
    // softmax of one tile runs, the tensor core works for the other.  The only commits are
    // the scores' and an item's last outputs' (each takes this warp over 100 cycles): what
    // else a tile's scores say is done, the softmax passes on.
    const uint32_t idesc_s = idesc_16(kBf16, 128, 128, false, p.scale_log2 < 0.0f), idesc_o = idesc_16(kBf16, 128, D, true, false);
    uint32_t step = 0, n_q = 0, made[2] = {0, 0};
    bool had[2] = {false, false}, fresh[2] = {false, false}, ends = false;
    auto output = [&](int t) -> bool {  // of the step before
      if (!had[t]) return true;
      const uint32_t load = 2 * step - 1, slot = load % kSlots;
      if (!wait(&sh.kv_full[slot], (load / kSlots) & 1)) return false;
      for (int part = 0; part < 2; ++part) {
        if (!wait(part == 0 ? &sh.p_early[t] : &sh.p_ready[t], made[t] & 1)) return false;
        tc_fence_after();
        issue_outputs<1>(tmem + C::kO + t * D, tmem + 128 * t, ring + slot * C::kTile, idesc_o, part, fresh[t], ends && part == 1 ? &sh.o_done[t] : nullptr);
      }
      ++made[t];
      return true;
    };
    auto scores = [&](int t) {
      tc_fence_after();
      issue_scores<D>(tmem + 128 * t, base + t * C::kTile, ring + 2 * step % kSlots * C::kTile, idesc_s, false, &sh.s_full[t]);
    };
    PromptItem it;
    bool ok = true;
    for (uint32_t n = 0; ok && take(n, it); ++n) {
      give(n);
      const int steps = max(it.n[0], it.n[1]);
      if (steps == 0) {  // (nothing later may wait for an item to come: the softmax needs these to let it go)
        if (!(ok = output(0) && output(1))) break;
        had[0] = had[1] = false;
      }
      for (int j = steps - 1; j >= 0; --j, ++step) {
        const bool now[2] = {j < it.n[0], j < it.n[1]};
        if (j == steps - 1) {  // the outputs of the item before do not wait for this one's queries
          if (step > 0 && !(ok = output(0) && output(1))) break;
          if (!(ok = wait(&sh.q_full, n_q++ & 1) && wait(&sh.kv_full[2 * step % kSlots], (2 * step / kSlots) & 1))) break;
          if (now[0]) scores(0);
          if (now[1]) scores(1);
        } else {
          if (!(ok = wait(&sh.kv_full[2 * step % kSlots], (2 * step / kSlots) & 1))) break;
          if (!(ok = output(0))) break;
          if (now[0]) scores(0);
          if (!(ok = output(1))) break;
          if (now[1]) scores(1);
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          had[t] = now[t];
          fresh[t] = j == it.n[t] - 1;
        }
        ends = j == 0;
      }
    }
    if (ok && step > 0 && *const_cast<volatile int*>(&sh.waits.stop) == 0 && output(0)) output(1);  // the last step's
  } else if (warp < kMmaWarp) {
    // ---------------------------------------------------------------- softmax, one tile a warpgroup
    more_registers<kSoftmaxRegs>();
    const int t = warp >> 3, half = (warp >> 2) & 1, r = (warp & 3) * 32 + lane;
    const uint32_t mine = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16), tm_s = mine + 128 * t, tm_o = mine + C::kO + t * D;
    Pair pair = {&sh.told[t][half][r], &sh.told[t][half ^ 1][r], &sh.met[t], 0};
    // positive, so that a masked score's -inf stays one; a negative scaling negates the queries in the product
    const float c = fmaxf(fabsf(p.scale_log2), 1e-36f);
    uint32_t count = 0, items = 0, before = 0;  // score tiles and items with some so far, steps of the items before
    const bool frees = (warp & 7) == 0;
    bool ok = true;
    for (uint32_t n = 0; ok && wait(&sh.item_full[n & 1], (n >> 1) & 1); ++n) {
      volatile const PromptItem& it = sh.item[n & 1];  // (read where it is needed: registers are short here)
      if (it.b < 0) break;
      const int steps = it.n[t], all = max(it.n[0], it.n[1]), t0 = it.tok + t * per_tile;
      RowState st = no_scores();
      {
        const int sees = min(t0 + r / p.group + 1, it.tokens);
        for (int j = steps - 1; j >= 0; --j, ++count) {
          if (!(ok = wait(&sh.s_full[t], count & 1))) break;
          tc_fence_after();
          const uint32_t load = 2 * (before + all - 1 - j);  // of the Key tile; the Value tile is the next
          if (frees && (t == 1 || j >= it.n[1])) {
            // The step's last scores are done, and with them all products before: the Key
            // tile is free, the Value tile of the step before, after the last step the queries.
            arrive_once(&sh.kv_empty[load % kSlots]);
            if (load > 0) arrive_once(&sh.kv_empty[(load - 1) % kSlots]);
            if (j == 0) arrive_once(&sh.q_empty);
          }
          if (!(ok = soften_tile<T, D, kPolyPairs, 1>(tm_s, tm_o, half, c, tile_masked(t0, j), sees - 128 * j, j == steps - 1, st, pair, &sh.p_early[t], &sh.p_ready[t], wait, [&] {
                                         const uint32_t slot = (load + 1) % kSlots;
                                         if (!wait(&sh.kv_full[slot], ((load + 1) / kSlots) & 1)) return false;
                                         if (scan_value<T, D>(ring_ptr + slot * C::kTile, min(128, it.tokens - 128 * j))) sh.bad[n & 1] = 1;
                                         return true;
                                       })))
            break;
        }
      }
      if (!ok) break;
      before += all;
      const int in_tile = r / p.group, head = r - in_tile * p.group, token = t0 + in_tile;
      const bool stored = in_tile < per_tile && token < it.rows;
      T* out = static_cast<T*>(p.out) + it.b * p.o_seq + (static_cast<int64_t>(it.first) + token) * p.o_tok +
               (it.h * p.group + head) * p.o_head + D / 2 * half;
      if (steps > 0) {
        if (!(ok = wait(&sh.o_done[t], items++ & 1))) break;
        if (!(ok = join_sums(st, pair, wait))) break;
        tc_fence_after();
      }
      if (steps > 0 && (*const_cast<volatile int*>(&sh.bad[n & 1]) != 0 || __any_sync(0xffffffffu, st.large && stored && token < it.tokens))) {
        const T* k = static_cast<const T*>(p.k) + it.b * p.k_seq + it.first * p.k_tok + it.h * p.k_head;
        const T* v = static_cast<const T*>(p.v) + it.b * p.v_seq + it.first * p.v_tok + it.h * p.v_head;
        for (int i = half; i < 32; i += 2) {
          const int x = (warp & 3) * 32 + i, tok = t0 + x / p.group, hd = it.h * p.group + x % p.group;
          if (x >= per_tile * p.group || tok >= it.rows) break;
          const int64_t row = static_cast<int64_t>(it.first) + tok;
          prompt_row<T, D>(static_cast<const T*>(p.q) + it.b * p.q_seq + row * p.q_tok + hd * p.q_head, k, p.k_tok, v, p.v_tok,
                           tok < it.tokens ? tok + 1 : 0, p.scale_log2, static_cast<T*>(p.out) + it.b * p.o_seq + row * p.o_tok + hd * p.o_head, &sh.waits.moved);
        }
      } else {
        // else 0: a row behind the sequence, or one of no score above -inf
        const bool live = steps > 0 && token < it.tokens && !st.empty();
        const float inv = 1.0f / st.sum;
#pragma unroll 1
        for (int i = 0; i < D / 32; ++i) {
          float o[16];
          if (steps > 0) tmem_ld_x16(tm_o + D / 2 * half + 16 * i, o);
          if (stored) {
            uint32_t w[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) w[x] = live ? pack_two<T>(o[2 * x] * inv, o[2 * x + 1] * inv) : 0u;
            store_row(out + 16 * i, w, p.wide_out);
          }
        }
      }
      tc_fence_before();
      give(n);
    }
  } else {
    fewer_registers<kOtherRegs>();  // (of a warpgroup, all warps at once)
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
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

// cuTensorMapEncodeTiled of the driver, found once.
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeTiled encode_tiled() {
  static std::atomic<void*> known{nullptr};
  void* f = known.load(std::memory_order_acquire);
  if (f == nullptr) {
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess)
      return nullptr;
    known.store(f, std::memory_order_release);
  }
  return reinterpret_cast<EncodeTiled>(f);
}
// A map of [..] 16-bit elements: 64 channels wide boxes in the 128-byte swizzle; extents,
// strides (elements) and box of the three dimensions over the channels.
static bool make_map(CUtensorMap* map, const void* at, bool bf16, int D, const int64_t (&extent)[3], const int64_t (&stride)[3],
                     const int (&box)[3]) {
  const EncodeTiled encode = encode_tiled();
  if (encode == nullptr) return false;
  cuuint64_t dims[4] = {static_cast<cuuint64_t>(D)}, strides[3];
  cuuint32_t boxes[4] = {64}, ones[4] = {1, 1, 1, 1};
  for (int i = 0; i < 3; ++i) {
    dims[i + 1] = static_cast<cuuint64_t>(extent[i]);
    strides[i] = static_cast<cuuint64_t>(extent[i] > 1 ? stride[i] : D) * 2;
    boxes[i + 1] = static_cast<cuuint32_t>(box[i]);
  }
  return encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(at), dims, strides, boxes,
                ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T>
static const void* prompt_kernel_of(int head_dim) {
  return head_dim == 128 ? reinterpret_cast<const void*>(prompt_kernel<T, 128>) : reinterpret_cast<const void*>(prompt_kernel<T, 64>);
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
  p.n_kv = a->n_kv;
  p.group = a->n_q / a->n_kv;
  p.wide_out = reinterpret_cast<uintptr_t>(a->out) % 32 == 0 && (p.o_seq | p.o_head | p.o_tok) % 16 == 0;
  const int sms = sm_count();
  if (sms <= 0) {
    set_error("lf_prompt_attend: the current device's SMs cannot be counted");
    return LF_ERR_CUDA;
  }
  const bool packed = a->starts != nullptr, bf16 = a->dtype == LF_BF16;
  const int per_tile = 128 / p.group, batches = packed ? 1 : a->batch;
  CUtensorMap q_map, k_map, v_map;
  if (!make_map(&q_map, a->q, bf16, a->head_dim, {a->n_q, a->tokens, batches}, {p.q_head, p.q_tok, p.q_seq}, {p.group, per_tile, 1}) ||
      !make_map(&k_map, a->k, bf16, a->head_dim, {a->tokens, a->n_kv, batches}, {p.k_tok, p.k_head, p.k_seq}, {128, 1, 1}) ||
      !make_map(&v_map, a->v, bf16, a->head_dim, {a->tokens, a->n_kv, batches}, {p.v_tok, p.v_head, p.v_seq}, {128, 1, 1})) {
    set_error("lf_prompt_attend: the driver makes no tensor map of these rows");
    return LF_ERR_CUDA;
  }
  // No more CTAs than items there can be (of sequences that do not overlap).
  const int64_t span = 2 * per_tile;
  const int64_t items = (packed ? a->tokens / span + a->batch : (a->tokens + span - 1) / span * a->batch) * a->n_kv;
  const void* kern = bf16 ? prompt_kernel_of<__nv_bfloat16>(a->head_dim) : prompt_kernel_of<__half>(a->head_dim);
  const int smem = a->head_dim == 128 ? PromptCfg<128>::kSmem : PromptCfg<64>::kSmem;
  cudaError_t err = raise_smem_limit(kern, smem, true);
  if (err != cudaSuccess) {
    set_error("lf_prompt_attend: %s", cudaGetErrorString(err));
    return LF_ERR_CUDA;
  }
  if (!launched_with(kern, kLaunchRegs)) {
    set_error("lf_prompt_attend: the kernel was not built for %d registers a thread", kLaunchRegs);
    return LF_ERR_LAUNCH;
  }
  void* args[] = {&p, &q_map, &k_map, &v_map};
  err = launch_programmatic(kern, dim3(static_cast<unsigned>(items < sms ? items : sms)), dim3(kPromptThreads), smem,
                            reinterpret_cast<cudaStream_t>(stream), args);
  if (err != cudaSuccess) {
    set_error("lf_prompt_attend: %s", cudaGetErrorString(err));
    return LF_ERR_LAUNCH;
  }
  return launch_status("lf_prompt_attend");
}
