// Rotary positions of a step's queries and Keys (lf_rotary_embed).
//
// Mathematics.  A pair (x, y) of a token at position p turns by the angle a = 2 pi f p:
//   x' = m (x cos a - y sin a),  y' = m (y cos a + x sin a).
// In fp32 the angle of a far position is off by more than the output's rounding: at
// p = 131072 and f = 1 / (2 pi), fp32 steps are 2^-7 radians.  Here f is a whole number
// of 2^-64 turns, and p f modulo one turn is one wrapping 64-bit product: exact for any
// position, up to f's own rounding (2^-65 turns a position).  The phase splits into the
// nearest quarter turn and a rest of at most 1/8 turn, kept to 2^-32 turns, and the rest
// goes through sincospif.
//
// What bounds it: every element is read and written once and the angles are shared by a
// token's heads, so a large call is bound by HBM.  A thread keeps the cosines and sines
// of its pairs (16 bytes of channels and their partners) in registers and walks over the
// token's heads, four in flight.  The block's angles are worked out once, each by one
// thread, while the first loads are on their way, and handed over in shared memory: when
// that brought 16384 tokens of 32 heads, D 128, to 57 us, each thread working out its own had
// taken 90 (the arithmetic of 8 angles for 4 heads).  In small calls there are as many threads to a
// token as it has heads, so that each makes one round of loads.  16384 tokens of 32 heads, D
// 128, bf16: 46 us replayed, 5.9 TB/s, 90 % of a plain copy's rate (D 256: 6.3 TB/s; fp32: 6.4);
// 16 tokens: 2.5 us replayed, 5.3 from Python, the host's issue.
#include <cmath>

#include "lf_common.cuh"

namespace lf {

struct RotaryParams {
  const void *q, *k;
  void *q_out, *k_out;
  int64_t q_seq, q_head, q_tok, qo_seq, qo_head, qo_tok;
  int64_t k_seq, k_head, k_tok, ko_seq, ko_head, ko_tok;
  const int64_t* freqs;
  const void* positions;
  int64_t pos_seq, pos_tok;
  const int32_t* start;
  float magnitude, sign;
  int positions_64, part, tokens, n_q, heads;
  int64_t total;                      // tokens of all sequences
  int per_row, head_lanes, per_block;  // items of a head's row, threads to a token and item, tokens of a block
};

constexpr int kRotaryAhead = 4;

// Threads of a block.  In a large call small blocks wait less at their barrier for the angles:
// 16384 tokens of 32 heads, D 128, bf16, take 46 us with 64 threads and 52 with 256, 600
// tokens 3.5 and 4.9, 300 (a quarter of the GPU's threads) 3.2 with either.  A small call
// wants a token's heads in one block: 16 tokens take 2.5 us with 256 threads and 2.9 with 64.
// Rows of single elements (up to 255 items) need 256.  (Replayed 20 or 40 times in a graph.)
constexpr int kSmallBlock = 64, kLargeBlock = 256;

constexpr int64_t kRotaryFill = 148 * 2048;  // threads that a B200 holds at once

template <typename T, int N> struct alignas(sizeof(T) * N) Pack { T x[N]; };

// Cosine and sine of 2 pi phase / 2^64.
__device__ __forceinline__ void turn_of(uint64_t phase, float& c, float& s) {
  const uint64_t quarter = (phase + (1ull << 61)) >> 62;
  const int32_t rest = static_cast<int32_t>((phase - (quarter << 62)) >> 32);  // of 2^-32 turns, |rest| <= 2^29
  float rs, rc;
  sincospif(static_cast<float>(rest) * 0x1p-31f, &rs, &rc);
  const bool swap = quarter & 1, minus_s = quarter & 2, minus_c = (quarter + 1) & 2;
  c = swap ? rs : rc;
  s = swap ? rc : rs;
  c = minus_c ? -c : c;
  s = minus_s ? -s : s;
}

// Sequence and token of a token of all sequences.  (A 64-bit division is some 100
// instructions: as many as the rest of what a thread does for a head.)
__device__ __forceinline__ void split(const RotaryParams& p, int64_t token, int64_t& b, int64_t& t) {
  if (p.total <= INT32_MAX) {
    b = static_cast<uint32_t>(token) / static_cast<uint32_t>(p.tokens);
    t = static_cast<uint32_t>(token) - static_cast<uint32_t>(b) * p.tokens;
  } else {
    b = token / p.tokens;
    t = token - b * p.tokens;
  }
}

// Pairs (u, w) turned: two of them at a time.
__device__ __forceinline__ void turn_two(float2& u, float2& w, float2 c, float2 s) {
  const float2 a = __fmul2_rn(w, make_float2(-s.x, -s.y)), b = __fmul2_rn(u, s);
  u = __ffma2_rn(u, c, a);
  w = __ffma2_rn(w, c, b);
}
// N pairs, of vectors x and y (half pairs).
template <typename T, int N>
__device__ __forceinline__ void turn_halves(Pack<T, N>& x, Pack<T, N>& y, const float (&c)[N], const float (&s)[N]) {
  if constexpr (N == 1) {
    const float u = Scalar<T>::load(x.x), w = Scalar<T>::load(y.x);
    Scalar<T>::store(x.x, fmaf(u, c[0], -w * s[0]));
    Scalar<T>::store(y.x, fmaf(w, c[0], u * s[0]));
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      float2 u, w;
      if constexpr (sizeof(T) == 4) {
        u = make_float2(x.x[i], x.x[i + 1]);
        w = make_float2(y.x[i], y.x[i + 1]);
      } else {
        u = unpack_two<T>(reinterpret_cast<uint32_t*>(x.x)[i / 2]);
        w = unpack_two<T>(reinterpret_cast<uint32_t*>(y.x)[i / 2]);
      }
      turn_two(u, w, make_float2(c[i], c[i + 1]), make_float2(s[i], s[i + 1]));
      if constexpr (sizeof(T) == 4) {
        x.x[i] = u.x;
        x.x[i + 1] = u.y;
        y.x[i] = w.x;
        y.x[i + 1] = w.y;
      } else {
        reinterpret_cast<uint32_t*>(x.x)[i / 2] = pack_two<T>(u.x, u.y);
        reinterpret_cast<uint32_t*>(y.x)[i / 2] = pack_two<T>(w.x, w.y);
      }
    }
  }
}
// N / 2 pairs of one vector (adjacent pairs).
template <typename T, int N>
__device__ __forceinline__ void turn_adjacent(Pack<T, N>& x, const float (&c)[N / 2], const float (&s)[N / 2]) {
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    float2 u;
    if constexpr (sizeof(T) == 4)
      u = make_float2(x.x[2 * i], x.x[2 * i + 1]);
    else
      u = unpack_two<T>(reinterpret_cast<uint32_t*>(x.x)[i]);
    u = make_float2(fmaf(u.x, c[i], -u.y * s[i]), fmaf(u.y, c[i], u.x * s[i]));
    if constexpr (sizeof(T) == 4) {
      x.x[2 * i] = u.x;
      x.x[2 * i + 1] = u.y;
    } else {
      reinterpret_cast<uint32_t*>(x.x)[i] = pack_two<T>(u.x, u.y);
    }
  }
}

// N elements a vector.  Half pairs: item v < part / 2 / N is the vectors at N v and N v +
// part / 2.  Adjacent pairs: item v < part / N is the vector at N v; for N = 1, item v <
// part / 2 is the elements at 2 v and 2 v + 1.  The items behind them are vectors of
// channels that are copied.
template <typename T, int N, bool kAdjacent>
__global__ void __launch_bounds__(kLargeBlock, 3) rotary_kernel(const __grid_constant__ RotaryParams p) {
  constexpr bool kInside = kAdjacent && N > 1;  // both channels of a pair in one vector
  constexpr int kPairs = kInside ? N / 2 : N;
  using Vec = Pack<T, N>;
  const int v = threadIdx.x % p.per_row, slot = threadIdx.x / p.per_row;
  const int first_head = slot % p.head_lanes, in_block = slot / p.head_lanes;
  const int64_t token = static_cast<int64_t>(blockIdx.x) * p.per_block + in_block;
  grid_dep_wait();
  const bool mine = in_block < p.per_block && token < p.total;
  int64_t b, t;
  split(p, token, b, t);
  const int turning = kInside ? p.part / N : p.part / 2 / N;
  const bool turns = v < turning;
  // The item's channel, and its partner's.
  const int at = !turns ? p.part + (v - turning) * N : kAdjacent && !kInside ? 2 * v : v * N;
  const int other = kAdjacent ? at + 1 : at + p.part / 2;
  // This thread's rows: of the queries from its first head on, then of the Keys.
  struct Rows {
    const T* in;
    T* out;
    int64_t in_step, out_step;
    int n;
  } rows[2];
  const int first_k = first_head < p.n_q ? first_head + (p.n_q - first_head + p.head_lanes - 1) / p.head_lanes * p.head_lanes - p.n_q
                                         : first_head - p.n_q;
  const int n_kv = p.heads - p.n_q;
  rows[0] = Rows{static_cast<const T*>(p.q) + b * p.q_seq + t * p.q_tok + first_head * p.q_head,
                 static_cast<T*>(p.q_out) + b * p.qo_seq + t * p.qo_tok + first_head * p.qo_head, p.head_lanes * p.q_head,
                 p.head_lanes * p.qo_head, mine && first_head < p.n_q ? (p.n_q - first_head + p.head_lanes - 1) / p.head_lanes : 0};
  rows[1] = Rows{static_cast<const T*>(p.k) + b * p.k_seq + t * p.k_tok + first_k * p.k_head,
                 static_cast<T*>(p.k_out) + b * p.ko_seq + t * p.ko_tok + first_k * p.ko_head, p.head_lanes * p.k_head,
                 p.head_lanes * p.ko_head, mine && first_k < n_kv ? (n_kv - first_k + p.head_lanes - 1) / p.head_lanes : 0};

  Vec x[kRotaryAhead], y[kRotaryAhead];
  auto load = [&](const Rows& r) {
#pragma unroll
    for (int j = 0; j < kRotaryAhead; ++j) {
      if (j >= r.n) break;
      x[j] = *reinterpret_cast<const Vec*>(r.in + j * r.in_step + at);
      if (!kInside && turns) y[j] = *reinterpret_cast<const Vec*>(r.in + j * r.in_step + other);
    }
  };
  const bool k_first = rows[0].n == 0;
  if (k_first)
    load(rows[1]);
  else
    load(rows[0]);

  // The block's tokens' angles, each by one thread.  Pair i of item v lies at place i *
  // turning + v of its token, so that a warp's reads do not meet in a bank.
  extern __shared__ float2 turn_s[];
  const int pairs = p.part / 2;
  for (int x = threadIdx.x; x < p.per_block * pairs; x += blockDim.x) {
    const int which = x / pairs, pair = x - which * pairs;
    const int64_t tok = static_cast<int64_t>(blockIdx.x) * p.per_block + which;
    if (tok >= p.total) break;
    int64_t bb, tt;
    split(p, tok, bb, tt);
    int64_t position;
    if (p.positions == nullptr)
      position = static_cast<int64_t>(p.start[bb]) + tt;
    else if (p.positions_64)
      position = static_cast<const int64_t*>(p.positions)[bb * p.pos_seq + tt * p.pos_tok];
    else
      position = static_cast<const int32_t*>(p.positions)[bb * p.pos_seq + tt * p.pos_tok];
    float c, s;
    turn_of(static_cast<uint64_t>(position) * static_cast<uint64_t>(p.freqs[pair]), c, s);
    turn_s[which * pairs + pair % kPairs * turning + pair / kPairs] = make_float2(c * p.magnitude, s * p.sign);
  }
  __syncthreads();
  if (!mine) return;
  float c[kPairs], s[kPairs];
  if (turns) {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const float2 y = turn_s[in_block * pairs + i * turning + v];
      c[i] = y.x;
      s[i] = y.y;
    }
  }
  bool loaded = true;
  auto go = [&](Rows r) {
    for (; r.n > 0; r.n -= kRotaryAhead, r.in += kRotaryAhead * r.in_step, r.out += kRotaryAhead * r.out_step) {
      if (!loaded) load(r);
      loaded = false;
#pragma unroll
      for (int j = 0; j < kRotaryAhead; ++j) {
        if (j >= r.n) break;
        if (turns) {
          if constexpr (kInside)
            turn_adjacent<T, N>(x[j], c, s);
          else
            turn_halves<T, N>(x[j], y[j], c, s);
          if (!kInside) *reinterpret_cast<Vec*>(r.out + j * r.out_step + other) = y[j];
        }
        *reinterpret_cast<Vec*>(r.out + j * r.out_step + at) = x[j];
      }
    }
  };
  go(rows[0]);
  go(rows[1]);
}

template <typename T>
static const void* rotary_kernel_of(bool adjacent, bool wide) {
  constexpr int kWide = 16 / sizeof(T);
  if (adjacent)
    return wide ? reinterpret_cast<const void*>(rotary_kernel<T, kWide, true>) : reinterpret_cast<const void*>(rotary_kernel<T, 1, true>);
  return wide ? reinterpret_cast<const void*>(rotary_kernel<T, kWide, false>) : reinterpret_cast<const void*>(rotary_kernel<T, 1, false>);
}

}  // namespace lf

extern "C" int lf_rotary_embed(const lf_rotary* a, lf_stream_t stream) {
  using namespace lf;
  LF_CHECK_ARG(a != nullptr, "lf_rotary_embed: null arguments");
  LF_CHECK_ARG(a->dtype == LF_F32 || a->dtype == LF_F16 || a->dtype == LF_BF16, "lf_rotary_embed: dtype %d", a->dtype);
  LF_CHECK_SUPPORTED(a->head_dim >= 2 && a->head_dim <= 256, "lf_rotary_embed: head_dim %d (2 to 256)", a->head_dim);
  LF_CHECK_ARG(a->part >= 2 && a->part <= a->head_dim && a->part % 2 == 0,
               "lf_rotary_embed: %d rotated channels of %d (an even number from 2 on)", a->part, a->head_dim);
  LF_CHECK_ARG(std::isfinite(a->magnitude), "lf_rotary_embed: magnitude is not a finite number");
  LF_CHECK_ARG(a->batch >= 0 && a->tokens >= 0 && a->n_q >= 0 && a->n_kv >= 0, "lf_rotary_embed: negative extent");
  LF_CHECK_SUPPORTED(a->n_q <= 65535 && a->n_kv <= 65535, "lf_rotary_embed: %d and %d heads (65535 at most)", a->n_q, a->n_kv);
  RotaryParams p;
  p.total = static_cast<int64_t>(a->batch) * a->tokens;
  p.heads = a->n_q + a->n_kv;
  if (p.total == 0 || p.heads == 0) return LF_OK;
  LF_CHECK_ARG((a->n_q == 0 || (a->q && a->q_out)) && (a->n_kv == 0 || (a->k && a->k_out)) && a->freqs && (a->positions || a->start),
               "lf_rotary_embed: null pointer");
  p.q = a->q;
  p.k = a->k;
  p.q_out = a->q_out;
  p.k_out = a->k_out;
  p.q_seq = a->q_seq_stride;
  p.q_head = a->q_head_stride;
  p.q_tok = a->q_tok_stride;
  p.qo_seq = a->q_out_seq_stride;
  p.qo_head = a->q_out_head_stride;
  p.qo_tok = a->q_out_tok_stride;
  p.k_seq = a->k_seq_stride;
  p.k_head = a->k_head_stride;
  p.k_tok = a->k_tok_stride;
  p.ko_seq = a->k_out_seq_stride;
  p.ko_head = a->k_out_head_stride;
  p.ko_tok = a->k_out_tok_stride;
  p.freqs = a->freqs;
  p.positions = a->positions;
  p.pos_seq = a->pos_seq_stride;
  p.pos_tok = a->pos_tok_stride;
  p.start = a->start;
  p.magnitude = a->magnitude;
  p.sign = a->transposed ? -a->magnitude : a->magnitude;
  p.positions_64 = a->positions_64;
  p.part = a->part;
  p.tokens = a->tokens;
  p.n_q = a->n_q;

  // Vectors of 16 bytes where every row, and the border between rotated halves and copied
  // channels, lies on such a boundary; else single elements.
  const int size = a->dtype == LF_F32 ? 4 : 2, lanes = 16 / size;
  uint64_t low = 0;
  if (a->n_q > 0)
    low |= reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->q_out) |
           static_cast<uint64_t>(p.q_seq | p.q_head | p.q_tok | p.qo_seq | p.qo_head | p.qo_tok) * size;
  if (a->n_kv > 0)
    low |= reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->k_out) |
           static_cast<uint64_t>(p.k_seq | p.k_head | p.k_tok | p.ko_seq | p.ko_head | p.ko_tok) * size;
  const int unit = a->interleaved ? a->part : a->part / 2;
  const bool wide = low % 16 == 0 && unit % lanes == 0 && a->head_dim % lanes == 0;
  p.per_row = wide ? (a->interleaved ? a->part : a->part / 2) / lanes + (a->head_dim - a->part) / lanes : a->head_dim - a->part / 2;

  // Threads to a token and item: as many as there are heads in a small call (a thread makes
  // one round of loads), down to one for each kRotaryAhead heads once the threads fill the
  // GPU.  16384 tokens, 32 heads, when that took 57 us: 59 with 8 heads to a thread, 61 with 16.
  int lanes_heads = p.heads;
  while (lanes_heads > 1 && static_cast<int64_t>(p.total) * p.per_row * lanes_heads > kRotaryFill && lanes_heads * kRotaryAhead > p.heads)
    lanes_heads = (lanes_heads + 1) / 2;
  const bool large = static_cast<int64_t>(p.total) * p.per_row * p.heads > kRotaryFill / 4;
  const int threads = wide && large ? kSmallBlock : kLargeBlock, slots = threads / p.per_row;
  p.head_lanes = lanes_heads < slots ? lanes_heads : slots;
  p.per_block = slots / p.head_lanes;
  const int64_t blocks = (p.total + p.per_block - 1) / p.per_block;
  LF_CHECK_SUPPORTED(blocks <= INT32_MAX, "lf_rotary_embed: %lld tokens are too many for one call", static_cast<long long>(p.total));
  const void* kern = a->dtype == LF_F32   ? rotary_kernel_of<float>(a->interleaved != 0, wide)
                     : a->dtype == LF_F16 ? rotary_kernel_of<__half>(a->interleaved != 0, wide)
                                          : rotary_kernel_of<__nv_bfloat16>(a->interleaved != 0, wide);
  void* args[] = {&p};
  const cudaError_t err = launch_programmatic(kern, dim3(static_cast<unsigned>(blocks)), dim3(threads),
                                              static_cast<size_t>(p.per_block) * (p.part / 2) * sizeof(float2),
                                              reinterpret_cast<cudaStream_t>(stream), args);
  if (err != cudaSuccess) {
    set_error("lf_rotary_embed: %s", cudaGetErrorString(err));
    return LF_ERR_LAUNCH;
  }
  return launch_status("lf_rotary_embed");
}
