// Which pages a sparse attention call reads: a bound on the scores of each page
// from its Key bounds, and the best of them (lf_int4_select).
//
// Mathematics.  For a page with channel bounds low_d <= K_d <= upper_d every
// score q . K is at most sum_d max(q_d, 0) upper_d + min(q_d, 0) low_d; summed over
// the heads that share the KV head, that is one dot product of the record's 2 D
// int8 entries with 2 D weights.  The weights are whole numbers (the queries
// scaled by one power of two per group and rounded), so the sum is exact in
// int32 and the choice the same on every run.
//
// One cluster per (query token, KV head): its CTAs share the candidate pages, a
// warp per record (a lane holds the weights of its 8 channels, two int16 x int8
// products an instruction, one warp sum), and put the scores into the first
// CTA's shared memory; that CTA then narrows the range of the top-th best score
// (a histogram of 256 steps over the range that is left, four rounds at most)
// and writes the chosen pages in order.
//
// Bound by the latency of dependent steps: lengths, queries and table, records,
// rounds of the histogram.  Measured at 64 sequences of 16k tokens, 40 heads on 8,
// D 128 (34 MB of records): 12.8 us (2.7 TB/s); 2 of 128k, 28 heads on 4 (4.2 MB):
// 10.3 us with clusters of 8, a warp on a run of records that lie one after another
// in its list (13.6 us when the warps took turns).  Loading the first ids beside the
// queries costs registers: 11.2 us.
#include "lf_int4.cuh"

namespace lf {

struct SelectParams {
  Int4Pool pool;
  const void* q;
  int64_t q_seq, q_head, q_tok;
  int q_len, group;
  const int8_t* bounds;
  int64_t bounds_page, bounds_head;
  const int32_t *lengths, *counts;
  int top, sink, recent, cluster;
  int32_t* picked;
  int32_t* status;
  float sign;  // of the scores' scaling: -1 chooses for the negated queries
};

constexpr int kSelectThreads = 256, kSelectWarps = kSelectThreads / 32;
constexpr int kMaxSelectPages = 32768;  // candidates whose scores fit in shared memory
constexpr int kMaxGroup = 64;           // query heads per KV head
constexpr int kPagesAtOnce = 16;        // records a warp has in flight

// A float's bits as an unsigned number of the same order.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x);
  return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// Stores into the shared memory of the cluster's first CTA, at this CTA's address of p.
__device__ __forceinline__ void store_first(uint32_t* p, uint32_t v) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(at) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))));
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}

// Sum of x over the threads before this one, and over all of them.
__device__ __forceinline__ uint32_t scan_before(uint32_t x, uint32_t* warp_sum, uint32_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t upto = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
  }
  __syncthreads();  // warp_sum may still be read from the scan before
  if (lane == 31) warp_sum[warp] = upto;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kSelectWarps; ++w) {
    if (w < warp) before += warp_sum[w];
    total += warp_sum[w];
  }
  return before + upto - x;
}

template <typename T, int D>
__global__ void __launch_bounds__(kSelectThreads, 4) int4_select_kernel(const __grid_constant__ SelectParams p) {
  extern __shared__ uint32_t key_s[];
  __shared__ __align__(16) int16_t weight_s[2 * D];
  __shared__ __align__(16) uint16_t query_s[kMaxGroup * D];
  __shared__ float most_s[kSelectWarps];
  __shared__ uint32_t hist_s[256], sum_s[kSelectWarps], low_s[kSelectWarps], high_s[kSelectWarps], pick_s[3];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = p.cluster > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int h = blockIdx.x / p.cluster, i = blockIdx.y, b = blockIdx.z;
  const int slots = p.top + p.sink + p.recent;
  grid_dep_wait();
  int32_t* picked = p.picked + ((static_cast<int64_t>(b) * p.q_len + i) * p.pool.kv_heads + h) * slots;
  const int seen = int4_seen(p.lengths[b], p.counts != nullptr ? p.counts[b] : p.q_len, i);
  const int n = min(seen / kInt4Page + (seen % kInt4Page != 0), p.pool.table_width);
  if (n <= slots || p.top == 0) {  // nothing to choose (the same in every CTA of the cluster)
    const int head = n <= slots ? n : p.sink;
    if (rank == 0)
      for (int s = tid; s < slots; s += kSelectThreads) picked[s] = s < head ? s : n <= slots ? -1 : n - slots + s;
    return;
  }

  if (p.cluster > 1) cluster_arrive();  // that every CTA of the cluster runs, before any stores to the first

  // Weights: the group's queries in whole numbers, split by sign.  All heads are
  // loaded at once, eight channels a thread.
  const T* q = static_cast<const T*>(p.q) + b * p.q_seq + static_cast<int64_t>(h) * p.group * p.q_head + i * p.q_tok;
  float most = 0.0f;
  for (int x = tid; x < p.group * (D / 8); x += kSelectThreads) {
    const uint4 w = *reinterpret_cast<const uint4*>(q + x / (D / 8) * p.q_head + x % (D / 8) * 8);
    *reinterpret_cast<uint4*>(query_s + 8 * x) = w;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t pair = k < 2 ? w.x : k < 4 ? w.y : k < 6 ? w.z : w.w;
      const uint16_t bits = static_cast<uint16_t>(k % 2 ? pair >> 16 : pair);
      const float v = fabsf(Scalar<T>::load(reinterpret_cast<const T*>(&bits)));
      most = v < INFINITY ? fmaxf(most, v) : most;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
  if (lane == 0) most_s[warp] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSelectWarps; ++w) most = fmaxf(most, most_s[w]);
  const float scale = pow2(-exponent127(most)) * p.sign;
  if (tid < D) {
    int plus = 0, minus = 0;
    for (int j = 0; j < p.group; ++j) {
      const float v = Scalar<T>::load(reinterpret_cast<const T*>(query_s + j * D + tid));
      const int c = isfinite(v) ? __float2int_rn(v * scale) : 0;
      plus += max(c, 0);
      minus += min(c, 0);
    }
    weight_s[tid] = static_cast<int16_t>(plus);
    weight_s[D + tid] = static_cast<int16_t>(minus);
  }
  __syncthreads();

  // Scores of this CTA's candidates (pages sink .. n - recent - 1): an equal run of
  // them per warp, the ids of 32 at a time, the records of kPagesAtOnce in flight.
  constexpr int kBytes = 2 * D / 32, kPairs = kBytes / 2;  // a lane's record entries and its weight pairs
  int wt[kPairs];
#pragma unroll
  for (int x = 0; x < kPairs; ++x) wt[x] = reinterpret_cast<const int*>(weight_s)[lane * kPairs + x];
  const int first = p.sink, count = n - p.sink - p.recent;
  if (p.cluster > 1) cluster_wait();
  const int run = (count + p.cluster * kSelectWarps - 1) / (p.cluster * kSelectWarps);
  const int run_end = min(count, (rank * kSelectWarps + warp + 1) * run);
  const int8_t* head_bounds = p.bounds + h * p.bounds_head;
  for (int c0 = (rank * kSelectWarps + warp) * run; c0 < run_end; c0 += 32) {
    int id = -1, e = 0, mine = 0;
    if (c0 + lane < run_end) {
      id = int4_page_id(p.pool, b, first + c0 + lane);
      if (id < 0 && p.status != nullptr) atomicExch(p.status, LF_ERR_OUT_OF_RANGE);
      if (id >= 0) e = head_bounds[id * p.bounds_page + 2 * D];
    }
    for (int x0 = 0; x0 < min(32, run_end - c0); x0 += kPagesAtOnce) {
      uint32_t w[kPagesAtOnce][kBytes / 4];
#pragma unroll
      for (int x = 0; x < kPagesAtOnce; ++x) {
        const int page = __shfl_sync(0xffffffffu, id, x0 + x);
#pragma unroll
        for (int y = 0; y < kBytes / 4; ++y) w[x][y] = 0;
        if (page >= 0) {
          const int8_t* rec = head_bounds + page * p.bounds_page + lane * kBytes;
          if constexpr (D == 128) {
            const uint2 y = *reinterpret_cast<const uint2*>(rec);
            w[x][0] = y.x;
            w[x][1] = y.y;
          } else {
            w[x][0] = *reinterpret_cast<const uint32_t*>(rec);
          }
        }
      }
#pragma unroll
      for (int x = 0; x < kPagesAtOnce; ++x) {
        int sum = 0;
#pragma unroll
        for (int y = 0; y < kBytes / 4; ++y) {
          sum = __dp2a_lo(wt[2 * y], static_cast<int>(w[x][y]), sum);
          sum = __dp2a_hi(wt[2 * y + 1], static_cast<int>(w[x][y]), sum);
        }
        sum = __reduce_add_sync(0xffffffffu, sum);
        mine = lane == x0 + x ? sum : mine;
      }
    }
    if (c0 + lane < run_end) {
      const uint32_t key = id < 0 ? 0u : ordered(__int2float_rn(mine) * pow2(e));
      if (p.cluster > 1)
        store_first(key_s + c0 + lane, key);
      else
        key_s[c0 + lane] = key;
    }
  }
  if (p.cluster > 1) {
    cluster_arrive();
    cluster_wait();
    if (rank != 0) return;
  } else {
    __syncthreads();
  }

  // The top-th best key: narrow [low, high] until all the keys in it are chosen, or
  // one value is left.  `want` keys of the range are chosen, and all above it.
  uint32_t low = UINT32_MAX, high = 0;
  for (int c = tid; c < count; c += kSelectThreads) {
    low = min(low, key_s[c]);
    high = max(high, key_s[c]);
  }
  low = __reduce_min_sync(0xffffffffu, low);
  high = __reduce_max_sync(0xffffffffu, high);
  if (lane == 0) {
    low_s[warp] = low;
    high_s[warp] = high;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSelectWarps; ++w) {
    low = min(low, low_s[w]);
    high = max(high, high_s[w]);
  }
  uint32_t want = p.top;
  while (low < high) {  // at most 4 rounds: the range loses 8 bits each
    const int shift = max(0, 24 - __clz(high - low));  // (high - low) >> shift is at most 255
    hist_s[tid] = 0;
    __syncthreads();
    for (int c = tid; c < count; c += kSelectThreads) {
      const uint32_t k = key_s[c];
      if (k >= low && k <= high) atomicAdd(&hist_s[255 - ((k - low) >> shift)], 1u);  // best step first
    }
    __syncthreads();
    const uint32_t mine = hist_s[tid];
    uint32_t total;
    const uint32_t before = scan_before(mine, sum_s, total);
    if (before < want && want <= before + mine) {
      pick_s[0] = 255 - tid;
      pick_s[1] = want - before;
      pick_s[2] = mine;
    }
    __syncthreads();
    want = pick_s[1];
    low += pick_s[0] << shift;
    high = low + min(high - low, (1u << shift) - 1u);
    if (want == pick_s[2]) break;
  }

  // Every key above the range, and the first `want` in it, in order.
  const int each = (count + kSelectThreads - 1) / kSelectThreads;
  const int from = min(count, tid * each), to = min(count, from + each);
  uint32_t found = 0;  // keys above in the low half, those in the range in the high half
  for (int c = from; c < to; ++c) found += key_s[c] > high ? 1u : key_s[c] >= low ? 0x10000u : 0u;
  uint32_t total;
  uint32_t place = scan_before(found, sum_s, total);
  for (int c = from; c < to; ++c) {
    const uint32_t k = key_s[c], within = place >> 16;
    if (k > high || (k >= low && within < want)) picked[p.sink + (place & 0xFFFFu) + min(within, want)] = first + c;
    place += k > high ? 1u : k >= low ? 0x10000u : 0u;
  }
  for (int s = tid; s < p.sink; s += kSelectThreads) picked[s] = s;
  for (int s = tid; s < p.recent; s += kSelectThreads) picked[p.sink + p.top + s] = n - p.recent + s;
}

template <typename T, int D>
static int launch_select(SelectParams p, cudaStream_t stream) {
  const void* kern = reinterpret_cast<const void*>(int4_select_kernel<T, D>);
  const int smem = p.pool.table_width * static_cast<int>(sizeof(uint32_t));
  cudaError_t err = raise_smem_limit(kern, smem, false);
  if (err != cudaSuccess) {
    set_error("lf_int4_select: %s", cudaGetErrorString(err));
    return LF_ERR_CUDA;
  }
  // More CTAs per unit while the units alone leave SMs idle and every warp keeps
  // eight records.  Measured: 8 units of 2048 pages 27.3 us with one CTA each, 10.3
  // with eight; 4 units of 515 pages 9.7 and 7.2; 512 units of 256 pages 12.8 with one
  // CTA each, 18.5 with two.
  const int64_t units = static_cast<int64_t>(p.pool.kv_heads) * p.q_len * p.pool.batch;
  p.cluster = 1;
  while (p.cluster < 8 && units * p.cluster < 148 && p.pool.table_width > p.cluster * kSelectWarps * 8) p.cluster *= 2;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.pool.kv_heads * p.cluster, p.q_len, p.pool.batch);
  cfg.blockDim = dim3(kSelectThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  void* args[] = {&p};
  err = cudaLaunchKernelExC(&cfg, kern, args);
  if (err != cudaSuccess) {
    set_error("lf_int4_select: %s", cudaGetErrorString(err));
    return LF_ERR_LAUNCH;
  }
  return launch_status("lf_int4_select");
}

// Checks the arguments and fills p; launches nothing.
static int check_select(const lf_int4_query* a, float sign, SelectParams& p) {
  LF_CHECK_ARG(a != nullptr, "lf_int4_select: null arguments");
  p.sign = sign;
  const int bad = check_int4_pool("lf_int4_select", a->pool, a->head_dim, p.pool);
  if (bad != LF_OK) return bad;
  LF_CHECK_ARG(a->q && a->bounds && a->lengths && a->picked, "lf_int4_select: null pointer");
  LF_CHECK_SUPPORTED(a->dtype == LF_F16 || a->dtype == LF_BF16, "lf_int4_select: query dtype %d (fp16 or bf16)", a->dtype);
  LF_CHECK_ARG(a->q_len > 0 && a->q_len <= 65535 && a->n_q > 0 && a->n_q % p.pool.kv_heads == 0,
               "lf_int4_select: q_len %d, %d query heads on %d KV heads", a->q_len, a->n_q, p.pool.kv_heads);
  p.group = a->n_q / p.pool.kv_heads;
  LF_CHECK_SUPPORTED(p.group <= kMaxGroup, "lf_int4_select: %d query heads per KV head (%d at most)", p.group, kMaxGroup);
  LF_CHECK_ARG(a->sink_pages >= 0 && a->recent_pages >= 1 && a->slots <= (1 << 24) &&
                   static_cast<int64_t>(a->sink_pages) + a->recent_pages <= a->slots,
               "lf_int4_select: sink %d, recent %d of %d pages (recent at least 1)", a->sink_pages, a->recent_pages,
               a->slots);
  LF_CHECK_ARG(a->bounds_page_stride > 2 * a->head_dim && a->bounds_head_stride > 2 * a->head_dim,
               "lf_int4_select: bounds records overlap");
  LF_CHECK_ARG((reinterpret_cast<uintptr_t>(a->bounds) & 7) == 0 && (a->bounds_page_stride | a->bounds_head_stride) % 8 == 0,
               "lf_int4_select: bounds records must be 8-byte aligned");
  LF_CHECK_ARG((reinterpret_cast<uintptr_t>(a->q) & 15) == 0 && (a->q_seq_stride | a->q_head_stride | a->q_tok_stride) % 8 == 0,
               "lf_int4_select: query rows must be 16-byte aligned");
  LF_CHECK_SUPPORTED(p.pool.table_width <= kMaxSelectPages, "lf_int4_select: %d pages per sequence (%d at most)",
                     p.pool.table_width, kMaxSelectPages);
  p.q = a->q;
  p.q_seq = a->q_seq_stride;
  p.q_head = a->q_head_stride;
  p.q_tok = a->q_tok_stride;
  p.q_len = a->q_len;
  p.bounds = a->bounds;
  p.bounds_page = a->bounds_page_stride;
  p.bounds_head = a->bounds_head_stride;
  p.lengths = a->lengths;
  p.counts = a->counts;
  p.top = a->slots - a->sink_pages - a->recent_pages;
  p.sink = a->sink_pages;
  p.recent = a->recent_pages;
  p.picked = a->picked;
  p.status = a->status;
  return LF_OK;
}

int check_int4_select(const lf_int4_query* a) {
  SelectParams p;
  return check_select(a, 1.0f, p);
}

int int4_select_pages(const lf_int4_query* a, float sign, cudaStream_t s) {
  SelectParams p;
  const int bad = check_select(a, sign, p);
  if (bad != LF_OK) return bad;
  if (a->dtype == LF_F16) return a->head_dim == 128 ? launch_select<__half, 128>(p, s) : launch_select<__half, 64>(p, s);
  return a->head_dim == 128 ? launch_select<__nv_bfloat16, 128>(p, s) : launch_select<__nv_bfloat16, 64>(p, s);
}

}  // namespace lf

extern "C" int lf_int4_select(const lf_int4_query* a, lf_stream_t stream) {
  return lf::int4_select_pages(a, 1.0f, reinterpret_cast<cudaStream_t>(stream));
}
