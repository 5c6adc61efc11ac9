// Sampling for a batch of rows, each under its own options, from given random
// numbers.
//
// A row's candidates are its finite FP16 logits in descending order (-0 below
// +0, equal bits by ascending index). top_k keeps the first k; the weight of a
// candidate is exp((v - max) / T) and their sum the total; top_p keeps the
// candidates before which less than top_p of the total lies, min_p those whose
// weight is at least min_p; the first always stays. The token is the first
// kept candidate at which the running sum exceeds uniform * (kept sum).
//
// Weights and sums are FP64, so a token depends on the order of additions only
// where the uniform number lies within about 1e-15 of a border. FP16 has 63,488
// finite values: the row is counted into a histogram of order keys, an exact
// and order-free sum, and each distinct value's weight is computed once.
//
// A cluster of 8 CTAs takes a row: each counts an eighth of the row's indexes
// into a histogram of 16-bit counts in its shared memory, then sums a
// contiguous range of 8,192 keys over the cluster's histograms and scans it.
// Ranges descend with the CTA's rank, so running sums go from rank 0 up.

#include <cooperative_groups.h>

#include "device.cuh"

namespace cg = cooperative_groups;

namespace mi {
namespace k {

namespace {

constexpr int kCtas = 8;
constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kKeys = 65536 / kCtas;      // keys a CTA scans
constexpr int kPer = kKeys / kThreads;    // keys a thread scans
static_assert(kPer == 8, "a thread reads its keys as one 16-byte word");

struct Shared {
  uint32_t hist[65536 / 2];  // two 16-bit counts to a word
  double warp_mass[kWarps];
  uint32_t warp_count[kWarps];
  // read by the cluster's other CTAs
  uint32_t top;              // largest key + 1
  uint32_t count;            // candidates of this CTA's range
  double mass;               // their weight (after top_k)
  double kept;               // running sum at this range's last kept candidate, or -1
  uint32_t key, place;       // the token's key + 1 and place (0: not here)
  uint32_t before[kWarps];
};

__device__ __forceinline__ float key_value(uint32_t key) {
  const uint16_t bits = (uint16_t)((key & 0x8000u) ? (key ^ 0x8000u) : (~key & 0xffffu));
  return __half2float(__ushort_as_half(bits));
}

// Sum over the threads before this one, and over the block.
template <class T>
__device__ __forceinline__ T block_exclusive(T v, T* warps, T& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  T x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) warps[warp] = x;
  __syncthreads();
  T w = warps[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T y = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += y;
  }
  total = __shfl_sync(0xffffffffu, w, 31);
  const T base = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
  T up = __shfl_up_sync(0xffffffffu, x, 1);
  if (lane == 0) up = T(0);
  return (warp ? base : T(0)) + up;
}

// The first / last thread for which `yes` holds, or -1.
__device__ __forceinline__ int block_first(bool yes, uint32_t* warps) {
  const unsigned has = __ballot_sync(0xffffffffu, yes);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = has;
  __syncthreads();
  const unsigned any = __ballot_sync(0xffffffffu, warps[threadIdx.x & 31] != 0);
  if (!any) return -1;
  const int w = __ffs(any) - 1;
  return 32 * w + __ffs(warps[w]) - 1;
}
__device__ __forceinline__ int block_last(bool yes, uint32_t* warps) {
  const unsigned has = __ballot_sync(0xffffffffu, yes);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = has;
  __syncthreads();
  const unsigned any = __ballot_sync(0xffffffffu, warps[threadIdx.x & 31] != 0);
  if (!any) return -1;
  const int w = 31 - __clz(any);
  return 32 * w + 31 - __clz(warps[w]);
}

__global__ void __cluster_dims__(kCtas, 1, 1) __launch_bounds__(kThreads, 1)
    sample_batch_kernel(const SampleBatch p) {
  extern __shared__ __align__(16) uint8_t smem[];
  Shared& sh = *reinterpret_cast<Shared*>(smem);
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank();
  const int row = blockIdx.x / kCtas;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  for (int i = tid; i < 65536 / 8; i += kThreads)
    reinterpret_cast<uint4*>(sh.hist)[i] = make_uint4(0, 0, 0, 0);
  if (tid == 0) {
    sh.top = 0;
    sh.key = 0;
  }
  pdl_trigger();
  pdl_wait();
  const float temperature = p.temperature[row], top_p = p.top_p[row], min_p = p.min_p[row];
  const float uniform = p.uniform[row];
  const uint32_t top_k = p.top_k[row];
  // written so that NaN fails
  const bool fine = temperature >= 0.f && temperature <= 3.4028234664e38f && top_p >= 0.f &&
                    top_p <= 1.f && min_p >= 0.f && min_p <= 1.f && uniform >= 0.f &&
                    uniform < 1.f;
  if (!fine) {  // the same in every CTA of the cluster
    if (rank == 0 && tid == 0) {
      p.tokens[row] = 0xFFFFFFFEu;
      report_fault(p.fault, kFaultSampling);
    }
    return;
  }
  __syncthreads();

  // ---- count ---------------------------------------------------------------------
  const uint16_t* x = reinterpret_cast<const uint16_t*>(p.logits) + (size_t)row * p.n;
  const int chunk = ((p.n + kCtas - 1) / kCtas + 7) / 8 * 8;
  const int first = min(p.n, rank * chunk), last = min(p.n, first + chunk);
  uint32_t top = 0;
  auto count = [&](uint32_t bits) {
    if ((bits & 0x7c00u) != 0x7c00u) {
      const uint32_t key = sample_key16((uint16_t)bits);
      top = max(top, key + 1);
      atomicAdd(&sh.hist[key >> 1], 1u << (16 * (key & 1)));
    }
  };
  {
    // 16-byte words of the range, and what lies before and behind them
    const int head = min(last - first, (int)((16 - (reinterpret_cast<uintptr_t>(x + first) & 15)) & 15) / 2);
    const int words = (last - first - head) / 8;
    if (tid < head) count(x[first + tid]);
    const uint4* w = reinterpret_cast<const uint4*>(x + first + head);
    for (int i = tid; i < words; i += kThreads) {
      const uint4 v = w[i];
      const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        count(u[e] & 0xffffu);
        count(u[e] >> 16);
      }
    }
    const int tail = first + head + words * 8 + tid;
    if (tail < last) count(x[tail]);
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0 && top) atomicMax(&sh.top, top);
  cluster.sync();
  top = 0;
  for (int c = 0; c < kCtas; ++c) top = max(top, *cluster.map_shared_rank(&sh.top, c));

  // ---- this thread's keys, descending from `high` ----------------------------------
  const int high = 65536 - rank * kKeys - tid * kPer;  // keys high - 1 ... high - kPer
  uint32_t c[kPer] = {};
  for (int r = 0; r < kCtas; ++r) {
    const uint4 v =
        *reinterpret_cast<const uint4*>(cluster.map_shared_rank(sh.hist, r) + (high - kPer) / 2);
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      c[kPer - 1 - 2 * e] += u[e] & 0xffffu;
      c[kPer - 2 - 2 * e] += u[e] >> 16;
    }
  }
  uint32_t place = 0, key = 0;  // the token, where it is in this thread's keys
  bool chosen = false;
  if (top == 0) {
    // no finite logit
  } else if (temperature == 0.f) {
    key = top - 1;
    chosen = rank == 0 && tid == 0;
  } else {
    const double most = (double)key_value(top - 1);
    if (top_k) {  // the first top_k candidates stay
      uint32_t own = 0, all;
#pragma unroll
      for (int e = 0; e < kPer; ++e) own += c[e];
      uint32_t at = block_exclusive(own, sh.warp_count, all);
      if (tid == 0) sh.count = all;
      cluster.sync();
      for (int r = 0; r < rank; ++r) at += *cluster.map_shared_rank(&sh.count, r);
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const uint32_t n = c[e];
        c[e] = at >= top_k ? 0u : min(n, top_k - at);
        at += n;
      }
    }
    double w[kPer], own = 0.0, all;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      w[e] = c[e] ? exp(((double)key_value(high - 1 - e) - most) / (double)temperature) : 0.0;
      own += c[e] * w[e];
    }
    double at = block_exclusive(own, sh.warp_mass, all);
    if (tid == 0) sh.mass = all;
    cluster.sync();
    double before = 0.0, total = 0.0;
    for (int r = 0; r < kCtas; ++r) {
      const double m = *cluster.map_shared_rank(&sh.mass, r);
      if (r < rank) before += m;
      total += m;
    }
    at += before;
    // What top_p and min_p keep is a prefix again: the kept sum is the sum at
    // the end of the last kept group.
    const double limit = top_p >= 1.f ? INFINITY : (double)top_p * total;
    double kept = -1.0, sum = at;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      uint32_t n = c[e];
      if (!(w[e] >= (double)min_p)) n = 0;
      if (n && limit != INFINITY) {
        // places j with sum + j w < limit
        const double j = ceil((limit - sum) / w[e]);
        uint32_t m = j <= 0.0 ? 0u : j >= (double)n ? n : (uint32_t)j;
        if (m && !(sum + (m - 1) * w[e] < limit)) --m;
        else if (m < n && sum + m * w[e] < limit) ++m;
        n = m;
      }
      if (c[e] && n == 0 && (uint32_t)(high - e) == top) n = 1;  // the first always stays
      if (n) kept = sum + n * w[e];
      sum += c[e] * w[e];
      c[e] = n;
    }
    const int last_thread = block_last(kept >= 0.0, sh.before);
    if (tid == last_thread) sh.kept = kept;
    if (tid == 0 && last_thread < 0) sh.kept = -1.0;
    cluster.sync();
    double sum_kept = 0.0;
    for (int r = 0; r < kCtas; ++r) {
      const double s = *cluster.map_shared_rank(&sh.kept, r);
      if (s >= 0.0) sum_kept = s;
    }
    // The first group whose sum exceeds the target: there is one, as the
    // last kept group's sum is the kept sum itself. Threads' sums meet within
    // rounding only, so the first of all is taken, not the one around it.
    const double target = (double)uniform * sum_kept;
    bool crosses = false;
    sum = at;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      if (c[e] && !crosses && sum + c[e] * w[e] > target) {
        const double j = floor((target - sum) / w[e]);
        uint32_t m = j <= 0.0 ? 0u : j >= (double)c[e] ? c[e] - 1 : (uint32_t)j;
        if (sum + (m + 1) * w[e] <= target && m + 1 < c[e]) ++m;
        else if (m && sum + m * w[e] > target) --m;
        crosses = true;
        key = high - 1 - e;
        place = m;
      }
      sum += c[e] * w[e];
    }
    chosen = tid == block_first(crosses, sh.before);
  }
  if (chosen) {
    sh.key = key + 1;
    sh.place = place;
  }
  cluster.sync();

  // ---- key and place to an index -----------------------------------------------------
  key = 0;
  for (int r = kCtas - 1; r >= 0; --r) {
    const uint32_t q = *cluster.map_shared_rank(&sh.key, r);
    if (q) {
      key = q;
      place = *cluster.map_shared_rank(&sh.place, r);
    }
  }
  if (key == 0) {
    if (rank == 0 && tid == 0) p.tokens[row] = 0xFFFFFFFFu;
  } else {
    --key;
    int at = (int)place;  // place among this CTA's and later ones' equals
    for (int r = 0; r < rank; ++r)
      at -= (cluster.map_shared_rank(sh.hist, r)[key >> 1] >> (16 * (key & 1))) & 0xffffu;
    const int here = (sh.hist[key >> 1] >> (16 * (key & 1))) & 0xffffu;
    if (at >= 0 && at < here) {
      // each warp takes a run of the range: equals per warp, then the warp
      // that holds the place walks its run
      const int run = (last - first + kWarps * 32 - 1) / (kWarps * 32) * 32;
      const int a = min(last, first + warp * run), b = min(last, a + run);
      int equals = 0;
      for (int i = a; i < b; i += 32) {
        const bool eq = i + lane < b && (x[i + lane] & 0x7c00u) != 0x7c00u &&
                        sample_key16(x[i + lane]) == key;
        equals += __popc(__ballot_sync(0xffffffffu, eq));
      }
      __syncthreads();
      if (lane == 0) sh.before[warp] = equals;
      __syncthreads();
      int rest = at;
      for (int q = 0; q < warp; ++q) rest -= (int)sh.before[q];
      if (rest >= 0 && rest < equals) {
        for (int i = a; i < b; i += 32) {
          const bool eq = i + lane < b && (x[i + lane] & 0x7c00u) != 0x7c00u &&
                          sample_key16(x[i + lane]) == key;
          const unsigned hits = __ballot_sync(0xffffffffu, eq);
          const int n = __popc(hits);
          if (rest < n) {
            if (eq && __popc(hits & ((1u << lane) - 1)) == rest) p.tokens[row] = i + lane;
            break;
          }
          rest -= n;
        }
      }
    }
  }
  cluster.sync();  // no CTA leaves while another reads its shared memory
}

}  // namespace

void sample_batch(const Launch& l, const SampleBatch& p) {
  if (p.rows == 0) return;
  allow_dynamic_smem(sample_batch_kernel, sizeof(Shared));
  launch_kernel(l, dim3(p.rows * kCtas), dim3(kThreads), sizeof(Shared), sample_batch_kernel, p);
}

}  // namespace k
}  // namespace mi
