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
// A cluster of 8 CTAs takes a row, of 4 where the rows fill the GPU: each
// counts its share of the row's indexes into a histogram of 16-bit counts in
// its shared memory, then sums its keys over the cluster's histograms and
// scans them. The keys go to the CTAs in blocks of 1,024 by turns, since a
// row's values share a few exponents; the scan is by descending key: threads,
// blocks of a CTA, then the 64 blocks' sums of all CTAs.

#include <cooperative_groups.h>

#include "device.cuh"

namespace cg = cooperative_groups;

namespace mi {
namespace k {

namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kBlockKeys = 1024;
constexpr int kBlocks = 65536 / kBlockKeys;
static_assert(kBlocks == 64, "a warp sums the blocks two to a lane");

struct Shared {
  uint32_t hist[65536 / 2];  // two 16-bit counts to a word
  double warp_mass[kWarps];
  uint32_t warp_count[kWarps];
  uint32_t equals[kWarps];
  // read by the cluster's other CTAs
  uint32_t top;                // largest key + 1
  uint32_t count[kBlocks / 4]; // candidates of this CTA's blocks
  double mass[kBlocks / 4];    // their weight (after top_k)
  uint32_t last;               // order + 1 of this CTA's last kept group
  double kept;                 // running sum at its end
  uint32_t first;              // ~order of this CTA's first group that crosses the target
  uint32_t key, place;         // its key + 1, the place among the equals
};

__device__ __forceinline__ float key_value(uint32_t key) {
  const uint16_t bits = (uint16_t)((key & 0x8000u) ? (key ^ 0x8000u) : (~key & 0xffffu));
  return __half2float(__ushort_as_half(bits));
}

// Sum over everything before this thread in descending key order, and over
// the row. `sums` (this CTA's blocks) is read by the cluster.
template <int kCtas, class T>
__device__ __forceinline__ T row_exclusive(cg::cluster_group& cluster, T v, T* warps, T* sums,
                                           T& total) {
  constexpr int kBlockWarps = kThreads / (kBlocks / kCtas) / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  T x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) warps[warp] = x;
  T before = __shfl_up_sync(0xffffffffu, x, 1);
  if (lane == 0) before = T(0);
  __syncthreads();
  const int block = warp / kBlockWarps;
  T all = T(0), base = T(0);
#pragma unroll
  for (int w = 0; w < kBlockWarps; ++w) {
    const T y = warps[block * kBlockWarps + w];
    if (w < warp % kBlockWarps) base += y;
    all += y;
  }
  if (lane == 0 && warp % kBlockWarps == 0) sums[block] = all;
  cluster.sync();
  // block b of the row is block b / kCtas of CTA b % kCtas
  const int mine = block * kCtas + (int)cluster.block_rank();
  T earlier = T(0), every = T(0);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int b = lane + 32 * i;
    const T y = cluster.map_shared_rank(sums, b % kCtas)[b / kCtas];
    every += y;
    if (b < mine) earlier += y;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    every += __shfl_xor_sync(0xffffffffu, every, o);
    earlier += __shfl_xor_sync(0xffffffffu, earlier, o);
  }
  total = every;
  return earlier + (base + before);
}

template <int kCtas>
__global__ void __launch_bounds__(kThreads, 1) sample_batch_kernel(const SampleBatch p) {
  constexpr int kPer = 65536 / kCtas / kThreads;  // keys of a thread
  constexpr int kBlockThreads = kBlockKeys / kPer;
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
    sh.last = 0;
    sh.first = 0;
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
    const int head =
        min(last - first, (int)((16 - (reinterpret_cast<uintptr_t>(x + first) & 15)) & 15) / 2);
    const int words = (last - first - head) / 8;
    if (tid < head) count(x[first + tid]);
    const uint4* w = reinterpret_cast<const uint4*>(x + first + head);
#pragma unroll 2
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
#pragma unroll
  for (int c = 0; c < kCtas; ++c) top = max(top, *cluster.map_shared_rank(&sh.top, c));

  // ---- this thread's keys, descending: high - 1 ... high - kPer ----------------------
  const int block = tid / kBlockThreads * kCtas + rank;
  const int high = 65536 - block * kBlockKeys - tid % kBlockThreads * kPer;
  const uint32_t order = block * kBlockThreads + tid % kBlockThreads;
  uint32_t c[kPer] = {};
#pragma unroll
  for (int r = 0; r < kCtas; ++r) {
    const uint4* h =
        reinterpret_cast<const uint4*>(cluster.map_shared_rank(sh.hist, r) + (high - kPer) / 2);
#pragma unroll
    for (int i = 0; i < kPer / 8; ++i) {
      const uint4 v = h[i];
      const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        c[kPer - 1 - 8 * i - 2 * e] += u[e] & 0xffffu;
        c[kPer - 2 - 8 * i - 2 * e] += u[e] >> 16;
      }
    }
  }
  if (top == 0) {
    // no finite logit
  } else if (temperature == 0.f) {
    if (rank == 0 && tid == 0) {
      sh.first = ~0u;
      sh.key = top;
      sh.place = 0;
    }
  } else {
    if (top_k) {  // the first top_k candidates stay
      uint32_t own = 0, all;
#pragma unroll
      for (int e = 0; e < kPer; ++e) own += c[e];
      uint32_t at = row_exclusive<kCtas>(cluster, own, sh.warp_count, sh.count, all);
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const uint32_t n = c[e];
        c[e] = at >= top_k ? 0u : min(n, top_k - at);
        at += n;
      }
    }
    const double most = (double)key_value(top - 1), inverse = 1.0 / (double)temperature;
    double w[kPer], own = 0.0, total;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      w[e] = c[e] ? exp(((double)key_value(high - 1 - e) - most) * inverse) : 0.0;
      own += c[e] * w[e];
    }
    const double at = row_exclusive<kCtas>(cluster, own, sh.warp_mass, sh.mass, total);
    // What top_p and min_p keep is a prefix again: the kept sum is the sum at
    // the end of the last kept group.
    const double limit = top_p >= 1.f ? INFINITY : (double)top_p * total;
    double kept = -1.0, sum = at;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      uint32_t n = w[e] >= (double)min_p ? c[e] : 0u;
      if (n && !(sum + (n - 1) * w[e] < limit)) {
        // places j with sum + j w < limit
        uint32_t m = 0;
        if (sum < limit) {
          const double j = ceil((limit - sum) / w[e]);
          m = j >= (double)n ? n : (uint32_t)j;
          if (m && !(sum + (m - 1) * w[e] < limit)) --m;
          else if (m < n && sum + m * w[e] < limit) ++m;
        }
        n = m;
      }
      if (c[e] && n == 0 && (uint32_t)(high - e) == top) n = 1;  // the first always stays
      if (n) kept = sum + n * w[e];
      sum += c[e] * w[e];
      c[e] = n;
    }
    const uint32_t mine = kept >= 0.0 ? order + 1 : 0u;
    const uint32_t warp_last = __reduce_max_sync(0xffffffffu, mine);
    if (lane == 0 && warp_last) atomicMax(&sh.last, warp_last);
    __syncthreads();
    if (mine && sh.last == mine) sh.kept = kept;
    cluster.sync();
    uint32_t final = 0;
    double sum_kept = 0.0;
#pragma unroll
    for (int r = 0; r < kCtas; ++r) {
      const uint32_t q = *cluster.map_shared_rank(&sh.last, r);
      if (q > final) {
        final = q;
        sum_kept = *cluster.map_shared_rank(&sh.kept, r);
      }
    }
    // The first group whose sum exceeds the target: there is one, as the
    // last kept group's sum is the kept sum itself. Threads' sums meet within
    // rounding only, so the first of all is taken, not the one around it.
    const double target = (double)uniform * sum_kept;
    bool crosses = false;
    sum = at;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      if (c[e] && sum + c[e] * w[e] > target) crosses = true;
      sum += c[e] * w[e];
    }
    const uint32_t hit = crosses ? ~order : 0u;
    const uint32_t warp_first = __reduce_max_sync(0xffffffffu, hit);
    if (lane == 0 && warp_first) atomicMax(&sh.first, warp_first);
    __syncthreads();
    if (hit && sh.first == hit) {
      sum = at;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        if (crosses && c[e] && sum + c[e] * w[e] > target) {
          const double j = floor((target - sum) / w[e]);
          uint32_t m = j <= 0.0 ? 0u : j >= (double)c[e] ? c[e] - 1 : (uint32_t)j;
          if (sum + (m + 1) * w[e] <= target && m + 1 < c[e]) ++m;
          else if (m && sum + m * w[e] > target) --m;
          sh.key = high - e;
          sh.place = m;
          crosses = false;
        }
        sum += c[e] * w[e];
      }
    }
  }
  cluster.sync();

  // ---- key and place to an index -----------------------------------------------------
  uint32_t key = 0, place = 0, best = 0;
#pragma unroll
  for (int r = 0; r < kCtas; ++r) {
    const uint32_t q = *cluster.map_shared_rank(&sh.first, r);
    if (q > best) {
      best = q;
      key = *cluster.map_shared_rank(&sh.key, r);
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
      // the FP16 bits of the key
      const uint16_t bits = (uint16_t)((key & 0x8000u) ? (key ^ 0x8000u) : (~key & 0xffffu));
      int equals = 0;
#pragma unroll 4
      for (int i = a; i < b; i += 32)
        equals += __popc(__ballot_sync(0xffffffffu, i + lane < b && x[i + lane] == bits));
      if (lane == 0) sh.equals[warp] = equals;
      __syncthreads();
      int rest = at;
      for (int q = 0; q < warp; ++q) rest -= (int)sh.equals[q];
      if (rest >= 0 && rest < equals) {
        for (int i = a; i < b; i += 32) {
          const bool eq = i + lane < b && x[i + lane] == bits;
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

template <int kCtas>
void launch_sample(const Launch& l, const SampleBatch& p) {
  auto kernel = sample_batch_kernel<kCtas>;
  allow_dynamic_smem(kernel, sizeof(Shared));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.rows * kCtas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(Shared);
  cfg.stream = l.stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kCtas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = l.pdl ? 2 : 1;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, p);
  if (err != cudaSuccess)
    fail(MI_ERR_COMMAND, "kernel launch failed: %s", cudaGetErrorString(err));
}

}  // namespace

void sample_batch(const Launch& l, const SampleBatch& p) {
  if (p.rows == 0) return;
  // Four CTAs to a row leave fewer fixed costs, eight are quicker with a row:
  // eight while the rows fit the GPU at once, or where a CTA's share of the
  // row would outgrow its 16-bit counts.
  if (p.rows * 8 <= l.sm_count || p.n > 4 * 65528)
    launch_sample<8>(l, p);
  else
    launch_sample<4>(l, p);
}

}  // namespace k
}  // namespace mi
