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
// and order-free sum, and weights belong to values, not to candidates. Eight
// neighbouring keys share an exponent, so their weights are one exponential
// and powers of another.
//
// A CTA counts 16 bits to a key (128 KB of shared memory). Counting sets the
// pace, so a row that shares the GPU with many others has one CTA and nothing
// to add up between CTAs; where rows are fewer, a cluster of 2, 4 or 8 CTAs
// takes a row: each counts its share of it, then adds up the keys of its own
// over the cluster's histograms (blocks of 64 keys by turns, as a row's values
// share a few exponents). Measured, 96 rows of 151,936: 115 us with 4 CTAs to a
// row, 120 with every CTA reading the whole row for its own keys, 40 so; one
// row 15 to 19 us. Of the some 60,000 clocks of a row's only CTA counting takes
// 27,000 (21,000 without its additions; more loads at a time, loads a step
// ahead and fewer instructions to a value change little), the weights 10,000,
// their sums 5,000, the borders of top_p and the crossing 5,000 each and the
// search for the token's index 7,000.

#include <cooperative_groups.h>

#include "device.cuh"

namespace cg = cooperative_groups;

namespace mi {
namespace k {

namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kGroups = 65536 / 8;  // of eight keys
constexpr int kBlocks = kGroups / 8; // a cluster's CTAs take blocks of 64 keys by turns
static_assert(kBlocks == kThreads, "a thread takes a block's sum");
// Finite keys, descending: 65535 - the order key, so that the largest value
// comes first; infinities and NaN lie outside of [kFirst, kEnd).
constexpr uint32_t kFirst = 0x400, kEnd = 0xFC00;
// A count may grow by a segment's elements before it is looked at again;
// those above kLarge then move to a list of their own.
constexpr int kSegment = 49152;
constexpr uint32_t kLarge = 65535 - kSegment;
constexpr int kLargeMax = kSampleBatchMax / (int)kLarge + 1;

// A thread has a group of eight keys in each of its rounds: 8 where the CTA
// has the row to itself, 1,024 groups apart, so that the few exponents that
// hold most of a row keep all warps busy; fewer where a cluster shares it.
template <int kCtas>
constexpr int kRounds = kGroups / kThreads / kCtas;

template <int kCtas>
struct Shared {
  uint32_t hist[65536 / 2];  // two 16-bit counts to a word
  double mass[kRounds<kCtas>][kThreads];  // sum of a thread's candidates, per round
  double warp_sums[kCtas == 1 ? kRounds<1> * kWarps : kWarps];
  double total;
  double blocks_before[kCtas == 1 ? 1 : kBlocks];
  double step[64];           // weight of one step of an exponent's values (sign in front)
  uint32_t equals[kWarps];
  uint32_t last, first;      // order + 1 of the last kept group, ~order of the first that crosses
  // read by the cluster's other CTAs
  uint32_t least;            // smallest key of this CTA's part - kFirst
  uint32_t large;            // counts moved out of the histogram
  uint32_t large_key[kLargeMax], large_count[kLargeMax];
  double block_sums[kCtas == 1 ? 1 : kBlocks / kCtas];
  double kept;               // running sum where this CTA's kept candidates end
  uint32_t kept_order;       // order + 1 of the group that has it, 0: none
  // written by them
  uint32_t cutoff[8][3];     // ~order, key, count of it that top_k leaves (a CTA's first)
  uint32_t crossing[8][3];   // ~order, key, place of a CTA's first crossing
  uint32_t matches[8];       // the token's equals in a CTA's part of the row
};

__device__ __forceinline__ uint16_t key_bits(uint32_t key) {
  return (uint16_t)(key < 0x8000u ? key ^ 0x7fffu : key);
}
__device__ __forceinline__ float key_value_f(uint32_t key) {
  return __half2float(__ushort_as_half(key_bits(key)));
}
__device__ __forceinline__ double key_value(uint32_t key) { return (double)key_value_f(key); }
// An exact conversion on the FP64 pipe, which is four times as wide as the
// converter: n as the low bits of 2^52.
__device__ __forceinline__ double count_value(uint32_t n) {
  return __hiloint2double(0x43300000, (int)n) - 4503599627370496.0;
}
// Descending keys of the two halves of a word: 0x7fff - bits for a positive
// value, bits for a negative one.
__device__ __forceinline__ uint32_t keys_of(uint32_t w) {
  uint32_t negative;  // each half's sign, spread over it
  asm("prmt.b32 %0, %1, 0, 0xBB99;" : "=r"(negative) : "r"(w));
  return w ^ (~negative & 0x7fff7fffu);
}

// A row as 16-byte words; places outside of it read as +inf, no candidate.
struct Row {
  const uint16_t* base;  // aligned down to 16 bytes
  int from, to;          // the row's places from `base`
  int whole0, whole1;    // words that lie inside
  __device__ Row(const uint16_t* x, int n) {
    from = (int)((reinterpret_cast<uintptr_t>(x) & 15) / 2);
    base = x - from;
    to = from + n;
    whole0 = from ? 1 : 0;
    whole1 = to / 8;
  }
  __device__ int words() const { return (to + 7) / 8; }
  __device__ uint4 word(int i) const {
    if (i >= whole0 && i < whole1) return reinterpret_cast<const uint4*>(base)[i];
    uint32_t u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int a = 8 * i + 2 * e, b = a + 1;
      const uint32_t lo = a >= from && a < to ? base[a] : 0x7c00u;
      const uint32_t hi = b >= from && b < to ? base[b] : 0x7c00u;
      u[e] = lo | hi << 16;
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
  // Words i, i + stride, ..., kMany of them (nothing from `end` on): the loads
  // of words inside the row are in flight together.
  template <int kMany>
  __device__ void load(uint4 (&v)[kMany], int i, int stride, int end) const {
    if (i >= whole0 && i + (kMany - 1) * stride < min(whole1, end)) {
#pragma unroll
      for (int k = 0; k < kMany; ++k) v[k] = reinterpret_cast<const uint4*>(base)[i + k * stride];
    } else {
#pragma unroll
      for (int k = 0; k < kMany; ++k)
        v[k] = i + k * stride < end ? word(i + k * stride)
                                    : make_uint4(0x7c007c00u, 0x7c007c00u, 0x7c007c00u, 0x7c007c00u);
    }
  }
};

template <int kCtas>
__device__ __forceinline__ void row_sync() {
  if constexpr (kCtas == 1)
    __syncthreads();
  else
    cg::this_cluster().sync();
}
template <int kCtas, class T>
__device__ __forceinline__ T* of_rank(T* p, int rank) {
  if constexpr (kCtas == 1)
    return p;
  else
    return cg::this_cluster().map_shared_rank(p, rank);
}

// Sums over the row before each of a thread's groups, and over the row: a
// count or a sum of weights, v[r] the thread's of round r.
template <int kCtas, class T>
__device__ __forceinline__ T row_exclusive(Shared<kCtas>& sh, int rank,
                                           const T (&v)[kRounds<kCtas>],
                                           T (&before)[kRounds<kCtas>]) {
  constexpr int kR = kRounds<kCtas>;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  T* sums = reinterpret_cast<T*>(sh.warp_sums);
  __syncthreads();
  if constexpr (kCtas == 1) {
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      T x = v[r];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const T y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      if (lane == 31) sums[r * kWarps + warp] = x;
      before[r] = __shfl_up_sync(0xffffffffu, x, 1);
      if (lane == 0) before[r] = T(0);
    }
    __syncthreads();
    if (warp == 0) {  // eight warp sums to a lane
      T z = T(0);
#pragma unroll
      for (int i = 0; i < kR; ++i) z += sums[lane * kR + i];
      T x = z;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const T y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      T at = __shfl_up_sync(0xffffffffu, x, 1);
      if (lane == 0) at = T(0);
#pragma unroll
      for (int i = 0; i < kR; ++i) {
        const T y = sums[lane * kR + i];
        sums[lane * kR + i] = at;
        at += y;
      }
      if (lane == 31) *reinterpret_cast<T*>(&sh.total) = at;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kR; ++r) before[r] += sums[r * kWarps + warp];
    return *reinterpret_cast<T*>(&sh.total);
  } else {
    // eight threads to a block, 128 blocks to a round; block b of the row is
    // block b / kCtas of CTA b % kCtas. Each CTA adds up all blocks.
    T* own = reinterpret_cast<T*>(sh.block_sums);
    T* all = reinterpret_cast<T*>(sh.blocks_before);
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      T x = v[r];
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) {
        const T y = __shfl_up_sync(0xffffffffu, x, o, 8);
        if (tid % 8 >= o) x += y;
      }
      before[r] = __shfl_up_sync(0xffffffffu, x, 1, 8);
      if (tid % 8 == 0) before[r] = T(0);
      if (tid % 8 == 7) own[r * (kThreads / 8) + tid / 8] = x;
    }
    row_sync<kCtas>();
    T z = of_rank<kCtas>(own, tid % kCtas)[tid / kCtas];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const T y = __shfl_up_sync(0xffffffffu, z, o);
      if (lane >= o) z += y;
    }
    if (lane == 31) sums[warp] = z;
    __syncthreads();
    T w = sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const T y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    const T total = __shfl_sync(0xffffffffu, w, 31);
    const T base = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
    T earlier = __shfl_up_sync(0xffffffffu, z, 1);
    if (lane == 0) earlier = T(0);
    if (warp) earlier += base;
    all[tid] = earlier;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kR; ++r)
      before[r] += all[(r * (kThreads / 8) + tid / 8) * kCtas + rank];
    return total;
  }
}

// Which of the row's threads comes first: `order` of this one where it has
// `hit`. The CTA's first runs f(out) and leaves out[0..1] beside ~order in
// `to` of every CTA; returns the row's first of them (0: none has hit).
template <int kCtas, class F>
__device__ __forceinline__ bool row_first(Shared<kCtas>& sh, int rank, bool has, uint32_t order,
                                          uint32_t (*to)[3], F f, uint32_t& a, uint32_t& b) {
  const uint32_t hit = has ? ~order : 0u;
  const uint32_t warp_first = __reduce_max_sync(0xffffffffu, hit);
  if ((threadIdx.x & 31) == 0 && warp_first) atomicMax(&sh.first, warp_first);
  __syncthreads();
  const uint32_t found = sh.first;
  if (hit ? found == hit : found == 0 && threadIdx.x == 0) {
    uint32_t out[2] = {0, 0};
    if (hit) f(out);
#pragma unroll
    for (int r = 0; r < kCtas; ++r) {
      uint32_t* q = of_rank<kCtas>(&to[rank][0], r);
      q[0] = hit;
      q[1] = out[0];
      q[2] = out[1];
    }
  }
  row_sync<kCtas>();
  if (threadIdx.x == 0) sh.first = 0;
  uint32_t best = 0;
#pragma unroll
  for (int r = 0; r < kCtas; ++r)
    if (to[r][0] > best) {
      best = to[r][0];
      a = to[r][1];
      b = to[r][2];
    }
  return best != 0;
}

template <int kCtas>
__global__ void __launch_bounds__(kThreads, 1) sample_batch_kernel(const SampleBatch p) {
  constexpr int kR = kRounds<kCtas>;
  extern __shared__ __align__(16) uint8_t smem[];
  Shared<kCtas>& sh = *reinterpret_cast<Shared<kCtas>*>(smem);
  const int rank = kCtas == 1 ? 0 : (int)(blockIdx.x % kCtas);
  const int row = blockIdx.x / kCtas;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  for (int i = tid; i < 65536 / 8; i += kThreads)
    reinterpret_cast<uint4*>(sh.hist)[i] = make_uint4(0, 0, 0, 0);
  if (tid == 0) {
    sh.least = 0xFFFFu;
    sh.last = 0;
    sh.first = 0;
    sh.large = 0;
    sh.kept_order = 0;
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
  if (!fine) {  // the same in every CTA of the row
    if (rank == 0 && tid == 0) {
      p.tokens[row] = 0xFFFFFFFEu;
      report_fault(p.fault, kFaultSampling);
    }
    return;
  }
  const double inverse = 1.0 / (double)temperature;
  if (tid < 64) {
    // values of exponent e are 2^(max(e, 1) - 25) apart
    sh.step[tid] = exp(-ldexp(1.0, max(tid & 31, 1) - 25) * inverse);
  }
  __syncthreads();

  // ---- count ---------------------------------------------------------------------
  const Row x(reinterpret_cast<const uint16_t*>(p.logits) + (size_t)row * p.n, p.n);
  // this CTA's words
  const int share = (x.words() + kCtas - 1) / kCtas;
  const int w0 = min(x.words(), rank * share), w1 = min(x.words(), w0 + share);
  {
    uint32_t least = 0xFFFFFFFFu;  // two smallest key - kFirst, wrapped below it
    auto add = [&](uint32_t d, uint32_t n) {
      if (d - kFirst < kEnd - kFirst) atomicAdd(&sh.hist[d >> 1], n << (16 * (d & 1)));
    };
    constexpr int kMany = 3;
    static_assert(kSegment % (8 * kMany * kThreads) == 0, "whole steps to a segment");
    for (int a = w0; a < w1; a += kSegment / 8) {
      const int b = min(w1, a + kSegment / 8);
      for (int i = a + tid; i - lane < b; i += kMany * kThreads) {
        uint4 v[kMany];
        x.load(v, i, kThreads, b);
#pragma unroll
        for (int k = 0; k < kMany; ++k) {
          const uint32_t u[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
          // a stretch of one value (a mask) is one addition
          const bool same = ((u[0] ^ u[1]) | (u[2] ^ u[3]) | (u[0] ^ u[2])) == 0;
          if (__all_sync(0xffffffffu, same)) {
            const uint32_t one = __shfl_sync(0xffffffffu, u[0], 0);
            if (__all_sync(0xffffffffu, u[0] == one) && (one & 0xffffu) == one >> 16) {
              const uint32_t d = keys_of(one);
              least = __viaddmin_u16x2(d, 0xFC00FC00u, least);
              if (lane == 0) add(d & 0xffffu, 256);
              continue;
            }
          }
          uint32_t d[4], most = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            d[e] = keys_of(u[e]);
            least = __viaddmin_u16x2(d[e], 0xFC00FC00u, least);
            most = __viaddmax_u16x2(d[e], 0xFC00FC00u, most);
          }
          // less kFirst, keys of infinities and NaN are the ones from kEnd - kFirst on
          const bool finite =
              most < (kEnd - kFirst) << 16 && (most & 0xffffu) < kEnd - kFirst;
          if (__all_sync(0xffffffffu, finite)) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              // word d / 2, and 1 or 2^16: 1 turned by 16 (d mod 2) bits
              char* const hist = reinterpret_cast<char*>(sh.hist);
              atomicAdd(reinterpret_cast<uint32_t*>(hist + ((d[e] << 1) & 0x1FFFCu)),
                        __funnelshift_l(1u, 1u, d[e] << 4));
              atomicAdd(reinterpret_cast<uint32_t*>(hist + ((d[e] >> 15) & 0x1FFFCu)),
                        __funnelshift_l(1u, 1u, (d[e] >> 12) & 16u));
            }
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              add(d[e] & 0xffffu, 1);
              add(d[e] >> 16, 1);
            }
          }
        }
      }
      if (b < w1) {  // more to come: room in every count
        __syncthreads();
        uint4* const words = reinterpret_cast<uint4*>(sh.hist);
        uint32_t most = 0;
#pragma unroll
        for (int i = tid; i < 65536 / 8; i += kThreads) {
          const uint4 c = words[i];
          most = __vmaxu2(most, __vmaxu2(__vmaxu2(c.x, c.y), __vmaxu2(c.z, c.w)));
        }
        if ((most & 0xffffu) > kLarge || most >> 16 > kLarge)
          for (int i = tid; i < 65536 / 8; i += kThreads)
            for (int h = 0; h < 8; ++h) {
              uint16_t& n = reinterpret_cast<uint16_t*>(words + i)[h];
              if (n <= kLarge) continue;
              const uint32_t at = atomicAdd(&sh.large, 1u);
              if (at >= kLargeMax) continue;  // more counts than the row has: cannot be
              sh.large_key[at] = 8 * i + h;
              sh.large_count[at] = n;
              n = 0;
            }
        __syncthreads();
      }
    }
    least = __reduce_min_sync(0xffffffffu, min(least & 0xffffu, least >> 16));
    if (lane == 0) atomicMin(&sh.least, least);
  }
  row_sync<kCtas>();
  uint32_t top = 0xFFFFu, large = 0;  // the row's largest value, as a descending key
#pragma unroll
  for (int r = 0; r < kCtas; ++r) {
    top = min(top, *of_rank<kCtas>(&sh.least, r));
    large |= *of_rank<kCtas>(&sh.large, r);
  }
  top += kFirst;

  uint32_t key = top, place = 0;
  if (top < kEnd && temperature != 0.f) {
    const double most = key_value(top);
    // this thread's group of a round, in descending order of keys
    auto group_of = [&](int r) -> uint32_t {
      return kCtas == 1 ? r * kThreads + tid
                        : ((r * (kThreads / 8) + tid / 8) * kCtas + rank) * 8 + tid % 8;
    };
    // Counts of a group's keys, over the cluster.
    auto counts = [&](uint32_t k0, uint32_t (&c)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) c[e] = 0;
      if (k0 < top / 8 * 8 || k0 >= kEnd) return;
#pragma unroll
      for (int r = 0; r < kCtas; ++r) {
        const uint4 v = *reinterpret_cast<const uint4*>(of_rank<kCtas>(sh.hist, r) + k0 / 2);
        const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          c[2 * e] += u[e] & 0xffffu;
          c[2 * e + 1] += u[e] >> 16;
        }
      }
      if (large)
        for (int r = 0; r < kCtas; ++r) {
          const uint32_t n = min(*of_rank<kCtas>(&sh.large, r), (uint32_t)kLargeMax);
          for (uint32_t i = 0; i < n; ++i) {
            const uint32_t k = of_rank<kCtas>(sh.large_key, r)[i] - k0;
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (k == e) c[e] += of_rank<kCtas>(sh.large_count, r)[i];
          }
        }
    };
    // A thread with one group adds up its counts over the cluster once.
    uint32_t group_counts[8];
    if constexpr (kR == 1) counts(group_of(0) * 8, group_counts);
    auto group = [&](int r, uint32_t (&c)[8]) {
      if constexpr (kR == 1) {
#pragma unroll
        for (int e = 0; e < 8; ++e) c[e] = group_counts[e];
      } else {
        counts(group_of(r) * 8, c);
      }
    };
    // top_k: of key `cutoff` the first `leaves` candidates stay, of later ones none.
    uint32_t cutoff = 0xFFFFFFFFu, leaves = 0;
    if (top_k) {
      uint32_t own[kR], before[kR];
#pragma unroll
      for (int r = 0; r < kR; ++r) {
        uint32_t c[8];
        group(r, c);
        own[r] = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) own[r] += c[e];
      }
      row_exclusive<kCtas, uint32_t>(sh, rank, own, before);
      int round = -1;
      uint32_t at = 0;
#pragma unroll
      for (int r = kR - 1; r >= 0; --r)
        if (own[r] && before[r] + own[r] >= top_k) {
          round = r;
          at = before[r];
        }
      uint32_t k = 0, n = 0;
      if (row_first<kCtas>(sh, rank, round >= 0, round >= 0 ? group_of(round) : 0, sh.cutoff,
                           [&](uint32_t (&out)[2]) {
                             uint32_t c[8];
                             group(round, c);
                             bool done = false;
#pragma unroll
                             for (int e = 0; e < 8; ++e) {
                               if (!done && at + c[e] >= top_k) {
                                 out[0] = group_of(round) * 8 + e;
                                 out[1] = top_k - at;
                                 done = true;
                               }
                               at += c[e];
                             }
                           },
                           k, n)) {
        cutoff = k;
        leaves = n;
      }
    }
    // Counts of a round's group that top_k leaves; returns the first key that
    // has one.
    constexpr uint32_t kNone = 0xFFFFFFFFu;
    auto candidates = [&](int r, uint32_t (&c)[8]) -> uint32_t {
      const uint32_t k0 = group_of(r) * 8;
      group(r, c);
      if (k0 + 7 >= cutoff) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          c[e] = k0 + e < cutoff ? c[e] : k0 + e == cutoff ? leaves : 0u;
      }
      uint32_t k1 = kNone;
#pragma unroll
      for (int e = 7; e >= 0; --e)
        if (c[e]) k1 = k0 + e;
      return k1;
    };
    // Runs f(key, count, weight) over the candidates of a round's group.
    auto walk = [&](int r, auto f) {
      uint32_t c[8];
      const uint32_t k0 = group_of(r) * 8, k1 = candidates(r, c);
      if (k1 == kNone) return;
      double w = exp((key_value(k1) - most) * inverse);
      const double step = sh.step[key_bits(k0) >> 10];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (c[e]) f(k0 + e, c[e], w);
        if (k0 + e >= k1) w *= step;
      }
    };
#pragma unroll 1
    for (int r = 0; r < kR; ++r) {
      // the walk without a branch to a key: keys without a count add 0
      const uint32_t k0 = group_of(r) * 8;
      uint32_t c[8];
      const uint32_t k1 = candidates(r, c);
      double sum = 0.0;
      if (k1 != kNone) {
        double w = exp((key_value(k1) - most) * inverse);
        const double step = sh.step[key_bits(k0) >> 10];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          sum += count_value(c[e]) * w;
          if (k0 + e >= k1) w *= step;
        }
      }
      sh.mass[r][tid] = sum;
    }
    double own[kR], before[kR];
#pragma unroll
    for (int r = 0; r < kR; ++r) own[r] = sh.mass[r][tid];
    const double total = row_exclusive<kCtas, double>(sh, rank, own, before);
    // What top_p and min_p keep is a prefix again: the kept sum is the sum at
    // the end of the last kept candidate. Only the groups around a border
    // are looked at one candidate at a time.
    const double limit = top_p >= 1.f ? INFINITY : (double)top_p * total;
    // f(key, kept count, weight, sum before it)
    auto walk_kept = [&](int r, double sum, auto f) {
      walk(r, [&](uint32_t k, uint32_t c, double w) {
        uint32_t n = w >= (double)min_p ? c : 0u;
        if (n && !(sum + (n - 1) * w < limit)) {
          // places j with sum + j w < limit
          uint32_t m = 0;
          if (sum < limit) {
            const double j = ceil((limit - sum) / w);
            m = j >= (double)n ? n : (uint32_t)j;
            if (m && !(sum + (m - 1) * w < limit)) --m;
            else if (m < n && sum + m * w < limit) ++m;
          }
          n = m;
        }
        if (k == top && n == 0) n = 1;  // the first always stays
        if (n) f(k, n, w, sum);
        sum += c * w;
      });
    };
    uint32_t final = 0xFFFFFFFFu;  // order + 1 of the last kept group
    double sum_kept = total;
    if (top_p < 1.f || min_p > 0.f) {
      // weights of a group are at least min_p where its exponents are above
      // log(min_p), none is where they are below; the margin is far above the
      // FP32 errors of both, and the groups between are looked at
      const float least_x = logf(min_p), most_f = key_value_f(top);
      const float inverse_f = (float)inverse;
      const float margin = 1e-3f - 1e-5f * least_x;
      uint32_t mine = 0, border = 0;
      double mine_end = 0.0;
#pragma unroll
      for (int r = 0; r < kR; ++r) {
        const uint32_t k0 = group_of(r) * 8;
        if (!(own[r] > 0.0)) continue;
        const double end = before[r] + own[r];
        const float high_x = (key_value_f(k0) - most_f) * inverse_f;
        const float low_x = (key_value_f(k0 + 7) - most_f) * inverse_f;
        // NaN (an exponent that overflows both ways) is looked at too
        if (end < limit && (min_p == 0.f || low_x > least_x + margin)) {
          mine = group_of(r) + 1;
          mine_end = end;
        } else if (top / 8 == k0 / 8 || (before[r] < limit && !(high_x < least_x - margin))) {
          border |= 1u << r;
        }
      }
      for (; border; border &= border - 1) {
        const int r = __ffs(border) - 1;
        double at = 0.0, end = -1.0;
#pragma unroll
        for (int q = 0; q < kR; ++q) at = q == r ? before[q] : at;
        walk_kept(r, at, [&](uint32_t, uint32_t n, double w, double sum) { end = sum + n * w; });
        if (end >= 0.0 && group_of(r) + 1 > mine) {
          mine = group_of(r) + 1;
          mine_end = end;
        }
      }
      const uint32_t warp_last = __reduce_max_sync(0xffffffffu, mine);
      if (lane == 0 && warp_last) atomicMax(&sh.last, warp_last);
      __syncthreads();
      if (mine && sh.last == mine) {
        sh.kept = mine_end;
        sh.kept_order = mine;
      }
      row_sync<kCtas>();
      final = 0;
#pragma unroll
      for (int r = 0; r < kCtas; ++r) {
        const uint32_t q = *of_rank<kCtas>(&sh.kept_order, r);
        const double e = *of_rank<kCtas>(&sh.kept, r);
        if (q > final) {
          final = q;
          sum_kept = e;
        }
      }
    }
    // The first group whose kept sum exceeds the target: there is one, as
    // uniform is at most 1 - 2^-24 and sums agree to about 1e-15. Groups' sums
    // meet within rounding only, so the first of all is taken, not the one
    // around it.
    const double target = (double)uniform * sum_kept;
    int round = -1;
    double at = 0.0;
#pragma unroll
    for (int r = kR - 1; r >= 0; --r) {
      const uint32_t o = group_of(r) + 1;
      if (own[r] > 0.0 && o <= final && (o == final ? sum_kept : before[r] + own[r]) > target) {
        round = r;
        at = before[r];
      }
    }
    row_first<kCtas>(sh, rank, round >= 0, round >= 0 ? group_of(round) : 0, sh.crossing,
                     [&](uint32_t (&out)[2]) {
                       bool crossed = false;
                       walk_kept(round, at, [&](uint32_t k, uint32_t n, double w, double sum) {
                         if (crossed) return;
                         // its first place whose sum exceeds the target; the last
                         // candidate of the group where rounding leaves none
                         const double j = floor((target - sum) / w);
                         uint32_t m = j <= 0.0 ? 0u : j >= (double)n ? n - 1 : (uint32_t)j;
                         if (sum + (m + 1) * w <= target && m + 1 < n) ++m;
                         else if (m && sum + m * w > target) --m;
                         crossed = sum + (m + 1) * w > target;
                         out[0] = k;
                         out[1] = m;
                       });
                     },
                     key, place);
  }

  // ---- key and place to an index -----------------------------------------------------
  // Each warp takes a run of its CTA's words: equals per warp, then the warp
  // that holds the place looks for it.
  if (top >= kEnd) {
    if (rank == 0 && tid == 0) p.tokens[row] = 0xFFFFFFFFu;
  } else {
    const uint32_t bits = key_bits(key) * 0x10001u;
    const int run = (w1 - w0 + kWarps - 1) / kWarps;
    const int a = min(w1, w0 + warp * run), b = min(w1, a + run);
    auto equal = [&](const uint4& v) {  // a bit for each of the word's equals
      const uint32_t u[4] = {v.x ^ bits, v.y ^ bits, v.z ^ bits, v.w ^ bits};
      uint32_t mask = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        mask |= ((u[e] & 0xffffu) == 0 ? 1u << (2 * e) : 0u) |
                (u[e] >> 16 == 0 ? 2u << (2 * e) : 0u);
      return mask;
    };
    uint32_t equals = 0;
    for (int i = a + lane; i < b; i += 4 * 32) {
      uint4 v[4];
      x.load(v, i, 32, b);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        // borrows of a zero half (or one above it): few words have an equal
        const uint32_t t[4] = {v[k].x ^ bits, v[k].y ^ bits, v[k].z ^ bits, v[k].w ^ bits};
        const uint32_t some = ((t[0] - 0x10001u) & ~t[0]) | ((t[1] - 0x10001u) & ~t[1]) |
                              ((t[2] - 0x10001u) & ~t[2]) | ((t[3] - 0x10001u) & ~t[3]);
        if (some & 0x80008000u) equals += __popc(equal(v[k]));
      }
    }
    equals = __reduce_add_sync(0xffffffffu, equals);
    if (lane == 0) sh.equals[warp] = equals;
    __syncthreads();
    int rest = (int)place;
    if constexpr (kCtas > 1) {
      if (warp == 0) {
        const uint32_t all = __reduce_add_sync(0xffffffffu, sh.equals[lane]);
        if (lane < kCtas) *of_rank<kCtas>(&sh.matches[rank], lane) = all;
      }
      row_sync<kCtas>();
      for (int r = 0; r < rank; ++r) rest -= (int)sh.matches[r];
    }
    for (int q = 0; q < warp; ++q) rest -= (int)sh.equals[q];
    if (rest >= 0 && rest < (int)equals) {
      for (int i = a; i < b; i += 4 * 32) {
        uint4 v[4];
        x.load(v, i + lane, 32, b);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t mask = equal(v[k]);
          int n = __popc(mask), upto = n;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
          }
          const int all = __shfl_sync(0xffffffffu, upto, 31);
          int j = rest - (upto - n);  // of this lane's equals
          if (j >= 0 && j < n) {
            for (; j > 0; --j) mask &= mask - 1;
            p.tokens[row] = 8 * (i + 32 * k + lane) + __ffs(mask) - 1 - x.from;
          }
          rest -= all;
        }
        if (rest < 0) break;
      }
    }
  }
  // no CTA leaves while another reads its shared memory
  if constexpr (kCtas > 1) row_sync<kCtas>();
}

template <int kCtas>
void launch_sample(const Launch& l, const SampleBatch& p) {
  auto kernel = sample_batch_kernel<kCtas>;
  allow_dynamic_smem(kernel, sizeof(Shared<kCtas>));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.rows * kCtas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(Shared<kCtas>);
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
  // As many CTAs to a row as fit the GPU at once, up to 8. Clusters of 8 and 4
  // leave SMs of a GPC empty, which the eighth below stands for (18 rows of
  // 151,936: 28 us with 8, 25 with 4; 36: 34 with 4, 30 with 2; 75 and more:
  // 39 with 1).
  const int sms = l.sm_count - l.sm_count / 8;
  if (p.rows * 8 <= sms)
    launch_sample<8>(l, p);
  else if (p.rows * 4 <= sms)
    launch_sample<4>(l, p);
  else if (p.rows * 2 <= l.sm_count)
    launch_sample<2>(l, p);
  else
    launch_sample<1>(l, p);
}

}  // namespace k
}  // namespace mi
