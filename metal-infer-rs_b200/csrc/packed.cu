// Attention over packed prompts: sequences of different lengths laid end to
// end, grouped heads, causal from the ends (a prefix of keys computed before
// is allowed) or not.
//
//   o = sum_j softmax_j(q . k_j / sqrt(d)) v_j
//
// Tensor-bound: 4 d operations per visible (query, key) pair and head on the
// tcgen05 pipe, with the exponentials (16 per clock and SM) close behind at
// head_dim 128 and ahead of it at 64; each has 0.55 of its pipe, the rest is the
// hand-over between the roles. Long prompts one after another also run at the
// board's power limit (8192 tokens: 1.545 of 1.965 GHz), where instructions cost
// clock: a quarter of the exponentials as polynomials on the FMA pipe shortened
// the softmax and lost 3% all the same.
//
// A CTA takes two row tiles of one sequence and KV head. The rows of a tile
// are the query heads of the group for up to 128 / group tokens, so a short
// prompt still fills a tile and a key tile is read once for the whole group.
// Roles (registers go from the last warpgroup to the softmax):
//   warps 0-3, 4-7  softmax of row tile 0 / 1, one row to a thread: scores from
//                   TMEM, the running maximum and sum in registers, FP16
//                   weights to TMEM; in the end the output
//   warps 8, 9      tcgen05.mma of row tile 0 / 1: S_t = Q_t K^T from shared
//                   memory, O_t += P_t V with P from TMEM. A wait costs a warp
//                   about 170 clocks even when it has nothing to wait for, so
//                   each tile has an issuer, and K and V come under one barrier
//   warp 10         TMA: the query tiles once, then a ring of stages, stage n
//                   holding K tile n and V tile n - 1, which are used together
//   warp 11         zeros over the rows behind a sequence's last value: what
//                   stands there (other sequences, padding) has weight 0, and
//                   0 * NaN would send the row to attention_row
// TMEM holds S, P and O of both tiles with P beside S, so the next key tile's
// scores are computed while the softmax of this one runs and the products
// leave its chain: 80 keys to a tile at head_dim 128 (2 (80 + 40 + 128)
// columns of 512), 128 at 64. With P over S and 128 keys the chain scores ->
// softmax -> values took 3,460 clocks to a tile (a hand-over between the
// roles is 150 to 370 of them) where the products take 1,024.
//
// O is rescaled only when a row's maximum has grown by more than 2^8 since the
// last time, once the product of the step before is done. Weights are taken
// over the row's maximum less 7 binary places, so that they lie below 2^15 and
// use all of FP16's exponents: one is rounded by at most half a step, which is
// 2^-11 of itself or, below 2^-14, 2^-25, and that is 2^-32 of the row's
// largest. The final division by the sum of the same weights takes both factors
// out.
//
// The tensor cores cut each product off at 2^-25 of the accumulator's power of
// two before they add it (measured: beside a first key of weight 1, 131,071
// keys of 2^-25.04 added nothing, of 2^-23.5 0.69 of their sum, and as many
// equal keys lost 6e-4 of their mean, more than the output's rounding). So every
// 8,240 keys (8,192 at head_dim 64) a row puts its output and its sum aside in
// device memory, in FP32, and its accumulators start from 0: what products lose
// then adds up to at most 2^-11.6 whatever the length (16,384 tokens of 32/8
// heads of 128: 2.00 ms without, 2.10 so; 65,536: 31.0 and 32.8).

#include <cuda.h>

#include "device.cuh"
#include "pipeline.cuh"

namespace mi {
namespace k {

namespace {

constexpr int kTile = 128;     // rows of a row tile
constexpr int kThreads = 384;
constexpr uint64_t kWaitNs = 200ull * 1000 * 1000;
constexpr int kLeadBlocks = 4; // key tiles from which row tile 1 starts after row tile 0
constexpr int kAsideKeys = 8192; // keys that are added up in TMEM at most, to whole key tiles
constexpr float kLift = 7.f;    // log2 of a largest weight when the base is set
constexpr float kGrowth = 15.f; // and what it may grow to

struct PackedArgs {
  const __half *q, *k, *v;
  __half* out;
  const uint32_t *query_starts, *key_starts;
  uint32_t* fault;
  int tokens, keys, sequences, qh, kvh, causal;
  int group;        // query heads per KV head
  int heads;        // of them in a row tile
  int head_tiles;   // row tiles to cover the group
  int span;         // tokens of a row tile
  float scale_log2; // log2(e) / sqrt(HD)
  const struct Plan* plan;
  float* parts;     // states of the parts of split work
  // Outputs put aside, for a CTA on every SM (more are never resident): a flag
  // to a place that says whether it is taken, null where no row is that long.
  uint32_t* taken;
  float4* aside;    // [places][2][HD / 4 + 1][kTile]: output, then base and sum
  int places;
};

template <int HD>
struct Packed {
  static constexpr int kKeys = HD == 128 ? 80 : 128;  // of a key tile
  static constexpr uint32_t kQBytes = kTile * HD * 2;
  static constexpr uint32_t kTileBytes = kKeys * HD * 2;  // a K or V tile
  static constexpr int kStages = 4;                       // of a K and a V tile
  static constexpr int kBytes = 1024 /*align*/ + 2 * kQBytes + 2 * kStages * kTileBytes + 512;
  static constexpr int kAside = (kAsideKeys + kKeys - 1) / kKeys;  // key tiles from 0 to aside
  // TMEM columns
  static constexpr uint32_t kS = HD == 128 ? 128 : 192;  // S_1's distance from S_0, which is at 0
  static constexpr uint32_t kP = kKeys;                  // P's distance from its S
  static constexpr uint32_t kO = HD == 128 ? 256 : 384;  // O_0; O_1 is HD further
  static_assert(kP + kKeys / 2 <= kS && kS + kP + kKeys / 2 <= kO && kO + 2 * HD <= 512, "TMEM");
};

// One row by one warp, from the formula, over the first `visible` keys and
// reading no others: rows whose products met infinities or NaN that they do
// not see (0 * NaN among the keys behind a causal row) are computed again this
// way.
template <int HD>
__device__ __noinline__ void attention_row(const __half* q, const __half* k, const __half* v,
                                           size_t stride, int visible, float scale_log2,
                                           __half* out) {
  constexpr int kV = HD / 32;
  const int lane = threadIdx.x & 31;
  float acc[kV] = {}, m = -INFINITY, l = 0.f;
  for (int j0 = 0; j0 < visible; j0 += 32) {
    const int j = j0 + lane;
    float s = -INFINITY;
    if (j < visible) {
      s = 0.f;
      const uint4* kr = reinterpret_cast<const uint4*>(k + (size_t)j * stride);
      const uint4* qr = reinterpret_cast<const uint4*>(q);
#pragma unroll 4
      for (int c = 0; c < HD / 8; ++c) s = chunk_dot(qr[c], kr[c], s);
      s *= scale_log2;
    }
    const float top = fmaxf(m, warp_max(s));
    const float base = top == -INFINITY ? 0.f : top;
    const float keep = m == -INFINITY ? 0.f : exp2f(m - base);
    const float p = j < visible ? exp2f(s - base) : 0.f;
    l = l * keep + warp_sum(p);
#pragma unroll
    for (int e = 0; e < kV; ++e) acc[e] *= keep;
    m = top;
    // these keys' own sum first: one by one, small weights would be lost beside
    // what the row has
    const int n = min(32, visible - j0);
    float sum[kV] = {};
    for (int i = 0; i < n; ++i) {
      const float w = __shfl_sync(0xffffffffu, p, i);
      const __half* vr = v + (size_t)(j0 + i) * stride + lane * kV;
#pragma unroll
      for (int e = 0; e < kV; ++e) sum[e] += w * __half2float(vr[e]);
    }
#pragma unroll
    for (int e = 0; e < kV; ++e) acc[e] += sum[e];
  }
#pragma unroll
  for (int e = 0; e < kV; ++e) out[lane * kV + e] = __float2half_rn(acc[e] / l);
}

// ---- PTX ------------------------------------------------------------------------
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, uint32_t* fault) {
  if (pipe::mbar_try_wait(bar, parity)) return true;
  const uint64_t start = pipe::global_ns();
  while (!pipe::mbar_try_wait(bar, parity))
    if (pipe::global_ns() - start > kWaitNs) {
      report_fault(fault, kFaultTimeout);
      return false;
    }
  return true;
}
// The same by a whole warp, with one answer for all of its lanes.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, uint32_t* fault) {
  return __all_sync(0xffffffffu, wait_for(bar, parity, fault));
}
// Whether a wait would return at once. Asked early, the answer comes while the
// asking warp works: even a wait that is over costs 150 to 200 clocks.
__device__ __forceinline__ bool is_over(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n"
      " mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}"
      : "=r"(ok)
      : "r"(pipe::smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ void arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(pipe::smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar, bool one) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.u32 q, %1, 0;\n"
      " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(
          pipe::smem_u32(bar)),
      "r"((uint32_t)one)
      : "memory");
}
__device__ __forceinline__ void tma_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0,
                                       int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, "
      "{%3, %4, %5}], [%2];" ::"r"(pipe::smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(pipe::smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
__device__ __forceinline__ void tma_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0,
                                       int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, "
      "{%3, %4, %5, %6}], [%2];" ::"r"(pipe::smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(pipe::smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2),
      "r"(c3)
      : "memory");
}
// Shared-memory matrix descriptor of a 128-byte-swizzled operand (version 1),
// low and high word: K-major (Q, K: rows of 64 values of the product's depth),
// 8-row groups 1024 bytes apart; MN-major (V: rows are keys, the depth; 64
// values of N to a row), the next 64 values of N `lead` bytes on, the next 8
// keys 1024 bytes on. A step inside the operand adds its bytes / 16.
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lead) {
  return (addr >> 4) | ((lead >> 4) << 16);
}
constexpr uint32_t kDescHi = (1024 >> 4) | (1u << 14) | (2u << 29);
// Instruction descriptor of kind::f16: F16 operands, F32 result, M = 128.
__host__ __device__ constexpr uint32_t idesc_f16(int n, bool b_mn_major) {
  return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
// The products are issued by a warp that runs their loop as a whole, `one` set
// in one lane: operands of tcgen05.mma live in uniform registers, and a loop
// that one lane runs alone moves each of them there every time (95 clocks to a
// product where the tensor cores take 64).
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc,
                                       bool accumulate, bool one) {
  asm volatile(
      "{\n .reg .pred p, q;\n .reg .b64 x, y;\n"
      " setp.ne.u32 p, %4, 0;\n setp.ne.u32 q, %5, 0;\n"
      " mov.b64 x, {%1, %6};\n mov.b64 y, {%2, %6};\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n}" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"((uint32_t)accumulate), "r"((uint32_t)one),
      "n"(kDescHi)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc,
                                       bool accumulate, bool one) {
  asm volatile(
      "{\n .reg .pred p, q;\n .reg .b64 y;\n"
      " setp.ne.u32 p, %4, 0;\n setp.ne.u32 q, %5, 0;\n"
      " mov.b64 y, {%2, %6};\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n}" ::"r"(d),
      "r"(a), "r"(b_lo), "r"(idesc), "r"((uint32_t)accumulate), "r"((uint32_t)one), "n"(kDescHi)
      : "memory");
}
// 16 or 32 columns of a thread's TMEM lane; r is an array indexed by constants.
__device__ __forceinline__ void tmem_ld16(uint32_t* r, uint32_t addr) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(addr));
}
__device__ __forceinline__ void tmem_ld32(uint32_t* r, uint32_t addr) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
               : "r"(addr));
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
               : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
// Ties loaded registers to this point, so that no use moves above the wait.
__device__ __forceinline__ void tie16(uint32_t* r) {
  asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]));
}
__device__ __forceinline__ void tie32(uint32_t* r) {
  asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two FP32 lanes in one instruction.
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void split(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// What a CTA works on: two row tiles.
struct alignas(16) Work {
  int q0, q1;      // the sequence's query rows
  int k0, keys;    // its first key row, its keys
  int token;       // first token (of the sequence) of row tile 0, -1: nothing
  int blocks[2];   // key tiles that row tile 0 / 1 sees
  int part;        // where a part's state goes, -1: the work is whole
};
static_assert(sizeof(Work) == 32, "two 16-byte words");

// The starts of a sequence and its successor.
struct Starts {
  uint32_t q0, q1, k0, k1;
  __device__ Starts(const PackedArgs& a, int s)
      : q0(a.query_starts[s]), q1(a.query_starts[s + 1]), k0(a.key_starts[s]),
        k1(a.key_starts[s + 1]) {}
  __device__ bool bad(const PackedArgs& a) const {
    return q0 > q1 || q1 > (uint32_t)a.tokens || k0 > k1 || k1 > (uint32_t)a.keys;
  }
};
// Sequence s owns the places floor(start_s / (2 span)) + s and on, which leaves
// it room for its tiles whatever the lengths are.
__device__ __forceinline__ long long first_place(const PackedArgs& a, uint32_t start, int s) {
  return (long long)(start / (uint32_t)(2 * a.span)) + s;
}
// The row tiles from token t on of a sequence.
__device__ __forceinline__ Work work_of(const PackedArgs& a, int key_tile, const Starts& st,
                                        long long t) {
  Work w{(int)st.q0, (int)st.q1, (int)st.k0, (int)(st.k1 - st.k0), -1, {0, 0}, -1};
  const int n = w.q1 - w.q0;
  w.token = t < n ? (int)t : -1;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int last = min((long long)n, t + (i + 1) * a.span) - 1;  // last token of the row tile
    if (w.token < 0 || last < t + i * a.span) continue;
    const long long seen = a.causal ? (long long)w.keys - (n - 1 - last) : w.keys;
    w.blocks[i] = seen > 0 ? (int)((seen + key_tile - 1) / key_tile) : 0;
  }
  return w;
}
// ---- the order of the work ------------------------------------------------------
// All sequences' row tiles, the ones that see most keys first (a counting sort
// by key tiles): the CTAs that start last are then the shortest. Without it the
// longest prompt's tiles may come last: 10 prompts of 20 to 2500 tokens took
// 100 us, 96 so, the plan's launch included. The order among equals depends on
// timing, the results do not.
struct alignas(16) Join {
  Work w;          // the whole work
  int part, parts; // its parts' states
  int pad[2];
};
struct Plan {
  uint32_t count, joins;
  uint32_t pad[6];
  Work work[1];
  __host__ __device__ Join* join(int works) { return reinterpret_cast<Join*>(work + works); }
  __host__ __device__ const Join* join(int works) const {
    return reinterpret_cast<const Join*>(work + works);
  }
};
__device__ __forceinline__ Work work_at_place(const PackedArgs& a, int key_tile, int place) {
  int lo = 0, hi = a.sequences;  // the last sequence that begins at or before it
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (first_place(a, a.query_starts[mid], mid) <= place) lo = mid + 1;
    else hi = mid;
  }
  if (lo == 0) return Work{0, 0, 0, 0, -1, {0, 0}, -1};
  const Starts st(a, lo - 1);
  return work_of(a, key_tile, st, (place - first_place(a, st.q0, lo - 1)) * 2 * a.span);
}

constexpr int kPlanThreads = 1024;
__device__ __forceinline__ void free_places(const PackedArgs& a, int tid) {
  for (int i = tid; a.taken && i < a.places; i += kPlanThreads) a.taken[i] = 0;
}
constexpr int kPlanBins = 2048;  // longer ones share the last

__global__ void __launch_bounds__(kPlanThreads) packed_plan_kernel(const PackedArgs a, Plan* plan,
                                                                   int places, int key_tile) {
  __shared__ uint32_t bins[kPlanBins];
  __shared__ uint32_t sums[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = tid; i < kPlanBins; i += kPlanThreads) bins[i] = 0;
  pdl_wait();
  pdl_trigger();
  free_places(a, tid);
  bool bad = false;
  for (int s = tid; s < a.sequences; s += kPlanThreads) bad |= Starts(a, s).bad(a);
  if (__syncthreads_or(bad)) {
    if (tid == 0) {
      report_fault(a.fault, kFaultStarts);
      plan->count = 0;
    }
    return;
  }
  auto work_at = [&](int place) { return work_at_place(a, key_tile, place); };
  auto bin_of = [&](const Work& w) {  // longest first
    return kPlanBins - 1 - min(kPlanBins - 1, max(w.blocks[0], w.blocks[1]));
  };
  for (int i = tid; i < places; i += kPlanThreads) {
    const Work w = work_at(i);
    if (w.token >= 0) atomicAdd(&bins[bin_of(w)], 1u);
  }
  __syncthreads();
  // sums before each bin, two bins to a thread
  const uint32_t b0 = bins[2 * tid], b1 = bins[2 * tid + 1];
  uint32_t x = b0 + b1;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) sums[warp] = x;
  __syncthreads();
  uint32_t base = 0, all = 0;
  for (int q = 0; q < 32; ++q) {
    if (q < warp) base += sums[q];
    all += sums[q];
  }
  bins[2 * tid] = base + x - b0 - b1;
  bins[2 * tid + 1] = base + x - b1;
  if (tid == 0) plan->count = all;
  __syncthreads();
  for (int i = tid; i < places; i += kPlanThreads) {
    const Work w = work_at(i);
    if (w.token >= 0) plan->work[atomicAdd(&bins[bin_of(w)], 1u)] = w;
  }
}
static_assert(kPlanBins == 2 * kPlanThreads, "two bins to a thread");

// ---- work split along its keys ------------------------------------------------------
// Few queries over many keys are a few row tiles with very much each, and a few
// waves of row tiles over long prefixes leave most SMs without work in the last
// wave. The work that does not fill a wave (the shortest) is cut along its keys
// into as many parts as there are places left in that wave (a part is work like
// any other over keys of its own), which leave their rows' maxima, sums and
// unnormalised outputs, and a last kernel joins them in order. With 32/8 heads
// of 128, 64 queries over 65,536 keys take 906 us in one piece and 103 so, 1,300
// over 9,300 (1.1 waves) 245 and 209, 1,200 over 5,200 122 and 108.
constexpr int kPartLeast = 8;       // key tiles of a part at least
constexpr int kSplitPlaces = 512;  // of a call that is split, at most (each is ranked among all)
constexpr int kSplitRest = 512;    // SMs and one, at most

__global__ void __launch_bounds__(kPlanThreads) packed_split_kernel(const PackedArgs a, Plan* plan,
                                                                    int places, int works,
                                                                    int key_tile, int columns,
                                                                    int sm_count) {
  // Never more works than `works`, nor parts than states: the parts have `room`.
  __shared__ int length[kSplitPlaces];  // key tiles of a place's work, -1: none
  __shared__ int rest[kSplitRest];      // of the works that are cut, from long to short
  __shared__ uint32_t count, states, joins;
  __shared__ int part_most;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) count = states = joins = 0;
  pdl_wait();
  pdl_trigger();
  free_places(a, tid);
  bool bad = false;
  for (int s = tid; s < a.sequences; s += kPlanThreads) bad |= Starts(a, s).bad(a);
  if (__syncthreads_or(bad)) {
    if (tid == 0) {
      report_fault(a.fault, kFaultStarts);
      plan->count = plan->joins = 0;
    }
    return;
  }
  Work w;  // of place `tid`
  w.token = -1;
  if (tid < places) w = work_at_place(a, key_tile, tid);
  const int mine = w.token < 0 ? -1 : max(w.blocks[0], w.blocks[1]);
  if (tid < kSplitPlaces) length[tid] = mine;
  const int n = __syncthreads_count(w.token >= 0);
  // its place in the order from long to short
  int order = 0;
  if (tid < places)
    for (int j = 0; j < places; ++j)
      order += length[j] > mine || (length[j] == mine && j < tid);
  // the works that fill whole waves, and the places of the wave behind them
  const int waves = (int)((long long)n * columns / sm_count);
  const int whole = (int)((long long)waves * sm_count / columns);
  const int room = (int)(((long long)(waves + 1) * sm_count - (long long)whole * columns) / columns);
  if (w.token >= 0 && order >= whole) rest[order - whole] = mine;
  __syncthreads();
  if (warp == 0) {  // the least length of a part at which all parts have room
    const int many = n - whole;  // <= sm_count / columns + 1
    auto parts_of = [&](int most) {
      uint32_t parts = 0;
      for (int i = lane; i < many; i += 32) parts += max(1, (rest[i] + most - 1) / most);
      return (int)__reduce_add_sync(0xffffffffu, parts);
    };
    int lo = kPartLeast, hi = many > 0 ? max(kPartLeast, rest[0]) : kPartLeast;
    while (lo < hi) {
      const int most = (lo + hi) / 2;
      if (parts_of(most) <= room) hi = most;
      else lo = most + 1;
    }
    if (lane == 0) part_most = lo;
  }
  __syncthreads();
  const int most = part_most;
  if (w.token >= 0 && order < whole) {
    plan->work[order] = w;
  } else if (w.token >= 0) {
    int parts = max(1, (mine + most - 1) / most);
    const int per = (mine + parts - 1) / parts;
    if (mine > 0) parts = (mine + per - 1) / per;
    const int at = whole + (int)atomicAdd(&count, (uint32_t)parts);
    const int state = parts > 1 ? (int)atomicAdd(&states, (uint32_t)parts) : 0;
    if (parts == 1) plan->work[at] = w;
    else plan->join(works)[atomicAdd(&joins, 1u)] = Join{w, state, parts, {0, 0}};
    for (int q = 0; parts > 1 && q < parts; ++q) {
      Work v = w;
      v.k0 += q * per * key_tile;
      v.keys -= q * per * key_tile;
      for (int t = 0; t < 2; ++t)
        v.blocks[t] = max(0, min(w.blocks[t], (q + 1) * per) - q * per);
      v.part = state + q;
      plan->work[at + q] = v;
    }
  }
  __syncthreads();
  if (tid == 0) {
    plan->count = whole + count;
    plan->joins = joins;
  }
}
static_assert(kSplitPlaces <= kPlanThreads, "a place to a thread");

// Floats of a part's state: (base, sum) and output of 2 x 128 rows.
constexpr size_t part_floats(int hd) { return 2 * kTile * (2 + (size_t)hd); }

// What a row is: token and head of the group, keys that it sees.
struct RowOf {
  int token, head, visible;
  bool valid;
  __device__ RowOf(const PackedArgs& a, const Work& w, int head0, int t, int row) {
    const int n = w.q1 - w.q0;
    token = w.token + t * a.span + row / a.heads;
    head = head0 + row % a.heads;
    valid = row < a.heads * a.span && token < n && head < a.group;
    const long long seen = a.causal ? (long long)w.keys - (n - 1 - token) : w.keys;
    visible = valid && seen > 0 ? (int)seen : 0;
  }
};

// A row to a warp.
template <int HD>
__global__ void __launch_bounds__(256) packed_join_kernel(const PackedArgs a, int works) {
  constexpr int kV = HD / 32;
  pdl_wait();
  pdl_trigger();
  const int columns = a.kvh * a.head_tiles;
  const int index = (int)(blockIdx.x / (uint32_t)columns);
  if (index >= (int)a.plan->joins) return;
  const Join j = a.plan->join(works)[index];
  const int column = (int)(blockIdx.x % (uint32_t)columns);
  const int lane = threadIdx.x & 31;
  const int r = blockIdx.y * 8 + (threadIdx.x >> 5);
  const int t = r / kTile, row = r % kTile;
  const int kv = column / a.head_tiles;
  const RowOf me(a, j.w, column % a.head_tiles * a.heads, t, row);
  if (!me.valid) return;
  const size_t at =
      ((size_t)(j.w.q0 + me.token) * a.qh + (size_t)kv * a.group + me.head) * HD;
  auto state = [&](int q) {
    return a.parts + ((size_t)(j.part + q) * columns + column) * part_floats(HD);
  };
  float top = -INFINITY;
  for (int q = lane; q < j.parts; q += 32) top = fmaxf(top, state(q)[2 * r]);
  top = warp_max(top);
  float acc[kV] = {}, total = 0.f;
#pragma unroll 4
  for (int q = 0; q < j.parts; ++q) {
    const float* s = state(q);
    const float2 ml = *reinterpret_cast<const float2*>(s + 2 * r);
    if (ml.x == -INFINITY && ml.y == 0.f) continue;  // sees nothing of this part
    const float w = ml.x == -INFINITY ? 0.f : exp2_fast(ml.x - top);
    total += w * ml.y;
    const float* o = s + 4 * kTile + (size_t)r * HD + lane * kV;
#pragma unroll
    for (int e = 0; e < kV; ++e) acc[e] += w * o[e];
  }
  bool odd = false;
  const float inv = 1.f / total;
#pragma unroll
  for (int e = 0; e < kV; ++e) {
    acc[e] = me.visible > 0 ? acc[e] * inv : 0.f;
    odd |= !(acc[e] * 0.f == 0.f);
    a.out[at + lane * kV + e] = __float2half_rn(acc[e]);
  }
  if (__any_sync(0xffffffffu, odd) && me.visible > 0) {
    const size_t stride = (size_t)a.kvh * HD;
    attention_row<HD>(a.q + at, a.k + (size_t)j.w.k0 * stride + kv * HD,
                      a.v + (size_t)j.w.k0 * stride + kv * HD, stride, me.visible, a.scale_log2,
                      a.out + at);
  }
}

// A free place for outputs put aside, by one thread: the SM's own, which the CTA
// before this one has given back (any other free one would do).
__device__ __forceinline__ int take_place(const PackedArgs& a) {
  uint32_t sm;
  asm volatile("mov.u32 %0, %%smid;" : "=r"(sm));
  for (int n = 0; n < 4 * a.places; ++n) {
    const int i = (int)((sm + n) % (uint32_t)a.places);
    if (atomicCAS(a.taken + i, 0u, 1u) == 0u) {
      __threadfence();
      return i;
    }
  }
  return -1;
}
// What a sum over base `from` is worth over base `to`.
__device__ __forceinline__ float rebase(float from, float to) {
  return from == to ? 1.f : from == -INFINITY ? 0.f : exp2_fast(from - to);
}

// A row's output and sum of weights go from the accumulators to the row's place
// aside, on top of what is there, and in the end come back: `at` is that of its
// first four values, `m` the base of the accumulators. Both are rare, and calls,
// so that they take no registers from the softmax.
template <int HD>
__device__ __noinline__ void put_aside(uint32_t to, float4* at, bool first, float m, float l) {
  float4* const stats = at + HD / 4 * kTile;
  const float2 before = first ? make_float2(m, 0.f) : *reinterpret_cast<const float2*>(stats);
  const float factor = rebase(before.x, m);
  *reinterpret_cast<float2*>(stats) = make_float2(m, factor * before.y + l);
#pragma unroll 1
  for (int c = 0; c < HD; c += 64) {
    float4 v[16] = {};
    if (!first)
#pragma unroll
      for (int q = 0; q < 16; ++q) v[q] = at[(c / 4 + q) * kTile];
    uint32_t o[64];
    tmem_ld32(o, to + c);
    tmem_ld32(o + 32, to + c + 32);
    tmem_wait_ld();
    tie32(o);
    tie32(o + 32);
#pragma unroll
    for (int q = 0; q < 16; ++q)
      at[(c / 4 + q) * kTile] = make_float4(factor * v[q].x + __uint_as_float(o[4 * q]),
                                            factor * v[q].y + __uint_as_float(o[4 * q + 1]),
                                            factor * v[q].z + __uint_as_float(o[4 * q + 2]),
                                            factor * v[q].w + __uint_as_float(o[4 * q + 3]));
  }
}
// Returns the sum.
template <int HD>
__device__ __noinline__ float take_back(uint32_t to, const float4* at, float m, float l) {
  const float2 before = *reinterpret_cast<const float2*>(at + HD / 4 * kTile);
  const float factor = rebase(before.x, m);
#pragma unroll 1
  for (int c = 0; c < HD; c += 64) {
    float4 v[16];
#pragma unroll
    for (int q = 0; q < 16; ++q) v[q] = at[(c / 4 + q) * kTile];
    uint32_t o[64];
    tmem_ld32(o, to + c);
    tmem_ld32(o + 32, to + c + 32);
    tmem_wait_ld();
    tie32(o);
    tie32(o + 32);
#pragma unroll
    for (int q = 0; q < 16; ++q) {
      const float x[4] = {v[q].x, v[q].y, v[q].z, v[q].w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        o[4 * q + e] = __float_as_uint(factor * x[e] + __uint_as_float(o[4 * q + e]));
    }
    tmem_st32(to + c, o);
    tmem_st32(to + c + 32, o + 32);
  }
  tmem_wait_st();
  return factor * before.y + l;
}

// How a CTA comes by its work: it looks for its place, it is in the plan's
// order, or it is in a plan that splits it. kLong: rows may be long enough to be
// put aside (a call of more keys than that; the others' softmax is spared what
// the registers for it cost: 8192 tokens, a call at a time, 452 us, 460 with it).
enum Mode { kOwnPlace, kPlanned, kSplit };
template <int HD, Mode kMode, bool kLong>
__global__ void __launch_bounds__(kThreads, 1)
    packed_kernel(const __grid_constant__ CUtensorMap map_q,
                  const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const PackedArgs a) {
  using C = Packed<HD>;
  constexpr int kStages = C::kStages, kKeys = C::kKeys;
  constexpr int kHalves = HD / 64;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* ring = smem + 2 * C::kQBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + 2 * kStages * C::kTileBytes);
  uint64_t* q_full = bars;         // [1]
  uint64_t* s_full = bars + 1;     // [2] scores are in TMEM
  uint64_t* s_free = bars + 3;     // [2] and have been read
  uint64_t* p_full = bars + 5;     // [2] weights are in TMEM
  uint64_t* o_full = bars + 7;     // [2] their product is done
  uint64_t* lead = bars + 9;       // tile 0 has its first maximum
  uint64_t* kv_full = bars + 10;   // [kStages]
  uint64_t* kv_empty = kv_full + kStages;
  uint64_t* tail_full = bars + 20; // the last V tile, before its end is zero
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(kv_empty + kStages);
  Work* work = reinterpret_cast<Work*>(bars + 24);
  int* place_slot = reinterpret_cast<int*>(bars + 28);  // of outputs put aside

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // heads of one place side by side: their key tiles are near each other
  const int columns = a.kvh * a.head_tiles;
  const int place_y = (int)(blockIdx.x / (uint32_t)columns);
  const int kv = (int)(blockIdx.x % (uint32_t)columns) / a.head_tiles;
  const int head0 = (int)(blockIdx.x % (uint32_t)a.head_tiles) * a.heads;  // first of the group

  if (tid == 0) {
    pipe::mbar_init(q_full, 1);
    pipe::mbar_init(lead, 4);
    pipe::mbar_init(tail_full, 1);
    for (int i = 0; i < 2; ++i) {
      pipe::mbar_init(s_full + i, 1);
      pipe::mbar_init(s_free + i, 4);
      pipe::mbar_init(p_full + i, 4);
      pipe::mbar_init(o_full + i, 1);
    }
    for (int i = 0; i < kStages; ++i) {
      pipe::mbar_init(kv_full + i, 1);
      pipe::mbar_init(kv_empty + i, 2);  // both tiles' issuers
    }
    pipe::fence_mbar_init();
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_q)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_k)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_v)) : "memory");
    work->token = -1;
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     pipe::smem_u32(tmem_slot)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if constexpr (kMode == kOwnPlace) __syncthreads();
  pdl_wait();
  pdl_trigger();

  // ---- which tokens ------------------------------------------------------------
  Work w;
  bool bad = false;
  if constexpr (kMode != kOwnPlace) {
    w.token = -1;
    if (place_y < (int)a.plan->count) {
      const uint4* src = reinterpret_cast<const uint4*>(&a.plan->work[place_y]);
      reinterpret_cast<uint4*>(&w)[0] = src[0];
      reinterpret_cast<uint4*>(&w)[1] = src[1];
    }
  } else {
    // A place lies in one sequence or in none. Late places first: with a causal
    // mask they are the longest of their prompt.
    const int place = (int)(gridDim.x / (uint32_t)columns) - 1 - place_y;
    for (int s = tid; s < a.sequences; s += kThreads) {
      const Starts st(a, s);
      bad |= st.bad(a);
      const long long f = first_place(a, st.q0, s);
      if (f <= place && place < first_place(a, st.q1, s + 1))
        *work = work_of(a, kKeys, st, (place - f) * 2 * a.span);
    }
  }
  fence_before();
  bad = __syncthreads_or(bad);
  fence_after();
  if constexpr (kMode == kOwnPlace) w = *work;
  if (bad || w.token < 0) {  // starts that do not rise or leave their rows, or nothing to do
    if (bad && tid == 0) report_fault(a.fault, kFaultStarts);
    if (warp == 8)
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(*tmem_slot),
                   "r"(512)
                   : "memory");
    return;
  }
  const int blocks = max(w.blocks[0], w.blocks[1]);
  const uint32_t tmem = *tmem_slot;
  if (kLong && blocks > C::kAside) {
    if (tid == 0) *place_slot = take_place(a);
    __syncthreads();
    if (*place_slot < 0) {  // cannot be: there is one for every resident CTA
      if (tid == 0) report_fault(a.fault, kFaultTimeout);
      if (warp == 8)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512)
                     : "memory");
      return;
    }
  }
  // rows of the CTA's last V tile that are its sequence's, 0: all
  const int tail = blocks > 0 && blocks == (w.keys + kKeys - 1) / kKeys ? w.keys % kKeys : 0;

  if (warp >= 8) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
  if (warp == 11) {
    if (tail && warp_wait(tail_full, 0, a.fault)) {
      const int st = blocks % kStages;
      uint8_t* at = ring + (2 * st + 1) * C::kTileBytes + tail * 128;
      for (int h = 0; h < kHalves; ++h)
        for (int i = lane; i < (kKeys - tail) * 8; i += 32)
          reinterpret_cast<uint4*>(at + h * (kKeys * 128))[i] = make_uint4(0, 0, 0, 0);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) arrive(kv_full + st);
    }
  } else if (warp == 10) {
    if (lane == 0 && blocks > 0) {
      // ---- TMA ------------------------------------------------------------------
      pipe::mbar_expect_tx(q_full, 2u * kHalves * a.heads * a.span * 128u);
      for (int t = 0; t < 2; ++t)
        for (int h = 0; h < kHalves; ++h)
          tma_4d(smem + t * C::kQBytes + h * (kTile * 128), &map_q, q_full, h * 64, head0, kv,
                 w.q0 + w.token + t * a.span);
      int n = 0;
      for (; n <= blocks; ++n) {
        const int st = n % kStages;
        if (!wait_for(kv_empty + st, ((n / kStages) & 1) ^ 1, a.fault)) break;
        uint8_t* at = ring + 2 * st * C::kTileBytes;
        // a V tile with an end is full when that is zero
        uint64_t* full = n == blocks && tail ? tail_full : kv_full + st;
        pipe::mbar_expect_tx(full, ((n < blocks ? 1u : 0u) + (n > 0 ? 1u : 0u)) * C::kTileBytes);
        for (int h = 0; h < kHalves; ++h) {
          if (n < blocks)
            tma_3d(at + h * (kKeys * 128), &map_k, full, h * 64, kv, w.k0 + n * kKeys);
          if (n > 0)
            tma_3d(at + C::kTileBytes + h * (kKeys * 128), &map_v, full, h * 64, kv,
                   w.k0 + (n - 1) * kKeys);
        }
      }
      // the copies land before the CTA leaves
      wait_for(q_full, 0, a.fault);
      if (n > blocks && tail) wait_for(tail_full, 0, a.fault);
      for (int i = max(0, n - kStages); i < n; ++i)
        wait_for(kv_full + i % kStages, (i / kStages) & 1, a.fault);
    }
  } else if (warp >= 8) {
    if (blocks > 0) {
      // ---- products -----------------------------------------------------------------
      constexpr uint32_t idesc_s = idesc_f16(kKeys, false);
      constexpr uint32_t idesc_o = idesc_f16(HD, true);
      const bool one = elect_one();
      const int t = __shfl_sync(0xffffffffu, warp - 8, 0);
      const int mine = __shfl_sync(0xffffffffu, w.blocks[t], 0);
      const uint32_t q_lo = desc_lo(pipe::smem_u32(smem) + t * C::kQBytes, 16);
      const uint32_t k_lo = desc_lo(pipe::smem_u32(ring), 16);
      const uint32_t v_lo = desc_lo(pipe::smem_u32(ring) + C::kTileBytes, kKeys * 128);
      const uint32_t d_s = tmem + t * C::kS, d_p = d_s + C::kP, d_o = tmem + C::kO + t * HD;
      bool ok = wait_for(q_full, 0, a.fault);
      // The tiles' softmaxes share the exponential unit; begun together they
      // would stay in step, both at their exponentials and then neither. Tile
      // 1 begins when tile 0 has its first maximum (head_dim 64, prompts over
      // prefixes: 136 us in step, 128 so; no difference at 128).
      if (t == 1 && min(w.blocks[0], w.blocks[1]) >= kLeadBlocks)
        ok = ok && wait_for(lead, 0, a.fault);
      // stage n: the scores of key tile n, then the values of n - 1
      int st = 0, fresh = 0;  // `fresh`: the next key tile whose products start from 0
      uint32_t phase = 0;
      for (int n = 0; n <= blocks && ok; ++n) {
        ok = wait_for(kv_full + st, phase, a.fault);
        if (n < mine) {
          if (n > 0) ok = ok && wait_for(s_free + t, (n - 1) & 1, a.fault);
          fence_after();
          if (ok) {
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk)
              mma_ss(d_s, q_lo + ((kk / 4) * (kTile * 128) + (kk % 4) * 32) / 16,
                     k_lo + (2 * st * C::kTileBytes + (kk / 4) * (kKeys * 128) + (kk % 4) * 32) / 16,
                     idesc_s, kk != 0, one);
            commit(s_full + t, one);
          }
        }
        if (n > 0 && n <= mine) {
          ok = ok && wait_for(p_full + t, (n - 1) & 1, a.fault);
          fence_after();
          if (ok) {
#pragma unroll
            for (int kk = 0; kk < kKeys / 16; ++kk)
              mma_ts(d_o, d_p + kk * 8, v_lo + (2 * st * C::kTileBytes + kk * 2048) / 16, idesc_o,
                     n - 1 != fresh || kk != 0, one);
            if (kLong && n - 1 == fresh) fresh += C::kAside;
            commit(o_full + t, one);
          }
        }
        commit(kv_empty + st, one);
        if (++st == kStages) st = 0, phase ^= 1;
      }
    }
  } else {
    // ---- softmax -------------------------------------------------------------------
    // 8 warps of 208 and 4 of 88 registers: the launch's 12 of 168
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int t = warp >> 2;                // row tile
    const int row = (warp & 3) * 32 + lane; // of the tile: the TMEM lane
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + t * C::kS;
    const uint32_t tp = ts + C::kP;
    const uint32_t to = tmem + lanes + C::kO + t * HD;
    const int n = w.q1 - w.q0;
    const RowOf me(a, w, head0, t, row);
    const int token = me.token, head = me.head, visible = me.visible;
    const bool valid = me.valid;
    // keys that every row of the tile sees
    const long long least =
        a.causal ? (long long)w.keys - (n - 1 - (w.token + t * a.span)) : w.keys;
    const int mine = w.blocks[t];
    float m = -INFINITY;  // the row's base: its maximum when it was set, less kLift
    uint64_t l2 = 0;  // two partial sums
    const uint64_t scale2 = pair_of(a.scale_log2, a.scale_log2);
    // this row's place aside
    auto aside = [&] {
      return a.aside + ((size_t)*place_slot * 2 + t) * (HD / 4 + 1) * kTile + row;
    };
    bool ok = true, scored = false;
    // key tiles whose products one accumulator takes
    for (int first = 0; ok && first < mine; first += kLong ? C::kAside : mine) {
      if (kLong && first > 0) {
        ok = warp_wait(o_full + t, (first - 1) & 1, a.fault);
        if (!ok) break;
        fence_after();
        float la, lb;
        split(l2, la, lb);
        put_aside<HD>(to, aside(), first == C::kAside, m, la + lb);
        l2 = 0;
      }
      const int last = kLong ? min(mine, first + C::kAside) : mine;
      for (int i = first; i < last; ++i) {
        if (!__all_sync(0xffffffffu, scored)) ok = warp_wait(s_full + t, i & 1, a.fault);
        if (!ok) break;
        fence_after();
        uint32_t s[kKeys];
#pragma unroll
        for (int c = 0; c + 32 <= kKeys; c += 32) tmem_ld32(s + c, ts + c);
        if constexpr (kKeys % 32 != 0) tmem_ld16(s + kKeys - 16, ts + kKeys - 16);
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c + 32 <= kKeys; c += 32) tie32(s + c);
        if constexpr (kKeys % 32 != 0) tie16(s + kKeys - 16);
        fence_before();
        __syncwarp();
        if (lane == 0) arrive(s_free + t);
        const int k0 = i * kKeys;
        if (k0 + kKeys > least) {
          const int left = visible - k0;
#pragma unroll
          for (int e = 0; e < kKeys; ++e)
            if (e >= left) s[e] = 0xff800000u;  // -inf
        }
        // a NaN or +inf that the row sees ends in the maximum
        float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < kKeys; e += 2)
          tops[(e >> 1) & 3] = max3_nan(tops[(e >> 1) & 3], __uint_as_float(s[e]),
                                        __uint_as_float(s[e + 1]));
        float top = max3_nan(max3_nan(tops[0], tops[1], tops[2]), tops[3], -INFINITY) * a.scale_log2;
        if (!(top < INFINITY)) {  // the row ends as NaN, and is done again below
          l2 = pair_of(__int_as_float(0x7fc00000), 0.f);
          top = m;
        }
        // a maximum that grew past the bound moves the row's base
        const bool grown = top > m + kGrowth || (m == -INFINITY && top > m);
        if (__any_sync(0xffffffffu, grown)) {
          const float base = grown ? top - kLift : m;
          const float factor = !grown ? 1.f : m == -INFINITY ? 0.f : exp2_fast(m - base);
          m = base;
          if (i > first) {
            l2 = fma2(l2, pair_of(factor, factor), 0);
            ok = warp_wait(o_full + t, (i - 1) & 1, a.fault);
            if (!ok) break;
            fence_after();
#pragma unroll 1
            for (int c = 0; c < HD; c += 32) {
              uint32_t o[32];
              tmem_ld32(o, to + c);
              tmem_wait_ld();
              tie32(o);
#pragma unroll
              for (int e = 0; e < 32; ++e)
                o[e] = __float_as_uint(__uint_as_float(o[e]) * factor);
              tmem_st32(to + c, o);
            }
          }
        }
        if (i == 0 && t == 0 && lane == 0) arrive(lead);
        // P is free once the product of the step before is done
        const bool free = i == first || is_over(o_full + t, (i - 1) & 1);
        const float base = m == -INFINITY ? 0.f : -m;
        const uint64_t base2 = pair_of(base, base);
        uint32_t p[kKeys / 2];
#pragma unroll
        for (int e = 0; e < kKeys / 2; ++e) {
          const uint64_t x = fma2(pair_of(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])),
                                  scale2, base2);
          float w0, w1;
          split(x, w0, w1);
          w0 = exp2_fast(w0);
          w1 = exp2_fast(w1);
          // the sum takes the weights before their rounding to FP16
          l2 = add2(l2, pair_of(w0, w1));
          const __half2 h = __floats2half2_rn(w0, w1);
          p[e] = *reinterpret_cast<const uint32_t*>(&h);
        }
        if (!__all_sync(0xffffffffu, free)) ok = warp_wait(o_full + t, (i - 1) & 1, a.fault);
        if (!ok) break;
        fence_after();
        scored = i + 1 < mine && is_over(s_full + t, (i + 1) & 1);
#pragma unroll
        for (int c = 0; c + 32 <= kKeys / 2; c += 32) tmem_st32(tp + c, p + c);
        if constexpr (kKeys % 64 != 0) tmem_st8(tp + kKeys / 2 - 8, p + kKeys / 2 - 8);
        tmem_wait_st();
        fence_before();
        __syncwarp();
        if (lane == 0) arrive(p_full + t);
      }
    }
    // ---- output ---------------------------------------------------------------------
    const size_t stride = (size_t)a.kvh * HD;
    const size_t at = ((size_t)(w.q0 + token) * a.qh + (size_t)kv * a.group + head) * HD;
    if (mine > 0 && ok && warp_wait(o_full + t, (mine - 1) & 1, a.fault)) {
      fence_after();
      float la, lb;
      split(l2, la, lb);
      if (kLong && mine > C::kAside) {
        la = take_back<HD>(to, aside(), m, la + lb);
        lb = 0.f;
      }
      if (kMode == kSplit && w.part >= 0) {
        float* state = a.parts + ((size_t)w.part * columns + blockIdx.x % (uint32_t)columns) *
                                     part_floats(HD);
        const int r = t * kTile + row;
        // a row that saw only scores of -inf is done again, as its values count
        const float sum = m == -INFINITY && visible > 0 ? __int_as_float(0x7fc00000) : la + lb;
        if (valid) *reinterpret_cast<float2*>(state + 2 * r) = make_float2(m, sum);
#pragma unroll 1
        for (int c = 0; c < HD; c += 32) {
          uint32_t o[32];
          tmem_ld32(o, to + c);
          tmem_wait_ld();
          tie32(o);
          float4* dst = reinterpret_cast<float4*>(state + 4 * kTile + (size_t)r * HD + c);
#pragma unroll
          for (int q = 0; q < 8; ++q)
            if (valid)
              dst[q] = make_float4(__uint_as_float(o[4 * q]), __uint_as_float(o[4 * q + 1]),
                                   __uint_as_float(o[4 * q + 2]), __uint_as_float(o[4 * q + 3]));
        }
      } else {
        const float inv = 1.f / (la + lb);
        uint64_t odd2 = 0;  // stays 0 while all is finite: a sum of 0 * value
        const uint64_t inv2 = pair_of(inv, inv);
        // The rows go through this tile's query tile in shared memory, which its
        // products have read, so that they leave as whole lines: a row to a
        // thread touches a line with every 16 bytes (5,100 clocks to a CTA, 2,900 so).
        uint8_t* stage = smem + t * C::kQBytes + (warp & 3) * 32 * (HD * 2);
        constexpr int kChunks = HD / 8;
#pragma unroll
        for (int c = 0; c < HD; c += 32) {
          uint32_t o[32];
          tmem_ld32(o, to + c);
          tmem_wait_ld();
          tie32(o);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint4 v;
            __half2* hv = reinterpret_cast<__half2*>(&v);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint64_t z = mul2(pair_of(__uint_as_float(o[q * 8 + 2 * e]),
                                              __uint_as_float(o[q * 8 + 2 * e + 1])),
                                      inv2);
              odd2 = fma2(z, 0, odd2);
              float x, y;
              split(z, x, y);
              hv[e] = __floats2half2_rn(x, y);
            }
            if (visible == 0) v = make_uint4(0, 0, 0, 0);
            const int chunk = c / 8 + q;
            *reinterpret_cast<uint4*>(stage + lane * (HD * 2) + ((chunk ^ (lane & 7)) << 4)) = v;
          }
        }
        __syncwarp();
        const unsigned long long mine_at = valid ? (unsigned long long)at : ~0ull;
#pragma unroll 4
        for (int r = lane / kChunks; r < 32; r += 32 / kChunks) {
          const unsigned long long to_row = __shfl_sync(0xffffffffu, mine_at, r);
          const int chunk = lane % kChunks;
          if (to_row != ~0ull)
            reinterpret_cast<uint4*>(a.out + to_row)[chunk] = *reinterpret_cast<const uint4*>(
                stage + r * (HD * 2) + ((chunk ^ (r & 7)) << 4));
        }
        __syncwarp();
        float odd0, odd1;
        split(odd2, odd0, odd1);
        unsigned again = __ballot_sync(0xffffffffu, !(odd0 + odd1 == 0.f) && visible > 0);
        while (again) {
          const int who = __ffs(again) - 1;
          again &= again - 1;
          const int seen_w = __shfl_sync(0xffffffffu, visible, who);
          const unsigned long long at_w = __shfl_sync(0xffffffffu, (unsigned long long)at, who);
          attention_row<HD>(a.q + at_w, a.k + (size_t)w.k0 * stride + kv * HD,
                            a.v + (size_t)w.k0 * stride + kv * HD, stride, seen_w, a.scale_log2,
                            a.out + at_w);
        }
      }
    } else if (kMode == kSplit && mine == 0 && w.part >= 0) {
      float* state = a.parts + ((size_t)w.part * columns + blockIdx.x % (uint32_t)columns) *
                                   part_floats(HD);
      if (valid)
        *reinterpret_cast<float2*>(state + 2 * (t * kTile + row)) = make_float2(-INFINITY, 0.f);
    } else if (mine == 0 && valid) {
      for (int c = 0; c < HD / 8; ++c)
        reinterpret_cast<uint4*>(a.out + at)[c] = make_uint4(0, 0, 0, 0);
    }
  }
  fence_before();
  __syncthreads();
  if (kLong && tid == 0 && blocks > C::kAside) {
    __threadfence();
    atomicExch(a.taken + *place_slot, 0u);
  }
  if (warp == 8) {
    __syncwarp();
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512)
                 : "memory");
  }
}

// From how many keys, saved on the longest way through a call, its split pays
// for two launches, the parts' beginnings and their states, some 15 us in all
// (32/8 heads of 128, in one piece and split: 64 queries over 2,048 keys 34 and
// 28 us; 32 over 1,024 16 and 20; 512 over 2,048 35 and 40; 1,300 over 2,600 55
// and 63).
constexpr int kSplitKeys = 1800;
constexpr int kSplitWaves = 8;  // the wave that is cut is a small part of more

// Heads of a row tile, its tokens, and the places of a call's row tile pairs.
struct Shape {
  int head_tiles, heads, span;
  long long places;
  Mode mode;
  int works, states, joins;  // a split plan's most
};
Shape shape_of(const PackedAttention& p, int sm_count) {
  Shape s;
  const int group = p.qh / p.kvh;
  s.head_tiles = (group + kTile - 1) / kTile;
  s.heads = (group + s.head_tiles - 1) / s.head_tiles;
  s.span = kTile / s.heads;
  s.places = (long long)p.tokens / (2 * s.span) + p.sequences;
  // One sequence's tiles are in order as they are, and so is what fits the GPU
  // about at once: the plan is a launch of some 4 us.
  const long long columns = p.kvh * s.head_tiles;
  const long long items = s.places * columns;
  s.mode = p.sequences > 1 && items > 2 * sm_count ? kPlanned : kOwnPlace;
  // The lengths are not known here: a sequence is taken to fill half of its last
  // place, and to see its share of the keys, less those that its own queries add
  // one by one.
  const long long likely =
      std::max(1ll, p.sequences == 1 ? (p.tokens + 2ll * s.span - 1) / (2 * s.span)
                                     : s.places - p.sequences / 2) * columns;
  const long long waves = likely / sm_count;
  const long long cut = likely - waves * sm_count;
  const long long parts = cut > 0 ? sm_count / cut : 1;
  long long seen = (long long)p.keys / p.sequences;
  if (p.causal && waves > 0) seen -= p.tokens / p.sequences;
  if (waves < kSplitWaves && s.places <= kSplitPlaces && sm_count < kSplitRest && parts > 1 &&
      seen - seen / parts >= kSplitKeys)
    s.mode = kSplit;
  s.works = (int)std::min<long long>(s.places + sm_count / columns + 2, 1 << 20);
  s.states = (int)(sm_count / columns + 2);
  s.joins = (int)std::min<long long>(s.places, s.states / 2);
  return s;
}

// Whether a row can be so long that its output is put aside.
bool has_aside(const PackedAttention& p) {
  return p.keys > kAsideKeys;
}
// Bytes of the flags of places, to a multiple of 16, and of the places.
size_t taken_bytes(int sm_count) { return ((size_t)sm_count * sizeof(uint32_t) + 15) / 16 * 16; }
size_t aside_bytes(int sm_count, int hd) {
  return (size_t)sm_count * 2 * kTile * (hd + 4) * sizeof(float);
}

// Bytes of the plan, to a multiple of 16.
size_t plan_bytes(const Shape& s) {
  if (s.mode == kOwnPlace) return 0;
  if (s.mode == kSplit)
    return sizeof(Plan) + (size_t)s.works * sizeof(Work) + (size_t)s.joins * sizeof(Join);
  return sizeof(Plan) + (size_t)s.places * sizeof(Work);
}

// Bytes of the states of parts.
size_t parts_bytes(const Shape& s, int columns, int hd) {
  return s.mode == kSplit ? (size_t)s.states * columns * part_floats(hd) * sizeof(float) : 0;
}

template <int HD, bool kLong>
auto kernel_of(Mode mode) {
  return mode == kSplit     ? packed_kernel<HD, kSplit, kLong>
         : mode == kPlanned ? packed_kernel<HD, kPlanned, kLong>
                            : packed_kernel<HD, kOwnPlace, kLong>;
}

template <int HD>
void launch_packed(const Launch& l, PackedArgs a, const Shape& s, bool aside, void* workspace) {
  using C = Packed<HD>;
  a.head_tiles = s.head_tiles;
  a.heads = s.heads;
  a.span = s.span;
  CUtensorMap mq, mk, mv;
  const uint64_t dq[4] = {(uint64_t)HD, (uint64_t)a.group, (uint64_t)a.kvh, (uint64_t)a.tokens};
  const uint32_t bq[4] = {64, (uint32_t)a.heads, 1, (uint32_t)a.span};
  const uint64_t dk[3] = {(uint64_t)HD, (uint64_t)a.kvh, (uint64_t)std::max(1, a.keys)};
  const uint32_t bk[3] = {64, 1, (uint32_t)C::kKeys};
  if (!make_f16_map(&mq, a.q, 4, dq, bq) || !make_f16_map(&mk, a.k, 3, dk, bk) ||
      !make_f16_map(&mv, a.v, 3, dk, bk))
    fail(MI_ERR_KERNEL, "packed attention: tensor map encoding failed");
  auto kernel = aside ? kernel_of<HD, true>(s.mode) : kernel_of<HD, false>(s.mode);
  allow_dynamic_smem(kernel, C::kBytes);
  const int columns = a.kvh * a.head_tiles;
  const long long grid = (s.mode == kSplit ? s.works : s.places) * (long long)columns;
  if (grid > 0x7FFFFFFF)
    fail(MI_ERR_SHAPE, "invalid tensor shape: %d tokens of %d sequences are too many for one call",
         a.tokens, a.sequences);
  Plan* plan = static_cast<Plan*>(workspace);
  a.plan = plan;
  if (aside) {
    char* at = static_cast<char*>(workspace) + plan_bytes(s) + parts_bytes(s, columns, HD);
    a.taken = reinterpret_cast<uint32_t*>(at);
    a.aside = reinterpret_cast<float4*>(at + taken_bytes(l.sm_count));
    a.places = l.sm_count;
    if (s.mode == kOwnPlace)  // no plan that clears them
      MI_CUDA(cudaMemsetAsync(a.taken, 0, taken_bytes(l.sm_count), l.stream));
  }
  if (s.mode == kPlanned)
    launch_kernel(l, dim3(1), dim3(kPlanThreads), 0, packed_plan_kernel, a, plan, (int)s.places,
                  C::kKeys);
  if (s.mode == kSplit) {
    a.parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + plan_bytes(s));
    launch_kernel(l, dim3(1), dim3(kPlanThreads), 0, packed_split_kernel, a, plan, (int)s.places,
                  s.works, C::kKeys, columns, l.sm_count);
  }
  launch_kernel(l, dim3((unsigned)grid), dim3(kThreads), C::kBytes, kernel, mq, mk, mv, a);
  if (s.mode == kSplit)
    launch_kernel(l, dim3((unsigned)s.joins * columns, 2 * kTile / 8), dim3(256), 0,
                  packed_join_kernel<HD>, a, s.works);
}

}  // namespace

size_t packed_attention_workspace(const PackedAttention& p, int sm_count) {
  const Shape s = shape_of(p, sm_count);
  size_t bytes = plan_bytes(s) + parts_bytes(s, p.kvh * s.head_tiles, p.hd);
  if (has_aside(p)) bytes += taken_bytes(sm_count) + aside_bytes(sm_count, p.hd);
  return bytes;
}

void packed_attention(const Launch& l, const PackedAttention& p, void* workspace) {
  if (p.tokens == 0 || p.sequences == 0) return;
  PackedArgs a{};
  a.q = p.q;
  a.k = p.k;
  a.v = p.v;
  a.out = p.out;
  a.query_starts = p.query_starts;
  a.key_starts = p.key_starts;
  a.fault = p.fault;
  a.tokens = p.tokens;
  a.keys = p.keys;
  a.sequences = p.sequences;
  a.qh = p.qh;
  a.kvh = p.kvh;
  a.causal = p.causal;
  a.group = p.qh / p.kvh;
  a.scale_log2 = (float)(1.4426950408889634 / sqrt((double)p.hd));
  const Shape s = shape_of(p, l.sm_count);
  if (p.hd == 128)
    launch_packed<128>(l, a, s, has_aside(p), workspace);
  else
    launch_packed<64>(l, a, s, has_aside(p), workspace);
}

}  // namespace k
}  // namespace mi
