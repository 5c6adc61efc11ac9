// Attention over packed prompts: sequences of different lengths laid end to
// end, grouped heads, causal from the ends (a prefix of keys computed before
// is allowed) or not.
//
//   o = sum_j softmax_j(q . k_j / sqrt(d)) v_j
//
// Tensor-bound: 4 d operations per visible (query, key) pair and head on the
// tcgen05 pipe, with the exponentials (16 per clock and SM) close behind at
// head_dim 128 and ahead of it at 64.
//
// A CTA takes two row tiles of one sequence and KV head. The rows of a tile
// are the query heads of the group for up to 128 / group tokens, so a short
// prompt still fills a tile and a key tile is read once for the whole group.
// Roles:
//   warps 0-3, 4-7  softmax of row tile 0 / 1, one row to a thread: scores from
//                   TMEM, the running maximum and sum in registers, FP16
//                   weights back to TMEM over the scores; in the end the output
//   warp 8          one thread issues tcgen05.mma: S_t = Q_t K^T from shared
//                   memory, O_t += P_t V with P from TMEM. The tiles alternate,
//                   so one tile's products run while the other's softmax does
//   warp 9          TMA: the query tiles once, then K and V tiles of 128 keys
//                   through one ring
// TMEM: S_0, S_1 (128 columns each, P over them), O_0, O_1.
//
// O is rescaled only when a row's maximum has grown by more than 2^8 since the
// last time (weights then stay below 2^8, far inside FP16, and the final
// division by the sum of the same weights takes the factor out); s_full of
// step i says that the product of step i - 1 is done, as its commit covers all
// earlier products, so the row's own thread may rescale O in TMEM.

#include <cuda.h>

#include "device.cuh"
#include "pipeline.cuh"

namespace mi {
namespace k {

namespace {

constexpr int kTile = 128;     // rows of a row tile, keys of a key tile
constexpr int kThreads = 320;
constexpr uint64_t kWaitNs = 200ull * 1000 * 1000;
constexpr float kGrowth = 8.f; // log2 of the weights' largest value

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
};

template <int HD>
struct PackedSmem {
  static constexpr int kTileBytes = kTile * HD * 2;
  static constexpr int kSlots = HD == 128 ? 5 : 10;  // K and V tiles of the ring
  static constexpr int kBytes = 1024 /*align*/ + (2 + kSlots) * kTileBytes + 512;
};

// One row by one warp, from the formula, over the first `visible` keys and
// reading no others: rows whose products met infinities or NaN that they do
// not see (0 * NaN in a tile's masked places) are computed again this way.
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
    const int n = min(32, visible - j0);
    for (int i = 0; i < n; ++i) {
      const float w = __shfl_sync(0xffffffffu, p, i);
      const __half* vr = v + (size_t)(j0 + i) * stride + lane * kV;
#pragma unroll
      for (int e = 0; e < kV; ++e) acc[e] += w * __half2float(vr[e]);
    }
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
__device__ __forceinline__ void arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(pipe::smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
          pipe::smem_u32(bar))
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
// Shared-memory matrix descriptor of a 128-byte-swizzled operand (version 1):
// K-major (Q, K: rows of 64 values of the product's depth), 8-row groups 1024
// bytes apart; MN-major (V: rows are keys, the depth; 64 values of N to a row),
// the next 64 values of N `lead` bytes on, the next 8 keys 1024 bytes on.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr, uint32_t lead) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(lead >> 4) << 16) |
         ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// Instruction descriptor of kind::f16: F16 operands, F32 result, M = 128.
__host__ __device__ constexpr uint32_t idesc_f16(int n, bool b_mn_major) {
  return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t (&r)[32], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,"
      "%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,"
      "%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(
          addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
      "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
      "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
      "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// What a CTA works on.
struct Work {
  int q0, q1;      // the sequence's query rows
  int k0, keys;    // its first key row, its keys
  int token;       // first token (of the sequence) of row tile 0
  int blocks[2];   // key tiles that row tile 0 / 1 sees
};

template <int HD>
__global__ void __launch_bounds__(kThreads, 1)
    packed_kernel(const __grid_constant__ CUtensorMap map_q,
                  const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const PackedArgs a) {
  using S = PackedSmem<HD>;
  constexpr int kSlots = S::kSlots;
  constexpr uint32_t kTileBytes = S::kTileBytes;
  constexpr int kHalves = HD / 64;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* ring = smem + 2 * kTileBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + kSlots * kTileBytes);
  uint64_t* q_full = bars;            // [1]
  uint64_t* s_full = bars + 1;        // [2] scores are in TMEM
  uint64_t* p_full = bars + 3;        // [2] weights are in TMEM
  uint64_t* o_full = bars + 5;        // [2] the last product is done
  uint64_t* kv_full = bars + 7;       // [kSlots]
  uint64_t* kv_empty = kv_full + kSlots;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(kv_empty + kSlots);
  Work* work = reinterpret_cast<Work*>(tmem_slot + 2);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kv = blockIdx.x / a.head_tiles;
  const int head0 = (blockIdx.x % a.head_tiles) * a.heads;  // first head of the group in the tile

  pdl_trigger();
  pdl_wait();

  // ---- which tokens ------------------------------------------------------------
  // Sequence s owns the places floor(start_s / (2 span)) + s and on, which
  // leaves it room for its tiles whatever the lengths are; a place's sequence
  // is the last one that begins at or before it. Late places first: with a
  // causal mask they are the longest.
  const int place = (int)gridDim.y - 1 - (int)blockIdx.y;
  const int pair = 2 * a.span;
  bool bad = false;
  int begun = 0;
  for (int s = tid; s < a.sequences; s += kThreads) {
    const uint32_t qb = a.query_starts[s], qe = a.query_starts[s + 1];
    const uint32_t kb = a.key_starts[s], ke = a.key_starts[s + 1];
    bad |= qb > qe || qe > (uint32_t)a.tokens || kb > ke || ke > (uint32_t)a.keys;
    begun += (unsigned long long)qb / pair + s <= (unsigned long long)place;
  }
  if (tid == 0) tmem_slot[1] = 0;
  if (__syncthreads_or(bad)) {
    if (tid == 0) report_fault(a.fault, kFaultStarts);
    return;
  }
  begun = __reduce_add_sync(0xffffffffu, begun);
  if (lane == 0 && begun) atomicAdd(tmem_slot + 1, (uint32_t)begun);
  __syncthreads();
  if (tid == 0) {
    const int s = (int)tmem_slot[1] - 1;
    Work w{0, 0, 0, 0, 0, {0, 0}};
    if (s >= 0) {
      w.q0 = (int)a.query_starts[s];
      w.q1 = (int)a.query_starts[s + 1];
      w.k0 = (int)a.key_starts[s];
      w.keys = (int)a.key_starts[s + 1] - w.k0;
      const long long t = (long long)(place - (w.q0 / pair + s)) * pair;
      w.token = t < w.q1 - w.q0 ? (int)t : -1;
      for (int i = 0; i < 2 && w.token >= 0; ++i) {
        const int n = w.q1 - w.q0;
        const int last = min(n, w.token + (i + 1) * a.span) - 1;  // last token of the row tile
        if (last < w.token + i * a.span) continue;
        const long long seen = a.causal ? (long long)w.keys - (n - 1 - last) : w.keys;
        w.blocks[i] = seen > 0 ? (int)((seen + kTile - 1) / kTile) : 0;
      }
    } else {
      w.token = -1;
    }
    *work = w;
    pipe::mbar_init(q_full, 1);
    for (int i = 0; i < 2; ++i) {
      pipe::mbar_init(s_full + i, 1);
      pipe::mbar_init(p_full + i, 4);
      pipe::mbar_init(o_full + i, 1);
    }
    for (int i = 0; i < kSlots; ++i) {
      pipe::mbar_init(kv_full + i, 1);
      pipe::mbar_init(kv_empty + i, 1);
    }
    pipe::fence_mbar_init();
  }
  __syncthreads();
  const Work w = *work;
  if (w.token < 0) return;  // a place without tokens
  const int blocks = max(w.blocks[0], w.blocks[1]);
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     pipe::smem_u32(tmem_slot)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tmem_o = tmem + 2 * kTile;

  if (warp == 9) {
    if (lane == 0 && blocks > 0) {
      // ---- TMA ------------------------------------------------------------------
      pipe::mbar_expect_tx(q_full, 2u * kHalves * a.heads * a.span * 128u);
      for (int t = 0; t < 2; ++t)
        for (int h = 0; h < kHalves; ++h)
          tma_4d(smem + t * kTileBytes + h * (kTile * 128), &map_q, q_full, h * 64, head0, kv,
                 w.q0 + w.token + t * a.span);
      bool ok = true;
      int n = 0;
      for (; n < 2 * blocks && ok; ++n) {
        const int slot = n % kSlots;
        ok = wait_for(kv_empty + slot, ((n / kSlots) & 1) ^ 1, a.fault);
        if (!ok) break;
        pipe::mbar_expect_tx(kv_full + slot, kTileBytes);
        for (int h = 0; h < kHalves; ++h)
          tma_3d(ring + slot * kTileBytes + h * (kTile * 128), n & 1 ? &map_v : &map_k,
                 kv_full + slot, h * 64, kv, w.k0 + (n >> 1) * kTile);
      }
      // the copies land before the CTA leaves
      wait_for(q_full, 0, a.fault);
      for (int i = max(0, n - kSlots); i < n; ++i)
        wait_for(kv_full + i % kSlots, (i / kSlots) & 1, a.fault);
    }
  } else if (warp == 8) {
    if (lane == 0 && blocks > 0) {
      // ---- products -----------------------------------------------------------------
      constexpr uint32_t idesc_s = idesc_f16(kTile, false);
      constexpr uint32_t idesc_o = idesc_f16(HD, true);
      auto scores = [&](int t, int slot) {
        const uint32_t qa = pipe::smem_u32(smem + t * kTileBytes);
        const uint32_t ka = pipe::smem_u32(ring + slot * kTileBytes);
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          const uint32_t off = (kk / 4) * (kTile * 128) + (kk % 4) * 32;
          mma_ss(tmem + t * kTile, desc_sw128(qa + off, 16), desc_sw128(ka + off, 16), idesc_s,
                 kk != 0);
        }
      };
      bool ok = wait_for(q_full, 0, a.fault) && wait_for(kv_full, 0, a.fault);
      if (ok) {
        fence_after();
        for (int t = 0; t < 2; ++t)
          if (w.blocks[t] > 0) {
            scores(t, 0);
            commit(s_full + t);
          }
        commit(kv_empty);
      }
      for (int i = 0; i < blocks && ok; ++i) {
        const int nv = 2 * i + 1, nk = 2 * i + 2;
        const int sv = nv % kSlots, sk = nk % kSlots;
        ok = wait_for(kv_full + sv, (nv / kSlots) & 1, a.fault);
        for (int t = 0; t < 2 && ok; ++t) {
          if (i < w.blocks[t]) {
            ok = wait_for(p_full + t, i & 1, a.fault);
            if (!ok) break;
            fence_after();
            const uint32_t va = pipe::smem_u32(ring + sv * kTileBytes);
#pragma unroll
            for (int kk = 0; kk < kTile / 16; ++kk)
              mma_ts(tmem_o + t * HD, tmem + t * kTile + kk * 8,
                     desc_sw128(va + kk * 2048, kTile * 128), idesc_o, (i | kk) != 0);
            if (i + 1 == w.blocks[t]) commit(o_full + t);
          }
          if (t == 1) commit(kv_empty + sv);
          if (i + 1 < w.blocks[t]) {
            ok = wait_for(kv_full + sk, (nk / kSlots) & 1, a.fault);
            if (!ok) break;
            fence_after();
            scores(t, sk);
            commit(s_full + t);
          }
        }
        if (ok && i + 1 < blocks) commit(kv_empty + sk);
      }
    }
  } else {
    // ---- softmax -------------------------------------------------------------------
    const int t = warp >> 2;                // row tile
    const int row = (warp & 3) * 32 + lane; // of the tile: the TMEM lane
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + t * kTile;
    const uint32_t to = tmem_o + lanes + t * HD;
    const int n = w.q1 - w.q0;
    const int token = w.token + t * a.span + row / a.heads;
    const int head = head0 + row % a.heads;
    const bool valid = row < a.heads * a.span && token < n && head < a.group;
    long long seen = a.causal ? (long long)w.keys - (n - 1 - token) : w.keys;
    const int visible = valid && seen > 0 ? (int)seen : 0;
    // keys that every row of the tile sees
    const long long least =
        a.causal ? (long long)w.keys - (n - 1 - (w.token + t * a.span)) : w.keys;
    const int mine = w.blocks[t];
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int i = 0; i < mine; ++i) {
      ok = wait_for(s_full + t, i & 1, a.fault);
      if (!ok) break;
      fence_after();
      uint32_t s[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(s[c], ts + c * 32);
      tmem_wait_ld();
      const int k0 = i * kTile;
      if (k0 + kTile > least) {
        const int left = visible - k0;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (c * 32 + e >= left) s[c][e] = 0xff800000u;  // -inf
      }
      float top = -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int e = 0; e < 32; ++e) top = fmaxf(top, __uint_as_float(s[c][e]));
      top *= a.scale_log2;
      // a maximum that grew past the bound moves the row's base
      const bool grown = top > m + kGrowth || (m == -INFINITY && top > m);
      if (__any_sync(0xffffffffu, grown)) {
        const float next = grown ? top : m;
        const float f = m == -INFINITY ? 0.f : exp2_fast(m - next);
        const float factor = grown ? f : 1.f;
        m = next;
        if (i > 0) {
          l *= factor;
#pragma unroll 1
          for (int c = 0; c < HD; c += 32) {
            uint32_t o[32];
            tmem_ld32(o, to + c);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e)
              o[e] = __float_as_uint(__uint_as_float(o[e]) * factor);
            tmem_st32(to + c, o);
          }
          tmem_wait_st();
        }
      }
      const float base = m == -INFINITY ? 0.f : -m;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t p[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          // weights rounded to FP16 for the product; the sum takes the rounded
          // ones, so that it is the sum of what the product weighs
          const float x0 = __uint_as_float(s[2 * c + (e >> 4)][2 * (e & 15)]);
          const float x1 = __uint_as_float(s[2 * c + (e >> 4)][2 * (e & 15) + 1]);
          const __half2 h = __floats2half2_rn(exp2_fast(fmaf(x0, a.scale_log2, base)),
                                              exp2_fast(fmaf(x1, a.scale_log2, base)));
          const uint32_t u = *reinterpret_cast<const uint32_t*>(&h);
          l = fma_f16_f32((unsigned short)(u & 0xffffu), 0x3c00, l);
          l = fma_f16_f32((unsigned short)(u >> 16), 0x3c00, l);
          p[e] = u;
        }
        tmem_st32(ts + c * 32, p);
      }
      tmem_wait_st();
      fence_before();
      __syncwarp();
      if (lane == 0) arrive(p_full + t);
    }
    // ---- output ---------------------------------------------------------------------
    const size_t stride = (size_t)a.kvh * HD;
    const size_t at = ((size_t)(w.q0 + token) * a.qh + (size_t)kv * a.group + head) * HD;
    if (mine > 0 && ok && wait_for(o_full + t, 0, a.fault)) {
      fence_after();
      const float inv = 1.f / l;
      bool odd = false;  // something that is not finite
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        uint32_t o[32];
        tmem_ld32(o, to + c);
        tmem_wait_ld();
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint4 v;
          __half2* hv = reinterpret_cast<__half2*>(&v);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = __uint_as_float(o[q * 8 + 2 * e]) * inv;
            const float y = __uint_as_float(o[q * 8 + 2 * e + 1]) * inv;
            odd |= !(fabsf(x) <= 65504.f) || !(fabsf(y) <= 65504.f);
            hv[e] = __floats2half2_rn(x, y);
          }
          if (visible == 0) v = make_uint4(0, 0, 0, 0);
          if (valid) reinterpret_cast<uint4*>(a.out + at + c)[q] = v;
        }
      }
      unsigned again = __ballot_sync(0xffffffffu, odd && visible > 0);
      while (again) {
        const int who = __ffs(again) - 1;
        again &= again - 1;
        const int seen_w = __shfl_sync(0xffffffffu, visible, who);
        const unsigned long long at_w = __shfl_sync(0xffffffffu, (unsigned long long)at, who);
        attention_row<HD>(a.q + at_w, a.k + (size_t)w.k0 * stride + kv * HD,
                          a.v + (size_t)w.k0 * stride + kv * HD, stride, seen_w, a.scale_log2,
                          a.out + at_w);
      }
    } else if (mine == 0 && valid) {
      for (int c = 0; c < HD / 8; ++c)
        reinterpret_cast<uint4*>(a.out + at)[c] = make_uint4(0, 0, 0, 0);
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 8) {
    __syncwarp();
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512)
                 : "memory");
  }
}

template <int HD>
void launch_packed(const Launch& l, PackedArgs a) {
  using S = PackedSmem<HD>;
  a.head_tiles = (a.group + kTile - 1) / kTile;
  a.heads = (a.group + a.head_tiles - 1) / a.head_tiles;
  a.span = kTile / a.heads;
  CUtensorMap mq, mk, mv;
  const uint64_t dq[4] = {(uint64_t)HD, (uint64_t)a.group, (uint64_t)a.kvh, (uint64_t)a.tokens};
  const uint32_t bq[4] = {64, (uint32_t)a.heads, 1, (uint32_t)a.span};
  const uint64_t dk[3] = {(uint64_t)HD, (uint64_t)a.kvh, (uint64_t)std::max(1, a.keys)};
  const uint32_t bk[3] = {64, 1, (uint32_t)kTile};
  if (!make_f16_map(&mq, a.q, 4, dq, bq) || !make_f16_map(&mk, a.k, 3, dk, bk) ||
      !make_f16_map(&mv, a.v, 3, dk, bk))
    fail(MI_ERR_KERNEL, "packed attention: tensor map encoding failed");
  auto kernel = packed_kernel<HD>;
  allow_dynamic_smem(kernel, S::kBytes);
  // a place for every pair of row tiles, whatever the lengths are
  const long long places = (long long)a.tokens / (2 * a.span) + a.sequences;
  if (places > 65535)
    fail(MI_ERR_SHAPE, "invalid tensor shape: %d tokens of %d sequences are too many for one call",
         a.tokens, a.sequences);
  launch_kernel(l, dim3(a.kvh * a.head_tiles, (unsigned)places), dim3(kThreads), S::kBytes, kernel,
                mq, mk, mv, a);
}

}  // namespace

void packed_attention(const Launch& l, const PackedAttention& p) {
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
  if (p.hd == 128)
    launch_packed<128>(l, a);
  else
    launch_packed<64>(l, a);
}

}  // namespace k
}  // namespace mi
