// Paged caches of a ragged batch: the append of rotated keys and values, and
// attention of one new token per sequence over its pages.
//
// A cache is [pages, page_size, kv_heads, head_dim] FP16; position p of
// sequence s lies in page table[s][p / page_size] at row p % page_size, so a
// contiguous [capacity, kv_heads, head_dim] cache reshaped into pages is one
// too. Page ids, lengths and starts live on the device (a captured graph
// serves every step); the kernels check each against its tensor, leave out
// what lies outside and say so in the context's fault word.

#include "device.cuh"
#include "pipeline.cuh"

namespace mi {
namespace k {

namespace {

// ---- append -------------------------------------------------------------------
// y = half(rot(x * rsqrt(mean(x^2) + eps) * w)) for Q and K heads (the norm is
// left out without weights), V as it is; each head row is read and written
// once. The arithmetic is that of qk_norm_rope_cache and rope (numerics.cuh),
// so a paged cache holds the same bits as a contiguous one.
//
// HBM-bound for prompts. A row has HD / 16 lanes, each with a chunk of eight
// values and the chunk that it rotates with: the first step of the canonical
// sum of squares and the whole rotation stay inside a lane (with a chunk to a
// lane and the partner fetched by shuffles, 5.7 K tokens of 32/8 heads took 55
// us, 32 so). A block takes kTok tokens at a time and first fills a table of
// their cosines and sines: the angles need double precision (numerics.cuh),
// which a thread per (token, pair) pays once for all heads, and a thread per
// pair the frequency's pow once for all of a block's tokens.
constexpr int kAppendThreads = 256;

struct AppendArgs {
  const __half *q, *k, *v, *qw, *kw;
  __half *q_out, *kc, *vc;
  const uint32_t *starts, *lengths, *table;
  uint32_t* fault;
  int tokens, sequences, qh, kvh, table_width, page;
  uint32_t pages;
  float theta, eps;
  float inverse_heads;  // 1 / (qh + 2 kvh), rows to a token
};

// Two FP32 values in one instruction, each rounded as by itself.
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ void split(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ void widen8(const uint4& raw, uint64_t (&x)[4]) {
  const __half2* h = reinterpret_cast<const __half2*>(&raw);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 f = __half22float2(h[e]);
    x[e] = pair_of(f.x, f.y);
  }
}
__device__ __forceinline__ uint4 narrow8(const uint64_t (&x)[4]) {
  uint4 packed;
  __half2* h = reinterpret_cast<__half2*>(&packed);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float lo, hi;
    split(x[e], lo, hi);
    h[e] = __floats2half2_rn(lo, hi);
  }
  return packed;
}

template <int HD, int kTok>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const AppendArgs a) {
  constexpr int kLanes = HD / 16;          // lanes of a head row
  constexpr int kRows = kAppendThreads / kLanes;
  constexpr int kPairs = HD / 2;
  __shared__ __align__(16) float cosines[kTok][kPairs], sines[kTok][kPairs];
  __shared__ float frequencies[kPairs];
  __shared__ uint32_t position[kTok];
  __shared__ uint32_t slot[kTok];          // cache row of the token
  const int tid = threadIdx.x;
  const int li = tid % kLanes;
  const int pair0 = tid % kPairs;
  if (tid < kPairs)
    frequencies[tid] = (float)pow((double)a.theta, (double)__fdiv_rn(-(float)(tid * 2), (float)HD));
  pdl_trigger();
  pdl_wait();

  for (int t0 = blockIdx.x * kTok; t0 < a.tokens; t0 += gridDim.x * kTok) {
    // The sequence of a token is the number of sequences that end at or
    // before it: one pass over the starts by the whole block.
    int before[kTok];
#pragma unroll
    for (int i = 0; i < kTok; ++i) before[i] = 0;
    bool bad = false;
    for (int s = tid; s < a.sequences; s += kAppendThreads) {
      const uint32_t b = a.starts[s], e = a.starts[s + 1];
      bad |= b > e || e > (uint32_t)a.tokens;
#pragma unroll
      for (int i = 0; i < kTok; ++i) before[i] += e <= (uint32_t)(t0 + i);
    }
    if (tid < kTok) slot[tid] = 0;
    bad = __syncthreads_or(bad);
    if (bad) {  // starts that do not rise or leave the tokens: nothing is done
      if (tid == 0) report_fault(a.fault, kFaultStarts);
      return;
    }
#pragma unroll
    for (int i = 0; i < kTok; ++i) {
      const int w = __reduce_add_sync(0xffffffffu, before[i]);
      if ((tid & 31) == 0 && w) atomicAdd(&slot[i], (uint32_t)w);
    }
    __syncthreads();
    if (tid < kTok) {
      const int t = t0 + tid;
      const uint32_t s = slot[tid];
      uint32_t row = 0xFFFFFFFFu, pos = 0;
      // a token before the first start or behind the last sequence is left out
      if (t < a.tokens && s < (uint32_t)a.sequences && a.starts[s] <= (uint32_t)t) {
        const uint32_t left = a.starts[s + 1] - t, len = a.lengths[s];
        const uint32_t n = a.starts[s + 1] - a.starts[s];
        if (len < n || (uint64_t)len > (uint64_t)a.table_width * a.page) {
          report_fault(a.fault, kFaultLength);
        } else {
          pos = len - left;
          const uint32_t pg = a.table[(size_t)s * a.table_width + pos / a.page];
          if (pg < a.pages)
            row = pg * a.page + pos % a.page;
          else
            report_fault(a.fault, kFaultPage);
        }
      }
      position[tid] = pos;
      slot[tid] = row;
    }
    __syncthreads();
    const int heads = a.qh + 2 * a.kvh;
    const int rows = min(kTok, a.tokens - t0) * heads;
    // the chunks of row r of the block's tokens, and where they go
    auto source = [&](int r, const __half*& src, __half*& dst, int& i, int& h) {
      i = kTok == 1 ? 0 : (int)(((float)r + 0.5f) * a.inverse_heads);
      h = r - i * heads;
      const size_t t = t0 + i;
      const uint32_t row = slot[i];
      src = nullptr;
      dst = nullptr;
      if (row == 0xFFFFFFFFu) return;
      if (h < a.qh) {
        src = a.q + (t * a.qh + h) * HD;
        dst = a.q_out + (t * a.qh + h) * HD;
      } else {
        const bool is_v = h >= a.qh + a.kvh;
        const int kv = h - a.qh - (is_v ? a.kvh : 0);
        src = (is_v ? a.v : a.k) + (t * a.kvh + kv) * HD;
        dst = (is_v ? a.vc : a.kc) + ((size_t)row * a.kvh + kv) * HD;
      }
    };
    // the first row's loads are in flight while the angles are computed
    const __half* src = nullptr;
    __half* dst = nullptr;
    int i = 0, h = 0;
    uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
    int r = tid / kLanes;
    auto fetch = [&] {
      if (r < rows) source(r, src, dst, i, h);
      if (r < rows && src) {
        lo = reinterpret_cast<const uint4*>(src)[li];
        hi = reinterpret_cast<const uint4*>(src)[li + kLanes];
      }
    };
    fetch();
    for (int j = tid; j < kTok * kPairs; j += kAppendThreads) {
      const int t = j / kPairs;
      if (slot[t] != 0xFFFFFFFFu) {
        double s, c;
        sincos((double)__fmul_rn((float)position[t], frequencies[pair0]), &s, &c);
        cosines[t][pair0] = (float)c;
        sines[t][pair0] = (float)s;
      }
    }
    __syncthreads();
    while (r - (tid & 31) / kLanes < rows) {  // whole warps
      // this row's, while the next one's are on their way
      const bool ok = r < rows && src;
      const bool rotates = h < a.qh + a.kvh;
      const __half* w = h < a.qh ? a.qw : a.kw;
      __half* const to = dst;
      const int token = i;
      uint4 first = lo, second = hi;
      r += kRows;
      fetch();
      if (!__any_sync(0xffffffffu, ok && rotates)) {  // values
        if (ok) {
          reinterpret_cast<uint4*>(to)[li] = first;
          reinterpret_cast<uint4*>(to)[li + kLanes] = second;
        }
        continue;
      }
      uint64_t x[4], y[4];
      widen8(first, x);
      widen8(second, y);
      if (a.kw) {  // all of the call's rows have weights, or none
        float total = __fadd_rn(chunk_sq(first, 0.f), chunk_sq(second, 0.f));
#pragma unroll
        for (int o = kLanes / 2; o >= 1; o >>= 1)
          total = __fadd_rn(total, __shfl_xor_sync(0xffffffffu, total, o));
        const float one = rms_scale(total, HD, a.eps);
        const uint64_t scale = pair_of(one, one);
        uint64_t g[4];
        widen8(reinterpret_cast<const uint4*>(w)[li], g);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = mul2(mul2(x[e], scale), g[e]);
        widen8(reinterpret_cast<const uint4*>(w)[li + kLanes], g);
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = mul2(mul2(y[e], scale), g[e]);
      }
      if (ok) {
        if (rotates) {
          uint64_t u[4], v[4];
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const float4 c = *reinterpret_cast<const float4*>(&cosines[token][8 * li + 4 * q]);
            const float4 s = *reinterpret_cast<const float4*>(&sines[token][8 * li + 4 * q]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              // The sums are scalar: a paired addition behind a paired product
              // is fused with it, and the product's rounding is lost.
              const uint64_t ce = e ? pair_of(c.z, c.w) : pair_of(c.x, c.y);
              const uint64_t se = e ? pair_of(s.z, s.w) : pair_of(s.x, s.y);
              const int k = 2 * q + e;
              float xc[2], xs[2], yc[2], ys[2];
              split(mul2(x[k], ce), xc[0], xc[1]);
              split(mul2(x[k], se), xs[0], xs[1]);
              split(mul2(y[k], ce), yc[0], yc[1]);
              split(mul2(y[k], se), ys[0], ys[1]);
              u[k] = pair_of(__fsub_rn(xc[0], ys[0]), __fsub_rn(xc[1], ys[1]));
              v[k] = pair_of(__fadd_rn(xs[0], yc[0]), __fadd_rn(xs[1], yc[1]));
            }
          }
          first = narrow8(u);
          second = narrow8(v);
        }
        reinterpret_cast<uint4*>(to)[li] = first;
        reinterpret_cast<uint4*>(to)[li + kLanes] = second;
      }
    }
    __syncthreads();
  }
}

template <int HD>
void launch_append(const Launch& l, const AppendArgs& a) {
  // Four tokens to a block share its barriers (one 42 us, two 33.9, four 32.7
  // for 5.7 K tokens, before the pow was shared); few tokens take a block each, since latency is then all
  // there is.
  if (a.tokens <= 2 * l.sm_count) {
    launch_kernel(l, dim3(a.tokens), dim3(kAppendThreads), 0, paged_append_kernel<HD, 1>, a);
  } else {
    const int grid = std::min((a.tokens + 3) / 4, 8 * l.sm_count);
    launch_kernel(l, dim3(grid), dim3(kAppendThreads), 0, paged_append_kernel<HD, 4>, a);
  }
}

// ---- attention of one token -----------------------------------------------------
// o = sum_j softmax_j(q . k_j / sqrt(d)) v_j over the positions of each
// sequence. HBM-bound: every key and value is read once for all query heads
// of its group.
//
// The products are m16n8k16 with keys (then dims) as rows and the group's
// heads as the 8 or 16 columns: S^T = K Q^T, O^T += V^T P^T. Heads as the 16
// rows would leave half or more of every product and twice the registers to
// padding at the usual 1 to 8 heads a group; P^T's operand layout is S^T's
// result layout transposed (movmatrix).
//
// The work is cut evenly whatever the lengths are: all (sequence, KV head,
// head tile) units are laid end to end, each its tiles of 64 or 128 keys and
// kUnitCost empty places for what its end costs, and CTA c of C takes the places
// [c N / C, (c + 1) N / C). (Without them the CTAs that met the many units of
// short sequences set the time: 64 sequences of 1 to 8192 took 78 us, 57 with
// them.) A unit that lies inside a CTA is
// finished there; one that crosses CTAs leaves unnormalised pieces that a
// second kernel joins in order of position, so results do not depend on
// timing. A CTA has at most two pieces: one that continues a unit from the
// CTA before it (slot 0), one that a later CTA continues (slot 1).
//
// Each of a CTA's four warps owns a quarter of a tile, with its own ring of
// cp.async stages (rows past the length are filled with zeros, so stale
// values never enter a product) and its own running maximum and sum; the
// warps meet only at a unit's end, where each leaves its state in the ring
// stage that it has just used up. Two CTAs to an SM keep about 130 KB of
// loads in flight.
//
// Weights are taken over a warp's maximum less 7 binary places, so that they lie
// below 2^8 and FP16 holds them to half a step of 2^-11 of themselves or 2^-32
// of the largest (over the maximum itself those of 2^-25 were 0). The tensor
// cores cut a product off at 2^-25 of the accumulator's power of two before they
// add it, so every kAsideSteps steps a warp puts its accumulators and sums aside,
// in FP32, and starts from 0. They go to device memory: a second set of registers
// cost 96/8 heads of 128 9%.
constexpr float kLift = 7.f;
constexpr int kAsideSteps = 128;
constexpr int kUnitCost = 1;
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kHeadsMax = 16;

struct PagedArgs {
  const __half *q, *kc, *vc;
  __half* out;
  const uint32_t *lengths, *table;
  float* pieces;    // [C][2][16 * HD + 32]
  float* aside;     // [C][kWarps][aside_floats][32]: accumulators, bases, sums
  uint4* meta;      // [C]: of the unit that slot 1 begins: sequence, unit, last CTA, flag
  uint32_t* fault;
  int sequences, qh, kvh, table_width, page;
  int group;        // query heads per KV head
  int head_tiles;   // head tiles of a group
  int heads;        // heads of a tile (the last may have fewer)
  int page_shift;   // log2 of the page size, -1 where it has none
  uint32_t pages;
  float scale_log2; // log2(e) / sqrt(HD)
};

template <int HD, int NT>
struct PagedShape {
  // k16 tiles of keys of a warp's step, keys of a CTA's tile. At head_dim 64 a
  // step of 32 keys has the bytes of 16 at 128 and pays the maximum's shuffles
  // and the loop once for them (256 sequences of 100 to 1500: 63 us with 16
  // keys and four CTAs to an SM, 58 so).
  static constexpr int kSteps = HD == 128 ? 1 : 2;
  static constexpr int kTileKeys = kWarps * kSteps * 16;
  static constexpr int kCtas = 2;  // to an SM
  static constexpr int kStages = 3;
  static constexpr int kStageBytes = 2 * kSteps * 16 * HD * 2;  // a warp's keys and values
  static constexpr int kBytes = kWarps * kStages * kStageBytes;
};
constexpr size_t piece_floats(int hd) { return kHeadsMax * hd + 2 * kHeadsMax; }
// Of a thread's accumulators, bases and sums of 8 nt heads.
constexpr int aside_floats(int hd, int nt) { return nt * (hd / 16 * 4 + 4); }

__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Weight of a state with maximum m under the common maximum `top`.
__device__ __forceinline__ float state_weight(float m, float top) {
  return m == -INFINITY ? 0.f : exp2_fast(m - top);
}

// Length of a sequence as the kernels use it: 0 where the table cannot hold it.
__device__ __forceinline__ uint32_t paged_length(const PagedArgs& a, int s) {
  const uint32_t n = a.lengths[s];
  return (uint64_t)n > (uint64_t)a.table_width * a.page ? 0u : n;
}

// Walks a CTA's tiles in order.
struct Cursor {
  unsigned long long place;  // of the tile
  int s, unit, tile;         // sequence, unit of the sequence, tile of the unit
  int tiles;                 // tiles of a unit of this sequence
  uint32_t len;
};
// Places of a unit of n keys.
template <int kTileKeys>
__device__ __forceinline__ uint32_t unit_places(uint32_t n) {
  return n ? (n + kTileKeys - 1) / kTileKeys + kUnitCost : 0;
}

// NT: 8-head column tiles. kRuns: the page size is a multiple of 16, so a
// 16 keys of a step lie in one page (one table entry and one address for them).
template <int HD, int NT, bool kRuns>
__global__ void __launch_bounds__(kThreads, PagedShape<HD, NT>::kCtas)
    paged_attention_kernel(const PagedArgs a) {
  using S = PagedShape<HD, NT>;
  constexpr int kStages = S::kStages, kSteps = S::kSteps, kTileKeys = S::kTileKeys;
  constexpr int kRowsStep = 16 * kSteps;  // keys of a warp's step
  constexpr int kK = HD / 16;      // k16 steps of a score, m16 tiles of an output column
  constexpr int kChunks = HD / 8;  // 16-byte chunks of a row
  // row of a state in the ring: padded against bank conflicts where it fits
  constexpr int kRow = NT == 1 ? HD + 4 : HD;
  static_assert(8 * NT * kRow * 4 <= S::kStageBytes, "a state fits a stage");
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float stats[kWarps][kHeadsMax][2];
  __shared__ float* states[kWarps];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int units = a.kvh * a.head_tiles;

  pdl_wait();

  // Where this CTA's places begin: places per sequence, summed by the block
  // (each thread a run of consecutive sequences).
  __shared__ unsigned long long scan[kWarps];
  __shared__ Cursor first;
  const int run = (a.sequences + kThreads - 1) / kThreads;
  unsigned long long mine = 0;
  for (int i = 0; i < run; ++i) {
    const int s = tid * run + i;
    if (s < a.sequences) {
      const uint32_t n = paged_length(a, s);
      mine += unit_places<kTileKeys>(n);
      if (n == 0 && s % gridDim.x == blockIdx.x && a.lengths[s] != 0)
        report_fault(a.fault, kFaultLength);
    }
  }
  unsigned long long all = 0;
  {
    unsigned long long v = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    if (lane == 31) scan[warp] = v;
    __syncthreads();
    unsigned long long base = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) base += scan[w];
      all += scan[w];
    }
    mine = base + v - mine;  // places before this thread's sequences
  }
  const unsigned long long total = all * units;
  // no more CTAs than places, so that every one between a unit's first and last
  // holds a piece of it
  const unsigned long long ctas = total < gridDim.x ? total : gridDim.x;
  const bool works = blockIdx.x < ctas;
  const unsigned long long begin = works ? blockIdx.x * total / ctas : 0;
  const unsigned long long end = works ? (blockIdx.x + 1) * total / ctas : 0;
  if (begin < end) {
    unsigned long long at = mine * units;
    for (int i = 0; i < run; ++i) {
      const int s = tid * run + i;
      if (s >= a.sequences) break;
      const uint32_t n = paged_length(a, s);
      const uint32_t places = unit_places<kTileKeys>(n);
      const unsigned long long next = at + (unsigned long long)places * units;
      if (at <= begin && begin < next) {
        const unsigned long long w = begin - at;
        first = Cursor{begin, s, (int)(w / places), (int)(w % places), (int)places - kUnitCost, n};
      }
      at = next;
    }
  }
  // Rows of sequences without keys are zero.
  for (int s = blockIdx.x; s < a.sequences; s += gridDim.x)
    if (paged_length(a, s) == 0)
      for (int i = tid; i < a.qh * HD / 8; i += kThreads)
        reinterpret_cast<uint4*>(a.out + (size_t)s * a.qh * HD)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  uint4 note = make_uint4(0, 0, 0, 0);

  auto advance = [&](Cursor& c) {
    ++c.place;
    if (++c.tile < c.tiles) return;
    c.place += c.tiles + kUnitCost - c.tile;  // the rest of the unit's places
    c.tile = 0;
    if (++c.unit < units) return;
    c.unit = 0;
    do {
      if (++c.s >= a.sequences) {
        c.place = end;
        return;
      }
      c.len = paged_length(a, c.s);
      c.tiles = (c.len + kTileKeys - 1) / kTileKeys;
    } while (c.tiles == 0);
  };

  const uint32_t ring = pipe::smem_u32(smem) + warp * kStages * S::kStageBytes;
  const uint32_t row_stride = a.kvh * HD;
  // Cache row of this warp's key `lane` of a tile (kRuns: of key 16 lane, the
  // first of a run); all ones where there is none.
  auto row_of = [&](const Cursor& c) -> uint32_t {
    const int key = kRuns ? (lane < kSteps ? lane * 16 : kRowsStep) : lane;
    const uint32_t p = (uint32_t)c.tile * kTileKeys + warp * kRowsStep + key;
    if (key >= kRowsStep || p >= c.len) return 0xFFFFFFFFu;
    const uint32_t pi = a.page_shift >= 0 ? p >> a.page_shift : p / (uint32_t)a.page;
    const uint32_t pg = a.table[(size_t)c.s * a.table_width + pi];
    if (pg >= a.pages) {
      report_fault(a.fault, kFaultPage);
      return 0xFFFFFFFFu;
    }
    return pg * a.page + (p - pi * a.page);
  };
  constexpr int kRowsPerPass = 32 / kChunks;
  const int chunk = lane % kChunks, row0 = lane / kChunks;
  auto issue = [&](const Cursor& c, uint32_t rows, int stage) {
    const uint32_t dst = ring + stage * S::kStageBytes + row0 * (HD * 2);
    const int kv = c.unit / a.head_tiles;
    const size_t head = (size_t)kv * HD + chunk * 8;
    if constexpr (kRuns) {
      const int last = (int)c.len - c.tile * kTileKeys - warp * kRowsStep - row0;
#pragma unroll
      for (int run = 0; run < kSteps; ++run) {
        const uint32_t first_row = __shfl_sync(0xffffffffu, rows, run);
        const bool none = first_row == 0xFFFFFFFFu;
        // rows past the length are not read
        const int left = none ? 0 : last - run * 16;
        const size_t off = none ? head : (size_t)(first_row + row0) * row_stride + head;
#pragma unroll
        for (int i = 0; i < 16 / kRowsPerPass; ++i) {
          const int r = i * kRowsPerPass;
          const uint32_t bytes = r < left ? 16 : 0;
          const size_t at = r < left ? off + (size_t)r * row_stride : head;
          const uint32_t d =
              dst + (run * 16 + r) * (HD * 2) + ((chunk ^ ((r + row0) & 7)) << 4);
          cp_async16_zfill(d, a.kc + at, bytes);
          cp_async16_zfill(d + kRowsStep * HD * 2, a.vc + at, bytes);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < kRowsStep / kRowsPerPass; ++i) {
        const int r = i * kRowsPerPass;
        const uint32_t row = __shfl_sync(0xffffffffu, rows, r + row0);
        const uint32_t bytes = row != 0xFFFFFFFFu ? 16 : 0;
        const size_t at = row != 0xFFFFFFFFu ? (size_t)row * row_stride + head : head;
        const uint32_t d = dst + r * (HD * 2) + ((chunk ^ ((r + row0) & 7)) << 4);
        cp_async16_zfill(d, a.kc + at, bytes);
        cp_async16_zfill(d + kRowsStep * HD * 2, a.vc + at, bytes);
      }
    }
  };
  // Q^T fragments of a unit: head lane / 4 of each column tile, two values a word.
  auto load_q = [&](const Cursor& c, uint32_t (&q)[NT][kK][2]) {
    const int kv = c.unit / a.head_tiles, ht = c.unit % a.head_tiles;
    const int here = min(a.heads, a.group - ht * a.heads);
    const __half* base = a.q + ((size_t)c.s * a.qh + kv * a.group + ht * a.heads) * HD;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int h = n * 8 + (lane >> 2);
#pragma unroll
      for (int kk = 0; kk < kK; ++kk)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          q[n][kk][e] = h < here ? *reinterpret_cast<const uint32_t*>(
                                       base + (size_t)h * HD + kk * 16 + e * 8 + (lane & 3) * 2)
                                 : 0u;
    }
  };

  Cursor comp = first;
  if (begin < end && comp.tile >= comp.tiles) {  // a unit's empty places come first
    advance(comp);
  }
  if (begin < end && comp.place < end) {
    Cursor load = comp;
    uint32_t rows = row_of(load);
    auto issue_next = [&](int stage) {
      const Cursor now = load;
      const uint32_t r = rows;
      advance(load);
      if (load.place < end) rows = row_of(load);
      issue(now, r, stage);
    };
    for (int i = 0; i < kStages - 1; ++i) {
      if (load.place < end) issue_next(i);
      pipe::cp_async_commit();
    }
    uint32_t qf[NT][kK][2];
    load_q(comp, qf);
    float o[kK][NT][4] = {};
    float m[NT][2], l[NT][2];  // m: maximum less kLift
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
    }
    int steps = 0;       // since the accumulators were 0
    bool aside = false;  // some are put aside
    // Adds what is aside to the accumulators.
    auto take_back = [&](const float* at) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float* p = at + (n * 2 + e) * (HD / 16 * 2 + 2) * 32;
          const float base = p[HD / 16 * 2 * 32];
          const float g = base == m[n][e] ? 1.f : state_weight(base, m[n][e]);
          l[n][e] += g * p[(HD / 16 * 2 + 1) * 32];
#pragma unroll
          for (int kk = 0; kk < kK; ++kk) {
            o[kk][n][e] += g * p[2 * kk * 32];
            o[kk][n][e + 2] += g * p[(2 * kk + 1) * 32];
          }
        }
    };
    auto put_aside = [&](float* at) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float* p = at + (n * 2 + e) * (HD / 16 * 2 + 2) * 32;
          p[HD / 16 * 2 * 32] = m[n][e];
          p[(HD / 16 * 2 + 1) * 32] = l[n][e];
          l[n][e] = 0.f;
#pragma unroll
          for (int kk = 0; kk < kK; ++kk) {
            p[2 * kk * 32] = o[kk][n][e];
            p[(2 * kk + 1) * 32] = o[kk][n][e + 2];
            o[kk][n][e] = o[kk][n][e + 2] = 0.f;
          }
        }
    };
    auto place_aside = [&] {
      return a.aside + ((size_t)blockIdx.x * kWarps + warp) * aside_floats(HD, NT) * 32 + lane;
    };
    bool begins = comp.tile == 0;  // this segment holds its unit's first tile
    int stage = 0;
    const int key_k = lane & 15, chunk_k = lane >> 4;                       // K as rows of keys
    const int key_v = (lane & 7) + 8 * (lane >> 4), chunk_v = (lane >> 3) & 1;  // V^T as rows of dims
    while (true) {
      // refill the stage that the previous step read
      int st = stage + kStages - 1;
      if (st >= kStages) st -= kStages;
      if (load.place < end) issue_next(st);
      pipe::cp_async_commit();
      cp_async_wait<kStages - 1>();
      __syncwarp();
      const uint32_t kbase = ring + stage * S::kStageBytes;
      const uint32_t vbase = kbase + kRowsStep * HD * 2;

      // scores of 16 kSteps keys x 8 NT heads
      float sc[kSteps][NT][4] = {};
#pragma unroll
      for (int u = 0; u < kSteps; ++u)
#pragma unroll
        for (int kk = 0; kk < kK; ++kk) {
          uint32_t k4[4];
          ldsm4(k4, kbase + (u * 16 + key_k) * (HD * 2) +
                        (((2 * kk + chunk_k) ^ (key_k & 7)) << 4));
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816(sc[u][n], k4, qf[n][kk][0], qf[n][kk][1]);
        }
      const uint32_t p0 = (uint32_t)comp.tile * kTileKeys + warp * kRowsStep + (lane >> 2);
      uint32_t pf[kSteps][NT][2];
      bool moved = false;
      float f[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = -INFINITY;
#pragma unroll
          for (int u = 0; u < kSteps; ++u) {
            float& s0 = sc[u][n][e];
            float& s1 = sc[u][n][e + 2];
            s0 = p0 + u * 16 < comp.len ? s0 * a.scale_log2 : -INFINITY;
            s1 = p0 + u * 16 + 8 < comp.len ? s1 * a.scale_log2 : -INFINITY;
            x = fmaxf(x, fmaxf(s0, s1));
          }
#pragma unroll
          for (int sh = 4; sh < 32; sh <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, sh));
          const float top = fmaxf(m[n][e], x - kLift);
          f[n][e] = state_weight(m[n][e], top);
          moved |= top > m[n][e];
          m[n][e] = top;
          const float z = top == -INFINITY ? 0.f : top;
#pragma unroll
          for (int u = 0; u < kSteps; ++u) {
            sc[u][n][e] = exp2_fast(sc[u][n][e] - z);
            sc[u][n][e + 2] = exp2_fast(sc[u][n][e + 2] - z);
          }
          l[n][e] *= f[n][e];
        }
#pragma unroll
        for (int u = 0; u < kSteps; ++u) {
          // weights rounded to FP16 for the product; the sum takes the rounded
          // ones, so a row of equal values keeps its value
          const __half2 h0 = __floats2half2_rn(sc[u][n][0], sc[u][n][1]);
          const __half2 h1 = __floats2half2_rn(sc[u][n][2], sc[u][n][3]);
          const float2 g0 = __half22float2(h0), g1 = __half22float2(h1);
          l[n][0] += g0.x + g1.x;
          l[n][1] += g0.y + g1.y;
          pf[u][n][0] = transpose8(*reinterpret_cast<const uint32_t*>(&h0));
          pf[u][n][1] = transpose8(*reinterpret_cast<const uint32_t*>(&h1));
        }
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int kk = 0; kk < kK; ++kk)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            o[kk][n][0] *= f[n][0];
            o[kk][n][1] *= f[n][1];
            o[kk][n][2] *= f[n][0];
            o[kk][n][3] *= f[n][1];
          }
      }
#pragma unroll
      for (int u = 0; u < kSteps; ++u)
#pragma unroll
        for (int kk = 0; kk < kK; ++kk) {
          uint32_t v4[4];
          ldsm4_trans(v4, vbase + (u * 16 + key_v) * (HD * 2) +
                              (((2 * kk + chunk_v) ^ (key_v & 7)) << 4));
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816(o[kk][n], v4, pf[u][n][0], pf[u][n][1]);
        }
      __syncwarp();

      const bool unit_done = comp.tile + 1 == comp.tiles;
      if (!unit_done && comp.place + 1 < end) {
        if (++steps == kAsideSteps) {
          if (aside) take_back(place_aside());
          put_aside(place_aside());
          steps = 0;
          aside = true;
        }
        ++comp.tile;
        ++comp.place;
        if (++stage == kStages) stage = 0;
        continue;
      }
      // ---- a segment ends: the four warps' states become one -----------------
      if (aside) take_back(place_aside());
      const Cursor done = comp;
      advance(comp);
      const bool more = comp.place < end;
      if (more) load_q(comp, qf);  // in flight during the join
      float* state = reinterpret_cast<float*>(smem + (warp * kStages + stage) * S::kStageBytes);
      if (lane == 0) states[warp] = state;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int h = n * 8 + (lane & 3) * 2 + e;
#pragma unroll
          for (int sh = 4; sh < 32; sh <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], sh);
          if (lane < 4) {
            stats[warp][h][0] = m[n][e];
            stats[warp][h][1] = l[n][e];
          }
#pragma unroll
          for (int kk = 0; kk < kK; ++kk) {
            state[h * kRow + kk * 16 + (lane >> 2)] = o[kk][n][e];
            state[h * kRow + kk * 16 + (lane >> 2) + 8] = o[kk][n][e + 2];
          }
        }
      __syncthreads();
      const int kv = done.unit / a.head_tiles, ht = done.unit % a.head_tiles;
      const int here = min(a.heads, a.group - ht * a.heads);
      const bool whole = begins && unit_done;
      float* piece = a.pieces + ((size_t)blockIdx.x * 2 + (begins ? 1 : 0)) * piece_floats(HD);
      __half* dst = a.out + ((size_t)done.s * a.qh + kv * a.group + ht * a.heads) * HD;
      // two dims to a thread
      for (int i = tid; i < here * (HD / 2); i += kThreads) {
        const int h = i / (HD / 2), d = i % (HD / 2) * 2;
        float top = -INFINITY, sum = 0.f, x = 0.f, y = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, stats[w][h][0]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float g = state_weight(stats[w][h][0], top);
          const float2 v = *reinterpret_cast<const float2*>(states[w] + h * kRow + d);
          sum += g * stats[w][h][1];
          x += g * v.x;
          y += g * v.y;
        }
        if (whole) {
          const float inv = 1.f / sum;
          *reinterpret_cast<__half2*>(dst + h * HD + d) = __floats2half2_rn(x * inv, y * inv);
        } else {
          *reinterpret_cast<float2*>(piece + h * HD + d) = make_float2(x, y);
          if (d == 0) {
            piece[kHeadsMax * HD + 2 * h] = top;
            piece[kHeadsMax * HD + 2 * h + 1] = sum;
          }
        }
      }
      if (begins && !unit_done && tid == 0) {
        // the CTA that holds the unit's last tile
        const unsigned long long last = done.place + (done.tiles - 1 - done.tile);
        note = make_uint4((uint32_t)done.s, (uint32_t)done.unit,
                          (uint32_t)(((last + 1) * ctas - 1) / total), 1);
      }
      if (!more) break;
      __syncthreads();
      begins = true;
      steps = 0;
      aside = false;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        m[n][0] = m[n][1] = -INFINITY;
        l[n][0] = l[n][1] = 0.f;
#pragma unroll
        for (int kk = 0; kk < kK; ++kk) o[kk][n][0] = o[kk][n][1] = o[kk][n][2] = o[kk][n][3] = 0.f;
      }
      if (++stage == kStages) stage = 0;
    }
    cp_async_wait<0>();
  }
  if (tid == 0) a.meta[blockIdx.x] = note;
  pdl_trigger();
}

// Joins the pieces of the unit that CTA blockIdx.x began, one head to a block:
// the pieces' maxima first, then their rows weighted by them. Four warps take
// the pieces in turn.
template <int HD>
__global__ void __launch_bounds__(128) paged_join_kernel(const PagedArgs a) {
  constexpr int kV = HD / 32;
  __shared__ float part[4][HD];
  __shared__ float sums[4];
  // The next op's grid starts only when this one's wait is over: launched
  // earlier, its waiting CTAs take the places of the ones that still work.
  pdl_wait();
  pdl_trigger();
  const uint4 note = a.meta[blockIdx.x];
  if (!note.w) return;
  const int kv = note.y / a.head_tiles, ht = note.y % a.head_tiles;
  const int h = blockIdx.y;
  if (ht * a.heads + h >= a.group) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c0 = blockIdx.x, n = (int)note.z - c0 + 1;
  auto piece = [&](int i) {
    return a.pieces + ((size_t)(c0 + i) * 2 + (i == 0 ? 1 : 0)) * piece_floats(HD);
  };
  float top = -INFINITY;
  for (int i = lane; i < n; i += 32) top = fmaxf(top, piece(i)[kHeadsMax * HD + 2 * h]);
  top = warp_max(top);
  float acc[kV] = {}, total = 0.f;
#pragma unroll 4
  for (int i = warp; i < n; i += 4) {
    const float* p = piece(i);
    const float w = state_weight(p[kHeadsMax * HD + 2 * h], top);
    total += w * p[kHeadsMax * HD + 2 * h + 1];
#pragma unroll
    for (int e = 0; e < kV; ++e) acc[e] += w * p[h * HD + lane * kV + e];
  }
#pragma unroll
  for (int e = 0; e < kV; ++e) part[warp][lane * kV + e] = acc[e];
  if (lane == 0) sums[warp] = total;
  __syncthreads();
  for (int d = threadIdx.x; d < HD; d += 128) {
    const float l = sums[0] + sums[1] + sums[2] + sums[3];
    const float v = part[0][d] + part[1][d] + part[2][d] + part[3][d];
    a.out[((size_t)note.x * a.qh + kv * a.group + ht * a.heads + h) * HD + d] =
        __float2half_rn(v / l);
  }
}

constexpr int kCtasMax = 2;

template <int HD, int NT, bool kRuns>
void launch_paged(const Launch& l, const PagedArgs& a) {
  auto kernel = paged_attention_kernel<HD, NT, kRuns>;
  using S = PagedShape<HD, NT>;
  static_assert(S::kCtas <= kCtasMax, "workspace");
  allow_dynamic_smem(kernel, S::kBytes);
  const int grid = S::kCtas * l.sm_count;
  launch_kernel(l, dim3(grid), dim3(kThreads), S::kBytes, kernel, a);
  launch_kernel(l, dim3(grid, a.heads), dim3(128), 0, paged_join_kernel<HD>, a);
}

template <int HD>
void launch_paged(const Launch& l, PagedArgs& a) {
  const bool runs = a.page % 16 == 0;
  const int most = a.group <= 8 ? 8 : kHeadsMax;
  a.head_tiles = (a.group + most - 1) / most;
  a.heads = (a.group + a.head_tiles - 1) / a.head_tiles;
  if (a.heads <= 8)
    runs ? launch_paged<HD, 1, true>(l, a) : launch_paged<HD, 1, false>(l, a);
  else
    runs ? launch_paged<HD, 2, true>(l, a) : launch_paged<HD, 2, false>(l, a);
}

}  // namespace

void paged_append(const Launch& l, const PagedAppend& p) {
  if (p.tokens == 0 || p.sequences == 0) return;
  AppendArgs a{p.q, p.k, p.v, p.qw, p.kw, p.q_out, p.key_cache, p.value_cache, p.starts,
               p.lengths, p.table, p.fault, p.tokens, p.sequences, p.qh, p.kvh, p.table_width,
               p.page, p.pages, p.theta, p.eps, 1.f / (float)(p.qh + 2 * p.kvh)};
  if (p.hd == 128)
    launch_append<128>(l, a);
  else
    launch_append<64>(l, a);
}

size_t paged_attention_workspace(int sm_count, int hd) {
  const size_t c = kCtasMax * sm_count;
  return c * (sizeof(uint4) + 2 * piece_floats(hd) * sizeof(float) +
              (size_t)kThreads * aside_floats(hd, kHeadsMax / 8) * sizeof(float));
}

void paged_attention(const Launch& l, const PagedAttention& p, void* workspace) {
  if (p.sequences == 0) return;
  const size_t c = kCtasMax * l.sm_count;
  PagedArgs a{};
  a.q = p.q;
  a.kc = p.key_cache;
  a.vc = p.value_cache;
  a.out = p.out;
  a.lengths = p.lengths;
  a.table = p.table;
  a.meta = static_cast<uint4*>(workspace);
  a.pieces = reinterpret_cast<float*>(a.meta + c);
  a.aside = a.pieces + c * 2 * piece_floats(p.hd);
  a.fault = p.fault;
  a.sequences = p.sequences;
  a.qh = p.qh;
  a.kvh = p.kvh;
  a.table_width = p.table_width;
  a.page = p.page;
  a.group = p.qh / p.kvh;
  a.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (p.page == 1 << i) a.page_shift = i;
  a.pages = p.pages;
  a.scale_log2 = (float)(1.4426950408889634 / sqrt((double)p.hd));
  if (p.hd == 128)
    launch_paged<128>(l, a);
  else
    launch_paged<64>(l, a);
}

}  // namespace k
}  // namespace mi
