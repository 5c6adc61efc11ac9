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
// once by HD / 8 lanes (16 bytes a lane). The arithmetic is that of
// qk_norm_rope_cache and rope (numerics.cuh), so a paged cache holds the same
// bits as a contiguous one.
//
// A block takes kTok tokens at a time and first fills a table of their
// cosines and sines: the angles need double precision (numerics.cuh), which a
// thread per (token, pair) pays once for all heads, and the frequency's pow
// once for all of a block's tokens.
constexpr int kAppendThreads = 256;

struct AppendArgs {
  const __half *q, *k, *v, *qw, *kw;
  __half *q_out, *kc, *vc;
  const uint32_t *starts, *lengths, *table;
  uint32_t* fault;
  int tokens, sequences, qh, kvh, table_width, page;
  uint32_t pages;
  float theta, eps;
};

template <int HD, int kTok>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const AppendArgs a) {
  constexpr int kLanes = HD / 8;           // lanes of a head row
  constexpr int kRows = kAppendThreads / kLanes;
  constexpr int kPairs = HD / 2;
  __shared__ float2 cs[kTok][kPairs];
  __shared__ uint32_t position[kTok];
  __shared__ uint32_t slot[kTok];          // cache row of the token
  const int tid = threadIdx.x;
  const int li = tid % kLanes;
  const int pair0 = tid % kPairs;
  float frequency = 0.f;
  if (tid < kTok * kPairs)
    frequency = (float)pow((double)a.theta, (double)__fdiv_rn(-(float)(pair0 * 2), (float)HD));
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
    for (int i = tid; i < kTok * kPairs; i += kAppendThreads) {
      const int t = i / kPairs;
      if (slot[t] != 0xFFFFFFFFu) {
        double s, c;
        sincos((double)__fmul_rn((float)position[t], frequency), &s, &c);
        cs[t][pair0] = make_float2((float)c, (float)s);
      }
    }
    __syncthreads();
    const int heads = a.qh + 2 * a.kvh;
    for (int r = tid / kLanes; r < kTok * heads; r += kRows) {
      const int i = r / heads, h = r - i * heads;
      const uint32_t row = slot[i];
      if (row == 0xFFFFFFFFu) continue;
      const size_t t = t0 + i;
      if (h >= a.qh + a.kvh) {
        const int kv = h - a.qh - a.kvh;
        reinterpret_cast<uint4*>(a.vc + ((size_t)row * a.kvh + kv) * HD)[li] =
            reinterpret_cast<const uint4*>(a.v + (t * a.kvh + kv) * HD)[li];
        continue;
      }
      // the lanes of a head row stay together, two or four rows to a warp
      const unsigned group = (kLanes == 32 ? 0xffffffffu : ((1u << kLanes) - 1))
                             << ((tid & 31) / kLanes * kLanes);
      const bool is_q = h < a.qh;
      if (is_q && !a.q) continue;
      const __half* src = is_q ? a.q + (t * a.qh + h) * HD : a.k + (t * a.kvh + h - a.qh) * HD;
      __half* dst = is_q ? a.q_out + (t * a.qh + h) * HD
                         : a.kc + ((size_t)row * a.kvh + h - a.qh) * HD;
      const uint4 raw = reinterpret_cast<const uint4*>(src)[li];
      const __half* w = is_q ? a.qw : a.kw;
      const __half2* hr = reinterpret_cast<const __half2*>(&raw);
      float x[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = __half22float2(hr[e]);
        x[2 * e] = f.x;
        x[2 * e + 1] = f.y;
      }
      if (w) {
        const float scale =
            rms_scale(canon_butterfly_mask(chunk_sq(raw, 0.f), kLanes, group), HD, a.eps);
        const uint4 wr = reinterpret_cast<const uint4*>(w)[li];
        const __half2* hw = reinterpret_cast<const __half2*>(&wr);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 g = __half22float2(hw[e]);
          x[2 * e] = norm_mul(x[2 * e], scale, g.x);
          x[2 * e + 1] = norm_mul(x[2 * e + 1], scale, g.y);
        }
      }
      const bool first = li < kLanes / 2;
      uint4 packed;
      __half2* hp = reinterpret_cast<__half2*>(&packed);
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float other = __shfl_xor_sync(group, x[e], kLanes / 2);
        const float2 t2 = cs[i][8 * (first ? li : li - kLanes / 2) + e];
        y[e] = first ? __fsub_rn(__fmul_rn(x[e], t2.x), __fmul_rn(other, t2.y))
                     : __fadd_rn(__fmul_rn(other, t2.y), __fmul_rn(x[e], t2.x));
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        hp[e] = __halves2half2(__float2half_rn(y[2 * e]), __float2half_rn(y[2 * e + 1]));
      reinterpret_cast<uint4*>(dst)[li] = packed;
    }
    __syncthreads();
  }
}

template <int HD>
void launch_append(const Launch& l, const AppendArgs& a) {
  // Four tokens to a block amortise the table's barriers; few tokens take a
  // block each, since latency is then all there is.
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
// of its group, which are the rows of an m16n8k16 product (a group of more
// than 16 takes several row tiles).
//
// The work is cut evenly whatever the lengths are: all (sequence, KV head,
// row tile) units are laid end to end in tiles of 64 keys, and CTA c of C
// takes tiles [c N / C, (c + 1) N / C). A unit that lies inside a CTA is
// finished there; one that crosses CTAs leaves unnormalised pieces that a
// second kernel joins in order of position, so results do not depend on
// timing. A CTA has at most two pieces: one that continues a unit from the
// CTA before it (slot 0), one that a later CTA continues (slot 1).
//
// Each of a CTA's four warps owns 16 keys of a tile, with its own ring of
// cp.async stages (rows past the length are filled with zeros, so stale
// values never enter a product) and its own running maximum and sum; the
// warps meet only at a unit's end.
constexpr int kTileKeys = 64;
constexpr int kWarps = 4;
constexpr int kStages = 3;
constexpr int kRowsMax = 16;

struct PagedArgs {
  const __half *q, *kc, *vc;
  __half* out;
  const uint32_t *lengths, *table;
  float* pieces;    // [C][2][16 * HD + 32]
  uint4* meta;      // [C]: of the unit that slot 1 begins: sequence, unit, last CTA, flag
  uint32_t* fault;
  int sequences, qh, kvh, table_width, page;
  uint32_t pages;
  float scale_log2; // log2(e) / sqrt(HD)
};

template <int HD>
struct PagedSmem {
  static constexpr int kStageBytes = 2 * 16 * HD * 2;  // a warp's keys and values
  static constexpr int kRing = kWarps * kStages * kStageBytes;
  static constexpr int kMerge = 2 * kRowsMax * HD * 4;
  static constexpr int kBytes = kRing + kMerge + kWarps * kRowsMax * 8 + 64;
};

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
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
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

// Length of a sequence as the kernels use it: 0 where the table cannot hold it.
__device__ __forceinline__ uint32_t paged_length(const PagedArgs& a, int s) {
  const uint32_t n = a.lengths[s];
  return (uint64_t)n > (uint64_t)a.table_width * a.page ? 0u : n;
}

// Walks a CTA's tiles in order.
struct Cursor {
  int s, unit, tile;  // sequence, unit of the sequence, tile of the unit
  int tiles;          // tiles of a unit of this sequence
  uint32_t len;
};

template <int HD>
__global__ void __launch_bounds__(kWarps * 32, 2) paged_attention_kernel(const PagedArgs a) {
  using S = PagedSmem<HD>;
  constexpr int kK = HD / 16;      // k16 steps of a score
  constexpr int kN = HD / 8;       // n8 tiles of an output row
  constexpr int kChunks = HD / 8;  // 16-byte chunks of a row
  extern __shared__ __align__(128) uint8_t smem[];
  float* merge = reinterpret_cast<float*>(smem + S::kRing);
  float* stats = reinterpret_cast<float*>(smem + S::kRing + S::kMerge);  // [warp][16][2]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int group = a.qh / a.kvh;
  const int row_tiles = (group + kRowsMax - 1) / kRowsMax;
  const int units = a.kvh * row_tiles;

  pdl_trigger();
  pdl_wait();

  // Where this CTA's tiles begin: tiles per sequence, summed by the block
  // (each thread a run of consecutive sequences).
  __shared__ unsigned long long scan[kWarps * 32 + 1];
  __shared__ Cursor first;
  const int run = (a.sequences + kWarps * 32 - 1) / (kWarps * 32);
  unsigned long long mine = 0;
  for (int i = 0; i < run; ++i) {
    const int s = tid * run + i;
    if (s < a.sequences) {
      const uint32_t n = paged_length(a, s);
      mine += (n + kTileKeys - 1) / kTileKeys;
      if (n == 0 && s % gridDim.x == blockIdx.x && a.lengths[s] != 0)
        report_fault(a.fault, kFaultLength);
    }
  }
  {
    unsigned long long v = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    if (lane == 31) scan[warp] = v;
    __syncthreads();
    unsigned long long base = 0, all = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) base += scan[w];
      all += scan[w];
    }
    __syncthreads();
    mine = base + v - mine;  // tiles before this thread's sequences
    if (tid == 0) {
      scan[0] = all;
      first.s = a.sequences;
    }
  }
  __syncthreads();
  const unsigned long long total = scan[0] * units;
  // no more CTAs than tiles, so that every one between a unit's first and last
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
      const int tiles = (n + kTileKeys - 1) / kTileKeys;
      const unsigned long long next = at + (unsigned long long)tiles * units;
      if (at <= begin && begin < next) {
        const unsigned long long w = begin - at;
        first = Cursor{s, (int)(w / tiles), (int)(w % tiles), tiles, n};
      }
      at = next;
    }
  }
  // Rows of sequences without keys are zero.
  for (int s = blockIdx.x; s < a.sequences; s += gridDim.x)
    if (paged_length(a, s) == 0)
      for (int i = tid; i < a.qh * HD / 8; i += kWarps * 32)
        reinterpret_cast<uint4*>(a.out + (size_t)s * a.qh * HD)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  uint4 note = make_uint4(0, 0, 0, 0);
  const long long count = (long long)(end - begin);

  auto advance = [&](Cursor& c) {
    if (++c.tile < c.tiles) return;
    c.tile = 0;
    if (++c.unit < units) return;
    c.unit = 0;
    do {
      if (++c.s >= a.sequences) return;
      c.len = paged_length(a, c.s);
      c.tiles = (c.len + kTileKeys - 1) / kTileKeys;
    } while (c.tiles == 0);
  };

  const uint32_t ring = pipe::smem_u32(smem) + warp * kStages * S::kStageBytes;
  const size_t row_stride = (size_t)a.kvh * HD;
  // Issues one stage: lane l looks up row l % 16, then copies 16-byte chunks.
  auto row_of = [&](const Cursor& c) -> uint32_t {
    const uint32_t p = (uint32_t)c.tile * kTileKeys + warp * 16 + (lane & 15);
    if (p >= c.len) return 0xFFFFFFFFu;
    const uint32_t pi = p / (uint32_t)a.page;
    const uint32_t pg = a.table[(size_t)c.s * a.table_width + pi];
    if (pg >= a.pages) {
      report_fault(a.fault, kFaultPage);
      return 0xFFFFFFFFu;
    }
    return pg * a.page + (p - pi * a.page);
  };
  auto issue = [&](const Cursor& c, uint32_t rows, int stage) {
    const uint32_t dst = ring + stage * S::kStageBytes;
    const int kv = c.unit / row_tiles;
    constexpr int kRowsPerPass = 32 / kChunks;
    const int chunk = lane % kChunks;
#pragma unroll
    for (int i = 0; i < 16 / kRowsPerPass; ++i) {
      const int r = i * kRowsPerPass + lane / kChunks;
      const uint32_t row = __shfl_sync(0xffffffffu, rows, r);
      const bool ok = row != 0xFFFFFFFFu;
      const size_t off = (size_t)(ok ? row : 0) * row_stride + kv * HD + chunk * 8;
      const uint32_t d = dst + r * (HD * 2) + ((chunk ^ (r & 7)) << 4);
      cp_async16_zfill(d, a.kc + off, ok ? 16 : 0);
      cp_async16_zfill(d + 16 * HD * 2, a.vc + off, ok ? 16 : 0);
    }
  };

  if (count > 0) {
    Cursor load = first, comp = first;
    long long loaded = 0;
    uint32_t rows = row_of(load);
    for (int i = 0; i < kStages - 1; ++i) {
      if (loaded < count) {
        const Cursor now = load;
        const uint32_t r = rows;
        if (++loaded < count) {
          advance(load);
          rows = row_of(load);
        }
        issue(now, r, i);
      }
      pipe::cp_async_commit();
    }
    uint32_t qf[kK][4];
    float o[kN][4];
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    bool fresh = true;
    bool begins = false;  // this segment holds its unit's first tile
    int stage = 0;
    long long issued = loaded < count ? loaded : count;
    for (long long it = 0; it < count; ++it) {
      const int unit = comp.unit;
      const int kv = unit / row_tiles, rt = unit % row_tiles;
      const int rows_here = min(kRowsMax, group - rt * kRowsMax);
      if (fresh) {
        fresh = false;
        begins = comp.tile == 0;
        const __half* q = a.q + ((size_t)comp.s * a.qh + kv * group + rt * kRowsMax) * HD;
        const int r0 = lane >> 2, c0 = (lane & 3) * 2;
#pragma unroll
        for (int kk = 0; kk < kK; ++kk) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = r0 + (e & 1) * 8, c = kk * 16 + c0 + (e >> 1) * 8;
            qf[kk][e] = r < rows_here ? *reinterpret_cast<const uint32_t*>(q + (size_t)r * HD + c)
                                      : 0u;
          }
        }
#pragma unroll
        for (int n = 0; n < kN; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
        m0 = m1 = -INFINITY;
        l0 = l1 = 0.f;
      }
      // refill the stage that the previous step read
      if (issued < count) {
        const Cursor now = load;
        const uint32_t r = rows;
        if (++issued < count) {
          advance(load);
          rows = row_of(load);
        }
        int st = stage + kStages - 1;
        if (st >= kStages) st -= kStages;
        issue(now, r, st);
      }
      pipe::cp_async_commit();
      cp_async_wait<kStages - 1>();
      __syncwarp();
      const uint32_t kbase = ring + stage * S::kStageBytes;
      const uint32_t vbase = kbase + 16 * HD * 2;
      if (++stage == kStages) stage = 0;

      // scores of 16 rows x 16 keys
      float sc[2][4] = {};
      const int key = lane & 15;
#pragma unroll
      for (int kk = 0; kk < kK; ++kk) {
        uint32_t b[4];
        const int chunk = 2 * kk + (lane >> 4);
        ldsm4(b, kbase + key * (HD * 2) + ((chunk ^ (key & 7)) << 4));
        mma16816(sc[0], qf[kk], b[0], b[2]);
        mma16816(sc[1], qf[kk], b[1], b[3]);
      }
      const int p0 = comp.tile * kTileKeys + warp * 16 + (lane & 3) * 2;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool seen = (uint32_t)(p0 + n * 8 + (e & 1)) < comp.len;
          sc[n][e] = seen ? sc[n][e] * a.scale_log2 : -INFINITY;
        }
      float x0 = fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[1][0], sc[1][1]));
      float x1 = fmaxf(fmaxf(sc[0][2], sc[0][3]), fmaxf(sc[1][2], sc[1][3]));
#pragma unroll
      for (int sh = 1; sh < 4; sh <<= 1) {
        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, sh));
        x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, sh));
      }
      const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
      if (__any_sync(0xffffffffu, n0 > m0 || n1 > m1)) {
        const float f0 = m0 == -INFINITY ? 0.f : exp2_fast(m0 - n0);
        const float f1 = m1 == -INFINITY ? 0.f : exp2_fast(m1 - n1);
        l0 *= f0;
        l1 *= f1;
#pragma unroll
        for (int n = 0; n < kN; ++n) {
          o[n][0] *= f0;
          o[n][1] *= f0;
          o[n][2] *= f1;
          o[n][3] *= f1;
        }
        m0 = n0;
        m1 = n1;
      }
      const float z0 = m0 == -INFINITY ? 0.f : m0, z1 = m1 == -INFINITY ? 0.f : m1;
      uint32_t pf[4];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        // weights rounded to FP16 for the product; the sum takes the rounded
        // ones, so a row of equal values keeps its value
        const __half2 h0 = __floats2half2_rn(exp2_fast(sc[n][0] - z0), exp2_fast(sc[n][1] - z0));
        const __half2 h1 = __floats2half2_rn(exp2_fast(sc[n][2] - z1), exp2_fast(sc[n][3] - z1));
        const float2 g0 = __half22float2(h0), g1 = __half22float2(h1);
        l0 += g0.x + g0.y;
        l1 += g1.x + g1.y;
        pf[2 * n] = *reinterpret_cast<const uint32_t*>(&h0);
        pf[2 * n + 1] = *reinterpret_cast<const uint32_t*>(&h1);
      }
#pragma unroll
      for (int nn = 0; nn < kN / 2; ++nn) {
        uint32_t b[4];
        const int chunk = 2 * nn + (lane >> 4);
        ldsm4_trans(b, vbase + key * (HD * 2) + ((chunk ^ (key & 7)) << 4));
        mma16816(o[2 * nn], pf, b[0], b[1]);
        mma16816(o[2 * nn + 1], pf, b[2], b[3]);
      }
      __syncwarp();

      const bool unit_done = comp.tile + 1 == comp.tiles;
      if (!unit_done && it + 1 < count) {
        advance(comp);
        continue;
      }
      // ---- a segment ends: the four warps' states become one -----------------
      fresh = true;
#pragma unroll
      for (int sh = 1; sh < 4; sh <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, sh);
        l1 += __shfl_xor_sync(0xffffffffu, l1, sh);
      }
      const int r0 = lane >> 2, c0 = (lane & 3) * 2;
      if ((lane & 3) == 0) {
        stats[(warp * 16 + r0) * 2] = m0;
        stats[(warp * 16 + r0) * 2 + 1] = l0;
        stats[(warp * 16 + r0 + 8) * 2] = m1;
        stats[(warp * 16 + r0 + 8) * 2 + 1] = l1;
      }
      __syncthreads();
      float M0 = -INFINITY, M1 = -INFINITY, L0 = 0.f, L1 = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        M0 = fmaxf(M0, stats[(w * 16 + r0) * 2]);
        M1 = fmaxf(M1, stats[(w * 16 + r0 + 8) * 2]);
      }
      auto weight = [](float m, float top) {
        return m == -INFINITY ? 0.f : exp2_fast(m - top);
      };
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        L0 += stats[(w * 16 + r0) * 2 + 1] * weight(stats[(w * 16 + r0) * 2], M0);
        L1 += stats[(w * 16 + r0 + 8) * 2 + 1] * weight(stats[(w * 16 + r0 + 8) * 2], M1);
      }
      const float f0 = weight(m0, M0), f1 = weight(m1, M1);
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        o[n][0] *= f0;
        o[n][1] *= f0;
        o[n][2] *= f1;
        o[n][3] *= f1;
      }
      auto put = [&](float* dst) {
#pragma unroll
        for (int n = 0; n < kN; ++n) {
          if (r0 < rows_here)
            *reinterpret_cast<float2*>(dst + r0 * HD + n * 8 + c0) = make_float2(o[n][0], o[n][1]);
          if (r0 + 8 < rows_here)
            *reinterpret_cast<float2*>(dst + (r0 + 8) * HD + n * 8 + c0) =
                make_float2(o[n][2], o[n][3]);
        }
      };
      auto take = [&](const float* src) {
#pragma unroll
        for (int n = 0; n < kN; ++n) {
          if (r0 < rows_here) {
            const float2 f = *reinterpret_cast<const float2*>(src + r0 * HD + n * 8 + c0);
            o[n][0] += f.x;
            o[n][1] += f.y;
          }
          if (r0 + 8 < rows_here) {
            const float2 f = *reinterpret_cast<const float2*>(src + (r0 + 8) * HD + n * 8 + c0);
            o[n][2] += f.x;
            o[n][3] += f.y;
          }
        }
      };
      if (warp >= 2) put(merge + (warp - 2) * kRowsMax * HD);
      __syncthreads();
      if (warp < 2) take(merge + warp * kRowsMax * HD);
      __syncthreads();
      if (warp == 1) put(merge);
      __syncthreads();
      if (warp == 0) {
        take(merge);
        if (begins && unit_done) {
          const float i0 = 1.f / L0, i1 = 1.f / L1;
          __half* dst = a.out + ((size_t)comp.s * a.qh + kv * group + rt * kRowsMax) * HD;
#pragma unroll
          for (int n = 0; n < kN; ++n) {
            if (r0 < rows_here)
              *reinterpret_cast<__half2*>(dst + (size_t)r0 * HD + n * 8 + c0) =
                  __floats2half2_rn(o[n][0] * i0, o[n][1] * i0);
            if (r0 + 8 < rows_here)
              *reinterpret_cast<__half2*>(dst + (size_t)(r0 + 8) * HD + n * 8 + c0) =
                  __floats2half2_rn(o[n][2] * i1, o[n][3] * i1);
          }
        } else {
          float* piece = a.pieces + ((size_t)blockIdx.x * 2 + (begins ? 1 : 0)) *
                                        (kRowsMax * HD + 2 * kRowsMax);
          put(piece);
          if ((lane & 3) == 0) {
            float* st = piece + kRowsMax * HD;
            st[r0 * 2] = M0;
            st[r0 * 2 + 1] = L0;
            st[(r0 + 8) * 2] = M1;
            st[(r0 + 8) * 2 + 1] = L1;
          }
          if (begins) {
            // the CTA that holds the unit's last tile
            const unsigned long long last = begin + it + (comp.tiles - 1 - comp.tile);
            const uint32_t c1 = (uint32_t)(((last + 1) * ctas - 1) / total);
            note = make_uint4((uint32_t)comp.s, (uint32_t)unit, c1, 1);
          }
        }
      }
      __syncthreads();
      if (it + 1 < count) advance(comp);
    }
    cp_async_wait<0>();
  }
  if (tid == 0) a.meta[blockIdx.x] = note;
}

// Joins the pieces of the unit that CTA blockIdx.x began, one row to a block:
// the pieces' maxima and sums first, then their rows weighted by them. Four
// warps take the pieces in turn.
template <int HD>
__global__ void __launch_bounds__(128) paged_join_kernel(const PagedArgs a) {
  constexpr int kV = HD / 32;
  __shared__ float part[4][HD];
  __shared__ float sums[4];
  pdl_trigger();
  pdl_wait();
  const uint4 note = a.meta[blockIdx.x];
  if (!note.w) return;
  const int group = a.qh / a.kvh;
  const int row_tiles = (group + kRowsMax - 1) / kRowsMax;
  const int kv = note.y / row_tiles, rt = note.y % row_tiles;
  const int row = blockIdx.y;
  if (rt * kRowsMax + row >= group) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c0 = blockIdx.x, n = (int)note.z - c0 + 1;
  constexpr size_t kPiece = kRowsMax * HD + 2 * kRowsMax;
  auto piece = [&](int i) {
    return a.pieces + ((size_t)(c0 + i) * 2 + (i == 0 ? 1 : 0)) * kPiece;
  };
  float top = -INFINITY;
  for (int i = lane; i < n; i += 32) top = fmaxf(top, piece(i)[kRowsMax * HD + 2 * row]);
  top = warp_max(top);
  float acc[kV] = {}, total = 0.f;
#pragma unroll 4
  for (int i = warp; i < n; i += 4) {
    const float* p = piece(i);
    const float m = p[kRowsMax * HD + 2 * row];
    const float w = m == -INFINITY ? 0.f : exp2_fast(m - top);
    total += w * p[kRowsMax * HD + 2 * row + 1];
#pragma unroll
    for (int e = 0; e < kV; ++e) acc[e] += w * p[row * HD + lane * kV + e];
  }
#pragma unroll
  for (int e = 0; e < kV; ++e) part[warp][lane * kV + e] = acc[e];
  if (lane == 0) sums[warp] = total;
  __syncthreads();
  for (int d = threadIdx.x; d < HD; d += 128) {
    const float l = sums[0] + sums[1] + sums[2] + sums[3];
    const float v = part[0][d] + part[1][d] + part[2][d] + part[3][d];
    a.out[((size_t)note.x * a.qh + kv * group + rt * kRowsMax + row) * HD + d] =
        __float2half_rn(v / l);
  }
}

int paged_grid(int sm_count) { return 2 * sm_count; }

template <int HD>
void launch_paged(const Launch& l, const PagedArgs& a) {
  auto kernel = paged_attention_kernel<HD>;
  allow_dynamic_smem(kernel, PagedSmem<HD>::kBytes);
  const int grid = paged_grid(l.sm_count);
  launch_kernel(l, dim3(grid), dim3(kWarps * 32), PagedSmem<HD>::kBytes, kernel, a);
  launch_kernel(l, dim3(grid, std::min(a.qh / a.kvh, kRowsMax)), dim3(128), 0,
                paged_join_kernel<HD>, a);
}

}  // namespace

void paged_append(const Launch& l, const PagedAppend& p) {
  if (p.tokens == 0 || p.sequences == 0) return;
  AppendArgs a{p.q, p.k, p.v, p.qw, p.kw, p.q_out, p.key_cache, p.value_cache, p.starts,
               p.lengths, p.table, p.fault, p.tokens, p.sequences, p.qh, p.kvh, p.table_width,
               p.page, p.pages, p.theta, p.eps};
  if (p.hd == 128)
    launch_append<128>(l, a);
  else
    launch_append<64>(l, a);
}

size_t paged_attention_workspace(int sm_count, int hd) {
  const size_t c = paged_grid(sm_count);
  return c * 2 * (kRowsMax * hd + 2 * kRowsMax) * 4 + c * sizeof(uint4);
}

void paged_attention(const Launch& l, const PagedAttention& p, void* workspace) {
  if (p.sequences == 0) return;
  const size_t c = paged_grid(l.sm_count);
  PagedArgs a{};
  a.q = p.q;
  a.kc = p.key_cache;
  a.vc = p.value_cache;
  a.out = p.out;
  a.lengths = p.lengths;
  a.table = p.table;
  a.meta = static_cast<uint4*>(workspace);
  a.pieces = reinterpret_cast<float*>(a.meta + c);
  a.fault = p.fault;
  a.sequences = p.sequences;
  a.qh = p.qh;
  a.kvh = p.kvh;
  a.table_width = p.table_width;
  a.page = p.page;
  a.pages = p.pages;
  a.scale_log2 = (float)(1.4426950408889634 / sqrt((double)p.hd));
  if (p.hd == 128)
    launch_paged<128>(l, a);
  else
    launch_paged<64>(l, a);
}

}  // namespace k
}  // namespace mi
