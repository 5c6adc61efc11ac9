// Attention over packed prompts: sequences of different lengths laid end to
// end, grouped heads, causal from the ends (a prefix of keys computed before
// is allowed) or not.

#include "device.cuh"

namespace mi {
namespace k {

namespace {

struct PackedArgs {
  const __half *q, *k, *v;
  __half* out;
  const uint32_t *query_starts, *key_starts;
  uint32_t* fault;
  int tokens, keys, sequences, qh, kvh, causal;
  float scale;
};

// One row by one warp, from the formula: o = sum_j softmax_j(q . k_j / sqrt(d))
// v_j over the first `visible` keys, 32 keys at a time with a running maximum
// and sum. Keys behind `visible` are never read.
template <int HD>
__device__ void attention_row(const __half* q, const __half* k, const __half* v, size_t stride,
                              int visible, float scale, __half* out) {
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
      s *= scale;
    }
    const float top = fmaxf(m, warp_max(s));
    const float base = top == -INFINITY ? 0.f : top;
    const float keep = m == -INFINITY ? 0.f : mi_exp(m - base);
    const float p = j < visible ? mi_exp(s - base) : 0.f;
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
  for (int e = 0; e < kV; ++e)
    out[lane * kV + e] = __float2half_rn(visible > 0 ? acc[e] / l : 0.f);
}

template <int HD>
__global__ void __launch_bounds__(128) packed_row_kernel(const PackedArgs a) {
  pdl_trigger();
  pdl_wait();
  if (blockIdx.x == 0)  // every pair of starts is looked at once
    for (int s = threadIdx.x; s < a.sequences; s += 128)
      if (a.query_starts[s] > a.query_starts[s + 1] || a.key_starts[s] > a.key_starts[s + 1] ||
          a.query_starts[s + 1] > (uint32_t)a.tokens || a.key_starts[s + 1] > (uint32_t)a.keys)
        report_fault(a.fault, kFaultStarts);
  const size_t row = (size_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= (size_t)a.tokens * a.qh) return;
  const uint32_t t = row / a.qh;
  const int head = row % a.qh;
  int lo = 0, hi = a.sequences;  // sequences that end at or before t
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (a.query_starts[mid + 1] <= t) lo = mid + 1;
    else hi = mid;
  }
  if (lo >= a.sequences || a.query_starts[lo] > t) return;
  const uint32_t qe = a.query_starts[lo + 1], kb = a.key_starts[lo], ke = a.key_starts[lo + 1];
  if (kb > ke || ke > (uint32_t)a.keys || qe > (uint32_t)a.tokens) return;
  const long long n = ke - kb;
  long long visible = a.causal ? n - (long long)(qe - 1 - t) : n;
  visible = visible < 0 ? 0 : visible;
  const int kv = head / (a.qh / a.kvh);
  const size_t stride = (size_t)a.kvh * HD;
  attention_row<HD>(a.q + row * HD, a.k + kb * stride + kv * HD, a.v + kb * stride + kv * HD,
                    stride, (int)visible, a.scale, a.out + row * HD);
}

template <int HD>
void launch_packed(const Launch& l, const PackedArgs& a) {
  const size_t rows = (size_t)a.tokens * a.qh;
  launch_kernel(l, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, packed_row_kernel<HD>, a);
}

}  // namespace

void packed_attention(const Launch& l, const PackedAttention& p) {
  if (p.tokens == 0 || p.sequences == 0) return;
  PackedArgs a{p.q, p.k, p.v, p.out, p.query_starts, p.key_starts, p.fault, p.tokens, p.keys,
               p.sequences, p.qh, p.kvh, p.causal, (float)(1.0 / sqrt((double)p.hd))};
  if (p.hd == 128)
    launch_packed<128>(l, a);
  else
    launch_packed<64>(l, a);
}

}  // namespace k
}  // namespace mi
