// What the kernels of the windowed attention (nemo_op_attention_window) share:
// the request a block works on, the visible keys of its queries, and the row
// by row recomputation of results that are not finite.
#pragma once

#include "layer_ops.cuh"

namespace nemo {

// 16 rows of one kv head's group per tile (k_attention_rows.cu).
cudaError_t launch_attention_rows(const AttnWindowArgs& a, cudaStream_t s);
// Keys that `rows` consecutive queries see, at most.
int64_t visible_keys(const AttnWindowArgs& a, int rows);

// Request b with its offsets clamped into the buffers, so that a wrong offset
// cannot make a kernel leave them.
struct AttnRequest {
  int q0, nq;  // first query row, queries
  int k0, nk;  // first key row, keys
  __device__ __forceinline__ AttnRequest() {}
  __device__ __forceinline__ AttnRequest(const AttnWindowArgs& a, int b) {
    const int qa = min(max(a.q_off[b], 0), a.q_rows), qe = min(max(a.q_off[b + 1], qa), a.q_rows);
    q0 = qa;
    nq = qe - qa;
    k0 = min(max(a.k_start[b], 0), a.k_rows);
    nk = min(max(a.k_len[b], 0), a.k_rows - k0);
  }
};

// The keys that the query at position p sees: j <= last and (j >= first or
// j < sinks). Formed in 64 bits: left and right reach 2^31 - 1.
struct RowKeys {
  int first, last, sinks;
  __device__ __forceinline__ RowKeys() {}
  __device__ __forceinline__ RowKeys(const AttnWindowArgs& a, int p, int nk) {
    const int64_t h = a.right < 0 ? (int64_t)nk - 1 : (int64_t)p + a.right;
    last = (int)(h < nk - 1 ? h : nk - 1);
    const int64_t l = a.left < 0 ? 0 : (int64_t)p - a.left;
    first = (int)(l > 0 ? l : 0);
    sinks = a.sinks;
  }
  __device__ __forceinline__ bool has(int j) const { return j <= last && (j >= first || j < sinks); }
};

// The keys that some query with a position in [p0, p1] sees: sinks [0, sink)
// in front of the window [lo, hi).
struct KeyRange {
  int sink, lo, hi;
  __device__ __forceinline__ KeyRange(const AttnWindowArgs& a, int p0, int p1, int nk) {
    int64_t h = a.right < 0 ? (int64_t)nk : (int64_t)p1 + a.right + 1;
    if (h > nk) h = nk;
    if (h < 0) h = 0;
    int64_t l = a.left < 0 ? 0 : (int64_t)p0 - a.left;
    if (l < 0) l = 0;
    if (l > h) l = h;
    hi = (int)h;
    lo = (int)l;
    sink = min(a.sinks, lo);
  }
};

// The output of query row i of request r for one head, columns [d0, d1), by one
// warp, key by key and touching only keys that the query sees. The tiled
// kernels multiply weights of 0 with values of keys that other queries of the
// tile see; where such a value is infinite or NaN the product is NaN, and the
// rows it reached are computed again here (up to the key that settles the row,
// so that a call on NaN throughout does not crawl).
template <typename T>
__device__ __noinline__ void attention_row(const AttnWindowArgs& a, AttnRequest r, int i, int head, int d0,
                                           int d1) {
  const int lane = threadIdx.x & 31, d = a.head_dim;
  const int kvh = head / (a.q_heads / a.kv_heads);
  const int p = i + r.nk - r.nq;
  const T* q = static_cast<const T*>(a.q) + (int64_t)(r.q0 + i) * a.ldq + head * d;
  const T* k = static_cast<const T*>(a.k) + (int64_t)r.k0 * a.ldk + kvh * d;
  const T* v = static_cast<const T*>(a.v) + (int64_t)r.k0 * a.ldv + kvh * d;
  const KeyRange range(a, p, p, r.nk);
  float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int j = 0; j < range.hi; ++j) {
    if (j == range.sink && range.lo > j) j = range.lo;
    if (j >= range.hi) break;
    float s = 0.f;
    for (int c = lane; c < d; c += 32) s += dev::to_f32(q[c]) * dev::to_f32(k[(int64_t)j * a.ldk + c]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    s *= a.scale * 1.4426950408889634f;
    if (!(s < INFINITY)) {  // a NaN or +infinity score makes the row NaN, as it does in a softmax
      l = __uint_as_float(0x7fc00000u);
      break;
    }
    const float mn = fmaxf(m, s);
    const float keep = m == -INFINITY ? 0.f : exp2f(m - mn);
    const float w = s == -INFINITY ? 0.f : exp2f(s - mn);
    l = l * keep + w;
    bool lost = true;
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (c * 32 + lane < d) {
        acc[c] = acc[c] * keep + w * dev::to_f32(v[(int64_t)j * a.ldv + c * 32 + lane]);
        lost &= isnan(acc[c]);
      }
    if (l > 0.f && __all_sync(0xffffffffu, lost)) break;  // every column is NaN: no later key changes that
    m = mn;
  }
  T* out = static_cast<T*>(a.out) + (int64_t)(r.q0 + i) * a.ldo + head * d;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int col = c * 32 + lane;
    if (col >= d0 && col < d1) out[col] = dev::from_f32<T>(l == 0.f ? 0.f : acc[c] / l);
  }
}

}  // namespace nemo
