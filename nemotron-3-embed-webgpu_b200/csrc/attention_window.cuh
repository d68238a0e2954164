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

// Weights are 2^(score - reference), with a reference this far (log2) below the
// running maximum. f16 has less than 11 bits below 2^-14: beside a weight of 1,
// the small ones of a long cache would lose them, or all round alike (one key with
// half of the weight, 131072 with the rest: 3.4e-3 off without, 1.4e-3 with). In
// the tile kernel more would leave too little room above an old maximum (7: 107 us
// where 0 and 4 take 103). Where scores are so large that the difference is
// rounded, it is at most 8.
template <typename T>
constexpr float weight_lift() {
  return 0.f;
}
template <>
constexpr float weight_lift<__half>() {
  return 4.f;
}

// Which of 8 elements have an exponent field of ones (an infinity or NaN), and
// which are NaN: a bit each.
template <typename T>
struct Special;
template <>
struct Special<__half> {
  static constexpr uint32_t kExp = 0x7c00;
};
template <>
struct Special<__nv_bfloat16> {
  static constexpr uint32_t kExp = 0x7f80;
};
template <typename T>
__device__ __forceinline__ bool any_special(const uint4& u) {
  constexpr uint32_t kExp2 = Special<T>::kExp * 0x10001u, kStep = (0x8000u - Special<T>::kExp) * 0x10001u;
  return ((((u.x & kExp2) + kStep) | ((u.y & kExp2) + kStep) | ((u.z & kExp2) + kStep) | ((u.w & kExp2) + kStep)) &
          0x80008000u) != 0;
}
template <typename T>
__device__ __forceinline__ void special8(const uint4& u, uint32_t& nans, uint32_t& infs) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  nans = infs = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t h = w[e / 2] >> (e & 1) * 16 & 0x7fff;
    nans |= (h > Special<T>::kExp ? 1u : 0u) << e;
    infs |= (h == Special<T>::kExp ? 1u : 0u) << e;
  }
}

// The elements of columns 8 g .. 8 g + 7 of a head's values (v) that are NaN or
// infinite in some key of `range`, as bits; by one warp, a key a lane. Ends once
// every column of `want` has a NaN, or an infinity where `inf_will_do`.
template <typename T>
__device__ __forceinline__ void seen_specials(const T* v, int64_t ldv, const KeyRange& range, int g, uint32_t want,
                                              uint32_t inf_will_do, uint32_t& nans, uint32_t& infs) {
  constexpr int kAhead = 4;
  const int lane = threadIdx.x & 31;
  nans = infs = 0;
  for (int part = 0; part < 2; ++part) {
    const int end = part ? range.hi : range.sink;
    for (int j = part ? range.lo : 0; j < end; j += 32 * kAhead) {
      uint4 u[kAhead];
      bool hit = false;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int key = j + i * 32 + lane;
        u[i] = make_uint4(0, 0, 0, 0);
        if (key < end) u[i] = *reinterpret_cast<const uint4*>(v + (int64_t)key * ldv + g * 8);
        hit |= any_special<T>(u[i]);
      }
      if (!__any_sync(0xffffffffu, hit)) continue;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        uint32_t n, f;
        special8<T>(u[i], n, f);
        nans |= __reduce_or_sync(0xffffffffu, n);
        infs |= __reduce_or_sync(0xffffffffu, f);
      }
      if (!(want & ~nans & ~(infs & inf_will_do))) return;
    }
  }
}

// Makes the columns [d0, d1) of the output of query row i of request r for one
// head right where the tiled kernels left an infinity or NaN there, by one warp.
// Those kernels multiply weights of 0 with values of keys that other queries of
// the tile see, so a value that is infinite or NaN reaches rows that do not see
// it. Only called where the row's sum of weights is finite, that is where no
// score of a key that it sees is NaN or +infinity. A column stands as it is if
// the row does see a NaN in it, or, where the result is an infinity (and so no
// NaN arose), sees an infinity: that takes one walk over the column's values.
// What is left is computed again from the keys that the row sees, 32 at a time.
// (8192 causal queries of 24 heads of 128 with one such value in sight of all: a
// walk key by key over every row took 228 ms where the clean call takes 0.4.)
template <typename T, int D>
__device__ __noinline__ void attention_row(const AttnWindowArgs& a, AttnRequest r, int i, int head, int d0, int d1) {
  constexpr uint32_t kAll = 0xffffffffu;
  constexpr int kLanes = D / 8;         // lanes with 8 columns each
  constexpr int kKeys = 32 / kLanes;    // keys side by side
  const int lane = threadIdx.x & 31, g = lane % kLanes, sub = lane / kLanes;
  const int kvh = head / (a.q_heads / a.kv_heads);
  const int p = i + r.nk - r.nq;
  const T* q = static_cast<const T*>(a.q) + (int64_t)(r.q0 + i) * a.ldq + head * D;
  const T* k = static_cast<const T*>(a.k) + (int64_t)r.k0 * a.ldk + kvh * D;
  const T* v = static_cast<const T*>(a.v) + (int64_t)r.k0 * a.ldv + kvh * D;
  T* out = static_cast<T*>(a.out) + (int64_t)(r.q0 + i) * a.ldo + head * D;
  const KeyRange range(a, p, p, r.nk);

  uint32_t need = 0, inf_out = 0;  // of the lane's columns: to be looked at, infinite
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int col = g * 8 + e;
    if (col < d0 || col >= d1) continue;
    const uint32_t h = *reinterpret_cast<const uint16_t*>(out + col) & 0x7fff;
    need |= (h >= Special<T>::kExp ? 1u : 0u) << e;
    inf_out |= (h == Special<T>::kExp ? 1u : 0u) << e;
  }
  for (uint32_t left = __ballot_sync(kAll, sub == 0 && need); left; left &= left - 1) {
    const int from = __ffs(left) - 1;
    const uint32_t want = __shfl_sync(kAll, need, from), inf_will_do = __shfl_sync(kAll, inf_out, from);
    uint32_t nans, infs;
    seen_specials<T>(v, a.ldv, range, from, want, inf_will_do, nans, infs);
    if (g == from) need &= ~(nans | (infs & inf_out));
  }
  if (!__any_sync(kAll, need)) return;

  float qv[8], m = -INFINITY, l = 0.f, acc[8];  // acc: the mean so far, of the lane's columns and keys
  dev::unpack8<T>(*reinterpret_cast<const uint4*>(q + g * 8), qv);
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = 0.f;
  bool done = false;
  for (int part = 0; part < 2 && !done; ++part) {
    const int end = part ? range.hi : range.sink;
    for (int base = part ? range.lo : 0; base < end && !done; base += 32) {
      const int n = min(32, end - base);
      float s = 0.f;
#pragma unroll 8
      for (int t = 0; t < kLanes; ++t) {
        const int key = t * kKeys + sub;
        float dot = 0.f;
        if (key < n) {
          float kv[8];
          dev::unpack8<T>(*reinterpret_cast<const uint4*>(k + (int64_t)(base + key) * a.ldk + g * 8), kv);
#pragma unroll
          for (int e = 0; e < 8; ++e) dot = fmaf(qv[e], kv[e], dot);
        }
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) dot += __shfl_xor_sync(kAll, dot, o);
        const float x = __shfl_sync(kAll, dot, lane % kKeys * kLanes);
        if (lane / kKeys == t) s = x;  // lane = key
      }
      s = lane < n ? s * (a.scale * 1.4426950408889634f) : -INFINITY;
      if (__any_sync(kAll, !(s < INFINITY))) {  // makes the row NaN, as in a softmax
        l = __uint_as_float(0x7fc00000u);
        done = true;
        break;
      }
      float mn = s, sum;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mn = fmaxf(mn, __shfl_xor_sync(kAll, mn, o));
      mn = fmaxf(mn, m);
      float w = s == -INFINITY ? 0.f : exp2f(s - mn);
      sum = w;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kAll, sum, o);
      const float kept = m == -INFINITY ? 0.f : l * exp2f(m - mn);
      m = mn, l = kept + sum;
      const float inv = l > 0.f ? 1.f / l : 0.f;
      w *= inv;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] *= kept * inv;
#pragma unroll 8
      for (int t = 0; t < kLanes; ++t) {
        const int key = t * kKeys + sub;
        const float wk = __shfl_sync(kAll, w, key);
        if (key < n && need) {
          float vv[8];
          dev::unpack8<T>(*reinterpret_cast<const uint4*>(v + (int64_t)(base + key) * a.ldv + g * 8), vv);
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[e] = fmaf(wk, vv[e], acc[e]);
        }
      }
      uint32_t lost = 0;  // columns that are NaN whatever follows
#pragma unroll
      for (int e = 0; e < 8; ++e) lost |= (isnan(acc[e]) ? 1u : 0u) << e;
#pragma unroll
      for (int o = kLanes; o < 32; o <<= 1) lost |= __shfl_xor_sync(kAll, lost, o);
      done = l > 0.f && __all_sync(kAll, !(need & ~lost));
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
#pragma unroll
    for (int o = kLanes; o < 32; o <<= 1) acc[e] += __shfl_xor_sync(kAll, acc[e], o);
    if (sub == 0 && (need >> e & 1)) out[g * 8 + e] = dev::from_f32<T>(l == 0.f ? 0.f : l > 0.f ? acc[e] : l);
  }
}

}  // namespace nemo
