// Windowed attention of few query rows (nemo_op_attention_window): single
// tokens, or a few, against a cache.
//
// Bound by memory: each visible K and V row is read once per kv head and meets
// only the query rows of its group. A tile is 16 such rows, (query, head of the
// group) pairs of one kv head, which is what an m16n8k16 instruction takes; a
// 128-row tcgen05 tile would be nearly empty. The keys are split over the 4
// warps of a block and over the blocks of a cluster, each warp running its own
// online softmax over chunks of 32 keys that it copies to shared memory
// itself (no block barriers in the loop); the partial results meet in shared
// memory and, over the cluster, in distributed shared memory, always in the
// same order.
//
// Scores and statistics are f32; weights are rounded to the 16-bit type for
// the product with V (relative error half a step, like the output's own
// rounding).
#include "attention_window.cuh"

namespace nemo {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kChunk = 32;  // keys per copy

template <int D, int STAGES>
struct RowsCfg {
  static constexpr int kRowBytes = D * 2;
  static constexpr int kStage = 2 * kChunk * kRowBytes;  // K, then V
  static constexpr int kRing = kWarps * STAGES * kStage;
  // the merge reuses the ring: [warp][16][D] f32, then [warp][16] max and sum;
  // the block's own [16][D], [16], [16] lie behind it
  static constexpr int kMerge = kWarps * 16 * (D + 2) * 4;
  static constexpr int kBlock = 16 * (D + 2) * 4;
  static constexpr int kSmem = (kRing > kMerge ? kRing : kMerge) + kBlock + 64;
};

template <typename T, int D, int STAGES>
__global__ void __launch_bounds__(kThreads) attention_rows_kernel(const __grid_constant__ AttnWindowArgs a, int splits,
                                                                  int row_tiles) {
  using C = RowsCfg<D, STAGES>;
  extern __shared__ __align__(1024) uint8_t smem[];
  dev::pdl_launch_dependents();
  dev::pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = blockIdx.x % splits, tile = blockIdx.x / splits;
  const int kvh = blockIdx.y;
  const AttnRequest rq(a, blockIdx.z);
  const int group = a.q_heads / a.kv_heads;
  const int nq = min(rq.nq, a.max_q);
  const int rows = nq * group;  // of this request and kv head
  if (tile * 16 >= rows) return;  // the whole cluster
  const int i_first = tile * 16 / group, i_last = min(tile * 16 + 15, rows - 1) / group;
  const int p_off = rq.nk - rq.nq;  // position of query 0
  const KeyRange range(a, i_first + p_off, i_last + p_off, rq.nk);
  const int sink_chunks = (range.sink + kChunk - 1) / kChunk;
  const int chunks = sink_chunks + (range.hi - range.lo + kChunk - 1) / kChunk;
  const int step = splits * kWarps, c_first = rank * kWarps + warp;
  auto chunk_keys = [&](int c, int& base, int& end) {
    if (c < sink_chunks) {
      base = c * kChunk, end = range.sink;
    } else {
      base = range.lo + (c - sink_chunks) * kChunk, end = range.hi;
    }
  };
  uint8_t* ring = smem + warp * STAGES * C::kStage;
  const uint8_t* kp = reinterpret_cast<const uint8_t*>(static_cast<const T*>(a.k) + (int64_t)rq.k0 * a.ldk + kvh * D);
  const uint8_t* vp = reinterpret_cast<const uint8_t*>(static_cast<const T*>(a.v) + (int64_t)rq.k0 * a.ldv + kvh * D);
  constexpr int UNITS = D / 8;           // 16-byte units of a row
  constexpr int KEYS = 32 / UNITS;       // keys per copy instruction
  auto load = [&](int c, int stage) {
    int base, end;
    chunk_keys(c, base, end);
    const uint32_t dk = dev::smem_u32(ring + stage * C::kStage), dv = dk + kChunk * C::kRowBytes;
    const int u = lane % UNITS;
#pragma unroll
    for (int i = 0; i < kChunk / KEYS; ++i) {
      const int key = i * KEYS + lane / UNITS;
      const bool in = base + key < end;  // keys no query sees are zeros: they may hold anything
      const int64_t j = in ? base + key : base;
      const uint32_t at = key * C::kRowBytes + ((u ^ (key & 7)) * 16);
      dev::cp_async16(dk + at, kp + j * a.ldk * 2 + u * 16, in ? 16 : 0);
      dev::cp_async16(dv + at, vp + j * a.ldv * 2 + u * 16, in ? 16 : 0);
    }
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) {
    if (c_first + s * step < chunks) load(c_first + s * step, s);
    dev::cp_async_commit();
  }
  // Q of the tile: rows g and g + 8 of the lane
  uint32_t qf[D / 16][4];
  RowKeys seen[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int row = tile * 16 + h * 8 + g;
    const int i = row / group, head = kvh * group + row % group;
    seen[h] = RowKeys(a, i + p_off, rq.nk);
    const bool live = row < rows;
    const uint32_t* src =
        reinterpret_cast<const uint32_t*>(static_cast<const T*>(a.q) + (int64_t)(rq.q0 + (live ? i : 0)) * a.ldq +
                                          (live ? head : 0) * D);
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      qf[k][h] = live ? src[k * 8 + t] : 0u;
      qf[k][h + 2] = live ? src[k * 8 + t + 4] : 0u;
    }
  }
  const float scale = a.scale * 1.4426950408889634f;  // scores in log2 units
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  float o[D / 8][4];
#pragma unroll
  for (int n = 0; n < D / 8; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[n][i] = 0.f;

  int it = 0;
  for (int c = c_first; c < chunks; c += step, ++it) {
    {
      const int ahead = c + (STAGES - 1) * step;
      if (ahead < chunks) load(ahead, (it + STAGES - 1) % STAGES);
      dev::cp_async_commit();
    }
    dev::cp_async_wait<STAGES - 1>();
    __syncwarp();
    const uint32_t sk = dev::smem_u32(ring + (it % STAGES) * C::kStage), sv = sk + kChunk * C::kRowBytes;
    int base, end;
    chunk_keys(c, base, end);
    float s[4][4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[n][i] = 0.f;
      const int key = n * 8 + (lane & 7);
#pragma unroll
      for (int k = 0; k < D / 32; ++k) {
        uint32_t b0, b1, b2, b3;
        dev::ldmatrix_x4(sk + key * C::kRowBytes + (((k * 4 + (lane >> 3)) ^ (key & 7)) * 16), b0, b1, b2, b3);
        dev::mma_16816<T>(s[n], qf[2 * k][0], qf[2 * k][1], qf[2 * k][2], qf[2 * k][3], b0, b1);
        dev::mma_16816<T>(s[n], qf[2 * k + 1][0], qf[2 * k + 1][1], qf[2 * k + 1][2], qf[2 * k + 1][3], b2, b3);
      }
    }
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = base + n * 8 + 2 * t + (i & 1);
        s[n][i] = j < end && seen[i >> 1].has(j) ? s[n][i] * scale : -INFINITY;
      }
    float keep[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float mx = m[h];
#pragma unroll
      for (int n = 0; n < 4; ++n) mx = fmaxf(mx, fmaxf(s[n][2 * h], s[n][2 * h + 1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float ref = mx == -INFINITY ? 0.f : mx;  // nothing seen yet: all weights 0
      keep[h] = dev::exp2_approx(m[h] - ref);
      m[h] = mx;
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float w = dev::exp2_approx(s[n][2 * h + i] - ref);
          s[n][2 * h + i] = w;
          sum += w;
        }
      l[h] = l[h] * keep[h] + sum;
    }
#pragma unroll
    for (int n = 0; n < D / 8; ++n) {
      o[n][0] *= keep[0], o[n][1] *= keep[0];
      o[n][2] *= keep[1], o[n][3] *= keep[1];
    }
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const uint32_t p0 = dev::pack2<T>(s[2 * ks][0], s[2 * ks][1]), p1 = dev::pack2<T>(s[2 * ks][2], s[2 * ks][3]);
      const uint32_t p2 = dev::pack2<T>(s[2 * ks + 1][0], s[2 * ks + 1][1]),
                     p3 = dev::pack2<T>(s[2 * ks + 1][2], s[2 * ks + 1][3]);
      const int key = ks * 16 + (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
      for (int n = 0; n < D / 16; ++n) {
        uint32_t b0, b1, b2, b3;
        dev::ldmatrix_x4_trans(sv + key * C::kRowBytes + (((n * 2 + (lane >> 4)) ^ (key & 7)) * 16), b0, b1, b2, b3);
        dev::mma_16816<T>(o[2 * n], p0, p1, p2, p3, b0, b1);
        dev::mma_16816<T>(o[2 * n + 1], p0, p1, p2, p3, b2, b3);
      }
    }
    __syncwarp();  // the stage is free for the next copy
  }
  dev::cp_async_wait<0>();
  __syncthreads();  // the ring becomes the merge buffer

  float* mo = reinterpret_cast<float*>(smem);  // [warp][16][D]
  float* mm = mo + kWarps * 16 * D;            // [warp][16]
  float* ml = mm + kWarps * 16;
  float* bo = reinterpret_cast<float*>(smem + (C::kRing > C::kMerge ? C::kRing : C::kMerge));  // [16][D]
  float* bm = bo + 16 * D;
  float* bl = bm + 16;
  uint32_t* bad = reinterpret_cast<uint32_t*>(bl + 16);  // rows with a result that is not finite
  if (threadIdx.x == 0) *bad = 0;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    if (t == 0) mm[warp * 16 + h * 8 + g] = m[h], ml[warp * 16 + h * 8 + g] = l[h];
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
      *reinterpret_cast<float2*>(mo + (warp * 16 + h * 8 + g) * D + n * 8 + 2 * t) =
          make_float2(o[n][2 * h], o[n][2 * h + 1]);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * D; i += kThreads) {
    const int row = i / D;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, mm[w * 16 + row]);
    const float ref = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = exp2f(mm[w * 16 + row] - ref);
      sum += ml[w * 16 + row] * f;
      acc += mo[w * 16 * D + i] * f;
    }
    bo[i] = acc;
    if (i % D == 0) bm[row] = mx, bl[row] = sum;
  }
  // this rank's columns [d0, d1) of every row
  const int d0 = rank * (D / splits), d1 = d0 + D / splits, width = D / splits;
  if (splits > 1) dev::cluster_sync();
  else __syncthreads();
  for (int i = threadIdx.x; i < 16 * width; i += kThreads) {
    const int row = i / width, col = d0 + i % width;
    const int global_row = tile * 16 + row;
    float acc, sum;
    if (splits > 1) {
      float mx = -INFINITY;
      for (int c = 0; c < splits; ++c) mx = fmaxf(mx, dev::ld_dsmem_f32(dev::mapa(dev::smem_u32(bm + row), c)));
      const float ref = mx == -INFINITY ? 0.f : mx;
      acc = sum = 0.f;
      for (int c = 0; c < splits; ++c) {
        const float f = exp2f(dev::ld_dsmem_f32(dev::mapa(dev::smem_u32(bm + row), c)) - ref);
        sum += dev::ld_dsmem_f32(dev::mapa(dev::smem_u32(bl + row), c)) * f;
        acc += dev::ld_dsmem_f32(dev::mapa(dev::smem_u32(bo + row * D + col), c)) * f;
      }
    } else {
      acc = bo[row * D + col], sum = bl[row];
    }
    if (global_row >= rows) continue;
    const float y = sum == 0.f ? 0.f : acc / sum;
    if (!isfinite(y)) atomicOr(bad, 1u << row);
    const int qi = global_row / group, head = kvh * group + global_row % group;
    static_cast<T*>(a.out)[(int64_t)(rq.q0 + qi) * a.ldo + head * D + col] = dev::from_f32<T>(y);
  }
  if (splits > 1) dev::cluster_sync();  // no block leaves while its partial results are read
  else __syncthreads();
  uint32_t rest = *bad;
  for (int n = 0; rest; ++n, rest &= rest - 1) {
    const int row = __ffs(rest) - 1, global_row = tile * 16 + row;
    if (n % kWarps == warp)
      attention_row<T>(a, rq, global_row / group, kvh * group + global_row % group, d0, d1);
  }
}

template <typename T, int D>
cudaError_t launch_rows(const AttnWindowArgs& a, cudaStream_t s) {
  constexpr int kStages = 3;
  using C = RowsCfg<D, kStages>;
  auto kernel = attention_rows_kernel<T, D, kStages>;
  static bool configured[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev]) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  const int group = a.q_heads / a.kv_heads;
  const int64_t tiles = ((int64_t)a.max_q * group + 15) / 16;
  // keys that a tile's queries see, at most
  int64_t keys = a.max_k;
  if (a.left >= 0) {
    const int64_t window = (int64_t)a.left + (a.right > 0 ? a.right : a.right < 0 ? a.max_k : 0) + 16 + a.sinks;
    if (window < keys) keys = window;
  }
  const int64_t chunks = (keys + kChunk - 1) / kChunk;
  // split the keys while there are fewer blocks than SMs and every warp keeps
  // two chunks
  int splits = 1;
  while (splits < 8 && tiles * a.kv_heads * a.batch * splits * 2 <= 148 && chunks >= splits * 2 * kWarps * 2) splits *= 2;
  const dim3 grid((unsigned)(tiles * splits), a.kv_heads, a.batch);
  return launch_overlapped(kernel, grid, dim3(kThreads), C::kSmem, s, dim3(splits, 1), a, splits, (int)tiles);
}

}  // namespace

cudaError_t launch_attention_rows(const AttnWindowArgs& a, cudaStream_t s) {
  if (a.head_dim == 64)
    return a.dtype == kDtBF16 ? launch_rows<__nv_bfloat16, 64>(a, s) : launch_rows<__half, 64>(a, s);
  return a.dtype == kDtBF16 ? launch_rows<__nv_bfloat16, 128>(a, s) : launch_rows<__half, 128>(a, s);
}

}  // namespace nemo
