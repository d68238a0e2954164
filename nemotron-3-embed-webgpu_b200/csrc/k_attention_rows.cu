// Windowed attention of few query rows (nemo_op_attention_window): single
// tokens, or a few, against a cache.
//
// Bound by memory: each visible K and V row is read once per kv head and meets
// only the query rows of its group. A tile is 16 such rows, (query, head of the
// group) pairs of one kv head, which is what an m16n8k16 instruction takes; a
// 128-row tcgen05 tile would be nearly empty. The keys are split over the 4
// warps of a block and over the blocks of a cluster, each warp running its own
// online softmax over chunks of 16 keys that it copies to shared memory
// itself (no block barriers in the loop); the partial results meet in shared
// memory and, over the cluster, in the shared memory of the block that writes
// their columns, always in the same order. 16 tokens on up to 5000 keys, window
// of 1024 and four sinks, 24 + 8 heads of 128 (f16): 16.4 us, 4.1 TB/s of the
// visible rows. A warp has only two or three chunks there, so the first copies
// and the two merges, not the stream between them, are what is left.
//
// Scores and statistics are f32; weights are rounded to the 16-bit type for
// the product with V (relative error half a step, like the output's own
// rounding).
#include "attention_window.cuh"

namespace nemo {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kChunk = 16;  // keys per copy
constexpr int kMaxSplits = 16;

template <int D, int STAGES>
struct RowsCfg {
  static constexpr int kRowBytes = D * 2;
  static constexpr int kStage = 2 * kChunk * kRowBytes;  // K, then V
  static constexpr int kRing = kWarps * STAGES * kStage;
  // the warps' partial results reuse the ring: [warp][16][D] f32
  static constexpr int kMerge = kWarps * 16 * D * 4;
  static constexpr int kArea = kRing > kMerge ? kRing : kMerge;
  // behind it: reference and sum of [warp][16], then what the cluster's blocks send:
  // of each rank 16 rows of this block's columns, reference and sum of 16 rows
  static constexpr int kStats = 2 * kWarps * 16 * 4;
  static constexpr int kSent = 16 * D * 4 + 2 * kMaxSplits * 16 * 4;
  static constexpr int kSmem = kArea + kStats + kSent + 64;
};

template <typename T, int D, int STAGES>
__global__ void __launch_bounds__(kThreads) attention_rows_kernel(const __grid_constant__ AttnWindowArgs a,
                                                                  int splits) {
  using C = RowsCfg<D, STAGES>;
  extern __shared__ __align__(1024) uint8_t smem[];
  dev::pdl_launch_dependents();
  if (splits > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // this block has started
  dev::pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = blockIdx.x % splits, tile = blockIdx.x / splits;
  const int kvh = blockIdx.y;
  const AttnRequest rq(a, blockIdx.z);
  const int group = a.q_heads / a.kv_heads;
  const int nq = min(rq.nq, a.max_q);
  const int rows = nq * group;  // of this request and kv head
  if (tile * 16 >= rows) {  // the whole cluster
    if (splits > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    return;
  }
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
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};  // m: the references of the weights
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
    float s[kChunk / 8][4];
#pragma unroll
    for (int n = 0; n < kChunk / 8; ++n) {
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
    for (int n = 0; n < kChunk / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = base + n * 8 + 2 * t + (i & 1);
        s[n][i] = j < end && seen[i >> 1].has(j) ? s[n][i] * scale : -INFINITY;
      }
    float keep[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float mx = -INFINITY;
#pragma unroll
      for (int n = 0; n < kChunk / 8; ++n) mx = fmaxf(mx, fmaxf(s[n][2 * h], s[n][2 * h + 1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      mx = fmaxf(m[h], mx - weight_lift<T>());
      const float ref = mx == -INFINITY ? 0.f : mx;  // nothing seen yet: all weights 0
      keep[h] = dev::exp2_approx(m[h] - ref);
      m[h] = mx;
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < kChunk / 8; ++n)
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
    for (int ks = 0; ks < kChunk / 16; ++ks) {
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

  float* mo = reinterpret_cast<float*>(smem);             // [warp][16][D]
  float* mm = reinterpret_cast<float*>(smem + C::kArea);  // [warp][16]
  float* ml = mm + kWarps * 16;
  const int width = D / splits;                           // columns that this block writes
  float* so = ml + kWarps * 16;                           // sent: [rank][16][width]
  float* sm = so + 16 * D;                                // [rank][16]
  float* sl = sm + kMaxSplits * 16;
  uint32_t* bad = reinterpret_cast<uint32_t*>(sl + kMaxSplits * 16);  // rows with a result that is not finite
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
  // Every other block of the cluster runs by now, so its shared memory may be written.
  if (splits > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  // The block's result: a thread has 16 / 4 rows of one column group of four. It
  // goes to the block that writes these columns (reference and sum to all).
  constexpr int kQuads = D / 4, kStep = kThreads / kQuads;
  const int quad = threadIdx.x % kQuads, col = quad * 4, owner = col / width;
  const uint32_t to_o = dev::smem_u32(so) + (rank * 16 * width + col - owner * width) * 4;
#pragma unroll
  for (int i = 0; i < 16 / kStep; ++i) {
    const int row = i * kStep + threadIdx.x / kQuads;
    float mw[kWarps], mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, mw[w] = mm[w * 16 + row]);
    const float ref = mx == -INFINITY ? 0.f : mx;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = dev::exp2_approx(mw[w] - ref);
      const float4 v = *reinterpret_cast<const float4*>(mo + (w * 16 + row) * D + col);
      sum += ml[w * 16 + row] * f;
      acc.x += v.x * f, acc.y += v.y * f, acc.z += v.z * f, acc.w += v.w * f;
    }
    if (splits > 1) {
      const uint32_t at = dev::mapa(to_o + row * width * 4, owner);
      asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(acc.x), "f"(acc.y), "f"(acc.z),
                   "f"(acc.w)
                   : "memory");
      if (quad < splits) {
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dev::mapa(dev::smem_u32(sm + rank * 16 + row), quad)), "f"(mx)
                     : "memory");
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dev::mapa(dev::smem_u32(sl + rank * 16 + row), quad)), "f"(sum)
                     : "memory");
      }
    } else {
      *reinterpret_cast<float4*>(so + row * D + col) = acc;
      if (quad == 0) sm[row] = mx, sl[row] = sum;
    }
  }
  if (splits > 1) dev::cluster_sync();
  else __syncthreads();
  // this rank's columns [d0, d1) of every row, over the ranks in order
  const int d0 = rank * width, d1 = d0 + width;
  for (int i = threadIdx.x; i < 16 * width / 4; i += kThreads) {
    const int row = i / (width / 4), c = i % (width / 4) * 4;
    const int global_row = tile * 16 + row;
    float mx = -INFINITY, sum = 0.f;
    for (int k = 0; k < splits; ++k) mx = fmaxf(mx, sm[k * 16 + row]);
    const float ref = mx == -INFINITY ? 0.f : mx;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < splits; ++k) {
      const float f = dev::exp2_approx(sm[k * 16 + row] - ref);
      const float4 v = *reinterpret_cast<const float4*>(so + (k * 16 + row) * width + c);
      sum += sl[k * 16 + row] * f;
      acc.x += v.x * f, acc.y += v.y * f, acc.z += v.z * f, acc.w += v.w * f;
    }
    if (global_row >= rows) continue;
    if (sum == 0.f) {
      acc = make_float4(0.f, 0.f, 0.f, 0.f);
    } else {
      const float inv = 1.f / sum;
      acc.x *= inv, acc.y *= inv, acc.z *= inv, acc.w *= inv;
    }
    // A mean of finite values is no larger than they are; the rounded weights' product may be, by half a step.
    uint2 y = make_uint2(dev::pack2_finite<T>(acc.x, acc.y), dev::pack2_finite<T>(acc.z, acc.w));
    if (!isfinite(acc.x + acc.y + acc.z + acc.w)) {
      y = make_uint2(dev::pack2<T>(acc.x, acc.y), dev::pack2<T>(acc.z, acc.w));
      if (isfinite(sum)) atomicOr(bad, 1u << row);  // (otherwise a score is not: the row is NaN)
    }
    const int qi = global_row / group, head = kvh * group + global_row % group;
    *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (int64_t)(rq.q0 + qi) * a.ldo + head * D + d0 + c) = y;
  }
  __syncthreads();
  uint32_t rest = *bad;
  for (int n = 0; rest; ++n, rest &= rest - 1) {
    const int row = __ffs(rest) - 1, global_row = tile * 16 + row;
    if (n % kWarps == warp)
      attention_row<T, D>(a, rq, global_row / group, kvh * group + global_row % group, d0, d1);
  }
}

// 16-row tiles of a request and kv head.
int64_t row_tiles(const AttnWindowArgs& a) { return ((int64_t)a.max_q * (a.q_heads / a.kv_heads) + 15) / 16; }

// Largest cluster of the kernel that the current device can place: 16 blocks are
// more than is portable, and a partition of a GPU may have no room for them.
template <typename K>
cudaError_t largest_cluster(K* kernel, size_t smem, int* blocks) {
  for (*blocks = kMaxSplits; *blocks > 1; *blocks /= 2) {
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = *blocks, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(*blocks), cfg.blockDim = dim3(kThreads), cfg.dynamicSmemBytes = smem;
    cfg.attrs = &attr, cfg.numAttrs = 1;
    int clusters = 0;
    const cudaError_t e = cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg);
    if (e == cudaSuccess && clusters > 0) break;
    if (e != cudaSuccess && e != cudaErrorInvalidClusterSize) return e;
    cudaGetLastError();
  }
  return cudaSuccess;
}

template <typename T, int D>
cudaError_t launch_rows(const AttnWindowArgs& a, cudaStream_t s) {
  constexpr int kStages = 3;
  using C = RowsCfg<D, kStages>;
  auto kernel = attention_rows_kernel<T, D, kStages>;
  static int max_splits[64] = {};  // 0: the kernel is not set up on that device yet
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64) return cudaErrorInvalidDevice;
  if (!max_splits[dev]) {
    int blocks = 1;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess) e = largest_cluster(kernel, C::kSmem, &blocks);
    if (e != cudaSuccess) return e;
    max_splits[dev] = blocks;
  }
  const int splits = attention_splits(a, max_splits[dev]);
  const dim3 grid((unsigned)(row_tiles(a) * splits), a.kv_heads, a.batch);
  return launch_overlapped(kernel, grid, dim3(kThreads), C::kSmem, s, dim3(splits, 1), a, splits);
}

}  // namespace

int attention_splits(const AttnWindowArgs& a, int max_splits) {
  const int64_t keys = visible_keys(a, 16);
  const int64_t chunks = (keys + kChunk - 1) / kChunk;
  // Split the keys over a cluster while two blocks an SM are not reached and
  // every warp keeps two chunks (16 tokens on 1028 keys: 16.3 us with two blocks
  // a tile, 24.9 with one); beyond that, up to eight, while it keeps 32, which
  // levels ragged lengths (16 tokens on up to 32768 keys: 193 us, 256 without).
  int splits = 1;
  const int64_t blocks = row_tiles(a) * a.kv_heads * a.batch, sms = a.sms;
  if (max_splits > kMaxSplits) max_splits = kMaxSplits;
  while (splits * 2 <= max_splits && chunks >= splits * 2 * kWarps * 2 &&
         (blocks * splits * 2 <= 2 * sms || (blocks * splits * 2 <= 8 * sms && chunks >= splits * 2 * kWarps * 32)))
    splits *= 2;
  return splits;
}

cudaError_t launch_attention_rows(const AttnWindowArgs& a, cudaStream_t s) {
  if (a.head_dim == 64)
    return a.dtype == kDtBF16 ? launch_rows<__nv_bfloat16, 64>(a, s) : launch_rows<__half, 64>(a, s);
  return a.dtype == kDtBF16 ? launch_rows<__nv_bfloat16, 128>(a, s) : launch_rows<__half, 128>(a, s);
}

}  // namespace nemo
