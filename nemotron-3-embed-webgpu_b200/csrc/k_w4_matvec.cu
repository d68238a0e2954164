// Matrix-vector products with 4-bit weights and group scales, 1 to 16 rows of
// x at once (nemo_op_w4_matvec).
//
//   y[m][r] = sum_g s[r][g] * ( sum_{c in g} x[m][c] * (q[r][c] - z[r][g]) )
//
// The inner sum runs on m16n8k16 tensor-core instructions: A = 16 weight rows
// as the exact small integers q - z in the type of x, B = up to 8 rows of x,
// f32 accumulation; each segment's sum is then scaled in f32. Nothing is
// rounded before y. (The 128-row tcgen05 tile would hold 16 rows of x against
// 128 of weights, but its operand would have to be written to shared or tensor
// memory; here the decoded integers go from registers straight into the
// instruction, and the bound is the stream of weights, not the tensor rate.)
//
// A segment is the shorter of the weight group and the group of x scales (32,
// 64 or 128 columns). A lane takes SEG/32 consecutive 32-bit words of a row per
// segment: the columns that an instruction's k index stands for are permuted,
// in the same way for the weights and for x, so that each lane reads its
// weights as one vector and each word's nibble pairs (k, k + 4) come out of
// one mask; x is stored in shared memory in that order once per block.
//
// One block owns 16 R rows and a panel of columns; its 8 warps divide the
// panel, each with its own asynchronous copies, so weights flow without block
// barriers. Panels of one row tile are blocks of one cluster, summed in rank
// order through distributed shared memory.
#include "layer_ops.cuh"

namespace nemo {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr size_t kSmemLimit = 227 * 1024;

struct W4Plan {
  W4Args a;
  int segs;         // segments of a row
  int panel_segs;   // segments of a block's panel
  int warp_segs;    // segments of a warp's slice of the panel (panel_segs / 8 rounded up)
  int panels;       // panels of a row
  int splits;       // blocks per row tile (cluster size)
  int mp;           // rows of x in shared memory: m rounded up to 1, 2, 4, 8 or 16
  int w_pitch;      // bytes between weight rows of a warp's slice in shared memory
  int off_x, off_s, off_xs, off_red;  // byte offsets in shared memory (weights at 0)
};

// The integers q - z of one 32-bit word as four pairs: (k, k+4), (k+1, k+5),
// (k+2, k+6), (k+3, k+7). zc = the pair (1024 + z) in f16, (128 + z) in bf16: a
// nibble masked under the exponent whose unit is 1 is that base plus q.
template <typename T>
struct Nibbles;
template <>
struct Nibbles<__half> {
  static constexpr float kBase = 1024.f;
  __device__ static __forceinline__ void decode(uint32_t w, uint32_t zc, uint32_t (&p)[4]) {
    const __half2 z = *reinterpret_cast<const __half2*>(&zc);
    // high nibbles sit four bits up: 1024 + 16 q, times 1/16 = 64 + q; 64 + z = (1024 + z) - 960
    const __half2 zh = __hsub2(__floats2half2_rn(960.f, 960.f), z);  // -(64 + z)
    const __half2 sixteenth = __floats2half2_rn(0.0625f, 0.0625f);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t lo = (w & 0x000f000fu) | 0x64006400u, hi = (w & 0x00f000f0u) | 0x64006400u;
      const __half2 a = __hsub2(*reinterpret_cast<const __half2*>(&lo), z);
      const __half2 b = __hfma2(*reinterpret_cast<const __half2*>(&hi), sixteenth, zh);
      p[2 * i] = *reinterpret_cast<const uint32_t*>(&a);
      p[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&b);
      w >>= 8;
    }
  }
};
template <>
struct Nibbles<__nv_bfloat16> {
  static constexpr float kBase = 128.f;
  __device__ static __forceinline__ void decode(uint32_t w, uint32_t zc, uint32_t (&p)[4]) {
    const __nv_bfloat162 z = *reinterpret_cast<const __nv_bfloat162*>(&zc);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t v = (w & 0x000f000fu) | 0x43004300u;
      const __nv_bfloat162 a = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), z);
      p[i] = *reinterpret_cast<const uint32_t*>(&a);
      w >>= 4;
    }
  }
};

// One element of x as f32 (8-bit codes without their scale).
__device__ __forceinline__ float load_x(const void* x, int dtype, int64_t i) {
  if (dtype == kDtF16) return __half2float(static_cast<const __half*>(x)[i]);
  if (dtype == kDtBF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(x)[i]);
  if (dtype == kDtI8) return (float)static_cast<const int8_t*>(x)[i];
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<const uint8_t*>(x)[i], __NV_E4M3)));
}

template <int N>
__device__ __forceinline__ void lds_words(const uint8_t* p, uint32_t (&w)[N]) {
  if (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1 % N] = v.y, w[2 % N] = v.z, w[3 % N] = v.w;
  } else if (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1 % N] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// T: type of the products (f16 also for 8-bit x, whose codes it holds
// exactly). R: 16-row tiles per block. NT: 8-row tiles of x. XG: x scales per
// group.
template <typename T, int SEG, int R, int NT, bool XG>
__global__ void __launch_bounds__(kThreads) w4_matvec_kernel(const __grid_constant__ W4Plan p) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int WPL = SEG / 32;  // words of a row per lane and segment
  constexpr int ROWS = 16 * R;
  const W4Args& a = p.a;
  dev::pdl_launch_dependents();
  dev::pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int row0 = blockIdx.x * ROWS, rank = blockIdx.y;
  const int seg_bytes = SEG / 2;
  uint8_t* sw = smem + (size_t)warp * ROWS * p.w_pitch;
  uint8_t* sx = smem + p.off_x;
  uint32_t* ss = reinterpret_cast<uint32_t*>(smem + p.off_s);
  float* sxs = reinterpret_cast<float*>(smem + p.off_xs);
  float* red = reinterpret_cast<float*>(smem + p.off_red);
  const int64_t row_bytes = a.k / 2;
  const int groups = a.k / a.group, seg_per_group = a.group / SEG;
  const int zero_bytes = (groups + 1) / 2;
  const int x_groups = (a.k + a.x_group - 1) / a.x_group;

  float acc[R][NT][4];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[r][n][i] = 0.f;

  for (int panel = rank; panel < p.panels; panel += p.splits) {
    const int seg0 = panel * p.panel_segs;
    const int nseg = min(p.panel_segs, p.segs - seg0);  // of the panel
    const int ws0 = warp * p.warp_segs;                 // the warp's first segment in the panel
    const int wn = max(0, min(p.warp_segs, nseg - ws0));
    // the warp's weights: rows past n repeat the last one (their sums are not stored)
    const int units = wn * seg_bytes / 16;
    for (int u0 = 0; u0 < units; u0 += 8) {
      const int u = u0 + (lane & 7);
#pragma unroll
      for (int i = 0; i < ROWS / 4; ++i) {
        const int row = i * 4 + (lane >> 3);
        if (u < units)
          dev::cp_async16(dev::smem_u32(sw + row * p.w_pitch + u * 16),
                          a.w + (int64_t)min(row0 + row, a.n - 1) * row_bytes + (int64_t)(seg0 + ws0) * seg_bytes + u * 16);
      }
    }
    dev::cp_async_commit();
    // x in the order of the instructions: for each 32-column step of a segment,
    // row and lane t, the 8 columns of that lane's word, paired (k, k + 4)
    for (int m = 0; m < p.mp; ++m)
      for (int u = threadIdx.x; u < nseg * (SEG / 8); u += kThreads) {
        const int seg = u / (SEG / 8), rem = u % (SEG / 8);
        const int64_t at = m * a.ldx + (int64_t)(seg0 + seg) * SEG + rem * 8;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = m < a.m ? load_x(a.x, a.x_dtype, at + i) : 0.f;
        uint4 o;
        o.x = dev::pack2<T>(v[0], v[4]);
        o.y = dev::pack2<T>(v[1], v[5]);
        o.z = dev::pack2<T>(v[2], v[6]);
        o.w = dev::pack2<T>(v[3], v[7]);
        const int step = seg * WPL + rem % WPL, l = rem / WPL;
        *reinterpret_cast<uint4*>(sx + ((step * p.mp + m) * 4 + l) * 16) = o;
      }
    // scale (low half, as stored) and zero constant (high half) of each group and row
    const int g0 = seg0 / seg_per_group, ng = (nseg + seg_per_group - 1) / seg_per_group;
    for (int i = threadIdx.x; i < ng * ROWS; i += kThreads) {
      const int row = i / ng, gr = i - row * ng;
      const int64_t r = min(row0 + row, a.n - 1);
      float z = 8.f;
      if (a.zeros) z = (float)((a.zeros[r * zero_bytes + (g0 + gr) / 2] >> (((g0 + gr) & 1) * 4)) & 15);
      const uint32_t zc = dev::pack2<T>(0.f, Nibbles<T>::kBase + z);
      ss[gr * ROWS + row] = zc | a.scales[r * groups + g0 + gr];
    }
    if (XG)
      for (int i = threadIdx.x; i < nseg * p.mp; i += kThreads) {
        const int m = i % p.mp, seg = i / p.mp;
        sxs[i] = m < a.m ? a.x_scales[(int64_t)m * x_groups + (seg0 + seg) * SEG / a.x_group] : 0.f;
      }
    dev::cp_async_wait<0>();
    __syncthreads();

    for (int s = 0; s < wn; ++s) {
      const int seg = ws0 + s, gr = seg / seg_per_group;
      uint32_t w[R][2][WPL], zc[R][2];
      float sc[R][2];
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = r * 16 + h * 8 + g;
          lds_words<WPL>(sw + row * p.w_pitch + s * seg_bytes + t * WPL * 4, w[r][h]);
          const uint32_t v = ss[gr * ROWS + row];
          zc[r][h] = __byte_perm(v, v, 0x3232);
          const uint16_t bits = (uint16_t)v;
          sc[r][h] = a.scale_dtype == kDtBF16 ? __uint_as_float(v << 16)
                                              : __half2float(*reinterpret_cast<const __half*>(&bits));
        }
      float part[R][NT][4];
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) part[r][n][i] = 0.f;
#pragma unroll
      for (int j = 0; j < WPL; ++j) {
        uint4 b[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          b[n] = make_uint4(0, 0, 0, 0);
          if (n * 8 + g < p.mp)
            b[n] = *reinterpret_cast<const uint4*>(sx + (((seg * WPL + j) * p.mp + n * 8 + g) * 4 + t) * 16);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          uint32_t lo[4], hi[4];
          Nibbles<T>::decode(w[r][0][j], zc[r][0], lo);
          Nibbles<T>::decode(w[r][1][j], zc[r][1], hi);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            dev::mma_16816<T>(part[r][n], lo[0], hi[0], lo[1], hi[1], b[n].x, b[n].y);
            dev::mma_16816<T>(part[r][n], lo[2], hi[2], lo[3], hi[3], b[n].z, b[n].w);
          }
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float f0 = 1.f, f1 = 1.f;  // x scales of the lane's two rows of x
        if (XG) {
          const int m = n * 8 + 2 * t;
          f0 = m < p.mp ? sxs[seg * p.mp + m] : 0.f;
          f1 = m + 1 < p.mp ? sxs[seg * p.mp + m + 1] : 0.f;
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          acc[r][n][0] = fmaf(part[r][n][0], XG ? sc[r][0] * f0 : sc[r][0], acc[r][n][0]);
          acc[r][n][1] = fmaf(part[r][n][1], XG ? sc[r][0] * f1 : sc[r][0], acc[r][n][1]);
          acc[r][n][2] = fmaf(part[r][n][2], XG ? sc[r][1] * f0 : sc[r][1], acc[r][n][2]);
          acc[r][n][3] = fmaf(part[r][n][3], XG ? sc[r][1] * f1 : sc[r][1], acc[r][n][3]);
        }
      }
    }
    __syncthreads();  // before the next panel overwrites shared memory
  }

  // sums over the warps, then over the cluster's panels, both in order
  constexpr int COLS = 8 * NT;
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        red[(warp * COLS + n * 8 + 2 * t + (i & 1)) * ROWS + r * 16 + (i >> 1) * 8 + g] = acc[r][n][i];
  __syncthreads();
  float* total = red;  // [COLS][ROWS], over warp 0's part
  constexpr int kEach = (COLS * ROWS + kThreads - 1) / kThreads;
  float v[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = e * kThreads + threadIdx.x;
    v[e] = 0.f;
    if (i < a.m * ROWS)
      for (int w = 0; w < kWarps; ++w) v[e] += red[w * COLS * ROWS + i];
  }
  if (p.splits > 1) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int i = e * kThreads + threadIdx.x;
      if (i < a.m * ROWS) total[i] = v[e];
    }
    dev::cluster_sync();
    if (rank == 0) {
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const int i = e * kThreads + threadIdx.x;
        if (i < a.m * ROWS)
          for (int c = 1; c < p.splits; ++c) v[e] += dev::ld_dsmem_f32(dev::mapa(dev::smem_u32(total + i), c));
      }
    }
    dev::cluster_sync();  // no block leaves while its sums are read
    if (rank) return;
  }
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = e * kThreads + threadIdx.x;
    const int m = i / ROWS, row = row0 + i % ROWS;
    if (i >= a.m * ROWS || row >= a.n) continue;
    const float y = !XG && a.x_scales ? v[e] * a.x_scales[m] : v[e];
    const int64_t at = m * a.ldy + row;
    if (a.y_dtype == kDtF32) static_cast<float*>(a.y)[at] = y;
    else if (a.y_dtype == kDtBF16) static_cast<__nv_bfloat16*>(a.y)[at] = __float2bfloat16_rn(y);
    else static_cast<__half*>(a.y)[at] = __float2half_rn(y);
  }
}

template <typename T, int SEG, int R, int NT, bool XG>
cudaError_t launch_kernel(const W4Plan& p, size_t smem, cudaStream_t s) {
  auto kernel = w4_matvec_kernel<T, SEG, R, NT, XG>;
  static bool configured[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev]) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemLimit);
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  const dim3 grid((unsigned)((p.a.n + 16 * R - 1) / (16 * R)), (unsigned)p.splits);
  return launch_overlapped(kernel, grid, dim3(kThreads), smem, s, dim3(1, p.splits), p);
}

template <typename T, int SEG, int R>
cudaError_t launch_r(const W4Plan& p, bool xg, size_t smem, cudaStream_t s) {
  if (p.mp <= 8)
    return xg ? launch_kernel<T, SEG, R, 1, true>(p, smem, s) : launch_kernel<T, SEG, R, 1, false>(p, smem, s);
  return xg ? launch_kernel<T, SEG, R, 2, true>(p, smem, s) : launch_kernel<T, SEG, R, 2, false>(p, smem, s);
}

template <typename T>
cudaError_t launch_seg(const W4Plan& p, int seg, int r, bool xg, size_t smem, cudaStream_t s) {
#define NEMO_W4(SEG) \
  (r == 1 ? launch_r<T, SEG, 1>(p, xg, smem, s) : launch_r<T, SEG, 2>(p, xg, smem, s))
  return seg == 128 ? NEMO_W4(128) : seg == 64 ? NEMO_W4(64) : NEMO_W4(32);
#undef NEMO_W4
}

}  // namespace

cudaError_t launch_w4_matvec(const W4Args& a, cudaStream_t s) {
  W4Plan p = {};
  p.a = a;
  const bool xg = a.x_scales && a.x_group < a.k;
  if (!a.x_scales || !xg) p.a.x_group = a.k;
  const int seg = xg && a.x_group < a.group ? a.x_group : a.group;
  p.segs = a.k / seg;
  p.mp = a.m <= 1 ? 1 : a.m <= 2 ? 2 : a.m <= 4 ? 4 : a.m <= 8 ? 8 : 16;
  const int nt = p.mp == 16 ? 2 : 1;
  const int r = a.n >= 32 * 148 ? 2 : 1;
  const int rows = 16 * r;
  // A panel's weights and rows of x take at most 64 KB of shared memory each;
  // a multiple of the weight group, so that no group is split.
  int panel_k = 64 * 1024 * 2 / rows;
  if (panel_k > 64 * 1024 / 2 / p.mp) panel_k = 64 * 1024 / 2 / p.mp;
  panel_k = panel_k < a.k ? panel_k / a.group * a.group : a.k;
  p.panels = (a.k + panel_k - 1) / panel_k;
  p.splits = p.panels < 8 ? p.panels : 8;
  panel_k = ((a.k + p.panels - 1) / p.panels + a.group - 1) / a.group * a.group;  // panels of one length
  p.panels = (a.k + panel_k - 1) / panel_k;
  p.splits = p.panels < p.splits ? p.panels : p.splits;
  p.panel_segs = panel_k / seg;
  p.warp_segs = (p.panel_segs + kWarps - 1) / kWarps;
  const int slice = p.warp_segs * seg / 2;
  p.w_pitch = (slice + 127) / 128 * 128 + 16 * (seg / 32);
  size_t off = (size_t)kWarps * rows * p.w_pitch;
  p.off_x = (int)off;
  off += (size_t)p.mp * panel_k * 2;
  p.off_s = (int)off;
  off += (size_t)(panel_k / a.group) * rows * 4;
  p.off_xs = (int)off;
  if (xg) off += (size_t)p.panel_segs * p.mp * 4;
  p.off_red = (int)((off + 15) / 16 * 16);
  off = p.off_red + (size_t)kWarps * 8 * nt * rows * 4;
  if (off > kSmemLimit) return cudaErrorInvalidValue;
  return a.x_dtype == kDtBF16 ? launch_seg<__nv_bfloat16>(p, seg, r, xg, off, s) : launch_seg<__half>(p, seg, r, xg, off, s);
}

}  // namespace nemo
