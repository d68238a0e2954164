// Residual RMSNorm with an 8-bit output (nemo_op_rmsnorm_q8).
//
// For a row s = x + r the normalised value is y = s * w * inv with one factor
// inv = 1 / sqrt(mean s^2 + eps) per row. A group's scale is max|y| / Q and its
// codes are y / scale = u * (Q / max|u|) with u = s * w: inv falls out, so the
// codes need the group's maximum only, and each is the product of two f32
// values whatever the order in which the row's sum is formed.
//
// Bound by memory: x, r in, sum and codes out, 7 bytes per element with a
// residual and 3 without; the row stays in registers between its one read and
// the writes. wpr warps share a row, NV 8-column vectors per thread. With a
// dozen scalar operations per element the kernel was bound by instructions (89
// us at 24000 x 2048, bf16 to e4m3); packed f32 pairs, maxima of three and one
// division per group brought it to 57, 93 % of the copy rate.
#include "layer_ops.cuh"

namespace nemo {
namespace {

constexpr uint32_t kInfBits = 0x7f800000u;
constexpr float kTinyTop = 1e-30f;  // groups no larger than this have codes 0: Q / top would overflow

// Up to 8 consecutive elements of a row of n left; elements past them are 0.
template <typename T, bool VEC>
__device__ __forceinline__ uint4 load8(const T* p, int n) {
  if constexpr (VEC) {
    return *reinterpret_cast<const uint4*>(p);
  } else {
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint16_t* h = reinterpret_cast<const uint16_t*>(p) + 2 * i;
      v[i] = (2 * i < n ? h[0] : 0u) | (2 * i + 1 < n ? (uint32_t)h[1] << 16 : 0u);
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
  }
}

template <typename T>
__device__ __forceinline__ void unpack_pairs(const uint4& u, float2 (&v)[4]) {
  v[0] = dev::unpack2<T>(u.x), v[1] = dev::unpack2<T>(u.y), v[2] = dev::unpack2<T>(u.z), v[3] = dev::unpack2<T>(u.w);
}

template <typename T, int OUT, int NV, bool VEC, int THREADS>
__global__ void __launch_bounds__(THREADS) rmsnorm_q8_kernel(const __grid_constant__ NormQ8Args a, int wpr) {
  __shared__ float red_ss[32];
  __shared__ uint32_t red_top[32];
  constexpr float kQ = OUT == kDtE4M3 ? 448.f : 127.f;
  dev::pdl_launch_dependents();
  dev::pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slot = warp / wpr, part = warp % wpr;  // the row of the block, the warp's part of it
  const int64_t row = (int64_t)blockIdx.x * ((blockDim.x >> 5) / wpr) + slot;
  const bool live = row < a.rows;
  const T* x = static_cast<const T*>(a.x) + row * a.ldx;
  const T* r = static_cast<const T*>(a.residual) + row * a.ldr;
  T* sum = static_cast<T*>(a.sum) + row * a.lds;
  // every load of the row first
  uint4 xv[NV], rv[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = ((v * wpr + part) * 32 + lane) * 8;
    xv[v] = rv[v] = make_uint4(0, 0, 0, 0);
    if (live && c < a.width) {
      xv[v] = load8<T, VEC>(x + c, a.width - c);
      if (a.residual) rv[v] = load8<T, VEC>(r + c, a.width - c);
    }
  }
  float2 u[NV][4];
  float top[NV], row_top = 0.f;  // largest |u| of the vector, of the thread; NaN where one is
  float2 ss2 = make_float2(0.f, 0.f);
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = ((v * wpr + part) * 32 + lane) * 8;
    unpack_pairs<T>(xv[v], u[v]);
    top[v] = 0.f;
    if (live && c < a.width) {
      if (a.residual) {
        float2 f[4];
        unpack_pairs<T>(rv[v], f);
#pragma unroll
        for (int i = 0; i < 4; ++i) u[v][i] = dev::add2(u[v][i], f[i]);
        const uint4 o = make_uint4(dev::pack2<T>(u[v][0].x, u[v][0].y), dev::pack2<T>(u[v][1].x, u[v][1].y),
                                   dev::pack2<T>(u[v][2].x, u[v][2].y), dev::pack2<T>(u[v][3].x, u[v][3].y));
        if (VEC) {
          *reinterpret_cast<uint4*>(sum + c) = o;
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (c + i < a.width) sum[c + i] = dev::from_f32<T>(i & 1 ? u[v][i / 2].y : u[v][i / 2].x);
        }
      }
      float2 w[4];
      if (VEC) {
        const float4 w0 = __ldg(reinterpret_cast<const float4*>(a.w + c));
        const float4 w1 = __ldg(reinterpret_cast<const float4*>(a.w + c) + 1);
        w[0] = make_float2(w0.x, w0.y), w[1] = make_float2(w0.z, w0.w);
        w[2] = make_float2(w1.x, w1.y), w[3] = make_float2(w1.z, w1.w);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i] = make_float2(c + 2 * i < a.width ? a.w[c + 2 * i] : 0.f, c + 2 * i + 1 < a.width ? a.w[c + 2 * i + 1] : 0.f);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ss2 = dev::fma2(u[v][i], u[v][i], ss2);
        u[v][i] = dev::mul2(u[v][i], w[i]);
        top[v] = dev::max3_abs_nan(top[v], u[v][i].x, u[v][i].y);
      }
      row_top = dev::max3_abs_nan(row_top, top[v], 0.f);
    }
  }
  float ss = ss2.x + ss2.y;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  // as integers magnitudes compare like floats, with NaN above infinity
  uint32_t row_bits = 0;
  if (a.group == 0) row_bits = __reduce_max_sync(0xffffffffu, __float_as_uint(row_top));
  if (wpr > 1) {
    if (lane == 0) red_ss[warp] = ss, red_top[warp] = row_bits;
    __syncthreads();
    // every warp of the row sums its parts in the same order
    ss = 0.f, row_bits = 0;
    for (int i = 0; i < wpr; ++i) {
      ss += red_ss[slot * wpr + i];
      row_bits = max(row_bits, red_top[slot * wpr + i]);
    }
  }
  const float inv = rsqrtf(__fadd_rn(__fdiv_rn(ss, (float)a.width), a.eps));
  uint32_t bits[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    bits[v] = row_bits;
    if (a.group) {
      uint32_t t = __float_as_uint(top[v]);
      t = max(t, __shfl_xor_sync(0xffffffffu, t, 1));
      t = max(t, __shfl_xor_sync(0xffffffffu, t, 2));
      if (a.group >= 64) t = max(t, __shfl_xor_sync(0xffffffffu, t, 4));
      if (a.group >= 128) t = max(t, __shfl_xor_sync(0xffffffffu, t, 8));
      bits[v] = t;
    }
  }
  // The two divisions of a group are made once: lane v of each four (a group
  // has four lanes or more) makes those of vector v and stores its scale.
  uint32_t t = bits[0];
  int vec = 0;
#pragma unroll
  for (int v = 1; v < NV; ++v)
    if ((lane & 3) == v) t = bits[v], vec = v;
  const float tf = __uint_as_float(t);
  const float to_mine = t < kInfBits && tf > kTinyTop ? __fdiv_rn(kQ, tf) : 0.f;
  if (live) {
    const int c = ((vec * wpr + part) * 32 + (lane & ~3)) * 8;  // of the four lanes' first column
    const bool first = a.group ? c % a.group == 0 : c == 0;
    if (first && (lane & 3) == vec && c < a.width)
      a.scales[row * a.groups + (a.group ? c / a.group : 0)] =
          t < kInfBits ? __fdiv_rn(tf > kTinyTop ? tf * inv : 0.f, kQ) : __uint_as_float(0x7fc00000u);
  }
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const float to = NV == 1 ? to_mine : __shfl_sync(0xffffffffu, to_mine, (lane & ~3) + v);
    const int c = ((v * wpr + part) * 32 + lane) * 8;
    if (!live || c >= a.width) continue;
    uint2 code;
    if (bits[v] < kInfBits) {
      float2 p[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] = dev::mul2(u[v][i], make_float2(to, to));
      if (OUT == kDtE4M3) {
        uint32_t h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __nv_cvt_float2_to_fp8x2(p[i], __NV_SATFINITE, __NV_E4M3);
        code = make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
      } else {
        // |p| <= 127: adding 1.5 * 2^23 rounds to a whole number, in the low byte
        // (a scalar addition: the packed one may be merged with the product)
        uint32_t h[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          h[2 * i] = __float_as_uint(__fadd_rn(p[i].x, 12582912.f));
          h[2 * i + 1] = __float_as_uint(__fadd_rn(p[i].y, 12582912.f));
        }
        code.x = __byte_perm(__byte_perm(h[0], h[1], 0x0040), __byte_perm(h[2], h[3], 0x0040), 0x5410);
        code.y = __byte_perm(__byte_perm(h[4], h[5], 0x0040), __byte_perm(h[6], h[7], 0x0040), 0x5410);
      }
    } else {
      code = make_uint2(0, 0);  // an infinity or NaN in the group, whose scale is NaN
    }
    uint8_t* q = static_cast<uint8_t*>(a.q) + row * a.ldq + c;
    if (VEC) {
      *reinterpret_cast<uint2*>(q) = code;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i < a.width) q[i] = (uint8_t)((i < 4 ? code.x : code.y) >> (i & 3) * 8);
    }
  }
}

template <typename T, int OUT, bool VEC>
cudaError_t launch_nv(const NormQ8Args& a, int nv, int wpr, dim3 grid, int threads, cudaStream_t s) {
  auto kernel = nv == 1   ? rmsnorm_q8_kernel<T, OUT, 1, VEC, 512>
                : nv == 2 ? rmsnorm_q8_kernel<T, OUT, 2, VEC, 512>
                          : rmsnorm_q8_kernel<T, OUT, 4, VEC, 1024>;
  return launch_overlapped(kernel, grid, dim3(threads), 0, s, dim3(1, 1), a, wpr);
}

}  // namespace

cudaError_t launch_rmsnorm_q8(const NormQ8Args& a, cudaStream_t s) {
  auto aligned = [](const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; };
  const bool vec = a.width % 8 == 0 && a.ldx % 8 == 0 && aligned(a.x, 16) && aligned(a.w, 16) && a.ldq % 8 == 0 &&
                   aligned(a.q, 8) &&
                   (!a.residual || (a.ldr % 8 == 0 && a.lds % 8 == 0 && aligned(a.residual, 16) && aligned(a.sum, 16)));
  const int vectors = (a.width + 7) / 8;
  if (vectors > 4096) return cudaErrorInvalidValue;  // more than 32768 columns
  // Vectors per thread. Few rows: one, the shortest chain of instructions (one
  // row of 2048: 2.0 us with one, 3.0 with four; 240 rows 3.2 and 3.6). Rows that
  // fit a warp: as many as that takes, so that no block barrier is needed (4000
  // rows of 1000: 5.7 us in one warp, 7.4 in two). Otherwise two, which keeps
  // enough rows in flight (2400 rows of 2048: 9.0 us, 10.2 with four, 10.9 with
  // one), and four where the grid is many waves and fewer instructions count
  // (24000 rows: 58 us with four, 61 with two, 84 with one).
  const int64_t total = (int64_t)a.rows * vectors;
  int nv = total <= a.sms * 256 ? 1 : vectors <= 128 ? (vectors <= 32 ? 1 : vectors <= 64 ? 2 : 4) : total < 4000000 ? 2 : 4;
  while (vectors > nv * (nv == 4 ? 1024 : 512)) nv *= 2;
  const int wpr = (vectors + 32 * nv - 1) / (32 * nv);
  const int rows_per_block = wpr >= 4 ? 1 : 4 / wpr;
  const int warps = rows_per_block * wpr;
  const dim3 grid((unsigned)((a.rows + rows_per_block - 1) / rows_per_block));
  const bool e4m3 = a.out_dtype == kDtE4M3;
#define NEMO_NORM(T)                                                                            \
  (vec ? (e4m3 ? launch_nv<T, kDtE4M3, true>(a, nv, wpr, grid, warps * 32, s)                   \
               : launch_nv<T, kDtI8, true>(a, nv, wpr, grid, warps * 32, s))                    \
       : (e4m3 ? launch_nv<T, kDtE4M3, false>(a, nv, wpr, grid, warps * 32, s)                  \
               : launch_nv<T, kDtI8, false>(a, nv, wpr, grid, warps * 32, s)))
  return a.dtype == kDtBF16 ? NEMO_NORM(__nv_bfloat16) : NEMO_NORM(__half);
#undef NEMO_NORM
}

}  // namespace nemo
