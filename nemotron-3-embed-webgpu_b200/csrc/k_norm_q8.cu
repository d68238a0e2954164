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
// the writes. W warps (a power of two) share a row, NV 8-column vectors per
// thread.
#include "layer_ops.cuh"

namespace nemo {
namespace {

constexpr uint32_t kInfBits = 0x7f800000u;
constexpr float kTinyTop = 1e-30f;  // groups no larger than this have codes 0: Q / top would overflow

// Up to 8 consecutive elements of a row of n left; elements past them are 0.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int n, float (&v)[8]) {
  if (VEC) {
    dev::unpack8<T>(*reinterpret_cast<const uint4*>(p), v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? dev::to_f32(p[i]) : 0.f;
  }
}

template <typename T, int OUT, int NV, bool VEC>
__global__ void __launch_bounds__(1024) rmsnorm_q8_kernel(const __grid_constant__ NormQ8Args a, int wpr) {
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
  float u[NV][8];
  uint32_t top[NV];
  float ss = 0.f;
  uint32_t row_top = 0;
  // every load of the row first
  float rr[NV][8];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = ((v * wpr + part) * 32 + lane) * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) u[v][i] = rr[v][i] = 0.f;
    if (live && c < a.width) {
      load8<T, VEC>(x + c, a.width - c, u[v]);
      if (a.residual) load8<T, VEC>(r + c, a.width - c, rr[v]);
    }
  }
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = ((v * wpr + part) * 32 + lane) * 8;
    top[v] = 0;
    if (live && c < a.width) {
      if (a.residual) {
#pragma unroll
        for (int i = 0; i < 8; ++i) u[v][i] = __fadd_rn(u[v][i], rr[v][i]);
        if (VEC) {
          *reinterpret_cast<uint4*>(sum + c) = dev::pack8<T>(u[v]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (c + i < a.width) sum[c + i] = dev::from_f32<T>(u[v][i]);
        }
      }
      float w[8];
      if (VEC) {
        const float4 w0 = __ldg(reinterpret_cast<const float4*>(a.w + c));
        const float4 w1 = __ldg(reinterpret_cast<const float4*>(a.w + c) + 1);
        w[0] = w0.x, w[1] = w0.y, w[2] = w0.z, w[3] = w0.w, w[4] = w1.x, w[5] = w1.y, w[6] = w1.z, w[7] = w1.w;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = c + i < a.width ? a.w[c + i] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        ss = fmaf(u[v][i], u[v][i], ss);
        u[v][i] = __fmul_rn(u[v][i], w[i]);
        // as integers |u| compare like floats, with NaN above infinity
        top[v] = max(top[v], __float_as_uint(u[v][i]) & 0x7fffffffu);
      }
      row_top = max(row_top, top[v]);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (a.group == 0) row_top = __reduce_max_sync(0xffffffffu, row_top);
  if (wpr > 1) {
    if (lane == 0) red_ss[warp] = ss, red_top[warp] = row_top;
    __syncthreads();
    // every warp of the row sums its parts in the same order
    ss = 0.f, row_top = 0;
    for (int i = 0; i < wpr; ++i) {
      ss += red_ss[slot * wpr + i];
      row_top = max(row_top, red_top[slot * wpr + i]);
    }
  }
  const float inv = rsqrtf(__fadd_rn(__fdiv_rn(ss, (float)a.width), a.eps));
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = ((v * wpr + part) * 32 + lane) * 8;
    uint32_t t = row_top;
    if (a.group) {
      t = top[v];
      t = max(t, __shfl_xor_sync(0xffffffffu, t, 1));
      t = max(t, __shfl_xor_sync(0xffffffffu, t, 2));
      if (a.group >= 64) t = max(t, __shfl_xor_sync(0xffffffffu, t, 4));
      if (a.group >= 128) t = max(t, __shfl_xor_sync(0xffffffffu, t, 8));
    }
    if (!live || c >= a.width) continue;
    const float tf = __uint_as_float(t);
    const float to = t < kInfBits && tf > kTinyTop ? __fdiv_rn(kQ, tf) : 0.f;
    uint8_t code[8];
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      // an infinity or NaN in the group: codes 0 (its scale below is NaN)
      const float p0 = t < kInfBits ? __fmul_rn(u[v][i], to) : 0.f;
      const float p1 = t < kInfBits ? __fmul_rn(u[v][i + 1], to) : 0.f;
      if (OUT == kDtE4M3) {
        const __nv_fp8x2_storage_t h = __nv_cvt_float2_to_fp8x2(make_float2(p0, p1), __NV_SATFINITE, __NV_E4M3);
        code[i] = (uint8_t)(h & 0xff), code[i + 1] = (uint8_t)(h >> 8);
      } else {
        code[i] = (uint8_t)min(127, max(-127, __float2int_rn(p0)));
        code[i + 1] = (uint8_t)min(127, max(-127, __float2int_rn(p1)));
      }
    }
    uint8_t* q = static_cast<uint8_t*>(a.q) + row * a.ldq + c;
    if (VEC) {
      *reinterpret_cast<uint2*>(q) = *reinterpret_cast<const uint2*>(code);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i < a.width) q[i] = code[i];
    }
    // the first thread of each group (of the row for group 0) stores the scale
    const bool first = a.group ? c % a.group == 0 : c == 0;
    if (first) {
      const float scale = t < kInfBits ? __fdiv_rn(tf > kTinyTop ? tf * inv : 0.f, kQ) : __uint_as_float(0x7fc00000u);
      a.scales[row * a.groups + (a.group ? c / a.group : 0)] = scale;
    }
  }
}

template <typename T, int OUT, bool VEC>
cudaError_t launch_nv(const NormQ8Args& a, int nv, int wpr, dim3 grid, int threads, cudaStream_t s) {
  auto kernel = nv == 1   ? rmsnorm_q8_kernel<T, OUT, 1, VEC>
                : nv == 2 ? rmsnorm_q8_kernel<T, OUT, 2, VEC>
                          : rmsnorm_q8_kernel<T, OUT, 4, VEC>;
  return launch_overlapped(kernel, grid, dim3(threads), 0, s, dim3(1, 1), a, wpr);
}

}  // namespace

cudaError_t launch_rmsnorm_q8(const NormQ8Args& a, cudaStream_t s) {
  auto aligned = [](const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; };
  const bool vec = a.width % 8 == 0 && a.ldx % 8 == 0 && aligned(a.x, 16) && aligned(a.w, 16) && a.ldq % 8 == 0 &&
                   aligned(a.q, 8) &&
                   (!a.residual || (a.ldr % 8 == 0 && a.lds % 8 == 0 && aligned(a.residual, 16) && aligned(a.sum, 16)));
  // One vector per thread while a row fits 32 warps that way.
  const int vectors = (a.width + 7) / 8;
  int nv = 1, wpr = 1;
  while (wpr * 32 < vectors && wpr < 32) wpr *= 2;
  while (nv * wpr * 32 < vectors) nv *= 2;
  if (nv > 4) return cudaErrorInvalidValue;  // more than 32768 columns
  const int warps = wpr < 8 ? 8 : wpr;
  const int64_t rows_per_block = warps / wpr;
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
