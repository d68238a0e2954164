// Rotary embedding for any head size, rotated part and pair layout
// (nemo_op_rope_apply), and the host frequencies of scaled contexts.
//
// The angle of position p and pair i is p * f_i; only its fraction of a turn
// matters. p * f_i / 2pi is formed in f64 (a position of 2^31 keeps the
// fraction to 2^-22 of a turn and one of a million to 2^-33), reduced there,
// and sincospi of the f32 remainder gives cos and sin.
//
// Bound by memory: every element is read and written once. All heads of a
// token turn by the same angles, so a block computes the cos and sin of its
// tokens' pairs once, in shared memory, and its threads then walk over the
// heads: thread column = one item of a head, thread row = head.
#include <math.h>

#include "layer_ops.cuh"

namespace nemo {
namespace {

// What one thread turns at a time.
enum RopeItem {
  kPairs8,   // pairs layout: 8 consecutive columns (4 pairs, or 8 copied columns)
  kHalves8,  // halves layout: 8 columns and their 8 partners (or 8 copied columns)
  kSingle,   // any layout and alignment: one pair (or one copied column)
};

template <typename T, int ITEM>
__global__ void __launch_bounds__(512) rope_apply_kernel(const __grid_constant__ RopeApplyArgs a, int tokens_per_block) {
  extern __shared__ float2 turns[];  // [tokens_per_block][rotary_dim / 2] (cos, sin)
  dev::pdl_launch_dependents();
  dev::pdl_wait();
  const int half = a.rotary_dim / 2;
  const int t0 = blockIdx.x * tokens_per_block;
  const int nt = min(tokens_per_block, a.tokens - t0);
  const int tid = threadIdx.y * blockDim.x + threadIdx.x;
  for (int i = tid; i < nt * half; i += blockDim.x * blockDim.y) {
    const int t = i / half, p = i - t * half;
    const double turn = (double)a.positions[t0 + t] * a.inv_freq[p] * 0.15915494309189533577;  // 1 / 2pi
    float sn, cs;
    sincospif((float)(2.0 * (turn - rint(turn))), &sn, &cs);
    turns[i] = make_float2(cs * a.magnitude, sn * a.magnitude);
  }
  __syncthreads();
  const int item = threadIdx.x, d = a.head_dim;
  const int heads = a.q_heads + a.k_heads;
  for (int t = 0; t < nt; ++t) {
    const float2* cs = turns + t * half;
    for (int h = threadIdx.y; h < heads; h += blockDim.y) {
      const bool is_q = h < a.q_heads;
      const int64_t tok = t0 + t;
      const T* src = is_q ? static_cast<const T*>(a.q) + tok * a.ldq + h * d
                          : static_cast<const T*>(a.k) + tok * a.ldk + (h - a.q_heads) * d;
      T* dst = is_q ? static_cast<T*>(a.qo) + tok * a.ldqo + h * d
                    : static_cast<T*>(a.ko) + tok * a.ldko + (h - a.q_heads) * d;
      if (ITEM == kPairs8) {
        const int c = item * 8;
        const uint4 in = *reinterpret_cast<const uint4*>(src + c);
        if (c < a.rotary_dim) {
          float v[8];
          dev::unpack8<T>(in, v);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = cs[c / 2 + i];
            const float x = v[2 * i], y = v[2 * i + 1];
            v[2 * i] = x * f.x - y * f.y;
            v[2 * i + 1] = x * f.y + y * f.x;
          }
          *reinterpret_cast<uint4*>(dst + c) = dev::pack8<T>(v);
        } else if (src != dst) {
          *reinterpret_cast<uint4*>(dst + c) = in;
        }
      } else if (ITEM == kHalves8) {
        const int turned = half / 8;
        if (item < turned) {
          const int c = item * 8;
          float x[8], y[8];
          dev::unpack8<T>(*reinterpret_cast<const uint4*>(src + c), x);
          dev::unpack8<T>(*reinterpret_cast<const uint4*>(src + half + c), y);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 f = cs[c + i];
            const float p = x[i], q = y[i];
            x[i] = p * f.x - q * f.y;
            y[i] = p * f.y + q * f.x;
          }
          *reinterpret_cast<uint4*>(dst + c) = dev::pack8<T>(x);
          *reinterpret_cast<uint4*>(dst + half + c) = dev::pack8<T>(y);
        } else if (src != dst) {
          const int c = a.rotary_dim + (item - turned) * 8;
          *reinterpret_cast<uint4*>(dst + c) = *reinterpret_cast<const uint4*>(src + c);
        }
      } else {
        if (item < half) {
          const int c0 = a.layout ? item : 2 * item, c1 = a.layout ? item + half : 2 * item + 1;
          const float2 f = cs[item];
          const float x = dev::to_f32(src[c0]), y = dev::to_f32(src[c1]);
          dst[c0] = dev::from_f32<T>(x * f.x - y * f.y);
          dst[c1] = dev::from_f32<T>(x * f.y + y * f.x);
        } else {
          const int c = a.rotary_dim + item - half;
          if (src != dst) dst[c] = src[c];
        }
      }
    }
  }
}

template <typename T>
cudaError_t launch_rope_t(const RopeApplyArgs& a, int item, dim3 grid, dim3 block, size_t smem, int tpb,
                          cudaStream_t s) {
  auto kernel = item == kPairs8    ? rope_apply_kernel<T, kPairs8>
                : item == kHalves8 ? rope_apply_kernel<T, kHalves8>
                                   : rope_apply_kernel<T, kSingle>;
  return launch_overlapped(kernel, grid, block, smem, s, dim3(1, 1), a, tpb);
}

}  // namespace

cudaError_t launch_rope_apply(const RopeApplyArgs& a, cudaStream_t s) {
  auto aligned = [](const void* p) { return ((uintptr_t)p & 15) == 0; };
  const bool vec = a.head_dim % 8 == 0 && a.ldq % 8 == 0 && a.ldqo % 8 == 0 && aligned(a.q) && aligned(a.qo) &&
                   (a.k_heads == 0 || (a.ldk % 8 == 0 && a.ldko % 8 == 0 && aligned(a.k) && aligned(a.ko)));
  int item = kSingle, items = a.rotary_dim / 2 + a.head_dim - a.rotary_dim;
  if (vec && !a.layout && a.rotary_dim % 8 == 0) item = kPairs8, items = a.head_dim / 8;
  if (vec && a.layout && a.rotary_dim % 16 == 0) {
    item = kHalves8;
    items = a.rotary_dim / 16 + (a.head_dim - a.rotary_dim) / 8;
  }
  const int heads = a.q_heads + a.k_heads;
  int rows = items >= 256 ? 1 : 256 / items;
  if (rows > heads) rows = heads;
  const int tpb = 1;
  const size_t smem = (size_t)tpb * (a.rotary_dim / 2) * sizeof(float2);
  const dim3 grid((unsigned)((a.tokens + tpb - 1) / tpb)), block(items, rows);
  return a.dtype == kDtBF16 ? launch_rope_t<__nv_bfloat16>(a, item, grid, block, smem, tpb, s)
                            : launch_rope_t<__half>(a, item, grid, block, smem, tpb, s);
}

}  // namespace nemo
