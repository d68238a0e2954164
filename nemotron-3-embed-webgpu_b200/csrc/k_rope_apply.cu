// Rotary embedding for any head size, rotated part and pair layout
// (nemo_op_rope_apply; its frequencies come from nemo_rope_inv_freq, layer_ops.cu).
//
// The angle of position p and pair i is p * f_i; only its fraction of a turn
// matters. p * f_i / 2pi is formed in f64 (a position of 2^31 keeps the
// fraction to 2^-22 of a turn and one of a million to 2^-33), reduced there,
// and sincospi of the f32 remainder gives cos and sin.
//
// Bound by memory: every element is read and written once. All heads of a
// token turn by the same angles, so a block computes the cos and sin of its
// token's pairs once, in shared memory, while its first loads are in flight, and
// its threads walk over the heads: thread column = one item of a head, thread
// row = head. Small blocks with few registers hide each other's latencies best:
// 24000 tokens of 24 + 8 heads of 128 take 60 us (the copy rate) with one token
// and 128 threads a block at 32 registers, 75 without the limit, 77 with 256
// threads, 72 to 88 with four tokens a block.
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

// U: items of a thread in flight.
template <typename T, int ITEM, int U>
__global__ void __launch_bounds__(512, 4) rope_apply_kernel(const __grid_constant__ RopeApplyArgs a) {
  __shared__ float2 turn[256];  // (cos, sin) of the token's pairs
  dev::pdl_launch_dependents();
  dev::pdl_wait();
  const int64_t token = blockIdx.x;
  const int half = a.rotary_dim / 2, d = a.head_dim, heads = a.q_heads + a.k_heads;
  const int item = threadIdx.x;

  // The thread's heads threadIdx.y + i * blockDim.y, U at a time: every load
  // before the first store, the first U before the angles are ready.
  int h = threadIdx.y;
  const T* src[U];
  T* dst[U];  // null: none left
  uint4 x[U], y[U];
  // columns of the item: c0 (and c1 its partner's); copied past the rotated ones
  const int turned = ITEM == kPairs8 ? a.rotary_dim / 8 : ITEM == kHalves8 ? half / 8 : half;
  const bool copied = item >= turned;
  int c0, c1 = 0;
  if (ITEM == kPairs8) {
    c0 = item * 8;
  } else if (ITEM == kHalves8) {
    c0 = copied ? a.rotary_dim + (item - turned) * 8 : item * 8, c1 = c0 + half;
  } else {
    c0 = copied ? a.rotary_dim + item - turned : a.layout ? item : 2 * item;
    c1 = a.layout ? c0 + half : c0 + 1;
  }
  auto fetch = [&]() {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      dst[i] = nullptr;
      if (h < heads) {
        const bool is_q = h < a.q_heads;
        src[i] = is_q ? static_cast<const T*>(a.q) + token * a.ldq + h * d
                      : static_cast<const T*>(a.k) + token * a.ldk + (h - a.q_heads) * d;
        dst[i] = is_q ? static_cast<T*>(a.qo) + token * a.ldqo + h * d
                      : static_cast<T*>(a.ko) + token * a.ldko + (h - a.q_heads) * d;
        if (ITEM == kSingle) {
          x[i].x = *reinterpret_cast<const uint16_t*>(src[i] + c0);
          if (!copied) x[i].y = *reinterpret_cast<const uint16_t*>(src[i] + c1);
        } else {
          x[i] = *reinterpret_cast<const uint4*>(src[i] + c0);
          if (ITEM == kHalves8 && !copied) y[i] = *reinterpret_cast<const uint4*>(src[i] + c1);
        }
        h += blockDim.y;
      }
    }
  };
  fetch();
  for (int i = threadIdx.y * blockDim.x + threadIdx.x; i < half; i += blockDim.x * blockDim.y) {
    const double t = (double)a.positions[token] * a.inv_freq[i] * 0.15915494309189533577;  // 1 / 2pi
    float sn, cs;
    sincospif((float)(2.0 * (t - rint(t))), &sn, &cs);
    turn[i] = make_float2(cs * a.magnitude, sn * a.magnitude);
  }
  __syncthreads();
  while (dst[0]) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (!dst[i]) break;
      if (ITEM == kSingle) {
        uint16_t* out = reinterpret_cast<uint16_t*>(dst[i]);
        if (copied) {
          if (src[i] != dst[i]) out[c0] = (uint16_t)x[i].x;
        } else {
          const float2 f = turn[item];
          const float p = dev::unpack2<T>(x[i].x).x, q = dev::unpack2<T>(x[i].y).x;
          dst[i][c0] = dev::from_f32<T>(p * f.x - q * f.y);
          dst[i][c1] = dev::from_f32<T>(p * f.y + q * f.x);
        }
      } else if (copied) {
        if (src[i] != dst[i]) *reinterpret_cast<uint4*>(dst[i] + c0) = x[i];
      } else if (ITEM == kPairs8) {
        float v[8];
        dev::unpack8<T>(x[i], v);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = turn[c0 / 2 + j];
          const float p = v[2 * j], q = v[2 * j + 1];
          v[2 * j] = p * f.x - q * f.y;
          v[2 * j + 1] = p * f.y + q * f.x;
        }
        *reinterpret_cast<uint4*>(dst[i] + c0) = dev::pack8<T>(v);
      } else {
        float v[8], w[8];
        dev::unpack8<T>(x[i], v);
        dev::unpack8<T>(y[i], w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float2 f = turn[c0 + j];
          const float p = v[j], q = w[j];
          v[j] = p * f.x - q * f.y;
          w[j] = p * f.y + q * f.x;
        }
        *reinterpret_cast<uint4*>(dst[i] + c0) = dev::pack8<T>(v);
        *reinterpret_cast<uint4*>(dst[i] + c1) = dev::pack8<T>(w);
      }
    }
    fetch();
  }
}

template <typename T>
cudaError_t launch_rope_t(const RopeApplyArgs& a, int item, dim3 block, cudaStream_t s) {
  auto kernel = item == kPairs8    ? rope_apply_kernel<T, kPairs8, 2>
                : item == kHalves8 ? rope_apply_kernel<T, kHalves8, 1>
                                   : rope_apply_kernel<T, kSingle, 2>;
  return launch_overlapped(kernel, dim3((unsigned)a.tokens), block, 0, s, dim3(1, 1), a);
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
  // few tokens: more threads each (one token 1.8 us with 256, 2.5 with 128)
  const int threads = a.tokens <= 8 * a.sms ? 256 : 128;
  int rows = items >= threads ? 1 : threads / items;
  if (rows > heads) rows = heads;
  const dim3 block(items, rows);
  return a.dtype == kDtBF16 ? launch_rope_t<__nv_bfloat16>(a, item, block, s) : launch_rope_t<__half>(a, item, block, s);
}

}  // namespace nemo
