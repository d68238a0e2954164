// C entry points of the layer operators of nemo_ops.h: argument checks, the
// device that owns the buffers, and the launch.
#include <math.h>

#include <exception>
#include <initializer_list>

#include "../../include/nemo_ops.h"
#include "layer_ops.cuh"

namespace nemo {
namespace {

static_assert(kDtF16 == NEMO_DTYPE_F16 && kDtBF16 == NEMO_DTYPE_BF16 && kDtF32 == NEMO_DTYPE_F32 &&
                  kDtE4M3 == NEMO_DTYPE_E4M3 && kDtI8 == NEMO_DTYPE_I8,
              "DType and NEMO_DTYPE_* are the same codes");

int refuse(const char* op, const char* what) {
  set_error(std::string(op) + ": " + what);
  return kErrArgs;
}

// Makes the device that owns a call's buffers the current one while the call
// launches, and the previous one again after it. All buffers given (null ones
// are skipped) have to be device memory of one device: a kernel handed
// anything else would fault.
class BufferDevice {
 public:
  int enter(const char* op, std::initializer_list<const void*> buffers) {
    int device = -1;
    for (const void* p : buffers) {
      if (!p) continue;
      cudaPointerAttributes at = {};
      const cudaError_t e = cudaPointerGetAttributes(&at, p);
      if (e != cudaSuccess) {
        cudaGetLastError();
        set_error(std::string(op) + ": " + cudaGetErrorString(e));
        return kErrCuda;
      }
      if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged)
        return refuse(op, "a buffer is not device memory");
      if (device >= 0 && at.device != device) return refuse(op, "buffers of more than one device");
      device = at.device;
    }
    NEMO_CUDA_TRY(cudaGetDevice(&before_));
    if (device >= 0 && device != before_) {
      NEMO_CUDA_TRY(cudaSetDevice(device));
      switched_ = true;
    }
    NEMO_CUDA_TRY(cudaDeviceGetAttribute(&sms_, cudaDevAttrMultiProcessorCount, device >= 0 ? device : before_));
    return kOk;
  }
  int sms() const { return sms_; }  // of the device
  ~BufferDevice() {
    if (switched_) cudaSetDevice(before_);
  }

 private:
  int before_ = 0, sms_ = 0;
  bool switched_ = false;
};

int launched(const char* op, cudaError_t e) {
  if (e == cudaSuccess) return kOk;
  cudaGetLastError();
  set_error(std::string(op) + ": kernel launch failed: " + cudaGetErrorString(e));
  return kErrCuda;
}

// No C++ exception leaves a C entry point.
template <typename F>
int guarded(const char* op, F&& f) {
  try {
    return f();
  } catch (const std::exception&) {
    return kErrState;  // out of host memory while a message was formed
  }
}

bool is16(int dtype) { return dtype == kDtF16 || dtype == kDtBF16; }
bool is8(int dtype) { return dtype == kDtE4M3 || dtype == kDtI8; }
bool misaligned(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) != 0; }
size_t dtype_bytes(int dtype) { return is16(dtype) ? 2 : is8(dtype) ? 1 : 4; }

}  // namespace
}  // namespace nemo

using namespace nemo;

extern "C" {

int nemo_op_rmsnorm_q8(int dtype, const void* d_x, int64_t ldx, const void* d_residual, int64_t ldr, const void* d_w,
                       int rows, int width, float eps, void* d_sum, int64_t lds, int out_dtype, int group, void* d_q,
                       int64_t ldq, void* d_scales, void* stream) {
  const char* op = "nemo_op_rmsnorm_q8";
  return guarded(op, [&]() -> int {
    if (!is16(dtype)) return refuse(op, "x must be f16 or bf16");
    if (!is8(out_dtype)) return refuse(op, "the output must be e4m3 or i8");
    if (rows < 0 || width < 1 || width > 32768) return refuse(op, "rows >= 0 and width in [1, 32768]");
    if (group != 0 && group != 32 && group != 64 && group != 128) return refuse(op, "group must be 0, 32, 64 or 128");
    if (!(eps >= 0.f) || isinf(eps)) return refuse(op, "eps must be finite and not negative");
    if (!d_x || !d_w || !d_q || !d_scales) return refuse(op, "null buffer");
    if (!d_residual != !d_sum) return refuse(op, "d_sum goes with d_residual");
    if (ldx < width || ldq < width || (d_residual && (ldr < width || lds < width)))
      return refuse(op, "a leading dimension is less than the width");
    if ((d_sum == d_x && lds != ldx) || (d_sum && d_sum == d_residual && lds != ldr))
      return refuse(op, "in place needs the same leading dimension");
    if (misaligned(d_x, 2) || misaligned(d_residual, 2) || misaligned(d_sum, 2) || misaligned(d_w, 4) ||
        misaligned(d_scales, 4))
      return refuse(op, "a buffer is not aligned to its element");
    if (rows == 0) return kOk;
    BufferDevice device;
    if (int rc = device.enter(op, {d_x, d_residual, d_w, d_sum, d_q, d_scales})) return rc;
    NormQ8Args a = {};
    a.x = d_x, a.residual = d_residual, a.w = (const float*)d_w, a.sum = d_sum, a.q = d_q;
    a.scales = (float*)d_scales;
    a.ldx = ldx, a.ldr = ldr, a.lds = lds, a.ldq = ldq;
    a.rows = rows, a.width = width, a.group = group, a.groups = group ? (width + group - 1) / group : 1;
    a.eps = eps, a.dtype = dtype, a.out_dtype = out_dtype, a.sms = device.sms();
    return launched(op, launch_rmsnorm_q8(a, (cudaStream_t)stream));
  });
}

int nemo_rope_inv_freq(int scaling, double theta, int rotary_dim, double factor, double original_context, double slow,
                       double fast, double* out, float* magnitude) {
  const char* op = "nemo_rope_inv_freq";
  return guarded(op, [&]() -> int {
    if (!out || !magnitude) return refuse(op, "null buffer");
    if (scaling < NEMO_ROPE_PLAIN || scaling > NEMO_ROPE_RAMP) return refuse(op, "unknown scaling");
    if (rotary_dim < 2 || rotary_dim % 2 || rotary_dim > 512) return refuse(op, "rotary_dim must be even and in [2, 512]");
    if (!(theta > 1.0) || isinf(theta)) return refuse(op, "theta must be finite and above 1");
    if (scaling != NEMO_ROPE_PLAIN && (!(factor >= 1.0) || isinf(factor)))
      return refuse(op, "factor must be finite and at least 1");
    if (scaling == NEMO_ROPE_NTK && rotary_dim < 4) return refuse(op, "this scaling needs a rotary_dim of 4 or more");
    if (scaling >= NEMO_ROPE_YARN && (!(original_context > 0) || !(slow > 0) || !(fast > slow) || isinf(fast) ||
                                      isinf(original_context)))
      return refuse(op, "original_context > 0 and 0 < slow < fast are needed");
    const int half = rotary_dim / 2;
    const double two_pi = 2.0 * M_PI;
    if (scaling == NEMO_ROPE_NTK) theta *= pow(factor, (double)rotary_dim / (rotary_dim - 2));
    if (isinf(theta)) return refuse(op, "the scaled theta is not finite");
    // the pair that turns `turns` times in the original context
    auto pair_of = [&](double turns) {
      return rotary_dim * log(original_context / (turns * two_pi)) / (2.0 * log(theta));
    };
    for (int i = 0; i < half; ++i) {
      const double f = pow(theta, -2.0 * i / rotary_dim);
      double keep = 1.0;  // share of f itself; the rest is f / factor
      if (scaling == NEMO_ROPE_LINEAR) {
        keep = 0.0;
      } else if (scaling == NEMO_ROPE_YARN) {
        const double low = floor(pair_of(fast)), high = ceil(pair_of(slow));
        keep = 1.0 - fmin(1.0, fmax(0.0, (i - low) / fmax(0.001, high - low)));
      } else if (scaling == NEMO_ROPE_RAMP) {
        keep = fmin(1.0, fmax(0.0, (original_context * f / two_pi - slow) / (fast - slow)));
      }
      out[i] = scaling == NEMO_ROPE_PLAIN || scaling == NEMO_ROPE_NTK ? f : f / factor * (1.0 - keep) + f * keep;
    }
    *magnitude = scaling == NEMO_ROPE_YARN ? (float)(0.1 * log(factor) + 1.0) : 1.0f;
    return kOk;
  });
}

int nemo_op_rope_apply(int dtype, int layout, const void* d_q, int64_t ldq, int q_heads, const void* d_k, int64_t ldk,
                       int k_heads, int head_dim, int rotary_dim, const void* d_inv_freq, float magnitude,
                       const void* d_positions, int tokens, void* d_qo, int64_t ldqo, void* d_ko, int64_t ldko,
                       void* stream) {
  const char* op = "nemo_op_rope_apply";
  return guarded(op, [&]() -> int {
    if (!is16(dtype)) return refuse(op, "q and k must be f16 or bf16");
    if (layout != NEMO_ROPE_PAIRS && layout != NEMO_ROPE_HALVES) return refuse(op, "unknown layout");
    if (q_heads < 1 || k_heads < 0 || q_heads > 65535 || k_heads > 65535 || tokens < 0)
      return refuse(op, "q_heads in [1, 65535], k_heads in [0, 65535], tokens >= 0");
    if (head_dim < 2 || head_dim > 512 || rotary_dim < 2 || rotary_dim % 2 || rotary_dim > head_dim)
      return refuse(op, "head_dim in [2, 512], rotary_dim even and in [2, head_dim]");
    if (!isfinite(magnitude)) return refuse(op, "magnitude must be finite");
    if (!d_q || !d_qo || !d_inv_freq || !d_positions || (k_heads && (!d_k || !d_ko))) return refuse(op, "null buffer");
    const int64_t wq = (int64_t)q_heads * head_dim, wk = (int64_t)k_heads * head_dim;
    if (ldq < wq || ldqo < wq || (k_heads && (ldk < wk || ldko < wk)))
      return refuse(op, "a leading dimension is less than the heads of a row");
    if ((d_q == d_qo && ldq != ldqo) || (k_heads && d_k == d_ko && ldk != ldko))
      return refuse(op, "in place needs the same leading dimension");
    if (misaligned(d_q, 2) || misaligned(d_qo, 2) || (k_heads && (misaligned(d_k, 2) || misaligned(d_ko, 2))) ||
        misaligned(d_inv_freq, 8) || misaligned(d_positions, 4))
      return refuse(op, "a buffer is not aligned to its element");
    if (tokens == 0) return kOk;
    BufferDevice device;
    if (int rc = device.enter(op, {d_q, d_qo, k_heads ? d_k : nullptr, k_heads ? d_ko : nullptr, d_inv_freq, d_positions}))
      return rc;
    RopeApplyArgs a = {};
    a.q = d_q, a.k = d_k, a.qo = d_qo, a.ko = d_ko;
    a.inv_freq = (const double*)d_inv_freq, a.positions = (const int*)d_positions;
    a.ldq = ldq, a.ldk = ldk, a.ldqo = ldqo, a.ldko = ldko;
    a.q_heads = q_heads, a.k_heads = k_heads, a.head_dim = head_dim, a.rotary_dim = rotary_dim, a.tokens = tokens;
    a.magnitude = magnitude, a.dtype = dtype, a.layout = layout, a.sms = device.sms();
    return launched(op, launch_rope_apply(a, (cudaStream_t)stream));
  });
}

int nemo_op_w4_matvec(int x_dtype, const void* d_x, int64_t ldx, const void* d_x_scales, int x_group, const void* d_w4,
                      int scale_dtype, const void* d_scales, const void* d_zeros, int group, int m, int n, int k,
                      int y_dtype, void* d_y, int64_t ldy, void* stream) {
  const char* op = "nemo_op_w4_matvec";
  return guarded(op, [&]() -> int {
    if (!is16(x_dtype) && !is8(x_dtype)) return refuse(op, "x must be f16, bf16, e4m3 or i8");
    if (!is16(scale_dtype)) return refuse(op, "scales must be f16 or bf16");
    if (!is16(y_dtype) && y_dtype != kDtF32) return refuse(op, "y must be f16, bf16 or f32");
    if (m < 0 || m > 16) return refuse(op, "m must be in [0, 16]: more rows take a call for each 16 of them");
    if (n < 1 || k < 1 || n > 1 << 30 || k > 1 << 30) return refuse(op, "n and k must be positive and at most 2^30");
    if (group != 32 && group != 64 && group != 128) return refuse(op, "group must be 32, 64 or 128");
    if (k % group) return refuse(op, "group must divide k");
    if (is8(x_dtype) != (d_x_scales != nullptr)) return refuse(op, "8-bit x needs d_x_scales, 16-bit x takes none");
    if (d_x_scales && x_group != 32 && x_group != 64 && x_group != 128 && x_group < k)
      return refuse(op, "x_group must be 32, 64, 128 or at least k");
    if (!d_x || !d_w4 || !d_scales || !d_y) return refuse(op, "null buffer");
    if (ldx < k || ldy < n) return refuse(op, "a leading dimension is less than the row");
    if (misaligned(d_w4, 16)) return refuse(op, "d_w4 must be 16-byte aligned");
    if (misaligned(d_x, dtype_bytes(x_dtype)) || misaligned(d_scales, 2) || misaligned(d_x_scales, 4) ||
        misaligned(d_y, dtype_bytes(y_dtype)))
      return refuse(op, "a buffer is not aligned to its element");
    if (m == 0) return kOk;
    BufferDevice device;
    if (int rc = device.enter(op, {d_x, d_x_scales, d_w4, d_scales, d_zeros, d_y})) return rc;
    W4Args a = {};
    a.x = d_x, a.x_scales = (const float*)d_x_scales, a.w = (const uint8_t*)d_w4;
    a.scales = (const uint16_t*)d_scales, a.zeros = (const uint8_t*)d_zeros, a.y = d_y;
    a.ldx = ldx, a.ldy = ldy, a.x_dtype = x_dtype, a.scale_dtype = scale_dtype, a.y_dtype = y_dtype;
    a.x_group = x_group, a.group = group, a.m = m, a.n = n, a.k = k, a.sms = device.sms();
    return launched(op, launch_w4_matvec(a, (cudaStream_t)stream));
  });
}

int nemo_op_w4_matvec_form(int x_dtype, int x_group, int group, int m, int n, int k, int sms, int* digits, int* rows,
                           int* slices, int* panels, int* blocks, int* shared_bytes) {
  const char* op = "nemo_op_w4_matvec_form";
  return guarded(op, [&]() -> int {
    if ((!is16(x_dtype) && !is8(x_dtype)) || m < 1 || m > 16 || n < 1 || k < 1 || n > 1 << 30 || k > 1 << 30 ||
        (group != 32 && group != 64 && group != 128) || k % group || sms < 1 ||
        (is8(x_dtype) && x_group != 32 && x_group != 64 && x_group != 128 && x_group < k))
      return refuse(op, "sizes or types out of range");
    if (!digits || !rows || !slices || !panels || !blocks || !shared_bytes) return refuse(op, "null buffer");
    W4Args a = {};
    a.x_dtype = x_dtype, a.x_group = x_group, a.group = group, a.m = m, a.n = n, a.k = k, a.sms = sms;
    W4Form f;
    if (!w4_form(a, is8(x_dtype), f)) return refuse(op, "no form fits");
    *digits = f.digits, *rows = f.rows, *slices = f.slices, *panels = f.panels, *blocks = f.blocks;
    *shared_bytes = (int)f.smem;
    return kOk;
  });
}

int nemo_op_attention_window(int dtype, const void* d_q, int64_t ldq, const void* d_k, int64_t ldk, const void* d_v,
                             int64_t ldv, int q_heads, int kv_heads, int head_dim, const void* d_q_off,
                             const void* d_k_start, const void* d_k_len, int batch, int q_rows, int k_rows, int max_q,
                             int max_k, int left, int right, int sinks, float scale, void* d_out, int64_t ldo,
                             void* d_err, void* stream) {
  const char* op = "nemo_op_attention_window";
  return guarded(op, [&]() -> int {
    if (!is16(dtype)) return refuse(op, "q, k and v must be f16 or bf16");
    if (head_dim != 64 && head_dim != 128) return refuse(op, "head_dim must be 64 or 128");
    if (kv_heads < 1 || kv_heads > 65535 || q_heads < 1 || q_heads > 65535 || q_heads % kv_heads)
      return refuse(op, "q_heads must be a multiple of kv_heads, both in [1, 65535]");
    if (batch < 0 || batch > 65535) return refuse(op, "batch must be in [0, 65535]");
    if (q_rows < 0 || k_rows < 0 || max_q < 0 || max_k < 0) return refuse(op, "row counts must not be negative");
    if (left < -1 || right < -1 || sinks < 0) return refuse(op, "left and right >= -1 and sinks >= 0");
    if (!(scale > 0.f) || isinf(scale)) return refuse(op, "scale must be finite and above 0");
    if (!d_q_off || !d_k_start || !d_k_len || !d_err) return refuse(op, "null buffer");
    if (q_rows && (!d_q || !d_out)) return refuse(op, "null buffer");
    if (k_rows && (!d_k || !d_v)) return refuse(op, "null buffer");
    if (ldq < (int64_t)q_heads * head_dim || ldo < (int64_t)q_heads * head_dim ||
        ldk < (int64_t)kv_heads * head_dim || ldv < (int64_t)kv_heads * head_dim)
      return refuse(op, "a leading dimension is less than the heads of a row");
    if (ldq % 8 || ldk % 8 || ldv % 8 || ldo % 8) return refuse(op, "leading dimensions must be multiples of 8");
    if (misaligned(d_q, 16) || misaligned(d_k, 16) || misaligned(d_v, 16) || misaligned(d_out, 16))
      return refuse(op, "q, k, v and out must be 16-byte aligned");
    if (misaligned(d_q_off, 4) || misaligned(d_k_start, 4) || misaligned(d_k_len, 4) || misaligned(d_err, 4))
      return refuse(op, "a buffer is not aligned to its element");
    if (batch == 0 || q_rows == 0 || max_q == 0) return kOk;
    BufferDevice device;
    if (int rc = device.enter(op, {d_q, k_rows ? d_k : nullptr, k_rows ? d_v : nullptr, d_out, d_q_off, d_k_start,
                                   d_k_len, d_err}))
      return rc;
    AttnWindowArgs a = {};
    a.q = d_q, a.k = d_k, a.v = d_v, a.out = d_out;
    a.q_off = (const int*)d_q_off, a.k_start = (const int*)d_k_start, a.k_len = (const int*)d_k_len;
    a.err = (uint32_t*)d_err;
    a.ldq = ldq, a.ldk = ldk, a.ldv = ldv, a.ldo = ldo;
    a.q_heads = q_heads, a.kv_heads = kv_heads, a.head_dim = head_dim, a.batch = batch;
    a.q_rows = q_rows, a.k_rows = k_rows, a.max_q = max_q < q_rows ? max_q : q_rows;
    a.max_k = max_k < k_rows ? max_k : k_rows;
    a.left = left, a.right = right, a.sinks = sinks, a.scale = scale, a.dtype = dtype, a.sms = device.sms();
    return launched(op, launch_attention_window(a, (cudaStream_t)stream));
  });
}

int nemo_op_attention_window_form(int q_heads, int kv_heads, int head_dim, int batch, int q_rows, int k_rows, int max_q,
                                  int max_k, int left, int right, int sinks, int sms, int max_cluster, int* tiles,
                                  int* splits) {
  const char* op = "nemo_op_attention_window_form";
  return guarded(op, [&]() -> int {
    if (kv_heads < 1 || q_heads < 1 || q_heads % kv_heads || batch < 1 || q_rows < 1 || k_rows < 0 || max_q < 1 ||
        max_k < 0 || left < -1 || right < -1 || sinks < 0 || sms < 1 || max_cluster < 1)
      return refuse(op, "sizes out of range");
    if (!tiles || !splits) return refuse(op, "null buffer");
    AttnWindowArgs a = {};
    a.q_heads = q_heads, a.kv_heads = kv_heads, a.head_dim = head_dim, a.batch = batch, a.q_rows = q_rows;
    a.k_rows = k_rows, a.max_q = max_q < q_rows ? max_q : q_rows, a.max_k = max_k < k_rows ? max_k : k_rows;
    a.left = left, a.right = right, a.sinks = sinks, a.sms = sms;
    *tiles = attention_on_tiles(a);
    *splits = *tiles ? 1 : attention_splits(a, max_cluster);
    return kOk;
  });
}

}  // extern "C"
