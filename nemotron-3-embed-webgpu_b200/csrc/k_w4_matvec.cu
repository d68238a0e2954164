// Matrix-vector products with 4-bit weights and group scales, 1 to 16 rows of
// x at once (nemo_op_w4_matvec).
//
//   y[m][r] = sum_g s[r][g] * ( sum_{c in g} x[m][c] * (q[r][c] - z[r][g]) )
//
// The inner sum runs on tensor-core instructions whose A is 16 weight rows and
// whose B holds up to 8 columns made from x; each segment's sum is then scaled in
// f32. (The 128-row tcgen05 tile would hold 16 rows of x against 128 of weights,
// but its operand would have to be written to shared or tensor memory; here the
// decoded integers go from registers straight into the instruction, and the
// bound is the stream of weights, not the tensor rate.) Two forms:
//
//   floating point (m16n8k16): A = the exact small integers q - z in the type of
//   x, B = up to 8 rows of x, f32 accumulation. A word of 8 nibbles takes 9
//   instructions to decode in f16, 11 in bf16.
//
//   digits (m16n8k32, integers): A = the nibbles q themselves, two masks and a
//   shift a word, B = the 8-bit digits of x as fixed-point numbers, four columns
//   a row of x (load_digits; i8 codes are one column). The sums are whole
//   numbers without any rounding; -z * (sum of the digits) is where they start.
//
// A segment is the shorter of the weight group and the group of x scales (32,
// 64 or 128 columns). A lane takes SEG/32 consecutive 32-bit words of a row per
// segment: the columns that an instruction's k index stands for are permuted,
// in the same way for the weights and for x, so that each lane reads its
// weights as one vector and the nibbles of a word that belong together come out
// of one mask (pairs (k, k + 4), or the even and the odd ones); x is stored in
// shared memory in that order.
//
// A warp's work is 16 R rows and a slice of a panel of columns, in chunks of 256
// columns (R x 2 KB). Each warp copies its own next chunks and their scales to
// shared memory while it works on this one, so weights flow without block
// barriers. The 8 warps of a block are wk slices of 8 / wk row tiles: one slice
// where there are rows enough for every warp of the GPU, so that nothing is
// summed over warps; more where there are few rows. Panels (of the columns
// whose x fits shared memory) of a row tile are blocks of one cluster, summed in
// rank order through distributed shared memory. (Chunks of all the block's tiles
// in one stream, an eighth for each warp, balanced better, 28.9 us against 31.0
// when the two were compared, but the sums of tiles that warps share cost 0.3 us in
// small calls and twice the time where a row takes several panels.)
//
// Bound: at 6.5 TB/s an SM gets 4 KB of weights (32 rows x 256 columns) in 180
// cycles, in which its schedulers issue 720 instructions; the floating-point form
// takes some 750 for them, digits about 450. One row of bf16 x against 131072 x
// 2048: 29.4 us with digits, 4.7 TB/s (37.7 without); 512 tiles are 1.7 rounds of
// 296 blocks, and the last round is the most of what is missing. (Earlier
// versions without digits: 16-row tiles 61, a fixed split of every tile over the 8
// warps 51, scales read in line and two logic operations a nibble pair 64.) One row
// against 5120 x 2048: 4.9 us.
#include <type_traits>

#include "layer_ops.cuh"

namespace nemo {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr size_t kSmemLimit = 227 * 1024;           // of a block
constexpr size_t kSmemOfTwo = (228 / 2 - 1) * 1024;  // of each of two blocks an SM, which keeps 1 KB for a block

constexpr int kChunk = 256;   // columns of a copy
constexpr int kPitch = kChunk / 2;

struct W4Plan {
  W4Args a;
  int segs;        // segments of a row
  int panel_segs;  // segments of a block's panel
  int slice_segs;  // segments of a warp's slice of the panel
  int wk;          // slices of a panel: 1, 2, 4 or 8
  int panels;      // panels of a row
  int splits;      // blocks per row tile (cluster size)
  int tiles;       // block tiles (8 / wk x 16 R rows)
  int blocks;      // blocks over the tiles
  int stages;      // chunks in flight
  int tile_rows;   // R: 16-row tiles of a warp
  bool digits;     // the form
  size_t smem;
  int cols;        // columns of x's operand in shared memory: m rounded up to 1, 2, 4, 8 or 16, or m's digits
  int off_x, off_xs, off_zero, off_red;  // byte offsets in shared memory (the warps' stages at 0)
};

// A warp's stage: the weights, then the scales of the groups that a chunk can
// touch (one more where it may start inside a group, which shorter groups of x
// scales allow).
template <int SEG, int R>
struct W4Cfg {
  static constexpr int kRows = 16 * R;
  static constexpr int kGroups = kChunk / SEG + (SEG < 128 ? 1 : 0);
  static constexpr int kStage = kRows * (kPitch + kGroups * 8);
};

// a & b | c in one instruction (the compiler makes two of constant b and c).
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}

// The integers q - z of one 32-bit word as four pairs: (k, k+4), (k+1, k+5),
// (k+2, k+6), (k+3, k+7). zc = the pair -(1024 + z) in f16, -(128 + z) in bf16: a
// nibble masked under the exponent whose unit is 1 is that base plus q.
template <typename T>
struct Nibbles;
template <>
struct Nibbles<__half> {
  static constexpr uint32_t kBase = 0xe400;  // -1024, whose last bits count ones
  // high nibbles sit four bits up: 1024 + 16 q, times 1/16 = 64 + q
  __device__ static __forceinline__ uint32_t high(uint32_t zc) {  // -(64 + z)
    uint32_t d;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(0x63806380u), "r"(zc));
    return d;
  }
  __device__ static __forceinline__ void decode(uint32_t w, uint32_t zc, uint32_t zh, uint32_t (&p)[4]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t lo = and_or(w, 0x000f000fu, 0x64006400u), hi = and_or(w, 0x00f000f0u, 0x64006400u);
      asm("add.rn.f16x2 %0, %1, %2;" : "=r"(p[2 * i]) : "r"(lo), "r"(zc));
      asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(p[2 * i + 1]) : "r"(hi), "r"(0x2c002c00u), "r"(zh));
      w >>= 8;
    }
  }
};
template <>
struct Nibbles<__nv_bfloat16> {
  static constexpr uint32_t kBase = 0xc300;  // -128
  __device__ static __forceinline__ uint32_t high(uint32_t) { return 0; }
  __device__ static __forceinline__ void decode(uint32_t w, uint32_t zc, uint32_t, uint32_t (&p)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // times 1, plus: one instruction, where a bf16 addition or subtraction takes two
      asm("fma.rn.bf16x2 %0, %1, %2, %3;"
          : "=r"(p[i])
          : "r"(and_or(w, 0x000f000fu, 0x43004300u)), "r"(0x3f803f80u), "r"(zc));
      w >>= 4;
    }
  }
};

// D[16 x 8] += A[16 x 32] . B[32 x 8], unsigned by signed 8-bit integers, in one warp.
__device__ __forceinline__ void mma_16832(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
constexpr int kMagic = 0x4b400000;  // 1.5 * 2^23 as bits: plus i, |i| < 2^22, the bits of 1.5 * 2^23 + i

// Eight elements of x as they lie in memory: 16 bytes of 16-bit ones, 8 of codes.
template <bool CODES>
__device__ __forceinline__ uint4 load_x8(const void* x, int64_t at) {
  if constexpr (CODES) {
    const uint8_t* p = static_cast<const uint8_t*>(x) + at;
    uint32_t b[2];
    if (((uintptr_t)p & 7) == 0) {
      const uint2 u = *reinterpret_cast<const uint2*>(p);
      b[0] = u.x, b[1] = u.y;
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        b[i] = p[4 * i] | (uint32_t)p[4 * i + 1] << 8 | (uint32_t)p[4 * i + 2] << 16 | (uint32_t)p[4 * i + 3] << 24;
    }
    return make_uint4(b[0], b[1], 0, 0);
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(x) + at;
    if (((uintptr_t)p & 15) == 0) return *reinterpret_cast<const uint4*>(p);
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = p[2 * i] | (uint32_t)p[2 * i + 1] << 16;
    return make_uint4(v[0], v[1], v[2], v[3]);
  }
}
// Codes as f16 (exact).
__device__ __forceinline__ uint4 codes_to_f16(uint4 u, int dtype) {
  uint32_t v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t two = (i < 2 ? u.x : u.y) >> (i & 1) * 16;
    if (dtype == kDtE4M3) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(two & 0xffff), __NV_E4M3);
      v[i] = h.x | (uint32_t)h.y << 16;
    } else {
      v[i] = dev::pack2<__half>((float)(int8_t)(two & 0xff), (float)(int8_t)(two >> 8 & 0xff));
    }
  }
  return make_uint4(v[0], v[1], v[2], v[3]);
}
// Eight 16-bit elements paired as one word's nibbles are: (0, 4), (1, 5), (2, 6), (3, 7).
__device__ __forceinline__ uint4 pair_x8(uint4 u) {
  const uint32_t v[4] = {u.x, u.y, u.z, u.w};
  return make_uint4(__byte_perm(v[0], v[2], 0x5410), __byte_perm(v[0], v[2], 0x7632), __byte_perm(v[1], v[3], 0x5410),
                    __byte_perm(v[1], v[3], 0x7632));
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

// A row of x and one of its units of eight elements. A block's threads walk over
// the units of all rows in order: one division each at the start.
struct Unit {
  int units, rows_on, units_on;  // of a row; a step of the block
  int m, u;
  __device__ __forceinline__ Unit(int units_, int thread)
      : units(units_), rows_on(kThreads / units_), units_on(kThreads % units_), m(thread / units_), u(thread % units_) {}
  __device__ __forceinline__ void advance() {
    m += rows_on, u += units_on;
    if (u >= units) u -= units, ++m;
  }
};

// T: type of the products (f16 also for 8-bit x, which it holds exactly; int8_t:
// digits). R: 16-row tiles per warp. NT: 8-column tiles of x's operand. XG: x
// scales per group (always with digits).
template <typename T, int SEG, int R, int NT, bool XG>
__global__ void __launch_bounds__(kThreads, 2) w4_matvec_kernel(const __grid_constant__ W4Plan p) {
  extern __shared__ __align__(128) uint8_t smem[];
  using C = W4Cfg<SEG, R>;
  constexpr int WPL = SEG / 32;  // words of a row per lane and segment
  constexpr int ROWS = C::kRows;
  constexpr int SEG_BYTES = SEG / 2, CHUNK_SEGS = kChunk / SEG;
  constexpr bool DIGITS = std::is_same<T, int8_t>::value;
  constexpr int XW = DIGITS ? (WPL < 2 ? 1 : 2) : 1;  // words of a lane whose x is one read of 16 (8 with WPL 1) bytes
  const W4Args& a = p.a;
  dev::pdl_launch_dependents();
  dev::pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = blockIdx.y;
  const int ks = warp % p.wk, wr = warp / p.wk, row_tiles = kWarps / p.wk;
  const int block_rows = row_tiles * ROWS;
  uint8_t* stages = smem + warp * p.stages * C::kStage;
  uint8_t* sx = smem + p.off_x;
  float* sxs = reinterpret_cast<float*>(smem + p.off_xs);            // [segment][column]
  int* sums = reinterpret_cast<int*>(sxs + p.panel_segs * p.cols);   // of the digits, alike
  float* red = reinterpret_cast<float*>(smem + p.off_red);  // two buffers of [wk][row of x][block_rows]
  const int groups = a.k / a.group;
  const int seg_shift = a.group == SEG ? 0 : a.group == 2 * SEG ? 1 : 2;  // segments of a group, log2
  const int zero_bytes = (groups + 1) / 2;
  const int x_groups = (a.k + a.x_group - 1) / a.x_group;
  const int x_shift = 31 - __clz(a.x_group);  // (a power of two where there is more than one)
  const int64_t row_bytes = a.k / 2;

  // The warp's chunks in order: tiles blockIdx.x, + gridDim.x, ...; of each, the
  // panels rank, + splits, ... (one, unless a row has more panels than a cluster
  // has blocks); of each panel, its slice.
  struct Cursor {
    int tile, panel;
    int seg, left;  // the chunk's first segment, segments of the slice from there on
  };
  auto enter = [&](Cursor& c) {  // the slice of c's tile and panel
    c.seg = c.panel * p.panel_segs + ks * p.slice_segs;
    c.left = max(0, min(min(p.slice_segs, p.panel_segs - ks * p.slice_segs), p.segs - c.seg));
  };
  // To the next chunk; whether that is of another slice. A slice counts as one
  // chunk at least, so that every warp meets every tile.
  auto advance = [&](Cursor& c) {
    c.seg += CHUNK_SEGS, c.left -= CHUNK_SEGS;
    if (c.left > 0) return false;
    c.panel += p.splits;
    if (c.panel >= p.panels) {
      c.panel = rank;
      c.tile += gridDim.x;
    }
    enter(c);
    return true;
  };
  Cursor next{(int)blockIdx.x, rank, 0, 0}, cur = next;  // to copy, to work on
  enter(next);
  enter(cur);

  // The copies. Lane: 16-byte unit lane % 8 of the rows lane / 8 + 4 i of the
  // weights, at unit u ^ (row % (8 / WPL)) * WPL of its row, so that the lanes'
  // reads meet no bank twice; the scales and zero points of row lane % ROWS. Rows
  // past the last one repeat it; their sums are not stored.
  const int unit = lane & 7, r0 = lane >> 3, own_row = lane % ROWS;
  const uint8_t* w_from = nullptr;    // the lane's unit of the chunk's first four rows
  const uint16_t* s_from = nullptr;   // the lane's row of scales
  const uint8_t* z_from = nullptr;    // and of zero points
  bool whole = true;                  // every row exists
  auto aim = [&]() {                  // at the slice of `next`
    const int row0 = next.tile * block_rows + wr * ROWS;
    whole = row0 + ROWS <= a.n;
    w_from = a.w + (int64_t)(row0 + r0) * row_bytes + (int64_t)next.seg * SEG_BYTES + unit * 16;
    const int64_t row = min(row0 + own_row, a.n - 1);
    s_from = a.scales + row * groups;
    z_from = a.zeros + row * zero_bytes;
  };
  auto load = [&](int stage) {
    if (next.tile < p.tiles && unit < next.left * (SEG_BYTES / 16)) {
      const uint32_t to = dev::smem_u32(stages) + stage * C::kStage + r0 * kPitch;
      if (whole) {
        const uint8_t* from = w_from;
#pragma unroll
        for (int i = 0; i < ROWS / 4; ++i, from += 4 * row_bytes)
          dev::cp_async16(to + i * 4 * kPitch + (unit ^ ((i * 4 + r0) % (8 / WPL) * WPL)) * 16, from);
      } else {
        const int row0 = next.tile * block_rows + wr * ROWS;
#pragma unroll 1
        for (int i = 0; i < ROWS / 4; ++i)
          dev::cp_async16(to + i * 4 * kPitch + (unit ^ ((i * 4 + r0) % (8 / WPL) * WPL)) * 16,
                          w_from + (int64_t)(min(row0 + i * 4 + r0, a.n - 1) - row0 - r0) * row_bytes);
      }
    }
    dev::cp_async_commit();
  };
  // Scales and zero points are read into registers before the work on another
  // chunk and put into shared memory after it, as [group][row] of the scale
  // (f32) and the pair of the zero constant.
  constexpr int kScales = (C::kGroups + 32 / ROWS - 1) / (32 / ROWS);
  uint32_t scale16[kScales], zero4[kScales];
  auto read_scales = [&]() {
    if (next.tile >= p.tiles) return;
    const int g0 = next.seg >> seg_shift, n = min(next.left, CHUNK_SEGS);
    const int ng = n > 0 ? ((next.seg + n - 1) >> seg_shift) - g0 + 1 : 0;
#pragma unroll
    for (int j = 0; j < kScales; ++j) {
      const int i = lane / ROWS + j * (32 / ROWS);
      scale16[j] = 0, zero4[j] = 8;
      if (i < ng) {
        scale16[j] = s_from[g0 + i];
        if (a.zeros) zero4[j] = (uint32_t)z_from[(g0 + i) >> 1] >> ((g0 + i) & 1) * 4;
      }
    }
  };
  auto put_scales = [&](int stage) {
    uint2* ss = reinterpret_cast<uint2*>(stages + stage * C::kStage + ROWS * kPitch);
#pragma unroll
    for (int j = 0; j < kScales; ++j) {
      const int i = lane / ROWS + j * (32 / ROWS);
      const uint16_t bits = (uint16_t)scale16[j];
      const float f = a.scale_dtype == kDtBF16 ? __uint_as_float(scale16[j] << 16)
                                               : __half2float(*reinterpret_cast<const __half*>(&bits));
      uint32_t zero = zero4[j] & 15;
      if constexpr (!DIGITS) zero = (Nibbles<T>::kBase + zero) * 0x10001u;
      if (i < C::kGroups) ss[i * ROWS + own_row] = make_uint2(__float_as_uint(f), zero);
    }
  };
  // x of a panel in the order of the instructions: for each 32-column step of a
  // segment, row of x and lane t, the 8 columns of that lane's word
  auto load_x = [&](int panel, auto codes) {
    constexpr bool CODES = decltype(codes)::value;
    const int seg0 = panel * p.panel_segs, n = min(p.panel_segs, p.segs - seg0);
    const int units = n * (SEG / 8);  // of a row
    constexpr int kAhead = 4;         // loads in flight
    Unit at(units, threadIdx.x);
    while (at.m < p.cols) {
      uint4 raw[kAhead];
      int to[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j, at.advance()) {
        const int seg = at.u / (SEG / 8), rem = at.u % (SEG / 8);
        to[j] = at.m < p.cols ? (((seg * WPL + rem % WPL) * p.cols + at.m) * 4 + rem / WPL) * 16 : -1;
        raw[j] = make_uint4(0, 0, 0, 0);
        if (at.m < a.m) raw[j] = load_x8<CODES>(a.x, at.m * a.ldx + (int64_t)seg0 * SEG + at.u * 8);
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        if (to[j] >= 0) *reinterpret_cast<uint4*>(sx + to[j]) = pair_x8(CODES ? codes_to_f16(raw[j], a.x_dtype) : raw[j]);
    }
    if (XG)
      for (int i = threadIdx.x; i < n * p.cols; i += kThreads) {
        const int m = i % p.cols, seg = i / p.cols;
        sxs[i] = m < a.m ? a.x_scales[(int64_t)m * x_groups + ((seg0 + seg) * SEG >> x_shift)] : 0.f;
      }
  };
  // The same as digits: element x of a segment whose largest magnitude is below
  // 2^(e + 1) is the integer X = x 2^(29 - e), |X| <= 2^30 (exact where x is at
  // least 2^-19 of the largest, otherwise rounded to 2^-30 of it), in four
  // balanced digits of 8 bits, a column of the operand each (column 4 m + s:
  // digit s, worth 2^(8 s + e - 29)). i8 codes are a digit themselves. Eight
  // elements a thread, the segment's lanes side by side.
  auto load_digits = [&](int panel, auto kind) {
    constexpr int KIND = decltype(kind)::value;  // dtype of x
    constexpr bool CODES = KIND == kDtE4M3 || KIND == kDtI8;
    constexpr int LANES = SEG / 8;
    const int seg0 = panel * p.panel_segs, n = min(p.panel_segs, p.segs - seg0);
    const int units = n * LANES, rows = KIND == kDtI8 ? p.cols : a.m;
    constexpr int kAhead = 4;
    // every lane of a warp takes part in the segments' sums until its warp is done
    Unit from(units, threadIdx.x);
    while (__any_sync(0xffffffffu, from.m < rows)) {
      uint4 raw[kAhead];
      Unit of = from;
#pragma unroll
      for (int j = 0; j < kAhead; ++j, of.advance()) {
        raw[j] = make_uint4(0, 0, 0, 0);
        if (of.m < a.m) raw[j] = load_x8<CODES>(a.x, of.m * a.ldx + (int64_t)seg0 * SEG + of.u * 8);
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j, from.advance()) {
        if (!__any_sync(0xffffffffu, from.m < rows)) break;
        const int m = from.m, u = from.u;
        const bool in = m < rows;
        const int seg = u / LANES, rem = u % LANES, word = rem % WPL;
        float xs = 1.f;
        if (in && a.x_group < a.k)
          xs = m < a.m ? a.x_scales[(int64_t)m * x_groups + ((seg0 + seg) * SEG >> x_shift)] : 0.f;
        const int at = (seg * (WPL / XW) + word / XW) * p.cols;  // the columns' rows of 4 lanes
        uint8_t* to = sx + (rem / WPL) * (XW * 8) + word % XW * 8;
        if constexpr (KIND == kDtI8) {
          const uint32_t even = __byte_perm(raw[j].x, raw[j].y, 0x6420), odd = __byte_perm(raw[j].x, raw[j].y, 0x7531);
          int sum = __dp4a((int)even, 0x01010101, __dp4a((int)odd, 0x01010101, 0));
#pragma unroll
          for (int o = 1; o < LANES; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
          if (in) {
            *reinterpret_cast<uint2*>(to + (at + m) * (XW * 32)) = make_uint2(even, odd);
            if (rem == 0) sxs[seg * p.cols + m] = xs, sums[seg * p.cols + m] = sum;
          }
        } else {
          float v[8];
          if constexpr (KIND == kDtBF16) dev::unpack8<__nv_bfloat16>(raw[j], v);
          else dev::unpack8<__half>(KIND == kDtE4M3 ? codes_to_f16(raw[j], KIND) : raw[j], v);
          uint32_t top = 0;  // as integers magnitudes compare like floats, NaN above infinity
#pragma unroll
          for (int c = 0; c < 8; ++c) top = max(top, __float_as_uint(v[c]) & 0x7fffffffu);
#pragma unroll
          for (int o = 1; o < LANES; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
          int e = (int)(top >> 23) - 127;
          // A factor 2^(29 - e) is finite from e = -97 on. bf16 goes on below: such segments are raised
          // by 2^23 first, to at least 2^-97 or all of them whole multiples of the unit 2^-149.
          const bool raised = KIND == kDtBF16 && e < -97;
          if (raised) {
#pragma unroll
            for (int c = 0; c < 8; ++c) v[c] *= 8388608.f;
            e += 23;
          }
          e = max(e, -97);
          const float up = __uint_as_float((uint32_t)(156 - e) << 23);
          uint32_t d[8];
#pragma unroll
          for (int c = 0; c < 8; ++c) d[c] = ((uint32_t)__float2int_rn(v[c] * up) + 0x00808080u) ^ 0x00808080u;
          uint32_t half[2][4];  // of even and odd columns, the digits s of four elements
          int sum[4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t a01 = __byte_perm(d[h], d[2 + h], 0x5140), a23 = __byte_perm(d[4 + h], d[6 + h], 0x5140);
            const uint32_t b01 = __byte_perm(d[h], d[2 + h], 0x7362), b23 = __byte_perm(d[4 + h], d[6 + h], 0x7362);
            half[h][0] = __byte_perm(a01, a23, 0x5410), half[h][1] = __byte_perm(a01, a23, 0x7632);
            half[h][2] = __byte_perm(b01, b23, 0x5410), half[h][3] = __byte_perm(b01, b23, 0x7632);
          }
#pragma unroll
          for (int c = 0; c < 4; ++c)
            sum[c] = __dp4a((int)half[0][c], 0x01010101, __dp4a((int)half[1][c], 0x01010101, 0));
          // two sums of at most 2^14 in a word
          int low = sum[0] + sum[1] * 65536, high = sum[2] + sum[3] * 65536;
#pragma unroll
          for (int o = 1; o < LANES; o <<= 1) {
            low += __shfl_xor_sync(0xffffffffu, low, o);
            high += __shfl_xor_sync(0xffffffffu, high, o);
          }
          if (in) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
              *reinterpret_cast<uint2*>(to + (at + 4 * m + c) * (XW * 32)) = make_uint2(half[0][c], half[1][c]);
            if (rem < 4) {  // a lane of the segment for each digit
              const int pair = rem & 2 ? high : low, first = (int16_t)(pair & 0xffff);
              sums[seg * p.cols + 4 * m + rem] = rem & 1 ? (pair - first) >> 16 : first;
              // an infinity or NaN makes every product of the row NaN
              float unit = __uint_as_float((uint32_t)(e + 98 + 8 * rem) << 23);
              if (raised) unit *= 1.f / 8388608.f;  // (exact, if subnormal)
              sxs[seg * p.cols + 4 * m + rem] = top < 0x7f800000u ? xs * unit : __uint_as_float(0x7fc00000u);
            }
          }
        }
      }
    }
  };
  auto stage_x = [&](int panel) {
    if constexpr (DIGITS) {
      if (a.x_dtype == kDtF16) load_digits(panel, std::integral_constant<int, kDtF16>{});
      else if (a.x_dtype == kDtBF16) load_digits(panel, std::integral_constant<int, kDtBF16>{});
      else if (a.x_dtype == kDtE4M3) load_digits(panel, std::integral_constant<int, kDtE4M3>{});
      else load_digits(panel, std::integral_constant<int, kDtI8>{});
    } else if (a.x_dtype == kDtE4M3 || a.x_dtype == kDtI8) {
      load_x(panel, std::true_type{});
    } else {
      load_x(panel, std::false_type{});
    }
  };

  const int ahead = p.stages - 1;
  aim();
  auto copy = [&](int stage) {  // the next chunk's weights; its scales into registers
    load(stage);
    read_scales();
    w_from += kPitch;
    if (advance(next)) aim();
  };
  for (int i = 0; i < ahead; ++i) {
    copy(i);
    put_scales(i);
  }
  if (threadIdx.x == 0) *reinterpret_cast<uint4*>(smem + p.off_zero) = make_uint4(0, 0, 0, 0);
  const bool one_panel = p.panels <= p.splits;
  if (one_panel) {
    stage_x(rank);
    __syncthreads();
  }
  // the lane's columns of the operand; those past the last one read zeros behind it
  constexpr int XB = DIGITS ? XW * 8 : 16;  // bytes of a read
  const uint8_t* x_at[NT];
  int x_step[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const bool live = n * 8 + g < p.cols;
    x_at[n] = live ? sx + ((n * 8 + g) * 4 + t) * XB : smem + p.off_zero;
    x_step[n] = live ? p.cols * 4 * XB : 0;
  }
  float acc[R][NT][4];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[r][n][i] = 0.f;
  int stage = 0, fill = ahead;  // of this chunk, of the next copy
  int turn = 0;                 // tiles done
  while (cur.tile < p.tiles) {
    copy(fill);
    if (!one_panel && cur.seg == cur.panel * p.panel_segs + ks * p.slice_segs) {
      __syncthreads();  // the last panel's x is done with
      stage_x(cur.panel);
      __syncthreads();
    }
    if (p.stages == 3) dev::cp_async_wait<2>();
    else dev::cp_async_wait<1>();
    __syncwarp();
    const uint8_t* st = stages + stage * C::kStage;
    const uint2* ss = reinterpret_cast<const uint2*>(st + ROWS * kPitch);
    const int seg0 = cur.seg, g0 = seg0 >> seg_shift, in_panel = seg0 - cur.panel * p.panel_segs;
    const int n_segs = cur.left;
    const uint8_t* wp = st + g * kPitch;  // (rows 8 apart have the same swizzle)
    const int flip = g % (8 / WPL) * WPL * 16;
    const uint8_t* xp[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) xp[n] = x_at[n] + in_panel * (WPL / XW) * x_step[n];
#pragma unroll
    for (int s = 0; s < CHUNK_SEGS; ++s) {
      if (s >= n_segs) break;
      const uint2* sp = ss + (((seg0 + s) >> seg_shift) - g0) * ROWS + g;
      uint32_t w[R][2][WPL], zc[R][2];
      float sc[R][2];
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          lds_words<WPL>(wp + (r * 16 + h * 8) * kPitch + ((s * SEG_BYTES + t * WPL * 4) ^ flip), w[r][h]);
          const uint2 v = sp[r * 16 + h * 8];
          sc[r][h] = __uint_as_float(v.x);
          zc[r][h] = v.y;
        }
      if constexpr (DIGITS) {
        // whole numbers throughout: the sums start at -zero * (sum of the digits),
        // and read as f32 they are 1.5 * 2^23 more than themselves
        float f[NT][2];
        int part[R][NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int col = n * 8 + 2 * t;
          float2 fs = make_float2(0.f, 0.f);
          int2 sd = make_int2(0, 0);
          if (col < p.cols) {
            fs = *reinterpret_cast<const float2*>(sxs + (in_panel + s) * p.cols + col);
            sd = *reinterpret_cast<const int2*>(sums + (in_panel + s) * p.cols + col);
          }
          f[n][0] = fs.x, f[n][1] = fs.y;
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) part[r][n][i] = kMagic - (int)zc[r][i >> 1] * (i & 1 ? sd.y : sd.x);
        }
#pragma unroll
        for (int j = 0; j < WPL; j += XW) {
          uint32_t b[NT][2 * XW];
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            lds_words<2 * XW>(xp[n], b[n]);
            xp[n] += x_step[n];
          }
#pragma unroll
          for (int i = 0; i < XW; ++i)
#pragma unroll
            for (int r = 0; r < R; ++r) {
              const uint32_t w0 = w[r][0][j + i], w1 = w[r][1][j + i];
              const uint32_t a0 = w0 & 0x0f0f0f0fu, a2 = w0 >> 4 & 0x0f0f0f0fu;
              const uint32_t a1 = w1 & 0x0f0f0f0fu, a3 = w1 >> 4 & 0x0f0f0f0fu;
#pragma unroll
              for (int n = 0; n < NT; ++n) mma_16832(part[r][n], a0, a1, a2, a3, b[n][2 * i], b[n][2 * i + 1]);
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              // (the unit of the digit first: exact for 16-bit x, and its product with a weight's scale may underflow)
              acc[r][n][i] = fmaf((__int_as_float(part[r][n][i]) - __int_as_float(kMagic)) * f[n][i & 1], sc[r][i >> 1],
                                  acc[r][n][i]);
      } else {
        uint32_t zh[R][2];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int h = 0; h < 2; ++h) zh[r][h] = Nibbles<T>::high(zc[r][h]);
        float part[R][NT][4];
#pragma unroll
        for (int j = 0; j < WPL; ++j) {
          uint4 b[NT];
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            b[n] = *reinterpret_cast<const uint4*>(xp[n]);
            xp[n] += x_step[n];
          }
#pragma unroll
          for (int r = 0; r < R; ++r) {
            uint32_t lo[4], hi[4];
            Nibbles<T>::decode(w[r][0][j], zc[r][0], zh[r][0], lo);
            Nibbles<T>::decode(w[r][1][j], zc[r][1], zh[r][1], hi);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              if (j == 0) dev::mma_16816_zero<T>(part[r][n], lo[0], hi[0], lo[1], hi[1], b[n].x, b[n].y);
              else dev::mma_16816<T>(part[r][n], lo[0], hi[0], lo[1], hi[1], b[n].x, b[n].y);
              dev::mma_16816<T>(part[r][n], lo[2], hi[2], lo[3], hi[3], b[n].z, b[n].w);
            }
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float f0 = 1.f, f1 = 1.f;  // x scales of the lane's two rows of x
          if (XG) {
            const int m = n * 8 + 2 * t;
            f0 = m < p.cols ? sxs[(in_panel + s) * p.cols + m] : 0.f;
            f1 = m + 1 < p.cols ? sxs[(in_panel + s) * p.cols + m + 1] : 0.f;
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
    }
    put_scales(fill);
    __syncwarp();  // the stage is free for the next copy
    stage = stage + 1 == p.stages ? 0 : stage + 1;
    fill = fill + 1 == p.stages ? 0 : fill + 1;
    const int tile = cur.tile;
    advance(cur);
    if (cur.tile == tile) continue;

    // the tile's sums
    auto store = [&](int m, int row, float y) {
      if (a.x_scales && a.x_group >= a.k) y *= a.x_scales[m];
      const int64_t at = m * a.ldy + row;
      if (a.y_dtype == kDtF32) static_cast<float*>(a.y)[at] = y;
      else if (a.y_dtype == kDtBF16) static_cast<__nv_bfloat16*>(a.y)[at] = __float2bfloat16_rn(y);
      else static_cast<__half*>(a.y)[at] = __float2half_rn(y);
    };
    const bool alone = p.wk == 1 && p.splits == 1;  // no other warp has a part of them
    float* mine = red + (turn++ & 1) * (p.wk * a.m * block_rows);
    auto give = [&](int m, int row, float y) {
      if (m >= a.m) return;
      if (!alone) mine[(ks * a.m + m) * block_rows + row] = y;
      else if (tile * block_rows + row < a.n) store(m, tile * block_rows + row, y);
    };
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int row = wr * ROWS + r * 16 + g;
        if (DIGITS && a.x_dtype != kDtI8) {
          // the four digits of a row of x: two here, two in the next lane
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float y = acc[r][n][2 * h] + acc[r][n][2 * h + 1];
            y += __shfl_xor_sync(0xffffffffu, y, 1);
            if (!(t & 1)) give(n * 2 + t / 2, row + h * 8, y);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) give(n * 8 + 2 * t + (i & 1), row + (i >> 1) * 8, acc[r][n][i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[r][n][i] = 0.f;
      }
    if (alone) continue;
    // over the warps, then over the cluster's panels, both in order; the buffers
    // alternate, so the next tile's sums need no second barrier
    __syncthreads();
    for (int i = threadIdx.x; i < a.m * block_rows; i += kThreads) {
      float v = 0.f;
      for (int w = 0; w < p.wk; ++w) v += mine[w * a.m * block_rows + i];
      if (p.splits > 1) mine[i] = v;  // over slice 0's part
      else if (tile * block_rows + i % block_rows < a.n) store(i / block_rows, tile * block_rows + i % block_rows, v);
    }
    if (p.splits > 1) {
      dev::cluster_sync();
      if (rank == 0)
        for (int i = threadIdx.x; i < a.m * block_rows; i += kThreads) {
          float v = mine[i];
          for (int c = 1; c < p.splits; ++c) v += dev::ld_dsmem_f32(dev::mapa(dev::smem_u32(mine + i), c));
          if (tile * block_rows + i % block_rows < a.n) store(i / block_rows, tile * block_rows + i % block_rows, v);
        }
    }
  }
  dev::cp_async_wait<0>();
  if (p.splits > 1) dev::cluster_sync();  // no block leaves while its sums are read
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
  const dim3 grid((unsigned)p.blocks, (unsigned)p.splits);
  return launch_overlapped(kernel, grid, dim3(kThreads), smem, s, dim3(1, p.splits), p);
}

template <typename T, int SEG, int R>
cudaError_t launch_r(const W4Plan& p, bool xg, size_t smem, cudaStream_t s) {
  if constexpr (std::is_same<T, int8_t>::value)
    return p.cols <= 8 ? launch_kernel<T, SEG, R, 1, true>(p, smem, s) : launch_kernel<T, SEG, R, 2, true>(p, smem, s);
  else if (p.cols <= 8)
    return xg ? launch_kernel<T, SEG, R, 1, true>(p, smem, s) : launch_kernel<T, SEG, R, 1, false>(p, smem, s);
  else
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

namespace {

// The plan of a call whose x has scales per group if xg. False if none fits.
bool plan_w4(const W4Args& a, bool xg, int seg, W4Plan& best) {
  double best_cost = 0;
  best.tile_rows = 0;
  // Digits or floating point, 16 or 32 rows a warp, slices of a panel: whatever
  // has the least modelled time. That is the rounds of blocks over the SMs,
  // times the chunks of a slice (1 with 32 rows, 0.6 with 16; digits cost less
  // of it the longer the segments are) plus a tile's sums (a third of a chunk;
  // two chunks with a cluster's barriers), plus a block's preparation of digits
  // for each eight elements a thread prepares. One f16 row, group 128, us with
  // digits and without: 131072 x 2048 29 / 38, 5120 x 2048 4.8 / 5.0, 2048 x 6144
  // 7.4 / 6.6; group 64, 6144 x 6144: 14.8 / 10.7; sixteen i8 rows, 131072 x 2048
  // 60 / 83, 5120 x 2048 11.4 / 11.0. Digits take four columns a row of x, so
  // they are for two rows at most (four rows against 131072 x 2048 took 50 us
  // with them; 39 without) and for i8, where they are one.
  const double digit_chunk = seg == 128 ? 0.8 : seg == 64 ? 1.0 : 1.2;
  for (int digits = 0; digits < (a.x_dtype == kDtI8 || a.m <= 2 ? 2 : 1); ++digits) {
    W4Plan p = {};
    p.a = a;
    if (!xg) p.a.x_group = a.k;
    p.segs = a.k / seg;
    p.cols = digits ? (a.x_dtype == kDtI8 ? (a.m + 1) / 2 * 2 : 4 * a.m)
                    : a.m <= 1 ? 1 : a.m <= 2 ? 2 : a.m <= 4 ? 4 : a.m <= 8 ? 8 : 16;
    const int x_bytes = digits ? p.cols : 2 * p.cols;  // of a column of the weights
    // A panel's rows of x take at most 48 KB of shared memory; a multiple of the
    // weight group, so that no group is split over panels.
    int panel_k = 48 * 1024 / x_bytes;
    const int panels = (a.k + panel_k - 1) / panel_k;
    panel_k = ((a.k + panels - 1) / panels + a.group - 1) / a.group * a.group;  // panels of one length
    p.panels = (a.k + panel_k - 1) / panel_k;
    p.splits = p.panels < 8 ? p.panels : 8;
    p.panel_segs = panel_k / seg;
    auto smem_of = [&](int r, int stages) {
      const int stage_bytes = 16 * r * (kPitch + (kChunk / seg + (seg < 128 ? 1 : 0)) * 8);
      size_t off = (size_t)kWarps * stages * stage_bytes;
      p.off_x = (int)((off + 127) / 128 * 128);
      off = p.off_x + (size_t)panel_k * x_bytes;
      p.off_xs = (int)off;
      if (xg || digits) off += (size_t)p.panel_segs * p.cols * (digits ? 8 : 4);
      p.off_zero = (int)((off + 15) / 16 * 16);
      p.off_red = p.off_zero + 16;
      return p.off_red + (size_t)2 * kWarps * a.m * 16 * r * 4;
    };
    // of a block: a thread's eight elements each, more for four digits
    const double prepare = digits ? (double)a.m * panel_k / 8 / kThreads * (a.x_dtype == kDtI8 ? 0.04 : 0.15) : 0;
    for (int r = 1; r <= 2; ++r) {
      // three stages where two blocks still fit an SM, or two
      p.stages = smem_of(r, 3) <= kSmemOfTwo ? 3 : 2;
      const size_t bytes = smem_of(r, p.stages);
      if (bytes > kSmemLimit) continue;
      const int resident = (bytes <= kSmemOfTwo ? 2 : 1) * a.sms / p.splits;
      for (p.wk = 1; p.wk <= 8; p.wk *= 2) {
        const int64_t block_rows = 16LL * r * (8 / p.wk), tiles = (a.n + block_rows - 1) / block_rows;
        p.slice_segs = (p.panel_segs + p.wk - 1) / p.wk;
        const int chunks = (p.slice_segs * seg + kChunk - 1) / kChunk;
        const double cost = (double)((tiles + resident - 1) / resident) *
                                (chunks * (r == 1 ? 0.6 : 1.0) * (digits ? digit_chunk : 1.0) + (p.splits > 1 ? 2.0 : 0.35)) +
                            prepare;
        if (best.tile_rows && cost >= best_cost) continue;
        p.tiles = (int)tiles;
        p.blocks = p.tiles < resident ? p.tiles : resident;
        p.tile_rows = r, p.digits = digits, p.smem = bytes;
        best = p, best_cost = cost;
      }
    }
  }
  return best.tile_rows > 0;
}

// Columns of a segment, and whether x has a scale for each of its groups.
int w4_segment(const W4Args& a, bool x_scales, bool& xg) {
  xg = x_scales && a.x_group < a.k;
  return xg && a.x_group < a.group ? a.x_group : a.group;
}

}  // namespace

bool w4_form(const W4Args& a, bool x_scales, W4Form& form) {
  bool xg;
  const int seg = w4_segment(a, x_scales, xg);
  W4Plan p;
  if (!plan_w4(a, xg, seg, p)) return false;
  form.digits = p.digits, form.rows = 16 * p.tile_rows, form.slices = p.wk, form.panels = p.panels;
  form.cluster = p.splits, form.smem = p.smem, form.blocks = p.blocks * p.splits;
  return true;
}

cudaError_t launch_w4_matvec(const W4Args& a, cudaStream_t s) {
  bool xg;
  const int seg = w4_segment(a, a.x_scales != nullptr, xg);
  W4Plan p;
  if (!plan_w4(a, xg, seg, p)) return cudaErrorInvalidValue;
  if (p.digits) return launch_seg<int8_t>(p, seg, p.tile_rows, xg, p.smem, s);
  return a.x_dtype == kDtBF16 ? launch_seg<__nv_bfloat16>(p, seg, p.tile_rows, xg, p.smem, s)
                              : launch_seg<__half>(p, seg, p.tile_rows, xg, p.smem, s);
}

}  // namespace nemo
