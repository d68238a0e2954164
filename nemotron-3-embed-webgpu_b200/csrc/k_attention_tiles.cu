// Windowed attention of prompts and documents (nemo_op_attention_window) on the
// 5th-generation tensor cores.
//
// Work is cut into units: 128 consecutive queries of one head. A block takes
// two units that follow one another in the order (query tile, head of the kv
// group), so that both read the same keys (two heads of one tile) or nearly
// the same (neighbouring tiles), and every K and V tile it loads serves both.
// For each unit and tile of 64 keys:
//   S = Q . K^T   (tcgen05, f32 in tensor memory)
//   online softmax by the unit's four warps, one query row per thread
//   P = 2^(S scale log2 e - m) rounded to the 16-bit type over the columns of S,
//   m the running maximum (f16: less weight_lift)
//   O += P . V    (tcgen05, P from tensor memory, O stays there)
// Each unit has two S tiles in tensor memory (2 x 64 columns beside 128 of O;
// two units fill the 512): the products of the next key tile are ready when a
// softmax ends, so neither side waits for the other's latency. (When they came in,
// 180 us for the 8,192 tokens below, 347 with tiles of 128 keys and one S of 128
// columns.)
//
// The window: a block's key tiles start at its first visible key, the sinks in
// front of it have tiles of their own behind the window's (the running maximum
// that a window leaves rarely moves again: sinks in front took 3 % more for
// sixteen requests of 1 to 1,500 tokens, 24 heads of 128, window 128 + 128 and one
// sink), and each product covers only the 32-key chunks that some
// query of the unit sees. Within a tile each warp leaves out the chunks that
// none of its 32 rows sees and masks only those that some of them do not see
// whole.
//
// Bound: both the tensor cores and the exponential unit need 512 cycles per
// 128 x 64 tile at head size 128. Measured: a prompt of 8,192 tokens, heads as
// above, causal with 2,048 keys a query 166 to 177 us on different cards (1.02 to
// 1.09 PFLOP/s of the visible pairs) in a row of launches, 201 for one launch
// between two events; the sixteen above 102 to 104 us, where half of the tiles are
// masked ones and each pair of units has six or seven: the masks and maxima are
// about 12 us of it, the output 16 and the sink 12.
//
// Warps (384 threads, persistent, one block per SM): 0 copies Q, K and V (TMA),
// 1 and 2 issue the units' products (a warp each: the tensor pipe takes one
// unit's while the other's warp waits or finds its next tile), 3 clears the rows
// of V behind a tile's last key, 4-7 and 8-11 are the units' softmax. The copies
// and first products of the next pair of units run under the output of this
// one. All waits are bounded.
#include <math.h>

#include "attention_window.cuh"
#include "kernels.cuh"

namespace nemo {
namespace {

constexpr int kRows = 128;          // queries of a unit
constexpr int kKeys = 64;           // keys of a tile
constexpr int kChunks = kKeys / 32;
constexpr int kMaxRequests = 1024;  // of one launch: their pair counts are summed in shared memory
constexpr int kListed = 48;         // items of a block that are worked out at its start
constexpr float kMaxSum = 32768.f;  // sum of a row's weights of one tile against an old reference, at most
constexpr float kMaxSlack = 14.f;   // and how far such a one may be exceeded (log2): f16 ends at 65504

template <int D>
struct TilesCfg {
  static constexpr int kQHalf = kRows * 128;     // 64 columns of Q: one 128-byte-swizzle block
  static constexpr int kQ = D / 64 * kQHalf;
  static constexpr int kHalf = kKeys * 128;      // 64 columns of K or V
  static constexpr int kTileBytes = D / 64 * kHalf;
  static constexpr int kStages = 4;              // K and V tiles in flight: two ahead of V for S, one to load
  static constexpr int kThreads = 384;
  static constexpr int kListedBytes = 96 * kListed;  // a Pair each
  static constexpr int kRedoBytes = 32 * kListed;    // a bit for each row of a Pair
  static constexpr int kSmem =
      1024 + 2 * kQ + kStages * 2 * kTileBytes + 256 + kListedBytes + kRedoBytes + (kMaxRequests + 1) * 4;
  static constexpr uint32_t kTmemCols = 512;
  static constexpr uint32_t kColS = 0, kColO = 256;  // S tile i of unit t at 128 t + 64 i, O_t at 256 + 128 t
};

// One unit of a block's pair.
struct Unit {
  int head, i0, rows;  // q head, first query, queries (0: no such unit)
  int lo, hi;          // window keys that some query of the unit sees
  int full0, full1;    // tiles [full0, full1) of the pair that are needed whole
};

// A pair of units and the key tiles it walks over: the window's, then the sinks'.
struct alignas(16) Pair {
  AttnRequest rq;
  int kvh, sink, lo, hi, window_tiles, tiles;
  Unit u[2];
  __device__ __forceinline__ Pair() {}
  __device__ __forceinline__ Pair(const AttnWindowArgs& a, int b, int kvh_, int pair) : rq(a, b), kvh(kvh_) {
    const int group = a.q_heads / a.kv_heads;
    const int nq = min(rq.nq, a.max_q), p_off = rq.nk - rq.nq;
    const int units = (nq + kRows - 1) / kRows * group;
    lo = rq.nk, hi = 0;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int n = pair * 2 + t;
      u[t].i0 = n / group * kRows;
      u[t].head = kvh * group + n % group;
      u[t].rows = n < units ? min(kRows, nq - u[t].i0) : 0;
      u[t].lo = u[t].hi = 0;
      if (u[t].rows) {
        const KeyRange r(a, u[t].i0 + p_off, u[t].i0 + u[t].rows - 1 + p_off, rq.nk);
        u[t].lo = r.lo, u[t].hi = r.hi;
        if (r.hi > 0) lo = min(lo, r.lo), hi = max(hi, r.hi);
      }
    }
    if (lo > hi) lo = hi;
    sink = min(a.sinks, lo);
    window_tiles = (hi - lo + kKeys - 1) / kKeys;
    tiles = window_tiles + (sink + kKeys - 1) / kKeys;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      u[t].full0 = (max(u[t].lo - lo, 0) + kKeys - 1) / kKeys;
      u[t].full1 = max(u[t].hi - lo, 0) / kKeys;
    }
  }
  __device__ __forceinline__ Unit unit(int t) const {  // by selects: an index would put the pair into local memory
    Unit r;
    r.head = t ? u[1].head : u[0].head, r.i0 = t ? u[1].i0 : u[0].i0, r.rows = t ? u[1].rows : u[0].rows;
    r.lo = t ? u[1].lo : u[0].lo, r.hi = t ? u[1].hi : u[0].hi;
    r.full0 = t ? u[1].full0 : u[0].full0, r.full1 = t ? u[1].full1 : u[0].full1;
    return r;
  }
  __device__ __forceinline__ void tile(int j, int& base, int& end) const {
    if (j < window_tiles) {
      base = lo + j * kKeys, end = hi;
    } else {
      base = (j - window_tiles) * kKeys, end = sink;
    }
    end = min(end, base + kKeys);
  }
  // The chunks [c0, c1) of 32 keys of a tile that a unit needs.
  __device__ __forceinline__ static void chunks(const Unit& u, int base, int end, int sinks, int& c0, int& c1) {
    const int w0 = max(base, u.lo), w1 = min(end, u.hi), s1 = min(end, min(sinks, u.hi));
    const bool window = w1 > w0, sinked = s1 > base;
    c0 = sinked ? 0 : (w0 - base) >> 5;
    const int last = max(window ? w1 : base, sinked ? s1 : base) - base;  // keys past the last needed one
    c1 = (last + 31) >> 5;
    if (last <= 0) c0 = c1 = 0;
  }
};

// Pairs of units over all requests: item -> (request, kv head, pair). A block's
// first kListed items are worked out once, in shared memory: every role reads
// them there instead of waiting for the request's offsets between two pairs.
struct Items {
  const int* before;   // items of the requests before each one, [requests + 1]
  const Pair* listed;  // items nth(0), nth(1), ...
  int batch, b;
  __device__ __forceinline__ Items(const int* s, const Pair* p, int n) : before(s), listed(p), batch(n), b(0) {}
  __device__ __forceinline__ int total() const { return before[batch]; }
  __device__ __forceinline__ Pair find(const AttnWindowArgs& a, int item) {
    while (item >= before[b + 1]) ++b;  // items only grow
    const int each = (before[b + 1] - before[b]) / a.kv_heads, in = item - before[b];
    const int pair = in / a.kv_heads;
    // the last queries, which see the most keys of a causal request, first: the
    // short pairs level the blocks at the end
    return Pair(a, b, in - pair * a.kv_heads, each - 1 - pair);
  }
  // The block's i-th item: every other round of the blocks runs backwards, so
  // that the blocks with the longest pairs of one round get the shortest of the
  // next (8192 causal queries when it came in: 178 us without, 167 with it).
  __device__ __forceinline__ int nth(int i) const {
    return i * (int)gridDim.x + (i & 1 ? (int)(gridDim.x - 1 - blockIdx.x) : (int)blockIdx.x);
  }
  __device__ __forceinline__ Pair at(const AttnWindowArgs& a, int i) {
    return i < kListed ? listed[i] : find(a, nth(i));
  }
};

static_assert(sizeof(Pair) == 96, "kListedBytes");

template <typename T>
constexpr uint32_t idesc_type() {
  return 0u;
}
template <>
constexpr uint32_t idesc_type<__nv_bfloat16>() {
  return (1u << 7) | (1u << 10);  // A and B bf16
}

__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// Bits first..last of a 32-bit word (either may lie outside).
__device__ __forceinline__ uint32_t bit_range(int first, int last) {
  const uint32_t from = first <= 0 ? 0xffffffffu : first > 31 ? 0u : 0xffffffffu << first;
  const uint32_t to = last >= 31 ? 0xffffffffu : last < 0 ? 0u : 0xffffffffu >> (31 - last);
  return from & to;
}

// One 32-byte store: a whole sector of a thread's own row. Rows are 16-byte
// aligned only; those that are not 32-byte aligned take two stores.
template <typename T>
__device__ __forceinline__ void store32(T* p, const uint32_t* v) {
  if (((uintptr_t)p & 31) == 0) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                 "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
  } else {
    reinterpret_cast<uint4*>(p)[0] = make_uint4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<uint4*>(p)[1] = make_uint4(v[4], v[5], v[6], v[7]);
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(384, 1)
    attention_tiles_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                           const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttnWindowArgs a) {
  using C = TilesCfg<D>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_s = dev::smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_s + 1023u) & ~1023u) - raw_s);
  uint8_t* sQ = smem;
  uint8_t* sKV = sQ + 2 * C::kQ;  // stage s: K at 2 s tiles, V behind it
  uint64_t* bars = reinterpret_cast<uint64_t*>(sKV + C::kStages * 2 * C::kTileBytes);
  const uint32_t q_full = dev::smem_u32(bars), q_empty = q_full + 8;
  // s_full, p_ready, pv_done: [unit][S tile]. One barrier for both S tiles would
  // not do: a side that is a tile behind cannot tell a phase from the next but one.
  const uint32_t s_full = q_full + 16, p_ready = s_full + 32, pv_done = p_ready + 32, mma_fin = pv_done + 32;
  const uint32_t kv_full = mma_fin + 8, kv_ready = kv_full + 8 * C::kStages, kv_empty = kv_ready + 8 * C::kStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 30);
  uint32_t* bad = tmem_slot + 1;  // some output of this block has to be looked at again
  Pair* listed = reinterpret_cast<Pair*>(bars + 32);
  uint32_t* redo = reinterpret_cast<uint32_t*>(bars + 32) + C::kListedBytes / 4;  // its rows: [item][unit][quarter]
  int* before = reinterpret_cast<int*>(redo) + C::kRedoBytes / 4;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (warp == 0 && lane == 0) {
    dev::prefetch_tmap(&map_q);
    dev::prefetch_tmap(&map_k);
    dev::prefetch_tmap(&map_v);
    dev::mbar_init(q_full, 1);
    dev::mbar_init(q_empty, 2);  // both units' warps
    for (int i = 0; i < 4; ++i) {
      dev::mbar_init(s_full + 8 * i, 1);
      dev::mbar_init(p_ready + 8 * i, 128);
      dev::mbar_init(pv_done + 8 * i, 1);
    }
    dev::mbar_init(mma_fin, 2);
    *bad = 0;
    for (int s = 0; s < C::kStages; ++s) {
      dev::mbar_init(kv_full + 8 * s, 1);
      dev::mbar_init(kv_ready + 8 * s, 1);
      dev::mbar_init(kv_empty + 8 * s, 2);
    }
    dev::fence_mbar_init();
  }
  // TMEM is taken only after the previous kernel of the stream has ended, and
  // the next one may start only once it is taken: neither can hold columns that
  // the other waits for.
  dev::pdl_wait();
  if (warp == 1) {
    dev::tmem_alloc(dev::smem_u32(tmem_slot), C::kTmemCols);
    dev::tmem_relinquish();
  }
  if (warp == 4) {
    // items of each request, summed by one warp
    const int group = a.q_heads / a.kv_heads;
    int sum = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 32) {
      const int b = b0 + lane;
      int n = 0;
      if (b < a.batch) {
        const int nq = min(AttnRequest(a, b).nq, a.max_q);
        n = ((nq + kRows - 1) / kRows * group + 1) / 2 * a.kv_heads;
      }
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, n, o);
        if (lane >= o) n += up;
      }
      if (b < a.batch) before[b + 1] = sum + n;
      sum += __shfl_sync(0xffffffffu, n, 31);
    }
    if (lane == 0) before[0] = 0;
  }
  dev::tc_fence_before();
  __syncthreads();
  dev::tc_fence_after();
  dev::pdl_launch_dependents();
  const uint32_t tmem = *tmem_slot;
  Items items(before, listed, a.batch);
  const int total = items.total();
  if (threadIdx.x < kListed) {
    Items mine(before, listed, a.batch);
    const int item = mine.nth(threadIdx.x);
    if (item < total) listed[threadIdx.x] = mine.find(a, item);
  }
  for (int i = threadIdx.x; i < C::kRedoBytes / 4; i += C::kThreads) redo[i] = 0;
  __syncthreads();

  if (warp == 0) {
    // ---- copies: the elected lane of the converged warp issues them ----
    int n = 0, issued_q = 0;  // K/V tiles and Q pairs issued
    bool ok = true;
    for (int i = 0; items.nth(i) < total && ok; ++i) {
      const Pair p = items.at(a, i);
      if (!p.tiles) continue;
      ok = __all_sync(0xffffffffu, dev::mbar_wait(q_empty, (issued_q & 1) ^ 1, a.err));
      if (!ok) break;
      if (dev::elect_one()) {
        dev::mbar_arrive_expect_tx(q_full, (p.u[1].rows ? 2 : 1) * C::kQ);
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (p.u[t].rows)
            for (int h = 0; h < D / 64; ++h)
              dev::tma_load_2d(dev::smem_u32(sQ + t * C::kQ + h * C::kQHalf), &map_q, p.u[t].head * D + h * 64,
                               p.rq.q0 + p.u[t].i0, q_full);
      }
      __syncwarp();
      ++issued_q;
      for (int j = 0; j < p.tiles; ++j, ++n) {
        const int st = n % C::kStages;
        ok = __all_sync(0xffffffffu, dev::mbar_wait(kv_empty + 8 * st, ((n / C::kStages) & 1) ^ 1, a.err));
        if (!ok) break;
        int base, end;
        p.tile(j, base, end);
        if (dev::elect_one()) {
          const uint32_t fb = kv_full + 8 * st, dk = dev::smem_u32(sKV + st * 2 * C::kTileBytes);
          const uint32_t dv = dk + C::kTileBytes;
          dev::mbar_arrive_expect_tx(fb, 2 * C::kTileBytes);
          for (int h = 0; h < D / 64; ++h)
            dev::tma_load_2d(dk + h * C::kHalf, &map_k, p.kvh * D + h * 64, p.rq.k0 + base, fb);
          for (int h = 0; h < D / 64; ++h)
            dev::tma_load_2d(dv + h * C::kHalf, &map_v, p.kvh * D + h * 64, p.rq.k0 + base, fb);
        }
        __syncwarp();
      }
    }
    // no copy of this block is in flight when it leaves
    if (issued_q) dev::mbar_wait(q_full, (issued_q - 1) & 1, a.err, 100000000ull);
    for (int i = n > C::kStages ? n - C::kStages : 0; i < n; ++i)
      dev::mbar_wait(kv_full + 8 * (i % C::kStages), (i / C::kStages) & 1, a.err, 100000000ull);
  } else if (warp <= 2) {
    // ---- products of unit t, by one thread. Step js of a pair: O += P . V of
    // tile js - 2, then S of tile js into the S tile that this P was in; the
    // tensor pipe runs them in the order of issue ----
    if (dev::elect_one()) {
      const int t = warp - 1;
      constexpr uint32_t kIdescO = dev::make_idesc_f16(kRows, D) | idesc_type<T>() | (1u << 16);  // V MN-major
      constexpr uint32_t kIdescS = dev::make_idesc_f16(kRows, 32) | idesc_type<T>();  // one chunk; N doubles for two
      constexpr uint32_t kN32 = 32u >> 3 << 17;
      const uint64_t desc_q = dev::make_sw128_desc(dev::smem_u32(sQ + t * C::kQ));
      const uint64_t desc_k = dev::make_sw128_desc(dev::smem_u32(sKV));
      const uint64_t desc_v = dev::make_sw128_desc_mn(dev::smem_u32(sKV + C::kTileBytes), C::kHalf, 1024);
      const uint32_t o_at = tmem + C::kColO + t * 128;
      constexpr uint32_t kWhole = kChunks << 2;  // the code of a tile that is needed whole
      uint32_t n = 0, nq = 0;                    // K/V tiles whose S, and Q pairs that, have been reached
      uint32_t s_count = 0, p_count = 0;         // S tiles issued, P tiles used
      bool ok = true;
      for (int i = 0; items.nth(i) < total && ok; ++i) {
        const Pair p = items.at(a, i);
        if (!p.tiles) continue;
        const Unit u = p.unit(t);
        if (!dev::mbar_wait(q_full, nq & 1, a.err)) break;
        ++nq;
        uint32_t begun = 0;  // O holds a product of this pair
        uint32_t codes = 0;  // chunks of the tiles js - 2, js - 1, js, a byte each: c0 | c1 << 2
        for (int js = 0; js < p.tiles + 2; ++js, ++n) {
          const uint32_t st_s = n % C::kStages, st_v = (n - 2) % C::kStages;
          codes >>= 8;
          if (js < p.tiles) {
            if (js >= u.full0 && js < u.full1) {
              codes |= kWhole << 16;
            } else {
              int base, end, c0, c1;
              p.tile(js, base, end);
              Pair::chunks(u, base, end, a.sinks, c0, c1);
              if (c0 < c1) codes |= (uint32_t)(c0 | c1 << 2) << 16;
            }
            ok = dev::mbar_wait(kv_ready + 8 * st_s, n / C::kStages & 1, a.err);
            if (!ok) break;
          }
          const uint32_t pv = codes & 15, sc = codes >> 16;
          if (pv) {
            const uint32_t at = 2 * t + (p_count & 1);
            ok = dev::mbar_wait(p_ready + 8 * at, p_count >> 1 & 1, a.err);
            if (!ok) break;
            dev::tc_fence_after();
            const uint32_t p_at = tmem + C::kColS + at * 64;
            const uint64_t v = desc_v + st_v * (2 * C::kTileBytes >> 4);
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
              if (pv != kWhole && (c < (int)(pv & 3) || c >= (int)(pv >> 2))) continue;
              dev::tc_mma_f16_ts(o_at, p_at + c * 16, v + c * (4096 >> 4), kIdescO, begun);
              dev::tc_mma_f16_ts(o_at, p_at + c * 16 + 8, v + c * (4096 >> 4) + (2048 >> 4), kIdescO, 1);
              begun = 1;
            }
            dev::tc_commit(pv_done + 8 * at);
            ++p_count;
          }
          if (sc) {
            // S for the keys of the chunks, at their own columns
            const uint32_t at = 2 * t + (s_count & 1);
            const uint32_t c0 = sc & 3, idesc = kIdescS + ((sc >> 2) - c0 - 1) * kN32;
            const uint32_t s_at = tmem + C::kColS + at * 64 + c0 * 32;
            const uint64_t k = desc_k + st_s * (2 * C::kTileBytes >> 4) + c0 * (4096 >> 4);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              dev::tc_mma_f16(s_at, desc_q + (kk >> 2) * (C::kQHalf >> 4) + (kk & 3) * 2,
                              k + (kk >> 2) * (C::kHalf >> 4) + (kk & 3) * 2, idesc, kk != 0 ? 1u : 0u);
            dev::tc_commit(s_full + 8 * at);
            ++s_count;
          }
          // every product of the unit that reads tile js - 2, or the pair's Q, has been issued
          if (js >= 2) dev::tc_commit(kv_empty + 8 * st_v);
          if (js == p.tiles - 1) dev::tc_commit(q_empty);
        }
        n -= 2;  // the last two steps had no S
      }
      dev::tc_commit(mma_fin);
    }
    __syncwarp();
    dev::mbar_wait(mma_fin, 0, a.err, 100000000ull);  // every product has retired before TMEM is freed
  } else if (warp == 3) {
    // ---- passes each K/V tile on to the products. Rows of V past a tile's last
    // key, up to the end of its 32-key chunk, are no request's or another one's:
    // their weights are 0, but they may hold infinities or NaN, so they become
    // zeros first ----
    uint32_t n = 0;
    bool ok = true;
    for (int i = 0; items.nth(i) < total && ok; ++i) {
      const Pair p = items.at(a, i);
      for (int j = 0; j < p.tiles; ++j, ++n) {
        const uint32_t st = n % C::kStages;
        ok = __all_sync(0xffffffffu, dev::mbar_wait(kv_full + 8 * st, n / C::kStages & 1, a.err));
        if (!ok) break;
        int base, end;
        p.tile(j, base, end);
        const int keys = end - base;
        if (keys & 31) {
          uint8_t* v = sKV + st * 2 * C::kTileBytes + C::kTileBytes;
          const int zero = ((keys + 31) & ~31) - keys;
          for (int i = lane; i < zero * 8 * (D / 64); i += 32) {
            const int h = i / (zero * 8), r = i % (zero * 8);
            *reinterpret_cast<uint4*>(v + h * C::kHalf + keys * 128 + r * 16) = make_uint4(0, 0, 0, 0);
          }
          dev::fence_proxy_async_smem();
          __syncwarp();
        }
        if (lane == 0) dev::mbar_arrive(kv_ready + 8 * st);
      }
    }
  } else {
    // ---- softmax of unit t: thread = query row ----
    const int t = (warp - 4) >> 2, quarter = warp & 3;
    const uint32_t rows_at = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t col_o = rows_at + C::kColO + t * 128;
    const float scale = a.scale * 1.4426950408889634f;  // scores in log2 units
    int count = 0;  // tiles of this unit so far, over all pairs
    bool ok = true;
    for (int i = 0; items.nth(i) < total && ok; ++i) {
      const Pair p = items.at(a, i);
      const Unit u = p.unit(t);
      if (!u.rows) continue;
      const int p_warp = u.i0 + quarter * 32 + p.rq.nk - p.rq.nq;
      const RowKeys mine(a, p_warp + lane, p.rq.nk), top(a, p_warp, p.rq.nk), bottom(a, p_warp + 31, p.rq.nk);
      // Window tiles [plain0, plain1) whose 64 keys every row of the warp sees.
      const int plain0 = (max(bottom.first - p.lo, 0) + kKeys - 1) / kKeys;
      const int plain1 = max(min(top.last + 1, u.hi) - p.lo, 0) / kKeys;
      float m = -INFINITY, l = 0.f;  // m: the reference of the weights
      int seen = 0;  // tiles of this pair
      for (int j = 0; j < p.tiles; ++j) {
        int base = 0, end = 0;
        uint32_t any = 3, whole = 3;  // chunks that some row sees, that every row sees whole
        if (j < plain0 || j >= plain1) {
          int c0, c1;
          p.tile(j, base, end);
          Pair::chunks(u, base, end, a.sinks, c0, c1);
          if (c0 >= c1) continue;
          any = whole = 0;
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            const int j0 = base + c * 32, j1 = j0 + 31;
            if (c >= c0 && c < c1 && j0 <= bottom.last && (j1 >= top.first || j0 < a.sinks)) any |= 1u << c;
            if (j1 <= top.last && j1 < end && (j0 >= bottom.first || j1 < a.sinks)) whole |= 1u << c;
          }
        }
        const int at = 2 * t + (count & 1);
        const uint32_t col_s = rows_at + C::kColS + at * 64;
        ok = __all_sync(0xffffffffu, dev::mbar_wait(s_full + 8 * at, count >> 1 & 1, a.err));
        if (!ok) break;
        dev::tc_fence_after();
        float s[kKeys];
        uint32_t pr[kKeys / 2];
        float2 sum = make_float2(0.f, 0.f), sum1 = sum;
        bool done = false;
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
          dev::tmem_ld_32x32b_x32(col_s + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&s[c * 32]));
        dev::tc_wait_ld();
        // A tile that every row sees takes its weights against the reference that
        // it has straight away. They stand if every row's sum is at most 2^15 (with 2^8 as
        // the limit more tiles go twice: 106 us for 102): then no
        // weight is above that either, inside the 16-bit types, and O needs no
        // rescaling. Otherwise the tile's own maximum is found, the reference
        // moves and the weights are taken again. (A NaN fails the comparison.)
        if (any == 3 && whole == 3 && seen) {
#pragma unroll
          for (int i = 0; i < kKeys; i += 2) {
            const float2 x = dev::fma2(make_float2(s[i], s[i + 1]), make_float2(scale, scale), make_float2(-m, -m));
            const float2 e = make_float2(dev::exp2_approx(x.x), dev::exp2_approx(x.y));
            if (i & 2) sum1 = dev::add2(sum1, e);
            else sum = dev::add2(sum, e);
            pr[i / 2] = dev::pack2<T>(e.x, e.y);
          }
          sum = dev::add2(sum, sum1);
          done = __all_sync(0xffffffffu, sum.x + sum.y <= kMaxSum);
        }
        if (!done) {
          sum = make_float2(0.f, 0.f);
          float part[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            if (!(any >> c & 1)) continue;
            if (!(whole >> c & 1)) {
              const int j0 = base + c * 32, last = min(mine.last, end - 1) - j0;
              const uint32_t bits = bit_range(mine.first - j0, last) | bit_range(0, min(last, a.sinks - 1 - j0));
#pragma unroll
              for (int i = 0; i < 32; ++i) s[c * 32 + i] = bits >> i & 1 ? s[c * 32 + i] : -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < 32; i += 8)
#pragma unroll
              for (int k = 0; k < 4; ++k) part[k] = dev::max3(part[k], s[c * 32 + i + 2 * k], s[c * 32 + i + 2 * k + 1]);
          }
          const float tmax = scale * fmaxf(dev::max3(part[0], part[1], part[2]), part[3]);
          const bool move = __any_sync(0xffffffffu, tmax > m + (whole == 3 ? weight_lift<T>() : kMaxSlack));
          const float mnew = move ? fmaxf(m, tmax - weight_lift<T>()) : m;
          const float neg = mnew == -INFINITY ? 0.f : -mnew;  // no key seen yet: all weights 0
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            if (any >> c & 1) {
#pragma unroll
              for (int i = c * 32; i < c * 32 + 32; i += 2) {
                const float2 x = dev::fma2(make_float2(s[i], s[i + 1]), make_float2(scale, scale), make_float2(neg, neg));
                const float2 e = make_float2(dev::exp2_approx(x.x), dev::exp2_approx(x.y));
                sum = dev::add2(sum, e);
                pr[i / 2] = dev::pack2<T>(e.x, e.y);
              }
            } else {
#pragma unroll
              for (int i = 0; i < 16; ++i) pr[c * 16 + i] = 0;
            }
          }
          if (move) {
            const float keep = m == -INFINITY ? 0.f : dev::exp2_approx(m - mnew);
            l *= keep;
            m = mnew;
            if (seen) {
              // O is stable once the previous tile's P.V is complete (the one
              // before that is: this tile's S was issued after it)
              ok = __all_sync(0xffffffffu, dev::mbar_wait(pv_done + 8 * (at ^ 1), (count - 1) >> 1 & 1, a.err));
              if (!ok) break;
              dev::tc_fence_after();
#pragma unroll
              for (int c = 0; c < D / 16; ++c) {
                uint32_t o[16];
                dev::tmem_ld_32x32b_x16(col_o + c * 16, o);
                dev::tc_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
                tmem_st_x16(col_o + c * 16, o);
              }
            }
          }
        }
        dev::tmem_st_32x32b_x32(col_s, pr);
        dev::tc_wait_st();
        l += sum.x + sum.y;
        dev::tc_fence_before();
        dev::mbar_arrive(p_ready + 8 * at);
        ++seen;
        ++count;
      }
      if (!ok) break;
      if (seen) {
        ok = __all_sync(0xffffffffu,
                        dev::mbar_wait(pv_done + 8 * (2 * t + ((count - 1) & 1)), (count - 1) >> 1 & 1, a.err));
        if (!ok) break;
        dev::tc_fence_after();
      }
      // output: O / l, one row per thread in 32-byte stores
      const float inv = l == 0.f ? 0.f : 1.0f / l;
      const int row = u.i0 + quarter * 32 + lane;
      const bool live = quarter * 32 + lane < u.rows;
      T* out = static_cast<T*>(a.out) + (int64_t)(p.rq.q0 + row) * a.ldo + u.head * D;
      float2 probe = make_float2(0.f, 0.f);  // stays 0 unless some value is infinite or NaN
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        float o[32];
        if (seen) {
          dev::tmem_ld_32x32b_x32(col_o + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&o[0]));
          dev::tc_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0.f;
        }
        uint32_t v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float2 y = dev::fma2(make_float2(o[2 * i], o[2 * i + 1]), make_float2(inv, inv), make_float2(0.f, 0.f));
          probe = dev::fma2(y, make_float2(0.f, 0.f), probe);
          // (a mean of finite values is no larger than they are; the rounded weights' product may be, by half a step)
          v[i] = dev::pack2_finite<T>(y.x, y.y);
        }
        if (live) {
          store32(out + c * 32, v);
          store32(out + c * 32 + 16, v + 8);
        }
      }
      const bool odd = live && !(probe.x + probe.y == 0.f);
      if (__any_sync(0xffffffffu, odd)) {
        // Such rows are written with their infinities, and rows without a key of any weight with zeros (O may
        // hold 0 times anything there). A sum that is NaN is a score that is NaN or +infinity, of a key that the
        // row sees: so is the row. Others are looked at again.
#pragma unroll 1
        for (int c = 0; c < D; c += 16) {
          uint32_t o[16];
          dev::tmem_ld_32x32b_x16(col_o + c, o);
          dev::tc_wait_ld();
          if (odd) {
#pragma unroll
            for (int k = 0; k < 16; k += 8) {
              float y[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) y[e] = l == 0.f ? 0.f : __uint_as_float(o[k + e]) * inv;
              *reinterpret_cast<uint4*>(out + c + k) = dev::pack8<T>(y);
            }
          }
          __syncwarp();
        }
        const uint32_t again = __ballot_sync(0xffffffffu, odd && l > 0.f);
        if (lane == 0 && again) {
          *bad = 1;
          if (i < kListed) redo[(i * 2 + t) * 4 + quarter] = again;
        }
      }
      dev::tc_fence_before();  // orders the loads above before the next arrival on p_ready
    }
  }
  dev::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    dev::tc_fence_after();
    dev::tmem_dealloc(tmem, C::kTmemCols);
  }
  if (!*bad) return;
  // Some row met an infinity or NaN, perhaps one that it does not see (weight 0
  // times the value): rows whose result is not finite are looked at again.
  Items again(before, listed, a.batch);
  for (int i = 0; again.nth(i) < total; ++i) {
    const Pair p = again.at(a, i);
#pragma unroll 1
    for (int t = 0; t < 2; ++t) {
      const Unit u = p.unit(t);
      for (int r = warp; r < u.rows; r += C::kThreads / 32) {
        if (i < kListed && !(redo[(i * 2 + t) * 4 + (r >> 5)] >> (r & 31) & 1)) continue;
        const T* out = static_cast<const T*>(a.out) + (int64_t)(p.rq.q0 + u.i0 + r) * a.ldo + u.head * D;
        bool wrong = false;
        for (int c = lane; c < D; c += 32) wrong |= !isfinite(dev::to_f32(out[c]));
        if (__any_sync(0xffffffffu, wrong)) attention_row<T, D>(a, p.rq, u.i0 + r, u.head, 0, D);
      }
    }
  }
}

}  // namespace

template <typename T, int D>
static cudaError_t launch_tiles(AttnWindowArgs a, cudaStream_t s) {
  using C = TilesCfg<D>;
  auto kernel = attention_tiles_kernel<T, D>;
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
  CUtensorMap mq, mk, mv;
  if (make_tmap_16bit(&mq, a.q, (uint64_t)a.q_heads * D, a.q_rows, a.ldq * 2, 64, kRows) ||
      make_tmap_16bit(&mk, a.k, (uint64_t)a.kv_heads * D, a.k_rows, a.ldk * 2, 64, kKeys) ||
      make_tmap_16bit(&mv, a.v, (uint64_t)a.kv_heads * D, a.k_rows, a.ldv * 2, 64, kKeys))
    return cudaErrorInvalidValue;
  const int group = a.q_heads / a.kv_heads;
  const int64_t pairs = (((int64_t)a.max_q + kRows - 1) / kRows * group + 1) / 2 * a.kv_heads;
  const int batch = a.batch;
  for (int b = 0; b < batch; b += kMaxRequests) {
    a.batch = batch - b < kMaxRequests ? batch - b : kMaxRequests;
    const int64_t items = pairs * a.batch;
    e = launch_overlapped(kernel, dim3((unsigned)(items < a.sms ? items : a.sms)), dim3(C::kThreads), C::kSmem, s,
                          dim3(1, 1), mq, mk, mv, a);
    if (e != cudaSuccess) return e;
    a.q_off += kMaxRequests, a.k_start += kMaxRequests, a.k_len += kMaxRequests;
  }
  return cudaSuccess;
}

// Keys that `rows` consecutive queries see, at most.
int64_t visible_keys(const AttnWindowArgs& a, int rows) {
  int64_t keys = a.max_k;
  if (a.left >= 0) {
    const int64_t window = (int64_t)a.left + (a.right > 0 ? a.right : a.right < 0 ? a.max_k : 0) + rows + a.sinks;
    if (window < keys) keys = window;
  }
  return keys;
}

// Prompts and documents run on the 128-row tiles, few queries on 16-row ones,
// whichever a model of both calls faster: 4 us + (row tiles x keys of all requests)
// over a rate for the 16-row kernel, 5 us + a time for each step of 64 keys and
// round of pairs over the SMs for this one. Measured with 24 + 8 heads, us (16-row
// against this), queries on keys of 128, then of 64 columns: 16 x 8 on 1500 32 / 53
// and 34 / 49, 16 x 32 89 / 53 and 55 / 50, 4 x 64 on 4096 112 / 65 and 71 / 61,
// 1 x 64 on 16384 112 / 238 and 74 / 223, 1 x 128 206 / 239 and 135 / 224, 1 x 256
// 394 / 239 and 259 / 226; 8 x 2 on 56 of 64 columns 4.0 / 6.6.
bool attention_on_tiles(const AttnWindowArgs& a) {
  const int group = a.q_heads / a.kv_heads;
  const double row_tiles = (double)(((int64_t)a.max_q * group + 15) / 16) * a.kv_heads * a.batch;
  const double pairs = (double)((((int64_t)a.max_q + kRows - 1) / kRows * group + 1) / 2) * a.kv_heads * a.batch;
  const double rate = a.head_dim == 64 ? 23500 : 15000, step = a.head_dim == 64 ? 0.86 : 0.92;
  const double few = 4 + row_tiles * visible_keys(a, 16) / rate;
  const double many = 5 + ceil(pairs / a.sms) * visible_keys(a, kRows + kKeys) * (step / kKeys);
  return few > many && a.k_rows > 0;
}

cudaError_t launch_attention_window(const AttnWindowArgs& a, cudaStream_t s) {
  if (!attention_on_tiles(a)) return launch_attention_rows(a, s);
  if (a.head_dim == 64)
    return a.dtype == kDtBF16 ? launch_tiles<__nv_bfloat16, 64>(a, s) : launch_tiles<__half, 64>(a, s);
  return a.dtype == kDtBF16 ? launch_tiles<__nv_bfloat16, 128>(a, s) : launch_tiles<__half, 128>(a, s);
}

}  // namespace nemo
