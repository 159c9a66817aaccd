// Attention of chunks of new tokens over a paged cache on the 5th-generation tensor
// cores: bf16 / f16 queries, head_dim 64 or 128, caches of the query's type (staged by
// TMA) or of e4m3 rows (converted while they are staged).
//
// A unit (chunk_plan.cuh) has up to 256 query rows of one kv head as two tiles of 128 (M), and
// a step takes 128 keys:
//   S = Q K^T [128 x 128] (Q and K K-major), P = 2^(S c - m), O += P V (V MN-major).
// Softmax and MMA of the two tiles alternate: while the tensor core works on one tile's
// products, the other tile's 128 threads (one row each) take its scores.
// A row keeps a reference that is raised only when a score exceeds it by 2^8 (f16: 2^15): then O is
// rescaled in TMEM, else O is never touched between the products.
//   warps 0-3, 4-7  softmax of tile 0 / 1: thread = row = TMEM lane; they write P to shared memory,
//                   and write out the finished rows
//   warp 8          loads Q (one copy per tile and 64 columns: 128 threads fetching rows took 14000
//                   cycles a unit), issues the MMAs of the scores
//   warps 9, 10     stage K and V by TMA
//   warp 11         issues the MMAs of P V: a wait takes some 200 cycles next to operand reads that fill
//                   shared memory's bandwidth, and the two streams cover each other's; in tiles that
//                   only some of a unit's queries see it takes infinities and NaN out of V before
//   warps 12-15     8-bit caches only: turn the staged rows into 16-bit stages
// P goes through shared memory, not through TMEM as an A operand: a kernel of this library that
// read A from TMEM ended in a launch failure whose cause was not found.
//   TMEM: S of tile 0 / 1 at columns 0 / 128, O at 256 / 256 + head_dim.
//   Shared memory: Q 2 x [128 x D], P [128 x 128], a ring of [128 x D] stages of K and one of V (128-byte
//   swizzle everywhere).  The tiles share one P buffer: a tile's P is written after the other's
//   product has read its own, which costs nothing while the tiles take turns, and the 32 KB are a
//   fourth stage (with three, every V was still on its way when it was needed: 4050 cycles a step of
//   2 x 128 x 128 scores).  Every ring has one producer and one consumer that go through it in
//   order, so a barrier's parity always tells the phase that is meant.
// Every wait is bounded and ends early once another role gave up; TMEM is released on
// every path.
// What bounds it is shared memory: a step of 2 x 128 x 128 scores reads 4 x 64 KB of operands, writes 64 KB of P
// and receives 64 KB of K and V, 3070 cycles at 128 bytes each (measured 3200 to 3300; the products
// themselves take 2048).  2048 new tokens behind 30720 cached ones, 32 heads over 8 of 128: 987 us, 1080
// TFLOP/s (replayed from a graph, as the other times here; back to back from Python, under the power
// cap, 1140 us).  Short units add 20000 cycles at the start of a CTA and 12000 a piece (a mixed step
// 176 us, 760 TFLOP/s).  Over 8-bit rows the converting warps add 48 KB a tile to the same traffic: 2700
// cycles a tile, 2000 of them without any conversion, 118 us and 493 TFLOP/s for a step of four
// chunks; fewer instructions, rows fetched ahead and conversions by bit operations did not help.
// Instructions count even where they do not run (the softmax loop is long, and what it and the other roles
// fetch from L2 is waited for): the handling of keys without a block costs 1 to 2% of every call,
// that of infinities in V up to 2.5% of a step of 8-bit chunks.
#include <cuda.h>

#include "chunk_plan.cuh"
#include "pairs.cuh"
#include "sm100.cuh"

namespace snapmind {
namespace {

using namespace tc;

constexpr int kTileM = 128, kKeys = 128;
constexpr int kConvert = 128;  // threads that convert e4m3 rows
constexpr uint32_t kBlockBytes = 128 * 128;  // 128 rows of 64 16-bit elements
constexpr uint32_t kPBytes = 2 * kBlockBytes;
// A raised reference stands 2^kLow below the maximum, and stays until a score exceeds it by 2^kRescale.
// f16 weights go up to 2^15: a weight 2^25 below a largest one of 1 would vanish, and the weights of
// thousands of keys behind a strong sink lie there; 2^7 further up, a weight is off by 2^-32 of the
// largest at most.
template <typename T> constexpr float kLow = std::is_same<T, __half>::value ? 7.f : 0.f;
template <typename T> constexpr float kRescale = kLow<T> + 8.f;

template <int D, bool kQuant> struct Shape {
  static constexpr uint32_t kTileBytes = D / 64 * kBlockBytes;  // a Q tile, a K or V stage
  static constexpr int kK = D == 64 ? 4 : 2, kV = kK - (kQuant ? 1 : 0);  // stages
  static constexpr uint32_t kRawBytes = kQuant ? 128 * D : 0;             // codes of a K or V tile
  static constexpr uint32_t kP = 2 * kTileBytes, kRing = kP + kPBytes;    // K's stages, then V's
  static constexpr uint32_t kRaw = kRing + (kK + kV) * kTileBytes, kCtrl = kRaw + 2 * kRawBytes;
  // K and V stages are [8-row group][64-column block][8 rows x 128 bytes]
  static constexpr uint32_t kGroup = D / 64 * 1024;
  // Stage and parity of the K (0) or V (1) tile with running number i.
  __device__ __forceinline__ static int stage(int kv, uint32_t i) { return kv == 0 ? i % kK : i % kV; }
  __device__ __forceinline__ static uint32_t parity(int kv, uint32_t i) { return (kv == 0 ? i / kK : i / kV) & 1; }
  __device__ __forceinline__ static uint32_t at(int kv, uint32_t i) { return kRing + (kv * kK + stage(kv, i)) * kTileBytes; }
};

struct Ctrl {
  uint64_t full[2][4], empty[2][4];  // K's and V's stages
  uint64_t q_full;      // the Q tiles of a piece have landed
  uint64_t s_full[2];   // MMA commit: scores ready
  uint64_t s_free[2];   // softmax threads: scores read (the group's next ones may replace them)
  uint64_t p_full[2];   // softmax threads: P written
  uint64_t pv_done[2];  // MMA commit: O += P V done
  uint64_t x_ml;        // split: group 1's maxima and sums are in `ml`, its O is final
  uint64_t x_done;      // split: group 0 has read them
  uint64_t raw_full[2], raw_empty[2];  // e4m3: codes and scales of a K / V tile
  uint64_t v_ready[2];  // MMA warp: V of an edge tile has landed (its unseen rows may be zeroed)
  uint32_t tmem_base;
  int32_t abort;
  // A K tile i with parts whose table entry is no block: its number and a bit per lost key, at i % 8.  (Its
  // scores are read before the loading warp is 8 tiles on: it waits for the products of 4 tiles ago, which
  // wait for the softmax threads to have read scores.)
  uint32_t lost_tile[8], lost[8][4];
  int32_t any_lost;  // there was one
  int32_t any_odd;  // values of V were taken out (in this piece, or one before)
  int32_t odd;  // f16 over e4m3: a row that f16 does not hold was met
  PlanShared plan;
  alignas(16) uint8_t scales[2][128];
  float2 ml[128];
};

static_assert(offsetof(Ctrl, scales) % 16 == 0, "16-byte copies land there");

template <int D, bool kQuant> constexpr size_t smem_bytes() { return 1024 + Shape<D, kQuant>::kCtrl + sizeof(Ctrl); }
static_assert(smem_bytes<128, false>() <= 232448 && smem_bytes<128, true>() <= 232448, "shared memory budget");
static_assert(smem_bytes<64, false>() <= 232448 && smem_bytes<64, true>() <= 232448, "shared memory budget");
static_assert(kPBytes >= kMaxChunkBatch * 4, "plan scratch in the P tiles");

// Rare, so not inlined: one bit per key of the parts `missing` (2^log_box keys each) of tile `tile`.
__device__ __noinline__ void mark_lost(Ctrl& C, uint32_t tile, uint32_t missing, int log_box) {
  if (!C.any_lost)
    for (int i = 0; i < 8; ++i) C.lost_tile[i] = ~0u;
  uint32_t* lost = C.lost[tile % 8];
#pragma unroll 1
  for (int key = 0; key < kKeys; key += 8) {
    if (key % 32 == 0) lost[key / 32] = 0;
    if (missing >> (key >> log_box) & 1) lost[key / 32] |= 0xFFu << (key % 32);
  }
  C.lost_tile[tile % 8] = tile;
  __threadfence_block();
  C.any_lost = 1;
}
__device__ __forceinline__ void give_up(Ctrl& C, int32_t* err) {
  atomicExch(&C.abort, 1);
  flag_error(err, SNAPMIND_DEVERR_TIMEOUT);
}

// The lowest k bits (none for k <= 0, all for k >= 32).
__device__ __forceinline__ uint32_t low_bits(int k) { return k <= 0 ? 0u : k >= 32 ? ~0u : (1u << k) - 1u; }
// A piece whose rows all fit tile 0 runs split: both softmax groups take tile 0's rows, group t
// the key tiles t, t + 2, ..., each with sums and an O of its own, added up at the end.

// Whether a key tile holds rows that no query of the unit sees: [u_s, u_lo) and from v_len on, on the
// virtual axis.  Their V is zeroed: a weight of 0 times an infinity or NaN would reach O.
struct EdgeTiles {
  int v_len, u_s, u_lo;
  __device__ __forceinline__ EdgeTiles(const ChunkParams& p, const KeyRange& r)
      : v_len(r.v_len), u_s(p.window > 0 ? min(p.sinks, r.v_sink) : 0), u_lo(r.win_lo - r.shift) {}
  __device__ __forceinline__ bool operator()(int tile) const {
    const int v0 = tile * kKeys;
    return v0 + kKeys > v_len || (v0 < u_lo && v0 + kKeys > u_s);
  }
  __device__ __forceinline__ bool unseen(int v) const { return v >= v_len || (v < u_lo && v >= u_s); }
};
// Rows that some queries of the unit see and others do not, from hi0 on and in [lo0, lo1): of their V
// the values that are not finite are taken out for the same reason, and the rows that see them get
// them at the end (add_odd).
struct MixedKeys {
  int hi0, hi1, lo0, lo1;
  __device__ __forceinline__ MixedKeys(const ChunkParams& p, const KeyRange& r, int tokens)
      : hi0(min(max(0, r.pos0 + 1 - r.shift), r.v_len)), hi1(r.v_len),
        lo0(p.window > 0 ? max(r.win_lo - r.shift, min(p.sinks, r.v_sink)) : 0),
        lo1(p.window > 0 ? max(0, r.pos0 + tokens - p.window) - r.shift : 0) {}
  __device__ __forceinline__ bool operator()(int v) const { return (v >= hi0 && v < hi1) || (v >= lo0 && v < lo1); }
  // Rows [first, last) of the tile at v0 hold all of its mixed keys.
  __device__ __forceinline__ int first(int v0) const {
    const int a = max(v0, hi0), b = max(v0, lo0);
    return min(a < hi1 ? a : INT32_MAX, b < lo1 ? b : INT32_MAX) - v0;
  }
  __device__ __forceinline__ int last(int v0) const {
    const int end = v0 + kKeys, a = min(end, hi1), b = min(end, lo1);
    return max(a > hi0 ? a : 0, b > lo0 ? b : 0) - v0;
  }
};

// 32 bytes, one sector, in one store (a lane stores a row of its own: with 16 bytes a store, a mixed
// step took 172 us, not 167).
__device__ __forceinline__ void store32(void* p, const uint32_t* x) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(x[0]), "r"(x[1]), "r"(x[2]),
               "r"(x[3]), "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7])
               : "memory");
}

// The tiles that hold such rows (and, below the last of a window's, others).
struct MixedTiles {
  int from, below;
  __device__ __forceinline__ explicit MixedTiles(const MixedKeys& m)
      : from(m.hi0 < m.hi1 ? m.hi0 / kKeys : INT32_MAX), below(m.lo0 < m.lo1 ? (m.lo1 + kKeys - 1) / kKeys : 0) {}
  __device__ __forceinline__ bool has(int tile) const { return tile >= from || tile < below; }
};

// 16 e4m3 codes of one row times 2^(byte - 127), as 16 elements of T.  The scale is a power of two:
// exact in bf16, and in f16 unless odd_row says otherwise.
template <typename T>
__device__ __forceinline__ void dequant16(const uint4& codes, uint32_t byte, uint4& lo, uint4& hi) {
  const float s = scale_byte_to_f(byte);
  const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
  uint32_t o[8];
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    uint32_t h[2];
    codes_f16(w[i / 2], h[0], h[1]);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float2 f = mul2(__half22float2(*reinterpret_cast<const __half2*>(&h[j])), s);
      o[i + j] = pack2<T>(f.x, f.y);
    }
  }
  lo = make_uint4(o[0], o[1], o[2], o[3]);
  hi = make_uint4(o[4], o[5], o[6], o[7]);
}

// Takes the infinities and NaN out of the mixed rows of the V stage of the tile whose first key is v0, by one
// warp; whether the lane met one.  Short code on purpose: it runs once or twice a unit, and instructions that
// come from L2 cost more than rounds of a loop (unrolled by 4 it took 4% of a step of chunks).
template <typename T, int D>
__device__ __forceinline__ bool take_odd(const MixedKeys& mixed, int v0, int lane, uint8_t* stage) {
  constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7C007C00u : 0x7F807F80u;  // an exponent of all ones
  constexpr uint32_t carry = std::is_same<T, __half>::value ? 0x04000400u : 0x00800080u;  // carries into the sign's place
  const int last = mixed.last(v0) * (D / 8);
  bool odd = false;
#pragma unroll 1
  for (int i = max(0, mixed.first(v0)) * (D / 8) + lane; i < last; i += 32) {  // 16 bytes of row r
    const int r = i / (D / 8), x = i % (D / 8);
    uint4* at = reinterpret_cast<uint4*>(stage + (r >> 3) * Shape<D, false>::kGroup + x / 8 * 1024 + (r & 7) * 128 + x % 8 * 16);
    const uint4 y = *at;
    if (((((y.x & e) + carry) | ((y.y & e) + carry) | ((y.z & e) + carry) | ((y.w & e) + carry)) & 0x80008000u) && mixed(v0 + r)) {
      uint32_t* w = reinterpret_cast<uint32_t*>(at);
#pragma unroll 1
      for (int k = 0; k < 4; ++k) w[k] &= ~((((w[k] & e) + carry) >> 15 & 0x00010001u) * 0xFFFFu);
      odd = true;
    }
  }
  return odd;
}

// Adds to an output row (`out`, or a piece's partial row) the infinities and NaN that were taken out of V: those of
// the piece's keys that token `tok` of the unit sees and another does not.  The rows of V come from
// the pool once more; nothing of this runs unless there is such a value.
template <typename T, int D, bool kQuant>
__device__ __noinline__ void add_odd(const ChunkParams& p, const Piece c, int tok, T* out, float* part) {
  const int tokens = min(p.tokens, c.n - c.i0);
  const KeyRange kr = key_range(p, c.len, c.n, c.i0, c.i0 + tokens);
  const MixedKeys mixed(p, kr, tokens);
  const int qpos = kr.pos0 + tok;
  const int32_t* table = p.tables + (int64_t)c.b * p.table_stride;
  for (int v = c.tile0 * kKeys; v < min(kr.v_len, c.tile1 * kKeys); ++v) {
    if (!mixed(v)) {
      if (v >= mixed.lo1 && v < mixed.hi0) v = mixed.hi0 - 1;
      continue;
    }
    const int pos = kr.position(v), j = p.by_block.div(pos);
    if (pos > qpos || (p.window > 0 && pos <= qpos - p.window && pos >= p.sinks)) continue;
    const int32_t phys = table[j];
    if (phys < 0 || phys >= p.num_blocks) continue;
    const int64_t tile = (int64_t)phys * p.n_kv_heads + c.kvh;
    const int64_t row = tile * p.block_size + (pos - j * p.block_size);
    const float scale = kQuant ? scale_byte_to_f(p.scales[row + tile * p.block_size + p.block_size]) : 1.f;
    for (int d = 0; d < D; ++d) {
      float x;
      if constexpr (kQuant) {
        x = Conv<T>::to_f(Conv<T>::from_f(e4m3_to_f(reinterpret_cast<const uint8_t*>(p.v_pool)[row * D + d]) * scale));
      } else {
        x = Conv<T>::to_f(reinterpret_cast<const T*>(p.v_pool)[row * D + d]);
      }
      if (fabsf(x) < INFINITY) continue;
      if (part != nullptr) part[d] += x;
      else out[d] = Conv<T>::from_f(Conv<T>::to_f(out[d]) + x);
    }
  }
}

// f16 over e4m3 rows.  K is staged times 2^5, which the scores' factor takes back, so that f16 holds
// it exactly for exponents from -20 (its smallest code is 2^-9 and f16's smallest number 2^-24) to 2
// (largest values of a row from 2e-4 to 1800); V as it is, for exponents up to 7, and up to 8 unless
// its values pass f16's largest.  (Smaller V lose at most 2^-25, half a step of the smallest f16 output.)
// A row outside that, zeros aside, makes the call odd: its results are of no use, and the CUDA-core
// kernel, which takes any exponent, does the call over.
template <typename T, bool kQuant> constexpr int kKeyUp = kQuant && std::is_same<T, __half>::value ? 5 : 0;
__device__ __forceinline__ bool odd_byte(int kv, uint32_t byte) { return kv == 0 ? byte - 107u > 22u : byte > 134u; }
__device__ __forceinline__ bool odd_row(int kv, const uint4& codes, const uint4& lo, const uint4& hi) {
  if (kv == 0) return ((codes.x | codes.y | codes.z | codes.w) & 0x7F7F7F7Fu) != 0;
  const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  uint32_t top = 0;  // an exponent of all ones carries into the sign's place
#pragma unroll
  for (int i = 0; i < 8; ++i) top |= (w[i] & 0x7C007C00u) + 0x04000400u;
  return (top & 0x80008000u) != 0;
}

// The third warpgroup (e4m3: and the fourth) gives up registers that the softmax threads, with a row
// of 128 scores each, need: 3 x 128 threads are launched with 168 each, 4 x 128 with 128.
template <bool kQuant> struct Roles {
  static constexpr int kThreads = kQuant ? 512 : 384, kLaunchRegs = kQuant ? 128 : 168;
  static constexpr int kScores = 8, kValues = 11, kLoad = 9, kConvertWarp = 12;
  static constexpr int kOther = kQuant ? 72 : 104, kSoftmax = kQuant ? 184 : 200;
  static_assert((kThreads - 256) * kOther + 256 * kSoftmax <= kThreads * kLaunchRegs, "register split");
};
template <int N> __device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }

// kStats: the rows' softmax sums go to p.stats.
template <typename T, int D, bool kQuant, bool kStats>
__global__ void __launch_bounds__(Roles<kQuant>::kThreads, 1)
    chunk_umma_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                      const __grid_constant__ CUtensorMap v_map, const __grid_constant__ CallParams<kStats> p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  using Sh = Shape<D, kQuant>;
  using Ro = Roles<kQuant>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t kIdescS = idesc_f16(kBf16, kTileM, kKeys, false, false);
  constexpr uint32_t kIdescO = idesc_f16(kBf16, kTileM, D, false, true);
  uint8_t* q_s = base;
  uint8_t* p_s = base + Sh::kP;
  Ctrl& C = *reinterpret_cast<Ctrl*>(base + Sh::kCtrl);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < 2 * Sh::kK; ++i) {
      mbar_init(smem_u32(&C.full[i & 1][i >> 1]), kQuant ? kConvert : 1);
      mbar_init(smem_u32(&C.empty[i & 1][i >> 1]), 1);
    }
    for (int kv = 0; kv < 2; ++kv) {
      mbar_init(smem_u32(&C.raw_full[kv]), 1 + 32);
      mbar_init(smem_u32(&C.raw_empty[kv]), kConvert);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(smem_u32(&C.s_full[t]), 1);
      mbar_init(smem_u32(&C.s_free[t]), 128);
      mbar_init(smem_u32(&C.p_full[t]), 128);
      mbar_init(smem_u32(&C.pv_done[t]), 1);
      mbar_init(smem_u32(&C.v_ready[t]), 1);
    }
    mbar_init(smem_u32(&C.q_full), 1);
    mbar_init(smem_u32(&C.x_ml), 128);
    mbar_init(smem_u32(&C.x_done), 128);
    C.abort = C.odd = 0;
    C.any_lost = C.any_odd = 0;
    mbar_init_fence();
  }
  if (warp == Ro::kScores) {
    tmem_alloc(smem_u32(&C.tmem_base), 512);
    tmem_relinquish();
  }
  prior_grid_wait();
  plan_block(p, C.plan, reinterpret_cast<int32_t*>(p_s));
  // rows of Q that no copy fills (128 / gw has a remainder) are zeros, not whatever lay there
  for (uint32_t i = tid; i < 2 * Sh::kTileBytes / 16; i += Ro::kThreads) reinterpret_cast<uint4*>(q_s)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = C.tmem_base;

  PieceWalk w;
  bool on = w.start(C.plan);
  if (warp >= Ro::kScores) {
    regs_dec<Ro::kOther>();
    if (kQuant && warp >= Ro::kConvertWarp) {
      // ------------------------------------------------------------------ e4m3 rows -> 16-bit stages
      // In the order in which the products need them: the first K tiles (1, split 2), then K(j + ahead),
      // while there is one, and V(j).  D / 16 threads share a row, 16 codes each.
      constexpr int kLanes = D / 16, kRowsPass = kConvert / kLanes;
      const int ct = tid - Ro::kConvertWarp * 32, ch = ct % kLanes, r0 = ct / kLanes;
      const uint32_t c0 = (ch % 4) * 2;
      const bool swap = ch >= 4;
      uint32_t tiles = 0;
      bool ok = true;
      for (; on && ok; on = w.next(p)) {
        const Piece& c = w.c;
        const int i1 = min(c.n, c.i0 + p.tokens), n = c.tile1 - c.tile0;
        const EdgeTiles edge(p, key_range(p, c.len, c.n, c.i0, i1));
        const int ahead = i1 - c.i0 <= p.tokens / 2 ? 2 : 1, lead = min(n, ahead);
        for (int i = 0; i < 2 * n; ++i) {
          const int x = i - lead;
          const int kv = x < 0 ? 0 : (x < 2 * (n - lead) ? x & 1 : 1);
          const int j = x < 0 ? i : (x < 2 * (n - lead) ? x / 2 + (kv ? 0 : ahead) : x - (n - lead));
          const uint32_t num = tiles + j;
          const int st = Sh::stage(kv, num);
          ok = role_wait(C.abort, smem_u32(&C.raw_full[kv]), num & 1) &&
               role_wait(C.abort, smem_u32(&C.empty[kv][st]), Sh::parity(kv, num) ^ 1);
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            break;
          }
          const uint8_t* raw = base + Sh::kRaw + kv * Sh::kRawBytes + ch * 16;
          uint8_t* dst = base + Sh::at(kv, num) + (ch / 4) * 1024;
          const int v0 = (c.tile0 + j) * kKeys;
          const bool edges = edge(c.tile0 + j);
#pragma unroll 1
          for (int r = r0; r < 128; r += kRowsPass) {
            uint4 codes = *reinterpret_cast<const uint4*>(raw + r * D);
            uint32_t byte = C.scales[kv][r];
            if (edges && edge.unseen(v0 + r)) {  // seen by no query of the unit: zeros, whatever lies there
              codes = make_uint4(0, 0, 0, 0);
              byte = 127;
            }
            uint4 lo, hi;
            dequant16<T>(codes, byte + (kv == 0 ? kKeyUp<T, kQuant> : 0), lo, hi);
            if constexpr (std::is_same<T, __half>::value) {
              if (odd_byte(kv, byte) && odd_row(kv, codes, lo, hi)) C.odd = 1;
            }
            uint8_t* row = dst + (r >> 3) * Sh::kGroup + (r & 7) * 128;
            const uint32_t sw = r & 7;
            // lanes of the two 64-element halves write opposite pieces: no bank is hit twice
            *reinterpret_cast<uint4*>(row + ((c0 + swap) ^ sw) * 16) = swap ? hi : lo;
            *reinterpret_cast<uint4*>(row + ((c0 + !swap) ^ sw) * 16) = swap ? lo : hi;
          }
          mbar_arrive(smem_u32(&C.raw_empty[kv]));
          fence_proxy_async_smem();
          mbar_arrive(smem_u32(&C.full[kv][st]));
        }
        tiles += n;
      }
      if (!ok && lane == 0) give_up(C, p.err);
    } else if (warp == Ro::kLoad || warp == Ro::kLoad + 1) {
      // ------------------------------------------------------------------ K and V copies
      const int kv = warp - Ro::kLoad;
      const uint32_t leader = elect_one_sync();
      const CUtensorMap* map = kv == 0 ? &k_map : &v_map;
      uint32_t issued = 0;
      bool ok = true;
      for (; on && ok; on = w.next(p)) {
        const Piece& c = w.c;
        const KeyRange kr = key_range(p, c.len, c.n, c.i0, min(c.n, c.i0 + p.tokens));
        // a part whose entry is no block is a copy from past the pool: zeros, not what the stage held
        TileRows at(p, kr, c, lane, p.num_blocks * p.n_kv_heads * p.block_size);
        const int box = at.box;
        for (int tile = c.tile0; tile < c.tile1; ++tile, ++issued) {
          at.advance(tile);
          const int st = Sh::stage(kv, issued);
          const uint32_t freed = smem_u32(kQuant ? &C.raw_empty[kv] : &C.empty[kv][st]);
          ok = __all_sync(0xffffffffu, role_wait(C.abort, freed, (kQuant ? issued & 1 : Sh::parity(kv, issued)) ^ 1));
          if (!ok) break;
          const uint32_t bar = smem_u32(kQuant ? &C.raw_full[kv] : &C.full[kv][st]);
          constexpr uint32_t kRowBytes = kQuant ? D : 2 * D;
          const uint32_t missing = at.missing(tile);
          if (kv == 0 && missing != 0 && leader) mark_lost(C, issued, missing, 7 - at.log_parts);
          mbar_arrive_expect_tx_p(leader, bar, __popc(at.have(tile)) * (uint32_t)box * kRowBytes);
          const uint32_t to = smem_u32(base + (kQuant ? Sh::kRaw + kv * Sh::kRawBytes : Sh::at(kv, issued)));
          if constexpr (kQuant) {  // the scale bytes: 16 (blocks of 8 keys: 8) a lane
            const int width = min(box, 16), key = lane * width, part = min(key, 127) >> (7 - at.log_parts);
            const int y = at.row(tile, part);
            if (missing >> part & 1) {  // its codes are zeros: any factor but the infinity that may lie there
              if (key < 128) *reinterpret_cast<uint2*>(&C.scales[kv][key]) = make_uint2(0x7F7F7F7Fu, 0x7F7F7F7Fu);
              if (key < 128 && width == 16) *reinterpret_cast<uint2*>(&C.scales[kv][key + 8]) = make_uint2(0x7F7F7F7Fu, 0x7F7F7F7Fu);
              __threadfence_block();
            } else if (key < 128 && y >= 0) {
              const uint8_t* src = p.scales + at.scale_at(y + (key - part * box), kv);
              const uint32_t sd = smem_u32(&C.scales[kv][key]);
              if (width == 16)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(sd), "l"(src) : "memory");
              else
                asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(sd), "l"(src) : "memory");
            }
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
          }
          for (int x0 = 0; x0 < at.parts; x0 += 8) {
            int y[8];  // all rows first: a shuffle between two copies costs more than the copies
#pragma unroll
            for (int x = 0; x < 8; ++x) y[x] = at.row(tile, (x0 + x) & (at.parts - 1));
#pragma unroll
            for (int x = 0; x < 8; ++x) {
              const uint32_t go = x0 + x < at.parts && y[x] >= 0 ? leader : 0u;
              if constexpr (kQuant) tma_load_2d_p(go, to + (x0 + x) * box * D, map, 0, y[x], bar);
              else tma_load_4d_p(go, to + (x0 + x) * box * (D * 2), map, 0, 0, 0, y[x] >> 3, bar);
            }
          }
        }
      }
      if (!ok && lane == 0) give_up(C, p.err);
      // before the shared memory goes: every copy issued has landed (bounded)
      if constexpr (kQuant) {
        if (issued > 0) mbar_wait(smem_u32(&C.raw_full[kv]), (issued - 1) & 1);
      } else {
        for (uint32_t i = issued > Sh::kK ? issued - Sh::kK : 0; i < issued; ++i)
          mbar_wait(smem_u32(&C.full[kv][Sh::stage(kv, i)]), Sh::parity(kv, i));
      }
    } else if (warp == Ro::kScores || warp == Ro::kValues) {
      // ------------------------------------------------------------------ MMA issuers
      const bool do_s = warp == Ro::kScores, do_o = warp == Ro::kValues;
      const uint32_t leader = elect_one_sync();
      uint32_t tiles = 0, piece = 0;  // key tiles, pieces before this one
      uint32_t s0[2] = {0, 0};  // steps of group 0 / 1 before this piece
      uint32_t last_bar = 0, last_parity = 0, q_pending = 0;
      bool ok = true;
      const auto wait = [&](uint64_t* bar, uint32_t parity) {
        ok = ok && __all_sync(0xffffffffu, role_wait(C.abort, smem_u32(bar), parity));
        if (ok) tc_fence_after();
        return ok;
      };
      // shared-memory descriptors: offsets only change the address field (in 16-byte units)
      const uint64_t q_desc = smem_desc(smem_u32(q_s), 16, 1024, kSwizzle128B);
      const uint64_t p_desc = smem_desc(smem_u32(p_s), 16, 1024, kSwizzle128B);
      const uint64_t k_desc = smem_desc(smem_u32(base + Sh::kRing), 16, Sh::kGroup, kSwizzle128B);
      const uint64_t v_desc = smem_desc(smem_u32(base + Sh::kRing + Sh::kK * Sh::kTileBytes), 1024, Sh::kGroup, kSwizzle128B);
      // S of group t = (Q of tile qt) K^T, K in stage st
      const auto scores = [&](int t, int qt, int st, uint32_t step) {
        const uint64_t qd = q_desc + qt * (Sh::kTileBytes >> 4), kd = k_desc + st * (Sh::kTileBytes >> 4);
#pragma unroll
        for (int kb = 0; kb < D / 64; ++kb)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            umma_f16_p(leader, tmem + t * kKeys, qd + ((kb * kBlockBytes + kk * 32) >> 4), kd + ((kb * 1024 + kk * 32) >> 4),
                       kIdescS, (kb > 0 || kk > 0) ? 1u : 0u);
        umma_commit_p(leader, smem_u32(&C.s_full[t]));
        last_bar = smem_u32(&C.s_full[t]);
        last_parity = step & 1;
      };
      // O of group t (+)= P V, V in stage st
      const auto values = [&](int t, int st, bool first, uint32_t step) {
        const uint64_t vd = v_desc + st * (Sh::kTileBytes >> 4);
#pragma unroll
        for (int ks = 0; ks < kKeys / 16; ++ks)
          umma_f16_p(leader, tmem + 2 * kKeys + t * D, p_desc + (((ks / 4) * kBlockBytes + (ks % 4) * 32) >> 4),
                     vd + ((ks * 2 * Sh::kGroup) >> 4), kIdescO, (!first || ks > 0) ? 1u : 0u);
        umma_commit_p(leader, smem_u32(&C.pv_done[t]));
        last_bar = smem_u32(&C.pv_done[t]);
        last_parity = step & 1;
      };
      for (; on && ok; on = w.next(p)) {
        const Piece& c = w.c;
        const int n = c.tile1 - c.tile0;
        const int i1 = min(c.n, c.i0 + p.tokens);
        const bool split = i1 - c.i0 <= p.tokens / 2;
        const int ahead = split ? 2 : 1;
        const KeyRange kr = key_range(p, c.len, c.n, c.i0, i1);
        const EdgeTiles edge(p, kr);
        const MixedTiles mixed(MixedKeys(p, kr, i1 - c.i0));
        if (do_s) {
          // the groups have read the last scores of the piece before: its products are done with Q
          for (int t = 0; t < 2 && ok; ++t)
            if (s0[t] > 0) wait(&C.s_free[t], (s0[t] - 1) & 1);
          if (!ok) break;
          const int qt = split ? 1 : 2, tpt = p.tokens / 2, head0 = c.kvh * p.group + c.slice * p.gw;
          const uint32_t bar = smem_u32(&C.q_full);
          mbar_arrive_expect_tx_p(leader, bar, qt * (D / 64) * tpt * p.gw * 128u);
          for (int t = 0; t < qt; ++t)
#pragma unroll
            for (int kb = 0; kb < D / 64; ++kb)
              tma_load_3d_p(leader, smem_u32(q_s + t * Sh::kTileBytes + kb * kBlockBytes), &q_map, 64 * kb, head0,
                            c.q_first + c.i0 + t * tpt, bar);
          q_pending = piece + 1;
          if (!wait(&C.q_full, piece & 1)) break;
        }
        // the scores of the first tile(s)
        for (int j = 0; j < min(n, ahead) && ok && do_s; ++j) {
          const uint32_t i = tiles + j;
          if (!wait(&C.full[0][Sh::stage(0, i)], Sh::parity(0, i))) break;
          for (int t = 0; t < (split ? 1 : 2) && ok; ++t) {
            scores(split ? j : t, t, Sh::stage(0, i), split && j == 1 ? s0[1] : s0[t]);
          }
          if (ok) umma_commit_p(leader, smem_u32(&C.empty[0][Sh::stage(0, i)]));
        }
        // Half steps h: group h & 1 takes its key tile.  Once it has read its scores, its next ones go
        // out, then the product of the half step before: the groups find their next scores ready, and
        // their products run under the other group's softmax.
        const int halves = split ? n : 2 * n;
        for (int h = 0; h <= halves && ok; ++h) {
          if (do_s && h < halves) {
            const int t = h & 1, j = split ? h : h >> 1;
            const uint32_t step = s0[t] + (h >> 1);
            if (j + ahead < n) {
              const uint32_t ik = tiles + j + ahead;
              if (!wait(&C.s_free[t], step & 1)) break;
              if ((split || t == 0) && !wait(&C.full[0][Sh::stage(0, ik)], Sh::parity(0, ik))) break;
              scores(t, split ? 0 : t, Sh::stage(0, ik), step + 1);
              if (split || t == 1) umma_commit_p(leader, smem_u32(&C.empty[0][Sh::stage(0, ik)]));
            }
          }
          if (do_o && h > 0) {
            const int t = (h - 1) & 1, j = split ? h - 1 : (h - 1) >> 1;
            const uint32_t step = s0[t] + ((h - 1) >> 1), iv = tiles + j;
            if ((split || t == 0) && !wait(&C.full[1][Sh::stage(1, iv)], Sh::parity(1, iv))) break;
            if (!kQuant && (split || t == 0) && edge(c.tile0 + j)) mbar_arrive_p(leader, smem_u32(&C.v_ready[t]));
            // under the group's softmax
            if ((split || t == 0) && mixed.has(c.tile0 + j)) {  // under the group's softmax
              const MixedKeys keys(p, key_range(p, c.len, c.n, c.i0, i1), i1 - c.i0);
              if (take_odd<T, D>(keys, (c.tile0 + j) * kKeys, lane, base + Sh::at(1, iv))) C.any_odd = 1;
              fence_proxy_async_smem();
              __syncwarp();
            }
            if (!wait(&C.p_full[t], step & 1)) break;
            values(t, Sh::stage(1, iv), step == s0[t], step);
            if (split || t == 1) umma_commit_p(leader, smem_u32(&C.empty[1][Sh::stage(1, iv)]));
          }
        }
        tiles += n;
        ++piece;
        s0[0] += split ? (n + 1) / 2 : n;
        s0[1] += split ? n / 2 : n;
      }
      if (!ok && lane == 0) give_up(C, p.err);
      if (q_pending) mbar_wait(smem_u32(&C.q_full), (q_pending - 1) & 1);  // Q has landed (bounded)
      if (last_bar) mbar_wait(last_bar, last_parity);  // MMAs in flight end (bounded) before TMEM goes
    }
  } else {
    // ------------------------------------------------------------------ softmax: thread = row
    regs_inc<Ro::kSoftmax>();
    const int t = warp >> 2, r = tid & 127;
    const uint32_t lanes = ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t t_s = tmem + lanes + t * kKeys, t_o = tmem + lanes + 2 * kKeys + t * D;
    const bool flip = p.scale < 0.f;  // then the scores change sign: the largest has the largest weight
    const float c2 = fmaxf(fabsf(p.scale) * (kLog2e / (1 << kKeyUp<T, kQuant>)), 1e-37f);
    uint8_t* prow = p_s + r * 128;
    const uint32_t sw = (uint32_t)(r & 7);
    uint32_t step = 0, tiles = 0, edges = 0, splits = 0, other_steps = 0;
    bool ok = true;
    while (on && ok) {
      const Piece c = w.c;
      const int n = c.tile1 - c.tile0;
      const int i1 = min(c.n, c.i0 + p.tokens), tpt = p.tokens / 2;
      const bool split = i1 - c.i0 <= tpt;
      // the row's token of the unit and head of the slice
      const int rt = p.by_gw.div(r), g = r - rt * p.gw, tok = (split ? 0 : t * tpt) + rt;
      const KeyRange kr = key_range(p, c.len, c.n, c.i0, i1);
      const EdgeTiles edge(p, kr);
      const int qpos = kr.pos0 + min(tok, i1 - c.i0 - 1);
      // on the virtual axis the row sees [v_lo, v_hi) and [0, v_s)
      const int v_hi = min(max(0, qpos + 1 - kr.shift), kr.v_len);
      const int v_lo = p.window > 0 ? max(0, qpos - p.window + 1) - kr.shift : 0;
      const int v_s = p.window > 0 ? min(p.sinks, v_hi) : 0;
      const uint32_t step0 = step;
      float m = -INFINITY, l = 0.f;
      for (int j = split ? t : 0; j < n; j += split ? 2 : 1) {
        const int v0 = (c.tile0 + j) * kKeys;
        ok = role_wait(C.abort, smem_u32(&C.s_full[t]), step & 1);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const bool any_lost = *reinterpret_cast<const volatile int32_t*>(&C.any_lost);  // lands with the scores
        float s[kKeys];
#pragma unroll
        for (int x = 0; x < kKeys; x += 32) tmem_ld32(t_s + x, s + x);
        tmem_wait_ld();
        tc_fence_before();
        mbar_arrive(smem_u32(&C.s_free[t]));
        if (!kQuant && (split || t == 0) && edge(c.tile0 + j)) {
          // rows of V that nobody sees are zeroed: 0 x (whatever lies there) must not reach O
          ok = __all_sync(0xffffffffu, role_wait(C.abort, smem_u32(&C.v_ready[t]), edges++ & 1));
          if (!ok) break;
          if (edge.unseen(v0 + r)) {
            uint8_t* vrow = base + Sh::at(1, tiles + j) + (r >> 3) * Sh::kGroup + (r & 7) * 128;
#pragma unroll
            for (int h = 0; h < D / 64; ++h)
#pragma unroll
              for (int x = 0; x < 8; ++x) *reinterpret_cast<uint4*>(vrow + h * 1024 + x * 16) = make_uint4(0, 0, 0, 0);
          }
        }
        if (flip) {
#pragma unroll
          for (int x = 0; x < kKeys; ++x) s[x] = -s[x];
        }
        {
          const int lo = v_lo - v0, hi = v_hi - v0, sk = v_s - v0;
          if (!__all_sync(0xffffffffu, hi >= kKeys && (lo <= 0 || sk >= kKeys))) {
#pragma unroll
            for (int x = 0; x < kKeys; x += 32) {  // bit i of `see`: key x + i
              const uint32_t see = (low_bits(hi - x) & ~low_bits(lo - x)) | low_bits(sk - x);
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!(see >> i & 1)) s[x + i] = -INFINITY;
            }
          }
        }
        if (any_lost && C.lost_tile[(tiles + j) % 8] == tiles + j) {
#pragma unroll
          for (int x = 0; x < kKeys; x += 32) {
            const uint32_t lost = C.lost[(tiles + j) % 8][x / 32];
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (lost >> i & 1) s[x + i] = -INFINITY;
          }
        }
        float mx[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) mx[x] = s[x];
#pragma unroll
        for (int x = 4; x < kKeys; x += 8)
#pragma unroll
          for (int i = 0; i < 4; ++i) mx[i] = x + 4 + i < kKeys ? fmaxf(mx[i], fmaxf(s[x + i], s[x + 4 + i])) : fmaxf(mx[i], s[x + i]);
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c2;
        const bool raise = top > m + kRescale<T>;
        if (__any_sync(0xffffffffu, raise)) {
          const float alpha = raise ? ex2(m - (top - kLow<T>)) : 1.f;
          if (raise) m = top - kLow<T>;
          l *= alpha;
          if (step > step0) {  // O += P V of the group's tile before is done: O may change
            ok = role_wait(C.abort, smem_u32(&C.pv_done[t]), (step - 1) & 1);
            if (!__all_sync(0xffffffffu, ok)) {
              ok = false;
              break;
            }
            tc_fence_after();
#pragma unroll 1
            for (int x = 0; x < D; x += 16) {
              float o[16];
              tmem_ld16(t_o + x, o);
              tmem_wait_ld();
#pragma unroll
              for (int y = 0; y < 16; ++y) o[y] *= alpha;
              tmem_st16(t_o + x, o);
            }
            tmem_wait_st();
          }
        }
        const float ref = m == -INFINITY ? 0.f : m;  // nothing seen yet: 2^-inf = 0 for any reference
        // products of the other group that come before this one's: they take turns, group 0 first
        const uint32_t before = other_steps + (step - step0) + t;
        // weights go to the tensor core in the query's type (off by half a step, 2^-8 of themselves in bf16 and 2^-11 in f16; one
        // product for P V instead of two), their sum stays f32: bf16 outputs have a relative RMS error of 0.0022, 0.0017 with
        // f32 weights
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        uint32_t pk[kKeys / 2];
#pragma unroll
        for (int x = 0; x < kKeys; x += 2) {
          float2 e = fma2(make_float2(s[x], s[x + 1]), make_float2(c2, c2), make_float2(-ref, -ref));
          e.x = ex2(e.x);
          e.y = ex2(e.y);
          sum[(x >> 1) & 1] = add2(sum[(x >> 1) & 1], e);
          pk[x / 2] = pack2<T>(e.x, e.y);
        }
        if (before > 0) {  // the other group's product has read the P buffer
          ok = role_wait(C.abort, smem_u32(&C.pv_done[t ^ 1]), (before - 1) & 1);
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            break;
          }
        }
#pragma unroll
        for (int x = 0; x < kKeys / 8; ++x)
          *reinterpret_cast<uint4*>(prow + (x / 8) * kBlockBytes + (((uint32_t)(x % 8) ^ sw) << 4)) =
              make_uint4(pk[4 * x], pk[4 * x + 1], pk[4 * x + 2], pk[4 * x + 3]);
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        fence_proxy_async_smem();
        tc_fence_before();
        mbar_arrive(smem_u32(&C.p_full[t]));
        ++step;
      }
      if (!ok) break;
      tiles += n;
      if (split) {
        other_steps += (n - (t ^ 1) + 1) / 2;
      } else {
        other_steps += n;
      }
      on = w.next(p);
      if (ok && step > step0) ok = role_wait(C.abort, smem_u32(&C.pv_done[t]), (step - 1) & 1);
      const uint32_t t_x = tmem + lanes + 2 * kKeys + (t ^ 1) * D;  // the other group's O
      float f = 1.f, fx = 0.f;
      if (split) {
        // group 1 hands its maxima and sums to group 0, which reads both O where they are and writes
        // the rows out
        if (t == 1) {
          C.ml[r] = make_float2(m, l);
          tc_fence_before();
          if (ok) mbar_arrive(smem_u32(&C.x_ml));
          ok = ok && role_wait(C.abort, smem_u32(&C.x_done), splits++ & 1);
          ok = __all_sync(0xffffffffu, ok);
          tc_fence_after();
          continue;
        }
        ok = ok && role_wait(C.abort, smem_u32(&C.x_ml), splits++ & 1);
        if (ok && other_steps > 0) ok = role_wait(C.abort, smem_u32(&C.pv_done[1]), (other_steps - 1) & 1);
        const float2 ml = C.ml[r];
        const float M = fmaxf(m, ml.x);
        f = m == -INFINITY ? l : ex2(m - M);  // sees nothing: 0; only NaN: NaN
        fx = ml.x == -INFINITY ? ml.y : ex2(ml.x - M);
        m = M;
        l = l * f + ml.y * fx;
      }
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const bool mine = rt < tpt && tok < i1 - c.i0 && g < slice_heads(p, c.slice), whole = c.whole();
      const int64_t slot = part_slot(c) * p.rows + tok * p.gw + g;
      T* out = reinterpret_cast<T*>(p.out) + (int64_t)(c.q_first + c.i0 + tok) * p.out_stride_tok +
               (int64_t)(c.kvh * p.group + c.slice * p.gw + g) * p.out_stride_head;
      if (!whole && mine) {
        p.part_ml[slot * 2] = m;
        p.part_ml[slot * 2 + 1] = l;
      }
      if constexpr (kStats)
        if (whole && mine) write_stats(p, c.q_first + c.i0 + tok, c.kvh * p.group + c.slice * p.gw + g, m, l);
      if (whole) {  // sees nothing: zeros
        const float inv = l == 0.f ? 0.f : 1.f / l;
        f *= inv;
        fx *= inv;
      }
#pragma unroll 1
      for (int x = 0; x < D; x += 16) {
        float o[16];
        tmem_ld16(t_o + x, o);
        if (split) {
          float o2[16];
          tmem_ld16(t_x + x, o2);
          tmem_wait_ld();
          // a group without a tile (or without a key its row sees) may hold anything
#pragma unroll
          for (int y = 0; y < 16; ++y) o[y] = (f == 0.f ? 0.f : o[y] * f) + (fx == 0.f ? 0.f : o2[y] * fx);
        } else {
          tmem_wait_ld();
#pragma unroll
          for (int y = 0; y < 16; ++y) o[y] = f == 0.f ? 0.f : o[y] * f;
        }
        if (!mine) continue;
        if (whole) {
#pragma unroll
          for (int y = 0; y < 16; y += 8)
            *reinterpret_cast<uint4*>(out + x + y) = make_uint4(pack2<T>(o[y], o[y + 1]), pack2<T>(o[y + 2], o[y + 3]),
                                                                pack2<T>(o[y + 4], o[y + 5]), pack2<T>(o[y + 6], o[y + 7]));
        } else {
#pragma unroll
          for (int y = 0; y < 16; y += 8) store32(p.part_o + slot * D + x + y, reinterpret_cast<const uint32_t*>(o + y));
        }
      }
      if (C.any_odd) {
        if (mine) add_odd<T, D, kQuant>(p, c, tok, out, whole ? nullptr : p.part_o + slot * D);
        __syncwarp();
      }
      tc_fence_before();
      if (split) mbar_arrive(smem_u32(&C.x_done));
    }
    if (!ok && lane == 0) give_up(C, p.err);
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0) {
    write_piece_info(p, C.plan);
    if (p.odd != nullptr) p.odd[blockIdx.x] = C.odd;
  }
  next_grid_may_launch();
  if (warp == Ro::kScores) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Q as [token][head][dim]: a box is the gw heads of a slice of 128 / gw tokens, 64 columns.
bool q_tiles_map(CUtensorMap* map, bool bf16, const ChunkParams& p, int D) {
  EncodeTiledFn fn = encode_tiled();
  if (!fn) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)p.n_q_heads, (cuuint64_t)p.total_q};
  const cuuint64_t strides[2] = {(cuuint64_t)p.q_stride_head * 2, (cuuint64_t)p.q_stride_tok * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)p.gw, (cuuint32_t)p.tokens / 2};
  const cuuint32_t estr[3] = {1, 1, 1};
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(p.q), dims,
            strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D, bool kQuant, bool kStats>
int launch(const WeighedParams& p, cudaStream_t st) {
  CUtensorMap q_map, k_map, v_map;
  const uint64_t rows = (uint64_t)p.num_blocks * p.n_kv_heads * p.block_size;
  const uint32_t box = p.block_size < kKeys ? p.block_size : kKeys;
  const bool bf16 = std::is_same<T, __nv_bfloat16>::value;
  const bool mapped = kQuant ? tensor_map_bytes(&k_map, p.k_pool, D, rows, box, false) && tensor_map_bytes(&v_map, p.v_pool, D, rows, box, false)
                             : tensor_map_row_groups(&k_map, bf16, p.k_pool, rows, D, box / 8) &&
                                   tensor_map_row_groups(&v_map, bf16, p.v_pool, rows, D, box / 8);
  if (!mapped || !q_tiles_map(&q_map, bf16, p, D)) return SNAPMIND_ERR_UNSUPPORTED;  // the caller takes the CUDA-core kernel
  auto kernel = chunk_umma_kernel<T, D, kQuant, kStats>;
  static bool done[kMaxDevices] = {};
  const cudaError_t e = kernel_attributes(reinterpret_cast<const void*>(kernel), smem_bytes<D, kQuant>(), done);
  if (e != cudaSuccess) return cuda_status(e, "paged_chunk smem attribute");
  return cuda_status(launch_dependent(kernel, dim3(p.n_ctas), Roles<kQuant>::kThreads, smem_bytes<D, kQuant>(), st, q_map,
                                      k_map, v_map, p),
                     "paged_chunk launch");
}

}  // namespace

// Shapes of the kernel: 16-bit queries and outputs in whole, aligned 16-byte vectors; head_dim 64
// or 128; blocks of 8, 16, 32, 64, 128 or a multiple of 128 tokens (a 128-key tile is whole
// blocks, or lies in one).
bool chunk_umma_supported(const ChunkParams& p, int dtype, int pool_dtype) {
  if (dtype != SNAPMIND_DTYPE_BF16 && dtype != SNAPMIND_DTYPE_F16) return false;
  if (p.head_dim != 64 && p.head_dim != 128) return false;
  const int bs = p.block_size;
  if (bs != 8 && bs != 16 && bs != 32 && bs != 64 && bs % 128 != 0) return false;
  const auto a16 = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; };
  if (!a16(p.q) || !a16(p.out) || !a16(p.k_pool) || !a16(p.v_pool)) return false;
  if (p.q_stride_tok <= 0 || p.q_stride_head <= 0 || p.q_stride_tok % 8 || p.q_stride_head % 8 || p.out_stride_tok % 8 || p.out_stride_head % 8) return false;
  if ((int64_t)p.num_blocks * p.n_kv_heads * bs >= (int64_t)1 << 31) return false;  // TMA row coordinate
  if (pool_dtype == SNAPMIND_DTYPE_E4M3 && !a16(p.scales)) return false;
  return encode_tiled() != nullptr;
}

int launch_chunk_umma(WeighedParams& p, int dtype, int pool_dtype, cudaStream_t st) {
  const int rc = plan_geometry(p, 2 * kTileM, kTileM, kKeys, num_sms());
  if (rc != SNAPMIND_OK) return rc;
  const bool quant = pool_dtype == SNAPMIND_DTYPE_E4M3;
  const auto go = [&](auto t) -> int {
    using T = decltype(t);
    const auto of = [&](auto stats) -> int {
      constexpr bool kStats = decltype(stats)::value;
      if (p.head_dim == 64) return quant ? launch<T, 64, true, kStats>(p, st) : launch<T, 64, false, kStats>(p, st);
      return quant ? launch<T, 128, true, kStats>(p, st) : launch<T, 128, false, kStats>(p, st);
    };
    return p.stats != nullptr ? of(std::true_type()) : of(std::false_type());
  };
  return dtype == SNAPMIND_DTYPE_BF16 ? go(__nv_bfloat16()) : go(__half());
}

}  // namespace snapmind
