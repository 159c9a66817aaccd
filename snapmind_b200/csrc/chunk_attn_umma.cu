// Attention of chunks of new tokens over a paged cache on the 5th-generation tensor
// cores: bf16 / f16 queries, head_dim 64 or 128, caches of the query's type (staged by
// TMA) or of e4m3 rows (converted while they are staged).
//
// A unit (chunk_plan.cuh) has up to 256 query rows of one kv head as two tiles of 128 (M), and
// a step takes 128 keys:
//   S = Q K^T [128 x 128] (Q and K K-major), P = 2^(S c - m), O += P V (V MN-major).
// Softmax and MMA of the two tiles alternate: while the tensor core works on one tile's
// products, the other tile's 128 threads (one row each) take its scores.
// A row keeps a reference maximum that is raised only when a score exceeds it by 2^8:
// then O is rescaled in TMEM, else O is never touched between the products.
//   warps 0-3, 4-7  softmax of tile 0 / 1: thread = row = TMEM lane; they load their Q tile,
//                   write P to shared memory, and write out the finished rows
//   warp 8          issues the MMAs
//   warps 9-11      stage K and V: warp 9 by TMA, or all three converting e4m3 rows
// P goes through shared memory, not through TMEM as an A operand: a kernel of this library that
// read A from TMEM ended in a launch failure whose cause was not found.
//   TMEM: S of tile 0 / 1 at columns 0 / 128, O at 256 / 256 + head_dim.
//   Shared memory: Q 2 x [128 x D], P 2 x [128 x 128], then a ring of [128 x D] stages that
//   K and V tiles take in the order K0, K1, V0, K2, V1, ... (128-byte swizzle everywhere).
// Every wait is bounded and ends early once another role gave up; TMEM is released on
// every path.
#include <cuda.h>
#include <cuda_fp8.h>

#include "chunk_plan.cuh"
#include "sm100.cuh"

namespace snapmind {
namespace {

using namespace tc;

constexpr int kTileM = 128, kKeys = 128;
constexpr int kMmaWarp = 8, kLoadWarp = 9;
constexpr int kConvert = 96;  // threads that convert e4m3 rows: warps 9-11
constexpr uint32_t kBlockBytes = 128 * 128;  // 128 rows of 64 16-bit elements
constexpr uint32_t kPBytes = 2 * kBlockBytes;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescale = 8.f;  // log2 headroom of the reference maximum

template <int D> struct Shape {
  static constexpr uint32_t kTileBytes = D / 64 * kBlockBytes;  // a Q tile, a K or V stage
  static constexpr int kStages = D == 64 ? 6 : 3;
  static constexpr uint32_t kP = 2 * kTileBytes, kRing = kP + 2 * kPBytes;
  static constexpr uint32_t kCtrl = kRing + kStages * kTileBytes;
};

struct Ctrl {
  uint64_t kv_full[6], kv_empty[6];
  uint64_t q_full[2];   // softmax threads: the Q tile of a piece is in shared memory
  uint64_t s_full[2];   // MMA commit: scores ready
  uint64_t p_full[2];   // softmax threads: P written, scores read
  uint64_t pv_done[2];  // MMA commit: O += P V done
  uint32_t tmem_base;
  int32_t abort;
  PlanShared plan;
};

template <int D> constexpr size_t smem_bytes() { return 1024 + Shape<D>::kCtrl + sizeof(Ctrl); }
static_assert(smem_bytes<128>() <= 232448 && smem_bytes<64>() <= 232448, "shared memory budget");
static_assert(2 * kPBytes >= kMaxChunkBatch * 4, "plan scratch in the P tiles");

__device__ __forceinline__ bool role_wait(const Ctrl& C, uint32_t bar, uint32_t parity) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity)) {
    if (*reinterpret_cast<const volatile int32_t*>(&C.abort)) return false;
    if (clock64() - t0 > kWaitTicks) return false;
  }
  return true;
}
__device__ __forceinline__ void give_up(Ctrl& C, int32_t* err) {
  atomicExch(&C.abort, 1);
  flag_error(err, SNAPMIND_DEVERR_TIMEOUT);
}

template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// The staged loads of a piece of n tiles, in order: K0, K1, V0, K2, V1, .., K(n-1), V(n-2), V(n-1).
__device__ __forceinline__ int k_index(int j) { return j == 0 ? 0 : 2 * j - 1; }
__device__ __forceinline__ int v_index(int j, int n) { return j == n - 1 ? 2 * n - 1 : 2 * j + 2; }

// Stage and parity of the load with running number i.
template <int D> __device__ __forceinline__ int stage_of(uint32_t i) { return i % Shape<D>::kStages; }
template <int D> __device__ __forceinline__ uint32_t full_parity(uint32_t i) { return (i / Shape<D>::kStages) & 1; }

// 16 e4m3 codes of one row times 2^(byte - 127), as 16 elements of T.  The scale is a power
// of two: exact in bf16, and in f16 as long as the value is a normal f16.
template <typename T>
__device__ __forceinline__ void dequant16(const uint4& codes, uint8_t byte, uint4& lo, uint4& hi) {
  const float s = __uint_as_float((uint32_t)byte << 23);
  const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
  uint32_t o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i / 2] >> (16 * (i & 1))), __NV_E4M3);
    float2 f = __half22float2(__half2(h));
    f.x *= s;
    f.y *= s;
    if constexpr (std::is_same<T, __half>::value) {  // hold to f16's range, keep NaN
      if (fabsf(f.x) > 65504.f) f.x = copysignf(65504.f, f.x);
      if (fabsf(f.y) > 65504.f) f.y = copysignf(65504.f, f.y);
    }
    o[i] = pack2<T>(f.x, f.y);
  }
  lo = make_uint4(o[0], o[1], o[2], o[3]);
  hi = make_uint4(o[4], o[5], o[6], o[7]);
}

// Three warpgroups.  They are launched with 168 registers a thread (3 x 128 x 168 = 64512); the third
// gives up what the softmax threads, with a row of 128 scores each, need more of.
constexpr int kThreads = 384;
template <bool kQuant> struct Regs {
  static constexpr int kOther = kQuant ? 120 : 56, kSoftmax = kQuant ? 192 : 224;
  static_assert(kOther + 2 * kSoftmax <= 3 * 168, "register split");
};
template <int N> __device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }

template <typename T, int D, bool kQuant>
__global__ void __launch_bounds__(kThreads, 1)
    chunk_umma_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                      ChunkParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  using Sh = Shape<D>;
  constexpr int kStages = Sh::kStages;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t kIdescS = idesc_f16(kBf16, kTileM, kKeys, false, false);
  constexpr uint32_t kIdescO = idesc_f16(kBf16, kTileM, D, false, true);
  uint8_t* q_s = base;
  uint8_t* p_s = base + Sh::kP;
  uint8_t* ring = base + Sh::kRing;
  Ctrl& C = *reinterpret_cast<Ctrl*>(base + Sh::kCtrl);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(smem_u32(&C.kv_full[i]), kQuant ? kConvert : 1);
      mbar_init(smem_u32(&C.kv_empty[i]), 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(smem_u32(&C.q_full[t]), 128);
      mbar_init(smem_u32(&C.s_full[t]), 1);
      mbar_init(smem_u32(&C.p_full[t]), 128);
      mbar_init(smem_u32(&C.pv_done[t]), 1);
    }
    C.abort = 0;
    mbar_init_fence();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(&C.tmem_base), 512);
    tmem_relinquish();
  }
  plan_block(p, C.plan, reinterpret_cast<int32_t*>(p_s));
  if (tid == 0) write_piece_info(p, C.plan);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = C.tmem_base;

  PieceWalk w;
  bool on = w.start(C.plan);
  if (warp >= kMmaWarp) {
  regs_dec<Regs<kQuant>::kOther>();
  if (warp >= kLoadWarp) {
    if (!kQuant && warp > kLoadWarp) on = false;
    // ------------------------------------------------------------------ K and V stages
    uint32_t issued = 0;
    bool ok = true;
    for (; on && ok; on = w.next(p)) {
      const Piece& c = w.c;
      const KeyRange kr = key_range(p, c.len, c.n, c.i0, min(c.n, c.i0 + p.tokens));
      const int n = c.tile1 - c.tile0, bs = p.block_size;
      const int32_t* table = p.tables + (int64_t)c.b * p.table_stride;
      const int box = min(bs, kKeys);  // rows of a tile that share a block
      const int per_tile = kKeys / box;
      // the physical block of part `lane` of tile j (lanes >= per_tile: none), -1 when nothing is there
      const auto block_of = [&](int j) -> int32_t {
        const int v = (c.tile0 + j) * kKeys + lane * box;
        if (j >= n || lane >= per_tile || v >= kr.v_len) return -1;
        const int lb = kr.position(v) / bs;
        if (lb >= p.table_width) {
          flag_error(p.err, SNAPMIND_DEVERR_TABLE);
          return -1;
        }
        const int32_t phys = table[lb];
        if (phys < 0 || phys >= p.num_blocks) {
          flag_error(p.err, SNAPMIND_DEVERR_BLOCK_ID);
          return -1;
        }
        return phys;
      };
      int32_t prev = -1, cur = block_of(0);  // blocks of the latest V's and K's tiles
      for (int i = 0; i < 2 * n && ok; ++i) {
        // load i of the piece: tile j of K (0) or V (1)
        const int kv = i == 0 ? 0 : (i == 2 * n - 1 ? 1 : (i & 1 ? 0 : 1));
        const int j = kv == 0 ? (i + 1) / 2 : (i == 2 * n - 1 ? n - 1 : i / 2 - 1);
        if (kv == 0 && i > 0) {
          prev = cur;
          cur = block_of(j);
        } else if (i == 2 * n - 1) {
          prev = cur;
        }
        const int32_t phys = kv == 0 ? cur : prev;
        const int st = stage_of<D>(issued);
        const int off = bs > kKeys ? kr.position((c.tile0 + j) * kKeys) % bs : 0;  // tile inside a larger block
        uint8_t* dst = ring + st * Sh::kTileBytes;
        if constexpr (!kQuant) {
          const uint32_t leader = elect_one_sync();
          ok = __all_sync(0xffffffffu, role_wait(C, smem_u32(&C.kv_empty[st]), full_parity<D>(issued) ^ 1));
          if (!ok) break;
          const uint32_t have = __ballot_sync(0xffffffffu, phys >= 0);
          const uint32_t bar = smem_u32(&C.kv_full[st]);
          mbar_arrive_expect_tx_p(leader, bar, __popc(have) * (uint32_t)box * 128u * (D / 64));
          const CUtensorMap* map = kv == 0 ? &k_map : &v_map;
          for (int x = 0; x < per_tile; ++x) {
            if (!(have >> x & 1)) continue;
            const int y = (__shfl_sync(0xffffffffu, phys, x) * p.n_kv_heads + c.kvh) * bs + off;
#pragma unroll
            for (int h = 0; h < D / 64; ++h)
              tma_load_2d_p(leader, smem_u32(dst + h * kBlockBytes + x * box * 128), map, 64 * h, y, bar);
          }
        } else {
          // D / 16 lanes share a row (16 codes each), kRowsPass rows a pass
          constexpr int kLanes = D / 16, kRowsPass = kConvert / kLanes, kPasses = (128 + kRowsPass - 1) / kRowsPass;
          const int ct = tid - kLoadWarp * 32, ch = ct % kLanes, r0 = ct / kLanes;
          const uint8_t* pool = static_cast<const uint8_t*>(kv == 0 ? p.k_pool : p.v_pool);
          uint4 codes[kPasses];
          uint8_t sc[kPasses];
#pragma unroll
          for (int x = 0; x < kPasses; ++x) {
            const int r = x * kRowsPass + r0;
            const int32_t ph = __shfl_sync(0xffffffffu, phys, r / box);
            const int v = (c.tile0 + j) * kKeys + r;
            // rows that no query of the unit sees are zeros: past the end, or in a block that is
            // read between the sinks and the first window
            const int pos = kr.position(v);
            const bool seen = r < 128 && ph >= 0 && v < kr.v_len && (pos >= kr.win_lo || pos < p.sinks);
            codes[x] = make_uint4(0, 0, 0, 0);
            sc[x] = 0;
            if (seen) {
              const int64_t tile = (int64_t)ph * p.n_kv_heads + c.kvh;
              const int slot = r % box + off;
              codes[x] = *reinterpret_cast<const uint4*>(pool + (tile * bs + slot) * D + ch * 16);
              sc[x] = p.scales[(tile * 2 + kv) * bs + slot];
            }
          }
          ok = role_wait(C, smem_u32(&C.kv_empty[st]), full_parity<D>(issued) ^ 1);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
#pragma unroll
          for (int x = 0; x < kPasses; ++x) {
            const int r = x * kRowsPass + r0;
            if (r >= 128) break;
            uint4 lo, hi;
            dequant16<T>(codes[x], sc[x], lo, hi);
            uint8_t* row = dst + (ch / 4) * kBlockBytes + r * 128;
            const uint32_t sw = r & 7, c0 = (ch % 4) * 2;
            // lanes of the two 64-element halves write opposite pieces: no bank is hit twice
            const bool swap = ch >= 4;
            *reinterpret_cast<uint4*>(row + ((c0 + swap) ^ sw) * 16) = swap ? hi : lo;
            *reinterpret_cast<uint4*>(row + ((c0 + !swap) ^ sw) * 16) = swap ? lo : hi;
          }
          fence_proxy_async_smem();
          mbar_arrive(smem_u32(&C.kv_full[st]));
        }
        ++issued;
      }
    }
    if (!ok && lane == 0) give_up(C, p.err);
    if constexpr (!kQuant) {  // before the shared memory goes: every copy issued has landed (bounded)
      for (uint32_t i = issued > kStages ? issued - kStages : 0; i < issued; ++i)
        mbar_wait(smem_u32(&C.kv_full[stage_of<D>(i)]), full_parity<D>(i));
    }
  } else {
    // ------------------------------------------------------------------ MMA issuer
    const uint32_t leader = elect_one_sync();
    uint32_t load0 = 0, piece = 0;
    uint32_t steps[2] = {0, 0}, pieces1 = 0;  // key tiles done by tile 0 / 1; pieces with a tile 1
    uint32_t last_bar = 0, last_parity = 0;
    bool ok = true;
    const auto wait = [&](uint64_t* bar, uint32_t parity) {
      ok = ok && __all_sync(0xffffffffu, role_wait(C, smem_u32(bar), parity));
      if (ok) tc_fence_after();
      return ok;
    };
    // S of tile t = Q K^T, K in stage st
    const auto scores = [&](int t, int st) {
#pragma unroll
      for (int kb = 0; kb < D / 64; ++kb)
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          umma_f16_p(leader, tmem + t * kKeys,
                     smem_desc(smem_u32(q_s + t * Sh::kTileBytes + kb * kBlockBytes + kk * 32), 16, 1024, kSwizzle128B),
                     smem_desc(smem_u32(ring + st * Sh::kTileBytes + kb * kBlockBytes + kk * 32), 16, 1024, kSwizzle128B),
                     kIdescS, (kb > 0 || kk > 0) ? 1u : 0u);
      umma_commit_p(leader, smem_u32(&C.s_full[t]));
      last_bar = smem_u32(&C.s_full[t]);
    };
    // O of tile t (+)= P V, V in stage st
    const auto values = [&](int t, int st, bool first) {
#pragma unroll
      for (int ks = 0; ks < kKeys / 16; ++ks)
        umma_f16_p(leader, tmem + 2 * kKeys + t * D,
                   smem_desc(smem_u32(p_s + t * kPBytes + (ks / 4) * kBlockBytes + (ks % 4) * 32), 16, 1024, kSwizzle128B),
                   smem_desc(smem_u32(ring + st * Sh::kTileBytes + ks * 16 * 128), kBlockBytes, 1024, kSwizzle128B),
                   kIdescO, (!first || ks > 0) ? 1u : 0u);
      umma_commit_p(leader, smem_u32(&C.pv_done[t]));
      last_bar = smem_u32(&C.pv_done[t]);
    };
    for (; on && ok; on = w.next(p)) {
      const Piece& c = w.c;
      const int n = c.tile1 - c.tile0;
      const int tiles = (min(c.n, c.i0 + p.tokens) - c.i0) * p.gw > kTileM ? 2 : 1;
      {
        const uint32_t i = load0;
        if (!wait(&C.kv_full[stage_of<D>(i)], full_parity<D>(i))) break;
        for (int t = 0; t < tiles && ok; ++t) {
          if (!wait(&C.q_full[t], (t == 0 ? piece : pieces1) & 1)) break;
          scores(t, stage_of<D>(i));
          last_parity = steps[t] & 1;
        }
        if (!ok) break;
        umma_commit_p(leader, smem_u32(&C.kv_empty[stage_of<D>(i)]));
      }
      for (int j = 0; j < n && ok; ++j) {
        const uint32_t ik = load0 + k_index(j + 1), iv = load0 + v_index(j, n);
        for (int t = 0; t < tiles; ++t) {
          // P of tile j written, so its scores are read: the next ones may replace them
          if (!wait(&C.p_full[t], steps[t] & 1)) break;
          if (j + 1 < n) {
            if (t == 0 && !wait(&C.kv_full[stage_of<D>(ik)], full_parity<D>(ik))) break;
            scores(t, stage_of<D>(ik));
            last_parity = (steps[t] + 1) & 1;
            if (t == tiles - 1) umma_commit_p(leader, smem_u32(&C.kv_empty[stage_of<D>(ik)]));
          }
          if (t == 0 && !wait(&C.kv_full[stage_of<D>(iv)], full_parity<D>(iv))) break;
          values(t, stage_of<D>(iv), j == 0);
          last_parity = steps[t] & 1;
          ++steps[t];
          if (t == tiles - 1) umma_commit_p(leader, smem_u32(&C.kv_empty[stage_of<D>(iv)]));
        }
      }
      load0 += 2 * n;
      ++piece;
      pieces1 += tiles - 1;
    }
    if (!ok && lane == 0) give_up(C, p.err);
    if (last_bar) mbar_wait(last_bar, last_parity);  // MMAs in flight end (bounded) before TMEM goes
  }
  } else {
    // ------------------------------------------------------------------ softmax: thread = row
    regs_inc<Regs<kQuant>::kSoftmax>();
    const int t = warp >> 2, r = tid & 127;
    const uint32_t lanes = ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t t_s = tmem + lanes + t * kKeys, t_o = tmem + lanes + 2 * kKeys + t * D;
    const bool flip = p.scale < 0.f;  // a negative scale is folded into Q, so the largest score has the largest weight
    const float c2 = fmaxf(fabsf(p.scale) * kLog2e, 1e-37f);
    uint8_t* prow = p_s + t * kPBytes + r * 128;
    const uint32_t sw = (uint32_t)(r & 7);
    uint32_t step = 0, load0 = 0;
    bool ok = true;
    for (; on && ok; on = w.next(p)) {
      const Piece& c = w.c;
      const int n = c.tile1 - c.tile0;
      const int i1 = min(c.n, c.i0 + p.tokens), n_rows = (i1 - c.i0) * p.gw;
      const uint32_t load = load0;
      load0 += 2 * n;
      if (t * kTileM >= n_rows) continue;
      const int heads = slice_heads(p, c.slice), head0 = c.kvh * p.group + c.slice * p.gw;
      // the Q tile (the scores of the piece before are all done: its last s_full was waited for)
      for (int e = r; e < kTileM * (D / 8); e += 128) {
        const int row = e / (D / 8), ch = e % (D / 8), R = t * kTileM + row, g = R % p.gw;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (R < n_rows && g < heads)
          x = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.q) +
                                              (int64_t)(c.q_first + c.i0 + R / p.gw) * p.q_stride_tok +
                                              (int64_t)(head0 + g) * p.q_stride_head + ch * 8);
        if (flip) {
          x.x ^= 0x80008000u;
          x.y ^= 0x80008000u;
          x.z ^= 0x80008000u;
          x.w ^= 0x80008000u;
        }
        *reinterpret_cast<uint4*>(q_s + t * Sh::kTileBytes + (ch / 8) * kBlockBytes + row * 128 + (((uint32_t)(ch % 8) ^ (row & 7)) << 4)) = x;
      }
      fence_proxy_async_smem();
      mbar_arrive(smem_u32(&C.q_full[t]));

      const KeyRange kr = key_range(p, c.len, c.n, c.i0, i1);
      const int R = t * kTileM + r;
      const int qpos = kr.pos0 + min(R, n_rows - 1) / p.gw;
      // on the virtual axis the row sees [v_lo, v_hi) and [0, v_s); no row of the unit sees
      // [u_s, u_lo) or past v_len
      const int v_hi = max(0, qpos + 1 - kr.shift);
      const int v_lo = p.window > 0 ? max(0, qpos - p.window + 1) - kr.shift : 0;
      const int v_s = p.window > 0 ? min(p.sinks, v_hi) : 0;
      const int u_s = p.window > 0 ? min(p.sinks, kr.v_sink) : 0, u_lo = kr.win_lo - kr.shift;
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < n; ++j) {
        const int v0 = (c.tile0 + j) * kKeys;
        ok = ok && role_wait(C, smem_u32(&C.s_full[t]), step & 1);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (!kQuant && t == 0) {
          const int key = v0 + r;
          if (v0 + kKeys > kr.v_len || (v0 < u_lo && v0 + kKeys > u_s)) {
            // rows of V that nobody sees are zeroed: 0 x (whatever lies there) must not reach O.
            // (After the scores: K of this tile has landed, so V's barrier is in the phase waited for.)
            const uint32_t i = load + v_index(j, n);
            ok = __all_sync(0xffffffffu, role_wait(C, smem_u32(&C.kv_full[stage_of<D>(i)]), full_parity<D>(i)));
            if (!ok) break;
            if (key >= kr.v_len || (key < u_lo && key >= u_s)) {
              uint8_t* vrow = ring + stage_of<D>(i) * Sh::kTileBytes + r * 128;
#pragma unroll
              for (int h = 0; h < D / 64; ++h)
#pragma unroll
                for (int x = 0; x < 8; ++x) *reinterpret_cast<uint4*>(vrow + h * kBlockBytes + x * 16) = make_uint4(0, 0, 0, 0);
            }
          }
        }
        float s[kKeys];
        const auto load_scores = [&]() {
#pragma unroll
          for (int x = 0; x < kKeys; x += 32) tmem_ld32(t_s + x, s + x);
          tmem_wait_ld();
          const int lo = v_lo - v0, hi = v_hi - v0, sk = v_s - v0;
          if (!__all_sync(0xffffffffu, hi >= kKeys && (lo <= 0 || sk >= kKeys))) {
#pragma unroll
            for (int x = 0; x < kKeys; ++x)
              if (!((x >= lo && x < hi) || x < sk)) s[x] = -INFINITY;
          }
        };
        load_scores();
        float mx[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) mx[x] = s[x];
#pragma unroll
        for (int x = 4; x < kKeys; ++x) mx[x & 3] = fmaxf(mx[x & 3], s[x]);
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c2;
        const bool raise = top > m + kRescale;
        bool waited = j == 0;  // O += P V of the tile before: P and O are free
        if (__any_sync(0xffffffffu, raise)) {
          const float alpha = raise ? ex2(m - top) : 1.f;
          if (raise) m = top;
          l *= alpha;
          if (j > 0) {
            ok = role_wait(C, smem_u32(&C.pv_done[t]), (step - 1) & 1);
            if (!__all_sync(0xffffffffu, ok)) {
              ok = false;
              break;
            }
            waited = true;
            tc_fence_after();
#pragma unroll 1
            for (int x = 0; x < D; x += 32) {
              float o[32];
              tmem_ld32(t_o + x, o);
              tmem_wait_ld();
#pragma unroll
              for (int y = 0; y < 32; ++y) o[y] *= alpha;
              tmem_st32(t_o + x, o);
            }
            tmem_wait_st();
            load_scores();  // again, rather than 128 registers kept over the rescaling
          }
        }
        const float ref = m == -INFINITY ? 0.f : m;  // nothing seen yet: 2^-inf = 0 for any reference
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        uint32_t pk[kKeys / 2];
#pragma unroll
        for (int x = 0; x < kKeys; x += 2) {
          const float a = ex2(fmaf(s[x], c2, -ref)), b = ex2(fmaf(s[x + 1], c2, -ref));
          sum[x & 2] += a;
          sum[(x & 2) + 1] += b;
          pk[x / 2] = pack2<T>(a, b);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        if (!waited) {
          ok = role_wait(C, smem_u32(&C.pv_done[t]), (step - 1) & 1);
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            break;
          }
        }
#pragma unroll
        for (int x = 0; x < kKeys / 8; ++x)
          *reinterpret_cast<uint4*>(prow + (x / 8) * kBlockBytes + (((uint32_t)(x % 8) ^ sw) << 4)) =
              make_uint4(pk[4 * x], pk[4 * x + 1], pk[4 * x + 2], pk[4 * x + 3]);
        fence_proxy_async_smem();
        tc_fence_before();
        mbar_arrive(smem_u32(&C.p_full[t]));
        ++step;
      }
      if (!ok) break;
      ok = role_wait(C, smem_u32(&C.pv_done[t]), (step - 1) & 1);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const int g = R % p.gw;
      const bool mine = R < n_rows && g < heads;
      if (c.whole()) {
        const float inv = m == -INFINITY ? 0.f : 1.f / l;
        T* out = reinterpret_cast<T*>(p.out) + (int64_t)(c.q_first + c.i0 + R / p.gw) * p.out_stride_tok +
                 (int64_t)(head0 + g) * p.out_stride_head;
#pragma unroll 1
        for (int x = 0; x < D; x += 32) {
          float o[32];
          tmem_ld32(t_o + x, o);
          tmem_wait_ld();
          if (mine) {
#pragma unroll
            for (int y = 0; y < 32; y += 8)
              *reinterpret_cast<uint4*>(out + x + y) =
                  make_uint4(pack2<T>(o[y] * inv, o[y + 1] * inv), pack2<T>(o[y + 2] * inv, o[y + 3] * inv),
                             pack2<T>(o[y + 4] * inv, o[y + 5] * inv), pack2<T>(o[y + 6] * inv, o[y + 7] * inv));
          }
        }
      } else {
        const int64_t slot = part_slot(c) * p.rows + R;
        if (mine) {
          p.part_ml[slot * 2] = m;
          p.part_ml[slot * 2 + 1] = l;
        }
#pragma unroll 1
        for (int x = 0; x < D; x += 32) {
          float o[32];
          tmem_ld32(t_o + x, o);
          tmem_wait_ld();
          if (mine) {
#pragma unroll
            for (int y = 0; y < 32; y += 4)
              *reinterpret_cast<float4*>(p.part_o + slot * D + x + y) = make_float4(o[y], o[y + 1], o[y + 2], o[y + 3]);
          }
        }
      }
      tc_fence_before();
    }
    if (!ok && lane == 0) give_up(C, p.err);
  }
  tc_fence_before();
  __syncthreads();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <typename T, int D, bool kQuant>
int launch(const ChunkParams& p, cudaStream_t st) {
  CUtensorMap k_map = {}, v_map = {};
  if (!kQuant) {
    const uint64_t rows = (uint64_t)p.num_blocks * p.n_kv_heads * p.block_size;
    const uint32_t box = p.block_size < kKeys ? p.block_size : kKeys;
    const bool bf16 = std::is_same<T, __nv_bfloat16>::value;
    if (!tensor_map_2d(&k_map, bf16, p.k_pool, D, rows, D * 2, 64, box) ||
        !tensor_map_2d(&v_map, bf16, p.v_pool, D, rows, D * 2, 64, box)) {
      set_last_error("paged_chunk: tensor map encoding failed");
      return SNAPMIND_ERR_CUDA;
    }
  }
  auto kernel = chunk_umma_kernel<T, D, kQuant>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes<D>());
  if (e != cudaSuccess) return cuda_status(e, "paged_chunk smem attribute");
  kernel<<<p.n_ctas, kThreads, smem_bytes<D>(), st>>>(k_map, v_map, p);
  return cuda_status(cudaGetLastError(), "paged_chunk launch");
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
  if (p.q_stride_tok % 8 || p.q_stride_head % 8 || p.out_stride_tok % 8 || p.out_stride_head % 8) return false;
  if ((int64_t)p.num_blocks * p.n_kv_heads * bs >= (int64_t)1 << 31) return false;  // TMA row coordinate
  return pool_dtype == SNAPMIND_DTYPE_E4M3 || encode_tiled() != nullptr;
}

int launch_chunk_umma(ChunkParams& p, int dtype, int pool_dtype, cudaStream_t st) {
  plan_geometry(p, 2 * kTileM, kKeys, num_sms());
  const bool quant = pool_dtype == SNAPMIND_DTYPE_E4M3;
  const auto go = [&](auto t) -> int {
    using T = decltype(t);
    if (p.head_dim == 64) return quant ? launch<T, 64, true>(p, st) : launch<T, 64, false>(p, st);
    return quant ? launch<T, 128, true>(p, st) : launch<T, 128, false>(p, st);
  };
  return dtype == SNAPMIND_DTYPE_BF16 ? go(__nv_bfloat16()) : go(__half());
}

}  // namespace snapmind
