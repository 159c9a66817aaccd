// The pass that adds the weights of a chunk's softmax to their keys (chunk_mass.cuh) on the 5th-generation
// tensor cores: bf16 / f16 queries, head_dim 64 or 128, caches of the query's type or of e4m3 rows.
//
//   mass[key] += sum_i 2^(c s(key, i) - x_i),  x_i = reference + log2(sum) of row i
//
// The scores are taken transposed, S^T = K Q^T with the keys as M, so that a thread owns a key (a TMEM lane) and sums
// its weights over the rows in a register: nothing is exchanged, nothing added atomically.  A unit is 256 keys, two
// tiles of 128 that stay in shared memory while tiles of 128 query rows go by; two S^T buffers a tile let
// the products of a step run under the exponentials of the one before.
//   warps 0-3, 4-7  the weights of key tile 0 / 1: thread = key
//   warp 8          stages K by TMA (8-bit caches: warps 12-15 convert the codes, without their scales, which
//                   go to the key's factor c)
//   warp 9          stages Q by TMA
//   warp 10         issues the MMAs
//   warp 11         stages the rows' x_i
// Rows of the last step that are no queries, and keys that a row does not see, are left out by intervals: the
// rows that see a key are one run of them.
// What bounds it is the exponentials: a step of 256 keys x 128 rows has 2048 cycles of them (an SM does 16 a cycle) and
// took 2900, the rest being what a warp waits for between its chunks (without them it took 1250, 1024 of them
// products).  2048 new tokens behind 30720 cached ones, 32 heads over 8 of 128: about 640 us behind the attention's 990;
// 16 x 5 tokens over 1 to 8 thousand: 44 us, of which K takes 21 to read.  Tried and no better: four warps a key tile more
// (1% here, 7 us more for the small case), a part of the exponentials by a polynomial on the FMA units (with
// those 6%, without 3% worse), four stages of Q.
#include <cuda.h>

#include "chunk_mass.cuh"
#include "pairs.cuh"
#include "sm100.cuh"

namespace snapmind {
namespace {

using namespace tc;

constexpr int kTile = 128, kUnit = 256, kRowsStep = 128;
constexpr uint32_t kBlockBytes = 128 * 128;  // 128 rows of 64 16-bit elements

template <int D> struct Shape {
  static constexpr uint32_t kTileBytes = D / 64 * kBlockBytes;
  static constexpr int kK = 2, kQ = 2;  // stages: of a unit's two K tiles, of Q
  static constexpr uint32_t kQRing = kK * 2 * kTileBytes, kCtrl = kQRing + kQ * kTileBytes;
  static constexpr uint32_t kGroup = D / 64 * 1024;  // K is [8-row group][64-column block][8 rows x 128 bytes]
};

struct Ctrl {
  uint64_t k_full[2], k_empty[2], q_full[2], q_empty[2], x_full[4], x_empty[4];
  uint64_t s_full[2][2], s_free[2][2];  // [key tile][buffer]
  uint64_t done;                        // every MMA has completed
  uint32_t tmem_base;
  int32_t abort;
  alignas(16) float x[4][kRowsStep];  // x_i of a step's rows
  MassShared plan;
};

template <int D> constexpr size_t smem_bytes() { return 1024 + Shape<D>::kCtrl + sizeof(Ctrl); }
static_assert(smem_bytes<128>() <= 232448, "shared memory budget");
static_assert(Shape<64>::kQRing >= kMaxChunkBatch * 4, "plan scratch in the K stages");

template <bool kQuant> struct Roles {
  static constexpr int kLoadK = 8, kLoadQ = kLoadK + 1, kMma = kLoadK + 2, kStats = kLoadK + 3, kConvert = kLoadK + 4;
  static constexpr int kThreads = (kConvert + (kQuant ? 4 : 0)) * 32;
};

__device__ __forceinline__ uint32_t low_bits(int k) { return k <= 0 ? 0u : k >= 32 ? ~0u : (1u << k) - 1u; }

__device__ __forceinline__ void give_up(Ctrl& C, int32_t* err) {
  atomicExch(&C.abort, 1);
  flag_error(err, SNAPMIND_DEVERR_TIMEOUT);
}

// A step: its first token, head and valid rows (a prefix).
struct Step {
  int i0, head0, valid;
  __device__ __forceinline__ Step(const ChunkParams& p, const MassPiece& c, int s) {
    const int run = p.n_slices == 1 ? s : s / p.n_slices, slice = s - run * p.n_slices;
    i0 = (c.r0 + run) * p.tokens;
    head0 = c.kvh * p.group + slice * p.gw;
    valid = (min(p.tokens, c.n - i0) - 1) * p.gw + slice_heads(p, slice);  // several slices: one token a step
  }
};

// tiles: mp.c for tiles of 128 keys.  kFull: no row of a step is left without a query (the heads divide 128), or its score
// does not matter: such a row is zeros of Q, and a key that holds an infinity would give it NaN, which an x of
// -infinity does not take out (an e4m3 row holds none, and with a NaN it is NaN for whoever sees it).  A NaN score of a row
// with a query goes with an x of NaN, so NaN scores may become numbers: one maximum each for the later half of the rows.  It
// costs calls of 3 heads a kv head 1% (2048 new of 32768: 1261 us, 1244 without); a branch on the row's number cost
// them 8%, and in the kernel of full steps 4%.
template <typename T, int D, bool kQuant, bool kFull>
__global__ void __launch_bounds__(Roles<kQuant>::kThreads, 1)
    mass_umma_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                     const __grid_constant__ MassParams mp, const __grid_constant__ ChunkParams tiles) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  using Sh = Shape<D>;
  using Ro = Roles<kQuant>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  const WeighedParams& p = mp.c;
  Ctrl& C = *reinterpret_cast<Ctrl*>(base + Sh::kCtrl);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&C.k_full[i]), kQuant ? 128 : 1);
      mbar_init(smem_u32(&C.k_empty[i]), 1);
      mbar_init(smem_u32(&C.q_full[i]), 1);
      mbar_init(smem_u32(&C.q_empty[i]), 1);
      for (int k = 2 * i; k < 2 * i + 2; ++k) {
        mbar_init(smem_u32(&C.x_full[k]), 2 * 32);
        mbar_init(smem_u32(&C.x_empty[k]), 8);
      }
      for (int t = 0; t < 2; ++t) {
        mbar_init(smem_u32(&C.s_full[t][i]), 1);
        mbar_init(smem_u32(&C.s_free[t][i]), 4);
      }
    }
    mbar_init(smem_u32(&C.done), 1);
    C.abort = 0;
    mbar_init_fence();
  }
  if (warp == Ro::kMma) {
    tmem_alloc(smem_u32(&C.tmem_base), 512);
    tmem_relinquish();
  }
  next_grid_may_launch();
  prior_grid_wait();
  mass_plan(mp, C.plan, reinterpret_cast<int32_t*>(base));
  // rows of Q that no copy fills (128 / gw has a remainder) are zeros, not whatever lay there
  for (uint32_t i = tid; i < Sh::kQ * Sh::kTileBytes / 16; i += Ro::kThreads)
    reinterpret_cast<uint4*>(base + Sh::kQRing)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = C.tmem_base;

  MassWalk w;
  bool on = w.start(p, C.plan), ok = true;
  if (warp >= Ro::kLoadK) {
    if (warp == Ro::kLoadK) {
      // ------------------------------------------------------------------ K copies
      if constexpr (!kQuant) {
        const uint32_t leader = elect_one_sync();
        uint32_t unit = 0;
        while (on && ok) {
          // one table walk for the tiles of a (sequence, head) that this CTA takes in a row
          Piece c = {};
          c.b = w.c.b;
          c.kvh = w.c.kvh;
          c.tile0 = 2 * w.c.tile;
          c.tile1 = 2 * w.n_tiles;
          TileRows at(tiles, w.kr, c, lane);
          const int b = w.c.b, kvh = w.c.kvh;
          for (int next = w.c.tile; on && w.c.b == b && w.c.kvh == kvh && w.c.tile == next; on = w.next(mp), ++unit, ++next) {
            const int st = unit % Sh::kK;
            ok = __all_sync(0xffffffffu, role_wait(C.abort, smem_u32(&C.k_empty[st]), ((unit / Sh::kK) & 1) ^ 1));
            if (!ok) break;
            const uint32_t bar = smem_u32(&C.k_full[st]);
            // both tiles' bytes are announced before either is copied (a batch of the table walk holds both)
            at.advance(2 * w.c.tile);
            const uint32_t have = __popc(at.have(2 * w.c.tile)) + __popc(at.have(2 * w.c.tile + 1));
            mbar_arrive_expect_tx_p(leader, bar, have * (uint32_t)at.box * (2 * D));
#pragma unroll 1
            for (int tile = 0; tile < 2; ++tile) {
              const uint32_t to = smem_u32(base + (st * 2 + tile) * Sh::kTileBytes);
#pragma unroll 1
              for (int x0 = 0; x0 < at.parts; x0 += 8) {
                int y[8];  // all rows first: a shuffle between two copies costs more than the copies
#pragma unroll
                for (int x = 0; x < 8; ++x) y[x] = at.row(2 * w.c.tile + tile, (x0 + x) & (at.parts - 1));
#pragma unroll
                for (int x = 0; x < 8; ++x)
                  tma_load_4d_p(x0 + x < at.parts && y[x] >= 0 ? leader : 0u, to + (x0 + x) * at.box * (D * 2), &k_map, 0, 0, 0, y[x] >> 3, bar);
              }
            }
          }
        }
        if (!ok && lane == 0) give_up(C, p.err);
        for (uint32_t i = unit > Sh::kK ? unit - Sh::kK : 0; i < unit; ++i)  // every copy issued has landed (bounded)
          mbar_wait(smem_u32(&C.k_full[i % Sh::kK]), (i / Sh::kK) & 1);
      }
    } else if (warp == Ro::kLoadQ) {
      // ------------------------------------------------------------------ Q copies
      const uint32_t leader = elect_one_sync();
      uint32_t q = 0;
      for (; on && ok; on = w.next(mp)) {
        for (int s = w.c.s0; s < w.c.s1; ++s, ++q) {
          const Step at(p, w.c, s);
          const int st = q % Sh::kQ;
          ok = __all_sync(0xffffffffu, role_wait(C.abort, smem_u32(&C.q_empty[st]), ((q / Sh::kQ) & 1) ^ 1));
          if (!ok) break;
          const uint32_t bar = smem_u32(&C.q_full[st]);
          mbar_arrive_expect_tx_p(leader, bar, D / 64 * p.tokens * p.gw * 128u);
#pragma unroll
          for (int kb = 0; kb < D / 64; ++kb)
            tma_load_3d_p(leader, smem_u32(base + Sh::kQRing + st * Sh::kTileBytes + kb * kBlockBytes), &q_map, 64 * kb, at.head0,
                          w.c.q_first + at.i0, bar);
        }
      }
      if (!ok && lane == 0) give_up(C, p.err);
      for (uint32_t i = q > Sh::kQ ? q - Sh::kQ : 0; i < q; ++i) mbar_wait(smem_u32(&C.q_full[i % Sh::kQ]), (i / Sh::kQ) & 1);
    } else if (warp == Ro::kMma) {
      // ------------------------------------------------------------------ MMA issue
      const uint32_t leader = elect_one_sync();
      constexpr uint32_t kIdesc = idesc_f16(kBf16, kTile, kRowsStep, false, false);
      const uint64_t k_desc = smem_desc(smem_u32(base), 16, Sh::kGroup, kSwizzle128B);
      const uint64_t q_desc = smem_desc(smem_u32(base + Sh::kQRing), 16, 1024, kSwizzle128B);
      uint32_t q = 0, unit = 0;
      const auto wait = [&](uint64_t* bar, uint32_t parity) {
        ok = ok && __all_sync(0xffffffffu, role_wait(C.abort, smem_u32(bar), parity));
        if (ok) tc_fence_after();
        return ok;
      };
      for (; on && ok; on = w.next(mp), ++unit) {
        if (!wait(&C.k_full[unit % Sh::kK], (unit / Sh::kK) & 1)) break;
        for (int s = w.c.s0; s < w.c.s1 && ok; ++s, ++q) {
          const int st = q % Sh::kQ, buf = q & 1;
          if (!wait(&C.q_full[st], (q / Sh::kQ) & 1)) break;
          for (int t = 0; t < 2; ++t) {
            if (!wait(&C.s_free[t][buf], ((q >> 1) & 1) ^ 1)) break;
            const uint64_t kd = k_desc + ((unit % Sh::kK) * 2 + t) * (Sh::kTileBytes >> 4), qd = q_desc + st * (Sh::kTileBytes >> 4);
#pragma unroll
            for (int kb = 0; kb < D / 64; ++kb)
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                umma_f16_p(leader, tmem + (t * 2 + buf) * kRowsStep, kd + ((kb * 1024 + kk * 32) >> 4),
                           qd + ((kb * kBlockBytes + kk * 32) >> 4), kIdesc, (kb > 0 || kk > 0) ? 1u : 0u);
            umma_commit_p(leader, smem_u32(&C.s_full[t][buf]));
          }
          if (ok) umma_commit_p(leader, smem_u32(&C.q_empty[st]));
        }
        if (ok) umma_commit_p(leader, smem_u32(&C.k_empty[unit % Sh::kK]));
      }
      if (!ok && lane == 0) give_up(C, p.err);
      // MMAs in flight end (bounded) before TMEM and shared memory go
      umma_commit_p(leader, smem_u32(&C.done));
      mbar_wait(smem_u32(&C.done), 0);
    } else if (warp == Ro::kStats) {
      // ------------------------------------------------------------------ x_i of the rows
      uint32_t q = 0;
      for (; on && ok; on = w.next(mp)) {
        for (int s = w.c.s0; s < w.c.s1; ++s, ++q) {
          const Step at(p, w.c, s);
          const uint32_t bar = smem_u32(&C.x_full[q & 3]);
          ok = __all_sync(0xffffffffu, role_wait(C.abort, smem_u32(&C.x_empty[q & 3]), ((q >> 2) & 1) ^ 1));
          if (!ok) break;
          // a step's rows lie side by side; they are copied, so that no step waits for the last one's
          const float* from = row_stats(p, w.c.kvh, w.c.q_first + at.i0, at.head0 - w.c.kvh * p.group);
          float* to = C.x[q & 3];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = lane + 32 * i;
            if (r < at.valid)
              asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(to + r)), "l"(from + r) : "memory");
            else
              to[r] = -INFINITY;
          }
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
          mbar_arrive(bar);
        }
      }
      if (!ok && lane == 0) give_up(C, p.err);
      asm volatile("cp.async.wait_all;" ::: "memory");  // no copy outlives the block
    } else if (kQuant && warp >= Ro::kConvert) {
      // ------------------------------------------------------------------ e4m3 codes -> 16-bit K tiles
      const int ct = tid - Ro::kConvert * 32;
      uint32_t unit = 0;
      for (; on && ok; on = w.next(mp), ++unit) {
        const int st = unit % Sh::kK;
        ok = __all_sync(0xffffffffu, role_wait(C.abort, smem_u32(&C.k_empty[st]), ((unit / Sh::kK) & 1) ^ 1));
        if (!ok) break;
        // D / 16 threads share a row, 16 codes each
        constexpr int kLanes = D / 16, kPass = 128 / kLanes;
        const int ch = ct % kLanes;
        for (int r = ct / kLanes; r < kUnit; r += kPass) {
          int pos;
          const int64_t row = mass_row(p, w.kr, w.c.b, w.c.kvh, w.c.tile, r, &pos);
          uint4 codes = make_uint4(0, 0, 0, 0);
          if (row >= 0) codes = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p.k_pool) + row * D + ch * 16);
          const uint32_t in[4] = {codes.x, codes.y, codes.z, codes.w};
          uint32_t o[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            codes_f16(in[i], o[2 * i], o[2 * i + 1]);
            if constexpr (kBf16) {
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&o[2 * i + j]));
                o[2 * i + j] = pack2<T>(f.x, f.y);
              }
            }
          }
          uint8_t* dst = base + (st * 2 + (r >> 7)) * Sh::kTileBytes + ((r & 127) >> 3) * Sh::kGroup + (ch / 4) * 1024 + (r & 7) * 128;
          const uint32_t c0 = (ch % 4) * 2, sw = r & 7;
          *reinterpret_cast<uint4*>(dst + ((c0 ^ sw) * 16)) = make_uint4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<uint4*>(dst + (((c0 + 1) ^ sw) * 16)) = make_uint4(o[4], o[5], o[6], o[7]);
        }
        fence_proxy_async_smem();
        mbar_arrive(smem_u32(&C.k_full[st]));
      }
      if (!ok && lane == 0) give_up(C, p.err);
    }
  } else {
    // ------------------------------------------------------------------ weights: thread = key
    const int t = warp >> 2, key = tid & 127;
    const uint32_t from0 = tmem + ((uint32_t)((warp & 3) * 32) << 16) + t * 2 * kRowsStep;
    const float c2 = p.scale * kLog2e;
    uint32_t q = 0;
    // the pool row of the thread's key is looked up a unit ahead
    int pos_next = 0;
    int64_t row_next = on ? mass_row(p, w.kr, w.c.b, w.c.kvh, w.c.tile, t * kTile + key, &pos_next) : -1;
    while (on && ok) {
      const MassPiece c = w.c;
      const int pos = pos_next, pos0 = w.kr.pos0;
      const int64_t row = row_next;
      float f = c2, old = 0.f;
      if (row >= 0) {
        if constexpr (kQuant) {
          const int64_t block = row / p.block_size;
          f = c2 * scale_byte_to_f(p.scales[block * p.block_size + row]);  // [block][head][2][slot]
        }
        if (c.whole()) old = mp.mass[row];
      }
      // of a row without a query (kFull): f low is finite; a query's score below it weighs nothing, or its x is NaN
      const float low = -3e38f / fmaxf(1.f, fabsf(f));
      on = w.next(mp);
      if (on) row_next = mass_row(p, w.kr, w.c.b, w.c.kvh, w.c.tile, t * kTile + key, &pos_next);
      // steps whose rows all see all of the warp's keys: first tokens from `from_i0` to `to_i0` (keys that are none do
      // not matter)
      const int far = 1 << 30;
      const int from_i0 = __reduce_max_sync(0xffffffffu, row >= 0 ? pos - pos0 : -far);
      const int to_i0 = min(c.n - p.tokens, __reduce_min_sync(0xffffffffu, row >= 0 && p.window > 0 && pos >= p.sinks
                                                                               ? (int)min((long long)pos + p.window - p.tokens - pos0, (long long)far)
                                                                               : far));
      int i0 = c.r0 * p.tokens + (p.n_slices == 1 ? c.s0 * p.tokens : 0);
      float sum = 0.f;
      for (int s = c.s0; s < c.s1; ++s, ++q, i0 += p.tokens) {
        ok = role_wait(C.abort, smem_u32(&C.x_full[q & 3]), (q >> 2) & 1) &&
             role_wait(C.abort, smem_u32(&C.s_full[t][q & 1]), (q >> 1) & 1);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t from = from0 + (q & 1) * kRowsStep;
        const float* xs = C.x[q & 3];
        float2 acc[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        if (i0 >= from_i0 && i0 <= to_i0 && p.n_slices == 1) {
          float v[2][32];
          tmem_ld32(from, v[0]);
#pragma unroll
          for (int k = 0; k < kRowsStep / 32; ++k) {
            float* u = v[k & 1];
            tmem_wait_ld32(u);
            if (k + 1 < kRowsStep / 32) {
              tmem_ld32(from + 32 * (k + 1), v[(k + 1) & 1]);
            } else {  // all scores have been read
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(smem_u32(&C.s_free[t][q & 1]));
            }
            if (!kFull && k >= kRowsStep / 64) {  // (more than half of a step's rows have queries)
#pragma unroll
              for (int i = 0; i < 32; ++i) u[i] = fmaxf(u[i], low);
            }
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const float4 x = *reinterpret_cast<const float4*>(xs + 32 * k + i);
              float2 a = fma2(make_float2(u[i], u[i + 1]), make_float2(f, f), make_float2(x.x, x.y));
              float2 b = fma2(make_float2(u[i + 2], u[i + 3]), make_float2(f, f), make_float2(x.z, x.w));
              a = make_float2(ex2(a.x), ex2(a.y));
              b = make_float2(ex2(b.x), ex2(b.y));
              acc[0] = add2(acc[0], a);
              acc[1] = add2(acc[1], b);
            }
          }
        } else {
          const Step at(p, c, s);
          // the rows that see the key: tokens [pos - qpos0, pos + window - qpos0) of the step's
          const int qpos0 = pos0 + at.i0;
          int lo = 0, hi = 0;
          if (row >= 0) {
            lo = min(max(pos - qpos0, 0), kRowsStep) * p.gw;
            hi = at.valid;
            if (p.window > 0 && pos >= p.sinks)
              hi = min(hi, (int)min(max((long long)pos + p.window - qpos0, 0ll), (long long)kRowsStep) * p.gw);
          }
          if (__any_sync(0xffffffffu, lo < hi)) {
#pragma unroll 1
            for (int x0 = 0; x0 < at.valid; x0 += 32) {
              float v[32];
              tmem_ld32(from + x0, v);
              const uint32_t see = low_bits(hi - x0) & ~low_bits(lo - x0);
              tmem_wait_ld32(v);
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                const float2 x = *reinterpret_cast<const float2*>(xs + x0 + i);
                float2 a = fma2(make_float2(v[i], v[i + 1]), make_float2(f, f), x);
                if (!(see >> i & 1)) a.x = -INFINITY;
                if (!(see >> (i + 1) & 1)) a.y = -INFINITY;
                a.x = ex2(a.x);
                a.y = ex2(a.y);
                acc[(i >> 1) & 1] = add2(acc[(i >> 1) & 1], a);
              }
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&C.s_free[t][q & 1]));
        }
        sum += (acc[0].x + acc[0].y) + (acc[1].x + acc[1].y);
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&C.x_empty[q & 3]));
      }
      if (!ok) break;
      if (!c.whole()) mp.part[mass_slot(c) * kUnit + t * kTile + key] = sum;
      else if (row >= 0) mp.mass[row] = old + sum;
    }
    if (!ok && lane == 0) give_up(C, p.err);
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0) write_mass_info(mp, C.plan);
  if (warp == Ro::kMma) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Q as [token][head][dim]: a box is the gw heads of a slice of 128 / gw tokens, 64 columns.
bool q_step_map(CUtensorMap* map, bool bf16, const ChunkParams& p, int D) {
  EncodeTiledFn fn = encode_tiled();
  if (!fn) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)p.n_q_heads, (cuuint64_t)p.total_q};
  const cuuint64_t strides[2] = {(cuuint64_t)p.q_stride_head * 2, (cuuint64_t)p.q_stride_tok * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)p.gw, (cuuint32_t)p.tokens};
  const cuuint32_t estr[3] = {1, 1, 1};
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(p.q), dims,
            strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D, bool kQuant, bool kFull>
int launch_geometry(MassParams& mp, cudaStream_t st) {
  ChunkParams tiles = mp.c;
  tiles.key_tile = kTile;
  tiles.by_tile = FastDiv(kTile);
  CUtensorMap q_map, k_map = {};
  const uint64_t rows = (uint64_t)mp.c.num_blocks * mp.c.n_kv_heads * mp.c.block_size;
  const uint32_t box = mp.c.block_size < kTile ? mp.c.block_size : kTile;
  const bool bf16 = std::is_same<T, __nv_bfloat16>::value;
  if ((!kQuant && !tensor_map_row_groups(&k_map, bf16, mp.c.k_pool, rows, D, box / 8)) || !q_step_map(&q_map, bf16, mp.c, D))
    return SNAPMIND_ERR_UNSUPPORTED;  // the caller takes the CUDA-core kernel
  auto kernel = mass_umma_kernel<T, D, kQuant, kFull>;
  static bool done[kMaxDevices] = {};
  const cudaError_t e = kernel_attributes(reinterpret_cast<const void*>(kernel), smem_bytes<D>(), done);
  if (e != cudaSuccess) return cuda_status(e, "paged_chunk mass smem attribute");
  const int status = cuda_status(launch_dependent(kernel, dim3(mp.c.n_ctas), Roles<kQuant>::kThreads, smem_bytes<D>(), st, q_map, k_map, mp, tiles),
                                 "paged_chunk mass launch");
  return status != SNAPMIND_OK ? status : launch_mass_merge(mp, st);
}

template <typename T, int D, bool kQuant>
int launch(MassParams& mp, cudaStream_t st) {
  const int rc = mass_geometry(mp, kRowsStep, kUnit, num_sms());
  if (rc != SNAPMIND_OK) return rc;
  if constexpr (!kQuant)
    if (mp.c.tokens * mp.c.gw < kRowsStep) return launch_geometry<T, D, kQuant, false>(mp, st);
  return launch_geometry<T, D, kQuant, true>(mp, st);
}

}  // namespace

int launch_mass_umma(MassParams& mp, int dtype, int pool_dtype, cudaStream_t st) {
  const bool quant = pool_dtype == SNAPMIND_DTYPE_E4M3;
  const auto go = [&](auto t) -> int {
    using T = decltype(t);
    if (mp.c.head_dim == 64) return quant ? launch<T, 64, true>(mp, st) : launch<T, 64, false>(mp, st);
    return quant ? launch<T, 128, true>(mp, st) : launch<T, 128, false>(mp, st);
  };
  return dtype == SNAPMIND_DTYPE_BF16 ? go(__nv_bfloat16()) : go(__half());
}

}  // namespace snapmind
