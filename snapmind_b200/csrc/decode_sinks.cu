// One token per sequence over a paged cache with a sliding window and sinks, or over an
// 8-bit cache: head_dim 128, query groups of up to 8 heads, bf16 / f16 queries.
//
// HBM bound (4 flop per 16-bit byte read), so the matrix product is mma.sync with the
// keys as M, as in paged_decode_fast.cu: S^T = K Q^T, O^T += V^T P^T, 16 keys per warp.  What
// is different: the CTAs (two per SM) walk equal shares of the work line of chunk_plan.cuh,
// which jumps from the sink blocks to the window's, and the pipeline runs on from
// one unit to the next, so a batch of uneven lengths keeps every SM streaming to the end.
// 128 sequences of 1024 to 8192 tokens, 32 heads over 8: a window of 4096 with 4 sinks 268 us (6.6 TB/s, a
// copy's rate), the whole 8-bit cache 211 us (6.05 TB/s, 0.93 of it).  One sequence and a window of 1024
// take 11.4 us, four 8-bit ones 18: launch, plan (2 to 3 us), one tile's latency and the merge.  (Replayed
// from a graph; called from Python back to back 274, 237, 15 and 19 us.)
//
// e4m3 rows (c 2^e, a byte e + 127 per row): the codes become f16 in registers (exact), and
// the scales never touch the elements: K's multiplies its key's score, V's its weight.
// With s the score in log2 units and e_v the exponent of V's row, the weight that multiplies the
// codes is 2^(s + e_v - R), R = max (s + e_v), a good f16 whatever the rows' scales are.  The sum
// has a reference of its own, 2^(s - M), M = max s: R - M may be anything in [-100, 120] and s + e_v
// differ by more than f32's exponents between rows that count alike (a row of zeros has e = -100), so
// neither can be had from the other.  A piece's result is O 2^(R - M) / sum, a mean of V.  Queries are
// brought to [2^8, 2^9) by a power of two per head, so f16 holds a bf16 query as exactly as the
// f32 sum needs.  Both type conversions take permuted dims (K) and pairs of dims (V), so that
// ldmatrix can move bytes in 16-bit units:
//   K: lane (g, t) holds dims 16 k + 4 t .. + 3 of key g as k-slots 2 t, 2 t + 1, 2 t + 8, 2 t + 9;
//   V: row g / g + 8 of a 16-dim step stands for dim 2 g / 2 g + 1.
#include <cuda.h>

#include "chunk_plan.cuh"
#include "pairs.cuh"
#include "sm100.cuh"

namespace snapmind {
namespace {

using namespace tc;

constexpr int kD = 128, kTile = 64, kConsumers = 4, kThreads = (kConsumers + 2) * 32, kHeads = 8;
constexpr int kScaleLanes = kTile / 16;  // lanes that fetch a tile's scale bytes of K, or of V, 16 each
// A raised reference stands 2^kLow below the maximum, and stays until a score passes it by 2^kRaise
// (weights up to 2^kRaise are as good as those up to 1).  f16 weights go up to 2^15: what is 2^25
// below the largest weight would vanish if that were 1, although thousands of such keys behind a
// strong sink may be all that shows; 2^7 further up, a weight is off by 2^-32 of the largest at most.
template <bool kBf16> constexpr float kLow = kBf16 ? 0.f : 7.f;
template <bool kBf16> constexpr float kRaise = kLow<kBf16> + 8.f;
constexpr float kNone = -3e38f;  // a reference before any score: finite, so that -infinity less it stays one

template <bool kQuant> struct Stage {
  static constexpr int kHalf = kTile * 128;                      // 64 rows of 128 bytes
  static constexpr int kK = 0, kV = kQuant ? kHalf : 2 * kHalf;  // 16-bit rows are two halves of 64 dims
  static constexpr int kBytes = kQuant ? 2 * kHalf : 4 * kHalf;
  static constexpr int kCount = kQuant ? 5 : 3;
};

template <bool kQuant>
struct Ctrl {
  static constexpr int N = Stage<kQuant>::kCount;
  float mo[2][kHeads][kD];
  alignas(16) uint8_t scales[kQuant ? N : 1][2][kTile];  // K, V bytes of a stage's rows (16-byte copies)
  float mm[kConsumers][kHeads], ml[kConsumers][kHeads];  // M, sum
  float mr[kConsumers][kHeads];                          // R (16-bit caches: M)
  uint64_t full[N], empty[N];
  uint32_t have[N];  // parts of a stage's tile that were there to be copied
  int32_t rows[N][kTile / 16];  // their score rows (kScores)
  int32_t abort;
  PlanShared plan;
};
template <bool kQuant> constexpr size_t smem_bytes() {
  return 1024 + Stage<kQuant>::kCount * Stage<kQuant>::kBytes + sizeof(Ctrl<kQuant>);
}
static_assert(2 * (smem_bytes<false>() + 1024) <= 233472 && 2 * (smem_bytes<true>() + 1024) <= 233472, "two CTAs per SM");
static_assert(Stage<true>::kCount * Stage<true>::kBytes >= kMaxChunkBatch * 4, "plan scratch in the ring");

__device__ __forceinline__ void ldsm_x4(uint32_t a, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a));
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t a, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a));
}
template <bool kBf16>
__device__ __forceinline__ void mma16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if constexpr (kBf16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Byte offset of 16-byte piece `ch` (0..7) of row `row` in rows of 128 bytes, 128-byte swizzle.
__device__ __forceinline__ uint32_t swz(int row, int ch) { return row * 128 + ((ch ^ (row & 7)) << 4); }

// 16 bytes global -> shared by the calling thread, then its arrival on `bar` once they landed.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ bool consumers_any(bool v) {
  uint32_t r;
  asm volatile("{ .reg .pred p, q; setp.ne.u32 p, %1, 0; bar.red.or.pred q, 1, 128, p; selp.u32 %0, 1, 0, q; }"
               : "=r"(r)
               : "r"((uint32_t)v)
               : "memory");
  return r != 0;
}

// kScores: the rows' softmax sums go to p.stats, and the scores of the tokens to p.scores where there is room for them, for
// the pass that adds their weights up (128 sequences of 1 to 8 thousand tokens: 3% more bytes than the decode without).
template <typename T, bool kQuant, bool kScores>
__global__ void __launch_bounds__(kThreads, 2)
    decode_sinks_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, CallParams<kScores> p) {
  extern __shared__ uint8_t smem_raw[];
  using St = Stage<kQuant>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr bool kMmaBf16 = kBf16 && !kQuant;
  // weights are the 16-bit operand of one product: off by half a step (2^-8 of themselves in bf16, 2^-11 in f16: outputs of
  // 8-bit caches have a relative RMS error of 0.00027, 0.00021 with f32 weights); their sum stays f32
  using Weight = typename std::conditional<kMmaBf16, __nv_bfloat16, __half>::type;
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  auto& S = *reinterpret_cast<Ctrl<kQuant>*>(ring + St::kCount * St::kBytes);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < St::kCount; ++i) {
      mbar_init(smem_u32(&S.full[i]), kQuant ? 2 * (1 + kScaleLanes) : 2);
      mbar_init(smem_u32(&S.empty[i]), kConsumers);
    }
    S.abort = 0;
    mbar_init_fence();
  }
  prior_grid_wait();
  plan_block(p, S.plan, reinterpret_cast<int32_t*>(ring));
  fence_proxy_async_smem();  // the scratch in the ring is done with before copies land there
  __syncthreads();

  PieceWalk w;
  bool on = w.start(S.plan);
  uint32_t tile = 0;  // running number of the CTA's tiles
  bool ok = true;
  if (warp >= kConsumers) {
    // ------------------------------------------------------------------ producers: K, V
    const int kv = warp - kConsumers;
    const CUtensorMap* map = kv == 0 ? &k_map : &v_map;
    const uint32_t leader = elect_one_sync();
    // the scale bytes that a lane fetches: keys scale_key .. + 15, from part scale_part
    const int scale_key = (lane & (kScaleLanes - 1)) * 16;
    const int scale_part = p.block_size < kTile ? p.by_block.div(scale_key) : 0;
    const int scale_in = scale_key - scale_part * min(p.block_size, kTile);
    for (; on && ok; on = w.next(p)) {
      const Piece& c = w.c;
      const KeyRange kr = key_range(p, c.len, c.n, c.i0, c.i0 + 1);
      TileRows at(p, kr, c, lane);
      const int box = at.box;
      for (int j = c.tile0; j < c.tile1; ++j, ++tile) {
        at.advance(j);
        const uint32_t have = at.have(j);
        const int st = tile % St::kCount;
        ok = __all_sync(0xffffffffu, role_wait(S.abort, smem_u32(&S.empty[st]), ((tile / St::kCount) & 1) ^ 1));
        if (!ok) break;
        const uint32_t bar = smem_u32(&S.full[st]);
        const uint32_t row_bytes = kQuant ? 128 : 2 * 128;
        if (kv == 0 && leader) S.have[st] = have;
        if constexpr (kScores) {
          const int y = at.row(j, lane & (at.parts - 1));
          if (kv == 0 && lane < at.parts)
            S.rows[st][lane] = p.scores_room > 0 ? (c.b * p.n_kv_heads + c.kvh) * p.scores_room + j * kTile + lane * box : y;
          __syncwarp();
        }
        mbar_arrive_expect_tx_p(leader, bar, __popc(have) * (uint32_t)box * row_bytes);
        const uint32_t dst = smem_u32(ring + st * St::kBytes + (kv == 0 ? St::kK : St::kV));
        if constexpr (kQuant) {
          // the scales go by plain 16-byte copies, not as small bulk copies beside the boxes
          const int sr = at.row(j, scale_part);
          if (lane < kScaleLanes) {
            if (sr >= 0) copy16(smem_u32(&S.scales[st][kv][scale_key]), p.scales + at.scale_at(sr + scale_in, kv));
            copies_arrive(bar);
          }
        }
        int ys[kTile / 16];  // all rows first: a shuffle between two copies costs more than the copies
#pragma unroll
        for (int x = 0; x < kTile / 16; ++x) ys[x] = at.row(j, x & (at.parts - 1));
#pragma unroll
        for (int x = 0; x < kTile / 16; ++x) {  // parts that are not there are predicated off
          const int y = ys[x];
          const uint32_t go = x < at.parts && y >= 0 ? leader : 0u;
          const uint32_t ro = x * box * 128;
          tma_load_2d_p(go, dst + ro, map, 0, y, bar);
          if constexpr (!kQuant) tma_load_2d_p(go, dst + St::kHalf + ro, map, 64, y, bar);
        }
      }
    }
    if (!ok && lane == 0) {
      flag_error(p.err, SNAPMIND_DEVERR_TIMEOUT);
      atomicExch(&S.abort, 1);
    }
    // every copy issued lands (bounded) before the shared memory goes
    for (uint32_t i = tile > St::kCount ? tile - St::kCount : 0; i < tile; ++i)
      mbar_wait(smem_u32(&S.full[i % St::kCount]), (i / St::kCount) & 1);
  } else {
    // ------------------------------------------------------------------ consumers
    const int g = lane >> 2, tig = lane & 3;
    const int lrow = (lane & 7) + ((lane >> 3) & 1) * 8, lchk = lane >> 4;
    const int vrow = (lane & 7) + ((lane >> 4) & 1) * 8, vchk = (lane >> 3) & 1;  // 16-bit V
    // offsets of the lane's rows in a stage: e4m3 pieces k + lchk of K and of V, 16-bit pieces 2 k + ..
    uint32_t k_off[4], v_off[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      k_off[k] = swz(16 * warp + lrow, 2 * k + lchk);
      v_off[k] = kQuant ? k_off[k] : swz(16 * warp + vrow, 2 * k + vchk);
    }
    const int part = p.block_size < kTile ? p.by_block.div(16 * warp) : 0;  // the warp's keys in a tile
    const bool flip = p.scale < 0.f;  // folded into Q: the largest score has the largest weight
    const float c2 = fmaxf(fabsf(p.scale) * kLog2e, 1e-37f);
    for (; on; on = w.next(p)) {
      const Piece& c = w.c;
      const KeyRange kr = key_range(p, c.len, c.n, c.i0, c.i0 + 1);
      const int heads = slice_heads(p, c.slice), head0 = c.kvh * p.group + c.slice * p.gw;
      // keys seen: [0, v_s) and [v_lo, v_len) of the virtual axis
      const int v_lo = kr.win_lo - kr.shift, v_s = p.window > 0 ? min(p.sinks, kr.v_sink) : 0;
      uint32_t qf[8][2];
      float q0 = c2, q1 = c2;            // factors of heads 2 tig, 2 tig + 1
      uint32_t down0 = 0, down1 = 0;     // e4m3: powers of two (in exponent bits) that K's scales leave to them
      {
        const T* qrow = reinterpret_cast<const T*>(p.q) + (int64_t)c.q_first * p.q_stride_tok +
                        (int64_t)(head0 + min(g, heads - 1)) * p.q_stride_head;
        if constexpr (kQuant) {
          float x[32], a = 0.f;
#pragma unroll
          for (int k = 0; k < 8; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              x[4 * k + i] = Conv<T>::to_f(qrow[16 * k + 4 * tig + i]);
              a = fmaxf(a, fabsf(x[4 * k + i]));
            }
          a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 1));
          a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 2));
          // a 2^-e in [2^8, 2^9); 0 and what is not finite keep any e
          const int e = min(max((int)(__float_as_uint(a) >> 23) - 127, -110), 127) - 8;
          const float up = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
          for (int k = 0; k < 8; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i) qf[k][i] = pack2<__half>(x[4 * k + 2 * i] * up, x[4 * k + 2 * i + 1] * up);
          // A sum of products is below 2^25 (128 x 448 x 2^9), K's scale at most 2^120: 2^17 of it goes
          // to the head's factor, so that what overflows is a score, not a step towards one.  (A query above
          // 2^110 has no room for it and needs none.)
          const int down = e < 100 ? 17 : 0;
          const float f = c2 * __uint_as_float((uint32_t)(127 + down + e) << 23);  // of head g
          q0 = __shfl_sync(0xffffffffu, f, 8 * tig);
          q1 = __shfl_sync(0xffffffffu, f, 8 * tig + 4);
          down0 = __shfl_sync(0xffffffffu, (uint32_t)down << 23, 8 * tig);
          down1 = __shfl_sync(0xffffffffu, (uint32_t)down << 23, 8 * tig + 4);
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i) qf[k][i] = *reinterpret_cast<const uint32_t*>(qrow + 16 * k + 8 * i + 2 * tig);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (g >= heads) qf[k][i] = 0u;
            if (flip) qf[k][i] ^= 0x80008000u;
          }
      }
      float o[8][4];
#pragma unroll
      for (int k = 0; k < 8; ++k) o[k][0] = o[k][1] = o[k][2] = o[k][3] = 0.f;
      float m0 = kNone, m1 = kNone, l0 = 0.f, l1 = 0.f;  // M (log2 units), sum
      float R0 = kNone, R1 = kNone;                      // R
      for (int j = c.tile0; j < c.tile1; ++j, ++tile) {
        const int st = tile % St::kCount;
        ok = __all_sync(0xffffffffu, role_wait(S.abort, smem_u32(&S.full[st]), (tile / St::kCount) & 1));
        if (!ok) break;
        uint8_t* stage = ring + st * St::kBytes;
        const uint32_t kb = smem_u32(stage + St::kK), vb = smem_u32(stage + St::kV);
        const int v0 = j * kTile + 16 * warp;
        const bool there = S.have[st] >> part & 1;
        const auto seen = [&](int i) { return there && v0 + i < kr.v_len && (v0 + i >= v_lo || v0 + i < v_s); };
        const bool all = there && v0 + 16 <= kr.v_len && (v0 >= v_lo || v0 + 16 <= v_s);
        if (all || __any_sync(0xffffffffu, seen(lane & 15))) {
          if (!all) {
            // rows of V that are not seen become zeros: 0 x (whatever lies there) must not reach O
            for (int e = lane; e < 16 * 8; e += 32) {
              const int i = e >> 3;
              if (!seen(i)) {
                const uint32_t off = swz(16 * warp + i, e & 7);
                *reinterpret_cast<uint4*>(stage + St::kV + off) = make_uint4(0, 0, 0, 0);
                if (!kQuant) *reinterpret_cast<uint4*>(stage + St::kV + St::kHalf + off) = make_uint4(0, 0, 0, 0);
              }
            }
            __syncwarp();
          }
          // ---- S^T = K Q^T: 16 keys x 8 heads; keys g and g + 8, heads 2 tig, 2 tig + 1
          float sc[4] = {0.f, 0.f, 0.f, 0.f};
          float sv0 = 0.f, sv1 = 0.f;  // e_v of V's rows g, g + 8
          if constexpr (kQuant) {
#pragma unroll
            for (int k = 0; k < 8; k += 2) {
              uint32_t r[4];
              ldsm_x4(kb + k_off[k / 2], r);
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                uint32_t a[4];
                codes_f16(r[2 * i], a[0], a[2]);
                codes_f16(r[2 * i + 1], a[1], a[3]);
                mma16816<false>(sc, a, qf[k + i][0], qf[k + i][1]);
              }
            }
            const uint8_t* bytes = &S.scales[st][0][16 * warp];
            const uint32_t e0 = (uint32_t)bytes[g] << 23, e1 = (uint32_t)bytes[g + 8] << 23;
            sv0 = (float)((int)bytes[kTile + g] - 127);
            sv1 = (float)((int)bytes[kTile + g + 8] - 127);
            sc[0] *= __uint_as_float(e0 - down0);
            sc[1] *= __uint_as_float(e0 - down1);
            sc[2] *= __uint_as_float(e1 - down0);
            sc[3] *= __uint_as_float(e1 - down1);
          } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              uint32_t a[4];
              ldsm_x4(kb + (k >> 2) * St::kHalf + k_off[k & 3], a);
              mma16816<kMmaBf16>(sc, a, qf[k][0], qf[k][1]);
            }
          }
          if constexpr (kScores) {
            if (p.scores != nullptr) {
              // a key's scores side by side: 16 bytes for four heads (rows past the last token, unseen ones: never read)
              const int64_t row = S.rows[st][part] + 16 * warp - part * p.block_size;
#pragma unroll
              for (int i = 0; i < 4; i += 2) {
                float* to = p.scores + (row + g + 4 * i) * heads + 2 * tig;
                const float a = sc[i] * q0, b = sc[i + 1] * q1;
                if (heads % 2 == 0) {
                  if (2 * tig < heads) *reinterpret_cast<float2*>(to) = make_float2(a, b);
                } else {
                  if (2 * tig < heads) to[0] = a;
                  if (2 * tig + 1 < heads) to[1] = b;
                }
              }
            }
          }
          // Scores less their references: xs for the sum, ys for the weights (16-bit caches: xs).  When a
          // reference is raised, what was summed is rescaled.
          float xs[4], ys[4];
          const auto refer = [&](float M0, float M1, float r0, float r1) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float f = i & 1 ? q1 : q0, sv = i & 2 ? sv1 : sv0;
              xs[i] = fmaf(sc[i], f, i & 1 ? -M1 : -M0);
              ys[i] = kQuant ? fmaf(sc[i], f, sv - (i & 1 ? r1 : r0)) : xs[i];
            }
            if (!all) {
              if (!seen(g)) xs[0] = xs[1] = ys[0] = ys[1] = -INFINITY;
              if (!seen(g + 8)) xs[2] = xs[3] = ys[2] = ys[3] = -INFINITY;
            }
          };
          refer(m0, m1, R0, R1);
          float top = fmaxf(fmaxf(xs[0], xs[1]), fmaxf(xs[2], xs[3]));
          if constexpr (kQuant) top = fmaxf(top, fmaxf(fmaxf(ys[0], ys[1]), fmaxf(ys[2], ys[3])));
          if (__any_sync(0xffffffffu, top > kRaise<kMmaBf16>)) {
            refer(0.f, 0.f, 0.f, 0.f);
            const auto raised = [](float& ref, float a, float b) {  // the factor of what was summed before
              float n = fmaxf(a, b);
#pragma unroll
              for (int off = 4; off < 32; off <<= 1) n = fmaxf(n, __shfl_xor_sync(0xffffffffu, n, off));
              n = fmaxf(n - kLow<kMmaBf16>, ref);
              const float f = ex2(ref - n);
              ref = n;
              return f;
            };
            float b0 = raised(m0, xs[0], xs[2]), b1 = raised(m1, xs[1], xs[3]);
            l0 *= b0;
            l1 *= b1;
            if constexpr (kQuant) {
              b0 = raised(R0, ys[0], ys[2]);
              b1 = raised(R1, ys[1], ys[3]);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              o[k][0] *= b0;
              o[k][1] *= b1;
              o[k][2] *= b0;
              o[k][3] *= b1;
            }
            refer(m0, m1, R0, R1);
          }
          const float p0 = ex2(ys[0]), p1 = ex2(ys[1]), p2 = ex2(ys[2]), p3 = ex2(ys[3]);
          l0 += kQuant ? ex2(xs[0]) + ex2(xs[2]) : p0 + p2;
          l1 += kQuant ? ex2(xs[1]) + ex2(xs[3]) : p1 + p3;
          // ---- P^T as the B operand: lane (g, tig) needs keys 2 tig, + 1, + 8, + 9 of head g
          const uint32_t pr01 = pack2<Weight>(p0, p1), pr23 = pack2<Weight>(p2, p3);
          const int src = 8 * tig + (g >> 1);
          const uint32_t sel = (g & 1) ? 0x7632u : 0x5410u;
          const auto operand = [&](uint32_t r) {
            const uint32_t x = __shfl_sync(0xffffffffu, r, src), y = __shfl_sync(0xffffffffu, r, src + 4);
            return __byte_perm(x, y, sel);
          };
          const uint32_t pb0 = operand(pr01), pb1 = operand(pr23);
          // bf16 weights next to scores that are kept: what their rounding leaves multiplies V as well (the weights are
          // then off by 2^-16 and not 2^-8 of themselves; the products of an HBM-bound kernel have the room)
          uint32_t rb0 = 0, rb1 = 0;
          if constexpr (kScores && kMmaBf16) {
            const auto left = [](uint32_t r, float lo, float hi) {
              return pack2<Weight>(lo - __uint_as_float(r << 16), hi - __uint_as_float(r & 0xFFFF0000u));
            };
            rb0 = operand(left(pr01, p0, p1));
            rb1 = operand(left(pr23, p2, p3));
          }
          // ---- O^T += V^T P^T: 128 dims x 8 heads
          if constexpr (kQuant) {
#pragma unroll
            for (int k = 0; k < 8; k += 2) {
              uint32_t r[4];
              ldsm_x4_t(vb + v_off[k / 2], r);
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                uint32_t a[4];
                codes_f16(__byte_perm(r[2 * i], 0, 0x3120), a[0], a[1]);
                codes_f16(__byte_perm(r[2 * i + 1], 0, 0x3120), a[2], a[3]);
                mma16816<false>(o[k + i], a, pb0, pb1);
              }
            }
          } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              uint32_t a[4];
              ldsm_x4_t(vb + (k >> 2) * St::kHalf + v_off[k & 3], a);
              mma16816<kMmaBf16>(o[k], a, pb0, pb1);
              if constexpr (kScores && kMmaBf16) mma16816<kMmaBf16>(o[k], a, rb0, rb1);
            }
          }
          if (!all) fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&S.empty[st]));
      }
      // ---- the four warps' states, merged; every consumer takes these barriers
      if (!kQuant) R0 = m0, R1 = m1;
      const auto known = [](float& ref) { ref = ref == kNone ? -INFINITY : ref; };  // nothing seen, or only NaN
      known(m0), known(m1), known(R0), known(R1);
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, off);
        l1 += __shfl_xor_sync(0xffffffffu, l1, off);
      }
      if (g == 0) {
        S.mm[warp][2 * tig] = m0;
        S.mm[warp][2 * tig + 1] = m1;
        S.ml[warp][2 * tig] = l0;
        S.ml[warp][2 * tig + 1] = l1;
        S.mr[warp][2 * tig] = R0;
        S.mr[warp][2 * tig + 1] = R1;
      }
      if (consumers_any(!ok)) {
        ok = false;
        break;
      }
      float M0 = -INFINITY, M1 = -INFINITY;  // of R
#pragma unroll
      for (int x = 0; x < kConsumers; ++x) {
        M0 = fmaxf(M0, S.mr[x][2 * tig]);
        M1 = fmaxf(M1, S.mr[x][2 * tig + 1]);
      }
      const float f0 = R0 == -INFINITY ? 0.f : ex2(R0 - M0), f1 = R1 == -INFINITY ? 0.f : ex2(R1 - M1);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        o[k][0] *= f0;
        o[k][1] *= f1;
        o[k][2] *= f0;
        o[k][3] *= f1;
      }
      const int slot = warp & 1;
#pragma unroll
      for (int half = 0; half < 2; ++half) {  // warps 2 and 3 write, then 0 and 1 add theirs
        if ((warp >= 2) == (half == 0)) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int d0 = 16 * k + (kQuant ? 2 * g : g), d1 = d0 + (kQuant ? 1 : 8);
            float* r0 = S.mo[slot][2 * tig];
            float* r1 = S.mo[slot][2 * tig + 1];
            if (half == 0) {
              r0[d0] = o[k][0];
              r1[d0] = o[k][1];
              r0[d1] = o[k][2];
              r1[d1] = o[k][3];
            } else {
              r0[d0] += o[k][0];
              r1[d0] += o[k][1];
              r0[d1] += o[k][2];
              r1[d1] += o[k][3];
            }
          }
        }
        consumers_sync();
      }
      const int h = tid >> 4, d = (tid & 15) * 8;  // a head's 8 dims per thread
      if (h < heads) {
        float M = -INFINITY, L = 0.f, x[8];
#pragma unroll
        for (int i = 0; i < kConsumers; ++i) M = fmaxf(M, S.mm[i][h]);
#pragma unroll
        for (int i = 0; i < kConsumers; ++i) L += S.mm[i][h] == -INFINITY ? S.ml[i][h] : S.ml[i][h] * ex2(S.mm[i][h] - M);  // 0, or NaN
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
          const float4 a = *reinterpret_cast<const float4*>(&S.mo[0][h][d + i]);
          const float4 b = *reinterpret_cast<const float4*>(&S.mo[1][h][d + i]);
          x[i] = a.x + b.x;
          x[i + 1] = a.y + b.y;
          x[i + 2] = a.z + b.z;
          x[i + 3] = a.w + b.w;
        }
        const float inv = L == 0.f ? 0.f : 1.f / L;  // nothing seen: zeros
        if constexpr (kQuant) {
          // the mean of V, of a piece too: 2^(R - M) in two halves, since R - M can pass f32's exponents
          float R = -INFINITY;
#pragma unroll
          for (int i = 0; i < kConsumers; ++i) R = fmaxf(R, S.mr[i][h]);
          const float half = R == -INFINITY ? 0.f : ex2(0.5f * (R - M));
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * half * half;
        }
        if (c.whole()) {
          if constexpr (kScores)
            if (d == 0) write_stats(p, c.q_first, head0 + h, M, L);
          if constexpr (!kQuant)
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] *= inv;
          T* out = reinterpret_cast<T*>(p.out) + (int64_t)c.q_first * p.out_stride_tok + (int64_t)(head0 + h) * p.out_stride_head + d;
          *reinterpret_cast<uint4*>(out) = make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]),
                                                      pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
        } else {
          const int64_t row = part_slot(c) * p.rows + h;
          if (d == 0) {
            p.part_ml[row * 2] = M;
            p.part_ml[row * 2 + 1] = L;
          }
          *reinterpret_cast<float4*>(p.part_o + row * kD + d) = make_float4(x[0], x[1], x[2], x[3]);
          *reinterpret_cast<float4*>(p.part_o + row * kD + d + 4) = make_float4(x[4], x[5], x[6], x[7]);
        }
      }
      // the next piece's mm and ml are written after its own barrier-free part only once every
      // thread has read these
      consumers_sync();
    }
    if (!ok && lane == 0) {
      flag_error(p.err, SNAPMIND_DEVERR_TIMEOUT);
      atomicExch(&S.abort, 1);
    }
  }
  __syncthreads();
  if (tid == 0) write_piece_info(p, S.plan);
  next_grid_may_launch();
}

template <typename T, bool kQuant, bool kScores>
int launch(const WeighedParams& p, cudaStream_t st) {
  CUtensorMap k_map, v_map;
  const uint64_t rows = (uint64_t)p.num_blocks * p.n_kv_heads * p.block_size;
  const uint32_t box = p.block_size < kTile ? p.block_size : kTile;
  const bool bf16 = std::is_same<T, __nv_bfloat16>::value;
  const bool mapped = kQuant ? tensor_map_bytes(&k_map, p.k_pool, kD, rows, box, true) && tensor_map_bytes(&v_map, p.v_pool, kD, rows, box, true)
                             : tensor_map_2d(&k_map, bf16, p.k_pool, kD, rows, kD * 2, 64, box) &&
                                   tensor_map_2d(&v_map, bf16, p.v_pool, kD, rows, kD * 2, 64, box);
  if (!mapped) {
    set_last_error("paged_chunk: tensor map encoding failed");
    return SNAPMIND_ERR_CUDA;
  }
  auto kernel = decode_sinks_kernel<T, kQuant, kScores>;
  static bool done[kMaxDevices] = {};
  const cudaError_t e = kernel_attributes(reinterpret_cast<const void*>(kernel), smem_bytes<kQuant>(), done);
  if (e != cudaSuccess) return cuda_status(e, "paged_chunk smem attribute");
  return cuda_status(launch_dependent(kernel, dim3(p.n_ctas), kThreads, smem_bytes<kQuant>(), st, k_map, v_map, p),
                     "paged_chunk launch");
}

}  // namespace

// One query per sequence, groups of at most 8 heads (the N of an MMA); blocks of 16, 32 or 64
// tokens or a multiple of 64 (a 64-key tile is whole blocks, or lies in one; 16 bytes of scales at
// least).  Wider groups run on the tcgen05 kernel, whose 128 rows they fill better.
bool decode_sinks_supported(const ChunkParams& p, int dtype, int pool_dtype) {
  if (p.cu_q != nullptr || (dtype != SNAPMIND_DTYPE_BF16 && dtype != SNAPMIND_DTYPE_F16)) return false;
  if (p.head_dim != kD || p.group > kHeads) return false;
  const int bs = p.block_size;
  if (bs != 16 && bs != 32 && bs % 64 != 0) return false;
  const auto a16 = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; };
  if (!a16(p.q) || !a16(p.out) || !a16(p.k_pool) || !a16(p.v_pool)) return false;
  if (p.q_stride_tok % 8 || p.q_stride_head % 8 || p.out_stride_tok % 8 || p.out_stride_head % 8) return false;
  if ((int64_t)p.num_blocks * p.n_kv_heads * bs >= (int64_t)1 << 31) return false;  // TMA row coordinate
  if (pool_dtype == SNAPMIND_DTYPE_E4M3 && !a16(p.scales)) return false;
  return encode_tiled() != nullptr;
}

int launch_decode_sinks(WeighedParams& p, int dtype, int pool_dtype, cudaStream_t st) {
  const int rc = plan_geometry(p, kHeads, kHeads, kTile, 2 * num_sms());
  if (rc != SNAPMIND_OK) return rc;
  p.tokens = 1;
  p.means = pool_dtype == SNAPMIND_DTYPE_E4M3;
  const bool quant = pool_dtype == SNAPMIND_DTYPE_E4M3;
  const auto go = [&](auto t) -> int {
    using T = decltype(t);
    if (p.stats != nullptr) return quant ? launch<T, true, true>(p, st) : launch<T, false, true>(p, st);
    return quant ? launch<T, true, false>(p, st) : launch<T, false, false>(p, st);
  };
  return dtype == SNAPMIND_DTYPE_BF16 ? go(__nv_bfloat16()) : go(__half());
}

}  // namespace snapmind
