// Attention of chunks of new tokens over a paged cache: entry point, the CUDA-core
// kernel (any head_dim up to 256, any block size, f32 / bf16 / f16 / e4m3 caches) and
// the merge of units that more than one CTA worked on.
//
//   o_i = sum_p softmax_p(scale q_i . k_p) v_p over the positions p that query i sees
//   (chunk_plan.cuh).
//
// The CUDA-core kernel: 64 query rows x 64 keys a step, thread (ty, tx) holding rows ty + 16 i and keys
// (then 4-dim pieces) tx + kTx j.  All arithmetic is f32, so it is the path of f32 caches.  What bounds
// it is shared memory and FMA issue together: with head_dim up to 64 a thread takes 4 x 8 products from
// 12 16-byte reads, three CTAs of 128 threads to an SM, which hide one another's loads: 4 prompts of 256
// tokens (32 heads over 4 of 64) take 55 us, 20 TFLOP/s of what is seen.  4 x 4 products from 8 reads, two CTAs of
// 256 threads and loads a step ahead took 60 us (63000 wavefronts of shared memory in 92000 cycles), loads
// element by element 92.  Larger rows need the threads: one CTA of 256, 4 x 4 products.
#include "chunk_plan.cuh"
#include "pairs.cuh"

namespace snapmind {
namespace {

constexpr int kRows = 64, kKeys = 64;
constexpr int kGenMaxD = 256;

// D4 = head_dim / 64 rounded up; smem rows are D = 64 * D4 floats (+4: 16-byte reads of
// 16 different rows then touch different banks), zero past head_dim.
template <int D4>
struct GenSmem {
  static constexpr int D = 64 * D4, P = D + 4;
  // threads that share a row, keys and 16-byte pieces of V of a thread; CTAs per SM
  static constexpr int kTx = D4 == 1 ? 8 : 16, kJ = kKeys / kTx, kX = D / (4 * kTx), kThreads = 16 * kTx;
  static constexpr int kCtas = D4 == 1 ? 3 : 1;
  static constexpr int PS = kKeys + (D4 == 1 ? 8 : 4);
  float q[kRows * P];
  float k[kKeys * P];
  float v[kKeys * P];
  float s[kRows * PS];
  int64_t row[2][kKeys];  // pool row of every key of a step, -1: seen by no row
  int32_t pos[2][kKeys];
  PlanShared plan;
};

// 16 bytes of pool elements as floats, stored to 16-byte-aligned shared memory; whether all are finite.
template <typename KV>
__device__ __forceinline__ bool spread(float* dst, const uint4& w, float scale) {
  constexpr int V = 16 / sizeof(KV);
  const KV* e = reinterpret_cast<const KV*>(&w);
  float f[V];
  bool finite = true;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if constexpr (std::is_same<KV, uint8_t>::value) f[i] = e4m3_to_f(e[i]) * scale;
    else f[i] = Conv<KV>::to_f(e[i]);
    finite &= fabsf(f[i]) < INFINITY;
  }
#pragma unroll
  for (int i = 0; i < V; i += 4) *reinterpret_cast<float4*>(dst + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
  return finite;
}

template <typename T>
__device__ __forceinline__ void store4(T* out, int d, int D, const float4& v, bool vec) {
  if (vec && d + 3 < D) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(out + d) = v;
    } else {
      __align__(8) T y[4] = {Conv<T>::from_f(v.x), Conv<T>::from_f(v.y), Conv<T>::from_f(v.z), Conv<T>::from_f(v.w)};
      *reinterpret_cast<uint2*>(out + d) = *reinterpret_cast<const uint2*>(y);
    }
    return;
  }
  const float y[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (d + u < D) out[d + u] = Conv<T>::from_f(y[u]);
}
// Whether 4 elements of an output row may be stored as one vector.
template <typename T>
__device__ __forceinline__ bool out_vec(const ChunkParams& p) {
  return p.out_stride_tok % 4 == 0 && p.out_stride_head % 4 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;
}

// p.odd: a second go at a call of the tcgen05 kernel, which only some CTA's odd rows make necessary.
template <typename T, typename KV, int D4>
__global__ void __launch_bounds__(GenSmem<D4>::kThreads, GenSmem<D4>::kCtas) chunk_generic_kernel(ChunkParams p) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  using Smem = GenSmem<D4>;
  constexpr int P = Smem::P, PS = Smem::PS, D = Smem::D, kTx = Smem::kTx, kJ = Smem::kJ, kX = Smem::kX;
  constexpr int kGenThreads = Smem::kThreads;
  constexpr bool kQuant = std::is_same<KV, uint8_t>::value;
  // whole 16-byte vectors of the pool: a row's, a thread's of K (and of V) a step
  constexpr int V = 16 / sizeof(KV), kRowVecs = D / V, kVecs = kKeys * kRowVecs / kGenThreads;
  constexpr bool kCanFetch = kVecs <= 8;                    // registers for a step of K and V
  constexpr bool kAhead = D4 > 1 && kCanFetch;              // ... while the step before is computed
  constexpr int kUnroll = D4 == 1 ? 2 : 4;                  // 4 spills with 168 registers
  constexpr int kHeld = kCanFetch ? kVecs : 1;
  Smem& S = *reinterpret_cast<Smem*>(smem_raw);
  const int tid = threadIdx.x, tx = tid % kTx, ty = tid / kTx;
  prior_grid_wait();
  if (p.odd != nullptr && !any_odd(p)) return;
  plan_block(p, S.plan, reinterpret_cast<int32_t*>(S.q));
  const float c2 = p.scale * kLog2e;
  const int bs = p.block_size, hd = p.head_dim;
  const bool fetches = kCanFetch && hd == D && ((reinterpret_cast<uintptr_t>(p.k_pool) | reinterpret_cast<uintptr_t>(p.v_pool)) & 15) == 0;
  const bool vec = out_vec<T>(p);
  constexpr int VQ = 16 / sizeof(T);
  const bool q_vec = hd == D && p.q_stride_tok % VQ == 0 && p.q_stride_head % VQ == 0 && (reinterpret_cast<uintptr_t>(p.q) & 15) == 0;

  PieceWalk w;
  for (bool on = w.start(S.plan); on; on = w.next(p)) {
    const Piece& c = w.c;
    const int heads = slice_heads(p, c.slice);
    const int i1 = min(c.n, c.i0 + p.tokens);
    const KeyRange kr = key_range(p, c.len, c.n, c.i0, i1);
    const int n_rows = (i1 - c.i0) * p.gw;
    const int head0 = c.kvh * p.group + c.slice * p.gw;
    // pool rows and positions of the keys of a step, by the first 64 threads
    const auto find = [&](int t) {
      if (tid >= kKeys) return;
      const int v = t * kKeys + tid;
      int64_t row = -1;
      int pos = INT32_MAX;
      if (t < c.tile1 && v < kr.v_len) {
        pos = kr.position(v);
        const int j = p.by_block.div(pos);
        const bool in_sink = p.window > 0 && pos < p.sinks;
        if (pos < kr.win_lo && !in_sink) {
          pos = INT32_MAX;  // in a block that is read, before every window
        } else {
          const int32_t phys = p.tables[(int64_t)c.b * p.table_stride + j];
          if (phys < 0 || phys >= p.num_blocks)
            flag_error(p.err, SNAPMIND_DEVERR_BLOCK_ID);
          else
            row = ((int64_t)phys * p.n_kv_heads + c.kvh) * bs + (pos - j * bs);
        }
      }
      S.row[t & 1][tid] = row;
      S.pos[t & 1][tid] = row < 0 ? INT32_MAX : pos;
    };
    // scales [block][head][2][slot]: K's byte of a pool row; V's is block_size further
    const auto scale_of = [&](int64_t row) {
      const int64_t tile = row / bs;
      return p.scales + tile * 2 * bs + (row - tile * bs);
    };
    uint4 held[2][kHeld];
    const auto fetch = [&](int t) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        const int e = tid + i * kGenThreads, r = e / kRowVecs, x = e % kRowVecs;
        const int64_t row = S.row[t & 1][r];
        held[0][i] = held[1][i] = make_uint4(0, 0, 0, 0);
        if (row >= 0) {
          held[0][i] = reinterpret_cast<const uint4*>(p.k_pool)[row * kRowVecs + x];
          held[1][i] = reinterpret_cast<const uint4*>(p.v_pool)[row * kRowVecs + x];
        }
      }
    };
    __syncthreads();
    find(c.tile0);
    if (q_vec) {
#pragma unroll
      for (int i = 0; i < kRows * D / VQ / kGenThreads; ++i) {
        const int e = tid + i * kGenThreads, r = e / (D / VQ), x = e % (D / VQ);
        const int tok = p.by_gw.div(r), g = r - tok * p.gw;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < n_rows && g < heads)
          v = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.q) + (int64_t)(c.q_first + c.i0 + tok) * p.q_stride_tok +
                                              (int64_t)(head0 + g) * p.q_stride_head + x * VQ);
        spread<T>(&S.q[r * P + x * VQ], v, 1.f);
      }
    } else for (int e = tid; e < kRows * D; e += kGenThreads) {
      const int r = e / D, d = e - r * D;
      const int tok = p.by_gw.div(r), g = r - tok * p.gw;
      float x = 0.f;
      if (r < n_rows && g < heads && d < hd)
        x = Conv<T>::to_f(reinterpret_cast<const T*>(p.q)[(int64_t)(c.q_first + c.i0 + tok) * p.q_stride_tok + (int64_t)(head0 + g) * p.q_stride_head + d]);
      S.q[r * P + d] = x;
    }
    __syncthreads();
    if (kAhead && fetches) fetch(c.tile0);
    float2 o[4][2 * kX];
    float m[4], l[4];
    int qpos[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.f;
      qpos[i] = kr.pos0 + p.by_gw.div(ty + 16 * i);
#pragma unroll
      for (int j = 0; j < 2 * kX; ++j) o[i][j] = make_float2(0.f, 0.f);
    }
    for (int t = c.tile0; t < c.tile1; ++t) {
      __syncthreads();  // the step before has been computed
      bool odd = false;  // a value of V that is not finite
      if (fetches) {
        if (!kAhead) fetch(t);
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
          const int e = tid + i * kGenThreads, r = e / kRowVecs, x = e % kRowVecs;
          float ks = 1.f, vs = 1.f;
          if constexpr (kQuant) {
            const int64_t row = S.row[t & 1][r];
            if (row >= 0) {
              const uint8_t* sc = scale_of(row);
              ks = scale_byte_to_f(sc[0]);
              vs = scale_byte_to_f(sc[bs]);
            }
          }
          spread<KV>(&S.k[r * P + x * V], held[0][i], ks);
          odd |= !spread<KV>(&S.v[r * P + x * V], held[1][i], vs);
        }
      } else {
        for (int e = tid; e < kKeys * D; e += kGenThreads) {
          const int r = e / D, d = e - r * D;
          const int64_t row = S.row[t & 1][r];
          float kx = 0.f, vx = 0.f;
          if (row >= 0 && d < hd) {
            if constexpr (kQuant) {
              const uint8_t* sc = scale_of(row);
              kx = e4m3_to_f(reinterpret_cast<const uint8_t*>(p.k_pool)[row * hd + d]) * scale_byte_to_f(sc[0]);
              vx = e4m3_to_f(reinterpret_cast<const uint8_t*>(p.v_pool)[row * hd + d]) * scale_byte_to_f(sc[bs]);
            } else {
              kx = Conv<KV>::to_f(reinterpret_cast<const KV*>(p.k_pool)[row * hd + d]);
              vx = Conv<KV>::to_f(reinterpret_cast<const KV*>(p.v_pool)[row * hd + d]);
            }
          }
          S.k[r * P + d] = kx;
          S.v[r * P + d] = vx;
          odd |= !(fabsf(vx) < INFINITY);
        }
      }
      find(t + 1);
      odd = __syncthreads_or(odd);
      if (kAhead && fetches && t + 1 < c.tile1) fetch(t + 1);  // lands while this step is computed
      float2 s2[4][kJ];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < kJ; ++j) s2[i][j] = make_float2(0.f, 0.f);
#pragma unroll kUnroll
      for (int d = 0; d < D; d += 4) {
        float4 a[4], b[kJ];
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = *reinterpret_cast<const float4*>(&S.q[(ty + 16 * i) * P + d]);
#pragma unroll
        for (int j = 0; j < kJ; ++j) b[j] = *reinterpret_cast<const float4*>(&S.k[(tx + kTx * j) * P + d]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < kJ; ++j) {
            s2[i][j] = fma2(make_float2(a[i].x, a[i].y), make_float2(b[j].x, b[j].y), s2[i][j]);
            s2[i][j] = fma2(make_float2(a[i].z, a[i].w), make_float2(b[j].z, b[j].w), s2[i][j]);
          }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float s[kJ];
        float mx = m[i];
#pragma unroll
        for (int j = 0; j < kJ; ++j) {
          const int pos = S.pos[t & 1][tx + kTx * j];
          const bool sees = pos <= qpos[i] && (p.window <= 0 || pos > qpos[i] - p.window || pos < p.sinks);
          s[j] = sees ? (s2[i][j].x + s2[i][j].y) * c2 : -INFINITY;
          mx = fmaxf(mx, s[j]);
        }
#pragma unroll
        for (int off = kTx / 2; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
        // nothing seen so far: any finite reference gives p = 2^-inf = 0
        const float ref = mx == -INFINITY ? 0.f : mx;
        const float alpha = ex2(m[i] - ref);
        m[i] = mx;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < kJ; ++j) {
          const float e = ex2(s[j] - ref);
          sum += e;
          S.s[(ty + 16 * i) * PS + tx + kTx * j] = e;
        }
        l[i] = l[i] * alpha + sum;  // this thread's share; summed over the row's threads at the end
#pragma unroll
        for (int j = 0; j < 2 * kX; ++j) {
          o[i][j].x *= alpha;
          o[i][j].y *= alpha;
        }
      }
      __syncwarp();  // a row's threads share a warp
      if (!odd) {
#pragma unroll 2
        for (int k = 0; k < kKeys; k += 4) {
          float a[4][4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<float4*>(a[i]) = *reinterpret_cast<const float4*>(&S.s[(ty + 16 * i) * PS + k]);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
#pragma unroll
            for (int j = 0; j < kX; ++j) {
              const float4 b = *reinterpret_cast<const float4*>(&S.v[(k + kk) * P + 4 * (kTx * j + tx)]);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float2 x = make_float2(a[i][kk], a[i][kk]);
                o[i][2 * j] = fma2(x, make_float2(b.x, b.y), o[i][2 * j]);
                o[i][2 * j + 1] = fma2(x, make_float2(b.z, b.w), o[i][2 * j + 1]);
              }
            }
        }
      } else {
        // infinities or NaN in V: they reach only the rows that see their token
        for (int k = 0; k < kKeys; ++k) {
          const int pos = S.pos[t & 1][k];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (!(pos <= qpos[i] && (p.window <= 0 || pos > qpos[i] - p.window || pos < p.sinks))) continue;
            const float a = S.s[(ty + 16 * i) * PS + k];
#pragma unroll
            for (int j = 0; j < 2 * kX; ++j) {
              const float* v = &S.v[k * P + 4 * (kTx * (j / 2) + tx) + 2 * (j % 2)];
              o[i][j].x = fmaf(a, v[0], o[i][j].x);
              o[i][j].y = fmaf(a, v[1], o[i][j].y);
            }
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int off = kTx / 2; off > 0; off >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], off);
      const int r = ty + 16 * i, tok = p.by_gw.div(r), g = r - tok * p.gw;
      if (r >= n_rows || g >= heads) continue;
      const bool whole = c.whole();
      const float f = !whole ? 1.f : l[i] == 0.f ? 0.f : 1.f / l[i];  // sees nothing: zeros (a NaN stays one)
      const int64_t slot = part_slot(c) * p.rows + r;
      T* out = reinterpret_cast<T*>(p.out) + (int64_t)(c.q_first + c.i0 + tok) * p.out_stride_tok + (int64_t)(head0 + g) * p.out_stride_head;
      if (!whole && tx == 0) {
        p.part_ml[slot * 2] = m[i];
        p.part_ml[slot * 2 + 1] = l[i];
      }
#pragma unroll
      for (int j = 0; j < kX; ++j) {
        const float4 y = make_float4(o[i][2 * j].x * f, o[i][2 * j].y * f, o[i][2 * j + 1].x * f, o[i][2 * j + 1].y * f);
        if (whole) store4(out, 4 * (kTx * j + tx), hd, y, vec);
        else store4(p.part_o + slot * hd, 4 * (kTx * j + tx), hd, y, hd % 4 == 0);
      }
    }
  }
  if (tid == 0) write_piece_info(p, S.plan);
}

// Merge of the cut units: block (c, y) works when CTA c holds the first cut inside a
// unit, on rows y, y + gridDim.y, ... (in groups of kMergeRows); pieces are CTA c - 1's slot 1, then
// slot 0 of CTAs c .. last.  M = max m_i, out = sum o_i 2^(m_i - M) / sum l_i 2^(m_i - M); pieces that left
// means (8-bit decodes: sums relative to M could pass f32's range) have l_i o_i for o_i.  A piece with
// m = -infinity saw nothing (l = 0, and o may hold anything) or only NaN (l is one, and so is out).
// The work is a few loads that wait for one another, so what counts is how many are in flight: a
// warp takes kMergeRows rows of a unit cut into up to 8 pieces at once (one row at a time, the 256-row
// units of a long chunk took 30 us), or one row of more pieces, 8 of them in flight (one at a
// time, the 17 pieces of a decode took 25 us).  A lane holds 4 dims (and 128 more).
constexpr int kMergeWarps = 4, kMergeBatch = 8, kMergeRows = 4;

__device__ __forceinline__ float4 load4(const float* o, int d, int D) {
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (D % 4 == 0) {
    if (d < D) v = *reinterpret_cast<const float4*>(o + d);
  } else {
    if (d < D) v.x = o[d];
    if (d + 1 < D) v.y = o[d + 1];
    if (d + 2 < D) v.z = o[d + 2];
    if (d + 3 < D) v.w = o[d + 3];
  }
  return v;
}
__device__ __forceinline__ void add4(float4& a, const float4& v, float f) {
  a.x = fmaf(v.x, f, a.x);
  a.y = fmaf(v.y, f, a.y);
  a.z = fmaf(v.z, f, a.z);
  a.w = fmaf(v.w, f, a.w);
}
__device__ __forceinline__ void mul4(float4& a, float f) {
  a.x *= f;
  a.y *= f;
  a.z *= f;
  a.w *= f;
}

template <typename T>
__device__ __forceinline__ void merge_units(const ChunkParams& p) {
  const int cta = blockIdx.x + 1;
  if (cta >= p.n_ctas) return;
  const int4 h0 = *reinterpret_cast<const int4*>(p.heads + (int64_t)cta * kPieceInts);
  const int4 h1 = *reinterpret_cast<const int4*>(p.heads + (int64_t)cta * kPieceInts + 4);
  if (h0.x < 0 || h1.x != cta - 1) return;
  const int kvh = h0.y, slice = h0.z, i0 = h0.w, n_pieces = h1.y - cta + 2, first = h1.z, n = h1.w;
  const int heads = slice_heads(p, slice), n_rows = (min(n, i0 + p.tokens) - i0) * p.gw;
  const int lane = threadIdx.x & 31, D = p.head_dim;
  const bool vec = out_vec<T>(p);
  const auto slot = [&](int i, int r) { return ((int64_t)(cta - 1 + i) * 2 + (i == 0 ? 1 : 0)) * p.rows + r; };
  const auto out_row = [&](int r, int g) {
    return reinterpret_cast<T*>(p.out) + (int64_t)(first + i0 + p.by_gw.div(r)) * p.out_stride_tok +
           (int64_t)(kvh * p.group + slice * p.gw + g) * p.out_stride_head;
  };
  const int warp = blockIdx.y * kMergeWarps + (threadIdx.x >> 5), warps = gridDim.y * kMergeWarps;

  if (n_pieces <= 8) {
    for (int r0 = warp * kMergeRows; r0 < n_rows; r0 += warps * kMergeRows) {
      // lane 8 x + i: piece i of row r0 + x
      const int rl = r0 + (lane >> 3), il = lane & 7;
      float2 ml = make_float2(-INFINITY, 0.f);
      if (rl < n_rows && il < n_pieces) ml = *reinterpret_cast<const float2*>(p.part_ml + slot(il, rl) * 2);
      float4 acc[kMergeRows][2] = {};
      float4 v[2][kMergeRows];  // the rows of two pieces at a time (each row's first 128 dims)
      const auto fetch = [&](int i, int c) {
#pragma unroll
        for (int x = 0; x < kMergeRows; ++x) {
          v[i & 1][x] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (i < n_pieces && r0 + x < n_rows) v[i & 1][x] = load4(p.part_o + slot(i, r0 + x) * D, 128 * c + 4 * lane, D);
        }
      };
      fetch(0, 0);
      fetch(1, 0);
      float M = ml.x;
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
      const float ref = M == -INFINITY ? 0.f : M;
      float f = ml.x == -INFINITY ? ml.y : ex2(ml.x - ref), L = ml.y * f;
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
      f *= L == 0.f ? 0.f : 1.f / L;  // a row that sees nothing: zeros
      if (p.means) f *= ml.y;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if (128 * c >= D) break;
        if (c > 0) {
          fetch(0, c);
          fetch(1, c);
        }
        for (int i = 0; i < n_pieces; i += 2) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int x = 0; x < kMergeRows; ++x) {
              const float fx = __shfl_sync(0xffffffffu, f, 8 * x + i + u);
              if (i + u < n_pieces && fx != 0.f) add4(acc[x][c], v[u][x], fx);  // weight 0: the piece may hold anything
            }
            if (i + u + 2 < n_pieces) fetch(i + u + 2, c);
          }
        }
      }
#pragma unroll
      for (int x = 0; x < kMergeRows; ++x) {
        const int r = r0 + x, g = r - p.by_gw.div(r) * p.gw;
        if (r >= n_rows || g >= heads) continue;
        T* out = out_row(r, g);
        store4(out, 4 * lane, D, acc[x][0], vec);
        if (D > 128) store4(out, 128 + 4 * lane, D, acc[x][1], vec);
      }
    }
    return;
  }
  for (int r = warp; r < n_rows; r += warps) {
    const int g = r - p.by_gw.div(r) * p.gw;
    if (g >= heads) continue;
    float M = -INFINITY, L = 0.f;
    float4 acc[2] = {};
    for (int k0 = 0; k0 < n_pieces; k0 += 32) {  // lane i holds the weight of piece k0 + i
      float2 ml = make_float2(-INFINITY, 0.f);
      if (k0 + lane < n_pieces) ml = *reinterpret_cast<const float2*>(p.part_ml + slot(k0 + lane, r) * 2);
      float mb = ml.x;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mb = fmaxf(mb, __shfl_xor_sync(0xffffffffu, mb, o));
      mb = fmaxf(mb, M);
      const float ref = mb == -INFINITY ? 0.f : mb, old = ex2(M - ref);
      M = mb;
      const float f = ml.x == -INFINITY ? ml.y : ex2(ml.x - ref);
      const float ls_mine = ml.y * f;
      float ls = ls_mine;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) ls += __shfl_xor_sync(0xffffffffu, ls, o);
      L = L * old + ls;
      mul4(acc[0], old);
      mul4(acc[1], old);
      const float fo = p.means ? ls_mine : f;
      const int here = min(32, n_pieces - k0);
      for (int k = 0; k < here; k += kMergeBatch) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (128 * c >= D) break;
          float4 v[kMergeBatch];
#pragma unroll
          for (int u = 0; u < kMergeBatch; ++u)
            v[u] = k + u < here ? load4(p.part_o + slot(k0 + k + u, r) * D, 128 * c + 4 * lane, D) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int u = 0; u < kMergeBatch; ++u) {
            const float fu = __shfl_sync(0xffffffffu, fo, (k + u) & 31);
            if (k + u < here && fu != 0.f) add4(acc[c], v[u], fu);
          }
        }
      }
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    mul4(acc[0], inv);
    mul4(acc[1], inv);
    T* out = out_row(r, g);
    store4(out, 4 * lane, D, acc[0], vec);
    if (D > 128) store4(out, 128 + 4 * lane, D, acc[1], vec);
  }
}

template <typename T>
__global__ void __launch_bounds__(32 * kMergeWarps) chunk_merge_kernel(ChunkParams p) {
  next_grid_may_launch();  // every block of this grid has started by then
  prior_grid_wait();
  merge_units<T>(p);
}
// After a call that may have been done over: `again` merges the units of that.
template <typename T>
__global__ void __launch_bounds__(32 * kMergeWarps)
    chunk_merge_either_kernel(const __grid_constant__ ChunkParams p, const __grid_constant__ ChunkParams again) {
  next_grid_may_launch();
  prior_grid_wait();
  if (any_odd(again)) merge_units<T>(again);
  else merge_units<T>(p);
}

dim3 merge_grid(const ChunkParams& p) {
  const int used = p.gw * p.tokens;
  return dim3(p.n_ctas - 1, (used + kMergeWarps * kMergeRows - 1) / (kMergeWarps * kMergeRows));
}

template <typename T, typename KV>
int launch_generic(const ChunkParams& p, cudaStream_t st) {
  const auto go = [&](auto kernel, int threads, size_t smem, bool (&done)[kMaxDevices]) -> int {
    const cudaError_t e = kernel_attributes(reinterpret_cast<const void*>(kernel), smem, done);
    if (e != cudaSuccess) return cuda_status(e, "paged_chunk smem attribute");
    return cuda_status(launch_dependent(kernel, dim3(p.n_ctas), threads, smem, st, p), "paged_chunk launch");
  };
  static bool done[3][kMaxDevices] = {};
  static_assert(sizeof(GenSmem<4>) <= 232448, "shared memory budget");
  static_assert(sizeof(GenSmem<1>().q) + sizeof(GenSmem<1>().k) >= kMaxChunkBatch * 4, "plan scratch");
  if (p.head_dim <= 64) return go(chunk_generic_kernel<T, KV, 1>, GenSmem<1>::kThreads, sizeof(GenSmem<1>), done[0]);
  if (p.head_dim <= 128) return go(chunk_generic_kernel<T, KV, 2>, GenSmem<2>::kThreads, sizeof(GenSmem<2>), done[1]);
  return go(chunk_generic_kernel<T, KV, 4>, GenSmem<4>::kThreads, sizeof(GenSmem<4>), done[2]);
}

int plan_generic(ChunkParams& p) {
  return plan_geometry(p, kRows, kRows, kKeys, num_sms() * (p.head_dim <= 64 ? GenSmem<1>::kCtas : 1));
}

// The tcgen05 kernel, then the CUDA-core kernel over the same call, which returns at once unless a
// CTA of the first met rows that f16 does not hold, then one merge for both.
int launch_f16_over_e4m3(ChunkParams& p, cudaStream_t st) {
  ChunkParams again = p;
  int rc = plan_generic(again);
  if (rc == SNAPMIND_OK) rc = launch_chunk_umma(p, SNAPMIND_DTYPE_F16, SNAPMIND_DTYPE_E4M3, st);
  if (rc != SNAPMIND_OK) return rc;
  again.n_odd = p.n_ctas;
  rc = launch_generic<__half, uint8_t>(again, st);
  if (rc != SNAPMIND_OK) return rc;
  const dim3 a = merge_grid(p), b = merge_grid(again);
  return cuda_status(launch_dependent(chunk_merge_either_kernel<__half>, dim3(a.x > b.x ? a.x : b.x, a.y > b.y ? a.y : b.y),
                                      32 * kMergeWarps, 0, st, p, again),
                     "paged_chunk merge");
}

// The largest workspace of the kernels: one CTA per SM with units of 256 rows, or three with 64.
int64_t max_ctas() { return num_sms(); }
constexpr int kMaxRows = 256;
static_assert(3 * kRows <= kMaxRows, "three CTAs per SM");
int64_t partials_bytes(int head_dim) {
  ChunkParams p = {};
  p.head_dim = head_dim;
  return plan_workspace(p, nullptr, 2 * max_ctas(), kMaxRows / 2);
}

}  // namespace

int launch_chunk_merge(const ChunkParams& p, int dtype, cudaStream_t st) {
  if (p.n_ctas < 2) return SNAPMIND_OK;
  const auto go = [&](auto kernel) {
    return cuda_status(launch_dependent(kernel, merge_grid(p), 32 * kMergeWarps, 0, st, p), "paged_chunk merge");
  };
  switch (dtype) {
    case SNAPMIND_DTYPE_F32: return go(chunk_merge_kernel<float>);
    case SNAPMIND_DTYPE_BF16: return go(chunk_merge_kernel<__nv_bfloat16>);
    default: return go(chunk_merge_kernel<__half>);
  }
}

}  // namespace snapmind

using namespace snapmind;

extern "C" {

int64_t snapmind_paged_gqa_chunk_workspace_bytes(int32_t head_dim) {
  if (head_dim <= 0 || head_dim > kGenMaxD) return 0;
  return partials_bytes(head_dim) + (max_ctas() * 4 + 255) / 256 * 256;
}

int snapmind_paged_gqa_chunk(const void* q, int64_t q_stride_tok, int64_t q_stride_head, int dtype, const void* k_pool,
                             const void* v_pool, const void* scales, int pool_dtype, const int32_t* block_tables,
                             int64_t table_stride_seq, int32_t table_width, const int32_t* seq_lens,
                             const int32_t* cu_q, void* out, int64_t out_stride_tok, int64_t out_stride_head,
                             float scale, int32_t batch, int32_t total_q, int32_t n_q_heads, int32_t n_kv_heads,
                             int32_t head_dim, int32_t block_size, int32_t num_blocks, int32_t window, int32_t sinks,
                             int32_t flags, void* workspace, int64_t workspace_bytes, int32_t* err_word, void* stream) {
  SNAPMIND_CHECK_ARG(dtype_size(dtype) > 0, "paged_chunk: unknown dtype");
  SNAPMIND_CHECK_ARG(pool_dtype == dtype || pool_dtype == SNAPMIND_DTYPE_E4M3,
                     "paged_chunk: the pool holds the query's dtype or e4m3");
  SNAPMIND_CHECK_ARG((pool_dtype == SNAPMIND_DTYPE_E4M3) == (scales != nullptr),
                     "paged_chunk: scales go with an e4m3 pool, and only with one");
  SNAPMIND_CHECK_ARG(batch >= 0 && batch <= kMaxChunkBatch && total_q >= 0 && n_q_heads > 0 && n_kv_heads > 0 &&
                         block_size > 0 && num_blocks > 0 && table_width >= 0,
                     "paged_chunk: bad sizes (batch at most %d)", kMaxChunkBatch);
  SNAPMIND_CHECK_ARG(n_q_heads % n_kv_heads == 0, "paged_chunk: n_q_heads (%d) must be a multiple of n_kv_heads (%d)",
                     n_q_heads, n_kv_heads);
  SNAPMIND_CHECK_ARG(head_dim > 0 && head_dim <= kGenMaxD, "paged_chunk: head_dim must be in [1, %d]", kGenMaxD);
  SNAPMIND_CHECK_ARG(window >= 0 && sinks >= 0, "paged_chunk: window and sinks must not be negative");
  SNAPMIND_CHECK_ARG(window > 0 || sinks == 0, "paged_chunk: sinks need a window");
  SNAPMIND_CHECK_ARG(cu_q != nullptr || total_q == batch, "paged_chunk: without cu_q there is one query per sequence");
  if (batch == 0 || total_q == 0) return SNAPMIND_OK;
  SNAPMIND_CHECK_ARG(q && k_pool && v_pool && block_tables && seq_lens && out, "paged_chunk: null pointer");
  ChunkParams p = {};
  // the stride of an axis of one is never used: give it the dense value, whatever the caller's is
  if (total_q == 1) q_stride_tok = out_stride_tok = (int64_t)n_q_heads * head_dim;
  if (n_q_heads == 1) q_stride_head = out_stride_head = head_dim;
  p.q = q;
  p.q_stride_tok = q_stride_tok;
  p.q_stride_head = q_stride_head;
  p.k_pool = k_pool;
  p.v_pool = v_pool;
  p.scales = static_cast<const uint8_t*>(scales);
  p.tables = block_tables;
  p.table_stride = table_stride_seq;
  p.seq_lens = seq_lens;
  p.cu_q = cu_q;
  p.out = out;
  p.out_stride_tok = out_stride_tok;
  p.out_stride_head = out_stride_head;
  p.scale = scale;
  p.batch = batch;
  p.total_q = total_q;
  p.n_q_heads = n_q_heads;
  p.n_kv_heads = n_kv_heads;
  p.group = n_q_heads / n_kv_heads;
  p.head_dim = head_dim;
  p.block_size = block_size;
  p.num_blocks = num_blocks;
  p.window = window < (1 << 30) ? window : (1 << 30);  // positions stay below 2^30
  p.sinks = sinks < (1 << 30) ? sinks : (1 << 30);
  const int64_t room = (int64_t)table_width * block_size;
  p.max_len = room < (1 << 30) ? (int32_t)room : (1 << 30);
  p.err = err_word;
  const int64_t need = snapmind_paged_gqa_chunk_workspace_bytes(head_dim);
  SNAPMIND_CHECK_ARG(workspace != nullptr && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0,
                     "paged_chunk: workspace needs %lld bytes on a 256-byte boundary, got %lld", (long long)need,
                     (long long)workspace_bytes);
  p.workspace = workspace;
  p.odd = nullptr;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool quant = pool_dtype == SNAPMIND_DTYPE_E4M3;
  if (!(flags & SNAPMIND_DECODE_FORCE_GENERIC) && decode_sinks_supported(p, dtype, pool_dtype)) {
    const int rc = launch_decode_sinks(p, dtype, pool_dtype, st);
    return rc != SNAPMIND_OK ? rc : launch_chunk_merge(p, dtype, st);
  }
  if (!(flags & SNAPMIND_DECODE_FORCE_GENERIC) && chunk_umma_supported(p, dtype, pool_dtype)) {
    if (quant && dtype == SNAPMIND_DTYPE_F16) {
      p.odd = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + partials_bytes(head_dim));
      const int rc = launch_f16_over_e4m3(p, st);
      if (rc != SNAPMIND_ERR_UNSUPPORTED) return rc;
      p.odd = nullptr;
    }
    const int rc = launch_chunk_umma(p, dtype, pool_dtype, st);
    if (rc != SNAPMIND_ERR_UNSUPPORTED) return rc != SNAPMIND_OK ? rc : launch_chunk_merge(p, dtype, st);
  }
  int rc = plan_generic(p);
  if (rc != SNAPMIND_OK) return rc;
  switch (dtype) {
    case SNAPMIND_DTYPE_F32: rc = quant ? launch_generic<float, uint8_t>(p, st) : launch_generic<float, float>(p, st); break;
    case SNAPMIND_DTYPE_BF16:
      rc = quant ? launch_generic<__nv_bfloat16, uint8_t>(p, st) : launch_generic<__nv_bfloat16, __nv_bfloat16>(p, st);
      break;
    default: rc = quant ? launch_generic<__half, uint8_t>(p, st) : launch_generic<__half, __half>(p, st); break;
  }
  return rc != SNAPMIND_OK ? rc : launch_chunk_merge(p, dtype, st);
}

}  // extern "C"
