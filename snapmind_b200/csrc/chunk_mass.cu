// Attention that adds the weights of its softmax to the cached tokens that they went to: entry point, the
// CUDA-core pass over the scores (any head_dim up to 256, any block size and type) and the merge of cut units.
//
// The CUDA-core pass: 64 query rows x 64 keys a step, thread (ty, tx) holding rows ty + 16 i and keys tx + 16 j,
// all in f32; the keys stay in shared memory while the rows go by.  FMA and shared-memory issue bound it: 4 prompts
// of 256 f32 tokens (32 heads over 4 of 64) take 56 us of attention and 40 for the weights.
#include "chunk_mass.cuh"
#include "pairs.cuh"

namespace snapmind {
namespace {

constexpr int kRows = 64, kKeys = 64, kThreads = 256;
constexpr int kGenMaxD = 256;

template <int D4>
struct MassSmem {
  static constexpr int D = 64 * D4, P = D + 4;  // +4: 16-byte reads of 16 different rows touch different banks
  static constexpr int kCtas = D4 == 1 ? 4 : D4 == 2 ? 2 : 1;
  float q[kRows * P];
  float k[kKeys * P];
  float x[kRows];
  int32_t qpos[kRows];
  int64_t row[kKeys];
  int32_t pos[kKeys];
  float sum[16][kKeys];
  MassShared plan;
};
static_assert(sizeof(MassSmem<1>) * 4 + 4 * 1024 <= 233472 && sizeof(MassSmem<2>) * 2 + 2 * 1024 <= 233472, "CTAs per SM");
static_assert(sizeof(MassSmem<4>) <= 232448, "shared memory budget");
static_assert(sizeof(MassSmem<1>().q) + sizeof(MassSmem<1>().k) >= kMaxChunkBatch * 4, "plan scratch");

// Rows into shared memory as f32, zero past head_dim: row r of 64 from src(r) (NULL: zeros) times scale(r).
template <typename T, int D4, typename Src, typename Scale>
__device__ __forceinline__ void load_rows(float* dst, int hd, bool vec, const Src& src, const Scale& scale) {
  using Smem = MassSmem<D4>;
  constexpr int V = 16 / sizeof(T), kVecs = Smem::D / V;
  const auto value = [](T x) {
    if constexpr (std::is_same<T, uint8_t>::value) return e4m3_to_f(x);
    else return Conv<T>::to_f(x);
  };
  if (vec) {  // head_dim a whole number of vectors
    for (int e = threadIdx.x; e < 64 * kVecs; e += kThreads) {
      const int r = e / kVecs, x = e % kVecs;
      const T* from = src(r);
      uint4 w = make_uint4(0, 0, 0, 0);
      const bool there = from != nullptr && x * V < hd;
      if (there) w = *reinterpret_cast<const uint4*>(from + x * V);
      const float f = there ? scale(r) : 0.f;
      const T* y = reinterpret_cast<const T*>(&w);
#pragma unroll
      for (int i = 0; i < V; i += 4)
        *reinterpret_cast<float4*>(dst + r * Smem::P + x * V + i) =
            make_float4(value(y[i]) * f, value(y[i + 1]) * f, value(y[i + 2]) * f, value(y[i + 3]) * f);
    }
  } else {
    for (int e = threadIdx.x; e < 64 * Smem::D; e += kThreads) {
      const int r = e / Smem::D, d = e % Smem::D;
      const T* from = src(r);
      dst[r * Smem::P + d] = from != nullptr && d < hd ? value(from[d]) * scale(r) : 0.f;
    }
  }
}

template <typename T, typename KV, int D4>
__global__ void __launch_bounds__(kThreads, MassSmem<D4>::kCtas) mass_generic_kernel(const __grid_constant__ MassParams mp) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  using Smem = MassSmem<D4>;
  constexpr int P = Smem::P, D = Smem::D;
  constexpr bool kQuant = std::is_same<KV, uint8_t>::value;
  const WeighedParams& p = mp.c;
  Smem& S = *reinterpret_cast<Smem*>(smem_raw);
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  next_grid_may_launch();
  prior_grid_wait();
  mass_plan(mp, S.plan, reinterpret_cast<int32_t*>(S.q));
  const float c2 = p.scale * kLog2e;
  const int hd = p.head_dim, bs = p.block_size;
  const auto aligned = [&](const void* x, int64_t bytes) { return ((reinterpret_cast<uintptr_t>(x) | (uintptr_t)bytes) & 15) == 0; };
  const bool q_vec = aligned(p.q, (hd | p.q_stride_tok | p.q_stride_head) * (int64_t)sizeof(T));
  const bool k_vec = aligned(p.k_pool, hd * (int64_t)sizeof(KV));
  MassWalk w;
  for (bool on = w.start(p, S.plan); on; on = w.next(mp)) {
    const MassPiece& c = w.c;
    __syncthreads();
    if (tid < kKeys) {
      int pos = INT32_MAX;
      S.row[tid] = mass_row(p, w.kr, c.b, c.kvh, c.tile, tid, &pos);
      S.pos[tid] = S.row[tid] < 0 ? INT32_MAX : pos;
    }
    __syncthreads();
    load_rows<KV, D4>(S.k, hd, k_vec,
                      [&](int r) { return S.row[r] < 0 ? nullptr : reinterpret_cast<const KV*>(p.k_pool) + S.row[r] * hd; },
                      [&](int r) {
                        if constexpr (kQuant) {
                          const int64_t block = S.row[r] / bs;
                          return scale_byte_to_f(p.scales[block * 2 * bs + (S.row[r] - block * bs)]);
                        } else {
                          return 1.f;
                        }
                      });
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = c.s0; s < c.s1; ++s) {
      const int run = s / p.n_slices, slice = s - run * p.n_slices;
      const int i0 = (c.r0 + run) * p.tokens, heads = slice_heads(p, slice), head0 = c.kvh * p.group + slice * p.gw;
      __syncthreads();  // the step before has been computed
      const auto query = [&](int r, int* tok, int* g) {  // whether row r of the step is a query
        const int t = p.by_gw.div(r);
        *tok = i0 + t;
        *g = r - t * p.gw;
        return t < p.tokens && *tok < c.n && *g < heads;
      };
      if (tid < kRows) {
        int tok, g;
        const bool there = query(tid, &tok, &g);
        S.x[tid] = there ? *row_stats(p, c.kvh, c.q_first + tok, slice * p.gw + g) : -INFINITY;
        S.qpos[tid] = there ? w.kr.pos0 + tok : INT32_MIN / 2;
      }
      load_rows<T, D4>(S.q, hd, q_vec,
                       [&](int r) -> const T* {
                         int tok, g;
                         if (!query(r, &tok, &g)) return nullptr;
                         return reinterpret_cast<const T*>(p.q) + (int64_t)(c.q_first + tok) * p.q_stride_tok + (int64_t)(head0 + g) * p.q_stride_head;
                       },
                       [](int) { return 1.f; });
      __syncthreads();
      float2 s2[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s2[i][j] = make_float2(0.f, 0.f);
#pragma unroll 4
      for (int d = 0; d < D; d += 4) {
        float4 a[4], b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = *reinterpret_cast<const float4*>(&S.q[(ty + 16 * i) * P + d]);
#pragma unroll
        for (int j = 0; j < 4; ++j) b[j] = *reinterpret_cast<const float4*>(&S.k[(tx + 16 * j) * P + d]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            s2[i][j] = fma2(make_float2(a[i].x, a[i].y), make_float2(b[j].x, b[j].y), s2[i][j]);
            s2[i][j] = fma2(make_float2(a[i].z, a[i].w), make_float2(b[j].z, b[j].w), s2[i][j]);
          }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = S.x[ty + 16 * i];
        const int q = S.qpos[ty + 16 * i];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float weight = ex2(fmaf(s2[i][j].x + s2[i][j].y, c2, x));
          if (sees(p, q, S.pos[tx + 16 * j])) acc[j] += weight;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) S.sum[ty][tx + 16 * j] = acc[j];
    __syncthreads();
    if (tid < kKeys) {
      float sum = 0.f;
#pragma unroll
      for (int y = 0; y < 16; ++y) sum += S.sum[y][tid];
      if (!c.whole()) mp.part[mass_slot(c) * kKeys + tid] = sum;
      else if (S.row[tid] >= 0) mp.mass[S.row[tid]] += sum;
    }
  }
  if (tid == 0) write_mass_info(mp, S.plan);
}

// Adds up the pieces of the units that CTAs cut: block c works when CTA c + 1 holds the first cut inside one.
__global__ void mass_merge_kernel(const __grid_constant__ MassParams mp) {
  next_grid_may_launch();
  prior_grid_wait();
  const ChunkParams& p = mp.c;
  const int cta = blockIdx.x + 1, i = threadIdx.x;
  const int32_t* h = mp.info + (int64_t)cta * kMassInts;
  if (cta >= p.n_ctas || h[0] < 0 || h[3] != cta - 1) return;
  const int b = h[0], last = h[4];
  int first;
  const int n = chunk_queries(p, b, &first);
  const KeyRange kr = mass_range(p, clamp_len(p, b), n);
  int pos;
  const int64_t row = mass_row(p, kr, b, h[1], h[2], i, &pos);
  if (row < 0) return;
  float sum = mp.part[((int64_t)(cta - 1) * 2 + 1) * p.key_tile + i];
  for (int k = cta; k <= last; ++k) sum += mp.part[(int64_t)k * 2 * p.key_tile + i];
  mp.mass[row] += sum;
}

template <typename T, typename KV>
int launch_generic(MassParams& mp, cudaStream_t st) {
  const auto go = [&](auto kernel, size_t smem, int ctas, bool (&done)[kMaxDevices]) -> int {
    int rc = mass_geometry(mp, kRows, kKeys, num_sms() * ctas);
    if (rc != SNAPMIND_OK) return rc;
    const cudaError_t e = kernel_attributes(reinterpret_cast<const void*>(kernel), smem, done);
    if (e != cudaSuccess) return cuda_status(e, "paged_chunk mass smem attribute");
    rc = cuda_status(launch_dependent(kernel, dim3(mp.c.n_ctas), kThreads, smem, st, mp), "paged_chunk mass launch");
    return rc != SNAPMIND_OK ? rc : launch_mass_merge(mp, st);
  };
  static bool done[3][kMaxDevices] = {};
  if (mp.c.head_dim <= 64) return go(mass_generic_kernel<T, KV, 1>, sizeof(MassSmem<1>), MassSmem<1>::kCtas, done[0]);
  if (mp.c.head_dim <= 128) return go(mass_generic_kernel<T, KV, 2>, sizeof(MassSmem<2>), MassSmem<2>::kCtas, done[1]);
  return go(mass_generic_kernel<T, KV, 4>, sizeof(MassSmem<4>), MassSmem<4>::kCtas, done[2]);
}

// Behind a decode that left its scores (decode_sinks.cu): the same CTAs on the same shares of the key line, four keys of
// a block a thread.  HBM bound: 4 bytes a query head and 8 of mass for each key and kv head, against the 512 of a
// 16-bit row of K and V that the decode read (scores taken from K anew would read half of those again).  A thread a key
// took 31 us beside the 440 of a decode of 128 sequences of 1 to 8 thousand tokens (32 heads over 8 of 128), this 25.  Tried and
// dropped: the merge of the output beside this kernel instead of before it, every warp putting a cut unit's sums
// together for itself (one sequence of 32768: 48 us, 43 without).
constexpr int kScoreThreads = 512;
template <int G>
__global__ void __launch_bounds__(kScoreThreads, 2) mass_scores_kernel(const __grid_constant__ WeighedParams p, float* mass) {
  extern __shared__ int32_t tiles[];
  __shared__ PlanShared plan;
  next_grid_may_launch();
  // the lengths are older than the call's first kernel, which has begun: only what it left is waited for
  plan_block(p, plan, tiles);
  prior_grid_wait();
  PieceWalk w;
  for (bool on = w.start(plan); on; on = w.next(p)) {
    const Piece& c = w.c;
    const KeyRange kr = key_range(p, c.len, c.n, c.i0, c.i0 + 1);
    const int group = G > 0 ? G : p.group;
    const float* stats = row_stats(p, c.kvh, c.q_first, 0);
    float st[G > 0 ? G : 1];
    if constexpr (G > 0) {
#pragma unroll
      for (int g = 0; g < G; ++g) st[g] = stats[g];
    }
    const int32_t* table = p.tables + (int64_t)c.b * p.table_stride;
    const int v1 = min(c.tile1 * p.key_tile, kr.v_len), q = kr.pos0;
    for (int v = c.tile0 * p.key_tile + 4 * threadIdx.x; v < v1; v += 4 * kScoreThreads) {
      const int pos = kr.position(v), j = p.by_block.div(pos);  // blocks are a multiple of 16 tokens: four in one
      const int32_t phys = table[j];
      if (phys < 0 || phys >= p.num_blocks) continue;
      const int64_t row = ((int64_t)phys * p.n_kv_heads + c.kvh) * p.block_size + (pos - j * p.block_size);
      float4* at = reinterpret_cast<float4*>(mass + row);
      const float* from = p.scores + (p.scores_room > 0 ? (int64_t)(c.b * p.n_kv_heads + c.kvh) * p.scores_room + v : row) * group;
      float4 m = *at;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
      if constexpr (G > 0) {
        float s[4 * G];
#pragma unroll
        for (int i = 0; i < G; ++i) *reinterpret_cast<float4*>(&s[4 * i]) = reinterpret_cast<const float4*>(from)[i];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int g = 0; g < G; ++g) sum[i] += ex2(s[i * G + g] + st[g]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          for (int g = 0; g < group; ++g) sum[i] += ex2(from[i * group + g] + stats[g]);
      }
      m = make_float4(m.x + sum[0], m.y + sum[1], m.z + sum[2], m.w + sum[3]);
      if (v + 4 <= v1 && (p.window <= 0 || pos > q - p.window || pos + 3 < p.sinks)) {
        *at = m;
        continue;
      }
      const float y[4] = {m.x, m.y, m.z, m.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (v + i < v1 && sees(p, q, pos + i)) mass[row + i] = y[i];
    }
  }
}

int launch_scores(const WeighedParams& p, float* mass, cudaStream_t st) {
  const auto go = [&](auto kernel) {
    return cuda_status(launch_dependent(kernel, dim3(p.n_ctas), kScoreThreads, (size_t)p.batch * 4, st, p, mass), "paged_chunk mass launch");
  };
  switch (p.group) {
    case 1: return go(mass_scores_kernel<1>);
    case 2: return go(mass_scores_kernel<2>);
    case 4: return go(mass_scores_kernel<4>);
    case 8: return go(mass_scores_kernel<8>);
    default: return go(mass_scores_kernel<0>);
  }
}

// Workspace: the attention's, then the rows' statistics, the cut units' pieces.
constexpr int64_t up256(int64_t x) { return (x + 255) / 256 * 256; }
int64_t max_ctas() { return 4 * (int64_t)num_sms(); }
int64_t info_bytes() { return up256(max_ctas() * kMassInts * 4); }
int64_t part_bytes() { return up256(max_ctas() * 2 * 128 * 4); }

}  // namespace

int launch_mass_merge(const MassParams& mp, cudaStream_t st) {
  if (mp.c.n_ctas < 2) return SNAPMIND_OK;
  return cuda_status(launch_dependent(mass_merge_kernel, dim3(mp.c.n_ctas - 1), mp.c.key_tile, 0, st, mp), "paged_chunk mass merge");
}

// After the attention kernels on the stream, which left p.stats.
int launch_mass(const WeighedParams& p, int dtype, int pool_dtype, int32_t flags, float* mass, void* workspace, cudaStream_t st) {
  if (p.scores != nullptr) return launch_scores(p, mass, st);
  MassParams mp = {};
  mp.c = p;
  mp.mass = mass;
  mp.info = static_cast<int32_t*>(workspace);
  mp.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + info_bytes());
  const bool quant = pool_dtype == SNAPMIND_DTYPE_E4M3;
  if (!(flags & SNAPMIND_DECODE_FORCE_GENERIC) && chunk_umma_supported(p, dtype, pool_dtype)) {
    const int rc = launch_mass_umma(mp, dtype, pool_dtype, st);
    if (rc != SNAPMIND_ERR_UNSUPPORTED) return rc;
  }
  switch (dtype) {
    case SNAPMIND_DTYPE_F32: return quant ? launch_generic<float, uint8_t>(mp, st) : launch_generic<float, float>(mp, st);
    case SNAPMIND_DTYPE_BF16:
      return quant ? launch_generic<__nv_bfloat16, uint8_t>(mp, st) : launch_generic<__nv_bfloat16, __nv_bfloat16>(mp, st);
    default: return quant ? launch_generic<__half, uint8_t>(mp, st) : launch_generic<__half, __half>(mp, st);
  }
}
int64_t mass_workspace_bytes() { return info_bytes() + part_bytes(); }

}  // namespace snapmind
