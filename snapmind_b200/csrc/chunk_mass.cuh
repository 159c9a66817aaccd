// Work plan of the kernels that add the weights of a call's softmax to their keys (chunk_mass.cu,
// chunk_mass_umma.cu).
//
//   mass[key] += sum over the call's rows i that see it of 2^(score(i, key) + x_i)
//
// with x_i = -log2 of the row's sum, as the attention kernels left it (WeighedParams::stats).  A weight is
// known only when its row's whole softmax is, so it takes a second pass over the scores, but not over V.
//
// The roles of chunk_plan.cuh are turned round: a unit is one (sequence, kv head, tile of key_tile keys),
// which stays where it is while the rows that see some of it go by in steps: step s is run
// r0 + s / n_slices (p.tokens tokens) and slice s % n_slices of the query heads.  The steps of all units, in the
// order (b, kv head, tile), form a line that the CTAs cut into equal shares, so a key's sum is taken in
// one place (or in a few, left in the workspace and added in order): no atomics, the same result every time.
#pragma once

#include "chunk_plan.cuh"

namespace snapmind {

struct MassParams {
  WeighedParams c;    // gw, n_slices, tokens, rows, key_tile, n_ctas: this kernel's own
  FastDiv by_tokens;  // by c.tokens
  float* mass;        // [block][kv head][slot] of the layer
  int32_t* info;      // workspace: [n_ctas][kMassInts]
  float* part;        // workspace: [n_ctas][2][key_tile] sums of the pieces of cut units
};

constexpr int kMassInts = 8;  // b, kv head, tile, first and last piece's CTA, -, -, -

struct MassPiece {
  int b, kvh, tile;     // the unit
  int n, len, q_first;  // new tokens, cached tokens, first query row of sequence b
  int r0, steps;        // the unit's first run, its steps
  int s0, s1;           // the piece's steps
  __device__ __forceinline__ bool whole() const { return s0 == 0 && s1 == steps; }
};

struct MassShared {
  PlanShared line;
  MassPiece first;
};

// All keys that some of sequence b's n new tokens sees.
__device__ __forceinline__ KeyRange mass_range(const ChunkParams& p, int len, int n) { return key_range(p, len, n, 0, n); }
__device__ __forceinline__ int mass_tiles(const ChunkParams& p, const KeyRange& kr) { return p.by_tile.div(kr.v_len + p.key_tile - 1); }

// Runs [r0, r1) of tokens of which some see a key of the tile (none: r0 = r1 = 0).
__device__ __forceinline__ int2 mass_runs(const MassParams& mp, const KeyRange& kr, int n, int tile) {
  const ChunkParams& p = mp.c;
  const int v0 = tile * p.key_tile, v1 = min(v0 + p.key_tile, kr.v_len);
  if (v0 >= v1) return make_int2(0, 0);
  const int lo = kr.position(v0);
  const int i_lo = max(0, lo - kr.pos0);
  int i_hi = n;
  if (p.window > 0 && lo >= p.sinks)
    i_hi = (int)min((long long)n, (long long)kr.position(v1 - 1) + p.window - kr.pos0);
  if (i_lo >= i_hi) return make_int2(0, 0);
  return make_int2(mp.by_tokens.div(i_lo), mp.by_tokens.div(i_hi + p.tokens - 1));
}

// The block's share of the line.  `tiles` is scratch for batch ints.  Every thread of the block calls
// it; ends with a barrier.
__device__ inline void mass_plan(const MassParams& mp, MassShared& S, int32_t* tiles) {
  const ChunkParams& p = mp.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  for (int b = warp; b < p.batch; b += nw) {
    int first;
    const int n = chunk_queries(p, b, &first);
    int s = 0;
    if (n > 0) {
      const KeyRange kr = mass_range(p, clamp_len(p, b), n);
      const int nt = mass_tiles(p, kr);
      for (int t = lane; t < nt; t += 32) {
        const int2 r = mass_runs(mp, kr, n, t);
        s += r.y - r.x;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    }
    if (lane == 0) tiles[b] = s * p.n_slices;
  }
  __syncthreads();
  long long t0, t1;
  line_share(p, S.line, tiles, p.n_kv_heads, t0, t1);
  if (warp == 0 && t0 < t1) {
    MassPiece f;
    f.b = S.line.b;
    f.kvh = (int)(S.line.rem / S.line.u);
    int rem = (int)(S.line.rem - (long long)f.kvh * S.line.u);
    f.n = chunk_queries(p, f.b, &f.q_first);
    f.len = clamp_len(p, f.b);
    f.tile = f.r0 = f.steps = f.s0 = 0;
    const KeyRange kr = mass_range(p, f.len, f.n);
    const int nt = mass_tiles(p, kr);
    for (int base = 0; base < nt; base += 32) {  // 32 tiles at a time; ends inside since rem < u
      const int2 r = base + lane < nt ? mass_runs(mp, kr, f.n, base + lane) : make_int2(0, 0);
      const int t = (r.y - r.x) * p.n_slices;
      int x = t;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      const uint32_t m = __ballot_sync(0xffffffffu, x > rem);
      if (m != 0) {
        const int l = __ffs(m) - 1;
        f.tile = base + l;
        f.r0 = __shfl_sync(0xffffffffu, r.x, l);
        f.steps = __shfl_sync(0xffffffffu, t, l);
        f.s0 = rem - (__shfl_sync(0xffffffffu, x, l) - f.steps);
        break;
      }
      rem -= __shfl_sync(0xffffffffu, x, 31);
    }
    f.s1 = (int)min((long long)f.steps, f.s0 + (t1 - t0));
    if (lane == 0) S.first = f;
  }
  __syncthreads();
}

// Walks the pieces of a CTA; the key range and the tiles of the sequence come with the piece.
struct MassWalk {
  MassPiece c;
  KeyRange kr;
  int n_tiles;
  long long left;
  __device__ __forceinline__ void range(const ChunkParams& p) {
    kr = mass_range(p, c.len, c.n);
    n_tiles = mass_tiles(p, kr);
  }
  __device__ __forceinline__ bool start(const ChunkParams& p, const MassShared& S) {
    left = S.line.t1 - S.line.t0;
    if (left <= 0) return false;
    c = S.first;
    range(p);
    left -= c.s1 - c.s0;
    return c.s1 > c.s0;
  }
  // The next unit with a step (`left` of the line's steps remain, so there is one).
  __device__ __forceinline__ bool next(const MassParams& mp) {
    const ChunkParams& p = mp.c;
    if (left <= 0) return false;
    for (;;) {
      if (++c.tile >= n_tiles) {
        c.tile = 0;
        if (++c.kvh == p.n_kv_heads) {
          c.kvh = 0;
          do {
            if (++c.b >= p.batch) return false;
            c.n = chunk_queries(p, c.b, &c.q_first);
          } while (c.n == 0);
          c.len = clamp_len(p, c.b);
          range(p);
          if (n_tiles == 0) {  // no key: on to the next sequence
            c.kvh = p.n_kv_heads - 1;
            continue;
          }
        }
      }
      const int2 r = mass_runs(mp, kr, c.n, c.tile);
      if (r.y > r.x) {
        c.r0 = r.x;
        c.steps = (r.y - r.x) * p.n_slices;
        break;
      }
    }
    c.s0 = 0;
    c.s1 = (int)min((long long)c.steps, left);
    left -= c.s1;
    return true;
  }
};

__device__ __forceinline__ int64_t mass_slot(const MassPiece& c) { return (int64_t)blockIdx.x * 2 + (c.s0 == 0 ? 1 : 0); }

// What the merge kernel reads about the unit that CTA c cuts at its start: by one thread.
__device__ inline void write_mass_info(const MassParams& mp, const MassShared& S) {
  int32_t* h = mp.info + (int64_t)blockIdx.x * kMassInts;
  const PlanShared& L = S.line;
  if (L.t0 >= L.t1 || S.first.s0 == 0) {
    h[0] = -1;
    return;
  }
  const long long s_u = L.t0 - S.first.s0, e_u = s_u + S.first.steps;
  h[1] = S.first.kvh;
  h[2] = S.first.tile;
  h[3] = cta_of(s_u, L.total, L.n);
  h[4] = cta_of(e_u - 1, L.total, L.n);
  h[0] = S.first.b;
}

// Pool row ((block * kv heads + head) * block_size + slot) of key i of a unit's tile, -1: there is none.
__device__ __forceinline__ int64_t mass_row(const ChunkParams& p, const KeyRange& kr, int b, int kvh, int tile, int i, int* pos) {
  const int v = tile * p.key_tile + i;
  if (v >= kr.v_len) return -1;
  *pos = kr.position(v);
  const int j = p.by_block.div(*pos);
  const int32_t phys = p.tables[(int64_t)b * p.table_stride + j];
  if (phys < 0 || phys >= p.num_blocks) {
    flag_error(p.err, SNAPMIND_DEVERR_BLOCK_ID);
    return -1;
  }
  return ((int64_t)phys * p.n_kv_heads + kvh) * p.block_size + (*pos - j * p.block_size);
}

// x_i of row (token, head g of the kv head's group).
__device__ __forceinline__ const float* row_stats(const WeighedParams& p, int kvh, int64_t token, int g) {
  return p.stats + (kvh * (int64_t)p.total_q + token) * p.group + g;
}

// Whether a query at position q sees position pos.
__device__ __forceinline__ bool sees(const ChunkParams& p, int q, int pos) {
  return pos <= q && (p.window <= 0 || pos > q - p.window || pos < p.sinks);
}

// Geometry: steps of `rows` query rows, tiles of key_tile keys, n_ctas CTAs.
inline int mass_geometry(MassParams& mp, int rows, int key_tile, int n_ctas) {
  ChunkParams& p = mp.c;
  const int rc = plan_geometry(p, rows, rows, key_tile, n_ctas);
  if (rc != SNAPMIND_OK) return rc;
  SNAPMIND_CHECK_ARG(((int64_t)p.total_q / p.tokens + p.batch) * p.n_slices * (p.max_len / key_tile + 2) < (int64_t)1 << 31,
                     "paged_chunk: %d new tokens over tables of %d positions are too many for one call", p.total_q, p.max_len);
  mp.by_tokens = FastDiv(p.tokens);
  return SNAPMIND_OK;
}

// chunk_mass.cu: the merge of cut units, behind a kernel of this plan; the whole pass behind the attention kernels
// of a call, in a workspace of mass_workspace_bytes().
int launch_mass_merge(const MassParams& mp, cudaStream_t st);
int launch_mass(const WeighedParams& p, int dtype, int pool_dtype, int32_t flags, float* mass, void* workspace, cudaStream_t st);
int64_t mass_workspace_bytes();

// chunk_mass_umma.cu: for the shapes of chunk_umma_supported.
int launch_mass_umma(MassParams& mp, int dtype, int pool_dtype, cudaStream_t st);

}  // namespace snapmind
