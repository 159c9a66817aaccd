// Work plan of the paged attention over chunks of new tokens (chunk_attn*.cu,
// decode_sinks.cu).
//
// A unit is one (sequence b, kv head, slice of its query group, run of query tokens): at
// most `rows` query rows that read the same keys.  Row r of a unit is token
// i0 + r / gw, query head r % gw of the slice (gw = the slice's heads).  A unit's
// work is the number of key tiles some row of it sees, and the tiles of all units,
// in the order (b, kv head, slice, run), form one line that the CTAs cut into equal
// pieces: CTA c of n takes tiles [c W / n, (c + 1) W / n) of W (n is at most W).  So every CTA streams
// the same number of tiles whatever the lengths are, and long caches with few rows are
// split over many CTAs by the same rule.  A unit cut by a boundary leaves one
// partial softmax state per piece in the workspace, and a second kernel merges them.
// The plan needs nothing from the host: lengths may come from a captured step.
//
// Keys of a unit.  Query position p sees keys j <= p, under a window w only
// j > p - w or j < sinks.  The unit's keys are the sink blocks, then the blocks from
// the first one that its first query's window reaches: a virtual axis v with one jump,
// position(v) = v + (v >= v_sink ? shift : 0), so nothing between is read.
#pragma once

#include "common.cuh"

namespace snapmind {

struct ChunkParams {
  const void* q;
  int64_t q_stride_tok, q_stride_head;  // elements
  const void* k_pool;
  const void* v_pool;
  const uint8_t* scales;  // e4m3 pools: [block][head][2][slot] exponents + 127 (else NULL)
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* seq_lens;
  const int32_t* cu_q;  // [batch + 1] first query row of every sequence; NULL: one each
  void* out;
  int64_t out_stride_tok, out_stride_head;  // elements
  float scale;
  int32_t batch, total_q, n_q_heads, n_kv_heads, group, head_dim, block_size, num_blocks;
  int32_t window, sinks;   // window 0: none
  int32_t max_len;         // positions that a table row has room for
  int32_t gw, n_slices;    // query heads of a slice, slices of a group
  int32_t tokens;          // query tokens of a unit
  int32_t rows;            // partial rows of a unit in the workspace (>= gw * tokens)
  int32_t key_tile;        // keys of a tile
  int32_t n_ctas;
  FastDiv by_gw, by_block, by_tile, by_ctas;  // divisions by gw, block_size, key_tile, n_ctas
  void* workspace;
  int32_t* heads;   // workspace: [n_ctas][kPieceInts], see PieceInfo
  float* part_ml;   // workspace: [n_ctas][2][rows][2] maximum (log2 units), sum
  float* part_o;    // workspace: [n_ctas][2][rows][head_dim]
  int32_t* odd;     // workspace: [n_odd] whether a CTA met rows that its kernel's types do not hold, or NULL
  int32_t n_odd;
  int32_t means;    // part_o holds a piece's weighted means of V (else its weighted sums)
  int32_t* err;
};

constexpr int kPieceInts = 8;   // b, kv head, slice, first token, first and last piece's CTA, first query row, new tokens
constexpr int kMaxChunkBatch = 8192;

// New tokens of sequence b: its first query row and their number.
__device__ __forceinline__ int chunk_queries(const ChunkParams& p, int b, int* first) {
  if (p.cu_q == nullptr) {
    *first = b;
    return 1;
  }
  const int lo = min(max(p.cu_q[b], 0), p.total_q);
  *first = lo;
  return min(max(p.cu_q[b + 1], lo), p.total_q) - lo;
}

// The keys that the query tokens [i0, i1) of n new ones see in a cache of len tokens.
struct KeyRange {
  int pos0;    // position of token i0
  int end;     // positions >= end are seen by none (or have no entry in the table row)
  int win_lo;  // first position inside token i0's window
  int v_sink, shift, v_len;
  __device__ __forceinline__ int position(int v) const { return v + (v >= v_sink ? shift : 0); }
};
__device__ __forceinline__ KeyRange key_range(const ChunkParams& p, int len, int n, int i0, int i1) {
  KeyRange r;
  r.pos0 = len - n + i0;
  r.end = max(0, min(min(len, p.max_len), len - n + i1));
  r.win_lo = p.window > 0 ? max(0, r.pos0 - p.window + 1) : 0;
  const int bs = p.block_size;
  const int n_sink = p.window > 0 ? p.by_block.div(min(p.sinks, r.end) + bs - 1) : 0;
  const int wb0 = p.window > 0 ? p.by_block.div(min(r.win_lo, r.end)) : 0;
  r.v_sink = n_sink * bs;
  r.shift = max(0, wb0 - n_sink) * bs;
  r.v_len = r.end - r.shift;
  return r;
}
// Key tiles of a unit; at least one, so that rows that see nothing are written as zeros.
__device__ __forceinline__ int key_tiles(const ChunkParams& p, int len, int n, int i0) {
  const KeyRange r = key_range(p, len, n, i0, min(n, i0 + p.tokens));
  return max(1, p.by_tile.div(r.v_len + p.key_tile - 1));
}

// A piece: consecutive tiles of one unit.
struct Piece {
  int b, kvh, slice, i0;     // the unit
  int n, len, q_first;       // new tokens, cached tokens, first query row of sequence b
  int tile0, tile1, n_tiles; // tiles of the piece, tiles of the unit
  __device__ __forceinline__ bool whole() const { return tile0 == 0 && tile1 == n_tiles; }
};

struct PlanShared {
  int32_t warp_sum[32];
  long long total, t0, t1;
  int32_t n;            // CTAs with work: min(n_ctas, total)
  long long rem;        // tiles of the sequence of tile t0 that come before it
  int32_t b;            // that sequence
  int32_t u;            // tiles of one (kv head, slice) of that sequence
  Piece first;
};

__device__ __forceinline__ int clamp_len(const ChunkParams& p, int b) { return max(0, p.seq_lens[b]); }

// A length past the table row: its positions there are left out, and flagged (once, by CTA 0).
__device__ __forceinline__ void check_len(const ChunkParams& p, int len) {
  if (len > p.max_len && blockIdx.x == 0) flag_error(p.err, SNAPMIND_DEVERR_TABLE);
}

// Tiles of one (kv head, slice) of sequence b, summed by a full warp.
__device__ __forceinline__ int seq_tiles(const ChunkParams& p, int b, int lane) {
  int first;
  const int n = chunk_queries(p, b, &first);
  const int len = clamp_len(p, b);
  if (n > 0 && lane == 0) check_len(p, len);
  int s = 0;
  for (int i0 = lane * p.tokens; i0 < n; i0 += 32 * p.tokens) s += key_tiles(p, len, n, i0);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

// First tile of a CTA's share, cta total / n; n is n_ctas, or total when that is less.
__device__ __forceinline__ long long cut(const ChunkParams& p, int cta, long long total) {
  if (total <= p.n_ctas) return cta;
  const long long x = cta * total;
  return x < (1ll << 31) ? p.by_ctas.div((int)x) : x / p.n_ctas;
}
// The CTA whose share holds tile t: the largest c with cut(c) <= t, which is
// ((t + 1) n - 1) / total rounded down.
__device__ __forceinline__ int cta_of(long long t, long long total, int n) {
  const long long x = (t + 1) * n - 1;
  return (int)(x < (1ll << 32) && total < (1ll << 32) ? (long long)((uint32_t)x / (uint32_t)total) : x / total);
}

// The block's share of the line: fills S (total, t0, t1, first piece).  `tiles` is
// scratch for batch ints.  Every thread of the block calls it; ends with a barrier.
__device__ inline void plan_block(const ChunkParams& p, PlanShared& S, int32_t* tiles) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = blockDim.x >> 5;
  const int per_head = p.n_kv_heads * p.n_slices;
  if (p.cu_q == nullptr) {
    for (int b = tid; b < p.batch; b += blockDim.x) {
      const int len = clamp_len(p, b);
      check_len(p, len);
      tiles[b] = key_tiles(p, len, 1, 0);
    }
  } else {
    for (int b = warp; b < p.batch; b += nw) {
      const int s = seq_tiles(p, b, lane);
      if (lane == 0) tiles[b] = s;
    }
  }
  __syncthreads();
  // The tile line's length, and where this CTA's share begins.  Up to kWarpBatch sequences: every
  // warp goes over them, 32 a step (no barrier, the last step finds the place); more: one run of
  // sequences per thread and a scan over the block.
  constexpr int kWarpBatch = 256;
  long long t0, t1;
  if (p.batch <= kWarpBatch) {
    int sum = 0;
    for (int b = lane; b < p.batch; b += 32) sum += tiles[b];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const long long total = (long long)sum * per_head;
    const int n = (int)min((long long)p.n_ctas, total);
    const bool works = (int)blockIdx.x < n;
    t0 = works ? cut(p, blockIdx.x, total) : total;
    t1 = works ? cut(p, blockIdx.x + 1, total) : total;
    if (warp == 0) {
      long long before = 0;
      for (int base = 0; base < p.batch && t0 < t1; base += 32) {
        const int b = base + lane, u = b < p.batch ? tiles[b] : 0;
        int x = u;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, x, o);
          if (lane >= o) x += y;
        }
        const long long end = before + (long long)x * per_head, at = end - (long long)u * per_head;
        if (t0 >= at && t0 < end) {
          S.b = b;
          S.u = u;
          S.rem = t0 - at;
        }
        before += (long long)__shfl_sync(0xffffffffu, x, 31) * per_head;
        if (t0 < before) break;
      }
      if (lane == 0) {
        S.total = total;
        S.n = n;
        S.t0 = t0;
        S.t1 = t1;
      }
      __syncwarp();
    }
  } else {
    const int run = (p.batch + blockDim.x - 1) / blockDim.x;
    const int b0 = min(p.batch, tid * run), b1 = min(p.batch, b0 + run);
    int s = 0;
    for (int b = b0; b < b1; ++b) s += tiles[b];
    int incl = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    if (lane == 31) S.warp_sum[warp] = incl;
    __syncthreads();
    long long before = 0, total = 0;
    for (int w = 0; w < nw; ++w) {
      if (w < warp) before += S.warp_sum[w];
      total += S.warp_sum[w];
    }
    before = (before + incl - s) * per_head;
    total *= per_head;
    const int n = (int)min((long long)p.n_ctas, total);
    const bool works = (int)blockIdx.x < n;
    t0 = works ? cut(p, blockIdx.x, total) : total;
    t1 = works ? cut(p, blockIdx.x + 1, total) : total;
    if (tid == 0) {
      S.total = total;
      S.n = n;
      S.t0 = t0;
      S.t1 = t1;
    }
    if (t0 < t1 && t0 >= before && t0 < before + (long long)s * per_head) {
      long long at = before;
      int b = b0;
      while (t0 >= at + (long long)tiles[b] * per_head) at += (long long)tiles[b++] * per_head;
      S.b = b;
      S.u = tiles[b];
      S.rem = t0 - at;
    }
    __syncthreads();
  }
  if (warp == 0 && t0 < t1) {
    Piece f;
    f.b = S.b;
    int hs = (int)__fdividef((float)S.rem, (float)S.u);  // off by one at most: hs is small
    hs -= hs * (long long)S.u > S.rem;
    hs += (hs + 1) * (long long)S.u <= S.rem;
    int rem = (int)(S.rem - hs * (long long)S.u);
    f.kvh = hs / p.n_slices;
    f.slice = hs - f.kvh * p.n_slices;
    f.n = chunk_queries(p, f.b, &f.q_first);
    f.len = clamp_len(p, f.b);
    f.i0 = 0;
    f.n_tiles = S.u;
    f.tile0 = rem;
    // 32 runs at a time; ends inside the sequence since rem < u (one query per sequence: one run)
    for (int base = 0; p.cu_q != nullptr; base += 32) {
      const int i0 = (base + lane) * p.tokens;
      const int t = i0 < f.n ? key_tiles(p, f.len, f.n, i0) : 0;
      int x = t;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      const uint32_t m = __ballot_sync(0xffffffffu, x > rem);
      if (m != 0 || i0 - lane * p.tokens >= f.n) {
        const int l = m != 0 ? __ffs(m) - 1 : 0;
        f.i0 = __shfl_sync(0xffffffffu, i0, l);
        f.n_tiles = __shfl_sync(0xffffffffu, t, l);
        f.tile0 = rem - (__shfl_sync(0xffffffffu, x, l) - f.n_tiles);
        break;
      }
      rem -= __shfl_sync(0xffffffffu, x, 31);
    }
    f.tile1 = (int)min((long long)f.n_tiles, f.tile0 + (t1 - t0));
    if (lane == 0) S.first = f;
  }
  __syncthreads();
}

// Walks the pieces of a CTA: `left` tiles remain after the current piece.
struct PieceWalk {
  Piece c;
  long long left;
  __device__ __forceinline__ bool start(const PlanShared& S) {
    c = S.first;
    left = S.t1 - S.t0;
    if (left <= 0) return false;
    left -= c.tile1 - c.tile0;
    return true;
  }
  __device__ __forceinline__ bool next(const ChunkParams& p) {
    if (left <= 0) return false;
    c.i0 += p.tokens;
    if (c.i0 >= c.n) {
      c.i0 = 0;
      if (++c.slice == p.n_slices) {
        c.slice = 0;
        if (++c.kvh == p.n_kv_heads) {
          c.kvh = 0;
          do {
            if (++c.b >= p.batch) return false;
            c.n = chunk_queries(p, c.b, &c.q_first);
          } while (c.n == 0);
          c.len = clamp_len(p, c.b);
        }
      }
    }
    c.n_tiles = key_tiles(p, c.len, c.n, c.i0);
    c.tile0 = 0;
    c.tile1 = (int)min((long long)c.n_tiles, left);
    left -= c.tile1;
    return true;
  }
};

// Where the key tiles of a unit lie in the pool, 32 / parts tiles at a time: lane i holds part
// i % parts (a block, or the tile's piece of a larger block) of tile first + i / parts as its pool
// row (block * kv heads + kv head) * block_size + slot, -1 (no keys there), or `bad` where the table's entry
// is no block of the pool: such keys are seen by nobody.  The entries of the next batch are
// read while the current one is staged, so that no tile waits for the table.  (A read, a check and a
// division per tile made the staging warp the bound of 8-bit decodes: 306 us for what takes 200 us
// of copies.)
struct TileRows {
  const ChunkParams& p;
  const KeyRange& kr;
  const int32_t* table;
  int kvh, end, lane;
  int box, parts, log_parts;  // keys of a part, parts of a tile
  int bad;                    // row of a part whose entry is no block: -1, or the first row past the pool
  int first, rows;            // the current batch
  bool none;                  // it has an entry that is no block (`bad` >= 0)
  int32_t next;               // table entry of the batch after it

  __device__ __forceinline__ TileRows(const ChunkParams& p_, const KeyRange& kr_, const Piece& c, int lane_, int bad_ = -1)
      : p(p_), kr(kr_), table(p_.tables + (int64_t)c.b * p_.table_stride), kvh(c.kvh), end(c.tile1), lane(lane_), bad(bad_) {
    box = min(p.block_size, p.key_tile);
    parts = p.block_size >= p.key_tile ? 1 : p.by_block.div(p.key_tile);
    log_parts = 31 - __clz(parts);  // a power of two: blocks of 8 .. 64 keys
    first = c.tile0 - (32 >> log_parts);
    rows = -1;
    none = false;
    next = entry(c.tile0);
  }
  __device__ __forceinline__ int position(int first_tile) const {
    const int v = (first_tile + (lane >> log_parts)) * p.key_tile + (lane & (parts - 1)) * box;
    return v < kr.v_len ? kr.position(v) : -1;
  }
  // Table entry of the lane's part; kNoKey: no key there.
  static constexpr int32_t kNoKey = INT32_MIN;
  __device__ __forceinline__ int32_t entry(int first_tile) const {
    const int pos = position(first_tile);
    if (pos < 0 || first_tile + (lane >> log_parts) >= end) return kNoKey;
    return table[p.by_block.div(pos)];
  }
  // Makes `tile` part of the current batch (tiles are asked for in ascending order).
  __device__ __forceinline__ void advance(int tile) {
    if (tile < first + (32 >> log_parts)) return;
    first = tile;
    const int32_t e = next;
    rows = -1;
    if (e >= 0 && e < p.num_blocks) {
      const int pos = position(first);
      rows = (e * p.n_kv_heads + kvh) * p.block_size + (pos - p.by_block.div(pos) * p.block_size);
    } else if (e != kNoKey) {
      flag_error(p.err, SNAPMIND_DEVERR_BLOCK_ID);
      rows = bad;
    }
    if (bad >= 0) none = __any_sync(0xffffffffu, rows == bad);
    next = entry(first + (32 >> log_parts));
  }
  // Pool row of part x of a tile of the current batch (all lanes take part).
  __device__ __forceinline__ int row(int tile, int x) const {
    return __shfl_sync(0xffffffffu, rows, ((tile - first) << log_parts) + x);
  }
  // Parts of the tile that hold keys; those whose entry is no block (with a `bad` of 0 or more they
  // count among the first, too).
  __device__ __forceinline__ uint32_t have(int tile) const { return of_tile(rows >= 0, tile); }
  __device__ __forceinline__ uint32_t missing(int tile) const { return none ? of_tile(rows == bad, tile) : 0u; }
  __device__ __forceinline__ uint32_t of_tile(bool mine, int tile) const {
    return __ballot_sync(0xffffffffu, mine) >> ((tile - first) << log_parts) & ((1u << parts) - 1u);
  }
  // The byte of a pool row's K (0) or V (1) scale: [block][head][2][slot].
  __device__ __forceinline__ int64_t scale_at(int row, int kv) const {
    const int slot = row - p.by_block.div(row) * p.block_size;
    return 2 * (int64_t)row - slot + kv * p.block_size;
  }
};

// Query heads of a slice (the last one of a group may be narrower).
__device__ __forceinline__ int slice_heads(const ChunkParams& p, int slice) {
  return min(p.gw, p.group - slice * p.gw);
}

// Partial slot of a piece: 0 = the unit began in an earlier CTA, 1 = it begins here.
__device__ __forceinline__ int64_t part_slot(const Piece& c) { return (int64_t)blockIdx.x * 2 + (c.tile0 == 0 ? 1 : 0); }

// What the merge kernel reads about the unit that CTA c cuts at its start: written by one
// thread, b = -1 when the CTA starts on a unit's first tile or has no work.
__device__ inline void write_piece_info(const ChunkParams& p, const PlanShared& S) {
  int32_t* h = p.heads + (int64_t)blockIdx.x * kPieceInts;
  if (S.t0 >= S.t1 || S.first.tile0 == 0) {
    h[0] = -1;
    return;
  }
  const Piece& c = S.first;
  const long long s_u = S.t0 - c.tile0, e_u = s_u + c.n_tiles;
  h[1] = c.kvh;
  h[2] = c.slice;
  h[3] = c.i0;
  h[4] = cta_of(s_u, S.total, S.n);  // the CTA that holds tile s_u
  h[5] = cta_of(e_u - 1, S.total, S.n);        // ... and tile e_u - 1
  h[6] = c.q_first;
  h[7] = c.n;
  h[0] = c.b;
}

// 2^x by the hardware approximation (2 ulp); -inf -> 0.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Whether some CTA of the tcgen05 kernel before met such rows (then the CUDA-core kernel does the call
// over); every thread of the block calls it.
__device__ __forceinline__ bool any_odd(const ChunkParams& p) {
  int x = 0;
  for (int i = threadIdx.x; i < p.n_odd; i += blockDim.x) x |= p.odd[i];
  return __syncthreads_or(x) != 0;
}

// chunk_attn.cu: merges the cut units, after the attention kernel on the stream.
int launch_chunk_merge(const ChunkParams& p, int dtype, cudaStream_t st);

// chunk_attn_umma.cu (tcgen05) and decode_sinks.cu (one token per sequence): whether the
// shapes fit, the unit geometry and CTA count they want, and the launch.
bool chunk_umma_supported(const ChunkParams& p, int dtype, int pool_dtype);
int launch_chunk_umma(ChunkParams& p, int dtype, int pool_dtype, cudaStream_t st);
bool decode_sinks_supported(const ChunkParams& p, int dtype, int pool_dtype);
int launch_decode_sinks(ChunkParams& p, int dtype, int pool_dtype, cudaStream_t st);

// Sets a kernel's shared-memory attributes once per device (`done` is the instantiation's own).
constexpr int kMaxDevices = 64;
inline cudaError_t kernel_attributes(const void* kernel, size_t smem, bool (&done)[kMaxDevices]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < kMaxDevices && done[dev])) return e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e == cudaSuccess)  // room for two CTAs where two are meant to share an SM
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  if (e == cudaSuccess && dev < kMaxDevices) done[dev] = true;
  return e;
}

// The kernels of a call, and calls in a row, are programmatic dependents: a kernel's launch and its
// set-up overlap the tail of the one before, and it waits for that one to be complete and visible
// (prior_grid_wait) before it reads or writes anything in global memory.
__device__ __forceinline__ void prior_grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void next_grid_may_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
template <typename... P, typename... A>
inline cudaError_t launch_dependent(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, const A&... args) {
  cudaLaunchAttribute pdl[1];
  pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = pdl;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Workspace regions of n_ctas CTAs: heads, then maxima and sums, then partial outputs.
inline int64_t plan_workspace(ChunkParams& p, void* workspace, int64_t n_ctas, int64_t rows) {
  const int64_t ml_off = (n_ctas * kPieceInts * 4 + 255) / 256 * 256;
  const int64_t o_off = ml_off + (n_ctas * 2 * rows * 2 * 4 + 255) / 256 * 256;
  char* w = static_cast<char*>(workspace);
  p.heads = reinterpret_cast<int32_t*>(w);
  p.part_ml = reinterpret_cast<float*>(w + ml_off);
  p.part_o = reinterpret_cast<float*>(w + o_off);
  return (o_off + n_ctas * 2 * rows * p.head_dim * 4 + 255) / 256 * 256;
}

// Unit geometry for kernels of `rows` query rows in tiles of `tile_rows` (whole tokens each),
// `key_tile` keys and `n_ctas` CTAs.
inline int plan_geometry(ChunkParams& p, int rows, int tile_rows, int key_tile, int n_ctas) {
  p.gw = p.group < tile_rows ? p.group : tile_rows;
  p.n_slices = (p.group + p.gw - 1) / p.gw;
  p.tokens = rows / tile_rows * (tile_rows / p.gw);
  p.rows = rows;
  // the plan counts the tiles of one kv head in 32 bits
  const int64_t units = p.cu_q == nullptr ? p.batch : (int64_t)p.total_q / p.tokens + p.batch;
  SNAPMIND_CHECK_ARG(units * (p.max_len / key_tile + 2) < (int64_t)1 << 31,
                     "paged_chunk: %d new tokens over tables of %d positions are too many for one call", p.total_q, p.max_len);
  p.key_tile = key_tile;
  p.n_ctas = n_ctas;
  p.by_gw = FastDiv(p.gw);
  p.by_block = FastDiv(p.block_size);
  p.by_tile = FastDiv(key_tile);
  p.by_ctas = FastDiv(n_ctas);
  plan_workspace(p, p.workspace, n_ctas, rows);
  return SNAPMIND_OK;
}

}  // namespace snapmind
