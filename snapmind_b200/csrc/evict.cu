// Eviction from a paged cache by accumulated attention weight: per (layer, sequence, kv head) the first
// `sinks` tokens, the newest `recent` and, of the others, those with the most weight stay (equal ones: the lowest
// index), up to `budget`, and move to the front in their order.
//
//   select  the kept indexes of every (layer, sequence, head), and their weights to their new places;
//   move    the kept rows of K and V (and 8-bit scales);
//   tables  lengths, table rows and the free stack (before the others when the rows go to other sequences).
//
// In place is safe because the i-th kept token stands at index p_i >= i: rows move towards the front in
// ascending order, a batch is read whole before it is written, and what a batch overwrites lies in front of all
// that is still to be read.
#include <type_traits>

#include "common.cuh"

namespace snapmind {
namespace {

struct EvictParams {
  int32_t* tables;
  int64_t table_stride;
  int32_t table_width;
  int32_t* seq_lens;
  const int32_t* src;  // [n] sequence ids, NULL: 0 .. n - 1
  const int32_t* dst;  // [n], NULL: in place
  int32_t n, n_layers, n_heads, block_size, num_blocks, budget, recent, sinks;
  FastDiv by_block;
  float* mass;
  int64_t mass_layer;  // elements
  int32_t* kept;       // [n_layers][n][n_heads][budget]
  uint8_t* pool[2];
  int64_t pool_layer;  // bytes
  uint8_t* scales;
  int64_t scale_layer;  // bytes
  int32_t row_bytes;
  int32_t slices, slice_bytes;  // a row's bytes are moved by `slices` blocks
  int32_t* free_stack;
  int32_t* free_top;
  int32_t* err;
};

__device__ __forceinline__ int src_id(const EvictParams& p, int i) { return p.src ? p.src[i] : i; }
__device__ __forceinline__ int dst_id(const EvictParams& p, int i) { return p.dst ? p.dst[i] : src_id(p, i); }
__device__ __forceinline__ int cached(const EvictParams& p, int seq) {
  const int64_t room = (int64_t)p.table_width * p.block_size;
  return (int)min((int64_t)max(0, p.seq_lens[seq]), room);
}
// Pool row of index j of the sequence whose table row is `table`, -1 (flagged): its entry is no block.
__device__ __forceinline__ int64_t row_of(const EvictParams& p, const int32_t* table, int head, int j) {
  const int k = p.by_block.div(j);
  const int32_t phys = table[k];
  if (phys < 0 || phys >= p.num_blocks) {
    flag_error(p.err, SNAPMIND_DEVERR_BLOCK_ID);
    return -1;
  }
  return ((int64_t)phys * p.n_heads + head) * p.block_size + (j - k * p.block_size);
}

// What tells the kernels of a call with targets that it was refused (their lengths do not: a target may have had its own
// before): the first kept index of a sequence's first layer and head is -1.  There evict_tables_kernel leaves it, and
// what selection writes in the end says the same: 0 or more, or -1 where a sequence keeps nothing.
__device__ __forceinline__ int32_t* mark_of(const EvictParams& p, int i) { return p.kept + (int64_t)i * p.n_heads * p.budget; }

// Order of weights as unsigned integers: -infinity lowest, infinity below NaN, -0 with 0.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x7FFFFFFFu) > 0x7F800000u ? 0xFFFFFFFFu : u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Selection: a block per (layer, sequence, head).  The weights lie in shared memory (a chunk of them when there
// are more), warp w holding run w of the chunk's indexes; the order of the last that stays is found from a histogram
// of the highest 11 bits, counted as the weights come in, and then among the few of its bin (or 11 bits at a time, if
// they are not few), and the kept indexes are counted per warp by ballots and written out in a second sweep.  What
// bounds it is instructions (64% of the issue slots: the sweeps, and orders made of weights), with a read of the
// table, one of the weights and a handful of barriers for latency, so blocks are small where sequences are short,
// several to an SM: 1024 units of 2112 tokens 26 us, 1024 of 1 to 8 thousand 67, 128 of 32768 47.  Tried and dropped:
// histogram additions put together by the lanes of a bin (128 units: 77 us, 54 without), fewer registers (76 us, 70).
constexpr int kRadix = 11, kBins = 1 << kRadix;
static_assert(2 * 49152 / 32 <= kBins + 1024, "bits of a chunk");
constexpr int kFew = 256;  // that many are listed and compared with one another (800 took 25 us more than another histogram)

template <int THREADS>
struct SelectSmem {
  int32_t bins[kBins + 1024];  // later two words of bits for every 32 indexes of a chunk
  int32_t above[THREADS / 32], equal[THREADS / 32];
  uint32_t prefix;  // of the lowest kept order
  int32_t need;     // how many with exactly that order stay
  int32_t there;    // indexes in the prefix's bin
  int32_t listed;
};

template <int THREADS>
__global__ void __launch_bounds__(THREADS) evict_select_kernel(const __grid_constant__ EvictParams p, int chunk) {
  extern __shared__ __align__(16) float held[];  // [chunk], a multiple of 4 * THREADS
  __shared__ SelectSmem<THREADS> S;
  constexpr int kWarps = THREADS / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int layer = blockIdx.x / (p.n * p.n_heads), u = blockIdx.x - layer * (p.n * p.n_heads);
  const int i = u / p.n_heads, head = u - i * p.n_heads;
  int32_t* kept = p.kept + (int64_t)blockIdx.x * p.budget;
  const bool copies = p.dst != nullptr, refused = copies && *mark_of(p, i) < 0;
  const int from = src_id(p, i), to = dst_id(p, i);
  const int len = cached(p, from), keep = min(len, p.budget);
  float* mass = p.mass + layer * p.mass_layer;
  const int32_t* table = p.tables + (int64_t)from * p.table_stride;
  const int32_t* new_table = p.tables + (int64_t)to * p.table_stride;
  for (int x = (refused ? 0 : keep) + tid; x < p.budget; x += THREADS) kept[x] = -1;
  if (refused) return;
  if (len <= p.budget) {
    for (int x = tid; x < keep; x += THREADS) {
      kept[x] = x;
      if (copies) {
        const int64_t a = row_of(p, table, head, x), b = row_of(p, new_table, head, x);
        if (a >= 0 && b >= 0) mass[b] = mass[a];
      }
    }
    return;
  }
  // what stays in any case takes no part: [0, lo) and [hi, len)
  const int lo = min(p.sinks, keep), hi = len - min(p.recent, keep - lo);
  const bool one = len <= chunk;
  int need = keep - lo - (len - hi);  // of [lo, hi)
  const bool none = need <= 0;
  const auto count = [&](int x, float m) {  // the first histogram: the highest bits
    if (x >= lo && x < hi) atomicAdd(&S.bins[order_of(m) >> (32 - kRadix)], 1);
  };
  // weights [c0, c0 + chunk) into shared memory (an index without a block: -infinity), counted on the way if all fit
  const auto load = [&](int c0) {
    const int n = min(chunk, len - c0);
    if ((p.block_size & 3) == 0) {
      constexpr int kDeep = 4;
      for (int x0 = 4 * tid; x0 < n; x0 += 4 * THREADS * kDeep) {
        float4 v[kDeep];
#pragma unroll
        for (int y = 0; y < kDeep; ++y) {
          const int x = x0 + y * 4 * THREADS;
          v[y] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
          if (x < n) {
            const int64_t row = row_of(p, table, head, c0 + x);  // four slots of a block
            if (row >= 0) v[y] = *reinterpret_cast<const float4*>(mass + row);
          }
        }
#pragma unroll
        for (int y = 0; y < kDeep; ++y)
          if (x0 + y * 4 * THREADS < n) {
            const int x = x0 + y * 4 * THREADS;
            *reinterpret_cast<float4*>(held + x) = v[y];
            if (one && !none) count(x, v[y].x), count(x + 1, v[y].y), count(x + 2, v[y].z), count(x + 3, v[y].w);
          }
      }
    } else {
      for (int x = tid; x < n; x += THREADS) {
        const int64_t row = row_of(p, table, head, c0 + x);
        held[x] = row < 0 ? -INFINITY : mass[row];
        if (one && !none) count(x, held[x]);
      }
    }
  };
  for (int x = tid; x < kBins; x += THREADS) S.bins[x] = 0;
  __syncthreads();
  if (one) load(0);
  uint32_t prefix = 0;
  int shift = 32;
  // the order of the need-th largest, 11, 11 and 10 bits at a time
  for (int pass = 0; pass < 3 && !none; ++pass) {
    const int bits = pass < 2 ? kRadix : 32 - 2 * kRadix;
    if (pass > 0) {
      for (int x = tid; x < kBins; x += THREADS) S.bins[x] = 0;
      __syncthreads();
    }
    for (int c0 = 0; c0 < len && !(one && pass == 0); c0 += chunk) {
      if (!one) {
        __syncthreads();
        load(c0);
        __syncthreads();
      }
      const int x1 = min(hi, c0 + chunk);
      for (int x = max(lo, c0) + tid; x < x1; x += THREADS) {
        const uint32_t k = order_of(held[x - c0]);
        if (shift == 32 || k >> shift == prefix >> shift) atomicAdd(&S.bins[(k >> (shift - bits)) & ((1u << bits) - 1)], 1);
      }
    }
    __syncthreads();
    // from the highest bin down: the bin where the count reaches `need`
    constexpr int kPer = kBins / THREADS;
    int mine[kPer], sum = 0;
#pragma unroll
    for (int y = 0; y < kPer; ++y) {
      mine[y] = S.bins[kBins - 1 - (tid * kPer + y)];
      sum += mine[y];
    }
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    if (lane == 31) S.above[warp] = incl;
    __syncthreads();
    int before = incl - sum;
    {
      int x = lane < warp ? S.above[lane] : 0;  // 32 warps at most
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
      before += x;
    }
#pragma unroll
    for (int y = 0; y < kPer; ++y) {
      if (before < need && before + mine[y] >= need) {
        S.prefix = prefix | (uint32_t)(kBins - 1 - (tid * kPer + y)) << (shift - bits);
        S.need = need - before;
        S.there = mine[y];
        S.listed = 0;
      }
      before += mine[y];
    }
    __syncthreads();
    prefix = S.prefix;
    need = S.need;
    shift -= bits;
    const int there = S.there;
    if (one && shift > 0 && there <= kFew) {
      // listed where the bins were, which all have read; each counts those above it
      uint32_t* list = reinterpret_cast<uint32_t*>(S.bins);
      for (int x = lo + tid; x < hi; x += THREADS) {
        const uint32_t k = order_of(held[x]);
        if (k >> shift == prefix >> shift) list[atomicAdd(&S.listed, 1)] = k;
      }
      __syncthreads();
      if (tid < there) {
        const uint32_t k = list[tid];
        int above = 0, same = 0;
        for (int j = 0; j < there; ++j) {
          const uint32_t other = list[j];
          above += other > k;
          same += other == k;
        }
        if (above < need && above + same >= need) {  // (its equals write the same)
          S.prefix = k;
          S.need = need - above;
        }
      }
      __syncthreads();
      prefix = S.prefix;
      need = S.need;
      break;
    }
  }
  // in ascending order: what is above the border stays, of those on it the first `need`.  A chunk is read whole
  // before its kept weights are written, which is never past its own end.
  int at = 0, equal = 0;
  for (int c0 = 0; c0 < len; c0 += chunk) {
    const int n = min(chunk, len - c0);
    if (!one) {
      __syncthreads();
      load(c0);
    }
    __syncthreads();
    const int run = (n + 32 * kWarps - 1) / (32 * kWarps) * 32, x0 = min(n, warp * run), x1 = min(n, x0 + run);  // x0 of a run with an index is a multiple of 32
    // 32 indexes' bits: those that stay, those on the border
    uint2* bits = reinterpret_cast<uint2*>(S.bins);
    int above = 0, on = 0;
    for (int x = x0; x < x1; x += 32) {
      const int j = c0 + x + lane;
      bool sure = j < lo || j >= hi, border = false;
      if (!sure && !none) {
        const uint32_t k = order_of(held[min(x + lane, x1 - 1)]);
        sure = k > prefix;
        border = k == prefix;
      }
      const bool there = x + lane < x1;
      const uint32_t a = __ballot_sync(0xffffffffu, there && sure), e = __ballot_sync(0xffffffffu, there && border);
      if (lane == 0) bits[x >> 5] = make_uint2(a, e);
      above += __popc(a);
      on += __popc(e);
    }
    if (lane == 0) {
      S.above[warp] = above;
      S.equal[warp] = on;
    }
    __syncthreads();
    int mine_at = at, mine_equal = equal, all_at = at, all_equal = equal;
    for (int w = 0; w < kWarps; ++w) {
      const int e = S.equal[w], k = S.above[w] + min(e, max(0, need - all_equal));
      if (w < warp) {
        mine_at += k;
        mine_equal += e;
      }
      all_at += k;
      all_equal += e;
    }
    const uint32_t below = (1u << lane) - 1u;
    for (int x = x0; x < x1; x += 32) {
      const uint2 m = bits[x >> 5];
      const bool stays = (m.x >> lane & 1) || ((m.y >> lane & 1) && mine_equal + __popc(m.y & below) < need);
      const uint32_t those = m.y == 0 ? m.x : __ballot_sync(0xffffffffu, stays);
      if (stays) {
        const int place = mine_at + __popc(those & below);
        kept[place] = c0 + x + lane;
        const int64_t b = row_of(p, new_table, head, place);
        if (b >= 0) mass[b] = held[x + lane];
      }
      mine_at += __popc(those);
      mine_equal += __popc(m.y);
    }
    at = all_at;
    equal = all_equal;
  }
}

// Rows of the kept tokens of one (layer, sequence, head): a block moves slice_bytes of each K or V row, TEAM lanes of
// W bytes a row, 32 rows a warp and step.  A lane works out where one row comes from and goes to (and moves its
// scale), and the teams fetch that by shuffles; the next step's indexes are read while this one's rows are on
// their way.  Where there are few units, a row's columns go to several blocks, which never meet.  HBM bound: 16 layers
// of 4096 rows of 256 bytes for each of 8 heads, K and V, take 105 us (5.1 TB/s; 227 with a row's place worked out by every
// lane of it), 8-bit rows of 1024 units 94 (5.6 TB/s).
constexpr int kMoveThreads = 256;
template <int W, int TEAM>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const __grid_constant__ EvictParams p) {
  using V = typename VecT<W>::type;
  constexpr int kTeams = 32 / TEAM, kDeep = TEAM;  // rows of a warp side by side, passes: 32 rows
  constexpr int kHold = kDeep < 16 ? kDeep : 16;   // passes whose rows are held at once
  constexpr int kRows = kHold * kTeams;            // of a warp and step
  const int unit = blockIdx.x, kv = blockIdx.y & 1, slice = blockIdx.y >> 1;
  const int layer = unit / (p.n * p.n_heads), u = unit - layer * (p.n * p.n_heads);
  const int i = u / p.n_heads, head = u - i * p.n_heads;
  const int from = src_id(p, i), to = dst_id(p, i);
  const int len = cached(p, from), keep = min(len, p.budget);
  const bool copies = p.dst != nullptr;
  const int32_t* kept = p.kept + (int64_t)unit * p.budget;
  if (copies ? *mark_of(p, i) < 0 : len <= p.budget) return;
  const int32_t* table = p.tables + (int64_t)from * p.table_stride;
  const int32_t* new_table = p.tables + (int64_t)to * p.table_stride;
  uint8_t* pool = p.pool[kv] + layer * p.pool_layer + slice * p.slice_bytes;
  uint8_t* scales = p.scales && slice == 0 ? p.scales + layer * p.scale_layer : nullptr;
  const int vecs = min(p.slice_bytes, p.row_bytes - slice * p.slice_bytes) / W;  // of a row
  int first = 0;
  if (!copies) {  // p_i - i never falls: the first that moves
    int hi = keep;
    while (first < hi) {
      const int mid = (first + hi) >> 1;
      if (kept[mid] > mid) hi = mid;
      else first = mid + 1;
    }
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane / TEAM, x = lane % TEAM;
  constexpr int kWarps = kMoveThreads / 32, kStep = kWarps * kRows;
  const auto scale_at = [&](int64_t row) {
    const int64_t block = row / p.block_size;
    return (block * 2 + kv) * p.block_size + (row - block * p.block_size);
  };
  const auto index = [&](int base) {
    const int k = base + warp * kRows + lane;
    return lane < kRows && k < keep ? kept[k] : -1;
  };
  int next = index(first);
  for (int base = first; base < keep; base += kStep) {
    const int k = base + warp * kRows + lane;
    int64_t a = -1, b = -1;
    if (next >= 0) {
      a = row_of(p, table, head, next);
      b = row_of(p, new_table, head, k);
      if (a < 0 || b < 0) a = b = -1;
    }
    V v[kHold];
#pragma unroll
    for (int y = 0; y < kHold; ++y) {
      const int64_t r = __shfl_sync(0xffffffffu, a, y * kTeams + sub);
      if (r >= 0 && x < vecs) v[y] = *reinterpret_cast<const V*>(pool + r * p.row_bytes + x * W);
    }
    uint8_t sc = 0;
    if (scales && a >= 0) sc = scales[scale_at(a)];
    next = index(base + kStep);
    if (!copies) __syncthreads();  // all of the step is read before any of it is written
#pragma unroll
    for (int y = 0; y < kHold; ++y) {
      const int64_t r = __shfl_sync(0xffffffffu, b, y * kTeams + sub);
      if (r >= 0 && x < vecs) *reinterpret_cast<V*>(pool + r * p.row_bytes + x * W) = v[y];
    }
    if (scales && b >= 0) scales[scale_at(b)] = sc;
  }
}

// Lengths, table rows and the free stack, by one block.  Sequence i of the call ends with
// min(length of its source, budget) tokens.  Blocks are taken from the top of the stack in ascending order of
// the call's sequences and come back in the reverse order, so that a pool that grows and evicts in turn gets the
// same blocks again.
constexpr int kTableThreads = 1024;
__global__ void __launch_bounds__(kTableThreads) evict_tables_kernel(const __grid_constant__ EvictParams p) {
  __shared__ int32_t s_pop[32], s_push[32];
  __shared__ int32_t s_total[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int run = (p.n + kTableThreads - 1) / kTableThreads;
  const int i0 = min(p.n, tid * run), i1 = min(p.n, i0 + run);
  const auto blocks = [&](int len) { return p.by_block.div(len + p.block_size - 1); };
  const auto ends = [&](int i) { return min(cached(p, src_id(p, i)), p.budget); };
  int pop = 0, push = 0;
  for (int i = i0; i < i1; ++i) {
    const int d = blocks(ends(i)) - blocks(cached(p, dst_id(p, i)));
    pop += max(d, 0);
    push += max(-d, 0);
  }
  int a = pop, b = push;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) a += x, b += y;
  }
  if (lane == 31) s_pop[warp] = a, s_push[warp] = b;
  __syncthreads();
  if (tid == 0) {
    int x = 0, y = 0;
    for (int w = 0; w < kTableThreads / 32; ++w) {
      const int px = s_pop[w], py = s_push[w];
      s_pop[w] = x, s_push[w] = y;
      x += px, y += py;
    }
    s_total[0] = x, s_total[1] = y;
  }
  __syncthreads();
  const int top = *p.free_top, pops = s_total[0], pushes = s_total[1];
  const int left = top - pops, end = left + pushes;
  const bool refused = left < 0 || end > p.num_blocks;
  if (p.dst != nullptr)  // (in place the other kernels have run already)
    for (int i = i0; i < i1; ++i) *mark_of(p, i) = refused ? -1 : 0;
  if (refused) {  // nothing changes
    if (tid == 0) flag_error(p.err, SNAPMIND_DEVERR_OUT_OF_BLOCKS);
    return;
  }
  // every length is read before one is written: a source is no target of another sequence
  int x = s_pop[warp] + a - pop, y = s_push[warp] + b - push;
  // all that is popped is read before anything is pushed over it
  for (int i = i0; i < i1; ++i) {
    const int d = dst_id(p, i), old = blocks(cached(p, d)), now = blocks(ends(i));
    int32_t* table = p.tables + (int64_t)d * p.table_stride;
    for (int k = old; k < now; ++k) table[k] = p.free_stack[top - 1 - x++];
  }
  __syncthreads();
  for (int i = i0; i < i1; ++i) {
    const int d = dst_id(p, i), old = blocks(cached(p, d)), len = ends(i), now = blocks(len);
    const int32_t* table = p.tables + (int64_t)d * p.table_stride;
    for (int k = now; k < old; ++k) p.free_stack[end - 1 - y++] = table[k];
  }
  __syncthreads();
  // in place a sequence's own length is its source's: after all reads of its own
  for (int i = i0; i < i1; ++i) {
    const int len = ends(i);
    p.seq_lens[dst_id(p, i)] = len;
  }
  if (tid == 0) *p.free_top = end;
}

// Weights of the newest tokens of every sequence: 0, in all layers.  Not after a reserve that failed: those of older tokens
// would go.
struct ClearParams {
  float* mass;
  int64_t mass_layer;
  const int32_t* tables;
  int64_t table_stride;
  int32_t table_width;
  const int32_t* seq_lens;
  const int32_t* counts;  // NULL: n_new each
  int32_t n_new, batch, n_layers, n_heads, block_size, num_blocks;
  const int32_t* status;  // of the reserve
};
__global__ void __launch_bounds__(256) clear_mass_kernel(const __grid_constant__ ClearParams p) {
  if (p.status != nullptr && (*p.status & (SNAPMIND_DEVERR_OUT_OF_BLOCKS | SNAPMIND_DEVERR_TABLE)) != 0) return;
  const int per = p.n_layers * p.n_heads;
  for (int b = blockIdx.y; b < p.batch; b += gridDim.y) {
    const int len = p.seq_lens[b], n = min(p.counts ? p.counts[b] : p.n_new, len);
    for (int64_t e = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; e < (int64_t)n * per; e += (int64_t)gridDim.x * blockDim.x) {
      // (layer, head) outer, tokens inner: a block's slots lie side by side
      const int lh = (int)(e / n), j = len - n + (int)(e - (int64_t)lh * n);
      const int layer = lh / p.n_heads, head = lh - layer * p.n_heads, k = j / p.block_size;
      if (k >= p.table_width) continue;
      const int32_t phys = p.tables[(int64_t)b * p.table_stride + k];
      if (phys < 0 || phys >= p.num_blocks) continue;
      p.mass[layer * p.mass_layer + ((int64_t)phys * p.n_heads + head) * p.block_size + (j - k * p.block_size)] = 0.f;
    }
  }
}

}  // namespace
}  // namespace snapmind

using namespace snapmind;

extern "C" {

int snapmind_kv_evict_by_mass(void* k_pool, void* v_pool, void* scales, int pool_dtype, int64_t pool_layer_stride,
                              int64_t scale_layer_stride, float* mass, int64_t mass_layer_stride, int32_t* block_tables,
                              int64_t table_stride_seq, int32_t table_width, int32_t* seq_lens, const int32_t* seqs,
                              const int32_t* into, int32_t n_seqs, int32_t budget, int32_t recent, int32_t sinks,
                              int32_t max_len, int32_t* kept, int32_t* free_stack, int32_t* free_top, int32_t n_layers,
                              int32_t n_heads, int32_t head_dim, int32_t block_size, int32_t num_blocks, int32_t* err_word,
                              void* stream) {
  const bool quant = pool_dtype == SNAPMIND_DTYPE_E4M3;
  SNAPMIND_CHECK_ARG(quant || dtype_size(pool_dtype) > 0, "kv_evict: unknown pool dtype");
  SNAPMIND_CHECK_ARG(quant == (scales != nullptr), "kv_evict: scales go with an e4m3 pool, and only with one");
  SNAPMIND_CHECK_ARG(n_seqs >= 0 && n_layers > 0 && n_heads > 0 && head_dim > 0 && block_size > 0 && num_blocks > 0 && table_width >= 0,
                     "kv_evict: bad sizes");
  SNAPMIND_CHECK_ARG(budget > 0 && recent >= 0 && sinks >= 0 && (int64_t)recent + sinks <= budget,
                     "kv_evict: the newest %d and the first %d tokens do not fit a budget of %d", recent, sinks, budget);
  SNAPMIND_CHECK_ARG((int64_t)table_width * block_size < (int64_t)1 << 31, "kv_evict: table rows of %d blocks are too long", table_width);
  const int64_t units = (int64_t)n_layers * n_seqs * n_heads;
  SNAPMIND_CHECK_ARG(units < (int64_t)1 << 31, "kv_evict: too many layers, sequences and heads for one call");
  if (n_seqs == 0) return SNAPMIND_OK;
  SNAPMIND_CHECK_ARG(k_pool && v_pool && mass && block_tables && seq_lens && kept && free_stack && free_top, "kv_evict: null pointer");
  SNAPMIND_CHECK_ARG(into == nullptr || seqs != nullptr, "kv_evict: targets need the sequences named");
  // weights are read four at a time where a block's are a multiple of four
  SNAPMIND_CHECK_ARG(block_size % 4 != 0 || ((reinterpret_cast<uintptr_t>(mass) & 15) == 0 && mass_layer_stride % 4 == 0),
                     "kv_evict: with blocks of %d tokens each layer of mass must stand on a 16-byte boundary", block_size);
  EvictParams p = {};
  p.tables = block_tables;
  p.table_stride = table_stride_seq;
  p.table_width = table_width;
  p.seq_lens = seq_lens;
  p.src = seqs;
  p.dst = into;
  p.n = n_seqs;
  p.n_layers = n_layers;
  p.n_heads = n_heads;
  p.block_size = block_size;
  p.num_blocks = num_blocks;
  p.budget = budget;
  p.recent = recent;
  p.sinks = sinks;
  p.by_block = FastDiv(block_size);
  p.mass = mass;
  p.mass_layer = mass_layer_stride;
  p.kept = kept;
  p.pool[0] = static_cast<uint8_t*>(k_pool);
  p.pool[1] = static_cast<uint8_t*>(v_pool);
  const int esz = quant ? 1 : dtype_size(pool_dtype);
  p.row_bytes = head_dim * esz;
  p.pool_layer = pool_layer_stride * esz;
  p.scales = static_cast<uint8_t*>(scales);
  p.scale_layer = scale_layer_stride;
  p.free_stack = free_stack;
  p.free_top = free_top;
  p.err = err_word;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (into) evict_tables_kernel<<<1, kTableThreads, 0, st>>>(p);
  // Sequences of up to 4096 tokens: 256 threads (4 blocks an SM), up to 16384: 512, above: 1024, each with room for
  // that many weights (above: 49152 at a time).  Calls that keep 256 rows of 16 bytes, us with 256 / 512 / 1024 threads: 1024 units
  // of 4096 tokens 66 / 76 / 104, of 8192 90 / 97 / 128 (16 units: 39 / 35 / 35), 512 units of 16384 109 / 87 / 104, 256
  // units of 17000 66 / 55 / 64, of 32768 158 / 100 / 85.
  const int64_t room = (int64_t)table_width * block_size, longest = max_len > 0 && max_len < room ? max_len : room;
  const auto select = [&](auto kernel, int threads, bool (&done)[64]) -> cudaError_t {
    const int64_t step = 4 * (int64_t)threads;
    const int chunk = (int)((longest < 49152 ? longest + step - 1 : (int64_t)49152) / step * step);
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev >= 64 || !done[dev])) {
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 49152 * 4);
      if (e == cudaSuccess)  // room for the blocks that are meant to share an SM
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
      if (e == cudaSuccess && dev < 64) done[dev] = true;
    }
    if (e == cudaSuccess) kernel<<<(uint32_t)units, threads, chunk * 4, st>>>(p, chunk);
    return e;
  };
  static bool done[3][64] = {};
  const cudaError_t e = longest <= 4096 ? select(evict_select_kernel<256>, 256, done[0])
                        : longest <= 16384 ? select(evict_select_kernel<512>, 512, done[1])
                                           : select(evict_select_kernel<1024>, 1024, done[2]);
  if (e != cudaSuccess) return cuda_status(e, "kv_evict select");
  const int w = vec_width(p.row_bytes, p.pool_layer, reinterpret_cast<intptr_t>(k_pool), reinterpret_cast<intptr_t>(v_pool));
  // a slice of up to 32 vectors a row; halves of it (128 bytes at least) while there are few blocks for the SMs
  p.slice_bytes = p.row_bytes < 32 * w ? p.row_bytes : 32 * w;
  while (p.slice_bytes % (2 * w) == 0 && p.slice_bytes >= 256 &&
         units * 2 * ((p.row_bytes + p.slice_bytes - 1) / p.slice_bytes) < 4 * num_sms())
    p.slice_bytes /= 2;
  p.slices = (p.row_bytes + p.slice_bytes - 1) / p.slice_bytes;
  SNAPMIND_CHECK_ARG(2 * (int64_t)p.slices <= 65535, "kv_evict: rows of %d bytes are too long", p.row_bytes);
  const dim3 grid((uint32_t)units, 2 * p.slices);
  const auto move = [&](auto width) {
    constexpr int W = decltype(width)::value;
    const int vecs = p.slice_bytes / W;
    if (vecs <= 4) evict_move_kernel<W, 4><<<grid, kMoveThreads, 0, st>>>(p);
    else if (vecs <= 8) evict_move_kernel<W, 8><<<grid, kMoveThreads, 0, st>>>(p);
    else if (vecs <= 16) evict_move_kernel<W, 16><<<grid, kMoveThreads, 0, st>>>(p);
    else evict_move_kernel<W, 32><<<grid, kMoveThreads, 0, st>>>(p);
  };
  switch (w) {
    case 16: move(std::integral_constant<int, 16>()); break;
    case 8: move(std::integral_constant<int, 8>()); break;
    case 4: move(std::integral_constant<int, 4>()); break;
    case 2: move(std::integral_constant<int, 2>()); break;
    default: move(std::integral_constant<int, 1>());
  }
  if (!into) evict_tables_kernel<<<1, kTableThreads, 0, st>>>(p);
  return cuda_status(cudaGetLastError(), "kv_evict launch");
}

int snapmind_kv_clear_mass(float* mass, int64_t mass_layer_stride, const int32_t* block_tables, int64_t table_stride_seq,
                           int32_t table_width, const int32_t* seq_lens, const int32_t* counts, int32_t n_new, int32_t batch,
                           int32_t n_layers, int32_t n_heads, int32_t block_size, int32_t num_blocks,
                           const int32_t* status, void* stream) {
  SNAPMIND_CHECK_ARG(batch >= 0 && n_new >= 0 && n_layers > 0 && n_heads > 0 && block_size > 0 && num_blocks > 0 && table_width >= 0,
                     "kv_clear_mass: bad sizes");
  if (batch == 0 || (counts == nullptr && n_new == 0)) return SNAPMIND_OK;
  SNAPMIND_CHECK_ARG(mass && block_tables && seq_lens, "kv_clear_mass: null pointer");
  const ClearParams p{mass, mass_layer_stride, block_tables, table_stride_seq, table_width, seq_lens, counts, n_new,
                      batch, n_layers, n_heads, block_size, num_blocks, status};
  const int64_t each = counts ? 4096 : (int64_t)n_new * n_layers * n_heads;
  const int64_t blocks = (each + 255) / 256;
  const dim3 grid((uint32_t)(blocks < 64 ? blocks : 64), (uint32_t)(batch < 1024 ? batch : 1024));
  clear_mass_kernel<<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(p);
  return cuda_status(cudaGetLastError(), "kv_clear_mass launch");
}

}  // extern "C"
