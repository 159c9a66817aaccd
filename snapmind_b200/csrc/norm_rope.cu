// Norms of queries and keys for each head, their rotation, and the store of the keys and values into a paged
// pool, in one pass over the projections' rows.
//
//   y = x / sqrt(mean x^2 + eps) * w                     (w given; else y = x)
//   z[d] = y[d] cos[p][d] + rot(y)[d] sin[p][d], d < R   rot(y)[d] = -y[d + R/2] (d < R/2), y[d - R/2] else
//   z[d] = y[d], d >= R
//
// for the queries (into q_out) and the keys; p is the token's own position, which is not its index in a
// cache that evicts.  Keys and values go to their slots of the pool (f32, 16-bit, or e4m3 rows quantised
// as the append kernel does), or the keys to a plain tensor.  All arithmetic is f32, rounded once on the way out.
//
// HBM bound: a row is read once and written once.  A team of lanes holds a row, eight elements a lane, so a
// sum of squares is a few shuffles and the rotation's partner is one lane away.
#include "pairs.cuh"

namespace snapmind {
namespace {

constexpr int kThreads = 256;

struct RowSet {  // rows [seq][head][token] of one of q, k, v: strides in elements
  const void* in;
  int64_t seq, head, tok;
  void* out;
  int64_t out_seq, out_head, out_tok;
  int32_t heads;
};

struct NormRopeParams {
  RowSet q, k, v;  // v.in NULL: no values, and k goes to k.out
  const void* q_norm;
  const void* k_norm;
  int64_t q_norm_head, k_norm_head;  // elements between the heads' weights (0: one for all)
  float eps;
  const float* cos_t;
  const float* sin_t;
  int32_t rot;  // dims that are rotated
  int64_t n_pos;
  const int64_t* positions;
  int64_t pos_seq;
  int32_t n_seq, n_tok, head_dim;
  // pool
  void* pool[2];
  uint8_t* scales;
  const int32_t* tables;
  int64_t table_stride;
  int32_t table_width, block_size, num_blocks, batch;
  const int32_t* seq_lens;
  const int32_t* cu;  // [batch + 1] or NULL: sequence b's only new token is token b
  int32_t* err;
};

// Where token i (of the packed ones) goes: *base = block * kv heads * block_size + slot; head h adds h * block_size.
// -1: nowhere (outside every sequence, or flagged).
__device__ __forceinline__ int64_t token_slot(const NormRopeParams& p, int i) {
  int b = i, back = 1;
  if (p.cu != nullptr) {
    b = upper_bound_i32(p.cu, p.batch + 1, i) - 1;
    if (b < 0 || b >= p.batch) return -1;
    back = p.cu[b + 1] - i;
  }
  const int slot = p.seq_lens[b] - back;
  const int j = slot < 0 ? 0 : slot / p.block_size;
  if (slot < 0 || j >= p.table_width) {
    flag_error(p.err, SNAPMIND_DEVERR_TABLE);
    return -1;
  }
  const int32_t phys = p.tables[(int64_t)b * p.table_stride + j];
  if (phys < 0 || phys >= p.num_blocks) {
    flag_error(p.err, SNAPMIND_DEVERR_BLOCK_ID);
    return -1;
  }
  return (int64_t)phys * p.k.heads * p.block_size + (slot - j * p.block_size);
}
// Byte of a pool row's exponent: [block][head][K, V][slot].
__device__ __forceinline__ int64_t scale_byte_at(const NormRopeParams& p, int64_t row, int kv) {
  const int64_t tile = row / p.block_size;
  return (tile * 2 + kv) * p.block_size + (row - tile * p.block_size);
}
// The token's position, -1: outside the tables (flagged).
__device__ __forceinline__ int64_t token_position(const NormRopeParams& p, int b, int t) {
  const int64_t pos = p.positions ? p.positions[(int64_t)b * p.pos_seq + t] : t;
  if (pos >= 0 && pos < p.n_pos) return pos;
  flag_error(p.err, SNAPMIND_DEVERR_POSITION);
  return -1;
}

// A lane's eight elements of a row: four from d0 and four from d1, as they lie in memory and as pairs of f32.
template <typename T> struct Four { using type = uint2; };
template <> struct Four<float> { using type = uint4; };
template <typename T> struct Raw { typename Four<T>::type w[2]; };
template <typename T>
__device__ __forceinline__ Raw<T> load_raw(const T* x, int d0, int d1) {
  using V = typename Four<T>::type;
  return Raw<T>{{*reinterpret_cast<const V*>(x + d0), *reinterpret_cast<const V*>(x + d1)}};
}
template <typename T>
__device__ __forceinline__ void spread8(const Raw<T>& r, float2* f) {
  const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = make_float2(Conv<T>::to_f(e[2 * i]), Conv<T>::to_f(e[2 * i + 1]));
}
template <typename T>
__device__ __forceinline__ void store4(T* x, float2 a, float2 b) {
  if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(x) = make_float4(a.x, a.y, b.x, b.y);
  else *reinterpret_cast<uint2*>(x) = make_uint2(pack2<T>(a.x, a.y), pack2<T>(b.x, b.y));
}

// A CTA takes a run of items (token, kHeads heads) of one of q, k and v; TEAM lanes hold a row, head_dim / 8 of them eight
// elements each: a lane of the rotated part four and the four that they turn with, so nothing is exchanged but the
// sum of squares, and a token's cosines and sines serve kHeads rows.  Where tokens come from and go to (positions,
// sequences, lengths, table entries: reads that wait for one another) is worked out for all of a CTA's tokens at
// once, and the next item's rows, cosines and sines are on their way while one is computed.  Fewer instructions
// made it fast: 8200 tokens of 48 heads of 128 (bf16) took 70 us with 219 a row and warp (64-bit
// addresses, partners by shuffles), 79 with 178 and cosines that a row waited for, 41 us (4.6 TB/s) with 115.  Now
// neither they (56% of the issue slots; into 8-bit rows 53%) nor HBM (41%; 25%) are full, at 16 warps an SM and one item
// ahead.
struct Rows32 { int32_t seq, head, tok, out_seq, out_head, out_tok; };  // RowSet's strides where they fit
struct Split {
  Rows32 at[3];        // q, k, v
  int32_t q, k;        // CTAs of q, of k (v's come last)
  int32_t items;       // of a CTA
  FastDiv by_groups[2], by_tok;  // groups of kHeads heads: of q, of k and v
  int32_t groups[2];
};
constexpr int kMostItems = 512, kHeads = 4;

template <typename T, typename KV, int TEAM>
__global__ void __launch_bounds__(kThreads, 2) norm_rope_kernel(const __grid_constant__ NormRopeParams p, const __grid_constant__ Split split) {
  constexpr int kTeams = kThreads / TEAM;
  constexpr bool kQuant = std::is_same<KV, uint8_t>::value;
  constexpr uint32_t kAll = 0xffffffffu;
  __shared__ int32_t at_turn[kMostItems + 2];  // of the CTA's tokens: the first of its cosines, -1: no such position
  __shared__ int64_t at_row[kMostItems + 2];   // pool row of head 0, -1: none
  __shared__ int64_t at_scale[kQuant ? kMostItems + 2 : 1];  // its K scale
  const int team = threadIdx.x / TEAM, lane = threadIdx.x % TEAM;
  const bool mine = 8 * lane < p.head_dim, turns = 8 * lane < p.rot;
  const int d0 = !mine ? 0 : turns ? 4 * lane : 8 * lane, d1 = !mine ? 4 : turns ? p.rot / 2 + d0 : d0 + 4;
  const int cta = blockIdx.x, kind = cta < split.q ? 0 : cta < split.q + split.k ? 1 : 2;
  const RowSet& set = kind == 0 ? p.q : kind == 1 ? p.k : p.v;
  const Rows32& by = split.at[kind];
  const FastDiv& by_groups = split.by_groups[kind > 0];
  const int n_groups = split.groups[kind > 0], all = p.n_seq * p.n_tok * n_groups;
  const int e0 = (cta - (kind == 0 ? 0 : kind == 1 ? split.q : split.q + split.k)) * split.items, e1 = min(all, e0 + split.items);
  const int token0 = by_groups.div(e0), tokens = by_groups.div(e1 - 1) - token0 + 1;
  const bool stores = kind > 0 && p.v.in != nullptr;
  const T* in = static_cast<const T*>(set.in);
  const auto sequence = [&](int token) { return p.n_seq == 1 ? 0 : split.by_tok.div(token); };
  struct Item { Raw<T> row[kHeads]; };
  const auto fetch = [&](Item& r, int e) {
    r = Item{};
    if (e >= e1 || !mine) return;
    const int token = by_groups.div(e), head = (e - token * n_groups) * kHeads, b = sequence(token);
    const T* from = in + (b * by.seq + head * by.head + (token - b * p.n_tok) * by.tok);
#pragma unroll
    for (int h = 0; h < kHeads; ++h)
      if (head + h < set.heads) r.row[h] = load_raw(from + h * by.head, d0, d1);
  };
  Raw<float> c_next = {}, s_next = {};
  const auto fetch_turn = [&](int e) {
    if (kind == 2 || !turns || e >= e1) return;
    const int turn = at_turn[by_groups.div(e) - token0];
    if (turn < 0) return;
    c_next = load_raw(p.cos_t + turn, d0, d1);
    s_next = load_raw(p.sin_t + turn, d0, d1);
  };
  Item next;
  fetch(next, e0 + team);
  for (int i = threadIdx.x; i < tokens; i += kThreads) {
    const int token = token0 + i, b = sequence(token), t = token - b * p.n_tok;
    const int64_t pos = token_position(p, b, t);
    at_turn[i] = pos < 0 ? -1 : (int)pos * p.rot;
    const int64_t row = stores && pos >= 0 ? token_slot(p, t) : -1;
    at_row[i] = row;
    if (kQuant && row >= 0) at_scale[i] = scale_byte_at(p, row, 0);
  }
  // a row's largest magnitude, by its team; infinities become NaN, as they are stored, and NaN do not count
  const auto magnitude = [&](float2* x) {
    const auto largest = [&] {
      float a = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) a = fmaxf(a, fmaxf(fabsf(x[k].x), fabsf(x[k].y)));
#pragma unroll
      for (int o = TEAM / 2; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(kAll, a, o));
      return a;
    };
    float a = largest();
    if (__any_sync(kAll, a == INFINITY)) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        x[k].x = fabsf(x[k].x) < INFINITY ? x[k].x : __uint_as_float(0x7FC00000u);
        x[k].y = fabsf(x[k].y) < INFINITY ? x[k].y : __uint_as_float(0x7FC00000u);
      }
      a = largest();
    }
    return a;
  };
  // a row into the pool: of token token0 + i, head h
  const auto put = [&](int i, int64_t row0, int h, const float2* x, float a) {
    KV* to = static_cast<KV*>(p.pool[kind > 1]) + (row0 + h * p.block_size) * p.head_dim;
    if constexpr (kQuant) {
      const int x2 = row_exponent(a);
      const float inv = __uint_as_float((uint32_t)(127 - x2) << 23);
      const auto codes = [&](float2 y, float2 z) {
        y = mul2(y, inv), z = mul2(z, inv);
        return codes4(y.x, y.y, z.x, z.y);
      };
      *reinterpret_cast<uint32_t*>(to + d0) = codes(x[0], x[1]);
      *reinterpret_cast<uint32_t*>(to + d1) = codes(x[2], x[3]);
      if (lane == 0) p.scales[at_scale[i] + (2 * h + kind - 1) * p.block_size] = (uint8_t)(x2 + 127);
    } else {
      store4(to + d0, x[0], x[1]);
      store4(to + d1, x[2], x[3]);
    }
  };
  if (kind == 2) {  // values: as they are, in the pool's type
    __syncthreads();
    for (int base = e0; base < e1; base += kTeams) {
      const int e = min(base + team, e1 - 1), i = by_groups.div(e) - token0, head0 = (e - (token0 + i) * n_groups) * kHeads;
      const int64_t row0 = at_row[i];
      const bool there = base + team < e1 && row0 >= 0 && mine;
#pragma unroll
      for (int h = 0; h < kHeads; ++h) {
        const bool on = there && head0 + h < set.heads;
        if constexpr (std::is_same<T, KV>::value) {
          if (on) {
            T* to = static_cast<T*>(p.pool[1]) + (row0 + (head0 + h) * p.block_size) * p.head_dim;
            *reinterpret_cast<typename Four<T>::type*>(to + d0) = next.row[h].w[0];
            *reinterpret_cast<typename Four<T>::type*>(to + d1) = next.row[h].w[1];
          }
        } else {
          float2 x[4];
          spread8(next.row[h], x);
          const float a = kQuant ? magnitude(x) : 0.f;
          if (on) put(i, row0, head0 + h, x, a);
        }
      }
      fetch(next, base + kTeams + team);
    }
    return;
  }
  const T* norm = static_cast<const T*>(kind == 0 ? p.q_norm : p.k_norm);
  const int norm_head = (int)(kind == 0 ? p.q_norm_head : p.k_norm_head);
  float2 w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) w[k] = make_float2(1.f, 1.f);
  if (norm != nullptr && norm_head == 0) spread8(load_raw(norm, d0, d1), w);
  const float inv_d = 1.f / p.head_dim;
  __syncthreads();
  fetch_turn(e0 + team);
  for (int base = e0; base < e1; base += kTeams) {
    const Item now = next;
    float2 c[4], s[4];
    spread8(c_next, c);
    spread8(s_next, s);
#pragma unroll
    for (int k = 0; k < 2; ++k) s[k] = make_float2(-s[k].x, -s[k].y);
    fetch(next, base + kTeams + team);
    fetch_turn(base + kTeams + team);
    const int e = min(base + team, e1 - 1), token = by_groups.div(e), i = token - token0, head0 = (e - token * n_groups) * kHeads;
    const int64_t row0 = at_row[i];
    const bool there = base + team < e1 && at_turn[i] >= 0 && mine && (!stores || row0 >= 0);
    const int b = sequence(token);
    T* to_out = static_cast<T*>(set.out) + (b * by.out_seq + head0 * by.out_head + (token - b * p.n_tok) * by.out_tok);
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      const bool on = there && head0 + h < set.heads;
      float2 x[4];
      spread8(now.row[h], x);
      if (norm != nullptr) {
        float2 sq = times(x[0], x[0]);
#pragma unroll
        for (int k = 1; k < 4; ++k) sq = fma2(x[k], x[k], sq);
        float sum = sq.x + sq.y;
#pragma unroll
        for (int o = TEAM / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(kAll, sum, o);
        const float f = rsqrtf(fmaf(sum, inv_d, p.eps));
        if (norm_head != 0 && on) spread8(load_raw(norm + (head0 + h) * norm_head, d0, d1), w);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = times(mul2(x[k], f), w[k]);
      }
      if (turns) {  // x[0 .. 1] turn with x[2 .. 3]
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float2 y0 = x[k], y1 = x[k + 2];
          x[k] = fma2(y1, s[k], times(y0, c[k]));
          x[k + 2] = fma2(y0, s[k + 2], times(y1, c[k + 2]));
        }
      }
      if (stores) {
        const float a = kQuant ? magnitude(x) : 0.f;
        if (on) put(i, row0, head0 + h, x, a);
      } else if (on) {
        store4(to_out + h * by.out_head + d0, x[0], x[1]);
        store4(to_out + h * by.out_head + d1, x[2], x[3]);
      }
    }
  }
}

// Any head_dim, strides and alignment: a warp per row, two passes over it.
template <typename T, typename KV>
__global__ void __launch_bounds__(kThreads) norm_rope_any_kernel(const __grid_constant__ NormRopeParams p) {
  constexpr bool kQuant = std::is_same<KV, uint8_t>::value;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = p.n_seq == 1 ? 0 : blockIdx.x / p.n_tok, t = blockIdx.x - b * p.n_tok;
  const bool stores = p.v.in != nullptr;
  const int64_t pos = token_position(p, b, t);
  if (pos < 0) return;
  const int64_t slot = stores ? token_slot(p, t) : -1;
  const int rows = p.q.heads + p.k.heads + (stores ? p.v.heads : 0), half = p.rot / 2;
  for (int r = warp; r < rows; r += kThreads / 32) {
    const int kind = r < p.q.heads ? 0 : r < p.q.heads + p.k.heads ? 1 : 2;
    const int h = kind == 0 ? r : kind == 1 ? r - p.q.heads : r - p.q.heads - p.k.heads;
    const RowSet& set = kind == 0 ? p.q : kind == 1 ? p.k : p.v;
    const T* in = static_cast<const T*>(set.in) + b * set.seq + h * set.head + t * set.tok;
    const T* norm = kind == 2 ? nullptr : static_cast<const T*>(kind == 0 ? p.q_norm : p.k_norm);
    if (norm) norm += h * (kind == 0 ? p.q_norm_head : p.k_norm_head);
    float f = 1.f;
    if (norm) {
      float sum = 0.f;
      for (int d = lane; d < p.head_dim; d += 32) sum = fmaf(Conv<T>::to_f(in[d]), Conv<T>::to_f(in[d]), sum);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      f = 1.f / sqrtf(fmaf(sum, 1.f / p.head_dim, p.eps));
    }
    const auto normed = [&](int d) { return norm ? Conv<T>::to_f(in[d]) * f * Conv<T>::to_f(norm[d]) : Conv<T>::to_f(in[d]); };
    // elements lane, lane + 32, ...: in place is safe, since a lane reads a rotated pair before it writes it
    const auto value = [&](int d, float x, float y) {  // y: the partner's
      if (kind == 2 || d >= p.rot) return x;
      const float s = p.sin_t[pos * p.rot + d];
      return fmaf(y, d < half ? -s : s, x * p.cos_t[pos * p.rot + d]);
    };
    const auto each = [&](auto&& put) {
      for (int d = lane; d < (kind == 2 ? 0 : half); d += 32) {
        const float x = normed(d), y = normed(d + half);
        put(d, value(d, x, y));
        put(d + half, value(d + half, y, x));
      }
      for (int d = (kind == 2 ? 0 : p.rot) + lane; d < p.head_dim; d += 32) put(d, normed(d));
    };
    if (kind == 0 || !stores) {
      T* out = static_cast<T*>(set.out) + b * set.out_seq + h * set.out_head + t * set.out_tok;
      each([&](int d, float z) { out[d] = Conv<T>::from_f(z); });
    } else if (slot >= 0) {
      const int64_t row = slot + (int64_t)h * p.block_size;
      KV* to = static_cast<KV*>(p.pool[kind - 1]) + row * p.head_dim;
      if constexpr (kQuant) {
        float a = 0.f;
        each([&](int, float z) { a = fmaxf(a, finite_abs(z)); });
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
        const int e = row_exponent(a);
        const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
        each([&](int d, float z) { to[d] = (uint8_t)codes2(scaled(z, inv), 0.f); });
        if (lane == 0) p.scales[scale_byte_at(p, row, kind - 1)] = (uint8_t)(e + 127);
      } else {
        each([&](int d, float z) { to[d] = Conv<KV>::from_f(z); });
      }
    }
  }
}

// Whether the rows are whole pieces of four elements, and their offsets fit 32 bits.
bool pieces_fit(const NormRopeParams& p, int esz, int pool_esz, Split& split) {
  if (p.head_dim % 8 || p.head_dim > 256 || p.rot % 8) return false;
  const auto aligned = [](const void* x, int to) { return (reinterpret_cast<uintptr_t>(x) & (to - 1)) == 0; };
  const RowSet* sets[3] = {&p.q, &p.k, &p.v};
  for (int i = 0; i < 3; ++i) {
    const RowSet& s = *sets[i];
    if (!aligned(s.in, 4 * esz) || !aligned(s.out, 4 * esz)) return false;
    const auto fit = [&](int64_t seq, int64_t head, int64_t tok) {
      if (seq < 0 || head < 0 || tok < 0 || seq % 4 || head % 4 || tok % 4) return false;
      const auto reach = [](int64_t stride, int64_t n) { return n <= 1 ? 0.0 : (double)stride * (double)(n - 1); };
      return reach(seq, p.n_seq) + reach(head, s.heads) + reach(tok, p.n_tok) + p.head_dim < 2147483648.0;
    };
    if (!fit(s.seq, s.head, s.tok) || !fit(s.out_seq, s.out_head, s.out_tok)) return false;
    const auto of = [](int64_t stride, int n) { return n <= 1 ? 0 : (int32_t)stride; };
    split.at[i] = Rows32{of(s.seq, p.n_seq), of(s.head, s.heads), of(s.tok, p.n_tok), of(s.out_seq, p.n_seq), of(s.out_head, s.heads), of(s.out_tok, p.n_tok)};
  }
  for (int64_t head : {p.q_norm_head, p.k_norm_head})
    if (head < 0 || head % 4 || head > 1 << 20) return false;
  if (!aligned(p.q_norm, 4 * esz) || !aligned(p.k_norm, 4 * esz) || !aligned(p.cos_t, 16) || !aligned(p.sin_t, 16)) return false;
  if (p.n_pos * p.rot >= (int64_t)1 << 31) return false;
  return aligned(p.pool[0], 4 * pool_esz) && aligned(p.pool[1], 4 * pool_esz);
}

template <typename T, typename KV>
int launch(const NormRopeParams& p, cudaStream_t st) {
  const int64_t tokens = (int64_t)p.n_seq * p.n_tok;
  Split split = {};
  if (pieces_fit(p, sizeof(T), sizeof(KV), split)) {
    const int lanes = p.head_dim / 8;
    // items of a CTA: one wave of two CTAs an SM, an item for every team at least
    for (int i = 0; i < 2; ++i) {
      split.groups[i] = ((i ? p.k.heads : p.q.heads) + kHeads - 1) / kHeads;
      split.by_groups[i] = FastDiv(split.groups[i] > 0 ? split.groups[i] : 1);
    }
    const int64_t all = tokens * (split.groups[0] + split.groups[1] * (p.v.in ? 2 : 1)), slots = 2 * (int64_t)num_sms() - 2;
    const int teams = kThreads / (lanes <= 8 ? 8 : lanes <= 16 ? 16 : 32);
    int64_t items = ((all + slots - 1) / slots + teams - 1) / teams * teams;
    items = items < kMostItems ? items : kMostItems;
    split.items = (int32_t)items;
    split.q = (int32_t)((tokens * split.groups[0] + items - 1) / items);
    split.k = (int32_t)((tokens * split.groups[1] + items - 1) / items);
    split.by_tok = FastDiv(p.n_tok);
    const uint32_t grid = split.q + split.k + (p.v.in ? split.k : 0);
    if (lanes <= 8) norm_rope_kernel<T, KV, 8><<<grid, kThreads, 0, st>>>(p, split);
    else if (lanes <= 16) norm_rope_kernel<T, KV, 16><<<grid, kThreads, 0, st>>>(p, split);
    else norm_rope_kernel<T, KV, 32><<<grid, kThreads, 0, st>>>(p, split);
  } else {
    norm_rope_any_kernel<T, KV><<<(uint32_t)tokens, kThreads, 0, st>>>(p);
  }
  return cuda_status(cudaGetLastError(), "norm_rope launch");
}

template <typename T>
int launch_for(const NormRopeParams& p, int pool_dtype, cudaStream_t st) {
  switch (pool_dtype) {
    case SNAPMIND_DTYPE_F32: return launch<T, float>(p, st);
    case SNAPMIND_DTYPE_BF16: return launch<T, __nv_bfloat16>(p, st);
    case SNAPMIND_DTYPE_F16: return launch<T, __half>(p, st);
    default: return launch<T, uint8_t>(p, st);
  }
}
int launch_any(const NormRopeParams& p, int dtype, int pool_dtype, cudaStream_t st) {
  switch (dtype) {
    case SNAPMIND_DTYPE_F32: return launch_for<float>(p, pool_dtype, st);
    case SNAPMIND_DTYPE_BF16: return launch_for<__nv_bfloat16>(p, pool_dtype, st);
    default: return launch_for<__half>(p, pool_dtype, st);
  }
}

// What both entry points check of the rows, norms and tables.
int check_common(const NormRopeParams& p, int dtype, int64_t tokens) {
  SNAPMIND_CHECK_ARG(dtype_size(dtype) > 0, "norm_rope: unknown dtype");
  SNAPMIND_CHECK_ARG(p.n_seq >= 0 && p.n_tok >= 0 && p.q.heads >= 0 && p.k.heads > 0 && p.head_dim > 0 && p.n_pos > 0 &&
                         tokens * (p.q.heads > p.k.heads ? p.q.heads : p.k.heads) < (int64_t)1 << 30,
                     "norm_rope: bad sizes");
  SNAPMIND_CHECK_ARG(p.rot >= 0 && p.rot <= p.head_dim && p.rot % 2 == 0, "norm_rope: %d rotated dims of %d (even, at most head_dim)",
                     p.rot, p.head_dim);
  SNAPMIND_CHECK_ARG(p.eps >= 0.f, "norm_rope: eps must not be negative");
  if (tokens == 0) return SNAPMIND_OK;
  SNAPMIND_CHECK_ARG((p.q.heads == 0 || (p.q.in && p.q.out)) && p.k.in && (p.rot == 0 || (p.cos_t && p.sin_t)),
                     "norm_rope: null pointer");
  return SNAPMIND_OK;
}

}  // namespace
}  // namespace snapmind

using namespace snapmind;

extern "C" {

int snapmind_norm_rope_qk(const void* q, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_t, void* q_out,
                          int64_t qo_stride_b, int64_t qo_stride_h, int64_t qo_stride_t, int32_t n_q_heads, const void* k,
                          int64_t k_stride_b, int64_t k_stride_h, int64_t k_stride_t, void* k_out, int64_t ko_stride_b,
                          int64_t ko_stride_h, int64_t ko_stride_t, int32_t n_kv_heads, int dtype, const void* q_norm,
                          int64_t q_norm_stride_h, const void* k_norm, int64_t k_norm_stride_h, float eps, int32_t batch,
                          int32_t n_tok, int32_t head_dim, const float* cos_table, const float* sin_table, int32_t rot_dim,
                          int64_t n_pos, const int64_t* positions, int64_t pos_stride_b, int32_t* err_word, void* stream) {
  NormRopeParams p = {};
  p.q = RowSet{q, q_stride_b, q_stride_h, q_stride_t, q_out, qo_stride_b, qo_stride_h, qo_stride_t, n_q_heads};
  p.k = RowSet{k, k_stride_b, k_stride_h, k_stride_t, k_out, ko_stride_b, ko_stride_h, ko_stride_t, n_kv_heads};
  p.q_norm = q_norm;
  p.k_norm = k_norm;
  p.q_norm_head = q_norm_stride_h;
  p.k_norm_head = k_norm_stride_h;
  p.eps = eps;
  p.cos_t = cos_table;
  p.sin_t = sin_table;
  p.rot = rot_dim;
  p.n_pos = n_pos;
  p.positions = positions;
  p.pos_seq = pos_stride_b;
  p.n_seq = batch;
  p.n_tok = n_tok;
  p.head_dim = head_dim;
  p.err = err_word;
  const int64_t tokens = (int64_t)batch * n_tok;
  const int rc = check_common(p, dtype, tokens);
  if (rc != SNAPMIND_OK || tokens == 0) return rc;
  SNAPMIND_CHECK_ARG(k_out != nullptr, "norm_rope: null pointer");
  return launch_any(p, dtype, dtype, static_cast<cudaStream_t>(stream));
}

int snapmind_norm_rope_append(const void* q, int64_t q_stride_tok, int64_t q_stride_head, void* q_out, int64_t qo_stride_tok,
                              int64_t qo_stride_head, int32_t n_q_heads, const void* k, int64_t k_stride_tok,
                              int64_t k_stride_head, const void* v, int64_t v_stride_tok, int64_t v_stride_head, int dtype,
                              const void* q_norm, int64_t q_norm_stride_head, const void* k_norm, int64_t k_norm_stride_head,
                              float eps, const float* cos_table, const float* sin_table, int32_t rot_dim, int64_t n_pos,
                              const int64_t* positions, void* k_pool, void* v_pool, void* scales, int pool_dtype,
                              const int32_t* block_tables, int64_t table_stride_seq, int32_t table_width,
                              const int32_t* seq_lens, const int32_t* cu_new, int32_t batch, int32_t total_new,
                              int32_t n_kv_heads, int32_t head_dim, int32_t block_size, int32_t num_blocks,
                              int32_t* err_word, void* stream) {
  SNAPMIND_CHECK_ARG(dtype_size(pool_dtype) > 0 || pool_dtype == SNAPMIND_DTYPE_E4M3, "norm_rope: unknown pool dtype");
  SNAPMIND_CHECK_ARG((pool_dtype == SNAPMIND_DTYPE_E4M3) == (scales != nullptr),
                     "norm_rope: scales go with an e4m3 pool, and only with one");
  SNAPMIND_CHECK_ARG(batch >= 0 && block_size > 0 && num_blocks > 0 && table_width >= 0, "norm_rope: bad sizes");
  SNAPMIND_CHECK_ARG(cu_new != nullptr || total_new == batch, "norm_rope: without cu_new there is one token per sequence");
  NormRopeParams p = {};
  p.q = RowSet{q, 0, q_stride_head, q_stride_tok, q_out, 0, qo_stride_head, qo_stride_tok, n_q_heads};
  p.k = RowSet{k, 0, k_stride_head, k_stride_tok, nullptr, 0, 0, 0, n_kv_heads};
  p.v = RowSet{v, 0, v_stride_head, v_stride_tok, nullptr, 0, 0, 0, n_kv_heads};
  p.q_norm = q_norm;
  p.k_norm = k_norm;
  p.q_norm_head = q_norm_stride_head;
  p.k_norm_head = k_norm_stride_head;
  p.eps = eps;
  p.cos_t = cos_table;
  p.sin_t = sin_table;
  p.rot = rot_dim;
  p.n_pos = n_pos;
  p.positions = positions;
  p.n_seq = 1;
  p.n_tok = total_new;
  p.head_dim = head_dim;
  p.pool[0] = k_pool;
  p.pool[1] = v_pool;
  p.scales = static_cast<uint8_t*>(scales);
  p.tables = block_tables;
  p.table_stride = table_stride_seq;
  p.table_width = table_width;
  p.block_size = block_size;
  p.num_blocks = num_blocks;
  p.batch = batch;
  p.seq_lens = seq_lens;
  p.cu = cu_new;
  p.err = err_word;
  const int rc = check_common(p, dtype, total_new);
  if (rc != SNAPMIND_OK || total_new == 0) return rc;
  SNAPMIND_CHECK_ARG(v && k_pool && v_pool && block_tables && seq_lens && positions, "norm_rope: null pointer");
  return launch_any(p, dtype, pool_dtype, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
