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
// sum of squares is a few shuffles and the rotation's partner is one lane away; a CTA takes a token, and a lane keeps
// the token's cosines and sines for all the rows that it does.
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

template <typename T>
__device__ __forceinline__ void load8(const T* x, float* f) {
  uint4 w[sizeof(T) / 2];
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const uint4*>(x)[i];
  const T* e = reinterpret_cast<const T*>(w);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = Conv<T>::to_f(e[i]);
}
template <typename T>
__device__ __forceinline__ void store8(T* x, const float* f) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(x)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(x)[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    *reinterpret_cast<uint4*>(x) = make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
  }
}

// One CTA per token; TEAM lanes per row, of which head_dim / 8 hold eight elements each.
template <typename T, typename KV, int TEAM>
__global__ void __launch_bounds__(kThreads) norm_rope_kernel(const __grid_constant__ NormRopeParams p) {
  constexpr int kTeams = kThreads / TEAM;
  constexpr bool kQuant = std::is_same<KV, uint8_t>::value;
  const int team = threadIdx.x / TEAM, lane = threadIdx.x % TEAM;
  const int b = p.n_seq == 1 ? 0 : blockIdx.x / p.n_tok, t = blockIdx.x - b * p.n_tok;
  const bool stores = p.v.in != nullptr;
  const bool mine = 8 * lane < p.head_dim, turns = 8 * lane < p.rot;
  const int d = mine ? 8 * lane : 0;
  // the lane that holds the rotation's partner, and its sign
  const int half = p.rot / 16, other = !turns ? lane : lane < half ? lane + half : lane - half;
  const float sign = lane < half ? -1.f : 1.f;
  const int64_t pos = token_position(p, b, t);
  if (pos < 0) return;
  const int64_t slot = stores ? token_slot(p, t) : -1;
  float c[8], s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = 1.f, s[i] = 0.f;
  if (turns) {
    load8(p.cos_t + pos * p.rot + d, c);
    load8(p.sin_t + pos * p.rot + d, s);
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] *= sign;
  }
  const int rows = p.q.heads + p.k.heads + (stores ? p.v.heads : 0);
  const float inv_d = 1.f / p.head_dim;
  for (int r0 = 0; r0 < rows; r0 += kTeams) {
    const int r = r0 + team;  // a warp's teams run together: shuffles inside
    const int kind = r < p.q.heads ? 0 : r < p.q.heads + p.k.heads ? 1 : 2;
    const int h = kind == 0 ? r : kind == 1 ? r - p.q.heads : r - p.q.heads - p.k.heads;
    const RowSet& set = kind == 0 ? p.q : kind == 1 ? p.k : p.v;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.f;
    if (r < rows && mine) load8(static_cast<const T*>(set.in) + b * set.seq + h * set.head + t * set.tok + d, x);
    // the teams of a warp may hold rows of different kinds: every shuffle is taken by all lanes
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
#pragma unroll
    for (int o = TEAM / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const void* norm = kind == 0 ? p.q_norm : kind == 1 ? p.k_norm : nullptr;
    if (norm != nullptr && r < rows) {
      float w[8];
      load8(static_cast<const T*>(norm) + h * (kind == 0 ? p.q_norm_head : p.k_norm_head) + d, w);
      const float f = 1.f / sqrtf(fmaf(sum, inv_d, p.eps));
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] * f * w[i];
    }
    __syncwarp();
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = __shfl_sync(0xffffffffu, x[i], other, TEAM);
    if (kind < 2) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = fmaf(y[i], s[i], x[i] * c[i]);
    }
    float a = 0.f;
    if (kQuant) {
#pragma unroll
      for (int i = 0; i < 8; ++i) a = fmaxf(a, finite_abs(x[i]));
#pragma unroll
      for (int o = TEAM / 2; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
    }
    if (r >= rows || !mine) continue;
    if (kind == 0 || !stores) {
      store8(static_cast<T*>(set.out) + b * set.out_seq + h * set.out_head + t * set.out_tok + d, x);
    } else if (slot >= 0) {
      const int64_t row = slot + (int64_t)h * p.block_size;
      KV* to = static_cast<KV*>(p.pool[kind - 1]) + row * p.head_dim + d;
      if constexpr (kQuant) {
        const int e = row_exponent(a);
        const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
        *reinterpret_cast<uint2*>(to) = make_uint2(codes4(scaled(x[0], inv), scaled(x[1], inv), scaled(x[2], inv), scaled(x[3], inv)),
                                                   codes4(scaled(x[4], inv), scaled(x[5], inv), scaled(x[6], inv), scaled(x[7], inv)));
        if (lane == 0) p.scales[scale_byte_at(p, row, kind - 1)] = (uint8_t)(e + 127);
      } else {
        store8(to, x);
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
        each([&](int d, float z) { to[d] = (uint8_t)codes4(scaled(z, inv), 0.f, 0.f, 0.f); });
        if (lane == 0) p.scales[scale_byte_at(p, row, kind - 1)] = (uint8_t)(e + 127);
      } else {
        each([&](int d, float z) { to[d] = Conv<KV>::from_f(z); });
      }
    }
  }
}

bool vectors_fit(const NormRopeParams& p, int esz, int pool_esz) {
  if (p.head_dim % 8 || p.head_dim > 256 || p.rot % 16) return false;
  const auto a16 = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; };
  const int v = 16 / esz;
  for (const RowSet* s : {&p.q, &p.k, &p.v}) {
    if (!a16(s->in) || !a16(s->out)) return false;
    if (s->seq % v || s->head % v || s->tok % v || s->out_seq % v || s->out_head % v || s->out_tok % v) return false;
  }
  if (!a16(p.q_norm) || !a16(p.k_norm) || p.q_norm_head % v || p.k_norm_head % v) return false;
  if (!a16(p.cos_t) || !a16(p.sin_t)) return false;
  return a16(p.pool[0]) && a16(p.pool[1]) && (p.head_dim * pool_esz) % 8 == 0;
}

template <typename T, typename KV>
int launch(const NormRopeParams& p, cudaStream_t st) {
  const int64_t tokens = (int64_t)p.n_seq * p.n_tok;
  if (vectors_fit(p, sizeof(T), sizeof(KV))) {
    const int lanes = p.head_dim / 8;
    if (lanes <= 8) norm_rope_kernel<T, KV, 8><<<(uint32_t)tokens, kThreads, 0, st>>>(p);
    else if (lanes <= 16) norm_rope_kernel<T, KV, 16><<<(uint32_t)tokens, kThreads, 0, st>>>(p);
    else norm_rope_kernel<T, KV, 32><<<(uint32_t)tokens, kThreads, 0, st>>>(p);
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
                         tokens < (int64_t)1 << 31,
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
