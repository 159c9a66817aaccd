// Rows written into a paged pool from ragged or uniform chunks, quantised to 8 bits when
// the pool holds e4m3, and 8-bit pools read back.
//
// Quantisation of a row x of one token and head (head_dim values, K or V):
//   e = the smallest integer in [-100, 120] with max |x| <= 448 2^e,
//   c = x 2^-e rounded to e4m3 (nearest even);
// the pool keeps the codes [block][head][slot][dim] (1 byte each) and one byte e + 127 per
// row, [block][head][K, V][slot], so a 16-token tile's 32 scale bytes are one sector.  The
// scale is a power of two, because then scaling is exact: no rounding but e4m3's own, codes
// that do not hang on a division's last bit, values that bf16 holds exactly, and nothing
// lost, since the relative step of e4m3 (2^-4 at most, half a step) is the same at
// every scale.  Infinities and NaN are stored as NaN and do not count for the scale.
//
// Both kernels are byte movers: a team of lanes owns a row (16-byte vectors of the wide
// side), several rows in flight per team.
#include "pairs.cuh"

namespace snapmind {
namespace {

constexpr int kThreads = 256;

struct ChunkAppendParams {
  uint8_t* pool[2];
  uint8_t* scales;
  const char* in[2];
  int64_t pool_layer_stride, scale_layer_stride;                          // bytes
  int64_t in_stride_layer, in_stride_seq, in_stride_head, in_stride_tok;  // bytes
  const int32_t* tables;
  int64_t table_stride;
  int32_t table_width;
  const int32_t* slot_starts;
  int32_t slot_start0;
  const int32_t* cu;  // [batch + 1] first row of every sequence, or NULL: n_tokens each
  int32_t batch, n_tokens, total, n_heads, head_dim, block_size, num_blocks;
  int32_t heads_inner;  // consecutive rows walk the heads (else the tokens)
  FastDiv by_heads, by_tokens, by_block;
  int32_t* err;
};

// Exponent of a row whose largest finite magnitude is a.
__device__ __forceinline__ int row_exponent(float a) {
  const uint32_t u = __float_as_uint(a);
  const int k = (int)(u >> 23) - 127;
  const int e = (u & 0x7FFFFFu) <= 0x600000u ? k - 8 : k - 7;  // a <= 1.75 2^(e + 8)
  return min(max(e, -100), 120);
}

__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;  // false for NaN too
}
__device__ __forceinline__ float scaled(float x, float inv) {
  return fabsf(x) < INFINITY ? x * inv : __uint_as_float(0x7FC00000u);
}
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

template <typename T> struct Vec { static constexpr int N = 16 / sizeof(T); };

template <typename T>
__device__ __forceinline__ void unpack(const uint4& w, float* f) {
  const T* t = reinterpret_cast<const T*>(&w);
#pragma unroll
  for (int i = 0; i < Vec<T>::N; ++i) f[i] = Conv<T>::to_f(t[i]);
}

// A row of the (layer, K or V) plane.
struct AppendRow {
  int b, i, h;  // sequence (cu_new: unknown yet), token (packed, or within the sequence), head
};
__device__ __forceinline__ AppendRow append_row(const ChunkAppendParams& p, int r) {
  AppendRow a;
  if (p.heads_inner) {
    a.i = p.by_heads.div(r);
    a.h = r - a.i * p.n_heads;
    a.b = 0;
    if (p.cu == nullptr) {
      a.b = p.by_tokens.div(a.i);
      a.i -= a.b * p.n_tokens;
    }
  } else {  // (sequence, head, token)
    const int bh = p.by_tokens.div(r);
    a.i = r - bh * p.n_tokens;
    a.b = p.by_heads.div(bh);
    a.h = bh - a.b * p.n_heads;
  }
  return a;
}
__device__ __forceinline__ const char* append_src(const ChunkAppendParams& p, const char* in, const AppendRow& a) {
  const int64_t seq = p.cu == nullptr ? (int64_t)a.b * p.in_stride_seq : 0;
  return in + seq + (int64_t)a.i * p.in_stride_tok + (int64_t)a.h * p.in_stride_head;
}
// Pool row of (block, head, slot), or -1 (skipped: outside every sequence, or flagged).
__device__ __forceinline__ int64_t append_dst(const ChunkAppendParams& p, const AppendRow& a) {
  int b = a.b, t = a.i, n = 0;
  if (p.cu != nullptr) {
    b = upper_bound_i32(p.cu, p.batch + 1, a.i) - 1;  // rows outside every sequence are not stored
    if (b < 0 || b >= p.batch) return -1;
    t = a.i - p.cu[b];
    n = p.cu[b + 1] - p.cu[b];
  }
  const int slot = (p.slot_starts ? p.slot_starts[b] : 0) + p.slot_start0 - n + t;
  const int j = slot < 0 ? 0 : p.by_block.div(slot);
  if (slot < 0 || j >= p.table_width) {
    flag_error(p.err, SNAPMIND_DEVERR_TABLE);
    return -1;
  }
  const int32_t phys = p.tables[(int64_t)b * p.table_stride + j];
  if (phys < 0 || phys >= p.num_blocks) {
    flag_error(p.err, SNAPMIND_DEVERR_BLOCK_ID);
    return -1;
  }
  return ((int64_t)phys * p.n_heads + a.h) * p.block_size + (slot - j * p.block_size);
}

// Byte of a row's exponent: row = (block * heads + head) * block_size + slot.
__device__ __forceinline__ int64_t scale_at(const ChunkAppendParams& p, int64_t row, int kv) {
  const int tile = p.by_block.div((int)row);
  return ((int64_t)tile * 2 + kv) * p.block_size + (row - (int64_t)tile * p.block_size);
}

// Largest magnitude of a 16-byte vector as the bits of |x| (16-bit types: both halves of
// a word hold candidates): unsigned order is the order of magnitudes, infinities and NaN
// above all finite values.
template <typename T> struct Bits {
  static constexpr uint32_t kInf = std::is_same<T, float>::value ? 0x7F800000u : std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
  __device__ __forceinline__ static uint32_t max2(uint32_t a, uint32_t b) {
    if constexpr (sizeof(T) == 4) return max(a, b);
    else return __vmaxu2(a, b);
  }
  __device__ __forceinline__ static uint32_t of(const uint4& w) {
    constexpr uint32_t m = sizeof(T) == 4 ? 0x7FFFFFFFu : 0x7FFF7FFFu;
    return max2(max2(w.x & m, w.y & m), max2(w.z & m, w.w & m));
  }
  __device__ __forceinline__ static uint32_t fold(uint32_t a) {
    if constexpr (sizeof(T) == 4) return a;
    else return max(a & 0xFFFFu, a >> 16);
  }
  __device__ __forceinline__ static float value(uint32_t a) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(a);
    else if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half((unsigned short)a));
    else return __uint_as_float(a << 16);
  }
};

// Rows of TEAM lanes x two 16-byte vectors each (head_dim * sizeof(T) = 32 TEAM bytes; a lane's
// vectors are TEAM apart, so a team reads whole lines).  blockIdx.y = layer * 2 + (K, V).  A warp
// takes kRows rows a step: lane i works out where row i comes from and goes to, and the teams
// fetch that by shuffles.  The magnitude is reduced on the bits, two 16-bit values a word.
// This kernel is bound by instructions first.  16 x 2049 tokens x 4 layers, 807 MB: 483 us with
// every lane resolving its rows and unpacked magnitudes, 296 us with the bits (228 instructions
// a vector), 168 us with a lane per row (124), 142 us (5.7 TB/s) with two vectors a lane.
template <typename T, int TEAM>
__global__ void __launch_bounds__(kThreads) quant_append_kernel(ChunkAppendParams p) {
  constexpr int N = Vec<T>::N, kTeams = 32 / TEAM, kUnroll = 4, kRows = kTeams * kUnroll;
  static_assert(kRows <= 32, "a lane per row");
  using B = Bits<T>;
  const int kv = blockIdx.y & 1, layer = blockIdx.y >> 1;
  const int lane = threadIdx.x & 31, piece = lane % TEAM, sub = lane / TEAM;
  const int rows = p.total * p.n_heads;
  const char* in = p.in[kv] + layer * p.in_stride_layer;
  uint8_t* pool = p.pool[kv] + layer * p.pool_layer_stride + piece * N;
  uint8_t* scales = p.scales + layer * p.scale_layer_stride;
  const int64_t stride = (int64_t)gridDim.x * (kThreads / 32) * kRows;
  for (int64_t r0 = ((int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * kRows; r0 < rows; r0 += stride) {
    AppendRow at;
    const char* src = nullptr;
    const bool mine = lane < kRows && r0 + lane < rows;
    if (mine) {
      at = append_row(p, (int)(r0 + lane));
      src = append_src(p, in, at);
    }
    uint4 w[kUnroll][2];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const char* from = reinterpret_cast<const char*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(src), u * kTeams + sub));
      w[u][0] = w[u][1] = make_uint4(0, 0, 0, 0);
      if (from != nullptr) {
        w[u][0] = reinterpret_cast<const uint4*>(from)[piece];
        w[u][1] = reinterpret_cast<const uint4*>(from)[piece + TEAM];
      }
    }
    int row = -1;  // num_blocks * heads * block_size < 2^31
    uint32_t scale = 0;
    if (mine) {
      row = (int)append_dst(p, at);
      if (row >= 0) scale = (uint32_t)scale_at(p, row, kv);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int to = __shfl_sync(0xffffffffu, row, u * kTeams + sub);
      const uint32_t sc = __shfl_sync(0xffffffffu, scale, u * kTeams + sub);
      uint32_t bits = B::max2(B::of(w[u][0]), B::of(w[u][1]));
#pragma unroll
      for (int o = TEAM / 2; o > 0; o >>= 1) bits = B::max2(bits, __shfl_xor_sync(0xffffffffu, bits, o));
      bits = B::fold(bits);
      float f[2][N];
      unpack<T>(w[u][0], f[0]);
      unpack<T>(w[u][1], f[1]);
      float a = B::value(bits);
      if (__any_sync(0xffffffffu, bits >= B::kInf)) {  // an infinity or NaN in some row of the warp
        float fa = 0.f;
#pragma unroll
        for (int i = 0; i < 2 * N; ++i) {
          float& x = f[i / N][i % N];
          fa = fmaxf(fa, finite_abs(x));
          x = scaled(x, 1.f);
        }
#pragma unroll
        for (int o = TEAM / 2; o > 0; o >>= 1) fa = fmaxf(fa, __shfl_xor_sync(0xffffffffu, fa, o));
        a = fa;
      }
      if (to < 0) continue;
      const int e = row_exponent(a);
      const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
      uint8_t* dst = pool + (int64_t)to * p.head_dim;
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        uint32_t c[N / 4];
#pragma unroll
        for (int i = 0; i < N; i += 4) {
          const float2 lo = mul2(make_float2(f[v][i], f[v][i + 1]), inv), hi = mul2(make_float2(f[v][i + 2], f[v][i + 3]), inv);
          c[i / 4] = codes4(lo.x, lo.y, hi.x, hi.y);
        }
        if constexpr (N == 8) *reinterpret_cast<uint2*>(dst + v * TEAM * N) = make_uint2(c[0], c[1]);
        else *reinterpret_cast<uint32_t*>(dst + v * TEAM * N) = c[0];
      }
      if (piece == 0) scales[sc] = (uint8_t)(e + 127);
    }
  }
}

// Any head_dim, stride and alignment: one warp per row, one element per lane and step.
template <typename T>
__global__ void __launch_bounds__(kThreads) quant_append_any_kernel(ChunkAppendParams p) {
  const int kv = blockIdx.y & 1, layer = blockIdx.y >> 1;
  const int lane = threadIdx.x & 31;
  const int rows = p.total * p.n_heads;
  const char* in = p.in[kv] + layer * p.in_stride_layer;
  uint8_t* pool = p.pool[kv] + layer * p.pool_layer_stride;
  const int warps = gridDim.x * (kThreads / 32);
  for (int64_t r = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); r < rows; r += warps) {  // warp-uniform
    const AppendRow at = append_row(p, (int)r);
    const int64_t row = append_dst(p, at);
    if (row < 0) continue;
    const T* x = reinterpret_cast<const T*>(append_src(p, in, at));
    float a = 0.f;
    for (int d = lane; d < p.head_dim; d += 32) a = fmaxf(a, finite_abs(Conv<T>::to_f(x[d])));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
    const int e = row_exponent(a);
    const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
    for (int d = lane; d < p.head_dim; d += 32)
      pool[row * p.head_dim + d] = __nv_cvt_float_to_fp8(scaled(Conv<T>::to_f(x[d]), inv), __NV_SATFINITE, __NV_E4M3);
    if (lane == 0) p.scales[layer * p.scale_layer_stride + scale_at(p, row, kv)] = (uint8_t)(e + 127);
  }
}

// A pool of the rows' own type, rows of 32 TEAM bytes: quant_append_kernel without the
// quantisation.  16 x 2049 tokens x 4 layers, 1074 MB: 183 us (5.9 TB/s); 608 us with every lane
// resolving its row.
template <int TEAM>
__global__ void __launch_bounds__(kThreads) copy_append_kernel(ChunkAppendParams p) {
  constexpr int kTeams = 32 / TEAM, kUnroll = 4, kRows = kTeams * kUnroll;
  static_assert(kRows <= 32, "a lane per row");
  const int kv = blockIdx.y & 1, layer = blockIdx.y >> 1;
  const int lane = threadIdx.x & 31, piece = lane % TEAM, sub = lane / TEAM;
  const int rows = p.total * p.n_heads;
  const char* in = p.in[kv] + layer * p.in_stride_layer;
  uint4* pool = reinterpret_cast<uint4*>(p.pool[kv] + layer * p.pool_layer_stride) + piece;
  const int64_t stride = (int64_t)gridDim.x * (kThreads / 32) * kRows;
  for (int64_t r0 = ((int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * kRows; r0 < rows; r0 += stride) {
    const char* src = nullptr;
    int row = -1;  // num_blocks * heads * block_size < 2^31
    if (lane < kRows && r0 + lane < rows) {
      const AppendRow at = append_row(p, (int)(r0 + lane));
      src = append_src(p, in, at);
      row = (int)append_dst(p, at);
    }
    uint4 w[kUnroll][2];
    int to[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const char* from = reinterpret_cast<const char*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(src), u * kTeams + sub));
      to[u] = __shfl_sync(0xffffffffu, row, u * kTeams + sub);
      if (to[u] < 0) continue;
      w[u][0] = reinterpret_cast<const uint4*>(from)[piece];
      w[u][1] = reinterpret_cast<const uint4*>(from)[piece + TEAM];
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (to[u] < 0) continue;
      uint4* dst = pool + (int64_t)to[u] * (2 * TEAM);
      dst[0] = w[u][0];
      dst[TEAM] = w[u][1];
    }
  }
}

// A pool of plain elements: the rows are stored as they are, or converted.
template <typename Tin, typename Tout>
__global__ void __launch_bounds__(kThreads) chunk_append_kernel(ChunkAppendParams p) {
  const int kv = blockIdx.y & 1, layer = blockIdx.y >> 1;
  const int lane = threadIdx.x & 31;
  const int rows = p.total * p.n_heads;
  const char* in = p.in[kv] + layer * p.in_stride_layer;
  Tout* pool = reinterpret_cast<Tout*>(p.pool[kv] + layer * p.pool_layer_stride);
  const int warps = gridDim.x * (kThreads / 32);
  for (int64_t r = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); r < rows; r += warps) {
    const AppendRow at = append_row(p, (int)r);
    const int64_t row = append_dst(p, at);
    if (row < 0) continue;
    const Tin* x = reinterpret_cast<const Tin*>(append_src(p, in, at));
    Tout* y = pool + row * p.head_dim;
    if constexpr (std::is_same<Tin, Tout>::value) {
      if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & 7) == 0 && p.head_dim * sizeof(Tin) % 8 == 0) {
        for (int d = lane; d < p.head_dim * (int)sizeof(Tin) / 8; d += 32)
          reinterpret_cast<uint2*>(y)[d] = reinterpret_cast<const uint2*>(x)[d];
        continue;
      }
    }
    for (int d = lane; d < p.head_dim; d += 32) y[d] = Conv<Tout>::from_f(Conv<Tin>::to_f(x[d]));
  }
}

// ---------------------------------------------------------------------------
// read back
// ---------------------------------------------------------------------------
struct QuantGatherParams {
  const uint8_t* pool[2];
  const uint8_t* scales;
  char* out[2];
  int64_t pool_layer_stride, scale_layer_stride, out_layer_stride;  // bytes
  int64_t out_capacity;                                             // elements one layer's output holds
  const int32_t* tables;
  int64_t table_stride;
  int32_t table_width;
  const int32_t* seq_lens;
  int32_t batch, n_heads, head_dim, block_size, num_blocks;
  FastDiv by_block;
  int32_t* err;
};

__device__ __forceinline__ float dequant_top(float) { return 3.402823466e38f; }
__device__ __forceinline__ float dequant_top(__nv_bfloat16) { return 3.389531390e38f; }
__device__ __forceinline__ float dequant_top(__half) { return 65504.f; }

// c 2^e, held to T's finite range (a NaN stays one)
template <typename T>
__device__ __forceinline__ float held(float y) {
  const float top = dequant_top(T());
  return fabsf(y) > top ? copysignf(top, y) : y;
}
// Largest scale byte at which no code can pass T's range: 448 2^e <= top.
template <typename T> constexpr int plain_bytes() { return std::is_same<T, __half>::value ? 127 + 7 : 127 + 118; }

// N codes (the low bytes of w) times 2^(byte - 127); kHold: the range is looked at.
template <typename T, int N, bool kHold>
__device__ __forceinline__ void dequant(const uint32_t* w, int byte, T* y) {
  const float s = scale_byte_to_f(byte);
  if constexpr (N == 1) {
    y[0] = Conv<T>::from_f(held<T>(e4m3_to_f((uint8_t)w[0]) * s));
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i / 4] >> (8 * (i & 3))), __NV_E4M3);
      float2 f = mul2(__half22float2(__half2(h)), s);
      if constexpr (kHold) {
        f.x = held<T>(f.x);
        f.y = held<T>(f.y);
      }
      if constexpr (std::is_same<T, float>::value) {
        y[i] = f.x;
        y[i + 1] = f.y;
      } else if constexpr (std::is_same<T, __half>::value) {
        *reinterpret_cast<__half2*>(y + i) = __floats2half2_rn(f.x, f.y);
      } else {
        *reinterpret_cast<__nv_bfloat162*>(y + i) = __floats2bfloat162_rn(f.x, f.y);
      }
    }
  }
}

// Work item = one block of one sequence: all its heads, K and V of one layer
// (blockIdx.y).  The items of a sequence start after those of the sequences before it; a
// CTA finds its sequences by a scan of the lengths, kept in shared memory.  Rows are handled
// as in quant_append_kernel: TEAM lanes x two 16-byte vectors of output, a lane per row resolving
// it (and reading its scale byte); TEAM 0 is a warp per row, for any head_dim and alignment.
// Bound by instructions and latency before DRAM: 16 x 2049 tokens x 4 layers, 807 MB: 249 us with
// every lane resolving its vector, 147 us with a lane per row, 137 us (5.9 TB/s) with two vectors a lane.
template <typename T, int TEAM>
__global__ void __launch_bounds__(kThreads, 4) quant_gather_kernel(QuantGatherParams p) {
  extern __shared__ int32_t cu[];  // [batch + 1] first block, then [batch + 1] first token
  int32_t* cu_tok = cu + p.batch + 1;
  __shared__ int32_t s_sum[2][kThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  {
    const int run = (p.batch + kThreads - 1) / kThreads, b0 = min(p.batch, tid * run), b1 = min(p.batch, b0 + run);
    int nb = 0, nt = 0;
    for (int b = b0; b < b1; ++b) {
      const int len = max(0, p.seq_lens[b]);
      nb += (len + p.block_size - 1) / p.block_size;
      nt += len;
    }
    int xb = nb, xt = nt;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int yb = __shfl_up_sync(0xffffffffu, xb, o), yt = __shfl_up_sync(0xffffffffu, xt, o);
      if (lane >= o) {
        xb += yb;
        xt += yt;
      }
    }
    if (lane == 31) {
      s_sum[0][warp] = xb;
      s_sum[1][warp] = xt;
    }
    __syncthreads();
    int fb = xb - nb, ft = xt - nt;
    for (int w = 0; w < warp; ++w) {
      fb += s_sum[0][w];
      ft += s_sum[1][w];
    }
    for (int b = b0; b < b1; ++b) {
      const int len = max(0, p.seq_lens[b]);
      cu[b] = fb;
      cu_tok[b] = ft;
      fb += (len + p.block_size - 1) / p.block_size;
      ft += len;
    }
    if (b0 < p.batch && b1 == p.batch) {
      cu[p.batch] = fb;
      cu_tok[p.batch] = ft;
    }
    __syncthreads();
  }
  const int row_elems = p.n_heads * p.head_dim;
  if ((int64_t)cu_tok[p.batch] * row_elems > p.out_capacity) {
    if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) flag_error(p.err, SNAPMIND_DEVERR_TABLE);
    return;
  }
  constexpr int N = TEAM ? Vec<T>::N : 1, kTeam = TEAM ? TEAM : 32, kTeams = 32 / kTeam, kV = TEAM ? 2 : 1;
  constexpr int kUnroll = TEAM ? 4 : 1, kRows = kTeams * kUnroll;
  static_assert(kRows <= 32, "a lane per row");
  const int layer = blockIdx.y, piece = lane % kTeam, sub = lane / kTeam;
  struct Item {
    int b, j;
    int32_t phys;
  };
  const auto locate = [&](int it) {  // the item's block: read one item ahead
    Item x{0, 0, -1};
    if (it < cu[p.batch]) {
      x.b = upper_bound_i32(cu, p.batch + 1, it) - 1;
      x.j = it - cu[x.b];
      if (x.j < p.table_width) x.phys = p.tables[(int64_t)x.b * p.table_stride + x.j];
    }
    return x;
  };
  Item next = locate(blockIdx.x);
  for (int it = blockIdx.x; it < cu[p.batch]; it += gridDim.x) {
    const int b = next.b, j = next.j;
    const int32_t phys = next.phys;
    next = locate(it + gridDim.x);
    const int len = cu_tok[b + 1] - cu_tok[b], valid = min(p.block_size, len - j * p.block_size);
    if (phys < 0 || phys >= p.num_blocks) {
      if (tid == 0) flag_error(p.err, j < p.table_width ? SNAPMIND_DEVERR_BLOCK_ID : SNAPMIND_DEVERR_TABLE);
      continue;
    }
    const uint8_t* sc = p.scales + layer * p.scale_layer_stride + (int64_t)phys * p.n_heads * 2 * p.block_size;
    const int64_t src0 = layer * p.pool_layer_stride + (int64_t)phys * p.n_heads * p.block_size * p.head_dim;
    const int64_t dst0 = (int64_t)cu_tok[b] * row_elems + (int64_t)j * p.block_size * p.head_dim;
    const int rows = 2 * p.n_heads * p.block_size;  // (K or V, head, slot)
    for (int r0 = warp * kRows; r0 < rows; r0 += kThreads / 32 * kRows) {
      int plane = -1, byte = 0;
      uint32_t from = 0;  // within the block: 2 * heads * head_dim * block_size < 2^31
      int64_t to = 0;
      const int row = r0 + lane;
      if (lane < kRows && row < rows) {
        const int th = p.by_block.div(row), t = row - th * p.block_size;
        if (t < valid) {  // slots past the sequence's end are skipped
          plane = th >= p.n_heads;
          const int h = th - plane * p.n_heads;
          byte = sc[(h * 2 + plane) * p.block_size + t];  // lands with the codes, not before them
          from = (uint32_t)(h * p.block_size + t) * p.head_dim;
          to = dst0 + ((int64_t)h * len + t) * p.head_dim;
        }
      }
      const bool hold = __any_sync(0xffffffffu, byte > plain_bytes<T>());
      for (int d0 = 0; d0 < p.head_dim; d0 += kTeam * N * kV) {  // one turn with TEAM lanes a row
        const int d = d0 + piece * N;
        uint32_t codes[kUnroll][kV][2];
        int kv[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          kv[u] = __shfl_sync(0xffffffffu, plane, u * kTeams + sub);
          const uint32_t f = __shfl_sync(0xffffffffu, from, u * kTeams + sub);
          if (d >= p.head_dim) kv[u] = -1;
          if (kv[u] < 0) continue;
          const uint8_t* src = p.pool[kv[u]] + src0 + f + d;
#pragma unroll
          for (int v = 0; v < kV; ++v, src += kTeam * N) {
            if constexpr (N == 8) {
              const uint2 x = *reinterpret_cast<const uint2*>(src);
              codes[u][v][0] = x.x;
              codes[u][v][1] = x.y;
            } else if constexpr (N == 4) {
              codes[u][v][0] = *reinterpret_cast<const uint32_t*>(src);
            } else {
              codes[u][v][0] = *src;
            }
          }
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          const int64_t dst = __shfl_sync(0xffffffffu, to, u * kTeams + sub) + d;
          const int by = __shfl_sync(0xffffffffu, byte, u * kTeams + sub);
          if (kv[u] < 0) continue;
          T* out = reinterpret_cast<T*>(p.out[kv[u]] + layer * p.out_layer_stride) + dst;
#pragma unroll
          for (int v = 0; v < kV; ++v, out += kTeam * N) {
            __align__(16) T y[N];
            if (hold) dequant<T, N, true>(codes[u][v], by, y);
            else dequant<T, N, false>(codes[u][v], by, y);
            if constexpr (TEAM != 0) *reinterpret_cast<uint4*>(out) = *reinterpret_cast<const uint4*>(y);
            else *out = y[0];
          }
        }
      }
    }
  }
}

inline bool aligned16(const void* a) { return (reinterpret_cast<uintptr_t>(a) & 15) == 0; }

// Whether rows and pool may be moved in 16-byte vectors.
inline bool append_vectors(const ChunkAppendParams& p) {
  return aligned16(p.in[0]) && aligned16(p.in[1]) && aligned16(p.pool[0]) && aligned16(p.pool[1]) &&
         p.in_stride_layer % 16 == 0 && p.in_stride_seq % 16 == 0 && p.in_stride_head % 16 == 0 &&
         p.in_stride_tok % 16 == 0 && p.pool_layer_stride % 8 == 0;
}
template <typename K>
int launch_append(K kernel, int rows_per_cta, const ChunkAppendParams& p, int n_layers, cudaStream_t st) {
  const int64_t want = ((int64_t)p.total * p.n_heads + rows_per_cta - 1) / rows_per_cta;
  const int planes = 2 * n_layers;
  const int64_t cap = ((int64_t)num_sms() * 8 + planes - 1) / planes;  // about one wave over all planes
  kernel<<<dim3((unsigned)(want < cap ? want : cap), planes), kThreads, 0, st>>>(p);
  return cuda_status(cudaGetLastError(), "kv_append_chunk launch");
}

template <typename T>
int launch_quant_append(const ChunkAppendParams& p, int n_layers, cudaStream_t st) {
  const int row_bytes = append_vectors(p) ? p.head_dim * (int)sizeof(T) : 0;
  switch (row_bytes) {
    case 16 * 32: return launch_append(quant_append_kernel<T, 16>, 4 * kThreads / 16, p, n_layers, st);
    case 8 * 32: return launch_append(quant_append_kernel<T, 8>, 4 * kThreads / 8, p, n_layers, st);
    case 4 * 32: return launch_append(quant_append_kernel<T, 4>, 4 * kThreads / 4, p, n_layers, st);
    default: return launch_append(quant_append_any_kernel<T>, kThreads / 32, p, n_layers, st);
  }
}

template <typename Tin>
int launch_plain_append(const ChunkAppendParams& p, int in_dtype, int pool_dtype, int n_layers, cudaStream_t st) {
  const bool copies = in_dtype == pool_dtype && append_vectors(p) && p.pool_layer_stride % 16 == 0;
  switch (copies ? p.head_dim * (int)sizeof(Tin) : 0) {
    case 16 * 32: return launch_append(copy_append_kernel<16>, 4 * kThreads / 16, p, n_layers, st);
    case 8 * 32: return launch_append(copy_append_kernel<8>, 4 * kThreads / 8, p, n_layers, st);
    case 4 * 32: return launch_append(copy_append_kernel<4>, 4 * kThreads / 4, p, n_layers, st);
  }
  switch (pool_dtype) {
    case SNAPMIND_DTYPE_F32: return launch_append(chunk_append_kernel<Tin, float>, kThreads / 32, p, n_layers, st);
    case SNAPMIND_DTYPE_BF16: return launch_append(chunk_append_kernel<Tin, __nv_bfloat16>, kThreads / 32, p, n_layers, st);
    default: return launch_append(chunk_append_kernel<Tin, __half>, kThreads / 32, p, n_layers, st);
  }
}

}  // namespace
}  // namespace snapmind

using namespace snapmind;

extern "C" {

int snapmind_kv_append_chunk(void* k_pool, void* v_pool, void* scales, int pool_dtype, int64_t pool_layer_stride,
                             int64_t scale_layer_stride, const void* k_new, const void* v_new, int in_dtype,
                             int64_t in_stride_layer, int64_t in_stride_seq, int64_t in_stride_head,
                             int64_t in_stride_tok, const int32_t* block_tables, int64_t table_stride_seq,
                             int32_t table_width, const int32_t* slot_starts, int32_t slot_start0,
                             const int32_t* cu_new, int32_t n_layers, int32_t batch, int32_t n_tokens,
                             int32_t total_new, int32_t n_heads, int32_t head_dim, int32_t block_size,
                             int32_t num_blocks, int32_t* err_word, void* stream) {
  const int esz_in = dtype_size(in_dtype);
  const bool quant = pool_dtype == SNAPMIND_DTYPE_E4M3;
  const int esz = quant ? 1 : dtype_size(pool_dtype);
  SNAPMIND_CHECK_ARG(esz_in > 0 && esz > 0, "kv_append_chunk: unknown dtype");
  SNAPMIND_CHECK_ARG(n_layers >= 0 && n_layers <= 32767 && batch >= 0 && n_tokens >= 0 && total_new >= 0 &&
                         n_heads > 0 && head_dim > 0 && block_size > 0 && num_blocks > 0 && table_width >= 0,
                     "kv_append_chunk: bad sizes");
  SNAPMIND_CHECK_ARG(cu_new != nullptr || (int64_t)batch * n_tokens == total_new,
                     "kv_append_chunk: without cu_new total_new is batch * n_tokens");
  SNAPMIND_CHECK_ARG((int64_t)total_new * n_heads < (1LL << 31) && (int64_t)num_blocks * n_heads * block_size < (1LL << 31),
                     "kv_append_chunk: too many rows");
  SNAPMIND_CHECK_ARG(quant == (scales != nullptr), "kv_append_chunk: scales go with an e4m3 pool, and only with one");
  if (n_layers == 0 || batch == 0 || total_new == 0) return SNAPMIND_OK;
  SNAPMIND_CHECK_ARG(k_pool && v_pool && k_new && v_new && block_tables, "kv_append_chunk: null pointer");
  ChunkAppendParams p;
  p.pool[0] = static_cast<uint8_t*>(k_pool);
  p.pool[1] = static_cast<uint8_t*>(v_pool);
  p.scales = static_cast<uint8_t*>(scales);
  p.in[0] = static_cast<const char*>(k_new);
  p.in[1] = static_cast<const char*>(v_new);
  p.pool_layer_stride = pool_layer_stride * esz;
  p.scale_layer_stride = scale_layer_stride;
  p.in_stride_layer = in_stride_layer * esz_in;
  p.in_stride_seq = in_stride_seq * esz_in;
  p.in_stride_head = in_stride_head * esz_in;
  p.in_stride_tok = in_stride_tok * esz_in;
  p.tables = block_tables;
  p.table_stride = table_stride_seq;
  p.table_width = table_width;
  p.slot_starts = slot_starts;
  p.slot_start0 = slot_start0;
  p.cu = cu_new;
  p.batch = batch;
  p.n_tokens = n_tokens;
  p.total = total_new;
  p.n_heads = n_heads;
  p.head_dim = head_dim;
  p.block_size = block_size;
  p.num_blocks = num_blocks;
  // neighbouring teams walk the axis whose rows are neighbours in the input
  p.by_heads = FastDiv(n_heads);
  p.by_tokens = FastDiv(n_tokens > 0 ? n_tokens : 1);
  p.by_block = FastDiv(block_size);
  p.heads_inner = cu_new != nullptr || p.in_stride_head < p.in_stride_tok;
  p.err = err_word;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (in_dtype) {
    case SNAPMIND_DTYPE_F32:
      return quant ? launch_quant_append<float>(p, n_layers, st) : launch_plain_append<float>(p, in_dtype, pool_dtype, n_layers, st);
    case SNAPMIND_DTYPE_BF16:
      return quant ? launch_quant_append<__nv_bfloat16>(p, n_layers, st)
                   : launch_plain_append<__nv_bfloat16>(p, in_dtype, pool_dtype, n_layers, st);
    default:
      return quant ? launch_quant_append<__half>(p, n_layers, st)
                   : launch_plain_append<__half>(p, in_dtype, pool_dtype, n_layers, st);
  }
}

int snapmind_kv_gather_quant(const void* k_pool, const void* v_pool, const void* scales, int64_t pool_layer_stride,
                             int64_t scale_layer_stride, void* k_out, void* v_out, int out_dtype,
                             int64_t out_layer_stride, int64_t out_layer_capacity, const int32_t* block_tables,
                             int64_t table_stride_seq, int32_t table_width, const int32_t* seq_lens,
                             int32_t n_layers, int32_t batch, int32_t n_heads, int32_t head_dim, int32_t block_size,
                             int32_t num_blocks, int32_t* err_word, void* stream) {
  const int esz = dtype_size(out_dtype);
  SNAPMIND_CHECK_ARG(esz > 0, "kv_gather_quant: unknown dtype");
  SNAPMIND_CHECK_ARG(n_layers >= 0 && n_layers <= 65535 && batch >= 0 && batch <= 8192 && n_heads > 0 && head_dim > 0 &&
                         block_size > 0 && num_blocks > 0 && table_width >= 0 &&
                         (int64_t)2 * n_heads * head_dim * block_size < (1LL << 31),
                     "kv_gather_quant: bad sizes");
  if (n_layers == 0 || batch == 0) return SNAPMIND_OK;
  SNAPMIND_CHECK_ARG(k_pool && v_pool && scales && k_out && v_out && block_tables && seq_lens,
                     "kv_gather_quant: null pointer");
  QuantGatherParams p;
  p.pool[0] = static_cast<const uint8_t*>(k_pool);
  p.pool[1] = static_cast<const uint8_t*>(v_pool);
  p.scales = static_cast<const uint8_t*>(scales);
  p.out[0] = static_cast<char*>(k_out);
  p.out[1] = static_cast<char*>(v_out);
  p.pool_layer_stride = pool_layer_stride;
  p.scale_layer_stride = scale_layer_stride;
  p.out_layer_stride = out_layer_stride * esz;
  p.out_capacity = out_layer_capacity;
  p.tables = block_tables;
  p.table_stride = table_stride_seq;
  p.table_width = table_width;
  p.seq_lens = seq_lens;
  p.batch = batch;
  p.n_heads = n_heads;
  p.head_dim = head_dim;
  p.block_size = block_size;
  p.num_blocks = num_blocks;
  p.err = err_word;
  const bool vec = aligned16(k_pool) && aligned16(v_pool) && aligned16(k_out) && aligned16(v_out) &&
                   head_dim * esz % 16 == 0 && p.out_layer_stride % 16 == 0 && pool_layer_stride % 8 == 0;
  p.by_block = FastDiv(block_size);
  const size_t smem = 2 * sizeof(int32_t) * (size_t)(batch + 1);
  const int cap = (num_sms() * 8 + n_layers - 1) / n_layers;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const auto go = [&](auto kernel) -> int {
    if (smem > 48 * 1024) {
      cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
      if (e != cudaSuccess) return cuda_status(e, "kv_gather_quant smem attribute");
    }
    kernel<<<dim3(cap, n_layers), kThreads, smem, st>>>(p);
    return cuda_status(cudaGetLastError(), "kv_gather_quant launch");
  };
  const int team = vec && head_dim * esz % 32 == 0 ? head_dim * esz / 32 : 0;
  const auto by_team = [&](auto t) -> int {
    using T = decltype(t);
    switch (team) {
      case 4: return go(quant_gather_kernel<T, 4>);
      case 8: return go(quant_gather_kernel<T, 8>);
      case 16: return go(quant_gather_kernel<T, 16>);
      default: return go(quant_gather_kernel<T, 0>);
    }
  };
  switch (out_dtype) {
    case SNAPMIND_DTYPE_F32: return by_team(float());
    case SNAPMIND_DTYPE_BF16: return by_team(__nv_bfloat16());
    default: return by_team(__half());
  }
}

}  // extern "C"
