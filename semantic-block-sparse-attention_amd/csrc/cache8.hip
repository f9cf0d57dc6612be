// The 8-bit key/value cache of a dense layer: new rows quantised block by block, attention of
// the newest rows over the cache, and the tables of a cache without its least attended blocks.
//
// A block is 64 tokens of one (sequence, KV head).  Keys lie [64][D], values [D][64]:
// both are then the A operand of their product as they lie (S^T = K Q^T takes 8 dims of
// a key per lane, O^T = V^T P^T 8 keys of a dim), and nothing is transposed in the attention.
#include "sbsa_common.h"

namespace {

constexpr int KB = SBSA_CACHE8_BLOCK;
constexpr int BUFFER_CONFIG = 0x00020000;   // raw buffer resource, 32-bit data format
constexpr float LOG2E = 1.44269504088896340736f;
constexpr float FLT_MOST = 3.402823466e38f;
constexpr float LN2 = 0.69314718055994530942f;
typedef __attribute__((ext_vector_type(16))) float f32x16_t;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2_t;

__device__ __forceinline__ f16x8_t as_f16x8(u32x4_t v) {
  f16x8_t r;
  __builtin_memcpy(&r, &v, 16);
  return r;
}

__device__ __forceinline__ uint32_t pack2h(float a, float b) {
  const f16x2_t v = __builtin_convertvector(f32x2_t{a, b}, f16x2_t);
  uint32_t r;
  __builtin_memcpy(&r, &v, 4);
  return r;
}

// Four codes of a word as bf16 (exact: e4m3 has 4 significant bits, int8 7).
template <int FMT>
__device__ __forceinline__ void decode4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (FMT == SBSA_CACHE8_E4M3) {
    const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false);
    const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true);
    __builtin_memcpy(&lo, &a, 4);
    __builtin_memcpy(&hi, &b, 4);
  } else {
    lo = pack2bf((float)(int8_t)(w & 0xff), (float)(int8_t)((w >> 8) & 0xff));
    hi = pack2bf((float)(int8_t)((w >> 16) & 0xff), (float)(int8_t)(w >> 24));
  }
}

template <int FMT>
__device__ __forceinline__ bf16x8_t decode8(uint32_t w0, uint32_t w1) {
  u32x4_t r;
  uint32_t a, b, c, d;
  decode4<FMT>(w0, a, b);
  decode4<FMT>(w1, c, d);
  r.x = a; r.y = b; r.z = c; r.w = d;
  return as_bf16x8(r);
}

// Four codes of a word as fp16 (exact too).
template <int FMT>
__device__ __forceinline__ void decode4h(uint32_t w, uint32_t& lo, uint32_t& hi) {
  f16x2_t a, b;
  if constexpr (FMT == SBSA_CACHE8_E4M3) {
    a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false);
    b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true);
  } else {
    // code + 128 under the exponent of 1024 is the fp16 number 1152 + code
    const uint32_t u = w ^ 0x80808080u;
    const uint32_t x = __builtin_amdgcn_perm(0x64646464u, u, 0x07010700u);
    const uint32_t y = __builtin_amdgcn_perm(0x64646464u, u, 0x07030702u);
    const f16x2_t off = {(_Float16)1152.f, (_Float16)1152.f};
    __builtin_memcpy(&a, &x, 4);
    __builtin_memcpy(&b, &y, 4);
    a -= off;
    b -= off;
  }
  __builtin_memcpy(&lo, &a, 4);
  __builtin_memcpy(&hi, &b, 4);
}

template <int FMT>
__device__ __forceinline__ f16x8_t decode8h(uint32_t w0, uint32_t w1) {
  u32x4_t r;
  uint32_t a, b, c, d;
  decode4h<FMT>(w0, a, b);
  decode4h<FMT>(w1, c, d);
  r.x = a; r.y = b; r.z = c; r.w = d;
  return as_f16x8(r);
}

template <int FMT>
__device__ __forceinline__ float decode1(uint8_t c) {
  uint32_t lo, hi;
  decode4<FMT>((uint32_t)c, lo, hi);
  return bf2f((bf16_t)(lo & 0xffff));
}

// Two values to codes, rounded to the nearest (even).  |x| is at most the largest code, up to
// the rounding of x's division.
template <int FMT>
__device__ __forceinline__ uint32_t encode2(float x, float y) {
  if constexpr (FMT == SBSA_CACHE8_E4M3) {
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x, y, 0, false) & 0xffffu;
  } else {
    return ((uint32_t)(int)rintf(x) & 0xffu) | (((uint32_t)(int)rintf(y) & 0xffu) << 8);
  }
}

__device__ __forceinline__ int64_t place_of(const sbsa_cache8& c, int64_t sh, int block) {
  int t = c.table[sh * c.num_blocks + block];
  t = t < 0 ? 0 : t;
  return sh * c.num_blocks + (t < c.num_blocks ? t : c.num_blocks - 1);
}

__device__ __forceinline__ int held_of(const sbsa_cache8& c, int64_t sh) {
  const int len = c.lengths[sh], most = c.num_blocks * KB;
  return len < 0 ? 0 : (len < most ? len : most);
}

// Rows of sequence s: first and count, kept inside the call's tokens whatever offsets hold.
__device__ __forceinline__ void rows_of(const int32_t* offsets, int s, int64_t uniform, int64_t tokens, int64_t& first,
                                        int& n) {
  if (!offsets) {
    first = (int64_t)s * uniform;
    n = (int)uniform;
    return;
  }
  int64_t a = offsets[s], b = offsets[s + 1];
  a = a < 0 ? 0 : (a < tokens ? a : tokens);
  b = b < a ? a : (b < tokens ? b : tokens);
  first = a;
  n = (int)(b - a);
}

// ---- append ---------------------------------------------------------------------------

struct AppendArgs {
  sbsa_cache8 c;
  const bf16_t* k;
  const bf16_t* v;
  int64_t k_st, k_sh, v_st, v_sh;
  int64_t tokens, uniform;
  const int32_t* offsets;
  const int32_t* start;
};

// x / s to the nearest, for |x / s| of at least 2^-11 and s of at least 2^-90 (else only near: what is below rounds to
// code 0 all the same).  With inv = 1 / s to the nearest a faithful quotient corrected by its exact residual
// is the nearest one (Markstein); the first correction makes it faithful.  5 operations to the division's 10 and more.
__device__ __forceinline__ float quotient(float x, float s, float inv) {
  float q = x * inv;
  q = __builtin_fmaf(__builtin_fmaf(-q, s, x), inv, q);
  return __builtin_fmaf(__builtin_fmaf(-q, s, x), inv, q);
}

typedef __attribute__((ext_vector_type(2))) uint16_t u16x2_t;

// A block of the grid takes a block of 64 tokens (and every gridDim.x-th after it) of one
// (sequence, head): its rows into registers, the largest magnitudes of the keys and of the values over the block, the
// codes out.  A thread holds PASSES consecutive rows of 8 columns, so its codes of a key row are 8 bytes of it and
// those of a value column PASSES bytes of that; the values' turn through LDS only to leave in whole rows of
// [dim][64].  The last of a (sequence, head)'s grid blocks to end moves the length on, so that none reads a moved one.
template <int D, int FMT>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
  constexpr int CH = D / 8;             // 16-byte pieces of a row
  constexpr int PASSES = KB * CH / 256; // consecutive rows of a thread: 4 or 8
  constexpr int LD = KB + 16;           // bytes of a value column in LDS: 16-byte pieces stay aligned
  constexpr float CODE_MAX = FMT == SBSA_CACHE8_E4M3 ? 448.f : 127.f;
  const sbsa_cache8& c = a.c;
  const int h = blockIdx.y, s = blockIdx.z, tid = threadIdx.x;
  const int64_t sh = (int64_t)s * c.num_kv_heads + h;
  const int64_t heads = (int64_t)c.num_seqs * c.num_kv_heads;
  __shared__ int red[2][4];
  __shared__ __attribute__((aligned(16))) unsigned char turn[D * LD];
  __shared__ int s_last;

  int64_t row0;
  int n;
  rows_of(a.offsets, s, a.uniform, a.tokens, row0, n);
  const int held = held_of(c, sh);
  int start = a.start ? a.start[s] : held;
  start = start < 0 ? 0 : (start < held ? start : held);
  const int room = c.num_blocks * KB;
  const int open = c.open_block[sh];
  const int end = (int64_t)start + n > room ? room : start + n;
  if ((int64_t)start + n > room && tid == 0 && blockIdx.x == 0) *c.overflow = 1;
  // no rows, or no room for any: the sequence ends at start, and no block is touched
  const bool grows = end > start;
  const int first = start / KB, last = grows ? (end - 1) / KB : first - 1;

  const int col = (tid % CH) * 8, r0 = tid / CH * PASSES;
  const bf16_t* src[2] = {a.k + row0 * a.k_st + h * a.k_sh, a.v + row0 * a.v_st + h * a.v_sh};
  const int64_t st[2] = {a.k_st, a.v_st};
  bf16_t* const tail = (bf16_t*)c.tail + sh * KB * D;
  const int64_t tail_v = heads * KB * D, scale_v = heads * c.num_blocks;
  for (int b = first + (int)blockIdx.x; b <= last; b += (int)gridDim.x) {
    const int64_t place = place_of(c, sh, b);
    uint8_t* const codes[2] = {(uint8_t*)c.codes_k + place * KB * D, (uint8_t*)c.codes_v + place * KB * D};
    u32x4_t x[2][PASSES];
    const bool fresh = b * KB >= start && (b + 1) * KB <= end;     // the block is new rows throughout
    if (fresh) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int p = 0; p < PASSES; ++p)
          x[t][p] = *reinterpret_cast<const u32x4_t*>(src[t] + (int64_t)(b * KB + r0 + p - start) * st[t] + col);
    } else {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
          const int j = r0 + p, pos = b * KB + j;
          u32x4_t w = {0u, 0u, 0u, 0u};
          if (pos >= start && pos < end) {
            w = *reinterpret_cast<const u32x4_t*>(src[t] + (int64_t)(pos - start) * st[t] + col);
          } else if (pos < start && open == b) {
            w = *reinterpret_cast<const u32x4_t*>(tail + t * tail_v + j * D + col);
          } else if (pos < start) {
            // the row is there in its codes alone
            const float old = c.scales[t * scale_v + place];
            bf16_t y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
              y[i] = f2bf(decode1<FMT>(codes[t][t ? (col + i) * KB + j : j * D + col + i]) * old);
            __builtin_memcpy(&w, y, 16);
          }
          x[t][p] = w;
        }
    }
    // the largest magnitudes, as bf16 bits without the sign: those that are not finite are 0x7f80 and up
    float scale[2];
    bool fine[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      u16x2_t most = {0, 0};
#pragma unroll
      for (int p = 0; p < PASSES; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t w = x[t][p][i] & 0x7fff7fffu;
          u16x2_t v;
          __builtin_memcpy(&v, &w, 4);
          most = __builtin_elementwise_max(most, v);
        }
      int m = most.x > most.y ? most.x : most.y;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) m = max(m, __shfl_xor(m, o, 64));
      if ((tid & 63) == 0) red[t][tid >> 6] = m;
    }
    __syncthreads();                    // and every row is read before a code or the tail is written
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int m = max(max(red[t][0], red[t][1]), max(red[t][2], red[t][3]));
      fine[t] = m < 0x7f80;
      scale[t] = fine[t] ? fmaxf(bf2f((bf16_t)m) / CODE_MAX, 0x1p-126f) : __uint_as_float(0x7fc00000u);
      if (tid == 0) c.scales[t * scale_v + place] = scale[t];
    }
    const bool easy = scale[0] >= 0x1p-90f && scale[1] >= 0x1p-90f;      // (no, where one is NaN)
    const float inv[2] = {1.f / scale[0], 1.f / scale[1]};
    auto value = [&](int t, int p, int i) {
      const uint32_t w = x[t][p][i >> 1];
      const float v = bf2f((bf16_t)(i & 1 ? w >> 16 : w & 0xffffu));
      return easy ? quotient(v, scale[t], inv[t]) : v / scale[t];
    };
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      uint32_t w[2] = {0u, 0u};
      if (fine[0]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i >> 1] |= encode2<FMT>(value(0, p, 2 * i), value(0, p, 2 * i + 1)) << (16 * (i & 1));
      }
      u32x2_t o;
      o.x = w[0]; o.y = w[1];
      *reinterpret_cast<u32x2_t*>(codes[0] + (r0 + p) * D + col) = o;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t w[PASSES / 4];
#pragma unroll
      for (int x4 = 0; x4 < PASSES / 4; ++x4)
        w[x4] = fine[1] ? encode2<FMT>(value(1, 4 * x4, i), value(1, 4 * x4 + 1, i)) |
                              encode2<FMT>(value(1, 4 * x4 + 2, i), value(1, 4 * x4 + 3, i)) << 16
                        : 0u;
      __builtin_memcpy(turn + (col + i) * LD + r0, w, PASSES);
    }
    if (b == last && first == last) {
      // the rows are kept: those that were the tail's already are there
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
          const int pos = b * KB + r0 + p;
          if (pos < end && (pos >= start || open != b))
            *reinterpret_cast<u32x4_t*>(tail + t * tail_v + (r0 + p) * D + col) = x[t][p];
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = tid; i < D * (KB / 16); i += 256)
      *reinterpret_cast<u32x4_t*>(codes[1] + i * 16) = *reinterpret_cast<const u32x4_t*>(turn + (i / 4) * LD + (i % 4) * 16);
    if (b * KB >= start && tid == 0) c.weights[sh * c.num_blocks + b] = 0.f;
    __syncthreads();                    // LDS is used again
  }

  if (gridDim.x > 1) {
    if (tid == 0) {
      __threadfence();
      s_last = atomicAdd(&c.counters[sh], 1) == (int)gridDim.x - 1;
    }
    __syncthreads();
    if (!s_last) return;
    if (tid == 0) c.counters[sh] = 0;
    // the last block's rows are kept: all of them are new where it is not the first
    for (int t = 0; t < 2 && last > first; ++t)
      for (int j = r0; j < r0 + PASSES && last * KB + j < end; ++j)
        *reinterpret_cast<u32x4_t*>(tail + t * tail_v + j * D + col) =
            *reinterpret_cast<const u32x4_t*>(src[t] + (int64_t)(last * KB + j - start) * st[t] + col);
  }
  if (tid == 0) {
    c.lengths[sh] = end;
    if (grows) c.open_block[sh] = last;
  }
}

// ---- attention --------------------------------------------------------------------------

struct AttendArgs {
  sbsa_cache8 c;
  const bf16_t* q;
  int64_t q_st, q_sh;
  bf16_t* out;
  int64_t o_st, o_sh;
  float* lse;                  // [tokens, Hq], natural
  float* part_o;               // [splits][tokens * Hq][D]
  // Sums of exponentials are kept as (m, l), 2^m l: the logarithm of one would round a weight by 10^-6
  f32x2_t* part_ml;            // [splits][tokens * Hq]
  f32x2_t* row_ml;             // [tokens * Hq], with 1 / l (accumulating)
  f32x2_t* part_w;             // [tokens * Hq][N]: each block's sum of a row (few rows, accumulating)
  const int32_t* offsets;
  int64_t tokens, uniform;
  int hq, g, splits, tile_queries, tiles_per_seq;
  float scale_log2;            // sm_scale * log2(e)
};

// The row tile of this block of the grid: sequence, its rows, and the tile's first query.  With
// offsets the tiles are counted along the sequences, 64 of them at a time; false: no tile is left.
__device__ __forceinline__ bool tile_of(const AttendArgs& a, int64_t t, int& s, int64_t& row0, int& n, int& q0) {
  if (!a.offsets) {
    s = (int)(t / a.tiles_per_seq);
    rows_of(nullptr, s, a.uniform, a.tokens, row0, n);
    q0 = (int)(t % a.tiles_per_seq) * a.tile_queries;
    return true;
  }
  const int lane = threadIdx.x & 63;
  int64_t before = 0;
  for (int s0 = 0; s0 < a.c.num_seqs; s0 += 64) {
    int64_t r = 0;
    int m = 0;
    if (s0 + lane < a.c.num_seqs) rows_of(a.offsets, s0 + lane, 0, a.tokens, r, m);
    const int mine = (m + a.tile_queries - 1) / a.tile_queries;
    const int upto = wave_incl_scan(mine);
    const unsigned long long past = __ballot(before + upto > t);
    if (past) {
      const int l = __builtin_amdgcn_readfirstlane(__ffsll((long long)past) - 1);
      s = s0 + l;
      rows_of(a.offsets, s, 0, a.tokens, row0, n);
      const int upto_l = __builtin_amdgcn_readlane(upto, l), mine_l = __builtin_amdgcn_readlane(mine, l);
      q0 = (int)(t - before - (upto_l - mine_l)) * a.tile_queries;
      return true;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

// 16 codes, those from `keep` on as 0: what lies behind a sequence's last token may be any bits
__device__ __forceinline__ u32x4_t clear_past(u32x4_t w, int keep) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int k = keep - 4 * i;
    w[i] = k >= 4 ? w[i] : (k <= 0 ? 0u : w[i] & ((1u << (8 * k)) - 1u));
  }
  return w;
}

__device__ __forceinline__ void finish_row(const AttendArgs& a, int64_t row, float m, float l) {
  if (a.lse) a.lse[row] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * LN2;
  if (a.row_ml) a.row_ml[row] = f32x2_t{m, l == 0.f ? 0.f : 1.f / l};
}

// A wave's state over R = 16 or 32 rows (columns of S^T and O^T).  Lane l holds row l % R, and of
// a block's 64 keys those of its part l / R: 16 or 32 consecutive ones, because the K rows
// are handed to the product in the order that leaves them so.  They are the B operand of
// O^T = V^T P^T as they lie, so the probabilities never leave the lane.
//
// P times the values' scale is rounded to fp16 (2^-11; bf16 would double the result's error).  For
// fp16's range the scale is taken relative to the largest so far (v_ref) and times 2^11: with the reference
// maximum at most 2^4 below the true one a probability is at most 2^15, and keeps its 11 bits down to 2^-25 of
// the largest block's.
template <int D, int FMT, int R>
struct WaveRows {
  static constexpr int PARTS = 64 / R;          // lanes that share a row
  static constexpr int MINE = KB / PARTS;       // a lane's keys of a block
  static constexpr int GROUPS = KB / R;         // products of R keys
  static constexpr int SEG = 16 * PARTS;        // dims that one 16-byte load of every part covers
  static constexpr int NT = D / R;              // R-dim tiles of O^T
  static constexpr int NI = R * R / 64;         // accumulator values of a lane
  static constexpr float P_SCALE = 0x1p11f, SLACK = 4.f;
  typedef __attribute__((ext_vector_type(NI))) float acc_t;
  typedef u32x4_t kcodes_t[GROUPS][D / SEG];
  typedef u32x4_t vcodes_t[NT][MINE / 16];

  acc_t o[NT];
  float m, l;
  float v_ref;

  static __device__ __forceinline__ acc_t mfma(bf16x8_t x, bf16x8_t y, acc_t z) {
    if constexpr (R == 16)
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, z, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, z, 0, 0, 0);
  }
  static __device__ __forceinline__ acc_t mfma(f16x8_t x, f16x8_t y, acc_t z) {
    if constexpr (R == 16)
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, z, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, z, 0, 0, 0);
  }

  __device__ __forceinline__ void start() {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < NI; ++i) o[t][i] = 0.f;
    m = -INFINITY;
    l = 0.f;
    v_ref = 0.f;
  }

  // piece x (of 2) of 16-byte step j of a row, for the lane's part; zeros without a row
  static __device__ __forceinline__ u32x4_t query_piece(const bf16_t* qrow, int j, int x, int lane) {
    const u32x4_t zero = {0u, 0u, 0u, 0u};
    return qrow ? *reinterpret_cast<const u32x4_t*>(qrow + j * SEG + (lane / R) * 16 + x * 8) : zero;
  }

  // the key (of a block's 64) that row r of product g takes
  static __device__ __forceinline__ int key_of(int r, int g) {
    if constexpr (R == 16)
      return (r >> 2) * 16 + g * 4 + (r & 3);
    else
      return ((r >> 2) & 1) * 32 + g * 16 + (r >> 3) * 4 + (r & 3);
  }

  // A block's codes through a buffer resource of its size: the address of a load is a scalar base, one lane
  // offset and a scalar or literal one.  (By pointers the compiler carries 64-bit lane addresses and spills.)
  static __device__ __forceinline__ void load_k(const uint8_t* kb, int lane, kcodes_t& kc) {
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)kb, 0, KB * D, BUFFER_CONFIG);
    const int off = key_of(lane % R, 0) * D + (lane / R) * 16;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
#pragma unroll
      for (int j = 0; j < D / SEG; ++j)
        kc[g][j] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, off + j * SEG, key_of(0, g) * D, 0);
  }
  static __device__ __forceinline__ void load_v(const uint8_t* vb, int lane, vcodes_t& vc) {
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)vb, 0, KB * D, BUFFER_CONFIG);
    const int off = (lane % R) * KB + (lane / R) * MINE;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int x = 0; x < MINE / 16; ++x)
        vc[t][x] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, off + x * 16, t * R * KB, 0);
  }

  // scores of a block's keys, times ks; q(j, x) gives the rows' pieces
  template <class Q>
  static __device__ __forceinline__ void scores(const kcodes_t& kc, Q&& q, float ks, acc_t (&sc)[GROUPS]) {
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
#pragma unroll
      for (int i = 0; i < NI; ++i) sc[g][i] = 0.f;
#pragma unroll
    for (int j = 0; j < D / SEG; ++j)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const bf16x8_t qq = as_bf16x8(q(j, x));
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
          u32x4_t w = kc[g][j];
          asm volatile("" : "+v"(w));           // decoded here, not where it was loaded
          sc[g] = mfma(x ? decode8<FMT>(w.z, w.w) : decode8<FMT>(w.x, w.y), qq, sc[g]);
        }
        // without these the compiler decodes far ahead and runs out of registers
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
#pragma unroll
      for (int i = 0; i < NI; ++i) sc[g][i] *= ks;
  }

  // a block's scores to probabilities p (fp16, with the values' scale), the state moved on.  seen: how
  // many of its keys the lane's row sees (all: every row every one).  Returns the lane's sum.
  __device__ __forceinline__ float softmax(acc_t (&sc)[GROUPS], float vs, int seen, bool all, int lane,
                                           u32x4_t (&p)[MINE / 8]) {
    const int part = lane / R;
    if (!all) {
#pragma unroll
      for (int g = 0; g < GROUPS; ++g)
#pragma unroll
        for (int i = 0; i < NI; ++i)
          if (part * MINE + g * NI + i >= seen) sc[g][i] = -INFINITY;
    }
    float top = -INFINITY;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
#pragma unroll
      for (int i = 0; i < NI; ++i) top = fmaxf(top, sc[g][i]);
    if constexpr (R == 16) top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    // the reference maximum moves only when a row has gone 2^SLACK above it, the reference
    // scale when a block's is larger
    if (__ballot(top > m + SLACK || fabsf(vs) > v_ref)) {
      // a score past fp32's range counts as its largest number (infinities would leave NaN)
      if (__ballot(top == INFINITY)) {
#pragma unroll
        for (int g = 0; g < GROUPS; ++g)
#pragma unroll
          for (int i = 0; i < NI; ++i) sc[g][i] = sc[g][i] == INFINITY ? FLT_MOST : sc[g][i];
        top = top == INFINITY ? FLT_MOST : top;
      }
      const float to = fmaxf(m, top);
      float f = m == to ? 1.f : __builtin_amdgcn_exp2f(m - to);
      l *= f;
      m = to;
      if (fabsf(vs) > v_ref) {
        f *= v_ref / fabsf(vs);
        v_ref = fabsf(vs);
      }
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < NI; ++i) o[t][i] *= f;
    }
    const float ref = m == -INFINITY ? 0.f : m;
    const float pv = v_ref > 0.f ? vs / v_ref * P_SCALE : vs * 0.f;       // a NaN scale stays one
    float sum = 0.f;
#pragma unroll
    for (int x = 0; x < MINE / 2; ++x) {
      const int i0 = 2 * x, i1 = 2 * x + 1;
      const float p0 = __builtin_amdgcn_exp2f(sc[i0 / NI][i0 % NI] - ref);
      const float p1 = __builtin_amdgcn_exp2f(sc[i1 / NI][i1 % NI] - ref);
      sum += p0 + p1;
      // an unseen key's product is 0 whatever the scale
      const bool h0 = !all && part * MINE + i0 >= seen, h1 = !all && part * MINE + i1 >= seen;
      p[x / 4][x % 4] = pack2h(h0 ? 0.f : p0 * pv, h1 ? 0.f : p1 * pv);
    }
    l += sum;
    return sum;
  }

  // filled: how many of the block's keys are there
  __device__ __forceinline__ void values(vcodes_t& vc, const u32x4_t (&p)[MINE / 8], int filled, int lane) {
    if (filled < KB) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int x = 0; x < MINE / 16; ++x) vc[t][x] = clear_past(vc[t][x], filled - ((lane / R) * MINE + x * 16));
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int x = 0; x < MINE / 16; ++x) {
        u32x4_t w = vc[t][x];
        asm volatile("" : "+v"(w));
        o[t] = mfma(decode8h<FMT>(w.x, w.y), as_f16x8(p[2 * x]), o[t]);
        o[t] = mfma(decode8h<FMT>(w.z, w.w), as_f16x8(p[2 * x + 1]), o[t]);
        __builtin_amdgcn_sched_barrier(0);
      }
  }

  // the row's sum over its lanes, and O as the wave's own result (normalised before it gets the values'
  // unit back, or a sum of large values would pass fp32's range).  A row without keys has sum 0 and gives 0; a NaN stays one.
  __device__ __forceinline__ void total() {
    if constexpr (R == 16) l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    const float f = l == 0.f ? 0.f : 1.f / P_SCALE / l;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < NI; ++i) o[t][i] = o[t][i] * f * v_ref;
  }

  // four consecutive dims of the lane's row: tile t, quarter x of the accumulator
  static __device__ __forceinline__ int dim_of(int t, int x, int lane) { return t * R + 8 * x + 4 * (lane / R); }

  // where a row's result goes: out, or its share's partial row
  static __device__ __forceinline__ void store(const AttendArgs& a, int split, int64_t token, int head, int t, int x,
                                               int lane, f32x4_t v) {
    if (a.splits == 1) {
      u32x2_t w;
      w.x = pack2bf(v.x, v.y);
      w.y = pack2bf(v.z, v.w);
      *reinterpret_cast<u32x2_t*>(a.out + token * a.o_st + head * a.o_sh + dim_of(t, x, lane)) = w;
    } else {
      const int64_t row = (split * a.tokens + token) * a.hq + head;
      *reinterpret_cast<f32x4_t*>(a.part_o + row * D + dim_of(t, x, lane)) = v;
    }
  }
  // m, l: a row without keys has l = 0
  static __device__ __forceinline__ void store_sum(const AttendArgs& a, int split, int64_t token, int head, float m, float l) {
    const int64_t row = token * a.hq + head;
    if (a.splits > 1)
      a.part_ml[split * a.tokens * a.hq + row] = f32x2_t{m, l};
    else
      finish_row(a, row, m, l);
  }
};

// This lane's row of a tile, what it sees, and the tile's share of the blocks.
template <int R>
struct LaneRow {
  int qi, head, vis, vis_most, vis_least, lo, hi, held;
  bool there;
  int64_t sh;

  __device__ __forceinline__ void find(const AttendArgs& a, int s, int h, int n, int q0, int r, int split) {
    sh = (int64_t)s * a.c.num_kv_heads + h;
    held = __builtin_amdgcn_readfirstlane(held_of(a.c, sh));
    qi = q0 + r / a.g;
    head = h * a.g + r % a.g;
    there = r < a.tile_queries * a.g && qi < n;
    vis = there ? held - n + qi + 1 : 0;
    vis = vis < 0 ? 0 : vis;
    vis_most = vis;
    vis_least = there ? vis : 0x7fffffff;
#pragma unroll
    for (int x = 1; x < R; x <<= 1) {
      vis_most = max(vis_most, __shfl_xor(vis_most, x, 64));
      vis_least = min(vis_least, __shfl_xor(vis_least, x, 64));
    }
    vis_most = __builtin_amdgcn_readfirstlane(vis_most);
    vis_least = __builtin_amdgcn_readfirstlane(vis_least);
    // the share: of the blocks that the tile's last row sees
    const int tile_last = q0 + a.tile_queries < n ? q0 + a.tile_queries : n;
    const int tile_vis = held - n + tile_last;
    const int blocks = tile_vis > 0 ? (tile_vis + KB - 1) / KB : 0;
    const int per = (blocks + a.splits - 1) / a.splits;
    lo = split * per;
    hi = lo + per < blocks ? lo + per : blocks;
  }
};

// Few rows per sequence: a tile of R rows over one share of the keys, every fourth block of keys to each
// wave, the waves joined through LDS.  The codes go from memory to the registers that the products read,
// the next block's on their way while this one's are used; no barrier and no LDS traffic but the queries'.
template <int D, int FMT, int R>
__global__ __launch_bounds__(256, R == 32 && D == 256 ? 1 : 2) void attend_keys_kernel(AttendArgs a) {
  using W = WaveRows<D, FMT, R>;
  constexpr int TILE = W::NT * W::NI * 64;          // floats of a wave's O
  constexpr int PIECES = D / W::SEG * 2;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem_keys[];
  float* fold = reinterpret_cast<float*>(smem_keys);
  __shared__ u32x4_t sq[PIECES * 64];
  __shared__ float sm[4 * 64], sl[4 * 64];
  const sbsa_cache8& c = a.c;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int split = (int)(blockIdx.x % a.splits);
  const int64_t tiles = gridDim.x / a.splits;
  int s, n, q0;
  int64_t row0;
  if (!tile_of(a, tiles - 1 - blockIdx.x / a.splits, s, row0, n, q0)) return;
  LaneRow<R> r;
  r.find(a, s, (int)blockIdx.y, n, q0, lane % R, split);
  const int64_t token = row0 + r.qi;
  const bf16_t* qrow = r.there ? a.q + token * a.q_st + r.head * a.q_sh : nullptr;
  for (int i = wave; i < PIECES; i += 4) sq[i * 64 + lane] = W::query_piece(qrow, i >> 1, i & 1, lane);

  W w;
  w.start();
  const int64_t heads = (int64_t)c.num_seqs * c.num_kv_heads;
  const int64_t base = r.sh * c.num_blocks;
  const uint8_t* codes_k = (const uint8_t*)c.codes_k + base * KB * D;
  const uint8_t* codes_v = (const uint8_t*)c.codes_v + base * KB * D;
  const int first = r.lo + wave;
  const int count = r.hi > first ? (r.hi - first + 3) / 4 : 0;
  // the places and scales of the wave's next 64 blocks, one per lane
  int place = 0;
  float ks = 0.f, vs = 0.f;
  auto fetch = [&](int i0) {
    const int b = first + 4 * (i0 + lane);
    place = 0;
    if (b < r.hi) {
      place = (int)(place_of(c, r.sh, b) - base);
      ks = c.scales[base + place] * a.scale_log2;
      vs = c.scales[heads * c.num_blocks + base + place];
    }
  };
  typename W::kcodes_t kc;
  typename W::vcodes_t vc;
  if (count > 0) {
    fetch(0);
    const int64_t at = (int64_t)__builtin_amdgcn_readlane(place, 0) * (KB * D);
    W::load_k(codes_k + at, lane, kc);
    W::load_v(codes_v + at, lane, vc);
  }
  __syncthreads();                                  // the queries are in LDS
  for (int i = 0; i < count; ++i) {
    const int b = first + 4 * i;
    const float ksi = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(ks), i & 63));
    const float vsi = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(vs), i & 63));
    if (((i + 1) & 63) == 0) fetch(i + 1);
    const int64_t at = (int64_t)__builtin_amdgcn_readlane(place, (i + 1) & 63) * (KB * D);
    typename W::acc_t sc[W::GROUPS];
    W::scores(kc, [&](int j, int x) { return sq[(2 * j + x) * 64 + lane]; }, ksi, sc);
    if (i + 1 < count) W::load_k(codes_k + at, lane, kc);
    u32x4_t p[W::MINE / 8];
    float sum = w.softmax(sc, vsi, r.vis - b * KB, (b + 1) * KB <= r.vis_least, lane, p);
    if (a.part_w) {
      // the block's share of each row's attention, for the blocks' weights
      if constexpr (R == 16) sum += __shfl_xor(sum, 16, 64);
      sum += __shfl_xor(sum, 32, 64);
      if (r.there && lane < R)
        a.part_w[(token * a.hq + r.head) * c.num_blocks + b] = f32x2_t{w.m, sum};
    }
    w.values(vc, p, r.held - b * KB, lane);
    if (i + 1 < count) W::load_v(codes_v + at, lane, vc);
    asm volatile("" ::: "memory");                  // the queries stay in LDS, not in registers
  }
  w.total();
#pragma unroll
  for (int t = 0; t < W::NT; ++t)
#pragma unroll
    for (int i = 0; i < W::NI; ++i) fold[wave * TILE + (t * W::NI + i) * 64 + lane] = w.o[t][i];
  sm[wave * 64 + lane] = w.m;
  sl[wave * 64 + lane] = w.l;
  __syncthreads();
  // each wave joins a quarter of the dims
  float top = -INFINITY, f[4], total = 0.f;
#pragma unroll
  for (int x = 0; x < 4; ++x) top = fmaxf(top, sm[x * 64 + lane]);
  const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    f[x] = sl[x * 64 + lane] * __builtin_amdgcn_exp2f(sm[x * 64 + lane] - ref);
    total += f[x];
  }
  if (!r.there) return;
  const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
  for (int x = 0; x < 4; ++x) f[x] *= inv;
  constexpr int OWN = W::NT / 4;
#pragma unroll
  for (int tt = 0; tt < OWN; ++tt) {
    const int t = wave * OWN + tt;
#pragma unroll
    for (int q = 0; q < W::NI / 4; ++q) {
      f32x4_t v;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = (t * W::NI + 4 * q + i) * 64 + lane;
        v[i] = (fold[at] * f[0] + fold[TILE + at] * f[1]) + (fold[2 * TILE + at] * f[2] + fold[3 * TILE + at] * f[3]);
      }
      W::store(a, split, token, r.head, t, q, lane, v);
    }
  }
  if (wave == 0 && lane < R) W::store_sum(a, split, token, r.head, top, total);
}

// Many rows: 32 of them to each wave, over one share of the keys.
template <int D, int FMT>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void attend_rows_kernel(AttendArgs a) {
  using W = WaveRows<D, FMT, 32>;
  const sbsa_cache8& c = a.c;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int split = (int)(blockIdx.x % a.splits);
  const int64_t tiles = gridDim.x / a.splits;
  int s, n, q0;
  int64_t row0;
  // late tiles see the most keys: they go first
  if (!tile_of(a, tiles - 1 - blockIdx.x / a.splits, s, row0, n, q0)) return;
  LaneRow<32> r;
  r.find(a, s, (int)blockIdx.y, n, q0, wave * 32 + lane % 32, split);
  const int64_t token = row0 + r.qi;
  const bf16_t* qrow = r.there ? a.q + token * a.q_st + r.head * a.q_sh : nullptr;
  u32x4_t q[D / W::SEG][2];
#pragma unroll
  for (int j = 0; j < D / W::SEG; ++j)
#pragma unroll
    for (int x = 0; x < 2; ++x) q[j][x] = W::query_piece(qrow, j, x, lane);
  W w;
  w.start();
  const int64_t heads = (int64_t)c.num_seqs * c.num_kv_heads;
  const int hi = min(r.hi, (r.vis_most + KB - 1) / KB);
  for (int b = r.lo; b < hi; ++b) {
    const int64_t place = place_of(c, r.sh, b);
    typename W::kcodes_t kc;
    typename W::vcodes_t vc;
    W::load_k((const uint8_t*)c.codes_k + place * (KB * D), lane, kc);
    W::load_v((const uint8_t*)c.codes_v + place * (KB * D), lane, vc);
    typename W::acc_t sc[W::GROUPS];
    W::scores(kc, [&](int j, int x) { return q[j][x]; }, c.scales[place] * a.scale_log2, sc);
    u32x4_t p[W::MINE / 8];
    w.softmax(sc, c.scales[heads * c.num_blocks + place], r.vis - b * KB, (b + 1) * KB <= r.vis_least, lane, p);
    w.values(vc, p, r.held - b * KB, lane);
  }
  w.total();
  if (!r.there) return;
#pragma unroll
  for (int t = 0; t < W::NT; ++t)
#pragma unroll
    for (int x = 0; x < W::NI / 4; ++x) {
      f32x4_t v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = w.o[t][4 * x + i];
      W::store(a, split, token, r.head, t, x, lane, v);
    }
  if (lane < 32) W::store_sum(a, split, token, r.head, w.m, w.l);
}

// The shares of a row joined: a grid block takes 64 dims of a row, 16 threads to a share's 64 dims and every
// 16th share to each.
template <int D>
__global__ __launch_bounds__(256) void join_kernel(AttendArgs a) {
  const int64_t row = blockIdx.x, rows = a.tokens * a.hq;
  const int lane = threadIdx.x & 63;
  const int64_t token = row / a.hq;
  const int head = (int)(row % a.hq);
  if (a.offsets && (token < a.offsets[0] || token >= a.offsets[a.c.num_seqs])) return;
  __shared__ f32x4_t fold[16 * 16];
  const f32x2_t* ml = a.part_ml + row;
  float top = -INFINITY;
  for (int x = lane; x < a.splits; x += 64) top = fmaxf(top, ml[x * rows].x);
  top = wave_max(top);
  const float ref = top == -INFINITY ? 0.f : top;
  float total = 0.f;
  for (int x = lane; x < a.splits; x += 64) {
    const f32x2_t v = ml[x * rows];
    total += v.y * __builtin_amdgcn_exp2f(v.x - ref);
  }
  total = wave_sum(total);
  const float inv = total == 0.f ? 0.f : 1.f / total;
  const int d = (int)blockIdx.y * 64 + (threadIdx.x & 15) * 4;
  f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int x = threadIdx.x >> 4; x < a.splits; x += 16) {
    const f32x2_t v = ml[x * rows];
    const f32x4_t o = *reinterpret_cast<const f32x4_t*>(a.part_o + (x * rows + row) * D + d);
    acc += o * (v.y * __builtin_amdgcn_exp2f(v.x - ref) * inv);      // a share without keys has an O of 0
  }
  fold[threadIdx.x] = acc;
  __syncthreads();
  if (threadIdx.x >= 16) return;
  f32x4_t sum = fold[threadIdx.x];
  for (int x = 1; x < 16; ++x) sum += fold[x * 16 + threadIdx.x];
  u32x2_t w;
  w.x = pack2bf(sum.x, sum.y);
  w.y = pack2bf(sum.z, sum.w);
  *reinterpret_cast<u32x2_t*>(a.out + token * a.o_st + head * a.o_sh + d) = w;
  if (threadIdx.x == 0 && blockIdx.y == 0) finish_row(a, row, top, total);
}

// The blocks' weights from the shares that few rows left block by block: a thread per block.
__global__ __launch_bounds__(256) void weigh_shares_kernel(AttendArgs a) {
  const sbsa_cache8& c = a.c;
  const int b = (int)(blockIdx.x * 256 + threadIdx.x), h = blockIdx.y, s = blockIdx.z;
  const int64_t sh = (int64_t)s * c.num_kv_heads + h;
  int64_t row0;
  int n;
  rows_of(a.offsets, s, a.uniform, a.tokens, row0, n);
  const int held = held_of(c, sh);
  if (n == 0 || b * KB >= held) return;
  float sum = 0.f;
  int qi = b * KB - (held - n);                      // the first row that sees the block
  for (qi = qi < 0 ? 0 : qi; qi < n; ++qi)
    for (int j = 0; j < a.g; ++j) {
      const int64_t row = (row0 + qi) * a.hq + h * a.g + j;
      const f32x2_t w = a.part_w[row * c.num_blocks + b], all = a.row_ml[row];
      sum += w.y == 0.f ? 0.f : w.y * __builtin_amdgcn_exp2f(w.x - all.x) * all.y;
    }
  c.weights[sh * c.num_blocks + b] += sum;
}

// The attention that each block receives: a wave holds a block of keys and goes over the rows that
// see it, their sums known (lse); one addition per block, so no order of atomics enters.
template <int D, int FMT>
__global__ __launch_bounds__(256) void weigh_kernel(AttendArgs a) {
  using W = WaveRows<D, FMT, 32>;
  const sbsa_cache8& c = a.c;
  const int lane = threadIdx.x & 63;
  const int b = (int)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int h = blockIdx.y, s = blockIdx.z;
  const int64_t sh = (int64_t)s * c.num_kv_heads + h;
  int64_t row0;
  int n;
  rows_of(a.offsets, s, a.uniform, a.tokens, row0, n);
  const int held = held_of(c, sh);
  if (n == 0 || b * KB >= held) return;
  const int64_t place = place_of(c, sh, b);
  typename W::kcodes_t kc;
  W::load_k((const uint8_t*)c.codes_k + place * (KB * D), lane, kc);
  const float ks = c.scales[place] * a.scale_log2;
  // the first row that sees the block's first key
  int first = b * KB - (held - n);
  first = first < 0 ? 0 : first;
  float sum = 0.f;
  for (int64_t r0 = (int64_t)first * a.g; r0 < (int64_t)n * a.g; r0 += 32) {
    const int64_t r = r0 + lane % 32;
    const bool there = r < (int64_t)n * a.g;
    const int64_t qi = there ? r / a.g : 0;
    const int head = h * a.g + (int)(r % a.g);
    const int seen = there ? (int)(held - n + qi + 1 - b * KB) : 0;
    const bf16_t* qrow = there ? a.q + (row0 + qi) * a.q_st + head * a.q_sh : nullptr;
    const f32x2_t none = {0.f, 0.f};
    const f32x2_t all = there ? a.row_ml[(row0 + qi) * a.hq + head] : none;
    typename W::acc_t sc[W::GROUPS];
    W::scores(kc, [&](int j, int x) { return W::query_piece(qrow, j, x, lane); }, ks, sc);
#pragma unroll
    for (int g = 0; g < W::GROUPS; ++g)
#pragma unroll
      for (int i = 0; i < W::NI; ++i)
        sum += (lane / 32) * W::MINE + g * W::NI + i < seen ? __builtin_amdgcn_exp2f(fminf(sc[g][i], FLT_MOST) - all.x) * all.y : 0.f;
  }
  sum = wave_sum(sum);
  if (lane == 0) c.weights[sh * c.num_blocks + b] += sum;
}

// ---- eviction ---------------------------------------------------------------------------

struct EvictArgs {
  const int32_t* table;
  const float* weights;
  const int32_t* lengths;
  const int32_t* open_block;
  int32_t* table_out;
  float* weights_out;
  int32_t* lengths_out;
  int32_t* open_out;
  int num_blocks, keep, sink, recent;
};

constexpr int EVICT_THREADS = 1024;

// One (sequence, head): tables into LDS whole (the outputs may be the inputs); the weight of the last block that
// stays by three histograms over its bits (not negative, so their order is that of the numbers), 11, 11
// and 9 of them; then each wave counts its run of blocks, and writes it in order behind those before.
__global__ __launch_bounds__(EVICT_THREADS) void evict_kernel(EvictArgs a) {
  constexpr int BINS = 2048, WAVES = EVICT_THREADS / 64;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem_evict[];
  int32_t* tab = reinterpret_cast<int32_t*>(smem_evict);
  uint32_t* bits = reinterpret_cast<uint32_t*>(tab + a.num_blocks);
  __shared__ int hist[BINS];
  __shared__ int part[WAVES], part_eq[WAVES];
  __shared__ int s_bin[2];
  const int64_t sh = blockIdx.x, base = sh * a.num_blocks;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int room = a.num_blocks;
  int len = a.lengths[sh];
  len = len < 0 ? 0 : (len < room * KB ? len : room * KB);
  const int open = a.open_block[sh];
  const int n = (len + KB - 1) / KB;
  for (int i = tid; i < room; i += EVICT_THREADS) {
    tab[i] = a.table[base + i];
    bits[i] = __float_as_uint(a.weights[base + i]);
  }
  const bool cuts = n > a.keep;
  const int stay = cuts ? a.keep : n;
  const int mid0 = a.sink, mid1 = n - a.recent;       // used where the sequence is cut
  auto key = [&](int i) -> uint32_t {
    const uint32_t b = bits[i];
    return __uint_as_float(b) > 0.f ? b : 0u;
  };
  // bound: the key of the last of the heaviest `wanted` of the middle; above: how many are heavier
  uint32_t bound = 0;
  int above = 0;
  const int wanted = a.keep - a.sink - a.recent;
  if (cuts && wanted > 0) {
    constexpr int SHIFT[3] = {20, 9, 0}, WIDTH[3] = {11, 11, 9};
#pragma unroll
    for (int round = 0; round < 3; ++round) {
      hist[tid] = 0;
      hist[tid + EVICT_THREADS] = 0;
      __syncthreads();
      for (int i = mid0 + tid; i < mid1; i += EVICT_THREADS) {
        const uint32_t k = key(i);
        if (round == 0 || k >> (SHIFT[round] + WIDTH[round]) == bound >> (SHIFT[round] + WIDTH[round]))
          atomicAdd(&hist[(k >> SHIFT[round]) & ((1u << WIDTH[round]) - 1)], 1);
      }
      __syncthreads();
      // keys in bins above this thread's pair, from the top: threads in reverse order
      const int hi = BINS - 1 - 2 * tid;
      const int h1 = hist[hi], h0 = hist[hi - 1];
      const int incl = wave_incl_scan(h1 + h0);
      if (lane == 63) part[wave] = incl;
      __syncthreads();
      int before = above + incl - h1 - h0;
      for (int i = 0; i < wave; ++i) before += part[i];
      if (before < wanted && before + h1 >= wanted) {
        s_bin[0] = hi;
        s_bin[1] = before;
      } else if (before + h1 < wanted && before + h1 + h0 >= wanted) {
        s_bin[0] = hi - 1;
        s_bin[1] = before + h1;
      }
      __syncthreads();
      bound |= (uint32_t)s_bin[0] << SHIFT[round];
      above = s_bin[1];
    }
  } else if (cuts) {
    bound = 0xffffffffu;                              // none of the middle stays
  }
  const int ties = wanted - above;                    // of those at the bound, the first that stay
  __syncthreads();
  // this wave's run of blocks: how many stay for sure, and how many are at the bound
  const int run = (room + WAVES * 64 - 1) / (WAVES * 64) * 64;
  const int i0 = wave * run, i1 = min(i0 + run, room);
  auto sure = [&](int i, bool& at_bound) {
    at_bound = false;
    if (i >= n) return false;
    if (!cuts || i < mid0 || i >= mid1) return true;
    const uint32_t k = key(i);
    at_bound = k == bound;
    return k > bound;
  };
  int kept = 0, eq = 0;
  for (int i = i0; i < i1; i += 64) {
    bool at_bound = false;
    const bool yes = i + lane < i1 && sure(i + lane, at_bound);
    kept += __popcll(__ballot(yes));
    eq += __popcll(__ballot(i + lane < i1 && at_bound));
  }
  if (lane == 0) {
    part[wave] = kept;
    part_eq[wave] = eq;
  }
  __syncthreads();
  int at = 0, seen = 0;
  for (int w = 0; w < wave; ++w) {
    at += part[w];
    seen += part_eq[w];
  }
  at += min(seen, max(ties, 0));                      // of the ties before, those that stay
  const unsigned long long below = (1ull << lane) - 1;
  for (int i = i0; i < i1; i += 64) {
    const int b = i + lane;
    bool at_bound = false;
    bool here = b < i1 && sure(b, at_bound);
    at_bound = at_bound && b < i1;
    const unsigned long long tied = __ballot(at_bound);
    here = here || (at_bound && seen + __popcll(tied & below) < ties);
    const unsigned long long all = __ballot(here);
    const int before = at + __popcll(all & below);    // blocks that stay before this one
    if (b < i1) {
      const int to = here ? before : (b < n ? stay + b - before : b);
      a.table_out[base + to] = tab[b];
      a.weights_out[base + to] = here ? __uint_as_float(bits[b]) : 0.f;
      if (b == open) a.open_out[sh] = here ? to : -1;
    }
    at += __popcll(all);
    seen += __popcll(tied);
  }
  if (tid == 0) {
    a.lengths_out[sh] = len - (n - stay) * KB;
    if (open < 0 || open >= room) a.open_out[sh] = -1;
  }
}

// ---- launches ---------------------------------------------------------------------------

bool bad_cache(const sbsa_cache8* c) {
  return !c || !c->codes_k || !c->codes_v || !c->scales || !c->tail || !c->table || !c->weights || !c->lengths ||
         !c->open_block || !c->counters || !c->overflow || c->num_seqs < 1 || c->num_kv_heads < 1 ||
         c->num_blocks < 1 || ((uintptr_t)c->codes_k | (uintptr_t)c->codes_v | (uintptr_t)c->tail) % 16;
}

bool unsupported_cache(const sbsa_cache8* c) {
  return (c->head_dim != 128 && c->head_dim != 256) || (c->format != SBSA_CACHE8_E4M3 && c->format != SBSA_CACHE8_INT8) ||
         c->num_blocks > SBSA_CACHE8_MAX_BLOCKS || c->num_seqs > 65535 || c->num_kv_heads > 65535;
}

// bf16 rows that are read or written in pieces of 16 bytes
bool bad_rows(const void* p, int64_t st, int64_t sh) { return !p || (uintptr_t)p % 16 || st % 8 || sh % 8; }

template <int D, int FMT>
void launch_append(const AppendArgs& a, dim3 grid, hipStream_t stream) {
  hipLaunchKernelGGL((append_kernel<D, FMT>), grid, dim3(256), 0, stream, a);
}

// How a call's rows go over the grid.
struct AttendPlan {
  bool keys;                 // the waves of a block share its rows and split its keys
  int rows;                  // of a wave
  int tile_queries, tiles_per_seq, splits;
  int64_t tiles;
};

AttendPlan plan_attend(const sbsa_cache8* c, int num_q_heads, int64_t tokens, int64_t max_rows, bool ragged) {
  AttendPlan p;
  const int g = num_q_heads / c->num_kv_heads;
  const int64_t uniform = tokens / c->num_seqs;
  int64_t most = ragged ? (max_rows < 1 || max_rows > tokens ? tokens : max_rows) : uniform;
  p.keys = most * g <= 32;
  p.rows = most * g <= 16 ? 16 : 32;
  p.tile_queries = (p.keys ? p.rows : 4 * p.rows) / g;
  p.tiles_per_seq = (int)((uniform + p.tile_queries - 1) / p.tile_queries);
  p.tiles = ragged ? tokens / p.tile_queries + c->num_seqs : (int64_t)p.tiles_per_seq * c->num_seqs;
  // enough grid blocks for two per compute unit of the card's 256, each with a block of keys per wave at least
  const int64_t have = p.tiles * c->num_kv_heads;
  int64_t splits = 512 / (have > 0 ? have : 1);
  const int64_t most_splits = (c->num_blocks + 3) / 4;
  splits = splits < most_splits ? splits : most_splits;
  p.splits = splits < 1 ? 1 : (int)splits;
  return p;
}

// The workspace's parts, in floats: the shares' O and sums, the rows' sums, and each row's sums block by block.
struct AttendSpace {
  size_t o, part, row, w;
  size_t bytes() const { return (o + part + row + w) * sizeof(float); }
};

AttendSpace attend_space(const AttendPlan& p, const sbsa_cache8* c, int64_t tokens, int num_q_heads, bool accumulate) {
  const size_t rows = (size_t)tokens * num_q_heads;
  AttendSpace x;
  x.o = p.splits > 1 ? p.splits * rows * c->head_dim : 0;
  x.part = p.splits > 1 ? 2 * p.splits * rows : 0;
  x.row = accumulate ? 2 * rows : 0;
  x.w = accumulate && p.keys ? 2 * rows * c->num_blocks : 0;
  return x;
}

template <int D, int FMT, int R>
bool launch_keys(const AttendArgs& a, dim3 grid, hipStream_t stream) {
  constexpr int lds = 4 * R * D * (int)sizeof(float);
  if (lds > 48 * 1024 && hipFuncSetAttribute(reinterpret_cast<const void*>(attend_keys_kernel<D, FMT, R>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess)
    return false;
  hipLaunchKernelGGL((attend_keys_kernel<D, FMT, R>), grid, dim3(256), lds, stream, a);
  return true;
}

template <int D, int FMT>
bool launch_attend(const AttendArgs& a, const AttendPlan& p, int accumulate, hipStream_t stream) {
  const dim3 grid((unsigned)(p.tiles * p.splits), (unsigned)a.c.num_kv_heads);
  if (p.keys) {
    if (!(p.rows == 16 ? launch_keys<D, FMT, 16>(a, grid, stream) : launch_keys<D, FMT, 32>(a, grid, stream))) return false;
  } else {
    hipLaunchKernelGGL((attend_rows_kernel<D, FMT>), grid, dim3(256), 0, stream, a);
  }
  if (p.splits > 1)
    hipLaunchKernelGGL((join_kernel<D>), dim3((unsigned)(a.tokens * a.hq), D / 64), dim3(256), 0, stream, a);
  if (accumulate && p.keys)
    hipLaunchKernelGGL(weigh_shares_kernel, dim3((unsigned)((a.c.num_blocks + 255) / 256), (unsigned)a.c.num_kv_heads,
                                                 (unsigned)a.c.num_seqs), dim3(256), 0, stream, a);
  else if (accumulate)
    hipLaunchKernelGGL((weigh_kernel<D, FMT>),
                       dim3((unsigned)((a.c.num_blocks + 3) / 4), (unsigned)a.c.num_kv_heads, (unsigned)a.c.num_seqs),
                       dim3(256), 0, stream, a);
  return true;
}

}  // namespace

extern "C" int sbsa_cache8_append(const sbsa_cache8* cache, const void* k, int64_t k_st, int64_t k_sh, const void* v,
                                  int64_t v_st, int64_t v_sh, int64_t tokens, const int32_t* offsets,
                                  const int32_t* start, int64_t max_rows, hipStream_t stream) {
  if (bad_cache(cache) || tokens < 0 || (tokens > 0 && (bad_rows(k, k_st, k_sh) || bad_rows(v, v_st, v_sh))) ||
      (!offsets && tokens % cache->num_seqs))
    return SBSA_ERR_ARG;
  if (unsupported_cache(cache) || tokens > (1 << 24)) return SBSA_ERR_UNSUPPORTED;
  if (tokens == 0 && !start) return SBSA_OK;
  AppendArgs a;
  a.c = *cache;
  a.k = (const bf16_t*)k; a.v = (const bf16_t*)v;
  a.k_st = k_st; a.k_sh = k_sh; a.v_st = v_st; a.v_sh = v_sh;
  a.tokens = tokens; a.uniform = tokens / cache->num_seqs; a.offsets = offsets; a.start = start;
  int64_t most = offsets ? (max_rows < 1 || max_rows > tokens ? tokens : max_rows) : a.uniform;
  int64_t blocks = most < 1 ? 1 : (most + KB - 2) / KB + 1;
  if (blocks > cache->num_blocks) blocks = cache->num_blocks;
  const dim3 grid((unsigned)blocks, (unsigned)cache->num_kv_heads, (unsigned)cache->num_seqs);
  if (cache->head_dim == 128)
    cache->format == SBSA_CACHE8_E4M3 ? launch_append<128, SBSA_CACHE8_E4M3>(a, grid, stream)
                                      : launch_append<128, SBSA_CACHE8_INT8>(a, grid, stream);
  else
    cache->format == SBSA_CACHE8_E4M3 ? launch_append<256, SBSA_CACHE8_E4M3>(a, grid, stream)
                                      : launch_append<256, SBSA_CACHE8_INT8>(a, grid, stream);
  SBSA_CHECK_LAUNCH();
  return SBSA_OK;
}

extern "C" size_t sbsa_cache8_attend_workspace_bytes(const sbsa_cache8* cache, int num_q_heads, int64_t tokens,
                                                     int64_t max_rows, int ragged, int accumulate) {
  if (!cache || cache->num_seqs < 1 || cache->num_kv_heads < 1 || num_q_heads < cache->num_kv_heads ||
      num_q_heads / cache->num_kv_heads > 16 || tokens < 1)
    return 0;
  return attend_space(plan_attend(cache, num_q_heads, tokens, max_rows, ragged != 0), cache, tokens, num_q_heads,
                      accumulate != 0).bytes();
}

extern "C" int sbsa_cache8_attend(const sbsa_cache8* cache, const void* q, int64_t q_st, int64_t q_sh, int num_q_heads,
                                  int64_t tokens, const int32_t* offsets, int64_t max_rows, float sm_scale, void* out,
                                  int64_t o_st, int64_t o_sh, float* lse, int accumulate, void* workspace,
                                  size_t workspace_bytes, hipStream_t stream) {
  if (bad_cache(cache) || tokens < 0 || num_q_heads < 1 || num_q_heads % cache->num_kv_heads ||
      (!offsets && tokens % cache->num_seqs))
    return SBSA_ERR_ARG;
  if (tokens > 0 && (bad_rows(q, q_st, q_sh) || bad_rows(out, o_st, o_sh))) return SBSA_ERR_ARG;
  if (unsupported_cache(cache) || num_q_heads / cache->num_kv_heads > 16 || tokens * num_q_heads >= (1 << 24))
    return SBSA_ERR_UNSUPPORTED;
  if (tokens == 0) return SBSA_OK;
  const AttendPlan p = plan_attend(cache, num_q_heads, tokens, max_rows, offsets != nullptr);
  if (p.tiles * p.splits >= (1 << 24)) return SBSA_ERR_UNSUPPORTED;
  const AttendSpace space = attend_space(p, cache, tokens, num_q_heads, accumulate != 0);
  if (workspace_bytes < space.bytes()) return SBSA_ERR_CAPACITY;
  if (space.bytes() > 0 && (!workspace || (uintptr_t)workspace % 16)) return SBSA_ERR_ARG;
  AttendArgs a;
  a.c = *cache;
  a.q = (const bf16_t*)q; a.q_st = q_st; a.q_sh = q_sh;
  a.out = (bf16_t*)out; a.o_st = o_st; a.o_sh = o_sh; a.lse = lse;
  a.part_o = (float*)workspace;
  a.part_ml = (f32x2_t*)(a.part_o + space.o);
  a.row_ml = accumulate ? (f32x2_t*)(a.part_o + space.o + space.part) : nullptr;
  a.part_w = space.w ? (f32x2_t*)(a.part_o + space.o + space.part + space.row) : nullptr;
  a.offsets = offsets; a.tokens = tokens; a.uniform = tokens / cache->num_seqs;
  a.hq = num_q_heads; a.g = num_q_heads / cache->num_kv_heads;
  a.splits = p.splits; a.tile_queries = p.tile_queries; a.tiles_per_seq = p.tiles_per_seq;
  a.scale_log2 = sm_scale * LOG2E;
  const bool e4m3 = cache->format == SBSA_CACHE8_E4M3;
  const bool ok = cache->head_dim == 128
                      ? (e4m3 ? launch_attend<128, SBSA_CACHE8_E4M3>(a, p, accumulate, stream)
                              : launch_attend<128, SBSA_CACHE8_INT8>(a, p, accumulate, stream))
                      : (e4m3 ? launch_attend<256, SBSA_CACHE8_E4M3>(a, p, accumulate, stream)
                              : launch_attend<256, SBSA_CACHE8_INT8>(a, p, accumulate, stream));
  if (!ok) return SBSA_ERR_LAUNCH;
  SBSA_CHECK_LAUNCH();
  return SBSA_OK;
}

extern "C" int sbsa_cache8_evict(const int32_t* table, const float* weights, const int32_t* lengths,
                                 const int32_t* open_block, int32_t* table_out, float* weights_out,
                                 int32_t* lengths_out, int32_t* open_block_out, int num_seqs, int num_kv_heads,
                                 int num_blocks, int keep, int sink, int recent, hipStream_t stream) {
  if (!table || !weights || !lengths || !open_block || !table_out || !weights_out || !lengths_out || !open_block_out ||
      num_seqs < 1 || num_kv_heads < 1 || num_blocks < 1 || sink < 0 || recent < 1 || keep < 1 ||
      (int64_t)sink + recent > keep)
    return SBSA_ERR_ARG;
  if (num_blocks > SBSA_CACHE8_MAX_BLOCKS || num_seqs > 65535 || num_kv_heads > 65535) return SBSA_ERR_UNSUPPORTED;
  const EvictArgs a{table, weights, lengths, open_block, table_out, weights_out, lengths_out, open_block_out,
                    num_blocks, keep, sink, recent};
  const size_t lds = (size_t)num_blocks * 8;
  if (lds > 48 * 1024 && hipFuncSetAttribute(reinterpret_cast<const void*>(evict_kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess)
    return SBSA_ERR_LAUNCH;
  hipLaunchKernelGGL(evict_kernel, dim3((unsigned)((int64_t)num_seqs * num_kv_heads)), dim3(EVICT_THREADS), lds, stream, a);
  SBSA_CHECK_LAUNCH();
  return SBSA_OK;
}
