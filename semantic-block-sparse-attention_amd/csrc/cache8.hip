// The 8-bit key/value cache of a dense layer: new rows quantised block by block, attention of
// the newest rows over the cache, and the tables of a cache without its least attended blocks.
//
// A block is 64 tokens of one (sequence, KV head).  Keys lie [64][D], values [D][64]:
// both are then the A operand of their product as they lie (S^T = K Q^T takes 8 dims of
// a key per lane, O^T = V^T P^T 8 keys of a dim), and nothing is transposed in the attention.
#include "sbsa_common.h"

namespace {

constexpr int KB = SBSA_CACHE8_BLOCK;
constexpr float LOG2E = 1.44269504088896340736f;
constexpr float LN2 = 0.69314718055994530942f;
typedef __attribute__((ext_vector_type(16))) float f32x16_t;

__device__ __forceinline__ f32x16_t mfma32x32x16(bf16x8_t a, bf16x8_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
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

// A block of the grid takes a block of 64 tokens (and every gridDim.x-th after it) of one
// (sequence, head), keys then values: its rows into registers, the largest
// magnitude over the block, the codes out; the values' codes turn through LDS.  The last of a
// (sequence, head)'s grid blocks to end moves the length on, so that none reads a moved one.
template <int D, int FMT>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
  constexpr int CH = D / 8;             // 16-byte pieces of a row
  constexpr int RP = 256 / CH;          // rows of one pass of the threads
  constexpr int PASSES = KB / RP;
  constexpr float CODE_MAX = FMT == SBSA_CACHE8_E4M3 ? 448.f : 127.f;
  const sbsa_cache8& c = a.c;
  const int h = blockIdx.y, s = blockIdx.z, tid = threadIdx.x;
  const int64_t sh = (int64_t)s * c.num_kv_heads + h;
  const int64_t heads = (int64_t)c.num_seqs * c.num_kv_heads;
  __shared__ float red[4];
  __shared__ uint32_t turn[D * (KB / 4 + 1)];
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

  const int col = (tid % CH) * 8, r0 = tid / CH;
  for (int b = first + (int)blockIdx.x; b <= last; b += (int)gridDim.x) {
    const int64_t place = place_of(c, sh, b);
#pragma unroll 1
    for (int t = 0; t < 2; ++t) {
      const bf16_t* src = t ? a.v + row0 * a.v_st + h * a.v_sh : a.k + row0 * a.k_st + h * a.k_sh;
      const int64_t st = t ? a.v_st : a.k_st;
      bf16_t* tail = (bf16_t*)c.tail + ((int64_t)t * heads + sh) * KB * D;
      const float old_scale = c.scales[(int64_t)t * heads * c.num_blocks + place];
      uint8_t* codes = t ? (uint8_t*)c.codes_v + place * KB * D : (uint8_t*)c.codes_k + place * KB * D;
      u32x4_t x[PASSES];
      float most = 0.f;
      bool fine = true;
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        const int j = p * RP + r0, pos = b * KB + j;
        u32x4_t w = {0u, 0u, 0u, 0u};
        if (pos >= start && pos < end) {
          w = *reinterpret_cast<const u32x4_t*>(src + (int64_t)(pos - start) * st + col);
        } else if (pos < start && open == b) {
          w = *reinterpret_cast<const u32x4_t*>(tail + (int64_t)j * D + col);
        } else if (pos < start) {
          // the row is there in its codes alone
          bf16_t y[8];
#pragma unroll
          for (int i = 0; i < 8; ++i)
            y[i] = f2bf(decode1<FMT>(codes[t ? (col + i) * KB + j : j * D + col + i]) * old_scale);
          __builtin_memcpy(&w, y, 16);
        }
        x[p] = w;
        bf16_t y[8];
        __builtin_memcpy(y, &w, 16);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          fine = fine && (y[i] & 0x7f80) != 0x7f80;
          most = fmaxf(most, fabsf(bf2f(y[i])));
        }
      }
      // the block's largest magnitude; one value that is not finite makes the scale NaN
      most = fine ? most : INFINITY;
      most = wave_max(most);
      __syncthreads();                  // every row is read before a code or the tail is written
      if ((tid & 63) == 0) red[tid >> 6] = most;
      __syncthreads();
      most = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
      fine = most < INFINITY;
      const float scale = fine ? fmaxf(most / CODE_MAX, 0x1p-126f) : __uint_as_float(0x7fc00000u);
      if (tid == 0) c.scales[(int64_t)t * heads * c.num_blocks + place] = scale;
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        const int j = p * RP + r0;
        bf16_t y[8];
        __builtin_memcpy(y, &x[p], 16);
        uint32_t w[2] = {0u, 0u};
        if (fine) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            w[i >> 1] |= encode2<FMT>(bf2f(y[2 * i]) / scale, bf2f(y[2 * i + 1]) / scale) << (16 * (i & 1));
        }
        if (t == 0) {
          u32x2_t o;
          o.x = w[0]; o.y = w[1];
          *reinterpret_cast<u32x2_t*>(codes + (int64_t)j * D + col) = o;
        } else {
          uint8_t* tb = reinterpret_cast<uint8_t*>(turn);
#pragma unroll
          for (int i = 0; i < 8; ++i) tb[(col + i) * (KB + 4) + j] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
        }
        if (b == last && first == last) {
          const int pos = b * KB + j;
          if (pos < end && (pos >= start || open != b))
            *reinterpret_cast<u32x4_t*>(tail + (int64_t)j * D + col) = x[p];
        }
      }
      if (t == 1) {
        __syncthreads();
        for (int i = tid; i < D * (KB / 4); i += 256)
          reinterpret_cast<uint32_t*>(codes)[i] = turn[(i / (KB / 4)) * (KB / 4 + 1) + i % (KB / 4)];
      }
    }
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
    for (int t = 0; t < 2 && last > first; ++t) {
      const bf16_t* src = t ? a.v + row0 * a.v_st + h * a.v_sh : a.k + row0 * a.k_st + h * a.k_sh;
      const int64_t st = t ? a.v_st : a.k_st;
      bf16_t* tail = (bf16_t*)c.tail + ((int64_t)t * heads + sh) * KB * D;
      for (int j = r0; last * KB + j < end && j < KB; j += RP)
        *reinterpret_cast<u32x4_t*>(tail + (int64_t)j * D + col) =
            *reinterpret_cast<const u32x4_t*>(src + (int64_t)(last * KB + j - start) * st + col);
    }
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
  float* part_lse;             // [splits][tokens * Hq], base 2
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
      const int l = __ffsll((long long)past) - 1;
      s = s0 + l;
      rows_of(a.offsets, s, 0, a.tokens, row0, n);
      q0 = (int)(t - before - (__shfl(upto, l, 64) - __shfl(mine, l, 64))) * a.tile_queries;
      return true;
    }
    before += __shfl(upto, 63, 64);
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

// A wave's state over R = 16 or 32 rows (columns of S^T and O^T).  Lane l holds row l % R, and of
// a block's 64 keys those of its part l / R: 16 or 32 consecutive ones, because the K rows
// are handed to the product in the order that leaves them so.  They are the B operand of
// O^T = V^T P^T as they lie, so the probabilities never leave the lane.
template <int D, int FMT, int R>
struct WaveRows {
  static constexpr int PARTS = 64 / R;          // lanes that share a row
  static constexpr int MINE = KB / PARTS;       // a lane's keys of a block
  static constexpr int GROUPS = KB / R;         // products of R keys
  static constexpr int SEG = 16 * PARTS;        // dims that one 16-byte load of every part covers
  static constexpr int NT = D / R;              // R-dim tiles of O^T
  static constexpr int NI = R * R / 64;         // accumulator values of a lane
  typedef __attribute__((ext_vector_type(NI))) float acc_t;

  bf16x8_t q[D / SEG][2];
  acc_t o[NT];
  float m, l;

  static __device__ __forceinline__ acc_t mfma(bf16x8_t x, bf16x8_t y, acc_t z) {
    if constexpr (R == 16)
      return mfma16x16x32(x, y, z);
    else
      return mfma32x32x16(x, y, z);
  }

  __device__ __forceinline__ void start(const bf16_t* qrow, int lane) {
    const int part = lane / R;
#pragma unroll
    for (int j = 0; j < D / SEG; ++j)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        u32x4_t w = {0u, 0u, 0u, 0u};
        if (qrow) w = *reinterpret_cast<const u32x4_t*>(qrow + j * SEG + part * 16 + x * 8);
        q[j][x] = as_bf16x8(w);
      }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < NI; ++i) o[t][i] = 0.f;
    m = -INFINITY;
    l = 0.f;
  }

  // the key (of a block's 64) that row r of product g takes
  static __device__ __forceinline__ int key_of(int r, int g) {
    if constexpr (R == 16)
      return (r >> 2) * 16 + g * 4 + (r & 3);
    else
      return ((r >> 2) & 1) * 32 + g * 16 + (r >> 3) * 4 + (r & 3);
  }

  // scores of a block's keys, times the keys' scale and log2(e) sm_scale
  static __device__ __forceinline__ void scores(const bf16x8_t (&q)[D / SEG][2], const uint8_t* kb, float ks, int lane,
                                                acc_t (&sc)[GROUPS]) {
    const int part = lane / R;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      const uint8_t* row = kb + key_of(lane % R, g) * D + part * 16;
      acc_t acc;
#pragma unroll
      for (int i = 0; i < NI; ++i) acc[i] = 0.f;
#pragma unroll
      for (int j = 0; j < D / SEG; ++j) {
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(row + j * SEG);
        acc = mfma(decode8<FMT>(w.x, w.y), q[j][0], acc);
        acc = mfma(decode8<FMT>(w.z, w.w), q[j][1], acc);
      }
#pragma unroll
      for (int i = 0; i < NI; ++i) acc[i] *= ks;
      sc[g] = acc;
    }
  }

  // one block: seen is how many of its keys the lane's row sees, filled how many are there (all: every row
  // sees every key)
  __device__ __forceinline__ void block(const uint8_t* kb, const uint8_t* vb, float ks, float vs, int seen, int filled,
                                        bool all, int lane) {
    const int part = lane / R;
    acc_t sc[GROUPS];
    scores(q, kb, ks, lane, sc);
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
    // the reference maximum moves only when a row has gone 2^8 above it: until then its
    // probabilities are at most 2^8, which neither bf16 nor the fp32 sums mind
    if (__ballot(top > m + 8.f)) {
      const float to = fmaxf(m, top);
      const float f = m == to ? 1.f : __builtin_amdgcn_exp2f(m - to);
      l *= f;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < NI; ++i) o[t][i] *= f;
      m = to;
    }
    const float ref = m == -INFINITY ? 0.f : m;
    u32x4_t p[MINE / 8];
#pragma unroll
    for (int x = 0; x < MINE / 2; ++x) {
      const int i0 = 2 * x, i1 = 2 * x + 1;
      const float p0 = __builtin_amdgcn_exp2f(sc[i0 / NI][i0 % NI] - ref);
      const float p1 = __builtin_amdgcn_exp2f(sc[i1 / NI][i1 % NI] - ref);
      l += p0 + p1;
      // the scale joins the probability before its one rounding; an unseen key's is 0 whatever the scale
      const bool h0 = !all && part * MINE + i0 >= seen, h1 = !all && part * MINE + i1 >= seen;
      p[x / 4][x % 4] = pack2bf(h0 ? 0.f : p0 * vs, h1 ? 0.f : p1 * vs);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const uint8_t* row = vb + (t * R + lane % R) * KB + part * MINE;
#pragma unroll
      for (int x = 0; x < MINE / 16; ++x) {
        u32x4_t w = *reinterpret_cast<const u32x4_t*>(row + x * 16);
        if (!all) w = clear_past(w, filled - (part * MINE + x * 16));
        o[t] = mfma(decode8<FMT>(w.x, w.y), as_bf16x8(p[2 * x]), o[t]);
        o[t] = mfma(decode8<FMT>(w.z, w.w), as_bf16x8(p[2 * x + 1]), o[t]);
      }
    }
  }

  // the row's sum over its lanes
  __device__ __forceinline__ void total() {
    if constexpr (R == 16) l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
  }

  // joins another wave's rows, left in LDS
  static constexpr int FOLD_FLOATS = NT * NI * 64 + 128;
  __device__ __forceinline__ void leave(float* to, int lane) const {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < NI; ++i) to[(t * NI + i) * 64 + lane] = o[t][i];
    to[NT * NI * 64 + lane] = m;
    to[NT * NI * 64 + 64 + lane] = l;
  }
  __device__ __forceinline__ void join(const float* from, int lane) {
    const float m1 = from[NT * NI * 64 + lane], l1 = from[NT * NI * 64 + 64 + lane];
    const float to = fmaxf(m, m1), ref = to == -INFINITY ? 0.f : to;
    const float f0 = __builtin_amdgcn_exp2f(m - ref), f1 = __builtin_amdgcn_exp2f(m1 - ref);
    m = to;
    l = l * f0 + l1 * f1;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < NI; ++i) o[t][i] = o[t][i] * f0 + from[(t * NI + i) * 64 + lane] * f1;
  }

  // four consecutive dims of the lane's row: tile t, quarter x of the accumulator
  static __device__ __forceinline__ int dim_of(int t, int x, int lane) { return t * R + 8 * x + 4 * (lane / R); }
};

// One grid block: a tile of rows of one (sequence, KV head) over one share of the keys.  KEYS: its
// four waves hold the same R rows and take every fourth block of keys each, joined through LDS at
// the end; otherwise each holds R rows of its own.
template <int D, int FMT, int R, bool KEYS>
__global__ __launch_bounds__(256, R == 32 && D == 256 ? 1 : 2) void attend_kernel(AttendArgs a) {
  using W = WaveRows<D, FMT, R>;
  const sbsa_cache8& c = a.c;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int split = (int)(blockIdx.x % a.splits);
  const int64_t tiles = gridDim.x / a.splits;
  __shared__ float fold[KEYS ? W::FOLD_FLOATS : 1];

  int s, n, q0;
  int64_t row0;
  // late tiles see the most keys: they go first
  if (!tile_of(a, tiles - 1 - blockIdx.x / a.splits, s, row0, n, q0)) return;
  const int h = blockIdx.y;
  const int64_t sh = (int64_t)s * c.num_kv_heads + h;
  const int64_t heads = (int64_t)c.num_seqs * c.num_kv_heads;
  const int held = held_of(c, sh);

  // this lane's row
  const int r = (KEYS ? 0 : wave * R) + lane % R;
  const int qi = q0 + r / a.g, head = h * a.g + r % a.g;
  const bool there = r < a.tile_queries * a.g && qi < n;
  int vis = there ? held - n + qi + 1 : 0;
  vis = vis < 0 ? 0 : vis;
  int vis_most = vis, vis_least = there ? vis : 0x7fffffff;
#pragma unroll
  for (int x = 1; x < R; x <<= 1) {
    vis_most = max(vis_most, __shfl_xor(vis_most, x, 64));
    vis_least = min(vis_least, __shfl_xor(vis_least, x, 64));
  }
  vis_most = __builtin_amdgcn_readfirstlane(vis_most);
  vis_least = __builtin_amdgcn_readfirstlane(vis_least);

  // the share: of the blocks that the tile's last row sees
  const int tile_last = q0 + a.tile_queries < n ? q0 + a.tile_queries : n;
  int tile_vis = held - n + tile_last;
  tile_vis = tile_vis < 0 ? 0 : tile_vis;
  const int blocks = (tile_vis + KB - 1) / KB;
  const int per = (blocks + a.splits - 1) / a.splits;
  const int lo = split * per;
  int hi = lo + per < blocks ? lo + per : blocks;
  if (!KEYS) hi = min(hi, (vis_most + KB - 1) / KB);

  W w;
  w.start(there ? a.q + (row0 + qi) * a.q_st + head * a.q_sh : nullptr, lane);
  const float* scales_v = c.scales + heads * c.num_blocks;
  for (int b = lo + (KEYS ? wave : 0); b < hi; b += KEYS ? 4 : 1) {
    const int64_t place = place_of(c, sh, b);
    w.block((const uint8_t*)c.codes_k + place * KB * D, (const uint8_t*)c.codes_v + place * KB * D,
            c.scales[place] * a.scale_log2, scales_v[place], vis - b * KB, held - b * KB, (b + 1) * KB <= vis_least, lane);
  }
  w.total();
  if constexpr (KEYS) {
    for (int x = 3; x > 0; --x) {
      if (wave == x) w.leave(fold, lane);
      __syncthreads();
      if (wave == 0) w.join(fold, lane);
      __syncthreads();
    }
    if (wave != 0) return;
  }
  if (!there) return;
  // a row without keys has sum 0 and gives 0; a NaN stays one
  const float inv = w.l == 0.f ? 0.f : 1.f / w.l;
  const float lse2 = w.l == 0.f ? -INFINITY : w.m + __builtin_amdgcn_logf(w.l);
  const int64_t row = (row0 + qi) * a.hq + head;
  if (a.splits == 1) {
    bf16_t* out = a.out + (row0 + qi) * a.o_st + head * a.o_sh;
#pragma unroll
    for (int t = 0; t < W::NT; ++t)
#pragma unroll
      for (int x = 0; x < W::NI / 4; ++x) {
        u32x2_t v;
        v.x = pack2bf(w.o[t][4 * x] * inv, w.o[t][4 * x + 1] * inv);
        v.y = pack2bf(w.o[t][4 * x + 2] * inv, w.o[t][4 * x + 3] * inv);
        *reinterpret_cast<u32x2_t*>(out + W::dim_of(t, x, lane)) = v;
      }
    if (a.lse && lane < R) a.lse[row] = lse2 * LN2;
    return;
  }
  float* po = a.part_o + ((int64_t)split * a.tokens * a.hq + row) * D;
#pragma unroll
  for (int t = 0; t < W::NT; ++t)
#pragma unroll
    for (int x = 0; x < W::NI / 4; ++x) {
      f32x4_t v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = w.o[t][4 * x + i] * inv;
      *reinterpret_cast<f32x4_t*>(po + W::dim_of(t, x, lane)) = v;
    }
  if (lane < R) a.part_lse[(int64_t)split * a.tokens * a.hq + row] = lse2;
}

// The shares of a row joined: a grid block per row, its waves every fourth share each.
template <int D>
__global__ __launch_bounds__(256) void join_kernel(AttendArgs a) {
  constexpr int PER = D / 64;
  const int64_t row = blockIdx.x, rows = a.tokens * a.hq;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t token = row / a.hq;
  const int head = (int)(row % a.hq);
  if (a.offsets && (token < a.offsets[0] || token >= a.offsets[a.c.num_seqs])) return;
  __shared__ float fold[4][64 * PER];
  float top = -INFINITY;
  for (int x = lane; x < a.splits; x += 64) top = fmaxf(top, a.part_lse[x * rows + row]);
  top = wave_max(top);
  const float ref = top == -INFINITY ? 0.f : top;
  float total = 0.f, acc[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) acc[i] = 0.f;
  for (int x = lane; x < a.splits; x += 64) total += __builtin_amdgcn_exp2f(a.part_lse[x * rows + row] - ref);
  total = wave_sum(total);
  for (int x = wave; x < a.splits; x += 4) {
    const float v = a.part_lse[x * rows + row];
    if (v == -INFINITY) continue;
    const float f = __builtin_amdgcn_exp2f(v - ref);
    const float* po = a.part_o + (x * rows + row) * D + lane * PER;
#pragma unroll
    for (int i = 0; i < PER; ++i) acc[i] += f * po[i];
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) fold[wave][lane * PER + i] = acc[i];
  __syncthreads();
  if (wave != 0) return;
  const float inv = total == 0.f ? 0.f : 1.f / total;
  bf16_t* out = a.out + token * a.o_st + head * a.o_sh + lane * PER;
#pragma unroll
  for (int i = 0; i < PER; i += 2) {
    const int d = lane * PER + i;
    const float x = (fold[0][d] + fold[1][d]) + (fold[2][d] + fold[3][d]);
    const float y = (fold[0][d + 1] + fold[1][d + 1]) + (fold[2][d + 1] + fold[3][d + 1]);
    *reinterpret_cast<uint32_t*>(out + i) = pack2bf(x * inv, y * inv);
  }
  if (a.lse && lane == 0) a.lse[row] = total == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(total)) * LN2;
}

// The attention that each block receives: a wave holds a block of keys and goes over the rows that
// see it, their sums known (lse); one addition per block, so no order of atomics enters.
template <int D, int FMT>
__global__ __launch_bounds__(256) void weigh_kernel(AttendArgs a) {
  using W = WaveRows<D, FMT, 32>;
  const sbsa_cache8& c = a.c;
  const int lane = threadIdx.x & 63;
  const int b = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6);
  const int h = blockIdx.y, s = blockIdx.z;
  const int64_t sh = (int64_t)s * c.num_kv_heads + h;
  int64_t row0;
  int n;
  rows_of(a.offsets, s, a.uniform, a.tokens, row0, n);
  const int held = held_of(c, sh);
  if (n == 0 || b * KB >= held) return;
  const int64_t place = place_of(c, sh, b);
  const uint8_t* kb = (const uint8_t*)c.codes_k + place * KB * D;
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
    W w;
    w.start(there ? a.q + (row0 + qi) * a.q_st + head * a.q_sh : nullptr, lane);
    const float lse2 = there ? a.lse[(row0 + qi) * a.hq + head] * LOG2E : 0.f;
    typename W::acc_t sc[W::GROUPS];
    W::scores(w.q, kb, ks, lane, sc);
#pragma unroll
    for (int g = 0; g < W::GROUPS; ++g)
#pragma unroll
      for (int i = 0; i < W::NI; ++i)
        sum += (lane / 32) * W::MINE + g * W::NI + i < seen ? __builtin_amdgcn_exp2f(sc[g][i] - lse2) : 0.f;
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

// Sum of a value over the block; `part` has a place per wave and is read by all afterwards.
__device__ __forceinline__ int block_sum(int v, int* part) {
  v = wave_sum_i32(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  int t = 0;
  for (int i = 0; i < EVICT_THREADS / 64; ++i) t += part[i];
  return t;
}

// One (sequence, head): tables into LDS whole (the outputs may be the inputs), the weight of the last block
// that stays found bit by bit over the weights' bits (not negative, so their order is that of the
// numbers), then every block's new place by a prefix sum over the threads' runs of blocks.
__global__ __launch_bounds__(EVICT_THREADS) void evict_kernel(EvictArgs a) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem_evict[];
  int32_t* tab = reinterpret_cast<int32_t*>(smem_evict);
  uint32_t* bits = reinterpret_cast<uint32_t*>(tab + a.num_blocks);
  __shared__ int part[EVICT_THREADS / 64];
  const int64_t sh = blockIdx.x, base = sh * a.num_blocks;
  const int tid = threadIdx.x;
  const int room = a.num_blocks;
  int len = a.lengths[sh];
  len = len < 0 ? 0 : (len < room * KB ? len : room * KB);
  const int open = a.open_block[sh];
  const int n = (len + KB - 1) / KB;
  for (int i = tid; i < room; i += EVICT_THREADS) {
    tab[i] = a.table[base + i];
    bits[i] = __float_as_uint(a.weights[base + i]);
  }
  __syncthreads();
  const int stay = n < a.keep ? n : a.keep;
  const int mid0 = a.sink < n ? a.sink : n, mid1 = n - a.recent > mid0 ? n - a.recent : mid0;
  const int wanted = n > a.keep ? a.keep - a.sink - a.recent : mid1 - mid0;
  auto key = [&](int i) -> uint32_t {
    const float w = __uint_as_float(bits[i]);
    return w > 0.f ? __float_as_uint(w) : 0u;
  };
  // the largest bound that at least `wanted` of the middle blocks reach
  uint32_t bound = 0;
  int above = 0;                      // of them, strictly above the bound
  if (n > a.keep) {
    for (int bit = 30; bit >= 0; --bit) {
      const uint32_t cand = bound | (1u << bit);
      int v = 0;
      for (int i = mid0 + tid; i < mid1; i += EVICT_THREADS) v += key(i) >= cand;
      if (block_sum(v, part) >= wanted) bound = cand;
    }
    int v = 0;
    for (int i = mid0 + tid; i < mid1; i += EVICT_THREADS) v += key(i) > bound;
    above = block_sum(v, part);
  }
  const int ties = wanted - above;    // of those at the bound, the first that stay
  // this thread's run of blocks
  const int per = (room + EVICT_THREADS - 1) / EVICT_THREADS;
  const int i0 = tid * per < room ? tid * per : room, i1 = i0 + per < room ? i0 + per : room;
  auto prefix = [&](int v) {          // sum over the threads before this one
    const int incl = wave_incl_scan(v);
    __syncthreads();
    if ((tid & 63) == 63) part[tid >> 6] = incl;
    __syncthreads();
    int t = incl - v;
    for (int i = 0; i < (tid >> 6); ++i) t += part[i];
    return t;
  };
  int eq = 0;
  for (int i = i0; i < i1; ++i) eq += n > a.keep && i >= mid0 && i < mid1 && key(i) == bound;
  const int eq_before = prefix(eq);
  auto stays = [&](int i, int& seen) {
    if (i >= n) return false;
    if (n <= a.keep || i < mid0 || i >= mid1) return true;
    const uint32_t k = key(i);
    if (k == bound) return seen++ < ties;
    return k > bound;
  };
  int kept = 0, seen = eq_before;
  for (int i = i0; i < i1; ++i) kept += stays(i, seen);
  int at = prefix(kept);
  seen = eq_before;
  for (int i = i0; i < i1; ++i) {
    int to = i;
    float w = 0.f;
    const bool here = stays(i, seen);
    if (here) {
      to = at++;
      w = __uint_as_float(bits[i]);
    } else if (i < n) {
      to = stay + i - at;             // behind those that stay: of the i blocks before, `at` stayed
    }
    a.table_out[base + to] = tab[i];
    a.weights_out[base + to] = w;
    if (i == open) a.open_out[sh] = here ? to : -1;
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

size_t attend_bytes(const AttendPlan& p, int64_t tokens, int num_q_heads, int dim) {
  return p.splits > 1 ? (size_t)p.splits * tokens * num_q_heads * (dim + 1) * sizeof(float) : 0;
}

template <int D, int FMT>
void launch_attend(const AttendArgs& a, const AttendPlan& p, int accumulate, hipStream_t stream) {
  const dim3 grid((unsigned)(p.tiles * p.splits), (unsigned)a.c.num_kv_heads);
  if (p.keys && p.rows == 16)
    hipLaunchKernelGGL((attend_kernel<D, FMT, 16, true>), grid, dim3(256), 0, stream, a);
  else if (p.keys)
    hipLaunchKernelGGL((attend_kernel<D, FMT, 32, true>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((attend_kernel<D, FMT, 32, false>), grid, dim3(256), 0, stream, a);
  if (p.splits > 1)
    hipLaunchKernelGGL((join_kernel<D>), dim3((unsigned)(a.tokens * a.hq)), dim3(256), 0, stream, a);
  if (accumulate)
    hipLaunchKernelGGL((weigh_kernel<D, FMT>),
                       dim3((unsigned)((a.c.num_blocks + 3) / 4), (unsigned)a.c.num_kv_heads, (unsigned)a.c.num_seqs),
                       dim3(256), 0, stream, a);
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
  (void)accumulate;
  if (!cache || cache->num_seqs < 1 || cache->num_kv_heads < 1 || num_q_heads < cache->num_kv_heads ||
      num_q_heads / cache->num_kv_heads > 16 || tokens < 1)
    return 0;
  return attend_bytes(plan_attend(cache, num_q_heads, tokens, max_rows, ragged != 0), tokens, num_q_heads,
                      cache->head_dim);
}

extern "C" int sbsa_cache8_attend(const sbsa_cache8* cache, const void* q, int64_t q_st, int64_t q_sh, int num_q_heads,
                                  int64_t tokens, const int32_t* offsets, int64_t max_rows, float sm_scale, void* out,
                                  int64_t o_st, int64_t o_sh, float* lse, int accumulate, void* workspace,
                                  size_t workspace_bytes, hipStream_t stream) {
  if (bad_cache(cache) || tokens < 0 || num_q_heads < 1 || num_q_heads % cache->num_kv_heads ||
      (!offsets && tokens % cache->num_seqs) || (accumulate && !lse))
    return SBSA_ERR_ARG;
  if (tokens > 0 && (bad_rows(q, q_st, q_sh) || bad_rows(out, o_st, o_sh))) return SBSA_ERR_ARG;
  if (unsupported_cache(cache) || num_q_heads / cache->num_kv_heads > 16 || tokens * num_q_heads >= (1 << 24))
    return SBSA_ERR_UNSUPPORTED;
  if (tokens == 0) return SBSA_OK;
  const AttendPlan p = plan_attend(cache, num_q_heads, tokens, max_rows, offsets != nullptr);
  if (p.tiles * p.splits >= (1 << 24)) return SBSA_ERR_UNSUPPORTED;
  if (workspace_bytes < attend_bytes(p, tokens, num_q_heads, cache->head_dim)) return SBSA_ERR_CAPACITY;
  if (p.splits > 1 && (!workspace || (uintptr_t)workspace % 16)) return SBSA_ERR_ARG;
  AttendArgs a;
  a.c = *cache;
  a.q = (const bf16_t*)q; a.q_st = q_st; a.q_sh = q_sh;
  a.out = (bf16_t*)out; a.o_st = o_st; a.o_sh = o_sh; a.lse = lse;
  a.part_o = (float*)workspace;
  a.part_lse = a.part_o + (size_t)p.splits * tokens * num_q_heads * cache->head_dim;
  a.offsets = offsets; a.tokens = tokens; a.uniform = tokens / cache->num_seqs;
  a.hq = num_q_heads; a.g = num_q_heads / cache->num_kv_heads;
  a.splits = p.splits; a.tile_queries = p.tile_queries; a.tiles_per_seq = p.tiles_per_seq;
  a.scale_log2 = sm_scale * LOG2E;
  if (cache->head_dim == 128)
    cache->format == SBSA_CACHE8_E4M3 ? launch_attend<128, SBSA_CACHE8_E4M3>(a, p, accumulate, stream)
                                      : launch_attend<128, SBSA_CACHE8_INT8>(a, p, accumulate, stream);
  else
    cache->format == SBSA_CACHE8_E4M3 ? launch_attend<256, SBSA_CACHE8_E4M3>(a, p, accumulate, stream)
                                      : launch_attend<256, SBSA_CACHE8_INT8>(a, p, accumulate, stream);
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
