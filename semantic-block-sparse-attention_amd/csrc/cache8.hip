// The 8-bit key/value cache of a dense layer: new rows quantised block by block, attention of
// the newest rows over the cache, and the tables of a cache without its least attended blocks.
//
// A block is 64 tokens of one (sequence, KV head).  Keys lie [64][D], values [D][64]:
// both are then the A operand of their product as they lie (S^T = K Q^T takes 8 dims of
// a key per lane, O^T = V^T P^T 8 keys of a dim), and nothing is transposed in the attention.
#include <algorithm>
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
typedef __attribute__((ext_vector_type(4))) int32_t i32x4_t;

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

// a value that is the same in every lane, in a scalar register
__device__ __forceinline__ float uniform(float v) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_readfirstlane((int)__float_as_uint(v)));
}

// a value joined with the one 32 (or 16) lanes away, without a round trip through LDS
__device__ __forceinline__ float max32(float v) {
  const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
}
__device__ __forceinline__ float max16(float v) {
  const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
}

// the lane's number, counted anew
__device__ __forceinline__ int lane_again() {
  int l = (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
  asm volatile("" : "+v"(l));
  return l;
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

// A block of the grid takes the keys (even grid x) or the values (odd) of a block of 64 tokens of one
// (sequence, head), and of every gridDim.x / 2-th block after it: its rows into registers, the largest magnitude
// over the block, the codes out.  A thread holds PASSES consecutive rows of 8 columns, so its codes of a key row are 8
// bytes of it and those of a value column PASSES bytes of that; the values' turn through LDS only to leave in
// whole rows of [dim][64].  No grid block moves a length that another may still read:
// ONE: the call touches one block of a (sequence, head) at most, and the last of its two grid blocks (by a ticket) moves the
// length on; otherwise append_end_kernel does (tickets of a long prompt's 1000 grid blocks on one address took 11 us).
//
// Memory bounds a prompt: 32768 tokens of 4 heads of 256 dims read 134 MB and write 67 in 43 us, 4.7 TB/s, and the closing
// kernel takes 4 more.  One token of 32 sequences takes 5.6 us: lengths, table, the open block's rows, one after another.
// (A device fence at each grid block's end, an L2 write-back, had made a prompt's 64 us 133.)
template <int D, int FMT, bool ONE>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
  constexpr int CH = D / 8;             // 16-byte pieces of a row
  constexpr int PASSES = KB * CH / 256; // consecutive rows of a thread: 4 or 8
  constexpr int LD = KB + 16;           // bytes of a value column in LDS: 16-byte pieces stay aligned
  constexpr float CODE_MAX = FMT == SBSA_CACHE8_E4M3 ? 448.f : 127.f;
  const sbsa_cache8& c = a.c;
  const int h = blockIdx.y, s = blockIdx.z, tid = threadIdx.x;
  const int t = blockIdx.x & 1, bx = blockIdx.x >> 1, step = gridDim.x >> 1;
  const int64_t sh = (int64_t)s * c.num_kv_heads + h;
  const int64_t heads = (int64_t)c.num_seqs * c.num_kv_heads;
  __shared__ int red[4];
  __shared__ __attribute__((aligned(16))) unsigned char turn[D * LD];

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
  const bf16_t* const src = t ? a.v + row0 * a.v_st + h * a.v_sh : a.k + row0 * a.k_st + h * a.k_sh;
  const int64_t st = t ? a.v_st : a.k_st;
  bf16_t* const tail = (bf16_t*)c.tail + (t * heads + sh) * KB * D;
  float* const scales = c.scales + t * heads * c.num_blocks;
  for (int b = first + bx; b <= last; b += step) {
    const int64_t place = place_of(c, sh, b);
    uint8_t* const codes = (t ? (uint8_t*)c.codes_v : (uint8_t*)c.codes_k) + place * KB * D;
    u32x4_t x[PASSES];
    if (b * KB >= start && (b + 1) * KB <= end) {     // the block is new rows throughout
#pragma unroll
      for (int p = 0; p < PASSES; ++p)
        x[p] = *reinterpret_cast<const u32x4_t*>(src + (int64_t)(b * KB + r0 + p - start) * st + col);
    } else {
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        const int j = r0 + p, pos = b * KB + j;
        u32x4_t w = {0u, 0u, 0u, 0u};
        if (pos >= start && pos < end) {
          w = *reinterpret_cast<const u32x4_t*>(src + (int64_t)(pos - start) * st + col);
        } else if (pos < start && open == b) {
          w = *reinterpret_cast<const u32x4_t*>(tail + j * D + col);
        } else if (pos < start) {
          // the row is there in its codes alone
          const float old = scales[place];
          const int at = t ? col * KB + j : j * D + col, by = t ? KB : 1;
          uint64_t half[2] = {0, 0};
#pragma unroll 1
          for (int i = 0; i < 8; ++i) {               // (rolled: rare, and 64 loads' addresses if not)
            const uint64_t y = f2bf(decode1<FMT>(codes[at + i * by]) * old);
            half[1] = half[1] >> 16 | half[0] << 48;
            half[0] = half[0] >> 16 | y << 48;
          }
          w.x = (uint32_t)half[1]; w.y = (uint32_t)(half[1] >> 32);
          w.z = (uint32_t)half[0]; w.w = (uint32_t)(half[0] >> 32);
        }
        x[p] = w;
      }
    }
    // the largest magnitude, as bf16 bits without the sign: one that is not finite is 0x7f80 and up
    u16x2_t top = {0, 0};
#pragma unroll
    for (int p = 0; p < PASSES; ++p)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w = x[p][i] & 0x7fff7fffu;
        u16x2_t v;
        __builtin_memcpy(&v, &w, 4);
        top = __builtin_elementwise_max(top, v);
      }
    int most = top.x > top.y ? top.x : top.y;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) most = max(most, __shfl_xor(most, o, 64));
    if ((tid & 63) == 0) red[tid >> 6] = most;
    __syncthreads();                    // and every row is read before a code or the tail is written
    most = max(max(red[0], red[1]), max(red[2], red[3]));
    const bool fine = most < 0x7f80;
    const float scale = fine ? fmaxf(bf2f((bf16_t)most) / CODE_MAX, 0x1p-126f) : __uint_as_float(0x7fc00000u);
    if (tid == 0) scales[place] = scale;
    const bool easy = scale >= 0x1p-90f;              // (no, where it is NaN)
    const float inv = 1.f / scale;
    // (a row or column at a time: the compiler would hold every quotient, and twice, for both divisions)
    auto codes_out = [&](auto&& divide) {
      auto value = [&](int p, int i) {
        const uint32_t w = x[p][i >> 1];
        return divide(bf2f((bf16_t)(i & 1 ? w >> 16 : w & 0xffffu)));
      };
      if (t == 0) {
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
          u32x2_t o;
#pragma unroll
          for (int i = 0; i < 2; ++i)
            o[i] = encode2<FMT>(value(p, 4 * i), value(p, 4 * i + 1)) | encode2<FMT>(value(p, 4 * i + 2), value(p, 4 * i + 3)) << 16;
          *reinterpret_cast<u32x2_t*>(codes + (r0 + p) * D + col) = o;
          __builtin_amdgcn_sched_barrier(0);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          uint32_t w[PASSES / 4];
#pragma unroll
          for (int q = 0; q < PASSES / 4; ++q)
            w[q] = encode2<FMT>(value(4 * q, i), value(4 * q + 1, i)) | encode2<FMT>(value(4 * q + 2, i), value(4 * q + 3, i)) << 16;
          __builtin_memcpy(turn + (col + i) * LD + r0, w, PASSES);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    };
    if (easy)
      codes_out([&](float v) { return quotient(v, scale, inv); });
    else if (fine)
      codes_out([&](float v) { return v / scale; });
    else
      codes_out([&](float) { return 0.f; });
    if (b == last && (ONE || first == last)) {
      // the rows are kept: those that were the tail's already are there (another grid block may still read the tail
      // otherwise)
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        const int pos = b * KB + r0 + p;
        if (pos < end && (pos >= start || open != b)) *reinterpret_cast<u32x4_t*>(tail + (r0 + p) * D + col) = x[p];
      }
    }
    if (t == 0 && b * KB >= start && tid == 0) c.weights[sh * c.num_blocks + b] = 0.f;
    __syncthreads();
    if (t == 1) {
#pragma unroll
      for (int i = tid; i < D * (KB / 16); i += 256)
        *reinterpret_cast<u32x4_t*>(codes + i * 16) = *reinterpret_cast<const u32x4_t*>(turn + (i / 4) * LD + (i % 4) * 16);
      __syncthreads();                  // LDS is used again
    }
  }

  if constexpr (!ONE) return;
  // Every read of this block has ended (its values were used before the barriers above), so the ticket needs no fence.
  __syncthreads();
  if (tid == 0 && atomicAdd(&c.counters[sh], 1) == 1) {
    c.counters[sh] = 0;
    c.lengths[sh] = end;
    if (grows) c.open_block[sh] = last;
  }
}

// The lengths moved on, and the last block's rows kept: all of them are new where it is not the first.  (Every row's piece on
// its way at once: 256 threads in a loop took 8.3 us for 4 heads.)
constexpr int END_THREADS = 1024;
template <int D>
__global__ __launch_bounds__(END_THREADS) void append_end_kernel(AppendArgs a) {
  const sbsa_cache8& c = a.c;
  const int h = blockIdx.x, s = blockIdx.y;
  const int64_t sh = (int64_t)s * c.num_kv_heads + h, heads = (int64_t)c.num_seqs * c.num_kv_heads;
  int64_t row0;
  int n;
  rows_of(a.offsets, s, a.uniform, a.tokens, row0, n);
  const int held = held_of(c, sh), room = c.num_blocks * KB;
  int start = a.start ? a.start[s] : held;
  start = start < 0 ? 0 : (start < held ? start : held);
  const int end = (int64_t)start + n > room ? room : start + n;
  const int first = start / KB, last = end > start ? (end - 1) / KB : -1;
  __syncthreads();                      // the length is read
  if (threadIdx.x == 0) {
    c.lengths[sh] = end;
    if (last >= 0) c.open_block[sh] = last;
  }
  if (last <= first) return;
  constexpr int CH = D / 8, EACH = 2 * KB * CH / END_THREADS;
  u32x4_t x[EACH];
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int i = threadIdx.x + e * END_THREADS, t = i / (KB * CH), j = i / CH % KB, col = i % CH * 8;
    const int pos = last * KB + j < end ? last * KB + j : end - 1;
    const bf16_t* from = t ? a.v + h * a.v_sh + (row0 + pos - start) * a.v_st : a.k + h * a.k_sh + (row0 + pos - start) * a.k_st;
    x[e] = *reinterpret_cast<const u32x4_t*>(from + col);
  }
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int i = threadIdx.x + e * END_THREADS, t = i / (KB * CH), j = i / CH % KB, col = i % CH * 8;
    if (last * KB + j < end) *reinterpret_cast<u32x4_t*>((bf16_t*)c.tail + ((t * heads + sh) * KB + j) * D + col) = x[e];
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
  float* part_o;               // [Hkv][slots][tile rows][D]
  // Sums of exponentials are kept as (m, l), 2^m l: the logarithm of one would round a weight by 10^-6
  f32x2_t* part_ml;            // [Hkv][slots][tile rows]
  i32x4_t* where;                 // [tokens * Hq]: a row's first slot, its slots, its place in the tile
  f32x2_t* row_ml;             // [tokens * Hq], with 1 / l (accumulating)
  f32x2_t* part_w;             // [tokens * Hq][N][steps of a block]: each one's sum of a row (few rows, accumulating)
  const int32_t* offsets;
  int64_t tokens, uniform;
  int hq, g, tile_queries, tile_rows, slots, target;
  float scale_log2;            // sm_scale * log2(e)
};

// The share of a slot (grid block x): a tile of rows of one sequence, and a run of the blocks that it sees.
struct Share {
  int s, n, q0, held, lo, hi, first, count;
  int64_t row0;
};

// The shares are equal runs of blocks over all tiles (target of them, or whole tiles where target is 0): a
// long sequence gets more of them than a short one.  Every wave works its own out from the sequences' lengths, a lane to
// a sequence, 64 sequences at a time.  False: the slot is left over.
__device__ __forceinline__ bool share_of(const AttendArgs& a, int h, int slot, Share& x) {
  const int lane = threadIdx.x & 63, seqs = a.c.num_seqs;
  auto look = [&](int s, int64_t& row0, int& n, int& held, int& tiles, int& blocks) {
    row0 = 0;
    n = held = tiles = blocks = 0;
    if (s < seqs) {
      rows_of(a.offsets, s, a.uniform, a.tokens, row0, n);
      held = held_of(a.c, (int64_t)s * a.c.num_kv_heads + h);
      tiles = (n + a.tile_queries - 1) / a.tile_queries;
      blocks = (held + KB - 1) / KB;
    }
  };
  int64_t row0;
  int n, held, tiles, blocks;
  look(lane, row0, n, held, tiles, blocks);
  int per = 0x7fffffff;
  if (a.target) {
    int total = tiles * blocks;
    for (int s0 = 64; s0 < seqs; s0 += 64) {
      int64_t r;
      int m, e, t, b;
      look(s0 + lane, r, m, e, t, b);
      total += t * b;
    }
    total = wave_sum_i32_dpp(total);
    per = (total + a.target - 1) / a.target;
    per = per < 4 ? 4 : per;
  }
  int before = 0;
  for (int s0 = 0;; s0 += 64) {
    const int shares = blocks <= per ? 1 : (blocks + per - 1) / per;
    const int mine = tiles * shares;
    const int upto = wave_incl_scan_dpp(mine);
    const unsigned long long past = __ballot(before + upto > slot);
    if (past) {
      const int l = __builtin_amdgcn_readfirstlane(__ffsll((long long)past) - 1);
      x.s = s0 + l;
      x.n = __builtin_amdgcn_readlane(n, l);
      x.held = __builtin_amdgcn_readlane(held, l);
      x.row0 = (int64_t)__builtin_amdgcn_readlane((int)row0, l);       // below 2^24
      const int count = __builtin_amdgcn_readlane(shares, l);
      const int own = before + __builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(mine, l);
      const int tile = (slot - own) / count, part = (slot - own) - tile * count;
      x.q0 = tile * a.tile_queries;
      x.first = slot - part;
      x.count = count;
      // the blocks that the tile's last row sees, of which this is share `part`
      const int last = x.q0 + a.tile_queries < x.n ? x.q0 + a.tile_queries : x.n;
      const int sees = x.held - x.n + last;
      const int all = sees > 0 ? (sees + KB - 1) / KB : 0;
      const int each = (all + count - 1) / count;
      x.lo = part * each;
      x.hi = x.lo + each < all ? x.lo + each : all;
      return true;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
    if (s0 + 64 >= seqs) return false;
    look(s0 + 64 + lane, row0, n, held, tiles, blocks);
  }
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
  static constexpr int STEPS = R == 16 ? 1 : 2; // a block of keys is taken in this many steps (32 rows: registers)
  static constexpr int GROUPS = KB / R / STEPS; // products of R keys in a step
  static constexpr int SEG = 16 * PARTS;        // dims that one 16-byte load of every part covers
  static constexpr int NT = D / R;              // R-dim tiles of O^T
  static constexpr int NI = R * R / 64;         // accumulator values of a lane
  static constexpr float P_SCALE = 0x1p11f, SLACK = 4.f;
  typedef __attribute__((ext_vector_type(NI))) float acc_t;
  typedef u32x4_t kcodes_t[GROUPS][D / SEG];
  static constexpr int KEYS = KB / PARTS / STEPS;       // a lane's keys of a step: 16
  typedef u32x4_t vcodes_t[NT];

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

  // the key of a step's that row r of product g takes
  static __device__ __forceinline__ int key_of(int r, int g) {
    if constexpr (R == 16)
      return (r >> 2) * 16 + g * 4 + (r & 3);
    else
      return ((r >> 2) & 1) * 16 + (r >> 3) * 4 + (r & 3);
  }
  // a lane's first key (of the block's 64) of a step
  static __device__ __forceinline__ int mine(int step, int lane) { return step * (KB / STEPS) + (lane / R) * KEYS; }

  // A block's codes through a buffer resource of its size: the address of a load is a scalar base, one lane
  // offset and a scalar or literal one.  (By pointers the compiler carries 64-bit lane addresses and spills.)
  static __device__ __forceinline__ void load_k(const uint8_t* kb, int step, int lane, kcodes_t& kc) {
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)kb, 0, KB * D, BUFFER_CONFIG);
    if constexpr (R * D > 4096) lane = lane_again();      // the offset made here: registers less to keep
    const int off = (step * (KB / STEPS) + key_of(lane % R, 0)) * D + (lane / R) * 16;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
#pragma unroll
      for (int j = 0; j < D / SEG; ++j)
        kc[g][j] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, off, key_of(0, g) * D + j * SEG, 0);
  }
  static __device__ __forceinline__ void load_v(const uint8_t* vb, int step, int lane, vcodes_t& vc) {
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)vb, 0, KB * D, BUFFER_CONFIG);
    if constexpr (R * D > 4096) lane = lane_again();
    const int off = (lane % R) * KB + mine(step, lane);
#pragma unroll
    for (int t = 0; t < NT; ++t) vc[t] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, off, t * R * KB, 0);
  }

  // scores of a step's keys, times ks; q(j, x) gives the rows' pieces
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

  // a step's scores to probabilities p (fp16, with the values' scale), the state moved on.  seen: how
  // many of the lane's keys of the step its row sees (all: every row every one).  Returns the lane's sum.
  __device__ __forceinline__ float softmax(acc_t (&sc)[GROUPS], float vs, int seen, bool all, u32x4_t (&p)[KEYS / 8]) {
    if (!all) {
#pragma unroll
      for (int g = 0; g < GROUPS; ++g)
#pragma unroll
        for (int i = 0; i < NI; ++i)
          if (g * NI + i >= seen) sc[g][i] = -INFINITY;
    }
    float top = -INFINITY;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
#pragma unroll
      for (int i = 0; i < NI; ++i) top = fmaxf(top, sc[g][i]);
    if constexpr (R == 16) top = max16(top);
    top = max32(top);
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
    for (int x = 0; x < KEYS / 2; ++x) {
      const int i0 = 2 * x, i1 = 2 * x + 1;
      const float p0 = __builtin_amdgcn_exp2f(sc[i0 / NI][i0 % NI] - ref);
      const float p1 = __builtin_amdgcn_exp2f(sc[i1 / NI][i1 % NI] - ref);
      sum += p0 + p1;
      // an unseen key's product is 0 whatever the scale
      const bool h0 = !all && i0 >= seen, h1 = !all && i1 >= seen;
      p[x / 4][x % 4] = pack2h(h0 ? 0.f : p0 * pv, h1 ? 0.f : p1 * pv);
    }
    l += sum;
    return sum;
  }

  // filled: how many of the lane's keys of the step are there (whole: all of every lane)
  __device__ __forceinline__ void values(vcodes_t& vc, const u32x4_t (&p)[KEYS / 8], int filled, bool whole) {
    if (!whole) {
#pragma unroll
      for (int t = 0; t < NT; ++t) vc[t] = clear_past(vc[t], filled);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      u32x4_t w = vc[t];
      asm volatile("" : "+v"(w));
      o[t] = mfma(decode8h<FMT>(w.x, w.y), as_f16x8(p[0]), o[t]);
      o[t] = mfma(decode8h<FMT>(w.z, w.w), as_f16x8(p[1]), o[t]);
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

};

// This lane's row of a tile, and what it sees.
template <int R>
struct LaneRow {
  int r, head, vis, vis_most, vis_least;
  bool there;
  int64_t token;

  __device__ __forceinline__ void find(const AttendArgs& a, int h, const Share& x, int row) {
    r = row;
    const int qi = x.q0 + r / a.g;
    head = h * a.g + r % a.g;
    there = r < a.tile_queries * a.g && qi < x.n;
    token = x.row0 + qi;
    auto sees = [&](int row) {
      const int v = x.held - x.n + x.q0 + row / a.g + 1;
      return v < 0 ? 0 : v;
    };
    vis = there ? sees(r) : 0;
    // the wave's rows are R in a row: the last one that is there sees the most, the first the least
    const int left = (x.n - x.q0 < a.tile_queries ? x.n - x.q0 : a.tile_queries) * a.g;
    const int first = __builtin_amdgcn_readfirstlane(row), last = first + R < left ? first + R - 1 : left - 1;
    vis_most = first < left ? sees(last) : 0;
    vis_least = first < left ? sees(first) : 0x7fffffff;
  }

  // four dims of the row's result: to out, or where its shares are joined
  __device__ __forceinline__ void store(const AttendArgs& a, int h, int slot, const Share& x, int D, int dim, f32x4_t v) const {
    if (x.count == 1) {
      u32x2_t w;
      w.x = pack2bf(v.x, v.y);
      w.y = pack2bf(v.z, v.w);
      *reinterpret_cast<u32x2_t*>(a.out + token * a.o_st + head * a.o_sh + dim) = w;
    } else {
      const int64_t at = ((int64_t)h * a.slots + slot) * a.tile_rows + r;
      *reinterpret_cast<f32x4_t*>(a.part_o + at * D + dim) = v;
    }
  }
  // the row's sum, by one lane of it: without keys it has l = 0
  __device__ __forceinline__ void store_sum(const AttendArgs& a, int h, int slot, const Share& x, float m, float l) const {
    const int64_t row = token * a.hq + head;
    if (a.target) {
      if (slot == x.first) a.where[row] = i32x4_t{x.first, x.count, r, 0};
      a.part_ml[((int64_t)h * a.slots + slot) * a.tile_rows + r] = f32x2_t{m, l};
    }
    if (x.count == 1) finish_row(a, row, m, l);
  }
};

// Few rows per sequence: a tile of R rows over one share of the keys, every fourth block of keys to each
// wave (with 32 rows every fourth half of one: few blocks come to a wave, and halves of them go round more evenly), the
// waves joined through LDS.  The codes go from memory to the registers that the products read, the next block's on their
// way while this one's are used; no barrier and no LDS traffic but the queries'.
//
// Memory bounds it: one token of 16 heads over 131272 keys of 4 heads of 256 dims (269 MB) takes 52 us, 5.2 TB/s, and
// its join 5.6.  5 rows of each of 4 sequences up to 40009 keys (164 MB) take 40 us, 49 with whole blocks to a wave:
// five halves come to each, and the start and the join of the waves show.
template <int D, int FMT, int R>
__global__ __launch_bounds__(256, 2) void attend_keys_kernel(AttendArgs a) {
  using W = WaveRows<D, FMT, R>;
  constexpr int TILE = W::NT * W::NI * 64;          // floats of a wave's O
  constexpr int PIECES = D / W::SEG * 2;
  constexpr int LEFT = R * D > 4096 ? 2 : 4;        // results that the last step joins
  __shared__ __attribute__((aligned(16))) unsigned char smem_keys[LEFT * TILE * sizeof(float)];
  float* fold = reinterpret_cast<float*>(smem_keys);      // after the keys
  u32x4_t* sq = reinterpret_cast<u32x4_t*>(smem_keys);    // before
  __shared__ float sm[4 * 64], sl[4 * 64];
  const sbsa_cache8& c = a.c;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int h = blockIdx.y, slot = blockIdx.x;
  Share sh;
  if (!share_of(a, h, slot, sh)) return;
  LaneRow<R> r;
  r.find(a, h, sh, lane % R);
  const bf16_t* qrow = r.there ? a.q + r.token * a.q_st + r.head * a.q_sh : nullptr;

  W w;
  w.start();
  const int64_t heads = (int64_t)c.num_seqs * c.num_kv_heads;
  const int64_t row = (int64_t)sh.s * c.num_kv_heads + h, base = row * c.num_blocks;
  const uint8_t* codes_k = (const uint8_t*)c.codes_k + base * KB * D;
  const uint8_t* codes_v = (const uint8_t*)c.codes_v + base * KB * D;
  constexpr int STRIDE = 4 / W::STEPS;
  const int step = wave % W::STEPS, first = sh.lo + wave / W::STEPS;
  const int count = sh.hi > first ? (sh.hi - first + STRIDE - 1) / STRIDE : 0;
  // the places and scales of the wave's next 64 blocks: fetched by a lane each, kept in LDS
  __shared__ int s_place[4 * 64];
  __shared__ float s_ks[4 * 64], s_vs[4 * 64];
  auto fetch = [&](int i0, auto&& then) {           // then: what goes on as soon as the places are there
    const int b = first + STRIDE * (i0 + lane);
    int place = 0;
    if (b < sh.hi) {
      place = (int)(place_of(c, row, b) - base);
      s_place[wave * 64 + lane] = place;
    }
    __builtin_amdgcn_wave_barrier();
    then();
    if (b < sh.hi) {
      s_ks[wave * 64 + lane] = c.scales[base + place] * a.scale_log2;
      s_vs[wave * 64 + lane] = c.scales[heads * c.num_blocks + base + place];
    }
    __builtin_amdgcn_wave_barrier();
  };
  auto place_at = [&](int i) {                      // in bytes of codes
    return (int64_t)__builtin_amdgcn_readfirstlane(s_place[wave * 64 + (i & 63)]) * (KB * D);
  };
  typename W::kcodes_t kc;
  typename W::vcodes_t vc;
  if (count > 0) {
    fetch(0, [&] {
      const int64_t at = place_at(0);
      W::load_k(codes_k + at, step, lane, kc);
      W::load_v(codes_v + at, step, lane, vc);
    });
  }
  for (int i = wave; i < PIECES; i += 4) sq[i * 64 + lane] = W::query_piece(qrow, i >> 1, i & 1, lane);
  __syncthreads();                                  // the queries are in LDS
  const int mine = W::mine(step, lane);
  for (int i = 0; i < count; ++i) {
    const int b = first + STRIDE * i;
    const float ksi = uniform(s_ks[wave * 64 + (i & 63)]), vsi = uniform(s_vs[wave * 64 + (i & 63)]);
    if (((i + 1) & 63) == 0) fetch(i + 1, [] {});
    const bool more = i + 1 < count;
    const int64_t next = more ? place_at(i + 1) : 0;
    typename W::acc_t sc[W::GROUPS];
    const int own = R * D > 4096 ? lane_again() : lane;         // a reload from scratch would wait for every load
    W::scores(kc, [&](int j, int x) { return sq[(2 * j + x) * 64 + own]; }, ksi, sc);
    if (more) W::load_k(codes_k + next, step, lane, kc);
    u32x4_t p[W::KEYS / 8];
    float sum = w.softmax(sc, vsi, r.vis - b * KB - mine, (b + 1) * KB <= r.vis_least, p);
    if (a.part_w) {
      // what the row gives to the block's keys here, for the blocks' weights
      if constexpr (R == 16) sum += __shfl_xor(sum, 16, 64);
      sum += __shfl_xor(sum, 32, 64);
      if (r.there && lane < R)
        a.part_w[((r.token * a.hq + r.head) * c.num_blocks + b) * W::STEPS + step] = f32x2_t{w.m, sum};
    }
    w.values(vc, p, sh.held - b * KB - mine, sh.held - b * KB >= KB);
    if (more) W::load_v(codes_v + next, step, lane, vc);
    asm volatile("" ::: "memory");                  // the queries stay in LDS, not in registers
  }
  w.total();
  // The waves' results joined.  Where all four do not fit LDS twice on a compute unit (32 rows of 256 dims),
  // the odd waves' go into the even ones' first.
  auto leave = [&](int at) {
#pragma unroll
    for (int t = 0; t < W::NT; ++t)
#pragma unroll
      for (int i = 0; i < W::NI; ++i) fold[at * TILE + (t * W::NI + i) * 64 + lane] = w.o[t][i];
    sm[at * 64 + lane] = w.m;
    sl[at * 64 + lane] = w.l;
  };
  if constexpr (LEFT == 2) {
    __syncthreads();                                // the queries' place in LDS is used again
    if (wave & 1) leave(wave >> 1);
    __syncthreads();
    if (!(wave & 1)) {
      const int at = wave >> 1;
      const float m1 = sm[at * 64 + lane], l1 = sl[at * 64 + lane];
      const float to = fmaxf(w.m, m1), ref = to == -INFINITY ? 0.f : to;
      float f0 = w.l * __builtin_amdgcn_exp2f(w.m - ref), f1 = l1 * __builtin_amdgcn_exp2f(m1 - ref);
      w.m = to;
      w.l = f0 + f1;
      const float inv = w.l == 0.f ? 0.f : 1.f / w.l;
      f0 *= inv;
      f1 *= inv;
#pragma unroll
      for (int t = 0; t < W::NT; ++t)
#pragma unroll
        for (int i = 0; i < W::NI; ++i)
          w.o[t][i] = w.o[t][i] * f0 + fold[at * TILE + (t * W::NI + i) * 64 + lane] * f1;
      leave(at);                                    // each lane into the place that it read
    }
  } else {
    __syncthreads();
    leave(wave);
  }
  __syncthreads();
  // each wave joins a quarter of the dims
  float top = -INFINITY, f[LEFT], total = 0.f;
#pragma unroll
  for (int x = 0; x < LEFT; ++x) top = fmaxf(top, sm[x * 64 + lane]);
  const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
  for (int x = 0; x < LEFT; ++x) {
    f[x] = sl[x * 64 + lane] * __builtin_amdgcn_exp2f(sm[x * 64 + lane] - ref);
    total += f[x];
  }
  if (!r.there) return;
  const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
  for (int x = 0; x < LEFT; ++x) f[x] *= inv;
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
        float y = fold[at] * f[0] + fold[TILE + at] * f[1];
        if constexpr (LEFT == 4) y += fold[2 * TILE + at] * f[2] + fold[3 * TILE + at] * f[3];
        v[i] = y;
      }
      r.store(a, h, slot, sh, D, W::dim_of(t, q, lane), v);
    }
  }
  if (wave == 0 && lane < R) r.store_sum(a, h, slot, sh, top, total);
}

// Many rows: 32 of them to each wave, the tiles of codes in LDS for all four.  The codes stay 8 bits wide there
// (half the LDS traffic of bf16 tiles, which would keep LDS as busy as the matrix cores) and each wave decodes what it reads;
// a block of keys is taken in two halves of 32, so that two grid blocks fit a compute unit's registers and one's
// softmax runs under the other's products.
//
// 2048 rows of 16 heads at 34777 keys of 4 heads of 256 dims take 1160 us, 980 TFLOP/s (a large bf16 product: 1220 to 1380).
// What is left is vector work, the codes' decoding and the softmax: two waves of a SIMD do not cover it and the latency of
// the LDS reads at every turn, and there are no registers for a third or for reads further ahead.
//
// LDS holds a block's tiles as 16-byte pieces, swizzled so that the 8 lanes of a read's cycle meet
// different banks: piece c of key row r at c ^ key_swizzle(r), piece c of dim row d at c ^ (d / 2) % 4.  They come straight from
// memory (loads into LDS), the next block's while this one is used.
typedef __attribute__((address_space(3))) void lds_void_t;

// 16 bytes per lane from memory straight to LDS, lane l's at lds_addr + 16 l.  In assembly, because the compiler waits for
// the builtin's loads before any LDS read that it cannot tell apart; the kernel waits (vmcnt) before the
// barrier that publishes a tile.  M0 holds the LDS base (a wait state lies between its write and its use); nothing else in the
// kernel uses it.
__device__ __forceinline__ void lds_load16(u32x4_t rsrc, uint32_t lds_addr, uint32_t voffset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(lds_addr), "v"(voffset), "s"(rsrc)
               : "memory", "m0");
}

// A load through the scalar cache, by an address that is the same in every lane (of memory that no block of the launch writes).
template <class T>
__device__ __forceinline__ T scalar_load(const T* p) {
  return *(const __attribute__((address_space(4))) T*)(uintptr_t)p;
}

template <int D, int FMT>
struct RowsTile {
  static constexpr int BYTES = KB * D;                 // of a block's keys, or values
  static constexpr int CH = D / 16;                    // pieces of a key row
  static constexpr int PER_WAVE = BYTES / 1024 / 4;    // loads of 64 pieces by each wave
  static __device__ __forceinline__ int key_swizzle(int r) {
    const int x = (r & 3) | ((r >> 5) & 1) << 2;
    return D == 256 ? x | ((r >> 2) & 1) << 3 : x;
  }
  // Load i of a wave takes pieces (4 i + wave) 64 + lane: rows (4 i + wave) 1024 / D + .., whose swizzle depends on
  // i in the row's bit 5 alone.
  static __device__ __forceinline__ void load(const uint8_t* kb, const uint8_t* vb, unsigned char* to, int wave, int lane) {
    const int p = wave * 64 + lane;
    const int koff = p / CH * D + ((p % CH) ^ key_swizzle(p / CH)) * 16;
    const int voff = p / 4 * KB + ((p % 4) ^ ((p >> 3) & 3)) * 16;
    const uint32_t at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_void_t*)(to + wave * 1024));
    const u32x4_t krs = codes_rsrc(kb), vrs = codes_rsrc(vb);
#pragma unroll
    for (int i = 0; i < PER_WAVE; ++i)
      lds_load16(krs, at + i * 4096, (uint32_t)((koff ^ (key_swizzle(i * 256 / CH) * 16)) + i * 4096));
#pragma unroll
    for (int i = 0; i < PER_WAVE; ++i) lds_load16(vrs, at + BYTES + i * 4096, (uint32_t)(voff + i * 4096));
  }
  static __device__ __forceinline__ u32x4_t codes_rsrc(const uint8_t* p) {
    const uint64_t b = (uint64_t)p;
    u32x4_t r;                                         // raw buffer resource: base, stride 0, bytes, config
    r.x = __builtin_amdgcn_readfirstlane((uint32_t)b);
    r.y = __builtin_amdgcn_readfirstlane((uint32_t)(b >> 32)) & 0xffffu;
    r.z = (uint32_t)BYTES;
    r.w = (uint32_t)BUFFER_CONFIG;
    return r;
  }
};

template <int D, int FMT>
__global__ __launch_bounds__(256, 2) void attend_rows_kernel(AttendArgs a) {
  using T = RowsTile<D, FMT>;
  constexpr int NT = D / 32, STEPS = D / 32;
  constexpr int K_AHEAD = 2, V_AHEAD = 2;
  constexpr float P_LOG2 = 11.f, SLACK = 4.f;          // as in WaveRows
  __shared__ __attribute__((aligned(16))) unsigned char tile[2][2 * T::BYTES];
  const sbsa_cache8& c = a.c;
  const int lane = threadIdx.x & 63, part = lane / 32;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  // late tiles see the most keys: they go first
  const int h = blockIdx.y, slot = (int)(gridDim.x - 1 - blockIdx.x);
  Share sh;
  if (!share_of(a, h, slot, sh)) return;
  LaneRow<32> r;
  r.find(a, h, sh, wave * 32 + lane % 32);
  const bf16_t* qrow = r.there ? a.q + r.token * a.q_st + r.head * a.q_sh : nullptr;
  // the queries in registers, but for what does not fit: that lies in LDS, by wave and lane
  constexpr int KEPT = D == 256 ? STEPS - 2 : STEPS;
  __shared__ u32x4_t sq[KEPT < STEPS ? (STEPS - KEPT) * 2 * 256 : 1];
  bf16x8_t q[KEPT][2];
#pragma unroll
  for (int j = 0; j < STEPS; ++j)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const u32x4_t w = WaveRows<D, FMT, 32>::query_piece(qrow, j, x, lane);
      if (j < KEPT)
        q[j][x] = as_bf16x8(w);
      else
        sq[(2 * (j - KEPT) + x) * 256 + threadIdx.x] = w;
    }
  f32x16_t o[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[t][i] = 0.f;
  float m = -INFINITY, l = 0.f, v_ref = 0.f;

  const int64_t heads = (int64_t)c.num_seqs * c.num_kv_heads;
  const int64_t head_row = (int64_t)sh.s * c.num_kv_heads + h;
  const float* scales_v = c.scales + heads * c.num_blocks;
  auto load = [&](int b, int64_t place) {
    T::load((const uint8_t*)c.codes_k + place * T::BYTES, (const uint8_t*)c.codes_v + place * T::BYTES, tile[b & 1], wave, lane);
  };
  // per-lane places in the tiles: the keys' row of each half (its swizzle does not depend on the half: bits 0, 1, 2
  // and 5 of the row), the values' row of a 32-dim tile
  using W = WaveRows<D, FMT, 32>;
  const int lane_row = lane % 32, krow = ((lane_row >> 2) & 1) * 32 + (lane_row >> 3) * 4 + (lane_row & 3);
  const uint32_t klane = krow * D + ((part ^ T::key_swizzle(krow)) * 16);
  const uint32_t vlane = (lane % 32) * KB + (((2 * part) ^ ((lane >> 1) & 3)) * 16);

  auto place_at = [&](int b) {                         // as place_of
    int t = scalar_load(c.table + head_row * c.num_blocks + (b < sh.hi ? b : sh.hi - 1));
    t = t < 0 ? 0 : t;
    return head_row * c.num_blocks + (t < c.num_blocks ? t : c.num_blocks - 1);
  };
  // places and scales are fetched a block ahead, so that no load is waited for but the tiles'
  int64_t next_place = 0;
  float next_ks = 0.f, next_vs = 0.f;
  if (sh.lo < sh.hi) {
    const int64_t place = place_at(sh.lo);
    next_ks = scalar_load(c.scales + place);
    next_vs = scalar_load(scales_v + place);
    next_place = place_at(sh.lo + 1);
    load(sh.lo, place);
  }
  for (int b = sh.lo; b < sh.hi; ++b) {
    const float ks = uniform(next_ks * a.scale_log2), vs = next_vs;
    const int64_t place = next_place;
    next_ks = scalar_load(c.scales + place);
    next_vs = scalar_load(scales_v + place);
    next_place = place_at(b + 2);
    // this block's tiles are there, and every wave is done with the last block's
    __builtin_amdgcn_s_waitcnt(0x0f70);               // vmcnt(0)
    __syncthreads();
    if (b + 1 < sh.hi) load(b + 1, place);
    if (b * KB >= r.vis_most) continue;
    // a step's or half's piece is a flip of address bits away; laundered, or the compiler keeps every address
    uint32_t kat = (b & 1) * (2 * T::BYTES) + klane, vat = (b & 1) * (2 * T::BYTES) + T::BYTES + vlane;
    asm volatile("" : "+v"(kat));
    asm volatile("" : "+v"(vat));
    const bool all = (b + 1) * KB <= r.vis_least, whole = sh.held - b * KB >= KB;
    const int seen = r.vis - b * KB;
    if (fabsf(vs) > v_ref) {
      const float f = v_ref / fabsf(vs);
      v_ref = uniform(fabsf(vs));
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] *= f;
    }
    // in (0, 1]; below 2^-60 fp16 has nothing left of the block's values, but its keys still count (as do those of
    // a block whose values are not finite)
    float ratio = v_ref > 0.f && vs == vs ? vs / v_ref : 1.f;
    ratio = ratio < 0x1p-60f ? 0x1p-60f : ratio;
    if (vs != vs) {                                    // NaN to every row that sees a value of the block
      const float none = seen > 0 ? vs : 0.f;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] += none;
    }
    const float lift = uniform(P_LOG2 + __builtin_amdgcn_logf(ratio)), drop = uniform(1.f / (ratio * 2048.f));
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      f32x16_t sc;
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[i] = 0.f;
      auto query = [&](int j, int x) {
        return j < KEPT ? q[j < KEPT ? j : 0][x] : as_bf16x8(sq[(2 * (j - KEPT) + x) * 256 + threadIdx.x]);
      };
      auto key_piece = [&](int j) {
        return *reinterpret_cast<const u32x4_t*>(&tile[0][0] + (kat ^ (32u * j)) + 16 * g * D);
      };
      auto value_piece = [&](int t) {
        return *reinterpret_cast<const u32x4_t*>(&tile[0][0] + (vat ^ (16u * g)) + t * 32 * KB);
      };
      // pieces K_AHEAD and V_AHEAD steps ahead, the values' first ones under the softmax; further, and the
      // compiler runs out of registers
      __builtin_amdgcn_s_setprio(1);                   // the products before the other block's softmax: 2 %
      u32x4_t kp[K_AHEAD], vp[V_AHEAD];
#pragma unroll
      for (int j = 0; j < K_AHEAD; ++j) kp[j] = key_piece(j);
#pragma unroll
      for (int j = 0; j < STEPS; ++j) {
        const u32x4_t w = kp[j % K_AHEAD];
        sc = W::mfma(decode8<FMT>(w.x, w.y), query(j, 0), sc);
        sc = W::mfma(decode8<FMT>(w.z, w.w), query(j, 1), sc);
        if (j + K_AHEAD < STEPS) kp[j % K_AHEAD] = key_piece(j + K_AHEAD);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int t = 0; t < V_AHEAD; ++t) vp[t] = value_piece(t);
      __builtin_amdgcn_s_setprio(0);
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        sc[i] *= ks;
        if (!all && part * 32 + g * 16 + i >= seen) sc[i] = -INFINITY;
        top = fmaxf(top, sc[i]);
      }
      top = max32(top);
      if (__ballot(top > m + SLACK)) {
        if (__ballot(top == INFINITY)) {               // as in WaveRows
#pragma unroll
          for (int i = 0; i < 16; ++i) sc[i] = sc[i] == INFINITY ? FLT_MOST : sc[i];
          top = top == INFINITY ? FLT_MOST : top;
        }
        const float to = fmaxf(m, top);
        const float f = m == to ? 1.f : __builtin_amdgcn_exp2f(m - to);
        m = to;
        l *= f;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[t][i] *= f;
      }
      // p times the values' relative scale and 2^11, by the exponent; the sum without them
      const float ref = (m == -INFINITY ? 0.f : m) - lift;
      u32x4_t p[2];
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        float p0 = __builtin_amdgcn_exp2f(sc[i] - ref), p1 = __builtin_amdgcn_exp2f(sc[i + 1] - ref);
        if (!all) {                                    // 0 whatever the scale
          p0 = part * 32 + g * 16 + i >= seen ? 0.f : p0;
          p1 = part * 32 + g * 16 + i + 1 >= seen ? 0.f : p1;
        }
        sum += p0 + p1;
        p[i / 8][i / 2 % 4] = pack2h(p0, p1);
      }
      l += sum * drop;
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        u32x4_t w = vp[t % V_AHEAD];
        if (!whole) w = clear_past(w, sh.held - b * KB - (part * 32 + g * 16));
        o[t] = W::mfma(decode8h<FMT>(w.x, w.y), as_f16x8(p[0]), o[t]);
        o[t] = W::mfma(decode8h<FMT>(w.z, w.w), as_f16x8(p[1]), o[t]);
        if (t + V_AHEAD < NT) vp[t % V_AHEAD] = value_piece(t + V_AHEAD);
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_setprio(0);
    }
  }
  l += __shfl_xor(l, 32, 64);
  if (!r.there) return;
  const float f = l == 0.f ? 0.f : 0x1p-11f / l;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      f32x4_t v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = o[t][4 * x + i] * f * v_ref;
      r.store(a, h, slot, sh, D, W::dim_of(t, x, lane), v);
    }
  if (lane < 32) r.store_sum(a, h, slot, sh, m, l);
}

// Whether a row's shares lie in the workspace.  Rows that no share reached (offsets that do not ascend) have none.
__device__ __forceinline__ bool shares_fit(const AttendArgs& a, const i32x4_t& w) {
  return w.x >= 0 && w.y >= 1 && w.y <= a.slots && w.x <= a.slots - w.y && w.z >= 0 && w.z < a.tile_rows;
}

// The shares joined.  The first blocks of the grid each take 64 dims of a row, 16 threads to a share's 64 dims and every
// 16th share to each (FEW: the 64 dims of 16 rows, every share of a row to its 16 threads); with part_w the others take 256
// blocks of keys of a (sequence, head) and add up what the rows left for each of them.  Latency bounds it: 5.6 us for one
// token's 128 shares of 4 heads.
template <int D, bool FEW>
__global__ __launch_bounds__(256) void join_kernel(AttendArgs a, int join_blocks) {
  const int tid = threadIdx.x, lane = tid & 63;
  const sbsa_cache8& c = a.c;
  if (FEW && (int)blockIdx.x < join_blocks) {
    const int64_t unit = (int64_t)blockIdx.x * 16 + (tid >> 4), row = unit / (D / 64), token = row / a.hq;
    const int d = (int)(unit % (D / 64)) * 64 + (tid & 15) * 4, head = (int)(row % a.hq);
    if (token >= a.tokens || (a.offsets && (token < a.offsets[0] || token >= a.offsets[c.num_seqs]))) return;
    const i32x4_t where = a.where[row];
    if (where.y == 1 || !shares_fit(a, where)) return;
    const int64_t at = ((int64_t)(head / a.g) * a.slots + where.x) * a.tile_rows + where.z;
    const f32x2_t* ml = a.part_ml + at;
    float top = -INFINITY, total = 0.f;
    for (int x = 0; x < where.y; ++x) top = fmaxf(top, ml[(int64_t)x * a.tile_rows].x);
    const float ref = top == -INFINITY ? 0.f : top;
    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
    for (int x = 0; x < where.y; ++x) {
      const f32x2_t v = ml[(int64_t)x * a.tile_rows];
      total += v.y * __builtin_amdgcn_exp2f(v.x - ref);
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    for (int x = 0; x < where.y; ++x) {
      const f32x2_t v = ml[(int64_t)x * a.tile_rows];
      const f32x4_t o = *reinterpret_cast<const f32x4_t*>(a.part_o + (at + (int64_t)x * a.tile_rows) * D + d);
      acc += o * (v.y * __builtin_amdgcn_exp2f(v.x - ref) * inv);
    }
    u32x2_t w;
    w.x = pack2bf(acc.x, acc.y);
    w.y = pack2bf(acc.z, acc.w);
    *reinterpret_cast<u32x2_t*>(a.out + token * a.o_st + head * a.o_sh + d) = w;
    if (d == 0) finish_row(a, row, top, total);
    return;
  }
  if (!FEW && (int)blockIdx.x < join_blocks) {
    const int64_t row = blockIdx.x / (D / 64);
    const int dims = (int)(blockIdx.x % (D / 64)) * 64;
    const int64_t token = row / a.hq;
    const int head = (int)(row % a.hq);
    if (a.offsets && (token < a.offsets[0] || token >= a.offsets[c.num_seqs])) return;
    const i32x4_t where = a.where[row];
    if (where.y == 1 || !shares_fit(a, where)) return; // (a single share wrote the result itself)
    __shared__ f32x4_t fold[16 * 16];
    const int64_t at = ((int64_t)(head / a.g) * a.slots + where.x) * a.tile_rows + where.z;
    const f32x2_t* ml = a.part_ml + at;
    float top = -INFINITY;
    for (int x = lane; x < where.y; x += 64) top = fmaxf(top, ml[(int64_t)x * a.tile_rows].x);
    top = wave_max(top);
    const float ref = top == -INFINITY ? 0.f : top;
    float total = 0.f;
    for (int x = lane; x < where.y; x += 64) {
      const f32x2_t v = ml[(int64_t)x * a.tile_rows];
      total += v.y * __builtin_amdgcn_exp2f(v.x - ref);
    }
    total = wave_sum(total);
    const float inv = total == 0.f ? 0.f : 1.f / total;
    const int d = dims + (tid & 15) * 4;
    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int x = tid >> 4; x < where.y; x += 16) {
      const f32x2_t v = ml[(int64_t)x * a.tile_rows];
      const f32x4_t o = *reinterpret_cast<const f32x4_t*>(a.part_o + (at + (int64_t)x * a.tile_rows) * D + d);
      acc += o * (v.y * __builtin_amdgcn_exp2f(v.x - ref) * inv);      // a share without keys has an O of 0
    }
    fold[tid] = acc;
    __syncthreads();
    if (tid >= 16) return;
    f32x4_t sum = fold[tid];
    for (int x = 1; x < 16; ++x) sum += fold[x * 16 + tid];
    u32x2_t w;
    w.x = pack2bf(sum.x, sum.y);
    w.y = pack2bf(sum.z, sum.w);
    *reinterpret_cast<u32x2_t*>(a.out + token * a.o_st + head * a.o_sh + d) = w;
    if (tid == 0 && dims == 0) finish_row(a, row, top, total);
    return;
  }
  // the blocks' weights: the rows' sums first (8 threads to a row, 32 rows at a time), then a thread per block
  const int per_head = (c.num_blocks + 255) / 256;
  const int i = (int)blockIdx.x - join_blocks, h = i / per_head % c.num_kv_heads, s = i / per_head / c.num_kv_heads;
  const int b = i % per_head * 256 + tid;
  const int64_t sh = (int64_t)s * c.num_kv_heads + h;
  int64_t row0;
  int n;
  rows_of(a.offsets, s, a.uniform, a.tokens, row0, n);
  const int held = held_of(c, sh);
  if (i % per_head * 256 * KB >= held) return;         // the same for the whole block
  __shared__ f32x2_t row_ml[32];
  float sum = 0.f;
  for (int64_t r0 = 0; r0 < (int64_t)n * a.g; r0 += 32) {
    const int64_t r = r0 + (tid >> 3);
    float top = -INFINITY, total = 0.f;
    i32x4_t where = {0, 0, 0, 0};                      // no shares, past the last row
    if (r < (int64_t)n * a.g) where = a.where[(row0 + r / a.g) * a.hq + h * a.g + r % a.g];
    if (!shares_fit(a, where)) where = i32x4_t{0, 0, 0, 0};
    const f32x2_t* ml = a.part_ml + ((int64_t)h * a.slots + where.x) * a.tile_rows + where.z;
    for (int x = tid & 7; x < where.y; x += 8) top = fmaxf(top, ml[(int64_t)x * a.tile_rows].x);
#pragma unroll
    for (int y = 1; y < 8; y <<= 1) top = fmaxf(top, __shfl_xor(top, y, 64));
    const float ref = top == -INFINITY ? 0.f : top;
    for (int x = tid & 7; x < where.y; x += 8) {
      const f32x2_t v = ml[(int64_t)x * a.tile_rows];
      total += v.y * __builtin_amdgcn_exp2f(v.x - ref);
    }
#pragma unroll
    for (int y = 1; y < 8; y <<= 1) total += __shfl_xor(total, y, 64);
    __syncthreads();
    if ((tid & 7) == 0) row_ml[tid >> 3] = f32x2_t{top, total == 0.f ? 0.f : 1.f / total};
    __syncthreads();
    for (int x = 0; x < 32 && r0 + x < (int64_t)n * a.g; ++x) {
      const int qi = (int)((r0 + x) / a.g);
      if (b * KB >= held - n + qi + 1 || b >= c.num_blocks) continue;      // the row does not see the block
      const int steps = a.tile_rows / 16;
      const f32x2_t* w = a.part_w + (((row0 + qi) * a.hq + h * a.g + (r0 + x) % a.g) * c.num_blocks + b) * steps;
      const f32x2_t all = row_ml[x];
      for (int y = 0; y < steps; ++y) sum += w[y].y == 0.f ? 0.f : w[y].y * __builtin_amdgcn_exp2f(w[y].x - all.x) * all.y;
    }
  }
  if (n > 0 && b < c.num_blocks && b * KB < held) c.weights[sh * c.num_blocks + b] += sum;
}

// The attention that each block receives: a wave holds a block of keys and goes over the rows that
// see it, their sums known; one addition per block, so no order of atomics enters.  The keys form leaves the
// sums to its join instead: for many rows, a float pair for each row and block would be more than the keys.  Decoding again for
// every 32 rows bounds it: 130 rows at 65000 keys of 4 heads of 128 dims 86 us, 132 with the rows not loaded ahead.
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
  typename W::kcodes_t kc[W::STEPS];
#pragma unroll
  for (int step = 0; step < W::STEPS; ++step) W::load_k((const uint8_t*)c.codes_k + place * (KB * D), step, lane, kc[step]);
  const float ks = c.scales[place] * a.scale_log2;
  // the rows from the first that sees the block's first key, 32 at a time, the next ones on their way meanwhile
  struct Rows {
    u32x4_t q[D / W::SEG][2];
    f32x2_t all;
    int seen;
  };
  auto fetch = [&](int64_t r0, Rows& x) {
    const int64_t r = r0 + lane % 32;
    const bool there = r < (int64_t)n * a.g;
    const int64_t qi = there ? r / a.g : 0;
    const int head = h * a.g + (int)(r % a.g);
    x.seen = there ? (int)(held - n + qi + 1 - b * KB) : 0;
    const bf16_t* qrow = there ? a.q + (row0 + qi) * a.q_st + head * a.q_sh : nullptr;
    const f32x2_t none = {0.f, 0.f};
    x.all = there ? a.row_ml[(row0 + qi) * a.hq + head] : none;
#pragma unroll
    for (int j = 0; j < D / W::SEG; ++j)
#pragma unroll
      for (int y = 0; y < 2; ++y) x.q[j][y] = W::query_piece(qrow, j, y, lane);
  };
  int first = b * KB - (held - n);
  first = first < 0 ? 0 : first;
  float sum = 0.f;
  Rows rows[2];
  auto add = [&](const Rows& x) {
#pragma unroll
    for (int step = 0; step < W::STEPS; ++step) {
      typename W::acc_t sc[W::GROUPS];
      W::scores(kc[step], [&](int j, int y) { return x.q[j][y]; }, ks, sc);
#pragma unroll
      for (int g = 0; g < W::GROUPS; ++g)
#pragma unroll
        for (int i = 0; i < W::NI; ++i)
          sum += W::mine(step, lane) + g * W::NI + i < x.seen
                     ? __builtin_amdgcn_exp2f(fminf(sc[g][i], FLT_MOST) - x.all.x) * x.all.y
                     : 0.f;
    }
  };
  const int64_t end = (int64_t)n * a.g;
  fetch((int64_t)first * a.g, rows[0]);
  for (int64_t r0 = (int64_t)first * a.g; r0 < end; r0 += 64) {
    if (r0 + 32 < end) fetch(r0 + 32, rows[1]);
    add(rows[0]);
    if (r0 + 32 >= end) break;
    if (r0 + 64 < end) fetch(r0 + 64, rows[0]);
    add(rows[1]);
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
constexpr int EVICT_MOST = SBSA_CACHE8_MAX_BLOCKS / EVICT_THREADS;      // blocks of a thread

// One (sequence, head).  The tables come through LDS into registers (the outputs may be the inputs), a run of 4 to 16 blocks to
// a thread, so that counts need one scan and no ballots; the weight of the last block that stays by three histograms over
// its bits (not negative, so their order is that of the numbers), 11, 11 and 9 of them; then the blocks in their new order
// through LDS and out.  Instructions and barriers bound it (one compute unit to a list): 128 lists of 8192 blocks take
// 14 us, 17.6 with a ballot for every 64 blocks; 4 of 2304 7.2 us and 8.2.
__global__ __launch_bounds__(EVICT_THREADS) void evict_kernel(EvictArgs a) {
  constexpr int BINS = 2048, WAVES = EVICT_THREADS / 64;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem_evict[];
  const int room = a.num_blocks, room4 = (room + 3) / 4 * 4;
  int32_t* tab = reinterpret_cast<int32_t*>(smem_evict);
  uint32_t* bits = reinterpret_cast<uint32_t*>(tab + room4);
  __shared__ int hist[BINS];
  __shared__ int part[WAVES];
  __shared__ int s_bin[2];
  const int64_t sh = blockIdx.x, base = sh * room;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int len = a.lengths[sh];
  len = len < 0 ? 0 : (len < room * KB ? len : room * KB);
  const int open = a.open_block[sh];
  const int n = (len + KB - 1) / KB;
  for (int i = tid; i < room; i += EVICT_THREADS) {
    tab[i] = a.table[base + i];
    bits[i] = __float_as_uint(a.weights[base + i]);
  }
  hist[tid] = 0;
  hist[tid + EVICT_THREADS] = 0;
  __syncthreads();
  const bool cuts = n > a.keep;
  const int stay = cuts ? a.keep : n;
  const int mid0 = a.sink, mid1 = cuts ? n - a.recent : 0;      // the blocks of which some go
  // this thread's blocks, and the keys of those in the middle (0 for a weight that is not above 0)
  const int per = (room + 4 * EVICT_THREADS - 1) / (4 * EVICT_THREADS) * 4, b0 = tid * per;
  u32x4_t t[EVICT_MOST / 4], w[EVICT_MOST / 4], k[EVICT_MOST / 4];
#pragma unroll
  for (int x = 0; x < EVICT_MOST; x += 4) {
    if (x >= per) continue;
    const int at = b0 + x < room4 ? b0 + x : 0;
    t[x / 4] = *reinterpret_cast<const u32x4_t*>(tab + at);
    w[x / 4] = *reinterpret_cast<const u32x4_t*>(bits + at);
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int b = b0 + x + y;
      k[x / 4][y] = b >= mid0 && b < mid1 && __uint_as_float(w[x / 4][y]) > 0.f ? w[x / 4][y] : 0u;
    }
  }
  // a sum over the threads before this one, and the wave's last lane's sum left for the others
  auto before_wave = [&] { return wave_sum_i32_dpp(lane < wave ? part[lane & (WAVES - 1)] : 0); };
  // bound: the key of the last of the heaviest `wanted` of the middle; above: how many are heavier
  uint32_t bound = 0;
  int above = 0;
  const int wanted = a.keep - a.sink - a.recent;
  if (cuts && wanted > 0) {
    constexpr int SHIFT[3] = {20, 9, 0}, WIDTH[3] = {11, 11, 9};
#pragma unroll
    for (int round = 0; round < 3; ++round) {
#pragma unroll
      for (int x = 0; x < EVICT_MOST; ++x) {
        if (x >= per) continue;
        const uint32_t key = k[x / 4][x % 4], digit = (key >> SHIFT[round]) & ((1u << WIDTH[round]) - 1);
        // (digit 0 need not be counted: it is where the bound lies if it is in no other bin)
        if (digit && (round == 0 || key >> (SHIFT[round] + WIDTH[round]) == bound >> (SHIFT[round] + WIDTH[round])))
          atomicAdd(&hist[digit], 1);
      }
      __syncthreads();
      // keys in bins above this thread's pair, from the top: threads in reverse order
      const int hi = BINS - 1 - 2 * tid;
      const int h1 = hist[hi], h0 = hist[hi - 1];
      hist[hi] = 0;
      hist[hi - 1] = 0;
      const int incl = wave_incl_scan_dpp(h1 + h0);
      if (lane == 63) part[wave] = incl;
      __syncthreads();
      const int before = above + incl - h1 - h0 + before_wave();
      if (before < wanted && before + h1 >= wanted) {
        s_bin[0] = hi;
        s_bin[1] = before;
      } else if (before + h1 < wanted && (before + h1 + h0 >= wanted || tid == EVICT_THREADS - 1)) {
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
  const int ties = wanted - above > 0 ? wanted - above : 0;     // of those at the bound, the first that stay
  auto look = [&](int x, bool& sure, bool& tied) {
    const int b = b0 + x;
    const bool middle = b >= mid0 && b < mid1;
    sure = b < n && (!middle || k[x / 4][x % 4] > bound);
    tied = middle && k[x / 4][x % 4] == bound;
  };
  // how many stay for sure (in the upper 16 bits) and how many are at the bound: at most 16384 each
  int mine = 0;
#pragma unroll
  for (int x = 0; x < EVICT_MOST; ++x) {
    if (x >= per) continue;
    bool sure, tied;
    look(x, sure, tied);
    mine += (sure ? 1 << 16 : 0) + (tied ? 1 : 0);
  }
  const int incl = wave_incl_scan_dpp(mine);
  if (lane == 63) part[wave] = incl;
  __syncthreads();                                    // and every thread has its blocks from LDS
  const int before = before_wave() + incl - mine;
  int seen = before & 0xffff, at = (before >> 16) + (seen < ties ? seen : ties);
#pragma unroll
  for (int x = 0; x < EVICT_MOST; ++x) {
    if (x >= per) continue;
    const int b = b0 + x;
    bool sure, tied;
    look(x, sure, tied);
    const bool here = sure || (tied && seen < ties);
    if (b < room) {
      const int to = here ? at : (b < n ? stay + b - at : b);
      tab[to] = (int32_t)t[x / 4][x % 4];
      bits[to] = here ? w[x / 4][x % 4] : 0u;
      if (b == open) a.open_out[sh] = here ? to : -1;
    }
    at += here;
    seen += tied;
  }
  __syncthreads();
  for (int i = tid; i < room; i += EVICT_THREADS) {
    a.table_out[base + i] = tab[i];
    a.weights_out[base + i] = __uint_as_float(bits[i]);
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
  if (grid.x == 2) {
    hipLaunchKernelGGL((append_kernel<D, FMT, true>), grid, dim3(256), 0, stream, a);
  } else {
    hipLaunchKernelGGL((append_kernel<D, FMT, false>), grid, dim3(256), 0, stream, a);
    hipLaunchKernelGGL((append_end_kernel<D>), dim3(grid.y, grid.z), dim3(END_THREADS), 0, stream, a);
  }
}

// How a call's rows go over the grid.
struct AttendPlan {
  bool keys;                 // the waves of a block share its rows and split its keys
  int tile_rows, tile_queries;
  int target;                // shares per KV head to aim for; 0: whole tiles
  int64_t slots;             // grid blocks per KV head
};

AttendPlan plan_attend(const sbsa_cache8* c, int num_q_heads, int64_t tokens, int64_t max_rows, bool ragged) {
  AttendPlan p;
  const int g = num_q_heads / c->num_kv_heads;
  const int64_t uniform = tokens / c->num_seqs;
  const int64_t most = ragged ? (max_rows < 1 || max_rows > tokens ? tokens : max_rows) : uniform;
  // Up to 32 rows of a sequence to a KV head, the waves split the keys; with more they split the rows.  (20 rows of 4 sequences up
  // to 40009 keys, D = 256: 47.8 us so, 53.5 in a tile of 128 rows; of 8 up to 16384, D = 128: 24.5 and 30.7.)  Up to 16
  // rows, in tiles of 16: 41.7 us for 16 rows where 20 take 47.8.
  p.keys = most * g <= 32;
  p.tile_rows = !p.keys ? 128 : most * g <= 16 ? 16 : 32;
  p.tile_queries = p.tile_rows / g;
  const int64_t tiles = ragged ? tokens / p.tile_queries + c->num_seqs
                               : (uniform + p.tile_queries - 1) / p.tile_queries * c->num_seqs;
  // The keys are shared out until there are two grid blocks for each of the card's 256 compute units.  (One token at
  // 131272 keys: 512 shares 60.7 us, 768 67, 1024 65, 1536 70.)  For tiles of 128 rows there are 1024 where the tiles alone
  // are 512 and more, or their last ones run alone: an 8192-token chunk at 16384 keys 885 us with 512 and 695 with 1024,
  // but a 512-token one at 16000 keys 178 and 221.
  // Up to 20 blocks of 128 dims or 10 of 256 stay whole, which saves the join (one token, 18 blocks of 128: 13.8 us so and
  // 14.0 to 15.2 shared, 29: 20.7 and 15.5; 18 of 256: 18.6 and 14.6 to 15.8).
  // No more shares than the room can fill: left-over grid blocks put the others two to a compute unit (57 blocks of 256
  // dims: 19.4 us with them, 15.8 without).
  const int64_t heads = c->num_kv_heads;
  p.target = 0;
  const int64_t want = p.keys || tiles * heads < 512 ? 512 : 1024;
  if (tiles * heads < want && c->num_blocks * c->head_dim > 20 * 128) {
    const int64_t useful = tiles * ((c->num_blocks + 3) / 4);     // of 4 blocks, a share's least
    p.target = (int)std::max<int64_t>(1, std::min(want / heads, useful));
  }
  p.slots = tiles + p.target;
  return p;
}

// The workspace's parts, in floats: the shares' O and sums, where each row's shares lie, the rows' sums, and each
// row's sums block by block.
struct AttendSpace {
  size_t o, part, where, row, w;
  size_t bytes() const { return (o + part + where + row + w) * sizeof(float); }
};

AttendSpace attend_space(const AttendPlan& p, const sbsa_cache8* c, int64_t tokens, int num_q_heads, bool accumulate) {
  const size_t rows = (size_t)tokens * num_q_heads, shares = p.target ? (size_t)c->num_kv_heads * p.slots * p.tile_rows : 0;
  AttendSpace x;
  x.o = shares * c->head_dim;
  x.part = 2 * shares;
  x.where = p.target ? 4 * rows : 0;
  x.row = accumulate && !(p.keys && p.target) ? (2 * rows + 3) / 4 * 4 : 0;
  x.w = accumulate && p.keys && p.target ? 2 * rows * c->num_blocks * (p.tile_rows / 16) : 0;
  return x;
}

// Few shares of many rows are joined, or many of few: 512 blocks of 16 row pieces fill the card (a 512-token chunk at
// 16000 keys 177 us so, 203 with a block per piece; 16 sequences' tokens at 8192 keys 42 so, 36 with a block per piece).
bool few_shares(const sbsa_cache8* c, int64_t tokens, int num_q_heads) {
  return tokens * num_q_heads * (c->head_dim / 64) >= 8192;
}

int64_t join_blocks(const sbsa_cache8* c, int64_t tokens, int num_q_heads) {
  const int64_t pieces = tokens * num_q_heads * (c->head_dim / 64);
  return few_shares(c, tokens, num_q_heads) ? (pieces + 15) / 16 : pieces;
}

int64_t weigh_blocks(const sbsa_cache8* c) {
  return (int64_t)((c->num_blocks + 255) / 256) * c->num_kv_heads * c->num_seqs;
}

template <int D, int FMT>
void launch_attend(const AttendArgs& a, const AttendPlan& p, int accumulate, hipStream_t stream) {
  const dim3 grid((unsigned)p.slots, (unsigned)a.c.num_kv_heads);
  if (!p.keys)
    hipLaunchKernelGGL((attend_rows_kernel<D, FMT>), grid, dim3(256), 0, stream, a);
  else if (p.tile_rows == 16)
    hipLaunchKernelGGL((attend_keys_kernel<D, FMT, 16>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((attend_keys_kernel<D, FMT, 32>), grid, dim3(256), 0, stream, a);
  if (p.target) {
    const int64_t join = join_blocks(&a.c, a.tokens, a.hq), weigh = a.part_w ? weigh_blocks(&a.c) : 0;
    if (few_shares(&a.c, a.tokens, a.hq))
      hipLaunchKernelGGL((join_kernel<D, true>), dim3((unsigned)(join + weigh)), dim3(256), 0, stream, a, (int)join);
    else
      hipLaunchKernelGGL((join_kernel<D, false>), dim3((unsigned)(join + weigh)), dim3(256), 0, stream, a, (int)join);
  }
  if (accumulate && !a.part_w)
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
  const dim3 grid((unsigned)(2 * blocks), (unsigned)cache->num_kv_heads, (unsigned)cache->num_seqs);
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
  // a grid's threads are below 2^32: fewer than 2^24 blocks of 256
  if (p.slots >= (1 << 24) || (p.target && join_blocks(cache, tokens, num_q_heads) + weigh_blocks(cache) >= (1 << 24)))
    return SBSA_ERR_UNSUPPORTED;
  const AttendSpace space = attend_space(p, cache, tokens, num_q_heads, accumulate != 0);
  if (workspace_bytes < space.bytes()) return SBSA_ERR_CAPACITY;
  if (space.bytes() > 0 && (!workspace || (uintptr_t)workspace % 16)) return SBSA_ERR_ARG;
  AttendArgs a;
  a.c = *cache;
  a.q = (const bf16_t*)q; a.q_st = q_st; a.q_sh = q_sh;
  a.out = (bf16_t*)out; a.o_st = o_st; a.o_sh = o_sh; a.lse = lse;
  a.part_o = (float*)workspace;
  float* at = a.part_o + space.o;
  a.part_ml = (f32x2_t*)at;
  at += space.part;
  a.where = (i32x4_t*)at;
  at += space.where;
  a.row_ml = space.row ? (f32x2_t*)at : nullptr;
  at += space.row;
  a.part_w = space.w ? (f32x2_t*)at : nullptr;
  a.offsets = offsets; a.tokens = tokens; a.uniform = tokens / cache->num_seqs;
  a.hq = num_q_heads; a.g = num_q_heads / cache->num_kv_heads;
  a.tile_queries = p.tile_queries; a.tile_rows = p.tile_rows; a.slots = (int)p.slots; a.target = p.target;
  a.scale_log2 = sm_scale * LOG2E;
  const bool e4m3 = cache->format == SBSA_CACHE8_E4M3;
  if (cache->head_dim == 128)
    e4m3 ? launch_attend<128, SBSA_CACHE8_E4M3>(a, p, accumulate, stream)
         : launch_attend<128, SBSA_CACHE8_INT8>(a, p, accumulate, stream);
  else
    e4m3 ? launch_attend<256, SBSA_CACHE8_E4M3>(a, p, accumulate, stream)
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
  const size_t lds = (size_t)(num_blocks + 3) / 4 * 32;
  if (lds > 48 * 1024 && hipFuncSetAttribute(reinterpret_cast<const void*>(evict_kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess)
    return SBSA_ERR_LAUNCH;
  hipLaunchKernelGGL(evict_kernel, dim3((unsigned)((int64_t)num_seqs * num_kv_heads)), dim3(EVICT_THREADS), lds, stream, a);
  SBSA_CHECK_LAUNCH();
  return SBSA_OK;
}
