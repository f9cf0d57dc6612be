// Rotary positions of a layer's queries and keys, one launch for both.
//
// A pair (a, b) turns by t = position x frequency.  The angle is kept as a fraction of a
// turn in 64-bit fixed point: position x turns mod 2^64 loses nothing at any position (in
// fp32 the angle of position 10^6 would be off by 0.06), and the sine unit takes turns.
//
// A thread takes a unit (VEC pairs: two vectors of VEC values; or VEC values that pass) of one token in
// HEADS heads, every HEADS-th group of them to a thread: the sines of its pairs are made once for HEADS heads, and its
// loads are all on their way before the first is used.  The work is a row of items over all threads, so
// that no thread is left over whatever the head count and the rotated share.
//
// Memory bounds it: 32768 tokens of 16 + 4 heads of 256 dims (671 MB) take 145 us, 4.6 TB/s.  One token takes 3.2 us, which is
// the chain of its loads (position, frequency, row).
#include "sbsa_common.h"

namespace {

struct RotaryArgs {
  const bf16_t* q;
  const bf16_t* k;
  bf16_t* qo;
  bf16_t* ko;
  int64_t q_st, q_sh, k_st, k_sh, qo_st, qo_sh, ko_st, ko_sh;
  const void* positions;
  int64_t pos_axis, pos_stride;
  const uint64_t* turns;
  const uint8_t* axes;
  float gain;
  int pos_bytes, inverse;
  int hq, hkv, rotary_dim, units, rot_units, groups;
  uint32_t items;
};

template <int VEC>
__device__ __forceinline__ void load_vec(const bf16_t* p, bf16_t (&x)[VEC]) {
  if constexpr (VEC == 8) {
    const u32x4_t v = *reinterpret_cast<const u32x4_t*>(p);
    __builtin_memcpy(x, &v, 16);
  } else if constexpr (VEC == 2) {
    const uint32_t v = *reinterpret_cast<const uint32_t*>(p);
    __builtin_memcpy(x, &v, 4);
  } else {
    x[0] = *p;
  }
}

template <int VEC>
__device__ __forceinline__ void store_vec(bf16_t* p, const bf16_t (&x)[VEC]) {
  if constexpr (VEC == 8) {
    u32x4_t v;
    __builtin_memcpy(&v, x, 16);
    *reinterpret_cast<u32x4_t*>(p) = v;
  } else if constexpr (VEC == 2) {
    uint32_t v;
    __builtin_memcpy(&v, x, 4);
    *reinterpret_cast<uint32_t*>(p) = v;
  } else {
    *p = x[0];
  }
}

template <int VEC, bool INTERLEAVED, int HEADS>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  // item = (token, group of heads, unit)
  const uint32_t item = blockIdx.x * 256u + threadIdx.x;
  if (item >= a.items) return;
  const uint32_t row = item / (uint32_t)a.units, u = item - row * (uint32_t)a.units;
  const int64_t tok = row / (uint32_t)a.groups;
  const int group = (int)(row - (uint32_t)tok * (uint32_t)a.groups);
  const bool rot = (int)u < a.rot_units;
  // the two vectors' places: (i, i + rotary_dim/2), neighbours, or one that passes
  const int d0 = rot ? (INTERLEAVED ? 2 * VEC * (int)u : VEC * (int)u) : a.rotary_dim + VEC * ((int)u - a.rot_units);
  const int d1 = INTERLEAVED ? d0 + VEC : d0 + a.rotary_dim / 2;
  bf16_t x[HEADS][VEC], y[HEADS][VEC];
#pragma unroll
  for (int j = 0; j < HEADS; ++j) {
    const int h = group + j * a.groups;
    if (h < a.hq + a.hkv) {
      const bf16_t* in = h < a.hq ? a.q + tok * a.q_st + h * a.q_sh : a.k + tok * a.k_st + (h - a.hq) * a.k_sh;
      load_vec<VEC>(in + d0, x[j]);
      if (rot) load_vec<VEC>(in + d1, y[j]);
    }
  }
  float c[VEC], s[VEC];
  if (rot) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int pair = VEC * (int)u + i;
      const int64_t at = (a.axes ? (int64_t)a.axes[pair] * a.pos_axis : 0) + tok * a.pos_stride;
      const int64_t pos = a.pos_bytes == 8 ? reinterpret_cast<const int64_t*>(a.positions)[at]
                                           : (int64_t)reinterpret_cast<const int32_t*>(a.positions)[at];
      const uint64_t angle = (uint64_t)pos * a.turns[pair];
      const float t = (float)(int32_t)(angle >> 32) * 0x1p-32f;      // in [-1/2, 1/2] turns
      c[i] = __builtin_amdgcn_cosf(t) * a.gain;
      s[i] = __builtin_amdgcn_sinf(a.inverse ? -t : t) * a.gain;
    }
  }
#pragma unroll
  for (int j = 0; j < HEADS; ++j) {
    const int h = group + j * a.groups;
    if (h < a.hq + a.hkv) {
      bf16_t* out = h < a.hq ? a.qo + tok * a.qo_st + h * a.qo_sh : a.ko + tok * a.ko_st + (h - a.hq) * a.ko_sh;
      if (rot) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          // where the pairs are neighbours, x and y are 2 VEC values in a row
          bf16_t& pa = !INTERLEAVED ? x[j][i] : 2 * i < VEC ? x[j][(2 * i) % VEC] : y[j][(2 * i) % VEC];
          bf16_t& pb = !INTERLEAVED ? y[j][i] : 2 * i + 1 < VEC ? x[j][(2 * i + 1) % VEC] : y[j][(2 * i + 1) % VEC];
          const float fa = bf2f(pa), fb = bf2f(pb);
          pa = f2bf(fa * c[i] - fb * s[i]);
          pb = f2bf(fb * c[i] + fa * s[i]);
        }
        store_vec<VEC>(out + d1, y[j]);
      }
      store_vec<VEC>(out + d0, x[j]);
    }
  }
}

bool aligned(const void* p, int64_t st, int64_t sh, int vec) {
  return ((uintptr_t)p % (2 * vec)) == 0 && st % vec == 0 && sh % vec == 0;
}

template <int VEC, int HEADS>
void launch_heads(RotaryArgs a, int64_t rows, int interleaved, hipStream_t stream) {
  a.groups = (a.hq + a.hkv + HEADS - 1) / HEADS;
  a.items = (uint32_t)(rows * a.groups);
  const dim3 grid((a.items + 255) / 256);
  if (interleaved)
    hipLaunchKernelGGL((rotary_kernel<VEC, true, HEADS>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((rotary_kernel<VEC, false, HEADS>), grid, dim3(256), 0, stream, a);
}

// False: more items than 32 bits count.
template <int VEC>
bool launch_rotary(RotaryArgs a, int64_t tokens, int head_dim, bool in_place, int interleaved, hipStream_t stream) {
  a.rot_units = a.rotary_dim / (2 * VEC);
  // what passes is there already where the outputs are the inputs
  a.units = a.rot_units + (in_place ? 0 : (head_dim - a.rotary_dim) / VEC);
  const int64_t rows = tokens * a.units;
  if (rows * (a.hq + a.hkv) >= (1ll << 32) - 256) return false;
  // a thread per head until there are threads for half of the card's 524288 places, then four heads to each (one token:
  // 3.2 us with one, 4.2 with four; 3001 tokens of 10 heads 7.5 and 7.3; 32768 of 20 heads 293 and 149)
  if (rows * (a.hq + a.hkv) <= 262144)
    launch_heads<VEC, 1>(a, rows, interleaved, stream);
  else
    launch_heads<VEC, 4>(a, rows, interleaved, stream);
  return true;
}

}  // namespace

extern "C" int sbsa_rotary(const void* q, int64_t q_st, int64_t q_sh, void* q_out, int64_t qo_st, int64_t qo_sh,
                           int num_q_heads, const void* k, int64_t k_st, int64_t k_sh, void* k_out, int64_t ko_st,
                           int64_t ko_sh, int num_kv_heads, const void* positions, int pos_bytes,
                           int64_t pos_axis_stride, int64_t pos_stride, int64_t tokens, int head_dim, int rotary_dim,
                           int interleaved, const uint64_t* turns, const uint8_t* axes, float gain, int inverse,
                           hipStream_t stream) {
  if (!turns || num_q_heads < 1 || num_kv_heads < 0 || tokens < 0 ||
      (tokens > 0 && (!q || !q_out || !positions || (num_kv_heads > 0 && (!k || !k_out)))) ||
      (pos_bytes != 4 && pos_bytes != 8) || rotary_dim < 2 || rotary_dim % 2 || rotary_dim > head_dim || !(gain > 0.f))
    return SBSA_ERR_ARG;
  if (head_dim > 512 || tokens >= (1 << 24)) return SBSA_ERR_UNSUPPORTED;
  if (tokens == 0) return SBSA_OK;
  RotaryArgs a;
  a.q = (const bf16_t*)q; a.k = (const bf16_t*)k; a.qo = (bf16_t*)q_out; a.ko = (bf16_t*)k_out;
  a.q_st = q_st; a.q_sh = q_sh; a.k_st = k_st; a.k_sh = k_sh;
  a.qo_st = qo_st; a.qo_sh = qo_sh; a.ko_st = ko_st; a.ko_sh = ko_sh;
  a.positions = positions; a.pos_axis = pos_axis_stride; a.pos_stride = pos_stride; a.pos_bytes = pos_bytes;
  a.turns = turns; a.axes = axes; a.gain = inverse ? 1.f / gain : gain; a.inverse = inverse;
  a.hq = num_q_heads; a.hkv = num_kv_heads; a.rotary_dim = rotary_dim;
  const bool in_place = q == q_out && q_st == qo_st && q_sh == qo_sh &&
                        (num_kv_heads == 0 || (k == k_out && k_st == ko_st && k_sh == ko_sh));
  auto fits = [&](int vec) {
    return rotary_dim % (2 * vec) == 0 && (head_dim - rotary_dim) % vec == 0 && aligned(q, q_st, q_sh, vec) &&
           aligned(q_out, qo_st, qo_sh, vec) &&
           (num_kv_heads == 0 || (aligned(k, k_st, k_sh, vec) && aligned(k_out, ko_st, ko_sh, vec)));
  };
  // pieces of 16 bytes where sizes and alignment allow them, else of 4 (32768 tokens: 149 us, 271 with 4), else single values
  const bool ok = fits(8)   ? launch_rotary<8>(a, tokens, head_dim, in_place, interleaved, stream)
                  : fits(2) ? launch_rotary<2>(a, tokens, head_dim, in_place, interleaved, stream)
                            : launch_rotary<1>(a, tokens, head_dim, in_place, interleaved, stream);
  if (!ok) return SBSA_ERR_UNSUPPORTED;
  SBSA_CHECK_LAUNCH();
  return SBSA_OK;
}
