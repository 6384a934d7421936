// The 8-bit paged pool: e4m3 codes and one power-of-two scale per (block, kv
// head), shared by the kernels that write, read and attend over it.
//
// A value is code * 2^e, e in [kExpMin, kExpMax]. The range is the one for which
// every value is an fp16 number: 2^-9 (e4m3's smallest step) * 2^-15 is fp16's
// smallest step, and codes at e = 8 stop at 240 (240 * 2^8 = 61440; the next code,
// 256, would be 2^16). Sources are fp16, so no smaller exponent would hold a row
// more exactly either.
#pragma once

#include "pa_common.h"

namespace pa {
namespace fp8 {

constexpr int kExpMin = -15;
constexpr int kExpMax = 8;
constexpr float kMaxValue = 61440.f;

// 2^e for e of fp32's normal range.
__device__ inline float exp2i(int e) { return __builtin_bit_cast(float, (e + 127) << 23); }

// The exponent of a stored scale, kept in range whatever the pool holds.
__device__ inline int scale_exp(float s) {
  const int e = (int)((__builtin_bit_cast(uint32_t, s) >> 23) & 255u) - 127;
  return e < kExpMin ? kExpMin : (e > kExpMax ? kExpMax : e);
}

// Smallest exponent of the range with amax <= 448 * 2^e (448, e4m3's largest
// value, is 1.75 * 2^8): adding 0x1fffff carries into the exponent exactly where
// the mantissa is above 1.75. amax is at most kMaxValue.
__device__ inline int exp_for(float amax) {
  const int e = (int)((__builtin_bit_cast(uint32_t, amax) + 0x1fffffu) >> 23) - 127 - 8;
  return e < kExpMin ? kExpMin : (e > kExpMax ? kExpMax : e);
}

// Two products rounded to e4m3 (to nearest, ties to even) into the low or high half
// of w. The products must be at most 448 in magnitude, or NaN.
template <bool HI>
__device__ inline int to_codes(float a, float b, int w) {
  return __builtin_amdgcn_cvt_pk_fp8_f32(a, b, w, HI);
}

// Codes of a 32-bit word's low or high half times scale (a power of two) as fp16.
template <bool HI>
__device__ inline f16x2 from_codes(unsigned w, float scale) {
  return __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, HI));
}

__device__ inline f16x8 from_codes8(unsigned lo, unsigned hi, float scale) {
  const f16x2 a = from_codes<false>(lo, scale), b = from_codes<true>(lo, scale);
  const f16x2 c = from_codes<false>(hi, scale), d = from_codes<true>(hi, scale);
  return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// What each sequence's rows and positions come from. qstart null: one row per
// sequence, row b.
struct Rows {
  const int32_t* bt;
  int64_t bt_sb, bt_sk;
  const int32_t* lens;
  const int32_t* qstart;
  int num_seqs, num_tokens, bs, num_blocks, max_blocks;
};

// First row of sequence b (b = num_seqs: one past the last row), kept in range.
__device__ inline int row_start(const Rows& r, int b) {
  if (!r.qstart) return b;
  const int q = r.qstart[b];
  return q < 0 ? 0 : (q > r.num_tokens ? r.num_tokens : q);
}

// Last b of [0, n) with key(b) <= x for a non-decreasing key (0 when there is none),
// found by a wavefront: 64 candidates a step.
template <typename Key>
__device__ inline int wave_search(int n, int x, int lane, Key key) {
  int lo = 0, len = n;
  while (len > 1) {
    const int step = (len + 63) / 64;
    const int at = lane * step;
    const uint64_t m = __ballot(at < len && key(lo + (at < len ? at : 0)) <= x);
    const int k = m ? 63 - (int)__builtin_clzll(m) : 0;
    lo += k * step;
    len = len - k * step < step ? len - k * step : step;
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

struct WriteArgs {
  Rows r;
  const uint16_t* src[2];  // key, value
  int64_t s_t[2], s_h[2], s_d[2];
  uint8_t* cache[2];
  int64_t c_sb[2], c_st[2], c_sh[2];
  float* scale[2];
  int64_t x_sb[2], x_sh[2];
  int hkv, D, slots;
};

struct ReadArgs {
  Rows r;
  const uint8_t* cache[2];
  int64_t c_sb[2], c_st[2], c_sh[2];
  const float* scale[2];
  int64_t x_sb[2], x_sh[2];
  f16* out[2];
  int64_t o_t[2], o_h[2];
  int hkv, D;
};

}  // namespace fp8
}  // namespace pa
