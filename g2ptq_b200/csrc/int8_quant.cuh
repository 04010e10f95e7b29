// Quantization of a token's row to int8: the scale from the largest magnitude,
// the codes of units of 16 elements.
#pragma once

#include <type_traits>

#include "rows.cuh"

namespace g2q {
namespace i8 {

using rows::of_f;
using rows::to_f;

constexpr unsigned kInfBits = 0x7f800000u;

// Sixteen consecutive elements of a row, raw; missing ones (beyond `have`) are zero.
template <typename S>
struct Unit {
  static constexpr int W = 16 * (int)sizeof(S) / 4;  // 32-bit words
  uint32_t raw[W];

  __device__ __forceinline__ void load(const S* p) {
#pragma unroll
    for (int i = 0; i < W / 4; ++i) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(p) + i);
      raw[4 * i] = v.x;
      raw[4 * i + 1] = v.y;
      raw[4 * i + 2] = v.z;
      raw[4 * i + 3] = v.w;
    }
  }
  // the same from any address
  __device__ __forceinline__ void load_any(const S* p) {
    if (sizeof(S) == 4 || (reinterpret_cast<uintptr_t>(p) & 3) == 0) {
#pragma unroll
      for (int i = 0; i < W; ++i) raw[i] = __ldg(reinterpret_cast<const uint32_t*>(p) + i);
    } else {
      const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
      for (int i = 0; i < W; ++i)
        raw[i] = (uint32_t)__ldg(h + 2 * i) | (uint32_t)__ldg(h + 2 * i + 1) << 16;
    }
  }
  __device__ __forceinline__ void load_part(const S* p, int have) {
    S e[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) e[i] = i < have ? p[i] : of_f<S>(0.f);
    memcpy(raw, e, sizeof(raw));
  }
  __device__ __forceinline__ float at(int i) const {
    if constexpr (sizeof(S) == 4) {
      return __uint_as_float(raw[i]);
    } else if constexpr (std::is_same_v<S, __nv_bfloat16>) {
      return __uint_as_float(i % 2 ? raw[i / 2] & 0xffff0000u : raw[i / 2] << 16);
    } else {
      __half2 h;
      memcpy(&h, &raw[i / 2], 4);
      return i % 2 ? __high2float(h) : __low2float(h);
    }
  }
  // the largest magnitude: the bits of a non-negative number order like an
  // unsigned integer, infinities and NaN at the top.  16-bit types: the two
  // halves of a word side by side, merged by top_of.
  __device__ __forceinline__ unsigned top_bits() const {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < W; ++i)
      m = sizeof(S) == 4 ? max(m, raw[i] & 0x7fffffffu) : __vmaxu2(m, raw[i] & 0x7fff7fffu);
    return m;
  }
};

// The larger of two such values
template <typename S>
__device__ __forceinline__ unsigned max_bits(unsigned a, unsigned b) {
  return sizeof(S) == 4 ? max(a, b) : __vmaxu2(a, b);
}

// fp32 bits of the magnitude that top_bits collected
template <typename S>
__device__ __forceinline__ unsigned top_of(unsigned m) {
  if constexpr (sizeof(S) == 4) {
    return m;
  } else {
    const uint16_t h = (uint16_t)max(m & 0xffffu, m >> 16);
    S v;
    memcpy(&v, &h, 2);
    return __float_as_uint(to_f<S>(v));
  }
}

// What a row's codes are made with: the scale, and factors just below and above
// its reciprocal, so that the real quotient v / scale lies between the products
// v * below and v * above.
struct RowScale {
  float scale, below, above;
};

constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: a sum's low bits are the integer's

// The real quotient's rounding, ties to even, where it lies next to the
// half-integer between the neighbouring integers of a and b (sums with kMagic, like
// the result): the sign of the exactly rounded residual v - h * scale tells on
// which side.  Of the smallest scales twice that: it is a multiple of 2^-150, which
// alone would round to zero.
__device__ __forceinline__ uint32_t settle(float v, float scale, float a, float b) {
  const float lo = fminf(a, b), hi = fmaxf(a, b), n = lo - kMagic;
  float res = fmaf(-(n + 0.5f), scale, v);
  if (scale < 1e-36f) res = fmaf(-(n + n + 1.f), scale, v + v);
  const float even = (__float_as_uint(lo) & 1) ? hi : lo;
  return __float_as_uint(res > 0.f ? hi : (res < 0.f ? lo : even));
}

// Codes of a unit, four to a word: round(v / scale) of the real quotient.  Where
// its two bounds round to the same integer the quotient does too; the others are
// settled one by one.  They are not that rare: in 16-bit inputs many values are
// exactly half of the row's largest one, whose quotient is 63.5 but for the
// scale's own rounding.
template <typename S>
__device__ __forceinline__ void unit_codes(const Unit<S>& u, const RowScale& rs, uint32_t (&w)[4]) {
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    uint32_t a[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float v = u.at(4 * g + i);
      a[i] = __float_as_uint(fmaf(v, rs.below, kMagic));
      b[i] = __float_as_uint(fmaf(v, rs.above, kMagic));
    }
    const uint32_t wa =
        __byte_perm(__byte_perm(a[0], a[1], 0x0040), __byte_perm(a[2], a[3], 0x0040), 0x5410);
    const uint32_t wb =
        __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    w[g] = wa;
    uint32_t differ = wa ^ wb;
    while (differ) {
      const int i = (__ffs(differ) - 1) / 8;
      const float v01 = i & 1 ? u.at(4 * g + 1) : u.at(4 * g);
      const float v23 = i & 1 ? u.at(4 * g + 3) : u.at(4 * g + 2);
      const float v = i & 2 ? v23 : v01;
      const uint32_t code = settle(v, rs.scale, fmaf(v, rs.below, kMagic), fmaf(v, rs.above, kMagic));
      const uint32_t mask = 255u << (8 * i);
      w[g] = (w[g] & ~mask) | ((code << (8 * i)) & mask);
      differ &= ~mask;
    }
  }
}

template <typename S>
__device__ __forceinline__ void store_codes(int8_t* dst, const Unit<S>& u, int have, bool vec,
                                            const RowScale& rs, bool finite) {
  uint32_t w[4] = {0, 0, 0, 0};
  if (finite) unit_codes<S>(u, rs, w);
  if (vec && have >= 16) {
    *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < have) dst[i] = static_cast<int8_t>(w[i / 4] >> (8 * (i % 4)));
  }
}

// Scale of a row from its largest magnitude's bits; false where a value is not
// finite, which makes the whole row NaN (codes zero).  The reciprocal is within
// 2^-24 of 1 / scale, so 2^-22 either way brackets it.
__device__ __forceinline__ bool row_scale(unsigned top, RowScale* rs) {
  float scale = __fdiv_rn(__uint_as_float(top), 127.f);
  if (scale < 1.17549435e-38f) scale = 1.f;  // zeros (and values below the normal range)
  const float inv = __frcp_rn(scale);
  rs->scale = scale;
  rs->below = __fmul_rd(inv, 1.f - 2.3841858e-7f);
  rs->above = __fmul_ru(inv, 1.f + 2.3841858e-7f);
  return top < kInfBits;
}

// One row by a whole block of THREADS threads (all call; `tops`: shared, one word
// per warp): its scale and its codes, the codes' row filled with zeros up to
// `pitch` bytes.  The row is read twice.  Ends with the block's reads of `tops`
// done, not with its writes visible.
template <typename S, int THREADS>
__device__ __forceinline__ void quantize_row(int8_t* codes, int pitch, float* scale, const S* row,
                                             int C, bool vec, unsigned* tops) {
  const int units = (C + 15) / 16;
  const int whole = vec ? C / 16 : 0;
  unsigned top = 0;
  auto fetch = [&](int i) {
    Unit<S> u;
    if (i < whole) u.load(row + 16LL * i);
    else u.load_part(row + 16LL * i, C - 16 * i);
    return u;
  };
  for (int i = threadIdx.x; i < units; i += THREADS) top = max(top, top_of<S>(fetch(i).top_bits()));
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) top = max(top, tops[w]);
  __syncthreads();
  RowScale rs;
  const bool finite = row_scale(top, &rs);
  if (threadIdx.x == 0) *scale = finite ? rs.scale : __uint_as_float(0x7fc00000u);
  for (int i = threadIdx.x; i < pitch / 16; i += THREADS) {
    uint32_t w[4] = {0, 0, 0, 0};
    if (finite && i < units) unit_codes<S>(fetch(i), rs, w);
    *reinterpret_cast<uint4*>(codes + 16LL * i) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

}  // namespace i8
}  // namespace g2q
