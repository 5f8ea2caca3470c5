// 8-bit activation checkpoints: what the kernels of act8.hip, act8_norm.hip and act8_wgrad.hip
// share.
//
// A row of C features is cut into blocks of 32 (the last one shorter where 32 does not divide C).
// A block with the largest magnitude a keeps
//     e = the smallest integer >= -126 with a <= 127 2^e,   q_i = round_half_even(x_i 2^-e)
// as q int8 [rows, P] (P = C rounded up to 32, zeros behind C) and scale uint8 [rows, P / 32] =
// e + 127, and stands for q_i 2^e.  A power of two, so that the value is exact in bf16 (|q| < 128
// is 7 bits) and a matrix product in bf16 sees exactly what the checkpoint stands for; an error
// of at most 2^e / 2 <= max(a / 127, 2^-127) a value (e stops at -126).  A block that holds a
// magnitude above 127 2^121 (3.376e38, where a rounded value can reach 2^128), an infinity or a NaN
// has scale 255 and q 0: 0 * 2^128 = NaN, so a non-finite activation stays visible in the backward
// pass.
//
// The unit of the kernels is a CHUNK of 8 consecutive features of a row: one 16-B load of bf16,
// two of f32, one 8-B store of q.  A block is the 4 chunks of an aligned quad of lanes.
#pragma once
#include "mfma_util.h"

namespace vs {
namespace {

constexpr int kBlock = 32;                       // features of a block
__host__ __device__ constexpr int padded32(int C) { return (C + 31) & ~31; }

// 16 B at any element alignment (one global_load / store_dwordx4: the memory path takes
// unaligned addresses, so an odd row pitch needs no kernel of its own)
typedef uint32_t unaligned16_t __attribute__((ext_vector_type(4), aligned(2)));
__device__ __forceinline__ uint4 ld16(const void* p) {
  const unaligned16_t v = *reinterpret_cast<const unaligned16_t*>(p);
  return make_uint4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void st16(void* p, uint4 a) {
  const unaligned16_t v = {a.x, a.y, a.z, a.w};
  *reinterpret_cast<unaligned16_t*>(p) = v;
}

// 8 features as loaded
template <typename T> struct Chunk;
template <> struct Chunk<bf16> {
  uint4 a;
  __device__ __forceinline__ void load(const bf16* p) { a = ld16(p); }
  // the first n (0..7) of 8
  __device__ __forceinline__ void load_some(const bf16* p, int n) {
    const unsigned short* s = reinterpret_cast<const unsigned short*>(p);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = (2 * i < n ? (uint32_t)s[2 * i] : 0u) | (2 * i + 1 < n ? (uint32_t)s[2 * i + 1] << 16 : 0u);
    a = make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ void zero() { a = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ void unpack(float* out) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      out[2 * i] = __uint_as_float(w[i] << 16);
      out[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  __device__ __forceinline__ void pack(const float* v) {       // rounded to nearest even
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = (uint32_t)(unsigned short)bf16_bits(v[2 * i]) | ((uint32_t)(unsigned short)bf16_bits(v[2 * i + 1]) << 16);
    a = make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ void store(bf16* p) const { st16(p, a); }
  __device__ __forceinline__ void store_some(bf16* p, int n) const {
    unsigned short* s = reinterpret_cast<unsigned short*>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) s[i] = (unsigned short)(w[i >> 1] >> (16 * (i & 1)));
  }
};
template <> struct Chunk<float> {
  uint4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = ld16(p);
    b = ld16(p + 4);
  }
  __device__ __forceinline__ void load_some(const float* p, int n) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = i < n ? __float_as_uint(p[i]) : 0u;
    a = make_uint4(w[0], w[1], w[2], w[3]);
    b = make_uint4(w[4], w[5], w[6], w[7]);
  }
  __device__ __forceinline__ void zero() { a = b = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ void unpack(float* out) const {
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = __uint_as_float(w[i]);
  }
  __device__ __forceinline__ void pack(const float* v) {
    a = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    b = make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
  }
  __device__ __forceinline__ void store(float* p) const {
    st16(p, a);
    st16(p + 4, b);
  }
  __device__ __forceinline__ void store_some(float* p, int n) const {
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = __uint_as_float(w[i]);
  }
};

// chunk j of a row of C features at p: whole, its first features, or (behind the row) zeros
template <typename T>
__device__ __forceinline__ void load_row_chunk(Chunk<T>& c, const T* p, int j, int C) {
  const int n = C - 8 * j;
  if (n >= 8)
    c.load(p + 8 * j);
  else if (n > 0)
    c.load_some(p + 8 * j, n);
  else
    c.zero();
}

template <typename T>
__device__ __forceinline__ void store_row_chunk(const Chunk<T>& c, T* p, int j, int C) {
  const int n = C - 8 * j;
  if (n >= 8)
    c.store(p + 8 * j);
  else if (n > 0)
    c.store_some(p + 8 * j, n);
}

// lane exchange inside a quad: CTRL 0xB1 = lanes 1 0 3 2, 0x4E = lanes 2 3 0 1
template <int CTRL>
__device__ __forceinline__ uint32_t quad(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true);
}

// The 8 values of a chunk -> 8 bytes of q and the block's scale byte (the same in its 4 lanes,
// all of which have to be active).  Magnitudes are compared as the integers that their bits
// are: ordered like the numbers, an infinity or NaN above every finite one.
__device__ __forceinline__ uint2 pack_chunk(const float* v, uint32_t& scale) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  m = max(m, quad<0xB1>(m));
  m = max(m, quad<0x4E>(m));
  // exponent field of a less 6 where its significand is <= 127 / 64 (mantissa 0x7e0000), else
  // less 5: the carry of adding 0x1ffff
  uint32_t sb = (m + 0x1ffffu) >> 23;
  sb = sb > 7u ? sb - 6u : 1u;
  const bool bad = m > 0x7f7e0000u;              // 127 2^121
  const float inv = __uint_as_float((254u - sb) << 23);       // 2^-e, normal for 1 <= sb <= 248
  // x 2^-e + 1.5 2^23 rounds the exact product to the integer (ties to even), which the sum's
  // low byte holds in two's complement
  uint32_t f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = __float_as_uint(fmaf(v[i], inv, 12582912.f));
  uint2 q;
  q.x = __builtin_amdgcn_perm(__builtin_amdgcn_perm(f[3], f[2], 0x0c0c0400u),
                              __builtin_amdgcn_perm(f[1], f[0], 0x0c0c0400u), 0x05040100u);
  q.y = __builtin_amdgcn_perm(__builtin_amdgcn_perm(f[7], f[6], 0x0c0c0400u),
                              __builtin_amdgcn_perm(f[5], f[4], 0x0c0c0400u), 0x05040100u);
  if (bad) q = make_uint2(0u, 0u);
  scale = bad ? 255u : sb;
  return q;
}

// what a chunk stands for (scale 255: 0 * infinity = NaN)
__device__ __forceinline__ void unpack_chunk(uint2 q, uint32_t scale, float* v) {
  const float s = __uint_as_float(scale << 23);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = (float)(signed char)(q.x >> (8 * i)) * s;
    v[4 + i] = (float)(signed char)(q.y >> (8 * i)) * s;
  }
}

// The normal distribution's tail by its Mills ratio M(a) = (1 - Phi(a)) / phi(a), a >= 0: smooth,
// falling from sqrt(pi / 2) like 1 / a, so t poly(t) with t = 1 / (1 + p a) fits it in RELATIVE
// error (least squares with the weights raised where the error is largest, until it is level,
// over 0 <= a <= 14.5): degree 6 to 9e-6 for bf16 results (half a step: 2e-3), degree 9 to 3.6e-8
// for f32 ones (half a step: 6e-8; with the coefficients as rounded to f32, whose last bits were
// searched for the smallest error).  gelu(x) and its slope then need one exponential and one reciprocal:
//     gelu(x)  = max(x, 0) - |x| M(|x|) phi(x)
//     gelu'(x) = [x >= 0] + sign(x) (|x| - M(|x|)) phi(x)
template <typename T> struct Mills;
template <> struct Mills<bf16> {
  __device__ __forceinline__ static float at(float a) {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.30f, a, 1.f));
    float s = -1.922598183e-01f;
    s = fmaf(s, t, 5.385463834e-01f);
    s = fmaf(s, t, -3.909720480e-02f);
    s = fmaf(s, t, 3.596343994e-01f);
    s = fmaf(s, t, 2.855621874e-01f);
    s = fmaf(s, t, 3.009393215e-01f);
    return s * t;
  }
};
template <> struct Mills<float> {
  __device__ __forceinline__ static float at(float a) {
    // M moves 2.35 times as much as t near a = 0, so what the denominator's rounding and the
    // reciprocal's leave, rho = 1 - (1 + p a) t, is taken back to first order: M(t + t rho) = M(t)
    // (1 + g rho), g = t M'(t) / M(t), 1 at t = 0 and 2.35 at t = 1
    const float d = fmaf(0.34f, a, 1.f), t = __builtin_amdgcn_rcpf(d);
    const float rho = fmaf(-fmaf(0.34f, a, 1.f - d), t, fmaf(-d, t, 1.f));
    float s = -6.486240029e-02f;
    s = fmaf(s, t, 3.468088210e-01f);
    s = fmaf(s, t, -6.789713502e-01f);
    s = fmaf(s, t, 5.006161928e-01f);
    s = fmaf(s, t, -1.080504805e-01f);
    s = fmaf(s, t, 2.875439227e-01f);
    s = fmaf(s, t, 2.891439795e-01f);
    s = fmaf(s, t, 3.411326110e-01f);
    s = fmaf(s, t, 3.399528861e-01f);
    const float m = s * t;
    return fmaf(m * fmaf(1.35f, t, 1.f), rho, m);
  }
};

// phi(a) = exp(-a^2 / 2) / sqrt(2 pi): the hardware's 2^x
__device__ __forceinline__ float normal_density(float a) {
  return 0.3989422804f * __builtin_amdgcn_exp2f(-0.7213475204f * a * a);
}

// |x| is cut at 40 (phi is 0 there), so that +-infinity gives its limit; a NaN stays one
template <typename T>
__device__ __forceinline__ float gelu_value(float x) {
  const float a = fminf(fabsf(x), 40.f);
  return (x < 0.f ? 0.f : x) - a * Mills<T>::at(a) * normal_density(a);
}

// x finite or NaN (a checkpoint's value)
template <typename T>
__device__ __forceinline__ float gelu_slope(float x) {
  const float a = fabsf(x);
  const float d = (a - Mills<T>::at(a)) * normal_density(a);
  return x < 0.f ? -d : 1.f + d;
}

// gelu and its slope of one value, from one exponential and one reciprocal
template <typename T>
__device__ __forceinline__ void gelu_both(float x, float& y, float& slope) {
  const float a = fabsf(x);
  const float m = Mills<T>::at(a), p = normal_density(a);
  const float d = (a - m) * p;
  slope = x < 0.f ? -d : 1.f + d;
  y = (x < 0.f ? 0.f : x) - fminf(a, 40.f) * m * p;
}

}  // namespace
}  // namespace vs
