// ea_fp8.h -- the 8-bit block format shared by ea_train.hip, ea_fp8.hip and ea_fp8_gemm.hip.
//
// A row of C values is cut into blocks of 128 (the last one padded with zero codes).  A block holds e4m3 codes (OCP: 4 exponent
// bits, 3 mantissa bits, largest 448, no infinity) and ONE exponent E: a code stands for code * 2^E.
//   E = the smallest whole number with max |x| <= 448 * 2^E  over the block's finite values (0 for a block of zeros), in
//   [-100, 120]; stored as the byte E + 127 (E8M0), which is what the matrix instruction v_mfma_scale_f32_16x16x128_f8f6f4 takes.
// A power of two costs a floating format nothing but the unused part of its top octave, makes x * 2^-E exact (the code is the only
// rounding: at most 2^-4 of the value, or 2^-10 * 2^E), and lets the matrix unit apply both operands' scales inside the product.
// Non-finite values become NaN codes (e4m3 has no infinity) and do not enter the maximum.
//   codes   [rows][Kp], Kp = C rounded up to 128
//   scales  [Kp / 128][Rp], Rp = rows rounded up to 16 (block-major: four consecutive rows' bytes are one 32-bit load)
//           a weight shares one exponent among 128 rows: [Kp / 128][ceil(rows / 128)]
#pragma once
#include "ea_platform.h"
#include "ea_prims.h"

#define EA_FP8_BLOCK 128
#define EA_FP8_E_MIN (-100)
#define EA_FP8_E_MAX 120
#define EA_INF_BITS 0x7f800000u

// 16 bytes at any element's alignment (global memory takes unaligned vector accesses; a row of odd length starts anywhere)
typedef f16x8 f16x8_any __attribute__((aligned(2)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));
__device__ __forceinline__ f16x8 ea_ld8u(const f16* p) { return *reinterpret_cast<const f16x8_any*>(p); }
__device__ __forceinline__ void ea_st8u(f16* p, f16x8 v) { *reinterpret_cast<f16x8_any*>(p) = v; }
__device__ __forceinline__ f32x4 ea_ld4u(const float* p) { return *reinterpret_cast<const f32x4_any*>(p); }
__device__ __forceinline__ void ea_st4u(float* p, f32x4 v) { *reinterpret_cast<f32x4_any*>(p) = v; }

__device__ __forceinline__ unsigned ea_f2u(float v) { return __builtin_bit_cast(unsigned, v); }
__device__ __forceinline__ float ea_u2f(unsigned v) { return __builtin_bit_cast(float, v); }
// |v| where it enters a block's maximum: NaN and infinity count as 0
__device__ __forceinline__ float ea_finite_abs(float v) {
  const unsigned u = ea_f2u(v) & 0x7fffffffu;
  return u < EA_INF_BITS ? ea_u2f(u) : 0.0f;
}
// the block's exponent byte from its maximum: 448 = 1.75 * 2^8
__device__ __forceinline__ int ea_fp8_exp_byte(float amax) {
  const unsigned u = ea_f2u(amax);
  int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = e < EA_FP8_E_MIN ? EA_FP8_E_MIN : (e > EA_FP8_E_MAX ? EA_FP8_E_MAX : e);
  return (u == 0 ? 0 : e) + 127;
}
__device__ __forceinline__ float ea_fp8_scale(int byte) { return ea_u2f((unsigned)byte << 23); }            // 2^E
__device__ __forceinline__ float ea_fp8_inv_scale(int byte) { return ea_u2f((unsigned)(254 - byte) << 23); }  // 2^-E

#ifdef EA_EMU
inline float ea_emu_fp8_to_f32(unsigned c) {
  const int s = c >> 7, e = (c >> 3) & 15, m = c & 7;
  if (e == 15 && m == 7) return NAN;
  const float v = e ? ldexpf(1.0f + m / 8.0f, e - 7) : ldexpf((float)m, -9);
  return s ? -v : v;
}
inline unsigned ea_emu_f32_to_fp8(float x) {   // round to nearest even; the callers keep |x| <= 448
  if (x != x) return 0x7f;
  const unsigned s = signbit(x) ? 0x80 : 0;
  const float a = fabsf(x);
  int e;
  frexpf(a < 0.015625f ? 0.015625f : a, &e);
  const float step = ldexpf(1.0f, e - 4);
  const float r = nearbyintf(a / step) * step;
  if (r >= 0.015625f) {
    int e2;
    const float f = frexpf(r, &e2);
    return s | (unsigned)((e2 - 1 + 7) << 3) | (unsigned)((f * 2.0f - 1.0f) * 8.0f);
  }
  return s | (unsigned)(r * 512.0f);
}
__device__ __forceinline__ unsigned ea_fp8_pack4(float a, float b, float c, float d) {
  return ea_emu_f32_to_fp8(a) | ea_emu_f32_to_fp8(b) << 8 | ea_emu_f32_to_fp8(c) << 16 | ea_emu_f32_to_fp8(d) << 24;
}
__device__ __forceinline__ void ea_fp8_unpack4(unsigned w, float* v) {
  for (int i = 0; i < 4; ++i) v[i] = ea_emu_fp8_to_f32((w >> (8 * i)) & 255);
}
#else
__device__ __forceinline__ unsigned ea_fp8_pack4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
__device__ __forceinline__ void ea_fp8_unpack4(unsigned w, float* v) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  v[0] = lo[0]; v[1] = lo[1]; v[2] = hi[0]; v[3] = hi[1];
}
#endif
// x * 2^-E for the conversion: what is not finite becomes a NaN code
__device__ __forceinline__ float ea_fp8_prep(float x, float inv) {
  return (ea_f2u(x) & 0x7fffffffu) < EA_INF_BITS ? x * inv : ea_u2f(0x7fc00000u);
}

// ---- reductions over aligned groups of LPR lanes (8, 16, 32, 64); every lane gets the result.  Up to 16 lanes they stay in the
// vector unit (DPP: quad permutes, half-row mirror, row rotate); 32 and 64 add a lane exchange.
#ifdef EA_EMU
#define EA_DPP(v, ctrl, mask) ea_shfl_xor(v, mask)
#else
template <int CTRL>
__device__ __forceinline__ float ea_dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
#define EA_DPP(v, ctrl, mask) ea_dpp<ctrl>(v)
#endif
template <int LPR, typename F>
__device__ __forceinline__ float ea_group_reduce(float v, F f) {
  v = f(v, EA_DPP(v, 0xB1, 1));                 // quad_perm [1, 0, 3, 2]
  v = f(v, EA_DPP(v, 0x4E, 2));                 // quad_perm [2, 3, 0, 1]
  v = f(v, EA_DPP(v, 0x141, 4));                // row_half_mirror: the other quad of the 8 (all four lanes of a quad agree)
  if (LPR >= 16) v = f(v, EA_DPP(v, 0x128, 8)); // row_ror:8
  if (LPR >= 32) v = f(v, ea_shfl_xor(v, 16));
  if (LPR >= 64) v = f(v, ea_shfl_xor(v, 32));
  return v;
}
template <int LPR>
__device__ __forceinline__ float ea_group_sum(float v) {
  return ea_group_reduce<LPR>(v, [](float a, float b) { return a + b; });
}
template <int LPR>
__device__ __forceinline__ float ea_group_max(float v) {
  return ea_group_reduce<LPR>(v, [](float a, float b) { return fmaxf(a, b); });
}

template <int LPR>
__device__ __forceinline__ unsigned ea_group_max_bits(unsigned v) {        // of |v|'s bits: their order is that of the values
  return ea_f2u(ea_group_reduce<LPR>(ea_u2f(v), [](float a, float b) { return ea_f2u(a) > ea_f2u(b) ? a : b; }));
}
// does any lane of the wave say so?
__device__ __forceinline__ bool ea_any(bool c) {
#ifdef EA_EMU
  char* s = ea_emu::wave_scratch();
  s[ea_emu::lane_id() * 64] = c;
  ea_emu::wave_sync();
  bool r = false;
  for (int l = 0; l < ea_emu::wave_lanes(); ++l) r = r || s[l * 64];
  ea_emu::wave_sync();
  return r;
#else
  return __builtin_amdgcn_ballot_w64(c) != 0;
#endif
}

// ---- encoding 8 finite values with their block's exponent byte: one instruction for two values, the power of two included
__device__ __forceinline__ u32x2 ea_fp8_pack8(const float* v, int byte) {
#ifdef EA_EMU
  const float f = ea_fp8_inv_scale(byte);
  return u32x2{ea_fp8_pack4(v[0] * f, v[1] * f, v[2] * f, v[3] * f), ea_fp8_pack4(v[4] * f, v[5] * f, v[6] * f, v[7] * f)};
#else
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  const float f = ea_fp8_scale(byte);
  s16x2 a = {0, 0}, b = {0, 0};
  a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(a, v[0], v[1], f, false);
  a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(a, v[2], v[3], f, true);
  b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, v[4], v[5], f, false);
  b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, v[6], v[7], f, true);
  return u32x2{__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b)};
#endif
}
__device__ __forceinline__ u32x2 ea_fp8_pack8(f16x8 v, int byte) {
#ifdef EA_EMU
  float t[8];
  for (int j = 0; j < 8; ++j) t[j] = (float)v[j];
  return ea_fp8_pack8(t, byte);
#else
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  typedef __fp16 h2 __attribute__((ext_vector_type(2)));
  const float f = ea_fp8_scale(byte);
  const u32x4 w = __builtin_bit_cast(u32x4, v);
  const unsigned w0 = w[0], w1 = w[1], w2 = w[2], w3 = w[3];
  s16x2 a = {0, 0}, b = {0, 0};
  a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(a, __builtin_bit_cast(h2, w0), f, false);
  a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(a, __builtin_bit_cast(h2, w1), f, true);
  b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(b, __builtin_bit_cast(h2, w2), f, false);
  b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(b, __builtin_bit_cast(h2, w3), f, true);
  return u32x2{__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b)};
#endif
}
// the largest |v| of 8 values, as fp32 bits (at least EA_INF_BITS where one of them is not finite)
__device__ __forceinline__ unsigned ea_max_bits8(const float* v) {
  unsigned m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const unsigned u = ea_f2u(v[j]) & 0x7fffffffu;
    m = u > m ? u : m;
  }
  return m;
}
__device__ __forceinline__ unsigned ea_max_bits8(f16x8 v) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  const u32x4 w = __builtin_bit_cast(u32x4, v);
  const unsigned a0 = w[0] & 0x7fff7fffu, a1 = w[1] & 0x7fff7fffu, a2 = w[2] & 0x7fff7fffu, a3 = w[3] & 0x7fff7fffu;
  const u16x2 p = __builtin_elementwise_max(__builtin_bit_cast(u16x2, a0), __builtin_bit_cast(u16x2, a1));
  const u16x2 q = __builtin_elementwise_max(__builtin_bit_cast(u16x2, a2), __builtin_bit_cast(u16x2, a3));
  const u16x2 m = __builtin_elementwise_max(p, q);
  const unsigned short h = m[0] > m[1] ? m[0] : m[1];
  return ea_f2u((float)__builtin_bit_cast(f16, h)) & 0x7fffffffu;
}
// One block of 128: 16 lanes (GRP; 8 columns each) turn their 8 values into codes and the block's exponent byte.  Every lane of the wave
// calls it.  Blocks with values that are not finite take the slow way: those become NaN codes and stay out of the maximum.
template <int GRP, typename V>
__device__ __forceinline__ u32x2 ea_fp8_block(const V& v, int& byte) {
  const unsigned m = ea_group_max_bits<GRP>(ea_max_bits8(v));
  if (!ea_any(m >= EA_INF_BITS)) {
    byte = ea_fp8_exp_byte(ea_u2f(m));
    return ea_fp8_pack8(v, byte);
  }
  float t[8], top = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    t[j] = (float)v[j];
    top = fmaxf(top, ea_finite_abs(t[j]));
  }
  byte = ea_fp8_exp_byte(ea_group_max<GRP>(top));
  const float inv = ea_fp8_inv_scale(byte);
#pragma unroll
  for (int j = 0; j < 8; ++j) t[j] = ea_fp8_prep(t[j], inv);
  return u32x2{ea_fp8_pack4(t[0], t[1], t[2], t[3]), ea_fp8_pack4(t[4], t[5], t[6], t[7])};
}

// 1 - Phi(a) = erfc(a / sqrt 2) / 2 by the polynomial of ea_gelu_erf (ea_platform.h), for a = |x| up to 4 sqrt 2
#define EA_FP8_GELU_END 5.65685424949238f
__device__ __forceinline__ float ea_fp8_gelu_tail(float a) {
  float q = -4.276626896171365e-06f;
  q = q * a + 1.2775987670465838e-05f;
  q = q * a + 0.0005758762708865106f;
  q = q * a - 0.007670961786061525f;
  q = q * a + 0.05294874310493469f;
  q = q * a + 0.45904383063316345f;
  q = q * a + 1.1511269807815552f;
  return ea_exp2_raw(-a * q - 1.0f);
}
// GELU to ea_gelu_erf's values.  That takes fmaxf(x, 0) and puts a NaN back afterwards; the
// comparison x < 0 lets a NaN through by itself, one instruction less.  The epilogue of the 256 x 256 product is bound by these
// instructions: with the scale's multiplication left out where it is 1, 16384 x 5120 x 1280 went from 137 to 128 us.
__device__ __forceinline__ float ea_fp8_gelu(float x) {
  const float a = fminf(fabsf(x), EA_FP8_GELU_END);
  return (x < 0.0f ? 0.0f : x) - a * ea_fp8_gelu_tail(a);
}

#define EA_FP8_ROWS (1 << 30)      // most rows of an entry that counts them in 32 bits: tile counts and row indexes stay below 2^31
// a launch holds fewer than 2^32 threads along x
static inline bool ea_launch_holds(long long workgroups, int threads) { return workgroups * threads < (1ll << 32); }
// Memory of a call: n bytes at p (NULL: none).  An output may not share bytes with an input or another output; `same` allows exactly the same
// bytes, where every element is read by the thread that writes it
struct ea_span { const void* p; long long n; };
static inline bool ea_apart(ea_span a, ea_span b, bool same = false) {
  const uintptr_t x = (uintptr_t)a.p, y = (uintptr_t)b.p;
  return !x || !y || (x < y ? (long long)(y - x) >= a.n : (long long)(x - y) >= b.n) || (same && x == y && a.n == b.n);
}
template <size_t O, size_t I>
static inline bool ea_outputs_apart(const ea_span (&out)[O], const ea_span (&in)[I]) {
  for (size_t o = 0; o < O; ++o) {
    for (size_t i = 0; i < I; ++i)
      if (!ea_apart(out[o], in[i])) return false;
    for (size_t i = 0; i < o; ++i)
      if (!ea_apart(out[o], out[i])) return false;
  }
  return true;
}
static inline int ea_fp8_blocks(int cols) { return (cols + EA_FP8_BLOCK - 1) / EA_FP8_BLOCK; }
static inline long long ea_fp8_scale_pitch(long long rows) { return (rows + 15) / 16 * 16; }
static inline ea_span ea_codes(const void* q, long long rows, int cols) { return {q, rows * ea_fp8_blocks(cols) * EA_FP8_BLOCK}; }
static inline ea_span ea_row_scales(const void* s, long long rows, int cols) { return {s, ea_fp8_scale_pitch(rows) * ea_fp8_blocks(cols)}; }
static inline ea_span ea_weight_scales(const void* s, long long rows, int cols) { return {s, (rows + 127) / 128 * ea_fp8_blocks(cols)}; }
