// ea_fp8_gemm.h -- out = epilogue(A W^T) on the 8-bit format of ea_fp8.h.
//
//   out[m][n] = residual + scale * act( sum_b 2^(Ea[b][m] + Ew[b][n / 128]) * sum_{k in block b} a[m][k] w[n][k]  + bias[n] )
//
// One instruction does a whole scale block: v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 16 x 128 by 128 x 16 codes and applies one
// exponent byte per row and per column, so scales cost no vector work and the accumulators are fp32 throughout.
//
// Layout (both kernels).  A K tile is one scale block: 128 bytes of a row, the LDS row of the fp16 kernels with K = 64, fetched by
// LDS-DMA with the same 16-byte XOR swizzle.  The order of K inside a block is free (both operands share it and one scale covers
// it), so a lane's 32 operand bytes are two 16-byte reads, chunks lq and lq + 4 of its row.  The order of ROWS inside a tile is free
// too (the DMA's source address is per lane) and is chosen so that
//   * the activation rows of 4 fragments are 4 i + f (fragment f, lane i): a lane's four scale bytes are one 32-bit load and the
//     instruction picks its byte by op_sel;
//   * the weight rows of 4 fragments are 16 (i >> 2) + 4 f + (i & 3): with the operands swapped (D^T = W A^T) a lane ends up with 16
//     consecutive outputs of one row, stored from registers with 16-byte stores.
#pragma once
#include "ea_fp8.h"
#include "../../include/editanything_hip.h"

typedef int i32x8 __attribute__((ext_vector_type(8)));

// A, B: 32 bytes per lane (row / column l & 15; K group l >> 4); SA, SB: which byte of the lane's scale word
template <int SA, int SB>
__device__ __forceinline__ f32x4 ea_mfma_fp8_128(i32x8 a, i32x8 b, f32x4 c, unsigned sa, unsigned sb) {
#ifdef EA_EMU
  char* s = ea_emu::wave_scratch();
  const int l = ea_emu::lane_id();
  memcpy(s + l * 64, &a, 32);
  memcpy(s + l * 64 + 32, &b, 32);
  ea_emu::wave_sync();
  uint8_t ra[4][128], rb[128];
  for (int g = 0; g < 4; ++g) {
    for (int r = 0; r < 4; ++r) memcpy(ra[r] + 32 * g, s + ((l >> 4) * 4 + r + 16 * g) * 64, 32);
    memcpy(rb + 32 * g, s + ((l & 15) + 16 * g) * 64 + 32, 32);
  }
  ea_emu::wave_sync();
  memcpy(s + l * 64, &sa, 4);
  memcpy(s + l * 64 + 4, &sb, 4);
  ea_emu::wave_sync();
  for (int r = 0; r < 4; ++r) {
    float acc = 0.0f;
    for (int g = 0; g < 4; ++g) {
      const int ea = (uint8_t)s[((l >> 4) * 4 + r + 16 * g) * 64 + SA], eb = (uint8_t)s[((l & 15) + 16 * g) * 64 + 4 + SB];
      float t = 0.0f;
      for (int k = 0; k < 32; ++k) t += ea_emu_fp8_to_f32(ra[r][32 * g + k]) * ea_emu_fp8_to_f32(rb[32 * g + k]);
      acc += ldexpf(t, ea + eb - 254);
    }
    c[r] += acc;
  }
  ea_emu::wave_sync();
  return c;
#else
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, SA, (int)sa, SB, (int)sb);
#endif
}

// 8 codes times a power of two in fp16 (exact for the power 1)
__device__ __forceinline__ f16x8 ea_f8_half8(unsigned w0, unsigned w1, float f) {
#ifdef EA_EMU
  f16x8 o;
  for (int j = 0; j < 8; ++j) o[j] = (f16)(ea_emu_fp8_to_f32(((j < 4 ? w0 : w1) >> (8 * (j & 3))) & 255) * f);
  return o;
#else
  return __builtin_bit_cast(f16x8, u32x4{__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, f, false)),
                                         __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, f, true)),
                                         __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, f, false)),
                                         __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, f, true))});
#endif
}

struct EaFp8GemmParams {
  const uint8_t* a; const uint8_t* sa;     // [M][Kp], [nb][Rp]
  const uint8_t* w; const uint8_t* sw;     // [N][Kp], [nb][nwb]
  int M, N, Kp, nb, nwb; long long Rp;
  const float* bias; const f16* residual; const float* residual32; void* out;
  int act, out_f32, ldc, ldr, vec; float scale;
  int raster_gm;
};

// Workgroup -> tile.  Workgroups are dealt round-robin to the 8 XCDs, each with its own L2: an XCD gets one contiguous run of tiles,
// and a run goes down `gm` row tiles before it moves to the next column tile, so that it re-reads few rows and few columns.
__device__ __forceinline__ void ea_fp8_tile(int wg, int tiles_m, int tiles_n, int gm, int& tm, int& tn) {
  const int n = tiles_m * tiles_n, q = n >> 3, r = n & 7, xcd = wg & 7;
  const int t = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (wg >> 3);
  const int grp = t / (gm * tiles_n), first = grp * gm;
  const int gsz = tiles_m - first < gm ? tiles_m - first : gm;
  const int u = t - grp * gm * tiles_n;
  tn = ea_uniform(u / gsz);
  tm = ea_uniform(first + u - tn * gsz);
}

// Output and residual rows through buffer descriptors that end with the last row of the matrix: a lane's byte offset is one addition
// per 16-byte access, rows behind the end are dropped (loads: zero) by the bounds check, and so are columns behind N (their lanes'
// offsets start at 2 GiB).  A descriptor starts at the workgroup's first row; the host keeps 256 rows within 2 GiB (p.vec).
#define EA_F8_NOWHERE 0x80000000u
#ifdef EA_EMU
struct ea_rows { char* p; unsigned n; };
__device__ __forceinline__ ea_rows ea_make_rows(const void* p, long long bytes) {
  return ea_rows{(char*)const_cast<void*>(p), (unsigned)(bytes > 0x7fffffffll ? 0x7fffffffll : bytes)};
}
__device__ __forceinline__ u32x4 ea_rows_load(ea_rows r, unsigned off) {
  u32x4 v = {0, 0, 0, 0};
  if (off < r.n && off + 16 <= r.n) memcpy(&v, r.p + off, 16);
  return v;
}
__device__ __forceinline__ void ea_rows_store(ea_rows r, unsigned off, u32x4 v) {
  if (off < r.n && off + 16 <= r.n) memcpy(r.p + off, &v, 16);
}
__device__ __forceinline__ unsigned ea_rows_load1(ea_rows r, unsigned off) {
  unsigned v = 0;
  if (off < r.n && off + 4 <= r.n) memcpy(&v, r.p + off, 4);
  return v;
}
__device__ __forceinline__ void ea_rows_store1(ea_rows r, unsigned off, unsigned v) {
  if (off < r.n && off + 4 <= r.n) memcpy(r.p + off, &v, 4);
}
#else
typedef __amdgpu_buffer_rsrc_t ea_rows;
__device__ __forceinline__ ea_rows ea_make_rows(const void* p, long long bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (unsigned)(bytes > 0x7fffffffll ? 0x7fffffffll : bytes), 0x00020000);
}
__device__ __forceinline__ u32x4 ea_rows_load(ea_rows r, unsigned off) {
  return __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0);
}
__device__ __forceinline__ void ea_rows_store(ea_rows r, unsigned off, u32x4 v) {
  __builtin_amdgcn_raw_buffer_store_b128(v, r, off, 0, 0);
}
__device__ __forceinline__ unsigned ea_rows_load1(ea_rows r, unsigned off) { return __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0); }
__device__ __forceinline__ void ea_rows_store1(ea_rows r, unsigned off, unsigned v) { __builtin_amdgcn_raw_buffer_store_b32(v, r, off, 0, 0); }
#endif

// acc[i][j] of one wave (16 x 16 fragments): activation fragments i (groups of FMG), weight fragments j (groups of FNG): a lane owns
// 4 FNG consecutive columns of FM rows.  The accumulators start from the bias.
template <int FM, int FN, int FMG, int FNG>
__device__ __forceinline__ void ea_fp8_start(const EaFp8GemmParams& p, f32x4 (&acc)[FM][FN], int n0) {
  const int lq = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int j = 0; j < FN; ++j) {
    const int n = n0 + 16 * FNG * (j / FNG) + 4 * FNG * lq + 4 * (j % FNG);
    f32x4 b = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (p.bias) {
#pragma unroll
      for (int r = 0; r < 4; ++r) b[r] = p.bias[n + r < p.N ? n + r : p.N - 1];      // (columns behind N are not stored)
    }
#pragma unroll
    for (int i = 0; i < FM; ++i) acc[i][j] = b;
  }
}

template <int ACT>
__device__ __forceinline__ float ea_fp8_act(float x) {
  return ACT == EA_ACT_SILU ? ea_silu(x) : ACT == EA_ACT_GELU ? ea_fp8_gelu(x) : x;
}
// 16-byte accesses.  m0: the workgroup's first row, mw: the wave's
template <int ACT, int FM, int FN, int FMG, int FNG>
__device__ __forceinline__ void ea_fp8_finish_vec(const EaFp8GemmParams& p, const f32x4 (&acc)[FM][FN], int mw, int m0, int n0) {
  const int lane = threadIdx.x & 63, l15 = lane & 15, lq = lane >> 4;
  const int es = p.out_f32 ? 4 : 2, rs = p.residual32 ? 4 : 2;
  const ea_rows out = ea_make_rows((char*)p.out + (long long)m0 * p.ldc * es, (long long)(p.M - m0) * p.ldc * es);
  const void* res = p.residual32 ? (const void*)p.residual32 : (const void*)p.residual;
  const ea_rows rr = ea_make_rows((const char*)res + (long long)m0 * p.ldr * rs, res ? (long long)(p.M - m0) * p.ldr * rs : 0);
  const unsigned oline = (unsigned)(p.ldc * es), rline = (unsigned)(p.ldr * rs);
  constexpr int NH = FNG / 2, NP = FN / FNG * NH;     // 8-column pieces of a lane's run, of a row
  unsigned oc[NP], rc[NP];
#pragma unroll
  for (int g = 0; g < NP; ++g) {
    const int n = n0 + 16 * FNG * (g / NH) + 4 * FNG * lq + 8 * (g % NH);
    oc[g] = n < p.N ? (unsigned)(n * es) : EA_F8_NOWHERE;
    rc[g] = n < p.N ? (unsigned)(n * rs) : EA_F8_NOWHERE;
  }
  auto row = [&](int i) { return (unsigned)(mw - m0 + 16 * FMG * (i / FMG) + FMG * l15 + i % FMG); };
  u32x4 r0[2][NP], r1[NP];                            // residual pieces, one row ahead (fp32: the second half when it is used)
  auto fetch = [&](int i) {
    if (res)
#pragma unroll
      for (int g = 0; g < NP; ++g) r0[i & 1][g] = ea_rows_load(rr, rc[g] + row(i) * rline);
  };
  fetch(0);
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    if (p.residual32)
#pragma unroll
      for (int g = 0; g < NP; ++g) r1[g] = ea_rows_load(rr, rc[g] + row(i) * rline + 16);
    if (i + 1 < FM) fetch(i + 1);
#pragma unroll
    for (int g = 0; g < NP; ++g) {
      const int j = g / NH * FNG + 2 * (g % NH);
      const unsigned o = oc[g] + row(i) * oline;
      float v[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) v[c] = ea_fp8_act<ACT>(acc[i][j + c / 4][c % 4]);
      if (p.scale != 1.0f)
#pragma unroll
        for (int c = 0; c < 8; ++c) v[c] *= p.scale;
      if (p.residual) {
        const f16x8 r = __builtin_bit_cast(f16x8, r0[i & 1][g]);
#pragma unroll
        for (int c = 0; c < 8; ++c) v[c] += (float)r[c];
      } else if (p.residual32) {
        const f32x4 a = __builtin_bit_cast(f32x4, r0[i & 1][g]), b = __builtin_bit_cast(f32x4, r1[g]);
#pragma unroll
        for (int c = 0; c < 8; ++c) v[c] += c < 4 ? a[c & 3] : b[c & 3];
      }
      if (p.out_f32) {
        ea_rows_store(out, o, __builtin_bit_cast(u32x4, f32x4{v[0], v[1], v[2], v[3]}));
        ea_rows_store(out, o + 16, __builtin_bit_cast(u32x4, f32x4{v[4], v[5], v[6], v[7]}));
      } else {
        f16x8 y;
#pragma unroll
        for (int c = 0; c < 8; ++c) y[c] = (f16)v[c];
        ea_rows_store(out, o, __builtin_bit_cast(u32x4, y));
      }
    }
  }
}
template <int FM, int FN, int FMG, int FNG>
__device__ __forceinline__ void ea_fp8_finish(const EaFp8GemmParams& p, const f32x4 (&acc)[FM][FN], int mw, int m0, int n0) {
  if constexpr (FNG > 1) {
    if (p.vec) {
      if (p.act == EA_ACT_GELU) ea_fp8_finish_vec<EA_ACT_GELU, FM, FN, FMG, FNG>(p, acc, mw, m0, n0);
      else if (p.act == EA_ACT_SILU) ea_fp8_finish_vec<EA_ACT_SILU, FM, FN, FMG, FNG>(p, acc, mw, m0, n0);
      else ea_fp8_finish_vec<EA_ACT_NONE, FM, FN, FMG, FNG>(p, acc, mw, m0, n0);
      return;
    }
  }
  const int lane = threadIdx.x & 63, l15 = lane & 15, lq = lane >> 4;
#pragma unroll
  for (int i = 0; i < FM; ++i)                        // any N, any alignment
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int m = mw + 16 * FMG * (i / FMG) + FMG * l15 + i % FMG, n = n0 + 16 * FNG * (j / FNG) + 4 * FNG * lq + 4 * (j % FNG) + r;
        float v = acc[i][j][r];
        if (m >= p.M || n >= p.N) continue;
        v = (p.act == EA_ACT_GELU ? ea_fp8_gelu(v) : p.act == EA_ACT_SILU ? ea_silu(v) : v) * p.scale;
        if (p.residual) v += (float)p.residual[(long long)m * p.ldr + n];
        else if (p.residual32) v += p.residual32[(long long)m * p.ldr + n];
        if (p.out_f32) ((float*)p.out)[(long long)m * p.ldc + n] = v;
        else ((f16*)p.out)[(long long)m * p.ldc + n] = (f16)v;
      }
}

// Scale bytes of up to EA_F8_CH K tiles in LDS, [tile][BM] of the rows and then [tile][4] of the columns (two 128-column blocks at
// most): loaded into registers in front of a chunk's first DMA, written behind it.  Kept out of the K loop's vector loads on purpose:
// as registers prefetched a tile ahead they made the compiler drain the DMA queue at every tile (vmcnt counts both), 0.5 us per tile of
// the small kernel.
#define EA_F8_CH 64
template <int BM, int NT>
struct EaF8Scales {
  static constexpr int W = EA_F8_CH * BM / 4 / NT;          // words per thread
  unsigned w[W], c[2];
  __device__ __forceinline__ void load(const EaFp8GemmParams& p, int t0, int n, int m0, int n0) {
#pragma unroll
    for (int u = 0; u < W; ++u) {
      const int i = u * NT + threadIdx.x, kb = i / (BM / 4);
      long long r = m0 + (i % (BM / 4)) * 4;
      if (r >= p.Rp) r = p.Rp - 4;                          // (rows behind the last use any stored byte: nothing of them is kept)
      w[u] = kb < n ? *reinterpret_cast<const unsigned*>(p.sa + (t0 + kb) * p.Rp + r) : 0;
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      int b = (n0 >> 7) + u;
      if (b >= p.nwb) b = p.nwb - 1;
      c[u] = threadIdx.x < (unsigned)n ? p.sw[(long long)(t0 + threadIdx.x) * p.nwb + b] : 0;
    }
  }
  __device__ __forceinline__ void store(char* lds) {
#pragma unroll
    for (int u = 0; u < W; ++u) *reinterpret_cast<unsigned*>(lds + (u * NT + threadIdx.x) * 4) = w[u];
    if (threadIdx.x < EA_F8_CH) *reinterpret_cast<unsigned*>(lds + EA_F8_CH * BM + threadIdx.x * 4) = c[0] | c[1] << 8;
  }
};
__device__ __forceinline__ i32x8 ea_f8_frag(const char* base, int s, int lq) {
  const u32x4 x = *reinterpret_cast<const u32x4*>(base + s * 128 + ((lq ^ ea_swz(s)) << 4));
  const u32x4 y = *reinterpret_cast<const u32x4*>(base + s * 128 + (((4 + lq) ^ ea_swz(s)) << 4));
  return i32x8{(int)x[0], (int)x[1], (int)x[2], (int)x[3], (int)y[0], (int)y[1], (int)y[2], (int)y[3]};
}

// ------------------------------------------------------------------------------------------------------- ring kernel
// BM x BN outputs, WM x WN waves, a ring of S stages of one K tile each, one barrier per tile.  At tile t a wave waits for its own
// DMA of tile t (the S - 2 younger tiles stay in flight), the barrier makes everybody's visible and says that tile t - 1 has been read;
// then tile t + S - 1 is issued into that buffer.
//
// EXACT: the 8-bit instruction keeps each of eight neighbouring products only to 2^-13 of the largest.  This form decodes both operands to fp16 (a
// code is an fp16 value) and multiplies with the fp16 instruction, whose products and sums are fp32's: four of them make a block's sum, which
// enters the accumulators with the block's power of two.  At the fp16 rate, half of the other's, and 8 vector instructions per
// fragment and block beside the decoding.  Error (root mean square, of the result's, 616 x 2560 x 1024): 8-bit instruction 1.5e-5, EXACT 3.4e-8; behind
// the rounding to fp16 2.083e-4 and 2.078e-4.
template <int BM, int BN, int WM, int WN, int S, bool EXACT>
__global__ __launch_bounds__(64 * WM * WN) void ea_fp8_ring_kernel(EaFp8GemmParams p) {
  constexpr int NT = 64 * WM * WN, FM = BM / WM / 16, FN = BN / WN / 16;
  constexpr int FMG = FM < 4 ? FM : 4, FNG = FN < 4 ? FN : 4;
  constexpr int STAGE = (BM + BN) * 128, DA = BM * 8 / NT, DB = BN * 8 / NT, D = DA + DB;
  static_assert(BM * 8 % NT == 0 && BN * 8 % NT == 0, "whole DMA instructions");
  static_assert(128 % BN == 0, "a workgroup's columns share one weight scale");
  EA_SMEM(smem);
  char* const scl = smem + S * STAGE;
  const int tid = threadIdx.x, lane = tid & 63, wave = ea_uniform(tid >> 6), wm = wave / WN, wn = wave % WN;
  const int l15 = lane & 15, lq = lane >> 4;
  const int tiles_n = (p.N + BN - 1) / BN, tiles_m = (p.M + BM - 1) / BM;
  int tm, tn;
  ea_fp8_tile(blockIdx.x, tiles_m, tiles_n, p.raster_gm, tm, tn);
  const int m0 = tm * BM, n0 = tn * BN;
  const ea_rsrc ra = ea_make_rsrc(p.a + (long long)m0 * p.Kp), rw = ea_make_rsrc(p.w + (long long)n0 * p.Kp);

  unsigned va[DA], vb[DB];
#pragma unroll
  for (int i = 0; i < DA; ++i) {
    const int s = (i * NT + tid) >> 3, w = s & (16 * FMG - 1);       // LDS row s holds tile row (s - w) + FMG * (w & 15) + (w >> 4)
    const int r = s - w + FMG * (w & 15) + (w >> 4);
    va[i] = m0 + r < p.M ? (unsigned)r * (unsigned)p.Kp + (unsigned)(((tid & 7) ^ ea_swz(s)) << 4) : EA_OOB;
  }
#pragma unroll
  for (int i = 0; i < DB; ++i) {
    const int s = (i * NT + tid) >> 3, w = s & (16 * FNG - 1);
    const int r = s - w + 4 * FNG * ((w & 15) >> 2) + 4 * (w >> 4) + (w & 3);
    vb[i] = n0 + r < p.N ? (unsigned)r * (unsigned)p.Kp + (unsigned)(((tid & 7) ^ ea_swz(s)) << 4) : EA_OOB;
  }
  int t0 = 0, n = 0;                       // the chunk: K tiles t0 ... t0 + n - 1
  auto stage = [&](int t) {
    char* buf = smem + (t % S) * STAGE;
    const unsigned k = (unsigned)(t0 + t) * 128u;
#pragma unroll
    for (int i = 0; i < DA; ++i) ea_dma16(ra, va[i], k, buf + (i * NT + wave * 64) * 16);
#pragma unroll
    for (int i = 0; i < DB; ++i) ea_dma16(rw, vb[i], k, buf + BM * 128 + (i * NT + wave * 64) * 16);
  };

  f32x4 acc[FM][FN];
  ea_fp8_start<FM, FN, FMG, FNG>(p, acc, n0 + wn * (BN / WN));
  for (; t0 < p.nb; t0 += EA_F8_CH) {
    n = p.nb - t0 < EA_F8_CH ? p.nb - t0 : EA_F8_CH;
    if (t0) ea_raw_barrier();              // the chunk before this one has been read
    EaF8Scales<BM, NT> sc;
    sc.load(p, t0, n, m0, n0);
#pragma unroll
    for (int t = 0; t < S - 1; ++t)
      if (t < n) stage(t);
    sc.store(scl);
    for (int t = 0; t < n; ++t) {
      if (S > 2 && t + S - 2 < n) ea_wait_dma<(S - 2) * D>();        // (tile t + S - 2 has been issued: S - 2 younger ones are in flight)
      else ea_wait_dma<0>();
      ea_raw_barrier();
      if (t + S - 1 < n) stage(t + S - 1);
      const char* ba = smem + (t % S) * STAGE + wm * (BM / WM) * 128;
      const char* bb = smem + (t % S) * STAGE + BM * 128 + wn * (BN / WN) * 128;
      unsigned sa[FM / FMG];
      const unsigned sb = *reinterpret_cast<const unsigned*>(scl + EA_F8_CH * BM + t * 4);
#pragma unroll
      for (int g = 0; g < FM / FMG; ++g) {
        const char* q = scl + t * BM + wm * (BM / WM) + 16 * FMG * g + FMG * l15;
        sa[g] = FMG == 4 ? *reinterpret_cast<const unsigned*>(q) : FMG == 2 ? *reinterpret_cast<const uint16_t*>(q) : *reinterpret_cast<const uint8_t*>(q);
      }
      i32x8 fa[FM], fb[FN];
#pragma unroll
      for (int j = 0; j < FN; ++j) fb[j] = ea_f8_frag(bb, j * 16 + l15, lq);
#pragma unroll
      for (int i = 0; i < FM; ++i) fa[i] = ea_f8_frag(ba, i * 16 + l15, lq);
      if constexpr (EXACT) {
        f32x4 sum[FM][FN];
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int j = 0; j < FN; ++j) sum[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          f16x8 ha[FM], hb[FN];
#pragma unroll
          for (int j = 0; j < FN; ++j) hb[j] = ea_f8_half8((unsigned)fb[j][2 * u], (unsigned)fb[j][2 * u + 1], 1.0f);
#pragma unroll
          for (int i = 0; i < FM; ++i) ha[i] = ea_f8_half8((unsigned)fa[i][2 * u], (unsigned)fa[i][2 * u + 1], 1.0f);
#pragma unroll
          for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) sum[i][j] = ea_mfma_16x16x32(hb[j], ha[i], sum[i][j]);
        }
#pragma unroll
        for (int i = 0; i < FM; ++i) {
          const int e = (int)((sa[i / FMG] >> (8 * (i % FMG))) & 255) + (int)(sb & 255) - 254;
#pragma unroll
          for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][j][r] += ldexpf(sum[i][j][r], e);
        }
      } else {
        ea_static_for<FM>([&](auto ic) {
          constexpr int i = decltype(ic)::value;
#pragma unroll
          for (int j = 0; j < FN; ++j) acc[i][j] = ea_mfma_fp8_128<0, i % FMG>(fb[j], fa[i], acc[i][j], sb, sa[i / FMG]);
        });
      }
    }
  }
  ea_fp8_finish<FM, FN, FMG, FNG>(p, acc, m0 + wm * (BM / WM), m0, n0 + wn * (BN / WN));
}

// --------------------------------------------------------------------------------------------------- large-tile kernel
// 256 x 256 outputs, 8 waves (2 x 4) of 128 x 64, the phase schedule of ea_gemm8.h: a K tile (64 KiB of LDS, two of them) is worked off in
// four phases of one 64 x 32 quadrant each, 8 instructions of 16x16x128 per phase; each phase issues one half tile of the next K tile
// and waits with a counted vmcnt(4), the two wave rows run one barrier apart so that on every SIMD one wave multiplies while the other
// reads and issues.
#define EA_F8L_KT 65536
#define EA_F8L_LDS (2 * EA_F8L_KT + EA_F8_CH * 260)

__device__ __forceinline__ void ea_f8l_barrier() {           // fragment reads fly across it
#ifdef EA_EMU
  ea_emu::block_sync();
#else
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
#endif
}

__global__ __launch_bounds__(512, 2) void ea_fp8_large_kernel(EaFp8GemmParams p) {
  EA_SMEM(smem);
  const int tid = threadIdx.x, lane = tid & 63, wave = ea_uniform(tid >> 6), wm = wave >> 2, wn = wave & 3;
  const int l15 = lane & 15, lq = lane >> 4;
  int tm, tn;
  ea_fp8_tile(blockIdx.x, (p.M + 255) >> 8, (p.N + 255) >> 8, p.raster_gm, tm, tn);
  const int m0 = tm * 256, n0 = tn * 256;
  const ea_rsrc ra = ea_make_rsrc(p.a + (long long)m0 * p.Kp), rw = ea_make_rsrc(p.w + (long long)n0 * p.Kp);

  // half h of the activation rows: wave row g >> 3, its 64-row quadrant h; of the weight rows: wave column g >> 2, its 32-row quadrant h
  // (8-row groups g = 2 * wave + i).  LDS row s holds tile row 4 (s & 15) + ((s >> 4) & 3) of its 64 (activations), 16 ((s & 15) >> 2) +
  // 4 ((s >> 4) & 3) + (s & 3) of its 64 (weights)
  int la[2][2], lb[2][2];
  unsigned va[2][2], vb[2][2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int g = 2 * wave + i;
      const int as = (g >> 3) * 128 + h * 64 + (g & 7) * 8, bs = (g >> 2) * 64 + h * 32 + (g & 3) * 8;
      la[h][i] = as * 128;
      lb[h][i] = 32768 + bs * 128;
      const int sa = as + (lane >> 3), sb = bs + (lane >> 3);
      const int ar = (sa & ~63) + 4 * (sa & 15) + ((sa >> 4) & 3);
      const int br = (sb & ~63) + 16 * ((sb & 15) >> 2) + 4 * ((sb >> 4) & 3) + (sb & 3);
      va[h][i] = m0 + ar < p.M ? (unsigned)ar * (unsigned)p.Kp + (unsigned)(((lane & 7) ^ ea_swz(sa)) << 4) : EA_OOB;
      vb[h][i] = n0 + br < p.N ? (unsigned)br * (unsigned)p.Kp + (unsigned)(((lane & 7) ^ ea_swz(sb)) << 4) : EA_OOB;
    }
  unsigned koff = 0;
  char* sbuf = smem;
  auto stage_a = [&](int h) {
#pragma unroll
    for (int i = 0; i < 2; ++i) ea_dma16(ra, va[h][i], koff, sbuf + la[h][i]);
  };
  auto stage_b = [&](int h) {
#pragma unroll
    for (int i = 0; i < 2; ++i) ea_dma16(rw, vb[h][i], koff, sbuf + lb[h][i]);
  };

  f32x4 acc[8][4];
  ea_fp8_start<8, 4, 4, 4>(p, acc, n0 + wn * 64);
  i32x8 fa[4], fb[2][2];
  unsigned sa[2] = {0, 0}, sb = 0;
  auto read_a = [&](const char* buf, int qa) {
#pragma unroll
    for (int i = 0; i < 4; ++i) fa[i] = ea_f8_frag(buf, wm * 128 + qa * 64 + i * 16 + l15, lq);
  };
  auto read_b = [&](const char* buf, int qb) {
#pragma unroll
    for (int j = 0; j < 2; ++j) fb[qb][j] = ea_f8_frag(buf + 32768, wn * 64 + qb * 32 + j * 16 + l15, lq);
  };
  auto mma = [&](auto qa_c, auto qb_c) {
    constexpr int qa = decltype(qa_c)::value, qb = decltype(qb_c)::value;
#ifndef EA_EMU
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_setprio(1);
#endif
    ea_static_for<4>([&](auto ic) {
      constexpr int i = decltype(ic)::value;
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[qa * 4 + i][qb * 2 + j] = ea_mfma_fp8_128<0, i>(fb[qb][j], fa[i], acc[qa * 4 + i][qb * 2 + j], sb, sa[qa]);
    });
#ifndef EA_EMU
    __builtin_amdgcn_s_setprio(0);
#endif
  };
  constexpr std::integral_constant<int, 0> c0{};
  constexpr std::integral_constant<int, 1> c1{};

  char* const scl = smem + 2 * EA_F8L_KT;
  int t0 = 0;
  auto body = [&](int t, auto more_c) {
    constexpr bool more = decltype(more_c)::value;
    const char* buf = smem + (t & 1) * EA_F8L_KT;
    // quadrant (A0, B0); A half 0 of the next tile
    read_a(buf, 0);
    read_b(buf, 0);
    sa[0] = *reinterpret_cast<const unsigned*>(scl + t * 256 + wm * 128 + l15 * 4);
    sa[1] = *reinterpret_cast<const unsigned*>(scl + t * 256 + wm * 128 + 64 + l15 * 4);
    sb = *reinterpret_cast<const uint8_t*>(scl + EA_F8_CH * 256 + t * 4 + (wn >> 1));
    if (more) { sbuf = smem + ((t + 1) & 1) * EA_F8L_KT; koff = ea_uniform((t0 + t + 1) * 128); stage_a(0); ea_wait_dma<4>(); } else ea_wait_dma<2>();
    ea_f8l_barrier();
    mma(c0, c0);
    ea_f8l_barrier();
    // (A0, B1); B half 0
    read_b(buf, 1);
    if (more) { stage_b(0); ea_wait_dma<4>(); } else ea_wait_dma<0>();
    ea_f8l_barrier();
    mma(c0, c1);
    ea_f8l_barrier();
    // (A1, B1); B half 1
    read_a(buf, 1);
    if (more) { stage_b(1); ea_wait_dma<4>(); }
    ea_f8l_barrier();
    mma(c1, c1);
    ea_f8l_barrier();
    // (A1, B0); A half 1
    if (more) { stage_a(1); ea_wait_dma<4>(); }
    ea_f8l_barrier();
    mma(c1, c0);
    ea_f8l_barrier();
  };
  for (; t0 < p.nb; t0 += EA_F8_CH) {
    const int n = p.nb - t0 < EA_F8_CH ? p.nb - t0 : EA_F8_CH;
    if (t0) ea_raw_barrier();              // the chunk before this one has been read
    EaF8Scales<256, 512> sc;
    sc.load(p, t0, n, m0, n0);
    sbuf = smem;
    koff = ea_uniform(t0 * 128);
    stage_a(0);
    stage_b(0);
    stage_b(1);
    stage_a(1);
    sc.store(scl);
    ea_wait_dma<4>();
    ea_raw_barrier();                      // (its lgkmcnt(0) covers the scale bytes)
    if (wm == 1) ea_f8l_barrier();         // wave row 1 runs one barrier behind wave row 0
    for (int t = 0; t + 1 < n; ++t) body(t, std::true_type{});
    body(n - 1, std::false_type{});
    if (wm == 0) ea_f8l_barrier();         // both wave rows execute the same number of barriers
  }
  ea_fp8_finish<8, 4, 4, 4>(p, acc, m0 + wm * 128, m0, n0 + wn * 64);
}
