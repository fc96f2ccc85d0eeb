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

__device__ __forceinline__ float ea_fp8_act(float v, int act) {
  return act == EA_ACT_SILU ? ea_silu(v) : act == EA_ACT_GELU ? ea_gelu_erf(v) : v;
}

// acc[i][j] of one wave: activation fragments i (groups of FMG), weight fragments j (groups of FNG)
template <int FM, int FN, int FMG, int FNG>
__device__ __forceinline__ void ea_fp8_epilogue(const EaFp8GemmParams& p, const f32x4 (&acc)[FM][FN], int m0, int n0) {
  const int lane = threadIdx.x & 63, l15 = lane & 15, lq = lane >> 4;
  constexpr int NC = 4 * FNG;                       // consecutive columns of a lane
#pragma unroll
  for (int gn = 0; gn < FN / FNG; ++gn) {
    const int n = n0 + 16 * FNG * gn + NC * lq;
    float bias[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) bias[c] = 0.0f;
    if (p.bias) {
#pragma unroll
      for (int c = 0; c < NC; ++c)
        if (n + c < p.N) bias[c] = p.bias[n + c];
    }
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int m = m0 + 16 * FMG * (i / FMG) + FMG * l15 + i % FMG;
      if (m >= p.M) continue;
      float v[NC];
#pragma unroll
      for (int c = 0; c < NC; ++c) v[c] = ea_fp8_act(acc[i][gn * FNG + c / 4][c % 4] + bias[c], p.act) * p.scale;
      const long long ro = (long long)m * p.ldr + n, co = (long long)m * p.ldc + n;
      if (p.vec) {
#pragma unroll
        for (int h = 0; h < NC / 8; ++h) {
          if (n + 8 * h >= p.N) continue;
          float* u = v + 8 * h;
          if (p.residual) {
            const f16x8 r = ea_ld8(p.residual + ro + 8 * h);
#pragma unroll
            for (int c = 0; c < 8; ++c) u[c] += (float)r[c];
          }
          if (p.residual32) {
#pragma unroll
            for (int c = 0; c < 8; ++c) u[c] += p.residual32[ro + 8 * h + c];
          }
          if (p.out_f32) {
            float* o = (float*)p.out + co + 8 * h;
            *reinterpret_cast<f32x4*>(o) = f32x4{u[0], u[1], u[2], u[3]};
            *reinterpret_cast<f32x4*>(o + 4) = f32x4{u[4], u[5], u[6], u[7]};
          } else {
            f16x8 y;
#pragma unroll
            for (int c = 0; c < 8; ++c) y[c] = (f16)u[c];
            ea_st8((f16*)p.out + co + 8 * h, y);
          }
        }
      } else {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          if (n + c >= p.N) continue;
          float u = v[c];
          if (p.residual) u += (float)p.residual[ro + c];
          if (p.residual32) u += p.residual32[ro + c];
          if (p.out_f32) ((float*)p.out)[co + c] = u;
          else ((f16*)p.out)[co + c] = (f16)u;
        }
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------------- ring kernel
// BM x BN outputs, WM x WN waves, a ring of S stages of one K tile each, one barrier per tile.  At tile t a wave waits for its own
// DMA of tile t (the S - 2 younger tiles stay in flight), the barrier makes everybody's visible and says that tile t - 1 has been read;
// then tile t + S - 1 is issued into that buffer.  The scale words of tile t + 1 are loaded in front of that DMA, so the counted wait of
// the next tile covers them.
template <int BM, int BN, int WM, int WN, int S>
__global__ __launch_bounds__(64 * WM * WN) void ea_fp8_ring_kernel(EaFp8GemmParams p) {
  constexpr int NT = 64 * WM * WN, FM = BM / WM / 16, FN = BN / WN / 16;
  constexpr int FMG = FM < 4 ? FM : 4, FNG = FN < 4 ? FN : 4;
  constexpr int STAGE = (BM + BN) * 128, DA = BM * 8 / NT, DB = BN * 8 / NT, D = DA + DB;
  static_assert(BM * 8 % NT == 0 && BN * 8 % NT == 0, "whole DMA instructions");
  static_assert(128 % (BN / WN) == 0, "a wave's columns share one weight scale");
  EA_SMEM(smem);
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
  auto stage = [&](int t) {
    char* buf = smem + (t % S) * STAGE;
    const unsigned k = (unsigned)t * 128u;
#pragma unroll
    for (int i = 0; i < DA; ++i) ea_dma16(ra, va[i], k, buf + (i * NT + wave * 64) * 16);
#pragma unroll
    for (int i = 0; i < DB; ++i) ea_dma16(rw, vb[i], k, buf + BM * 128 + (i * NT + wave * 64) * 16);
  };
  // scale words: one per group of FMG fragments (rows behind M clamp to the last group of 16 stored bytes), one byte for the columns
  unsigned sa[FM / FMG], sb;
  auto scales = [&](int t) {
#pragma unroll
    for (int g = 0; g < FM / FMG; ++g) {
      long long r = m0 + wm * (BM / WM) + 16 * FMG * g + FMG * l15;
      if (r >= p.Rp) r = p.Rp - FMG;
      const uint8_t* q = p.sa + t * p.Rp + r;
      sa[g] = FMG == 4 ? *reinterpret_cast<const unsigned*>(q) : FMG == 2 ? *reinterpret_cast<const uint16_t*>(q) : *q;
    }
    int b = (n0 + wn * (BN / WN)) >> 7;
    if (b >= p.nwb) b = p.nwb - 1;
    sb = p.sw[(long long)t * p.nwb + b];
  };

  f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  scales(0);
#pragma unroll
  for (int t = 0; t < S - 1; ++t)
    if (t < p.nb) stage(t);
  for (int t = 0; t < p.nb; ++t) {
    if (S > 2 && t + 1 < p.nb) ea_wait_dma<(S - 2) * D>();
    else ea_wait_dma<0>();
    ea_raw_barrier();
    unsigned csa[FM / FMG], csb = sb;
#pragma unroll
    for (int g = 0; g < FM / FMG; ++g) csa[g] = sa[g];
    scales(t + 1 < p.nb ? t + 1 : t);
    if (t + S - 1 < p.nb) stage(t + S - 1);
    const char* ba = smem + (t % S) * STAGE + wm * (BM / WM) * 128;
    const char* bb = smem + (t % S) * STAGE + BM * 128 + wn * (BN / WN) * 128;
    i32x8 fa[FM], fb[FN];
    auto frag = [&](const char* base, int s) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(base + s * 128 + ((lq ^ ea_swz(s)) << 4));
      const u32x4 y = *reinterpret_cast<const u32x4*>(base + s * 128 + (((4 + lq) ^ ea_swz(s)) << 4));
      return i32x8{(int)x[0], (int)x[1], (int)x[2], (int)x[3], (int)y[0], (int)y[1], (int)y[2], (int)y[3]};
    };
#pragma unroll
    for (int j = 0; j < FN; ++j) fb[j] = frag(bb, j * 16 + l15);
#pragma unroll
    for (int i = 0; i < FM; ++i) fa[i] = frag(ba, i * 16 + l15);
    ea_static_for<FM>([&](auto ic) {
      constexpr int i = decltype(ic)::value;
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = ea_mfma_fp8_128<0, i % FMG>(fb[j], fa[i], acc[i][j], csb, csa[i / FMG]);
    });
  }
  ea_fp8_epilogue<FM, FN, FMG, FNG>(p, acc, m0 + wm * (BM / WM), n0 + wn * (BN / WN));
}
