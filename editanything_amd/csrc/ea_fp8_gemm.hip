// ea_fp8_gemm.hip -- the contractions on the 8-bit format: ea_gemm_fp8 (both operands in 8 bits; ea_fp8_gemm.h) and
// ea_gemm_fp8_wgrad, the weight and bias gradient of a Linear from its 8-bit input.
#include "ea_fp8_gemm.h"

int ea_forced_variant();          // ea_gemm.hip: the calling thread's ea_tuning.variant and .splits (tests)
int ea_forced_splits();

namespace {

// ---------------------------------------------------------------------------------------------------- weight gradient
//   dw[n][k] = sum_m dy[m][n] x[m][k],  x[m][k] = code * 2^E[m][k / 128];     db[n] = sum_m dy[m][n]
// The sum runs over rows, and each row has its own exponents, so the matrix unit's block scales do not apply (they belong to runs of
// the contracted axis).  x is decoded to fp16 instead and multiplied by dy as it is: every product is exact, the sums are fp32.
// fp16 holds 40 octaves, the format 220, so x goes in as x / 2^U and the accumulators count in units of 2^U: a code times 2^f, f = E - U,
// is an fp16 value for -15 <= f <= 7 (the code's smallest step 2^-9 times 2^-15 is fp16's, 448 * 2^7 is 57344).  U belongs to a block column
// of 128 and is chosen for up to 2048 rows at a time (WxUnit): from the exponents of those rows, and where it changes, the accumulators are
// multiplied by the power of two between.  Rows that do not fit one window of 23 octaves are taken in several passes over the same rows, each with
// the others' factors 0 (a block of zeros has E = 0, so padding rows among tiny ones do that).  Choosing a unit costs 0.4 us (128 x 128
// tiles) to 1 us per 2048 rows: the scale bytes' extremes are joined over the workgroup before the first factor can be written (616 x 1280 x 1024 13.8 ->
// 14.2 us, 8192^3 971 -> 988).
// Both operands have the contracted axis as their ROW axis, so they go to LDS row-major and the fragments are read transposed: 16 lanes
// take a 4 x 16 (fp16) or 8 x 16 (codes) block and each ends up with consecutive rows of one column.  Bound by the matrix unit at
// the fp16 rate: 8192^3 937 us = 1173 TFLOP/s (the library's fp16 product on the same card: 1314).
// First the kernel for any N and alignment: 128 x 128 tiles, both operands through registers, x decoded on the way to LDS.
struct WgradParams {
  const f16* dy; const uint8_t* x; const uint8_t* sx;
  float* dw; float* db;              // or one [N][K] + [N] partial per slice
  int M, N, K, Kp, tiles_n, tiles_k, splits, rows_per_split; long long Rp, part;
  int vec;                           // dy rows are 16-byte aligned (N a multiple of 8)
};

constexpr int WG_T = 128, WG_R = 64;                     // tile columns of n and of k, rows per step
constexpr int WG_BUF = WG_R * WG_T * 2;                  // one operand's tile: 16 KiB
constexpr int WG_CH = 32 * WG_R, WG_LDS = 2 * WG_BUF + 16;      // rows under one choice of the unit; the tiles and the waves' extremes
// byte of (row, column) in a tile
__device__ __forceinline__ int wg_at(int r, int c) { return r * 256 + ((((c >> 4) ^ r) & 7) << 5) + (c & 15) * 2; }

// 4 rows of one column of fp16 (the builtin, not ea_prims.h's inline assembly: the compiler then knows when the registers are written)
__device__ __forceinline__ f16x4 wg_read_tr16(const char* ptr) {
#ifdef EA_EMU
  return ea_lds_read_tr16<0>(ptr);
#else
  typedef __fp16 h4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) h4*)ptr));
#endif
}
__device__ __forceinline__ f16x8 wg_frag(const char* buf, int r0, int c0, int lane) {
  const int q = lane >> 4, i = lane & 15;
  // rows r0 + 4 q .. + 3 and r0 + 16 + 4 q .. + 3: the order of rows inside a step is the same for both operands
  const char* a = buf + wg_at(r0 + 4 * q + (i >> 2), c0 + (i & 3) * 4);
  const char* b = buf + wg_at(r0 + 16 + 4 * q + (i >> 2), c0 + (i & 3) * 4);
  const f16x4 lo = wg_read_tr16(a), hi = wg_read_tr16(b);
  return f16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

// The unit 2^(u - 127) of the accumulators of one block column and the exponent bytes that are still to be taken of the rows at hand.
// Accumulators are below 2^62 units (2^30 rows of |dy| 65504 times 57344) and worth keeping from 2^-72 on (2^-24 of the smallest product, 2^-24
// times 2^-24), so within WX_REACH octaves a change of units neither overflows fp32 nor loses anything in its subnormal numbers; a wider one adds the
// sums to the output and starts them anew.
constexpr int WX_NONE = -1000, WX_REACH = 50;
struct WxUnit {
  int u = WX_NONE, bottom = 0, top = 0, lo = 0, hi = -1;
  // The next pass: the unit becomes u, its rows have the bytes from ... to (none: from > to).  Returns true where the sums, still in
  // units of `old`, have to be put away first
  __device__ __forceinline__ bool next(int& from, int& to, int& old) {
    old = u;
    from = lo;
    to = hi;
    if (hi < lo) return false;
    if (hi - u > 7 || lo - u < -15) {
      if (hi - 22 > from) from = hi - 22;
      u = hi - 7;
    }
    hi = from - 1;
    const int b = u < bottom ? u : bottom, t = u > top ? u : top;
    const bool first = old == WX_NONE, away = !first && t - b > WX_REACH;
    bottom = first || away ? u : b;
    top = first || away ? u : t;
    if (first) old = u;
    return away;
  }
};
// The lane's number, made anew: what is needed once in 32 steps is not kept in registers over them (kept ones were spilled, and reading a spilled one
// back waits for all DMA in flight)
__device__ __forceinline__ int wg_fresh_lane() {
#ifdef EA_EMU
  return ea_emu::lane_id();
#else
  unsigned z = 0;
  asm volatile("" : "+s"(z));
  return (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, z));
#endif
}
// Extremes of the bytes of some rows: (hi, 255 - lo) in the halves of a word, whose maximum is taken for both at once
__device__ __forceinline__ unsigned wx_max(unsigned a, unsigned b) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
__device__ __forceinline__ unsigned wx_word(int byte) { return (unsigned)byte | (unsigned)(255 - byte) << 16; }
// each wave's word to red[wave]; after a barrier the words of waves first, first + step, ... are joined
__device__ __forceinline__ void wx_range_put(unsigned* red, unsigned w, int lane, int wave) {
  w = ea_f2u(ea_group_reduce<64>(ea_u2f(w), [](float a, float b) { return ea_u2f(wx_max(ea_f2u(a), ea_f2u(b))); }));
  if (lane == 0) red[wave] = w;
}
template <int FIRST, int STEP, int WAVES>
__device__ __forceinline__ void wx_range_get(const unsigned* red, WxUnit& x) {
  unsigned w = red[FIRST];
#pragma unroll
  for (int i = FIRST + STEP; i < WAVES; i += STEP) w = wx_max(w, red[i]);
  w = (unsigned)ea_uniform((int)w);
  x.hi = (int)(w & 0xffff);
  x.lo = 255 - (int)(w >> 16);
}
// acc *= 2^d, or = 0
template <int I, int J>
__device__ __forceinline__ void wx_rescale(f32x4 (&acc)[I][J], bool zero, int d) {
  if (!zero && d == 0) return;
#pragma unroll
  for (int i = 0; i < I; ++i)
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[i][j][r] = zero ? 0.0f : ldexpf(acc[i][j][r], d);
}

__device__ __forceinline__ void wg_decode16(u32x4 w, float s, f16x8& a, f16x8& b) {
  float v[16];
#pragma unroll
  for (int i = 0; i < 4; ++i) ea_fp8_unpack4(w[i], v + 4 * i);
#pragma unroll
  for (int j = 0; j < 8; ++j) { a[j] = (f16)(v[j] * s); b[j] = (f16)(v[8 + j] * s); }
}

// Accumulators in units of 2^(u - 127) to dw, or added to it: fragment (i, j) holds the 4 columns k + 16 j of row row(i) + l of the tile (D^T: a
// lane has 4 consecutive k of one n).  `out` starts at the tile's first row and ends with the matrix; columns that are not there lie 2 GiB on.
template <int I, int J, typename F>
__device__ __forceinline__ void wg_put(ea_rows out, const f32x4 (&acc)[I][J], F row, int l, int k, int K, int u, bool add) {
#ifndef EA_EMU
  asm volatile("" : "+v"(l), "+v"(k));     // (the offsets are made here: over the loop they would take the accumulators' registers)
#endif
  if ((K & 3) == 0) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const unsigned c = k + 16 * j < K ? (unsigned)(k + 16 * j) * 4u : EA_F8_NOWHERE;
#pragma unroll
      for (int i = 0; i < I; ++i) {
        const unsigned o = c + (unsigned)(row(i) + l) * (unsigned)K * 4u;
        f32x4 v = acc[i][j];
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = ldexpf(v[r], u - 127);
        if (add) v += __builtin_bit_cast(f32x4, ea_rows_load(out, o));
        ea_rows_store(out, o, __builtin_bit_cast(u32x4, v));
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const unsigned c = k + 16 * j + r < K ? (unsigned)(k + 16 * j + r) * 4u : EA_F8_NOWHERE;
#pragma unroll
        for (int i = 0; i < I; ++i) {
          const unsigned o = c + (unsigned)(row(i) + l) * (unsigned)K * 4u;
          float v = ldexpf(acc[i][j][r], u - 127);
          if (add) v += ea_u2f(ea_rows_load1(out, o));
          ea_rows_store1(out, o, ea_f2u(v));
        }
      }
  }
}

__global__ __launch_bounds__(256) void ea_fp8_wgrad_kernel(WgradParams p) {
  EA_SMEM(smem);
  const int tid = threadIdx.x, lane = tid & 63, wave = ea_uniform(tid >> 6), wn = wave >> 1, wk = wave & 1;
  const int tile = blockIdx.x, tn = tile / p.tiles_k, tk = tile - tn * p.tiles_k;
  const int n0 = tn * WG_T, k0 = tk * WG_T;
  const int m_begin = blockIdx.y * p.rows_per_split;
  const int m_end = m_begin + p.rows_per_split < p.M ? m_begin + p.rows_per_split : p.M;

  u32x4 xr[2];
  float xs[2];
  f16x8 dr[4];
  WxUnit unit;
  int from = 0, to = 0;
  auto load = [&](int m0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = i * 32 + (tid >> 3), m = m0 + r, c = (tid & 7) * 16;
      const bool ok = m < m_end;
      const long long mm = ok ? m : m_begin;
      xr[i] = *reinterpret_cast<const u32x4*>(p.x + mm * p.Kp + k0 + c);
      const int b = p.sx[(long long)tk * p.Rp + mm];
      xs[i] = ok && b >= from && b <= to ? ldexpf(1.0f, b - unit.u) : 0.0f;
      if (!ok) xr[i] = u32x4{0, 0, 0, 0};                  // (a NaN code must not reach the sum)
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = i * 16 + (tid >> 4), m = m0 + r, n = n0 + (tid & 15) * 8;
      const bool ok = m < m_end;
      const f16* d = p.dy + (long long)(ok ? m : m_begin) * p.N;
      if (p.vec) {
        dr[i] = ea_ld8(d + (n < p.N ? n : 0));
        if (!ok || n >= p.N) dr[i] = ea_zero8();
      } else if (ok && n + 8 <= p.N) {
        dr[i] = ea_ld8u(d + n);            // (rows that start anywhere)
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) dr[i][j] = ok && n + j < p.N ? d[n + j] : (f16)0.0f;
      }
    }
  };
  auto store = [&]() {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = i * 32 + (tid >> 3), c = (tid & 7) * 16;
      f16x8 a, b;
      wg_decode16(xr[i], xs[i], a, b);
      *reinterpret_cast<f16x8*>(smem + WG_BUF + wg_at(r, c)) = a;
      *reinterpret_cast<f16x8*>(smem + WG_BUF + wg_at(r, c) + 16) = b;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<f16x8*>(smem + wg_at(i * 16 + (tid >> 4), (tid & 15) * 8)) = dr[i];
  };

  f32x4 acc[4][4], accb[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    accb[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  f16x8 ones;
#pragma unroll
  for (int j = 0; j < 8; ++j) ones[j] = (f16)1.0f;
  unsigned* const red = reinterpret_cast<unsigned*>(smem + 2 * WG_BUF);
  float* const dw = p.dw + (long long)blockIdx.y * p.part;
  const ea_rows out = ea_make_rows(dw + (long long)n0 * p.K, (long long)(p.N - n0) * p.K * 4);
  const int l15 = lane & 15, lq = lane >> 4;
  bool stored = false;
  auto put = [&](int u) {
    wg_put(out, acc, [&](int i) { return wn * 64 + i * 16; }, l15, k0 + wk * 64 + 4 * lq, p.K, u, stored);
    stored = true;
  };
  bool again = false;                      // another pass over the same rows
  for (int c0 = m_begin;;) {
    const bool end = c0 >= m_end;
    const int c1 = m_end - c0 < WG_CH ? m_end : c0 + WG_CH;
    if (!end && !again) {
      unsigned w = 0;
#pragma unroll
      for (int u = 0; u < WG_CH / 256; ++u) {
        const int m = c0 + u * 256 + tid;
        w = wx_max(w, wx_word(p.sx[(long long)tk * p.Rp + (m < c1 ? m : c0)]));      // (the first row once more changes nothing)
      }
      wx_range_put(red, w, lane, wave);
      __syncthreads();
      wx_range_get<0, 1, 4>(red, unit);
    }
    int old;
    const bool away = unit.next(from, to, old);
    if (end || away) put(old);
    if (end) break;
    wx_rescale(acc, away, old - unit.u);
    const bool sums = tk == 0 && wk == 0 && !again;
    load(c0);
    for (int m0 = c0; m0 < c1; m0 += WG_R) {
      __syncthreads();
      store();
      __syncthreads();
      if (m0 + WG_R < c1) load(m0 + WG_R);
#pragma unroll
      for (int h = 0; h < WG_R; h += 32) {
        f16x8 fd[4], fx[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) fd[i] = wg_frag(smem, h, wn * 64 + i * 16, lane);
#pragma unroll
        for (int j = 0; j < 4; ++j) fx[j] = wg_frag(smem + WG_BUF, h, wk * 64 + j * 16, lane);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = ea_mfma_16x16x32(fx[j], fd[i], acc[i][j]);
        if (sums)
#pragma unroll
          for (int i = 0; i < 4; ++i) accb[i] = ea_mfma_16x16x32(ones, fd[i], accb[i]);
      }
    }
    again = unit.lo <= unit.hi;
    if (!again) c0 += WG_CH;
  }
  float* db = p.splits > 1 ? dw + (long long)p.N * p.K : p.db;
  if (tk == 0 && wk == 0 && lq == 0)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = n0 + wn * 64 + i * 16 + l15;
      if (n < p.N) db[n] = accb[i][0];
    }
}

// -------------------------------------------------------------------------------------------- weight gradient, large tiles
// 256 n x 256 k, 8 waves (2 x 4) of 128 x 64, 64 rows per step, two steps of LDS, in the manner of ea_fp8_gemm.h's large kernel: four
// phases of one 64 x 32 quadrant (16 MFMAs), each a load part and a multiply part with a barrier behind either, the two wave rows one
// barrier apart, so that on every SIMD one wave multiplies while the other reads, decodes and issues DMA.
// Both operands go to LDS as they are.  dy: half h holds the 64-column quadrants h of both wave rows, rows of 256 bytes, read with
// ds_read_b64_tr_b16; x: half h holds the 32-column quadrants h of the four wave columns, rows of 128 bytes of CODES, read with
// ds_read_b64_tr_b8: 16 lanes take 8 rows x 16 bytes and each gets 8 rows of one column.  The codes become fp16 in registers,
//     x / 2^U = (code 2^-8) * 2^(E - U + 8):   the conversion's own scale does the first factor, a packed fp16 product with the rows' 8
// scale factors (one 16-byte LDS read for 8 rows) the second; both are exact inside the unit's window.
// The load parts: L0 reads dy quadrant 0, L1 reads and decodes x quadrant 1, L2 reads dy quadrant 1, L3 reads and decodes the next
// step's x quadrant 0 (1.58 us per step with the chip two fifths full; decoding in the multiply parts
// 1.71, spreading the dy reads over all four load parts 1.61).  DMA of the next step: x in L0, dy 0 in L1,
// dy 1 in L2.  What L(q) issues is waited for in L(q + 2) (counted: the younger two parts' DMA stays in flight) and first read in
// L(q + 3), one barrier after the lagging wave row's wait.
constexpr int WL_DY = 32768, WL_X = 16384, WL_STEP = WL_DY + WL_X, WL_CH = 32;      // bytes per step; steps whose scale factors are in LDS
constexpr int WL_SCL = 2 * WL_STEP, WL_RED = WL_SCL + WL_CH * 2 * 64 * 2, WL_LDS = WL_RED + 32;

// 32-byte piece of a dy row, 16-byte piece of an x row: XORed so that the rows that a wave reads together cover the banks evenly
__device__ __forceinline__ int wl_dy_swz(int r) { return (r & 3) | ((r >> 1) & 4); }
__device__ __forceinline__ int wl_x_swz(int r) { return (r >> 1) & 7; }

#ifdef EA_EMU
// ds_read_b64_tr_b8: 16 lanes take 8 rows x 16 bytes (lanes 2 r, 2 r + 1: row r); lane i gets column i
inline u32x2 wl_emu_tr8(const char* ptr) {
  char* sc = ea_emu::wave_scratch();
  const int l = ea_emu::lane_id(), g = l & ~15, i = l & 15;
  memcpy(sc + l * 64, ptr, 8);
  ea_emu::wave_sync();
  uint8_t b[8];
  for (int r = 0; r < 8; ++r) b[r] = (uint8_t)sc[(g + 2 * r + (i >> 3)) * 64 + (i & 7)];
  ea_emu::wave_sync();
  u32x2 v;
  memcpy(&v, b, 8);
  return v;
}
#endif
// The fragment reads of one phase.  Inline assembly, because the compiler waits for all LDS-DMA in front of a transposed read that it
// knows (its address may be the one being filled); with the wait for the reads in the same block, no register is in flight behind it.
// Fragment i: rows 8 lq ... + 7 of both 32-row halves.
template <int Q>
__device__ __forceinline__ void wl_read_d(const char* a0, const char* a1, const char* a2, const char* a3, f16x8 (&f)[4][2]) {
  const char* const ptr[4] = {a0, a1, a2, a3};
#ifdef EA_EMU
  for (int i = 0; i < 4; ++i)
    for (int ks = 0; ks < 2; ++ks) {
      const f16x4 lo = ea_lds_read_tr16<0>(ptr[i] + Q + ks * 8192), hi = ea_lds_read_tr16<0>(ptr[i] + Q + ks * 8192 + 1024);
      f[i][ks] = f16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    }
#else
  unsigned ad[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) ad[i] = (unsigned)(uintptr_t)ptr[i];
  f16x4 r[4][4];
  asm volatile(
      "ds_read_b64_tr_b16 %0, %16 offset:%20\n\tds_read_b64_tr_b16 %1, %16 offset:%21\n\t"
      "ds_read_b64_tr_b16 %2, %16 offset:%22\n\tds_read_b64_tr_b16 %3, %16 offset:%23\n\t"
      "ds_read_b64_tr_b16 %4, %17 offset:%20\n\tds_read_b64_tr_b16 %5, %17 offset:%21\n\t"
      "ds_read_b64_tr_b16 %6, %17 offset:%22\n\tds_read_b64_tr_b16 %7, %17 offset:%23\n\t"
      "ds_read_b64_tr_b16 %8, %18 offset:%20\n\tds_read_b64_tr_b16 %9, %18 offset:%21\n\t"
      "ds_read_b64_tr_b16 %10, %18 offset:%22\n\tds_read_b64_tr_b16 %11, %18 offset:%23\n\t"
      "ds_read_b64_tr_b16 %12, %19 offset:%20\n\tds_read_b64_tr_b16 %13, %19 offset:%21\n\t"
      "ds_read_b64_tr_b16 %14, %19 offset:%22\n\tds_read_b64_tr_b16 %15, %19 offset:%23\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(r[0][0]), "=&v"(r[0][1]), "=&v"(r[0][2]), "=&v"(r[0][3]), "=&v"(r[1][0]), "=&v"(r[1][1]), "=&v"(r[1][2]), "=&v"(r[1][3]),
        "=&v"(r[2][0]), "=&v"(r[2][1]), "=&v"(r[2][2]), "=&v"(r[2][3]), "=&v"(r[3][0]), "=&v"(r[3][1]), "=&v"(r[3][2]), "=&v"(r[3][3])
      : "v"(ad[0]), "v"(ad[1]), "v"(ad[2]), "v"(ad[3]), "n"(Q), "n"(Q + 1024), "n"(Q + 8192), "n"(Q + 9216)
      : "memory");
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
      f[i][ks] = __builtin_shufflevector(r[i][2 * ks], r[i][2 * ks + 1], 0, 1, 2, 3, 4, 5, 6, 7);
#endif
}
template <int Q>
__device__ __forceinline__ void wl_read_x(const char* a0, const char* a1, u32x2 (&f)[2][2]) {
#ifdef EA_EMU
  for (int j = 0; j < 2; ++j)
    for (int ks = 0; ks < 2; ++ks) f[j][ks] = wl_emu_tr8((j ? a1 : a0) + Q + ks * 4096);
#else
  asm volatile("ds_read_b64_tr_b8 %0, %4 offset:%6\n\tds_read_b64_tr_b8 %1, %4 offset:%7\n\t"
               "ds_read_b64_tr_b8 %2, %5 offset:%6\n\tds_read_b64_tr_b8 %3, %5 offset:%7\n\ts_waitcnt lgkmcnt(0)"
               : "=&v"(f[0][0]), "=&v"(f[0][1]), "=&v"(f[1][0]), "=&v"(f[1][1])
               : "v"((unsigned)(uintptr_t)a0), "v"((unsigned)(uintptr_t)a1), "n"(Q), "n"(Q + 4096)
               : "memory");
#endif
}
// LDS-DMA through a descriptor with an end: what lies behind it arrives as zeros
__device__ __forceinline__ void wl_dma16(ea_rows r, unsigned off, char* lds_base) {
#ifdef EA_EMU
  const u32x4 v = ea_rows_load(r, off);
  memcpy(lds_base + 16 * ea_emu::lane_id(), &v, 16);
#else
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds_base, 16, off, 0, 0, 0);
#endif
}
// 8 codes times their rows' factors
__device__ __forceinline__ f16x8 wl_decode8(u32x2 w, f16x8 s) {
  const f16x8 h = ea_f8_half8(w[0], w[1], 0.00390625f);
#ifdef EA_EMU
  f16x8 o;
  for (int j = 0; j < 8; ++j) o[j] = (f16)((float)h[j] * (float)s[j]);
  return o;
#else
  return h * s;
#endif
}
// 2^(E - U + 8) as fp16 from the stored byte (-7 ... 15 inside a window; less where the unit could not follow); 0 for a row of another pass
__device__ __forceinline__ f16 wl_factor(int byte, int unit, int from, int to) {
  const int e = byte - unit + 8;
  const unsigned short u = byte < from || byte > to ? 0 : e >= -14 ? (unsigned short)((e + 15) << 10) : e >= -24 ? (unsigned short)(1 << (e + 24)) : 0;
  return __builtin_bit_cast(f16, u);
}

// an MFMA operand of ones: every row of the product is the column sums of the other operand.  One accumulator per fragment: where two
// fragments shared one (each with a single row of ones), the zeros times an infinity of one's column made NaN of the other's sum.  On
// the vector unit the sums cost 3 % of 8192^3 and 5 % of 616 x 1280 x 1024.
__device__ __forceinline__ f16x8 wl_ones() {
  unsigned u = 0x3c003c00u;
#ifndef EA_EMU
  asm volatile("" : "+v"(u));              // (made where it is used: kept over the loop, its four registers were spilled)
#endif
  return __builtin_bit_cast(f16x8, u32x4{u, u, u, u});
}

// ------------------------------------------------------------------------------------- weight gradient, 128 x 128 tiles
// Few or small outputs: 4 waves (2 x 2) of 64 x 64, a ring of three 64-row steps (24 KiB each, two workgroups per CU), one barrier per
// step; operands, fragment reads and decoding as in the large kernel.
constexpr int WR_S = 3, WR_DY = 16384, WR_STEP = 24576, WR_CH = 32, WR_SCL = WR_S * WR_STEP, WR_RED = WR_SCL + WR_CH * 64 * 2, WR_LDS = WR_RED + 16;
__global__ __launch_bounds__(256, 2) void ea_fp8_wgrad_ring_kernel(WgradParams p) {
  EA_SMEM(smem);
  const int tid = threadIdx.x, lane = tid & 63, wave = ea_uniform(tid >> 6), wm = wave >> 1, wn = wave & 1;
  const int l15 = lane & 15, lq = lane >> 4;
  const int tn = ea_uniform((int)blockIdx.x / p.tiles_k), tk = ea_uniform((int)blockIdx.x - tn * p.tiles_k);
  const int n0 = tn * 128, k0 = tk * 128;
  const int m_begin = blockIdx.y * p.rows_per_split;
  const int m_end = m_begin + p.rows_per_split < p.M ? m_begin + p.rows_per_split : p.M;
  const int steps = (m_end - m_begin + 63) >> 6;
  unsigned vd[4], vx[2];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 4 * (4 * wave + i) + (lane >> 4), c = ((((lane & 15) >> 1) ^ wl_dy_swz(r)) * 16) + (lane & 1) * 8;
    vd[i] = n0 + c < p.N ? ((unsigned)r * (unsigned)p.N + (unsigned)c) * 2u : EA_F8_NOWHERE;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 8 * (2 * wave + i) + (lane >> 3);
    vx[i] = (unsigned)r * (unsigned)p.Kp + (unsigned)(((lane & 7) ^ wl_x_swz(r)) * 16);
  }
  ea_rows rd = ea_make_rows(p.dy, 0), rx = ea_make_rows(p.x, 0);
  auto stage = [&](int t) {                // t: step of the chunk
    char* buf = smem + (t % WR_S) * WR_STEP;
    const unsigned od = ea_uniform((unsigned)t * 64u * (unsigned)p.N * 2u), ox = ea_uniform((unsigned)t * 64u * (unsigned)p.Kp);
#pragma unroll
    for (int i = 0; i < 4; ++i) wl_dma16(rd, vd[i] + od, buf + (4 * wave + i) * 1024);
#pragma unroll
    for (int i = 0; i < 2; ++i) wl_dma16(rx, vx[i] + ox, buf + WR_DY + (2 * wave + i) * 1024);
  };
  int ad[4], ax[4];                        // fragment i is the wave's 16-column group i ^ 2 wn: it sums dy over the groups of fragments 0 and 1
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 8 * lq + (l15 >> 2), s = 8 * lq + (l15 >> 1);
    ad[i] = r * 256 + (((wm * 4 + (i ^ (2 * wn))) ^ wl_dy_swz(r)) << 5) + (l15 & 3) * 8;
    ax[i] = WR_DY + s * 128 + (((wn * 4 + i) ^ wl_x_swz(s)) << 4) + (l15 & 1) * 8;
  }
  f32x4 acc[4][4], accb[2] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}, f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  char* const scl = smem + WR_SCL;
  unsigned* const red = reinterpret_cast<unsigned*>(smem + WR_RED);
  WxUnit unit;
  float* const dw = p.dw + (long long)blockIdx.y * p.part;
  const ea_rows out = ea_make_rows(dw + (long long)n0 * p.K, (long long)(p.N - n0) * p.K * 4);
  bool stored = false;
  auto put = [&](int u) {
    wg_put(out, acc, [&](int i) { return wm * 64 + (i ^ (2 * wn)) * 16; }, l15, k0 + wn * 64 + 4 * lq, p.K, u, stored);
    stored = true;
  };
  bool again = false;                      // another pass over the same chunk
  for (int t0 = 0;;) {
    const bool end = t0 >= steps;
    const int n = steps - t0 < WR_CH ? steps - t0 : WR_CH;
    const long long mc = m_begin + t0 * 64ll;
    const bool sums = tk == 0 && !again;
    if (t0 || again) ea_raw_barrier();     // the chunk (pass) before this one has been read
    int sb[WR_CH * 64 / 256];
    if (!end) {
      const int left = (int)(m_end - mc);
      const uint8_t* const sx = p.sx + tk * p.Rp + mc;
#pragma unroll
      for (int u = 0; u < WR_CH * 64 / 256; ++u) sb[u] = sx[u * 256 + tid < left ? u * 256 + tid : left - 1];      // (behind the end: zeros, any factor)
      rd = ea_make_rows(p.dy + mc * p.N + n0, ((m_end - mc) * p.N - n0) * 2);
      rx = ea_make_rows(p.x + mc * p.Kp + k0, (m_end - mc) * p.Kp - k0);
#pragma unroll
      for (int t = 0; t < WR_S - 1; ++t)
        if (t < n) stage(t);
      if (!again) {
        unsigned w = 0;
#pragma unroll
        for (int u = 0; u < WR_CH * 64 / 256; ++u) w = wx_max(w, wx_word(sb[u]));
        wx_range_put(red, w, lane, wave);
        ea_raw_barrier();
        wx_range_get<0, 1, 4>(red, unit);
      }
    }
    int from, to, old;
    const bool away = unit.next(from, to, old);
    if (end || away) put(old);
    if (end) break;
    wx_rescale(acc, away, old - unit.u);
#pragma unroll
    for (int u = 0; u < WR_CH * 64 / 256; ++u) *reinterpret_cast<f16*>(scl + (u * 256 + tid) * 2) = wl_factor(sb[u], unit.u, from, to);
    for (int t = 0; t < n; ++t) {
      if (t + WR_S - 2 < n) ea_wait_dma<(WR_S - 2) * 6>();           // (step t + WR_S - 2 has been issued: it alone may be in flight)
      else ea_wait_dma<0>();
      ea_raw_barrier();
      if (t + WR_S - 1 < n) stage(t + WR_S - 1);
      const char* buf = smem + (t % WR_S) * WR_STEP;
      f16x8 sc[2], fa[4][2], fx[4][2];
      u32x2 w[2][2];
      sc[0] = *reinterpret_cast<const f16x8*>(scl + (t * 64 + 8 * lq) * 2);
      sc[1] = *reinterpret_cast<const f16x8*>(scl + (t * 64 + 32 + 8 * lq) * 2);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        wl_read_x<0>(buf + ax[2 * h], buf + ax[2 * h + 1], w);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int ks = 0; ks < 2; ++ks) fx[2 * h + j][ks] = wl_decode8(w[j][ks], sc[ks]);
      }
      wl_read_d<0>(buf + ad[0], buf + ad[1], buf + ad[2], buf + ad[3], fa);
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = ea_mfma_16x16x32(fx[j][ks], fa[i][ks], acc[i][j]);
        if (sums) {
          accb[0] = ea_mfma_16x16x32(wl_ones(), fa[0][ks], accb[0]);
          accb[1] = ea_mfma_16x16x32(wl_ones(), fa[1][ks], accb[1]);
        }
      }
    }
    again = unit.lo <= unit.hi;
    if (!again) t0 += WR_CH;
  }
  float* db = p.splits > 1 ? dw + (long long)p.N * p.K : p.db;
  if (tk == 0 && lq == 0)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int n = n0 + wm * 64 + (i ^ (2 * wn)) * 16 + l15;
      if (n < p.N) db[n] = accb[i][0];
    }
}

__global__ __launch_bounds__(512, 2) void ea_fp8_wgrad_large_kernel(WgradParams p) {
  EA_SMEM(smem);
  const int tid = threadIdx.x, lane = tid & 63, wave = ea_uniform(tid >> 6), wm = wave >> 2, wn = wave & 3;
  const int l15 = lane & 15, lq = lane >> 4;
  int tn, tk;
  {   // an XCD's workgroups share dy columns and x columns: one contiguous run of tiles, all k tiles of an n tile first
    const int n = p.tiles_n * p.tiles_k, q = n >> 3, r = n & 7, xcd = blockIdx.x & 7;
    const int t = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (blockIdx.x >> 3);
    tn = ea_uniform(t / p.tiles_k);
    tk = ea_uniform(t - tn * p.tiles_k);
  }
  const int n0 = tn * 256, k0 = tk * 256;
  const int m_begin = blockIdx.y * p.rows_per_split;
  const int m_end = m_begin + p.rows_per_split < p.M ? m_begin + p.rows_per_split : p.M;
  const int steps = (m_end - m_begin + 63) >> 6;

  // DMA: dy half h, instruction i of this wave: rows 4 (2 wave + i) ... + 3 (256 bytes each: columns 64 h of wave row 0, then of wave row 1);
  // x half h: rows 8 wave ... + 7 (128 bytes each: 32 h of the four wave columns)
  unsigned vd[2][2], vx[2];                // columns that are not there start at 2 GiB, behind every descriptor
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 4 * (2 * wave + i) + (lane >> 4), piece = ((lane & 15) >> 1) ^ wl_dy_swz(r);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = (piece >> 2) * 128 + h * 64 + (piece & 3) * 16 + (lane & 1) * 8;
      vd[h][i] = n0 + c < p.N ? ((unsigned)r * (unsigned)p.N + (unsigned)c) * 2u : EA_F8_NOWHERE;
    }
  }
  {
    const int r = 8 * wave + (lane >> 3), piece = (lane & 7) ^ wl_x_swz(r);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = (piece >> 1) * 64 + h * 32 + (piece & 1) * 16;
      vx[h] = k0 + c < p.Kp ? (unsigned)r * (unsigned)p.Kp + (unsigned)c : EA_F8_NOWHERE;
    }
  }
  char* sbuf = smem;
  unsigned od = 0, ox = 0;
  // descriptors of a chunk: from its first row to the slice's last one (rows behind it read as zeros)
  ea_rows rd = ea_make_rows(p.dy, 0), rx = ea_make_rows(p.x, 0);
  int t0 = 0;                              // the chunk's first step
  auto begin = [&](int t) {                // t: step of the chunk
    sbuf = smem + (t & 1) * WL_STEP;
    od = ea_uniform((unsigned)t * 64u * (unsigned)p.N * 2u);
    ox = ea_uniform((unsigned)t * 64u * (unsigned)p.Kp);
  };
  auto stage_d = [&](int h) {
#pragma unroll
    for (int i = 0; i < 2; ++i) wl_dma16(rd, vd[h][i] + od, sbuf + h * 16384 + (2 * wave + i) * 1024);
  };
  auto stage_x = [&](int h) { wl_dma16(rx, vx[h] + ox, sbuf + WL_DY + h * 8192 + wave * 1024); };

  f32x4 acc[8][4], accb = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  f16x8 fa[4][2];
  f16x8 fb0[2][2], fb1[2][2], fbn[2][2];  // quadrants 0 and 1, the next step's 0
  // rows 8 lq ... + 7 of a 32-row half of the step are this lane group's share of one MFMA, for both operands.  The swizzle does not
  // change over the 32-row halves or the 4-row quarters of a group: one address per fragment, the rest are immediate offsets
  // (fragment i is the quadrant's 16-column group i ^ wn: each wave column sums dy over the group of its own fragment 0)
  int ad[4], ax[2];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 8 * lq + (l15 >> 2);
    ad[i] = r * 256 + (((wm * 4 + (i ^ wn)) ^ wl_dy_swz(r)) << 5) + (l15 & 3) * 8;
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int r = 8 * lq + (l15 >> 1);
    ax[j] = WL_DY + r * 128 + (((wn * 2 + j) ^ wl_x_swz(r)) << 4) + (l15 & 1) * 8;
  }
  auto read_d = [&](const char* buf, auto qa_c) { wl_read_d<decltype(qa_c)::value * 16384>(buf + ad[0], buf + ad[1], buf + ad[2], buf + ad[3], fa); };
  constexpr std::integral_constant<int, 0> c0{};
  constexpr std::integral_constant<int, 1> c1{};
  char* const scl = smem + WL_SCL;         // [step of the chunk][kb of the tile][64]
  auto read_x = [&](int t, auto qb_c, f16x8 (&f)[2][2]) {          // codes and factors of one quadrant -> fragments
    const char* buf = smem + (t & 1) * WL_STEP;
    f16x8 sc[2];
    u32x2 w[2][2];
    sc[0] = *reinterpret_cast<const f16x8*>(scl + (t * 128 + (wn >> 1) * 64 + 8 * lq) * 2);
    sc[1] = *reinterpret_cast<const f16x8*>(scl + (t * 128 + (wn >> 1) * 64 + 32 + 8 * lq) * 2);
    wl_read_x<decltype(qb_c)::value * 8192>(buf + ax[0], buf + ax[1], w);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) f[j][ks] = wl_decode8(w[j][ks], sc[ks]);
  };
  auto mma = [&](auto qa_c, auto qb_c, const f16x8 (&fb)[2][2], bool sums) {
    constexpr int qa = decltype(qa_c)::value, qb = decltype(qb_c)::value;
#ifndef EA_EMU
    __builtin_amdgcn_s_setprio(1);
#endif
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[qa * 4 + i][qb * 2 + j] = ea_mfma_16x16x32(fb[j][ks], fa[i][ks], acc[qa * 4 + i][qb * 2 + j]);
      if (sums) accb = ea_mfma_16x16x32(wl_ones(), fa[0][ks], accb);
    }
#ifndef EA_EMU
    __builtin_amdgcn_s_setprio(0);
#endif
  };
  // dy's column sums, one accumulator's worth per workgroup: quadrants 0 by the first k tile, 1 by the second (there are two: wgrad_plan)
  bool again = false;                      // another pass over the same chunk
  auto body = [&](int t, auto more_c) {
    constexpr bool more = decltype(more_c)::value;
    const char* buf = smem + (t & 1) * WL_STEP;
    if (more) { begin(t + 1); stage_x(0); stage_x(1); }
    read_d(buf, c0);
    if (more) ea_wait_dma<2>(); else ea_wait_dma<0>();
    ea_f8l_barrier();
    mma(c0, c0, fb0, tk == 0 && !again);
    ea_f8l_barrier();
    if (more) stage_d(0);
    read_x(t, c1, fb1);
    if (more) ea_wait_dma<4>();
    ea_f8l_barrier();
    mma(c0, c1, fb1, false);
    ea_f8l_barrier();
    if (more) stage_d(1);
    read_d(buf, c1);
    if (more) ea_wait_dma<4>();
    ea_f8l_barrier();
    mma(c1, c1, fb1, tk == 1 && !again);
    ea_f8l_barrier();
    if (more) {
      read_x(t + 1, c0, fbn);
      ea_wait_dma<2>();
    }
    ea_f8l_barrier();
    mma(c1, c0, fb0, false);
    if (more)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) fb0[j][ks] = fbn[j][ks];
    ea_f8l_barrier();
  };
  unsigned* const red = reinterpret_cast<unsigned*>(smem + WL_RED);
  WxUnit unit0, unit1;                     // of the tile's two block columns
  float* const dw = p.dw + (long long)blockIdx.y * p.part;
  const ea_rows out = ea_make_rows(dw + (long long)n0 * p.K, (long long)(p.N - n0) * p.K * 4);
  bool stored = false;
  auto put = [&](int u) {
    const int fl = wg_fresh_lane();
    wg_put(out, acc, [&](int i) { return wm * 128 + (i >> 2) * 64 + ((i & 3) ^ wn) * 16; }, fl & 15, k0 + wn * 64 + 4 * (fl >> 4), p.K, u, stored);
    stored = true;
  };
  for (;;) {
    const bool end = t0 >= steps;
    const int n = steps - t0 < WL_CH ? steps - t0 : WL_CH;
    const long long mc = m_begin + t0 * 64ll;
    if (t0 || again) ea_raw_barrier();     // the chunk (pass) before this one has been read
    const int fl = wg_fresh_lane(), ft = wave * 64 + fl;
    int sb[WL_CH * 128 / 512];
    if (!end) {
      int kb = 2 * tk + (wave & 1);
      if (kb >= (p.Kp >> 7)) kb = (p.Kp >> 7) - 1;
      const int mt = (wave >> 1) * 64 + fl, left = (int)(m_end - mc);
      const uint8_t* const sx = p.sx + kb * p.Rp + mc;
#pragma unroll
      for (int u = 0; u < WL_CH * 128 / 512; ++u) sb[u] = sx[mt + u * 256 < left ? mt + u * 256 : left - 1];      // (behind the end: zeros, any factor)
      rd = ea_make_rows(p.dy + mc * p.N + n0, ((m_end - mc) * p.N - n0) * 2);
      rx = ea_make_rows(p.x + mc * p.Kp + k0, (m_end - mc) * p.Kp - k0);
      begin(0);
      stage_x(0);
      stage_x(1);
      stage_d(0);
      stage_d(1);
      if (!again) {
        unsigned w = 0;
#pragma unroll
        for (int u = 0; u < WL_CH * 128 / 512; ++u) w = wx_max(w, wx_word(sb[u]));
        wx_range_put(red, w, fl, wave);      // (even waves: the first block column, odd ones the second)
        ea_raw_barrier();
        wx_range_get<0, 2, 8>(red, unit0);
        wx_range_get<1, 2, 8>(red, unit1);
      }
    }
    int from0, to0, from1, to1, old0, old1;
    const bool away0 = unit0.next(from0, to0, old0), away1 = unit1.next(from1, to1, old1);
    const bool away = wn >> 1 ? away1 : away0;
    const int old = wn >> 1 ? old1 : old0;
    if (end || away) put(old);
    if (end) break;
    wx_rescale(acc, away, old - (wn >> 1 ? unit1.u : unit0.u));
    const int fu = wave & 1 ? unit1.u : unit0.u, from = wave & 1 ? from1 : from0, to = wave & 1 ? to1 : to0;
#pragma unroll
    for (int u = 0; u < WL_CH * 128 / 512; ++u) *reinterpret_cast<f16*>(scl + (u * 512 + ft) * 2) = wl_factor(sb[u], fu, from, to);
    ea_wait_dma<2>();
    ea_raw_barrier();
    read_x(0, c0, fb0);
    if (wm == 1) ea_f8l_barrier();         // wave row 1 runs one barrier behind wave row 0
    for (int t = 0; t + 1 < n; ++t) body(t, std::true_type{});
    body(n - 1, std::false_type{});
    if (wm == 0) ea_f8l_barrier();         // both wave rows execute the same number of barriers
    again = unit0.lo <= unit0.hi || unit1.lo <= unit1.hi;
    if (!again) t0 += WL_CH;
  }
  float* db = p.splits > 1 ? dw + (long long)p.N * p.K : p.db;
  if (tk < 2 && lq == 0) {
    const int n = n0 + wm * 128 + tk * 64 + wn * 16 + l15;
    if (n < p.N) db[n] = accb[0];
  }
}

// sum of the slices, in their order
__global__ __launch_bounds__(64) void ea_fp8_wgrad_join_kernel(const float* part, float* dw, float* db, long long nk, long long total, int splits) {
  const long long i = ((long long)blockIdx.x * 64 + threadIdx.x) * 4;
  if (i >= total) return;
  const long long left = total - i;
  f32x4 s = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
  for (int t = 0; t < splits; ++t) s += *reinterpret_cast<const f32x4*>(part + t * ((total + 3) & ~3ll) + i);      // (slices are padded to whole vectors)
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < left) (i + j < nk ? dw[i + j] : db[i + j - nk]) = s[j];
}

// Kernel (256, 128: the DMA kernels; 0: the one for any N and alignment) and number of slices of the rows: the least time by a model of
// what was measured.  A 64-row step takes a 256 x 256 workgroup 1.65 us, a 128 x 128 one 0.87 us alone on its CU and 1.25 us beside
// another, the any-N kernel's 2.7 and 3.5; a workgroup's start and end 10 / 5 us; joining s slices 4 us and 2 s + 1 passes over the output at 8 TB/s.
//   16384 x 1280 x 5120 (M x N x K): 256 with 5 slices 216 us (2: 225, 1: 400; 128: 263 at best), 32768 x 2560 x 320: 256 with 12 slices 89
//   (128 with 8: 103), 8192 x 640 x 640: 128 with 10 slices 25 (1: 111; 256 with 24: 32), 616 x 1280 x 1024: 128 with 1 slice 14 (2: 19; 256: 27)
//   any N: 616 x 1281 x 1024 5 slices 25.5 (1: 30.3, 2: 25.6), 16384 x 1281 x 1280 9 slices 198 (4: 246, 16: 188), 8192 x 641 x 640 16 slices 46 (8: 63)
// Workspace and launch go by the same answer, which depends on the sizes alone.
struct WgradPlan { int kernel, splits, rows; };
WgradPlan wgrad_plan(int M, int N, int K) {
  WgradPlan w{-1, 1, 64};
  const int v = ea_forced_variant();       // tests: 101, 102, 103 pin a kernel
  const bool large = K > 256;              // (two k tiles: each sums one half of its dy columns for db)
  const bool dma = (N & 7) == 0 && N <= (1 << 18) && K <= (1 << 18) && v != 103;
  const double nk = (double)N * K;
  const int steps = (M + 63) / 64;
  int f = ea_forced_splits();              // tests: this many slices, where that leaves none empty
  if (f < 1 || f > steps || f > 64) f = 0;
  if (f) {
    const int per = (steps + f - 1) / f;
    if ((steps + per - 1) / per != f) f = 0;
  }
  double best = 0;
  for (int kernel = 256; kernel >= 0; kernel -= 128) {
    if (kernel ? !dma || (kernel == 256 ? !large || v == 102 : large && v == 101) : dma) continue;
    const int tile = kernel == 256 ? 256 : 128;
    const double beside = kernel ? 1.25 : 3.5, alone = kernel ? 0.87 : 2.7;      // us per step of a 128 x 128 workgroup
    const long long tiles = (long long)((N + tile - 1) / tile) * ((K + tile - 1) / tile);
    for (int s = 1; s <= steps && s <= 64; ++s) {
      const int per = (steps + s - 1) / s;
      if ((steps + per - 1) / per != s) continue;                    // (this many slices leave one empty)
      if (f && s != f) continue;
      const long long wgs = tiles * s;
      const double t = (kernel == 256 ? (wgs + 255) / 256 * (per * 1.65 + 10)
                                      : wgs / 512 * (per * beside + 5) + (wgs % 512 > 256 ? per * beside + 5 : wgs % 512 ? per * alone + 5 : 0)) +
                       (s > 1 ? 4 + (2 * s + 1) * nk * 4 / 8e6 : 0);
      if (w.kernel < 0 || t < best) {
        best = t;
        w = WgradPlan{kernel, s, per * 64};
      }
    }
  }
  return w;
}

long long fp8_tiles(const EaFp8GemmParams& p, int bm, int bn) { return (long long)((p.M + bm - 1) / bm) * ((p.N + bn - 1) / bn); }

// (apart: the output shares no memory with the operands; it is looked at last, behind every size)
template <int BM, int BN, int WM, int WN, int S, bool EXACT = false>
int fp8_ring_launch(const EaFp8GemmParams& p, bool apart, void* stream) {
  auto k = ea_fp8_ring_kernel<BM, BN, WM, WN, S, EXACT>;
  const int smem = (BM + BN) * 128 * S + EA_F8_CH * (BM + 4);
  const long long tiles = fp8_tiles(p, BM, BN);
  if (!ea_launch_holds(tiles, 64 * WM * WN)) return EA_ERR_BAD_SHAPE;
  if (!apart) return EA_ERR_BAD_ARG;
  ea_allow_big_lds(k, smem);
  EA_LAUNCH(k, dim3((unsigned)tiles), dim3(64 * WM * WN), smem, stream, p);
  return ea_launch_status();
}
int fp8_large_launch(const EaFp8GemmParams& p, bool apart, void* stream) {
  const long long tiles = fp8_tiles(p, 256, 256);
  if (!ea_launch_holds(tiles, 512)) return EA_ERR_BAD_SHAPE;
  if (!apart) return EA_ERR_BAD_ARG;
  auto k = ea_fp8_large_kernel;
  ea_allow_big_lds(k, EA_F8L_LDS);
  EA_LAUNCH(k, dim3((unsigned)tiles), dim3(512), EA_F8L_LDS, stream, p);
  return ea_launch_status();
}

// Which kernel (times in us on the MI355X, M x N x K):
//   256 x 256 tiles, one workgroup per CU: from 8 K tiles on, where the last round of 256 workgroups is at least as full as three
//       quarters of all rounds.  16384 x 5120 x 1280 113 (128 x 128: 125), 8192^3 383 (492); 16384 x 1280 x 5120 fills 1.25 rounds:
//       111.5 (110.5), and 5 K tiles do not carry the larger tile's start and end: 8192 x 5120 x 640 45.4 (43.4)
//   128 x 128, two workgroups per CU (one multiplies while the other starts or stores): from 256 tiles on.  32768 x 320 x 320 12.8
//       (64 x 128: 14.1, 64 x 64: 21.1), 16384 x 5120 x 1280 125 (150, 234)
//   64 x 128: from 160 tiles on.  616 x 2560 x 1024 6.7 (64 x 64: 7.5, 128 x 128: 8.5), 2048 x 1280 x 1280 9.9 (13.2, 10.0)
//   64 x 64 with a ring of four: few tiles, where each K tile's latency counts.  512 x 1280 x 5120 15.4 (64 x 128: 23.1),
//       77 x 1024 x 1024 6.1 (6.0)
int fp8_launch(EaFp8GemmParams& p, bool apart, void* stream) {
  p.raster_gm = 8;                         // (4 and 16: within 2 %)
  const int v = ea_forced_variant();
  const long long large = fp8_tiles(p, 256, 256), rounds = (large + 255) / 256;
  if (v == 101 || (v < 101 && p.nb >= 8 && large * 4 >= rounds * 256 * 3)) return fp8_large_launch(p, apart, stream);
  if (v == 102 || (v < 101 && fp8_tiles(p, 128, 128) >= 256)) return fp8_ring_launch<128, 128, 2, 4, 2>(p, apart, stream);
  if (v == 103 || (v < 101 && fp8_tiles(p, 64, 128) >= 160)) return fp8_ring_launch<64, 128, 2, 4, 2>(p, apart, stream);
  return fp8_ring_launch<64, 64, 2, 2, 4>(p, apart, stream);
}
// The same with exact products (the 8-bit kernels' time behind it): 128 x 128 from 512 tiles on: 16384 x 5120 x 1280 252 us (64 x 128: 292, 64 x 64:
// 369; 111), 32768 x 320 x 320 18.2 (19.9, 23.9; 12.1), 8192^3 1029 = 1070 TFLOP/s (390); but 8192 x 640 x 640, 320 tiles, 17.0 (15.4, 18.0; 10.2).
// 64 x 128 from 160 tiles on: 616 x 2560 x 1024 9.7 (64 x 64: 10.6; 6.6), 2048 x 1280 x 1280 16.5 (17.8; 9.6).  64 x 64 below: 512 x 1280 x
// 5120 25.5 (64 x 128: 31.5; 15.0).
int fp8_exact_launch(EaFp8GemmParams& p, bool apart, void* stream) {
  p.raster_gm = 8;
  const int v = ea_forced_variant();
  if (v == 102 || (v < 101 && fp8_tiles(p, 128, 128) >= 512)) return fp8_ring_launch<128, 128, 2, 2, 2, true>(p, apart, stream);
  if (v == 103 || (v < 101 && fp8_tiles(p, 64, 128) >= 160)) return fp8_ring_launch<64, 128, 2, 4, 2, true>(p, apart, stream);
  return fp8_ring_launch<64, 64, 2, 2, 4, true>(p, apart, stream);
}

// rows of `width` bytes, `pitch` apart, against other memory: rows of the same pitch, or one piece (pitch 0)
struct RowSpan { const void* p; long long rows, pitch, width; };
bool rows_apart(const RowSpan& a, const RowSpan& b) {
  const ea_span x = {a.p, (a.rows - 1) * a.pitch + a.width}, y = {b.p, (b.rows - 1) * b.pitch + b.width};
  if (ea_apart(x, y)) return true;
  if (b.pitch && b.pitch != a.pitch) return false;
  const RowSpan& lo = (uintptr_t)a.p <= (uintptr_t)b.p ? a : b;
  const RowSpan& hi = &lo == &a ? b : a;
  if (!lo.pitch) return false;
  const long long d = (long long)((uintptr_t)hi.p - (uintptr_t)lo.p) % lo.pitch;         // beside lo's columns?
  return d >= lo.width && d + hi.width <= lo.pitch;
}

int gemm_fp8_entry(const void* a, const unsigned char* a_scale, const void* w, const unsigned char* w_scale, int M, int N, int K, const ea_epilogue* e,
                   bool exact, void* stream) {
  if (!a || !a_scale || !w || !w_scale || !e || !e->out) return EA_ERR_BAD_ARG;
  if (M <= 0 || N <= 0 || K <= 0 || M > EA_FP8_ROWS || N > (1 << 22) || K > (1 << 20)) return EA_ERR_BAD_SHAPE;
  if (((uintptr_t)a & 15) || ((uintptr_t)w & 15) || ((uintptr_t)a_scale & 3)) return EA_ERR_BAD_ARG;
  if (e->act != EA_ACT_NONE && e->act != EA_ACT_SILU && e->act != EA_ACT_GELU) return EA_ERR_UNSUPPORTED;
  if (e->bias_per_row || e->rowvec || e->row_scale || e->ln_stats || e->row_stats_out || e->gn_stats_out || e->gn_next_out || e->acc_scale_k)
    return EA_ERR_UNSUPPORTED;
  if (e->ldc < N || ((e->residual || e->residual32) && e->ldr < N) || (e->residual && e->residual32)) return EA_ERR_BAD_ARG;
  EaFp8GemmParams p;
  memset(&p, 0, sizeof(p));
  p.a = (const uint8_t*)a; p.sa = a_scale; p.w = (const uint8_t*)w; p.sw = w_scale;
  p.M = M; p.N = N; p.nb = ea_fp8_blocks(K); p.Kp = p.nb * EA_FP8_BLOCK; p.nwb = (N + 127) / 128; p.Rp = ea_fp8_scale_pitch(M);
  p.bias = e->bias; p.residual = (const f16*)e->residual; p.residual32 = e->residual32; p.out = e->out;
  p.act = e->act; p.out_f32 = e->out_f32; p.ldc = e->ldc; p.ldr = e->ldr; p.scale = e->scale;
  // 16-byte accesses; a tile's 256 rows within 2 GiB
  p.vec = (N & 7) == 0 && (e->ldc & 7) == 0 && e->ldc < (1 << 21) && ((uintptr_t)e->out & 15) == 0;
  if (e->residual || e->residual32)
    p.vec = p.vec && (e->ldr & 7) == 0 && e->ldr < (1 << 21) && ((((uintptr_t)e->residual) | ((uintptr_t)e->residual32)) & 15) == 0;
  const int es = e->out_f32 ? 4 : 2, rs = e->residual32 ? 4 : 2;
  const RowSpan out = {e->out, M, (long long)e->ldc * es, (long long)N * es};
  const void* const res = e->residual32 ? (const void*)e->residual32 : e->residual;
  bool apart = true;
  for (const ea_span& in : {ea_codes(a, M, K), ea_row_scales(a_scale, M, K), ea_codes(w, N, K), ea_weight_scales(w_scale, N, K), ea_span{e->bias, 4ll * N}})
    apart = apart && rows_apart(out, {in.p, 1, 0, in.n});
  if (res && !(res == e->out && rs == es && e->ldr == e->ldc)) apart = apart && rows_apart(out, {res, M, (long long)e->ldr * rs, (long long)N * rs});
  return exact ? fp8_exact_launch(p, apart, stream) : fp8_launch(p, apart, stream);
}

}  // namespace

extern "C" int ea_gemm_fp8(const void* a, const unsigned char* a_scale, const void* w, const unsigned char* w_scale, int M, int N, int K,
                           const ea_epilogue* e, void* stream) {
  return gemm_fp8_entry(a, a_scale, w, w_scale, M, N, K, e, false, stream);
}
extern "C" int ea_gemm_fp8_exact(const void* a, const unsigned char* a_scale, const void* w, const unsigned char* w_scale, int M, int N, int K,
                                 const ea_epilogue* e, void* stream) {
  return gemm_fp8_entry(a, a_scale, w, w_scale, M, N, K, e, true, stream);
}

extern "C" size_t ea_gemm_fp8_wgrad_workspace_bytes(int M, int N, int K) {
  if (M <= 0 || N <= 0 || K <= 0 || M > EA_FP8_ROWS) return 0;
  const int s = wgrad_plan(M, N, K).splits;
  return s == 1 ? 0 : (size_t)s * ((((size_t)N * K + N) + 3) & ~(size_t)3) * sizeof(float);
}

extern "C" int ea_gemm_fp8_wgrad(const void* dy, const void* x, const unsigned char* x_scale, float* dw, float* db, int M, int N, int K,
                                 void* workspace, size_t ws_bytes, void* stream) {
  if (!dy || !x || !x_scale || !dw || !db) return EA_ERR_BAD_ARG;
  if (M <= 0 || N <= 0 || K <= 0 || M > EA_FP8_ROWS || N > (1 << 20) || K > (1 << 20)) return EA_ERR_BAD_SHAPE;
  if (((uintptr_t)x & 15) || ((uintptr_t)dw & 15) || ((uintptr_t)workspace & 15)) return EA_ERR_BAD_ARG;
  if (ws_bytes < ea_gemm_fp8_wgrad_workspace_bytes(M, N, K) || (!workspace && ws_bytes)) return EA_ERR_WORKSPACE;
  WgradParams p;
  memset(&p, 0, sizeof(p));
  const WgradPlan w = wgrad_plan(M, N, K);
  p.splits = w.splits;
  p.rows_per_split = w.rows;
  if (p.splits > 1 && !workspace) return EA_ERR_WORKSPACE;
  const int kernel = ((uintptr_t)dy & 15) ? 0 : w.kernel, tile = kernel == 256 ? 256 : 128;
  p.dy = (const f16*)dy; p.x = (const uint8_t*)x; p.sx = x_scale;
  p.M = M; p.N = N; p.K = K; p.Kp = ea_fp8_blocks(K) * EA_FP8_BLOCK; p.Rp = ea_fp8_scale_pitch(M);
  p.tiles_n = (N + tile - 1) / tile; p.tiles_k = (K + tile - 1) / tile;
  p.part = p.splits > 1 ? (((long long)N * K + N + 3) & ~3ll) : 0;
  p.dw = p.splits > 1 ? (float*)workspace : dw;
  p.db = db;
  p.vec = (N & 7) == 0 && ((uintptr_t)dy & 15) == 0;
  const long long tiles = (long long)p.tiles_n * p.tiles_k;
  const long long total = (long long)N * K + N;
  if (!ea_launch_holds(tiles, 512) || (p.splits > 1 && !ea_launch_holds((total + 255) / 256, 64))) return EA_ERR_BAD_SHAPE;
  if (!ea_outputs_apart({{dw, 4ll * N * K}, {db, 4ll * N}, {p.splits > 1 ? workspace : nullptr, p.splits * p.part * 4}},
                        {{dy, 2ll * M * N}, ea_codes(x, M, K), ea_row_scales(x_scale, M, K)}))
    return EA_ERR_BAD_ARG;
  if (kernel == 256) {
    auto k = ea_fp8_wgrad_large_kernel;
    ea_allow_big_lds(k, WL_LDS);
    EA_LAUNCH(k, dim3((unsigned)tiles, p.splits), dim3(512), WL_LDS, stream, p);
  } else if (kernel == 128) {
    auto k = ea_fp8_wgrad_ring_kernel;
    ea_allow_big_lds(k, WR_LDS);
    EA_LAUNCH(k, dim3((unsigned)tiles, p.splits), dim3(256), WR_LDS, stream, p);
  } else {
    auto k = ea_fp8_wgrad_kernel;
    EA_LAUNCH(k, dim3((unsigned)tiles, p.splits), dim3(256), WG_LDS, stream, p);
  }
  int st = ea_launch_status();
  if (st != EA_OK || p.splits == 1) return st;
  auto j = ea_fp8_wgrad_join_kernel;
  EA_LAUNCH(j, dim3((unsigned)((total + 255) / 256)), dim3(64), 0, stream, (const float*)workspace, dw, db, (long long)N * K, total, p.splits);
  return ea_launch_status();
}
