// ea_fp8_gemm.hip -- the contractions on the 8-bit format: ea_gemm_fp8 (both operands in 8 bits; ea_fp8_gemm.h) and
// ea_gemm_fp8_wgrad, the weight and bias gradient of a Linear from its 8-bit input.
#include "ea_fp8_gemm.h"

int ea_forced_variant();          // ea_gemm.hip: the calling thread's ea_tuning.variant (tests)

namespace {

// ---------------------------------------------------------------------------------------------------- weight gradient
//   dw[n][k] = sum_m dy[m][n] x[m][k],  x[m][k] = code * 2^E[m][k / 128];     db[n] = sum_m dy[m][n]
// The sum runs over rows, and each row has its own exponents, so the matrix unit's block scales do not apply (they belong to runs of
// the contracted axis).  x is decoded to fp16 instead -- four significant bits, exact -- and multiplied by dy as it is: every product
// is exact, the sums are fp32.  x is decoded as x / 2 and the accumulators are doubled: e4m3 rounding can carry an fp16 maximum
// (65504) to 65536, and at the small end x / 2 loses less than fp16's own last step.  Values beyond +-131008 become infinite.
//
// Both operands have the contracted axis as their ROW axis.  Tiles go to LDS row-major and the fragments are read transposed
// (ds_read_b64_tr_b16): 16 lanes take a 4 x 16 block and each ends up with 4 consecutive rows of one column.  A wave reads 16 rows of
// 32 bytes at once; 32-byte pieces are XORed with the row so that these cover all 64 banks twice, the minimum.
struct WgradParams {
  const f16* dy; const uint8_t* x; const uint8_t* sx;
  float* dw; float* db;              // or one [N][K] + [N] partial per slice
  int M, N, K, Kp, tiles_n, tiles_k, splits, rows_per_split; long long Rp, part;
  int vec;                           // dy rows are 16-byte aligned (N a multiple of 8)
};

constexpr int WG_T = 128, WG_R = 64;                     // tile columns of n and of k, rows per step
constexpr int WG_BUF = WG_R * WG_T * 2;                  // one operand's tile: 16 KiB
// byte of (row, column) in a tile
__device__ __forceinline__ int wg_at(int r, int c) { return r * 256 + ((((c >> 4) ^ r) & 7) << 5) + (c & 15) * 2; }

__device__ __forceinline__ f16x8 wg_frag(const char* buf, int r0, int c0, int lane) {
  const int q = lane >> 4, i = lane & 15;
  // rows r0 + 4 q .. + 3 and r0 + 16 + 4 q .. + 3: the order of rows inside a step is the same for both operands
  const char* a = buf + wg_at(r0 + 4 * q + (i >> 2), c0 + (i & 3) * 4);
  const char* b = buf + wg_at(r0 + 16 + 4 * q + (i >> 2), c0 + (i & 3) * 4);
  const f16x4 lo = ea_lds_read_tr16<0>(a), hi = ea_lds_read_tr16<0>(b);
  return f16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

__device__ __forceinline__ void wg_decode16(u32x4 w, float s, f16x8& a, f16x8& b) {
  float v[16];
#pragma unroll
  for (int i = 0; i < 4; ++i) ea_fp8_unpack4(w[i], v + 4 * i);
#pragma unroll
  for (int j = 0; j < 8; ++j) { a[j] = (f16)(v[j] * s); b[j] = (f16)(v[8 + j] * s); }
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
  auto load = [&](int m0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = i * 32 + (tid >> 3), m = m0 + r, c = (tid & 7) * 16;
      const bool ok = m < m_end;
      const long long mm = ok ? m : m_begin;
      xr[i] = *reinterpret_cast<const u32x4*>(p.x + mm * p.Kp + k0 + c);
      xs[i] = ok ? ea_fp8_scale(p.sx[(long long)tk * p.Rp + mm]) * 0.5f : 0.0f;
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
  if (m_begin < m_end) load(m_begin);
  for (int m0 = m_begin; m0 < m_end; m0 += WG_R) {
    __syncthreads();
    store();
    __syncthreads();
    if (m0 + WG_R < m_end) load(m0 + WG_R);
#pragma unroll
    for (int h = 0; h < WG_R; h += 32) {
      f16x8 fd[4], fx[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) fd[i] = wg_frag(smem, h, wn * 64 + i * 16, lane);
#pragma unroll
      for (int j = 0; j < 4; ++j) fx[j] = wg_frag(smem + WG_BUF, h, wk * 64 + j * 16, lane);
      ea_lds_tr_wait();
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = ea_mfma_16x16x32(fd[i], fx[j], acc[i][j]);
      if (tk == 0 && wk == 0)
#pragma unroll
        for (int i = 0; i < 4; ++i) accb[i] = ea_mfma_16x16x32(fd[i], ones, accb[i]);
    }
  }
  float* dw = p.dw + (long long)blockIdx.y * p.part;
  float* db = p.splits > 1 ? dw + (long long)p.N * p.K : p.db;
  const int l15 = lane & 15, lq = lane >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int n = n0 + wn * 64 + i * 16 + 4 * lq + r;
      if (n >= p.N) continue;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = k0 + wk * 64 + j * 16 + l15;
        if (k < p.K) dw[(long long)n * p.K + k] = acc[i][j][r] * 2.0f;
      }
      if (tk == 0 && wk == 0 && l15 == 0) db[n] = accb[i][r];
    }
}

// sum of the slices, in their order
__global__ __launch_bounds__(256) void ea_fp8_wgrad_join_kernel(const float* part, float* dw, float* db, long long nk, long long total, int splits) {
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= total) return;
  const long long left = total - i;
  f32x4 s = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int t = 0; t < splits; ++t) {
    const float* q = part + t * ((total + 3) & ~3ll) + i;          // (slices are padded to whole vectors)
    s += *reinterpret_cast<const f32x4*>(q);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < left) (i + j < nk ? dw[i + j] : db[i + j - nk]) = s[j];
}

int wgrad_splits(int M, int N, int K) {
  const int tiles = ((N + WG_T - 1) / WG_T) * ((K + WG_T - 1) / WG_T), steps = (M + WG_R - 1) / WG_R;
  int s = tiles >= 512 ? 1 : 512 / tiles;
  if (s > steps / 4) s = steps / 4;
  return s < 1 ? 1 : s;
}

long long fp8_tiles(const EaFp8GemmParams& p, int bm, int bn) { return (long long)((p.M + bm - 1) / bm) * ((p.N + bn - 1) / bn); }

template <int BM, int BN, int WM, int WN, int S>
int fp8_ring_launch(const EaFp8GemmParams& p, void* stream) {
  auto k = ea_fp8_ring_kernel<BM, BN, WM, WN, S>;
  const int smem = (BM + BN) * 128 * S + EA_F8_CH * (BM + 4);
  const long long tiles = fp8_tiles(p, BM, BN);
  if (tiles > 0x7fffffffll) return EA_ERR_BAD_SHAPE;
  ea_allow_big_lds(k, smem);
  EA_LAUNCH(k, dim3((unsigned)tiles), dim3(64 * WM * WN), smem, stream, p);
  return ea_launch_status();
}
int fp8_large_launch(const EaFp8GemmParams& p, void* stream) {
  const long long tiles = fp8_tiles(p, 256, 256);
  if (tiles > 0x7fffffffll) return EA_ERR_BAD_SHAPE;
  auto k = ea_fp8_large_kernel;
  ea_allow_big_lds(k, EA_F8L_LDS);
  EA_LAUNCH(k, dim3((unsigned)tiles), dim3(512), EA_F8L_LDS, stream, p);
  return ea_launch_status();
}

// Which kernel (times in us on the MI355X, M x N x K):
//   256 x 256 tiles, one workgroup per CU: from 8 K tiles on, where the last round of 256 workgroups is at least as full as three
//       quarters of all rounds.  16384 x 5120 x 1280 115 (128 x 128: 126), 8192^3 391 (504); 16384 x 1280 x 5120 fills 1.25 rounds:
//       123 (115), and 5 K tiles do not carry the larger tile's start and end: 8192 x 5120 x 640 62 (57)
//   128 x 128, two workgroups per CU (one multiplies while the other starts or stores): from 256 tiles on.  32768 x 320 x 320 17.0
//       (64 x 128: 16.1, 64 x 64: 22.7), 16384 x 5120 x 1280 126 (154, 231)
//   64 x 128: from 160 tiles on.  616 x 2560 x 1024 6.6 (64 x 64: 7.3, 128 x 128: 8.5), 2048 x 1280 x 1280 9.9 (12.9, 9.9)
//   64 x 64 with a ring of four: few tiles, where each K tile's latency counts.  512 x 1280 x 5120 15.8 (64 x 128: 24.1),
//       77 x 1024 x 1024 5.7 (5.9)
int fp8_launch(EaFp8GemmParams& p, void* stream) {
  p.raster_gm = 8;                         // (4 and 16: within 2 %)
  const int v = ea_forced_variant();
  const long long large = fp8_tiles(p, 256, 256), rounds = (large + 255) / 256;
  if (v == 101 || (v < 101 && p.nb >= 8 && large * 4 >= rounds * 256 * 3)) return fp8_large_launch(p, stream);
  if (v == 102 || (v < 101 && fp8_tiles(p, 128, 128) >= 256)) return fp8_ring_launch<128, 128, 2, 4, 2>(p, stream);
  if (v == 103 || (v < 101 && fp8_tiles(p, 64, 128) >= 160)) return fp8_ring_launch<64, 128, 2, 4, 2>(p, stream);
  return fp8_ring_launch<64, 64, 2, 2, 4>(p, stream);
}

}  // namespace

extern "C" int ea_gemm_fp8(const void* a, const unsigned char* a_scale, const void* w, const unsigned char* w_scale, int M, int N, int K,
                           const ea_epilogue* e, void* stream) {
  if (!a || !a_scale || !w || !w_scale || !e || !e->out) return EA_ERR_BAD_ARG;
  if (M <= 0 || N <= 0 || K <= 0 || K > (1 << 20)) return EA_ERR_BAD_SHAPE;
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
  return fp8_launch(p, stream);
}

extern "C" size_t ea_gemm_fp8_wgrad_workspace_bytes(int M, int N, int K) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const int s = wgrad_splits(M, N, K);
  return s == 1 ? 0 : (size_t)s * ((((size_t)N * K + N) + 3) & ~(size_t)3) * sizeof(float);
}

extern "C" int ea_gemm_fp8_wgrad(const void* dy, const void* x, const unsigned char* x_scale, float* dw, float* db, int M, int N, int K,
                                 void* workspace, size_t ws_bytes, void* stream) {
  if (!dy || !x || !x_scale || !dw || !db) return EA_ERR_BAD_ARG;
  if (M <= 0 || N <= 0 || K <= 0 || N > (1 << 20) || K > (1 << 20)) return EA_ERR_BAD_SHAPE;
  if (((uintptr_t)x & 15) || ((uintptr_t)dw & 15) || ((uintptr_t)workspace & 15)) return EA_ERR_BAD_ARG;
  if (ws_bytes < ea_gemm_fp8_wgrad_workspace_bytes(M, N, K) || (!workspace && ws_bytes)) return EA_ERR_WORKSPACE;
  WgradParams p;
  memset(&p, 0, sizeof(p));
  p.splits = wgrad_splits(M, N, K);
  if (p.splits > 1 && !workspace) return EA_ERR_WORKSPACE;
  const int steps = (M + WG_R - 1) / WG_R;
  p.rows_per_split = (steps + p.splits - 1) / p.splits * WG_R;
  p.dy = (const f16*)dy; p.x = (const uint8_t*)x; p.sx = x_scale;
  p.M = M; p.N = N; p.K = K; p.Kp = ea_fp8_blocks(K) * EA_FP8_BLOCK; p.Rp = ea_fp8_scale_pitch(M);
  p.tiles_n = (N + WG_T - 1) / WG_T; p.tiles_k = (K + WG_T - 1) / WG_T;
  p.part = p.splits > 1 ? (((long long)N * K + N + 3) & ~3ll) : 0;
  p.dw = p.splits > 1 ? (float*)workspace : dw;
  p.db = db;
  p.vec = (N & 7) == 0 && ((uintptr_t)dy & 15) == 0;
  const long long tiles = (long long)p.tiles_n * p.tiles_k;
  if (tiles > 0x7fffffffll) return EA_ERR_BAD_SHAPE;
  auto k = ea_fp8_wgrad_kernel;
  EA_LAUNCH(k, dim3((unsigned)tiles, p.splits), dim3(256), 2 * WG_BUF, stream, p);
  int st = ea_launch_status();
  if (st != EA_OK || p.splits == 1) return st;
  auto j = ea_fp8_wgrad_join_kernel;
  const long long total = (long long)N * K + N;
  EA_LAUNCH(j, dim3((unsigned)((total + 1023) / 1024)), dim3(256), 0, stream, (const float*)workspace, dw, db, (long long)N * K, total, p.splits);
  return ea_launch_status();
}
