// ea_fp8.hip -- activations and weights in 8 bits (format: ea_fp8.h): quantisation of rows and of 128 x 128 weight blocks, its
// inverse, and activation functions that keep their INPUT in 8 bits for the backward pass.
//
//   save   h = f(z),  saved = q8(z)         f: SiLU, exact GELU, GEGLU (h = value * gelu(gate), z = [value | gate]); h fp16 or q8(h)
//   use    dz = dh f'(z),  z decoded from `saved`
//             SiLU'(z) = s (1 + z (1 - s)), s = sigmoid(z);   GELU'(z) = Phi(z) + z phi(z)
// Each is one pass bound by HBM.  Sixteen lanes own one block of 128 (a 16-byte load of 8 values each), so the block's maximum is
// four DPP steps and the codes go out as 128 contiguous bytes; a workgroup covers 16 rows x 4 blocks, four blocks' loads in flight per
// lane, and the 16 rows' scale bytes of a block are adjacent.
// Measured: quantising 16384 x 5120 fp16 38 us = 6.6 TB/s; save, GELU, 16384 x 5120: 81 us with fp16 output (5.2 TB/s), 70 us with 8-bit
// output (4.8 TB/s: about 20 vector instructions per value; 92 us before the maxima were taken on packed halves and the conversions
// took the power of two along); use, GEGLU, 32768 x 1280: 65 us = 5.2 TB/s.
#include "ea_fp8.h"
#include "../../include/editanything_hip.h"

namespace {

constexpr int Q_KB = 4;        // blocks of 128 columns per thread

template <bool F32, bool VEC>
__device__ __forceinline__ void q_load8(const void* x, long long row, int cols, int c, float* v) {
  if constexpr (VEC) {
    const int cc = c < cols ? c : 0;                          // clamped, unconditional loads: four blocks in flight
    if constexpr (F32) {
      const float* p = (const float*)x + row * cols + cc;
      const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
    } else {
      const f16x8 h = ea_ld8((const f16*)x + row * cols + cc);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = (float)h[j];
    }
    if (c >= cols)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.0f;
  } else if (c + 8 <= cols) {                                 // a row that starts anywhere
    if constexpr (F32) {
      const float* p = (const float*)x + row * cols + c;
      const f32x4 a = ea_ld4u(p), b = ea_ld4u(p + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
    } else {
      const f16x8 h = ea_ld8u((const f16*)x + row * cols + c);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = (float)h[j];
    }
  } else {                                                    // its end
#pragma unroll
    for (int j = 0; j < 8; ++j)
      v[j] = c + j < cols ? (F32 ? ((const float*)x)[row * cols + c + j] : (float)((const f16*)x)[row * cols + c + j]) : 0.0f;
  }
}

// 8 fp16 values of a row, as they are
template <bool VEC>
__device__ __forceinline__ f16x8 q_load8h(const f16* x, long long row, int cols, int c) {
  if constexpr (VEC) {
    f16x8 h = ea_ld8(x + row * cols + (c < cols ? c : 0));
    if (c >= cols) h = ea_zero8();
    return h;
  } else {
    f16x8 h;
    if (c + 8 <= cols) return ea_ld8u(x + row * cols + c);
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] = c + j < cols ? x[row * cols + c + j] : (f16)0.0f;
    return h;
  }
}

template <typename V>
__device__ __forceinline__ void q_store(const V& v, uint8_t* q, uint8_t* scale, long long row, int Kp, long long Rp, int kb, int l,
                                        bool live) {        // every lane of the wave calls it; rows that are not there store nothing
  int e;
  const u32x2 w = ea_fp8_block<16>(v, e);
  if (live) *reinterpret_cast<u32x2*>(q + row * Kp + kb * 128 + l * 8) = w;
  if (live && l == 0) scale[(long long)kb * Rp + row] = (uint8_t)e;
}

// ----------------------------------------------------------------------------------------------------- rows -> 8 bits
template <bool F32, bool VEC>
__global__ __launch_bounds__(256) void ea_quant_rows_kernel(const void* x, uint8_t* q, uint8_t* scale, long long rows, int cols, int nb,
                                                            long long Rp, int gx) {
  const int l = threadIdx.x & 15;
  const long long rt = blockIdx.x / gx;
  const long long row = rt * 16 + (threadIdx.x >> 4);
  const int kb0 = (blockIdx.x - (int)(rt * gx)) * Q_KB;
  const bool live = row < rows;
  const long long r = live ? row : rows - 1;
  if constexpr (F32) {
    float v[Q_KB][8];
#pragma unroll
    for (int u = 0; u < Q_KB; ++u) q_load8<true, VEC>(x, r, cols, (kb0 + u) * 128 + l * 8, v[u]);
#pragma unroll
    for (int u = 0; u < Q_KB; ++u)
      if (kb0 + u < nb) q_store((const float*)v[u], q, scale, row, nb * 128, Rp, kb0 + u, l, live);
  } else {
    f16x8 v[Q_KB];
#pragma unroll
    for (int u = 0; u < Q_KB; ++u) v[u] = q_load8h<VEC>((const f16*)x, r, cols, (kb0 + u) * 128 + l * 8);
#pragma unroll
    for (int u = 0; u < Q_KB; ++u)
      if (kb0 + u < nb) q_store(v[u], q, scale, row, nb * 128, Rp, kb0 + u, l, live);
  }
}

// ------------------------------------------------------------------------------------------- a 128 x 128 weight block
template <bool F32, bool VEC>
__global__ __launch_bounds__(256) void ea_quant_weight_kernel(const void* w, uint8_t* q, uint8_t* scale, int N, int K, int nb) {
  EA_SMEM(smem);
  float* red = reinterpret_cast<float*>(smem);
  const int l = threadIdx.x & 15, gy = threadIdx.x >> 4, kb = blockIdx.x;
  const int n0 = blockIdx.y * 128;
  float v[8][8];
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int n = n0 + gy + 16 * i;
    q_load8<F32, VEC>(w, n < N ? n : N - 1, K, kb * 128 + l * 8, v[i]);      // (a repeated last row leaves the maximum as it is)
#pragma unroll
    for (int j = 0; j < 8; ++j) m = fmaxf(m, ea_finite_abs(v[i][j]));
  }
  m = ea_group_max<64>(m);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  const int e = ea_fp8_exp_byte(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
  const float inv = ea_fp8_inv_scale(e);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int n = n0 + gy + 16 * i;
    float t[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = ea_fp8_prep(v[i][j], inv);
    if (n < N)
      *reinterpret_cast<u32x2*>(q + (long long)n * nb * 128 + kb * 128 + l * 8) =
          u32x2{ea_fp8_pack4(t[0], t[1], t[2], t[3]), ea_fp8_pack4(t[4], t[5], t[6], t[7])};
  }
  if (threadIdx.x == 0) scale[(long long)kb * gridDim.y + blockIdx.y] = (uint8_t)e;
}

// ------------------------------------------------------------------------------------------------------ 8 bits -> rows
__device__ __forceinline__ void q_decode8(const uint8_t* p, float s, float* v) {
  const u32x2 w = *reinterpret_cast<const u32x2*>(p);
  ea_fp8_unpack4(w[0], v);
  ea_fp8_unpack4(w[1], v + 4);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] *= s;
}
template <bool VEC>
__device__ __forceinline__ void h_load8(const f16* p, int c, int cols, float* v) {
  if constexpr (VEC) {
    const f16x8 h = ea_ld8(p + (c < cols ? c : 0));
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (float)h[j];
  } else if (c + 8 <= cols) {
    const f16x8 h = ea_ld8u(p + c);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (float)h[j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c + j < cols ? (float)p[c + j] : 0.0f;
  }
}
template <bool VEC>
__device__ __forceinline__ void h_store8(f16* p, int c, int cols, const float* v) {
  if constexpr (VEC) {
    f16x8 h;
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] = (f16)v[j];
    if (c < cols) ea_st8(p + c, h);
  } else if (c + 8 <= cols) {
    f16x8 h;
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] = (f16)v[j];
    ea_st8u(p + c, h);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j < cols) p[c + j] = (f16)v[j];
  }
}

template <bool F32, bool VEC>
__global__ __launch_bounds__(256) void ea_dequant_kernel(const uint8_t* q, const uint8_t* scale, void* out, long long rows, int cols, int nb,
                                                         long long pitch, int row_shift, int gx) {
  const int l = threadIdx.x & 15;
  const long long rt = blockIdx.x / gx;
  const long long row = rt * 16 + (threadIdx.x >> 4);
  const int kb0 = (blockIdx.x - (int)(rt * gx)) * Q_KB;
  if (row >= rows) return;
#pragma unroll
  for (int u = 0; u < Q_KB; ++u) {
    const int kb = kb0 + u, c = kb * 128 + l * 8;
    if (kb >= nb) break;
    float v[8];
    q_decode8(q + row * nb * 128 + c, ea_fp8_scale(scale[kb * pitch + (row >> row_shift)]), v);
    if constexpr (F32) {
      float* o = (float*)out + row * cols;
      if (VEC && c < cols) {
        *reinterpret_cast<f32x4*>(o + c) = f32x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4*>(o + c + 4) = f32x4{v[4], v[5], v[6], v[7]};
      } else if (!VEC && c + 8 <= cols) {
        ea_st4u(o + c, f32x4{v[0], v[1], v[2], v[3]});
        ea_st4u(o + c + 4, f32x4{v[4], v[5], v[6], v[7]});
      } else if (!VEC) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c + j < cols) o[c + j] = v[j];
      }
    } else h_store8<VEC>((f16*)out + row * cols, c, cols, v);
  }
}

// ------------------------------------------------------------------------------------------------ activation, forward
struct ActParams {
  const f16* z; f16* h; uint8_t* hq; uint8_t* hs;      // forward: z [M][g H], h fp16 or 8-bit
  uint8_t* zq; uint8_t* zs;                            // z as [g M][H] rows in 8 bits
  const f16* dh; f16* dz;                              // backward
  long long M; int H, nb, gx; long long RpH, RpZ;
};

template <int ACT>
__device__ __forceinline__ float act_f(float z) { return ACT == EA_ACT_SILU ? ea_silu(z) : ea_fp8_gelu(z); }

// GELU(x) as in the forward pass, Phi(x) and x phi(x).  (x Phi(x) would not do for GELU(x): Phi ends at 7.7e-9, not at 0, and x does not end)
__device__ __forceinline__ void gelu_parts(float x, float& gelu, float& phi_c, float& xp) {
  const float a = fminf(fabsf(x), EA_FP8_GELU_END), t = ea_fp8_gelu_tail(a);
  gelu = (x < 0.0f ? 0.0f : x) - a * t;
  phi_c = x > 0.0f ? 1.0f - t : t;
  const float c = fminf(fmaxf(x, -13.0f), 13.0f);              // (phi(13) = 8e-38: the exponent ends inside fp32's, and so does x)
  xp = c * 0.3989422804014327f * ea_exp2_raw(c * c * -0.7213475204444817f);
  if (x != x) phi_c = xp = x;
}
template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  if (ACT == EA_ACT_SILU) {
    const float s = 1.0f / (1.0f + ea_expf(-z)), c = fminf(fmaxf(z, -200.0f), 200.0f);      // (1 - s or s is 0 there; a NaN is in s)
    return s * (1.0f + c * (1.0f - s));
  }
  float f, P, xp;
  gelu_parts(z, f, P, xp);
  return P + xp;
}

template <int ACT, bool VEC, bool OUT8>
__global__ __launch_bounds__(256) void ea_act_save_kernel(ActParams p) {
  constexpr int G = ACT == EA_ACT_GEGLU ? 2 : 1;
  const int l = threadIdx.x & 15;
  const long long rt = blockIdx.x / p.gx;
  const long long row = rt * 16 + (threadIdx.x >> 4);
  const int kb0 = (blockIdx.x - (int)(rt * p.gx)) * Q_KB;
  const bool live = row < p.M;
  const long long r = live ? row : p.M - 1;
  f16x8 v[G][Q_KB];
#pragma unroll
  for (int u = 0; u < Q_KB; ++u)
#pragma unroll
    for (int g = 0; g < G; ++g) v[g][u] = q_load8h<VEC>(p.z, r * G + g, p.H, (kb0 + u) * 128 + l * 8);
#pragma unroll
  for (int u = 0; u < Q_KB; ++u) {
    const int kb = kb0 + u, c = kb * 128 + l * 8;
    if (kb >= p.nb) break;
#pragma unroll
    for (int g = 0; g < G; ++g) q_store(v[g][u], p.zq, p.zs, row * G + g, p.nb * 128, p.RpZ, kb, l, live);
    float h[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] = G == 2 ? (float)v[0][u][j] * act_f<EA_ACT_GELU>((float)v[G - 1][u][j]) : act_f<ACT>((float)v[0][u][j]);
    if constexpr (OUT8) q_store((const float*)h, p.hq, p.hs, row, p.nb * 128, p.RpH, kb, l, live);     // (f(0) = 0: the padding stays zero codes)
    else if (live) h_store8<VEC>(p.h + row * p.H, c, p.H, h);
  }
}

// ----------------------------------------------------------------------------------------------- activation, backward
template <int ACT, bool VEC>
__global__ __launch_bounds__(256) void ea_act_use_kernel(ActParams p) {
  constexpr int G = ACT == EA_ACT_GEGLU ? 2 : 1;
  const int l = threadIdx.x & 15;
  const long long rt = blockIdx.x / p.gx;
  const long long row = rt * 16 + (threadIdx.x >> 4);
  const int kb0 = (blockIdx.x - (int)(rt * p.gx)) * Q_KB;
  if (row >= p.M) return;
#pragma unroll
  for (int u = 0; u < Q_KB; ++u) {
    const int kb = kb0 + u, c = kb * 128 + l * 8;
    if (kb >= p.nb) break;
    float z[G][8], d[8], o[G][8];
#pragma unroll
    for (int g = 0; g < G; ++g)
      q_decode8(p.zq + (row * G + g) * p.nb * 128 + c, ea_fp8_scale(p.zs[kb * p.RpZ + row * G + g]), z[g]);
    h_load8<VEC>(p.dh + row * p.H, c, p.H, d);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (G == 2) {
        float f, P, xp;
        gelu_parts(z[1][j], f, P, xp);
        o[0][j] = d[j] * f;
        o[1][j] = d[j] * z[0][j] * (P + xp);
      } else o[0][j] = d[j] * act_slope<ACT>(z[0][j]);
    }
#pragma unroll
    for (int g = 0; g < G; ++g) h_store8<VEC>(p.dz + (row * G + g) * p.H, c, p.H, o[g]);
  }
}

bool al16(const void* a, const void* b = nullptr, const void* c = nullptr) {
  return ((((uintptr_t)a) | ((uintptr_t)b) | ((uintptr_t)c)) & 15) == 0;
}
// workgroups of 16 rows x Q_KB blocks, column tiles fastest; 0: more than a launch holds
unsigned q_grid(long long rows, int nb, int& gx) {
  gx = (nb + Q_KB - 1) / Q_KB;
  if (rows > (1ll << 40)) return 0u;
  const long long g = (rows + 15) / 16 * gx;
  return ea_launch_holds(g, 256) ? (unsigned)g : 0u;
}

}  // namespace

extern "C" int ea_quantize_fp8(const void* x, int in_f32, void* q, unsigned char* scale, long long rows, int cols, void* stream) {
  if (!x || !q || !scale) return EA_ERR_BAD_ARG;
  if (rows <= 0 || cols <= 0 || cols > (1 << 24)) return EA_ERR_BAD_SHAPE;
  if (!al16(q)) return EA_ERR_BAD_ARG;
  int gx;
  const int nb = ea_fp8_blocks(cols);
  const unsigned grid = q_grid(rows, nb, gx);
  if (!grid) return EA_ERR_BAD_SHAPE;
  if (!ea_outputs_apart({ea_codes(q, rows, cols), ea_row_scales(scale, rows, cols)}, {{x, rows * cols * (in_f32 ? 4 : 2)}})) return EA_ERR_BAD_ARG;
  const bool vec = (cols & 7) == 0 && al16(x);
  auto k = in_f32 ? (vec ? ea_quant_rows_kernel<true, true> : ea_quant_rows_kernel<true, false>)
                  : (vec ? ea_quant_rows_kernel<false, true> : ea_quant_rows_kernel<false, false>);
  EA_LAUNCH(k, dim3(grid), dim3(256), 0, stream, x, (uint8_t*)q, scale, rows, cols, nb, ea_fp8_scale_pitch(rows), gx);
  return ea_launch_status();
}

extern "C" int ea_quantize_fp8_weight(const void* w, int in_f32, void* q, unsigned char* scale, int N, int K, void* stream) {
  if (!w || !q || !scale) return EA_ERR_BAD_ARG;
  if (N <= 0 || K <= 0 || N > (1 << 22) || K > (1 << 24)) return EA_ERR_BAD_SHAPE;
  if (!al16(q)) return EA_ERR_BAD_ARG;
  if (!ea_outputs_apart({ea_codes(q, N, K), ea_weight_scales(scale, N, K)}, {{w, (long long)N * K * (in_f32 ? 4 : 2)}})) return EA_ERR_BAD_ARG;
  const bool vec = (K & 7) == 0 && al16(w);
  auto k = in_f32 ? (vec ? ea_quant_weight_kernel<true, true> : ea_quant_weight_kernel<true, false>)
                  : (vec ? ea_quant_weight_kernel<false, true> : ea_quant_weight_kernel<false, false>);
  EA_LAUNCH(k, dim3(ea_fp8_blocks(K), (N + 127) / 128), dim3(256), 64, stream, w, (uint8_t*)q, scale, N, K, ea_fp8_blocks(K));
  return ea_launch_status();
}

extern "C" int ea_dequantize_fp8(const void* q, const unsigned char* scale, int block_rows, void* out, int out_f32, long long rows, int cols,
                                 void* stream) {
  if (!q || !scale || !out) return EA_ERR_BAD_ARG;
  if (rows <= 0 || cols <= 0 || cols > (1 << 24)) return EA_ERR_BAD_SHAPE;
  if (!al16(q) || (block_rows != 1 && block_rows != 128)) return EA_ERR_BAD_ARG;
  int gx;
  const int nb = ea_fp8_blocks(cols);
  const unsigned grid = q_grid(rows, nb, gx);
  if (!grid) return EA_ERR_BAD_SHAPE;
  if (!ea_outputs_apart({{out, rows * cols * (out_f32 ? 4 : 2)}},
                        {ea_codes(q, rows, cols), block_rows == 1 ? ea_row_scales(scale, rows, cols) : ea_weight_scales(scale, rows, cols)}))
    return EA_ERR_BAD_ARG;
  const bool vec = (cols & 7) == 0 && al16(out);
  auto k = out_f32 ? (vec ? ea_dequant_kernel<true, true> : ea_dequant_kernel<true, false>)
                   : (vec ? ea_dequant_kernel<false, true> : ea_dequant_kernel<false, false>);
  EA_LAUNCH(k, dim3(grid), dim3(256), 0, stream, (const uint8_t*)q, scale, out, rows, cols, nb,
            block_rows == 1 ? ea_fp8_scale_pitch(rows) : (rows + 127) / 128, block_rows == 1 ? 0 : 7, gx);
  return ea_launch_status();
}

static int act_params(ActParams& p, int act, long long M, int H, unsigned& grid) {
  if (act != EA_ACT_SILU && act != EA_ACT_GELU && act != EA_ACT_GEGLU) return EA_ERR_BAD_ARG;
  if (M <= 0 || H <= 0 || H > (1 << 24)) return EA_ERR_BAD_SHAPE;
  memset(&p, 0, sizeof(p));
  p.M = M; p.H = H; p.nb = ea_fp8_blocks(H);
  p.RpH = ea_fp8_scale_pitch(M);
  p.RpZ = ea_fp8_scale_pitch(act == EA_ACT_GEGLU ? 2 * M : M);
  grid = q_grid(M, p.nb, p.gx);
  return grid ? EA_OK : EA_ERR_BAD_SHAPE;
}

extern "C" int ea_activation_fp8(const void* z, int act, void* h, void* hq, unsigned char* hscale, void* zq, unsigned char* zscale, long long M,
                                 int H, void* stream) {
  if (!z || !zq || !zscale || (!h == !hq) || (hq && !hscale)) return EA_ERR_BAD_ARG;
  ActParams p;
  unsigned grid;
  const int st = act_params(p, act, M, H, grid);
  if (st != EA_OK) return st;
  if (!al16(zq, hq)) return EA_ERR_BAD_ARG;
  const int g = act == EA_ACT_GEGLU ? 2 : 1;
  const ea_span in = {z, M * g * H * 2}, ho = {h, M * H * 2};
  if (!ea_outputs_apart({ho, ea_codes(hq, M, H), ea_row_scales(hq ? hscale : nullptr, M, H), ea_codes(zq, g * M, H), ea_row_scales(zscale, g * M, H)},
                        {{nullptr, 0}}) ||
      !ea_outputs_apart({ea_codes(hq, M, H), ea_row_scales(hq ? hscale : nullptr, M, H), ea_codes(zq, g * M, H), ea_row_scales(zscale, g * M, H)}, {in}) ||
      !ea_apart(ho, in, g == 1))
    return EA_ERR_BAD_ARG;
  p.z = (const f16*)z; p.h = (f16*)h; p.hq = (uint8_t*)hq; p.hs = hscale; p.zq = (uint8_t*)zq; p.zs = zscale;
  const bool vec = (H & 7) == 0 && al16(z, h), o8 = hq != nullptr;
#define EA_ACT_PICK(A) (vec ? (o8 ? ea_act_save_kernel<A, true, true> : ea_act_save_kernel<A, true, false>) \
                            : (o8 ? ea_act_save_kernel<A, false, true> : ea_act_save_kernel<A, false, false>))
  auto k = act == EA_ACT_SILU ? EA_ACT_PICK(EA_ACT_SILU) : act == EA_ACT_GELU ? EA_ACT_PICK(EA_ACT_GELU) : EA_ACT_PICK(EA_ACT_GEGLU);
#undef EA_ACT_PICK
  EA_LAUNCH(k, dim3(grid), dim3(256), 0, stream, p);
  return ea_launch_status();
}

extern "C" int ea_activation_fp8_bwd(const void* dh, const void* zq, const unsigned char* zscale, int act, void* dz, long long M, int H,
                                     void* stream) {
  if (!dh || !zq || !zscale || !dz) return EA_ERR_BAD_ARG;
  ActParams p;
  unsigned grid;
  const int st = act_params(p, act, M, H, grid);
  if (st != EA_OK) return st;
  if (!al16(zq)) return EA_ERR_BAD_ARG;
  const int g = act == EA_ACT_GEGLU ? 2 : 1;
  const ea_span out = {dz, M * g * H * 2};
  if (!ea_outputs_apart({out}, {ea_codes(zq, g * M, H), ea_row_scales(zscale, g * M, H)}) || !ea_apart(out, {dh, M * H * 2}, g == 1))
    return EA_ERR_BAD_ARG;
  p.dh = (const f16*)dh; p.dz = (f16*)dz; p.zq = (uint8_t*)const_cast<void*>(zq); p.zs = const_cast<unsigned char*>(zscale);
  const bool vec = (H & 7) == 0 && al16(dh, dz);
  auto k = act == EA_ACT_SILU ? (vec ? ea_act_use_kernel<EA_ACT_SILU, true> : ea_act_use_kernel<EA_ACT_SILU, false>)
         : act == EA_ACT_GELU ? (vec ? ea_act_use_kernel<EA_ACT_GELU, true> : ea_act_use_kernel<EA_ACT_GELU, false>)
                              : (vec ? ea_act_use_kernel<EA_ACT_GEGLU, true> : ea_act_use_kernel<EA_ACT_GEGLU, false>);
  EA_LAUNCH(k, dim3(grid), dim3(256), 0, stream, p);
  return ea_launch_status();
}
