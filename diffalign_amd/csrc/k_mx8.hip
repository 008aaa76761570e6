// 8-bit activation checkpoints of the training step (MXINT8, mx8_util.h) and their use in the backward pass:
//   k_mx8_quant / k_mx8_dequant     activation (rows, D) <-> codes (rows, D) + scale bytes (rows, ceil(D / 32))
//   k_relu_drop_bwd_mx8             backward of ReLU + dropout from the codes of its result
//   k_mx8_wgrad                     weight / bias gradient of a Linear whose input is held in 8 bits
// The training forward of the reference keeps every per-pair activation at full width for loss.backward() (training/helpers.py:139-142).
#include "mfma_util.h"
#include "mx8_util.h"
#include "dropout_util.h"

// ---------------------------------------------------------------------------------------------------------------------------------
// Quantise / restore.  Streaming: D (s + 1 + 1/32) bytes per row, a dozen integer and float operations per element.  HBM-bound: 313,600 x 256
// bf16 (243 MB each way) 47 us = 5.2 TB/s to quantise, 34 us to restore right after (the codes are still in the 256 MB cache; non-temporal
// stores of them cost both: 52 and 39 us); fp32 (404 MB) 76 us to quantise = 5.3 TB/s.
__device__ __forceinline__ void ld8(const float* p, float (&v)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void unpack8(uint4 a, float (&v)[8]) {
  v[0] = bf16_lo(a.x); v[1] = bf16_hi(a.x); v[2] = bf16_lo(a.y); v[3] = bf16_hi(a.y);
  v[4] = bf16_lo(a.z); v[5] = bf16_hi(a.z); v[6] = bf16_lo(a.w); v[7] = bf16_hi(a.w);
}
__device__ __forceinline__ void ld8(const bf16_t* p, float (&v)[8]) { unpack8(*reinterpret_cast<const uint4*>(p), v); }
__device__ __forceinline__ void st8(float* p, const float (&v)[8]) {
  *reinterpret_cast<float4*>(p) = float4{v[0], v[1], v[2], v[3]};
  *reinterpret_cast<float4*>(p + 4) = float4{v[4], v[5], v[6], v[7]};
}
__device__ __forceinline__ void st8(bf16_t* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) = uint4{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])};
}
__device__ __forceinline__ float ld1(const float* p) { return *p; }
__device__ __forceinline__ float ld1(const bf16_t* p) { return bf2f(*p); }
__device__ __forceinline__ void st1(float* p, float v) { *p = v; }
__device__ __forceinline__ void st1(bf16_t* p, float v) { *p = f2bf(v); }
__device__ __forceinline__ void codes8(uint2 w, float step, float (&v)[8]) {
  v[0] = mx8_elem<0>(w.x) * step; v[1] = mx8_elem<1>(w.x) * step; v[2] = mx8_elem<2>(w.x) * step; v[3] = mx8_elem<3>(w.x) * step;
  v[4] = mx8_elem<0>(w.y) * step; v[5] = mx8_elem<1>(w.y) * step; v[6] = mx8_elem<2>(w.y) * step; v[7] = mx8_elem<3>(w.y) * step;
}

// D % 32 == 0 and aligned: the groups are consecutive in memory.  A thread holds 8 elements, a group lies on 4 neighbouring lanes.
template <class T, bool KEEP>
__global__ void __launch_bounds__(256) k_mx8_quant(const T* __restrict__ x, uint2* __restrict__ codes, uint8_t* __restrict__ scales, long long octs) {
  for (long long t = (long long)blockIdx.x * 256 + threadIdx.x; t < octs; t += (long long)gridDim.x * 256) {
    float v[8];
    ld8(x + t * 8, v);
    unsigned m = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) m = dpp_max_u32(m, abs_bits(v[k]));
    const unsigned b = mx8_scale(quad_max(m));                          // octs % 4 == 0: the four lanes of a group run together
    const float inv = mx8_inv(b);
    codes[t] = uint2{mx8_pack4<KEEP>(v[0], v[1], v[2], v[3], inv), mx8_pack4<KEEP>(v[4], v[5], v[6], v[7], inv)};
    if ((t & 3) == 0) scales[t >> 2] = (uint8_t)b;
  }
}
// any D, any alignment: 32 lanes per group of a row, one element each
template <class T, bool KEEP>
__global__ void __launch_bounds__(256) k_mx8_quant_any(const T* __restrict__ x, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, long long groups,
                                                       int D, int G) {
  const int l32 = threadIdx.x & 31;
  for (long long g = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); g < groups; g += (long long)gridDim.x * 8) {
    const long long row = g / G;
    const int c = (int)(g - row * G) * MX8_GROUP + l32;
    const float v = c < D ? ld1(x + row * D + c) : 0.f;
    unsigned m = abs_bits(v);
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) m = dpp_max_u32(m, (unsigned)__shfl_xor((int)m, k, 32));
    const unsigned b = mx8_scale(m);
    if (c < D) codes[row * D + c] = (uint8_t)mx8_code<KEEP>(v, mx8_inv(b));
    if (l32 == 0) scales[g] = (uint8_t)b;
  }
}
template <class T>
__global__ void __launch_bounds__(256) k_mx8_dequant(const uint2* __restrict__ codes, const uint8_t* __restrict__ scales, T* __restrict__ out, long long octs) {
  for (long long t = (long long)blockIdx.x * 256 + threadIdx.x; t < octs; t += (long long)gridDim.x * 256) {
    float v[8];
    codes8(codes[t], mx8_step(scales[t >> 2]), v);
    st8(out + t * 8, v);
  }
}
template <class T>
__global__ void __launch_bounds__(256) k_mx8_dequant_any(const int8_t* __restrict__ codes, const uint8_t* __restrict__ scales, T* __restrict__ out,
                                                         long long numel, int D, int G) {
  for (long long t = (long long)blockIdx.x * 256 + threadIdx.x; t < numel; t += (long long)gridDim.x * 256) {
    const long long row = t / D;
    const int c = (int)(t - row * D);
    st1(out + t, (float)codes[t] * mx8_step(scales[row * G + c / MX8_GROUP]));
  }
}

// dx = dy * scale where the code is not 0 (the forward result was not zero: passed the ReLU and kept by the dropout), else 0.  HBM-bound, 1 + 2 s
// bytes an element: 313,600 x 128 bf16 (201 MB) 32 us, fp32 (361 MB) 67 us = 5.4 TB/s (a copy of 4 GiB: 4.75; part of dy is still cached).
template <class T>
__global__ void __launch_bounds__(256) k_relu_drop_bwd_mx8(const uint2* __restrict__ codes, const T* __restrict__ dy, T* __restrict__ dx, long long octs,
                                                           float scale) {
  for (long long t = (long long)blockIdx.x * 256 + threadIdx.x; t < octs; t += (long long)gridDim.x * 256) {
    const uint2 w = codes[t];
    float v[8];
    ld8(dy + t * 8, v);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[k] = (w.x >> (8 * k)) & 0xffu ? v[k] * scale : 0.f;
      v[4 + k] = (w.y >> (8 * k)) & 0xffu ? v[4 + k] * scale : 0.f;
    }
    st8(dx + t * 8, v);
  }
}
template <class T>
__global__ void __launch_bounds__(256) k_relu_drop_bwd_mx8_any(const int8_t* __restrict__ codes, const T* __restrict__ dy, T* __restrict__ dx, long long numel,
                                                               float scale) {
  for (long long t = (long long)blockIdx.x * 256 + threadIdx.x; t < numel; t += (long long)gridDim.x * 256)
    st1(dx + t, codes[t] != 0 ? ld1(dy + t) * scale : 0.f);
}

// ---------------------------------------------------------------------------------------------------------------------------------
// Weight / bias gradient from the 8-bit input: dW (OUT,IN) = dY^T x^, db = column sums of dY, over R rows.  A tiny result with a huge
// reduction: HBM-bound (IN (1 + 1/32) + OUT s bytes for 2 IN OUT flops per row), so the rows are split over the chip, each workgroup
// keeps the whole (OUT,IN) result in accumulators, and the slices' partial results are folded in slice order (no atomics).
// v_mfma_f32_32x32x16_bf16 sums over 16 rows at a time and wants 8 rows of one feature per lane, while memory is contiguous along the
// features: tiles of KR rows go through LDS row-major and come back through the transposing read (ds_read_b64_tr_b16: 4 rows of 16
// features per 16 lanes).  x^ = q 2^e is exact in bf16.  dY: bf16 as it is; fp32 as the sum of three bf16 parts (8 + 8 + 8 bits, each cut
// toward zero: the whole significand, down to 2^-133, the unit of the subnormal bf16, which the instruction takes as they are), one product
// each, so nothing of it is rounded away.  Products are exact, sums fp32.
// A tile's next rows are loaded into registers while the matrix instructions of the present one run (a second LDS buffer in place of the second
// barrier changes nothing).  313,600 rows: 64 -> 256 bf16 41 us (181 MB, 4.5 TB/s), 256 -> 64 fp32 50 us (163 MB, 3.3 TB/s: neither HBM nor the
// VALU, busy 52 %, is full; a tile's load, stage, products and two barriers follow one another), and 8 us for the fold of 512 partial results.
// Row pitch in LDS: OUT or IN elements + 64 bytes from 64 features on -- the four rows of a transposing read then start 16 banks apart.
__host__ __device__ constexpr int tr_pitch(int feats) { return feats * 2 + (feats >= 64 ? 64 : 0); }   // bytes

template <int IN, int OUT, class TY>
struct WgradCfg {
  static constexpr int TI = IN / 32, TO = OUT / 32, TILES = TI * TO;
  static constexpr int WT = TILES < 4 ? TILES : 4, WK = 4 / WT;         // waves over result tiles x waves over rows
  static constexpr int WO = TO >= WT ? WT : (TO >= 2 && WT == 4 ? 2 : TO), WI = WT / WO;
  static constexpr int AO = TO / WO, AI = TI / WI;                      // tiles per wave
  static constexpr int PLANES = sizeof(TY) == 4 ? 3 : 1;
  static constexpr int PY = tr_pitch(OUT), PX = tr_pitch(IN);
  // rows per LDS tile: 64 where two workgroups still fit a CU (fp32 64 -> 256 does not: 131 KB)
  static constexpr int KR = 64 * (PLANES * PY + PX) + 8192 <= 80 * 1024 ? 64 : 32, KSTEPS = KR / 16;
  static constexpr int Y_BYTES = KR * PY, X_BYTES = KR * PX;
  static constexpr int NYT = KR * OUT / 8;                              // chunks of 8 features in a tile
  static constexpr int NXT = KR * IN / 8;
  static constexpr int CY = (NYT + 255) / 256, CX = (NXT + 255) / 256;
};
// the upper halves of two floats: bf16 cut toward zero, so that no finite value becomes infinite (rounded to nearest, 3.3953e38 and more does)
__device__ __forceinline__ unsigned hi_bf16(float a, float b) {
  return __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, b), __builtin_bit_cast(unsigned, a), 0x07060302u);
}
typedef __attribute__((ext_vector_type(4))) short i16x4;
__device__ __forceinline__ bf16x8 tr_frag(const char* base, int pitch, int row, int feat, int lane) {
  // rows row + 8 h .. + 7 (two reads of 4), features feat .. feat + 31: lane i of 16 addresses row i / 4, features 4 (i % 4) ..
  const int i = lane & 15, h = lane >> 5, f = feat + ((lane >> 4) & 1) * 16 + 4 * (i & 3);
  const char* p = base + (row + 8 * h + (i >> 2)) * pitch + f * 2;
  typedef __attribute__((address_space(3))) i16x4* lp;
  const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)p), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(p + 4 * pitch));
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

template <int IN, int OUT, class TY>
__global__ void __launch_bounds__(256) k_mx8_wgrad(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, const TY* __restrict__ dY,
                                                   float* __restrict__ part, float* __restrict__ bpart, long long R, int rows_per_wg) {
  using C = WgradCfg<IN, OUT, TY>;
  __shared__ __attribute__((aligned(16))) char s_y[C::PLANES * C::Y_BYTES];
  __shared__ __attribute__((aligned(16))) char s_x[C::X_BYTES];
  __shared__ float s_b[256 * 8];
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
  const int wt = w % C::WT, wk = w / C::WT, wo = wt / C::WI, wi = wt % C::WI;
  const long long r0 = (long long)blockIdx.x * rows_per_wg, r1 = min(R, r0 + rows_per_wg);
  f32x16 acc[C::AO][C::AI];
#pragma unroll
  for (int a = 0; a < C::AO; ++a)
#pragma unroll
    for (int b = 0; b < C::AI; ++b) acc[a][b] = splat16(0.f);
  float bs[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  // the tile in flight: raw dY (8 features a chunk), codes and scale bytes.  Rows past the slice are clamped and their dY dropped.
  uint4 ry[C::CY][sizeof(TY) / 2];
  uint2 rx[C::CX];
  unsigned rs[C::CX];
  auto load = [&](long long r) {
#pragma unroll
    for (int u = 0; u < C::CY; ++u) {
      const int t = tid + 256 * u, row = t / (OUT / 8), f = (t % (OUT / 8)) * 8;
      const uint4* p = reinterpret_cast<const uint4*>(dY + min(r + row, r1 - 1) * OUT + f);
      if (C::NYT % 256 == 0 || t < C::NYT) {
#pragma unroll
        for (int k = 0; k < (int)sizeof(TY) / 2; ++k) ry[u][k] = p[k];
      }
    }
#pragma unroll
    for (int u = 0; u < C::CX; ++u) {
      const int t = tid + 256 * u, row = t / (IN / 8), f = (t % (IN / 8)) * 8;
      const long long rr = min(r + row, r1 - 1);
      if (C::NXT % 256 == 0 || t < C::NXT) {
        rx[u] = *reinterpret_cast<const uint2*>(codes + rr * IN + f);
        rs[u] = scales[rr * (IN / MX8_GROUP) + f / MX8_GROUP];
      }
    }
  };
  auto stage = [&](long long r) {
#pragma unroll
    for (int u = 0; u < C::CY; ++u) {
      const int t = tid + 256 * u, row = t / (OUT / 8), f = (t % (OUT / 8)) * 8;
      if (C::NYT % 256 != 0 && t >= C::NYT) break;
      const bool ok = r + row < r1;
      float v[8];
      if constexpr (C::PLANES == 1) unpack8(ry[u][0], v);
      else {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          v[4 * k] = __builtin_bit_cast(float, ry[u][k].x); v[4 * k + 1] = __builtin_bit_cast(float, ry[u][k].y);
          v[4 * k + 2] = __builtin_bit_cast(float, ry[u][k].z); v[4 * k + 3] = __builtin_bit_cast(float, ry[u][k].w);
        }
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) { v[k] = ok ? v[k] : 0.f; bs[k] += v[k]; }
      char* d = s_y + row * C::PY + f * 2;
#pragma unroll
      for (int pl = 0; pl < C::PLANES; ++pl) {
        uint4 o;
        if constexpr (C::PLANES == 1) o = uint4{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])};
        else o = uint4{hi_bf16(v[0], v[1]), hi_bf16(v[2], v[3]), hi_bf16(v[4], v[5]), hi_bf16(v[6], v[7])};
        *reinterpret_cast<uint4*>(d + pl * C::Y_BYTES) = o;
        if (pl + 1 < C::PLANES) {                                      // what this part leaves, exactly; nothing of an infinity, NaN of a NaN
          float p8[8];
          unpack8(o, p8);
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = v[k] == p8[k] ? 0.f : v[k] - p8[k];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < C::CX; ++u) {
      const int t = tid + 256 * u, row = t / (IN / 8), f = (t % (IN / 8)) * 8;
      if (C::NXT % 256 != 0 && t >= C::NXT) break;
      float v[8];
      codes8(rx[u], mx8_step(rs[u]), v);
      *reinterpret_cast<uint4*>(s_x + row * C::PX + f * 2) = uint4{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])};
    }
  };
  load(r0);
  for (long long r = r0; r < r1; r += C::KR) {
    stage(r);
    __syncthreads();
    load(r + C::KR);                                                    // (past the slice: clamped, never staged)
#pragma unroll
    for (int ks = 0; ks < C::KSTEPS; ks += C::WK) {
      const int row = (ks + wk) * 16;
      bf16x8 x[C::AI];
#pragma unroll
      for (int b = 0; b < C::AI; ++b) x[b] = tr_frag(s_x, C::PX, row, (wi * C::AI + b) * 32, lane);
#pragma unroll
      for (int pl = 0; pl < C::PLANES; ++pl)
#pragma unroll
        for (int a = 0; a < C::AO; ++a) {
          const bf16x8 y = tr_frag(s_y + pl * C::Y_BYTES, C::PY, row, (wo * C::AO + a) * 32, lane);
#pragma unroll
          for (int b = 0; b < C::AI; ++b) acc[a][b] = mfma32(y, x[b], acc[a][b]);
        }
    }
    __syncthreads();
  }
  const int h = lane >> 5, l32 = lane & 31;
  float* pw = part + ((size_t)blockIdx.x * C::WK + wk) * (OUT * IN);
#pragma unroll
  for (int a = 0; a < C::AO; ++a)
#pragma unroll
    for (int b = 0; b < C::AI; ++b)
#pragma unroll
      for (int v = 0; v < 16; ++v) pw[((wo * C::AO + a) * 32 + crow(v, h)) * IN + (wi * C::AI + b) * 32 + l32] = acc[a][b][v];
  // column sums: the threads of one 8-feature chunk (tid, tid + OUT / 8, ..) hold different rows
#pragma unroll
  for (int k = 0; k < 8; ++k) s_b[tid * 8 + k] = bs[k];
  __syncthreads();
  for (int o = tid; o < OUT; o += 256) {
    float t = 0.f;
    for (int q = 0; q < 256 / (OUT / 8); ++q) t += s_b[(q * (OUT / 8) + o / 8) * 8 + (o & 7)];
    bpart[(size_t)blockIdx.x * OUT + o] = t;
  }
}
// Fold of the partial results in slice order: 16 result quads x 16 groups of slices per workgroup, a thread sums its group's partials, the
// groups are added in order through LDS.  nW, nB: quads of dW (GW partials) and of db (GB partials).
__global__ void __launch_bounds__(256) k_mx8_wgrad_fold(const float4* __restrict__ part, const float4* __restrict__ bpart, float4* __restrict__ dW,
                                                        float4* __restrict__ db, int GW, int GB, int nW, int nB) {
  __shared__ float4 s_p[16][16];
  const int q = threadIdx.x & 15, gg = threadIdx.x >> 4;
  const int t = blockIdx.x * 16 + q;
  const bool isW = t < nW, isB = !isW && t < nW + nB;
  const int G = isW ? GW : GB, per = (G + 15) / 16, g0 = gg * per, g1 = min(G, g0 + per), n = isW ? nW : nB;
  const float4* src = isW ? part + t : bpart + (t - nW);
  float4 s = {0.f, 0.f, 0.f, 0.f};
  if (isW || isB)
    for (int g = g0; g < g1; g += 8) {
      float4 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = src[(size_t)min(g + u, g1 - 1) * n];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (g + u < g1) { s.x += v[u].x; s.y += v[u].y; s.z += v[u].z; s.w += v[u].w; }
    }
  s_p[gg][q] = s;
  __syncthreads();
  if (gg == 0 && (isW || isB)) {
    for (int k = 1; k < 16; ++k) { const float4 o = s_p[k][q]; s.x += o.x; s.y += o.y; s.z += o.z; s.w += o.w; }
    if (isW) dW[t] = s; else if (db) db[t - nW] = s;
  }
}

// Rows of a slice, a multiple of 64.  Up to 131,072 rows 256 slices (one workgroup a CU), beyond that 512: the second workgroup hides the
// first one's waits, and its partial result costs the fold.  The two cross between 80,000 and 150,000 rows, by shape; 256 / 512 slices, us a call:
//   rows             60,000     100,000     131,072     150,000     220,000     313,600
//   64 -> 256 bf16   17.7/20.3  21.5/24.7   28.9/31.4   31.7/31.3   41.7/38.8   53.0/47.7
//   128 -> 64 bf16   15.0/18.3  17.2/17.1   17.5/17.5   19.7/18.4   24.0/21.5   36.3/27.8
//   256 -> 64 fp32   21.6/22.5  27.7/26.5   31.7/29.9   36.6/32.3   47.0/42.7   61.9/52.3
//   64 -> 64 fp32    14.3/15.6  17.1/16.2   19.1/17.2   21.2/18.5   30.2/23.4   41.0/29.8
static long long wgrad_slice_rows(long long R) {
  const long long G = R <= 131072 ? 256 : 512, per = (R + G - 1) / G;
  return (per + 63) / 64 * 64;
}
static int wgrad_wk(int in_features, int out_features) { const int tiles = in_features * out_features / 1024; return tiles < 4 ? 4 / tiles : 1; }
static bool wgrad_built(int i, int o) {
  auto ok = [](int f) { return f == 32 || f == 64 || f == 128 || f == 256; };
  return ok(i) && ok(o) && i * o <= 64 * 256;
}
template <int IN, int OUT, class TY>
static void launch_mx8_wgrad(const uint8_t* codes, const uint8_t* scales, const TY* dY, float* dW, float* db, float* ws, long long R, hipStream_t s) {
  using C = WgradCfg<IN, OUT, TY>;
  const long long per = wgrad_slice_rows(R);
  const int G = (int)((R + per - 1) / per);
  float* bpart = ws + (size_t)G * C::WK * OUT * IN;
  k_mx8_wgrad<IN, OUT, TY><<<G, 256, 0, s>>>(codes, scales, dY, ws, bpart, R, (int)per);
  const int nW = IN * OUT / 4, nB = OUT / 4;
  k_mx8_wgrad_fold<<<(nW + nB + 15) / 16, 256, 0, s>>>((const float4*)ws, (const float4*)bpart, (float4*)dW, (float4*)db, G * C::WK, G, nW, nB);
}
template <class TY>
static void wgrad_shape(const uint8_t* codes, const uint8_t* scales, const TY* dY, float* dW, float* db, float* ws, long long R, int i, int o, hipStream_t s) {
#define WG(I, O) case I * 1000 + O: launch_mx8_wgrad<I, O, TY>(codes, scales, dY, dW, db, ws, R, s); break
  switch (i * 1000 + o) {
    WG(32, 32); WG(32, 64); WG(32, 128); WG(32, 256); WG(64, 32); WG(64, 64); WG(64, 128); WG(64, 256); WG(128, 32); WG(128, 64); WG(128, 128);
    WG(256, 32); WG(256, 64);
  }
#undef WG
}

static unsigned stream_grid(long long items, int per_wg) {
  const long long g = (items + per_wg - 1) / per_wg;
  return (unsigned)(g < 1 ? 1 : g > 8192 ? 8192 : g);
}

extern "C" {

int da_mx8_quant(const void* x, int x_bf16, void* codes, uint8_t* scales, long long rows, int D, int keep_nonzero, void* stream) {
  DA_CHECK_ARG(rows >= 0 && D >= 1, "da_mx8_quant: rows = %lld, D = %d", rows, D);
  if (rows == 0) return DA_OK;
  DA_CHECK_ARG(x && codes && scales, "da_mx8_quant: null pointer");
  DA_CHECK_ARG(((uintptr_t)x & (x_bf16 ? 1 : 3)) == 0, "da_mx8_quant: x is not aligned to its type");
  hipStream_t s = (hipStream_t)stream;
  const int G = (D + MX8_GROUP - 1) / MX8_GROUP;
  if (D % MX8_GROUP == 0 && (((uintptr_t)x & 15) | ((uintptr_t)codes & 7)) == 0) {
    const long long octs = rows * (D / 8);
    const unsigned g = stream_grid(octs, 256);
#define Q(T, K) k_mx8_quant<T, K><<<g, 256, 0, s>>>((const T*)x, (uint2*)codes, scales, octs)
    if (x_bf16) { if (keep_nonzero) Q(bf16_t, true); else Q(bf16_t, false); } else { if (keep_nonzero) Q(float, true); else Q(float, false); }
#undef Q
  } else {
    const unsigned g = stream_grid(rows * G, 8);
#define Q(T, K) k_mx8_quant_any<T, K><<<g, 256, 0, s>>>((const T*)x, (uint8_t*)codes, scales, rows * G, D, G)
    if (x_bf16) { if (keep_nonzero) Q(bf16_t, true); else Q(bf16_t, false); } else { if (keep_nonzero) Q(float, true); else Q(float, false); }
#undef Q
  }
  DA_CHECK_LAUNCH("da_mx8_quant");
  return DA_OK;
}

int da_mx8_dequant(const void* codes, const uint8_t* scales, void* out, int out_bf16, long long rows, int D, void* stream) {
  DA_CHECK_ARG(rows >= 0 && D >= 1, "da_mx8_dequant: rows = %lld, D = %d", rows, D);
  if (rows == 0) return DA_OK;
  DA_CHECK_ARG(out && codes && scales, "da_mx8_dequant: null pointer");
  DA_CHECK_ARG(((uintptr_t)out & (out_bf16 ? 1 : 3)) == 0, "da_mx8_dequant: out is not aligned to its type");
  hipStream_t s = (hipStream_t)stream;
  const int G = (D + MX8_GROUP - 1) / MX8_GROUP;
  if (D % MX8_GROUP == 0 && (((uintptr_t)out & 15) | ((uintptr_t)codes & 7)) == 0) {
    const long long octs = rows * (D / 8);
    const unsigned g = stream_grid(octs, 256);
    if (out_bf16) k_mx8_dequant<bf16_t><<<g, 256, 0, s>>>((const uint2*)codes, scales, (bf16_t*)out, octs);
    else k_mx8_dequant<float><<<g, 256, 0, s>>>((const uint2*)codes, scales, (float*)out, octs);
  } else {
    const unsigned g = stream_grid(rows * D, 256);
    if (out_bf16) k_mx8_dequant_any<bf16_t><<<g, 256, 0, s>>>((const int8_t*)codes, scales, (bf16_t*)out, rows * D, D, G);
    else k_mx8_dequant_any<float><<<g, 256, 0, s>>>((const int8_t*)codes, scales, (float*)out, rows * D, D, G);
  }
  DA_CHECK_LAUNCH("da_mx8_dequant");
  return DA_OK;
}

int da_relu_dropout_bwd_mx8(const void* codes, const void* dy, void* dx, int is_bf16, long long numel, float p, void* stream) {
  DA_CHECK_ARG(numel >= 0, "da_relu_dropout_bwd_mx8: numel = %lld", numel);
  DA_CHECK_ARG(p >= 0.f && p < 1.f, "da_relu_dropout_bwd_mx8: p in [0,1)");
  if (numel == 0) return DA_OK;
  DA_CHECK_ARG(codes && dy && dx, "da_relu_dropout_bwd_mx8: null pointer");
  DA_CHECK_ARG((((uintptr_t)dy | (uintptr_t)dx) & (is_bf16 ? 1 : 3)) == 0, "da_relu_dropout_bwd_mx8: not aligned to its type");
  hipStream_t s = (hipStream_t)stream;
  unsigned thr; float scale;
  drop_consts(p, &thr, &scale);
  if (numel % 8 == 0 && (((uintptr_t)dy | (uintptr_t)dx) & 15) == 0 && ((uintptr_t)codes & 7) == 0) {
    const unsigned g = stream_grid(numel / 8, 256);
    if (is_bf16) k_relu_drop_bwd_mx8<bf16_t><<<g, 256, 0, s>>>((const uint2*)codes, (const bf16_t*)dy, (bf16_t*)dx, numel / 8, scale);
    else k_relu_drop_bwd_mx8<float><<<g, 256, 0, s>>>((const uint2*)codes, (const float*)dy, (float*)dx, numel / 8, scale);
  } else {
    const unsigned g = stream_grid(numel, 256);
    if (is_bf16) k_relu_drop_bwd_mx8_any<bf16_t><<<g, 256, 0, s>>>((const int8_t*)codes, (const bf16_t*)dy, (bf16_t*)dx, numel, scale);
    else k_relu_drop_bwd_mx8_any<float><<<g, 256, 0, s>>>((const int8_t*)codes, (const float*)dy, (float*)dx, numel, scale);
  }
  DA_CHECK_LAUNCH("da_relu_dropout_bwd_mx8");
  return DA_OK;
}

long long da_linear_wgrad_mx8_workspace(long long R, int in_features, int out_features) {
  if (R < 0 || !wgrad_built(in_features, out_features)) return -1;
  const int wk = wgrad_wk(in_features, out_features);
  const long long per = R ? wgrad_slice_rows(R) : 1, G = (R + per - 1) / per;
  return (long long)sizeof(float) * G * ((long long)wk * in_features * out_features + out_features);
}
int da_linear_wgrad_mx8(const void* codes, const uint8_t* scales, const void* dY, int dy_bf16, float* dW, float* db, void* workspace,
                        long long workspace_bytes, long long R, int in_features, int out_features, void* stream) {
  DA_CHECK_ARG(R >= 1, "da_linear_wgrad_mx8: R = %lld", R);
  if (!wgrad_built(in_features, out_features)) {
    da_set_error("da_linear_wgrad_mx8: %d -> %d features not built", in_features, out_features);
    return DA_ERR_UNSUPPORTED;
  }
  DA_CHECK_ARG(codes && scales && dY && dW, "da_linear_wgrad_mx8: null pointer");
  DA_CHECK_ARG(((((uintptr_t)dY | (uintptr_t)dW | (uintptr_t)db | (uintptr_t)workspace) & 15) | ((uintptr_t)codes & 7)) == 0,
               "da_linear_wgrad_mx8: dY, dW, db and the workspace must be 16-byte aligned, the codes 8-byte");
  DA_CHECK_ARG(workspace && workspace_bytes >= da_linear_wgrad_mx8_workspace(R, in_features, out_features), "da_linear_wgrad_mx8: workspace too small");
  hipStream_t s = (hipStream_t)stream;
  if (dy_bf16) wgrad_shape<bf16_t>((const uint8_t*)codes, scales, (const bf16_t*)dY, dW, db, (float*)workspace, R, in_features, out_features, s);
  else wgrad_shape<float>((const uint8_t*)codes, scales, (const float*)dY, dW, db, (float*)workspace, R, in_features, out_features, s);
  DA_CHECK_LAUNCH("da_linear_wgrad_mx8");
  return DA_OK;
}

}  // extern "C"
