// Per-head edge attention, forward and backward: the core of NodeEdgeBlockImproved (neuralnet/layers.py:115-141), where the edge-modulated
// products of a head are summed into one score and the softmax over the keys is per head (the plain block, k_backward.hip, has one per
// channel).  Per pair (i,j) and channel c of head h(c), m_ij = m_i m_j:
//   Y_ijc = s Q_ic K_jc (1 + m_ij E1_ijc) + m_ij E2_ijc            the input of e_out
//   S_ijh = sum over the head's channels of Y;   S' = cap tanh(S / cap) where cap > 0, else S
//   P_ijh = softmax over the keys j with group_j == group_i >= 0 (all keys without groups);   wV_ic = sum_j P_ijh V_jc
// A row without a key gets wV = 0.  With G_ijc = dY_ijc + dS_ijh, dS = P (dP - D) (1 - (S'/cap)^2), dP_ijh = dwV_i . V_j and
// D_ih = dwV_i . wV_i (sums over the head's channels) the gradients are
//   dE2 = m G;  dE1 = m G s Q K;  dQ_i = sum_j G s (1 + m E1) K_j;  dK_j = sum_i G s (1 + m E1) Q_i;  dV_j = sum_i P dwV_i.
// The forward leaves S' (B,n,n,H) and the softmax statistics, 4 H bytes a pair beside 2-4 dx for each of E1 and E2: the backward then
// needs neither E2 nor the scores' sum again, and E1, the one wide operand left, may be held in 8 bits (mx8_util.h).
//
// Bound: HBM.  Forward E1, E2 in, Y out; backward E1, dY in, dE1, dE2 out: 3 and 4 (3.5 with 8 bits of E1 beside bf16) streams of B n n dx
// elements against about 12 operations per element each way.  So every stream is touched once, in 16-byte accesses, and what repeats stays in
// registers: a lane holds C channels of one head, LP = dx / C lanes (a power of two) a pair, a wave 64 / LP keys at a time for RW query
// rows, whose Q (dwV, dQ) never move; K_j and V_j are fetched once for the RW rows.  A head's sum runs over df / C neighbouring lanes
// (DPP).  E1 and E2 are read through a buffer descriptor whose range ends at the rows in hand: a masked pair, a row past the end and a
// channel past dx get an offset outside it, so the hardware returns the 0 that the formula wants and moves no data.
// Measured, dx = 256, 8 heads, graphs padded by a quarter on average: B = 16, n = 140 bf16 forward 88 us, backward 135 us (607 MB, 4.5 TB/s) + fold
// 6.8; B = 16, n = 300 bf16 with 8-bit E1, cap and groups 449 us (2.0 GB, 4.5 TB/s), 528 us (2.5 GB, 4.75 TB/s) + 19; B = 16, n = 140 fp32 158,
// 256 + 6.8 us.  A copy of 4 GiB runs at 4.75 TB/s on the same card.
#include "mfma_util.h"
#include "mx8_util.h"
#include <initializer_list>
#include <type_traits>

// Which product is fused into which sum is written out (fmaf) and left to nobody else: the variants of a kernel then round alike, and the
// forward gives the same bits with and without a backward to come.
#pragma clang fp contract(off)
__device__ __forceinline__ float fma_(float a, float b, float c) { return __builtin_fmaf(a, b, c); }

struct HeadArgs {
  const float *Q, *K, *V;
  const void *E1, *E2;                  // E1: TE, or its codes (8-bit backward)
  const uint8_t* E1s;                   // scale bytes of E1's codes
  const uint8_t* nm;
  const int* grp;                       // nullable
  float qscale, cap;
  int n, dx, H, lp_log;                 // lp_log: log2 of the lanes a pair takes
  // forward out
  void* Y;
  float *wV, *S, *stat;                 // S (B,n,n,H) and stat (B,n,H,2) = {max, 1 / sum}: nullable (no backward wanted)
  uint8_t *q1, *q1s;                    // 8-bit copy of E1: nullable
  // backward
  const void* dY;
  const float* dwV;
  float *dQp, *dKp, *dVp;               // (jchunks, B, n, dx), (iblocks, B, n, dx) x 2
  void *dE1, *dE2;
  int B, jchunk, njc, nib;
};

#define OOB 0x80000000u                 // past every descriptor's range, also with a row's offset added (the host keeps both below 2^31)
// cache policy of the streams that pass once (E1, E2, Y, dY, dE1, dE2): non-temporal where a lane's channels are one 16-byte access, so that K
// and V keep the L2 (bf16: forward B = 16, n = 140 96 -> 88 us, backward n = 300 565 -> 532 us; fp32: 169 -> 158 and 518 -> 498 us).  Eight
// fp32 channels take two accesses that share every 64 bytes, and want the line kept for the second (n = 93: 49 / 49 us, non-temporal 52 / 55)
template <class TE, int C> constexpr int nt() { return sizeof(TE) * C == 16 ? 2 : 0; }
template <class TE, int C> struct Raw { unsigned w[sizeof(TE) * C / 4]; };
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void* p, unsigned bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)bytes, 0x00027000);
}
typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
typedef __attribute__((ext_vector_type(2))) unsigned u32x2;
template <int AUX = 0, int W>
__device__ __forceinline__ void bld(__amdgpu_buffer_rsrc_t r, unsigned off, unsigned (&w)[W], unsigned soff = 0) {
  if constexpr (W == 1) w[0] = __builtin_amdgcn_raw_buffer_load_b32(r, off, soff, AUX);
  else if constexpr (W == 2) { const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(r, off, soff, AUX); w[0] = v.x; w[1] = v.y; }
  else {
#pragma unroll
    for (int k = 0; k < W / 4; ++k) {
      const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(r, off + 16 * k, soff, AUX);
      w[4 * k] = v.x; w[4 * k + 1] = v.y; w[4 * k + 2] = v.z; w[4 * k + 3] = v.w;
    }
  }
}
template <class TE, int C>
__device__ __forceinline__ void widen(const Raw<TE, C>& r, float (&v)[C]) {
#pragma unroll
  for (int k = 0; k < C; ++k) {
    if constexpr (sizeof(TE) == 2) v[k] = k & 1 ? bf16_hi(r.w[k / 2]) : bf16_lo(r.w[k / 2]);
    else v[k] = __builtin_bit_cast(float, r.w[k]);
  }
}
// C values of type TE through a descriptor: offsets outside its range store nothing.  No scalar offset on these: after a 16-byte buffer store
// with an SGPR offset the compiler inserts no wait state, and here the next vector instruction overwrote the store's first data register
// before it had been read.
template <class TE, int C>
__device__ __forceinline__ void bst(__amdgpu_buffer_rsrc_t r, unsigned off, const float (&v)[C]) {
  if constexpr (sizeof(TE) == 2 && C == 8) {
    const u32x4 o = {pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])};
    __builtin_amdgcn_raw_buffer_store_b128(o, r, off, 0, nt<TE, C>());
  } else if constexpr (sizeof(TE) == 2) {
    const u32x2 o = {pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
    __builtin_amdgcn_raw_buffer_store_b64(o, r, off, 0, nt<TE, C>());
  } else {
#pragma unroll
    for (int k = 0; k < C; k += 4) {
      const u32x4 o = {__builtin_bit_cast(unsigned, v[k]), __builtin_bit_cast(unsigned, v[k + 1]), __builtin_bit_cast(unsigned, v[k + 2]),
                       __builtin_bit_cast(unsigned, v[k + 3])};
      __builtin_amdgcn_raw_buffer_store_b128(o, r, off + 4 * k, 0, nt<TE, C>());
    }
  }
}
template <class TE, int C>
__device__ __forceinline__ void gst(TE* p, const float (&v)[C]) {
  if constexpr (sizeof(TE) == 2 && C == 8) {
    *reinterpret_cast<uint4*>(p) = uint4{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])};
  } else if constexpr (sizeof(TE) == 2) {
    *reinterpret_cast<uint2*>(p) = uint2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
  } else {
#pragma unroll
    for (int k = 0; k < C; k += 4) *reinterpret_cast<float4*>(p + k) = float4{v[k], v[k + 1], v[k + 2], v[k + 3]};
  }
}
#define DPPF(v, ctrl) __builtin_bit_cast(float, MX8_DPP(__builtin_bit_cast(unsigned, v), ctrl))
// sum over 2^HLOG neighbouring lanes, in every one of them
template <int HLOG>
__device__ __forceinline__ float head_sum(float v) {
  if constexpr (HLOG >= 1) v += DPPF(v, 0xB1);
  if constexpr (HLOG >= 2) v += DPPF(v, 0x4E);
  if constexpr (HLOG >= 3) v += DPPF(v, 0x141);
  if constexpr (HLOG >= 4) v += DPPF(v, 0x140);
  return v;
}

// ---------------------------------------------------------------------------------------------------------------------------------
// Forward.  A workgroup owns RW query rows; its 4 waves x 64 / LP key slots walk the keys, each with an online softmax of its own (running
// maximum, sum, weighted V in registers), merged over the slots by lane exchange and over the waves in LDS.
template <class TE, int C, int HLOG, int RW, bool SAVE, bool MX8>
__global__ void __launch_bounds__(256) k_attn_head_fwd(HeadArgs a) {
  extern __shared__ float s_st[];                                       // [4][RW][dx] weighted V, [4][RW][H][2] maximum, sum
  const int n = a.n, dx = a.dx, H = a.H;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, slot = lane >> a.lp_log, li = lane & ((1 << a.lp_log) - 1);
  const int NS = 64 >> a.lp_log, JS = 4 * NS;
  const bool act = li * C < dx;
  const int c = act ? li * C : 0, h = c / (C << HLOG);
  const int nblk = (n + RW - 1) / RW, b = blockIdx.x / nblk, i0 = (blockIdx.x - b * nblk) * RW;
  const int rows = min(RW, n - i0);
  const size_t node0 = (size_t)b * n, row0 = node0 + i0;
  const uint8_t* nm = a.nm + node0;
  const int* grp = a.grp ? a.grp + node0 : nullptr;
  const unsigned es = sizeof(TE);
  const __amdgpu_buffer_rsrc_t r1 = rsrc((const TE*)a.E1 + row0 * n * dx, rows * n * dx * es), r2 = rsrc((const TE*)a.E2 + row0 * n * dx, rows * n * dx * es);
  const __amdgpu_buffer_rsrc_t rk = rsrc(a.K + node0 * dx, n * dx * 4), rv = rsrc(a.V + node0 * dx, n * dx * 4);
  const __amdgpu_buffer_rsrc_t rq = rsrc(a.Q + row0 * dx, rows * dx * 4);
  float q[RW][C], acc[RW][C], m[RW], l[RW];
  bool mi[RW];
  int gi[RW];
#pragma unroll
  for (int t = 0; t < RW; ++t) {
    Raw<float, C> rw;
    bld(rq, act ? (t * dx + c) * 4 : OOB, rw.w);
    widen(rw, q[t]);
    const int i = min(i0 + t, n - 1);
    mi[t] = __builtin_amdgcn_readfirstlane(t < rows ? (int)nm[i] : 0) != 0;
    gi[t] = grp ? grp[i] : 0;
    m[t] = -INFINITY; l[t] = 0.f;
#pragma unroll
    for (int k = 0; k < C; ++k) { q[t][k] *= a.qscale; acc[t][k] = 0.f; }
  }
  const float inv_cap = a.cap > 0.f ? 1.f / a.cap : 0.f;
  const __amdgpu_buffer_rsrc_t ry = rsrc((TE*)a.Y + row0 * n * dx, rows * n * dx * es);
  const __amdgpu_buffer_rsrc_t rS = rsrc(SAVE ? a.S + row0 * n * H : nullptr, SAVE ? rows * n * H * 4 : 0);
  const __amdgpu_buffer_rsrc_t rc = rsrc(MX8 ? a.q1 + row0 * n * dx : nullptr, MX8 ? rows * n * dx : 0);
  const __amdgpu_buffer_rsrc_t rcs = rsrc(MX8 ? a.q1s + row0 * n * (dx / MX8_GROUP) : nullptr, MX8 ? rows * n * (dx / MX8_GROUP) : 0);
  Raw<TE, C> e1n[RW], e2n[RW];          // a row's operands of the next key: loaded as soon as the present key's are widened
  Raw<float, C> kn, vn;
  // node flags of a key two steps ahead of its use: they decide the addresses of the next step's loads
  struct Meta { uint8_t m; int g; };
  auto meta = [&](int j) { const int jc = min(j, n - 1); return Meta{nm[jc], grp ? grp[jc] : 0}; };
  auto fetch_kv = [&](int j) {
    const unsigned ko = act && j < n ? (unsigned)(j * dx + c) * 4 : OOB;
    bld(rk, ko, kn.w); bld(rv, ko, vn.w);
  };
  // byte offset of a row's pair = the key's offset (one register for all rows) + the row's (uniform: the instruction's scalar offset); a row
  // past the end, a masked pair, a key past the end: OOB.  E1 and E2 of masked pairs are not read
  const unsigned row_c = (unsigned)(n * dx), row_e = row_c * es;
  auto fetch = [&](int t, unsigned eo) {
    const unsigned o = mi[t] ? eo : OOB, so = mi[t] ? t * row_e : 0;
    bld<nt<TE, C>()>(r1, o, e1n[t].w, so); bld<nt<TE, C>()>(r2, o, e2n[t].w, so);
  };
  auto key_off = [&](int j, uint8_t mj) { return act & (j < n) & (mj != 0) ? (unsigned)(j * dx + c) * es : OOB; };
  const int jf = w * NS + slot;
  Meta f0 = meta(jf), f1 = meta(jf + JS);
  fetch_kv(jf);
#pragma unroll
  for (int t = 0; t < RW; ++t) fetch(t, key_off(jf, f0.m));
  for (int j0 = 0; j0 < n; j0 += JS) {
    const int j = j0 + jf;
    float kk[C], vv[C];
    widen(kn, kk); widen(vn, vv);
    const int gj = j < n ? f0.g : -1;
    f0 = f1;
    f1 = meta(j + 2 * JS);
    fetch_kv(j + JS);
    const bool st = act & (j < n);
    const unsigned nx = key_off(j + JS, f0.m), jc = (unsigned)(j * dx + c), oY = st ? jc * es : OOB, oC = st ? jc : OOB;
    const unsigned oS = st & ((li & ((1 << HLOG) - 1)) == 0) ? (unsigned)(j * H + h) * 4 : OOB;
    const unsigned oCs = st & (c % MX8_GROUP == 0) ? (unsigned)(j * (dx / MX8_GROUP) + c / MX8_GROUP) : OOB;
#pragma unroll
    for (int t = 0; t < RW; ++t) {
      float e1[C], e2[C], y[C];
      widen(e1n[t], e1); widen(e2n[t], e2);
      fetch(t, nx);
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < C; ++k) { const float x = q[t][k] * kk[k]; y[k] = fma_(x, e1[k], x + e2[k]); s += y[k]; }
      bst<TE, C>(ry, oY + t * row_e, y);
      if constexpr (MX8) {
        unsigned mb = 0;
#pragma unroll
        for (int k = 0; k < C; ++k) mb = dpp_max_u32(mb, abs_bits(e1[k]));
        const unsigned sb = mx8_scale(C == 8 ? quad_max(mb) : oct_max(mb));
        const float inv = mx8_inv(sb);
        const unsigned w0 = mx8_pack4<false>(e1[0], e1[1], e1[2], e1[3], inv), co = oC + t * row_c;
        if constexpr (C == 8) __builtin_amdgcn_raw_buffer_store_b64(u32x2{w0, mx8_pack4<false>(e1[4], e1[5], e1[6], e1[7], inv)}, rc, co, 0, nt<TE, C>());
        else __builtin_amdgcn_raw_buffer_store_b32(w0, rc, co, 0, nt<TE, C>());
        __builtin_amdgcn_raw_buffer_store_b8((uint8_t)sb, rcs, oCs + t * (row_c / MX8_GROUP), 0, 0);
      }
      s = head_sum<HLOG>(s);
      if (a.cap > 0.f) s = a.cap * tanhf(s * inv_cap);
      const bool on = (gj >= 0) & (gj == gi[t]) & (s != -INFINITY);      // (a score of -inf shuts the key out like a group does: V is not looked at)
      s = on ? s : -INFINITY;
      if constexpr (SAVE)
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, s), rS, oS + t * (unsigned)(n * H) * 4, 0, 0);
      const float mx = fmaxf(m[t], s), mg = mx == -INFINITY ? 0.f : mx;
      const float sc = __expf(m[t] - mg), p = on ? __expf(s - mg) : 0.f;
      m[t] = mx;
      l[t] = fma_(l[t], sc, p);
#pragma unroll
      for (int k = 0; k < C; ++k) acc[t][k] = fma_(p, on ? vv[k] : 0.f, acc[t][k] * sc);
    }
  }
  for (int off = 1 << a.lp_log; off < 64; off <<= 1)                    // the key slots of the wave
#pragma unroll
    for (int t = 0; t < RW; ++t) {
      const float mo = __shfl_xor(m[t], off), M = fmaxf(m[t], mo), mg = M == -INFINITY ? 0.f : M;
      const float x = __expf(m[t] - mg), y = __expf(mo - mg);
      l[t] = fma_(l[t], x, __shfl_xor(l[t], off) * y);
      m[t] = M;
#pragma unroll
      for (int k = 0; k < C; ++k) acc[t][k] = fma_(acc[t][k], x, __shfl_xor(acc[t][k], off) * y);
    }
  float* s_ml = s_st + 4 * RW * dx;
  if (slot == 0 && act) {
#pragma unroll
    for (int t = 0; t < RW; ++t) {
      gst(s_st + (w * RW + t) * dx + c, acc[t]);
      if ((li & ((1 << HLOG) - 1)) == 0) { s_ml[((w * RW + t) * H + h) * 2] = m[t]; s_ml[((w * RW + t) * H + h) * 2 + 1] = l[t]; }
    }
  }
  __syncthreads();
  const int df = C << HLOG;
  for (int u = threadIdx.x; u < rows * dx; u += 256) {
    const int t = u / dx, cc = u - t * dx, hh = cc / df;
    float M = -INFINITY, L = 0.f, A = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) M = fmaxf(M, s_ml[((k * RW + t) * H + hh) * 2]);
    const float mg = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float x = __expf(s_ml[((k * RW + t) * H + hh) * 2] - mg);
      L = fma_(s_ml[((k * RW + t) * H + hh) * 2 + 1], x, L); A = fma_(s_st[(k * RW + t) * dx + cc], x, A);
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;                         // no key: 0
    a.wV[(row0 + t) * dx + cc] = L == 0.f ? 0.f : A * inv;
    if (SAVE && cc % df == 0) *reinterpret_cast<float2*>(a.stat + ((row0 + t) * H + hh) * 2) = float2{mg, inv};
  }
}

// ---------------------------------------------------------------------------------------------------------------------------------
// Backward.  A workgroup of NW waves owns NW RW query rows (RW a wave) and a chunk of keys; its waves take the same keys at the same time, so dK_j
// and dV_j are summed over the workgroup's rows in registers and LDS, and only one partial result per NW RW rows reaches memory.  dQ
// stays in registers over the chunk.  k_attn_head_fold adds the partial results in order (no atomics: the sums do not depend on timing).
#define HEAD_NW 8
// rows a wave: what its registers hold without spilling (two waves a SIMD)
__host__ __device__ constexpr int head_rw(bool bf16, int C) { return bf16 || C == 4 ? 4 : 2; }
// Workgroups are dealt to the 8 XCDs in turn, each with an L2 of its own: the blocks are cut into 8 runs, so that the row blocks of a chunk of
// keys meet in one of them (dx = 64, B = 60, n = 150 158 -> 151 us, dx = 256, B = 16, n = 300 531 -> 524 us).  The forward stays dealt in turn:
// it skips what padding masks, and 8 runs of graphs of different sizes do not end together (n = 300 187 -> 198 us).
__device__ __forceinline__ unsigned xcd_run(unsigned bid, unsigned grid) {
  const unsigned x = bid & 7, q = grid >> 3, r = grid & 7;
  return x * q + (x < r ? x : r) + (bid >> 3);
}
template <class TY, int C, int HLOG, bool MX8>
__global__ void __launch_bounds__(64 * HEAD_NW) k_attn_head_bwd(HeadArgs a) {
  constexpr int RW = head_rw(sizeof(TY) == 2, C), NW = HEAD_NW;
  extern __shared__ float s_kv[];                                       // [2][NW][NS][2][dx]
  const int n = a.n, dx = a.dx, H = a.H;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, slot = lane >> a.lp_log, li = lane & ((1 << a.lp_log) - 1);
  const int NS = 64 >> a.lp_log;
  const bool act = li * C < dx;
  const int c = act ? li * C : 0, h = c / (C << HLOG);
  const int bid = (int)xcd_run(blockIdx.x, gridDim.x), ib = bid % a.nib, jc = (bid / a.nib) % a.njc, b = bid / a.nib / a.njc;
  const int i0 = (ib * NW + w) * RW, rows = __builtin_amdgcn_readfirstlane(max(0, min(RW, n - i0)));      // (uniform: descriptors are made of it)
  const int j_lo = jc * a.jchunk, j_hi = min(n, j_lo + a.jchunk);
  const size_t node0 = (size_t)b * n, row0 = node0 + min(i0, n - 1);
  const uint8_t* nm = a.nm + node0;
  const unsigned es = sizeof(TY), range = (unsigned)(rows * n) * dx;
  const __amdgpu_buffer_rsrc_t r1 = MX8 ? rsrc((const uint8_t*)a.E1 + row0 * n * dx, range) : rsrc((const TY*)a.E1 + row0 * n * dx, range * es);
  const __amdgpu_buffer_rsrc_t rsc = rsrc(MX8 ? a.E1s + row0 * n * (dx / MX8_GROUP) : nullptr, MX8 ? range / MX8_GROUP : 0);
  const __amdgpu_buffer_rsrc_t ry = rsrc((const TY*)a.dY + row0 * n * dx, range * es);
  const __amdgpu_buffer_rsrc_t r1o = rsrc((TY*)a.dE1 + row0 * n * dx, range * es), r2o = rsrc((TY*)a.dE2 + row0 * n * dx, range * es);
  const __amdgpu_buffer_rsrc_t rS = rsrc(a.S + row0 * n * H, rows * n * H * 4);
  const __amdgpu_buffer_rsrc_t rk = rsrc(a.K + node0 * dx, n * dx * 4), rv = rsrc(a.V + node0 * dx, n * dx * 4);
  const __amdgpu_buffer_rsrc_t rq = rsrc(a.Q + row0 * dx, rows * dx * 4), ro = rsrc(a.wV + row0 * dx, rows * dx * 4), rg = rsrc(a.dwV + row0 * dx, rows * dx * 4);
  float q[RW][C], g[RW][C], dq[RW][C], D[RW], mx[RW], il[RW];
  bool mi[RW];
#pragma unroll
  for (int t = 0; t < RW; ++t) {
    const unsigned off = act ? (unsigned)(t * dx + c) * 4 : OOB;        // rows past the end: zeros throughout
    Raw<float, C> x;
    bld(rq, off, x.w); widen(x, q[t]);
    bld(rg, off, x.w); widen(x, g[t]);
    float o[C], d = 0.f;
    bld(ro, off, x.w); widen(x, o);
#pragma unroll
    for (int k = 0; k < C; ++k) { d = fma_(g[t][k], o[k], d); q[t][k] *= a.qscale; dq[t][k] = 0.f; }
    D[t] = head_sum<HLOG>(d);
    const int i = min(i0 + t, n - 1);
    mi[t] = __builtin_amdgcn_readfirstlane(t < rows ? (int)nm[i] : 0) != 0;
    const float2 st = *reinterpret_cast<const float2*>(a.stat + ((node0 + i) * H + h) * 2);
    mx[t] = t < rows ? st.x : 0.f; il[t] = t < rows ? st.y : 0.f;
  }
  const float inv_cap = a.cap > 0.f ? 1.f / a.cap : 0.f;
  constexpr int W1 = MX8 ? C / 4 : (int)sizeof(TY) * C / 4;
  struct Ops { unsigned e1[W1], sc, s; Raw<TY, C> dy; };
  Ops op[RW];                           // a row's operands of the next key: loaded as soon as the present key's are widened
  Raw<float, C> kn, vn;
  auto meta = [&](int j) { return nm[min(j, n - 1)]; };
  auto fetch_kv = [&](int j) {
    const unsigned ko = act && j < j_hi ? (unsigned)(j * dx + c) * 4 : OOB;
    bld(rk, ko, kn.w); bld(rv, ko, vn.w);
  };
  // (offsets as in the forward: the key's in one register for all rows, the row's uniform)
  struct Off { unsigned e1, sc, y, s; };
  auto key_off = [&](int j, uint8_t mj) {
    const bool on = act & (j < j_hi), pm = on & (mj != 0);
    const unsigned jc = (unsigned)(j * dx + c);
    return Off{pm ? (MX8 ? jc : jc * es) : OOB, pm ? (unsigned)(j * (dx / MX8_GROUP) + c / MX8_GROUP) : OOB, on ? jc * es : OOB,
               on ? (unsigned)(j * H + h) * 4 : OOB};
  };
  const unsigned row_c = (unsigned)(n * dx), row_e = row_c * es;
  auto fetch = [&](int t, const Off& o) {
    const bool in = t < rows;
    bld<nt<TY, C>()>(r1, mi[t] ? o.e1 : OOB, op[t].e1, mi[t] ? t * (MX8 ? row_c : row_e) : 0);
    if constexpr (MX8) op[t].sc = __builtin_amdgcn_raw_buffer_load_b8(rsc, mi[t] ? o.sc : OOB, mi[t] ? t * (row_c / MX8_GROUP) : 0, 0);
    bld<nt<TY, C>()>(ry, in ? o.y : OOB, op[t].dy.w, in ? t * row_e : 0);
    op[t].s = __builtin_amdgcn_raw_buffer_load_b32(rS, in ? o.s : OOB, in ? (unsigned)(t * n * H) * 4 : 0, 0);
  };
  uint8_t m0 = meta(j_lo + slot), m1 = meta(j_lo + slot + NS);
  fetch_kv(j_lo + slot);
#pragma unroll
  for (int t = 0; t < RW; ++t) fetch(t, key_off(j_lo + slot, m0));
  // what this thread adds up of the waves' dK_j, dV_j: one quad of one key slot (NS 2 dx / 4 <= 256 of them)
  const int quads = 2 * dx / 4, r_sl = threadIdx.x / quads, r_c = (threadIdx.x - r_sl * quads) * 4, r_src = r_sl * 2 * dx + r_c;
  const bool red = r_sl < NS, red_k = r_c < dx;
  const size_t part0 = (((size_t)ib * a.B + b) * n + j_lo) * dx;
  const __amdgpu_buffer_rsrc_t rdk = rsrc(a.dKp + part0, (j_hi - j_lo) * dx * 4), rdv = rsrc(a.dVp + part0, (j_hi - j_lo) * dx * 4);
  unsigned r_off = (unsigned)(r_sl * dx + (red_k ? r_c : r_c - dx)) * 4;
  int buf = 0;
  for (int j0 = j_lo; j0 < j_hi; j0 += NS, buf ^= 1) {
    const int j = j0 + slot;
    float kk[C], vv[C], dk[C], dv[C];
    widen(kn, kk); widen(vn, vv);
    const bool mj = (j < j_hi) & (m0 != 0);
    m0 = m1;
    m1 = meta(j + 2 * NS);
    fetch_kv(j + NS);
    const Off nx = key_off(j + NS, m0);
    const unsigned oE = act & (j < j_hi) ? (unsigned)(j * dx + c) * es : OOB;
#pragma unroll
    for (int k = 0; k < C; ++k) dk[k] = dv[k] = 0.f;
#pragma unroll
    for (int t = 0; t < RW; ++t) {
      float e1[C], G[C], o1[C], o2[C], dp = 0.f;
      if constexpr (MX8) {
        const float step = mx8_step(op[t].sc);                            // (a masked pair reads 0, and codes of 0)
#pragma unroll
        for (int k = 0; k < C; k += 4) {
          e1[k] = mx8_elem<0>(op[t].e1[k / 4]) * step; e1[k + 1] = mx8_elem<1>(op[t].e1[k / 4]) * step;
          e1[k + 2] = mx8_elem<2>(op[t].e1[k / 4]) * step; e1[k + 3] = mx8_elem<3>(op[t].e1[k / 4]) * step;
        }
      } else {
        Raw<TY, C> r;
#pragma unroll
        for (int k = 0; k < W1; ++k) r.w[k] = op[t].e1[k];
        widen(r, e1);
      }
      widen(op[t].dy, G);
      const float s = __builtin_bit_cast(float, op[t].s), cs = s * inv_cap;
      fetch(t, nx);
#pragma unroll
      for (int k = 0; k < C; ++k) dp = fma_(g[t][k], vv[k], dp);
      dp = head_sum<HLOG>(dp);
      const bool on = (t < rows) & (j < j_hi) & (s != -INFINITY);
      const float p = on ? __expf(s - mx[t]) * il[t] : 0.f;
      const float ds = on ? p * (dp - D[t]) * fma_(-cs, cs, 1.f) : 0.f;
      const bool pm = mj & mi[t];
#pragma unroll
      for (int k = 0; k < C; ++k) {
        G[k] += ds;
        o2[k] = pm ? G[k] : 0.f;
        o1[k] = o2[k] * (q[t][k] * kk[k]);
        const float x = fma_(G[k], e1[k], G[k]);
        dq[t][k] = fma_(x, kk[k], dq[t][k]);
        dk[k] = fma_(x, q[t][k], dk[k]);
        dv[k] = fma_(p, on ? g[t][k] : 0.f, dv[k]);                     // (an unseen key: the row's dwV is not looked at)
      }
      bst<TY, C>(r1o, oE + t * row_e, o1); bst<TY, C>(r2o, oE + t * row_e, o2);
      __builtin_amdgcn_sched_barrier(0);                                // one row's temporaries at a time: mixed, the rows spill
    }
    float* mine = s_kv + (((buf * NW + w) * NS + slot) * 2) * dx + c;
    if (act) { gst(mine, dk); gst(mine + dx, dv); }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");     // LDS only: the global loads in flight stay in flight
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    // the waves' sums; the other buffer is written next, and this one again only after the barrier that follows this read
    if (red) {
      const float* src = s_kv + (size_t)buf * NW * NS * 2 * dx + r_src;
      float4 t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < NW; ++k) {
        const float4 x = *reinterpret_cast<const float4*>(src + k * NS * 2 * dx);
        t.x += x.x; t.y += x.y; t.z += x.z; t.w += x.w;
      }
      const u32x4 o = __builtin_bit_cast(u32x4, t);
      __builtin_amdgcn_raw_buffer_store_b128(o, rdk, red_k ? r_off : OOB, 0, 0);         // (keys past the chunk are outside the range)
      __builtin_amdgcn_raw_buffer_store_b128(o, rdv, red_k ? OOB : r_off, 0, 0);
      r_off += (unsigned)(NS * dx) * 4;
    }
  }
  for (int off = 1 << a.lp_log; off < 64; off <<= 1)
#pragma unroll
    for (int t = 0; t < RW; ++t)
#pragma unroll
      for (int k = 0; k < C; ++k) dq[t][k] += __shfl_xor(dq[t][k], off);
  if (slot == 0 && act)
#pragma unroll
    for (int t = 0; t < RW; ++t)
      if (t < rows) {
#pragma unroll
        for (int k = 0; k < C; ++k) dq[t][k] *= a.qscale;
        gst(a.dQp + (((size_t)jc * a.B + b) * n + i0 + t) * dx + c, dq[t]);
      }
}
// partial results in order: dQ over the key chunks, dK and dV over the row blocks
__global__ void __launch_bounds__(256) k_attn_head_fold(const float4* __restrict__ pQ, const float4* __restrict__ pK, const float4* __restrict__ pV,
                                                        float4* __restrict__ dQ, float4* __restrict__ dK, float4* __restrict__ dV, int njc, int nib,
                                                        long long quads) {
  const long long t = (long long)blockIdx.x * 256 + threadIdx.x;
  if (t >= quads) return;
  const int which = blockIdx.y + (njc > 1 ? 0 : 1);                     // what has one partial result is in place already
  const float4* src = which == 0 ? pQ : which == 1 ? pK : pV;
  const int G = which == 0 ? njc : nib;
  float4 s = {0.f, 0.f, 0.f, 0.f};
  for (int g = 0; g < G; g += 5) {                                        // five in flight, added in order
    float4 x[5];
#pragma unroll
    for (int u = 0; u < 5; ++u) x[u] = src[(size_t)min(g + u, G - 1) * quads + t];
#pragma unroll
    for (int u = 0; u < 5; ++u)
      if (g + u < G) { s.x += x[u].x; s.y += x[u].y; s.z += x[u].z; s.w += x[u].w; }
  }
  (which == 0 ? dQ : which == 1 ? dK : dV)[t] = s;
}

// ---------------------------------------------------------------------------------------------------------------------------------
// channels per lane and lanes per head; false: not built.  16 bytes of the pair tensors per lane (8 bf16, 4 fp32 channels) where a pair then fits
// 64 lanes and a head 16: fp32 B = 16, n = 140 backward + fold 263 us, with 8 channels 309 us
static bool head_shape(int dx, int H, bool bf16, int* C, int* hlog, int* lp_log) {
  if (dx < 4 || H < 1 || dx % H) return false;
  const int df = dx / H;
  *C = df == 4 || (!bf16 && dx <= 256 && df <= 64) ? 4 : 8;
  int l = 0;
  while ((*C << l) < df) ++l;
  if ((*C << l) != df || l > 4 || dx / *C > 64) return false;
  *hlog = l;
  int p = 0;
  while ((1 << p) < dx / *C) ++p;
  *lp_log = p;
  return true;
}
// backward: row blocks, and the keys cut into chunks so that the workgroups fill the 256 CUs in whole rounds.  One workgroup runs on a CU at a
// time (its registers); it takes its chunk's steps and HEAD_FIXED more for its beginning and end.
#define HEAD_FIXED 6
static void head_chunks(int B, int n, int C, int lp_log, bool bf16, int* nib, int* njc, int* jchunk) {
  const int NS = 64 >> lp_log, rows = HEAD_NW * head_rw(bf16, C);
  *nib = (n + rows - 1) / rows;
  long long best = -1;
  for (int want = 1; want <= 64 && (want == 1 || (want - 1) * 4 * NS < n); ++want) {
    const int ch = ((n + want - 1) / want + NS - 1) / NS * NS, nc = (n + ch - 1) / ch;
    const long long rounds = ((long long)B * *nib * nc + 255) / 256, cost = rounds * (ch / NS + HEAD_FIXED);
    if (best < 0 || cost < best) { best = cost; *jchunk = ch; *njc = nc; }
  }
}

// rows per workgroup: 2 share K_j and V_j (3 and 4 take registers that are waves: 194 against 199 and 213 us, 1 row 226 us, bf16 B = 8, n = 300)
// where that still gives 2 workgroups per CU, else 1
#define HEAD_WIDE 2
static int fwd_rows(int B, int n) { return (long long)B * ((n + HEAD_WIDE - 1) / HEAD_WIDE) >= 512 ? HEAD_WIDE : 1; }
// a launch has fewer than 2^32 threads
static bool fits_grid(long long groups, int threads) { return groups * threads < (1LL << 32); }

template <class TE, int C, int HLOG>
static void fwd_launch(const HeadArgs& a, bool save, bool mx8, hipStream_t s) {
  constexpr int WIDE = HEAD_WIDE;
  const int RW = fwd_rows(a.B, a.n);
  const bool wide = RW == WIDE;
  const long long grid = (long long)a.B * ((a.n + RW - 1) / RW);
  const size_t lds = sizeof(float) * 4 * RW * (a.dx + 2 * a.H);
#define F(R, S, M) k_attn_head_fwd<TE, C, HLOG, R, S, M><<<(unsigned)grid, 256, lds, s>>>(a)
  if (wide) { if (mx8) F(WIDE, true, true); else if (save) F(WIDE, true, false); else F(WIDE, false, false); }
  else { if (mx8) F(1, true, true); else if (save) F(1, true, false); else F(1, false, false); }
#undef F
}
template <class TY, int C, int HLOG>
static void bwd_launch(const HeadArgs& a, bool mx8, hipStream_t s) {
  const unsigned grid = (unsigned)((long long)a.B * a.nib * a.njc);
  const size_t lds = sizeof(float) * 2 * HEAD_NW * (64 >> a.lp_log) * 2 * a.dx;             // 64 KB at most
  if (mx8) k_attn_head_bwd<TY, C, HLOG, true><<<grid, 64 * HEAD_NW, lds, s>>>(a);
  else k_attn_head_bwd<TY, C, HLOG, false><<<grid, 64 * HEAD_NW, lds, s>>>(a);
}
// f(type, channels per lane, log2 of the lanes per head)
template <int C, int L> struct Shape { static constexpr int c = C, hlog = L; };
template <class F>
static void by_shape(bool bf16, int C, int hlog, F f) {
#define S(T, C, L) f((T*)nullptr, Shape<C, L>{})
  if (C == 4 && bf16) S(bf16_t, 4, 0);                                  // (4 channels per head)
  else if (C == 4) switch (hlog) { case 0: S(float, 4, 0); break; case 1: S(float, 4, 1); break; case 2: S(float, 4, 2); break; case 3: S(float, 4, 3); break; default: S(float, 4, 4); }
  else if (bf16) switch (hlog) { case 0: S(bf16_t, 8, 0); break; case 1: S(bf16_t, 8, 1); break; case 2: S(bf16_t, 8, 2); break; case 3: S(bf16_t, 8, 3); break; default: S(bf16_t, 8, 4); }
  else switch (hlog) { case 0: S(float, 8, 0); break; case 1: S(float, 8, 1); break; case 2: S(float, 8, 2); break; case 3: S(float, 8, 3); break; default: S(float, 8, 4); }
#undef S
}
static bool al16(std::initializer_list<const void*> ps) {
  uintptr_t v = 0;
  for (const void* p : ps) v |= (uintptr_t)p;
  return (v & 15) == 0;
}
// sizes both passes take: the descriptors' ranges and offsets are 32-bit (4 rows of a graph's pairs), the grid one-dimensional
static int head_sizes(const char* who, int B, int n, int dx, int H, bool bf16, int* C, int* hlog, int* lp_log) {
  DA_CHECK_ARG(B >= 0 && n >= 0 && dx >= 1 && H >= 1, "%s: B = %d, n = %d, dx = %d, n_head = %d", who, B, n, dx, H);
  if (!head_shape(dx, H, bf16, C, hlog, lp_log)) {
    da_set_error("%s: dx = %d with %d heads not built (channels per head 4, 8, 16, .. 128; dx <= 512, 256 with 4 channels per head)", who, dx, H);
    return DA_ERR_UNSUPPORTED;
  }
  DA_CHECK_ARG(4LL * n * dx * 4 < (1LL << 31) && 16LL * n * H < (1LL << 31) && (long long)B * n < (1LL << 31), "%s: B = %d, n = %d too large", who, B, n);
  return DA_OK;
}

extern "C" {

int da_attn_head_fwd(const float* Q, const float* K, const float* V, const void* E1, const void* E2, int e_bf16, const uint8_t* node_mask,
                     const int* groups, float qscale, float cap, void* Y, float* wV, float* S, float* stat, void* E1_codes, uint8_t* E1_scales, int B,
                     int n, int dx, int n_head, void* stream) {
  HeadArgs a = {};
  int C, hlog;
  if (int rc = head_sizes("da_attn_head_fwd", B, n, dx, n_head, e_bf16 != 0, &C, &hlog, &a.lp_log)) return rc;
  if (B == 0 || n == 0) return DA_OK;
  DA_CHECK_ARG(Q && K && V && E1 && E2 && node_mask && Y && wV, "da_attn_head_fwd: null pointer");
  const int RW = fwd_rows(B, n);
  DA_CHECK_ARG(fits_grid((long long)B * ((n + RW - 1) / RW), 256), "da_attn_head_fwd: B = %d, n = %d too large for one launch", B, n);
  DA_CHECK_ARG((S == nullptr) == (stat == nullptr) && (E1_codes == nullptr) == (E1_scales == nullptr) && (!E1_codes || S),
               "da_attn_head_fwd: S and stat go together, E1's codes and scales with both");
  DA_CHECK_ARG(!E1_codes || dx % MX8_GROUP == 0, "da_attn_head_fwd: 8-bit E1 needs dx %% 32 == 0, dx = %d", dx);
  DA_CHECK_ARG(cap == 0.f || (cap >= 1e-30f && cap <= 1e30f), "da_attn_head_fwd: cap = %g: 0 (none) or in [1e-30, 1e30]", cap);
  DA_CHECK_ARG(al16({Q, K, V, E1, E2, Y, wV, E1_codes}) && ((uintptr_t)stat & 7) == 0 && ((uintptr_t)S & 3) == 0, "da_attn_head_fwd: unaligned tensor (16 bytes)");
  a.Q = Q; a.K = K; a.V = V; a.E1 = E1; a.E2 = E2; a.nm = node_mask; a.grp = groups; a.qscale = qscale; a.cap = cap; a.n = n; a.dx = dx; a.H = n_head;
  a.Y = Y; a.wV = wV; a.S = S; a.stat = stat; a.q1 = (uint8_t*)E1_codes; a.q1s = E1_scales; a.B = B;
  by_shape(e_bf16 != 0, C, hlog, [&](auto* t, auto sh) {
    fwd_launch<std::remove_pointer_t<decltype(t)>, sh.c, sh.hlog>(a, S != nullptr, E1_codes != nullptr, (hipStream_t)stream);
  });
  DA_CHECK_LAUNCH("da_attn_head_fwd");
  return DA_OK;
}

long long da_attn_head_bwd_workspace(int B, int n, int dx, int n_head, int dy_bf16) {
  int C, hlog, lp, nib, njc, jchunk;
  if (B < 0 || n < 0 || !head_shape(dx, n_head, dy_bf16 != 0, &C, &hlog, &lp)) return -1;
  if (B == 0 || n == 0) return 0;
  head_chunks(B, n, C, lp, dy_bf16 != 0, &nib, &njc, &jchunk);
  return (long long)sizeof(float) * ((nib > 1 ? 2LL * nib : 0) + (njc > 1 ? njc : 0)) * B * n * dx;
}

int da_attn_head_bwd(const float* Q, const float* K, const float* V, const void* E1, const void* E1_codes, const uint8_t* E1_scales,
                     const uint8_t* node_mask, float qscale, float cap, const float* wV, const float* S, const float* stat, const void* dY,
                     int dy_bf16, const float* dwV, float* dQ, float* dK, float* dV, void* dE1, void* dE2, void* workspace,
                     long long workspace_bytes, int B, int n, int dx, int n_head, void* stream) {
  HeadArgs a = {};
  int C, hlog;
  if (int rc = head_sizes("da_attn_head_bwd", B, n, dx, n_head, dy_bf16 != 0, &C, &hlog, &a.lp_log)) return rc;
  if (B == 0 || n == 0) return DA_OK;
  DA_CHECK_ARG(Q && K && V && node_mask && wV && S && stat && dY && dwV && dQ && dK && dV && dE1 && dE2, "da_attn_head_bwd: null pointer");
  DA_CHECK_ARG((E1 != nullptr) != (E1_codes != nullptr) && (E1_codes == nullptr) == (E1_scales == nullptr),
               "da_attn_head_bwd: E1 either at full width or as codes and scales");
  DA_CHECK_ARG(!E1_codes || dx % MX8_GROUP == 0, "da_attn_head_bwd: 8-bit E1 needs dx %% 32 == 0, dx = %d", dx);
  DA_CHECK_ARG(cap == 0.f || (cap >= 1e-30f && cap <= 1e30f), "da_attn_head_bwd: cap = %g: 0 (none) or in [1e-30, 1e30]", cap);
  DA_CHECK_ARG(al16({Q, K, V, E1, E1_codes, wV, dY, dwV, dQ, dK, dV, dE1, dE2, workspace}) && ((uintptr_t)stat & 7) == 0 && ((uintptr_t)S & 3) == 0,
               "da_attn_head_bwd: unaligned tensor (16 bytes)");
  const long long need = da_attn_head_bwd_workspace(B, n, dx, n_head, dy_bf16);
  DA_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need), "da_attn_head_bwd: workspace too small");
  a.Q = Q; a.K = K; a.V = V; a.E1 = E1_codes ? E1_codes : E1; a.E1s = E1_scales; a.nm = node_mask; a.qscale = qscale; a.cap = cap; a.n = n; a.dx = dx;
  a.H = n_head; a.wV = (float*)wV; a.S = (float*)S; a.stat = (float*)stat; a.dY = dY; a.dwV = dwV; a.dE1 = dE1; a.dE2 = dE2; a.B = B;
  head_chunks(B, n, C, a.lp_log, dy_bf16 != 0, &a.nib, &a.njc, &a.jchunk);
  DA_CHECK_ARG(fits_grid((long long)B * a.nib * a.njc, 64 * HEAD_NW), "da_attn_head_bwd: B = %d, n = %d too large for one launch", B, n);
  const size_t one = (size_t)B * n * dx;
  float* ws = (float*)workspace;
  a.dKp = dK; a.dVp = dV; a.dQp = dQ;
  if (a.nib > 1) { a.dKp = ws; a.dVp = ws + a.nib * one; ws += 2 * a.nib * one; }
  if (a.njc > 1) a.dQp = ws;
  hipStream_t s = (hipStream_t)stream;
  by_shape(dy_bf16 != 0, C, hlog, [&](auto* t, auto sh) { bwd_launch<std::remove_pointer_t<decltype(t)>, sh.c, sh.hlog>(a, E1_codes != nullptr, s); });
  if (a.nib > 1 || a.njc > 1) {
    const long long quads = (long long)one / 4;
    const unsigned gx = (unsigned)((quads + 255) / 256);
    k_attn_head_fold<<<dim3(gx, (a.njc > 1 ? 1 : 0) + (a.nib > 1 ? 2 : 0)), 256, 0, s>>>((const float4*)a.dQp, (const float4*)a.dKp, (const float4*)a.dVp, (float4*)dQ, (float4*)dK,
                                                                 (float4*)dV, a.njc, a.nib, quads);
  }
  DA_CHECK_LAUNCH("da_attn_head_bwd");
  return DA_OK;
}

}  // extern "C"
