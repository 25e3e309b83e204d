// vmscan_cached.cuh — the selective scan and the causal conv1d + SiLU over a
// cache of request states, for packed prompts and single tokens.
//
// The reference has no cached or ragged form; the recurrence is its
// selective_scan (mlx_vision_mamba/mamba_block.py:45-73, gate :190) and the
// conv its conv1d + SiLU (:129-132,170-171), started from a stored state:
//   h_t[n] = exp(delta_t A[d, n]) h_{t-1}[n] + delta_t u_t B_t[n]
//   y_t    = (sum_n C_t[n] h_t[n] + D[d] u_t) * silu(z_t)
//   out_t  = silu(bias + sum_k w[c, k] x_{t-K+1+k})
// with h_{-1} and the K - 1 rows before the first one read from the request's
// source slot (zeros for a fresh request) and the last ones written to its
// slot.
//
// Requests are packed row after row.  The host cuts them into pieces (int32[8]
// records, PieceField below) of consecutive rows of one request; a request of
// no rows is one empty piece, which only carries its state over.
#pragma once

#include "vmscan_common.cuh"

namespace vmscan {

// One piece: rows [T0, T1) of the request that owns rows [BEGIN, END).
// SOURCE: slot its state is read from (-1: zeros), SLOT: slot written (-1: a
// padding request, whose rows are set to zero).  CARRY: row of the carry
// arrays when the request is scanned in several pieces, else -1.
enum PieceField { PF_T0, PF_T1, PF_BEGIN, PF_END, PF_SOURCE, PF_SLOT, PF_CARRY, PF_PAD, PF_COUNT };

struct Piece {
  int t0, t1, begin, end, source, slot, carry;
};

// Reads a piece and keeps it inside the arrays whatever the table holds: rows
// inside [0, rows), a slot or source outside the cache is no slot.
__device__ __forceinline__ Piece load_piece(const int32_t* __restrict__ pieces, int64_t i, int rows, int64_t n_slots) {
  const int4 a = reinterpret_cast<const int4*>(pieces)[2 * i];
  const int4 b = reinterpret_cast<const int4*>(pieces)[2 * i + 1];
  Piece p;
  p.begin = min(max(a.z, 0), rows);
  p.end = min(max(a.w, p.begin), rows);
  p.t0 = min(max(a.x, p.begin), p.end);
  p.t1 = min(max(a.y, p.t0), p.end);
  p.source = b.x < n_slots ? b.x : -1;
  p.slot = b.y < n_slots ? b.y : -1;
  p.carry = b.z;
  return p;
}

template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);  // the output's one rounding (half a bf16 step)
}

struct CachedScanArgs {
  const void* u;
  const void* delta;
  const void* B;
  const void* C;
  const void* z;
  void* y;
  const float* A;
  const float* D;
  float* state;
  int64_t ldu, ldd, ldb, ldc, ldz, ldy;  // row strides in elements
  int64_t n_slots;
  int rows, dn;
};

// ---------------------------------------------------------------------------
// Prompts: a warp owns 32 channels of one piece, a lane one channel and its 16
// states.  B and C of CSC_ROWS rows are staged in the warp's shared memory.
// CARRY: only the state at the piece's end from a zero state and the sum of
// delta (the piece maps h to exp(A sum delta) h + carry_h).
// ---------------------------------------------------------------------------
constexpr int CSC_WARPS = 4;
constexpr int CSC_ROWS = 8;

template <typename T, bool HAS_Z, bool CARRY>
__global__ void __launch_bounds__(CSC_WARPS * 32)
    cached_scan_kernel(const CachedScanArgs a, const int32_t* __restrict__ pieces, int groups,
                       const float* __restrict__ h_start, float* __restrict__ carry_h, float* __restrict__ carry_s) {
  __shared__ float bc[CSC_WARPS][CSC_ROWS][2 * NS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Piece p = load_piece(pieces, blockIdx.x / groups, a.rows, a.n_slots);
  const int d = ((blockIdx.x % groups) * CSC_WARPS + warp) * 32 + lane;
  if (d - lane >= a.dn) return;  // whole warps only: the rest of the kernel shuffles and syncs by warp
  const bool ok = d < a.dn;
  const int dc = ok ? d : a.dn - 1;
  const T* __restrict__ u = static_cast<const T*>(a.u) + dc;
  const T* __restrict__ dl = static_cast<const T*>(a.delta) + dc;
  const T* __restrict__ z = static_cast<const T*>(a.z) + (HAS_Z ? dc : 0);
  T* __restrict__ y = static_cast<T*>(a.y) + dc;
  if (p.slot < 0) {  // padding request
    if (!CARRY && ok)
      for (int t = p.t0; t < p.t1; ++t) y[t * a.ldy] = from_f<T>(0.f);
    return;
  }
  float2 A2[8], h[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float4 v = *reinterpret_cast<const float4*>(a.A + int64_t(dc) * NS + 4 * j);
    A2[2 * j] = make_float2(v.x, v.y);
    A2[2 * j + 1] = make_float2(v.z, v.w);
  }
  const float* src = nullptr;
  if (!CARRY) {
    if (p.carry >= 0)  // also for a first piece: another piece may write the source's slot meanwhile
      src = h_start + (int64_t(p.carry) * a.dn + dc) * NS;
    else if (p.source >= 0)
      src = a.state + (int64_t(p.source) * a.dn + dc) * NS;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float4 v = src != nullptr ? *reinterpret_cast<const float4*>(src + 4 * j) : make_float4(0.f, 0.f, 0.f, 0.f);
    h[2 * j] = make_float2(v.x, v.y);
    h[2 * j + 1] = make_float2(v.z, v.w);
  }
  const float Dd = a.D[dc];
  float dsum = 0.f;
  const int brow = lane >> 2, bcol = (lane & 3) * 4;  // B / C values this lane stages
  for (int t0 = p.t0; t0 < p.t1; t0 += CSC_ROWS) {
    const int nr = min(CSC_ROWS, p.t1 - t0);
    float uv[CSC_ROWS], dv[CSC_ROWS], zv[CSC_ROWS];
#pragma unroll
    for (int r = 0; r < CSC_ROWS; ++r) {
      const int64_t t = min(t0 + r, p.t1 - 1);
      uv[r] = ld_one(u + t * a.ldu);
      dv[r] = ld_one(dl + t * a.ldd);
      if (HAS_Z && !CARRY) zv[r] = ld_one(z + t * a.ldz);
    }
    __syncwarp();
    if (brow < nr) {
      const T* pb = static_cast<const T*>(a.B) + (t0 + brow) * a.ldb + bcol;
      const T* pc = static_cast<const T*>(a.C) + (t0 + brow) * a.ldc + bcol;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        bc[warp][brow][bcol + k] = ld_one(pb + k);
        if (!CARRY) bc[warp][brow][NS + bcol + k] = ld_one(pc + k);
      }
    }
    __syncwarp();
#pragma unroll
    for (int r = 0; r < CSC_ROWS; ++r) {
      if (r < nr) {
        const float2 du = bcast2(dv[r] * uv[r]), dlog = bcast2(dv[r] * kLog2e), off = bcast2(kEx2ArgBias);
        if (CARRY) dsum += dv[r];
        float2 acc0 = make_float2(0.f, 0.f), acc1 = make_float2(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float2 arg = fma2(dlog, A2[j], off);
          const float2 e = make_float2(ex2_approx(arg.x), ex2_approx(arg.y));
          h[j] = fma2(e, h[j], mul2(du, lds2(&bc[warp][r][2 * j])));
          if (!CARRY) {
            const float2 c2 = lds2(&bc[warp][r][NS + 2 * j]);
            if (j & 1)
              acc1 = fma2(c2, h[j], acc1);
            else
              acc0 = fma2(c2, h[j], acc0);
          }
        }
        if (!CARRY) {
          const float2 acc = add2(acc0, acc1);
          float yy = fmaf(uv[r], Dd, acc.x + acc.y);
          if (HAS_Z) yy *= silu_f(zv[r]);
          if (ok) y[(t0 + r) * a.ldy] = from_f<T>(yy);
        }
      }
    }
  }
  if (!ok) return;
  float* dst = nullptr;
  if (CARRY) {
    dst = carry_h + (int64_t(p.carry) * a.dn + d) * NS;
    carry_s[int64_t(p.carry) * a.dn + d] = dsum;
  } else if (p.t1 == p.end) {
    dst = a.state + (int64_t(p.slot) * a.dn + d) * NS;
  }
  if (dst != nullptr) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<float4*>(dst + 4 * j) = make_float4(h[2 * j].x, h[2 * j].y, h[2 * j + 1].x, h[2 * j + 1].y);
  }
}

// State entering every piece of the split requests: chain i =
// {first carry row, pieces, source slot, 0}; one thread per (chain, channel,
// state) walks the pieces' maps.
__global__ void cached_chain_kernel(const int32_t* __restrict__ chains, const float* __restrict__ A,
                                    const float* __restrict__ state, int64_t n_slots,
                                    const float* __restrict__ carry_h, const float* __restrict__ carry_s,
                                    float* __restrict__ h_start, int dn) {
  const int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= int64_t(dn) * NS) return;
  const int4 c = reinterpret_cast<const int4*>(chains)[blockIdx.y];
  const float An = A[i];
  float h = c.z >= 0 && c.z < n_slots ? state[int64_t(c.z) * dn * NS + i] : 0.f;
  h_start[int64_t(c.x) * dn * NS + i] = h;
  for (int k = 0; k + 1 < c.y; ++k) {
    const int64_t row = c.x + k;
    h = fmaf(expf(An * carry_s[row * dn + i / NS]), h, carry_h[row * dn * NS + i]);
    h_start[(row + 1) * dn * NS + i] = h;
  }
}

// ---------------------------------------------------------------------------
// Single tokens: row i is request i.  A warp owns 32 channels of one row; four
// lanes share a channel (four states each), so the state moves as whole
// 512-byte warp accesses.
// ---------------------------------------------------------------------------
constexpr int CST_WARPS = 4;

template <typename T, bool HAS_Z>
__global__ void __launch_bounds__(CST_WARPS * 32)
    cached_step_kernel(const CachedScanArgs a, const int32_t* __restrict__ slots, const int32_t* __restrict__ sources,
                       int groups) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = blockIdx.x / groups;
  const int d0 = ((blockIdx.x % groups) * CST_WARPS + warp) * 32;
  if (d0 >= a.dn) return;
  const int d = d0 + lane;
  const bool ok = d < a.dn;
  const int slot = slots[row], source = sources[row];
  T* __restrict__ y = static_cast<T*>(a.y) + row * a.ldy;
  if (slot < 0 || slot >= a.n_slots) {
    if (ok) y[d] = from_f<T>(0.f);
    return;
  }
  const int dc = ok ? d : a.dn - 1;
  const float u = ld_one(static_cast<const T*>(a.u) + row * a.ldu + dc);
  const float dl = ld_one(static_cast<const T*>(a.delta) + row * a.ldd + dc);
  const float z = HAS_Z ? ld_one(static_cast<const T*>(a.z) + row * a.ldz + dc) : 0.f;
  const float Dd = a.D[dc];
  const int q = lane & 3;
  float Bq[4], Cq[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    Bq[k] = ld_one(static_cast<const T*>(a.B) + row * a.ldb + 4 * q + k);
    Cq[k] = ld_one(static_cast<const T*>(a.C) + row * a.ldc + 4 * q + k);
  }
  const bool kept = source >= 0 && source < a.n_slots;
  float mine = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int k = 8 * i + (lane >> 2);  // channel of this round, in the warp's 32
    const int c = d0 + k;
    const bool in = c < a.dn;
    const float du = __shfl_sync(0xffffffffu, dl * u, k);
    const float dlog = __shfl_sync(0xffffffffu, dl * kLog2e, k);
    float part = 0.f;
    if (in) {
      const float4 A4 = *reinterpret_cast<const float4*>(a.A + int64_t(c) * NS + 4 * q);
      float4 h = make_float4(0.f, 0.f, 0.f, 0.f);
      if (kept) h = *reinterpret_cast<const float4*>(a.state + (int64_t(source) * a.dn + c) * NS + 4 * q);
      h.x = fmaf(ex2_approx(fmaf(dlog, A4.x, kEx2ArgBias)), h.x, du * Bq[0]);
      h.y = fmaf(ex2_approx(fmaf(dlog, A4.y, kEx2ArgBias)), h.y, du * Bq[1]);
      h.z = fmaf(ex2_approx(fmaf(dlog, A4.z, kEx2ArgBias)), h.z, du * Bq[2]);
      h.w = fmaf(ex2_approx(fmaf(dlog, A4.w, kEx2ArgBias)), h.w, du * Bq[3]);
      part = fmaf(Cq[1], h.y, Cq[0] * h.x) + fmaf(Cq[3], h.w, Cq[2] * h.z);
      *reinterpret_cast<float4*>(a.state + (int64_t(slot) * a.dn + c) * NS + 4 * q) = h;
    }
    part += __shfl_xor_sync(0xffffffffu, part, 1);
    part += __shfl_xor_sync(0xffffffffu, part, 2);
    // lane l owns channel l of the warp: round l / 8, lane group l % 8
    const float got = __shfl_sync(0xffffffffu, part, 4 * (lane & 7));
    if ((lane >> 3) == i) mine = got;
  }
  float yy = fmaf(u, Dd, mine);
  if (HAS_Z) yy *= silu_f(z);
  if (ok) y[d] = from_f<T>(yy);
}

// ---------------------------------------------------------------------------
// Causal conv1d + SiLU.  A thread owns VEC adjacent channels of one piece and
// slides the K-row window along its rows.  The first piece of a request (and
// the only one that can reach rows before it: pieces hold CCV_ROWS >= K - 1
// rows) reads the stored window, and writes the new one: the request's last
// K - 1 rows, reaching back into the old window when it has fewer.  The same
// thread reads the old window before it writes, so a slot may be both.
// ---------------------------------------------------------------------------
constexpr int CCV_ROWS = 32;
constexpr int CCV_THREADS = 64;
constexpr int CCV_KMAX = 8;

template <typename T, int VEC>
__device__ __forceinline__ void ldv(const T* p, float v[VEC]) {
  if constexpr (VEC == 1) {
    v[0] = ld_one(p);
  } else if constexpr (sizeof(T) == 4) {
    const float4 q = *reinterpret_cast<const float4*>(p);
    v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
  } else {
    const uint2 q = *reinterpret_cast<const uint2*>(p);
    const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&q.x));
    const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&q.y));
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
  }
}

template <typename T, int VEC>
__device__ __forceinline__ void stv(T* p, const float v[VEC]) {
  if constexpr (VEC == 1) {
    *p = from_f<T>(v[0]);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    uint2 q;
    *reinterpret_cast<__nv_bfloat162*>(&q.x) = __floats2bfloat162_rn(v[0], v[1]);
    *reinterpret_cast<__nv_bfloat162*>(&q.y) = __floats2bfloat162_rn(v[2], v[3]);
    *reinterpret_cast<uint2*>(p) = q;
  }
}

struct CachedConvArgs {
  const void* x;
  void* out;
  void* state;  // (n_slots, K - 1, channels), oldest row first
  const float* w;
  const float* bias;
  int64_t ldx, ldo, n_slots;
  int rows, channels, K;
};

template <typename T, int VEC>
__global__ void __launch_bounds__(CCV_THREADS)
    cached_conv_kernel(const CachedConvArgs a, const int32_t* __restrict__ pieces, int groups) {
  const Piece p = load_piece(pieces, blockIdx.x / groups, a.rows, a.n_slots);
  const int c = ((blockIdx.x % groups) * CCV_THREADS + threadIdx.x) * VEC;
  if (c >= a.channels) return;
  const int K = a.K;
  T* out = static_cast<T*>(a.out) + c;
  if (p.slot < 0) {
    const float zero[VEC] = {};
    for (int t = p.t0; t < p.t1; ++t) stv<T, VEC>(out + t * a.ldo, zero);
    return;
  }
  const T* x = static_cast<const T*>(a.x) + c;
  T* state = static_cast<T*>(a.state) + c;
  const int64_t C = a.channels;
  float w[CCV_KMAX][VEC], win[CCV_KMAX][VEC], bias[VEC];
#pragma unroll
  for (int m = 0; m < CCV_KMAX; ++m) {
    const int k = m - (CCV_KMAX - K);  // tap of window slot m: the K taps sit at the newest end
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      w[m][v] = k >= 0 ? a.w[int64_t(c + v) * K + k] : 0.f;
      win[m][v] = 0.f;
    }
  }
#pragma unroll
  for (int v = 0; v < VEC; ++v) bias[v] = a.bias[c + v];
  // rows before the piece: rows of the request, or of the stored window
#pragma unroll
  for (int m = 1; m < CCV_KMAX; ++m) {
    const int t = p.t0 - (CCV_KMAX - m);  // row of window slot m before the first shift
    if (CCV_KMAX - m < K) {
      if (t >= p.begin)
        ldv<T, VEC>(x + t * a.ldx, win[m]);
      else if (p.source >= 0)
        ldv<T, VEC>(state + (int64_t(p.source) * (K - 1) + (K - 1 - (p.begin - t))) * C, win[m]);
    }
  }
  if (p.t0 == p.begin) {
    // the new window: its row j is row end - (K - 1) + j of the request, and
    // where that lies before the request, the old window's row j + length
    // (read above: slot m of win is row begin - (CCV_KMAX - m))
    const int len = p.end - p.begin;
#pragma unroll
    for (int m = 1; m < CCV_KMAX; ++m) {
      const int j = K - 1 - (CCV_KMAX - m);
      if (j >= 0) {
        float v[VEC] = {};
        const int t = p.end - (CCV_KMAX - m);
        if (t >= p.begin) {
          ldv<T, VEC>(x + t * a.ldx, v);
        } else {
#pragma unroll
          for (int s = 1; s < CCV_KMAX; ++s)
            if (s == m + len)
#pragma unroll
              for (int q = 0; q < VEC; ++q) v[q] = win[s][q];
        }
        stv<T, VEC>(state + (int64_t(p.slot) * (K - 1) + j) * C, v);
      }
    }
  }
  for (int t = p.t0; t < p.t1; ++t) {
#pragma unroll
    for (int m = 0; m < CCV_KMAX - 1; ++m)
#pragma unroll
      for (int v = 0; v < VEC; ++v) win[m][v] = win[m + 1][v];
    ldv<T, VEC>(x + t * a.ldx, win[CCV_KMAX - 1]);
    float acc[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      acc[v] = bias[v];
#pragma unroll
      for (int m = 0; m < CCV_KMAX; ++m) acc[v] = fmaf(w[m][v], win[m][v], acc[v]);
      acc[v] = silu_f(acc[v]);
    }
    stv<T, VEC>(out + t * a.ldo, acc);
  }
}

}  // namespace vmscan
