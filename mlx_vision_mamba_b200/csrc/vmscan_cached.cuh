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
// arrays when the request is scanned in several pieces, else -1; ORDINAL: the
// piece's place among them (their carry rows are consecutive).
enum PieceField { PF_T0, PF_T1, PF_BEGIN, PF_END, PF_SOURCE, PF_SLOT, PF_CARRY, PF_ORDINAL, PF_COUNT };

struct Piece {
  int t0, t1, begin, end, source, slot, carry, ordinal;
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
  p.ordinal = b.w;
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

// The launches of a small split scan overlap: a kernel lets the next one's CTAs
// start while it runs (`launch_next`), and that one waits for all of it to be
// done and visible (`wait_previous`) before it touches what they share.  Every
// CTA of such a kernel waits, so that the end of the last one is the end of
// all.  In a launch that does not overlap both do nothing.  What the launch
// before writes (states, carries) is read through plain pointers only: a
// `const __restrict__` parameter says that nobody writes the data while the
// kernel runs, and its loads need not stay behind wait_previous.
__device__ __forceinline__ void launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

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

// Four adjacent elements as fp32; `wide`: the address takes one access.
template <typename T>
__device__ __forceinline__ float4 ld_four(const T* p, bool wide) {
  if (!wide) return make_float4(ld_one(p), ld_one(p + 1), ld_one(p + 2), ld_one(p + 3));
  if constexpr (sizeof(T) == 4) {
    return __ldg(reinterpret_cast<const float4*>(p));
  } else {
    const uint2 q = __ldg(reinterpret_cast<const uint2*>(p));
    const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&q.x));
    const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&q.y));
    return make_float4(a.x, a.y, b.x, b.y);
  }
}

// ---------------------------------------------------------------------------
// Prompts: a warp owns 32 channels of one piece.  A lane pair owns two adjacent
// channels and each lane 8 of the 16 states of both, so a B / C value read from
// shared memory serves two channels.  The rows travel through a ring of
// CSC_STAGES blocks of CSC_ROWS rows in the warp's own shared memory, filled by
// asynchronous copies: a warp needs no other warp and no barrier, and one warp
// alone on its scheduler still has two blocks in flight.
// G: bytes of one copy, the widest that the rows' alignment allows
// (cached_scan_grain): 16, 4 (two bf16 or one fp32) or 2 (odd bf16 rows: plain
// loads, kept in registers while the block before is computed).  bc_grain: the
// same for B and C.
// A request that would keep a few warps busy long after the others is split
// into pieces.  CARRY: a piece whose start is not known yet only yields its
// map h -> exp(A sum delta) h + (its end state from zero).
//
// Bound: the exponential unit.  A row of 32 channels is 512 decays, the gate's
// exponential and reciprocal: 18 warp instructions of 8 cycles on that unit,
// 144 cycles a scheduler, against 88 cycles of HBM traffic for fp32 at full
// rate over all SMs and about 92 instructions to issue.  Measured on B200: 180
// cycles with four warps a scheduler (64 requests of 512 rows x 1536, fp32,
// gated: 277 us, 2.9e12 decays/s), 250 with one; the unit is busy 79 % of the
// time in the first phase of 32 uneven prompts, 71 % in the second.  Of what
// that took: rows through the ring instead of one register block ahead, an
// explicit global store (338 -> 316 us on those 64 requests, with the decays
// computed one row ahead), A in exponent units (-5 %).  Tried and slower:
// part of the decays by a polynomial on the FMA pipe (one of eight pairs:
// within 3 %, two: +9 %), one channel and 16 states a lane (fp32 +3 to 5 %),
// five CTAs an SM.
// Whole calls: 32 prompts of 32768 rows x 1536, bf16: 358 us; one prompt of
// 32768 x 768 fp32: 255 us (in 96 pieces; 4.3 ms in one); 24 requests, 9001
// rows x 768, fp32: 75 us (1.8x rows from splitting, and single tokens are pieces
// of this kernel); 196 rows x 768: 11.5 us (three dependent launches; pieces that
// pass their states on inside a cluster, in one launch, are not built).
// ---------------------------------------------------------------------------
constexpr int CSC_WARPS = 4;
constexpr int CSC_ROWS = 8;
constexpr int CSC_STAGES = 3;

template <int BYTES>
__device__ __forceinline__ void cp_async(void* dst, const void* src) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(dst)), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// First column (of 32) that a lane copies, and the copies of CSC_ROWS rows
// into dst[row][32].  p: that column of row 0; rows past `last` repeat it.
template <typename T, int G>
__device__ __forceinline__ int copy_col(int lane) {
  constexpr int E = G / int(sizeof(T));
  return lane % (32 / E) * E;
}
template <typename T, int G>
__device__ __forceinline__ void copy_rows(T* dst, const T* p, int64_t ld, int t0, int last, int lane) {
  constexpr int E = G / int(sizeof(T)), LPR = 32 / E;  // E rows at a time
  static_assert(CSC_ROWS % E == 0, "a copy must not reach past the block's rows");
  dst += lane / LPR * 32 + lane % LPR * E;
  if (t0 + CSC_ROWS - 1 <= last) {
    const T* q = p + (t0 + lane / LPR) * ld;
#pragma unroll
    for (int r0 = 0; r0 < CSC_ROWS; r0 += E) cp_async<G>(dst + r0 * 32, q + r0 * ld);
  } else {
#pragma unroll
    for (int r0 = 0; r0 < CSC_ROWS; r0 += E) cp_async<G>(dst + r0 * 32, p + min(t0 + r0 + lane / LPR, last) * ld);
  }
}

// One stage of a warp's ring.
template <typename T>
struct ScanStage {
  T u[CSC_ROWS][32], dl[CSC_ROWS][32], z[CSC_ROWS][32], bc[CSC_ROWS][32];
};
template <typename T>
struct ScanRing {
  ScanStage<T> st[CSC_STAGES];
  float wide[sizeof(T) == 4 ? 1 : CSC_ROWS][32];  // bf16: the block's B | C as fp32
};
template <typename T>
constexpr size_t cached_scan_smem() {
  return sizeof(ScanRing<T>) * CSC_WARPS;
}

// Where the pieces of split requests leave and find their states.
struct ScanCarries {
  float* h;             // (carry rows, dn, 16): state at a piece's end (a first piece: the true one; later: from zero)
  float* sum;           // (carry rows, dn): sum of delta over a later piece
  const float* start;   // (carry rows, dn, 16): state entering a later piece, or NULL: chained here
  int rows;             // carry rows
};

// A later piece's map: half^2 h + local, half = exp(A sum delta / 2).  With
// A > 0 the factor may leave fp32's range where the state does not (it is tiny,
// or still zero); in halves it does so only with the state itself.
__device__ __forceinline__ float apply_map(float half, float h, float local) {
  return h == 0.f ? local : fmaf(half, half * h, local);
}

template <typename T, int G, bool HAS_Z, bool CARRY>
__device__ __forceinline__ void cached_scan_piece(const CachedScanArgs& a, const Piece& p, int group, int bc_grain,
                                                  bool later, const ScanCarries& k, unsigned char* smem_raw) {
  constexpr bool LOAD_Z = HAS_Z && !CARRY;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  ScanRing<T>& ring = reinterpret_cast<ScanRing<T>*>(smem_raw)[warp];
  const int d0 = (group * CSC_WARPS + warp) * 32;
  if (later && (d0 >= a.dn || p.slot < 0)) wait_previous();
  if (d0 >= a.dn) return;  // whole warps: the rest shuffles and syncs by warp only
  const int hb = lane & 1, pc = lane & ~1;
  const int own = d0 + lane, dp = d0 + pc;
  const bool ok = own < a.dn;
  T* __restrict__ y = static_cast<T*>(a.y) + min(own, a.dn - 1);
  if (p.slot < 0) {  // padding request
    if (!CARRY && ok)
      for (int t = p.t0; t < p.t1; ++t) y[t * a.ldy] = from_f<T>(0.f);
    return;
  }
  // what this lane copies: columns past the last channel repeat the last ones
  const int last = p.t1 - 1;
  constexpr int E = G / int(sizeof(T));
  const int col = min(d0 + copy_col<T, G>(lane), a.dn - E);
  const T* __restrict__ pu = static_cast<const T*>(a.u) + col;
  const T* __restrict__ pd = static_cast<const T*>(a.delta) + col;
  const T* __restrict__ pz = static_cast<const T*>(a.z) + (LOAD_Z ? col : 0);
  const int bcol = bc_grain == 16 ? copy_col<T, 16>(lane) : bc_grain == 4 ? copy_col<T, 4>(lane) : lane;
  const bool is_b = bcol < NS;
  const T* __restrict__ pbc = is_b ? static_cast<const T*>(a.B) + bcol : static_cast<const T*>(a.C) + bcol - NS;
  const int64_t ldbc = is_b ? a.ldb : a.ldc;
  T ru[G == 2 ? CSC_ROWS : 1], rd[G == 2 ? CSC_ROWS : 1], rz[G == 2 ? CSC_ROWS : 1], rbc[sizeof(T) == 2 ? CSC_ROWS : 1];

  auto issue = [&](int t0, ScanStage<T>& st) {
    if (t0 < p.t1) {
      if constexpr (G == 2) {
#pragma unroll
        for (int r = 0; r < CSC_ROWS; ++r) {
          const int64_t t = min(t0 + r, last);
          ru[r] = pu[t * a.ldu];
          rd[r] = pd[t * a.ldd];
          if (LOAD_Z) rz[r] = pz[t * a.ldz];
        }
      } else {
        copy_rows<T, G>(&st.u[0][0], pu, a.ldu, t0, last, lane);
        copy_rows<T, G>(&st.dl[0][0], pd, a.ldd, t0, last, lane);
        if (LOAD_Z) copy_rows<T, G>(&st.z[0][0], pz, a.ldz, t0, last, lane);
      }
      if (!CARRY || is_b) {
        if (bc_grain == 16) {
          copy_rows<T, 16>(&st.bc[0][0], pbc, ldbc, t0, last, lane);
        } else if (bc_grain == 4) {
          copy_rows<T, 4>(&st.bc[0][0], pbc, ldbc, t0, last, lane);
        } else if constexpr (sizeof(T) == 2) {
#pragma unroll
          for (int r = 0; r < CSC_ROWS; ++r) rbc[r] = pbc[min(t0 + r, last) * ldbc];
        }
      }
    }
    cp_async_commit();
  };
  // what `issue` left in registers, into its stage
  auto settle = [&](int t0, ScanStage<T>& st) {
    if (t0 >= p.t1) return;
    if constexpr (G == 2) {
#pragma unroll
      for (int r = 0; r < CSC_ROWS; ++r) {
        st.u[r][lane] = ru[r];
        st.dl[r][lane] = rd[r];
        if (LOAD_Z) st.z[r][lane] = rz[r];
      }
    }
    if constexpr (sizeof(T) == 2) {
      if (bc_grain == 2 && (!CARRY || is_b)) {
#pragma unroll
        for (int r = 0; r < CSC_ROWS; ++r) st.bc[r][lane] = rbc[r];
      }
    }
  };
#pragma unroll
  for (int k = 0; k < CSC_STAGES - 1; ++k) {
    issue(p.t0 + k * CSC_ROWS, ring.st[k]);
    settle(p.t0 + k * CSC_ROWS, ring.st[k]);
  }

  if (later) wait_previous();  // the rows are on their way; states and carries from here on
  float2 A2[2][4], h[2][4];
  const float* src = nullptr;
  if (!CARRY) {
    if (p.carry < 0 || p.ordinal == 0)
      src = p.source >= 0 ? a.state + int64_t(p.source) * a.dn * NS : nullptr;
    else
      src = k.start != nullptr ? k.start + int64_t(p.carry) * a.dn * NS : k.h + int64_t(p.carry - p.ordinal) * a.dn * NS;
  }
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int64_t off = int64_t(min(dp + c, a.dn - 1)) * NS + 8 * hb;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float4 v = *reinterpret_cast<const float4*>(a.A + off + 4 * j);
      A2[c][2 * j] = make_float2(v.x * kLog2e, v.y * kLog2e);
      A2[c][2 * j + 1] = make_float2(v.z * kLog2e, v.w * kLog2e);
      const float4 g = src != nullptr ? *reinterpret_cast<const float4*>(src + off + 4 * j) : make_float4(0.f, 0.f, 0.f, 0.f);
      h[c][2 * j] = make_float2(g.x, g.y);
      h[c][2 * j + 1] = make_float2(g.z, g.w);
    }
  }
  if (!CARRY && p.carry >= 0 && k.start == nullptr) {
    // the maps of the later pieces before this one, onto the first piece's end
    for (int i = 1; i < p.ordinal; ++i) {
      const int64_t at = int64_t(p.carry - p.ordinal + i) * a.dn;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int64_t ch = at + min(dp + c, a.dn - 1);
        const float sum = k.sum[ch];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 g = *reinterpret_cast<const float2*>(k.h + ch * NS + 8 * hb + 2 * j);
          h[c][j].x = apply_map(exp2f(0.5f * (A2[c][j].x * sum)), h[c][j].x, g.x);
          h[c][j].y = apply_map(exp2f(0.5f * (A2[c][j].y * sum)), h[c][j].y, g.y);
        }
      }
    }
  }
  const float Dd = a.D[min(own, a.dn - 1)];
  float2 dsum = make_float2(0.f, 0.f);

  int stage = 0;
  for (int t0 = p.t0; t0 < p.t1; t0 += CSC_ROWS) {
    cp_async_wait<CSC_STAGES - 2>();
    __syncwarp();  // this block has arrived for every lane, and every lane has left the one before
    const ScanStage<T>& st = ring.st[stage];
    const float* bc;
    if constexpr (sizeof(T) == 4) {
      bc = &st.bc[0][0];
    } else {
      const uint4 q = *reinterpret_cast<const uint4*>(&st.bc[lane >> 2][(lane & 3) * 8]);
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
      float2 f[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) f[k] = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[k]));
      float* o = &ring.wide[lane >> 2][(lane & 3) * 8];
      *reinterpret_cast<float4*>(o) = make_float4(f[0].x, f[0].y, f[1].x, f[1].y);
      *reinterpret_cast<float4*>(o + 4) = make_float4(f[2].x, f[2].y, f[3].x, f[3].y);
      __syncwarp();
      bc = &ring.wide[0][0];
    }
    const int ahead = t0 + (CSC_STAGES - 1) * CSC_ROWS;
    ScanStage<T>& free_stage = ring.st[stage == 0 ? CSC_STAGES - 1 : stage - 1];
    issue(ahead, free_stage);
    // decays of a row; computed one row ahead of their use, so that the exp
    // unit works while the row before is summed
    struct Decay {
      float2 e[2][4];
      float2 u, d;
    };
    auto decay = [&](int r, Decay& w) {
      w.u = ld_pair(&st.u[r][pc]);
      w.d = ld_pair(&st.dl[r][pc]);
      const float2 off = bcast2(kEx2ArgBias);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float2 dg = bcast2(c ? w.d.y : w.d.x);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 arg = fma2(dg, A2[c][j], off);
          w.e[c][j] = make_float2(ex2_approx(arg.x), ex2_approx(arg.y));
        }
      }
    };
    auto row = [&](int r, const Decay& w) {
      const float2 du = mul2(w.d, w.u);
      if (CARRY) dsum = add2(dsum, w.d);
      const float* s = bc + r * 32 + 8 * hb;
      const float4 b0 = lds4(s), b1 = lds4(s + 4);
      const float2 B2[4] = {make_float2(b0.x, b0.y), make_float2(b0.z, b0.w), make_float2(b1.x, b1.y),
                            make_float2(b1.z, b1.w)};
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float2 db = bcast2(c ? du.y : du.x);
#pragma unroll
        for (int j = 0; j < 4; ++j) h[c][j] = fma2(w.e[c][j], h[c][j], mul2(db, B2[j]));
      }
      if (!CARRY) {
        const float4 e0 = lds4(s + NS), e1 = lds4(s + NS + 4);
        const float2 C2[4] = {make_float2(e0.x, e0.y), make_float2(e0.z, e0.w), make_float2(e1.x, e1.y),
                              make_float2(e1.z, e1.w)};
        float part[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float2 acc =
              fma2(C2[3], h[c][3], fma2(C2[2], h[c][2], fma2(C2[1], h[c][1], mul2(C2[0], h[c][0]))));
          part[c] = acc.x + acc.y;
        }
        float yy = fmaf(hb ? w.u.y : w.u.x, Dd, pair_scatter(part[0], part[1], hb));
        if (HAS_Z) yy *= silu_f(ld_one(&st.z[r][lane]));
        // an explicit global store: a generic one could alias the ring, and would keep the next row's
        // shared loads behind it
        stg_if_t<T>(y + (t0 + r) * a.ldy, yy, ok);
      }
    };
    const int nr = min(CSC_ROWS, p.t1 - t0);
    Decay ka, kb;
    decay(0, ka);
    if (nr == CSC_ROWS) {
#pragma unroll
      for (int r = 0; r < CSC_ROWS; ++r) {
        if (r + 1 < CSC_ROWS) decay(r + 1, kb);
        row(r, ka);
        ka = kb;
      }
    } else {
      for (int r = 0; r < nr; ++r) {
        row(r, ka);
        if (r + 1 < nr) decay(r + 1, ka);
      }
    }
    settle(ahead, free_stage);
    stage = stage + 1 == CSC_STAGES ? 0 : stage + 1;
  }
  float* dst = nullptr;
  if (CARRY) {
    dst = k.h + int64_t(p.carry) * a.dn * NS;
    if (ok) k.sum[int64_t(p.carry) * a.dn + own] = hb ? dsum.y : dsum.x;
  } else if (p.t1 == p.end) {
    dst = a.state + int64_t(p.slot) * a.dn * NS;
  } else if (p.carry >= 0 && p.ordinal == 0) {
    dst = k.h + int64_t(p.carry) * a.dn * NS;
  }
  if (dst == nullptr) return;
#pragma unroll
  for (int c = 0; c < 2; ++c)
    if (dp + c < a.dn) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
        *reinterpret_cast<float4*>(dst + int64_t(dp + c) * NS + 8 * hb + 4 * j) =
            make_float4(h[c][2 * j].x, h[c][2 * j].y, h[c][2 * j + 1].x, h[c][2 * j + 1].y);
    }
}

// A launch runs pieces of one phase (the request's pieces in two launches, so
// that a later piece finds its start and no slot is written before it is read):
// first: whole requests and first pieces from their source's state, and the
//        carries of the pieces between the first and the last one;
// later: pieces after the first, from the chained carries;
// whole: no request is split, there is one launch.
enum ScanPhase { SCAN_WHOLE, SCAN_FIRST, SCAN_LATER };
template <typename T, int G, bool HAS_Z>
__global__ void __launch_bounds__(CSC_WARPS * 32)
    cached_scan_kernel(const CachedScanArgs a, const int32_t* __restrict__ pieces, int groups, int bc_grain,
                       int phase, const ScanCarries k) {
  extern __shared__ __align__(16) unsigned char scan_raw[];
  Piece p = load_piece(pieces, blockIdx.x / groups, a.rows, a.n_slots);
  p.carry = p.carry < k.rows ? p.carry : -1;
  p.ordinal = min(max(p.ordinal, 0), max(p.carry, 0));
  if (phase == SCAN_FIRST) launch_next();
  if (phase == SCAN_FIRST && p.carry >= 0 && p.ordinal > 0)
    cached_scan_piece<T, G, HAS_Z, true>(a, p, blockIdx.x % groups, bc_grain, false, k, scan_raw);
  else
    cached_scan_piece<T, G, HAS_Z, false>(a, p, blockIdx.x % groups, bc_grain, phase == SCAN_LATER, k, scan_raw);
}

// State entering every later piece of the split requests: chain i = {first
// carry row, pieces, 0, 0}; one thread per (chain, channel, state) walks the
// pieces' maps, the loads of CCH_AHEAD pieces at a time.  Only for requests of
// many pieces: a few are chained by the pieces themselves.
constexpr int CCH_AHEAD = 8;
__global__ void cached_chain_kernel(const int32_t* __restrict__ chains, const float* __restrict__ A,
                                    const float* carry_h, const float* carry_s, float* h_start, int64_t dn, int rows,
                                    int blocks) {
  launch_next();
  wait_previous();
  const int64_t i = int64_t(blockIdx.x % blocks) * blockDim.x + threadIdx.x;
  if (i >= dn * NS) return;
  int4 c = reinterpret_cast<const int4*>(chains)[blockIdx.x / blocks];
  if (c.x < 0 || c.x >= rows) return;
  c.y = min(c.y, rows - c.x);
  const float An = A[i];
  const int64_t ch = i / NS;
  float h = carry_h[int64_t(c.x) * dn * NS + i];
  for (int k0 = 1; k0 < c.y; k0 += CCH_AHEAD) {
    float s[CCH_AHEAD], g[CCH_AHEAD];
#pragma unroll
    for (int q = 0; q < CCH_AHEAD; ++q) {
      const bool in = k0 + q + 1 < c.y;  // the last piece has no map
      const int64_t row = c.x + (in ? k0 + q : 0);
      s[q] = in ? carry_s[row * dn + ch] : 0.f;
      g[q] = in ? carry_h[row * dn * NS + i] : 0.f;
    }
#pragma unroll
    for (int q = 0; q < CCH_AHEAD; ++q) {
      if (k0 + q < c.y) {
        h_start[int64_t(c.x + k0 + q) * dn * NS + i] = h;
        h = apply_map(expf(0.5f * (An * s[q])), h, g[q]);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Single tokens: row i is request i.  A warp owns 32 channels of one row; four
// lanes share a channel (four states each), so the state moves as whole
// 512-byte warp accesses, 2 KB of it in flight a warp.  In turn i the quad g
// works on channel 8 i + g; a transposing sum over the quad leaves lane 4 g + q
// the output of channel 8 q + g, its own.
// Bound: HBM, 128 bytes of state a channel and token.  256 x 1536 fp32, gated,
// states from HBM: 12.1 us, 4.7 TB/s (16.2 in scalar arithmetic, 390
// instructions a warp instead of about 130; 13.4 with two rows a warp, whose
// registers halve the warps an SM holds; 14.0 with ten CTAs an SM, which
// spill); 1024 x 1536: 40 to 43 us, 5.3 to 5.7 TB/s; 333 x 768 bf16 8.2 us, fp32
// 8.6, 333 x 771 8.4 to 9.0 (rows of scalars cost little beside the states);
// 1 x 768: 2.0 us.
// ---------------------------------------------------------------------------
constexpr int CST_WARPS = 4;
constexpr int CST_CTAS = 8;  // an SM is to hold

template <typename T, bool HAS_Z>
__global__ void __launch_bounds__(CST_WARPS * 32, CST_CTAS)
    cached_step_kernel(const CachedScanArgs a, const int32_t* __restrict__ slots, const int32_t* __restrict__ sources,
                       int groups, int bc_wide) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int row = blockIdx.x / groups;
  const int d0 = ((blockIdx.x % groups) * CST_WARPS + warp) * 32;
  if (d0 >= a.dn) return;
  const int own = d0 + 8 * q + g;
  const bool ok = own < a.dn;
  const int oc = min(own, a.dn - 1);
  const int slot = slots[row], source = sources[row];
  const float u = ld_one(static_cast<const T*>(a.u) + row * a.ldu + oc);
  const float dl = ld_one(static_cast<const T*>(a.delta) + row * a.ldd + oc);
  const float z = HAS_Z ? ld_one(static_cast<const T*>(a.z) + row * a.ldz + oc) : 0.f;
  const float4 B4 = ld_four(static_cast<const T*>(a.B) + row * a.ldb + 4 * q, bc_wide != 0);
  const float4 C4 = ld_four(static_cast<const T*>(a.C) + row * a.ldc + 4 * q, bc_wide != 0);
  T* y = static_cast<T*>(a.y) + row * a.ldy + oc;
  if (slot < 0 || slot >= a.n_slots) {  // padding request
    stg_if_t<T>(y, 0.f, ok);
    return;
  }
  // turns past the last channel repeat it and store nothing
  int64_t at[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) at[i] = int64_t(min(d0 + 8 * i + g, a.dn - 1)) * NS + 4 * q;
  const bool kept = source >= 0 && source < a.n_slots;
  const float* from = a.state + int64_t(kept ? source : 0) * a.dn * NS;
  float* to = a.state + int64_t(slot) * a.dn * NS;
  float4 h[4], A4[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    h[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (kept) h[i] = *reinterpret_cast<const float4*>(from + at[i]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) A4[i] = *reinterpret_cast<const float4*>(a.A + at[i]);
  const float Dd = a.D[oc];
  const float du = dl * u, dlog = dl * kLog2e;
  const float2 B0 = make_float2(B4.x, B4.y), B1 = make_float2(B4.z, B4.w);
  const float2 C0 = make_float2(C4.x, C4.y), C1 = make_float2(C4.z, C4.w);
  float part[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 du2 = bcast2(__shfl_sync(0xffffffffu, du, (lane & ~3) + i));
    const float2 dg = bcast2(__shfl_sync(0xffffffffu, dlog, (lane & ~3) + i)), off = bcast2(kEx2ArgBias);
    const float2 e0 = fma2(dg, make_float2(A4[i].x, A4[i].y), off), e1 = fma2(dg, make_float2(A4[i].z, A4[i].w), off);
    const float2 h0 = fma2(make_float2(ex2_approx(e0.x), ex2_approx(e0.y)), make_float2(h[i].x, h[i].y), mul2(du2, B0));
    const float2 h1 = fma2(make_float2(ex2_approx(e1.x), ex2_approx(e1.y)), make_float2(h[i].z, h[i].w), mul2(du2, B1));
    const float2 s = fma2(C1, h1, mul2(C0, h0));
    part[i] = s.x + s.y;
    if (d0 + 8 * i + g < a.dn) *reinterpret_cast<float4*>(to + at[i]) = make_float4(h0.x, h0.y, h1.x, h1.y);
  }
  // lane q of the quad keeps the sum of part[q] over the quad
  const float p0 = (q & 1 ? part[1] : part[0]) + __shfl_xor_sync(0xffffffffu, q & 1 ? part[0] : part[1], 1);
  const float p1 = (q & 1 ? part[3] : part[2]) + __shfl_xor_sync(0xffffffffu, q & 1 ? part[2] : part[3], 1);
  const float sum = (q & 2 ? p1 : p0) + __shfl_xor_sync(0xffffffffu, q & 2 ? p0 : p1, 2);
  float yy = fmaf(u, Dd, sum);
  if (HAS_Z) yy *= silu_f(z);
  stg_if_t<T>(y, yy, ok);
}

// ---------------------------------------------------------------------------
// Causal conv1d + SiLU.  A thread owns VEC adjacent channels of one piece and
// slides the K-row window along its rows.  The first piece of a request (and
// the only one that can reach rows before it: pieces hold at least K - 1
// rows) reads the stored window, and writes the new one: the request's last
// K - 1 rows, reaching back into the old window when it has fewer.  The same
// thread reads the old window before it writes, so a slot may be both.
// Bound: HBM, a read and a write of each element.  32768 x 1536, K = 4: fp32
// 70 us, 5.7 TB/s (148 with one row's loads at a time); bf16 46 us, more than
// its bytes (31) or the exponential unit (22, two operations an element) take:
// an access of four channels is 8 bytes there; K = 8 fp32 111 us (the window of 7
// rows before each piece and 140 registers); 64 tokens x 768: 2.9 to 3.1 us.
// ---------------------------------------------------------------------------
constexpr int CCV_ROWS = 32;       // rows of a piece
constexpr int CCV_FEW_ROWS = 16;   // where those would give the SMs too few threads (both at least K - 1)
constexpr int CCV_THREADS = 64;
constexpr int CCV_KMAX = 8;
constexpr int CCV_AHEAD = 8;  // rows whose loads are issued together

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

template <typename T, int VEC, int K>
__global__ void __launch_bounds__(CCV_THREADS)
    cached_conv_kernel(const CachedConvArgs a, const int32_t* __restrict__ pieces, int groups) {
  const Piece p = load_piece(pieces, blockIdx.x / groups, a.rows, a.n_slots);
  const int c = ((blockIdx.x % groups) * CCV_THREADS + threadIdx.x) * VEC;
  if (c >= a.channels) return;
  T* __restrict__ out = static_cast<T*>(a.out) + c;
  if (p.slot < 0) {
    const float zero[VEC] = {};
    for (int t = p.t0; t < p.t1; ++t) stv<T, VEC>(out + t * a.ldo, zero);
    return;
  }
  const T* __restrict__ x = static_cast<const T*>(a.x) + c;
  T* state = static_cast<T*>(a.state) + c;
  const int64_t C = a.channels;
  // the thread's taps lie together: VEC channels x K
  float w[VEC * K], bias[VEC], win[K][VEC];
  if constexpr (VEC == 4) {
#pragma unroll
    for (int i = 0; i < K; ++i) {
      const float4 q = __ldg(reinterpret_cast<const float4*>(a.w + int64_t(c) * K) + i);
      w[4 * i] = q.x, w[4 * i + 1] = q.y, w[4 * i + 2] = q.z, w[4 * i + 3] = q.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < K; ++i) w[i] = __ldg(a.w + int64_t(c) * K + i);
  }
#pragma unroll
  for (int v = 0; v < VEC; ++v) bias[v] = __ldg(a.bias + c + v);
  // rows before the piece: rows of the request, or of the stored window.  Slot
  // m is row t0 - (K - m) before the first shift.
#pragma unroll
  for (int m = 1; m < K; ++m) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) win[m][v] = 0.f;
    const int t = p.t0 - (K - m);
    if (t >= p.begin)
      ldv<T, VEC>(x + t * a.ldx, win[m]);
    else if (p.source >= 0)
      ldv<T, VEC>(state + (int64_t(p.source) * (K - 1) + (K - 1 - (p.begin - t))) * C, win[m]);
  }
  if (p.t0 == p.begin) {
    // the new window: its row m - 1 is row end - (K - m) of the request, and
    // where that lies before the request, the old window's (read above: slot s
    // is row begin - (K - s))
    const int len = p.end - p.begin;
#pragma unroll
    for (int m = 1; m < K; ++m) {
      float v[VEC] = {};
      const int t = p.end - (K - m);
      if (t >= p.begin) {
        ldv<T, VEC>(x + t * a.ldx, v);
      } else {
#pragma unroll
        for (int s = m; s < K; ++s)
          if (s == m + len) {
#pragma unroll
            for (int q = 0; q < VEC; ++q) v[q] = win[s][q];
          }
      }
      stv<T, VEC>(state + (int64_t(p.slot) * (K - 1) + m - 1) * C, v);
    }
  }
  for (int t0 = p.t0; t0 < p.t1; t0 += CCV_AHEAD) {
    float xs[CCV_AHEAD][VEC];
#pragma unroll
    for (int u = 0; u < CCV_AHEAD; ++u) ldv<T, VEC>(x + min(t0 + u, p.t1 - 1) * a.ldx, xs[u]);
#pragma unroll
    for (int u = 0; u < CCV_AHEAD; ++u) {
      if (t0 + u < p.t1) {
        float acc[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
#pragma unroll
          for (int m = 0; m < K - 1; ++m) win[m][v] = win[m + 1][v];
          win[K - 1][v] = xs[u][v];
        }
        if constexpr (VEC == 4) {  // channels in packed pairs
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            float2 s = make_float2(bias[2 * q], bias[2 * q + 1]);
#pragma unroll
            for (int m = 0; m < K; ++m)
              s = fma2(make_float2(w[2 * q * K + m], w[(2 * q + 1) * K + m]),
                       make_float2(win[m][2 * q], win[m][2 * q + 1]), s);
            acc[2 * q] = s.x;
            acc[2 * q + 1] = s.y;
          }
        } else {
          acc[0] = bias[0];
#pragma unroll
          for (int m = 0; m < K; ++m) acc[0] = fmaf(w[m], win[m][0], acc[0]);
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) acc[v] = silu_f(acc[v]);
        stv<T, VEC>(out + (t0 + u) * a.ldo, acc);
      }
    }
  }
}

}  // namespace vmscan
