// vmscan_lora.cuh — low-rank adapters of many requests beside a shared
// projection: out_t = base_t + scale_a (x_t A_a^T) B_a^T, a = the adapter of
// row t's request (no counterpart in the reference).
//
// The host sorts the rows by adapter and cuts them into tiles of at most
// LORA_ROWS rows of one adapter (int32[4] records: first entry of the row
// list, entries, adapter or -1, 0).  One CTA owns a tile and a share of the
// output columns: its warps split d_in and form partial products
// S = x A^T (rows x rank), which are added in shared memory in a fixed order,
// and then split the columns for out = base + S B^T.  Nothing but base, x and
// out crosses HBM; the rank-wide S never leaves the SM.
//
// Both products run on mma.sync: a tile has a few rows of one adapter, too
// little work per operand byte for tcgen05 to matter at a rank of up to 16,
// where the kernel is bound by the bytes of base and out.  That no longer holds
// at a rank of 64 on many rows of one adapter (figures below), for which this is
// not the best design.  Operands go from global
// memory straight to fragments: the order of a product's inner index is free,
// so a lane's four (fp32) or eight (bf16) adjacent elements stand for the
// inner indices that its fragment registers hold, on both operands alike, and
// every access is a 16-byte one.
//   fp32: TF32 hi / lo parts, hi hi + hi lo + lo hi (lo lo is 2^-22 of a
//         product at most).  The tensor pipe cuts off, towards zero, what lies
//         below the last place of its accumulator, so that a chain of products
//         in one accumulator drifts: 768 -> 1536, rank 64, was off by 1.2e-6
//         of the norm (plain fp32 products: 3.7e-7).  A chain therefore covers
//         16 inner indices, starts from zero, and is added to the sum in fp32,
//         rounded to nearest: 1.7e-7, whatever the lengths, for 1 to 9 % of
//         the time (9: rank 24 on unaligned rows).
//   bf16: x, A, B are exact operands; S enters the second product as three
//         bf16 parts (24 bits).  The output is rounded once, to 2^-9 of its
//         norm, far above what the chains lose (3e-6).
//
// Measured on B200: 16384 rows of 16 uneven requests, 384 -> 1536, rank 16, fp32
// 52 us, 4.4 TB/s of the 227 MB that have to move (the floor is 35 us; 14 warps
// an SM wait for base and B); the same rows 768 -> 1536, rank 64, bf16 68 us and
// fp32 139 us (128 with even requests; floors 20 and 39.  Three TF32 products a
// term: the tensor pipe alone takes about 50; the rest is mostly A, B and their
// parts, loaded and split again for each tile of 32 rows); 64 rows of 32
// adapters 384 -> 1536, rank 16: 6.3 to 6.6 us (latency: row list, x and A, S, B).
// Rings of asynchronous copies for x, base and B cost more occupancy than they
// hid (62 to 74 us on the first case at the time, 53 without).
#pragma once

#include "vmscan_common.cuh"

namespace vmscan {

constexpr int LORA_ROWS = 32;
constexpr int LORA_WARPS = 4;
constexpr int LORA_RMAX = 128;
constexpr int LORA_LD = 18;       // row of 16 products in shared memory (two more keep the rows off each other's banks)
constexpr int LORA_RCHUNK = 32;  // rank columns whose partial products a warp holds at a time

struct LoraArgs {
  const void* x;
  const void* a;      // (adapters, rank, lda), columns from d_in on zero
  const void* b;      // (adapters, d_out, rank)
  const void* base;
  void* out;
  const float* scale; // (adapters)
  const int32_t* row_index;
  const int32_t* tiles;
  int64_t lda, ldx, ldbase, ldout;
  int rows, d_in, d_out, rank, adapters, n_index;
};

__device__ __forceinline__ void mma_tf32(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Sixteen bytes of a row from column c on, zero past `limit`.
template <typename T>
struct Chunk {
  static constexpr int N = 16 / int(sizeof(T));
  uint32_t w[4];
};
template <typename T, bool WIDE>
__device__ __forceinline__ Chunk<T> ld_chunk(const T* row, int c, int limit) {
  Chunk<T> k;
  if constexpr (WIDE) {  // limit is a multiple of N: a chunk is inside or outside
    const uint4 q = c < limit ? __ldg(reinterpret_cast<const uint4*>(row + c)) : make_uint4(0, 0, 0, 0);
    k.w[0] = q.x, k.w[1] = q.y, k.w[2] = q.z, k.w[3] = q.w;
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) k.w[i] = c + i < limit ? __float_as_uint(row[c + i]) : 0u;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = c + 2 * i < limit ? __bfloat16_as_ushort(row[c + 2 * i]) : 0;
      const uint32_t hi = c + 2 * i + 1 < limit ? __bfloat16_as_ushort(row[c + 2 * i + 1]) : 0;
      k.w[i] = lo | hi << 16;
    }
  }
  return k;
}

// Four elements of a row from column c on as they lie in memory (fp32: 4
// words, bf16: 2), zero from `limit` (a multiple of 4) on.  Ordinary loads
// (base may be the output: no read-only path), which the compiler may still
// move across the stores of other columns.
template <typename T>
struct Four {
  uint32_t w[sizeof(T)];
};
template <typename T>
__device__ __forceinline__ Four<T> ld_quad(const T* row, int c, int limit) {
  Four<T> k{};
  if constexpr (sizeof(T) == 4) {
    if (c < limit)
      asm("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];"
          : "=r"(k.w[0]), "=r"(k.w[1]), "=r"(k.w[2]), "=r"(k.w[3])
          : "l"(row + c));
  } else {
    if (c < limit) asm("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(k.w[0]), "=r"(k.w[1]) : "l"(row + c));
  }
  return k;
}

__device__ __forceinline__ float ld_scalar(const float* p) {
  float v;
  asm("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ float ld_scalar(const __nv_bfloat16* p) {
  unsigned short v;
  asm("ld.global.u16 %0, [%1];" : "=h"(v) : "l"(p));
  return __uint_as_float(uint32_t(v) << 16);
}

template <typename T>
__device__ __forceinline__ float4 four_f(const Four<T>& k) {
  if constexpr (sizeof(T) == 4) {
    return make_float4(__uint_as_float(k.w[0]), __uint_as_float(k.w[1]), __uint_as_float(k.w[2]),
                       __uint_as_float(k.w[3]));
  } else {
    const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&k.w[0]));
    const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&k.w[1]));
    return make_float4(a.x, a.y, b.x, b.y);
  }
}

// Columns c .. c + 3 of a row, c and limit multiples of 4.
template <typename T>
__device__ __forceinline__ void st_quad(T* row, int c, int limit, const float4& v) {
  if (c >= limit) return;
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(row + c) = v;
  } else {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    uint2 q;
    q.x = *reinterpret_cast<const uint32_t*>(&a);
    q.y = *reinterpret_cast<const uint32_t*>(&b);
    *reinterpret_cast<uint2*>(row + c) = q;
  }
}

// TF32 parts of an fp32 word.  The integer rounding of hi carries a NaN whose
// mantissa is all ones (the one the hardware makes) over to zero; the rounding
// of lo is the conversion instruction, which keeps the NaN that x - hi then is,
// as it is for infinities, so that neither is lost (lo rounded the integer way
// too lost them and took 6.1 instead of 6.3 us for 64 rows of 32 adapters, 384 ->
// 1536, rank 16, 106 instead of 108 us for 16384 rows of the same at rank 64;
// both parts by conversion 6.7 and 113).
__device__ __forceinline__ uint32_t tf32_hi(uint32_t x) { return (x + 0x1000u) & 0xFFFFE000u; }
__device__ __forceinline__ uint32_t tf32_lo(uint32_t x, uint32_t hi) {
  uint32_t lo;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(__uint_as_float(x) - __uint_as_float(hi)));
  return lo;
}

// Fragments of S for 16 rank columns and one 16-row block, as groups of four
// words a lane: fp32 two steps of hi and two of lo, bf16 three parts.
template <typename T>
struct LoraFrag {
  static constexpr int GROUPS = sizeof(T) == 4 ? 4 : 3;
};
template <typename T>
constexpr size_t lora_smem(int rank) {
  return (size_t(LORA_WARPS) * LORA_ROWS * (LORA_RCHUNK + 1) +
          size_t(2) * ((rank + 15) / 16) * 32 * 4 * LoraFrag<T>::GROUPS) * 4;
}

// MT: 16-row blocks of the tile in use.  WIDE: every row of x, base and out
// takes whole accesses (x 16 bytes, base and out four elements); A and B
// always do.  Without, base and out move as rows of 16 adjacent elements, two
// rows an access, and the products cross to that layout in shared memory (as
// scalars in the products' own layout, 4 columns of 8 rows an access, 16384
// rows 700 -> 1411, rank 10, bf16 took 119 us).  STEPS: 16-column steps of the
// rank, 0: any number.
template <typename T, bool WIDE, int MT, int STEPS>
__device__ __forceinline__ void lora_tile(const LoraArgs& a, const int* row, int n, int ad, int c_begin, int c_end,
                                          float* part, uint32_t* frag) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  constexpr int CN = Chunk<T>::N;
  // The products with a lo part, 2^-11 of the others, may stay in accumulators
  // of their own for the whole of d_in, which shortens the chains that a short
  // call waits for: 1 x 768 -> 768, rank 8, 5.5 us (6.6 in the one chain), 64
  // rows of 32 adapters, 384 -> 1536, rank 16, 6.3 (6.7).  More columns of S or
  // unaligned rows leave no registers for them (16384 rows 768 -> 1536, rank 64:
  // 180 us for 128).  By variant and not by the tile's rows, so that a row's
  // result does not depend on the rows beside it.
  constexpr bool APART = sizeof(T) == 4 && WIDE && STEPS == 1;
  constexpr int NT = STEPS == 1 ? 2 : LORA_RCHUNK / 8;  // 8-column blocks of S a warp holds
  int r[2 * MT];  // rows g, g + 8, ... of the tile; those past the last repeat it
#pragma unroll
  for (int i = 0; i < 2 * MT; ++i) r[i] = row[min(g + 8 * i, n - 1)];
  const int steps = STEPS > 0 ? STEPS : (a.rank + 15) / 16;
  if (ad >= 0) {
    const T* A = static_cast<const T*>(a.a) + int64_t(ad) * a.rank * a.lda;
    const T* xr[2 * MT];
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) xr[i] = static_cast<const T*>(a.x) + r[i] * a.ldx;
    const float scale = a.scale[ad];
    for (int rc = 0; rc < a.rank; rc += LORA_RCHUNK) {
      float acc[MT][NT][4] = {};
      float small[APART ? MT : 1][APART ? NT : 1][4] = {};
      const int nt = min(NT, (a.rank - rc + 7) / 8);
      const T* ar[NT];  // row of A whose products this lane's B fragments hold
#pragma unroll
      for (int j = 0; j < NT; ++j) ar[j] = A + int64_t(min(rc + 8 * j + g, a.rank - 1)) * a.lda;
#pragma unroll (APART && MT == 2 ? 1 : 2)  // (16384 rows, rank 16: 51.4 us, 52.3 with two chunks)
      for (int c = (warp * 4 + t) * CN; c - t * CN < a.d_in; c += LORA_WARPS * 4 * CN) {
        Chunk<T> x[2 * MT], ab[NT];
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) x[i] = ld_chunk<T, WIDE>(xr[i], c, a.d_in);
#pragma unroll
        for (int j = 0; j < NT; ++j) ab[j] = ld_chunk<T, true>(ar[j], c, int(a.lda));  // rows past the rank: never summed
        uint32_t xl[2 * MT][4];
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int i = 0; i < 2 * MT; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t hi = tf32_hi(x[i].w[k]);
              xl[i][k] = tf32_lo(x[i].w[k], hi);
              x[i].w[k] = hi;
            }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          if (j < nt) {
            const Chunk<T>& b = ab[j];
            float sum[MT][4] = {};  // fp32: the chain of this chunk
#pragma unroll
            for (int h = 0; h < 2; ++h) {  // words 2h and 2h + 1 of the chunk are one step of the product
              uint32_t bh[2] = {b.w[2 * h], b.w[2 * h + 1]}, bl[2];
              if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                  const uint32_t hi = tf32_hi(bh[q]);
                  bl[q] = tf32_lo(bh[q], hi);
                  bh[q] = hi;
                }
              }
#pragma unroll
              for (int m = 0; m < MT; ++m) {
                const uint32_t xa[4] = {x[2 * m].w[2 * h], x[2 * m + 1].w[2 * h], x[2 * m].w[2 * h + 1],
                                        x[2 * m + 1].w[2 * h + 1]};
                if constexpr (sizeof(T) == 4) {
                  const uint32_t la[4] = {xl[2 * m][2 * h], xl[2 * m + 1][2 * h], xl[2 * m][2 * h + 1],
                                          xl[2 * m + 1][2 * h + 1]};
                  mma_tf32(APART ? small[m][j] : sum[m], la, bh[0], bh[1]);
                  mma_tf32(APART ? small[m][j] : sum[m], xa, bl[0], bl[1]);
                  mma_tf32(sum[m], xa, bh[0], bh[1]);
                } else {
                  mma_bf16(acc[m][j], xa, bh[0], bh[1]);
                }
              }
            }
            if constexpr (sizeof(T) == 4) {
#pragma unroll
              for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int q = 0; q < 4; ++q) acc[m][j][q] += sum[m][q];
            }
          }
        }
      }
      if constexpr (APART) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[m][j][q] += small[m][j][q];
      }
      // partial products of the warps, then their sum in a fixed order as the
      // fragments of the second product
      constexpr int LD = LORA_RCHUNK + 1;
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < NT; ++j)
          if (j < nt) {
            float* p = part + (warp * LORA_ROWS + 16 * m + g) * LD + 8 * j + 2 * t;
            p[0] = acc[m][j][0];
            p[1] = acc[m][j][1];
            p[8 * LD] = acc[m][j][2];
            p[8 * LD + 1] = acc[m][j][3];
          }
      __syncthreads();
      const int here = min(NT / 2, steps - rc / 16);  // 16-column steps of this chunk
      for (int e = threadIdx.x; e < MT * here * 32; e += LORA_WARPS * 32) {
        const int fl = e & 31, s = (e >> 5) % here, m = (e >> 5) / here;
        const int fr = 16 * m + (fl >> 2), fc = 16 * s + 4 * (fl & 3);
        float v[2][4];  // rows fr, fr + 8; columns fc .. fc + 3
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float sum = 0.f;
            if (rc + fc + q < a.rank) {
#pragma unroll
              for (int w = 0; w < LORA_WARPS; ++w) sum += part[(w * LORA_ROWS + fr + 8 * i) * LD + fc + q];
            }
            v[i][q] = scale * sum;
          }
        uint32_t* f = frag + (size_t(m * steps + rc / 16 + s) * LoraFrag<T>::GROUPS * 32 + fl) * 4;
        if constexpr (sizeof(T) == 4) {
          // groups 0, 1: hi of step h = 0, 1 (columns fc + 2h, fc + 2h + 1); 2, 3: lo
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const uint32_t x = __float_as_uint(v[q & 1][2 * h + (q >> 1)]), hi = tf32_hi(x);
              f[128 * h + q] = hi;
              f[128 * (2 + h) + q] = tf32_lo(x, hi);
            }
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float x0 = v[q & 1][2 * (q >> 1)], x1 = v[q & 1][2 * (q >> 1) + 1];
#pragma unroll
            for (int w = 0; w < 3; ++w) {
              const __nv_bfloat162 b2 = __floats2bfloat162_rn(x0, x1);
              f[128 * w + q] = *reinterpret_cast<const uint32_t*>(&b2);
              const float2 back = __bfloat1622float2(b2);
              x0 -= back.x;
              x1 -= back.y;
            }
          }
        }
      }
      if (rc + LORA_RCHUNK < a.rank) __syncthreads();  // part is read before the next chunk's is written
    }
  }
  // columns in groups of 16, two 8-column blocks of the product.  WIDE: lane t
  // of a quad owns columns 4t .. 4t + 3 of its rows, which stand for columns
  // 2t, 2t + 1 of the two blocks; else lane l owns column l % 16 of rows
  // l / 16, l / 16 + 2, ...
  const T* B = static_cast<const T*>(a.b) + int64_t(max(ad, 0)) * a.d_out * a.rank;
  const T* br[2 * MT];
  T* outr[2 * MT];
#pragma unroll
  for (int i = 0; i < 2 * MT; ++i) {
    br[i] = static_cast<const T*>(a.base) + r[i] * a.ldbase;
    outr[i] = static_cast<T*>(a.out) + r[i] * a.ldout;
  }
  constexpr int HELD = STEPS == 0 ? 1 : STEPS;  // steps of B loaded together
  const int half = lane >> 4, lcol = lane & 15;
  float* stage = part + warp * LORA_ROWS * (LORA_RCHUNK + 1);  // !WIDE: the warp's products, free since S is complete
  struct Group {
    Four<T> base[WIDE ? 2 * MT : 1];
    float one[WIDE ? 1 : 8 * MT];
    Four<T> b[HELD][2];
  };
  auto load_b = [&](int c0, int s, Four<T> b[2]) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int col = c0 + (WIDE ? 4 * (g >> 1) + (g & 1) + 2 * j : 8 * j + g);
      b[j] = ld_quad<T>(B + int64_t(min(col, a.d_out - 1)) * a.rank, 16 * s + 4 * t, a.rank);
    }
  };
  auto load = [&](int c0, Group& k) {
    if constexpr (WIDE) {
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i) k.base[i] = ld_quad<T>(br[i], c0 + 4 * t, a.d_out);
    } else {
#pragma unroll
      for (int i = 0; i < 8 * MT; ++i) {
        k.one[i] = 0.f;
        if (c0 + lcol < a.d_out)
          k.one[i] = ld_scalar(static_cast<const T*>(a.base) + row[min(2 * i + half, n - 1)] * a.ldbase + c0 + lcol);
      }
    }
    if (STEPS > 0 && ad >= 0) {
#pragma unroll
      for (int s = 0; s < HELD; ++s) load_b(c0, s, k.b[s]);
    }
  };
  auto multiply = [&](const Four<T> b[2], int s, float acc[MT][2][4]) {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const uint4* f = reinterpret_cast<const uint4*>(frag) + size_t(m * steps + s) * LoraFrag<T>::GROUPS * 32 + lane;
      if constexpr (sizeof(T) == 4) {
        float sum[2][4] = {};  // the chain of this step
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4 fh = f[32 * h], fl = f[32 * (2 + h)];
          const uint32_t sh[4] = {fh.x, fh.y, fh.z, fh.w}, sl[4] = {fl.x, fl.y, fl.z, fl.w};
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t h0 = tf32_hi(b[j].w[2 * h]), h1 = tf32_hi(b[j].w[2 * h + 1]);
            mma_tf32(sum[j], sl, h0, h1);
            mma_tf32(sum[j], sh, tf32_lo(b[j].w[2 * h], h0), tf32_lo(b[j].w[2 * h + 1], h1));
            mma_tf32(sum[j], sh, h0, h1);
          }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) acc[m][j][q] = STEPS == 1 ? sum[j][q] : acc[m][j][q] + sum[j][q];
      } else {
#pragma unroll
        for (int w = 2; w >= 0; --w) {
          const uint4 fw = f[32 * w];
          const uint32_t sw[4] = {fw.x, fw.y, fw.z, fw.w};
#pragma unroll
          for (int j = 0; j < 2; ++j) mma_bf16(acc[m][j], sw, b[j].w[0], b[j].w[1]);
        }
      }
    }
  };
  constexpr int STEP = 16 * LORA_WARPS;
  Group cur, nxt;
  if (c_begin + 16 * warp < c_end) load(c_begin + 16 * warp, cur);
  if (ad >= 0) __syncthreads();  // S is complete
  for (int c0 = c_begin + 16 * warp; c0 < c_end; c0 += STEP) {
    if (c0 + STEP < c_end) load(c0 + STEP, nxt);
    float acc[MT][2][4] = {};
    if (ad >= 0) {
      if constexpr (STEPS > 0) {
#pragma unroll
        for (int s = 0; s < STEPS; ++s) multiply(cur.b[s], s, acc);
      } else {
#pragma unroll 2
        for (int s = 0; s < steps; ++s) {
          Four<T> b[2];
          load_b(c0, s, b);
          multiply(b, s, acc);
        }
      }
    }
    if constexpr (WIDE) {
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i) {
        const float4 v = four_f(cur.base[i]);
        const float* p0 = &acc[i >> 1][0][2 * (i & 1)];
        const float* p1 = &acc[i >> 1][1][2 * (i & 1)];
        if (g + 8 * i < n)
          st_quad(outr[i], c0 + 4 * t, a.d_out, make_float4(v.x + p0[0], v.y + p0[1], v.z + p1[0], v.w + p1[1]));
      }
    } else {
      __syncwarp();  // every lane has read the group before
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          *reinterpret_cast<float2*>(stage + (g + 8 * i) * LORA_LD + 8 * j + 2 * t) =
              make_float2(acc[i >> 1][j][2 * (i & 1)], acc[i >> 1][j][2 * (i & 1) + 1]);
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 8 * MT; ++i) {
        const int rr = 2 * i + half;
        stg_if_t<T>(static_cast<T*>(a.out) + row[min(rr, n - 1)] * a.ldout + c0 + lcol,
                    cur.one[i] + stage[rr * LORA_LD + lcol], rr < n && c0 + lcol < a.d_out);
      }
    }
    cur = nxt;
  }
}

// CTAs an SM is to hold (registers), measured with the fp32 products in one
// chain: 16384 rows 384 -> 1536, rank 16, fp32 took 50 us with four, 54 with
// five, 72 with three; 768 -> 1536, rank 64, fp32 141 with four, 129 with three;
// 5000 rows 457 -> 763, rank 10, bf16 29 with four, 23 with five.
template <typename T, bool WIDE, int STEPS>
constexpr int lora_ctas() {
  return STEPS == 1 ? (WIDE ? 4 : 5) : STEPS == 4 && sizeof(T) == 4 ? 3 : 4;
}

template <typename T, bool WIDE, int STEPS>
__global__ void __launch_bounds__(LORA_WARPS * 32, (lora_ctas<T, WIDE, STEPS>())) lora_add_kernel(const LoraArgs a, int cols_per_cta) {
  extern __shared__ __align__(16) unsigned char lora_raw[];
  __shared__ int row[LORA_ROWS];
  float* part = reinterpret_cast<float*>(lora_raw);
  uint32_t* frag = reinterpret_cast<uint32_t*>(part + LORA_WARPS * LORA_ROWS * (LORA_RCHUNK + 1));
  const int4 tile = reinterpret_cast<const int4*>(a.tiles)[blockIdx.x];
  const int first = max(tile.x, 0);
  const int n = min(min(tile.y, LORA_ROWS), a.n_index - first);
  if (n <= 0) return;
  const int ad = tile.z < a.adapters ? tile.z : -1;
  if (ad < 0 && a.out == a.base) return;
  for (int i = threadIdx.x; i < n; i += LORA_WARPS * 32) row[i] = min(max(a.row_index[first + i], 0), a.rows - 1);
  __syncthreads();
  const int c0 = blockIdx.y * cols_per_cta, c1 = min(c0 + cols_per_cta, a.d_out);
  if (n > 16)
    lora_tile<T, WIDE, 2, STEPS>(a, row, n, ad, c0, c1, part, frag);
  else
    lora_tile<T, WIDE, 1, STEPS>(a, row, n, ad, c0, c1, part, frag);
}

}  // namespace vmscan
