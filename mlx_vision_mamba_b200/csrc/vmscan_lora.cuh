// vmscan_lora.cuh — low-rank adapters of many requests beside a shared
// projection: out_t = base_t + scale_a (x_t A_a^T) B_a^T, a = the adapter of
// row t's request (no counterpart in the reference).
//
// The host sorts the rows by adapter and cuts them into tiles of at most
// LORA_ROWS rows of one adapter (int32[4] records: first entry of the row
// list, entries, adapter or -1, 0).  A CTA forms the tile's rank-wide products
// in fp32 in shared memory and expands them into its share of the columns.
#pragma once

#include "vmscan_common.cuh"

namespace vmscan {

constexpr int LORA_ROWS = 16;
constexpr int LORA_THREADS = 128;
constexpr int LORA_RMAX = 128;

struct LoraArgs {
  const void* x;
  const void* a;      // (adapters, rank, d_in)
  const void* b;      // (adapters, d_out, rank)
  const void* base;
  void* out;
  const float* scale; // (adapters)
  const int32_t* row_index;
  const int32_t* tiles;
  int64_t ldx, ldbase, ldout;
  int rows, d_in, d_out, rank, adapters, n_index;
};

template <typename T>
__global__ void __launch_bounds__(LORA_THREADS) lora_add_kernel(const LoraArgs a, int cols_per_cta) {
  __shared__ float s[LORA_ROWS][LORA_RMAX];
  __shared__ int row[LORA_ROWS];
  const int4 tile = reinterpret_cast<const int4*>(a.tiles)[blockIdx.x];
  const int first = max(tile.x, 0);
  const int n = min(min(tile.y, LORA_ROWS), a.n_index - first);
  if (n <= 0) return;
  const int ad = tile.z < a.adapters ? tile.z : -1;
  if (ad < 0 && a.out == a.base) return;
  for (int i = threadIdx.x; i < n; i += LORA_THREADS) row[i] = min(max(a.row_index[first + i], 0), a.rows - 1);
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c0 = blockIdx.y * cols_per_cta, c1 = min(c0 + cols_per_cta, a.d_out);
  if (ad >= 0) {
    const T* A = static_cast<const T*>(a.a) + int64_t(ad) * a.rank * a.d_in;
    const float scale = a.scale[ad];
    for (int i = warp; i < n * a.rank; i += LORA_THREADS / 32) {
      const int r = i / a.rank, k = i % a.rank;
      const T* x = static_cast<const T*>(a.x) + row[r] * a.ldx;
      float acc = 0.f;
      for (int j = lane; j < a.d_in; j += 32) acc = fmaf(ld_one(x + j), ld_one(A + int64_t(k) * a.d_in + j), acc);
#pragma unroll
      for (int m = 16; m > 0; m >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, m);
      if (lane == 0) s[r][k] = scale * acc;
    }
  }
  __syncthreads();
  for (int c = c0 + threadIdx.x; c < c1; c += LORA_THREADS) {
    float acc[LORA_ROWS];
#pragma unroll
    for (int r = 0; r < LORA_ROWS; ++r)
      acc[r] = r < n ? ld_one(static_cast<const T*>(a.base) + row[r] * a.ldbase + c) : 0.f;
    if (ad >= 0) {
      const T* B = static_cast<const T*>(a.b) + (int64_t(ad) * a.d_out + c) * a.rank;
      for (int k = 0; k < a.rank; ++k) {
        const float bk = ld_one(B + k);
#pragma unroll
        for (int r = 0; r < LORA_ROWS; ++r)
          if (r < n) acc[r] = fmaf(s[r][k], bk, acc[r]);
      }
    }
#pragma unroll
    for (int r = 0; r < LORA_ROWS; ++r)
      if (r < n) {
        T* o = static_cast<T*>(a.out) + row[r] * a.ldout + c;
        if constexpr (sizeof(T) == 4)
          *o = acc[r];
        else
          *o = __float2bfloat16_rn(acc[r]);
      }
  }
}

}  // namespace vmscan
