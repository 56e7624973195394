// residual_device.h - what the kernels of the residual stream (norm_kernels.hip,
// embed_kernels.hip) share: runs of elements between memory and fp32, and sums over
// wavefronts.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace flagcx_amd {

typedef _Float16 h16;
typedef __bf16 b16;
typedef uint32_t raw2 __attribute__((ext_vector_type(2)));
typedef uint32_t raw4 __attribute__((ext_vector_type(4)));
typedef float float4v __attribute__((ext_vector_type(4)));

// Cache-policy bits of the buffer instructions on gfx950.  nt marks what is streamed: 3 to 4 %
// of a block end's time for its loads (and for its gradient's), 3 to 8 % for its stores.
enum : int { kAuxPlain = 0, kAuxStream = 2 };

// One row (or a part of one) as a buffer: lanes beyond its end read zeros and write
// nothing, so a row of any length needs no branches.  The address is the same in all
// lanes of a wavefront.
struct Row {
  __amdgpu_buffer_rsrc_t r;
  __device__ __forceinline__ Row(const void *p, uint32_t bytes)
      : r(__builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, (int)bytes, 0x00020000)) {}
};

// A lane's number and the number of lanes, of which the compiler knows nothing from here on:
// offsets that derive from them are computed where they are used instead of being kept in a
// register each over the whole loop.
__device__ __forceinline__ void afresh(uint32_t &lane, uint32_t &lanes) {
  lanes = __builtin_amdgcn_readfirstlane(lanes);
  __asm__ volatile("" : "+v"(lane));
  __asm__ volatile("" : "+s"(lanes));
}

// N consecutive elements of type T as they lie in memory.  A run of several elements lies on
// an 8-byte boundary if it is 8 bytes long, else on a 16-byte one; a single element on its own.
//
// A run is at most 16 bytes: a wavefront's access then covers consecutive bytes.  Runs of 32
// bytes (eight fp32 next to eight bf16) take two accesses that each touch every line of both
// halves, which costs: a block end of 16384 x 6144 with bf16 partials and an fp32 stream took
// 301 us so, 290 us with runs of four elements of both types, its gradient 359 and 345.
template <typename T, int N>
struct Run {
  static constexpr int kBytes = N * (int)sizeof(T);
  static_assert(N == 1 || kBytes == 8 || kBytes % 16 == 0, "a run is one element, 8 bytes or whole 16-byte vectors");
  alignas(N == 1 ? sizeof(T) : kBytes == 8 ? 8 : 16) T v[N];

  // from / to element skip + at of the row
  template <int AUX = kAuxPlain>
  __device__ __forceinline__ void load(const Row &row, uint32_t skip, uint32_t at) {
    const uint32_t off = (skip + at) * (uint32_t)sizeof(T);
    if constexpr (kBytes >= 16) {
      raw4 d[kBytes / 16];
#pragma unroll
      for (int i = 0; i < kBytes / 16; i++) d[i] = __builtin_amdgcn_raw_buffer_load_b128(row.r, off + 16 * i, 0, AUX);
      __builtin_memcpy(v, d, kBytes);
    } else if constexpr (kBytes == 8) {
      const raw2 d = __builtin_amdgcn_raw_buffer_load_b64(row.r, off, 0, AUX);
      __builtin_memcpy(v, &d, 8);
    } else if constexpr (kBytes == 4) {
      v[0] = __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b32(row.r, off, 0, AUX));
    } else {
      v[0] = __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b16(row.r, off, 0, AUX));
    }
  }
  template <int AUX = kAuxPlain>
  __device__ __forceinline__ void store(const Row &row, uint32_t skip, uint32_t at) const {
    const uint32_t off = (skip + at) * (uint32_t)sizeof(T);
    if constexpr (kBytes >= 16) {
      raw4 d[kBytes / 16];
      __builtin_memcpy(d, v, kBytes);
#pragma unroll
      for (int i = 0; i < kBytes / 16; i++) __builtin_amdgcn_raw_buffer_store_b128(d[i], row.r, off + 16 * i, 0, AUX);
    } else if constexpr (kBytes == 8) {
      raw2 d;
      __builtin_memcpy(&d, v, 8);
      __builtin_amdgcn_raw_buffer_store_b64(d, row.r, off, 0, AUX);
    } else if constexpr (kBytes == 4) {
      __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, v[0]), row.r, off, 0, AUX);
    } else {
      __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, v[0]), row.r, off, 0, AUX);
    }
  }
  __device__ __forceinline__ float at(int i) const { return (float)v[i]; }
  // one rounding, to nearest even (v_cvt_pk_bf16_f32, v_cvt_f16_f32)
  __device__ __forceinline__ void set(int i, float x) { v[i] = (T)x; }
};

// M runs of a vector of weights, `step` elements apart from element skip + at on, of the activations'
// type or fp32, as fp32.  All are loaded before the first is used: run by run behind a branch each
// would wait out the memory's latency.
template <typename T, int N, int M>
__device__ __forceinline__ void loadWeights(float (&w)[M][N], const void *p, bool isF32, uint32_t dim, uint32_t skip, uint32_t step,
                                            uint32_t at) {
  if (isF32) {
    const Row in(p, dim * 4u);
    Run<float, N> r[M];
#pragma unroll
    for (int m = 0; m < M; m++) r[m].load(in, skip + m * step, at);
#pragma unroll
    for (int m = 0; m < M; m++)
#pragma unroll
      for (int i = 0; i < N; i++) w[m][i] = r[m].v[i];
  } else {
    const Row in(p, dim * (uint32_t)sizeof(T));
    Run<T, N> r[M];
#pragma unroll
    for (int m = 0; m < M; m++) r[m].load(in, skip + m * step, at);
#pragma unroll
    for (int m = 0; m < M; m++)
#pragma unroll
      for (int i = 0; i < N; i++) w[m][i] = r[m].at(i);
  }
}

// x of another lane of the same row of 16 lanes (DPP control word CTRL)
template <int CTRL>
__device__ __forceinline__ float rowLane(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}

// Sum over a row of 16 lanes, in all of them.
__device__ __forceinline__ float rowSum(float x) {
  x += rowLane<0xB1>(x);  // quad_perm [1,0,3,2]
  x += rowLane<0x4E>(x);  // quad_perm [2,3,0,1]
  x += rowLane<0x141>(x); // row_half_mirror
  x += rowLane<0x140>(x); // row_mirror
  return x;
}

// Sum over the 64 lanes, the same bits in every lane: pairs, quads, eights and rows of 16
// inside the vector unit, the four rows through scalar registers - no trip through LDS.
__device__ __forceinline__ float waveSum(float x) {
  x = rowSum(x);
  const int b = __builtin_bit_cast(int, x);
  const float r0 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 0));
  const float r1 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 16));
  const float r2 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 32));
  const float r3 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 48));
  return (r0 + r1) + (r2 + r3);
}

} // namespace flagcx_amd
