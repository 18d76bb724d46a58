// Rows of 16- and 32-bit floats in registers: eight consecutive elements a step and thread, whatever the row's
// alignment, converted to fp32 and back.  Shared by the kernels that take rows of any width.
#pragma once
#include "common.h"
#include "quant_rows.h"

namespace {

__device__ __forceinline__ uint16_t f32_to_f16(float f) {
  const _Float16 h = (_Float16)f;  // round to nearest even, overflow to infinity
  uint16_t u;
  __builtin_memcpy(&u, &h, 2);
  return u;
}

// what a value becomes in a tensor of the type, as fp32
template <int DT>
__device__ __forceinline__ float round_to(float f) {
  if constexpr (DT == OMNI_DT_BF16) return round_bf16(f);
  else if constexpr (DT == OMNI_DT_F16) return f16_to_f32(f32_to_f16(f));
  else return f;
}
template <int DT>
__device__ __forceinline__ typename Elem<DT>::T to_elem(float f) {
  if constexpr (DT == OMNI_DT_BF16) return f32_to_bf16(f);
  else if constexpr (DT == OMNI_DT_F16) return f32_to_f16(f);
  else return f;
}

// 16 bytes at the alignment of an element: one load or store instruction on this target, which has unaligned
// access to global memory switched on
template <int ALIGN>
struct __attribute__((packed, aligned(ALIGN))) Piece16 {
  v4i v;
};

// elements [8*vi, 8*vi + 8) of a row of n elements; those past the end are 0
template <int DT, bool ALIGNED>
__device__ __forceinline__ void load8(const typename Elem<DT>::T* __restrict__ row, int vi, int n, float* v) {
  typedef typename Elem<DT>::T ET;
  const ET* p = row + (size_t)vi * 8;
  if (ALIGNED || vi * 8 + 8 <= n) {
    constexpr int AL = ALIGNED ? 16 : (int)sizeof(ET);
    if constexpr (sizeof(ET) == 2) {
      const v4i raw = ((const Piece16<AL>*)p)->v;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = Elem<DT>::cvt((uint16_t)((uint32_t)raw[j] & 0xffffu));
        v[2 * j + 1] = Elem<DT>::cvt((uint16_t)((uint32_t)raw[j] >> 16));
      }
    } else {
      const v4i a = ((const Piece16<AL>*)p)[0].v, b = ((const Piece16<AL>*)p)[1].v;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[j] = __int_as_float(a[j]);
        v[4 + j] = __int_as_float(b[j]);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = vi * 8 + j < n ? Elem<DT>::cvt(p[j]) : 0.0f;
  }
}

template <int DT, bool ALIGNED>
__device__ __forceinline__ void store8(typename Elem<DT>::T* __restrict__ row, int vi, int n, const float* v) {
  typedef typename Elem<DT>::T ET;
  ET* p = row + (size_t)vi * 8;
  if (ALIGNED || vi * 8 + 8 <= n) {
    constexpr int AL = ALIGNED ? 16 : (int)sizeof(ET);
    if constexpr (sizeof(ET) == 2) {
      v4i o;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        o[j] = (int)((uint32_t)to_elem<DT>(v[2 * j]) | ((uint32_t)to_elem<DT>(v[2 * j + 1]) << 16));
      ((Piece16<AL>*)p)->v = o;
    } else {
      v4i a, b;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        a[j] = __float_as_int(v[j]);
        b[j] = __float_as_int(v[4 + j]);
      }
      ((Piece16<AL>*)p)[0].v = a;
      ((Piece16<AL>*)p)[1].v = b;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (vi * 8 + j < n) p[j] = to_elem<DT>(v[j]);
  }
}

// eight int8 values of a row whose scale is s
template <bool ALIGNED>
__device__ __forceinline__ void store_q8(int8_t* __restrict__ row, int vi, int n, const float* v, float s) {
  int8_t* p = row + (size_t)vi * 8;
  // a row of zeros, or one that holds an infinity or a NaN (its scale says so): zeros
  const bool live = s > 0.0f && s < __builtin_inff();
  uint32_t w[2] = {0, 0};
  if (live) {
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j / 4] |= ((uint32_t)(quant_i8(v[j], s) & 0xff)) << (8 * (j % 4));
  }
  if (ALIGNED || vi * 8 + 8 <= n) {
    struct __attribute__((packed, aligned(ALIGNED ? 8 : 1))) Piece8 { v2i v; };
    ((Piece8*)p)->v = v2i{(int)w[0], (int)w[1]};
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (vi * 8 + j < n) p[j] = (int8_t)(w[j / 4] >> (8 * (j % 4)));
  }
}

// sum over the block, the same in every thread: the 64 lanes of a wavefront by the butterfly, the wavefronts in
// order.  `red` holds a word per wavefront and is written by this call alone.
template <int THREADS>
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = wave_allsum_f(v);
  if ((threadIdx.x & (WAVE - 1)) == 0) red[threadIdx.x / WAVE] = v;
  __syncthreads();
  float t = red[0];
#pragma unroll
  for (int i = 1; i < THREADS / WAVE; ++i) t = t + red[i];
  return t;
}

// largest magnitude over the block, from the bit patterns of the magnitudes: they order like the values, and a NaN
// comes out above everything instead of being dropped
template <int THREADS>
__device__ __forceinline__ float block_absmax(uint32_t bits, uint32_t* red) {
  bits = wave_allmax_u32(bits);
  if ((threadIdx.x & (WAVE - 1)) == 0) red[threadIdx.x / WAVE] = bits;
  __syncthreads();
  uint32_t m = red[0];
#pragma unroll
  for (int i = 1; i < THREADS / WAVE; ++i) m = max(m, red[i]);
  return __uint_as_float(m);
}
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// a launch is a block per row of up to 1024 threads, and a grid holds fewer than 2^32 threads
constexpr int64_t ROWS_MAX = (1 << 22) - 1;

}  // namespace
