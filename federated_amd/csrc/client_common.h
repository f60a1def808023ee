// Shared by the client-step operators (client_rows.hip, client_linear.hip): element
// types, unaligned vector access, row tiles and wave reductions.  gfx950 only.
#ifndef FEDERATED_AMD_CLIENT_COMMON_H_
#define FEDERATED_AMD_CLIENT_COMMON_H_

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "../../include/fedcodec.h"

// fc_last_error()'s message (fedcodec.hip); returns `code`.
extern "C" __attribute__((visibility("hidden"))) int fc_internal_fail(int code, const char* msg);
extern "C" __attribute__((visibility("hidden"))) int fc_internal_check_launch(const char* what);

namespace fc {

using bf16 = __bf16;
using f16 = _Float16;

template <typename T> struct Elem;
template <> struct Elem<float> { static constexpr int kVec = 4; };
template <> struct Elem<bf16> { static constexpr int kVec = 8; };
template <> struct Elem<f16> { static constexpr int kVec = 8; };

// 16 bytes of T, at T's own alignment: parameters live at any element offset of a
// client's flat row, and global memory takes unaligned dwordx4.
template <typename T> struct VecOf {
  typedef T type __attribute__((ext_vector_type(Elem<T>::kVec)));
  typedef T loose __attribute__((ext_vector_type(Elem<T>::kVec), aligned(sizeof(T))));
  typedef T quad __attribute__((ext_vector_type(4)));
  typedef T loose_quad __attribute__((ext_vector_type(4), aligned(sizeof(T))));
};

// `valid` (<= kVec, may be <= 0) elements from p, zeros behind them.
template <typename T>
__device__ __forceinline__ typename VecOf<T>::type load_vec(const T* p, int64_t valid) {
  typename VecOf<T>::type v = {};
  if (valid >= Elem<T>::kVec) {
    v = *(const typename VecOf<T>::loose*)p;
  } else {
#pragma unroll
    for (int e = 0; e < Elem<T>::kVec; ++e)
      if (e < valid) v[e] = p[e];
  }
  return v;
}

template <typename T>
__device__ __forceinline__ void store_vec(T* p, typename VecOf<T>::type v, int64_t valid) {
  if (valid >= Elem<T>::kVec) {
    *(typename VecOf<T>::loose*)p = v;
  } else {
#pragma unroll
    for (int e = 0; e < Elem<T>::kVec; ++e)
      if (e < valid) p[e] = v[e];
  }
}

// One entry of a batch's row-tile table: rows [begin, begin + rows) of client `client`.
struct RowTile {
  int32_t client, begin, rows, pad;
};

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
  return v;
}

}  // namespace fc

#endif  // FEDERATED_AMD_CLIENT_COMMON_H_
