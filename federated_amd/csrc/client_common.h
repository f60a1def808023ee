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

// N elements of T (16 bytes unless said otherwise), and the same at T's own alignment:
// parameters live at any element offset of a client's flat row, and global memory takes
// unaligned dwordx4 (at multiples of 4 bytes for nothing, at odd 16-bit elements at about
// two thirds of the rate, measured).
template <typename T, int N = Elem<T>::kVec> struct VecOf {
  typedef T type __attribute__((ext_vector_type(N)));
  typedef T loose __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};

// `valid` (<= N, may be <= 0) elements from p, zeros behind them.
template <typename T, int N = Elem<T>::kVec>
__device__ __forceinline__ typename VecOf<T, N>::type load_vec(const T* p, int64_t valid) {
  typename VecOf<T, N>::type v = {};
  if (valid >= N) {
    v = *(const typename VecOf<T, N>::loose*)p;
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e < valid) v[e] = p[e];
  }
  return v;
}

// A part vector leaves in pieces of 8, 4 and 2 bytes: three stores instead of up to seven.
template <typename T, int N = Elem<T>::kVec>
__device__ __forceinline__ void store_vec(T* p, typename VecOf<T, N>::type v, int64_t valid) {
  if (valid >= N) {
    *(typename VecOf<T, N>::loose*)p = v;
  } else if (valid > 0) {
    const int left = (int)valid;
    if constexpr (N >= 8)
      if (left & 4) {
        *(typename VecOf<T, 4>::loose*)p = __builtin_shufflevector(v, v, 0, 1, 2, 3);
        v = __builtin_shufflevector(v, v, 4, 5, 6, 7, 4, 5, 6, 7);
        p += 4;
      }
    if constexpr (N >= 4)
      if (left & 2) {
        *(typename VecOf<T, 2>::loose*)p = __builtin_shufflevector(v, v, 0, 1);
        v[0] = v[2];
        p += 2;
      }
    if (left & 1) *p = v[0];
  }
}

// Columns [c, c + N) of a row of `dim` >= N: read as the last N where they go past its end,
// with no branch, and put right by settle() where they are used (a wait for the load).
template <typename T, int N>
__device__ __forceinline__ typename VecOf<T, N>::type load_columns(const T* row, int c, int dim) {
  return *(const typename VecOf<T, N>::loose*)(row + min(c, dim - N));
}

// Those columns, zeros behind the row's end.
template <typename T, int N>
__device__ __forceinline__ typename VecOf<T, N>::type settle(typename VecOf<T, N>::type v, int c, int dim) {
  const int over = c - (dim - N);
  if (over <= 0) return v;
  const int bits = min(over, N) * 8 * (int)sizeof(T);
  if constexpr (N == 1) {
    return v;  // its one column past the end: not asked for
  } else if constexpr (N * sizeof(T) == 8) {
    const uint64_t q = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(typename VecOf<T, N>::type, bits >= 64 ? 0 : q >> bits);
  } else {
    typedef uint64_t pair __attribute__((ext_vector_type(2)));
    pair q = __builtin_bit_cast(pair, v);
    if (bits >= 128) {
      q.x = q.y = 0;
    } else if (bits >= 64) {
      q.x = q.y >> (bits - 64);
      q.y = 0;
    } else {
      q.x = q.x >> bits | q.y << (64 - bits);
      q.y >>= bits;
    }
    return __builtin_bit_cast(typename VecOf<T, N>::type, q);
  }
}

// One entry of a batch's row-tile table: rows [begin, begin + rows) of client `client`.
struct RowTile {
  int32_t client, begin, rows, pad;
};

// The DPP value of v under control CTRL: lanes it does not reach hold `old`.
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ float dpp(float old, float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, old), __builtin_bit_cast(int, v),
                                                               CTRL, ROWS, 0xf, false));
}

// Over the 64 lanes, the result in all of them: shifts inside rows of 16 lanes, then the
// rows' last lanes broadcast, and lane 63 read back (six adds, no LDS).
__device__ __forceinline__ float wave_sum(float v) {
  v += dpp<0x111>(0.0f, v);
  v += dpp<0x112>(0.0f, v);
  v += dpp<0x114>(0.0f, v);
  v += dpp<0x118>(0.0f, v);
  v += dpp<0x142, 0xa>(0.0f, v);
  v += dpp<0x143, 0xc>(0.0f, v);
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, dpp<0x111>(v, v));
  v = fmaxf(v, dpp<0x112>(v, v));
  v = fmaxf(v, dpp<0x114>(v, v));
  v = fmaxf(v, dpp<0x118>(v, v));
  v = fmaxf(v, dpp<0x142, 0xa>(v, v));
  v = fmaxf(v, dpp<0x143, 0xc>(v, v));
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

}  // namespace fc

#endif  // FEDERATED_AMD_CLIENT_COMMON_H_
