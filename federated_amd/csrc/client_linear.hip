// Matrix products of a client's local step, batched over a round's clients: every
// client has its own weight W_c [M, K] (inside its flat parameter row) and its own
// rows of the activations.
//
//   forward   z = x W_c^T + b_c;  y = act(z) + residual          (rows x M, over K)
//   input     dx = (dz W_c) * act'(z_in) + residual              (rows x K, over M)
//   weight    dW_c = sum_r dz_r x_r^T, db_c = sum_r dz_r         (M x K, over the client's rows)
//
// All three are out(i, j) = sum_k A(i, k) B(j, k) with A and B read either along k
// ("KC": a row of 16-byte chunks along k) or along their own index ("XC").
#include "client_common.h"

#include <algorithm>
#include <type_traits>

namespace {

using namespace fc;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

enum Act { kNone = 0, kRelu = 1, kGelu = 2, kSilu = 3 };

// The normal distribution function Phi and exp(-z^2 / 2), with the relative error of the
// negative tail kept: Phi(-|z|) = t exp(-z^2 / 2) P(t), t = 1 / (1 + p |z| / sqrt 2), P fitted to
// erfcx(|z| / sqrt 2) / (2 t) for the least largest error relative to a multiple of 1 + z^2 (what
// the rounding of the exponential's argument costs anyway).
// float32: p = 1/2, P to within 2^-25 (1 + z^2 / 4); its relative error stays below that of
// (12 + 2 z^2) 2^-24, where 1 + erf has lost every digit by z = -5.5; no slower than erff.
// 16-bit outputs: p = 3/5, hardware exponential; below (1 + z^2) 2^-19 down to z = -13, where
// float32's exponential ends: 2^-15 at z = -4, a sixteenth of float16's half step, and 2^-11.6
// at -13, a twelfth of bfloat16's.
template <typename T>
__device__ __forceinline__ float normal_cdf(float z, float& bell) {
  float q;
  if constexpr (sizeof(T) == 4) {
    const float t = __builtin_amdgcn_rcpf(1.0f + 0.35355338f * fabsf(z));
    bell = expf(-0.5f * z * z);
    q = -0.025849622f;
    q = q * t + 0.12417259f;
    q = q * t - 0.20580198f;
    q = q * t + 0.09546222f;
    q = q * t + 0.016917551f;
    q = q * t + 0.08847369f;
    q = q * t + 0.124818854f;
    q = q * t + 0.1407379f;
    q = q * t + 0.14106877f;
    q *= t * bell;
  } else {
    const float t = __builtin_amdgcn_rcpf(1.0f + 0.42426407f * fabsf(z));
    bell = __builtin_amdgcn_exp2f(-0.72134752f * z * z);
    q = 0.059716813f;
    q = q * t - 0.23668773f;
    q = q * t + 0.25189537f;
    q = q * t + 0.07624174f;
    q = q * t + 0.18033396f;
    q = q * t + 0.16849965f;
    q *= t * bell;
  }
  return z < 0.0f ? q : 1.0f - q;
}

template <typename T>
__device__ __forceinline__ float logistic(float z) {
  if constexpr (sizeof(T) == 4) return 1.0f / (1.0f + expf(-z));
  else return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * z));
}

template <typename T>
__device__ __forceinline__ float act_value(int act, float z) {
  float bell;
  if (act == kRelu) return z > 0.0f ? z : (z != z ? z : 0.0f);
  if (act == kGelu) return z * normal_cdf<T>(z, bell);
  if (act == kSilu) return z * logistic<T>(z);
  return z;
}

template <typename T>
__device__ __forceinline__ float act_slope(int act, float z) {
  if (act == kRelu) return z > 0.0f ? 1.0f : (z != z ? z : 0.0f);
  if (act == kGelu) {
    float bell;
    const float cdf = normal_cdf<T>(z, bell);
    return cdf + z * 0.39894228f * bell;
  }
  if (act == kSilu) {
    const float s = logistic<T>(z);
    return s * (1.0f + z * (1.0f - s));
  }
  return 1.0f;
}

// acc += A B^T over one 16-byte fragment per lane: lane l holds index l % 16 and the
// fragment's k chunk l / 16.  The first operand's index lands in the registers (4
// consecutive ones per lane), so outputs are stored 4 elements at a time.
template <typename T> __device__ __forceinline__ f32x4 mma(typename VecOf<T>::type j, typename VecOf<T>::type i,
                                                           f32x4 acc);
template <> __device__ __forceinline__ f32x4 mma<bf16>(VecOf<bf16>::type j, VecOf<bf16>::type i, f32x4 acc) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(j, i, acc, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x4 mma<f16>(VecOf<f16>::type j, VecOf<f16>::type i, f32x4 acc) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(j, i, acc, 0, 0, 0);
}
// float32: element e of the four k chunks is one k-step of 4; both operands permute k alike.
template <> __device__ __forceinline__ f32x4 mma<float>(VecOf<float>::type j, VecOf<float>::type i, f32x4 acc) {
#pragma unroll
  for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(j[e], i[e], acc, 0, 0, 0);
  return acc;
}

// 16 bytes per lane from base + off straight to LDS (dword-aligned source): lane l's land
// at lds + 16 l.  Untracked by the compiler: the caller waits for vmcnt(0).  M0 is named as
// changed: a value of the compiler's own in it is set anew (the compiler warns that it
// would not be kept, which is what is meant).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_lds16(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds)
               : "memory", "m0");
}

__device__ __forceinline__ void load_lds16_at(const void* p, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "s"(lds) : "memory", "m0");
}
#pragma clang diagnostic pop

// The thread's number, to the compiler a new value each time: addresses made from it
// are not carried in registers through the main loop.
__device__ __forceinline__ int hidden_thread() {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));
  return t;
}

// A staged operand tile of X indices by one k-step of 128 bytes of k, NT threads.
//  KC: [X][128 bytes], 16-byte chunk c of row x at chunk c ^ turn(x).
//  XC: [k][X], groups of 16 indices of row k at group g ^ swz(k).
template <typename T, int X, bool KC, int NT>
struct Stage {
  static constexpr int ROW = 128;
  static constexpr int kVec = Elem<T>::kVec;
  static constexpr int kK = ROW / (int)sizeof(T);   // k per staged tile
  static constexpr int kPer = ROW / 16;             // chunks per KC row
  static constexpr int kChunks = X * kPer / NT;  // 16-byte chunks per thread (either layout)
  static constexpr int kBytes = X * ROW;
  typedef typename VecOf<T>::type vec;

  // A 16-byte read takes lanes {0-3, 12-15, 20-23, 24-27}, then {4-7, 8-11, 16-19, 28-31},
  // and so on in the upper half, at once (measured): their 16 chunks then cover all banks.
  static __device__ __forceinline__ int turn(int x) { return x & 7; }

  static __device__ __forceinline__ int swz(int k) {
    // the rows one read instruction touches differ in these bits
    if (sizeof(T) == 2) return ((k & 3) | ((k >> 3) & 1) << 2) & (X / 16 - 1);
    return (k >> 2) & 3 & (X / 16 - 1);
  }

  static __device__ __forceinline__ int slot(int s) {  // byte offset of this thread's chunk s
    const int q = threadIdx.x + s * NT;
    if (KC) return (q / kPer) * ROW + (((q % kPer) ^ turn(q / kPer)) << 4);
    constexpr int kPerRow = X / kVec;  // chunks per k row
    const int k = q / kPerRow, c = q % kPerRow;
    constexpr int kPerGroup = 16 / kVec;
    return k * X * (int)sizeof(T) + (((c / kPerGroup) ^ swz(k)) * kPerGroup + c % kPerGroup) * 16;
  }

  // base: element (index 0 of the tile, k 0); nx / nk: indices and ks that exist from there.
  static __device__ __forceinline__ void load(vec (&r)[kChunks], const T* base, int64_t ld, int nx, int64_t nk) {
#pragma unroll
    for (int s = 0; s < kChunks; ++s) {
      const int q = threadIdx.x + s * NT;
      if (KC) {
        const int x = min(q / kPer, nx - 1);  // rows past the end repeat the last: their outputs are not stored
        const int k = (q % kPer) * kVec;
        r[s] = load_vec(base + x * ld + k, nk - k);
      } else {
        constexpr int kPerRow = X / kVec;
        const int k = q / kPerRow, x = (q % kPerRow) * kVec;
        r[s] = load_vec(base + k * ld + x, k < nk ? (int64_t)(nx - x) : 0);
      }
    }
  }

  static __device__ __forceinline__ void put(const vec (&r)[kChunks], char* lds) {
#pragma unroll
    for (int s = 0; s < kChunks; ++s) *(vec*)(lds + slot(s)) = r[s];
  }

  // Direct to LDS: wave w's instruction s fills bytes [NT 16 s + 1024 w, + 1024) in lane
  // order, so the swizzle is applied to the source.  Byte offsets of this thread's
  // chunks from the tile's base; indices past the end repeat a valid one.  An XC tile
  // whose chunks lie a multiple of 16 ks apart (swz's period) needs the first alone.
  static constexpr int kChunkRows = KC ? NT / kPer : NT * kVec / X;
  static constexpr int kOffsets = !KC && kChunkRows % 16 == 0 ? 1 : kChunks;
  static __device__ __forceinline__ void offsets(uint32_t (&o)[kOffsets], int64_t ld, int nx) {
#pragma unroll
    for (int s = 0; s < kOffsets; ++s) {
      int x, k;
      source(s, threadIdx.x, x, k);
      if (KC) x = min(x, nx - 1);
      else if (x >= nx) x = 0;
      o[s] = (uint32_t)((KC ? x * ld + k : k * ld + x) * (int64_t)sizeof(T));
    }
  }

  // Index and k of the chunk that lands in this thread's LDS slot s.
  static __device__ __forceinline__ void source(int s, int tid, int& x, int& k) {
    const int q = tid + s * NT;
    if (KC) {
      x = q / kPer;
      k = ((q % kPer) ^ turn(x)) * kVec;
    } else {
      constexpr int kPerRow = X / kVec, kPerGroup = 16 / kVec;
      const int c = q % kPerRow;
      k = q / kPerRow;
      x = (((c / kPerGroup) ^ swz(k)) * kPerGroup + c % kPerGroup) * kVec;
    }
  }

  static __device__ __forceinline__ void direct(const uint32_t (&o)[kOffsets], const T* base, int64_t ld,
                                                const char* lds) {
    const uint32_t at = wave_base(lds);
#pragma unroll
    for (int s = 0; s < kChunks; ++s) {
      if (kOffsets == 1) load_lds16(base + s * kChunkRows * ld, o[0], at + s * NT * 16);
      else load_lds16(base, o[s], at + s * NT * 16);
    }
  }

  // direct() of the chunks whose k lies in [0, nk): the others' LDS stays as it is.
  static __device__ __forceinline__ void direct_some(const uint32_t (&o)[kOffsets], const T* base, int64_t ld,
                                                     int64_t nk, const char* lds) {
    const uint32_t at = wave_base(lds);
#pragma unroll
    for (int s = 0; s < kChunks; ++s) {
      int x, k;
      source(s, threadIdx.x, x, k);
      if (k < nk) {
        if (kOffsets == 1) load_lds16(base + s * kChunkRows * ld, o[0], at + s * NT * 16);
        else load_lds16(base, o[s], at + s * NT * 16);
      }
    }
  }

  // LDS address of this wave's first instruction in the buffer `lds`.
  static __device__ __forceinline__ uint32_t wave_base(const char* lds) {
    return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)lds +
                                          (threadIdx.x >> 6) * 1024);
  }

  // The same where k or the indices end inside the tile: part chunks go through
  // registers, ks past the end are zero.  `back`: the rows begin before `base`.  Rolled,
  // with its own addresses: few steps take it, and the main loop keeps its registers.
  static __device__ __forceinline__ void direct_edge(const T* base, int64_t ld, int nx, int64_t nk, bool back,
                                                     char* lds) {
    const uint32_t at = wave_base(lds);
    const int tid = hidden_thread();
    // elements of chunk s that exist (0: zeros; negative: past the indices, any will do), and where it is
    auto find = [&](int s, const T*& p, bool& room) -> int {
      int x, k;
      source(s, tid, x, k);
      const int valid = KC ? (int)min((int64_t)kVec, nk - k) : k < nk ? min(kVec, nx - x) : 0;
      room = (KC ? k : x) > 0 || back;
      if (KC) x = min(x, nx - 1);
      else if (x >= nx) x = 0;
      p = base + (KC ? x * ld + k : k * ld + x);
      if (!KC && k < nk && valid <= 0) return nx >= kVec ? kVec : 0;
      return max(valid, 0);
    };
    const T* p;
    bool room;
#pragma unroll 1
    for (int s = 0; s < kChunks; ++s) {
      const int valid = find(s, p, room);
      if (valid == kVec) load_lds16_at(p, at + s * NT * 16);
      else if (valid == 0) *(vec*)(lds + (tid + s * NT) * 16) = vec{};
    }
    constexpr int kAtOnce = NT == 512 && kChunks >= 2 ? 2 : kChunks;
#pragma unroll 1
    for (int s0 = 0; s0 < kChunks; s0 += kAtOnce) {
      vec r[kAtOnce];
      int valid[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        valid[u] = find(s0 + u, p, room);
        if (valid[u] > 0 && valid[u] < kVec) r[u] = load_tail(p, valid[u], room);
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u)
        if (valid[u] > 0 && valid[u] < kVec) *(vec*)(lds + (tid + (s0 + u) * NT) * 16) = r[u];
    }
    // vmcnt(0), here: a wait the compiler would else place behind, in every step's way
    __builtin_amdgcn_s_waitcnt(0x0f70);
  }

  // The last `valid` elements of a row, at p, and zeros: read as the vector that ends
  // with them where the row has `room` for it, so that one load does.
  static __device__ __forceinline__ vec load_tail(const T* p, int valid, bool room) {
    if (!room) return load_vec(p, valid);
    typedef uint64_t pair __attribute__((ext_vector_type(2)));
    pair q = __builtin_bit_cast(pair, *(const typename VecOf<T>::loose*)(p + valid - kVec));
    const int bits = (kVec - valid) * 8 * (int)sizeof(T);
    if (bits >= 64) {
      q.x = q.y >> (bits - 64);
      q.y = 0;
    } else {
      q.x = q.x >> bits | q.y << (64 - bits);
      q.y >>= bits;
    }
    return __builtin_bit_cast(vec, q);
  }

  // Column sums of an XC tile: thread t adds up the 4-byte column group t % kCols4 of
  // every kSumRows-th k row (v: one float per element of the group).
  static constexpr int kCols4 = X * (int)sizeof(T) / 4, kSumGroups = NT / kCols4;
  static __device__ __forceinline__ void add_rows(const char* lds, float (&v)[4 / sizeof(T)]) {
    typedef T group __attribute__((ext_vector_type(4 / sizeof(T))));
    const int tid = hidden_thread(), c = tid % kCols4, i = c * (4 / (int)sizeof(T));
#pragma unroll 4
    for (int k = tid / kCols4; k < kK; k += kSumGroups) {
      const group q =
          *(const group*)(lds + k * X * (int)sizeof(T) + (((i >> 4) ^ swz(k)) * 16 + (i & 15)) * (int)sizeof(T));
#pragma unroll
      for (int e = 0; e < 4 / (int)sizeof(T); ++e) v[e] += (float)q[e];
    }
  }

  // Byte offset of this lane's part of the fragment at indices x0.., first half step (64
  // bytes of k).  Fragment f further on (f 16 indices; f and x0 / 16 share no bits) and
  // the second half are at at(base, f, 1).
  static __device__ __forceinline__ uint32_t lane_base(int x0) {
    const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
    if (KC) return (x0 + r) * ROW + ((g ^ turn(x0 + r)) << 4);
    // transposing read: 16 lanes read 4 k rows of 16 indices, lane i gets index i's 4 ks
    if (sizeof(T) == 2) {
      const int k = g * 8 + (r >> 2);
      return k * X * 2 + (((x0 >> 4) ^ swz(k)) << 5) + (r & 3) * 8;
    }
    return g * 4 * X * 4 + (((x0 >> 4) ^ swz(g * 4)) << 6) + r * 4;
  }

  static __device__ __forceinline__ vec frag(const char* lds, uint32_t base, int f, int ks) {
    if (KC) return *(const vec*)(lds + (base ^ (ks << 6)) + f * 16 * ROW);
    if constexpr (sizeof(T) == 2) {
      const char* p = lds + (base ^ (f << 5)) + ks * 32 * X * 2;
      s16x8 v;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const s16x4 t =
            __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p + h * 4 * X * 2));
#pragma unroll
        for (int e = 0; e < 4; ++e) v[h * 4 + e] = t[e];
      }
      return __builtin_bit_cast(vec, v);
    } else {
      const char* p = lds + (base ^ (f << 6)) + ks * 16 * X * 4;
      vec v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = *(const T*)(p + e * X * 4);
      return v;
    }
  }
};

enum Kind { kForward = 0, kInput = 1, kWeight = 2 };

constexpr int64_t kMaxBlocks = (1LL << 32) / 256 - 1;  // a launch has fewer than 2^32 threads
constexpr int64_t kMaxSide = 1LL << 31;

struct Args {
  const void* a;       // rows operand: x (forward), dz (input, weight)
  const void* b;       // W (forward, input), x (weight)
  int64_t lda, ldb;    // row strides
  int64_t b_client;    // W's client stride
  const RowTile* tiles;  // forward, input: row tiles; weight: one entry per client (all its rows)
  int32_t nclients;
  int64_t nj, nk;      // output columns; contraction length (weight: rows, per client)
  int64_t ni;          // weight: output rows (M)
  const void* bias;    // forward
  int64_t bias_client;
  const void* extra;   // residual [rows, nj]
  int64_t ld_extra;
  const void* pre;     // input: pre-activation [rows, nj]; act' multiplies
  int64_t ld_pre;
  void* out;
  int64_t ld_out, out_client;
  void* z;             // forward: pre-activation out
  int64_t ld_z;
  float* db;           // weight
  int64_t db_client;
  int32_t accumulate;
  int32_t act;
  int32_t tiles_i, tiles_j;
  int32_t splits;      // parts of the contraction, joined through `part`
  float* part;         // [tile][split][BM BN + BM]
  int32_t walk;        // column tiles a k_linear_short block walks
};

// Workgroups go round the 8 XCDs; tiles are dealt to them kRun at a time, so that what
// an XCD's blocks read at once (8 row tiles by kRun / 8 column tiles) lies in its own
// L2, and clients of uneven size still spread over all XCDs.
__device__ __forceinline__ int xcd_order(int b, int total) {
  constexpr int kRun = 32;
  const int turn = b / (8 * kRun) * (8 * kRun);
  if (turn + 8 * kRun > total) return b;  // the last, partial turn
  const int r = b - turn;
  return turn + (r & 7) * kRun + (r >> 3);
}

__device__ __forceinline__ void tile_of(int b, int tiles_i, int tiles_j, int& ti, int& tj) {
  constexpr int kGroup = 8;
  const int per = kGroup * tiles_j, g = b / per, first = g * kGroup;
  const int rows = min(kGroup, tiles_i - first), r = b - g * per;
  ti = first + r % rows;
  tj = r / rows;
}

// Output elements of a row, columns [j, j + VEC), from float32 accumulators, the bias (or
// pre-activation) and residual vectors already read.
template <typename T, int KIND>
__device__ __forceinline__ void finish(const Args& p, float (&v)[Elem<T>::kVec], typename VecOf<T>::type bias,
                                       typename VecOf<T>::type pre, typename VecOf<T>::type extra, int64_t row,
                                       int64_t j, int left) {
  constexpr int VEC = Elem<T>::kVec;
  typename VecOf<T>::type o;
  if (KIND == kForward) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] += (float)bias[e];
    if (p.z) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[e] = (T)v[e];
      store_vec((T*)p.z + row * p.ld_z + j, o, left);
    }
    if (p.act) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = act_value<T>(p.act, v[e]);
    }
  } else if (p.pre) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] *= act_slope<T>(p.act, (float)pre[e]);
  }
  if (p.extra) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] += (float)extra[e];
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) o[e] = (T)v[e];
  store_vec((T*)p.out + row * p.ld_out + j, o, left);
}

template <int VEC>
__device__ __forceinline__ void store_weight(const Args& p, const float (&v)[VEC], int client, int64_t i, int64_t j,
                                             int left) {
  float* o = (float*)p.out + client * p.out_client + i * p.ld_out + j;
#pragma unroll
  for (int h = 0; h < VEC / 4; ++h) {
    VecOf<float>::type q = {v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]};
    if (p.accumulate) q += load_vec(o + 4 * h, left - 4 * h);
    store_vec(o + 4 * h, q, left - 4 * h);
  }
}

// Which tile of the output a workgroup makes, and of which rows and client.
struct Place {
  int client, ni, nj;   // rows and columns of the tile
  int64_t i0, j0;       // forward, input: activation row; weight: out feature
  int64_t nk;           // contraction
  int32_t row0;         // weight: the client's first row
  bool first_column;
};

template <int KIND, int BM, int BN>
__device__ __forceinline__ Place place_of(const Args& p, int b) {
  Place o;
  int ti, tj, client = 0;
  if (KIND == kWeight) {
    const int per = p.tiles_i * p.tiles_j;
    client = b / per;
    b -= client * per;
  }
  tile_of(b, p.tiles_i, p.tiles_j, ti, tj);
  const RowTile rt = p.tiles[KIND == kWeight ? client : ti];
  o.j0 = (int64_t)tj * BN;
  o.nj = (int)min((int64_t)BN, p.nj - o.j0);
  o.first_column = tj == 0;
  o.row0 = rt.begin;
  if (KIND == kWeight) {
    o.client = client;
    o.i0 = (int64_t)ti * BM;
    o.ni = (int)min((int64_t)BM, p.ni - o.i0);
    o.nk = rt.rows;
  } else {
    o.client = rt.client;
    o.i0 = rt.begin;
    o.ni = rt.rows;
    o.nk = p.nk;
  }
  return o;
}

// Bound by the matrix unit (and its power) where the contraction is long: bfloat16, 8 clients
// of 2048 rows, 4096 to 8192: 1.08 ms forward with residual and pre-activation, 1.08 input,
// 1.19 weight gradient, 1017 / 1019 / 922 TFLOP/s; the library's plain product of that size
// class reaches 1407 / 1237 / 1100 by layout.  By memory where it is short or rows are few:
// one row, 4096 to 14336: 117 MB of weight in 19 us.  Float32 products run at the unit's 153.
// Tiles: 256 x 256 loads each operand half as often as 128 x 128, 32 x 128 wastes less on
// few rows and keeps four blocks on a CU; the caller's cost model picks by their measured
// steps.  LDS reads are free of bank conflicts in every layout (counted: none).
//
// 128-byte k-steps staged to two LDS buffers: straight from memory where every address
// is a multiple of 4 bytes, else (REG: 16-bit rows of odd length) through registers.
// During a half step's products the next half's fragments are read, so a buffer is free
// half a step before its products are done: there, at the step's one barrier, the next
// buffer has landed and the load of the step after it starts.
template <typename T, int KIND, int BM, int BN, int WM, int WN, bool REG>
__global__ __launch_bounds__(WM * WN * 64, 8 / (WM * WN)) void k_linear(const Args p) {
  constexpr bool kA_KC = KIND != kWeight, kB_KC = KIND == kForward;
  constexpr int NT = WM * WN * 64;
  typedef Stage<T, BM, kA_KC, NT> SA;
  typedef Stage<T, BN, kB_KC, NT> SB;
  constexpr int kK = SA::kK, kStage = SA::kBytes + SB::kBytes, VEC = SA::kVec;
  constexpr int MF = BM / WM / 16, NF = BN / WN / 16;  // fragments per wave
  __shared__ __attribute__((aligned(1024))) char lds[2 * kStage];

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wi = wave / WN * (BM / WM), wj = wave % WN * (BN / WN);
  const int tile = xcd_order(blockIdx.x, gridDim.x);
  const Place at = place_of<KIND, BM, BN>(p, tile);
  const int ni = at.ni, nj = at.nj, client = at.client;
  const int64_t i0 = at.i0, j0 = at.j0;
  const int64_t step_a = kA_KC ? kK : kK * p.lda, step_b = kB_KC ? kK : kK * p.ldb;
  const T* pa = (const T*)p.a + (KIND == kWeight ? at.row0 * p.lda + i0 : i0 * p.lda);
  const T* pb = (const T*)p.b + (KIND == kWeight ? at.row0 * p.ldb + j0
                                                 : client * p.b_client + (KIND == kForward ? j0 * p.ldb : j0));
  int64_t nk = at.nk;
  if (p.splits > 1) {
    const int64_t per = ((nk + kK - 1) / kK + p.splits - 1) / p.splits, first = blockIdx.y * per;
    nk = max((int64_t)0, min(nk - first * kK, per * kK));
    pa += first * step_a;
    pb += first * step_b;
  }
  // An XC tile whose indices end inside a vector reads on into the next row: into columns
  // that are not stored.  The last step, with no next row, goes by the edges, and so does
  // every step where the vector would go past that row too.
  const bool edge_a = !kA_KC && ni < BM && ni % VEC, edge_b = !kB_KC && nj < BN && nj % VEC, edge = edge_a || edge_b;
  uint32_t oa[SA::kOffsets], ob[SB::kOffsets];
  if (!REG) {
    SA::offsets(oa, p.lda, ni);
    SB::offsets(ob, p.ldb, nj);
  }
  const int steps = (int)((nk + kK - 1) / kK);
  int full = (int)(nk / kK);  // steps whose loads are all direct
  if (edge) full = (edge_a && p.lda < VEC) || (edge_b && p.ldb < VEC) ? 0 : min(full, steps - 1);
  typename SA::vec ra[REG ? SA::kChunks : 1];
  typename SB::vec rb[REG ? SB::kChunks : 1];

  auto load = [&](int t) {
    char* d = lds + (t & 1) * kStage;
    const T *a = pa + t * step_a, *b = pb + t * step_b;
    const int64_t left = nk - (int64_t)t * kK;
    if constexpr (REG) {
      if (t < steps) {
        SA::load(ra, a, p.lda, ni, left);
        SB::load(rb, b, p.ldb, nj, left);
      }
    } else if (t < full) {
      SA::direct(oa, a, p.lda, d);
      SB::direct(ob, b, p.ldb, d + SA::kBytes);
    } else if (t < steps) {
      SA::direct_edge(a, p.lda, ni, left, kA_KC ? t > 0 || blockIdx.y > 0 : i0 > 0, d);
      SB::direct_edge(b, p.ldb, nj, left, kB_KC ? t > 0 || blockIdx.y > 0 : j0 > 0, d + SA::kBytes);
    }
  };
  auto put = [&](int t) {
    if constexpr (REG) {
      if (t < steps) {
        SA::put(ra, lds + (t & 1) * kStage);
        SB::put(rb, lds + (t & 1) * kStage + SA::kBytes);
      }
    }
  };
  // every wave is here, its fragments read and its loads landed
  auto arrive = []() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };

  f32x4 acc[MF][NF] = {};
  float colsum[4 / sizeof(T)] = {};  // of dz (the first column tile's blocks)
  const bool want_db = KIND == kWeight && p.db && at.first_column;
  typename SA::vec fa[2][MF];
  typename SB::vec fb[2][NF];
  uint32_t base_a = SA::lane_base(wi), base_b = SB::lane_base(wj);

  auto half = [&](auto which, const char* next) {
    constexpr int cur = decltype(which)::value, nxt = cur ^ 1;
    asm volatile("" : "+v"(base_a), "+v"(base_b));  // fragments' addresses are made as needed, not kept in registers
#pragma unroll
    for (int n = 0; n < NF; ++n) {
      fb[nxt][n] = SB::frag(next + SA::kBytes, base_b, n, nxt);
#pragma unroll
      for (int m = n * MF / NF; m < (n + 1) * MF / NF; ++m) fa[nxt][m] = SA::frag(next, base_a, m, nxt);
#pragma unroll
      for (int m = 0; m < MF; ++m) acc[m][n] = mma<T>(fb[cur][n], fa[cur][m], acc[m][n]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // this lane's columns on the way out, and their bias: there before it is needed
  constexpr int kCols = BN / WN, kLanes = kCols / VEC;
  const int jt = (lane % kLanes) * VEC, left = nj - wj - jt;
  const int64_t jg = j0 + wj + jt;
  typename VecOf<T>::type bias = {};
  if (KIND == kForward && p.bias) bias = load_vec((const T*)p.bias + client * p.bias_client + jg, left);
  if (steps > 0) {
    load(0);
    put(0);
    load(1);
    put(1);
    arrive();
#pragma unroll
    for (int m = 0; m < MF; ++m) fa[0][m] = SA::frag(lds, base_a, m, 0);
#pragma unroll
    for (int n = 0; n < NF; ++n) fb[0][n] = SB::frag(lds + SA::kBytes, base_b, n, 0);
#pragma unroll 1
    for (int t = 0; t < steps; ++t) {
      if constexpr (KIND == kWeight)
        if (want_db) SA::add_rows(lds + (t & 1) * kStage, colsum);
      half(std::integral_constant<int, 0>(), lds + (t & 1) * kStage);
      arrive();
      load(t + 2);
      half(std::integral_constant<int, 1>(), lds + (~t & 1) * kStage);
      put(t + 2);
    }
  }

  // The accumulators leave through LDS, each wave through its own part, so that global
  // memory sees whole row segments of 16 bytes per lane.
  constexpr int kRows = BM / WM, kRowB = kCols * 4, kPart = 2 * kStage / (WM * WN);
  constexpr int kFit = kPart / kRowB >= kRows ? kRows : kPart / kRowB >= 64 ? 64 : kPart / kRowB >= 32 ? 32 : 16;
  constexpr int kPass = 64 / kLanes;  // rows per read
  constexpr int kChunkMask = kCols / 4 < 16 ? kCols / 4 - 1 : 15;
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  float* part = p.part + ((int64_t)tile * p.splits + blockIdx.y) * (BM * BN + BM);
  if constexpr (KIND == kWeight) {
    if (want_db) {
      constexpr int kPer = 4 / (int)sizeof(T);
      float* sums = (float*)lds;
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        sums[threadIdx.x / SA::kCols4 * BM + threadIdx.x % SA::kCols4 * kPer + e] = colsum[e];
      __syncthreads();
      if ((int)threadIdx.x < ni) {
        float sum = 0.0f;
#pragma unroll
        for (int g = 0; g < SA::kSumGroups; ++g) sum += sums[g * BM + threadIdx.x];
        if (p.splits > 1) {
          part[BM * BN + threadIdx.x] = sum;
        } else {
          float* o = p.db + client * p.db_client + i0 + threadIdx.x;
          *o = p.accumulate ? *o + sum : sum;
        }
      }
      __syncthreads();
    }
  }
  char* mine = lds + wave * kPart;
#pragma unroll
  for (int half = 0; half < kRows / kFit; ++half) {
#pragma unroll
    for (int m = 0; m < kFit / 16; ++m)
#pragma unroll
      for (int n = 0; n < NF; ++n) {
        const int r = m * 16 + (lane & 15), c = n * 4 + (lane >> 4);
        *(f32x4*)(mine + r * kRowB + ((c ^ (r & kChunkMask)) << 4)) = acc[half * (kFit / 16) + m][n];
      }
    __builtin_amdgcn_wave_barrier();
    // kUnroll rows at a time, what they read from memory first
    constexpr int kUnroll = kFit / kPass >= 4 ? 4 : kFit / kPass;
#pragma unroll 1
    for (int r0 = lane / kLanes; r0 < kFit; r0 += kPass * kUnroll) {
      typename VecOf<T>::type pre[kUnroll] = {}, extra[kUnroll] = {};
      if (KIND != kWeight && p.splits == 1) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          const int i = wi + half * kFit + r0 + u * kPass;
          const int64_t row = i0 + i;
          if (KIND == kInput && p.pre) pre[u] = load_vec((const T*)p.pre + row * p.ld_pre + jg, i < ni ? left : 0);
          if (p.extra) extra[u] = load_vec((const T*)p.extra + row * p.ld_extra + jg, i < ni ? left : 0);
        }
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int r = r0 + u * kPass, i = wi + half * kFit + r;
        if (i >= ni || left <= 0) continue;
        float v[VEC];
#pragma unroll
        for (int h = 0; h < VEC / 4; ++h) {
          const f32x4 q = *(const f32x4*)(mine + r * kRowB + (((jt / 4 + h) ^ (r & kChunkMask)) << 4));
#pragma unroll
          for (int e = 0; e < 4; ++e) v[4 * h + e] = q[e];
        }
        if (p.splits > 1) {
          float* o = part + i * BN + wj + jt;
#pragma unroll
          for (int e = 0; e < VEC; ++e) o[e] = v[e];
        } else if (KIND == kWeight) {
          store_weight<VEC>(p, v, client, i0 + i, jg, left);
        } else {
          finish<T, KIND>(p, v, bias, pre[u], extra[u], i0 + i, jg, left);
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// A contraction of at most two 128-byte steps and many columns (an output head's forward:
// 96 to 10004), bound by its outputs' write: a block that makes one tile spends most of its
// time on its start and end (20480 rows, 64 clients, bfloat16: 287 to 318 us).  So a block
// keeps its 128 rows of A in LDS and walks along `walk` column tiles, the next one's B
// loading while this one's outputs leave: 204 us (190 in a trace), 2.1 TB/s.  What is left
// is the chain of one tile (LDS reads, products, way out) in two blocks a CU; the writes
// alone, in such tiles at rows of 20008 bytes, take 110.  In float32 the products are the
// chain, and it gains nothing (64 to 10004: 214 us in tiles, 239 walking).
template <typename T, int KIND, int STEPS>
__global__ __launch_bounds__(256, 2) void k_linear_short(const Args p) {
  constexpr bool kB_KC = KIND == kForward;
  constexpr int kTile = 128, NT = 256, MF = 4, NF = 4;
  typedef Stage<T, kTile, true, NT> SA;
  typedef Stage<T, kTile, kB_KC, NT> SB;
  constexpr int kK = SA::kK, VEC = SA::kVec, kStep = SA::kBytes;
  constexpr int kCols = 64, kFit = 16, kRowB = kCols * 4, kLanes = kCols / VEC, kPass = 64 / kLanes;
  // A's steps, B's steps, the waves' parts of the way out
  __shared__ __attribute__((aligned(1024))) char lds[2 * STEPS * kStep + 4 * kFit * kRowB];

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int wi = (wave >> 1) * 64, wj = (wave & 1) * 64;
  const int chunks = (p.tiles_j + p.walk - 1) / p.walk, block = xcd_order(blockIdx.x, gridDim.x);
  const int ti = block / chunks, first = (block - ti * chunks) * p.walk, last = min(first + p.walk, p.tiles_j);
  const RowTile rt = p.tiles[ti];
  const int ni = rt.rows;
  const int64_t i0 = rt.begin;
  const T* pb = (const T*)p.b + rt.client * p.b_client;

  // Both steps of an operand's tile.  Chunks past the contraction's end are zero from the
  // start; only part chunks go through registers.
  auto stage = [&](auto s_type, auto kc, const T* base, int64_t ld, int nx, bool before, char* d) {
    typedef typename decltype(s_type)::type S;
    constexpr bool KC = decltype(kc)::value;
    uint32_t o[S::kOffsets];
    S::offsets(o, ld, nx);
    const bool columns = !KC && nx < kTile && nx % VEC;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const T* b = base + s * (KC ? kK : kK * ld);
      const int64_t left = p.nk - s * kK;
      if (columns && (s == STEPS - 1 || ld < VEC)) S::direct_edge(b, ld, nx, left, before, d + s * kStep);
      else if (KC && left < kK && left % VEC) S::direct_edge(b, ld, nx, left, s > 0, d + s * kStep);
      else if (left < kK) S::direct_some(o, b, ld, left, d + s * kStep);
      else S::direct(o, b, ld, d + s * kStep);
    }
  };
  auto stage_b = [&](int tj) {
    const int64_t j0 = (int64_t)tj * kTile;
    stage(std::common_type<SB>(), std::integral_constant<bool, kB_KC>(), pb + (kB_KC ? j0 * p.ldb : j0), p.ldb,
          (int)min((int64_t)kTile, p.nj - j0), tj > 0, lds + STEPS * kStep);
  };
  if (p.nk % kK) {
    for (int q = tid; q < 2 * STEPS * kStep / 16; q += NT) *(typename SA::vec*)(lds + q * 16) = typename SA::vec{};
    __syncthreads();
  }
  stage(std::common_type<SA>(), std::true_type(), (const T*)p.a + i0 * p.lda, p.lda, ni, false, lds);
  stage_b(first);
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");

  const uint32_t base_a = SA::lane_base(wi), base_b = SB::lane_base(wj);
  char* mine = lds + 2 * STEPS * kStep + wave * kFit * kRowB;
  const int jt = (lane % kLanes) * VEC;
#pragma unroll 1
  for (int tj = first; tj < last; ++tj) {
    const int64_t j0 = (int64_t)tj * kTile, jg = j0 + wj + jt;
    const int left = (int)min((int64_t)kTile, p.nj - j0) - wj - jt;
    typename VecOf<T>::type bias = {};
    if (KIND == kForward && p.bias) bias = load_vec((const T*)p.bias + rt.client * p.bias_client + jg, left);
    f32x4 acc[MF][NF] = {};
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        typename SA::vec fa[MF];
        typename SB::vec fb[NF];
#pragma unroll
        for (int m = 0; m < MF; ++m) fa[m] = SA::frag(lds + s * kStep, base_a, m, h);
#pragma unroll
        for (int n = 0; n < NF; ++n) fb[n] = SB::frag(lds + (STEPS + s) * kStep, base_b, n, h);
#pragma unroll
        for (int m = 0; m < MF; ++m)
#pragma unroll
          for (int n = 0; n < NF; ++n) acc[m][n] = mma<T>(fb[n], fa[m], acc[m][n]);
      }
    // B is read
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (tj + 1 < last) stage_b(tj + 1);
    // out through the wave's own part of LDS, 16 rows at a time
#pragma unroll
    for (int m = 0; m < MF; ++m) {
#pragma unroll
      for (int n = 0; n < NF; ++n) {
        const int r = lane & 15, c = n * 4 + (lane >> 4);
        *(f32x4*)(mine + r * kRowB + ((c ^ r) << 4)) = acc[m][n];
      }
      __builtin_amdgcn_wave_barrier();
      // the next B has landed, before these outputs are in its queue
      if (m == 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
      for (int u = 0; u < kFit / kPass; ++u) {
        const int r = lane / kLanes + u * kPass, i = wi + m * 16 + r;
        const int64_t row = i0 + i;
        if (i >= ni || left <= 0) continue;
        typename VecOf<T>::type pre = {}, extra = {};
        if (KIND == kInput && p.pre) pre = load_vec((const T*)p.pre + row * p.ld_pre + jg, left);
        if (p.extra) extra = load_vec((const T*)p.extra + row * p.ld_extra + jg, left);
        float v[VEC];
#pragma unroll
        for (int h = 0; h < VEC / 4; ++h) {
          const f32x4 q = *(const f32x4*)(mine + r * kRowB + (((jt / 4 + h) ^ r) << 4));
#pragma unroll
          for (int e = 0; e < 4; ++e) v[4 * h + e] = q[e];
        }
        finish<T, KIND>(p, v, bias, pre, extra, row, jg, left);
      }
      __builtin_amdgcn_wave_barrier();
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  }
}

// A split contraction's parts, added up in their order, and the way out.
template <typename T, int KIND, int BM, int BN>
__global__ __launch_bounds__(256) void k_linear_join(const Args p) {
  constexpr int VEC = Elem<T>::kVec, kLanes = BN / VEC;
  const Place at = place_of<KIND, BM, BN>(p, blockIdx.x);
  const float* part = p.part + (int64_t)blockIdx.x * p.splits * (BM * BN + BM);
  constexpr int64_t kNext = BM * BN + BM;
  const int i = (blockIdx.y * 256 + threadIdx.x) / kLanes, jt = threadIdx.x % kLanes * VEC, left = at.nj - jt;
  if (KIND == kWeight && p.db && at.first_column && blockIdx.y == 0)
    for (int r = threadIdx.x; r < at.ni; r += 256) {
      float* o = p.db + at.client * p.db_client + at.i0 + r;
      float sum = p.accumulate ? *o : 0.0f;
      for (int s = 0; s < p.splits; ++s) sum += part[s * kNext + BM * BN + r];
      *o = sum;
    }
  if (i >= at.ni || left <= 0) return;
  float v[VEC] = {};
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) {
    const float* q = part + s * kNext + i * BN + jt;
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] += q[e];
  }
  const int64_t row = at.i0 + i, j = at.j0 + jt;
  if (KIND == kWeight) {
    store_weight<VEC>(p, v, at.client, row, j, left);
  } else {
    typename VecOf<T>::type bias = {}, pre = {}, extra = {};
    if (KIND == kForward && p.bias) bias = load_vec((const T*)p.bias + at.client * p.bias_client + j, left);
    if (KIND == kInput && p.pre) pre = load_vec((const T*)p.pre + row * p.ld_pre + j, left);
    if (p.extra) extra = load_vec((const T*)p.extra + row * p.ld_extra + j, left);
    finish<T, KIND>(p, v, bias, pre, extra, row, j, left);
  }
}

// The weight gradient of clients with few rows: what bounds it is the write of M x K
// float32, and a matrix tile's start and end (loads, LDS, way out) take longer than its
// 64 KB of writes do.  So each thread keeps R rows of its four columns of x in registers,
// reads the rows' dz of an output row from LDS (the same for a whole wave) and writes one
// 16-byte vector per output row, 4 R multiply-adds each.  More rows than R are added in
// turns.  TPR threads side by side on a row, I output rows per block.  Neighbours in memory
// are made on one XCD: rows begin anywhere in a 128-byte line, and a line that two L2s
// write in parts costs twice (6 x 3062 x 6547, one row: 140 us without, 107 with).
template <typename T, int R, int TPR, int I>
__global__ __launch_bounds__(256) void k_weight_few(const Args p) {
  constexpr int G = 256 / TPR, kPad = R + 4;
  __shared__ __attribute__((aligned(16))) float dz[I * kPad];
  const int tile = xcd_order(blockIdx.x, gridDim.x);
  const int per = p.tiles_i * p.tiles_j, client = tile / per, b = tile - client * per;
  const int ti = b / p.tiles_j, tj = b - ti * p.tiles_j, tid = threadIdx.x;
  const RowTile rt = p.tiles[client];
  const int64_t i0 = (int64_t)ti * I, j = ((int64_t)tj * TPR + tid % TPR) * 4;
  const int ni = (int)min((int64_t)I, p.ni - i0), left = (int)min((int64_t)4, p.nj - j);
  for (int r0 = 0; r0 == 0 || r0 < rt.rows; r0 += R) {
    const int rows = min(R, rt.rows - r0);
    const bool add = p.accumulate || r0 > 0;
    const T* a = (const T*)p.a + (int64_t)(rt.begin + r0) * p.lda + i0;
    const T* x = (const T*)p.b + (int64_t)(rt.begin + r0) * p.ldb + j;
    float xr[R][4];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const auto v = load_vec<T, 4>(x + r * p.ldb, r < rows ? left : 0);
#pragma unroll
      for (int e = 0; e < 4; ++e) xr[r][e] = (float)v[e];
    }
    for (int q = tid; q < I * R; q += 256) {
      const int r = q / I, i = q % I;
      dz[i * kPad + r] = r < rows && i < ni ? (float)a[r * p.lda + i] : 0.0f;
    }
    __syncthreads();
    if (p.db && tj == 0 && tid < ni) {
      float* o = p.db + client * p.db_client + i0 + tid;
      float sum = 0.0f;
#pragma unroll
      for (int r = 0; r < R; ++r) sum += dz[tid * kPad + r];
      *o = add ? *o + sum : sum;
    }
    if (left > 0) {
      for (int i = tid / TPR; i < ni; i += G) {
        float* o = (float*)p.out + client * p.out_client + (i0 + i) * p.ld_out + j;
        VecOf<float>::type v = {}, old = {};
        if (add) old = load_vec(o, left);
#pragma unroll
        for (int r = 0; r < R; r += 4) {
          const f32x4 d = *(const f32x4*)&dz[i * kPad + r];
#pragma unroll
          for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(d[u], xr[r + u][e], v[e]);
        }
        store_vec(o, v + old, left);
      }
    }
    __syncthreads();
  }
}

template <typename T, int R, int TPR, int I>
int few_launch(Args p, hipStream_t s) {
  p.tiles_i = (int32_t)((p.ni + I - 1) / I);
  p.tiles_j = (int32_t)((p.nj + 4 * TPR - 1) / (4 * TPR));
  const int64_t blocks = (int64_t)p.tiles_i * p.tiles_j * p.nclients;
  if (blocks > kMaxBlocks) return fc_internal_fail(-1, "too many tiles");
  hipLaunchKernelGGL((k_weight_few<T, R, TPR, I>), dim3((unsigned)blocks), dim3(256), 0, s, p);
  return fc_internal_check_launch("k_weight_few");
}

template <typename T>
int few_pick(const Args& p, int longest, hipStream_t s) {
  // narrow rows: 16 threads each, so that a wave writes four
  if (p.nj <= 64) return longest <= 8 ? few_launch<T, 8, 16, 256>(p, s) : few_launch<T, 16, 16, 256>(p, s);
  if constexpr (sizeof(T) == 4)  // 16-bit rows beyond 8 are better off in matrix tiles, or in turns
    if (longest > 8) return few_launch<T, 16, 64, 128>(p, s);
  return few_launch<T, 8, 64, 64>(p, s);
}

// Rows of 16-bit elements copied to a stride of whole 16-byte vectors: [clients][rows]
// [out_ld], zeros behind `cols`.  A thread per vector.
typedef f16 T16;  // a copy: 16 bits are 16 bits
__global__ __launch_bounds__(256) void k_pack_rows(const T16* src, int64_t client, int64_t ld, int32_t blocks, int64_t rows,
                                                   int32_t cols, T16* dst, int32_t out_ld) {
  constexpr int VEC = Elem<T16>::kVec;
  const int64_t which = blockIdx.x / blocks, per = out_ld / VEC;
  const int64_t q = (blockIdx.x - which * blocks) * 256 + threadIdx.x;
  if (q >= rows * per) return;
  const int64_t r = q / per;
  const int c = (int)(q - r * per) * VEC;
  const T16* from = src + which * client + r * ld + c;
  *(VecOf<T16>::type*)(dst + (which * rows + r) * out_ld + c) = load_vec(from, cols - c);
}

// Every address of the operand a multiple of 4 bytes: row stride, client stride, base.
bool dword_aligned(const void* base, int64_t ld, int64_t client, size_t size) {
  return ((uintptr_t)base | (uintptr_t)(ld * (int64_t)size) | (uintptr_t)(client * (int64_t)size)) % 4 == 0;
}

template <typename T, int KIND, int BM, int BN, int WM, int WN>
int launch(Args p, int32_t ntiles, int64_t workspace_bytes, hipStream_t s) {
  constexpr int NT = WM * WN * 64;
  if (p.ni >= kMaxSide || p.nj >= kMaxSide || p.nk >= kMaxSide) return fc_internal_fail(-1, "bad sizes");
  p.tiles_j = (int32_t)((p.nj + BN - 1) / BN);
  p.tiles_i = KIND == kWeight ? (int32_t)((p.ni + BM - 1) / BM) : ntiles;
  const int64_t blocks = (int64_t)p.tiles_i * p.tiles_j * (KIND == kWeight ? p.nclients : 1);
  if (blocks > kMaxBlocks / std::max(1, NT / 256)) return fc_internal_fail(-1, "too many tiles");
  if (p.splits > 1 && (!p.part || workspace_bytes < blocks * p.splits * (BM * BN + BM) * (int64_t)sizeof(float)))
    return fc_internal_fail(-1, "workspace too small");
  const dim3 grid((unsigned)blocks, (unsigned)p.splits), block(NT);
  const bool direct = dword_aligned(p.a, p.lda, 0, sizeof(T)) && dword_aligned(p.b, p.ldb, p.b_client, sizeof(T)) &&
                      p.lda < (1 << 22) && p.ldb < (1 << 22);  // offsets inside a tile in 32 bits
  if (direct) {
    hipLaunchKernelGGL((k_linear<T, KIND, BM, BN, WM, WN, false>), grid, block, 0, s, p);
  } else if constexpr (BM < 256) {
    hipLaunchKernelGGL((k_linear<T, KIND, BM, BN, WM, WN, true>), grid, block, 0, s, p);
  } else {
    return fc_internal_fail(-1, "256-row tiles need operands at multiples of 4 bytes");
  }
  if (const int rc = fc_internal_check_launch("k_linear")) return rc;
  if (p.splits == 1) return 0;
  hipLaunchKernelGGL((k_linear_join<T, KIND, BM, BN>), dim3((unsigned)blocks, BM * BN / Elem<T>::kVec / 256), dim3(256),
                     0, s, p);
  return fc_internal_check_launch("k_linear_join");
}

template <typename T, int KIND>
int walk(Args p, int32_t ntiles, int tile_rows, hipStream_t s) {
  if (sizeof(T) != 2 || tile_rows != 128 || p.nk * (int64_t)sizeof(T) > 256 || p.lda >= (1 << 22) || p.ldb >= (1 << 22) ||
      !dword_aligned(p.a, p.lda, 0, sizeof(T)) || !dword_aligned(p.b, p.ldb, p.b_client, sizeof(T)))
    return fc_internal_fail(-1, "splits FC_WALK: 16-bit types, tiles of 128 rows, at most 256 bytes of contraction, "
                                "operands at multiples of 4 bytes");
  if (p.nj >= kMaxSide) return fc_internal_fail(-1, "bad sizes");
  p.tiles_j = (int32_t)((p.nj + 127) / 128);
  // some four blocks for each that the chip holds, so that the last ones are short
  const int64_t total = (int64_t)ntiles * p.tiles_j;
  p.walk = (int32_t)std::min<int64_t>(std::max<int64_t>(1, total / 2048), p.tiles_j);
  const int64_t blocks = (int64_t)ntiles * ((p.tiles_j + p.walk - 1) / p.walk);
  if (blocks > kMaxBlocks) return fc_internal_fail(-1, "too many tiles");
  if constexpr (sizeof(T) == 2) {
    const dim3 grid((unsigned)blocks), block(256);
    if (p.nk * (int64_t)sizeof(T) <= 128) hipLaunchKernelGGL((k_linear_short<T, KIND, 1>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((k_linear_short<T, KIND, 2>), grid, block, 0, s, p);
  }
  return fc_internal_check_launch("k_linear_short");
}

template <typename T, int KIND>
int pick(const Args& p, int32_t ntiles, int tile_rows, int64_t workspace_bytes, hipStream_t s) {
  if constexpr (KIND != kWeight)
    if (p.splits == FC_WALK) return walk<T, KIND>(p, ntiles, tile_rows, s);
  switch (tile_rows) {
    case 32: return launch<T, KIND, 32, 128, 1, 4>(p, ntiles, workspace_bytes, s);
    case 128: return launch<T, KIND, 128, 128, 2, 2>(p, ntiles, workspace_bytes, s);
    case 256:
      if constexpr (sizeof(T) == 2) return launch<T, KIND, 256, 256, 2, 4>(p, ntiles, workspace_bytes, s);
  }
  return fc_internal_fail(-1, "bad tile_rows");
}

template <int KIND>
int dispatch(int dtype, const Args& p, int32_t ntiles, int tile_rows, int64_t workspace_bytes, hipStream_t s) {
  if ((p.splits < 1 && (KIND == kWeight || p.splits != FC_WALK)) || p.splits > 1024) return fc_internal_fail(-1, "bad splits");
  switch (dtype) {
    case FC_FLOAT32: return pick<float, KIND>(p, ntiles, tile_rows, workspace_bytes, s);
    case FC_BFLOAT16: return pick<bf16, KIND>(p, ntiles, tile_rows, workspace_bytes, s);
    case FC_FLOAT16: return pick<f16, KIND>(p, ntiles, tile_rows, workspace_bytes, s);
  }
  return fc_internal_fail(-1, "bad dtype");
}

}  // namespace

extern "C" {

int64_t fc_linear_workspace_bytes(int64_t blocks, int tile_rows, int splits) {
  if (blocks < 0 || (tile_rows != 32 && tile_rows != 128 && tile_rows != 256) || splits < 1 || splits > 1024)
    return fc_internal_fail(-1, "bad tile_rows or splits");
  const int64_t columns = tile_rows == 256 ? 256 : 128;
  return splits == 1 ? 0 : blocks * splits * (tile_rows * columns + tile_rows) * (int64_t)sizeof(float);
}

int fc_pack_rows(const void* src, int64_t client_stride, int64_t stride, int dtype, int32_t nclients, int64_t rows,
                 int64_t cols, void* dst, int64_t dst_stride, void* stream) {
  if (nclients <= 0 || rows < 0 || cols <= 0 || dst_stride < cols || dst_stride > 0x7fffffff)
    return fc_internal_fail(-1, "bad sizes");
  if (rows == 0) return 0;
  if (!src || !dst) return fc_internal_fail(-1, "null pointer");
  if (dtype != FC_BFLOAT16 && dtype != FC_FLOAT16) return fc_internal_fail(-1, "bad dtype");
  constexpr int64_t vec = Elem<T16>::kVec;
  if (dst_stride % vec || (uintptr_t)dst % 16) return fc_internal_fail(-1, "dst is not in whole 16-byte vectors");
  if (rows >= kMaxSide) return fc_internal_fail(-1, "bad sizes");
  const int64_t blocks = (rows * (dst_stride / vec) + 255) / 256;
  if (blocks > kMaxBlocks / nclients) return fc_internal_fail(-1, "too many rows");
  const dim3 grid((unsigned)(blocks * nclients));
  hipStream_t s = (hipStream_t)stream;
  hipLaunchKernelGGL(k_pack_rows, grid, dim3(256), 0, s, (const T16*)src, client_stride, stride, (int32_t)blocks, rows,
                     (int32_t)cols, (T16*)dst, (int32_t)dst_stride);
  return fc_internal_check_launch("k_pack_rows");
}

int fc_linear(const void* x, int64_t x_stride, int dtype, const int32_t* tiles, int32_t ntiles, int tile_rows,
              int32_t nclients, int64_t in_features, int64_t out_features, const void* weight,
              int64_t weight_client_stride, int64_t weight_stride, const void* bias, int64_t bias_client_stride,
              int activation, const void* residual, int64_t residual_stride, void* preactivation,
              int64_t preactivation_stride, void* y, int64_t y_stride, int splits, void* workspace, int64_t workspace_bytes, void* stream) {
  if (ntiles < 0 || nclients <= 0 || in_features <= 0 || out_features <= 0) return fc_internal_fail(-1, "bad sizes");
  if (activation < 0 || activation > 3) return fc_internal_fail(-1, "bad activation");
  if (ntiles == 0) return 0;
  if (!x || !tiles || !weight || !y) return fc_internal_fail(-1, "null pointer");
  Args p = {};
  p.a = x; p.lda = x_stride;
  p.b = weight; p.ldb = weight_stride; p.b_client = weight_client_stride;
  p.tiles = (const RowTile*)tiles; p.nclients = nclients;
  p.nj = out_features; p.nk = in_features;
  p.bias = bias; p.bias_client = bias_client_stride;
  p.extra = residual; p.ld_extra = residual_stride;
  p.z = preactivation; p.ld_z = preactivation_stride;
  p.out = y; p.ld_out = y_stride;
  p.act = activation;
  p.splits = splits; p.part = (float*)workspace;
  return dispatch<kForward>(dtype, p, ntiles, tile_rows, workspace_bytes, (hipStream_t)stream);
}

int fc_linear_backward_input(const void* dz, int64_t dz_stride, int dtype, const int32_t* tiles, int32_t ntiles,
                             int tile_rows, int32_t nclients, int64_t in_features, int64_t out_features, const void* weight,
                             int64_t weight_client_stride, int64_t weight_stride, int activation,
                             const void* preactivation, int64_t preactivation_stride, const void* residual,
                             int64_t residual_stride, void* dx, int64_t dx_stride, int splits, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  if (ntiles < 0 || nclients <= 0 || in_features <= 0 || out_features <= 0) return fc_internal_fail(-1, "bad sizes");
  if (activation < 0 || activation > 3) return fc_internal_fail(-1, "bad activation");
  if (ntiles == 0) return 0;
  if (!dz || !tiles || !weight || !dx) return fc_internal_fail(-1, "null pointer");
  Args p = {};
  p.a = dz; p.lda = dz_stride;
  p.b = weight; p.ldb = weight_stride; p.b_client = weight_client_stride;
  p.tiles = (const RowTile*)tiles; p.nclients = nclients;
  p.nj = in_features; p.nk = out_features;
  p.pre = activation ? preactivation : nullptr; p.ld_pre = preactivation_stride;
  p.extra = residual; p.ld_extra = residual_stride;
  p.out = dx; p.ld_out = dx_stride;
  p.act = activation;
  if (activation && !preactivation) return fc_internal_fail(-1, "an activation needs its pre-activation");
  p.splits = splits; p.part = (float*)workspace;
  return dispatch<kInput>(dtype, p, ntiles, tile_rows, workspace_bytes, (hipStream_t)stream);
}

int fc_linear_backward_weight(const void* dz, int64_t dz_stride, const void* x, int64_t x_stride, int dtype,
                              const int32_t* clients, int32_t nclients, int64_t in_features, int64_t out_features,
                              float* dweight, int64_t dweight_client_stride, int64_t dweight_stride, float* dbias,
                              int64_t dbias_client_stride, int accumulate, int tile_rows, int splits, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  if (nclients <= 0 || in_features <= 0 || out_features <= 0) return fc_internal_fail(-1, "bad sizes");
  if (!dz || !x || !clients || !dweight) return fc_internal_fail(-1, "null pointer");
  Args p = {};
  p.a = dz; p.lda = dz_stride;
  p.b = x; p.ldb = x_stride;
  p.tiles = (const RowTile*)clients; p.nclients = nclients;
  p.ni = out_features; p.nj = in_features;
  p.out = dweight; p.ld_out = dweight_stride; p.out_client = dweight_client_stride;
  p.db = dbias; p.db_client = dbias_client_stride;
  p.accumulate = accumulate;
  p.splits = splits; p.part = (float*)workspace;
  return dispatch<kWeight>(dtype, p, 0, tile_rows, workspace_bytes, (hipStream_t)stream);
}

int fc_linear_backward_weight_few(const void* dz, int64_t dz_stride, const void* x, int64_t x_stride, int dtype,
                                  const int32_t* clients, int32_t nclients, int64_t longest, int64_t in_features,
                                  int64_t out_features, float* dweight, int64_t dweight_client_stride,
                                  int64_t dweight_stride, float* dbias, int64_t dbias_client_stride, int accumulate,
                                  void* stream) {
  if (nclients <= 0 || longest < 0 || in_features <= 0 || out_features <= 0 || in_features >= kMaxSide ||
      out_features >= kMaxSide)
    return fc_internal_fail(-1, "bad sizes");
  if (!clients || !dweight || (longest > 0 && (!dz || !x))) return fc_internal_fail(-1, "null pointer");
  Args p = {};
  p.a = dz; p.lda = dz_stride;
  p.b = x; p.ldb = x_stride;
  p.tiles = (const RowTile*)clients; p.nclients = nclients;
  p.ni = out_features; p.nj = in_features;
  p.out = dweight; p.ld_out = dweight_stride; p.out_client = dweight_client_stride;
  p.db = dbias; p.db_client = dbias_client_stride;
  p.accumulate = accumulate;
  const int rows = (int)std::min<int64_t>(longest, 1 << 30);
  switch (dtype) {
    case FC_FLOAT32: return few_pick<float>(p, rows, (hipStream_t)stream);
    case FC_BFLOAT16: return few_pick<bf16>(p, rows, (hipStream_t)stream);
    case FC_FLOAT16: return few_pick<f16>(p, rows, (hipStream_t)stream);
  }
  return fc_internal_fail(-1, "bad dtype");
}

}  // extern "C"
