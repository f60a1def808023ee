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

namespace {

using namespace fc;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256;
constexpr int kRowBytes = 128;  // a KC tile's row: one k-step of a staged tile

enum Act { kNone = 0, kRelu = 1, kGelu = 2, kSilu = 3 };

__device__ __forceinline__ float act_value(int act, float z) {
  if (act == kRelu) return z > 0.0f ? z : (z != z ? z : 0.0f);
  if (act == kGelu) return 0.5f * z * (1.0f + erff(z * 0.70710678f));
  if (act == kSilu) return z / (1.0f + expf(-z));
  return z;
}

__device__ __forceinline__ float act_slope(int act, float z) {
  if (act == kRelu) return z > 0.0f ? 1.0f : (z != z ? z : 0.0f);
  if (act == kGelu)
    return 0.5f * (1.0f + erff(z * 0.70710678f)) + z * 0.39894228f * expf(-0.5f * z * z);
  if (act == kSilu) {
    const float s = 1.0f / (1.0f + expf(-z));
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

// A staged operand tile of X indices by one k-step (128 bytes of k).
//  KC: [X][128 B], 16-byte chunk c of row x at chunk c ^ (x & 7).
//  XC: [k][X], groups of 16 indices of row k at group g ^ swz(k).
template <typename T, int X, bool KC>
struct Stage {
  static constexpr int kVec = Elem<T>::kVec;
  static constexpr int kK = kRowBytes / (int)sizeof(T);  // k per staged tile
  static constexpr int kChunks = X * 8 / kThreads;       // 16-byte chunks per thread (either layout)
  static constexpr int kBytes = X * kRowBytes;
  typedef typename VecOf<T>::type vec;

  static __device__ __forceinline__ int swz(int k) {
    // the rows one read instruction touches differ in these bits
    if (sizeof(T) == 2) return ((k & 3) | ((k >> 3) & 1) << 2) & (X / 16 - 1);
    return (k >> 2) & 3 & (X / 16 - 1);
  }

  static __device__ __forceinline__ int slot(int s) {  // byte offset of this thread's chunk s
    const int q = threadIdx.x + s * kThreads;
    if (KC) return (q >> 3) * kRowBytes + (((q & 7) ^ ((q >> 3) & 7)) << 4);
    constexpr int kPerRow = X / kVec;  // chunks per k row
    const int k = q / kPerRow, c = q % kPerRow;
    constexpr int kPerGroup = 16 / kVec;
    return k * X * (int)sizeof(T) + (((c / kPerGroup) ^ swz(k)) * kPerGroup + c % kPerGroup) * 16;
  }

  // base: element (index 0 of the tile, k 0); nx / nk: indices and ks that exist from there.
  static __device__ __forceinline__ void load(vec (&r)[kChunks], const T* base, int64_t ld, int nx, int64_t nk) {
#pragma unroll
    for (int s = 0; s < kChunks; ++s) {
      const int q = threadIdx.x + s * kThreads;
      if (KC) {
        const int x = min(q >> 3, nx - 1);  // rows past the end repeat the last: their outputs are not stored
        const int k = (q & 7) * kVec;
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

  // Fragment of indices [x0, x0 + 16), k chunk-step ks (64 bytes of k: 4 chunks).
  static __device__ __forceinline__ vec frag(const char* lds, int x0, int ks) {
    const int lane = threadIdx.x & 63, g = lane >> 4;
    if (KC) {
      const int x = x0 + (lane & 15);
      return *(const vec*)(lds + x * kRowBytes + (((ks * 4 + g) ^ (x & 7)) << 4));
    }
    if constexpr (sizeof(T) == 2) {
      // the transposing read: 16 lanes read 4 k rows of 16 indices, lane i gets index i's 4 ks
      s16x8 v;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = ks * 32 + g * 8 + h * 4 + ((lane & 15) >> 2);
        const char* p = lds + k * X * 2 + (((x0 >> 4) ^ swz(k)) << 5) + (lane & 3) * 8;
        const s16x4 t = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[h * 4 + e] = t[e];
      }
      return __builtin_bit_cast(vec, v);
    } else {
      vec v;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int k = ks * 16 + g * 4 + e;
        v[e] = *(const T*)(lds + k * X * 4 + (((x0 >> 4) ^ swz(k)) << 6) + (lane & 15) * 4);
      }
      return v;
    }
  }
};

enum Kind { kForward = 0, kInput = 1, kWeight = 2 };

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
};

// 128-byte k-steps, staged through registers into two LDS buffers: the next step's
// global loads are in flight while this one's matrix instructions run.
template <typename T, int KIND, int BM, int BN>
__global__ __launch_bounds__(kThreads) void k_linear(const Args p) {
  constexpr bool kA_KC = KIND != kWeight, kB_KC = KIND == kForward;
  typedef Stage<T, BM, kA_KC> SA;
  typedef Stage<T, BN, kB_KC> SB;
  constexpr int kK = SA::kK;
  constexpr int MF = BM / 32, NF = BN / 32;  // 2 x 2 waves, 16 x 16 fragments
  __shared__ __attribute__((aligned(16))) char lds[2][SA::kBytes + SB::kBytes];

  const int ti = blockIdx.x / p.tiles_j, tj = blockIdx.x % p.tiles_j;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wi = (wave >> 1) * (BM / 2), wj = (wave & 1) * (BN / 2);
  const int64_t j0 = (int64_t)tj * BN;
  const int nj = (int)min((int64_t)BN, p.nj - j0);

  int client, ni;
  int64_t i0, nk;
  const T *a, *b;
  if (KIND == kWeight) {
    client = blockIdx.y;
    const RowTile t = p.tiles[client];
    i0 = (int64_t)ti * BM;
    ni = (int)min((int64_t)BM, p.ni - i0);
    nk = t.rows;
    a = (const T*)p.a + t.begin * p.lda + i0;
    b = (const T*)p.b + t.begin * p.ldb + j0;
  } else {
    const RowTile t = p.tiles[ti];
    client = t.client;
    i0 = t.begin;
    ni = t.rows;
    nk = p.nk;
    a = (const T*)p.a + i0 * p.lda;
    b = (const T*)p.b + client * p.b_client + (KIND == kForward ? j0 * p.ldb : j0);
  }
  const int64_t step_a = kA_KC ? kK : kK * p.lda, step_b = kB_KC ? kK : kK * p.ldb;

  f32x4 acc[MF][NF] = {};
  f32x4 colsum[MF] = {};
  const bool want_db = KIND == kWeight && p.db && tj == 0 && (wave & 1) == 0;
  typename SA::vec ones;
#pragma unroll
  for (int e = 0; e < SA::kVec; ++e) ones[e] = (T)1.0f;

  typename SA::vec ra[SA::kChunks];
  typename SB::vec rb[SB::kChunks];
  const int steps = (int)((nk + kK - 1) / kK);
  if (steps > 0) {
    SA::load(ra, a, p.lda, ni, nk);
    SB::load(rb, b, p.ldb, nj, nk);
    SA::put(ra, lds[0]);
    SB::put(rb, lds[0] + SA::kBytes);
  }
  __syncthreads();
  for (int t = 0; t < steps; ++t) {
    const bool more = t + 1 < steps;
    if (more) {
      const int64_t left = nk - (int64_t)(t + 1) * kK;
      SA::load(ra, a + (t + 1) * step_a, p.lda, ni, left);
      SB::load(rb, b + (t + 1) * step_b, p.ldb, nj, left);
    }
    const char* la = lds[t & 1];
    const char* lb = la + SA::kBytes;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      typename SA::vec fa[MF];
      typename SB::vec fb[NF];
#pragma unroll
      for (int m = 0; m < MF; ++m) fa[m] = SA::frag(la, wi + m * 16, ks);
#pragma unroll
      for (int n = 0; n < NF; ++n) fb[n] = SB::frag(lb, wj + n * 16, ks);
#pragma unroll
      for (int m = 0; m < MF; ++m)
#pragma unroll
        for (int n = 0; n < NF; ++n) acc[m][n] = mma<T>(fb[n], fa[m], acc[m][n]);
      if (want_db) {  // column sums as a product with ones: float32, in row order
#pragma unroll
        for (int m = 0; m < MF; ++m) colsum[m] = mma<T>(ones, fa[m], colsum[m]);
      }
    }
    if (more) {
      char* w = lds[(t + 1) & 1];
      SA::put(ra, w);
      SB::put(rb, w + SA::kBytes);
    }
    __syncthreads();
  }

  // lane: output row wi + 16 m + lane % 16, columns wj + 16 n + 4 (lane / 16) + 0..3
#pragma unroll
  for (int m = 0; m < MF; ++m) {
    const int i = wi + m * 16 + (lane & 15);
    if (i >= ni) continue;
#pragma unroll
    for (int n = 0; n < NF; ++n) {
      const int jt = wj + n * 16 + (lane >> 4) * 4;
      const int left = nj - jt;
      if (left <= 0) continue;
      const int64_t j = j0 + jt;
      f32x4 v = acc[m][n];
      if (KIND == kWeight) {
        float* o = (float*)p.out + client * p.out_client + (i0 + i) * p.ld_out + j;
        if (left >= 4) {
          VecOf<float>::loose_quad* q = (VecOf<float>::loose_quad*)o;
          *q = p.accumulate ? *q + v : v;
        } else {
#pragma unroll
          for (int e = 0; e < 3; ++e)
            if (e < left) o[e] = p.accumulate ? o[e] + v[e] : v[e];
        }
        continue;
      }
      const int64_t row = i0 + i;
      typedef typename VecOf<T>::quad quad;
      typedef typename VecOf<T>::loose_quad loose_quad;
      auto get = [&](const void* base, int64_t at) -> quad {
        const T* s = (const T*)base + at;
        quad q = {};
        if (left >= 4) {
          q = *(const loose_quad*)s;
        } else {
#pragma unroll
          for (int e = 0; e < 3; ++e)
            if (e < left) q[e] = s[e];
        }
        return q;
      };
      auto set = [&](void* base, int64_t at, quad q) {
        T* s = (T*)base + at;
        if (left >= 4) {
          *(loose_quad*)s = q;
        } else {
#pragma unroll
          for (int e = 0; e < 3; ++e)
            if (e < left) s[e] = q[e];
        }
      };
      quad o;
      if (KIND == kForward) {
        if (p.bias) {
          const quad q = get(p.bias, client * p.bias_client + j);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] += (float)q[e];
        }
        if (p.z) {
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = (T)v[e];
          set(p.z, row * p.ld_z + j, o);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = act_value(p.act, v[e]);
      } else if (p.pre) {
        const quad q = get(p.pre, row * p.ld_pre + j);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] *= act_slope(p.act, (float)q[e]);
      }
      if (p.extra) {
        const quad q = get(p.extra, row * p.ld_extra + j);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += (float)q[e];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = (T)v[e];
      set(p.out, row * p.ld_out + j, o);
    }
    if (want_db && lane < 16) {
      float* o = p.db + client * p.db_client + i0 + i;
      *o = p.accumulate ? *o + colsum[m][0] : colsum[m][0];
    }
  }
}

template <typename T, int KIND>
int launch(Args p, int32_t ntiles, hipStream_t s) {
  constexpr int BM = 128, BN = 128;
  p.tiles_j = (int32_t)((p.nj + BN - 1) / BN);
  p.tiles_i = KIND == kWeight ? (int32_t)((p.ni + BM - 1) / BM) : ntiles;
  const int64_t blocks = (int64_t)p.tiles_i * p.tiles_j;
  if (blocks > 0x7fffffffLL) return fc_internal_fail(-1, "too many tiles");
  hipLaunchKernelGGL((k_linear<T, KIND, BM, BN>), dim3((unsigned)blocks, KIND == kWeight ? p.nclients : 1),
                     dim3(kThreads), 0, s, p);
  return fc_internal_check_launch("k_linear");
}

template <int KIND>
int dispatch(int dtype, const Args& p, int32_t ntiles, hipStream_t s) {
  switch (dtype) {
    case FC_FLOAT32: return launch<float, KIND>(p, ntiles, s);
    case FC_BFLOAT16: return launch<bf16, KIND>(p, ntiles, s);
    case FC_FLOAT16: return launch<f16, KIND>(p, ntiles, s);
  }
  return fc_internal_fail(-1, "bad dtype");
}

}  // namespace

extern "C" {

int fc_linear(const void* x, int64_t x_stride, int dtype, const int32_t* tiles, int32_t ntiles, int32_t nclients,
              int64_t in_features, int64_t out_features, const void* weight, int64_t weight_client_stride,
              int64_t weight_stride, const void* bias, int64_t bias_client_stride, int activation,
              const void* residual, int64_t residual_stride, void* preactivation, int64_t preactivation_stride,
              void* y, int64_t y_stride, void* stream) {
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
  return dispatch<kForward>(dtype, p, ntiles, (hipStream_t)stream);
}

int fc_linear_backward_input(const void* dz, int64_t dz_stride, int dtype, const int32_t* tiles, int32_t ntiles,
                             int32_t nclients, int64_t in_features, int64_t out_features, const void* weight,
                             int64_t weight_client_stride, int64_t weight_stride, int activation,
                             const void* preactivation, int64_t preactivation_stride, const void* residual,
                             int64_t residual_stride, void* dx, int64_t dx_stride, void* stream) {
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
  return dispatch<kInput>(dtype, p, ntiles, (hipStream_t)stream);
}

int fc_linear_backward_weight(const void* dz, int64_t dz_stride, const void* x, int64_t x_stride, int dtype,
                              const int32_t* clients, int32_t nclients, int64_t in_features, int64_t out_features,
                              float* dweight, int64_t dweight_client_stride, int64_t dweight_stride, float* dbias,
                              int64_t dbias_client_stride, int accumulate, void* stream) {
  if (nclients <= 0 || nclients > 65535 || in_features <= 0 || out_features <= 0)
    return fc_internal_fail(-1, "bad sizes");
  if (!clients || !dweight) return fc_internal_fail(-1, "null pointer");
  Args p = {};
  p.a = dz; p.lda = dz_stride;
  p.b = x; p.ldb = x_stride;
  p.tiles = (const RowTile*)clients; p.nclients = nclients;
  p.ni = out_features; p.nj = in_features;
  p.out = dweight; p.ld_out = dweight_stride; p.out_client = dweight_client_stride;
  p.db = dbias; p.db_client = dbias_client_stride;
  p.accumulate = accumulate;
  return dispatch<kWeight>(dtype, p, 0, (hipStream_t)stream);
}

}  // extern "C"
