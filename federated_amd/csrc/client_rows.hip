// Row operators of a client's local step: layer norm with its gradients, a row's top
// logits, and the distillation loss that reads them.  Batched over a round's clients:
// rows [begin, begin + rows) of a tile belong to one client, whose parameters and
// gradients lie in its own flat row.
#include "client_common.h"

#include <algorithm>
#include <type_traits>

namespace {

using namespace fc;

constexpr float kLog2e = 1.44269504f;

// ---------------------------------------------------------------------------
// Layer norm
//   y = (x - mu) s g_c + b_c,  s = 1 / sqrt(var + eps)
//   dx = s (a - mean(a) - xh mean(a xh)) + residual,  a = dy g_c, xh = (x - mu) s
//   dg_c = sum_r dy xh,  db_c = sum_r dy
// ---------------------------------------------------------------------------

// Sum of v over the TPR threads of a row group; TPR > 64 spans whole waves of the
// block through `slot` (TPR / 64 floats per value, alternating buffers: one barrier).
template <int TPR, int NVAL>
__device__ __forceinline__ void group_sum(float (&v)[NVAL], float* slot) {
#pragma unroll
  for (int i = 0; i < NVAL; ++i) v[i] = wave_sum(v[i]);
  if constexpr (TPR > 64) {
    constexpr int W = TPR / 64;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < NVAL; ++i) slot[i * W + (threadIdx.x >> 6)] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NVAL; ++i) {
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) s += slot[i * W + w];
      v[i] = s;
    }
  }
}

struct NormArgs {
  const void *x, *weight, *bias, *dy, *residual;
  int64_t ld_x, ld_w, ld_b, ld_dy, ld_res, ld_out;
  const RowTile* tiles;
  int32_t ntiles;
  int32_t dim;
  float eps;
  void* out;
  float *mean, *rstd;
  float* part;  // [ntiles][2][dim]
};

// TPR threads per row, NV vectors of VEC elements per thread: the row stays in registers, the next
// row's are on their way while this one is summed, and the client's weights stay too.  Bound
// by memory: one read and one write (backward: two and one).  A row's last vector is read
// where it ends, so that no lane goes element by element (2500 bfloat16 elements, backward:
// 564 us with such a tail, 321 without).
template <typename T, int TPR, int NV, int VEC>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void k_norm(const NormArgs p) {
  constexpr int G = TPR > 256 ? 1 : 256 / TPR;
  typedef typename VecOf<T, VEC>::type vec;
  __shared__ float slots[2][2 * (TPR > 64 ? TPR / 64 : 1)];
  const RowTile t = p.tiles[blockIdx.x];
  const int lane = threadIdx.x % TPR, g = threadIdx.x / TPR;
  const float inv = 1.0f / (float)p.dim;
  vec gw[NV], gb[NV], next[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + lane) * VEC;
    gw[i] = gb[i] = vec{};
    if (p.weight) {
      gw[i] = settle<T, VEC>(load_columns<T, VEC>((const T*)p.weight + t.client * p.ld_w, c, p.dim), c, p.dim);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) gw[i][e] = (T)1.0f;
    }
    if (p.bias) gb[i] = settle<T, VEC>(load_columns<T, VEC>((const T*)p.bias + t.client * p.ld_b, c, p.dim), c, p.dim);
    next[i] = load_columns<T, VEC>((const T*)p.x + (t.begin + min(g, t.rows - 1)) * p.ld_x, c, p.dim);
  }
  // every group walks the same number of rows: barriers are uniform
  for (int r = 0; r < t.rows; r += G) {
    const int64_t row = t.begin + min(r + g, t.rows - 1);
    const bool live = r + g < t.rows;
    vec v[NV];
    float f[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = settle<T, VEC>(next[i], (i * TPR + lane) * VEC, p.dim);
    if (r + G < t.rows) {
      const T* x = (const T*)p.x + (t.begin + min(r + G + g, t.rows - 1)) * p.ld_x;
#pragma unroll
      for (int i = 0; i < NV; ++i) next[i] = load_columns<T, VEC>(x, (i * TPR + lane) * VEC, p.dim);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[0] += (float)v[i][e];
    group_sum<TPR>(f, slots[0]);
    const float mu = f[0] * inv;
    f[0] = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = (float)v[i][e] - mu;
        f[0] += c + e < p.dim ? d * d : 0.0f;
      }
    }
    group_sum<TPR>(f, slots[1]);
    const float s = 1.0f / sqrtf(f[0] * inv + p.eps);
    if (!live) continue;
    if (lane == 0) {
      p.mean[row] = mu;
      p.rstd[row] = s;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      vec o;
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[e] = (T)(((float)v[i][e] - mu) * s * (float)gw[i][e] + (float)gb[i][e]);
      store_vec<T, VEC>((T*)p.out + row * p.ld_out + c, o, p.dim - c);
    }
  }
}

template <typename T, int TPR, int NV, int VEC>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void k_norm_backward(const NormArgs p) {
  constexpr int G = TPR > 256 ? 1 : 256 / TPR;
  typedef typename VecOf<T, VEC>::type vec;
  __shared__ float slots[2][2 * (TPR > 64 ? TPR / 64 : 1)];
  __shared__ float join[G > 1 ? TPR * VEC * NV : 1];
  const RowTile t = p.tiles[blockIdx.x];
  const int lane = threadIdx.x % TPR, g = threadIdx.x / TPR;
  const float inv = 1.0f / (float)p.dim;
  float dg[NV][VEC] = {}, db[NV][VEC] = {};
  vec gw[NV], nx[NV], nd[NV];
  float nmu, ns;
  auto fetch = [&](int r) {
    const int64_t row = t.begin + min(r + g, t.rows - 1);
    nmu = p.mean[row];
    ns = p.rstd[row];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      nx[i] = load_columns<T, VEC>((const T*)p.x + row * p.ld_x, c, p.dim);
      nd[i] = load_columns<T, VEC>((const T*)p.dy + row * p.ld_dy, c, p.dim);
    }
  };
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + lane) * VEC;
    if (p.weight) {
      gw[i] = settle<T, VEC>(load_columns<T, VEC>((const T*)p.weight + t.client * p.ld_w, c, p.dim), c, p.dim);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) gw[i][e] = (T)(c + e < p.dim ? 1.0f : 0.0f);
    }
  }
  fetch(0);
  int turn = 0;
  for (int r = 0; r < t.rows; r += G, turn ^= 1) {
    const int64_t row = t.begin + min(r + g, t.rows - 1);
    const bool live = r + g < t.rows;
    const float mu = live ? nmu : 0.0f, s = live ? ns : 0.0f;
    vec vx[NV], vd[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      // a group past the tile's rows adds zeros
      vx[i] = live ? settle<T, VEC>(nx[i], c, p.dim) : vec{};
      vd[i] = live ? settle<T, VEC>(nd[i], c, p.dim) : vec{};
    }
    if (r + G < t.rows) fetch(r + G);
    float f[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        // columns past the end have dy = weight = 0: 0 times a finite xh
        const float d = (float)vd[i][e], xh = ((float)vx[i][e] - mu) * s, a = d * (float)gw[i][e];
        f[0] += a;
        f[1] += (i * TPR + lane) * VEC + e < p.dim ? a * xh : 0.0f;
        dg[i][e] += d * xh;
        db[i][e] += d;
      }
    group_sum<TPR>(f, slots[turn]);
    const float m0 = f[0] * inv, m1 = f[1] * inv;
    if (!live) continue;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      vec res = {};
      if (p.residual) res = settle<T, VEC>(load_columns<T, VEC>((const T*)p.residual + row * p.ld_res, c, p.dim), c, p.dim);
      vec o;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float xh = ((float)vx[i][e] - mu) * s, a = (float)vd[i][e] * (float)gw[i][e];
        o[e] = (T)(s * (a - m0 - xh * m1) + (float)res[e]);
      }
      store_vec<T, VEC>((T*)p.out + row * p.ld_out + c, o, p.dim - c);
    }
  }
  if (!p.part) return;
  // the block's groups join in group order, then one partial row per tile and sum
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if constexpr (G > 1) {
      for (int turn2 = 0; turn2 < G; ++turn2) {
        __syncthreads();
        if (g == turn2) {
#pragma unroll
          for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              float& acc = which ? db[i][e] : dg[i][e];
              float* j = &join[(i * VEC + e) * TPR + lane];
              if (turn2) acc += *j;
              *j = acc;
            }
        }
      }
    }
    if (g == G - 1) {
      float* o = p.part + ((int64_t)blockIdx.x * 2 + which) * p.dim;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + lane) * VEC;
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (c + e < p.dim) o[c + e] = which ? db[i][e] : dg[i][e];
      }
    }
  }
}

// Rows longer than the registers of a block hold (the row is read once per sum), and rows
// shorter than a vector (N 1).
template <typename T, int NT, int N>
__global__ __launch_bounds__(NT) void k_norm_long(const NormArgs p) {
  typedef typename VecOf<T, N>::type vec;
  __shared__ float slots[2][2 * NT / 64];
  const RowTile t = p.tiles[blockIdx.x];
  const int first = threadIdx.x * N;
  const float inv = 1.0f / (float)p.dim;
  const T* w = (const T*)p.weight + t.client * p.ld_w;
  const T* b = (const T*)p.bias + t.client * p.ld_b;
  auto read = [&](const T* row, int c) { return settle<T, N>(load_columns<T, N>(row, c, p.dim), c, p.dim); };
  for (int r = 0; r < t.rows; ++r) {
    const int64_t row = t.begin + r;
    const T* x = (const T*)p.x + row * p.ld_x;
    float f[1] = {0.0f};
#pragma unroll 4
    for (int c = first; c < p.dim; c += NT * N) {
      const vec v = read(x, c);
#pragma unroll
      for (int e = 0; e < N; ++e) f[0] += (float)v[e];
    }
    group_sum<NT>(f, slots[0]);
    const float mu = f[0] * inv;
    f[0] = 0.0f;
#pragma unroll 4
    for (int c = first; c < p.dim; c += NT * N) {
      const vec v = read(x, c);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float d = (float)v[e] - mu;
        f[0] += c + e < p.dim ? d * d : 0.0f;
      }
    }
    group_sum<NT>(f, slots[1]);
    const float s = 1.0f / sqrtf(f[0] * inv + p.eps);
    if (threadIdx.x == 0) {
      p.mean[row] = mu;
      p.rstd[row] = s;
    }
    T* o = (T*)p.out + row * p.ld_out;
#pragma unroll 2
    for (int c = first; c < p.dim; c += NT * N) {
      vec v = read(x, c), gw = {}, gb = {};
      if (p.weight) gw = read(w, c);
      if (p.bias) gb = read(b, c);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        float y = ((float)v[e] - mu) * s;
        if (p.weight) y *= (float)gw[e];
        v[e] = (T)(y + (float)gb[e]);
      }
      store_vec<T, N>(o + c, v, p.dim - c);
    }
  }
}

template <typename T, int NT, int N>
__global__ __launch_bounds__(NT) void k_norm_backward_long(const NormArgs p) {
  typedef typename VecOf<T, N>::type vec;
  __shared__ float slots[2][2 * NT / 64];
  const RowTile t = p.tiles[blockIdx.x];
  const int first = threadIdx.x * N;
  const float inv = 1.0f / (float)p.dim;
  const T* w = (const T*)p.weight + t.client * p.ld_w;
  auto read = [&](const T* row, int c) { return settle<T, N>(load_columns<T, N>(row, c, p.dim), c, p.dim); };
  for (int r = 0; r < t.rows; ++r) {
    const int64_t row = t.begin + r;
    const T* x = (const T*)p.x + row * p.ld_x;
    const T* dy = (const T*)p.dy + row * p.ld_dy;
    const float mu = p.mean[row], s = p.rstd[row];
    float f[2] = {0.0f, 0.0f};
#pragma unroll 2
    for (int c = first; c < p.dim; c += NT * N) {
      const vec vx = read(x, c), vd = read(dy, c);
      vec gw = {};
      if (p.weight) gw = read(w, c);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float a = p.weight ? (float)vd[e] * (float)gw[e] : (float)vd[e];
        f[0] += a;
        f[1] += c + e < p.dim ? a * ((float)vx[e] - mu) * s : 0.0f;
      }
    }
    group_sum<NT>(f, slots[r & 1]);
    const float m0 = f[0] * inv, m1 = f[1] * inv;
#pragma unroll 2
    for (int c = first; c < p.dim; c += NT * N) {
      const vec vx = read(x, c), vd = read(dy, c);
      vec gw = {}, res = {};
      if (p.weight) gw = read(w, c);
      if (p.residual) res = read((const T*)p.residual + row * p.ld_res, c);
      vec o;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float a = p.weight ? (float)vd[e] * (float)gw[e] : (float)vd[e];
        o[e] = (T)(s * (a - m0 - ((float)vx[e] - mu) * s * m1) + (float)res[e]);
      }
      store_vec<T, N>((T*)p.out + row * p.ld_out + c, o, p.dim - c);
    }
  }
  if (!p.part) return;
  for (int c = first; c < p.dim; c += NT * N) {
    float dg[N] = {}, db[N] = {};
#pragma unroll 2
    for (int r = 0; r < t.rows; ++r) {
      const int64_t row = t.begin + r;
      const float mu = p.mean[row], s = p.rstd[row];
      const vec vx = read((const T*)p.x + row * p.ld_x, c), vd = read((const T*)p.dy + row * p.ld_dy, c);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        dg[e] += (float)vd[e] * ((float)vx[e] - mu) * s;
        db[e] += (float)vd[e];
      }
    }
    float* o = p.part + (int64_t)blockIdx.x * 2 * p.dim + c;
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (c + e < p.dim) {
        o[e] = dg[e];
        o[p.dim + e] = db[e];
      }
  }
}

// dg_c, db_c: the client's tiles' partial rows.  A block adds up 64 columns, its four waves
// every fourth tile each, joined in wave order.
__global__ __launch_bounds__(256) void k_norm_join(const float* part, const int32_t* first_tile, int32_t dim,
                                                   int32_t blocks, float* dw, int64_t ld_dw, float* db, int64_t ld_db,
                                                   int accumulate) {
  __shared__ float sums[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int client = blockIdx.x / blocks, c = (blockIdx.x - client * blocks) * 64 + lane, which = blockIdx.y;
  float* o = which ? db : dw;
  if (!o) return;
  const int hi = first_tile[client + 1];
  float s = 0.0f;
  if (c < dim) {
    int k = first_tile[client] + wave;
    for (; k + 28 < hi; k += 32) {
      float t[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) t[u] = part[((int64_t)(k + 4 * u) * 2 + which) * dim + c];
#pragma unroll
      for (int u = 0; u < 8; ++u) s += t[u];
    }
    for (; k < hi; k += 4) s += part[((int64_t)k * 2 + which) * dim + c];
  }
  sums[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && c < dim) {
    o += client * (which ? ld_db : ld_dw) + c;
    s = accumulate ? *o : 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) s += sums[w][lane];
    *o = s;
  }
}

// ---------------------------------------------------------------------------
// Top logits: the k largest of a row (ties to the lowest index, NaN below every
// number), and log sum exp(l / tau).
//
// One read of the row: each thread keeps its elements' maximum, running maximum and sum.
// The k-th largest of the threads' maxima is a lower bound of the k-th largest logit, so
// only the elements of the few threads whose maximum reaches it are looked at again, and
// what is at or above it is put in order: by counting for each how many are greater, a
// few hundred and more by a bitonic network (300,000 rows of 2000, k 300: 10.6 ms, counted
// 188).  When too many elements tie at the bound, it is made exact by a radix select first.  Bound by the read: 4096 rows of 131072
// (bfloat16, k 64) in 224 us, 4.8 TB/s.
// ---------------------------------------------------------------------------

// A row of n elements as N-element vectors at multiples of their size: it starts `head`
// elements into its first vector, so a row at an odd address (an odd row length) is still
// read in aligned vectors.  Offsets c count from that vector's start, `end` = head + n;
// elements outside the row come as -inf and are not stored.
template <typename T, int N>
struct Row {
  typedef typename VecOf<T, N>::type vec;
  const T* base;  // not to be read before head
  uint32_t head, end;

  __device__ __forceinline__ Row(const T* row, uint32_t n) {
    head = (uint32_t)((uintptr_t)row / sizeof(T)) % N;
    base = row - head;
    end = head + n;
  }

  __device__ __forceinline__ bool whole(uint32_t c) const { return c >= head && c + N <= end; }

  __device__ __forceinline__ vec load(uint32_t c) const {
    if (whole(c)) return *(const vec*)(base + c);
    vec v;
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = c + e >= head && c + e < end ? base[c + e] : (T)-INFINITY;
    return v;
  }

  // to another row of the same length, element 0 at `to`; PASSING: not to be kept in the
  // caches
  template <bool PASSING>
  __device__ __forceinline__ void store(T* to, uint32_t c, vec v) const {
    typedef typename VecOf<T, N>::loose loose;
    T* p = to + (int64_t)c - head;
    if (whole(c)) {
      if (PASSING) __builtin_nontemporal_store((loose)v, (loose*)p);
      else *(loose*)p = v;
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (c + e >= head && c + e < end) p[e] = v[e];
    }
  }
};

// A running maximum m of f and sum of exp2((f - c) scale), c = m (0 while nothing but -inf
// and NaN came by).  The difference comes before the scale: a row of nothing but a type's
// lowest values is a uniform one.  A NaN makes the sum NaN, and so does +inf.
struct Softmax {
  float m = -INFINITY, c = 0.0f, sum = 0.0f;

  __device__ __forceinline__ void raise(float to, float scale) {
    if (to > m) {
      sum *= m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((c - to) * scale);
      m = c = to;
    }
  }

  template <int N>
  __device__ __forceinline__ void add(const float (&f)[N], float scale) {
    float high = f[0];
#pragma unroll
    for (int e = 1; e < N; ++e) high = fmaxf(high, f[e]);
    raise(high, scale);
#pragma unroll
    for (int e = 0; e < N; ++e) sum += __builtin_amdgcn_exp2f((f[e] - c) * scale);
  }

  // log sum exp(f / tau), scale = log2(e) / tau
  __device__ __forceinline__ float lse(float inv_tau) const {
    if (m == -INFINITY) return sum == 0.0f ? -INFINITY : sum;
    return m * inv_tau + logf(sum);
  }
};

// Orders as the float does; -0 = +0; NaN lowest.
__device__ __forceinline__ uint32_t order_key(float f) {
  if (f != f) return 0;
  const uint32_t u = __float_as_uint(f + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ unsigned long long candidate(uint32_t key, int64_t c) {
  return (unsigned long long)key << 32 | (uint32_t)~(uint32_t)c;
}

template <typename T, int NT, int VEC>
__global__ __launch_bounds__(NT) void k_top_logits(const T* logits, int64_t ld, int32_t vocab, int32_t k, float inv_tau,
                                                   int32_t* index, T* values, float* lse) {
  constexpr int W = NT / 64, kProbes = 16 / W;
  constexpr int kTopCap = NT == 64 ? 512 : 2048;  // candidates put in order in LDS
  constexpr uint32_t kCounted = 256;              // up to here by counting
  typedef typename VecOf<T, VEC>::type vec;
  __shared__ uint32_t maxima[NT], active[NT];
  __shared__ unsigned long long cand[kTopCap];
  __shared__ uint32_t hist[256];
  __shared__ float red[2][W];
  __shared__ uint32_t count[2][16];
  __shared__ uint32_t bound, ncand, nactive, want, ties;
  const int64_t row = blockIdx.x;
  const T* x = logits + row * ld;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float scale = kLog2e * inv_tau;

  const Row<T, VEC> at_row(x, vocab);
  Softmax sm;
  auto add = [&](const vec& v) {
    float f[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = (float)v[e];
    sm.add(f, scale);
  };
  constexpr uint32_t kStride = NT * VEC;
  uint32_t c0 = tid * VEC;
  for (; c0 + 3 * kStride < at_row.end; c0 += 4 * kStride) {
    vec v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = at_row.load(c0 + u * kStride);
#pragma unroll
    for (int u = 0; u < 4; ++u) add(v[u]);
  }
  for (; c0 < at_row.end; c0 += kStride) add(at_row.load(c0));

  // 16-bit types: by the key's high half, from which a bfloat16's low half follows; a float16
  // keeps its last three bits there, so its bound is up to eight values low (more candidates)
  constexpr int kBits = 8 * (int)sizeof(T);
  const uint32_t best = sm.m == -INFINITY ? 0 : order_key(sm.m);  // nothing but -inf and NaN bounds nothing
  maxima[tid] = best;
  const float wm = wave_max(sm.m);
  if (lane == 0) red[0][wave] = wm;
  if (tid == 0) ncand = nactive = ties = 0;
  __syncthreads();
  float bm = red[0][0];
#pragma unroll
  for (int w = 1; w < W; ++w) bm = fmaxf(bm, red[0][w]);
  sm.raise(bm, scale);
  const float ws = wave_sum(sm.sum);
  if (lane == 0) red[1][wave] = ws;

  // the k-th largest of the maxima, four bits a round: the waves count 16 probes
  // (0 when fewer threads than k hold any)
  uint32_t t0 = 0;
  {
    uint32_t m[W];
#pragma unroll
    for (int i = 0; i < W; ++i) m[i] = maxima[i * 64 + lane];
#pragma unroll 1
    for (int shift = 28, turn = 0; shift >= 32 - kBits; shift -= 4, turn ^= 1) {
#pragma unroll
      for (int q = 0; q < kProbes; ++q) {
        const uint32_t probe = t0 | (uint32_t)(wave * kProbes + q) << shift;
        int n = 0;
#pragma unroll
        for (int i = 0; i < W; ++i) n += __popcll(__ballot(m[i] >= probe));
        if (lane == 0) count[turn][wave * kProbes + q] = n;
      }
      __syncthreads();
      const unsigned long long ok = __ballot(lane < 16 && (lane == 0 || (int)count[turn][lane & 15] >= k));
      t0 |= (uint32_t)(63 - __clzll((long long)ok)) << shift;
    }
  }
  if (bm == INFINITY) {  // the sum is NaN; the row's is +inf unless it holds a NaN
    bool nan = false;
    for (int64_t c = tid; c < vocab; c += NT) nan |= (float)x[c] != (float)x[c];
    nan = __syncthreads_or(nan);
    if (tid == 0) lse[row] = nan ? NAN : INFINITY;
  } else if (tid == 0) {
    sm.sum = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) sm.sum += red[1][w];
    lse[row] = sm.lse(inv_tau);
  }
  const int chunks = (int)((at_row.end + kStride - 1) / kStride);  // per thread
  if (best >= t0) active[atomicAdd(&nactive, 1u)] = tid;
  __syncthreads();
  const int total = (int)nactive * chunks;
  for (int q = tid; q < total; q += NT) {
    const uint32_t c = active[q / chunks] * VEC + q % chunks * kStride;
    if (c >= at_row.end) continue;
    const vec v = at_row.load(c);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const uint32_t key = order_key((float)v[e]);
      if (key < t0 || c + e < at_row.head || c + e >= at_row.end) continue;
      const uint32_t at = atomicAdd(&ncand, 1u);
      if (at < kTopCap) cand[at] = candidate(key, c + e - at_row.head);
    }
  }
  __syncthreads();
  uint32_t n = ncand;
  if (n > kTopCap) {
    // exact k-th key by four 8-bit digits, then everything above it and the first ties
    uint32_t prefix = 0, need = k;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += NT) hist[i] = 0;
      __syncthreads();
      for (int64_t c = tid; c < vocab; c += NT) {
        const uint32_t key = order_key((float)x[c]);
        if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(key >> shift) & 255], 1u);
      }
      __syncthreads();
      if (tid == 0) {
        uint32_t left = need;
        int d = 255;
        while (d > 0 && hist[d] < left) left -= hist[d--];
        want = left;
        bound = prefix | (uint32_t)d << shift;
      }
      __syncthreads();
      prefix = bound;
      need = want;
      __syncthreads();
    }
    if (tid == 0) ncand = 0;
    __syncthreads();
    // ties are taken in index order: `need` of them
    for (int64_t c1 = 0; c1 < vocab; c1 += NT) {
      const int64_t c = c1 + tid;
      const uint32_t key = c < vocab ? order_key((float)x[c]) : 0;
      const bool tie = c < vocab && key == prefix;
      if (c < vocab && key > prefix) cand[atomicAdd(&ncand, 1u)] = candidate(key, c);
      const unsigned long long b = __ballot(tie);
      if (lane == 0) hist[wave] = __popcll(b);
      __syncthreads();
      uint32_t before = ties + __popcll(b & ((1ull << lane) - 1)), all = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        if (w < wave) before += hist[w];
        all += hist[w];
      }
      if (tie && before < need) cand[atomicAdd(&ncand, 1u)] = candidate(key, c);
      __syncthreads();
      if (tid == 0) ties += all;
      __syncthreads();
    }
    n = ncand;
  }
  if (n > kCounted) {  // in falling order by a bitonic network
    uint32_t m = 2 * kCounted;
    while (m < n) m *= 2;
    for (uint32_t i = n + tid; i < m; i += NT) cand[i] = 0;  // below every candidate
    for (uint32_t size = 2; size <= m; size *= 2)
      for (uint32_t stride = size / 2; stride > 0; stride /= 2) {
        __syncthreads();
        for (uint32_t q = tid; q < m / 2; q += NT) {
          const uint32_t i = 2 * q - (q & (stride - 1)), j = i + stride;
          const unsigned long long a = cand[i], b = cand[j];
          if ((a < b) == ((i & size) == 0)) {
            cand[i] = b;
            cand[j] = a;
          }
        }
      }
    __syncthreads();
    for (int i = tid; i < k; i += NT) {
      const uint32_t at = ~(uint32_t)cand[i];
      index[row * k + i] = (int32_t)at;
      values[row * k + i] = x[at];
    }
    return;
  }
  // a candidate's rank: how many are greater, counted by 8 lanes
  for (uint32_t i0 = 0; i0 < n; i0 += NT / 8) {
    const uint32_t i = i0 + tid / 8;
    const unsigned long long mine = i < n ? cand[i] : 0;
    int rank = 0;
    for (uint32_t j = tid & 7; j < n; j += 8) rank += cand[j] > mine;
    rank += __shfl_xor(rank, 1);
    rank += __shfl_xor(rank, 2);
    rank += __shfl_xor(rank, 4);
    if (i < n && rank < k && (tid & 7) == 0) {
      const uint32_t at = ~(uint32_t)mine;
      index[row * k + rank] = (int32_t)at;
      values[row * k + rank] = x[at];
    }
  }
}

// ---------------------------------------------------------------------------
// Distillation from top logits
//   p_k = exp(t_k / tau - L), m = sum p_k;  q = softmax(s / tau)
//   loss_r = w_r tau^2 sum_k p_k (log p_k - log q_{i_k})
//   ds_j = w_r tau (m q_j - sum_{k: i_k = j} p_k)
//
// Bound by one read of the logits and one write of the gradient: 20480 rows of 10004
// (float32, k 32) in 328 us, 5.0 TB/s; 8197 of 131072 (bfloat16, k 64) in 919, 4.7 TB/s.
// ---------------------------------------------------------------------------

constexpr int kDistillMax = 1024;  // teacher entries per row

struct DistillArgs {
  const void* logits;
  int64_t ld;
  const int32_t* index;
  const float* values;  // [rows][k]
  const float* teacher_lse;
  const float* row_weights;
  const float* dloss;  // [clients]
  const int32_t* row_client;
  const int32_t* offsets;  // [clients + 1]
  int32_t vocab, k;
  float tau;
  float* row_loss;
  float* lse;   // of s / tau; out (loss) or in (gradient alone)
  void* grad;
  int64_t ld_grad;
};

// Over the block's NT threads, through `red` (NT / 64 floats of this call's own: one barrier).
template <int NT>
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = wave_sum(v);
  if (NT == 64) return v;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.0f;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) v += red[w];
  return v;
}

template <int NT>
__device__ __forceinline__ float block_max(float v, float* red) {
  v = wave_max(v);
  if (NT == 64) return v;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int w = 1; w < NT / 64; ++w) v = fmaxf(v, red[w]);
  return v;
}

// LOSS: row loss and lse; GRAD: the gradient (with LOSS unset from the saved lse).
// NV > 0: the row stays in registers, NV 16-byte vectors per thread, so that loss and
// gradient read it once; NV = 0 streams it, once per use.
template <typename T, int NT, int NV, bool LOSS, bool GRAD>
__global__ __launch_bounds__(NT) void k_distill(const DistillArgs a) {
  constexpr int VEC = Elem<T>::kVec;
  constexpr uint32_t kStride = NT * VEC;  // offsets in a row stay below 2^31: a uniform base and 32 bits
  typedef typename VecOf<T>::type vec;
  extern __shared__ int32_t entries[];  // 4 k words
  int32_t *at = entries, *lead = entries + a.k;
  float *prob = (float*)(entries + 2 * a.k), *own = (float*)(entries + 3 * a.k);
  __shared__ float red[6][NT / 64];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  const T* s = (const T*)a.logits + row * a.ld;
  T* grad = (T*)a.grad + row * a.ld_grad;
  const float inv_tau = 1.0f / a.tau, scale = kLog2e * inv_tau;
  const uint32_t first = tid * VEC;
  const Row<T, VEC> at_row(s, a.vocab);
  typedef uint32_t raw __attribute__((ext_vector_type(4)));
  raw held[NV > 0 ? NV : 1];  // packed: unpacked to float32 the row would not fit
  auto past = [&](int i) { return i * kStride >= at_row.end; };  // no thread's vector i lies in the row
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (past(i)) continue;
    held[i] = __builtin_bit_cast(raw, at_row.load(first + i * kStride));
  }
  // vector by vector, and each use unpacks it anew
  auto held_at = [&](int i) {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" : "+v"(held[i]));
    return __builtin_bit_cast(vec, held[i]);
  };
  const int client = a.row_client[row];
  const float weight = a.row_weights ? a.row_weights[row]
                                     : 1.0f / (float)(a.offsets[client + 1] - a.offsets[client]);

  // the teacher's row
  float high = -INFINITY;
  for (int i = tid; i < a.k; i += NT) {
    int32_t j = a.index[row * a.k + i];
    const float t = a.values[row * a.k + i];
    if ((uint32_t)j >= (uint32_t)a.vocab || t == -INFINITY) j = -1;
    at[i] = j;
    prob[i] = t;
    lead[i] = i;
    if (j >= 0) high = t != t ? t : fmaxf(high, t);
  }
  const bool any = __syncthreads_or(high != -INFINITY);
  if (!any || weight == 0.0f) {  // nothing to learn from: no loss, no gradient, whatever the logits
    if (LOSS && tid == 0) {
      a.row_loss[row] = 0.0f;
      if (a.lse) a.lse[row] = NAN;  // not summed: a gradient that looks at the row sums it
    }
    if (GRAD) {
      const vec zero = {};
      for (uint32_t c = first; c < at_row.end; c += kStride) at_row.template store<false>(grad, c, zero);
    }
    return;
  }
  // log p = (t - base) / tau - L
  float base = 0.0f, L;
  if (a.teacher_lse) {
    L = a.teacher_lse[row];
  } else {
    base = block_max<NT>(high, red[0]);
    float z = 0.0f;
    for (int i = tid; i < a.k; i += NT)
      if (at[i] >= 0) z += expf((prob[i] - base) * inv_tau);
    L = logf(block_sum<NT>(z, red[1]));
  }
  if (GRAD) {  // the first of the entries that share an index
    // waves take the earlier entries in turn, lanes the later ones
    for (int i = tid & 63; i < a.k; i += 64) {
      const int32_t mine = at[i];
      int best = i;
#pragma unroll 4
      for (int h = tid >> 6; h < a.k; h += NT / 64) best = at[h] == mine ? min(best, h) : best;
      if (best < i) atomicMin(&lead[i], best);
    }
  }

  // The student's softmax: q_j = exp2((s_j - c) scale) / sum.  A saved lse is c = lse tau and
  // a sum of 1, and its four roundings (m / tau twice, the sum, c) cost q a relative error of
  // |lse| 2^-22: beyond kFar (1.5e-5 in float32, as the softmax's own; an eighth of float16's
  // half step) the row is summed again.
  constexpr float kFar = sizeof(T) == 4 ? 64.0f : 256.0f;
  Softmax sm;
  float lse = LOSS ? 0.0f : a.lse[row];
  const bool scan = LOSS || !(fabsf(lse) <= kFar);
  if (scan) {
    auto unpack = [](const vec& v, float (&f)[VEC]) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] = (float)v[e];
    };
    float f[VEC];
    if constexpr (NV > 0) {
      float high = -INFINITY;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (past(i)) continue;
        unpack(held_at(i), f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) high = fmaxf(high, f[e]);
      }
      sm.raise(block_max<NT>(high, red[2]), scale);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (past(i)) continue;
        unpack(held_at(i), f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) sm.sum += __builtin_amdgcn_exp2f((f[e] - sm.c) * scale);
      }
    } else {
      uint32_t c = first;
      for (; c + 3 * kStride < at_row.end; c += 4 * kStride) {
        vec v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = at_row.load(c + u * kStride);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          unpack(v[u], f);
          sm.add(f, scale);
        }
      }
      for (; c < at_row.end; c += kStride) {
        unpack(at_row.load(c), f);
        sm.add(f, scale);
      }
      sm.raise(block_max<NT>(sm.m, red[2]), scale);
    }
    sm.sum = block_sum<NT>(sm.sum, red[3]);
    if (LOSS && tid == 0 && a.lse) a.lse[row] = sm.lse(inv_tau);
  } else {
    sm.c = lse * a.tau;
    sm.sum = 1.0f;
  }
  const bool none = sm.sum == 0.0f;  // all -inf, no student distribution: q = 0
  const float unit = none ? 0.0f : 1.0f / sm.sum;
  // q before the division by the sum
  auto part = [&](float f) { return __builtin_amdgcn_exp2f((f - sm.c) * scale); };

  // teacher entries: probability, student logit, loss
  float loss = 0.0f, mass = 0.0f;
  const float log_sum = logf(sm.sum);
  for (int i = tid; i < a.k; i += NT) {
    const int32_t j = at[i];
    float pr = 0.0f, st = 0.0f;
    if (j >= 0) {
      const float logp = (prob[i] - base) * inv_tau - L;
      pr = expf(logp);
      st = (float)s[j];
      const float logq = st == -INFINITY ? -INFINITY : (st - sm.c) * inv_tau - log_sum;
      if (LOSS && pr != 0.0f) loss += pr * (logp - logq);
    }
    prob[i] = pr;
    own[i] = st;
    mass += pr;
  }
  if (LOSS) {
    loss = block_sum<NT>(loss, red[4]);
    if (tid == 0) a.row_loss[row] = weight * a.tau * a.tau * loss;
  }
  if (!GRAD) return;
  mass = block_sum<NT>(mass, red[5]);
  float w = weight * a.tau;
  if (a.dloss) w *= a.dloss[client];
  const float wm = w * mass * unit;
  // a streamed row's gradient leaves the caches to the logits that are read again (8197 rows
  // of 131072 bfloat16: 961 us, kept 1006); of a row read once it costs up to a tenth
  constexpr bool kPassing = LOSS && NV == 0;
  auto emit = [&](const vec& v, uint32_t c) {
    vec o;
#pragma unroll
    for (int e = 0; e < VEC; ++e) o[e] = (T)(none ? 0.0f : wm * part((float)v[e]));
    at_row.template store<kPassing>(grad, c, o);
  };
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (past(i)) continue;
      emit(held_at(i), first + i * kStride);
    }
  } else {
    // backwards: what the sum read last is in the caches still
    int i = (int)((at_row.end + kStride - 1) / kStride) - 1;
    for (; i >= 3; i -= 4) {
      vec v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = at_row.load(first + (i - u) * kStride);
#pragma unroll
      for (int u = 0; u < 4; ++u) emit(v[u], first + (i - u) * kStride);
    }
    for (; i >= 0; --i) emit(at_row.load(first + i * kStride), first + i * kStride);
  }
  __syncthreads();  // the gradient's columns are written, `lead` is settled
  // the teacher's columns: the first entry of an index takes all of its entries, in order
  for (int i = tid; i < a.k; i += NT) {
    const int32_t j = at[i];
    if (j < 0 || lead[i] != i) continue;
    float pr = prob[i];
    for (int h = i + 1; h < a.k; ++h)
      if (lead[h] == i) pr += prob[h];
    grad[j] = (T)(none ? -w * pr : wm * part(own[i]) - w * pr);
  }
}

// loss_c: the client's rows, each thread a fixed set, joined in a fixed order.
__global__ __launch_bounds__(256) void k_distill_join(const float* row_loss, const int32_t* offsets, float* loss) {
  __shared__ float red[4];
  const int lo = offsets[blockIdx.x], hi = offsets[blockIdx.x + 1];
  float s = 0.0f;
  for (int r = lo + threadIdx.x; r < hi; r += 256) s += row_loss[r];
  s = block_sum<256>(s, red);
  if (threadIdx.x == 0) loss[blockIdx.x] = s;
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------

// A launch has fewer than 2^32 threads: `blocks` workgroups of NT in as many launches as
// that takes, go(first, how many).
template <int NT, typename Go>
void in_parts(int64_t blocks, Go go) {
  constexpr int64_t most = ((1LL << 32) - 1) / NT;
  for (int64_t first = 0; first < blocks; first += most) go(first, dim3((unsigned)std::min(most, blocks - first)));
}

// A norm's kernel over its tiles.
template <int NT>
void norm_go(void (*kernel)(const NormArgs), const NormArgs& all, hipStream_t s) {
  in_parts<NT>(all.ntiles, [&](int64_t first, dim3 grid) {
    NormArgs p = all;
    p.tiles += first;
    if (p.part) p.part += first * 2 * p.dim;
    hipLaunchKernelGGL(kernel, grid, dim3(NT), 0, s, p);
  });
}

template <typename T, int TPR, int NV, int VEC>
void norm_forward(const NormArgs& p, hipStream_t s) {
  norm_go<(TPR > 256 ? TPR : 256)>(k_norm<T, TPR, NV, VEC>, p, s);
}

template <typename T, int TPR, int NV, int VEC>
void norm_launch(const NormArgs& p, bool backward, hipStream_t s) {
  if (!backward) norm_forward<T, TPR, NV, VEC>(p, s);
  else norm_go<(TPR > 256 ? TPR : 256)>(k_norm_backward<T, TPR, NV, VEC>, p, s);
}

template <typename T, int NT, int N>
void norm_long(const NormArgs& p, bool backward, hipStream_t s) {
  if (backward) norm_go<NT>(k_norm_backward_long<T, NT, N>, p, s);
  else norm_go<NT>(k_norm_long<T, NT, N>, p, s);
}

template <typename T>
int norm_dispatch(const NormArgs& p, bool backward, hipStream_t s) {
  // Threads per row, vectors per thread, elements per vector.  8-byte vectors where a 16-bit
  // row fills 16-byte ones no better: more waves for the same registers, which is what
  // keeps the loads coming (backward, bfloat16, rows of 2500: 3.9 TB/s in 256 x 3 x 4, 3.3 in
  // 256 x 2 x 8; 8000: 4.1 in 1024 x 2 x 4, 3.7 in 512 x 2 x 8).  float32 takes more threads:
  // 1500 in 512 x 1 x 4 4.4 / 4.3 TB/s (forward / backward), in 256 x 2 x 4 4.3 / 3.8.
  constexpr bool wide = sizeof(T) == 4;
  const int quads = (p.dim + 3) / 4;
  if (p.dim < 4) norm_long<T, 64, 1>(p, backward, s);
  else if (quads <= 64) norm_launch<T, 64, 1, 4>(p, backward, s);
  else if (quads <= 64 * 2) norm_launch<T, 64, 2, 4>(p, backward, s);
  else if (quads <= 64 * 3) norm_launch<T, 64, 3, 4>(p, backward, s);
  else if (quads <= 64 * 4) norm_launch<T, 64, 4, 4>(p, backward, s);
  else if (quads <= 256 * 2) norm_launch<T, wide ? 512 : 256, wide ? 1 : 2, 4>(p, backward, s);
  else if (quads <= 256 * 3 && !wide) norm_launch<T, wide ? 512 : 256, wide ? 2 : 3, 4>(p, backward, s);
  else if (quads <= 512 * 2) norm_launch<T, 512, 2, 4>(p, backward, s);
  else if (quads <= 512 * 3 && !wide) norm_launch<T, wide ? 1024 : 512, wide ? 2 : 3, 4>(p, backward, s);
  else if (quads <= 1024 * 2) norm_launch<T, 1024, 2, 4>(p, backward, s);
  // Wider rows: forward in registers still (16000: 4.8 TB/s, streamed 2.7); backward, with
  // its two accumulators per column, spills there (float32: 1.1 TB/s, streamed 1.8).
  else if (quads <= 1024 * 4 && !backward) norm_forward<T, wide ? 1024 : 512, 4, Elem<T>::kVec>(p, s);
  else norm_long<T, 1024, Elem<T>::kVec>(p, backward, s);
  return fc_internal_check_launch("k_norm");
}

int norm_dtype(int dtype, const NormArgs& p, bool backward, hipStream_t s) {
  switch (dtype) {
    case FC_FLOAT32: return norm_dispatch<float>(p, backward, s);
    case FC_BFLOAT16: return norm_dispatch<bf16>(p, backward, s);
    case FC_FLOAT16: return norm_dispatch<f16>(p, backward, s);
  }
  return fc_internal_fail(-1, "bad dtype");
}

template <typename T, int NT, int NV>
void distill_go(const DistillArgs& all, int64_t rows, bool loss, hipStream_t s) {
  in_parts<NT>(rows, [&](int64_t first, dim3 grid) {
    DistillArgs a = all;
    a.logits = (const T*)a.logits + first * a.ld;
    a.index += first * a.k;
    a.values += first * a.k;
    a.row_client += first;
    if (a.teacher_lse) a.teacher_lse += first;
    if (a.row_weights) a.row_weights += first;
    if (a.row_loss) a.row_loss += first;
    if (a.lse) a.lse += first;
    if (a.grad) a.grad = (T*)a.grad + first * a.ld_grad;
    const dim3 block(NT);
    const size_t lds = 16 * (size_t)a.k;
    if constexpr (NV > 0) {
      hipLaunchKernelGGL((k_distill<T, NT, NV, true, true>), grid, block, lds, s, a);
    } else {
      if (loss && a.grad) hipLaunchKernelGGL((k_distill<T, NT, 0, true, true>), grid, block, lds, s, a);
      else if (loss) hipLaunchKernelGGL((k_distill<T, NT, 0, true, false>), grid, block, lds, s, a);
      else hipLaunchKernelGGL((k_distill<T, NT, 0, false, true>), grid, block, lds, s, a);
    }
  });
}

template <typename T>
int distill_launch(const DistillArgs& a, int64_t rows, bool loss, hipStream_t s) {
  const int64_t vecs = (a.vocab + Elem<T>::kVec - 1) / Elem<T>::kVec;
  // One wave for a short row (100,000 rows of 3000 bfloat16: 375 us, 256 threads 498);
  // loss and gradient together hold the row while it leaves registers for two blocks a
  // CU, else stream it: what 512 blocks read comes back from the last-level cache (8197
  // rows of 131072 bfloat16: 1019 us, held 1113).
  if (!loss || !a.grad) {
    if (vecs <= 512) distill_go<T, 64, 0>(a, rows, loss, s);
    else if (vecs <= 4096) distill_go<T, 256, 0>(a, rows, loss, s);
    else distill_go<T, 1024, 0>(a, rows, loss, s);
  } else if (vecs < 64 * 4) {
    distill_go<T, 64, 4>(a, rows, loss, s);
  } else if (vecs < 64 * 8) {
    distill_go<T, 64, 8>(a, rows, loss, s);
  } else if (vecs < 256 * 5) {
    distill_go<T, 256, 5>(a, rows, loss, s);
  } else if (vecs < 256 * 10) {
    distill_go<T, 256, 10>(a, rows, loss, s);
  } else if (vecs < 1024 * 4) {
    distill_go<T, 1024, 4>(a, rows, loss, s);
  } else if (vecs < 1024 * 8 && vecs >= 1024 * 7 && sizeof(T) == 4) {
    // 3e8 elements, us held / streamed: rows of 20000 541 / 491, 24000 526 / 490, 28000 497 / 497,
    // 28700 519 / 515, 30000 506 / 511, 32000 480 / 499, 32700 481 / 522
    distill_go<T, 1024, sizeof(T) == 4 ? 8 : 4>(a, rows, loss, s);
  } else {
    distill_go<T, 1024, 0>(a, rows, loss, s);
  }
  return fc_internal_check_launch("k_distill");
}

int distill_dtype(int dtype, const DistillArgs& a, int64_t rows, bool loss, hipStream_t s) {
  switch (dtype) {
    case FC_FLOAT32: return distill_launch<float>(a, rows, loss, s);
    case FC_BFLOAT16: return distill_launch<bf16>(a, rows, loss, s);
    case FC_FLOAT16: return distill_launch<f16>(a, rows, loss, s);
  }
  return fc_internal_fail(-1, "bad dtype");
}

template <typename T>
int top_launch(const void* logits, int64_t stride, int64_t rows, int64_t vocab, int32_t k, float inv_tau, int32_t* index,
               void* values, float* lse, hipStream_t s) {
  // The bound is close while there are several times as many threads with elements as k,
  // and a block is no larger than its row keeps busy (bfloat16, us): 200,000 rows of 3000, k
  // 16: 64 threads 462, 256 676; 60,000 of 10004: 256 threads 303 (k 16), 802 (200), 4063
  // (300), 4551 (1000), 1024 threads 924, 1394, 2021, 9058: where the bound is close for
  // neither, the exact select's barriers cost the larger block more.  600,000 of 1000, k 128:
  // vectors of two 4212, of eight, which leave half of the threads without, 9661.  The limits
  // at other widths (2e8 elements, 256 / 1024 threads): k 200 6000 wide 408 / 698, 32000 189 /
  // 208; k 256 1218 / 1047, 586 / 270; k 800 10004 wide 1608 / 1294, 24000 1363 / 579; k 1000
  // 1622 / 3198, 1372 / 1961: beyond 10,000 wide and between 700 and some 950 the larger
  // block would be faster.
  auto go = [&](auto threads, auto vec) {
    constexpr int NT = decltype(threads)::value, VEC = decltype(vec)::value;
    in_parts<NT>(rows, [&](int64_t first, dim3 grid) {
      hipLaunchKernelGGL((k_top_logits<T, NT, VEC>), grid, dim3(NT), 0, s, (const T*)logits + first * stride, stride,
                         (int32_t)vocab, k, inv_tau, index + first * k, (T*)values + first * k, lse + first);
    });
  };
  typedef std::integral_constant<int, Elem<T>::kVec> wide;
  if (vocab <= 4096 && k <= 32) go(std::integral_constant<int, 64>(), wide());
  else if (vocab <= 2048) go(std::integral_constant<int, 256>(), std::integral_constant<int, 2>());
  else if (vocab <= 8192 || (vocab <= 32768 && (k <= 200 || k > 700))) go(std::integral_constant<int, 256>(), wide());
  else go(std::integral_constant<int, 1024>(), wide());
  return fc_internal_check_launch("k_top_logits");
}

constexpr int64_t kMaxDim = 1 << 24;
constexpr int64_t kMaxBlocks = (1LL << 32) / 256 - 1;  // of 256 threads in one launch

bool bad_temperature(float t) { return !(t >= FC_MIN_TEMPERATURE && t <= FC_MAX_TEMPERATURE); }

}  // namespace

extern "C" {

int64_t fc_client_tiles(const int64_t* counts, int32_t nclients, int32_t tile_rows, int32_t* tiles,
                        int32_t* first_tile) {
  if (!counts || nclients <= 0 || tile_rows <= 0) return fc_internal_fail(-1, "bad batch");
  int64_t row = 0, n = 0;
  for (int32_t c = 0; c < nclients; ++c) {
    if (counts[c] < 0) return fc_internal_fail(-1, "negative row count");
    if (first_tile) first_tile[c] = (int32_t)n;
    for (int64_t r = 0; r < counts[c]; r += tile_rows, ++n) {
      if (row + r + tile_rows > 0x7fffffffLL) return fc_internal_fail(-1, "too many rows");
      if (!tiles) continue;
      tiles[4 * n] = c;
      tiles[4 * n + 1] = (int32_t)(row + r);
      tiles[4 * n + 2] = (int32_t)std::min<int64_t>(tile_rows, counts[c] - r);
      tiles[4 * n + 3] = 0;
    }
    row += counts[c];
  }
  if (first_tile) first_tile[nclients] = (int32_t)n;
  return n;
}

int fc_layer_norm(const void* x, int64_t x_stride, int dtype, const int32_t* tiles, int32_t ntiles, int64_t dim,
                  const void* weight, int64_t weight_stride, const void* bias, int64_t bias_stride, float eps,
                  void* y, int64_t y_stride, float* mean, float* rstd, void* stream) {
  if (ntiles < 0 || dim <= 0 || dim > kMaxDim) return fc_internal_fail(-1, "bad sizes");
  if (!(eps >= 0.0f)) return fc_internal_fail(-1, "bad eps");
  if (ntiles == 0) return 0;
  if (!x || !tiles || !y || !mean || !rstd) return fc_internal_fail(-1, "null pointer");
  NormArgs p = {};
  p.x = x; p.ld_x = x_stride;
  p.weight = weight; p.ld_w = weight_stride;
  p.bias = bias; p.ld_b = bias_stride;
  p.tiles = (const RowTile*)tiles; p.ntiles = ntiles;
  p.dim = (int32_t)dim; p.eps = eps;
  p.out = y; p.ld_out = y_stride; p.mean = mean; p.rstd = rstd;
  return norm_dtype(dtype, p, false, (hipStream_t)stream);
}

int fc_layer_norm_backward(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, int dtype,
                           const float* mean, const float* rstd, const int32_t* tiles, int32_t ntiles,
                           const int32_t* first_tile, int32_t nclients, int64_t dim, const void* weight,
                           int64_t weight_stride, const void* residual, int64_t residual_stride, void* dx,
                           int64_t dx_stride, float* dweight, int64_t dweight_stride, float* dbias,
                           int64_t dbias_stride, int accumulate, float* partials, void* stream) {
  if (ntiles < 0 || nclients <= 0 || dim <= 0 || dim > kMaxDim) return fc_internal_fail(-1, "bad sizes");
  const bool want = dweight || dbias;
  if (want && !first_tile) return fc_internal_fail(-1, "null pointer");
  const int64_t columns = (dim + 63) / 64;  // blocks per client that join the gradients
  if (want && nclients * columns > kMaxBlocks) return fc_internal_fail(-1, "bad sizes");
  hipStream_t s = (hipStream_t)stream;
  if (ntiles > 0) {
    if (!x || !dy || !tiles || !dx || !mean || !rstd || (want && !partials)) return fc_internal_fail(-1, "null pointer");
    NormArgs p = {};
    p.x = x; p.ld_x = x_stride;
    p.dy = dy; p.ld_dy = dy_stride;
    p.weight = weight; p.ld_w = weight_stride;
    p.residual = residual; p.ld_res = residual_stride;
    p.tiles = (const RowTile*)tiles; p.ntiles = ntiles;
    p.dim = (int32_t)dim;
    p.out = dx; p.ld_out = dx_stride;
    p.mean = const_cast<float*>(mean); p.rstd = const_cast<float*>(rstd);
    p.part = want ? partials : nullptr;
    if (const int rc = norm_dtype(dtype, p, true, s)) return rc;
  }
  if (!want) return 0;
  hipLaunchKernelGGL(k_norm_join, dim3((unsigned)(nclients * columns), 2), dim3(256), 0, s, (const float*)partials,
                     first_tile, (int32_t)dim, (int32_t)columns, dweight, dweight_stride, dbias, dbias_stride,
                     accumulate);
  return fc_internal_check_launch("k_norm_join");
}

int fc_top_logits(const void* logits, int64_t stride, int dtype, int64_t rows, int64_t vocab, int32_t k,
                  float temperature, int32_t* index, void* values, float* lse, void* stream) {
  if (rows < 0 || rows > 0x7fffffffLL || vocab <= 0 || vocab > 0x7fffffffLL - 65536) return fc_internal_fail(-1, "bad sizes");
  if (k <= 0 || k > vocab || k > FC_MAX_TOP) return fc_internal_fail(-1, "bad k");
  if (bad_temperature(temperature)) return fc_internal_fail(-1, "bad temperature");
  if (rows == 0) return 0;
  if (!logits || !index || !values || !lse) return fc_internal_fail(-1, "null pointer");
  const float inv_tau = 1.0f / temperature;
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case FC_FLOAT32: return top_launch<float>(logits, stride, rows, vocab, k, inv_tau, index, values, lse, s);
    case FC_BFLOAT16: return top_launch<bf16>(logits, stride, rows, vocab, k, inv_tau, index, values, lse, s);
    case FC_FLOAT16: return top_launch<f16>(logits, stride, rows, vocab, k, inv_tau, index, values, lse, s);
  }
  return fc_internal_fail(-1, "bad dtype");
}

int fc_distill(const void* logits, int64_t stride, int dtype, int64_t rows, int64_t vocab, const int32_t* index,
               const float* values, int32_t k, const int32_t* row_client, const int32_t* offsets, int32_t nclients,
               float temperature, const float* teacher_lse, const float* row_weights, const float* dloss,
               float* row_loss, float* lse, float* loss, void* grad, int64_t grad_stride, void* stream) {
  if (rows < 0 || rows > 0x7fffffffLL || nclients <= 0 || vocab <= 0 || vocab > 0x7fffffffLL - 65536)
    return fc_internal_fail(-1, "bad sizes");
  if (k <= 0 || k > kDistillMax) return fc_internal_fail(-1, "bad k");
  if (bad_temperature(temperature)) return fc_internal_fail(-1, "bad temperature");
  // without rows every tensor of them may be empty, its pointer null
  if (!offsets || (rows && ((!loss && !grad) || (!loss && !lse) || (loss && !row_loss))))
    return fc_internal_fail(-1, "null pointer");
  if (loss && dloss) return fc_internal_fail(-1, "dloss goes with the gradient alone");
  hipStream_t s = (hipStream_t)stream;
  if (rows > 0) {
    if (!logits || !index || !values || !row_client) return fc_internal_fail(-1, "null pointer");
    DistillArgs a = {};
    a.logits = logits; a.ld = stride;
    a.index = index; a.values = values; a.k = k;
    a.teacher_lse = teacher_lse; a.row_weights = row_weights; a.dloss = dloss;
    a.row_client = row_client; a.offsets = offsets;
    a.vocab = (int32_t)vocab; a.tau = temperature;
    a.row_loss = row_loss; a.lse = lse;
    a.grad = grad; a.ld_grad = grad_stride;
    if (const int rc = distill_dtype(dtype, a, rows, loss != nullptr, s)) return rc;
  }
  if (!loss) return 0;
  in_parts<256>(nclients, [&](int64_t first, dim3 grid) {
    hipLaunchKernelGGL(k_distill_join, grid, dim3(256), 0, s, (const float*)row_loss, offsets + first, loss + first);
  });
  return fc_internal_check_launch("k_distill_join");
}

}  // extern "C"
