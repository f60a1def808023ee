// Row operators of a client's local step: layer norm with its gradients, a row's top
// logits, and the distillation loss that reads them.  Batched over a round's clients:
// rows [begin, begin + rows) of a tile belong to one client, whose parameters and
// gradients lie in its own flat row.
#include "client_common.h"

#include <algorithm>
#include <cmath>

namespace {

using namespace fc;

constexpr float kLog2e = 1.44269504f;
constexpr float kLn2 = 0.69314718f;

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

// TPR threads per row, NV 16-byte vectors per thread: the row stays in registers.
template <typename T, int TPR, int NV>
__global__ __launch_bounds__(256) void k_norm(const NormArgs p) {
  constexpr int VEC = Elem<T>::kVec, G = 256 / TPR;
  typedef typename VecOf<T>::type vec;
  __shared__ float slots[2][2 * 4];
  const RowTile t = p.tiles[blockIdx.x];
  const int lane = threadIdx.x % TPR, g = threadIdx.x / TPR;
  const float inv = 1.0f / (float)p.dim;
  const T* w = (const T*)p.weight + t.client * p.ld_w;
  const T* b = (const T*)p.bias + t.client * p.ld_b;
  // every group walks the same number of rows: barriers are uniform
  for (int r = 0; r < t.rows; r += G) {
    const int64_t row = t.begin + min(r + g, t.rows - 1);
    const bool live = r + g < t.rows;
    const T* x = (const T*)p.x + row * p.ld_x;
    vec v[NV];
    float f[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      v[i] = load_vec(x + c, (int64_t)p.dim - c);
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[0] += (float)v[i][e];
    }
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
      const int64_t left = (int64_t)p.dim - c;
      vec gw = {}, gb = {};
      if (p.weight) gw = load_vec(w + c, left);
      if (p.bias) gb = load_vec(b + c, left);
      vec o;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float y = ((float)v[i][e] - mu) * s;
        if (p.weight) y *= (float)gw[e];
        if (p.bias) y += (float)gb[e];
        o[e] = (T)y;
      }
      store_vec((T*)p.out + row * p.ld_out + c, o, left);
    }
  }
}

template <typename T, int TPR, int NV>
__global__ __launch_bounds__(256) void k_norm_backward(const NormArgs p) {
  constexpr int VEC = Elem<T>::kVec, G = 256 / TPR;
  typedef typename VecOf<T>::type vec;
  __shared__ float slots[2][2 * 4];
  __shared__ float join[G > 1 ? TPR * VEC * NV : 1];
  const RowTile t = p.tiles[blockIdx.x];
  const int lane = threadIdx.x % TPR, g = threadIdx.x / TPR;
  const float inv = 1.0f / (float)p.dim;
  const T* w = (const T*)p.weight + t.client * p.ld_w;
  float dg[NV][VEC] = {}, db[NV][VEC] = {};
  int turn = 0;
  for (int r = 0; r < t.rows; r += G, turn ^= 1) {
    const int64_t row = t.begin + min(r + g, t.rows - 1);
    const bool live = r + g < t.rows;
    const float mu = p.mean[row], s = p.rstd[row];
    const T* x = (const T*)p.x + row * p.ld_x;
    const T* dy = (const T*)p.dy + row * p.ld_dy;
    vec vx[NV], vd[NV];
    float f[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      const int64_t left = live ? (int64_t)p.dim - c : 0;
      vx[i] = load_vec(x + c, left);
      vd[i] = load_vec(dy + c, left);
      vec gw = {};
      if (p.weight) gw = load_vec(w + c, left);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        // columns past the end (and rows past the tile) have dy = 0: they add nothing
        const float d = (float)vd[i][e], xh = ((float)vx[i][e] - mu) * s;
        const float a = p.weight ? d * (float)gw[e] : d;
        const bool in = e < left;
        f[0] += in ? a : 0.0f;
        f[1] += in ? a * xh : 0.0f;
        dg[i][e] += in ? d * xh : 0.0f;
        db[i][e] += in ? d : 0.0f;
      }
    }
    group_sum<TPR>(f, slots[turn]);
    const float m0 = f[0] * inv, m1 = f[1] * inv;
    if (!live) continue;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      const int64_t left = (int64_t)p.dim - c;
      vec gw = {}, res = {};
      if (p.weight) gw = load_vec(w + c, left);
      if (p.residual) res = load_vec((const T*)p.residual + row * p.ld_res + c, left);
      vec o;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = (float)vd[i][e], xh = ((float)vx[i][e] - mu) * s;
        const float a = p.weight ? d * (float)gw[e] : d;
        float v = s * (a - m0 - xh * m1);
        if (p.residual) v += (float)res[e];
        o[e] = (T)v;
      }
      store_vec((T*)p.out + row * p.ld_out + c, o, left);
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

// Rows longer than the registers of a block hold: the row is read once per sum.
template <typename T>
__global__ __launch_bounds__(256) void k_norm_long(const NormArgs p) {
  __shared__ float slots[2][2 * 4];
  const RowTile t = p.tiles[blockIdx.x];
  const float inv = 1.0f / (float)p.dim;
  const T* w = (const T*)p.weight + t.client * p.ld_w;
  const T* b = (const T*)p.bias + t.client * p.ld_b;
  for (int r = 0; r < t.rows; ++r) {
    const int64_t row = t.begin + r;
    const T* x = (const T*)p.x + row * p.ld_x;
    float f[1] = {0.0f};
    for (int c = threadIdx.x; c < p.dim; c += 256) f[0] += (float)x[c];
    group_sum<256>(f, slots[0]);
    const float mu = f[0] * inv;
    f[0] = 0.0f;
    for (int c = threadIdx.x; c < p.dim; c += 256) {
      const float d = (float)x[c] - mu;
      f[0] += d * d;
    }
    group_sum<256>(f, slots[1]);
    const float s = 1.0f / sqrtf(f[0] * inv + p.eps);
    if (threadIdx.x == 0) {
      p.mean[row] = mu;
      p.rstd[row] = s;
    }
    T* o = (T*)p.out + row * p.ld_out;
    for (int c = threadIdx.x; c < p.dim; c += 256) {
      float y = ((float)x[c] - mu) * s;
      if (p.weight) y *= (float)w[c];
      if (p.bias) y += (float)b[c];
      o[c] = (T)y;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void k_norm_backward_long(const NormArgs p) {
  __shared__ float slots[2][2 * 4];
  const RowTile t = p.tiles[blockIdx.x];
  const float inv = 1.0f / (float)p.dim;
  const T* w = (const T*)p.weight + t.client * p.ld_w;
  for (int r = 0; r < t.rows; ++r) {
    const int64_t row = t.begin + r;
    const T* x = (const T*)p.x + row * p.ld_x;
    const T* dy = (const T*)p.dy + row * p.ld_dy;
    const float mu = p.mean[row], s = p.rstd[row];
    float f[2] = {0.0f, 0.0f};
    for (int c = threadIdx.x; c < p.dim; c += 256) {
      const float a = (float)dy[c] * (p.weight ? (float)w[c] : 1.0f);
      f[0] += a;
      f[1] += a * ((float)x[c] - mu) * s;
    }
    group_sum<256>(f, slots[r & 1]);
    const float m0 = f[0] * inv, m1 = f[1] * inv;
    for (int c = threadIdx.x; c < p.dim; c += 256) {
      const float a = (float)dy[c] * (p.weight ? (float)w[c] : 1.0f);
      float v = s * (a - m0 - ((float)x[c] - mu) * s * m1);
      if (p.residual) v += (float)((const T*)p.residual)[row * p.ld_res + c];
      ((T*)p.out)[row * p.ld_out + c] = (T)v;
    }
  }
  if (!p.part) return;
  for (int c = threadIdx.x; c < p.dim; c += 256) {
    float dg = 0.0f, db = 0.0f;
    for (int r = 0; r < t.rows; ++r) {
      const int64_t row = t.begin + r;
      const float d = (float)((const T*)p.dy)[row * p.ld_dy + c];
      dg += d * ((float)((const T*)p.x)[row * p.ld_x + c] - p.mean[row]) * p.rstd[row];
      db += d;
    }
    p.part[((int64_t)blockIdx.x * 2) * p.dim + c] = dg;
    p.part[((int64_t)blockIdx.x * 2 + 1) * p.dim + c] = db;
  }
}

// dg_c, db_c: the client's tiles' partial rows, summed in tile order.
__global__ __launch_bounds__(256) void k_norm_join(const float* part, const int32_t* first_tile, int32_t dim,
                                                   float* dw, int64_t ld_dw, float* db, int64_t ld_db,
                                                   int accumulate) {
  const int c = blockIdx.y * 256 + threadIdx.x, client = blockIdx.x, which = blockIdx.z;
  float* o = which ? db : dw;
  if (c >= dim || !o) return;
  o += client * (which ? ld_db : ld_dw) + c;
  const int lo = first_tile[client], hi = first_tile[client + 1];
  float s = accumulate ? *o : 0.0f;
  float t[8];
  int k = lo;
  for (; k + 8 <= hi; k += 8) {
#pragma unroll
    for (int u = 0; u < 8; ++u) t[u] = part[((int64_t)(k + u) * 2 + which) * dim + c];
#pragma unroll
    for (int u = 0; u < 8; ++u) s += t[u];
  }
  for (; k < hi; ++k) s += part[((int64_t)k * 2 + which) * dim + c];
  *o = s;
}

// ---------------------------------------------------------------------------
// Top logits: the k largest of a row (ties to the lowest index, NaN below every
// number), and log sum exp(l / tau).
//
// The k-th largest of the threads' own maxima is a lower bound of the k-th largest
// logit, so only the few threads whose maximum reaches it look at their elements
// again; what they hold at or above it is ranked by counting.  When too many
// elements tie there, the bound is made exact by a radix select first.
// ---------------------------------------------------------------------------

constexpr int kTopThreads = 1024;
constexpr int kTopCap = 2048;  // candidates ranked in LDS

// Orders as the float does; -0 = +0; NaN lowest.
__device__ __forceinline__ uint32_t order_key(float f) {
  if (f != f) return 0;
  const uint32_t u = __float_as_uint(f + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

template <typename T>
__global__ __launch_bounds__(kTopThreads) void k_top_logits(const T* logits, int64_t ld, int32_t vocab, int32_t k,
                                                            float scale, int32_t* index, T* values, float* lse) {
  constexpr int VEC = Elem<T>::kVec;
  typedef typename VecOf<T>::type vec;
  __shared__ uint32_t maxima[kTopThreads];
  __shared__ unsigned long long cand[kTopCap];
  __shared__ uint32_t hist[256];
  __shared__ float red[2][kTopThreads / 64];
  __shared__ uint32_t bound, ncand, want, ties;
  const int64_t row = blockIdx.x;
  const T* x = logits + row * ld;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;

  uint32_t best = 0;
  bool nan = false;
  float mx = -INFINITY, sum = 0.0f;  // running maximum and sum of exp2((l - mx) scale)
  for (int64_t c = (int64_t)tid * VEC; c < vocab; c += (int64_t)kTopThreads * VEC) {
    const vec v = load_vec(x + c, vocab - c);
    float m = -INFINITY;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float f = c + e < vocab ? (float)v[e] : -INFINITY;
      nan |= f != f;
      m = fmaxf(m, f);
      if (c + e < vocab) best = max(best, order_key(f));
    }
    if (m > mx) {
      sum *= exp2f((mx - m) * scale);
      mx = m;
    }
    if (mx > -INFINITY)
#pragma unroll
      for (int e = 0; e < VEC; ++e) sum += c + e < vocab ? exp2f(((float)v[e] - mx) * scale) : 0.0f;
  }
  maxima[tid] = best;
  const float wm = wave_max(mx);
  if (lane == 0) red[0][wave] = wm;
  if (tid == 0) ncand = ties = 0;
  const bool any_nan = __syncthreads_or(nan);
  float bm = red[0][0];
#pragma unroll
  for (int w = 1; w < kTopThreads / 64; ++w) bm = fmaxf(bm, red[0][w]);
  const float ws = wave_sum(mx > -INFINITY ? sum * exp2f((mx - bm) * scale) : 0.0f);
  if (lane == 0) red[1][wave] = ws;
  if (wave == 0) {
    // the k-th largest of the maxima, bit by bit (0 when fewer threads than k hold any)
    uint32_t m[kTopThreads / 64];
#pragma unroll
    for (int i = 0; i < kTopThreads / 64; ++i) m[i] = maxima[i * 64 + lane];
    uint32_t t = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t probe = t | (1u << bit);
      int n = 0;
#pragma unroll
      for (int i = 0; i < kTopThreads / 64; ++i) n += __popcll(__ballot(m[i] >= probe));
      if (n >= k) t = probe;
    }
    if (lane == 0) bound = t;
  }
  __syncthreads();
  if (tid == 0) {
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < kTopThreads / 64; ++w) s += red[1][w];
    lse[row] = any_nan ? NAN : fabsf(bm) == INFINITY ? bm : bm * scale * kLn2 + logf(s);
  }
  const uint32_t t0 = bound;
  if (best >= t0)
    for (int64_t c = (int64_t)tid * VEC; c < vocab; c += (int64_t)kTopThreads * VEC) {
      const vec v = load_vec(x + c, vocab - c);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        if (c + e >= vocab) break;
        const uint32_t key = order_key((float)v[e]);
        if (key < t0) continue;
        const uint32_t at = atomicAdd(&ncand, 1u);
        if (at < kTopCap) cand[at] = (unsigned long long)key << 32 | (uint32_t)~(uint32_t)(c + e);
      }
    }
  __syncthreads();
  uint32_t n = ncand;
  if (n > kTopCap) {
    // exact k-th key by four 8-bit digits, then everything above it and the first ties
    uint32_t prefix = 0, need = k;
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int64_t c = tid; c < vocab; c += kTopThreads) {
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
    for (int64_t c0 = 0; c0 < vocab; c0 += kTopThreads) {
      const int64_t c = c0 + tid;
      const uint32_t key = c < vocab ? order_key((float)x[c]) : 0;
      const bool tie = c < vocab && key == prefix;
      if (c < vocab && key > prefix) cand[atomicAdd(&ncand, 1u)] = (unsigned long long)key << 32 | (uint32_t)~(uint32_t)c;
      const unsigned long long b = __ballot(tie);
      if (lane == 0) hist[wave] = __popcll(b);
      __syncthreads();
      uint32_t before = ties + __popcll(b & ((1ull << lane) - 1)), all = 0;
#pragma unroll
      for (int w = 0; w < kTopThreads / 64; ++w) {
        if (w < wave) before += hist[w];
        all += hist[w];
      }
      if (tie && before < need) cand[atomicAdd(&ncand, 1u)] = (unsigned long long)key << 32 | (uint32_t)~(uint32_t)c;
      __syncthreads();
      if (tid == 0) ties += all;
      __syncthreads();
    }
    n = ncand;
  }
  for (uint32_t i = tid; i < n; i += kTopThreads) {
    const unsigned long long mine = cand[i];
    int rank = 0;
    for (uint32_t j = 0; j < n; ++j) rank += cand[j] > mine;
    if (rank < k) {
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
// ---------------------------------------------------------------------------

constexpr int kDistillThreads = 256;
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

template <int NT>
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = wave_sum(v);
  __syncthreads();
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
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int w = 1; w < NT / 64; ++w) v = fmaxf(v, red[w]);
  return v;
}

// LOSS: row loss and lse; GRAD: the gradient (with LOSS unset from the saved lse).
template <typename T, bool LOSS, bool GRAD>
__global__ __launch_bounds__(kDistillThreads) void k_distill(const DistillArgs a) {
  constexpr int VEC = Elem<T>::kVec, NT = kDistillThreads;
  typedef typename VecOf<T>::type vec;
  __shared__ int32_t at[kDistillMax];
  __shared__ float prob[kDistillMax], own[kDistillMax];
  __shared__ float red[NT / 64];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  const int client = a.row_client[row];
  const float weight = a.row_weights ? a.row_weights[row]
                                     : 1.0f / (float)(a.offsets[client + 1] - a.offsets[client]);
  const T* s = (const T*)a.logits + row * a.ld;
  T* grad = (T*)a.grad + row * a.ld_grad;
  const float inv_tau = 1.0f / a.tau, scale = kLog2e * inv_tau;

  // the teacher's row
  float high = -INFINITY;
  for (int i = tid; i < a.k; i += NT) {
    int32_t j = a.index[row * a.k + i];
    const float t = a.values[row * a.k + i] * inv_tau;
    if ((uint32_t)j >= (uint32_t)a.vocab || t == -INFINITY) j = -1;
    at[i] = j;
    prob[i] = t;
    if (j >= 0) high = t != t ? t : fmaxf(high, t);
  }
  const bool any = __syncthreads_or(high != -INFINITY);
  if (!any || weight == 0.0f) {  // nothing to learn from: no loss, no gradient, logits not looked at
    if (LOSS && tid == 0) {
      a.row_loss[row] = 0.0f;
      if (a.lse) a.lse[row] = 0.0f;
    }
    if (GRAD) {
      const vec zero = {};
      for (int64_t c = (int64_t)tid * VEC; c < a.vocab; c += NT * VEC) store_vec(grad + c, zero, a.vocab - c);
    }
    return;
  }
  float L;
  if (a.teacher_lse) {
    L = a.teacher_lse[row];
  } else {
    high = block_max<NT>(high, red);
    float z = 0.0f;
    for (int i = tid; i < a.k; i += NT)
      if (at[i] >= 0) z += expf(prob[i] - high);
    L = high + logf(block_sum<NT>(z, red));
  }

  // the student's softmax
  float mx, lse;
  if (LOSS) {
    float m = -INFINITY, z = 0.0f;
    for (int64_t c = (int64_t)tid * VEC; c < a.vocab; c += NT * VEC) {
      const vec v = load_vec(s + c, a.vocab - c);
      float vm = -INFINITY;
#pragma unroll
      for (int e = 0; e < VEC; ++e) vm = fmaxf(vm, c + e < a.vocab ? (float)v[e] : -INFINITY);
      if (vm > m) {
        z *= exp2f((m - vm) * scale);
        m = vm;
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float f = (float)v[e];
        if (c + e < a.vocab && f != -INFINITY) z += exp2f((f - m) * scale);
      }
    }
    mx = block_max<NT>(m, red);
    z = block_sum<NT>(m > -INFINITY ? z * exp2f((m - mx) * scale) : z, red);
    lse = mx == -INFINITY && z == 0.0f ? -INFINITY : mx * inv_tau + logf(z);
    if (tid == 0 && a.lse) a.lse[row] = lse;
    if (!GRAD) mx = 0.0f;
  } else {
    lse = a.lse[row];
  }

  // teacher entries: probability, student logit, loss
  float loss = 0.0f, mass = 0.0f;
  for (int i = tid; i < a.k; i += NT) {
    const int32_t j = at[i];
    float pr = 0.0f, st = 0.0f;
    if (j >= 0) {
      const float logp = prob[i] - L;
      pr = expf(logp);
      st = (float)s[j];
      const float logq = st == -INFINITY ? -INFINITY : st * inv_tau - lse;
      if (pr != 0.0f) loss += pr * (logp - logq);
    }
    prob[i] = pr;
    own[i] = st;
    mass += pr;
  }
  if (LOSS) {
    loss = block_sum<NT>(loss, red);
    if (tid == 0) a.row_loss[row] = weight * a.tau * a.tau * loss;
  }
  if (!GRAD) return;
  mass = block_sum<NT>(mass, red);
  float w = weight * a.tau;
  if (a.dloss) w *= a.dloss[client];
  const float wm = w * mass;
  const bool none = lse == -INFINITY;  // no student distribution: q = 0
  const float shift = lse;
  for (int64_t c = (int64_t)tid * VEC; c < a.vocab; c += NT * VEC) {
    const vec v = load_vec(s + c, a.vocab - c);
    vec o;
#pragma unroll
    for (int e = 0; e < VEC; ++e) o[e] = (T)(none ? 0.0f : wm * expf((float)v[e] * inv_tau - shift));
    store_vec(grad + c, o, a.vocab - c);
  }
  __syncthreads();
  // the teacher's columns: the first entry of an index takes all of its entries, in order
  for (int i = tid; i < a.k; i += NT) {
    const int32_t j = at[i];
    if (j < 0) continue;
    bool first = true;
    for (int h = 0; h < i; ++h) first &= at[h] != j;
    if (!first) continue;
    float pr = prob[i];
    for (int h = i + 1; h < a.k; ++h)
      if (at[h] == j) pr += prob[h];
    const float q = none ? 0.0f : mass * expf(own[i] * inv_tau - shift);
    grad[j] = (T)(w * (q - pr));
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

template <typename T, int TPR, int NV>
void norm_launch(const NormArgs& p, bool backward, hipStream_t s) {
  if (backward) hipLaunchKernelGGL((k_norm_backward<T, TPR, NV>), dim3(p.ntiles), dim3(256), 0, s, p);
  else hipLaunchKernelGGL((k_norm<T, TPR, NV>), dim3(p.ntiles), dim3(256), 0, s, p);
}

template <typename T>
int norm_dispatch(const NormArgs& p, bool backward, hipStream_t s) {
  const int64_t vecs = (p.dim + Elem<T>::kVec - 1) / Elem<T>::kVec;
  if (vecs <= 64) norm_launch<T, 64, 1>(p, backward, s);
  else if (vecs <= 128) norm_launch<T, 64, 2>(p, backward, s);
  else if (vecs <= 256) norm_launch<T, 256, 1>(p, backward, s);
  else if (vecs <= 512) norm_launch<T, 256, 2>(p, backward, s);
  else if (vecs <= 1024) norm_launch<T, 256, 4>(p, backward, s);
  else if (vecs <= 2048) norm_launch<T, 256, 8>(p, backward, s);
  else if (backward) hipLaunchKernelGGL((k_norm_backward_long<T>), dim3(p.ntiles), dim3(256), 0, s, p);
  else hipLaunchKernelGGL((k_norm_long<T>), dim3(p.ntiles), dim3(256), 0, s, p);
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

template <typename T>
int distill_launch(const DistillArgs& a, int64_t rows, bool loss, hipStream_t s) {
  const dim3 grid((unsigned)rows), block(kDistillThreads);
  if (loss && a.grad) hipLaunchKernelGGL((k_distill<T, true, true>), grid, block, 0, s, a);
  else if (loss) hipLaunchKernelGGL((k_distill<T, true, false>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((k_distill<T, false, true>), grid, block, 0, s, a);
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

constexpr int64_t kMaxDim = 1 << 24;

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
  hipLaunchKernelGGL(k_norm_join, dim3((unsigned)nclients, (unsigned)((dim + 255) / 256), 2), dim3(256), 0, s,
                     (const float*)partials, first_tile, (int32_t)dim, dweight, dweight_stride, dbias, dbias_stride,
                     accumulate);
  return fc_internal_check_launch("k_norm_join");
}

int fc_top_logits(const void* logits, int64_t stride, int dtype, int64_t rows, int64_t vocab, int32_t k,
                  float temperature, int32_t* index, void* values, float* lse, void* stream) {
  if (rows < 0 || rows > 0x7fffffffLL || vocab <= 0 || vocab > 0x7fffffffLL - 65536) return fc_internal_fail(-1, "bad sizes");
  if (k <= 0 || k > vocab || k > FC_MAX_TOP) return fc_internal_fail(-1, "bad k");
  if (!(temperature > 0.0f) || std::isinf(temperature)) return fc_internal_fail(-1, "bad temperature");
  if (rows == 0) return 0;
  if (!logits || !index || !values || !lse) return fc_internal_fail(-1, "null pointer");
  const float scale = kLog2e / temperature;
  const dim3 grid((unsigned)rows), block(kTopThreads);
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case FC_FLOAT32:
      hipLaunchKernelGGL((k_top_logits<float>), grid, block, 0, s, (const float*)logits, stride, (int32_t)vocab, k,
                         scale, index, (float*)values, lse);
      break;
    case FC_BFLOAT16:
      hipLaunchKernelGGL((k_top_logits<bf16>), grid, block, 0, s, (const bf16*)logits, stride, (int32_t)vocab, k,
                         scale, index, (bf16*)values, lse);
      break;
    case FC_FLOAT16:
      hipLaunchKernelGGL((k_top_logits<f16>), grid, block, 0, s, (const f16*)logits, stride, (int32_t)vocab, k, scale,
                         index, (f16*)values, lse);
      break;
    default: return fc_internal_fail(-1, "bad dtype");
  }
  return fc_internal_check_launch("k_top_logits");
}

int fc_distill(const void* logits, int64_t stride, int dtype, int64_t rows, int64_t vocab, const int32_t* index,
               const float* values, int32_t k, const int32_t* row_client, const int32_t* offsets, int32_t nclients,
               float temperature, const float* teacher_lse, const float* row_weights, const float* dloss,
               float* row_loss, float* lse, float* loss, void* grad, int64_t grad_stride, void* stream) {
  if (rows < 0 || rows > 0x7fffffffLL || nclients <= 0 || vocab <= 0 || vocab > 0x7fffffffLL - 65536)
    return fc_internal_fail(-1, "bad sizes");
  if (k <= 0 || k > kDistillMax) return fc_internal_fail(-1, "bad k");
  if (!(temperature > 0.0f) || std::isinf(temperature)) return fc_internal_fail(-1, "bad temperature");
  if (!offsets || (!loss && !grad) || (!loss && rows && !lse) || (loss && rows && !row_loss))
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
  hipLaunchKernelGGL(k_distill_join, dim3((unsigned)nclients), dim3(256), 0, s, (const float*)row_loss, offsets, loss);
  return fc_internal_check_launch("k_distill_join");
}

}  // extern "C"
