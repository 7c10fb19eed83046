// Losses on the log-probabilities of chosen ids (atom types, or tokens of any vocabulary), x = logits / temperature:
//   logp_t = x[t, id_t] - log sum_v exp(x[t, v])            d logp_t / d x[t, v] = [v = id_t] - p[t, v]
// so every loss below reaches the logits as  d_logits[t, v] = coef_t / temperature ([v = id_t] - p[t, v])  with one number
// coef_t = d loss / d logp_t for each row.  All of them are bound by HBM: a logit costs a handful of vector operations and
// its bytes are read once (and a gradient of the same size written once).
#include "token_common.h"

#define TK_LOG2E 1.44269504088896340736

struct TokenRows {
  const void* x;
  int64_t stride;      // elements between rows
  int64_t n;           // rows
  int32_t V;
  TokenView tok;
  float c;             // log2(e) / temperature: exp(x / temperature) = exp2(c x)
  double inv_t;        // 1 / temperature
};

// log(s) of the softmax sum, in 64 bits: losses use differences of log-probabilities of two policies, which are small
// against the log-probabilities.  s = 2^k f with f in [sqrt(1/2), sqrt(2)), z = (f - 1) / (f + 1),
// log f = 2 (z + z^3/3 + z^5/5 + ...): |z| < 0.172, six terms leave 5e-11 (the fp32 sum itself is good to ~1e-7).
// The quotient is the fp32 reciprocal with one correction step.
__device__ __forceinline__ double log_of_sum(float s) {
  if (!(s < __builtin_inff())) return (double)s;   // NaN and +inf pass through
  const uint32_t u = __float_as_uint(s);
  int k = (int)(u >> 23) - 127;
  float f = __uint_as_float((u & 0x7fffffu) | 0x3f800000u);
  if (f > 1.41421354f) { f *= 0.5f; ++k; }
  const double num = (double)f - 1.0, den = (double)f + 1.0;
  const double r = (double)__builtin_amdgcn_rcpf((float)den);
  double z = num * r;
  z = fma(fma(-den, z, num), r, z);
  const double q = z * z;
  const double poly = fma(q, fma(q, fma(q, fma(q, fma(q, 1.0 / 11, 1.0 / 9), 1.0 / 7), 1.0 / 5), 1.0 / 3), 1.0);
  return fma((double)k, 0.69314718055994530942, 2.0 * z * poly);
}

// exp(q) - 1 and exp(q) - 1 - q without cancellation (the second is ~q^2 / 2): Taylor for |q| < 1/2, eight terms leave 2e-9.
__device__ __forceinline__ void kl_terms(float q, float& em1, float& kl) {
  if (fabsf(q) < 0.5f) {
    float p = 1.0f / 362880.0f;
    p = fmaf(p, q, 1.0f / 40320.0f);
    p = fmaf(p, q, 1.0f / 5040.0f);
    p = fmaf(p, q, 1.0f / 720.0f);
    p = fmaf(p, q, 1.0f / 120.0f);
    p = fmaf(p, q, 1.0f / 24.0f);
    p = fmaf(p, q, 1.0f / 6.0f);
    p = fmaf(p, q, 0.5f);
    kl = q * q * p;
    em1 = q + kl;
  } else {
    em1 = expf(q) - 1.0f;
    kl = em1 - q;
  }
}

enum { TK_LOGP = 0, TK_POLICY = 1 };

struct PolicyIn {
  const int32_t* seq_of;     // [n] sequence of a row, -1 for rows that take no part
  const int32_t* seq_len;    // [S] rows of each sequence that take part (mean over sequences)
  const int32_t* chunk_len;  // [n_chunks] rows of each chunk that take part (mean over rows)
  int32_t n_chunks;
  double denom;              // <= 0: the count / the number of sequences
  int32_t n_seq, per_seq_mean;
  const float* adv;          // [S] or [n]
  int32_t adv_per_token;
  const float* old_logp;     // may be null: the policy itself
  const float* ref_logp;     // may be null: no KL term
  float clip_lo, clip_hi, kl_coef, grad_scale;
  double* partial;           // [gridDim.x][3]
  uint32_t* counter;
  float* result;             // loss, surrogate, kl, clip fraction
};
struct RowOut {
  float* logp;               // [n] or null
  const float* minus;        // [n] or null: subtracted from logp (difference of two policies)
  float* stats;              // [n][2]: row maximum and 1 / sum, for the gradient kernel; may be null
  float* coef;               // [n] d loss / d logp (TK_POLICY); may be null
  void* d;                   // gradient of the logits or null
  int64_t d_stride;
  uint32_t* clear;           // a counter of a later launch to set to 0, or null
};

// What a row contributes once its maximum M and sum S are known, the same in every lane of the row; returns the gradient's
// factor d loss / d logp * grad_scale / temperature.
template <int MODE>
__device__ __forceinline__ float row_epilogue(const TokenRows& a, const PolicyIn& p, const RowOut& o, int64_t t, int id, int seq,
                                              float xt, float M, float S, float inv_s, bool writer, double w, double (&acc)[3]) {
  // a row of -inf only has no distribution: S = 0, logp = -inf, no gradient
  const double lp = S == 0.f ? -__builtin_inf() : ((double)xt - (double)M) * a.inv_t - log_of_sum(S);
  float g = 0.f, coef = 0.f;
  if constexpr (MODE == TK_POLICY) {
    const float A = p.adv[p.adv_per_token ? t : (int64_t)seq];
    const float rho = p.old_logp ? expf((float)(lp - (double)p.old_logp[t])) : lp == lp ? 1.0f : (float)lp;
    const float hi = 1.0f + p.clip_hi, lo = 1.0f - p.clip_lo;
    const bool clipped = (A > 0.f && rho > hi) || (A < 0.f && rho < lo);
    const float gain = A == 0.f ? 0.f : fminf(rho * A, fminf(fmaxf(rho, lo), hi) * A);
    float slope = clipped || A == 0.f ? 0.f : -A * rho;
    float em1 = 0.f, kl = 0.f;
    if (p.ref_logp) {
      kl_terms((float)((double)p.ref_logp[t] - lp), em1, kl);
      slope -= p.kl_coef * em1;
    }
    if (rho != rho) slope = rho;   // fminf drops a NaN
    acc[0] -= w * (double)(rho != rho ? rho : gain);
    acc[1] += w * (double)kl;
    acc[2] += clipped ? w : 0.0;
    coef = (float)(w * (double)slope);
    if (S != 0.f) g = (float)(w * (double)slope * (double)p.grad_scale * a.inv_t);
  }
  if (writer) {
    if (o.logp) o.logp[t] = (float)(o.minus ? lp - (double)o.minus[t] : lp);
    if (o.stats) { o.stats[2 * t] = M; o.stats[2 * t + 1] = inv_s; }
    if (o.coef) o.coef[t] = coef;
  }
  return g;
}

// A row that takes no part: nothing of it is read, its log-probability and its gradient are 0.
template <typename T>
__device__ __forceinline__ void row_skip(const RowOut& o, int64_t t, int V, int r, int tpr, bool writer) {
  if (writer) {
    if (o.logp) o.logp[t] = 0.f;
    if (o.stats) { o.stats[2 * t] = 0.f; o.stats[2 * t + 1] = 0.f; }
    if (o.coef) o.coef[t] = 0.f;
  }
  if (o.d) {
    T* d = reinterpret_cast<T*>(o.d) + t * o.d_stride;
    constexpr int N = Pack<T>::N;
    const float z[N] = {};
    const int nb = V / N;
    for (int i = r; i < nb; i += tpr) store_pack(d + (int64_t)i * N, z);
    if (r < V - nb * N) d[nb * N + r] = (T)0.f;
  }
}

// The weight that a row has in the mean.
__device__ __forceinline__ double row_weight(const PolicyIn& p, int seq, double inv_total) {
  return p.per_seq_mean ? inv_total / (double)p.seq_len[seq] : inv_total;
}
template <int NT> __device__ __forceinline__ double inverse_total(const PolicyIn& p, double* red) {
  double total = p.denom;
  if (!(total > 0.0)) {
    if (p.per_seq_mean) total = (double)p.n_seq;
    else {
      double v = 0.0;
      for (int i = threadIdx.x; i < p.n_chunks; i += NT) v += (double)p.chunk_len[i];
      total = block_sum<NT>(v, red);
    }
  }
  return total > 0.0 ? 1.0 / total : 0.0;
}
// Per-block sums to memory; the last block adds them up in block order.
template <int NT> __device__ __forceinline__ void policy_finish(const PolicyIn& p, double (&acc)[3], double* red) {
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const double v = block_sum<NT>(acc[k], red);
    if (threadIdx.x == 0) p.partial[(int64_t)blockIdx.x * 3 + k] = v;
  }
  if (!last_block(p.counter)) return;
  double v[3] = {0.0, 0.0, 0.0};
  for (int b = threadIdx.x; b < (int)gridDim.x; b += NT)
#pragma unroll
    for (int k = 0; k < 3; ++k) v[k] += p.partial[(int64_t)b * 3 + k];
#pragma unroll
  for (int k = 0; k < 3; ++k) v[k] = block_sum<NT>(v[k], red);
  if (threadIdx.x == 0) {
    p.result[0] = (float)(v[0] + (double)p.kl_coef * v[1]);
    p.result[1] = (float)v[0];
    p.result[2] = (float)v[1];
    p.result[3] = (float)v[2];
  }
}

// Rows that fit the registers of TPR lanes, NV packs a lane: the logits are read once, exponentiated once, and the policy
// loss writes its gradient from the same registers.  TPR = 16 / 64: several rows a block and no barrier; 256 / 1024: one
// row a block, whose waves take the maximum and sum of their own part and exchange the pair once.
template <typename T, int TPR, int NV, int MODE>
__global__ __launch_bounds__(TPR <= 64 ? 256 : TPR) void k_token_rows(TokenRows a, PolicyIn p, RowOut o) {
  constexpr int N = Pack<T>::N, NT = TPR <= 64 ? 256 : TPR, RPB = NT / TPR, NW = TPR / 64;
  __shared__ float2 sh[2][NW > 1 ? NW : 1];
  __shared__ double red[NT / 64];
  const int r = threadIdx.x % TPR;
  const int V = a.V, nb = V / N, tail = V - nb * N;
  double inv_total = 0.0, acc[3] = {0.0, 0.0, 0.0};
  if constexpr (MODE == TK_POLICY) inv_total = inverse_total<NT>(p, red);
  if (o.clear && blockIdx.x == 0 && threadIdx.x == 0) *o.clear = 0;
  int parity = 0;
  for (int64_t base = (int64_t)blockIdx.x * RPB; base < a.n; base += (int64_t)gridDim.x * RPB) {
    const int64_t t = base + threadIdx.x / TPR;
    if (TPR <= 64 && t >= a.n) continue;
    int id = a.tok.at(t), seq = 0;
    if constexpr (MODE == TK_POLICY) {
      seq = p.seq_of[t];
      if (seq < 0) id = -1;
    }
    if (id < 0) {
      row_skip<T>(o, t, V, r, TPR, r == 0);
      continue;
    }
    const T* row = reinterpret_cast<const T*>(a.x) + t * a.stride;
    float e[NV][N], et = -__builtin_inff();
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (r + k * TPR < nb) load_pack(row + (int64_t)(r + k * TPR) * N, e[k]);
      else
#pragma unroll
        for (int j = 0; j < N; ++j) e[k][j] = -__builtin_inff();
    }
    if (r < tail) et = (float)row[nb * N + r];
    const float xt = (float)row[id];
    double w = 0.0;
    if constexpr (MODE == TK_POLICY) w = row_weight(p, seq, inv_total);
    float m = et;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int j = 0; j < N; ++j) m = fmaxf(m, e[k][j]);
    m = group_max<(TPR < 64 ? TPR : 64)>(m);
    const float mm = m == -__builtin_inff() ? 0.f : m;
    float s = et = __builtin_amdgcn_exp2f((et - mm) * a.c);
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int j = 0; j < N; ++j) s += e[k][j] = __builtin_amdgcn_exp2f((e[k][j] - mm) * a.c);
    s = group_sum<(TPR < 64 ? TPR : 64)>(s);
    float M = mm, S = s, f = 1.0f;
    if constexpr (NW > 1) {
      // (the buffers alternate between rows: a wave that runs ahead writes the other one)
      if ((threadIdx.x & 63) == 0) sh[parity][threadIdx.x >> 6] = make_float2(m, s);
      __syncthreads();
      M = -__builtin_inff();
#pragma unroll
      for (int i = 0; i < NW; ++i) M = fmaxf(M, sh[parity][i].x);
      if (M == -__builtin_inff()) M = 0.f;
      S = 0.f;
#pragma unroll
      for (int i = 0; i < NW; ++i) S += sh[parity][i].y * __builtin_amdgcn_exp2f((sh[parity][i].x - M) * a.c);
      f = __builtin_amdgcn_exp2f((mm - M) * a.c);
      if (m == -__builtin_inff()) f = 0.f;
      parity ^= 1;
    }
    const float inv_s = S == 0.f ? 0.f : 1.0f / S;
    const float g = row_epilogue<MODE>(a, p, o, t, id, seq, xt, M, S, inv_s, r == 0, w, acc);
    if constexpr (MODE == TK_POLICY) {
      if (o.d == nullptr) continue;
      T* d = reinterpret_cast<T*>(o.d) + t * o.d_stride;
      // a factor of 0 sends no gradient, also where the row holds a NaN
      const float q = g == 0.f ? 0.f : -g * f * inv_s;
      const int it = id / N;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int i = r + k * TPR;
        if (i < nb) {
          float v[N];
#pragma unroll
          for (int j = 0; j < N; ++j) v[j] = g == 0.f ? 0.f : q * e[k][j];
          if (i == it) {
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] += j == id - it * N ? g : 0.f;
          }
          store_pack(d + (int64_t)i * N, v);
        }
      }
      if (r < tail) d[nb * N + r] = (T)((g == 0.f ? 0.f : q * et) + (nb * N + r == id ? g : 0.f));
    }
  }
  if constexpr (MODE == TK_POLICY) {
    if (r != 0) acc[0] = acc[1] = acc[2] = 0.0;
    policy_finish<NT>(p, acc, red);
  }
}

// Longer rows: one block a row, running maximum and sum over the packs, and a second read for the gradient.
template <typename T, int MODE>
__global__ __launch_bounds__(1024) void k_token_rows_long(TokenRows a, PolicyIn p, RowOut o) {
  constexpr int N = Pack<T>::N, NT = 1024, NW = NT / 64;
  __shared__ float2 sh[2][NW];
  __shared__ double red[NW];
  const int r = threadIdx.x;
  const int V = a.V, nb = V / N, tail = V - nb * N;
  double inv_total = 0.0, acc[3] = {0.0, 0.0, 0.0};
  if constexpr (MODE == TK_POLICY) inv_total = inverse_total<NT>(p, red);
  if (o.clear && blockIdx.x == 0 && threadIdx.x == 0) *o.clear = 0;
  int parity = 0;
  for (int64_t t = blockIdx.x; t < a.n; t += gridDim.x) {
    int id = a.tok.at(t), seq = 0;
    if constexpr (MODE == TK_POLICY) {
      seq = p.seq_of[t];
      if (seq < 0) id = -1;
    }
    if (id < 0) {
      row_skip<T>(o, t, V, r, NT, r == 0);
      continue;
    }
    const T* row = reinterpret_cast<const T*>(a.x) + t * a.stride;
    const float xt = (float)row[id];
    double w = 0.0;
    if constexpr (MODE == TK_POLICY) w = row_weight(p, seq, inv_total);
    float m = -__builtin_inff(), s = 0.f;
    const auto take = [&](float mx, const float* v, int n) {
      const float nm = fmaxf(m, mx), z = nm == -__builtin_inff() ? 0.f : nm;
      if (m != -__builtin_inff()) s *= __builtin_amdgcn_exp2f((m - z) * a.c);
      for (int j = 0; j < n; ++j) s += __builtin_amdgcn_exp2f((v[j] - z) * a.c);
      m = nm;
    };
    for (int i = r; i < nb; i += NT) {
      float v[N];
      load_pack(row + (int64_t)i * N, v);
      float mx = v[0];
#pragma unroll
      for (int j = 1; j < N; ++j) mx = fmaxf(mx, v[j]);
      take(mx, v, N);
    }
    if (r < tail) {
      const float v = (float)row[nb * N + r];
      take(v, &v, 1);
    }
    const float wm = group_max<64>(m), wmm = wm == -__builtin_inff() ? 0.f : wm;
    s = group_sum<64>(m == -__builtin_inff() ? s : s * __builtin_amdgcn_exp2f((m - wmm) * a.c));
    if ((threadIdx.x & 63) == 0) sh[parity][threadIdx.x >> 6] = make_float2(wm, s);
    __syncthreads();
    float M = -__builtin_inff(), S = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) M = fmaxf(M, sh[parity][i].x);
    if (M == -__builtin_inff()) M = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) S += sh[parity][i].y * __builtin_amdgcn_exp2f((sh[parity][i].x - M) * a.c);
    parity ^= 1;
    const float inv_s = S == 0.f ? 0.f : 1.0f / S;
    const float g = row_epilogue<MODE>(a, p, o, t, id, seq, xt, M, S, inv_s, r == 0, w, acc);
    if constexpr (MODE == TK_POLICY) {
      if (o.d == nullptr) continue;
      T* d = reinterpret_cast<T*>(o.d) + t * o.d_stride;
      const float q = -g * inv_s;
      for (int i = r; i < nb; i += NT) {
        float v[N];
        load_pack(row + (int64_t)i * N, v);
#pragma unroll
        for (int j = 0; j < N; ++j)
          v[j] = g == 0.f ? 0.f : q * __builtin_amdgcn_exp2f((v[j] - M) * a.c) + (i * N + j == id ? g : 0.f);
        store_pack(d + (int64_t)i * N, v);
      }
      if (r < tail) {
        const int v = nb * N + r;
        d[v] = (T)(g == 0.f ? 0.f : q * __builtin_amdgcn_exp2f(((float)row[v] - M) * a.c) + (v == id ? g : 0.f));
      }
    }
  }
  if constexpr (MODE == TK_POLICY) {
    if (r != 0) acc[0] = acc[1] = acc[2] = 0.0;
    policy_finish<NT>(p, acc, red);
  }
}

// d_logits[t, v] = coef mult upstream / temperature ([v = id_t] - p[t, v]) from the saved maximum and 1 / sum: no reduction,
// the rows are streamed.  coef is that of the row, or of its sequence when an index is given.
template <typename T, int TPR>
__global__ __launch_bounds__(256) void k_token_grad(TokenRows a, const float* __restrict__ stats, const float* __restrict__ coef,
                                                    const int32_t* __restrict__ index, int64_t n_coef, float mult, const float* __restrict__ upstream, T* __restrict__ d, int64_t d_stride) {
  constexpr int N = Pack<T>::N, RPB = 256 / TPR;
  const int r = threadIdx.x % TPR;
  const int V = a.V, nb = V / N, tail = V - nb * N;
  const double k = (double)mult * a.inv_t * (upstream ? (double)*upstream : 1.0);
  for (int64_t t = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR; t < a.n; t += (int64_t)gridDim.x * RPB) {
    const int id = a.tok.at(t);
    const int64_t ci = index ? (int64_t)index[t] : t;
    const float g = id < 0 || ci < 0 || ci >= n_coef ? 0.f : (float)((double)coef[ci] * k);
    T* out = d + t * d_stride;
    if (g == 0.f || stats[2 * t + 1] == 0.f) {   // sends no gradient, also where the row holds a NaN; or -inf only
      row_skip<T>(RowOut{nullptr, nullptr, nullptr, nullptr, d, d_stride, nullptr}, t, V, r, TPR, false);
      continue;
    }
    const float M = stats[2 * t], q = -g * stats[2 * t + 1];
    const T* row = reinterpret_cast<const T*>(a.x) + t * a.stride;
    const int it = id / N;
#pragma unroll 4
    for (int i = r; i < nb; i += TPR) {
      float v[N];
      load_pack(row + (int64_t)i * N, v);
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = q * __builtin_amdgcn_exp2f((v[j] - M) * a.c);
      if (i == it) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] += j == id - it * N ? g : 0.f;
      }
      store_pack(out + (int64_t)i * N, v);
    }
    if (r < tail) {
      const int v = nb * N + r;
      out[v] = (T)(q * __builtin_amdgcn_exp2f(((float)row[v] - M) * a.c) + (v == id ? g : 0.f));
    }
  }
}

// Rows in chunks of SEG_ROWS, one block a chunk: the sequence of each row by bisection of seq_ptr (bounded whatever
// seq_ptr holds; -1 for ignored rows and rows outside every sequence), the chunk's number of taking rows, and for every
// sequence that meets the chunk the sum and the number of its rows in it, from prefix sums in 64 bits.  What sequence s has
// in chunk c goes to place c + s: both grow along the rows, so no two parts share a place.  A sequence of any length is
// then the sum of its parts, and no block waits for one long sequence.
#define SEG_ROWS 1024
__device__ __forceinline__ int seq_at(const int32_t* __restrict__ seq_ptr, int lo, int hi, int64_t t) {
  // the last s in [lo, hi] with seq_ptr[s] <= t, lo - 1 if there is none
  while (lo <= hi) {
    const int mid = (int)(((int64_t)lo + hi) >> 1);
    if ((int64_t)seq_ptr[mid] <= t) lo = mid + 1; else hi = mid - 1;
  }
  return hi;
}
template <bool SUM>
__global__ __launch_bounds__(256) void k_row_segments(TokenView tok, int64_t n, const int32_t* __restrict__ seq_ptr, int32_t S,
                                                      const float* __restrict__ diff, int32_t* __restrict__ seq_of,
                                                      double* __restrict__ part_sum, int32_t* __restrict__ part_len,
                                                      int32_t* __restrict__ chunk_len, uint32_t* __restrict__ clear) {
  __shared__ double pre[SUM ? SEG_ROWS + 1 : 1];
  __shared__ int cnt[SEG_ROWS + 1];
  __shared__ double wsum[4];
  __shared__ int wcnt[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (clear && blockIdx.x == 0 && tid == 0) *clear = 0;
  const int64_t c = blockIdx.x, c0 = c * SEG_ROWS;
  const int rows = (int)(n - c0 < SEG_ROWS ? n - c0 : SEG_ROWS);
  const int64_t first = seq_ptr ? seq_ptr[0] : 0, last = seq_ptr ? seq_ptr[S] : n;
  double v[4];
  int k[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = tid * 4 + j;
    const int64_t t = c0 + i;
    k[j] = i < rows && t >= first && t < last && tok.at(t) >= 0;
    v[j] = SUM && k[j] ? (double)diff[t] : 0.0;
  }
  int ci = (k[0] + k[1]) + (k[2] + k[3]);
  double vi = (v[0] + v[1]) + (v[2] + v[3]);
  const int own_c = ci;
  const double own_v = vi;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int cu = __shfl_up(ci, o);
    const double vu = SUM ? __shfl_up(vi, o) : 0.0;
    if (lane >= o) { ci += cu; vi += vu; }
  }
  if (lane == 63) { wcnt[wave] = ci; wsum[wave] = vi; }
  __syncthreads();
  int cb = ci - own_c;
  double vb = vi - own_v;
  for (int w = 0; w < wave; ++w) { cb += wcnt[w]; vb += wsum[w]; }
  if (tid == 0) { cnt[0] = 0; if (SUM) pre[0] = 0.0; }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    cb += k[j]; vb += v[j];
    cnt[tid * 4 + j + 1] = cb;
    if (SUM) pre[tid * 4 + j + 1] = vb;
  }
  __syncthreads();
  if (tid == 0 && chunk_len) chunk_len[c] = cnt[rows];
  const int s0 = seq_ptr ? seq_at(seq_ptr, 0, S, c0) : 0, s1 = seq_ptr ? seq_at(seq_ptr, 0, S, c0 + rows - 1) : 0;
  for (int i = tid; i < rows; i += 256) {
    int s = -1;
    if (cnt[i + 1] != cnt[i]) {
      s = seq_ptr ? seq_at(seq_ptr, s0 < 0 ? 0 : s0, s1, c0 + i) : 0;
      if (s >= S) s = -1;
    }
    seq_of[c0 + i] = s;
  }
  if (!part_len) return;
  for (int64_t s = (int64_t)(s0 < 0 ? 0 : s0) + tid; s <= s1 && s < S; s += 256) {
    const int64_t t0 = seq_ptr ? seq_ptr[s] : 0, t1 = seq_ptr ? seq_ptr[s + 1] : n;
    const int a = t0 <= c0 ? 0 : t0 - c0 < rows ? (int)(t0 - c0) : rows;
    const int b = t1 <= c0 ? 0 : t1 - c0 < rows ? (int)(t1 - c0) : rows;
    if (b > a) {
      part_len[c + s] = cnt[b] - cnt[a];
      if (SUM) part_sum[c + s] = pre[b] - pre[a];
    }
  }
}
// The parts of sequence s, added up by the 64 lanes of a wave.
template <bool SUM>
__device__ __forceinline__ void join_parts(const int32_t* __restrict__ seq_ptr, int64_t n, int64_t s, const double* __restrict__ part_sum,
                                           const int32_t* __restrict__ part_len, double& sum, int& len) {
  int64_t t0 = seq_ptr ? seq_ptr[s] : 0, t1 = seq_ptr ? seq_ptr[s + 1] : n;
  t0 = t0 < 0 ? 0 : t0;
  t1 = t1 > n ? n : t1;
  sum = 0.0; len = 0;
  if (t1 > t0)
    for (int64_t c = t0 / SEG_ROWS + (threadIdx.x & 63); c <= (t1 - 1) / SEG_ROWS; c += 64) {
      len += part_len[c + s];
      if (SUM) sum += part_sum[c + s];
    }
  len = wave_sum_i32(len);
  if (SUM) sum = wave_sum_f64(sum);
}
__global__ __launch_bounds__(256) void k_sequence_lengths(const int32_t* __restrict__ seq_ptr, int64_t n, int32_t S,
                                                          const int32_t* __restrict__ part_len, int32_t* __restrict__ seq_len) {
  const int64_t s = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (s >= S) return;
  double sum;
  int len;
  join_parts<false>(seq_ptr, n, s, nullptr, part_len, sum, len);
  if ((threadIdx.x & 63) == 0) seq_len[s] = len;
}

struct PrefIn {
  int64_t n;
  const int32_t* seq_ptr;
  int32_t P;
  const double* part_sum;
  const int32_t* part_len;
  float beta, smooth;
  int32_t kind, average;
  double denom, grad_scale;
  float* loss; float* log_ratio; float* margin; float* slope;
  double* partial;          // [gridDim.x]
  uint32_t* counter;
};
// Pairs: sequence p is preferred over sequence P + p.  A wave joins both sequences' differences (a margin is what two long
// sums leave: 64 bits), forms the loss and d loss / d logp of either sequence's rows; the last block adds the losses.
__global__ __launch_bounds__(256) void k_preference(PrefIn a) {
  __shared__ double red[4];
  const int lane = threadIdx.x & 63;
  double total = 0.0;
  for (int64_t pr = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); pr < a.P; pr += (int64_t)gridDim.x * 4) {
    double ratio[2], share[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      double sum;
      int len;
      join_parts<true>(a.seq_ptr, a.n, pr + (int64_t)h * a.P, a.part_sum, a.part_len, sum, len);
      share[h] = a.average && len > 0 ? 1.0 / (double)len : 1.0;
      ratio[h] = sum * share[h];
    }
    if (lane != 0) continue;
    const double gap = ratio[0] - ratio[1];
    double loss, slope;
    if (a.kind == LIGDIFF_PREFERENCE_SIGMOID) {
      // -(1 - e) log sigmoid(z) - e log sigmoid(-z) = log(1 + exp(-z)) + e z
      const double z = (double)a.beta * gap, x = exp(-fabs(z));
      loss = log1p(x) + (z < 0.0 ? -z : 0.0) + (double)a.smooth * z;
      const double sig = z >= 0.0 ? 1.0 / (1.0 + x) : x / (1.0 + x);
      slope = (double)a.beta * (sig - 1.0 + (double)a.smooth);
    } else {
      const double z = gap - 0.5 / (double)a.beta;
      loss = z * z;
      slope = 2.0 * z;
    }
    total += loss;
    slope *= a.grad_scale / a.denom;
    a.log_ratio[pr] = (float)ratio[0];
    a.log_ratio[pr + a.P] = (float)ratio[1];
    a.margin[pr] = (float)gap;
    a.slope[pr] = (float)(slope * share[0]);
    a.slope[pr + a.P] = (float)(-slope * share[1]);
  }
  total = block_sum<256>(total, red);
  if (threadIdx.x == 0) a.partial[blockIdx.x] = total;
  if (!last_block(a.counter)) return;
  double v = 0.0;
  for (int b = threadIdx.x; b < (int)gridDim.x; b += 256) v += a.partial[b];
  v = block_sum<256>(v, red);
  if (threadIdx.x == 0) a.loss[0] = (float)(v / a.denom);
}

// An empty batch: no row kernel runs.
__global__ void k_clear(uint32_t* counter) { if (threadIdx.x == 0) *counter = 0; }
__global__ void k_empty_policy(float* result) { if (threadIdx.x < 4) result[threadIdx.x] = 0.f; }

// ------------------------------------------------------------------ host side
// A persistent grid: enough blocks to fill the chip several times over, few enough that the per-block sums of a loss are
// added up by one block.
static int row_grid(int64_t groups, int most) { return (int)(groups < most ? groups : most); }

template <typename T, int TPR, int NV, int MODE>
static void launch_rows_as(const TokenRows& a, const PolicyIn& p, const RowOut& o, int grid_cap, hipStream_t s) {
  constexpr int NT = TPR <= 64 ? 256 : TPR, RPB = NT / TPR;
  const int grid = row_grid((a.n + RPB - 1) / RPB, grid_cap);
  hipLaunchKernelGGL((k_token_rows<T, TPR, NV, MODE>), dim3(grid), dim3(NT), 0, s, a, p, o);
}
#define TK_GRID_CAP 2048
// The least lanes whose registers hold a row: 16 lanes up to 64 packs, a wave up to 512, 256 lanes up to 2048, 1024 up to
// 8192 (32768 fp32 or 65536 half-precision logits); beyond that the row is read twice.
template <typename T, int MODE>
static void launch_rows(const TokenRows& a, const PolicyIn& p, const RowOut& o, hipStream_t s) {
  const int packs = a.V / Pack<T>::N;
  if (packs <= 16) launch_rows_as<T, 16, 1, MODE>(a, p, o, TK_GRID_CAP, s);
  else if (packs <= 32) launch_rows_as<T, 16, 2, MODE>(a, p, o, TK_GRID_CAP, s);
  else if (packs <= 64) launch_rows_as<T, 16, 4, MODE>(a, p, o, TK_GRID_CAP, s);
  else if (packs <= 128) launch_rows_as<T, 64, 2, MODE>(a, p, o, TK_GRID_CAP, s);
  else if (packs <= 256) launch_rows_as<T, 64, 4, MODE>(a, p, o, TK_GRID_CAP, s);
  else if (packs <= 512) launch_rows_as<T, 64, 8, MODE>(a, p, o, TK_GRID_CAP, s);
  else if (packs <= 1024) launch_rows_as<T, 256, 4, MODE>(a, p, o, TK_GRID_CAP, s);
  else if (packs <= 2048) launch_rows_as<T, 256, 8, MODE>(a, p, o, TK_GRID_CAP, s);
  else if (packs <= 4096) launch_rows_as<T, 1024, 4, MODE>(a, p, o, TK_GRID_CAP, s);
  else if (packs <= 8192) launch_rows_as<T, 1024, 8, MODE>(a, p, o, TK_GRID_CAP, s);
  else hipLaunchKernelGGL((k_token_rows_long<T, MODE>), dim3(row_grid(a.n, TK_GRID_CAP)), dim3(1024), 0, s, a, p, o);
}
template <int MODE> static void launch_rows_dtype(int dtype, const TokenRows& a, const PolicyIn& p, const RowOut& o, hipStream_t s) {
  if (a.n == 0) return;
  if (dtype == LIGDIFF_F32) launch_rows<float, MODE>(a, p, o, s);
  else if (dtype == LIGDIFF_BF16) launch_rows<bf16_t, MODE>(a, p, o, s);
  else launch_rows<f16_t, MODE>(a, p, o, s);
}
template <typename T>
static void launch_grad(const TokenRows& a, const float* stats, const float* coef, const int32_t* index, int64_t n_coef, float mult, const float* up, void* d,
                        int64_t d_stride, hipStream_t s) {
  const int packs = a.V / Pack<T>::N;
  const int cap = 8192;
  if (packs <= 64)
    hipLaunchKernelGGL((k_token_grad<T, 16>), dim3(row_grid((a.n + 15) / 16, cap)), dim3(256), 0, s, a, stats, coef, index, n_coef, mult, up, (T*)d, d_stride);
  else if (packs <= 512)
    hipLaunchKernelGGL((k_token_grad<T, 64>), dim3(row_grid((a.n + 3) / 4, cap)), dim3(256), 0, s, a, stats, coef, index, n_coef, mult, up, (T*)d, d_stride);
  else
    hipLaunchKernelGGL((k_token_grad<T, 256>), dim3(row_grid(a.n, cap)), dim3(256), 0, s, a, stats, coef, index, n_coef, mult, up, (T*)d, d_stride);
}
static void launch_grad_dtype(int dtype, const TokenRows& a, const float* stats, const float* coef, const int32_t* index,
                              int64_t n_coef, float mult, const float* up, void* d, int64_t d_stride, hipStream_t s) {
  if (a.n == 0) return;
  if (dtype == LIGDIFF_F32) launch_grad<float>(a, stats, coef, index, n_coef, mult, up, d, d_stride, s);
  else if (dtype == LIGDIFF_BF16) launch_grad<bf16_t>(a, stats, coef, index, n_coef, mult, up, d, d_stride, s);
  else launch_grad<f16_t>(a, stats, coef, index, n_coef, mult, up, d, d_stride, s);
}

static int fill_rows(TokenRows* r, const ligdiff_token_args* a) {
  if (!a || a->n_tokens < 0 || a->n_tokens > 0x7fffffffLL || a->vocab < 1 || a->row_stride < a->vocab ||
      a->dtype < LIGDIFF_F32 || a->dtype > LIGDIFF_F16 || (a->token_bytes != 4 && a->token_bytes != 8) ||
      !(a->temperature > 0.f) || !(a->temperature <= 3.0e38f))
    return LIGDIFF_ERR_ARG;
  if (a->n_tokens > 0 && (!a->logits || !a->tokens)) return LIGDIFF_ERR_ARG;
  r->x = a->logits; r->stride = a->row_stride; r->n = a->n_tokens; r->V = a->vocab;
  r->tok = TokenView{a->tokens, a->token_bytes, a->vocab};
  r->c = (float)(TK_LOG2E / (double)a->temperature);
  r->inv_t = 1.0 / (double)a->temperature;
  return LIGDIFF_OK;
}

extern "C" int ligdiff_token_logprob(const ligdiff_token_args* args, float* logp, float* stats, void* stream) {
  TokenRows a;
  const int rc = fill_rows(&a, args);
  if (rc) return rc;
  if (a.n > 0 && !logp) return LIGDIFF_ERR_ARG;
  launch_rows_dtype<TK_LOGP>(args->dtype, a, PolicyIn{}, RowOut{logp, nullptr, stats, nullptr, nullptr, 0, nullptr}, (hipStream_t)stream);
  LD_CHECK_LAUNCH();
  return LIGDIFF_OK;
}

extern "C" int ligdiff_token_logprob_grad(const ligdiff_token_args* args, const float* stats, const float* coef,
                                          const int32_t* coef_index, int64_t n_coef, float mult, const float* upstream,
                                          void* d_logits, int64_t d_stride, void* stream) {
  TokenRows a;
  const int rc = fill_rows(&a, args);
  if (rc) return rc;
  if (a.n > 0 && (!stats || !coef || !d_logits || d_stride < a.V || n_coef < (coef_index ? 1 : a.n))) return LIGDIFF_ERR_ARG;
  launch_grad_dtype(args->dtype, a, stats, coef, coef_index, n_coef, mult, upstream, d_logits, d_stride, (hipStream_t)stream);
  LD_CHECK_LAUNCH();
  return LIGDIFF_OK;
}

static int64_t seg_chunks(int64_t n) { return (n + SEG_ROWS - 1) / SEG_ROWS; }
// A workspace is cut into 256-byte aligned pieces.
struct Pieces {
  char* base;
  size_t used = 0;
  template <typename P> P* take(size_t n) {
    P* p = reinterpret_cast<P*>(base + used);
    used += align_up(n * sizeof(P), 256);
    return p;
  }
};
#define PREF_BLOCKS 1024
struct PrefWs { uint32_t* counter; double* partial; float* diff; double* part_sum; int32_t* part_len; size_t bytes; };
static PrefWs pref_ws(void* base, int64_t n, int32_t P) {
  Pieces w{(char*)base};
  const size_t parts = (size_t)(seg_chunks(n) + 2 * (int64_t)P);
  PrefWs r;
  r.counter = w.take<uint32_t>(1);
  r.partial = w.take<double>(PREF_BLOCKS);
  r.diff = w.take<float>((size_t)n);
  r.part_sum = w.take<double>(parts);
  r.part_len = w.take<int32_t>(parts);
  r.bytes = w.used;
  return r;
}
extern "C" size_t ligdiff_preference_workspace_bytes(int64_t n_tokens, int32_t n_pairs) {
  if (n_tokens < 0 || n_tokens > 0x7fffffffLL || n_pairs < 1 || n_pairs > 0x3fffffff) return 0;
  return pref_ws(nullptr, n_tokens, n_pairs).bytes;
}

extern "C" int ligdiff_preference_loss(const ligdiff_token_args* args, const ligdiff_preference_args* q, void* stream) {
  TokenRows a;
  const int rc = fill_rows(&a, args);
  if (rc) return rc;
  if (!q || !q->seq_ptr || q->n_pairs < 1 || q->n_pairs > 0x3fffffff || !(q->beta > 0.f) || !(q->beta <= 3.0e38f) ||
      !(q->label_smoothing >= 0.f) || !(q->label_smoothing < 0.5f) ||
      (q->kind != LIGDIFF_PREFERENCE_SIGMOID && q->kind != LIGDIFF_PREFERENCE_IPO) || !q->loss || !q->log_ratio || !q->margin ||
      !q->slope || !q->workspace || q->denominator != q->denominator || q->grad_scale != q->grad_scale)
    return LIGDIFF_ERR_ARG;
  if (a.n > 0 && (!q->stats || !q->row_seq)) return LIGDIFF_ERR_ARG;
  if (a.n > 0 && q->d_logits && q->d_stride < a.V) return LIGDIFF_ERR_ARG;
  const PrefWs w = pref_ws(q->workspace, a.n, q->n_pairs);
  if (q->workspace_bytes < w.bytes) return LIGDIFF_ERR_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  if (a.n > 0) {
    launch_rows_dtype<TK_LOGP>(args->dtype, a, PolicyIn{}, RowOut{w.diff, q->ref_logp, q->stats, nullptr, nullptr, 0, w.counter}, s);
    hipLaunchKernelGGL((k_row_segments<true>), dim3((unsigned)seg_chunks(a.n)), dim3(256), 0, s, a.tok, a.n, q->seq_ptr,
                       2 * q->n_pairs, w.diff, q->row_seq, w.part_sum, w.part_len, (int32_t*)nullptr, (uint32_t*)nullptr);
  } else {
    hipLaunchKernelGGL(k_clear, dim3(1), dim3(64), 0, s, w.counter);
  }
  PrefIn p;
  p.n = a.n; p.seq_ptr = q->seq_ptr; p.P = q->n_pairs; p.part_sum = w.part_sum; p.part_len = w.part_len;
  p.beta = q->beta; p.smooth = q->label_smoothing; p.kind = q->kind; p.average = q->average != 0;
  p.denom = q->denominator > 0.f ? (double)q->denominator : (double)q->n_pairs;
  p.grad_scale = (double)q->grad_scale;
  p.loss = q->loss; p.log_ratio = q->log_ratio; p.margin = q->margin; p.slope = q->slope;
  p.partial = w.partial; p.counter = w.counter;
  hipLaunchKernelGGL(k_preference, dim3(row_grid(((int64_t)q->n_pairs + 3) / 4, PREF_BLOCKS)), dim3(256), 0, s, p);
  if (q->d_logits)
    launch_grad_dtype(args->dtype, a, q->stats, q->slope, q->row_seq, 2 * (int64_t)q->n_pairs, 1.0f, nullptr, q->d_logits, q->d_stride, s);
  LD_CHECK_LAUNCH();
  return LIGDIFF_OK;
}

struct PolicyWs { uint32_t* counter; double* partial; int32_t* chunk_len; int32_t* seq_of; int32_t* part_len; int32_t* seq_len; size_t bytes; };
static PolicyWs policy_ws(void* base, int64_t n, int32_t S, bool per_seq) {
  Pieces w{(char*)base};
  PolicyWs r;
  r.counter = w.take<uint32_t>(1);
  r.partial = w.take<double>(TK_GRID_CAP * 3);
  r.chunk_len = w.take<int32_t>((size_t)seg_chunks(n));
  r.seq_of = w.take<int32_t>((size_t)n);
  r.part_len = w.take<int32_t>(per_seq ? (size_t)(seg_chunks(n) + S) : 0);
  r.seq_len = w.take<int32_t>(per_seq ? (size_t)S : 0);
  r.bytes = w.used;
  return r;
}
extern "C" size_t ligdiff_policy_workspace_bytes(int64_t n_tokens, int32_t n_seq, int32_t aggregate) {
  if (n_tokens < 0 || n_tokens > 0x7fffffffLL || n_seq < 1) return 0;
  return policy_ws(nullptr, n_tokens, n_seq, aggregate == LIGDIFF_POLICY_SEQUENCE_MEAN).bytes;
}

extern "C" int ligdiff_policy_loss(const ligdiff_token_args* args, const ligdiff_policy_args* q, void* stream) {
  TokenRows a;
  const int rc = fill_rows(&a, args);
  if (rc) return rc;
  if (!q || q->n_seq < 1 || (!q->seq_ptr && q->n_seq != 1) || !(q->clip_low >= 0.f) || !(q->clip_low <= 1.f) ||
      !(q->clip_high >= 0.f) || !(q->clip_high <= 3.0e38f) || !(q->kl_coef >= 0.f) || !(q->kl_coef <= 3.0e38f) ||
      (q->aggregate != LIGDIFF_POLICY_TOKEN_MEAN && q->aggregate != LIGDIFF_POLICY_SEQUENCE_MEAN) || !q->result ||
      !q->workspace || q->denominator != q->denominator || q->grad_scale != q->grad_scale)
    return LIGDIFF_ERR_ARG;
  if (a.n > 0 && (!q->advantage || (q->d_logits && q->d_stride < a.V))) return LIGDIFF_ERR_ARG;
  const bool per_seq = q->aggregate == LIGDIFF_POLICY_SEQUENCE_MEAN;
  const PolicyWs w = policy_ws(q->workspace, a.n, q->n_seq, per_seq);
  if (q->workspace_bytes < w.bytes) return LIGDIFF_ERR_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  if (a.n == 0) {
    hipLaunchKernelGGL(k_empty_policy, dim3(1), dim3(64), 0, s, q->result);
    LD_CHECK_LAUNCH();
    return LIGDIFF_OK;
  }
  const int chunks = (int)seg_chunks(a.n);
  hipLaunchKernelGGL((k_row_segments<false>), dim3(chunks), dim3(256), 0, s, a.tok, a.n, q->seq_ptr, q->n_seq, (const float*)nullptr,
                     w.seq_of, (double*)nullptr, per_seq ? w.part_len : nullptr, w.chunk_len, w.counter);
  if (per_seq)
    hipLaunchKernelGGL(k_sequence_lengths, dim3(ceil_div(q->n_seq, 4)), dim3(256), 0, s, q->seq_ptr, a.n, q->n_seq, w.part_len, w.seq_len);
  PolicyIn p;
  p.seq_of = w.seq_of; p.seq_len = w.seq_len; p.chunk_len = w.chunk_len; p.n_chunks = chunks;
  p.denom = (double)q->denominator; p.n_seq = q->n_seq; p.per_seq_mean = per_seq;
  p.adv = q->advantage; p.adv_per_token = q->advantage_per_token != 0;
  p.old_logp = q->old_logp; p.ref_logp = q->ref_logp;
  p.clip_lo = q->clip_low; p.clip_hi = q->clip_high; p.kl_coef = q->kl_coef; p.grad_scale = q->grad_scale;
  p.partial = w.partial; p.counter = w.counter; p.result = q->result;
  launch_rows_dtype<TK_POLICY>(args->dtype, a, p, RowOut{q->logp, nullptr, q->stats, q->coef, q->d_logits, q->d_stride, nullptr}, s);
  LD_CHECK_LAUNCH();
  return LIGDIFF_OK;
}
