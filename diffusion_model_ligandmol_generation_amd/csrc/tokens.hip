// Losses on the log-probabilities of chosen ids (atom types, or tokens of any vocabulary), x = logits / temperature:
//   logp_t = x[t, id_t] - log sum_v exp(x[t, v])            d logp_t / d x[t, v] = [v = id_t] - p[t, v]
// so every loss below reaches the logits as  d_logits[t, v] = coef_t / temperature ([v = id_t] - p[t, v])  with one number
// coef_t = d loss / d logp_t for each row.  All of them are bound by HBM: a logit costs a handful of vector operations and
// its bytes are read once (and a gradient of the same size written once): log-probabilities of 8192 rows of 32000 bf16 in
// 94 us (5.3 TB/s), policy loss with gradient 207 us (4.9 TB/s), of 593920 rows of 119 fp32 116 us (4.9 TB/s).
#include "token_common.h"

#define TK_LOG2E 1.44269504088896340736

struct TokenRows {
  const void* x;
  int64_t stride;      // elements between rows
  int64_t n;           // rows
  int32_t V;
  TokenView tok;
  float c, c_lo;       // log2(e) / temperature = c + c_lo, 0 < c_lo <= the last place of c: exp(x / temperature) = exp2((c + c_lo) x)
  double inv_t;        // 1 / temperature
};

// exp((x - m) / temperature) of a row with maximum m is exp2(exponent(x)).  x - m is exact where it matters (near m), the product
// is rounded once.  One constant would do for the exponentials, but its rounding is a temperature that is off by up to 2^-25:
// the same error 1.3e-8 (z - E[z]) in every log-probability, which sums over a sequence add up (29 atoms: twice the error
// of the plain form).  Both parts are above 0, so that a masked -inf stays -inf.
__device__ __forceinline__ float scaled(const TokenRows& a, float d) { return fmaf(d, a.c, d * a.c_lo); }
__device__ __forceinline__ float exponent(const TokenRows& a, float x, float m) {
  return scaled(a, x - m);
}

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
// In 32 bits: see row_epilogue.
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
    kl = em1 < __builtin_inff() ? em1 - q : em1;   // (q = inf: infinite, and NaN stays NaN)
  }
}

enum { TK_LOGP = 0, TK_POLICY = 1, TK_SMALL = 2 };   // TK_SMALL: the policy loss of at most SMALL_ROWS rows, by one block
#define SMALL_ROWS 64

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
  double* partial;           // [gridDim.x][3]: surrogate, kl, share of clipped rows
  const int32_t* seq_ptr;    // small batches: their one block finds the sequences itself
  float* result;             // and writes the result
};
struct RowOut {
  float* logp;               // [n] or null
  const float* minus;        // [n] or null: subtracted from logp (difference of two policies)
  float* stats;              // [n][2]: row maximum and 1 / sum, for the gradient kernel; may be null
  float* coef;               // [n] d loss / d logp (TK_POLICY); may be null
  void* d;                   // gradient of the logits or null
  int64_t d_stride;
};

// What is known of a row besides its logits; loaded one row ahead, so that a row costs one memory latency.
struct RowScalars { int id, seq; float old, ref; };
// A value that all lanes of the wave share, in a scalar register.
__device__ __forceinline__ float uniform(float v) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v))); }
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ double uniform(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)u), hi = __builtin_amdgcn_readfirstlane((uint32_t)(u >> 32));
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int MODE> __device__ __forceinline__ RowScalars row_scalars(const TokenRows& a, const PolicyIn& p, const RowOut& o, int64_t t) {
  RowScalars r{-1, 0, 0.f, 0.f};
  if (t >= a.n) return r;
  r.id = a.tok.at(t);
  if constexpr (MODE != TK_LOGP) {
    if (MODE == TK_POLICY) r.seq = p.seq_of[t];
    if (p.old_logp) r.old = p.old_logp[t];
    if (p.ref_logp) r.ref = p.ref_logp[t];
  } else if (o.minus) r.ref = o.minus[t];
  return r;
}

// What a row contributes once its maximum M and sum S are known, the same in every lane of the row; returns the gradient's
// factor d loss / d logp * grad_scale / temperature.
// logp is in 64 bits up to its differences with old_logp and ref_logp, which are rounded once to 32; ratio, clip bounds, gain, KL
// term and slope are in 32 bits from there on: the softmax sum under them is (its error, up to 1e-7, reaches all of them), and
// a row of 119 logits has as much work in these few numbers as in its exponentials.  Their sums are in 64 bits again.
template <int MODE>
__device__ __forceinline__ float row_epilogue(const TokenRows& a, const PolicyIn& p, const RowOut& o, int64_t t, const RowScalars& c,
                                              float xt, float M, float S, float inv_s, bool writer, float A, double w, double* acc) {
  // a row of -inf only has no distribution: S = 0, logp = -inf, no gradient
  const double z = ((double)xt - (double)M) * a.inv_t;
  const double lp = S == 0.f ? -__builtin_inf() : z - log_of_sum(S);
  float g = 0.f, coef = 0.f;
  if constexpr (MODE != TK_LOGP) {
    const float rho = p.old_logp ? expf((float)(lp - (double)c.old)) : lp == lp ? 1.0f : (float)lp;
    const float hi = 1.0f + p.clip_hi, lo = 1.0f - p.clip_lo;
    const bool clipped = (A > 0.f && rho > hi) || (A < 0.f && rho < lo);
    const float gain = A == 0.f ? 0.f : fminf(rho * A, fminf(fmaxf(rho, lo), hi) * A);
    float slope = clipped || A == 0.f ? 0.f : -A * rho;
    float em1 = 0.f, kl = 0.f;
    if (p.ref_logp) {
      kl_terms((float)((double)c.ref - lp), em1, kl);
      if (p.kl_coef != 0.f) slope -= p.kl_coef * em1;   // (an infinite term that does not count reaches nothing)
    }
    if (rho != rho) slope = rho;   // fminf drops a NaN
    if (writer) {
      acc[0] -= w * (double)(rho != rho ? rho : gain);
      acc[1] += w * (double)kl;
      acc[2] += clipped ? w : 0.0;
    }
    coef = (float)(w * (double)slope);
    if (S != 0.f) g = (float)(w * (double)slope * (double)p.grad_scale * a.inv_t);
  }
  if (writer) {
    if (o.logp) o.logp[t] = (float)(MODE == TK_LOGP ? lp - (double)c.ref : lp);
    if (o.stats) { o.stats[2 * t] = M; o.stats[2 * t + 1] = inv_s; }
    if (o.coef) o.coef[t] = coef;
  }
  return g;
}

template <typename T> __device__ __forceinline__ void row_zero(T* d, int V, int r, int tpr) {
  constexpr int N = Pack<T>::N;
  const float z[N] = {};
  const int nb = V / N;
  for (int i = r; i < nb; i += tpr) store_pack(d + (int64_t)i * N, z);
  if (r < V - nb * N) d[nb * N + r] = (T)0.f;
}
// Writes the rows that a wave has left in LDS as one run of memory.  Rows of a few hundred bytes that end inside cache lines,
// written by 8 lanes each, would touch every line in two or three pieces.  A wave's LDS operations are in order: no barrier.
template <typename T> __device__ __forceinline__ void write_flat(const T* stage, T* d, int count) {
  constexpr int N = Pack<T>::N;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  const int lane = threadIdx.x & 63, packs = count / N;
#pragma unroll 4
  for (int i = lane; i < packs; i += 64)
    *reinterpret_cast<typename Pack<T>::Mem*>(d + (int64_t)i * N) = *reinterpret_cast<const u32x4*>(stage + i * N);
  if (lane < count - packs * N) d[packs * N + lane] = stage[packs * N + lane];
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

// A row that takes no part: nothing of it is read, its log-probability and its gradient are 0.
template <typename T>
__device__ __forceinline__ void row_skip(const RowOut& o, int64_t t, int V, int r, int tpr, bool writer) {
  if (writer) {
    if (o.logp) o.logp[t] = 0.f;
    if (o.stats) { o.stats[2 * t] = 0.f; o.stats[2 * t + 1] = 0.f; }
    if (o.coef) o.coef[t] = 0.f;
  }
  if (o.d) row_zero(reinterpret_cast<T*>(o.d) + t * o.d_stride, V, r, tpr);
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
// Per-block sums to memory; k_policy_final adds them up in block order.  (A last block that did it inside this launch would
// need a release fence in every block, which writes back its XCD's L2: 30 us for 1200 blocks against 3 for a launch.)
template <int RPB> __device__ __forceinline__ void policy_partial(const PolicyIn& p, const double (&acc)[RPB][3]) {
  __syncthreads();
  if (threadIdx.x < 3) {
    double v = acc[0][threadIdx.x];
    for (int g = 1; g < RPB; ++g) v += acc[g][threadIdx.x];
    p.partial[(int64_t)blockIdx.x * 3 + threadIdx.x] = v;
  }
}
// The only block of a small batch: the sequence of each row and the number of its sequence's rows, and 1 / the total.
__device__ __forceinline__ double small_rows(const TokenRows& a, const PolicyIn& p, int* seq, int* len) {
  const int t = threadIdx.x;
  __shared__ int count;
  if (t < 64) {
    int s = -1;
    if (t < (int)a.n && a.tok.at(t) >= 0) {
      s = 0;
      if (p.seq_ptr) {
        uint32_t lo = 0, hi = (uint32_t)p.n_seq + 1u;   // the number of offsets <= t
        while (lo < hi) {
          const uint32_t mid = lo + ((hi - lo) >> 1);
          if (p.seq_ptr[mid] <= t) lo = mid + 1; else hi = mid;
        }
        s = lo > (uint32_t)p.n_seq ? -1 : (int)lo - 1;
      }
    }
    seq[t] = s;
    int same = 0;
    for (int k = 0; k < 64; ++k) same += __shfl(s, k) == s;
    len[t] = same;
    const int all = __popcll(__ballot(s >= 0));
    if (t == 0) count = all;
  }
  __syncthreads();
  const double total = p.denom > 0.0 ? p.denom : p.per_seq_mean ? (double)p.n_seq : (double)count;
  return total > 0.0 ? 1.0 / total : 0.0;
}
template <int RPB> __device__ __forceinline__ void policy_result(const PolicyIn& p, const double (&acc)[RPB][3]) {
  __syncthreads();
  if (threadIdx.x == 0) {
    double v[3] = {0.0, 0.0, 0.0};
    for (int g = 0; g < RPB; ++g)
#pragma unroll
      for (int k = 0; k < 3; ++k) v[k] += acc[g][k];
    p.result[0] = (float)(p.kl_coef != 0.f ? v[0] + (double)p.kl_coef * v[1] : v[0]);
    p.result[1] = (float)v[0];
    p.result[2] = (float)v[1];
    p.result[3] = (float)v[2];
  }
}
__global__ __launch_bounds__(256) void k_policy_final(const double* __restrict__ partial, int blocks, double kl_coef, float* __restrict__ result) {
  __shared__ double red[4];
  double v[3] = {0.0, 0.0, 0.0};
#pragma unroll 4
  for (int b = threadIdx.x; b < blocks; b += 256)
#pragma unroll
    for (int k = 0; k < 3; ++k) v[k] += partial[(int64_t)b * 3 + k];
#pragma unroll
  for (int k = 0; k < 3; ++k) v[k] = block_sum<256>(v[k], red);
  if (threadIdx.x == 0) {
    result[0] = (float)(kl_coef != 0.0 ? v[0] + kl_coef * v[1] : v[0]);
    result[1] = (float)v[0];
    result[2] = (float)v[1];
    result[3] = (float)v[2];
  }
}

// What a sum relative to a maximum m counts in a row with maximum M (m = -inf: nothing).
__device__ __forceinline__ float part_factor(const TokenRows& a, float m, float M) { return __builtin_amdgcn_exp2f(exponent(a, m, M)); }
// The maximum and sum of a row from those of its 4, 8 or 16 waves (0 and 0 for a row of -inf only).
template <int NW> __device__ __forceinline__ void join_waves(const TokenRows& a, const float2* sh, float& M, float& S) {
  const float2 v = sh[threadIdx.x & (NW - 1)];
  M = v.x;
  M = fmaxf(M, dpp_move<0xB1>(M));
  M = fmaxf(M, dpp_move<0x4E>(M));
  if (NW >= 8) M = fmaxf(M, dpp_move<0x141>(M));
  if (NW == 16) M = fmaxf(M, dpp_move<0x140>(M));
  if (M == -__builtin_inff()) M = 0.f;
  S = v.y * part_factor(a, v.x, M);
  S += dpp_move<0xB1>(S);
  S += dpp_move<0x4E>(S);
  if (NW >= 8) S += dpp_move<0x141>(S);
  if (NW == 16) S += dpp_move<0x140>(S);
}
// The maximum of a pack and m; fp16 in packed instructions.
template <typename T> __device__ __forceinline__ float max_pack(const u32x4& x, float m) {
  if constexpr (std::is_same<T, f16_t>::value) {
    f16x2 v = __builtin_elementwise_max(__builtin_bit_cast(f16x2, (uint32_t)x[0]), __builtin_bit_cast(f16x2, (uint32_t)x[1]));
    v = __builtin_elementwise_max(v, __builtin_elementwise_max(__builtin_bit_cast(f16x2, (uint32_t)x[2]), __builtin_bit_cast(f16x2, (uint32_t)x[3])));
    return fmaxf(m, fmaxf((float)v[0], (float)v[1]));
  }
#pragma unroll
  for (int j = 0; j < Pack<T>::N; ++j) m = fmaxf(m, raw_get<T>(x, j));
  return m;
}
// The exponentials of a lane's packs, handed on one pack at a time.  Half-precision packs stay packed until then (the compiler
// would keep the values that it unpacked for the maximum, twice the registers): the policy loss exponentiates them a second
// time for its gradient rather than hold 32-bit results, which halves the rows in flight.
__device__ __forceinline__ void set_pack(u32x4& x, const float (&v)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = __float_as_uint(v[j]);
}
template <typename T, int NV, int TPR, typename F>
__device__ __forceinline__ void exponentials(const TokenRows& a, u32x4 (&x)[NV], int nb, float m, F&& take) {
  constexpr int N = Pack<T>::N;
  float one = 1.f;   // (not known to the compiler: fp16 converts and subtracts in one instruction, a mixed fma)
  if (std::is_same<T, f16_t>::value) asm volatile("" : "+s"(one));
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    if (k > 0 && k * TPR >= nb) break;   // no lane has a pack here
    if (sizeof(T) == 2) asm volatile("" : "+v"(x[k]));
    float e[N];
#pragma unroll
    for (int j = 0; j < N; ++j) e[j] = __builtin_amdgcn_exp2f(scaled(a, std::is_same<T, f16_t>::value ? fmaf(raw_get<T>(x[k], j), one, -m) : raw_get<T>(x[k], j) - m));
    take(k, e);
    __builtin_amdgcn_sched_barrier(0);
  }
}
// A pack's exponentials added to a lane's sum.  Eight go by pairs: one after the other, 16 packs would be 128 additions to one
// sum, twice those of a row of fp32.
template <int N> __device__ __forceinline__ float add_pack(float s, const float (&e)[N]) {
  if constexpr (N == 8) return s + (((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7])));
#pragma unroll
  for (int j = 0; j < N; ++j) s += e[j];
  return s;
}
// Half-precision rows that start between two 32-bit words (odd strides): packs across word borders come slower.  Where many
// blocks of few lanes hold rows in registers it shows less (6007 rows of 32003 bf16 92 us, of 32004 75); the kernel that streams
// longer rows reads whole words, five a pack, and shifts them (another partition of the row would be another order of its sum,
// which would then change with the stride).  The halves before and behind the pack that come with the words lie in words of
// the row's own ends.  (Log-probabilities of 1601 rows of 120001 bf16 94 us without, 86 with them.)
template <typename T, int TPR> __device__ __forceinline__ bool between_words(const T* row) {
  return sizeof(T) == 2 && TPR >= 256 && uniform((int)reinterpret_cast<uintptr_t>(row) & 2);
}
template <typename T> __device__ __forceinline__ u32x4 load_words(const T* p, uint32_t& last) {
  typedef uint32_t words __attribute__((ext_vector_type(4), aligned(4)));
  last = *reinterpret_cast<const uint32_t*>(p + 7);
  return *reinterpret_cast<const words*>(p - 1);
}
__device__ __forceinline__ void shift_words(u32x4& x, uint32_t last) {
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = __builtin_amdgcn_alignbit(j < 3 ? x[j < 3 ? j + 1 : 3] : last, x[j], 16);
}
// Short rows are loaded one row ahead of their arithmetic: a wave has two rows' bytes under way.
#define ROW_AHEAD(REGS) ((REGS) <= 8)
// Waves a SIMD holds at once: what the registers of a row allow.
#define ROW_WAVES(REGS, MODE) ((REGS) > 16 ? 4 : (MODE) == TK_LOGP ? 8 : (REGS) <= 8 ? 6 : 5)

// Rows that fit the registers of TPR lanes, NV packs a lane: the logits are read once, exponentiated once, and the policy
// loss writes its gradient from the same registers.  TPR = 8 / 16 / 64: several rows a block and no barrier; 256 / 512 / 1024:
// one row a block, whose waves take the maximum and sum of their own part and exchange the pair once.
// STAGE: gradients of ragged short rows are written through LDS.
template <typename T, int TPR, int NV, int MODE, bool STAGE = false>
__global__ __launch_bounds__(TPR <= 64 ? 256 : TPR, ROW_WAVES(NV * 4, MODE)) void k_token_rows(TokenRows a, PolicyIn p, RowOut o) {
  constexpr int N = Pack<T>::N, NT = TPR <= 64 ? 256 : TPR, RPB = NT / TPR, NW = TPR / 64, GRP = TPR < 64 ? TPR : 64;
  constexpr bool KEEP = MODE != TK_LOGP && sizeof(T) == 4;   // the exponentials take the logits' registers
  constexpr bool AHEAD = ROW_AHEAD(NV * 4);
  constexpr int STAGE_ROWS = 64 / (TPR < 64 ? TPR : 64), STAGE_V = TPR * NV * N + N;   // (a multiple of a pack)
  __shared__ __attribute__((aligned(16))) T stage[STAGE ? NT / 64 * STAGE_ROWS * STAGE_V : 1];
  __shared__ float2 sh[2][NW > 1 ? NW : 1];
  __shared__ double red[NT / 64];
  __shared__ double acc[MODE != TK_LOGP ? RPB : 1][3];
  __shared__ int small_seq[MODE == TK_SMALL ? SMALL_ROWS : 1], small_len[MODE == TK_SMALL ? SMALL_ROWS : 1];
  const int r = TPR <= 64 ? threadIdx.x % TPR : threadIdx.x;
  const int mine = TPR < 64 ? threadIdx.x / TPR : TPR == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x / 64) : 0;
  const int V = a.V, nb = V / N, tail = V - nb * N;
  double inv_total = 0.0;
  if constexpr (MODE != TK_LOGP) {
    if (threadIdx.x < RPB * 3) acc[threadIdx.x / 3][threadIdx.x % 3] = 0.0;
    if constexpr (MODE == TK_SMALL) inv_total = small_rows(a, p, small_seq, small_len);
    else inv_total = uniform(inverse_total<NT>(p, red));
    __syncthreads();
  }
  int parity = 0;
  const int64_t step = (int64_t)gridDim.x * RPB;
  const auto scalars = [&](int64_t t) {
    RowScalars c = row_scalars<MODE>(a, p, o, t);
    if (MODE == TK_SMALL && t < a.n) c.seq = small_seq[t];
    if (MODE != TK_LOGP && c.seq < 0) c.id = -1;
    return c;
  };
  const auto load = [&](const RowScalars& c, int64_t t, u32x4 (&x)[NV], float& et, float& xt, float& A, int& len) {
    const T* row = reinterpret_cast<const T*>(a.x) + t * a.stride;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      x[k] = raw_minus_inf<T>();
      if (r + k * TPR < nb) x[k] = load_raw(row + (int64_t)(r + k * TPR) * N);
    }
    et = -__builtin_inff();
    if (r < tail) et = (float)row[nb * N + r];
    xt = (float)row[c.id];
    if constexpr (MODE != TK_LOGP) {
      A = p.adv[p.adv_per_token ? t : (int64_t)c.seq];
      len = !p.per_seq_mean ? 1 : MODE == TK_SMALL ? small_len[t] : p.seq_len[c.seq];
    }
  };
  RowScalars next = scalars((int64_t)blockIdx.x * RPB + mine), after{};
  u32x4 x1[AHEAD ? NV : 1];
  float et1 = 0.f, xt1 = 0.f, A1 = 0.f;
  int len1 = 1;
  if constexpr (AHEAD) {
    if (next.id >= 0) load(next, (int64_t)blockIdx.x * RPB + mine, x1, et1, xt1, A1, len1);
    after = scalars((int64_t)blockIdx.x * RPB + mine + step);
  }
  for (int64_t base = (int64_t)blockIdx.x * RPB; base < a.n; base += step) {
    const int64_t t = base + mine;
    RowScalars c = next;
    u32x4 x[NV];
    float et, xt, A = 0.f;
    int len = 1;
    if constexpr (AHEAD) {
#pragma unroll
      for (int k = 0; k < NV; ++k) x[k] = x1[k];
      et = et1; xt = xt1; A = A1; len = len1;
      next = after;
      if (next.id >= 0) load(next, t + step, x1, et1, xt1, A1, len1);
      after = scalars(t + 2 * step);
    } else {
      if constexpr (TPR >= 64) c = RowScalars{uniform(c.id), uniform(c.seq), uniform(c.old), uniform(c.ref)};
      next = scalars(t + step);
    }
    const auto work = [&]() {
    if (TPR <= 64 && t >= a.n) return;
    const int id = c.id;
    T* const staged = stage + (STAGE ? (threadIdx.x >> 6) * STAGE_ROWS * STAGE_V + (threadIdx.x & 63) / TPR * V : 0);
    if (id < 0) {
      row_skip<T>(STAGE ? RowOut{o.logp, nullptr, o.stats, o.coef, nullptr, 0} : o, t, V, r, TPR, r == 0);
      if constexpr (STAGE) row_zero(staged, V, r, TPR);
      return;
    }
    if constexpr (!AHEAD) load(c, t, x, et, xt, A, len);
    double w = 0.0;
    if constexpr (MODE != TK_LOGP) w = p.per_seq_mean ? inv_total / (double)len : inv_total;
    float m = et;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (k > 0 && k * TPR >= nb) break;
      m = max_pack<T>(x[k], m);
    }
    m = group_max<GRP>(m);
    // this wave's own part, relative to its own maximum
    const bool none = m == -__builtin_inff();
    if (none) m = 0.f;
    float s = et = __builtin_amdgcn_exp2f(exponent(a, et, m));
    exponentials<T, NV, TPR>(a, x, nb, m, [&](int k, float (&e)[N]) {
      s = add_pack(s, e);
      if constexpr (KEEP) set_pack(x[k], e);
    });
    s = group_sum<GRP>(s);
    float M = m, S = s, f = 1.0f;
    if constexpr (NW > 1) {
      // (the buffers alternate between rows: a wave that runs ahead writes the other one)
      if ((threadIdx.x & 63) == 0) sh[parity][threadIdx.x >> 6] = make_float2(none ? -__builtin_inff() : m, s);
      __syncthreads();
      join_waves<NW>(a, sh[parity], M, S);
      f = none ? 0.f : part_factor(a, m, M);
      parity ^= 1;
    }
    float inv_s = S == 0.f ? 0.f : 1.0f / S;
    if constexpr (TPR >= 64) {
      inv_s = uniform(inv_s);
      xt = uniform(xt); M = uniform(M); S = uniform(S);
      if constexpr (MODE != TK_LOGP) { A = uniform(A); w = uniform(w); }
    }
    float g = row_epilogue<MODE>(a, p, o, t, c, xt, M, S, inv_s, r == 0, A, w, acc[MODE != TK_LOGP ? mine : 0]);
    if constexpr (TPR >= 64) g = uniform(g);
    if constexpr (MODE != TK_LOGP) {
      if (!STAGE && o.d == nullptr) return;
      const auto write = [&](T* d) {
        if (g == 0.f) {   // sends no gradient, also where the row holds a NaN
          row_zero(d, V, r, TPR);
          return;
        }
        const float q = -g * f * inv_s;
        const int it = id / N;
        const auto out = [&](int k, float (&e)[N]) {
          const int i = r + k * TPR;
#pragma unroll
          for (int j = 0; j < N; ++j) e[j] *= q;
          if (i == it) {
#pragma unroll
            for (int j = 0; j < N; ++j) e[j] += j == id - it * N ? g : 0.f;
          }
          if (i < nb) store_pack(d + (int64_t)i * N, e);
        };
        if constexpr (KEEP) {
#pragma unroll
          for (int k = 0; k < NV; ++k) {
            float e[N];
#pragma unroll
            for (int j = 0; j < N; ++j) e[j] = raw_get<T>(x[k], j);
            out(k, e);
          }
        } else {
          exponentials<T, NV, TPR>(a, x, nb, m, out);
        }
        if (r < tail) d[nb * N + r] = (T)(q * et + (nb * N + r == id ? g : 0.f));
      };
      if constexpr (STAGE) write(staged);
      else write(reinterpret_cast<T*>(o.d) + t * o.d_stride);
    }
    };
    work();
    if constexpr (STAGE) {
      const int64_t t0 = base + (int64_t)(threadIdx.x >> 6) * STAGE_ROWS;
      if (t0 < a.n)
        write_flat(stage + (threadIdx.x >> 6) * STAGE_ROWS * STAGE_V, reinterpret_cast<T*>(o.d) + t0 * V,
                   (int)(a.n - t0 < STAGE_ROWS ? a.n - t0 : STAGE_ROWS) * V);
    }
  }
  if constexpr (MODE == TK_POLICY) policy_partial<RPB>(p, acc);
  if constexpr (MODE == TK_SMALL) policy_result<RPB>(p, acc);
}

// One row's gradient from its logits, maximum and 1 / sum, by TPR lanes: g ([v = id] - p[v]).  A factor of 0 sends no
// gradient, also where the row holds a NaN, and a row of -inf only (1 / sum is 0) has none.
template <typename T, int TPR>
__device__ __forceinline__ void row_gradient(const TokenRows& a, const T* row, T* d, int id, int r, float M, float inv_s, float g) {
  constexpr int N = Pack<T>::N;
  // long rows: packs from the first cache line of the gradient on, which a wave then writes whole; the elements before and
  // behind them go to a lane each (preference loss of 6007 rows of 32003 bf16 284 -> 274 us, 20000 of 8201 fp32 408 -> 400)
  const int V = a.V, head = TPR >= 256 ? uniform((int)(-reinterpret_cast<uintptr_t>(d) & 127) / (int)sizeof(T)) : 0;
  const int shift = head < V ? head : V, nb = (V - shift) / N, edges = V - nb * N;
  const bool off = g == 0.f || inv_s == 0.f;
  const float q = -g * inv_s;
  const int at = id - shift, it = at < 0 ? -1 : at / N;   // (an element before the packs is in none)
  if (off) {
    row_zero(d, V, r, TPR);
    return;
  }
#pragma unroll 4
  for (int i = r; i < nb; i += TPR) {
    float v[N];
    load_pack(row + shift + (int64_t)i * N, v);
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = q * __builtin_amdgcn_exp2f(exponent(a, v[j], M));
    if (i == it) {
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] += j == at - it * N ? g : 0.f;
    }
    store_pack(d + shift + (int64_t)i * N, v);
  }
  if (r < edges) {
    const int v = r < shift ? r : nb * N + r;
    const float x = (float)row[v];
    d[v] = (T)(q * __builtin_amdgcn_exp2f(exponent(a, x, M)) + (v == id ? g : 0.f));
  }
}

// Longer rows: one block a row, running maximum and sum over the packs, and a second read for the gradient.  Log-probabilities
// at 5.0 TB/s (1373 rows of 140000 bf16 77 us).
template <typename T, int MODE>
__global__ __launch_bounds__(1024) void k_token_rows_long(TokenRows a, PolicyIn p, RowOut o) {
  constexpr int N = Pack<T>::N, NT = 1024, NW = NT / 64;
  __shared__ float2 sh[2][NW];
  __shared__ double red[NW];
  const int r = threadIdx.x;
  const int V = a.V, nb = V / N, tail = V - nb * N;
  __shared__ double acc[1][3];
  double inv_total = 0.0;
  if constexpr (MODE == TK_POLICY) {
    if (threadIdx.x < 3) acc[0][threadIdx.x] = 0.0;
    inv_total = uniform(inverse_total<NT>(p, red));
    __syncthreads();
  }
  int parity = 0;
  for (int64_t t = blockIdx.x; t < a.n; t += gridDim.x) {
    const RowScalars c = row_scalars<MODE>(a, p, o, t);
    const int id = c.id;
    if (id < 0 || c.seq < 0) {
      row_skip<T>(o, t, V, r, NT, r == 0);
      continue;
    }
    const T* row = reinterpret_cast<const T*>(a.x) + t * a.stride;
    const bool words = between_words<T, NT>(row);
    const float xt = (float)row[id];
    double w = 0.0;
    float A = 0.f;
    if constexpr (MODE == TK_POLICY) {
      A = p.adv[p.adv_per_token ? t : (int64_t)c.seq];
      w = p.per_seq_mean ? inv_total / (double)p.seq_len[c.seq] : inv_total;
    }
    float m = -__builtin_inff(), s = 0.f;   // of this lane: s relative to m
    for (int i = r; i < nb + (r < tail ? NT : 0); i += NT) {
      float v[N];
      if (i < nb) {
        u32x4 x;
        if (words) {
          uint32_t last;
          x = load_words(row + (int64_t)i * N, last);
          shift_words(x, last);
        } else x = load_raw(row + (int64_t)i * N);
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = raw_get<T>(x, j);
      } else {   // one element of the tail
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = -__builtin_inff();
        v[0] = (float)row[nb * N + r];
      }
      float mx = v[0];
#pragma unroll
      for (int j = 1; j < N; ++j) mx = fmaxf(mx, v[j]);
      if (mx > m) {
        s *= part_factor(a, m, mx);
        m = mx;
      }
      const float base = m == -__builtin_inff() ? 0.f : m;
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = __builtin_amdgcn_exp2f(exponent(a, v[j], base));
      s = add_pack(s, v);
    }
    const float wm = group_max<64>(m);
    s = group_sum<64>(s * part_factor(a, m, wm == -__builtin_inff() ? 0.f : wm));
    if ((threadIdx.x & 63) == 0) sh[parity][threadIdx.x >> 6] = make_float2(wm, s);
    __syncthreads();
    float M, S;
    join_waves<NW>(a, sh[parity], M, S);
    parity ^= 1;
    const float inv_s = S == 0.f ? 0.f : 1.0f / S;
    const float g = row_epilogue<MODE>(a, p, o, t, c, xt, M, S, inv_s, r == 0, A, w, acc[0]);
    if constexpr (MODE == TK_POLICY) {
      if (o.d) row_gradient<T, NT>(a, row, reinterpret_cast<T*>(o.d) + t * o.d_stride, id, r, M, inv_s, g);
    }
  }
  if constexpr (MODE == TK_POLICY) policy_partial<1>(p, acc);
}

// The loss of a preference step, added up by the last block of its gradient launch.
struct LossTail { const double* partial; int blocks; double denom; float* loss; };
__device__ __forceinline__ void preference_final(const LossTail& f);
// d_logits[t, v] = coef mult upstream / temperature ([v = id_t] - p[t, v]) from the saved maximum and 1 / sum: no reduction,
// the rows are streamed, 5.6 TB/s for long ones (6007 rows of 32003 bf16 130 us).  coef is that of the row, or of its sequence when an index is given.
// FLAT: 0, or the packs of the longest row that is written through LDS (and a part of one more).
template <typename T, int TPR, int FLAT>
__global__ __launch_bounds__(256) void k_token_grad(TokenRows a, LossTail f, const float* __restrict__ stats, const float* __restrict__ coef,
                                                    const int32_t* __restrict__ index, int64_t n_coef, float mult, const float* __restrict__ upstream, T* __restrict__ d, int64_t d_stride) {
  constexpr int RPB = 256 / TPR;
  const int r = threadIdx.x % TPR;
  const double k = (double)mult * a.inv_t * (upstream ? (double)*upstream : 1.0);
  const int blocks = gridDim.x - (f.loss != nullptr);
  if ((int)blockIdx.x == blocks) { preference_final(f); return; }
  constexpr int ROWS = TPR < 64 ? 64 / TPR : 1;
  constexpr int FLAT_V = (FLAT + 1) * Pack<T>::N;
  __shared__ __attribute__((aligned(16))) T stage[FLAT ? 4 * ROWS * FLAT_V : 1];
  T* const mine = stage + (FLAT ? (threadIdx.x >> 6) * ROWS * FLAT_V : 0);
  for (int64_t from = (int64_t)blockIdx.x * RPB; from < a.n; from += (int64_t)blocks * RPB) {
    // long rows from the last one back: a preference step has just read them, and the last ones may still be in the last-level
    // cache (a logits buffer that is used again and again: 6007 rows of 32003 bf16 266 us against 270, 3000 of 32000 fp32 231
    // against 234; several buffers in turn: no more than 1 % either way)
    const int64_t base = TPR == 256 ? a.n - 1 - from : from;
    const int64_t t = base + threadIdx.x / TPR;
    if (t < a.n) {
      const int id = a.tok.at(t);
      const int64_t ci = index ? (int64_t)index[t] : t;
      const float g = id < 0 || ci < 0 || ci >= n_coef ? 0.f : (float)((double)coef[ci] * k);
      const T* row = reinterpret_cast<const T*>(a.x) + t * a.stride;
      if constexpr (FLAT) row_gradient<T, TPR>(a, row, mine + (threadIdx.x & 63) / TPR * a.V, id, r, stats[2 * t], stats[2 * t + 1], g);
      else row_gradient<T, TPR>(a, row, d + t * d_stride, id, r, stats[2 * t], stats[2 * t + 1], g);
    }
    if constexpr (FLAT) {
      const int64_t t0 = base + (int64_t)(threadIdx.x >> 6) * ROWS;
      if (t0 < a.n) write_flat(mine, d + t0 * a.V, (int)(a.n - t0 < ROWS ? a.n - t0 : ROWS) * a.V);
    }
  }
}

// Rows in chunks of SEG_ROWS, one block a chunk: the sequence of each row (-1 for ignored rows and rows outside every
// sequence), the chunk's number of taking rows, and for every sequence that meets the chunk the sum and the number of its
// rows in it.  The sums are running ones in 64 bits that start anew with every sequence: differences of one running sum over
// the whole chunk would carry an infinity or NaN of one sequence into those behind it.  What sequence s has in chunk c goes to
// place c + s: both grow along the rows, so no two parts share a place.  A sequence of any length is then the sum of its
// parts, and no block waits for one long sequence.  Bound by its dependent loads: 4.6 us for 18944 rows, 5.8 for 593920.
#define SEG_ROWS 1024
// The number of seq_ptr[0 .. n) that are <= t, by a whole wave: 64 probes a step.  (In 32 bits: n <= 2^31, a probe lies
// below 2^31 + 2^25.  The compiler's scalar code for the 64-bit form selects by a stale condition bit.)
__device__ __forceinline__ uint32_t wave_count_upto(const int32_t* __restrict__ seq_ptr, uint32_t n, int32_t t) {
  uint32_t lo = 0, hi = n;     // the answer lies in [lo, hi], which shrinks to 1/64 a step whatever seq_ptr holds
  while (lo < hi) {
    const uint32_t step = (hi - lo + 63) >> 6, at = lo + ((threadIdx.x & 63) + 1) * step - 1;
    const uint64_t below = __ballot(at < hi && seq_ptr[at < hi ? at : lo] <= t);
    const uint32_t k = (uint32_t)__popcll(below), next = lo + (k + 1) * step - 1;
    lo += k * step;
    hi = next < hi ? next : hi;
    hi = hi < lo ? lo : hi;
  }
  return lo;
}
struct SegRows {
  TokenView tok; int64_t n;
  const int32_t* seq_ptr; int32_t S;
  const float* diff;          // [n]
  int32_t* seq_of;            // [n]
  double* part_sum;           // [chunks + S]
  int32_t* part_len;          // [chunks + S] or null
  int32_t* chunk_len;         // [chunks] or null
};
template <bool SUM> struct SegShared {
  double run[SUM ? SEG_ROWS : 1], wsum[4];    // a row's sequence up to it, within the chunk
  int cnt[SEG_ROWS + 1], wcnt[4], wmax[4], wkey[4], ends[2];
};
template <bool SUM> __device__ __forceinline__ void row_segments(const SegRows& g, int64_t c, SegShared<SUM>& sh) {
  const TokenView& tok = g.tok;
  const int64_t n = g.n;
  const int32_t* __restrict__ seq_ptr = g.seq_ptr;
  const int32_t S = g.S;
  int* const cnt = sh.cnt;
  int* const mark = cnt;   // (the counts replace the marks once every thread has read its own)
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t c0 = c * SEG_ROWS;
  const int rows = (int)(n - c0 < SEG_ROWS ? n - c0 : SEG_ROWS);
  bool on[4];
  float d[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {   // (loads of a place that exists, so that all of them are under way at once)
    const int i = tid * 4 + j;
    const int64_t at = c0 + (i < rows ? i : rows - 1);
    on[j] = (tok.at(at) >= 0) & (i < rows);
    d[j] = SUM ? g.diff[at] : 0.f;
  }
  // sequences of the chunk's first and last row (-1: before the first, S: behind the last)
  if (seq_ptr && wave < 2) {
    const int k = (int)wave_count_upto(seq_ptr, (uint32_t)S + 1u, (int32_t)(wave ? c0 + rows - 1 : c0)) - 1;
    if (lane == 0) sh.ends[wave] = k;
  }
  if (!seq_ptr && tid < 2) sh.ends[tid] = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) mark[tid * 4 + j] = -1;
  __syncthreads();
  const int s0 = sh.ends[0], s1 = sh.ends[1], sa = s0 < 0 ? 0 : s0;
  // a row's sequence is the last that starts at or before it: starts are marked, then a running maximum
  if (seq_ptr)
    for (int64_t s = (int64_t)sa + tid; s <= s1; s += 256) {
      const int64_t at = seq_ptr[s] - c0;
      if (at >= 0 && at < rows) atomicMax(&mark[at], (int)s);
    }
  __syncthreads();
  int m[4], top = s0;
#pragma unroll
  for (int j = 0; j < 4; ++j) { const int v = mark[tid * 4 + j]; top = v > top ? v : top; m[j] = top; }
  int run = top;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) { const int u = __shfl_up(run, o); if (lane >= o && u > run) run = u; }
  if (lane == 63) sh.wmax[wave] = run;
  int before = __shfl_up(run, 1);
  if (lane == 0) before = s0;
  __syncthreads();
  for (int w = 0; w < wave; ++w) before = sh.wmax[w] > before ? sh.wmax[w] : before;
  int k[4];
  double v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    m[j] = before > m[j] ? before : m[j];
    k[j] = on[j] && m[j] >= 0 && m[j] < S;
    v[j] = SUM && k[j] ? (double)d[j] : 0.0;
    const int i = tid * 4 + j;
    if (i < rows) g.seq_of[c0 + i] = k[j] ? m[j] : -1;
  }
  // running sums that start anew with a sequence: the sequences never fall along the rows, so two places are of one run
  // exactly if they are of one sequence
  if (SUM) {
#pragma unroll
    for (int j = 1; j < 4; ++j)
      if (m[j] == m[j - 1]) v[j] += v[j - 1];
  }
  int ci = (k[0] + k[1]) + (k[2] + k[3]);
  const int own_c = ci, key = m[3];
  double vi = v[3];
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int cu = __shfl_up(ci, o), ku = SUM ? __shfl_up(key, o) : 0;
    const double vu = SUM ? __shfl_up(vi, o) : 0.0;
    if (lane >= o) {
      ci += cu;
      if (SUM && ku == key) vi += vu;
    }
  }
  const int key_below = SUM ? __shfl_up(key, 1) : 0, first = SUM ? __shfl(m[0], 0) : 0;
  double add = SUM ? __shfl_up(vi, 1) : 0.0;    // what came before the lane's first row, in this wave
  if (lane == 0 || key_below != m[0]) add = 0.0;
  if (lane == 63) {
    sh.wcnt[wave] = ci;
    if (SUM) { sh.wsum[wave] = vi; sh.wkey[wave] = key; }
  }
  __syncthreads();
  int cb = ci - own_c;
  for (int w = 0; w < wave; ++w) {
    cb += sh.wcnt[w];
    if (SUM && m[0] == first && sh.wkey[w] == first) add += sh.wsum[w];
  }
  if (tid == 0) cnt[0] = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    cb += k[j];
    cnt[tid * 4 + j + 1] = cb;
    if (SUM) sh.run[tid * 4 + j] = m[j] == m[0] ? v[j] + add : v[j];
  }
  __syncthreads();
  if (tid == 0 && g.chunk_len) g.chunk_len[c] = cnt[rows];
  if (!g.part_len) return;
  for (int64_t s = (int64_t)sa + tid; s <= s1 && s < S; s += 256) {
    const int64_t t0 = seq_ptr ? seq_ptr[s] : 0, t1 = seq_ptr ? seq_ptr[s + 1] : n;
    const int a = t0 <= c0 ? 0 : t0 - c0 < rows ? (int)(t0 - c0) : rows;
    const int b = t1 <= c0 ? 0 : t1 - c0 < rows ? (int)(t1 - c0) : rows;
    if (b > a) {
      g.part_len[c + s] = cnt[b] - cnt[a];
      if (SUM) g.part_sum[c + s] = sh.run[b - 1];
    }
  }
}
template <bool SUM> __global__ __launch_bounds__(256) void k_row_segments(SegRows g) {
  __shared__ SegShared<SUM> sh;
  row_segments<SUM>(g, blockIdx.x, sh);
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
  for (int64_t s = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); s < S; s += (int64_t)gridDim.x * 4) {
    double sum;
    int len;
    join_parts<false>(seq_ptr, n, s, nullptr, part_len, sum, len);
    if ((threadIdx.x & 63) == 0) seq_len[s] = len;
  }
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
  float* loss;
  float* log_ratio; float* margin; float* slope;
  double* partial;          // [gridDim.x]
};
// The loss of pair pr from both sequences' sums and numbers of rows, and d loss / d logp of either sequence's rows.
__device__ __forceinline__ double pair_loss(const PrefIn& a, int64_t pr, double sum0, int len0, double sum1, int len1) {
  const double share0 = a.average && len0 > 0 ? 1.0 / (double)len0 : 1.0, share1 = a.average && len1 > 0 ? 1.0 / (double)len1 : 1.0;
  const double ratio0 = sum0 * share0, ratio1 = sum1 * share1, gap = ratio0 - ratio1;
  double loss, slope;
  if (a.kind == LIGDIFF_PREFERENCE_SIGMOID) {
    // -(1 - e) log sigmoid(z) - e log sigmoid(-z) = log(1 + exp(-|z|)) + (z < 0 ? -(1 - e) z : e z).  The margin may be infinite
    // (a chosen id without probability): then x = 0 and the other term is the loss, 0 for z = inf and e = 0, else inf.
    const double z = (double)a.beta * gap, e = (double)a.smooth, x = exp(-fabs(z));
    loss = log1p(x) + (z < 0.0 ? -(1.0 - e) * z : e != 0.0 ? e * z : 0.0);
    const double sig = z >= 0.0 ? 1.0 / (1.0 + x) : x / (1.0 + x);
    slope = (double)a.beta * (sig - 1.0 + e);
  } else {
    const double z = gap - 0.5 / (double)a.beta;
    loss = z * z;
    slope = 2.0 * z;
  }
  slope *= a.grad_scale / a.denom;
  a.log_ratio[pr] = (float)ratio0;
  a.log_ratio[pr + a.P] = (float)ratio1;
  a.margin[pr] = (float)gap;
  a.slope[pr] = (float)(slope * share0);
  a.slope[pr + a.P] = (float)(-slope * share1);
  return loss;
}
// Pairs: sequence p is preferred over sequence P + p.  A wave joins the parts of both (a margin is what two long sums leave:
// 64 bits).  5 us for 512 pairs.
__global__ __launch_bounds__(256) void k_preference(PrefIn a) {
  __shared__ double red[4];
  double total = 0.0;
  for (int64_t pr = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); pr < a.P; pr += (int64_t)gridDim.x * 4) {
    double s0, s1;
    int l0, l1;
    join_parts<true>(a.seq_ptr, a.n, pr, a.part_sum, a.part_len, s0, l0);
    join_parts<true>(a.seq_ptr, a.n, pr + a.P, a.part_sum, a.part_len, s1, l1);
    if ((threadIdx.x & 63) == 0) total += pair_loss(a, pr, s0, l0, s1, l1);
  }
  total = block_sum<256>(total, red);
  if (threadIdx.x == 0) a.partial[blockIdx.x] = total;
}
// A batch of one chunk, where every sequence is one part: rows -> sequences, pairs (a thread each) and the loss in one launch
// of one block.
__global__ __launch_bounds__(256) void k_preference_small(SegRows g, PrefIn a) {
  __shared__ SegShared<true> sh;
  __shared__ double red[4];
  row_segments<true>(g, 0, sh);
  __syncthreads();
  double total = 0.0;
  for (int64_t pr = threadIdx.x; pr < a.P; pr += 256) {
    double sum[2] = {0.0, 0.0};
    int len[2] = {0, 0};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t q = pr + (int64_t)h * a.P, t0 = a.seq_ptr[q] < 0 ? 0 : a.seq_ptr[q], t1 = a.seq_ptr[q + 1] > a.n ? a.n : a.seq_ptr[q + 1];
      if (t1 > t0) { sum[h] = g.part_sum[q]; len[h] = g.part_len[q]; }
    }
    total += pair_loss(a, pr, sum[0], len[0], sum[1], len[1]);
  }
  total = block_sum<256>(total, red);
  if (threadIdx.x == 0) *a.loss = (float)(total / a.denom);
}
__device__ __forceinline__ void preference_final(const LossTail& f) {
  __shared__ double red[4];
  double v = 0.0;
#pragma unroll 4
  for (int b = threadIdx.x; b < f.blocks; b += 256) v += f.partial[b];
  v = block_sum<256>(v, red);
  if (threadIdx.x == 0) *f.loss = (float)(v / f.denom);
}
__global__ __launch_bounds__(256) void k_preference_final(LossTail f) { preference_final(f); }

// An empty batch: no row kernel runs.
__global__ void k_empty_policy(float* result) { if (threadIdx.x < 4) result[threadIdx.x] = 0.f; }

// ------------------------------------------------------------------ host side
// A persistent grid: enough blocks to fill the chip several times over, few enough that the per-block sums of a loss are
// added up by one block.
static int row_grid(int64_t groups, int most) { return (int)(groups < most ? groups : most); }

#define TK_GRID_CAP 2048
// Rows next to each other that end inside cache lines.
static bool ragged_lines(int32_t V, int64_t d_stride, size_t size) { return d_stride == V && (V * size) % 128 != 0; }
template <typename T, int TPR, int NV, int MODE, bool STAGE = false>
static int launch_rows_as(const TokenRows& a, const PolicyIn& p, const RowOut& o, hipStream_t s) {
  constexpr int NT = TPR <= 64 ? 256 : TPR, RPB = NT / TPR;
  const int grid = row_grid((a.n + RPB - 1) / RPB, TK_GRID_CAP * 256 / NT);
  hipLaunchKernelGGL((k_token_rows<T, TPR, NV, MODE, STAGE>), dim3(grid), dim3(NT), 0, s, a, p, o);
  return grid;
}
// A batch of at most SMALL_ROWS short rows is one launch of one block: three launches take longer than its two rounds.
static bool rows_of_8_lanes(int dtype, int32_t V) { return V / (dtype == LIGDIFF_F32 ? 4 : 8) <= 64; }
// Few lanes with many packs each (up to 16: 64 registers) before more lanes: more lanes wait for each other more often, hold fewer
// rows under way, have lanes without a pack in their last round, and do the work per row (64-bit log, ratio, KL term) for
// fewer rows at a time.  Measured on 419 MB, lanes x packs, log-probabilities / policy loss with gradient, us.
//   fp32: 24 packs 8x4 77/186, 8x8 93/168; 48 packs 8x8 81/169, 8x16 72, 16x4 74/181; 96 packs 8x16 72/184, 16x8 80/167, 16x12 74/167;
//     192 packs 16x16 72/182, 16x12 74/169, 64x4 76/186; 1024 packs 64x16 76/171, 256x4 74/169; 2048 packs 256x12 76/168, 1024x4 91/171;
//     5000 packs 512x12 72/173, 1024x6 83/170, twice read 81/244; 8192 packs 1024x12 78/170, twice read 74/236
//   bf16: 24 packs 8x4 88/194, 8x8 99/196; 48 packs 8x8 86/174, 8x16 81/181; 96 packs 8x16 76/194, 16x8 85/173, 16x12 80/173, 64x4
//     137/265; 192 packs 16x16 75/191, 16x12 78/176, 64x4 90/187; 300 packs 64x12 91/178, 256x4 185/330; 1024 packs 64x16 82/178, 256x4
//     89/176; 2500 packs 256x16 85/183, 512x8 91/179, 1024x4 111/203; 4000 packs 256x16 79/180, 512x8 86/175, 1024x4 87/177;
//     5000 packs 512x12 81/176, 1024x6 99/188, twice read 88/277; 7500 packs 1024x12 96/186, twice read 83/265; 16384 packs 1024x16
//     95/215, twice read 84/260
// So beyond 6144 packs the log-probabilities stream the row (they need one read in either form), and the policy loss keeps it up
// to 16384 packs.  Returns the number of blocks.
template <typename T, int MODE>
static int launch_rows(const TokenRows& a, const PolicyIn& p, const RowOut& o, hipStream_t s) {
  const int packs = a.V / Pack<T>::N;
  if (MODE == TK_POLICY && a.n <= SMALL_ROWS && packs <= 64) {
    if (packs <= 16) hipLaunchKernelGGL((k_token_rows<T, 8, 2, TK_SMALL>), dim3(1), dim3(256), 0, s, a, p, o);
    else if (packs <= 32) hipLaunchKernelGGL((k_token_rows<T, 8, 4, TK_SMALL>), dim3(1), dim3(256), 0, s, a, p, o);
    else hipLaunchKernelGGL((k_token_rows<T, 8, 8, TK_SMALL>), dim3(1), dim3(256), 0, s, a, p, o);
    return 1;
  }
  if constexpr (MODE == TK_POLICY) {
    // (through LDS: 119 fp32 a row 69 us against 86 for 147 MB, 200 fp32 61 against 72, 500 bf16 70 against 76; but 30 fp32 57
    // against 52 and 90 bf16 78 against 74: rows of two lines at most are as well written directly)
    const bool few = packs <= (sizeof(T) == 4 ? 16 : 24);
    if (packs <= 64 && (size_t)a.V * sizeof(T) > 256 && o.d && ragged_lines(a.V, o.d_stride, sizeof(T))) {
      if (sizeof(T) == 2 && packs <= 32) return launch_rows_as<T, 8, 4, MODE, true>(a, p, o, s);
      return launch_rows_as<T, 8, 8, MODE, true>(a, p, o, s);
    }
    if (packs <= 16) return launch_rows_as<T, 8, 2, MODE>(a, p, o, s);
    if (few) return launch_rows_as<T, 8, 4, MODE>(a, p, o, s);
    if (packs <= 64) return launch_rows_as<T, 8, 8, MODE>(a, p, o, s);
    if (packs <= 192) return launch_rows_as<T, 16, 12, MODE>(a, p, o, s);
    if (packs <= 256) return launch_rows_as<T, 64, 4, MODE>(a, p, o, s);
  } else {
    if (packs <= 16) return launch_rows_as<T, 8, 2, MODE>(a, p, o, s);
    if (packs <= 32) return launch_rows_as<T, 8, 4, MODE>(a, p, o, s);
    if (packs <= 128) return launch_rows_as<T, 8, 16, MODE>(a, p, o, s);
    if (packs <= 256) return launch_rows_as<T, 16, 16, MODE>(a, p, o, s);
  }
  if (packs <= 768) return launch_rows_as<T, 64, 12, MODE>(a, p, o, s);
  if (packs <= 1024) return launch_rows_as<T, 64, 16, MODE>(a, p, o, s);
  if (packs <= 2048) return launch_rows_as<T, 256, 12, MODE>(a, p, o, s);
  if constexpr (MODE == TK_POLICY) {
    if (packs <= 4096) return launch_rows_as<T, 512, 8, MODE>(a, p, o, s);
  } else {
    if (packs <= 4096) return launch_rows_as<T, 256, 16, MODE>(a, p, o, s);
  }
  if (packs <= 6144) return launch_rows_as<T, 512, 12, MODE>(a, p, o, s);
  if constexpr (MODE == TK_POLICY) {
    if (packs <= 12288) return launch_rows_as<T, 1024, 12, MODE>(a, p, o, s);
    if (packs <= 16384) return launch_rows_as<T, 1024, 16, MODE>(a, p, o, s);
  }
  const int grid = row_grid(a.n, TK_GRID_CAP);
  hipLaunchKernelGGL((k_token_rows_long<T, MODE>), dim3(grid), dim3(1024), 0, s, a, p, o);
  return grid;
}
template <int MODE> static int launch_rows_dtype(int dtype, const TokenRows& a, const PolicyIn& p, const RowOut& o, hipStream_t s) {
  if (a.n == 0) return 0;
  if (dtype == LIGDIFF_F32) return launch_rows<float, MODE>(a, p, o, s);
  if (dtype == LIGDIFF_BF16) return launch_rows<bf16_t, MODE>(a, p, o, s);
  return launch_rows<f16_t, MODE>(a, p, o, s);
}
struct GradIn { const float* stats; const float* coef; const int32_t* index; int64_t n_coef; float mult; const float* up; void* d; int64_t d_stride; };
template <typename T, int TPR, int FLAT> static void launch_grad_as(const TokenRows& a, const GradIn& g, const LossTail& f, hipStream_t s) {
  constexpr int RPB = 256 / TPR;
  const int grid = row_grid((a.n + RPB - 1) / RPB, 8192) + (f.loss != nullptr);
  hipLaunchKernelGGL((k_token_grad<T, TPR, FLAT>), dim3(grid), dim3(256), 0, s, a, f, g.stats, g.coef, g.index, g.n_coef, g.mult, g.up, (T*)g.d, g.d_stride);
}
template <typename T> static void launch_grad(const TokenRows& a, const GradIn& g, const LossTail& f, hipStream_t s) {
  const int packs = a.V / Pack<T>::N;
  // Rows that fill cache lines: 8 lanes a row (512 bytes 50 us against 61 with 16 lanes, 147 MB), 16 from 32 packs on (1024 bytes
  // 52 against 50).  Ragged rows: 8 lanes up to 192 bytes (45 fp32 39 us, 42 through LDS, 50 with 16 lanes), longer ones
  // through LDS (119 fp32 72 us, 97 with 8 and 76 with 16 lanes; 250 fp32 70, 96, 79; 119 bf16 72, 81, 86).
  const bool ragged = ragged_lines(a.V, g.d_stride, sizeof(T)), flat = ragged && (size_t)a.V * sizeof(T) > 192;
  if (flat && packs <= 32) launch_grad_as<T, 8, 32>(a, g, f, s);
  else if (flat && packs <= 64) launch_grad_as<T, 8, 64>(a, g, f, s);
  else if (packs <= 32) launch_grad_as<T, 8, 0>(a, g, f, s);
  else if (packs <= 64) launch_grad_as<T, 16, 0>(a, g, f, s);
  else if (packs <= 512) launch_grad_as<T, 64, 0>(a, g, f, s);
  else launch_grad_as<T, 256, 0>(a, g, f, s);
}
// (the caller has seen to it that there are rows)
static void launch_grad_dtype(int dtype, const TokenRows& a, const GradIn& g, const LossTail& f, hipStream_t s) {
  if (dtype == LIGDIFF_F32) launch_grad<float>(a, g, f, s);
  else if (dtype == LIGDIFF_BF16) launch_grad<bf16_t>(a, g, f, s);
  else launch_grad<f16_t>(a, g, f, s);
}

static int fill_rows(TokenRows* r, const ligdiff_token_args* a) {
  if (!a || a->n_tokens < 0 || a->n_tokens > 0x7fffffffLL || a->vocab < 1 || a->row_stride < a->vocab ||
      a->dtype < LIGDIFF_F32 || a->dtype > LIGDIFF_F16 || (a->token_bytes != 4 && a->token_bytes != 8) ||
      !(a->temperature >= 1e-20f) || !(a->temperature <= 1e20f))
    return LIGDIFF_ERR_ARG;
  if (a->n_tokens > 0 && (!a->logits || !a->tokens)) return LIGDIFF_ERR_ARG;
  r->x = a->logits; r->stride = a->row_stride; r->n = a->n_tokens; r->V = a->vocab;
  r->tok = TokenView{a->tokens, a->token_bytes, a->vocab};
  const double c = TK_LOG2E / (double)a->temperature;
  r->c = (float)c;
  if ((double)r->c >= c) r->c = nextafterf(r->c, 0.f);
  r->c_lo = (float)(c - (double)r->c);
  r->inv_t = 1.0 / (double)a->temperature;
  return LIGDIFF_OK;
}

extern "C" int ligdiff_token_logprob(const ligdiff_token_args* args, float* logp, float* stats, void* stream) {
  TokenRows a;
  const int rc = fill_rows(&a, args);
  if (rc) return rc;
  if (a.n > 0 && !logp) return LIGDIFF_ERR_ARG;
  launch_rows_dtype<TK_LOGP>(args->dtype, a, PolicyIn{}, RowOut{logp, nullptr, stats, nullptr, nullptr, 0}, (hipStream_t)stream);
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
  if (a.n > 0)
    launch_grad_dtype(args->dtype, a, GradIn{stats, coef, coef_index, n_coef, mult, upstream, d_logits, d_stride}, LossTail{},
                      (hipStream_t)stream);
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
struct PrefWs { double* partial; float* diff; double* part_sum; int32_t* part_len; size_t bytes; };
static PrefWs pref_ws(void* base, int64_t n, int32_t P) {
  Pieces w{(char*)base};
  const size_t parts = (size_t)(seg_chunks(n) + 2 * (int64_t)P);
  PrefWs r;
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
  PrefIn p;
  p.n = a.n; p.seq_ptr = q->seq_ptr; p.P = q->n_pairs; p.part_sum = w.part_sum; p.part_len = w.part_len;
  p.beta = q->beta; p.smooth = q->label_smoothing; p.kind = q->kind; p.average = q->average != 0;
  p.denom = q->denominator > 0.f ? (double)q->denominator : (double)q->n_pairs;
  p.grad_scale = (double)q->grad_scale;
  p.loss = q->loss; p.log_ratio = q->log_ratio; p.margin = q->margin; p.slope = q->slope;
  p.partial = w.partial;
  LossTail f{};
  const SegRows g{a.tok, a.n, q->seq_ptr, 2 * q->n_pairs, w.diff, q->row_seq, w.part_sum, w.part_len, nullptr};
  if (a.n > 0) launch_rows_dtype<TK_LOGP>(args->dtype, a, PolicyIn{}, RowOut{w.diff, q->ref_logp, q->stats, nullptr, nullptr, 0}, s);
  // one block while it has a chunk at most and the pairs do not keep it longer than two launches would take
  if (a.n > 0 && a.n <= SEG_ROWS && q->n_pairs <= 1024) {
    hipLaunchKernelGGL(k_preference_small, dim3(1), dim3(256), 0, s, g, p);
  } else {
    if (a.n > 0) hipLaunchKernelGGL((k_row_segments<true>), dim3((unsigned)seg_chunks(a.n)), dim3(256), 0, s, g);
    const int blocks = row_grid(((int64_t)q->n_pairs + 3) / 4, PREF_BLOCKS);
    hipLaunchKernelGGL(k_preference, dim3(blocks), dim3(256), 0, s, p);
    f = LossTail{w.partial, blocks, p.denom, q->loss};
  }
  if (a.n > 0 && q->d_logits)
    launch_grad_dtype(args->dtype, a, GradIn{q->stats, q->slope, q->row_seq, 2 * (int64_t)q->n_pairs, 1.0f, nullptr, q->d_logits, q->d_stride}, f, s);
  else if (f.loss) hipLaunchKernelGGL(k_preference_final, dim3(1), dim3(256), 0, s, f);
  LD_CHECK_LAUNCH();
  return LIGDIFF_OK;
}

struct PolicyWs { double* partial; int32_t* chunk_len; int32_t* seq_of; int32_t* part_len; int32_t* seq_len; size_t bytes; };
static PolicyWs policy_ws(void* base, int64_t n, int32_t S, bool per_seq) {
  Pieces w{(char*)base};
  PolicyWs r;
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
  const bool small = a.n <= SMALL_ROWS && rows_of_8_lanes(args->dtype, a.V);
  if (!small)
    hipLaunchKernelGGL((k_row_segments<false>), dim3(chunks), dim3(256), 0, s,
                       SegRows{a.tok, a.n, q->seq_ptr, q->n_seq, nullptr, w.seq_of, nullptr, per_seq ? w.part_len : nullptr, w.chunk_len});
  // (in a batch of one chunk a sequence is its one part)
  if (per_seq && !small && chunks > 1)
    hipLaunchKernelGGL(k_sequence_lengths, dim3(row_grid(((int64_t)q->n_seq + 3) / 4, 1 << 20)), dim3(256), 0, s, q->seq_ptr, a.n, q->n_seq, w.part_len, w.seq_len);
  PolicyIn p;
  p.seq_of = w.seq_of; p.seq_len = chunks > 1 ? w.seq_len : w.part_len; p.chunk_len = w.chunk_len; p.n_chunks = chunks;
  p.denom = (double)q->denominator; p.n_seq = q->n_seq; p.per_seq_mean = per_seq;
  p.adv = q->advantage; p.adv_per_token = q->advantage_per_token != 0;
  p.old_logp = q->old_logp; p.ref_logp = q->ref_logp;
  p.clip_lo = q->clip_low; p.clip_hi = q->clip_high; p.kl_coef = q->kl_coef; p.grad_scale = q->grad_scale;
  p.partial = w.partial; p.result = q->result; p.seq_ptr = q->seq_ptr;
  const int blocks = launch_rows_dtype<TK_POLICY>(args->dtype, a, p, RowOut{q->logp, nullptr, q->stats, q->coef, q->d_logits, q->d_stride}, s);
  if (!small) hipLaunchKernelGGL(k_policy_final, dim3(1), dim3(256), 0, s, w.partial, blocks, (double)q->kl_coef, q->result);
  LD_CHECK_LAUNCH();
  return LIGDIFF_OK;
}
