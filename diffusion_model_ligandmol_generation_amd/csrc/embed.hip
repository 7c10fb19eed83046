// Embedding lookup with scaling, and its gradient by sorted tokens.
//   out[i, :] = scale W[tok_i, :]                       d_W[v, :] = scale sum_{i: tok_i = v} d_out[i, :]
// Both are bound by HBM, small calls by their launches.  The gradient reads every row of d_out once and adds in 32 bits and in a
// fixed order, no float atomics, so the result does not change from run to run.  The tokens of a batch are very uneven (half
// of a ligand's atoms are carbon), so the work is cut into equal numbers of rows whatever their tokens are.  Tables of up to
// 128 rows are added up in LDS (two launches).  For larger ones the token positions are sorted (a stable radix sort of 8-byte
// records, small against the rows) and cut into chunks; a token whose positions lie in several chunks leaves one partial row
// in each, and a last launch joins them.
#include "embed.h"
#include <algorithm>

// ------------------------------------------------------------------ lookup
// TPR lanes a row, four rows in flight per group: the token, then the row, then the store are dependent accesses.  29696 rows of
// 256 fp32 8.5 us, 65536 rows of 1024 bf16 of a table of 32000 33-44 us (the table in the last-level cache or not).
template <typename T, int TPR>
__global__ __launch_bounds__(256) void k_embed(const T* __restrict__ table, int64_t row_stride, TokenView tok, int64_t n, int32_t D,
                                               float scale, T* __restrict__ out, int64_t out_stride) {
  constexpr int N = Pack<T>::N, RPB = 256 / TPR, RU = 4;
  const int r = threadIdx.x % TPR, nb = D / N, tail = D - nb * N;
  for (int64_t t0 = ((int64_t)blockIdx.x * RPB + threadIdx.x / TPR) * RU; t0 < n; t0 += (int64_t)gridDim.x * RPB * RU) {
    int id[RU];
#pragma unroll
    for (int u = 0; u < RU; ++u) id[u] = t0 + u < n ? tok.at(t0 + u) : -1;
    for (int i = r; i < nb; i += TPR) {
      u32x4 v[RU];
#pragma unroll
      for (int u = 0; u < RU; ++u) {
        v[u] = u32x4{0, 0, 0, 0};
        if (id[u] >= 0) v[u] = load_raw(table + id[u] * row_stride + (int64_t)i * N);
      }
#pragma unroll
      for (int u = 0; u < RU; ++u)
        if (t0 + u < n) {
          float f[N];
#pragma unroll
          for (int j = 0; j < N; ++j) f[j] = raw_get<T>(v[u], j) * scale;
          store_pack(out + (t0 + u) * out_stride + (int64_t)i * N, f);
        }
    }
    if (r < tail)
#pragma unroll
      for (int u = 0; u < RU; ++u)
        if (t0 + u < n)
          out[(t0 + u) * out_stride + nb * N + r] = id[u] >= 0 ? (T)((float)table[id[u] * row_stride + nb * N + r] * scale) : (T)0.f;
  }
}

template <typename T>
static void launch_embed(const void* table, int64_t row_stride, TokenView tok, int64_t n, int32_t D, float scale, void* out,
                         int64_t out_stride, hipStream_t s) {
  const int packs = D / Pack<T>::N;
#define LAUNCH_EMBED(TPR)                                                                                                 \
  do {                                                                                                                    \
    const int64_t blocks = (n + 4 * (256 / TPR) - 1) / (4 * (256 / TPR));                                                 \
    hipLaunchKernelGGL((k_embed<T, TPR>), dim3((unsigned)(blocks < 16384 ? blocks : 16384)), dim3(256), 0, s, (const T*)table, \
                       row_stride, tok, n, D, scale, (T*)out, out_stride);                                                \
  } while (0)
  if (packs <= 8) LAUNCH_EMBED(8);
  else if (packs <= 16) LAUNCH_EMBED(16);
  else if (packs <= 32) LAUNCH_EMBED(32);
  else LAUNCH_EMBED(64);
}

static bool bad_embed(int dtype, int64_t n_rows, int32_t width, int token_bytes, int64_t n) {
  return dtype < LIGDIFF_F32 || dtype > LIGDIFF_F16 || n_rows < 1 || n_rows > 0x7ffffffeLL || width < 1 ||
         (token_bytes != 4 && token_bytes != 8) || n < 0 || n > 0x7fffffffLL;
}

extern "C" int ligdiff_embed(const void* table, int32_t dtype, int64_t n_rows, int32_t width, int64_t row_stride,
                             const void* tokens, int32_t token_bytes, int64_t n_tokens, float scale, void* out,
                             int64_t out_stride, void* stream) {
  if (bad_embed(dtype, n_rows, width, token_bytes, n_tokens) || row_stride < width || out_stride < width || !table)
    return LIGDIFF_ERR_ARG;
  if (n_tokens == 0) return LIGDIFF_OK;
  if (!tokens || !out) return LIGDIFF_ERR_ARG;
  const TokenView tok{tokens, token_bytes, (int32_t)n_rows};
  hipStream_t s = (hipStream_t)stream;
  if (dtype == LIGDIFF_F32) launch_embed<float>(table, row_stride, tok, n_tokens, width, scale, out, out_stride, s);
  else if (dtype == LIGDIFF_BF16) launch_embed<bf16_t>(table, row_stride, tok, n_tokens, width, scale, out, out_stride, s);
  else launch_embed<f16_t>(table, row_stride, tok, n_tokens, width, scale, out, out_stride, s);
  LD_CHECK_LAUNCH();
  return LIGDIFF_OK;
}

// ------------------------------------------------------------------ stable radix sort of the positions by token
// Bound by latency: 65536 positions take 22 us in two passes of two launches, 4096 or fewer about 7 us in one launch.
#define SORT_NT 512
#define SORT_WAVES (SORT_NT / 64)
struct SortPass {
  TokenView tok;                       // first pass: the key of position i is its token, tok.n_rows for tokens outside
  const uint32_t* key_in; const int32_t* pos_in;   // later passes
  uint32_t* key_out; int32_t* pos_out;
  int64_t n;
  int32_t shift, per_block;            // per_block: a multiple of SORT_NT
  int32_t* hist;                       // [blocks][bins]
  int32_t* row_ptr; int32_t rows;      // one-pass sorts: block 0 writes the first position of every token, [rows + 1]
  int32_t blocks;                      // that sort; those behind them clear a part of the table
  u32x4* clear; int64_t n_clear;
};
// A sort keeps few compute units busy and waits for memory most of the time: the others write zeros to the table meanwhile.
__device__ __forceinline__ void clear_part(const SortPass& a) {
  const int64_t step = (int64_t)(gridDim.x - a.blocks) * blockDim.x;
  for (int64_t i = (int64_t)(blockIdx.x - a.blocks) * blockDim.x + threadIdx.x; i < a.n_clear; i += step) a.clear[i] = u32x4{0, 0, 0, 0};
}
template <bool FIRST> __device__ __forceinline__ uint32_t sort_key(const SortPass& a, int64_t i) {
  if (!FIRST) return a.key_in[i];
  const int id = a.tok.at(i);
  return id < 0 ? (uint32_t)a.tok.n_rows : (uint32_t)id;
}
template <int BITS, bool FIRST, bool CLEAR>
__global__ __launch_bounds__(SORT_NT) void k_sort_count(SortPass a) {
  constexpr int NB = 1 << BITS;
  __shared__ int cnt[NB];
  if (CLEAR && (int)blockIdx.x >= a.blocks) return clear_part(a);
  for (int d = threadIdx.x; d < NB; d += SORT_NT) cnt[d] = 0;
  __syncthreads();
  const int64_t b0 = (int64_t)blockIdx.x * a.per_block;
  for (int k = threadIdx.x; k < a.per_block; k += SORT_NT)
    if (b0 + k < a.n) atomicAdd(&cnt[(sort_key<FIRST>(a, b0 + k) >> a.shift) & (NB - 1)], 1);
  __syncthreads();
  for (int d = threadIdx.x; d < NB; d += SORT_NT) a.hist[(int64_t)blockIdx.x * NB + d] = cnt[d];
}
// Each block finds its own offsets from the count table (no scan launch): total and preceding blocks' counts of every digit,
// a prefix sum over the digits, then one over its waves; a wave ranks 64 positions at a time by the lanes that hold the
// same digit, so positions of equal digits keep their order.
template <int BITS, bool FIRST, bool CLEAR>
__global__ __launch_bounds__(SORT_NT) void k_sort_scatter(SortPass a) {
  constexpr int NB = 1 << BITS, K = NB > SORT_NT ? NB / SORT_NT : 1, LIVE = NB / K;
  __shared__ int cnt[SORT_WAVES][NB];
  __shared__ int wtot[SORT_WAVES];
  if (CLEAR && (int)blockIdx.x >= a.blocks) return clear_part(a);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // this wave's first keys are on their way while the count table is read
  constexpr int PRE = 2;
  const int64_t w0 = (int64_t)blockIdx.x * a.per_block + (int64_t)wave * (a.per_block / SORT_WAVES);
  uint32_t pre_key[PRE];
  int32_t pre_pos[PRE];
#pragma unroll
  for (int k = 0; k < PRE; ++k) {
    const int64_t i = w0 + k * 64 + lane;   // (a wave's part is at least PRE * 64 positions)
    pre_key[k] = 0; pre_pos[k] = 0;
    if (i < a.n) { pre_key[k] = sort_key<FIRST>(a, i); pre_pos[k] = FIRST ? (int32_t)i : a.pos_in[i]; }
  }
  for (int i = tid; i < SORT_WAVES * NB; i += SORT_NT) (&cnt[0][0])[i] = 0;
  int total[K] = {}, before[K] = {};
  if (tid < LIVE) {
#pragma unroll 8
    for (int b = 0; b < (CLEAR ? a.blocks : (int)gridDim.x); ++b)
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int h = a.hist[(int64_t)b * NB + tid * K + k];
        total[k] += h;
        before[k] += b < (int)blockIdx.x ? h : 0;
      }
  }
  int own = 0;
#pragma unroll
  for (int k = 0; k < K; ++k) own += total[k];
  int scan = own;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(scan, o);
    if (lane >= o) scan += u;
  }
  if (lane == 63) wtot[wave] = scan;
  __syncthreads();
  int excl = scan - own;
  for (int w = 0; w < wave; ++w) excl += wtot[w];
  // counts of this block's waves
#pragma unroll
  for (int k = 0; k < PRE; ++k)
    if (w0 + k * 64 + lane < a.n) atomicAdd(&cnt[wave][(pre_key[k] >> a.shift) & (NB - 1)], 1);
  for (int k = PRE * 64 + lane; k < a.per_block / SORT_WAVES; k += 64)
    if (w0 + k < a.n) atomicAdd(&cnt[wave][(sort_key<FIRST>(a, w0 + k) >> a.shift) & (NB - 1)], 1);
  __syncthreads();
  if (tid < LIVE) {
    int start = excl;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int d = tid * K + k;
      if (a.row_ptr && blockIdx.x == 0 && d <= a.rows) a.row_ptr[d] = start;
      int run = start + before[k];
      for (int w = 0; w < SORT_WAVES; ++w) {
        const int c = cnt[w][d];
        cnt[w][d] = run;
        run += c;
      }
      start += total[k];
    }
  }
  __syncthreads();
  const auto place = [&](bool on, uint32_t key, int32_t pos) {
    const int d = (int)(key >> a.shift) & (NB - 1);
    uint64_t same = __ballot(on);
#pragma unroll
    for (int b = 0; b < BITS; ++b) {
      const uint64_t set = __ballot((d >> b) & 1);
      same &= (d >> b) & 1 ? set : ~set;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1));
    int at = 0;
    if (on) at = cnt[wave][d];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (on && rank == 0) cnt[wave][d] = at + __popcll(same);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (on) {
      a.key_out[at + rank] = key;
      a.pos_out[at + rank] = pos;
    }
  };
#pragma unroll
  for (int k = 0; k < PRE; ++k) place(w0 + k * 64 + lane < a.n, pre_key[k], pre_pos[k]);
  for (int k = PRE * 64; k < a.per_block / SORT_WAVES && w0 + k < a.n; k += 64) {
    const int64_t i = w0 + k + lane;
    const bool on = i < a.n;
    uint32_t key = 0;
    int32_t pos = 0;
    if (on) { key = sort_key<FIRST>(a, i); pos = FIRST ? (int32_t)i : a.pos_in[i]; }
    place(on, key, pos);
  }
}

// Up to SORT_SMALL positions: all passes of 8 bits by one block in LDS, one launch instead of two a pass.
#define SORT_SMALL 4096
#define SORT_SMALL_NT 1024
template <int PASSES>
__global__ __launch_bounds__(SORT_SMALL_NT) void k_sort_small(SortPass a) {
  constexpr int WAVES = SORT_SMALL_NT / 64, EACH = SORT_SMALL / SORT_SMALL_NT;   // positions of a lane: 64 apart in its wave's part
  __shared__ uint32_t key[SORT_SMALL];
  __shared__ uint16_t pos[SORT_SMALL];
  __shared__ int cnt[WAVES][256];
  __shared__ int wtot[4];
  if (blockIdx.x > 0) return clear_part(a);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = (int)a.n, w0 = wave * 64 * EACH;
  uint32_t k[EACH];
  uint16_t p[EACH];
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int i = w0 + e * 64 + lane;
    k[e] = i < n ? sort_key<true>(a, i) : 0;
    p[e] = (uint16_t)i;
  }
#pragma unroll
  for (int pass = 0; pass < PASSES; ++pass) {
    for (int i = tid; i < WAVES * 256; i += SORT_SMALL_NT) (&cnt[0][0])[i] = 0;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < EACH; ++e)
      if (w0 + e * 64 + lane < n) atomicAdd(&cnt[wave][(k[e] >> (8 * pass)) & 255], 1);
    __syncthreads();
    int total = 0, scan = 0;
    if (tid < 256) {
      for (int w = 0; w < WAVES; ++w) total += cnt[w][tid];
      scan = total;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) { const int u = __shfl_up(scan, o); if (lane >= o) scan += u; }
      if (lane == 63) wtot[wave] = scan;
    }
    __syncthreads();
    if (tid < 256) {
      int run = scan - total;
      for (int w = 0; w < wave; ++w) run += wtot[w];
      if (PASSES == 1 && a.row_ptr && tid <= a.rows) a.row_ptr[tid] = run;
      for (int w = 0; w < WAVES; ++w) { const int c = cnt[w][tid]; cnt[w][tid] = run; run += c; }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const bool on = w0 + e * 64 + lane < n;
      const int d = (int)(k[e] >> (8 * pass)) & 255;
      uint64_t same = __ballot(on);
#pragma unroll
      for (int b = 0; b < 8; ++b) {
        const uint64_t set = __ballot((d >> b) & 1);
        same &= (d >> b) & 1 ? set : ~set;
      }
      const int rank = __popcll(same & ((1ull << lane) - 1));
      int at = 0;
      if (on) at = cnt[wave][d];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if (on && rank == 0) cnt[wave][d] = at + __popcll(same);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if (on) {
        if (pass == PASSES - 1) { a.key_out[at + rank] = k[e]; a.pos_out[at + rank] = p[e]; }
        else { key[at + rank] = k[e]; pos[at + rank] = p[e]; }
      }
    }
    if (pass < PASSES - 1) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        const int i = w0 + e * 64 + lane;
        if (i < n) { k[e] = key[i]; p[e] = pos[i]; }
      }
      __syncthreads();
    }
  }
}

// ------------------------------------------------------------------ sums of rows of equal tokens
struct SegIn {
  const void* d_out; int64_t d_stride;
  const uint32_t* key; const int32_t* pos;   // sorted
  int64_t n;
  int32_t* row_ptr; bool have_ptr;
  int32_t rows, D, R, n_chunks, n_tiles;
  float scale;
  float* part;                               // [n_chunks][2][D], a chunk here SUM_WAVES * R positions
  void* d_table; int64_t t_stride;
  bool accumulate, cleared;                  // cleared: the sort wrote zeros to the table
  int32_t zero_blocks;
};
#define SUM_WAVES 8
#define ZERO_ROWS 64   // rows of the table a block of the first part looks after

template <typename TO> __device__ __forceinline__ void put(TO* p, float v, bool add) { *p = (TO)(add ? (float)*p + v : v); }
// the first `live` of N columns
template <typename TO, int N> __device__ __forceinline__ void put_columns(TO* p, const float (&v)[N], float scale, int live, bool add) {
  if (live == N && !add) {
    typedef TO Raw __attribute__((ext_vector_type(N), aligned(sizeof(TO))));
    Raw r;
#pragma unroll
    for (int j = 0; j < N; ++j) r[j] = (TO)(v[j] * scale);
    *reinterpret_cast<Raw*>(p) = r;
    return;
  }
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (j < live) put(p + j, v[j] * scale, add);
}

// Blocks [0, zero_blocks): find where each token's positions start (bisection, unless the sort wrote it) and write the rows
// of tokens that do not occur.  The other blocks: SUM_WAVES chunks of R sorted positions and 64 packs of columns, a wave a chunk.  A wave
// writes the tokens that lie inside its chunk; the first and the last, which may go on in the neighbours', meet in LDS, and
// only what goes on beyond the block's chunks leaves it as a partial row: slot 0 the block's first token, slot 1 its last.
// 65536 rows of 1024 bf16 in random order, table of 32000: 49 us, 4.1 TB/s.
template <typename T, typename TO>
__global__ __launch_bounds__(SUM_WAVES * 64) void k_segment_sums(SegIn a) {
  constexpr int N = Pack<T>::N, U = 8, NT = SUM_WAVES * 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if ((int)blockIdx.x < a.zero_blocks) {
    __shared__ int ptr[ZERO_ROWS + 1];
    const int v0 = blockIdx.x * ZERO_ROWS;
    for (int k = threadIdx.x; k <= ZERO_ROWS; k += NT) {
      const int64_t v = (int64_t)v0 + k;
      if (v > a.rows) continue;
      int p;
      if (a.have_ptr) p = a.row_ptr[v];
      else {
        int64_t lo = 0, hi = a.n;   // the number of keys below v
        while (lo < hi) {
          const int64_t mid = (lo + hi) >> 1;
          if ((int64_t)a.key[mid] < v) lo = mid + 1; else hi = mid;
        }
        p = (int)lo;
        if (k < ZERO_ROWS || v == a.rows) a.row_ptr[v] = p;
      }
      ptr[k] = p;
    }
    __syncthreads();
    if (a.accumulate || a.cleared) return;
    for (int k = wave; k < ZERO_ROWS && v0 + k < a.rows; k += SUM_WAVES) {
      if (ptr[k + 1] != ptr[k]) continue;
      TO* row = reinterpret_cast<TO*>(a.d_table) + (int64_t)(v0 + k) * a.t_stride;
      constexpr int M = Pack<TO>::N;
      const float z[M] = {};
      const int nb = a.D / M;
      for (int i = lane; i < nb; i += 64) store_pack(row + (int64_t)i * M, z);
      if (lane < a.D - nb * M) row[nb * M + lane] = (TO)0.f;
    }
    return;
  }
  const int chunk = (int)((blockIdx.x - a.zero_blocks) / a.n_tiles), tile = (int)((blockIdx.x - a.zero_blocks) % a.n_tiles);
  __shared__ float sum[SUM_WAVES][2][64 * N];
  __shared__ uint32_t key0[SUM_WAVES], key1[SUM_WAVES];   // a wave's first and last token
  const int64_t b0 = (int64_t)chunk * a.R * SUM_WAVES, c0 = b0 + (int64_t)wave * a.R;
  const int64_t left_of = a.n - c0;
  const int rows = left_of <= 0 ? 0 : (int)(left_of < a.R ? left_of : a.R);
  const int col = tile * 64 * N + lane * N;
  const int live = a.D - col < 0 ? 0 : a.D - col < N ? a.D - col : N;   // columns of this lane
  const uint32_t limit = (uint32_t)a.rows, none = 0xffffffffu;
  float acc[N] = {};
  uint32_t cur = none, head = none;
  const T* base = reinterpret_cast<const T*>(a.d_out) + col;
  const auto flush = [&]() {   // token `cur` ends inside the chunk
    if (cur == head) {
#pragma unroll
      for (int j = 0; j < N; ++j) sum[wave][0][lane * N + j] = acc[j];
    } else {
      put_columns<TO, N>(reinterpret_cast<TO*>(a.d_table) + (int64_t)cur * a.t_stride + col, acc, a.scale, live, a.accumulate);
    }
  };
  bool done = false;
  for (int b = 0; b < rows && !done; b += 64) {
    const int left = rows - b < 64 ? rows - b : 64;
    uint32_t kv = none;
    int32_t pv = 0;
    if (lane < left) { kv = a.key[c0 + b + lane]; pv = a.pos[c0 + b + lane]; }
    if (b == 0) {
      cur = head = (uint32_t)__builtin_amdgcn_readfirstlane((int)kv);
      if (cur >= limit) { cur = head = none; break; }
    }
    for (int g = 0; g < left && !done; g += U) {
      u32x4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (g + u >= left) continue;
        const int64_t p = __builtin_amdgcn_readlane(pv, g + u);
        if (live == N) v[u] = load_raw(base + p * a.d_stride);
        else v[u] = load_raw_part(base + p * a.d_stride, live);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (g + u >= left || done) continue;
        const uint32_t key = (uint32_t)__builtin_amdgcn_readlane((int)kv, g + u);
        if (key >= limit) { done = true; continue; }   // tokens without a row are sorted last
        if (key != cur) {
          flush();
          cur = key;
#pragma unroll
          for (int j = 0; j < N; ++j) acc[j] = 0.f;
        }
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] += raw_get<T>(v[u], j);
      }
    }
  }
  // the last token: slot 1, or slot 0 when the chunk holds one token only
#pragma unroll
  for (int j = 0; j < N; ++j) sum[wave][cur == head ? 0 : 1][lane * N + j] = acc[j];
  if (lane == 0) { key0[wave] = head; key1[wave] = cur; }
  __syncthreads();
  // join: a thread a column, the chunks in order
  const int64_t b1 = a.n < b0 + (int64_t)a.R * SUM_WAVES ? a.n : b0 + (int64_t)a.R * SUM_WAVES;
  const uint32_t in = b0 > 0 ? a.key[b0 - 1] : none, out = b1 < a.n ? a.key[b1] : none;   // the neighbours' tokens
  float* part = a.part + (int64_t)chunk * 2 * a.D;
  for (int k = threadIdx.x; k < 64 * N; k += NT) {
    const int c = tile * 64 * N + k;
    if (c >= a.D) continue;
    uint32_t open = none;   // the token that is being added up
    float v = 0.f;
    const auto close = [&](bool goes_on) {
      if (open == none) return;
      const bool first = open == key0[0];
      if ((first && open == in) || goes_on) part[(first ? 0 : 1) * a.D + c] = v;
      else put(reinterpret_cast<TO*>(a.d_table) + (int64_t)open * a.t_stride + c, v * a.scale, a.accumulate);
    };
#pragma unroll
    for (int w = 0; w < SUM_WAVES; ++w) {
      if (key0[w] == none) continue;
      if (key0[w] == open) v += sum[w][0][k];
      else { close(false); open = key0[w]; v = sum[w][0][k]; }
      if (key1[w] != key0[w]) { close(false); open = key1[w]; v = sum[w][1][k]; }
    }
    close(open != none && open == out);
  }
}

#define JOIN_WAVES 8
// One block for each block of the sums; it joins the partial rows of the token that starts there and goes on in the next.
template <typename TO>
__global__ __launch_bounds__(JOIN_WAVES * 64) void k_segment_join(SegIn a) {
  const int chunk = blockIdx.x / a.n_tiles, tile = blockIdx.x % a.n_tiles;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t per = (int64_t)a.R * SUM_WAVES, c0 = chunk * per;
  const int64_t end = a.n - c0 < per ? a.n : c0 + per;
  const uint32_t key = a.key[end - 1];
  if (key >= (uint32_t)a.rows) return;
  const int s = a.row_ptr[key], e = a.row_ptr[key + 1];
  if (s < c0 || e <= end) return;
  const int last = (int)((e - 1) / per), count = last - chunk + 1;
  const int slot = s == c0 ? 0 : 1;
  __shared__ float sh[JOIN_WAVES][4][64];
  // 256 columns a block: 64 lanes x 4
  const int col = tile * 256 + lane * 4;
  const int live = a.D - col < 0 ? 0 : a.D - col < 4 ? a.D - col : 4;
  float acc[4] = {};
  const auto add = [&](auto whole) {
#pragma unroll 8
    for (int k = wave; k < count; k += JOIN_WAVES) {
      const float* p = a.part + ((int64_t)(chunk + k) * 2 + (k == 0 ? slot : 0)) * a.D + col;
      float v[4] = {};
      if (decltype(whole)::value) load_pack(p, v);
      else
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j < live) v[j] = p[j];
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] += v[j];
    }
  };
  if (live == 4) add(std::true_type());
  else if (live > 0) add(std::false_type());
#pragma unroll
  for (int j = 0; j < 4; ++j) sh[wave][j][lane] = acc[j];
  __syncthreads();
  if (wave != 0) return;
  TO* out = reinterpret_cast<TO*>(a.d_table) + (int64_t)key * a.t_stride + col;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float v = sh[0][j][lane];
#pragma unroll
    for (int w = 1; w < JOIN_WAVES; ++w) v += sh[w][j][lane];
    if (j < live) put(out + j, v * a.scale, a.accumulate);
  }
}

// ------------------------------------------------------------------ tables that fit into LDS
// Up to TABLE_ROWS rows need no sort: a wave adds its rows of d_out to a table of its own in LDS, 64 columns wide, lane by lane and
// in order; a row more takes the tokens without one.  The block joins its waves' tables and writes one part; k_table_join
// adds the parts in order.  Four rows make one trip to LDS; read, add and write take a third of the time that LDS's float
// atomics (29696 x 256 rows and 119 tokens: 52 us with atomics, 16 so, 20 sorted).  What bounds it at 119 rows, where one
// block of four waves fits into a compute unit, is the instructions of its waves; many rows come at 3.9 to 4.2 TB/s.
#define TABLE_ROWS 128
#define TABLE_WAVES 4
#define TABLE_U 16   // rows in flight, twice
#define TABLE_CHAIN 1024   // rows a wave adds at most: as many additions of one 32-bit sum, if all are of one token
struct TableIn {
  const void* d_out; int64_t d_stride;
  TokenView tok; int64_t n;
  int32_t rows, D, n_tiles, n_chunks;
  int64_t per_wave;
  float scale;
  float* part;                               // [n_chunks][rows][D]
  void* d_table; int64_t t_stride;
  bool accumulate;
};
template <typename T> struct RawBits { typedef uint16_t type; };
template <> struct RawBits<float> { typedef float type; };
template <typename T, int ROWS>
__global__ __launch_bounds__(TABLE_WAVES * 64) void k_table_sums(TableIn a) {
  __shared__ __attribute__((aligned(16))) float tab[TABLE_WAVES][ROWS + 1][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int chunk = blockIdx.x / a.n_tiles, tile = blockIdx.x % a.n_tiles;
  const int col = tile * 64 + lane;
  const uint32_t at = (uint32_t)(col < a.D ? col : a.D - 1) * (uint32_t)sizeof(T);
  const int64_t w0 = ((int64_t)chunk * TABLE_WAVES + wave) * a.per_wave, left = a.n - w0;
  const int rows = left <= 0 ? 0 : (int)(left < a.per_wave ? left : a.per_wave);
  f32x4* const clear = reinterpret_cast<f32x4*>(&tab[wave][0][0]);
#pragma unroll 4
  for (int k = lane; k < (a.rows + 1) * 16; k += 64) clear[k] = f32x4{0.f, 0.f, 0.f, 0.f};
  // a lane only ever touches its own column of its own wave's table
  typename RawBits<T>::type v[2][TABLE_U];    // as loaded (a conversion right behind the load would wait for it)
  int id[2];                                  // of 64 rows, a lane each
  const auto tokens = [&](int b) {
    int k = a.rows;
    if (b + lane < rows) {
      k = a.tok.at(w0 + b + lane);
      if (k < 0) k = a.tok.n_rows;            // (row n_rows of the table, or the one behind it)
    }
    return k;
  };
  // the rows of a batch lie at fixed 32-bit offsets from its first (the host sees to it), behind the last row at the last one's
  const int64_t step = a.d_stride * (int64_t)sizeof(T);
  const char* row = reinterpret_cast<const char*>(a.d_out) + w0 * step;
  uint32_t off[TABLE_U];
#pragma unroll
  for (int u = 0; u < TABLE_U; ++u) off[u] = at + (uint32_t)u * (uint32_t)step;
  const auto fetch = [&](int b, typename RawBits<T>::type (&x)[TABLE_U]) {
    if (b >= rows) return;
    if (rows - b < TABLE_U) {
#pragma unroll
      for (int u = 0; u < TABLE_U; ++u)
        off[u] = at + (uint32_t)(u < rows - b ? u : rows - b - 1) * (uint32_t)step;
    }
#pragma unroll
    for (int u = 0; u < TABLE_U; ++u) {
      asm("" : "+v"(off[u]));     // a 32-bit offset to the row's scalar address
      x[u] = *reinterpret_cast<const typename RawBits<T>::type*>(row + off[u]);
    }
    row += TABLE_U * step;
  };
  float* const own = &tab[wave][0][lane];
  if (rows > 0) {
    id[0] = tokens(0);
    fetch(0, v[0]);
    for (int b = 0; b < rows; b += 64) {
      id[1] = tokens(b + 64);
#pragma unroll
      for (int q = 0; q < 64 / TABLE_U; ++q) {
        if (b + q * TABLE_U >= rows) break;
        fetch(b + (q + 1) * TABLE_U, v[(q + 1) & 1]);
#pragma unroll
        for (int u = 0; u < TABLE_U; u += 4) {   // four at a time: one trip to LDS; a later row of the same token adds to the earlier
          float x[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            asm("" : "+v"(v[q & 1][u + j]));
            x[j] = (float)__builtin_bit_cast(T, v[q & 1][u + j]);
          }
          const int k0 = __builtin_amdgcn_readlane(id[0], q * TABLE_U + u), k1 = __builtin_amdgcn_readlane(id[0], q * TABLE_U + u + 1);
          const int k2 = __builtin_amdgcn_readlane(id[0], q * TABLE_U + u + 2), k3 = __builtin_amdgcn_readlane(id[0], q * TABLE_U + u + 3);
          const float t0 = own[k0 * 64], t1 = own[k1 * 64], t2 = own[k2 * 64], t3 = own[k3 * 64];
          const float s0 = t0 + x[0];
          float s1 = k1 == k0 ? s0 : t1;
          s1 += x[1];
          float s2 = k2 == k0 ? s0 : t2;
          s2 = k2 == k1 ? s1 : s2;
          s2 += x[2];
          float s3 = k3 == k0 ? s0 : t3;
          s3 = k3 == k1 ? s1 : s3;
          s3 = k3 == k2 ? s2 : s3;
          s3 += x[3];
          own[k0 * 64] = s0;
          own[k1 * 64] = s1;
          own[k2 * 64] = s2;
          own[k3 * 64] = s3;
        }
      }
      id[0] = id[1];
    }
  }
  __syncthreads();
  float* part = a.part + (int64_t)chunk * a.rows * a.D;
  if (col < a.D)
#pragma unroll 4
    for (int k = wave; k < a.rows; k += TABLE_WAVES) {
      float sum = tab[0][k][lane];
#pragma unroll
      for (int w = 1; w < TABLE_WAVES; ++w) sum += tab[w][k][lane];
      part[(int64_t)k * a.D + col] = sum;
    }
}
template <typename TO>
__global__ __launch_bounds__(512) void k_table_join(TableIn a) {
  __shared__ float sh[8][64];
  const int row = blockIdx.x / a.n_tiles, tile = blockIdx.x % a.n_tiles;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = tile * 64 + lane;
  float sum = 0.f;
  if (col < a.D) {
    const float* p = a.part + (int64_t)row * a.D + col;
#pragma unroll 8
    for (int c = wave; c < a.n_chunks; c += 8) sum += p[(int64_t)c * a.rows * a.D];
  }
  sh[wave][lane] = sum;
  __syncthreads();
  if (wave > 0 || col >= a.D) return;
#pragma unroll
  for (int w = 1; w < 8; ++w) sum += sh[w][lane];
  put(reinterpret_cast<TO*>(a.d_table) + (int64_t)row * a.t_stride + col, sum * a.scale, a.accumulate);
}

// ------------------------------------------------------------------ host side
// Sort: passes of 8 bits while they take no more passes than 11 bits would (a pass of 2048 bins costs twice one of 256: each
// block reads the whole count table): one pass for up to 255 rows (the token outside is one more key), two below 65536 rows;
// from there two passes of 11 bits up to 2^22 rows, three beyond.
static int sort_bits(int32_t rows) { return rows < 65536 ? 8 : 11; }
static int sort_passes(int32_t n_rows, int bits) {
  int p = 1;
  while (p * bits < 31 && (n_rows >> (p * bits)) != 0) ++p;
  return p;
}
// Blocks of a sort pass: 1024 positions or more each; every block reads the whole count table, so there are at most 64 blocks
// with 2048 bins and 512 with 256.
static int sort_per_block(int64_t n, int bits) {
  const int64_t most = bits == 8 ? 512 : 64;
  const int64_t per = (n + most - 1) / most;
  return (int)((per < 1024 ? 1024 : per + SORT_NT - 1) / SORT_NT * SORT_NT);
}
// Positions of a wave: about 8192 waves over the chip, at least 8 positions.
static int chunk_rows(int64_t n, int tiles) {
  int r = 8;
  while (r < 512 && n * tiles > (int64_t)r * 8192) r *= 2;
  return r;
}
// Blocks of the table sums: as many as the chip holds at once (a block takes rows + 1 KB of LDS), 32 rows a wave or more; whole
// multiples of that many where a wave would add more than TABLE_CHAIN rows (600000 x 256 fp32: 143 -> 156 us, 400000 x 2048 702 ->
// 791, the parts that the join reads; 8192 x 16448, where the chip was not full, 243 -> 199).
static int64_t table_per_wave(int64_t n, int32_t rows, int32_t width) {
  const int64_t tiles = (width + 63) / 64, held = 256 * (rows <= 32 ? 4 : rows <= 64 ? 2 : 1);
  const int64_t waves = (tiles < held ? held / tiles : 1) * TABLE_WAVES;
  const int64_t rounds = (n + waves * TABLE_CHAIN - 1) / (waves * TABLE_CHAIN);
  const int64_t per = rounds > 1 ? (n + waves * rounds - 1) / (waves * rounds) : (n + waves - 1) / waves;
  return per < 32 ? 32 : (per + 7) / 8 * 8;
}
static int64_t table_chunks(int64_t n, int32_t rows, int32_t width) {
  const int64_t per = table_per_wave(n, rows, width) * TABLE_WAVES;
  return (n + per - 1) / per;
}
// Measured against the sort (119 rows, us): 29 x 256 7 against 10, 29696 x 256 16 against 20, 29696 x 1024 32 against 39,
// 600000 x 64 38 against 107, 600000 x 256 156 against 153; bf16 29696 x 1024 31 against 31.  (A batch's offsets are 32 bits.)
static bool table_form(int64_t n, int32_t rows, int64_t d_stride) { return n > 0 && rows <= TABLE_ROWS && d_stride <= (1 << 24); }
struct EmbedWs { uint32_t* key[2]; int32_t* pos[2]; int32_t* hist; int32_t* row_ptr; float* part; size_t bytes; };
static EmbedWs embed_ws(void* base, int64_t n, int32_t rows, int32_t width) {
  char* p = (char*)base;
  size_t used = 0;
  const auto take = [&](size_t bytes) { char* r = p + used; used += align_up(bytes, 256); return r; };
  EmbedWs w;
  for (int k = 0; k < 2; ++k) { w.key[k] = (uint32_t*)take((size_t)n * 4); w.pos[k] = (int32_t*)take((size_t)n * 4); }
  const int bits = sort_bits(rows);
  const int64_t blocks = n ? (n + sort_per_block(n, bits) - 1) / sort_per_block(n, bits) : 0;
  w.hist = (int32_t*)take((size_t)blocks * (1 << bits) * 4);
  w.row_ptr = (int32_t*)take(((size_t)rows + 1) * 4);
  // (half-precision tiles are the widest: fewest tiles, shortest chunks, most partial rows)
  const int64_t r = (int64_t)chunk_rows(n, (width + 511) / 512) * SUM_WAVES;
  const size_t parts = (size_t)((n + r - 1) / r) * 2, table = table_form(n, rows, 0) ? (size_t)table_chunks(n, rows, width) * rows : 0;
  w.part = (float*)take((parts > table ? parts : table) * (size_t)width * 4);
  w.bytes = used;
  return w;
}
size_t embed_grad_workspace(int64_t n, int32_t rows, int32_t width) { return embed_ws(nullptr, n, rows, width).bytes; }

// The table in 16-byte units if the sort's launches clear it: it has to be one aligned piece of memory, and where the sort takes
// several launches of several blocks, most of its rows empty; else every row that is written twice costs more than the others
// gain (bf16, us: 32000 x 1024 with 4096 positions 31 -> 28, 8192 35 -> 38, 65536 61 -> 69; 10^6 x 64 with 10^5 171 -> 152).
static int64_t table_units(const EmbedGrad& g) {
  const int64_t bytes = (int64_t)g.rows * g.width * (g.grad_dtype == LIGDIFF_F32 ? 4 : 2);
  if (g.accumulate || g.n == 0 || g.t_stride != g.width || (reinterpret_cast<uintptr_t>(g.d_table) | bytes) % 16) return 0;
  return g.n <= SORT_SMALL || g.rows / 8 >= g.n ? bytes / 16 : 0;
}
static int clear_blocks(int64_t units, int threads) { return (int)std::min<int64_t>((units + threads - 1) / threads, 1024); }
// Sorts into key[0] / pos[0]; returns whether it wrote row_ptr.
static bool sort_small(const EmbedGrad& g, const EmbedWs& w, hipStream_t s) {
  SortPass a{};
  a.tok = g.tok; a.n = g.n; a.key_out = w.key[0]; a.pos_out = w.pos[0]; a.rows = g.rows;
  const int passes = sort_passes(g.tok.n_rows, 8);
  const bool ptr = passes == 1 && g.rows < 256;
  a.row_ptr = ptr ? w.row_ptr : nullptr;
  a.blocks = 1; a.clear = (u32x4*)g.d_table; a.n_clear = table_units(g);
  const dim3 grid(1 + clear_blocks(a.n_clear, SORT_SMALL_NT));
  if (passes == 1) hipLaunchKernelGGL(k_sort_small<1>, grid, dim3(SORT_SMALL_NT), 0, s, a);
  else if (passes == 2) hipLaunchKernelGGL(k_sort_small<2>, grid, dim3(SORT_SMALL_NT), 0, s, a);
  else if (passes == 3) hipLaunchKernelGGL(k_sort_small<3>, grid, dim3(SORT_SMALL_NT), 0, s, a);
  else hipLaunchKernelGGL(k_sort_small<4>, grid, dim3(SORT_SMALL_NT), 0, s, a);
  return ptr;
}
template <int BITS> static int sort_tokens(const EmbedGrad& g, const EmbedWs& w, hipStream_t s) {
  SortPass a;
  a.tok = g.tok; a.n = g.n; a.per_block = sort_per_block(g.n, BITS); a.hist = w.hist; a.rows = g.rows;
  const int blocks = (int)((g.n + a.per_block - 1) / a.per_block);
  const int passes = sort_passes(g.tok.n_rows, BITS);
  a.blocks = blocks;
  const int64_t units = table_units(g), each = (units + 2 * passes - 1) / (2 * passes);
  int64_t from = 0;
  const auto clear = [&]() {    // the next part of the table; returns the launch's grid
    a.clear = (u32x4*)g.d_table + from;
    a.n_clear = std::min(each, units - from);
    from += a.n_clear;
    return dim3(blocks + clear_blocks(a.n_clear, SORT_NT));
  };
  const auto pass = [&](auto first) {
    constexpr bool FIRST = decltype(first)::value;
    const dim3 count = clear();
    if (units) hipLaunchKernelGGL((k_sort_count<BITS, FIRST, true>), count, dim3(SORT_NT), 0, s, a);
    else hipLaunchKernelGGL((k_sort_count<BITS, FIRST, false>), count, dim3(SORT_NT), 0, s, a);
    const dim3 scatter = clear();
    if (units) hipLaunchKernelGGL((k_sort_scatter<BITS, FIRST, true>), scatter, dim3(SORT_NT), 0, s, a);
    else hipLaunchKernelGGL((k_sort_scatter<BITS, FIRST, false>), scatter, dim3(SORT_NT), 0, s, a);
  };
  for (int p = 0; p < passes; ++p) {
    a.shift = p * BITS;
    a.key_in = w.key[(p + 1) & 1]; a.pos_in = w.pos[(p + 1) & 1];
    a.key_out = w.key[p & 1]; a.pos_out = w.pos[p & 1];
    a.row_ptr = passes == 1 && g.rows < (1 << BITS) ? w.row_ptr : nullptr;
    if (p == 0) pass(std::true_type());
    else pass(std::false_type());
  }
  return passes;
}

template <typename T, typename TO> static void table_sums(const TableIn& a, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)a.n_chunks * a.n_tiles)), block(TABLE_WAVES * 64);
  if (a.rows <= 32) hipLaunchKernelGGL((k_table_sums<T, 32>), grid, block, 0, s, a);
  else if (a.rows <= 64) hipLaunchKernelGGL((k_table_sums<T, 64>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((k_table_sums<T, TABLE_ROWS>), grid, block, 0, s, a);
  hipLaunchKernelGGL((k_table_join<TO>), dim3((unsigned)((int64_t)a.rows * a.n_tiles)), dim3(512), 0, s, a);
}
template <typename T, typename TO> static void segment_sums(SegIn a, hipStream_t s) {
  a.n_tiles = (a.D + 64 * Pack<T>::N - 1) / (64 * Pack<T>::N);
  a.R = chunk_rows(a.n, a.n_tiles);
  const int64_t per = (int64_t)a.R * SUM_WAVES;
  a.n_chunks = (int)((a.n + per - 1) / per);
  a.zero_blocks = (a.rows + ZERO_ROWS - 1) / ZERO_ROWS;
  hipLaunchKernelGGL((k_segment_sums<T, TO>), dim3((unsigned)(a.zero_blocks + (int64_t)a.n_chunks * a.n_tiles)), dim3(SUM_WAVES * 64),
                     0, s, a);
  if (a.n_chunks > 1) {
    SegIn j = a;
    j.n_tiles = (a.D + 255) / 256;
    hipLaunchKernelGGL((k_segment_join<TO>), dim3((unsigned)((int64_t)j.n_chunks * j.n_tiles)), dim3(JOIN_WAVES * 64), 0, s, j);
  }
}

void embed_grad(const EmbedGrad& g, void* workspace, hipStream_t s) {
  const EmbedWs w = embed_ws(workspace, g.n, g.rows, g.width);
  const bool wide = g.grad_dtype == LIGDIFF_F32;
  if (table_form(g.n, g.rows, g.d_stride)) {
    TableIn t;
    t.d_out = g.d_out; t.d_stride = g.d_stride; t.tok = g.tok; t.n = g.n; t.rows = g.rows; t.D = g.width; t.scale = g.scale;
    t.n_tiles = (g.width + 63) / 64; t.per_wave = table_per_wave(g.n, g.rows, g.width);
    t.n_chunks = (int)table_chunks(g.n, g.rows, g.width); t.part = w.part;
    t.d_table = g.d_table; t.t_stride = g.t_stride; t.accumulate = g.accumulate;
    if (g.dtype == LIGDIFF_F32) table_sums<float, float>(t, s);
    else if (g.dtype == LIGDIFF_BF16) { if (wide) table_sums<bf16_t, float>(t, s); else table_sums<bf16_t, bf16_t>(t, s); }
    else { if (wide) table_sums<f16_t, float>(t, s); else table_sums<f16_t, f16_t>(t, s); }
    return;
  }
  SegIn a;
  a.have_ptr = false;
  int passes = 1;
  if (g.n > 0 && g.n <= SORT_SMALL) {
    a.have_ptr = sort_small(g, w, s);
  } else if (g.n > 0) {
    const int bits = sort_bits(g.rows);
    passes = bits == 8 ? sort_tokens<8>(g, w, s) : sort_tokens<11>(g, w, s);
    a.have_ptr = passes == 1 && g.rows < (1 << bits);
  }
  a.d_out = g.d_out; a.d_stride = g.d_stride; a.key = w.key[(passes - 1) & 1]; a.pos = w.pos[(passes - 1) & 1]; a.n = g.n;
  a.row_ptr = w.row_ptr; a.rows = g.rows; a.D = g.width; a.scale = g.scale; a.part = w.part;
  a.d_table = g.d_table; a.t_stride = g.t_stride; a.accumulate = g.accumulate; a.cleared = table_units(g) > 0;
  if (g.dtype == LIGDIFF_F32) segment_sums<float, float>(a, s);
  else if (g.dtype == LIGDIFF_BF16) { if (wide) segment_sums<bf16_t, float>(a, s); else segment_sums<bf16_t, bf16_t>(a, s); }
  else { if (wide) segment_sums<f16_t, float>(a, s); else segment_sums<f16_t, f16_t>(a, s); }
}

// A launch holds fewer than 2^32 threads: 2^29 rows of a table that is sorted for, 2^29 columns over the rows of a small one.
static bool launches_fit(const EmbedGrad& g) {
  const int64_t most = 0xffffffffLL;
  if (table_form(g.n, g.rows, g.d_stride)) {
    const int64_t tiles = ((int64_t)g.width + 63) / 64;
    return table_chunks(g.n, g.rows, g.width) * tiles * TABLE_WAVES * 64 <= most && g.rows * tiles * 512 <= most;
  }
  const int64_t columns = 64 * (g.dtype == LIGDIFF_F32 ? Pack<float>::N : Pack<bf16_t>::N), tiles = (g.width + columns - 1) / columns;
  const int64_t per = (int64_t)chunk_rows(g.n, (int)tiles) * SUM_WAVES, chunks = (g.n + per - 1) / per;
  return (((int64_t)g.rows + ZERO_ROWS - 1) / ZERO_ROWS + chunks * tiles) * SUM_WAVES * 64 <= most &&
         chunks * (((int64_t)g.width + 255) / 256) * JOIN_WAVES * 64 <= most;
}

extern "C" size_t ligdiff_embed_grad_workspace_bytes(int64_t n_tokens, int64_t n_rows, int32_t width) {
  if (bad_embed(LIGDIFF_F32, n_rows, width, 4, n_tokens)) return 0;
  return embed_grad_workspace(n_tokens, (int32_t)n_rows, width);
}

extern "C" int ligdiff_embed_grad(const void* d_out, int32_t dtype, int64_t d_stride, const void* tokens, int32_t token_bytes,
                                  int64_t n_tokens, int64_t n_rows, int32_t width, float scale, void* d_table,
                                  int32_t grad_dtype, int64_t table_stride, int32_t accumulate, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  if (bad_embed(dtype, n_rows, width, token_bytes, n_tokens) || (grad_dtype != dtype && grad_dtype != LIGDIFF_F32) ||
      d_stride < width || table_stride < width || !d_table || !workspace)
    return LIGDIFF_ERR_ARG;
  if (n_tokens > 0 && (!d_out || !tokens)) return LIGDIFF_ERR_ARG;
  const EmbedGrad g{d_out, dtype, d_stride, TokenView{tokens, token_bytes, (int32_t)n_rows}, n_tokens, (int32_t)n_rows, width, scale,
              d_table, grad_dtype, table_stride, accumulate != 0};
  if (!launches_fit(g)) return LIGDIFF_ERR_ARG;
  if (workspace_bytes < embed_grad_workspace(n_tokens, (int32_t)n_rows, width)) return LIGDIFF_ERR_WORKSPACE;
  embed_grad(g, workspace, (hipStream_t)stream);
  LD_CHECK_LAUNCH();
  return LIGDIFF_OK;
}

// ------------------------------------------------------------------ atom types of the score network
// Atom branch of the input embedding per TYPE (model1.py:599-609 on one-hot rows): u = Wa[:, v] + ba, GELU(LN(u)); row LD_A
// is that of a zero feature row.  One wave a type; the atoms then look their row up (k_pos_embed), 120 rows of
// arithmetic instead of one per atom and no [N,119] features to read.
__global__ __launch_bounds__(256) void k_type_embed(const float* __restrict__ Wa, const float* __restrict__ ba,
                                                    const float* __restrict__ ga, const float* __restrict__ bea,
                                                    float* __restrict__ pre, float* __restrict__ emb) {
  const int lane = threadIdx.x & 63;
  const int v = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (v > LD_A) return;
  f32x4 u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int col = lane * 4 + i;
    u[i] = ba[col] + (v < LD_A ? Wa[(size_t)col * LD_A + v] : 0.f);
  }
  const float mean = wave_sum((u[0] + u[1]) + (u[2] + u[3])) * (1.0f / 256.0f);
  const f32x4 d = u - mean;
  const float var = wave_sum((d[0] * d[0] + d[1] * d[1]) + (d[2] * d[2] + d[3] * d[3])) * (1.0f / 256.0f);
  const float rstd = 1.0f / sqrtf(var + 1e-5f);
  f32x4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = gelu_exact(d[i] * rstd * ga[lane * 4 + i] + bea[lane * 4 + i]);
  *reinterpret_cast<f32x4*>(pre + (size_t)v * 256 + lane * 4) = u;
  *reinterpret_cast<f32x4*>(emb + (size_t)v * 256 + lane * 4) = o;
}

// Gradient of the per-type atom branch: du [LD_A + 1, 256] before LayerNorm -> Wa[:, v] += du[v], ba += sum_v du[v].  Block v
// writes column v of Wa; block LD_A the bias (a column a thread, in the order of the types).
__global__ __launch_bounds__(256) void k_type_embed_dw(const float* __restrict__ du, float* __restrict__ dWa, float* __restrict__ dba) {
  const int c = threadIdx.x, v = blockIdx.x;
  if (v < LD_A) {
    dWa[(size_t)c * LD_A + v] += du[(size_t)v * 256 + c];
    return;
  }
  float sum = 0.f;
#pragma unroll 8
  for (int k = 0; k <= LD_A; ++k) sum += du[(size_t)k * 256 + c];
  dba[c] += sum;
}

void type_embed(const float* Wa, const float* ba, const float* ga, const float* bea, float* pre, float* emb, hipStream_t s) {
  hipLaunchKernelGGL(k_type_embed, dim3(ceil_div(LD_A + 1, 4)), dim3(256), 0, s, Wa, ba, ga, bea, pre, emb);
}
void type_embed_dw(const float* du, float* dWa, float* dba, hipStream_t s) {
  hipLaunchKernelGGL(k_type_embed_dw, dim3(LD_A + 1), dim3(256), 0, s, du, dWa, dba);
}
