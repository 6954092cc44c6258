// Log probabilities of given tokens, with entropy and the likeliest
// alternatives, over rows of V logits of any type and row stride:
//   m = max x,  s = sum exp(x - m),  logp = x_target - m - log s,
//   entropy = log s - sum exp(x - m) (x - m) / s,
//   top: the K largest (ties: the lowest index) with their log probabilities;
// and the gradient, p = exp(x - m) / s:
//   dx_j = d_logp ([j = target] - p_j) - d_entropy p_j (log p_j + entropy)
//          + sum_k d_top_k ([j = id_k] - p_j).
//
// Forward reads a row once (a running maximum, sum and weighted sum in each
// thread, rescaled when the maximum grows), backward reads and writes it once:
// both are bound by memory.  The top K need no second pass over the row: the
// row's threads form 64 groups, the K-th largest of the 64 group maxima is a
// lower bound of the K-th largest logit, and only threads whose own maximum
// reaches it read their few elements again (from L2) and list those at or
// above it; the list (about K long for logits without many ties) is ranked.
// A list that overflows (constant rows) takes K passes over the row instead.
//
// A row of nothing but -inf has no distribution: logp and top_logp -inf,
// entropy 0, gradient 0.  NaN or +inf in a row makes its results NaN; NaN
// ranks lowest among the alternatives.  Sums, maxima and logs are fp32.
#include "kernels/elem.h"
#include "kernels/lm.h"

namespace mfl {
namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kList = 1024;  // candidates of a row (LDS)

// Running maximum, sum of exp(x - m) and sum of exp(x - m) (x - m).
struct Soft {
  float m, s, t;
};
__device__ __forceinline__ Soft soft_none() { return {-INFINITY, 0.f, 0.f}; }
// t of a sum whose maximum goes from m to M: each (x - m) grows by (m - M)
__device__ __forceinline__ void soft_raise(Soft& a, float M) {
  if (a.s != 0.f) {
    const float d = a.m - M, c = exp2f(d * kLog2e);
    a.t = c * (a.t + (c > 0.f ? d * a.s : 0.f));
    a.s *= c;
  }
  a.m = M;
}
__device__ __forceinline__ Soft soft_join(Soft a, Soft b) {
  const float M = fmaxf(a.m, b.m);
  soft_raise(a, M);
  soft_raise(b, M);
  return {M, a.s + b.s, a.t + b.t};
}
// N more elements (fill: -inf)
template <int N>
__device__ __forceinline__ void soft_add(Soft& a, const float* x) {
  float M = a.m;
#pragma unroll
  for (int k = 0; k < N; ++k) M = fmaxf(M, x[k]);
  if (M > a.m) soft_raise(a, M);
  const float m = a.m == -INFINITY ? 0.f : a.m;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const float d = x[k] - m, e = __builtin_amdgcn_exp2f(d * kLog2e);
    a.s += e;
    a.t = fmaf(e, fmaxf(d, -1e4f), a.t);  // a masked logit adds 0, not 0 * -inf
  }
}

// Order of the alternatives as whole numbers: larger logit first, then lower
// index.  -0 and 0 tie, NaN ranks as -inf.
__device__ __forceinline__ int order_of(float v) {
  if (!(v == v)) v = -INFINITY;
  const int b = __float_as_int(v + 0.f);
  return b ^ ((b >> 31) & 0x7fffffff);
}
__device__ __forceinline__ uint64_t rank_key(int order, uint32_t id) {
  return ((uint64_t)((uint32_t)order ^ 0x80000000u) << 32) | (0xffffffffu - id);
}
__device__ __forceinline__ uint32_t key_id(uint64_t k) { return 0xffffffffu - (uint32_t)k; }
__device__ __forceinline__ float key_value(uint64_t k) {
  const int o = (int)((uint32_t)(k >> 32) ^ 0x80000000u);
  return __int_as_float(o ^ ((o >> 31) & 0x7fffffff));
}

template <int THREADS>
struct RowShared {
  float m[16], s[16], t[16];
  int group[64];
  int bound, count;
  uint64_t best[16], top[kTopMax], list[THREADS > 64 ? kList : 256];
};

template <int THREADS>
__device__ __forceinline__ void row_sync() {
  if constexpr (THREADS > 64) __syncthreads();
  else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"), __builtin_amdgcn_wave_barrier();
}

// The K largest keys of x[0 .. n) into sh.top, each thread holding the largest
// order `mine` of its own elements (those its loop visits).
template <typename T, int THREADS>
__device__ void row_top(const T* x, int n, uint32_t first, int K, int mine, RowShared<THREADS>& sh) {
  constexpr int N = Vec<T>::N, GROUP = THREADS / 64, CAP = THREADS > 64 ? kList : 256;
  const int tid = threadIdx.x % THREADS;
  int g = mine;
#pragma unroll
  for (int o = 1; o < GROUP; o <<= 1) g = max(g, __shfl_xor(g, o, 64));
  if (tid % GROUP == 0) sh.group[tid / GROUP] = g;
  if (tid == 0) sh.count = 0;
  row_sync<THREADS>();
  if (tid < 64) {
    const int v = sh.group[tid];
    int rank = 0;
    for (int j = 0; j < 64; ++j) {
      const int w = sh.group[j];
      rank += w > v || (w == v && j < tid);
    }
    if (rank == K - 1) sh.bound = v;
  }
  row_sync<THREADS>();
  const int bound = sh.bound;
  if (mine >= bound) {
    for (int c = tid * N; c < n; c += THREADS * N)
      for (int k = 0; k < N; ++k)
        if (c + k < n) {
          const int o = order_of(to_f(x[c + k]));
          if (o >= bound) {
            const int at = atomicAdd(&sh.count, 1);
            if (at < CAP) sh.list[at] = rank_key(o, first + c + k);
          }
        }
  }
  row_sync<THREADS>();
  const int count = sh.count;
  if (count <= CAP) {
    for (int i = tid; i < count; i += THREADS) {
      const uint64_t v = sh.list[i];
      int rank = 0;
      for (int j = 0; j < count; ++j) rank += sh.list[j] > v;
      if (rank < K) sh.top[rank] = v;
    }
    row_sync<THREADS>();
    return;
  }
  uint64_t last = ~0ull;  // K passes, each for the largest key below the last one
  for (int k = 0; k < K; ++k) {
    uint64_t best = 0;
    for (int c = tid; c < n; c += THREADS) {
      const uint64_t v = rank_key(order_of(to_f(x[c])), first + c);
      if (v < last && v > best) best = v;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const uint64_t w = __shfl_xor((unsigned long long)best, o, 64);
      best = w > best ? w : best;
    }
    row_sync<THREADS>();
    if ((tid & 63) == 0) sh.best[tid >> 6] = best;
    row_sync<THREADS>();
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) best = sh.best[w] > best ? sh.best[w] : best;
    if (tid == 0) sh.top[k] = best;
    last = best;
  }
  row_sync<THREADS>();
}

// One pass over x[0 .. n): the row's (or its part's) running sums in all
// threads of the row, and the largest order of this thread's elements.
template <typename T, int THREADS>
__device__ __forceinline__ Soft row_pass(const T* x, int n, int& mine, RowShared<THREADS>& sh) {
  constexpr int N = Vec<T>::N, UNROLL = 4;
  const int tid = threadIdx.x % THREADS;
  Soft a = soft_none();
  float largest = -INFINITY;
  int c = tid * N;
  for (; c + (UNROLL - 1) * THREADS * N + N <= n; c += UNROLL * THREADS * N) {
    float f[UNROLL][N];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) load_row<T, N>(x, c + u * THREADS * N, n, -INFINITY, f[u]);
    soft_add<UNROLL * N>(a, &f[0][0]);
  }
  for (; c < n; c += THREADS * N) {
    float f[N];
    load_row<T, N>(x, c, n, -INFINITY, f);
    soft_add<N>(a, f);
  }
  largest = a.m;
  mine = order_of(largest);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const Soft b = {__shfl_xor(a.m, o, 64), __shfl_xor(a.s, o, 64), __shfl_xor(a.t, o, 64)};
    a = soft_join(a, b);
  }
  if constexpr (THREADS > 64) {
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
      sh.m[w] = a.m;
      sh.s[w] = a.s;
      sh.t[w] = a.t;
    }
    __syncthreads();
    a = {sh.m[0], sh.s[0], sh.t[0]};
    for (int i = 1; i < THREADS / 64; ++i) a = soft_join(a, {sh.m[i], sh.s[i], sh.t[i]});
  }
  return a;
}

__device__ __forceinline__ int64_t target_of(const int64_t* t64, const int32_t* t32, int64_t row) {
  return t64 ? t64[row] : (int64_t)t32[row];
}

// Results of a row from its sums (and sh.top), by the row's threads.
template <typename T, int THREADS>
__device__ __forceinline__ void row_write(const TokenLogprobs& a, const T* x, int64_t row, Soft r,
                                          RowShared<THREADS>& sh) {
  const int tid = threadIdx.x % THREADS;
  const float logs = logf(r.s);
  const bool empty = r.m == -INFINITY && r.s == 0.f;
  if (tid == 0) {
    const int64_t t = target_of(a.target64, a.target32, row);
    float lp = 0.f;
    if (t >= 0 && t < a.V) lp = empty ? -INFINITY : (to_f(x[t]) - r.m) - logs;
    a.logp[row] = lp;
    const float entropy = empty ? 0.f : logs - r.t / r.s;
    a.entropy[row] = entropy;
    a.stats[3 * row] = r.m;
    a.stats[3 * row + 1] = r.s;
    a.stats[3 * row + 2] = entropy;
  }
  if (tid < a.K) {
    const uint64_t k = sh.top[tid];
    a.top_logp[row * a.K + tid] = empty ? -INFINITY : (key_value(k) - r.m) - logs;
    a.top_ids[row * a.K + tid] = key_id(k);
  }
}

template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS > 256 ? THREADS : 256) void logprobs_kernel(TokenLogprobs a) {
  constexpr int ROWS = THREADS < 256 ? 256 / THREADS : 1;
  __shared__ RowShared<THREADS> shared[ROWS];
  RowShared<THREADS>& sh = shared[threadIdx.x / THREADS];
  for (int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / THREADS; row < a.N; row += (int64_t)gridDim.x * ROWS) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    int mine;
    const Soft r = row_pass<T, THREADS>(x, a.V, mine, sh);
    if (a.K) row_top<T, THREADS>(x, a.V, 0, a.K, mine, sh);
    row_write<T, THREADS>(a, x, row, r, sh);
    row_sync<THREADS>();
  }
}

// Backward: a workgroup takes kBack elements of a row; p recomputed from the
// row's maximum and sum.  The target's and the alternatives' own terms are
// added by a rewrite of their elements behind a barrier.
constexpr int kBack = 16384;
template <typename T>
__global__ __launch_bounds__(256) void logprobs_bwd_kernel(TokenLogprobsBwd a, int parts) {
  constexpr int N = Vec<T>::N;
  const int64_t items = (int64_t)a.N * parts;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t row = item / parts;
    const int part = (int)(item - row * parts);
    const int lo = part * kBack, hi = min(a.C, lo + kBack);
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    T* dx = static_cast<T*>(a.dx) + row * a.C;
    const int64_t t = target_of(a.target64, a.target32, row);
    const bool has = t >= 0 && t < a.V;
    const float m = a.stats[3 * row], s = a.stats[3 * row + 1];
    const bool empty = m == -INFINITY && s == 0.f;
    const float dl = has && a.d_logp ? a.d_logp[row] : 0.f;
    const float dh = a.d_entropy ? a.d_entropy[row] : 0.f;
    float all = dl;
    if (a.d_top)
      for (int k = 0; k < a.K; ++k) all += a.d_top[row * a.K + k];
    // dx_j = -p_j (all + dh (log p_j + entropy)) + own terms
    const float inv = 1.f / s;
    const float ent = a.stats[3 * row + 2] - logf(s);
    const float base = empty ? 0.f : m;
    auto grad = [&](float v) -> float {
      if (empty) return 0.f;
      const float d = v - base, p = __builtin_amdgcn_exp2f(d * kLog2e) * inv;
      float w = all;
      if (dh != 0.f) w = fmaf(dh, fmaxf(d, -1e4f) + ent, w);
      return -p * w;
    };
    for (int c = lo + threadIdx.x * N; c < hi; c += 256 * N) {
      float f[N];
      load_row<T, N>(x, c, a.V, -INFINITY, f);
#pragma unroll
      for (int k = 0; k < N; ++k) f[k] = c + k < a.V ? grad(f[k]) : 0.f;
      store_row<T, N>(dx, c, hi, f);
    }
    __syncthreads();
    const int own = a.d_top ? a.K : 0;
    for (int i = threadIdx.x; i <= own; i += 256) {
      // thread i: alternative i; the last one: the target, unless an alternative
      // is the target (its thread adds both)
      int64_t j = i < own ? a.top_ids[row * a.K + i] : (has ? t : -1);
      if (j < lo || j >= hi || j >= a.V || empty) continue;
      float extra = i < own ? a.d_top[row * a.K + i] : dl;
      bool mine = true;
      for (int k = 0; k < own; ++k)
        if (k != i && a.top_ids[row * a.K + k] == j) {
          if (k < i) mine = false;  // the lowest place adds for all of them
          extra += a.d_top[row * a.K + k];
        }
      if (!mine) continue;
      if (i < own && has && t == j) extra += dl;
      dx[j] = from_f<T>(grad(to_f(x[j])) + extra);
    }
    __syncthreads();
  }
}

template <typename T>
void fwd_typed(const TokenLogprobs& a, hipStream_t s) {
  const int64_t cap = 1 << 20;
  if (a.V <= 2048) {
    const int64_t want = ((int64_t)a.N + 3) / 4;
    logprobs_kernel<T, 64><<<(unsigned)(want < cap ? want : cap), 256, 0, s>>>(a);
  } else if (a.V <= 16384) {
    logprobs_kernel<T, 256><<<(unsigned)(a.N < cap ? a.N : cap), 256, 0, s>>>(a);
  } else {
    logprobs_kernel<T, 1024><<<(unsigned)(a.N < cap ? a.N : cap), 1024, 0, s>>>(a);
  }
}
template <typename T>
void bwd_typed(const TokenLogprobsBwd& a, hipStream_t s) {
  const int parts = (a.C + kBack - 1) / kBack;
  const int64_t items = (int64_t)a.N * parts, cap = 1 << 20;
  logprobs_bwd_kernel<T><<<(unsigned)(items < cap ? items : cap), 256, 0, s>>>(a, parts);
}

}  // namespace

size_t token_logprobs_workspace(int, int, int, int) { return 0; }

void launch_token_logprobs(const TokenLogprobs& a, hipStream_t s) {
  if (a.type == ELEM_F32) fwd_typed<float>(a, s);
  else if (a.type == ELEM_BF16) fwd_typed<BF16>(a, s);
  else fwd_typed<F16>(a, s);
}
void launch_token_logprobs_bwd(const TokenLogprobsBwd& a, hipStream_t s) {
  if (a.type == ELEM_F32) bwd_typed<float>(a, s);
  else if (a.type == ELEM_BF16) bwd_typed<BF16>(a, s);
  else bwd_typed<F16>(a, s);
}

}  // namespace mfl
