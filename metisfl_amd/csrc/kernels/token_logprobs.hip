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
// A list that overflows (constant rows) takes K passes over the row instead: 64
// x 128000 bf16 zeros take 81 us with 4 alternatives and 397 us with 32, 2048 x
// 30522 2.7 ms with 32.
//
// Measured, calls among others over three sets of inputs in turn (copies of 1
// GiB: 4.7 to 5.1 TB/s; a pass that only reads goes above):
//   2560 x 30522   bf16  forward 36.7 us, 4.3 TB/s   backward 65 us, 4.8 TB/s
//   2560 x 30522   fp32  forward 53.9 us, 5.8 TB/s   backward 117 us, 5.3 TB/s
//   8192 x 128000  bf16  forward 348 us with 4 alternatives, 6.0 TB/s
//                        backward 790 us, with the entropy's gradient 782, 5.3 TB/s
//   509 x 50021    fp32  forward 24.5 us with 20 alternatives, 4.2 TB/s
//   130 x 128000   bf16  forward 14.9 us with 5 alternatives, 2.2 TB/s
//   1 x 30522      bf16  forward 7.0 us on the GPU with 5 alternatives, 7.4 us a call
//
// A row of nothing but -inf has no distribution: logp and top_logp -inf,
// entropy 0, gradient 0.  NaN or +inf in a row makes its results NaN; NaN
// ranks lowest among the alternatives.  Sums, maxima and logs are fp32.
#include "kernels/elem.h"
#include "kernels/lm.h"

#include <type_traits>

namespace mfl {
namespace {

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr int kList = 1024;  // candidates of a row (LDS)
constexpr int kSplitRows = 128, kSplitWidth = 98304, kSplitGroups = 512;  // see part_span

// Running maximum m, sum of exp(x - m) and sum of exp(x - m) (x - m) log2 e.
// exp(x - m) = exp2(x L - fl(m L)) with L = log2 e is one fused multiply-add
// and one v_exp_f32; what fl(m L) is rounded by (soft_off) is a factor common
// to the sum: soft_grow exchanges it with the maximum and soft_exact takes it
// out at the end, so the error of a term is a few times 2^-24 of |x - m|, not
// of |x|.  Up to |m| = 4096 it is at most 2^-12 and soft_exact's first order
// leaves 2^-25; beyond (logits of a large common part, rows masked with -1e9
// throughout) the difference x - m is taken first, and nothing is left over.
struct Soft {
  float m, s, t;
};
constexpr float kFar = 4096.f;
__device__ __forceinline__ float scaled_max(float m) { return m == -INFINITY ? 0.f : m * kLog2e; }
__device__ __forceinline__ float soft_off(float m) {  // x L - fl(m L) - off = (x - m) L
  return fabsf(m) > kFar ? 0.f : fmaf(m, kLog2e, -scaled_max(m));
}
// the sums to maximum M >= a.m: each exponent grows by d
__device__ __forceinline__ void soft_shift(Soft& a, float M, float d) {
  const float c = __builtin_amdgcn_exp2f(d);
  a.t = c * (a.t + (c > 0.f ? d * a.s : 0.f));
  a.s *= c;
  a.m = M;
}
// of exact sums (s is 0 only where nothing but -inf was added)
__device__ __forceinline__ void soft_raise(Soft& a, float M) {
  if (a.s != 0.f) soft_shift(a, M, (a.m - M) * kLog2e);
  a.m = M;
}
// of sums with their offset
__device__ __forceinline__ void soft_grow(Soft& a, float M) {
  if (a.s != 0.f) soft_shift(a, M, (a.m - M) * kLog2e - soft_off(a.m) + soft_off(M));
  a.m = M;
}
__device__ __forceinline__ void soft_exact(Soft& a) {
  const float off = soft_off(a.m);
  const float c = fmaf(-off, kLn2, 1.f);  // 2^-off
  a.t = c * fmaf(-off, a.s, a.t);
  a.s *= c;
}
// N more elements (fill: -inf) with the largest of them
template <int N>
__device__ __forceinline__ void soft_add(Soft& a, const float* x, float largest) {
  if (largest > a.m) soft_grow(a, largest);
  if (fabsf(a.m) > kFar && a.m != -INFINITY) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float d = (x[k] - a.m) * kLog2e, e = __builtin_amdgcn_exp2f(d);
      a.s += e;
      a.t = fmaf(e, fmaxf(d, -1e4f), a.t);
    }
    return;
  }
  const float ml = scaled_max(a.m);
  float s0 = 0.f, s1 = 0.f, t0 = 0.f, t1 = 0.f;
#pragma unroll
  for (int k = 0; k < N; k += 2) {
    const float d0 = fmaf(x[k], kLog2e, -ml), e0 = __builtin_amdgcn_exp2f(d0);
    s0 += e0;
    t0 = fmaf(e0, fmaxf(d0, -1e4f), t0);  // a masked logit adds 0, not 0 * -inf
    if (k + 1 < N) {
      const float d1 = fmaf(x[k + 1], kLog2e, -ml), e1 = __builtin_amdgcn_exp2f(d1);
      s1 += e1;
      t1 = fmaf(e1, fmaxf(d1, -1e4f), t1);
    }
  }
  a.s += s0 + s1;
  a.t += t0 + t1;
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
  float group[64];
  float bound;
  int count;
  uint64_t best[16], top[kTopMax], list[THREADS > 64 ? kList : 256];
};

template <int THREADS>
__device__ __forceinline__ void row_sync() {
  if constexpr (THREADS > 64) __syncthreads();
  else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"), __builtin_amdgcn_wave_barrier();
}

// What a thread saw of the row: the largest element of each of its two batches
// with the largest ones, those batches, and the largest element of the others.
struct Seen {
  float largest, second, others;
  int batch, batch2;
};
constexpr int kUnroll = 4;  // packs of a batch: the loads in flight of a thread

// The packs of batch `b` of a row of `n` elements: element u * N + k of f is
// x[((b * kUnroll + u) * THREADS + tid) * N + k], -inf behind the last whole pack.
template <typename T, int THREADS>
struct Batch {
  static constexpr int N = Vec<T>::N;
  Pack<T, N> v[kUnroll];
  __device__ __forceinline__ void load(const T* x, int b, int packs) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int i = (b * kUnroll + u) * THREADS + (int)(threadIdx.x % THREADS);
      v[u] = load_pack<T, N>(x + (int64_t)(i < packs ? i : packs - 1) * N);
    }
  }
  __device__ __forceinline__ void get(int b, int packs, float* f) const {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
#pragma unroll
      for (int k = 0; k < N; ++k) f[u * N + k] = to_f(v[u].e[k]);
    }
    if ((b + 1) * kUnroll * THREADS > packs) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int i = (b * kUnroll + u) * THREADS + (int)(threadIdx.x % THREADS);
#pragma unroll
        for (int k = 0; k < N; ++k) f[u * N + k] = i < packs ? f[u * N + k] : -INFINITY;
      }
    }
  }
};

// The K largest keys of x[0 .. n) into sh.top (ids counted from `first`).
template <typename T, int THREADS>
__device__ void row_top(const T* x, int n, uint32_t first, int K, Seen seen, RowShared<THREADS>& sh) {
  constexpr int N = Vec<T>::N, GROUP = THREADS / 64, CAP = THREADS > 64 ? kList : 256;
  const int tid = threadIdx.x % THREADS;
  // 64 groups of neighbouring threads; the K-th largest of their maxima
  float g = seen.largest;
  if constexpr (GROUP == 16) {
    g = max16(g);
  } else if constexpr (GROUP > 1) {
    g = max4(g);
    if constexpr (GROUP == 8)  // the eight lanes mirrored
      g = fmaxf(g, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(g), 0x141, 0xf, 0xf, false)));
  }
  if constexpr (GROUP > 1) {
    if (tid % GROUP == 0) sh.group[tid / GROUP] = g;
    __syncthreads();
    g = sh.group[tid & 63];
  }
  if (tid < 64) {  // (the first wave)
    int above = 0;  // groups above this lane's
    if (K <= 8) {   // four groups together: 16 to rank, about K log 2 elements more above the bound
      g = max4(g);
#pragma unroll
      for (int j = 0; j < 64; j += 4) above += lane_of(g, j) > g;
    } else {
#pragma unroll
      for (int j = 0; j < 64; ++j) above += lane_of(g, j) > g;
    }
    const float least = -max64(above < K ? -g : -INFINITY);
    if (tid == 0) {
      sh.bound = least;
      sh.count = 0;
    }
  }
  row_sync<THREADS>();
  const float bound = sh.bound;
  // threads that saw an element of that size list theirs (and NaN, which ranks
  // lowest: it is never below the bound)
  const int packs = n / N, batches = (packs + THREADS * kUnroll - 1) / (THREADS * kUnroll);
  auto list = [&](int id) {
    const int at = atomicAdd(&sh.count, 1);
    if (at < CAP) sh.list[at] = rank_key(order_of(to_f(x[id])), first + (uint32_t)id);
  };
  if (packs && !(seen.largest < bound)) {
    const bool few = seen.batch >= 0 && seen.others < bound;
    const int turns = !few ? batches : seen.second < bound ? 1 : 2;
    for (int turn = 0; turn < turns; ++turn) {
      const int b = !few ? turn : turn ? seen.batch2 : seen.batch;
      Batch<T, THREADS> v;
      v.load(x, b, packs);
      uint32_t mask = 0;  // a bit an element: their values are read again (from L1)
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        uint32_t part = 0;
#pragma unroll
        for (int k = 0; k < N; ++k) part |= to_f(v.v[u].e[k]) < bound ? 0u : 1u << k;
        mask |= (b * kUnroll + u) * THREADS + tid < packs ? part << (u * N) : 0u;
      }
      for (; mask; mask &= mask - 1) {
        const int e = __ffs(mask) - 1;
        list(((b * kUnroll + e / N) * THREADS + tid) * N + e % N);
      }
    }
  }
  // behind the last whole pack: one element of the first threads
  if (packs * N + tid < n && !(to_f(x[packs * N + tid]) < bound)) list(packs * N + tid);
  row_sync<THREADS>();
  const int count = sh.count;
  if (count <= CAP) {
    for (int i = tid; i < count; i += THREADS) {
      const uint64_t v = sh.list[i];
      int rank = 0;
#pragma unroll 8
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
      const uint64_t v = rank_key(order_of(to_f(x[c])), first + (uint32_t)c);
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

// One pass over x[0 .. n): the row's sums in all its threads, and what this
// thread saw.
template <typename T, int THREADS>
__device__ __forceinline__ Soft row_pass(const T* x, int n, Seen& seen, RowShared<THREADS>& sh) {
  constexpr int N = Vec<T>::N;
  const int tid = threadIdx.x % THREADS;
  const int packs = n / N, batches = (packs + THREADS * kUnroll - 1) / (THREADS * kUnroll);
  Soft a = {-INFINITY, 0.f, 0.f};
  seen = {-INFINITY, -INFINITY, -INFINITY, -1, -1};
  Batch<T, THREADS> v;
  if (batches) v.load(x, 0, packs);
  float tail = -INFINITY;
  if (packs * N + tid < n) tail = to_f(x[packs * N + tid]);
  for (int b = 0; b < batches; ++b) {
    float f[kUnroll * N];
    v.get(b, packs, f);
    if (b + 1 < batches) v.load(x, b + 1, packs);  // in flight while this batch is added
    float largest = f[0];
#pragma unroll
    for (int k = 1; k < kUnroll * N; ++k) largest = fmaxf(largest, f[k]);
    const bool first = largest > seen.largest, next = largest > seen.second;
    seen.others = fmaxf(seen.others, next ? seen.second : largest);
    seen.second = first ? seen.largest : next ? largest : seen.second;
    seen.batch2 = first ? seen.batch : next ? b : seen.batch2;
    seen.largest = first ? largest : seen.largest;
    seen.batch = first ? b : seen.batch;
    soft_add<kUnroll * N>(a, f, largest);
  }
  soft_add<1>(a, &tail, tail);
  soft_exact(a);
  const float wave = max64(a.m);
  soft_raise(a, wave);
  a.s = lane_sum<64>(a.s);
  a.t = lane_sum<64>(a.t);
  if constexpr (THREADS > 64) {
    const int w = threadIdx.x >> 6, j = threadIdx.x & 15;
    if ((threadIdx.x & 63) == 0) {
      sh.m[w] = a.m;
      sh.s[w] = a.s;
      sh.t[w] = a.t;
    }
    __syncthreads();
    a = {-INFINITY, 0.f, 0.f};
    if (j < THREADS / 64) a = {sh.m[j], sh.s[j], sh.t[j]};
    soft_raise(a, max16(a.m));
    a.s = sum16(a.s);
    a.t = sum16(a.t);
  }
  a.t *= kLn2;
  return a;
}

__device__ __forceinline__ int64_t target_of(const int64_t* t64, const int32_t* t32, int64_t row) {
  return t64 ? t64[row] : (int64_t)t32[row];
}

// Results of a row from its sums (and sh.top), by the row's threads.
template <typename T, int THREADS>
__device__ __forceinline__ void row_write(const TokenLogprobs& a, int64_t row, Soft r, bool has, float given,
                                          RowShared<THREADS>& sh) {
  const int tid = threadIdx.x % THREADS;
  const float logs = logf(r.s);
  const bool empty = r.m == -INFINITY && r.s == 0.f;
  if (tid == 0) {
    a.logp[row] = !has ? 0.f : empty ? -INFINITY : (given - r.m) - logs;
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
__global__ __launch_bounds__(THREADS > 256 ? THREADS : 256, 5) void logprobs_kernel(TokenLogprobs a) {
  constexpr int ROWS = THREADS < 256 ? 256 / THREADS : 1;
  __shared__ RowShared<THREADS> shared[ROWS];
  const int group = __builtin_amdgcn_readfirstlane(threadIdx.x / THREADS);
  RowShared<THREADS>& sh = shared[group];
  const int64_t step = (int64_t)gridDim.x * ROWS;
  for (int64_t row = (int64_t)blockIdx.x * ROWS + group; row < a.N; row += step) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const int64_t t = target_of(a.target64, a.target32, row);
    const bool has = t >= 0 && t < a.V;
    const float given = has ? to_f(x[t]) : 0.f;  // the target's logit, on its way during the pass
    Seen seen;
    const Soft r = row_pass<T, THREADS>(x, a.V, seen, sh);
    if (a.K) row_top<T, THREADS>(x, a.V, 0, a.K, seen, sh);
    row_write<T, THREADS>(a, row, r, has, given, sh);
    row_sync<THREADS>();
  }
}

// Few long rows: a workgroup to each part of a row (a whole number of batches)
// writes the part's sums and its K largest; a wave to each row joins them.
struct PartSums {
  float m, s, t, unused;
};
template <typename T>
__global__ __launch_bounds__(256) void logprobs_part_kernel(TokenLogprobs a, int span) {
  __shared__ RowShared<256> sh;
  const int part = blockIdx.x, parts = gridDim.x;
  const int64_t row = blockIdx.y;
  const int lo = part * span, n = min(span, a.V - lo);
  const T* x = static_cast<const T*>(a.x) + row * a.ldx + lo;
  Seen seen;
  const Soft r = row_pass<T, 256>(x, n, seen, sh);
  const int K = min(a.K, n);
  if (K) row_top<T, 256>(x, n, (uint32_t)lo, K, seen, sh);
  PartSums* sums = static_cast<PartSums*>(a.work);
  uint64_t* keys = reinterpret_cast<uint64_t*>(sums + (int64_t)a.N * parts);
  if (threadIdx.x == 0) sums[row * parts + part] = {r.m, r.s, r.t, 0.f};
  if ((int)threadIdx.x < a.K) keys[(row * parts + part) * a.K + threadIdx.x] = (int)threadIdx.x < K ? sh.top[threadIdx.x] : 0;
}
template <typename T>
__global__ __launch_bounds__(64) void logprobs_join_kernel(TokenLogprobs a, int parts) {
  __shared__ RowShared<64> sh;
  __shared__ uint64_t lists[64 * kTopMax];
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.ldx;
  const PartSums* sums = static_cast<const PartSums*>(a.work);
  const uint64_t* keys = reinterpret_cast<const uint64_t*>(sums + (int64_t)a.N * parts) + row * parts * a.K;
  for (int i = lane; i < parts * a.K; i += 64) lists[i] = keys[i];
  const int64_t t = target_of(a.target64, a.target32, row);
  const bool has = t >= 0 && t < a.V;
  const float given = has ? to_f(x[t]) : 0.f;
  Soft r = {-INFINITY, 0.f, 0.f};
  if (lane < parts) {
    const PartSums p = sums[row * parts + lane];
    r = {p.m, p.s, p.t * kLog2e};
  }
  soft_raise(r, max64(r.m));
  r.s = lane_sum<64>(r.s);
  r.t = lane_sum<64>(r.t) * kLn2;
  row_sync<64>();
  // each part's list is in order, and so are the parts' ids: the first lane
  // with the largest head has the next alternative
  int next = 1;
  uint64_t head = lane < parts && a.K ? lists[lane * a.K] : 0;
  for (int k = 0; k < a.K; ++k) {
    const uint32_t mine = (uint32_t)(head >> 32);  // (0 behind a list's end, below every logit's)
    uint32_t best = mine;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) best = max(best, (uint32_t)__shfl_xor((int)best, o, 64));
    if (lane == __ffsll((unsigned long long)__ballot(mine == best)) - 1) {
      sh.top[k] = head;
      head = next < a.K ? lists[lane * a.K + next] : 0;
      ++next;
    }
  }
  row_sync<64>();
  row_write<T, 64>(a, row, r, has, given, sh);
}
// Elements of a part, or 0 for rows that are not split: only long rows that
// leave most of the chip idle are, into batches of 256 threads, at most 64
// (128000 bf16 logits: one row 10.4 us against 13.5 us, 32 rows 11.6 against
// 14.4, 96 rows 15.5 against 14.8, 128 rows 16.3 against 15.0, 160 rows 18.0
// against 15.3; 128 rows of 200000 fp32 25.8 against 25.7; 32 rows of 65000 bf16
// 10 against 8.5, the join's launch being 2 us).
int part_span(int N, int V, int type) {
  const int batch = 256 * kUnroll * (type == ELEM_F32 ? 4 : 8);
  if (N > kSplitRows || V < kSplitWidth) return 0;
  const int64_t batches = ((int64_t)V + batch - 1) / batch;
  int64_t parts = kSplitGroups / N;
  parts = parts < 64 ? parts : 64;
  parts = parts < batches ? parts : batches;
  return (int)((batches + parts - 1) / parts * batch);
}

// Backward: THREADS threads take a batch of a row; p is recomputed from the
// row's maximum and sum, and a thread whose pack has the target or an
// alternative adds its own term (the alternatives of the batch are a mask of
// the row's, so a pack asks about few).  The gradient is streamed out (2560 x
// 30522 bf16 75 -> 69 us, 8192 x 128000 830 -> 795 us): this launch alone was
// timed, not the products that read the gradient next.
template <typename T, int THREADS>
__global__ __launch_bounds__(256) void logprobs_bwd_kernel(TokenLogprobsBwd a, int parts) {
  constexpr int N = Vec<T>::N, SPAN = THREADS * kUnroll, GROUPS = 256 / THREADS;
  const int64_t items = (int64_t)a.N * parts, step = (int64_t)gridDim.x * GROUPS;
  const int tid = threadIdx.x % THREADS;
  int64_t item = (int64_t)blockIdx.x * GROUPS + __builtin_amdgcn_readfirstlane(threadIdx.x / THREADS);
  for (; item < items; item += step) {
    const int64_t row = item / parts;
    const int part = (int)(item - row * parts);
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    T* dx = static_cast<T*>(a.dx) + row * a.C;
    const int packs = a.V / N;
    Batch<T, THREADS> v;
    if (packs) v.load(x, part, packs);
    const float m = a.stats[3 * row], s = a.stats[3 * row + 1];
    const bool empty = m == -INFINITY && s == 0.f;
    int64_t t = target_of(a.target64, a.target32, row);
    t = t >= 0 && t < a.V && a.d_logp && !empty ? t : -1;
    const float dl = t >= 0 ? a.d_logp[row] : 0.f;
    const float dh = a.d_entropy ? a.d_entropy[row] : 0.f;
    const int lo = part * SPAN * N, hi = part == parts - 1 ? a.V : lo + SPAN * N;
    float all = dl;
    uint32_t here = 0;  // the alternatives of this batch
    if (a.d_top)
      for (int k = 0; k < a.K; ++k) {
        all += a.d_top[row * a.K + k];
        const int64_t j = a.top_ids[row * a.K + k];
        if (j >= lo && j < hi && !empty) here |= 1u << k;
      }
    // dx_j = -p_j (all + dh (log p_j + entropy)) + own terms
    const float inv = 1.f / s, base = empty ? 0.f : m;
    const float ent = a.stats[3 * row + 2] - logf(s);
    auto grad = [&](float z) -> float {
      const float d = z - base, p = __builtin_amdgcn_exp2f(d * kLog2e) * inv;
      float w = all;
      if (dh != 0.f) w = fmaf(dh, fmaxf(d, -1e4f) + ent, w);
      return empty ? 0.f : -p * w;
    };
    // together, the waves' stores run along the row (8192 x 128000 bf16: 795 us against 838 us)
    row_sync<THREADS>();
    // the own terms of n elements from column j
    auto add_own = [&](int j, auto n, float* f) {
      auto add = [&](int64_t id, float d) {
        const int64_t e = id - j;
        if (e >= 0 && e < n) {
#pragma unroll
          for (int k = 0; k < n; ++k) f[k] += k == e ? d : 0.f;
        }
      };
      if (t >= 0) add(t, dl);
      for (uint32_t left = here; left; left &= left - 1) {
        const int k = __ffs(left) - 1;
        add(a.top_ids[row * a.K + k], a.d_top[row * a.K + k]);
      }
    };
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int i = part * SPAN + u * THREADS + tid;
      if (i < packs) {
        float f[N];
#pragma unroll
        for (int k = 0; k < N; ++k) f[k] = grad(to_f(v.v[u].e[k]));
        add_own(i * N, std::integral_constant<int, N>(), f);
        Pack<T, N> o;
#pragma unroll
        for (int k = 0; k < N; ++k) o.e[k] = from_f<T>(f[k]);
        stream_pack<T, N>(dx + (int64_t)i * N, o);
      }
    }
    // what is left of V, and the columns behind it: the last part's
    if (part == parts - 1)
      for (int j = packs * N + tid; j < a.C; j += THREADS) {
        float f = 0.f;
        if (j < a.V) {
          f = grad(to_f(x[j]));
          add_own(j, std::integral_constant<int, 1>(), &f);
        }
        dx[j] = from_f<T>(f);
      }
  }
}

template <typename T>
void fwd_typed(const TokenLogprobs& a, hipStream_t s) {
  const int64_t cap = 1 << 20;
  if (const int span = part_span(a.N, a.V, a.type)) {
    const int parts = (a.V + span - 1) / span;
    logprobs_part_kernel<T><<<dim3(parts, a.N), 256, 0, s>>>(a, span);
    logprobs_join_kernel<T><<<a.N, 64, 0, s>>>(a, parts);
    return;
  }
  // Threads to a row, both sides measured with 5 alternatives (4160 rows where
  // none are named).  A wave where rows are short, up to 16384 if there are
  // enough to fill the chip (fp16 2500: 14.4 us against 25.1 with 256, 8000:
  // 21.5 against 25.5, 16000: 37.8 against 37.7, 30522: 62 against 56; fp32
  // 2500: 13.9 against 18.2, 8000: 32.4 against 31.2, 16000: 58 against 52;
  // 1024 x 2500 fp32: 7.2 against 7.9 the other way).  Else 256 up to 64 KB
  // (fp16 30522: 56 against 75 with 512; fp32 16000: 130 rows 7.4 against 7.1)
  // and 512 above (2048 x 30522 fp32: 47.8 against 50.8, 18000: 59.0 against
  // 56.5, fp16 40000: 88 against 66 the other way) and for long rows that do not
  // fill the chip (one row of 30522 bf16: 7.8 against 8.4; 100 x 18000 fp32: 7.4
  // against 7.9).  The limits were set on bf16: fp32 from 8000 and rows of 64
  // to 80 KB would be faster with 256.
  const int64_t few = ((int64_t)a.N + 3) / 4;
  if (a.V <= 2048 || (a.V <= 16384 && a.N >= 2048))
    logprobs_kernel<T, 64><<<(unsigned)(few < cap ? few : cap), 256, 0, s>>>(a);
  else if ((int64_t)a.V * (int64_t)sizeof(T) <= 65536 && (a.V <= 16384 || a.N > 128))
    logprobs_kernel<T, 256><<<(unsigned)(a.N < cap ? a.N : cap), 256, 0, s>>>(a);
  else
    logprobs_kernel<T, 512><<<(unsigned)(a.N < cap ? a.N : cap), 512, 0, s>>>(a);
}
template <typename T>
void bwd_typed(const TokenLogprobsBwd& a, hipStream_t s) {
  // a wave to a row that is one batch of it (4099 x 1001 bf16: 7.4 us against 15 us), else 256 threads
  const int packs = a.V / Vec<T>::N, cap = 1 << 20;
  if (packs <= 64 * kUnroll) {
    const int64_t want = ((int64_t)a.N + 3) / 4;
    logprobs_bwd_kernel<T, 64><<<(unsigned)(want < cap ? want : cap), 256, 0, s>>>(a, 1);
    return;
  }
  const int span = 256 * kUnroll, parts = (packs + span - 1) / span;
  const int64_t items = (int64_t)a.N * parts;
  logprobs_bwd_kernel<T, 256><<<(unsigned)(items < cap ? items : cap), 256, 0, s>>>(a, parts);
}

}  // namespace

size_t token_logprobs_workspace(int N, int V, int K, int type) {
  const int span = part_span(N, V, type);
  return span ? (size_t)N * ((V + span - 1) / span) * (sizeof(PartSums) + (size_t)K * sizeof(uint64_t)) : 0;
}

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
