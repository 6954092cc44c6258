// LayerNorm of any width, type and row stride:
//   y = (x - mean) rstd gamma + beta,  rstd = 1 / sqrt(mean((x - mean)^2) + eps)
// and backward, with xh = (x - mean) rstd, u = dy gamma:
//   dx = rstd (u - mean(u) - xh mean(u xh)),  dgamma = sum dy xh,  dbeta = sum dy.
//
// Both directions are bound by memory: forward reads x and writes y, backward
// reads x and dy and writes dx, each once.  LANES lanes hold a row in
// registers (16 lanes for narrow rows, a wave, 256 or 1024 threads), VPL packs
// of 16 or 8 bytes each, so mean and variance are two passes over registers (no
// cancellation of E[x^2] - mean^2); the second also sums x - mean, which is
// what the fp32 mean is off by (row_rest).  Workgroups stay for several rows,
// the next row's loads in flight.  The weights' gradients are sums over all
// rows: each workgroup keeps the partial sums of its columns in registers over
// its rows, writes one row of partials, and a second launch adds the
// workgroups' rows in a fixed order, so results repeat bit for bit (no
// atomics).  All sums are fp32.
//
// Measured, calls among others over three sets of inputs in turn, fp32 weights
// (copies of 1 GiB: 4.7 to 5.1 TB/s; of 64 MiB: 5.1 TB/s over three pairs of
// buffers in turn, 6.9 TB/s over one pair, which stays cached):
//   16384 x 768    bf16  forward  10.7 us, 4.7 TB/s  backward  16.8 us, 4.5 TB/s
//   16384 x 4096   bf16  forward  57 us,   4.7 TB/s  backward  83 us,   4.8 TB/s
//   24576 x 5120   fp32  forward  199 us,  5.1 TB/s  backward  279 us,  5.4 TB/s
//   4099 x 1001    fp16  forward  6.1 us,  2.7 TB/s  backward  12.3 us, 2.0 TB/s
//   4096 x 16384   fp32  forward  97 us,   5.6 TB/s  backward  191 us,  4.2 TB/s
//   2048 x 40000   bf16  forward  105 us,  3.1 TB/s  backward  240 us,  2.1 TB/s
//   1 x 768        fp32  forward  1.8 us on the GPU, 5.2 us a call
// Weights of the input's type: 16384 x 768 bf16 11.8 and 17.0 us.
#include "kernels/elem.h"
#include "kernels/lm.h"

#include <type_traits>

namespace mfl {
namespace {

// Which of a workgroup's rows a thread works on: a scalar where a wave has one row.
template <int LANES>
__device__ __forceinline__ int row_group() {
  const int g = threadIdx.x / LANES;
  if constexpr (LANES >= 64) return __builtin_amdgcn_readfirstlane(g);
  return g;
}

// Sums of a and b over the LANES threads of a row; with more than one wave
// through LDS (`buf` 2 x 16 floats, two of them used in turn).
template <int LANES>
__device__ __forceinline__ void row_sum2(float& a, float& b, float* buf) {
  constexpr int L = LANES < 64 ? LANES : 64;
  a = lane_sum<L>(a);
  b = lane_sum<L>(b);
  if constexpr (LANES > 64) {
    constexpr int W = LANES / 64;
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
      buf[w] = a;
      buf[16 + w] = b;
    }
    __syncthreads();
    if constexpr (W == 16) {
      a = sum16(buf[threadIdx.x & 15]);
      b = sum16(buf[16 + (threadIdx.x & 15)]);
    } else {
      a = b = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        a += buf[i];
        b += buf[16 + i];
      }
    }
  }
}

// The packs of N columns that a lane has of every row: pack i starts at
// column c[i]; one that would end behind the row (or lie there) is moved back
// to end with it, and its first skip[i] elements, another lane's, count for
// nothing.  So every load is whole and in the row, whatever its width (>= N).
// EXACT: the row is as wide as the packs, nothing is skipped.
template <int LANES, int VPL, int N, bool EXACT>
struct Columns {
  int c[VPL], skip[VPL];
  // shapes hold a row in no more packs than needed: the first ones are whole
  static constexpr bool whole(int i) { return EXACT || (VPL > 1 && i < VPL / 2); }
  __device__ __forceinline__ Columns(int lane, int H) {
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int at = (i * LANES + lane) * N;
      c[i] = whole(i) || at <= H - N ? at : H - N;
      skip[i] = at - c[i];
    }
  }
  __device__ __forceinline__ bool has(int i, int k) const { return whole(i) || k >= skip[i]; }
  __device__ __forceinline__ bool full(int i) const { return whole(i) || skip[i] == 0; }
};
template <typename T, int LANES, int VPL, int N, bool EXACT>
__device__ __forceinline__ void load_packs(const T* row, const Columns<LANES, VPL, N, EXACT>& at, Pack<T, N> (&v)[VPL]) {
#pragma unroll
  for (int i = 0; i < VPL; ++i) v[i] = load_pack<T, N>(row + at.c[i]);
}
template <typename P, int LANES, int VPL, int N, bool EXACT>
__device__ __forceinline__ void load_weights(const void* p, const Columns<LANES, VPL, N, EXACT>& at, float none,
                                             float (&w)[VPL][N]) {
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    Pack<P, N> v;
    if (p) v = load_pack<P, N>(static_cast<const P*>(p) + at.c[i]);
#pragma unroll
    for (int k = 0; k < N; ++k) w[i][k] = p ? to_f(v.e[k]) : none;
  }
}

template <typename T, int LANES, int VPL, int N, bool EXACT>
__device__ __forceinline__ void store_packs(T* row, const Columns<LANES, VPL, N, EXACT>& at, const float (&f)[VPL][N]) {
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    Pack<T, N> o;
#pragma unroll
    for (int k = 0; k < N; ++k) o.e[k] = from_f<T>(f[i][k]);
    if (at.full(i)) {
      store_pack<T, N>(row + at.c[i], o);
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (at.has(i, k)) row[at.c[i] + k] = o.e[k];
    }
  }
}

// 1 / sqrt(variance + eps) from the mean square of x - mean and the mean of
// x - mean, `rest`, which is what the fp32 mean is off by.
__device__ __forceinline__ float row_rstd(float square, float rest, float eps) {
  const float var = square - rest * rest;
  return 1.f / sqrtf((var < 0.f ? 0.f : var) + eps);
}
// The correction of the mean.  Rows far from zero need it, and there x - mean
// is exact; near zero the differences are rounded, alike for x of few bits, and
// the sum itself is nearer.
__device__ __forceinline__ float row_rest(float mean, float rest, float rstd) {
  return fabsf(mean) * rstd > 1.f ? rest : 0.f;
}

// A workgroup's rows: its BLOCK / LANES groups take rows in turn, the next
// row's loads in flight while this one is worked on.
template <typename T, typename P, int BLOCK, int LANES, int VPL, int N, bool EXACT>
__global__ __launch_bounds__(BLOCK) void ln_fwd_kernel(LayerNormFwd a) {
  constexpr int ROWS = BLOCK / LANES;
  static_assert(LANES <= 64 || ROWS == 1, "a barrier belongs to one row");
  __shared__ float lds[2][32];
  const int lane = threadIdx.x % LANES;
  const Columns<LANES, VPL, N, EXACT> at(lane, a.H);
  const float width = (float)a.H;
  const int64_t step = (int64_t)gridDim.x * ROWS;
  int64_t row = (int64_t)blockIdx.x * ROWS + row_group<LANES>();
  Pack<T, N> next[VPL];
  if (row < a.M) load_packs<T>(static_cast<const T*>(a.x) + row * a.ldx, at, next);
  float g[VPL][N], b[VPL][N];
  load_weights<P>(a.gamma, at, 1.f, g);
  load_weights<P>(a.beta, at, 0.f, b);
  for (; row < a.M; row += step) {
    float v[VPL][N];
    float s = 0.f, zero = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i)
#pragma unroll
      for (int k = 0; k < N; ++k) {
        v[i][k] = at.has(i, k) ? to_f(next[i].e[k]) : 0.f;
        s += v[i][k];
      }
    if (row + step < a.M) load_packs<T>(static_cast<const T*>(a.x) + (row + step) * a.ldx, at, next);
    row_sum2<LANES>(s, zero, lds[0]);
    float mean = s / width;
    float q = 0.f, rest = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i)
#pragma unroll
      for (int k = 0; k < N; ++k) {
        v[i][k] = at.has(i, k) ? v[i][k] - mean : 0.f;
        q = fmaf(v[i][k], v[i][k], q);
        rest += v[i][k];
      }
    row_sum2<LANES>(q, rest, lds[1]);
    rest /= width;
    const float rstd = row_rstd(q / width, rest, a.eps);
    rest = row_rest(mean, rest, rstd);
    mean += rest;
    if (lane == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
    const float shift = -rest * rstd;
#pragma unroll
    for (int i = 0; i < VPL; ++i)
#pragma unroll
      for (int k = 0; k < N; ++k) v[i][k] = fmaf(fmaf(v[i][k], rstd, shift), g[i][k], b[i][k]);
    store_packs<T>(static_cast<T*>(a.y) + row * a.H, at, v);
  }
}

// Rows wider than registers hold: f(c, n, elements) for the n = N elements from
// column c of each whole pack of this thread, then for single ones behind them.
template <int N, typename F>
__device__ __forceinline__ void each_pack(int H, F&& f) {
  const int packs = H / N;
  for (int i = threadIdx.x; i < packs; i += 1024) f(i * N, std::integral_constant<int, N>());
  if (packs * N + (int)threadIdx.x < H) f(packs * N + (int)threadIdx.x, std::integral_constant<int, 1>());
}

// 1024 threads read such a row three times (the later two from L2).
template <typename T, typename P>
__global__ __launch_bounds__(1024) void ln_fwd_long_kernel(LayerNormFwd a) {
  constexpr int N = Vec<T>::N;
  __shared__ float lds[2][32];
  const float width = (float)a.H;
  for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    float s = 0.f, zero = 0.f;
    each_pack<N>(a.H, [&](int c, auto n) {
      const auto v = load_pack<T, n>(x + c);
#pragma unroll
      for (int k = 0; k < n; ++k) s += to_f(v.e[k]);
    });
    row_sum2<1024>(s, zero, lds[0]);
    const float mean = s / width;
    float q = 0.f, rest = 0.f;
    each_pack<N>(a.H, [&](int c, auto n) {
      const auto v = load_pack<T, n>(x + c);
#pragma unroll
      for (int k = 0; k < n; ++k) {
        const float d = to_f(v.e[k]) - mean;
        q = fmaf(d, d, q);
        rest += d;
      }
    });
    row_sum2<1024>(q, rest, lds[1]);
    rest /= width;
    const float rstd = row_rstd(q / width, rest, a.eps);
    rest = row_rest(mean, rest, rstd);
    if (threadIdx.x == 0) {
      a.mean[row] = mean + rest;
      a.rstd[row] = rstd;
    }
    T* y = static_cast<T*>(a.y) + row * a.H;
    each_pack<N>(a.H, [&](int c, auto n) {
      const auto v = load_pack<T, n>(x + c);
      Pack<P, n> g, b;
      if (a.gamma) g = load_pack<P, n>(static_cast<const P*>(a.gamma) + c);
      if (a.beta) b = load_pack<P, n>(static_cast<const P*>(a.beta) + c);
      Pack<T, n> o;
#pragma unroll
      for (int k = 0; k < n; ++k)
        o.e[k] = from_f<T>((to_f(v.e[k]) - mean - rest) * rstd * (a.gamma ? to_f(g.e[k]) : 1.f) +
                           (a.beta ? to_f(b.e[k]) : 0.f));
      store_pack<T, n>(y + c, o);
    });
  }
}

template <typename T, typename P, int BLOCK, int LANES, int VPL, int N, bool EXACT>
__global__ __launch_bounds__(BLOCK) void ln_bwd_kernel(LayerNormBwd a) {
  constexpr int ROWS = BLOCK / LANES;
  constexpr int WIDE = LANES * VPL * N;  // columns the registers of a row's lanes hold
  static_assert(LANES <= 64 || ROWS == 1, "a barrier belongs to one row");
  __shared__ float lds[2][32];
  __shared__ float sums[ROWS > 1 ? ROWS * WIDE : 1];
  const int lane = threadIdx.x % LANES, grp = row_group<LANES>();
  const Columns<LANES, VPL, N, EXACT> at(lane, a.H);
  const float inv = 1.f / (float)a.H;
  const int64_t step = (int64_t)gridDim.x * ROWS;
  int64_t row = (int64_t)blockIdx.x * ROWS + grp;
  Pack<T, N> nx[VPL], nd[VPL];
  float mean = 0.f, rstd = 0.f;
  if (row < a.M) {
    load_packs<T>(static_cast<const T*>(a.x) + row * a.ldx, at, nx);
    load_packs<T>(static_cast<const T*>(a.dy) + row * a.lddy, at, nd);
    mean = a.mean[row];
    rstd = a.rstd[row];
  }
  float g[VPL][N], dg[VPL][N], db[VPL][N];
  load_weights<P>(a.gamma, at, 1.f, g);
#pragma unroll
  for (int i = 0; i < VPL; ++i)
#pragma unroll
    for (int k = 0; k < N; ++k) dg[i][k] = db[i][k] = 0.f;
  for (int turn = 0; row < a.M; row += step, turn ^= 1) {
    float xh[VPL][N], u[VPL][N];
#pragma unroll
    for (int i = 0; i < VPL; ++i)
#pragma unroll
      for (int k = 0; k < N; ++k) {
        xh[i][k] = (to_f(nx[i].e[k]) - mean) * rstd;
        u[i][k] = to_f(nd[i].e[k]);
      }
    const float scale = rstd;
    if (row + step < a.M) {
      load_packs<T>(static_cast<const T*>(a.x) + (row + step) * a.ldx, at, nx);
      load_packs<T>(static_cast<const T*>(a.dy) + (row + step) * a.lddy, at, nd);
      mean = a.mean[row + step];
      rstd = a.rstd[row + step];
    }
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i)
#pragma unroll
      for (int k = 0; k < N; ++k) {
        dg[i][k] += u[i][k] * xh[i][k];
        db[i][k] += u[i][k];
        u[i][k] = at.has(i, k) ? u[i][k] * g[i][k] : 0.f;  // another lane's element adds nothing
        s1 += u[i][k];
        s2 += u[i][k] * xh[i][k];
      }
    row_sum2<LANES>(s1, s2, lds[turn]);
    s1 *= inv;
    s2 *= inv;
#pragma unroll
    for (int i = 0; i < VPL; ++i)
#pragma unroll
      for (int k = 0; k < N; ++k) u[i][k] = scale * (u[i][k] - s1 - xh[i][k] * s2);
    store_packs<T>(static_cast<T*>(a.dx) + row * a.H, at, u);
  }
  if (!a.dgamma) return;
  // the workgroup's sums: dgamma, then dbeta, the groups' added by column; a
  // row of partials, or the results themselves if it is alone
  for (int which = 0; which < 2; ++which) {
    const float(&mine)[VPL][N] = which ? db : dg;
    float* out = a.part + ((int64_t)blockIdx.x * 2 + which) * a.H;
    P* result = static_cast<P*>(which ? a.dbeta : a.dgamma);
    if constexpr (ROWS == 1) {
      if (a.part) store_packs<float>(out, at, mine);
      else store_packs<P>(result, at, mine);
    } else {
      if (which) __syncthreads();
      store_packs<float>(sums + grp * WIDE, at, mine);
      __syncthreads();
      for (int c = threadIdx.x; c < a.H; c += BLOCK) {
        float s = 0.f;
#pragma unroll 16
        for (int r = 0; r < ROWS; ++r) s += sums[r * WIDE + c];
        if (a.part) out[c] = s;
        else result[c] = from_f<P>(s);
      }
    }
  }
}

// Rows wider than registers hold: a workgroup takes a row at a time for dx
// (read twice), and the weights' gradients are column sums in launches of
// their own.
template <typename T, typename P>
__global__ __launch_bounds__(1024) void ln_bwd_long_kernel(LayerNormBwd a) {
  constexpr int N = Vec<T>::N;
  __shared__ float lds[2][32];
  const float inv = 1.f / (float)a.H;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x, turn ^= 1) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* dy = static_cast<const T*>(a.dy) + row * a.lddy;
    T* dx = static_cast<T*>(a.dx) + row * a.H;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s1 = 0.f, s2 = 0.f;
    auto pass = [&](auto write) {
      each_pack<N>(a.H, [&](int c, auto n) {
        const auto v = load_pack<T, n>(x + c);
        const auto d = load_pack<T, n>(dy + c);
        Pack<P, n> g;
        if (a.gamma) g = load_pack<P, n>(static_cast<const P*>(a.gamma) + c);
        Pack<T, n> o;
#pragma unroll
        for (int k = 0; k < n; ++k) {
          const float xh = (to_f(v.e[k]) - mean) * rstd, u = to_f(d.e[k]) * (a.gamma ? to_f(g.e[k]) : 1.f);
          if constexpr (write) {
            o.e[k] = from_f<T>(rstd * (u - s1 - xh * s2));
          } else {
            s1 += u;
            s2 += u * xh;
          }
        }
        if constexpr (write) store_pack<T, n>(dx + c, o);
      });
    };
    pass(std::false_type());
    row_sum2<1024>(s1, s2, lds[turn]);
    s1 *= inv;
    s2 *= inv;
    pass(std::true_type());
  }
}
// partials of 256 columns (blockIdx.x) over every gridDim.y-th row, four rows' loads in flight
template <typename T>
__global__ __launch_bounds__(256) void ln_colsum_long_kernel(LayerNormBwd a) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.H) return;
  float dg = 0.f, db = 0.f;
  for (int64_t row = blockIdx.y; row < a.M; row += 4 * (int64_t)gridDim.y) {
    float d[4], x[4], mean[4], rstd[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t at = row + j * (int64_t)gridDim.y, r = at < a.M ? at : a.M - 1;
      d[j] = to_f(static_cast<const T*>(a.dy)[r * a.lddy + c]);
      x[j] = to_f(static_cast<const T*>(a.x)[r * a.ldx + c]);
      mean[j] = a.mean[r];
      rstd[j] = a.rstd[r];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (row + j * (int64_t)gridDim.y >= a.M) break;
      dg += d[j] * ((x[j] - mean[j]) * rstd[j]);
      db += d[j];
    }
  }
  a.part[((int64_t)blockIdx.y * 2) * a.H + c] = dg;
  a.part[((int64_t)blockIdx.y * 2 + 1) * a.H + c] = db;
}

// dgamma (blockIdx.y = 0) / dbeta (1): the G rows of partials added in a fixed
// order, 32 columns (a 128-byte line) and 32 row lanes to a workgroup, eight
// loads of a lane in flight.
template <typename P>
__global__ __launch_bounds__(1024) void ln_wgrad_kernel(const float* __restrict__ part, P* dgamma, P* dbeta, int G,
                                                        int H) {
  __shared__ float lds[32][33];
  const int col = threadIdx.x & 31, r = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + col, which = blockIdx.y;
  float s = 0.f;
  if (c < H)
    for (int i = r; i < G; i += 8 * 32) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = part[((int64_t)min(i + 32 * j, G - 1) * 2 + which) * H + c];
#pragma unroll
      for (int j = 0; j < 8; ++j) s += i + 32 * j < G ? v[j] : 0.f;
    }
  lds[r][col] = s;
  __syncthreads();
  if (r == 0 && c < H) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += lds[i][col];
    P* out = which ? dbeta : dgamma;
    out[c] = from_f<P>(s);
  }
}

// Lanes and packs of a row, elements of a pack (16 bytes, or 8 where that
// leaves fewer lanes idle), exactness: the fewest lanes that hold the row in
// about 16 elements each.  A backward thread of 1024 has 128 registers, and with
// the weights and their sums some shapes need more: fp32 above 8192 columns
// spills 41 to 46 (4096 x 12288: 186 us, 3.2 TB/s; 4096 x 8192, which does not
// spill: 82 us, 4.9 TB/s), 16-bit rows of 8193 to 16383 columns 6 to 12 (8192 x
// 16000 bf16: 190 us, 4.1 TB/s; 16384 columns 164 us, 4.9), and with 16-bit
// weights 16384 columns 2 and 769 to 1023 columns 4 to 9 (16384 x 900 bf16:
// 26.5 us against 23.2 with fp32 weights).  Rows of fewer elements than a pack
// take one element a lane.
template <typename T, bool BACK, typename F>
bool with_shape(int H, F&& f) {
  constexpr int N = Vec<T>::N;
#define MFL_LN_EXACT(L_, V_, N_)                                                                           \
  if (H == L_ * V_ * N_)                                                                                   \
    return f(std::integral_constant<int, L_>(), std::integral_constant<int, V_>(),                         \
             std::integral_constant<int, N_>(), std::true_type()), true;
#define MFL_LN_UP_TO(L_, V_, N_)                                                                           \
  if (H <= L_ * V_ * N_)                                                                                   \
    return f(std::integral_constant<int, L_>(), std::integral_constant<int, V_>(),                         \
             std::integral_constant<int, N_>(), std::false_type()), true;
#define MFL_LN(L_, V_, N_) MFL_LN_EXACT(L_, V_, N_) MFL_LN_UP_TO(L_, V_, N_)
  if (H < N) {
    MFL_LN_UP_TO(16, 1, 1)
  }
  MFL_LN(16, 1, N)
  if constexpr (N == 4 || !BACK) {
    MFL_LN(16, 2, N)
  } else {
    MFL_LN_EXACT(16, 2, N)  // (masks are registers too many)
    MFL_LN_UP_TO(64, 1, 4)
  }
  if constexpr (N == 4 && !BACK) {
    MFL_LN(16, 4, N)
  }
  if constexpr (N == 8 || BACK) {
    MFL_LN(64, 1, N)
  }
  if constexpr (N == 8) {
    MFL_LN(64, 3, 4)
  }
  MFL_LN(64, 2, N)
  if constexpr (N == 4) {
    MFL_LN(64, 3, N)
  }
  if constexpr (N == 4 && !BACK) {  // (backward: 32 registers of loads ahead are too many)
    MFL_LN(64, 4, N)
  }
  if constexpr (N == 8 || BACK) {
    MFL_LN(256, 1, N)
  }
  MFL_LN(256, 2, N)
  if constexpr (N == 4) {
    MFL_LN(256, 4, N)
  }
  if constexpr (N == 8 && !BACK) {
    MFL_LN(256, 3, N)
  }
  if constexpr (N == 8) {
    MFL_LN(1024, 1, N)
  }
  MFL_LN(1024, 2, N)
  if constexpr (N == 4) {
    MFL_LN(1024, 4, N)
  }
#undef MFL_LN
#undef MFL_LN_UP_TO
#undef MFL_LN_EXACT
  return false;
}
constexpr int fwd_block(int lanes) { return lanes > 256 ? lanes : 256; }
constexpr int bwd_block(int lanes) { return lanes == 256 ? 256 : 1024; }

template <typename T, typename P>
void fwd_typed(const LayerNormFwd& a, hipStream_t s) {
  const bool done = with_shape<T, false>(a.H, [&](auto L, auto V, auto N, auto exact) {
    constexpr int BLOCK = fwd_block(L), ROWS = BLOCK / L;
    const int64_t want = ((int64_t)a.M + ROWS - 1) / ROWS, cap = 2048 * 256 / BLOCK;
    ln_fwd_kernel<T, P, BLOCK, L, V, N, exact><<<(unsigned)(want < cap ? want : cap), BLOCK, 0, s>>>(a);
  });
  if (!done) ln_fwd_long_kernel<T, P><<<(unsigned)(a.M < (1 << 20) ? a.M : (1 << 20)), 1024, 0, s>>>(a);
}

// Workgroups of the backward: what the chip holds at a time, fewer for few
// rows, and one where its groups have at most four rows each, which spares the
// second launch (a call on one row of 768 fp32: 4.5 us against 7.4; 4 rows of
// 1024: 4.7 against 7.5; 4 rows of 8192: 6.9 against 7.4; 64 rows of 768, four to
// a group: 7.9 against 7.2 to 8.5).  Rows wider than registers hold: the parts
// that the columns' sums are split into.
template <typename T>
int bwd_blocks(int M, int H) {
  int G = M < 64 ? M : 64;
  with_shape<T, true>(H, [&](auto L, auto, auto, auto) {
    constexpr int BLOCK = bwd_block(L), ROWS = BLOCK / L;
    const int want = (int)(((int64_t)M + ROWS - 1) / ROWS), cap = BLOCK == 1024 ? 256 : 512;
    G = want <= 4 ? 1 : want < cap ? want : cap;
  });
  return G;
}

template <typename T, typename P>
void bwd_typed(const LayerNormBwd& a, hipStream_t s) {
  const int G = bwd_blocks<T>(a.M, a.H);
  const bool done = with_shape<T, true>(a.H, [&](auto L, auto V, auto N, auto exact) {
    constexpr int BLOCK = bwd_block(L);
    ln_bwd_kernel<T, P, BLOCK, L, V, N, exact><<<G, BLOCK, 0, s>>>(a);
  });
  if (!done) {
    ln_bwd_long_kernel<T, P><<<(unsigned)(a.M < (1 << 20) ? a.M : (1 << 20)), 1024, 0, s>>>(a);
    if (a.dgamma) ln_colsum_long_kernel<T><<<dim3((a.H + 255) / 256, G), 256, 0, s>>>(a);
  }
  if (a.part)
    ln_wgrad_kernel<P><<<dim3((a.H + 31) / 32, 2), 1024, 0, s>>>(a.part, static_cast<P*>(a.dgamma),
                                                                static_cast<P*>(a.dbeta), G, a.H);
}

}  // namespace

int layer_norm_bwd_parts(int M, int H, int type) {
  const int G = type == ELEM_F32 ? bwd_blocks<float>(M, H) : bwd_blocks<BF16>(M, H);
  const bool held = type == ELEM_F32 ? with_shape<float, true>(H, [](auto...) {})
                                     : with_shape<BF16, true>(H, [](auto...) {});
  return held && G == 1 ? 0 : G;
}

// Parameters are fp32 or of the input's own type.
#define MFL_LN_TYPES(FN_)                                                        \
  switch (a.type) {                                                              \
    case ELEM_F32: FN_<float, float>(a, s); break;                               \
    case ELEM_BF16:                                                              \
      if (a.param_type == ELEM_F32) FN_<BF16, float>(a, s);                      \
      else FN_<BF16, BF16>(a, s);                                                \
      break;                                                                     \
    default:                                                                     \
      if (a.param_type == ELEM_F32) FN_<F16, float>(a, s);                       \
      else FN_<F16, F16>(a, s);                                                  \
  }
void launch_layer_norm_fwd(const LayerNormFwd& a, hipStream_t s) { MFL_LN_TYPES(fwd_typed) }
void launch_layer_norm_bwd(const LayerNormBwd& a, hipStream_t s) { MFL_LN_TYPES(bwd_typed) }
#undef MFL_LN_TYPES

}  // namespace mfl
