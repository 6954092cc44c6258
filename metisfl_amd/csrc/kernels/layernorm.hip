// LayerNorm of any width, type and row stride:
//   y = (x - mean) rstd gamma + beta,  rstd = 1 / sqrt(mean((x - mean)^2) + eps)
// and backward, with xh = (x - mean) rstd, u = dy gamma:
//   dx = rstd (u - mean(u) - xh mean(u xh)),  dgamma = sum dy xh,  dbeta = sum dy.
//
// Both directions are bound by memory: forward reads x and writes y, backward
// reads x and dy and writes dx, each once.  LANES lanes hold a row in
// registers (16 lanes for narrow rows, a wave, 256 or 1024 threads), VPL
// packs of 16 bytes each, so mean and variance are two passes over registers
// (no cancellation of E[x^2] - mean^2); the second also sums x - mean and what
// these differences were rounded by (x of few bits round alike, so it would
// not average out), which is what the fp32 mean is off by, and corrects it: a
// constant row gives 0.  The weights' gradients are sums over
// all rows: each workgroup keeps the partial sums of its columns in registers
// over its rows, writes one row of partials, and a second launch adds the
// workgroups' rows in a fixed order, so results repeat bit for bit (no
// atomics).  All sums are fp32.
#include "kernels/elem.h"
#include "kernels/lm.h"

namespace mfl {
namespace {

template <int LANES>
constexpr int block_of() {
  return LANES > 256 ? LANES : 256;
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
    a = b = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      a += buf[i];
      b += buf[16 + i];
    }
  }
}

template <typename T, typename P, int LANES, int VPL>
__global__ __launch_bounds__(block_of<LANES>()) void ln_fwd_kernel(LayerNormFwd a) {
  constexpr int N = Vec<T>::N, ROWS = block_of<LANES>() / LANES;
  __shared__ float lds[2][32];
  const int lane = threadIdx.x % LANES, grp = threadIdx.x / LANES;
  const float width = (float)a.H;
  for (int64_t row = (int64_t)blockIdx.x * ROWS + grp; row < a.M; row += (int64_t)gridDim.x * ROWS) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    float v[VPL][N];
    float s = 0.f, zero = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      load_row<T, N>(x, (i * LANES + lane) * N, a.H, 0.f, v[i]);
#pragma unroll
      for (int k = 0; k < N; ++k) s += v[i][k];
    }
    row_sum2<LANES>(s, zero, lds[0]);
    const float mean = s / width;
    float q = 0.f, rest = 0.f, low = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i)
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const bool in = (i * LANES + lane) * N + k < a.H;
        const float x0 = v[i][k], d = in ? x0 - mean : 0.f;
        low += in ? (x0 - d) - mean : 0.f;  // what the difference was rounded by
        q += d * d;
        rest += d;
        v[i][k] = d;
      }
    rest += low;
    row_sum2<LANES>(q, rest, lds[1]);
    rest /= width;
    const float var = q / width - rest * rest, rstd = 1.f / sqrtf((var < 0.f ? 0.f : var) + a.eps);
    if (lane == 0) {
      a.mean[row] = mean + rest;
      a.rstd[row] = rstd;
    }
    T* y = static_cast<T*>(a.y) + row * a.H;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int c = (i * LANES + lane) * N;
      float g[N], b[N];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        g[k] = 1.f;
        b[k] = 0.f;
      }
      if (a.gamma) load_row<P, N>(static_cast<const P*>(a.gamma), c, a.H, 0.f, g);
      if (a.beta) load_row<P, N>(static_cast<const P*>(a.beta), c, a.H, 0.f, b);
#pragma unroll
      for (int k = 0; k < N; ++k) v[i][k] = (v[i][k] - rest) * rstd * g[k] + b[k];
      store_row<T, N>(y, c, a.H, v[i]);
    }
  }
}

// Rows wider than registers hold: 1024 threads read the row three times (the
// later two from L2).
template <typename T, typename P>
__global__ __launch_bounds__(1024) void ln_fwd_long_kernel(LayerNormFwd a) {
  __shared__ float lds[2][32];
  const float width = (float)a.H;
  for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    float s = 0.f, zero = 0.f;
    for (int c = threadIdx.x; c < a.H; c += 1024) s += to_f(x[c]);
    row_sum2<1024>(s, zero, lds[0]);
    const float mean = s / width;
    float q = 0.f, rest = 0.f, low = 0.f;
    for (int c = threadIdx.x; c < a.H; c += 1024) {
      const float x0 = to_f(x[c]), d = x0 - mean;
      low += (x0 - d) - mean;
      q += d * d;
      rest += d;
    }
    rest += low;
    row_sum2<1024>(q, rest, lds[1]);
    rest /= width;
    const float var = q / width - rest * rest, rstd = 1.f / sqrtf((var < 0.f ? 0.f : var) + a.eps);
    if (threadIdx.x == 0) {
      a.mean[row] = mean + rest;
      a.rstd[row] = rstd;
    }
    T* y = static_cast<T*>(a.y) + row * a.H;
    for (int c = threadIdx.x; c < a.H; c += 1024) {
      const float g = a.gamma ? to_f(static_cast<const P*>(a.gamma)[c]) : 1.f;
      const float b = a.beta ? to_f(static_cast<const P*>(a.beta)[c]) : 0.f;
      y[c] = from_f<T>((to_f(x[c]) - mean - rest) * rstd * g + b);
    }
  }
}

template <typename T, typename P, int LANES, int VPL>
__global__ __launch_bounds__(block_of<LANES>()) void ln_bwd_kernel(LayerNormBwd a) {
  constexpr int N = Vec<T>::N, ROWS = block_of<LANES>() / LANES;
  constexpr int WIDE = LANES * VPL * N;  // columns the registers of a row's lanes hold
  __shared__ float lds[2][32];
  __shared__ float sums[ROWS > 1 ? ROWS * WIDE : 1];
  const int lane = threadIdx.x % LANES, grp = threadIdx.x / LANES;
  const float inv = 1.f / (float)a.H;
  float g[VPL][N], dg[VPL][N], db[VPL][N];
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      g[i][k] = 1.f;
      dg[i][k] = db[i][k] = 0.f;
    }
    if (a.gamma) load_row<P, N>(static_cast<const P*>(a.gamma), (i * LANES + lane) * N, a.H, 0.f, g[i]);
  }
  int turn = 0;
  for (int64_t row = (int64_t)blockIdx.x * ROWS + grp; row < a.M; row += (int64_t)gridDim.x * ROWS, turn ^= 1) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* dy = static_cast<const T*>(a.dy) + row * a.lddy;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float xh[VPL][N], u[VPL][N];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int c = (i * LANES + lane) * N;
      load_row<T, N>(x, c, a.H, mean, xh[i]);
      load_row<T, N>(dy, c, a.H, 0.f, u[i]);
    }
#pragma unroll
    for (int i = 0; i < VPL; ++i)
#pragma unroll
      for (int k = 0; k < N; ++k) {
        xh[i][k] = (xh[i][k] - mean) * rstd;
        dg[i][k] += u[i][k] * xh[i][k];
        db[i][k] += u[i][k];
        u[i][k] *= g[i][k];
        s1 += u[i][k];
        s2 += u[i][k] * xh[i][k];
      }
    row_sum2<LANES>(s1, s2, lds[turn]);
    s1 *= inv;
    s2 *= inv;
    T* dx = static_cast<T*>(a.dx) + row * a.H;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
#pragma unroll
      for (int k = 0; k < N; ++k) u[i][k] = rstd * (u[i][k] - s1 - xh[i][k] * s2);
      store_row<T, N>(dx, (i * LANES + lane) * N, a.H, u[i]);
    }
  }
  if (!a.part) return;
  // one row of partial sums for the workgroup: dgamma, then dbeta
  for (int which = 0; which < 2; ++which) {
    float* out = a.part + ((int64_t)blockIdx.x * 2 + which) * a.H;
    if constexpr (ROWS == 1) {
#pragma unroll
      for (int i = 0; i < VPL; ++i) store_row<float, N>(out, (i * LANES + lane) * N, a.H, which ? db[i] : dg[i]);
    } else {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < VPL; ++i)
#pragma unroll
        for (int k = 0; k < N; ++k) sums[grp * WIDE + (i * LANES + lane) * N + k] = which ? db[i][k] : dg[i][k];
      __syncthreads();
      for (int c = threadIdx.x; c < a.H; c += block_of<LANES>()) {
        float s = 0.f;
#pragma unroll
        for (int r = 0; r < ROWS; ++r) s += sums[r * WIDE + c];
        out[c] = s;
      }
    }
  }
}

// Rows wider than registers hold: a workgroup takes a row at a time for dx,
// and the weights' gradients are column sums in launches of their own.
template <typename T, typename P>
__global__ __launch_bounds__(1024) void ln_bwd_long_kernel(LayerNormBwd a) {
  __shared__ float lds[2][32];
  const float inv = 1.f / (float)a.H;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x, turn ^= 1) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* dy = static_cast<const T*>(a.dy) + row * a.lddy;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s1 = 0.f, s2 = 0.f;
    for (int c = threadIdx.x; c < a.H; c += 1024) {
      const float u = to_f(dy[c]) * (a.gamma ? to_f(static_cast<const P*>(a.gamma)[c]) : 1.f);
      s1 += u;
      s2 += u * ((to_f(x[c]) - mean) * rstd);
    }
    row_sum2<1024>(s1, s2, lds[turn]);
    s1 *= inv;
    s2 *= inv;
    T* dx = static_cast<T*>(a.dx) + row * a.H;
    for (int c = threadIdx.x; c < a.H; c += 1024) {
      const float u = to_f(dy[c]) * (a.gamma ? to_f(static_cast<const P*>(a.gamma)[c]) : 1.f);
      dx[c] = from_f<T>(rstd * (u - s1 - (to_f(x[c]) - mean) * rstd * s2));
    }
  }
}
// partials of 256 columns (blockIdx.x) over every gridDim.y-th row
template <typename T>
__global__ __launch_bounds__(256) void ln_colsum_long_kernel(LayerNormBwd a) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.H) return;
  float dg = 0.f, db = 0.f;
  for (int64_t row = blockIdx.y; row < a.M; row += gridDim.y) {
    const float d = to_f(static_cast<const T*>(a.dy)[row * a.lddy + c]);
    dg += d * ((to_f(static_cast<const T*>(a.x)[row * a.ldx + c]) - a.mean[row]) * a.rstd[row]);
    db += d;
  }
  a.part[((int64_t)blockIdx.y * 2) * a.H + c] = dg;
  a.part[((int64_t)blockIdx.y * 2 + 1) * a.H + c] = db;
}

// dgamma (blockIdx.y = 0) / dbeta (1): the G rows of partials added in a fixed
// order, 32 columns (a 128-byte line) and 32 row lanes to a workgroup.
template <typename P>
__global__ __launch_bounds__(1024) void ln_wgrad_kernel(const float* __restrict__ part, P* dgamma, P* dbeta, int G,
                                                        int H) {
  __shared__ float lds[32][33];
  const int col = threadIdx.x & 31, r = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + col, which = blockIdx.y;
  float s = 0.f;
  if (c < H)
    for (int i = r; i < G; i += 32) s += part[((int64_t)i * 2 + which) * H + c];
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

// Lanes and packs a row takes: the fewest that hold it, so that one load of
// each lane covers the row as far as possible.  0 lanes: no variant holds it.
struct Shape {
  int lanes, vpl;
};
Shape shape_of(int H, int type, bool back) {
  const int n = type == ELEM_F32 ? 4 : 8;
  const Shape all[] = {{16, 1}, {64, 1}, {64, 2}, {64, 4}, {256, 2}, {256, 4}, {1024, 2}, {1024, 4}};
  for (const Shape& s : all)
    if (H <= s.lanes * s.vpl * n) return s;
  return {0, 0};
}
int rows_of(const Shape& s) { return s.lanes > 256 ? 1 : 256 / s.lanes; }

template <typename T, typename P>
void fwd_typed(const LayerNormFwd& a, hipStream_t s) {
  const Shape sh = shape_of(a.H, a.type, false);
  const int rows = sh.lanes ? rows_of(sh) : 1;
  const int64_t want = ((int64_t)a.M + rows - 1) / rows;
  const unsigned grid = (unsigned)(want < (1 << 20) ? want : (1 << 20));
#define MFL_LN(L_, V_)                                                              \
  if (sh.lanes == L_ && sh.vpl == V_) {                                             \
    ln_fwd_kernel<T, P, L_, V_><<<grid, block_of<L_>(), 0, s>>>(a);                 \
    return;                                                                         \
  }
  MFL_LN(16, 1)
  MFL_LN(64, 1) MFL_LN(64, 2) MFL_LN(64, 4) MFL_LN(256, 2) MFL_LN(256, 4) MFL_LN(1024, 2) MFL_LN(1024, 4)
#undef MFL_LN
  ln_fwd_long_kernel<T, P><<<grid, 1024, 0, s>>>(a);
}

template <typename T, typename P>
void bwd_typed(const LayerNormBwd& a, hipStream_t s) {
  const Shape sh = shape_of(a.H, a.type, true);
  const int G = layer_norm_bwd_blocks(a.M, a.H, a.type);
  bool done = false;
#define MFL_LN(L_, V_)                                                              \
  if (sh.lanes == L_ && sh.vpl == V_) {                                             \
    ln_bwd_kernel<T, P, L_, V_><<<G, block_of<L_>(), 0, s>>>(a);                    \
    done = true;                                                                    \
  }
  MFL_LN(16, 1)
  MFL_LN(64, 1) MFL_LN(64, 2) MFL_LN(64, 4) MFL_LN(256, 2) MFL_LN(256, 4) MFL_LN(1024, 2) MFL_LN(1024, 4)
#undef MFL_LN
  if (!done) {
    ln_bwd_long_kernel<T, P><<<(unsigned)(a.M < (1 << 20) ? a.M : (1 << 20)), 1024, 0, s>>>(a);
    if (a.part) ln_colsum_long_kernel<T><<<dim3((a.H + 255) / 256, G), 256, 0, s>>>(a);
  }
  if (a.part)
    ln_wgrad_kernel<P><<<dim3((a.H + 31) / 32, 2), 1024, 0, s>>>(a.part, static_cast<P*>(a.dgamma),
                                                                static_cast<P*>(a.dbeta), G, a.H);
}

}  // namespace

// Workgroups of the backward (rows of partial sums): enough to fill the chip
// four times over, fewer for few rows.
int layer_norm_bwd_blocks(int M, int H, int type) {
  const Shape sh = shape_of(H, type, true);
  if (!sh.lanes) return M < 64 ? M : 64;
  const int rows = rows_of(sh);
  const int64_t want = ((int64_t)M + rows - 1) / rows;
  return (int)(want < 1024 ? want : 1024);
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
