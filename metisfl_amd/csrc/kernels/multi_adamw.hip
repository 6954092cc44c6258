// AdamW over many tensors in one launch, states in 32 or 8 bits:
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,
//   p -= lr ((m c1) / (sqrt(v) c2 + eps) + wd p),
//   c1 = 1 / (1 - b1^t),  c2 = 1 / sqrt(1 - b2^t).
//
// Bound by memory: p, m, v are read and written and g read once (28 bytes an
// element with fp32 states and gradients, 16 with 8-bit states).  The
// parameters' table and the list of their chunks live on the device
// from the optimizer's construction; a step hands over only the gradients'
// addresses, as kernel arguments, so a step is two launches for up to 384
// tensors and holds in a captured graph.  The first launch (one thread)
// advances the step counter and evaluates c1, c2 (in 64 bits) and the
// rounding key once instead of in every workgroup.  Up to 512 workgroups do
// that themselves in a single launch (six tensors of 118282 elements: 5.9 us a
// step instead of 9.3 us in two launches; the arrivals of 50000 workgroups
// would take longer than the step).
//
// 8-bit states: 128 elements share a power of two 2^E that puts their largest
// into [128, 256) of e4m3; m is kept as it is and v by its root, which halves
// the range its exponent has to span (2^17 of sqrt(v) below the largest).  An
// element between two codes goes up with the chance of its distance (16 bits
// of a mix of step, seed and place), because a nearest rounding would never
// move: b2 = 0.999 changes v by 0.1 % of (g^2 / v - 1) a step and half a code
// is 3 % or more.  sqrt(v) > 0 never becomes 0, so the quotient stays bounded.
// bf16 parameters are rounded the same way for the same reason.  Non-finite
// states are kept as NaN.
//
// Measured: 110 million elements in 199 tensors, bf16 gradients and mirrors,
// 593 us (5.2 TB/s) with 32-bit and 354 us (5.0 TB/s) with 8-bit states.
//
// The arithmetic is a fixed order of single fp32 operations (no contraction),
// so results do not depend on the launch and repeat bit for bit.
#include "kernels/elem.h"
#include "kernels/lm.h"

#pragma clang fp contract(off)

namespace mfl {
namespace {

__device__ __forceinline__ uint32_t mix32_rest(uint32_t x) {
  x ^= x >> 15;
  x *= 0x6A09E667u;  // fraction of sqrt(2)
  asm("" : "+v"(x));  // one product: a shift of it by 16 is not to become a second one
  return x ^ (x >> 16);
}
__device__ __forceinline__ uint32_t mix32(uint32_t x) { return mix32_rest(x * 0x9E3779B1u); }  // 2^32 / golden ratio, odd

// Correctly rounded root and quotient in the range where their residuals and
// results are normal numbers (in_range): one Newton step on v_rsq_f32 with
// the residual x - g^2 by a fused multiply-add, and Markstein's quotient
// correction with a correctly rounded reciprocal.  The root and the reciprocal
// were compared with 64 bits for every one of the 2^24 significands (root:
// both parities of the exponent), the quotient for 8.6e9 pairs: none differs.
// They take 8 and 9 issue slots where the general forms, which also scale, take
// 19 and 15; the 8-bit step is bound by these as much as by memory (83 ragged
// bf16 tensors 60 -> 57 us).
__device__ __forceinline__ float root_in_range(float x) {
  const float y = __builtin_amdgcn_rsqf(x), g = x * y;
  return fmaf(fmaf(-g, g, x), 0.5f * y, g);
}
__device__ __forceinline__ float quotient_in_range(float n, float d) {
  float r = __builtin_amdgcn_rcpf(d);
  r = fmaf(fmaf(-d, r, 1.f), r, r);
  const float q = n * r;
  return fmaf(fmaf(-d, q, n), r, q);
}
// That range.  v from 2^-100 to 2^40 and |m| from 2^-60 to 2^50, with c1, c2 (at
// least 1) at most 2^27 and eps at most 2^20: the denominator is between 2^-50
// and 2^48, the quotient between 2^-108 and 2^127.
constexpr uint32_t pow2(int e) { return (uint32_t)(127 + e) << 23; }
__device__ __forceinline__ bool in_range(uint32_t m_low, uint32_t m_high, uint32_t v_low, uint32_t v_high) {
  return m_low >= pow2(-60) && m_high <= pow2(50) && v_low >= pow2(-100) && v_high <= pow2(40);
}
__device__ __forceinline__ bool in_range(float c1, float c2, float eps) {
  return c1 <= 0x1p27f && c2 <= 0x1p27f && eps >= 0.f && eps <= 0x1p20f;
}

// b^t by squaring, in 64 bits
__device__ double power(double b, uint32_t t) {
  double r = 1.0;
  for (; t; t >>= 1, b *= b)
    if (t & 1) r *= b;
  return r;
}

__device__ __forceinline__ AdamScalars adam_scalars(const AdamStep& a, int t) {
  AdamScalars s;
  s.c1 = (float)(1.0 / (1.0 - power(a.beta1, (uint32_t)t)));
  s.c2 = (float)(1.0 / sqrt(1.0 - power(a.beta2, (uint32_t)t)));
  s.lr = a.lr_scale ? a.lr * a.lr_scale[0] : a.lr;
  s.key = mix32((uint32_t)t ^ a.seed);
  return s;
}

__global__ void adam_begin_kernel(AdamStep a) {
  const int t = a.step[0] + 1;
  a.step[0] = t;
  a.scalars[0] = adam_scalars(a, t);
}

// The same within a launch of few workgroups: each reads the counter, and the
// last of them to have read it writes the new one (and clears the arrivals).
// The empty statement holds t, so an arrival follows its read.
__device__ __forceinline__ AdamScalars adam_begin_here(const AdamStep& a) {
  __shared__ AdamScalars sh;
  if (threadIdx.x == 0) {
    const int t = __hip_atomic_load(a.step, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1;
    asm volatile("" ::"v"(t) : "memory");
    const int before = __hip_atomic_fetch_add(a.arrived, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    sh = adam_scalars(a, t);
    if (before == (int)gridDim.x - 1) {
      __hip_atomic_store(a.arrived, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(a.step, t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  __syncthreads();
  return sh;
}

// Read-only tables through scalar loads.
template <typename T>
__device__ __forceinline__ T table_entry(const T* table, int64_t i) {
  typedef const __attribute__((address_space(4))) uint32_t* Words;
  const Words w = (Words)(uintptr_t)(table + i);
  uint32_t words[sizeof(T) / 4];
#pragma unroll
  for (size_t k = 0; k < sizeof(T) / 4; ++k) words[k] = w[k];
  T v;
  __builtin_memcpy(&v, words, sizeof(T));
  return v;
}

// 8 codes of a thread as values.
__device__ __forceinline__ void unpack_states(uint2 w, float scale, float* f) {
  typedef float v2 __attribute__((ext_vector_type(2)));
  const uint32_t u[2] = {w.x, w.y};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const v2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)u[i], false);
    const v2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)u[i], true);
    f[4 * i] = a.x * scale;
    f[4 * i + 1] = a.y * scale;
    f[4 * i + 2] = b.x * scale;
    f[4 * i + 3] = b.y * scale;
  }
}

constexpr uint32_t kInf = 0x7f800000u;
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t row_max(uint32_t v) {  // over a row of 16 lanes
#define MFL_ROR(N_) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 + N_, 0xf, 0xf, false))
  MFL_ROR(8);
  MFL_ROR(4);
  MFL_ROR(2);
  MFL_ROR(1);
#undef MFL_ROR
  return v;
}

// Codes of 8 values and their block's 2^E (16 threads, a row of the wave, have
// a block).  The conversion with a dither adds the dither's high bits to those
// a code drops, below 2^-6 too, where codes are 2^-9 apart; HIGH picks the half
// of the mixed bits, LEAST keeps values above zero above zero.  Infinities
// become NaN and do not raise the scale.
template <bool HIGH, bool LEAST>
__device__ __forceinline__ uint2 pack_states(const float* x, const uint32_t* bits, float* scale) {
  uint32_t top = 0;  // magnitudes order as whole numbers, the non-finite ones on top
#pragma unroll
  for (int k = 0; k < 8; ++k) top = max(top, magnitude(x[k]));
  top = row_max(top);
  if (top >= kInf) {
    top = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) top = magnitude(x[k]) < kInf ? max(top, magnitude(x[k])) : top;
    top = row_max(top);
  }
  // biased exponent of 2^E: a block whose largest is below 2^-110 (or zero) takes the least
  int e = (int)(top >> 23) - 7;
  e = e < 10 ? 10 : e;
  *scale = __uint_as_float((uint32_t)e << 23);
  const float up = __uint_as_float((uint32_t)(254 - e) << 23);
  int out[2] = {0, 0};
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    float y = x[k] * up;
    if (LEAST) y = y > 0.f ? fmaxf(y, 0.001953125f) : y;
    const uint32_t d = HIGH ? bits[k] & 0xffff0000u : bits[k] << 16;
    int& w = out[k / 4];
    w = k % 4 == 0   ? __builtin_amdgcn_cvt_sr_fp8_f32(y, d, w, 0)
        : k % 4 == 1 ? __builtin_amdgcn_cvt_sr_fp8_f32(y, d, w, 1)
        : k % 4 == 2 ? __builtin_amdgcn_cvt_sr_fp8_f32(y, d, w, 2)
                     : __builtin_amdgcn_cvt_sr_fp8_f32(y, d, w, 3);
  }
  return make_uint2((uint32_t)out[0], (uint32_t)out[1]);
}

// n (at most 8) elements of any alignment; the others 0
template <typename T>
__device__ __forceinline__ Pack<T, 8> load8(const T* p, int n) {
  if (n >= 8) return load_pack<T, 8>(p);
  Pack<T, 8> v;
#pragma unroll
  for (int k = 0; k < 8; ++k) v.e[k] = k < n ? p[k] : T{};
  return v;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int n, const Pack<T, 8>& v) {
  if (n >= 8) {
    store_pack<T, 8>(p, v);
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (k < n) p[k] = v.e[k];
}

// What a thread reads of 8 elements.
template <int BITS, typename PT, typename GT>
struct AdamIn {
  Pack<PT, 8> p;
  Pack<GT, 8> g;
  Pack<float, 8> m, v;  // 32 bits
  uint2 mq, vq;         // 8 bits
  float ms, vs;
  __device__ __forceinline__ void load(const PT* pp, const GT* gp, const void* mp, const void* vp, const float* msp,
                                       const float* vsp, int i, int left) {
    if constexpr (BITS == 8) {
      mq = static_cast<const uint2*>(mp)[i >> 3];
      vq = static_cast<const uint2*>(vp)[i >> 3];
      ms = msp[i >> 7];
      vs = vsp[i >> 7];
    } else {
      m = load_pack<float, 8>(static_cast<const float*>(mp) + i);
      v = load_pack<float, 8>(static_cast<const float*>(vp) + i);
    }
    p = load8(pp + i, left);
    g = load8(gp + i, left);
  }
};

// One chunk: elements chunk * kAdamChunk .. of tensor t, 8 to a thread, all of
// a thread's loads in flight together.  The pointers are the workgroup's (scalars).
template <int BITS, bool WHOLE, typename PT, typename GT>
__device__ __forceinline__ void adam_chunk(const AdamStep& a, const AdamTensor& t, const GT* g, int chunk) {
  const int64_t first = (int64_t)chunk * kAdamChunk, at0 = t.offset + first;
  const int n = (int)(t.numel - first < kAdamChunk ? t.numel - first : kAdamChunk);
  const int i = threadIdx.x * 8, left = n - i;
  // whole blocks of 128: the 16 threads of a scale stay together
  const bool on = i < ((n + kAdamBlock - 1) & ~(kAdamBlock - 1));
  PT* p0 = static_cast<PT*>(t.p) + first;
  BF16* mirror = t.mirror ? reinterpret_cast<BF16*>(t.mirror) + first : nullptr;
  const int state = BITS == 8 ? 1 : 4;
  char* m0 = static_cast<char*>(a.m) + at0 * state;
  char* v0 = static_cast<char*>(a.v) + at0 * state;
  float* ms0 = BITS == 8 ? a.m_scale + at0 / kAdamBlock : nullptr;
  float* vs0 = BITS == 8 ? a.v_scale + at0 / kAdamBlock : nullptr;
  const float b1 = (float)a.beta1, b2 = (float)a.beta2, n1 = (float)(1.0 - a.beta1), n2 = (float)(1.0 - a.beta2);
  AdamIn<BITS, PT, GT> in;
  if (on) in.load(p0, g + first, m0, v0, ms0, vs0, i, left);
  AdamScalars sc;
  if constexpr (WHOLE) sc = adam_begin_here(a);
  else sc = table_entry(a.scalars, 0);
  if (!on) return;
  float p[8], m[8], v[8], r[8];
  uint32_t bits[8];
  if constexpr (BITS == 8) {
    unpack_states(in.mq, in.ms, m);
    unpack_states(in.vq, in.vs, v);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = v[k] * v[k];
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      m[k] = in.m.e[k];
      v[k] = in.v.e[k];
    }
  }
  uint32_t m_low = kInf, m_high = 0, v_low = kInf, v_high = 0;  // (v has no sign but a NaN's)
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float gk = to_f(in.g.e[k]);
    m[k] = m[k] * b1 + gk * n1;
    v[k] = v[k] * b2 + (gk * n2) * gk;
    m_low = min(m_low, magnitude(m[k]));
    m_high = max(m_high, magnitude(m[k]));
    v_low = min(v_low, __float_as_uint(v[k]));
    v_high = max(v_high, __float_as_uint(v[k]));
  }
  if (in_range(m_low, m_high, v_low, v_high) && in_range(sc.c1, sc.c2, a.eps)) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      r[k] = root_in_range(v[k]);
      p[k] = quotient_in_range(m[k] * sc.c1, r[k] * sc.c2 + a.eps);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      r[k] = sqrtf(v[k]);
      p[k] = (m[k] * sc.c1) / (r[k] * sc.c2 + a.eps);
    }
  }
  const float wd = t.decays ? a.wd : 0.f;
  const int64_t at = at0 + i;
  // mix32(((at + k) ^ key) + high part), its first product by parts: at is a
  // multiple of 8, so (at + k) ^ key is (at ^ key with the low bits 0) + (k ^ the key's)
  const uint32_t key = (uint32_t)__builtin_amdgcn_readfirstlane((int)sc.key);
  const uint32_t base = (((uint32_t)at ^ (key & ~7u)) + (uint32_t)(at >> 32) * 0x9E3779B1u) * 0x9E3779B1u;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float pk = to_f(in.p.e[k]);
    p[k] = pk - (p[k] + pk * wd) * sc.lr;
    if (BITS == 8 || sizeof(PT) == 2) bits[k] = mix32_rest(base + (((uint32_t)k ^ key) & 7u) * 0x9E3779B1u);
  }
  if constexpr (BITS == 8) {
    float ms, vs;
    const uint2 mq = pack_states<false, false>(m, bits, &ms);
    const uint2 vq = pack_states<true, true>(r, bits, &vs);
    reinterpret_cast<uint2*>(m0)[i >> 3] = mq;
    reinterpret_cast<uint2*>(v0)[i >> 3] = vq;
    if ((threadIdx.x & 15) == 0) {
      ms0[i >> 7] = ms;
      vs0[i >> 7] = vs;
    }
  } else {
    Pack<float, 8> mo, vo;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      mo.e[k] = m[k];
      vo.e[k] = v[k];
    }
    store_pack<float, 8>(reinterpret_cast<float*>(m0) + i, mo);
    store_pack<float, 8>(reinterpret_cast<float*>(v0) + i, vo);
  }
  Pack<PT, 8> po;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if constexpr (sizeof(PT) == 2) {
      const uint32_t b = __float_as_uint(p[k]);
      if (fabsf(p[k]) < INFINITY) p[k] = __uint_as_float((b + (mix32(bits[k]) >> 16)) & 0xffff0000u);
    }
    po.e[k] = from_f<PT>(p[k]);
  }
  store8(p0 + i, left, po);
  if (mirror) {
    Pack<BF16, 8> q;
#pragma unroll
    for (int k = 0; k < 8; ++k) q.e[k] = from_f<BF16>(p[k]);
    store8(mirror + i, left, q);
  }
}

template <int BITS, bool WHOLE>
__global__ __launch_bounds__(256) void adam_chunk_kernel(AdamStep a, AdamGrads grads, int first_tensor,
                                                         int64_t first_chunk) {
  const AdamChunk ch = table_entry(a.chunks, first_chunk + blockIdx.x);
  const void* g = grads.g[ch.tensor - first_tensor];
  if (!g) {  // no gradient: the tensor and its states stay as they are
    if constexpr (WHOLE) adam_begin_here(a);
    return;
  }
  const int gtype = grads.type[ch.tensor - first_tensor];
  const AdamTensor t = table_entry(a.tensors, ch.tensor);
#define MFL_ADAM(P_, G_) adam_chunk<BITS, WHOLE, P_, G_>(a, t, static_cast<const G_*>(g), ch.chunk)
  if (t.param_type == ELEM_F32) {
    if (gtype == ELEM_F32) MFL_ADAM(float, float);
    else if (gtype == ELEM_BF16) MFL_ADAM(float, BF16);
    else MFL_ADAM(float, F16);
  } else {
    if (gtype == ELEM_F32) MFL_ADAM(BF16, float);
    else if (gtype == ELEM_BF16) MFL_ADAM(BF16, BF16);
    else MFL_ADAM(BF16, F16);
  }
#undef MFL_ADAM
}

}  // namespace

void launch_adam_begin(const AdamStep& a, hipStream_t s) { adam_begin_kernel<<<1, 1, 0, s>>>(a); }

void launch_adam_chunks(const AdamStep& a, const AdamGrads& g, int first_tensor, int64_t first_chunk, int64_t chunks,
                        bool whole, hipStream_t s) {
  const unsigned n = (unsigned)chunks;
  if (a.state_bits == 8 && whole) adam_chunk_kernel<8, true><<<n, 256, 0, s>>>(a, g, first_tensor, first_chunk);
  else if (a.state_bits == 8) adam_chunk_kernel<8, false><<<n, 256, 0, s>>>(a, g, first_tensor, first_chunk);
  else if (whole) adam_chunk_kernel<32, true><<<n, 256, 0, s>>>(a, g, first_tensor, first_chunk);
  else adam_chunk_kernel<32, false><<<n, 256, 0, s>>>(a, g, first_tensor, first_chunk);
}

}  // namespace mfl
