// AdamW over many tensors in one launch, states in 32 or 8 bits:
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,
//   p -= lr ((m c1) / (sqrt(v) c2 + eps) + wd p),
//   c1 = 1 / (1 - b1^t),  c2 = 1 / sqrt(1 - b2^t).
//
// Bound by memory: p, m, v are read and written and g read once (28 bytes an
// element with fp32 states and gradients, 16 with 8-bit states).  The
// parameters' table and the list of 4096-element chunks live on the device
// from the optimizer's construction; a step hands over only the gradients'
// addresses, as kernel arguments, so a step is two launches for up to 384
// tensors and holds in a captured graph.  The first launch (one thread)
// advances the step counter and evaluates c1, c2 (in 64 bits) and the
// rounding key once instead of in every workgroup.
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
// The arithmetic is a fixed order of single fp32 operations (no contraction),
// so results do not depend on the launch and repeat bit for bit.
#include "kernels/elem.h"
#include "kernels/lm.h"

#pragma clang fp contract(off)

namespace mfl {
namespace {

__device__ __forceinline__ uint32_t mix32(uint32_t x) {
  x *= 0x9E3779B1u;  // 2^32 / golden ratio, odd
  x ^= x >> 15;
  x *= 0x6A09E667u;  // fraction of sqrt(2)
  return x ^ (x >> 16);
}

// b^t by squaring, in 64 bits
__device__ double power(double b, uint32_t t) {
  double r = 1.0;
  for (; t; t >>= 1, b *= b)
    if (t & 1) r *= b;
  return r;
}

__global__ void adam_begin_kernel(AdamStep a) {
  const int t = a.step[0] + 1;
  a.step[0] = t;
  AdamScalars s;
  s.c1 = (float)(1.0 / (1.0 - power(a.beta1, (uint32_t)t)));
  s.c2 = (float)(1.0 / sqrt(1.0 - power(a.beta2, (uint32_t)t)));
  s.lr = a.lr_scale ? a.lr * a.lr_scale[0] : a.lr;
  s.key = mix32((uint32_t)t ^ a.seed);
  a.scalars[0] = s;
}

// 8 states of a thread; 16 threads (a row of the wave) share a scale.
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

// Codes of 8 values and the block's 2^E; SHIFT picks the dither's half of the
// mixed bits, LEAST keeps values above zero above zero.
template <bool HIGH, bool LEAST>
__device__ __forceinline__ uint2 pack_states(const float* x, const uint32_t* bits, float* scale) {
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const uint32_t b = __float_as_uint(x[k]) & 0x7fffffffu;
    if (b < 0x7f800000u && b > top) top = b;
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
    const uint32_t w = __shfl_xor(top, o, 64);
    top = w > top ? w : top;
  }
  // biased exponent of 2^E: a block whose largest is below 2^-110 (or zero) takes the least
  int e = (int)(top >> 23) - 7;
  e = e < 10 ? 10 : e;
  *scale = __uint_as_float((uint32_t)e << 23);
  const float up = __uint_as_float((uint32_t)(254 - e) << 23);
  uint32_t out[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = 4 * h + i;
      const float y = fabsf(x[k]) * up;
      const float low = y < 0.015625f ? 0.015625f : 0.f;  // below 2^-6 the codes are 2^-9 apart
      const uint32_t d = HIGH ? bits[k] >> 16 : bits[k] & 0xffffu;
      float z = __uint_as_float((__float_as_uint(y + low) + (d << 4)) & ~0xfffffu) - low;
      if (LEAST && y > 0.f) z = fmaxf(z, 0.001953125f);
      z = y < 512.f ? z : __uint_as_float(0x7fc00000u);
      q[i] = copysignf(z, x[k]);
    }
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w, true);
    out[h] = (uint32_t)w;
  }
  return make_uint2(out[0], out[1]);
}

// 8 elements from i of n (fill 0) and back, any alignment of the tensor
template <typename T>
__device__ __forceinline__ void load8(const T* p, int64_t i, int64_t n, float* f) {
  if (i + 8 <= n) {
    const Pack<T, 8> v = load_pack<T, 8>(p + i);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = to_f(v.e[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = i + k < n ? to_f(p[i + k]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int64_t i, int64_t n, const T* v) {
  if (i + 8 <= n) {
    __builtin_memcpy(p + i, v, 8 * sizeof(T));
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i + k < n) p[i + k] = v[k];
  }
}

__device__ __forceinline__ void load_grad(const void* g, int type, int64_t i, int64_t n, float* f) {
  if (type == ELEM_F32) load8(static_cast<const float*>(g), i, n, f);
  else if (type == ELEM_BF16) load8(static_cast<const BF16*>(g), i, n, f);
  else load8(static_cast<const F16*>(g), i, n, f);
}

template <int BITS>
__global__ __launch_bounds__(256) void adam_chunk_kernel(AdamStep a, AdamGrads grads, int first_tensor,
                                                         int64_t first_chunk) {
  const AdamChunk ch = a.chunks[first_chunk + blockIdx.x];
  const void* g = grads.g[ch.tensor - first_tensor];
  if (!g) return;  // no gradient: the tensor and its states stay as they are
  const int gtype = grads.type[ch.tensor - first_tensor];
  const AdamTensor t = a.tensors[ch.tensor];
  const AdamScalars sc = a.scalars[0];
  const float b1 = (float)a.beta1, b2 = (float)a.beta2, n1 = (float)(1.0 - a.beta1), n2 = (float)(1.0 - a.beta2);
  const int64_t end = t.numel < (int64_t)(ch.chunk + 1) * kAdamChunk ? t.numel : (int64_t)(ch.chunk + 1) * kAdamChunk;
  // whole blocks of 128: the 16 threads of a scale stay together
  for (int64_t i = (int64_t)ch.chunk * kAdamChunk + threadIdx.x * 8; i < ((end + kAdamBlock - 1) & ~(int64_t)(kAdamBlock - 1));
       i += 2048) {
    float gf[8], p[8], m[8], v[8], r[8];
    load_grad(g, gtype, i, end, gf);
    if (t.param_type == ELEM_F32) load8(static_cast<const float*>(t.p), i, end, p);
    else load8(static_cast<const BF16*>(t.p), i, end, p);
    const int64_t at = t.offset + i;
    if constexpr (BITS == 8) {
      unpack_states(reinterpret_cast<const uint2*>(a.m)[at >> 3], a.m_scale[at >> 7], m);
      unpack_states(reinterpret_cast<const uint2*>(a.v)[at >> 3], a.v_scale[at >> 7], v);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = v[k] * v[k];
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        *reinterpret_cast<float4*>(m + 4 * h) = reinterpret_cast<const float4*>(a.m)[(at >> 2) + h];
        *reinterpret_cast<float4*>(v + 4 * h) = reinterpret_cast<const float4*>(a.v)[(at >> 2) + h];
      }
    }
    uint32_t bits[8];
    const uint32_t high = (uint32_t)(at >> 32) * 0x9E3779B1u;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      m[k] = m[k] * b1 + gf[k] * n1;
      v[k] = v[k] * b2 + (gf[k] * n2) * gf[k];
      r[k] = sqrtf(v[k]);
      p[k] = p[k] - ((m[k] * sc.c1) / (r[k] * sc.c2 + a.eps) + p[k] * t.wd) * sc.lr;
      bits[k] = mix32((((uint32_t)at + k) ^ sc.key) + high);
    }
    if constexpr (BITS == 8) {
      float ms, vs;
      const uint2 mq = pack_states<false, false>(m, bits, &ms);
      const uint2 vq = pack_states<true, true>(r, bits, &vs);
      reinterpret_cast<uint2*>(a.m)[at >> 3] = mq;
      reinterpret_cast<uint2*>(a.v)[at >> 3] = vq;
      if ((threadIdx.x & 15) == 0) {
        a.m_scale[at >> 7] = ms;
        a.v_scale[at >> 7] = vs;
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        reinterpret_cast<float4*>(a.m)[(at >> 2) + h] = *reinterpret_cast<float4*>(m + 4 * h);
        reinterpret_cast<float4*>(a.v)[(at >> 2) + h] = *reinterpret_cast<float4*>(v + 4 * h);
      }
    }
    if (t.param_type == ELEM_F32) {
      store8(static_cast<float*>(t.p), i, end, p);
    } else {
      BF16 q[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t b = __float_as_uint(p[k]);
        const bool finite = (b & 0x7f800000u) != 0x7f800000u;
        if (finite) p[k] = __uint_as_float((b + (mix32(bits[k]) >> 16)) & 0xffff0000u);
        q[k] = from_f<BF16>(p[k]);
      }
      store8(static_cast<BF16*>(t.p), i, end, q);
    }
    if (t.mirror) {
      BF16 q[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) q[k] = from_f<BF16>(p[k]);
      store8(reinterpret_cast<BF16*>(t.mirror), i, end, q);
    }
  }
}

}  // namespace

void launch_adam_begin(const AdamStep& a, hipStream_t s) { adam_begin_kernel<<<1, 1, 0, s>>>(a); }

void launch_adam_chunks(const AdamStep& a, const AdamGrads& g, int first_tensor, int64_t first_chunk, int64_t chunks,
                        hipStream_t s) {
  if (a.state_bits == 8)
    adam_chunk_kernel<8><<<(unsigned)chunks, 256, 0, s>>>(a, g, first_tensor, first_chunk);
  else
    adam_chunk_kernel<32><<<(unsigned)chunks, 256, 0, s>>>(a, g, first_tensor, first_chunk);
}

}  // namespace mfl
