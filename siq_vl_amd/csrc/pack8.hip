// Activations kept in 8 bits for the backward pass: packing, unpacking, and the
// gated MLP activation h = silu(gate) up that packs its two inputs as it reads
// them and works on the unpacked values in its backward.
//
// 32 neighbours share one scale byte b.  With a the largest magnitude of the
// group and 2^E the power of two below it (doubled where a would round past
// the largest code), b = E + 127 and
//   int8:  code = rint(x / step),  step = 2^(E - 6),  |code| <= 127;
//   e4m3:  code = e4m3(x / step),  step = 2^(E - 8),  |value| <= 448.
// A power of two as the step costs up to one bit of int8's range (half a bit on
// average) and makes everything exact but the one rounding to the code:
// x / step is exact, and so is the value code * step in bf16 (at most 8
// significant bits) and in fp32.  step is held at 2^-126 or more.  A group
// with an infinity or a NaN has b = 255 and unpacks to NaN.
#include <type_traits>

#include "common.h"
#include "pack8.h"

namespace siq {

namespace {

template <bool F32>
struct Elem;
template <>
struct Elem<false> {
  typedef bf16 T;
};
template <>
struct Elem<true> {
  typedef float T;
};

// All four kernels are bound by memory: one pass, 16-byte accesses, two vectors
// of eight elements a thread (four: up to 3% slower, eight: up to 45%).  Everything
// read is read once, and codes are not looked at again before the backward: those
// accesses are nontemporal.  Measured, with and without: pack 65536 x 1536 48.5
// and 52.4 us (6.3 TB/s), unpack 46.7 and 52.5, swiglu8 forward 16384 x 6144 120
// and 146 (6.8 TB/s, a large copy: 5.0), its backward 127 and 142 (there the
// gradients are stored so too; for the forward's h that costs 14 us, for unpack 3).
//
// Eight neighbouring elements from p, those past `have` zero.
__device__ __forceinline__ void load8(const bf16* p, int have, float (&x)[8]) {
  if (have >= 8) {
    const bf16x8 v = __builtin_nontemporal_load(reinterpret_cast<const bf16x8*>(p));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)v[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i < have ? (float)p[i] : 0.f;
  }
}
__device__ __forceinline__ void load8(const float* p, int have, float (&x)[8]) {
  if (have >= 8) {
    const f32x4 a = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p));
    const f32x4 b = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p + 4));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = a[i];
      x[4 + i] = b[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i < have ? p[i] : 0.f;
  }
}
template <bool NT, class V, class T>
__device__ __forceinline__ void put(T* p, const V& v) {
  if (NT)
    __builtin_nontemporal_store(v, reinterpret_cast<V*>(p));
  else
    *reinterpret_cast<V*>(p) = v;
}
template <bool NT = false>
__device__ __forceinline__ void store8(bf16* p, int have, const float (&x)[8]) {
  if (have >= 8) {
    bf16x8 v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (bf16)x[i];
    put<NT>(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < have) p[i] = (bf16)x[i];
  }
}
template <bool NT = false>
__device__ __forceinline__ void store8(float* p, int have, const float (&x)[8]) {
  if (have >= 8) {
    put<NT>(p, f32x4{x[0], x[1], x[2], x[3]});
    put<NT>(p + 4, f32x4{x[4], x[5], x[6], x[7]});
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < have) p[i] = x[i];
  }
}

// The same maximum in the four lanes of a group (quad_perm 1 0 3 2, 2 3 0 1).
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true));
  return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true));
}

// Bits of the step and of its reciprocal for scale byte b (both normal numbers
// over the range of b that pack writes).
template <bool E4M3>
__device__ __forceinline__ float step_of(int b) {
  return __uint_as_float(b == 255 ? 0x7FC00000u : (uint32_t)(b - (E4M3 ? 8 : 6)) << 23);
}
template <bool E4M3>
__device__ __forceinline__ float inv_step_of(int b) {
  return __uint_as_float((uint32_t)((E4M3 ? 262 : 260) - b) << 23);
}

// Codes of 8 elements of a group that lies in four lanes (all four active),
// and its scale byte.  Magnitudes are compared as the integers that their bits
// are: NaN is above everything.
template <bool E4M3>
__device__ __forceinline__ u32x2 encode8(const float (&x)[8], int& b) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7FFFFFFFu);
  m = quad_max(m);
  if (m >= 0x7F800000u) {
    b = 255;
    return u32x2{0u, 0u};
  }
  // int8: from 127.5 steps on the largest would round to 128; e4m3: from above 464 to 480
  b = (int)((m + (E4M3 ? 0x17FFFFu : 0x10000u)) >> 23);
  b = min(max(b, E4M3 ? 9 : 7), 254);
  const float inv = inv_step_of<E4M3>(b);
  u32x2 c;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (E4M3) {
      float y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = __builtin_amdgcn_fmed3f(x[4 * k + i] * inv, -448.f, 448.f);
      int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
      c[k] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
    } else {
      // rounded to a whole number by adding 1.5 * 2^23: the low byte of the sum is the code
      uint32_t q[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        q[i] = __float_as_uint(__builtin_amdgcn_fmed3f(x[4 * k + i] * inv, -127.f, 127.f) + 12582912.f);
      const uint32_t lo = __builtin_amdgcn_perm(q[1], q[0], 0x0C0C0400u), hi = __builtin_amdgcn_perm(q[3], q[2], 0x04000C0Cu);
      c[k] = lo | hi;
    }
  }
  return c;
}

template <bool E4M3>
__device__ __forceinline__ void decode8(const u32x2& c, int b, float (&x)[8]) {
  const float s = step_of<E4M3>(b);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (E4M3) {
      const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[k], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[k], true);
      x[4 * k] = lo[0] * s;
      x[4 * k + 1] = lo[1] * s;
      x[4 * k + 2] = hi[0] * s;
      x[4 * k + 3] = hi[1] * s;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * k + i] = (float)(int)(int8_t)(c[k] >> (8 * i)) * s;
    }
  }
}

__device__ __forceinline__ u32x2 load_codes(const uint8_t* p, int have) {
  if (have >= 8) return __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p));
  u32x2 c = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < have) c[i / 4] |= (uint32_t)p[i] << (8 * (i & 3));
  return c;
}
__device__ __forceinline__ void store_codes(uint8_t* p, int have, const u32x2& c) {
  if (have >= 8) {
    put<true>(p, c);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < have) p[i] = (uint8_t)(c[i / 4] >> (8 * (i & 3)));
  }
}

constexpr int kThreads = 256;

// Elements of vector v (8 neighbours) that exist.
__device__ __forceinline__ int have_of(int64_t v, int64_t numel) {
  const int64_t left = numel - 8 * v;
  return left >= 8 ? 8 : left > 0 ? (int)left : 0;
}

template <bool F32, bool E4M3, int U>
__global__ __launch_bounds__(kThreads) void pack8_kernel(const void* __restrict__ xp, int64_t numel,
                                                         uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  typedef typename Elem<F32>::T T;
  const T* x = static_cast<const T*>(xp);
  const int64_t v0 = (int64_t)blockIdx.x * kThreads * U + threadIdx.x;
  float e[U][8];
#pragma unroll
  for (int u = 0; u < U; ++u) load8(x + 8 * (v0 + u * kThreads), have_of(v0 + u * kThreads, numel), e[u]);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t v = v0 + u * kThreads;
    const int have = have_of(v, numel);
    int b;
    const u32x2 c = encode8<E4M3>(e[u], b);
    store_codes(codes + 8 * v, have, c);
    if (have > 0 && (v & 3) == 0) scales[v >> 2] = (uint8_t)b;
  }
}

template <bool F32, bool E4M3, int U>
__global__ __launch_bounds__(kThreads) void unpack8_kernel(const uint8_t* __restrict__ codes,
                                                           const uint8_t* __restrict__ scales, int64_t numel,
                                                           void* __restrict__ xp) {
  typedef typename Elem<F32>::T T;
  T* x = static_cast<T*>(xp);
  const int64_t v0 = (int64_t)blockIdx.x * kThreads * U + threadIdx.x;
  u32x2 c[U];
  int b[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t v = v0 + u * kThreads;
    const int have = have_of(v, numel);
    c[u] = load_codes(codes + 8 * v, have);
    b[u] = have > 0 ? scales[v >> 2] : 0;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t v = v0 + u * kThreads;
    float e[8];
    decode8<E4M3>(c[u], b[u], e);
    store8(x + 8 * v, have_of(v, numel), e);
  }
}

// sigmoid(g) = r k with k = 1.  LOW: 2^-64 where g < -64, so that silu(g) = (g k) r and its slope are normal numbers
// down to g = -91.9; 1 / (1 + e^-g) is none from -87.3 on, and its reciprocal would be taken as zero.  (A path of its
// own, that vectors with such a gate alone take: in all of them it cost the backward 6%.)
template <bool LOW>
__device__ __forceinline__ void sigmoid(float g, float& r, float& k) {
  const bool low = LOW && g < -64.f;
  k = low ? 0x1p-64f : 1.f;
  r = __builtin_amdgcn_rcpf(k + exp2f_fast(__builtin_fmaf(-g, kLog2e, low ? -64.f : 0.f)));
}
// f(LOW) for eight gates.
template <class F>
__device__ __forceinline__ void with_gates(const float (&g)[8], F f) {
  const float m = fminf(fminf(fminf(g[0], g[1]), fminf(g[2], g[3])), fminf(fminf(g[4], g[5]), fminf(g[6], g[7])));
  if (m < -64.f)
    f(std::true_type());
  else
    f(std::false_type());
}

// Offset of vector v in a [rows, cols] tensor whose rows are ld elements apart
// (STRIDED: cols is a multiple of 8 then, so no vector straddles two rows).
template <bool STRIDED>
__device__ __forceinline__ int64_t at(int64_t v, int64_t cols, int64_t ld) {
  if (!STRIDED) return 8 * v;
  const int64_t vpr = cols >> 3, row = v / vpr;
  return row * ld + 8 * (v - row * vpr);
}

template <bool F32, bool E4M3, bool KEEP, bool STRIDED, int U>
__global__ __launch_bounds__(kThreads) void swiglu8_fwd_kernel(const SwigluArgs p) {
  typedef typename Elem<F32>::T T;
  const T *gate = static_cast<const T*>(p.gate), *up = static_cast<const T*>(p.up);
  T* h = static_cast<T*>(p.h);
  const int64_t numel = p.rows * p.cols, v0 = (int64_t)blockIdx.x * kThreads * U + threadIdx.x;
  float g[U][8], w[U][8];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t v = v0 + u * kThreads;
    const int have = have_of(v, numel);
    load8(gate + (have > 0 ? at<STRIDED>(v, p.cols, p.ld0) : 0), have, g[u]);
    load8(up + (have > 0 ? at<STRIDED>(v, p.cols, p.ld1) : 0), have, w[u]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t v = v0 + u * kThreads;
    const int have = have_of(v, numel);
    float o[8];
    with_gates(g[u], [&](auto low) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float r, k;
        sigmoid<decltype(low)::value>(g[u][i], r, k);
        o[i] = g[u][i] * k * r * w[u][i];
      }
    });
    store8(h + 8 * v, have, o);
    if (KEEP) {
      int gb, ub;
      const u32x2 gc = encode8<E4M3>(g[u], gb), uc = encode8<E4M3>(w[u], ub);
      store_codes(p.gcodes + 8 * v, have, gc);
      store_codes(p.ucodes + 8 * v, have, uc);
      if (have > 0 && (v & 3) == 0) {
        p.gscales[v >> 2] = (uint8_t)gb;
        p.uscales[v >> 2] = (uint8_t)ub;
      }
    }
  }
}

// du = dh g s,  dg = dh u s (1 + g (1 - s)),  h = g s u on the unpacked g, u.
template <bool F32, bool E4M3, bool STRIDED, int U>
__global__ __launch_bounds__(kThreads) void swiglu8_bwd_kernel(const SwigluArgs p) {
  typedef typename Elem<F32>::T T;
  const T* dh = static_cast<const T*>(p.dh);
  T *dgate = static_cast<T*>(p.dgate), *dup = static_cast<T*>(p.dup), *h = static_cast<T*>(p.h);
  const int64_t numel = p.rows * p.cols, v0 = (int64_t)blockIdx.x * kThreads * U + threadIdx.x;
  float d[U][8];
  u32x2 gc[U], uc[U];
  int gb[U], ub[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t v = v0 + u * kThreads;
    const int have = have_of(v, numel);
    load8(dh + 8 * v, have, d[u]);
    gc[u] = load_codes(p.gcodes + 8 * v, have);
    uc[u] = load_codes(p.ucodes + 8 * v, have);
    gb[u] = have > 0 ? p.gscales[v >> 2] : 0;
    ub[u] = have > 0 ? p.uscales[v >> 2] : 0;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t v = v0 + u * kThreads;
    const int have = have_of(v, numel);
    float g[8], w[8], dg[8], du[8], o[8];
    decode8<E4M3>(gc[u], gb[u], g);
    decode8<E4M3>(uc[u], ub[u], w);
    with_gates(g, [&](auto low) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float r, k;
        sigmoid<decltype(low)::value>(g[i], r, k);
        const float gs = g[i] * k * r;
        du[i] = d[u][i] * gs;
        dg[i] = d[u][i] * w[i] * r * (k * __builtin_fmaf(g[i], 1.f - r * k, 1.f));
        o[i] = gs * w[i];
      }
    });
    if (have > 0) {
      store8<true>(dgate + at<STRIDED>(v, p.cols, p.ld0), have, dg);
      store8<true>(dup + at<STRIDED>(v, p.cols, p.ld1), have, du);
      if (h != nullptr) store8(h + 8 * v, have, o);
    }
  }
}

template <int U>
unsigned blocks_of(int64_t numel) {
  const int64_t nvec = (numel + 7) / 8;
  return (unsigned)((nvec + kThreads * U - 1) / (kThreads * U));
}

// f(F32, E4M3) for the two runtime types.
template <class F>
void with_types(bool f32, bool e4m3, F f) {
  if (f32)
    e4m3 ? f(std::true_type(), std::true_type()) : f(std::true_type(), std::false_type());
  else
    e4m3 ? f(std::false_type(), std::true_type()) : f(std::false_type(), std::false_type());
}

}  // namespace

hipError_t launch_pack8(const void* x, int64_t numel, bool f32, bool e4m3, uint8_t* codes, uint8_t* scales,
                        hipStream_t stream) {
  constexpr int U = 2;
  with_types(f32, e4m3, [&](auto tf, auto te) {
    hipLaunchKernelGGL((pack8_kernel<decltype(tf)::value, decltype(te)::value, U>), dim3(blocks_of<U>(numel)),
                       dim3(kThreads), 0, stream, x, numel, codes, scales);
  });
  return hipGetLastError();
}

hipError_t launch_unpack8(const uint8_t* codes, const uint8_t* scales, int64_t numel, bool f32, bool e4m3, void* x,
                          hipStream_t stream) {
  constexpr int U = 2;
  with_types(f32, e4m3, [&](auto tf, auto te) {
    hipLaunchKernelGGL((unpack8_kernel<decltype(tf)::value, decltype(te)::value, U>), dim3(blocks_of<U>(numel)),
                       dim3(kThreads), 0, stream, codes, scales, numel, x);
  });
  return hipGetLastError();
}

hipError_t launch_swiglu8_fwd(const SwigluArgs& a, hipStream_t stream) {
  constexpr int U = 2;
  const bool strided = a.ld0 != a.cols || a.ld1 != a.cols, keep = a.gcodes != nullptr;
  with_types(a.f32, a.e4m3, [&](auto tf, auto te) {
    constexpr bool F = decltype(tf)::value, E = decltype(te)::value;
    const auto kept = strided ? swiglu8_fwd_kernel<F, E, true, true, U> : swiglu8_fwd_kernel<F, E, true, false, U>;
    const auto lone = strided ? swiglu8_fwd_kernel<F, false, false, true, U> : swiglu8_fwd_kernel<F, false, false, false, U>;
    hipLaunchKernelGGL((keep ? kept : lone), dim3(blocks_of<U>(a.rows * a.cols)), dim3(kThreads), 0, stream, a);
  });
  return hipGetLastError();
}

hipError_t launch_swiglu8_bwd(const SwigluArgs& a, hipStream_t stream) {
  constexpr int U = 2;
  const bool strided = a.ld0 != a.cols || a.ld1 != a.cols;
  with_types(a.f32, a.e4m3, [&](auto tf, auto te) {
    constexpr bool F = decltype(tf)::value, E = decltype(te)::value;
    const auto k = strided ? swiglu8_bwd_kernel<F, E, true, U> : swiglu8_bwd_kernel<F, E, false, U>;
    hipLaunchKernelGGL(k, dim3(blocks_of<U>(a.rows * a.cols)), dim3(kThreads), 0, stream, a);
  });
  return hipGetLastError();
}

}  // namespace siq
