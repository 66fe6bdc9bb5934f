// Rows of 16- or 32-bit values to 8-bit integers with one scale a row: the operands of the 8-bit product.
//
//   quantise   t = x
//   norm       h = x (+ r, rounded to x's type), t = h * w in 32 bits
//   both       a = max_k |t|,  q = 127 t / a rounded half to even,  s = a / 127 (norm: / sqrt(mean(h^2) + eps))
//
// The norm's root is the same for the whole row, so it cancels out of q and only enters s: one pass over the row gives
// the sum of squares and the maximum together, and q needs nothing else.
//
// q is exact, not "within one", without 64-bit arithmetic on the way.  What can go wrong is the rounding of a quotient next
// to half way between two integers, and values of few bits (bf16, fp16) sit exactly there all the time (t = a / 2 gives 63.5):
//   rows of 16-bit values (quantise): 127 t is exact in 32 bits; the quotient by a reciprocal is corrected once by its
//     remainder, which gives the exact quotient where 32 bits hold it (half way among them), and elsewhere one nearer to
//     the true one than that is to half way (by 254 T 2^-s - (2k + 1) A being a whole multiple of 2^-s: at least 2^-s / 2A off).
//   otherwise: t * (127 / a) inside a fused multiply-add is off by less than 8e-6, so only a value further than
//     0.5 - 2e-5 from its integer is in doubt.  A vector with such a value takes the sign of 254 t - (2 n +- 1) a for each:
//     next to half way the two products agree in their leading bits, so their difference is exact in 32 bits.
// Rows whose maximum is so small or large that these products leave the range of 32 bits are divided in 64.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace wb {

struct RowParams {
  const void* x;
  const void* r;  // residual, or null
  const void* w;  // norm weights
  void* h;        // x + r as stored
  int8_t* q;
  float* scale;
  long long ldx, ldr, ldh, ldq;  // elements between rows
  int M, K;
  float eps;
};

template <class T>
struct RowVec;  // 16 bytes of T, unpacked to 32 bits and back
template <>
struct RowVec<__nv_bfloat16> {
  static constexpr int E = 8;
  static __device__ __forceinline__ void unpack(const uint4& v, float* f) {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(u[i] << 16), f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 p = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      u[i] = *reinterpret_cast<const uint32_t*>(&p);
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
};
template <>
struct RowVec<__half> {
  static constexpr int E = 8;
  static __device__ __forceinline__ void unpack(const uint4& v, float* f) {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      f[2 * i] = p.x, f[2 * i + 1] = p.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 p = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      u[i] = *reinterpret_cast<const uint32_t*>(&p);
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
};
template <>
struct RowVec<float> {
  static constexpr int E = 4;
  static __device__ __forceinline__ void unpack(const uint4& v, float* f) {
    f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};

// Where a thread's values sit in its row: slot v (of E values).  VEC: one 16-byte vector; else values `nt` apart, so that
// the lanes of a warp read neighbouring values whatever the rows' alignment.
template <class T, bool VEC>
struct RowSlot {
  using V = RowVec<T>;
  static constexpr int E = V::E;
  static __device__ __forceinline__ int at(int v, int e, int t, int nt) { return VEC ? (v * nt + t) * E + e : (v * E + e) * nt + t; }

  static __device__ __forceinline__ uint4 load(const T* row, int v, int t, int nt, int K) {
    if (VEC && at(v, E - 1, t, nt) < K) return *reinterpret_cast<const uint4*>(row + at(v, 0, t, nt));
    T part[E];
#pragma unroll
    for (int e = 0; e < E; ++e) part[e] = at(v, e, t, nt) < K ? row[at(v, e, t, nt)] : T(0.0f);
    uint4 u;
    memcpy(&u, part, 16);
    return u;
  }
  static __device__ __forceinline__ void store(T* row, const uint4& u, int v, int t, int nt, int K) {
    if (VEC && at(v, E - 1, t, nt) < K) {
      *reinterpret_cast<uint4*>(row + at(v, 0, t, nt)) = u;
      return;
    }
    T part[E];
    memcpy(part, &u, 16);
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (at(v, e, t, nt) < K) row[at(v, e, t, nt)] = part[e];
  }
  static __device__ __forceinline__ void store_q(int8_t* row, const uint32_t* q4, int v, int t, int nt, int K) {
    if (VEC && at(v, E - 1, t, nt) < K) {
      if constexpr (E == 8) *reinterpret_cast<uint2*>(row + at(v, 0, t, nt)) = make_uint2(q4[0], q4[1]);
      else *reinterpret_cast<uint32_t*>(row + at(v, 0, t, nt)) = q4[0];
      return;
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (at(v, e, t, nt) < K) row[at(v, e, t, nt)] = int8_t(q4[e / 4] >> (8 * (e % 4)));
  }
};

// A row's maximum and how its values are divided by it.
struct RowDiv {
  float amax, inv;
  bool zero;   // nothing to divide by: q = 0
  bool wide;   // divide in 64 bits
};

// max_k |t| arrives as bits: NaN and infinity are above every finite value.  ONE: inv is 1 / amax, else 127 / amax.
template <bool ONE>
__device__ __forceinline__ RowDiv row_div(uint32_t amax_bits) {
  RowDiv d;
  d.amax = __uint_as_float(amax_bits);
  d.zero = amax_bits == 0u || amax_bits >= 0x7f800000u;
  d.wide = !(d.amax > 0x1p-90f && d.amax < 0x1p118f);
  d.inv = (ONE ? 1.0f : 127.0f) / d.amax;
  return d;
}

template <int E>
__device__ __noinline__ void row_quantise_wide(const float* t, float amax, uint32_t* b) {
#pragma unroll 1
  for (int e = 0; e < E; ++e) b[e] = uint32_t(int(rint(127.0 * double(t[e]) / double(amax))));
}

// SHORT: t has at most 11 bits (the first of the two ways above)
template <int E, bool SHORT>
__device__ __forceinline__ void row_quantise(const float* t, const RowDiv& d, uint32_t* q4) {
  constexpr float MAGIC = 12582912.0f;  // 1.5 * 2^23: adding it leaves the nearest integer in the low bits
  uint32_t b[E];
  if (d.wide) {
    float c[E];
    uint32_t n[E];
#pragma unroll
    for (int e = 0; e < E; ++e) c[e] = t[e];
    if (!d.zero) row_quantise_wide<E>(c, d.amax, n);
#pragma unroll
    for (int e = 0; e < E; ++e) b[e] = d.zero ? 0u : n[e];
  } else if constexpr (SHORT) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float c = __fmul_rn(127.0f, t[e]), q0 = __fmul_rn(c, d.inv);
      const float q1 = __fmaf_rn(__fmaf_rn(-q0, d.amax, c), d.inv, q0);
      b[e] = __float_as_uint(__fadd_rn(q1, MAGIC));
    }
  } else {
    float far = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float r = __fmaf_rn(t[e], d.inv, MAGIC), n = __fadd_rn(r, -MAGIC);
      b[e] = __float_as_uint(r);
      far = fmaxf(far, fabsf(__fmaf_rn(t[e], d.inv, -n)));
    }
    if (far > 0.5f - 2e-5f) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float n = __fadd_rn(__uint_as_float(b[e]), -MAGIC), off = __fmaf_rn(t[e], d.inv, -n);
        const float side = off < 0.0f ? -1.0f : 1.0f, half = __fmaf_rn(2.0f, n, side);  // 2 x the half way point next to t
        const float hi = __fmul_rn(half, d.amax), lo = __fmaf_rn(half, d.amax, -hi);
        const float past = __fmul_rn(__fadd_rn(__fmaf_rn(254.0f, t[e], -hi), -lo), side);
        if (fabsf(off) > 0.5f - 2e-5f && (past > 0.0f || (past == 0.0f && (b[e] & 1u)))) b[e] += off < 0.0f ? 0xffffffffu : 1u;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < E / 4; ++i) {
    const uint32_t lo = __byte_perm(b[4 * i], b[4 * i + 1], 0x0040), hi = __byte_perm(b[4 * i + 2], b[4 * i + 3], 0x0040);
    q4[i] = __byte_perm(lo, hi, 0x5410);
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// blockDim = (threads a row, rows a block): more than 32 threads a row only with one row a block.  VPT vectors of 16
// bytes a thread; LOOP: rows longer than a block holds, read a second time (from L2) for the second half of the work.
template <class T, bool NORM, bool RES, bool VEC, int VPT, bool LOOP>
__global__ void __launch_bounds__(VPT <= 2 ? 1024 : 512) rows_kernel(const RowParams p) {
  static_assert(NORM || !RES, "the residual comes with the norm");
  using S = RowSlot<T, VEC>;
  constexpr int E = S::E;
  constexpr bool SHORT = !NORM && sizeof(T) == 2;
  constexpr bool AHEAD = !LOOP && VPT <= 2;  // the next row's loads are out while this row is reduced
  constexpr bool KEEP_W = !LOOP && VPT <= 4;
  __shared__ float2 part[2][32];
  __shared__ double dpart[32];
  const int t = int(threadIdx.x), nt = int(blockDim.x), lane = t & 31, warp = t >> 5, nw = nt >> 5;
  const int step = int(gridDim.x * blockDim.y), chunk = nt * VPT * E;
  const T* const w = static_cast<const T*>(p.w);
  int buf = 0;

  uint4 wv[KEEP_W ? VPT : 1];
  if constexpr (NORM && KEEP_W) {
#pragma unroll
    for (int v = 0; v < VPT; ++v) wv[v] = S::load(w, v, t, nt, p.K);
  }
  uint4 nx[AHEAD ? VPT : 1], nr[AHEAD && RES ? VPT : 1];
  long long row = (long long)(blockIdx.x) * blockDim.y + threadIdx.y;
  auto fetch = [&](long long i) {
    if constexpr (AHEAD) {
#pragma unroll
      for (int v = 0; v < VPT; ++v) {
        nx[v] = S::load(static_cast<const T*>(p.x) + i * p.ldx, v, t, nt, p.K);
        if constexpr (RES) nr[v] = S::load(static_cast<const T*>(p.r) + i * p.ldr, v, t, nt, p.K);
      }
    }
  };
  if (row < p.M) fetch(row);

  for (; row < p.M; row += step) {
    const T* const x = static_cast<const T*>(p.x) + row * p.ldx;
    const T* const r = RES ? static_cast<const T*>(p.r) + row * p.ldr : nullptr;
    T* const h = RES ? static_cast<T*>(p.h) + row * p.ldh : nullptr;
    uint4 hv[VPT];
    float sum = 0.0f;
    uint32_t top = 0u;
    // h of one chunk of the row (into registers, and out where there is a residual), its sum of squares and maximum
    auto first = [&](int c) {
#pragma unroll
      for (int v = 0; v < VPT; ++v) {
        uint4 a;
        if constexpr (AHEAD) a = nx[v];
        else a = S::load(x + c, v, t, nt, p.K - c);
        float f[E];
        if constexpr (RES) {
          uint4 b;
          if constexpr (AHEAD) b = nr[v];
          else b = S::load(r + c, v, t, nt, p.K - c);
          float g[E];
          S::V::unpack(a, f), S::V::unpack(b, g);
#pragma unroll
          for (int e = 0; e < E; ++e) f[e] += g[e];
          a = S::V::pack(f);
          S::store(h + c, a, v, t, nt, p.K - c);
        }
        hv[v] = a;
        S::V::unpack(a, f);
        if constexpr (NORM) {
          float g[E];
          if constexpr (KEEP_W) S::V::unpack(wv[v], g);
          else S::V::unpack(S::load(w + c, v, t, nt, p.K - c), g);
#pragma unroll
          for (int e = 0; e < E; ++e) sum = fmaf(f[e], f[e], sum), f[e] *= g[e];
        }
#pragma unroll
        for (int e = 0; e < E; ++e) top = max(top, __float_as_uint(f[e]) & 0x7fffffffu);
      }
    };
    auto second = [&](int c, const RowDiv& d) {
#pragma unroll
      for (int v = 0; v < VPT; ++v) {
        float f[E];
        if constexpr (LOOP) S::V::unpack(S::load((RES ? h : x) + c, v, t, nt, p.K - c), f);
        else S::V::unpack(hv[v], f);
        if constexpr (NORM) {
          float g[E];
          if constexpr (KEEP_W) S::V::unpack(wv[v], g);
          else S::V::unpack(S::load(w + c, v, t, nt, p.K - c), g);
#pragma unroll
          for (int e = 0; e < E; ++e) f[e] *= g[e];
        }
        uint32_t q4[E / 4];
        row_quantise<E, SHORT>(f, d, q4);
        S::store_q(p.q + row * p.ldq + c, q4, v, t, nt, p.K - c);
      }
    };

    if constexpr (LOOP) {
      for (int c = 0; c < p.K; c += chunk) first(c);
    } else {
      first(0);
    }
    if (row + step < p.M) fetch(row + step);

    if constexpr (NORM) sum = warp_sum(sum);
    top = __reduce_max_sync(0xffffffffu, top);
    if (nt > 32) {
      if (lane == 0) part[buf][warp] = make_float2(sum, __uint_as_float(top));
      __syncthreads();
      const float2 o = lane < nw ? part[buf][lane] : make_float2(0.0f, 0.0f);
      if constexpr (NORM) sum = warp_sum(o.x);
      top = __reduce_max_sync(0xffffffffu, __float_as_uint(o.y));
      buf ^= 1;
    }
    const RowDiv d = row_div<SHORT>(top);
    float s = d.amax / 127.0f;
    if constexpr (NORM) {
      // squares that 32 bits cannot hold (or hold with too few of them): the sum again in 64
      if (!(sum > 0x1p-90f && sum < 0x1p126f) && !d.zero) {
        double ds = 0.0;
        auto squares = [&](const uint4& a) {
          float f[E];
          S::V::unpack(a, f);
#pragma unroll
          for (int e = 0; e < E; ++e) ds = fma(double(f[e]), double(f[e]), ds);
        };
        if constexpr (LOOP) {
          for (int c = 0; c < p.K; c += chunk)
            for (int v = 0; v < VPT; ++v) squares(S::load((RES ? h : x) + c, v, t, nt, p.K - c));
        } else {
#pragma unroll
          for (int v = 0; v < VPT; ++v) squares(hv[v]);
        }
        ds = warp_sum(ds);
        if (nt > 32) {
          if (lane == 0) dpart[warp] = ds;
          __syncthreads();
          ds = warp_sum(lane < nw ? dpart[lane] : 0.0);
        }
        s = float(double(d.amax) / (127.0 * sqrt(ds / p.K + double(p.eps))));
      } else {
        s = s / sqrtf(sum / float(p.K) + p.eps);
      }
    }
    if (top == 0u) s = 0.0f;
    if (top >= 0x7f800000u) s = __uint_as_float(0x7fc00000u);
    if (t == 0) p.scale[row] = s;

    if constexpr (LOOP) {
      for (int c = 0; c < p.K; c += chunk) second(c, d);
    } else {
      second(0, d);
    }
  }
}

}  // namespace wb
