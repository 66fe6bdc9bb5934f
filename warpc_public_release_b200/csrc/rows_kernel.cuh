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
//   otherwise: t times a factor just below 127 / a and t times one just above are both rounded (each in one fused
//     multiply-add); where the two agree, so does what lies between them.  A vector in which some do not (values within
//     6e-5 of half way) takes the sign of 254 t - (2 n +- 1) a for each value: next to half way the two products agree in
//     their leading bits, so their difference is exact in 32 bits.
// Rows whose maximum is so small or large that these products leave the range of 32 bits are divided in 64.
//
// What bounds it is memory in the end and instructions on the way: at 6.5 TB/s an SM has about 16 instruction slots a value of a
// 16-bit row that is only read and quantised.  So the arithmetic is in pairs (f32x2), a 16-bit row's maximum is taken on the packed
// values, what only the row's scale needs (roots, exact divisions, the sum over the warps) is left to one warp, and a thread
// holds sixteen values (of 16 bits; eight of 32) and more, so that the reductions are spread over them.
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
  long long ldx, ldr, ldh, ldq;                  // elements between rows
  long long step_x, step_r, step_h, step_q;      // and between a block's (a warp's) rows: gridDim.x * blockDim.y of them
  int step;
  int M, K;
  float eps;
};

// ---------------------------------------------------------------- pairs of 32-bit values
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair(float a, float b) {
  f32x2 d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ void split(f32x2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// the larger of two magnitudes; NaN if either is
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(fabsf(b)));
  return d;
}

// 16 bytes of T: pairs of 32-bit values and back; magnitudes on the packed words (`top` of a row, kept packed, NaN kept).
template <class T>
struct RowVec;
template <>
struct RowVec<__nv_bfloat16> {
  static constexpr int E = 8;
  static __device__ __forceinline__ void unpack(const uint4& v, f32x2* f) {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = pair(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
  }
  static __device__ __forceinline__ uint4 pack(const f32x2* f) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a, b;
      split(f[i], a, b);
      const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
      u[i] = *reinterpret_cast<const uint32_t*>(&p);
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
  static __device__ __forceinline__ uint32_t larger(uint32_t top, uint32_t u) {
    u &= 0x7fff7fffu;
    const __nv_bfloat162 p = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&top), *reinterpret_cast<const __nv_bfloat162*>(&u));
    return *reinterpret_cast<const uint32_t*>(&p);
  }
  static __device__ __forceinline__ float larger_of(uint32_t top) { return max_nan(__uint_as_float(top << 16), __uint_as_float(top & 0xffff0000u)); }
};
template <>
struct RowVec<__half> {
  static constexpr int E = 8;
  static __device__ __forceinline__ void unpack(const uint4& v, f32x2* f) {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      f[i] = pair(p.x, p.y);
    }
  }
  static __device__ __forceinline__ uint4 pack(const f32x2* f) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a, b;
      split(f[i], a, b);
      const __half2 p = __floats2half2_rn(a, b);
      u[i] = *reinterpret_cast<const uint32_t*>(&p);
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
  static __device__ __forceinline__ uint32_t larger(uint32_t top, uint32_t u) {
    u &= 0x7fff7fffu;
    const __half2 p = __hmax2_nan(*reinterpret_cast<const __half2*>(&top), *reinterpret_cast<const __half2*>(&u));
    return *reinterpret_cast<const uint32_t*>(&p);
  }
  static __device__ __forceinline__ float larger_of(uint32_t top) {
    const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&top));
    return max_nan(p.x, p.y);
  }
};
template <>
struct RowVec<float> {
  static constexpr int E = 4;
  static __device__ __forceinline__ void unpack(const uint4& v, f32x2* f) {
    f[0] = pair(__uint_as_float(v.x), __uint_as_float(v.y)), f[1] = pair(__uint_as_float(v.z), __uint_as_float(v.w));
  }
  static __device__ __forceinline__ uint4 pack(const f32x2* f) {
    float a, b, c, d;
    split(f[0], a, b), split(f[1], c, d);
    return make_uint4(__float_as_uint(a), __float_as_uint(b), __float_as_uint(c), __float_as_uint(d));
  }
};

// Where a thread's values sit in its row.  Memory is accessed W bytes at a time, as wide as the rows' alignment allows; a slot is 16
// bytes of a thread, 16 / W accesses that lie `nt` threads' accesses apart, so that the lanes of a warp always touch neighbouring
// memory.  `mine` points at the thread's first value, `left` is how many values of the row lie from there to its end.
template <class T, int W>
struct RowSlot {
  using V = RowVec<T>;
  static constexpr int E = V::E, EW = W / int(sizeof(T)), S = 16 / W;
  static __device__ __forceinline__ int first(int t) { return t * EW; }
  static __device__ __forceinline__ int at(int v, int e, int nt) { return (v * S + e / EW) * nt * EW + e % EW; }
  // all E values exist; with several accesses a slot asked for all threads at once (the last thread has the fewest left)
  static __device__ __forceinline__ bool whole(int v, int t, int nt, int left) { return S == 1 ? at(v, E - 1, nt) < left : (v + 1) * S * nt * EW - first(t) <= left; }

  // access j of slot v: does it lie inside the row / does any of it
  static __device__ __forceinline__ bool inside(int v, int j, int nt, int left) { return at(v, j * EW + EW - 1, nt) < left; }
  static __device__ __forceinline__ bool touches(int v, int j, int nt, int left) { return EW > 1 && at(v, j * EW, nt) < left; }

  static __device__ __forceinline__ uint4 load(const T* mine, int v, int t, int nt, int left) {
    if constexpr (W == 16) {
      if (inside(v, 0, nt, left)) return *reinterpret_cast<const uint4*>(mine + at(v, 0, nt));
    }
    uint32_t u[4] = {0u, 0u, 0u, 0u};
    const bool all = W != 16 && whole(v, t, nt, left);
#pragma unroll
    for (int j = 0; j < S; ++j) {
      const T* const from = mine + at(v, j * EW, nt);
      if (W != 16 && (all || inside(v, j, nt, left))) {
        if constexpr (W == 8) {
          const uint2 d = *reinterpret_cast<const uint2*>(from);
          u[(2 * j) % 4] = d.x, u[(2 * j + 1) % 4] = d.y;
        } else if constexpr (W == 4) {
          u[j] = *reinterpret_cast<const uint32_t*>(from);
        } else if constexpr (W == 2) {
          u[j / 2] |= uint32_t(*reinterpret_cast<const uint16_t*>(from)) << (16 * (j % 2));
        }
      } else if (touches(v, j, nt, left)) {  // the row ends inside
        T part[EW];
#pragma unroll
        for (int e = 0; e < EW; ++e) part[e] = at(v, j * EW + e, nt) < left ? from[e] : T(0.0f);
        memcpy(reinterpret_cast<char*>(u) + j * W, part, W);
      }
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
  static __device__ __forceinline__ void store(T* mine, const uint4& w, int v, int t, int nt, int left) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    const bool all = whole(v, t, nt, left);
#pragma unroll
    for (int j = 0; j < S; ++j) {
      T* const to = mine + at(v, j * EW, nt);
      if (all || inside(v, j, nt, left)) {
        if constexpr (W == 16) *reinterpret_cast<uint4*>(to) = w;
        else if constexpr (W == 8) *reinterpret_cast<uint2*>(to) = make_uint2(u[(2 * j) % 4], u[(2 * j + 1) % 4]);
        else if constexpr (W == 4) *reinterpret_cast<uint32_t*>(to) = u[j];
        else *reinterpret_cast<uint16_t*>(to) = uint16_t(u[j / 2] >> (16 * (j % 2)));
      } else if (touches(v, j, nt, left)) {
        T part[EW];
        memcpy(part, reinterpret_cast<const char*>(u) + j * W, W);
#pragma unroll
        for (int e = 0; e < EW; ++e)
          if (at(v, j * EW + e, nt) < left) to[e] = part[e];
      }
    }
  }
  static __device__ __forceinline__ void store_q(int8_t* mine, const uint32_t* q4, int v, int t, int nt, int left) {
    const bool all = whole(v, t, nt, left);
#pragma unroll
    for (int j = 0; j < S; ++j) {
      int8_t* const to = mine + at(v, j * EW, nt);
      if (all || inside(v, j, nt, left)) {
        if constexpr (EW == 8) *reinterpret_cast<uint2*>(to) = make_uint2(q4[0], q4[1]);
        else if constexpr (EW == 4) *reinterpret_cast<uint32_t*>(to) = q4[j];
        else if constexpr (EW == 2) *reinterpret_cast<uint16_t*>(to) = uint16_t(q4[j / 2] >> (16 * (j % 2)));
        else *to = int8_t(q4[j / 4] >> (8 * (j % 4)));
      } else if (touches(v, j, nt, left)) {
#pragma unroll
        for (int e = 0; e < EW; ++e)
          if (at(v, j * EW + e, nt) < left) to[e] = int8_t(q4[(j * EW + e) / 4] >> (8 * ((j * EW + e) % 4)));
      }
    }
  }
};

// Copies of 16 bytes into shared memory that no register waits for; what lies past the row's end arrives as zeros.
__device__ __forceinline__ void copy_ahead(uint32_t to, const void* from, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_close() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A row's maximum and how its values are divided by it.
struct RowDiv {
  float amax, inv;  // inv: 127 / amax, or 1 / amax where the quotient is corrected by its remainder
  bool wide;        // zeros, values that are not finite, or too small or large for 32 bits
};

template <bool SHORT>
__device__ __forceinline__ RowDiv row_div(float top) {
  RowDiv d;
  d.amax = top;
  d.wide = !(top > 0x1p-90f && top < 0x1p118f);  // (NaN too)
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(d.inv) : "f"(top));
  if (!SHORT) d.inv *= 127.0f;
  return d;
}

template <int E>
__device__ __noinline__ void row_quantise_wide(const float* t, float amax, uint32_t* b) {
  const bool zero = !(amax > 0.0f) || !(amax < __int_as_float(0x7f800000));
#pragma unroll 1
  for (int e = 0; e < E; ++e) b[e] = zero ? 0u : uint32_t(int(rint(127.0 * double(t[e]) / double(amax))));
}

// SHORT: t has at most 11 bits (the first of the two ways above)
template <int E, bool SHORT>
__device__ __forceinline__ void row_quantise(const f32x2* t, const RowDiv& d, uint32_t* q4) {
  constexpr float MAGIC = 12582912.0f;  // 1.5 * 2^23: adding it leaves the nearest integer in the low bits
  const f32x2 magic = pair(MAGIC, MAGIC), inv = pair(d.inv, d.inv);
  uint32_t b[E];
  auto keep = [&](int i, f32x2 r) {
    float x, y;
    split(r, x, y);
    b[2 * i] = __float_as_uint(x), b[2 * i + 1] = __float_as_uint(y);
  };
  if (d.wide) {
    float c[E];
#pragma unroll
    for (int i = 0; i < E / 2; ++i) split(t[i], c[2 * i], c[2 * i + 1]);
    uint32_t n[E];
    row_quantise_wide<E>(c, d.amax, n);
#pragma unroll
    for (int e = 0; e < E; ++e) b[e] = n[e];
  } else if constexpr (SHORT) {
    const f32x2 c127 = pair(127.0f, 127.0f), minus = pair(-d.amax, -d.amax);
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      const f32x2 c = mul2(c127, t[i]), q0 = mul2(c, inv);
      keep(i, add2(fma2(fma2(q0, minus, c), inv, q0), magic));
    }
  } else {
    // (the reciprocal and its product with 127 are good to 2^-22)
    const f32x2 above = pair(d.inv * (1.0f + 0x1p-21f), d.inv * (1.0f + 0x1p-21f)), below = pair(d.inv * (1.0f - 0x1p-21f), d.inv * (1.0f - 0x1p-21f));
    uint32_t differ = 0u;
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      keep(i, fma2(t[i], above, magic));
      float x, y;
      split(fma2(t[i], below, magic), x, y);
      differ |= (__float_as_uint(x) ^ b[2 * i]) | (__float_as_uint(y) ^ b[2 * i + 1]);
    }
    if (differ != 0u) {
      float c[E];
#pragma unroll
      for (int i = 0; i < E / 2; ++i) split(t[i], c[2 * i], c[2 * i + 1]);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float n = __fadd_rn(__uint_as_float(b[e]), -MAGIC), off = __fmaf_rn(c[e], d.inv, -n);
        const float side = off < 0.0f ? -1.0f : 1.0f, half = __fmaf_rn(2.0f, n, side);  // 2 x the half way point next to t
        const float hi = __fmul_rn(half, d.amax), lo = __fmaf_rn(half, d.amax, -hi);
        const float past = __fmul_rn(__fadd_rn(__fmaf_rn(254.0f, c[e], -hi), -lo), side);
        if (fabsf(off) > 0.49f && (past > 0.0f || (past == 0.0f && (b[e] & 1u)))) b[e] += off < 0.0f ? 0xffffffffu : 1u;
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

// blockDim = (threads a row, rows a block): more than 32 threads a row only with one row a block.  NT: the threads a row where
// they are known (rows of narrow accesses: their addresses become constants), else 0.  VPT vectors of 16 bytes a thread; LOOP: rows longer
// than a block holds, read a second time (from L2) for the second half of the work.
// RING: rows of vectors that are only quantised have the loads of the next three rows out while one is reduced and written, in
// slots of shared memory that only the thread itself reads (so nothing but its own copies is waited for): with the next row in
// registers, 32 bytes a thread are in flight, too few at 6.5 TB/s (8192 x 8192, fp32 56 -> 50.5 us = 6.6 TB/s, bf16 38 -> 33.6).  With the
// norm that measured slower (16384 x 4096 bf16 45.1 -> 49.4 us, with a residual 84.7 -> 87.4; 4096 x 8192 fp32 69 -> 75): what is
// short there is instructions and registers.  SHARED_W: the norm's weights, the same for all of a block's rows, in such slots too:
// two loads a row instead of eight registers held (49 -> 45.1, fp32 71.9 -> 69.3, 40.9 -> 34.4 without a residual).
constexpr int kRowStages = 4;
template <bool NORM, int W, int VPT, bool LOOP>
constexpr bool kRowRing = !NORM && W == 16 && VPT == 2 && !LOOP;
template <bool NORM, int W, int VPT, bool LOOP>
constexpr bool kRowSharedW = NORM && W == 16 && VPT == 2 && !LOOP;
template <bool NORM>  // 16-byte words of shared memory a thread of these kernels
constexpr int kRowWords = 2 * (NORM ? 1 : kRowStages);

template <class T, bool NORM, bool RES, int W, int NT, int VPT, bool LOOP>
__global__ void __launch_bounds__(VPT <= 2 ? 1024 : 512, VPT <= 2 ? 1 : 2) rows_kernel(const RowParams p) {
  static_assert(NORM || !RES, "the residual comes with the norm");
  using S = RowSlot<T, W>;
  using V = typename S::V;
  constexpr int E = S::E, P = E / 2;
  constexpr bool SHORT = !NORM && sizeof(T) == 2, RING = kRowRing<NORM, W, VPT, LOOP>, SHARED_W = kRowSharedW<NORM, W, VPT, LOOP>;
  constexpr int STAGES = kRowStages;
  extern __shared__ uint4 row_slots[];  // RING: [stage][v][thread]; SHARED_W: [v][thread]
  __shared__ float2 part[2][32];
  // as the product's kernels: placed while the launch before ends, nothing read before it is complete
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int t = int(threadIdx.x), nt = NT ? NT : int(blockDim.x), lane = t & 31, warp = t >> 5, nw = nt >> 5;
  const int chunk = nt * VPT * E, left = p.K - S::first(t);
  const T* const w = static_cast<const T*>(p.w) + S::first(t);
  int buf = 0;

  const int block = int(blockDim.x * blockDim.y), me = int(threadIdx.y * blockDim.x) + t;
  auto slot = [&](int stage, int v) { return row_slots + (stage * VPT + v) * block + me; };
  uint4 wv[NORM && !LOOP && !SHARED_W ? VPT : 1];
  if constexpr (NORM && !LOOP) {
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      if constexpr (SHARED_W) *slot(0, v) = S::load(w, v, t, nt, left);
      else wv[v] = S::load(w, v, t, nt, left);
    }
  }
  long long row = (long long)(blockIdx.x) * blockDim.y + threadIdx.y;
  // this thread's place in the row (in the next one to be fetched, where rows are fetched ahead), moved on row by row
  const T* x = static_cast<const T*>(p.x) + row * p.ldx + S::first(t);
  const T* r = RES ? static_cast<const T*>(p.r) + row * p.ldr + S::first(t) : nullptr;
  T* h = RES ? static_cast<T*>(p.h) + row * p.ldh + S::first(t) : nullptr;
  int8_t* q = p.q + row * p.ldq + S::first(t);

  // otherwise the next row's loads are out, into registers
  uint4 nx[LOOP ? 1 : VPT], nr[!LOOP && RES ? VPT : 1];
  auto ahead = [&](int stage, bool there) {
    if constexpr (RING) {
      if (there) {
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
          const int at = S::at(v, 0, nt), bytes = max(0, min(16, (left - at) * int(sizeof(T))));
          // (nothing left: a copy of no bytes, from the row's own memory all the same)
          copy_ahead(uint32_t(__cvta_generic_to_shared(slot(stage, v))), bytes > 0 ? x + at : x - S::first(t), bytes);
        }
        x += p.step_x;
      }
      copy_close();
    }
  };
  auto fetch = [&]() {
    if constexpr (!LOOP && !RING) {
#pragma unroll
      for (int v = 0; v < VPT; ++v) {
        nx[v] = S::load(x, v, t, nt, left);
        if constexpr (RES) nr[v] = S::load(r, v, t, nt, left);
      }
      x += p.step_x;
      if constexpr (RES) r += p.step_r;
    }
  };
  int stage = 0;
  if constexpr (RING) {
    for (int i = 0; i < STAGES - 1; ++i) ahead(i, row + (long long)(i) * p.step < p.M);
  } else if (row < p.M) {
    fetch();
  }

  for (; row < p.M; row += p.step) {
    if constexpr (RING) {  // the row STAGES - 1 on goes where the last one was: its values are in registers since before the barrier
      ahead(stage == 0 ? STAGES - 1 : stage - 1, row + (long long)(STAGES - 1) * p.step < p.M);
      copy_wait<STAGES - 1>();
#pragma unroll
      for (int v = 0; v < VPT; ++v) nx[v] = *slot(stage, v);
      stage = stage + 1 == STAGES ? 0 : stage + 1;
    }
    uint4 hv[SHORT && !LOOP ? VPT : 1];           // quantise, 16-bit: the values as they are
    f32x2 tv[!SHORT && !LOOP ? VPT * P : 1];      // otherwise: t
    f32x2 sum2 = 0ull;
    float top = 0.0f;
    uint32_t top2 = 0u;
    // h of one chunk of the row (out, where there is a residual), t, the sum of squares and the maximum
    auto first = [&](int c) {
#pragma unroll
      for (int v = 0; v < VPT; ++v) {
        uint4 a;
        if constexpr (LOOP) a = S::load(x + c, v, t, nt, left - c);
        else a = nx[v];
        if constexpr (SHORT) {
          top2 = V::larger(V::larger(top2, a.x), a.y), top2 = V::larger(V::larger(top2, a.z), a.w);
          if constexpr (!LOOP) hv[v] = a;
        } else {
          f32x2 f[P];
          V::unpack(a, f);
          if constexpr (RES) {
            uint4 b;
            if constexpr (LOOP) b = S::load(r + c, v, t, nt, left - c);
            else b = nr[v];
            f32x2 g[P];
            V::unpack(b, g);
#pragma unroll
            for (int i = 0; i < P; ++i) f[i] = add2(f[i], g[i]);
            a = V::pack(f);
            S::store(h + c, a, v, t, nt, left - c);
            V::unpack(a, f);
          }
          if constexpr (NORM) {
            f32x2 g[P];
            if constexpr (LOOP) V::unpack(S::load(w + c, v, t, nt, left - c), g);
            else if constexpr (SHARED_W) V::unpack(*slot(0, v), g);
            else V::unpack(wv[v], g);
#pragma unroll
            for (int i = 0; i < P; ++i) sum2 = fma2(f[i], f[i], sum2), f[i] = mul2(f[i], g[i]);
          }
#pragma unroll
          for (int i = 0; i < P; ++i) {
            float lo, hi;
            split(f[i], lo, hi);
            top = max_nan(max_nan(top, lo), hi);
            if constexpr (!LOOP) tv[v * P + i] = f[i];
          }
        }
      }
    };
    auto second = [&](int c, const RowDiv& d) {
#pragma unroll
      for (int v = 0; v < VPT; ++v) {
        f32x2 f[P];
        if constexpr (LOOP) {
          V::unpack(S::load((RES ? h : x) + c, v, t, nt, left - c), f);
          if constexpr (NORM) {
            f32x2 g[P];
            V::unpack(S::load(w + c, v, t, nt, left - c), g);
#pragma unroll
            for (int i = 0; i < P; ++i) f[i] = mul2(f[i], g[i]);
          }
        } else if constexpr (SHORT) {
          V::unpack(hv[v], f);
        } else {
#pragma unroll
          for (int i = 0; i < P; ++i) f[i] = tv[v * P + i];
        }
        uint32_t q4[E / 4];
        row_quantise<E, SHORT>(f, d, q4);
        S::store_q(q + c, q4, v, t, nt, left - c);
      }
    };

    if constexpr (LOOP) {
      for (int c = 0; c < p.K; c += chunk) first(c);
    } else {
      first(0);
    }
    if (!LOOP && !RING && row + p.step < p.M) fetch();

    if constexpr (SHORT) top = V::larger_of(top2);
    // magnitudes order as their bits do, NaN above all
    top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
    float sum = 0.0f;
    if constexpr (NORM) {
      float lo, hi;
      split(sum2, lo, hi);
      sum = warp_sum(lo + hi);
    }
    if (nt > 32) {
      if (lane == 0) part[buf][warp] = make_float2(sum, top);
      __syncthreads();
      const float2 o = lane < nw ? part[buf][lane] : make_float2(0.0f, 0.0f);
      top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(o.y)));
      if (NORM && warp == 0) sum = warp_sum(o.x);
      buf ^= 1;
    }
    const RowDiv d = row_div<SHORT>(top);
    if (warp == 0) {  // the row's scale, by one warp alone
      float s = top / 127.0f;
      if constexpr (NORM) {
        if (!(sum > 0x1p-90f && sum < 0x1p126f) && top > 0.0f && top < __int_as_float(0x7f800000)) {
          // squares that 32 bits cannot hold (or hold with too few of them): the row again, in 64
          __syncwarp();  // a warp a row: what its lanes have just written
          double ds = 0.0;
          const T* const again = RES ? h - S::first(t) : static_cast<const T*>(p.x) + row * p.ldx;
          for (int i = lane; i < p.K; i += 32) {
            const double v = double(float(again[i]));
            ds = fma(v, v, ds);
          }
          s = float(double(top) / (127.0 * sqrt(warp_sum(ds) / p.K + double(p.eps))));
        } else {
          s = s / sqrtf(sum / float(p.K) + p.eps);
        }
      }
      if (top == 0.0f) s = 0.0f;
      if (!(top < __int_as_float(0x7f800000))) s = __int_as_float(0x7fc00000);
      if (t == 0) p.scale[row] = s;
    }

    if constexpr (LOOP) {
      for (int c = 0; c < p.K; c += chunk) second(c, d);
      x += p.step_x;
      if constexpr (RES) r += p.step_r;
    } else {
      second(0, d);
    }
    if constexpr (RES) h += p.step_h;
    q += p.step_q;
  }
}

}  // namespace wb
