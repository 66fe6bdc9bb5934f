// The product of 8-bit integers  Y[m, n] = sA[m] sB[n] sum_k A[m, k] Bt[n, k] (+ bias[n]),  in three forms:
//
//   i8_tile_kernel   many tokens: a tile of tokens (accumulator lanes) x channels (columns) per CTA or CTA pair, persistent
//   i8_few_kernel    few tokens: channels on the lanes, a tile of tokens as columns, K shared by the CTAs of a cluster
//   i8_gemv_kernel   one to eight tokens: no tensor cores; the weights stream through the integer dot-product lanes
//
// The tensor cores multiply with kind::i8 (32 values of K an instruction at the rate kind::f16 takes 16) and add in 32-bit
// integers: exact for K <= 131071, so how K is cut or in which order the parts are added changes nothing, and every
// launch gives the same bits.  The sum is rounded once to fp32, scaled there, and rounded once to the output type.
//
// Every launch carries the programmatic-stream-serialization attribute: a kernel may be set up (its CTAs placed, barriers and
// tensor memory made) while the launch before it in the stream ends, and waits (griddepcontrol.wait) until that launch is complete
// and its writes are visible before it touches global memory.  Stream order is what it was; what a launch costs before its first
// load is hidden behind its predecessor's tail (calls back to back: 32x8192x8192 18.3 -> 15.0 us, 512x4096x4096 14.3 -> 11.7, 2048^3
// 12.3 -> 10.3, 77x1003x1111 8.0 -> 5.3, 1x4096x4096 5.1 -> 3.6).
//
// Operand rows are 128-byte boxes of K (128 values a k-step), swizzled by the copy engine as in the fp16 kernel; K past the
// end of a row is filled with zeros by the copy engine, so any K works.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stddef.h>

#include "sm100_ptx.cuh"

namespace wb {

enum : int { I8_BF16 = 0, I8_FP16 = 1, I8_FP32 = 2 };

// status[0]: the wait that gave up (the codes of the fp16 kernel)
enum : uint32_t { I8_WAIT_EMPTY = 1, I8_WAIT_FULL = 2, I8_WAIT_ACC_EMPTY = 3, I8_WAIT_ACC_FULL = 4 };

struct I8Params {
  int M, N, K;           // tokens, channels, depth
  int kt;                // k-steps of 128
  int tiles_m, tiles_n;  // tiles of tokens and of channels
  int depth;             // ring rounds (of KSUB k-steps)
  int group;             // tile rows walked down before moving across
  int store_bytes;       // what Y's rows are aligned to: 16 (whole boxes go out through the copy engine), 8, 4 or 2
  int wk;                // gemv: warps that share a channel's K
  const int8_t* A;       // gemv reads plain memory
  const int8_t* Bt;
  long long lda, ldb, ldc;
  const float* sa;
  const float* sb;
  const float* bias;     // or null
  void* C;
  uint32_t* status;      // 4 words
  unsigned long long timeout_ns;
};

struct I8Ctrl {
  uint64_t full[16], empty[16], acc_full[2], acc_empty[2];
  uint64_t tmem_ready;  // pair leader's: the other CTA's tensor memory is allocated
  uint32_t tmem_base, abort;
};
static_assert(sizeof(I8Ctrl) <= 512, "control block");

// ---------------------------------------------------------------- waits, all bounded
WB_DEV uint32_t i8_ld_abort(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
WB_DEV void i8_st_abort(uint32_t addr) { asm volatile("st.volatile.shared.u32 [%0], 1;" ::"r"(addr) : "memory"); }

template <bool WARP>
__device__ __noinline__ bool i8_wait_timed(const I8Params& p, uint32_t abort_addr, uint32_t bar, uint32_t parity, uint32_t code, uint32_t detail) {
  const uint64_t t0 = globaltimer();
  for (;;) {
    const uint32_t ok = mbar_spin_wait<false>(bar, parity, 64);
    if (WARP ? (__all_sync(0xffffffffu, ok) != 0) : (ok != 0u)) return true;
    const uint32_t bad = i8_ld_abort(abort_addr) | ld_relaxed_gpu(p.status);
    const bool late = globaltimer() - t0 > p.timeout_ns;
    if (late && bad == 0u && atomicCAS(p.status, 0u, code) == 0u) {
      p.status[1] = detail, p.status[2] = blockIdx.x, p.status[3] = parity;
      __threadfence();
    }
    const bool stop = bad != 0u || late;
    if (WARP ? (__any_sync(0xffffffffu, stop) != 0) : stop) {
      i8_st_abort(abort_addr);
      return false;
    }
  }
}
// one lane alone: polls that return at once (a suspended try_wait wakes hundreds of cycles late)
WB_DEV bool i8_wait_lane(const I8Params& p, uint32_t abort_addr, uint32_t bar, uint32_t parity, uint32_t code, uint32_t detail) {
  for (int n = 0; n < (1 << 14); ++n)
    if (mbar_test_wait(bar, parity)) return true;
  return i8_wait_timed<false>(p, abort_addr, bar, parity, code, detail);
}
WB_DEV bool i8_wait_warp(const I8Params& p, uint32_t abort_addr, uint32_t bar, uint32_t parity, uint32_t code, uint32_t detail) {
  const uint32_t ok = mbar_spin_wait<false>(bar, parity, 1u << 12);
  if (__all_sync(0xffffffffu, ok) != 0) return true;
  return i8_wait_timed<true>(p, abort_addr, bar, parity, code, detail);
}

// ---------------------------------------------------------------- kind::i8
// instruction descriptor: 32-bit integer accumulator, both operands signed 8-bit, both K-major
constexpr uint32_t i8_idesc(int m, int n) { return (2u << 4) | (1u << 7) | (1u << 10) | (uint32_t(n >> 3) << 17) | (uint32_t(m >> 4) << 24); }
// operand tiles: K-major, 128-byte swizzle, 8-row groups 1024 bytes apart; the descriptor's low word holds the address
constexpr uint32_t I8_DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);
WB_DEV uint32_t i8_desc_lo(uint32_t addr) { return ((addr & 0x3FFFFu) >> 4) | (1u << 16); }

// One CTA's (pair's) operands of a tile: 128 rows of P a CTA on the accumulator's lanes, NT rows of Q as its columns.
// The ring is handed over KSUB k-steps at a time (a round): a k-step of four MMAs narrower than N = 256 on a pair is shorter than
// what its barriers, commit and bookkeeping cost the issuing thread.
template <int CG_, int NT_, int KSUB_>
struct I8Cfg {
  static constexpr int CG = CG_, NT = NT_, KSUB = KSUB_;
  static constexpr int Q_ROWS = NT / CG;
  static constexpr int P_BYTES = 128 * 128, Q_BYTES = Q_ROWS * 128, STAGE = P_BYTES + Q_BYTES, ROUND = KSUB * STAGE;
  static constexpr uint32_t IDESC = i8_idesc(128 * CG, NT);
  static_assert(NT % 32 == 0 && NT <= 256 && Q_BYTES % 1024 == 0, "tile");
};

// The rows that one CTA loads of an operand for a tile: its block of `box` rows, through the operand's map of whole boxes or, for the
// last rows, through one whose box is as high as they are.  A box is never asked for rows past the operand's end: those are
// zeros for the asking but not for free (48 x 5888 x 896 in 128-row boxes, 10.4 us, in 48-row ones 5.9; 16 x 5888 x 896 12.3 and 5.7: every CTA's missing rows
// are fetched from one place).  The slot's other rows hold whatever was there; nobody looks at what they are multiplied to.
struct I8Rows {
  bool last;   // through the map of the last rows
  int row, rows;
};
WB_DEV I8Rows i8_rows(int block, int size, int box) {
  const int whole = size / box, rest = size % box;
  if (block < whole) return {false, block * box, box};
  if (rest != 0 && (block == whole || whole == 0)) return {true, whole * box, rest};
  return {false, 0, box};  // no rows left for this CTA of a pair: any will do
}

// Producer, one lane: k-steps [kb, ke) of a tile, two boxes a step.  For a pair both CTAs' bytes (`rows` of them, 128 each) arrive
// on the leader's barrier.
template <class C>
WB_DEV bool i8_load(const I8Params& p, uint32_t abort_addr, uint32_t ring, uint32_t ctrl, uint32_t rank, const void* map_p, int row_p, const void* map_q,
                    int row_q, int rows, int kb, int ke, uint32_t& stage, uint32_t& phase) {
  const uint32_t full0 = ctrl + offsetof(I8Ctrl, full), empty0 = ctrl + offsetof(I8Ctrl, empty);
  const uint32_t full_to = C::CG == 2 ? mapa(full0, 0) : full0;
  const uint64_t policy = l2_policy_evict_normal();
  uint32_t left = uint32_t(ke - kb);
  int x = kb * 128;
  while (left != 0u) {
    uint32_t gave_up;
    if constexpr (C::KSUB == 1)
      gave_up = load_k_loop<C::CG, 128>(1u, left, uint32_t(p.depth), stage, phase, x, empty0, full0, full_to, rank == 0 ? 1u : 0u, uint32_t(rows * 128),
                                        ring, uint32_t(C::STAGE), uint32_t(C::P_BYTES), map_p, row_p, map_q, row_q, 1u << 14, 0u, policy);
    else
      gave_up = load_rounds<C::CG, C::KSUB, 128>(1u, left, uint32_t(p.depth), stage, phase, x, empty0, full0, full_to, rank == 0 ? 1u : 0u,
                                                 uint32_t(rows * 128), ring, uint32_t(C::ROUND), uint32_t(C::P_BYTES), map_p, row_p, map_q, row_q,
                                                 1u << 14, 0u, uint32_t(C::STAGE), policy);
    if (gave_up != 0u && !i8_wait_lane(p, abort_addr, empty0 + 8 * stage, phase ^ 1u, I8_WAIT_EMPTY, stage)) return false;
  }
  return true;
}
// Every round loaded has been handed back before the CTA leaves.
WB_DEV bool i8_load_done(const I8Params& p, uint32_t abort_addr, uint32_t ctrl, uint32_t stage, uint32_t phase) {
  for (int i = 0; i < p.depth; ++i) {
    if (!i8_wait_lane(p, abort_addr, ctrl + offsetof(I8Ctrl, empty) + 8 * stage, phase ^ 1u, I8_WAIT_EMPTY, 0x100u + stage)) return false;
    if (++stage == uint32_t(p.depth)) stage = 0, phase ^= 1u;
  }
  return true;
}

// MMA issuer, one lane (of the pair's leader): `left` k-steps of a tile into the accumulator at column d.
template <class C>
WB_DEV bool i8_mma(const I8Params& p, uint32_t abort_addr, uint32_t ring, uint32_t ctrl, uint32_t d, uint32_t left, uint32_t& stage, uint32_t& phase) {
  const uint32_t full0 = ctrl + offsetof(I8Ctrl, full), empty0 = ctrl + offsetof(I8Ctrl, empty);
  const uint32_t p_lo = i8_desc_lo(ring), q_lo = p_lo + (C::P_BYTES >> 4);
  uint32_t accumulate = 0;
  while (left != 0u) {
    uint32_t gave_up;
    if constexpr (C::KSUB == 1)
      gave_up = mma_k_loop<C::CG, 1, KIND_I8>(1u, left, uint32_t(p.depth), stage, phase, accumulate, full0, empty0, d, uint32_t(C::NT), p_lo, 0u, q_lo,
                                              uint32_t(C::STAGE >> 4), I8_DESC_HI, C::IDESC, 1u << 14);
    else
      gave_up = mma_rounds<C::CG, C::KSUB, KIND_I8>(1u, left, uint32_t(p.depth), stage, phase, accumulate, full0, empty0, d, uint32_t(C::NT), p_lo,
                                                    uint32_t(C::STAGE >> 4), q_lo, uint32_t(C::ROUND >> 4), I8_DESC_HI, C::IDESC, 1u << 14);
    if (gave_up != 0u && !i8_wait_lane(p, abort_addr, full0 + 8 * stage, phase, I8_WAIT_FULL, stage)) return false;
  }
  return true;
}

// ---------------------------------------------------------------- outputs
// A sum to its value in fp32, the same operations in every kernel (written out, so that no compiler contracts them one way
// here and another there): every program gives the same bits.
WB_DEV float i8_value(int sum, float sa, float sb) { return __fmul_rn(__fmul_rn(__int2float_rn(sum), sa), sb); }
WB_DEV float i8_value(int sum, float sa, float sb, float bias) { return __fmaf_rn(__fmul_rn(__int2float_rn(sum), sa), sb, bias); }
template <int OUT>
struct I8Out;
template <>
struct I8Out<I8_BF16> {
  using T = __nv_bfloat16;
  static WB_DEV T one(float v) { return __float2bfloat16_rn(v); }
  static WB_DEV uint32_t two(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};
template <>
struct I8Out<I8_FP16> {
  using T = __half;
  static WB_DEV T one(float v) { return __float2half_rn(v); }
  static WB_DEV uint32_t two(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};
template <>
struct I8Out<I8_FP32> {
  using T = float;
  static WB_DEV T one(float v) { return v; }
};

WB_DEV void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// ---------------------------------------------------------------- many tokens
// Warps: 0 loads, 1 multiplies (and owns the tensor memory), 2 prefetches the tensor maps, 4-11 store: two warps a quarter of the
// accumulator's lanes, half the columns each (64 columns: one, 4-7; a tile that nothing follows is stored with nothing beside it: 2048^3, one tile a
// pair, 14.9 -> 12.6 us against one warp a quarter; 4096 x 4096 x 1024 to fp32, 33.5 -> 23.8).
template <class C, int OUT>
struct I8Tile {
  static constexpr int NBUF = C::NT <= 256 ? 2 : 1;
  static constexpr int COLS = NBUF * C::NT;  // 128, 256 or 512: powers of two
  // one staging copy a warp, 32 rows of 128 bytes.  (Two, at the price of a ring stage, measured slower: 2048^3 12.6 -> 13.1 us,
  // 4096 x 4096 x 1024 to fp32 23.8 -> 24.3, 8192^3 330-341 -> 351.)
  static constexpr int COPY = 32 * 128;
  static constexpr int EPI_WARPS = C::NT == 64 ? 4 : 8, THREADS = 32 * (4 + EPI_WARPS);
  static constexpr int STAGING = EPI_WARPS * COPY;
  static constexpr int BLOCKS = C::NT / 32 / (EPI_WARPS / 4);  // of 32 columns, a storing warp's share of a tile
  static constexpr int WIDTH = OUT == I8_FP32 ? 32 : 64;       // channels a copy holds
  static_assert(BLOCKS % (WIDTH / 32) == 0, "whole copies");
  static constexpr size_t smem(int depth) { return 1024 + size_t(depth) * C::ROUND + STAGING + sizeof(I8Ctrl); }
};

// Tile number -> (tile of tokens, tile of channels): bands of `group` token tiles, down a band before across it, so that
// the tiles in flight share their operands in the L2.
WB_DEV void i8_tile_at(const I8Params& p, int tile, int& tm, int& tn) {
  const int band = tile / (p.group * p.tiles_n), first = band * p.group;
  const int rows = min(p.group, p.tiles_m - first), in = tile - first * p.tiles_n;
  tm = first + in % rows, tn = in / rows;
}

WB_DEV void i8_prefetch(const float* p) { asm volatile("prefetch.global.L1 [%0];" ::"l"(p)); }

// 32 channels' scales (and biases), from memory every lane reads alike
WB_DEV void i8_channel(const float* src, int n, int N, float* out) {
  if (n + 32 <= N) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(src + n) + i);
      out[4 * i] = v.x, out[4 * i + 1] = v.y, out[4 * i + 2] = v.z, out[4 * i + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) out[i] = n + i < N ? __ldg(src + n + i) : 0.0f;
  }
}

// A staged copy (32 rows of 128 bytes, swizzled) to rows of Y aligned to U bytes only: U bytes a lane, neighbouring lanes
// neighbouring memory, as many rows at a time as that leaves lanes for.
template <class T, int U>
WB_DEV void i8_store_rows(uint32_t copy, T* out, int m0, int M, int n0, int N, long long ldc, uint32_t lane) {
  constexpr int LANES = 128 / U < 32 ? 128 / U : 32, ROWS = 32 / LANES, E = U / int(sizeof(T)), AT_ONCE = 8;
  const uint32_t mine = lane / LANES;
#pragma unroll
  for (uint32_t byte = (lane % LANES) * U, pass = 0; pass < 128 / (LANES * U); ++pass, byte += LANES * U) {
    const int n = n0 + int(byte) / int(sizeof(T));
#pragma unroll 1
    for (uint32_t i = 0; i < 32; i += ROWS * AT_ONCE) {
      uint2 w[AT_ONCE];
#pragma unroll
      for (uint32_t j = 0; j < AT_ONCE; ++j) {
        const uint32_t row = i + j * ROWS + mine, at = copy + row * 128u + (((byte >> 4) ^ (row & 7u)) << 4) + (byte & 15u);
        if constexpr (U == 8) {
          asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[j].x), "=r"(w[j].y) : "r"(at) : "memory");
        } else if constexpr (U == 4) {
          asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[j].x) : "r"(at) : "memory");
        } else {
          uint16_t d;
          asm volatile("ld.shared.u16 %0, [%1];" : "=h"(d) : "r"(at) : "memory");
          w[j].x = d;
        }
      }
#pragma unroll
      for (uint32_t j = 0; j < AT_ONCE; ++j) {
        const int m = m0 + int(i + j * ROWS + mine);
        T* const to = out + (long long)m * ldc + n;
        if (m < M && n + E <= N) {
          if constexpr (U == 8) *reinterpret_cast<uint2*>(to) = w[j];
          else if constexpr (U == 4) *reinterpret_cast<uint32_t*>(to) = w[j].x;
          else *reinterpret_cast<uint16_t*>(to) = uint16_t(w[j].x);
        } else if (E > 1 && m < M) {  // the row ends inside
          T v[E];
          memcpy(v, &w[j], U);
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (n + e < N) to[e] = v[e];
        }
      }
    }
  }
}

template <class C, int OUT>
__global__ void __launch_bounds__(I8Tile<C, OUT>::THREADS, 1) i8_tile_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_a_last,
                                                         const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_b_last,
                                                         const __grid_constant__ CUtensorMap map_c, const __grid_constant__ I8Params p) {
  using L = I8Tile<C, OUT>;
  using T = typename I8Out<OUT>::T;
  extern __shared__ uint8_t i8_smem[];
  const uint32_t ring = (smem_u32(i8_smem) + 1023u) & ~1023u;
  const uint32_t staging = ring + uint32_t(p.depth) * uint32_t(C::ROUND), ctrl = staging + L::STAGING;
  const uint32_t abort_addr = ctrl + offsetof(I8Ctrl, abort);
  const uint32_t warp = warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31u;
  const uint32_t rank = C::CG == 2 ? cluster_ctarank() : 0u;
  const int first = int(blockIdx.x) / C::CG, step = int(gridDim.x) / C::CG, ntiles = p.tiles_m * p.tiles_n;
  griddep_launch_dependents();

  // The tensor memory is allocated after the arrival: nothing needs it before the first MMA.  The storing warps learn of it
  // at a barrier of their own, the leader's MMA lane (it writes into both CTAs') at tmem_ready.
  if (warp == 0 && lane == 0) {
    for (int i = 0; i < p.depth; ++i) mbar_init(ctrl + offsetof(I8Ctrl, full) + 8 * i, 1), mbar_init(ctrl + offsetof(I8Ctrl, empty) + 8 * i, 1);
    for (int i = 0; i < 2; ++i) mbar_init(ctrl + offsetof(I8Ctrl, acc_full) + 8 * i, 1), mbar_init(ctrl + offsetof(I8Ctrl, acc_empty) + 8 * i, L::EPI_WARPS * C::CG);
    mbar_init(ctrl + offsetof(I8Ctrl, tmem_ready), 1);
    asm volatile("st.shared.u32 [%0], 0;" ::"r"(abort_addr) : "memory");
    fence_mbar_init();
    __threadfence_block();  // the abort word too, ahead of the relaxed arrival
  }
  if (warp == 2 && lane == 0) {
    prefetch_tmap(p.M >= 128 ? &map_a : &map_a_last), prefetch_tmap(&map_b);
    if (p.store_bytes == 16) prefetch_tmap(&map_c);
  }
  __syncwarp();
  if constexpr (C::CG == 2) cluster_arrive_relaxed(), cluster_wait();
  else __syncthreads();
  if (warp == 1) {
    tmem_alloc<C::CG>(ctrl + offsetof(I8Ctrl, tmem_base), L::COLS);
    tmem_relinquish<C::CG>();
    tc_fence_before();
    named_bar_arrive(1, 32 * (L::EPI_WARPS + 1));
    if constexpr (C::CG == 2) mbar_arrive_cluster_relaxed_if(rank == 1 && lane == 0 ? 1u : 0u, mapa(ctrl + uint32_t(offsetof(I8Ctrl, tmem_ready)), 0));
  }
  if (warp >= 4) named_bar_sync(1, 32 * (L::EPI_WARPS + 1));
  griddep_wait();  // nothing in global memory has been read or written yet, and no bounded wait begun
  tc_fence_after();
  uint32_t tmem = 0;
  if (warp == 1 || warp >= 4) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(ctrl + uint32_t(offsetof(I8Ctrl, tmem_base))) : "memory");

  if (warp == 0) {
    if (lane == 0) {
      uint32_t stage = 0, phase = 0;
      bool ok = true;
      for (int tile = first; ok && tile < ntiles; tile += step) {
        int tm, tn;
        i8_tile_at(p, tile, tm, tn);
        const I8Rows a = i8_rows(tm * C::CG + int(rank), p.M, 128), b = i8_rows(tn * C::CG + int(rank), p.N, C::Q_ROWS);
        int rows = a.rows + b.rows;
        if (C::CG == 2) rows += i8_rows(tm * C::CG + 1 - int(rank), p.M, 128).rows + i8_rows(tn * C::CG + 1 - int(rank), p.N, C::Q_ROWS).rows;
        ok = i8_load<C>(p, abort_addr, ring, ctrl, rank, a.last ? &map_a_last : &map_a, a.row, b.last ? &map_b_last : &map_b, b.row, rows, 0, p.kt, stage, phase);
      }
      if (ok) i8_load_done(p, abort_addr, ctrl, stage, phase);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0 && lane == 0) {
      uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
      bool ok = C::CG == 1 || i8_wait_lane(p, abort_addr, ctrl + offsetof(I8Ctrl, tmem_ready), 0u, I8_WAIT_ACC_EMPTY, 0x200u);
      for (int tile = first; ok && tile < ntiles; tile += step) {
        ok = i8_wait_lane(p, abort_addr, ctrl + offsetof(I8Ctrl, acc_empty) + 8 * acc, acc_phase ^ 1u, I8_WAIT_ACC_EMPTY, acc);
        tc_fence_after();
        ok = ok && i8_mma<C>(p, abort_addr, ring, ctrl, tmem + acc * C::NT, uint32_t(p.kt), stage, phase);
        if (ok) umma_commit<C::CG>(ctrl + offsetof(I8Ctrl, acc_full) + 8 * acc, C::CG == 2 ? 0x3 : 0x1);
        if (++acc == L::NBUF) acc = 0, acc_phase ^= 1u;
      }
      for (int i = 0; ok && i < L::NBUF; ++i) {  // every accumulator has been read before the CTAs leave
        ok = i8_wait_lane(p, abort_addr, ctrl + offsetof(I8Ctrl, acc_empty) + 8 * acc, acc_phase ^ 1u, I8_WAIT_ACC_EMPTY, 0x100u + acc);
        if (++acc == L::NBUF) acc = 0, acc_phase ^= 1u;
      }
    }
    __syncwarp();
  } else if (warp >= 4) {
    const uint32_t q = warp & 3u, side = (warp - 4u) >> 2;  // which lanes, which half of the columns
    const uint32_t copy = staging + (warp - 4u) * L::COPY, line = copy + lane * 128u, turn = lane & 7u;
    const uint32_t release = C::CG == 2 ? mapa(ctrl + uint32_t(offsetof(I8Ctrl, acc_empty)), 0) : ctrl + uint32_t(offsetof(I8Ctrl, acc_empty));
    constexpr int BLOCKS = L::BLOCKS;
    uint32_t acc = 0, acc_phase = 0;
    T* const out = static_cast<T*>(p.C);
    for (int tile = first; tile < ntiles; tile += step) {
      int tm, tn;
      i8_tile_at(p, tile, tm, tn);
      const int m0 = (tm * C::CG + int(rank)) * 128 + int(q) * 32, n0 = tn * C::NT + int(side) * 32 * BLOCKS;
      const float sa = m0 + int(lane) < p.M ? __ldg(p.sa + m0 + lane) : 0.0f;
      if (int(lane) < BLOCKS && n0 + 32 * int(lane) < p.N) {  // a block's scales are a line
        i8_prefetch(p.sb + n0 + 32 * int(lane));
        if (p.bias != nullptr) i8_prefetch(p.bias + n0 + 32 * int(lane));
      }
      if (!i8_wait_warp(p, abort_addr, ctrl + offsetof(I8Ctrl, acc_full) + 8 * acc, acc_phase, I8_WAIT_ACC_FULL, acc)) break;
      tc_fence_after();
      const uint32_t from = tmem + acc * C::NT + side * 32u * BLOCKS + (q << 21);
      uint32_t v[2][32];
      tmem_ld_x32(from, v[0]);
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
        const int n = n0 + 32 * b, half = OUT == I8_FP32 ? 0 : b & 1;
        const bool last = b + 1 == BLOCKS;
        float s[32];
        i8_channel(p.sb, n, p.N, s);
        tmem_wait_ld();
        if (!last) {
          tmem_ld_x32(from + 32 * (b + 1), v[(b + 1) & 1]);
        } else {  // read out, as far as this warp goes: the next tile but one may have the accumulator
          tc_fence_before();
          __syncwarp();
          if constexpr (C::CG == 2) mbar_arrive_cluster_relaxed_if(lane == 0 ? 1u : 0u, release + 8 * acc);
          else mbar_arrive_if(lane == 0 ? 1u : 0u, release + 8 * acc);
        }
        if (p.bias != nullptr) {
          float add[32];
          i8_channel(p.bias, n, p.N, add);
#pragma unroll
          for (int i = 0; i < 32; ++i) s[i] = i8_value(int(v[b & 1][i]), sa, s[i], add[i]);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) s[i] = i8_value(int(v[b & 1][i]), sa, s[i]);
        }
        // into a staging copy, 16-byte pieces swizzled over a row's 128 bytes (the copy engine's 128-byte swizzle)
        if (half == 0) {  // the copy's last store has been read
          if (lane == 0) bulk_wait_read<0>();
          __syncwarp();
        }
        if constexpr (OUT == I8_FP32) {
#pragma unroll
          for (uint32_t c = 0; c < 8; ++c)
            st_shared_v4(line + ((c ^ turn) << 4), __float_as_uint(s[4 * c]), __float_as_uint(s[4 * c + 1]), __float_as_uint(s[4 * c + 2]),
                         __float_as_uint(s[4 * c + 3]));
        } else {
#pragma unroll
          for (uint32_t c = 0; c < 4; ++c)
            st_shared_v4(line + (((c + 4u * half) ^ turn) << 4), I8Out<OUT>::two(s[8 * c], s[8 * c + 1]), I8Out<OUT>::two(s[8 * c + 2], s[8 * c + 3]),
                         I8Out<OUT>::two(s[8 * c + 4], s[8 * c + 5]), I8Out<OUT>::two(s[8 * c + 6], s[8 * c + 7]));
        }
        if (OUT != I8_FP32 && half == 0) continue;
        const int nc = n0 + (OUT == I8_FP32 ? 32 * b : 32 * (b - half));
        if (p.store_bytes == 16) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (m0 < p.M && nc < p.N) tma_store_2d(&map_c, nc, m0, copy);
            bulk_commit();
          }
        } else {  // rows of Y that the copy engine cannot write
          __syncwarp();
          if (p.store_bytes == 8) i8_store_rows<T, 8>(copy, out, m0, p.M, nc, p.N, p.ldc, lane);
          else if (sizeof(T) == 4 || p.store_bytes == 4) i8_store_rows<T, 4>(copy, out, m0, p.M, nc, p.N, p.ldc, lane);
          else i8_store_rows<T, sizeof(T) == 4 ? 4 : 2>(copy, out, m0, p.M, nc, p.N, p.ldc, lane);
          __syncwarp();
        }
      }
      if (++acc == L::NBUF) acc = 0, acc_phase ^= 1u;
    }
    if (lane == 0) bulk_wait_read<0>();  // the last stores have read their copies
    __syncwarp();
  }

  __syncwarp();
  if (i8_ld_abort(abort_addr) != 0u) {  // giving up: copies and MMAs in flight land before their memory goes away
    const uint64_t t0 = globaltimer();
    while (globaltimer() - t0 < 200000ull) {
    }
  }
  // No barrier between the pair's CTAs: every word one sends the other has been waited for by a role of the other by now (the
  // loads that report to the leader by its MMA lane, the commits by both producers and the storing warps, the releases of the
  // accumulators and tmem_ready by the leader's MMA lane).
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<C::CG>(tmem, L::COLS);
  }
}

// ---------------------------------------------------------------- few tokens
// The weights' rows on the lanes (128 channels a CTA), NT tokens as columns.  The CTAs of a cluster share a tile's K; each
// sends its part of every token's sums to the CTA of the cluster that finishes that token (integers: the order of the
// additions does not matter), through shared memory, so nothing is kept in global memory between or after launches.
template <class C>
struct I8Few {
  static constexpr int COLS = C::NT < 32 ? 32 : C::NT;
  static constexpr int slice(int split) { return (C::NT + split - 1) / split; }  // tokens a CTA finishes
  static constexpr size_t parts(int split) { return size_t(split) * slice(split) * 512; }
  static constexpr size_t smem(int depth, int split) { return 1024 + size_t(depth) * C::ROUND + parts(split) + sizeof(I8Ctrl); }
};

template <class C, int OUT>
__global__ void __launch_bounds__(256) i8_few_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_a_last,
                                                     const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_b_last,
                                                     const __grid_constant__ I8Params p) {
  static_assert(C::CG == 1, "one CTA a tile");
  using L = I8Few<C>;
  using T = typename I8Out<OUT>::T;
  extern __shared__ uint8_t i8_smem[];
  griddep_launch_dependents();
  uint32_t split, rank = cluster_ctarank();
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(split));
  const int slice = (C::NT + int(split) - 1) / int(split);
  const uint32_t ring = (smem_u32(i8_smem) + 1023u) & ~1023u;
  const uint32_t parts = ring + uint32_t(p.depth) * uint32_t(C::ROUND), ctrl = parts + split * uint32_t(slice) * 512u;
  const uint32_t abort_addr = ctrl + offsetof(I8Ctrl, abort);
  const uint32_t warp = warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31u;
  const int tile = int(blockIdx.x / split), tn = tile % p.tiles_n, tm = tile / p.tiles_n;
  const int n0 = tn * 128, m0 = tm * C::NT;
  const int kb = int((long long)p.kt * rank / split), ke = int((long long)p.kt * (rank + 1) / split);  // at least one step: split <= kt

  if (warp == 0 && lane == 0) {
    for (int i = 0; i < p.depth; ++i) mbar_init(ctrl + offsetof(I8Ctrl, full) + 8 * i, 1), mbar_init(ctrl + offsetof(I8Ctrl, empty) + 8 * i, 1);
    mbar_init(ctrl + offsetof(I8Ctrl, acc_full), 1);
    asm volatile("st.shared.u32 [%0], 0;" ::"r"(abort_addr) : "memory");
    fence_mbar_init();
  }
  if (warp == 2 && lane == 0) prefetch_tmap(p.M >= C::NT ? &map_a : &map_a_last), prefetch_tmap(&map_b);
  __syncthreads();
  cluster_arrive();  // every CTA of the cluster runs before another writes into its shared memory (waited for below)
  if (warp == 1) {   // after the barrier: the first loads go out meanwhile
    tmem_alloc<1>(ctrl + offsetof(I8Ctrl, tmem_base), L::COLS);
    tmem_relinquish<1>();
    tc_fence_before();
    named_bar_arrive(1, 160);
  }
  if (warp >= 4) named_bar_sync(1, 160);
  griddep_wait();  // as in the tile kernel
  tc_fence_after();
  uint32_t tmem = 0;
  if (warp == 1 || warp >= 4) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(ctrl + uint32_t(offsetof(I8Ctrl, tmem_base))) : "memory");

  if (warp == 0) {
    if (lane == 0) {
      uint32_t stage = 0, phase = 0;
      const I8Rows a = i8_rows(tm, p.M, C::NT), b = i8_rows(tn, p.N, 128);
      if (i8_load<C>(p, abort_addr, ring, ctrl, 0u, b.last ? &map_b_last : &map_b, b.row, a.last ? &map_a_last : &map_a, a.row, a.rows + b.rows, kb, ke, stage, phase)) i8_load_done(p, abort_addr, ctrl, stage, phase);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      uint32_t stage = 0, phase = 0;
      if (i8_mma<C>(p, abort_addr, ring, ctrl, tmem, uint32_t(ke - kb), stage, phase)) umma_commit<1>(ctrl + offsetof(I8Ctrl, acc_full), 0x1);
    }
    __syncwarp();
  }
  cluster_wait();
  // what the end needs from memory, while the MMAs run: this lane's four channels, and the tokens this CTA finishes (one a lane)
  const int n = n0 + 4 * int(lane), m_first = m0 + int(rank) * slice;
  float sb[4], add[4], sa[C::NT / 32];
#pragma unroll
  for (int i = 0; i < 4; ++i) sb[i] = n + i < p.N ? __ldg(p.sb + n + i) : 0.0f, add[i] = p.bias != nullptr && n + i < p.N ? __ldg(p.bias + n + i) : 0.0f;
#pragma unroll
  for (int i = 0; i < C::NT / 32; ++i) sa[i] = m_first + 32 * i + int(lane) < p.M ? __ldg(p.sa + m_first + 32 * i + lane) : 0.0f;
  if (i8_wait_warp(p, abort_addr, ctrl + offsetof(I8Ctrl, acc_full), 0, I8_WAIT_ACC_FULL, 0)) {
    tc_fence_after();
    // all eight warps, two a quarter of the lanes, half the tokens each (warps 0-3 are done with their roles)
    constexpr int HALF = C::NT / 2;
    if (warp < 4) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(ctrl + uint32_t(offsetof(I8Ctrl, tmem_base))) : "memory");
    const uint32_t q = warp & 3u, t0 = warp < 4 ? HALF : 0;
    const int here = min(HALF, p.M - m0 - int(t0));
    // this warp's channels, in the slot that this CTA has in the CTA of the cluster that finishes the token
    const uint32_t word = rank * uint32_t(slice) * 512u + (q * 32u + lane) * 4u;
    uint32_t dest = t0 / uint32_t(slice);
    int left = slice - int(t0 % uint32_t(slice));
    uint32_t to = mapa(parts, min(dest, split - 1u)) + word + uint32_t(slice - left) * 512u;
    if (here > 0) {
      uint32_t v[HALF];
      tmem_ld<HALF>(tmem + (q << 21) + t0, v);
      tmem_wait_ld();
#pragma unroll
      for (int i = 0; i < HALF; ++i) {
        if (i < here) {
          st_cluster_u32(to, v[i]);
          to += 512u;
          if (--left == 0) left = slice, dest = min(dest + 1u, split - 1u), to = mapa(parts, dest) + word;
        }
      }
    }
    tc_fence_before();
  }
  __syncwarp();
  cluster_arrive();
  cluster_wait();
  if (i8_ld_abort(abort_addr) == 0u) {
    T* const out = static_cast<T*>(p.C);
#pragma unroll
    for (int r = 0; r < C::NT / 32; ++r) {
#pragma unroll 2
      for (int i = 32 * r + int(warp); i < min(slice, 32 * r + 32); i += 8) {
        const int m = m_first + i;
        if (int(rank) * slice + i >= C::NT || m >= p.M) break;
        int sum[4] = {0, 0, 0, 0};
        for (uint32_t s = 0; s < split; ++s) {
          int a, b, c, d;
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(a), "=r"(b), "=r"(c), "=r"(d) : "r"(parts + (s * uint32_t(slice) + uint32_t(i)) * 512u + lane * 16u) : "memory");
          sum[0] += a, sum[1] += b, sum[2] += c, sum[3] += d;
        }
        const float scale = __shfl_sync(0xffffffffu, sa[r], i & 31);
        float y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = p.bias != nullptr ? i8_value(sum[j], scale, sb[j], add[j]) : i8_value(sum[j], scale, sb[j]);
        T* const to = out + (long long)m * p.ldc + n;
        if (p.store_bytes >= 4 * int(sizeof(T)) && n + 4 <= p.N) {
          if constexpr (OUT == I8_FP32) *reinterpret_cast<float4*>(to) = make_float4(y[0], y[1], y[2], y[3]);
          else *reinterpret_cast<uint2*>(to) = make_uint2(I8Out<OUT>::two(y[0], y[1]), I8Out<OUT>::two(y[2], y[3]));
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (n + j < p.N) to[j] = I8Out<OUT>::one(y[j]);
        }
      }
    }
  }
  if (i8_ld_abort(abort_addr) != 0u) {
    const uint64_t t0 = globaltimer();
    while (globaltimer() - t0 < 200000ull) {
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<1>(tmem, L::COLS);
  }
}

// ---------------------------------------------------------------- one to eight tokens
// A warp takes R channels; its lanes take 16 bytes of K each, 512 apart; `wk` warps of the block share a channel's K.  Rows are
// 16-byte aligned and whole 16-byte pieces are read: what a row's last piece holds past K is multiplied by zeros.
template <int MT, int R, int OUT>
__global__ void __launch_bounds__(256) i8_gemv_kernel(const __grid_constant__ I8Params p) {
  using T = typename I8Out<OUT>::T;
  __shared__ int part[8][R * MT];
  griddep_launch_dependents();
  griddep_wait();
  const int warp = int(threadIdx.x >> 5), lane = int(threadIdx.x & 31u);
  const int wk = p.wk, wn = 8 / wk, kw = warp % wk, n0 = (int(blockIdx.x) * wn + warp / wk) * R;
  const int8_t* rows[R];
#pragma unroll
  for (int r = 0; r < R; ++r) rows[r] = p.Bt + (long long)min(n0 + r, p.N - 1) * p.ldb;
  int sum[R * MT];
#pragma unroll
  for (int i = 0; i < R * MT; ++i) sum[i] = 0;
#pragma unroll 2
  for (int k = (kw * 32 + lane) * 16; k < p.K; k += wk * 512) {
    int4 b[R];
#pragma unroll
    for (int r = 0; r < R; ++r) b[r] = __ldg(reinterpret_cast<const int4*>(rows[r] + k));
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      int4 a = __ldg(reinterpret_cast<const int4*>(p.A + (long long)min(m, p.M - 1) * p.lda + k));
      if (k + 16 > p.K) {
        const int left = p.K - k;  // 1 to 15 values of this piece exist
        auto keep = [&](int word, int at) { return left >= at + 4 ? word : left <= at ? 0 : word & int((1u << (8 * (left - at))) - 1u); };
        a.x = keep(a.x, 0), a.y = keep(a.y, 4), a.z = keep(a.z, 8), a.w = keep(a.w, 12);
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        int s = sum[r * MT + m];
        s = __dp4a(a.x, b[r].x, s), s = __dp4a(a.y, b[r].y, s), s = __dp4a(a.z, b[r].z, s), s = __dp4a(a.w, b[r].w, s);
        sum[r * MT + m] = s;
      }
    }
  }
  int mine = 0;  // lane i keeps sum i: channel i / MT, token i % MT
#pragma unroll
  for (int i = 0; i < R * MT; ++i) {
    const int total = __reduce_add_sync(0xffffffffu, sum[i]);
    if (lane == i) mine = total;
  }
  if (wk > 1) {
    if (lane < R * MT) part[warp][lane] = mine;
    __syncthreads();
    if (kw != 0) return;
    mine = 0;
    if (lane < R * MT)
      for (int i = 0; i < wk; ++i) mine += part[warp + i][lane];
  }
  const int n = n0 + lane / MT, m = lane % MT;
  if (lane < R * MT && n < p.N && m < p.M) {
    const float sa = __ldg(p.sa + m), sb = __ldg(p.sb + n);
    const float y = p.bias != nullptr ? i8_value(mine, sa, sb, __ldg(p.bias + n)) : i8_value(mine, sa, sb);
    static_cast<T*>(p.C)[(long long)m * p.ldc + n] = I8Out<OUT>::one(y);
  }
}

}  // namespace wb
