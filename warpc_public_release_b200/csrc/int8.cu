// C ABI of the 8-bit operators: rows to 8 bits (with or without the root-mean-square norm before it), and the product of
// 8-bit integers with a scale for each token and channel.
#include <algorithm>
#include <atomic>
#include <cstring>
#include <new>

#include "../../include/warpc_b200.h"
#include "host_cuda.h"
#include "int8_kernel.cuh"
#include "rows_kernel.cuh"

namespace {

using namespace wb;

constexpr int kSms = 148;

bool aligned(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
bool known_type(int dtype) { return dtype == WG_BF16 || dtype == WG_FP16 || dtype == WG_FP32; }
int type_size(int dtype) { return dtype == WG_FP32 ? 4 : 2; }

// One launch that may be set up while the one before it in the stream ends (the kernels wait for it before they touch global
// memory); cluster: CTAs a cluster, 0 for a launch without clusters.
int launch_kernel(const void* fn, dim3 grid, dim3 block, size_t smem, int cluster, cudaStream_t stream, void** args) {
  cudaLaunchConfig_t cfg;
  std::memset(&cfg, 0, sizeof cfg);
  cfg.gridDim = grid, cfg.blockDim = block, cfg.dynamicSmemBytes = smem, cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = unsigned(cluster), attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr, cfg.numAttrs = cluster > 0 ? 2 : 1;
  return int(cudaLaunchKernelExC(&cfg, fn, args));
}

// ------------------------------------------------------------------ rows
struct RowLaunch {
  int vpt, threads, rows, grid;
  bool loop;
};

// How a row is spread: `slots` vectors of 16 bytes.  A warp a row up to 64 of them (no barrier); else a block a row.  Rows of 16-
// or 8-byte accesses: one slot a thread where there are too few rows to fill the machine and only a row's own latency counts, two
// otherwise, and as many threads as that takes.  Rows of 4- or 2-byte accesses: 256 threads with one or two slots, then 512 or
// 1024 with two, as constants (a slot is four or eight accesses, whose addresses are constants then: 16384 x 4095 bf16 with a
// residual 232 -> 138-148 us; with 8-byte accesses the slots that stay empty cost more: 1792 x 4516 fp16 16.9 against 30.5).
// Rows beyond 2048 slots are read twice.
RowLaunch row_launch(int M, int slots, bool wide) {
  RowLaunch l;
  l.loop = slots > 2048, l.rows = 1;
  if (slots <= 64) {
    l.vpt = slots <= 32 ? 1 : 2, l.threads = 32, l.rows = M > 4 * kSms ? 8 : 1;
  } else if (l.loop) {
    l.vpt = wide ? 4 : 2, l.threads = 512;
  } else if (wide) {
    l.vpt = slots <= 1024 && M <= 2 * kSms ? 1 : 2;
    l.threads = (((slots + l.vpt - 1) / l.vpt) + 31) / 32 * 32;
  } else {
    l.vpt = slots <= 256 ? 1 : 2;
    l.threads = slots <= 512 ? 256 : slots <= 1024 ? 512 : 1024;
  }
  l.grid = int(std::min(((long long)M + l.rows - 1) / l.rows, (long long)kSms * std::max(1, 1024 / (l.threads * l.rows))));
  return l;
}

// The kernels that keep rows or weights in shared memory (kRowRing, kRowSharedW): the limit is raised once a device.
template <class T, bool NORM, bool RES>
int launch_rows_shared(const RowParams& p, const RowLaunch& l, cudaStream_t stream) {
  static std::atomic<unsigned long long> raised{0};
  const auto kernel = &rows_kernel<T, NORM, RES, 16, 0, 2, false>;
  const size_t bytes = size_t(l.threads) * l.rows * kRowWords<NORM> * 16;
  if (bytes > 32 * 1024) {  // with the kernel's own words, 48 KB need no asking
    int device = 0;
    WG_CUDA(cudaGetDevice(&device));
    const unsigned long long bit = 1ull << (device & 63);
    if (!(raised.load() & bit)) {
      WG_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 1024 * kRowWords<NORM> * 16));
      raised.fetch_or(bit);
    }
  }
  void* args[] = {const_cast<RowParams*>(&p)};
  return launch_kernel((const void*)kernel, dim3(unsigned(l.grid)), dim3(unsigned(l.threads), unsigned(l.rows)), bytes, 0, stream, args);
}

template <class T, bool NORM, bool RES, int W>
int launch_rows(RowParams p, cudaStream_t stream) {
  const RowLaunch l = row_launch(p.M, (p.K + RowVec<T>::E - 1) / RowVec<T>::E, W >= 8);
  p.step = l.grid * l.rows;
  p.step_x = p.step * p.ldx, p.step_r = p.step * p.ldr, p.step_h = p.step * p.ldh, p.step_q = p.step * p.ldq;
  const void* kernel;
  if constexpr (W >= 8) {
    if (l.loop) kernel = (const void*)rows_kernel<T, NORM, RES, W, 0, 4, true>;
    else if (l.vpt == 1) kernel = (const void*)rows_kernel<T, NORM, RES, W, 0, 1, false>;
    else if constexpr (W == 16) return launch_rows_shared<T, NORM, RES>(p, l, stream);
    else kernel = (const void*)rows_kernel<T, NORM, RES, W, 0, 2, false>;
  } else {
    if (l.loop) kernel = (const void*)rows_kernel<T, NORM, RES, W, 512, 2, true>;
    else if (l.threads == 32) kernel = l.vpt == 1 ? (const void*)rows_kernel<T, NORM, RES, W, 32, 1, false> : (const void*)rows_kernel<T, NORM, RES, W, 32, 2, false>;
    else if (l.threads == 256) kernel = l.vpt == 1 ? (const void*)rows_kernel<T, NORM, RES, W, 256, 1, false> : (const void*)rows_kernel<T, NORM, RES, W, 256, 2, false>;
    else kernel = l.threads == 512 ? (const void*)rows_kernel<T, NORM, RES, W, 512, 2, false> : (const void*)rows_kernel<T, NORM, RES, W, 1024, 2, false>;
  }
  void* args[] = {&p};
  return launch_kernel(kernel, dim3(unsigned(l.grid)), dim3(unsigned(l.threads), unsigned(l.rows)), 0, 0, stream, args);
}

// The widest access that every row of every operand is aligned to.
template <class T, bool NORM, bool RES>
int launch_rows_as(const RowParams& p, cudaStream_t stream) {
  auto fits = [&](unsigned width) {
    auto rows = [&](const void* at, long long ld) { return aligned(at, width) && (p.M == 1 || (ld * int(sizeof(T))) % width == 0); };
    const unsigned bytes = width / unsigned(sizeof(T));  // of q
    return rows(p.x, p.ldx) && aligned(p.q, bytes) && (p.M == 1 || p.ldq % bytes == 0) && (!NORM || aligned(p.w, width)) &&
           (!RES || (rows(p.r, p.ldr) && rows(p.h, p.ldh)));
  };
  if (fits(16)) return launch_rows<T, NORM, RES, 16>(p, stream);
  if (fits(8)) return launch_rows<T, NORM, RES, 8>(p, stream);
  if (sizeof(T) == 4 || fits(4)) return launch_rows<T, NORM, RES, 4>(p, stream);
  return launch_rows<T, NORM, RES, sizeof(T) == 4 ? 4 : 2>(p, stream);
}

template <bool NORM, bool RES>
int launch_rows_of(int dtype, const RowParams& p, cudaStream_t stream) {
  switch (dtype) {
    case WG_BF16: return launch_rows_as<__nv_bfloat16, NORM, RES>(p, stream);
    case WG_FP16: return launch_rows_as<__half, NORM, RES>(p, stream);
    default: return launch_rows_as<float, NORM, RES>(p, stream);
  }
}

// ------------------------------------------------------------------ the product
struct I8Plan {
  int device = 0, N = 0, K = 0, out = 0;
  const int8_t* Bt = nullptr;
  long long ldb = 0;
  const float *sb = nullptr, *bias = nullptr;
  CUtensorMap map_b128, map_b64;            // the weights in boxes of 128 and of 64 rows
  CUtensorMap map_b128_last, map_b64_last;  // and their last rows, fewer than that, in one box
  uint32_t* d_status = nullptr;
  unsigned long long timeout_ns = 2000ull * 1000ull * 1000ull;
  wg_int8_info named{};  // the program a caller named, or kernel 0
};

int encode_rows(CUtensorMap* map, CUtensorMapDataType type, int size, const void* ptr, long long rows, long long cols, long long ld, int box_rows) {
  EncodeTiledFn enc = encode_tiled();
  if (!enc) return WG_E_NODRIVER;
  cuuint64_t dims[2] = {cuuint64_t(cols), cuuint64_t(rows)};
  cuuint64_t strides[1] = {cuuint64_t(ld) * cuuint64_t(size)};
  cuuint32_t box[2] = {cuuint32_t(128 / size), cuuint32_t(box_rows)}, estr[2] = {1, 1};
  if (box_rows == 0) {  // no such rows: a map that nothing loads through
    std::memset(map, 0, sizeof *map);
    return WG_OK;
  }
  const CUresult r = enc(map, type, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? WG_OK : int(r);
}

constexpr size_t kI8MaxSmem = 232448;
constexpr int kI8MaxDepth = 16;

// ring rounds that fit beside `fixed` bytes
int ring_depth(size_t fixed, size_t round, int most) { return int(std::min<size_t>(size_t(std::min(most, kI8MaxDepth)), (kI8MaxSmem - fixed) / round)); }

// k-steps a round (I8Cfg)
constexpr int kFewKsub = 2;
constexpr int tile_ksub(int tile_m, int tile_n) { return tile_m == 256 && tile_n == 256 ? 1 : 2; }
template <int TILE_M, int TILE_N>
using TileCfg = I8Cfg<TILE_M / 128, TILE_N, tile_ksub(TILE_M, TILE_N)>;
template <int TILE_M>
using FewCfg = I8Cfg<1, TILE_M, kFewKsub>;

// The launch of a named program; WG_E_VARIANT where there is none.
int i8_derive(int M, int N, int K, wg_int8_info* o) {
  const int kt = (K + 127) / 128;
  auto up = [](int a, int b) { return int(((long long)a + b - 1) / b); };
  o->threads = 256, o->depth = 0, o->dynsmem = 0, o->cluster = 1;
  if (o->kernel == WG_INT8_GEMV) {
    if (o->tile_m != 1 && o->tile_m != 2 && o->tile_m != 4 && o->tile_m != 8) return WG_E_VARIANT;
    if (M > o->tile_m) return WG_E_VARIANT;
    if (o->split != 1 && o->split != 2 && o->split != 4 && o->split != 8) return WG_E_VARIANT;
    o->tile_n = 4 * (8 / o->split), o->tiles = up(N, o->tile_n), o->grid = o->tiles;
    return WG_OK;
  }
  if (o->kernel == WG_INT8_FEW) {
    if ((o->tile_m != 32 && o->tile_m != 64) || o->tile_n != 128) return WG_E_VARIANT;
    if ((o->split != 1 && o->split != 2 && o->split != 4 && o->split != 8) || o->split > kt) return WG_E_VARIANT;
    const size_t round = kFewKsub * size_t(128 + o->tile_m) * 128, fixed = 1024 + sizeof(I8Ctrl) + size_t(o->split) * up(o->tile_m, o->split) * 512;
    // (two CTAs an SM, each with half the ring, where there are more tiles than SMs: 32x28672x8192 46.7 -> 49.0 us, 32x40000x4096 42 -> 48)
    o->depth = ring_depth(fixed, round, std::max(2, up(up(kt, o->split), kFewKsub)));
    o->dynsmem = int(fixed + o->depth * round), o->cluster = o->split;
    const long long tiles = (long long)up(M, o->tile_m) * up(N, 128);
    if (tiles * o->split > 0x7fffffffll) return WG_E_LIMIT;
    o->tiles = int(tiles), o->grid = o->tiles * o->split;
    return WG_OK;
  }
  if (o->kernel == WG_INT8_TILE) {
    const int cg = o->tile_m / 128;
    const bool known = (o->tile_m == 256 && (o->tile_n == 256 || o->tile_n == 128)) || (o->tile_m == 128 && (o->tile_n == 128 || o->tile_n == 64));
    if (!known || o->split != 1) return WG_E_VARIANT;
    const size_t round = tile_ksub(o->tile_m, o->tile_n) * size_t(128 + o->tile_n / cg) * 128, fixed = 1024 + sizeof(I8Ctrl) + (o->tile_n == 64 ? 4 : 8) * 4096;
    o->threads = o->tile_n == 64 ? 256 : 384;
    o->depth = ring_depth(fixed, round, 8);
    o->dynsmem = int(fixed + o->depth * round), o->cluster = cg;
    const long long tiles = (long long)up(M, o->tile_m) * up(N, o->tile_n);
    if (tiles > 0x3fffffffll) return WG_E_LIMIT;
    o->tiles = int(tiles), o->grid = cg * std::min(o->tiles, kSms / cg);
    return WG_OK;
  }
  return WG_E_VARIANT;
}

// Which program, by estimated microseconds: what a launch costs besides its k-steps, plus its k-steps, as measured on a B200 with
// launches back to back.
//   gemv   1.7 us, and 0.2 / 0.3 / 0.5 / 0.9 us a megabyte of weights for 1 / 2 / 4 / 8 tokens (2048 x 2048: 2.9 / 3.2 / 4.0 / 6.1)
//   few    512 channels, 32 tokens: 3.7 us with one k-step, 9.9 with 32, 5.2 with 32 shared by four CTAs; 64 tokens: 4.9, 11.4, 5.9;
//          weights out of memory rather than the L2 add 0.11 us a megabyte
//   tile   256 x 512 with one k-step / 32: 128 x 64 3.5 / 10.4, 128 x 128 3.9 / 13.5, 256 x 128 3.9 / 11.2, 256 x 256 4.9 / 14.3 (more
//          a k-step with every SM at work); of several tiles each takes the slower of its k-steps and its store (4096 x 4096 x 1024);
//          rows of Y that the copy engine cannot write: 0.7, 0.8, 0.8, 2.2 a tile
// Clusters that run at once (a GPC holds a whole number of them): 74 of two CTAs, 33 of four, 15 of eight.
int i8_choose(int M, int N, int K, bool aligned, wg_int8_info* o) {
  std::memset(o, 0, sizeof *o);
  const int kt = (K + 127) / 128;
  auto up = [](long long a, long long b) { return (a + b - 1) / b; };
  const double megabytes = double(N) * K * 1e-6;
  double best = 1e300;
  auto take = [&](double cost, int kernel, int tile_m, int tile_n, int split) {
    if (cost < best) best = cost, o->kernel = kernel, o->tile_m = tile_m, o->tile_n = tile_n, o->split = split;
  };
  if (M <= 8) {
    const int t = M <= 1 ? 0 : M <= 2 ? 1 : M <= 4 ? 2 : 3;
    static const double mb[] = {0.2, 0.3, 0.5, 0.9};
    // four channels a warp: warps enough to keep the loads of a whole machine in flight, each with 512 values of K at least
    int wk = 1;
    while (wk < 8 && up(N, 4) * wk < (M <= 1 ? 4096 : 2048) && K > 512 * wk) wk *= 2;
    take(1.7 + megabytes * mb[t], WG_INT8_GEMV, 1 << t, 0, wk);
  }
  for (int t = 32; t <= 64; t *= 2)
    for (int s = 1; s <= 8 && s <= kt; s *= 2) {
      static const int at_once[] = {0, 148, 74, 0, 33, 0, 0, 0, 15};
      const double waves = double(up(up(M, t) * up(N, 128), at_once[s])), steps = double(up(kt, s));
      take(waves * (t == 32 ? 3.2 + 0.3 / s + 0.2 * steps : 3.6 + 1.1 / s + 0.22 * steps) + 0.11 * megabytes, WG_INT8_FEW, t, 128, s);
    }
  static const struct { int m, n; double launch, step, store, scattered; } tiles[] = {
      {256, 256, 4.7, 0.35, 3.1, 2.2}, {256, 128, 3.7, 0.235, 2.3, 0.8}, {128, 128, 3.6, 0.29, 2.8, 0.8}, {128, 64, 3.2, 0.21, 2.1, 0.7}};
  for (const auto& t : tiles) {
    const double each = double(up(up(M, t.m) * up(N, t.n), kSms / (t.m / 128))), store = t.store + (aligned ? 0.0 : t.scattered);
    take(t.launch + t.step * kt + (each - 1) * std::max(t.step * kt, store) + (aligned ? 0.0 : t.scattered) + 0.11 * megabytes, WG_INT8_TILE, t.m, t.n, 1);
  }
  return i8_derive(M, N, K, o);
}

int launch(const void* fn, const wg_int8_info& li, cudaStream_t stream, void** args) {
  return launch_kernel(fn, dim3(unsigned(li.grid)), dim3(unsigned(li.threads)), size_t(li.dynsmem), li.kernel == WG_INT8_GEMV ? 0 : li.cluster, stream, args);
}

// The kernels of one output type; `set_up` raises their shared-memory limit instead of launching.
template <int OUT>
struct I8Kernels {
  static int set_up() {
    const void* fns[] = {(const void*)i8_tile_kernel<TileCfg<256, 256>, OUT>, (const void*)i8_tile_kernel<TileCfg<256, 128>, OUT>,
                         (const void*)i8_tile_kernel<TileCfg<128, 128>, OUT>, (const void*)i8_tile_kernel<TileCfg<128, 64>, OUT>,
                         (const void*)i8_few_kernel<FewCfg<32>, OUT>,   (const void*)i8_few_kernel<FewCfg<64>, OUT>};
    for (const void* fn : fns) WG_CUDA(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kI8MaxSmem)));
    return WG_OK;
  }
  static int run(const wg_int8_info& li, cudaStream_t stream, CUtensorMap* a, CUtensorMap* a_last, CUtensorMap* b, CUtensorMap* b_last, CUtensorMap* c, I8Params* p) {
    if (li.kernel == WG_INT8_GEMV) {
      void* args[] = {p};
      switch (li.tile_m) {
        case 1: return launch((const void*)i8_gemv_kernel<1, 4, OUT>, li, stream, args);
        case 2: return launch((const void*)i8_gemv_kernel<2, 4, OUT>, li, stream, args);
        case 4: return launch((const void*)i8_gemv_kernel<4, 4, OUT>, li, stream, args);
        default: return launch((const void*)i8_gemv_kernel<8, 4, OUT>, li, stream, args);
      }
    }
    if (li.kernel == WG_INT8_FEW) {
      void* args[] = {a, a_last, b, b_last, p};
      return li.tile_m == 32 ? launch((const void*)i8_few_kernel<FewCfg<32>, OUT>, li, stream, args) : launch((const void*)i8_few_kernel<FewCfg<64>, OUT>, li, stream, args);
    }
    void* args[] = {a, a_last, b, b_last, c, p};
    if (li.tile_m == 256) return li.tile_n == 256 ? launch((const void*)i8_tile_kernel<TileCfg<256, 256>, OUT>, li, stream, args) : launch((const void*)i8_tile_kernel<TileCfg<256, 128>, OUT>, li, stream, args);
    return li.tile_n == 128 ? launch((const void*)i8_tile_kernel<TileCfg<128, 128>, OUT>, li, stream, args) : launch((const void*)i8_tile_kernel<TileCfg<128, 64>, OUT>, li, stream, args);
  }
};

constexpr int kMaxK = 131071;     // 128 * 128 * K stays below 2^31
constexpr int kMaxSize = 1 << 30;  // tokens, channels, values a row: a tile past the end is still an int

}  // namespace

extern "C" int wg_quantise_rows(int device, int M, int K, int dtype, const void* dX, long long ldx, signed char* dQ, long long ldq, float* dScale,
                                void* cuda_stream) {
  if (!known_type(dtype) || M < 0 || K <= 0 || ldx < K || ldq < K) return WG_E_ARG;
  if (K > kMaxSize) return WG_E_LIMIT;
  if (M == 0) return WG_OK;
  if (!dX || !dQ || !dScale || !aligned(dX, unsigned(type_size(dtype))) || !aligned(dScale, 4)) return WG_E_ARG;
  RowParams p;
  std::memset(&p, 0, sizeof p);
  p.x = dX, p.q = reinterpret_cast<int8_t*>(dQ), p.scale = dScale, p.ldx = ldx, p.ldq = ldq, p.M = M, p.K = K;
  WG_ON_DEVICE(device);
  return launch_rows_of<false, false>(dtype, p, static_cast<cudaStream_t>(cuda_stream));
}

extern "C" int wg_norm_quantise_rows(int device, int M, int K, int dtype, const void* dX, long long ldx, const void* dR, long long ldr, const void* dW,
                                     float eps, void* dH, long long ldh, signed char* dQ, long long ldq, float* dScale, void* cuda_stream) {
  if (!known_type(dtype) || M < 0 || K <= 0 || ldx < K || ldq < K || !(eps >= 0.0f)) return WG_E_ARG;
  if ((dR == nullptr) != (dH == nullptr) || (dR && (ldr < K || ldh < K))) return WG_E_ARG;
  if (K > kMaxSize) return WG_E_LIMIT;
  if (M == 0) return WG_OK;
  const unsigned size = unsigned(type_size(dtype));
  if (!dX || !dW || !dQ || !dScale || !aligned(dX, size) || !aligned(dW, size) || !aligned(dR, size) || !aligned(dH, size) || !aligned(dScale, 4))
    return WG_E_ARG;
  if ((dH == dX && ldh != ldx) || (dH && dH == dR && ldh != ldr)) return WG_E_ARG;
  RowParams p;
  std::memset(&p, 0, sizeof p);
  p.x = dX, p.r = dR, p.w = dW, p.h = dH, p.q = reinterpret_cast<int8_t*>(dQ), p.scale = dScale;
  p.ldx = ldx, p.ldr = ldr, p.ldh = ldh, p.ldq = ldq, p.M = M, p.K = K, p.eps = eps;
  WG_ON_DEVICE(device);
  const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  return dR ? launch_rows_of<true, true>(dtype, p, stream) : launch_rows_of<true, false>(dtype, p, stream);
}

extern "C" int wg_int8_choose(int M, int N, int K, wg_int8_info* out) {
  if (!out || M <= 0 || N <= 0 || K <= 0) return WG_E_ARG;
  if (K > kMaxK || M > kMaxSize || N > kMaxSize) return WG_E_LIMIT;
  return i8_choose(M, N, K, true, out);
}

extern "C" int wg_int8_plan_create(int device, int N, int K, const signed char* dBt, long long ldb, const float* dScaleB, const float* dBias, int out_dtype,
                                   void** plan) {
  if (!plan) return WG_E_ARG;
  *plan = nullptr;
  if (!known_type(out_dtype) || N <= 0 || K <= 0 || ldb < K || ldb % 16 != 0) return WG_E_ARG;
  if (!dBt || !dScaleB || !aligned(dBt, 16) || !aligned(dScaleB, 16) || !aligned(dBias, 16)) return WG_E_ARG;
  if (K > kMaxK || N > kMaxSize) return WG_E_LIMIT;
  WG_ON_DEVICE(device);
  I8Plan* pl = new (std::nothrow) I8Plan();
  if (!pl) return WG_E_ARG;
  pl->device = device, pl->N = N, pl->K = K, pl->out = out_dtype;
  pl->Bt = reinterpret_cast<const int8_t*>(dBt), pl->ldb = ldb, pl->sb = dScaleB, pl->bias = dBias;
  int r = encode_rows(&pl->map_b128, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, dBt, N, K, ldb, 128);
  if (r == WG_OK) r = encode_rows(&pl->map_b64, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, dBt, N, K, ldb, 64);
  if (r == WG_OK) r = encode_rows(&pl->map_b128_last, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, dBt, N, K, ldb, N % 128);
  if (r == WG_OK) r = encode_rows(&pl->map_b64_last, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, dBt, N, K, ldb, N % 64);
  if (r == WG_OK) r = int(cudaMalloc(&pl->d_status, 4 * sizeof(uint32_t)));
  if (r == WG_OK) r = int(cudaMemsetAsync(pl->d_status, 0, 4 * sizeof(uint32_t), 0));
  if (r == WG_OK) r = int(cudaStreamSynchronize(0));  // zero before any stream, blocking or not, can launch on the plan
  if (r == WG_OK) r = out_dtype == WG_BF16 ? I8Kernels<I8_BF16>::set_up() : out_dtype == WG_FP16 ? I8Kernels<I8_FP16>::set_up() : I8Kernels<I8_FP32>::set_up();
  if (r != WG_OK) {
    wg_int8_plan_destroy(pl);
    return r;
  }
  *plan = pl;
  return WG_OK;
}

extern "C" int wg_int8_plan_set_program(void* plan, const wg_int8_info* program) {
  I8Plan* pl = static_cast<I8Plan*>(plan);
  if (!pl) return WG_E_ARG;
  wg_int8_info named;
  std::memset(&named, 0, sizeof named);
  if (program) {
    named.kernel = program->kernel, named.tile_m = program->tile_m, named.tile_n = program->tile_n, named.split = program->split;
    wg_int8_info probe = named;
    const int r = i8_derive(1, pl->N, pl->K, &probe);
    if (r != WG_OK) return r;
  }
  pl->named = named;
  return WG_OK;
}

extern "C" int wg_int8_plan_set_timeout_ms(void* plan, unsigned ms) {
  I8Plan* pl = static_cast<I8Plan*>(plan);
  if (!pl) return WG_E_ARG;
  pl->timeout_ns = (ms ? ms : 2000u) * 1000000ull;
  return WG_OK;
}

extern "C" int wg_int8_launch(void* plan, int M, const signed char* dA, long long lda, const float* dScaleA, void* dC, long long ldc, void* cuda_stream) {
  I8Plan* pl = static_cast<I8Plan*>(plan);
  if (!pl || M < 0) return WG_E_ARG;
  const int size = type_size(pl->out);
  if (lda < pl->K || lda % 16 != 0 || ldc < pl->N) return WG_E_ARG;
  if (M > kMaxSize) return WG_E_LIMIT;
  if (M == 0) return WG_OK;
  if (!dA || !dScaleA || !dC || !aligned(dA, 16) || !aligned(dScaleA, 4) || !aligned(dC, unsigned(size))) return WG_E_ARG;
  int store_bytes = 16;  // what the rows of C are aligned to
  while (store_bytes > size && !(aligned(dC, unsigned(store_bytes)) && (ldc * size) % store_bytes == 0)) store_bytes /= 2;
  wg_int8_info li = pl->named;
  int r = li.kernel ? i8_derive(M, pl->N, pl->K, &li) : i8_choose(M, pl->N, pl->K, store_bytes == 16, &li);
  if (r != WG_OK) return r;
  I8Params p;
  std::memset(&p, 0, sizeof p);
  p.M = M, p.N = pl->N, p.K = pl->K, p.kt = (pl->K + 127) / 128;
  p.tiles_m = int(((long long)M + li.tile_m - 1) / li.tile_m), p.tiles_n = (pl->N + li.tile_n - 1) / li.tile_n;
  p.depth = li.depth, p.group = 8, p.wk = li.split;
  p.A = reinterpret_cast<const int8_t*>(dA), p.Bt = pl->Bt, p.lda = lda, p.ldb = pl->ldb, p.ldc = ldc;
  p.sa = dScaleA, p.sb = pl->sb, p.bias = pl->bias, p.C = dC, p.status = pl->d_status, p.timeout_ns = pl->timeout_ns;
  p.store_bytes = store_bytes;
  WG_ON_DEVICE(pl->device);
  CUtensorMap map_a, map_a_last, map_c;
  std::memset(&map_a, 0, sizeof map_a), std::memset(&map_a_last, 0, sizeof map_a_last), std::memset(&map_c, 0, sizeof map_c);
  const bool b64 = li.kernel == WG_INT8_TILE && li.tile_n / li.cluster == 64;
  CUtensorMap *map_b = b64 ? &pl->map_b64 : &pl->map_b128, *map_b_last = b64 ? &pl->map_b64_last : &pl->map_b128_last;
  if (li.kernel != WG_INT8_GEMV) {
    const int box = li.kernel == WG_INT8_FEW ? li.tile_m : 128;
    if (M >= box && (r = encode_rows(&map_a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, dA, M, pl->K, lda, box)) != WG_OK) return r;
    if ((r = encode_rows(&map_a_last, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, dA, M, pl->K, lda, M % box)) != WG_OK) return r;
  }
  if (li.kernel == WG_INT8_TILE && p.store_bytes == 16) {
    const CUtensorMapDataType type = pl->out == WG_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : pl->out == WG_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
    if ((r = encode_rows(&map_c, type, size, dC, M, pl->N, ldc, 32)) != WG_OK) return r;
  }
  const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  switch (pl->out) {
    case WG_BF16: return I8Kernels<I8_BF16>::run(li, stream, &map_a, &map_a_last, map_b, map_b_last, &map_c, &p);
    case WG_FP16: return I8Kernels<I8_FP16>::run(li, stream, &map_a, &map_a_last, map_b, map_b_last, &map_c, &p);
    default: return I8Kernels<I8_FP32>::run(li, stream, &map_a, &map_a_last, map_b, map_b_last, &map_c, &p);
  }
}

extern "C" int wg_int8_last_device_status(void* plan, unsigned out[4]) {
  I8Plan* pl = static_cast<I8Plan*>(plan);
  if (!pl || !out) return WG_E_ARG;
  WG_ON_DEVICE(pl->device);
  WG_CUDA(cudaDeviceSynchronize());
  WG_CUDA(cudaMemcpy(out, pl->d_status, 4 * sizeof(uint32_t), cudaMemcpyDeviceToHost));
  return out[0] == 0 ? WG_OK : WG_E_DEVICE_WAIT;
}

extern "C" int wg_int8_plan_reset(void* plan) {
  I8Plan* pl = static_cast<I8Plan*>(plan);
  if (!pl) return WG_E_ARG;
  WG_ON_DEVICE(pl->device);
  WG_CUDA(cudaDeviceSynchronize());
  WG_CUDA(cudaMemset(pl->d_status, 0, 4 * sizeof(uint32_t)));
  return WG_OK;
}

extern "C" int wg_int8_plan_destroy(void* plan) {
  I8Plan* pl = static_cast<I8Plan*>(plan);
  if (!pl) return WG_OK;
  DeviceGuard guard(pl->device);
  if (pl->d_status) cudaFree(pl->d_status);
  delete pl;
  return WG_OK;
}
