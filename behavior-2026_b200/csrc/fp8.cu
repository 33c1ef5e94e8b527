// fp8.cu — the 8-bit operators of the C ABI: block quantisation, the linear layer on quantised operands, writing
// and reading an 8-bit K/V cache, attention over it.  They need no engine: each call works on the current device and
// the caller's stream and allocates nothing.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <mutex>
#include <type_traits>

#include "../../include/pi05.h"
#include "fp8.cuh"
#include "fp8_gemm.cuh"
#include "kv8_attention.cuh"
#include "kv8_attention_tc.cuh"

using namespace p5;

namespace {

int fail(char* err, size_t err_len, int code, const char* fmt, ...) {
  if (err && err_len) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(err, err_len, fmt, ap);
    va_end(ap);
  }
  return code;
}
int launched(const char* what, char* err, size_t err_len) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(err, err_len, PI05_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  return PI05_OK;
}
bool aligned(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }
// SMs of the current device; a B200's where there is none (a host that only asks for sizes)
int num_sms() {
  static std::atomic<int> known[64];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
    cudaGetLastError();
    return 148;
  }
  n = known[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) {
      cudaGetLastError();
      return 148;
    }
    known[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}
// rows of `width` elements at b * sample + t * token (token >= width): none shares an element with another, whichever axis is outer
bool apart(int batch, int T, int64_t sample, int64_t token, int64_t width) {
  return batch == 1 || sample >= token * (T - 1) + width || (sample >= width && token >= sample * (batch - 1) + width);
}

// ------------------------------------------------------------------ quantisation
// Eight lanes take a block of 128 values, 16 each, and ITEMS consecutive blocks, whose loads are all issued before the first
// block is worked on.  Measured, 61952 x 2048 bf16: 56 us, 6.75 TB/s of its 381 MB, 1.03 of
// the copy rate (8 values a lane, maxima by redux.sync over half warps: 70 us at 78 % of the issue slots); fp32 16384 x 4304 52 us, 6.75.
template <typename X, bool VEC, int ITEMS>
__global__ void __launch_bounds__(256)
    fp8_quantize_kernel(const X* x, long ldx, int cols, uint32_t blocks, uint32_t items, uint8_t* q, long ldq, uint8_t* scales,
                        long lds) {
  const int lane = threadIdx.x & 7;
  const uint32_t first = (blockIdx.x * (blockDim.x >> 3) + (threadIdx.x >> 3)) * ITEMS;
  const uint32_t row0 = first / blocks, blk0 = first - row0 * blocks;
  Fp8Raw<X> raw[ITEMS];
  uint32_t row = row0, blk = blk0;
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const int c0 = (int)blk * FP8_BLOCK + 16 * lane;
    raw[k].clear();
    if (first + k < items && c0 < cols) {
      const X* src = x + (long)row * ldx + c0;
      if (VEC)
        raw[k].load(src);
      else
        raw[k].load_some(src, min(16, cols - c0));
    }
    if (++blk == blocks) blk = 0, ++row;
  }
  row = row0, blk = blk0;
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    int byte;
    const uint4 code = fp8_encode16<8>(raw[k], byte);
    if (first + k < items) {
      const int c0 = (int)blk * FP8_BLOCK + 16 * lane;
      uint8_t* dst = q + (long)row * ldq + c0;
      if (c0 + 16 <= cols) {
        *reinterpret_cast<uint4*>(dst) = code;
      } else {
        const uint32_t w[4] = {code.x, code.y, code.z, code.w};
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (c0 + i < cols) dst[i] = (uint8_t)(w[i / 4] >> (8 * (i & 3)));
      }
      if (lane == 0) scales[(long)row * lds + blk] = (uint8_t)byte;
    }
    if (++blk == blocks) blk = 0, ++row;
  }
}

// ------------------------------------------------------------------ the cache
struct KvRows {
  const bf16 *k, *v;  // write: sources
  bf16 *ko, *vo;      // read: destinations
  long b_stride, t_stride;
  uint8_t *k8, *ks, *v8, *vs;
  const int *start, *count, *slots;
  int n_slots, capacity, batch, T, kv_heads;
};

// rows [0, n) of sample b that have a place in the cache start at position p0 (may be negative)
__device__ __forceinline__ bool kv_span(const KvRows& a, int b, int& slot, long& p0, int& n) {
  slot = a.slots ? a.slots[b] : b;
  p0 = a.start ? a.start[b] : 0;
  n = a.count ? max(0, min(a.count[b], a.T)) : a.T;
  return slot >= 0 && slot < a.n_slots;
}

// One thread a piece of VALS values of a head row, HD / VALS neighbouring lanes a row, ITEMS rows a thread with their loads issued
// together; grid (rows, batch, K | V).  Where two samples of a call name the same slot and position the later sample's
// row is kept.
template <int HD, bool WRITE, int ITEMS>
__global__ void __launch_bounds__(256) kv8_rows_kernel(const KvRows a) {
  constexpr int VALS = WRITE ? 16 : 8, LANES = HD / VALS;
  const int b = blockIdx.y;
  const int per = blockDim.x / LANES, piece = threadIdx.x % LANES;
  const long first = (long)blockIdx.x * per * ITEMS + threadIdx.x / LANES;  // head row of the sample
  const bf16* src = blockIdx.z ? a.v : a.k;
  bf16* dst = blockIdx.z ? a.vo : a.ko;
  uint8_t* codes = (blockIdx.z ? a.v8 : a.k8) + VALS * piece;
  uint8_t* bytes = blockIdx.z ? a.vs : a.ks;
  uint32_t t[ITEMS], h[ITEMS];
  long at[ITEMS];
  Fp8Raw<bf16> raw[WRITE ? ITEMS : 1];
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const uint32_t i = (uint32_t)(first + k * per);  // head rows of a sample: fewer than 2^31
    t[k] = i / (uint32_t)a.kv_heads;
    h[k] = i - t[k] * (uint32_t)a.kv_heads;
    at[k] = (long)b * a.b_stride + (long)t[k] * a.t_stride + (long)h[k] * HD + VALS * piece;
    if (WRITE) {  // on their way while the indices are read
      raw[k].clear();
      if (t[k] < (uint32_t)a.T) raw[k].load(src + at[k]);
    }
  }
  int slot, n;
  long p0;
  const bool mine = kv_span(a, b, slot, p0, n);
  bool later = false;  // a later sample names this slot: rows are compared one by one
  if (WRITE && a.slots) {
    for (int o = b + 1 + threadIdx.x; o < a.batch; o += blockDim.x) later |= a.slots[o] == slot;
    later = __syncthreads_or(later);
  }
  if (!mine) return;
  long head[ITEMS];
  bool ok[ITEMS];
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const long pos = p0 + t[k];
    ok[k] = t[k] < (uint32_t)n && pos >= 0 && pos < a.capacity;
    if (WRITE && later && ok[k]) {
      for (int o = b + 1; o < a.batch; ++o) {
        int so, no;
        long po;
        if (kv_span(a, o, so, po, no) && so == slot && pos >= po && pos < po + no) ok[k] = false;
      }
    }
    head[k] = ((long)slot * a.capacity + pos) * a.kv_heads + h[k];
  }
  if (WRITE) {
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      int byte;
      const uint4 code = fp8_encode16<LANES>(raw[k], byte);
      if (ok[k]) {
        *reinterpret_cast<uint4*>(codes + head[k] * HD) = code;
        if (piece == 0) bytes[head[k]] = (uint8_t)byte;
      }
    }
  } else {
    uint2 code[ITEMS];
    int byte[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      code[k] = ok[k] ? *reinterpret_cast<const uint2*>(codes + head[k] * HD) : make_uint2(0u, 0u);
      byte[k] = ok[k] ? bytes[head[k]] : 0;
    }
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      if (!ok[k]) continue;
      const float s = fp8_scale_value(byte[k]);
      const float2 x0 = fp8_to_f2((uint16_t)code[k].x), x1 = fp8_to_f2((uint16_t)(code[k].x >> 16));
      const float2 x2 = fp8_to_f2((uint16_t)code[k].y), x3 = fp8_to_f2((uint16_t)(code[k].y >> 16));
      *reinterpret_cast<uint4*>(dst + at[k]) = make_uint4(pack_bf2(x0.x * s, x0.y * s), pack_bf2(x1.x * s, x1.y * s),
                                                          pack_bf2(x2.x * s, x2.y * s), pack_bf2(x3.x * s, x3.y * s));
    }
  }
}

template <bool WRITE>
int kv8_rows(const char* what, const KvRows& a, int head_dim, void* stream, char* err, size_t err_len) {
  if (a.batch < 1 || a.batch > 65535 || a.T < 1 || a.kv_heads < 1 || a.n_slots < 1 || a.capacity < 1 ||
      (head_dim != 64 && head_dim != 128 && head_dim != 256))
    return fail(err, err_len, PI05_ERR_ARG,
                "%s: needs 1 <= batch <= 65535, T, kv_heads, n_slots, capacity >= 1, head_dim 64, 128 or 256", what);
  const void* x0 = WRITE ? (const void*)a.k : a.ko;
  const void* x1 = WRITE ? (const void*)a.v : a.vo;
  if (!x0 || !x1 || !a.k8 || !a.ks || !a.v8 || !a.vs || !aligned(x0, 16) || !aligned(x1, 16) || !aligned(a.k8, 16) ||
      !aligned(a.v8, 16) || a.b_stride % 8 || a.t_stride % 8 || a.t_stride < (long)a.kv_heads * head_dim || a.b_stride < 0)
    return fail(err, err_len, PI05_ERR_ARG,
                "%s: k, v and the caches must be 16-byte aligned device pointers, rows at least kv_heads * head_dim "
                "elements and a multiple of 8 apart", what);
  if (!WRITE && !apart(a.batch, a.T, a.b_stride, a.t_stride, (long)a.kv_heads * head_dim))
    return fail(err, err_len, PI05_ERR_ARG, "%s: samples of k, v overlap", what);
  // what is written must be two things: K and V rows nearer to each other than a row is long, or caches that overlap, are not
  const auto near = [](const void* p, const void* q, double bytes) {
    return (double)((uintptr_t)p > (uintptr_t)q ? (uintptr_t)p - (uintptr_t)q : (uintptr_t)q - (uintptr_t)p) < bytes;
  };
  const double heads = (double)a.n_slots * a.capacity * a.kv_heads;
  if (WRITE ? near(a.k8, a.v8, heads * head_dim) || near(a.ks, a.vs, heads) : near(x0, x1, 2.0 * a.kv_heads * head_dim))
    return fail(err, err_len, PI05_ERR_ARG, "%s: what is written for K and for V overlaps", what);
  if (!a.slots && a.batch > a.n_slots)
    return fail(err, err_len, PI05_ERR_ARG, "%s: batch exceeds the cache's slots", what);
  const long head_rows = (long)a.T * a.kv_heads;
  // several rows a thread, one where the call has too few for that to fill the machine.  Measured (16 x 4099 x 8 x 128, 404 MB):
  // writing 68 us with 16 values a thread and 2 rows (8 and 4: 95), reading 62 us with 8 and 4 (16 and 2: 71)
  constexpr int MANY = WRITE ? 2 : 4;
  const int threads = 256, per = threads / (head_dim / (WRITE ? 16 : 8));
  const bool few = head_rows * a.batch < 8L * num_sms() * per;
  const long gx = (head_rows + per * (few ? 1 : MANY) - 1) / (per * (few ? 1 : MANY));
  if (head_rows > 0x7fffffffL) return fail(err, err_len, PI05_ERR_ARG, "%s: T * kv_heads must be below 2^31", what);
  const dim3 grid((unsigned)gx, a.batch, 2);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto go = [&](auto hd) {
    constexpr int HD = decltype(hd)::value;
    if (few)
      kv8_rows_kernel<HD, WRITE, 1><<<grid, threads, 0, st>>>(a);
    else
      kv8_rows_kernel<HD, WRITE, MANY><<<grid, threads, 0, st>>>(a);
  };
  if (head_dim == 64)
    go(std::integral_constant<int, 64>());
  else if (head_dim == 128)
    go(std::integral_constant<int, 128>());
  else
    go(std::integral_constant<int, 256>());
  return launched(what, err, err_len);
}

// ------------------------------------------------------------------ linear layer
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn g_encode = nullptr;
std::mutex g_mu;
int g_sms[64];  // SMs of a device, 0 before its first call

// [rows][K] codes, rows ld bytes apart, in boxes of one 128-byte K block x box_rows
bool tmap(CUtensorMap* m, const void* base, long rows, int K, long ld, int box_rows) {
  cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld};
  cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
  cuuint32_t es[2] = {1, 1};
  return g_encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, es,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool set_smem(const void* f, int bytes) {
  return cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess;
}

// its warpgroups' register shares must fit what the block is launched with, else a share would never be granted
template <int HD>
bool attention_attributes() {
  cudaFuncAttributes f;
  return set_smem((const void*)kv8_attn_tc_kernel<HD>, Kv8TcCfg<HD>::SMEM) &&
         cudaFuncGetAttributes(&f, (const void*)kv8_attn_tc_kernel<HD>) == cudaSuccess &&
         (f.numRegs + 7) / 8 * 8 * Kv8TcCfg<HD>::THREADS >= Kv8TcCfg<HD>::REGS;
}

template <int EPI>
bool linear_attributes() {
  auto set = set_smem;
  return set((const void*)fp8_few_kernel<32, EPI>, Fp8FewCfg<32>::SMEM) &&
         set((const void*)fp8_few_kernel<64, EPI>, Fp8FewCfg<64>::SMEM) &&
         set((const void*)fp8_few_kernel<128, EPI>, Fp8FewCfg<128>::SMEM) &&
         set((const void*)fp8_pair_kernel<EPI>, Fp8PairCfg::SMEM);
}

// once per device, with that device current
int setup(char* err, size_t err_len, int* sms) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return fail(err, err_len, PI05_ERR_CUDA, "no current device");
  std::lock_guard<std::mutex> lk(g_mu);
  if (!g_sms[dev]) {
    if (!g_encode) {
      void* fn = nullptr;
      cudaDriverEntryPointQueryResult q;
      if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess || !fn ||
          q != cudaDriverEntryPointSuccess)
        return fail(err, err_len, PI05_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
      g_encode = reinterpret_cast<EncodeTiledFn>(fn);
    }
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 2 || !linear_attributes<FP8_STORE>() ||
        !linear_attributes<FP8_GELU>() || !linear_attributes<FP8_RESID>() || !linear_attributes<FP8_GATED>() ||
        !linear_attributes<FP8_GEGLU>() || !linear_attributes<FP8_F32>() ||
        !attention_attributes<64>() || !attention_attributes<128>() || !attention_attributes<256>() ||
        !set_smem((const void*)kv8_attn_rows_kernel<64>, Kv8RowsCfg<64>::SMEM) ||
        !set_smem((const void*)kv8_attn_rows_kernel<128>, Kv8RowsCfg<128>::SMEM) ||
        !set_smem((const void*)kv8_attn_rows_kernel<256>, Kv8RowsCfg<256>::SMEM))
      return fail(err, err_len, PI05_ERR_CUDA, "preparing the 8-bit kernels failed: %s", cudaGetErrorString(cudaGetLastError()));
    g_sms[dev] = n;
  }
  *sms = g_sms[dev];
  return PI05_OK;
}

cudaError_t launch_cluster(const void* fn, unsigned grid, int threads, int smem, unsigned cluster, cudaStream_t st, void** params) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = cluster;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelExC(&cfg, fn, params);
}

struct LinearPlan {
  int few_bn;  // 0: the pair kernel
  int bn, splits;
};

// Picks the kernel and its tile by an estimate of its time in microseconds, fitted to measurements of 27 shapes (tokens
// 1 to 7744, features 1024 to 32768, K 1024 to 16384; each plan forced in turn).  A K block costs an SM what its operand
// bytes take to arrive; a cluster's exchange grows with its CTAs and its tile.  E.g. 50 x 8192 x 1024: 32-token tiles 6.9, 64
// 8.1, pair kernel 11.4; 968 x 2560 x 2048: pair 11.8 (160 features), 12.9 (240), 64-token tiles 18.3; 50 x 1024 x 4096:
// one CTA a tile 13.2, clusters of four 7.4; 768 x 1152 x 4304: 128-token tiles in clusters of two 14.8, of one 18.6, pair
// 18.9; 7744 x 2048 x 16384: pair 204 (240), 262 (128), 128-token tiles 413.
LinearPlan linear_plan(int T, int F, int blocks, int sms) {
  LinearPlan best = {0, 0, 1};
  double best_cost = 1e300;
  for (int bn = 240; bn >= 128; bn -= 16) {
    const double units = (double)((T + 255) / 256) * ((F + bn - 1) / bn);
    const double cost = 5.5 + 0.012 * bn + ceil(units / (sms / 2)) * (blocks * (0.26 + 0.0005 * bn) + 0.3);
    if (cost < best_cost) best_cost = cost, best = {0, bn, 1};
  }
  for (int bn = 32; bn <= 128; bn *= 2) {
    if (bn > 32 && T <= bn / 2) break;
    const double tiles = (double)((F + 127) / 128) * ((T + bn - 1) / bn);
    const double block = bn == 32 ? 0.36 : (bn == 64 ? 0.47 : 0.42);
    for (int s = 1; s <= 8 && s <= blocks; s *= 2) {
      const double exchange = s == 1 ? 0 : (bn == 32 ? 0.3 + 0.3 * s : (bn == 64 ? 0.6 + 0.4 * s : 3.0 + 0.5 * s));
      // two CTAs of the smaller tiles share an SM, so a second one's fill and epilogue are hidden; of the largest they add up
      const double work = (blocks + s - 1) / s * block + exchange;
      const double cost = bn == 128 ? 0.2 + ceil(tiles * s / sms) * (work + 4.5) : 3.7 + std::max(1.0, tiles * s / sms) * work;
      if (cost < best_cost) best_cost = cost, best = {bn, bn, s};
    }
  }
  return best;
}

template <int BN, int EPI>
cudaError_t launch_few(Fp8Args& a, const void* x, long ldx, const void* w, long ldw, int K, cudaStream_t st, bool& mapped) {
  CUtensorMap tw, tx;
  mapped = tmap(&tw, w, a.F, K, ldw, 128) && tmap(&tx, x, a.T, K, ldx, BN);
  if (!mapped) return cudaSuccess;
  a.tiles_f = (a.F + 127) / 128;
  a.tiles_t = (a.T + BN - 1) / BN;
  void* params[] = {&tw, &tx, &a};
  return launch_cluster((const void*)fp8_few_kernel<BN, EPI>, (unsigned)((long)a.tiles_f * a.tiles_t * a.splits), 256,
                        Fp8FewCfg<BN>::SMEM, a.splits, st, params);
}

template <int EPI>
int linear(Fp8Args& a, const void* x, long ldx, const void* w, long ldw, int K, int sms, cudaStream_t st, char* err, size_t err_len) {
  const LinearPlan p = linear_plan(a.T, a.F, a.blocks, sms);
  a.splits = p.splits;
  a.bn = p.bn;
  bool mapped = true;
  cudaError_t e;
  if (p.few_bn == 32) {
    e = launch_few<32, EPI>(a, x, ldx, w, ldw, K, st, mapped);
  } else if (p.few_bn == 64) {
    e = launch_few<64, EPI>(a, x, ldx, w, ldw, K, st, mapped);
  } else if (p.few_bn == 128) {
    e = launch_few<128, EPI>(a, x, ldx, w, ldw, K, st, mapped);
  } else {
    CUtensorMap tx, tw;
    mapped = tmap(&tx, x, a.T, K, ldx, 128) && tmap(&tw, w, a.F, K, ldw, a.bn / 2);
    a.tiles_t = (a.T + 255) / 256;
    a.tiles_f = (a.F + a.bn - 1) / a.bn;
    a.group_t = std::min(a.tiles_t, 8);
    const unsigned clusters = (unsigned)std::min<long>((long)a.tiles_t * a.tiles_f, sms / 2);
    void* params[] = {&tx, &tw, &a};
    e = mapped ? launch_cluster((const void*)fp8_pair_kernel<EPI>, 2 * clusters, Fp8PairCfg::THREADS, Fp8PairCfg::SMEM, 2, st, params)
               : cudaSuccess;
  }
  if (!mapped) return fail(err, err_len, PI05_ERR_ARG, "pi05_fp8_linear: tensor map rejected the operands");
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(err, err_len, PI05_ERR_CUDA, "pi05_fp8_linear: %s", cudaGetErrorString(e));
  }
  return launched("pi05_fp8_linear", err, err_len);
}

// ------------------------------------------------------------------ attention
// what attention and the query of its workspace take
bool attention_shape(int batch, int T, int heads, int kv_heads, int head_dim, int capacity) {
  return batch >= 1 && T >= 1 && heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0 && capacity >= 1 &&
         (head_dim == 64 || head_dim == 128 || head_dim == 256) && (int64_t)batch * kv_heads <= 65535 &&
         (int64_t)T * (heads / kv_heads) <= (1 << 30) && (int64_t)batch * T <= 0x7fffffff / heads &&
         (int64_t)kv_heads * head_dim * capacity < (1LL << 40);
}

struct AttentionPlan {
  bool tc;              // kv8_attn_tc_kernel (128 rows a CTA) or kv8_attn_rows_kernel (8)
  int splits, cluster;  // key splits, CTAs of a cluster (splits is a multiple)
};

// By sizes that the host knows (the lengths are on the device): the kernel and its key splits by an estimate in microseconds of
// waves x (fixed + steps), fitted to measurements.  E.g. 1018 keys, 8 heads on one of 256: one chunk of 50 tokens
// 14.2 (rows, 2 splits), 18.2 (tc, 8 splits); 64 chunks 365 (rows), 50.6 (tc); 8 x 5 tokens 14.1 (rows), 16.7 (tc).
// Heads of 64: 8 x 500 tokens, 16 heads, 2,000 keys 322 (rows), 105 (tc); 8 x 50 tokens, 8 on 2, 1,000 keys 14.1 (rows, 1 split),
// 16.4 (tc, 1 split), 13.4 (the plan's).
AttentionPlan attention_plan(int batch, int T, int heads, int kv_heads, int head_dim, int capacity) {
  const double rows = (double)T * (heads / kv_heads), pairs = (double)batch * kv_heads;
  AttentionPlan best = {false, 1, 1};
  double best_cost = 1e300;
  const int sms = num_sms();
  {  // a step: 32 keys of one of four warps
    const double tiles = pairs * ceil(rows / 8), steps = ceil(capacity / 128.0);
    const double places = (double)sms * (head_dim == 256 ? 1 : (head_dim == 128 ? 2 : 4));
    const double step = head_dim == 256 ? 1.8 : (head_dim == 128 ? 1.0 : 0.9);
    for (int s = 1; s <= 256 && (s == 1 || s <= steps); s *= 2) {
      const double cost = ceil(tiles * s / places) * (6 + ceil(steps / s) * step) + (s > 8 ? 3 : 0);
      if (cost < best_cost) best_cost = cost, best = {false, s, s < 8 ? s : 8};
      if (tiles * s > 2 * places) break;
    }
  }
  {  // a step: 64 keys
    const double tiles = pairs * ceil(rows / 128), steps = ceil(capacity / 64.0);
    const double fixed = head_dim == 256 ? 10 : (head_dim == 128 ? 8 : 6), step = head_dim == 256 ? 0.9 : 0.65;
    for (int s = 1; s <= 64 && (s == 1 || 2 * s <= steps); s += 1 + s / 3) {
      const double cost = ceil(tiles * s / sms) * (fixed + ceil(steps / s) * step) + (s > 1 ? 3 : 0);
      if (cost < best_cost) best_cost = cost, best = {true, s, 1};
      if (tiles * s > 2 * sms) break;
    }
  }
  return best;
}

// [slots][capacity][kv_heads][head_dim] codes in boxes of 64 positions x 128 (64) bytes of one head, swizzled as wide
bool cache_map(CUtensorMap* m, const void* base, const Kv8Args& a, int head_dim) {
  const cuuint64_t head = head_dim, pos = head * a.kv_heads;
  cuuint64_t dims[4] = {head, (cuuint64_t)a.kv_heads, (cuuint64_t)a.capacity, (cuuint64_t)a.n_slots};
  cuuint64_t strides[3] = {head, pos, pos * a.capacity};
  cuuint32_t box[4] = {head_dim < 128 ? 64u : 128u, 1, 64, 1};
  cuuint32_t es[4] = {1, 1, 1, 1};
  return g_encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(base), dims, strides, box, es,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, head_dim < 128 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int HD>
int attention_tc(const Kv8Args& a, int batch, cudaStream_t st, char* err, size_t err_len) {
  CUtensorMap tk, tv;
  if (!cache_map(&tk, a.k, a, HD) || !cache_map(&tv, a.v, a, HD))
    return fail(err, err_len, PI05_ERR_ARG, "pi05_kv8_attention: tensor map rejected the cache");
  const dim3 grid((unsigned)(((long)a.T * a.G + 127) / 128), batch * a.kv_heads, a.splits);
  kv8_attn_tc_kernel<HD><<<grid, Kv8TcCfg<HD>::THREADS, Kv8TcCfg<HD>::SMEM, st>>>(tk, tv, a);
  if (a.groups > 1) {
    const long rows = (long)batch * a.T * a.heads;
    kv8_attn_combine_kernel<HD><<<(unsigned)((rows + 3) / 4), 128, 0, st>>>(a, batch);
  }
  return launched("pi05_kv8_attention", err, err_len);
}

template <int HD>
int attention(const Kv8Args& a, int batch, int cluster, cudaStream_t st, char* err, size_t err_len) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((a.T * a.G + 7) / 8, batch * a.kv_heads, a.splits);
  cfg.blockDim = dim3(32 * Kv8RowsCfg<HD>::W);
  cfg.dynamicSmemBytes = Kv8RowsCfg<HD>::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = at.val.clusterDim.y = 1;
  at.val.clusterDim.z = cluster;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  void* params[] = {const_cast<Kv8Args*>(&a)};
  const cudaError_t e = cudaLaunchKernelExC(&cfg, (const void*)kv8_attn_rows_kernel<HD>, params);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(err, err_len, PI05_ERR_CUDA, "pi05_kv8_attention: %s", cudaGetErrorString(e));
  }
  if (a.groups > 1) {
    const long rows = (long)batch * a.T * a.heads;
    kv8_attn_combine_kernel<HD><<<(unsigned)((rows + 3) / 4), 128, 0, st>>>(a, batch);
  }
  return launched("pi05_kv8_attention", err, err_len);
}

}  // namespace

extern "C" PI05_API int pi05_fp8_quantize(int64_t rows, int64_t cols, const void* x, int x_type, int64_t ldx, void* q,
                                          int64_t ldq, uint8_t* scales, int64_t ld_scales, void* stream, char* err,
                                          size_t err_len) {
  const int64_t blocks = (cols + FP8_BLOCK - 1) / FP8_BLOCK;
  if (rows < 1 || cols < 1 || cols > 0x7fffff00L || rows > 0x7fffffffL || rows * blocks > 0x7fffffffL || (x_type != 0 && x_type != 1))
    return fail(err, err_len, PI05_ERR_ARG,
                "pi05_fp8_quantize: needs rows, cols >= 1, fewer than 2^31 blocks of 128, x_type 0 (bf16) or 1 (fp32)");
  const int xb = x_type ? 4 : 2;
  if (!x || !q || !scales || !aligned(x, xb) || !aligned(q, 16) || ldq % 16 || ldx < cols || ldq < cols || ld_scales < blocks)
    return fail(err, err_len, PI05_ERR_ARG,
                "pi05_fp8_quantize: q must be 16-byte aligned with rows a multiple of 16 bytes apart, rows of x, q and "
                "scales at least cols, cols and ceil(cols / 128) elements apart");
  // 16-byte loads where every row starts on a 16-byte boundary and ends on a whole 16-value piece
  const bool vec = aligned(x, 16) && (ldx * xb) % 16 == 0 && cols % 16 == 0;
  constexpr int ITEMS = 2;
  const uint32_t items = (uint32_t)(rows * blocks), per = 256 / 8 * ITEMS;
  const unsigned grid = (items + per - 1) / per;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* q8 = static_cast<uint8_t*>(q);
  const uint32_t nb = (uint32_t)blocks;
  if (x_type == 0) {
    const bf16* xp = static_cast<const bf16*>(x);
    if (vec) fp8_quantize_kernel<bf16, true, ITEMS><<<grid, 256, 0, st>>>(xp, ldx, (int)cols, nb, items, q8, ldq, scales, ld_scales);
    else fp8_quantize_kernel<bf16, false, ITEMS><<<grid, 256, 0, st>>>(xp, ldx, (int)cols, nb, items, q8, ldq, scales, ld_scales);
  } else {
    const float* xp = static_cast<const float*>(x);
    if (vec) fp8_quantize_kernel<float, true, ITEMS><<<grid, 256, 0, st>>>(xp, ldx, (int)cols, nb, items, q8, ldq, scales, ld_scales);
    else fp8_quantize_kernel<float, false, ITEMS><<<grid, 256, 0, st>>>(xp, ldx, (int)cols, nb, items, q8, ldq, scales, ld_scales);
  }
  return launched("pi05_fp8_quantize", err, err_len);
}

extern "C" PI05_API int pi05_fp8_linear(int T, int F, int K, const void* x, int64_t ldx, const uint8_t* x_scales,
                                        int64_t ld_xs, const void* w, int64_t ldw, const uint8_t* w_scales, int64_t ld_ws,
                                        const void* bias, const void* res, const void* gate, int epi, void* out,
                                        void* stream, char* err, size_t err_len) {
  if (T < 1 || F < 1 || K < 1 || T > (1 << 24) || F > (1 << 24) || K > (1 << 24) || epi < 0 || epi > 5 || (epi == 4 && F % 2))
    return fail(err, err_len, PI05_ERR_ARG, "pi05_fp8_linear: needs 1 <= T, F, K <= 2^24, epi 0..5, an even F for epi 4");
  const int blocks = (K + FP8_BLOCK - 1) / FP8_BLOCK;
  if (!x || !x_scales || !w || !w_scales || !out || ((epi == 2 || epi == 3) && !res) || (epi == 3 && !gate))
    return fail(err, err_len, PI05_ERR_ARG, "pi05_fp8_linear: missing operand (res for epi 2 and 3, gate for epi 3)");
  if (!aligned(x, 16) || !aligned(w, 16) || ldx % 16 || ldw % 16 || ldx < K || ldw < K || !aligned(x_scales, 4) ||
      !aligned(w_scales, 4) || ld_xs % 4 || ld_ws % 4 || ld_xs < blocks || ld_ws < blocks || ldx >= (1LL << 39) || ldw >= (1LL << 39) ||
      !aligned(out, 16) || !aligned(bias, 16) || !aligned(res, 16) || !aligned(gate, 16))
    return fail(err, err_len, PI05_ERR_ARG,
                "pi05_fp8_linear: x and w must be 16-byte aligned with rows a multiple of 16 bytes apart, their scales "
                "4-byte aligned with rows a multiple of 4 bytes apart, out, bias, res and gate 16-byte aligned");
  if (((int64_t)T + 31) / 32 * (((int64_t)F + 127) / 128) > 0x0fffffff)
    return fail(err, err_len, PI05_ERR_ARG, "pi05_fp8_linear: too many output tiles");
  int sms = 0;
  const int rc = setup(err, err_len, &sms);
  if (rc != PI05_OK) return rc;
  Fp8Args a = {};
  a.xs = x_scales;
  a.ws = w_scales;
  a.ld_xs = ld_xs;
  a.ld_ws = ld_ws;
  a.bias = static_cast<const bf16*>(bias);
  a.res = static_cast<const bf16*>(res);
  a.gate = static_cast<const bf16*>(gate);
  a.out = out;
  a.T = T;
  a.F = F;
  a.blocks = blocks;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (epi) {
    case FP8_STORE: return linear<FP8_STORE>(a, x, ldx, w, ldw, K, sms, st, err, err_len);
    case FP8_GELU: return linear<FP8_GELU>(a, x, ldx, w, ldw, K, sms, st, err, err_len);
    case FP8_RESID: return linear<FP8_RESID>(a, x, ldx, w, ldw, K, sms, st, err, err_len);
    case FP8_GATED: return linear<FP8_GATED>(a, x, ldx, w, ldw, K, sms, st, err, err_len);
    case FP8_GEGLU: return linear<FP8_GEGLU>(a, x, ldx, w, ldw, K, sms, st, err, err_len);
    default: return linear<FP8_F32>(a, x, ldx, w, ldw, K, sms, st, err, err_len);
  }
}

// Waits for `stream`, then reads and clears the status word that the kernels' bounded waits write.
extern "C" PI05_API int pi05_fp8_status(void* stream, char* err, size_t err_len) {
  cudaError_t e = cudaStreamSynchronize(static_cast<cudaStream_t>(stream));
  int word = 0;
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&word, g_fp8_status, sizeof word);
  if (e != cudaSuccess) return fail(err, err_len, PI05_ERR_CUDA, "pi05_fp8_status: %s", cudaGetErrorString(e));
  if (word == 0) return PI05_OK;
  const int zero = 0;
  e = cudaMemcpyToSymbol(g_fp8_status, &zero, sizeof zero);
  if (e != cudaSuccess) return fail(err, err_len, PI05_ERR_CUDA, "pi05_fp8_status: %s", cudaGetErrorString(e));
  return fail(err, err_len, PI05_ERR_DEVICE, "pi05_fp8_*/pi05_kv8_*: a device-side wait gave up (status %d); that call's output is incomplete", word);
}

extern "C" PI05_API int pi05_kv8_write(int batch, int T, int kv_heads, int head_dim, const void* k, const void* v,
                                       int64_t sample_stride, int64_t token_stride, int n_slots, int capacity, void* k8,
                                       uint8_t* k_scales, void* v8, uint8_t* v_scales, const int32_t* start,
                                       const int32_t* count, const int32_t* slots, void* stream, char* err, size_t err_len) {
  const KvRows a = {static_cast<const bf16*>(k), static_cast<const bf16*>(v), nullptr, nullptr, sample_stride, token_stride,
                    static_cast<uint8_t*>(k8), k_scales, static_cast<uint8_t*>(v8), v_scales, start, count, slots,
                    n_slots, capacity, batch, T, kv_heads};
  return kv8_rows<true>("pi05_kv8_write", a, head_dim, stream, err, err_len);
}

extern "C" PI05_API int pi05_kv8_read(int batch, int T, int kv_heads, int head_dim, void* k, void* v, int64_t sample_stride,
                                      int64_t token_stride, int n_slots, int capacity, const void* k8,
                                      const uint8_t* k_scales, const void* v8, const uint8_t* v_scales,
                                      const int32_t* start, const int32_t* count, const int32_t* slots, void* stream,
                                      char* err, size_t err_len) {
  const KvRows a = {nullptr, nullptr, static_cast<bf16*>(k), static_cast<bf16*>(v), sample_stride, token_stride,
                    (uint8_t*)k8, (uint8_t*)k_scales, (uint8_t*)v8, (uint8_t*)v_scales, start, count, slots,
                    n_slots, capacity, batch, T, kv_heads};
  return kv8_rows<false>("pi05_kv8_read", a, head_dim, stream, err, err_len);
}

extern "C" PI05_API int64_t pi05_kv8_attention_workspace(int batch, int T, int heads, int kv_heads, int head_dim, int capacity) {
  if (!attention_shape(batch, T, heads, kv_heads, head_dim, capacity)) return PI05_ERR_ARG;
  const AttentionPlan p = attention_plan(batch, T, heads, kv_heads, head_dim, capacity);
  const int64_t groups = p.splits / p.cluster;
  return groups == 1 ? 0 : groups * batch * T * heads * ((int64_t)head_dim * 4 + 8);
}

extern "C" PI05_API int pi05_kv8_attention(int batch, int T, int heads, int kv_heads, int head_dim, const void* q,
                                           int64_t q_sample_stride, int64_t q_token_stride, int n_slots, int capacity,
                                           const void* k8, const uint8_t* k_scales, const void* v8, const uint8_t* v_scales,
                                           const int32_t* lens, const int32_t* count, const int32_t* slots, int causal, float scale,
                                           void* out,
                                           int64_t out_sample_stride, int64_t out_token_stride, void* workspace,
                                           int64_t workspace_bytes, void* stream, char* err, size_t err_len) {
  if (n_slots < 1 || !attention_shape(batch, T, heads, kv_heads, head_dim, capacity))
    return fail(err, err_len, PI05_ERR_ARG,
                "pi05_kv8_attention: needs batch, T, n_slots, capacity >= 1, heads a multiple of kv_heads, head_dim 64, 128 "
                "or 256, batch * kv_heads <= 65535, T * heads / kv_heads <= 2^30, batch * T * heads < 2^31, a slot of the cache "
                "smaller than 2^40 bytes");
  const int64_t width = (int64_t)heads * head_dim;
  if (!q || !k8 || !k_scales || !v8 || !v_scales || !lens || !out || !aligned(q, 16) || !aligned(k8, 16) || !aligned(v8, 16) ||
      !aligned(out, 16) || q_sample_stride % 8 || q_token_stride % 8 || out_sample_stride % 8 || out_token_stride % 8 ||
      q_token_stride < width || out_token_stride < width || q_sample_stride < 0 || out_sample_stride < 0 ||
      !apart(batch, T, out_sample_stride, out_token_stride, width))
    return fail(err, err_len, PI05_ERR_ARG,
                "pi05_kv8_attention: q, out and the caches must be 16-byte aligned device pointers, tokens of q and out "
                "at least heads * head_dim elements and a multiple of 8 apart, samples of out not overlapping");
  if (!slots && batch > n_slots) return fail(err, err_len, PI05_ERR_ARG, "pi05_kv8_attention: batch exceeds the cache's slots");
  if (!(scale == scale) || scale - scale != 0.f) return fail(err, err_len, PI05_ERR_ARG, "pi05_kv8_attention: scale must be finite");
  Kv8Args a = {};
  a.q = static_cast<const bf16*>(q);
  a.q_b = q_sample_stride;
  a.q_t = q_token_stride;
  a.k = static_cast<const uint8_t*>(k8);
  a.ks = k_scales;
  a.v = static_cast<const uint8_t*>(v8);
  a.vs = v_scales;
  a.lens = lens;
  a.count = count;
  a.slots = slots;
  a.out = static_cast<bf16*>(out);
  a.o_b = out_sample_stride;
  a.o_t = out_token_stride;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.n_slots = n_slots;
  a.capacity = capacity;
  a.T = T;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.G = heads / kv_heads;
  a.causal = causal != 0;
  const AttentionPlan plan = attention_plan(batch, T, heads, kv_heads, head_dim, capacity);
  a.splits = plan.splits;
  a.groups = plan.splits / plan.cluster;
  const int64_t need = pi05_kv8_attention_workspace(batch, T, heads, kv_heads, head_dim, capacity);
  if (need > 0) {
    if (!workspace || workspace_bytes < need || !aligned(workspace, 16))
      return fail(err, err_len, PI05_ERR_ARG, "pi05_kv8_attention: needs a 16-byte aligned workspace of %lld bytes", (long long)need);
    a.ws_o = static_cast<float*>(workspace);
    a.ws_ml = reinterpret_cast<float2*>(a.ws_o + (int64_t)a.groups * batch * T * heads * head_dim);
  }
  int sms = 0;
  const int rc = setup(err, err_len, &sms);
  if (rc != PI05_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (plan.tc)
    return head_dim == 64    ? attention_tc<64>(a, batch, st, err, err_len)
           : head_dim == 128 ? attention_tc<128>(a, batch, st, err, err_len)
                             : attention_tc<256>(a, batch, st, err, err_len);
  if (head_dim == 64) return attention<64>(a, batch, plan.cluster, st, err, err_len);
  if (head_dim == 128) return attention<128>(a, batch, plan.cluster, st, err, err_len);
  return attention<256>(a, batch, plan.cluster, st, err, err_len);
}
