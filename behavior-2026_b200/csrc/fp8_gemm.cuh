// fp8_gemm.cuh — the linear layer on block-quantised operands (fp8.cuh) on the 5th-generation tensor cores:
//   y[t][f] = sum over blocks b of 2^(xs[t][b] + ws[f][b] - 254) sum_{k in b} x[t][k] w[f][k],  out = epilogue(y)
//
// tcgen05.mma kind::mxf8f6f4 multiplies e4m3 by e4m3 at twice the bf16 rate and applies a power-of-two scale to each
// row of either operand for every 32 values of K by itself, so the 128-wide blocks cost no pass over the accumulator:
// the four K = 32 steps of a block name the same scale.  The scales are read from tensor memory: for the rows 32 j + i of
// an operand, lane i (the same in each of the four 32-lane quarters) of column j holds one 32-bit word whose four bytes are
// the row's scales of four consecutive blocks, and the instruction descriptor names the byte.  Such a word is what four
// consecutive bytes of the caller's scale rows are, so four warps, one for each lane quarter, load the words and
// tcgen05.st them, a "chunk" of four blocks (512 of K) at a time.
#pragma once
#include "fp8.cuh"

namespace p5 {

// device-side status of this file's bounded waits (0: none gave up)
__device__ int g_fp8_status;

struct Fp8Args {
  const uint8_t *xs, *ws;  // scales: [T][ld_xs], [F][ld_ws]
  long ld_xs, ld_ws;
  const bf16 *bias, *res, *gate;
  void* out;
  int T, F, blocks;  // blocks = ceil(K / 128)
  int tiles_t, tiles_f, group_t;
  int bn;      // pair kernel: features of a tile
  int splits;  // few-token kernel: CTAs of a cluster along K
};

// instruction descriptor of kind::mxf8f6f4: e4m3 x e4m3, ue8m0 scales, both operands K-major; `sf` is the
// byte of both operands' scale words
__device__ __forceinline__ uint32_t fp8_idesc(int M, int N, int sf) {
  return ((uint32_t)sf << 4) | ((uint32_t)(N >> 3) << 17) | (1u << 23) | ((uint32_t)(M >> 4) << 24) | ((uint32_t)sf << 29);
}
// The issuing warp runs its loop as a whole and one elected lane issues: in a branch that a single lane takes the
// operands cannot stay in uniform registers, and moving them there for each instruction made every MMA cost about
// 180 clocks whatever its N (256 x 128 and 256 x 240 tiles took the same time).
__device__ __forceinline__ void tc_mma_mxf8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tc_mma2_mxf8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "@e tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}
// tc_commit and tc_commit2_mc by the elected lane of a whole warp
__device__ __forceinline__ void tc_commit_warp(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tc_commit2_mc_warp(uint64_t* bar, uint16_t mask) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(
          smem_u32(bar)),
      "h"(mask)
      : "memory");
}
// a bounded wait by a whole warp: every lane gets the same answer
__device__ __forceinline__ bool mbar_wait_warp(uint64_t* bar, uint32_t parity, int* status, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, status, code));
}
__device__ __forceinline__ bool mbar_wait_cl_warp(uint64_t* bar, uint32_t parity, int* status, int code) {
  return __all_sync(0xffffffffu, mbar_wait_cl(bar, parity, status, code));
}
__device__ __forceinline__ void tmem_st4(uint32_t taddr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(taddr), "r"(a), "r"(b), "r"(c), "r"(d)
               : "memory");
}

// the scales of blocks 4 chunk .. 4 chunk + 3 of row r as one word; 2^0 where there is no such row or block
__device__ __forceinline__ uint32_t fp8_scale_word(const uint8_t* s, long ld, int r, int rows, int chunk, int blocks) {
  if (r >= rows) return 0x7f7f7f7fu;
  const uint8_t* p = s + (long)r * ld + 4 * chunk;
  if (4 * chunk + 4 <= blocks) return *reinterpret_cast<const uint32_t*>(p);
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) w |= (uint32_t)(4 * chunk + i < blocks ? p[i] : 0x7f) << (8 * i);
  return w;
}

// the same of blocks 4 chunk .. 4 chunk + 15; `vec`: the rows start on 16-byte boundaries
__device__ __forceinline__ uint4 fp8_scale_quad(const uint8_t* s, long ld, int r, int rows, int chunk, int blocks, bool vec) {
  if (r < rows && vec && 4 * chunk + 16 <= blocks) return *reinterpret_cast<const uint4*>(s + (long)r * ld + 4 * chunk);
  return make_uint4(fp8_scale_word(s, ld, r, rows, chunk, blocks), fp8_scale_word(s, ld, r, rows, chunk + 1, blocks),
                    fp8_scale_word(s, ld, r, rows, chunk + 2, blocks), fp8_scale_word(s, ld, r, rows, chunk + 3, blocks));
}
// After a wait that gave up: the producer lets its last loads land (with a limit) before the CTA can leave.
__device__ __forceinline__ void fp8_drain(uint64_t* full, int stages, int issued, volatile int* flags, int* status) {
  if (!flags[0]) return;
  for (int i = max(0, issued - stages); i < issued; ++i)
    mbar_wait(&full[i % stages], (uint32_t)(i / stages) & 1u, status, P5_ERR_WAIT_FULL);
}

enum Fp8Epi : int { FP8_STORE = 0, FP8_GELU = 1, FP8_RESID = 2, FP8_GATED = 3, FP8_GEGLU = 4, FP8_F32 = 5 };

// The epilogue's arithmetic on eight consecutive features f.. of token t, in fp32 (F % 8 == 0, f < F): v becomes the result,
// its first four elements for GeGLU.
template <int EPI>
__device__ __forceinline__ void fp8_math8(const Fp8Args& a, float (&v)[8], int t, int f) {
  if (a.bias) {
    float b[8];
    unpack8(*reinterpret_cast<const uint4*>(a.bias + f), b);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += b[i];
  }
  if (EPI == FP8_GEGLU) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = gelu_tanh(v[2 * i]) * v[2 * i + 1];
  }
  if (EPI == FP8_GELU) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = gelu_tanh(v[i]);
  }
  if (EPI == FP8_GATED) {
    float g[8];
    unpack8(*reinterpret_cast<const uint4*>(a.gate + f), g);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= g[i];
  }
  if (EPI == FP8_RESID || EPI == FP8_GATED) {
    float r[8];
    unpack8(*reinterpret_cast<const uint4*>(a.res + (long)t * a.F + f), r);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += r[i];
  }
}

// The same for rows that are not a multiple of 16 bytes: element by element, features past F left alone.
template <int EPI>
__device__ __forceinline__ void fp8_math8_any(const Fp8Args& a, float (&v)[8], int t, int f) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (f + i >= a.F) break;
    if (a.bias) v[i] += bf(a.bias[f + i]);
    if (EPI == FP8_GELU) v[i] = gelu_tanh(v[i]);
    if (EPI == FP8_GATED) v[i] *= bf(a.gate[f + i]);
    if (EPI == FP8_RESID || EPI == FP8_GATED) v[i] += bf(a.res[(long)t * a.F + f + i]);
  }
  if (EPI == FP8_GEGLU) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = gelu_tanh(v[2 * i]) * v[2 * i + 1];
  }
}
// 16-byte accesses: rows of out, res start on 16-byte boundaries (the bases do)
template <int EPI>
__device__ __forceinline__ bool fp8_rows_aligned(const Fp8Args& a) {
  return a.F % (EPI == FP8_GEGLU ? 16 : 8) == 0;
}

// Epilogue of eight consecutive features f.. of token t (t < T; f + 8 may pass F), fp32 throughout and rounded once.
template <int EPI>
__device__ __forceinline__ void fp8_epilogue8(const Fp8Args& a, float (&v)[8], int t, int f) {
  if (f >= a.F) return;
  if (fp8_rows_aligned<EPI>(a)) {
    fp8_math8<EPI>(a, v, t, f);
    const long at = (long)t * a.F + f;
    if (EPI == FP8_F32) {
      float4* d = reinterpret_cast<float4*>(static_cast<float*>(a.out) + at);
      d[0] = make_float4(v[0], v[1], v[2], v[3]);
      d[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else if (EPI == FP8_GEGLU) {
      *reinterpret_cast<uint2*>(static_cast<bf16*>(a.out) + at / 2) = make_uint2(pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]));
    } else {
      *reinterpret_cast<uint4*>(static_cast<bf16*>(a.out) + at) =
          make_uint4(pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]), pack_bf2(v[4], v[5]), pack_bf2(v[6], v[7]));
    }
    return;
  }
  fp8_math8_any<EPI>(a, v, t, f);
  constexpr int PER = EPI == FP8_GEGLU ? 2 : 1;
  const int n = (min(8, a.F - f)) / PER;
  const long at = ((long)t * a.F + f) / PER;
#pragma unroll
  for (int i = 0; i < 8 / PER; ++i) {
    if (i >= n) break;
    if (EPI == FP8_F32)
      static_cast<float*>(a.out)[at + i] = v[i];
    else
      static_cast<bf16*>(a.out)[at + i] = tobf(v[i]);
  }
}

// ------------------------------------------------------------------ few tokens
// D[128 features][BN tokens] of one tile by a cluster of `splits` CTAs, each with its share of the K blocks: the weights
// are on the 128-row side, so a handful of tokens still reads each weight once and at full width.  The fp32 partial tiles
// meet over distributed shared memory: CTA p receives the token slice p of every partial in one bulk copy each and adds
// them in rank order (reruns give the same bits).
// Below 10 us bound by a CTA's fixed chain and by tiles that do not fill the machine (50 x 8192 x 1024 GeGLU 6.6 us, bytes
// alone 1.4: 64 CTAs), above by uneven shares: a weight of 32768 rows is 256 tiles, two on 108 SMs and one on 40 (50 x 32768 x 2048
// 17.8 us, 3.8 TB/s of weights; 1 x 32768 x 2048 15.7 us, 4.3).
//   warp 0  TMA producer, warp 1  MMA issuer, warp 2  TMEM, warps 4-7  scales, then the accumulator
template <int BN>
struct Fp8FewCfg {
  static constexpr int A_BYTES = 128 * 128, B_BYTES = BN * 128, STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = BN >= 128 ? 5 : (BN >= 64 ? 3 : 4);
  static constexpr int PER_SM = BN >= 128 ? 1 : 2;  // two CTAs share an SM: one's fill and epilogue run under the other's loads
  static constexpr int TILE = BN * 128 * 4;  // fp32 partial tile [token][feature]
  static constexpr int SF_SLOTS = 4, SF_COL = BN, SF_PITCH = 8;  // scale words: 4 columns of A, BN / 32 of B
  static constexpr uint32_t TMEM_COLS = BN >= 128 ? 256 : (BN >= 64 ? 128 : 64);
  static constexpr int SMEM = 1024 + STAGES * STAGE + TILE + 512;
  static_assert(TILE <= STAGES * STAGE && SF_COL + SF_SLOTS * SF_PITCH <= (int)TMEM_COLS && SMEM * PER_SM <= 232448 - 1024, "");
};

template <int BN, int EPI>
__global__ void __launch_bounds__(256, Fp8FewCfg<BN>::PER_SM)
    fp8_few_kernel(const __grid_constant__ CUtensorMap tw, const __grid_constant__ CUtensorMap tx, const Fp8Args a) {
  using C = Fp8FewCfg<BN>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* ring = smem_raw + (((raw + 1023) & ~1023u) - raw);
  uint8_t* recv = ring + C::STAGES * C::STAGE;  // [splits][BN / splits][128] fp32
  uint64_t* full = reinterpret_cast<uint64_t*>(recv + C::TILE);
  uint64_t* empty = full + C::STAGES;
  uint64_t* sf_full = empty + C::STAGES;
  uint64_t* sf_empty = sf_full + C::SF_SLOTS;
  uint64_t* done = sf_empty + C::SF_SLOTS;
  uint64_t* got = done + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(got + 1);
  volatile int* flags = reinterpret_cast<volatile int*>(tmem_slot + 1);  // [0] abort
  int* status = &g_fp8_status;

  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int tile = blockIdx.x / a.splits;
  const int f0 = (tile % a.tiles_f) * 128, t0 = (tile / a.tiles_f) * BN;
  const int per = (a.blocks + a.splits - 1) / a.splits;
  const int kb0 = min((int)rank * per, a.blocks), n = min(kb0 + per, a.blocks) - kb0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < C::SF_SLOTS; ++s) {
      mbar_init(&sf_full[s], 4);
      mbar_init(&sf_empty[s], 1);
    }
    mbar_init(done, 1);
    mbar_init(got, 1);
    flags[0] = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tw);
    tma_prefetch_desc(&tx);
  }
  if (warp == 2) {
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  cluster_sync();  // every CTA's barriers exist before a peer's copy can arrive
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  const int c_first = kb0 >> 2;  // chunks of four blocks, counted from the start of K

  if (warp == 0) {
    if (lane == 0) {
      int issued = 0;
      for (int i = 0; i < n && !flags[0]; ++i) {
        const int s = i % C::STAGES;
        if (!mbar_wait(&empty[s], ((uint32_t)(i / C::STAGES) & 1u) ^ 1u, status, P5_ERR_WAIT_EMPTY)) {
          flags[0] = 1;
          break;
        }
        mbar_arrive_expect_tx(&full[s], C::STAGE);
        tma_load_2d(ring + s * C::STAGE, &tw, &full[s], (kb0 + i) * 128, f0);
        tma_load_2d(ring + s * C::STAGE + C::A_BYTES, &tx, &full[s], (kb0 + i) * 128, t0);
        issued = i + 1;
      }
      fp8_drain(full, C::STAGES, issued, flags, status);
    }
    __syncwarp();
  } else if (warp == 1) {
    int cur = -1, slot = 0;
    for (int i = 0; i < n; ++i) {
      const int s = i % C::STAGES, kb = kb0 + i;
      bool ok = true;
      if ((kb >> 2) != cur) {
        cur = kb >> 2;
        const int ci = cur - c_first;
        slot = ci % C::SF_SLOTS;
        ok = mbar_wait_warp(&sf_full[slot], (uint32_t)(ci / C::SF_SLOTS) & 1u, status, P5_ERR_WAIT_FULL);
      }
      if (!ok || !mbar_wait_warp(&full[s], (uint32_t)(i / C::STAGES) & 1u, status, P5_ERR_WAIT_FULL)) {
        flags[0] = 1;
        break;
      }
      tc_fence_after();
      const uint32_t wa = smem_u32(ring) + s * C::STAGE, xa = wa + C::A_BYTES;
      const uint32_t sf = tmem + (uint32_t)(C::SF_COL + slot * C::SF_PITCH);
      const uint32_t idesc = fp8_idesc(128, BN, kb & 3);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        tc_mma_mxf8(tmem, sw128_kmajor_desc(wa + kk * 32), sw128_kmajor_desc(xa + kk * 32), idesc, sf, sf + 4,
                    (i > 0 || kk > 0) ? 1u : 0u);
      tc_commit_warp(&empty[s]);
      if ((kb & 3) == 3 || i == n - 1) tc_commit_warp(&sf_empty[slot]);
    }
    tc_commit_warp(done);
  } else if (warp >= 4) {
    // ---- scale words, a chunk ahead of the wait for its slot
    const uint32_t t_sf = tmem + ((uint32_t)((warp & 3) * 32) << 16) + C::SF_COL;
    const int chunks = n > 0 ? ((kb0 + n - 1) >> 2) - c_first + 1 : 0;
    for (int ci = 0; ci < chunks; ++ci) {
      const int slot = ci % C::SF_SLOTS;
      uint32_t wv[4], xv[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) wv[j] = fp8_scale_word(a.ws, a.ld_ws, f0 + 32 * j + lane, a.F, c_first + ci, a.blocks);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        xv[j] = j < BN / 32 ? fp8_scale_word(a.xs, a.ld_xs, t0 + 32 * j + lane, a.T, c_first + ci, a.blocks) : 0u;
      const bool ok = !flags[0] && mbar_wait(&sf_empty[slot], ((uint32_t)(ci / C::SF_SLOTS) & 1u) ^ 1u, status, P5_ERR_WAIT_EMPTY);
      if (__any_sync(0xffffffffu, !ok)) {
        flags[0] = 1;
        break;
      }
      tc_fence_after();
      tmem_st4(t_sf + (uint32_t)(slot * C::SF_PITCH), wv[0], wv[1], wv[2], wv[3]);
      tmem_st4(t_sf + (uint32_t)(slot * C::SF_PITCH) + 4u, xv[0], xv[1], xv[2], xv[3]);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sf_full[slot]);
    }
    // ---- partial tile -> shared memory [token][feature] (the ring is idle once every MMA is done)
    const bool ok = mbar_wait(done, 0, status, P5_ERR_WAIT_ACCUM) && n > 0;
    tc_fence_after();
    float* dst = reinterpret_cast<float*>(a.splits == 1 ? recv : ring) + (warp & 3) * 32 + lane;
    const uint32_t t_acc = tmem + ((uint32_t)((warp & 3) * 32) << 16);
#pragma unroll 1
    for (int c = 0; c < BN; c += 32) {
      uint32_t r[32];
      __syncwarp();
      tmem_ld32(t_acc + (uint32_t)c, r);
      tmem_wait_ld();
#pragma unroll
      for (int i = 0; i < 32; ++i) dst[(c + i) * 128] = ok ? __uint_as_float(r[i]) : 0.f;
    }
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 2) tmem_dealloc(tmem, C::TMEM_COLS);

  const int slice = BN / a.splits;  // tokens that this CTA finishes
  if (a.splits > 1) {
    const uint32_t bytes = (uint32_t)slice * 512u;
    if (threadIdx.x == 0) mbar_arrive_expect_tx(got, bytes * (uint32_t)a.splits);
    if (threadIdx.x < (unsigned)a.splits)
      bulk_copy_to_peer(map_peer(smem_u32(recv) + rank * bytes, threadIdx.x), smem_u32(ring) + threadIdx.x * bytes, bytes,
                        map_peer(smem_u32(got), threadIdx.x));
    // A peer whose own waits give up still sends, up to four limits later: this CTA must not free what that copy writes, nor
    // pass the barrier that keeps the peer's copy readable, so it waits for it all the same.
    for (int k = 0; k < 8 && !mbar_wait_cl(got, 0, status, P5_ERR_WAIT_SPLITK); ++k) flags[0] = 1;
    __syncthreads();
    cluster_arrive_relaxed();
  }
  const float* part = reinterpret_cast<const float*>(recv);
  if (!flags[0]) {
    for (int i = threadIdx.x; i < slice * 16; i += 256) {
      const int j = i >> 4, fo = (i & 15) * 8;
      const int t = t0 + (int)rank * slice + j;
      if (t >= a.T) continue;
      float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      for (int p = 0; p < a.splits; ++p) {
        const float4* s = reinterpret_cast<const float4*>(part + (long)(p * slice + j) * 128 + fo);
        const float4 u = s[0], w = s[1];
        v[0] += u.x, v[1] += u.y, v[2] += u.z, v[3] += u.w, v[4] += w.x, v[5] += w.y, v[6] += w.z, v[7] += w.w;
      }
      fp8_epilogue8<EPI>(a, v, t, f0 + fo);
    }
  }
  __syncwarp();
  if (a.splits > 1) cluster_wait_acquire();  // no CTA leaves while a peer's copy may still read its shared memory
}

// ------------------------------------------------------------------ many tokens
// A cluster of two CTAs owns 256 tokens x bn features (bn <= 240, a multiple of 16): each stages 128 token rows and
// bn / 2 weight rows per K block, and one thread of the even CTA issues tcgen05.mma.cta_group::2 over both, as in
// gemm_pair.cuh (the same ring, relay and commit protocol).  Measured: 7744 x 32768 x 2048 GeGLU 411 us, 2.5 PFLOP/s in short
// bursts (tensor pipes 69 % busy); run for seconds the power cap holds it near 2.2, where a library product with one
// scale a tensor and no epilogue gets 2.26.  7744 x 2048 x 16384 211 us.  Announcing the odd CTA's scale words soundly is 2 and 6 %
// of these.  Tensor memory holds two accumulators of bn columns and, in the
// rest, chunks of scale words (4 columns of tokens, 8 of features); bn = 256 would leave room for one accumulator only,
// and its epilogue could not run under the next tile's products.
//   warp 0 TMA, warp 1 MMA (odd CTA: relay), warp 2 TMEM, warp 3 the odd CTA's scales, warps 4-11 epilogue, warps 12-15 scales
struct Fp8PairCfg {
  static constexpr int A_BYTES = 128 * 128, B_BYTES = 120 * 128, STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = 5;
  static constexpr int MAX_BN = 240, SF_PITCH = 12, MAX_SLOTS = 8;
  // chunks of scale words that fit in tensor memory beside two accumulators of bn columns (2 at 240, 5 at 224, 8 from 208 down)
  __host__ __device__ static constexpr int slots(int bn) { return (512 - 2 * bn) / SF_PITCH < MAX_SLOTS ? (512 - 2 * bn) / SF_PITCH : MAX_SLOTS; }
  static constexpr int SF_BYTES = 2 * 384 * 16;  // scales of 16 blocks of every row, two buffers
  static constexpr int OUT_PITCH = 144, OUT_WARP = 32 * OUT_PITCH;  // staged output: 32 rows of 128 bytes, conflict-free pitch
  static constexpr int SMEM = 1024 + STAGES * STAGE + SF_BYTES + 8 * OUT_WARP + 512;
  static constexpr int THREADS = 512;
};

template <int EPI>
__global__ void __launch_bounds__(Fp8PairCfg::THREADS, 1)
    fp8_pair_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tw, const Fp8Args a) {
  using C = Fp8PairCfg;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* ring = smem_raw + (((raw + 1023) & ~1023u) - raw);
  uint4* sf_rows = reinterpret_cast<uint4*>(ring + C::STAGES * C::STAGE);
  uint8_t* out_rows = ring + C::STAGES * C::STAGE + C::SF_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(out_rows + 8 * C::OUT_WARP);  // own TMA landed
  uint64_t* empty = full + C::STAGES;        // pair MMAs done with the stage (multicast commit)
  uint64_t* pair = empty + C::STAGES;        // even CTA: the odd CTA's stage landed (relay)
  uint64_t* tfull = pair + C::STAGES;        // [2] accumulator complete (multicast commit)
  uint64_t* tempty = tfull + 2;              // [2] even CTA: accumulator drained by 16 epilogue warps
  uint64_t* sf_full = tempty + 2;                // [slots] this CTA's scale words in place (4 warps)
  uint64_t* sf_empty = sf_full + C::MAX_SLOTS;   // [slots] MMAs done with the scale words (multicast commit)
  uint64_t* rows_full = sf_empty + C::MAX_SLOTS;  // [2] sf_rows buffer written by the four scale warps
  uint64_t* sf_peer = rows_full + 2;              // [slots] even CTA: the odd CTA's scale words in place (its warp 3)
  uint64_t* done = sf_peer + C::MAX_SLOTS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* flags = reinterpret_cast<volatile int*>(tmem_slot + 1);  // [0] abort
  int* status = &g_fp8_status;

  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const bool even = rank == 0;
  const int cid = blockIdx.x >> 1, nclusters = gridDim.x >> 1;
  const int n_units = a.tiles_t * a.tiles_f;
  const uint32_t b_bytes = (uint32_t)(a.bn / 2) * 128u;
  const int slots = C::slots(a.bn);

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
      mbar_init(&pair[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], 16);
      mbar_init(&rows_full[i], 4);
    }
    for (int i = 0; i < C::MAX_SLOTS; ++i) {
      mbar_init(&sf_full[i], 4);
      mbar_init(&sf_peer[i], 1);
      mbar_init(&sf_empty[i], 1);
    }
    mbar_init(done, 1);
    flags[0] = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tx);
    tma_prefetch_desc(&tw);
  }
  cluster_sync();
  if (warp == 2) {
    tmem_alloc2(tmem_slot, 512);
    tmem_relinquish2();
  }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);

  auto decode = [&](int u, int& tt, int& tf) {  // tiles walk down group_t token tiles, then to the next features
    const int per_group = a.group_t * a.tiles_f;
    const int group = u / per_group, first = group * a.group_t;
    const int gt = min(a.group_t, a.tiles_t - first), in = u % per_group;
    tt = first + in % gt;
    tf = in / gt;
  };

  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      for (int u = cid; u < n_units && !flags[0]; u += nclusters) {
        int tt, tf;
        decode(u, tt, tf);
        const int xrow = tt * 256 + (int)rank * 128, wrow = tf * a.bn + (int)rank * (a.bn / 2);
        for (int i = 0; i < a.blocks; ++i, ++it) {
          const int s = it % C::STAGES;
          if (!mbar_wait(&empty[s], ((uint32_t)(it / C::STAGES) & 1u) ^ 1u, status, P5_ERR_WAIT_EMPTY)) {
            flags[0] = 1;
            break;
          }
          mbar_arrive_expect_tx(&full[s], C::A_BYTES + b_bytes);
          tma_load_2d(ring + s * C::STAGE, &tx, &full[s], i * 128, xrow);
          tma_load_2d(ring + s * C::STAGE + C::A_BYTES, &tw, &full[s], i * 128, wrow);
        }
      }
      fp8_drain(full, C::STAGES, it, flags, status);
    }
    __syncwarp();
  } else if (warp == 1 && even) {
    int it = 0, j = 0, slot = -1;
    uint32_t sf_ph = 1;
    bool ok = true;
    for (int u = cid; u < n_units && ok; u += nclusters, ++j) {
      const int acc = j & 1;
      ok = mbar_wait_cl_warp(&tempty[acc], ((uint32_t)(j >> 1) & 1u) ^ 1u, status, P5_ERR_WAIT_ACCUM);
      tc_fence_after();
      const uint32_t d = tmem + (uint32_t)(acc * a.bn);
      for (int i = 0; i < a.blocks && ok; ++i, ++it) {
        const int s = it % C::STAGES;
        const uint32_t ph = (uint32_t)(it / C::STAGES) & 1u;
        if ((i & 3) == 0) {
          if (++slot == slots) slot = 0;
          if (slot == 0) sf_ph ^= 1u;
          ok = mbar_wait_warp(&sf_full[slot], sf_ph, status, P5_ERR_WAIT_FULL) &&
               mbar_wait_cl_warp(&sf_peer[slot], sf_ph, status, P5_ERR_WAIT_FULL);
        }
        ok = ok && mbar_wait_warp(&full[s], ph, status, P5_ERR_WAIT_FULL) && mbar_wait_warp(&pair[s], ph, status, P5_ERR_WAIT_FULL);
        if (!ok) break;
        tc_fence_after();
        const uint32_t xa = smem_u32(ring) + s * C::STAGE, wa = xa + C::A_BYTES;
        const uint32_t sf = tmem + (uint32_t)(2 * a.bn + slot * C::SF_PITCH);
        const uint32_t idesc = fp8_idesc(256, a.bn, i & 3);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          tc_mma2_mxf8(d, sw128_kmajor_desc(xa + kk * 32), sw128_kmajor_desc(wa + kk * 32), idesc, sf, sf + 4,
                       (i > 0 || kk > 0) ? 1u : 0u);
        tc_commit2_mc_warp(&empty[s], 3);
        if ((i & 3) == 3 || i == a.blocks - 1) tc_commit2_mc_warp(&sf_empty[slot], 3);
      }
      if (ok) tc_commit2_mc_warp(&tfull[acc], 3);
    }
    if (!ok) flags[0] = 1;
    tc_commit2_mc_warp(done, 3);
  } else if (warp == 1) {
    if (lane == 0) {
      // relaxed, as in gemm_pair.cuh: nothing but a completion that the TMA has signalled is passed on
      const uint32_t pair0 = map_peer(smem_u32(pair), 0);
      int it = 0;
      for (int u = cid; u < n_units && !flags[0]; u += nclusters) {
        for (int i = 0; i < a.blocks; ++i, ++it) {
          const int s = it % C::STAGES;
          if (!mbar_wait(&full[s], (uint32_t)(it / C::STAGES) & 1u, status, P5_ERR_WAIT_FULL)) {
            flags[0] = 1;
            break;
          }
          mbar_arrive_cluster_relaxed(pair0 + (uint32_t)s * 8u);
        }
      }
    }
    __syncwarp();
  } else if (warp == 3) {
    // The odd CTA's scale words are written by its warps: this lane announces them with a release at cluster scope, which the
    // issuer acquires once a chunk.  A warp of its own, because a release holds its thread up (7744 x 32768 x 2048: by the relay
    // 445 us, by the scale warps 435, here 423).
    if (!even && lane == 0) {
      const uint32_t sf_peer0 = map_peer(smem_u32(sf_peer), 0);
      int slot = -1;
      uint32_t sf_ph = 1;
      for (int u = cid; u < n_units && !flags[0]; u += nclusters) {
        for (int i = 0; i < a.blocks; i += 4) {
          if (++slot == slots) slot = 0;
          if (slot == 0) sf_ph ^= 1u;
          if (!mbar_wait(&sf_full[slot], sf_ph, status, P5_ERR_WAIT_FULL)) {
            flags[0] = 1;
            break;
          }
          tc_fence_after();
          tc_fence_before();
          mbar_arrive_cluster(sf_peer0 + (uint32_t)slot * 8u);
        }
      }
    }
    __syncwarp();
  } else if (warp >= 12) {
    // ---- scale words of this CTA's 128 tokens and of all bn (<= 256) features.  Every quarter of the lanes needs all of
    // them, but a gather of 4 bytes a row takes a pass of the shared-memory pipe for each row (loaded by each warp for
    // itself it slowed the whole kernel by a third), so the four warps load 96 of the 384 rows each, 16 blocks at a
    // time and that far ahead, and share them through shared memory.
    const int sw = warp - 12;
    const uint32_t t_sf = tmem + ((uint32_t)(sw * 32) << 16) + (uint32_t)(2 * a.bn);
    const int chunks = (a.blocks + 3) >> 2;
    const bool vec_x = a.ld_xs % 16 == 0 && ((uintptr_t)a.xs & 15) == 0, vec_w = a.ld_ws % 16 == 0 && ((uintptr_t)a.ws & 15) == 0;
    int u = cid, k = 0, xrow = 0, wrow = 0;  // the next piece of 16 blocks: tile u, chunks k .. k + 3
    auto enter = [&]() {
      int tt, tf;
      decode(u, tt, tf);
      xrow = tt * 256 + (int)rank * 128;
      wrow = tf * a.bn;
    };
    uint4 next[3];
    auto load = [&]() {
#pragma unroll
      for (int j = 0; j < 3; ++j) {
        const int r = (3 * sw + j) * 32 + lane;
        next[j] = r < 128 ? fp8_scale_quad(a.xs, a.ld_xs, xrow + r, a.T, k, a.blocks, vec_x)
                          : fp8_scale_quad(a.ws, a.ld_ws, wrow + r - 128, a.F, k, a.blocks, vec_w);
      }
    };
    if (u < n_units) {
      enter();
      load();
    }
    bool ok = true;
    int slot = -1;
    uint32_t sf_ph = 1;
    for (int piece = 0; u < n_units && ok; ++piece) {
      uint4* buf = sf_rows + (piece & 1) * 384;
#pragma unroll
      for (int j = 0; j < 3; ++j) buf[(3 * sw + j) * 32 + lane] = next[j];
      // a buffer is written again two pieces later, after this wait for the piece between: every warp has read it by then
      __syncwarp();
      if (lane == 0) mbar_arrive(&rows_full[piece & 1]);
      ok = mbar_wait_warp(&rows_full[piece & 1], (uint32_t)(piece >> 1) & 1u, status, P5_ERR_WAIT_FULL);
      const int here = min(4, chunks - k);
      k += 4;
      if (k >= chunks) {
        k = 0;
        u += nclusters;
        if (u < n_units) enter();
      }
      for (int c = 0; c < here && ok; ++c) {
        if (++slot == slots) slot = 0;
        if (slot == 0) sf_ph ^= 1u;
        uint32_t v[12];
#pragma unroll
        for (int j = 0; j < 12; ++j) v[j] = reinterpret_cast<const uint32_t*>(buf + 32 * j + lane)[c];
        if (c == 0 && u < n_units) load();
        ok = !flags[0] && mbar_wait(&sf_empty[slot], sf_ph ^ 1u, status, P5_ERR_WAIT_EMPTY);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const uint32_t ta = t_sf + (uint32_t)(slot * C::SF_PITCH);
        tmem_st4(ta, v[0], v[1], v[2], v[3]);
        tmem_st4(ta + 4u, v[4], v[5], v[6], v[7]);
        tmem_st4(ta + 8u, v[8], v[9], v[10], v[11]);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sf_full[slot]);
      }
    }
    if (!ok) flags[0] = 1;
  } else if (warp >= 4) {
    // ---- epilogue: this CTA's 128 tokens, each half of the warps one half of the features
    const int sub = warp & 3, half = (warp - 4) >> 2;
    const uint32_t lane_addr = (uint32_t)(sub * 32) << 16;
    const uint32_t tempty0 = map_peer(smem_u32(tempty), 0);
    // the halves meet at a multiple of 16 columns, so that output rows start on 32-byte sectors
    const int middle = (a.bn / 2 + 15) / 16 * 16;
    const int c_begin = half ? middle : 0, c_end = half ? a.bn : middle;
    // Rows of 128 output bytes are staged in shared memory and written by whole rows: a thread owns one token, so its own
    // 16-byte stores lie a row apart and reach L2 as half sectors (7744 x 32768 x 2048 GeGLU 474 us, no stores 340).
    constexpr int ES = EPI == FP8_F32 ? 4 : 2, PER = EPI == FP8_GEGLU ? 2 : 1;  // output bytes; columns an output value
    constexpr int PASS = 128 / ES * PER;                                       // columns of 128 output bytes
    const bool rows16 = fp8_rows_aligned<EPI>(a);
    uint8_t* stage = out_rows + (warp - 4) * C::OUT_WARP;
    const long out_pitch = (long)(a.F / PER) * ES;
    int j = 0;
    for (int u = cid; u < n_units; u += nclusters, ++j) {
      int tt, tf;
      decode(u, tt, tf);
      const int acc = j & 1;
      const bool ok = !flags[0] && mbar_wait_warp(&tfull[acc], (uint32_t)(j >> 1) & 1u, status, P5_ERR_WAIT_ACCUM);
      if (!ok) flags[0] = 1;
      tc_fence_after();
      const uint32_t t_acc = tmem + lane_addr + (uint32_t)(acc * a.bn);
      const int t_warp = tt * 256 + (int)rank * 128 + sub * 32, fb = tf * a.bn;
      const int t = t_warp + lane;
#pragma unroll 1
      for (int c = c_begin; ok && c < c_end; c += PASS) {
        const int width = min(PASS, c_end - c);  // a multiple of 16
#pragma unroll
        for (int q = 0; q < PASS; q += 32) {
          if (q >= width) break;
          uint32_t r[32];
          __syncwarp();  // lanes behind the last token have skipped the arithmetic below
          if (q + 32 <= width) {
            tmem_ld32(t_acc + (uint32_t)(c + q), r);
          } else {
            uint32_t r16[16];
            tmem_ld16(t_acc + (uint32_t)(c + q), r16);
#pragma unroll
            for (int i = 0; i < 16; ++i) r[i] = r16[i], r[16 + i] = 0u;
          }
          tmem_wait_ld();
#pragma unroll
          for (int p = 0; p < 32; p += 8) {
            if (q + p >= width) break;
            const int f = fb + c + q + p;
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[p + i]);
            if (f >= a.F || t >= a.T) continue;
            if (rows16)
              fp8_math8<EPI>(a, v, t, f);
            else
              fp8_math8_any<EPI>(a, v, t, f);
            uint8_t* d = stage + lane * C::OUT_PITCH + (q + p) / PER * ES;
            if (EPI == FP8_F32) {
              reinterpret_cast<float4*>(d)[0] = make_float4(v[0], v[1], v[2], v[3]);
              reinterpret_cast<float4*>(d)[1] = make_float4(v[4], v[5], v[6], v[7]);
            } else if (EPI == FP8_GEGLU) {
              *reinterpret_cast<uint2*>(d) = make_uint2(pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]));
            } else {
              *reinterpret_cast<uint4*>(d) =
                  make_uint4(pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]), pack_bf2(v[4], v[5]), pack_bf2(v[6], v[7]));
            }
          }
        }
        __syncwarp();
        const int bytes = min(width, a.F - fb - c) / PER * ES;  // of a row (none where fb + c >= F)
        uint8_t* dst = static_cast<uint8_t*>(a.out) + (long)(fb + c) / PER * ES;
        if (rows16) {
          const int piece = (lane & 7) * 16;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int row = 4 * i + (lane >> 3);
            if (piece < bytes && t_warp + row < a.T)
              *reinterpret_cast<uint4*>(dst + (long)(t_warp + row) * out_pitch + piece) =
                  *reinterpret_cast<const uint4*>(stage + row * C::OUT_PITCH + piece);
          }
        } else {
          for (int row = 0; row < 32 && t_warp + row < a.T; ++row)
            for (int e = lane * ES; e < bytes; e += 32 * ES) {
              uint8_t* d = dst + (long)(t_warp + row) * out_pitch + e;
              const uint8_t* sp = stage + row * C::OUT_PITCH + e;
              if (ES == 4)
                *reinterpret_cast<uint32_t*>(d) = *reinterpret_cast<const uint32_t*>(sp);
              else
                *reinterpret_cast<uint16_t*>(d) = *reinterpret_cast<const uint16_t*>(sp);
            }
        }
        __syncwarp();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (even)
          mbar_arrive(&tempty[acc]);
        else
          mbar_arrive_cluster(tempty0 + (uint32_t)acc * 8u);
      }
      if (!ok) break;
    }
  }

  // ---- exit: the issuer's last commit has landed in both CTAs, then both meet
  __syncthreads();
  if (threadIdx.x == 0) mbar_wait_cl(done, 0, status, P5_ERR_WAIT_ACCUM);
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc2(tmem, 512);
  }
}

}  // namespace p5
