// kv8_attention_tc.cuh — attention over the 8-bit K/V cache for many query rows, on the 5th-generation tensor cores
// (the mathematics and the arguments are kv8_attention.cuh's).
//
// A CTA owns 128 folded query rows (r = t * G + g) of one (sample, K/V head) and one key split, and walks its keys in
// tiles of 64:
//   S = Q K^T     kind::f8f6f4, the K codes straight from the cache by TMA.  Q keeps 8 bits as two e4m3 operands, Q ~ 2^e (hi + lo)
//                 with lo = e4m3(q - hi): off by at most 2^-10 where the row's largest element is 256 or more, and the two
//                 products at twice the fp16 rate cost what one fp16 product would, without widening K.  Q lives in tensor
//                 memory (HD / 2 columns), so a product reads only K from shared memory.
//   softmax       thread = row = TMEM lane; two warpgroups take turns, one the even tiles and one the odd, so a tile's long
//                 chain (load, scale, maximum, exponentials, store) runs beside the next one's.  They share the running maximum
//                 of a row through shared memory: a tile's warp waits for its turn, raises the maximum if it must, and passes
//                 the turn on before its exponentials.  Each keeps its own sum.
//   O += P V      kind::f16, P in fp16 (11 bits; as 2^7 p, which keeps weights down to 2^-31 of the largest), V widened to fp16
//                 and scaled by its row's power of two relative to an exponent eb by four converter warps (exact: eb follows the
//                 tiles so that their scales lie within eb - 15 .. eb + 7; keys that no row sees become zeros, whatever the cache
//                 holds there).  An e4m3 P would need three operands to keep the small weights of a long cache.
//                 Where a tile's scales span more, or lie more than 2^64 from those before (a key that some rows do not see
//                 counts as well: it must not cost them bits), the CTA goes through its keys again with V and P in bf16, into which any scale fits; V is exact,
//                 weights keep 8 bits.  A choice of type for each tile made every call 2 to 7 % slower, in each form tried.
// Measured: 64 chunks of 50 tokens, 8 heads on one of 256, 1,018 keys 50.6 us (527 TFLOP/s); 8 x 968 x 968 98 us (629); 2 x 2,049
// tokens, causal over 8,192 keys, 16 heads on 4 of 128 315 us (764) and on 2 of 64 270 us (446); where the second pass is needed the
// chunks take 92 us, the third 683.  No unit is full (at HD 128 tensor pipes 43 %, exponentials
// 43 %, issue 56 %, shared memory 53 %): a tile waits on the chain of its softmax, about 2,400 clocks for two tiles in
// turn, and at HD 256 a short call on the 10 us that a CTA takes to load its queries and to store.  Three warpgroups were
// slower than two (349 against 328 us then): they leave a thread 128 registers.
// The running maximum moves only when a tile exceeds it by 2^8 and the V exponent eb only when a scale leaves its window;
// both rescale O through tcgen05.ld/st.  eb is the same for all rows and kept by the warp that loads the scales.
//   warp 0 TMA, warp 1 MMA issue, warp 2 TMEM, warp 3 scales, warps 4-11 softmax, warps 12-15 V
#pragma once
#include "fp8_gemm.cuh"
#include "kv8_attention.cuh"

namespace p5 {

template <int HD>
struct Kv8TcCfg {
  static constexpr int ROWS = 128, KT = 64;
  static constexpr int ROWB = HD < 128 ? HD : 128;  // bytes of a key row in one swizzled block
  static constexpr int ATOMS = HD / ROWB;           // such blocks
  static constexpr int TILE8 = KT * HD;            // codes of a K or V tile
  static constexpr int TILE16 = KT * HD * 2;       // a widened V tile
  static constexpr int NK = HD == 256 ? 3 : 4;     // K and V code rings
  static constexpr int NSC = 4;                    // scale slots
  static constexpr int K_OFF = 0, V_OFF = NK * TILE8, W_OFF = 2 * NK * TILE8;
  static constexpr int Q_BYTES = ROWS * (HD * 2 + 16);  // query rows on their way in, over the widened V
  static constexpr int SC_OFF = W_OFF + (2 * TILE16 > Q_BYTES ? 2 * TILE16 : (Q_BYTES + 127) / 128 * 128);
  static constexpr int SC_SLOT = (2 * KT + 4) * 4;  // kf[64] (fp32), vf[64] (fp16 or bf16, twice), rescale factor of O, unit of kf
  static constexpr int X_OFF = SC_OFF + NSC * SC_SLOT;  // [5][128] floats between the two softmax warpgroups
  static constexpr int BAR_OFF = X_OFF + 5 * ROWS * 4;
  static constexpr int BARS = 4 * NK + 2 * NSC + 21;  // barriers of a pass
  static constexpr int SMEM = 1024 + BAR_OFF + 2 * BARS * 8 + 64;
  // Tensor memory: Q hi | lo, S, P[2], O.  P lies here because all of this competes for the shared memory; at HD 256 that
  // leaves room for one S buffer only (two, and P in shared memory: 64 chunks 49.7 us).
  static constexpr int NS = HD == 256 ? 1 : 2;
  static constexpr int Q_COL = 0, S_COL = HD / 2, P_COL = S_COL + NS * KT, O_COL = P_COL + KT;
  static constexpr int OUT_PITCH = HD * 2 + 16;
  static constexpr int THREADS = 512;
  // registers a thread: warps 0-3, softmax, V; their sum over the block is what 128 a thread at launch make (the host checks)
  static constexpr int REG_ROLE = 64, REG_SOFT = 184, REG_V = 80;
  static constexpr int REGS = 128 * REG_ROLE + 256 * REG_SOFT + 128 * REG_V;
  static_assert(O_COL + HD <= 512 && REGS <= 65536 && ROWS * OUT_PITCH <= SC_OFF && SMEM <= 232448, "");
};

// D (+)= A[tmem] B[smem]^T, kind::f8f6f4 (e4m3 x e4m3), issued by the elected lane of a whole warp
__device__ __forceinline__ void tc_mma_f8_ta(uint32_t d, uint32_t a_tmem, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a_tmem), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tc_mma_f16_ta_warp(uint32_t d, uint32_t a_tmem, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a_tmem), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// descriptor of a K-major tile of 64-byte rows written by TMA with the 64-byte swizzle: 8-row groups 512 bytes apart
__device__ __forceinline__ uint64_t sw64_kmajor_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | (uint64_t)1 << 16 | (uint64_t)(512 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)4 << 61;
}
__device__ __forceinline__ void tmem_st_n(uint32_t taddr, const uint32_t (&r)[16]) { tmem_st16(taddr, r); }
__device__ __forceinline__ void tmem_st_n(uint32_t taddr, const uint32_t (&r)[8]) {
  tmem_st4(taddr, r[0], r[1], r[2], r[3]);
  tmem_st4(taddr + 4, r[4], r[5], r[6], r[7]);
}
// Each warpgroup sets its share of the block's registers once.
template <int N>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
// two fp32 operations in one instruction (sm_100 packed arithmetic)
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
  return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
  return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(d)
      : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)), "l"(*reinterpret_cast<uint64_t*>(&c)));
  return *reinterpret_cast<float2*>(&d);
}

__device__ __forceinline__ float2 sub2(float2 a, float2 b) {
  return fma2(b, make_float2(-1.f, -1.f), a);
}

template <int HD>
__global__ void __launch_bounds__(512, 1)
    kv8_attn_tc_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const Kv8Args a) {
  using C = Kv8TcCfg<HD>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw + 1023) & ~1023u) - raw);
  // barriers, those of a second pass over the keys C::BARS behind them
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);  // [NK] codes landed
  uint64_t* k_empty = k_full + C::NK;                                // [NK] S product done
  uint64_t* v_full = k_empty + C::NK;                                // [NK]
  uint64_t* v_empty = v_full + C::NK;                                // [NK] widened (4 warps)
  uint64_t* w_full = v_empty + C::NK;                                // [2] widened V in place (4 warps)
  uint64_t* w_empty = w_full + 2;                                    // [2] P V product done
  uint64_t* sc_full = w_empty + 2;                                   // [NSC] scales in place
  uint64_t* sc_empty = sc_full + C::NSC;                             // [NSC] read by the tile's 4 softmax warps and the 4 of V
  uint64_t* s_full = sc_empty + C::NSC;                              // [2] of the even and the odd tiles
  uint64_t* s_empty = s_full + 2;                                    // [2] (4 warps)
  uint64_t* p_full = s_empty + 2;                                    // [2] (4 warps)
  uint64_t* p_empty = p_full + 2;                                    // [2] P V product done
  uint64_t* turn = p_empty + 2;                                      // [2][4] the other warpgroup's warp has passed the turn
  uint64_t* o_full = turn + 8;                                       // every MMA complete
  uint64_t* q_full = k_full + 2 * C::BARS;                           // Q in tensor memory (8 warps)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(q_full + 1);
  volatile int* flags = reinterpret_cast<volatile int*>(tmem_slot + 1);  // [0] abort, [1] eb at the end, [2] go through the keys again
  float* exch = reinterpret_cast<float*>(smem + C::X_OFF);
  int* status = &g_fp8_status;

  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int b = blockIdx.y / a.kv_heads, kvh = blockIdx.y % a.kv_heads;
  const int tokens = kv8_tokens(a, b), rows = tokens * a.G;
  // the last rows first: under a causal mask they have the most keys
  const int row0 = ((int)gridDim.x - 1 - (int)blockIdx.x) * C::ROWS;
  const int split = blockIdx.z;
  // the 128 query rows into shared memory, before anything that waits for slots and lengths: each softmax warp loads
  // 16 whole rows, of the 32 that its lanes (thread = row) will convert
  const int g = (warp - 4) >> 2, sub = warp & 3;  // softmax warps: warpgroup, lane quarter
  const int r = sub * 32 + lane, row = row0 + r;
  const bool in = row < rows;
  const int t = in ? row / a.G : 0, h = kvh * a.G + (in ? row - t * a.G : 0);
  if (warp >= 4 && warp < 12) {
    const uint32_t sq = smem_u32(smem + C::W_OFF) + (uint32_t)(sub * 32 + g * 16) * C::OUT_PITCH;
    const bf16* src = a.q + (long)b * a.q_b + (long)t * a.q_t + (long)h * HD;
    constexpr int PER = HD / 8;  // 16-byte pieces of a row
#pragma unroll
    for (int k = 0; k < 16 * PER / 32; ++k) {
      const int id = k * 32 + lane, rr = id / PER, p = id % PER;
      const uint64_t from = __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(src), g * 16 + rr);
      const bool there = __shfl_sync(0xffffffffu, (int)in, g * 16 + rr);
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(sq + rr * C::OUT_PITCH + p * 16),
                   "l"(from + (there ? (uint64_t)p * 16 : 0)), "r"(there ? 16 : 0)
                   : "memory");
    }
    cp_async_commit();
  }
  const int slot = a.slots ? a.slots[b] : b;
  const int len = (slot < 0 || slot >= a.n_slots) ? 0 : max(0, min(a.lens[b], a.capacity));
  const int t_last = (min(row0 + C::ROWS, rows) - 1) / a.G;
  // keys that any of the rows sees
  const int top = row0 >= rows ? 0 : (a.causal ? max(0, min(len, len - tokens + t_last + 1)) : len);
  const int tiles = (top + C::KT - 1) / C::KT;
  const int per = (tiles + a.splits - 1) / a.splits;
  const int j0 = min(split * per, tiles), n = min(j0 + per, tiles) - j0;

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::NK; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 4);
    }
    for (int i = 0; i < C::NSC; ++i) {
      mbar_init(&sc_full[i], 1);
      mbar_init(&sc_empty[i], 8);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&w_full[i], 4);
      mbar_init(&w_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&s_empty[i], 4);
      mbar_init(&p_full[i], 4);
      mbar_init(&p_empty[i], 1);
    }
    for (int i = 0; i < 8; ++i) mbar_init(&turn[i], 1);
    mbar_init(o_full, 1);
    mbar_init(q_full, 8);
    flags[0] = flags[2] = 0;
    flags[1] = -1000;
    fence_barrier_init();
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
  }
  if (warp == 2) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);

  // A role's pass over the keys, and a second one in bf16 where a tile needs it, on barriers of its own.  The softmax, the scales and the
  // V warps have a copy of their code for each; one copy of the issuing loop runs twice (a second copy made head_dim 128 a third
  // slower).  What the second pass costs the calls that do not need it: at head_dim 128 1.5 %, at 256 4 %.
  auto met = [&]() -> bool {  // every thread; true: once more
    tc_fence_before();
    asm volatile("bar.sync 2, 512;" ::: "memory");
    tc_fence_after();
    return __builtin_expect(flags[2] && !flags[0], 0);
  };
  auto meet = [&]() -> bool {
    if (__builtin_expect(!met(), 1)) return false;
    asm volatile("bar.sync 2, 512;" ::: "memory");  // warp 2 has set the second pass' barriers up
    return true;
  };
  auto passes = [&](auto role) {
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
      role(pass);
      if (pass || __builtin_expect(!meet(), 1)) break;
    }
  };

  if (warp < 4) {
    regs_dec<C::REG_ROLE>();
    if (warp == 0) {
      passes([&](int pass) {
        const int of = pass * C::BARS;
        if (lane == 0) {
          int issued = 0;
          for (int i = 0; i < n && !flags[0]; ++i) {
            const int s = i % C::NK;
            const uint32_t ph = (uint32_t)(i / C::NK) & 1u;
            const int key0 = (j0 + i) * C::KT;
            if (!mbar_wait(&k_empty[of + s], ph ^ 1u, status, P5_ERR_WAIT_ATTN)) {
              flags[0] = 1;
              break;
            }
            mbar_arrive_expect_tx(&k_full[of + s], C::TILE8);
            for (int c = 0; c < C::ATOMS; ++c)
              tma_load_4d(smem + C::K_OFF + s * C::TILE8 + c * C::KT * C::ROWB, &tk, &k_full[of + s], c * C::ROWB, kvh, key0, slot);
            if (!mbar_wait(&v_empty[of + s], ph ^ 1u, status, P5_ERR_WAIT_ATTN)) {
              flags[0] = 1;
              mbar_wait(&k_full[of + s], ph, status, P5_ERR_WAIT_ATTN);
              break;
            }
            mbar_arrive_expect_tx(&v_full[of + s], C::TILE8);
            for (int c = 0; c < C::ATOMS; ++c)
              tma_load_4d(smem + C::V_OFF + s * C::TILE8 + c * C::KT * C::ROWB, &tv, &v_full[of + s], c * C::ROWB, kvh, key0, slot);
            issued = i + 1;
          }
          fp8_drain(k_full + of, C::NK, issued, flags, status);
          fp8_drain(v_full + of, C::NK, issued, flags, status);
        }
        __syncwarp();
      });
    } else if (warp == 1) {
      passes([&](int pass) {
        const int of = pass * C::BARS;
        constexpr uint32_t idesc_s = (1u << 4) | ((uint32_t)(C::KT >> 3) << 17) | (8u << 24);
        // fp16 or bf16, B MN-major
        const uint32_t idesc_o = (1u << 4) | (pass ? (1u << 7) | (1u << 10) : 0u) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | (8u << 24);
        const uint32_t base = smem_u32(smem);
        bool ok = mbar_wait_warp(q_full, 0, status, P5_ERR_WAIT_ATTN);
        // S runs two tiles ahead of P V: its buffer is free as soon as the softmax has read it, long before P is there
        for (int i = 0; i < n + 2 && ok; ++i) {
          if (i < n) {
            const int s = i % C::NK, sb = i & 1;
            ok = mbar_wait_warp(&k_full[of + s], (uint32_t)(i / C::NK) & 1u, status, P5_ERR_WAIT_ATTN) &&
                 (i < C::NS || mbar_wait_warp(&s_empty[of + ((i - C::NS) & 1)], (uint32_t)((i - C::NS) >> 1) & 1u, status, P5_ERR_WAIT_ATTN));
            if (!ok) break;
            tc_fence_after();
            const uint32_t ka = base + C::K_OFF + s * C::TILE8;
            const uint32_t d = tmem + (uint32_t)(C::S_COL + sb % C::NS * C::KT);
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
              for (int kk = 0; kk < HD / 32; ++kk)
                tc_mma_f8_ta(d, tmem + (uint32_t)(C::Q_COL + half * (HD / 4) + kk * 8),
                             HD == 64 ? sw64_kmajor_desc(ka + kk * 32) : sw128_kmajor_desc(ka + (kk >> 2) * (C::KT * 128) + (kk & 3) * 32), idesc_s, (half | kk) ? 1u : 0u);
            tc_commit_warp(&k_empty[of + s]);
            tc_commit_warp(&s_full[of + sb]);
          }
          if (i >= 2) {
            const int j = i - 2, pb = j & 1;
            const uint32_t ph = (uint32_t)(j >> 1) & 1u;
            ok = mbar_wait_warp(&w_full[of + pb], ph, status, P5_ERR_WAIT_ATTN) && mbar_wait_warp(&p_full[of + pb], ph, status, P5_ERR_WAIT_ATTN);
            if (!ok) break;
            tc_fence_after();
            const uint32_t va = base + C::W_OFF + pb * C::TILE16;
#pragma unroll
            for (int kk = 0; kk < C::KT / 16; ++kk)
              tc_mma_f16_ta_warp(tmem + C::O_COL, tmem + (uint32_t)(C::P_COL + pb * (C::KT / 2) + kk * 8),
                                 sw128_mnmajor_desc(va + kk * 2048, C::KT * 128), idesc_o, (j | kk) ? 1u : 0u);
            tc_commit_warp(&w_empty[of + pb]);
            tc_commit_warp(&p_empty[of + pb]);
          }
        }
        if (!ok) flags[0] = 1;
        tc_commit_warp(&o_full[of]);
      });
    } else if (warp == 3) {
      // ---- scales: two keys a lane, loaded a tile ahead
      const long c0 = (long)slot * a.capacity * a.kv_heads + kvh;
      int kb[2], vb[2];
      auto load = [&](int i) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int key = (j0 + i) * C::KT + 2 * lane + q;
          const bool in = i < n && key < top;
          kb[q] = in ? (int)a.ks[c0 + (long)key * a.kv_heads] : 127;
          vb[q] = in ? (int)a.vs[c0 + (long)key * a.kv_heads] : -1;  // no key
        }
      };
      int e_top = -1000, e_low = 1000;      // the largest and the smallest V exponent of the keys
      constexpr int E_UP = 7, E_DOWN = 15;  // an fp16 tile: eb - E_DOWN .. eb + E_UP
      auto scales = [&](auto in_bf16) {
        constexpr bool WIDE = decltype(in_bf16)::value;
        constexpr int of = WIDE ? C::BARS : 0;
        // O's unit: none yet, or one for all tiles
        int eb = WIDE ? max(min(e_low, e_top), e_top - KV8_E_SPAN) : -1000;
        load(0);
        for (int i = 0; i < n; ++i) {
          const int s = i % C::NSC;
          float kf[2];
          uint32_t vf[2];
          int ev[2], kt = 0;
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            kt = max(kt, kb[q] == 255 ? 0 : kb[q]);
            ev[q] = (vb[q] < 0 || vb[q] == 255) ? -1000 : vb[q] - 127;
          }
          // A tile's largest K factor is kept to 2^100, with the rest (kh) for the row's own factor: codes (2^26) and K factor
          // alone, up to 2^146, would leave the float range where the logit does not.
          const int kh = max(__reduce_max_sync(0xffffffffu, kt) - (127 + 100), 0);
#pragma unroll
          for (int q = 0; q < 2; ++q)
            kf[q] = (kb[q] == 255 || vb[q] == 255) ? NAN : exp2_int(kb[q] - 127 - kh);  // a NaN row: NaN for the rows that see it
          load(i + 1);
          float rescale = 1.f;
          if constexpr (!WIDE) {
            // the largest and the smallest exponent; that of a row of zeros (byte 0: or below 2^-117) is never the smallest
            const int em = __reduce_max_sync(0xffffffffu, max(ev[0], ev[1]));
            const int en = __reduce_min_sync(0xffffffffu, min(ev[0] > -127 ? ev[0] : 1000, ev[1] > -127 ? ev[1] : 1000));
            e_top = max(e_top, em);
            e_low = min(e_low, en);
            if (em > eb + E_UP || en < eb - E_DOWN) {
              const int to = en >= em - E_DOWN ? em : em - E_UP;
              // what is already summed must fit the new unit as well
              if (em - en > E_UP + E_DOWN || e_top - to > KV8_E_SPAN || to - e_low > KV8_E_SPAN) flags[2] = 1;
              if (i > 0) rescale = exp2_int(eb - to);  // 0 where there was no exponent yet: O is 0
              eb = to;
            }
          }
#pragma unroll
          for (int q = 0; q < 2; ++q) {  // 2^(ev - eb) for two dims at a time: fp16, at most 2^E_UP, or bf16, at most 2^KV8_E_SPAN
            const int e = ev[q] - eb;
            const uint32_t f = WIDE ? (e < -133 ? 0u : (e < -126 ? 1u << (e + 133) : (uint32_t)(e + 127) << 7))
                                    : (e < -24 ? 0u : (e < -14 ? 1u << (e + 24) : (uint32_t)(e + 15) << 10));
            vf[q] = f * 0x10001u;
          }
          bool ok = !flags[0] && mbar_wait(&sc_empty[of + s], ((uint32_t)(i / C::NSC) & 1u) ^ 1u, status, P5_ERR_WAIT_ATTN);
          if (!__all_sync(0xffffffffu, ok)) {
            flags[0] = 1;
            break;
          }
          float* sc = reinterpret_cast<float*>(smem + C::SC_OFF + s * C::SC_SLOT);
          *reinterpret_cast<float2*>(sc + 2 * lane) = make_float2(kf[0], kf[1]);
          *reinterpret_cast<uint2*>(sc + C::KT + 2 * lane) = make_uint2(vf[0], vf[1]);
          if (lane == 0) {
            *reinterpret_cast<float2*>(sc + 2 * C::KT) = make_float2(rescale, exp2_int(kh));
            flags[1] = eb;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&sc_full[of + s]);
        }
      };
      scales(std::false_type());
      if (__builtin_expect(meet(), 0)) scales(std::true_type());
    } else if (met()) {  // the second pass' barriers, in the first's order
      for (int i = lane; i < C::BARS; i += 32) {
        const uint64_t* b = k_full + i;
        const int count = b >= sc_empty && b < s_full ? 8 : ((b >= v_empty && b < w_empty) || (b >= s_empty && b < p_empty) ? 4 : 1);
        mbar_init(k_full + C::BARS + i, count);
      }
      fence_barrier_init();
      asm volatile("bar.sync 2, 512;" ::: "memory");
    }
  } else if (warp >= 12) {
    regs_dec<C::REG_V>();
    // ---- V codes -> fp16 or bf16, MN-major boxes of 64 dims with the 128-byte swizzle.  Eight lanes take four neighbouring
    // 16-byte pieces of rows r and r ^ 5: their reads and their two writes each hit different banks.
    const int cw = warp - 12;
    auto widen = [&](auto in_bf16) {
      constexpr bool WIDE = decltype(in_bf16)::value;
      constexpr int of = WIDE ? C::BARS : 0;
      if (!mbar_wait_warp(q_full, 0, status, P5_ERR_WAIT_ATTN)) flags[0] = 1;  // Q is staged where widened V goes
      for (int i = 0; i < n; ++i) {
        const int s = i % C::NK, wb = i & 1;
        const int ss = i % C::NSC;
        const bool ok = !flags[0] && mbar_wait(&v_full[of + s], (uint32_t)(i / C::NK) & 1u, status, P5_ERR_WAIT_ATTN) &&
                        mbar_wait(&sc_full[of + ss], (uint32_t)(i / C::NSC) & 1u, status, P5_ERR_WAIT_ATTN) &&
                        mbar_wait(&w_empty[of + wb], ((uint32_t)(i >> 1) & 1u) ^ 1u, status, P5_ERR_WAIT_ATTN);
        if (!__all_sync(0xffffffffu, ok)) {
          flags[0] = 1;
          break;
        }
        const int valid = top - (j0 + i) * C::KT;  // rows from here on become zeros
        const uint8_t* src = smem + C::V_OFF + s * C::TILE8;
        const uint32_t* vf = reinterpret_cast<const uint32_t*>(smem + C::SC_OFF + ss * C::SC_SLOT) + C::KT;
        uint8_t* dst = smem + C::W_OFF + wb * C::TILE16;
#pragma unroll
        for (int k = 0; k < C::KT * HD / 16 / 128; ++k) {
          const int id = k * 128 + cw * 32 + lane;  // [row pair][4 pieces of a group][2 rows] ...
          const int j4 = id & 3, hi = (id >> 2) & 1, rest = id >> 3;
          const int group = rest % (HD / 64), pair = rest / (HD / 64);  // 64-dim box, pair of rows of an 8-row group
          const int row = (pair >> 2) * 8 + ((pair & 3) ^ (hi ? 5 : 0));
          const int piece = group * 4 + j4;  // 16-byte piece of the key's codes
          uint4 u = *reinterpret_cast<const uint4*>(HD == 64 ? src + row * 64 + ((piece ^ ((row >> 1) & 3)) << 4)
                                                             : src + (piece >> 3) * (C::KT * 128) + row * 128 + (((piece & 7) ^ (row & 7)) << 4));
          if (row >= valid) u = make_uint4(0, 0, 0, 0);
          const uint32_t f = vf[row];
          auto two = [&](uint32_t c) {
            const uint32_t h = fp8_to_h2((uint16_t)c);
            if constexpr (WIDE) {
              const uint32_t w = h2_to_bf2(h);
              const __nv_bfloat162 x = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&w), *reinterpret_cast<const __nv_bfloat162*>(&f));
              return *reinterpret_cast<const uint32_t*>(&x);
            } else {
              const __half2 x = __hmul2(*reinterpret_cast<const __half2*>(&h), *reinterpret_cast<const __half2*>(&f));
              return *reinterpret_cast<const uint32_t*>(&x);
            }
          };
          uint8_t* d = dst + group * (C::KT * 128) + row * 128;
          *reinterpret_cast<uint4*>(d + (((2 * j4) ^ (row & 7)) << 4)) = make_uint4(two(u.x), two(u.x >> 16), two(u.y), two(u.y >> 16));
          *reinterpret_cast<uint4*>(d + (((2 * j4 + 1) ^ (row & 7)) << 4)) = make_uint4(two(u.z), two(u.z >> 16), two(u.w), two(u.w >> 16));
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&v_empty[of + s]);
          mbar_arrive(&sc_empty[of + ss]);
          mbar_arrive(&w_full[of + wb]);
        }
      }
    };
    widen(std::false_type());
    if (__builtin_expect(meet(), 0)) widen(std::true_type());
  } else {
    regs_inc<C::REG_SOFT>();
    // ---- softmax: thread = row = TMEM lane; warpgroup g takes the tiles j with j % 2 == g, and half of the head dims of
    // Q and O at the start and the end
    const uint32_t t_lane = tmem + ((uint32_t)(sub * 32) << 16);
    const int lim = !in ? 0 : (a.causal ? min(len, len - tokens + t + 1) : len);
    float row_factor;
    {
      const uint8_t* sq = smem + C::W_OFF;
      cp_async_wait<0>();
      asm volatile("bar.sync 1, 256;" ::: "memory");
      const uint4* src = reinterpret_cast<const uint4*>(sq + r * C::OUT_PITCH + g * HD);
      uint32_t mb = 0;  // the largest magnitude as a bf16 pattern
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) {
        const uint4 u = src[i];
        const uint32_t v = __vmaxu2(__vmaxu2(u.x & 0x7fff7fffu, u.y & 0x7fff7fffu), __vmaxu2(u.z & 0x7fff7fffu, u.w & 0x7fff7fffu));
        mb = max(mb, max(v >> 16, v & 0xffffu));
      }
      exch[g * 128 + r] = __uint_as_float(mb << 16);
      asm volatile("bar.sync 1, 256;" ::: "memory");
      mb = max(__float_as_uint(exch[r]), __float_as_uint(exch[128 + r]));
      const bool bad = mb >= 0x7f800000u;  // a query with a NaN or an infinity: its row is NaN, unless it sees no key
      const int byte = bad ? 127 : fp8_scale_byte(__uint_as_float(mb));
      // the row's factor is >= 0: the sign of the softmax scale goes into Q, and a scale of 0 makes Q zero.  A query with a NaN or an
      // infinity has NaN codes, which make every logit of its row NaN.
      const float sign = a.scale_log2 < 0.f ? -1.f : (a.scale_log2 == 0.f ? 0.f : 1.f);
      const float up = bad ? 0.f : sign * fp8_scale_inverse(byte);
      const float2 up2 = make_float2(up, up);
      row_factor = fp8_scale_value(byte) * fabsf(a.scale_log2);
      constexpr int NC = HD / 8;  // columns of this half: four codes each
      constexpr int CH = NC < 16 ? NC : 16;
#pragma unroll 1
      for (int i = 0; i < NC; i += CH) {
        uint32_t hi[CH], lo[CH];
#pragma unroll
        for (int k = 0; k < CH; k += 2) {
          const uint4 u = src[(i + k) / 2];
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float2 x0 = mul2(unpack_bf2(w[2 * e]), up2), x1 = mul2(unpack_bf2(w[2 * e + 1]), up2);
            // x rounded to the 4 bits of a normal code: c - (c - x) with c = (2^20 + 1) x (Dekker's splitting); where the codes are
            // subnormal the conversion rounds it once more, by at most the 2^-10 that lo is off by anyway
            const float2 c0 = mul2(x0, make_float2(1048577.f, 1048577.f)), c1 = mul2(x1, make_float2(1048577.f, 1048577.f));
            const float2 h0 = sub2(c0, sub2(c0, x0)), h1 = sub2(c1, sub2(c1, x1));
            const float2 l0 = sub2(x0, h0), l1 = sub2(x1, h1);
            hi[k + e] = fp8_pack4(h0.x, h0.y, h1.x, h1.y);
            lo[k + e] = fp8_pack4(l0.x, l0.y, l1.x, l1.y);
          }
        }
        __syncwarp();
        tmem_st_n(t_lane + (uint32_t)(C::Q_COL + g * NC + i), hi);
        tmem_st_n(t_lane + (uint32_t)(C::Q_COL + HD / 4 + g * NC + i), lo);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }
    float* m_ref = exch + 4 * C::ROWS + r;  // the row's running maximum
    float m_run, l_run;
    bool alive;
    auto softmax = [&](auto in_bf16) {
      constexpr bool WIDE = decltype(in_bf16)::value;
      constexpr int of = WIDE ? C::BARS : 0;
      m_run = -INFINITY, l_run = 0.f;
      alive = true;
      for (int j = g; j < n; j += 2) {
        const int ss = j % C::NSC;
        const uint32_t ph = (uint32_t)(j >> 1) & 1u;
        bool ok = !flags[0] && mbar_wait(&sc_full[of + ss], (uint32_t)(j / C::NSC) & 1u, status, P5_ERR_WAIT_ATTN) &&
                  mbar_wait(&s_full[of + g], ph, status, P5_ERR_WAIT_ATTN);
        if (!__all_sync(0xffffffffu, ok)) {
          flags[0] = 1;
          alive = false;
          break;
        }
        tc_fence_after();
        const float* sc = reinterpret_cast<const float*>(smem + C::SC_OFF + ss * C::SC_SLOT);
        float x[C::KT];
        {
          uint32_t lo[32], hi[32];
          tmem_ld32(t_lane + (uint32_t)(C::S_COL + g % C::NS * C::KT), lo);
          tmem_ld32(t_lane + (uint32_t)(C::S_COL + g % C::NS * C::KT + 32), hi);
          tmem_wait_ld();
#pragma unroll
          for (int c = 0; c < 32; ++c) x[c] = __uint_as_float(lo[c]), x[32 + c] = __uint_as_float(hi[c]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_empty[of + g]);
        const int valid = lim - (j0 + j) * C::KT;  // columns of the tile that this row sees (may be <= 0)
        // each column by its key's power of two
#pragma unroll
        for (int c = 0; c < C::KT; c += 4) {
          const float4 k = *reinterpret_cast<const float4*>(sc + c);
          const float2 a0 = mul2(make_float2(x[c], x[c + 1]), make_float2(k.x, k.y));
          const float2 a1 = mul2(make_float2(x[c + 2], x[c + 3]), make_float2(k.z, k.w));
          x[c] = a0.x, x[c + 1] = a0.y, x[c + 2] = a1.x, x[c + 3] = a1.y;
        }
        if (valid < C::KT) {
#pragma unroll
          for (int c = 0; c < C::KT; ++c)
            if (c >= valid) x[c] = -INFINITY;
        }
        float mx[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) mx[k] = fmaxf(x[k], x[8 + k]);
#pragma unroll
        for (int c = 16; c < C::KT; c += 16)
#pragma unroll
          for (int k = 0; k < 8; ++k) mx[k] = fmax3(mx[k], x[c + k], x[c + 8 + k]);
        // in base 2: rf carries the row's power of two, the softmax scale, log2 e and the unit of the K factors.  It is positive
        // and finite, so that a masked logit of -inf stays one and a sum of 0 gives 0; the smallest float makes no logit of 2^-23.
        const float2 tile = *reinterpret_cast<const float2*>(sc + 2 * C::KT);
        const float rf = fminf(fmaxf(row_factor * tile.y, 1.4012985e-45f), 3.4028235e38f);
        const float mt = fmaxf(fmax3(mx[0], mx[1], mx[2]), fmax3(mx[3], mx[4], fmax3(mx[5], mx[6], mx[7]))) * rf;
        const float rescale = tile.x;
        __syncwarp();
        if (lane == 0) mbar_arrive(&sc_empty[of + ss]);
        bool need = rescale != 1.f;
        float alpha = rescale, m = mt;
        if (j > 0) {  // the turn: the maximum after tile j - 1
          ok = mbar_wait(&turn[of + 4 * g + sub], (uint32_t)((j >> 1) - 1 + g) & 1u, status, P5_ERR_WAIT_ATTN);
          const float before = *m_ref;
          m = before;
          if (mt > before + 8.f) {
            need = true;
            m = mt;
            alpha *= before == -INFINITY ? 0.f : ex2_approx(before - mt);
          }
        }
        *m_ref = m;
        __syncwarp();
        if (lane == 0) mbar_arrive(&turn[of + 4 * (g ^ 1) + sub]);
        l_run *= m_run == m ? 1.f : (m_run == -INFINITY ? 0.f : ex2_approx(m_run - m));
        m_run = m;
        const float msc = m == -INFINITY ? 0.f : m - 7.f;  // p and l as 2^7 of themselves, which O / l forgets
        float2 ls[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        const float2 rf2 = make_float2(rf, rf), nm2 = make_float2(-msc, -msc);
        uint32_t pk[C::KT / 2];
#pragma unroll
        for (int c = 0; c < C::KT; c += 4) {
          const float2 x0 = fma2(make_float2(x[c], x[c + 1]), rf2, nm2);
          const float2 x1 = fma2(make_float2(x[c + 2], x[c + 3]), rf2, nm2);
          const float2 p0 = make_float2(ex2_approx(x0.x), ex2_approx(x0.y)), p1 = make_float2(ex2_approx(x1.x), ex2_approx(x1.y));
          ls[0] = add2(ls[0], p0);
          ls[1] = add2(ls[1], p1);
          if constexpr (WIDE) {
            pk[c / 2] = pack_bf2(p0.x, p0.y);
            pk[c / 2 + 1] = pack_bf2(p1.x, p1.y);
          } else {
            const __half2 h0 = __floats2half2_rn(p0.x, p0.y), h1 = __floats2half2_rn(p1.x, p1.y);
            pk[c / 2] = *reinterpret_cast<const uint32_t*>(&h0);
            pk[c / 2 + 1] = *reinterpret_cast<const uint32_t*>(&h1);
          }
        }
        l_run += (ls[0].x + ls[0].y) + (ls[1].x + ls[1].y);
        // P buffer g was last read by the P V product of tile j - 2
        ok = ok && mbar_wait(&p_empty[of + g], ph ^ 1u, status, P5_ERR_WAIT_ATTN);
        __syncwarp();
        tc_fence_after();
        tmem_st32(t_lane + (uint32_t)(C::P_COL + g * (C::KT / 2)), pk);
        tmem_wait_st();
        if (j > 0 && __any_sync(0xffffffffu, need)) {
          // wait for the P V product of tile j - 1, then rescale this warp's rows of O
          ok = ok && mbar_wait(&p_empty[of + (g ^ 1)], (uint32_t)((j - 1) >> 1) & 1u, status, P5_ERR_WAIT_ATTN);
          if (__all_sync(0xffffffffu, ok)) {
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < HD; c += 32) {
              uint32_t o[32];
              tmem_ld32(t_lane + (uint32_t)(C::O_COL + c), o);
              tmem_wait_ld();
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
              tmem_st32(t_lane + (uint32_t)(C::O_COL + c), o);
            }
            tmem_wait_st();
          }
        }
        if (!__all_sync(0xffffffffu, ok)) {
          flags[0] = 1;
          alive = false;
          break;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[of + g]);
      }
      alive = mbar_wait(&o_full[of], 0, status, P5_ERR_WAIT_ATTN) && alive;
    };
    softmax(std::false_type());
    if (__builtin_expect(meet(), 0)) softmax(std::true_type());
    const uint32_t t_o = t_lane + (uint32_t)(C::O_COL + g * (HD / 2));

    // ---- O / l, of the split where there are more
    tc_fence_after();
    const bool good = __all_sync(0xffffffffu, alive) && !flags[0];
    // the later tile's maximum is the larger; O is in units of it
    exch[g * 128 + r] = l_run;
    exch[(2 + g) * 128 + r] = m_run;
    asm volatile("bar.sync 1, 256;" ::: "memory");
    const float m0 = exch[256 + r], m1 = exch[384 + r];
    m_run = fmaxf(m0, m1);
    const float l = (m0 == m_run ? 1.f : ex2_approx(m0 - m_run)) * exch[r] + (m1 == m_run ? 1.f : ex2_approx(m1 - m_run)) * exch[128 + r];
    const float unit = exp2_int(n > 0 ? (int)flags[1] : 0);
    // l is 0 for a row without keys (its output is 0), NaN for one that sees a NaN
    const float f = l == 0.f ? 0.f : unit / l;
    const long part = ((long)split * (gridDim.y / a.kv_heads) + b) * ((long)a.T * a.heads);
#pragma unroll 1
    for (int c = 0; c < HD / 2; c += 32) {
      uint32_t o[32];
      __syncwarp();
      tmem_ld32(t_o + (uint32_t)c, o);
      tmem_wait_ld();
      if (n == 0) {  // no MMA wrote this accumulator
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] = 0u;
      }
      if (a.groups == 1) {
        uint4* dst = reinterpret_cast<uint4*>(smem + r * C::OUT_PITCH + (g * (HD / 2) + c) * 2);
#pragma unroll
        for (int q = 0; q < 4; ++q)
          dst[q] = make_uint4(pack_bf2(__uint_as_float(o[8 * q]) * f, __uint_as_float(o[8 * q + 1]) * f),
                              pack_bf2(__uint_as_float(o[8 * q + 2]) * f, __uint_as_float(o[8 * q + 3]) * f),
                              pack_bf2(__uint_as_float(o[8 * q + 4]) * f, __uint_as_float(o[8 * q + 5]) * f),
                              pack_bf2(__uint_as_float(o[8 * q + 6]) * f, __uint_as_float(o[8 * q + 7]) * f));
      } else if (in && good) {
        float4* dst = reinterpret_cast<float4*>(a.ws_o + (part + (long)h * a.T + t) * HD + g * (HD / 2) + c);
#pragma unroll
        for (int q = 0; q < 8; ++q)
          dst[q] = make_float4(__uint_as_float(o[4 * q]) * f, __uint_as_float(o[4 * q + 1]) * f, __uint_as_float(o[4 * q + 2]) * f,
                               __uint_as_float(o[4 * q + 3]) * f);
      }
    }
    if (a.groups > 1) {
      if (in && good && g == 0) a.ws_ml[part + (long)h * a.T + t] = make_float2(m_run, l);
    } else {
      // staged above (K and V buffers are idle: every MMA is done); each thread sends its half row by one bulk copy
      fence_proxy_async_smem();
      if (good && in) {
        bulk_store_global(a.out + (long)b * a.o_b + (long)t * a.o_t + (long)h * HD + g * (HD / 2),
                          smem_u32(smem + r * C::OUT_PITCH + g * HD), HD);
        bulk_store_wait_read();  // the staging must outlive the copy's reads
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 2) tmem_dealloc(tmem, 512);
}

}  // namespace p5
