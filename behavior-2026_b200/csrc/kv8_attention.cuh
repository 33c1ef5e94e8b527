// kv8_attention.cuh — attention over the 8-bit K/V cache (fp8.cuh) for few query rows.
//
//   out[b][t][h][:] = sum_j p_j V_j,  p = softmax_j(scale * q . K_j),  j < lens[b] (causal: j < lens[b] - n + t + 1)
// for the tokens t < n of sample b, n = count[b] (T without counts)
//
// The query heads of a K/V head and the T tokens of a sample are folded into rows r = t * G + g.  A CTA owns 8 of the
// rows of one (sample, K/V head) and one key split; its warps walk steps of 32 keys, each warp the steps w, w + W, ... of the
// split with a running maximum and sum of its own, merged through shared memory at the end, then over the cluster's
// CTAs (the neighbouring splits) through distributed shared memory, then, where there are more splits than a cluster
// holds, by kv8_attn_combine_kernel.
//
// One new token reads the whole cache once for a handful of products, so what counts is bytes in flight: each warp
// keeps a ring of its own of STAGES steps (cp.async, no barrier between warps), 48 to 192 KB an SM.  Measured, 16 samples of 32
// heads on 8 of 128: 46 us and 5.8 TB/s at 8,192 keys each, 71 us and 4.9 TB/s at 4,000 to 16,387 (the longest sample decides);
// one sample of 1,018 keys on one head of 256 9.9 us, its chain of latencies, of 30,000 25 us.
//
// Everything is computed transposed, keys and head dims on the 16-row side of mma.m16n8k16 and query rows on
// the 8-column side, because one token of 8 heads has 8 rows, not 16:
//   S^T[16 keys][8 rows] = K Q^T      O^T[16 dims][8 rows] += V^T P^T
// The order of the reduction index and of the output rows of an MMA is free, so each thread takes the operands
// that it can read in 16-byte pieces: lane (g, c) = (lane / 4, lane % 4) holds head dims 64 i + 16 c .. + 15 of
// keys g and g + 8, and head dims 128 i + 16 g .. + 15 of keys 2c, 2c + 1, 2c + 8, 2c + 9, widened to fp16 in
// registers (exact).  P^T goes from the accumulator layout to the operand layout by movmatrix.
//
// fp16 operands: a query row is scaled by a power of two so that its largest element is near 2^15 (elements
// down to 2^-29 of it keep all 8 bits of a bf16); P carries the V row's scale relative to an exponent eb of the warp
// (p * 2^(ev - eb)).  Logits, maxima, sums and O are fp32.
// The running maximum moves only when a logit exceeds it by 2^4, and eb only when a scale leaves eb .. eb + 11, so
// p * 2^(ev - eb) stays within 2^15, a weight keeps 11 bits (or 2^-25 of the largest) whatever other keys' scales are, and O is
// rarely rescaled.  A step whose scales span more than that (a key that a row does not see counts as well: its scale must
// not push that row's weights below the range) takes V and P in bf16, P as two operands hi + lo (16 bits): any scale fits
// (every step so: 60 us for the 46 above).
#pragma once
#include <type_traits>

#include "fp8.cuh"

namespace p5 {

struct Kv8Args {
  const bf16* q;
  long q_b, q_t;  // elements between samples, tokens; heads are head_dim apart
  const uint8_t *k, *ks, *v, *vs;
  const int* lens;
  const int* count;  // query tokens of a sample; NULL: T
  const int* slots;  // NULL: sample b is slot b
  bf16* out;
  long o_b, o_t;
  float scale_log2;  // scale * log2(e)
  int n_slots, capacity, T, heads, kv_heads, G, causal;
  int splits, groups;  // key splits, and clusters of them: splits = groups * CTAs of a cluster
  float* ws_o;         // [groups][batch][heads * T][head_dim], O / l of the group: never above the largest |V|
  float2* ws_ml;       // [groups][batch][heads * T] (m, l)
};

// query tokens of sample b
__device__ __forceinline__ int kv8_tokens(const Kv8Args& a, int b) { return a.count ? max(0, min(a.count[b], a.T)) : a.T; }

__device__ __forceinline__ uint32_t movmatrix_b16(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ void mma_f16_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// the smaller one; NaN if either is
__device__ __forceinline__ float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// two fp16 -> two bf16 (exact for widened e4m3 codes: 4 bits)
__device__ __forceinline__ uint32_t h2_to_bf2(uint32_t h) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
  return pack_bf2(f.x, f.y);
}
// Exponents of V scales that one accumulator holds.  A term is at most 2^15 (weight) * 2^9 (code) * 2^(scale - unit), summed over up
// to 2^28 keys, so scales up to 2^64 above the unit (and the rest of a window) stay within the fp32 range; and a unit at most
// 2^64 above the smallest scale leaves rows that see only that one all their bits.
constexpr int KV8_E_SPAN = 64;
// 2^n for any integer n (0 below 2^-127, 2^127 above)
__device__ __forceinline__ float exp2_int(int n) {
  return n < -127 ? 0.f : __uint_as_float(n == -127 ? 0x400000u : (uint32_t)(min(n, 127) + 127) << 23);
}
// x 2^n for n from -252 to 127
__device__ __forceinline__ float mul_exp2(float x, int n) { return x * exp2_int(max(n, -126)) * exp2_int(min(n + 126, 0)); }

template <int HD>
struct Kv8RowsCfg {
  static constexpr int W = 4, KEYS = 32, STAGES = 3;
  static constexpr int HALF = KEYS * HD, STAGE = 2 * HALF;  // bytes of a step: K rows, V rows
  static constexpr int SMEM = W * STAGES * STAGE;
  static constexpr int PER_SM = HD == 256 ? 1 : (HD == 128 ? 2 : 4);
  static_assert(8 * HD * 4 <= STAGES * STAGE, "a warp's O tile is staged in its ring");
};

// byte offset of 16-byte piece p of key row `key` of a stage.  Pieces are swizzled so that the eight lanes of a
// 16-byte (V of HD 64: sixteen of an 8-byte) access hit different banks: K pieces 4 i + c of keys g, g + 1, V pieces g, g + 1 of
// keys 2 c.
template <int HD>
__device__ __forceinline__ int kv8_k_at(int key, int p) {
  return HD == 64 ? key * 64 + p * 16 : key * HD + ((p ^ ((key & 1) << 2)) << 4);
}
template <int HD>
__device__ __forceinline__ int kv8_v_at(int key, int p) {
  return HD == 64 ? (key >> 1) * 128 + (((key & 1) ^ ((key >> 1) & 1)) << 6) + ((p ^ (((key >> 2) & 1) << 1)) << 4)
                  : key * HD + ((p ^ (key & 6)) << 4);
}

template <int HD>
__global__ void __launch_bounds__(32 * Kv8RowsCfg<HD>::W, Kv8RowsCfg<HD>::PER_SM)
    kv8_attn_rows_kernel(const Kv8Args a) {
  using C = Kv8RowsCfg<HD>;
  constexpr int W = C::W, KI = HD / 64, VI = HD >= 128 ? HD / 128 : 1;
  constexpr int VB = HD >= 128 ? 16 : 8;  // bytes of a lane's V piece
  constexpr int MT = HD / 16;             // 16-dim tiles of O^T
  constexpr int PIECES = HD / 16;         // 16-byte pieces of a key row
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float sm_m[W][8], sm_l[W][8];
  __shared__ int sm_e[W];
  __shared__ float cta_m[8], cta_l[8];
  __shared__ int cta_e;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int b = blockIdx.y / a.kv_heads, kvh = blockIdx.y % a.kv_heads;
  const int tokens = kv8_tokens(a, b), rows = tokens * a.G, row0 = blockIdx.x * 8;
  const int split = blockIdx.z;
  const int slot = a.slots ? a.slots[b] : b;
  const int len = (slot < 0 || slot >= a.n_slots) ? 0 : max(0, min(a.lens[b], a.capacity));
  // keys that any of the CTA's rows sees
  const int t_last = min(row0 + 8, rows) - 1;
  const int top = row0 >= rows ? 0 : (a.causal ? max(0, min(len, len - tokens + t_last / a.G + 1)) : len);
  // the split's steps
  const int steps = (top + C::KEYS - 1) / C::KEYS;
  const int per = (steps + a.splits - 1) / a.splits;
  const int s_begin = min(split * per, steps), s_end = min(s_begin + per, steps);

  const long key_pitch = (long)a.kv_heads * HD;
  const long cache0 = (long)slot * a.capacity * a.kv_heads + kvh;  // in heads
  const uint8_t* kp = a.k + cache0 * HD;
  const uint8_t* vp = a.v + cache0 * HD;
  const uint8_t* ksp = a.ks + cache0;
  const uint8_t* vsp = a.vs + cache0;
  uint8_t* ring = smem + warp * C::STAGES * C::STAGE;

  // One step's K and V rows into a stage (keys from `top` on become zeros), and this lane's scale bytes: K and V of
  // key `lane`.  255 where there is no key: no exponent of its own, and its p is 0.
  int kq[C::STAGES], vq[C::STAGES];
  auto fetch = [&](int step, int st) {
    if (step < s_end) {
      const int key0 = step * C::KEYS;
      uint8_t* dst = ring + st * C::STAGE;
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int q = i * 32 + lane, key = q / PIECES, p = q % PIECES;
        const bool in = key0 + key < top;
        const long off = in ? (long)(key0 + key) * key_pitch + 16 * p : 0;
        cp_async16(dst + kv8_k_at<HD>(key, p), kp + off, in);
        cp_async16(dst + C::HALF + kv8_v_at<HD>(key, p), vp + off, in);
      }
      const bool in = key0 + lane < top;
      kq[st] = in ? (int)ksp[(long)(key0 + lane) * a.kv_heads] : 255;
      vq[st] = in ? (int)vsp[(long)(key0 + lane) * a.kv_heads] : 255;
    }
    cp_async_commit();
  };
  int step = s_begin + warp;
#pragma unroll
  for (int i = 0; i < C::STAGES - 1; ++i) fetch(step + i * W, i);

  // ---- Q^T operand: row g, scaled to fp16
  uint32_t qf[KI][8];
  float rf[2];  // this thread's accumulator columns: rows 2c, 2c + 1
  int lim[2];
  {
    const int r = row0 + g;
    const bool in = r < rows;
    const int t = in ? r / a.G : 0, h = kvh * a.G + (in ? r % a.G : 0);
    const bf16* src = a.q + (long)b * a.q_b + (long)t * a.q_t + (long)h * HD;
    uint32_t mb = 0;
#pragma unroll
    for (int i = 0; i < KI; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint4 u = in ? *reinterpret_cast<const uint4*>(src + 64 * i + 16 * c + 8 * j) : make_uint4(0, 0, 0, 0);
        qf[i][4 * j] = u.x, qf[i][4 * j + 1] = u.y, qf[i][4 * j + 2] = u.z, qf[i][4 * j + 3] = u.w;
      }
#pragma unroll
    for (int i = 0; i < KI; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) mb = __vmaxu2(mb, qf[i][j] & 0x7fff7fffu);  // magnitudes as bf16 patterns
    mb = max(mb >> 16, mb & 0xffffu);
    mb = max(mb, __shfl_xor_sync(0xffffffffu, mb, 1));
    mb = max(mb, __shfl_xor_sync(0xffffffffu, mb, 2));
    // |q| < 2^(e + 1); the row is scaled by 2^(14 - e) (kept within the float range)
    const int e = min(max((int)(mb >> 7) - 127, -112), 127);
    // a query with a NaN or an infinity: its row is NaN, unless it sees no key.  The sign of the softmax scale goes into Q.
    const float up = mb >= 0x7f80u ? NAN : (a.scale_log2 < 0.f ? -exp2_int(14 - e) : exp2_int(14 - e));
#pragma unroll
    for (int i = 0; i < KI; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 f = unpack_bf2(qf[i][j]);
        const __half2 hh = __floats2half2_rn(f.x * up, f.y * up);
        qf[i][j] = *reinterpret_cast<const uint32_t*>(&hh);
      }
    const float down = fminf(fabsf(a.scale_log2) * exp2_int(e - 14), 3.4028235e38f);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      rf[j] = __shfl_sync(0xffffffffu, down, (2 * c + j) * 4);
      const int rr = row0 + 2 * c + j;
      lim[j] = rr >= rows ? 0 : (a.causal ? min(len, len - tokens + rr / a.G + 1) : len);
    }
  }

  float o[MT][4];
  float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
  int eb = -1000;              // O is in units of 2^eb (-1000: no V scale yet, O is 0)
  int e_top = -1000, e_low = 1000;  // the largest and the smallest V exponent so far, a window's width loose
  constexpr int E_WINDOW = 11;  // fp16 steps: eb .. eb + E_WINDOW
#pragma unroll
  for (int i = 0; i < MT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

  for (; step < s_end;) {
#pragma unroll
    for (int st = 0; st < C::STAGES; ++st) {
      if (step >= s_end) break;
      cp_async_wait<C::STAGES - 2>();
      __syncwarp();
      // the stage of the step before last is free: every lane has read it
      fetch(step + (C::STAGES - 1) * W, (st + C::STAGES - 1) % C::STAGES);
      const uint8_t* sk = ring + st * C::STAGE;
      const uint8_t* sv = sk + C::HALF;
      // ---- S^T = K Q^T, two chains a 16-key tile
      float s[2][4], s2[2][4];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = s2[n][e] = 0.f;
#pragma unroll
      for (int i = 0; i < KI; ++i)
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const uint4 u0 = *reinterpret_cast<const uint4*>(sk + kv8_k_at<HD>(16 * n + g, 4 * i + c));
          const uint4 u1 = *reinterpret_cast<const uint4*>(sk + kv8_k_at<HD>(16 * n + g + 8, 4 * i + c));
          const uint32_t w0[4] = {u0.x, u0.y, u0.z, u0.w}, w1[4] = {u1.x, u1.y, u1.z, u1.w};
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            const uint32_t af[4] = {fp8_to_h2((uint16_t)w0[p]), fp8_to_h2((uint16_t)w1[p]), fp8_to_h2((uint16_t)(w0[p] >> 16)),
                                    fp8_to_h2((uint16_t)(w1[p] >> 16))};
            mma_f16_16816(p & 1 ? s2[n] : s[n], af, qf[i][2 * p], qf[i][2 * p + 1]);
          }
        }
      // ---- logits in base 2; a cached NaN row (scale byte 255) makes the rows that see it NaN
      const int key0 = step * C::KEYS + g;
      const int kb = kq[st], vb = vq[st];  // of key `lane`
      const float kf1 = (kb == 255 || vb == 255) ? NAN : fp8_scale_value(kb);
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const float kf = __shfl_sync(0xffffffffu, kf1, 16 * n + 8 * q + g);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            // the row's and the key's factors first: each may be near the float range where their product is not (and where
            // that passes it, a sum of 0 is still a logit of 0)
            const float x = (s[n][2 * q + j] + s2[n][2 * q + j]) * min_nan(rf[j] * kf, 3.4028235e38f);
            s[n][2 * q + j] = key0 + 16 * n + 8 * q < lim[j] ? x : -INFINITY;
          }
        }
      float mt[2];
      // a scale outside the window; that of a row of zeros (byte 0: or below 2^-117) counts only where there is no window yet
      bool grow = vb != 255 && (uint32_t)(vb - 127 - eb) > (uint32_t)E_WINDOW && (vb != 0 || eb == -1000);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        mt[j] = fmaxf(fmaxf(s[0][j], s[0][2 + j]), fmaxf(s[1][j], s[1][2 + j]));
        grow |= mt[j] > m_run[j] + 4.f;
      }
      bool wide = false;  // this step's products in bf16
      if (__any_sync(0xffffffffu, grow)) {
        const int em = __reduce_max_sync(0xffffffffu, vb == 255 ? -1000 : vb - 127);
        int en = __reduce_min_sync(0xffffffffu, vb == 255 || vb == 0 ? 1000 : vb - 127), to = eb;
        if (em > eb + E_WINDOW || en < eb) {
          e_low = min(e_low, en);
          en = min(en, em);
          e_top = max(e_top, em);
          to = max(min(en, em - 9), -127);  // a little room above
          // what is already summed must fit the new unit as well
          wide = em - en > E_WINDOW || e_top - to > KV8_E_SPAN || to - e_low > KV8_E_SPAN;
          if (wide) to = eb == -1000 ? max(en, em - KV8_E_SPAN) : max(eb, em - KV8_E_SPAN);
          else if (e_low < 1000) e_low = min(e_low, to);
        }
        const float ealpha = exp2_int(eb - to);  // 0 at first, when O is 0 anyway
        eb = to;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float m = mt[j];
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
          m = fmaxf(m, m_run[j]);
          const float alpha = m_run[j] == -INFINITY ? 0.f : ex2_approx(m_run[j] - m);
          m_run[j] = m;
          l_run[j] *= alpha;
          const float al = alpha * ealpha;
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            o[i][j] *= al;
            o[i][2 + j] *= al;
          }
        }
      }
      // ---- P^T, each key's V scale folded in, and O^T += V^T P^T: tile (i, j) holds dims 16 g + 2 j and + 1 of the 128-dim
      // part i.  WIDE: in bf16, P as hi + lo.
      auto product = [&](auto in_bf16) {
        constexpr bool WIDE = decltype(in_bf16)::value;
        const float vf1 = vb == 255 ? 0.f : __uint_as_float((uint32_t)max(vb - eb, 0) << 23);  // 2^(vb - 127 - eb), at most 2^KV8_E_SPAN
        uint32_t pf[2][2], pl[2][2];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const float vf = __shfl_sync(0xffffffffu, vf1, 16 * n + 8 * q + g);
            float p[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              p[j] = ex2_approx(s[n][2 * q + j] - (m_run[j] == -INFINITY ? 0.f : m_run[j]));
              l_run[j] += p[j];
              p[j] *= vf;
            }
            if constexpr (WIDE) {
              const uint32_t hi = pack_bf2(p[0], p[1]);
              const float2 f = unpack_bf2(hi);
              pf[n][q] = movmatrix_b16(hi);
              pl[n][q] = movmatrix_b16(pack_bf2(p[0] - f.x, p[1] - f.y));
            } else {
              const __half2 h = __floats2half2_rn(p[0], p[1]);
              pf[n][q] = movmatrix_b16(*reinterpret_cast<const uint32_t*>(&h));
            }
          }
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int i = 0; i < VI; ++i) {
            uint32_t w[4][4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int key = 16 * n + 2 * c + (k & 1) + 8 * (k >> 1);
              if (VB == 16) {
                const uint4 u = *reinterpret_cast<const uint4*>(sv + kv8_v_at<HD>(key, 8 * i + g));
                w[k][0] = u.x, w[k][1] = u.y, w[k][2] = u.z, w[k][3] = u.w;
              } else {
                const uint2 u = *reinterpret_cast<const uint2*>(sv + kv8_v_at<HD>(key, g >> 1) + (g & 1) * 8);
                w[k][0] = u.x, w[k][1] = u.y;
              }
            }
#pragma unroll
            for (int q = 0; q < VB / 4; ++q)
#pragma unroll
              for (int hlf = 0; hlf < 2; ++hlf) {
                // bytes (2 hlf, 2 hlf + 1) of the word of two keys, interleaved by key
                const uint32_t lo = __byte_perm(w[0][q], w[1][q], hlf ? 0x7362 : 0x5140);
                const uint32_t hi = __byte_perm(w[2][q], w[3][q], hlf ? 0x7362 : 0x5140);
                uint32_t af[4] = {fp8_to_h2((uint16_t)lo), fp8_to_h2((uint16_t)(lo >> 16)), fp8_to_h2((uint16_t)hi),
                                  fp8_to_h2((uint16_t)(hi >> 16))};
                float(&acc)[4] = o[i * (VB / 2) + 2 * q + hlf];
                if constexpr (WIDE) {
#pragma unroll
                  for (int k = 0; k < 4; ++k) af[k] = h2_to_bf2(af[k]);
                  mma_bf16_16816(acc, af, pf[n][0], pf[n][1]);
                  mma_bf16_16816(acc, af, pl[n][0], pl[n][1]);
                } else {
                  mma_f16_16816(acc, af, pf[n][0], pf[n][1]);
                }
              }
          }
      };
      if (wide)
        product(std::true_type());
      else
        product(std::false_type());
      step += W;
    }
  }
  cp_async_wait<0>();

  // ---- merge the warps: maxima and exponents first, then O in warp order (reruns give the same bits)
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) l_run[j] += __shfl_xor_sync(0xffffffffu, l_run[j], d);
  if (g == 0) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      sm_m[warp][2 * c + j] = m_run[j];
      sm_l[warp][2 * c + j] = l_run[j];
    }
  }
  if (lane == 0) sm_e[warp] = e_top;
  __syncthreads();
  // one unit for all: warps that saw only small rows keep their bits beside one that saw only a large one
  int e_all = -1000;
#pragma unroll
  for (int w = 0; w < W; ++w) e_all = max(e_all, sm_e[w]);
  e_all = max(e_all - KV8_E_SPAN, -127);
  const float e1 = exp2_int(max(eb - e_all, -126)), e2 = exp2_int(min(eb - e_all + 126, 0));
  float* tile = reinterpret_cast<float*>(smem);  // [W][8][HD], each warp's in its own ring
  constexpr int TILE = C::STAGES * C::STAGE / 4;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) m = fmaxf(m, sm_m[w][2 * c + j]);
    const float f = m_run[j] == -INFINITY ? 0.f : ex2_approx(m_run[j] - m) * e2;
    float* dst = tile + warp * TILE + (2 * c + j) * HD;
#pragma unroll
    for (int i = 0; i < VI; ++i)
#pragma unroll
      for (int q = 0; q < VB; q += 4) {
        const int k = i * (VB / 2) + q / 2;
        *reinterpret_cast<float4*>(dst + 128 * i + VB * g + q) =
            make_float4(o[k][j] * e1 * f, o[k][2 + j] * e1 * f, o[k + 1][j] * e1 * f, o[k + 1][2 + j] * e1 * f);
      }
  }
  if (threadIdx.x < 8) {
    const int r = threadIdx.x;
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) m = fmaxf(m, sm_m[w][r]);
#pragma unroll
    for (int w = 0; w < W; ++w) l += sm_m[w][r] == -INFINITY ? sm_l[w][r] : sm_l[w][r] * ex2_approx(sm_m[w][r] - m);  // 0 or NaN
    cta_m[r] = m;
    cta_l[r] = l;
  }
  if (threadIdx.x == 0) cta_e = e_all;
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * HD; i += 32 * W) {  // 8 rows of HD in float4s, summed into the first warp's tile
    float4 x = reinterpret_cast<const float4*>(tile)[i];
#pragma unroll
    for (int w = 1; w < W; ++w) {
      const float4 y = reinterpret_cast<const float4*>(tile + w * TILE)[i];
      x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
    }
    reinterpret_cast<float4*>(tile)[i] = x;
  }

  // ---- merge the cluster's CTAs: CTA p finishes rows p, p + size, ... , in rank order
  const int size = a.splits / a.groups, rank = split % size, group = split / size;
  if (size > 1)
    cluster_sync();
  else
    __syncthreads();
  const int out_rows = a.T * a.heads;
  for (int r = rank + size * warp; r < 8; r += size * W) {
    const int row = row0 + r;
    if (row >= rows) continue;
    float m = -INFINITY, l = 0.f, x[HD / 32];
    int e = -1000;
#pragma unroll
    for (int k = 0; k < HD / 32; ++k) x[k] = 0.f;
    for (int p = 0; p < size; ++p) {
      m = fmaxf(m, size > 1 ? ld_peer_f32(map_peer(smem_u32(&cta_m[r]), p)) : cta_m[r]);
      e = max(e, size > 1 ? __float_as_int(ld_peer_f32(map_peer(smem_u32(&cta_e), p))) : cta_e);
    }
    for (int p = 0; p < size; ++p) {
      const float mp = size > 1 ? ld_peer_f32(map_peer(smem_u32(&cta_m[r]), p)) : cta_m[r];
      const float lp = size > 1 ? ld_peer_f32(map_peer(smem_u32(&cta_l[r]), p)) : cta_l[r];
      const int ep = size > 1 ? __float_as_int(ld_peer_f32(map_peer(smem_u32(&cta_e), p))) : cta_e;
      const float f = mp == -INFINITY ? 0.f : ex2_approx(mp - m);
      l += mp == -INFINITY ? lp : lp * f;
#pragma unroll
      for (int k = 0; k < HD / 64; ++k) {
        const float* q = tile + r * HD + 64 * k + 2 * lane;
        const uint32_t at = size > 1 ? map_peer(smem_u32(q), p) : 0u;
        x[2 * k] += f * mul_exp2(size > 1 ? ld_peer_f32(at) : q[0], ep - e);
        x[2 * k + 1] += f * mul_exp2(size > 1 ? ld_peer_f32(at + 4) : q[1], ep - e);
      }
    }
    const float unit = exp2_int(e);
    const int t = row / a.G, h = kvh * a.G + row % a.G;
    // l is 0 for a row without keys (its output is 0), NaN for one that sees a NaN
    const float inv = l == 0.f ? 0.f : unit / l;
    if (a.groups == 1) {
      bf16* dst = a.out + (long)b * a.o_b + (long)t * a.o_t + (long)h * HD;
#pragma unroll
      for (int k = 0; k < HD / 64; ++k)
        *reinterpret_cast<uint32_t*>(dst + 64 * k + 2 * lane) = pack_bf2(x[2 * k] * inv, x[2 * k + 1] * inv);
    } else {
      const long i = ((long)group * (gridDim.y / a.kv_heads) + b) * out_rows + (long)h * a.T + t;
#pragma unroll
      for (int k = 0; k < HD / 64; ++k)
        *reinterpret_cast<float2*>(a.ws_o + i * HD + 64 * k + 2 * lane) = make_float2(x[2 * k] * inv, x[2 * k + 1] * inv);
      if (lane == 0) a.ws_ml[i] = make_float2(m, l);
    }
  }
  if (size > 1) {
    __syncwarp();
    cluster_sync();  // no CTA leaves while a peer reads its shared memory
  }
}

// Joins the groups of key splits of a row: out = sum_s w_s O_s / sum_s w_s with w_s = 2^(m_s - m) l_s, in order.
// One warp a row.
template <int HD>
__global__ void kv8_attn_combine_kernel(const Kv8Args a, int batch) {
  const int lane = threadIdx.x & 31;
  const long rows = (long)batch * a.T * a.heads;
  const long i = (long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (i >= rows || (a.count && (int)(i % a.T) >= kv8_tokens(a, (int)(i / ((long)a.T * a.heads))))) return;
  float2 ml[2];  // lane: groups lane and lane + 32 (there are at most 64)
#pragma unroll
  for (int k = 0; k < 2; ++k) ml[k] = lane + 32 * k < a.groups ? a.ws_ml[(lane + 32 * k) * rows + i] : make_float2(-INFINITY, 0.f);
  float m = fmaxf(ml[0].x, ml[1].x);
#pragma unroll
  for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  float w[2], l;
#pragma unroll
  for (int k = 0; k < 2; ++k) w[k] = ml[k].x == -INFINITY && ml[k].y == 0.f ? 0.f : ml[k].y * ex2_approx(ml[k].x - m);
  l = w[0] + w[1];
#pragma unroll
  for (int d = 16; d; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  float acc[HD / 32];
#pragma unroll
  for (int k = 0; k < HD / 32; ++k) acc[k] = 0.f;
  for (int s = 0; s < a.groups; ++s) {
    const float f = __shfl_sync(0xffffffffu, s < 32 ? w[0] : w[1], s & 31) * inv;
    if (f == 0.f) continue;
#pragma unroll
    for (int k = 0; k < HD / 64; ++k) {
      const float2 x = *reinterpret_cast<const float2*>(a.ws_o + (s * rows + i) * HD + 64 * k + 2 * lane);
      acc[2 * k] += x.x * f;
      acc[2 * k + 1] += x.y * f;
    }
  }
  const long per = (long)a.T * a.heads;
  const long b = i / per;
  const int h = (int)(i % per / a.T), t = (int)(i % a.T);
  bf16* dst = a.out + b * a.o_b + (long)t * a.o_t + (long)h * HD;
#pragma unroll
  for (int k = 0; k < HD / 64; ++k)
    *reinterpret_cast<uint32_t*>(dst + 64 * k + 2 * lane) = pack_bf2(acc[2 * k], acc[2 * k + 1]);
}

}  // namespace p5
