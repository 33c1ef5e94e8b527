// kv8_attention.cuh — attention over the 8-bit K/V cache (fp8.cuh) for few query rows.
//
//   out[b][t][h][:] = sum_j p_j V_j,  p = softmax_j(scale * q . K_j),  j < lens[b] (causal: j < lens[b] - T + t + 1)
//
// The query heads of a K/V head and the T tokens of a sample are folded into rows r = t * G + g.  A CTA owns
// 8 * NT rows of one (sample, K/V head) and one key split; its warps walk 16-key steps, each warp the steps
// w, w + W, ... of the split with a running maximum and sum of its own, merged through shared memory at the end.
//
// Everything is computed transposed, keys and head dims on the 16-row side of mma.m16n8k16 and query rows on
// the 8-column side, because one token of 8 heads has 8 rows, not 16:
//   S^T[16 keys][8 rows] = K Q^T      O^T[16 dims][8 rows] += V^T P^T
// The order of the reduction index and of the output rows of an MMA is free, so each thread takes the operands
// that it can load in 16-byte pieces: lane (g, c) = (lane / 4, lane % 4) holds head dims 64 i + 16 c .. + 15 of
// keys g and g + 8, and head dims 128 i + 16 g .. + 15 of keys 2c, 2c + 1, 2c + 8, 2c + 9.  K and V go from
// global memory to registers, are widened to fp16 there (exact) and never touch shared memory.  P^T goes
// from the accumulator layout to the operand layout by movmatrix.
//
// fp16 operands: a query row is scaled by a power of two so that its largest element is near 2^15 (elements
// down to 2^-29 of it keep all 8 bits of a bf16); P carries the V row's scale relative to a running exponent
// eb (p * 2^(ev - eb)), 11 bits of mantissa, against the 8 that bf16 would keep.  Logits, maxima, sums and O are fp32.
// The running maximum moves only when a logit exceeds it by 2^8, and eb when a scale exceeds it by 2^7, so
// p * 2^(ev - eb) stays within 2^15 and O is rarely rescaled.
#pragma once
#include "fp8.cuh"

namespace p5 {

struct Kv8Args {
  const bf16* q;
  long q_b, q_t;  // elements between samples, tokens; heads are head_dim apart
  const uint8_t *k, *ks, *v, *vs;
  const int* lens;
  const int* slots;  // NULL: sample b is slot b
  bf16* out;
  long o_b, o_t;
  float scale_log2;  // scale * log2(e)
  int n_slots, capacity, T, heads, kv_heads, G, causal;
  int splits;
  float* ws_o;   // [splits][batch][heads * T][head_dim], O in units of the split's 2^m
  float2* ws_ml; // [splits][batch][heads * T] (m, l)
};

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
__device__ __forceinline__ uint4 ldg_stream(const uint8_t* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}
// 2^n for any integer n (0 below 2^-127, 2^127 above)
__device__ __forceinline__ float exp2_int(int n) {
  return n < -127 ? 0.f : __uint_as_float(n == -127 ? 0x400000u : (uint32_t)(min(n, 127) + 127) << 23);
}

template <int HD, int NT, int W>
__global__ void __launch_bounds__(32 * W)
    kv8_attn_rows_kernel(const Kv8Args a) {
  constexpr int KI = HD / 64;                      // 16-byte K pieces of a key per lane
  constexpr int VI = HD >= 128 ? HD / 128 : 1;     // 16-byte V pieces of a key per lane (HD 64: 8 bytes)
  constexpr int VB = HD >= 128 ? 16 : 8;           // bytes of a V piece
  constexpr int MT = HD / 16;                      // 16-dim tiles of O^T
  constexpr int R = 8 * NT;
  __shared__ float sm_o[R][HD + 4];
  __shared__ float sm_m[W][R], sm_l[W][R];
  __shared__ int sm_e[W];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int b = blockIdx.y / a.kv_heads, kvh = blockIdx.y % a.kv_heads;
  const int rows = a.T * a.G, row0 = blockIdx.x * R;
  const int split = blockIdx.z;
  const int slot = a.slots ? a.slots[b] : b;
  const int len = (slot < 0 || slot >= a.n_slots) ? 0 : max(0, min(a.lens[b], a.capacity));
  // keys that any of the CTA's rows sees
  const int t_last = min(row0 + R, rows) - 1;
  const int top = a.causal ? max(0, min(len, len - a.T + t_last / a.G + 1)) : len;
  // the split's steps of 16 keys
  const int steps = (top + 15) >> 4;
  const int per = (steps + a.splits - 1) / a.splits;
  const int s_begin = min(split * per, steps), s_end = min(s_begin + per, steps);

  // ---- Q^T operand: row g of each 8-row tile, scaled to fp16
  uint32_t qf[NT][KI][8];
  float rf[NT][2];  // this thread's accumulator columns: rows 2c, 2c + 1 of each tile
  int lim[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = row0 + 8 * n + g;
    const bool in = r < rows;
    const int t = in ? r / a.G : 0, h = kvh * a.G + (in ? r % a.G : 0);
    const bf16* src = a.q + (long)b * a.q_b + (long)t * a.q_t + (long)h * HD;
    uint32_t raw[KI][8];
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < KI; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint4 u = in ? *reinterpret_cast<const uint4*>(src + 64 * i + 16 * c + 8 * j) : make_uint4(0, 0, 0, 0);
        raw[i][4 * j] = u.x, raw[i][4 * j + 1] = u.y, raw[i][4 * j + 2] = u.z, raw[i][4 * j + 3] = u.w;
      }
#pragma unroll
    for (int i = 0; i < KI; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 f = unpack_bf2(raw[i][j]);
        m = fmaxf(m, fmaxf(fabsf(f.x), fabsf(f.y)));
      }
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
    // e: |q| < 2^(e + 1); rows are scaled by 2^(14 - e) (kept within the float range)
    const int e = min(max((int)(__float_as_uint(m) >> 23) - 127, -112), 127);
    const float up = exp2_int(14 - e);
#pragma unroll
    for (int i = 0; i < KI; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 f = unpack_bf2(raw[i][j]);
        const __half2 hh = __floats2half2_rn(f.x * up, f.y * up);
        qf[n][i][j] = *reinterpret_cast<const uint32_t*>(&hh);
      }
    const float down = a.scale_log2 * exp2_int(e - 14);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      rf[n][j] = __shfl_sync(0xffffffffu, down, (2 * c + j) * 4);
      const int rr = row0 + 8 * n + 2 * c + j;
      lim[n][j] = rr >= rows ? 0 : (a.causal ? min(len, len - a.T + rr / a.G + 1) : len);
    }
  }

  float o[NT][MT][4];
  float m_run[NT][2], l_run[NT][2];
  int eb = -1000;  // exponent of the V scales that O is in units of
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m_run[n][0] = m_run[n][1] = -INFINITY;
    l_run[n][0] = l_run[n][1] = 0.f;
#pragma unroll
    for (int i = 0; i < MT; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
  }

  const long key_pitch = (long)a.kv_heads * HD;
  const long cache0 = ((long)slot * a.capacity * a.kv_heads + kvh);  // in heads
  const uint8_t* kp = a.k + cache0 * HD;
  const uint8_t* vp = a.v + cache0 * HD;
  const uint8_t* ksp = a.ks + cache0;
  const uint8_t* vsp = a.vs + cache0;

  uint4 kr[2][KI], vr[4][VI];
  int kb[2], vb[2];
  auto load_k = [&](int step) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int key = step * 16 + g + 8 * j;
      const bool in = key < top;
      kb[j] = in ? (int)ksp[(long)key * a.kv_heads] : 127;
      vb[j] = in ? (int)vsp[(long)key * a.kv_heads] : 255;  // no exponent of its own; p is 0
#pragma unroll
      for (int i = 0; i < KI; ++i)
        kr[j][i] = in ? ldg_stream(kp + key * key_pitch + 64 * i + 16 * c) : make_uint4(0, 0, 0, 0);
    }
  };
  auto load_v = [&](int step) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int key = step * 16 + 2 * c + (j & 1) + 8 * (j >> 1);
      const bool in = key < top;
#pragma unroll
      for (int i = 0; i < VI; ++i) {
        if (VB == 16) {
          vr[j][i] = in ? ldg_stream(vp + key * key_pitch + 128 * i + 16 * g) : make_uint4(0, 0, 0, 0);
        } else {
          const uint2 u = in ? *reinterpret_cast<const uint2*>(vp + key * key_pitch + 8 * g) : make_uint2(0, 0);
          vr[j][i] = make_uint4(u.x, u.y, 0, 0);
        }
      }
    }
  };

  int step = s_begin + warp;
  if (step < s_end) {
    load_k(step);
    load_v(step);
  }
  for (; step < s_end; step += W) {
    // ---- S^T = K Q^T
    float s[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int i = 0; i < KI; ++i) {
      const uint32_t w0[4] = {kr[0][i].x, kr[0][i].y, kr[0][i].z, kr[0][i].w};
      const uint32_t w1[4] = {kr[1][i].x, kr[1][i].y, kr[1][i].z, kr[1][i].w};
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const uint32_t af[4] = {fp8_to_h2((uint16_t)w0[p]), fp8_to_h2((uint16_t)w1[p]), fp8_to_h2((uint16_t)(w0[p] >> 16)),
                                fp8_to_h2((uint16_t)(w1[p] >> 16))};
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_f16_16816(s[n], af, qf[n][i][2 * p], qf[n][i][2 * p + 1]);
      }
    }
    const int kb0 = kb[0], kb1 = kb[1], vb0 = vb[0], vb1 = vb[1];
    const int key0 = step * 16 + g;
    if (step + W < s_end) load_k(step + W);

    // ---- logits in base 2; a cached NaN row (scale byte 255) makes the rows that see it NaN
    const float kf0 = (kb0 == 255 || vb0 == 255) ? NAN : fp8_scale_value(kb0);
    const float kf1 = (kb1 == 255 || vb1 == 255) ? NAN : fp8_scale_value(kb1);
    bool grow = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float x0 = s[n][j] * rf[n][j] * kf0, x1 = s[n][2 + j] * rf[n][j] * kf1;
        s[n][j] = key0 < lim[n][j] ? x0 : -INFINITY;
        s[n][2 + j] = key0 + 8 < lim[n][j] ? x1 : -INFINITY;
        grow |= fmaxf(s[n][j], s[n][2 + j]) > m_run[n][j] + 8.f;
      }
    const int ev0 = vb0 == 255 ? -1000 : vb0 - 127, ev1 = vb1 == 255 ? -1000 : vb1 - 127;
    grow |= max(ev0, ev1) > eb + 7;
    if (__any_sync(0xffffffffu, grow)) {
      int em = max(ev0, ev1);
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) em = max(em, __shfl_xor_sync(0xffffffffu, em, d));
      em = max(em, eb);
      const float ealpha = exp2_int(eb - em);  // eb = -1000 at first: 0, O is 0 anyway
      eb = em;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float m = fmaxf(s[n][j], s[n][2 + j]);
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
          m = fmaxf(m, m_run[n][j]);
          const float alpha = m_run[n][j] == -INFINITY ? 0.f : ex2_approx(m_run[n][j] - m);
          m_run[n][j] = m;
          l_run[n][j] *= alpha;
          const float al = alpha * ealpha;
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            o[n][i][j] *= al;
            o[n][i][2 + j] *= al;
          }
        }
    }
    // ---- P^T, each key's V scale folded in
    const float vf0 = exp2_int(ev0 - eb), vf1 = exp2_int(ev1 - eb);
    uint32_t pf[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float p[4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float mm = m_run[n][j] == -INFINITY ? 0.f : m_run[n][j];
        p[j] = ex2_approx(s[n][j] - mm);
        p[2 + j] = ex2_approx(s[n][2 + j] - mm);
        l_run[n][j] += p[j] + p[2 + j];
      }
      const __half2 h0 = __floats2half2_rn(p[0] * vf0, p[1] * vf0), h1 = __floats2half2_rn(p[2] * vf1, p[3] * vf1);
      pf[n][0] = movmatrix_b16(*reinterpret_cast<const uint32_t*>(&h0));
      pf[n][1] = movmatrix_b16(*reinterpret_cast<const uint32_t*>(&h1));
    }
    // ---- O^T += V^T P^T: tile (i, j) holds dims 16 g + 2 j and + 1 of the 128-dim part i
#pragma unroll
    for (int i = 0; i < VI; ++i) {
      const uint32_t w[4][4] = {{vr[0][i].x, vr[0][i].y, vr[0][i].z, vr[0][i].w},
                                {vr[1][i].x, vr[1][i].y, vr[1][i].z, vr[1][i].w},
                                {vr[2][i].x, vr[2][i].y, vr[2][i].z, vr[2][i].w},
                                {vr[3][i].x, vr[3][i].y, vr[3][i].z, vr[3][i].w}};
#pragma unroll
      for (int q = 0; q < VB / 4; ++q) {
#pragma unroll
        for (int hlf = 0; hlf < 2; ++hlf) {
          // bytes (2 hlf, 2 hlf + 1) of the word of two keys, interleaved by key
          const uint32_t lo = __byte_perm(w[0][q], w[1][q], hlf ? 0x7362 : 0x5140);
          const uint32_t hi = __byte_perm(w[2][q], w[3][q], hlf ? 0x7362 : 0x5140);
          const uint32_t af[4] = {fp8_to_h2((uint16_t)lo), fp8_to_h2((uint16_t)(lo >> 16)), fp8_to_h2((uint16_t)hi),
                                  fp8_to_h2((uint16_t)(hi >> 16))};
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16_16816(o[n][i * (VB / 2) + 2 * q + hlf], af, pf[n][0], pf[n][1]);
        }
      }
    }
    if (step + W < s_end) load_v(step + W);
  }

  // ---- merge the warps: row maxima and exponents first, then O in warp order (reruns give the same bits)
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l_run[n][j] += __shfl_xor_sync(0xffffffffu, l_run[n][j], d);
  if (g == 0) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        sm_m[warp][8 * n + 2 * c + j] = m_run[n][j];
        sm_l[warp][8 * n + 2 * c + j] = l_run[n][j];
      }
  }
  if (lane == 0) sm_e[warp] = eb;
  __syncthreads();
  int e_all = -1000;
#pragma unroll
  for (int w = 0; w < W; ++w) e_all = max(e_all, sm_e[w]);
  float fac[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float m = -INFINITY;
#pragma unroll
      for (int w = 0; w < W; ++w) m = fmaxf(m, sm_m[w][8 * n + 2 * c + j]);
      fac[n][j] = m_run[n][j] == -INFINITY ? 0.f : ex2_approx(m_run[n][j] - m) * exp2_int(eb - e_all);
    }
#pragma unroll 1
  for (int w = 0; w < W; ++w) {
    if (warp == w) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float* dst = sm_o[8 * n + 2 * c + j];
#pragma unroll
          for (int i = 0; i < VI; ++i)
#pragma unroll
            for (int q = 0; q < VB; ++q) {
              const float x = o[n][i * (VB / 2) + q / 2][(q & 1) * 2 + j] * fac[n][j];
              float* d = dst + 128 * i + VB * g + q;
              *d = w == 0 ? x : *d + x;
            }
        }
    }
    __syncthreads();
  }
  const float unit = exp2_int(e_all);
  const int out_rows = a.T * a.heads;
  for (int r = warp; r < R; r += W) {
    const int row = row0 + r;
    if (row >= rows) continue;
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) m = fmaxf(m, sm_m[w][r]);
#pragma unroll
    for (int w = 0; w < W; ++w) l += sm_m[w][r] == -INFINITY ? sm_l[w][r] : sm_l[w][r] * ex2_approx(sm_m[w][r] - m);  // 0 or NaN
    const int t = row / a.G, h = kvh * a.G + row % a.G;
    if (a.splits == 1) {
      // l is 0 for a row without keys (its output is 0), NaN for one that sees a NaN
      const float inv = l == 0.f ? 0.f : unit / l;
      bf16* dst = a.out + (long)b * a.o_b + (long)t * a.o_t + (long)h * HD;
      for (int d = 2 * lane; d < HD; d += 64)
        *reinterpret_cast<uint32_t*>(dst + d) = pack_bf2(sm_o[r][d] * inv, sm_o[r][d + 1] * inv);
    } else {
      const long i = ((long)split * (gridDim.y / a.kv_heads) + b) * out_rows + (long)h * a.T + t;
      for (int d = lane; d < HD; d += 32) a.ws_o[i * HD + d] = sm_o[r][d] * unit;
      if (lane == 0) a.ws_ml[i] = make_float2(m, l);
    }
  }
}

// Joins the key splits of a row: out = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s, splits in order.
// One warp a row.
template <int HD>
__global__ void kv8_attn_combine_kernel(const Kv8Args a, int batch) {
  const int lane = threadIdx.x & 31;
  const long rows = (long)batch * a.T * a.heads;
  const long i = (long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (i >= rows) return;
  float m = -INFINITY;
  for (int s = 0; s < a.splits; ++s) m = fmaxf(m, a.ws_ml[s * rows + i].x);
  float l = 0.f, acc[HD / 32];
#pragma unroll
  for (int k = 0; k < HD / 32; ++k) acc[k] = 0.f;
  for (int s = 0; s < a.splits; ++s) {
    const float2 ml = a.ws_ml[s * rows + i];
    if (ml.x == -INFINITY && ml.y == 0.f) continue;
    const float f = ex2_approx(ml.x - m);
    l += ml.y * f;
#pragma unroll
    for (int k = 0; k < HD / 64; ++k) {
      const float2 x = *reinterpret_cast<const float2*>(a.ws_o + (s * rows + i) * HD + 64 * k + 2 * lane);
      acc[2 * k] += x.x * f;
      acc[2 * k + 1] += x.y * f;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const long per = (long)a.T * a.heads;
  const long b = i / per;
  const int h = (int)(i % per / a.T), t = (int)(i % a.T);
  bf16* dst = a.out + b * a.o_b + (long)t * a.o_t + (long)h * HD;
#pragma unroll
  for (int k = 0; k < HD / 64; ++k)
    *reinterpret_cast<uint32_t*>(dst + 64 * k + 2 * lane) = pack_bf2(acc[2 * k] * inv, acc[2 * k + 1] * inv);
}

}  // namespace p5
