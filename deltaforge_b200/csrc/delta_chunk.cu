// The gated delta rule over several new tokens of a sequence (a prompt, or a tree of drafted tokens), sm_100a.
//
// Per value head (key head h / (Hv / Hk)), token by token (src/deltaforge/reference.py:450-458):
//   S <- e^g_t S;  r = S^T k_t;  d = beta_t (v_t - r);  S <- S + k_t d^T;  o_t = S^T q_t
// Over a chunk of C = 64 tokens, with G_i = g_1 + .. + g_i, the same thing is
//   A_ij = beta_i e^(G_i - G_j) k_i.k_j (j < i),  T = (I + A)^-1 diag(beta),  P_ij = e^(G_i - G_j) q_i.k_j (j <= i)
//   R = V - diag(e^G) K S;  V' = T R;  O = diag(e^G) Q S + P V';  S <- e^G_C S + sum_j e^(G_C - G_j) k_j v'_j^T
// T, P and the scalars do not depend on S: delta_prep_kernel makes them for all chunks at once. delta_scan_kernel then walks
// through the chunks of a head; its work is matrix products with S.
// For a tree, "j <= i" reads "j is i or an ancestor of i" and G_i is summed along the path of i; there is one chunk and no
// new state (the accepted path is run through the prompt form afterwards).
//
// Precision. S is fp32 from end to end and so is the new state's bar: an operand rounded to 8 bits (bf16) would cost
// 2e-3 per product. All matrix operands are therefore fp16 (11 bits), scaled by powers of two to the top of fp16's range
// (per token for k and q, which are bf16 and stay exact; per matrix for T, P; per warp and chunk for S, R, V'), and S, T, R and
// V' are split in two, hi + lo = 22 bits, wherever the product leads into the state: hi hi + hi lo + lo hi, fp32
// accumulation. Products that lead into the bf16 output alone take hi (2^-12). The state's update is accumulated apart and
// added in fp32 (the tensor core truncates what it adds to a large accumulator). Log decays are summed in fp64 and kept as
// two floats, so that differences of large sums stay exact.
//
// Scan: one warp owns 16 value columns and all key rows of its head's state, in registers, as the accumulators of
// S^T (16 x dk). Their layout is that of the A operand of the next product, so R^T, V'^T, O^T and S^T follow from one
// another inside the warp without an exchange or a barrier; k, q, T, P of the chunk come from shared memory, which two loader
// warps fill by cp.async one to two chunks ahead. No wait spins.
#include <cuda_fp16.h>

#include "common.cuh"
#include "kernels.h"

namespace dfb {

namespace {

constexpr int C = 64;                // tokens per chunk
constexpr int SQ = C * C * 2;        // bytes of one 64 x 64 fp16 image
constexpr int SCAL = 4 * C * 4;      // scalars of a (chunk, value head): three per token, then a few
constexpr int HEAD_BYTES = 3 * SQ + SCAL;
constexpr float MIN_LOG_DECAY = -150.f;  // e^-150 is 0 in fp32: keeps sums finite when a log decay is -inf

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void stsm4_t(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t h2(float a, float b) {
  __half2 v = __floats2half2_rn(a, b);
  return *(uint32_t*)&v;
}
// (a, b) as fp16 pair hi and the remainder as fp16 pair lo: hi + lo carries 22 bits
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2 f = __half22float2(h);
  hi = *(const uint32_t*)&h;
  lo = h2(a - f.x, b - f.y);
}
// Exponent that takes a largest magnitude m to [2^12, 2^13); 0 for m = 0. Clamped so that 2^e and 2^-e are normal numbers.
__device__ __forceinline__ int scale_exp(float m) {
  if (m == 0.f) return 0;
  const int e = (int)((__float_as_uint(m) >> 23) & 255) - 127 - 12;
  return e < -110 ? -110 : e > 110 ? 110 : e;
}
// Largest of the lanes' non-negative values, whose bit patterns order like the values
__device__ __forceinline__ float warp_max_abs(float m) { return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m))); }
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

// Images are rows of W fp16 with 16-byte chunks permuted within 128 bytes, so that 8x8 matrix loads are free of conflicts.
template <int W> __device__ __forceinline__ uint32_t img_off(int row, int chunk) {
  return (uint32_t)(row * W * 2 + ((chunk ^ (row & 7)) << 4));
}

constexpr int PREP_THREADS = 256;
constexpr int TS = 68;  // row stride (floats) of the 64 x 64 fp32 matrices: 16-byte rows, neighbouring rows in other banks

// One CTA per (chunk, key head, sequence). Warps 0-3 form K K^T, warps 4-7 Q K^T, 16 rows each, once for all value heads of
// the key head; then per value head the decays, A, T = (I + A)^-1 diag(beta) by blocks (16 x 16 by substitution, then two
// doublings: the lower left block of a pair is -T22 A21 T11) and the images.
template <int DKP, bool TREE>
__global__ void __launch_bounds__(PREP_THREADS) delta_prep_kernel(const DeltaChunkParams p) {
  extern __shared__ __align__(128) unsigned char smem[];
  unsigned char* kt = smem;                                  // bf16 [64][DKP]
  unsigned char* qt = smem + C * DKP * 2;
  float* A = (float*)(smem + 2 * C * DKP * 2);               // [64][TS]
  float* T = A + C * TS;
  float* X = T + C * TS;                                     // [32][TS / 2 ..]: product of two blocks
  __shared__ float rk[C], rq[C], ghi[C], glo[C], bet[C], sk[C], sq[C];
  __shared__ float wmax[8];
  __shared__ unsigned long long anc[C];
  __shared__ int up[C];
  __shared__ double gsum[C];

  const int cl = blockIdx.x, hk = blockIdx.y, b = blockIdx.z;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31, g = lane >> 2, c = lane & 3;
  const int tok0 = (p.chunk0 + cl) * C;
  const int len = p.lengths ? min(max(p.lengths[b], 0), p.tokens) : p.tokens;
  const int live = min(len - tok0, C);  // tokens of this chunk; the scan does not read chunks without any
  if (live <= 0) return;

  if (TREE) {  // bit j of anc[i]: j is i or an ancestor of i; 0 where row i holds no node
    if (t < C) {
      const int pa = t < live ? p.parents[(long)b * p.parents_stride + t] : -2;
      const bool node = pa >= -1 && pa < t;
      anc[t] = node ? 1ull << t : 0ull;
      up[t] = node ? pa : -1;
    }
    __syncthreads();
    for (int step = 1; step < C; step *= 2) {
      unsigned long long bits = 0;
      int u = -1;
      if (t < C) {
        bits = anc[t], u = up[t];
        if (u >= 0) bits |= anc[u], u = up[u];
      }
      __syncthreads();
      if (t < C) anc[t] = bits, up[t] = u;
      __syncthreads();
    }
  }

  // ---- the chunk's keys and queries: bf16 tiles for the products, norms, fp16 images for the scan ----
  const long sbase = ((long)b * p.seg_chunks + cl) * (p.hk * (2L * C * DKP * 2) + p.hv * (long)HEAD_BYTES);
  unsigned char* kimg = p.scratch + sbase + (long)hk * (2 * C * DKP * 2);
  {
    // four threads per row: key rows 0 .. 63 by threads 0 .. 255, then query rows
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const int row = t >> 2, part = t & 3;
      const bf16* src = which ? p.q + b * p.q_stride[0] + (long)(tok0 + row) * p.q_stride[1] + hk * p.q_stride[2]
                              : p.k + b * p.k_stride[0] + (long)(tok0 + row) * p.k_stride[1] + hk * p.k_stride[2];
      const bool ok = row < live && (!TREE || anc[row] != 0);
      constexpr int N = DKP / 8 / 4;  // 16-byte chunks per thread
      uint4 raw[N];
      float ss = 0.f, mx = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int ch = part + 4 * i;
        raw[i] = ok && ch * 8 < p.dk ? *(const uint4*)(src + ch * 8) : make_uint4(0, 0, 0, 0);
        const bf16* e = (const bf16*)&raw[i];
#pragma unroll
        for (int y = 0; y < 8; ++y) {
          const float x = bf2f(e[y]);
          ss = fmaf(x, x, ss);
          mx = fmaxf(mx, fabsf(x));
        }
      }
      ss += __shfl_xor_sync(0xffffffffu, ss, 1);
      ss += __shfl_xor_sync(0xffffffffu, ss, 2);
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const int e2 = scale_exp(mx);
      const float down = pow2(-e2);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int ch = part + 4 * i;
        const bf16* e = (const bf16*)&raw[i];
        *(uint4*)((which ? qt : kt) + img_off<DKP>(row, ch)) = raw[i];
        uint4 im;
        im.x = h2(bf2f(e[0]) * down, bf2f(e[1]) * down), im.y = h2(bf2f(e[2]) * down, bf2f(e[3]) * down);
        im.z = h2(bf2f(e[4]) * down, bf2f(e[5]) * down), im.w = h2(bf2f(e[6]) * down, bf2f(e[7]) * down);
        *(uint4*)(kimg + which * (C * DKP * 2) + img_off<DKP>(row, ch)) = im;
      }
      if (part == 0) {
        float r = p.l2norm ? rsqrt_2step(__fadd_rn(ss, 1e-6f)) : 1.f;
        if (which && p.l2norm) r = __fdiv_rn(r, sqrtf((float)p.dk));
        (which ? rq : rk)[row] = r;
        (which ? sq : sk)[row] = r * pow2(e2);
      }
    }
  }
  __syncthreads();

  // ---- rows 16 (warp % 4) .. + 15 of K K^T (warps 0-3) or Q K^T (warps 4-7) ----
  const int r0 = (warp & 3) * 16;
  float dot[8][4];
#pragma unroll
  for (int nt = 0; nt < 8; ++nt) dot[nt][0] = dot[nt][1] = dot[nt][2] = dot[nt][3] = 0.f;
  {
    const uint32_t as = smem_u32(warp < 4 ? kt : qt), bs = smem_u32(kt);
#pragma unroll
    for (int ks = 0; ks < DKP / 16; ++ks) {
      uint32_t a[4];
      ldsm4(as + img_off<DKP>(r0 + (lane & 15), 2 * ks + (lane >> 4)), a);
#pragma unroll
      for (int n2 = 0; n2 < 4; ++n2) {
        if (16 * n2 > r0) continue;  // above the diagonal
        uint32_t kb[4];
        ldsm4(bs + img_off<DKP>(16 * n2 + (lane & 7) + 8 * (lane >> 4), 2 * ks + ((lane >> 3) & 1)), kb);
        mma_bf16(dot[2 * n2], a, kb[0], kb[1]);
        mma_bf16(dot[2 * n2 + 1], a, kb[2], kb[3]);
      }
    }
  }

  const int group = p.hv / p.hk;
  for (int r = 0; r < group; ++r) {
    const int hv = hk * group + r;
    unsigned char* himg = p.scratch + sbase + p.hk * (2L * C * DKP * 2) + (long)hv * HEAD_BYTES;
    __syncthreads();  // the previous head's matrices have been read
    if (t < C) {
      const bool ok = t < live && (!TREE || anc[t] != 0);
      float gv = 0.f, bv = 0.f;
      if (ok) {
        gv = p.g[((long)b * p.tokens + tok0 + t) * p.hv + hv];
        bv = p.beta[((long)b * p.tokens + tok0 + t) * p.hv + hv];
        gv = gv < MIN_LOG_DECAY ? MIN_LOG_DECAY : gv;
      }
      bet[t] = bv;
      gsum[t] = gv;
    }
    __syncthreads();
    if (!TREE) {
      if (warp == 0) {  // prefix sums of 64 values, two per lane
        const double a0 = gsum[2 * lane], a1 = gsum[2 * lane + 1];
        double s = a0 + a1;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
          const double y = __shfl_up_sync(0xffffffffu, s, o);
          if (lane >= o) s += y;
        }
        gsum[2 * lane] = s - a1;
        gsum[2 * lane + 1] = s;
      }
      __syncthreads();
      if (t < C) {
        const double s = gsum[t];
        ghi[t] = (float)s;
        glo[t] = (float)(s - (double)(float)s);
      }
    } else if (t < C) {  // along the path
      double s = 0.;
      unsigned long long bits = anc[t];
      while (bits) {
        s += gsum[__ffsll(bits) - 1];
        bits &= bits - 1;
      }
      ghi[t] = (float)s;
      glo[t] = (float)(s - (double)(float)s);
    }
    __syncthreads();
    // decayed entries of this warp's rows; A to shared memory, P kept for its scale
    float pm = 0.f;
    float pr[8][4];
#pragma unroll
    for (int nt = 0; nt < 8; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = r0 + g + 8 * (e >> 1), j = nt * 8 + 2 * c + (e & 1);
        const bool seen = TREE ? (anc[i] >> j) & 1 : j <= i;
        float x = 0.f;
        if (seen && i < live) {
          const float d = expf((ghi[i] - ghi[j]) + (glo[i] - glo[j]));
          x = dot[nt][e] * rk[j] * d * (warp < 4 ? rk[i] * bet[i] : rq[i]);
        }
        if (warp < 4)
          A[i * TS + j] = i == j ? 0.f : x;
        else
          pr[nt][e] = x, pm = fmaxf(pm, fabsf(x));
      }
    pm = warp_max(pm);
    if (lane == 0) wmax[warp] = pm;
    __syncthreads();
    const int ep = scale_exp(fmaxf(fmaxf(wmax[4], wmax[5]), fmaxf(wmax[6], wmax[7])));
    if (warp >= 4) {
      const float down = pow2(-ep);
#pragma unroll
      for (int nt = 0; nt < 8; ++nt) {
        *(uint32_t*)(himg + 2 * SQ + img_off<C>(r0 + g, nt) + 4 * c) = h2(pr[nt][0] * down, pr[nt][1] * down);
        *(uint32_t*)(himg + 2 * SQ + img_off<C>(r0 + g + 8, nt) + 4 * c) = h2(pr[nt][2] * down, pr[nt][3] * down);
      }
    }
    // (I + A)^-1: the four diagonal blocks, a column per lane
    if (warp < 4) {
      const int j = lane & 15, base = warp * 16;
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float s = 0.f;
#pragma unroll
        for (int m = 0; m < i; ++m) s = fmaf(A[(base + i) * TS + base + m], x[m], s);
        x[i] = (i == j ? 1.f : 0.f) - s;
      }
      if (lane < 16) {
#pragma unroll
        for (int i = 0; i < 16; ++i) T[(base + i) * TS + base + j] = x[i];
      }
    } else {  // zeros above the diagonal blocks
      for (int i = t - 128; i < C * C; i += 128)
        if ((i & 63) / 16 > (i >> 6) / 16) T[(i >> 6) * TS + (i & 63)] = 0.f;
    }
    __syncthreads();
    // pairs of 16: X = A21 T11 (two products of 16 x 16), T21 = -T22 X
    {
      const int pair = t >> 7, i = (t >> 3) & 15, j = (t & 7) * 2, o = 32 * pair;
      float x0 = 0.f, x1 = 0.f;
#pragma unroll
      for (int m = 0; m < 16; ++m) {
        const float a = A[(o + 16 + i) * TS + o + m];
        const float2 y = *(const float2*)&T[(o + m) * TS + o + j];
        x0 = fmaf(a, y.x, x0), x1 = fmaf(a, y.y, x1);
      }
      *(float2*)&X[(pair * 16 + i) * 36 + j] = make_float2(x0, x1);
      __syncthreads();
      x0 = x1 = 0.f;
#pragma unroll
      for (int m = 0; m < 16; ++m) {
        const float a = T[(o + 16 + i) * TS + o + 16 + m];
        const float2 y = *(const float2*)&X[(pair * 16 + m) * 36 + j];
        x0 = fmaf(a, y.x, x0), x1 = fmaf(a, y.y, x1);
      }
      *(float2*)&T[(o + 16 + i) * TS + o + j] = make_float2(-x0, -x1);
    }
    __syncthreads();
    // the pair of 32
    {
      const int i = t >> 3, j = (t & 7) * 4;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
      for (int m = 0; m < 32; ++m) {
        const float a = A[(32 + i) * TS + m];
        const float4 y = *(const float4*)&T[m * TS + j];
        x.x = fmaf(a, y.x, x.x), x.y = fmaf(a, y.y, x.y), x.z = fmaf(a, y.z, x.z), x.w = fmaf(a, y.w, x.w);
      }
      *(float4*)&X[i * 36 + j] = x;
      __syncthreads();
      x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
      for (int m = 0; m < 32; ++m) {
        const float a = T[(32 + i) * TS + 32 + m];
        const float4 y = *(const float4*)&X[m * 36 + j];
        x.x = fmaf(a, y.x, x.x), x.y = fmaf(a, y.y, x.y), x.z = fmaf(a, y.z, x.z), x.w = fmaf(a, y.w, x.w);
      }
      *(float4*)&T[(32 + i) * TS + j] = make_float4(-x.x, -x.y, -x.z, -x.w);
    }
    __syncthreads();
    // T diag(beta) as hi and lo images
    float tv[2][8], tm = 0.f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int i = (t + k * PREP_THREADS) >> 3, j0 = (t & 7) * 8;
#pragma unroll
      for (int y = 0; y < 8; ++y) {
        tv[k][y] = T[i * TS + j0 + y] * bet[j0 + y];
        tm = fmaxf(tm, fabsf(tv[k][y]));
      }
    }
    tm = warp_max(tm);
    if (lane == 0) wmax[warp] = tm;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) tm = fmaxf(tm, wmax[w]);
    const int et = scale_exp(tm);
    const float down = pow2(-et);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int i = (t + k * PREP_THREADS) >> 3;
      uint4 hi, lo;
      split2(tv[k][0] * down, tv[k][1] * down, hi.x, lo.x);
      split2(tv[k][2] * down, tv[k][3] * down, hi.y, lo.y);
      split2(tv[k][4] * down, tv[k][5] * down, hi.z, lo.z);
      split2(tv[k][6] * down, tv[k][7] * down, hi.w, lo.w);
      *(uint4*)(himg + img_off<C>(i, t & 7)) = hi;
      *(uint4*)(himg + SQ + img_off<C>(i, t & 7)) = lo;
    }
    float* sc = (float*)(himg + 3 * SQ);
    if (t < C) {
      const float eg = expf(ghi[t] + glo[t]);
      sc[t] = eg * sk[t];                                                                  // on K S
      sc[C + t] = expf((ghi[C - 1] - ghi[t]) + (glo[C - 1] - glo[t])) * sk[t];             // on V' into the state
      sc[2 * C + t] = eg * sq[t];                                                          // on Q S
      if (t == C - 1) sc[3 * C] = eg;                                                      // decay of the state
      if (t == 0) sc[3 * C + 1] = pow2(et), sc[3 * C + 2] = pow2(ep);
    }
  }
}

// ---- the scan -------------------------------------------------------------------------------------------------------

template <int DKP, int NW> struct Scan {
  static constexpr int THREADS = (NW + 2) * 32;
  static constexpr int VROW = NW * 32;  // bytes of a token's values in a stage
  static constexpr int Q_OFF = C * DKP * 2, H_OFF = 2 * C * DKP * 2, V_OFF = H_OFF + HEAD_BYTES;
  static constexpr int STAGE = V_OFF + C * VROW;
  static constexpr int OUT = NW * C * 32;  // per warp: 64 tokens x 16 columns
  static constexpr int FIT = (224 * 1024 - OUT) / STAGE;
  static constexpr int STAGES = FIT > 3 ? 3 : FIT;
  static constexpr int SMEM = STAGES * STAGE + OUT;
};

template <int VROW> __device__ __forceinline__ uint32_t v_off(int row, int chunk) {
  const int x = VROW >= 128 ? (chunk ^ (row & 7)) : (chunk ^ ((row >> 1) & (VROW / 16 - 1)));
  return (uint32_t)(row * VROW + (x << 4));
}

template <int DKP, int NW, int NB, bool TREE>
__global__ void __launch_bounds__((NW + 2) * 32, 1) delta_scan_kernel(const DeltaChunkParams p) {
  using S_ = Scan<DKP, NW>;
  constexpr int NT = DKP / 8;
  extern __shared__ __align__(128) unsigned char smem[];
  const int vb = blockIdx.x, hv = blockIdx.y, b = blockIdx.z, hk = hv / (p.hv / p.hk);
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31, g = lane >> 2, c = lane & 3;
  const int len = p.lengths ? min(max(p.lengths[b], 0), p.tokens) : p.tokens;
  const int nlive = min(max((len + C - 1) / C - p.chunk0, 0), p.chunks);  // chunks of this segment with tokens
  const int col_cta = vb * NW * 16;

  if (warp >= NW) {  // ---- loader warps ----
    const int lt = t - NW * 32;
    const long per = p.hk * (2L * C * DKP * 2) + p.hv * (long)HEAD_BYTES;
    auto load = [&](int n) {
      if (n < nlive) {
        const unsigned char* base = p.scratch + ((long)b * p.seg_chunks + n) * per;
        const unsigned char* kq = base + (long)hk * (2 * C * DKP * 2);
        const unsigned char* hd = base + p.hk * (2L * C * DKP * 2) + (long)hv * HEAD_BYTES;
        const uint32_t st = smem_u32(smem + (n % S_::STAGES) * S_::STAGE);
#pragma unroll 8
        for (int i = lt; i < 2 * C * DKP * 2 / 16; i += 64) cp_async16(st + i * 16, kq + i * 16, 16);
#pragma unroll 5
        for (int i = lt; i < HEAD_BYTES / 16; i += 64) cp_async16(st + S_::H_OFF + i * 16, hd + i * 16, 16);
        const int tok0 = (p.chunk0 + n) * C;
#pragma unroll 4
        for (int i = lt; i < C * NW * 2; i += 64) {
          const int row = i / (NW * 2), ch = i % (NW * 2), col = col_cta + ch * 8, tok = tok0 + row;
          bool ok = tok < len && col < p.dv;
          if (TREE && ok) {  // a row without a node may hold anything
            const int pa = p.parents[(long)b * p.parents_stride + tok];
            ok = pa >= -1 && pa < tok;
          }
          cp_async16(st + S_::V_OFF + v_off<S_::VROW>(row, ch),
                     p.v + b * p.v_stride[0] + (ok ? tok : 0) * p.v_stride[1] + hv * p.v_stride[2] + (ok ? col : 0), ok ? 16 : 0);
        }
      }
      cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < S_::STAGES - 1; ++i) load(i);
    for (int n = 0; n < nlive; ++n) {
      cp_async_wait<S_::STAGES - 2>();
      __syncthreads();  // chunk n is there, chunk n - 1 has been used up
      load(n + S_::STAGES - 1);
    }
    cp_async_wait<0>();
    return;
  }

  // ---- compute warps: 16 value columns each ----
  const int col0 = col_cta + warp * 16;
  const bool cok0 = col0 + g < p.dv, cok1 = col0 + g + 8 < p.dv;
  const long sb = ((long)b * p.hv + hv) * p.dk * p.dv;
  const float* Sin = p.first ? p.state + sb : p.state_out + sb;
  float S[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = 8 * n + 2 * c + (e & 1);
      const bool ok = d < p.dk && (e < 2 ? cok0 : cok1);
      S[n][e] = ok ? Sin[(long)d * p.dv + col0 + g + 8 * (e >> 1)] : 0.f;
    }
  unsigned char* obuf = smem + S_::STAGES * S_::STAGE + warp * (C * 32);
  bf16* out = p.out + ((long)b * p.tokens * p.hv + hv) * p.dv + col0;
  const long orow = (long)p.hv * p.dv;

  for (int n = 0; n < nlive; ++n) {
    __syncthreads();
    const unsigned char* st = smem + (n % S_::STAGES) * S_::STAGE;
    const uint32_t ks_s = smem_u32(st), qs_s = ks_s + S_::Q_OFF, ti_s = ks_s + S_::H_OFF, vs_s = ks_s + S_::V_OFF;
    const float* sc = (const float*)(st + S_::H_OFF + 3 * SQ);
    const int tok0 = (p.chunk0 + n) * C;

    // 1. S^T K^T (hi and lo) and S^T Q^T (hi)
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < NT; ++i) m = fmaxf(m, fmaxf(fmaxf(fabsf(S[i][0]), fabsf(S[i][1])), fmaxf(fabsf(S[i][2]), fabsf(S[i][3]))));
    const int es = scale_exp(warp_max_abs(m));
    const float sdown = pow2(-es), sup = pow2(es);
    float x[2 * NB][4], oq[2 * NB][4];
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[i][e] = oq[i][e] = 0.f;
#pragma unroll
    for (int ks = 0; ks < NT / 2; ++ks) {
      uint32_t hi[4], lo[4];
      split2(S[2 * ks][0] * sdown, S[2 * ks][1] * sdown, hi[0], lo[0]);
      split2(S[2 * ks][2] * sdown, S[2 * ks][3] * sdown, hi[1], lo[1]);
      split2(S[2 * ks + 1][0] * sdown, S[2 * ks + 1][1] * sdown, hi[2], lo[2]);
      split2(S[2 * ks + 1][2] * sdown, S[2 * ks + 1][3] * sdown, hi[3], lo[3]);
#pragma unroll
      for (int n2 = 0; n2 < NB; ++n2) {
        uint32_t kb[4], qb[4];
        const uint32_t off = img_off<DKP>(16 * n2 + (lane & 7) + 8 * (lane >> 4), 2 * ks + ((lane >> 3) & 1));
        ldsm4(ks_s + off, kb);
        ldsm4(qs_s + off, qb);
        mma_f16(x[2 * n2], hi, kb[0], kb[1]);
        mma_f16(x[2 * n2 + 1], hi, kb[2], kb[3]);
        mma_f16(oq[2 * n2], hi, qb[0], qb[1]);
        mma_f16(oq[2 * n2 + 1], hi, qb[2], qb[3]);
        mma_f16(x[2 * n2], lo, kb[0], kb[1]);
        mma_f16(x[2 * n2 + 1], lo, kb[2], kb[3]);
      }
    }
    // 2. R = V - diag(e^G) K S, then its halves
    m = 0.f;
#pragma unroll
    for (int n2 = 0; n2 < NB; ++n2) {
      uint32_t vr[4];
      ldsm4_t(vs_s + v_off<S_::VROW>(16 * n2 + (lane & 15), warp * 2 + (lane >> 4)), vr);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int nt = 2 * n2 + h;
        const float2 w = *(const float2*)&sc[8 * nt + 2 * c];
        const float2 v0 = __bfloat1622float2(*(const __nv_bfloat162*)&vr[h]), v1 = __bfloat1622float2(*(const __nv_bfloat162*)&vr[2 + h]);
        x[nt][0] = v0.x - x[nt][0] * (w.x * sup);
        x[nt][1] = v0.y - x[nt][1] * (w.y * sup);
        x[nt][2] = v1.x - x[nt][2] * (w.x * sup);
        x[nt][3] = v1.y - x[nt][3] * (w.y * sup);
        m = fmaxf(m, fmaxf(fmaxf(fabsf(x[nt][0]), fabsf(x[nt][1])), fmaxf(fabsf(x[nt][2]), fabsf(x[nt][3]))));
      }
    }
    const int er = scale_exp(warp_max_abs(m));
    const float rdown = pow2(-er);
    uint32_t rh[NB][4], rl[NB][4];
#pragma unroll
    for (int k = 0; k < NB; ++k) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        split2(x[2 * k + h][0] * rdown, x[2 * k + h][1] * rdown, rh[k][2 * h], rl[k][2 * h]);
        split2(x[2 * k + h][2] * rdown, x[2 * k + h][3] * rdown, rh[k][2 * h + 1], rl[k][2 * h + 1]);
      }
    }
    // 3. V'^T = R^T T^T; block (i, j) of T is zero for j > i
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0.f;
#pragma unroll
    for (int k = 0; k < NB; ++k) {
#pragma unroll
      for (int n2 = k; n2 < NB; ++n2) {
        uint32_t th[4], tl[4];
        const uint32_t off = img_off<C>(16 * n2 + (lane & 7) + 8 * (lane >> 4), 2 * k + ((lane >> 3) & 1));
        ldsm4(ti_s + off, th);
        ldsm4(ti_s + SQ + off, tl);
        mma_f16(x[2 * n2], rh[k], th[0], th[1]);
        mma_f16(x[2 * n2 + 1], rh[k], th[2], th[3]);
        mma_f16(x[2 * n2], rl[k], th[0], th[1]);
        mma_f16(x[2 * n2 + 1], rl[k], th[2], th[3]);
        mma_f16(x[2 * n2], rh[k], tl[0], tl[1]);
        mma_f16(x[2 * n2 + 1], rh[k], tl[2], tl[3]);
      }
    }
    m = 0.f;
    {
      const float up = pow2(er) * sc[3 * C + 1];
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[i][e] *= up, m = fmaxf(m, fabsf(x[i][e]));
    }
    // 4. O^T = (S^T Q^T) diag(e^G) + V'^T P^T
    const int ev = scale_exp(warp_max_abs(m));
    {
      const float vdown = pow2(-ev);
      float o[2 * NB][4];
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        const uint32_t a[4] = {h2(x[2 * k][0] * vdown, x[2 * k][1] * vdown), h2(x[2 * k][2] * vdown, x[2 * k][3] * vdown),
                               h2(x[2 * k + 1][0] * vdown, x[2 * k + 1][1] * vdown), h2(x[2 * k + 1][2] * vdown, x[2 * k + 1][3] * vdown)};
#pragma unroll
        for (int n2 = k; n2 < NB; ++n2) {
          uint32_t pb[4];
          ldsm4(ti_s + 2 * SQ + img_off<C>(16 * n2 + (lane & 7) + 8 * (lane >> 4), 2 * k + ((lane >> 3) & 1)), pb);
          mma_f16(o[2 * n2], a, pb[0], pb[1]);
          mma_f16(o[2 * n2 + 1], a, pb[2], pb[3]);
        }
      }
      const float up = pow2(ev) * sc[3 * C + 2];
      __syncwarp();  // the previous chunk's outputs have left the buffer
#pragma unroll
      for (int n2 = 0; n2 < NB; ++n2) {
        uint32_t w[4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int nt = 2 * n2 + h;
          const float2 f = *(const float2*)&sc[2 * C + 8 * nt + 2 * c];
          const float f0 = f.x * sup, f1 = f.y * sup;
          const __nv_bfloat162 a = __floats2bfloat162_rn(oq[nt][0] * f0 + o[nt][0] * up, oq[nt][1] * f1 + o[nt][1] * up);
          const __nv_bfloat162 z = __floats2bfloat162_rn(oq[nt][2] * f0 + o[nt][2] * up, oq[nt][3] * f1 + o[nt][3] * up);
          w[2 * h] = *(const uint32_t*)&a, w[2 * h + 1] = *(const uint32_t*)&z;
        }
        const int row = 16 * n2 + 8 * (lane >> 4) + (lane & 7), half = (lane >> 3) & 1;
        stsm4_t(smem_u32(obuf) + row * 32 + ((half ^ ((row >> 2) & 1)) << 4), w[0], w[1], w[2], w[3]);
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int row = 16 * i + (lane >> 1), half = lane & 1, tok = tok0 + row;
        if (tok < p.tokens && col0 + half * 8 < p.dv)
          *(uint4*)(out + tok * orow + half * 8) = *(const uint4*)(obuf + row * 32 + ((half ^ ((row >> 2) & 1)) << 4));
      }
    }
    if (TREE) break;
    // 5. S^T = e^G_C S^T + (V' diag(e^(G_C - G)))^T K, accumulated apart
    m = 0.f;
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) {
      const float2 w = *(const float2*)&sc[C + 8 * i + 2 * c];
      x[i][0] *= w.x, x[i][1] *= w.y, x[i][2] *= w.x, x[i][3] *= w.y;
      m = fmaxf(m, fmaxf(fmaxf(fabsf(x[i][0]), fabsf(x[i][1])), fmaxf(fabsf(x[i][2]), fabsf(x[i][3]))));
    }
    const int eu = scale_exp(warp_max_abs(m));
    const float udown = pow2(-eu), uup = pow2(eu), decay = sc[3 * C];
#pragma unroll
    for (int k = 0; k < NB; ++k) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        split2(x[2 * k + h][0] * udown, x[2 * k + h][1] * udown, rh[k][2 * h], rl[k][2 * h]);
        split2(x[2 * k + h][2] * udown, x[2 * k + h][3] * udown, rh[k][2 * h + 1], rl[k][2 * h + 1]);
      }
    }
#pragma unroll
    for (int j2 = 0; j2 < NT / 2; ++j2) {
      float a0[4] = {0.f, 0.f, 0.f, 0.f}, a1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        uint32_t kb[4];
        ldsm4_t(ks_s + img_off<DKP>(16 * k + (lane & 15), 2 * j2 + (lane >> 4)), kb);
        mma_f16(a0, rh[k], kb[0], kb[1]);
        mma_f16(a1, rh[k], kb[2], kb[3]);
        mma_f16(a0, rl[k], kb[0], kb[1]);
        mma_f16(a1, rl[k], kb[2], kb[3]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        S[2 * j2][e] = fmaf(a0[e], uup, S[2 * j2][e] * decay);
        S[2 * j2 + 1][e] = fmaf(a1[e], uup, S[2 * j2 + 1][e] * decay);
      }
    }
  }

  // rows of tokens that no chunk covered: zeros
  {
    const int from = (p.chunk0 + nlive) * C, to = min(p.tokens, (p.chunk0 + p.chunks) * C);
    for (int i = lane; i < (to - from) * 2; i += 32) {
      const int tok = from + (i >> 1), half = i & 1;
      if (col0 + half * 8 < p.dv) *(uint4*)(out + tok * orow + half * 8) = make_uint4(0u, 0u, 0u, 0u);
    }
  }
  if (TREE) return;
  float* So = p.state_out + sb;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = 8 * n + 2 * c + (e & 1);
      if (d < p.dk && (e < 2 ? cok0 : cok1)) So[(long)d * p.dv + col0 + g + 8 * (e >> 1)] = S[n][e];
    }
}

int pad_dk(int dk) { return dk <= 64 ? 64 : 128; }
size_t chunk_bytes(int hk, int hv, int dk) { return (size_t)hk * 2 * C * pad_dk(dk) * 2 + (size_t)hv * HEAD_BYTES; }

// Chunks per segment: a segment's images (1.3 MB per chunk at 16 key and 32 value heads) stay in the L2 between the kernel that
// writes them and the one that reads them, and the scratch of a long prompt stays bounded.
int segment_chunks(int batch, int tokens, int hk, int hv, int dk) {
  const int chunks = (tokens + C - 1) / C;
  const size_t per = chunk_bytes(hk, hv, dk) * batch;
  long fit = (long)((size_t)64 * 1024 * 1024 / per);
  if (fit < 4) fit = 4;
  if (fit >= chunks) return chunks;
  const int parts = (int)((chunks + fit - 1) / fit);
  return (chunks + parts - 1) / parts;
}

template <int DKP> constexpr int prep_smem() { return 2 * C * DKP * 2 + 2 * C * TS * 4 + 32 * 36 * 4; }

// Blocks of 16 tokens that a chunk computes: all four, or fewer where the whole call has no more tokens (a draft).
int token_blocks(int tokens) { return tokens <= 16 ? 1 : tokens <= 32 ? 2 : 4; }

// Calls f.template operator()<DKP, NW, NB, TREE>() for the instance that serves (dkp, nw, nb).
template <bool TREE, int DKP, int NW, typename F>
int with_nb(int nb, F f) {
  return nb == 1 ? f.template operator()<DKP, NW, 1, TREE>() : nb == 2 ? f.template operator()<DKP, NW, 2, TREE>() : f.template operator()<DKP, NW, 4, TREE>();
}
template <bool TREE, int DKP, typename F>
int with_nw(int nw, int nb, F f) {
  return nw == 2 ? with_nb<TREE, DKP, 2>(nb, f) : nw == 4 ? with_nb<TREE, DKP, 4>(nb, f) : with_nb<TREE, DKP, 8>(nb, f);
}
template <typename F>
int with_instance(bool tree, int dkp, int nw, int nb, F f) {
  if (tree) return dkp == 64 ? with_nw<true, 64>(nw, nb, f) : with_nw<true, 128>(nw, nb, f);
  return dkp == 64 ? with_nw<false, 64>(nw, nb, f) : with_nw<false, 128>(nw, nb, f);
}

struct Configure {
  template <int DKP, int NW, int NB, bool TREE>
  int operator()() const {
    cudaError_t e = cudaFuncSetAttribute(delta_prep_kernel<DKP, TREE>, cudaFuncAttributeMaxDynamicSharedMemorySize, prep_smem<DKP>());
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(delta_scan_kernel<DKP, NW, NB, TREE>, cudaFuncAttributeMaxDynamicSharedMemorySize, Scan<DKP, NW>::SMEM);
    return e == cudaSuccess ? 0 : check_launch("delta rule: shared-memory opt-in");
  }
};
int configure_all() {
  for (int tree = 0; tree < 2; ++tree)
    for (int dkp = 64; dkp <= 128; dkp *= 2)
      for (int nw = 2; nw <= 8; nw *= 2)
        for (int nb = 1; nb <= 4; nb *= 2)
          if (const int rc = with_instance(tree, dkp, nw, nb, Configure())) return rc;
  return 0;
}

struct LaunchSegment {
  const DeltaChunkParams& p;
  cudaStream_t stream;
  template <int DKP, int NW, int NB, bool TREE>
  int operator()() const {
    delta_prep_kernel<DKP, TREE><<<dim3(p.chunks, p.hk, p.batch), PREP_THREADS, prep_smem<DKP>(), stream>>>(p);
    const int rc = check_launch("delta rule preparation");
    if (rc) return rc;
    delta_scan_kernel<DKP, NW, NB, TREE>
        <<<dim3((p.dv + 16 * NW - 1) / (16 * NW), p.hv, p.batch), Scan<DKP, NW>::THREADS, Scan<DKP, NW>::SMEM, stream>>>(p);
    return check_launch("delta rule scan");
  }
};

}  // namespace

size_t delta_chunk_scratch_bytes(int batch, int tokens, int hk, int hv, int dk) {
  return chunk_bytes(hk, hv, dk) * batch * segment_chunks(batch, tokens, hk, hv, dk);
}

int launch_delta_chunk(const DeltaChunkParams& args, cudaStream_t stream) {
  static OncePerDevice once;
  int rc = once.run(configure_all);
  if (rc) return rc;
  DeltaChunkParams p = args;
  const bool tree = p.parents != nullptr;
  const int chunks = (p.tokens + C - 1) / C;
  p.seg_chunks = segment_chunks(p.batch, p.tokens, p.hk, p.hv, p.dk);
  // Columns per CTA: few (32) while that is what it takes to put every SM to work, else as many as share the loads.
  const long warps = (long)p.batch * p.hv * ((p.dv + 15) / 16);
  const int nw = warps <= 2 * 148 ? 2 : warps <= 4 * 148 ? 4 : 8;
  for (int at = 0; at < chunks; at += p.seg_chunks) {
    p.chunk0 = at;
    p.chunks = chunks - at < p.seg_chunks ? chunks - at : p.seg_chunks;
    p.first = at == 0;
    p.last = at + p.chunks == chunks;
    rc = with_instance(tree, pad_dk(p.dk), nw, token_blocks(p.tokens), LaunchSegment{p, stream});
    if (rc) return rc;
  }
  return 0;
}

}  // namespace dfb
