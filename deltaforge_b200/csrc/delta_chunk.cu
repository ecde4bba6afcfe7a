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
// Scan: two warps own 16 value columns of a head's state, half of the key rows each, in registers, as the accumulators of
// S^T (16 x dk/2). Their layout is that of the A operand of the next product, so R^T, V'^T and S^T follow from one another
// inside the warp; the two exchange their partial sums of K S once per chunk. A third warp makes the output of the chunk
// before from S and V', handed over as fp16 fragments, so that only what the next state needs is in the chain from chunk to
// chunk. k, q, T, P come through shared memory, which two loader warps fill by cp.async. No wait spins.
#include <cuda_fp16.h>

#include "common.cuh"
#include "kernels.h"

namespace dfb {

namespace {

constexpr int C = 64;                // tokens per chunk
constexpr int SQ = C * C * 2;        // bytes of one 64 x 64 fp16 image
constexpr int SCAL = 4 * C * 4;      // scalars of a (chunk, value head): three per token, the state's decay, four scales each of T and P
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
// The same for a row whose sum of squares is ss: no element exceeds its root.
__device__ __forceinline__ int norm_exp(float ss) { return (((int)((__float_as_uint(ss) >> 23) & 255) - 127 + 2) >> 1) - 13; }
// Largest of the lanes' non-negative values, whose bit patterns order like the values
__device__ __forceinline__ float warp_max_abs(float m) { return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m))); }
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

// Images are rows of W fp16 with 16-byte chunks permuted within 128 bytes, so that 8x8 matrix loads are free of conflicts.
template <int W> __device__ __forceinline__ uint32_t img_off(int row, int chunk) {
  return (uint32_t)(row * W * 2 + ((chunk ^ (row & 7)) << 4));
}

constexpr int PREP_THREADS = 128;
constexpr int TS = 68;  // row stride (floats) of the 64 x 64 fp32 matrices: 16-byte rows, neighbouring rows in other banks

// 2^x: one instruction, 2 ulp
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// z[r] = sum over m < M of a[4 r][m] y[m]: every fourth row of a (stride TS) against one column of y (stride TS). The four groups
// of lanes take neighbouring rows, which lie in different banks.
template <int R, int M>
__device__ __forceinline__ void block_product(float (&z)[R], const float* a, const float* y) {
#pragma unroll
  for (int r = 0; r < R; ++r) z[r] = 0.f;
#pragma unroll
  for (int m = 0; m < M; m += 4) {
    const float y0 = y[m * TS], y1 = y[(m + 1) * TS], y2 = y[(m + 2) * TS], y3 = y[(m + 3) * TS];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float4 x = *(const float4*)(a + 4 * r * TS + m);
      z[r] = fmaf(x.x, y0, fmaf(x.y, y1, fmaf(x.z, y2, fmaf(x.w, y3, z[r]))));
    }
  }
}

// One CTA per (chunk, value head, sequence); warp w owns rows 16 w .. 16 w + 15 of all 64 x 64 matrices.
//   1. keys and queries to shared memory (bf16), their norms and fp16 images; log decays summed (in units of log 2)
//   2. K K^T and Q K^T rows by mma; decays; A to shared memory, P to its image
//   3. the 16 x 16 diagonal blocks of (I + A)^-1 by substitution, a column per lane
//   4. two doublings, 16 -> 32 -> 64
//   5. T diag(beta) in halves to its images
// Bound by latency: three to four CTAs share an SM. Scales are per warp (16 rows), so no CTA-wide maximum is needed.
template <int DKP, bool TREE>
__global__ void __launch_bounds__(PREP_THREADS, 4) delta_prep_kernel(const DeltaChunkParams p) {
  extern __shared__ __align__(128) unsigned char smem[];
  unsigned char* kt = smem;                                  // bf16 [64][DKP]
  unsigned char* qt = smem + C * DKP * 2;
  float* A = (float*)(smem + (2 * C * DKP * 2 > C * TS * 4 ? 2 * C * DKP * 2 : C * TS * 4));  // [64][TS]
  float* T = (float*)smem;                                   // [64][TS], over the tiles once they have been read
  __shared__ float4 col[C];                                  // per token: log2 decay sum (hi, lo), 1/|k|, beta
  __shared__ float rq[C], sk[C], sq[C];
  __shared__ unsigned long long anc[C];
  __shared__ int up[C];
  __shared__ double gsum[C];

  const int cl = blockIdx.x, hv = blockIdx.y, b = blockIdx.z, group = p.hv / p.hk, hk = hv / group;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31, g = lane >> 2, c = lane & 3;
  const int tok0 = (p.chunk0 + cl) * C;
  const int len = p.lengths ? min(max(p.lengths[b], 0), p.tokens) : p.tokens;
  const int live = min(len - tok0, C);  // tokens of this chunk; the scan does not read chunks without any
  // Launched beside the scan of the segment before: whatever follows this grid must find that scan done too, so one CTA stays
  // until it is.
  const bool stays = p.beside && blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1 && blockIdx.z == gridDim.z - 1;
  if (live <= 0) {
    if (stays) pdl_wait();
    return;
  }

  if (TREE) {  // bit j of anc[i]: j is i or an ancestor of i; 0 where row i holds no node
    if (t < C) {
      const int pa = t < live ? p.parents[(long)b * p.parents_stride + t] : -2;
      const bool node = pa >= -1 && pa < t;
      anc[t] = node ? 1ull << t : 0ull;
      up[t] = node ? pa : -1;
    }
    __syncthreads();
    for (int step = 1; step < live; step *= 2) {
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

  const long sbase = ((long)b * p.seg_chunks + cl) * (p.hk * (2L * C * DKP * 2) + p.hv * (long)HEAD_BYTES);
  unsigned char* kimg = p.scratch + sbase + (long)hk * (2 * C * DKP * 2);
  unsigned char* himg = p.scratch + sbase + p.hk * (2L * C * DKP * 2) + (long)hv * HEAD_BYTES;
  const bool first = hv % group == 0;  // the first value head of a key head writes the key head's images

  // ---- 1 ----
  {
    constexpr int N = DKP / 64;  // 16-byte chunks per thread and row: eight threads per row, 16 rows per pass
    const int part = t & 7;
    uint4 raw[2][4][N];
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
      for (int pass = 0; pass < 4; ++pass) {
        const int row = pass * 16 + (t >> 3);
        const bf16* src = which ? p.q + b * p.q_stride[0] + (long)(tok0 + row) * p.q_stride[1] + hk * p.q_stride[2]
                                : p.k + b * p.k_stride[0] + (long)(tok0 + row) * p.k_stride[1] + hk * p.k_stride[2];
        const bool ok = row < live && (!TREE || anc[row] != 0);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int ch = part + 8 * i;
          raw[which][pass][i] = ok && ch * 8 < p.dk ? *(const uint4*)(src + ch * 8) : make_uint4(0, 0, 0, 0);
        }
      }
    // decays and beta: warps 0 and 1 one token per lane; the sum by warp 0 while the tiles arrive
    float bv = 0.f;
    if (t < C) {
      float gv = 0.f;
      if (t < live && (!TREE || anc[t] != 0)) {
        gv = p.g[((long)b * p.tokens + tok0 + t) * p.hv + hv];
        bv = p.beta[((long)b * p.tokens + tok0 + t) * p.hv + hv];
        gv = gv < MIN_LOG_DECAY ? MIN_LOG_DECAY : gv;
      }
      gsum[t] = (double)gv * 1.4426950408889634074;  // log2(e)
      col[t].w = bv;
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
        const double s0 = s - a1;
        col[2 * lane].x = (float)s0, col[2 * lane].y = (float)(s0 - (double)(float)s0);
        col[2 * lane + 1].x = (float)s, col[2 * lane + 1].y = (float)(s - (double)(float)s);
      }
    } else if (t < C) {  // along the path
      double s = 0.;
      unsigned long long bits = anc[t];
      while (bits) {
        s += gsum[__ffsll(bits) - 1];
        bits &= bits - 1;
      }
      col[t].x = (float)s, col[t].y = (float)(s - (double)(float)s);
    }
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
      for (int pass = 0; pass < 4; ++pass) {
        const int row = pass * 16 + (t >> 3);
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const bf16* e = (const bf16*)&raw[which][pass][i];
#pragma unroll
          for (int y = 0; y < 8; ++y) ss = fmaf(bf2f(e[y]), bf2f(e[y]), ss);
        }
#pragma unroll
        for (int o = 1; o < 8; o *= 2) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float down = pow2(-norm_exp(ss));
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int ch = part + 8 * i;
          const bf16* e = (const bf16*)&raw[which][pass][i];
          *(uint4*)((which ? qt : kt) + img_off<DKP>(row, ch)) = raw[which][pass][i];
          if (first) {
            uint4 im;
            im.x = h2(bf2f(e[0]) * down, bf2f(e[1]) * down), im.y = h2(bf2f(e[2]) * down, bf2f(e[3]) * down);
            im.z = h2(bf2f(e[4]) * down, bf2f(e[5]) * down), im.w = h2(bf2f(e[6]) * down, bf2f(e[7]) * down);
            *(uint4*)(kimg + which * (C * DKP * 2) + img_off<DKP>(row, ch)) = im;
          }
        }
        if (part == 0) (which ? sq : sk)[row] = ss;
      }
  }
  __syncthreads();
  {  // norms and image scales, a row per thread (used behind the next barrier)
    const int row = t & 63;
    const bool is_q = t >= 64;
    const float ss = (is_q ? sq : sk)[row];
    float r = p.l2norm ? rsqrt_2step(__fadd_rn(ss, 1e-6f)) : 1.f;
    if (is_q && p.l2norm) r = __fdiv_rn(r, sqrtf((float)p.dk));
    if (is_q) rq[row] = r;
    else col[row].z = r;
    (is_q ? sq : sk)[row] = r * pow2(norm_exp(ss));
  }

  // ---- 2 ----
  const int r0 = warp * 16;
  {
    float kk[8][4], qk[8][4];
#pragma unroll
    for (int nt = 0; nt < 8; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) kk[nt][e] = qk[nt][e] = 0.f;
    const uint32_t ks_s = smem_u32(kt), qs_s = smem_u32(qt);
#pragma unroll
    for (int ks = 0; ks < DKP / 16; ++ks) {
      uint32_t ka[4], qa[4];
      ldsm4(ks_s + img_off<DKP>(r0 + (lane & 15), 2 * ks + (lane >> 4)), ka);
      ldsm4(qs_s + img_off<DKP>(r0 + (lane & 15), 2 * ks + (lane >> 4)), qa);
#pragma unroll
      for (int n2 = 0; n2 < 4; ++n2) {
        if (n2 > warp) continue;  // above the diagonal
        uint32_t kb[4];
        ldsm4(ks_s + img_off<DKP>(16 * n2 + (lane & 7) + 8 * (lane >> 4), 2 * ks + ((lane >> 3) & 1)), kb);
        mma_bf16(kk[2 * n2], ka, kb[0], kb[1]);
        mma_bf16(kk[2 * n2 + 1], ka, kb[2], kb[3]);
        mma_bf16(qk[2 * n2], qa, kb[0], kb[1]);
        mma_bf16(qk[2 * n2 + 1], qa, kb[2], kb[3]);
      }
    }
    __syncthreads();
    float pm = 0.f;
    float ri[2], qi[2], hi[2], lo[2];
    unsigned long long bits[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int i = r0 + g + 8 * r;
      const float4 v = col[i];
      hi[r] = v.x, lo[r] = v.y, ri[r] = v.z * v.w, qi[r] = rq[i];
      bits[r] = TREE ? anc[i] : i < live ? (2ull << i) - 1 : 0ull;  // row i sees columns 0 .. i (2 << 63 wraps to 0: all of them)
    }
#pragma unroll
    for (int nt = 0; nt < 8; ++nt) {
      if (nt > 2 * warp + 1) {  // above the diagonal: kk and qk are zero there
        continue;
      }
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int j = nt * 8 + 2 * c + y;
        const float4 v = col[j];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float d = (bits[r] >> j) & 1 ? v.z * exp2_fast((hi[r] - v.x) + (lo[r] - v.y)) : 0.f;
          const int e = 2 * r + y;
          kk[nt][e] = d == 0.f ? 0.f : kk[nt][e] * (ri[r] * d);
          qk[nt][e] = d == 0.f ? 0.f : qk[nt][e] * (qi[r] * d);
          pm = fmaxf(pm, fabsf(qk[nt][e]));
        }
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) *(float2*)&A[(r0 + g + 8 * r) * TS + nt * 8 + 2 * c] = make_float2(kk[nt][2 * r], kk[nt][2 * r + 1]);
    }
    const int ep = scale_exp(warp_max_abs(pm));
    const float down = pow2(-ep);
#pragma unroll
    for (int nt = 0; nt < 8; ++nt) {
      *(uint32_t*)(himg + 2 * SQ + img_off<C>(r0 + g, nt) + 4 * c) = h2(qk[nt][0] * down, qk[nt][1] * down);
      *(uint32_t*)(himg + 2 * SQ + img_off<C>(r0 + g + 8, nt) + 4 * c) = h2(qk[nt][2] * down, qk[nt][3] * down);
    }
    if (lane == 0) ((float*)(himg + 3 * SQ))[3 * C + 8 + warp] = pow2(ep);
  }
  __syncwarp();

  // ---- 3: column (lane & 15) of this warp's diagonal block, rows in registers ----
  float x[16];
  {
    const int j = lane & 15;
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = i == j ? 1.f : 0.f;
#pragma unroll
    for (int i = 1; i < 16; ++i) {
      float a[16];
#pragma unroll
      for (int m = 0; m < i; m += 4) *(float4*)&a[m] = *(const float4*)&A[(r0 + i) * TS + r0 + m];
      float s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int m = 0; m < i; ++m) (m & 1 ? s1 : s0) = fmaf(a[m], x[m], m & 1 ? s1 : s0);
      x[i] -= s0 + s1;
    }
  }
  __syncthreads();  // A is complete, the tiles have been read
  if (lane < 16) {
#pragma unroll
    for (int i = 0; i < 16; ++i) T[(r0 + i) * TS + r0 + lane] = x[i];
  }
  // zeros right of the diagonal block
  for (int i = lane; i < 16 * 4 * (3 - warp); i += 32) {
    const int r = i & 15, q4 = i >> 4;
    *(float4*)&T[(r0 + r) * TS + r0 + 16 + 4 * q4] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __syncthreads();

  // ---- 4 ----
  // The lower left block of a pair of diagonal blocks is -T22 (A21 T11); A21 T11 waits in its place in T. All rows of a column
  // belong to one warp: lanes are eight columns by four groups of rows.
  {
    const int pair = 32 * (warp >> 1), j = pair + 8 * (warp & 1) + (lane & 7), i0 = pair + 16 + (lane >> 3);
    float z[4];
    block_product<4, 16>(z, A + i0 * TS + pair, T + pair * TS + j);
#pragma unroll
    for (int r = 0; r < 4; ++r) T[(i0 + 4 * r) * TS + j] = z[r];
    __syncwarp();
    block_product<4, 16>(z, T + i0 * TS + pair + 16, T + (pair + 16) * TS + j);
    __syncwarp();
#pragma unroll
    for (int r = 0; r < 4; ++r) T[(i0 + 4 * r) * TS + j] = -z[r];
  }
  __syncthreads();
  {
    const int j = 8 * warp + (lane & 7), i0 = 32 + (lane >> 3);
    float z[8];
    block_product<8, 32>(z, A + i0 * TS, T + j);
#pragma unroll
    for (int r = 0; r < 8; ++r) T[(i0 + 4 * r) * TS + j] = z[r];
    __syncwarp();
    block_product<8, 32>(z, T + i0 * TS + 32, T + 32 * TS + j);
    __syncwarp();
#pragma unroll
    for (int r = 0; r < 8; ++r) T[(i0 + 4 * r) * TS + j] = -z[r];
  }
  __syncthreads();

  // ---- 5: this warp's 16 rows, eight columns per lane and pass ----
  {
    float tv[4][8], tm = 0.f;
    const int j0 = (lane & 7) * 8;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float* src = &T[(r0 + 4 * k + (lane >> 3)) * TS + j0];
      *(float4*)&tv[k][0] = *(const float4*)src;
      *(float4*)&tv[k][4] = *(const float4*)(src + 4);
#pragma unroll
      for (int y = 0; y < 8; ++y) {
        tv[k][y] *= col[j0 + y].w;
        tm = fmaxf(tm, fabsf(tv[k][y]));
      }
    }
    const int et = scale_exp(warp_max_abs(tm));
    const float down = pow2(-et);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint4 hi, lo;
      split2(tv[k][0] * down, tv[k][1] * down, hi.x, lo.x);
      split2(tv[k][2] * down, tv[k][3] * down, hi.y, lo.y);
      split2(tv[k][4] * down, tv[k][5] * down, hi.z, lo.z);
      split2(tv[k][6] * down, tv[k][7] * down, hi.w, lo.w);
      *(uint4*)(himg + img_off<C>(r0 + 4 * k + (lane >> 3), lane & 7)) = hi;
      *(uint4*)(himg + SQ + img_off<C>(r0 + 4 * k + (lane >> 3), lane & 7)) = lo;
    }
    float* sc = (float*)(himg + 3 * SQ);
    if (lane == 0) sc[3 * C + 4 + warp] = pow2(et);
    if (t < C) {
      const float4 v = col[t], e = col[C - 1];
      const float eg = exp2_fast(v.x + v.y);
      sc[t] = eg * sk[t];                                             // on K S
      sc[C + t] = exp2_fast((e.x - v.x) + (e.y - v.y)) * sk[t];       // on V' into the state
      sc[2 * C + t] = eg * sq[t];                                     // on Q S
      if (t == C - 1) sc[3 * C] = eg;                                 // decay of the state
    }
  }
  if (stays) pdl_wait();
}

// ---- the scan -------------------------------------------------------------------------------------------------------

// NW: column tiles (of 16) per CTA; two warps each for the recurrence, one for the output, and two loader warps.
template <int DKP, int NW> struct Scan {
  static constexpr int WARPS = 3 * NW + 2, THREADS = WARPS * 32;
  static constexpr int VROW = NW * 32;  // bytes of a token's values in a stage
  // two stages of what the recurrence reads of a chunk: k, T (hi, lo), scalars, values
  static constexpr int T_OFF = C * DKP * 2, A_SC = T_OFF + 2 * SQ, V_OFF = A_SC + SCAL, A_STAGE = V_OFF + C * VROW;
  // two stages of what the output reads, a chunk behind: q, P, scalars
  static constexpr int P_OFF = C * DKP * 2, B_SC = P_OFF + SQ, B_STAGE = B_SC + SCAL;
  // per column tile: partial sums K S of both warps; two handovers (S as fp16 fragments, V' likewise); output rows
  static constexpr int SWAP = 2 * 8 * 32 * 16, HAND = (DKP / 16 + 4) * 32 * 16, OUT = C * 32;
  static constexpr int B_AT = 2 * A_STAGE, SWAP_AT = B_AT + 2 * B_STAGE, HAND_AT = SWAP_AT + NW * SWAP, OUT_AT = HAND_AT + 2 * NW * HAND;
  static constexpr int SMEM = OUT_AT + NW * OUT;
  // NW == 2 leaves room for a CTA of the preparation on the same SM: 55 KB of shared memory, and a quarter of the registers
  static constexpr int REGS = NW == 2 ? 192 : 128;
};

template <int VROW> __device__ __forceinline__ uint32_t v_off(int row, int chunk) {
  const int x = VROW >= 128 ? (chunk ^ (row & 7)) : (chunk ^ ((row >> 1) & (VROW / 16 - 1)));
  return (uint32_t)(row * VROW + (x << 4));
}

template <int DKP, int NW, int NB, bool TREE>
__global__ void __launch_bounds__((3 * NW + 2) * 32) __maxnreg__((Scan<DKP, NW>::REGS)) delta_scan_kernel(const DeltaChunkParams p) {
  using S_ = Scan<DKP, NW>;
  constexpr int NT = DKP / 16;  // 8-wide tiles of key rows per recurrence warp: half of them
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int hand_exp[2][NW][3];  // scales of a handover: S of the two warps, V'
  const int vb = blockIdx.x, hv = blockIdx.y, b = blockIdx.z, hk = hv / (p.hv / p.hk);
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31, g = lane >> 2, c = lane & 3;
  const int len = p.lengths ? min(max(p.lengths[b], 0), p.tokens) : p.tokens;
  const int nlive = min(max((len + C - 1) / C - p.chunk0, 0), p.chunks);  // chunks of this segment with tokens
  const int col_cta = vb * NW * 16;
  pdl_launch_dependents();  // the preparation of the next segment may run beside this one

  // One barrier per chunk for all warps: behind barrier n the recurrence works on chunk n, the output on chunk n - 1, the loads
  // bring chunk n + 1 of the one and chunk n of the other.
  if (warp >= 3 * NW) {  // ---- loader warps ----
    const int lt = t - 3 * NW * 32;
    const long per = p.hk * (2L * C * DKP * 2) + p.hv * (long)HEAD_BYTES;
    auto copy = [&](uint32_t to, const unsigned char* from, int bytes) {
#pragma unroll 4
      for (int i = lt * 16; i < bytes; i += 64 * 16) cp_async16(to + i, from + i, 16);
    };
    for (int n = -1; n <= nlive; ++n) {
      cp_async_wait<0>();
      if (n >= 0) __syncthreads();
      const unsigned char* base = p.scratch + (long)b * p.seg_chunks * per + (long)hk * (2 * C * DKP * 2);
      const unsigned char* head = p.scratch + (long)b * p.seg_chunks * per + p.hk * (2L * C * DKP * 2) + (long)hv * HEAD_BYTES;
      if (n + 1 < nlive) {
        const uint32_t st = smem_u32(smem + ((n + 1) & 1) * S_::A_STAGE);
        copy(st, base + (n + 1) * per, C * DKP * 2);
        copy(st + S_::T_OFF, head + (n + 1) * per, 2 * SQ);
        copy(st + S_::A_SC, head + (n + 1) * per + 3 * SQ, SCAL);
        const int tok0 = (p.chunk0 + n + 1) * C;
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
      if (n >= 0 && n < nlive) {
        const uint32_t st = smem_u32(smem + S_::B_AT + (n & 1) * S_::B_STAGE);
        copy(st, base + n * per + C * DKP * 2, C * DKP * 2);
        copy(st + S_::P_OFF, head + n * per + 2 * SQ, SQ);
        copy(st + S_::B_SC, head + n * per + 3 * SQ, SCAL);
      }
      cp_async_commit();
    }
    return;
  }

  if (warp >= 2 * NW) {  // ---- output warps: 16 value columns each ----
    const int ct = warp - 2 * NW, col0 = col_cta + ct * 16;
    unsigned char* obuf = smem + S_::OUT_AT + ct * S_::OUT;
    bf16* out = p.out + ((long)b * p.tokens * p.hv + hv) * p.dv + col0;
    const long orow = (long)p.hv * p.dv;
    for (int n = 0; n <= nlive; ++n) {
      __syncthreads();
      if (n == 0) continue;
      const int k_ = n - 1, buf = k_ & 1, tok0 = (p.chunk0 + k_) * C;
      const unsigned char* st = smem + S_::B_AT + buf * S_::B_STAGE;
      const uint32_t qs_s = smem_u32(st);
      const float* sc = (const float*)(st + S_::B_SC);
      const uint4* hand = (const uint4*)(smem + S_::HAND_AT + (buf * NW + ct) * S_::HAND) + lane;
      // O^T = (S^T Q^T) diag(e^G) + V'^T P^T
      float o[2 * NB][4];
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
#pragma unroll
      for (int hd = 0; hd < 2; ++hd) {
        float x[2 * NB][4];
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0.f;
#pragma unroll
        for (int ks = 0; ks < NT / 2; ++ks) {
          const uint4 av = hand[(hd * (NT / 2) + ks) * 32];
          const uint32_t a[4] = {av.x, av.y, av.z, av.w};
#pragma unroll
          for (int n2 = 0; n2 < NB; ++n2) {
            uint32_t qb[4];
            ldsm4(qs_s + img_off<DKP>(16 * n2 + (lane & 7) + 8 * (lane >> 4), hd * NT + 2 * ks + ((lane >> 3) & 1)), qb);
            mma_f16(x[2 * n2], a, qb[0], qb[1]);
            mma_f16(x[2 * n2 + 1], a, qb[2], qb[3]);
          }
        }
        const float up = pow2(hand_exp[buf][ct][hd]);
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][e] = fmaf(x[i][e], up, o[i][e]);
      }
      float x[2 * NB][4];
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i) x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0.f;
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        const uint4 av = hand[(DKP / 16 + k) * 32];
        const uint32_t a[4] = {av.x, av.y, av.z, av.w};
#pragma unroll
        for (int n2 = k; n2 < NB; ++n2) {
          uint32_t pb[4];
          ldsm4(qs_s + S_::P_OFF + img_off<C>(16 * n2 + (lane & 7) + 8 * (lane >> 4), 2 * k + ((lane >> 3) & 1)), pb);
          mma_f16(x[2 * n2], a, pb[0], pb[1]);
          mma_f16(x[2 * n2 + 1], a, pb[2], pb[3]);
        }
      }
      const float vup = pow2(hand_exp[buf][ct][2]);
      __syncwarp();  // the previous chunk's outputs have left the buffer
#pragma unroll
      for (int n2 = 0; n2 < NB; ++n2) {
        uint32_t w[4];
        const float up = vup * sc[3 * C + 8 + n2];  // P is scaled per 16 rows
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int nt = 2 * n2 + h;
          const float2 f = *(const float2*)&sc[2 * C + 8 * nt + 2 * c];
          const __nv_bfloat162 y = __floats2bfloat162_rn(o[nt][0] * f.x + x[nt][0] * up, o[nt][1] * f.y + x[nt][1] * up);
          const __nv_bfloat162 z = __floats2bfloat162_rn(o[nt][2] * f.x + x[nt][2] * up, o[nt][3] * f.y + x[nt][3] * up);
          w[2 * h] = *(const uint32_t*)&y, w[2 * h + 1] = *(const uint32_t*)&z;
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
    // rows of tokens that no chunk covered: zeros
    const int from = (p.chunk0 + nlive) * C, to = min(p.tokens, (p.chunk0 + p.chunks) * C);
    for (int i = lane; i < (to - from) * 2; i += 32) {
      const int tok = from + (i >> 1), half = i & 1;
      if (col0 + half * 8 < p.dv) *(uint4*)(out + tok * orow + half * 8) = make_uint4(0u, 0u, 0u, 0u);
    }
    return;
  }

  // ---- recurrence warps: 16 value columns and half of the key rows each ----
  const int ct = warp >> 1, hd = warp & 1;
  const int col0 = col_cta + ct * 16;
  const bool cok0 = col0 + g < p.dv, cok1 = col0 + g + 8 < p.dv;
  const long sb = ((long)b * p.hv + hv) * p.dk * p.dv;
  const float* Sin = p.first ? p.state + sb : p.state_out + sb;
  float S[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = 8 * (hd * NT + n) + 2 * c + (e & 1);
      const bool ok = d < p.dk && (e < 2 ? cok0 : cok1);
      S[n][e] = ok ? Sin[(long)d * p.dv + col0 + g + 8 * (e >> 1)] : 0.f;
    }
  float4* swap = (float4*)(smem + S_::SWAP_AT + ct * S_::SWAP);
  float4 *mine = swap + hd * (8 * 32) + lane, *other = swap + (hd ^ 1) * (8 * 32) + lane;

  for (int n = 0; n <= nlive; ++n) {
    __syncthreads();
    if (n == nlive) break;
    const unsigned char* st = smem + (n & 1) * S_::A_STAGE;
    const uint32_t ks_s = smem_u32(st), ti_s = ks_s + S_::T_OFF, vs_s = ks_s + S_::V_OFF;
    const float* sc = (const float*)(st + S_::A_SC);
    uint4* hand = (uint4*)(smem + S_::HAND_AT + ((n & 1) * NW + ct) * S_::HAND) + lane;

    // 1. S^T K^T over this warp's key rows; hi goes to the output warp too
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < NT; ++i) m = fmaxf(m, fmaxf(fmaxf(fabsf(S[i][0]), fabsf(S[i][1])), fmaxf(fabsf(S[i][2]), fabsf(S[i][3]))));
    const int es = scale_exp(warp_max_abs(m));
    const float sdown = pow2(-es), sup = pow2(es);
    if (lane == 0) hand_exp[n & 1][ct][hd] = es;
    float x[2 * NB][4];
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[i][e] = 0.f;
#pragma unroll
    for (int ks = 0; ks < NT / 2; ++ks) {
      uint32_t hi[4], lo[4];
      split2(S[2 * ks][0] * sdown, S[2 * ks][1] * sdown, hi[0], lo[0]);
      split2(S[2 * ks][2] * sdown, S[2 * ks][3] * sdown, hi[1], lo[1]);
      split2(S[2 * ks + 1][0] * sdown, S[2 * ks + 1][1] * sdown, hi[2], lo[2]);
      split2(S[2 * ks + 1][2] * sdown, S[2 * ks + 1][3] * sdown, hi[3], lo[3]);
      hand[(hd * (NT / 2) + ks) * 32] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      uint32_t kb[NB][4];
#pragma unroll
      for (int n2 = 0; n2 < NB; ++n2) {
        ldsm4(ks_s + img_off<DKP>(16 * n2 + (lane & 7) + 8 * (lane >> 4), hd * NT + 2 * ks + ((lane >> 3) & 1)), kb[n2]);
        mma_f16(x[2 * n2], hi, kb[n2][0], kb[n2][1]);
        mma_f16(x[2 * n2 + 1], hi, kb[n2][2], kb[n2][3]);
      }
#pragma unroll
      for (int n2 = 0; n2 < NB; ++n2) {
        mma_f16(x[2 * n2], lo, kb[n2][0], kb[n2][1]);
        mma_f16(x[2 * n2 + 1], lo, kb[n2][2], kb[n2][3]);
      }
    }
    // the other warp of these columns has the other key rows
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[i][e] *= sup;
      mine[i * 32] = make_float4(x[i][0], x[i][1], x[i][2], x[i][3]);
    }
    asm volatile("bar.sync %0, 64;" ::"r"(1 + ct) : "memory");
    // 2. R = V - diag(e^G) K S, then its halves
    m = 0.f;
#pragma unroll
    for (int n2 = 0; n2 < NB; ++n2) {
      uint32_t vr[4];
      ldsm4_t(vs_s + v_off<S_::VROW>(16 * n2 + (lane & 15), ct * 2 + (lane >> 4)), vr);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int nt = 2 * n2 + h;
        const float2 w = *(const float2*)&sc[8 * nt + 2 * c];
        const float4 y = other[nt * 32];
        const float2 v0 = __bfloat1622float2(*(const __nv_bfloat162*)&vr[h]), v1 = __bfloat1622float2(*(const __nv_bfloat162*)&vr[2 + h]);
        x[nt][0] = v0.x - (x[nt][0] + y.x) * w.x;
        x[nt][1] = v0.y - (x[nt][1] + y.y) * w.y;
        x[nt][2] = v1.x - (x[nt][2] + y.z) * w.x;
        x[nt][3] = v1.y - (x[nt][3] + y.w) * w.y;
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
    // 3. V'^T = R^T T^T (both warps); block (i, j) of T is zero for j > i
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
      const float up = pow2(er);
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i) {
        const float u = up * sc[3 * C + 4 + i / 2];  // T is scaled per 16 rows
#pragma unroll
        for (int e = 0; e < 4; ++e) x[i][e] *= u, m = fmaxf(m, fabsf(x[i][e]));
      }
    }
    {  // V' for the output warp, every second block of 16 tokens
      const int ev = scale_exp(warp_max_abs(m));
      const float vdown = pow2(-ev);
      if (lane == 0) hand_exp[n & 1][ct][2] = ev;  // (both warps have the same)
#pragma unroll
      for (int k = 0; k < NB; ++k)
        if ((k & 1) == hd)
          hand[(DKP / 16 + k) * 32] = make_uint4(h2(x[2 * k][0] * vdown, x[2 * k][1] * vdown), h2(x[2 * k][2] * vdown, x[2 * k][3] * vdown),
                                                 h2(x[2 * k + 1][0] * vdown, x[2 * k + 1][1] * vdown), h2(x[2 * k + 1][2] * vdown, x[2 * k + 1][3] * vdown));
    }
    if (TREE) continue;
    // 4. S^T = e^G_C S^T + (V' diag(e^(G_C - G)))^T K over this warp's key rows, accumulated apart
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
    // two pairs of tiles at a time: four chains of products
#pragma unroll
    for (int j4 = 0; j4 < NT / 4; ++j4) {
      float a[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i][0] = a[i][1] = a[i][2] = a[i][3] = 0.f;
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        uint32_t k0[4], k1[4];
        ldsm4_t(ks_s + img_off<DKP>(16 * k + (lane & 15), hd * NT + 4 * j4 + (lane >> 4)), k0);
        ldsm4_t(ks_s + img_off<DKP>(16 * k + (lane & 15), hd * NT + 4 * j4 + 2 + (lane >> 4)), k1);
        mma_f16(a[0], rh[k], k0[0], k0[1]);
        mma_f16(a[1], rh[k], k0[2], k0[3]);
        mma_f16(a[2], rh[k], k1[0], k1[1]);
        mma_f16(a[3], rh[k], k1[2], k1[3]);
        mma_f16(a[0], rl[k], k0[0], k0[1]);
        mma_f16(a[1], rl[k], k0[2], k0[3]);
        mma_f16(a[2], rl[k], k1[0], k1[1]);
        mma_f16(a[3], rl[k], k1[2], k1[3]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) S[4 * j4 + i][e] = fmaf(a[i][e], uup, S[4 * j4 + i][e] * decay);
    }
  }
  if (TREE) return;
  float* So = p.state_out + sb;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = 8 * (hd * NT + n) + 2 * c + (e & 1);
      if (d < p.dk && (e < 2 ? cok0 : cok1)) So[(long)d * p.dv + col0 + g + 8 * (e >> 1)] = S[n][e];
    }
}

// ---- a few tokens, one by one ---------------------------------------------------------------------------------------

// One or a few tokens per sequence: the recurrence itself in fp32, bound by reading and writing the state once. A CTA owns 32
// value columns of a head: lane = column, each of the eight warps holds 16 key rows of them in registers from the first
// token to the last; the two sums over the key rows go through shared memory.
constexpr int FEW = 4;  // most tokens (what the chunked form needs for one chunk is reached at about that many)
constexpr int FEW_THREADS = 256, FEW_ROWS = 16;

__global__ void __launch_bounds__(FEW_THREADS) delta_few_kernel(const DeltaChunkParams p) {
  __shared__ float qn[FEW][128], kn[FEW][128], gate[FEW][2];
  __shared__ float red[2][8][32];
  const int vb = blockIdx.x, hv = blockIdx.y, b = blockIdx.z, hk = hv / (p.hv / p.hk);
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31, col = vb * 32 + lane;
  const bool cok = col < p.dv;
  const long sb = ((long)b * p.hv + hv) * p.dk * p.dv;
  float s[FEW_ROWS];
#pragma unroll
  for (int i = 0; i < FEW_ROWS; ++i) {
    const int k = warp * FEW_ROWS + i;
    s[i] = cok && k < p.dk ? p.state[sb + (long)k * p.dv + col] : 0.f;
  }
  const int len = p.lengths ? min(max(p.lengths[b], 0), p.tokens) : p.tokens;
  // queries by warps 0 .. 3, keys by warps 4 .. 7, a token each
  const int tok = warp & 3, is_k = warp >> 2;
  if (tok < len) {
    const bf16* src = is_k ? p.k + b * p.k_stride[0] + tok * p.k_stride[1] + hk * p.k_stride[2] : p.q + b * p.q_stride[0] + tok * p.q_stride[1] + hk * p.q_stride[2];
    float x[4], ss = 0.f;
    uint2 raw = make_uint2(0u, 0u);
    if (4 * lane < p.dk) raw = *(const uint2*)(src + 4 * lane);
    const bf16* e = (const bf16*)&raw;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = bf2f(e[i]), ss = fmaf(x[i], x[i], ss);
    float r = 1.f;
    if (p.l2norm) {
      r = rsqrt_2step(__fadd_rn(warp_sum(ss), 1e-6f));
      if (!is_k) r = __fdiv_rn(r, sqrtf((float)p.dk));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) (is_k ? kn : qn)[tok][4 * lane + i] = x[i] * r;
    if (is_k && lane == 0) {
      gate[tok][0] = expf(p.g[((long)b * p.tokens + tok) * p.hv + hv]);
      gate[tok][1] = p.beta[((long)b * p.tokens + tok) * p.hv + hv];
    }
  }
  float v[FEW];
#pragma unroll
  for (int n = 0; n < FEW; ++n) v[n] = cok && n < len ? bf2f(p.v[b * p.v_stride[0] + n * p.v_stride[1] + hv * p.v_stride[2] + col]) : 0.f;
  __syncthreads();
#pragma unroll 1
  for (int n = 0; n < len; ++n) {
    const float decay = gate[n][0];
    float r = 0.f;
#pragma unroll
    for (int i = 0; i < FEW_ROWS; ++i) {
      s[i] *= decay;
      r = fmaf(s[i], kn[n][warp * FEW_ROWS + i], r);
    }
    red[0][warp][lane] = r;
    __syncthreads();
    r = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) r += red[0][w][lane];
    float vn = v[0];
#pragma unroll
    for (int i = 1; i < FEW; ++i) vn = n == i ? v[i] : vn;
    const float d = (vn - r) * gate[n][1];
    float o = 0.f;
#pragma unroll
    for (int i = 0; i < FEW_ROWS; ++i) {
      s[i] = fmaf(kn[n][warp * FEW_ROWS + i], d, s[i]);
      o = fmaf(s[i], qn[n][warp * FEW_ROWS + i], o);
    }
    red[1][warp][lane] = o;
    __syncthreads();
    if (warp == 0 && cok) {
      o = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) o += red[1][w][lane];
      p.out[(((long)b * p.tokens + n) * p.hv + hv) * p.dv + col] = f2bf(o);
    }
  }
#pragma unroll
  for (int i = 0; i < FEW_ROWS; ++i) {
    const int k = warp * FEW_ROWS + i;
    if (cok && k < p.dk) p.state_out[sb + (long)k * p.dv + col] = s[i];
  }
  for (int n = len + warp; n < p.tokens; n += 8)
    if (cok) p.out[(((long)b * p.tokens + n) * p.hv + hv) * p.dv + col] = f2bf(0.f);
}

int pad_dk(int dk) { return dk <= 64 ? 64 : 128; }
size_t chunk_bytes(int hk, int hv, int dk) { return (size_t)hk * 2 * C * pad_dk(dk) * 2 + (size_t)hv * HEAD_BYTES; }

// How a prompt is walked through: in segments, each prepared by one kernel and scanned by the next. The scratch of a long prompt
// so stays bounded, and in the L2 (1.3 MB per chunk at 16 key and 32 value heads).
// Where the scan fills the SMs once with its smaller CTAs (one or few sequences), segments are short and the preparation of
// each runs beside the scan of the one before, out of the other half of the scratch; only the first is waited for. One
// sequence of 8192 tokens and 32 heads: 422 us one after the other, of which 120 preparation.
struct Walk {
  int nw;      // column tiles per CTA of the scan
  int chunks;  // per segment
  bool beside;
};
Walk plan_walk(int batch, int tokens, int hk, int hv, int dk, int dv) {
  Walk w;
  const int chunks = (tokens + C - 1) / C;
  const long col_tiles = (long)batch * hv * ((dv + 15) / 16);
  // Columns per CTA: few (32) while that is what it takes to put every SM to work, else as many as share the loads.
  w.nw = col_tiles <= 2 * 148 ? 2 : 4;
  const size_t per = chunk_bytes(hk, hv, dk) * batch;
  const long fit = (long)((size_t)64 * 1024 * 1024 / per);
  long seg = fit < 4 ? 4 : fit;
  const long wave = 4 * 148 / ((long)batch * hv);  // chunks whose preparation fills the SMs once
  w.beside = w.nw == 2 && wave >= 4 && chunks > wave;
  if (w.beside) seg = wave < fit / 2 ? wave : fit / 2;
  const int parts = (int)((chunks + seg - 1) / seg);
  w.chunks = (chunks + parts - 1) / parts;
  return w;
}

template <int DKP> constexpr int prep_smem() { return (2 * C * DKP * 2 > C * TS * 4 ? 2 * C * DKP * 2 : C * TS * 4) + C * TS * 4; }

// Blocks of 16 tokens that a chunk computes: all four, or fewer where the whole call has no more tokens (a draft).
int token_blocks(int tokens) { return tokens <= 16 ? 1 : tokens <= 32 ? 2 : 4; }

// Calls f.template operator()<DKP, NW, NB, TREE>() for the instance that serves (dkp, nw, nb).
template <bool TREE, int DKP, int NW, typename F>
int with_nb(int nb, F f) {
  return nb == 1 ? f.template operator()<DKP, NW, 1, TREE>() : nb == 2 ? f.template operator()<DKP, NW, 2, TREE>() : f.template operator()<DKP, NW, 4, TREE>();
}
template <bool TREE, int DKP, typename F>
int with_nw(int nw, int nb, F f) {
  return nw == 2 ? with_nb<TREE, DKP, 2>(nb, f) : with_nb<TREE, DKP, 4>(nb, f);
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
      for (int nw = 2; nw <= 4; nw *= 2)
        for (int nb = 1; nb <= 4; nb *= 2)
          if (const int rc = with_instance(tree, dkp, nw, nb, Configure())) return rc;
  return 0;
}

struct LaunchSegment {
  const DeltaChunkParams& p;
  cudaStream_t stream;
  template <int DKP, int NW, int NB, bool TREE>
  int operator()() const {
    const dim3 grid(p.chunks, p.hv, p.batch);
    if (p.beside) (void)launch_pdl(delta_prep_kernel<DKP, TREE>, grid, dim3(PREP_THREADS), prep_smem<DKP>(), stream, p);
    else delta_prep_kernel<DKP, TREE><<<grid, PREP_THREADS, prep_smem<DKP>(), stream>>>(p);
    const int rc = check_launch("delta rule preparation");
    if (rc) return rc;
    delta_scan_kernel<DKP, NW, NB, TREE>
        <<<dim3((p.dv + 16 * NW - 1) / (16 * NW), p.hv, p.batch), Scan<DKP, NW>::THREADS, Scan<DKP, NW>::SMEM, stream>>>(p);
    return check_launch("delta rule scan");
  }
};

}  // namespace

size_t delta_chunk_scratch_bytes(int batch, int tokens, int hk, int hv, int dk, int dv, bool tree) {
  if (!tree && tokens <= FEW) return 0;
  const Walk w = plan_walk(batch, tokens, hk, hv, dk, dv);
  return chunk_bytes(hk, hv, dk) * batch * w.chunks * (w.beside ? 2 : 1);
}

int launch_delta_chunk(const DeltaChunkParams& args, cudaStream_t stream) {
  static OncePerDevice once;
  int rc = once.run(configure_all);
  if (rc) return rc;
  DeltaChunkParams p = args;
  const bool tree = p.parents != nullptr;
  if (!tree && p.tokens <= FEW) {
    delta_few_kernel<<<dim3((p.dv + 31) / 32, p.hv, p.batch), FEW_THREADS, 0, stream>>>(p);
    return check_launch("delta rule, few tokens");
  }
  const Walk w = plan_walk(p.batch, p.tokens, p.hk, p.hv, p.dk, p.dv);
  const int chunks = (p.tokens + C - 1) / C;
  const size_t half = chunk_bytes(p.hk, p.hv, p.dk) * p.batch * w.chunks;
  p.seg_chunks = w.chunks;
  for (int at = 0, i = 0; at < chunks; at += w.chunks, ++i) {
    p.chunk0 = at;
    p.chunks = chunks - at < w.chunks ? chunks - at : w.chunks;
    p.first = at == 0;
    p.beside = w.beside && i > 0;
    p.scratch = args.scratch + (w.beside && (i & 1) ? half : 0);
    rc = with_instance(tree, pad_dk(p.dk), w.nw, token_blocks(p.tokens), LaunchSegment{p, stream});
    if (rc) return rc;
  }
  return 0;
}

}  // namespace dfb
