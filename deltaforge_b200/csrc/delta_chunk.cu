// The gated delta rule over several new tokens of a sequence (a prompt, or a tree of drafted tokens), sm_100a.
//
// Per value head (key head h / (Hv / Hk)), token by token (src/deltaforge/reference.py:450-458):
//   S <- e^g_t S;  r = S^T k_t;  d = beta_t (v_t - r);  S <- S + k_t d^T;  o_t = S^T q_t
// Over a chunk of C = 64 tokens, with G_i = g_1 + .. + g_i, the same thing is
//   A_ij = beta_i e^(G_i - G_j) k_i.k_j (j < i),  T = (I + A)^-1 diag(beta),  P_ij = e^(G_i - G_j) q_i.k_j (j <= i)
//   W = T diag(e^G) K;  V' = T V - W S;  O = diag(e^G) Q S + P V';  S <- e^G_C S + sum_j e^(G_C - G_j) k_j v'_j^T
// T, W, P and the scalars do not depend on S: delta_prep_kernel makes them for all chunks at once. delta_scan_kernel then walks
// through the chunks of a head; its work is matrix products with S.
// For a tree, "j <= i" reads "j is i or an ancestor of i" and G_i is summed along the path of i; there is one chunk and no
// new state (the accepted path is run through the prompt form afterwards).
//
// Precision. S is fp32 from end to end and so is the new state's bar: an operand rounded to 8 bits (bf16) would cost
// 2e-3 per product. Products with S or V' take fp16 operands (11 bits), scaled by powers of two to the top of fp16's range
// (per token for k and q, which are bf16 and stay exact; per 16 rows for W, P; per value column for S, V'), and S, W and V'
// are split in two, hi + lo = 22 bits, wherever the product leads into the state: hi hi + hi lo + lo hi, fp32 accumulation.
// (The update's V' are scaled by the larger of the two halves of a chunk, each its largest V' times its largest weight: values
// 2^13 times above what the half leaves in the state begin to cost the update bits.)
// Products that lead into the bf16 output alone take hi (2^-12). T V is a product of bf16: the values as they are, T in three
// parts (24 bits); so is W, the left factor in three parts and the keys as they are. The state's update is accumulated apart
// and added in fp32 (the tensor core truncates what it adds to a large accumulator). Log decays are summed in fp64 and kept as
// two floats, so that differences of large sums stay exact.
//
// delta_scan.cu has the scan.
#include "delta.cuh"
#include "tcgen05.cuh"

namespace dfb {

namespace {

constexpr float MIN_LOG_DECAY = -150.f;  // e^-150 is 0 in fp32: keeps sums finite when a log decay is -inf

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// (a, b) as three pairs of bf16 that add up to them: 24 bits
__device__ __forceinline__ void split3(float a, float b, uint32_t& p0, uint32_t& p1, uint32_t& p2) {
  const __nv_bfloat162 x = __floats2bfloat162_rn(a, b);
  const float2 xf = __bfloat1622float2(x);
  const __nv_bfloat162 y = __floats2bfloat162_rn(a - xf.x, b - xf.y);
  const float2 yf = __bfloat1622float2(y);
  const __nv_bfloat162 z = __floats2bfloat162_rn(a - xf.x - yf.x, b - xf.y - yf.y);
  p0 = *(const uint32_t*)&x, p1 = *(const uint32_t*)&y, p2 = *(const uint32_t*)&z;
}

// What the lanes of a warp wrote to shared memory goes to memory by itself; lane 0 has it to wait for
__device__ __forceinline__ void send(unsigned char* dst, const unsigned char* src, uint32_t bytes) {
  fence_async();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) {
    bulk_store(dst, smem_u32(src), bytes);
    bulk_stores_commit();
  }
}

constexpr int PREP_THREADS = 128;
constexpr int TS = 68;  // row stride (floats) of the 64 x 64 fp32 matrices: 16-byte rows, neighbouring rows in other banks

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
//   5. W by mma, T diag(beta) in parts and W in halves to their images
// Bound by latency: four CTAs of one warp per scheduler share an SM and issue in half of the cycles (six prompts of 1001 tokens
// and 32 heads: 73 us, 4400 shared-memory passes and 13000 warp instructions per CTA; no single cause of waiting has a fifth).
// Eight warps per CTA with half of the registers, and the doublings by mma in three parts, were not faster. Scales are per warp
// (16 rows), so no CTA-wide maximum is needed.
template <int DKP, bool TREE>
__global__ void __launch_bounds__(PREP_THREADS, 4) delta_prep_kernel(const DeltaChunkParams p) {
  extern __shared__ __align__(128) unsigned char smem[];
  unsigned char* kt = smem;                                  // bf16 [64][DKP]
  unsigned char* qt = smem + C * DKP * 2;
  float* T = (float*)qt;                                     // [64][TS], over the queries once they have been read
  float* A = T + C * TS;                                     // [64][TS]
  __shared__ float4 col[C];                                  // per token: log2 decay sum (hi, lo), 1/|k|, beta
  __shared__ float rq[C], sk[C], sq[C];
  __shared__ __align__(16) float on_w[C], beta_s[C];
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
  pdl_launch_dependents();  // the scan may set itself up
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

  const long sbase = ((long)b * p.seg_chunks + cl) * (p.hk * (long)key_bytes(DKP) + p.hv * (long)head_bytes(DKP));
  unsigned char* kimg = p.scratch + sbase + (long)hk * key_bytes(DKP);
  unsigned char* himg = p.scratch + sbase + p.hk * (long)key_bytes(DKP) + (long)hv * head_bytes(DKP);
  unsigned char *pimg = himg + 3 * SQ, *wimg = himg + 4 * SQ;
  float* sc = (float*)(wimg + 2 * w_bytes(DKP));
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
      col[t].w = beta_s[t] = bv;
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
            *(uint4*)(kimg + i * (2 * C * 128) + which * (C * 128) + img_off<64>(row, part)) = im;
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
    unsigned char* stage = (unsigned char*)(T + r0 * TS);  // where this warp's rows of T will be; the queries have been read
#pragma unroll
    for (int nt = 0; nt < 8; ++nt) {
      *(uint32_t*)(stage + img_off<C>(g, nt) + 4 * c) = h2(qk[nt][0] * down, qk[nt][1] * down);
      *(uint32_t*)(stage + img_off<C>(g + 8, nt) + 4 * c) = h2(qk[nt][2] * down, qk[nt][3] * down);
    }
    send(pimg + r0 * 128, stage, 2048);
    if (lane == 0) sc[2 * C + 8 + warp] = pow2(ep);
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
  if (t < C) {
    const float4 v = col[t];
    on_w[t] = exp2_fast(v.x + v.y) * v.z * v.w;
  }
  if (lane == 0) bulk_stores_read();  // T may take the place of P's rows
  __syncthreads();  // A is complete, the queries have been read
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

  // ---- 5: W = T diag(beta e^G / |k|) K for this warp's 16 rows, the left factor in three bf16 parts (K is bf16) ----
  {
    float w[DKP / 8][4];
#pragma unroll
    for (int nt = 0; nt < DKP / 8; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) w[nt][e] = 0.f;
    const uint32_t ks_s = smem_u32(kt);
#pragma unroll 1
    for (int ks = 0; ks <= warp; ++ks) {
      uint32_t ta[3][4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // rows g, g + 8 of columns 2 c, then of columns 2 c + 8
        const int row = r0 + g + 8 * (e & 1), j = 16 * ks + 2 * c + 8 * (e >> 1);
        const float2 x = *(const float2*)&T[row * TS + j], f = *(const float2*)&on_w[j];
        split3(x.x * f.x, x.y * f.y, ta[0][e], ta[1][e], ta[2][e]);
      }
#pragma unroll
      for (int n2 = 0; n2 < DKP / 16; ++n2) {
        uint32_t kb[4];
        ldsm4_t(ks_s + img_off<DKP>(16 * ks + (lane & 15), 2 * n2 + (lane >> 4)), kb);
#pragma unroll
        for (int part = 2; part >= 0; --part) {
          mma_bf16(w[2 * n2], ta[part], kb[0], kb[1]);
          mma_bf16(w[2 * n2 + 1], ta[part], kb[2], kb[3]);
        }
      }
    }
    float wm = 0.f;
#pragma unroll
    for (int nt = 0; nt < DKP / 8; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) wm = fmaxf(wm, fabsf(w[nt][e]));
    const int ew = scale_exp(warp_max_abs(wm));
    const float down = pow2(-ew);
    if (lane == 0) sc[2 * C + 4 + warp] = pow2(ew);
    // T diag(beta), this warp's 16 rows, eight columns per lane and pass
    const int j0 = (lane & 7) * 8;
    float bj[8];
    *(float4*)&bj[0] = *(const float4*)&beta_s[j0];
    *(float4*)&bj[4] = *(const float4*)&beta_s[j0 + 4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float* src = &T[(r0 + 4 * k + (lane >> 3)) * TS + j0];
      float tv[8];
      *(float4*)&tv[0] = *(const float4*)src;
      *(float4*)&tv[4] = *(const float4*)(src + 4);
      uint32_t part[3][4];
#pragma unroll
      for (int y = 0; y < 4; ++y) split3(tv[2 * y] * bj[2 * y], tv[2 * y + 1] * bj[2 * y + 1], part[0][y], part[1][y], part[2][y]);
#pragma unroll
      for (int i = 0; i < 3; ++i)
        *(uint4*)(himg + i * SQ + img_off<C>(r0 + 4 * k + (lane >> 3), lane & 7)) = make_uint4(part[i][0], part[i][1], part[i][2], part[i][3]);
    }
    __syncwarp();
    // W leaves through this warp's rows of A and then of T, 64 key dims each: 16 rows are 2 KB in a row of either half's image
#pragma unroll
    for (int x = 0; x < DKP / 64; ++x) {
      unsigned char* stage = (unsigned char*)((x ? T : A) + r0 * TS);
#pragma unroll
      for (int nt = 0; nt < 8; ++nt)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          uint32_t hi, lo;
          split2(w[8 * x + nt][2 * r] * down, w[8 * x + nt][2 * r + 1] * down, hi, lo);
          *(uint32_t*)(stage + img_off<64>(g + 8 * r, nt) + 4 * c) = hi;
          *(uint32_t*)(stage + 2048 + img_off<64>(g + 8 * r, nt) + 4 * c) = lo;
        }
      send(wimg + x * SQ + r0 * 128, stage, 2048);
      send(wimg + w_bytes(DKP) + x * SQ + r0 * 128, stage + 2048, 2048);
    }
  }
  if (t < C) {
    const float4 v = col[t], e = col[C - 1];
    const float eg = exp2_fast(v.x + v.y), on_v = exp2_fast((e.x - v.x) + (e.y - v.y)) * sk[t];
    sc[t] = on_v;
    sc[C + t] = eg * sq[t];
    if (t == C - 1) sc[2 * C] = eg;
    const float m = warp_max_abs(on_v);
    const unsigned counts = __ballot_sync(0xffffffffu, t < live && (!TREE || anc[t] != 0));
    if (lane == 0) sc[2 * C + 12 + warp] = m, sc[2 * C + 14 + warp] = __uint_as_float(counts);
  }
  if (lane == 0) bulk_stores_done();
  if (stays) pdl_wait();
}

// ---- a few tokens, one by one ---------------------------------------------------------------------------------------

// One or a few tokens per sequence: the recurrence itself in fp32. For one token it is bound by reading and writing the state
// once (16 sequences x 32 heads of 128 x 128: 67 MB in 17 us; 19 without the streaming hints, 21 with four CTAs per SM instead
// of five), then by its two reductions per token. A CTA owns 32 value columns of a head: lane = column, each of the eight
// warps holds 16 key rows of them in registers from the first token to the last; the two sums over the key rows go through
// shared memory.
constexpr int FEW = 24;  // most tokens
constexpr int FEW_THREADS = 256, FEW_ROWS = 16;

__global__ void __launch_bounds__(FEW_THREADS, 5) delta_few_kernel(const DeltaChunkParams p) {
  __shared__ __align__(16) float qn[FEW][128], kn[FEW][128];
  __shared__ float gate[FEW][2];
  __shared__ bf16 vs[FEW][32];
  __shared__ float red[2][8][32];
  const int vb = blockIdx.x, hv = blockIdx.y, b = blockIdx.z, hk = hv / (p.hv / p.hk);
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31, col = vb * 32 + lane;
  const bool cok = col < p.dv;
  const long sb = ((long)b * p.hv + hv) * p.dk * p.dv;
  float s[FEW_ROWS];
#pragma unroll
  for (int i = 0; i < FEW_ROWS; ++i) {
    const int k = warp * FEW_ROWS + i;
    s[i] = cok && k < p.dk ? __ldcs(&p.state[sb + (long)k * p.dv + col]) : 0.f;
  }
  const int len = p.lengths ? min(max(p.lengths[b], 0), p.tokens) : p.tokens;
  // queries by warps 0 .. 3, keys by warps 4 .. 7, every fourth token each
  const bool is_k = warp >= 4;
  for (int tok = warp & 3; tok < len; tok += 4) {
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
    *(float4*)&(is_k ? kn : qn)[tok][4 * lane] = make_float4(x[0] * r, x[1] * r, x[2] * r, x[3] * r);
    if (is_k && lane == 0) {
      gate[tok][0] = expf(p.g[((long)b * p.tokens + tok) * p.hv + hv]);
      gate[tok][1] = p.beta[((long)b * p.tokens + tok) * p.hv + hv];
    }
    if (!is_k) vs[tok][lane] = cok ? p.v[b * p.v_stride[0] + tok * p.v_stride[1] + hv * p.v_stride[2] + col] : f2bf(0.f);
  }
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
    const float d = (bf2f(vs[n][lane]) - r) * gate[n][1];
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
    if (cok && k < p.dk) __stcs(&p.state_out[sb + (long)k * p.dv + col], s[i]);
  }
  for (int n = len + warp; n < p.tokens; n += 8)
    if (cok) p.out[(((long)b * p.tokens + n) * p.hv + hv) * p.dv + col] = f2bf(0.f);
}

// Where this form is taken. us, token by token / chunked, 32 heads of 128 x 128: one sequence 4 tokens 4.5 / 19, 12 tokens 9 / 18,
// 24 tokens 13 / 18; two sequences 24 tokens 17 / 18; four 12 tokens 18 / 20, 16 tokens 23 / 20; 16 sequences 4 tokens 27 / 61, 12
// tokens 51 / 61, 16 tokens 68 / 61.
bool few_tokens(int batch, int tokens, int hv, int dv) {
  return tokens <= ((long)batch * hv * ((dv + 31) / 32) <= 2 * 148 ? FEW : 12);
}

int pad_dk(int dk) { return dk <= 64 ? 64 : 128; }
size_t chunk_bytes(int hk, int hv, int dk) { return (size_t)hk * key_bytes(pad_dk(dk)) + (size_t)hv * head_bytes(pad_dk(dk)); }

// How a prompt is walked through: in segments, each prepared by one kernel and scanned by the next. The scratch of a long prompt
// so stays bounded: 256 MB, or four chunks of every sequence (2.6 MB per chunk at 16 key and 32 value heads. One prompt of 8192
// tokens / six of 1001: 128 MB 402 / 179 us, 256 MB 390 / 161, 512 MB 404 / 160: fewer starts against a longer first wait).
// Where the scan leaves most SMs idle (one CTA per head and sequence), the preparation of a segment runs beside the scan of the
// one before, out of the other half of the scratch; only the first, short one is waited for. us, beside / one after the other,
// 4096 tokens: 64 heads 291 / 334, 96 heads 393 / 412, 128 heads 516 / 509.
struct Walk {
  int first, chunks;  // chunks of the first segment, and of the others at most
  bool beside;
};
Walk plan_walk(int batch, int tokens, int hk, int hv, int dk, int dv) {
  Walk w;
  const int chunks = (tokens + C - 1) / C;
  const long fit = (long)((size_t)256 * 1024 * 1024 / (chunk_bytes(hk, hv, dk) * batch));
  const long heads = (long)batch * hv, wave = 4 * 148 / heads;  // chunks whose preparation fills the SMs once
  w.beside = heads * ((dv + 127) / 128) <= 100 && chunks > wave;
  long seg = w.beside ? fit / 2 : fit;
  if (seg < 4) seg = 4;
  w.first = (int)(w.beside ? (wave < 4 ? 4 : wave < seg ? wave : seg) : (chunks < seg ? chunks : seg));
  const int rest = chunks - w.first;
  const int parts = rest > 0 ? (int)((rest + seg - 1) / seg) : 1;
  w.chunks = rest > 0 ? (rest + parts - 1) / parts : w.first;
  return w;
}

// keys, then T (or the queries, which need less), then A
template <int DKP> constexpr int prep_smem() { return C * DKP * 2 + 2 * C * TS * 4; }

template <int DKP, bool TREE>
int configure() {
  return cudaFuncSetAttribute(delta_prep_kernel<DKP, TREE>, cudaFuncAttributeMaxDynamicSharedMemorySize, prep_smem<DKP>()) == cudaSuccess
             ? 0
             : check_launch("delta rule preparation: shared-memory opt-in");
}
int configure_all() {
  int rc = configure<64, false>();
  if (!rc) rc = configure<64, true>();
  if (!rc) rc = configure<128, false>();
  if (!rc) rc = configure<128, true>();
  return rc;
}

template <int DKP, bool TREE>
int launch_prep(const DeltaChunkParams& p, cudaStream_t stream) {
  const dim3 grid(p.chunks, p.hv, p.batch);
  if (p.beside) (void)launch_pdl(delta_prep_kernel<DKP, TREE>, grid, dim3(PREP_THREADS), prep_smem<DKP>(), stream, p);
  else delta_prep_kernel<DKP, TREE><<<grid, PREP_THREADS, prep_smem<DKP>(), stream>>>(p);
  return check_launch("delta rule preparation");
}

}  // namespace

size_t delta_chunk_scratch_bytes(int batch, int tokens, int hk, int hv, int dk, int dv, bool tree) {
  if (!tree && few_tokens(batch, tokens, hv, dv)) return 0;
  const Walk w = plan_walk(batch, tokens, hk, hv, dk, dv);
  return chunk_bytes(hk, hv, dk) * batch * (w.first > w.chunks ? w.first : w.chunks) * (w.beside ? 2 : 1);
}

int launch_delta_chunk(const DeltaChunkParams& args, cudaStream_t stream) {
  static OncePerDevice once;
  int rc = once.run(configure_all);
  if (rc) return rc;
  DeltaChunkParams p = args;
  const bool tree = p.parents != nullptr, wide = p.dk > 64;
  if (!tree && few_tokens(p.batch, p.tokens, p.hv, p.dv)) {
    delta_few_kernel<<<dim3((p.dv + 31) / 32, p.hv, p.batch), FEW_THREADS, 0, stream>>>(p);
    return check_launch("delta rule, few tokens");
  }
  const Walk w = plan_walk(p.batch, p.tokens, p.hk, p.hv, p.dk, p.dv);
  const int chunks = (p.tokens + C - 1) / C;
  p.seg_chunks = w.first > w.chunks ? w.first : w.chunks;
  const size_t half = chunk_bytes(p.hk, p.hv, p.dk) * p.batch * p.seg_chunks;
  for (int at = 0, i = 0; at < chunks; at += p.chunks, ++i) {
    const int most = i == 0 ? w.first : w.chunks;
    p.chunk0 = at;
    p.chunks = chunks - at < most ? chunks - at : most;
    p.first = i == 0;
    p.beside = w.beside && i > 0;
    p.scratch = args.scratch + (w.beside && (i & 1) ? half : 0);
    if (tree) rc = wide ? launch_prep<128, true>(p, stream) : launch_prep<64, true>(p, stream);
    else rc = wide ? launch_prep<128, false>(p, stream) : launch_prep<64, false>(p, stream);
    if (!rc) rc = launch_delta_scan(p, stream);
    if (rc) return rc;
  }
  return 0;
}

}  // namespace dfb
