// Attention of a tree of drafted tokens over the KV cache, sm_100a.
//
// Node i of sequence b sees the cache rows 0 .. len_b - 1 (the accepted prefix), the rows len_b + j of its ancestors j, and its
// own row len_b + i; o = softmax(scale q K^T) V over those rows. It is the many-token form of the split-KV decode
// attention (src/deltaforge/kernels/flash_decode_splitkv.py:177-256). With one node it is the decode attention itself; with a
// chain of nodes it is causal attention of the new tokens.
//
// One pass over the keys with a running maximum and sum. The query heads of one KV head and all nodes form the rows of
// m16n8k16 tiles (row = node * group + head), so K and V are read once per 16 * MT rows. A CTA takes a range of key tiles
// (a split) of one (sequence, KV head, row tile); its eight warps are 8 / MT groups of MT warps: a group owns every
// (8 / MT)-th tile of the range, each of its warps 16 rows. Groups keep rings of their own, filled by cp.async: no barrier
// across groups, no wait that could spin, rows past the end filled with zeros by the copy itself (so that what a cache
// holds behind its last row, NaN included, never meets a zero probability).
//
// Tree: bit j of anc[i] says that j is i or an ancestor of i, built from the parents by doubling (six rounds for 64 nodes).
// Only tiles at or past row len_b look at it. A masked node's value row may hold NaN or infinity, and 0 * NaN in
// P V would reach every row: values of tree rows that are not finite are zeroed in shared memory and added back, row by
// row, for the nodes that do see them (no cost when there are none but the look itself).
//
// Rounding: q, k, v as they are; scores, maximum, sum and accumulators in fp32; probabilities are rounded to the cache's
// type for the second product (relative 2^-9 each in bf16, of random sign), the sum takes them unrounded. fp16 has five bits of
// exponent: relative to the largest of a row, probabilities below 2^-14 would lose bits there and those below 2^-25 vanish, and
// behind one dominant key (an attention sink) they are the output. So for fp16 the reference of the exponentials lies 2^15 below
// the maximum; sums and accumulators refer to it alike, and the factor goes out in the division. 17 e-folds below the
// dominant key the output was off by 7 %.
//
// A row without a node (parent below -1 or not before the node) gets zeros, and so does one that sees no key: without a
// prefix, of a tree that reaches past the cache. Splits leave (m, l, acc) in scratch and
// tree_merge_kernel adds them in split order: results do not depend on which CTA ends first.
#include "common.cuh"
#include "kernels.h"

namespace dfb {

namespace {

constexpr int TA_WARPS = 8;
constexpr int TA_THREADS = TA_WARPS * 32;
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// 16 bytes global -> shared; bytes == 0 writes zeros and reads nothing
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <typename T> __device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16<bf16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
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
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<bf16>(float a, float b) {
  __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *(uint32_t*)&v;
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  __half2 v = __floats2half2_rn(a, b);
  return *(uint32_t*)&v;
}
template <typename T> __device__ __forceinline__ float elem_f(T v);
template <> __device__ __forceinline__ float elem_f(bf16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float elem_f(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ uint16_t exp_mask() { return 0x7f80; }  // all ones: infinity or NaN
template <> __device__ __forceinline__ uint16_t exp_mask<__half>() { return 0x7c00; }

// How far the reference of the exponentials lies below the maximum, in powers of two: probabilities are at most 2^this. The
// subtraction rounds upwards, which keeps that true for scores of any size.
template <typename T> __device__ __forceinline__ float headroom() { return 0.f; }
template <> __device__ __forceinline__ float headroom<__half>() { return 15.f; }

// One row of a tile is D elements; its 16-byte chunks are permuted within 128-byte lines so that the eight rows an 8x8
// matrix load touches lie in different banks.
template <int D> __device__ __forceinline__ uint32_t tile_off(int row, int chunk) {
  const int x = D >= 64 ? (chunk ^ (row & 7)) : (chunk ^ ((row >> 1) & 3));
  return (uint32_t)(row * D * 2 + x * 16);
}

// 2^x for x <= 0 (and NaN, -inf): one instruction, 2 ulp; the argument is exact to fp32
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int D, int MT> struct Shape {
  // keys per tile: 16 KB of keys and values together where the head is 256 or 128 wide, less for narrow heads, whose
  // scores would not fit the registers
  static constexpr int TK = D == 256 ? 16 : 32;
  static constexpr int BYTES = 2 * TK * D * 2;
  // the groups' rings beside each other in 224 KB, six stages at most
  static constexpr int FIT = 224 * 1024 / ((TA_WARPS / MT) * BYTES);
  static constexpr int STAGES = FIT > 6 ? 6 : FIT;
  static constexpr int RING = (TA_WARPS / MT) * STAGES * BYTES, MERGE = TA_WARPS * 16 * D * 4;
  static constexpr int SMEM = RING > MERGE ? RING : MERGE;
};

template <typename T, int D, int MT>
__global__ void __launch_bounds__(TA_THREADS, 1) tree_attention_kernel(const TreeAttnParams p) {
  constexpr int TK = Shape<D, MT>::TK, TILEB = Shape<D, MT>::BYTES, KG = TA_WARPS / MT, STAGES = Shape<D, MT>::STAGES;
  constexpr int CH = D / 8;  // 16-byte chunks per row
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ unsigned long long anc[MAX_TREE_NODES];
  __shared__ int up[MAX_TREE_NODES];
  __shared__ float ml_s[TA_WARPS][16][2];

  const int split = blockIdx.x, b = blockIdx.z;
  const int row_tiles = (p.rows + 16 * MT - 1) / (16 * MT);
  const int hk = blockIdx.y / row_tiles, rt = blockIdx.y % row_tiles;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31, g = lane >> 2, c = lane & 3;
  const int group = warp / MT, gt = t - group * MT * 32;  // group of warps, thread within it

  pdl_launch_dependents();  // the merge may set itself up; it waits for this grid's end before it reads

  // ---- which rows of the cache this CTA scans ----
  const int cached = min(max(p.cache_len[b], 0), p.max_seq);
  const int L = (int)min((long)cached + p.nodes, (long)p.max_seq);
  const int ntiles = (L + TK - 1) / TK, per = (ntiles + p.splits - 1) / p.splits;
  const int tile0 = split * per, tile1 = min(ntiles, tile0 + per);
  const int first_tree_tile = cached / TK;

  // ---- ancestors ----
  if (tile1 > first_tree_tile && tile1 > tile0) {
    if (t < p.nodes) {
      const int pa = p.parents[(long)b * p.parents_stride + t];
      const bool node = pa >= -1 && pa < t;
      anc[t] = node ? 1ull << t : 0ull;
      up[t] = node ? pa : -1;
    }
    __syncthreads();
    for (int step = 1; step < p.nodes; step *= 2) {  // bits of up to 2 * step ancestors
      unsigned long long bits = 0;
      int u = -1;
      if (t < p.nodes) {
        bits = anc[t], u = up[t];
        if (u >= 0) bits |= anc[u], u = up[u];
      }
      __syncthreads();
      if (t < p.nodes) anc[t] = bits, up[t] = u;
      __syncthreads();
    }
  }

  // ---- query rows of this warp: fragments in registers ----
  const int m0 = (rt * MT + warp % MT) * 16;  // first row of the warp
  const T* kbase = (const T*)p.kcache + b * p.k_stride[0] + hk * p.k_stride[1];
  const T* vbase = (const T*)p.vcache + b * p.v_stride[0] + hk * p.v_stride[1];
  uint32_t qa[D / 16][4];
  int node_of[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = m0 + g + 8 * r;
    const bool ok = row < p.rows;
    node_of[r] = ok ? row / p.group : 0;
    const T* q = (const T*)p.q + b * p.q_stride[0] + node_of[r] * p.q_stride[1] + (hk * p.group + (ok ? row % p.group : 0)) * p.q_stride[2];
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      qa[ks][r] = ok ? *(const uint32_t*)(q + 16 * ks + 2 * c) : 0u;
      qa[ks][2 + r] = ok ? *(const uint32_t*)(q + 16 * ks + 8 + 2 * c) : 0u;
    }
  }

  unsigned char* ring = smem + (size_t)group * STAGES * TILEB;
  // i-th tile of this group, keys (half 0) or values (half 1), into its slot of the ring
  auto load_half = [&](int i, int half) {
    const int tile = tile0 + group + i * KG;
    if (tile >= tile1) return;
    const uint32_t dst = smem_u32(ring + (i % STAGES) * TILEB) + half * (TILEB / 2);
    const T* base = half ? vbase : kbase;
    const long stride = half ? p.v_stride[2] : p.k_stride[2];
    const int key0 = tile * TK;
#pragma unroll
    for (int x = gt; x < TK * CH; x += MT * 32) {
      const int r = x / CH, ch = x % CH, key = key0 + r;
      cp_async16(dst + tile_off<D>(r, ch), base + (key < L ? key : 0) * stride + ch * 8, key < L ? 16 : 0);
    }
  };
  auto group_sync = [&]() {
    if (MT == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(MT * 32) : "memory");
  };

  float o[D / 8][4];
#pragma unroll
  for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  float mrun[2] = {-INFINITY, -INFINITY}, lrun[2] = {0.f, 0.f};
  const float sl = p.scale * LOG2E;  // scores are kept in units of log 2

  // MT == 1: a warp has its ring to itself. It refills the key slot as soon as the scores are done and the value slot after
  // the second product, so half a tile is always on its way even with one stage. MT > 1: keys and values of a stage
  // travel together, and one barrier of the group per tile covers both "has landed" and "may be refilled".
#pragma unroll
  for (int i = 0; i < (MT == 1 ? STAGES : STAGES - 1); ++i) {
    load_half(i, 0);
    if (MT == 1) cp_async_commit();
    load_half(i, 1);
    cp_async_commit();
  }
  for (int i = 0; tile0 + group + i * KG < tile1; ++i) {
    if (MT == 1) {
      cp_async_wait<2 * STAGES - 1>();
      __syncwarp();
    } else {
      cp_async_wait<(MT == 1 ? 0 : STAGES - 2)>();
      group_sync();  // tile i has landed for every warp of the group, and tile i - 1 has been read by all of them
      load_half(i + STAGES - 1, 0);
      load_half(i + STAGES - 1, 1);
      cp_async_commit();
    }
    const int tile = tile0 + group + i * KG, key0 = tile * TK;
    unsigned char* st = ring + (i % STAGES) * TILEB;
    const uint32_t ks_s = smem_u32(st), vs_s = ks_s + TK * D * 2;

    float s[TK / 8][4];
#pragma unroll
    for (int nt = 0; nt < TK / 8; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
#pragma unroll
      for (int n2 = 0; n2 < TK / 16; ++n2) {
        uint32_t kb[4];  // keys 16 n2 + 0..7 (dims +0..7, +8..15), then keys + 8
        ldsm4(ks_s + tile_off<D>(16 * n2 + (lane & 7) + 8 * (lane >> 4), 2 * ks + ((lane >> 3) & 1)), kb);
        mma16<T>(s[2 * n2], qa[ks], kb[0], kb[1]);
        mma16<T>(s[2 * n2 + 1], qa[ks], kb[2], kb[3]);
      }
    }
    if (MT == 1) {
      __syncwarp();
      load_half(i + STAGES, 0);
      cp_async_commit();
      cp_async_wait<2 * STAGES - 1>();  // the values of tile i
      __syncwarp();
    }
    // scores in units of log 2; keys past the end and nodes that are no ancestors are taken out
    const bool tree = key0 + TK > cached;
#pragma unroll
    for (int nt = 0; nt < TK / 8; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[nt][e] *= sl;
    if (tree) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const unsigned long long bits = anc[node_of[r]];
#pragma unroll
        for (int nt = 0; nt < TK / 8; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int j = key0 + nt * 8 + 2 * c + e - cached;  // node number, negative in the prefix
            const bool seen = j < 0 || (j < MAX_TREE_NODES && j + cached < L && ((bits >> j) & 1));
            if (!seen) s[nt][2 * r + e] = -INFINITY;
          }
      }
    }
    // values of tree rows that are not finite: zeroed here, added back below for the rows that see them
    bool odd = false;  // there are such values in this tile
    if (tree) {
      bool mine = false;
      for (int x = gt; x < TK * CH; x += MT * 32) {
        const int r = x / CH, ch = x % CH, key = key0 + r;
        if (key < cached || key >= L) continue;
        const uint16_t* e = (const uint16_t*)(st + TK * D * 2 + tile_off<D>(r, ch));
#pragma unroll
        for (int y = 0; y < 8; ++y) mine |= (e[y] & exp_mask<T>()) == exp_mask<T>();
      }
      int any = __any_sync(0xffffffffu, mine);
      if (MT > 1) {
        asm volatile(
            "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
            : "=r"(any)
            : "r"(any), "r"(1 + group), "n"(MT * 32)
            : "memory");
      }
      if (any) {
        for (int x = gt; x < TK * CH; x += MT * 32) {
          const int r = x / CH, ch = x % CH, key = key0 + r;
          if (key < cached || key >= L) continue;
          uint16_t* e = (uint16_t*)(st + TK * D * 2 + tile_off<D>(r, ch));
#pragma unroll
          for (int y = 0; y < 8; ++y)
            if ((e[y] & exp_mask<T>()) == exp_mask<T>()) e[y] = 0;
        }
        group_sync();
        odd = true;
      }
    }
    // running maximum and sum of rows g and g + 8
    float corr[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float mx = -INFINITY;
#pragma unroll
      for (int nt = 0; nt < TK / 8; ++nt) mx = fmaxf(mx, fmaxf(s[nt][2 * r], s[nt][2 * r + 1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float mn = fmaxf(mrun[r], __fadd_ru(mx, -headroom<T>()));
      const float ref = mn == -INFINITY ? 0.f : mn;  // nothing seen yet: every probability is 2^-inf = 0
      corr[r] = exp2_fast(mrun[r] - ref);
      float sum = 0.f;
#pragma unroll
      for (int nt = 0; nt < TK / 8; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float pr = exp2_fast(s[nt][2 * r + e] - ref);
          s[nt][2 * r + e] = pr;
          sum += pr;
        }
      lrun[r] = lrun[r] * corr[r] + sum;
      mrun[r] = mn;
    }
    if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
      for (int j = 0; j < D / 8; ++j) {
        o[j][0] *= corr[0], o[j][1] *= corr[0];
        o[j][2] *= corr[1], o[j][3] *= corr[1];
      }
    }
#pragma unroll
    for (int k2 = 0; k2 < TK / 16; ++k2) {
      uint32_t pa[4];
      pa[0] = pack2<T>(s[2 * k2][0], s[2 * k2][1]);
      pa[1] = pack2<T>(s[2 * k2][2], s[2 * k2][3]);
      pa[2] = pack2<T>(s[2 * k2 + 1][0], s[2 * k2 + 1][1]);
      pa[3] = pack2<T>(s[2 * k2 + 1][2], s[2 * k2 + 1][3]);
#pragma unroll
      for (int j2 = 0; j2 < D / 16; ++j2) {
        uint32_t vb[4];
        ldsm4_t(vs_s + tile_off<D>(16 * k2 + (lane & 15), 2 * j2 + (lane >> 4)), vb);
        mma16<T>(o[2 * j2], pa, vb[0], vb[1]);
        mma16<T>(o[2 * j2 + 1], pa, vb[2], vb[3]);
      }
    }
    if (MT == 1) {
      __syncwarp();
      load_half(i + STAGES, 1);
      cp_async_commit();
    }
    if (odd) {  // p * v for the values that were zeroed, from global memory, for the rows that see them
#pragma unroll 1
      for (int r = 0; r < TK; ++r) {
        const int j = key0 + r - cached;
        if (j < 0 || j + cached >= L) continue;
        const T* v = vbase + (long)(key0 + r) * p.v_stride[2];
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
          if (!((anc[node_of[rr]] >> j) & 1)) continue;
          // the probability of this key sits in another lane of the quad; what it multiplies is infinite or NaN, so its sign
          // (never negative) and whether it is zero is all that matters
#pragma unroll
          for (int jj = 0; jj < D / 8; ++jj)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float x = elem_f<T>(v[8 * jj + 2 * c + e]);
              if (!isfinite(x)) o[jj][2 * rr + e] += x;
            }
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    lrun[r] += __shfl_xor_sync(0xffffffffu, lrun[r], 1);
    lrun[r] += __shfl_xor_sync(0xffffffffu, lrun[r], 2);
  }
  cp_async_wait<0>();
  __syncthreads();  // all tiles have been read: the rings become the buffer in which the groups' results meet

  // ---- merge of the groups: acc[group][row][D], rows of the CTA 0 .. 16 MT - 1 ----
  constexpr int ROWS = 16 * MT;
  float* acc = (float*)smem;
  if (KG > 1) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = (warp % MT) * 16 + g + 8 * r;
      float* a = acc + ((size_t)group * ROWS + row) * D;
#pragma unroll
      for (int j = 0; j < D / 8; ++j) {
        const int at = 8 * (j ^ (g & 3)) + 2 * c;  // blocks of eight permuted by row: conflict-free writes
        *(float2*)(a + at) = make_float2(o[j][2 * r], o[j][2 * r + 1]);
      }
      if (c == 0) ml_s[warp][g + 8 * r][0] = mrun[r], ml_s[warp][g + 8 * r][1] = lrun[r];
    }
    __syncthreads();
  }
  const long pbase = (((long)b * p.hkv + hk) * p.splits + split) * p.rows;
  constexpr int PAIRS = D / 2;
  for (int x = t; x < ROWS * PAIRS; x += TA_THREADS) {
    const int row = x / PAIRS, d2 = (x % PAIRS) * 2;
    const int gr = rt * ROWS + row;
    if (gr >= p.rows) break;
    const int mt = row >> 4, r16 = row & 15;
    float m = -INFINITY, l = 0.f;
    float2 a = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < KG; ++k) m = fmaxf(m, ml_s[k * MT + mt][r16][0]);
    const float ref = m == -INFINITY ? 0.f : m;
    const int at = ((d2 >> 3) ^ (r16 & 3)) * 8 + (d2 & 7);
#pragma unroll
    for (int k = 0; k < KG; ++k) {
      const float w = exp2_fast(ml_s[k * MT + mt][r16][0] - ref);
      const float2 v = *(const float2*)(acc + ((size_t)k * ROWS + row) * D + at);
      l = fmaf(ml_s[k * MT + mt][r16][1], w, l);
      a.x = fmaf(v.x, w, a.x), a.y = fmaf(v.y, w, a.y);
    }
    if (p.splits == 1) {
      const int node = gr / p.group;
      const int pa = p.parents[(long)b * p.parents_stride + node];
      const bool ok = pa >= -1 && pa < node;
      const float inv = l == 0.f ? 0.f : 1.f / l;  // 0: nothing seen
      T* out = (T*)p.out + (((long)b * p.nodes + node) * p.hq + hk * p.group + gr % p.group) * D + d2;
      *(uint32_t*)out = ok ? pack2<T>(a.x * inv, a.y * inv) : 0u;
    } else {
      *(float2*)(p.part_acc + (pbase + gr) * D + d2) = a;
      if (d2 == 0) *(float2*)(p.part_ml + (pbase + gr) * 2) = make_float2(m, l);
    }
  }
}

// One CTA per output row: D / 4 lanes of four dims each, times as many groups as 256 threads hold; group i adds splits i, i +
// GROUPS, .. in order, then the groups' sums are added in order. All loads of a thread are independent of one another.
template <typename T, int D>
__global__ void __launch_bounds__(256) tree_merge_kernel(const TreeAttnParams p) {
  constexpr int LANES = D / 4, GROUPS = 256 / LANES;
  __shared__ float4 part[GROUPS][LANES];
  __shared__ float part_l[GROUPS], top[8];
  const int t = threadIdx.x, li = t % LANES, gi = t / LANES;
  const long r = blockIdx.x;
  const int row = (int)(r % p.rows);
  const long bh = r / p.rows;
  const int hk = (int)(bh % p.hkv), b = (int)(bh / p.hkv), node = row / p.group;
  const int pa = p.parents[(long)b * p.parents_stride + node];
  const bool ok = pa >= -1 && pa < node;
  pdl_wait();
  const float2* ml = (const float2*)p.part_ml + bh * p.splits * p.rows + row;
  const float* acc = p.part_acc + (bh * p.splits * p.rows + row) * D + 4 * li;
  float m = t < p.splits ? __ldcg(ml + (long)t * p.rows).x : -INFINITY;  // at most 128 splits
  m = warp_max(m);
  if ((t & 31) == 0) top[t >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) m = fmaxf(m, top[w]);
  const float ref = m == -INFINITY ? 0.f : m;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
#pragma unroll 8
  for (int s = gi; s < p.splits; s += GROUPS) {
    const float2 v = __ldcg(ml + (long)s * p.rows);
    const float4 y = __ldcg((const float4*)(acc + (long)s * p.rows * D));
    const float w = exp2_fast(v.x - ref);
    l = fmaf(v.y, w, l);
    a.x = fmaf(y.x, w, a.x), a.y = fmaf(y.y, w, a.y), a.z = fmaf(y.z, w, a.z), a.w = fmaf(y.w, w, a.w);
  }
  part[gi][li] = a;
  if (li == 0) part_l[gi] = l;
  __syncthreads();
  if (gi) return;
#pragma unroll
  for (int i = 1; i < GROUPS; ++i) {
    const float4 y = part[i][li];
    a.x += y.x, a.y += y.y, a.z += y.z, a.w += y.w;
    l += part_l[i];
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;  // 0: nothing seen
  T* out = (T*)p.out + (((long)b * p.nodes + node) * p.hq + hk * p.group + row % p.group) * D + 4 * li;
  uint2 v = make_uint2(pack2<T>(a.x * inv, a.y * inv), pack2<T>(a.z * inv, a.w * inv));
  if (!ok) v = make_uint2(0u, 0u);
  *(uint2*)out = v;
}

template <typename T, int D, int MT>
int configure_one() {
  return cudaFuncSetAttribute(tree_attention_kernel<T, D, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<D, MT>::SMEM) == cudaSuccess
             ? 0
             : check_launch("tree attention: shared-memory opt-in");
}
template <typename T, int D>
int configure_mt() {
  int rc = configure_one<T, D, 1>();
  if (!rc) rc = configure_one<T, D, 2>();
  if (!rc) rc = configure_one<T, D, 4>();
  return rc;
}
template <typename T>
int configure_d() {
  int rc = configure_mt<T, 32>();
  if (!rc) rc = configure_mt<T, 64>();
  if (!rc) rc = configure_mt<T, 128>();
  if (!rc) rc = configure_mt<T, 256>();
  return rc;
}
int configure_all() {
  const int rc = configure_d<bf16>();
  return rc ? rc : configure_d<__half>();
}

template <typename T, int D>
int launch_d(const TreeAttnParams& p, cudaStream_t stream) {
  const int rows_cta = 16 * p.mt;
  const dim3 grid(p.splits, p.hkv * ((p.rows + rows_cta - 1) / rows_cta), p.batch);
  if (p.mt == 1) tree_attention_kernel<T, D, 1><<<grid, TA_THREADS, Shape<D, 1>::SMEM, stream>>>(p);
  else if (p.mt == 2) tree_attention_kernel<T, D, 2><<<grid, TA_THREADS, Shape<D, 2>::SMEM, stream>>>(p);
  else tree_attention_kernel<T, D, 4><<<grid, TA_THREADS, Shape<D, 4>::SMEM, stream>>>(p);
  int rc = check_launch("tree attention");
  if (rc || p.splits == 1) return rc;
  const long rows = (long)p.batch * p.hkv * p.rows;
  if (launch_pdl(tree_merge_kernel<T, D>, dim3((unsigned)rows), dim3(256), 0, stream, p) != cudaSuccess)
    return check_launch("tree attention: merge");
  return check_launch("tree attention: merge");
}

template <typename T>
int launch_t(const TreeAttnParams& p, cudaStream_t stream) {
  switch (p.d) {
    case 32: return launch_d<T, 32>(p, stream);
    case 64: return launch_d<T, 64>(p, stream);
    case 128: return launch_d<T, 128>(p, stream);
    default: return launch_d<T, 256>(p, stream);
  }
}

}  // namespace

TreePlan tree_plan(int batch, int nodes, int hq, int hkv, int d, int max_seq, bool tc_ok) {
  TreePlan pl = {};
  const int rows = nodes * (hq / hkv);
  // Which form (us, mma.sync / tcgen05; sequences x cache rows, 4 KV heads of 256 dims or 8 of 128): the products on tcgen05 are
  // faster and read the cache once for up to 128 rows, but its pipeline takes 4 us more to fill and to merge.
  // Many heads fill the SMs either way: 8 x 4096, 16 rows 37 / 31, 32 rows 41 / 32 (256 dims), 47 / 31 (128 dims); 8 x 512, 32 rows
  // 15 / 14 and 13 / 14; only at 16 rows and long caches (8 x 32768: 165 / 169) does the other stay ahead.
  // Few heads: one pass over 32 rows is enough for mma.sync, 1 x 32768: 34 / 42 and 31 / 38; 48 rows 52 / 43 and 43 / 38; unless
  // there is little to do at all: 1 x 4096, 48 rows 18 / 17 and 14 / 20, 128 rows 24 / 22 and 19 / 23.
  const long units = (long)batch * hkv;
  if (tc_ok && d >= 64 && (units >= 32 ? rows > 16 : rows > 32 && (double)units * max_seq * rows * d > 5e8)) {
    const long row_tiles = (rows + 127) / 128, tiles = units * ((max_seq + 127) / 128);
    const long most = row_tiles < 148 ? 148 / row_tiles : 1, groups = (tiles + TREE_TC_MIN_TILES - 1) / TREE_TC_MIN_TILES;
    pl.tc_groups = (int)(groups < most ? groups : most);
    pl.slots = (size_t)(pl.tc_groups + units) * row_tiles * 128;
    return pl;
  }
  pl.mt = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  const long base = (long)batch * hkv * ((rows + 16 * pl.mt - 1) / (16 * pl.mt));
  // Splits: enough CTAs for the 148 SMs, as full a last wave as can be had, and no split of fewer than 64 keys of the
  // cache's capacity (the live length is known on the device alone).
  const int most = max_seq / 64 < 1 ? 1 : max_seq / 64 > 128 ? 128 : max_seq / 64;
  pl.splits = 1;
  double best_cost = 1e30;
  for (int s = 1; s <= most; ++s) {
    const double waves = (double)((base * s + 147) / 148);
    const double cost = waves / s * (1.0 + 0.02 * s * waves / (waves + 8.0)) + 0.0005 * s;
    if (cost < best_cost * 0.999) best_cost = cost, pl.splits = s;
    if (base * s > 148 * 8) break;
  }
  pl.slots = pl.splits > 1 ? (size_t)batch * hkv * rows * pl.splits : 0;
  return pl;
}

int launch_tree_attention(const TreeAttnParams& p, cudaStream_t stream) {
  if (p.tc_groups) return launch_tree_attention_tc(p, stream);
  static OncePerDevice once;
  const int rc = once.run(configure_all);
  if (rc) return rc;
  return p.is_fp16 ? launch_t<__half>(p, stream) : launch_t<bf16>(p, stream);
}

}  // namespace dfb
