// Attention of a tree of drafted tokens over the KV cache on tcgen05 (sm_100a), for many heads or more than a few query rows.
//
// Same contract as tree_attention.cu, which serves the others (tree_plan there has the rule). There the 16-row tiles of mma.sync read a key once per 64
// rows and reach a quarter of the tensor rate; 64 nodes with 4 query heads per KV head (256 rows) were bound by that.
// Here 128 rows (node * group + head) are the M of tcgen05.mma: S = Q K^T into TMEM, P = 2^(S - m) back into TMEM as the A
// operand of O += P V, O in TMEM as well (S and its successor 128 columns each, O one column per dim: 512 at head dim 256).
//
// Work: the (sequence, KV head) units are laid out one behind the other in tiles of 128 keys, as many as each sequence
// really has, and every group of CTAs takes an equal stretch of that line, whatever units it crosses (the lengths are on the
// device; a grid planned on the host from the cache's capacity waits for its longest sequence); cut_line has the
// exception. The CTAs of a group are the row tiles: they walk through the same keys side by side, so that the second
// reads them from the L2 (row tiles as units of their own read 1.80 GB instead of 0.9 at 8 sequences x 32K rows). A unit that
// one group covers is finished there; of the others every CTA leaves (m, l, acc) in a slot of its own, and
// tree_tc_merge_kernel adds them in order.
//
// Roles: warp 0 loads (TMA boxes 64 dims wide, 128-byte swizzle; a ring of K and V pieces), warp 1 issues the products, warps
// 2 and 3 look after values that must not meet a zero probability, warps 4-11 have two threads per row, half of a tile's
// keys each: scores out of TMEM, masks, maximum, exponentials, P into the columns of S. The product of tile i + 1 runs under
// the softmax of tile i. The maximum that P refers to is moved only when a row's true maximum is more than 2^8 (fp16: 2^4) above
// it, so that O rarely has to be rescaled; sums stay exact because l refers to the same maximum.
//
// Bounds per tile of 128 keys at head dim 256: 1024 cycles of ex2, 128 KB of K and V from the L2, and of tensor time 16 products
// Q K^T with both operands in shared memory (104 cycles each, measured, where the arithmetic takes 64) and 8 products P V with
// P in TMEM and N = 256 (138): 2770 cycles, 161 of the 188 us that 8 sequences x 64 nodes x 32K rows take. (Q in TMEM would take
// 74 cycles, but O, two S and Q are 640 columns; with tiles of 64 keys it was slower.) Run back to back for seconds, that case
// draws 1000 W, the clock falls from 1965 to 1380 MHz and the call takes 215 to 240 us.
//
// Every wait is bounded; one that runs out makes the CTA leave NaN, wait (again with a limit) for its own copies and products, and
// return.
#include <cuda.h>

#include "common.cuh"
#include "kernels.h"
#include "tcgen05.cuh"

namespace dfb {

namespace {

constexpr int TM = 128;          // query rows per tile
constexpr int TN = 128;          // keys per tile
constexpr int TC_WARPS = 12, TC_THREADS = TC_WARPS * 32;
constexpr float LOG2E = 1.4426950408889634f;

// In powers of two: how far the reference of the exponentials lies below the maximum it was taken from, and by how much the
// maximum may grow before O is rescaled. Probabilities are at most 2^(HEADROOM + LAZY): for fp16, 2^15, so that its five bits of
// exponent begin at 2^-25 of the largest and not at 2^-14 (see tree_attention.cu). Roundings go the way that keeps this true for
// scores of any size.
template <typename T> struct Range { static constexpr float HEADROOM = 0.f, LAZY = 8.f; };
template <> struct Range<__half> { static constexpr float HEADROOM = 11.f, LAZY = 4.f; };

template <int D> struct Tc {
  static constexpr int BLOCKS = D / 64;                          // 64-dim blocks of a row
  static constexpr int Q_BYTES = BLOCKS * TM * 128;
  // A K or V tile comes in one or two pieces of at most 32 KB, one slot of the ring each: K cut along the dims (the first
  // product contracts over them), V along the keys, so that every product has the widest N there is.
  static constexpr int PIECES = D == 256 ? 2 : 1;
  static constexpr int K_BLOCKS = BLOCKS / PIECES, V_KEYS = TN / PIECES;
  static constexpr int PIECE = K_BLOCKS * TN * 128;
  static constexpr int RING = D == 256 ? 5 : 6;
  static constexpr int SMEM = Q_BYTES + RING * PIECE + 1024;
  static_assert(RING * PIECE >= 40960 + 3 * TM * 4, "the ring serves as the result's staging buffer");
  // TMEM columns: O, one per dim; two S of 128, each with its P (two values per column) over its first half
  static constexpr int O_COL = 0, S_COL = 256;
};

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
template <typename T> __device__ __forceinline__ uint32_t exp_mask() { return 0x7f80; }  // all ones: infinity or NaN
template <> __device__ __forceinline__ uint32_t exp_mask<__half>() { return 0x7c00; }
__device__ __forceinline__ int live_rows(const TreeAttnParams& p, int b) {
  return (int)min((long)min(max(p.cache_len[b], 0), p.max_seq) + p.nodes, (long)p.max_seq);
}
__device__ __forceinline__ int live_tiles(const TreeAttnParams& p, int b) { return (live_rows(p, b) + TN - 1) / TN; }
// How the line of tiles is cut, found by one warp (the same in the kernel and in the merge).
struct Cut {
  int before;  // tiles per unit of the sequences before b
  int per_unit;  // > 0: that many CTAs for every unit, whose cuts then start with the unit; 0: equal stretches of the line
  long share;    // tiles per CTA (equal stretches)
};
// Equal stretches keep every CTA busy whatever the lengths; a CTA that crosses into another unit, though, pays for its start
// and its result twice (about EXTRA tiles' time), so units that are about equally long are cut each by itself.
constexpr int EXTRA = 5;
__device__ __forceinline__ Cut cut_line(const TreeAttnParams& p, int b, int lane) {
  int before = 0, all = 0, longest = 0;
  for (int i = lane; i < p.batch; i += 32) {
    const int n = live_tiles(p, i);
    all += n;
    if (i < b) before += n;
    longest = max(longest, n);
  }
  before = __reduce_add_sync(0xffffffffu, before);
  all = __reduce_add_sync(0xffffffffu, all);
  longest = __reduce_max_sync(0xffffffffu, longest);
  Cut c;
  c.before = before;
  const long even = ((long)all * p.hkv + p.tc_groups - 1) / p.tc_groups;
  c.share = even < TREE_TC_MIN_TILES ? TREE_TC_MIN_TILES : even;
  const long per = p.tc_groups / ((long)p.batch * p.hkv);
  c.per_unit = per > 0 && (longest + per - 1) / per <= c.share + EXTRA ? (int)per : 0;
  return c;
}
__device__ __forceinline__ int unit_share(const Cut& c, int tiles) { return (tiles + c.per_unit - 1) / c.per_unit; }

template <typename T, int D>
__global__ void __launch_bounds__(TC_THREADS, 1) tree_attention_tc_kernel(const __grid_constant__ CUtensorMap kmap,
                                                                          const __grid_constant__ CUtensorMap vmap, const TreeAttnParams p) {
  using S_ = Tc<D>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* sm = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  unsigned char* ring = sm + S_::Q_BYTES;
  __shared__ uint64_t full[S_::RING], freed[S_::RING], s_full[2], p_full[2], pv_done[2], at_tree, v_fixed, drained;
  // The largest score of each half of a row, in fp32: it is the reference of the exponentials, and rounded to eight bits it was off by
  // 16 at a score of 4096, which is the whole range of an fp16 probability.
  __shared__ float part_m[2][TM];
  float *row_l = (float*)(ring + 40960), *row_m = row_l + 2 * TM;  // at a unit's end, when the ring is idle: [2][TM] sums, [TM] maxima
  __shared__ unsigned long long anc[MAX_TREE_NODES];
  __shared__ unsigned char up[MAX_TREE_NODES];
  __shared__ uint32_t tmem_slot;
  __shared__ int failed_s, odd_s, where[5], sent_s;  // sent_s: ring pieces asked for
  volatile int* failed = &failed_s;

  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  if (t == 0) {
    for (int i = 0; i < S_::RING; ++i) mbar_init(&full[i], 1), mbar_init(&freed[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&s_full[i], 1), mbar_init(&p_full[i], 8), mbar_init(&pv_done[i], 1);
    mbar_init(&at_tree, 8);
    mbar_init(&v_fixed, 2);
    mbar_init(&drained, 1);
    failed_s = sent_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_launch_dependents();  // the merge may set itself up; it waits for this grid's end before it reads

  // ---- this CTA's stretch of the line of tiles ----
  const int row_tiles = (p.rows + TM - 1) / TM, upb = p.hkv;  // units per sequence
  const int rt = blockIdx.x % row_tiles, grp = blockIdx.x / row_tiles;
  if (warp == 2) {
    const Cut cut = cut_line(p, 0, lane);
    int w_b = 0, w_unit = 0, w_tile = 0, w_left = 0;
    if (cut.per_unit) {
      const int u = grp / cut.per_unit, part = grp % cut.per_unit;
      if (u < p.batch * upb) {
        const int n = live_tiles(p, u / upb), share = unit_share(cut, n);
        w_b = u / upb, w_unit = u % upb, w_tile = part * share, w_left = max(min(share, n - w_tile), 0);
      }
    } else {
      const long w0 = grp * cut.share;
      int before = 0;
      bool found = false;
      for (int at = 0; at < p.batch && !found; at += 32) {  // the sequence that holds tile w0
        const int n = at + lane < p.batch ? live_tiles(p, at + lane) : 0;
        int s = n;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
          const int y = __shfl_up_sync(0xffffffffu, s, o);
          if (lane >= o) s += y;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, at + lane < p.batch && (long)(before + s) * upb > w0);
        if (hit) {
          const int l = __ffs(hit) - 1, tiles = __shfl_sync(0xffffffffu, n, l);
          const long inside = w0 - (long)(before + __shfl_sync(0xffffffffu, s - n, l)) * upb;
          w_b = at + l, w_unit = (int)(inside / tiles), w_tile = (int)(inside % tiles);
          w_left = (int)cut.share;  // (the last CTA's stretch ends with the last sequence)
          found = true;
        }
        before += __shfl_sync(0xffffffffu, s, 31);
      }
    }
    if (lane == 0) where[0] = w_b, where[1] = w_unit, where[2] = w_tile, where[3] = w_left, where[4] = cut.per_unit;
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_slot;
  int b = where[0], unit = where[1], tile = where[2], left = where[3];  // left: tiles still to do
  int pieces = 0, done = 0, fixes = 0;  // ring pieces, tiles and (warps 1 to 3) tiles with tree rows so far: what the barriers' parities follow
  bool ok = true;

  const int per_unit = where[4];

  while (left > 0 && b < p.batch) {
    const int L = live_rows(p, b), cached = min(max(p.cache_len[b], 0), p.max_seq), tiles = (L + TN - 1) / TN;
    const int n = min(left, tiles - tile);  // this segment: tiles tile .. tile + n - 1 of the unit
    const int hk = unit;
    const bool has_tree = (tile + n) * TN > cached;

    // ---- queries to shared memory (warps 4 to 11; K-major, swizzled), ancestors (warps 2 and 3), while warp 0 starts loading ----
    auto sync_others = []() { asm volatile("bar.sync 2, %0;" ::"n"(TC_THREADS - 32) : "memory"); };
    const int half = (warp - 4) >> 2, r = (warp & 3) * 32 + lane, row = rt * TM + r;  // (warps 4 to 11)
    const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    if (warp >= 4) {
      constexpr int CH = D / 8, BATCH = CH / 4, N = 256;  // BATCH loads under way per thread, TM * CH in four rounds or fewer
      const int count = min(TM, p.rows - rt * TM) * CH;    // (rows past the last compute on what they find: nobody reads them)
#pragma unroll 1
      for (int i0 = t - 128; i0 < count; i0 += N * BATCH) {
        uint4 v[BATCH];
#pragma unroll
        for (int x = 0; x < BATCH; ++x) {
          const int i = i0 + x * N, qr = i / CH, ch = i % CH, qrow = rt * TM + qr, node = qrow / p.group;
          if (i < count)
            v[x] = *(const uint4*)((const T*)p.q + b * p.q_stride[0] + node * p.q_stride[1] + (hk * p.group + qrow - node * p.group) * p.q_stride[2] + ch * 8);
        }
#pragma unroll
        for (int x = 0; x < BATCH; ++x) {
          const int i = i0 + x * N, qr = i / CH, ch = i % CH;
          if (i < count) *(uint4*)(sm + (ch >> 3) * (TM * 128) + (qr >> 3) * 1024 + (qr & 7) * 128 + (((ch & 7) ^ (qr & 7)) << 4)) = v[x];
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    } else if (warp >= 2) {
      const int i = t - 64;
      if (i == 0) odd_s = 0;
      if (has_tree) {
        auto sync_two = []() { asm volatile("bar.sync 3, 64;" ::: "memory"); };
        if (i < p.nodes) {
          const int pa = p.parents[(long)b * p.parents_stride + i];
          const bool node = pa >= -1 && pa < i;
          anc[i] = node ? 1ull << i : 0ull;
          up[i] = node && pa >= 0 ? pa : 255;
        }
        sync_two();
        for (int step = 1; step < p.nodes; step *= 2) {  // bits of up to 2 * step ancestors
          unsigned long long bits = 0;
          int u = 255;
          if (i < p.nodes) {
            bits = anc[i], u = up[i];
            if (u < 255) bits |= anc[u], u = up[u];
          }
          sync_two();
          if (i < p.nodes) anc[i] = bits, up[i] = u;
          sync_two();
        }
      }
    }
    if (warp > 0) sync_others();

    if (warp == 0) {
      // ---------------- loads: K 0, then K i + 1 and V i in turn ----------------
      if (elect_one()) {
        int c = pieces;
        auto slot = [&]() {  // the next slot, once it is free
          const int s = c % S_::RING;
          if (c >= S_::RING) ok = ok && wait_for(&freed[s], (c / S_::RING - 1) & 1, failed);
          if (ok) mbar_expect_tx(&full[s], S_::PIECE), sent_s = c + 1;
          ++c;
          return s;
        };
        auto load_k = [&](int i) {
          for (int h = 0; h < S_::PIECES; ++h) {
            const int s = slot();
            if (!ok) return;
#pragma unroll
            for (int x = 0; x < S_::K_BLOCKS; ++x)
              tma_box(smem_u32(ring + s * S_::PIECE) + x * (TN * 128), &kmap, (h * S_::K_BLOCKS + x) * 64, (tile + i) * TN, hk, b, &full[s]);
          }
        };
        auto load_v = [&](int i) {
          for (int h = 0; h < S_::PIECES; ++h) {
            const int s = slot();
            if (!ok) return;
#pragma unroll
            for (int x = 0; x < S_::BLOCKS; ++x)
              tma_box(smem_u32(ring + s * S_::PIECE) + x * (S_::V_KEYS * 128), &vmap, x * 64, (tile + i) * TN + h * S_::V_KEYS, hk, b, &full[s]);
          }
        };
        load_k(0);
        for (int i = 0; i < n && ok; ++i) {
          if (i + 1 < n) load_k(i + 1);
          load_v(i);
        }
      }
      __syncwarp();
    } else if (warp == 1) {
      // ---------------- products ----------------
      if (elect_one()) {
        int c = pieces;
        const uint32_t qa = smem_u32(sm), ra = smem_u32(ring);
        const uint32_t id_s = instr_desc<T>(TN, false), id_o = instr_desc<T>(D, true);
        auto scores = [&](int i) {
          const int gi = done + i;
          for (int h = 0; h < S_::PIECES && ok; ++h, ++c) {
            const int s = c % S_::RING;
            ok = wait_for(&full[s], (c / S_::RING) & 1, failed);
            if (!ok) return;
            const uint64_t qd = smem_desc(qa + h * S_::K_BLOCKS * (TM * 128), 0), kd = smem_desc(ra + s * S_::PIECE, 0);
#pragma unroll
            for (int k = 0; k < S_::K_BLOCKS * 4; ++k) {  // (a descriptor's low bits are the address in units of 16 bytes)
              const uint64_t at = (k >> 2) * (TM * 128 / 16) + (k & 3) * 2;
              mma_ss(tmem + S_::S_COL + (gi & 1) * TN, qd + at, kd + at, id_s, (h | k) != 0);
            }
            commit(&freed[s]);
          }
          if (ok) commit(&s_full[gi & 1]);
        };
        scores(0);
        for (int i = 0; i < n && ok; ++i) {
          if (i + 1 < n) scores(i + 1);
          const int gi = done + i;
          ok = ok && wait_for(&p_full[gi & 1], (gi >> 1) & 1, failed);
          if ((tile + i + 1) * TN > cached) {
            ok = ok && wait_for(&v_fixed, fixes & 1, failed);
            ++fixes;
          }
          if (!ok) break;
          fence_after();
          for (int h = 0; h < S_::PIECES && ok; ++h, ++c) {
            const int s = c % S_::RING;
            ok = wait_for(&full[s], (c / S_::RING) & 1, failed);
            if (!ok) break;
            const uint64_t vd = smem_desc(ra + s * S_::PIECE, S_::V_KEYS * 128);
            const uint32_t pa = tmem + S_::S_COL + (gi & 1) * TN + h * (S_::V_KEYS / 2);
#pragma unroll
            for (int k = 0; k < S_::V_KEYS / 16; ++k) mma_ts(tmem + S_::O_COL, pa + k * 8, vd + k * (2048 / 16), id_o, (i | h | k) != 0);
            commit(&freed[s]);
          }
          if (ok) commit(&pv_done[gi & 1]);
        }
      }
      __syncwarp();
    } else if (warp >= 4) {
      // ---------------- softmax: two threads per row, half of the tile's keys each ----------------
      const int in_cache = L - cached;  // nodes that have a cache row
      const unsigned long long bits = !has_tree || row >= p.rows ? 0ull : anc[row / p.group] & (in_cache >= 64 ? ~0ull : (1ull << in_cache) - 1);
      const float sl0 = p.scale * LOG2E;
      float mref = -INFINITY, l = 0.f;
      for (int i = 0; i < n; ++i) {
        const int gi = done + i, key0 = (tile + i) * TN + half * 64;
        const uint32_t scol = lane_base + S_::S_COL + (gi & 1) * TN;
        ok = ok && wait_for(&s_full[gi & 1], (gi >> 1) & 1, failed);
        fence_after();
        uint32_t v[64];
        tmem_ld32(scol + half * 64, v);
        tmem_ld32(scol + half * 64 + 32, v + 32);
        tmem_wait_ld(v);
        tmem_wait_ld(v + 32);
        float sl = sl0;
        if (sl <= 0.f) {  // (a scale that is not positive: applied first, so that masks and the maximum mean the same)
#pragma unroll
          for (int x = 0; x < 64; ++x) v[x] = __float_as_uint(__uint_as_float(v[x]) * sl);
          sl = 1.f;
        }
        if ((tile + i + 1) * TN > cached) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&at_tree);
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const int j0 = key0 + 32 * w - cached;  // node number of the first key, negative in the prefix
            const uint32_t seen = j0 <= -32 ? ~0u : j0 >= MAX_TREE_NODES ? 0u : j0 >= 0 ? (uint32_t)(bits >> j0) : (uint32_t)(bits << -j0) | ((1u << -j0) - 1);
#pragma unroll
            for (int x = 0; x < 32; ++x)
              if (!((seen >> x) & 1)) v[32 * w + x] = 0xff800000u;
          }
        }
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int x = 0; x < 64; ++x) m4[x & 3] = fmaxf(m4[x & 3], __uint_as_float(v[x]));
        float top = __fmul_ru(fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])), sl);
        asm volatile("bar.sync %0, 64;" ::"r"(4 + (warp & 3)) : "memory");  // the tile before's have been read
        part_m[half][r] = top;
        {  // the two warps of these rows meet: both have read S, and both go on or both give up
          uint32_t go;
          asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.and.pred q, %2, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                       : "=r"(go)
                       : "r"((uint32_t)ok), "r"(4 + (warp & 3))
                       : "memory");
          ok = go != 0;
        }
        if (!ok) break;
        top = __fadd_ru(fmaxf(top, part_m[half ^ 1][r]), -Range<T>::HEADROOM);
        if (i == 0) {
          mref = top;
        } else {
          const bool move = top > __fadd_rd(mref, Range<T>::LAZY);
          if (__any_sync(0xffffffffu, move)) {  // (the same in both warps)
            ok = wait_for(&pv_done[(gi - 1) & 1], ((gi - 1) >> 1) & 1, failed);
            fence_after();
            const float f = move ? exp2_fast(mref - top) : 1.f;
            if (move) mref = top, l *= f;
#pragma unroll 1
            for (int x = half * (D / 2); x < (half + 1) * (D / 2); x += 32) {
              uint32_t o[32];
              tmem_ld32(lane_base + S_::O_COL + x, o);
              tmem_wait_ld(o);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st32(lane_base + S_::O_COL + x, o);
            }
          }
        }
        const float ref = mref == -INFINITY ? 0.f : mref;
        float l4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < 64; x += 2) {
          const float p0 = exp2_fast(fmaf(__uint_as_float(v[x]), sl, -ref)), p1 = exp2_fast(fmaf(__uint_as_float(v[x + 1]), sl, -ref));
          l4[(x >> 1) & 3] += p0 + p1;
          v[x >> 1] = pack2<T>(p0, p1);
        }
        l += (l4[0] + l4[1]) + (l4[2] + l4[3]);
        tmem_st32(scol + half * 32, v);
        tmem_wait_st();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[gi & 1]);
      }
      if (ok) ok = wait_for(&pv_done[(done + n - 1) & 1], ((done + n - 1) >> 1) & 1, failed);
      row_l[half * TM + r] = ok ? l : __int_as_float(0x7fffffff);  // (a wait that ran out: NaN)
      if (half == 0) row_m[r] = mref;
    } else {
      // ---------------- warps 2 and 3: values that must not meet a zero probability ----------------
      // Those of rows past the end are zeroed, and so are values of tree rows that are not finite; the latter are added back
      // below for the rows that see them.
      const int first = max(cached / TN - tile, 0);
      for (int i = first; i < n; ++i) {
        const int gi = done + i, key0 = (tile + i) * TN, fr = t - 64;
        // A parity cannot tell "this round has come" from "the round before the last has": the softmax warps say that they are at
        // tile i (S i is there, hence PV i - 2 has been done), then PV i - 1 is waited for: nothing younger was in V i's slots.
        ok = ok && wait_for(&at_tree, fixes & 1, failed);
        ++fixes;
        if (i > 0) ok = ok && wait_for(&pv_done[(gi - 1) & 1], ((gi - 1) >> 1) & 1, failed);
        bool odd = false;
        for (int h = 0; h < S_::PIECES; ++h) {
          const int c = pieces + (i + 1 < n ? 2 * i + 2 : 2 * n - 1) * S_::PIECES + h, s = c % S_::RING;
          ok = ok && wait_for(&full[s], (c / S_::RING) & 1, failed);
          // eight threads per row: its 16-byte chunks in any order, since each is looked at for itself
          const int k0 = key0 + h * S_::V_KEYS;
          for (int y = max(cached - k0, 0) + (fr >> 3); ok && y < S_::V_KEYS; y += 8) {
            uint4* at = (uint4*)(ring + s * S_::PIECE + (y >> 3) * 1024 + (y & 7) * 128 + (fr & 7) * 16);
#pragma unroll
            for (int x = 0; x < S_::BLOCKS; ++x, at += S_::V_KEYS * 128 / 16) {
              if (k0 + y >= L) {
                *at = make_uint4(0u, 0u, 0u, 0u);
                continue;
              }
              uint32_t v[4] = {at->x, at->y, at->z, at->w};
              bool change = false;
              const uint32_t m = exp_mask<T>();
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if ((v[e] & m) == m) v[e] &= 0xffff0000u, change = true;
                if (((v[e] >> 16) & m) == m) v[e] &= 0x0000ffffu, change = true;
              }
              if (change) *at = make_uint4(v[0], v[1], v[2], v[3]), odd = true;
            }
          }
        }
        if (odd) odd_s = 1;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_fixed);
      }
    }
    fence_before();
    __syncthreads();
    fence_after();

    // ---------------- the unit's result, or this CTA's part of it: warps 0 to 7, half of the columns each four ----------------
    if (warp < 8) {
      const int quarter = warp & 3;
      const bool odd = odd_s != 0 && has_tree, whole = n == tiles;
      const uint32_t o_base = lane_base + S_::O_COL;
      const long slot = (per_unit ? grp : grp + (long)b * upb + unit) * row_tiles + rt;
      const float2 ml = make_float2(row_m[r], row_l[r] + row_l[TM + r]);
      const float w = !whole ? 1.f : ml.y == 0.f ? 0.f : 1.f / ml.y;  // (a sum of 0: nothing seen)
      float* stage = (float*)ring + warp * (32 * 36);  // the ring is idle: a row's 32 columns leave as whole lines
#pragma unroll 1
      for (int x = (warp >> 2) * (D / 2); x < (warp >> 2) * (D / 2) + D / 2; x += 32) {
        uint32_t o[32];
        tmem_ld32(o_base + x, o);
        tmem_wait_ld(o);
        if (odd && row < p.rows) {
          for (int j = 0; j < p.nodes; ++j) {
            const int key = cached + j;
            if (!((anc[row / p.group] >> j) & 1) || key >= L || key < tile * TN || key >= (tile + n) * TN) continue;
            const T* y = (const T*)p.vcache + b * p.v_stride[0] + hk * p.v_stride[1] + key * p.v_stride[2] + x;
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const float z = elem_f<T>(y[e]);
              if (!isfinite(z)) o[e] = __float_as_uint(__uint_as_float(o[e]) + z);
            }
          }
        }
#pragma unroll
        for (int e = 0; e < 32; e += 4)
          *(float4*)(stage + lane * 36 + e) = make_float4(__uint_as_float(o[e]) * w, __uint_as_float(o[e + 1]) * w, __uint_as_float(o[e + 2]) * w,
                                                          __uint_as_float(o[e + 3]) * w);
        __syncwarp();
        float4 z[8];
#pragma unroll
        for (int y = 0; y < 8; ++y) z[y] = *(const float4*)(stage + (y * 4 + (lane >> 3)) * 36 + (lane & 7) * 4);
        const int rr0 = quarter * 32 + (lane >> 3), c4 = (lane & 7) * 4;
        if (whole) {
#pragma unroll
          for (int y = 0; y < 8; ++y) {
            const int orow = rt * TM + rr0 + 4 * y;
            if (orow >= p.rows) break;
            const int node = orow / p.group, pa = p.parents[(long)b * p.parents_stride + node];
            T* out = (T*)p.out + (((long)b * p.nodes + node) * p.hq + hk * p.group + orow - node * p.group) * D + x + c4;
            const bool is_node = pa >= -1 && pa < node;
            *(uint2*)out = is_node ? make_uint2(pack2<T>(z[y].x, z[y].y), pack2<T>(z[y].z, z[y].w)) : make_uint2(0u, 0u);
          }
        } else {
          float* acc = p.part_acc + (slot * TM + rr0) * D + x + c4;
#pragma unroll
          for (int y = 0; y < 8; ++y)
            if (rt * TM + rr0 + 4 * y < p.rows) *(float4*)(acc + 4 * y * D) = z[y];
        }
        __syncwarp();
      }
      if (warp < 4 && row < p.rows && !whole) *(float2*)(p.part_ml + (slot * TM + r) * 2) = ml;
    }
    fence_async();  // the ring was written by ordinary stores (row sums, the result's rows): the next unit's copies come after them
    fence_before();
    __syncthreads();  // queries, O and the flags may be written again
    fence_after();
    ok = ok && !*failed;
    pieces += 2 * n * S_::PIECES;
    done += n;
    left -= n;
    tile += n;
    if (tile == tiles) {
      tile = 0;
      if (++unit == upb) unit = 0, ++b;
    }
  }
  if (*failed) {  // a wait ran out: what is still under way ends before its memory is given back
    if (warp == 0 && elect_one()) {
      for (int c = max(sent_s - S_::RING, 0); c < sent_s; ++c) wait_out(&full[c % S_::RING], (c / S_::RING) & 1);
    }
    if (warp == 1 && elect_one()) {
      commit(&drained);
      wait_out(&drained, 0);
    }
  }
  __syncthreads();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
}

// D / 4 lanes per output row, as many rows per CTA as 256 threads hold: the parts of the row's unit in the order of the groups
// that left them, with a running maximum; the loads of four parts are under way at once (8 x 64 nodes, measured side by side: 186 us, with eight 188).
template <typename T, int D>
__global__ void __launch_bounds__(256) tree_tc_merge_kernel(const TreeAttnParams p) {
  constexpr int LANES = D / 4, ROWS = 256 / LANES, AHEAD = 4;
  __shared__ long first_s;
  __shared__ int count_s;
  const int t = threadIdx.x, li = t % LANES;
  const int row = blockIdx.x * ROWS + t / LANES, hk = blockIdx.y, b = blockIdx.z;
  const int row_tiles = (p.rows + TM - 1) / TM;
  if (t < 32) {
    const Cut cut = cut_line(p, b, t);
    const int mine = live_tiles(p, b), u = b * p.hkv + hk;
    if (t == 0) {
      if (cut.per_unit) {
        const int share = unit_share(cut, mine);
        first_s = (long)u * cut.per_unit;
        count_s = (mine + share - 1) / share;
      } else {
        const long w = (long)cut.before * p.hkv + (long)hk * mine;  // first tile of the unit
        const long c0 = w / cut.share;
        first_s = c0 + u;
        count_s = (int)((w + mine - 1) / cut.share - c0) + 1;
      }
    }
  }
  __syncthreads();
  const int count = count_s;
  pdl_wait();  // by every thread, with or without work here: what follows this grid may rely on the attention grid's end
  if (count == 1 || row >= p.rows) return;  // one part: finished by the CTA that had all of it
  const int node = row / p.group, pa = p.parents[(long)b * p.parents_stride + node];
  const bool ok = pa >= -1 && pa < node;
  const long step = (long)row_tiles * TM, at = (first_s * row_tiles + row / TM) * TM + row % TM;  // rows from one part to the next
  const float2* ml = (const float2*)p.part_ml + at;
  const float* acc = p.part_acc + at * D + 4 * li;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  float m = -INFINITY, l = 0.f;
  for (int s0 = 0; s0 < count; s0 += AHEAD) {
    float2 v[AHEAD];
    float4 y[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int s = min(s0 + i, count - 1);
      v[i] = __ldcg(ml + s * step);
      y[i] = __ldcg((const float4*)(acc + s * step * D));
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (s0 + i >= count) break;
      const float mn = fmaxf(m, v[i].x), ref = mn == -INFINITY ? 0.f : mn, f = exp2_fast(m - ref), w = exp2_fast(v[i].x - ref);
      m = mn;
      l = l * f + v[i].y * w;
      a.x = a.x * f + y[i].x * w, a.y = a.y * f + y[i].y * w, a.z = a.z * f + y[i].z * w, a.w = a.w * f + y[i].w * w;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;  // 0: nothing seen
  T* out = (T*)p.out + (((long)b * p.nodes + node) * p.hq + hk * p.group + row - node * p.group) * D + 4 * li;
  *(uint2*)out = ok ? make_uint2(pack2<T>(a.x * inv, a.y * inv), pack2<T>(a.z * inv, a.w * inv)) : make_uint2(0u, 0u);
}

// The cache as [sequence][KV head][row][D] with the caller's strides; boxes of 64 dims x `rows` rows.
bool encode_cache(CUtensorMap* map, const void* base, const long* stride, int rows, const TreeAttnParams& p) {
  return encode_map(map, base, p.is_fp16, {p.d, p.max_seq, p.hkv, p.batch}, {stride[2], stride[1], stride[0]}, {64, rows, 1, 1}, true);
}

template <typename T, int D>
int configure_one() {
  return cudaFuncSetAttribute(tree_attention_tc_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Tc<D>::SMEM) == cudaSuccess
             ? 0
             : check_launch("tree attention (tcgen05): shared-memory opt-in");
}
int configure_all() {
  int rc = configure_one<bf16, 64>();
  if (!rc) rc = configure_one<bf16, 128>();
  if (!rc) rc = configure_one<bf16, 256>();
  if (!rc) rc = configure_one<__half, 64>();
  if (!rc) rc = configure_one<__half, 128>();
  if (!rc) rc = configure_one<__half, 256>();
  return rc;
}

template <typename T, int D>
int launch_one(const CUtensorMap& kmap, const CUtensorMap& vmap, const TreeAttnParams& p, cudaStream_t stream) {
  tree_attention_tc_kernel<T, D><<<p.tc_groups * ((p.rows + TM - 1) / TM), TC_THREADS, Tc<D>::SMEM, stream>>>(kmap, vmap, p);
  const int rc = check_launch("tree attention (tcgen05)");
  if (rc) return rc;
  if (launch_pdl(tree_tc_merge_kernel<T, D>, dim3((p.rows + 1024 / D - 1) / (1024 / D), p.hkv, p.batch), dim3(256), 0, stream, p) != cudaSuccess)
    return check_launch("tree attention (tcgen05): merge");
  return check_launch("tree attention (tcgen05): merge");
}
template <typename T>
int launch_t(const CUtensorMap& kmap, const CUtensorMap& vmap, const TreeAttnParams& p, cudaStream_t stream) {
  switch (p.d) {
    case 64: return launch_one<T, 64>(kmap, vmap, p, stream);
    case 128: return launch_one<T, 128>(kmap, vmap, p, stream);
    default: return launch_one<T, 256>(kmap, vmap, p, stream);
  }
}

}  // namespace

int launch_tree_attention_tc(const TreeAttnParams& p, cudaStream_t stream) {
  static OncePerDevice once;
  const int rc = once.run(configure_all);
  if (rc) return rc;
  CUtensorMap kmap, vmap;
  if (!encode_cache(&kmap, p.kcache, p.k_stride, TN, p) || !encode_cache(&vmap, p.vcache, p.v_stride, p.d == 256 ? TN / 2 : TN, p)) {
    set_error("tree attention (tcgen05): tensor map for the cache failed");
    return 1;
  }
  return p.is_fp16 ? launch_t<__half>(kmap, vmap, p, stream) : launch_t<bf16>(kmap, vmap, p, stream);
}

}  // namespace dfb
