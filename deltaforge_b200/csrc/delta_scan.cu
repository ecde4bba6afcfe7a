// The scan of the chunked delta rule on tcgen05 (sm_100a): the chunks of a head one after the other, the state in registers.
//
// The mathematics and the precision are those of delta_chunk.cu, which prepares k, q, T, W, P and the scalars of every chunk:
//   V' = T V - W S;  O = diag(e^G) Q S + P V';  S <- e^G_C S + sum_j e^(G_C - G_j) k_j v'_j^T
// Everything is done transposed: 128 value columns of a head are the M of the products, tokens or key dims the N. The left
// operand then is always what was just computed (S^T, V'^T), written to TMEM by the threads that have it, a thread per column,
// and the right one an image of the chunk in shared memory as it came. A column's scale belongs to its threads alone. T V does
// not wait for the state: it is computed a chunk ahead from the values as they are (bf16 rows in shared memory).
//
// Warps 0-15: four threads per value column, a quarter of the key rows (of S) and of the tokens (of V') each; S stays there in
// fp32 from the first chunk to the last. Warps 16-19: the output, a thread per column, from TMEM to memory, while the others go
// on. Warp 20 fills the two stages of shared memory by bulk copies, warp 21 issues the products.
//
// Trees are one chunk each and leave no state: 148 CTAs walk through all of them, the next state on its way while the products
// of this one run (16 trees x 32 heads: 53 us with a CTA for each, 42 so).
//
// Bound by the chain from chunk to chunk, 4800 cycles (one 8192-token prompt of 32 heads: 128 chunks, 383 us, of which the
// preparation of the first chunks and the four segments' starts take 60): 1000 until S lies in halves in TMEM, 1000 of tensor
// time for W S, 1400 until V' does, 330 for half of the update, 200 for the new S, and three handovers between threads and
// tensor core of 300 each. The conversions, some 450 instructions per thread and chunk, fill half of all issue slots.
// What it replaced: T R with R = V - diag(e^G) K S in place of W, a product and a handover more per chunk (490 us); and a scan by
// mma.sync on four times the SMs, whose products share their issue slots with all other arithmetic (380 us for one prompt, but
// 229 against 154 for six of 1001 tokens).
#include "delta.cuh"
#include "tcgen05.cuh"

namespace dfb {

namespace {

constexpr int COLS = 128;  // value columns per CTA
constexpr int BY_LENGTH = 256;  // sequences that are put in order (a comparison of each with each in every CTA)
constexpr int SCAN_WARPS = 22, SCAN_THREADS = SCAN_WARPS * 32;

template <int DKP> struct Stage {
  static constexpr int P = key_bytes(DKP), W = P + SQ, BYTES = W + 2 * w_bytes(DKP);
  // two stages; T and the values, which one product reads; the scalars of three chunks (the output reads them last); the
  // output's rows; alignment
  static constexpr int T = 2 * BYTES, V = T + 3 * SQ, ROWS = V + C * COLS * 2, SC = ROWS + C * COLS * 2, SMEM = SC + 3 * SCAL + 1024;
};
// TMEM columns. S and V' are A operands, two fp16 values per column (V' twice: in halves with the decays into the state, and as
// it is for the output); the others are accumulators. The update takes the place of W S, V' in halves that of the lower halves of S.
constexpr int SH = 0, SL = 64, WS = 128, UP = 128, RH = 64, RL = 96, QS = 256, TV = 320, PV = 384, VH = 448;

struct Unit {
  int vb, hv, b;  // block of value columns, value head, sequence
};

template <int DKP, bool TREE>
__global__ void __launch_bounds__(SCAN_THREADS, 1)
    delta_scan_kernel(const __grid_constant__ CUtensorMap vmap, const __grid_constant__ CUtensorMap omap, const DeltaChunkParams p) {
  using G = Stage<DKP>;
  constexpr int NS = DKP / 4;  // key rows per thread
  extern __shared__ unsigned char smem_raw[];
  unsigned char* sm = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ uint64_t full[2], v_full, v_in, s_in[2], tv_out, ws_out, u_in, p_in, u_out[2], o_out[2], o_read, drained;
  __shared__ float s_max[4][COLS], vp_max[4][COLS], r_max[4][COLS];  // of S, V', and the images of V' on their way into S
  __shared__ int s_exp[2][COLS], v_exp[2][COLS];  // by chunk parity, for the output
  __shared__ uint32_t tmem_slot;
  __shared__ int failed_s, seq_s;
  volatile int* failed = &failed_s;

  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  // What is walked through: the chunks of one unit (value columns, head, sequence); for trees units, one chunk each.
  const int wide = (p.dv + COLS - 1) / COLS;
  auto nth = [&](unsigned u) {
    const int rest = u / wide;
    return Unit{(int)u - rest * wide, rest % p.hv, rest / p.hv};
  };
  Unit here = nth(blockIdx.x);
  // The longest prompts first, where not all CTAs run at once (us, as they come / so, 32 heads: six drawn batches of 12 prompts
  // of up to 2000 tokens 407 .. 528 / 390 .. 504, of 6 up to 1001 107 .. 166 / 105 .. 160)
  const bool by_length = !TREE && p.lengths && gridDim.x > 148 && p.batch <= BY_LENGTH;
  if (by_length && t < p.batch) {
    const int mine = p.lengths[t];
    int rank = 0;
    for (int i = 0; i < p.batch; ++i) {
      const int other = p.lengths[i];
      rank += other > mine || (other == mine && i < t);
    }
    if (rank == here.b) seq_s = t;
  }
  if (t == 0) {
    for (int i = 0; i < 2; ++i) mbar_init(&full[i], 1), mbar_init(&s_in[i], 16), mbar_init(&u_out[i], 1), mbar_init(&o_out[i], 1);
    mbar_init(&v_full, 1), mbar_init(&v_in, 1), mbar_init(&tv_out, 1), mbar_init(&ws_out, 1);
    mbar_init(&u_in, 16), mbar_init(&p_in, 16), mbar_init(&o_read, 4), mbar_init(&drained, 1);
    failed_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 21) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (by_length) here.b = seq_s;
  auto unit = [&](int n) { return TREE && n > 0 ? nth(blockIdx.x + n * gridDim.x) : here; };
  int nlive;
  if (TREE) {
    nlive = (wide * p.hv * p.batch - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;
  } else {
    const int len = p.lengths ? min(max(p.lengths[here.b], 0), p.tokens) : p.tokens;
    nlive = min(max((len + C - 1) / C - p.chunk0, 0), p.chunks);  // chunks of this segment with tokens
  }
  const uint32_t tmem = tmem_slot;
  const int q = warp & 3, col = q * 32 + lane;
  const uint32_t base = tmem + ((uint32_t)(q * 32) << 16);
  bool ok = true;  // a wait that ran out lets everything run to its end on garbage; NaN is what is left then

  if (warp < 16) {
    // ---------------- the recurrence ----------------
    const int h = warp >> 2;
    auto meet = [&]() { asm volatile("bar.sync %0, 128;" ::"r"(1 + q) : "memory"); };  // the four warps of these columns
    auto most = [&](const float (&m)[4][COLS]) { return fmaxf(fmaxf(m[0][col], m[1][col]), fmaxf(m[2][col], m[3][col])); };
    // hi and lo of two values
    auto split = [](F2 v, uint32_t& hi, uint32_t& lo) {
      hi = h2(v.x, v.y);
      const float2 f = __half22float2(*(const __half2*)&hi);
      const F2 r = fma2({f.x, f.y}, {-1.f, -1.f}, v);
      lo = h2(r.x, r.y);
    };
    F2 S[NS / 2];
    long sb = 0;  // this thread's column in the state
    bool cok = false;
    auto load = [&](int n) {
      const Unit u = unit(n);
      const int gcol = u.vb * COLS + col;
      cok = gcol < p.dv;
      sb = ((long)u.b * p.hv + u.hv) * p.dk * p.dv + gcol;
      const float* Sin = p.first ? p.state + sb : p.state_out + sb;
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const int d = h * NS + i;
        const float v = cok && d < p.dk ? Sin[(long)d * p.dv] : 0.f;
        (i & 1 ? S[i / 2].y : S[i / 2].x) = v;
      }
    };
    // (The first segment's state is there before the preparation starts; nothing else here comes but through the loads.)
    load(0);
    float ms;
    int es;
    auto scale = [&]() {  // the columns' largest
      ms = 0.f;
#pragma unroll
      for (int i = 0; i < NS / 2; ++i) ms = fmaxf(fmaxf(ms, fabsf(S[i].x)), fabsf(S[i].y));
      s_max[h][col] = ms;
      meet();
      es = scale_exp(most(s_max));
      meet();
    };
    if (!TREE) scale();
    for (int n = 0; n < nlive; ++n) {
      const float* sc = (const float*)(sm + G::SC + n % 3 * SCAL);
      if (TREE) {
        scale();
        if (n > 0) {  // the products of the unit before have read its state
          ok = wait_for(&o_out[(n - 1) & 1], ((n - 1) >> 1) & 1, failed) && ok;
          fence_after();
        }
      }
      // S in halves to TMEM, 16 key rows at a time; its largest on the side
      {
        const float sdown = pow2(-es);
        __half2 top = __float2half2_rn(0.f);
#pragma unroll
        for (int x = 0; x < NS; x += 16) {
          uint32_t hi[8], lo[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            split(mul2(S[x / 2 + i], {sdown, sdown}), hi[i], lo[i]);
            top = __hmax2_nan(top, __habs2(*(const __half2*)&hi[i]));
          }
          if (!TREE && x == 0 && n > 0 && h < 2 && DKP > 64) {  // the lower halves' place: all of the update before has read it
            ok = wait_for(&u_out[1], (n & 1) ^ 1, failed) && ok;
            fence_after();
          }
          tmem_st8(base + SH + h * (NS / 2) + x / 2, hi);
          tmem_st8(base + SL + h * (NS / 2) + x / 2, lo);
          tmem_wait_st();
          fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_in[x / 16]);
        }
        ms = fmaxf(__low2float(top), __high2float(top));
      }
      s_max[h][col] = ms * pow2(es);
      if (h == 0) s_exp[n & 1][col] = es;
      if (TREE && n + 1 < nlive) load(n + 1);

      // V' = T V - W S
      ok = wait_for(&full[n & 1], (n >> 1) & 1, failed) && ok;
      const float wscale = pow2(es) * sc[2 * C + 4 + h], decay = sc[2 * C];  // W is scaled per 16 rows
      ok = wait_for(&tv_out, n & 1, failed) && ok;
      fence_after();
      float uup;
      uint32_t hi[8];
      {
        uint32_t x[16], lo[8];
        tmem_ld16(base + TV + 16 * h, x);
        tmem_wait_ld16(x);
        ok = wait_for(&ws_out, n & 1, failed) && ok;
        fence_after();
        float m0 = 0.f, m1 = 0.f;
#pragma unroll
        for (int y = 0; y < 16; y += 8) {
          uint32_t z[8];
          tmem_ld8(base + WS + 16 * h + y, z);
          tmem_wait_ld8(z);
#pragma unroll
          for (int i = 0; i < 8; i += 2) {
            const F2 r = fma2({__uint_as_float(z[i]), __uint_as_float(z[i + 1])}, {-wscale, -wscale}, {__uint_as_float(x[y + i]), __uint_as_float(x[y + i + 1])});
            x[y + i] = __float_as_uint(r.x), x[y + i + 1] = __float_as_uint(r.y);
            m0 = fmaxf(m0, fabsf(r.x)), m1 = fmaxf(m1, fabsf(r.y));
          }
        }
        vp_max[h][col] = fmaxf(m0, m1);
        meet();
        const float m = most(vp_max);
        const int ev = scale_exp(m), eu = scale_exp(fmaxf(fmaxf(vp_max[0][col], vp_max[1][col]) * sc[2 * C + 12], fmaxf(vp_max[2][col], vp_max[3][col]) * sc[2 * C + 13]));
        if (h == 0) v_exp[n & 1][col] = ev;
        uup = pow2(eu);
        const float a = pow2(-ev), u = pow2(-eu);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const F2 y = mul2({__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])}, {a, a});
          hi[i] = h2(y.x, y.y);
        }
        tmem_st8(base + VH + 8 * h, hi);
        if (!TREE) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 w = *(const float2*)&sc[16 * h + 2 * i];
            split(mul2({__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])}, mul2({w.x, w.y}, {u, u})), hi[i], lo[i]);
          }
          tmem_st8(base + RH + 8 * h, hi);
          tmem_st8(base + RL + 8 * h, lo);
        }
      }
      tmem_wait_st();
      fence_before();
      __syncwarp();
      if (lane == 0) {
        if (!TREE) mbar_arrive(&u_in);
        mbar_arrive(&p_in);
      }
      if (TREE) continue;
      {
        __half2 top = __habs2(*(const __half2*)&hi[0]);
#pragma unroll
        for (int i = 1; i < 8; ++i) top = __hmax2(top, __habs2(*(const __half2*)&hi[i]));
        r_max[h][col] = fmaxf(__low2float(top), __high2float(top));
        // The next S is at most decay |S| + |U|, and U is a sum of 64 products of an image of V', as large as these really are, with one
        // of K, at most 2^13. (An update may be nothing at all, or its largest values forgotten within the chunk: a bound from
        // 2^13, or from a scale that stands for "nothing", pushes S down into fp16's subnormal numbers. Found out here, under the
        // products, it costs nothing; a maximum of V' times its weight per token before them cost 15 to 40 of 382 us.)
        const float both = most(s_max);
        meet();
        es = scale_exp(fmaf(both, fabsf(decay), uup * most(r_max) * (64.f * 8192.f)));
      }

      // S: the update was accumulated apart and is added in fp32
      ok = wait_for(&u_out[h >> 1], n & 1, failed) && ok;
      fence_after();
#pragma unroll
      for (int x = 0; x < NS; x += 16) {
        uint32_t u[16];
        tmem_ld16(base + UP + h * NS + x, u);
        tmem_wait_ld16(u);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          S[x / 2 + i] = fma2({__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1])}, {uup, uup}, mul2(S[x / 2 + i], {decay, decay}));
      }
    }
    if (!TREE) {
      float* So = p.state_out + sb;
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const int d = h * NS + i;
        if (cok && d < p.dk) So[(long)d * p.dv] = ok ? (i & 1 ? S[i / 2].y : S[i / 2].x) : __int_as_float(0x7fffffff);
      }
    }
  } else if (warp < 20) {
    // ---------------- output ----------------
    bf16* rows_s = (bf16*)(sm + G::ROWS);  // a chunk's output rows on their way out
    for (int n = 0; n < nlive; ++n) {
      const float* sc = (const float*)(sm + G::SC + n % 3 * SCAL);
      ok = wait_for(&o_out[n & 1], (n >> 1) & 1, failed) && ok;
      fence_after();
      const float sup = pow2(s_exp[n & 1][col]), vup = ok ? pow2(v_exp[n & 1][col]) : __int_as_float(0x7fffffff);
      if (n > 0) {
        if (warp == 16 && lane == 0) bulk_stores_read();
        asm volatile("bar.sync 5, 128;" ::: "memory");  // the rows of the chunk before have left
      }
#pragma unroll 1
      for (int x = 0; x < C; x += 16) {
        uint32_t a[16], z[16];
        tmem_ld16(base + QS + x, a);
        tmem_ld16(base + PV + x, z);
        tmem_wait_ld16(a);
        tmem_wait_ld16(z);
        const float pscale = vup * sc[2 * C + 8 + x / 16];  // P is scaled per 16 rows
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const float4 w = *(const float4*)&sc[C + x + i];
#pragma unroll
          for (int y = 0; y < 4; y += 2) {
            const F2 o = fma2({__uint_as_float(a[i + y]), __uint_as_float(a[i + y + 1])}, mul2(y ? F2{w.z, w.w} : F2{w.x, w.y}, {sup, sup}),
                              mul2({__uint_as_float(z[i + y]), __uint_as_float(z[i + y + 1])}, {pscale, pscale}));
            const __nv_bfloat162 r = __floats2bfloat162_rn(o.x, o.y);
            rows_s[(x + i + y) * COLS + col] = r.x;
            rows_s[(x + i + y + 1) * COLS + col] = r.y;
          }
        }
      }
      fence_before();
      fence_async();
      asm volatile("bar.sync 5, 128;" ::: "memory");
      if (lane == 0) mbar_arrive(&o_read);  // TMEM and the scalars have been read
      if (warp == 16 && lane == 0) {  // (rows and columns past the ends are left out)
        const Unit u = unit(n);
        tma_store_box(&omap, smem_u32(rows_s), u.vb * COLS, u.hv, TREE ? 0 : (p.chunk0 + n) * C, u.b);
        bulk_stores_commit();
      }
    }
    if (warp == 16 && lane == 0) bulk_stores_done();
    if (!TREE) {  // rows of tokens that no chunk covered: zeros
      const Unit u = here;
      const int from = (p.chunk0 + nlive) * C, to = min(p.tokens, (p.chunk0 + p.chunks) * C), gcol = u.vb * COLS + col;
      const long orow = (long)p.hv * p.dv;
      bf16* out = p.out + ((long)u.b * p.tokens * p.hv + u.hv) * p.dv + gcol;
      for (int i = from; i < to; ++i)
        if (gcol < p.dv) out[(long)i * orow] = f2bf(0.f);
    }
  } else if (warp == 20) {
    // ---------------- loads ----------------
    pdl_wait();
    pdl_launch_dependents();  // the preparation of the next segment may run beside this scan, but not beside the one before
    const long per = p.hk * (long)key_bytes(DKP) + p.hv * (long)head_bytes(DKP);
    int sent = 0, v_sent = 0;  // chunks and values asked for
    for (int n = 0; n < nlive; ++n) {
      // the products of chunk n - 2 are done; they came after the output of chunk n - 3, whose scalars are replaced
      if (n >= 2) ok = wait_for(&o_out[n & 1], ((n >> 1) - 1) & 1, failed) && ok;
      if (!__all_sync(0xffffffffu, ok)) break;
      const Unit u = unit(n);
      const unsigned char* src = p.scratch + ((long)u.b * p.seg_chunks + (TREE ? 0 : n)) * per;
      const unsigned char* head = src + p.hk * (long)key_bytes(DKP) + (long)u.hv * head_bytes(DKP);
      const uint32_t st = smem_u32(sm + (n & 1) * G::BYTES);
      unsigned char* scn = sm + G::SC + n % 3 * SCAL;
      if (elect_one()) {
        uint64_t* bar = &full[n & 1];
        mbar_expect_tx(bar, G::BYTES + SCAL);
        bulk_copy(st, src + (long)(u.hv / (p.hv / p.hk)) * key_bytes(DKP), key_bytes(DKP), bar);
        bulk_copy(st + G::P, head + 3 * SQ, SQ + 2 * w_bytes(DKP), bar);
        bulk_copy(smem_u32(scn), head + 4 * SQ + 2 * w_bytes(DKP), SCAL, bar);
      }
      __syncwarp();
      sent = n + 1;
      if (n > 0) ok = wait_for(&tv_out, (n - 1) & 1, failed) && ok;
      if (!__all_sync(0xffffffffu, ok)) break;
      if (elect_one()) {
        mbar_expect_tx(&v_full, 3 * SQ + C * COLS * 2);
        bulk_copy(smem_u32(sm + G::T), head, 3 * SQ, &v_full);
        for (int i = 0; i < 2; ++i)  // (zeros past the ends)
          tma_box(smem_u32(sm + G::V + i * C * 128), &vmap, u.vb * COLS + 64 * i, u.hv, TREE ? 0 : (p.chunk0 + n) * C, u.b, &v_full);
      }
      __syncwarp();
      v_sent = n + 1;
      // values of tokens that do not count may be anything: zeros take their place
      ok = wait_for(&full[n & 1], (n >> 1) & 1, failed) && ok;
      ok = wait_for(&v_full, n & 1, failed) && ok;
      if (!__all_sync(0xffffffffu, ok)) break;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t empty = ~__float_as_uint(((const float*)scn)[2 * C + 14 + i]);
        if (empty) {
          while (empty) {
            const int row = 32 * i + __ffs(empty) - 1;
            empty &= empty - 1;
            *(uint2*)(sm + G::V + (lane >> 4) * C * 128 + row * 128 + (lane & 15) * 8) = make_uint2(0, 0);
          }
          fence_async();
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&v_in);
    }
    if (!__all_sync(0xffffffffu, ok)) {  // a wait ran out (else all that was asked for has been waited for)
      for (int n = max(sent - 2, 0); n < sent; ++n) wait_out(&full[n & 1], (n >> 1) & 1);
      if (v_sent > 0) wait_out(&v_full, (v_sent - 1) & 1);
    }
  } else {
    // ---------------- products ----------------
    if (elect_one()) {
      const uint32_t i64 = instr_desc<__half>(64, false), u64 = instr_desc<__half>(64, true);
      const uint32_t t64 = instr_desc<bf16>(64, false) | 1u << 15;  // the values' rows run along the contraction
      auto values = [&](int n) {  // T V of chunk n
        ok = wait_for(&v_in, n & 1, failed) && ok;
        fence_after();
        if (!ok) return;
        const uint32_t ts = smem_u32(sm + G::T), vs = smem_u32(sm + G::V);
#pragma unroll
        for (int k = 0; k < C / 16; ++k)
#pragma unroll
          for (int i = 2; i >= 0; --i) mma_ss(tmem + TV, smem_desc(vs + k * 2048, C * 128), smem_desc(ts + i * SQ + k * 32, 0), t64, k != 0 || i != 2);
        commit(&tv_out);
      };
      if (nlive > 0) values(0);
      for (int n = 0; n < nlive; ++n) {
        const uint32_t st = smem_u32(sm + (n & 1) * G::BYTES), ph = n & 1;
        ok = wait_for(&full[n & 1], (n >> 1) & 1, failed) && ok;
        // W S, the key rows as they come: the first 16 of each quarter, then the others
#pragma unroll
        for (int x = 0; x < NS / 16; ++x) {
          ok = wait_for(&s_in[x], ph, failed) && ok;
          fence_after();
          if (!ok) continue;
#pragma unroll
          for (int k = x; k < DKP / 16; k += NS / 16) {
            const uint32_t at = st + G::W + (k >> 2) * SQ + (k & 3) * 32;
            const uint64_t wh = smem_desc(at, 0), wl = smem_desc(at + w_bytes(DKP), 0);
            mma_ts(tmem + WS, tmem + SH + k * 8, wh, i64, k != 0);
            mma_ts(tmem + WS, tmem + SL + k * 8, wh, i64, true);
            mma_ts(tmem + WS, tmem + SH + k * 8, wl, i64, true);
          }
        }
        if (!ok) break;
        commit(&ws_out);
        // Q S, once the output of the chunk before has been read
        if (n > 0) ok = wait_for(&o_read, ph ^ 1, failed) && ok;
        fence_after();
        if (ok) {
#pragma unroll
          for (int k = 0; k < DKP / 16; ++k) mma_ts(tmem + QS, tmem + SH + k * 8, smem_desc(st + (k >> 2) * (2 * C * 128) + C * 128 + (k & 3) * 32, 0), i64, k != 0);
        }
        // the update, 64 key dims at a time, then P V' and the next chunk's T V
        if (!TREE) {
          ok = wait_for(&u_in, ph, failed) && ok;
          fence_after();
          if (!ok) break;
#pragma unroll
          for (int x = 0; x < DKP / 64; ++x) {
#pragma unroll
            for (int k = 0; k < C / 16; ++k) {
              const uint64_t kd = smem_desc(st + x * (2 * C * 128) + k * 2048, 0);
              mma_ts(tmem + UP + x * 64, tmem + RH + k * 8, kd, u64, k != 0);
              mma_ts(tmem + UP + x * 64, tmem + RL + k * 8, kd, u64, true);
            }
            commit(&u_out[x]);
          }
          if (DKP == 64) commit(&u_out[1]);
        }
        ok = wait_for(&p_in, ph, failed) && ok;
        fence_after();
        if (!ok) break;
#pragma unroll
        for (int k = 0; k < C / 16; ++k) mma_ts(tmem + PV, tmem + VH + k * 8, smem_desc(st + G::P + k * 32, 0), i64, k != 0);
        commit(&o_out[ph]);
        if (n + 1 < nlive) values(n + 1);
      }
    }
    __syncwarp();
  }
  fence_before();
  __syncthreads();
  if (*failed) {  // products that are still under way end before their memory is given back
    if (warp == 21 && elect_one()) {
      commit(&drained);
      wait_out(&drained, 0);
    }
    __syncthreads();
  }
  if (warp == 21) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
}

template <int DKP, bool TREE>
int configure() {
  return cudaFuncSetAttribute(delta_scan_kernel<DKP, TREE>, cudaFuncAttributeMaxDynamicSharedMemorySize, Stage<DKP>::SMEM) == cudaSuccess
             ? 0
             : check_launch("delta rule scan: shared-memory opt-in");
}
int configure_all() {
  int rc = configure<64, false>();
  if (!rc) rc = configure<64, true>();
  if (!rc) rc = configure<128, false>();
  if (!rc) rc = configure<128, true>();
  return rc;
}

template <int DKP, bool TREE>
int launch_one(const CUtensorMap& vmap, const CUtensorMap& omap, const DeltaChunkParams& p, dim3 grid, cudaStream_t stream) {
  // Set up beside the preparation (16 x 64 tree nodes: 57.0 -> 54.7 us); a later segment's has another scan to wait for, and
  // its CTAs would only take room from the preparation (8192 tokens: 389 us, with it 407).
  if (p.first) (void)launch_pdl(delta_scan_kernel<DKP, TREE>, grid, dim3(SCAN_THREADS), Stage<DKP>::SMEM, stream, vmap, omap, p);
  else delta_scan_kernel<DKP, TREE><<<grid, SCAN_THREADS, Stage<DKP>::SMEM, stream>>>(vmap, omap, p);
  return check_launch("delta rule scan");
}

}  // namespace

int launch_delta_scan(const DeltaChunkParams& p, cudaStream_t stream) {
  static OncePerDevice once;
  const int rc = once.run(configure_all);
  if (rc) return rc;
  CUtensorMap vmap, omap;
  const long dims[4] = {p.dv, p.hv, p.tokens, p.batch};
  if (!encode_map(&vmap, p.v, false, dims, {p.v_stride[2], p.v_stride[1], p.v_stride[0]}, {64, 1, C, 1}, true) ||
      !encode_map(&omap, p.out, false, dims, {p.dv, (long)p.hv * p.dv, (long)p.tokens * p.hv * p.dv}, {COLS, 1, C, 1}, false)) {
    set_error("delta rule scan: tensor map for the values or the output failed");
    return 1;
  }
  const bool tree = p.parents != nullptr, wide = p.dk > 64;
  const long units = (long)((p.dv + COLS - 1) / COLS) * p.hv * p.batch;
  if (units > 0x7fffffff) {
    set_error("delta rule scan: %d sequences of %d heads are too many", p.batch, p.hv);
    return 2;
  }
  const dim3 grid((unsigned)(tree && units > 148 ? 148 : units));
  if (tree) return wide ? launch_one<128, true>(vmap, omap, p, grid, stream) : launch_one<64, true>(vmap, omap, p, grid, stream);
  return wide ? launch_one<128, false>(vmap, omap, p, grid, stream) : launch_one<64, false>(vmap, omap, p, grid, stream);
}

}  // namespace dfb
