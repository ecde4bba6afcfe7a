// Rotary positions for several new tokens, sm_100a: queries and keys turned by the angles of integer positions, and, in the
// appending form, keys and values written straight into the KV cache. It is the many-token counterpart of what
// attn_prep_kernel does for one token (src/deltaforge/reference.py:638-650) without cos/sin tables.
//
//   a_i = position * inv_freq[i];  (x, y) -> (x c - y s, y c + x s),  c = factor cos a_i, s = factor sin a_i
//   pairs (x, y): dims (i, i + r/2) in the half layout, (2i, 2i + 1) in the interleaved one; dims >= r pass through
//
// Angles: a position of 2^18 times a frequency near 1 has only six fraction bits left in fp32, so the angle is formed in
// turns in fp64 (position * inv_freq / 2 pi), its whole turns are dropped there, and only the fraction is rounded to fp32 for
// sincospif. That is r/2 fp64 products per token, shared by all its heads.
//
// Bound: HBM. Each input element is read once and each output element written once, in 16-byte vectors; a CTA owns a
// token, and its threads have up to five vectors each under way while the angles are computed.
#include "common.cuh"
#include "kernels.h"

namespace dfb {

namespace {

constexpr int ROT_THREADS = 256;

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(bf16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ bf16 from_f(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ float from_f(float v) { return v; }

template <typename T, int V> struct alignas(sizeof(T) * V) Vec { T e[V]; };

__device__ __forceinline__ int fast_div(int x, unsigned long long mul) { return (int)(((unsigned long long)(unsigned)x * mul) >> 32); }

// V elements per access: 16 bytes where every address allows it, else single elements. One CTA per token. Its work is two
// lists: vectors that turn (half layout: a vector and its partner r/2 further on) of the query and key heads, and vectors that
// pass through (dims from r on of those heads, and the value heads of the appending form as a whole).
template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(ROT_THREADS) rotary_kernel(const RotaryParams p) {
  __shared__ float2 cs[MAX_ROTARY_DIM / 2];
  using Pack = Vec<T, V>;
  constexpr int COPIES = 3, TURNS = INTERLEAVED ? 2 : 1;  // under way per thread before the first use
  constexpr bool PAIRS = !INTERLEAVED || V == 1;          // a unit is two vectors
  const int tok = blockIdx.x % p.tokens, b = blockIdx.x / p.tokens, t = threadIdx.x;
  const int half = p.rotary_dim / 2;
  const bool append = p.kcache != nullptr;
  bool row_ok = true;
  long row = 0;
  if (append) {
    row = (long)p.cache_len[b] + tok;
    row_ok = row >= 0 && row < p.max_seq;  // a row the cache does not have is not written
  }
  const T *q = (const T*)p.q + b * p.q_stride[0] + tok * p.q_stride[1], *k = (const T*)p.k + b * p.k_stride[0] + tok * p.k_stride[1];
  const long bt = (long)b * p.tokens + tok;
  T *qo = (T*)p.q_out + bt * p.hq * p.d, *ko = append ? (T*)p.kcache + b * p.kc_stride[0] + row * p.kc_stride[2] : (T*)p.k_out + bt * p.hkv * p.d;
  const long ko_stride = append ? p.kc_stride[1] : p.d;
  const T* v = append ? (const T*)p.v + b * p.v_stride[0] + tok * p.v_stride[1] : nullptr;
  T* vo = append ? (T*)p.vcache + b * p.vc_stride[0] + row * p.vc_stride[2] : nullptr;
  const int heads = row_ok ? p.hq + p.hkv : p.hq;
  const int n_turn = heads * p.turn_units, n_pass = heads * p.pass_units, n_copy = n_pass + (append && row_ok ? p.hkv * (p.d / V) : 0);

  // places of copy i and of turn i
  auto copy_at = [&](int i, const T*& from, T*& to) {
    if (i < n_pass) {
      const int h = fast_div(i, p.pass_mul), at = p.rotary_dim + (i - h * p.pass_units) * V;
      if (h < p.hq) from = q + h * p.q_stride[2] + at, to = qo + h * p.d + at;
      else from = k + (h - p.hq) * p.k_stride[2] + at, to = ko + (h - p.hq) * ko_stride + at;
    } else {
      const int h = fast_div(i - n_pass, p.value_mul), at = (i - n_pass - h * (p.d / V)) * V;
      from = v + h * p.v_stride[2] + at, to = vo + h * p.vc_stride[1] + at;
    }
  };
  auto turn_at = [&](int i, const T*& from, T*& to, int& u) {
    const int h = fast_div(i, p.turn_mul);
    u = i - h * p.turn_units;
    const int at = INTERLEAVED && V == 1 ? 2 * u : u * V;
    if (h < p.hq) from = q + h * p.q_stride[2] + at, to = qo + h * p.d + at;
    else from = k + (h - p.hq) * p.k_stride[2] + at, to = ko + (h - p.hq) * ko_stride + at;
  };
  const int second = INTERLEAVED ? 1 : half;  // from the first vector of a pair to the second

  bool angles = false;
  for (int c0 = t, r0 = t; c0 < n_copy || r0 < n_turn || !angles; c0 += COPIES * ROT_THREADS, r0 += TURNS * ROT_THREADS) {
    Pack cv[COPIES], x[TURNS], y[TURNS];
    const T* from;
    T* to;
    int u;
#pragma unroll
    for (int i = 0; i < COPIES; ++i)
      if (c0 + i * ROT_THREADS < n_copy) {
        copy_at(c0 + i * ROT_THREADS, from, to);
        cv[i] = *(const Pack*)from;
      }
#pragma unroll
    for (int i = 0; i < TURNS; ++i)
      if (r0 + i * ROT_THREADS < n_turn) {
        turn_at(r0 + i * ROT_THREADS, from, to, u);
        x[i] = *(const Pack*)from;
        if (PAIRS) y[i] = *(const Pack*)(from + second);
      }
    if (!angles) {  // while the first loads are on their way
      const long pi = (long)b * p.pos_stride + tok;
      const double position = p.pos_is_i64 ? (double)((const int64_t*)p.pos)[pi] : (double)((const int*)p.pos)[pi];
      for (int i = t; i < half; i += ROT_THREADS) {
        const double f = p.freq_is_f64 ? ((const double*)p.inv_freq)[i] : (double)((const float*)p.inv_freq)[i];
        const double turns = position * (f * 0.15915494309189533577);  // 1 / (2 pi)
        float sn, cn;
        sincospif(2.f * (float)(turns - rint(turns)), &sn, &cn);
        cs[i] = make_float2(cn * p.factor, sn * p.factor);
      }
      __syncthreads();
      angles = true;
    }
#pragma unroll
    for (int i = 0; i < COPIES; ++i)
      if (c0 + i * ROT_THREADS < n_copy) {
        copy_at(c0 + i * ROT_THREADS, from, to);
        *(Pack*)to = cv[i];
      }
#pragma unroll
    for (int i = 0; i < TURNS; ++i)
      if (r0 + i * ROT_THREADS < n_turn) {
        turn_at(r0 + i * ROT_THREADS, from, to, u);
        if (PAIRS) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float a = to_f<T>(x[i].e[e]), z = to_f<T>(y[i].e[e]);
            const float2 w = cs[u * V + e];
            x[i].e[e] = from_f<T>(a * w.x - z * w.y);
            y[i].e[e] = from_f<T>(z * w.x + a * w.y);
          }
          *(Pack*)to = x[i];
          *(Pack*)(to + second) = y[i];
        } else {
#pragma unroll
          for (int e = 0; e + 1 < V; e += 2) {
            const float a = to_f<T>(x[i].e[e]), z = to_f<T>(x[i].e[e + 1]);
            const float2 w = cs[(u * V + e) / 2];
            x[i].e[e] = from_f<T>(a * w.x - z * w.y);
            x[i].e[e + 1] = from_f<T>(z * w.x + a * w.y);
          }
          *(Pack*)to = x[i];
        }
      }
  }
}

template <typename T>
int launch_rotary_t(RotaryParams p, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  auto whole = [&](const void* ptr, const long* stride) {  // null: not part of this call
    return ptr == nullptr || ((uintptr_t)ptr % 16 == 0 && stride[0] % V == 0 && stride[1] % V == 0 && stride[2] % V == 0);
  };
  const long none[3] = {0, 0, 0};
  const bool vec = p.d % V == 0 && p.rotary_dim % V == 0 && (p.interleaved || (p.rotary_dim / 2) % V == 0) && whole(p.q, p.q_stride) &&
                   whole(p.k, p.k_stride) && whole(p.v, p.v_stride) && whole(p.kcache, p.kc_stride) && whole(p.vcache, p.vc_stride) &&
                   whole(p.q_out, none) && whole(p.k_out, none);
  const int v = vec ? V : 1;
  p.turn_units = p.interleaved ? p.rotary_dim / (v == 1 ? 2 : v) : p.rotary_dim / 2 / v;
  p.pass_units = (p.d - p.rotary_dim) / v;
  // x / n = x * mul >> 32 with mul = 2^32 / n rounded up by e / n, for all x with x e < 2^32: any x where n is a power of two, and
  // below 2^32 / n always. Heads of many thousand dims can go beyond that, and a wrong quotient is another head's address.
  bool exact = true;
  auto mul = [&exact](int n, long heads) {
    if (n <= 0) return 0ull;
    const unsigned long long m = ((1ull << 32) + n - 1) / n, e = m * n - (1ull << 32), most = (unsigned long long)heads * n;
    if (most > 0x7fffffff || (most - 1) * e >= 1ull << 32) exact = false;
    return m;
  };
  p.turn_mul = mul(p.turn_units, (long)p.hq + p.hkv);
  p.pass_mul = mul(p.pass_units, (long)p.hq + p.hkv);
  p.value_mul = mul(p.d / v, p.hkv);
  if (!exact) {
    set_error("rotary positions: %d + %d heads of %d dims are too many for one call", p.hq, p.hkv, p.d);
    return 2;
  }
  const dim3 grid((unsigned)((long)p.batch * p.tokens)), block(ROT_THREADS);
  if (vec && p.interleaved) rotary_kernel<T, V, true><<<grid, block, 0, stream>>>(p);
  else if (vec) rotary_kernel<T, V, false><<<grid, block, 0, stream>>>(p);
  else if (p.interleaved) rotary_kernel<T, 1, true><<<grid, block, 0, stream>>>(p);
  else rotary_kernel<T, 1, false><<<grid, block, 0, stream>>>(p);
  return check_launch("rotary positions");
}

}  // namespace

int launch_rotary(const RotaryParams& p, cudaStream_t stream) {
  if (p.batch == 0 || p.tokens == 0) return 0;
  switch (p.dtype) {
    case DTYPE_BF16: return launch_rotary_t<bf16>(p, stream);
    case DTYPE_FP16: return launch_rotary_t<__half>(p, stream);
    default: return launch_rotary_t<float>(p, stream);
  }
}

}  // namespace dfb
