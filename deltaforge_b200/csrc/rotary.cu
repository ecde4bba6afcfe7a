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
// Bound: HBM. Each input element is read once and each output element written once, in 16-byte vectors; one CTA owns a
// token, a group of lanes a head, and every lane issues the loads of UNROLL heads before the first use.
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

// V elements per access: 16 bytes where every address allows it, else single elements. A "unit" of a head is what one
// lane moves at a time: a rotated vector (half layout: the vector and its partner r/2 further on), or a vector beyond r.
template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(ROT_THREADS) rotary_kernel(const RotaryParams p) {
  __shared__ float2 cs[MAX_ROTARY_DIM / 2];
  using Pack = Vec<T, V>;
  const int tok = blockIdx.x % p.tokens, b = blockIdx.x / p.tokens, t = threadIdx.x;
  const int half = p.rotary_dim / 2;
  const long pi = (long)b * p.pos_stride + tok;
  const double position = p.pos_is_i64 ? (double)((const int64_t*)p.pos)[pi] : (double)((const int*)p.pos)[pi];
  for (int i = t; i < half; i += ROT_THREADS) {
    const double f = p.freq_is_f64 ? ((const double*)p.inv_freq)[i] : (double)((const float*)p.inv_freq)[i];
    const double turns = position * (f * 0.15915494309189533577);  // 1 / (2 pi)
    float s, c;
    sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
    cs[i] = make_float2(c * p.factor, s * p.factor);
  }
  __syncthreads();

  const int rot_units = INTERLEAVED ? p.rotary_dim / (V == 1 ? 2 : V) : half / V;
  const int units = rot_units + (p.d - p.rotary_dim) / V;
  const int lph = p.lanes_per_head, u0 = t % lph, slots = ROT_THREADS / lph;
  const bool append = p.kcache != nullptr;
  long row = 0;
  bool row_ok = true;
  if (append) {
    row = (long)p.cache_len[b] + tok;
    row_ok = row >= 0 && row < p.max_seq;
  }
  const int heads = p.hq + p.hkv;
#pragma unroll 2
  for (int h = t / lph; h < heads; h += slots) {
    const bool is_q = h < p.hq;
    const int hk = h - p.hq;
    const T* in = is_q ? (const T*)p.q + b * p.q_stride[0] + tok * p.q_stride[1] + h * p.q_stride[2]
                       : (const T*)p.k + b * p.k_stride[0] + tok * p.k_stride[1] + hk * p.k_stride[2];
    T* out;
    if (is_q)
      out = (T*)p.q_out + (((long)b * p.tokens + tok) * p.hq + h) * p.d;
    else if (append)
      out = (T*)p.kcache + b * p.kc_stride[0] + hk * p.kc_stride[1] + row * p.kc_stride[2];
    else
      out = (T*)p.k_out + (((long)b * p.tokens + tok) * p.hkv + hk) * p.d;
    if (!is_q && !row_ok) continue;  // a row the cache does not have is not written
    for (int u = u0; u < units; u += lph) {
      if (u >= rot_units) {
        const int at = p.rotary_dim + (u - rot_units) * V;
        *(Pack*)(out + at) = *(const Pack*)(in + at);
      } else if (INTERLEAVED && V == 1) {  // one pair, element by element
        const float x = to_f<T>(in[2 * u]), y = to_f<T>(in[2 * u + 1]);
        const float2 w = cs[u];
        out[2 * u] = from_f<T>(x * w.x - y * w.y);
        out[2 * u + 1] = from_f<T>(y * w.x + x * w.y);
      } else if (INTERLEAVED) {
        Pack v = *(const Pack*)(in + u * V);
#pragma unroll
        for (int e = 0; e + 1 < V; e += 2) {
          const float x = to_f<T>(v.e[e]), y = to_f<T>(v.e[e + 1]);
          const float2 w = cs[(u * V + e) / 2];
          v.e[e] = from_f<T>(x * w.x - y * w.y);
          v.e[e + 1] = from_f<T>(y * w.x + x * w.y);
        }
        *(Pack*)(out + u * V) = v;
      } else {
        Pack v = *(const Pack*)(in + u * V), z = *(const Pack*)(in + half + u * V);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float x = to_f<T>(v.e[e]), y = to_f<T>(z.e[e]);
          const float2 w = cs[u * V + e];
          v.e[e] = from_f<T>(x * w.x - y * w.y);
          z.e[e] = from_f<T>(y * w.x + x * w.y);
        }
        *(Pack*)(out + u * V) = v;
        *(Pack*)(out + half + u * V) = z;
      }
    }
  }
  if (!append || !row_ok) return;
  const int vvec = p.d / V;
  for (int i = t; i < p.hkv * vvec; i += ROT_THREADS) {
    const int h = i / vvec, at = (i - h * vvec) * V;
    *(Pack*)((T*)p.vcache + b * p.vc_stride[0] + h * p.vc_stride[1] + row * p.vc_stride[2] + at) =
        *(const Pack*)((const T*)p.v + b * p.v_stride[0] + tok * p.v_stride[1] + h * p.v_stride[2] + at);
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
  const int units = (p.interleaved ? p.rotary_dim / (v == 1 ? 2 : v) : p.rotary_dim / 2 / v) + (p.d - p.rotary_dim) / v;
  p.lanes_per_head = 1;
  while (p.lanes_per_head < units && p.lanes_per_head < 32) p.lanes_per_head *= 2;
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
