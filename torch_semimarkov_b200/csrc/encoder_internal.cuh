// Internal declarations of the encoder operators: the gated linear recurrence
// (recurrence.cu), the gated residual norm (blocknorm.cu) and the 8-bit
// activation checkpoints (packed.cu, packgrad.cu).
//
// Activations are float32, bfloat16 or float16 (semicrf_dtype); every sum,
// state and statistic is float32, and a value is rounded to its type once,
// when it is stored.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/semicrf.h"

namespace semicrf {

template <class T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }

template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// N values of T that are loaded and stored together
template <class T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

// A (batch, time, channel) tensor: contiguous channels, strides in elements.
template <class T>
struct Seq {
  T* p;
  int64_t sb, st;
  __device__ __forceinline__ T* row(int64_t b, int64_t t) const { return p + b * sb + t * st; }
};
template <class T>
Seq<T> as_seq(const semicrf_sequence& s) {
  return Seq<T>{static_cast<T*>(s.data), s.batch_stride, s.time_stride};
}

// True when every row of s can be read in vectors of n elements.
inline bool seq_aligned(const semicrf_sequence& s, int64_t B, int64_t T, int elem, int n) {
  if (!s.data) return true;
  return reinterpret_cast<uintptr_t>(s.data) % ((uintptr_t)elem * n) == 0 &&
         (B <= 1 || s.batch_stride % n == 0) && (T <= 1 || s.time_stride % n == 0);
}

// Division by a fixed T for values below 2^31: multiply by a rounded-up
// reciprocal and shift (Granlund and Montgomery).
struct Divider {
  unsigned d, mul, shift;
};
inline Divider make_divider(unsigned d) {
  unsigned s = 0;
  while ((1ull << s) < d) ++s;
  return Divider{d, (unsigned)(((1ull << 32) * ((1ull << s) - d)) / d + 1), s};
}
__device__ __forceinline__ unsigned quotient(unsigned n, const Divider& v) {
  return (__umulhi(n, v.mul) + n) >> v.shift;
}

// Position n of a batch of sequences of T positions: its sequence and place there.
struct Places {
  int64_t T;
  Divider by_t;
  bool small;  // every n is below 2^31
};
inline Places make_places(int64_t B, int64_t T) {
  const bool small = B * T < (1ll << 31);
  return Places{T, make_divider(small && T ? (unsigned)T : 1u), small};
}
__device__ __forceinline__ void locate(const Places& p, int64_t n, int64_t& b, int64_t& t) {
  b = p.small ? (int64_t)quotient((unsigned)n, p.by_t) : n / p.T;
  t = n - b * p.T;
}

// Number of valid positions of sequence b (all T without lengths).
__device__ __forceinline__ int64_t valid_length(const int64_t* lengths, int64_t b, int64_t T) {
  if (!lengths) return T;
  const int64_t n = lengths[b];
  return n < 0 ? 0 : (n > T ? T : n);
}

// sigmoid(g) and sigmoid(-g): with e = exp(-g) they are 1 / (1 + e) and
// e / (1 + e), so neither cancels.  e is held to 2^126, where the first is
// 2^-126; a NaN stays one.  Six operations, two of them special functions.
// Two errors are taken back where they count.  The rounding of g / ln 2 puts e
// off by |g| 2^-24 of itself: for float32 activations T the remainder is kept
// and added.  The approximate reciprocal errs to one side, which over the
// hundreds of positions that a gate near 1 remembers adds up (8e-7 of the
// state, against 3e-7): in a CHAIN, and for float32, it gets one Newton step.
constexpr float kInvLn2 = 1.4426950408889634f, kInvLn2Low = 1.925963033500907e-8f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float exp2_capped(float t) {
  float e;
  asm("{.reg .f32 t; min.NaN.f32 t, %1, 0f42FC0000; ex2.approx.ftz.f32 %0, t;}"
      : "=f"(e)
      : "f"(t));
  return e;
}
__device__ __forceinline__ float reciprocal(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// Two channels at once: products and sums go two to an instruction.
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 sub2(float2 a, float2 b) {
  return __ffma2_rn(b, make_float2(-1.f, -1.f), a);  // exactly a - b rounded once
}
template <class T, bool CHAIN = false>
__device__ __forceinline__ void sigmoid_pair2(float2 g, float2& pos, float2& neg) {
  const float2 t = __fmul2_rn(g, both(-kInvLn2));
  float2 e = make_float2(exp2_capped(t.x), exp2_capped(t.y));
  if (sizeof(T) == 4) {
    float2 rest = __ffma2_rn(g, both(-kInvLn2), make_float2(-t.x, -t.y));
    rest = __ffma2_rn(g, both(-kInvLn2Low), rest);
    // past |t| = 128 e is 0 or held, and the remainder of an infinite g is NaN
    rest.x = fabsf(t.x) < 128.f ? rest.x * kLn2 : 0.f;
    rest.y = fabsf(t.y) < 128.f ? rest.y * kLn2 : 0.f;
    e = __ffma2_rn(e, rest, e);
  }
  const float2 d = __fadd2_rn(e, both(1.f));
  pos = make_float2(reciprocal(d.x), reciprocal(d.y));
  if (CHAIN || sizeof(T) == 4)
    pos = __ffma2_rn(pos, __ffma2_rn(make_float2(-d.x, -d.y), pos, both(1.f)), pos);
  neg = __fmul2_rn(e, pos);
}
template <class T, bool CHAIN = false>
__device__ __forceinline__ void sigmoid_pair(float g, float& pos, float& neg) {
  const float t = g * -kInvLn2;
  float e = exp2_capped(t);
  if (sizeof(T) == 4) {
    const float rest = fmaf(g, -kInvLn2Low, fmaf(g, -kInvLn2, -t));
    e = fmaf(e, fabsf(t) < 128.f ? rest * kLn2 : 0.f, e);
  }
  const float d = 1.f + e;
  pos = reciprocal(d);
  if (CHAIN || sizeof(T) == 4) pos = fmaf(pos, fmaf(-d, pos, 1.f), pos);
  neg = e * pos;
}

template <class T>
__device__ __forceinline__ float2 to_f32x2(const Pack<T, 2>& v) {
  return make_float2(to_f32(v.v[0]), to_f32(v.v[1]));
}
template <>
__device__ __forceinline__ float2 to_f32x2(const Pack<__half, 2>& v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
template <class T>
__device__ __forceinline__ Pack<T, 2> from_f32x2(float2 v);
template <>
__device__ __forceinline__ Pack<float, 2> from_f32x2<float>(float2 v) {
  Pack<float, 2> q;
  q.v[0] = v.x, q.v[1] = v.y;
  return q;
}
template <>
__device__ __forceinline__ Pack<__nv_bfloat16, 2> from_f32x2<__nv_bfloat16>(float2 v) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
  return *reinterpret_cast<const Pack<__nv_bfloat16, 2>*>(&h);
}
template <>
__device__ __forceinline__ Pack<__half, 2> from_f32x2<__half>(float2 v) {
  const __half2 h = __floats2half2_rn(v.x, v.y);
  return *reinterpret_cast<const Pack<__half, 2>*>(&h);
}

// ---------------------------------------------------------------------------
// 8-bit checkpoints: 32 channels of a position share the scale 2^e, e + 127 in
// a byte.  A power of two costs up to one bit against a free scale, and makes
// both directions exact operations: the codes do not depend on how a division
// rounds, and a decoded value has 7 bits, so it is exact in bfloat16.
// ---------------------------------------------------------------------------
constexpr int kPackGroup = 32;
__host__ __device__ inline int64_t pack_groups(int64_t D) {
  return (D + kPackGroup - 1) / kPackGroup;
}

template <class T>
__device__ __forceinline__ float largest_finite();
template <>
__device__ __forceinline__ float largest_finite<float>() { return 3.402823466e38f; }
template <>
__device__ __forceinline__ float largest_finite<__nv_bfloat16>() { return 3.389531390e38f; }
template <>
__device__ __forceinline__ float largest_finite<__half>() { return 65504.f; }

__device__ __forceinline__ float pack_scale(uint8_t byte) {  // 255 (inf) times code 0 is NaN
  return __int_as_float((int)byte << 23);
}

// The largest magnitude of a lane's values, as the bits of a float.
template <class T, int V>
__device__ __forceinline__ unsigned pack_top(const Pack<T, V>& v, unsigned lanes) {
  unsigned top = 0;
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
    // 16-bit types order by their bits without the sign: two at a time
    const unsigned* w = reinterpret_cast<const unsigned*>(v.v);
#pragma unroll
    for (int j = 0; j < V / 2; ++j) top = __vmaxu2(top, w[j] & 0x7fff7fffu);
#pragma unroll
    for (int o = 1; o < kPackGroup / V; o <<= 1) top = __vmaxu2(top, __shfl_xor_sync(lanes, top, o));
    const unsigned short one = (unsigned short)max(top & 0xffffu, top >> 16);
    return __float_as_uint(to_f32(*reinterpret_cast<const T*>(&one)));
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) top = max(top, __float_as_uint(to_f32(v.v[j])) & 0x7fffffffu);
#pragma unroll
    for (int o = 1; o < kPackGroup / V; o <<= 1) top = max(top, __shfl_xor_sync(lanes, top, o));
    return top;
  }
}

// Codes of a group whose values lie V to a lane in 32 / V neighbouring lanes
// (all of `lanes` call this together); returns the scale byte.
template <class T, int V>
__device__ __forceinline__ uint8_t pack_encode(const Pack<T, V>& v, Pack<int8_t, V>& q,
                                               unsigned lanes = ~0u) {
  // top = m 2^p, 1/2 <= m < 1, exponent field p + 126: e is p - 7 where m <= 127/128, else p - 6
  const unsigned top = pack_top(v, lanes);
  const int field = (int)(top >> 23);
  int byte = max(1, field - 6 + ((top & 0x7fffffu) > 0x7e0000u));
  if (top == 0) byte = 0;
  const bool finite = field < 255;
  if (!finite) byte = 255;
  const float inv = __int_as_float((254 - (finite ? byte : 254)) << 23);
  // adding 1.5 * 2^23 rounds to the nearest integer, ties to even, into the low bits
  int r[V];
#pragma unroll
  for (int j = 0; j < V; ++j) r[j] = __float_as_int(fmaf(to_f32(v.v[j]), inv, 12582912.f));
  const float most = floorf(largest_finite<T>() * inv);
  if (!finite || most < 127.f) {  // the topmost scale of the type: no code past its largest value
#pragma unroll
    for (int j = 0; j < V; ++j)
      r[j] = finite ? (int)fminf(fmaxf(rintf(to_f32(v.v[j]) * inv), -most), most) : 0;
  }
  if constexpr (V % 4 == 0) {
    unsigned* w = reinterpret_cast<unsigned*>(q.v);
#pragma unroll
    for (int j = 0; j < V; j += 4)
      w[j / 4] = __byte_perm(__byte_perm(r[j], r[j + 1], 0x0040),
                             __byte_perm(r[j + 2], r[j + 3], 0x0040), 0x5410);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) q.v[j] = (int8_t)r[j];
  }
  return (uint8_t)byte;
}

// 8 codes to 8 bfloat16 values: code byte q = (q & 127) - (q & 128); either
// part OR 0x4300 is a bfloat16 of 128 more, so their difference is q, exactly.
__device__ __forceinline__ uint4 pack_decode(uint2 q, uint8_t byte) {
  const __nv_bfloat162 unit = __bfloat162bfloat162(__float2bfloat16_rn(pack_scale(byte)));
  unsigned o[4];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const unsigned w = k ? q.y : q.x;
    const unsigned lo = w & 0x7f7f7f7fu, hi = w & 0x80808080u;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const unsigned pick = h ? 0x4342u : 0x4140u;  // two bytes, each below a 0x43
      const unsigned a = __byte_perm(lo, 0x43434343u, pick), c = __byte_perm(hi, 0x43434343u, pick);
      const __nv_bfloat162 v = __hmul2(__hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                               *reinterpret_cast<const __nv_bfloat162*>(&c)),
                                       unit);
      o[2 * k + h] = *reinterpret_cast<const unsigned*>(&v);
    }
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// The same for the checkpoint of a float16 activation, whose decoded values are
// all float16: code byte q + 128 below 0x64 is 1024 + q + 128.  The scale may lie
// below float16's range and is then multiplied in two steps; the first is exact,
// since 2^-14 is the smallest normal number, and the second ends on a float16.
__device__ __forceinline__ uint4 pack_decode_half(uint2 q, uint8_t byte) {
  const bool low = byte < 127 - 14;
  const __half2 unit = __half2half2(__float2half_rn(low ? 6.103515625e-5f : pack_scale(byte)));
  const __half2 rest = __half2half2(__float2half_rn(low ? pack_scale(byte + 14) : 1.f));
  const __half2 zero_at = __half2half2(__float2half_rn(1152.f));
  unsigned o[4];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const unsigned w = (k ? q.y : q.x) ^ 0x80808080u;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const unsigned a = __byte_perm(w, 0x64646464u, h ? 0x4342u : 0x4140u);
      const __half2 v = __hmul2(
          __hmul2(__hsub2(*reinterpret_cast<const __half2*>(&a), zero_at), unit), rest);
      o[2 * k + h] = *reinterpret_cast<const unsigned*>(&v);
    }
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

inline int launch_status() {
  return cudaGetLastError() == cudaSuccess ? SEMICRF_OK : SEMICRF_ERR_CUDA;
}

// recurrence.cu
size_t recurrence_saved_bytes(const semicrf_recurrence* p);
size_t recurrence_workspace_bytes(const semicrf_recurrence* p);
int recurrence_forward(const semicrf_recurrence* p, const semicrf_sequence& h, float* final_state,
                       void* saved, void* workspace, cudaStream_t stream);
int recurrence_backward(const semicrf_recurrence* p, const void* saved,
                        const semicrf_sequence& grad_h, const float* grad_state,
                        const semicrf_sequence& grad_x, const semicrf_sequence& grad_gate,
                        float* grad_initial, void* workspace, cudaStream_t stream);
int recurrence_step(int64_t B, int64_t D, int dtype, const void* x, int64_t x_stride,
                    const void* gate, int64_t gate_stride, const uint8_t* active,
                    const float* state, float* state_out, void* h, cudaStream_t stream);

// blocknorm.cu
size_t block_norm_workspace_bytes(const semicrf_block_norm* p);
int block_norm_forward(const semicrf_block_norm* p, const semicrf_sequence& residual_out,
                       const semicrf_sequence& normed, float* statistics, int8_t* codes,
                       uint8_t* scales, cudaStream_t stream);
int block_norm_backward(const semicrf_block_norm* p, const float* statistics,
                        const semicrf_sequence& grad_residual_out,
                        const semicrf_sequence& grad_normed, const semicrf_sequence& grad_residual,
                        const semicrf_sequence& grad_branch, const semicrf_sequence& grad_gate,
                        float* grad_weights, void* workspace, cudaStream_t stream);

// packed.cu
int pack_rows(int64_t B, int64_t T, int64_t D, int dtype, const semicrf_sequence& x,
              const int64_t* lengths, int8_t* codes, uint8_t* scales, cudaStream_t stream);
int unpack_rows(int64_t rows, int64_t D, int dtype, const int8_t* codes, const uint8_t* scales,
                void* out, cudaStream_t stream);

// packgrad.cu
size_t packed_weight_grad_workspace_bytes(int64_t B, int64_t T, int64_t D, int64_t M, int dtype);
int packed_weight_grad(int64_t B, int64_t T, int64_t D, int64_t M, int dtype, int packed_dtype,
                       const semicrf_sequence& grad_output, const int8_t* codes,
                       const uint8_t* scales, const int64_t* lengths, int out_dtype, void* out,
                       void* workspace, cudaStream_t stream);

}  // namespace semicrf
