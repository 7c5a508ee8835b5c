// packed.cu -- 8-bit activation checkpoints: store and read back.
//
// Both directions are one pass, bound by memory: 2 + 1 + 1/32 bytes an
// element for 16-bit activations.  A lane takes 16 bytes of a row, so the
// lanes of a group of 32 channels are neighbours and its maximum is a few
// shuffles.

#include "encoder_internal.cuh"

namespace semicrf {
namespace {

template <class T, int V>
__global__ void __launch_bounds__(256) pack_kernel(int64_t rows, int64_t T_, int64_t D, Seq<const T> x,
                                                   const int64_t* __restrict__ lengths,
                                                   int8_t* __restrict__ codes,
                                                   uint8_t* __restrict__ scales) {
  const int64_t G = pack_groups(D), per = G * (kPackGroup / V);
  const int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t row = id / per, d = (id - row * per) * V;
  const bool in = row < rows;  // lanes past the end still take part in the shuffles
  float v[V] = {};
  if (in) {
    const int64_t b = row / T_, t = row - b * T_;
    if (d < D && t < valid_length(lengths, b, T_)) {
      const Pack<T, V> q = *reinterpret_cast<const Pack<T, V>*>(x.row(b, t) + d);
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] = to_f32(q.v[k]);
    }
  }
  int8_t c[V];
  const uint8_t byte = pack_encode<T, V>(v, c);
  if (!in) return;
  Pack<int8_t, V> pc;
#pragma unroll
  for (int k = 0; k < V; ++k) pc.v[k] = c[k];
  *reinterpret_cast<Pack<int8_t, V>*>(codes + row * G * kPackGroup + d) = pc;
  if (d % kPackGroup == 0) scales[row * G + d / kPackGroup] = byte;
}

template <class T, int V>
__global__ void __launch_bounds__(256) unpack_kernel(int64_t rows, int64_t D,
                                                     const int8_t* __restrict__ codes,
                                                     const uint8_t* __restrict__ scales,
                                                     T* __restrict__ out) {
  const int64_t G = pack_groups(D), per = (D + V - 1) / V;
  const int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t row = id / per, d = (id - row * per) * V;
  if (row >= rows) return;
  const float unit = pack_scale(scales[row * G + d / kPackGroup]);
  const Pack<int8_t, V> c =
      *reinterpret_cast<const Pack<int8_t, V>*>(codes + row * G * kPackGroup + d);
  Pack<T, V> q;
#pragma unroll
  for (int k = 0; k < V; ++k) q.v[k] = from_f32<T>((float)c.v[k] * unit);
  *reinterpret_cast<Pack<T, V>*>(out + row * D + d) = q;
}

template <class T, int V>
int launch_pack(int64_t B, int64_t T_, int64_t D, const semicrf_sequence& x,
                const int64_t* lengths, int8_t* codes, uint8_t* scales, cudaStream_t stream) {
  const int64_t n = B * T_ * pack_groups(D) * (kPackGroup / V);
  const int64_t grid = (n + 255) / 256;
  if (grid > 0x7fffffff) return SEMICRF_ERR_UNSUPPORTED;
  if (grid)
    pack_kernel<T, V><<<(unsigned)grid, 256, 0, stream>>>(B * T_, T_, D, as_seq<const T>(x),
                                                          lengths, codes, scales);
  return launch_status();
}

template <class T>
int run_pack(int64_t B, int64_t T_, int64_t D, const semicrf_sequence& x, const int64_t* lengths,
             int8_t* codes, uint8_t* scales, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  if (D % V == 0 && seq_aligned(x, B, T_, sizeof(T), V))
    return launch_pack<T, V>(B, T_, D, x, lengths, codes, scales, stream);
  return launch_pack<T, 1>(B, T_, D, x, lengths, codes, scales, stream);
}

template <class T, int V>
int launch_unpack(int64_t rows, int64_t D, const int8_t* codes, const uint8_t* scales, void* out,
                  cudaStream_t stream) {
  const int64_t n = rows * ((D + V - 1) / V);
  const int64_t grid = (n + 255) / 256;
  if (grid > 0x7fffffff) return SEMICRF_ERR_UNSUPPORTED;
  if (grid)
    unpack_kernel<T, V><<<(unsigned)grid, 256, 0, stream>>>(rows, D, codes, scales,
                                                            static_cast<T*>(out));
  return launch_status();
}

template <class T>
int run_unpack(int64_t rows, int64_t D, const int8_t* codes, const uint8_t* scales, void* out,
               cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  if (D % V == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0)
    return launch_unpack<T, V>(rows, D, codes, scales, out, stream);
  return launch_unpack<T, 1>(rows, D, codes, scales, out, stream);
}

}  // namespace

int pack_rows(int64_t B, int64_t T, int64_t D, int dtype, const semicrf_sequence& x,
              const int64_t* lengths, int8_t* codes, uint8_t* scales, cudaStream_t stream) {
  switch (dtype) {
    case SEMICRF_F32: return run_pack<float>(B, T, D, x, lengths, codes, scales, stream);
    case SEMICRF_BF16: return run_pack<__nv_bfloat16>(B, T, D, x, lengths, codes, scales, stream);
    default: return run_pack<__half>(B, T, D, x, lengths, codes, scales, stream);
  }
}

int unpack_rows(int64_t rows, int64_t D, int dtype, const int8_t* codes, const uint8_t* scales,
                void* out, cudaStream_t stream) {
  switch (dtype) {
    case SEMICRF_F32: return run_unpack<float>(rows, D, codes, scales, out, stream);
    case SEMICRF_BF16: return run_unpack<__nv_bfloat16>(rows, D, codes, scales, out, stream);
    default: return run_unpack<__half>(rows, D, codes, scales, out, stream);
  }
}

}  // namespace semicrf
