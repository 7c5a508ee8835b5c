// packed.cu -- 8-bit activation checkpoints: store and read back.
//
// Both directions are one pass, bound by memory: 2 + 1 + 1/32 bytes an
// element for 16-bit activations.  A lane takes 16 bytes of a row, so the
// lanes of a group of 32 channels are neighbours and its maximum is a few
// shuffles.  A thread keeps its columns and takes 4 rows, all requested
// before the first is used.
//
// Measured, bfloat16, 10^6 x 512: storing 278 us, reading back 265 us, 3.03
// bytes an element at 5.6 and 5.9 TB/s.
//
// Rows that do not start on 16-byte boundaries are packed by the same lanes,
// which load value by value (64 x 5,000 x 203: 65 us; lanes of one value each,
// 182 us).  Reading back, such rows are written by lanes of one value, whose
// neighbours' stores join, 8 rows to a thread (74 us; with 4 rows 88 us; by the
// wide lanes 186 us).

#include <algorithm>
#include <type_traits>

#include "encoder_internal.cuh"

namespace semicrf {
namespace {

constexpr int kThreads = 256;
// rows of a thread: more where its values are single ones (2 and 8 rows of
// vectors or 4 and 16 of single values are slower)
template <int V>
constexpr int kUnroll = V == 1 ? 8 : 4;

// A lane's values, the first `left` of them where rows are not ALIGNED.
template <class T, int V, bool ALIGNED>
__device__ __forceinline__ void load_values(const T* p, int64_t left, Pack<T, V>& q) {
  if (ALIGNED) {
    q = *reinterpret_cast<const Pack<T, V>*>(p);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (k < left) q.v[k] = p[k];
  }
}

// FLAT: every position is valid and all lie at one distance (x.st).
template <class T, int V, bool FLAT, bool ALIGNED>
__global__ void __launch_bounds__(kThreads) pack_kernel(int64_t rows, Places places, int64_t D,
                                                        int64_t G, Seq<const T> x,
                                                        const int64_t* __restrict__ lengths,
                                                        int8_t* __restrict__ codes,
                                                        uint8_t* __restrict__ scales) {
  constexpr int kRows = kUnroll<V>;
  const int64_t first = ((int64_t)blockIdx.x * kRows) * blockDim.y + threadIdx.y;
  const int64_t d = ((int64_t)blockIdx.y * blockDim.x + threadIdx.x) * V;
  const int deep = blockDim.y;
  const int left = (int)min((rows - first + deep - 1) / deep, (int64_t)kRows);  // rows here
  const bool in = d < D;
  Pack<T, V> q[kRows];
  const T* src = x.p + first * x.st + d;
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
#pragma unroll
    for (int k = 0; k < V; ++k) q[u].v[k] = from_f32<T>(0.f);
    if (u < left && in) {
      if (FLAT) {
        load_values<T, V, ALIGNED>(src, D - d, q[u]);
      } else {
        int64_t b, t;
        locate(places, first + u * deep, b, t);
        if (!lengths || t < lengths[b]) load_values<T, V, ALIGNED>(x.row(b, t) + d, D - d, q[u]);
      }
    }
    src += deep * x.st;
  }
  const bool stored = d < G * kPackGroup, opens = d % kPackGroup == 0;
  codes += first * G * kPackGroup + d;
  scales += first * G + d / kPackGroup;
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    Pack<int8_t, V> c;
    const uint8_t byte = pack_encode(q[u], c);  // lanes past the end hold zeros
    if (u < left && stored) {
      *reinterpret_cast<Pack<int8_t, V>*>(codes) = c;
      if (opens) *scales = byte;
    }
    codes += deep * G * kPackGroup;
    scales += deep * G;
  }
}

template <class T, int V>
__global__ void __launch_bounds__(kThreads) unpack_kernel(int64_t rows, int64_t D, int64_t G,
                                                          const int8_t* __restrict__ codes,
                                                          const uint8_t* __restrict__ scales,
                                                          T* __restrict__ out) {
  constexpr int kRows = kUnroll<V>;
  const int64_t first = ((int64_t)blockIdx.x * kRows) * blockDim.y + threadIdx.y;
  const int64_t d = ((int64_t)blockIdx.y * blockDim.x + threadIdx.x) * V;
  const int deep = blockDim.y;
  const int left = (int)min((rows - first + deep - 1) / deep, (int64_t)kRows);  // rows here
  if (d >= D) return;
  Pack<int8_t, V> c[kRows];
  uint8_t byte[kRows];
  codes += first * G * kPackGroup + d;
  scales += first * G + d / kPackGroup;
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    if (u < left) {
      byte[u] = *scales;
      c[u] = *reinterpret_cast<const Pack<int8_t, V>*>(codes);
    }
    codes += deep * G * kPackGroup;
    scales += deep * G;
  }
  out += first * D + d;
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    if (u < left) {
      Pack<T, V> q;
      if constexpr (V == 8 && std::is_same<T, __nv_bfloat16>::value) {
        *reinterpret_cast<uint4*>(&q) = pack_decode(*reinterpret_cast<const uint2*>(&c[u]), byte[u]);
      } else {
        const float unit = pack_scale(byte[u]);
#pragma unroll
        for (int k = 0; k < V; ++k) q.v[k] = from_f32<T>((float)c[u].v[k] * unit);
      }
      *reinterpret_cast<Pack<T, V>*>(out) = q;
    }
    out += deep * D;
  }
}

// A block as wide as a row's lane items (at most 256 of them), with as many
// rows as fill its threads.  Items come in whole groups of 32 channels, so a
// group never straddles two warps.
struct Grid {
  dim3 grid, block;
  bool ok;
};
template <int V>
Grid grid_of(int64_t rows, int64_t G) {
  const int64_t per = G * (kPackGroup / V);
  const unsigned wide = (unsigned)std::min<int64_t>(per, kThreads), deep = kThreads / wide;
  const int64_t across = (per + wide - 1) / wide;
  const int64_t down = (rows + (int64_t)deep * kUnroll<V> - 1) / ((int64_t)deep * kUnroll<V>);
  return Grid{dim3((unsigned)down, (unsigned)across), dim3(wide, deep),
              down <= 0x7fffffff && across <= 65535};
}

template <class T, int V, bool ALIGNED>
int launch_pack(int64_t B, int64_t T_, int64_t D, const semicrf_sequence& x,
                const int64_t* lengths, int8_t* codes, uint8_t* scales, cudaStream_t stream) {
  const int64_t G = pack_groups(D);
  const Grid g = grid_of<V>(B * T_, G);
  if (!g.ok) return SEMICRF_ERR_UNSUPPORTED;
  Seq<const T> xs = as_seq<const T>(x);
  if (!lengths && (B == 1 || T_ == 1 || x.batch_stride == T_ * x.time_stride)) {
    if (T_ == 1) xs.st = xs.sb;
    pack_kernel<T, V, true, ALIGNED>
        <<<g.grid, g.block, 0, stream>>>(B * T_, Places{}, D, G, xs, nullptr, codes, scales);
  } else {
    pack_kernel<T, V, false, ALIGNED><<<g.grid, g.block, 0, stream>>>(
        B * T_, make_places(B, T_), D, G, xs, lengths, codes, scales);
  }
  return launch_status();
}

template <class T>
int run_pack(int64_t B, int64_t T_, int64_t D, const semicrf_sequence& x, const int64_t* lengths,
             int8_t* codes, uint8_t* scales, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  if (D % V == 0 && seq_aligned(x, B, T_, sizeof(T), V))
    return launch_pack<T, V, true>(B, T_, D, x, lengths, codes, scales, stream);
  return launch_pack<T, V, false>(B, T_, D, x, lengths, codes, scales, stream);
}

template <class T, int V>
int launch_unpack(int64_t rows, int64_t D, const int8_t* codes, const uint8_t* scales, void* out,
                  cudaStream_t stream) {
  const int64_t G = pack_groups(D);
  const Grid g = grid_of<V>(rows, G);
  if (!g.ok) return SEMICRF_ERR_UNSUPPORTED;
  unpack_kernel<T, V>
      <<<g.grid, g.block, 0, stream>>>(rows, D, G, codes, scales, static_cast<T*>(out));
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
