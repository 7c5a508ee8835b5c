// packgrad.cu -- the gradient of a linear layer's weight from the 8-bit
// checkpoint of its input: out (M, D) = sum_n dy[n, :]^T x[n, :].
//
// A CTA of 256 threads owns 64 x 64 outputs and a run of positions, 4 x 4
// outputs to a thread; runs are summed by a second kernel in order.

#include <algorithm>

#include "encoder_internal.cuh"

namespace semicrf {
int device_sm_count();  // api.cu

namespace {

constexpr int kTileOut = 64, kStep = 16;

template <class T>
__global__ void __launch_bounds__(256) weight_grad_kernel(int64_t N, int64_t T_, int64_t D, int64_t M,
                                                          int64_t run, Seq<const T> dy,
                                                          const int8_t* __restrict__ codes,
                                                          const uint8_t* __restrict__ scales,
                                                          const int64_t* __restrict__ lengths,
                                                          float* __restrict__ partial) {
  __shared__ float a[kStep][kTileOut], x[kStep][kTileOut];
  const int64_t m0 = (int64_t)blockIdx.x * kTileOut, d0 = (int64_t)blockIdx.y * kTileOut;
  const int64_t G = pack_groups(D);
  const int64_t first = blockIdx.z * run, last = first + run < N ? first + run : N;
  const int c = threadIdx.x & 63, r = threadIdx.x >> 6;
  const int tm = (threadIdx.x >> 4) * 4, td = (threadIdx.x & 15) * 4;
  float acc[4][4] = {};
  for (int64_t n0 = first; n0 < last; n0 += kStep) {
#pragma unroll
    for (int k = 0; k < kStep; k += 4) {
      const int64_t n = n0 + k + r;
      float va = 0.f, vx = 0.f;
      if (n < last) {
        const int64_t b = n / T_, t = n - b * T_;
        if (t < valid_length(lengths, b, T_)) {
          if (m0 + c < M) va = to_f32(dy.row(b, t)[m0 + c]);
          if (d0 + c < D)
            vx = (float)codes[n * G * kPackGroup + d0 + c] *
                 pack_scale(scales[n * G + (d0 + c) / kPackGroup]);
        }
      }
      a[k + r][c] = va;
      x[k + r][c] = vx;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kStep; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(a[k][tm + i], x[k][td + j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j)
      if (m0 + tm + i < M && d0 + td + j < D)
        partial[(blockIdx.z * M + m0 + tm + i) * D + d0 + td + j] = acc[i][j];
}

template <class O>
__global__ void sum_runs_kernel(int64_t n, int runs, const float* __restrict__ partial,
                                O* __restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  float s = 0.f;
  for (int k = 0; k < runs; ++k) s += partial[k * n + i];
  out[i] = from_f32<O>(s);
}

int runs_of(int64_t N, int64_t D, int64_t M) {
  const int64_t tiles = ((M + kTileOut - 1) / kTileOut) * ((D + kTileOut - 1) / kTileOut);
  const int64_t want = std::max<int64_t>(1, 4 * device_sm_count() / tiles);
  return (int)std::min<int64_t>(want, std::max<int64_t>(1, N / 256));
}

template <class T>
int run(int64_t B, int64_t T_, int64_t D, int64_t M, const semicrf_sequence& dy,
        const int8_t* codes, const uint8_t* scales, const int64_t* lengths, int out_dtype,
        void* out, void* workspace, cudaStream_t stream) {
  const int64_t N = B * T_;
  const int runs = runs_of(N, D, M);
  const int64_t run_len = N ? (N + runs - 1) / runs : 0;
  float* partial = static_cast<float*>(workspace);
  const dim3 grid((unsigned)((M + kTileOut - 1) / kTileOut),
                  (unsigned)((D + kTileOut - 1) / kTileOut), (unsigned)runs);
  weight_grad_kernel<T><<<grid, 256, 0, stream>>>(N, T_, D, M, run_len, as_seq<const T>(dy), codes,
                                                  scales, lengths, partial);
  const unsigned sg = (unsigned)((M * D + 255) / 256);
  switch (out_dtype) {
    case SEMICRF_F32:
      sum_runs_kernel<<<sg, 256, 0, stream>>>(M * D, runs, partial, static_cast<float*>(out));
      break;
    case SEMICRF_BF16:
      sum_runs_kernel<<<sg, 256, 0, stream>>>(M * D, runs, partial,
                                              static_cast<__nv_bfloat16*>(out));
      break;
    default:
      sum_runs_kernel<<<sg, 256, 0, stream>>>(M * D, runs, partial, static_cast<__half*>(out));
  }
  return launch_status();
}

}  // namespace

size_t packed_weight_grad_workspace_bytes(int64_t B, int64_t T, int64_t D, int64_t M, int) {
  return sizeof(float) * M * D * runs_of(B * T, D, M);
}

int packed_weight_grad(int64_t B, int64_t T, int64_t D, int64_t M, int dtype,
                       const semicrf_sequence& dy, const int8_t* codes, const uint8_t* scales,
                       const int64_t* lengths, int out_dtype, void* out, void* workspace,
                       cudaStream_t stream) {
  switch (dtype) {
    case SEMICRF_F32:
      return run<float>(B, T, D, M, dy, codes, scales, lengths, out_dtype, out, workspace, stream);
    case SEMICRF_BF16:
      return run<__nv_bfloat16>(B, T, D, M, dy, codes, scales, lengths, out_dtype, out, workspace,
                                stream);
    default:
      return run<__half>(B, T, D, M, dy, codes, scales, lengths, out_dtype, out, workspace, stream);
  }
}

}  // namespace semicrf
