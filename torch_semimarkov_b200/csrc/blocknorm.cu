// blocknorm.cu -- the norms around a block fused with its gate, its residual
// scale and the residual sum, forward and backward.
//
//   zh = z / rms(z),  b = zh w1,  r = x + s silu(g) b,  rh = r / rms(r),  n = rh w2
//
// Gradient, with D the row's width and sums over it:
//   d  = dr + (dn w2 - rh sum(dn w2 rh) / D) / rms(r)     (= dx)
//   db = d s silu(g),  dg = d s b silu'(g)
//   dz = (db w1 - zh sum(db w1 zh) / D) / rms(z)
//   dw1 = sum_rows db zh,  ds = sum_rows d silu(g) b,  dw2 = sum_rows dn rh
//
// A row lies in the registers of WR warps, PER channels to a lane, so each
// input is read once.  The backward recomputes r from the block's inputs in
// 32 bits; it reads x where it would else read the rounded r.  Weight
// gradients are summed per thread over the rows that its CTA walks, then over
// the CTAs in a fixed order: no atomics.

#include <algorithm>

#include "encoder_internal.cuh"

namespace semicrf {
int device_sm_count();  // api.cu

namespace {

template <class T>
struct NormArgs {
  int64_t rows, T_, D;
  float eps, inv_d;
  Seq<const T> x, z, g;
  Seq<T> r, n;
  const float *w1, *s, *w2;
  const int64_t* lengths;
  float* stats;
  int8_t* codes;
  uint8_t* scales;
  Seq<const T> dr, dn;
  Seq<T> dx, dz, dg;
  float* partial;  // (grid, 3, D)
};

// Sums over the row's lanes; every lane gets the result.  `red` alternates
// between two slots, so one barrier per sum is enough.
template <int WR>
struct RowSum {
  float (*red)[WR];
  int slot, w, lane, barrier;
  __device__ __forceinline__ float operator()(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    if (WR > 1) {
      slot ^= 1;
      if (lane == 0) red[slot][w] = v;
      asm volatile("bar.sync %0, %1;" ::"r"(barrier), "n"(32 * WR) : "memory");
      v = 0.f;
#pragma unroll
      for (int k = 0; k < WR; ++k) v += red[slot][k];
    }
    return v;
  }
};

template <class T, int V, int WR, int PER>
struct Layout {
  static constexpr int J = PER / V;                      // vectors of a lane
  static constexpr int kRows = WR >= 4 ? 1 : 4 / WR;     // rows that a CTA works on at once
  static constexpr int kThreads = 32 * WR * kRows;
};

template <class T, int V>
__device__ __forceinline__ void get(const T* row, int64_t d, bool ok, float (&v)[V]) {
  Pack<T, V> q;
  if (ok) q = *reinterpret_cast<const Pack<T, V>*>(row + d);
#pragma unroll
  for (int k = 0; k < V; ++k) v[k] = ok ? to_f32(q.v[k]) : 0.f;
}
template <class T, int V>
__device__ __forceinline__ void put(T* row, int64_t d, bool ok, const float (&v)[V]) {
  if (!ok) return;
  Pack<T, V> q;
#pragma unroll
  for (int k = 0; k < V; ++k) q.v[k] = from_f32<T>(v[k]);
  *reinterpret_cast<Pack<T, V>*>(row + d) = q;
}
template <int V>
__device__ __forceinline__ void weights(const float* w, int64_t d, bool ok, float (&v)[V]) {
#pragma unroll
  for (int k = 0; k < V; ++k) v[k] = ok && w ? w[d + k] : 0.f;
}

template <class T, int V, int WR, int PER, bool BRANCH>
__global__ void __launch_bounds__(Layout<T, V, WR, PER>::kThreads) norm_forward_kernel(NormArgs<T> a) {
  using L = Layout<T, V, WR, PER>;
  constexpr int J = L::J;
  __shared__ float red[L::kRows][2][WR];
  const int group = threadIdx.x / (32 * WR), l = threadIdx.x % (32 * WR);
  RowSum<WR> row_sum{red[group], 0, l >> 5, l & 31, 1 + group};
  const int64_t G = pack_groups(a.D);
  int64_t d[J];
  bool ok[J];
#pragma unroll
  for (int j = 0; j < J; ++j) d[j] = (int64_t)(j * 32 * WR + l) * V, ok[j] = d[j] < a.D;

  for (int64_t row = (int64_t)blockIdx.x * L::kRows + group; row < a.rows;
       row += (int64_t)gridDim.x * L::kRows) {
    const int64_t b = row / a.T_, t = row - b * a.T_;
    const bool live = t < valid_length(a.lengths, b, a.T_);
    float r[J][V];
    float rz = 0.f;
#pragma unroll
    for (int j = 0; j < J; ++j) get<T, V>(a.x.row(b, t), d[j], ok[j] && live, r[j]);
    if (BRANCH) {
      float z[J][V], g[J][V];
      float q = 0.f;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        get<T, V>(a.z.row(b, t), d[j], ok[j] && live, z[j]);
        get<T, V>(a.g.row(b, t), d[j], ok[j] && live, g[j]);
      }
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int k = 0; k < V; ++k) q = fmaf(z[j][k], z[j][k], q);
      rz = rsqrtf(row_sum(q) * a.inv_d + a.eps);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        float w1[V], sc[V];
        weights<V>(a.w1, d[j], ok[j], w1);
        weights<V>(a.s, d[j], ok[j], sc);
#pragma unroll
        for (int k = 0; k < V; ++k) {
          float sig, neg;
          sigmoid_pair(g[j][k], sig, neg);
          r[j][k] = fmaf(sc[k] * (g[j][k] * sig), z[j][k] * rz * w1[k], r[j][k]);
        }
      }
    }
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int k = 0; k < V; ++k) q = fmaf(r[j][k], r[j][k], q);
    const float rr = rsqrtf(row_sum(q) * a.inv_d + a.eps);
    if (a.stats && l == 0) {
      a.stats[2 * row] = rz;
      a.stats[2 * row + 1] = rr;
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
      float w2[V], n[V];
      weights<V>(a.w2, d[j], ok[j], w2);
      if (BRANCH) put<T, V>(a.r.row(b, t), d[j], ok[j], r[j]);
#pragma unroll
      for (int k = 0; k < V; ++k) n[k] = live ? r[j][k] * rr * w2[k] : 0.f;
      put<T, V>(a.n.row(b, t), d[j], ok[j], n);
      if (a.codes) {  // the checkpoint holds what n holds after rounding
        Pack<int8_t, V> c;
        Pack<T, V> rounded;
#pragma unroll
        for (int k = 0; k < V; ++k) rounded.v[k] = from_f32<T>(ok[j] ? n[k] : 0.f);
        const uint8_t byte = pack_encode(rounded, c);
        if (d[j] < G * kPackGroup) {
          *reinterpret_cast<Pack<int8_t, V>*>(a.codes + row * G * kPackGroup + d[j]) = c;
          if (d[j] % kPackGroup == 0) a.scales[row * G + d[j] / kPackGroup] = byte;
        }
      }
    }
  }
}

template <class T, int V, int WR, int PER, bool BRANCH>
__global__ void __launch_bounds__(Layout<T, V, WR, PER>::kThreads) norm_backward_kernel(NormArgs<T> a) {
  using L = Layout<T, V, WR, PER>;
  constexpr int J = L::J;
  __shared__ float red[L::kRows][2][WR];
  __shared__ float sums[L::kRows > 1 ? 32 * WR * PER : 1];
  const int group = threadIdx.x / (32 * WR), l = threadIdx.x % (32 * WR);
  RowSum<WR> row_sum{red[group], 0, l >> 5, l & 31, 1 + group};
  int64_t d[J];
  bool ok[J];
#pragma unroll
  for (int j = 0; j < J; ++j) d[j] = (int64_t)(j * 32 * WR + l) * V, ok[j] = d[j] < a.D;
  float acc[3][J][V];
#pragma unroll
  for (int m = 0; m < 3; ++m)
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int k = 0; k < V; ++k) acc[m][j][k] = 0.f;

  for (int64_t row = (int64_t)blockIdx.x * L::kRows + group; row < a.rows;
       row += (int64_t)gridDim.x * L::kRows) {
    const int64_t b = row / a.T_, t = row - b * a.T_;
    const bool live = t < valid_length(a.lengths, b, a.T_);
    const float zero[V] = {};
    if (!live) {  // the whole row group takes this branch together
#pragma unroll
      for (int j = 0; j < J; ++j) {
        put<T, V>(a.dx.row(b, t), d[j], ok[j], zero);
        if (BRANCH) {
          put<T, V>(a.dz.row(b, t), d[j], ok[j], zero);
          put<T, V>(a.dg.row(b, t), d[j], ok[j], zero);
        }
      }
      continue;
    }
    const float rz = a.stats[2 * row], rr = a.stats[2 * row + 1];
    float r[J][V], z[J][V], g[J][V], dn[J][V], dr[J][V];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      get<T, V>(a.x.row(b, t), d[j], ok[j], r[j]);
      if (BRANCH) {
        get<T, V>(a.z.row(b, t), d[j], ok[j], z[j]);
        get<T, V>(a.g.row(b, t), d[j], ok[j], g[j]);
      }
      get<T, V>(a.dn.p ? a.dn.row(b, t) : nullptr, d[j], ok[j] && a.dn.p, dn[j]);
      get<T, V>(a.dr.p ? a.dr.row(b, t) : nullptr, d[j], ok[j] && a.dr.p, dr[j]);
    }
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      float w1[V], sc[V], w2[V];
      weights<V>(a.w2, d[j], ok[j], w2);
      if (BRANCH) {
        weights<V>(a.w1, d[j], ok[j], w1);
        weights<V>(a.s, d[j], ok[j], sc);
      }
#pragma unroll
      for (int k = 0; k < V; ++k) {
        if (BRANCH) {
          float sig, neg;
          sigmoid_pair(g[j][k], sig, neg);
          z[j][k] *= rz;
          r[j][k] = fmaf(sc[k] * (g[j][k] * sig), z[j][k] * w1[k], r[j][k]);
        }
        r[j][k] *= rr;  // rh
        acc[2][j][k] = fmaf(dn[j][k], r[j][k], acc[2][j][k]);
        dn[j][k] *= w2[k];
        q = fmaf(dn[j][k], r[j][k], q);
      }
    }
    const float c2 = row_sum(q) * a.inv_d;
    q = 0.f;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      float w1[V], sc[V];
      if (BRANCH) {
        weights<V>(a.w1, d[j], ok[j], w1);
        weights<V>(a.s, d[j], ok[j], sc);
      }
      float dg[V];
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float dd = fmaf(rr, dn[j][k] - r[j][k] * c2, dr[j][k]);
        dr[j][k] = dd;
        if (BRANCH) {
          float sig, neg;
          sigmoid_pair(g[j][k], sig, neg);
          const float u = g[j][k] * sig, bn = z[j][k] * w1[k];
          const float db = dd * sc[k] * u;
          acc[0][j][k] = fmaf(db, z[j][k], acc[0][j][k]);
          acc[1][j][k] = fmaf(dd * u, bn, acc[1][j][k]);
          dg[k] = dd * sc[k] * bn * sig * fmaf(g[j][k], neg, 1.f);
          dn[j][k] = db * w1[k];  // the row's db w1 takes dn's place
          q = fmaf(dn[j][k], z[j][k], q);
        }
      }
      put<T, V>(a.dx.row(b, t), d[j], ok[j], dr[j]);
      if (BRANCH) put<T, V>(a.dg.row(b, t), d[j], ok[j], dg);
    }
    if (BRANCH) {
      const float c1 = row_sum(q) * a.inv_d;
#pragma unroll
      for (int j = 0; j < J; ++j) {
#pragma unroll
        for (int k = 0; k < V; ++k) dn[j][k] = rz * (dn[j][k] - z[j][k] * c1);
        put<T, V>(a.dz.row(b, t), d[j], ok[j], dn[j]);
      }
    }
  }

  // the CTA's sums, its row groups added in order
#pragma unroll
  for (int m = BRANCH ? 0 : 2; m < 3; ++m) {
    if (L::kRows > 1) {
      for (int turn = L::kRows - 1; turn > 0; --turn) {
        __syncthreads();
        if (group == turn)
#pragma unroll
          for (int j = 0; j < J; ++j)
#pragma unroll
            for (int k = 0; k < V; ++k) sums[(j * V + k) * 32 * WR + l] = acc[m][j][k];
        __syncthreads();
        if (group == turn - 1)
#pragma unroll
          for (int j = 0; j < J; ++j)
#pragma unroll
            for (int k = 0; k < V; ++k) acc[m][j][k] += sums[(j * V + k) * 32 * WR + l];
      }
    }
    if (group == 0)
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int k = 0; k < V; ++k)
          if (ok[j]) a.partial[((int64_t)blockIdx.x * 3 + m) * a.D + d[j] + k] = acc[m][j][k];
  }
}

// Sums the CTAs' partials in a fixed order: a block takes 32 channels, its
// eight rows of threads every eighth CTA.
__global__ void norm_reduce_kernel(int64_t D, int first, int ctas,
                                   const float* __restrict__ partial, float* __restrict__ out) {
  __shared__ float part[8][33];
  const int64_t n = (int64_t)blockIdx.x * 32 + threadIdx.x + first * D;
  float s = 0.f;
  if (n < 3 * D)
    for (int c = threadIdx.y; c < ctas; c += 8) s += partial[(int64_t)c * 3 * D + n];
  part[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y || n >= 3 * D) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) s += part[k][threadIdx.x];
  out[n] = s;
}

template <class T>
NormArgs<T> norm_args(const semicrf_block_norm* p) {
  NormArgs<T> a{};
  a.rows = p->batch * p->T;
  a.T_ = p->T;
  a.D = p->D;
  a.eps = p->eps;
  a.inv_d = 1.f / (float)p->D;
  a.x = as_seq<const T>(p->residual);
  a.z = as_seq<const T>(p->branch);
  a.g = as_seq<const T>(p->gate);
  a.w1 = p->branch_weight;
  a.s = p->residual_scale;
  a.w2 = p->next_weight;
  a.lengths = p->lengths;
  return a;
}

int64_t backward_ctas(int64_t rows, int at_once) {
  const int64_t all = (rows + at_once - 1) / at_once;
  return std::max<int64_t>(1, std::min<int64_t>(all, 4 * device_sm_count()));
}

template <class T, int V, int WR, int PER, bool BRANCH>
int launch(const NormArgs<T>& a, bool backward, float* grad_weights, cudaStream_t stream) {
  using L = Layout<T, V, WR, PER>;
  if (!backward) {
    const int64_t all = (a.rows + L::kRows - 1) / L::kRows;
    const unsigned grid = (unsigned)std::min<int64_t>(all, 16 * device_sm_count());
    if (grid) norm_forward_kernel<T, V, WR, PER, BRANCH><<<grid, L::kThreads, 0, stream>>>(a);
    return launch_status();
  }
  const int ctas = (int)backward_ctas(a.rows, L::kRows);
  norm_backward_kernel<T, V, WR, PER, BRANCH><<<ctas, L::kThreads, 0, stream>>>(a);
  const int first = BRANCH ? 0 : 2;
  const unsigned rg = (unsigned)(((3 - first) * a.D + 31) / 32);
  norm_reduce_kernel<<<rg, dim3(32, 8), 0, stream>>>(a.D, first, ctas, a.partial, grad_weights);
  return launch_status();
}

// The fewest warps whose registers hold a row: up to 16 channels a lane.
template <class T, int V, bool BRANCH>
int launch_width(const NormArgs<T>& a, bool backward, float* gw, cudaStream_t s) {
  if (a.D <= 256) return launch<T, V, 1, 8, BRANCH>(a, backward, gw, s);
  if (a.D <= 512) return launch<T, V, 1, 16, BRANCH>(a, backward, gw, s);
  if (a.D <= 1024) return launch<T, V, 2, 16, BRANCH>(a, backward, gw, s);
  if (a.D <= 2048) return launch<T, V, 4, 16, BRANCH>(a, backward, gw, s);
  if (a.D <= 4096) return launch<T, V, 8, 16, BRANCH>(a, backward, gw, s);
  return launch<T, V, 16, 16, BRANCH>(a, backward, gw, s);
}

template <class T>
int launch_type(const NormArgs<T>& a, bool vec, bool branch, bool backward, float* gw,
                cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  if (branch)
    return vec ? launch_width<T, V, true>(a, backward, gw, s)
               : launch_width<T, 1, true>(a, backward, gw, s);
  return vec ? launch_width<T, V, false>(a, backward, gw, s)
             : launch_width<T, 1, false>(a, backward, gw, s);
}

template <class T>
int run_forward(const semicrf_block_norm* p, const semicrf_sequence& r, const semicrf_sequence& n,
                float* stats, int8_t* codes, uint8_t* scales, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  NormArgs<T> a = norm_args<T>(p);
  a.r = as_seq<T>(r);
  a.n = as_seq<T>(n);
  a.stats = stats;
  a.codes = codes;
  a.scales = scales;
  bool vec = p->D % V == 0;
  for (const semicrf_sequence* s : {&p->residual, &p->branch, &p->gate, &r, &n})
    vec = vec && seq_aligned(*s, p->batch, p->T, sizeof(T), V);
  return launch_type<T>(a, vec, p->branch.data != nullptr, false, nullptr, stream);
}

template <class T>
int run_backward(const semicrf_block_norm* p, const float* stats, const semicrf_sequence& dr,
                 const semicrf_sequence& dn, const semicrf_sequence& dx,
                 const semicrf_sequence& dz, const semicrf_sequence& dg, float* grad_weights,
                 void* workspace, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  NormArgs<T> a = norm_args<T>(p);
  a.stats = const_cast<float*>(stats);
  a.dr = as_seq<const T>(dr);
  a.dn = as_seq<const T>(dn);
  a.dx = as_seq<T>(dx);
  a.dz = as_seq<T>(dz);
  a.dg = as_seq<T>(dg);
  a.partial = static_cast<float*>(workspace);
  bool vec = p->D % V == 0;
  for (const semicrf_sequence* s : {&p->residual, &p->branch, &p->gate, &dr, &dn, &dx, &dz, &dg})
    vec = vec && seq_aligned(*s, p->batch, p->T, sizeof(T), V);
  return launch_type<T>(a, vec, p->branch.data != nullptr, true, grad_weights, stream);
}

}  // namespace

size_t block_norm_workspace_bytes(const semicrf_block_norm* p) {
  // at most one CTA a row, whatever the layout
  return sizeof(float) * 3 * p->D * backward_ctas(p->batch * p->T, 1);
}

int block_norm_forward(const semicrf_block_norm* p, const semicrf_sequence& r,
                       const semicrf_sequence& n, float* stats, int8_t* codes, uint8_t* scales,
                       cudaStream_t stream) {
  switch (p->dtype) {
    case SEMICRF_F32: return run_forward<float>(p, r, n, stats, codes, scales, stream);
    case SEMICRF_BF16: return run_forward<__nv_bfloat16>(p, r, n, stats, codes, scales, stream);
    default: return run_forward<__half>(p, r, n, stats, codes, scales, stream);
  }
}

int block_norm_backward(const semicrf_block_norm* p, const float* stats,
                        const semicrf_sequence& dr, const semicrf_sequence& dn,
                        const semicrf_sequence& dx, const semicrf_sequence& dz,
                        const semicrf_sequence& dg, float* grad_weights, void* workspace,
                        cudaStream_t stream) {
  switch (p->dtype) {
    case SEMICRF_F32:
      return run_backward<float>(p, stats, dr, dn, dx, dz, dg, grad_weights, workspace, stream);
    case SEMICRF_BF16:
      return run_backward<__nv_bfloat16>(p, stats, dr, dn, dx, dz, dg, grad_weights, workspace,
                                         stream);
    default:
      return run_backward<__half>(p, stats, dr, dn, dx, dz, dg, grad_weights, workspace, stream);
  }
}

}  // namespace semicrf
