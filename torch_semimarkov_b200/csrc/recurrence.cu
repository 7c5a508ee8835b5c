// recurrence.cu -- the gated linear recurrence, its gradient and its
// single-position form.
//
//   f = sigmoid(g),  h_u = f_u h_{u-1} + (1 - f_u) x_u
//
// u counts positions in scan order (t = u, or T-1-u when reversed); masked
// positions have f = 1 and contribute nothing, so they pass the state on.
// Steps compose: (P, S) with h_out = P h_in + S, P the product of f, S the
// result from zero.  f <= 1, so nothing overflows and no logarithm is needed.
//
// Gradient: lam_u = dh_u + f_{u+1} lam_{u+1}.  With mu_u = f_u lam_u it is
// the same recurrence from the other end, mu_u = f_u (dh_u + mu_{u+1}), and
//   dx_u = lam_u (1 - f_u),  dg_u = lam_u (h_{u-1} - x_u) f_u (1 - f_u).
// h_{u-1} is recomputed from the float32 state kept at the start of each
// chunk, which is more exact than rereading the rounded h and one read less.
//
// The time axis is cut into chunks of kChunk positions.  A CTA of kWarps
// warps owns one chunk of kTile channels: a warp owns kRun consecutive
// positions, a lane two channels.  One pass composes each chunk, one joins
// the chunks in order, one writes the outputs.

#include "encoder_internal.cuh"

namespace semicrf {
namespace {

constexpr int kRun = 8;                 // positions of a thread
constexpr int kWarps = 8;               // threads along time
constexpr int kChunk = kRun * kWarps;   // positions of a CTA
constexpr int kLane = 2;                // channels of a thread
constexpr int kTile = 32 * kLane;       // channels of a CTA

template <class T>
struct ScanArgs {
  int64_t B, T_, D, chunks, tiles;
  bool reverse;
  Seq<const T> x, g, dh;
  Seq<T> h, dx, dg;
  const int64_t* lengths;
  float2* agg;    // (B, chunks, D): a chunk's (P, S)
  float* carry;   // (B, chunks, D): the state entering each chunk (forward)
  float* gcarry;  // (B, chunks, D): mu entering each chunk from its successor (backward)
};

// Where a CTA works: its sequence, chunk and channels.
template <bool VEC>
struct Place {
  int64_t b, c, u0, len;
  int d[kLane];
  bool ok[kLane];
  int lane, w;
  template <class T>
  __device__ Place(const ScanArgs<T>& a) {
    const int64_t id = blockIdx.x;
    const int64_t tile = id % a.tiles;
    c = (id / a.tiles) % a.chunks;
    b = id / a.tiles / a.chunks;
    lane = threadIdx.x & 31;
    w = threadIdx.x >> 5;
    u0 = c * kChunk + w * kRun;
    len = valid_length(a.lengths, b, a.T_);
#pragma unroll
    for (int j = 0; j < kLane; ++j) {
      d[j] = (int)(tile * kTile) + (VEC ? lane * kLane + j : lane + 32 * j);
      ok[j] = d[j] < a.D;
    }
  }
  template <class T>
  __device__ int64_t time(const ScanArgs<T>& a, int i) const {
    return a.reverse ? a.T_ - 1 - (u0 + i) : u0 + i;
  }
  __device__ bool valid(int64_t t) const { return t >= 0 && t < len; }
};

template <bool VEC, class T>
__device__ __forceinline__ void load_row(const T* row, const int (&d)[kLane], const bool (&ok)[kLane],
                                         bool live, float (&v)[kLane]) {
  if (VEC) {
    Pack<T, kLane> q;
    if (live && ok[0]) {
      q = *reinterpret_cast<const Pack<T, kLane>*>(row + d[0]);
#pragma unroll
      for (int j = 0; j < kLane; ++j) v[j] = to_f32(q.v[j]);
    } else {
#pragma unroll
      for (int j = 0; j < kLane; ++j) v[j] = 0.f;
    }
  } else {
#pragma unroll
    for (int j = 0; j < kLane; ++j) v[j] = live && ok[j] ? to_f32(row[d[j]]) : 0.f;
  }
}

template <bool VEC, class T>
__device__ __forceinline__ void store_row(T* row, const int (&d)[kLane], const bool (&ok)[kLane],
                                          const float (&v)[kLane]) {
  if (VEC) {
    if (!ok[0]) return;
    Pack<T, kLane> q;
#pragma unroll
    for (int j = 0; j < kLane; ++j) q.v[j] = from_f32<T>(v[j]);
    *reinterpret_cast<Pack<T, kLane>*>(row + d[0]) = q;
  } else {
#pragma unroll
    for (int j = 0; j < kLane; ++j)
      if (ok[j]) row[d[j]] = from_f32<T>(v[j]);
  }
}

// Composes a chunk: (P, S) of the forward state, or with BWD of mu.
template <class T, bool VEC, bool BWD>
__global__ void __launch_bounds__(32 * kWarps) compose_kernel(ScanArgs<T> a) {
  const Place<VEC> at(a);
  __shared__ float2 part[kWarps][kTile];
  float P[kLane], S[kLane];
#pragma unroll
  for (int j = 0; j < kLane; ++j) P[j] = 1.f, S[j] = 0.f;
#pragma unroll
  for (int k = 0; k < kRun; ++k) {
    const int i = BWD ? kRun - 1 - k : k;
    const int64_t t = at.time(a, i);
    if (!at.valid(t)) continue;
    float v[kLane], g[kLane];
    load_row<VEC>(BWD ? a.dh.p ? a.dh.row(at.b, t) : nullptr : a.x.row(at.b, t), at.d, at.ok,
                  !BWD || a.dh.p, v);
    load_row<VEC>(a.g.row(at.b, t), at.d, at.ok, true, g);
#pragma unroll
    for (int j = 0; j < kLane; ++j) {
      float f, n;
      sigmoid_pair(g[j], f, n);
      P[j] *= f;
      S[j] = BWD ? f * (v[j] + S[j]) : fmaf(f, S[j], n * v[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < kLane; ++j) part[at.w][at.lane + 32 * j] = make_float2(P[j], S[j]);
  __syncthreads();
  if (at.w) return;
#pragma unroll
  for (int j = 0; j < kLane; ++j) {
    float p = 1.f, s = 0.f;
    for (int w = 0; w < kWarps; ++w) {
      const float2 q = part[BWD ? kWarps - 1 - w : w][at.lane + 32 * j];
      s = fmaf(q.x, s, q.y);
      p *= q.x;
    }
    if (at.ok[j]) a.agg[(at.b * a.chunks + at.c) * a.D + at.d[j]] = make_float2(p, s);
  }
}

// Joins the chunks of a channel in order.
__global__ void join_kernel(int64_t B, int64_t chunks, int64_t D, bool descending,
                            const float2* __restrict__ agg, const float* __restrict__ first,
                            float* __restrict__ carry, float* __restrict__ last) {
  const int64_t n = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (n >= B * D) return;
  const int64_t base = n / D * chunks * D + n % D;
  float s = first ? first[n] : 0.f;
#pragma unroll 8
  for (int64_t k = 0; k < chunks; ++k) {
    const int64_t i = base + (descending ? chunks - 1 - k : k) * D;
    carry[i] = s;
    const float2 q = agg[i];
    s = fmaf(q.x, s, q.y);
  }
  if (last) last[n] = s;
}

template <class T, bool VEC>
__global__ void __launch_bounds__(32 * kWarps) forward_kernel(ScanArgs<T> a) {
  const Place<VEC> at(a);
  __shared__ float2 part[kWarps][kTile];
  float f[kRun][kLane], b[kRun][kLane];
  float P[kLane], S[kLane];
#pragma unroll
  for (int j = 0; j < kLane; ++j) P[j] = 1.f, S[j] = 0.f;
#pragma unroll
  for (int i = 0; i < kRun; ++i) {
    const int64_t t = at.time(a, i);
    const bool live = at.valid(t);
    float x[kLane], g[kLane];
    load_row<VEC>(a.x.row(at.b, t), at.d, at.ok, live, x);
    load_row<VEC>(a.g.row(at.b, t), at.d, at.ok, live, g);
#pragma unroll
    for (int j = 0; j < kLane; ++j) {
      float n;
      sigmoid_pair(g[j], f[i][j], n);
      b[i][j] = live ? n * x[j] : 0.f;
      if (!live) f[i][j] = 1.f;
      P[j] *= f[i][j];
      S[j] = fmaf(f[i][j], S[j], b[i][j]);
    }
  }
#pragma unroll
  for (int j = 0; j < kLane; ++j) part[at.w][at.lane + 32 * j] = make_float2(P[j], S[j]);
  __syncthreads();
  float s[kLane];
#pragma unroll
  for (int j = 0; j < kLane; ++j) {
    s[j] = at.ok[j] ? a.carry[(at.b * a.chunks + at.c) * a.D + at.d[j]] : 0.f;
    for (int w = 0; w < at.w; ++w) {
      const float2 q = part[w][at.lane + 32 * j];
      s[j] = fmaf(q.x, s[j], q.y);
    }
  }
#pragma unroll
  for (int i = 0; i < kRun; ++i) {
    const int64_t t = at.time(a, i);
    if (t < 0 || t >= a.T_) continue;
    float out[kLane];
#pragma unroll
    for (int j = 0; j < kLane; ++j) {
      s[j] = fmaf(f[i][j], s[j], b[i][j]);
      out[j] = at.valid(t) ? s[j] : 0.f;
    }
    store_row<VEC>(a.h.row(at.b, t), at.d, at.ok, out);
  }
}

template <class T, bool VEC>
__global__ void __launch_bounds__(32 * kWarps) backward_kernel(ScanArgs<T> a) {
  const Place<VEC> at(a);
  __shared__ float2 part[kWarps][kTile];
  __shared__ float gpart[kWarps][kTile];
  float f[kRun][kLane], n[kRun][kLane], x[kRun][kLane], dh[kRun][kLane];
  float P[kLane], S[kLane];
#pragma unroll
  for (int j = 0; j < kLane; ++j) P[j] = 1.f, S[j] = 0.f;
#pragma unroll
  for (int i = 0; i < kRun; ++i) {
    const int64_t t = at.time(a, i);
    const bool live = at.valid(t);
    float g[kLane];
    load_row<VEC>(a.x.row(at.b, t), at.d, at.ok, live, x[i]);
    load_row<VEC>(a.g.row(at.b, t), at.d, at.ok, live, g);
    load_row<VEC>(a.dh.p ? a.dh.row(at.b, t) : nullptr, at.d, at.ok, live && a.dh.p, dh[i]);
#pragma unroll
    for (int j = 0; j < kLane; ++j) {
      sigmoid_pair(g[j], f[i][j], n[i][j]);
      if (!live) f[i][j] = 1.f, n[i][j] = 0.f;
      P[j] *= f[i][j];
      S[j] = fmaf(f[i][j], S[j], n[i][j] * x[i][j]);
    }
  }
#pragma unroll
  for (int j = 0; j < kLane; ++j) {
    float m = 0.f;
#pragma unroll
    for (int i = kRun - 1; i >= 0; --i) m = f[i][j] * (dh[i][j] + m);
    part[at.w][at.lane + 32 * j] = make_float2(P[j], S[j]);
    gpart[at.w][at.lane + 32 * j] = m;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kLane; ++j) {
    const int64_t k = (at.b * a.chunks + at.c) * a.D + at.d[j];
    float s = at.ok[j] ? a.carry[k] : 0.f;
    float mu = at.ok[j] ? a.gcarry[k] : 0.f;
    for (int w = 0; w < at.w; ++w) {
      const float2 q = part[w][at.lane + 32 * j];
      s = fmaf(q.x, s, q.y);
    }
    for (int w = kWarps - 1; w > at.w; --w)
      mu = fmaf(part[w][at.lane + 32 * j].x, mu, gpart[w][at.lane + 32 * j]);
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const float before = s;
      s = fmaf(f[i][j], s, n[i][j] * x[i][j]);
      x[i][j] = before - x[i][j];
    }
#pragma unroll
    for (int i = kRun - 1; i >= 0; --i) {
      const float lam = dh[i][j] + mu;
      mu = f[i][j] * lam;
      dh[i][j] = lam * n[i][j];              // dx
      x[i][j] = mu * n[i][j] * x[i][j];      // dg
    }
  }
#pragma unroll
  for (int i = 0; i < kRun; ++i) {
    const int64_t t = at.time(a, i);
    if (t < 0 || t >= a.T_) continue;
    if (!at.valid(t)) {
#pragma unroll
      for (int j = 0; j < kLane; ++j) dh[i][j] = x[i][j] = 0.f;
    }
    store_row<VEC>(a.dx.row(at.b, t), at.d, at.ok, dh[i]);
    store_row<VEC>(a.dg.row(at.b, t), at.d, at.ok, x[i]);
  }
}

template <class T, bool VEC>
__global__ void step_kernel(int64_t B, int64_t D, const T* __restrict__ x, int64_t xs,
                            const T* __restrict__ g, int64_t gs,
                            const uint8_t* __restrict__ active, const float* state,
                            float* state_out, T* __restrict__ h) {
  constexpr int V = VEC ? 4 : 1;
  const int64_t per = D / V;
  const int64_t n = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (n >= B * per) return;
  const int64_t b = n / per, d = (n - b * per) * V;
  const Pack<float, V> s = *reinterpret_cast<const Pack<float, V>*>(state + b * D + d);
  Pack<float, V> o = s;
  Pack<T, V> y;
  if (!active || active[b]) {
    const Pack<T, V> xv = *reinterpret_cast<const Pack<T, V>*>(x + b * xs + d);
    const Pack<T, V> gv = *reinterpret_cast<const Pack<T, V>*>(g + b * gs + d);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float f, m;
      sigmoid_pair(to_f32(gv.v[j]), f, m);
      o.v[j] = fmaf(f, s.v[j], m * to_f32(xv.v[j]));
      y.v[j] = from_f32<T>(o.v[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) y.v[j] = from_f32<T>(0.f);
  }
  *reinterpret_cast<Pack<float, V>*>(state_out + b * D + d) = o;
  *reinterpret_cast<Pack<T, V>*>(h + b * D + d) = y;
}

int64_t chunks_of(int64_t T) { return (T + kChunk - 1) / kChunk; }

template <class T>
ScanArgs<T> scan_args(const semicrf_recurrence* p) {
  ScanArgs<T> a{};
  a.B = p->batch;
  a.T_ = p->T;
  a.D = p->D;
  a.chunks = chunks_of(p->T);
  a.tiles = (p->D + kTile - 1) / kTile;
  a.reverse = p->reverse != 0;
  a.x = as_seq<const T>(p->x);
  a.g = as_seq<const T>(p->gate);
  a.lengths = p->lengths;
  return a;
}

template <class T>
int run_forward(const semicrf_recurrence* p, const semicrf_sequence& h, float* final_state,
                void* saved, void* workspace, cudaStream_t stream) {
  ScanArgs<T> a = scan_args<T>(p);
  a.h = as_seq<T>(h);
  a.agg = static_cast<float2*>(workspace);
  a.carry = saved ? static_cast<float*>(saved)
                  : reinterpret_cast<float*>(a.agg + a.B * a.chunks * a.D);
  const unsigned grid = (unsigned)(a.B * a.chunks * a.tiles);
  const bool vec = p->D % kLane == 0 && seq_aligned(p->x, a.B, a.T_, sizeof(T), kLane) &&
                   seq_aligned(p->gate, a.B, a.T_, sizeof(T), kLane) &&
                   seq_aligned(h, a.B, a.T_, sizeof(T), kLane);
  if (grid) {
    if (vec)
      compose_kernel<T, true, false><<<grid, 32 * kWarps, 0, stream>>>(a);
    else
      compose_kernel<T, false, false><<<grid, 32 * kWarps, 0, stream>>>(a);
  }
  const unsigned jg = (unsigned)((a.B * a.D + 127) / 128);
  join_kernel<<<jg, 128, 0, stream>>>(a.B, a.chunks, a.D, false, a.agg, p->initial_state, a.carry,
                                      final_state);
  if (grid) {
    if (vec)
      forward_kernel<T, true><<<grid, 32 * kWarps, 0, stream>>>(a);
    else
      forward_kernel<T, false><<<grid, 32 * kWarps, 0, stream>>>(a);
  }
  return launch_status();
}

template <class T>
int run_backward(const semicrf_recurrence* p, const void* saved, const semicrf_sequence& grad_h,
                 const float* grad_state, const semicrf_sequence& grad_x,
                 const semicrf_sequence& grad_gate, float* grad_initial, void* workspace,
                 cudaStream_t stream) {
  ScanArgs<T> a = scan_args<T>(p);
  a.dh = as_seq<const T>(grad_h);
  a.dx = as_seq<T>(grad_x);
  a.dg = as_seq<T>(grad_gate);
  a.carry = const_cast<float*>(static_cast<const float*>(saved));
  a.agg = static_cast<float2*>(workspace);
  a.gcarry = reinterpret_cast<float*>(a.agg + a.B * a.chunks * a.D);
  const unsigned grid = (unsigned)(a.B * a.chunks * a.tiles);
  const bool vec = p->D % kLane == 0 && seq_aligned(p->x, a.B, a.T_, sizeof(T), kLane) &&
                   seq_aligned(p->gate, a.B, a.T_, sizeof(T), kLane) &&
                   seq_aligned(grad_h, a.B, a.T_, sizeof(T), kLane) &&
                   seq_aligned(grad_x, a.B, a.T_, sizeof(T), kLane) &&
                   seq_aligned(grad_gate, a.B, a.T_, sizeof(T), kLane);
  if (grid) {
    if (vec)
      compose_kernel<T, true, true><<<grid, 32 * kWarps, 0, stream>>>(a);
    else
      compose_kernel<T, false, true><<<grid, 32 * kWarps, 0, stream>>>(a);
  }
  const unsigned jg = (unsigned)((a.B * a.D + 127) / 128);
  join_kernel<<<jg, 128, 0, stream>>>(a.B, a.chunks, a.D, true, a.agg, grad_state, a.gcarry,
                                      grad_initial);
  if (grid) {
    if (vec)
      backward_kernel<T, true><<<grid, 32 * kWarps, 0, stream>>>(a);
    else
      backward_kernel<T, false><<<grid, 32 * kWarps, 0, stream>>>(a);
  }
  return launch_status();
}

template <class T>
int run_step(int64_t B, int64_t D, const void* x, int64_t xs, const void* g, int64_t gs,
             const uint8_t* active, const float* state, float* state_out, void* h,
             cudaStream_t stream) {
  const auto aligned = [](const void* p, size_t n) {
    return reinterpret_cast<uintptr_t>(p) % n == 0;
  };
  const bool vec = D % 4 == 0 && xs % 4 == 0 && gs % 4 == 0 && aligned(x, 4 * sizeof(T)) &&
                   aligned(g, 4 * sizeof(T)) && aligned(h, 4 * sizeof(T)) && aligned(state, 16) &&
                   aligned(state_out, 16);
  const int64_t n = B * D / (vec ? 4 : 1);
  const unsigned grid = (unsigned)((n + 127) / 128);
  const T* xp = static_cast<const T*>(x);
  const T* gp = static_cast<const T*>(g);
  if (vec)
    step_kernel<T, true><<<grid, 128, 0, stream>>>(B, D, xp, xs, gp, gs, active, state, state_out,
                                                   static_cast<T*>(h));
  else
    step_kernel<T, false><<<grid, 128, 0, stream>>>(B, D, xp, xs, gp, gs, active, state, state_out,
                                                    static_cast<T*>(h));
  return launch_status();
}

}  // namespace

size_t recurrence_saved_bytes(const semicrf_recurrence* p) {
  return sizeof(float) * p->batch * chunks_of(p->T) * p->D;
}
size_t recurrence_workspace_bytes(const semicrf_recurrence* p) {
  return (sizeof(float2) + sizeof(float)) * p->batch * chunks_of(p->T) * p->D;
}

int recurrence_forward(const semicrf_recurrence* p, const semicrf_sequence& h, float* final_state,
                       void* saved, void* workspace, cudaStream_t stream) {
  switch (p->dtype) {
    case SEMICRF_F32: return run_forward<float>(p, h, final_state, saved, workspace, stream);
    case SEMICRF_BF16:
      return run_forward<__nv_bfloat16>(p, h, final_state, saved, workspace, stream);
    default: return run_forward<__half>(p, h, final_state, saved, workspace, stream);
  }
}

int recurrence_backward(const semicrf_recurrence* p, const void* saved,
                        const semicrf_sequence& grad_h, const float* grad_state,
                        const semicrf_sequence& grad_x, const semicrf_sequence& grad_gate,
                        float* grad_initial, void* workspace, cudaStream_t stream) {
  switch (p->dtype) {
    case SEMICRF_F32:
      return run_backward<float>(p, saved, grad_h, grad_state, grad_x, grad_gate, grad_initial,
                                 workspace, stream);
    case SEMICRF_BF16:
      return run_backward<__nv_bfloat16>(p, saved, grad_h, grad_state, grad_x, grad_gate,
                                         grad_initial, workspace, stream);
    default:
      return run_backward<__half>(p, saved, grad_h, grad_state, grad_x, grad_gate, grad_initial,
                                  workspace, stream);
  }
}

int recurrence_step(int64_t B, int64_t D, int dtype, const void* x, int64_t x_stride,
                    const void* gate, int64_t gate_stride, const uint8_t* active,
                    const float* state, float* state_out, void* h, cudaStream_t stream) {
  switch (dtype) {
    case SEMICRF_F32:
      return run_step<float>(B, D, x, x_stride, gate, gate_stride, active, state, state_out, h,
                             stream);
    case SEMICRF_BF16:
      return run_step<__nv_bfloat16>(B, D, x, x_stride, gate, gate_stride, active, state,
                                     state_out, h, stream);
    default:
      return run_step<__half>(B, D, x, x_stride, gate, gate_stride, active, state, state_out, h,
                              stream);
  }
}

}  // namespace semicrf
