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
// dw1 and ds share their sum over rows: A = sum d silu(g) zh gives dw1 = s A
// and ds = w1 A, so two sums a channel are carried, and w1 and s enter the rows
// only as their product.
//
// A row lies in the registers of WR warps, PER channels to a lane, so each
// input is read once.  The backward recomputes r from the block's inputs in
// 32 bits; it reads x where it would else read the rounded r.  Weight
// gradients are summed per thread over the rows that its CTA walks, then over
// the CTAs in a fixed order: no atomics.  Products and sums go two channels to
// an instruction.
//
// Bound by memory: 5 values an element forward, 8 backward.  Measured at 32 x
// 4,096 x 512, bfloat16: forward 111 us and backward 170 us (6.1 and 6.3 TB/s),
// the sums over CTAs 5 us.  Other widths with whole 16-byte vectors reach 0.8
// to 1.5 times their bytes' time at the copy rate, up to 4,096; wider rows have
// one CTA an SM, and of 16-bit types a ring beside which the weights find no
// room: 8,192 takes 2.8 and 4.1 times it.  Rows without 16-byte alignment go
// value by value: 1.0 to 1.7 times for float32, 1.5 to 3 for 16-bit types.

#include <algorithm>
#include <type_traits>

#include "encoder_internal.cuh"
#include "tma.cuh"

namespace semicrf {
int device_sm_count();  // api.cu

namespace {

template <class T>
struct NormArgs {
  int64_t rows, D;
  Places places;
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
  float* partial;  // (grid, 2, D): A and the sum of dn rh
};

// Sums over the row's lanes; every lane gets the result.  `red` alternates
// between two slots, so one barrier per sum is enough.
template <class L>
struct RowSum {
  static constexpr int WR = L::WR;
  float (*red)[WR];
  int slot, w, lane, barrier;
  __device__ __forceinline__ float operator()(float v) {
#pragma unroll
    for (int o = 16 / L::SPLIT; o > 0; o >>= 1) v += __shfl_xor_sync(L::peers(), v, o);
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

// PER channels to a lane in vectors of V, WR warps to a row or SPLIT rows to a warp.
template <class T, int V_, int WR_, int PER_, int SPLIT_ = 1>
struct Layout {
  static constexpr int V = V_, WR = WR_, PER = PER_, SPLIT = SPLIT_;
  static constexpr int J = PER / V;                   // vectors of a lane
  static constexpr int H = PER / 2;                   // pairs of a lane
  static constexpr int NL = 32 * WR / SPLIT;          // lanes of a row
  static constexpr int kRows = SPLIT * (WR >= 4 ? 1 : 4 / WR);  // rows that a CTA works on at once
  // whether the lanes that share a group of the checkpoint share a row
  static constexpr bool kCodes = NL * V >= kPackGroup;
  static constexpr int kThreads = NL * kRows;
  // CTAs of the backward on an SM: 8 warps of 24 channels a lane (255 registers),
  // 12 of 16 (168), 16 of 8 (128), 24 of 4 (80)
  static constexpr int kWarpsPerSm = PER == 24 ? 8 : PER == 16 ? 12 : PER == 8 ? 16 : 24;
  static constexpr int kPerSm = NL * kRows < 32 * kWarpsPerSm ? 32 * kWarpsPerSm / kThreads : 1;
  // shared memory of a CTA beside a ring, and what a CTA may take if n of them are to lie on an SM
  static constexpr bool kSharedWeights = H * NL <= 2048;
  static constexpr int kFixedBytes =
      (kSharedWeights ? 16 * H * NL : 16) + (kRows > 1 ? 8 * H * NL : 8) + 8 * kRows * WR + 2048;
  static constexpr int share(int n) { return 228 * 1024 / n - kFixedBytes; }
  // the lanes of a warp that work on this lane's row; others may be elsewhere
  __device__ static __forceinline__ unsigned peers() {
    return SPLIT == 1 ? ~0u : ((1u << (32 / SPLIT)) - 1) << (threadIdx.x & 31 & ~(32 / SPLIT - 1));
  }
  // channel of vector j of lane l
  __device__ static __forceinline__ int channel(int j, int l) { return (j * NL + l) * V; }
  // channel of half k of pair i of lane l
  __device__ static __forceinline__ int channel_of(int i, int k, int l) {
    const int e = 2 * i + k;
    return channel(e / V, l) + e % V;
  }
};

// A lane's part of a row as it lies in memory, and as pairs.
template <class T, class L>
struct Held {
  Pack<T, L::V> v[L::J];
  __device__ __forceinline__ void get(const T* row, int l, const bool (&ok)[L::J], bool live) {
#pragma unroll
    for (int j = 0; j < L::J; ++j) {
#pragma unroll
      for (int k = 0; k < L::V; ++k) v[j].v[k] = from_f32<T>(0.f);
      if (live && ok[j])
        v[j] = *reinterpret_cast<const Pack<T, L::V>*>(row + L::channel(j, l));
    }
  }
  __device__ __forceinline__ float2 pair(int i) const {
    Pack<T, 2> q;
    q.v[0] = v[2 * i / L::V].v[2 * i % L::V];
    q.v[1] = v[(2 * i + 1) / L::V].v[(2 * i + 1) % L::V];
    return to_f32x2(q);
  }
  __device__ __forceinline__ void set(int i, float2 f) {
    const Pack<T, 2> q = from_f32x2<T>(f);
    v[2 * i / L::V].v[2 * i % L::V] = q.v[0];
    v[(2 * i + 1) / L::V].v[(2 * i + 1) % L::V] = q.v[1];
  }
  __device__ __forceinline__ void put(T* row, int l, const bool (&ok)[L::J]) const {
#pragma unroll
    for (int j = 0; j < L::J; ++j)
      if (ok[j]) *reinterpret_cast<Pack<T, L::V>*>(row + L::channel(j, l)) = v[j];
  }
};

// The two weight vectors that rows need, s w1 and w2, by pair and lane: from
// shared memory, or in the widest layout (64 KB of them) from global memory.
template <class L, bool BRANCH>
struct Weights {
  static constexpr bool kShared = L::kSharedWeights;
  static constexpr int kSize = kShared ? L::H * L::NL : 1;
  float2 *sw_, *w2_;
  const float *s, *w1, *w2g;
  int64_t D;
  int l;
  __device__ __forceinline__ float2 from_global(int i, const float* p, const float* q) const {
    const int d0 = L::channel_of(i, 0, l), d1 = L::channel_of(i, 1, l);
    return make_float2(d0 < D ? (q ? p[d0] * q[d0] : p[d0]) : 0.f,
                       d1 < D ? (q ? p[d1] * q[d1] : p[d1]) : 0.f);
  }
  __device__ __forceinline__ float2 sw(int i) const {
    return kShared ? sw_[i * L::NL + l] : from_global(i, s, w1);
  }
  __device__ __forceinline__ float2 w2(int i) const {
    return kShared ? w2_[i * L::NL + l] : from_global(i, w2g, nullptr);
  }
  template <class T>
  __device__ Weights(const NormArgs<T>& a, float2* sw, float2* w2)
      : sw_(sw), w2_(w2), s(a.s), w1(a.w1), w2g(a.w2), D(a.D) {
    if (kShared)
      for (int k = threadIdx.x; k < kSize; k += L::kThreads) {
        l = k % L::NL;
        w2[k] = from_global(k / L::NL, w2g, nullptr);
        if (BRANCH) sw[k] = from_global(k / L::NL, s, w1);
      }
    __syncthreads();
    l = threadIdx.x % L::NL;
  }
};

// How a row's inputs reach the pairs that are worked on.  Plain: into
// registers.  Where a lane's vectors are 16 bytes, asynchronous copies keep the
// next rows on their way to shared memory: it takes some 40 KB in flight on an
// SM to keep HBM busy, and the sums and factors leave no registers for that.
// A lane reads only what it copied itself, so no barrier is involved.
enum Input { kX, kZ, kG, kDn, kDr };

template <class T, class L, int N>
struct PlainRows {
  static constexpr int kSlots = 0;
  Held<T, L> held[N];
  __device__ __forceinline__ float2 pair(int k, int i) const { return held[k].pair(i); }
};
template <class T, class L, int N>
struct RingRows {
  static constexpr int kSlotBytes = N * L::J * L::kThreads * 16;
  static constexpr int kCtas = N == 5 ? L::kPerSm : 1;  // that have to fit an SM
  static constexpr int kRoom = L::share(kCtas) / kSlotBytes;
  static constexpr int kSlots = kRoom >= 3 && 3 * kSlotBytes <= 96 * 1024 ? 3 : kRoom >= 2 ? 2 : 0;
  unsigned char* at;  // this thread's part of the present slot
  __device__ __forceinline__ float2 pair(int k, int i) const {
    const int j = 2 * i / L::V;
    const Pack<T, L::V> v =
        *reinterpret_cast<const Pack<T, L::V>*>(at + (k * L::J + j) * L::kThreads * 16);
    Pack<T, 2> q;
    q.v[0] = v.v[2 * i % L::V];
    q.v[1] = v.v[2 * i % L::V + 1];
    return to_f32x2(q);
  }
};

// Requests a row of N tensors into a slot of the ring: one group of copies a
// row, whatever it holds.
template <int N, class T, class L>
__device__ __forceinline__ void request_row(const NormArgs<T>& a, const Seq<const T> (&src)[N],
                                            unsigned char* ring, int slot, int64_t row, int l,
                                            const bool (&ok)[L::J], L) {
  int64_t b, t;
  bool live = row < a.rows;
  if (live) {
    locate(a.places, row, b, t);
    live = !a.lengths || t < a.lengths[b];
  }
  if (live)
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
      for (int j = 0; j < L::J; ++j) {
        const bool has = src[k].p && ok[j];
        asm volatile(
            "cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(
                ring + slot * RingRows<T, L, N>::kSlotBytes +
                ((k * L::J + j) * L::kThreads + threadIdx.x) * 16)),
            "l"(has ? src[k].row(b, t) + L::channel(j, l) : a.x.p), "r"(has ? 16 : 0)
            : "memory");
      }
  asm volatile("cp.async.commit_group;" ::: "memory");
}

// The checkpoint of n as it was rounded.
template <class T, class L>
__device__ __forceinline__ void put_codes(const NormArgs<T>& a, int64_t row, int l,
                                          const bool (&ok)[L::J], const Held<T, L>& n) {
  const int64_t G = pack_groups(a.D);
#pragma unroll
  for (int j = 0; j < L::J; ++j) {
    const int d = L::channel(j, l);
    Pack<T, L::V> v = n.v[j];
    if (!ok[j])
#pragma unroll
      for (int k = 0; k < L::V; ++k) v.v[k] = from_f32<T>(0.f);
    Pack<int8_t, L::V> c;
    const uint8_t byte = pack_encode(v, c, L::peers());
    if (d < G * kPackGroup) {
      *reinterpret_cast<Pack<int8_t, L::V>*>(a.codes + row * G * kPackGroup + d) = c;
      if (d % kPackGroup == 0) a.scales[row * G + d / kPackGroup] = byte;
    }
  }
}

// A gate as the rows use it: below -128 its sigmoid is held to 2^-126, which times
// a gate near the type's lowest value would not be silu's 0 any more (-4 at bfloat16's).
__device__ __forceinline__ float2 held_gate(float2 g) {
  asm("max.NaN.f32 %0, %0, 0fC3000000;" : "+f"(g.x));
  asm("max.NaN.f32 %0, %0, 0fC3000000;" : "+f"(g.y));
  return g;
}

template <class T, class L, bool BRANCH, bool RING>
__global__ void __launch_bounds__(L::kThreads) norm_forward_kernel(const NormArgs<T> a) {
  constexpr int H = L::H, NL = L::NL;
  using Rows = typename std::conditional<RING, RingRows<T, L, 3>, PlainRows<T, L, 3>>::type;
  constexpr int SLOTS = Rows::kSlots;
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ float red[L::kRows][2][L::WR];
  __shared__ float2 sw_at[BRANCH ? Weights<L, BRANCH>::kSize : 1], w2_at[Weights<L, BRANCH>::kSize];
  const int group = threadIdx.x / NL, l = threadIdx.x % NL;
  RowSum<L> row_sum{red[group], 0, l >> 5, l & 31, 1 + group};
  bool ok[L::J];
#pragma unroll
  for (int j = 0; j < L::J; ++j) ok[j] = L::channel(j, l) < a.D;

  const Seq<const T> src[3] = {a.x, a.z, a.g};
  const int64_t first = (int64_t)blockIdx.x * L::kRows + group;
  const int64_t stride = (int64_t)gridDim.x * L::kRows;
  Rows in;
  const auto request = [&](int64_t row, int slot) {
    if constexpr (RING) request_row<3>(a, src, ring, slot, row, l, ok, L());
  };
#pragma unroll
  for (int k = 0; k < SLOTS - 1; ++k) request(first + k * stride, k);
  const Weights<L, BRANCH> weight(a, sw_at, w2_at);
  int slot = 0;
  for (int64_t row = first; row < a.rows; row += stride) {
    int64_t b, t;
    locate(a.places, row, b, t);
    const bool live = !a.lengths || t < a.lengths[b];
    if constexpr (RING) {
      request(row + (SLOTS - 1) * stride, slot == 0 ? SLOTS - 1 : slot - 1);
      asm volatile("cp.async.wait_group %0;" ::"n"(SLOTS > 0 ? SLOTS - 1 : 0) : "memory");
      in.at = ring + slot * Rows::kSlotBytes + threadIdx.x * 16;
      slot = slot == SLOTS - 1 ? 0 : slot + 1;
    }
    Held<T, L> out;
    if (!live) {  // the whole row group takes this branch together
#pragma unroll
      for (int i = 0; i < H; ++i) out.set(i, both(0.f));
      if (BRANCH) out.put(a.r.row(b, t), l, ok);
      out.put(a.n.row(b, t), l, ok);
      if (L::kCodes && a.codes) put_codes<T, L>(a, row, l, ok, out);
      continue;
    }
    if constexpr (!RING) {
#pragma unroll
      for (int k = 0; k < (BRANCH ? 3 : 1); ++k) in.held[k].get(src[k].row(b, t), l, ok, true);
    }
    float rz = 0.f;
    float2 r[H], q = both(0.f);
    if (BRANCH) {
#pragma unroll
      for (int i = 0; i < H; ++i) {
        const float2 z = in.pair(kZ, i);
        q = __ffma2_rn(z, z, q);
      }
      rz = rsqrtf(row_sum(q.x + q.y) * a.inv_d + a.eps);
      q = both(0.f);
    }
#pragma unroll
    for (int i = 0; i < H; ++i) {
      r[i] = in.pair(kX, i);
      if (BRANCH) {
        float2 sig, neg;
        const float2 g = held_gate(in.pair(kG, i));
        sigmoid_pair2<T>(g, sig, neg);
        const float2 u = __fmul2_rn(__fmul2_rn(g, sig), weight.sw(i));
        r[i] = __ffma2_rn(u, __fmul2_rn(in.pair(kZ, i), both(rz)), r[i]);
      }
      q = __ffma2_rn(r[i], r[i], q);
    }
    const float rr = rsqrtf(row_sum(q.x + q.y) * a.inv_d + a.eps);
    if (a.stats && l == 0) {
      a.stats[2 * row] = rz;
      a.stats[2 * row + 1] = rr;
    }
    if (BRANCH) {
#pragma unroll
      for (int i = 0; i < H; ++i) out.set(i, r[i]);
      out.put(a.r.row(b, t), l, ok);
    }
#pragma unroll
    for (int i = 0; i < H; ++i) out.set(i, __fmul2_rn(__fmul2_rn(r[i], both(rr)), weight.w2(i)));
    out.put(a.n.row(b, t), l, ok);
    if (L::kCodes && a.codes) put_codes<T, L>(a, row, l, ok, out);
  }
  if (RING) asm volatile("cp.async.wait_all;" ::: "memory");
}

template <class T, class L, bool BRANCH, bool RING>
__global__ void __launch_bounds__(L::kThreads, L::kPerSm) norm_backward_kernel(const NormArgs<T> a) {
  constexpr int H = L::H, NL = L::NL;
  using Rows = typename std::conditional<RING, RingRows<T, L, 5>, PlainRows<T, L, 5>>::type;
  constexpr int SLOTS = Rows::kSlots;
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ float red[L::kRows][2][L::WR];
  __shared__ float2 sw_at[BRANCH ? Weights<L, BRANCH>::kSize : 1], w2_at[Weights<L, BRANCH>::kSize];
  __shared__ float2 sums[L::kRows > L::SPLIT ? H * NL : 1];
  const Weights<L, BRANCH> weight(a, sw_at, w2_at);
  const int group = threadIdx.x / NL, l = threadIdx.x % NL;
  RowSum<L> row_sum{red[group], 0, l >> 5, l & 31, 1 + group};
  bool ok[L::J];
#pragma unroll
  for (int j = 0; j < L::J; ++j) ok[j] = L::channel(j, l) < a.D;
  float2 acc[2][H];
#pragma unroll
  for (int i = 0; i < H; ++i) acc[0][i] = acc[1][i] = both(0.f);

  const Seq<const T> src[5] = {a.x, a.z, a.g, a.dn, a.dr};
  const int64_t first = (int64_t)blockIdx.x * L::kRows + group;
  const int64_t stride = (int64_t)gridDim.x * L::kRows;
  Rows in;
  const auto request = [&](int64_t row, int slot) {
    if constexpr (RING) request_row<5>(a, src, ring, slot, row, l, ok, L());
  };
  float next_z = 0.f, next_r = 0.f;
  if (RING) {
#pragma unroll
    for (int k = 0; k < SLOTS - 1; ++k) request(first + k * stride, k);
    if (first < a.rows) next_z = a.stats[2 * first], next_r = a.stats[2 * first + 1];
  }
  int slot = 0;
  for (int64_t row = first; row < a.rows; row += stride) {
    int64_t b, t;
    locate(a.places, row, b, t);
    const bool live = !a.lengths || t < a.lengths[b];
    float2 rz, rr;
    if constexpr (RING) {
      request(row + (SLOTS - 1) * stride, slot == 0 ? SLOTS - 1 : slot - 1);
      rz = both(next_z), rr = both(next_r);
      if (row + stride < a.rows) {
        next_z = a.stats[2 * (row + stride)];
        next_r = a.stats[2 * (row + stride) + 1];
      }
      asm volatile("cp.async.wait_group %0;" ::"n"(SLOTS > 0 ? SLOTS - 1 : 0) : "memory");
      in.at = ring + slot * Rows::kSlotBytes + threadIdx.x * 16;
      slot = slot == SLOTS - 1 ? 0 : slot + 1;
    }
    Held<T, L> out;
    if (!live) {  // the whole row group takes this branch together
#pragma unroll
      for (int i = 0; i < H; ++i) out.set(i, both(0.f));
      out.put(a.dx.row(b, t), l, ok);
      if (BRANCH) {
        out.put(a.dz.row(b, t), l, ok);
        out.put(a.dg.row(b, t), l, ok);
      }
      continue;
    }
    if constexpr (!RING) {
#pragma unroll
      for (int k = 0; k < 5; ++k)
        if (BRANCH || (k != kZ && k != kG))
          in.held[k].get(src[k].row(b, t), l, ok, src[k].p != nullptr);
      rz = both(a.stats[2 * row]), rr = both(a.stats[2 * row + 1]);
    }
    float2 rh[H], sig[BRANCH ? H : 1], q = both(0.f);
#pragma unroll
    for (int i = 0; i < H; ++i) {
      rh[i] = in.pair(kX, i);
      if (BRANCH) {
        float2 neg;
        const float2 g = held_gate(in.pair(kG, i));
        sigmoid_pair2<T>(g, sig[i], neg);
        rh[i] = __ffma2_rn(__fmul2_rn(__fmul2_rn(g, sig[i]), weight.sw(i)),
                           __fmul2_rn(in.pair(kZ, i), rz), rh[i]);
      }
      rh[i] = __fmul2_rn(rh[i], rr);
      const float2 dn = in.pair(kDn, i);
      acc[1][i] = __ffma2_rn(dn, rh[i], acc[1][i]);
      q = __ffma2_rn(__fmul2_rn(dn, weight.w2(i)), rh[i], q);
    }
    const float2 c2 = both(-row_sum(q.x + q.y) * a.inv_d);
    q = both(0.f);
    Held<T, L> gate;
#pragma unroll
    for (int i = 0; i < H; ++i) {
      const float2 p = __fmul2_rn(in.pair(kDn, i), weight.w2(i));
      const float2 d = __ffma2_rn(rr, __ffma2_rn(rh[i], c2, p), in.pair(kDr, i));
      out.set(i, d);
      if (BRANCH) {
        const float2 zh = __fmul2_rn(in.pair(kZ, i), rz),
                     g = held_gate(in.pair(kG, i));
        const float2 du = __fmul2_rn(d, __fmul2_rn(g, sig[i]));
        acc[0][i] = __ffma2_rn(du, zh, acc[0][i]);
        // silu'(g) = sig (1 + g (1 - sig))
        const float2 slope =
            __fmul2_rn(sig[i], __ffma2_rn(g, sub2(both(1.f), sig[i]), both(1.f)));
        gate.set(i, __fmul2_rn(__fmul2_rn(__fmul2_rn(d, weight.sw(i)), zh), slope));
        rh[i] = __fmul2_rn(du, weight.sw(i));  // db w1 takes rh's place
        q = __ffma2_rn(rh[i], zh, q);
      }
    }
    out.put(a.dx.row(b, t), l, ok);
    if (BRANCH) {
      gate.put(a.dg.row(b, t), l, ok);
      const float2 c1 = both(-row_sum(q.x + q.y) * a.inv_d);
#pragma unroll
      for (int i = 0; i < H; ++i)
        out.set(i, __fmul2_rn(rz, __ffma2_rn(__fmul2_rn(in.pair(kZ, i), rz), c1, rh[i])));
      out.put(a.dz.row(b, t), l, ok);
    }
  }
  if (RING) asm volatile("cp.async.wait_all;" ::: "memory");

  // the CTA's sums: over the rows of a warp, then its row groups in order
  constexpr int kGroups = L::kRows / L::SPLIT;
  const int mine = group / L::SPLIT;
#pragma unroll
  for (int m = BRANCH ? 0 : 1; m < 2; ++m) {
#pragma unroll
    for (int o = NL; o < 32; o <<= 1)
#pragma unroll
      for (int i = 0; i < H; ++i) {
        acc[m][i].x += __shfl_xor_sync(~0u, acc[m][i].x, o);
        acc[m][i].y += __shfl_xor_sync(~0u, acc[m][i].y, o);
      }
    if (kGroups > 1) {
#pragma unroll 1
      for (int turn = kGroups - 1; turn > 0; --turn) {
        __syncthreads();
        if (group == turn * L::SPLIT)
#pragma unroll
          for (int i = 0; i < H; ++i) sums[i * NL + l] = acc[m][i];
        __syncthreads();
        if (mine == turn - 1)
#pragma unroll
          for (int i = 0; i < H; ++i) acc[m][i] = __fadd2_rn(acc[m][i], sums[i * NL + l]);
      }
    }
    if (group == 0)
#pragma unroll
      for (int i = 0; i < H; ++i) {
        float* p = a.partial + ((int64_t)blockIdx.x * 2 + m) * a.D;
        const int d0 = L::channel_of(i, 0, l), d1 = L::channel_of(i, 1, l);
        if (d0 < a.D) p[d0] = acc[m][i].x;
        if (d1 < a.D) p[d1] = acc[m][i].y;
      }
  }
}

// Sums the CTAs' partials in a fixed order: a block takes 8 channels of one of
// the two sums, its 32 rows of threads every 32nd CTA.
__global__ void __launch_bounds__(256) norm_reduce_kernel(int64_t D, int first, int ctas,
                                                          const float* __restrict__ w1,
                                                          const float* __restrict__ s,
                                                          const float* __restrict__ partial,
                                                          float* __restrict__ out) {
  __shared__ float part[32][9];
  const int m = blockIdx.y + first, x = threadIdx.x & 7, y = threadIdx.x >> 3;
  const int64_t d = (int64_t)blockIdx.x * 8 + x;
  float v = 0.f;
  if (d < D) {
    const float* p = partial + m * D + d;
#pragma unroll 8
    for (int c = y; c < ctas; c += 32) v += p[(int64_t)c * 2 * D];
  }
  part[y][x] = v;
  __syncthreads();
  if (y || d >= D) return;
#pragma unroll
  for (int k = 1; k < 32; ++k) v += part[k][x];
  if (m) {
    out[2 * D + d] = v;
  } else {
    out[d] = s[d] * v;
    out[D + d] = w1[d] * v;
  }
}

template <class T>
NormArgs<T> norm_args(const semicrf_block_norm* p) {
  NormArgs<T> a{};
  a.rows = p->batch * p->T;
  a.places = make_places(p->batch, p->T);
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

// CTAs of a backward launch: what is resident at once, so that each walks an
// equal share of the rows.
int64_t backward_ctas(int64_t rows, int at_once, int per_sm) {
  const int64_t all = (rows + at_once - 1) / at_once;
  return std::max<int64_t>(1, std::min<int64_t>(all, (int64_t)per_sm * device_sm_count()));
}

template <class T, class L, bool BRANCH>
int launch(const NormArgs<T>& a, bool backward, float* grad_weights, cudaStream_t stream) {
  if (!backward) {
    const int64_t all = (a.rows + L::kRows - 1) / L::kRows;
    constexpr bool kRing = BRANCH && L::V * sizeof(T) == 16 && RingRows<T, L, 3>::kSlots > 0;
    const auto kernel = norm_forward_kernel<T, L, BRANCH, kRing>;
    constexpr int bytes = kRing ? RingRows<T, L, 3>::kSlots * RingRows<T, L, 3>::kSlotBytes : 0;
    const int64_t most = (int64_t)std::max(1, 1024 / L::kThreads) * device_sm_count();
    const unsigned grid = (unsigned)std::min<int64_t>(all, most);
    if (bytes && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      bytes) != cudaSuccess)
      return SEMICRF_ERR_CUDA;
    if (grid) kernel<<<grid, L::kThreads, bytes, stream>>>(a);
    return launch_status();
  }
  const int ctas = (int)backward_ctas(a.rows, L::kRows, L::kPerSm);
  constexpr bool kRing = BRANCH && L::V * sizeof(T) == 16 && RingRows<T, L, 5>::kSlots > 0;
  const auto kernel = norm_backward_kernel<T, L, BRANCH, kRing>;
  constexpr int bytes = kRing ? RingRows<T, L, 5>::kSlots * RingRows<T, L, 5>::kSlotBytes : 0;
  if (bytes && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) !=
                   cudaSuccess)
    return SEMICRF_ERR_CUDA;
  kernel<<<ctas, L::kThreads, bytes, stream>>>(a);
  const int first = BRANCH ? 0 : 1;
  const dim3 grid((unsigned)((a.D + 7) / 8), 2 - first);
  norm_reduce_kernel<<<grid, 256, 0, stream>>>(a.D, first, ctas, a.w1, a.s, a.partial,
                                                        grad_weights);
  return launch_status();
}

// The first of the layouts whose lanes hold a row, and its codes where wanted.
template <class T, bool BRANCH, class L, class... Wider>
int launch_first(const NormArgs<T>& a, bool backward, float* gw, cudaStream_t s) {
  if constexpr (sizeof...(Wider) > 0)
    if (a.D > L::NL * L::PER || (a.codes && !L::kCodes))
      return launch_first<T, BRANCH, Wider...>(a, backward, gw, s);
  return launch<T, L, BRANCH>(a, backward, gw, s);
}

// The fewest lanes whose registers hold a row.  16-byte rows of 16-bit types:
// 16 or 24 channels a lane, few idle ones at any width, since the more a lane
// holds the more of its arithmetic overlaps (eight, one row to a warp: width
// 256 backward 236 us for the 218 of sixteen and two rows; width 64 in a whole
// warp 618 us for 232).  Else 4 or 8, at most 16 warps; narrow rows share a
// warp there too, unless their codes are wanted (37 channels without alignment,
// backward, 1036 us in a whole warp and 538 in half of one).
template <class T, int V, bool BRANCH>
int launch_width(const NormArgs<T>& a, bool backward, float* gw, cudaStream_t s) {
  if constexpr (V == 8)
    return launch_first<T, BRANCH, Layout<T, V, 1, 8, 8>, Layout<T, V, 1, 16, 8>,
                        Layout<T, V, 1, 24, 8>, Layout<T, V, 1, 16, 4>, Layout<T, V, 1, 24, 4>,
                        Layout<T, V, 1, 16, 2>, Layout<T, V, 1, 24, 2>, Layout<T, V, 1, 16>,
                        Layout<T, V, 1, 24>, Layout<T, V, 2, 16>, Layout<T, V, 2, 24>,
                        Layout<T, V, 4, 16>, Layout<T, V, 4, 24>, Layout<T, V, 8, 16>,
                        Layout<T, V, 16, 16>>(a, backward, gw, s);
  else if constexpr (V == 4)
    return launch_first<T, BRANCH, Layout<T, V, 1, 4, 4>, Layout<T, V, 1, 4, 2>,
                        Layout<T, V, 1, 4>, Layout<T, V, 1, 8>, Layout<T, V, 2, 8>,
                        Layout<T, V, 4, 8>, Layout<T, V, 8, 8>, Layout<T, V, 16, 8>,
                        Layout<T, V, 16, 16>>(a, backward, gw, s);
  else
    return launch_first<T, BRANCH, Layout<T, V, 1, 4, 4>, Layout<T, V, 1, 4, 2>,
                        Layout<T, V, 1, 4>, Layout<T, V, 1, 8>, Layout<T, V, 2, 8>,
                        Layout<T, V, 4, 8>, Layout<T, V, 8, 8>, Layout<T, V, 16, 8>,
                        Layout<T, V, 16, 16>>(a, backward, gw, s);
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
  // the most CTAs that any layout launches
  return sizeof(float) * 2 * p->D * backward_ctas(p->batch * p->T, 1, 6);
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
