// recurrence.cu -- the gated linear recurrence, its gradient and its
// single-position form.
//
//   f = sigmoid(g),  h_u = f_u h_{u-1} + (1 - f_u) x_u
//
// u counts positions in scan order (t = u; reversed, from the end of the last
// chunk down); masked positions have f = 1 and contribute nothing, so they pass the state on.
// Steps compose: (P, S) with h_out = P h_in + S, P the product of f, S the
// result from zero.  f <= 1, so nothing overflows and no logarithm is needed.
//
// Gradient: lam_u = dh_u + f_{u+1} lam_{u+1}.  With mu_u = f_u lam_u it is
// the same recurrence from the other end, mu_u = f_u (dh_u + mu_{u+1}), and
//   dx_u = lam_u (1 - f_u),  dg_u = lam_u (h_{u-1} - x_u) f_u (1 - f_u).
// h_{u-1} is recomputed from the float32 state kept at the start of each
// chunk, which is more exact than rereading the rounded h and one read less.
//
// A CTA of eight warps walks a column (a sequence's tile of channels) in
// chunks of 64 positions: a warp owns eight consecutive positions, a lane its
// channels.  Each warp composes its positions, one barrier a chunk makes the
// compositions known, and each warp goes from the state that entered the
// chunk over the earlier warps' to its own start.  The next chunk's rows are
// requested before the present one is joined, so loads are always in flight.
//
// Where there are fewer columns than CTAs fit on the device, a column's chunks
// are cut into segments, one to a CTA.  A first launch composes each segment
// but the last one; the walk then joins the segments before its own.  That
// reads two of the tensors twice, against a device mostly idle.  (A single
// pass in which CTAs wait for their predecessors' compositions was slower:
// each held its registers through several dependent trips to L2.)
// Every order of operations depends on sizes alone.

#include <algorithm>
#include <type_traits>

#include "encoder_internal.cuh"
#include "tma.cuh"

namespace semicrf {
int device_sm_count();  // api.cu

namespace {

constexpr int kRun = 8;                 // positions of a thread
constexpr int kWarps = 8;               // threads along time
constexpr int kChunk = kRun * kWarps;   // positions of a CTA at a time

template <class T>
struct ScanArgs {
  int64_t B, T_, D;
  int64_t chunks, per;  // chunks of a sequence, of a segment
  int tiles, segments;
  bool reverse;
  Seq<const T> x, g, dh;
  Seq<T> h, dx, dg;
  const int64_t* lengths;
  const float* first;  // (B, D): state before the first position / gradient of the last state
  float* last;         // (B, D): state after the last / gradient of the first; may be null
  float* carry;        // (B, chunks, D): the state entering each chunk; may be null (forward)
  float2* composed;    // (B, segments, D)
};

__device__ __forceinline__ float2 then(float2 a, float2 b) {  // b after a
  return make_float2(b.x * a.x, fmaf(b.x, a.y, b.y));
}

// Where a CTA works.  A lane holds L channels: neighbours where rows can be
// read as vectors, else 32 apart.  Slot lane + 32 j of a tile is lane's j-th.
template <class T, int L, bool VEC>
struct Place {
  static constexpr int kTile = 32 * L;
  int64_t b, len, d0;
  int segment, lane, w;
  bool ok[L];
  __device__ explicit Place(const ScanArgs<T>& a) {
    const int64_t id = blockIdx.x, tile = id % a.tiles, rest = id / a.tiles;
    segment = (int)(rest % a.segments);
    b = rest / a.segments;
    lane = threadIdx.x & 31;
    w = threadIdx.x >> 5;
    len = valid_length(a.lengths, b, a.T_);
    d0 = tile * kTile;
#pragma unroll
    for (int j = 0; j < L; ++j) ok[j] = channel(lane + 32 * j) < a.D;
  }
  __device__ __forceinline__ int64_t channel(int slot) const {
    return d0 + (VEC ? (slot & 31) * L + (slot >> 5) : slot);
  }
  __device__ __forceinline__ int64_t column0() const { return d0 + lane * (VEC ? L : 1); }
  // position of scan index u
  __device__ __forceinline__ int64_t time(const ScanArgs<T>& a, int64_t u) const {
    return a.reverse ? a.chunks * kChunk - 1 - u : u;
  }
  // whether all of scan indexes [u, u + n) are valid positions
  __device__ __forceinline__ bool whole(const ScanArgs<T>& a, int64_t u, int n) const {
    const int64_t lo = a.reverse ? a.chunks * kChunk - u - n : u;
    return lo + n <= len;
  }
};

template <bool VEC, class T, int L>
__device__ __forceinline__ void load_lane(const T* p, const bool (&ok)[L], bool live,
                                          Pack<T, L>& q) {
#pragma unroll
  for (int j = 0; j < L; ++j) q.v[j] = from_f32<T>(0.f);
  if (VEC) {
    if (live && ok[0]) q = *reinterpret_cast<const Pack<T, L>*>(p);
  } else {
#pragma unroll
    for (int j = 0; j < L; ++j)
      if (live && ok[j]) q.v[j] = p[32 * j];
  }
}
template <bool VEC, class T, int L>
__device__ __forceinline__ void store_lane(T* p, const bool (&ok)[L], const float (&v)[L]) {
  if (VEC) {
    if (!ok[0]) return;
    Pack<T, L> q;
#pragma unroll
    for (int j = 0; j < L; ++j) q.v[j] = from_f32<T>(v[j]);
    *reinterpret_cast<Pack<T, L>*>(p) = q;
  } else {
#pragma unroll
    for (int j = 0; j < L; ++j)
      if (ok[j]) p[32 * j] = from_f32<T>(v[j]);
  }
}

// kRun rows of one tensor, from scan index u on.
template <bool VEC, class T, int L>
__device__ __forceinline__ void load_run(const ScanArgs<T>& a, const Place<T, L, VEC>& at,
                                         const Seq<const T>& s, int64_t u, bool whole,
                                         Pack<T, L> (&q)[kRun]) {
  const int64_t dir = a.reverse ? -1 : 1, t0 = at.time(a, u);
  const T* p = s.row(at.b, t0) + at.column0();
#pragma unroll
  for (int i = 0; i < kRun; ++i) {
    const int64_t t = t0 + dir * i;
    load_lane<VEC>(p, at.ok, s.p && (whole || t < at.len), q[i]);
    p += dir * s.st;
  }
}

// The state that enters this CTA's segment: the segments before it, in order,
// after `first`.  For slot tid of the tile.
template <class T, int L, bool VEC>
__device__ __forceinline__ float enter_segment(const ScanArgs<T>& a, const Place<T, L, VEC>& at,
                                               bool descending, int64_t d) {
  float state = a.first ? a.first[at.b * a.D + d] : 0.f;
  const float2* p = a.composed + at.b * a.segments * a.D + d;
  const int n = descending ? a.segments - 1 - at.segment : at.segment;
#pragma unroll 8
  for (int k = 0; k < n; ++k) {
    const float2 q = p[(descending ? a.segments - 1 - k : k) * a.D];
    state = fmaf(q.x, state, q.y);
  }
  return state;
}

// Composes every segment that another one follows: (P, S) of the state, or
// with BWD of mu.  A warp composes one eighth of the segment's runs of eight
// positions, in scan order.
template <class T, int L, bool VEC, bool BWD>
__global__ void __launch_bounds__(32 * kWarps) compose_kernel(const ScanArgs<T> a) {
  using Pl = Place<T, L, VEC>;
  const Pl at(a);
  if (at.segment == (BWD ? 0 : a.segments - 1)) return;
  __shared__ float2 part[kWarps][Pl::kTile];
  const int64_t c0 = at.segment * a.per, c1 = min(c0 + a.per, a.chunks);
  const int64_t runs = c1 - c0;  // of a warp: the segment has kWarps times as many
  float2 sum[L];
#pragma unroll
  for (int j = 0; j < L; ++j) sum[j] = make_float2(1.f, 0.f);
  Pack<T, L> v[kRun], g[kRun];
  const auto index = [&](int64_t r) {
    return c0 * kChunk + (at.w * runs + (BWD ? runs - 1 - r : r)) * kRun;
  };
  const auto fetch = [&](int64_t r) {
    const int64_t u = index(r);
    const bool whole = at.whole(a, u, kRun);
    load_run<VEC, T, L>(a, at, BWD ? a.dh : a.x, u, whole, v);
    load_run<VEC, T, L>(a, at, a.g, u, whole, g);
  };
  fetch(0);
  for (int64_t r = 0; r < runs; ++r) {
    const int64_t u = index(r);
    const bool whole = at.whole(a, u, kRun);
    float f[kRun][L], s[kRun][L];
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const int64_t t = at.time(a, u + i);
      const bool live = whole || t < at.len;
#pragma unroll
      for (int j = 0; j < L; ++j) {
        float n;
        sigmoid_pair<T, true>(to_f32(g[i].v[j]), f[i][j], n);
        s[i][j] = BWD ? to_f32(v[i].v[j]) : n * to_f32(v[i].v[j]);
        if (!live) f[i][j] = 1.f, s[i][j] = 0.f;
      }
    }
    if (r + 1 < runs) fetch(r + 1);
#pragma unroll
    for (int k = 0; k < kRun; ++k) {
      const int i = BWD ? kRun - 1 - k : k;
#pragma unroll
      for (int j = 0; j < L; ++j) {
        sum[j].y = BWD ? f[i][j] * (s[i][j] + sum[j].y) : fmaf(f[i][j], sum[j].y, s[i][j]);
        sum[j].x *= f[i][j];
      }
    }
  }
#pragma unroll
  for (int j = 0; j < L; ++j) part[at.w][at.lane + 32 * j] = sum[j];
  __syncthreads();
  const int tid = threadIdx.x;
  if (tid >= Pl::kTile || at.channel(tid) >= a.D) return;
  float2 own = make_float2(1.f, 0.f);
#pragma unroll
  for (int w = 0; w < kWarps; ++w) own = then(own, part[BWD ? kWarps - 1 - w : w][tid]);
  a.composed[(at.b * a.segments + at.segment) * a.D + at.channel(tid)] = own;
}

template <class T, int L, bool VEC>
__global__ void __launch_bounds__(32 * kWarps, 2) forward_kernel(const ScanArgs<T> a) {
  using Pl = Place<T, L, VEC>;
  constexpr int TILE = Pl::kTile;
  __shared__ float2 part[2][kWarps][TILE];
  __shared__ float enter[2][TILE];
  const Pl at(a);
  const int64_t dir = a.reverse ? -1 : 1;
  const int64_t c0 = at.segment * a.per, c1 = min(c0 + a.per, a.chunks);
  const int tid = threadIdx.x;
  Pack<T, L> x[kRun], g[kRun];
  const auto fetch = [&](int64_t c) {
    const int64_t u = c * kChunk + at.w * kRun;
    const bool whole = at.whole(a, c * kChunk, kChunk);
    load_run<VEC, T, L>(a, at, a.x, u, whole, x);
    load_run<VEC, T, L>(a, at, a.g, u, whole, g);
  };
  fetch(c0);
  if (tid < TILE) {
    const int64_t d = at.channel(tid);
    enter[0][tid] = d < a.D ? enter_segment(a, at, false, d) : 0.f;
  }
  for (int64_t c = c0; c < c1; ++c) {
    const int turn = (int)(c - c0) & 1;
    const int64_t t0 = at.time(a, c * kChunk + at.w * kRun);
    const bool whole = at.whole(a, c * kChunk, kChunk);
    float f[kRun][L], s[kRun][L];
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const int64_t t = t0 + dir * i;
      const bool live = whole || t < at.len;
#pragma unroll
      for (int j = 0; j < L; ++j) {
        float n;
        sigmoid_pair<T, true>(to_f32(g[i].v[j]), f[i][j], n);
        s[i][j] = n * to_f32(x[i].v[j]);
        if (!live) f[i][j] = 1.f, s[i][j] = 0.f;
      }
    }
    if (c + 1 < c1) fetch(c + 1);
#pragma unroll
    for (int j = 0; j < L; ++j) {
      float2 q = make_float2(f[0][j], s[0][j]);
#pragma unroll
      for (int i = 1; i < kRun; ++i) q = then(q, make_float2(f[i][j], s[i][j]));
      part[turn][at.w][at.lane + 32 * j] = q;
    }
    __syncthreads();
    float h[L];
#pragma unroll
    for (int j = 0; j < L; ++j) h[j] = enter[turn][at.lane + 32 * j];
    if (a.carry && at.w == 0)
#pragma unroll
      for (int j = 0; j < L; ++j)
        if (at.ok[j]) a.carry[(at.b * a.chunks + c) * a.D + at.channel(at.lane + 32 * j)] = h[j];
    for (int w = 0; w < at.w; ++w)
#pragma unroll
      for (int j = 0; j < L; ++j) {
        const float2 q = part[turn][w][at.lane + 32 * j];
        h[j] = fmaf(q.x, h[j], q.y);
      }
    T* hp = a.h.row(at.b, t0) + at.column0();
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const int64_t t = t0 + dir * i;
      float out[L];
#pragma unroll
      for (int j = 0; j < L; ++j) {
        h[j] = fmaf(f[i][j], h[j], s[i][j]);
        out[j] = whole || t < at.len ? h[j] : 0.f;
      }
      if (whole || t < a.T_) store_lane<VEC>(hp, at.ok, out);
      hp += dir * a.h.st;
    }
    if (at.w == kWarps - 1)
#pragma unroll
      for (int j = 0; j < L; ++j) {
        enter[turn ^ 1][at.lane + 32 * j] = h[j];
        if (a.last && c + 1 == a.chunks && at.ok[j])
          a.last[at.b * a.D + at.channel(at.lane + 32 * j)] = h[j];
      }
  }
}

template <class T, int L, bool VEC>
__global__ void __launch_bounds__(32 * kWarps, 2) backward_kernel(const ScanArgs<T> a) {
  using Pl = Place<T, L, VEC>;
  constexpr int TILE = Pl::kTile;
  __shared__ float2 part[2][kWarps][TILE];
  __shared__ float mpart[2][kWarps][TILE];
  __shared__ float enter[2][TILE];
  const Pl at(a);
  const int64_t dir = a.reverse ? -1 : 1;
  const int64_t c0 = at.segment * a.per, c1 = min(c0 + a.per, a.chunks);
  const int tid = threadIdx.x;
  Pack<T, L> xq[kRun], gq[kRun], dq[kRun];
  float before[L];  // the state entering the chunk
  const auto fetch = [&](int64_t c) {
    const int64_t u = c * kChunk + at.w * kRun;
    const bool whole = at.whole(a, c * kChunk, kChunk);
    load_run<VEC, T, L>(a, at, a.x, u, whole, xq);
    load_run<VEC, T, L>(a, at, a.g, u, whole, gq);
    load_run<VEC, T, L>(a, at, a.dh, u, whole, dq);
#pragma unroll
    for (int j = 0; j < L; ++j)
      before[j] = at.ok[j] ? a.carry[(at.b * a.chunks + c) * a.D + at.channel(at.lane + 32 * j)] : 0.f;
  };
  fetch(c1 - 1);
  if (tid < TILE) {
    const int64_t d = at.channel(tid);
    enter[0][tid] = d < a.D ? enter_segment(a, at, true, d) : 0.f;
  }
  for (int64_t c = c1 - 1; c >= c0; --c) {
    const int turn = (int)(c1 - 1 - c) & 1;
    const int64_t t0 = at.time(a, c * kChunk + at.w * kRun);
    const bool whole = at.whole(a, c * kChunk, kChunk);
    float f[kRun][L], n[kRun][L], x[kRun][L], dh[kRun][L], h[L];
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const int64_t t = t0 + dir * i;
      const bool live = whole || t < at.len;
#pragma unroll
      for (int j = 0; j < L; ++j) {
        sigmoid_pair<T, true>(to_f32(gq[i].v[j]), f[i][j], n[i][j]);
        if (!live) f[i][j] = 1.f, n[i][j] = 0.f;
        x[i][j] = to_f32(xq[i].v[j]);
        dh[i][j] = to_f32(dq[i].v[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < L; ++j) h[j] = before[j];
    if (c > c0) fetch(c - 1);
#pragma unroll
    for (int j = 0; j < L; ++j) {
      float2 q = make_float2(1.f, 0.f);
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < kRun; ++i) q = then(q, make_float2(f[i][j], n[i][j] * x[i][j]));
#pragma unroll
      for (int i = kRun - 1; i >= 0; --i) m = f[i][j] * (dh[i][j] + m);
      part[turn][at.w][at.lane + 32 * j] = q;
      mpart[turn][at.w][at.lane + 32 * j] = m;
    }
    __syncthreads();
    float mu[L];
#pragma unroll
    for (int j = 0; j < L; ++j) {
      const int slot = at.lane + 32 * j;
      mu[j] = enter[turn][slot];
      for (int w = 0; w < at.w; ++w) {
        const float2 q = part[turn][w][slot];
        h[j] = fmaf(q.x, h[j], q.y);
      }
      for (int w = kWarps - 1; w > at.w; --w)
        mu[j] = fmaf(part[turn][w][slot].x, mu[j], mpart[turn][w][slot]);
#pragma unroll
      for (int i = 0; i < kRun; ++i) {  // x becomes h_{u-1} - x_u
        const float prev = h[j];
        h[j] = fmaf(f[i][j], h[j], n[i][j] * x[i][j]);
        x[i][j] = prev - x[i][j];
      }
    }
    T* xp = a.dx.row(at.b, t0 + dir * (kRun - 1)) + at.column0();
    T* gp = a.dg.row(at.b, t0 + dir * (kRun - 1)) + at.column0();
#pragma unroll
    for (int i = kRun - 1; i >= 0; --i) {
      const int64_t t = t0 + dir * i;
      const bool live = whole || t < at.len;
      float dx[L], dg[L];
#pragma unroll
      for (int j = 0; j < L; ++j) {
        const float lam = dh[i][j] + mu[j];
        mu[j] = f[i][j] * lam;
        dx[j] = live ? lam * n[i][j] : 0.f;
        dg[j] = live ? mu[j] * n[i][j] * x[i][j] : 0.f;
      }
      if (whole || t < a.T_) {
        store_lane<VEC>(xp, at.ok, dx);
        store_lane<VEC>(gp, at.ok, dg);
      }
      xp -= dir * a.dx.st;
      gp -= dir * a.dg.st;
    }
    if (at.w == 0)
#pragma unroll
      for (int j = 0; j < L; ++j) {
        enter[turn ^ 1][at.lane + 32 * j] = mu[j];
        if (a.last && c == 0 && at.ok[j])
          a.last[at.b * a.D + at.channel(at.lane + 32 * j)] = mu[j];
      }
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
      sigmoid_pair<T, true>(to_f32(gv.v[j]), f, m);
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

// ---------------------------------------------------------------------------
// The walk with its inputs brought by bulk copies: rows on 16-byte boundaries.
// A producer thread keeps a ring of chunks of every input on their way to
// shared memory; rows there lie at fixed offsets, so reading them costs no
// address arithmetic, and nothing waits in registers.  A lane takes H pairs of
// channels: two of 16-bit types forward, one else (the run's factors and, in
// the backward, its inputs fill the registers).  Products and sums go two
// channels to an instruction: issue slots are what comes next after DRAM.
// ---------------------------------------------------------------------------
template <class T>
constexpr int forward_pairs() { return sizeof(T) == 2 ? 2 : 1; }
constexpr int kBackwardPairs = 1;
constexpr int box_bytes(int elem, int pairs) { return 64 * elem * pairs * kChunk; }
// chunks in the ring: what lets two CTAs share an SM
constexpr int kForwardStages = 3;
template <class T>
constexpr int backward_stages() { return sizeof(T) == 2 ? 3 : 2; }
constexpr int ring_bytes(int elem, int pairs, int tensors, int stages) {
  return tensors * stages * box_bytes(elem, pairs) + 128;
}

__device__ __forceinline__ void compute_barrier() {
  asm volatile("bar.sync 1, %0;" ::"n"(32 * kWarps) : "memory");
}

// A lane's pairs of row i of a warp's run, in scan order, in a tile in shared memory.
template <class T, int H>
__device__ __forceinline__ void tile_row(const unsigned char* tile, int w, int lane, int i,
                                         bool reverse, float2 (&v)[H]) {
  constexpr int kBytes = 2 * H * (int)sizeof(T);
  const int row = reverse ? kChunk - 1 - (w * kRun + i) : w * kRun + i;
  const Pack<Pack<T, 2>, H> q =
      *reinterpret_cast<const Pack<Pack<T, 2>, H>*>(tile + (row * 32 + lane) * kBytes);
#pragma unroll
  for (int j = 0; j < H; ++j) v[j] = to_f32x2(q.v[j]);
}
template <class T, int H>
__device__ __forceinline__ void store_pairs(T* p, bool ok, const float2 (&v)[H]) {
  if (!ok) return;
  Pack<Pack<T, 2>, H> q;
#pragma unroll
  for (int j = 0; j < H; ++j) q.v[j] = from_f32x2<T>(v[j]);
  *reinterpret_cast<Pack<Pack<T, 2>, H>*>(p) = q;
}

// (P, S) of two channels
struct Affine {
  float2 P, S;
};
__device__ __forceinline__ Affine then(const Affine& a, const Affine& b) {  // b after a
  return Affine{__fmul2_rn(b.P, a.P), __ffma2_rn(b.P, a.S, b.S)};
}

// Keeps the ring full: N tensors a chunk, `descending` in scan order for the backward.
template <int BOX, class T, int N, int STAGES, class At>
__device__ void produce(const ScanArgs<T>& a, const At& at, const CUtensorMap* const (&maps)[N],
                        unsigned char* ring, uint64_t* full, uint64_t* empty, int64_t c0,
                        int64_t c1, bool descending) {
  int it = 0;
  const int n = (int)(c1 - c0);
  for (; it < n; ++it) {
    const int slot = it % STAGES;
    if (it >= STAGES && !barrier_wait(&empty[slot], (unsigned)(it / STAGES - 1) & 1)) break;
    const int64_t c = descending ? c1 - 1 - it : c0 + it;
    const int row = (int)(a.reverse ? a.chunks - 1 - c : c) * kChunk;
    expect_bytes(&full[slot], N * BOX);
#pragma unroll
    for (int k = 0; k < N; ++k)
      fetch_tile(smem_addr(ring + (slot * N + k) * BOX), maps[k], (int)at.d0, row, (int)at.b,
                 &full[slot]);
  }
  // no copy may still be in flight when the CTA's memory is given up
  for (int k = it > STAGES ? it - STAGES : 0; k < it; ++k)
    barrier_wait(&full[k % STAGES], (unsigned)(k / STAGES) & 1);
}

template <int STAGES>
__device__ __forceinline__ void init_ring(uint64_t* full, uint64_t* empty) {
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      barrier_init(&full[s], 1);
      barrier_init(&empty[s], kWarps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
}

__device__ __forceinline__ unsigned char* align_ring(unsigned char* p) {
  return reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(p) + 127) &
                                          ~(uintptr_t)127);
}

// The chunks of a segment that hold valid positions, in scan order.  The other
// chunks take no part in a walk: the state passes them unchanged.
struct Range {
  int64_t c0, c1;  // the segment's chunks
  int64_t v0, v1;  // those with valid positions
};
template <class T, class At>
__device__ __forceinline__ Range range_of(const ScanArgs<T>& a, const At& at) {
  Range r;
  r.c0 = at.segment * a.per;
  r.c1 = min(r.c0 + a.per, a.chunks);
  const int64_t n = (at.len + kChunk - 1) / kChunk;
  r.v0 = a.reverse ? max(r.c0, a.chunks - n) : r.c0;
  r.v1 = a.reverse ? r.c1 : min(r.c1, n);
  if (r.v1 < r.v0) r.v1 = r.v0;
  return r;
}
// Zeros in every row of the segment's other chunks, by the CTA's first 256 threads.
template <int H, class T, class At>
__device__ void clear_rest(const ScanArgs<T>& a, const At& at, const Range& r, const Seq<T>& out) {
  const int64_t rest = (r.c1 - r.c0) - (r.v1 - r.v0);
  const float2 zero[H] = {};
  for (int64_t k = 0; k < rest; ++k) {
    const int64_t c = a.reverse ? r.c0 + k : r.v1 + k;
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const int64_t t = at.time(a, c * kChunk + at.w * kRun + i);
      if (t < a.T_) store_pairs(out.row(at.b, t) + at.column0(), at.ok[0], zero);
    }
  }
}
// First channel of pair number k = lane + 32 j of a tile.
template <int H>
__device__ __forceinline__ int pair_channel(int k) { return (k & 31) * 2 * H + 2 * (k >> 5); }

// The state entering the segment, of the pair of channels that thread tid < 32 H looks after.
template <int H, class T, class At>
__device__ __forceinline__ float2 enter_pair(const ScanArgs<T>& a, const At& at, bool descending) {
  const int64_t d = at.d0 + pair_channel<H>(threadIdx.x);
  if (d >= a.D) return both(0.f);
  return make_float2(enter_segment(a, at, descending, d), enter_segment(a, at, descending, d + 1));
}

struct Masked { static constexpr bool value = true; };
struct Whole { static constexpr bool value = false; };

// The forward walk, or with COMPOSE its (P, S) alone.
template <class T, bool COMPOSE>
__global__ void __launch_bounds__(32 * kWarps + 32, 2)
    forward_bulk_kernel(const ScanArgs<T> a, const __grid_constant__ CUtensorMap x_map,
                        const __grid_constant__ CUtensorMap g_map) {
  constexpr int H = forward_pairs<T>(), PAIRS = 32 * H, ST = kForwardStages;
  constexpr int kBox = box_bytes(sizeof(T), H);
  constexpr int kParts = COMPOSE ? kWarps : kWarps - 1;  // the last warp's has no reader in a walk
  extern __shared__ unsigned char raw[];
  __shared__ uint64_t full[ST], empty[ST];
  __shared__ Affine part[2][kParts][PAIRS];
  __shared__ float2 enter[2][COMPOSE ? 1 : PAIRS];
  unsigned char* ring = align_ring(raw);
  const Place<T, 2 * H, true> at(a);
  if (COMPOSE && at.segment == a.segments - 1) return;
  const Range range = range_of(a, at);
  const int tid = threadIdx.x;
  init_ring<ST>(full, empty);
  if (at.w == kWarps) {
    const CUtensorMap* const maps[2] = {&x_map, &g_map};
    if (at.lane == 0)
      produce<kBox, T, 2, ST>(a, at, maps, ring, full, empty, range.v0, range.v1, false);
    return;
  }
  Affine own{both(1.f), both(0.f)};
  if (!COMPOSE && tid < PAIRS) enter[0][tid] = enter_pair<H>(a, at, false);
  bool ok = true;
  const int64_t step = a.reverse ? -a.h.st : a.h.st;
  int turn = 0;
  const auto chunk = [&](int64_t c, auto kind) {
    constexpr bool kMasked = decltype(kind)::value;
    const int it = (int)(c - range.v0), slot = it % ST;
    const int64_t t0 = at.time(a, c * kChunk + at.w * kRun), dir = a.reverse ? -1 : 1;
    if (ok) ok = barrier_wait(&full[slot], (unsigned)(it / ST) & 1);
    const unsigned char* xt = ring + slot * 2 * kBox;
    Affine u[kRun][H];
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      float2 x[H], g[H];
      tile_row<T>(xt, at.w, at.lane, i, a.reverse, x);
      tile_row<T>(xt + kBox, at.w, at.lane, i, a.reverse, g);
#pragma unroll
      for (int j = 0; j < H; ++j) {
        float2 n;
        sigmoid_pair2<T, true>(g[j], u[i][j].P, n);
        u[i][j].S = __fmul2_rn(n, x[j]);
        if (kMasked && t0 + dir * i >= at.len) u[i][j] = Affine{both(1.f), both(0.f)};
      }
    }
    __syncwarp();
    if (at.lane == 0) barrier_arrive_here(&empty[slot]);
    if (!ok) u[0][0].P.x = __uint_as_float(0x7fc00000u);  // a copy that never came shows as NaN
    if (COMPOSE || at.w < kParts)
#pragma unroll
      for (int j = 0; j < H; ++j) {
        Affine q = u[0][j];
#pragma unroll
        for (int i = 1; i < kRun; ++i) q = then(q, u[i][j]);
        part[turn][at.w][at.lane + 32 * j] = q;
      }
    compute_barrier();
    if (COMPOSE) {
      if (tid < PAIRS)
#pragma unroll
        for (int w = 0; w < kParts; ++w) own = then(own, part[turn][w][tid]);
      turn ^= 1;
      return;
    }
    float2 h[H];
#pragma unroll
    for (int j = 0; j < H; ++j) h[j] = enter[turn][at.lane + 32 * j];
    if (a.carry && at.w == 0 && at.ok[0]) {
      float* p = a.carry + (at.b * a.chunks + c) * a.D + at.column0();
#pragma unroll
      for (int j = 0; j < H; ++j) p[2 * j] = h[j].x, p[2 * j + 1] = h[j].y;
    }
    for (int w = 0; w < at.w; ++w)
#pragma unroll
      for (int j = 0; j < H; ++j) {
        const Affine q = part[turn][w][at.lane + 32 * j];
        h[j] = __ffma2_rn(q.P, h[j], q.S);
      }
    T* hp = a.h.row(at.b, t0) + at.column0();
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const int64_t t = t0 + dir * i;
      float2 out[H];
#pragma unroll
      for (int j = 0; j < H; ++j) {
        h[j] = __ffma2_rn(u[i][j].P, h[j], u[i][j].S);
        out[j] = kMasked && t >= at.len ? both(0.f) : h[j];
      }
      if (!kMasked || t < a.T_) store_pairs(hp, at.ok[0], out);
      hp += step;
    }
    turn ^= 1;
    if (at.w == kWarps - 1)
#pragma unroll
      for (int j = 0; j < H; ++j) enter[turn][at.lane + 32 * j] = h[j];
  };
  for (int64_t c = range.v0; c < range.v1; ++c) {
    if (at.whole(a, c * kChunk, kChunk))
      chunk(c, Whole());
    else
      chunk(c, Masked());
  }
  const int64_t d = at.d0 + pair_channel<H>(tid);
  if (COMPOSE) {
    if (tid < PAIRS && d < a.D) {
      float2* p = a.composed + (at.b * a.segments + at.segment) * a.D + d;
      p[0] = make_float2(own.P.x, own.S.x);
      p[1] = make_float2(own.P.y, own.S.y);
    }
    return;
  }
  clear_rest<H>(a, at, range, a.h);
  if (!a.last || at.segment != a.segments - 1) return;
  compute_barrier();
  if (tid < PAIRS && d < a.D) {
    a.last[at.b * a.D + d] = enter[turn][tid].x;
    a.last[at.b * a.D + d + 1] = enter[turn][tid].y;
  }
}

// mu's (P, S) of every segment but the first.
template <class T>
__global__ void __launch_bounds__(32 * kWarps + 32, 2)
    backward_compose_kernel(const ScanArgs<T> a, const __grid_constant__ CUtensorMap d_map,
                            const __grid_constant__ CUtensorMap g_map) {
  constexpr int H = kBackwardPairs, PAIRS = 32 * H, ST = backward_stages<T>();
  constexpr int kBox = box_bytes(sizeof(T), H);
  extern __shared__ unsigned char raw[];
  __shared__ uint64_t full[ST], empty[ST];
  __shared__ Affine part[2][kWarps][PAIRS];
  unsigned char* ring = align_ring(raw);
  const Place<T, 2 * H, true> at(a);
  if (at.segment == 0) return;
  const Range range = range_of(a, at);
  const int tid = threadIdx.x;
  init_ring<ST>(full, empty);
  if (at.w == kWarps) {
    const CUtensorMap* const maps[2] = {&d_map, &g_map};
    if (at.lane == 0)
      produce<kBox, T, 2, ST>(a, at, maps, ring, full, empty, range.v0, range.v1, true);
    return;
  }
  Affine own{both(1.f), both(0.f)};
  bool ok = true;
  int turn = 0;
  const auto chunk = [&](int64_t c, auto kind) {
    constexpr bool kMasked = decltype(kind)::value;
    const int it = (int)(range.v1 - 1 - c), slot = it % ST;
    const int64_t t0 = at.time(a, c * kChunk + at.w * kRun), dir = a.reverse ? -1 : 1;
    if (ok) ok = barrier_wait(&full[slot], (unsigned)(it / ST) & 1);
    const unsigned char* dt = ring + slot * 2 * kBox;
    Affine q[H];
#pragma unroll
    for (int j = 0; j < H; ++j)
      q[j] = Affine{both(ok ? 1.f : __uint_as_float(0x7fc00000u)), both(0.f)};
#pragma unroll
    for (int i = kRun - 1; i >= 0; --i) {
      float2 d[H], g[H];
      tile_row<T>(dt, at.w, at.lane, i, a.reverse, d);
      tile_row<T>(dt + kBox, at.w, at.lane, i, a.reverse, g);
      if (kMasked && t0 + dir * i >= at.len) continue;
#pragma unroll
      for (int j = 0; j < H; ++j) {
        float2 f, n;
        sigmoid_pair2<T, true>(g[j], f, n);
        q[j].P = __fmul2_rn(q[j].P, f);
        q[j].S = __fmul2_rn(f, __fadd2_rn(d[j], q[j].S));
      }
    }
    __syncwarp();
    if (at.lane == 0) barrier_arrive_here(&empty[slot]);
#pragma unroll
    for (int j = 0; j < H; ++j) part[turn][at.w][at.lane + 32 * j] = q[j];
    compute_barrier();
    if (tid < PAIRS)
#pragma unroll
      for (int w = kWarps - 1; w >= 0; --w) own = then(own, part[turn][w][tid]);
    turn ^= 1;
  };
  for (int64_t c = range.v1 - 1; c >= range.v0; --c) {
    if (at.whole(a, c * kChunk, kChunk))
      chunk(c, Whole());
    else
      chunk(c, Masked());
  }
  const int64_t d = at.d0 + pair_channel<H>(tid);
  if (tid < PAIRS && d < a.D) {
    float2* p = a.composed + (at.b * a.segments + at.segment) * a.D + d;
    p[0] = make_float2(own.P.x, own.S.x);
    p[1] = make_float2(own.P.y, own.S.y);
  }
}

template <class T>
__global__ void __launch_bounds__(32 * kWarps + 32, 2)
    backward_bulk_kernel(const ScanArgs<T> a, const __grid_constant__ CUtensorMap x_map,
                         const __grid_constant__ CUtensorMap g_map,
                         const __grid_constant__ CUtensorMap d_map) {
  constexpr int H = kBackwardPairs, PAIRS = 32 * H, ST = backward_stages<T>();
  constexpr int kBox = box_bytes(sizeof(T), H);
  extern __shared__ unsigned char raw[];
  __shared__ uint64_t full[ST], empty[ST];
  __shared__ Affine part[2][kWarps][PAIRS];
  __shared__ float2 mpart[2][kWarps][PAIRS];
  __shared__ float2 enter[2][PAIRS];
  unsigned char* ring = align_ring(raw);
  const Place<T, 2 * H, true> at(a);
  const Range range = range_of(a, at);
  const int tid = threadIdx.x;
  init_ring<ST>(full, empty);
  if (at.w == kWarps) {
    const CUtensorMap* const maps[3] = {&x_map, &g_map, &d_map};
    if (at.lane == 0)
      produce<kBox, T, 3, ST>(a, at, maps, ring, full, empty, range.v0, range.v1, true);
    return;
  }
  if (tid < PAIRS) enter[0][tid] = enter_pair<H>(a, at, true);
  bool ok = true;
  int turn = 0;
  const auto chunk = [&](int64_t c, auto kind) {
    constexpr bool kMasked = decltype(kind)::value;
    const int it = (int)(range.v1 - 1 - c), slot = it % ST;
    const int64_t t0 = at.time(a, c * kChunk + at.w * kRun), dir = a.reverse ? -1 : 1;
    const auto off = [&](int i) { return kMasked && t0 + dir * i >= at.len; };
    float2 h[H] = {};
    if (at.ok[0]) {
      const float* p = a.carry + (at.b * a.chunks + c) * a.D + at.column0();
#pragma unroll
      for (int j = 0; j < H; ++j) h[j] = make_float2(p[2 * j], p[2 * j + 1]);
    }
    if (ok) ok = barrier_wait(&full[slot], (unsigned)(it / ST) & 1);
    const unsigned char* xt = ring + slot * 3 * kBox;
    const unsigned char *gt = xt + kBox, *dt = gt + kBox;
    // the factors and inputs of the run; masked positions have f = 1 and zeros
    float2 f[kRun][H], n[kRun][H], x[kRun][H], d[kRun][H];
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      float2 g[H];
      tile_row<T>(gt, at.w, at.lane, i, a.reverse, g);
      tile_row<T>(xt, at.w, at.lane, i, a.reverse, x[i]);
      tile_row<T>(dt, at.w, at.lane, i, a.reverse, d[i]);
#pragma unroll
      for (int j = 0; j < H; ++j) {
        sigmoid_pair2<T, true>(g[j], f[i][j], n[i][j]);
        if (off(i)) f[i][j] = both(1.f), n[i][j] = x[i][j] = d[i][j] = both(0.f);
      }
    }
    __syncwarp();
    if (at.lane == 0) barrier_arrive_here(&empty[slot]);
    if (!ok) f[0][0].x = __uint_as_float(0x7fc00000u);  // a copy that never came shows as NaN
#pragma unroll
    for (int j = 0; j < H; ++j) {
      Affine q{f[0][j], __fmul2_rn(n[0][j], x[0][j])};
#pragma unroll
      for (int i = 1; i < kRun; ++i) q = then(q, Affine{f[i][j], __fmul2_rn(n[i][j], x[i][j])});
      float2 m = both(0.f);
#pragma unroll
      for (int i = kRun - 1; i >= 0; --i) m = __fmul2_rn(f[i][j], __fadd2_rn(d[i][j], m));
      part[turn][at.w][at.lane + 32 * j] = q;
      mpart[turn][at.w][at.lane + 32 * j] = m;
    }
    compute_barrier();
    float2 mu[H];
#pragma unroll
    for (int j = 0; j < H; ++j) {
      const int at_slot = at.lane + 32 * j;
      mu[j] = enter[turn][at_slot];
      for (int w = 0; w < at.w; ++w) {
        const Affine q = part[turn][w][at_slot];
        h[j] = __ffma2_rn(q.P, h[j], q.S);
      }
      for (int w = kWarps - 1; w > at.w; --w)
        mu[j] = __ffma2_rn(part[turn][w][at_slot].P, mu[j], mpart[turn][w][at_slot]);
#pragma unroll
      for (int i = 0; i < kRun; ++i) {  // x becomes (1 - f) (h_{u-1} - x_u)
        const float2 before = h[j];
        h[j] = __ffma2_rn(f[i][j], before, __fmul2_rn(n[i][j], x[i][j]));
        x[i][j] = __fmul2_rn(n[i][j], sub2(before, x[i][j]));
      }
    }
    const int64_t last = t0 + dir * (kRun - 1);
    T* xp = a.dx.row(at.b, last) + at.column0();
    T* gp = a.dg.row(at.b, last) + at.column0();
#pragma unroll
    for (int i = kRun - 1; i >= 0; --i) {
      float2 dx[H], dg[H];
#pragma unroll
      for (int j = 0; j < H; ++j) {
        const float2 lam = __fadd2_rn(d[i][j], mu[j]);
        mu[j] = __fmul2_rn(f[i][j], lam);
        dx[j] = off(i) ? both(0.f) : __fmul2_rn(lam, n[i][j]);
        dg[j] = off(i) ? both(0.f) : __fmul2_rn(mu[j], x[i][j]);
      }
      if (!kMasked || t0 + dir * i < a.T_) {
        store_pairs(xp, at.ok[0], dx);
        store_pairs(gp, at.ok[0], dg);
      }
      xp -= dir * a.dx.st;
      gp -= dir * a.dg.st;
    }
    turn ^= 1;
    if (at.w == 0)
#pragma unroll
      for (int j = 0; j < H; ++j) enter[turn][at.lane + 32 * j] = mu[j];
  };
  for (int64_t c = range.v1 - 1; c >= range.v0; --c) {
    if (at.whole(a, c * kChunk, kChunk))
      chunk(c, Whole());
    else
      chunk(c, Masked());
  }
  clear_rest<H>(a, at, range, a.dx);
  clear_rest<H>(a, at, range, a.dg);
  if (!a.last || at.segment != 0) return;
  compute_barrier();
  const int64_t d = at.d0 + pair_channel<H>(tid);
  if (tid < PAIRS && d < a.D) {
    a.last[at.b * a.D + d] = enter[turn][tid].x;
    a.last[at.b * a.D + d + 1] = enter[turn][tid].y;
  }
}

int64_t chunks_of(int64_t T) { return (T + kChunk - 1) / kChunk; }

// Channels of a lane where rows are read by plain loads.
template <class T>
constexpr int forward_lane() { return 2 * forward_pairs<T>(); }
template <class T>
constexpr int backward_lane() { return sizeof(T) == 2 ? 2 : 1; }

struct Cut {
  int tiles, segments;
  int64_t per;
};
// Segments: as many as fill the device's CTA slots once.
Cut cut_of(int64_t B, int64_t T, int64_t D, int tile) {
  Cut c;
  c.tiles = (int)((D + tile - 1) / tile);
  const int64_t columns = B * c.tiles, chunks = chunks_of(T), slots = 2 * device_sm_count();
  const int64_t want = columns ? std::max<int64_t>(1, std::min(slots / columns, chunks)) : 1;
  c.per = (chunks + want - 1) / want;
  c.segments = c.per ? (int)((chunks + c.per - 1) / c.per) : 1;
  return c;
}

template <class T>
ScanArgs<T> scan_args(const semicrf_recurrence* p, int tile, void* workspace) {
  const Cut c = cut_of(p->batch, p->T, p->D, tile);
  ScanArgs<T> a{};
  a.B = p->batch;
  a.T_ = p->T;
  a.D = p->D;
  a.chunks = chunks_of(p->T);
  a.per = c.per;
  a.tiles = c.tiles;
  a.segments = c.segments;
  a.reverse = p->reverse != 0;
  a.x = as_seq<const T>(p->x);
  a.g = as_seq<const T>(p->gate);
  a.lengths = p->lengths;
  a.composed = static_cast<float2*>(workspace);
  return a;
}

// Without positions the last state is the first.
int copy_state(const semicrf_recurrence* p, const float* first, float* last, cudaStream_t stream) {
  if (!last) return SEMICRF_OK;
  const size_t bytes = sizeof(float) * p->batch * p->D;
  const cudaError_t e = first ? cudaMemcpyAsync(last, first, bytes, cudaMemcpyDeviceToDevice, stream)
                              : cudaMemsetAsync(last, 0, bytes, stream);
  return e == cudaSuccess ? SEMICRF_OK : SEMICRF_ERR_CUDA;
}

template <class T, int L, bool VEC, bool BWD>
int launch_scan(const ScanArgs<T>& a, cudaStream_t stream) {
  const unsigned grid = (unsigned)(a.B * a.tiles * a.segments);
  if (a.segments > 1) compose_kernel<T, L, VEC, BWD><<<grid, 32 * kWarps, 0, stream>>>(a);
  if constexpr (BWD)
    backward_kernel<T, L, VEC><<<grid, 32 * kWarps, 0, stream>>>(a);
  else
    forward_kernel<T, L, VEC><<<grid, 32 * kWarps, 0, stream>>>(a);
  return launch_status();
}

// Whether bulk copies can read s: 16-byte rows, no two of them overlapping.
bool bulk_readable(const semicrf_sequence& s, int64_t B, int64_t T, int64_t D, int elem) {
  return s.data && T < (1ll << 30) && B < (1ll << 30) && seq_aligned(s, B, T, elem, 16 / elem) &&
         (T == 1 || (s.time_stride >= D && s.time_stride < (1ll << 36))) &&
         (B == 1 || (s.batch_stride >= D && s.batch_stride < (1ll << 36)));
}

template <class T>
bool sequence_map(CUtensorMap* map, const semicrf_sequence& s, int64_t B, int64_t T_, int64_t D,
                  int lane) {
  const CUtensorMapDataType type = sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : std::is_same<T, __half>::value
                                       ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                       : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const cuuint64_t row = (cuuint64_t)((D * sizeof(T) + 15) / 16 * 16);  // where there is one row
  const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)T_, (cuuint64_t)B};
  const cuuint64_t strides[2] = {T_ == 1 ? row : (cuuint64_t)s.time_stride * sizeof(T),
                                 B == 1 ? row : (cuuint64_t)s.batch_stride * sizeof(T)};
  const cuuint32_t box[3] = {(cuuint32_t)(32 * lane), (cuuint32_t)kChunk, 1};
  return make_tensor_map(map, type, 3, s.data, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
}

template <class K>
bool allow_shared(K kernel, int bytes) {
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) ==
         cudaSuccess;
}

template <class T>
int run_forward(const semicrf_recurrence* p, const semicrf_sequence& h, float* final_state,
                void* saved, void* workspace, cudaStream_t stream) {
  if (p->T == 0) return copy_state(p, p->initial_state, final_state, stream);
  constexpr int L = forward_lane<T>();
  ScanArgs<T> a = scan_args<T>(p, 32 * L, workspace);
  a.h = as_seq<T>(h);
  a.first = p->initial_state;
  a.last = final_state;
  a.carry = static_cast<float*>(saved);
  bool vec = p->D % L == 0;
  for (const semicrf_sequence* s : {&p->x, &p->gate, &h})
    vec = vec && seq_aligned(*s, a.B, a.T_, sizeof(T), L);
  if (vec && bulk_readable(p->x, a.B, a.T_, a.D, sizeof(T)) &&
      bulk_readable(p->gate, a.B, a.T_, a.D, sizeof(T))) {
    CUtensorMap xm, gm;
    const auto walk = forward_bulk_kernel<T, false>;
    const auto compose = forward_bulk_kernel<T, true>;
    constexpr int bytes = ring_bytes(sizeof(T), forward_pairs<T>(), 2, kForwardStages);
    // the runtime's calls come first: they give a thread that has none yet the
    // device's context, which encoding a map needs
    if (!allow_shared(walk, bytes) || !allow_shared(compose, bytes) ||
        !sequence_map<T>(&xm, p->x, a.B, a.T_, a.D, L) ||
        !sequence_map<T>(&gm, p->gate, a.B, a.T_, a.D, L))
      return SEMICRF_ERR_CUDA;
    const unsigned grid = (unsigned)(a.B * a.tiles * a.segments);
    if (a.segments > 1) compose<<<grid, 32 * kWarps + 32, bytes, stream>>>(a, xm, gm);
    walk<<<grid, 32 * kWarps + 32, bytes, stream>>>(a, xm, gm);
    return launch_status();
  }
  return vec ? launch_scan<T, L, true, false>(a, stream) : launch_scan<T, L, false, false>(a, stream);
}

template <class T>
int run_backward(const semicrf_recurrence* p, const void* saved, const semicrf_sequence& grad_h,
                 const float* grad_state, const semicrf_sequence& grad_x,
                 const semicrf_sequence& grad_gate, float* grad_initial, void* workspace,
                 cudaStream_t stream) {
  if (p->T == 0) return copy_state(p, grad_state, grad_initial, stream);
  constexpr int L = backward_lane<T>(), BL = 2 * kBackwardPairs;
  bool vec = p->D % L == 0, bulk = p->D % BL == 0;
  for (const semicrf_sequence* s : {&p->x, &p->gate, &grad_h, &grad_x, &grad_gate}) {
    vec = vec && seq_aligned(*s, p->batch, p->T, sizeof(T), L);
    bulk = bulk && seq_aligned(*s, p->batch, p->T, sizeof(T), BL);
  }
  for (const semicrf_sequence* s : {&p->x, &p->gate, &grad_h})
    bulk = bulk && bulk_readable(*s, p->batch, p->T, p->D, sizeof(T));
  ScanArgs<T> a = scan_args<T>(p, 32 * (bulk ? BL : L), workspace);
  a.dh = as_seq<const T>(grad_h);
  a.dx = as_seq<T>(grad_x);
  a.dg = as_seq<T>(grad_gate);
  a.first = grad_state;
  a.last = grad_initial;
  a.carry = const_cast<float*>(static_cast<const float*>(saved));
  if (bulk) {
    CUtensorMap xm, gm, dm;
    const auto walk = backward_bulk_kernel<T>;
    const auto compose = backward_compose_kernel<T>;
    constexpr int walk_bytes = ring_bytes(sizeof(T), kBackwardPairs, 3, backward_stages<T>());
    constexpr int compose_bytes = ring_bytes(sizeof(T), kBackwardPairs, 2, backward_stages<T>());
    if (!allow_shared(walk, walk_bytes) || !allow_shared(compose, compose_bytes) ||
        !sequence_map<T>(&xm, p->x, a.B, a.T_, a.D, BL) ||
        !sequence_map<T>(&gm, p->gate, a.B, a.T_, a.D, BL) ||
        !sequence_map<T>(&dm, grad_h, a.B, a.T_, a.D, BL))
      return SEMICRF_ERR_CUDA;
    const unsigned grid = (unsigned)(a.B * a.tiles * a.segments);
    if (a.segments > 1) compose<<<grid, 32 * kWarps + 32, compose_bytes, stream>>>(a, dm, gm);
    walk<<<grid, 32 * kWarps + 32, walk_bytes, stream>>>(a, xm, gm, dm);
    return launch_status();
  }
  return vec ? launch_scan<T, L, true, true>(a, stream) : launch_scan<T, L, false, true>(a, stream);
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
  const bool wide = p->dtype == SEMICRF_F32;
  const int tiles[3] = {32 * (wide ? forward_lane<float>() : forward_lane<__half>()),
                        32 * (wide ? backward_lane<float>() : backward_lane<__half>()),
                        64 * kBackwardPairs};
  int segments = 1;
  for (const int tile : tiles)
    segments = std::max(segments, cut_of(p->batch, p->T, p->D, tile).segments);
  return sizeof(float2) * p->batch * segments * p->D;
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
