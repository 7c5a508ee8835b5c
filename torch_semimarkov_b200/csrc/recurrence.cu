// recurrence.cu -- the gated linear recurrence, its gradient and its
// single-position form.
//
//   f = sigmoid(g),  h_u = f_u h_{u-1} + (1 - f_u) x_u
//
// u counts positions in scan order (t = u; reversed, from the end of the last
// chunk down); masked positions have f = 1 and contribute nothing, so they
// pass the state on.
// Steps compose: (P, S) with h_out = P h_in + S, P the product of f, S the
// result from zero.  f <= 1, so nothing overflows and no logarithm is needed.
//
// Gradient: lam_u = dh_u + f_{u+1} lam_{u+1}.  With mu_u = f_u lam_u it is
// the same recurrence from the other end, mu_u = f_u (dh_u + mu_{u+1}), and
//   dx_u = lam_u (1 - f_u),  dg_u = lam_u (h_{u-1} - x_u) f_u (1 - f_u).
// h_{u-1} is recomputed from the float32 state kept at the start of each
// chunk, which is more exact than rereading the rounded h and one read less.
//
// A CTA walks a column (a sequence's tile of channels) in chunks of 64
// positions.  Of its eight computing warps each owns eight consecutive
// positions of a chunk, a lane H pairs of channels.  Each warp composes its
// positions, one barrier a chunk makes the compositions known, and each warp
// goes from the state that entered the chunk over the earlier warps' to its
// own start.  Products and sums go two channels to an instruction.
//
// One or two more warps keep a ring of chunks of every input on their way to
// shared memory, so that nothing waits in registers.  Rows on 16-byte
// boundaries come by bulk tensor copies (TMA), one thread issuing 16 KB at a
// time.  Other rows come by 4-byte asynchronous copies of their aligned words;
// a 16-bit row that starts in the middle of a word lies one element on in its
// tile, and its first or last element, where the rest of the word is another
// row's, is copied by itself.
//
// Where there are fewer columns than CTAs fit on the device, a column's chunks
// are cut into segments, one to a CTA.  A first launch composes each segment
// but the last one; the walk then joins the segments before its own.  That
// reads two of the tensors twice, against a device mostly idle.  (A single
// pass in which CTAs wait for their predecessors' compositions was slower:
// each held its registers through several dependent trips to L2.)
// Every order of operations depends on sizes alone.
//
// Measured, bfloat16: batch 64 of 10^4 positions with ragged lengths, 512
// channels, forward 317 us and backward 645 us, where their bytes (3 and 5
// values an element) take 255 and 425 at the device's copy rate; float32, half
// the batch, 292 and 550 us for the same bytes.  The backward's 512 columns are
// 1.73 waves of CTAs; counted over both (64 x 1,500 x 512) 63% of issue slots and
// 47% of DRAM are used, and what its 18 warps an SM wait for most is the fixed
// latency of their own chains of steps.  One sequence of 10^6 positions: composing
// 355 us, walking 508 us, whose own bytes take 315 and 473.  Rows without 16-byte
// alignment (64 x 5,000 x 203): 217 and 418 us, 3.6 and 4.2 times their bytes (208
// channels take 124 and 193); their elements are loaded, converted and stored one
// by one.

#include <algorithm>
#include <type_traits>

#include "encoder_internal.cuh"
#include "tma.cuh"

namespace semicrf {
int device_sm_count();  // api.cu

namespace {

constexpr int kRun = 8;                 // positions of a thread
constexpr int kWarps = 8;               // computing warps, threads along time
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
  float2* composed;    // (B, segments, D): their (P, S)
};

// (P, S) of two channels
struct Affine {
  float2 P, S;
};
__device__ __forceinline__ Affine then(const Affine& a, const Affine& b) {  // b after a
  return Affine{__fmul2_rn(b.P, a.P), __ffma2_rn(b.P, a.S, b.S)};
}

// The product of a run as it is handed on: one too small for float32 stays above 0,
// as every f is, so that an infinite state passes it as it passes the single steps
// (0 times infinity would be NaN, and where runs end depends on the launch).  A
// finite state is off by less than 5e-7 at 3e38.
__device__ __forceinline__ float2 held_product(float2 P) {
  asm("max.NaN.f32 %0, %0, 0f00000001;" : "+f"(P.x));
  asm("max.NaN.f32 %0, %0, 0f00000001;" : "+f"(P.y));
  return P;
}

// What becomes of values whose chunk never came: NaN in every channel of the lane.
// Marked are the product of a run's first step, from which NaN reaches every later
// state (and the run's composition, so every later run), and in the backward also
// the gradient at the run's last position, from which it reaches every earlier one.
__device__ __forceinline__ void mark_lost(float2& v) { v = both(__uint_as_float(0x7fc00000u)); }

// Where a CTA works, and how its rows lie in shared memory.  Pair lane + 32 j
// is lane's j-th.  BULK: a lane's channels are neighbours, else 32 apart.
template <class T, int H, bool BULK>
struct Column {
  static constexpr int kPairs = 32 * H, kTile = 64 * H;
  static constexpr int kPitch = kTile * (int)sizeof(T) + (BULK ? 0 : 8);
  static constexpr int kBox = kPitch * kChunk;  // bytes of a chunk of one tensor
  static constexpr int kProducers = BULK ? 1 : 2;
  static constexpr int kThreads = 32 * (kWarps + kProducers);
  int64_t b, len, d0;
  int segment, lane, w;
  bool ok[2 * H];
  int64_t c0, c1;  // the segment's chunks
  int64_t v0, v1;  // those with valid positions: the state passes the others unchanged

  __device__ explicit Column(const ScanArgs<T>& a) {
    const int64_t id = blockIdx.x, tile = id % a.tiles, rest = id / a.tiles;
    segment = (int)(rest % a.segments);
    b = rest / a.segments;
    lane = threadIdx.x & 31;
    w = threadIdx.x >> 5;
    len = valid_length(a.lengths, b, a.T_);
    d0 = tile * kTile;
#pragma unroll
    for (int k = 0; k < 2 * H; ++k) ok[k] = channel(lane + 32 * (k >> 1), k & 1) < a.D;
    c0 = segment * a.per;
    c1 = min(c0 + a.per, a.chunks);
    const int64_t n = (len + kChunk - 1) / kChunk;
    v0 = a.reverse ? max(c0, a.chunks - n) : c0;
    v1 = a.reverse ? c1 : min(c1, n);
    if (v1 < v0) v1 = v0;
  }
  __device__ __forceinline__ int64_t channel(int pair, int half) const {
    return d0 + (BULK ? (pair & 31) * 2 * H + 2 * (pair >> 5) + half
                      : (pair & 31) + 64 * (pair >> 5) + 32 * half);
  }
  // first position of chunk c
  __device__ __forceinline__ int64_t chunk_time(const ScanArgs<T>& a, int64_t c) const {
    return (a.reverse ? a.chunks - 1 - c : c) * kChunk;
  }
  // a row of the chunk's tile: scan index i of this warp's run
  __device__ __forceinline__ int row(const ScanArgs<T>& a, int i) const {
    return a.reverse ? kChunk - 1 - (w * kRun + i) : w * kRun + i;
  }
  // whether 16-bit row r of s starts in the middle of a word
  __device__ __forceinline__ int shift(const Seq<const T>& s, int r) const {
    if (BULK || sizeof(T) == 4) return 0;
    return (int)(reinterpret_cast<uintptr_t>(s.row(b, r) + d0) >> 1 & 1);
  }
  __device__ __forceinline__ void load(const unsigned char* tile, int r, int shift,
                                       float2 (&v)[H]) const {
    if (BULK) {
      const Pack<Pack<T, 2>, H> q = *reinterpret_cast<const Pack<Pack<T, 2>, H>*>(
          tile + r * kPitch + lane * 2 * H * (int)sizeof(T));
#pragma unroll
      for (int j = 0; j < H; ++j) v[j] = to_f32x2(q.v[j]);
    } else {
      const T* p = reinterpret_cast<const T*>(tile + r * kPitch) + shift + lane;
#pragma unroll
      for (int j = 0; j < H; ++j) v[j] = make_float2(to_f32(p[64 * j]), to_f32(p[64 * j + 32]));
    }
  }
  // this lane's first channel of a row of an output
  __device__ __forceinline__ T* out(const Seq<T>& s, int64_t t) const {
    return s.row(b, t) + d0 + lane * (BULK ? 2 * H : 1);
  }
  __device__ __forceinline__ void store(T* p, const float2 (&v)[H]) const {
    if (BULK) {
      if (!ok[0]) return;
      Pack<Pack<T, 2>, H> q;
#pragma unroll
      for (int j = 0; j < H; ++j) q.v[j] = from_f32x2<T>(v[j]);
      *reinterpret_cast<Pack<Pack<T, 2>, H>*>(p) = q;
    } else {
#pragma unroll
      for (int j = 0; j < H; ++j) {
        const Pack<T, 2> q = from_f32x2<T>(v[j]);
        if (ok[2 * j]) p[64 * j] = q.v[0];
        if (ok[2 * j + 1]) p[64 * j + 32] = q.v[1];
      }
    }
  }
};

__device__ __forceinline__ void compute_barrier() {
  asm volatile("bar.sync 1, %0;" ::"n"(32 * kWarps) : "memory");
}
__device__ __forceinline__ unsigned char* align_ring(unsigned char* p) {
  return reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(p) + 127) &
                                          ~(uintptr_t)127);
}

// The ring of one CTA: N tensors a chunk.
template <class T, class C, int N, int STAGES>
struct Ring {
  static constexpr int kBytes = N * STAGES * C::kBox + 128;
  uint64_t *full, *empty;
  unsigned char* at;
  __device__ __forceinline__ unsigned char* tile(int slot, int k) const {
    return at + (slot * N + k) * C::kBox;
  }
  // what arrives on `full`: a bulk copy's bytes, or each copying thread and each of its warps
  static __device__ constexpr unsigned arrivals() {
    return C::kProducers == 1 ? 1 : 33 * C::kProducers;
  }
  __device__ void init() const {
    if (threadIdx.x == 0) {
      for (int s = 0; s < STAGES; ++s) {
        barrier_init(&full[s], arrivals());
        barrier_init(&empty[s], kWarps);
      }
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
  }
  __device__ __forceinline__ void release(int slot) const {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) barrier_arrive_here(&empty[slot]);
  }

  __device__ int64_t chunk_at(const C& at, bool descending, int it) const {
    return descending ? at.v1 - 1 - it : at.v0 + it;
  }
  __device__ void produce_bulk(const ScanArgs<T>& a, const C& col, const CUtensorMap* const (&maps)[N],
                               bool descending) const {
    if (col.lane) return;
    int it = 0;
    const int n = (int)(col.v1 - col.v0);
    for (; it < n; ++it) {
      const int slot = it % STAGES;
      if (it >= STAGES && !barrier_wait(&empty[slot], (unsigned)(it / STAGES - 1) & 1)) break;
      const int row = (int)col.chunk_time(a, chunk_at(col, descending, it));
      expect_bytes(&full[slot], N * C::kBox);
#pragma unroll
      for (int k = 0; k < N; ++k)
        fetch_tile(smem_addr(tile(slot, k)), maps[k], (int)col.d0, row, (int)col.b, &full[slot]);
    }
    // no copy may still be in flight when the CTA's memory is given up
    for (int k = it > STAGES ? it - STAGES : 0; k < it; ++k)
      barrier_wait(&full[k % STAGES], (unsigned)(k / STAGES) & 1);
  }
  __device__ void produce_words(const ScanArgs<T>& a, const C& col, const Seq<const T> (&src)[N],
                                bool descending) const {
    constexpr int kPer = 4 / (int)sizeof(T);           // elements of a word
    constexpr int kRows = kChunk / C::kProducers;      // rows of a warp
    static_assert(kRows == 32 || C::kProducers == 1, "a lane looks after a row's edges");
    const int n = (int)(col.v1 - col.v0), r0 = (col.w - kWarps) * kRows;
    const int width = (int)min((int64_t)C::kTile, a.D - col.d0);
    bool ok = true;
    for (int it = 0; it < n && ok; ++it) {
      const int slot = it % STAGES;
      if (it >= STAGES) {
        ok = __all_sync(~0u, barrier_wait(&empty[slot], (unsigned)(it / STAGES - 1) & 1));
        if (!ok) break;
      }
      const int64_t t0 = col.chunk_time(a, chunk_at(col, descending, it));
      const int rows = (int)min((int64_t)kRows, col.len - t0 - r0);  // with valid positions
      T head[N], tail[N];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        if (!src[k].p) continue;
        const T* p = src[k].row(col.b, t0 + r0) + col.d0;
        if (kPer == 2 && col.lane < rows) {
          const T* mine = p + col.lane * src[k].st;
          const int s = (int)(reinterpret_cast<uintptr_t>(mine) >> 1 & 1);
          if (s) head[k] = mine[0];
          if ((s + width) & 1) tail[k] = mine[width - 1];
        }
        unsigned dst = smem_addr(tile(slot, k)) + r0 * C::kPitch;
        for (int r = 0; r < rows; ++r) {
          const int s = kPer == 2 ? (int)(reinterpret_cast<uintptr_t>(p) >> 1 & 1) : 0;
#pragma unroll
          for (int j = 0; j < C::kTile / kPer; j += 32) {
            const int word = j + col.lane;
            if (word >= s && (word + 1) * kPer <= s + width)
              asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst + word * 4),
                           "l"(p - s + word * kPer)
                           : "memory");
          }
          p += src[k].st;
          dst += C::kPitch;
        }
      }
      if (kPer == 2 && col.lane < rows) {
#pragma unroll
        for (int k = 0; k < N; ++k) {
          if (!src[k].p) continue;
          const int r = r0 + col.lane;
          const T* mine = src[k].row(col.b, t0 + r) + col.d0;
          const int s = (int)(reinterpret_cast<uintptr_t>(mine) >> 1 & 1);
          T* row = reinterpret_cast<T*>(tile(slot, k) + r * C::kPitch);
          if (s) row[1] = head[k];
          if ((s + width) & 1) row[s + width - 1] = tail[k];
        }
      }
      asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(smem_addr(&full[slot]))
                   : "memory");
      __syncwarp();
      if (col.lane == 0) barrier_arrive_here(&full[slot]);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
};

// The state entering the segment, of the pair of channels that thread tid looks
// after: the segments before it, in order, after `first`.
template <class T, class C>
__device__ __forceinline__ float2 enter_segment(const ScanArgs<T>& a, const C& col,
                                                bool descending) {
  float v[2] = {0.f, 0.f};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t d = col.channel(threadIdx.x, h);
    if (d >= a.D) continue;
    float state = a.first ? a.first[col.b * a.D + d] : 0.f;
    const float2* p = a.composed + col.b * a.segments * a.D + d;
    const int n = descending ? a.segments - 1 - col.segment : col.segment;
#pragma unroll 8
    for (int k = 0; k < n; ++k) {
      const float2 q = p[(descending ? a.segments - 1 - k : k) * a.D];
      state = fmaf(q.x, state, q.y);
    }
    v[h] = state;
  }
  return make_float2(v[0], v[1]);
}
template <class T, class C>
__device__ __forceinline__ void put_composed(const ScanArgs<T>& a, const C& col, const Affine& own) {
  const float2 P = held_product(own.P);
  const float2 v[2] = {make_float2(P.x, own.S.x), make_float2(P.y, own.S.y)};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t d = col.channel(threadIdx.x, h);
    if (d < a.D) a.composed[(col.b * a.segments + col.segment) * a.D + d] = v[h];
  }
}
template <class T, class C>
__device__ __forceinline__ void put_last(const ScanArgs<T>& a, const C& col, float2 v) {
  const int64_t d = col.channel(threadIdx.x, 0), e = col.channel(threadIdx.x, 1);
  if (d < a.D) a.last[col.b * a.D + d] = v.x;
  if (e < a.D) a.last[col.b * a.D + e] = v.y;
}
// Zeros in every row of the segment's chunks without valid positions.
template <int H, class T, class C>
__device__ void clear_rest(const ScanArgs<T>& a, const C& col, const Seq<T>& out) {
  const int64_t rest = (col.c1 - col.c0) - (col.v1 - col.v0);
  const float2 zero[H] = {};
  for (int64_t k = 0; k < rest; ++k) {
    const int64_t t0 = col.chunk_time(a, a.reverse ? col.c0 + k : col.v1 + k);
#pragma unroll
    for (int i = 0; i < kRun; ++i)
      if (t0 + col.row(a, i) < a.T_) col.store(col.out(out, t0 + col.row(a, i)), zero);
  }
}

struct Masked { static constexpr bool value = true; };
struct Whole { static constexpr bool value = false; };

// The forward walk, or with COMPOSE its (P, S) alone.
template <class T, int H, bool BULK, int STAGES, bool COMPOSE>
__global__ void __launch_bounds__(Column<T, H, BULK>::kThreads, 2)
    forward_kernel(const ScanArgs<T> a, const __grid_constant__ CUtensorMap x_map,
                   const __grid_constant__ CUtensorMap g_map) {
  using C = Column<T, H, BULK>;
  constexpr int PAIRS = C::kPairs;
  constexpr int kParts = COMPOSE ? kWarps : kWarps - 1;  // the last warp's has no reader in a walk
  extern __shared__ unsigned char raw[];
  __shared__ uint64_t full[STAGES], empty[STAGES];
  __shared__ Affine part[2][kParts][PAIRS];
  __shared__ float2 enter[2][COMPOSE ? 1 : PAIRS];
  const C col(a);
  if (COMPOSE && col.segment == a.segments - 1) return;
  const Ring<T, C, 2, STAGES> ring{full, empty, align_ring(raw)};
  ring.init();
  const int tid = threadIdx.x;
  if (col.w >= kWarps) {
    if constexpr (BULK)
      ring.produce_bulk(a, col, {&x_map, &g_map}, false);
    else
      ring.produce_words(a, col, {a.x, a.g}, false);
    return;
  }
  Affine own{both(1.f), both(0.f)};
  if (!COMPOSE && tid < PAIRS) enter[0][tid] = enter_segment(a, col, false);
  bool ok = true;
  int turn = 0;
  const auto chunk = [&](int64_t c, auto kind) {
    constexpr bool kMasked = decltype(kind)::value;
    const int it = (int)(c - col.v0), slot = it % STAGES;
    const int64_t t0 = col.chunk_time(a, c);
    if (ok) ok = barrier_wait(&full[slot], (unsigned)(it / STAGES) & 1);
    const unsigned char *xt = ring.tile(slot, 0), *gt = ring.tile(slot, 1);
    Affine u[kRun][H];
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      float2 x[H], g[H];
      const int r = col.row(a, i);
      col.load(xt, r, col.shift(a.x, r), x);
      col.load(gt, r, col.shift(a.g, r), g);
#pragma unroll
      for (int j = 0; j < H; ++j) {
        float2 n;
        sigmoid_pair2<T, true>(g[j], u[i][j].P, n);
        u[i][j].S = __fmul2_rn(n, x[j]);
        if (kMasked && t0 + r >= col.len) u[i][j] = Affine{both(1.f), both(0.f)};
      }
    }
    ring.release(slot);
    if (!ok)
#pragma unroll
      for (int j = 0; j < H; ++j) mark_lost(u[0][j].P);
    if (COMPOSE || col.w < kParts)
#pragma unroll
      for (int j = 0; j < H; ++j) {
        Affine q = u[0][j];
#pragma unroll
        for (int i = 1; i < kRun; ++i) q = then(q, u[i][j]);
        q.P = held_product(q.P);
        part[turn][col.w][col.lane + 32 * j] = q;
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
    for (int j = 0; j < H; ++j) h[j] = enter[turn][col.lane + 32 * j];
    if (a.carry && col.w == 0) {
      float* p = a.carry + (col.b * a.chunks + c) * a.D;
#pragma unroll
      for (int j = 0; j < H; ++j) {
        if (col.ok[2 * j]) p[col.channel(col.lane + 32 * j, 0)] = h[j].x;
        if (col.ok[2 * j + 1]) p[col.channel(col.lane + 32 * j, 1)] = h[j].y;
      }
    }
    for (int w = 0; w < col.w; ++w)
#pragma unroll
      for (int j = 0; j < H; ++j) {
        const Affine q = part[turn][w][col.lane + 32 * j];
        h[j] = __ffma2_rn(q.P, h[j], q.S);
      }
    T* hp = col.out(a.h, t0 + col.row(a, 0));
    const int64_t step = a.reverse ? -a.h.st : a.h.st;
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const int64_t t = t0 + col.row(a, i);
      float2 out[H];
#pragma unroll
      for (int j = 0; j < H; ++j) {
        h[j] = __ffma2_rn(u[i][j].P, h[j], u[i][j].S);
        out[j] = kMasked && t >= col.len ? both(0.f) : h[j];
      }
      if (!kMasked || t < a.T_) col.store(hp, out);
      hp += step;
    }
    turn ^= 1;
    if (col.w == kWarps - 1)
#pragma unroll
      for (int j = 0; j < H; ++j) enter[turn][col.lane + 32 * j] = h[j];
  };
  for (int64_t c = col.v0; c < col.v1; ++c) {
    if (col.chunk_time(a, c) + kChunk <= col.len)
      chunk(c, Whole());
    else
      chunk(c, Masked());
  }
  if (COMPOSE) {
    if (tid < PAIRS) put_composed(a, col, own);
    return;
  }
  clear_rest<H>(a, col, a.h);
  if (!a.last || col.segment != a.segments - 1) return;
  compute_barrier();
  if (tid < PAIRS) put_last(a, col, enter[turn][tid]);
}

// mu's (P, S) of every segment but the first.
template <class T, bool BULK, int STAGES>
__global__ void __launch_bounds__(Column<T, 1, BULK>::kThreads, 2)
    backward_compose_kernel(const ScanArgs<T> a, const __grid_constant__ CUtensorMap d_map,
                            const __grid_constant__ CUtensorMap g_map) {
  using C = Column<T, 1, BULK>;
  constexpr int PAIRS = C::kPairs;
  extern __shared__ unsigned char raw[];
  __shared__ uint64_t full[STAGES], empty[STAGES];
  __shared__ Affine part[2][kWarps][PAIRS];
  const C col(a);
  if (col.segment == 0) return;
  const Ring<T, C, 2, STAGES> ring{full, empty, align_ring(raw)};
  ring.init();
  const int tid = threadIdx.x;
  if (col.w >= kWarps) {
    if constexpr (BULK)
      ring.produce_bulk(a, col, {&d_map, &g_map}, true);
    else
      ring.produce_words(a, col, {a.dh, a.g}, true);
    return;
  }
  Affine own{both(1.f), both(0.f)};
  bool ok = true;
  int turn = 0;
  const auto chunk = [&](int64_t c, auto kind) {
    constexpr bool kMasked = decltype(kind)::value;
    const int it = (int)(col.v1 - 1 - c), slot = it % STAGES;
    const int64_t t0 = col.chunk_time(a, c);
    if (ok) ok = barrier_wait(&full[slot], (unsigned)(it / STAGES) & 1);
    const unsigned char *dt = ring.tile(slot, 0), *gt = ring.tile(slot, 1);
    Affine q{both(1.f), both(0.f)};
    if (!ok) mark_lost(q.P);
#pragma unroll
    for (int i = kRun - 1; i >= 0; --i) {
      const int r = col.row(a, i);
      if (kMasked && t0 + r >= col.len) continue;
      float2 d[1] = {both(0.f)}, g[1], f, n;
      if (BULK || a.dh.p) col.load(dt, r, col.shift(a.dh, r), d);
      col.load(gt, r, col.shift(a.g, r), g);
      sigmoid_pair2<T, true>(g[0], f, n);
      q.P = __fmul2_rn(q.P, f);
      q.S = __fmul2_rn(f, __fadd2_rn(d[0], q.S));
    }
    ring.release(slot);
    q.P = held_product(q.P);
    part[turn][col.w][col.lane] = q;
    compute_barrier();
    if (tid < PAIRS)
#pragma unroll
      for (int w = kWarps - 1; w >= 0; --w) own = then(own, part[turn][w][tid]);
    turn ^= 1;
  };
  for (int64_t c = col.v1 - 1; c >= col.v0; --c) {
    if (col.chunk_time(a, c) + kChunk <= col.len)
      chunk(c, Whole());
    else
      chunk(c, Masked());
  }
  if (tid < PAIRS) put_composed(a, col, own);
}

// One pair of channels a lane: the factors and inputs of a run fill the registers.
template <class T, bool BULK, int STAGES>
__global__ void __launch_bounds__(Column<T, 1, BULK>::kThreads, 2)
    backward_kernel(const ScanArgs<T> a, const __grid_constant__ CUtensorMap x_map,
                    const __grid_constant__ CUtensorMap g_map,
                    const __grid_constant__ CUtensorMap d_map) {
  using C = Column<T, 1, BULK>;
  constexpr int PAIRS = C::kPairs;
  extern __shared__ unsigned char raw[];
  __shared__ uint64_t full[STAGES], empty[STAGES];
  __shared__ Affine part[2][kWarps][PAIRS];
  __shared__ float2 mpart[2][kWarps][PAIRS];
  __shared__ float2 enter[2][PAIRS];
  const C col(a);
  const Ring<T, C, 3, STAGES> ring{full, empty, align_ring(raw)};
  ring.init();
  const int tid = threadIdx.x;
  if (col.w >= kWarps) {
    if constexpr (BULK)
      ring.produce_bulk(a, col, {&x_map, &g_map, &d_map}, true);
    else
      ring.produce_words(a, col, {a.x, a.g, a.dh}, true);
    return;
  }
  if (tid < PAIRS) enter[0][tid] = enter_segment(a, col, true);
  bool ok = true;
  int turn = 0;
  const auto chunk = [&](int64_t c, auto kind) {
    constexpr bool kMasked = decltype(kind)::value;
    const int it = (int)(col.v1 - 1 - c), slot = it % STAGES;
    const int64_t t0 = col.chunk_time(a, c);
    const auto off = [&](int i) { return kMasked && t0 + col.row(a, i) >= col.len; };
    float2 h = both(0.f);
    {
      const float* p = a.carry + (col.b * a.chunks + c) * a.D;
      if (col.ok[0]) h.x = p[col.channel(col.lane, 0)];
      if (col.ok[1]) h.y = p[col.channel(col.lane, 1)];
    }
    if (ok) ok = barrier_wait(&full[slot], (unsigned)(it / STAGES) & 1);
    const unsigned char* xt = ring.tile(slot, 0);
    const unsigned char *gt = xt + C::kBox, *dt = gt + C::kBox;
    // the factors and inputs of the run; masked positions have f = 1 and zeros
    float2 f[kRun], n[kRun], x[kRun], d[kRun];
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      float2 g[1], xv[1], dv[1] = {both(0.f)};
      const int r = col.row(a, i);
      col.load(gt, r, col.shift(a.g, r), g);
      col.load(xt, r, col.shift(a.x, r), xv);
      if (BULK || a.dh.p) col.load(dt, r, col.shift(a.dh, r), dv);
      x[i] = xv[0], d[i] = dv[0];
      sigmoid_pair2<T, true>(g[0], f[i], n[i]);
      if (off(i)) f[i] = both(1.f), n[i] = x[i] = d[i] = both(0.f);
    }
    ring.release(slot);
    if (!ok) mark_lost(f[0]), mark_lost(d[kRun - 1]);
    {
      Affine q{f[0], __fmul2_rn(n[0], x[0])};
#pragma unroll
      for (int i = 1; i < kRun; ++i) q = then(q, Affine{f[i], __fmul2_rn(n[i], x[i])});
      float2 m = both(0.f);
#pragma unroll
      for (int i = kRun - 1; i >= 0; --i) m = __fmul2_rn(f[i], __fadd2_rn(d[i], m));
      q.P = held_product(q.P);
      part[turn][col.w][col.lane] = q;
      mpart[turn][col.w][col.lane] = m;
    }
    compute_barrier();
    float2 mu = enter[turn][col.lane];
    for (int w = 0; w < col.w; ++w) {
      const Affine q = part[turn][w][col.lane];
      h = __ffma2_rn(q.P, h, q.S);
    }
    for (int w = kWarps - 1; w > col.w; --w)
      mu = __ffma2_rn(part[turn][w][col.lane].P, mu, mpart[turn][w][col.lane]);
#pragma unroll
    for (int i = 0; i < kRun; ++i) {  // x becomes (1 - f) (h_{u-1} - x_u)
      const float2 before = h;
      h = __ffma2_rn(f[i], before, __fmul2_rn(n[i], x[i]));
      x[i] = __fmul2_rn(n[i], sub2(before, x[i]));
    }
    const int64_t end = t0 + col.row(a, kRun - 1);
    T* xp = col.out(a.dx, end);
    T* gp = col.out(a.dg, end);
    const int64_t dir = a.reverse ? -1 : 1;
#pragma unroll
    for (int i = kRun - 1; i >= 0; --i) {
      const float2 lam = __fadd2_rn(d[i], mu);
      mu = __fmul2_rn(f[i], lam);
      const float2 dx[1] = {off(i) ? both(0.f) : __fmul2_rn(lam, n[i])};
      const float2 dg[1] = {off(i) ? both(0.f) : __fmul2_rn(mu, x[i])};
      if (!kMasked || t0 + col.row(a, i) < a.T_) {
        col.store(xp, dx);
        col.store(gp, dg);
      }
      xp -= dir * a.dx.st;
      gp -= dir * a.dg.st;
    }
    turn ^= 1;
    if (col.w == 0) enter[turn][col.lane] = mu;
  };
  for (int64_t c = col.v1 - 1; c >= col.v0; --c) {
    if (col.chunk_time(a, c) + kChunk <= col.len)
      chunk(c, Whole());
    else
      chunk(c, Masked());
  }
  clear_rest<1>(a, col, a.dx);
  clear_rest<1>(a, col, a.dg);
  if (!a.last || col.segment != 0) return;
  compute_barrier();
  if (tid < PAIRS) put_last(a, col, enter[turn][tid]);
}

// One position of B streams: 1.8 us for 4 streams of 512 channels, 2.4 us for
// 512 of 1,024 (10.5 MB); what a caller waits for is the launch.
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

int64_t chunks_of(int64_t T) { return (T + kChunk - 1) / kChunk; }

// Chunks in the ring.  Two keep DRAM busy; a third and fourth, where two CTAs
// still fit an SM, were slower (backward at batch 64 x 10^4 x 512: 646, 686 and
// 748 us), since shared memory leaves that much less of the SM to L1.
constexpr int kStages = 2;

struct Cut {
  int tiles, segments;
  int64_t per;
};
// Segments: one, or as many as fill the SMs with one CTA or with two, whichever
// is the least by this measure: a CTA's chunks, 1.6 times as slow where two
// share an SM, and with segments `compose` times the walk on top (0.7 forward,
// 0.35 backward).  Measured on aligned 16-bit rows and used for all types and
// alignments, us for one / few / many segments:
// forward of 128 columns of 4000 positions 99 / - / 136, of 64 columns of
// 20000 495 / 406 / 315; backward of 64 columns of 40000 - / 733 / 524.
Cut cut_of(int64_t B, int64_t T, int64_t D, int tile, float compose) {
  Cut best{};
  const int64_t tiles = (D + tile - 1) / tile, columns = B * tiles, chunks = chunks_of(T);
  const int64_t sms = device_sm_count();
  float least = 0.f;
  for (const int64_t slots : {columns, sms, 2 * sms}) {
    const int64_t want = std::max<int64_t>(1, std::min(slots / std::max<int64_t>(1, columns), chunks));
    Cut c;
    c.tiles = (int)tiles;
    c.per = (chunks + want - 1) / want;
    c.segments = c.per ? (int)((chunks + c.per - 1) / c.per) : 1;
    const int64_t ctas = columns * c.segments;
    const float cost = (float)c.per * (c.segments > 1 ? 1.f + compose : 1.f) *
                       (ctas > sms ? 1.6f * (float)((ctas + 2 * sms - 1) / (2 * sms)) : 1.f);
    if (best.segments == 0 || cost < least) best = c, least = cost;
  }
  return best;
}
constexpr float kComposeForward = 0.7f, kComposeBackward = 0.35f;

template <class T>
ScanArgs<T> scan_args(const semicrf_recurrence* p, int tile, float compose, void* workspace) {
  const Cut c = cut_of(p->batch, p->T, p->D, tile, compose);
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

// Whether bulk copies can read s: 16-byte rows, no two of them overlapping.
bool bulk_readable(const semicrf_sequence& s, int64_t B, int64_t T, int64_t D, int elem) {
  return s.data && T < (1ll << 30) && B < (1ll << 30) && seq_aligned(s, B, T, elem, 16 / elem) &&
         (T == 1 || (s.time_stride >= D && s.time_stride < (1ll << 36))) &&
         (B == 1 || (s.batch_stride >= D && s.batch_stride < (1ll << 36)));
}

template <class T>
bool sequence_map(CUtensorMap* map, const semicrf_sequence& s, int64_t B, int64_t T_, int64_t D,
                  int tile) {
  const CUtensorMapDataType type = sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : std::is_same<T, __half>::value
                                       ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                       : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const cuuint64_t row = (cuuint64_t)((D * sizeof(T) + 15) / 16 * 16);  // where there is one row
  const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)T_, (cuuint64_t)B};
  const cuuint64_t strides[2] = {T_ == 1 ? row : (cuuint64_t)s.time_stride * sizeof(T),
                                 B == 1 ? row : (cuuint64_t)s.batch_stride * sizeof(T)};
  const cuuint32_t box[3] = {(cuuint32_t)tile, (cuuint32_t)kChunk, 1};
  return make_tensor_map(map, type, 3, s.data, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
}

template <class K>
bool allow_shared(K kernel, int bytes) {
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) ==
         cudaSuccess;
}

// The runtime's calls come before the maps: they give a thread that has none
// yet the device's context, which encoding a map needs.
template <class T, int H, bool BULK>
int launch_forward(const semicrf_recurrence* p, const ScanArgs<T>& a, cudaStream_t stream) {
  using C = Column<T, H, BULK>;
  constexpr int S = kStages;
  using R = Ring<T, C, 2, S>;
  const auto walk = forward_kernel<T, H, BULK, S, false>;
  const auto compose = forward_kernel<T, H, BULK, S, true>;
  CUtensorMap xm{}, gm{};
  if (!allow_shared(walk, R::kBytes) || !allow_shared(compose, R::kBytes) ||
      (BULK && (!sequence_map<T>(&xm, p->x, a.B, a.T_, a.D, C::kTile) ||
                !sequence_map<T>(&gm, p->gate, a.B, a.T_, a.D, C::kTile))))
    return SEMICRF_ERR_CUDA;
  const unsigned grid = (unsigned)(a.B * a.tiles * a.segments);
  if (a.segments > 1) compose<<<grid, C::kThreads, R::kBytes, stream>>>(a, xm, gm);
  walk<<<grid, C::kThreads, R::kBytes, stream>>>(a, xm, gm);
  return launch_status();
}

template <class T, bool BULK>
int launch_backward(const semicrf_recurrence* p, const semicrf_sequence& grad_h,
                    const ScanArgs<T>& a, cudaStream_t stream) {
  using C = Column<T, 1, BULK>;
  constexpr int S = kStages;
  using R = Ring<T, C, 3, S>;
  using RC = Ring<T, C, 2, S>;
  const auto walk = backward_kernel<T, BULK, S>;
  const auto compose = backward_compose_kernel<T, BULK, S>;
  CUtensorMap xm{}, gm{}, dm{};
  if (!allow_shared(walk, R::kBytes) || !allow_shared(compose, RC::kBytes) ||
      (BULK && (!sequence_map<T>(&xm, p->x, a.B, a.T_, a.D, C::kTile) ||
                !sequence_map<T>(&gm, p->gate, a.B, a.T_, a.D, C::kTile) ||
                !sequence_map<T>(&dm, grad_h, a.B, a.T_, a.D, C::kTile))))
    return SEMICRF_ERR_CUDA;
  const unsigned grid = (unsigned)(a.B * a.tiles * a.segments);
  if (a.segments > 1) compose<<<grid, C::kThreads, RC::kBytes, stream>>>(a, dm, gm);
  walk<<<grid, C::kThreads, R::kBytes, stream>>>(a, xm, gm, dm);
  return launch_status();
}

// Forward, a lane of 16-bit types takes two pairs of channels; one where D is
// at most 64, whose second would lie idle, and of float32, whose ring is twice
// the size.
template <class T>
int run_forward(const semicrf_recurrence* p, const semicrf_sequence& h, float* final_state,
                void* saved, void* workspace, cudaStream_t stream) {
  if (p->T == 0) return copy_state(p, p->initial_state, final_state, stream);
  const int H = sizeof(T) == 2 && p->D > 64 ? 2 : 1;
  ScanArgs<T> a = scan_args<T>(p, 64 * H, kComposeForward, workspace);
  a.h = as_seq<T>(h);
  a.first = p->initial_state;
  a.last = final_state;
  a.carry = static_cast<float*>(saved);
  bool bulk = p->D % (2 * H) == 0;
  for (const semicrf_sequence* s : {&p->x, &p->gate, &h})
    bulk = bulk && seq_aligned(*s, a.B, a.T_, sizeof(T), 2 * H);
  for (const semicrf_sequence* s : {&p->x, &p->gate})
    bulk = bulk && bulk_readable(*s, a.B, a.T_, a.D, sizeof(T));
  if constexpr (sizeof(T) == 2)
    if (H == 2)
      return bulk ? launch_forward<T, 2, true>(p, a, stream)
                  : launch_forward<T, 2, false>(p, a, stream);
  return bulk ? launch_forward<T, 1, true>(p, a, stream) : launch_forward<T, 1, false>(p, a, stream);
}

template <class T>
int run_backward(const semicrf_recurrence* p, const void* saved, const semicrf_sequence& grad_h,
                 const float* grad_state, const semicrf_sequence& grad_x,
                 const semicrf_sequence& grad_gate, float* grad_initial, void* workspace,
                 cudaStream_t stream) {
  if (p->T == 0) return copy_state(p, grad_state, grad_initial, stream);
  ScanArgs<T> a = scan_args<T>(p, 64, kComposeBackward, workspace);
  a.dh = as_seq<const T>(grad_h);
  a.dx = as_seq<T>(grad_x);
  a.dg = as_seq<T>(grad_gate);
  a.first = grad_state;
  a.last = grad_initial;
  a.carry = const_cast<float*>(static_cast<const float*>(saved));
  bool bulk = p->D % 2 == 0;
  for (const semicrf_sequence* s : {&p->x, &p->gate, &grad_h, &grad_x, &grad_gate})
    bulk = bulk && seq_aligned(*s, a.B, a.T_, sizeof(T), 2);
  for (const semicrf_sequence* s : {&p->x, &p->gate, &grad_h})
    bulk = bulk && bulk_readable(*s, a.B, a.T_, a.D, sizeof(T));
  return bulk ? launch_backward<T, true>(p, grad_h, a, stream)
              : launch_backward<T, false>(p, grad_h, a, stream);
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
  const int segments = std::max({cut_of(p->batch, p->T, p->D, 64, kComposeForward).segments,
                                 cut_of(p->batch, p->T, p->D, 128, kComposeForward).segments,
                                 cut_of(p->batch, p->T, p->D, 64, kComposeBackward).segments});
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
