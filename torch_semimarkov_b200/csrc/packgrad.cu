// packgrad.cu -- the gradient of a linear layer's weight from the 8-bit
// checkpoint of its input: out (M, D) = sum over positions n of dy[n, :]^T x[n, :].
//
// A matrix product over positions, on the tensor cores (tcgen05.mma,
// kind::f16, bfloat16 operands, float32 accumulators in tensor memory).  Both
// operands lie in memory with their channels contiguous, so both are
// MN-major; a position is one row of the shared-memory tile.
//
// x: a code times a power of two has 7 bits, so its bfloat16 value is exact,
// and its float16 value too where the checkpoint is of a float16 tensor.
// dy: bfloat16 as it is, and float16 as it is over a float16 checkpoint; else
// float16 and float32 are cut into 2 and 3 bfloat16 pieces of 8 bits each
// (exact: 11 and 24 bits), one product each.  So every product is exact and
// only the float32 sums round.
//
// Tiles: 256 x 256 outputs to a pair of CTAs (cta_group::2: a CTA brings 128
// channels of either operand, so each code is decoded for 256 outputs), or
// 128 x 128 to one CTA where M or D is at most 128 and for float32.  Each
// tile takes a run of positions; the runs' partial results are summed in
// order by a second kernel.
//
// Bound by the tensor cores with wide products, by decoding with narrow ones.
// Measured, 131,072 positions, M 1,536, D 512, the runs' sum (10 us) included,
// 16-bit types by bulk copies: 187 us, 1,160 TFLOP/s in the product, 0.7 of the
// library product's measured rate (the decoding warps' fences and the hand-over of
// a stage leave the tensor pipe idle for the rest).  Through registers (odd strides)
// bfloat16 351 us and float16, in two pieces, 433, over a bfloat16 checkpoint 600;
// float32 with M 768 630 us.
//
// The tensor cores truncate their float32 sums, always towards zero, so a long
// chain of them shrinks the result: values of one sign summed in one run of 131,072
// positions lost 6.3e-4, of 640,000 4.0e-3 (two pieces 6.0e-3).  No chain is longer
// than a segment: every kSums positions tensor memory is emptied into float32 sums
// that round to nearest.  For 16-bit dy those are the partial result itself, to which
// four warps of their own add one buffer of tensor memory while the next one fills.
// For float32 they are registers, the segments shorter and the leading piece summed
// apart from the others.  Errors then, at either length: 0.9e-6 for one piece, 5.2e-6
// for two, 2e-7 for float32 (random signs 0.5e-6, 2.1e-6, 3e-7).  Segments of 1,024
// positions would make them 0.4e-6 and 1.4e-6 and take 5% longer.

#include <algorithm>
#include <type_traits>

#include "encoder_internal.cuh"
#include "tma.cuh"

namespace semicrf {
int device_sm_count();  // api.cu

namespace {

constexpr int kTile = 128;      // channels of dy, and of x, that a CTA brings
constexpr int kStep = 64;       // positions of a stage
constexpr int kAtom = kStep * 128;  // bytes of 64 channels of a stage: 64 rows of 128
constexpr int kOperand = 2 * kAtom; // bytes of an operand of a stage
constexpr int kReaders = 16;    // 16-bit dy: warps that read the last segment's sums
constexpr int kAdders = 4;      // 16-bit dy: warps that add the others', one a quarter of the rows
constexpr int kGroupWarps = 4;  // warps that produce a stage together
constexpr int kSums = 2048;     // 16-bit dy: positions of a segment

template <class T>
struct Form;  // pieces of a value; positions of a stage; warps that produce, that read tensor
              // memory at the end of a segment or of all, and both; warps after those: one
              // issues, and the last kAdders add where others > 1
template <>
struct Form<__nv_bfloat16> {
  static constexpr int pieces = 1, step = 32, producers = 16, readers = 16, warps = 16;
  static constexpr int others = 4 + kAdders;
};
template <>
struct Form<__half> {
  static constexpr int pieces = 2, step = 32, producers = 16, readers = 16, warps = 16;
  static constexpr int others = 4 + kAdders;
};
template <>
struct Form<float> {
  static constexpr int pieces = 3, step = 32, producers = 8, readers = 8, warps = 16, others = 1;
};

// Registers a thread of the 16-bit forms: what the launch gives all of them, and
// what the producing and the other warpgroups make of it.  With the same for all,
// the rows on their way would spill (131,072 x 512 x 1,536 bfloat16: 495 us for
// 351).  What is taken has to be what is given, or the warps that take would wait.
constexpr int kLaunchRegs = 80, kProducerRegs = 96, kOtherRegs = 48;
static_assert(16 * kProducerRegs + 8 * kOtherRegs == 24 * kLaunchRegs, "of 16 and 8 warps");

template <class T>
struct Shape {
  static constexpr int kAtom = Form<T>::step * 128;
  static constexpr int kOperand = 2 * kAtom;
  static constexpr int kStage = (Form<T>::pieces + 1) * kOperand;
  static constexpr int kStages = 200 * 1024 / kStage < 8 ? 200 * 1024 / kStage : 8;
  static constexpr int kBytes = kStages * kStage + 1024;  // and room to align
};

struct GradArgs {
  int64_t N, M, Dp, G;  // positions, width of dy, code row bytes, scale row bytes
  int64_t run;          // positions of a tile, a multiple of kStep
  const void* dy;
  int64_t sb, st;
  bool vec;             // rows of dy start on 16-byte boundaries
  bool flat;            // position n of all sequences lies n * st from the first
  const int8_t* codes;
  const uint8_t* scales;
  const int64_t* lengths;
  unsigned T_;
  Divider by_t;
  int tiles_m, tiles_d;  // of 128 rows; of 128 CG columns
  float* partial;  // (runs, tiles_m, tiles_d, 128 CG, 128): a tile's columns one after another
};

__device__ __forceinline__ unsigned peer_addr(unsigned addr, unsigned rank) {
  unsigned r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
// Arrives on the barrier of the pair's first CTA (its own without a pair).
template <int CG>
__device__ __forceinline__ void barrier_arrive(uint64_t* b) {
  if (CG == 1)
    barrier_arrive_here(b);
  else
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(
                     peer_addr(smem_addr(b), 0))
                 : "memory");
}
// The barrier (of both CTAs of a pair) completes when the products issued so far have.
template <int CG>
__device__ __forceinline__ void commit_to(uint64_t* b) {
  if (CG == 1)
    asm volatile(
        "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
            smem_addr(b))
        : "memory");
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
        "[%0], %1;" ::"r"(smem_addr(b)),
        "h"((uint16_t)3)
        : "memory");
}
template <int CG, class T>
__device__ __forceinline__ void product(unsigned d, uint64_t a, uint64_t b, bool add) {
  // float32 accumulator, both operands of type T and MN-major, 128 CG x 128 CG
  constexpr unsigned type = std::is_same<T, __half>::value ? 0 : 1;
  constexpr unsigned kind = (1u << 4) | (type << 7) | (type << 10) | (1u << 15) | (1u << 16) |
                            ((unsigned)(kTile * CG >> 3) << 17) |
                            ((unsigned)(kTile * CG >> 4) << 24);
  if (CG == 1)
    asm volatile(
        "{.reg .pred p; setp.ne.u32 p, %4, 0;"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;}" ::"r"(d),
        "l"(a), "l"(b), "r"(kind), "r"((unsigned)add)
        : "memory");
  else
    asm volatile(
        "{.reg .pred p; setp.ne.u32 p, %4, 0;"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;}" ::"r"(d),
        "l"(a), "l"(b), "r"(kind), "r"((unsigned)add)
        : "memory");
}
template <int CG>
__device__ __forceinline__ void sync_all() {  // the CTA, or the pair
  if (CG == 1) {
    __syncthreads();
  } else {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
}
// 16 columns of this warp's 32 rows of tensor memory, one row a lane
__device__ __forceinline__ void read_columns(unsigned at, float (&f)[16]) {
  unsigned v[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(at));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int k = 0; k < 16; ++k) f[k] = __uint_as_float(v[k]);
}
// Adds N columns of this warp's rows of tensor memory to a tile of the partial
// result, a lane's row at `out` and its columns kTile apart; the first segment's
// are stored as they are.  The sums are formed in L2, by additions that no one
// waits for (640,000 x 512 x 1,536 bfloat16 927 us; read here and written back,
// 960).  One CTA adds to an address, a segment after the other, so the order is
// fixed.  These additions round to nearest and take subnormal numbers for zeros.
template <int N>
__device__ __forceinline__ void add_columns(unsigned at, float* out, bool first) {
  float v[16];
#pragma unroll 2
  for (int c = 0; c < N; c += 16) {
    float* p = out + (int64_t)c * kTile;
    read_columns(at + c, v);
#pragma unroll
    for (int k = 0; k < 16; ++k)
      if (first)
        __stcg(p + k * kTile, v[k]);
      else
        asm volatile("red.relaxed.gpu.global.add.f32 [%0], %1;" ::"l"(p + k * kTile), "f"(v[k])
                     : "memory");
  }
}
// This lane's row of a quarter of a tile's rows, column 0.
__device__ __forceinline__ float* partial_row(const GradArgs& a, int tm, int td, int cols,
                                              int quarter) {
  return a.partial +
         (((int64_t)blockIdx.y * a.tiles_m + tm) * a.tiles_d + td) * cols * kTile + quarter * 32 +
         (threadIdx.x & 31);
}
// Every segment's sums but the last one's, by one warp a quarter of the rows.
// A buffer is `ready` when its segment's products are done, and `taken` when
// all of these warps (of both CTAs) have read it, which the issuing thread
// waits for; so no wait is more than one phase ahead of its barrier.
template <int CG>
__device__ __forceinline__ void add_segments(const GradArgs& a, int tm, int td, unsigned tmem,
                                             int segments, uint64_t* ready, uint64_t* taken,
                                             int* lost) {
  constexpr int kCols = kTile * CG;
  const int quarter = (int)(threadIdx.x >> 5) & 3;
  float* const out = partial_row(a, tm, td, kCols, quarter);
  for (int g = 0; g + 1 < segments; ++g) {
    const int buffer = g & 1;
    if (!__all_sync(~0u, barrier_wait(&ready[buffer], (unsigned)(g / 2) & 1))) {
      *lost = 1;
      return;
    }
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    add_columns<kCols>(tmem + ((unsigned)(quarter * 32) << 16) + (unsigned)(buffer * kCols), out,
                       g == 0);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncwarp();
    if ((threadIdx.x & 31) == 0) barrier_arrive<CG>(&taken[buffer]);
  }
}
// The last segment's, by kReaders warps, after a barrier of the CTA.
template <int CG>
__device__ __forceinline__ void add_last_segment(const GradArgs& a, int tm, int td, unsigned tmem,
                                                 int segments, uint64_t* ready, bool lost) {
  constexpr int kCols = kTile * CG, kShare = kCols / (kReaders / 4);
  const int warp = threadIdx.x >> 5, quarter = warp & 3, c0 = (warp >> 2) * kShare;
  const int last = segments - 1, buffer = last & 1;
  float* const out = partial_row(a, tm, td, kCols, quarter) + (int64_t)c0 * kTile;
  const bool good = !lost && (!segments || __all_sync(~0u, barrier_wait(&ready[buffer],
                                                                        (unsigned)(last / 2) & 1)));
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (segments && good) {
    add_columns<kShare>(
        tmem + ((unsigned)(quarter * 32) << 16) + (unsigned)(buffer * kCols + c0), out, last == 0);
  } else {  // no positions: zeros; a wait that ran out shows as NaN
#pragma unroll 16
    for (int k = 0; k < kShare; ++k) out[k * kTile] = good ? 0.f : __uint_as_float(0x7fc00000u);
  }
}

// Shared-memory operand, MN-major, 128-byte swizzle: 64 channels are one row
// of 128 bytes, 8 positions 1024 bytes, the next 64 channels `atom` further.
__device__ __forceinline__ uint64_t operand(unsigned addr, int atom) {
  return (uint64_t)((addr & 0x3ffff) >> 4) | ((uint64_t)(atom >> 4) << 16) |
         ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// Eight values' pieces, two to a word: each the leading 8 bits of what is
// left, by truncation, so no piece overflows and the last leaves nothing.  An
// infinity has itself and zeros (what is left of it is NaN, whose larger
// partner 0 is taken); a NaN is made to show in the leading piece.
template <int NP, class T>
__device__ __forceinline__ void cut(const Pack<T, 8>& v, uint4 (&piece)[NP]) {
  if constexpr (NP == 1) {
    piece[0] = *reinterpret_cast<const uint4*>(&v);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      unsigned rest[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float f = to_f32(v.v[2 * k + h]);
        if (NP == 3) f += 0.f;  // any NaN to the one whose leading bits are set
        rest[h] = __float_as_uint(f);
      }
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const unsigned w = __byte_perm(rest[0], rest[1], 0x7632);
        (&piece[j].x)[k] = w;
        if (j + 1 < NP)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float f = __uint_as_float(rest[h]);
            const float left = fmaxf(fabsf(f - __uint_as_float(rest[h] & 0xffff0000u)), 0.f);
            rest[h] = __float_as_uint(left) | (rest[h] & 0x80000000u);
          }
      }
    }
  }
}

// dy of any type, stride and alignment, through registers.  Groups of four
// warps take the stages in turn.  A group publishes a stage, then requests the
// one it takes next, whose loads arrive while the other groups' stages are
// worked off.  (A fence before publishing waits for every load in flight, so a
// warp must not have any of its own then.)  A group waits for the products of
// the stage that used its slot before; products are done in order and there
// are no more groups than slots, so that wait is never more than one phase
// ahead of its barrier.
template <class T, int CG>
__global__ void __launch_bounds__(32 * (Form<T>::warps + Form<T>::others), 1)
    weight_grad_kernel(const GradArgs a) {
  using F = Form<T>;
  using S = Shape<T>;
  constexpr int NP = F::pieces, NS = S::kStages, STEP = F::step, W = F::warps;
  constexpr int kGroups = F::producers / kGroupWarps, kPart = 32 * kGroupWarps;
  constexpr int kPasses = STEP / 8;     // 16 threads a row, 8 rows at once
  constexpr bool kApart = NP == 3;      // float32: lower pieces apart, sums in registers
  constexpr int kSegment = (kApart ? 512 : kSums) / STEP;  // stages that tensor memory sums
  constexpr int kCols = kTile * CG;     // columns of the accumulator
  constexpr int kTmem = kApart ? 512 : 2 * kCols;
  static_assert(!kApart || CG == 1, "tensor memory holds two segments and the lower pieces");
  static_assert(kGroups <= NS, "see above");
  extern __shared__ unsigned char raw[];
  __shared__ uint64_t full[NS], empty[NS], ready[2], taken[2];
  __shared__ unsigned tmem_at;
  __shared__ int lost;
  unsigned char* ring = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = CG == 1 ? 0 : (int)(blockIdx.x % CG);
  const int pairs_m = a.tiles_m / CG, tile = (int)blockIdx.x / CG;
  const int tm = tile % pairs_m * CG + rank, td = tile / pairs_m;
  const int64_t first = blockIdx.y * a.run;
  const int64_t left = a.N - first;
  const int count = (int)(left < a.run ? (left < 0 ? 0 : left) : a.run);
  const int steps = (count + STEP - 1) / STEP;
  const int segments = (steps + kSegment - 1) / kSegment;

  if (tid == 0) {
    lost = 0;
    for (int s = 0; s < NS; ++s) {
      barrier_init(&full[s], kGroupWarps * CG);
      barrier_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      barrier_init(&ready[s], 1);
      barrier_init(&taken[s], kApart ? F::readers : kAdders * CG);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == W) {
    if (CG == 1) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                       smem_addr(&tmem_at)),
                   "n"(kTmem)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    } else {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                       smem_addr(&tmem_at)),
                   "n"(kTmem)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (CG > 1) sync_all<CG>();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const unsigned tmem = tmem_at;

  bool ok = true;
  if constexpr (!kApart) {
    static_assert(F::producers == 16 && W + F::others == 24, "see kLaunchRegs");
    if (warp < F::producers)
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kProducerRegs));
    else
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
  }
  if (warp < F::producers) {
    // this thread's 8 channels of dy and of x, and its first row of a stage
    const int group = tid / kPart, col = tid & 15, row0 = tid % kPart >> 4;
    const int64_t m = (int64_t)tm * kTile + col * 8;
    const int64_t d = ((int64_t)td * CG + rank) * kTile + col * 8;
    const bool has_m = m < a.M, has_d = d < a.Dp;
    const unsigned width = !has_m ? 0u : (unsigned)(a.M - m < 8 ? a.M - m : 8);
    // where its 16-byte piece of a row lies; later passes are 8 rows on
    const unsigned dst = (unsigned)(col >> 3) * S::kAtom + (unsigned)((col & 7) ^ row0) * 16 +
                         (unsigned)row0 * 128;
    const int64_t start = first + group * STEP + row0;
    const T* const dy0 = static_cast<const T*>(a.dy) + (has_m ? m : 0);
    const int8_t* const codes0 = a.codes + (has_d ? d : 0);
    const uint8_t* const scales0 = a.scales + (has_d ? d / kPackGroup : 0);
    // the row of pass 0 of the stage that is requested next: in the tensors
    // (dy where its positions are at one distance), and its sequence and position
    const T* dy = dy0 + start * a.st;
    const int8_t* codes = codes0 + start * a.Dp;
    const uint8_t* scales = scales0 + start * a.G;
    const bool placed = a.lengths || !a.flat;
    int64_t b = placed ? start / a.T_ : 0;
    unsigned t = (unsigned)(start - b * a.T_);
    // WIDE: every row holds whole 16-byte pieces.  Else values are loaded, and
    // held, one by one: packing them is work for when they have arrived.
    const auto produce = [&](auto kind) {
      constexpr bool kWide = decltype(kind)::value;
      struct Values {
        Pack<T, 8> whole;
        T single[8];
      } v[kPasses];
      uint2 q[kPasses];
      unsigned byte[kPasses];
      unsigned valid = 0;  // bit p: the row of pass p counts
      const auto request = [&](int it) {
        valid = 0;
#pragma unroll
        for (int p = 0; p < kPasses; ++p) {
          bool live = it * STEP + row0 + p * 8 < count;
          const T* src = dy + p * 8 * a.st;
          if (placed) {
            unsigned tt = t + p * 8;
            int64_t bb = b;
            if (tt >= a.T_) {
              const unsigned k = quotient(tt, a.by_t);
              bb += k;
              tt -= k * a.T_;
            }
            live = live && (!a.lengths || (int64_t)tt < a.lengths[bb]);
            if (!a.flat) src = dy0 + bb * a.sb + (int64_t)tt * a.st;
          }
          if (!live) continue;
          valid |= 1u << p;
          if (kWide) {
            constexpr int V = 16 / sizeof(T);
            if (has_m)
#pragma unroll
              for (int k = 0; k < 8; k += V)
                *reinterpret_cast<Pack<T, V>*>(&v[p].whole.v[k]) =
                    *reinterpret_cast<const Pack<T, V>*>(src + k);
          } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
              if (k < width) v[p].single[k] = src[k];
          }
          if (has_d) {
            q[p] = *reinterpret_cast<const uint2*>(codes + p * 8 * a.Dp);
            byte[p] = scales[p * 8 * a.G];
          }
        }
        dy += kGroups * STEP * a.st;
        codes += kGroups * STEP * a.Dp;
        scales += kGroups * STEP * a.G;
        t += kGroups * STEP;
        if (placed && t >= a.T_) {
          const unsigned k = quotient(t, a.by_t);
          b += k;
          t -= k * a.T_;
        }
      };
      if (group < steps) request(group);
      for (int it = group; it < steps; it += kGroups) {
        const int slot = it % NS;
        if (it >= NS) {
          ok = __all_sync(~0u, barrier_wait(&empty[slot], (unsigned)(it / NS - 1) & 1));
          if (!ok) break;
        }
        unsigned char* base = ring + slot * S::kStage + dst;
#pragma unroll
        for (int p = 0; p < kPasses; ++p) {
          unsigned char* at = base + p * 8 * 128;
          const bool live = valid >> p & 1;
          if (!kWide)
#pragma unroll
            for (int k = 0; k < 8; ++k)
              v[p].whole.v[k] = k < width ? v[p].single[k] : from_f32<T>(0.f);
          uint4 piece[NP];
          cut<NP>(v[p].whole, piece);
#pragma unroll
          for (int j = 0; j < NP; ++j)
            *reinterpret_cast<uint4*>(at + j * S::kOperand) =
                live && has_m ? piece[j] : make_uint4(0, 0, 0, 0);
          *reinterpret_cast<uint4*>(at + NP * S::kOperand) =
              live && has_d ? pack_decode(q[p], (uint8_t)byte[p]) : make_uint4(0, 0, 0, 0);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) barrier_arrive<CG>(&full[slot]);
        if (it + kGroups < steps) request(it + kGroups);
      }
    };
    if (a.vec && a.M % 8 == 0)
      produce(std::true_type());
    else
      produce(std::false_type());
  } else if (warp == W && lane == 0 && rank == 0) {
    int slot = 0;
    unsigned parity = 0;
    for (int segment = 0; segment < segments && ok; ++segment) {
      const int buffer = segment & 1, n = min(steps - segment * kSegment, kSegment);
      const unsigned sums = tmem + buffer * kCols;
      if (segment >= 2) ok = barrier_wait(&taken[buffer], (unsigned)(segment / 2 - 1) & 1);
      for (int i = 0; i < n; ++i) {
        ok = ok && barrier_wait(&full[slot], parity);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const unsigned at = smem_addr(ring + slot * S::kStage);
#pragma unroll
        for (int k = 0; k < STEP / 16; ++k) {
          const uint64_t bd = operand(at + NP * S::kOperand + k * 2048, S::kAtom);
#pragma unroll
          for (int j = 0; j < NP; ++j) {
            const uint64_t ad = operand(at + j * S::kOperand + k * 2048, S::kAtom);
            if (kApart && j)
              product<CG, __nv_bfloat16>(tmem + 2 * kCols, ad, bd,
                                         segment > 0 || i > 0 || k > 0 || j > 1);
            else
              product<CG, __nv_bfloat16>(sums, ad, bd, i > 0 || k > 0 || j > 0);
          }
        }
        commit_to<CG>(&empty[slot]);
        if (++slot == NS) slot = 0, parity ^= 1;
      }
      if (ok) commit_to<CG>(&ready[buffer]);
    }
  } else if (!kApart && warp >= W + F::others - kAdders) {
    add_segments<CG>(a, tm, td, tmem, segments, ready, taken, &lost);
  }
  __syncwarp();

  // Tensor memory to the partial result: a warp reads its 32 lanes (rows of
  // the tile) and a share of the columns; a column's rows are contiguous.
  if constexpr (!kApart) {
    static_assert(F::readers == kReaders, "the warps that read the last segment");
    __syncthreads();
    if (warp < kReaders) add_last_segment<CG>(a, tm, td, tmem, segments, ready, lost != 0);
  } else if (warp >= W - F::readers && warp < W) {
    constexpr int kShare = kCols / (F::readers / 4);
    static_assert(kShare % 16 == 0, "a warp reads 16 columns at once");
    const int quarter = warp & 3, c0 = (warp - (W - F::readers)) / 4 * kShare;
    const unsigned at = tmem + ((unsigned)(quarter * 32) << 16) + (unsigned)c0;
    float sum[kShare];
#pragma unroll
    for (int k = 0; k < kShare; ++k) sum[k] = 0.f;
    bool good = true;
    for (int g = 0; g < segments && good; ++g) {
      const int buffer = g & 1;
      good = __all_sync(~0u, barrier_wait(&ready[buffer], (unsigned)(g / 2) & 1));
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (!good) break;
#pragma unroll
      for (int c = 0; c < kShare; c += 16) {
        float v[16];
        read_columns(at + buffer * kCols + c, v);
#pragma unroll
        for (int k = 0; k < 16; ++k) sum[c + k] += v[k];
        if (g == segments - 1) {
          read_columns(at + 2 * kCols + c, v);
#pragma unroll
          for (int k = 0; k < 16; ++k) sum[c + k] += v[k];
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) barrier_arrive<1>(&taken[buffer]);
    }
    float* out = partial_row(a, tm, td, kCols, quarter) + (int64_t)c0 * kTile;
#pragma unroll
    for (int k = 0; k < kShare; ++k)  // a wait that ran out shows as NaN
      out[(int64_t)k * kTile] = good ? sum[k] : __uint_as_float(0x7fc00000u);
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (CG > 1) sync_all<CG>();
  if (warp == W) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (CG == 1)
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kTmem));
    else
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kTmem));
  }
}

// ---------------------------------------------------------------------------
// bfloat16 dy, or float16 with a checkpoint of float16 values (both operands
// float16 then: one product for the two of the pieces), whose positions are
// evenly spaced: the bulk-copy form.  One
// thread fetches codes and one dy (into the operand tile, swizzled) by TMA.
// The decoding warps read their scales from global memory right after they
// publish a stage, for the stage they take next, so that their fence before a
// stage is published never waits for a load.  A stage still takes a warp a
// few thousand cycles of waiting and decoding: five groups of four warps each
// take every fifth stage.  A group owns one slot of the operand ring.  It
// waits for the products of the slot's earlier stage first; those are done in
// order, so by then every stage that used its next code slot before has
// landed, and no wait is ever more than one phase ahead of its barrier.
// The issuing thread waits for one barrier a stage: another thread reports
// dy's arrival to it.
// ---------------------------------------------------------------------------
constexpr int kGroups = 5;                   // decoding groups and slots of the operand ring
constexpr int kDecoders = kGroups * kGroupWarps;
constexpr int kCodeSlots = 7;
constexpr int kCodes = kStep * kTile;        // bytes of a stage's codes
constexpr int kBulkBytes = kGroups * 2 * kOperand + kCodeSlots * kCodes + 1024;
constexpr int kBulkThreads = 32 * (kDecoders + 4 + kAdders);

template <class T, int CG>
__global__ void __launch_bounds__(kBulkThreads, 1)
    weight_grad_bulk_kernel(const GradArgs a, const __grid_constant__ CUtensorMap dy_map,
                            const __grid_constant__ CUtensorMap code_map) {
  constexpr int NS = kGroups, NC = kCodeSlots, kCols = kTile * CG, kTmem = 2 * kCols;
  constexpr int kSegment = kSums / kStep;  // stages that tensor memory sums
  extern __shared__ unsigned char raw[];
  __shared__ uint64_t code_landed[NC], code_free[NC], dy_landed[NS], full[NS], empty[NS];
  __shared__ uint64_t ready[2], taken[2];
  __shared__ unsigned tmem_at;
  __shared__ int lost;
  unsigned char* ring = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  unsigned char* code_ring = ring + NS * 2 * kOperand;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = CG == 1 ? 0 : (int)(blockIdx.x % CG);
  const int pairs_m = a.tiles_m / CG, tile = (int)blockIdx.x / CG;
  const int tm = tile % pairs_m * CG + rank, td = tile / pairs_m;
  const int64_t first = blockIdx.y * a.run;
  const int64_t left = a.N - first;
  const int count = (int)(left < a.run ? (left < 0 ? 0 : left) : a.run);
  const int steps = (count + kStep - 1) / kStep;
  const int segments = (steps + kSegment - 1) / kSegment;

  if (tid == 0) {
    lost = 0;
    for (int s = 0; s < NC; ++s) {
      barrier_init(&code_landed[s], 1);
      barrier_init(&code_free[s], kGroupWarps);
    }
    for (int s = 0; s < NS; ++s) {
      barrier_init(&dy_landed[s], 1);
      barrier_init(&full[s], (kGroupWarps + 1) * CG);  // each CTA's group, and its dy
      barrier_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      barrier_init(&ready[s], 1);
      barrier_init(&taken[s], kAdders * CG);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kDecoders) {
    if (CG == 1) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                       smem_addr(&tmem_at)),
                   "n"(kTmem)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    } else {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                       smem_addr(&tmem_at)),
                   "n"(kTmem)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (CG > 1) sync_all<CG>();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const unsigned tmem = tmem_at;

  bool ok = true;
  if (warp < kDecoders) {
    // rows row0, row0 + 8, ...; a warp's sixteen rows are 2 w, 2 w + 1, + 8, ...
    constexpr int kPart = 32 * kGroupWarps, kRows = kPart / 16, kPasses = kStep / kRows;
    static_assert(kRows == 8, "the swizzle and the lanes' rows repeat every 8 rows");
    const int part = tid % kPart, col = part & 15, row0 = part >> 4;
    const unsigned dst = (unsigned)(col >> 3) * kAtom + (unsigned)((col & 7) ^ row0) * 16 +
                         (unsigned)row0 * 128;
    const int slot = tid / kPart;
    unsigned char* base = ring + slot * 2 * kOperand + dst;
    // lane l < 16 brings the four scale bytes of row 2 w + l % 2 + 8 (l / 2)
    const int my_row = (row0 & ~1) + (lane & 1) + 8 * (lane >> 1 & 7);
    const int g0 = (td * CG + rank) * (kTile / kPackGroup);
    const bool whole =
        a.G % 4 == 0 && g0 + 4 <= a.G && reinterpret_cast<uintptr_t>(a.scales) % 4 == 0;
    const int64_t b0 = first / a.T_;
    const unsigned t0 = (unsigned)(first - b0 * a.T_);
    unsigned scale = 0;
    bool live = false;
    const auto request = [&](int it) {
      const int n = it * kStep + my_row;
      scale = 0;
      live = n < count;
      if (live && a.lengths) {
        const unsigned k = t0 + (unsigned)n, q = quotient(k, a.by_t);
        live = (int64_t)(k - q * a.T_) < a.lengths[b0 + q];
      }
      if (!live) return;
      const uint8_t* src = a.scales + (first + n) * a.G + g0;
      if (whole) {
        scale = *reinterpret_cast<const unsigned*>(src);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (g0 + k < a.G) scale |= (unsigned)src[k] << 8 * k;
      }
    };
    request(slot);
    for (int it = slot; it < steps; it += kGroups) {
      const int cs = it % NC;
      const unsigned use = (unsigned)(it / NS);
      if (use) ok = __all_sync(~0u, barrier_wait(&empty[slot], (use - 1) & 1));
      ok = ok && __all_sync(~0u, barrier_wait(&code_landed[cs], (unsigned)(it / NC) & 1));
      if (!ok) break;
      const unsigned char* codes = code_ring + cs * kCodes + row0 * kTile + col * 8;
      const unsigned on = __ballot_sync(~0u, live);
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        const uint2 q = *reinterpret_cast<const uint2*>(codes + p * kRows * kTile);
        const unsigned bytes = __shfl_sync(~0u, scale, (row0 & 1) + 2 * p);
        const uint8_t byte = (uint8_t)(bytes >> (col >> 2) * 8);
        *reinterpret_cast<uint4*>(base + kOperand + p * kRows * 128) =
            std::is_same<T, __half>::value ? pack_decode_half(q, byte) : pack_decode(q, byte);
      }
      __syncwarp();
      if (lane == 0) barrier_arrive<1>(&code_free[cs]);
      if ((on & 0xffffu) != 0xffffu) {  // clear the masked rows of dy
        ok = __all_sync(~0u, barrier_wait(&dy_landed[slot], use & 1));
        if (!ok) break;
#pragma unroll
        for (int p = 0; p < kPasses; ++p)
          if (!(on >> ((row0 & 1) + 2 * p) & 1))
            *reinterpret_cast<uint4*>(base + p * kRows * 128) = make_uint4(0, 0, 0, 0);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) barrier_arrive<CG>(&full[slot]);
      request(it + kGroups);
    }
  } else if (warp == kDecoders) {
    if (lane == 0 && rank == 0) {
      int slot = 0;
      unsigned parity = 0;
      for (int segment = 0; segment < segments && ok; ++segment) {
        const int buffer = segment & 1, n = min(steps - segment * kSegment, kSegment);
        const unsigned sums = tmem + buffer * kCols;
        if (segment >= 2) ok = barrier_wait(&taken[buffer], (unsigned)(segment / 2 - 1) & 1);
        for (int i = 0; i < n; ++i) {
          ok = ok && barrier_wait(&full[slot], parity);
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const unsigned at = smem_addr(ring + slot * 2 * kOperand);
          const uint64_t ad = operand(at, kAtom), bd = operand(at + kOperand, kAtom);
#pragma unroll
          for (int k = 0; k < kStep / 16; ++k)  // 16 positions are 2048 bytes
            product<CG, T>(sums, ad + k * (2048 >> 4), bd + k * (2048 >> 4), i > 0 || k > 0);
          commit_to<CG>(&empty[slot]);
          if (++slot == NS) slot = 0, parity ^= 1;
        }
        if (ok) commit_to<CG>(&ready[buffer]);
      }
    }
  } else if (warp == kDecoders + 1) {
    if (lane == 0) {
      const int m0 = tm * kTile;
      int it = 0;
      for (; it < steps; ++it) {
        const int slot = it % NS;
        if (it >= NS) {
          ok = barrier_wait(&empty[slot], (unsigned)(it / NS - 1) & 1);
          if (!ok) break;
        }
        const unsigned at = smem_addr(ring + slot * 2 * kOperand);
        const int n0 = (int)first + it * kStep;
        expect_bytes(&dy_landed[slot], kOperand);
        fetch_tile(at, &dy_map, m0, n0, &dy_landed[slot]);
        fetch_tile(at + kAtom, &dy_map, m0 + 64, n0, &dy_landed[slot]);
      }
      // no copy may still be in flight when the CTA's memory is given up
      for (int k = it > NS ? it - NS : 0; k < it; ++k)
        barrier_wait(&dy_landed[k % NS], (unsigned)(k / NS) & 1);
    }
  } else if (warp == kDecoders + 2) {
    if (lane == 0) {
      const int d0 = (td * CG + rank) * kTile;
      int it = 0;
      for (; it < steps; ++it) {
        const int cs = it % NC;
        if (it >= NC) {
          ok = barrier_wait(&code_free[cs], (unsigned)(it / NC - 1) & 1);
          if (!ok) break;
        }
        expect_bytes(&code_landed[cs], kCodes);
        fetch_tile(smem_addr(code_ring + cs * kCodes), &code_map, d0, (int)first + it * kStep,
                   &code_landed[cs]);
      }
      for (int k = it > NC ? it - NC : 0; k < it; ++k)
        barrier_wait(&code_landed[k % NC], (unsigned)(k / NC) & 1);
    }
  } else if (warp > kDecoders + 3) {
    add_segments<CG>(a, tm, td, tmem, segments, ready, taken, &lost);
  } else {
    if (lane == 0)
      for (int it = 0; it < steps; ++it) {
        const int slot = it % NS;
        ok = barrier_wait(&dy_landed[slot], (unsigned)(it / NS) & 1);
        if (!ok) break;
        barrier_arrive<CG>(&full[slot]);
      }
  }
  __syncwarp();

  __syncthreads();
  if (warp < kReaders) add_last_segment<CG>(a, tm, td, tmem, segments, ready, lost != 0);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (CG > 1) sync_all<CG>();
  if (warp == kDecoders) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (CG == 1)
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kTmem));
    else
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kTmem));
  }
}

// Sums the runs in order.  A block takes 32 x 32 outputs of a tile: reads
// along the tile's rows, writes along the output's.
template <class O>
__global__ void __launch_bounds__(256) sum_runs_kernel(int64_t D, int64_t M, int tiles_m, int64_t cols,
                                                       int runs, const float* __restrict__ partial,
                                                       O* __restrict__ out) {
  __shared__ float tile[32][33];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int64_t m0 = (int64_t)blockIdx.x * 32, d0 = (int64_t)blockIdx.y * 32;
  const int64_t size = (int64_t)tiles_m * cols * kTile;
  const float* src = partial + (m0 / kTile * cols + d0) * kTile + m0 % kTile + x;
#pragma unroll
  for (int k = 0; k < 32; k += 8) {
    float s = 0.f;
    for (int r = 0; r < runs; ++r) s += src[r * size + (int64_t)(y + k) * kTile];
    tile[y + k][x] = s;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 32; k += 8)
    if (m0 + y + k < M && d0 + x < D) out[(m0 + y + k) * D + d0 + x] = from_f32<O>(tile[x][y + k]);
}

struct Plan {
  int group, tiles_m, tiles_d, runs;  // CTAs of a tile; its tiles of 128 rows, 128 group columns
  int64_t run;
};

// Runs: as many as fill the SMs once, of four stages at least.
Plan plan(int64_t N, int64_t D, int64_t M, int dtype) {
  Plan p;
  p.group = dtype != SEMICRF_F32 && M > kTile && D > kTile ? 2 : 1;
  const int64_t edge = (int64_t)kTile * p.group;
  p.tiles_m = (int)((M + edge - 1) / edge) * p.group;
  p.tiles_d = (int)((D + edge - 1) / edge);
  const int64_t steps = (N + kStep - 1) / kStep;
  const int64_t ctas = (int64_t)p.tiles_m * p.tiles_d;
  int64_t runs = std::max<int64_t>(1, device_sm_count() / ctas);
  runs = std::max<int64_t>(1, std::min(runs, steps / 4));
  const int64_t per = std::max<int64_t>(1, (steps + runs - 1) / runs);
  p.run = per * kStep;
  p.runs = (int)std::max<int64_t>(1, (steps + per - 1) / per);
  return p;
}

template <class T, int CG>
int launch(const GradArgs& a, int runs, cudaStream_t stream) {
  const auto kernel = weight_grad_kernel<T, CG>;
  constexpr int bytes = Shape<T>::kBytes;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) !=
      cudaSuccess)
    return SEMICRF_ERR_CUDA;
  if (sizeof(T) == 2) {  // no launch with other registers than its warpgroups count on
    cudaFuncAttributes at{};
    if (cudaFuncGetAttributes(&at, kernel) != cudaSuccess || at.numRegs != kLaunchRegs)
      return SEMICRF_ERR_CUDA;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a.tiles_m * a.tiles_d), (unsigned)runs);
  cfg.blockDim = dim3(32 * (Form<T>::warps + Form<T>::others));
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = CG;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, a) == cudaSuccess ? SEMICRF_OK : SEMICRF_ERR_CUDA;
}

// (width, rows) bytes or 16-bit values, in boxes of one stage's positions
bool make_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, int64_t width,
              int64_t rows, int64_t row_bytes, int box, CUtensorMapSwizzle swizzle) {
  const cuuint64_t dims[2] = {(cuuint64_t)width, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)row_bytes};
  const cuuint32_t boxes[2] = {(cuuint32_t)box, (cuuint32_t)kStep};
  return make_tensor_map(map, type, 2, base, dims, strides, boxes, swizzle);
}

template <class T, int CG>
int launch_bulk(const GradArgs& a, int runs, cudaStream_t stream) {
  const auto kernel = weight_grad_bulk_kernel<T, CG>;
  CUtensorMap dy, codes;
  // the runtime's call comes first: it gives a thread that has none yet the
  // device's context, which encoding a map needs
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBulkBytes) !=
          cudaSuccess ||
      !make_map(&dy,
                std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                               : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                a.dy, a.M, a.N, a.st * 2, 64,
                CU_TENSOR_MAP_SWIZZLE_128B) ||
      !make_map(&codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.codes, a.Dp, a.N, a.Dp, kTile,
                CU_TENSOR_MAP_SWIZZLE_NONE))
    return SEMICRF_ERR_CUDA;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a.tiles_m * a.tiles_d), (unsigned)runs);
  cfg.blockDim = dim3(kBulkThreads);
  cfg.dynamicSmemBytes = kBulkBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = CG;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, a, dy, codes) == cudaSuccess ? SEMICRF_OK
                                                                       : SEMICRF_ERR_CUDA;
}

template <class T>
int launch_bulk_group(const GradArgs& a, const Plan& p, cudaStream_t stream) {
  return p.group == 2 ? launch_bulk<T, 2>(a, p.runs, stream) : launch_bulk<T, 1>(a, p.runs, stream);
}
template <class T>
int launch_group(const GradArgs& a, const Plan& p, cudaStream_t stream) {
  return p.group == 2 ? launch<T, 2>(a, p.runs, stream) : launch<T, 1>(a, p.runs, stream);
}

}  // namespace

size_t packed_weight_grad_workspace_bytes(int64_t B, int64_t T, int64_t D, int64_t M,
                                          int dtype) {
  const Plan p = plan(B * T, D, M, dtype);
  return sizeof(float) * p.runs * p.tiles_m * kTile * p.tiles_d * p.group * kTile;
}

int packed_weight_grad(int64_t B, int64_t T, int64_t D, int64_t M, int dtype, int packed_dtype,
                       const semicrf_sequence& dy, const int8_t* codes, const uint8_t* scales,
                       const int64_t* lengths, int out_dtype, void* out, void* workspace,
                       cudaStream_t stream) {
  const Plan p = plan(B * T, D, M, dtype);
  if (T >= (1 << 30) || p.run >= (1 << 30)) return SEMICRF_ERR_UNSUPPORTED;  // Divider's range
  GradArgs a{};
  a.N = B * T;
  a.M = M;
  a.G = pack_groups(D);
  a.Dp = a.G * kPackGroup;
  a.run = p.run;
  a.dy = dy.data;
  a.sb = dy.batch_stride;
  a.st = dy.time_stride;
  a.codes = codes;
  a.scales = scales;
  a.vec = seq_aligned(dy, B, T, dtype == SEMICRF_F32 ? 4 : 2, dtype == SEMICRF_F32 ? 4 : 8);
  a.flat = B == 1 || T == 1 || a.sb == T * a.st;
  a.lengths = lengths;
  a.T_ = (unsigned)std::max<int64_t>(T, 1);
  a.by_t = make_divider(a.T_);
  a.tiles_m = p.tiles_m;
  a.tiles_d = p.tiles_d;
  a.partial = static_cast<float*>(workspace);
  if (a.flat) a.st = T > 1 ? a.st : B > 1 ? a.sb : (M + 7) / 8 * 8;
  // bulk copies want aligned rows at one distance, and a row index in 31 bits
  const bool bulk = a.vec && a.N && a.N < (1ll << 31) - kStep &&
                    reinterpret_cast<uintptr_t>(codes) % 16 == 0 && a.flat && a.st >= M &&
                    a.st < (1ll << 36);
  int st;
  if (dtype == SEMICRF_F32)
    st = launch<float, 1>(a, p.runs, stream);
  else if (dtype == SEMICRF_BF16)
    st = bulk ? launch_bulk_group<__nv_bfloat16>(a, p, stream)
              : launch_group<__nv_bfloat16>(a, p, stream);
  else
    st = bulk && packed_dtype == SEMICRF_F16 ? launch_bulk_group<__half>(a, p, stream)
                                             : launch_group<__half>(a, p, stream);
  if (st != SEMICRF_OK) return st;
  const dim3 grid((unsigned)((M + 31) / 32), (unsigned)((D + 31) / 32));
  const int64_t cols = (int64_t)p.tiles_d * p.group * kTile;
  switch (out_dtype) {
    case SEMICRF_F32:
      sum_runs_kernel<<<grid, 256, 0, stream>>>(D, M, p.tiles_m, cols, p.runs, a.partial,
                                                static_cast<float*>(out));
      break;
    case SEMICRF_BF16:
      sum_runs_kernel<<<grid, 256, 0, stream>>>(D, M, p.tiles_m, cols, p.runs, a.partial,
                                                static_cast<__nv_bfloat16*>(out));
      break;
    default:
      sum_runs_kernel<<<grid, 256, 0, stream>>>(D, M, p.tiles_m, cols, p.runs, a.partial,
                                                static_cast<__half*>(out));
  }
  return launch_status();
}

}  // namespace semicrf
