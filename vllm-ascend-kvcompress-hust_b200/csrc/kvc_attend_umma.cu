// Paged attention for chunks of new tokens on the 5th-generation tensor cores
// (tcgen05, sm_100a).  kvc_attend.cuh has the mathematics and how work is
// shared out.
//
// Floor: the tensor cores (4 D flops per row and visible key) and the SM's
// exponential unit beside them (128 keys x 128 rows are 16,384 exponentials at
// 16 a cycle, 1024 cycles, against 8 D cycles of tensor work).  Bound: neither.
// 2048 new tokens over 16,384 at 40 / 8 heads of 128 take 1.2 million cycles in
// which both are busy half the time (51 %): S in 64-key parts reads 6 KB of shared
// memory for 32 cycles of products (48), the two halves' products and
// exponentials wait for each other, and a tile's start and end take 25,000
// cycles.  0.75 to 0.83 ms, 880 to 970 TFLOP/s, as calls follow each other and the
// 1000 W cap takes the clock to 1.45 to 1.65 GHz; a library product under that cap
// keeps 1,397 TFLOP/s, so the cap alone is not the bound, though changes that saved
// a tenth of the cycles (an eighth of the exponentials as polynomials on the FMA
// pipes) left the time as it was.  K and V are read through L2 once for each 256
// (128) rows: 3.3 GB for 118 MB here, 2.3 GB for 180 MB in 12 ragged requests at
// head_dim 256.
//
// Roles of a CTA (one per SM: it holds all 512 TMEM columns):
//  * producer lane: queries of each tile and K/V blocks of 16 or 32 KB into a
//    ring of shared-memory slots, by TMA with the 128-byte swizzle;
//  * two MMA lanes: S = Q K^T with both operands in shared memory, O += P V with
//    P from tensor memory and V read from the very tile that TMA wrote, as an
//    N-major operand: nothing is transposed;
//  * two softmax warpgroups: a thread owns one row, so maximum and sum need no
//    exchange; S row from TMEM, masked, 2^(c s - c m), rounded to the cache's
//    type (the instruction wants A and B alike) and stored back as P.
// head_dim 64 and 128: a tile has two halves of 128 rows, one per warpgroup and
// MMA lane, that share every K/V block.  S comes in parts of 64 keys with two
// buffers to a half (P goes over the S it came from): the next part's S is
// computed under this one's exponentials.  S of 128 keys at a time left no TMEM
// for that, and each product then waited for the exponentials before it (955 us
// for the above).  head_dim 256: O alone takes 256 columns, so a tile has 128
// rows, P lies beside S, and each warpgroup takes 64 of a block's 128 keys (row
// maxima by shared memory).
//
// The maximum that the weights are taken with is raised only when it has to be:
// when a part's own exceeds it by 2^8, which at head_dim 64 and 128 is looked at
// only when the sum of 64 weights passes 2^15, so that most parts need no pass
// over the scores for their maximum.  Weights above 1 lose nothing in fp32 or
// bf16, and the output in TMEM is rescaled in the first parts of a row alone.
//
// Rounding of P: half a step of the weight at most in bf16, whose range is
// fp32's, as the output's own rounding.  fp16 ends at 2^16 and loses bits below
// 2^-14, so a weight at the maximum is 2^3 there (2^7 at head_dim 256), and 2^9
// (2^10) once a block's weights have averaged less than 2^-10.  What rounding takes
// from weights that are below the range all the same is 2^-15 of the row's sum at
// most, and from then on 2^-34 of it a key; against a maximum of 1, keys under 2^-25
// vanished beside a sum that counts them, which many keys behind one strong first
// token feel.  Not 2^10 from the start: the running maximum then outgrew the type
// too often (178 us for 119 in a windowed 8,191-token prompt at head_dim 64).  The
// range costs that case 2 % (117 us without), and up to a sixth where scores are
// spread over tens of bits.
//
// Every wait is bounded (KVC_DEV_TIMEOUT); a softmax warp whose wait ran out
// goes on without waiting, so every named barrier is met, the other roles
// stop, and all meet at the last CTA barrier after copies and MMAs in flight
// have drained.
#include <algorithm>
#include <type_traits>

#include "kvc_attend.cuh"
#include "kvc_umma.cuh"

namespace kvc {
namespace {

constexpr int kThreads = 384;
constexpr int kProducer = 8, kMma = 9;  // warps (kMma and the one after it); one more fills the third warpgroup
// A softmax thread holds a row of S: registers of the third warpgroup go to the
// other two, 2 x 128 x 216 + 128 x 72 = 384 x 168, what the block is launched with.
constexpr int kSoftmaxRegs = 216, kOtherRegs = 72, kLaunchRegs = 168;
static_assert(2 * kSoftmaxRegs + kOtherRegs <= 3 * kLaunchRegs, "registers");
constexpr int KB = 128;                 // keys per unit
constexpr int kSpan = 64;               // elements of a 128-byte swizzle span
constexpr int kMeta = 16;

// log2 of the weights: at the maximum, at first and once others were small; of the largest that leave the maximum as
// it is.  kMost: the sum of 64 that does, at head_dim 64 and 128; 64 of 2^kTop have to be within it.
template <bool FP16, int NT>
struct Lift {
  static constexpr float kFirst = FP16 ? (NT == 2 ? 3.f : 7.f) : 0.f;
  static constexpr float kSmall = FP16 ? (NT == 2 ? 9.f : 10.f) : 0.f;
  static constexpr float kTop = FP16 ? (NT == 2 ? 9.f : 15.f) : 8.f;
  static constexpr float kMost = FP16 ? 49152.f : 32768.f;
};
constexpr float kMean = 1.f / 1024.f;  // weights are small where they average less

template <int D>
struct Geom {
  static constexpr int NT = D <= 128 ? 2 : 1;      // 128-row halves
  static constexpr int SK = D <= 128 ? 128 : 64;   // keys of a ring slot
  static constexpr int HV = KB / SK;               // slots of a K (or V) block
  static constexpr int kSlot = SK * D * 2;
  static constexpr int kBox = SK * 128;            // one 64-element span of a slot
  static constexpr int kQ = 128 * D * 2;           // queries of a half
  static constexpr int kFit = (225 * 1024 - NT * kQ) / kSlot;
  static constexpr int S = kFit > 10 ? 10 : kFit;
  static constexpr int OC = NT == 2 ? D : D / 2;   // O columns of a softmax thread
  // Room of a tile on the line beside its units: cycles of its start and end (first loads, output) over those
  // of a unit, 24,000 / 2,900, 25,000 / 3,900 and 7,000 / 3,400.  Against none: 12 ragged requests at 16 / 2 heads
  // of 256 295 -> 274 us, an 8,191-token windowed prompt at 16 / 8 of 64 122 -> 115 us; doubled, 278 and 117 (the
  // prompt is 119 now that fp16 weights are taken higher).
  static constexpr int kExtra = D == 256 ? 8 : D == 128 ? 6 : 2;
  // barriers, 8 bytes each: places in their array
  enum Bar : int { kFull = 0, kEmpty = S, kQFull = 2 * S, kQEmpty, kSFull, kPFull = kSFull + 4, kODone = kPFull + 4,
                   kSRead = kODone + 4, kOFree, kDone = kOFree + 2, kRead, kCleared, kBars };
  static constexpr int kTail = kBars * 8 + kMeta * 4 + 48 + (NT == 1 ? 2048 : 0);
  static constexpr int kSmem = NT * kQ + S * kSlot + kTail;
  static_assert(S >= 5 && kSmem <= 227 * 1024 && kSmem > 116 * 1024, "one CTA per SM: it holds every TMEM column");
  static_assert(S * kSlot >= (kMaxAttendRequests + 1 + kLocateInts) * 4, "the prefix sums lie in the ring");
  // TMEM columns.  Two halves: S of a half's 64-key parts, P over the S it came from.  One: S of 128 keys, P
  // of even and odd units.  O from 256 on.
  static __device__ __forceinline__ uint32_t s_col(int half, int part) { return 128 * half + 64 * part; }
  static __device__ __forceinline__ uint32_t p_col(int half, int part, uint32_t g) {
    return NT == 2 ? 128 * half + 64 * part : 128 + 64 * (g & 1) + 32 * part;
  }
  static __device__ __forceinline__ uint32_t o_col(int half) { return 256 + D * half; }
  // place of unit g's K and V among the 2 n blocks of the CTA's n units, as the MMA warps take them
  static __device__ __forceinline__ uint32_t k_at(uint32_t g) { return NT == 2 ? 2 * g : g == 0 ? 0 : 2 * g - 1; }
  static __device__ __forceinline__ uint32_t v_at(uint32_t g, uint32_t n) {
    return NT == 2 ? 2 * g + 1 : g + 1 == n ? 2 * n - 1 : 2 * g + 2;
  }
};

// what the producer says of a unit
constexpr uint32_t kSkip = 1, kFirst = 2, kLast = 4, kTwo = 8;  // no block to read; first, last of its piece; both halves have rows

// kind::f16, f32 accumulator, A K-major, B K-major or N-major, M = 128
constexpr uint32_t idesc(bool fp16, int n, bool b_mn) {
  return (1u << 4) | ((fp16 ? 0u : 1u) << 7) | ((fp16 ? 0u : 1u) << 10) | ((b_mn ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

__device__ __forceinline__ void tma_3d(uint32_t dst, const void* map, int c0, int c1, int c2, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_4d(uint32_t dst, const void* map, int c0, int c1, int c2, int c3, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
      : "memory");
}

// Named barriers.  With two halves a warpgroup may run ahead of the other by a tile, so each id has one set of
// threads that ever comes to it, and what both have to meet for are mbarriers, whose waits are bounded: both
// warpgroups (one half); each one's look at the values; a warpgroup by itself.
constexpr int kBarBoth = 1, kBarLook = 2, kBarOwn = 4;

__device__ __forceinline__ void named_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ bool named_or(int id, int threads, bool x) {
  uint32_t y;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, %3, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(y)
      : "r"((uint32_t)x), "r"(threads), "r"(id)
      : "memory");
  return y != 0;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
template <bool FP16>
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  uint32_t d;
  if constexpr (FP16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
template <bool FP16>
__device__ __forceinline__ bool odd_pair(uint32_t w) {  // an infinite or NaN value among the two
  constexpr uint32_t e = FP16 ? 0x7c00u : 0x7f80u;
  return (w & e) == e || ((w >> 16) & e) == e;
}

template <int D, bool FP16>
__global__ void __launch_bounds__(kThreads, 1) attend_umma_kernel(const __grid_constant__ AttendArgs a) {
  using G_ = Geom<D>;
  using E = std::conditional_t<FP16, Fp16, Bf16>;
  using Lift_ = Lift<FP16, G_::NT>;
  constexpr int NT = G_::NT, S = G_::S, HV = G_::HV, SK = G_::SK;
  pdl_wait();
  pdl_trigger();
  extern __shared__ __align__(1024) uint8_t base[];
  const uint32_t q0 = smem_u32(base), ring0 = q0 + NT * G_::kQ;
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + NT * G_::kQ + S * G_::kSlot);
  const uint32_t full0 = smem_u32(bars);
  const uint32_t empty0 = full0 + 8 * G_::kEmpty;
  const uint32_t qfull = full0 + 8 * G_::kQFull, qempty = full0 + 8 * G_::kQEmpty;
  const uint32_t sfull = full0 + 8 * G_::kSFull;  // [half][part] S is complete (one half: [0][0])
  const uint32_t pfull = full0 + 8 * G_::kPFull;  // [half][part] P is in its place
  const uint32_t odone = full0 + 8 * G_::kODone;  // [half][part], or [unit & 1] with one half: P V is complete
  const uint32_t sread = full0 + 8 * G_::kSRead;  // S has been read (one half)
  const uint32_t ofree = full0 + 8 * G_::kOFree;  // [half] the tile's output has been read
  const uint32_t done = full0 + 8 * G_::kDone;    // every product is complete
  const uint32_t vread = full0 + 8 * G_::kRead, vclear = full0 + 8 * G_::kCleared;  // a block's odd values (two halves)
  volatile uint32_t* meta = reinterpret_cast<uint32_t*>(bars + G_::kBars);  // per unit, from the producer
  uint32_t* tmem_slot = const_cast<uint32_t*>(meta + kMeta);
  uint32_t* odd_keys = tmem_slot + 4;  // [warpgroup][4] keys of a block that hold infinite or NaN values, a bit each
  float* xch = reinterpret_cast<float*>(tmem_slot + 12);  // [2][2][128] (NT == 1)
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if ((q0 & 1023u) != 0) {  // the swizzle goes by the address
    if (tid == 0) {
      raise_flag(a.error_flag, KVC_DEV_TIMEOUT);
      a.record[blockIdx.x] = make_int4(0, 0, 0, 0);
    }
    return;
  }
  if (tid == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, NT);  // MMA warps that read a slot
    }
    mbar_init(qfull, 1);
    mbar_init(qempty, NT);
    for (int i = 0; i < 4; ++i) {
      mbar_init(sfull + 8 * i, 1);
      mbar_init(pfull + 8 * i, 4);  // softmax warps arrive once each
      mbar_init(odone + 8 * i, 1);
    }
    mbar_init(sread, 8);
    for (int i = 0; i < 2; ++i) mbar_init(ofree + 8 * i, NT == 2 ? 4 : 8);
    mbar_init(done, 2);
    mbar_init(vread, 8);
    mbar_init(vclear, 8);
    for (int i = 0; i < 8; ++i) odd_keys[i] = 0;
    mbar_init_fence();
  }
  if (warp == kMma) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  AttendLine line;
  AttendCursor c = attend_locate<KB, kThreads, G_::kExtra>(a, reinterpret_cast<int32_t*>(base + NT * G_::kQ), &line);
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the ring held the prefix sums
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t units = (uint32_t)c.left;  // of this CTA

  if (warp >= kProducer) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == kProducer) {
      // ---------------- producer ----------------
      if (lane == 0) {
        if (units == 0) a.record[blockIdx.x] = make_int4(0, 0, 0, 0);
        uint32_t it = 0, g = 0, pc = 0;  // slots, units, pieces
        bool ok = true;
        auto fill = [&](const CUtensorMap* map, int h, int blk) {  // a K or V block: HV slots
#pragma unroll
          for (int hv = 0; hv < HV; ++hv, ++it) {
            const int s = it % S;
            if (!mbar_wait_short(empty0 + 8 * s, ((it / S) & 1) ^ 1, a.error_flag)) return false;
            if (blk < 0) {
              mbar_arrive(full0 + 8 * s);
              continue;
            }
            mbar_expect_tx(full0 + 8 * s, G_::kSlot);
#pragma unroll
            for (int b = 0; b < D / kSpan; ++b)
              tma_4d(ring0 + s * G_::kSlot + b * G_::kBox, map, b * kSpan, h, hv * SK, blk, full0 + 8 * s);
          }
          return true;
        };
        int prev_blk = -1, prev_h = 0;  // (one half) the unit whose V is still to come
        while (ok && c.left > 0) {
          const AttendTile t = attend_tile<KB>(a, c.r, c.i);
          const int n = (int)min64(t.units - c.u, c.left);
          const int halves = NT == 2 && t.ntok > a.sub ? 2 : 1;
          if (!mbar_wait_short(qempty, (pc & 1) ^ 1, a.error_flag)) break;
          mbar_expect_tx(qfull, halves * a.sub * a.G * D * 2);
          for (int s = 0; s < halves; ++s)
#pragma unroll
            for (int b = 0; b < D / kSpan; ++b)
              tma_3d(q0 + s * G_::kQ + b * 128 * 128, &a.qmap, b * kSpan, c.h * a.G, t.row0 + s * a.sub, qfull);
          ++pc;
          for (int u = 0; ok && u < n; ++u, ++g) {
            const int blk = t.last() < 0 ? -1 : attend_block<KB>(a, t, t.block_of(c.u + u));
            meta[g % kMeta] = (blk < 0 ? kSkip : 0) | (u == 0 ? kFirst : 0) | (u + 1 == n ? kLast : 0) |
                              (halves == 2 ? kTwo : 0);
            ok = fill(&a.kmap, c.h, blk);
            if constexpr (NT == 2) {
              ok = ok && fill(&a.vmap, c.h, blk);
            } else {
              if (g > 0) ok = ok && fill(&a.vmap, prev_h, prev_blk);
              prev_blk = blk;
              prev_h = c.h;
            }
          }
          c.left -= n;
          if (c.left > 0) attend_advance(a, c);
        }
        if constexpr (NT == 1) {
          if (ok && g > 0) fill(&a.vmap, prev_h, prev_blk);
        }
        // every copy has landed before the CTA may end
        for (uint32_t k = 0; k < (uint32_t)S && k < it; ++k) {
          const uint32_t j = it - 1 - k;
          if (!mbar_wait_short(full0 + 8 * (j % S), (j / S) & 1, a.error_flag)) break;
        }
        if (pc > 0) mbar_wait_short(qfull, (pc - 1) & 1, a.error_flag);
      }
      __syncwarp();
    } else if (warp <= kMma + 1) {
      // ---------------- MMA issuers: a lane each for the two halves, or for S and for O with one half ----------------
      // An issued product holds the lane until the tensor pipe takes it, and with one lane for everything the
      // pipe stood still through the waits of one half where the other's products were ready.  A wait that is
      // met takes the lane through some 20 dependent instructions, so slots and phases are carried along
      // instead of divided out.
      if (elect_one()) {
        constexpr uint32_t id_s = idesc(FP16, 64, false), id_o = idesc(FP16, D, true);
        const int role = warp - kMma;
        const int half = NT == 2 ? role : 0;
        bool ok = true;
        auto wait = [&](uint32_t bar, uint32_t parity) {
          if (ok) ok = mbar_wait_short(bar, parity, a.error_flag);
        };
        auto advance = [&](uint32_t& s, uint32_t& parity, uint32_t by) {  // a slot and its phase
          s += by;
          if (s >= S) {
            s -= S;
            parity ^= 1;
          }
        };
        const uint64_t qd = sw128_desc(q0 + half * G_::kQ), ring_k = sw128_desc(ring0),
                       ring_v = sw128_mn_desc(ring0, G_::kBox);  // start addresses count 16 bytes
        auto qk = [&](uint32_t d, uint64_t kd) {  // S of 64 keys
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            mma_ss(d, qd + (k >> 2) * (128 * 128 / 16) + (k & 3) * 2, kd + (k >> 2) * (G_::kBox / 16) + (k & 3) * 2,
                   id_s, k > 0 ? 1u : 0u);
        };
        auto pv = [&](uint32_t p, uint64_t vd, bool acc) {  // O (+)= P V of 64 keys
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_ts(tmem + G_::o_col(half), p + 8 * k, vd + k * (2048 / 16), id_o, acc || k > 0 ? 1u : 0u);
        };
        uint32_t pieces = 0, n_o = 0;  // whose queries, whose place for the output have been waited for
        bool acc = false;
        if constexpr (NT == 2) {
          // Parts of 64 keys: S of the next part runs under this one's softmax, in the buffer that the part
          // before this one has left.  Products of different shapes have no order among each other, so that
          // part's P V is waited for.
          const uint32_t s_bar = sfull + 16 * half, p_bar = pfull + 16 * half, o_bar = odone + 16 * half;
          uint32_t ks = 0, kp = 0, vs = 1, vp = 0;
          uint32_t f = 0, n = 0;  // flags of the unit; units of this half
          auto first_part = [&](uint32_t g, uint32_t n) {  // S of unit g's first 64 keys; the unit's flags
            wait(full0 + 8 * ks, kp);
            const uint32_t nf = meta[g % kMeta];
            if (nf & kFirst) wait(qfull, pieces++ & 1);
            if (half == 0 || (nf & kTwo)) {
              if (n > 0) wait(o_bar, (n - 1) & 1);
              tc_fence_after();
              if (ok && !(nf & kSkip)) qk(tmem + G_::s_col(half, 0), ring_k + ks * (G_::kSlot / 16));
              tc_commit(s_bar);
            }
            return nf;
          };
          if (units > 0) f = first_part(0, 0);
          for (uint32_t g = 0; ok && g < units; ++g) {
            const bool live = half == 0 || (f & kTwo);  // a tile without a second half: its blocks pass by
            const bool more = g + 1 < units;
            uint32_t nf = 0;
            if (live) {
              if (n > 0) wait(o_bar + 8, (n - 1) & 1);
              tc_fence_after();
              if (ok && !(f & kSkip)) qk(tmem + G_::s_col(half, 1), ring_k + ks * (G_::kSlot / 16) + 64 * 128 / 16);
              tc_commit(s_bar + 8);
            }
            tc_commit(empty0 + 8 * ks);
            if (f & kLast) tc_commit(qempty);
            advance(ks, kp, 2);
            if (live && (f & kFirst)) {
              wait(ofree + 8 * half, (n_o++ & 1) ^ 1);
              acc = false;
            }
            wait(full0 + 8 * vs, vp);
            if (live) {
              wait(p_bar, n & 1);
              tc_fence_after();
              if (ok && !(f & kSkip)) pv(tmem + G_::p_col(half, 0, g), ring_v + vs * (G_::kSlot / 16), acc);
              tc_commit(o_bar);
              acc = acc || !(f & kSkip);
            }
            // at a tile's end the next queries are still on their way: P V first
            if (more && !(f & kLast)) nf = first_part(g + 1, n + live);
            if (live) {
              wait(p_bar + 8, n & 1);
              tc_fence_after();
              if (ok && !(f & kSkip)) pv(tmem + G_::p_col(half, 1, g), ring_v + vs * (G_::kSlot / 16) + 64 * 128 / 16, acc);
              tc_commit(o_bar + 8);
            }
            tc_commit(empty0 + 8 * vs);
            advance(vs, vp, 2);
            if (more && (f & kLast)) nf = first_part(g + 1, n + live);
            n += live;
            f = nf;
          }
        } else if (role == 0) {
          uint32_t ks = 0, kp = 0;
          for (uint32_t g = 0; ok && g < units; ++g) {
            wait(full0 + 8 * ks, kp);
            const uint32_t f = meta[g % kMeta];
            if (f & kFirst) wait(qfull, pieces++ & 1);
            if (g > 0) wait(sread, (g - 1) & 1);
#pragma unroll 1
            for (int hv = 0; hv < 2; ++hv) {
              if (hv > 0) wait(full0 + 8 * ks, kp);
              tc_fence_after();
              if (ok && !(f & kSkip)) qk(tmem + G_::s_col(0, hv), ring_k + ks * (G_::kSlot / 16));
              tc_commit(empty0 + 8 * ks);
              advance(ks, kp, 1);
            }
            tc_commit(sfull);
            if (f & kLast) tc_commit(qempty);
            if (g > 0) advance(ks, kp, 2);  // V(g - 1) lies between K(g) and K(g + 1)
          }
        } else {
          uint32_t vs = 0, vp = 0;
          advance(vs, vp, units > 1 ? 4 : 2);  // K(0), K(1), V(0), K(2), V(1), ..
          for (uint32_t g = 0; ok && g < units; ++g) {
            // P first: either warpgroup may still be rescaling its columns of O.  What was in V's slots before
            // has arrived for certain only then, so that the barrier's phase means this V; and the unit's
            // flags have.
            wait(pfull, g & 1);
            wait(pfull + 8, g & 1);
            const uint32_t f = meta[g % kMeta];
            if (f & kFirst) {
              wait(ofree, (n_o++ & 1) ^ 1);
              acc = false;
            }
#pragma unroll 1
            for (int hv = 0; hv < 2; ++hv) {
              wait(full0 + 8 * vs, vp);
              tc_fence_after();
              if (ok && !(f & kSkip)) pv(tmem + G_::p_col(0, hv, g), ring_v + vs * (G_::kSlot / 16), acc || hv > 0);
              tc_commit(empty0 + 8 * vs);
              advance(vs, vp, 1);
            }
            tc_commit(odone + 8 * (g & 1));
            acc = acc || !(f & kSkip);
            if (g + 2 < units) advance(vs, vp, 2);  // K(g + 2) lies between V(g) and V(g + 1)
          }
        }
        tc_commit(done);  // arrives once every MMA issued above has completed
        mbar_wait_short(done, 0, a.error_flag);
      }
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    // ---------------- softmax ----------------
    constexpr int OC = G_::OC;
    const int wg = warp >> 2;
    const int half = NT == 2 ? wg : 0;
    const int r = tid & 127;  // row of the half = TMEM lane
    const uint32_t lane_base = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
    const uint32_t ocol = lane_base + G_::o_col(half) + (NT == 1 ? wg * OC : 0);
    const int tk = r / a.G;  // token of the half
    uint32_t g = 0, ga = 0;  // units of this half, and of the CTA
    uint32_t odd_blocks = 0;  // that both halves have cleared
    bool dead = false;
    auto wait = [&](uint32_t bar, uint32_t parity) {
      if (!dead) dead = !mbar_wait_short(bar, parity, a.error_flag);
      __syncwarp();  // the lanes may leave the wait apart, and what follows wants the warp as a whole
    };
    // The products so far, up to the part before (unit x, part) of this half, are in O.  A barrier tells two
    // phases apart; the one before the phase waited for has always been met: by the S that came after it (two
    // halves), or here, before P's place is written again (one).
    auto wait_o = [&](uint32_t x, int part) {
      if (NT == 1) wait(odone + 8 * ((x - 1) & 1), ((x - 1) >> 1) & 1);
      else if (part == 1) wait(odone + 16 * half, x & 1);
      else wait(odone + 16 * half + 8, (x - 1) & 1);
      tc_fence_after();
    };
    auto arrive = [&](uint32_t bar) {  // all lanes' TMEM accesses are ordered before it
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    while (c.left > 0) {
      const AttendTile t = attend_tile<KB>(a, c.r, c.i);
      const int n = (int)min64(t.units - c.u, c.left);
      const bool starts = c.u == 0, ends = c.u + n == t.units;
      const int halves = NT == 2 && t.ntok > a.sub ? 2 : 1;
      if (wg < halves || NT == 1) {
        const int token = half * a.sub + tk;
        const bool live = tk < a.sub && token < t.ntok;
        const int pos = live ? t.pos0 + token : -1;
        const int64_t part = 2 * (int64_t)blockIdx.x + (starts ? 1 : 0);
        float* mine = a.part_o + (part * a.rows + (int64_t)token * a.G + r - tk * a.G) * D + (NT == 1 ? wg * OC : 0);
        // positions of this half's rows
        const int pos_first = t.pos0 + half * a.sub, pos_last = min(t.last(), pos_first + a.sub - 1);
        float m = -INFINITY, l = 0.f;
        float base = -Lift_::kFirst;  // weights are 2^(c s - c m - base)
        bool any = false;     // a unit of the piece has been multiplied
        bool poison = false;  // `mine` holds infinite and NaN values to add to the output
        bool ready = false;   // every row of the warp has a maximum
        for (int u = 0; u < n; ++u, ++g, ++ga) {
          const int k0 = t.block_of(c.u + u) * KB;
          const bool whole = attend_whole(a, t.pos0, t.last(), k0, KB);  // for the tile
#pragma unroll 1
          for (int part = NT == 1 ? wg : 0; part < 2; part += NT == 1 ? 2 : 1) {  // 64 keys of the block
            wait(sfull + 16 * half + (NT == 2 ? 8 * part : 0), g & 1);
            tc_fence_after();
            const bool skip = (meta[ga % kMeta] & kSkip) != 0;
            const uint32_t scol = lane_base + G_::s_col(half, part), pcol = lane_base + G_::p_col(half, part, g);
            uint32_t w[64];  // the row's scores
            float* s = reinterpret_cast<float*>(w);
            tmem_ld32_async(scol, w);
            tmem_ld32_async(scol + 32, w + 32);
            if (!skip && !whole && (NT == 1 || part == 0)) {
              // A masked key weighs nothing whatever its value row holds, but 0 * inf
              // is not 0 in the product: infinite and NaN values leave the block
              // here and reach the rows that do see them by addition at the end.
              // Only the keys that hold some are gone through: NaN past every length
              // (pages that were never written) costs 12 chunks of 300 tokens 1 (head_dim
              // 128) to 9 % (256), where a walk through the block's keys took 2.5 and 4
              // times the whole call.  A key that rows do see costs each of them its dims.
              const uint32_t vs = HV * G_::v_at(ga, units);
              if (NT == 1 && g > 0) wait_o(g, 0);  // its V has been in the slots before this one's
#pragma unroll
              for (int hv = 0; hv < HV; ++hv) wait(full0 + 8 * ((vs + hv) % S), ((vs + hv) / S) & 1);
              bool odd = false;
              constexpr int kVec = KB * D / 8;
              auto vaddr = [&](int i) { return ring0 + ((vs + i / (SK * D / 8)) % S) * G_::kSlot + (i % (SK * D / 8)) * 16; };
              // Each warpgroup looks for itself (with one half they share the block), and nothing is cleared
              // before both have looked, so both find the same.
              constexpr int kLook = NT == 1 ? 256 : 128;
              for (int i = tid % kLook; i < kVec; i += kLook) {
                uint32_t w[4];
                lds128(vaddr(i), w);
                odd |= odd_pair<FP16>(w[0]) | odd_pair<FP16>(w[1]) | odd_pair<FP16>(w[2]) | odd_pair<FP16>(w[3]);
              }
              const int team = NT == 1 || halves == 2 ? 256 : 128;
              auto meet = [&](uint32_t bar) {  // the team's warps; two halves' by mbarrier
                if (NT == 1) {
                  named_sync(kBarBoth, 256);
                } else if (halves == 1) {
                  named_sync(kBarOwn, 128);
                } else {
                  __syncwarp();
                  if (lane == 0) mbar_arrive(bar);
                  wait(bar, odd_blocks & 1);
                }
              };
              if (named_or(kBarLook + (NT == 1 ? 0 : wg), kLook, odd)) {
                const int d0 = NT == 1 ? wg * OC : 0;
                uint32_t* keys = odd_keys + (NT == 1 ? 0 : 4 * wg);
                for (int i = tid % kLook; odd && i < kVec; i += kLook) {
                  uint32_t w[4];
                  lds128(vaddr(i), w);
                  const int key = i / (SK * D / 8) * SK + i % (SK * 8) / 8;  // rows of a box are 8 vectors
                  if (odd_pair<FP16>(w[0]) | odd_pair<FP16>(w[1]) | odd_pair<FP16>(w[2]) | odd_pair<FP16>(w[3]))
                    atomicOr(keys + key / 32, 1u << (key % 32));
                }
                named_sync(kBarLook + (NT == 1 ? 0 : wg), kLook);
                // the keys that hold some, where a row sees them (past a request's length none does)
                for (int k = 0; k < KB / 32; ++k)
                  for (uint32_t left = live ? *reinterpret_cast<volatile uint32_t*>(keys + k) : 0; left; left &= left - 1) {
                    const int key = 32 * k + __ffs(left) - 1, row = key % SK;
                    if (!attend_sees(a, pos, k0 + key)) continue;
                    if (!poison) {
                      for (int d = 0; d < OC; ++d) mine[d] = 0.f;
                      poison = true;
                    }
                    const uint32_t slot = ring0 + ((vs + key / SK) % S) * G_::kSlot;
                    for (int d = d0; d < d0 + OC; d += 2) {
                      uint32_t w;
                      asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w)
                                   : "r"(slot + (d / kSpan) * G_::kBox + row * 128 + ((((d % kSpan) / 8) ^ (row & 7)) << 4) +
                                         (d % 8) * 2)
                                   : "memory");
                      if (!odd_pair<FP16>(w)) continue;
                      const float2 v = unpack2(w, E{});
                      if (!isfinite(v.x)) mine[d - d0] += v.x;
                      if (!isfinite(v.y)) mine[d - d0 + 1] += v.y;
                    }
                  }
                meet(vread);  // read by all before it is cleared
                if (tid % kLook < KB / 32) keys[tid % kLook] = 0;
                for (int i = team == 256 ? tid : r; i < kVec; i += team) {
                  const uint32_t ad = vaddr(i);
                  uint32_t w[4];
                  lds128(ad, w);
#pragma unroll
                  for (int j = 0; j < 4; ++j)
                    if (odd_pair<FP16>(w[j])) {
                      const float2 v = unpack2(w[j], E{});
                      w[j] = (isfinite(v.x) ? w[j] & 0xffffu : 0u) | (isfinite(v.y) ? w[j] & 0xffff0000u : 0u);
                      asm volatile("st.shared.b32 [%0], %1;" ::"r"(ad + 4 * j), "r"(w[j]) : "memory");
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                meet(vclear);
                if (halves == 2) ++odd_blocks;
              }
            }
            tmem_ld_wait();
            tmem_ready32(w);
            tmem_ready32(w + 32);
            if (NT == 1) {
              arrive(sread);
              if (g > 1) wait_o(g - 1, 0);  // the unit before the last has left P's place
            }
            if (!skip) {
              // weights of the 64 keys, rounded into p; returns the sum of the unrounded ones
              uint32_t p[32];
              auto weigh = [&]() {
                const float ms = m == -INFINITY ? 0.f : FP16 ? fmaf(m, a.scale_log2, base) : m * a.scale_log2;
                const float2 c2 = make_float2(a.scale_log2, a.scale_log2), n2 = make_float2(-ms, -ms);
                float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                  const float2 x = __ffma2_rn(make_float2(s[2 * j], s[2 * j + 1]), c2, n2);
                  const float2 e = make_float2(exp2_approx(x.x), exp2_approx(x.y));
                  sum[j & 1] = __fadd2_rn(sum[j & 1], e);
                  p[j] = pack<FP16>(e.x, e.y);
                }
                sum[0] = __fadd2_rn(sum[0], sum[1]);
                return sum[0].x + sum[0].y;
              };
              auto largest = [&]() {
                float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int j = 4; j < 60; j += 8)
#pragma unroll
                  for (int k = 0; k < 4; ++k) top[k] = max3(top[k], s[j + k], s[j + 4 + k]);
#pragma unroll
                for (int k = 0; k < 4; ++k) top[k] = fmaxf(top[k], s[60 + k]);
                return max3(fmaxf(top[0], top[1]), top[2], top[3]);
              };
              // a new maximum: the row's sum and its output so far times f
              auto rescale = [&](float f) {
                l *= f;
                wait_o(g, NT == 1 ? 0 : part);
#pragma unroll 1
                for (int i = 0; i < OC; i += 32) {
                  uint32_t o[32];
                  tmem_ld32(ocol + i, o);
#pragma unroll
                  for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                  tmem_st32(ocol + i, o);
                }
              };
              float sum = 0.f;
              // The weights are taken with the maximum as it stands, and only a sum that is too large (or a row's
              // first keys) asks for the scores' own: no pass for the maximum in most blocks.
              bool fine = false;
              const bool seen = whole || attend_whole(a, pos_first, pos_last, k0 + 64 * part, 64);  // by this half's rows
              if (NT == 2 && seen && ready) {
                sum = weigh();
                fine = __all_sync(0xffffffffu,
                                  !live || (sum <= Lift_::kMost && (!FP16 || base != -Lift_::kFirst || sum >= 64.f * kMean)));
              }
              if (__builtin_expect(!fine, 0)) {
                if (!seen) {
                  const int c0 = k0 + 64 * part;  // attend_sees, relative to the row's columns
                  const int hi = pos - c0, lo = a.window > 0 ? hi - a.window : -1, first = a.sinks - c0;
#pragma unroll
                  for (int j = 0; j < 64; ++j) s[j] = j <= hi && (j > lo || j < first) ? s[j] : -INFINITY;
                }
                float mx = largest();
                if constexpr (NT == 1) {
                  xch[((g & 1) * 2 + wg) * 128 + r] = mx;
                  named_sync(kBarBoth, 256);
                  mx = fmaxf(mx, xch[((g & 1) * 2 + (wg ^ 1)) * 128 + r]);
                }
                const float top = (mx - m) * a.scale_log2 - base;  // log2 of the largest weight
                float f = 1.f;
                if (!(mx <= m) && m == -INFINITY) {
                  m = mx;
                } else if (FP16 ? top > Lift_::kTop : !(mx <= m) && !(top <= Lift_::kTop)) {
                  f = exp2_approx((m - mx) * a.scale_log2);
                  m = mx;
                } else if (FP16 && base == -Lift_::kFirst) {
                  // keys of the part (with one half, of the block) that the row sees
                  const int c0 = k0 + (NT == 2 ? 64 * part : 0), lo = a.window > 0 ? pos - c0 - a.window : -1;
                  const int hi = min(pos - c0, NT == 2 ? 63 : KB - 1);
                  const int n = max(0, hi - max(lo, -1)) + max(0, min(min(a.sinks - c0 - 1, lo), hi) + 1);
                  if (exp2_approx(top) < n * kMean) {
                    f = (float)(1 << (int)(Lift_::kSmall - Lift_::kFirst));
                    base = -Lift_::kSmall;
                  }
                }
                if (__any_sync(0xffffffffu, f != 1.f)) rescale(f);
                sum = weigh();
                // 64 of the largest weights and as much again for the rounding of large scores
                if (live && !(sum <= (FP16 ? 4194304.f : 32768.f))) sum = NAN;  // a score is infinite or NaN
                ready = __all_sync(0xffffffffu, !live || m > -INFINITY);
              }
              l += sum;
              any = true;
              tmem_st32(pcol, p);
              tc_wait_st();
            }
            arrive(pfull + 16 * half + 8 * part);
          }
        }
        // ---- the piece's output ----
        if constexpr (NT == 1) {
          named_sync(kBarBoth, 256);
          xch[wg * 128 + r] = l;
          named_sync(kBarBoth, 256);
          l += xch[(wg ^ 1) * 128 + r];
          named_sync(kBarBoth, 256);
        }
        wait_o(g, 0);
        const int head = c.h * a.G + r - tk * a.G;
        // A row that has seen nothing answers 0.  The sum tells: NaN scores leave no maximum, but a NaN sum.
        if (l == 0.f) any = false;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const float unit = FP16 ? __int_as_float((127 + (int)base) << 23) : 1.f;  // 2^base, for parts and lse
        l *= unit;
        uint16_t* dst = a.out + (int64_t)(t.row0 + token) * a.o_tok + (int64_t)head * a.o_head + (NT == 1 ? wg * OC : 0);
#pragma unroll 1
        for (int i = 0; i < OC; i += 32) {
          uint32_t o[32];
          tmem_ld32(ocol + i, o);
          if (!live) continue;
          float* x = reinterpret_cast<float*>(o);
#pragma unroll
          for (int j = 0; j < 32; ++j) x[j] = any ? x[j] : 0.f;
          if (starts && ends) {
#pragma unroll
            for (int j = 0; j < 32; ++j) x[j] *= inv;
            if (poison) {
#pragma unroll
              for (int j = 0; j < 32; ++j) x[j] += mine[i + j];
            }
#pragma unroll
            for (int j = 0; j < 32; j += 8)
              *reinterpret_cast<uint4*>(dst + i + j) =
                  make_uint4(pack<FP16>(x[j], x[j + 1]), pack<FP16>(x[j + 2], x[j + 3]), pack<FP16>(x[j + 4], x[j + 5]),
                             pack<FP16>(x[j + 6], x[j + 7]));
          } else {
            if constexpr (FP16) {
#pragma unroll
              for (int j = 0; j < 32; ++j) x[j] *= unit;
            }
            if (poison) {
#pragma unroll
              for (int j = 0; j < 32; ++j) x[j] += mine[i + j];
            }
#pragma unroll
            for (int j = 0; j < 32; j += 4)
              *reinterpret_cast<float4*>(mine + i + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
          }
        }
        if (live && (NT == 2 || wg == 0)) {
          if (!(starts && ends)) a.part_ml[part * a.rows + token * a.G + r - tk * a.G] = make_float2(m, l);
          else if (a.lse)
            a.lse[(int64_t)(t.row0 + token) * a.Hq + head] = l == 0.f ? -INFINITY : m * a.scale + logf(l);
        }
        arrive(ofree + 8 * half);
      } else {
        ga += n;
      }
      c.left -= n;
      if (c.left == 0 && tid == 0) {
        int4 rec = make_int4(0, t.row0, t.ntok, c.h);
        if (starts && !ends) {  // later CTAs hold the rest of this tile
          const int64_t u1 = attend_div(((int64_t)blockIdx.x + 1) * line.total, line.used);
          rec.x = (int)(attend_owner(line, u1 - 1 + (t.units - n)) - blockIdx.x);
        }
        a.record[blockIdx.x] = rec;
      }
      if (c.left > 0) attend_advance(a, c);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMma) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int D, bool FP16>
int launch_t(const AttendArgs& a, cudaStream_t st) {
  static bool configured[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return KVC_ECUDA;
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(attend_umma_kernel<D, FP16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             Geom<D>::kSmem) != cudaSuccess)
      return KVC_ECUDA;
    configured[dev] = true;
  }
  launch_dep(attend_umma_kernel<D, FP16>, dim3((unsigned)a.ctas), dim3(kThreads), (size_t)Geom<D>::kSmem, st, a);
  return launch_status();
}

}  // namespace

int attend_umma_rows(int D) { return D <= 128 ? 256 : 128; }
int attend_umma_slot_keys(int D) { return D <= 128 ? 128 : 64; }

int attend_umma_launch(const AttendArgs& a, bool fp16, cudaStream_t st) {
  if (a.D == 64) return fp16 ? launch_t<64, true>(a, st) : launch_t<64, false>(a, st);
  if (a.D == 128) return fp16 ? launch_t<128, true>(a, st) : launch_t<128, false>(a, st);
  return fp16 ? launch_t<256, true>(a, st) : launch_t<256, false>(a, st);
}

}  // namespace kvc
