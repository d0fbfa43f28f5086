// Paged attention for chunks of new tokens on the 5th-generation tensor cores
// (tcgen05, sm_100a).  kvc_attend.cuh has the mathematics and how work is
// shared out.
//
// Bound: the tensor cores (4 D flops per row and visible key) and, next to
// them, the SM's exponential unit: 128 keys x 128 rows are 16,384 exponentials
// at 16 a cycle, 1024 cycles, against 8 D cycles of tensor work (1024 at
// head_dim 128, half of that at 64).
//
// Roles of a CTA (one per SM: it holds all 512 TMEM columns):
//  * producer lane: queries of each tile and K/V blocks of 16 or 32 KB into a
//    ring of shared-memory slots, by TMA with the 128-byte swizzle;
//  * MMA lane: S = Q K^T with both operands in shared memory, O += P V with P
//    from tensor memory (it overwrites the S it came from) and V read from the
//    very tile that TMA wrote, as an N-major operand: nothing is transposed;
//  * two softmax warpgroups: a thread owns one row, so maximum and sum need no
//    exchange; S row from TMEM, masked, 2^(c s - c m), rounded to the cache's
//    type (the instruction wants A and B alike; off by half a step of the
//    weight at most, as the output's own rounding) and stored back as P.
// head_dim 64 and 128: a tile has two halves of 128 rows, one per warpgroup,
// that share every K/V block, and the MMA lane alternates between them, so one
// half's products run under the other's exponentials.  head_dim 256: O alone
// takes 256 columns, so a tile has 128 rows, S is double-buffered and each
// warpgroup takes 64 of a block's 128 keys (row maxima by shared memory).
//
// The running maximum is raised only when a block's exceeds it by 2^8: weights
// up to 256 lose nothing in fp32, bf16 or fp16, and the output in TMEM is
// rescaled in the first blocks of a row alone.
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
constexpr int kProducer = 8, kMma = 9;  // warps; two more fill the third warpgroup
// A softmax thread holds a row of S: registers of the third warpgroup go to the
// other two, 2 x 128 x 224 + 128 x 56 = 384 x 168, what the block is launched with.
constexpr int kSoftmaxRegs = 224, kOtherRegs = 56, kLaunchRegs = 168;
static_assert(2 * kSoftmaxRegs + kOtherRegs <= 3 * kLaunchRegs, "registers");
constexpr int KB = 128;                 // keys per unit
constexpr int kSpan = 64;               // elements of a 128-byte swizzle span
constexpr int kMeta = 16;
constexpr float kSlack = 8.f;           // log2 of the largest weight

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
  static constexpr int SC = NT == 2 ? KB : KB / 2;  // S columns of a softmax thread
  static constexpr int OC = NT == 2 ? D : D / 2;    // O columns of a softmax thread
  static constexpr int kBars = 2 * S + 11;
  static constexpr int kTail = kBars * 8 + kMeta * 4 + 16 + (NT == 1 ? 2048 : 0);
  static constexpr int kSmem = NT * kQ + S * kSlot + kTail;
  static_assert(S >= 4 && kSmem <= 227 * 1024 && kSmem > 116 * 1024, "one CTA per SM: it holds every TMEM column");
  static_assert(S * kSlot >= (kMaxAttendRequests + 41) * 4, "the prefix sums lie in the ring");
  // place of unit u's K and V among the 2 n blocks of a piece of n units, in the order of the MMA lane's use
  static __device__ __forceinline__ int kpos(int u) { return NT == 2 ? 2 * u : (u == 0 ? 0 : 2 * u - 1); }
  static __device__ __forceinline__ int vpos(int u, int n) {
    return NT == 2 ? 2 * u + 1 : (u == n - 1 ? 2 * n - 1 : 2 * u + 2);
  }
};

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

__device__ __forceinline__ void named_sync(int threads) {
  asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory");
}
__device__ __forceinline__ bool named_or(int threads, bool x) {
  uint32_t y;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 2, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(y)
      : "r"((uint32_t)x), "r"(threads)
      : "memory");
  return y != 0;
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
  constexpr int NT = G_::NT, S = G_::S, HV = G_::HV, SK = G_::SK;
  pdl_wait();
  pdl_trigger();
  extern __shared__ __align__(1024) uint8_t base[];
  const uint32_t q0 = smem_u32(base), ring0 = q0 + NT * G_::kQ;
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + NT * G_::kQ + S * G_::kSlot);
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * S;
  const uint32_t qfull = empty0 + 8 * S, qempty = qfull + 8;
  const uint32_t sfull = qempty + 8;   // [2] S is complete (per half, or per S buffer)
  const uint32_t pfull = sfull + 16;   // [2] P is in its place
  const uint32_t odone = pfull + 16;   // [2] P V is complete
  const uint32_t ofree = odone + 16;   // [2] the tile's output has been read
  const uint32_t done = ofree + 16;
  int* meta = reinterpret_cast<int*>(bars + G_::kBars);  // per unit: whether there is no block to read
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(meta + kMeta);
  float* xch = reinterpret_cast<float*>(tmem_slot + 4);  // [2][2][128] (NT == 1)
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if ((q0 & 1023u) != 0) {  // the swizzle goes by the address
    if (tid == 0) raise_flag(a.error_flag, KVC_DEV_TIMEOUT);
    if (tid == 0) a.record[blockIdx.x] = make_int4(0, 0, 0, 0);
    return;
  }
  if (tid == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, 1);
    }
    mbar_init(qfull, 1);
    mbar_init(qempty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(sfull + 8 * i, 1);
      mbar_init(pfull + 8 * i, NT == 2 ? 128 : 256);
      mbar_init(odone + 8 * i, 1);
      mbar_init(ofree + 8 * i, NT == 2 ? 128 : 256);
    }
    mbar_init(done, 1);
    mbar_init_fence();
  }
  if (warp == kMma) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  AttendLine line;
  AttendCursor c = attend_locate<KB, kThreads>(a, reinterpret_cast<int32_t*>(base + NT * G_::kQ), &line);
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the ring held the prefix sums
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // TMEM columns: S of the halves (or the two S buffers) at 0 and 128, O from 256 on
  constexpr uint32_t kO = 256;

  if (warp >= kProducer) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
  if (warp == kProducer) {
    // ---------------- producer ----------------
    if (lane == 0) {
      if (c.left == 0) a.record[blockIdx.x] = make_int4(0, 0, 0, 0);
      uint32_t it = 0, g = 0, pc = 0;  // slots, units, pieces
      bool ok = true;
      auto fill = [&](const CUtensorMap* map, int h, int blk) {  // a K or V block of the unit: HV slots
#pragma unroll
        for (int hv = 0; hv < HV; ++hv, ++it) {
          const int s = it % S;
          if (!mbar_wait(empty0 + 8 * s, ((it / S) & 1) ^ 1, a.error_flag)) return false;
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
      while (ok && c.left > 0) {
        const AttendTile t = attend_tile<KB>(a, c.r, c.i);
        const int n = (int)min64(t.units - c.u, c.left);
        const int halves = NT == 2 && t.ntok > a.sub ? 2 : 1;
        if (!mbar_wait(qempty, (pc & 1) ^ 1, a.error_flag)) break;
        mbar_expect_tx(qfull, halves * a.sub * a.G * D * 2);
        for (int s = 0; s < halves; ++s)
#pragma unroll
          for (int b = 0; b < D / kSpan; ++b)
            tma_3d(q0 + s * G_::kQ + b * 128 * 128, &a.qmap, b * kSpan, c.h * a.G, t.row0 + s * a.sub, qfull);
        ++pc;
        int prev = -1;
        for (int u = 0; ok && u < n; ++u, ++g) {
          const int blk = t.last() < 0 ? -1 : attend_block<KB>(a, t, t.block_of(c.u + u));
          meta[g % kMeta] = blk < 0;
          ok = fill(&a.kmap, c.h, blk);
          if constexpr (NT == 2) ok = ok && fill(&a.vmap, c.h, blk);
          else if (u > 0) ok = ok && fill(&a.vmap, c.h, prev);
          prev = blk;
        }
        if constexpr (NT == 1) ok = ok && fill(&a.vmap, c.h, prev);
        c.left -= n;
        if (c.left > 0) attend_advance(a, c);
      }
      // every copy has landed before the CTA may end
      for (uint32_t k = 0; k < (uint32_t)S && k < it; ++k) {
        const uint32_t j = it - 1 - k;
        if (!mbar_wait(full0 + 8 * (j % S), (j / S) & 1, a.error_flag)) break;
      }
      if (pc > 0) mbar_wait(qfull, (pc - 1) & 1, a.error_flag);
    }
    __syncwarp();
  } else if (warp == kMma) {
    // ---------------- MMA issuer ----------------
    if (lane == 0) {
      constexpr uint32_t id_s = idesc(FP16, SK, false), id_o = idesc(FP16, D, true);
      bool ok = true;
      auto wait = [&](uint32_t bar, uint32_t parity) {
        if (ok) ok = mbar_wait(bar, parity, a.error_flag);
        return ok;
      };
      // S[dst] = Q[half] K of the slots from sequence number `seq` on
      auto qk = [&](uint32_t dst, int half, uint32_t seq, bool skip, bool release) {
#pragma unroll 1
        for (int hv = 0; hv < HV; ++hv) {
          const uint32_t s = (seq + hv) % S;
          if (!wait(full0 + 8 * s, ((seq + hv) / S) & 1)) return;
          tc_fence_after();
          if (!skip) {
            const uint32_t kt = ring0 + s * G_::kSlot, qt = q0 + half * G_::kQ;
            const uint64_t qd = sw128_desc(qt), kd = sw128_desc(kt);  // start addresses count 16 bytes
#pragma unroll 2
            for (int k = 0; k < D / 16; ++k)
              mma_ss(dst + hv * SK, qd + (k >> 2) * (128 * 128 / 16) + (k & 3) * 2, kd + (k >> 2) * (G_::kBox / 16) + (k & 3) * 2,
                     id_s, k > 0 ? 1u : 0u);
          }
          if (release) tc_commit(empty0 + 8 * s);
        }
      };
      // O[dst] (+)= P[src] V
      auto pv = [&](uint32_t dst, uint32_t src, uint32_t seq, bool skip, bool acc, bool release) {
#pragma unroll 1
        for (int hv = 0; hv < HV; ++hv) {
          const uint32_t s = (seq + hv) % S;
          if (!wait(full0 + 8 * s, ((seq + hv) / S) & 1)) return;
          tc_fence_after();
          if (!skip) {
            const uint32_t vt = ring0 + s * G_::kSlot;
            const uint64_t vd = sw128_mn_desc(vt, G_::kBox);
#pragma unroll 2
            for (int k = 0; k < SK / 16; ++k)
              mma_ts(dst, src + hv * (SK / 2) + 8 * k, vd + k * (2048 / 16), id_o, acc || hv + k > 0 ? 1u : 0u);
          }
          if (release) tc_commit(empty0 + 8 * s);
        }
      };
      uint32_t g = 0, pc = 0;         // units and pieces issued
      uint32_t gb = 0, pcb = 0;       // those of the second half
      uint32_t seq0 = 0;              // slots before the piece
      int n = 0, halves = 1;
      auto next_piece = [&]() {       // sizes of the piece at the cursor
        const AttendTile t = attend_tile<KB>(a, c.r, c.i);
        n = (int)min64(t.units - c.u, c.left);
        halves = NT == 2 && t.ntok > a.sub ? 2 : 1;
        c.left -= n;
        if (c.left > 0) attend_advance(a, c);
      };
      bool have = c.left > 0;
      if (have) next_piece();
      while (ok && have) {
        // first unit of the piece
        if (!wait(qfull, pc & 1)) break;
        bool skip;
        {
          const uint32_t ks = seq0 + HV * G_::kpos(0);
          // meta is the producer's: read it behind the slot's barrier
          if (!wait(full0 + 8 * (ks % S), (ks / S) & 1)) break;
          skip = *(volatile int*)&meta[g % kMeta] != 0;
          qk(tmem + (NT == 1 ? (g & 1) * 128 : 0), 0, ks, skip, halves == 1);
          tc_commit(sfull + 8 * (NT == 1 ? (g & 1) : 0));
          if (halves == 2) {
            qk(tmem + 128, 1, ks, skip, true);
            tc_commit(sfull + 8);
          }
          if (n == 1) tc_commit(qempty);
        }
        bool acc = false;
        const int cn = n, ch = halves;
        for (int u = 0; ok && u < cn; ++u) {
          const uint32_t vs = seq0 + HV * G_::vpos(u, cn), ks = seq0 + HV * G_::kpos(u + 1);
          const bool more = u + 1 < cn;
          bool next_skip = false;
          if (more) {
            if (NT == 1) {  // the other S buffer, under this unit's softmax
              if (!wait(full0 + 8 * (ks % S), (ks / S) & 1)) break;
              next_skip = *(volatile int*)&meta[(g + 1) % kMeta] != 0;
              qk(tmem + ((g + 1) & 1) * 128, 0, ks, next_skip, true);
              tc_commit(sfull + 8 * ((g + 1) & 1));
              if (u + 2 == cn) tc_commit(qempty);
            }
          }
          if constexpr (NT == 1) {
            if (!wait(pfull + 8 * (g & 1), (g >> 1) & 1)) break;
            if (u == 0 && !wait(ofree, (pc & 1) ^ 1)) break;
            pv(tmem + kO, tmem + (g & 1) * 128, vs, skip, acc, true);
            tc_commit(odone);
          } else {
            if (!wait(pfull, g & 1)) break;
            if (u == 0 && !wait(ofree, (pc & 1) ^ 1)) break;
            pv(tmem + kO, tmem, vs, skip, acc, ch == 1);
            tc_commit(odone);
            if (more) {
              if (!wait(full0 + 8 * (ks % S), (ks / S) & 1)) break;
              next_skip = *(volatile int*)&meta[(g + 1) % kMeta] != 0;
              qk(tmem, 0, ks, next_skip, ch == 1);
              tc_commit(sfull);
            }
            if (ch == 2) {
              if (!wait(pfull + 8, gb & 1)) break;
              if (u == 0 && !wait(ofree + 8, (pcb & 1) ^ 1)) break;
              pv(tmem + kO + D, tmem + 128, vs, skip, acc, true);
              tc_commit(odone + 8);
              if (more) {
                qk(tmem + 128, 1, ks, next_skip, true);
                tc_commit(sfull + 8);
              }
              ++gb;
            }
            if (more && u + 2 == cn) tc_commit(qempty);
          }
          acc = acc || !skip;
          skip = next_skip;
          ++g;
        }
        seq0 += 2 * HV * cn;
        ++pc;
        if (ch == 2) ++pcb;
        have = c.left > 0;
        if (have) next_piece();
      }
      tc_commit(done);  // arrives once every MMA issued above has completed
      mbar_wait(done, 0, a.error_flag);
    }
    __syncwarp();
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    // ---------------- softmax ----------------
    constexpr int SC = G_::SC, OC = G_::OC;
    const int wg = warp >> 2;
    const int r = tid & 127;  // row of the half = TMEM lane
    const uint32_t lane_base = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
    const uint32_t ocol = lane_base + kO + wg * OC;
    const int tk = r / a.G;  // token of the half
    uint32_t g = 0, ga = 0, pc = 0;  // units of this half; units of the CTA; pieces of this half
    uint32_t seq0 = 0;
    bool dead = false;
    auto wait = [&](uint32_t bar, uint32_t parity) {  // voted warp-wide
      if (!dead) dead = !__all_sync(0xffffffffu, mbar_wait(bar, parity, a.error_flag));
    };
    while (c.left > 0) {
      const AttendTile t = attend_tile<KB>(a, c.r, c.i);
      const int n = (int)min64(t.units - c.u, c.left);
      const bool starts = c.u == 0, ends = c.u + n == t.units;
      const int halves = NT == 2 && t.ntok > a.sub ? 2 : 1;
      if (wg < halves || NT == 1) {
        const int half = NT == 2 ? wg : 0;
        const int token = half * a.sub + tk;
        const bool live = tk < a.sub && token < t.ntok;
        const int pos = live ? t.pos0 + token : -1;
        const int64_t part = 2 * (int64_t)blockIdx.x + (starts ? 1 : 0);
        float* mine = a.part_o + (part * a.rows + (int64_t)token * a.G + r - tk * a.G) * D + (NT == 1 ? wg * OC : 0);
        const int team = NT == 1 ? 256 : 128 * halves;  // threads that look at a V block together
        float m = -INFINITY, l = 0.f;
        bool any = false;     // a unit of the piece has been multiplied
        bool poison = false;  // `mine` holds infinite and NaN values to add to the output
        for (int u = 0; u < n; ++u, ++g, ++ga) {
          const int b = NT == 1 ? (int)(g & 1) : half;
          wait(sfull + 8 * b, NT == 1 ? (g >> 1) & 1 : g & 1);
          tc_fence_after();
          const bool skip = *(volatile int*)&meta[ga % kMeta] != 0;
          const uint32_t scol = lane_base + b * 128 + (NT == 1 ? wg * SC : 0);
          const int k0 = t.block_of(c.u + u) * KB;
          const bool whole = attend_whole<KB>(a, t, k0);
          if (!skip && !whole) {
            // A masked key weighs nothing whatever its value row holds, but 0 * inf
            // is not 0 in the product: infinite and NaN values leave the block
            // here and reach the rows that do see them by addition at the end.
            const uint32_t vs = seq0 + HV * G_::vpos(u, n);
#pragma unroll
            for (int hv = 0; hv < HV; ++hv) wait(full0 + 8 * ((vs + hv) % S), ((vs + hv) / S) & 1);
            bool odd = false;
            constexpr int kVec = KB * D / 8;
            auto vaddr = [&](int i) { return ring0 + ((vs + i / (SK * D / 8)) % S) * G_::kSlot + (i % (SK * D / 8)) * 16; };
            const int me = team == 256 ? tid : r;
            for (int i = me; i < kVec; i += team) {
              uint32_t w[4];
              lds128(vaddr(i), w);
              odd |= odd_pair<FP16>(w[0]) | odd_pair<FP16>(w[1]) | odd_pair<FP16>(w[2]) | odd_pair<FP16>(w[3]);
            }
            if (named_or(team, odd)) {
              const int d0 = NT == 1 ? wg * OC : 0;
              if (live && !poison) {
                for (int d = 0; d < OC; ++d) mine[d] = 0.f;
                poison = true;
              }
              for (int key = 0; key < KB; ++key) {
                if (!live || !attend_sees(a, pos, k0 + key)) continue;
                const int row = key % SK;
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
              named_sync(team);  // read by all before it is cleared
              for (int i = me; i < kVec; i += team) {
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
              named_sync(team);
            }
          }
          if (!skip) {
            uint32_t w[SC];
#pragma unroll
            for (int i = 0; i < SC; i += 32) tmem_ld32(scol + i, w + i);
            float* s = reinterpret_cast<float*>(w);
            if (!whole) {
              const int c0 = k0 + (NT == 1 ? wg * SC : 0);  // attend_sees, relative to the row's columns
              const int hi = pos - c0, lo = a.window > 0 ? hi - a.window : -1, first = a.sinks - c0;
#pragma unroll
              for (int i = 0; i < SC; ++i) s[i] = i <= hi && (i > lo || i < first) ? s[i] : -INFINITY;
            }
            float mx = s[0];
#pragma unroll
            for (int i = 1; i < SC; ++i) mx = fmaxf(mx, s[i]);
            if constexpr (NT == 1) {
              xch[((g & 1) * 2 + wg) * 128 + r] = mx;
              tc_fence_before();
              named_sync(256);  // and both halves of S are read: P may overwrite them
              tc_fence_after();
              mx = fmaxf(mx, xch[((g & 1) * 2 + (wg ^ 1)) * 128 + r]);
            }
            const bool raise = m > -INFINITY && mx * a.scale_log2 > m * a.scale_log2 + kSlack;
            if (__any_sync(0xffffffffu, raise)) {  // rescale the output and the sum
              const float f = raise ? exp2_approx((m - mx) * a.scale_log2) : 1.f;
              l *= f;
              if (raise) m = mx;
              wait(odone + (NT == 2 ? 8 * half : 0), (g & 1) ^ 1);  // the unit before this one
              tc_fence_after();
#pragma unroll
              for (int i = 0; i < OC; i += 32) {
                uint32_t o[32];
                tmem_ld32(ocol + i, o);
#pragma unroll
                for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                tmem_st32(ocol + i, o);
              }
            }
            if (m == -INFINITY) m = mx;  // nothing seen so far: l and the output row are 0
            const float ms = m == -INFINITY ? 0.f : m * a.scale_log2;
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < SC; i += 64) {
              uint32_t p[32];
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                const float e0 = exp2_approx(fmaf(s[i + 2 * j], a.scale_log2, -ms));
                const float e1 = exp2_approx(fmaf(s[i + 2 * j + 1], a.scale_log2, -ms));
                sum[(2 * j) & 3] += e0;
                sum[(2 * j + 1) & 3] += e1;
                p[j] = pack<FP16>(e0, e1);
              }
              // P over the S columns that it came from
              tmem_st32(lane_base + b * 128 + (NT == 1 ? wg * 32 : 0) + i / 2, p);
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            any = true;
            tc_wait_st();
          }
          tc_fence_before();
          mbar_arrive(pfull + 8 * b);
        }
        // ---- the piece's output ----
        if constexpr (NT == 1) {
          named_sync(256);
          xch[wg * 128 + r] = l;
          named_sync(256);
          l += xch[(wg ^ 1) * 128 + r];
          named_sync(256);
        }
        wait(odone + (NT == 2 ? 8 * half : 0), (g & 1) ^ 1);
        tc_fence_after();
        const int head = c.h * a.G + r - tk * a.G;
        const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees nothing answers 0
        uint16_t* dst = a.out + (int64_t)(t.row0 + token) * a.o_tok + (int64_t)head * a.o_head + (NT == 1 ? wg * OC : 0);
#pragma unroll
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
        tc_fence_before();
        mbar_arrive(ofree + (NT == 2 ? 8 * half : 0));
        ++pc;
      } else {
        ga += n;
      }
      seq0 += 2 * HV * n;
      c.left -= n;
      if (c.left == 0 && tid == 0) {
        int4 rec = make_int4(0, t.row0, t.ntok, c.h);
        if (starts && !ends) {  // later CTAs hold the rest of this tile
          const int64_t u1 = ((int64_t)blockIdx.x + 1) * line.total / line.used;
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
