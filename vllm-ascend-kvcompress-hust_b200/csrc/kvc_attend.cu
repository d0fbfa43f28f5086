// Paged attention for few rows per request: single tokens and short chunks
// (sm_100a).  kvc_attend.cuh has the mathematics and how work is shared out.
//
// Bound: HBM.  A decode step reads every K and V row of its requests once (4 D
// bytes per key and KV head) and does 4 G D flops on it, a flop a byte for each
// of the G query heads: two orders of magnitude under the tensor cores' rate.  So the tile is as small as the tensor instruction allows (16 rows:
// the heads of one KV head, for as many tokens as fit) and everything serves
// the stream: one persistent CTA per SM whose TMA producer keeps 128 to 192 KB of
// K/V blocks in flight, four consumer warps that split a block's keys, so no
// warp waits for another inside a tile, and a line of units cut evenly over the
// SMs, so a batch of unlike lengths ends everywhere at once.
//
// Measured on the device, call behind call: 16 decodes at 8k-52k keys, 16 / 2 heads
// of 256, 1.15 GB: 171 us, the copy rate (175 us); 32 at 4,608, 40 / 8 of 128, 0.61
// GB: 101 us, 0.92 of it; 4 decodes of 1k-6k: 12.5 us, 2 of them to find the CTA's
// piece, 2 to the first block, 3 to join the parts.
//
// A consumer warp holds the tile's queries, its running maximum, sum and
// output in registers: S = Q K^T by mma.sync (K by ldmatrix from the swizzled
// tile), the masked exponentials rounded to the cache's type as the A operand
// of O += P V (V by transposing ldmatrix), the sums taken from the unrounded
// exponentials.  P is rounded to the cache's 16 bits because the tensor
// instruction wants both operands alike.  In bf16, whose range is fp32's, each
// weight is off by half a step at most (2^-8 of it), independent from key to key,
// which is no more than the output's own rounding.  In fp16 the weights are taken
// 14 bits higher than against a maximum of 1 (lift_of): half a step (2^-11 of it)
// for weights down to 2^-28 of the row's largest, and 2^-39 of the largest for
// those below; against 1, weights under 2^-25 would vanish beside a sum that
// counts them, which many keys behind one strong first token feel.
// mma.sync rather than tcgen05: with 5 to 16 of 128 rows in use a 128-row
// instruction computes mostly padding, and the legacy path is far from being the
// bound.
#include <algorithm>
#include <type_traits>

#include "kvc_attend.cuh"

namespace kvc {
namespace {

constexpr int kRows = 16;
constexpr int kConsumers = 4;
constexpr int kThreads = (kConsumers + 1) * 32;
constexpr int kSpan = 64;  // elements of a 128-byte swizzle span
// Bits that the weights of a row with the (scaled) maximum ms are taken higher by, so that small ones stay in fp16's
// range; taken off where the warps' parts are joined.  2^14 is the type's highest power but one; past 2^22 the
// rounding of c m itself moves all weights of a row by a bit and more, and they keep that room.
template <bool FP16>
__device__ __forceinline__ float lift_of(float ms) {
  return FP16 && fabsf(ms) < 4194304.f ? 14.f : 0.f;
}
constexpr int kExtra = 2;  // units' time that a tile's start and end take (2,600 cycles, a unit 1,450)

template <int D>
struct Geom {
  static constexpr int KB = D <= 128 ? 128 : 64;   // keys per unit (rows_keys)
  static constexpr int kTile = KB * D * 2;         // bytes of a K (or V) block
  static constexpr int kStage = 2 * kTile;
  static constexpr int kPitch = D + 8;             // of a row in the merge buffers: 8 rows on different banks
  static constexpr int kMerge = kConsumers * kRows * kPitch * 4;
  static constexpr int kFit = (226 * 1024 - kMerge) / kStage;
  static constexpr int kStages = kFit > 6 ? 6 : kFit;
  static constexpr int kTail = kConsumers * kRows * 8 + kStages * (2 * 8 + 4);  // (m, l) of the warps, barriers, keys
  static constexpr int kKeys = KB / kConsumers;    // keys per warp and unit
  static constexpr int kSmem = kStages * kStage + kMerge + kTail;
  static_assert(kStages >= 2 && kSmem <= 227 * 1024, "shared memory");
  static_assert(kStages * kStage >= (kMaxAttendRequests + 1 + kLocateInts) * 4, "the prefix sums lie in the stages");
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

template <bool FP16>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t* a, uint32_t b0, uint32_t b1) {
  if constexpr (FP16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <bool FP16>
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  uint32_t d;
  if constexpr (FP16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}

__device__ __forceinline__ void tma_box(uint32_t dst, const void* map, int c0, int c1, int c2, int c3, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
      : "memory");
}

// Byte address of element (row, dim) of a KB-row tile of 64-element spans (128-byte swizzle).
template <int KB>
__device__ __forceinline__ uint32_t tile_addr(uint32_t tile, int row, int dim) {
  return tile + (dim / kSpan) * (KB * 128) + row * 128 + ((((dim % kSpan) / 8) ^ (row & 7)) << 4) + (dim % 8) * 2;
}

__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kConsumers * 32) : "memory"); }

// whether one of the two packed 16-bit values is infinite or NaN
template <bool FP16>
__device__ __forceinline__ bool odd_pair(uint32_t w) {
  constexpr uint32_t e = FP16 ? 0x7c00u : 0x7f80u;
  return (w & e) == e || ((w >> 16) & e) == e;
}

template <int D, bool FP16>
__global__ void __launch_bounds__(kThreads, 1) attend_rows_kernel(const __grid_constant__ AttendArgs a) {
  using G_ = Geom<D>;
  using E = std::conditional_t<FP16, Fp16, Bf16>;
  constexpr int KB = G_::KB, S = G_::kStages, NK = G_::kKeys;
  pdl_wait();
  pdl_trigger();
  extern __shared__ __align__(1024) uint8_t base[];
  float* merge_o = reinterpret_cast<float*>(base + S * G_::kStage);  // [warp][row][kPitch]
  auto merge_ml = reinterpret_cast<float2(*)[kRows]>(base + S * G_::kStage + G_::kMerge);  // [warp][row]
  uint64_t* bars = reinterpret_cast<uint64_t*>(merge_ml + kConsumers);
  volatile int* stage_key = reinterpret_cast<int*>(bars + 2 * S);  // first key of the stage's block, or -1: none to read
  const uint32_t stage0 = smem_u32(base), full0 = smem_u32(bars), empty0 = full0 + 8 * S;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if ((stage0 & 1023u) != 0) {  // the swizzle goes by the address
    if (tid == 0) {
      raise_flag(a.error_flag, KVC_DEV_TIMEOUT);
      a.record[blockIdx.x] = make_int4(0, 0, 0, 0);
    }
    return;
  }
  if (tid == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, kConsumers);
    }
    mbar_init_fence();
  }
  AttendLine line;
  AttendCursor c = attend_locate<KB, kThreads, kExtra>(a, reinterpret_cast<int32_t*>(base), &line);  // synchronises
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the stages held the prefix sums
  __syncthreads();
  const int64_t end = c.left;

  if (warp == kConsumers) {
    // ---------------- producer: one lane streams the blocks of every unit ----------------
    if (lane == 0) {
      if (end == 0) a.record[blockIdx.x] = make_int4(0, 0, 0, 0);
      uint32_t it = 0;
      bool ok = true;
      while (c.left > 0 && ok) {
        const AttendTile t = attend_tile<KB>(a, c.r, c.i);
        const int n = (int)min64(t.units - c.u, c.left);
        for (int u = c.u; u < c.u + n; ++u, ++it) {
          const int s = it % S;
          const int kb = t.block_of(u);
          const int blk = t.last() < 0 ? -1 : attend_block<KB>(a, t, kb);
          if (!mbar_wait(empty0 + 8 * s, ((it / S) & 1) ^ 1, a.error_flag)) {
            ok = false;
            break;
          }
          if (blk < 0) {
            stage_key[s] = -1;
            mbar_arrive(full0 + 8 * s);
            continue;
          }
          stage_key[s] = kb * KB;
          mbar_expect_tx(full0 + 8 * s, G_::kStage);
          const uint32_t st = stage0 + s * G_::kStage;
          const int in = (kb * KB) % kBlock;
#pragma unroll
          for (int b = 0; b < D / kSpan; ++b) tma_box(st + b * KB * 128, &a.kmap, b * kSpan, c.h, in, blk, full0 + 8 * s);
#pragma unroll
          for (int b = 0; b < D / kSpan; ++b)
            tma_box(st + G_::kTile + b * KB * 128, &a.vmap, b * kSpan, c.h, in, blk, full0 + 8 * s);
        }
        c.left -= n;
        if (c.left > 0) attend_advance(a, c);
      }
      // every copy has landed before the CTA may end
      for (uint32_t k = 0; k < (uint32_t)S && k < it; ++k) {
        const uint32_t j = it - 1 - k;
        if (!mbar_wait(full0 + 8 * (j % S), (j / S) & 1, a.error_flag)) break;
      }
    }
    return;
  }

  // ---------------- consumers ----------------
  uint32_t it = 0;
  bool dead = false;  // a wait ran out: go through the motions without waiting, so every barrier is met
  while (c.left > 0) {
    const AttendTile t = attend_tile<KB>(a, c.r, c.i);
    const int n = (int)min64(t.units - c.u, c.left);
    const int rows = t.ntok * a.G;
    // queries: A fragments, rows lane / 4 and lane / 4 + 8
    uint32_t qf[D / 16][4];
    int pos[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int row = lane / 4 + 8 * j, tk = row / a.G;
      const bool live = row < rows;
      pos[j] = live ? t.pos0 + tk : -1;
      const uint16_t* src = a.q + (int64_t)(t.row0 + tk) * a.q_tok + (int64_t)(c.h * a.G + row - tk * a.G) * a.q_head +
                            2 * (lane & 3);
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        qf[k][j] = live ? __ldg(reinterpret_cast<const uint32_t*>(src + 16 * k)) : 0u;
        qf[k][j + 2] = live ? __ldg(reinterpret_cast<const uint32_t*>(src + 16 * k + 8)) : 0u;
      }
    }
    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    for (int u = 0; u < n; ++u, ++it) {
      const int s = it % S;
      // waits are voted warp-wide
      if (!dead) dead = !__all_sync(0xffffffffu, mbar_wait(full0 + 8 * s, (it / S) & 1, a.error_flag));
      const int k0 = stage_key[s];
      if (!dead && k0 >= 0) {
        const uint32_t kt = stage0 + s * G_::kStage, vt = kt + G_::kTile;
        const int w0 = warp * NK;  // this warp's keys of the block
        const bool whole = attend_whole(a, t.pos0, t.last(), k0, KB);
        float x[NK / 8][4];
#pragma unroll
        for (int i = 0; i < NK / 8; ++i) x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0.f;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
#pragma unroll
          for (int i = 0; i < NK / 16; ++i) {  // 16 keys: matrices (keys 0-7, dims 0-7), (0-7, 8-15), (8-15, 0-7), (8-15, 8-15)
            uint32_t b[4];
            ldsm4(tile_addr<KB>(kt, w0 + 16 * i + (lane & 7) + (lane >> 4) * 8, 16 * k + ((lane >> 3) & 1) * 8), b);
            mma<FP16>(x[2 * i], qf[k], b[0], b[1]);
            mma<FP16>(x[2 * i + 1], qf[k], b[2], b[3]);
          }
        }
        if (!whole) {
#pragma unroll
          for (int i = 0; i < NK / 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!attend_sees(a, pos[e >> 1], k0 + w0 + 8 * i + 2 * (lane & 3) + (e & 1))) x[i][e] = -INFINITY;
          // A masked key weighs nothing whatever its value row holds, but 0 * inf
          // is not 0 in the product: infinite and NaN values leave the tile here
          // and reach the rows that do see them by addition.
          bool odd = false;
          for (int i = lane; i < NK * (D / 8); i += 32) {
            uint32_t w[4];
            const uint32_t ad = tile_addr<KB>(vt, w0 + i / (D / 8), (i % (D / 8)) * 8);
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(ad) : "memory");
            odd |= odd_pair<FP16>(w[0]) | odd_pair<FP16>(w[1]) | odd_pair<FP16>(w[2]) | odd_pair<FP16>(w[3]);
          }
          if (__any_sync(0xffffffffu, odd)) {
            uint32_t keys = 0;  // that hold some, a bit each
            static_assert(NK <= 32, "");
            for (int i = lane; i < NK * (D / 2); i += 32) {
              uint32_t w;
              asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w)
                           : "r"(tile_addr<KB>(vt, w0 + i / (D / 2), (i % (D / 2)) * 2)) : "memory");
              if (odd_pair<FP16>(w)) keys |= 1u << (i / (D / 2));
            }
            keys = __reduce_or_sync(0xffffffffu, keys);
            for (uint32_t left = keys; left; left &= left - 1) {
              const int key = __ffs(left) - 1;
              const bool sees0 = attend_sees(a, pos[0], k0 + w0 + key), sees1 = attend_sees(a, pos[1], k0 + w0 + key);
              if (!__any_sync(0xffffffffu, sees0 || sees1)) continue;  // past a request's length no row sees it
#pragma unroll
              for (int i = 0; i < D / 8; ++i) {
                uint32_t w;
                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w)
                             : "r"(tile_addr<KB>(vt, w0 + key, 8 * i + 2 * (lane & 3))) : "memory");
                if (odd_pair<FP16>(w)) {
                  const float2 v = unpack2(w, E{});
                  const float v0 = isfinite(v.x) ? 0.f : v.x, v1 = isfinite(v.y) ? 0.f : v.y;
                  if (sees0) o[i][0] += v0, o[i][1] += v1;
                  if (sees1) o[i][2] += v0, o[i][3] += v1;
                }
              }
            }
            __syncwarp();
            for (int i = lane; i < NK * (D / 2); i += 32) {
              const uint32_t ad = tile_addr<KB>(vt, w0 + i / (D / 2), (i % (D / 2)) * 2);
              uint32_t w;
              asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(ad) : "memory");
              if (odd_pair<FP16>(w)) {
                const float2 v = unpack2(w, E{});
                w = (isfinite(v.x) ? w & 0xffffu : 0u) | (isfinite(v.y) ? w & 0xffff0000u : 0u);
                asm volatile("st.shared.b32 [%0], %1;" ::"r"(ad), "r"(w) : "memory");
              }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the stage's next TMA write
            __syncwarp();
          }
        }
        // running maximum; rows that have seen nothing yet keep their weights at 0
        float ms[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float mx = m[j];
#pragma unroll
          for (int i = 0; i < NK / 8; ++i) mx = fmaxf(mx, fmaxf(x[i][2 * j], x[i][2 * j + 1]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const float top = mx * a.scale_log2, old = m[j] * a.scale_log2;
          ms[j] = mx == -INFINITY ? 0.f : top - lift_of<FP16>(top);
          const float keep = m[j] == -INFINITY ? 0.f : exp2_approx(old - lift_of<FP16>(old) - ms[j]);
          if (mx != m[j]) {
            l[j] *= keep;
            if (m[j] != -INFINITY) {
#pragma unroll
              for (int i = 0; i < D / 8; ++i) o[i][2 * j] *= keep, o[i][2 * j + 1] *= keep;
            }
            m[j] = mx;
          }
        }
#pragma unroll
        for (int i = 0; i < NK / 8; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[i][e] = exp2_approx(fmaf(x[i][e], a.scale_log2, -ms[e >> 1]));
            l[e >> 1] += x[i][e];
          }
#pragma unroll
        for (int k = 0; k < NK / 16; ++k) {  // 16 keys of P V
          const uint32_t p[4] = {pack<FP16>(x[2 * k][0], x[2 * k][1]), pack<FP16>(x[2 * k][2], x[2 * k][3]),
                                 pack<FP16>(x[2 * k + 1][0], x[2 * k + 1][1]),
                                 pack<FP16>(x[2 * k + 1][2], x[2 * k + 1][3])};
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {  // matrices (keys 0-7, dims 0-7), (8-15, 0-7), (0-7, 8-15), (8-15, 8-15)
            uint32_t b[4];
            ldsm4t(tile_addr<KB>(vt, w0 + 16 * k + (lane & 15), 16 * i + (lane >> 4) * 8), b);
            mma<FP16>(o[2 * i], p, b[0], b[1]);
            mma<FP16>(o[2 * i + 1], p, b[2], b[3]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty0 + 8 * s);
    }

    // ---- join the four warps' parts ----
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      l[j] += __shfl_xor_sync(0xffffffffu, l[j], 1);
      l[j] += __shfl_xor_sync(0xffffffffu, l[j], 2);
      if ((lane & 3) == 0) merge_ml[warp][lane / 4 + 8 * j] = make_float2(m[j], l[j]);
      float* dst = merge_o + (warp * kRows + lane / 4 + 8 * j) * G_::kPitch + 2 * (lane & 3);
#pragma unroll
      for (int i = 0; i < D / 8; ++i) *reinterpret_cast<float2*>(dst + 8 * i) = make_float2(o[i][2 * j], o[i][2 * j + 1]);
    }
    consumers_sync();
    const bool starts = c.u == 0, ends = c.u + n == t.units;
    const int64_t part = 2 * (int64_t)blockIdx.x + (starts ? 1 : 0);
    for (int i = tid; i < rows * (D / 4); i += kConsumers * 32) {
      const int row = i / (D / 4), d = (i % (D / 4)) * 4;
      float mx = -INFINITY;
#pragma unroll
      for (int w = 0; w < kConsumers; ++w) mx = fmaxf(mx, merge_ml[w][row].x);
      float sum = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kConsumers; ++w) {
        const float2 ml = merge_ml[w][row];
        // an empty part has o = l = 0, or, with values that are not finite, what it has to add
        const float f = ml.x == -INFINITY ? 1.f : exp2_approx((ml.x - mx) * a.scale_log2 - lift_of<FP16>(ml.x * a.scale_log2));
        const float4 v = *reinterpret_cast<const float4*>(merge_o + (w * kRows + row) * G_::kPitch + d);
        sum += f * ml.y;
        acc.x += f * v.x, acc.y += f * v.y, acc.z += f * v.z, acc.w += f * v.w;
      }
      if (starts && ends) {
        const int tk = row / a.G, head = c.h * a.G + row - tk * a.G;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;  // a row that sees nothing answers 0
        uint2 w;
        w.x = pack<FP16>(acc.x * inv, acc.y * inv);
        w.y = pack<FP16>(acc.z * inv, acc.w * inv);
        *reinterpret_cast<uint2*>(a.out + (int64_t)(t.row0 + tk) * a.o_tok + (int64_t)head * a.o_head + d) = w;
        if (a.lse && d == 0)
          a.lse[(int64_t)(t.row0 + tk) * a.Hq + head] = sum == 0.f ? -INFINITY : mx * a.scale + logf(sum);
      } else {
        *reinterpret_cast<float4*>(a.part_o + (part * kRows + row) * D + d) = acc;
        if (d == 0) a.part_ml[part * kRows + row] = make_float2(mx, sum);
      }
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
    consumers_sync();  // the merge buffers are read
    if (c.left > 0) attend_advance(a, c);
  }
}

template <int D, bool FP16>
int launch_t(const AttendArgs& a, cudaStream_t st) {
  static bool configured[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return KVC_ECUDA;
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(attend_rows_kernel<D, FP16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             Geom<D>::kSmem) != cudaSuccess)
      return KVC_ECUDA;
    configured[dev] = true;
  }
  launch_dep(attend_rows_kernel<D, FP16>, dim3((unsigned)a.ctas), dim3(kThreads), (size_t)Geom<D>::kSmem, st, a);
  return launch_status();
}

// ---------------------------------------------------------------------------
// joins the parts of tiles cut by a CTA boundary
// ---------------------------------------------------------------------------

constexpr int kCombineWarps = 4;

// blockIdx.x: the CTA in which the tile starts; the warps of blockIdx.y share the rows.  Four parts at a time
// are on their way with their (m, l), and joined with a running maximum, so that nothing but the record comes
// before the loads: 250 rows of 128 values in 2 to 3 parts for each of 148 CTAs, 40 MB.
template <int D, bool FP16>
__global__ void __launch_bounds__(kCombineWarps * 32) attend_combine_kernel(const __grid_constant__ AttendArgs a) {
  pdl_wait();
  pdl_trigger();
  constexpr int kLanes = D < 128 ? D / 4 : 32;  // of a row, 4 values each, kVec times
  constexpr int kVec = D / (4 * kLanes), kRowsAtOnce = 32 / kLanes, kParts = 4;
  const int4 rec = a.record[blockIdx.x];
  if (rec.x == 0) return;
  const int lane = threadIdx.x & 31, in_row = lane % kLanes;
  const int rows = rec.z * a.G, parts = rec.x + 1;
  const int64_t first = 2 * (int64_t)blockIdx.x;  // part 0 is slot first + 1, part j slot first + 2 j
  for (int row = (blockIdx.y * kCombineWarps + (threadIdx.x >> 5)) * kRowsAtOnce + lane / kLanes; row < rows;
       row += gridDim.y * kCombineWarps * kRowsAtOnce) {
    float m = -INFINITY, sum = 0.f;
    float4 acc[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j0 = 0; j0 < parts; j0 += kParts) {  // in unit order
      float2 ml[kParts];
      float4 v[kParts][kVec];
#pragma unroll
      for (int j = 0; j < kParts; ++j) {
        ml[j] = make_float2(-INFINITY, 0.f);
        if (j0 + j >= parts) continue;
        const int64_t at = (j0 + j == 0 ? first + 1 : first + 2 * (int64_t)(j0 + j)) * a.rows + row;
        ml[j] = a.part_ml[at];
#pragma unroll
        for (int i = 0; i < kVec; ++i)
          v[j][i] = *reinterpret_cast<const float4*>(a.part_o + at * D + 4 * (in_row + i * kLanes));
      }
      float mx = m;
#pragma unroll
      for (int j = 0; j < kParts; ++j) mx = fmaxf(mx, ml[j].x);
      // an empty part has o = l = 0, or, with values that are not finite, what it has to add
      const float keep = m == -INFINITY ? 1.f : exp2_approx((m - mx) * a.scale_log2);
      m = mx;
      sum *= keep;
#pragma unroll
      for (int i = 0; i < kVec; ++i) acc[i].x *= keep, acc[i].y *= keep, acc[i].z *= keep, acc[i].w *= keep;
#pragma unroll
      for (int j = 0; j < kParts; ++j) {
        if (j0 + j >= parts) continue;
        const float f = ml[j].x == -INFINITY ? 1.f : exp2_approx((ml[j].x - mx) * a.scale_log2);
        sum += f * ml[j].y;
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          acc[i].x += f * v[j][i].x, acc[i].y += f * v[j][i].y;
          acc[i].z += f * v[j][i].z, acc[i].w += f * v[j][i].w;
        }
      }
    }
    const int tk = row / a.G, head = rec.w * a.G + row - tk * a.G;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;  // a row that sees nothing answers 0
    uint16_t* dst = a.out + (int64_t)(rec.y + tk) * a.o_tok + (int64_t)head * a.o_head;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      uint2 w;
      w.x = pack<FP16>(acc[i].x * inv, acc[i].y * inv);
      w.y = pack<FP16>(acc[i].z * inv, acc[i].w * inv);
      *reinterpret_cast<uint2*>(dst + 4 * (in_row + i * kLanes)) = w;
    }
    if (a.lse && in_row == 0)
      a.lse[(int64_t)(rec.y + tk) * a.Hq + head] = sum == 0.f ? -INFINITY : m * a.scale + logf(sum);
  }
}

int rows_launch(const AttendArgs& a, bool fp16, cudaStream_t st) {
  if (a.D == 64) return fp16 ? launch_t<64, true>(a, st) : launch_t<64, false>(a, st);
  if (a.D == 128) return fp16 ? launch_t<128, true>(a, st) : launch_t<128, false>(a, st);
  return fp16 ? launch_t<256, true>(a, st) : launch_t<256, false>(a, st);
}

int combine_launch(const AttendArgs& a, bool fp16, cudaStream_t st) {
  const unsigned y = (unsigned)a.rows / (a.rows > kRows ? 16 : 8);
  const dim3 grid((unsigned)a.ctas, y), block(kCombineWarps * 32);
  if (a.D == 64) launch_dep(fp16 ? attend_combine_kernel<64, true> : attend_combine_kernel<64, false>, grid, block, 0, st, a);
  else if (a.D == 128)
    launch_dep(fp16 ? attend_combine_kernel<128, true> : attend_combine_kernel<128, false>, grid, block, 0, st, a);
  else launch_dep(fp16 ? attend_combine_kernel<256, true> : attend_combine_kernel<256, false>, grid, block, 0, st, a);
  return launch_status();
}

int encode_cache_map(CUtensorMap* map, const void* cache, bool fp16, int D, int Hkv, int64_t block_stride,
                     int64_t num_blocks, int keys) {
  PFN_cuTensorMapEncodeTiled_v12000 fn = encode_fn();
  if (!fn) return KVC_ECUDA;
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)Hkv, (cuuint64_t)kBlock, (cuuint64_t)num_blocks};
  const cuuint64_t strides[3] = {(cuuint64_t)D * 2, (cuuint64_t)Hkv * D * 2, (cuuint64_t)block_stride * 2};
  const cuuint32_t box[4] = {(cuuint32_t)kSpan, 1, (cuuint32_t)keys, 1};
  const cuuint32_t one[4] = {1, 1, 1, 1};
  const CUresult rc =
      fn(map, fp16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(cache),
         dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return rc == CUDA_SUCCESS ? KVC_OK : KVC_ECUDA;
}

// [token][head][dim], boxes of 64 dims x the heads of a KV head x a tile half's tokens
int encode_query_map(CUtensorMap* map, const AttendArgs& a, bool fp16) {
  PFN_cuTensorMapEncodeTiled_v12000 fn = encode_fn();
  if (!fn) return KVC_ECUDA;
  const cuuint64_t dims[3] = {(cuuint64_t)a.D, (cuuint64_t)a.Hq, (cuuint64_t)a.num_tokens};
  const cuuint64_t strides[2] = {(cuuint64_t)a.q_head * 2, (cuuint64_t)a.q_tok * 2};
  const cuuint32_t box[3] = {(cuuint32_t)kSpan, (cuuint32_t)a.G, (cuuint32_t)a.sub};
  const cuuint32_t one[3] = {1, 1, 1};
  const CUresult rc =
      fn(map, fp16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<uint16_t*>(a.q),
         dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return rc == CUDA_SUCCESS ? KVC_OK : KVC_ECUDA;
}

constexpr int rows_keys(int D) { return D <= 128 ? 128 : 64; }

}  // namespace
}  // namespace kvc

using namespace kvc;

// Rows of a tile.  Up to 16 rows in the longest request: the 16-row kernel, which
// reads each K/V block once and streams at 0.9 of the copy rate and more; past
// that it reads them once per 16 rows, and the tcgen05 kernel, whose products are
// 128 rows wide whatever the rows in use, is ahead.  Measured, 32 requests at
// 4,608 keys, 5 query heads of 128 to a KV head, us (16-row / tcgen05): 5 rows 100 /
// 122, 15 rows 104 / 140, 20 rows 193 / 139; 16 requests at 30k, 8 of 256: 8 rows
// 165 / 169, 16 rows 184 / 177, 24 rows 328 / 187.
static int tile_rows(int max_query_len, int group, int head_dim) {
  return (int64_t)max_query_len * group <= kRows ? kRows : attend_umma_rows(head_dim);
}

// Workspace: parts' outputs, their (m, l), and one record per CTA.
static int64_t workspace_bytes(int ctas, int rows, int D) {
  return (int64_t)ctas * (2 * (int64_t)rows * (4 * D + 8) + 16);
}

extern "C" int64_t kvc_paged_attention_workspace_bytes(int max_query_len, int heads, int kv_heads, int head_dim) {
  if (max_query_len < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || heads / kv_heads > kRows ||
      (head_dim != 64 && head_dim != 128 && head_dim != 256))
    return 0;
  return workspace_bytes(sm_count(), tile_rows(max_query_len, heads / kv_heads, head_dim), head_dim);
}

extern "C" int kvc_paged_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, int dtype,
                                   int64_t num_tokens, int max_query_len, int heads, int kv_heads, int head_dim,
                                   const void* k_cache, int64_t k_block_stride, const void* v_cache,
                                   int64_t v_block_stride, int64_t num_blocks, const int32_t* block_table,
                                   int64_t table_stride, int table_width, const int32_t* query_start_loc,
                                   const int32_t* seq_lens, int num_requests, float scale, int window, int sinks,
                                   void* out, int64_t out_token_stride, int64_t out_head_stride, float* lse,
                                   void* workspace, int64_t workspace_size, int32_t* error_flag, void* stream) {
  KVC_CHECK_ARG(num_tokens >= 0 && num_tokens <= INT32_MAX && max_query_len >= 0 && heads > 0 && kv_heads > 0 &&
                    heads % kv_heads == 0 && num_requests >= 0 && num_blocks > 0 && num_blocks <= INT32_MAX &&
                    table_width >= 0 && table_stride >= 0 && (dtype == KVC_BF16 || dtype == KVC_FP16) &&
                    window >= 0 && sinks >= 0 && scale > 0.f && scale <= 3.0e38f,
                KVC_EINVAL);
  KVC_CHECK_ARG(heads / kv_heads <= kRows && (head_dim == 64 || head_dim == 128 || head_dim == 256) &&
                    num_requests <= kMaxAttendRequests && table_width <= kMaxAttendWidth,
                KVC_EUNSUPPORTED);
  if (num_requests == 0 || num_tokens == 0 || max_query_len == 0) return KVC_OK;
  KVC_CHECK_ARG(q && k_cache && v_cache && query_start_loc && seq_lens && out && workspace &&
                    (block_table || table_width == 0),
                KVC_ENULL);
  const int64_t page = (int64_t)kBlock * kv_heads * head_dim;
  KVC_CHECK_ARG(k_block_stride >= page && v_block_stride >= page, KVC_EINVAL);
  const int64_t strides[] = {q_token_stride, q_head_stride, out_token_stride, out_head_stride, k_block_stride,
                             v_block_stride};
  for (int64_t s : strides) KVC_CHECK_ARG(s > 0 && s % 8 == 0, KVC_EALIGN);
  const void* ptrs[] = {q, k_cache, v_cache, out, workspace};
  for (const void* p : ptrs) KVC_CHECK_ARG(aligned(p, 16), KVC_EALIGN);
  KVC_CHECK_ARG(aligned(lse, 4) && aligned(block_table, 4), KVC_EALIGN);
  AttendArgs a{};
  const bool fp16 = dtype == KVC_FP16;
  a.ctas = sm_count();
  a.rows = tile_rows(max_query_len, heads / kv_heads, head_dim);
  const bool wide = a.rows != kRows;
  KVC_CHECK_ARG(workspace_size >= workspace_bytes(a.ctas, a.rows, head_dim), KVC_EINVAL);
  a.q = (const uint16_t*)q;
  a.out = (uint16_t*)out;
  a.lse = lse;
  a.table = block_table;
  a.starts = query_start_loc;
  a.lens = seq_lens;
  a.part_o = (float*)workspace;
  a.part_ml = reinterpret_cast<float2*>(a.part_o + 2 * (int64_t)a.ctas * a.rows * head_dim);
  a.record = reinterpret_cast<int4*>(a.part_ml + 2 * (int64_t)a.ctas * a.rows);
  a.error_flag = error_flag;
  a.q_tok = q_token_stride, a.q_head = q_head_stride, a.o_tok = out_token_stride, a.o_head = out_head_stride;
  a.table_stride = table_stride, a.table_width = table_width, a.num_blocks = (int)num_blocks;
  a.num_tokens = num_tokens;
  a.R = num_requests, a.Hq = heads, a.Hkv = kv_heads, a.G = heads / kv_heads, a.D = head_dim;
  // past any cache: 2^30 is as good as more, and positions plus or minus it stay inside an int
  a.window = std::min(window, 1 << 30), a.sinks = window > 0 ? std::min(sinks, 1 << 30) : 0;
  a.sub = 128 / a.G;
  a.tok = wide ? a.rows / 128 * a.sub : kRows / a.G;
  a.scale = scale;
  a.scale_log2 = scale * 1.44269504088896340736f;
  const int keys = wide ? attend_umma_slot_keys(head_dim) : rows_keys(head_dim);
  int rc = encode_cache_map(&a.kmap, k_cache, fp16, head_dim, kv_heads, k_block_stride, num_blocks, keys);
  if (rc == KVC_OK)
    rc = encode_cache_map(&a.vmap, v_cache, fp16, head_dim, kv_heads, v_block_stride, num_blocks, keys);
  if (rc == KVC_OK && wide) rc = encode_query_map(&a.qmap, a, fp16);
  if (rc == KVC_OK) rc = wide ? attend_umma_launch(a, fp16, (cudaStream_t)stream) : rows_launch(a, fp16, (cudaStream_t)stream);
  if (rc == KVC_OK) rc = combine_launch(a, fp16, (cudaStream_t)stream);
  return rc;
}
