// Rotary positions with several axes, and the write of a step's keys and
// values into the paged cache (sm_100a).
//
// Frequency f of token t turns by theta = position[axis(f)][t] * omega[f]; the
// pair (x[f], x[F + f]) of every query and key head becomes
//     (x[f] cos - x[F+f] sin, x[F+f] cos + x[f] sin),
// the dims past rotary_dim = 2F pass.  Queries go to q_out, keys and values to
// the token's slot of the cache.
//
// Bound: HBM, 4 bytes per element of q, k and v (one read, one write), so q, k
// and v are touched once, in 16-byte vectors, and the rotated keys never exist
// outside the cache.  The angles are formed here rather than read from a
// table: a token's F angles serve its (q + kv) heads, so a CTA computes them
// once into shared memory.  An angle of a far position loses fp32's bits
// (position 50,000 at omega = 1 would be off by 2e-3), so the product and its
// reduction to (-1, 1] half turns are taken in fp64, which is F products per
// token next to 2 (q + 2 kv) D bytes of traffic; sine and cosine of the reduced
// angle, and the rotation, are fp32, rounded once to 16 bits.
//
// Four tokens a CTA once there are enough of them to fill the GPU several times
// (8,191 tokens, 16 q and 2 kv heads of 256 dims, 64 of them turned: 34.5 us, 4.9
// TB/s; 2 tokens 39, 8 tokens 44, one token 42 us), else one, for latency.
#include <algorithm>
#include <type_traits>

#include "kvc_common.cuh"

namespace {

constexpr int kMaxFreq = 128;
constexpr int kMaxAxes = 8;
constexpr int kThreads = 128, kTokens = 4;

struct RotaryArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* q_out;
  uint16_t* k_cache;
  uint16_t* v_cache;
  const int64_t* positions;
  const int64_t* slots;
  const float* omega;
  const int32_t* axis;
  int32_t* error_flag;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head, o_tok, o_head;  // strides in elements
  int64_t pos_stride, k_block, v_block;                                // block strides in elements
  int64_t num_slots, num_tokens;
  int Hq, Hk, D, F, axes;
  uint32_t per_magic, vec_magic;  // ceil(2^32 / vectors of a q or k head), and of a v head
  bool in_place;  // q_out is q: the pass band is already there
};

// read once; not the read-only path, since q_out may be q
__device__ __forceinline__ uint4 load16(const uint16_t* p) {
  uint4 r;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p)
               : "memory");
  return r;
}

template <class E>
__device__ __forceinline__ void rotate8(uint4& x, uint4& y, const float* cs, const float* sn) {
  uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 u = kvc::unpack2(xw[i], E{}), w = kvc::unpack2(yw[i], E{});
    const float c0 = cs[2 * i], c1 = cs[2 * i + 1], s0 = sn[2 * i], s1 = sn[2 * i + 1];
    xw[i] = (uint32_t)kvc::pack1(u.x * c0 - w.x * s0, E{}) | (uint32_t)kvc::pack1(u.y * c1 - w.y * s1, E{}) << 16;
    yw[i] = (uint32_t)kvc::pack1(w.x * c0 + u.x * s0, E{}) | (uint32_t)kvc::pack1(w.y * c1 + u.y * s1, E{}) << 16;
  }
  x = make_uint4(xw[0], xw[1], xw[2], xw[3]);
  y = make_uint4(yw[0], yw[1], yw[2], yw[3]);
}

// A token's work in 16-byte pieces: of each q and k head first the F / 8 pairs of
// vectors that turn into each other, then the passing ones; then the v heads.
// A CTA takes T tokens: a thread works out where its piece lies once for all of
// them, has their T (or 2 T) loads on their way at once, the first ones while
// the angles are formed, and the T F angles keep every thread busy.
template <class E, int T>
__global__ void __launch_bounds__(kThreads) rotary_write_kernel(const __grid_constant__ RotaryArgs a) {
  kvc::pdl_wait();
  kvc::pdl_trigger();
  __shared__ __align__(16) float cs[T][kMaxFreq], sn[T][kMaxFreq];
  const int64_t t0 = (int64_t)blockIdx.x * T;
  const int n = T == 1 ? 1 : (int)kvc::min64(T, a.num_tokens - t0);
  const int tid = threadIdx.x;
  const int pairs = a.F / 8, per = pairs + (a.D - 2 * a.F) / 8, vec = a.D / 8;
  const int turned = (a.Hq + a.Hk) * per, items = turned + a.Hk * vec;
  __shared__ int64_t place[2][T];  // of the tokens' rows in the K and V caches, or -1
  bool angles = false;
  for (int base = 0; base < items; base += kThreads) {
    const int i = base + tid;
    const bool mine = i < items, value = i >= turned;
    const int k = value ? i - turned : i, of = value ? vec : per;
    const int h = of == 1 ? k : (int)__umulhi((uint32_t)k, value ? a.vec_magic : a.per_magic);
    const bool key = !value && h >= a.Hq, query = !value && !key;
    const bool pair = !value && k - h * of < pairs;
    const int dim = 8 * (k - h * of) + (value || pair ? 0 : a.F);  // 2 F + 8 (j - pairs) past the pairs
    const uint16_t* src = value ? a.v + t0 * a.v_tok + h * a.v_head
                          : key ? a.k + t0 * a.k_tok + (h - a.Hq) * a.k_head
                                : a.q + t0 * a.q_tok + h * a.q_head;
    const int64_t step = value ? a.v_tok : key ? a.k_tok : a.q_tok;
    uint4 x[T], y[T];
    if (mine) {
#pragma unroll
      for (int j = 0; j < T; ++j)
        if (j < n) {
          x[j] = load16(src + j * step + dim);
          if (pair) y[j] = load16(src + j * step + dim + a.F);
        }
    }
    if (!angles) {
      angles = true;
      if (tid < T) {
        int64_t slot = tid < n ? __ldg(a.slots + t0 + tid) : -1;
        if (slot >= a.num_slots) {
          kvc::raise_flag(a.error_flag, KVC_DEV_TOKEN_RANGE);
          slot = -1;
        }
        const int64_t block = slot / kvc::kBlock, row = (slot % kvc::kBlock) * a.Hk * a.D;
        place[0][tid] = slot < 0 ? -1 : block * a.k_block + row;
        place[1][tid] = slot < 0 ? -1 : block * a.v_block + row;
      }
      for (int e = tid; e < n * a.F; e += kThreads) {
        const int j = T == 1 ? 0 : e / a.F, f = e - j * a.F;
        int ax = a.axis ? __ldg(a.axis + f) : 0;
        if (ax < 0 || ax >= a.axes) {
          kvc::raise_flag(a.error_flag, KVC_DEV_INDEX_RANGE);
          ax = 0;
        }
        // half turns, reduced to [-1, 1]
        const double u = (double)__ldg(a.positions + ax * a.pos_stride + t0 + j) * (double)__ldg(a.omega + f) *
                         0.31830988618379067154;
        sincospif((float)(u - 2.0 * rint(0.5 * u)), &sn[j][f], &cs[j][f]);
      }
      __syncthreads();
    }
    if (!mine || (query && !pair && a.in_place)) continue;
    uint16_t* to = query ? a.q_out + t0 * a.o_tok + h * a.o_head + dim
                   : value ? a.v_cache + h * a.D + dim
                           : a.k_cache + (h - a.Hq) * a.D + dim;
#pragma unroll
    for (int j = 0; j < T; ++j) {
      if (j >= n) continue;
      const int64_t off = query ? j * a.o_tok : place[value][j];
      if (off < 0) continue;
      uint16_t* dst = to + off;
      if (pair) {
        rotate8<E>(x[j], y[j], cs[j] + dim, sn[j] + dim);
        *reinterpret_cast<uint4*>(dst + a.F) = y[j];
      }
      *reinterpret_cast<uint4*>(dst) = x[j];
    }
  }
}

template <int T>
void launch(const RotaryArgs& a, bool bf16, cudaStream_t st) {
  const dim3 grid((unsigned)((a.num_tokens + T - 1) / T)), block(kThreads);
  if (bf16) kvc::launch_dep(rotary_write_kernel<kvc::Bf16, T>, grid, block, 0, st, a);
  else kvc::launch_dep(rotary_write_kernel<kvc::Fp16, T>, grid, block, 0, st, a);
}

}  // namespace

extern "C" int kvc_rotary_write(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
                                int64_t k_token_stride, int64_t k_head_stride, const void* v, int64_t v_token_stride,
                                int64_t v_head_stride, int dtype, int64_t num_tokens, int heads, int kv_heads,
                                int head_dim, int rotary_dim, const int64_t* positions, int axes,
                                int64_t position_stride, const float* omega, const int32_t* axis_of_frequency,
                                const int64_t* slot_mapping, void* q_out, int64_t out_token_stride,
                                int64_t out_head_stride, void* k_cache, int64_t k_block_stride, void* v_cache,
                                int64_t v_block_stride, int64_t num_blocks, int32_t* error_flag, void* stream) {
  KVC_CHECK_ARG(num_tokens >= 0 && num_tokens <= INT32_MAX && heads > 0 && kv_heads > 0 && num_blocks > 0 &&
                    (dtype == KVC_BF16 || dtype == KVC_FP16) && axes >= 1 && axes <= kMaxAxes && head_dim > 0 &&
                    rotary_dim > 0 && rotary_dim <= head_dim && position_stride >= 0,
                KVC_EINVAL);
  KVC_CHECK_ARG(head_dim % 8 == 0 && rotary_dim % 16 == 0 && rotary_dim / 2 <= kMaxFreq && head_dim <= 1024 &&
                    heads <= 4096 && kv_heads <= 4096,
                KVC_EUNSUPPORTED);
  if (num_tokens == 0) return KVC_OK;
  KVC_CHECK_ARG(q && k && v && positions && omega && slot_mapping && q_out && k_cache && v_cache, KVC_ENULL);
  KVC_CHECK_ARG(axes == 1 || axis_of_frequency, KVC_ENULL);
  KVC_CHECK_ARG((num_tokens == 1 || out_token_stride > 0) && (heads == 1 || out_head_stride > 0), KVC_EINVAL);
  const int64_t row = (int64_t)kvc::kBlock * kv_heads * head_dim;
  KVC_CHECK_ARG(k_block_stride >= row && v_block_stride >= row, KVC_EINVAL);
  const int64_t strides[] = {q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride,
                             v_head_stride, out_token_stride, out_head_stride, k_block_stride, v_block_stride};
  for (int64_t s : strides) KVC_CHECK_ARG(s >= 0 && s % 8 == 0, KVC_EALIGN);
  const void* ptrs[] = {q, k, v, q_out, k_cache, v_cache};
  for (const void* p : ptrs) KVC_CHECK_ARG(kvc::aligned(p, 16), KVC_EALIGN);
  RotaryArgs a{};
  a.q = (const uint16_t*)q;
  a.k = (const uint16_t*)k;
  a.v = (const uint16_t*)v;
  a.q_out = (uint16_t*)q_out;
  a.k_cache = (uint16_t*)k_cache;
  a.v_cache = (uint16_t*)v_cache;
  a.positions = positions;
  a.slots = slot_mapping;
  a.omega = omega;
  a.axis = axis_of_frequency;
  a.error_flag = error_flag;
  a.q_tok = q_token_stride, a.q_head = q_head_stride;
  a.k_tok = k_token_stride, a.k_head = k_head_stride;
  a.v_tok = v_token_stride, a.v_head = v_head_stride;
  a.o_tok = out_token_stride, a.o_head = out_head_stride;
  a.pos_stride = position_stride;
  a.k_block = k_block_stride, a.v_block = v_block_stride;
  a.num_slots = num_blocks * kvc::kBlock;
  a.Hq = heads, a.Hk = kv_heads, a.D = head_dim, a.F = rotary_dim / 2, a.axes = axes;
  a.in_place = q_out == q && out_token_stride == q_token_stride && out_head_stride == q_head_stride;
  const auto magic = [](int n) { return (uint32_t)(((1ull << 32) + n - 1) / n); };  // exact for i * n < 2^32, n > 1
  a.per_magic = magic(rotary_dim / 16 + (head_dim - rotary_dim) / 8);
  a.vec_magic = magic(head_dim / 8);
  a.num_tokens = num_tokens;
  if (num_tokens >= kTokens * 4 * kvc::sm_count()) launch<kTokens>(a, dtype == KVC_BF16, (cudaStream_t)stream);
  else launch<1>(a, dtype == KVC_BF16, (cudaStream_t)stream);
  return kvc::launch_status();
}
