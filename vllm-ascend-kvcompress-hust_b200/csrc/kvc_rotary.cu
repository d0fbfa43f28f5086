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
// table: a token's F angles serve its (q + kv) heads, so one CTA per token
// computes them once into shared memory.  An angle of a far position loses
// fp32's bits (position 50,000 at omega = 1 would be off by 2e-3), so the
// product and its reduction to (-1, 1] half turns are taken in fp64, which is
// F products per token next to 2 (q + 2 kv) D bytes of traffic; sine and cosine
// of the reduced angle, and the rotation, are fp32, rounded once to 16 bits.
#include <algorithm>
#include <type_traits>

#include "kvc_common.cuh"

namespace {

constexpr int kMaxFreq = 128;
constexpr int kMaxAxes = 8;

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
  int64_t num_slots;
  int Hq, Hk, D, F, axes;
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

template <class E>
__global__ void __launch_bounds__(256) rotary_write_kernel(const __grid_constant__ RotaryArgs a) {
  kvc::pdl_wait();
  kvc::pdl_trigger();
  __shared__ __align__(16) float cs[kMaxFreq], sn[kMaxFreq];
  const int64_t t = blockIdx.x;
  const int tid = threadIdx.x, nt = blockDim.x;
  for (int f = tid; f < a.F; f += nt) {
    int ax = a.axis ? __ldg(a.axis + f) : 0;
    if (ax < 0 || ax >= a.axes) {
      kvc::raise_flag(a.error_flag, KVC_DEV_INDEX_RANGE);
      ax = 0;
    }
    // half turns, reduced to [-1, 1]
    const double u = (double)__ldg(a.positions + ax * a.pos_stride + t) * (double)__ldg(a.omega + f) *
                     0.31830988618379067154;
    sincospif((float)(u - 2.0 * rint(0.5 * u)), &sn[f], &cs[f]);
  }
  int64_t slot = __ldg(a.slots + t);
  if (slot >= a.num_slots) {
    if (tid == 0) kvc::raise_flag(a.error_flag, KVC_DEV_TOKEN_RANGE);
    slot = -1;
  }
  const int64_t block = slot / kvc::kBlock, row = (slot % kvc::kBlock) * a.Hk;
  uint16_t* kd = a.k_cache + block * a.k_block + row * a.D;
  uint16_t* vd = a.v_cache + block * a.v_block + row * a.D;
  __syncthreads();

  const int pairs = a.F / 8, pass = (a.D - 2 * a.F) / 8, per = pairs + pass;
  const int heads = slot < 0 ? a.Hq : a.Hq + a.Hk;  // a token without a slot turns its queries alone
  for (int i = tid; i < heads * per; i += nt) {
    const int h = i / per, j = i - h * per;
    const bool key = h >= a.Hq;
    const uint16_t* src = key ? a.k + t * a.k_tok + (h - a.Hq) * a.k_head : a.q + t * a.q_tok + h * a.q_head;
    uint16_t* dst = key ? kd + (h - a.Hq) * a.D : a.q_out + t * a.o_tok + h * a.o_head;
    if (j < pairs) {
      uint4 x = load16(src + 8 * j), y = load16(src + a.F + 8 * j);
      rotate8<E>(x, y, cs + 8 * j, sn + 8 * j);
      *reinterpret_cast<uint4*>(dst + 8 * j) = x;
      *reinterpret_cast<uint4*>(dst + a.F + 8 * j) = y;
    } else if (key || !a.in_place) {
      const int d = 2 * a.F + 8 * (j - pairs);
      *reinterpret_cast<uint4*>(dst + d) = load16(src + d);
    }
  }
  if (slot < 0) return;
  const int vec = a.D / 8;
  for (int i = tid; i < a.Hk * vec; i += nt) {
    const int h = i / vec, d = (i - h * vec) * 8;
    *reinterpret_cast<uint4*>(vd + h * a.D + d) = load16(a.v + t * a.v_tok + h * a.v_head + d);
  }
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
  KVC_CHECK_ARG(head_dim % 8 == 0 && rotary_dim % 16 == 0 && rotary_dim / 2 <= kMaxFreq, KVC_EUNSUPPORTED);
  if (num_tokens == 0) return KVC_OK;
  KVC_CHECK_ARG(q && k && v && positions && omega && slot_mapping && q_out && k_cache && v_cache, KVC_ENULL);
  KVC_CHECK_ARG(axes == 1 || axis_of_frequency, KVC_ENULL);
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
  const dim3 grid((unsigned)num_tokens), block(128);
  if (dtype == KVC_BF16)
    kvc::launch_dep(rotary_write_kernel<kvc::Bf16>, grid, block, 0, (cudaStream_t)stream, a);
  else
    kvc::launch_dep(rotary_write_kernel<kvc::Fp16>, grid, block, 0, (cudaStream_t)stream, a);
  return kvc::launch_status();
}
