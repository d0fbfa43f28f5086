// Attention of each request's newest tokens over its paged KV cache: what the
// two kernels (kvc_attend.cu, kvc_attend_umma.cu) share.
//
// Request r has n new tokens, already written to its cache of `len` physical
// tokens; new token j sits at physical position p = len - n + j and sees
//     keys i <= p                                  (window == 0)
//     keys i <= p with i > p - window or i < sinks (window > 0)
// out = sum_i softmax_i(scale * q.k_i) v_i in base 2: with c = scale * log2(e)
// and the running maximum m, p_i = 2^(c s_i - c m), l = sum p_i, o = sum p_i v_i.
//
// A *tile* is the G query heads of one KV head for up to `tok` consecutive new
// tokens of a request (row = token * G + head in group), so a KV block is read
// once for all the heads that share it.  A *unit* is one KB-key block of a
// tile that some row sees.  The units of all tiles, KV heads outermost, form
// one line, on which a tile also takes the room of `Extra` units, about what its
// start and end cost; each CTA has an equal length of it, whatever the requests'
// lengths.  A tile whose units all fall to one CTA is finished there; the
// parts of a tile cut by a CTA boundary go to the workspace as (o, m, l) and
// attend_combine_kernel joins them in unit order, so results do not depend on
// timing.  Every CTA finds its piece from the lengths on the device: no plan
// has to be kept or refreshed, and a captured graph follows new lengths.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include "kvc_async.cuh"

namespace kvc {

constexpr float kLn2 = 0.69314718055994530942f;
constexpr int kMaxAttendRequests = 8192;
constexpr int kMaxAttendWidth = 1 << 22;  // entries of a table row: units of a block's threads stay within 32 bits

struct AttendArgs {
  CUtensorMap kmap, vmap;  // [block][token][head][dim], boxes of 64 dims x KB tokens of one head
  CUtensorMap qmap;        // [token][head][dim] (tcgen05 kernel)
  const uint16_t* q;
  uint16_t* out;
  float* lse;  // [tokens][Hq] or null
  const int32_t* table;
  const int32_t* starts;  // [R + 1]
  const int32_t* lens;    // [R]
  float* part_o;          // [2 * ctas][rows][D]
  float2* part_ml;        // [2 * ctas][rows] (m in score units, l)
  int4* record;           // [ctas] {parts after the first, first query token, tokens, KV head} of the tile cut at the CTA's end
  int32_t* error_flag;
  int64_t q_tok, q_head, o_tok, o_head, table_stride;
  int64_t num_tokens;  // rows of q
  int table_width, num_blocks;
  int R, Hq, Hkv, G, D;
  int window, sinks;
  int tok;   // tokens per tile
  int sub;   // tokens per 128-row half of a tile (tcgen05 kernel)
  int rows;  // rows of a partial
  int ctas;  // CTAs that share the line of units
  float scale, scale_log2;
};

// One tile: tokens [row0, row0 + ntok) of the batch at physical positions pos0, pos0 + 1, ..
struct AttendTile {
  int r, row0, ntok, pos0;
  int head_blocks;  // leading KB-key blocks that hold visible first tokens and lie before the window
  int lo_block;     // first block of the window
  int units;
  __device__ __forceinline__ int block_of(int u) const { return u < head_blocks ? u : lo_block + u - head_blocks; }
  __device__ __forceinline__ int last() const { return pos0 + ntok - 1; }
};

template <int KB>
__device__ __forceinline__ AttendTile attend_tile(const AttendArgs& a, int r, int i) {
  AttendTile t;
  const int q0 = __ldg(a.starts + r), q1 = __ldg(a.starts + r + 1), n = q1 - q0;
  t.r = r;
  t.row0 = q0 + i * a.tok;
  t.ntok = min(a.tok, n - i * a.tok);
  t.pos0 = max(__ldg(a.lens + r), 0) - n + i * a.tok;  // no keys: every row is before the first
  t.head_blocks = t.lo_block = 0;
  const int last = t.last();
  const int past = a.table_width * (kBlock / KB);  // of the blocks past the table a tile has this one, which raises the error
  if (a.window > 0 && t.pos0 >= a.window) {
    t.lo_block = min((t.pos0 - a.window + 1) / KB, past);
    t.head_blocks = min((a.sinks + KB - 1) / KB, t.lo_block);
  }
  // a tile that sees nothing still has one unit, so that its rows are written
  t.units = last < 0 ? 1 : t.head_blocks + min(last / KB, past) - t.lo_block + 1;
  return t;
}

__device__ __forceinline__ int attend_tiles(const AttendArgs& a, int r) {
  const int q0 = __ldg(a.starts + r), q1 = __ldg(a.starts + r + 1);
  if (q0 < 0 || q1 < q0 || q1 > a.num_tokens) {  // rows that q does not have: the request is left out
    raise_flag(a.error_flag, KVC_DEV_INDEX_RANGE);
    return 0;
  }
  return (q1 - q0 + a.tok - 1) / a.tok;
}

// Position on the line of units: tile i of request r, KV head h, unit u of the tile.
struct AttendCursor {
  int h, r, i, u;
  int64_t left;  // units of this CTA from here on
};

// the line, and how it is shared: CTA c has the units [c * total / used, (c + 1) * total / used)
struct AttendLine {
  int64_t total;  // units of all KV heads
  int64_t used;   // CTAs that have work
};

// a / b, a < 2^53: a quotient that is no whole number lies 1 / b under the next one, more than the division's
// rounding (a few dozen instructions, against a few hundred for 64-bit integers)
__device__ __forceinline__ int64_t attend_div(int64_t a, int64_t b) { return (int64_t)__ddiv_rd((double)a, (double)b); }

// CTA that owns place x of the line
__device__ __forceinline__ int64_t attend_owner(const AttendLine& l, int64_t x) {
  return attend_div((x + 1) * l.used - 1, l.total);
}

constexpr int kLocateInts = 72;  // shared memory of attend_locate beside the R + 1 prefix sums, in ints

// All threads: this CTA's piece of the line.  `sh`: kLocateInts + R + 1 ints of shared memory, free again on return.
template <int KB, int NT, int Extra>
__device__ AttendCursor attend_locate(const AttendArgs& a, int32_t* sh, AttendLine* line) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int32_t* first = sh + kLocateInts;  // [R + 1] tiles before each request
  constexpr int kWarps = NT / 32;
  static_assert(kWarps <= 32, "");
  auto scan = [&](auto n, auto& all) {  // exclusive prefix of n over the threads
    using T = decltype(n);
    T* totals = reinterpret_cast<T*>(sh);  // [32]
    T v = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const T u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 31) totals[warp] = v;
    __syncthreads();
    T before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const T t = totals[w];
      if (w < warp) before += t;
      all += t;
    }
    return before + v - n;
  };
  // In 64 bits: starts that go back can name q's rows any number of times.  Requests with rows of their own have no
  // more tiles than rows, and with more than that and one for each request none is served.
  int64_t carry = 0, some = 0;
  for (int r0 = 0; r0 < a.R; r0 += NT) {
    const int r = r0 + tid;
    const int64_t before = scan((int64_t)(r < a.R ? attend_tiles(a, r) : 0), some);
    if (r < a.R) first[r] = (int32_t)min64(carry + before, INT32_MAX);
    carry += some;
  }
  if (carry > min64(a.num_tokens + a.R, INT32_MAX)) {
    raise_flag(a.error_flag, KVC_DEV_INDEX_RANGE);
    carry = 0;
  }
  if (tid == 0) first[a.R] = (int32_t)carry;
  __syncthreads();
  const int tiles = (int)carry;
  int all = 0;
  auto tile_of = [&](int t, int& r) {  // request of tile t: the last that starts at or before it
    int lo = 0, hi = a.R - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first[mid] <= t) lo = mid; else hi = mid - 1;
    }
    r = lo;
    return t - first[lo];
  };
  // length of one KV head, and -- when one round of threads covers the tiles -- each tile's place
  int64_t sum = 0;
  int mine = 0, before = 0, my_r = 0, my_i = 0;
  auto measure = [&](int t) {
    mine = 0;
    if (t < tiles) {
      my_i = tile_of(t, my_r);
      mine = Extra + attend_tile<KB>(a, my_r, my_i).units;
    }
    before = scan(mine, all);
  };
  for (int t0 = 0; t0 < tiles; t0 += NT) {
    measure(t0 + tid);
    sum += all;
  }
  AttendCursor c{0, 0, 0, 0, 0};
  line->total = sum * a.Hkv;
  line->used = min((int64_t)a.ctas, line->total);
  int32_t* found = sh + 64;  // start: request, tile of it, tile of the head, place in the tile; end: the last two
  if ((int64_t)blockIdx.x < line->used) {  // the same for the whole CTA
    const int64_t x0 = attend_div((int64_t)blockIdx.x * line->total, line->used);
    const int64_t x1 = attend_div(((int64_t)blockIdx.x + 1) * line->total, line->used);
    const int64_t h0 = attend_div(x0, sum), h1 = attend_div(x1, sum);
    const int64_t want0 = x0 - h0 * sum, want1 = x1 - h1 * sum;
    int64_t base = 0;
    for (int t0 = 0; t0 < tiles; t0 += NT) {
      const int t = t0 + tid;
      if (tiles > NT) measure(t);
      const int64_t at = base + before;
      if (at <= want0 && want0 < at + mine) {
        found[0] = my_r;
        found[1] = my_i;
        found[2] = t;
        found[3] = (int)(want0 - at);
      }
      if (at <= want1 && want1 < at + mine) {
        found[4] = t;
        found[5] = (int)(want1 - at);
      }
      base += all;
      if (base > want0 && base > want1) break;
    }
    __syncthreads();
    // units before a place: its distance, less the extra room of the tiles before it and of its own
    const int64_t u0 = x0 - Extra * (h0 * tiles + found[2]) - min(found[3], Extra);
    const int64_t u1 = x1 - Extra * (h1 * tiles + found[4]) - min(found[5], Extra);
    c = AttendCursor{(int)h0, found[0], found[1], max(0, found[3] - Extra), u1 - u0};
  }
  __syncthreads();
  return c;
}

// the next tile on the line
__device__ __forceinline__ void attend_advance(const AttendArgs& a, AttendCursor& c) {
  c.u = 0;
  if (++c.i < attend_tiles(a, c.r)) return;
  c.i = 0;
  do {
    if (++c.r == a.R) {
      c.r = 0;
      ++c.h;
    }
  } while (attend_tiles(a, c.r) == 0);
}

// whether rows at positions first to last see all n keys from k0 on
__device__ __forceinline__ bool attend_whole(const AttendArgs& a, int first, int last, int k0, int n) {
  if (k0 + n - 1 > first) return false;
  return a.window == 0 || k0 > last - a.window || k0 + n <= a.sinks;
}

__device__ __forceinline__ bool attend_sees(const AttendArgs& a, int pos, int key) {
  return key <= pos && (a.window == 0 || key > pos - a.window || key < a.sinks);
}

// Block id of the tile's KB-key block, or -1 (with the error raised) when the
// table does not name one inside the cache.
template <int KB>
__device__ __forceinline__ int attend_block(const AttendArgs& a, const AttendTile& t, int key_block) {
  const int page = key_block / (kBlock / KB);
  const int id = page < a.table_width ? __ldg(a.table + (int64_t)t.r * a.table_stride + page) : -1;
  if (id < 0 || id >= a.num_blocks) {
    raise_flag(a.error_flag, KVC_DEV_BLOCK_RANGE);
    return -1;
  }
  return id;
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn();  // kvc_score_tc.cu

// kvc_attend_umma.cu: tiles of up to 256 rows
int attend_umma_rows(int D);       // rows of a tile
int attend_umma_slot_keys(int D);  // keys of a K/V box
int attend_umma_launch(const AttendArgs& a, bool fp16, cudaStream_t st);

}  // namespace kvc
