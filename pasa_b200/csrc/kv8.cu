// Keys and values in 8 bits, in pages of 64 tokens, and attention over them.
//
// A page holds 64 tokens of every key/value head as e4m3, with one scale a head
// and page: the smallest power of two (2^-100 at least) that brings the largest
// absolute value to 448 or below.  A power of two costs an e4m3 value nothing
// but range at the very bottom, and makes x / scale and q * scale exact, so the
// only rounding is the one to e4m3 and it does not depend on the order of
// anything.  A request's tokens lie in the pages that its row of a block table
// names.  A page with an infinity or NaN among its values has the scale NaN, and
// reads as NaN.
//
//   write      rounds new tokens into pages.  Where a page has earlier tokens its
//              scale is the larger of theirs and the new ones', and they are
//              rounded again to it.  Bound: HBM, 2 bytes read and 1 written a value.
//   attention  out = softmax(q k^T scale) v over a request's first `length`
//              tokens.  Bound: the tensor cores for many queries, HBM (one byte a
//              value) for single tokens.
//
// Attention on the tensor cores (tcgen05) takes the pages as they are, without
// converting them: both products run on e4m3 operands (twice the rate of bf16),
// and the 16-bit operand of each goes in as two e4m3 terms, hi + lo.  A bf16
// value has 8 significant bits and an e4m3 value 4, so q = s (hi + lo) is exact
// for a row's elements down to 2^-11 of its largest, and 2^-19 of the largest
// off below (s: a power of two for each row); the probabilities are kept to 8
// significant bits or 2^-16 of the largest, as a bf16 one would be.  The two
// terms together take the time of one bf16 product and read 8-bit keys and
// values from shared memory.  Scores, maxima, sums and the output are fp32.
//
// Work split.  A unit is a request, a key/value head and 256 of the rows
// (query, query head of the group) that attend with it; its cost is its steps of
// 128 tokens and two more.  The line of all units is cut into equal parts, one
// for each of the GPU's SMs, so neither the number of units nor their lengths
// leave SMs idle; a unit that is cut leaves its parts (fp32 sums, maximum and
// denominator) in the workspace, and a second kernel joins them.  With at most
// 128 rows (single tokens) the two tiles of a unit hold the same rows and take
// the steps in turn, which hides the one's softmax behind the other's products.
#include <cuda_fp16.h>

#include "umma.cuh"

namespace pasa {
namespace kv8 {

constexpr int kPage = 64;
constexpr int kMinScaleExp = -100;

// 8 consecutive bf16 values.
struct Bf8 {
  uint4 r;
  __device__ __forceinline__ float operator[](int i) const {
    const uint32_t w = i < 2 ? r.x : i < 4 ? r.y : i < 6 ? r.z : r.w;
    return __uint_as_float(i & 1 ? (w & 0xFFFF0000u) : (w << 16));
  }
  // the largest absolute value's bits
  __device__ __forceinline__ uint32_t amax() const {
    const uint32_t m = __vmaxu2(__vmaxu2(r.x & 0x7FFF7FFFu, r.y & 0x7FFF7FFFu),
                                __vmaxu2(r.z & 0x7FFF7FFFu, r.w & 0x7FFF7FFFu));
    return max(m & 0xFFFFu, m >> 16);
  }
};

// The scale for a largest absolute value given as bf16 bits; NaN if that is not finite.
__device__ __forceinline__ float scale_of(uint32_t amax) {
  if (amax >= 0x7F80u) return __uint_as_float(0x7FC00000u);
  // amax = 1.f * 2^e <= 448 * 2^t = 1.75 * 2^(8 + t)
  const int e = int(amax >> 7) - 127;
  const int t = max(e - 8 + ((amax & 0x7Fu) > 0x60u ? 1 : 0), kMinScaleExp);
  return __uint_as_float(uint32_t(t + 127) << 23);
}
// 1 / scale, exact.
__device__ __forceinline__ float inverse(float scale) {
  const uint32_t b = __float_as_uint(scale);
  return b >= 0x7F800000u ? scale : __uint_as_float((254u << 23) - b);
}

__device__ __forceinline__ uint16_t to_e4m3x2(float lo, float hi) {
  uint16_t d;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint16_t v) {
  uint32_t d;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(d) : "h"(v));
  return d;
}
__device__ __forceinline__ uint16_t f16x2_to_e4m3x2(uint32_t v) {
  uint16_t d;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(d) : "r"(v));
  return d;
}
__device__ __forceinline__ float2 unpack_e4m3x2(uint16_t v) {
  const uint32_t h = e4m3x2_to_f16x2(v);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// ---------------------------------------------------------------------------
// write: a block takes one page and head of k or of v
// ---------------------------------------------------------------------------
constexpr int kWriteThreads = 128;

struct WriteArgs {
  const __nv_bfloat16* x[2];   // new keys, values
  int64_t xs[2][3];            // strides of batch, head, token
  uint8_t* cache[2];           // [pages][heads][64][dim]
  float* scale[2];             // [pages][heads]
  const int32_t* table;        // [batch][width]
  const int32_t* starts;       // [batch] tokens before the new ones
  const int32_t* counts;       // [batch] new tokens, or null: all
  int64_t pages, width, tokens;
  int heads;
  uint32_t* err;
};

template <int D>
__global__ void __launch_bounds__(kWriteThreads) write_kernel(const __grid_constant__ WriteArgs a) {
  constexpr int kRowVecs = D / 8, kVecs = kPage * kRowVecs / kWriteThreads;
  __shared__ uint32_t amax_of[kWriteThreads / 32];
  const int which = int(blockIdx.y) & 1, head = int(blockIdx.y) >> 1, b = int(blockIdx.z), tid = threadIdx.x;
  const int64_t start = a.starts[b];
  int64_t count = a.counts ? a.counts[b] : a.tokens;
  if (count > a.tokens) count = a.tokens;
  if (start < 0 || count <= 0) return;
  const int64_t block = start / kPage + blockIdx.x, at = block * kPage;  // the page's first token
  if (at >= start + count) return;
  const int held = start > at ? int(start - at) : 0;  // earlier tokens of the page
  const int end = start + count - at < kPage ? int(start + count - at) : kPage;
  const int64_t page = block < a.width ? a.table[b * a.width + block] : -1;
  if (page < 0 || page >= a.pages) {
    if (tid == 0) atomicOr(a.err, PASA_DEVERR_BAD_PAGE);
    return;
  }
  const __nv_bfloat16* x = a.x[which] + b * a.xs[which][0] + head * a.xs[which][1];
  Bf8 v[kVecs];
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int vec = tid + i * kWriteThreads, row = vec / kRowVecs, c = vec % kRowVecs * 8;
    v[i].r = make_uint4(0u, 0u, 0u, 0u);
    if (row >= held && row < end)
      v[i].r = *reinterpret_cast<const uint4*>(x + (at + row - start) * a.xs[which][2] + c);
    amax = max(amax, v[i].amax());
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, off));
  if ((tid & 31) == 0) amax_of[tid >> 5] = amax;
  float* at_scale = a.scale[which] + page * a.heads + head;
  const float old = held > 0 ? *at_scale : 0.f;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWriteThreads / 32; ++w) amax = max(amax, amax_of[w]);
  float scale = scale_of(amax);
  if (held > 0 && !(scale >= old)) scale = isnan(scale) ? scale : old;  // the larger, NaN before all
  const float inv = inverse(scale);
  uint8_t* cache = a.cache[which] + (page * a.heads + head) * (kPage * D);
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int vec = tid + i * kWriteThreads, row = vec / kRowVecs, c = vec % kRowVecs * 8;
    uint2* dst = reinterpret_cast<uint2*>(cache + row * D + c);
    uint16_t o[4];
    if (row >= held && row < end) {
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = to_e4m3x2(v[i][2 * e] * inv, v[i][2 * e + 1] * inv);
    } else if (row < held && scale != old) {  // round the earlier tokens again
      const uint2 was = *dst;
      const uint16_t q[4] = {uint16_t(was.x), uint16_t(was.x >> 16), uint16_t(was.y), uint16_t(was.y >> 16)};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = unpack_e4m3x2(q[e]);
        o[e] = to_e4m3x2(f.x * (old * inv), f.y * (old * inv));
      }
    } else {
      continue;
    }
    *dst = make_uint2(uint32_t(o[0]) | uint32_t(o[1]) << 16, uint32_t(o[2]) | uint32_t(o[3]) << 16);
  }
  if (tid == 0) *at_scale = scale;
}

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------
constexpr int kTile = 128;          // rows of a tile
constexpr int kStep = 128;          // tokens of a step: two pages
constexpr int kSlotBytes = kStep * 128;
constexpr int kMaxSlots = 4;        // ring of keys' and values' steps
constexpr int kQTile = 2 * kTile * 128;  // hi, lo
constexpr int kQBuf = 2 * kQTile;   // two tiles
constexpr int kThreads = 512;       // 0 TMA, 1 MMA + TMEM, 2-3 and 12-15 queries, 4-7 and 8-11 softmax
constexpr int kLoaders = 6;
constexpr int kOverhead = 2;        // steps' time that a unit takes besides its steps
constexpr float kLog2P = 4.f;       // probabilities are held times 2^4 ...
constexpr float kRescale = 4.f;     // ... and their reference lags the maximum by up to 2^4: at most 2^8 < 448
constexpr int kOffQ = 0;                        // [2 buffers][2 tiles][hi, lo][128 rows][128 bytes]
constexpr int kOffRing = 2 * kQBuf;
constexpr int kOffOut = kOffRing + kMaxSlots * kSlotBytes;   // [8 warps][32 rows][64 bytes]
constexpr int kOffScale = kOffOut + 8 * 32 * 64;  // f32 [2 buffers][256 rows]: the queries' scales
constexpr int kSmem = kOffScale + 2 * 2 * kTile * 4 + 1024;
// Tile t: scores at kColS + 128 t, the probabilities (hi, then lo, 32 columns
// each) over the first 64 of them; output at kColO + 128 t.
constexpr uint32_t kColS = 0, kColO = 256;
static_assert(kSmem + 1024 <= 232448, "shared memory budget");

struct Maps {
  CUtensorMap k, v;
};
struct Args {
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  int64_t qs[3], os[3];        // strides of batch, head, query
  const float* k_scale;        // [pages][heads]
  const float* v_scale;
  const int32_t* table;        // [batch][width]
  const int32_t* lengths;      // [batch]
  int64_t pages, width;
  int batch, heads, group;     // key/value heads; query heads of each
  int rows, blocks;            // rows of a key/value head (queries x group); units of 256 of them
  int both;                    // 1: both tiles hold the same rows and take the steps in turn
  float scale_log2;            // softmax scale * log2(e)
  float* part_o;               // [2 parts a CTA][256][D]
  float2* part_ml;             // [2 parts a CTA][256]: maximum, denominator
  uint32_t* err;
};

__device__ __forceinline__ int request_tokens(const Args& a, int b) {
  const int64_t most = a.width * kPage;
  const int n = a.lengths[b];
  return n < 0 ? 0 : n > most ? int(most) : n;
}
__device__ __forceinline__ int request_steps(const Args& a, int b) {
  return (request_tokens(a, b) + kStep - 1) / kStep;
}

// Ticks of the line of all units: a unit takes kOverhead and its steps.  All lanes.
__device__ __forceinline__ int64_t total_ticks(const Args& a, int lane) {
  int64_t sum = 0;
  for (int b = lane; b < a.batch; b += 32) sum += request_steps(a, b) + kOverhead;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  return sum * a.heads * a.blocks;
}
__device__ __forceinline__ int64_t part_begin(int64_t total, int part, int parts) {
  return total / parts * part + total % parts * part / parts;
}

struct Unit {
  int b, head, block;
  int steps;       // of the request
  int64_t begin;   // first tick
};

// The unit that holds a tick.  All lanes.
__device__ __forceinline__ Unit find_unit(const Args& a, int64_t tick, int lane) {
  const int64_t units = int64_t(a.heads) * a.blocks;
  int64_t before = 0;
  for (int b0 = 0;; b0 += 32) {
    const int b = b0 + lane;
    const int steps = b < a.batch ? request_steps(a, b) : 0;
    const int64_t own = b < a.batch ? (steps + kOverhead) * units : 0;
    int64_t upto = own;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= off) upto += v;
    }
    const uint32_t reached = __ballot_sync(0xffffffffu, before + upto > tick);
    if (reached != 0) {
      const int src = __ffs(int(reached)) - 1;
      Unit u;
      u.b = b0 + src;
      u.steps = __shfl_sync(0xffffffffu, steps, src);
      const int64_t first = before + __shfl_sync(0xffffffffu, upto - own, src);
      const int64_t index = (tick - first) / (u.steps + kOverhead);
      u.begin = first + index * (u.steps + kOverhead);
      u.head = int(index / a.blocks);
      u.block = int(index % a.blocks);
      return u;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
    if (b0 + 32 >= a.batch) return Unit{0, 0, 0, 0, before};  // (no unit: a tick behind the last)
  }
}

// What a CTA does of a unit.
struct Piece {
  Unit u;
  int first, count;  // steps
  bool whole;        // the unit's only piece
  bool zero;         // the request has no tokens and this CTA writes its zeros
  int part;          // 0 if it begins with the CTA's part of the line, else 1
};

// Goes through a CTA's part of the line of units.  Every warp has one of its own.
struct Walk {
  int64_t at, begin, end;
  __device__ __forceinline__ Walk(const Args& a, int lane) {
    const int64_t total = total_ticks(a, lane);
    begin = at = part_begin(total, int(blockIdx.x), int(gridDim.x));
    end = part_begin(total, int(blockIdx.x) + 1, int(gridDim.x));
  }
  __device__ __forceinline__ bool next(const Args& a, int lane, Piece& p) {
    while (at < end) {
      p.u = find_unit(a, at, lane);
      const int lo = int(at - p.u.begin), most = p.u.steps + kOverhead;
      const int hi = end - p.u.begin < most ? int(end - p.u.begin) : most;
      p.first = max(lo - kOverhead, 0);
      p.count = max(hi - kOverhead, 0) - p.first;
      p.whole = p.first == 0 && p.count == p.u.steps;
      p.zero = p.u.steps == 0 && lo == 0;
      p.part = at == begin ? 0 : 1;
      at = p.u.begin + hi;
      if (p.count > 0 || p.zero) return true;
    }
    return false;
  }
};

// A place in the ring of keys' and values' steps.  They lie there in the order in
// which the products need them: where both tiles take every step K0 V0 K1 V1 ...,
// where they take them in turn K0 K1 V0 K2 V1 K3 ...
struct Cursor {
  int at;
  uint32_t parity;
  __device__ __forceinline__ void next(int slots) {
    if (++at == slots) { at = 0; parity ^= 1u; }
  }
  __device__ __forceinline__ void skip(int n, int slots) {
    const int to = at + n;
    at = to % slots;
    parity ^= uint32_t(to / slots) & 1u;
  }
};

// kind::f8f6f4: e4m3 operands, fp32 accumulator.
__device__ __forceinline__ void mma8_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void mma8_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], %2, %3, p;\n\t}"
      :: "r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__host__ __device__ constexpr uint32_t idesc_e4m3(int M, int N, bool b_mn_major) {
  return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | (uint32_t(N >> 3) << 17) | (uint32_t(M >> 4) << 24);
}

template <int N> __device__ __forceinline__ void set_max_registers_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(N));
}
template <int N> __device__ __forceinline__ void set_max_registers_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(N));
}

// Row r of a unit's (query, query head): its place in q or out.
__device__ __forceinline__ int64_t row_offset(const Args& a, const int64_t (&s)[3], const Unit& u, int row) {
  const int query = row / a.group, h = u.head * a.group + (row - query * a.group);
  return u.b * s[0] + h * s[1] + query * s[2];
}

// A page's scales.  They are read a step before they are used, and the page's
// number (-1: all tokens of the page are masked) a step before that.
struct PageScale {
  float k;
  uint32_t v;
};
__device__ __forceinline__ int page_number(const Args& a, const Unit& u, int tokens, int64_t index) {
  if (index * kPage >= tokens) return -1;
  const int page = a.table[u.b * a.width + index];
  return page < 0 || page >= a.pages ? 0 : page;  // (reported where the page is loaded)
}
__device__ __forceinline__ PageScale page_scale(const Args& a, const Unit& u, int page) {
  // (masked: scores are -infinity whatever the scale, the values' is below any other)
  if (page < 0) return PageScale{1.f, 0x00800000u};
  const int64_t at = int64_t(page) * a.heads + u.head;
  return PageScale{a.k_scale[at], __float_as_uint(a.v_scale[at])};
}
// The exponent of a values' scale; NaN for NaN, and for what is no power of two (an error).
__device__ __forceinline__ float scale_log2(const Args& a, uint32_t v) {
  if (v >= 0x7F800000u || (v & 0x7FFFFFu) || v == 0) {
    if (v != 0x7FC00000u) atomicOr(a.err, PASA_DEVERR_BAD_SCALE);
    return __uint_as_float(0x7FC00000u);
  }
  return float(int(v >> 23) - 127);
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1) attention_kernel(const __grid_constant__ Maps maps,
                                                                const __grid_constant__ Args a) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* sm =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[kMaxSlots], empty[kMaxSlots], q_full[2], q_empty[2], o_free[2];
  __shared__ uint64_t s_full[2], p_full[2][2], pv_done[2];  // of a tile; p_full: of a page of a step
  __shared__ uint32_t tmem_slot;
  float* q_scale = reinterpret_cast<float*>(sm + kOffScale);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int both = a.both;
  constexpr int slots = kMaxSlots;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kMaxSlots; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full[t], kLoaders);
      mbar_init(&q_empty[t], 1 + 8);  // the last product that reads it, and the softmax warps (its scales)
      mbar_init(&o_free[t], 4);
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t][0], 4);
      mbar_init(&p_full[t][1], 4);
      mbar_init(&pv_done[t], 1);
    }
    fence_barrier_init();
  }
  if (warp == 1) { tmem_alloc(&tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  Walk walk(a, lane);
  Piece p;

  if (warp < 4 || warp >= 12) {
    set_max_registers_down<56>();
    if (warp == 0) {
      // ================= keys and values =================
      Cursor c{0, 1};
      int issued = 0;
      bool ok = true;
      while (ok && walk.next(a, lane, p)) {
        const int n = p.count, ahead = both ? 2 : 1;
        const int left = (request_tokens(a, p.u.b) + kPage - 1) / kPage - 2 * p.first;  // pages from the first step on
        const int32_t* row = a.table + p.u.b * a.width + 2 * p.first;
        int k_pages = 0, v_pages = 0;  // of 16 steps, a page a lane
        for (int jk = 0, jv = 0; jv < n && ok;) {
          // the next load: keys until they are `ahead` of the values, then in turn
          const bool values = jk >= min(n, jv + ahead);
          const int j = values ? jv++ : jk++;
          if ((j & 15) == 0) {
            int page = 2 * j + lane < left ? row[2 * j + lane] : 0;
            if (page < 0 || page >= a.pages) {
              if (2 * j + lane < 2 * n) atomicOr(a.err, PASA_DEVERR_BAD_PAGE);
              page = 0;
            }
            if (values) v_pages = page;
            else k_pages = page;
          }
          const int pages = values ? v_pages : k_pages, at = 2 * (j & 15);
          const int z0 = __shfl_sync(0xffffffffu, pages, at) * a.heads + p.u.head;
          const int z1 = __shfl_sync(0xffffffffu, pages, at + 1) * a.heads + p.u.head;
          const bool second = 2 * j + 1 < left;
          ok = __all_sync(0xffffffffu, mbar_wait_bounded(&empty[c.at], c.parity));
          if (!ok) break;
          if (elect_one()) {
            unsigned char* dst = sm + kOffRing + c.at * kSlotBytes;
            const CUtensorMap* map = values ? &maps.v : &maps.k;
            mbar_arrive_expect_tx(&full[c.at], second ? uint32_t(kSlotBytes) : uint32_t(kSlotBytes / 2));
            tma_load_3d(dst, map, &full[c.at], 0, 0, z0);
            if (second) tma_load_3d(dst + kSlotBytes / 2, map, &full[c.at], 0, 0, z1);
          }
          __syncwarp();
          ++issued;
          c.next(slots);
        }
      }
      if (!ok && lane == 0) report_operator_timeout(a.err);
      // the copies in flight land before the block can end
      for (int l = issued > slots ? issued - slots : 0; l < issued; ++l)
        mbar_wait_bounded(&full[l % slots], uint32_t((l / slots) & 1));
    } else if (warp == 1) {
      // ================= products =================
      // One elected lane waits and issues: a wait by the whole warp, its vote and a new election around every product
      // took 1000 clocks a product.
      constexpr uint32_t id_s = idesc_e4m3(128, kStep, false), id_o = idesc_e4m3(128, D, true);
      Cursor start{0, 0};
      int buf = 0;
      uint32_t q_parity = 0, p_parity = 0, o_parity = 3;  // p_parity, o_parity: bit t
      bool ok = true;
      const uint64_t desc = umma_desc_sw128(smem_u32(sm), 16, 1024);  // of the start of shared memory
      while (ok && walk.next(a, lane, p)) {
        if (p.count == 0) continue;
        const int n = p.count;
        const int last_valid = request_tokens(a, p.u.b) - (p.first + n - 1) * kStep;  // tokens of the last step
        const int tiles = both ? min(n, 2) : (p.u.block * 2 + 1) * kTile < a.rows ? 2 : 1;
        auto wait = [&](uint64_t* bar, uint32_t parity) {
          if (ok) ok = mbar_wait_bounded(bar, parity);
        };
        // scores of tile t with the keys in `slot`
        auto scores = [&](int t, int slot, bool frees_keys, bool frees_queries) {
          if (!ok) return;
          tc_fence_after();
          const uint64_t qd = desc + uint64_t((kOffQ + buf * kQBuf + (both ? 0 : t) * kQTile) >> 4);
          const uint64_t kd = desc + uint64_t((kOffRing + slot * kSlotBytes) >> 4);
          const uint32_t d = tmem + kColS + uint32_t(128 * t);
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int kk = 0; kk < D / 32; ++kk)
              mma8_ss(d, qd + uint64_t((x * kTile * 128 + kk * 32) >> 4), kd + uint64_t((kk * 32) >> 4), id_s,
                      x > 0 || kk > 0 ? 1u : 0u);
          tc_commit(&s_full[t]);
          if (frees_keys) tc_commit(&empty[slot]);
          if (frees_queries) tc_commit(&q_empty[buf]);
        };
        // output of tile t += probabilities times the values in `slot`, a page as soon as its probabilities are there
        auto output = [&](int t, int slot, bool first, bool frees_values) {
          if (first) {
            wait(&o_free[t], (o_parity >> t) & 1u);
            o_parity ^= 1u << t;
          }
          const uint64_t vd = desc + uint64_t((kOffRing + slot * kSlotBytes) >> 4);
          const uint32_t d = tmem + kColO + uint32_t(128 * t), pt = tmem + kColS + uint32_t(128 * t);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            wait(&p_full[t][h], (p_parity >> t) & 1u);
            if (!ok) return;
            tc_fence_after();
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
              for (int kk = 0; kk < 2; ++kk)
                mma8_ts(d, pt + uint32_t(x * 32 + h * 16 + kk * 8), vd + uint64_t((h * 8192 + kk * 4096) >> 4), id_o,
                        !first || h > 0 || x > 0 || kk > 0 ? 1u : 0u);
          }
          p_parity ^= 1u << t;
          tc_commit(&pv_done[t]);
          if (frees_values) tc_commit(&empty[slot]);
        };
        if (elect_one()) {
          Cursor c = start;
          wait(&q_full[buf], q_parity);
          // all but the last step's output
          if (both) {
            for (int j = 0; j < tiles; ++j, c.next(slots)) {
              wait(&full[c.at], c.parity);
              scores(j, c.at, true, j == n - 1);
            }
            for (int j = 0; j < n - 1 && ok; ++j) {
              wait(&full[c.at], c.parity);
              output(j & 1, c.at, j < 2, true);
              c.next(slots);
              if (j + 2 < n) {
                wait(&full[c.at], c.parity);
                scores(j & 1, c.at, true, j + 2 == n - 1);
                c.next(slots);
              }
            }
          } else {
            wait(&full[c.at], c.parity);
            for (int t = 0; t < tiles; ++t) scores(t, c.at, t == tiles - 1, n == 1 && t == tiles - 1);
            c.next(slots);
            for (int j = 0; j < n - 1 && ok; ++j) {
              const int values = c.at;
              wait(&full[c.at], c.parity);
              c.next(slots);
              output(0, values, j == 0, tiles == 1);
              wait(&full[c.at], c.parity);
              scores(0, c.at, tiles == 1, tiles == 1 && j == n - 2);
              if (tiles == 2) {
                output(1, values, j == 0, true);
                scores(1, c.at, true, j == n - 2);
              }
              c.next(slots);
            }
          }
        }
        __syncwarp();
        start.skip(2 * n - 1, slots);
        if (last_valid < kStep) {
          // what lies behind the last token is no value: it may be a NaN's bits, and 0 * NaN is NaN
          mbar_wait_bounded(&full[start.at], start.parity);
          unsigned char* vs = sm + kOffRing + start.at * kSlotBytes;
          for (int i = lane; i < (kStep - last_valid) * 8; i += 32)
            *reinterpret_cast<uint4*>(vs + last_valid * 128 + i * 16) = make_uint4(0u, 0u, 0u, 0u);
          fence_proxy_async();
          __syncwarp();
        }
        if (elect_one()) {
          wait(&full[start.at], start.parity);
          if (both) {
            output((n - 1) & 1, start.at, n <= 2, true);
          } else {
            for (int t = 0; t < tiles; ++t) output(t, start.at, n == 1, t == tiles - 1);
          }
        }
        ok = __all_sync(0xffffffffu, ok);  // the elected lane's, the others' is true
        start.skip(1, slots);
        if ((buf ^= 1) == 0) q_parity ^= 1u;
      }
      if (!ok && lane == 0) report_operator_timeout(a.err);
    } else {
      // ================= queries =================
      // four lanes a row, eight rows a warp: the row's largest value, its scale, hi and lo
      const int loader = warp < 4 ? warp - 2 : warp - 10;
      const int sub = lane >> 2, part = lane & 3;
      constexpr int kVecs = D / 32;  // 16-byte vectors of a lane: part + 4 i
      int buf = 0;
      uint32_t parity = 1;
      bool ok = true;
      while (ok && walk.next(a, lane, p)) {
        if (p.count == 0) continue;
        const int r0 = p.u.block * 2 * kTile, live = min(a.rows - r0, both ? kTile : 2 * kTile);
        unsigned char* qs = sm + kOffQ + buf * kQBuf;
        Bf8 v[kVecs];
        auto load = [&](int row) {
          if (row >= live) return;
          const __nv_bfloat16* src = a.q + row_offset(a, a.qs, p.u, r0 + row) + part * 8;
#pragma unroll
          for (int i = 0; i < kVecs; ++i) v[i].r = *reinterpret_cast<const uint4*>(src + 32 * i);
        };
        load(loader * 8 + sub);  // the first rows are on their way while the buffer is still in use
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(&q_empty[buf], parity));
        if (!ok) break;
        for (int row8 = loader * 8; row8 < live; row8 += kLoaders * 8) {
          const int row = row8 + sub;
          uint4 now[kVecs];
          uint32_t amax = 0;
#pragma unroll
          for (int i = 0; i < kVecs; ++i) {
            now[i] = v[i].r;
            amax = max(amax, v[i].amax());
          }
          load(row + kLoaders * 8);
          amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
          amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
          if (row >= live) continue;  // (what the rows behind the last hold makes only rows that are not kept)
          const float scale = scale_of(amax), inv = inverse(scale);
          unsigned char* at = qs + (row / kTile) * kQTile + (row % kTile) * 128;
#pragma unroll
          for (int i = 0; i < kVecs; ++i) {
            const uint32_t in[4] = {now[i].x, now[i].y, now[i].z, now[i].w};
            uint16_t hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {  // exact in fp16: 8 significant bits, 448 at most
              const __half2 x = __floats2half2_rn(__uint_as_float(in[e] << 16) * inv,
                                                  __uint_as_float(in[e] & 0xFFFF0000u) * inv);
              hi[e] = f16x2_to_e4m3x2(*reinterpret_cast<const uint32_t*>(&x));
              const uint32_t h = e4m3x2_to_f16x2(hi[e]);
              const __half2 rest = __hsub2(x, *reinterpret_cast<const __half2*>(&h));
              lo[e] = f16x2_to_e4m3x2(*reinterpret_cast<const uint32_t*>(&rest));
            }
            // byte c of the row, 16-byte pieces swizzled by the row
            const int c = part * 8 + 32 * i;
            unsigned char* dst = at + (((c >> 4) ^ (row & 7)) << 4) + (c & 15);
            *reinterpret_cast<uint2*>(dst) =
                make_uint2(uint32_t(hi[0]) | uint32_t(hi[1]) << 16, uint32_t(hi[2]) | uint32_t(hi[3]) << 16);
            *reinterpret_cast<uint2*>(dst + kTile * 128) =
                make_uint2(uint32_t(lo[0]) | uint32_t(lo[1]) << 16, uint32_t(lo[2]) | uint32_t(lo[3]) << 16);
          }
          if (part == 0) q_scale[buf * 2 * kTile + row] = scale;
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[buf]);
        if ((buf ^= 1) == 0) parity ^= 1u;
      }
      if (!ok && lane == 0) report_operator_timeout(a.err);
    }
  } else {
    set_max_registers_up<200>();
    // ================= softmax of tile t: a thread a row =================
    const int t = (warp - 4) >> 2, w = warp & 3, row = w * 32 + lane;
    const uint32_t lanes = uint32_t(w * 32) << 16;
    const uint32_t s_tmem = tmem + lanes + kColS + 128u * uint32_t(t), o_tmem = tmem + lanes + kColO + 128u * uint32_t(t);
    int buf = 0;
    uint32_t q_parity = 0, k_parity = 0;  // k_parity: of the tile's next step
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      if (ok && !mbar_wait_bounded(bar, parity)) {
        ok = false;
        report_operator_timeout(a.err);
      }
    };
    while (walk.next(a, lane, p)) {
      const int r0 = p.u.block * 2 * kTile + (both ? 0 : t * kTile);
      const int r = r0 + row;  // the row of the key/value head
      const bool live = r < a.rows, warp_live = r0 + w * 32 < a.rows;
      if (p.zero) {
        if (live && !(both && t == 1)) {
          __nv_bfloat16* out = a.out + row_offset(a, a.os, p.u, r);
#pragma unroll
          for (int c = 0; c < D; c += 8) *reinterpret_cast<uint4*>(out + c) = make_uint4(0u, 0u, 0u, 0u);
        }
        continue;
      }
      const int n = p.count, tokens = request_tokens(a, p.u.b);
      const int tiles = both ? min(n, 2) : (p.u.block * 2 + 1) * kTile < a.rows ? 2 : 1;
      wait(&q_full[buf], q_parity);
      const float q_row = q_scale[buf * 2 * kTile + (both ? 0 : t * kTile) + row] * a.scale_log2;
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_empty[buf]);
      if ((buf ^= 1) == 0) q_parity ^= 1u;
      // References (log2): m of the probabilities in the denominator l, v_ref of the values' scales; the output's is
      // m + v_ref.  They are a row's own.
      float m = -INFINITY, l = 0.f, v_ref = 0.f;
      const int stride = both ? 2 : 1, begin = both ? t : 0;
      if (t < tiles) {
        PageScale next[2];
        int number[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          next[h] = page_scale(a, p.u, page_number(a, p.u, tokens, int64_t(p.first + begin) * 2 + h));
          number[h] = page_number(a, p.u, tokens, int64_t(p.first + begin + stride) * 2 + h);
        }
        for (int j = begin; j < n; j += stride, k_parity ^= 1u) {
          const PageScale page[2] = {next[0], next[1]};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            next[h] = page_scale(a, p.u, number[h]);
            number[h] = page_number(a, p.u, tokens, int64_t(p.first + j + 2 * stride) * 2 + h);
          }
          wait(&s_full[t], k_parity);
          if (!warp_live) {  // (its rows' probabilities are whatever the scores' bits are: they make rows not kept)
            __syncwarp();  // a lane still in its wait could miss the phase that lane 0's arrivals let begin
            if (lane == 0) {
              mbar_arrive(&p_full[t][0]);
              mbar_arrive(&p_full[t][1]);
            }
            continue;
          }
          tc_fence_after();
          uint32_t s[4][32];
#pragma unroll
          for (int i = 0; i < 4; ++i) tmem_ld32(s_tmem + 32u * uint32_t(i), s[i]);
          float c[2], v_log2[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            c[h] = q_row * page[h].k;
            if (c[h] < 1e-37f) c[h] = 1e-37f;  // -infinity times it stays that; a NaN stays NaN
            v_log2[h] = scale_log2(a, page[h].v);
          }
          tmem_wait_ld();
          const int valid = tokens - (p.first + j) * kStep;
          if (valid < kStep) {
#pragma unroll
            for (int i = 0; i < 128; ++i)
              if (i >= valid) s[i >> 5][i & 31] = 0xFF800000u;
          }
          const float top0 = fmaxf(max_tree32(s[0]), max_tree32(s[1])) * c[0];
          const float top1 = fmaxf(max_tree32(s[2]), max_tree32(s[3])) * c[1];
          const float top = fmaxf(top0, top1), v_top = fmaxf(top0 + v_log2[0], top1 + v_log2[1]);
          // the references move when a probability, or one times its value's scale, is more than 2^4 above them
          const bool moves = top > m + kRescale || v_top > m + v_ref + kRescale;
          if (__any_sync(0xffffffffu, moves)) {
            const float m_new = moves ? fmaxf(m, top) : m;
            const float v_new = moves ? (j > begin ? fmaxf(m + v_ref, v_top) : v_top) - m_new : v_ref;
            if (j > begin) {
              const float fall = exp2_ftz(fmaxf(m - m_new, -200.f));
              const float factor = exp2_ftz(fmaxf((m + v_ref) - (m_new + v_new), -200.f));
              wait(&pv_done[t], k_parity ^ 1u);
              tc_fence_after();
#pragma unroll 1
              for (int i = 0; i < D / 32; ++i) {
                uint32_t o[32];
                tmem_ld32(o_tmem + 32u * uint32_t(i), o);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * factor);
                tmem_st32(o_tmem + 32u * uint32_t(i), o);
              }
              l *= fall;
            }
            m = m_new;
            v_ref = v_new;
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            // probabilities times the page's value scale over the reference; times 2^-60 at the least, which is nothing
            // next to what set the reference
            const float dv = v_log2[h] == v_log2[h] ? fmaxf(v_log2[h] - v_ref, -60.f) : v_log2[h];
            const float shift = dv + kLog2P - (m == -INFINITY ? 0.f : m);
            const float2 mul = make_float2(c[h], c[h]), add = make_float2(shift, shift);
            float2 sum0 = make_float2(0.f, 0.f), sum1 = make_float2(0.f, 0.f);
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              uint32_t hi[8], lo[8];
#pragma unroll
              for (int e = 0; e < 32; e += 4) {
                const uint32_t* x = &s[2 * h + g][e];
                float2 x01 = __ffma2_rn(make_float2(__uint_as_float(x[0]), __uint_as_float(x[1])), mul, add);
                float2 x23 = __ffma2_rn(make_float2(__uint_as_float(x[2]), __uint_as_float(x[3])), mul, add);
                x01.x = exp2_ftz(x01.x); x01.y = exp2_ftz(x01.y);
                x23.x = exp2_ftz(x23.x); x23.y = exp2_ftz(x23.y);
                sum0 = __fadd2_rn(sum0, x01);
                sum1 = __fadd2_rn(sum1, x23);
                const __half2 p01 = __floats2half2_rn(x01.x, x01.y), p23 = __floats2half2_rn(x23.x, x23.y);
                const uint16_t h01 = f16x2_to_e4m3x2(*reinterpret_cast<const uint32_t*>(&p01));
                const uint16_t h23 = f16x2_to_e4m3x2(*reinterpret_cast<const uint32_t*>(&p23));
                const uint32_t b01 = e4m3x2_to_f16x2(h01), b23 = e4m3x2_to_f16x2(h23);
                const __half2 l01 = __hsub2(p01, *reinterpret_cast<const __half2*>(&b01));
                const __half2 l23 = __hsub2(p23, *reinterpret_cast<const __half2*>(&b23));
                hi[e >> 2] = uint32_t(h01) | uint32_t(h23) << 16;
                lo[e >> 2] = uint32_t(f16x2_to_e4m3x2(*reinterpret_cast<const uint32_t*>(&l01))) |
                             uint32_t(f16x2_to_e4m3x2(*reinterpret_cast<const uint32_t*>(&l23))) << 16;
              }
              tmem_st8(s_tmem + uint32_t(16 * h + 8 * g), hi);
              tmem_st8(s_tmem + uint32_t(32 + 16 * h + 8 * g), lo);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[t][h]);
            l += ((sum0.x + sum0.y) + (sum1.x + sum1.y)) * exp2_ftz(-dv - kLog2P);
          }
        }
        wait(&pv_done[t], k_parity ^ 1u);  // the last step's output
        tc_fence_after();
      }
      const float to_true = exp2f(v_ref - kLog2P);  // the accumulator's unit
      if (!p.whole) {
        // a part of the unit: sums, maximum and denominator for the second kernel
        const int64_t at = (int64_t(blockIdx.x) * 2 + p.part) * 2 * kTile + t * kTile + row;
        if (live) a.part_ml[at] = make_float2(m, l);
        if (t < tiles) {
          float4* dst = reinterpret_cast<float4*>(a.part_o + at * D);
#pragma unroll 1
          for (int i = 0; i < D / 16; ++i) {
            uint32_t o[16];
            __syncwarp();
            tmem_ld16(o_tmem + 16u * uint32_t(i), o);
            tmem_wait_ld();
            if (live) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                dst[4 * i + e] = make_float4(__uint_as_float(o[4 * e]) * to_true, __uint_as_float(o[4 * e + 1]) * to_true,
                                             __uint_as_float(o[4 * e + 2]) * to_true,
                                             __uint_as_float(o[4 * e + 3]) * to_true);
            }
          }
        }
      } else if (both && tiles == 2) {
        // both tiles have the same rows: tile 1 hands its sums over through shared memory, 32 columns at a time (the
        // space of a second tile of queries, and of its scales in either buffer)
        float4* xch = reinterpret_cast<float4*>(sm + kOffQ + kQTile);
        float* xch_ml = q_scale + kTile;
        if (t == 1) {
          xch_ml[row] = m;
          xch_ml[2 * kTile + row] = l;
        }
        __nv_bfloat16* out = a.out + row_offset(a, a.os, p.u, live ? r : 0);
        float f0 = 0.f, f1 = 0.f;
#pragma unroll 1
        for (int i = 0; i < D / 32; ++i) {
          uint32_t o[32];
          __syncwarp();
          tmem_ld32(o_tmem + 32u * uint32_t(i), o);
          tmem_wait_ld();
          if (t == 1) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              xch[e * kTile + row] = make_float4(__uint_as_float(o[4 * e]) * to_true, __uint_as_float(o[4 * e + 1]) * to_true,
                                                 __uint_as_float(o[4 * e + 2]) * to_true,
                                                 __uint_as_float(o[4 * e + 3]) * to_true);
          }
          named_bar_sync(1, 256);
          if (t == 0) {
            if (i == 0) {
              const float m1 = xch_ml[row], l1 = xch_ml[2 * kTile + row], top = fmaxf(m, m1);
              const float e0 = exp2_ftz(fmaxf(m - top, -200.f)), e1 = exp2_ftz(fmaxf(m1 - top, -200.f));
              const float inv = 1.f / (l * e0 + l1 * e1);
              f0 = to_true * e0 * inv;
              f1 = e1 * inv;
            }
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              const float4 u0 = xch[(2 * v) * kTile + row], u1 = xch[(2 * v + 1) * kTile + row];
              const uint32_t* x = &o[8 * v];
              const uint4 y = make_uint4(
                  pack_bf16x2(fmaf(u0.x, f1, __uint_as_float(x[0]) * f0), fmaf(u0.y, f1, __uint_as_float(x[1]) * f0)),
                  pack_bf16x2(fmaf(u0.z, f1, __uint_as_float(x[2]) * f0), fmaf(u0.w, f1, __uint_as_float(x[3]) * f0)),
                  pack_bf16x2(fmaf(u1.x, f1, __uint_as_float(x[4]) * f0), fmaf(u1.y, f1, __uint_as_float(x[5]) * f0)),
                  pack_bf16x2(fmaf(u1.z, f1, __uint_as_float(x[6]) * f0), fmaf(u1.w, f1, __uint_as_float(x[7]) * f0)));
              if (live) *reinterpret_cast<uint4*>(out + 32 * i + 8 * v) = y;
            }
          }
          named_bar_sync(2, 256);  // the space may be written again
        }
      } else if (t < tiles) {
        // through shared memory, 32 columns at a time: 4 lanes then write 64 bytes of a row
        const float f = to_true / l;
        unsigned char* stage = sm + kOffOut + (warp - 4) * 2048;
        int64_t at[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int rr = r0 + w * 32 + x * 8 + (lane >> 2);
          at[x] = rr < a.rows ? row_offset(a, a.os, p.u, rr) + (lane & 3) * 8 : -1;
        }
#pragma unroll 1
        for (int i = 0; i < D / 32; ++i) {
          uint32_t o[32];
          __syncwarp();
          tmem_ld32(o_tmem + 32u * uint32_t(i), o);
          tmem_wait_ld();
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const uint32_t* x = &o[8 * v];
            *reinterpret_cast<uint4*>(stage + lane * 64 + ((v ^ ((lane >> 1) & 3)) << 4)) =
                make_uint4(pack_bf16x2(__uint_as_float(x[0]) * f, __uint_as_float(x[1]) * f),
                           pack_bf16x2(__uint_as_float(x[2]) * f, __uint_as_float(x[3]) * f),
                           pack_bf16x2(__uint_as_float(x[4]) * f, __uint_as_float(x[5]) * f),
                           pack_bf16x2(__uint_as_float(x[6]) * f, __uint_as_float(x[7]) * f));
          }
          __syncwarp();
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int rr = x * 8 + (lane >> 2);
            const uint4 y = *reinterpret_cast<const uint4*>(stage + rr * 64 + (((lane & 3) ^ ((rr >> 1) & 3)) << 4));
            if (at[x] >= 0) *reinterpret_cast<uint4*>(a.out + at[x] + 32 * i) = y;
          }
        }
      }
      if (t < tiles) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_free[t]);
      }
    }
  }
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// Joins the parts of a unit that was cut.  Block (c, y): the unit that begins in
// CTA c's part of the line and goes on in the next; a warp a row.
template <int D>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ Args a, int parts) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  wait_for_predecessor();
  const int64_t total = total_ticks(a, lane);
  const int64_t cut = part_begin(total, int(blockIdx.x) + 1, parts);
  if (cut >= total) return;
  const Unit u = find_unit(a, cut, lane);
  // the unit's steps before the cut: some, and all of them CTA c's
  if (cut - u.begin <= kOverhead || part_begin(total, int(blockIdx.x), parts) > u.begin + kOverhead) return;
  const int row = int(blockIdx.y) * 8 + warp, r = u.block * 2 * kTile + row;
  if (r >= a.rows || (a.both && row >= kTile)) return;
  constexpr int kCols = D / 32;
  float o[kCols] = {}, m = -INFINITY, l = 0.f;
  const int64_t end = u.begin + kOverhead + u.steps;
  for (int c = int(blockIdx.x); c < parts; ++c) {
    const int64_t begin = part_begin(total, c, parts), stop = part_begin(total, c + 1, parts);
    if (begin >= end) break;
    const int64_t first = max(begin - u.begin - kOverhead, int64_t(0));
    if (min(stop, end) - u.begin - kOverhead <= first) continue;  // none of the unit's steps
    const int part = begin >= u.begin ? 0 : 1;
    for (int t = 0; t < (a.both ? 2 : 1); ++t) {
      const int64_t at = (int64_t(c) * 2 + part) * 2 * kTile + t * kTile + row;
      const float2 ml = a.part_ml[at];
      if (ml.x == -INFINITY && ml.y == 0.f) continue;  // a tile without steps
      const float top = fmaxf(m, ml.x);
      const float e0 = m == -INFINITY ? 0.f : exp2f(m - top), e1 = exp2f(ml.x - top);
#pragma unroll
      for (int i = 0; i < kCols; ++i) o[i] = o[i] * e0 + a.part_o[at * D + lane * kCols + i] * e1;
      l = l * e0 + ml.y * e1;
      m = top;
    }
  }
  __nv_bfloat16* out = a.out + row_offset(a, a.os, u, r) + lane * kCols;
  const float inv = 1.f / l;
#pragma unroll
  for (int i = 0; i < kCols; i += 2) *reinterpret_cast<uint32_t*>(out + i) = pack_bf16x2(o[i] * inv, o[i + 1] * inv);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
// e4m3 [pages * heads][64][dim]; a box is a page of one head, its rows 128 bytes
// apart in shared memory (dim 64: the rest of a row is filled with zeros).
bool make_page_map(CUtensorMap* m, const void* base, int64_t pages, int heads, int dim) {
  const auto fn = tensor_map_encoder();
  if (!fn) return false;
  const cuuint64_t dims[3] = {cuuint64_t(dim), cuuint64_t(kPage), cuuint64_t(pages * heads)};
  const cuuint64_t strides[2] = {cuuint64_t(dim), cuuint64_t(dim) * kPage};
  const cuuint32_t box[3] = {128u, cuuint32_t(kPage), 1u};
  const cuuint32_t step[3] = {1u, 1u, 1u};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, step,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

int check_cache(const void* k, const void* v, const float* ks, const float* vs, int64_t pages, int64_t heads, int dim,
                const int32_t* table, int64_t width, int64_t batch) {
  if (dim != 64 && dim != 128) return PASA_ERR_UNSUPPORTED;
  if (pages < 0 || heads < 1 || heads > 32767 || width < 0 || batch < 0 || batch > 65535) return PASA_ERR_SHAPE;
  if (pages * heads > INT32_MAX || width > INT32_MAX / kPage) return PASA_ERR_SHAPE;
  if (pages && (!k || !v || !ks || !vs)) return PASA_ERR_NULL;
  if (batch && width && !table) return PASA_ERR_NULL;
  return misaligned(k) || misaligned(v) ? PASA_ERR_ALIGN : PASA_OK;
}

int check_rows(const void* x, const int64_t* stride) {
  if (!x || !stride) return PASA_ERR_NULL;
  if (misaligned(x)) return PASA_ERR_ALIGN;
  for (int i = 0; i < 3; ++i)
    if (stride[i] % 8) return PASA_ERR_ALIGN;
  return PASA_OK;
}

int device_sms(int* sms) {
  int dev = 0, major = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess ||
      cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return PASA_ERR_CUDA;
  return major == 10 ? PASA_OK : PASA_ERR_DEVICE;
}

size_t part_bytes(int sms, int dim) { return size_t(sms) * 2 * 2 * kTile * (size_t(dim) * 4 + sizeof(float2)); }

template <int D>
cudaError_t launch_attention(cudaStream_t st, const Maps& maps, const Args& a, int sms) {
  cudaError_t e = cudaFuncSetAttribute(attention_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) return e;
  attention_kernel<D><<<unsigned(sms), kThreads, kSmem, st>>>(maps, a);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const int rows = a.rows < 2 * kTile ? a.rows : 2 * kTile;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(sms - 1), unsigned(cdiv(rows, 8)));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, join_kernel<D>, a, sms);
}

}  // namespace kv8
}  // namespace pasa

using namespace pasa;

extern "C" {

int pasa_kv8_write(void* stream, const void* k, const int64_t* k_stride, const void* v, const int64_t* v_stride,
                   void* k_cache, void* v_cache, float* k_scale, float* v_scale, int64_t pages, int64_t heads, int dim,
                   const int32_t* table, int64_t width, const int32_t* starts, const int32_t* counts, int64_t batch,
                   int64_t tokens) {
  using namespace pasa::kv8;
  int st = check_cache(k_cache, v_cache, k_scale, v_scale, pages, heads, dim, table, width, batch);
  if (st) return st;
  if (tokens < 0 || tokens > INT32_MAX - kPage) return PASA_ERR_SHAPE;
  if (batch == 0 || tokens == 0) return PASA_OK;
  if ((st = check_rows(k, k_stride)) || (st = check_rows(v, v_stride))) return st;
  if (!starts) return PASA_ERR_NULL;
  int sms = 0;
  if ((st = device_sms(&sms))) return st;
  WriteArgs a{};
  a.x[0] = static_cast<const __nv_bfloat16*>(k);
  a.x[1] = static_cast<const __nv_bfloat16*>(v);
  for (int i = 0; i < 3; ++i) {
    a.xs[0][i] = k_stride[i];
    a.xs[1][i] = v_stride[i];
  }
  a.cache[0] = static_cast<uint8_t*>(k_cache);
  a.cache[1] = static_cast<uint8_t*>(v_cache);
  a.scale[0] = k_scale;
  a.scale[1] = v_scale;
  a.table = table;
  a.starts = starts;
  a.counts = counts;
  a.pages = pages;
  a.width = width;
  a.tokens = tokens;
  a.heads = int(heads);
  a.err = operator_error_word();
  if (!a.err) return PASA_ERR_CUDA;
  const dim3 grid(unsigned(cdiv(tokens + kPage - 1, kPage)), unsigned(2 * heads), unsigned(batch));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dim == 64) write_kernel<64><<<grid, kWriteThreads, 0, s>>>(a);
  else write_kernel<128><<<grid, kWriteThreads, 0, s>>>(a);
  return cudaGetLastError() == cudaSuccess ? PASA_OK : PASA_ERR_CUDA;
}

int pasa_kv8_attention_workspace_size(int dim, size_t* bytes) {
  if (!bytes) return PASA_ERR_NULL;
  if (dim != 64 && dim != 128) return PASA_ERR_UNSUPPORTED;
  int sms = 0;
  const int st = kv8::device_sms(&sms);
  if (st) return st;
  *bytes = kv8::part_bytes(sms, dim);
  return PASA_OK;
}

int pasa_kv8_attention(void* stream, const void* q, const int64_t* q_stride, const void* k_cache, const void* v_cache,
                       const float* k_scale, const float* v_scale, int64_t pages, int64_t heads, int dim,
                       const int32_t* table, int64_t width, const int32_t* lengths, int64_t batch, int64_t queries,
                       int64_t group, float scale, void* out, const int64_t* out_stride, void* workspace,
                       size_t workspace_bytes) {
  using namespace pasa::kv8;
  int st = check_cache(k_cache, v_cache, k_scale, v_scale, pages, heads, dim, table, width, batch);
  if (st) return st;
  if (queries < 0 || group < 1 || queries > (1 << 30) / group || heads * group > INT32_MAX) return PASA_ERR_SHAPE;
  if (!(scale > 0.f) || !(scale <= 3.0e38f)) return PASA_ERR_SHAPE;
  if (batch == 0 || queries == 0) return PASA_OK;
  if ((st = check_rows(q, q_stride)) || (st = check_rows(out, out_stride))) return st;
  if (!lengths) return PASA_ERR_NULL;
  if (!workspace) return PASA_ERR_WORKSPACE;
  if (misaligned(workspace)) return PASA_ERR_ALIGN;
  int sms = 0;
  if ((st = device_sms(&sms))) return st;
  if (workspace_bytes < part_bytes(sms, dim)) return PASA_ERR_WORKSPACE;
  Maps maps;
  Args a{};
  a.err = operator_error_word();
  if (!a.err) return PASA_ERR_CUDA;
  // (without pages no request has tokens: the maps are not used)
  const void* some = pages ? k_cache : workspace;
  if (!make_page_map(&maps.k, some, pages ? pages : 1, int(heads), dim) ||
      !make_page_map(&maps.v, pages ? v_cache : workspace, pages ? pages : 1, int(heads), dim))
    return PASA_ERR_CUDA;
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.out = static_cast<__nv_bfloat16*>(out);
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = q_stride[i];
    a.os[i] = out_stride[i];
  }
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.table = table;
  a.lengths = lengths;
  a.pages = pages;
  a.width = pages ? width : 0;
  a.batch = int(batch);
  a.heads = int(heads);
  a.group = int(group);
  a.rows = int(queries * group);
  a.blocks = int(cdiv(a.rows, 2 * kTile));
  a.both = a.rows <= kTile ? 1 : 0;
  a.scale_log2 = scale * kLog2e;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + size_t(sms) * 2 * 2 * kTile * size_t(dim));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dim == 64 ? launch_attention<64>(s, maps, a, sms) : launch_attention<128>(s, maps, a, sms);
  return e == cudaSuccess ? PASA_OK : PASA_ERR_CUDA;
}

}  // extern "C"
