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
//              rounded again to it.  Reads 2 bytes and writes 1 a value; a block has
//              a page and head and waits for its maximum before it writes, which is
//              what bounds it (4680 tokens, 12 heads of 128, 43 MB: 12 us, 3.6 TB/s;
//              one token of 8 requests, 8 heads: 4.2 us).
//   attention  out = softmax(q k^T scale) v over a request's first `length`
//              tokens.  Bound: the tensor cores for many queries, HBM (one byte a
//              value) for single tokens.
//
// Attention on the tensor cores (tcgen05).  The scores' products run on the pages
// as they are: a bf16 value has 8 significant bits and an e4m3 value 4, so a query
// goes in as two e4m3 terms, q = s (hi + lo) (s: a power of two for each row), exact
// for a row's elements down to 2^-9 of its largest and 2^-17 of the largest off
// below.  The two terms take the time of one bf16 product (e4m3 has twice its rate)
// and read 8-bit keys from shared memory.  The probabilities' products run in fp16:
// four warps widen the values once, which is exact, and a probability is held times
// 2^11 over a reference that lags the maximum by up to 2^4.  So it keeps 11
// significant bits, or 2^-36 of the largest, and a long tail far below one key
// weighs what the denominator says.  (As two e4m3 terms, which end at 2^-14 of the
// largest, half of such a tail of 18720 tokens was lost.)  Scores, maxima, sums and
// the output are fp32.
//
// Work split.  A unit is a request, a key/value head and 256 of the rows
// (query, query head of the group) that attend with it; its cost is its steps of
// 128 tokens and an overhead.  The line of all units is cut into equal parts, one
// for each of the GPU's SMs, so neither the number of units nor their lengths
// leave SMs idle; a unit that is cut leaves its parts (fp32 sums, maximum and
// denominator) in the workspace, and a second kernel joins them in order.  With
// at most 128 rows the two tiles of a unit hold the same rows and take the steps
// in turn, which hides the one's softmax behind the other's products.  With at
// most 32 rows (single tokens) each of a tile's four warps has those rows and a
// quarter of a step's tokens as well, and the rings of keys and values are longer.
//
// What bounds it (12 heads, 4680 queries over 18720 tokens, D = 128: 530 us, 1.01
// PFLOP/s): a step of a pair of tiles takes some 4000 clocks, of which the products
// take 2100 and 2^x 2050.  They overlap between the two tiles only, since scores,
// probabilities and outputs of two tiles fill TMEM; 64-token steps with two places
// for scores made the products the bound (one of N = 64 takes as long as one of
// N = 128).  Units of few steps (40 heads, 32760 queries over 512 and 77 tokens:
// 840 us) wait for their queries, whose copying and splitting takes 15000 clocks a
// buffer.  Single tokens (8 requests of 130 to 32767 tokens, 8 heads of 128, 333 MB
// of pages: 103 us) wait for the chain scores, softmax, output of two tiles, some
// 2700 clocks a step; widening the values is 14 us of it, and the rings' lengths
// make no difference.
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
constexpr int kKeyBytes = kStep * 128;   // a step's keys
constexpr int kRawBytes = kPage * 128;   // a page's values as they lie in the cache
constexpr int kWideBytes = kPage * 256;  // in fp16: for every 64 dimensions the tokens' rows of 128 bytes
// Places of the three rings; the second number where both tiles have the same rows.
constexpr int key_slots(bool both) { return both ? 4 : 2; }
constexpr int raw_slots(bool both) { return both ? 5 : 2; }
constexpr int wide_slots(bool both) { return both ? 2 : 2; }
constexpr int kMaxSlots = 5;
constexpr int kScaleSteps = 8;      // ring of the steps' scales: a step's stay until both its products are done
constexpr int kQTile = 2 * kTile * 128;  // hi, lo
constexpr int kQBuf = 2 * kQTile;   // two tiles
constexpr int kThreads = 640;       // 0 TMA, 1 MMA + TMEM, 2-3 and 12-15 queries, 4-7 and 8-11 softmax, 16-19 values
constexpr int kLoaders = 6;
constexpr int kWideners = 4;
constexpr int kRegisters = 96, kRegistersSoftmax = 128, kRegistersQueries = 88, kRegistersValues = 48;  // of a thread
static_assert(2 * kRegistersSoftmax + 2 * kRegistersQueries + kRegistersValues <= kThreads / 128 * kRegisters,
              "the warpgroups share what the block was launched with");
constexpr float kLog2P = 11.f;      // probabilities are held times 2^11 ...
constexpr float kRescale = 4.f;     // ... and their reference lags the maximum by up to 2^4: at most 2^15, fp16 ends at 2^16
constexpr int kOffQ = 0;            // [2 buffers][2 tiles][hi, lo][128 rows][128 bytes], then the rings and the output
constexpr int out_bytes(bool both) { return both ? 16384 : 8192; }  // on its way
constexpr int off_keys(bool both) { return 2 * (both ? kQTile : kQBuf); }
constexpr int off_raw(bool both) { return off_keys(both) + key_slots(both) * kKeyBytes; }
constexpr int off_wide(bool both) { return off_raw(both) + raw_slots(both) * kRawBytes; }
constexpr int off_out(bool both) { return off_wide(both) + wide_slots(both) * kWideBytes; }
constexpr int kOffScale = off_out(true) + out_bytes(true);  // f32 [2 buffers][256 rows]: the queries' scales
static_assert(off_out(false) + out_bytes(false) == kOffScale, "both layouts end there");
constexpr int kSmem = kOffScale + 2 * 2 * kTile * 4 + 1024;
// Tile t: scores at kColS + 128 t, over them the probabilities (of 32 tokens: in the
// first 16 columns of their scores); output at kColO + 128 t.
constexpr uint32_t kColS = 0, kColO = 256;
static_assert(kSmem + 4096 <= 232448, "shared memory budget");

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
  uint32_t group_magic;        // 2^32 / group + 1, rounded down; 0 for 1
  int rows, blocks;            // rows of a key/value head (queries x group); units of 256 of them
  int overhead;                // steps' time that a unit takes besides its steps
  int quarters;                // 1: the 4 warps of a tile have the same rows, each with a quarter of a step's tokens
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

// Ticks of the line of all units: a unit takes a.overhead and its steps.  All lanes.
__device__ __forceinline__ int64_t total_ticks(const Args& a, int lane) {
  int64_t sum = 0;
  for (int b = lane; b < a.batch; b += 32) sum += request_steps(a, b) + a.overhead;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  return sum * a.heads * a.blocks;
}
// The line's parts: part c is [begin(c), begin(c + 1)).
struct Parts {
  int64_t total, each;
  int rest, parts;
  __device__ __forceinline__ Parts(int64_t total_, int parts_) : total(total_), each(total_ / parts_), parts(parts_) {
    rest = int(total_ - each * parts_);
  }
  __device__ __forceinline__ int64_t begin(int c) const { return each * c + unsigned(rest * c) / unsigned(parts); }
};

struct Unit {
  int b, head, block;
  int tokens, steps;  // of the request
  int64_t begin;   // first tick
};

// The unit that holds a tick.  All lanes.
__device__ __forceinline__ Unit find_unit(const Args& a, int64_t tick, int lane) {
  const int64_t units = int64_t(a.heads) * a.blocks;
  int64_t before = 0;
  for (int b0 = 0;; b0 += 32) {
    const int b = b0 + lane;
    const int tokens = b < a.batch ? request_tokens(a, b) : 0, steps = (tokens + kStep - 1) / kStep;
    const int64_t own = b < a.batch ? (steps + a.overhead) * units : 0;
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
      u.tokens = __shfl_sync(0xffffffffu, tokens, src);
      u.steps = (u.tokens + kStep - 1) / kStep;
      const int64_t first = before + __shfl_sync(0xffffffffu, upto - own, src);
      const int64_t index = (tick - first) / (u.steps + a.overhead);
      u.begin = first + index * (u.steps + a.overhead);
      u.block = int(index / a.heads);
      u.head = int(index % a.heads);
      return u;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
    if (b0 + 32 >= a.batch) return Unit{0, 0, 0, 0, 0, before};  // (no unit: a tick behind the last)
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

// Goes through a CTA's part of the line of units.
struct Walk {
  int64_t at, begin, end;
  Unit u;
  __device__ __forceinline__ Walk(const Args& a, int lane) {
    const Parts line(total_ticks(a, lane), int(gridDim.x));
    begin = at = line.begin(int(blockIdx.x));
    end = line.begin(int(blockIdx.x) + 1);
    u = find_unit(a, at, lane);
  }
  __device__ __forceinline__ bool next(const Args& a, Piece& p) {
    while (at < end) {
      const int lo = int(at - u.begin), most = u.steps + a.overhead;
      const int hi = end - u.begin < most ? int(end - u.begin) : most;
      p.u = u;
      p.first = max(lo - a.overhead, 0);
      p.count = max(hi - a.overhead, 0) - p.first;
      p.whole = p.first == 0 && p.count == u.steps;
      p.zero = u.steps == 0 && lo == 0;
      p.part = at == begin ? 0 : 1;
      at = u.begin + hi;
      if (at < end) {  // the next unit
        u.begin = at;
        if (++u.head == a.heads) {
          u.head = 0;
          if (++u.block == a.blocks) {
            u.block = 0;
            u.tokens = request_tokens(a, ++u.b);
            u.steps = (u.tokens + kStep - 1) / kStep;
          }
        }
      }
      if (p.count > 0 || p.zero) return true;
    }
    return false;
  }
};

// A place in a ring and the parity of the phase that comes next there.
struct Cursor {
  int at;
  uint32_t parity;
  __device__ __forceinline__ void next(int slots) {
    if (++at == slots) { at = 0; parity ^= 1u; }
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
// The types' code is 0 for e4m3 under kind::f8f6f4 and for fp16 under kind::f16; fp32 accumulator.
__host__ __device__ constexpr uint32_t idesc_of(int M, int N, bool b_mn_major) {
  return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | (uint32_t(N >> 3) << 17) | (uint32_t(M >> 4) << 24);
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

template <int N> __device__ __forceinline__ void set_max_registers_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(N));
}
template <int N> __device__ __forceinline__ void set_max_registers_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(N));
}

// Row r of a unit's (query, query head): its place in q or out, from the unit's first.
__device__ __forceinline__ int64_t unit_offset(const Args& a, const int64_t (&s)[3], const Unit& u) {
  return u.b * s[0] + u.head * a.group * s[1];
}
__device__ __forceinline__ int64_t row_offset(const Args& a, const int64_t (&s)[3], int row) {
  // row < 2^30, so the product is 1 too large at most
  int query = a.group_magic ? int(__umulhi(uint32_t(row), a.group_magic)) : row;
  if (query * int64_t(a.group) > row) --query;
  return (row - query * a.group) * s[1] + query * s[2];
}

// A page's scale as it is; NaN for NaN, and for what is no power of two (an error).
__device__ __forceinline__ float checked_scale(const Args& a, float scale) {
  const uint32_t v = __float_as_uint(scale);
  if (v < 0x7F800000u && !(v & 0x7FFFFFu) && v != 0) return scale;
  if (v != 0x7FC00000u) atomicOr(a.err, PASA_DEVERR_BAD_SCALE);
  return __uint_as_float(0x7FC00000u);
}
// The exponent of a checked scale.
__device__ __forceinline__ float scale_log2(float scale) {
  return scale == scale ? float(int(__float_as_uint(scale) >> 23) - 127) : scale;
}

// 2^(x mul + shift) of 32 scores in fp16, and their fp32 sums.
__device__ __forceinline__ void probabilities(const uint32_t (&s)[32], float mul_, float shift, uint32_t (&p)[16],
                                              float2& sum0, float2& sum1) {
  const float2 mul = make_float2(mul_, mul_), add = make_float2(shift, shift);
#pragma unroll
  for (int e = 0; e < 32; e += 4) {
    const uint32_t* x = &s[e];
    float2 x01 = __ffma2_rn(make_float2(__uint_as_float(x[0]), __uint_as_float(x[1])), mul, add);
    float2 x23 = __ffma2_rn(make_float2(__uint_as_float(x[2]), __uint_as_float(x[3])), mul, add);
    x01.x = exp2_ftz(x01.x); x01.y = exp2_ftz(x01.y);
    x23.x = exp2_ftz(x23.x); x23.y = exp2_ftz(x23.y);
    sum0 = __fadd2_rn(sum0, x01);
    sum1 = __fadd2_rn(sum1, x23);
    const __half2 p01 = __floats2half2_rn(x01.x, x01.y), p23 = __floats2half2_rn(x23.x, x23.y);
    p[e >> 1] = *reinterpret_cast<const uint32_t*>(&p01);
    p[(e >> 1) + 1] = *reinterpret_cast<const uint32_t*>(&p23);
  }
}

// both: both tiles hold the same rows and take the steps in turn.
template <int D, bool both>
__global__ void __launch_bounds__(kThreads, 1) attention_kernel(const __grid_constant__ Maps maps,
                                                                const __grid_constant__ Args a) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* sm =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t key_full[kMaxSlots], key_empty[kMaxSlots], raw_full[kMaxSlots], raw_empty[kMaxSlots];
  __shared__ uint64_t wide_full[kMaxSlots], wide_empty[kMaxSlots], q_full[2], q_empty[2], o_free[2];
  __shared__ uint64_t s_full[2], p_full[2][2], pv_done[2];  // of a tile; p_full: of a page of a step
  __shared__ uint32_t tmem_slot;
  __shared__ float2 step_scale[kScaleSteps][2];  // of a step's two pages: the keys' scale, log2 of the values'
  __shared__ int raw_rows[kMaxSlots];            // tokens of a page of values; -1: the end
  __shared__ float2 copy_ml[2 * kTile];          // maximum and denominator of every copy of a row
  __shared__ uint64_t copies;
  __shared__ Piece work[2];                      // what a buffer of queries is for; no steps: the end
  float* q_scale = reinterpret_cast<float*>(sm + kOffScale);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int q_buf = both ? kQTile : kQBuf;  // bytes of a buffer of queries
  constexpr int keys_at = off_keys(both), raw_at = off_raw(both), wide_at = off_wide(both), out_at = off_out(both);

  if (threadIdx.x == 0) {
    for (int s = 0; s < kMaxSlots; ++s) {
      mbar_init(&key_full[s], 1);
      mbar_init(&key_empty[s], 1);
      mbar_init(&raw_full[s], 1);
      mbar_init(&raw_empty[s], kWideners);
      mbar_init(&wide_full[s], kWideners);
      mbar_init(&wide_empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full[t], kLoaders);
      mbar_init(&q_empty[t], 1 + 8);  // the last product that reads it, and the softmax warps (its scales)
      mbar_init(&o_free[t], 4);
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t][0], 4);
      mbar_init(&p_full[t][1], 4);
      mbar_init(&pv_done[t], 1);
    }
    mbar_init(&copies, 8);
    fence_barrier_init();
  }
  if (warp == 1) { tmem_alloc(&tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  if (warp < 4 || (warp >= 12 && warp < 16)) {
    set_max_registers_down<kRegistersQueries>();
    if (warp == 0) {
      // ================= keys and values =================
      Walk walk(a, lane);
      auto next_steps = [&](Piece& x) {
        while (walk.next(a, x))
          if (x.count > 0) return true;
        return false;
      };
      auto pages_left = [&](const Piece& x, int j) { return (x.u.tokens + kPage - 1) / kPage - 2 * (x.first + j); };
      // the table's entry for this lane's page of 16 steps
      auto entry = [&](const Piece& x, int j) {
        return lane < pages_left(x, j) ? a.table[x.u.b * a.width + 2 * (x.first + j) + lane] : 0;
      };
      Piece p, after;
      bool more = next_steps(p), ok = true;
      int coming = more ? entry(p, 0) : 0;  // the entry for the next 16 steps of keys, read that much ahead
      Cursor keys{0, 1}, raw{0, 1};
      int issued_keys = 0, issued_raw = 0, step = 0;  // step: of step_scale
      for (bool more_after; more && ok; more = more_after, p = after) {
        more_after = next_steps(after);
        const int n = p.count, ahead = both ? 2 : 1;
        int k_pages = 0, v_pages = 0;  // of 16 steps, a page a lane
        float2 scales = make_float2(1.f, 0.f);
        for (int jk = 0, jv = 0; jv < n && ok;) {
          // the next load: keys until they are `ahead` of the values, then in turn
          const bool values = jk >= min(n, jv + ahead);
          const int j = values ? jv++ : jk++;
          if ((j & 15) == 0) {
            if (values) {
              v_pages = k_pages;  // (the keys are less than 16 steps ahead)
            } else {
              const bool mine = lane < pages_left(p, j) && lane < 2 * (n - j);
              const bool bad = coming < 0 || coming >= a.pages;
              if (bad && mine) atomicOr(a.err, PASA_DEVERR_BAD_PAGE);
              k_pages = bad ? 0 : coming;
              // (a page behind the last token is masked: scores are -infinity whatever the scale, the values' is below any)
              scales = make_float2(1.f, __uint_as_float(0x00800000u));
              if (bad && mine) {  // (what is read in its place is another request's)
                scales.x = scales.y = __uint_as_float(0x7FC00000u);
              } else if (mine) {
                const int64_t z = int64_t(k_pages) * a.heads + p.u.head;
                scales = make_float2(a.k_scale[z], a.v_scale[z]);
              }
              coming = j + 16 < n ? entry(p, j + 16) : more_after ? entry(after, 0) : 0;
            }
          }
          const int pages = values ? v_pages : k_pages, at = 2 * (j & 15);
          const int z[2] = {__shfl_sync(0xffffffffu, pages, at) * a.heads + p.u.head,
                            __shfl_sync(0xffffffffu, pages, at + 1) * a.heads + p.u.head};
          if (values) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              ok = ok && __all_sync(0xffffffffu, mbar_wait_bounded(&raw_empty[raw.at], raw.parity));
              if (!ok) break;
              if (elect_one()) {
                const int rows = min(max(p.u.tokens - (p.first + j) * kStep - h * kPage, 0), kPage);
                raw_rows[raw.at] = rows;
                if (rows > 0) {
                  mbar_arrive_expect_tx(&raw_full[raw.at], uint32_t(kPage * D));
                  tma_load_3d(sm + raw_at + raw.at * kRawBytes, &maps.v, &raw_full[raw.at], 0, 0, z[h]);
                } else {
                  mbar_arrive(&raw_full[raw.at]);
                }
              }
              __syncwarp();
              ++issued_raw;
              raw.next(raw_slots(both));
            }
            continue;
          }
          const bool second = pages_left(p, j) > 1;
          ok = __all_sync(0xffffffffu, mbar_wait_bounded(&key_empty[keys.at], keys.parity));
          if (!ok) break;
          if (elect_one()) {
            unsigned char* dst = sm + keys_at + keys.at * kKeyBytes;
            tma_load_3d(dst, &maps.k, &key_full[keys.at], 0, 0, z[0]);
            if (second) tma_load_3d(dst + kKeyBytes / 2, &maps.k, &key_full[keys.at], 0, 0, z[1]);
          }
          // the scales are on their way while the tiles are: what the barrier expects comes behind them
          if ((j & 15) == 0) scales = make_float2(checked_scale(a, scales.x), scale_log2(checked_scale(a, scales.y)));
          if ((lane >> 1) == (j & 15)) step_scale[step % kScaleSteps][lane & 1] = scales;
          ++step;
          __syncwarp();
          if (elect_one())
            mbar_arrive_expect_tx(&key_full[keys.at], second ? uint32_t(kKeyBytes) : uint32_t(kKeyBytes / 2));
          __syncwarp();
          ++issued_keys;
          keys.next(key_slots(both));
        }
      }
      if (ok) {  // the end of the values
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(&raw_empty[raw.at], raw.parity));
        if (ok) {
          if (elect_one()) {
            raw_rows[raw.at] = -1;
            mbar_arrive(&raw_full[raw.at]);
          }
          ++issued_raw;
        }
      }
      if (!ok && lane == 0) report_operator_timeout(a.err);
      // the copies in flight land before the block can end
      auto land = [&](uint64_t* full, int issued, int slots) {
        for (int l = issued > slots ? issued - slots : 0; l < issued; ++l)
          mbar_wait_bounded(&full[l % slots], uint32_t((l / slots) & 1));
      };
      land(key_full, issued_keys, key_slots(both));
      land(raw_full, issued_raw, raw_slots(both));
    } else if (warp == 1) {
      // ================= products =================
      // One elected lane waits and issues: a wait by the whole warp, its vote and a new election around every product
      // took 1000 clocks a product.
      constexpr uint32_t id_s = idesc_of(128, kStep, false), id_o = idesc_of(128, D, true);
      Cursor keys{0, 0}, wide{0, 0};  // the elected lane's
      int buf = 0;
      uint32_t q_parity = 0, p_parity = 0, o_parity = 3;  // p_parity, o_parity: bit t
      bool ok = true;
      const uint64_t desc = umma_desc_sw128(smem_u32(sm), 16, 1024);  // of the start of shared memory
      const uint64_t wide_desc = umma_desc_sw128(smem_u32(sm + wide_at), kPage * 128, 1024);
      for (;;) {
        ok = __all_sync(0xffffffffu, ok && mbar_wait_bounded(&q_full[buf], q_parity));
        if (!ok) break;
        const int n = work[buf].count;
        if (n == 0) break;
        const int tiles = both ? min(n, 2) : (work[buf].u.block * 2 + 1) * kTile < a.rows ? 2 : 1;
        __syncwarp();
        auto wait = [&](uint64_t* bar, uint32_t parity) {
          if (ok) ok = mbar_wait_bounded(bar, parity);
        };
        // scores of tile t with the keys at their ring's cursor
        auto scores = [&](int t, bool frees_keys, bool frees_queries) {
          wait(&key_full[keys.at], keys.parity);
          if (!ok) return;
          tc_fence_after();
          const uint64_t qd = desc + uint64_t((kOffQ + buf * q_buf + (both ? 0 : t) * kQTile) >> 4);
          const uint64_t kd = desc + uint64_t((keys_at + keys.at * kKeyBytes) >> 4);
          const uint32_t d = tmem + kColS + uint32_t(128 * t);
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int kk = 0; kk < D / 32; ++kk)
              mma8_ss(d, qd + uint64_t((x * kTile * 128 + kk * 32) >> 4), kd + uint64_t((kk * 32) >> 4), id_s,
                      x > 0 || kk > 0 ? 1u : 0u);
          tc_commit(&s_full[t]);
          if (frees_keys) {
            tc_commit(&key_empty[keys.at]);
            keys.next(key_slots(both));
          }
          if (frees_queries) tc_commit(&q_empty[buf]);
        };
        // output of tile t += probabilities times the values of the two pages at their ring's cursor, a page as soon as
        // its probabilities are there
        auto output = [&](int t, bool first, bool frees_values) {
          if (first) {
            wait(&o_free[t], (o_parity >> t) & 1u);
            o_parity ^= 1u << t;
          }
          const uint32_t d = tmem + kColO + uint32_t(128 * t), pt = tmem + kColS + uint32_t(128 * t);
          Cursor c = wide;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            wait(&wide_full[c.at], c.parity);
            wait(&p_full[t][h], (p_parity >> t) & 1u);
            if (!ok) return;
            tc_fence_after();
            const uint64_t vd = wide_desc + uint64_t((c.at * kWideBytes) >> 4);
#pragma unroll
            for (int kk = 0; kk < kPage / 16; ++kk)
              mma_ts(d, pt + uint32_t(h * 64 + (kk >> 1) * 32 + (kk & 1) * 8), vd + uint64_t((kk * 2048) >> 4), id_o,
                     !first || h > 0 || kk > 0 ? 1u : 0u);
            if (frees_values) tc_commit(&wide_empty[c.at]);
            c.next(wide_slots(both));
          }
          p_parity ^= 1u << t;
          tc_commit(&pv_done[t]);
          if (frees_values) wide = c;
        };
        if (elect_one()) {
          if (both) {
            for (int j = 0; j < tiles; ++j) scores(j, true, j == n - 1);
            for (int j = 0; j < n && ok; ++j) {
              output(j & 1, j < 2, true);
              if (j + 2 < n) scores(j & 1, true, j + 2 == n - 1);
            }
          } else {
            for (int t = 0; t < tiles; ++t) scores(t, t == tiles - 1, n == 1 && t == tiles - 1);
            for (int j = 0; j < n && ok; ++j) {
              const bool more = j + 1 < n, last = j + 2 == n;
              output(0, j == 0, tiles == 1);
              if (more) scores(0, tiles == 1, tiles == 1 && last);
              if (tiles == 2) {
                output(1, j == 0, true);
                if (more) scores(1, true, last);
              }
            }
          }
        }
        ok = __all_sync(0xffffffffu, ok);  // the elected lane's, the others' is true
        if ((buf ^= 1) == 0) q_parity ^= 1u;
      }
      if (!ok && lane == 0) report_operator_timeout(a.err);
    } else {
      // ================= queries =================
      // Four lanes a row, eight rows a warp at a time: the row's largest value, its scale, hi and lo.  The bf16 row has
      // the size of its two e4m3 rows: it is copied to their place asynchronously, all rows of the buffer at once (48 in
      // flight, through registers, took 20000 clocks a buffer, this takes 15000), and split there.
      const int loader = warp < 4 ? warp - 2 : warp - 10;
      const int sub = lane >> 2, part = lane & 3;
      constexpr int kVecs = D / 32;  // 16-byte vectors of a lane: part + 4 i
      constexpr int kRounds = (2 * kTile + 8 * kLoaders - 1) / (8 * kLoaders);
      constexpr int kRowLanes = D / 8, kRowsAtOnce = 32 / kRowLanes;  // a copy's lanes in a row, its rows
      Walk walk(a, lane);
      Piece p{};
      int buf = 0;
      uint32_t parity = 1;
      bool ok = true;
      for (bool here = true; here;) {
        here = walk.next(a, p);
        const int r0 = p.u.block * 2 * kTile;
        // rows of the buffer; with quarters every 32 of them are the same
        const bool quarters = both && a.quarters;
        const int mask = quarters ? 31 : 255, kept = min(a.rows - r0, 2 * kTile);
        const int live = !here ? 0 : quarters ? kTile : kept;
        if (here && p.zero) {
          for (int row = loader * 8 + sub; row < kept; row += kLoaders * 8) {
            __nv_bfloat16* dst = a.out + unit_offset(a, a.os, p.u) + row_offset(a, a.os, r0 + row) + part * 8;
#pragma unroll
            for (int i = 0; i < kVecs; ++i) *reinterpret_cast<uint4*>(dst + 32 * i) = make_uint4(0u, 0u, 0u, 0u);
          }
          continue;
        }
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(&q_empty[buf], parity));
        if (!ok) break;
        const __nv_bfloat16* q = a.q + unit_offset(a, a.qs, p.u) + lane % kRowLanes * 8;
        unsigned char* qs = sm + kOffQ + buf * q_buf;
        auto place = [&](int row) { return qs + (row / kTile) * kQTile + (row % kTile) * 128; };
        // (what the rows behind the last hold makes only rows that are not kept)
        auto has = [&](int row) { return row < live && (row & mask) < kept; };
#pragma unroll 1
        for (int x = 0; x < kRounds; ++x) {
#pragma unroll
          for (int i = 0; i < kVecs; ++i) {
            const int row = x * 8 * kLoaders + loader * 8 + i * kRowsAtOnce + lane / kRowLanes, c = lane % kRowLanes;
            if (has(row))  // the first 128 bytes lie in the row of hi, the others in that of lo
              cp_async16(smem_u32(place(row)) + uint32_t((c & 7) * 16 + (c >> 3) * kTile * 128),
                         q + row_offset(a, a.qs, r0 + (row & mask)));
          }
        }
        auto split = [&](int x) {
          const int first = x * 8 * kLoaders + loader * 8, row = first + sub;
          if (first >= live) return;
          unsigned char* at = place(row < live ? row : first);
          Bf8 v[kVecs];
          uint32_t amax = 0;
#pragma unroll
          for (int i = 0; i < kVecs; ++i) {
            v[i].r = *reinterpret_cast<const uint4*>(at + part * 16 + (i & 1) * 64 + (i >> 1) * kTile * 128);
            amax = max(amax, v[i].amax());
          }
          amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
          amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
          __syncwarp();  // all of a row is read before any of it is written
          if (!has(row)) return;
          const float scale = scale_of(amax), inv = inverse(scale);
#pragma unroll
          for (int i = 0; i < kVecs; ++i) {
            const uint32_t in[4] = {v[i].r.x, v[i].r.y, v[i].r.z, v[i].r.w};
            uint16_t hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {  // exact in fp16: 8 significant bits, 448 at most
              const __half2 h = __floats2half2_rn(__uint_as_float(in[e] << 16) * inv,
                                                  __uint_as_float(in[e] & 0xFFFF0000u) * inv);
              hi[e] = f16x2_to_e4m3x2(*reinterpret_cast<const uint32_t*>(&h));
              const uint32_t back = e4m3x2_to_f16x2(hi[e]);
              const __half2 rest = __hsub2(h, *reinterpret_cast<const __half2*>(&back));
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
        };
        cp_async_wait_all();
        __syncwarp();
#pragma unroll 1
        for (int x = 0; x < kRounds; ++x) split(x);
        if (loader == 0 && lane == 0) {
          if (!here) p.count = 0;
          work[buf] = p;
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[buf]);
        if ((buf ^= 1) == 0) parity ^= 1u;
      }
      if (!ok && lane == 0) report_operator_timeout(a.err);
    }
  } else if (warp >= 16) {
    set_max_registers_down<kRegistersValues>();
    // ================= values: from e4m3 to fp16, which is exact =================
    // A warp 16 tokens of a page, a lane 16 dimensions of a token; what lies behind the last token is no value (it may
    // be a NaN's bits, and 0 * NaN is NaN) and becomes zero.
    constexpr int kRowLanes = D / 16, kRowsAtOnce = 32 / kRowLanes, kVecs = kPage / kWideners / kRowsAtOnce;
    const int row0 = (warp - 16) * (kPage / kWideners) + lane / kRowLanes, c = lane % kRowLanes;
    Cursor raw{0, 0}, wide{0, 1};
    bool ok = true;
    for (;;) {
      ok = __all_sync(0xffffffffu, mbar_wait_bounded(&wide_empty[wide.at], wide.parity) &&
                                       mbar_wait_bounded(&raw_full[raw.at], raw.parity));
      if (!ok) break;
      const int rows = raw_rows[raw.at];
      if (rows < 0) break;
      const unsigned char* src = sm + raw_at + raw.at * kRawBytes + c * 16;
      uint4 x[kVecs];
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        const int row = row0 + i * kRowsAtOnce;
        x[i] = row < rows ? *reinterpret_cast<const uint4*>(src + row * D) : make_uint4(0u, 0u, 0u, 0u);
      }
      unsigned char* dst = sm + wide_at + wide.at * kWideBytes + (c >> 2) * (kPage * 128);
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        const int row = row0 + i * kRowsAtOnce;
        const uint32_t in[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
        uint32_t v[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[2 * e] = e4m3x2_to_f16x2(uint16_t(in[e]));
          v[2 * e + 1] = e4m3x2_to_f16x2(uint16_t(in[e] >> 16));
        }
        // the row's 16-byte pieces are swizzled by the row; the lanes of the second 64 dimensions store their second
        // piece first, so that eight lanes meet no bank twice
        const bool swap = (c >> 2) != 0;
        unsigned char* at = dst + row * 128;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int piece = (c & 3) * 2 + (k ^ int(swap));
          const bool high = (k != 0) != swap;
          *reinterpret_cast<uint4*>(at + ((piece ^ (row & 7)) << 4)) =
              make_uint4(high ? v[4] : v[0], high ? v[5] : v[1], high ? v[6] : v[2], high ? v[7] : v[3]);
        }
      }
      fence_proxy_async();
      __syncwarp();
      // (the page's place is handed back when what was read of it has been used: an arrival does not wait for loads
      // before it, which took 1500 clocks behind another warp's stores)
      if (lane == 0) {
        mbar_arrive(&wide_full[wide.at]);
        mbar_arrive(&raw_empty[raw.at]);
      }
      raw.next(raw_slots(both));
      wide.next(wide_slots(both));
    }
    if (!ok && lane == 0) report_operator_timeout(a.err);
  } else {
    set_max_registers_up<kRegistersSoftmax>();
    // ================= softmax of tile t: a thread a row =================
    const int t = (warp - 4) >> 2, w = warp & 3, row = w * 32 + lane;
    const uint32_t lanes = uint32_t(w * 32) << 16;
    const uint32_t s_tmem = tmem + lanes + kColS + 128u * uint32_t(t), o_tmem = tmem + lanes + kColO + 128u * uint32_t(t);
    const bool quarters = both && a.quarters;
    int buf = 0;
    uint32_t q_parity = 0, k_parity = 0;  // k_parity: of the tile's next step
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      if (ok && !mbar_wait_bounded(bar, parity)) {
        ok = false;
        report_operator_timeout(a.err);
      }
    };
    uint32_t copies_parity = 0;
    auto all_copies = [&] {  // a barrier of the 8 warps that ends
      __syncwarp();
      if (lane == 0) mbar_arrive(&copies);
      wait(&copies, copies_parity);
      copies_parity ^= 1u;
    };
    for (int base = 0;;) {  // base: the piece's first step in step_scale
      wait(&q_full[buf], q_parity);
      if (!__all_sync(0xffffffffu, ok)) break;
      const Piece p = work[buf];
      const int n = p.count, tokens = p.u.tokens;
      if (n == 0) break;
      const int r0 = p.u.block * 2 * kTile + (both ? 0 : t * kTile);
      const int r = r0 + (quarters ? lane : row);  // the row of the key/value head
      const bool live = r < a.rows, warp_live = quarters || r0 + w * 32 < a.rows;
      const int tiles = both ? min(n, 2) : (p.u.block * 2 + 1) * kTile < a.rows ? 2 : 1;
      const float q_row = q_scale[buf * 2 * kTile + (both ? 0 : t * kTile) + row] * a.scale_log2;
      __threadfence_block();  // an arrival does not wait for loads before it
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_empty[buf]);
      if ((buf ^= 1) == 0) q_parity ^= 1u;
      // References (log2): m of the probabilities in the denominator l, v_ref of the values' scales; the output's is
      // m + v_ref.  They are a row's own.
      float m = -INFINITY, l = 0.f, v_ref = 0.f;
      const int stride = both ? 2 : 1, begin = both ? t : 0;
      // The references move when a probability, or one times its value's scale, is more than 2^4 above them.
      auto follow = [&](float top, float v_top, bool first) {
        const bool moves = top > m + kRescale || v_top > m + v_ref + kRescale;
        if (!__any_sync(0xffffffffu, moves)) return;
        const float m_new = moves ? fmaxf(m, top) : m;
        const float v_new = moves ? (first ? v_top : fmaxf(m + v_ref, v_top)) - m_new : v_ref;
        if (!first) {
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
      };
      // log2 of a page's value scale over the reference; -60 at the least, which is nothing next to what set the reference
      auto value_shift = [&](float v_log2) { return v_log2 == v_log2 ? fmaxf(v_log2 - v_ref, -60.f) : v_log2; };
      if (t < tiles) {
        for (int j = begin; j < n; j += stride, k_parity ^= 1u) {
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
          const float2 page[2] = {step_scale[(base + j) % kScaleSteps][0], step_scale[(base + j) % kScaleSteps][1]};
          const int valid = tokens - (p.first + j) * kStep;
          auto score_scale = [&](int h) {
            const float c = q_row * page[h].x;
            return c < 1e-37f ? 1e-37f : c;  // -infinity times it stays that; a NaN stays NaN
          };
          if (quarters) {
            uint32_t s[32];
            tmem_ld32(s_tmem + 32u * uint32_t(w), s);
            const float c = score_scale(w >> 1), v_log2 = page[w >> 1].y;
            tmem_wait_ld();
            if (valid < kStep) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (i + 32 * w >= valid) s[i] = 0xFF800000u;
            }
            const float top = max_tree32(s) * c;
            follow(top, top + v_log2, j == begin);
            const float dv = value_shift(v_log2);
            float2 sum0 = make_float2(0.f, 0.f), sum1 = make_float2(0.f, 0.f);
            uint32_t pk[16];
            probabilities(s, c, dv + kLog2P - (m == -INFINITY ? 0.f : m), pk, sum0, sum1);
#pragma unroll
            for (int g = 0; g < 4; ++g) {  // nothing for the tokens of the other quarters
              uint32_t x[16];
#pragma unroll
              for (int e = 0; e < 16; ++e) x[e] = g == w ? pk[e] : 0u;
              tmem_st16(s_tmem + uint32_t(32 * g), x);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              mbar_arrive(&p_full[t][0]);
              mbar_arrive(&p_full[t][1]);
            }
            l += ((sum0.x + sum0.y) + (sum1.x + sum1.y)) * exp2_ftz(-dv - kLog2P);
            continue;
          }
          const float c0 = score_scale(0), c1 = score_scale(1);
          auto load = [&](int h, uint32_t (&s)[2][32]) {  // a page's scores
            tmem_ld32(s_tmem + 64u * uint32_t(h), s[0]);
            tmem_ld32(s_tmem + 64u * uint32_t(h) + 32u, s[1]);
            tmem_wait_ld();
            if (valid < kStep) {
#pragma unroll
              for (int i = 0; i < 64; ++i)
                if (i + 64 * h >= valid) s[i >> 5][i & 31] = 0xFF800000u;
            }
          };
          float top = -INFINITY, v_top = -INFINITY;
#pragma unroll 1
          for (int h = 0; h < 2; ++h) {
            uint32_t s[2][32];
            load(h, s);
            const float x = fmaxf(max_tree32(s[0]), max_tree32(s[1])) * (h ? c1 : c0);
            top = fmaxf(top, x);
            v_top = fmaxf(v_top, x + (h ? page[1].y : page[0].y));
          }
          follow(top, v_top, j == begin);
#pragma unroll 1
          for (int h = 0; h < 2; ++h) {
            const float dv = value_shift(h ? page[1].y : page[0].y), shift = dv + kLog2P - (m == -INFINITY ? 0.f : m);
            float2 sum0 = make_float2(0.f, 0.f), sum1 = make_float2(0.f, 0.f);
            uint32_t s[2][32];
            load(h, s);
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              uint32_t pk[16];
              probabilities(s[g], h ? c1 : c0, shift, pk, sum0, sum1);
              tmem_st16(s_tmem + uint32_t(64 * h + 32 * g), pk);
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
      base += n;
      __nv_bfloat16* out = a.out + unit_offset(a, a.os, p.u);
      const float to_true = exp2f(v_ref - kLog2P);  // the accumulator's unit
      const int64_t part_row = (int64_t(blockIdx.x) * 2 + p.part) * 2 * kTile;  // the first of a part of the unit
      if (both) {
        // the copies of a row (2 tiles, or 8 warps) are added through shared memory, 16 columns at a time
        float4* xch = reinterpret_cast<float4*>(sm + out_at);
        const int me = t * kTile + row, rows = quarters ? 32 : kTile, r_me = me & (rows - 1);
        copy_ml[me] = make_float2(m, l);
        all_copies();
        float top = m, sum = 0.f;
        for (int c = r_me; c < 2 * kTile; c += rows) top = fmaxf(top, copy_ml[c].x);
        for (int c = r_me; c < 2 * kTile; c += rows)
          sum += copy_ml[c].y * exp2_ftz(fmaxf(copy_ml[c].x - top, -200.f));
        float f = to_true * exp2_ftz(fmaxf(m - top, -200.f));
        if (p.whole) f /= sum;
        else if (me < rows && live) a.part_ml[part_row + me] = make_float2(top, sum);
        const bool none = l == 0.f;  // (the output of a tile without steps is not set)
#pragma unroll 1
        for (int i = 0; i < D / 16; ++i) {
          uint32_t o[16];
          __syncwarp();
          tmem_ld16(o_tmem + 16u * uint32_t(i), o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = none ? 0u : __float_as_uint(__uint_as_float(o[e]) * f);
#pragma unroll
          for (int v = 0; v < 4; ++v)
            xch[v * 2 * kTile + me] = *reinterpret_cast<const float4*>(&o[4 * v]);
          all_copies();
          for (int at = me; at < 4 * rows; at += 2 * kTile) {
            const int v = at / rows, rr = at & (rows - 1);
            float4 y = xch[v * 2 * kTile + rr];
            for (int c = rr + rows; c < 2 * kTile; c += rows) {
              const float4 z = xch[v * 2 * kTile + c];
              y.x += z.x; y.y += z.y; y.z += z.z; y.w += z.w;
            }
            if (rr >= a.rows) continue;
            const int col = 16 * i + 4 * v;
            if (p.whole)
              *reinterpret_cast<uint2*>(out + row_offset(a, a.os, rr) + col) =
                  make_uint2(pack_bf16x2(y.x, y.y), pack_bf16x2(y.z, y.w));
            else
              *reinterpret_cast<float4*>(a.part_o + (part_row + rr) * D + col) = y;
          }
          all_copies();  // the space may be written again
        }
      } else if (!p.whole) {
        // sums, maximum and denominator for the second kernel
        const int64_t at = part_row + t * kTile + row;
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
      } else if (t < tiles) {
        // through shared memory, 16 columns at a time: 2 lanes then write 32 bytes of a row
        const float f = to_true / l;
        unsigned char* stage = sm + out_at + (warp - 4) * 1024;
        int64_t at[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int rr = r0 + w * 32 + x * 16 + (lane >> 1);
          at[x] = rr < a.rows ? row_offset(a, a.os, rr) + (lane & 1) * 8 : -1;
        }
#pragma unroll 1
        for (int i = 0; i < D / 16; ++i) {
          uint32_t o[16];
          __syncwarp();
          tmem_ld16(o_tmem + 16u * uint32_t(i), o);
          tmem_wait_ld();
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            const uint32_t* x = &o[8 * v];
            *reinterpret_cast<uint4*>(stage + lane * 32 + ((v ^ ((lane >> 2) & 1)) << 4)) =
                make_uint4(pack_bf16x2(__uint_as_float(x[0]) * f, __uint_as_float(x[1]) * f),
                           pack_bf16x2(__uint_as_float(x[2]) * f, __uint_as_float(x[3]) * f),
                           pack_bf16x2(__uint_as_float(x[4]) * f, __uint_as_float(x[5]) * f),
                           pack_bf16x2(__uint_as_float(x[6]) * f, __uint_as_float(x[7]) * f));
          }
          __syncwarp();
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int rr = x * 16 + (lane >> 1);
            const uint4 y = *reinterpret_cast<const uint4*>(stage + rr * 32 + (((lane & 1) ^ ((rr >> 2) & 1)) << 4));
            if (at[x] >= 0) *reinterpret_cast<uint4*>(out + at[x] + 16 * i) = y;
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
// CTA c's part of the line and goes on in the next; a warp four rows.  The
// parts' maxima and denominators are read by a lane each, so that the loads of
// their sums wait for nothing: 16 us for 147 cut units of 256 rows, 6 us for 5.
constexpr int kJoinWarps = 8, kJoinRows = 4;
template <int D>
__global__ void __launch_bounds__(32 * kJoinWarps) join_kernel(const __grid_constant__ Args a, int parts) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  wait_for_predecessor();
  const int first = int(blockIdx.x);
  const Parts line(total_ticks(a, lane), parts);
  const int64_t cut = line.begin(first + 1);
  if (cut >= line.total) return;
  const Unit u = find_unit(a, cut, lane);
  // the unit's steps before the cut: some, and all of them CTA c's
  if (cut - u.begin <= a.overhead || line.begin(first) > u.begin + a.overhead) return;
  const int64_t end = u.begin + a.overhead + u.steps;
  int count = 1;  // CTAs with steps of the unit
  for (int c0 = first + 1; c0 < parts; c0 += 32) {
    const uint32_t has = __ballot_sync(0xffffffffu, c0 + lane < parts && line.begin(c0 + lane) < end);
    count += __popc(has);
    if (has != 0xffffffffu) break;
  }
  const int part = line.begin(first) >= u.begin ? 0 : 1;  // the first one's; the others' begin with the unit
  constexpr int kCols = D / 32;
  const int rows = min(a.rows - u.block * 2 * kTile, 2 * kTile);
  const int row0 = (int(blockIdx.y) * kJoinWarps + warp) * kJoinRows;
  if (row0 >= rows) return;
  float o[kJoinRows][kCols] = {}, m[kJoinRows], l[kJoinRows] = {};
#pragma unroll
  for (int x = 0; x < kJoinRows; ++x) m[x] = -INFINITY;
  for (int c0 = 0; c0 < count; c0 += 32) {
    const int c = c0 + lane;
    const int64_t mine = (int64_t(first + c) * 2 + (c ? 0 : part)) * 2 * kTile + row0;
    // (with fewer ticks than CTAs some have none)
    const bool some = c < count && line.begin(first + c + 1) > line.begin(first + c);
    float2 ml[kJoinRows];
    float share[kJoinRows];
#pragma unroll
    for (int x = 0; x < kJoinRows; ++x)
      ml[x] = some && row0 + x < rows ? a.part_ml[mine + x] : make_float2(-INFINITY, 0.f);
#pragma unroll
    for (int x = 0; x < kJoinRows; ++x) {
      float top = fmaxf(m[x], ml[x].x);
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
      const float fall = exp2_ftz(fmaxf(m[x] - top, -200.f));
      share[x] = exp2_ftz(fmaxf(ml[x].x - top, -200.f));
      l[x] *= fall;
      m[x] = top;
#pragma unroll
      for (int i = 0; i < kCols; ++i) o[x][i] *= fall;
    }
    for (uint32_t left = __ballot_sync(0xffffffffu, some); left != 0; left &= left - 1) {
      const int src = __ffs(int(left)) - 1;
      const float* from = a.part_o + __shfl_sync(0xffffffffu, mine, src) * D + lane * kCols;
      float v[kJoinRows][kCols];
#pragma unroll
      for (int x = 0; x < kJoinRows; ++x) {
        if (row0 + x >= rows) continue;
        if constexpr (kCols == 4) *reinterpret_cast<float4*>(v[x]) = *reinterpret_cast<const float4*>(from + x * D);
        else *reinterpret_cast<float2*>(v[x]) = *reinterpret_cast<const float2*>(from + x * D);
      }
#pragma unroll
      for (int x = 0; x < kJoinRows; ++x) {  // (in order, wherever CTAs without ticks lie)
        const float f = __shfl_sync(0xffffffffu, share[x], src), part_l = __shfl_sync(0xffffffffu, ml[x].y, src);
        if (part_l == 0.f) continue;  // (one without tokens has no sums)
        l[x] = fmaf(part_l, f, l[x]);
#pragma unroll
        for (int i = 0; i < kCols; ++i) o[x][i] = fmaf(v[x][i], f, o[x][i]);
      }
    }
  }
  __nv_bfloat16* out = a.out + unit_offset(a, a.os, u) + lane * kCols;
#pragma unroll
  for (int x = 0; x < kJoinRows; ++x) {
    if (row0 + x >= rows) continue;
    __nv_bfloat16* at = out + row_offset(a, a.os, u.block * 2 * kTile + row0 + x);
    const float inv = 1.f / l[x];
#pragma unroll
    for (int i = 0; i < kCols; i += 2)
      *reinterpret_cast<uint32_t*>(at + i) = pack_bf16x2(o[x][i] * inv, o[x][i + 1] * inv);
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
// e4m3 [pages * heads][64][dim]; a box is a page of one head.  Keys: its rows 128
// bytes apart in shared memory (dim 64: the rest of a row is filled with zeros) and
// swizzled for the products; values: as they lie in the cache.
bool make_page_map(CUtensorMap* m, const void* base, int64_t pages, int heads, int dim, bool keys) {
  const auto fn = tensor_map_encoder();
  if (!fn) return false;
  const cuuint64_t dims[3] = {cuuint64_t(dim), cuuint64_t(kPage), cuuint64_t(pages * heads)};
  const cuuint64_t strides[2] = {cuuint64_t(dim), cuuint64_t(dim) * kPage};
  const cuuint32_t box[3] = {keys ? 128u : cuuint32_t(dim), cuuint32_t(kPage), 1u};
  const cuuint32_t step[3] = {1u, 1u, 1u};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, step,
            CU_TENSOR_MAP_INTERLEAVE_NONE, keys ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
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

// The warpgroups share out the registers that the block is launched with: with fewer they would wait for good.
int registers_of(void (*kernel)(Maps, Args)) {
  cudaFuncAttributes at{};
  return cudaFuncGetAttributes(&at, reinterpret_cast<const void*>(kernel)) == cudaSuccess ? at.numRegs : 0;
}

template <int D>
cudaError_t launch_attention(cudaStream_t st, const Maps& maps, const Args& a, int sms) {
  const auto kernel = a.rows <= kTile ? attention_kernel<D, true> : attention_kernel<D, false>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) return e;
  static const int registers[2] = {registers_of(attention_kernel<D, false>), registers_of(attention_kernel<D, true>)};
  if (registers[a.rows <= kTile] != kRegisters) return cudaErrorInvalidKernelImage;
  kernel<<<unsigned(sms), kThreads, kSmem, st>>>(maps, a);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  const int rows = a.rows < 2 * kTile ? a.rows : 2 * kTile;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(sms - 1), unsigned(cdiv(rows, kJoinRows * kJoinWarps)));
  cfg.blockDim = dim3(32 * kJoinWarps);
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
  if (!make_page_map(&maps.k, some, pages ? pages : 1, int(heads), dim, true) ||
      !make_page_map(&maps.v, pages ? v_cache : workspace, pages ? pages : 1, int(heads), dim, false))
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
  a.group_magic = group == 1 ? 0u : uint32_t((uint64_t(1) << 32) / uint64_t(group) + 1);
  a.rows = int(queries * group);
  a.blocks = int(cdiv(a.rows, 2 * kTile));
  a.quarters = a.rows <= 32 ? 1 : 0;
  // a unit takes about as long as that many steps besides its own (one token, 8 requests of 130 to 32767: 165 us at 2,
  // 92 at 12; 32760 queries over 512 and 77 tokens: 966 at 2, 810 at 4, 840 at 6)
  a.overhead = a.quarters ? 12 : 4;
  a.scale_log2 = scale * kLog2e;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + size_t(sms) * 2 * 2 * kTile * size_t(dim));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dim == 64 ? launch_attention<64>(s, maps, a, sms) : launch_attention<128>(s, maps, a, sms);
  return e == cudaSuccess ? PASA_OK : PASA_ERR_CUDA;
}

}  // extern "C"
