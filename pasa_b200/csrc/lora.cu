// Low-rank adapters of many requests beside a shared projection.  Request q
// owns the rows [rows[q], rows[q+1]) and the adapter slots[q] (none if outside
// [0, adapters)); with that adapter's A [R, K], B [N, R] and scale s
//     h = s x A^T            (down)      out = y + h B^T          (up)
// and backwards, from dy,
//     g = s dy B             (down)      dx  = base + g A         (up)
//     dA = g^T x,  dB = dy^T h           (grad), summed over the adapter's rows.
//
// Bound: HBM.  R is at most 128, so a row of x costs 2 R operations for every
// 2 bytes: a quarter of the tensor cores' balance at most.  The tensor cores
// (tcgen05) are still needed: at R = 64 a step at Wan2.1-14B's size is 0.2
// TFLOP.  The products run as three kernels, each reading its large operands
// once: down reads x (or dy), up reads y and writes out (or dx), grad reads x
// and dy.  h and g are R wide; passing them through memory costs R / K of the
// traffic and lets each kernel split its own long axis: down splits K over a
// cluster of up to 8 CTAs when there are few rows (the partial sums meet in
// distributed shared memory, in rank order), up splits N.  Measured: 75600 rows,
// 5120 -> 5120, R = 32: down 133 us (5.8 TB/s), up 332 us (4.7 TB/s); 32760 rows,
// R = 64: grad 131 us (5.1 TB/s).
//
// Rounding: h and g are products' operands again, and are kept as two bf16
// terms, v = hi + lo to 2^-17 of v, each multiplied and accumulated in fp32:
// one term would cost 2^-9.  The second term doubles the small products, which
// are not what bounds the kernels.  Results are rounded once.
//
// Rows are worked on in spans: a span begins at every multiple of 128 rows (4 in
// the kernels for few rows) and at every request's first row, and ends at the
// next of either, so a span has one adapter.  Every block finds its span from `rows` on the device (no host
// copy; a captured graph follows new lengths).
#include <atomic>

#include "umma.cuh"

namespace pasa {
namespace lora {

constexpr int kRows = 128;          // rows of a span at most: the lanes of the accumulator
constexpr int kThreads = 192;       // warp 0 TMA, warp 1 MMA + TMEM, warps 2-5 epilogue
constexpr int kBox = 32;            // rows of a TMA box of x, y, out and h: a short span loads only what it has
constexpr int kBoxBytes = kBox * 128;
constexpr int kMaxStages = 8;
constexpr int kMaxRank = 128;
constexpr int kSmemTwo = 112 * 1024;  // shared memory of a block when two share an SM

struct Rows {
  const int32_t* rows;   // [requests + 1]
  const int32_t* slots;  // [requests]
  const float* scale;    // [adapters] or null
  int requests, adapters;
  int64_t m;
};

struct Span {
  int64_t begin;
  int count;  // 0: nothing to do
  int slot;   // -1: no adapter
};

// Span t, in the order of the rows; count 0 behind the last one.  Segment 0 is
// the rows before the first request, then the requests, then the rows behind
// the last; each lane of the warp takes a segment's bounds and a prefix sum over
// their spans finds the one with span t.  All lanes of a warp call it.
template <int ROWS>
__device__ __forceinline__ Span find_span(const Rows& a, int64_t t, int lane) {
  Span s{0, 0, -1};
  for (int first = 0; first <= a.requests + 1; first += 32) {
    const int segment = first + lane;
    int64_t begin = 0, end = 0;
    if (segment <= a.requests + 1) {
      begin = segment == 0 ? 0 : a.rows[segment - 1];
      end = segment <= a.requests ? a.rows[segment] : a.m;
      if (begin < 0) begin = 0;
      if (end > a.m) end = a.m;
    }
    const int64_t own = end > begin ? (end - 1) / ROWS - begin / ROWS + 1 : 0;
    int64_t upto = own;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= off) upto += v;
    }
    const uint32_t reached = __ballot_sync(0xffffffffu, upto > t);
    if (reached == 0) {
      t -= __shfl_sync(0xffffffffu, upto, 31);
      continue;
    }
    const int src = __ffs(int(reached)) - 1;
    t -= __shfl_sync(0xffffffffu, upto - own, src);
    begin = __shfl_sync(0xffffffffu, begin, src);
    end = __shfl_sync(0xffffffffu, end, src);
    s.begin = t == 0 ? begin : (begin / ROWS + t) * ROWS;
    const int64_t next = (s.begin / ROWS + 1) * ROWS;
    s.count = int((next < end ? next : end) - s.begin);
    const int request = first + src - 1;
    if (request >= 0 && request < a.requests) {
      const int slot = a.slots[request];
      if (slot >= 0 && slot < a.adapters) s.slot = slot;
    }
    return s;
  }
  return s;
}

// v = hi + lo in two bf16 terms; an infinity or NaN is hi alone.  (Times an infinite element of the other operand the
// two terms may differ in sign: such a sum is infinite or NaN.)
__device__ __forceinline__ void split2(float v0, float v1, uint32_t& hi, uint32_t& lo) {
  hi = pack_bf16x2(v0, v1);
  const float h0 = __uint_as_float(hi << 16), h1 = __uint_as_float(hi & 0xFFFF0000u);
  lo = pack_bf16x2(isfinite(h0) ? v0 - h0 : 0.f, isfinite(h1) ? v1 - h1 : 0.f);
}

// Shared memory is carved up by the block itself: a short span needs fewer
// bytes a stage and gets more stages, which is what a span of few rows, bound
// by the latency of reading weights, needs.
struct Ring {
  int stages, stage_bytes;
};
__device__ __forceinline__ Ring ring_in(int room, int stage_bytes) {
  const int stages = room / stage_bytes;
  return Ring{stages < kMaxStages ? stages : kMaxStages, stage_bytes};
}

// ---------------------------------------------------------------------------
// down: h[rows, R] = scale * u[rows, C] w^T, w = A [R, C] (K-major) or B [C, R]
// (MN-major, its ranks contiguous)
// ---------------------------------------------------------------------------
struct DownMaps {
  CUtensorMap u, w;
};
struct DownArgs {
  Rows rows;
  int room;        // bytes of shared memory for the ring
  int rank, rp;    // R, and rounded up to 16: h is zero behind R, whatever x holds (infinity times the zeros of w is NaN)
  int64_t steps;   // 64-wide steps of C
  int split;       // CTAs of a cluster, each a share of the steps
  __nv_bfloat16* h;  // [2][m][rp]
  uint32_t* err;
};

__host__ __device__ constexpr int down_w_bytes(bool mn, int rp) { return mn ? ((rp + 63) / 64) * 8192 : rp * 128; }

template <bool MN>
__global__ void __launch_bounds__(kThreads) down_kernel(const __grid_constant__ DownMaps maps,
                                                        const __grid_constant__ DownArgs a) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* sm =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages], done;
  __shared__ uint32_t tmem_slot;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = int(blockIdx.x % unsigned(a.split));
  const Span span = find_span<kRows>(a.rows, blockIdx.x / unsigned(a.split), lane);
  if (span.count == 0 || span.slot < 0) return;  // the same for the whole cluster

  const uint32_t cols = a.rp <= 32 ? 32 : a.rp <= 64 ? 64 : 128;
  const int boxes = (span.count + kBox - 1) / kBox;
  const int w_bytes = down_w_bytes(MN, a.rp), u_bytes = boxes * kBoxBytes;
  // (every MMA reads 128 rows: where a span has fewer boxes the others' rows
  // are the weights and stages behind them, and only make rows that are not kept;
  // the last stage is followed by the rest of a full tile)
  const Ring ring = ring_in(a.room - (kRows * 128 - u_bytes), u_bytes + w_bytes);
  if (threadIdx.x == 0) {
    for (int s = 0; s < ring.stages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    mbar_init(&done, 1);
    fence_barrier_init();
  }
  if (warp == 1) { tmem_alloc(&tmem_slot, cols); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  dependents_may_start();  // they take TMEM too: not before this block has its own
  const int first = int(a.steps * rank / a.split), last = int(a.steps * (rank + 1) / a.split);

  if (warp == 0) {
    if (elect_one()) {
      int issued = 0;
      for (int i = 0; first + i < last; ++i) {
        const int s = i % ring.stages;
        if (!mbar_wait_bounded(&empty[s], uint32_t((i / ring.stages) & 1) ^ 1u)) {
          report_operator_timeout(a.err);
          break;
        }
        unsigned char* st = sm + s * ring.stage_bytes;
        const int32_t c0 = (first + i) * 64;
        mbar_arrive_expect_tx(&full[s], uint32_t(u_bytes + w_bytes));
        for (int b = 0; b < boxes; ++b)
          tma_load_3d(st + b * kBoxBytes, &maps.u, &full[s], c0, int32_t(span.begin) + b * kBox, 0);
        unsigned char* w = st + u_bytes;
        if (MN) {
          for (int r = 0; r < a.rp; r += 64) tma_load_3d(w + r * 128, &maps.w, &full[s], r, c0, span.slot);
        } else {
          tma_load_3d(w, &maps.w, &full[s], c0, 0, span.slot);
        }
        issued = i + 1;
      }
      // the copies in flight land before the block can end
      for (int i = issued > ring.stages ? issued - ring.stages : 0; i < issued; ++i)
        mbar_wait_bounded(&full[i % ring.stages], uint32_t((i / ring.stages) & 1));
    }
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t idesc = umma_idesc_bf16(128, a.rp, false, MN);
      for (int i = 0; first + i < last; ++i) {
        const int s = i % ring.stages;
        if (!mbar_wait_bounded(&full[s], uint32_t((i / ring.stages) & 1))) {
          report_operator_timeout(a.err);
          break;
        }
        tc_fence_after();
        const uint32_t st = smem_u32(sm + s * ring.stage_bytes);
        const uint64_t ud = umma_desc_sw128(st, 16, 1024);
        const uint64_t wd = umma_desc_sw128(st + u_bytes, MN ? 8192 : 16, 1024);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          mma_ss(tmem, ud + uint64_t((kk * 32) >> 4), wd + uint64_t((kk * (MN ? 2048 : 32)) >> 4), idesc,
                 i > 0 || kk > 0 ? 1u : 0u);
        tc_commit(&empty[s]);
      }
      tc_commit(&done);
    }
  } else {
    const int q = warp & 3, row = q * 32 + lane;
    if (!mbar_wait_bounded(&done, 0)) report_operator_timeout(a.err);
    tc_fence_after();
    const bool live = row < span.count;
    const float scale = a.rows.scale ? a.rows.scale[span.slot] : 1.f;
    __nv_bfloat16* hi = a.h + (span.begin + row) * a.rp;
    __nv_bfloat16* lo = hi + a.rows.m * a.rp;
    float* part = reinterpret_cast<float*>(sm) + row * (a.rp + 4);  // the ring is free once `done`
    for (int c = 0; c < a.rp; c += 16) {
      uint32_t v[16];
      __syncwarp();
      tmem_ld16(tmem + (uint32_t(q * 32) << 16) + uint32_t(c), v);
      tmem_wait_ld();
      if (a.split > 1) {
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *reinterpret_cast<uint4*>(part + c + i) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
      } else if (live) {
        uint32_t h[8], l[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          split2(scale * __uint_as_float(v[2 * i]), scale * __uint_as_float(v[2 * i + 1]), h[i], l[i]);
          if (c + 2 * i >= a.rank) h[i] = l[i] = 0u;  // (R is a multiple of 8)
        }
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
          *reinterpret_cast<uint4*>(hi + c + 2 * i) = make_uint4(h[i], h[i + 1], h[i + 2], h[i + 3]);
          *reinterpret_cast<uint4*>(lo + c + 2 * i) = make_uint4(l[i], l[i + 1], l[i + 2], l[i + 3]);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, cols);
  if (a.split == 1) return;

  // The cluster's partial sums, in rank order; each CTA sums a share of the rows.
  __syncwarp();
  cluster_sync_all();
  const float scale = a.rows.scale ? a.rows.scale[span.slot] : 1.f;
  const int quads = a.rp / 4;
  for (int i = int(threadIdx.x) + rank * kThreads; i < span.count * quads; i += kThreads * a.split) {
    const int row = i / quads, c = (i - row * quads) * 4;
    const uint32_t at = smem_u32(sm) + uint32_t(row * (a.rp + 4) + c) * 4u;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int r = 0; r < a.split; ++r) {
      const float4 v = cluster_load4(cluster_map(at, uint32_t(r)));
      sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
    }
    uint32_t h[2], l[2];
    split2(scale * sum.x, scale * sum.y, h[0], l[0]);
    split2(scale * sum.z, scale * sum.w, h[1], l[1]);
    if (c >= a.rank) h[0] = h[1] = l[0] = l[1] = 0u;
    __nv_bfloat16* hi = a.h + (span.begin + row) * a.rp + c;
    *reinterpret_cast<uint2*>(hi) = make_uint2(h[0], h[1]);
    *reinterpret_cast<uint2*>(hi + a.rows.m * a.rp) = make_uint2(l[0], l[1]);
  }
  __syncwarp();
  cluster_sync_all();  // no CTA ends while another reads its partial sums
}

// ---------------------------------------------------------------------------
// up: out[rows, C] = base[rows, C] + h[rows, R] w, w^T = B [C, R] (K-major) or
// w = A [R, C] (MN-major).  A unit of work is a span and a share of its
// 64-column chunks; two blocks an SM go through their units, and their loads
// run ahead into the next unit.  h (hi and lo) lies in TMEM as the products'
// first operand.  The base's chunk lands in shared memory by TMA, is added to
// in place and leaves by TMA from there (by plain stores where a box of 32 rows
// reaches into another span).  The base and the weights have rings of their
// own: the weights' is freed by the product, the base's only when its store has
// left.  The epilogue is a chain of latencies, 1200 clocks a chunk for its four
// warps (waits 330, TMEM 320, sums and shared memory 510), which the SM's
// second block fills; issuing the stores and waiting for them, 400 more, is a
// warp of its own.  (One block an SM with two sets of epilogue warps in turn
// needs both sets to see every phase of both rings, and was slower.)
// ---------------------------------------------------------------------------
constexpr int kChunk = 64;
constexpr int kMaxAcc = 3;          // accumulators in flight
constexpr int kUpThreads = 256;     // warp 0 base, 1 MMA + TMEM, 2 weights, 3-6 epilogue, 7 stores
constexpr int kUpEpi = 4;
constexpr uint32_t kUpTmem = 256;   // accumulators from column 0; h (hi, then lo, rp / 2 each) at the end

struct UpMaps {
  CUtensorMap base, out, w;
};
struct UpArgs {
  Rows rows;
  int room;        // bytes of shared memory for the rings
  int rp;
  int64_t chunks;  // of C
  int split;       // units of a span
  int64_t units;   // at most (spans without end, where the rows decrease, end there)
  int64_t cols, ldo;
  const __nv_bfloat16* h;  // [2][m][rp]
  __nv_bfloat16* out;
  int has_base;    // else the base is zero
  int in_place;    // out is base: spans without an adapter are done
  uint32_t* err;
};

__host__ __device__ constexpr int up_w_bytes(bool mn, int rp) { return mn ? rp * 128 : ((rp + 63) / 64) * 8192; }

struct Unit {
  Span span;
  int first, chunks;
  bool adapts;
  int live_boxes;
};

__device__ __forceinline__ Unit find_unit(const UpArgs& a, int64_t id, int lane) {
  Unit u;
  u.span = find_span<kRows>(a.rows, id / a.split, lane);
  const int part = int(id % a.split);
  u.first = int(a.chunks * part / a.split);
  u.chunks = int(a.chunks * (part + 1) / a.split) - u.first;
  u.adapts = u.span.slot >= 0;
  u.live_boxes = (u.span.count + kBox - 1) / kBox;
  if (!u.adapts && a.in_place) u.chunks = 0;
  return u;
}

// A place in a ring and the parity of the phase that comes next there.
struct Cursor {
  int at;
  uint32_t parity;
  __device__ __forceinline__ void next(int slots) {
    if (++at == slots) { at = 0; parity ^= 1u; }
  }
};

template <bool MN>
__global__ void __launch_bounds__(kUpThreads, 2) up_kernel(const __grid_constant__ UpMaps maps,
                                                           const __grid_constant__ UpArgs a) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* sm =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t y_full[kMaxStages], y_done[kMaxStages], y_empty[kMaxStages], w_full[kMaxStages], w_empty[kMaxStages];
  __shared__ uint64_t acc_full[kMaxAcc], acc_empty[kMaxAcc], h_full;
  __shared__ uint32_t tmem_slot;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // a slot of the base's ring holds a full span's chunk: boxes of 32 rows
  const int box_rows = a.rows.m >= kRows ? kRows / kBox : int((a.rows.m + kBox - 1) / kBox);
  const int y_bytes = box_rows * kBoxBytes, w_bytes = up_w_bytes(MN, a.rp);
  // three base chunks to two of the weights' at the most
  const int n_w = min(kMaxStages, a.room / (w_bytes + y_bytes + y_bytes / 2));
  const int n_y = min(kMaxStages, (a.room - n_w * w_bytes) / y_bytes);
  const int n_acc = a.rp <= 64 ? 3 : 2;
  unsigned char* ys = sm + n_w * w_bytes;

  if (threadIdx.x == 0) {
    for (int s = 0; s < n_y; ++s) { mbar_init(&y_full[s], 1); mbar_init(&y_done[s], kUpEpi); mbar_init(&y_empty[s], 1); }
    for (int s = 0; s < n_w; ++s) { mbar_init(&w_full[s], 1); mbar_init(&w_empty[s], 1); }
    for (int b = 0; b < n_acc; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], kUpEpi); }
    mbar_init(&h_full, kUpEpi);
    fence_barrier_init();
  }
  if (warp == 1) { tmem_alloc(&tmem_slot, kUpTmem); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot, h_tmem = tmem + kUpTmem - uint32_t(a.rp);

  if (warp == 0 || warp == 2) {
    // the base and the weights do not depend on the kernel before
    const bool weights = warp == 2;
    uint64_t* full = weights ? w_full : y_full;
    uint64_t* empty = weights ? w_empty : y_empty;
    const int slots = weights ? n_w : n_y;
    Cursor c{0, 1};
    int64_t issued = 0;
    bool ok = true;
    for (int64_t id = blockIdx.x; ok && id < a.units; id += gridDim.x) {
      const Unit u = find_unit(a, id, lane);
      if (u.span.count == 0) break;
      if (weights ? !u.adapts : !a.has_base) continue;
      if (elect_one()) {
        for (int i = 0; i < u.chunks; ++i) {
          if (!mbar_wait_bounded(&empty[c.at], c.parity)) {
            report_operator_timeout(a.err);
            ok = false;
            break;
          }
          const int32_t c0 = (u.first + i) * kChunk;
          if (weights) {
            unsigned char* w = sm + c.at * w_bytes;
            mbar_arrive_expect_tx(&full[c.at], uint32_t(w_bytes));
            if (MN) {
              tma_load_3d(w, &maps.w, &full[c.at], c0, 0, u.span.slot);
            } else {
              for (int r = 0; r < a.rp; r += 64) tma_load_3d(w + r * 128, &maps.w, &full[c.at], r, c0, u.span.slot);
            }
          } else {
            mbar_arrive_expect_tx(&full[c.at], uint32_t(u.live_boxes * kBoxBytes));
            for (int b = 0; b < u.live_boxes; ++b)
              tma_load_3d(ys + c.at * y_bytes + b * kBoxBytes, &maps.base, &full[c.at], c0,
                          int32_t(u.span.begin) + b * kBox, 0);
          }
          ++issued;
          c.next(slots);
        }
      }
      ok = __all_sync(0xffffffffu, ok);
    }
    if (elect_one())  // the copies in flight land before the block can end
      for (int64_t i = issued > slots ? issued - slots : 0; i < issued; ++i)
        mbar_wait_bounded(&full[i % slots], uint32_t((i / slots) & 1));
  } else if (warp == 1) {
    const uint32_t idesc = umma_idesc_bf16(128, kChunk, false, MN);
    Cursor w{0, 0}, c{0, 1};
    uint32_t h_parity = 0;
    bool ok = true;
    for (int64_t id = blockIdx.x; ok && id < a.units; id += gridDim.x) {
      const Unit u = find_unit(a, id, lane);
      if (u.span.count == 0) break;
      if (!u.adapts) continue;
      if (elect_one()) {
        ok = mbar_wait_bounded(&h_full, h_parity);
        for (int i = 0; i < u.chunks && ok; ++i) {
          if (!mbar_wait_bounded(&w_full[w.at], w.parity) || !mbar_wait_bounded(&acc_empty[c.at], c.parity)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t wd =
              umma_desc_sw128(smem_u32(sm + w.at * w_bytes), MN ? 8192 : 16, 1024);
          for (int t = 0; t < 2; ++t)
            for (int kk = 0; kk < a.rp / 16; ++kk) {
              const int w_off = MN ? kk * 2048 : (kk / 4) * 8192 + (kk % 4) * 32;
              mma_ts(tmem + uint32_t(c.at * kChunk), h_tmem + uint32_t(t * (a.rp / 2) + kk * 8),
                     wd + uint64_t(w_off >> 4), idesc, t > 0 || kk > 0 ? 1u : 0u);
            }
          tc_commit(&w_empty[w.at]);
          tc_commit(&acc_full[c.at]);
          w.next(n_w);
          c.next(n_acc);
        }
        if (!ok) report_operator_timeout(a.err);
      }
      h_parity ^= 1u;
      ok = __all_sync(0xffffffffu, ok);  // the elected lane's, the others' is true
    }
  } else if (warp == 7) {
    // full boxes leave by TMA; a slot is free when its boxes have left shared memory
    wait_for_predecessor();
    bool ok = true;
    Cursor y{0, 0};
    int before = -1;  // the slot whose stores may still read it
    for (int64_t id = blockIdx.x; ok && id < a.units; id += gridDim.x) {
      const Unit u = find_unit(a, id, lane);
      if (u.span.count == 0) break;
      if (elect_one()) {
        for (int i = 0; i < u.chunks; ++i) {
          if (!mbar_wait_bounded(&y_done[y.at], y.parity)) {
            report_operator_timeout(a.err);
            ok = false;
            break;
          }
          for (int b = 0; (b + 1) * kBox <= u.span.count; ++b)
            tma_store_3d(&maps.out, ys + y.at * y_bytes + b * kBoxBytes, (u.first + i) * kChunk,
                         int32_t(u.span.begin) + b * kBox, 0);
          bulk_commit();
          bulk_wait_read<1>();
          if (before >= 0) mbar_arrive(&y_empty[before]);
          before = y.at;
          y.next(n_y);
        }
      }
      ok = __all_sync(0xffffffffu, ok);
    }
    if (elect_one()) bulk_wait<0>();
  } else {
    const int q = warp & 3;
    const uint32_t lanes = uint32_t(q * 32) << 16;
    wait_for_predecessor();
    bool ok = true;
    Cursor y{0, a.has_base ? 0u : 1u}, c{0, 0};  // of the base's arrivals, or of the slots that are free
    uint64_t* ready = a.has_base ? y_full : y_empty;
    for (int64_t id = blockIdx.x; id < a.units; id += gridDim.x) {
      const Unit u = find_unit(a, id, lane);
      if (u.span.count == 0) break;
      const int live = min(max(u.span.count - q * kBox, 0), kBox);  // this warp's rows of the span
      if (u.adapts) {
        // h of the warp's rows, rows behind the span zero.  (The products of the unit before have ended: this warp
        // has waited for the last one's accumulator.)
        const __nv_bfloat16* row = a.h + (u.span.begin + q * kBox + lane) * a.rp;
        for (int t = 0; t < 2; ++t, row += a.rows.m * a.rp)
          for (int r = 0; r < a.rp; r += 32) {  // 16 columns of two values; rp is a multiple of 16
            uint32_t v[16];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint4 x = make_uint4(0u, 0u, 0u, 0u);
              if (lane < live && r + 8 * i < a.rp) x = *reinterpret_cast<const uint4*>(row + r + 8 * i);
              v[4 * i] = x.x; v[4 * i + 1] = x.y; v[4 * i + 2] = x.z; v[4 * i + 3] = x.w;
            }
            __syncwarp();
            const uint32_t at = h_tmem + lanes + uint32_t(t * (a.rp / 2) + r / 2);
            if (r + 32 <= a.rp) tmem_st16(at, v);
            else tmem_st8(at, v);
          }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&h_full);
      }
      for (int i = 0; i < u.chunks; ++i) {
        unsigned char* box = ys + y.at * y_bytes + q * kBoxBytes;
        if (ok) {
          ok = mbar_wait_bounded(&ready[y.at], y.parity) &&
               (!u.adapts || mbar_wait_bounded(&acc_full[c.at], c.parity));
          if (!ok) report_operator_timeout(a.err);
        }
        ok = __all_sync(0xffffffffu, ok);
        const int64_t c0 = int64_t(u.first + i) * kChunk, r0 = u.span.begin + q * kBox;
        const bool works = live > 0 && ok;
        if (works) {
          if (u.adapts || !a.has_base) {
            unsigned char* mine = box + lane * 128;  // the row's eight 16-byte vectors, swizzled
            uint32_t d[2][32];
            if (u.adapts) {
              tc_fence_after();
              const uint32_t t = tmem + lanes + uint32_t(c.at * kChunk);
              tmem_ld32(t, d[0]);
              tmem_ld32(t + 32, d[1]);
            } else {
#pragma unroll
              for (int e = 0; e < 32; ++e) d[0][e] = d[1][e] = 0u;
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              uint4 x[4];
#pragma unroll
              for (int v = 0; v < 4; ++v)
                x[v] = a.has_base ? *reinterpret_cast<uint4*>(mine + (((4 * e + v) ^ (lane & 7)) << 4))
                                  : make_uint4(0u, 0u, 0u, 0u);
              if (e == 0 && u.adapts) {
                tmem_wait_ld();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&acc_empty[c.at]);
              }
#pragma unroll
              for (int v = 0; v < 16; ++v) {
                uint32_t& w = reinterpret_cast<uint32_t*>(&x[v / 4])[v & 3];
                w = pack_bf16x2(__uint_as_float(w << 16) + __uint_as_float(d[e][2 * v]),
                                __uint_as_float(w & 0xFFFF0000u) + __uint_as_float(d[e][2 * v + 1]));
              }
#pragma unroll
              for (int v = 0; v < 4; ++v)
                *reinterpret_cast<uint4*>(mine + (((4 * e + v) ^ (lane & 7)) << 4)) = x[v];
            }
          }
          fence_proxy_async();  // the slot's next reader or writer is TMA
          __syncwarp();
          if (live < kBox)  // the box's other rows are another span's
            for (int r = lane >> 3; r < live; r += 4) {
              const int64_t col = c0 + (lane & 7) * 8;
              if (col < a.cols)
                *reinterpret_cast<uint4*>(a.out + (r0 + r) * a.ldo + col) =
                    *reinterpret_cast<uint4*>(box + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
            }
        } else if (lane == 0 && u.adapts) {
          mbar_arrive(&acc_empty[c.at]);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&y_done[y.at]);
        y.next(n_y);
        if (u.adapts) c.next(n_acc);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, kUpTmem);
}

// ---------------------------------------------------------------------------
// Few rows (single tokens of many requests): both products read the requests'
// weights once and do next to nothing with them, so what counts is how many
// loads are in flight.  On the tensor cores a span of one row still takes 128
// rows' epilogue, 1500 clocks for 8 KB of weights; here 24 single rows of
// 5120 -> 30720 at rank 64 (76 MB) take 33 us where they took 57 us.
// ---------------------------------------------------------------------------
// Rows of a span; 5120 -> 30720 at rank 64 with 2, 4 and 8: one request of 16 rows 14.3, 14.3 and 17.8 us, 64 requests of
// one row 63, 72 and 80; 1536 -> 8960 at rank 128, one request of 32 rows: 17.3, 15.1 and 18.3.
constexpr int kFewRows = 4;
constexpr int kFewMost = 64;        // rows of a call that may take this way: few_rows
constexpr int kFewRanks = 8;        // ranks of a down block
constexpr int kFewWarps = 8;
constexpr int kFewCols = 128;       // columns of an up block, one a thread

struct FewArgs {
  Rows rows;
  const __nv_bfloat16* x;
  const __nv_bfloat16* w;
  const __nv_bfloat16* base;
  __nv_bfloat16* h;  // [2][m][rp]
  __nv_bfloat16* out;
  int64_t ldx, ldbase, ldo, k, cols;
  int rank, rp, in_place;
};

__device__ __forceinline__ void unpack8(const uint4& r, float (&f)[8]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}

// h of a span (blockIdx.x) and 8 ranks (blockIdx.y).  The warps take every
// eighth 512 bytes of the rows of A and x, so a warp has eight rows' loads in
// flight at once (a warp a rank had four: 14.2 against 11.6 us);
// their sums meet in shared memory.
__global__ void __launch_bounds__(32 * kFewWarps) down_few_kernel(const __grid_constant__ FewArgs a) {
  __shared__ float part[kFewWarps][kFewRanks][kFewRows];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Span span = find_span<kFewRows>(a.rows, blockIdx.x, lane);
  dependents_may_start();
  if (span.count == 0 || span.slot < 0) return;
  const int r0 = int(blockIdx.y) * kFewRanks;
  float sum[kFewRanks][kFewRows] = {};
  if (r0 < a.rank) {  // a multiple of 8; the ranks that fill up to rp are zero
    const __nv_bfloat16* w = a.w + (int64_t(span.slot) * a.rank + r0) * a.k;
    const __nv_bfloat16* x = a.x + span.begin * a.ldx;
    for (int64_t c = warp * 256 + lane * 8; c < a.k; c += kFewWarps * 256) {
      uint4 f[kFewRanks], v[kFewRows];
#pragma unroll
      for (int r = 0; r < kFewRanks; ++r) f[r] = *reinterpret_cast<const uint4*>(w + r * a.k + c);
#pragma unroll
      for (int i = 0; i < kFewRows; ++i)
        if (i < span.count) v[i] = *reinterpret_cast<const uint4*>(x + i * a.ldx + c);
#pragma unroll
      for (int i = 0; i < kFewRows; ++i) {
        if (i >= span.count) break;
        float xv[8];
        unpack8(v[i], xv);
#pragma unroll
        for (int r = 0; r < kFewRanks; ++r) {
          float fv[8];
          unpack8(f[r], fv);
#pragma unroll
          for (int e = 0; e < 8; ++e) sum[r][i] = fmaf(fv[e], xv[e], sum[r][i]);
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < kFewRanks; ++r)
#pragma unroll
    for (int i = 0; i < kFewRows; ++i) {
      if (i >= span.count) break;
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) sum[r][i] += __shfl_xor_sync(0xffffffffu, sum[r][i], off);
      if (lane == 0) part[warp][r][i] = sum[r][i];
    }
  __syncthreads();
  if (threadIdx.x < kFewRanks * kFewRows) {
    const int r = threadIdx.x / kFewRows, i = threadIdx.x % kFewRows;
    if (i < span.count) {
      float total = 0.f;
#pragma unroll
      for (int w = 0; w < kFewWarps; ++w) total += part[w][r][i];
      uint32_t hi, lo;
      split2((a.rows.scale ? a.rows.scale[span.slot] : 1.f) * total, 0.f, hi, lo);
      __nv_bfloat16* h = a.h + (span.begin + i) * a.rp + r0 + r;
      *reinterpret_cast<uint16_t*>(h) = uint16_t(hi);
      *reinterpret_cast<uint16_t*>(h + a.rows.m * a.rp) = uint16_t(lo);
    }
  }
}

// out of a span (blockIdx.y) and 128 columns (blockIdx.x): the columns' rows of
// B, which lie one behind the other, go through shared memory (a thread's row 16
// bytes further than the one before, so that its 16-byte reads meet no other's
// bank).
__global__ void __launch_bounds__(kFewCols) up_few_kernel(const __grid_constant__ FewArgs a) {
  extern __shared__ uint4 few_smem[];
  __shared__ float h[kFewRows][kMaxRank];
  const int tid = threadIdx.x;
  const Span span = find_span<kFewRows>(a.rows, blockIdx.y, tid & 31);
  if (span.count == 0 || (span.slot < 0 && a.in_place)) {
    wait_for_predecessor();  // this grid does not end before the one that it depends on
    return;
  }
  const int64_t c0 = int64_t(blockIdx.x) * kFewCols, col = c0 + tid;
  const int vecs = a.rank / 8, pitch = vecs + 1;
  const int live = int(a.cols - c0 < kFewCols ? a.cols - c0 : kFewCols);
  if (span.slot >= 0) {
    const uint4* src = reinterpret_cast<const uint4*>(a.w + (int64_t(span.slot) * a.cols + c0) * a.rank);
    for (int i = tid; i < live * vecs; i += kFewCols)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                   :: "r"(smem_u32(few_smem + (i / vecs) * pitch + i % vecs)), "l"(src + i) : "memory");
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  float acc[kFewRows];
#pragma unroll
  for (int i = 0; i < kFewRows; ++i)
    acc[i] = i < span.count && col < a.cols ? __bfloat162float(a.base[(span.begin + i) * a.ldbase + col]) : 0.f;
  wait_for_predecessor();
  if (span.slot >= 0) {
    for (int i = tid; i < span.count * a.rank; i += kFewCols) {
      const int row = i / a.rank, r = i - row * a.rank;
      const __nv_bfloat16* src = a.h + (span.begin + row) * a.rp + r;
      h[row][r] = __bfloat162float(*src) + __bfloat162float(src[a.rows.m * a.rp]);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    if (col < a.cols) {
      float sum[kFewRows] = {};
      for (int v = 0; v < vecs; ++v) {
        float f[8];
        unpack8(few_smem[tid * pitch + v], f);
#pragma unroll
        for (int i = 0; i < kFewRows; ++i) {
          if (i >= span.count) break;
#pragma unroll
          for (int e = 0; e < 8; ++e) sum[i] = fmaf(f[e], h[i][8 * v + e], sum[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < kFewRows; ++i) acc[i] += sum[i];
    }
  }
#pragma unroll
  for (int i = 0; i < kFewRows; ++i)
    if (i < span.count && col < a.cols) a.out[(span.begin + i) * a.ldo + col] = __float2bfloat16_rn(acc[i]);
}

// ---------------------------------------------------------------------------
// grad: for each adapter, d[C, R] = sum over its rows of u[row, C]^T h[row, R]:
// dA = (x, g) and dB = (dy, h) in one launch.
//
// The rows go by in stages of 32 (64 above rank 64) of one request, adapter by
// adapter; the list of all stages is cut into equal shares, so adapters of very
// different numbers of rows keep all SMs busy.  A block owns 512 columns (256
// above rank 64) of x or of dy and one share; where its share passes from one
// adapter to the next it puts down what it has summed.  An adapter that lies in
// one share is written at once; the others' sums, two a share at most (of the
// adapter that it begins in and of the one that it ends in), go to the workspace
// and a second kernel adds them in the order of the shares.
//
// A stage's rows behind the request's last are zeroed in shared memory: they
// hold another request's values, which may be NaN.  hi and lo sit side by side
// as the columns of one operand, so 16 rows and 128 columns are one MMA of
// N = 128 (256 above rank 64); the two halves are added at the end.  h is read
// again by every column block, which is why a block is as wide as TMEM allows.
// ---------------------------------------------------------------------------
constexpr int kMaxAdapters = 4096;
__host__ __device__ constexpr int grad_cols(int atoms) { return atoms == 1 ? 512 : 256; }
__host__ __device__ constexpr int grad_rows(int atoms) { return atoms == 1 ? 32 : 64; }

struct GradMaps {
  CUtensorMap u[2], h[2];
};
struct GradArgs {
  Rows rows;
  Ring ring;
  int rank, atoms;
  int problem0;                // the first problem computed (0: dA, 1: dB)
  int64_t cols[2], blocks[2];  // columns and column blocks
  int shares;
  float* partial;         // [shares][2][rank * cols] for each problem
  __nv_bfloat16* out[2];  // [adapters][rank][cols], [adapters][cols][rank]
  uint32_t* err;
};

// Stages of request q, and the adapter that they belong to (-1: none).
__device__ __forceinline__ int request_stages(const Rows& a, int q, int stage_rows, int& slot, int64_t& begin,
                                              int64_t& end) {
  slot = -1;
  begin = end = 0;
  if (q >= a.requests) return 0;
  const int s = a.slots[q];
  if (s < 0 || s >= a.adapters) return 0;
  begin = a.rows[q];
  end = a.rows[q + 1];
  if (begin < 0) begin = 0;
  if (end > a.m) end = a.m;
  if (end <= begin) return 0;
  slot = s;
  return int((end - begin + stage_rows - 1) / stage_rows);
}

// All stages, from their sum over the requests; none where the rows decrease and there are more than there can be.
__device__ __forceinline__ int total_stages(const Rows& a, int stage_rows, unsigned long long sum) {
  return sum <= (unsigned long long)((a.m + stage_rows - 1) / stage_rows + a.requests) ? int(sum) : 0;
}

// First stage of a share, of `total`.
__device__ __forceinline__ int share_begin(int total, int share, int shares) {
  return int(int64_t(total) * share / shares);
}

// The part of a share that belongs to one adapter: its stages [first, first + count) of that adapter.
struct Piece {
  int slot, first, count;
  int base;    // stages of the adapters before
  bool whole;  // all of the adapter's
};

// The place of the sums that share `share`, which begins at stage g0, has of an adapter with `base` stages before it and
// more in other shares: such an adapter is the one that the share begins in, or else the one that it ends in.
__device__ __forceinline__ int64_t partial_index(int share, int base, int g0) {
  return int64_t(share) * 2 + (base > g0 ? 1 : 0);
}

// The piece of the share [g0, g1) behind `after` (slot -1, base 0: the first); count 0: there is none.  All lanes.
__device__ __forceinline__ Piece next_piece(const int* stages, int adapters, int g0, int g1, const Piece& after,
                                            int lane) {
  Piece p{-1, 0, 0, after.base, false};
  int from = after.slot + 1;
  if (after.slot >= 0) p.base += stages[after.slot];
  for (; from < adapters && p.base < g1; from += 32) {
    const int own = from + lane < adapters ? stages[from + lane] : 0;
    int upto = own;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= off) upto += v;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, own > 0 && p.base + upto > g0);
    if (hit != 0) {
      const int src = __ffs(int(hit)) - 1;
      const int n = __shfl_sync(0xffffffffu, own, src);
      p.base += __shfl_sync(0xffffffffu, upto, src) - n;
      p.slot = from + src;
      p.first = max(g0 - p.base, 0);
      p.count = max(min(g1 - p.base, n) - p.first, 0);
      p.whole = p.count == n;
      return p;
    }
    p.base += __shfl_sync(0xffffffffu, upto, 31);
  }
  return p;
}

__global__ void __launch_bounds__(kThreads) grad_kernel(const __grid_constant__ GradMaps maps,
                                                        const __grid_constant__ GradArgs a) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* sm =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  int* stages = reinterpret_cast<int*>(sm + a.ring.stages * a.ring.stage_bytes);  // [adapters]
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages], acc_full, acc_empty;
  __shared__ uint32_t tmem_slot;
  __shared__ int valid[kMaxStages];  // rows of a stage that are the request's
  __shared__ unsigned long long sum;  // of the requests' stages
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int width = grad_cols(a.atoms), stage_rows = grad_rows(a.atoms), box = stage_rows * 128;
  int64_t id = blockIdx.x;
  int problem = a.problem0;
  if (problem == 0 && id >= a.blocks[0] * a.shares) { id -= a.blocks[0] * a.shares; problem = 1; }
  const int64_t col0 = (id % a.blocks[problem]) * width;
  const int share = int(id / a.blocks[problem]);
  const int n = 128 * a.atoms;                // accumulator columns of 128 matrix columns: hi, then lo
  constexpr uint32_t cols = 512;

  if (threadIdx.x == 0) {
    for (int s = 0; s < a.ring.stages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    mbar_init(&acc_full, 1);
    mbar_init(&acc_empty, 4);
    fence_barrier_init();
    sum = 0;
  }
  for (int s = int(threadIdx.x); s < a.rows.adapters; s += kThreads) stages[s] = 0;
  if (warp == 1) { tmem_alloc(&tmem_slot, cols); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  for (int q = int(threadIdx.x); q < a.rows.requests; q += kThreads) {
    int slot;
    int64_t begin, end;
    const int own = request_stages(a.rows, q, stage_rows, slot, begin, end);
    if (own > 0) { atomicAdd(&stages[slot], own); atomicAdd(&sum, (unsigned long long)own); }
  }
  __syncthreads();
  const uint32_t tmem = tmem_slot;
  const int total = total_stages(a.rows, stage_rows, sum);
  const int g0 = share_begin(total, share, a.shares), g1 = share_begin(total, share + 1, a.shares);
  const Piece none{-1, 0, 0, 0, false};

  if (warp == 0) {
    // all lanes look for the pieces' requests, one issues
    Cursor c{0, 1};
    int issued = 0;
    bool ok = true;
    for (Piece p = next_piece(stages, a.rows.adapters, g0, g1, none, lane); p.count > 0 && ok;
         p = next_piece(stages, a.rows.adapters, g0, g1, p, lane)) {
      int base = 0, done = 0;  // the adapter's stages in the requests so far; the piece's stages so far
      for (int q0 = 0; q0 < a.rows.requests && done < p.count && ok; q0 += 32) {
        int64_t begin, end;
        int slot;
        int own = request_stages(a.rows, q0 + lane, stage_rows, slot, begin, end);
        if (slot != p.slot) own = 0;
        int upto = own;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, upto, off);
          if (lane >= off) upto += v;
        }
        for (uint32_t left = __ballot_sync(0xffffffffu, own > 0); left != 0 && done < p.count && ok;
             left &= left - 1) {
          const int src = __ffs(int(left)) - 1;
          const int count = __shfl_sync(0xffffffffu, own, src);
          const int before = base + __shfl_sync(0xffffffffu, upto, src) - count;
          const int64_t r0 = __shfl_sync(0xffffffffu, begin, src), r1 = __shfl_sync(0xffffffffu, end, src);
          for (int t = max(0, p.first + done - before); t < count && done < p.count && ok; ++t, ++done) {
            ok = mbar_wait_bounded(&empty[c.at], c.parity);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            if (elect_one()) {
              const int64_t row = r0 + int64_t(t) * stage_rows;
              unsigned char* st = sm + c.at * a.ring.stage_bytes;
              valid[c.at] = int(r1 - row < stage_rows ? r1 - row : stage_rows);
              mbar_arrive_expect_tx(&full[c.at], uint32_t(a.ring.stage_bytes));
              for (int x = 0; x < width / 64; ++x)
                tma_load_3d(st + x * box, &maps.u[problem], &full[c.at], int32_t(col0) + x * 64, int32_t(row), 0);
              for (int x = 0; x < 2 * a.atoms; ++x)
                tma_load_3d(st + (width / 64 + x) * box, &maps.h[problem], &full[c.at], (x % a.atoms) * 64,
                            int32_t(row), x / a.atoms);
            }
            __syncwarp();
            ++issued;
            c.next(a.ring.stages);
          }
        }
        base += __shfl_sync(0xffffffffu, upto, 31);
      }
    }
    if (!ok && lane == 0) report_operator_timeout(a.err);
    for (int j = issued > a.ring.stages ? issued - a.ring.stages : 0; j < issued; ++j)
      mbar_wait_bounded(&full[j % a.ring.stages], uint32_t((j / a.ring.stages) & 1));
  } else if (warp == 1) {
    const uint32_t idesc = umma_idesc_bf16(128, n, true, true);
    Cursor c{0, 0};
    uint32_t acc_parity = 1;
    bool ok = true;
    for (Piece p = next_piece(stages, a.rows.adapters, g0, g1, none, lane); p.count > 0 && ok;
         p = next_piece(stages, a.rows.adapters, g0, g1, p, lane)) {
      ok = __all_sync(0xffffffffu, mbar_wait_bounded(&acc_empty, acc_parity));
      acc_parity ^= 1u;
      for (int i = 0; i < p.count && ok; ++i) {
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(&full[c.at], c.parity));
        if (!ok) break;
        unsigned char* st = sm + c.at * a.ring.stage_bytes;
        const int rows = valid[c.at];
        if (rows < stage_rows) {  // zero the other rows of every box
          const int boxes = width / 64 + 2 * a.atoms;
          for (int b = 0; b < boxes; ++b)
            for (int at = rows * 128 + lane * 16; at < box; at += 512)
              *reinterpret_cast<uint4*>(st + b * box + at) = make_uint4(0u, 0u, 0u, 0u);
          fence_proxy_async();
          __syncwarp();
        }
        if (elect_one()) {
          tc_fence_after();
          const uint64_t ud = umma_desc_sw128(smem_u32(st), uint32_t(box), 1024);
          const uint64_t hd = umma_desc_sw128(smem_u32(st) + uint32_t(width / 64 * box), uint32_t(box), 1024);
          for (int x = 0; x < width / 128; ++x)
            for (int kk = 0; kk < stage_rows / 16; ++kk)
              mma_ss(tmem + uint32_t(x * n), ud + uint64_t((x * 2 * box + kk * 2048) >> 4),
                     hd + uint64_t((kk * 2048) >> 4), idesc, i > 0 || kk > 0 ? 1u : 0u);
          tc_commit(&empty[c.at]);
          if (i == p.count - 1) tc_commit(&acc_full);
        }
        __syncwarp();
        c.next(a.ring.stages);
      }
    }
    if (!ok && lane == 0) report_operator_timeout(a.err);
  } else {
    const int q = warp & 3;
    const int64_t size = int64_t(a.rank) * a.cols[problem];
    uint32_t acc_parity = 0;
    for (Piece p = next_piece(stages, a.rows.adapters, g0, g1, none, lane); p.count > 0;
         p = next_piece(stages, a.rows.adapters, g0, g1, p, lane)) {
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(&acc_full, acc_parity))) {
        if (lane == 0) report_operator_timeout(a.err);
        break;
      }
      acc_parity ^= 1u;
      tc_fence_after();
      float* partial = a.partial + (problem == 1 && a.problem0 == 0 ? int64_t(a.shares) * 2 * a.rank * a.cols[0] : 0) +
                       partial_index(share, p.base, g0) * size;
      __nv_bfloat16* out = a.out[problem] + int64_t(p.slot) * size;
      for (int x = 0; x < width / 128; ++x) {
        const int64_t col = col0 + x * 128 + q * 32 + lane;
        for (int r0 = 0; r0 < a.rank; r0 += 16) {
          uint32_t hi[16], lo[16];
          __syncwarp();
          const uint32_t t = tmem + (uint32_t(q * 32) << 16) + uint32_t(x * n + r0);
          tmem_ld16(t, hi);
          tmem_ld16(t + uint32_t(n / 2), lo);
          tmem_wait_ld();
          float v[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(hi[i]) + __uint_as_float(lo[i]);
          if (col < a.cols[problem]) {
#pragma unroll
            for (int i = 0; i < 16; i += 8) {
              if (r0 + i >= a.rank) continue;  // a multiple of 8
              if (problem == 0) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                  const int64_t at = int64_t(r0 + i + e) * a.cols[0] + col;
                  if (p.whole) out[at] = __float2bfloat16_rn(v[i + e]);
                  else partial[at] = v[i + e];
                }
              } else {
                const int64_t at = col * a.rank + r0 + i;
                if (p.whole) {
                  *reinterpret_cast<uint4*>(out + at) =
                      make_uint4(pack_bf16x2(v[i], v[i + 1]), pack_bf16x2(v[i + 2], v[i + 3]),
                                 pack_bf16x2(v[i + 4], v[i + 5]), pack_bf16x2(v[i + 6], v[i + 7]));
                } else {
                  *reinterpret_cast<float4*>(partial + at) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                  *reinterpret_cast<float4*>(partial + at + 4) = make_float4(v[i + 4], v[i + 5], v[i + 6], v[i + 7]);
                }
              }
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, cols);
}

// The adapters (blockIdx.y) whose stages lie in several shares: out = bf16(sum
// over the shares, in order); and zero for those without rows.  8 values a
// thread, dA's and then dB's.
struct SumArgs {
  Rows rows;
  int stage_rows, shares;
  const float* partial;
  int64_t size[2];  // of one adapter; 0: not computed
  __nv_bfloat16* out[2];
};

__global__ void __launch_bounds__(256) grad_sum_kernel(const __grid_constant__ SumArgs a) {
  __shared__ int before, mine;
  __shared__ unsigned long long all;
  const int adapter = int(blockIdx.y);
  if (threadIdx.x == 0) { before = mine = 0; all = 0; }
  __syncthreads();
  int sum[2] = {0, 0};
  unsigned long long own_all = 0;
  for (int q = int(threadIdx.x); q < a.rows.requests; q += 256) {
    int slot;
    int64_t begin, end;
    const int own = request_stages(a.rows, q, a.stage_rows, slot, begin, end);
    if (own > 0) {
      own_all += own;
      if (slot < adapter) sum[0] += own;
      if (slot == adapter) sum[1] += own;
    }
  }
  if (own_all > 0) { atomicAdd(&before, sum[0]); atomicAdd(&mine, sum[1]); atomicAdd(&all, own_all); }
  __syncthreads();
  const int total = total_stages(a.rows, a.stage_rows, all);
  int first = 0, last = -1;  // the shares of the adapter's first and last stage
  if (total > 0 && mine > 0) {
    while (share_begin(total, first + 1, a.shares) <= before) ++first;
    last = first;
    while (share_begin(total, last + 1, a.shares) < before + mine) ++last;
    if (first == last) return;  // written whole
  }
  int64_t i = (int64_t(blockIdx.x) * 256 + threadIdx.x) * 8;
  const float* partial = a.partial;
  int problem = 0;
  if (i >= a.size[0]) {
    i -= a.size[0];
    partial += int64_t(a.shares) * 2 * a.size[0];
    problem = 1;
    if (i >= a.size[1]) return;
  }
  float v[8] = {};
  for (int share = first; share <= last; ++share) {
    // (a share without stages of its own, when there are fewer stages than shares, wrote nothing)
    const int g0 = share_begin(total, share, a.shares);
    if (g0 == share_begin(total, share + 1, a.shares)) continue;
    const float4* src = reinterpret_cast<const float4*>(partial + partial_index(share, before, g0) * a.size[problem] + i);
    const float4 x = src[0], y = src[1];
    v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
    v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
  }
  *reinterpret_cast<uint4*>(a.out[problem] + adapter * a.size[problem] + i) =
      make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
// bf16 [batch][rows][cols], row stride ld; a box of 64 x box_rows, 128-byte swizzle.
bool make_map(CUtensorMap* m, const void* base, int64_t cols, int64_t rows, int64_t batch, int64_t ld,
              int box_rows) {
  const auto fn = tensor_map_encoder();
  if (!fn) return false;
  const cuuint64_t dims[3] = {cuuint64_t(cols), cuuint64_t(rows), cuuint64_t(batch)};
  const cuuint64_t strides[2] = {cuuint64_t(ld) * 2, cuuint64_t(rows) * cuuint64_t(ld) * 2};
  const cuuint32_t box[3] = {64u, cuuint32_t(box_rows), 1u};
  const cuuint32_t step[3] = {1u, 1u, 1u};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, step,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

Ring ring_of(int stage_bytes, int room) {
  int stages = room / stage_bytes;
  if (stages > kMaxStages) stages = kMaxStages;
  return Ring{stages, stage_bytes};
}

// Lets a kernel have `bytes` (the same for every call) of shared memory; once for each device.
template <auto kKernel>
cudaError_t allow_smem(int bytes) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if (e != cudaSuccess || (done.load(std::memory_order_acquire) & bit)) return e;
  e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return e;
}

// at most: every segment ends one
int64_t span_count(const Rows& r) { return cdiv(r.m, kRows) + r.requests + 1; }
// spans that have rows, about: every request ends one, at most one a row
int64_t busy_spans(const Rows& r) {
  const int64_t most = cdiv(r.m, kRows) + (r.requests > 0 ? r.requests - 1 : 0);
  return most < r.m ? most : r.m;
}

struct Matrix {
  const void* p;
  int64_t ld;
};

template <bool MN>
cudaError_t down(cudaStream_t st, const Rows& r, Matrix u, int64_t c, const void* w, int rank, __nv_bfloat16* h,
                 int sms, uint32_t* err) {
  DownMaps maps;
  DownArgs a{};
  a.rank = rank;
  a.rp = int(cdiv(rank, 16)) * 16;
  if (!make_map(&maps.u, u.p, c, r.m, 1, u.ld, kBox)) return cudaErrorInvalidValue;
  if (!(MN ? make_map(&maps.w, w, rank, c, r.adapters, rank, 64)
           : make_map(&maps.w, w, c, rank, r.adapters, c, a.rp)))
    return cudaErrorInvalidValue;
  a.rows = r;
  a.room = kSmemTwo - 2048;
  a.steps = cdiv(c, 64);
  a.h = h;
  a.err = err;
  // few rows: K is split while that still adds blocks that find an SM free
  a.split = 1;
  while (a.split < 8 && busy_spans(r) * a.split * 2 <= 2 * sms && a.steps >= a.split * 4) a.split *= 2;
  const int smem = a.room + 1024;
  cudaError_t e = allow_smem<down_kernel<MN>>(smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(span_count(r) * a.split));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = size_t(smem);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = unsigned(a.split);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, down_kernel<MN>, maps, a);
}

template <bool MN>
cudaError_t up(cudaStream_t st, const Rows& r, const __nv_bfloat16* h, const void* w, int rank, int64_t c,
               Matrix base, Matrix out, int sms, uint32_t* err) {
  UpMaps maps;
  UpArgs a{};
  a.rp = int(cdiv(rank, 16)) * 16;
  if (!make_map(&maps.out, out.p, c, r.m, 1, out.ld, kBox)) return cudaErrorInvalidValue;
  if (base.p == nullptr) maps.base = maps.out;
  else if (!make_map(&maps.base, base.p, c, r.m, 1, base.ld, kBox)) return cudaErrorInvalidValue;
  if (!(MN ? make_map(&maps.w, w, c, rank, r.adapters, c, a.rp)
           : make_map(&maps.w, w, rank, c, r.adapters, rank, kChunk)))  // 64 ranks of 128 columns
    return cudaErrorInvalidValue;
  a.rows = r;
  a.room = kSmemTwo - 2048;
  a.h = h;
  a.chunks = cdiv(c, kChunk);
  a.cols = c;
  a.ldo = out.ld;
  a.out = static_cast<__nv_bfloat16*>(const_cast<void*>(out.p));
  a.has_base = base.p != nullptr;
  a.in_place = base.p == out.p;
  a.err = err;
  // Units of a span: those with which the block that has most to do is done
  // first.  A unit costs its chunks and the time of about two more until its h
  // is in TMEM; blocks that are as good as equal still end up to one unit apart.
  double best = 0.0;
  for (int64_t split = 1; split <= a.chunks && split <= 8 * sms; ++split) {
    const double time =
        (double(cdiv(busy_spans(r) * split, 2 * sms)) + 0.5) * (double(cdiv(a.chunks, split)) + 2.0);
    if (split == 1 || time < best * 0.98) { best = time; a.split = int(split); }
  }
  a.units = span_count(r) * a.split;
  const int smem = a.room + 1024;
  cudaError_t e = allow_smem<up_kernel<MN>>(smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(a.units < 2 * sms ? a.units : 2 * sms));
  cfg.blockDim = dim3(kUpThreads);
  cfg.dynamicSmemBytes = size_t(smem);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, up_kernel<MN>, maps, a);
}

// Whether a call takes the kernels for few rows.  They read an adapter's weights for every four rows of a request, the
// others for every 128, and take 6 us less to begin with; what a read costs beside is fitted to the times of 1 to 128
// rows.  (us, here / there.  5120 -> 30720, rank 64: one request of 16, 24 and 64 rows 14.3 / 16.2, 17.2 / 16.8 and
// 28.8 / 17.1, 16 and 64 requests of one row 21 / 41 and 72 / 120.  1536 -> 8960, rank 128: 24, 32 and 64 rows 14.8 /
// 14.9, 15.1 / 15.5 and 26 / 16.7; 64 and 128 requests 50 / 48 and 98 / 90.  5120 -> 5120, rank 16: one request of 64
// rows 9.2 / 13.5, 64 requests 13 / 35.)  The requests' lengths are not known here: they are taken to be equal.
bool few_rows(const Rows& r, int64_t k, int64_t n, int rank) {
  if (r.m > kFewMost) return false;
  const double mb = double(rank) * double(k + n) * 2e-6;
  const int64_t requests = r.requests < 1 ? 1 : r.requests < r.m ? r.requests : r.m;
  const int64_t reads = requests * cdiv(cdiv(r.m, requests), kFewRows);
  return 0.35 * mb * double(reads) <= 6.0 + double(requests) * (0.3 + 0.3 * mb);
}

unsigned few_spans(const Rows& r) {
  const int64_t spans = cdiv(r.m, kFewRows) + r.requests + 1;
  return unsigned(spans < r.m ? spans : r.m);  // every span has a row
}

FewArgs few_args(const Rows& r, int rank, __nv_bfloat16* h, const void* w) {
  FewArgs a{};
  a.rows = r;
  a.rank = rank;
  a.rp = int(cdiv(rank, 16)) * 16;
  a.h = h;
  a.w = static_cast<const __nv_bfloat16*>(w);
  return a;
}

cudaError_t down_few(cudaStream_t st, const Rows& r, Matrix x, int64_t k, const void* w, int rank, __nv_bfloat16* h) {
  FewArgs a = few_args(r, rank, h, w);
  a.x = static_cast<const __nv_bfloat16*>(x.p);
  a.ldx = x.ld;
  a.k = k;
  down_few_kernel<<<dim3(few_spans(r), unsigned(a.rp / kFewRanks)), 32 * kFewWarps, 0, st>>>(a);
  return cudaGetLastError();
}

cudaError_t up_few(cudaStream_t st, const Rows& r, __nv_bfloat16* h, const void* w, int rank, int64_t n, Matrix y,
                   Matrix out) {
  FewArgs a = few_args(r, rank, h, w);
  a.base = static_cast<const __nv_bfloat16*>(y.p);
  a.out = static_cast<__nv_bfloat16*>(const_cast<void*>(out.p));
  a.ldbase = y.ld;
  a.ldo = out.ld;
  a.cols = n;
  a.in_place = y.p == out.p;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(cdiv(n, kFewCols)), few_spans(r));
  cfg.blockDim = dim3(kFewCols);
  cfg.dynamicSmemBytes = size_t(kFewCols) * size_t(rank / 8 + 1) * 16;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, up_few_kernel, a);
}

// h of x, the same wherever it is computed.
cudaError_t down_a(cudaStream_t st, const Rows& r, Matrix x, int64_t k, int64_t n, const void* a, int rank,
                   __nv_bfloat16* h, int sms, uint32_t* err) {
  return few_rows(r, k, n, rank) ? down_few(st, r, x, k, a, rank, h) : down<false>(st, r, x, k, a, rank, h, sms, err);
}

int64_t grad_blocks(int64_t c, int rank) { return cdiv(c, grad_cols(rank <= 64 ? 1 : 2)); }

// Shares of the rows, of 1 to 3 waves of blocks (a block takes an SM for
// itself): those with the least time, counted in stages.  Every request ends a
// stage.  A block takes as long as about six more for every adapter that it
// puts down, and every share is read again by the second kernel.  (20 column
// blocks and 1024 stages: 7 shares take 127 us, 22 take 146 us; 27 rows of 16
// adapters, 240 and 224 columns, rank 120: 8 shares take 24 us, one 153 us.)
int grad_shares(int64_t m, int64_t blocks, int rank, int64_t adapters, int64_t requests, int sms) {
  const int64_t busy = requests < m ? requests : m, pieces = busy < adapters ? busy : adapters;
  const double stages = double(m) / double(grad_rows(rank <= 64 ? 1 : 2)) + double(busy) * 0.5;
  int64_t best = 1;
  double best_time = 0.0;
  for (int64_t shares = 1; shares == 1 || (blocks * shares <= 3 * sms && double(shares) <= stages); ++shares) {
    const double put = 6.0 * double(cdiv(pieces, shares)) + (shares > 1 ? 6.0 : 0.0) * double(pieces > 1);
    const double time =
        double(cdiv(blocks * shares, sms)) * (stages / double(shares) + put) + 0.5 * double(shares > 1 ? shares : 0);
    if (shares == 1 || time < best_time) { best = shares; best_time = time; }
  }
  return int(best);
}

size_t grad_partial_bytes(int64_t m, int64_t k, int64_t n, int rank, int64_t adapters, int64_t requests, int sms) {
  const int64_t shares = grad_shares(m, grad_blocks(k, rank) + grad_blocks(n, rank), rank, adapters, requests, sms);
  return shares > 1 ? size_t(shares) * 2 * size_t(rank) * size_t(k + n) * 4 : 0;
}

cudaError_t grad(cudaStream_t st, const Rows& r, int rank, Matrix x, int64_t k, Matrix dy, int64_t n,
                 const __nv_bfloat16* g, const __nv_bfloat16* h, void* da, void* db, void* workspace, int sms,
                 uint32_t* err) {
  GradMaps maps;
  GradArgs a{};
  const int rp = int(cdiv(rank, 16)) * 16;
  a.atoms = rp <= 64 ? 1 : 2;
  const int rows = grad_rows(a.atoms);
  if (!make_map(&maps.u[0], x.p, k, r.m, 1, x.ld, rows) || !make_map(&maps.u[1], dy.p, n, r.m, 1, dy.ld, rows) ||
      !make_map(&maps.h[0], g, rp, r.m, 2, rp, rows) || !make_map(&maps.h[1], h, rp, r.m, 2, rp, rows))
    return cudaErrorInvalidValue;
  a.rows = r;
  a.rank = rank;
  const int list = int(cdiv(r.adapters, 256)) * 1024;  // the adapters' stages in shared memory
  a.ring = ring_of((grad_cols(a.atoms) / 64 + 2 * a.atoms) * rows * 128, 2 * kSmemTwo - 2048 - list);
  a.problem0 = da ? 0 : 1;
  a.cols[0] = k;
  a.cols[1] = n;
  a.blocks[0] = grad_blocks(k, rank);
  a.blocks[1] = grad_blocks(n, rank);
  const int64_t blocks = (da ? a.blocks[0] : 0) + (db ? a.blocks[1] : 0);
  a.shares = grad_shares(r.m, grad_blocks(k, rank) + grad_blocks(n, rank), rank, r.adapters, r.requests, sms);
  a.partial = static_cast<float*>(workspace);
  a.out[0] = static_cast<__nv_bfloat16*>(da);
  a.out[1] = static_cast<__nv_bfloat16*>(db);
  a.err = err;
  const int smem = a.ring.stages * a.ring.stage_bytes + list + 1024;
  cudaError_t e = allow_smem<grad_kernel>(2 * kSmemTwo);
  if (e != cudaSuccess) return e;
  grad_kernel<<<unsigned(blocks * a.shares), kThreads, smem, st>>>(maps, a);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  SumArgs sum{r, rows, a.shares, a.partial, {da ? rank * k : 0, db ? rank * n : 0}, {a.out[0], a.out[1]}};
  const dim3 grid(unsigned(cdiv((sum.size[0] + sum.size[1]) / 8, 256)), unsigned(r.adapters));
  grad_sum_kernel<<<grid, 256, 0, st>>>(sum);
  return cudaGetLastError();
}

bool misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

int check(int64_t m, int64_t k, int64_t n, int rank, int64_t adapters, int64_t requests) {
  if (m < 0 || k < 1 || n < 1 || adapters < 1 || requests < 0) return PASA_ERR_SHAPE;
  if (k % 8 || n % 8 || rank < 8 || rank > kMaxRank || rank % 8) return PASA_ERR_SHAPE;
  if (m > (int64_t(1) << 30) || k > (1 << 24) || n > (1 << 24) || adapters > kMaxAdapters || requests > (1 << 20))
    return PASA_ERR_SHAPE;
  return PASA_OK;
}

int check_matrix(const void* p, int64_t ld, int64_t cols) {
  if (!p) return PASA_ERR_NULL;
  if (misaligned(p)) return PASA_ERR_ALIGN;
  return ld < cols || ld % 8 || ld > (int64_t(1) << 32) ? PASA_ERR_SHAPE : PASA_OK;
}

int device_sms(int* sms) {
  int dev = 0, major = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess ||
      cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return PASA_ERR_CUDA;
  return major == 10 ? PASA_OK : PASA_ERR_DEVICE;
}

}  // namespace lora
}  // namespace pasa

using namespace pasa;

extern "C" {

int pasa_lora_h_size(int64_t m, int rank, size_t* bytes) {
  if (!bytes) return PASA_ERR_NULL;
  const int st = lora::check(m, 8, 8, rank, 1, 0);
  if (st) return st;
  *bytes = size_t(2 * m) * size_t(cdiv(rank, 16) * 16) * 2;
  return PASA_OK;
}

int pasa_lora_update(void* stream, const void* x, int64_t ldx, const void* y, int64_t ldy, const void* a,
                     const void* b, const float* scale, int64_t m, int64_t k, int64_t n, int rank, int64_t adapters,
                     const int32_t* rows, const int32_t* slots, int64_t requests, void* h, void* out, int64_t ldo) {
  using namespace pasa::lora;
  int st = check(m, k, n, rank, adapters, requests);
  if (st || m == 0) return st;
  if ((st = check_matrix(x, ldx, k)) || (st = check_matrix(y, ldy, n)) || (st = check_matrix(out, ldo, n))) return st;
  if (!a || !b || !rows || !h || (requests && !slots)) return PASA_ERR_NULL;
  if (misaligned(a) || misaligned(b) || misaligned(h)) return PASA_ERR_ALIGN;
  if (out == y && ldo != ldy) return PASA_ERR_SHAPE;
  int sms = 0;
  if ((st = device_sms(&sms))) return st;
  uint32_t* err = operator_error_word();
  if (!err) return PASA_ERR_CUDA;
  const Rows r{rows, slots, scale, int(requests), int(adapters), m};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  __nv_bfloat16* hh = static_cast<__nv_bfloat16*>(h);
  cudaError_t e = down_a(s, r, Matrix{x, ldx}, k, n, a, rank, hh, sms, err);
  if (e == cudaSuccess)
    e = few_rows(r, k, n, rank) ? up_few(s, r, hh, b, rank, n, Matrix{y, ldy}, Matrix{out, ldo})
                                : up<false>(s, r, hh, b, rank, n, Matrix{y, ldy}, Matrix{out, ldo}, sms, err);
  return e == cudaSuccess ? PASA_OK : PASA_ERR_CUDA;
}

int pasa_lora_backward_workspace_size(int64_t m, int64_t k, int64_t n, int rank, int64_t adapters, int64_t requests,
                                      size_t* bytes) {
  using namespace pasa::lora;
  if (!bytes) return PASA_ERR_NULL;
  int st = check(m, k, n, rank, adapters, requests);
  if (st) return st;
  int sms = 0;
  if ((st = device_sms(&sms))) return st;
  size_t h = 0;
  pasa_lora_h_size(m, rank, &h);
  *bytes = align256(h) + (m && requests ? grad_partial_bytes(m, k, n, rank, adapters, requests, sms) : 0);
  return PASA_OK;
}

int pasa_lora_update_backward(void* stream, const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* a,
                              const void* b, const float* scale, int64_t m, int64_t k, int64_t n, int rank,
                              int64_t adapters, const int32_t* rows, const int32_t* slots, int64_t requests, void* h,
                              int h_given, const void* dx_base, int64_t ldbase, void* dx, int64_t lddx, void* da,
                              void* db, void* workspace, size_t workspace_bytes) {
  using namespace pasa::lora;
  int st = check(m, k, n, rank, adapters, requests);
  if (st) return st;
  if (m && ((st = check_matrix(dy, lddy, n)) || (st = check_matrix(x, ldx, k)) ||
            (dx && (st = check_matrix(dx, lddx, k))) || (dx && dx_base && (st = check_matrix(dx_base, ldbase, k)))))
    return st;
  if (!a || !b || !rows || (requests && !slots) || (m && db && !h)) return PASA_ERR_NULL;
  if (misaligned(a) || misaligned(b) || misaligned(h) || misaligned(da) || misaligned(db)) return PASA_ERR_ALIGN;
  if (dx && dx == dx_base && lddx != ldbase) return PASA_ERR_SHAPE;
  size_t need = 0;
  if ((st = pasa_lora_backward_workspace_size(m, k, n, rank, adapters, requests, &need))) return st;
  if (need && (!workspace || workspace_bytes < need)) return PASA_ERR_WORKSPACE;
  if (misaligned(workspace)) return PASA_ERR_ALIGN;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (m == 0 || requests == 0) {  // no row has an adapter
    const size_t grad_bytes = size_t(adapters) * size_t(rank) * 2;
    if (da && cudaMemsetAsync(da, 0, grad_bytes * size_t(k), s) != cudaSuccess) return PASA_ERR_CUDA;
    if (db && cudaMemsetAsync(db, 0, grad_bytes * size_t(n), s) != cudaSuccess) return PASA_ERR_CUDA;
    if (m == 0 || !dx) return PASA_OK;
  }
  int sms = 0;
  if ((st = device_sms(&sms))) return st;
  uint32_t* err = operator_error_word();
  if (!err) return PASA_ERR_CUDA;
  const Rows r{rows, slots, scale, int(requests), int(adapters), m};
  __nv_bfloat16* g = static_cast<__nv_bfloat16*>(workspace);
  __nv_bfloat16* hh = static_cast<__nv_bfloat16*>(h);
  size_t h_bytes = 0;
  pasa_lora_h_size(m, rank, &h_bytes);
  cudaError_t e = cudaSuccess;
  if (db && !h_given && requests) e = down_a(s, r, Matrix{x, ldx}, k, n, a, rank, hh, sms, err);
  if (e == cudaSuccess && (dx || da)) e = down<true>(s, r, Matrix{dy, lddy}, n, b, rank, g, sms, err);
  if (e == cudaSuccess && dx)
    e = up<true>(s, r, g, a, rank, k, Matrix{dx_base, ldbase}, Matrix{dx, lddx}, sms, err);
  if (e == cudaSuccess && (da || db) && requests)
    e = grad(s, r, rank, Matrix{x, ldx}, k, Matrix{dy, lddy}, n, g, hh, da, db,
             static_cast<unsigned char*>(workspace) + align256(h_bytes), sms, err);
  return e == cudaSuccess ? PASA_OK : PASA_ERR_CUDA;
}

}  // extern "C"
