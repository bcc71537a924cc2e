// Rotary positions with several axes (frame, row, column, ...) of queries and
// keys, without a table: pair p of axis i is turned by the angle
//     pos_i * f_p,   (u, v) -> (u cos - v sin, u sin + v cos)
// and the dimensions behind the last pair are kept.  The inverse turns by the
// negative angle, which is also the gradient of the forward pass: a rotation's
// transpose is its inverse.  Positions are a grid's points in row-major order,
// computed from the token's index, or one vector per token.
//
// Arithmetic.  The angle is formed in turns in fp64 (pos * f / 2 pi) and its
// whole turns are dropped there, so a position of 2^30 keeps its angle to
// about 1e-7; sine and cosine of what is left are fp32 (sincospi of the
// leading 24 bits, and the rest of the angle by one step of the addition
// theorem), the rotation is fp32 and rounded once.
//
// Bound: HBM.  Every value is read once and written once; an angle costs about
// as many instructions as rotating 15 values, so a thread computes the angles
// of one 16-byte vector of one token and applies them to up to kMaxHeads heads
// (of q and of k), four heads' loads in flight.  With fewer tokens than fill
// the GPU the heads are split over more threads instead, down to one head a
// thread.  Measured: q and k of 75600 tokens, 40 heads of 128 (3.1 GB moved) in
// 512 us, 6.05 TB/s; of 1560 tokens, 24 heads (38 MB, two heads a thread: bound by
// the angles) in 17.7 us.
#include "common.cuh"

namespace pasa {
namespace rope {

constexpr int kMaxAxes = 4;
constexpr int kMaxPairs = 128;
constexpr int kThreads = 256;
constexpr int kMaxHeads = 16;  // heads a thread turns by the same angles
constexpr int kUnroll = 4;     // heads whose loads are in flight together

struct Tensor {
  const void* x;
  void* out;
  int64_t xs[3], os[3];  // strides of batch, head, token in elements
};

struct Args {
  Tensor t[2];           // q, k
  int heads0, heads;     // heads of q; of q and k together
  int heads_per_thread;
  int64_t tokens, slots; // tokens of a batch entry; batch * tokens * units
  int units;             // threads of one token
  int dim, pairs;        // pairs: rotated pairs (2 * pairs <= dim)
  const void* positions; // [batch or 1, tokens, axes], or null: a grid
  int pos_type;
  int64_t pos_batch;     // stride between batch entries (0: shared)
  int axes;
  int64_t grid[kMaxAxes], origin[kMaxAxes];
  int axis_end[kMaxAxes];     // first pair behind axis i
  double turns[kMaxPairs];    // f_p / 2 pi, negated for the inverse
};

__device__ __forceinline__ double load_position(const Args& a, int64_t i) {
  switch (a.pos_type) {
    case PASA_POS_I32: return double(static_cast<const int32_t*>(a.positions)[i]);
    case PASA_POS_I64: return double(static_cast<const int64_t*>(a.positions)[i]);
    case PASA_POS_F32: return double(static_cast<const float*>(a.positions)[i]);
    default: return static_cast<const double*>(a.positions)[i];
  }
}

// The token's position on every axis.
__device__ __forceinline__ void token_position(const Args& a, int64_t b, int64_t token, double (&pos)[kMaxAxes]) {
  if (a.positions != nullptr) {
#pragma unroll
    for (int i = 0; i < kMaxAxes; ++i)
      pos[i] = i < a.axes ? load_position(a, b * a.pos_batch + token * a.axes + i) : 0.0;
    return;
  }
  uint32_t rest = uint32_t(token);  // a grid has fewer than 2^31 points
#pragma unroll
  for (int i = kMaxAxes - 1; i >= 0; --i) {
    if (i >= a.axes) { pos[i] = 0.0; continue; }
    const uint32_t n = uint32_t(a.grid[i]), q = rest / n;
    pos[i] = double(int64_t(rest - q * n) + a.origin[i]);
    rest = q;
  }
}

// cos and sin of pair p's angle.
__device__ __forceinline__ float2 pair_rotation(const Args& a, const double (&pos)[kMaxAxes], int p) {
  double where = pos[0];
#pragma unroll
  for (int i = 1; i < kMaxAxes; ++i)
    if (i < a.axes && p >= a.axis_end[i - 1]) where = pos[i];
  const double turn = where * a.turns[p];
  const double half_turns = 2.0 * (turn - rint(turn));  // in [-1, 1]
  const float lead = float(half_turns);
  const float rest = float(half_turns - double(lead)) * 3.14159265f;
  float s, c;
  sincospif(lead, &s, &c);
  return make_float2(fmaf(-s, rest, c), fmaf(c, rest, s));
}

__device__ __forceinline__ float2 turn(float u, float v, float2 cs) {
  return make_float2(u * cs.x - v * cs.y, u * cs.y + v * cs.x);
}

// One 16-byte vector as fp32 values and back.
template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4& r, float (&f)[4]) {
    f[0] = __uint_as_float(r.x); f[1] = __uint_as_float(r.y); f[2] = __uint_as_float(r.z); f[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& r, float (&f)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                      pack_bf16x2(f[6], f[7]));
  }
};

// Offsets of head h (of q, then of k) at this token.
template <typename T>
__device__ __forceinline__ void head_pointers(const Args& a, int h, int64_t b, int64_t token, const T*& x, T*& out) {
  const bool second = h >= a.heads0;
  const Tensor& t = a.t[second ? 1 : 0];
  const int64_t hh = second ? h - a.heads0 : h;
  x = static_cast<const T*>(t.x) + b * t.xs[0] + hh * t.xs[1] + token * t.xs[2];
  out = static_cast<T*>(t.out) + b * t.os[0] + hh * t.os[1] + token * t.os[2];
}

// Vectors of 16 bytes.  HALVES: unit u < pairs / N holds the pairs of the
// vectors at u * N and pairs + u * N, the units behind them copy the tail's;
// otherwise unit u is the vector at u * N with N / 2 adjacent pairs.
template <typename T, bool HALVES>
__global__ void __launch_bounds__(kThreads) rope_vec_kernel(const __grid_constant__ Args a) {
  constexpr int N = Vec<T>::N;
  constexpr int P = HALVES ? N : N / 2;  // pairs of a unit
  const int64_t slot = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  if (slot >= a.slots) return;
  const int64_t row = slot / a.units;
  const int u = int(slot - row * a.units);
  const int64_t b = row / a.tokens, token = row - b * a.tokens;
  const int h_begin = int(blockIdx.y) * a.heads_per_thread;
  const int h_end = min(h_begin + a.heads_per_thread, a.heads);
  const int turned_units = HALVES ? a.pairs / N : (2 * a.pairs + N - 1) / N;
  const bool copies = u >= turned_units;
  const int first = HALVES && copies ? 2 * a.pairs + (u - turned_units) * N : u * N;  // its first value
  const int p0 = HALVES ? u * N : u * (N / 2);
  float2 cs[P];
  if (!copies) {
    double pos[kMaxAxes];
    token_position(a, b, token, pos);
#pragma unroll
    for (int i = 0; i < P; ++i)
      cs[i] = p0 + i < a.pairs ? pair_rotation(a, pos, p0 + i) : make_float2(1.f, 0.f);
  }
  for (int h0 = h_begin; h0 < h_end; h0 += kUnroll) {
    uint4 lo[kUnroll], hi[kUnroll];
    const T* x;
    T* out;
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      if (h0 + j >= h_end) break;
      head_pointers<T>(a, h0 + j, b, token, x, out);
      lo[j] = *reinterpret_cast<const uint4*>(x + first);
      if (HALVES && !copies) hi[j] = *reinterpret_cast<const uint4*>(x + first + a.pairs);
    }
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      if (h0 + j >= h_end) break;
      head_pointers<T>(a, h0 + j, b, token, x, out);
      if (!copies) {
        float f[N], g[N];
        Vec<T>::unpack(lo[j], f);
        if (HALVES) {
          Vec<T>::unpack(hi[j], g);
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const float2 r = turn(f[i], g[i], cs[i % P]);
            f[i] = r.x;
            g[i] = r.y;
          }
          *reinterpret_cast<uint4*>(out + first + a.pairs) = Vec<T>::pack(g);
        } else {
#pragma unroll
          for (int i = 0; i < N / 2; ++i) {
            if (p0 + i >= a.pairs) continue;  // values behind the last pair are kept as they are
            const float2 r = turn(f[2 * i], f[2 * i + 1], cs[i]);
            f[2 * i] = r.x;
            f[2 * i + 1] = r.y;
          }
        }
        lo[j] = Vec<T>::pack(f);
      }
      *reinterpret_cast<uint4*>(out + first) = lo[j];
    }
  }
}

// Any alignment and any sizes: unit u < pairs is one pair, the units behind
// them are the tail's values.
template <typename T, bool HALVES>
__global__ void __launch_bounds__(kThreads) rope_pair_kernel(const __grid_constant__ Args a) {
  const int64_t slot = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  if (slot >= a.slots) return;
  const int64_t row = slot / a.units;
  const int u = int(slot - row * a.units);
  const int64_t b = row / a.tokens, token = row - b * a.tokens;
  const int h_begin = int(blockIdx.y) * a.heads_per_thread;
  const int h_end = min(h_begin + a.heads_per_thread, a.heads);
  float2 cs = make_float2(1.f, 0.f);
  if (u < a.pairs) {
    double pos[kMaxAxes];
    token_position(a, b, token, pos);
    cs = pair_rotation(a, pos, u);
  }
  const int d0 = u < a.pairs ? (HALVES ? u : 2 * u) : a.pairs + u, d1 = HALVES ? u + a.pairs : 2 * u + 1;
  for (int h = h_begin; h < h_end; ++h) {
    const T* x;
    T* out;
    head_pointers<T>(a, h, b, token, x, out);
    if (u < a.pairs) {
      const float2 r = turn(Elem<T>::load(x + d0), Elem<T>::load(x + d1), cs);
      Elem<T>::store(out + d0, r.x);
      Elem<T>::store(out + d1, r.y);
    } else {
      out[d0] = x[d0];
    }
  }
}

bool vector_aligned(const Args& a, int tensors, int esize) {
  for (int i = 0; i < tensors; ++i) {
    if ((reinterpret_cast<uintptr_t>(a.t[i].x) | reinterpret_cast<uintptr_t>(a.t[i].out)) & 15u) return false;
    for (int j = 0; j < 3; ++j)
      if (((a.t[i].xs[j] * esize) & 15) || ((a.t[i].os[j] * esize) & 15)) return false;
  }
  return true;
}

template <typename T, bool HALVES>
cudaError_t launch(cudaStream_t stream, Args& a, int tensors, int64_t batch, int sms) {
  constexpr int N = Vec<T>::N;
  const bool vec = vector_aligned(a, tensors, int(sizeof(T))) && a.dim % N == 0 && (!HALVES || a.pairs % N == 0);
  a.units = vec ? (HALVES ? (a.dim - a.pairs) / N : a.dim / N) : a.dim - a.pairs;
  a.slots = batch * a.tokens * a.units;
  const int64_t blocks = cdiv(a.slots, kThreads);
  // as many heads a thread as leave eight blocks for every SM (a full one)
  int per = kMaxHeads;
  while (per > 1 && blocks * cdiv(a.heads, per) < int64_t(sms) * 8) per >>= 1;
  if (cdiv(a.heads, per) > 65535) per = int(cdiv(a.heads, 65535));
  a.heads_per_thread = per;
  const dim3 grid(unsigned(blocks), unsigned(cdiv(a.heads, per)), 1);
  if (vec) rope_vec_kernel<T, HALVES><<<grid, kThreads, 0, stream>>>(a);
  else rope_pair_kernel<T, HALVES><<<grid, kThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace rope
}  // namespace pasa

using namespace pasa;

extern "C" int pasa_rope_axes(void* stream, const pasa_rope_tensor* tensors, int n_tensors, int dtype, int64_t batch,
                              int64_t tokens, int dim, const void* positions, int pos_type, int64_t pos_batch_stride,
                              const int64_t* grid, const int64_t* origin, int n_axes, const int* axes,
                              const double* freqs, int pairing, int inverse) {
  using namespace pasa::rope;
  if (dtype != PASA_BF16 && dtype != PASA_F32) return PASA_ERR_DTYPE;
  if (!tensors || !axes || !freqs || (!positions && !grid)) return PASA_ERR_NULL;
  if (n_tensors < 1 || n_tensors > 2 || n_axes < 1 || n_axes > kMaxAxes || batch < 0 || tokens < 0 || dim < 1)
    return PASA_ERR_SHAPE;
  if (pairing != PASA_PAIRS_INTERLEAVED && pairing != PASA_PAIRS_HALVES) return PASA_ERR_UNSUPPORTED;
  if (positions && (pos_type < PASA_POS_I32 || pos_type > PASA_POS_F64)) return PASA_ERR_DTYPE;
  if (dim > (1 << 20) || tokens > INT32_MAX || batch > INT32_MAX) return PASA_ERR_SHAPE;
  Args a{};
  int pairs = 0;
  for (int i = 0; i < n_axes; ++i) {
    if (axes[i] < 0 || axes[i] % 2 || axes[i] > 2 * kMaxPairs) return PASA_ERR_SHAPE;
    pairs += axes[i] / 2;
    a.axis_end[i] = pairs;
  }
  if (pairs < 1 || pairs > kMaxPairs || 2 * pairs > dim) return PASA_ERR_SHAPE;
  if (!positions) {
    int64_t points = 1;
    for (int i = 0; i < n_axes; ++i) {
      if (grid[i] < 0 || grid[i] > INT32_MAX) return PASA_ERR_SHAPE;
      points *= grid[i];
      if (points > INT32_MAX) return PASA_ERR_SHAPE;
      a.grid[i] = grid[i];
      a.origin[i] = origin ? origin[i] : 0;
    }
    if (points != tokens) return PASA_ERR_SHAPE;
  }
  int64_t heads = 0;
  for (int i = 0; i < n_tensors; ++i) {
    if (tensors[i].heads < 0 || tensors[i].heads > INT32_MAX / 2) return PASA_ERR_SHAPE;
    heads += tensors[i].heads;
    if (i == 0) a.heads0 = int(heads);
    a.t[i].x = tensors[i].x;
    a.t[i].out = tensors[i].out;
    for (int j = 0; j < 3; ++j) {
      a.t[i].xs[j] = tensors[i].x_stride[j];
      a.t[i].os[j] = tensors[i].out_stride[j];
    }
  }
  if (heads == 0 || batch == 0 || tokens == 0) return PASA_OK;
  for (int i = 0; i < n_tensors; ++i)
    if (tensors[i].heads && (!tensors[i].x || !tensors[i].out)) return PASA_ERR_NULL;
  if (cdiv(batch * tokens, kThreads) > INT32_MAX / dim) return PASA_ERR_SHAPE;
  int dev = 0, major = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return PASA_ERR_CUDA;
  if (major != 10) return PASA_ERR_DEVICE;
  a.heads = int(heads);
  a.tokens = tokens;
  a.dim = dim;
  a.pairs = pairs;
  a.positions = positions;
  a.pos_type = pos_type;
  a.pos_batch = pos_batch_stride;
  a.axes = n_axes;
  constexpr double kTurn = 6.283185307179586476925286766559;
  for (int p = 0; p < pairs; ++p) a.turns[p] = (inverse ? -freqs[p] : freqs[p]) / kTurn;
  const bool halves = pairing == PASA_PAIRS_HALVES;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (dtype == PASA_BF16)
    e = halves ? launch<__nv_bfloat16, true>(st, a, n_tensors, batch, sms)
               : launch<__nv_bfloat16, false>(st, a, n_tensors, batch, sms);
  else
    e = halves ? launch<float, true>(st, a, n_tensors, batch, sms) : launch<float, false>(st, a, n_tensors, batch, sms);
  return e == cudaSuccess ? PASA_OK : PASA_ERR_CUDA;
}
