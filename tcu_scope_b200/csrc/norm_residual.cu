// The norms around a block, fused with the block's gate and its residual connection, and the gradient:
//     n = z / rms(z) * post        (z itself without post)
//     o = residual + scale * act(gate) * n
//     u = o / rms(o) * pre         rms(y) = sqrt(mean(y^2) + eps)
// With c = scale act(gate) post, which rows share, and a = 1 / rms(z), o = residual + a c z, so that the second
// norm's sum is known from sums that need no first:
//     sum o^2 = sum residual^2 + 2 a sum residual c z + a^2 sum (c z)^2
// and threads meet once a row.  Where the branch cancels most of the residual (sum o^2 below a quarter of what is
// added up) that would lose digits, and o is summed itself, at another meeting.
//
// Gradient, per row, with v = du pre, b = 1 / rms(o), zn = a z:
//     d  = do + b (v - o b mean(v o b))                 = dresidual
//     dz = a (c d - zn mean(c d zn))
//     dpre = sum over rows of du o b;  q = sum over rows of d zn;  dpost = scale act(gate) q;  dgate = scale act'(gate) post q
// and again every mean follows from sums of products of what is read:
//     sum v o = sum v residual + a sum v c z
//     sum c d z = sum c z do + b sum v c z - b^2 mean(v o b) (sum residual c z + a sum (c z)^2)
// The sums over rows are kept by every block for its own rows, in registers, and joined by a second kernel in
// the order of the blocks: no atomics, the same bits every time.
//
// Bound by HBM: 4 arrays forward, 6 backward.  Rows come through a ring in shared memory, each thread copying (cp.async)
// what it will read itself: nothing is waited for but a thread's own copies and the one meeting.
// Measured, bf16, of the copy bandwidth: forward 16384 x 4096 106 us (77 %; without post and gate 103, without residual, too,
// 88), 65536 x 256 80 % (a warp a row, no meeting), 8192 x 5120 65 %, bound by the instructions a row takes; gradient 226 us (54 %;
// 218, 190), of which its seven sums take 62: it needs up to 127 registers, so that one block of 512 threads is on an SM and
// nothing runs while that meets.  Gradient of rows a warp holds, 65536 x 256, 39 %; of 16 elements a thread, 8192 x 5120, 34 %;
// element by element, 4096 x 12288, 15 %.  (Two meetings forward and four backward took 129 and 509 us; pairs of
// floats in one instruction 131 and 237.)
#include <type_traits>

#include "lm_common.cuh"

namespace tcu_lm {
namespace {

constexpr int kNone = 0, kSigmoid = 1, kSilu = 2;

struct NormArgs {
  const void *z, *residual, *post, *gate, *pre, *dout, *dnormed;
  void *out, *normed, *dz, *dresidual;
  void* dgate;        // written where one worker holds all rows of a gate row
  float* gate_parts;  // else one row of floats per unit
  float *post_parts, *pre_parts;  // one row of floats per worker
  int64_t rows, rows_per_gate, slice_rows;
  int64_t z_row, residual_row, gate_row, dout_row, dnormed_row;
  int64_t units;      // backward: slices of the rows of one gate row
  int64_t workers;    // blocks, or warps, that take consecutive units (forward: rows)
  int slices;         // per gate row
  int dim, act, row_bytes;  // row_bytes: of a row in the ring
  float scale, eps;
};

__device__ __forceinline__ float act_of(int act, float g) {
  if (act == kNone) return g;
  const float s = reciprocal(1.f + exp2_fast(-g * kLog2E));
  return act == kSigmoid ? s : g * s;
}

__device__ __forceinline__ float slope_of(int act, float g) {
  if (act == kNone) return 1.f;
  const float s = reciprocal(1.f + exp2_fast(-g * kLog2E)), r = reciprocal(1.f + exp2_fast(g * kLog2E));  // r = 1 - s
  return act == kSigmoid ? s * r : s * (1.f + g * r);
}

// ------------------------------------------------------------------ sums over a row's threads
// Each of N sums over a warp (WARP) or the block, in every thread, always added up in the same order: the
// lanes halve the sums among them, so that 8 take 9 exchanges and not 40.  `scratch`: N x 33 floats that the previous
// call did not use.
template <bool WARP, int N>
__device__ __forceinline__ void row_sums(float (&s)[N], float* scratch) {
  const int lane = threadIdx.x & 31;
  constexpr int kLanes = 32 / N;  // lanes that end up with the same sum
  int o = 16;
#pragma unroll
  for (int n = N / 2; n >= 1; n /= 2, o /= 2) {
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float keep = lane & o ? s[i + n] : s[i], give = lane & o ? s[i] : s[i + n];
      s[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
    }
  }
  float x = s[0];
#pragma unroll
  for (int q = kLanes / 2; q >= 1; q /= 2) x += __shfl_xor_sync(0xffffffffu, x, q);
  if constexpr (!WARP) {
    const int warps = blockDim.x >> 5, mine = lane / kLanes, sub = lane % kLanes;
    if (warps > 1) {
      if (sub == 0) scratch[mine * 33 + (threadIdx.x >> 5)] = x;
      __syncthreads();
      x = 0.f;
      for (int w = sub; w < warps; w += kLanes) x += scratch[mine * 33 + w];
#pragma unroll
      for (int q = kLanes / 2; q >= 1; q /= 2) x += __shfl_xor_sync(0xffffffffu, x, q);
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] = __shfl_sync(0xffffffffu, x, i * kLanes);
}

// ------------------------------------------------------------------ rows
// A thread's elements of a row: vectors first, first + width, ... of VEC elements, E elements in all.
template <int VEC, int E>
struct Part {
  int first, width, dim;
  __device__ __forceinline__ int at(int k) const { return (first + k * width) * VEC; }
};

template <typename T, int VEC, int E>
__device__ __forceinline__ void load_part(float (&x)[E], const Part<VEC, E>& t, const T* row) {
#pragma unroll
  for (int k = 0; k < E / VEC; ++k) {
    const Vec<T, VEC> r = t.at(k) < t.dim ? load_vec<T, VEC>(row + t.at(k)) : zero_vec<T, VEC>();
    float y[VEC];
    to_floats<T, VEC>(r, y);
#pragma unroll
    for (int c = 0; c < VEC; ++c) x[k * VEC + c] = y[c];
  }
}

template <typename T, int VEC, int E>
__device__ __forceinline__ void store_part(T* row, const Part<VEC, E>& t, const float (&x)[E]) {
#pragma unroll
  for (int k = 0; k < E / VEC; ++k) {
    float y[VEC];
#pragma unroll
    for (int c = 0; c < VEC; ++c) y[c] = x[k * VEC + c];
    if (t.at(k) < t.dim) store_vec<T, VEC>(row + t.at(k), y);
  }
}

constexpr int kStages = 3;  // rows in the ring

// An array's rows on their way through the ring (VEC == 1: read from where they are, an element at a time; those rows are not
// aligned for copies, or the ring does not hold them, which 16-byte loads past the ring would not need: not built).
// The gate's rows do not take it: with a gate for each row each row waits for its gate, too.
template <typename T, int VEC, int E>
struct Stream {
  const T* base;
  int64_t stride;
  unsigned char* ring;  // of stage 0
  int stage_bytes;

  __device__ __forceinline__ void fetch(const Part<VEC, E>& t, int64_t row, int stage) const {
    if (VEC == 1 || base == nullptr) return;
    const T* from = base + row * stride;
    T* to         = reinterpret_cast<T*>(ring + stage * stage_bytes);
#pragma unroll
    for (int k = 0; k < E / VEC; ++k)
      if (t.at(k) < t.dim) copy_async16(to + t.at(k), from + t.at(k));
  }
  __device__ __forceinline__ void load(float (&x)[E], const Part<VEC, E>& t, int64_t row, int stage) const {
    if (base == nullptr) {
#pragma unroll
      for (int i = 0; i < E; ++i) x[i] = 0.f;
    } else {
      load_part<T, VEC, E>(x, t, VEC == 1 ? base + row * stride : reinterpret_cast<const T*>(ring + stage * stage_bytes));
    }
  }
};

// c = scale act(gate) post, of the gate's row `group`.
template <typename T, typename W, int VEC, int E>
__device__ __forceinline__ void coefficients(float (&c)[E], const Part<VEC, E>& t, const NormArgs& p, int64_t group) {
#pragma unroll
  for (int i = 0; i < E; ++i) c[i] = p.scale;
  float x[E];
  if (p.gate) {
    load_part<T, VEC, E>(x, t, static_cast<const T*>(p.gate) + group * p.gate_row);
#pragma unroll
    for (int i = 0; i < E; ++i) c[i] *= act_of(p.act, x[i]);
  }
  if (p.post) {
    load_part<W, VEC, E>(x, t, static_cast<const W*>(p.post));
#pragma unroll
    for (int i = 0; i < E; ++i) c[i] *= x[i];
  }
}

// Whether sum o^2, of terms of this size, has lost digits, or a part left float32 (which o itself need not do).
__device__ __forceinline__ bool cancelled(float sum, float residual_part, float branch_part) {
  const float parts = residual_part + branch_part;
  return !(sum >= 0.25f * parts) || parts == INFINITY;
}

template <typename T, typename W, int VEC, int E, bool WARP, int THREADS, int BLOCKS>
__global__ void __launch_bounds__(THREADS, BLOCKS)
norm_residual_kernel(const NormArgs p) {
  __shared__ float scratch[2][4 * 33], again[2][2 * 33];
  extern __shared__ __align__(16) unsigned char rings[];
  const Part<VEC, E> t = {WARP ? int(threadIdx.x & 31) : int(threadIdx.x), WARP ? 32 : int(blockDim.x), p.dim};
  const int64_t worker = WARP ? int64_t(blockIdx.x) * (THREADS / 32) + (threadIdx.x >> 5) : blockIdx.x;
  if (worker >= p.workers) return;
  unsigned char* ring = rings + (WARP ? (threadIdx.x >> 5) * kStages * 2 * p.row_bytes : 0);
  const Stream<T, VEC, E> z = {static_cast<const T*>(p.z), p.z_row, ring, 2 * p.row_bytes};
  const Stream<T, VEC, E> residual = {static_cast<const T*>(p.residual), p.residual_row, ring + p.row_bytes, 2 * p.row_bytes};
  const float inv_dim = 1.f / float(p.dim);
  const int64_t begin = worker * p.rows / p.workers, end = (worker + 1) * p.rows / p.workers;
  auto fetch = [&](int64_t row, int stage) {
    if (row < end) z.fetch(t, row, stage), residual.fetch(t, row, stage);
    copy_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages; ++i) fetch(begin + i, i);
  float c[E], pre[E];
  if (p.pre) load_part<W, VEC, E>(pre, t, static_cast<const W*>(p.pre));
  int64_t group = begin / p.rows_per_gate, group_end = (group + 1) * p.rows_per_gate;
  coefficients<T, W, VEC, E>(c, t, p, group);
  int stage = 0, side = 0;
  for (int64_t row = begin; row < end; ++row, side ^= 1) {
    if (row == group_end) {
      ++group, group_end += p.rows_per_gate;
      coefficients<T, W, VEC, E>(c, t, p, group);
    }
    copy_wait(kStages - 1);
    float x[E], r[E];
    z.load(x, t, row, stage);
    residual.load(r, t, row, stage);
    float s[4] = {0.f, 0.f, 0.f, 0.f};  // of z z, r r, r c z, c z c z
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float cz = c[i] * x[i];
      s[0] = fmaf(x[i], x[i], s[0]);
      s[1] = fmaf(r[i], r[i], s[1]);
      s[2] = fmaf(r[i], cz, s[2]);
      s[3] = fmaf(cz, cz, s[3]);
      x[i] = cz;
    }
    row_sums<WARP, 4>(s, scratch[side]);
    const float rz = p.post ? rsqrtf(fmaf(s[0], inv_dim, p.eps)) : 1.f;
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = fmaf(rz, x[i], r[i]);
    store_part<T, VEC, E>(static_cast<T*>(p.out) + row * p.dim, t, x);
    if (p.pre) {
      float so = s[1] + rz * fmaf(rz, s[3], 2.f * s[2]);
      if (cancelled(so, s[1], rz * rz * s[3])) {
        float o[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < E; ++i) o[0] = fmaf(x[i], x[i], o[0]);
        row_sums<WARP, 2>(o, again[side]);
        so = o[0];
      }
      const float ro = rsqrtf(fmaf(so, inv_dim, p.eps));
#pragma unroll
      for (int i = 0; i < E; ++i) x[i] *= ro * pre[i];
      store_part<T, VEC, E>(static_cast<T*>(p.normed) + row * p.dim, t, x);
    }
    fetch(row + kStages, stage);
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }
}

template <typename T, typename W, int VEC, int E, bool WARP, int THREADS>
__global__ void __launch_bounds__(THREADS)
norm_residual_backward_kernel(const NormArgs p) {
  __shared__ float scratch[2][8 * 33], again[2][2][2 * 33];
  extern __shared__ __align__(16) unsigned char rings[];
  const Part<VEC, E> t = {WARP ? int(threadIdx.x & 31) : int(threadIdx.x), WARP ? 32 : int(blockDim.x), p.dim};
  const int64_t worker = WARP ? int64_t(blockIdx.x) * (THREADS / 32) + (threadIdx.x >> 5) : blockIdx.x;
  if (worker >= p.workers) return;
  unsigned char* ring = rings + (WARP ? (threadIdx.x >> 5) * kStages * 4 * p.row_bytes : 0);
  const int stage_bytes = 4 * p.row_bytes;
  const Stream<T, VEC, E> z = {static_cast<const T*>(p.z), p.z_row, ring, stage_bytes};
  const Stream<T, VEC, E> residual = {static_cast<const T*>(p.pre ? p.residual : nullptr), p.residual_row, ring + p.row_bytes, stage_bytes};
  const Stream<T, VEC, E> dout = {static_cast<const T*>(p.dout), p.dout_row, ring + 2 * p.row_bytes, stage_bytes};
  const Stream<T, VEC, E> dnormed = {static_cast<const T*>(p.pre ? p.dnormed : nullptr), p.dnormed_row, ring + 3 * p.row_bytes, stage_bytes};
  const float inv_dim = 1.f / float(p.dim);
  auto begin_of = [&](int64_t unit) { return unit / p.slices * p.rows_per_gate + unit % p.slices * p.slice_rows; };
  const int64_t first_unit = worker * p.units / p.workers, last_unit = (worker + 1) * p.units / p.workers;
  int64_t end = begin_of(last_unit);  // the worker's rows lie one behind the other
  if (end > p.rows) end = p.rows;
  auto fetch = [&](int64_t row, int stage) {
    if (row < end) z.fetch(t, row, stage), residual.fetch(t, row, stage), dout.fetch(t, row, stage), dnormed.fetch(t, row, stage);
    copy_commit();
  };
  int64_t row = begin_of(first_unit);
#pragma unroll
  for (int i = 0; i < kStages; ++i) fetch(row + i, i);
  float c[E], pre[E], dpost[E], dpre[E];
#pragma unroll
  for (int i = 0; i < E; ++i) dpost[i] = dpre[i] = pre[i] = 0.f;
  if (p.pre) load_part<W, VEC, E>(pre, t, static_cast<const W*>(p.pre));
  int stage = 0, side = 0;
  for (int64_t unit = first_unit; unit < last_unit; ++unit) {
    const int64_t group = unit / p.slices;
    int64_t unit_end    = begin_of(unit) + p.slice_rows;
    if (unit_end > (group + 1) * p.rows_per_gate) unit_end = (group + 1) * p.rows_per_gate;
    coefficients<T, W, VEC, E>(c, t, p, group);
    float q[E];  // the sum over rows of d zn
#pragma unroll
    for (int i = 0; i < E; ++i) q[i] = 0.f;
    for (; row < unit_end; ++row, side ^= 1) {
      copy_wait(kStages - 1);
      float x[E], r[E], d[E], du[E];
      z.load(x, t, row, stage);
      residual.load(r, t, row, stage);
      dout.load(d, t, row, stage);
      dnormed.load(du, t, row, stage);
      // of z z, r r, r c z, c z c z, v r, v c z, c z do
      float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float cz = c[i] * x[i], v = du[i] * pre[i];
        s[0] = fmaf(x[i], x[i], s[0]);
        s[1] = fmaf(r[i], r[i], s[1]);
        s[2] = fmaf(r[i], cz, s[2]);
        s[3] = fmaf(cz, cz, s[3]);
        s[4] = fmaf(v, r[i], s[4]);
        s[5] = fmaf(v, cz, s[5]);
        s[6] = fmaf(cz, d[i], s[6]);
      }
      row_sums<WARP, 8>(s, scratch[side]);
      const float rz = p.post ? rsqrtf(fmaf(s[0], inv_dim, p.eps)) : 1.f;
      // d = do + ro (v - m on), on = ro o, m = mean(v on);  mean: of c d z, times dim.  (Only one ro is multiplied at a
      // time: ro^2 and ro^3 leave float32 for rows whose sum of squares does not.)
      float ro = 0.f, m = 0.f, mean = s[6];
      if (p.pre) {
        float so = s[1] + rz * fmaf(rz, s[3], 2.f * s[2]), vo = fmaf(rz, s[5], s[4]);
        const bool careful = cancelled(so, s[1], rz * rz * s[3]);
        if (careful) {
          float y[2] = {0.f, 0.f};
#pragma unroll
          for (int i = 0; i < E; ++i) {
            const float o = fmaf(rz * c[i], x[i], r[i]);
            y[0] = fmaf(o, o, y[0]);
            y[1] = fmaf(du[i] * pre[i], o, y[1]);
          }
          row_sums<WARP, 2>(y, again[side][0]);
          so = y[0], vo = y[1];
        }
        ro   = rsqrtf(fmaf(so, inv_dim, p.eps));
        m    = ro * vo * inv_dim;
        mean = fmaf(ro, fmaf(-m, ro * fmaf(rz, s[3], s[2]), s[5]), s[6]);
        if (careful) {
          float y[2] = {0.f, 0.f};
#pragma unroll
          for (int i = 0; i < E; ++i) {
            const float o = fmaf(rz * c[i], x[i], r[i]);
            y[0] = fmaf(c[i] * x[i], fmaf(ro, fmaf(-m, o * ro, du[i] * pre[i]), d[i]), y[0]);
          }
          row_sums<WARP, 2>(y, again[side][1]);
          mean = y[0];
        }
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const float on = fmaf(rz * c[i], x[i], r[i]) * ro;
          dpre[i] = fmaf(du[i], on, dpre[i]);
          d[i]    = fmaf(ro, fmaf(-m, on, du[i] * pre[i]), d[i]);
        }
      }
      if (p.dresidual) store_part<T, VEC, E>(static_cast<T*>(p.dresidual) + row * p.dim, t, d);
      const float shift = p.post ? -(rz * mean * inv_dim) * rz : 0.f;  // dz = rz (c d + shift z), rz inside: mean(c d zn) zn
#pragma unroll
      for (int i = 0; i < E; ++i) {
        q[i] = fmaf(d[i], rz * x[i], q[i]);
        d[i] = rz * fmaf(shift, x[i], c[i] * d[i]);
      }
      store_part<T, VEC, E>(static_cast<T*>(p.dz) + row * p.dim, t, d);
      fetch(row + kStages, stage);
      stage = stage + 1 == kStages ? 0 : stage + 1;
    }
    // dpost += scale act(gate) q, dgate = scale act'(gate) post q
    float gate[E];
    if (p.gate) load_part<T, VEC, E>(gate, t, static_cast<const T*>(p.gate) + group * p.gate_row);
    if (p.post_parts) {
#pragma unroll
      for (int i = 0; i < E; ++i) dpost[i] = fmaf(p.gate ? p.scale * act_of(p.act, gate[i]) : p.scale, q[i], dpost[i]);
    }
    if (p.dgate || p.gate_parts) {
#pragma unroll
      for (int i = 0; i < E; ++i) q[i] *= p.scale * slope_of(p.act, gate[i]);
      if (p.post) {
        load_part<W, VEC, E>(gate, t, static_cast<const W*>(p.post));
#pragma unroll
        for (int i = 0; i < E; ++i) q[i] *= gate[i];
      }
      if (p.dgate) store_part<T, VEC, E>(static_cast<T*>(p.dgate) + group * p.dim, t, q);
      if (p.gate_parts) store_part<float, VEC, E>(p.gate_parts + unit * p.dim, t, q);
    }
  }
  if (p.post_parts) store_part<float, VEC, E>(p.post_parts + worker * p.dim, t, dpost);
  if (p.pre_parts) store_part<float, VEC, E>(p.pre_parts + worker * p.dim, t, dpre);
}

// out[g][c] = sum over k of parts[g * count + k][c], in a fixed order; blockIdx.y is g over three jobs.
struct Job {
  const float* parts;
  void* out;
  int64_t groups, count;
  int type;
};
struct Jobs {
  Job job[3];
  int dim;
};

constexpr int kSumWarps = 32;

__device__ __forceinline__ void store_typed(void* out, int64_t at, float x, int type) {
  if (type == TCU_TYPE_F32)
    static_cast<float*>(out)[at] = x;
  else if (type == TCU_TYPE_F16)
    static_cast<__half*>(out)[at] = __float2half_rn(x);
  else
    static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(x);
}

__global__ void __launch_bounds__(kSumWarps * 32)
column_sums_kernel(const Jobs jobs) {
  __shared__ float part[kSumWarps][33];
  int64_t g = blockIdx.y;
  int j = 0;
  while (j < 2 && g >= jobs.job[j].groups) g -= jobs.job[j].groups, ++j;
  const Job& job = jobs.job[j];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t column = int64_t(blockIdx.x) * 32 + lane;
  float s = 0.f;
  if (column < jobs.dim) {
    const float* p = job.parts + g * job.count * jobs.dim + column;
#pragma unroll 4
    for (int64_t k = warp; k < job.count; k += kSumWarps) s += p[k * jobs.dim];
  }
  part[warp][lane] = s;
  __syncthreads();
  s = warp_sum(part[lane][warp]);  // column `warp` of this block
  const int64_t mine = int64_t(blockIdx.x) * 32 + warp;
  if (lane == 0 && mine < jobs.dim) store_typed(job.out, g * jobs.dim + mine, s, job.type);
}

// ------------------------------------------------------------------ host side
constexpr int kMaxDim      = 16384;
constexpr int kWarpThreads = 256;  // rows that a warp holds (up to 256 elements): eight to a block
constexpr int kWarpDim     = 256;

// A row's threads, whole warps, for E elements a thread.
int row_threads(int64_t dim, int e) { return int((dim + e * 32 - 1) / (e * 32) * 32); }

// Elements per thread: 8, but not more threads than `most`.
int elements(int64_t dim, int most) { return dim <= most * 8 ? 8 : 16; }

// Workers of the backward pass, which needs 122 registers and more: as many as 512 threads on each of the 148 SMs
// are (a number that leaves some SMs with one more than others takes twice as long: 236 blocks of 320 threads).  Rows of up to 256
// elements are 296 blocks of 8 warps, of which the 146 ... 164 registers a thread that their kernels take let an SM
// hold one at a time; above 4096 elements the kernels spill (480 bytes a thread, 1200 above 8192).
int64_t backward_workers(int64_t dim) {
  const int threads = dim <= kWarpDim ? 32 : row_threads(dim, elements(dim, 512));
  return threads > 512 ? 148 : 148 * (512 / threads);
}

template <typename K>
cudaError_t allow_shared(K kernel, bool* configured, int bytes) {
  const int dev = current_device();
  if (dev < 0) return cudaErrorInvalidDevice;
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  return cudaSuccess;
}
constexpr int kMostShared = 216 << 10;

// Launches a kernel whose ring holds kStages rows of `arrays` arrays for each of `rings` rows at a time.
template <typename K>
int launch_rows(K kernel, bool* configured, NormArgs p, int elem, int vec, int arrays, int rings, unsigned grid, int threads,
                cudaStream_t st) {
  p.row_bytes     = vec > 1 ? (p.dim * elem + 15) / 16 * 16 : 0;
  const int bytes = kStages * arrays * rings * p.row_bytes;
  if (allow_shared(kernel, configured, kMostShared) != cudaSuccess) return TCU_ERR_CUDA;
  kernel<<<grid, threads, bytes, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? TCU_OK : TCU_ERR_CUDA;
}

// Whether a ring of rows of `arrays` arrays fits into shared memory (two of 32 bits: up to 9212 elements, four: 4604).
bool ring_fits(int64_t dim, size_t elem, int arrays) { return kStages * arrays * (dim * int64_t(elem) + 15) / 16 * 16 <= kMostShared; }

bool row_vectors(const void* p, size_t elem, int64_t stride, int vec) {
  return aligned(p, elem * vec < 16 ? elem * vec : 16) && stride % vec == 0;
}

template <typename F>
int for_norm_types(int64_t type, int64_t w_type, F&& f) {
  if (type == TCU_TYPE_F32) return f(float{}, float{});
  if (type == TCU_TYPE_F16) return w_type == TCU_TYPE_F32 ? f(__half{}, float{}) : f(__half{}, __half{});
  return w_type == TCU_TYPE_F32 ? f(__nv_bfloat16{}, float{}) : f(__nv_bfloat16{}, __nv_bfloat16{});
}

// How the rows of a backward call are cut: units (slices of the rows of one gate row), and workers that take
// consecutive units.
struct Cut {
  int64_t units, workers, slice_rows;
  int slices;
};

Cut cut_rows(int64_t rows, int64_t dim, int64_t gate_rows) {
  const int64_t most = backward_workers(dim);
  const int64_t per  = rows / gate_rows;
  Cut c;
  int64_t slices = gate_rows >= most ? 1 : most / gate_rows;
  if (slices > per) slices = per;
  c.slice_rows = (per + slices - 1) / slices;
  slices       = (per + c.slice_rows - 1) / c.slice_rows;
  c.slices     = int(slices);
  c.units      = gate_rows * slices;
  c.workers    = c.units < most ? c.units : most;
  return c;
}

int check_norm(int64_t type, int64_t w_type, int64_t act, int64_t rows, int64_t dim, const void* gate, int64_t gate_rows) {
  if (!known_type(type) || (w_type != type && w_type != TCU_TYPE_F32)) return TCU_ERR_UNSUPPORTED;
  if (act < kNone || act > kSilu || dim > kMaxDim) return TCU_ERR_UNSUPPORTED;
  if (rows < 0 || dim < 0 || rows > (int64_t(1) << 40)) return TCU_ERR_INVALID_ARG;
  if (gate && rows > 0 && (gate_rows <= 0 || rows % gate_rows != 0)) return TCU_ERR_INVALID_ARG;
  return TCU_OK;
}

}  // namespace
}  // namespace tcu_lm

using namespace tcu_lm;

extern "C" {

int tcu_norm_residual(const tcu_norm_residual_args* g, void* stream) {
  if (!g) return TCU_ERR_INVALID_ARG;
  if (const int e = check_norm(g->type, g->weight_type, g->act, g->rows, g->dim, g->gate, g->gate_rows)) return e;
  if (g->rows == 0 || g->dim == 0) return TCU_OK;
  if (!g->z || !g->out || (g->pre_weight && !g->normed)) return TCU_ERR_INVALID_ARG;
  const size_t e = type_bytes(g->type), ew = type_bytes(g->weight_type);
  if (!aligned(g->z, e) || !aligned(g->residual, e) || !aligned(g->gate, e) || !aligned(g->out, e) ||
      !aligned(g->normed, e) || !aligned(g->post_weight, ew) || !aligned(g->pre_weight, ew))
    return TCU_ERR_INVALID_ARG;
  const int sms = sm_count();
  if (sms <= 0) return TCU_ERR_CUDA;
  NormArgs p{};
  p.z = g->z, p.residual = g->residual, p.post = g->post_weight, p.gate = g->gate, p.pre = g->pre_weight;
  p.out = g->out, p.normed = g->normed;
  p.rows = g->rows, p.dim = int(g->dim), p.rows_per_gate = g->gate ? g->rows / g->gate_rows : g->rows;
  p.z_row = g->z_row_stride, p.residual_row = g->residual_row_stride, p.gate_row = g->gate_row_stride;
  p.act = int(g->act), p.scale = float(g->scale), p.eps = float(g->eps);
  return for_norm_types(g->type, g->weight_type, [&](auto t, auto w) -> int {
    using T = decltype(t);
    using W = decltype(w);
    constexpr int V = 16 / sizeof(T);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool wide = p.dim % V == 0 && ring_fits(p.dim, e, 2) && row_vectors(p.z, e, p.z_row, V) && row_vectors(p.residual, e, p.residual_row, V) &&
                      row_vectors(p.gate, e, p.gate_row, V) && row_vectors(p.post, ew, 0, V) &&
                      row_vectors(p.pre, ew, 0, V) && aligned(p.out, 16) && aligned(p.normed, 16);
    auto go = [&](auto vec) -> int {
      constexpr int VEC = decltype(vec)::value;
      if (p.dim <= kWarpDim) {
        static bool ready[kMaxDevices];
        p.workers = p.rows < int64_t(sms) * 64 ? p.rows : int64_t(sms) * 64;
        return launch_rows(norm_residual_kernel<T, W, VEC, 8, true, kWarpThreads, 4>, ready, p, sizeof(T), VEC, 2, 8,
                           unsigned((p.workers + 7) / 8), kWarpThreads, st);
      }
      const int e8 = elements(p.dim, 512), threads = row_threads(p.dim, e8);
      const int blocks = threads > 512 ? 1 : e8 == 16 ? 1024 / threads : 2048 / threads;  // for an SM
      p.workers        = p.rows < int64_t(sms) * blocks ? p.rows : int64_t(sms) * blocks;
      const unsigned grid = unsigned(p.workers);
      if (e8 == 8) {
        static bool ready[kMaxDevices];
        return launch_rows(norm_residual_kernel<T, W, VEC, 8, false, 512, 2>, ready, p, sizeof(T), VEC, 2, 1, grid, threads, st);
      }
      if (threads <= 512) {
        static bool ready[kMaxDevices];
        return launch_rows(norm_residual_kernel<T, W, VEC, 16, false, 512, 2>, ready, p, sizeof(T), VEC, 2, 1, grid, threads, st);
      }
      static bool ready[kMaxDevices];
      return launch_rows(norm_residual_kernel<T, W, VEC, 16, false, 1024, 1>, ready, p, sizeof(T), VEC, 2, 1, grid, threads, st);
    };
    return wide ? go(std::integral_constant<int, V>{}) : go(std::integral_constant<int, 1>{});
  });
}

size_t tcu_norm_residual_workspace_bytes(size_t rows, size_t dim, size_t gate_rows) {
  if (rows == 0 || dim == 0 || dim > kMaxDim) return 0;
  if (gate_rows == 0 || rows % gate_rows != 0) gate_rows = 1;
  const Cut c = cut_rows(int64_t(rows), int64_t(dim), int64_t(gate_rows));
  return size_t(2 * c.workers + (c.slices > 1 ? c.units : 0)) * dim * sizeof(float) + 3 * 16;
}

int tcu_norm_residual_backward(const tcu_norm_residual_backward_args* g, void* stream) {
  if (!g) return TCU_ERR_INVALID_ARG;
  if (const int e = check_norm(g->type, g->weight_type, g->act, g->rows, g->dim, g->gate, g->gate_rows)) return e;
  const size_t e = type_bytes(g->type), ew = type_bytes(g->weight_type);
  if (!aligned(g->z, e) || !aligned(g->residual, e) || !aligned(g->gate, e) || !aligned(g->dout, e) ||
      !aligned(g->dnormed, e) || !aligned(g->dz, e) || !aligned(g->dresidual, e) || !aligned(g->dgate, e) ||
      !aligned(g->post_weight, ew) || !aligned(g->pre_weight, ew) || !aligned(g->dpost_weight, ew) ||
      !aligned(g->dpre_weight, ew))
    return TCU_ERR_INVALID_ARG;
  if ((g->dpost_weight && !g->post_weight) || (g->dgate && !g->gate) || (g->dpre_weight && !g->pre_weight))
    return TCU_ERR_INVALID_ARG;
  if (g->dim == 0) return TCU_OK;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (g->rows == 0) {  // sums of nothing
    if (g->dpost_weight && cudaMemsetAsync(g->dpost_weight, 0, g->dim * ew, st) != cudaSuccess) return TCU_ERR_CUDA;
    if (g->dpre_weight && cudaMemsetAsync(g->dpre_weight, 0, g->dim * ew, st) != cudaSuccess) return TCU_ERR_CUDA;
    if (g->dgate && g->gate_rows > 0 && cudaMemsetAsync(g->dgate, 0, g->gate_rows * g->dim * e, st) != cudaSuccess)
      return TCU_ERR_CUDA;
    return TCU_OK;
  }
  if (!g->z || !g->dz) return TCU_ERR_INVALID_ARG;
  const int64_t gate_rows = g->gate ? g->gate_rows : 1;
  const size_t need       = tcu_norm_residual_workspace_bytes(g->rows, g->dim, gate_rows);
  if (!g->workspace || g->workspace_bytes < int64_t(need) || !aligned(g->workspace, 16)) return TCU_ERR_WORKSPACE;
  const Cut c = cut_rows(g->rows, g->dim, gate_rows);
  NormArgs p{};
  p.z = g->z, p.residual = g->residual, p.post = g->post_weight, p.gate = g->gate, p.pre = g->pre_weight;
  p.dout = g->dout, p.dnormed = g->dnormed, p.dz = g->dz, p.dresidual = g->dresidual;
  p.rows = g->rows, p.dim = int(g->dim), p.rows_per_gate = g->rows / gate_rows;
  p.z_row = g->z_row_stride, p.residual_row = g->residual_row_stride, p.gate_row = g->gate_row_stride;
  p.dout_row = g->dout_row_stride, p.dnormed_row = g->dnormed_row_stride;
  p.act = int(g->act), p.scale = float(g->scale), p.eps = float(g->eps);
  p.units = c.units, p.workers = c.workers, p.slices = c.slices, p.slice_rows = c.slice_rows;
  const size_t part = (size_t(c.workers) * g->dim + 3) / 4 * 4;  // each array begins at a multiple of 16 bytes
  float* ws = static_cast<float*>(g->workspace);
  if (g->dpost_weight) p.post_parts = ws;
  if (g->dpre_weight) p.pre_parts = ws + part;
  if (g->dgate) {
    if (c.slices > 1)
      p.gate_parts = ws + 2 * part;
    else
      p.dgate = g->dgate;
  }
  const int err = for_norm_types(g->type, g->weight_type, [&](auto t, auto w) -> int {
    using T = decltype(t);
    using W = decltype(w);
    constexpr int V = 16 / sizeof(T);
    const bool wide = p.dim % V == 0 && ring_fits(p.dim, e, 4) && row_vectors(p.z, e, p.z_row, V) && row_vectors(p.residual, e, p.residual_row, V) &&
                      row_vectors(p.gate, e, p.gate_row, V) && row_vectors(p.dout, e, p.dout_row, V) &&
                      row_vectors(p.dnormed, e, p.dnormed_row, V) && row_vectors(p.post, ew, 0, V) &&
                      row_vectors(p.pre, ew, 0, V) && aligned(p.dz, 16) && aligned(p.dresidual, 16) && aligned(p.dgate, 16);
    auto go = [&](auto vec) -> int {
      constexpr int VEC = decltype(vec)::value;
      const int e8 = elements(p.dim, 512), threads = row_threads(p.dim, e8);
      const unsigned grid = unsigned(c.workers);
      if (p.dim <= kWarpDim) {
        static bool ready[kMaxDevices];
        return launch_rows(norm_residual_backward_kernel<T, W, VEC, 8, true, kWarpThreads>, ready, p, sizeof(T), VEC, 4, 8,
                           (grid + 7) / 8, kWarpThreads, st);
      }
      if (e8 == 8) {
        static bool ready[kMaxDevices];
        return launch_rows(norm_residual_backward_kernel<T, W, VEC, 8, false, 512>, ready, p, sizeof(T), VEC, 4, 1, grid, threads, st);
      }
      if (threads <= 512) {
        static bool ready[kMaxDevices];
        return launch_rows(norm_residual_backward_kernel<T, W, VEC, 16, false, 512>, ready, p, sizeof(T), VEC, 4, 1, grid, threads, st);
      }
      // (a ring of rows of more than 8192 elements does not fit with four arrays of 32 bits, of 16 bits up to 9209: read
      // element by element, whatever their type and alignment)
      static bool ready[kMaxDevices];
      return launch_rows(norm_residual_backward_kernel<T, W, 1, 16, false, 1024>, ready, p, sizeof(T), 1, 4, 1, grid, threads, st);
    };
    return wide ? go(std::integral_constant<int, V>{}) : go(std::integral_constant<int, 1>{});
  });
  if (err != TCU_OK) return err;
  Jobs jobs{};
  jobs.dim = p.dim;
  int n = 0;
  int64_t groups = 0;
  auto add = [&](const float* parts, void* out, int64_t count_groups, int64_t count, int64_t type) {
    if (!parts) return;
    jobs.job[n++] = {parts, out, count_groups, count, int(type)};
    groups += count_groups;
  };
  add(p.post_parts, g->dpost_weight, 1, c.workers, g->weight_type);
  add(p.pre_parts, g->dpre_weight, 1, c.workers, g->weight_type);
  add(p.gate_parts, g->dgate, gate_rows, c.slices, g->type);
  if (n == 0) return TCU_OK;
  column_sums_kernel<<<dim3(unsigned((p.dim + 31) / 32), unsigned(groups)), kSumWarps * 32, 0, st>>>(jobs);
  return cudaGetLastError() == cudaSuccess ? TCU_OK : TCU_ERR_CUDA;
}

}  // extern "C"
