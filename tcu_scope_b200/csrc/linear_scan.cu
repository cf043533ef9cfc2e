// Gated linear recurrence h_t = f_t h_{t-1} + u_t along time, channel by channel, and its gradient.
//
// The step h -> f h + u is a linear map, and maps compose: (A2, H2) after (A1, H1) is
// (A2 A1, A2 H1 + H2).  So time is cut into pieces whose maps are computed independently, and
// only the maps are passed along:
//   - a warp holds 8 consecutive rows of 32 * VEC channels in registers and computes their map;
//   - the 8 warps of a block hold 64 consecutive rows (a chunk) and exchange maps in shared memory;
//   - the P blocks of a cluster hold P consecutive chunks (a window) of the same channels and
//     exchange maps in each other's shared memory;
//   - the cluster goes through its sequence window by window, the state in registers, the next window's
//     rows already on their way.
// Every element is read and written once.  All maps are joined in the order of time, so the result does not depend on timing.
//
// Backwards, with g_t = f_t dh_t passing from row t to row t-1 (dh_t = dy_t + g_{t+1}) the same
// holds with time reversed; h_{t-1} is recomputed from the state before each chunk, which the
// forward pass leaves behind (one row of floats for 64 rows of elements).
//
// Bound by HBM: 3 arrays forward, 5 backward.
#include <cooperative_groups.h>

#include <type_traits>

#include "lm_common.cuh"

namespace tcu_lm {
namespace {

namespace cg = cooperative_groups;

constexpr int kWarps      = 8;
constexpr int kRows       = 8;               // rows per warp and window
constexpr int kChunk      = kWarps * kRows;  // rows per block and window; also the spacing of the states
constexpr int kMaxCluster = 8;

struct ScanArgs {
  const void *a, *x, *dh;
  void *h, *da, *dx;
  const float *h0, *dlast;
  float *last, *states, *dh0;
  const void* offsets;
  int64_t batch, tokens, dim;
  int64_t a_batch, a_row, x_batch, x_row, dh_batch, dh_row;
  int columns;
  bool wide;
  bool clear_rest;  // with offsets: rows outside all sequences become 0
};

// f and u of one element, and 1 - f (SIGMOID only), computed without cancellation.
template <int GATE>
__device__ __forceinline__ void gate_of(float a, float x, float& f, float& u, float& one_minus_f) {
  if constexpr (GATE == TCU_GATE_SIGMOID) {
    const float e = expf(-fabsf(a));
    const float r = __fdividef(1.f, 1.f + e);
    const float s = e * r;
    f           = a >= 0.f ? r : s;
    one_minus_f = a >= 0.f ? s : r;
    u           = one_minus_f * x;
  } else {
    f = GATE == TCU_GATE_LOG ? expf(a) : a;
    u = x;
  }
}

// The rows of the block's sequence: where they begin, how many, and where its chunks' states lie.
struct Sequence {
  int64_t a, x, dh, out;  // element offsets of the first row
  int64_t chunk;          // row of `states` of the first chunk
  int64_t length;
};

__device__ __forceinline__ Sequence sequence_of(const ScanArgs& p, int64_t b) {
  Sequence s;
  if (p.offsets == nullptr) {
    s.length = p.tokens;
    s.a      = b * p.a_batch;
    s.x      = b * p.x_batch;
    s.dh     = b * p.dh_batch;
    s.out    = b * p.tokens * p.dim;
    s.chunk  = b * ((p.tokens + kChunk - 1) / kChunk);
    return s;
  }
  int64_t first = load_index(p.offsets, b, p.wide), end = load_index(p.offsets, b + 1, p.wide);
  if (first < 0 || end < first || end > p.tokens) {
    if (threadIdx.x == 0) raise_index_error();
    first = end = 0;
  }
  s.length = end - first;
  s.a      = first * p.a_row;
  s.x      = first * p.x_row;
  s.dh     = first * p.dh_row;
  s.out    = first * p.dim;
  s.chunk  = first / kChunk + b;  // distinct: a sequence has at most length / kChunk + 1 chunks
  return s;
}

template <typename T, int VEC>
__device__ __forceinline__ void load_rows(Vec<T, VEC> (&r)[kRows], const T* base, int64_t row_stride,
                                          int64_t row, int64_t length, bool in_dim) {
#pragma unroll
  for (int i = 0; i < kRows; ++i)
    r[i] = in_dim && row + i < length ? load_vec<T, VEC>(base + (row + i) * row_stride) : zero_vec<T, VEC>();
}

// Rows that no sequence holds, of the channels of this block: those before the first sequence and
// behind the last one.
template <typename T, int VEC>
__device__ __forceinline__ void clear_rest(const ScanArgs& p, T* out, int64_t b, int64_t ch, int part, int parts) {
  const float zero[VEC] = {};
  const int warp = part * kWarps + (threadIdx.x >> 5), warps = parts * kWarps;
  if (ch >= p.dim) return;
  if (b == 0) {
    const int64_t first = load_index(p.offsets, 0, p.wide);
    for (int64_t r = warp; r < first && r < p.tokens; r += warps) store_vec<T, VEC>(out + r * p.dim + ch, zero);
  }
  if (b == p.batch - 1) {
    const int64_t end = load_index(p.offsets, p.batch, p.wide);
    for (int64_t r = (end < 0 ? 0 : end) + warp; r < p.tokens; r += warps) store_vec<T, VEC>(out + r * p.dim + ch, zero);
  }
}

// VEC floats of every lane, in shared memory, lanes side by side.
template <int VEC>
struct Lanes {
  Vec<float, VEC> lane[32];
};

template <int VEC>
__device__ __forceinline__ void apply(float (&h)[VEC], const Vec<float, VEC>& A, const Vec<float, VEC>& H) {
#pragma unroll
  for (int c = 0; c < VEC; ++c) h[c] = h[c] == 0.f ? H.v[c] : fmaf(A.v[c], h[c], H.v[c]);
  // (a product of gates that overflowed must not turn a state of 0 into NaN)
}

template <typename T, typename A, int GATE, int VEC>
__global__ void __launch_bounds__(kWarps * 32)
linear_scan_kernel(const ScanArgs p) {
  __shared__ Lanes<VEC> warp_a[2][kWarps], warp_h[2][kWarps];
  __shared__ Lanes<VEC> block_a[2][kMaxCluster], block_h[2][kMaxCluster];
  const cg::cluster_group cluster = cg::this_cluster();
  const int parts = int(cluster.num_blocks()), part = int(cluster.block_rank());
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t group = blockIdx.x / parts;
  const int64_t b     = group / p.columns;
  const int64_t ch    = (group % p.columns) * (32 * VEC) + lane * VEC;
  const bool in_dim   = ch < p.dim;
  const Sequence s    = sequence_of(p, b);
  const A* a = static_cast<const A*>(p.a) + s.a + ch;
  const T* x = static_cast<const T*>(p.x) + s.x + ch;
  T* out     = static_cast<T*>(p.h) + s.out + ch;

  float carry[VEC];  // the state before the current window
#pragma unroll
  for (int c = 0; c < VEC; ++c) carry[c] = 0.f;
  if (p.h0 && in_dim) {
#pragma unroll
    for (int c = 0; c < VEC; ++c) carry[c] = p.h0[b * p.dim + ch + c];
  }

  if (parts > 1) cluster.sync();  // no block writes to another's shared memory before that has begun
  const int64_t step = int64_t(parts) * kChunk;
  int64_t row        = int64_t(part) * kChunk + warp * kRows;
  Vec<A, VEC> next_a[kRows];
  Vec<T, VEC> next_x[kRows];
  load_rows<A, VEC>(next_a, a, p.a_row, row, s.length, in_dim);
  load_rows<T, VEC>(next_x, x, p.x_row, row, s.length, in_dim);
  int side = 0;
  for (int64_t window = 0; window < s.length; window += step, row += step, side ^= 1) {
    float f[kRows][VEC], u[kRows][VEC];
    Vec<float, VEC> prod, sum;
#pragma unroll
    for (int c = 0; c < VEC; ++c) prod.v[c] = 1.f, sum.v[c] = 0.f;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const bool inside = row + i < s.length;  // rows behind the end: the identity
#pragma unroll
      for (int c = 0; c < VEC; ++c) {
        float unused;
        gate_of<GATE>(to_float(next_a[i].v[c]), to_float(next_x[i].v[c]), f[i][c], u[i][c], unused);
        f[i][c] = inside ? f[i][c] : 1.f;
        u[i][c] = inside ? u[i][c] : 0.f;
        sum.v[c] = fmaf(f[i][c], sum.v[c], u[i][c]);
        prod.v[c] *= f[i][c];
      }
    }
    if (window + step < s.length) {
      load_rows<A, VEC>(next_a, a, p.a_row, row + step, s.length, in_dim);
      load_rows<T, VEC>(next_x, x, p.x_row, row + step, s.length, in_dim);
    }
    warp_a[side][warp].lane[lane] = prod;
    warp_h[side][warp].lane[lane] = sum;
    __syncthreads();
    float h[VEC];  // becomes the state before this warp's rows
    if (parts > 1) {
      // this block's map to all blocks of the cluster: warp r writes to block r
      Vec<float, VEC> A_ = warp_a[side][0].lane[lane];
      Vec<float, VEC> H_ = warp_h[side][0].lane[lane];
#pragma unroll
      for (int j = 1; j < kWarps; ++j) {
        const Vec<float, VEC> aj = warp_a[side][j].lane[lane], hj = warp_h[side][j].lane[lane];
        apply<VEC>(H_.v, aj, hj);
#pragma unroll
        for (int c = 0; c < VEC; ++c) A_.v[c] *= aj.v[c];
      }
      if (warp < parts) {
        cluster.map_shared_rank(&block_a[side][part], warp)->lane[lane] = A_;
        cluster.map_shared_rank(&block_h[side][part], warp)->lane[lane] = H_;
      }
      cluster.sync();
      float before[VEC];
#pragma unroll
      for (int c = 0; c < VEC; ++c) before[c] = carry[c];
      for (int q = 0; q < parts; ++q) {
        if (q == part) {
#pragma unroll
          for (int c = 0; c < VEC; ++c) before[c] = carry[c];
        }
        apply<VEC>(carry, block_a[side][q].lane[lane], block_h[side][q].lane[lane]);
      }
#pragma unroll
      for (int c = 0; c < VEC; ++c) h[c] = before[c];
    } else {
#pragma unroll
      for (int c = 0; c < VEC; ++c) h[c] = carry[c];
#pragma unroll
      for (int j = 0; j < kWarps; ++j)
        apply<VEC>(carry, warp_a[side][j].lane[lane], warp_h[side][j].lane[lane]);
    }
    const int64_t chunk = window / kChunk + part;
    if (p.states && warp == 0 && in_dim && chunk * kChunk < s.length)
      store_vec<float, VEC>(p.states + (s.chunk + chunk) * p.dim + ch, h);
    for (int j = 0; j < warp; ++j)
      apply<VEC>(h, warp_a[side][j].lane[lane], warp_h[side][j].lane[lane]);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
#pragma unroll
      for (int c = 0; c < VEC; ++c) h[c] = fmaf(f[i][c], h[c], u[i][c]);
      if (in_dim && row + i < s.length) store_vec<T, VEC>(out + (row + i) * p.dim, h);
    }
  }
  if (p.clear_rest) clear_rest<T, VEC>(p, static_cast<T*>(p.h), b, ch, part, parts);
  if (p.last && part == 0 && warp == 0 && in_dim) store_vec<float, VEC>(p.last + b * p.dim + ch, carry);
}

template <typename T, typename A, int GATE, int VEC>
__global__ void __launch_bounds__(kWarps * 32)
linear_scan_backward_kernel(const ScanArgs p) {
  __shared__ Lanes<VEC> warp_a[2][kWarps], warp_h[2][kWarps], warp_g[2][kWarps];
  __shared__ Lanes<VEC> block_a[2][kMaxCluster], block_g[2][kMaxCluster];
  const cg::cluster_group cluster = cg::this_cluster();
  const int parts = int(cluster.num_blocks()), part = int(cluster.block_rank());
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t group = blockIdx.x / parts;
  const int64_t b     = group / p.columns;
  const int64_t ch    = (group % p.columns) * (32 * VEC) + lane * VEC;
  const bool in_dim   = ch < p.dim;
  const Sequence s    = sequence_of(p, b);
  const A* a  = static_cast<const A*>(p.a) + s.a + ch;
  const T* x  = static_cast<const T*>(p.x) + s.x + ch;
  const T* dy = static_cast<const T*>(p.dh) + s.dh + ch;
  A* da       = static_cast<A*>(p.da) + s.out + ch;
  T* dx       = static_cast<T*>(p.dx) + s.out + ch;

  float carry[VEC];  // what the rows behind the current window pass back
#pragma unroll
  for (int c = 0; c < VEC; ++c) carry[c] = 0.f;
  if (p.dlast && in_dim) {
#pragma unroll
    for (int c = 0; c < VEC; ++c) carry[c] = p.dlast[b * p.dim + ch + c];
  }

  if (parts > 1) cluster.sync();
  const int64_t step    = int64_t(parts) * kChunk;
  const int64_t windows = (s.length + step - 1) / step;
  int64_t row           = (windows - 1) * step + int64_t(part) * kChunk + warp * kRows;
  Vec<A, VEC> next_a[kRows];
  Vec<T, VEC> next_x[kRows], next_d[kRows];
  const bool has_dy = p.dh != nullptr;
  if (windows > 0) {
    load_rows<A, VEC>(next_a, a, p.a_row, row, s.length, in_dim);
    load_rows<T, VEC>(next_x, x, p.x_row, row, s.length, in_dim);
    load_rows<T, VEC>(next_d, dy, p.dh_row, row, s.length, in_dim && has_dy);
  }
  int side = 0;
  for (int64_t window = (windows - 1) * step; window >= 0; window -= step, row -= step, side ^= 1) {
    const int64_t chunk = window / kChunk + part;
    float h[VEC];  // the state before this chunk
#pragma unroll
    for (int c = 0; c < VEC; ++c) h[c] = 0.f;
    if (in_dim && chunk * kChunk < s.length) {
      const Vec<float, VEC> st = load_vec<float, VEC>(p.states + (s.chunk + chunk) * p.dim + ch);
#pragma unroll
      for (int c = 0; c < VEC; ++c) h[c] = st.v[c];
    }
    float f[kRows][VEC], u[kRows][VEC], rest[kRows][VEC], d[kRows][VEC];
    Vec<float, VEC> prod, sum, back;
#pragma unroll
    for (int c = 0; c < VEC; ++c) prod.v[c] = 1.f, sum.v[c] = 0.f, back.v[c] = 0.f;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const bool inside = row + i < s.length;
#pragma unroll
      for (int c = 0; c < VEC; ++c) {
        gate_of<GATE>(to_float(next_a[i].v[c]), to_float(next_x[i].v[c]), f[i][c], u[i][c], rest[i][c]);
        f[i][c] = inside ? f[i][c] : 1.f;
        u[i][c] = inside ? u[i][c] : 0.f;
        d[i][c] = to_float(next_d[i].v[c]);
        sum.v[c] = fmaf(f[i][c], sum.v[c], u[i][c]);
        prod.v[c] *= f[i][c];
      }
    }
#pragma unroll
    for (int i = kRows - 1; i >= 0; --i) {
#pragma unroll
      for (int c = 0; c < VEC; ++c) back.v[c] = f[i][c] * (d[i][c] + back.v[c]);
    }
    float xs[kRows][VEC];  // only SIGMOID needs x again
    if constexpr (GATE == TCU_GATE_SIGMOID) {
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
#pragma unroll
        for (int c = 0; c < VEC; ++c) xs[i][c] = to_float(next_x[i].v[c]);
      }
    }
    if (window > 0) {
      load_rows<A, VEC>(next_a, a, p.a_row, row - step, s.length, in_dim);
      load_rows<T, VEC>(next_x, x, p.x_row, row - step, s.length, in_dim);
      load_rows<T, VEC>(next_d, dy, p.dh_row, row - step, s.length, in_dim && has_dy);
    }
    warp_a[side][warp].lane[lane] = prod;
    warp_h[side][warp].lane[lane] = sum;
    warp_g[side][warp].lane[lane] = back;
    __syncthreads();
    float g[VEC];  // becomes what the rows behind this warp's pass back
    if (parts > 1) {
      Vec<float, VEC> A_ = warp_a[side][kWarps - 1].lane[lane];
      Vec<float, VEC> G_ = warp_g[side][kWarps - 1].lane[lane];
#pragma unroll
      for (int j = kWarps - 2; j >= 0; --j) {
        const Vec<float, VEC> aj = warp_a[side][j].lane[lane], gj = warp_g[side][j].lane[lane];
        apply<VEC>(G_.v, aj, gj);
#pragma unroll
        for (int c = 0; c < VEC; ++c) A_.v[c] *= aj.v[c];
      }
      if (warp < parts) {
        cluster.map_shared_rank(&block_a[side][part], warp)->lane[lane] = A_;
        cluster.map_shared_rank(&block_g[side][part], warp)->lane[lane] = G_;
      }
      cluster.sync();
      float behind[VEC];
#pragma unroll
      for (int c = 0; c < VEC; ++c) behind[c] = carry[c];
      for (int q = parts - 1; q >= 0; --q) {
        if (q == part) {
#pragma unroll
          for (int c = 0; c < VEC; ++c) behind[c] = carry[c];
        }
        apply<VEC>(carry, block_a[side][q].lane[lane], block_g[side][q].lane[lane]);
      }
#pragma unroll
      for (int c = 0; c < VEC; ++c) g[c] = behind[c];
    } else {
#pragma unroll
      for (int c = 0; c < VEC; ++c) g[c] = carry[c];
#pragma unroll
      for (int j = kWarps - 1; j >= 0; --j)
        apply<VEC>(carry, warp_a[side][j].lane[lane], warp_g[side][j].lane[lane]);
    }
    for (int j = kWarps - 1; j > warp; --j)
      apply<VEC>(g, warp_a[side][j].lane[lane], warp_g[side][j].lane[lane]);
    for (int j = 0; j < warp; ++j)
      apply<VEC>(h, warp_a[side][j].lane[lane], warp_h[side][j].lane[lane]);
    float before[kRows][VEC];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
#pragma unroll
      for (int c = 0; c < VEC; ++c) {
        before[i][c] = h[c];
        h[c]         = fmaf(f[i][c], h[c], u[i][c]);
      }
    }
#pragma unroll
    for (int i = kRows - 1; i >= 0; --i) {
      float ga[VEC], gx[VEC];
#pragma unroll
      for (int c = 0; c < VEC; ++c) {
        const float dh = d[i][c] + g[c];
        if constexpr (GATE == TCU_GATE_SIGMOID) {
          ga[c] = dh * (before[i][c] - xs[i][c]) * f[i][c] * rest[i][c];
          gx[c] = dh * rest[i][c];
        } else {
          ga[c] = GATE == TCU_GATE_LOG ? dh * before[i][c] * f[i][c] : dh * before[i][c];
          gx[c] = dh;
        }
        g[c] = f[i][c] * dh;
      }
      if (in_dim && row + i < s.length) {
        store_vec<A, VEC>(da + (row + i) * p.dim, ga);
        store_vec<T, VEC>(dx + (row + i) * p.dim, gx);
      }
    }
  }
  if (p.clear_rest) {
    clear_rest<A, VEC>(p, static_cast<A*>(p.da), b, ch, part, parts);
    clear_rest<T, VEC>(p, static_cast<T*>(p.dx), b, ch, part, parts);
  }
  if (p.dh0 && part == 0 && warp == 0 && in_dim) store_vec<float, VEC>(p.dh0 + b * p.dim + ch, carry);
}

struct StepArgs {
  const void *a, *x;
  void* h;
  float* state;
  const void* slots;
  int64_t batch, pool, dim, a_row, x_row;
  int blocks_per_row;
  bool wide, clear_rest;
};

constexpr int kStepThreads = 256;

// One token.  A block takes kStepThreads * VEC channels of one row; with slots it first looks
// whether an earlier row has the same one (two rows must not update a state at a time).
template <typename T, typename A, int GATE, int VEC>
__global__ void __launch_bounds__(kStepThreads)
linear_scan_step_kernel(const StepArgs p) {
  const int64_t b  = blockIdx.x / p.blocks_per_row;
  const int64_t ch = (int64_t(blockIdx.x % p.blocks_per_row) * kStepThreads + threadIdx.x) * VEC;
  const bool in_dim = ch < p.dim;
  int64_t slot = b;
  if (p.slots) {
    slot      = load_index(p.slots, b, p.wide);
    bool same = false;
    if (slot >= 0)
      for (int64_t i = threadIdx.x; i < b; i += kStepThreads) same |= load_index(p.slots, i, p.wide) == slot;
    const bool taken = __syncthreads_or(same);
    if (slot < 0 || taken || slot >= p.pool) {
      if (slot >= 0 && threadIdx.x == 0) raise_index_error();
      const float zero[VEC] = {};
      if (p.clear_rest && in_dim) store_vec<T, VEC>(static_cast<T*>(p.h) + b * p.dim + ch, zero);
      return;
    }
  }
  if (!in_dim) return;
  const Vec<A, VEC> a = load_vec<A, VEC>(static_cast<const A*>(p.a) + b * p.a_row + ch);
  const Vec<T, VEC> x = load_vec<T, VEC>(static_cast<const T*>(p.x) + b * p.x_row + ch);
  float* state        = p.state + slot * p.dim + ch;
  const Vec<float, VEC> before = load_vec<float, VEC>(state);
  float h[VEC];
#pragma unroll
  for (int c = 0; c < VEC; ++c) {
    float f, u, unused;
    gate_of<GATE>(to_float(a.v[c]), to_float(x.v[c]), f, u, unused);
    h[c] = fmaf(f, before.v[c], u);
  }
  store_vec<float, VEC>(state, h);
  store_vec<T, VEC>(static_cast<T*>(p.h) + b * p.dim + ch, h);
}

// ------------------------------------------------------------------ host side

// Whether rows that begin at p, a row (and a batch) stride apart, can be read VEC elements at a time.
bool vector_rows(const void* p, size_t elem, int64_t batch_stride, int64_t row_stride, int vec) {
  return aligned(p, elem * vec) && batch_stride % vec == 0 && row_stride % vec == 0;
}

// Calls f with the types T (of x) and A (of a) and the gate as template arguments.
template <typename F>
cudaError_t for_types(int64_t type, int64_t a_type, int64_t gate, F&& f) {
  auto with_gate = [&](auto t, auto a) -> cudaError_t {
    if (gate == TCU_GATE_DECAY) return f(t, a, std::integral_constant<int, TCU_GATE_DECAY>{});
    if (gate == TCU_GATE_LOG) return f(t, a, std::integral_constant<int, TCU_GATE_LOG>{});
    return f(t, a, std::integral_constant<int, TCU_GATE_SIGMOID>{});
  };
  if (type == TCU_TYPE_F32) return with_gate(float{}, float{});
  if (type == TCU_TYPE_F16)
    return a_type == TCU_TYPE_F32 ? with_gate(__half{}, float{}) : with_gate(__half{}, __half{});
  return a_type == TCU_TYPE_F32 ? with_gate(__nv_bfloat16{}, float{}) : with_gate(__nv_bfloat16{}, __nv_bfloat16{});
}

int check_types(int64_t type, int64_t a_type, int64_t gate) {
  if (!known_type(type) || (a_type != type && a_type != TCU_TYPE_F32)) return TCU_ERR_UNSUPPORTED;
  if (gate < TCU_GATE_DECAY || gate > TCU_GATE_SIGMOID) return TCU_ERR_UNSUPPORTED;
  return TCU_OK;
}

// Blocks per sequence and column of channels: as many as it takes to give every SM two blocks, if
// the sequences have the rows for them.
int cluster_size(int64_t blocks, int64_t tokens_each, int sms) {
  int parts = 1;
  while (parts < kMaxCluster && blocks * parts < 2 * sms && tokens_each > int64_t(parts) * kChunk) parts *= 2;
  return parts;
}

cudaError_t launch_clusters(void (*kernel)(const ScanArgs), ScanArgs args, int vec, int sms, cudaStream_t st) {
  args.columns         = int((args.dim + 32 * vec - 1) / (32 * vec));
  const int64_t groups = args.batch * args.columns;
  const int64_t each   = args.offsets ? 2 * args.tokens / args.batch : args.tokens;
  const int parts      = cluster_size(groups, each, sms);
  if (groups * parts > int64_t(0x7fffffff)) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim            = dim3(unsigned(groups * parts));
  cfg.blockDim           = dim3(kWarps * 32);
  cfg.stream             = st;
  cudaLaunchAttribute attr[1];
  attr[0].id                 = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x   = unsigned(parts);
  attr[0].val.clusterDim.y   = 1;
  attr[0].val.clusterDim.z   = 1;
  cfg.attrs    = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args);
}

bool bad_sizes(int64_t batch, int64_t tokens, int64_t dim) {
  const int64_t most = int64_t(1) << 40;  // keeps every product below 2^62
  return batch < 0 || tokens < 0 || dim < 0 || batch > most || tokens > most || dim > (1 << 21) ||
         (tokens > 0 && batch > (int64_t(1) << 40) / tokens);
}

}  // namespace
}  // namespace tcu_lm

using namespace tcu_lm;

extern "C" {

size_t tcu_linear_scan_states_rows(size_t batch, size_t tokens, int packed) {
  return packed ? tokens / kChunk + batch : batch * ((tokens + kChunk - 1) / kChunk);
}

int tcu_linear_scan(const tcu_linear_scan_args* g, void* stream) {
  if (!g) return TCU_ERR_INVALID_ARG;
  if (const int e = check_types(g->type, g->a_type, g->gate)) return e;
  if (bad_sizes(g->batch, g->tokens, g->dim)) return TCU_ERR_INVALID_ARG;
  if (g->batch == 0 || g->dim == 0) return TCU_OK;
  if (g->tokens > 0 && (!g->a || !g->x || !g->h)) return TCU_ERR_INVALID_ARG;
  const size_t ea = type_bytes(g->a_type), e = type_bytes(g->type);
  if (!aligned(g->a, ea) || !aligned(g->x, e) || !aligned(g->h, e) || !aligned(g->h0, 4) || !aligned(g->last, 4) ||
      !aligned(g->states, 4) || !aligned(g->offsets, g->offsets_are_64bit ? 8 : 4))
    return TCU_ERR_INVALID_ARG;
  const int sms = sm_count();
  if (sms <= 0) return TCU_ERR_CUDA;
  ScanArgs p{};
  p.a = g->a, p.x = g->x, p.h = g->h, p.h0 = g->h0, p.last = g->last, p.states = g->states, p.offsets = g->offsets;
  p.batch = g->batch, p.tokens = g->tokens, p.dim = g->dim;
  p.a_batch = g->offsets ? 0 : g->a_batch_stride, p.a_row = g->a_row_stride;
  p.x_batch = g->offsets ? 0 : g->x_batch_stride, p.x_row = g->x_row_stride;
  p.wide = g->offsets_are_64bit != 0;
  p.clear_rest = g->offsets && g->clear_rest;
  auto fits = [&](int v) {
    return p.dim % v == 0 && vector_rows(p.a, ea, p.a_batch, p.a_row, v) && vector_rows(p.x, e, p.x_batch, p.x_row, v) &&
           aligned(p.h, e * v) && aligned(p.last, 4 * v) && aligned(p.states, 4 * v);
  };
  const cudaError_t err = for_types(g->type, g->a_type, g->gate, [&](auto t, auto a, auto gate) {
    using T = decltype(t);
    using A = decltype(a);
    constexpr int G = decltype(gate)::value;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if constexpr (sizeof(T) == 2) {
      if (fits(4)) return launch_clusters(linear_scan_kernel<T, A, G, 4>, p, 4, sms, st);
    }
    if (fits(2)) return launch_clusters(linear_scan_kernel<T, A, G, 2>, p, 2, sms, st);
    return launch_clusters(linear_scan_kernel<T, A, G, 1>, p, 1, sms, st);
  });
  return err == cudaSuccess ? TCU_OK : TCU_ERR_CUDA;
}

int tcu_linear_scan_backward(const tcu_linear_scan_backward_args* g, void* stream) {
  if (!g) return TCU_ERR_INVALID_ARG;
  if (const int e = check_types(g->type, g->a_type, g->gate)) return e;
  if (bad_sizes(g->batch, g->tokens, g->dim)) return TCU_ERR_INVALID_ARG;
  if (g->batch == 0 || g->dim == 0) return TCU_OK;
  if (g->tokens > 0 && (!g->a || !g->x || !g->da || !g->dx || !g->states)) return TCU_ERR_INVALID_ARG;
  const size_t ea = type_bytes(g->a_type), e = type_bytes(g->type);
  if (!aligned(g->a, ea) || !aligned(g->x, e) || !aligned(g->dh, e) || !aligned(g->da, ea) || !aligned(g->dx, e) ||
      !aligned(g->dlast, 4) || !aligned(g->dh0, 4) || !aligned(g->states, 4) ||
      !aligned(g->offsets, g->offsets_are_64bit ? 8 : 4))
    return TCU_ERR_INVALID_ARG;
  const int sms = sm_count();
  if (sms <= 0) return TCU_ERR_CUDA;
  ScanArgs p{};
  p.a = g->a, p.x = g->x, p.dh = g->dh, p.states = const_cast<float*>(g->states), p.dlast = g->dlast;
  p.da = g->da, p.dx = g->dx, p.dh0 = g->dh0, p.offsets = g->offsets;
  p.batch = g->batch, p.tokens = g->tokens, p.dim = g->dim;
  p.a_batch = g->offsets ? 0 : g->a_batch_stride, p.a_row = g->a_row_stride;
  p.x_batch = g->offsets ? 0 : g->x_batch_stride, p.x_row = g->x_row_stride;
  p.dh_batch = g->offsets ? 0 : g->dh_batch_stride, p.dh_row = g->dh_row_stride;
  p.wide = g->offsets_are_64bit != 0;
  p.clear_rest = g->offsets && g->clear_rest;
  auto fits = [&](int v) {
    return p.dim % v == 0 && vector_rows(p.a, ea, p.a_batch, p.a_row, v) && vector_rows(p.x, e, p.x_batch, p.x_row, v) &&
           vector_rows(p.dh, e, p.dh_batch, p.dh_row, v) && aligned(p.da, ea * v) && aligned(p.dx, e * v) &&
           aligned(p.dh0, 4 * v) && aligned(p.states, 4 * v);
  };
  const cudaError_t err = for_types(g->type, g->a_type, g->gate, [&](auto t, auto a, auto gate) {
    using T = decltype(t);
    using A = decltype(a);
    constexpr int G = decltype(gate)::value;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (fits(2)) return launch_clusters(linear_scan_backward_kernel<T, A, G, 2>, p, 2, sms, st);
    return launch_clusters(linear_scan_backward_kernel<T, A, G, 1>, p, 1, sms, st);
  });
  return err == cudaSuccess ? TCU_OK : TCU_ERR_CUDA;
}

int tcu_linear_scan_step(const tcu_linear_scan_step_args* g, void* stream) {
  if (!g) return TCU_ERR_INVALID_ARG;
  if (const int e = check_types(g->type, g->a_type, g->gate)) return e;
  if (bad_sizes(g->batch, g->pool, g->dim)) return TCU_ERR_INVALID_ARG;
  if (!g->slots && g->batch > g->pool) return TCU_ERR_INVALID_ARG;
  if (g->batch == 0 || g->dim == 0) return TCU_OK;
  if (!g->a || !g->x || !g->h || !g->state) return TCU_ERR_INVALID_ARG;
  const size_t ea = type_bytes(g->a_type), e = type_bytes(g->type);
  if (!aligned(g->a, ea) || !aligned(g->x, e) || !aligned(g->h, e) || !aligned(g->state, 4) ||
      !aligned(g->slots, g->slots_are_64bit ? 8 : 4))
    return TCU_ERR_INVALID_ARG;
  StepArgs p{};
  p.a = g->a, p.x = g->x, p.h = g->h, p.state = g->state, p.slots = g->slots;
  p.batch = g->batch, p.pool = g->pool, p.dim = g->dim, p.a_row = g->a_row_stride, p.x_row = g->x_row_stride;
  p.wide = g->slots_are_64bit != 0, p.clear_rest = g->clear_rest != 0;
  auto fits = [&](int v) {
    return p.dim % v == 0 && vector_rows(p.a, ea, 0, p.a_row, v) && vector_rows(p.x, e, 0, p.x_row, v) &&
           aligned(p.h, e * v) && aligned(p.state, 4 * v);
  };
  const cudaError_t err = for_types(g->type, g->a_type, g->gate, [&](auto t, auto a, auto gate) -> cudaError_t {
    using T = decltype(t);
    using A = decltype(a);
    constexpr int G = decltype(gate)::value;
    const int vec   = fits(4) ? 4 : 1;
    const int64_t per = int64_t(kStepThreads) * vec;
    p.blocks_per_row  = int((p.dim + per - 1) / per);
    if (p.batch > int64_t(0x7fffffff) / p.blocks_per_row) return cudaErrorInvalidConfiguration;
    const unsigned grid = unsigned(p.batch * p.blocks_per_row);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (vec == 4)
      linear_scan_step_kernel<T, A, G, 4><<<grid, kStepThreads, 0, st>>>(p);
    else
      linear_scan_step_kernel<T, A, G, 1><<<grid, kStepThreads, 0, st>>>(p);
    return cudaGetLastError();
  });
  return err == cudaSuccess ? TCU_OK : TCU_ERR_CUDA;
}

int tcu_error_word_linear_scan(unsigned int* bits, int clear) { return read_error_word(bits, clear); }

}  // extern "C"
