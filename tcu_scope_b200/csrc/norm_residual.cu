// The norms around a block, fused with the block's gate and its residual connection, and the gradient:
//     n = z / rms(z) * post        (z itself without post)
//     o = residual + scale * act(gate) * n
//     u = o / rms(o) * pre         rms(y) = sqrt(mean(y^2) + eps)
// Row sums of squares of two arrays, the second known only after the first sum: a row stays in the
// registers of one block (or warp) between its single read and its single write.
//
// Gradient, per row, with v = du pre, on = o / rms(o), zn = z / rms(z):
//     d  = do + (v - on mean(v on)) / rms(o)     = dresidual
//     dn = scale act(gate) d,   w = dn post
//     dz = (w - zn mean(w zn)) / rms(z)
//     dpre = sum over rows of du on, dpost = sum of dn zn, dgate = sum of scale act'(gate) d n
// The sums over rows are kept by every block for its own rows, in registers, and joined by a second kernel in
// the order of the blocks: no atomics, the same bits every time.
//
// Bound by HBM: 4 arrays forward, 6 backward.
#include <type_traits>

#include "lm_common.cuh"

namespace tcu_lm {
namespace {

constexpr int kNone = 0, kSigmoid = 1, kSilu = 2;

struct NormArgs {
  const void *z, *residual, *post, *gate, *pre, *dout, *dnormed;
  void *out, *normed, *dz, *dresidual;
  void* dgate;        // written where one worker holds all rows of a gate row
  float* gate_parts;  // else one row of floats per worker
  float *post_parts, *pre_parts;  // one row of floats per worker
  int64_t rows, rows_per_gate, slice_rows;
  int64_t z_row, residual_row, gate_row, dout_row, dnormed_row;
  int64_t units;      // backward: slices of the rows of one gate row
  int64_t workers;    // blocks, or warps, that take consecutive units
  int slices;         // per gate row
  int dim, act;
  float scale, eps;
};

__device__ __forceinline__ float act_of(int act, float g) {
  if (act == kNone) return g;
  const float s = __fdividef(1.f, 1.f + expf(-g));
  return act == kSigmoid ? s : g * s;
}

__device__ __forceinline__ float slope_of(int act, float g) {
  if (act == kNone) return 1.f;
  const float s = __fdividef(1.f, 1.f + expf(-g)), r = __fdividef(1.f, 1.f + expf(g));  // r = 1 - s
  return act == kSigmoid ? s * r : s * (1.f + g * r);
}

// Sum over the threads of a row: a warp (WARP) or the block.  `scratch`: 32 floats that the previous
// call did not use.  Every thread gets the sum, always added up in the same order.
template <bool WARP>
__device__ __forceinline__ float row_sum(float x, float* scratch) {
  x = warp_sum(x);
  if constexpr (WARP) return x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  if (warps == 1) return x;
  if (lane == 0) scratch[warp] = x;
  __syncthreads();
  return warp_sum(lane < warps ? scratch[lane] : 0.f);
}

// Elements v * VEC ... of a row that this thread holds, v = first, first + width, ...: E in all.
template <typename T, int VEC, int E>
__device__ __forceinline__ void load_part(float (&x)[E], const void* row, int64_t offset, int first, int width, int dim) {
  const T* p = static_cast<const T*>(row) + offset;
#pragma unroll
  for (int k = 0; k < E / VEC; ++k) {
    const int at = (first + k * width) * VEC;
    const Vec<T, VEC> r = at < dim ? load_vec<T, VEC>(p + at) : zero_vec<T, VEC>();
    float y[VEC];
    to_floats<T, VEC>(r, y);
#pragma unroll
    for (int c = 0; c < VEC; ++c) x[k * VEC + c] = y[c];
  }
}

template <typename T, int VEC, int E>
__device__ __forceinline__ void store_part(void* row, int64_t offset, const float (&x)[E], int first, int width, int dim) {
  T* p = static_cast<T*>(row) + offset;
#pragma unroll
  for (int k = 0; k < E / VEC; ++k) {
    const int at = (first + k * width) * VEC;
    float y[VEC];
#pragma unroll
    for (int c = 0; c < VEC; ++c) y[c] = x[k * VEC + c];
    if (at < dim) store_vec<T, VEC>(p + at, y);
  }
}

template <typename T, typename W, int VEC, int E, bool WARP, int THREADS>
__global__ void __launch_bounds__(THREADS)
norm_residual_kernel(const NormArgs p) {
  __shared__ float scratch[2][32];
  const int first = WARP ? threadIdx.x & 31 : threadIdx.x, width = WARP ? 32 : blockDim.x;
  const int64_t workers = WARP ? int64_t(gridDim.x) * (THREADS / 32) : gridDim.x;
  int64_t row           = WARP ? int64_t(blockIdx.x) * (THREADS / 32) + (threadIdx.x >> 5) : blockIdx.x;
  const float inv_dim   = 1.f / float(p.dim);
  for (; row < p.rows; row += workers) {
    float z[E], o[E];
    load_part<T, VEC, E>(z, p.z, row * p.z_row, first, width, p.dim);
    if (p.residual)
      load_part<T, VEC, E>(o, p.residual, row * p.residual_row, first, width, p.dim);
    else {
#pragma unroll
      for (int i = 0; i < E; ++i) o[i] = 0.f;
    }
    float rz = 1.f;
    if (p.post) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) s = fmaf(z[i], z[i], s);
      rz = rsqrtf(row_sum<WARP>(s, scratch[0]) * inv_dim + p.eps);
      float w[E];
      load_part<W, VEC, E>(w, p.post, 0, first, width, p.dim);
#pragma unroll
      for (int i = 0; i < E; ++i) z[i] *= rz * w[i];
    }
    if (p.gate) {
      float g[E];
      load_part<T, VEC, E>(g, p.gate, row / p.rows_per_gate * p.gate_row, first, width, p.dim);
#pragma unroll
      for (int i = 0; i < E; ++i) z[i] *= act_of(p.act, g[i]);
    }
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = fmaf(p.scale, z[i], o[i]);
    store_part<T, VEC, E>(p.out, row * p.dim, o, first, width, p.dim);
    if (p.pre) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) s = fmaf(o[i], o[i], s);
      const float ro = rsqrtf(row_sum<WARP>(s, scratch[1]) * inv_dim + p.eps);
      float w[E];
      load_part<W, VEC, E>(w, p.pre, 0, first, width, p.dim);
#pragma unroll
      for (int i = 0; i < E; ++i) o[i] *= ro * w[i];
      store_part<T, VEC, E>(p.normed, row * p.dim, o, first, width, p.dim);
    }
    if (!WARP && !(p.post && p.pre)) __syncthreads();  // one sum a row: its scratch is used again at once
  }
}

template <typename T, typename W, int VEC, int E, bool WARP, int THREADS>
__global__ void __launch_bounds__(THREADS)
norm_residual_backward_kernel(const NormArgs p) {
  __shared__ float scratch[4][32];
  const int first = WARP ? threadIdx.x & 31 : threadIdx.x, width = WARP ? 32 : blockDim.x;
  const int64_t workers = p.workers;
  const int64_t worker  = WARP ? int64_t(blockIdx.x) * (THREADS / 32) + (threadIdx.x >> 5) : blockIdx.x;
  if (worker >= workers) return;
  const float inv_dim = 1.f / float(p.dim);
  float dpost[E], dpre[E];
#pragma unroll
  for (int i = 0; i < E; ++i) dpost[i] = dpre[i] = 0.f;
  const int64_t unit_end = (worker + 1) * p.units / workers;
  for (int64_t unit = worker * p.units / workers; unit < unit_end; ++unit) {
    const int64_t group = unit / p.slices, slice = unit % p.slices;
    const int64_t begin = group * p.rows_per_gate + slice * p.slice_rows;
    int64_t end         = begin + p.slice_rows;
    if (end > (group + 1) * p.rows_per_gate) end = (group + 1) * p.rows_per_gate;
    float dgate[E];
#pragma unroll
    for (int i = 0; i < E; ++i) dgate[i] = 0.f;
    for (int64_t row = begin; row < end; ++row) {
      float z[E], o[E], d[E], du[E];
      load_part<T, VEC, E>(z, p.z, row * p.z_row, first, width, p.dim);
#pragma unroll
      for (int i = 0; i < E; ++i) o[i] = d[i] = du[i] = 0.f;
      if (p.pre && p.residual) load_part<T, VEC, E>(o, p.residual, row * p.residual_row, first, width, p.dim);
      if (p.dout) load_part<T, VEC, E>(d, p.dout, row * p.dout_row, first, width, p.dim);
      if (p.pre && p.dnormed) load_part<T, VEC, E>(du, p.dnormed, row * p.dnormed_row, first, width, p.dim);
      float rz = 1.f;
      if (p.post) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) s = fmaf(z[i], z[i], s);
        rz = rsqrtf(row_sum<WARP>(s, scratch[0]) * inv_dim + p.eps);
#pragma unroll
        for (int i = 0; i < E; ++i) z[i] *= rz;  // z / rms(z) from here on
      }
      float post[E], gate[E];
#pragma unroll
      for (int i = 0; i < E; ++i) post[i] = gate[i] = 1.f;
      if (p.post) load_part<W, VEC, E>(post, p.post, 0, first, width, p.dim);
      if (p.gate) {
        load_part<T, VEC, E>(gate, p.gate, group * p.gate_row, first, width, p.dim);
#pragma unroll
        for (int i = 0; i < E; ++i) gate[i] = act_of(p.act, gate[i]);
      }
      if (p.pre) {
        float pre[E], so = 0.f, sv = 0.f;
        load_part<W, VEC, E>(pre, p.pre, 0, first, width, p.dim);
#pragma unroll
        for (int i = 0; i < E; ++i) {
          o[i] = fmaf(p.scale * gate[i], z[i] * post[i], o[i]);
          so   = fmaf(o[i], o[i], so);
          sv   = fmaf(du[i] * pre[i], o[i], sv);
        }
        const float ro   = rsqrtf(row_sum<WARP>(so, scratch[1]) * inv_dim + p.eps);
        const float mean = row_sum<WARP>(sv, scratch[2]) * inv_dim * ro;  // of v on
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const float on = o[i] * ro;
          dpre[i] = fmaf(du[i], on, dpre[i]);
          d[i]    = fmaf(ro, fmaf(-on, mean, du[i] * pre[i]), d[i]);
        }
      }
      if (p.dresidual) store_part<T, VEC, E>(p.dresidual, row * p.dim, d, first, width, p.dim);
      float sw = 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        d[i] *= p.scale;
        dgate[i] = fmaf(d[i], z[i] * post[i], dgate[i]);
        d[i] *= gate[i];  // dn
        dpost[i] = fmaf(d[i], z[i], dpost[i]);
        d[i] *= post[i];  // w
        sw = fmaf(d[i], z[i], sw);
      }
      if (p.post) {
        const float mean = row_sum<WARP>(sw, scratch[3]) * inv_dim;  // of w zn
#pragma unroll
        for (int i = 0; i < E; ++i) d[i] = rz * fmaf(-z[i], mean, d[i]);
      }
      store_part<T, VEC, E>(p.dz, row * p.dim, d, first, width, p.dim);
    }
    if (p.gate && p.act != kNone) {
      float gate[E];
      load_part<T, VEC, E>(gate, p.gate, group * p.gate_row, first, width, p.dim);
#pragma unroll
      for (int i = 0; i < E; ++i) dgate[i] *= slope_of(p.act, gate[i]);
    }
    if (p.dgate) store_part<T, VEC, E>(p.dgate, group * p.dim, dgate, first, width, p.dim);
    if (p.gate_parts) store_part<float, VEC, E>(p.gate_parts, unit * p.dim, dgate, first, width, p.dim);
  }
  if (p.post_parts) store_part<float, VEC, E>(p.post_parts, worker * p.dim, dpost, first, width, p.dim);
  if (p.pre_parts) store_part<float, VEC, E>(p.pre_parts, worker * p.dim, dpre, first, width, p.dim);
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
constexpr int kMaxDim       = 16384;
constexpr int kForwardE     = 16;    // elements per thread
constexpr int kWarpThreads  = 256;   // rows that a warp holds: eight to a block
constexpr int kBackwardThreads = 148 * 1024;  // of the backward pass: 1024 on each SM

int warp_dim(int e) { return 32 * e; }

// A row's threads, whole warps.
int row_threads(int64_t dim, int e) { return int((dim + e * 32 - 1) / (e * 32) * 32); }

// Elements per thread of the backward pass: it keeps sums for each of them.
int backward_e(int64_t dim) { return dim <= 512 * 8 ? 8 : 16; }

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
  const int64_t most = kBackwardThreads / row_threads(dim, backward_e(dim));
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
    const bool wide = p.dim % V == 0 && row_vectors(p.z, e, p.z_row, V) && row_vectors(p.residual, e, p.residual_row, V) &&
                      row_vectors(p.gate, e, p.gate_row, V) && row_vectors(p.post, ew, 0, V) &&
                      row_vectors(p.pre, ew, 0, V) && aligned(p.out, 16) && aligned(p.normed, 16);
    const bool warp   = p.dim <= warp_dim(kForwardE);
    const int threads = warp ? kWarpThreads : row_threads(p.dim, kForwardE);
    const int64_t blocks = warp ? (p.rows + 7) / 8 : p.rows;
    const int64_t most   = int64_t(sms) * (2048 / threads);
    const unsigned grid  = unsigned(blocks < most ? blocks : most);
    if (wide) {
      if (warp)
        norm_residual_kernel<T, W, V, kForwardE, true, kWarpThreads><<<grid, threads, 0, st>>>(p);
      else
        norm_residual_kernel<T, W, V, kForwardE, false, 1024><<<grid, threads, 0, st>>>(p);
    } else {
      if (warp)
        norm_residual_kernel<T, W, 1, kForwardE, true, kWarpThreads><<<grid, threads, 0, st>>>(p);
      else
        norm_residual_kernel<T, W, 1, kForwardE, false, 1024><<<grid, threads, 0, st>>>(p);
    }
    return cudaGetLastError() == cudaSuccess ? TCU_OK : TCU_ERR_CUDA;
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
    const bool wide = p.dim % V == 0 && row_vectors(p.z, e, p.z_row, V) && row_vectors(p.residual, e, p.residual_row, V) &&
                      row_vectors(p.gate, e, p.gate_row, V) && row_vectors(p.dout, e, p.dout_row, V) &&
                      row_vectors(p.dnormed, e, p.dnormed_row, V) && row_vectors(p.post, ew, 0, V) &&
                      row_vectors(p.pre, ew, 0, V) && aligned(p.dz, 16) && aligned(p.dresidual, 16) && aligned(p.dgate, 16);
    auto go = [&](auto vec) {
      constexpr int VEC = decltype(vec)::value;
      if (p.dim <= warp_dim(8)) {
        const unsigned grid = unsigned((c.workers + 7) / 8);
        norm_residual_backward_kernel<T, W, VEC, 8, true, kWarpThreads><<<grid, kWarpThreads, 0, st>>>(p);
      } else if (p.dim <= 512 * 8) {
        norm_residual_backward_kernel<T, W, VEC, 8, false, 512><<<unsigned(c.workers), row_threads(p.dim, 8), 0, st>>>(p);
      } else if (p.dim <= 512 * 16) {
        norm_residual_backward_kernel<T, W, VEC, 16, false, 512><<<unsigned(c.workers), row_threads(p.dim, 16), 0, st>>>(p);
      } else {
        norm_residual_backward_kernel<T, W, VEC, 16, false, 1024><<<unsigned(c.workers), row_threads(p.dim, 16), 0, st>>>(p);
      }
    };
    if (wide)
      go(std::integral_constant<int, V>{});
    else
      go(std::integral_constant<int, 1>{});
    return cudaGetLastError() == cudaSuccess ? TCU_OK : TCU_ERR_CUDA;
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
