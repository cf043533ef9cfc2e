// The entry points of the gated linear recurrence, and its form for single tokens.
#include "linear_scan.cuh"

namespace tcu_lm {
namespace {

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
// whether an earlier row has the same one (two rows must not update a state at a time).  64 x 2048: 2.1 us, all latency.
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
    float f, rest;
    gate_of<GATE>(to_float(a.v[c]), f, rest);
    h[c] = fmaf(f, before.v[c], rest * to_float(x.v[c]));
  }
  store_vec<float, VEC>(state, h);
  store_vec<T, VEC>(static_cast<T*>(p.h) + b * p.dim + ch, h);
}

// ------------------------------------------------------------------ host side

// Whether rows that begin at p, a row stride apart, can be read VEC elements at a time.
bool vector_rows(const void* p, size_t elem, int64_t row_stride, int vec) {
  return aligned(p, elem * vec) && row_stride % vec == 0;
}

template <typename F>
cudaError_t for_type(int64_t type, F&& f) {
  if (type == TCU_TYPE_F32) return f(float{});
  return type == TCU_TYPE_F16 ? f(__half{}) : f(__nv_bfloat16{});
}

int check_types(int64_t type, int64_t a_type, int64_t gate) {
  if (!known_type(type) || (a_type != type && a_type != TCU_TYPE_F32)) return TCU_ERR_UNSUPPORTED;
  if (gate < TCU_GATE_DECAY || gate > TCU_GATE_SIGMOID) return TCU_ERR_UNSUPPORTED;
  return TCU_OK;
}

// How many bytes of rows that begin at p can be copied at a time.
int piece_of(const void* p, size_t elem, int64_t dim, int64_t batch_stride, int64_t row_stride) {
  auto fits = [&](int64_t bytes) {
    return aligned(p, bytes) && dim * int64_t(elem) % bytes == 0 && batch_stride * int64_t(elem) % bytes == 0 &&
           row_stride * int64_t(elem) % bytes == 0;
  };
  return fits(16) ? 16 : fits(4) ? 4 : int(elem);
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
  return packed ? tokens / kSpacing + batch : batch * ((tokens + kSpacing - 1) / kSpacing);
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
  p.a_piece = piece_of(p.a, ea, p.dim, p.a_batch, p.a_row), p.x_piece = piece_of(p.x, e, p.dim, p.x_batch, p.x_row);
  p.pairs   = p.dim % 2 == 0 && aligned(p.h, 2 * e);
  const cudaError_t err = for_type(g->type, [&](auto t) {
    return launch_linear_scan<decltype(t)>(p, g->a_type, g->gate, sms, static_cast<cudaStream_t>(stream));
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
  p.a_piece = piece_of(p.a, ea, p.dim, p.a_batch, p.a_row), p.x_piece = piece_of(p.x, e, p.dim, p.x_batch, p.x_row);
  p.dh_piece = piece_of(p.dh, e, p.dim, p.dh_batch, p.dh_row);
  p.pairs    = p.dim % 2 == 0 && aligned(p.da, 2 * ea) && aligned(p.dx, 2 * e);
  const cudaError_t err = for_type(g->type, [&](auto t) {
    return launch_linear_scan_backward<decltype(t)>(p, g->a_type, g->gate, sms, static_cast<cudaStream_t>(stream));
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
    return p.dim % v == 0 && vector_rows(p.a, ea, p.a_row, v) && vector_rows(p.x, e, p.x_row, v) &&
           aligned(p.h, e * v) && aligned(p.state, 4 * v);
  };
  const cudaError_t err = for_type(g->type, [&](auto t) {
    using T = decltype(t);
    return for_gates<T>(g->a_type, g->gate, [&](auto a, auto gate) -> cudaError_t {
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
  });
  return err == cudaSuccess ? TCU_OK : TCU_ERR_CUDA;
}

int tcu_error_word_linear_scan_f16(unsigned int* bits, int clear);
int tcu_error_word_linear_scan_bf16(unsigned int* bits, int clear);
int tcu_error_word_linear_scan_f32(unsigned int* bits, int clear);

int tcu_error_word_linear_scan(unsigned int* bits, int clear) {
  unsigned int each[4] = {0, 0, 0, 0};
  if (read_error_word(&each[0], clear) != TCU_OK || tcu_error_word_linear_scan_f16(&each[1], clear) != TCU_OK ||
      tcu_error_word_linear_scan_bf16(&each[2], clear) != TCU_OK || tcu_error_word_linear_scan_f32(&each[3], clear) != TCU_OK)
    return TCU_ERR_CUDA;
  *bits = each[0] | each[1] | each[2] | each[3];
  return TCU_OK;
}

}  // extern "C"
