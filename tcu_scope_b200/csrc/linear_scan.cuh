// What the translation units of the gated linear recurrence share: linear_scan.cu has the entry points and the form for
// single tokens, linear_scan_f16.cu, _bf16.cu and _f32.cu the kernels for x of one type.
#pragma once

#include <type_traits>

#include "lm_common.cuh"

namespace tcu_lm {

struct ScanArgs {
  const void *a, *x, *dh;
  void *h, *da, *dx;
  const float *h0, *dlast;
  float *last, *states, *dh0;
  const void* offsets;
  int64_t batch, tokens, dim;
  int64_t a_batch, a_row, x_batch, x_row, dh_batch, dh_row;
  int columns, stages;
  int a_piece, x_piece, dh_piece;  // bytes that can be copied at a time: 16, 4 or an element
  bool pairs;                      // outputs can be written two elements at a time
  bool wide;
  bool clear_rest;  // with offsets: rows outside all sequences become 0
};

constexpr int kSpacing = 16;  // of the states

// Launch the forward (backward) pass for x of type T; a_type: T's or TCU_TYPE_F32.
template <typename T>
cudaError_t launch_linear_scan(const ScanArgs& args, int64_t a_type, int64_t gate, int sms, cudaStream_t st);
template <typename T>
cudaError_t launch_linear_scan_backward(const ScanArgs& args, int64_t a_type, int64_t gate, int sms, cudaStream_t st);

// Calls f with the type A of a and the gate as template arguments.
template <typename T, typename F>
cudaError_t for_gates(int64_t a_type, int64_t gate, F&& f) {
  auto with_gate = [&](auto a) -> cudaError_t {
    if (gate == TCU_GATE_DECAY) return f(a, std::integral_constant<int, TCU_GATE_DECAY>{});
    if (gate == TCU_GATE_LOG) return f(a, std::integral_constant<int, TCU_GATE_LOG>{});
    return f(a, std::integral_constant<int, TCU_GATE_SIGMOID>{});
  };
  if (std::is_same<T, float>::value || a_type != TCU_TYPE_F32) return with_gate(T{});
  return with_gate(float{});
}

// f of one element, and what u takes of x: 1 - f (SIGMOID, computed without cancellation) or 1.  exp(a) = 2^(a log2(e)): the product's
// rounding makes f off by |a| half steps, relative, which is where f is small and counts for little.
template <int GATE>
__device__ __forceinline__ void gate_of(float a, float& f, float& one_minus_f) {
  if constexpr (GATE == TCU_GATE_SIGMOID) {
    const float e = exp2_fast(-fabsf(a) * kLog2E);
    const float r = reciprocal(1.f + e);
    const float s = e * r;
    f           = a >= 0.f ? r : s;
    one_minus_f = a >= 0.f ? s : r;
    if (a != a) f = one_minus_f = a;
  } else {
    f           = GATE == TCU_GATE_LOG ? exp2_fast(a * kLog2E) : a;
    one_minus_f = 1.f;  // what u takes of x
  }
}

template <int GATE>
__device__ __forceinline__ void gate_of(float2 a, float2& f, float2& one_minus_f) {
  gate_of<GATE>(a.x, f.x, one_minus_f.x);
  gate_of<GATE>(a.y, f.y, one_minus_f.y);
}

}  // namespace tcu_lm
