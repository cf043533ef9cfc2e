// The gated linear recurrence and its gradient for x of one type (see linear_scan_kernels.cuh).
#include "linear_scan_kernels.cuh"

namespace tcu_lm {
template cudaError_t launch_linear_scan<float>(const ScanArgs&, int64_t, int64_t, int, cudaStream_t);
template cudaError_t launch_linear_scan_backward<float>(const ScanArgs&, int64_t, int64_t, int, cudaStream_t);
}  // namespace tcu_lm

extern "C" int tcu_error_word_linear_scan_f32(unsigned int* bits, int clear) { return tcu_lm::read_error_word(bits, clear); }
