// Log probabilities of given tokens with the entropy and the best alternatives, and the gradient of the
// logits, for rows x_0 ... x_{V-1}:
//     lse = log sum exp(x_j),   logprob = x_target - lse,   entropy = - sum p_j log p_j,  p_j = exp(x_j - lse)
// in one pass over the row.  With the largest x so far as reference r
//     s = sum 2^d_j,  t = sum 2^d_j d_j,   d_j = (x_j - r) log2(e)
// and a larger reference r' turns (s, t) into 2^q (s, t + q s), q = (r - r') log2(e).  In the end
//     lse = r + log2(s) log 2,   entropy = (log2(s) - t / s) log 2,
// both terms of the entropy being >= 0: nothing cancels.  (x - r is taken before the product: a row
// that holds nothing but the lowest value of its type is then as even a distribution as any other.)
//
// The best k (up to 32) are found in the same pass: every warp keeps its best in its lanes, sorted, and looks
// only at elements above its k-th; ties go to the lower index, NaN counts as the largest.
//
// A row is read by the P blocks of a cluster, P > 1 where there are few rows, which join their sums
// and lists in shared memory of the first.  Bound by HBM: one read forward, a read and a write backward.
#include <cooperative_groups.h>

#include "lm_common.cuh"

namespace tcu_lm {
namespace {

namespace cg = cooperative_groups;

constexpr int kMaxCluster = 8;
constexpr int kMaxThreads = 512;
constexpr int kMaxWarps   = kMaxThreads / 32;
constexpr int kUnroll     = 4;
constexpr float kLog2E    = 1.44269504088896341f;
constexpr float kLn2      = 0.693147180559945309f;
// 2^this is 0 (subnormal results are: a probability below 2^-126 of the sum counts as none); stands for
// -inf, which 0 * -inf would turn into NaN.
constexpr float kZeroExp = -160.f;

struct LogprobArgs {
  const void *logits, *targets;
  float *logprob, *entropy, *lse, *top_logprob;
  int64_t* top_index;
  const float *in_lse, *in_entropy, *dlogprob, *dentropy;
  void* dlogits;
  int64_t rows, vocab, row_stride, ignore_index, vectors_per_block, blocks_per_row;
  int top;
  bool wide;
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The larger of two, NaN if one is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// Whole numbers that order as the values do: -0 as 0, NaN above all; never 0.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) {
  if (o == 0xffffffffu) return __uint_as_float(0x7fffffffu);
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

// Sum of exponentials against a reference.
struct Sums {
  float ref = -INFINITY, s = 0.f, t = 0.f;
};

__device__ __forceinline__ void rebase(Sums& a, float ref) {
  if (a.ref == ref || a.s == 0.f) {  // s is 0 while everything so far was -inf
    a.ref = ref;
    return;
  }
  const float q = (a.ref - ref) * kLog2E, f = exp2_fast(q);
  a.t   = q <= kZeroExp ? 0.f : f * fmaf(q, a.s, a.t);
  a.s *= f;
  a.ref = ref;
}

__device__ __forceinline__ void join(Sums& a, Sums b) {
  const float ref = max_nan(a.ref, b.ref);
  if (ref == -INFINITY) return;
  rebase(a, ref);
  rebase(b, ref);
  a.s += b.s;
  a.t += b.t;
}

template <typename T>
constexpr int kVec = 16 / int(sizeof(T));

// A row as 16-byte vectors: vector v holds elements v * kVec - shift ..., the first and the last may
// reach over the row's ends.
template <typename T>
struct Row {
  const T* p;
  int64_t vocab, shift, vectors;
  __device__ __forceinline__ Row(const T* row, int64_t n) : p(row), vocab(n) {
    shift   = int64_t(reinterpret_cast<uintptr_t>(row) % 16) / int64_t(sizeof(T));
    vectors = (shift + n + kVec<T> - 1) / kVec<T>;
  }
  __device__ __forceinline__ int64_t element(int64_t v) const { return v * kVec<T> - shift; }
  // vector v; -inf where it lies outside the row
  __device__ __forceinline__ Vec<T, kVec<T>> load(int64_t v) const {
    const int64_t e = element(v);
    if (e >= 0 && e + kVec<T> <= vocab) return load_vec<T, kVec<T>>(p + e);
    Vec<T, kVec<T>> r;
#pragma unroll
    for (int c = 0; c < kVec<T>; ++c)
      r.v[c] = e + c >= 0 && e + c < vocab ? p[e + c] : from_float<T>(-INFINITY);
    return r;
  }
};

// Adds the elements of a vector, none of them above a.ref.
template <typename T>
__device__ __forceinline__ void add_vector(Sums& a, const Vec<T, kVec<T>>& x) {
  const float ref = a.ref == -INFINITY ? 0.f : a.ref;
#pragma unroll
  for (int c = 0; c < kVec<T>; ++c) {
    const float d = max_nan((to_float(x.v[c]) - ref) * kLog2E, kZeroExp);
    const float e = exp2_fast(d);
    a.s += e;
    a.t = fmaf(e, d, a.t);
  }
}

__device__ __forceinline__ Sums join_warp(Sums a) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Sums b;
    b.ref = __shfl_xor_sync(0xffffffffu, a.ref, o);
    b.s   = __shfl_xor_sync(0xffffffffu, a.s, o);
    b.t   = __shfl_xor_sync(0xffffffffu, a.t, o);
    join(a, b);
  }
  return a;
}

using Key = unsigned long long;

__device__ __forceinline__ Key key_of(float x, int64_t index) {
  return Key(order_of(x)) << 32 | uint32_t(~uint32_t(index));
}

// The best of a warp, sorted, one in each lane; 0 is none.
__device__ __forceinline__ Key merge_best(Key mine, Key other_reversed, int lane) {
  Key x = mine > other_reversed ? mine : other_reversed;  // the 32 largest, a bitonic sequence
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Key y = __shfl_xor_sync(0xffffffffu, x, o);
    x = (lane & o) == 0 ? (x > y ? x : y) : (x < y ? x : y);
  }
  return x;
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(kMaxThreads, 2)
token_logprobs_kernel(const LogprobArgs p) {
  __shared__ Sums warp_sums[kMaxWarps], block_sums[kMaxCluster];
  __shared__ Key warp_best[TOP ? kMaxWarps : 1][32], block_best[TOP ? kMaxCluster : 1][32];
  __shared__ uint32_t shared_bar;  // the largest k-th best of the block's warps: nothing below it matters
  const cg::cluster_group cluster = cg::this_cluster();
  const int parts = int(cluster.num_blocks()), part = int(cluster.block_rank());
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int64_t r = blockIdx.x / parts;
  const T* logits = static_cast<const T*>(p.logits) + r * p.row_stride;
  const Row<T> row(logits, p.vocab);
  constexpr int V = kVec<T>;
  if (TOP && threadIdx.x == 0) shared_bar = 0;
  if (parts > 1) cluster.sync();  // no block writes to another's shared memory before that has begun
  else if (TOP) __syncthreads();

  Sums a;
  Key best   = 0;
  float kth  = 0.f;   // value of the k-th best, once there are k
  bool full  = false;
  float gate = -INFINITY;  // before that: a value that k elements of this warp are known to reach
  bool fresh = true;
  const int64_t begin = row.vectors * part / parts, end = row.vectors * (part + 1) / parts;
  for (int64_t v0 = begin + warp * 32; v0 < end; v0 += int64_t(blockDim.x) * kUnroll) {
    Vec<T, V> raw[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      const int64_t v = v0 + int64_t(k) * blockDim.x + lane;
      if (v < end) raw[k] = row.load(v);
      else {
#pragma unroll
        for (int c = 0; c < V; ++c) raw[k].v[c] = from_float<T>(-INFINITY);
      }
    }
    float most[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      most[k] = to_float(raw[k].v[0]);
#pragma unroll
      for (int c = 1; c < V; ++c) most[k] = max_nan(most[k], to_float(raw[k].v[c]));
    }
    float m = most[0];
#pragma unroll
    for (int k = 1; k < kUnroll; ++k) m = max_nan(m, most[k]);
    if (!(m <= a.ref)) rebase(a, m);
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) add_vector<T>(a, raw[k]);
    if constexpr (TOP) {
      const float bar = value_of(*static_cast<volatile uint32_t*>(&shared_bar));  // NaN while it is 0
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        if (fresh) {
          // the k-th largest of the lanes' largest: sorted as whole numbers, lane by lane
          uint32_t x = order_of(most[k]);
#pragma unroll
          for (int size = 2; size <= 32; size <<= 1) {
#pragma unroll
            for (int o = size >> 1; o > 0; o >>= 1) {
              const uint32_t y = __shfl_xor_sync(0xffffffffu, x, o);
              const bool down  = (lane & size) == 0 || size == 32;
              x = ((lane & o) == 0) == down ? (x > y ? x : y) : (x < y ? x : y);
            }
          }
          const float floor = value_of(__shfl_sync(0xffffffffu, x, p.top - 1));
          gate  = floor != floor ? INFINITY : floor;
          fresh = false;
        }
        const int64_t v = v0 + int64_t(k) * blockDim.x + lane;
        const int64_t e = row.element(v);
        uint32_t pending = 0;
        if (v < end && (full ? !(most[k] <= kth) : !(most[k] < gate)) && !(most[k] < bar)) {
#pragma unroll
          for (int c = 0; c < V; ++c) {
            const float x = to_float(raw[k].v[c]);
            if ((full ? !(x <= kth) : !(x < gate)) && !(x < bar) && e + c >= 0 && e + c < p.vocab) pending |= 1u << c;
          }
        }
        uint32_t lanes;
        bool changed = false;
        while ((lanes = __ballot_sync(0xffffffffu, pending != 0)) != 0) {
          const int from = __ffs(lanes) - 1, c = __ffs(pending) - 1;
          float x = 0.f;
#pragma unroll
          for (int i = 0; i < V; ++i) x = i == c ? to_float(raw[k].v[i]) : x;
          const Key cand = __shfl_sync(0xffffffffu, key_of(x, e + c), from);
          if (lane == from) pending &= pending - 1;
          const int place = __popc(__ballot_sync(0xffffffffu, best > cand));
          if (place >= p.top) continue;
          const Key above = __shfl_up_sync(0xffffffffu, best, 1);
          best    = lane < place ? best : lane == place ? cand : above;
          changed = true;
        }
        if (changed) {
          const Key last = __shfl_sync(0xffffffffu, best, p.top - 1);
          if (last != 0) {
            full = true;
            kth  = value_of(uint32_t(last >> 32));
            if (lane == 0) atomicMax(&shared_bar, uint32_t(last >> 32));
          }
        }
      }
    }
  }

  a = join_warp(a);
  if (lane == 0) warp_sums[warp] = a;
  if constexpr (TOP) warp_best[warp][lane] = best;
  __syncthreads();
  if (warp == 0) {
    a = warp_sums[0];
    for (int w = 1; w < warps; ++w) join(a, warp_sums[w]);
    if constexpr (TOP)
      for (int w = 1; w < warps; ++w) best = merge_best(best, warp_best[w][31 - lane], lane);
  }
  if (parts > 1) {
    if (warp == 0) {
      if (lane == 0) *cluster.map_shared_rank(&block_sums[part], 0) = a;
      if constexpr (TOP) cluster.map_shared_rank(block_best[part], 0)[lane] = best;
    }
    cluster.sync();
    if (part != 0) return;
    if (warp == 0) {
      for (int q = 1; q < parts; ++q) {
        join(a, block_sums[q]);
        if constexpr (TOP) best = merge_best(best, block_best[q][31 - lane], lane);
      }
    }
  }
  if (warp != 0) return;
  const float log_s = log2f(a.s);  // a row of -inf: s = 0
  const float lse   = a.s == 0.f ? -INFINITY : fmaf(log_s, kLn2, a.ref);
  // an element's log probability, from the reference: more exact than x - lse
  auto logprob_of = [&](float x) {
    return a.s == 0.f || x == -INFINITY ? (lse != lse ? lse : -INFINITY) : fmaf(-log_s, kLn2, x - a.ref);
  };
  if (lane == 0) {
    if (p.lse) p.lse[r] = lse;
    if (p.entropy) p.entropy[r] = a.s == 0.f ? 0.f : (log_s - a.t / a.s) * kLn2;
    if (p.logprob) {
      const int64_t target = load_index(p.targets, r, p.wide);
      float lp = 0.f;
      if (target >= 0 && target < p.vocab && target != p.ignore_index)
        lp = logprob_of(to_float(logits[target]));
      else if (target != p.ignore_index)
        raise_index_error();
      p.logprob[r] = lp;
    }
  }
  if constexpr (TOP) {
    if (lane < p.top) {
      p.top_logprob[r * p.top + lane] = logprob_of(value_of(uint32_t(best >> 32)));
      p.top_index[r * p.top + lane]   = int64_t(uint32_t(~uint32_t(best)));
    }
  }
}

constexpr int kBackThreads = 256;

// Above this size lse has lost more than 2^-16 of log p to its own rounding, and the gradient goes by the
// row's largest element and the sum against it instead, for which every block reads the row once more.
constexpr float kExactLse = 256.f;

template <typename T>
__device__ __noinline__ Sums block_row_sums(const Row<T>& row, Sums* scratch) {
  Sums a;
  for (int64_t v = threadIdx.x; v < row.vectors; v += kBackThreads) {
    const Vec<T, kVec<T>> x = row.load(v);
    float m = to_float(x.v[0]);
#pragma unroll
    for (int c = 1; c < kVec<T>; ++c) m = max_nan(m, to_float(x.v[c]));
    if (!(m <= a.ref)) rebase(a, m);
    add_vector<T>(a, x);
  }
  a = join_warp(a);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = a;
  __syncthreads();
  a = scratch[0];
  for (int w = 1; w < kBackThreads / 32; ++w) join(a, scratch[w]);
  return a;
}

// dx_j = dlp ([j = target] - p_j) - dH p_j (log p_j + H), H the entropy.
template <typename T>
__global__ void __launch_bounds__(kBackThreads)
token_logprobs_backward_kernel(const LogprobArgs p) {
  __shared__ Sums scratch[kBackThreads / 32];
  constexpr int V   = kVec<T>;
  const int64_t r   = blockIdx.x / p.blocks_per_row;
  const T* logits   = static_cast<const T*>(p.logits) + r * p.row_stride;
  T* out            = static_cast<T*>(p.dlogits) + r * p.vocab;
  const Row<T> row(logits, p.vocab);
  const bool same_shift = (reinterpret_cast<uintptr_t>(out) - reinterpret_cast<uintptr_t>(logits)) % 16 == 0;
  const float lse = p.in_lse[r], entropy = p.in_entropy ? p.in_entropy[r] : 0.f;
  const bool empty = lse == -INFINITY;  // every element -inf: no gradient
  float dlp = p.dlogprob ? p.dlogprob[r] : 0.f;
  const float dent = p.dentropy ? p.dentropy[r] : 0.f;
  int64_t target = -1;
  if (p.dlogprob) {
    target = load_index(p.targets, r, p.wide);
    if (target < 0 || target >= p.vocab || target == p.ignore_index) {
      if (target != p.ignore_index && threadIdx.x == 0) raise_index_error();
      target = -1;
      dlp    = 0.f;
    }
  }
  if (empty) target = -1;
  // log2 p = (x - ref) log2(e) - shift
  float ref = empty ? 0.f : lse, shift = 0.f;
  if (!empty && fabsf(lse) > kExactLse) {
    const Sums a = block_row_sums<T>(row, scratch);
    ref   = a.ref;
    shift = log2f(a.s);
  }
  const float c0 = -fmaf(dent, entropy, dlp), c1 = -dent * kLn2;
  const int64_t begin = (blockIdx.x % p.blocks_per_row) * p.vectors_per_block;
  const int64_t end   = begin + p.vectors_per_block < row.vectors ? begin + p.vectors_per_block : row.vectors;
  for (int64_t v0 = begin + threadIdx.x; v0 < end; v0 += kBackThreads * kUnroll) {
    Vec<T, V> raw[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k)
      if (v0 + k * kBackThreads < end) raw[k] = row.load(v0 + k * kBackThreads);
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      const int64_t v = v0 + k * kBackThreads;
      if (v >= end) break;
      const int64_t e = row.element(v);
      float g[V];
#pragma unroll
      for (int c = 0; c < V; ++c) {
        const float d = max_nan(fmaf(to_float(raw[k].v[c]) - ref, kLog2E, -shift), kZeroExp);  // log2 p
        g[c]          = exp2_fast(d) * fmaf(c1, d, c0);
        if (e + c == target) g[c] += dlp;
      }
      if (same_shift && e >= 0 && e + V <= p.vocab)
        store_vec<T, V>(out + e, g);
      else {
#pragma unroll
        for (int c = 0; c < V; ++c)
          if (e + c >= 0 && e + c < p.vocab) out[e + c] = from_float<T>(g[c]);
      }
    }
  }
}

// ------------------------------------------------------------------ host side
template <typename F>
cudaError_t for_type(int64_t type, F&& f) {
  if (type == TCU_TYPE_F32) return f(float{});
  return type == TCU_TYPE_F16 ? f(__half{}) : f(__nv_bfloat16{});
}

int check_logits(const void* logits, int64_t type, int64_t rows, int64_t vocab) {
  if (!known_type(type)) return TCU_ERR_UNSUPPORTED;
  if (rows < 0 || vocab < 0 || rows > 0x7fffffff || vocab > 0x7fffffff) return TCU_ERR_INVALID_ARG;
  if (rows > 0 && (vocab == 0 || !logits)) return TCU_ERR_INVALID_ARG;
  return aligned(logits, type_bytes(type)) ? TCU_OK : TCU_ERR_INVALID_ARG;
}

}  // namespace
}  // namespace tcu_lm

using namespace tcu_lm;

extern "C" {

int tcu_token_logprobs(const tcu_token_logprobs_args* g, void* stream) {
  if (!g) return TCU_ERR_INVALID_ARG;
  if (const int e = check_logits(g->logits, g->type, g->rows, g->vocab)) return e;
  if (g->top < 0 || g->top > TCU_MAX_TOP) return TCU_ERR_UNSUPPORTED;
  if (g->rows == 0) return TCU_OK;
  if (g->top > g->vocab || (g->top > 0 && (!g->top_logprob || !g->top_index)) || (g->logprob && !g->targets))
    return TCU_ERR_INVALID_ARG;
  if (!aligned(g->targets, g->targets_are_64bit ? 8 : 4) || !aligned(g->logprob, 4) || !aligned(g->entropy, 4) ||
      !aligned(g->lse, 4) || !aligned(g->top_logprob, 4) || !aligned(g->top_index, 8))
    return TCU_ERR_INVALID_ARG;
  const int sms = sm_count();
  if (sms <= 0) return TCU_ERR_CUDA;
  LogprobArgs p{};
  p.logits = g->logits, p.targets = g->targets, p.logprob = g->logprob, p.entropy = g->entropy, p.lse = g->lse;
  p.top_logprob = g->top_logprob, p.top_index = g->top_index;
  p.rows = g->rows, p.vocab = g->vocab, p.row_stride = g->row_stride, p.ignore_index = g->ignore_index;
  p.top = int(g->top), p.wide = g->targets_are_64bit != 0;
  const cudaError_t err = for_type(g->type, [&](auto t) {
    using T = decltype(t);
    const int64_t vectors = (p.vocab + kVec<T> - 1) / kVec<T> + 1;
    int parts = 1;
    while (parts < kMaxCluster && p.rows * parts < 2 * sms && vectors > int64_t(parts) * kMaxThreads) parts *= 2;
    const int64_t want = ((vectors + parts - 1) / parts + kUnroll - 1) / kUnroll;
    const int threads  = want >= kMaxThreads ? kMaxThreads : int((want + 31) / 32 * 32);
    if (p.rows * parts > int64_t(0x7fffffff)) return cudaErrorInvalidConfiguration;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim            = dim3(unsigned(p.rows * parts));
    cfg.blockDim           = dim3(threads);
    cfg.stream             = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id               = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(parts);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs    = attr;
    cfg.numAttrs = 1;
    return p.top > 0 ? cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, true>, p)
                     : cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, false>, p);
  });
  return err == cudaSuccess ? TCU_OK : TCU_ERR_CUDA;
}

int tcu_token_logprobs_backward(const tcu_token_logprobs_backward_args* g, void* stream) {
  if (!g) return TCU_ERR_INVALID_ARG;
  if (const int e = check_logits(g->logits, g->type, g->rows, g->vocab)) return e;
  if (g->rows == 0) return TCU_OK;
  if (!g->lse || !g->dlogits || (g->dlogprob && !g->targets) || (g->dentropy && !g->entropy)) return TCU_ERR_INVALID_ARG;
  if (!aligned(g->targets, g->targets_are_64bit ? 8 : 4) || !aligned(g->lse, 4) || !aligned(g->entropy, 4) ||
      !aligned(g->dlogprob, 4) || !aligned(g->dentropy, 4) || !aligned(g->dlogits, type_bytes(g->type)))
    return TCU_ERR_INVALID_ARG;
  LogprobArgs p{};
  p.logits = g->logits, p.targets = g->targets, p.in_lse = g->lse, p.in_entropy = g->entropy;
  p.dlogprob = g->dlogprob, p.dentropy = g->dentropy, p.dlogits = g->dlogits;
  p.rows = g->rows, p.vocab = g->vocab, p.row_stride = g->row_stride, p.ignore_index = g->ignore_index;
  p.wide = g->targets_are_64bit != 0;
  const cudaError_t err = for_type(g->type, [&](auto t) {
    using T = decltype(t);
    const int64_t vectors = (p.vocab + kVec<T> - 1) / kVec<T> + 1;
    p.vectors_per_block   = kBackThreads * kUnroll;
    p.blocks_per_row      = (vectors + p.vectors_per_block - 1) / p.vectors_per_block;
    if (p.rows * p.blocks_per_row > int64_t(0x7fffffff)) return cudaErrorInvalidConfiguration;
    token_logprobs_backward_kernel<T>
        <<<unsigned(p.rows * p.blocks_per_row), kBackThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
    return cudaGetLastError();
  });
  return err == cudaSuccess ? TCU_OK : TCU_ERR_CUDA;
}

int tcu_error_word_token_logprobs(unsigned int* bits, int clear) { return read_error_word(bits, clear); }

}  // extern "C"
