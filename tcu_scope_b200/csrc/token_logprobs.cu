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
// The best k (up to 32) are found in the same pass: a block's first vectors give a bar that k elements are
// known to reach, the few elements that reach it are set aside, and in the end each of them counts how many are
// better.  Ties go to the lower index, NaN counts as the largest.
//
// A row is read by the P blocks of a cluster, P > 1 where there are few rows, which join their sums
// and lists in shared memory of the first.  Bound by HBM: one read forward, a read and a write backward.
// Measured, bf16: 4096 x 128000 164 ... 175 us (97 ... 91 % of the copy bandwidth) without, 212 us with 8 alternatives: 64 % of
// the issue slots are taken, and 56 % of what the exponentials' unit can do; gradient of 2048 x 100003 141 us (88 %).
#include <cooperative_groups.h>

#include <type_traits>

#include "lm_common.cuh"

namespace tcu_lm {
namespace {

namespace cg = cooperative_groups;

constexpr int kMaxCluster = 8;
constexpr int kMaxThreads = 256;
constexpr int kBlocksPerSm = 4;
constexpr int kMaxWarps   = kMaxThreads / 32;
constexpr int kUnroll     = 4;
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

// ------------------------------------------------------------------ rows
// 16 bytes of logits: kVec<T> elements, kVec<T> / 2 pairs.
template <typename T>
constexpr int kVec = 16 / int(sizeof(T));

// Elements far below the reference are first raised to kFloor<T>, whose exponential is 0 against any
// reference for which near_reference() holds: no -inf, of which 0 * -inf makes NaN, gets any further.
template <typename T>
struct Limits {
  static constexpr float kFloor = -1e38f;
  static __device__ __forceinline__ bool near_reference(float ref) { return fabsf(ref) < 1e37f; }
};
template <>
struct Limits<__half> {
  static constexpr float kFloor = -65504.f;
  static __device__ __forceinline__ bool near_reference(float ref) { return ref > -60000.f; }
};

template <typename T>
struct Block16 {
  uint4 w;

  __device__ __forceinline__ void fill(float x) {
    Vec<T, kVec<T>> v;
#pragma unroll
    for (int c = 0; c < kVec<T>; ++c) v.v[c] = from_float<T>(x);
    w = *reinterpret_cast<uint4*>(&v);
  }
  __device__ __forceinline__ uint32_t word(int i) const { return i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w; }
  __device__ __forceinline__ float2 pair(int i) const {
    if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(word(2 * i)), __uint_as_float(word(2 * i + 1)));
    else return unpack_pair<T>(word(i));
  }
  __device__ __forceinline__ float element(int c) const {
    const float2 x = pair(c / 2);
    return c & 1 ? x.y : x.x;
  }
  // the largest element, NaN if there is one
  __device__ __forceinline__ float most() const {
    if constexpr (sizeof(T) == 4) {
      return max_nan(max_nan(element(0), element(1)), max_nan(element(2), element(3)));
    } else {
      using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
      auto as2 = [](uint32_t x) { return *reinterpret_cast<T2*>(&x); };
      const T2 m = __hmax2_nan(__hmax2_nan(as2(w.x), as2(w.y)), __hmax2_nan(as2(w.z), as2(w.w)));
      return max_nan(to_float(m.x), to_float(m.y));
    }
  }
  // pair i, with what is below `floor` raised to it (no NaN)
  __device__ __forceinline__ float2 raised(int i, float floor) const {
    if constexpr (sizeof(T) == 4) {
      const float2 x = pair(i);
      return make_float2(fmaxf(x.x, floor), fmaxf(x.y, floor));
    } else {
      using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
      const uint32_t x = word(i);
      T2 f;
      f.x = f.y = from_float<T>(floor);
      Block16 r;
      const T2 m = __hmax2(*reinterpret_cast<const T2*>(&x), f);
      r.w.x = *reinterpret_cast<const uint32_t*>(&m);
      return r.pair(0);
    }
  }
};

// A row as 16-byte vectors: vector v holds elements v * kVec - shift ..., the first and the last may
// reach over the row's ends.
template <typename T>
struct Row {
  const uint4* p;  // of vector 0
  int vocab, shift, vectors;
  __device__ __forceinline__ Row(const T* row, int64_t n) : vocab(int(n)) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(row);
    shift   = int(at % 16) / int(sizeof(T));
    vectors = int((shift + n + kVec<T> - 1) / kVec<T>);
    p       = reinterpret_cast<const uint4*>(at - at % 16);
  }
  __device__ __forceinline__ const T* first() const { return reinterpret_cast<const T*>(p) + shift; }
  __device__ __forceinline__ int element(int v) const { return v * kVec<T> - shift; }
  __device__ __forceinline__ bool whole(int v) const {
    const int e = element(v);
    return e >= 0 && e <= vocab - kVec<T>;
  }
  // vector v; -inf where it lies outside the row
  __device__ __forceinline__ Block16<T> load(int v) const {
    Block16<T> r;
    if (whole(v)) {
      r.w = p[v];
      return r;
    }
    Vec<T, kVec<T>> x;
    const int e = element(v);
#pragma unroll
    for (int c = 0; c < kVec<T>; ++c)
      x.v[c] = e + c >= 0 && e + c < vocab ? first()[e + c] : from_float<T>(-INFINITY);
    r.w = *reinterpret_cast<uint4*>(&x);
    return r;
  }
};

// The largest element of N vectors, NaN if there is one.
template <typename T, int N>
__device__ __forceinline__ float most_of(const Block16<T> (&x)[N]) {
  if constexpr (sizeof(T) == 4) {
    float m = x[0].most();
#pragma unroll
    for (int k = 1; k < N; ++k) m = max_nan(m, x[k].most());
    return m;
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    auto as2 = [](uint32_t w) { return *reinterpret_cast<T2*>(&w); };
    T2 m = as2(x[0].w.x);
#pragma unroll
    for (int i = 1; i < 4 * N; ++i) m = __hmax2_nan(m, as2(x[i / 4].word(i % 4)));
    return max_nan(to_float(m.x), to_float(m.y));
  }
}

// ------------------------------------------------------------------ sums of exponentials
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

// The sums of a warp's lanes, in every lane.
__device__ __forceinline__ Sums join_warp(Sums a) {
  float ref = a.ref;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ref = max_nan(ref, __shfl_xor_sync(0xffffffffu, ref, o));
  if (ref != -INFINITY) rebase(a, ref);
  a.s = warp_sum(a.s);
  a.t = warp_sum(a.t);
  return a;
}

// Adds the elements of N vectors, the largest of which is `most`.
template <typename T, int N>
__device__ __forceinline__ void add_vectors(Sums& a, const Block16<T> (&x)[N], float most) {
  if (!(most <= a.ref)) rebase(a, most);
  if (Limits<T>::near_reference(a.ref)) {
    float2 s = make_float2(a.s, 0.f), t = make_float2(a.t, 0.f);
    const float2 minus_ref = both(-a.ref), scale = both(kLog2E);
#pragma unroll
    for (int k = 0; k < N; ++k) {
#pragma unroll
      for (int i = 0; i < kVec<T> / 2; ++i) {
        const float2 d = mul2(add2(x[k].raised(i, Limits<T>::kFloor), minus_ref), scale);
        const float2 e = make_float2(exp2_fast(d.x), exp2_fast(d.y));
        s = add2(s, e);
        t = fma2(e, d, t);
      }
    }
    a.s = s.x + s.y;
    a.t = t.x + t.y;
    return;
  }
  const float ref = a.ref == -INFINITY ? 0.f : a.ref;
#pragma unroll
  for (int k = 0; k < N; ++k) {
#pragma unroll 1
    for (int c = 0; c < kVec<T>; ++c) {
      const float d = max_nan((x[k].element(c) - ref) * kLog2E, kZeroExp);
      const float e = exp2_fast(d);
      a.s += e;
      a.t = fmaf(e, d, a.t);
    }
  }
}

// ------------------------------------------------------------------ the best alternatives
using Key = unsigned long long;

__device__ __forceinline__ Key key_of(float x, int index) {
  return Key(order_of(x)) << 32 | uint32_t(~uint32_t(index));
}

// What may be among the best: vectors with an element not below a bar that k elements of the row are
// known to reach, and, in the end, the keys of those elements, -inf apart.
constexpr int kSetAside = 1024;

struct Candidates {
  Key key[kSetAside];
  uint4 vector[kSetAside];
  int place[kSetAside];
  uint32_t group[2][64];
  int vectors, count;
};

// 32 whole numbers, one in each lane, sorted: the largest in lane 0.
__device__ __forceinline__ uint32_t sort_lanes(uint32_t x, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1) {
#pragma unroll
    for (int o = size >> 1; o > 0; o >>= 1) {
      const uint32_t y = __shfl_xor_sync(0xffffffffu, x, o);
      const bool down  = (lane & size) == 0 || size == 32;
      x = ((lane & o) == 0) == down ? (x > y ? x : y) : (x < y ? x : y);
    }
  }
  return x;
}

// A bar below which none of the best k lies: the block's threads make groups, k of which hold an element
// that reaches the k-th largest of the groups' largest.  `most`: of what this thread holds so far.  32 groups, or 64
// where k is more than half of 32: the 32nd of 32 would be a low bar (of 128000 normal numbers, 1000 reach it; the 32nd
// of 64, 350).  A block of one warp has 32 threads and as many groups.  Two calls in a row use different `group`s.
__device__ __forceinline__ float bar_of(float most, int k, uint32_t* group) {
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;  // 2^n warps
  const bool more = k > 16 && warps > 1;
  const int width = more ? warps / 2 : warps;  // lanes in a group
  uint32_t x = order_of(most);
  for (int o = 1; o < width; o <<= 1) {
    const uint32_t y = __shfl_xor_sync(0xffffffffu, x, o);
    x = x > y ? x : y;
  }
  if ((lane & (width - 1)) == 0) group[threadIdx.x / width] = x;
  __syncthreads();
  x = sort_lanes(group[lane], lane);
  if (more) {
    const uint32_t y = __shfl_sync(0xffffffffu, sort_lanes(group[32 + lane], lane), 31 - lane);
    x = x > y ? x : y;  // the 32 largest of both, a bitonic sequence
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const uint32_t z = __shfl_xor_sync(0xffffffffu, x, o);
      x = (lane & o) == 0 ? (x > z ? x : z) : (x < z ? x : z);
    }
  }
  return value_of(__shfl_sync(0xffffffffu, x, k - 1));
}

// (-inf, with which vectors behind the end are filled, is no candidate)
__device__ __forceinline__ void set_aside(Candidates& c, uint4 x, int v) {
  const int at = atomicAdd(&c.vectors, 1);
  if (at < kSetAside) c.vector[at] = x, c.place[at] = v;
}

// The keys of what was set aside, by all threads of the block; false if there are too many or fewer than k.
template <typename T>
__device__ __forceinline__ bool collect(Candidates& c, const Row<T>& row, int k, float bar) {
  constexpr int V = kVec<T>;
  const int n = c.vectors;
  if (n <= kSetAside) {
    for (int i = threadIdx.x; i < n * V; i += blockDim.x) {
      const float x = to_float(reinterpret_cast<const T*>(&c.vector[i / V])[i % V]);
      const int e   = row.element(c.place[i / V]) + i % V;
      if (x < bar || x == -INFINITY || e < 0 || e >= row.vocab) continue;
      const int at = atomicAdd(&c.count, 1);
      if (at < kSetAside) c.key[at] = key_of(x, e);
    }
  }
  __syncthreads();
  return n <= kSetAside && c.count >= k && c.count <= kSetAside;
}

// best[r] = the key that r of the n keys are greater than, for r < k.
__device__ __forceinline__ void rank_keys(const Key* keys, int n, int k, Key* best) {
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const Key mine = keys[i];
    int above = 0;
    for (int j = 0; j < n; ++j) above += keys[j] > mine;
    if (above < k) best[above] = mine;
  }
}

// The best of two sorted lists of 32, one key in each lane, the second one reversed; 0 is none.
__device__ __forceinline__ Key merge_best(Key mine, Key other_reversed, int lane) {
  Key x = mine > other_reversed ? mine : other_reversed;  // the 32 largest, a bitonic sequence
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Key y = __shfl_xor_sync(0xffffffffu, x, o);
    x = (lane & o) == 0 ? (x > y ? x : y) : (x < y ? x : y);
  }
  return x;
}

// Where there were too many candidates (a row that rises steadily) or fewer than k (a row with fewer tokens
// left than alternatives asked for): every warp reads its part of vectors begin ... end-1 again and keeps its best,
// sorted, one in each lane.  lists: 32 keys for each warp.
template <typename T>
__device__ __noinline__ void best_by_insertion(const Row<T>& row, int begin, int end, int k, Key* lists, Key* best_out) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  Key best  = 0;
  float kth = 0.f;  // value of the k-th best, once there are k
  bool full = false;
  for (int v0 = begin + warp * 32; v0 < end; v0 += blockDim.x) {
    const int v = v0 + lane, e = row.element(v);
    Block16<T> x;
    uint32_t pending = 0;
    if (v < end) {
      x = row.load(v);
      for (int c = 0; c < kVec<T>; ++c)
        if ((!full || !(x.element(c) <= kth)) && e + c >= 0 && e + c < row.vocab) pending |= 1u << c;
    }
    uint32_t lanes;
    while ((lanes = __ballot_sync(0xffffffffu, pending != 0)) != 0) {
      const int from = __ffs(lanes) - 1, c = pending ? __ffs(pending) - 1 : 0;
      const Key cand = __shfl_sync(0xffffffffu, key_of(x.element(c), e + c), from);
      if (lane == from) pending &= pending - 1;
      const int place = __popc(__ballot_sync(0xffffffffu, best > cand));
      const Key above = __shfl_up_sync(0xffffffffu, best, 1);
      if (place < 32) best = lane < place ? best : lane == place ? cand : above;
    }
    const Key last = __shfl_sync(0xffffffffu, best, k - 1);
    full = last != 0;
    kth  = value_of(uint32_t(last >> 32));
  }
  lists[warp * 32 + lane] = best;
  __syncthreads();
  if (warp == 0) {
    for (int w = 1; w < warps; ++w) best = merge_best(best, lists[w * 32 + 31 - lane], lane);
    if (lane < k) best_out[lane] = best;
  }
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(kMaxThreads, kBlocksPerSm)
token_logprobs_kernel(const LogprobArgs p) {
  __shared__ Sums warp_sums[kMaxWarps], block_sums[kMaxCluster];
  __shared__ typename std::conditional<TOP, Candidates, int>::type candidates;
  __shared__ Key best[TOP ? 32 : 1], block_best[TOP ? kMaxCluster * 32 : 1];
  const cg::cluster_group cluster = cg::this_cluster();
  const int parts = int(cluster.num_blocks()), part = int(cluster.block_rank());
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5, width = blockDim.x;
  const int64_t r = blockIdx.x / parts;
  const Row<T> row(static_cast<const T*>(p.logits) + r * p.row_stride, p.vocab);
  if (parts > 1) cluster.sync();  // no block writes to another's shared memory before that has begun

  const int begin = int(int64_t(row.vectors) * part / parts), end = int(int64_t(row.vectors) * (part + 1) / parts);
  const int stride = width * kUnroll;
  auto load = [&](Block16<T>(&x)[kUnroll], int v0) {
    const uint4* at = row.p + v0 + threadIdx.x;
    if (v0 > 0 && v0 + stride < row.vectors && v0 + stride <= end) {  // nothing of it outside the row or the part
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) x[k].w = at[k * width];
      return;
    }
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      const int v = v0 + int(threadIdx.x) + k * width;
      if (v < end)
        x[k] = row.load(v);
      else
        x[k].fill(-INFINITY);
    }
  };
  Sums a;
  float bar = 0.f, top_most = -INFINITY;
  int renew = 0, group = 0;
  auto add = [&](const Block16<T>(&x)[kUnroll], int v0) {
    float m;
    if constexpr (TOP) {
      float most[kUnroll];
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) most[k] = x[k].most();
      m = most[0];
#pragma unroll
      for (int k = 1; k < kUnroll; ++k) m = max_nan(m, most[k]);
      top_most = max_nan(top_most, m);
      if (v0 >= renew) {  // at the first step, and then when there are eight times as many elements
        if (v0 == begin && threadIdx.x == 0) candidates.vectors = candidates.count = 0;
        bar   = bar_of(top_most, p.top, candidates.group[group]);
        renew = begin + (v0 + stride - begin) * 8 - stride;
        group ^= 1;
      }
      if (!(m < bar)) {
        const int v = v0 + threadIdx.x;
#pragma unroll
        for (int k = 0; k < kUnroll; ++k)
          if (!(most[k] < bar)) set_aside(candidates, x[k].w, v + k * width);
      }
    } else {
      m = most_of<T>(x);
    }
    add_vectors<T, kUnroll>(a, x, m);
  };
  // Two sets of vectors in turn, one on its way while the other is worked on.  Every thread takes the same
  // number of steps: in some of them they meet.
  Block16<T> x[kUnroll], y[kUnroll];
  load(x, begin);
  int v0 = begin;
  do {
    if (v0 + stride < end) load(y, v0 + stride);
    add(x, v0);
    v0 += stride;
    if (v0 >= end) break;
    if (v0 + stride < end) load(x, v0 + stride);
    add(y, v0);
    v0 += stride;
  } while (v0 < end);

  a = join_warp(a);
  if (lane == 0) warp_sums[warp] = a;
  __syncthreads();
  if constexpr (TOP) {
    if (threadIdx.x < 32) best[threadIdx.x] = 0;
    if (collect<T>(candidates, row, p.top, bar))
      rank_keys(candidates.key, candidates.count, p.top, best);
    else
      best_by_insertion<T>(row, begin, end, p.top, candidates.key, best);
    __syncthreads();
  }
  if (warp == 0) {
    a = lane < warps ? warp_sums[lane] : Sums();
    a = join_warp(a);
  }
  if (parts > 1) {
    if (warp == 0) {
      if (lane == 0) *cluster.map_shared_rank(&block_sums[part], 0) = a;
      if constexpr (TOP)
        if (lane < p.top) cluster.map_shared_rank(block_best, 0)[part * p.top + lane] = best[lane];
    }
    cluster.sync();
    if (part != 0) return;
    if constexpr (TOP) {
      rank_keys(block_best, parts * p.top, p.top, best);
      __syncthreads();
    }
    if (warp == 0) {
      a = lane < parts ? block_sums[lane] : Sums();
      a = join_warp(a);
    }
  }
  if (warp != 0) return;
  const float log_s = log2f(a.s);  // a row of -inf: s = 0
  const float lse   = a.s == 0.f ? -INFINITY : fmaf(log_s, kLn2, a.ref);
  // an element's log probability, from the reference: more exact than x - lse
  auto logprob_of = [&](float y) {
    return a.s == 0.f || y == -INFINITY ? (lse != lse ? lse : -INFINITY) : fmaf(-log_s, kLn2, y - a.ref);
  };
  if (lane == 0) {
    if (p.lse) p.lse[r] = lse;
    if (p.entropy) p.entropy[r] = a.s == 0.f ? 0.f : (log_s - a.t / a.s) * kLn2;
    if (p.logprob) {
      const int64_t target = load_index(p.targets, r, p.wide);
      float lp = 0.f;
      if (target >= 0 && target < p.vocab && target != p.ignore_index)
        lp = logprob_of(to_float(row.first()[target]));
      else if (target != p.ignore_index)
        raise_index_error();
      p.logprob[r] = lp;
    }
  }
  if constexpr (TOP) {
    if (lane < p.top) {
      p.top_logprob[r * p.top + lane] = logprob_of(value_of(uint32_t(best[lane] >> 32)));
      p.top_index[r * p.top + lane]   = int64_t(uint32_t(~uint32_t(best[lane])));
    }
  }
}

constexpr int kBackThreads = 256;

// lse comes in 32 bits, and its rounding, half a step of it, is the relative error of every p.  Above this size
// (2^-20 for gradients of 32 bits; 2^-16, where they are rounded to 2^-9 or 2^-12 themselves) the gradient goes by the
// row's largest element and the sum against it instead, for which the row is read once more.  Such a row is one
// block's: the gradient may lie over the logits, and no block may write while another still sums.  (600 x 100003
// fp32, all rows such: 155 us against 81, and 1140 where each of a row's blocks read it; 16 x 128000 fp32 62 against 6.)
template <typename T>
constexpr float kExactLse = sizeof(T) == 4 ? 32.f : 256.f;

// The sums of a row, in every thread; no thread returns before all have read their elements.
template <typename T>
__device__ __noinline__ Sums block_row_sums(const Row<T>& row, Sums* scratch) {
  Sums a;
  for (int v0 = threadIdx.x; v0 < row.vectors; v0 += kBackThreads * kUnroll) {
    Block16<T> x[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      if (v0 + k * kBackThreads < row.vectors)
        x[k] = row.load(v0 + k * kBackThreads);
      else
        x[k].fill(-INFINITY);
    }
    add_vectors<T, kUnroll>(a, x, most_of<T>(x));
  }
  a = join_warp(a);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = a;
  __syncthreads();
  return join_warp((threadIdx.x & 31) < kBackThreads / 32 ? scratch[threadIdx.x & 31] : Sums());
}

// dx_j = dlp ([j = target] - p_j) - dH p_j (log p_j + H), H the entropy.  Six blocks on an SM (40 registers) hide one
// another's loads: 2048 x 100003 bf16 141 us, 153 with five, 170 with the four that 61 registers leave room for.
template <typename T>
__global__ void __launch_bounds__(kBackThreads, 6)
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
  int target = -1;
  if (p.dlogprob) {
    const int64_t t = load_index(p.targets, r, p.wide);
    if (t < 0 || t >= p.vocab || t == p.ignore_index) {
      if (t != p.ignore_index && threadIdx.x == 0) raise_index_error();
      dlp = 0.f;
    } else if (!empty) {
      target = int(t);
    }
  }
  // log2 p = (x - ref) log2(e) - shift
  float ref = empty ? 0.f : lse, shift = 0.f;
  const int64_t block = blockIdx.x % p.blocks_per_row;
  int64_t vectors     = p.vectors_per_block;
  if (!empty && fabsf(lse) > kExactLse<T>) {
    if (block != 0) return;
    const Sums a = block_row_sums<T>(row, scratch);
    ref     = a.ref;
    shift   = log2f(a.s);
    vectors = row.vectors;
  }
  const float c0 = -fmaf(dent, entropy, dlp), c1 = -dent * kLn2;
  // Elements 200 (and up to 32 for the rounding to T) below lse have p = 0; raised to that, neither they
  // nor -inf make log2 p so large that 0 times it is not 0.
  const bool near   = fabsf(ref) < 1e4f && !empty;
  const float floor = ref - 200.f;
  const int begin = int(block * vectors), end = begin + int(vectors) < row.vectors ? begin + int(vectors) : row.vectors;
  for (int v0 = begin + threadIdx.x; v0 < end; v0 += kBackThreads * kUnroll) {
    Block16<T> raw[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k)
      if (v0 + k * kBackThreads < end) raw[k] = row.load(v0 + k * kBackThreads);
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      const int v = v0 + k * kBackThreads;
      if (v >= end) break;
      const int e = row.element(v);
      float g[V];
      if (near && raw[k].most() == raw[k].most()) {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
          const float2 d = fma2(add2(raw[k].raised(i, floor), both(-ref)), both(kLog2E), both(-shift));  // log2 p
          const float2 q = mul2(make_float2(exp2_fast(d.x), exp2_fast(d.y)), fma2(both(c1), d, both(c0)));
          g[2 * i] = q.x, g[2 * i + 1] = q.y;
        }
      } else {
#pragma unroll
        for (int c = 0; c < V; ++c) {
          const float d = max_nan(fmaf(raw[k].element(c) - ref, kLog2E, -shift), kZeroExp);
          g[c]          = exp2_fast(d) * fmaf(c1, d, c0);
        }
      }
      if (unsigned(target - e) < unsigned(V) && target >= 0) {
#pragma unroll
        for (int c = 0; c < V; ++c)
          if (e + c == target) g[c] += dlp;
      }
      if (same_shift && row.whole(v))
        store_vec<T, V>(out + e, g);
      else {
#pragma unroll
        for (int c = 0; c < V; ++c)
          if (e + c >= 0 && e + c < row.vocab) out[e + c] = from_float<T>(g[c]);
      }
    }
  }
}

// ------------------------------------------------------------------ host side
constexpr int kRowCost = 1000;

template <typename F>
cudaError_t for_type(int64_t type, F&& f) {
  if (type == TCU_TYPE_F32) return f(float{});
  return type == TCU_TYPE_F16 ? f(__half{}) : f(__nv_bfloat16{});
}

int check_logits(const void* logits, int64_t type, int64_t rows, int64_t vocab) {
  if (!known_type(type)) return TCU_ERR_UNSUPPORTED;
  if (rows < 0 || vocab < 0 || rows > 0x7fffffff || vocab > (1 << 30)) return TCU_ERR_INVALID_ARG;
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
    // Blocks per row: enough to half fill the SMs, of kRowCost vectors or more each.  (More than that costs: 512
    // rows of 32000 take 12.5 us with one block each, 14.7 us with two; 2048 rows of 100003 80 us and 98 us.)
    int parts = 1;
    while (parts < kMaxCluster && p.rows * parts < 2 * sms && vectors / (2 * parts) >= kRowCost) parts *= 2;
    const int64_t want = ((vectors + parts - 1) / parts + kUnroll - 1) / kUnroll;
    int threads        = 32;  // 2^n warps
    while (threads < kMaxThreads && threads < want) threads *= 2;
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
