// Gated linear recurrence h_t = f_t h_{t-1} + u_t along time, channel by channel, and its gradient.
//
// The step h -> f h + u is a linear map, and maps compose: (A2, H2) after (A1, H1) is (A2 A1, A2 H1 + H2).  So time is
// cut: a warp takes 64 channels of a sequence, two channels a lane, and 16 rows at a time; the warps of a block (4 or
// 8) and, with few channels, the blocks of a cluster (up to 8) take consecutive rows (a window).  Each warp computes
// the map of its rows, all exchange the maps in shared memory, each joins those before its own to the
// state, and then goes through its rows (still in shared memory, their gates in registers) once more.  All maps are joined
// in the order of time, so the result does not depend on timing.
//
// A warp copies its rows into a ring of its own in shared memory (cp.async, 16 bytes a lane) and waits for
// nothing but its own copies and its neighbours' maps.  What that costs: one warp alone issues an instruction every 3.5
// cycles, so 64 channels of 2048 tokens take one warp 90 us and 8 warps an SM are wanted; the backward pass
// of 1184 columns of 64 channels and more is one warp per column, without maps (113 us for 64 x 512 x 2048; 156 with
// maps, when one warp took 118).
// Measured, bf16, of the copy bandwidth: 64 x 512 x 2048 89 % forward, 90 % backward; 8 x 2048 x 2560 (320 columns, so that
// some SMs have three and some two) 73 % and 67 %; 1 x 65537 x 1024 (16 columns, clusters of 8, one meeting of the
// cluster for 1024 rows) 42 %.
//
// Backwards, with g_t = f_t dh_t passing from row t to row t-1 (dh_t = dy_t + g_{t+1}), the same
// holds with time reversed; h_{t-1} is recomputed from the state before every 16th row, which the
// forward pass leaves behind (one row of floats for 16 rows of elements).
//
// Every element is read from and written to memory once.  Bound by HBM: 3 arrays forward, 5 backward.
#pragma once

#include <cooperative_groups.h>

#include "linear_scan.cuh"

namespace tcu_lm {
namespace {

namespace cg = cooperative_groups;

constexpr int kLoneRows   = 32;  // rows per window of a warp that goes through a sequence alone
constexpr int kJoinedRows = 16;  // and of one that shares it with others: more warps, each with less to do
constexpr int kGroup      = 8;   // rows of the backward pass that are worked on side by side
constexpr int kWidth      = 64;  // channels per warp
constexpr int kMaxWarps   = 8;
constexpr int kMaxCluster = 8;
constexpr int kMaxStages  = 3;   // windows in a warp's ring
// Blocks of 8 warps that the registers of an SM hold.  The gradient of SIGMOID gates spills 400 bytes a thread at 128
// registers, and is faster with half the warps (packed fp16, 37 sequences of 1000 channels: 82 us against 112).
constexpr int kForwardBlocks = 2;
template <int GATE>
constexpr int kBackwardBlocks = GATE == TCU_GATE_SIGMOID ? 1 : 2;

// The rows of the block's sequence: where they begin, how many, and where its states lie.
struct Sequence {
  int64_t a, x, dh, out;  // element offsets of the first row
  int64_t chunk;          // row of `states` of the first rows
  int64_t length;
};

template <bool PACKED>
__device__ __forceinline__ Sequence sequence_of(const ScanArgs& p, int64_t b) {
  Sequence s;
  if (!PACKED) {
    s.length = p.tokens;
    s.a      = b * p.a_batch;
    s.x      = b * p.x_batch;
    s.dh     = b * p.dh_batch;
    s.out    = b * p.tokens * p.dim;
    s.chunk  = b * ((p.tokens + kSpacing - 1) / kSpacing);
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
  s.chunk  = first / kSpacing + b;  // distinct: a sequence has at most length / kSpacing + 1 states
  return s;
}

// Packed sequences of many lengths: blocks of the longest begin first, so that the others fill in beside them; up to
// kRankedBatch sequences.  They are compared in the room of the ring, before it is used (400 bytes more of shared memory
// and two blocks of the gradient no longer fit on an SM).
//
// Where offsets decrease, sequences may share rows, or lie in another order than their numbers and so share states.  Two
// such blocks would write the same memory, so only sequences that are in order may run.
constexpr int kRankedBatch = 96;

// The sequence that `rank` of the others come before; left out if a later one begins before its end.
__device__ __forceinline__ int sequence_of_rank(const ScanArgs& p, int batch, int rank, void* room, int& left_out) {
  __shared__ int found;
  int64_t* offset = static_cast<int64_t*>(room);
  int* length     = reinterpret_cast<int*>(offset + kRankedBatch + 1);
  if (threadIdx.x == 0) left_out = 0;
  for (int i = threadIdx.x; i < batch; i += blockDim.x) {
    const int64_t first = load_index(p.offsets, i, p.wide), end = load_index(p.offsets, i + 1, p.wide), n = end - first;
    offset[i] = first;
    if (i == batch - 1) offset[batch] = end;
    length[i] = n < 0 ? -1 : n > 0x7fffffff ? 0x7fffffff : int(n);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < batch; i += blockDim.x) {
    const int mine = length[i];
    int before = 0;
    for (int j = 0; j < batch; ++j) before += length[j] > mine || (length[j] == mine && j < i);
    if (before == rank) found = i;
  }
  __syncthreads();
  const int b = found;
  for (int i = b + 1 + threadIdx.x; i < batch; i += blockDim.x)
    if (length[i] > 0 && offset[i] >= 0 && offset[i] < offset[b + 1] && offset[i + 1] <= p.tokens) left_out = 1;
  __syncthreads();
  return found;
}

template <bool PACKED>
__device__ __forceinline__ int64_t sequence_at(const ScanArgs& p, int64_t place, void* room, int& left_out) {
  if (!PACKED || p.batch > kRankedBatch) return place;
  return sequence_of_rank(p, int(p.batch), int(place), room, left_out);
}

// A search for the last sequence that begins at or before a row, 32 ways at a time, gives each row one sequence, and a
// later row never one before it, whatever the offsets.  Whether it gives the first and the last row of sequence b to b, for
// a warp: as the steps that lead to b are known, its loads do not wait for each other.
__device__ __forceinline__ bool search_finds(const ScanArgs& p, uint32_t b, int64_t first, int64_t end) {
  const uint32_t lane = threadIdx.x & 31, batch = uint32_t(p.batch);  // (a grid has fewer than 2^31 blocks)
  bool wrong = false;
  for (uint32_t shift = 0; shift < 32 && (batch - 1) >> shift != 0; shift += 5) {
    const uint32_t way = b >> shift & 31;
    const uint64_t i   = uint64_t((b >> shift) - way + lane) << shift;
    if (lane < way || i >= batch) continue;
    const int64_t begin = load_index(p.offsets, int64_t(i), p.wide);
    wrong |= lane == way ? begin < 0 || begin > first : begin >= 0 && begin < end;
  }
  return !__any_sync(0xffffffffu, wrong);
}

// More sequences than kRankedBatch are not all compared: those that the search finds (all, where no offset decreases) are in
// order among themselves, and of the others those run that are in order with all.  By all threads of a block, when its
// first rows are on their way, and through shared memory: values that the compiler does not know to be one for the
// block make the gradient's loop spill.  (bf16, forward + backward, and without the search: 4000 sequences of 10 x 1024 359 + 272
// us, 312 + 249; 300 of 67 x 2048 75 + 106, 72 + 110; 97 of 206 x 2048 61 + 127, 59 + 136.)
__device__ __forceinline__ void leave_out(const ScanArgs& p, int64_t b, int& left_out) {
  if (p.batch > kRankedBatch) {
    if (threadIdx.x < 32) {
      const int64_t first = load_index(p.offsets, b, p.wide), end = load_index(p.offsets, b + 1, p.wide);
      bool wrong = false;
      if (!search_finds(p, uint32_t(b), first, end)) {
#pragma unroll 1
        for (int64_t i = threadIdx.x; i < p.batch; i += 32) {
          const int64_t f = load_index(p.offsets, i, p.wide), e = load_index(p.offsets, i + 1, p.wide);
          wrong |= f >= 0 && f < e && e <= p.tokens && (i < b ? e > first : i > b && f < end);
        }
        wrong = __any_sync(0xffffffffu, wrong);
      }
      if (threadIdx.x == 0) left_out = wrong;
    }
    __syncthreads();
  }
  if (left_out) {
    if (threadIdx.x == 0) raise_index_error();
    copy_wait(0);
  }
}

// ------------------------------------------------------------------ the ring
// Copies kRows rows from `row` on (those that are below `length`) of the warp's channels, the first `left` of them,
// to `to`, kWidth elements a row.  `base`: the block's first channel in the sequence's first row.
template <typename T, int kRows>
__device__ __forceinline__ void copy_rows(T* to, const T* base, int64_t row_stride, int64_t row, int64_t length,
                                          int left, int piece) {
  const int lane = threadIdx.x & 31;
  const int rows = length - row < kRows ? int(length - row) : kRows;  // may be negative
  const T* from  = base + row * row_stride;
  if (piece == 16) {
    constexpr int kLanes = kWidth * int(sizeof(T)) / 16, kAtOnce = 32 / kLanes, kElems = 16 / int(sizeof(T));
    const int r0 = lane / kLanes, c = lane % kLanes * kElems;
    if (c >= left) return;
    from += r0 * row_stride + c;
    to += r0 * kWidth + c;
#pragma unroll
    for (int i = 0; i < kRows; i += kAtOnce, from += kAtOnce * row_stride, to += kAtOnce * kWidth)
      if (i + r0 < rows) copy_async16(to, from);
  } else if (piece == 4) {
    constexpr int kElems = 4 / int(sizeof(T));
#pragma unroll 4
    for (int i = 0; i < kRows; ++i, from += row_stride, to += kWidth)
#pragma unroll
      for (int c = lane * kElems; c < kWidth; c += 32 * kElems)
        if (i < rows && c < left) copy_async4(to + c, from + c);
  } else {
    T x[kRows / 2][2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int i = 0; i < kRows / 2; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k)
          if (half * (kRows / 2) + i < rows && lane + 32 * k < left) x[i][k] = from[i * row_stride + lane + 32 * k];
#pragma unroll
      for (int i = 0; i < kRows / 2; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k)
          if (half * (kRows / 2) + i < rows && lane + 32 * k < left) to[i * kWidth + lane + 32 * k] = x[i][k];
      from += kRows / 2 * row_stride;
      to += kRows / 2 * kWidth;
    }
  }
}

// A lane's two channels of a row in shared memory.
template <typename T>
__device__ __forceinline__ float2 pair_at(const T* row) {
  float y[2];
  to_floats<T, 2>(load_vec<T, 2>(row + (threadIdx.x & 31) * 2), y);
  return make_float2(y[0], y[1]);
}

// Stores a lane's two channels, of which `count` exist.
template <typename T>
__device__ __forceinline__ void store_pair(T* p, float2 x, int count, bool pairs) {
  if (pairs) {
    const float y[2] = {x.x, x.y};
    if (count > 0) store_vec<T, 2>(p, y);
  } else {
    if (count > 0) p[0] = from_float<T>(x.x);
    if (count > 1) p[1] = from_float<T>(x.y);
  }
}
// Stores a lane's two channels of N rows, `rows` of them if that is less.
template <typename T, int N>
__device__ __forceinline__ void store_rows(T* p, const float2 (&x)[N], int64_t dim, int rows, int count, bool pairs) {
  if (rows >= N && pairs) {
    if (count > 0) {
#pragma unroll
      for (int i = 0; i < N; ++i, p += dim) store_pair<T>(p, x[i], 2, true);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i, p += dim)
      if (i < rows) store_pair<T>(p, x[i], count, pairs);
  }
}
__device__ __forceinline__ float2 load_pair(const float* p, int count) {
  return make_float2(count > 0 ? p[0] : 0.f, count > 1 ? p[1] : 0.f);
}

// Rows that no sequence holds: those before the first sequence and behind the last one, which the blocks of these
// two (b) clear.  Where offsets decrease other sequences may lie there: only what is before or behind all counts.  By all
// threads of a block.
struct Rest {
  int64_t before, behind;  // rows 0 ... before-1 and behind ... tokens-1
};
__device__ __forceinline__ Rest rest_of(const ScanArgs& p, int64_t b) {
  Rest rest = {b == 0 ? load_index(p.offsets, 0, p.wide) : 0, b == p.batch - 1 ? load_index(p.offsets, p.batch, p.wide) : p.tokens};
  if (rest.before <= 0 && rest.behind >= p.tokens) return {0, p.tokens};
  __shared__ long long ends[2];
  if (threadIdx.x == 0) ends[0] = p.tokens, ends[1] = 0;
  __syncthreads();
  int64_t low = p.tokens, high = 0;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < p.batch; i += blockDim.x) {
    const int64_t f = load_index(p.offsets, i, p.wide), e = load_index(p.offsets, i + 1, p.wide);
    if (f >= 0 && f < e && e <= p.tokens) low = f < low ? f : low, high = e > high ? e : high;
  }
  atomicMin(&ends[0], low), atomicMax(&ends[1], high);
  __syncthreads();
  low = ends[0], high = ends[1];
  return {rest.before < low ? rest.before : low, rest.behind > high ? rest.behind : high};
}

// Clears them, of the channels of this block.
template <typename T>
__device__ __forceinline__ void clear_rest(const ScanArgs& p, T* out, const Rest& rest, int count, int part, int parts) {
  const int warp = part * (blockDim.x >> 5) + (threadIdx.x >> 5), warps = parts * (blockDim.x >> 5);
  for (int64_t r = warp; r < rest.before; r += warps) store_pair<T>(out + r * p.dim, make_float2(0.f, 0.f), count, p.pairs);
  for (int64_t r = rest.behind + warp; r < p.tokens; r += warps) store_pair<T>(out + r * p.dim, make_float2(0.f, 0.f), count, p.pairs);
}

// ------------------------------------------------------------------ maps
// A product of gates stays finite, so that it does not turn a state of 0 into NaN.  (The sums hold what is not
// a number in the gates: 0 times it is added to them.)
__device__ __forceinline__ float2 finite(float2 a) {
  constexpr float kMost = 3.402823466e38f;
  return make_float2(fminf(fmaxf(a.x, -kMost), kMost), fminf(fmaxf(a.y, -kMost), kMost));
}

struct Map {  // h -> a h + b, of a lane's two channels
  float2 a, b;
};

// What the backward kernel begins with: a block's place.  (The forward kernel has its own variables for it.)
struct Place {
  int64_t b, first, ch;  // sequence, the block's first channel, the lane's
  int left, count;       // channels of the block from `first`; of the lane: above 0, above 1
};
template <bool PACKED>
__device__ __forceinline__ Place place_of(const ScanArgs& p, int64_t group, void* room, int& left_out) {
  Place w;
  w.b     = sequence_at<PACKED>(p, group / p.columns, room, left_out);
  w.first = group % p.columns * kWidth, w.ch = w.first + (threadIdx.x & 31) * 2;
  w.left  = p.dim - w.first < kWidth ? int(p.dim - w.first) : kWidth;
  w.count = w.left - int(threadIdx.x & 31) * 2;
  return w;
}

// The maps of a block's warps and of a cluster's blocks, lanes side by side; two sets, used in turn.
struct Maps {
  float2 warp_a[2][kMaxWarps][32], warp_b[2][kMaxWarps][32];
  float2 block_a[2][kMaxCluster][32], block_b[2][kMaxCluster][32];
};

// Joins the maps of all warps and blocks of a window: `state` goes from before them to behind them
// (REVERSE: time runs backwards, from the last block and warp to the first); returns the state this warp's rows
// start from.
template <bool REVERSE>
__device__ __forceinline__ float2 join_maps(Maps& m, const Map& mine, float2& state, int side,
                                            const cg::cluster_group& cluster, int part, int parts) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int at = REVERSE ? warps - 1 - warp : warp;
  m.warp_a[side][at][lane] = finite(mine.a);
  m.warp_b[side][at][lane] = mine.b;
  __syncthreads();
  float2 before = state;
  if (parts > 1) {
    Map all = {m.warp_a[side][0][lane], m.warp_b[side][0][lane]};
    for (int j = 1; j < warps; ++j) {
      const float2 a = m.warp_a[side][j][lane];
      all.b = fma2(a, all.b, m.warp_b[side][j][lane]);
      all.a = mul2(a, all.a);
    }
    all.a = finite(all.a);
    const int place = REVERSE ? parts - 1 - part : part;
    for (int q = warp; q < parts; q += warps) {
      cluster.map_shared_rank(m.block_a[side][place], q)[lane] = all.a;
      cluster.map_shared_rank(m.block_b[side][place], q)[lane] = all.b;
    }
    cluster.sync();
    for (int q = 0; q < parts; ++q) {
      if (q == place) before = state;
      state = fma2(m.block_a[side][q][lane], state, m.block_b[side][q][lane]);
    }
    for (int j = 0; j < at; ++j) before = fma2(m.warp_a[side][j][lane], before, m.warp_b[side][j][lane]);
  } else {
    for (int j = 0; j < warps; ++j) {
      if (j == at) before = state;
      state = fma2(m.warp_a[side][j][lane], state, m.warp_b[side][j][lane]);
    }
  }
  return before;
}

// ------------------------------------------------------------------ forward
// PACKED: the sequences lie one behind the other, by p.offsets.
template <typename T, typename A, int GATE, bool PACKED>
__global__ void __launch_bounds__(kMaxWarps * 32, kForwardBlocks)
linear_scan_kernel(const ScanArgs p) {
  constexpr int kRows = kJoinedRows;
  __shared__ Maps maps;
  extern __shared__ __align__(16) unsigned char ring[];
  const cg::cluster_group cluster = cg::this_cluster();
  const int parts = int(cluster.num_blocks()), part = int(cluster.block_rank());
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int64_t group = blockIdx.x / parts;
  __shared__ int left_out;
  const int64_t b     = sequence_at<PACKED>(p, group / p.columns, ring, left_out);
  const int64_t first = (group % p.columns) * kWidth, ch = first + lane * 2;
  const int left = p.dim - first < kWidth ? int(p.dim - first) : kWidth;  // channels of the block
  const int count = left - lane * 2;                                      // of the lane: above 0, above 1
  const Sequence s = sequence_of<PACKED>(p, b);
  const A* a = static_cast<const A*>(p.a) + s.a + first;
  const T* x = static_cast<const T*>(p.x) + s.x + first;
  T* out     = static_cast<T*>(p.h) + s.out + ch;

  float2 state = p.h0 ? load_pair(p.h0 + b * p.dim + ch, count) : make_float2(0.f, 0.f);  // before the window
  if (parts > 1) cluster.sync();  // no block writes to another's shared memory before that has begun

  constexpr int kStage = kRows * kWidth * int(sizeof(A) + sizeof(T));
  unsigned char* mine  = ring + warp * p.stages * kStage;
  const int64_t step   = int64_t(parts) * warps * kRows;
  int64_t row          = (int64_t(part) * warps + warp) * kRows;  // of this warp in the window
  auto fetch = [&](int64_t from, int stage) {
    A* to = reinterpret_cast<A*>(mine + stage * kStage);
    if (from < s.length) {
      copy_rows<A, kRows>(to, a, p.a_row, from, s.length, left, p.a_piece);
      copy_rows<T, kRows>(reinterpret_cast<T*>(to + kRows * kWidth), x, p.x_row, from, s.length, left, p.x_piece);
    }
    copy_commit();
  };
  for (int i = 0; i < p.stages; ++i) fetch(row + i * step, i);
  if constexpr (PACKED) leave_out(p, b, left_out);
  int side = 0, stage = 0;
  for (int64_t window = PACKED && left_out ? s.length : 0; window < s.length; window += step, row += step, side ^= 1) {
    copy_wait(p.stages - 1);
    __syncwarp();
    const A* sa = reinterpret_cast<const A*>(mine + stage * kStage);
    const T* sx = reinterpret_cast<const T*>(sa + kRows * kWidth);
    const int rows = s.length - row < kRows ? int(s.length - row) : kRows;  // of this warp; may be negative
    float2 f[kRows], rest[kRows] = {};  // rest: 1 - f, SIGMOID only
    Map map = {make_float2(1.f, 1.f), make_float2(0.f, 0.f)};
    auto input_at = [&](int i) {  // u of row i
      const float2 gx = pair_at<T>(sx + i * kWidth);
      if constexpr (GATE == TCU_GATE_SIGMOID) return mul2(rest[i], gx);
      return gx;
    };
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const float2 ga = pair_at<A>(sa + i * kWidth);
      gate_of<GATE>(ga.x, f[i].x, rest[i].x);
      gate_of<GATE>(ga.y, f[i].y, rest[i].y);
    }
    if (rows == kRows) {
#pragma unroll
      for (int i = 0; i < kRows; ++i) map.b = fma2(f[i], map.b, input_at(i)), map.a = mul2(map.a, f[i]);
    } else {
#pragma unroll
      for (int i = 0; i < kRows; ++i)  // (rows behind the end: the identity)
        if (i < rows) map.b = fma2(f[i], map.b, input_at(i)), map.a = mul2(map.a, f[i]);
    }
    float2 h = join_maps<false>(maps, map, state, side, cluster, part, parts);
    if (p.states && rows > 0) {
      float* st = p.states + (s.chunk + row / kSpacing) * p.dim + ch;
      if (count > 0) st[0] = h.x;
      if (count > 1) st[1] = h.y;
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) f[i] = h = fma2(f[i], h, input_at(i));
    store_rows<T>(out + row * p.dim, f, p.dim, rows, count, p.pairs);
    __syncwarp();  // every lane has read the stage
    fetch(row + p.stages * step, stage);
    stage = stage + 1 == p.stages ? 0 : stage + 1;
  }
  if (PACKED && p.clear_rest && (b == 0 || b == p.batch - 1)) clear_rest<T>(p, static_cast<T*>(p.h) + ch, rest_of(p, b), count, part, parts);
  if (p.last && part == 0 && warp == 0) {
    float* last = p.last + b * p.dim + ch;
    if (count > 0) last[0] = state.x;
    if (count > 1) last[1] = state.y;
  }
}

// ------------------------------------------------------------------ backward
// JOINED: the warps of a block and the blocks of a cluster share a sequence's time; else a block is one warp.
template <typename T, typename A, int GATE, bool JOINED, bool PACKED>
__global__ void __launch_bounds__(JOINED ? kMaxWarps * 32 : 32, JOINED ? kBackwardBlocks<GATE> : 1)
linear_scan_backward_kernel(const ScanArgs p) {
  constexpr int kRows = JOINED ? kJoinedRows : kLoneRows;
  __shared__ typename std::conditional<JOINED, Maps, int>::type maps;
  extern __shared__ __align__(16) unsigned char ring[];
  const cg::cluster_group cluster = cg::this_cluster();
  const int parts = JOINED ? int(cluster.num_blocks()) : 1, part = JOINED ? int(cluster.block_rank()) : 0;
  const int warp = JOINED ? threadIdx.x >> 5 : 0, warps = JOINED ? blockDim.x >> 5 : 1;
  __shared__ int left_out;
  const Place w    = place_of<PACKED>(p, blockIdx.x / parts, ring, left_out);
  const Sequence s = sequence_of<PACKED>(p, w.b);
  const A* a  = static_cast<const A*>(p.a) + s.a + w.first;
  const T* x  = static_cast<const T*>(p.x) + s.x + w.first;
  const T* dy = static_cast<const T*>(p.dh) + s.dh + w.first;
  A* da       = static_cast<A*>(p.da) + s.out + w.ch;
  T* dx       = static_cast<T*>(p.dx) + s.out + w.ch;
  const bool has_dy = p.dh != nullptr;
  // what the rows behind the window pass back
  float2 state = p.dlast ? load_pair(p.dlast + w.b * p.dim + w.ch, w.count) : make_float2(0.f, 0.f);
  if (parts > 1) cluster.sync();  // no block writes to another's shared memory before that has begun

  constexpr int kStage  = kRows * kWidth * int(sizeof(A) + 2 * sizeof(T));
  unsigned char* mine   = ring + warp * p.stages * kStage;
  const int64_t step    = int64_t(parts) * warps * kRows;
  const int64_t windows = (s.length + step - 1) / step;
  int64_t row           = (windows - 1) * step + (int64_t(part) * warps + warp) * kRows;
  auto fetch = [&](int64_t from, int stage) {
    A* to = reinterpret_cast<A*>(mine + stage * kStage);
    T* tx = reinterpret_cast<T*>(to + kRows * kWidth);
    if (from >= 0 && from < s.length) {
      copy_rows<A, kRows>(to, a, p.a_row, from, s.length, w.left, p.a_piece);
      copy_rows<T, kRows>(tx, x, p.x_row, from, s.length, w.left, p.x_piece);
      if (has_dy) copy_rows<T, kRows>(tx + kRows * kWidth, dy, p.dh_row, from, s.length, w.left, p.dh_piece);
    }
    copy_commit();
  };
  auto state_at = [&](int64_t from) {  // the state before row `from` of the sequence
    return from >= 0 && from < s.length ? load_pair(p.states + (s.chunk + from / kSpacing) * p.dim + w.ch, w.count)
                                        : make_float2(0.f, 0.f);
  };
  for (int i = 0; i < p.stages; ++i) fetch(row - i * step, i);
  if constexpr (PACKED) leave_out(p, w.b, left_out);
  int stage = 0;
  constexpr int kParts = kRows / kSpacing;
  float2 next_h[kParts];
#pragma unroll
  for (int k = 0; k < kParts; ++k) next_h[k] = state_at(row + k * kSpacing);
  for (uint32_t n = PACKED && left_out ? uint32_t(windows) : 0; n < windows; ++n, row -= step) {
    const int rows = s.length - row < kRows ? int(s.length - row) : kRows;
    float2 h[kParts];
#pragma unroll
    for (int k = 0; k < kParts; ++k) h[k] = next_h[k], next_h[k] = state_at(row - step + k * kSpacing);
    copy_wait(p.stages - 1);
    __syncwarp();
    const A* sa = reinterpret_cast<const A*>(mine + stage * kStage);
    const T* sx = reinterpret_cast<const T*>(sa + kRows * kWidth);
    const T* sd = sx + kRows * kWidth;
    // gates of rows i ... i + kGroup - 1
    auto gates_at = [&](int i, float2 (&f)[kGroup], float2 (&rest)[kGroup]) {
#pragma unroll
      for (int k = 0; k < kGroup; ++k) f[k] = pair_at<A>(sa + (i + k) * kWidth);
#pragma unroll
      for (int k = 0; k < kGroup; ++k) gate_of<GATE>(f[k], f[k], rest[k]);
    };
    // dy of rows i ... i + kGroup - 1; the rows from `rows` on pass on what they get: f 1 and dy 0
    auto gradients_at = [&](int i, float2 (&d)[kGroup], float2 (&f)[kGroup]) {
#pragma unroll
      for (int k = 0; k < kGroup; ++k) d[k] = has_dy ? pair_at<T>(sd + (i + k) * kWidth) : make_float2(0.f, 0.f);
      if (i + kGroup > rows) {
#pragma unroll
        for (int k = 0; k < kGroup; ++k)
          if (i + k >= rows) f[k] = make_float2(1.f, 1.f), d[k] = make_float2(0.f, 0.f);
      }
    };
    float2 g = state;
    if constexpr (JOINED) {
      // g passes back f_0 (dy_0 + f_1 (dy_1 + ...)), the sum of dy_i times the product of f_0 ... f_i
      Map back = {make_float2(1.f, 1.f), make_float2(0.f, 0.f)};
#pragma unroll 1
      for (int i = 0; i < kRows; i += kGroup) {
        float2 f[kGroup], rest[kGroup], d[kGroup];
        gates_at(i, f, rest);
        gradients_at(i, d, f);
#pragma unroll
        for (int k = 0; k < kGroup; ++k) back.a = mul2(back.a, f[k]), back.b = fma2(back.a, d[k], back.b);
      }
      g = join_maps<true>(maps, back, state, n & 1, cluster, part, parts);
    }
    float2 before[kRows];
#pragma unroll
    for (int n0 = 0; n0 < kParts; ++n0) {
#pragma unroll
      for (int i = n0 * kSpacing; i < (n0 + 1) * kSpacing; i += kGroup) {
        float2 f[kGroup], rest[kGroup], u[kGroup];
        gates_at(i, f, rest);
#pragma unroll
        for (int k = 0; k < kGroup; ++k) {
          u[k] = pair_at<T>(sx + (i + k) * kWidth);
          if constexpr (GATE == TCU_GATE_SIGMOID) u[k] = mul2(rest[k], u[k]);
        }
#pragma unroll
        for (int k = 0; k < kGroup; ++k) before[i + k] = h[n0], h[n0] = fma2(f[k], h[n0], u[k]);
      }
    }
#pragma unroll
    for (int i = kRows - kGroup; i >= 0; i -= kGroup) {
      if (i >= rows) continue;
      float2 f[kGroup], rest[kGroup], d[kGroup], ga[kGroup];
      gates_at(i, f, rest);
      gradients_at(i, d, f);
#pragma unroll
      for (int k = kGroup - 1; k >= 0; --k) {
        d[k] = add2(d[k], g);  // dh
        g    = mul2(f[k], d[k]);
        if constexpr (GATE == TCU_GATE_SIGMOID) {
          const float2 v = pair_at<T>(sx + (i + k) * kWidth);
          ga[k] = mul2(mul2(d[k], add2(before[i + k], make_float2(-v.x, -v.y))), mul2(f[k], rest[k]));
          d[k]  = mul2(d[k], rest[k]);
        } else {
          ga[k] = mul2(GATE == TCU_GATE_LOG ? g : d[k], before[i + k]);
        }
      }
      store_rows<A>(da + (row + i) * p.dim, ga, p.dim, rows - i, w.count, p.pairs);
      store_rows<T>(dx + (row + i) * p.dim, d, p.dim, rows - i, w.count, p.pairs);
    }
    if constexpr (!JOINED) state = g;
    __syncwarp();
    fetch(row - p.stages * step, stage);
    stage = stage + 1 == p.stages ? 0 : stage + 1;
  }
  if (PACKED && p.clear_rest && (w.b == 0 || w.b == p.batch - 1)) {
    const Rest rest = rest_of(p, w.b);
    clear_rest<A>(p, static_cast<A*>(p.da) + w.ch, rest, w.count, part, parts);
    clear_rest<T>(p, static_cast<T*>(p.dx) + w.ch, rest, w.count, part, parts);
  }
  if (p.dh0 && part == 0 && warp == 0) {
    float* dh0 = p.dh0 + w.b * p.dim + w.ch;
    if (w.count > 0) dh0[0] = state.x;
    if (w.count > 1) dh0[1] = state.y;
  }
}

constexpr int kSharedPerSm = 224 << 10;

// With eight columns of 64 channels for every SM a warp goes through a sequence alone.  With fewer, time is
// cut: blocks of 8 warps (fewer where their rings would not leave room for a second block on the SM, or all blocks would
// not fit on the SMs at once), and with fewer columns than SMs clusters of up to 8 such blocks, as
// long as the sequences have the rows for them.  (Clusters of 8 blocks that fill an SM each do not all find 8 free SMs
// side by side: 15 of 16 did.)  A ring takes what shared memory is left, two windows at least.
constexpr int kLoneColumns = 8;

template <void (*Lone)(const ScanArgs), void (*Joined)(const ScanArgs)>
cudaError_t launch_scan(ScanArgs args, int row_bytes, int blocks, int sms, cudaStream_t st) {
  constexpr int kStatic = int(sizeof(Maps));  // of a joined block
  static bool configured[kMaxDevices];
  const int dev = current_device();
  if (dev < 0) return cudaErrorInvalidDevice;
  if (!configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(Lone, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedPerSm - kStatic);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(Joined, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedPerSm - kStatic);
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  args.columns         = int((args.dim + kWidth - 1) / kWidth);
  const int64_t groups = args.batch * args.columns;
  const int64_t each   = args.offsets ? 2 * args.tokens / args.batch : args.tokens;  // (packed: a guess)
  int warps = 1, parts = 1;
  auto bytes_of = [&](int stages) {
    return stages * warps * row_bytes * (warps > 1 ? kJoinedRows : kLoneRows);
  };
  auto fit = [&] {  // blocks on an SM
    const int by_memory = kSharedPerSm / (bytes_of(2) + kStatic + 1024), by_registers = blocks * kMaxWarps / warps;
    return by_memory < by_registers ? by_memory : by_registers;
  };
  if (Lone == Joined || (groups < int64_t(kLoneColumns) * sms && each > kLoneRows)) {
    warps = kMaxWarps;
    // (packed sequences need not all fit at once: few are long)
    const bool at_once = !args.offsets || args.batch > kRankedBatch;
    while (warps > 2 && (2 * (bytes_of(2) + 17 * 1024) > (226 << 10) ||
                         (warps > 4 && at_once && groups > int64_t(sms) * fit())))
      warps /= 2;
    while (parts < kMaxCluster && groups * parts < sms && each > int64_t(parts) * warps * kJoinedRows) parts *= 2;
  }
  if (groups * parts > int64_t(0x7fffffff)) return cudaErrorInvalidConfiguration;
  int64_t per_sm = (groups * parts + sms - 1) / sms;  // blocks that there are for an SM
  int stages = 2;
  while (parts == 1 && stages < kMaxStages && per_sm * (bytes_of(stages + 1) + (warps > 1 ? kStatic : 0) + 1024) <= kSharedPerSm) ++stages;
  args.stages            = stages;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim            = dim3(unsigned(groups * parts));
  cfg.blockDim           = dim3(warps * 32);
  cfg.dynamicSmemBytes   = bytes_of(stages);
  cfg.stream             = st;
  cudaLaunchAttribute attr[1];
  attr[0].id                 = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x   = unsigned(parts);
  attr[0].val.clusterDim.y   = 1;
  attr[0].val.clusterDim.z   = 1;
  cfg.attrs    = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, warps > 1 ? Joined : Lone, args);
}

}  // namespace

template <typename T>
cudaError_t launch_linear_scan(const ScanArgs& args, int64_t a_type, int64_t gate, int sms, cudaStream_t st) {
  return for_gates<T>(a_type, gate, [&](auto a, auto g) {
    using A = decltype(a);
    constexpr int G = decltype(g)::value;
    auto go = [&](auto packed) {
      constexpr auto kernel = linear_scan_kernel<T, A, G, decltype(packed)::value>;
      return launch_scan<kernel, kernel>(args, kWidth * int(sizeof(A) + sizeof(T)), kForwardBlocks, sms, st);
    };
    return args.offsets ? go(std::true_type{}) : go(std::false_type{});
  });
}

template <typename T>
cudaError_t launch_linear_scan_backward(const ScanArgs& args, int64_t a_type, int64_t gate, int sms, cudaStream_t st) {
  return for_gates<T>(a_type, gate, [&](auto a, auto g) {
    using A = decltype(a);
    constexpr int G = decltype(g)::value;
    auto go = [&](auto packed) {
      constexpr bool P = decltype(packed)::value;
      return launch_scan<linear_scan_backward_kernel<T, A, G, false, P>, linear_scan_backward_kernel<T, A, G, true, P>>(
          args, kWidth * int(sizeof(A) + 2 * sizeof(T)), kBackwardBlocks<G>, sms, st);
    };
    return args.offsets ? go(std::true_type{}) : go(std::false_type{});
  });
}

}  // namespace tcu_lm
