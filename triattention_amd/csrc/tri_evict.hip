// Eviction by accumulated attention weight: the rows the top-k runs on, and the move of the weights with their tokens.
// Weights lie beside the cache, [layer][physical block][token in block][KV head] fp32, as the scales of an fp8 cache do.
#include <algorithm>

#include "tri_common.h"

namespace tri {
namespace {

// fin[row][t] = the weights of token t reduced over layers (and, shared, over heads), +inf where the token is guarded, -inf
// behind the sequence; keep[row][j] = -1 behind the sequence's budget.  A thread has one token and kHeads heads (as they
// lie, one piece of 16 bytes where it can be), lanes are tokens as the rows lie; the mean is summed in 64 bits and rounded once.
// Bound by reading the weights: 36 layers of 8 x 8192 tokens of 8 heads, a row per layer, 75 MB read and as much written in
// 36 us (4.2 TB/s); one request of 2176 tokens 10 us, 36 layers' reads one behind the other.
__device__ __forceinline__ float larger(float a, float b) { return __builtin_isnan(a) || a > b ? a : b; }

constexpr int kHeads = 4;
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <bool VEC>
__device__ __forceinline__ f32x4 load_heads(const float* w, int left) {
  if (VEC) return *reinterpret_cast<const f32x4*>(w);
  return f32x4{w[0], w[left > 1 ? 1 : 0], w[left > 2 ? 2 : 0], w[left > 3 ? 3 : 0]};
}

template <bool VEC>
__global__ __launch_bounds__(256) void weight_rows_kernel(EvictLaunch a, int width) {
  const int per_layer = a.layer_reduce < 0;
  const int chunks = ceil_div(width, 256), quads = a.shared ? 1 : ceil_div(a.Hkv, kHeads);
  int entry = blockIdx.x;
  const int t = entry % chunks * 256 + threadIdx.x;
  entry /= chunks;
  const int h0 = entry % quads * kHeads;
  entry /= quads;
  if (t >= width) return;
  const int b = entry / (per_layer ? a.L : 1), only = per_layer ? entry % a.L : 0;
  const int T = min(max(a.seq_lens[b], 0), a.Tmax);
  const int heads = a.shared ? 1 : a.Hkv, mine = a.shared ? 1 : min(kHeads, a.Hkv - h0);
  const int64_t row = (int64_t)entry * heads + h0;
  if (t < a.max_budget && t >= min(a.budgets[b], T))
    for (int e = 0; e < mine; ++e) a.keep[(row + e) * a.max_budget + t] = -1;
  if (t >= a.Tmax) return;
  float* const out = a.fin + row * a.Tmax + t;
  const int page = t >= T ? -1 : a.block_table ? a.block_table[(int64_t)b * a.block_table_pitch + t / a.block_size] : b;
  f32x4 v = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  if (t < T && (t >= T - a.window_size || (a.protect_prefill && a.prefill_lens && t < a.prefill_lens[b]))) {
    v = f32x4{INFINITY, INFINITY, INFINITY, INFINITY};
  } else if (page >= 0 && page < a.num_blocks) {
    const float* w = a.weights + ((int64_t)page * a.block_size + t % a.block_size) * a.Hkv;
    const int last = a.shared ? a.Hkv : h0 + 1;
    for (int h = h0; h < last; h += kHeads) {
      const int left = a.Hkv - h;
      f32x4 x;
      if (per_layer) {
        x = load_heads<VEC>(w + only * a.weights_stride_layer + h, left);
      } else if (a.layer_reduce == TRI_REDUCE_MAX) {
        x = load_heads<VEC>(w + h, left);
#pragma unroll 8
        for (int l = 1; l < a.L; ++l) {
          const f32x4 y = load_heads<VEC>(w + l * a.weights_stride_layer + h, left);
#pragma unroll
          for (int e = 0; e < kHeads; ++e) x[e] = larger(x[e], y[e]);
        }
      } else {
        double sum[kHeads] = {};
#pragma unroll 8
        for (int l = 0; l < a.L; ++l) {
          const f32x4 y = load_heads<VEC>(w + l * a.weights_stride_layer + h, left);
#pragma unroll
          for (int e = 0; e < kHeads; ++e) sum[e] += (double)y[e];
        }
#pragma unroll
        for (int e = 0; e < kHeads; ++e) x[e] = (float)(sum[e] / a.L);
      }
      if (!a.shared) v = x;
      else
        for (int e = 0; e < min(kHeads, left); ++e) v[0] = larger(x[e], v[0]);
    }
  }
  // (one NaN for all: the top-k orders by the bits, where those of negative sign lie below every number)
#pragma unroll
  for (int e = 0; e < kHeads; ++e)
    if (e < mine) out[(int64_t)e * a.Tmax] = __builtin_isnan(v[e]) ? __builtin_nanf("") : v[e];
}

// One workgroup per (sequence, layer) moves the weights of all heads as their rows move: slot j of head h receives the
// weight of token keep[h][j].  Lists ascend (keep[j] >= j), so a tile whose reads all precede its writes never reads what
// an earlier tile wrote.  2048 of 2176 tokens, 8 heads, 36 layers: 16 us, two tiles' chain of list, table and weight; the move of K
// and V before it takes 119.
constexpr int kMoveThreads = 1024, kMoveEach = 8;
__global__ __launch_bounds__(kMoveThreads) void move_weights_kernel(EvictLaunch a) {
  const int l = blockIdx.x % a.L, b = blockIdx.x / a.L;
  const int T = min(max(a.seq_lens[b], 0), a.Tmax);
  const int k = min(min(a.budgets[b], T), a.max_budget);
  if (k <= 0 || k >= T) return;                  // (a list of everything moves nothing)
  const int rows = a.shared ? 1 : a.Hkv;
  const int32_t* keep = a.keep + (int64_t)(a.layer_reduce < 0 ? b * a.L + l : b) * rows * a.max_budget;
  const int32_t* table = a.block_table + (int64_t)b * a.block_table_pitch;
  float* const w = a.weights + l * a.weights_stride_layer;
  const int64_t pairs = (int64_t)k * a.Hkv;
  for (int64_t p0 = 0; p0 < pairs; p0 += kMoveThreads * kMoveEach) {
    // Every level of the dependent lookups (list, table, weight) is issued for all of a thread's pairs before the next one.
    int src[kMoveEach];
    int64_t from[kMoveEach], to[kMoveEach];
    float v[kMoveEach];
#pragma unroll
    for (int i = 0; i < kMoveEach; ++i) {
      const int64_t p = min(p0 + i * kMoveThreads + threadIdx.x, pairs - 1);
      const int j = (int)(p / a.Hkv), h = (int)(p % a.Hkv);
      src[i] = keep[(int64_t)(a.shared ? 0 : h) * a.max_budget + j];
      to[i] = ((int64_t)table[j / a.block_size] * a.block_size + j % a.block_size) * a.Hkv + h;
    }
#pragma unroll
    for (int i = 0; i < kMoveEach; ++i) {
      const int64_t p = min(p0 + i * kMoveThreads + threadIdx.x, pairs - 1);
      from[i] = ((int64_t)table[src[i] / a.block_size] * a.block_size + src[i] % a.block_size) * a.Hkv + p % a.Hkv;
    }
#pragma unroll
    for (int i = 0; i < kMoveEach; ++i) v[i] = w[from[i]];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kMoveEach; ++i)
      if (p0 + i * kMoveThreads + threadIdx.x < pairs) w[to[i]] = v[i];
  }
}

}  // namespace

hipError_t launch_weight_rows(const EvictLaunch& a, hipStream_t s) {
  const int width = std::max(a.Tmax, a.max_budget);
  const int64_t quads = a.shared ? 1 : ceil_div(a.Hkv, kHeads);
  const dim3 grid((unsigned)(ceil_div(width, 256) * quads * a.B * (a.layer_reduce < 0 ? a.L : 1)));
  if (a.Hkv % kHeads == 0 && a.weights_stride_layer % 4 == 0 && reinterpret_cast<uintptr_t>(a.weights) % 16 == 0)
    hipLaunchKernelGGL(weight_rows_kernel<true>, grid, dim3(256), 0, s, a, width);
  else
    hipLaunchKernelGGL(weight_rows_kernel<false>, grid, dim3(256), 0, s, a, width);
  return hipGetLastError();
}

hipError_t launch_move_weights(const EvictLaunch& a, hipStream_t s) {
  hipLaunchKernelGGL(move_weights_kernel, dim3(a.B * a.L), dim3(kMoveThreads), 0, s, a);
  return hipGetLastError();
}

}  // namespace tri
