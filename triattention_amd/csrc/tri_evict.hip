// Eviction by accumulated attention weight: the rows the top-k runs on, and the move of the weights with their tokens.
// Weights lie beside the cache, [layer][physical block][token in block][KV head] fp32, as the scales of an fp8 cache do.
#include <algorithm>

#include "tri_common.h"

namespace tri {
namespace {

// fin[row][t] = the weights of token t reduced over layers (and, shared, over heads), +inf where the token is guarded, -inf
// behind the sequence; keep[row][j] = -1 behind the sequence's budget.  One thread per (token, head), heads fastest as
// they lie; the mean is summed in 64 bits and rounded once.
__global__ __launch_bounds__(256) void weight_rows_kernel(EvictLaunch a, int width) {
  const int heads = a.shared ? 1 : a.Hkv;
  const int chunks = (int)ceil_div64((int64_t)width * heads, 256), entry = blockIdx.x / chunks;
  const int64_t at = (int64_t)(blockIdx.x % chunks) * 256 + threadIdx.x;
  const int t = (int)(at / heads), h = (int)(at % heads);
  if (t >= width) return;
  const int per_layer = a.layer_reduce < 0;
  const int b = entry / (per_layer ? a.L : 1), only = per_layer ? entry % a.L : 0;
  const int T = min(max(a.seq_lens[b], 0), a.Tmax);
  const int64_t row = (int64_t)entry * heads + h;
  if (t < a.max_budget && t >= min(a.budgets[b], T)) a.keep[row * a.max_budget + t] = -1;
  if (t >= a.Tmax) return;
  float* const out = a.fin + row * a.Tmax + t;
  if (t >= T) {
    *out = -INFINITY;
    return;
  }
  if (t >= T - a.window_size || (a.protect_prefill && a.prefill_lens && t < a.prefill_lens[b])) {
    *out = INFINITY;
    return;
  }
  const int page = a.block_table ? a.block_table[(int64_t)b * a.block_table_pitch + t / a.block_size] : b;
  if (page < 0 || page >= a.num_blocks) {
    *out = -INFINITY;
    return;
  }
  const float* w = a.weights + ((int64_t)page * a.block_size + t % a.block_size) * a.Hkv;
  float best = -INFINITY;
  for (int hh = a.shared ? 0 : h; hh < (a.shared ? a.Hkv : h + 1); ++hh) {
    float v;
    if (per_layer) {
      v = w[only * a.weights_stride_layer + hh];
    } else if (a.layer_reduce == TRI_REDUCE_MAX) {
      v = -INFINITY;
#pragma unroll 8
      for (int l = 0; l < a.L; ++l) {
        const float x = w[l * a.weights_stride_layer + hh];
        v = __builtin_isnan(v) || v > x ? v : x;
      }
    } else {
      double sum = 0.;
#pragma unroll 8
      for (int l = 0; l < a.L; ++l) sum += (double)w[l * a.weights_stride_layer + hh];
      v = (float)(sum / a.L);
    }
    best = hh == 0 || !a.shared ? v : (__builtin_isnan(best) || best > v ? best : v);
  }
  *out = best;
}

// One workgroup per (sequence, layer) moves the weights of all heads as their rows move: slot j of head h receives the
// weight of token keep[h][j].  Lists ascend (keep[j] >= j), so a tile whose reads all precede its writes never reads what
// an earlier tile wrote.
constexpr int kMoveThreads = 1024, kMoveEach = 16;
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
    float v[kMoveEach];
#pragma unroll
    for (int i = 0; i < kMoveEach; ++i) {
      const int64_t p = p0 + i * kMoveThreads + threadIdx.x;
      if (p >= pairs) continue;
      const int j = (int)(p / a.Hkv), h = (int)(p % a.Hkv);
      const int src = keep[(int64_t)(a.shared ? 0 : h) * a.max_budget + j];
      v[i] = w[((int64_t)table[src / a.block_size] * a.block_size + src % a.block_size) * a.Hkv + h];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kMoveEach; ++i) {
      const int64_t p = p0 + i * kMoveThreads + threadIdx.x;
      if (p >= pairs) continue;
      const int j = (int)(p / a.Hkv), h = (int)(p % a.Hkv);
      w[((int64_t)table[j / a.block_size] * a.block_size + j % a.block_size) * a.Hkv + h] = v[i];
    }
  }
}

}  // namespace

hipError_t launch_weight_rows(const EvictLaunch& a, hipStream_t s) {
  const int width = std::max(a.Tmax, a.max_budget);
  const dim3 grid((unsigned)(ceil_div64((int64_t)width * (a.shared ? 1 : a.Hkv), 256) * a.B * (a.layer_reduce < 0 ? a.L : 1)));
  hipLaunchKernelGGL(weight_rows_kernel, grid, dim3(256), 0, s, a, width);
  return hipGetLastError();
}

hipError_t launch_move_weights(const EvictLaunch& a, hipStream_t s) {
  hipLaunchKernelGGL(move_weights_kernel, dim3(a.B * a.L), dim3(kMoveThreads), 0, s, a);
  return hipGetLastError();
}

}  // namespace tri
