// What follows attend_kernel (tri_attend_device.h): the splits of a sequence joined, and the weights its tokens received
// added up beside the cache.
#include "tri_attend_device.h"

namespace tri {
namespace {

// out = sum_s 2^(M_s - M) O_s / sum_s 2^(M_s - M) L_s over the splits that hold tokens of the sequence, in the order of the
// splits.  D / 4 lanes a row; reads nsplit * (D + 2) * 4 bytes of a row once, bound by that or, mostly, by its latency.
template <int QT, int D>
__global__ __launch_bounds__(256) void attend_join_kernel(AttendLaunch a) {
  constexpr int kLanes = D / 4, kRows = 256 / kLanes;
  const int rows_max = a.max_rows * a.G;
  const int64_t at = (int64_t)blockIdx.x * kRows + threadIdx.x / kLanes;
  if (at >= (int64_t)a.B * a.Hkv * rows_max) return;
  const int m = (int)(at % rows_max);
  const int h = (int)(at / rows_max % a.Hkv), b = (int)(at / rows_max / a.Hkv);
  const RowRange rows = rows_of(a, b);
  if (m >= rows.n * a.G) return;
  const int T = min(max(a.seq_lens[b], 0), a.Tmax);
  const int live = max(1, ceil_div(tokens_of(a, b, T), a.split_tokens));
  const int64_t first = ((int64_t)b * a.Hkv + h) * a.nsplit * rows_max + m;
  const int d = (threadIdx.x % kLanes) * 4;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  float top = -INFINITY, total = 0.f;
  constexpr int kAtOnce = 8;                 // splits asked for together
  for (int s0 = 0; s0 < live; s0 += kAtOnce) {
    f32x2 ml[kAtOnce];
    f32x4 o[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int64_t row = first + (int64_t)min(s0 + u, live - 1) * rows_max;
      ml[u] = *reinterpret_cast<const f32x2*>(a.part_ml + row * 2);
      o[u] = *reinterpret_cast<const f32x4*>(a.part_out + row * D + d);
    }
    float now = top;
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) now = fmaxf(now, ml[u][0]);
    const float old_f = rescale(top, now);
    v *= old_f;
    total *= old_f;
    top = now;
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const float f = s0 + u < live ? rescale(ml[u][0], now) : 0.f;
      if (f != 0.f) {
        v += o[u] * f;
        total += ml[u][1] * f;
      }
    }
  }
  const int64_t i = rows.first + m / a.G;
  const int hq = h * a.G + m % a.G;
  const float inv = total == 0.f ? 0.f : a.v_scale / total;
  uint16_t* dst = reinterpret_cast<uint16_t*>(a.out) + i * a.out_stride_row + (int64_t)hq * a.out_stride_head + d;
  *reinterpret_cast<uint2*>(dst) = uint2{Half<QT>::pack(v[0] * inv, v[1] * inv), Half<QT>::pack(v[2] * inv, v[3] * inv)};
  if (d == 0) {
    const float l2 = lse_of(top, total);
    if (a.lse) a.lse[i * a.Hq + hq] = l2 * 0.69314718055994530942f;
    if (a.lse2) a.lse2[i * a.Hq + hq] = l2;
  }
}

// weight[token][head] (+)= sum over the rows of the head of 2^(s - lse): every token and head by one thread, rows in order.
// A lane is a token (the scores lie token by token), a wave takes four heads, whose weights it reads and writes as one
// piece (VEC).  Reads a score once, weights once, writes them once.
template <bool VEC>
__global__ __launch_bounds__(256) void attend_weights_kernel(AttendLaunch a, float* weights, int set) {
  const int lane = threadIdx.x % kWave;
  const int quads = ceil_div(a.Hkv, 4), chunks = ceil_div(a.Tmax, kWave);
  int64_t unit = (int64_t)blockIdx.x * (256 / kWave) + threadIdx.x / kWave;
  const int h0 = (int)(unit % quads) * 4;
  unit /= quads;
  const int t = (int)(unit % chunks) * kWave + lane;
  const int64_t b = unit / chunks;
  if (b >= a.B) return;
  const int T = min(max(a.seq_lens[b], 0), a.Tmax);
  if (t >= T) return;
  const RowRange rows = rows_of(a, (int)b);
  const int page = a.block_table ? a.block_table[b * a.block_table_pitch + t / a.block_size] : (int)b;
  if (page < 0 || page >= a.num_blocks) return;
  float* const w = weights + ((int64_t)page * a.block_size + t % a.block_size) * a.Hkv + h0;
  const bool fresh = set || t >= T - rows.n;      // the rows' own tokens: nothing has been added for them yet
  f32x4 had = {0.f, 0.f, 0.f, 0.f};
  if (!fresh) {
    if (VEC) had = *reinterpret_cast<const f32x4*>(w);
    else
      for (int e = 0; e < 4; ++e) had[e] = h0 + e < a.Hkv ? w[e] : 0.f;
  }
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  const int64_t per_head = (int64_t)a.max_rows * a.G * a.score_pitch;
  const float* s = a.scores + (b * a.Hkv + h0) * per_head + t;
  for (int i = 0; i < rows.n; ++i) {
    const float* lse = a.lse2 + (int64_t)(rows.first + i) * a.Hq + h0 * a.G;
#pragma unroll 4
    for (int g = 0; g < a.G; ++g) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int ee = VEC ? e : min(e, a.Hkv - 1 - h0);
        const float l = lse[ee * a.G + g];
        // (a row without tokens, lse -inf: nothing)
        sum[e] += pow2(s[ee * per_head + (int64_t)(i * a.G + g) * a.score_pitch] - (l == -INFINITY ? INFINITY : l));
      }
    }
  }
  sum += had;
  if (VEC) *reinterpret_cast<f32x4*>(w) = sum;
  else
    for (int e = 0; e < 4; ++e)
      if (h0 + e < a.Hkv) w[e] = sum[e];
}

template <int QT>
hipError_t launch_join_typed(const AttendLaunch& a, hipStream_t s) {
  const int64_t rows = (int64_t)a.B * a.Hkv * a.max_rows * a.G;
  auto go = [&](auto kernel, int per) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)ceil_div64(rows, per)), dim3(256), 0, s, a);
    return hipGetLastError();
  };
  if (a.D == 64) return go(attend_join_kernel<QT, 64>, 16);
  if (a.D == 128) return go(attend_join_kernel<QT, 128>, 8);
  return go(attend_join_kernel<QT, 256>, 4);
}

}  // namespace

hipError_t launch_attend(const AttendLaunch& a, hipStream_t s) {
  const bool bf16 = a.q_dtype == TRI_KV_BF16;
  if (a.D == 64) return bf16 ? launch_attend_64_bf16(a, s) : launch_attend_64_fp16(a, s);
  if (a.D == 128) return bf16 ? launch_attend_128_bf16(a, s) : launch_attend_128_fp16(a, s);
  return bf16 ? launch_attend_256_bf16(a, s) : launch_attend_256_fp16(a, s);
}

hipError_t launch_attend_join(const AttendLaunch& a, hipStream_t s) {
  return a.q_dtype == TRI_KV_BF16 ? launch_join_typed<TRI_KV_BF16>(a, s) : launch_join_typed<TRI_KV_FP16>(a, s);
}

hipError_t launch_attend_weights(const AttendLaunch& a, float* weights, int set, hipStream_t s) {
  const int64_t waves = (int64_t)a.B * ceil_div(a.Tmax, kWave) * ceil_div(a.Hkv, 4);
  const dim3 grid((unsigned)ceil_div64(waves, 256 / kWave));
  if (a.Hkv % 4 == 0 && reinterpret_cast<uintptr_t>(weights) % 16 == 0)
    hipLaunchKernelGGL(attend_weights_kernel<true>, grid, dim3(256), 0, s, a, weights, set);
  else
    hipLaunchKernelGGL(attend_weights_kernel<false>, grid, dim3(256), 0, s, a, weights, set);
  return hipGetLastError();
}

}  // namespace tri
