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
  for (int s = 0; s < live; ++s) {
    const int64_t row = first + (int64_t)s * rows_max;
    const f32x2 ml = *reinterpret_cast<const f32x2*>(a.part_ml + row * 2);
    const f32x4 o = *reinterpret_cast<const f32x4*>(a.part_out + row * D + d);
    const float now = fmaxf(top, ml[0]);
    const float old_f = rescale(top, now), new_f = rescale(ml[0], now);
    v = v * old_f + o * new_f;
    total = total * old_f + ml[1] * new_f;
    top = now;
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
// A lane is a token (the scores lie token by token), a wave takes every fourth head; the four bytes a lane writes are
// joined with those of the other heads in L2.
__global__ __launch_bounds__(256) void attend_weights_kernel(AttendLaunch a, float* weights, int set) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int chunks = ceil_div(a.Tmax, kWave);
  const int b = blockIdx.x / chunks;
  const int T = min(max(a.seq_lens[b], 0), a.Tmax);
  const int t = blockIdx.x % chunks * kWave + lane;
  if (t >= T) return;
  const RowRange rows = rows_of(a, b);
  const int page = a.block_table ? a.block_table[(int64_t)b * a.block_table_pitch + t / a.block_size] : b;
  if (page < 0 || page >= a.num_blocks) return;
  float* const w = weights + ((int64_t)page * a.block_size + t % a.block_size) * a.Hkv;
  const bool fresh = set || t >= T - rows.n;      // the rows' own tokens: nothing has been added for them yet
  for (int h = wave; h < a.Hkv; h += 4) {
    const float* s = a.scores + ((int64_t)b * a.Hkv + h) * a.max_rows * a.G * a.score_pitch + t;
    float sum = 0.f;
    for (int i = 0; i < rows.n; ++i) {
      const float* lse = a.lse2 + (int64_t)(rows.first + i) * a.Hq + h * a.G;
      for (int g = 0; g < a.G; ++g) {
        const float l = lse[g];
        if (l != -INFINITY) sum += pow2(s[(int64_t)(i * a.G + g) * a.score_pitch] - l);
      }
    }
    w[h] = fresh ? sum : w[h] + sum;
  }
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
  hipLaunchKernelGGL(attend_weights_kernel, dim3((unsigned)((int64_t)ceil_div(a.Tmax, kWave) * a.B)), dim3(256), 0, s, a, weights, set);
  return hipGetLastError();
}

}  // namespace tri
