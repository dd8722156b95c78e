// What follows the attention itself (tri_attend_device.h): the splits of a sequence joined, and the weights its tokens received
// added up beside the cache.
#include <algorithm>

#include "tri_attend_device.h"

namespace tri {
namespace {

constexpr int kThreads = 256;
constexpr int kWideSplits = 8;      // more splits than that: several lanes side by side over them, where rows are few
constexpr int kWideRows = 1024;

struct Joined {
  f32x4 v;
  float top, total;
};
__device__ __forceinline__ void join_two(Joined& a, const Joined& b) {
  const float top = fmaxf(a.top, b.top), fa = rescale(a.top, top), fb = rescale(b.top, top);
  // (0 * NaN on purpose: a value that is no number shows, however the sequence is cut; a part without tokens holds zeros)
  a.v = a.v * fa + b.v * fb;
  a.total = a.total * fa + b.total * fb;
  a.top = top;
}

// out = sum_s 2^(M_s - M) O_s / sum_s 2^(M_s - M) L_s over the splits that hold tokens of the sequence, in a fixed order.
// D / 4 lanes take a row, PARTS of them side by side every PARTS-th split.  Reads nsplit * (D + 2) * 4 bytes of a row
// once; bound by their latency.
template <int QT, int D, int PARTS>
__device__ __forceinline__ void join_rows(const AttendLaunch& a, int64_t group) {
  constexpr int kLanes = D / 4, kRows = kThreads / kLanes / PARTS;
  constexpr int kAtOnce = PARTS > 1 ? 4 : 8;         // splits asked for together
  __shared__ Joined s_part[PARTS > 1 ? PARTS : 1][kRows][kLanes];
  const int rows_max = a.max_rows * a.G;
  const int lane = threadIdx.x % kLanes, part = threadIdx.x / kLanes % PARTS, mine = threadIdx.x / kLanes / PARTS;
  const int64_t at = group * kRows + mine;
  const bool in = at < (int64_t)a.B * a.Hkv * rows_max;
  const int m = in ? (int)(at % rows_max) : 0;
  const int h = in ? (int)(at / rows_max % a.Hkv) : 0, b = in ? (int)(at / rows_max / a.Hkv) : 0;
  const int T = min(max(a.seq_lens[b], 0), a.Tmax);
  const RowRange rows = rows_of(a, b, T);
  const bool live_row = in && m < rows.n * a.G;
  const int live = max(1, ceil_div(tokens_of(a, b, T), a.split_tokens));
  const int64_t first = ((int64_t)b * a.Hkv + h) * a.nsplit * rows_max + m;
  const int d = lane * 4;
  Joined j{{0.f, 0.f, 0.f, 0.f}, -INFINITY, 0.f};
  if (live_row) {
    for (int s0 = part; s0 < live; s0 += kAtOnce * PARTS) {
      f32x2 ml[kAtOnce];
      f32x4 o[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const int64_t row = first + (int64_t)min(s0 + u * PARTS, live - 1) * rows_max;
        ml[u] = *reinterpret_cast<const f32x2*>(a.part_ml + row * 2);
        o[u] = *reinterpret_cast<const f32x4*>(a.part_out + row * D + d);
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u)
        if (s0 + u * PARTS < live) join_two(j, Joined{o[u], ml[u][0], ml[u][1]});
    }
  }
  if (PARTS > 1) {
    s_part[part][mine][lane] = j;
    __syncthreads();
    if (part != 0) return;
#pragma unroll 4
    for (int p = 1; p < PARTS; ++p) join_two(j, s_part[p][mine][lane]);
  }
  if (!live_row) return;
  const int64_t i = rows.first + m / a.G;
  const int hq = h * a.G + m % a.G;
  const float inv = j.total == 0.f ? 0.f : a.v_scale / j.total;
  uint16_t* dst = reinterpret_cast<uint16_t*>(a.out) + i * a.out_stride_row + (int64_t)hq * a.out_stride_head + d;
  *reinterpret_cast<uint2*>(dst) = uint2{Half<QT>::pack(j.v[0] * inv, j.v[1] * inv), Half<QT>::pack(j.v[2] * inv, j.v[3] * inv)};
  if (d == 0) {
    const float l2 = lse_of(j.top, j.total);
    if (a.lse) a.lse[i * a.Hq + hq] = l2 * 0.69314718055994530942f;
    if (a.lse2) a.lse2[i * a.Hq + hq] = l2;
  }
}

// weight[token][head] (+)= sum over the rows of the head of 2^(s - lse): every token and head by one thread, rows in order.
// A lane is a token (the scores lie token by token), a wave takes four heads, whose weights it reads and writes as one
// piece (VEC), and sixteen rows at a time: four lanes find the lse of a row, from its splits where the sequence is
// cut.  Where the four heads have more rows than sixteen, the workgroup's waves take four pieces of one sequence's tokens and find
// the lse of 64 rows TOGETHER (a wave would read as much for them as of scores: 24 ragged sequences of 64 query heads 22 ->
// 17 us; with sixteen rows three waves would wait for one, 18 -> 21).  Reads a score once, weights once, writes them once.
template <bool VEC, bool TOGETHER>
__device__ __forceinline__ void add_weights(const AttendLaunch& a, float* weights, int set, int64_t group) {
  constexpr int kWaves = kThreads / kWave, kSpan = TOGETHER ? kThreads : kWave, kRows = kSpan / 4;
  __shared__ float s_lse[kThreads / 4];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int of_unit = TOGETHER ? 0 : wave * kRows;          // the unit's part of s_lse
  const int quads = ceil_div(a.Hkv, 4), spans = ceil_div(a.Tmax, kSpan);
  int64_t unit = TOGETHER ? group : group * kWaves + wave;
  const int h0 = (int)(unit % quads) * 4;
  unit /= quads;
  const int t0 = (int)(unit % spans) * kSpan;
  const int64_t b = unit / spans;
  if (b >= a.B) return;
  const int T = min(max(a.seq_lens[b], 0), a.Tmax);
  if (t0 >= T) return;
  const int mine = t0 + (TOGETHER ? (int)threadIdx.x : lane);
  const RowRange rows = rows_of(a, (int)b, T);
  const int t = min(mine, T - 1);
  const int page = a.block_table ? a.block_table[b * a.block_table_pitch + t / a.block_size] : (int)b;
  const bool ok = mine < T && page >= 0 && page < a.num_blocks;
  float* const w = weights + (ok ? ((int64_t)page * a.block_size + t % a.block_size) * a.Hkv + h0 : 0);
  const bool fresh = set || t >= T - rows.fresh;  // new tokens: nothing has been added for them yet
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  if (ok && !fresh) {
    if (VEC) sum = *reinterpret_cast<const f32x4*>(w);
    else
      for (int e = 0; e < 4; ++e) sum[e] = h0 + e < a.Hkv ? w[e] : 0.f;
  }
  f32x4 more = {0.f, 0.f, 0.f, 0.f};
  const int per_head = rows.n * a.G, heads = min(4, a.Hkv - h0), rows_max = a.max_rows * a.G;
  const int live = max(1, ceil_div(T, a.split_tokens));
  const int all = heads * per_head;
  for (int r0 = 0; r0 < all; r0 += kRows) {
    const int r = min(r0 + (TOGETHER ? wave * 16 : 0) + (lane & 15), all - 1), h = h0 + r / per_head, m = r % per_head;
    float l;
    if (a.nsplit > 1) {
      const float* ml = a.part_ml + (((b * a.Hkv + h) * a.nsplit) * rows_max + m) * 2;
      float top = -INFINITY, total = 0.f;
#pragma unroll 4
      for (int s = lane >> 4; s < live; s += 4) {
        const f32x2 x = *reinterpret_cast<const f32x2*>(ml + (int64_t)s * rows_max * 2);
        const float now = fmaxf(top, x[0]);
        total = total * rescale(top, now) + x[1] * rescale(x[0], now);
        top = now;
      }
#pragma unroll
      for (int step = 16; step <= 32; step *= 2) {
        const float other = __shfl_xor(top, step), now = fmaxf(top, other);
        total = total * rescale(top, now) + __shfl_xor(total, step) * rescale(other, now);
        top = now;
      }
      l = lse_of(top, total);
    } else {
      l = a.lse2[(int64_t)(rows.first + m / a.G) * a.Hq + h * a.G + m % a.G];
    }
    auto meet = [] {
      if (TOGETHER) __syncthreads();
      else order_lds_of_wave();
    };
    meet();
    if (lane < 16) s_lse[wave * 16 + lane] = l == -INFINITY ? INFINITY : l;             // (a row without tokens adds nothing)
    meet();
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float* s = a.scores + (b * a.Hkv + min(h0 + e, a.Hkv - 1)) * rows_max * a.score_pitch + t;
      const int from = max(r0, e * per_head), to = min(min(r0 + kRows, all), (e + 1) * per_head);
#pragma unroll 4
      for (int x = from; x < to; ++x)
        more[e] += pow2(s[(int64_t)(x - e * per_head) * a.score_pitch] - s_lse[of_unit + x - r0]);
    }
  }
  sum += more;
  if (!ok) return;
  if (VEC) *reinterpret_cast<f32x4*>(w) = sum;
  else
    for (int e = 0; e < 4; ++e)
      if (h0 + e < a.Hkv) w[e] = sum[e];
}

// The splits joined and the weights added up, in one launch: both start from what the attention left.  3 to 10 us, with the
// weights of 16 x 16384 tokens of 32 query heads 18 (34 MB of scores, 8 of weights twice), of 24 ragged sequences of 64 heads 17.
template <int QT, int D, int PARTS, bool VEC, bool TOGETHER>
__global__ __launch_bounds__(kThreads) void attend_finish_kernel(AttendLaunch a, int join_groups, float* weights, int set) {
  if ((int)blockIdx.x < join_groups) join_rows<QT, D, PARTS>(a, blockIdx.x);
  else add_weights<VEC, TOGETHER>(a, weights, set, blockIdx.x - join_groups);
}

template <int QT, int D>
hipError_t launch_finish_typed(const AttendLaunch& a, float* weights, int set, hipStream_t s) {
  constexpr int kRows = kThreads / (D / 4);
  const int64_t rows = a.nsplit > 1 ? (int64_t)a.B * a.Hkv * a.max_rows * a.G : 0;
  // Many splits of few rows: a workgroup a row, its lanes side by side over the splits.  1 and 2 x 32768 tokens of 128 dimensions,
  // without and with it: 128 rows 13.7 and 5.2 us, 640 8.1 and 5.7, 1024 8.4 and 6.9, 2048 6.8 and 8.5 (64 dimensions: 1024 7.9 and
  // 5.8, 2048 8.4 and 9.2; 256: 10.5 and 9.5, 9.1 and 10.1).  Up to eight splits are asked for at once either way (4.2 and 4.2 us;
  // 640 rows 4.2 and 5.2).
  const bool wide = a.nsplit > kWideSplits && rows <= kWideRows;
  const int64_t joins = wide ? rows : ceil_div64(rows, kRows);
  const bool together = weights && (int64_t)std::min(a.Hkv, 4) * a.max_rows * a.G > 16;
  const int64_t quads = (int64_t)a.B * ceil_div(a.Hkv, 4);
  const int64_t adds = !weights ? 0 : together ? quads * ceil_div(a.Tmax, kThreads) : ceil_div64(quads * ceil_div(a.Tmax, kWave), kThreads / kWave);
  if (joins + adds == 0) return hipSuccess;
  if (joins + adds > INT32_MAX) return hipErrorInvalidValue;
  const bool vec = a.Hkv % 4 == 0 && reinterpret_cast<uintptr_t>(weights) % 16 == 0;
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)(joins + adds)), dim3(kThreads), 0, s, a, (int)joins, weights, set);
    return hipGetLastError();
  };
  auto pick = [&](auto parts, auto four) {
    constexpr int P = decltype(parts)::value;
    constexpr bool V = decltype(four)::value;
    return together ? go(attend_finish_kernel<QT, D, P, V, true>) : go(attend_finish_kernel<QT, D, P, V, false>);
  };
  using One = std::integral_constant<int, 1>;
  using Wide = std::integral_constant<int, kRows>;
  if (wide) return vec ? pick(Wide{}, std::true_type{}) : pick(Wide{}, std::false_type{});
  return vec ? pick(One{}, std::true_type{}) : pick(One{}, std::false_type{});
}

// 16 bytes a thread.
__global__ __launch_bounds__(kThreads) void copy_queries_kernel(AttendLaunch a, uint4* dst) {
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x, row = i / (a.D / 8);
  if (row >= (int64_t)a.num_rows * a.Hq) return;
  const uint16_t* q = reinterpret_cast<const uint16_t*>(a.q) + row / a.Hq * a.q_stride_row + row % a.Hq * a.q_stride_head + i % (a.D / 8) * 8;
  dst[i] = *reinterpret_cast<const uint4*>(q);
}

}  // namespace

hipError_t launch_copy_queries(const AttendLaunch& a, void* dst, hipStream_t s) {
  const int64_t groups = ceil_div64((int64_t)a.num_rows * a.Hq * (a.D / 8), kThreads);
  hipLaunchKernelGGL(copy_queries_kernel, dim3((unsigned)groups), dim3(kThreads), 0, s, a, reinterpret_cast<uint4*>(dst));
  return hipGetLastError();
}

hipError_t launch_attend(const AttendLaunch& a, hipStream_t s) {
  const bool bf16 = a.q_dtype == TRI_KV_BF16;
  if (a.D == 64) return bf16 ? launch_attend_64_bf16(a, s) : launch_attend_64_fp16(a, s);
  if (a.D == 128) return bf16 ? launch_attend_128_bf16(a, s) : launch_attend_128_fp16(a, s);
  return bf16 ? launch_attend_256_bf16(a, s) : launch_attend_256_fp16(a, s);
}

hipError_t launch_attend_finish(const AttendLaunch& a, float* weights, int set, hipStream_t s) {
  const bool bf16 = a.q_dtype == TRI_KV_BF16;
  if (a.D == 64) return bf16 ? launch_finish_typed<TRI_KV_BF16, 64>(a, weights, set, s) : launch_finish_typed<TRI_KV_FP16, 64>(a, weights, set, s);
  if (a.D == 128) return bf16 ? launch_finish_typed<TRI_KV_BF16, 128>(a, weights, set, s) : launch_finish_typed<TRI_KV_FP16, 128>(a, weights, set, s);
  return bf16 ? launch_finish_typed<TRI_KV_BF16, 256>(a, weights, set, s) : launch_finish_typed<TRI_KV_FP16, 256>(a, weights, set, s);
}

}  // namespace tri
