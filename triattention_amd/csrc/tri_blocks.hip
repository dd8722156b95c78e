// Bounds of the keys of a block, and the scores by which a query's blocks are chosen.
//
//   low[d] = min over the block's tokens of k[d],  high[d] = max
//   score  = max (or mean) over the query heads of a KV head of  sum_d max(q[d] low[d], q[d] high[d])
// which no q . k of the block exceeds.
#include <algorithm>

#include "tri_common.h"
#include "tri_mma_device.h"
#include "tri_score_device.h"

namespace tri {
namespace {

// The smaller / larger of two numbers, NaN if either is one.
__device__ __forceinline__ float low_of(float a, float b) { return __builtin_isnan(a) || a < b ? a : b; }
__device__ __forceinline__ float high_of(float a, float b) { return __builtin_isnan(a) || a > b ? a : b; }

template <int DT>
__device__ __forceinline__ void unpack8(const uint4& w, float (&x)[8]) {
  const uint32_t* p = reinterpret_cast<const uint32_t*>(&w);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = elem_lo<DT>(p[i]);
    x[2 * i + 1] = elem_hi<DT>(p[i]);
  }
}
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (DT == TRI_KV_FP16) {
    f16x2 v = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, v);
  } else {
    bf16x2 v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, v);
  }
}
template <int DT>
__device__ __forceinline__ void store8(uint16_t* dst, const float (&x)[8]) {
  *reinterpret_cast<uint4*>(dst) = uint4{pack2<DT>(x[0], x[1]), pack2<DT>(x[2], x[3]), pack2<DT>(x[4], x[5]), pack2<DT>(x[6], x[7])};
}

// A wave reduces 64 pieces of 8 elements (of all heads, one behind the other) of one block over its tokens: every key is
// read once, 16 bytes a lane (fp8: 8).  Bound by reading the keys.
template <int DT>
__global__ __launch_bounds__(256) void block_bounds_kernel(BoundsLaunch a, int blocks_per_seq, int waves_per_block) {
  constexpr int ES = DT == TRI_KV_FP8_E4M3 ? 1 : 2;
  constexpr int BT = DT == TRI_KV_FP8_E4M3 ? TRI_KV_BF16 : DT;
  const int lane = threadIdx.x % kWave;
  int64_t unit = (int64_t)blockIdx.x * (256 / kWave) + threadIdx.x / kWave;
  const int piece = (int)(unit % waves_per_block) * kWave + lane;
  unit /= waves_per_block;
  int j = (int)(unit % blocks_per_seq);
  unit /= blocks_per_seq;
  const int l = (int)(unit % a.L);
  const int64_t b = unit / a.L;
  if (b >= a.B || piece >= a.Hkv * (a.D / 8)) return;
  const int T = min(max(a.seq_lens[b], 0), a.Tmax);
  if (a.new_tokens > 0) j += max(T - a.new_tokens, 0) / a.block_size;
  const int t0 = j * a.block_size, count = min(a.block_size, T - t0);
  if (count <= 0) return;
  const int page = a.block_table ? a.block_table[b * a.block_table_pitch + j] : (int)b;
  if (page < 0 || page >= a.num_blocks) return;
  const int h = piece / (a.D / 8), d = piece % (a.D / 8) * 8;
  const char* src = reinterpret_cast<const char*>(a.k_layers[l]) + ((int64_t)page * a.stride_block + (int64_t)h * a.stride_head + d) * ES;
  const float* sc = a.k_scale_layers ? a.k_scale_layers[l] + (int64_t)page * a.block_size * a.Hkv + h : nullptr;
  float low[8], high[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) { low[e] = INFINITY; high[e] = -INFINITY; }
#pragma unroll 8
  for (int t = 0; t < count; ++t) {
    float x[8];
    const char* row = src + (int64_t)t * a.stride_token * ES;
    if constexpr (DT == TRI_KV_FP8_E4M3) {
      const uint2 w = *reinterpret_cast<const uint2*>(row);
      x[0] = fp8_byte<0>(w.x); x[1] = fp8_byte<1>(w.x); x[2] = fp8_byte<2>(w.x); x[3] = fp8_byte<3>(w.x);
      x[4] = fp8_byte<0>(w.y); x[5] = fp8_byte<1>(w.y); x[6] = fp8_byte<2>(w.y); x[7] = fp8_byte<3>(w.y);
      if (sc) {
        const float f = sc[(int64_t)t * a.Hkv];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= f;
      }
    } else {
      unpack8<DT>(*reinterpret_cast<const uint4*>(row), x);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      low[e] = low_of(low[e], x[e]);
      high[e] = high_of(high[e], x[e]);
    }
  }
  uint16_t* dst = reinterpret_cast<uint16_t*>(a.bounds) + (int64_t)l * a.bounds_stride_layer + ((int64_t)page * a.Hkv + h) * 2 * a.D + d;
  store8<BT>(dst, low);
  store8<BT>(dst + a.D, high);
}

template <int CTRL>
__device__ __forceinline__ double dpp64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xf, 0xf, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xf, 0xf, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

constexpr int kScoreBlocks = 64;       // blocks of a (sequence, KV head) per workgroup
constexpr int kHeadsAtOnce = 4;

// D / 8 lanes a block, 8 elements each, the queries of up to four heads in registers: a positive element of a query meets the
// largest key, a negative one the least.  Products and sums are 64-bit: which blocks are read must not depend on the
// order of a sum.  Bound by reading the bounds and, from four heads on, by the 64-bit products of every head
// (selection, conversion and product are three instructions an element).
template <int BT, int QT, int D>
__global__ __launch_bounds__(256) void block_scores_kernel(BlockScoreLaunch a) {
  constexpr int LPB = D / 8, kBlocks = 256 / LPB;
  const int chunks = ceil_div(a.max_count, kScoreBlocks);
  int idx = blockIdx.x;
  const int h = idx % a.Hkv; idx /= a.Hkv;
  const int chunk = idx % chunks;
  const int b = idx / chunks;
  const int T = min(max(a.seq_lens[b], 0), a.Tmax);
  const int count = ceil_div(T, a.block_size), taken = min(a.top, count);
  const int64_t row = (int64_t)b * a.Hkv + h;
  if (chunk == 0) {
    if (h == 0 && threadIdx.x == 0) {
      a.counts[b] = count;
      a.counts[a.B + b] = taken;
    }
    for (int i = taken + threadIdx.x; i < a.top; i += 256) a.blocks[row * a.top + i] = -1;
  }
  const int sub = threadIdx.x % LPB;
  float best[kScoreBlocks / kBlocks];
  double total[kScoreBlocks / kBlocks];
#pragma unroll
  for (int i = 0; i < kScoreBlocks / kBlocks; ++i) { best[i] = -INFINITY; total[i] = 0.; }
  for (int g0 = 0; g0 < a.G; g0 += kHeadsAtOnce) {
    float q[8];
    double q64[kHeadsAtOnce][8];
    bool up[kHeadsAtOnce][8];
#pragma unroll
    for (int g = 0; g < kHeadsAtOnce; ++g) {
      const int gg = min(g0 + g, a.G - 1);
      const uint16_t* src = reinterpret_cast<const uint16_t*>(a.q) + (int64_t)b * a.q_stride_row + (int64_t)(h * a.G + gg) * a.q_stride_head + sub * 8;
      unpack8<QT>(*reinterpret_cast<const uint4*>(src), q);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        q64[g][e] = (double)q[e];
        up[g][e] = q[e] > 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < kScoreBlocks / kBlocks; ++i) {
      const int j = chunk * kScoreBlocks + i * kBlocks + threadIdx.x / LPB;
      if (j >= count) continue;
      const int page = a.block_table ? a.block_table[(int64_t)b * a.block_table_pitch + j] : b;
      const bool ok = page >= 0 && page < a.num_blocks;
      const uint16_t* src = reinterpret_cast<const uint16_t*>(a.bounds) + ((int64_t)(ok ? page : 0) * a.Hkv + h) * 2 * D + sub * 8;
      float low[8], high[8];
      unpack8<BT>(*reinterpret_cast<const uint4*>(src), low);
      unpack8<BT>(*reinterpret_cast<const uint4*>(src + D), high);
#pragma unroll
      for (int g = 0; g < kHeadsAtOnce; ++g) {
        double s = 0.;
#pragma unroll
        for (int e = 0; e < 8; ++e) s = __builtin_fma(q64[g][e], (double)(up[g][e] ? high[e] : low[e]), s);
        s += dpp64<kDppXor1>(s);
        s += dpp64<kDppXor2>(s);
        s += dpp64<kDppHalfMirror>(s);
        if (LPB >= 16) s += dpp64<kDppRor8>(s);
        if (LPB >= 32) s += __shfl_xor(s, 16);
        if (!ok) s = -INFINITY;
        if (g0 + g < a.G) {
          total[i] += s;
          best[i] = high_of((float)s, best[i]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kScoreBlocks / kBlocks; ++i) {
    const int j = chunk * kScoreBlocks + i * kBlocks + threadIdx.x / LPB;
    if (j >= count || sub != 0) continue;
    float s = a.group_max ? best[i] : (float)(total[i] / a.G);
    // (a NaN in a query or a key must come out of the attention as it would without the selection: its block is read)
    if (j < a.sinks || j >= count - a.recent || __builtin_isnan(s)) s = INFINITY;
    a.scores[row * a.max_count + j] = s;
  }
}

template <int BT, int QT>
hipError_t launch_scores_typed(const BlockScoreLaunch& a, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)a.B * ceil_div(a.max_count, kScoreBlocks) * a.Hkv));
  if (a.D == 64) hipLaunchKernelGGL((block_scores_kernel<BT, QT, 64>), grid, dim3(256), 0, s, a);
  else if (a.D == 128) hipLaunchKernelGGL((block_scores_kernel<BT, QT, 128>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((block_scores_kernel<BT, QT, 256>), grid, dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_block_bounds(const BoundsLaunch& a, hipStream_t s) {
  const int all = ceil_div(a.Tmax, a.block_size);
  const int per_seq = a.new_tokens > 0 ? std::min(all, (a.new_tokens + a.block_size - 2) / a.block_size + 1) : all;
  const int waves = ceil_div(a.Hkv * (a.D / 8), kWave);
  const int64_t units = (int64_t)a.B * a.L * per_seq * waves;
  const dim3 grid((unsigned)ceil_div64(units, 256 / kWave));
  if (a.kv_dtype == TRI_KV_BF16) hipLaunchKernelGGL(block_bounds_kernel<TRI_KV_BF16>, grid, dim3(256), 0, s, a, per_seq, waves);
  else if (a.kv_dtype == TRI_KV_FP16) hipLaunchKernelGGL(block_bounds_kernel<TRI_KV_FP16>, grid, dim3(256), 0, s, a, per_seq, waves);
  else hipLaunchKernelGGL(block_bounds_kernel<TRI_KV_FP8_E4M3>, grid, dim3(256), 0, s, a, per_seq, waves);
  return hipGetLastError();
}

hipError_t launch_block_scores(const BlockScoreLaunch& a, hipStream_t s) {
  if (a.bounds_dtype == TRI_KV_FP16) return launch_scores_typed<TRI_KV_FP16, TRI_KV_FP16>(a, s);
  return a.q_dtype == TRI_KV_FP16 ? launch_scores_typed<TRI_KV_BF16, TRI_KV_FP16>(a, s) : launch_scores_typed<TRI_KV_BF16, TRI_KV_BF16>(a, s);
}

}  // namespace tri
