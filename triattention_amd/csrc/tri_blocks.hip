// Bounds of the keys of a block, and the scores by which a query's blocks are chosen.
//
//   low[d] = min over the block's tokens of k[d],  high[d] = max
//   score  = max (or mean) over the query heads of a KV head of  sum_d max(q[d] low[d], q[d] high[d])
// which no q . k of the block exceeds, where the bounds are keys of the cache: bf16, fp16 and fp8 without scales of its rows.  Scaled fp8
// keys are products in fp32, their bounds the nearest bf16 numbers: a key lies outside by half a step (2^-8 of the bound)
// at most, and a q . k above the score by 2^-8 sum_d |q[d] bound[d]|, which is how far such scores tell blocks apart.
#include <algorithm>
#include <cfloat>

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
// read once, 16 bytes a lane (fp8: 8).  Bound by reading the keys: 2 x 131072 tokens of 4 x 128 bf16 in 66 us (4.1 TB/s), the
// blocks of sixteen sequences' newest tokens in 7, the latency of dependent reads.
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
  const int count = min(a.block_size, T - j * a.block_size);
  if (count <= 0) return;
  const int page = a.block_table ? a.block_table[b * a.block_table_pitch + j] : (int)b;
  if (page < 0 || page >= a.num_blocks) return;
  const int h = piece / (a.D / 8), d = piece % (a.D / 8) * 8;
  const char* src = reinterpret_cast<const char*>(a.k_layers[l]) + ((int64_t)page * a.stride_block + (int64_t)h * a.stride_head + d) * ES;
  const float* sc = a.k_scale_layers ? a.k_scale_layers[l] + (int64_t)page * a.block_size * a.Hkv + h : nullptr;
  float low[8], high[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) { low[e] = INFINITY; high[e] = -INFINITY; }
  constexpr int kAtOnce = 16;         // tokens asked for together (the last one again where the block has fewer)
  for (int t0 = 0; t0 < count; t0 += kAtOnce) {
    uint4 w[kAtOnce];
    float f[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int t = min(t0 + u, count - 1);
      const char* row = src + (int64_t)t * a.stride_token * ES;
      if constexpr (DT == TRI_KV_FP8_E4M3) {
        const uint2 x = *reinterpret_cast<const uint2*>(row);
        w[u] = uint4{x.x, x.y, 0, 0};
        f[u] = sc ? sc[(int64_t)t * a.Hkv] : 1.f;
      } else {
        w[u] = *reinterpret_cast<const uint4*>(row);
      }
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      float x[8];
      if constexpr (DT == TRI_KV_FP8_E4M3) {
        x[0] = fp8_byte<0>(w[u].x); x[1] = fp8_byte<1>(w[u].x); x[2] = fp8_byte<2>(w[u].x); x[3] = fp8_byte<3>(w[u].x);
        x[4] = fp8_byte<0>(w[u].y); x[5] = fp8_byte<1>(w[u].y); x[6] = fp8_byte<2>(w[u].y); x[7] = fp8_byte<3>(w[u].y);
        if (sc) {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] *= f[u];
        }
      } else {
        unpack8<DT>(w[u], x);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        low[e] = low_of(low[e], x[e]);
        high[e] = high_of(high[e], x[e]);
      }
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
// order of a sum.  16 x 1024 blocks of 8 x 128, four query heads each: 67 MB in 23 to 24 us, 2.8 TB/s.  Counters of that call: vector
// instructions keep a SIMD busy for 12 us of it (one in seven is a 64-bit product, the others select, convert and exchange:
// low and high are converted anew for every head), and waves spend 45 % of their time waiting, for the loads of a workgroup's
// blocks, which all come first.  Neither bounds it alone; they hardly overlap.
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
  const int sub = threadIdx.x % LPB, slot = threadIdx.x / LPB;
  const bool b0 = (sub ^ sub >> 2) & 1, b1 = (sub >> 1 ^ sub >> 2) & 1;      // (the same in the lanes that the half mirror pairs)
  constexpr int kEach = kScoreBlocks / kBlocks;
  float best[kEach];
  double total[kEach];
  uint4 low_w[kEach], high_w[kEach];
  bool ok[kEach];
  int page[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int j = min(chunk * kScoreBlocks + i * kBlocks + slot, max(count - 1, 0));
    page[i] = a.block_table ? a.block_table[(int64_t)b * a.block_table_pitch + j] : b;
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    best[i] = -INFINITY;
    total[i] = 0.;
    ok[i] = page[i] >= 0 && page[i] < a.num_blocks;
    const uint16_t* src = reinterpret_cast<const uint16_t*>(a.bounds) + ((int64_t)(ok[i] ? page[i] : 0) * a.Hkv + h) * 2 * D + sub * 8;
    low_w[i] = *reinterpret_cast<const uint4*>(src);
    high_w[i] = *reinterpret_cast<const uint4*>(src + D);
  }
  for (int g0 = 0; g0 < a.G; g0 += kHeadsAtOnce) {
    double q64[kHeadsAtOnce][8];
    bool up[kHeadsAtOnce][8];
#pragma unroll
    for (int g = 0; g < kHeadsAtOnce; ++g) {
      float q[8];
      const uint16_t* src = reinterpret_cast<const uint16_t*>(a.q) + (int64_t)b * a.q_stride_row + (int64_t)(h * a.G + min(g0 + g, a.G - 1)) * a.q_stride_head + sub * 8;
      unpack8<QT>(*reinterpret_cast<const uint4*>(src), q);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        q64[g][e] = (double)q[e];
        up[g][e] = q[e] > 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      float low[8], high[8];
      unpack8<BT>(low_w[i], low);
      unpack8<BT>(high_w[i], high);
      double s[kHeadsAtOnce];
#pragma unroll
      for (int g = 0; g < kHeadsAtOnce; ++g) {
        s[g] = 0.;
#pragma unroll
        for (int e = 0; e < 8; ++e) s[g] = __builtin_fma(q64[g][e], (double)(up[g][e] ? high[e] : low[e]), s[g]);
      }
      // Over the block's lanes: the first two exchanges leave head 2 * b0 + b1 to a lane, the others add up.
      double s0 = (b0 ? s[2] : s[0]) + dpp64<kDppXor1>(b0 ? s[0] : s[2]);
      double s1 = (b0 ? s[3] : s[1]) + dpp64<kDppXor1>(b0 ? s[1] : s[3]);
      double mine = (b1 ? s1 : s0) + dpp64<kDppXor2>(b1 ? s0 : s1);
      mine += dpp64<kDppHalfMirror>(mine);
      if (LPB >= 16) mine += dpp64<kDppRor8>(mine);
      if (LPB >= 32) mine += __shfl_xor(mine, 16);
      const bool in = g0 + (b0 ? 2 : 0) + (b1 ? 1 : 0) < a.G;
      total[i] += in ? mine : 0.;
      best[i] = in ? high_of((float)mine, best[i]) : best[i];
    }
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    // (the four lanes at the front hold the heads)
    best[i] = high_of(best[i], dpp<kDppXor1>(best[i]));
    best[i] = high_of(best[i], dpp<kDppXor2>(best[i]));
    total[i] += dpp64<kDppXor1>(total[i]);
    total[i] += dpp64<kDppXor2>(total[i]);
    const int j = chunk * kScoreBlocks + i * kBlocks + slot;
    if (j >= count || sub != 0) continue;
    float s = a.group_max ? best[i] : (float)(total[i] / a.G);
    if (!ok[i]) s = -INFINITY;
    // (a NaN in a query or a key should come out of the attention as it would without the selection: its block comes first, but for
    // those asked for by their place)
    if (__builtin_isnan(s) || s > FLT_MAX) s = FLT_MAX;
    if (j < a.sinks || j >= count - a.recent) s = INFINITY;
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
