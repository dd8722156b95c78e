// New tokens' rows into the paged cache, and cached rows out of it (gfx950).
//
//  write_paged_kernel : q and k normalised per head and rotated, q stored, K and V stored (quantised) in their slots
//  read_paged_kernel  : rows of sequences as dense K and V, scales multiplied in
//
//   y = x rsqrt(mean(x^2) + eps) w                          (with a norm; w of the head's dimensions)
//   (z1, z2) = (y1 cos t - y2 sin t, y2 cos t + y1 sin t) c,   t = position[axis(f)] inv_freq[f]
// for the pairs (f, f + D/2) or (2f, 2f + 1) of a head, c the rotary scale.
#include <algorithm>
#include <cfloat>

#include "tri_common.h"
#include "tri_mma_device.h"
#include "tri_rows_device.h"
#include "tri_score_device.h"

namespace tri {
namespace {

constexpr int kWriteThreads = 256;
constexpr int kWriteWaves = kWriteThreads / kWave;
constexpr int kStepsAtOnce = 4;            // steps of a wave asked for together
typedef __attribute__((address_space(1))) char* GlobalOut;
typedef __attribute__((address_space(1))) u32x2* GlobalOutU2;
typedef __attribute__((address_space(1))) uint32_t* GlobalOutU1;
typedef __attribute__((address_space(1))) float* GlobalOutF32;
enum CacheKind { kPlainRows = 0, kTensorScale = 1, kRowScales = 2 };

// cos and sin of position * inv_freq.  The product and its reduction by pi / 2 are 64-bit: the remainder of an angle of 2^31
// is off by 2^-54 a step, where an angle in 32 bits would be off by whole turns.  On [-pi/4, pi/4] the Taylor series up to r^9
// and r^10 in 32 bits (the next terms are below 2e-9).
__device__ __forceinline__ void turn(double position, float inv_freq, float scale, float& c_out, float& s_out) {
  const double x = position * (double)inv_freq;
  const double n = __builtin_rint(x * 0.636619772367581343075535);
  double rest = __builtin_fma(-n, 1.57079632679489655799898, x);
  rest = __builtin_fma(-n, 6.12323399573676603586882e-17, rest);
  const int quadrant = (int)(n - 4.0 * __builtin_floor(n * 0.25));
  const float r = (float)rest, z = r * r;
  const float s = r + r * z * (-1.f / 6 + z * (1.f / 120 + z * (-1.f / 5040 + z * (1.f / 362880))));
  const float c = 1.f + z * (-0.5f + z * (1.f / 24 + z * (-1.f / 720 + z * (1.f / 40320 + z * (-1.f / 3628800)))));
  const float cq = quadrant & 1 ? s : c, sq = quadrant & 1 ? c : s;
  c_out = (quadrant == 1 || quadrant == 2 ? -cq : cq) * scale;
  s_out = (quadrant >= 2 ? -sq : sq) * scale;
}

// Over the lanes of a head (8, 16 or 32 of them), the result in each.
template <int LPH>
__device__ __forceinline__ float sum_of_head(float v) {
  v += dpp<kDppXor1>(v);
  v += dpp<kDppXor2>(v);
  v += dpp<kDppHalfMirror>(v);
  if constexpr (LPH >= 16) v += dpp<kDppRor8>(v);
  if constexpr (LPH >= 32) v += __shfl_xor(v, 16);
  return v;
}
template <int LPH>
__device__ __forceinline__ float max_of_head(float v) {
  v = fmaxf(v, dpp<kDppXor1>(v));
  v = fmaxf(v, dpp<kDppXor2>(v));
  v = fmaxf(v, dpp<kDppHalfMirror>(v));
  if constexpr (LPH >= 16) v = fmaxf(v, dpp<kDppRor8>(v));
  if constexpr (LPH >= 32) v = fmaxf(v, __shfl_xor(v, 16));
  return v;
}

template <int T>
__device__ __forceinline__ uint32_t pack_half(float a, float b) {
  if constexpr (T == TRI_KV_FP16) {
    f16x2 v = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, v);
  } else {
    bf16x2 v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, v);
  }
}
__device__ __forceinline__ bool is_number(float x) { return fabsf(x) <= FLT_MAX; }

// Four e4m3 codes of x * inv: rounded to nearest, beyond 448 the largest; infinities and NaN are NaN.
__device__ __forceinline__ uint32_t pack_codes(const float* x, float inv) {
  float y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float v = x[e] * inv;
    y[e] = is_number(x[e]) ? fminf(fmaxf(v, -448.f), 448.f) : __builtin_nanf("");
  }
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
}

// A wave's step is 64 / (D / 8) heads of one kind (queries, keys or values) of a row, eight elements a lane: those whose pairs lie in
// the lane (4l to 4l + 3 and the same behind the head's middle, or 8l to 8l + 7), so that the rotation needs no other lane, and a lane
// has the same four angles in every head.  A row's steps are shared by waves_per_row waves, which find the angles once each.
template <int D, int QT, int KIND>
__global__ __launch_bounds__(kWriteThreads) void write_paged_kernel(WriteLaunch a) {
  constexpr int LPH = D / 8, HPW = kWave / LPH;
  const int lane = threadIdx.x % kWave, l = lane % LPH, sub = lane / LPH;
  const int unit = blockIdx.x * kWriteWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int row = unit / a.waves_per_row, part = unit % a.waves_per_row;
  if (row >= a.num_rows) return;
  int b = row;
  if (a.row_starts) {
    b = __builtin_amdgcn_readfirstlane(sequence_of_row(a.row_starts, a.B, row, lane));
    if (b < 0) return;
  }
  const int q_steps = ceil_div(a.Hq, HPW), kv_steps = ceil_div(a.Hkv, HPW), steps = q_steps + 2 * kv_steps;
  // elements of a head that are this lane's: first to first + 3 and second to second + 3
  const bool half = a.rope_style == TRI_ROPE_HALF;
  const int first = half ? 4 * l : 8 * l, second = half ? D / 2 + 4 * l : 8 * l + 4;

  float cs[4], sn[4];
  if (part < q_steps + kv_steps) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int f = 4 * l + e;
      int axis = a.freq_axes ? a.freq_axes[f] : 0;
      if (axis < 0 || axis >= a.num_axes) axis = 0;
      const int64_t at = axis * a.position_stride + row;
      const double position = a.positions_64 ? (double)reinterpret_cast<const int64_t*>(a.positions)[at]
                                             : (double)reinterpret_cast<const int32_t*>(a.positions)[at];
      turn(position, a.inv_freq[f], a.rotary_scale, cs[e], sn[e]);
    }
  }
  int page = -1, off = 0;
  if (part + (steps - 1 - part) / a.waves_per_row * a.waves_per_row >= q_steps) {
    const int t = token_of_row(a.row_starts, a.seq_lens, a.Tmax, b, row);
    if (t >= 0) {
      page = page_of_token(a.block_table, a.block_table_pitch, a.block_size, a.num_blocks, b, t);
      off = t % a.block_size;
    }
  }

  float w[8];
  const void* have = nullptr;
  for (int s0 = part; s0 < steps; s0 += kStepsAtOnce * a.waves_per_row) {
    uint2 raw[kStepsAtOnce][2];
#pragma unroll
    for (int u = 0; u < kStepsAtOnce; ++u) {
      const int s = s0 + u * a.waves_per_row;
      const int kind = s < q_steps ? 0 : s < q_steps + kv_steps ? 1 : 2;
      const int h = (s - (kind == 0 ? 0 : kind == 1 ? q_steps : q_steps + kv_steps)) * HPW + sub;
      raw[u][0] = raw[u][1] = uint2{0, 0};
      if (s < steps && h < (kind == 0 ? a.Hq : a.Hkv)) {
        const uint16_t* src = reinterpret_cast<const uint16_t*>(kind == 0 ? a.q : kind == 1 ? a.k : a.v) +
                              row * (kind == 0 ? a.q_stride_row : kind == 1 ? a.k_stride_row : a.v_stride_row) +
                              h * (kind == 0 ? a.q_stride_head : kind == 1 ? a.k_stride_head : a.v_stride_head);
        raw[u][0] = *reinterpret_cast<const uint2*>(src + first);
        raw[u][1] = *reinterpret_cast<const uint2*>(src + second);
      }
    }
#pragma unroll
    for (int u = 0; u < kStepsAtOnce; ++u) {
      const int s = s0 + u * a.waves_per_row;
      if (s >= steps) break;
      const int kind = s < q_steps ? 0 : s < q_steps + kv_steps ? 1 : 2;
      const int h = (s - (kind == 0 ? 0 : kind == 1 ? q_steps : q_steps + kv_steps)) * HPW + sub;
      const bool mine = h < (kind == 0 ? a.Hq : a.Hkv);
      const uint32_t word[4] = {raw[u][0].x, raw[u][0].y, raw[u][1].x, raw[u][1].y};
      float x[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[2 * e] = elem_lo<QT>(word[e]);
        x[2 * e + 1] = elem_hi<QT>(word[e]);
      }
      if (kind != 2) {
        const void* norm = kind == 0 ? a.q_norm : a.k_norm;
        if (norm) {
          if (norm != have) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int d = e < 4 ? first + e : second + e - 4;
              if (a.norm_fp32) w[e] = reinterpret_cast<const float*>(norm)[d];
              else w[e] = elem_lo<QT>(reinterpret_cast<const uint16_t*>(norm)[d]);
            }
            have = norm;
          }
          float squares = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) squares += x[e] * x[e];
          const float inv = rsqrtf(sum_of_head<LPH>(squares) * (1.f / D) + a.eps);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = x[e] * inv * w[e];
        }
        if (half) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float y = x[e], z = x[4 + e];
            x[e] = y * cs[e] - z * sn[e];
            x[4 + e] = z * cs[e] + y * sn[e];
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float y = x[2 * e], z = x[2 * e + 1];
            x[2 * e] = y * cs[e] - z * sn[e];
            x[2 * e + 1] = z * cs[e] + y * sn[e];
          }
        }
      }
      if (kind == 0) {
        if (!mine) continue;
        uint16_t* dst = reinterpret_cast<uint16_t*>(a.out) + row * a.out_stride_row + h * a.out_stride_head;
        *reinterpret_cast<uint2*>(dst + first) = uint2{pack_half<QT>(x[0], x[1]), pack_half<QT>(x[2], x[3])};
        *reinterpret_cast<uint2*>(dst + second) = uint2{pack_half<QT>(x[4], x[5]), pack_half<QT>(x[6], x[7])};
        continue;
      }
      if (page < 0) continue;
      const GlobalOut base = (GlobalOut)(uintptr_t)(kind == 1 ? a.k_layers : a.v_layers)[a.layer];
      const int64_t at = (int64_t)page * a.stride_block + off * a.stride_token + h * a.stride_head;
      if constexpr (KIND == kPlainRows) {
        if (!mine) continue;
        *(GlobalOutU2)(base + (at + first) * 2) = u32x2{pack_half<QT>(x[0], x[1]), pack_half<QT>(x[2], x[3])};
        *(GlobalOutU2)(base + (at + second) * 2) = u32x2{pack_half<QT>(x[4], x[5]), pack_half<QT>(x[6], x[7])};
      } else {
        float inv = kind == 1 ? a.k_inv_scale : a.v_inv_scale;
        float scale = 0.f;
        if constexpr (KIND == kRowScales) {
          // of the finite elements: an infinity or NaN is a NaN in its place and leaves the others as they are
          float most = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) most = fmaxf(most, is_number(x[e]) ? fabsf(x[e]) : 0.f);
          scale = fmaxf(max_of_head<LPH>(most) / 448.f, FLT_MIN);
          inv = 1.f / scale;
        }
        if (!mine) continue;
        *(GlobalOutU1)(base + at + first) = pack_codes(x, inv);
        *(GlobalOutU1)(base + at + second) = pack_codes(x + 4, inv);
        if constexpr (KIND == kRowScales)
          if (l == 0)
            *((GlobalOutF32)(uintptr_t)(kind == 1 ? a.k_scale_layers : a.v_scale_layers)[a.layer] + ((int64_t)page * a.block_size + off) * a.Hkv + h) = scale;
      }
    }
  }
}

// A wave takes rows_per_wave rows one behind the other; their places are found a row a lane.  Lanes are pieces of eight elements
// of the row's K, then of its V.
constexpr int kReadAtOnce = 8;             // pieces of a lane asked for together

template <int CT, int OT>
__global__ __launch_bounds__(kWriteThreads) void read_paged_kernel(ReadLaunch a) {
  const int lane = threadIdx.x % kWave;
  const int64_t r0 = ((int64_t)blockIdx.x * kWriteWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave)) * a.rows_per_wave;
  if (r0 >= a.num_rows) return;
  const int rows = (int)min((int64_t)a.rows_per_wave, a.num_rows - r0);
  // lane i has row i's place: slot >= 0, -1 for a row without a cached token (zeros), -2 for one that no sequence has
  int page = -2, off = 0;
  if (lane < rows) {
    const int row = (int)r0 + lane;
    int lo = 0, n = a.B;
    while (n > 1) {
      const int m = n / 2;
      if (a.row_starts[lo + m] <= row) { lo += m; n -= m; }
      else n = m;
    }
    if (a.row_starts[lo] <= row && row < a.row_starts[lo + 1]) {
      const int t = token_of_row(a.row_starts, a.seq_lens, a.Tmax, lo, row);
      page = t < 0 ? -1 : page_of_token(a.block_table, a.block_table_pitch, a.block_size, a.num_blocks, lo, t);
      off = t < 0 ? 0 : t % a.block_size;
    }
  }
  const int shift = a.D == 64 ? 3 : a.D == 128 ? 4 : 5, pieces = a.Hkv << shift, per_row = ceil_div(2 * pieces, kWave);
  const int total = rows * per_row;
  for (int i0 = 0; i0 < total; i0 += kReadAtOnce) {
    uint4 raw[kReadAtOnce];
    float scale[kReadAtOnce];
#pragma unroll
    for (int u = 0; u < kReadAtOnce; ++u) {
      const int i = min(i0 + u, total - 1), r = i / per_row, item = (i - r * per_row) * kWave + lane;
      const bool v = item >= pieces;
      const int piece = v ? item - pieces : item, h = piece >> shift, d = (piece & ((1 << shift) - 1)) * 8;
      const int p = __builtin_amdgcn_readlane(page, r), o = __builtin_amdgcn_readlane(off, r);
      raw[u] = uint4{0, 0, 0, 0};
      scale[u] = 0.f;
      if (p >= 0 && item < 2 * pieces) {
        const int64_t at = (int64_t)p * a.stride_block + o * a.stride_token + h * a.stride_head + d;
        const GlobalBytes base = (GlobalBytes)(uintptr_t)(v ? a.v_layers : a.k_layers)[a.layer];
        scale[u] = v ? a.v_scale : a.k_scale;
        if constexpr (CT == TRI_KV_FP8_E4M3) {
          const u32x2 x = *(GlobalU2)(base + at);
          raw[u] = uint4{x.x, x.y, 0, 0};
          if (a.k_scale_layers)
            scale[u] *= *((GlobalF32)(uintptr_t)(v ? a.v_scale_layers : a.k_scale_layers)[a.layer] + ((int64_t)p * a.block_size + o) * a.Hkv + h);
        } else {
          const u32x4 x = *(GlobalU4)(base + at * 2);
          raw[u] = uint4{x.x, x.y, x.z, x.w};
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kReadAtOnce; ++u) {
      const int i = i0 + u;
      if (i >= total) break;
      const int r = i / per_row, item = (i - r * per_row) * kWave + lane;
      const bool v = item >= pieces;
      const int piece = v ? item - pieces : item;
      if (__builtin_amdgcn_readlane(page, r) == -2 || item >= 2 * pieces) continue;
      float x[8];
      if constexpr (CT == TRI_KV_FP8_E4M3) {
        x[0] = fp8_byte<0>(raw[u].x); x[1] = fp8_byte<1>(raw[u].x); x[2] = fp8_byte<2>(raw[u].x); x[3] = fp8_byte<3>(raw[u].x);
        x[4] = fp8_byte<0>(raw[u].y); x[5] = fp8_byte<1>(raw[u].y); x[6] = fp8_byte<2>(raw[u].y); x[7] = fp8_byte<3>(raw[u].y);
      } else {
        const uint32_t word[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[2 * e] = elem_lo<CT>(word[e]);
          x[2 * e + 1] = elem_hi<CT>(word[e]);
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= scale[u];
      const int64_t to = ((r0 + r) * pieces + piece) * 8;
      void* const out = v ? a.v_out : a.k_out;
      if constexpr (OT == TRI_REAL_FP32) {
        float4* dst = reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + to);
        dst[0] = float4{x[0], x[1], x[2], x[3]};
        dst[1] = float4{x[4], x[5], x[6], x[7]};
      } else {
        *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(out) + to) =
            uint4{pack_half<OT>(x[0], x[1]), pack_half<OT>(x[2], x[3]), pack_half<OT>(x[4], x[5]), pack_half<OT>(x[6], x[7])};
      }
    }
  }
}

template <int D, int QT>
void write_of_kind(const WriteLaunch& a, hipStream_t s) {
  const dim3 grid((unsigned)ceil_div64((int64_t)a.num_rows * a.waves_per_row, kWriteWaves));
  if (a.kv_dtype != TRI_KV_FP8_E4M3) hipLaunchKernelGGL((write_paged_kernel<D, QT, kPlainRows>), grid, dim3(kWriteThreads), 0, s, a);
  else if (!a.k_scale_layers) hipLaunchKernelGGL((write_paged_kernel<D, QT, kTensorScale>), grid, dim3(kWriteThreads), 0, s, a);
  else hipLaunchKernelGGL((write_paged_kernel<D, QT, kRowScales>), grid, dim3(kWriteThreads), 0, s, a);
}
template <int D>
void write_of_type(const WriteLaunch& a, hipStream_t s) {
  if (a.q_dtype == TRI_KV_FP16) write_of_kind<D, TRI_KV_FP16>(a, s);
  else write_of_kind<D, TRI_KV_BF16>(a, s);
}
template <int CT>
void read_to_type(const ReadLaunch& a, hipStream_t s) {
  const dim3 grid((unsigned)ceil_div64(ceil_div64(a.num_rows, a.rows_per_wave), kWriteWaves));
  if (a.out_dtype == TRI_REAL_FP32) hipLaunchKernelGGL((read_paged_kernel<CT, TRI_REAL_FP32>), grid, dim3(kWriteThreads), 0, s, a);
  else if (a.out_dtype == TRI_REAL_FP16) hipLaunchKernelGGL((read_paged_kernel<CT, TRI_REAL_FP16>), grid, dim3(kWriteThreads), 0, s, a);
  else hipLaunchKernelGGL((read_paged_kernel<CT, TRI_REAL_BF16>), grid, dim3(kWriteThreads), 0, s, a);
}

}  // namespace

hipError_t launch_write_paged(WriteLaunch a, hipStream_t s) {
  const int heads = kWave / (a.D / 8), steps = ceil_div(a.Hq, heads) + 2 * ceil_div(a.Hkv, heads);
  // As many waves a row as fill the chip, down to a step each.
  a.waves_per_row = (int)std::min<int64_t>(steps, std::max<int64_t>(1, 8192 / a.num_rows));
  if (a.D == 64) write_of_type<64>(a, s);
  else if (a.D == 128) write_of_type<128>(a, s);
  else write_of_type<256>(a, s);
  return hipGetLastError();
}

hipError_t launch_read_paged(ReadLaunch a, hipStream_t s) {
  a.rows_per_wave = (int)std::min<int64_t>(8, std::max<int64_t>(1, a.num_rows / 8192));
  if (a.kv_dtype == TRI_KV_FP8_E4M3) read_to_type<TRI_KV_FP8_E4M3>(a, s);
  else if (a.kv_dtype == TRI_KV_FP16) read_to_type<TRI_KV_FP16>(a, s);
  else read_to_type<TRI_KV_BF16>(a, s);
  return hipGetLastError();
}

}  // namespace tri
