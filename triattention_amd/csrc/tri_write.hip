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
constexpr int kStepsAtOnce = 2;            // steps of a wave asked for together
typedef __attribute__((address_space(1))) char* GlobalOut;
typedef __attribute__((address_space(1))) u32x2* GlobalOutU2;
typedef __attribute__((address_space(1))) uint32_t* GlobalOutU1;
typedef __attribute__((address_space(1))) u32x4* GlobalOutU4;
typedef __attribute__((address_space(1))) float* GlobalOutF32;
enum CacheKind { kPlainRows = 0, kTensorScale = 1, kRowScales = 2 };
enum PastCaches { kCached = 0, kReadPast = 1, kAllPast = 2 };       // what goes past the caches: reads of q, k and v, stores of q too

// cos and sin of position * inv_freq, times scale, rounded once.  The angle is the 64-bit product: exact for positions below 2^29, at 2^31 off by up to
// 2^-23, at 2^40 by 2^-14.  What is left of it beside a multiple of pi / 2 is off by 2^-53, and on [-pi/4, pi/4] the Taylor series up to r^13 and
// r^14 by 2^-45.  (In 32 bits the series were off by a step: one rotated number in 30000 was its neighbour in fp16.)
__device__ __forceinline__ void turn(double position, float inv_freq, float scale, float& c_out, float& s_out) {
  const double x = position * (double)inv_freq;
  const double n = __builtin_rint(x * 0.636619772367581343075535);
  double r = __builtin_fma(-n, 1.57079632679489655799898, x);
  r = __builtin_fma(-n, 6.12323399573676603586882e-17, r);
  const int quadrant = (int)(n - 4.0 * __builtin_floor(n * 0.25));
  const double z = r * r;
  double s = 1.0 / 6227020800, c = -1.0 / 87178291200;
  s = __builtin_fma(s, z, -1.0 / 39916800);
  c = __builtin_fma(c, z, 1.0 / 479001600);
  s = __builtin_fma(s, z, 1.0 / 362880);
  c = __builtin_fma(c, z, -1.0 / 3628800);
  s = __builtin_fma(s, z, -1.0 / 5040);
  c = __builtin_fma(c, z, 1.0 / 40320);
  s = __builtin_fma(s, z, 1.0 / 120);
  c = __builtin_fma(c, z, -1.0 / 720);
  s = __builtin_fma(s, z, -1.0 / 6);
  c = __builtin_fma(c, z, 1.0 / 24);
  s = __builtin_fma(s * z, r, r);
  c = __builtin_fma(__builtin_fma(c, z, -0.5), z, 1.0);
  const double cq = quadrant & 1 ? s : c, sq = quadrant & 1 ? c : s;
  c_out = (float)((quadrant == 1 || quadrant == 2 ? -cq : cq) * scale);
  s_out = (float)((quadrant >= 2 ? -sq : sq) * scale);
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
    // (numbers of 32 bits: the rounding is not drawn into the product before it)
    asm("" : "+v"(a), "+v"(b));
    f16x2 v = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, v);
  } else {
    bf16x2 v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, v);
  }
}
__device__ __forceinline__ bool is_number(float x) { return fabsf(x) <= FLT_MAX; }

// What an fp8 row's numbers are divided by: a power of two away from where reciprocals and remainders lose bits, and its reciprocal.
struct Unit {
  float up, unit, inv;
  __device__ __forceinline__ explicit Unit(float scale)
      : up(scale < 0x1p-64f ? 0x1p64f : scale > 0x1p64f ? 0x1p-64f : 1.f), unit(scale * up), inv(1.f / unit) {}
};
// Four e4m3 codes of the 32-bit quotients x / scale: rounded to nearest, beyond 448 the largest; infinities and NaN are NaN.  A product by the
// reciprocal is off by up to 1.5 steps, and one remainder corrects it but for quotients within 2^-22 of a step of the middle between two
// numbers.  Where one of those is a tie of codes (17, 19 .. 31 times a power of two) and the scale's mantissa hence within 8 of a multiple of 2^20, all
// corrected products are the quotients: the codes are those of a division, which takes more (11392 rows into fp8 38.0 us, this 37.1, the product
// alone 36.8, but 1 code in 2000 its neighbour).
__device__ __forceinline__ uint32_t pack_codes(const float* x, const Unit& u) {
  float y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float a = x[e] * u.up, q = fminf(fmaxf(a * u.inv, -512.f), 512.f);
    const float over = __builtin_fmaf(q, u.unit, -a), v = __builtin_fmaf(-over, u.inv, q);      // (of - 0 that is - 0)
    y[e] = is_number(x[e]) ? fminf(fmaxf(v, -448.f), 448.f) : __builtin_nanf("");
  }
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
}

// A wave's step is 64 / (D / 8) heads of one kind (queries, keys or values) of a row, eight elements a lane: four pairs of the rotation (4l to
// 4l + 3 and the same behind the head's middle, or 8l to 8l + 7), so that it needs no other lane, and a lane has the same four
// angles in every head.  A row's steps are shared by waves_per_row waves, which find the angles once each.  Norm and rotation
// are a product by the head's 1 / sqrt(mean) and one by (w1 cos, w2 sin, w2 cos, w1 sin), the same in every head.
//
// Bound by reading and writing the rows: 16384 rows of 32 + 2 x 8 heads of 128, 403 MB, in 80 us (5.0 TB/s, a copy's 5.2 to 5.4); without a norm,
// whose sums over lanes are not all hidden, in 69; interleaved, whose loads and stores of 8 bytes take turns in a line, in 103.  The same
// into fp8 with scales 370 MB in 81; 11392 rows of 28 + 2 x 4 heads into fp8, 199 MB, in 37.  One row 5.4 us, 64 rows of 64 + 2 x 8 heads with
// scales 7.2: a launch and its dependent reads.  11392 rows took 53 while angles were found four times over and products of norm and
// rotation made in every head; four steps at once with five waves a SIMD, and eight waves, which spill, were a tenth slower than two steps and six.
template <int D, int QT, int KIND, bool HALF, int PAST>
__global__ __launch_bounds__(kWriteThreads, 6) void write_paged_kernel(WriteLaunch a) {
  constexpr int LPH = D / 8, HPW = kWave / LPH;
  // elements of a head that are this lane's: first to first + 3 and first + apart to first + apart + 3
  constexpr int apart = HALF ? D / 2 : 4;
  const int lane = threadIdx.x % kWave, l = lane % LPH, sub = lane / LPH, first = HALF ? 4 * l : 8 * l;
  const int unit = blockIdx.x * kWriteWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int row = unit / a.waves_per_row, part = unit % a.waves_per_row, W = a.waves_per_row;
  if (row >= a.num_rows) return;
  const int q_steps = ceil_div(a.Hq, HPW), kv_steps = ceil_div(a.Hkv, HPW);
  // this wave's first step of each kind; the steps of a row are dealt out one behind the other
  const int q_from = part, k_from = (part - q_steps % W + W) % W, v_from = (part - (q_steps + kv_steps) % W + W) % W;

  // kStepsAtOnce steps from `from` on
  struct Source {
    GlobalBytes row;
    int64_t step;          // bytes from a step to the next
    uint32_t lane;         // of this lane
    int heads;
  };
  auto source = [&](const void* x, int64_t stride_row, int64_t stride_head, int heads) {
    return Source{(GlobalBytes)(uintptr_t)x + row * stride_row * 2, HPW * stride_head * 2, (uint32_t)(sub * (int)stride_head + first) * 2, heads};
  };
  auto load = [&](const Source& x, int from, u32x2 (&raw)[kStepsAtOnce][2]) {
#pragma unroll
    for (int u = 0; u < kStepsAtOnce; ++u) {
      const int s = from + u * W;
      raw[u][0] = raw[u][1] = u32x2{0, 0};
      if (s * HPW + sub < x.heads) {
        const GlobalBytes at = x.row + s * x.step;
        if constexpr (PAST != kCached) {
          raw[u][0] = __builtin_nontemporal_load((GlobalU2)(at + x.lane));
          raw[u][1] = __builtin_nontemporal_load((GlobalU2)(at + (x.lane + apart * 2)));
        } else {
          raw[u][0] = *(GlobalU2)(at + x.lane);
          raw[u][1] = *(GlobalU2)(at + (x.lane + apart * 2));
        }
      }
    }
  };
  const Source q = source(a.q, a.q_stride_row, a.q_stride_head, a.Hq), k = source(a.k, a.k_stride_row, a.k_stride_head, a.Hkv),
               v = source(a.v, a.v_stride_row, a.v_stride_head, a.Hkv);
  u32x2 now[kStepsAtOnce][2], next[kStepsAtOnce][2];
  load(q, q_from, now);

  auto load_norm = [&](const void* norm, float (&w)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = e < 4 ? first + e : first + apart + e - 4;
      w[e] = !norm ? 1.f : a.norm_fp32 ? reinterpret_cast<const float*>(norm)[d] : elem_lo<QT>(reinterpret_cast<const uint16_t*>(norm)[d]);
    }
  };
  float qw[8], kw[8], cs[4], sn[4];
  load_norm(a.q_norm, qw);
  load_norm(a.k_norm, kw);
  // the angles of all D / 2 frequencies, each found by one lane (two, of 256 dimensions), then handed to the lanes that use them
  {
    constexpr int own = D == 256 ? 2 : 1;
    float c[own], s[own];
#pragma unroll
    for (int i = 0; i < own; ++i) {
      const int f = (lane * own + i) % (D / 2);
      int axis = a.freq_axes ? a.freq_axes[f] : 0;
      if (axis < 0 || axis >= a.num_axes) axis = 0;
      const int64_t at = axis * a.position_stride + row;
      const double position = a.positions_64 ? (double)reinterpret_cast<const int64_t*>(a.positions)[at]
                                             : (double)reinterpret_cast<const int32_t*>(a.positions)[at];
      turn(position, a.inv_freq[f], a.rotary_scale, c[i], s[i]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      cs[e] = __shfl(c[e % own], (4 * l + e) / own);
      sn[e] = __shfl(s[e % own], (4 * l + e) / own);
    }
  }
  int b = row;
  if (a.row_starts) {
    b = __builtin_amdgcn_readfirstlane(sequence_of_row(a.row_starts, a.B, row, lane));
    if (b < 0) return;
  }

  float by[4][4];
  auto make_products = [&](const float (&w)[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float w1 = HALF ? w[e] : w[2 * e], w2 = HALF ? w[4 + e] : w[2 * e + 1];
      by[e][0] = w1 * cs[e];
      by[e][1] = w2 * sn[e];
      by[e][2] = w2 * cs[e];
      by[e][3] = w1 * sn[e];
    }
  };
  // four pairs of a head, normalised and rotated
  auto turned = [&](const u32x2 (&raw)[2], bool norm, float (&x)[8]) {
    float y[8] = {elem_lo<QT>(raw[0].x), elem_hi<QT>(raw[0].x), elem_lo<QT>(raw[0].y), elem_hi<QT>(raw[0].y),
                  elem_lo<QT>(raw[1].x), elem_hi<QT>(raw[1].x), elem_lo<QT>(raw[1].y), elem_hi<QT>(raw[1].y)};
    float inv = 1.f;
    if (norm) {
      float squares = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) squares += y[e] * y[e];
      inv = rsqrtf(sum_of_head<LPH>(squares) * (1.f / D) + a.eps);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = HALF ? e : 2 * e, j = HALF ? 4 + e : 2 * e + 1;
      // (the norm first: a product beyond 32 bits times nothing is no number)
      const float y1 = y[i] * inv, y2 = y[j] * inv;
      x[i] = y1 * by[e][0] - y2 * by[e][1];
      x[j] = y2 * by[e][2] + y1 * by[e][3];
    }
  };

  make_products(qw);
  {
    const uint32_t out_lane = (sub * (int)a.out_stride_head + first) * 2;
    const GlobalOut out = (GlobalOut)(uintptr_t)a.out + row * a.out_stride_row * 2;
    const int64_t out_step = HPW * a.out_stride_head * 2;
    for (int s0 = q_from; s0 < q_steps; s0 += kStepsAtOnce * W) {
      const bool more = s0 + kStepsAtOnce * W < q_steps;
      if (more) load(q, s0 + kStepsAtOnce * W, next);
#pragma unroll
      for (int u = 0; u < kStepsAtOnce; ++u) {
        const int s = s0 + u * W;
        if (s >= q_steps) break;
        float x[8];
        turned(now[u], a.q_norm != nullptr, x);
        if (s * HPW + sub < a.Hq) {
          const GlobalOut dst = out + s * out_step;
          const u32x2 low = {pack_half<QT>(x[0], x[1]), pack_half<QT>(x[2], x[3])}, high = {pack_half<QT>(x[4], x[5]), pack_half<QT>(x[6], x[7])};
          if constexpr (PAST == kAllPast) {
            __builtin_nontemporal_store(low, (GlobalOutU2)(dst + out_lane));
            __builtin_nontemporal_store(high, (GlobalOutU2)(dst + (out_lane + apart * 2)));
          } else {
            *(GlobalOutU2)(dst + out_lane) = low;
            *(GlobalOutU2)(dst + (out_lane + apart * 2)) = high;
          }
        }
      }
      if (more) {
#pragma unroll
        for (int u = 0; u < kStepsAtOnce; ++u) {
          now[u][0] = next[u][0];
          now[u][1] = next[u][1];
        }
      }
    }
  }

  if (k_from >= kv_steps && v_from >= kv_steps) return;
  const int t = __builtin_amdgcn_readfirstlane(token_of_row(a.row_starts, a.seq_lens, a.Tmax, b, row));
  if (t < 0) return;
  load(k, k_from, now);
  load(v, v_from, next);
  const int page = __builtin_amdgcn_readfirstlane(page_of_token(a.block_table, a.block_table_pitch, a.block_size, a.num_blocks, b, t));
  if (page < 0) return;
  const int off = t % a.block_size;
  const int64_t row_at = (page * a.stride_block + off * a.stride_token) * (KIND == kPlainRows ? 2 : 1);
  const int64_t beside = ((int64_t)page * a.block_size + off) * a.Hkv;
  const uint32_t cache_lane = (sub * (int)a.stride_head + first) * (KIND == kPlainRows ? 2 : 1);
  const int64_t cache_step = HPW * a.stride_head * (KIND == kPlainRows ? 2 : 1);
  // a step of K or V into the cache
  auto store = [&](int s, const float (&x)[8], GlobalOut rows, GlobalOutF32 scales, float scale) {
    const GlobalOut dst = rows + s * cache_step;
    if constexpr (KIND == kPlainRows) {
      if (s * HPW + sub >= a.Hkv) return;
      *(GlobalOutU2)(dst + cache_lane) = u32x2{pack_half<QT>(x[0], x[1]), pack_half<QT>(x[2], x[3])};
      *(GlobalOutU2)(dst + (cache_lane + apart * 2)) = u32x2{pack_half<QT>(x[4], x[5]), pack_half<QT>(x[6], x[7])};
    } else {
      if constexpr (KIND == kRowScales) {
        // of the finite elements: an infinity or NaN is a NaN in its place and leaves the others as they are
        float most = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) most = fmaxf(most, is_number(x[e]) ? fabsf(x[e]) : 0.f);
        scale = fmaxf(max_of_head<LPH>(most) / 448.f, FLT_MIN);
      }
      if (s * HPW + sub >= a.Hkv) return;
      const Unit unit(scale);
      *(GlobalOutU1)(dst + cache_lane) = pack_codes(x, unit);
      *(GlobalOutU1)(dst + (cache_lane + apart)) = pack_codes(x + 4, unit);
      if constexpr (KIND == kRowScales)
        if (l == 0) scales[s * HPW + sub] = scale;
    }
  };
  make_products(kw);
  {
    const GlobalOut rows = (GlobalOut)(uintptr_t)a.k_layers[a.layer] + row_at;
    const GlobalOutF32 scales = KIND == kRowScales ? (GlobalOutF32)(uintptr_t)a.k_scale_layers[a.layer] + beside : nullptr;
    for (int s0 = k_from; s0 < kv_steps; s0 += kStepsAtOnce * W) {
      if (s0 != k_from) load(k, s0, now);
#pragma unroll
      for (int u = 0; u < kStepsAtOnce; ++u) {
        const int s = s0 + u * W;
        if (s >= kv_steps) break;
        float x[8];
        turned(now[u], a.k_norm != nullptr, x);
        store(s, x, rows, scales, a.k_scale);
      }
    }
  }
  const GlobalOut rows = (GlobalOut)(uintptr_t)a.v_layers[a.layer] + row_at;
  const GlobalOutF32 scales = KIND == kRowScales ? (GlobalOutF32)(uintptr_t)a.v_scale_layers[a.layer] + beside : nullptr;
  for (int s0 = v_from; s0 < kv_steps; s0 += kStepsAtOnce * W) {
    if (s0 != v_from) load(v, s0, next);
#pragma unroll
    for (int u = 0; u < kStepsAtOnce; ++u) {
      const int s = s0 + u * W;
      if (s >= kv_steps) break;
      const u32x2 (&raw)[2] = next[u];
      if constexpr (KIND == kPlainRows) {
        if (s * HPW + sub >= a.Hkv) continue;
        const GlobalOut dst = rows + s * cache_step;
        *(GlobalOutU2)(dst + cache_lane) = raw[0];
        *(GlobalOutU2)(dst + (cache_lane + apart * 2)) = raw[1];
      } else {
        const float x[8] = {elem_lo<QT>(raw[0].x), elem_hi<QT>(raw[0].x), elem_lo<QT>(raw[0].y), elem_hi<QT>(raw[0].y),
                            elem_lo<QT>(raw[1].x), elem_hi<QT>(raw[1].x), elem_lo<QT>(raw[1].y), elem_hi<QT>(raw[1].y)};
        store(s, x, rows, scales, a.v_scale);
      }
    }
  }
}

// A wave takes rows_per_wave rows; their places are found a row a lane.  Lanes are pieces of a row's K and V alike (of several rows, where a
// row has fewer than 64) that make 16 bytes of the output, so that a wave's store is whole lines; stores go past the caches.  Bound by
// memory: 88798 rows of 8 x 128 fp8 with scales into bf16, 551 MB, in 102 us (5.4 TB/s, a copy's rate), 2176 rows of bf16 5.1.  (Lanes
// that read 16 bytes of fp8 and wrote twice 16: 132 us, past the caches 199; sixteen rows a wave 131, eight 110, four 106, two 103.)
constexpr int kRowsAtOnce = 2;

template <int WORDS>
__device__ __forceinline__ void load_words(GlobalBytes at, uint32_t (&x)[WORDS]) {
  if constexpr (WORDS == 4) {
    const u32x4 w = *(GlobalU4)at;
    x[0] = w.x; x[1] = w.y; x[2] = w.z; x[3] = w.w;
  } else if constexpr (WORDS == 2) {
    const u32x2 w = *(GlobalU2)at;
    x[0] = w.x; x[1] = w.y;
  } else {
    x[0] = *(const __attribute__((address_space(1))) uint32_t*)at;
  }
}

template <int CT, int OT>
__global__ __launch_bounds__(kWriteThreads) void read_paged_kernel(ReadLaunch a) {
  constexpr int EPL = OT == TRI_REAL_FP32 ? 4 : 8, ES = elem_size<CT>(), words = EPL * ES / 4;
  const int lane = threadIdx.x % kWave;
  const int64_t r0 = ((int64_t)blockIdx.x * kWriteWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave)) * a.rows_per_wave;
  if (r0 >= a.num_rows) return;
  const int rows = (int)min((int64_t)a.rows_per_wave, a.num_rows - r0);
  const GlobalBytes k = (GlobalBytes)(uintptr_t)a.k_layers[a.layer], v = (GlobalBytes)(uintptr_t)a.v_layers[a.layer];
  GlobalF32 ks = nullptr, vs = nullptr;
  if (a.k_scale_layers) {
    ks = (GlobalF32)(uintptr_t)a.k_scale_layers[a.layer];
    vs = (GlobalF32)(uintptr_t)a.v_scale_layers[a.layer];
  }
  // lane i has row i's place: a page, -1 for a row without a cached token (zeros), -2 for one that no sequence has
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
  const int shift = 31 - __clz(a.D / EPL), pieces = a.Hkv << shift;
  // lanes of a row: all 64, or the power of two that holds its pieces
  const int width = pieces >= kWave ? kWave : 1 << (32 - __clz(pieces - 1)), together = kWave / width, own = lane / width;
  for (int p0 = 0; p0 < pieces; p0 += width) {
    const int piece = p0 + lane % width, h = piece >> shift;
    const int64_t head_at = h * a.stride_head + (piece & ((1 << shift) - 1)) * EPL;
    for (int i0 = 0; i0 < rows; i0 += kRowsAtOnce * together) {
      uint32_t x[kRowsAtOnce][2][words];
      float scale[kRowsAtOnce][2];
      int pg[kRowsAtOnce];
#pragma unroll
      for (int u = 0; u < kRowsAtOnce; ++u) {
        const int r = i0 + u * together + own;
        const int o = __shfl(off, min(r, kWave - 1));
        pg[u] = __shfl(page, min(r, kWave - 1));
        if (r >= rows || piece >= pieces) pg[u] = -2;
#pragma unroll
        for (int i = 0; i < words; ++i) x[u][0][i] = x[u][1][i] = 0;
        scale[u][0] = scale[u][1] = 0.f;
        if (pg[u] >= 0) {
          const int64_t at = (pg[u] * a.stride_block + o * a.stride_token + head_at) * ES;
          load_words<words>(k + at, x[u][0]);
          load_words<words>(v + at, x[u][1]);
          if constexpr (CT == TRI_KV_FP8_E4M3)
            if (a.k_scale_layers) {
              const int64_t slot = ((int64_t)pg[u] * a.block_size + o) * a.Hkv + h;
              scale[u][0] = ks[slot];
              scale[u][1] = vs[slot];
            }
        }
      }
#pragma unroll
      for (int u = 0; u < kRowsAtOnce; ++u) {
        if (pg[u] == -2) continue;
        const int64_t to = ((r0 + i0 + u * together + own) * pieces + piece) * EPL;
#pragma unroll
        for (int side = 0; side < 2; ++side) {
          float f = side ? a.v_scale : a.k_scale;
          if constexpr (CT == TRI_KV_FP8_E4M3)
            if (a.k_scale_layers) f *= scale[u][side];
          float y[EPL];
#pragma unroll
          for (int i = 0; i < words; ++i) {
            const uint32_t word = x[u][side][i];
            if constexpr (CT == TRI_KV_FP8_E4M3) {
              y[4 * i] = fp8_byte<0>(word) * f;
              y[4 * i + 1] = fp8_byte<1>(word) * f;
              y[4 * i + 2] = fp8_byte<2>(word) * f;
              y[4 * i + 3] = fp8_byte<3>(word) * f;
            } else {
              y[2 * i] = elem_lo<CT>(word) * f;
              y[2 * i + 1] = elem_hi<CT>(word) * f;
            }
          }
          const GlobalOut out = (GlobalOut)(uintptr_t)(side ? a.v_out : a.k_out) + to * (OT == TRI_REAL_FP32 ? 4 : 2);
          if constexpr (OT == TRI_REAL_FP32)
            __builtin_nontemporal_store(u32x4{__float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]), __float_as_uint(y[3])}, (GlobalOutU4)out);
          else
            __builtin_nontemporal_store(u32x4{pack_half<OT>(y[0], y[1]), pack_half<OT>(y[2], y[3]), pack_half<OT>(y[4], y[5]), pack_half<OT>(y[6], y[7])}, (GlobalOutU4)out);
        }
      }
    }
  }
}

template <int D, int QT, bool HALF, int PAST>
void write_of_kind(const WriteLaunch& a, hipStream_t s) {
  const dim3 grid((unsigned)ceil_div64((int64_t)a.num_rows * a.waves_per_row, kWriteWaves));
  if (a.kv_dtype != TRI_KV_FP8_E4M3) hipLaunchKernelGGL((write_paged_kernel<D, QT, kPlainRows, HALF, PAST>), grid, dim3(kWriteThreads), 0, s, a);
  else if (!a.k_scale_layers) hipLaunchKernelGGL((write_paged_kernel<D, QT, kTensorScale, HALF, PAST>), grid, dim3(kWriteThreads), 0, s, a);
  else hipLaunchKernelGGL((write_paged_kernel<D, QT, kRowScales, HALF, PAST>), grid, dim3(kWriteThreads), 0, s, a);
}
template <int D, int QT, bool HALF>
void write_past(const WriteLaunch& a, PastCaches past, hipStream_t s) {
  if (past == kAllPast) write_of_kind<D, QT, HALF, kAllPast>(a, s);
  else if (past == kReadPast) write_of_kind<D, QT, HALF, kReadPast>(a, s);
  else write_of_kind<D, QT, HALF, kCached>(a, s);
}
template <int D, int QT>
void write_of_style(const WriteLaunch& a, PastCaches past, hipStream_t s) {
  if (a.rope_style == TRI_ROPE_HALF) write_past<D, QT, true>(a, past, s);
  else write_past<D, QT, false>(a, past, s);
}
template <int D>
void write_of_type(const WriteLaunch& a, PastCaches past, hipStream_t s) {
  if (a.q_dtype == TRI_KV_FP16) write_of_style<D, TRI_KV_FP16>(a, past, s);
  else write_of_style<D, TRI_KV_BF16>(a, past, s);
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
  // Waves a row: as many as make 2048 waves, down to a step each.  More waves of a row find its angles more often: rows of 32 + 2 x 8
  // heads of 128, calls aiming at 8192, 4096 and 2048 waves: 256 rows 6.1, 6.1, 6.2 us, 512 rows 8.9, 9.2, 7.2, 1024 rows 16.1, 11.4, 10.8,
  // 2048 rows 18.5, 13.8, 13.9.
  a.waves_per_row = (int)std::min<int64_t>(steps, std::max<int64_t>(1, 2048 / a.num_rows));
  // Many rows are read past the caches, which keep what is written; of even more rows the queries go past them too, and what is
  // cached stays.  Between a copy that writes q, k and v and an addition that reads the queries, the three together on three sets of rows in turn,
  // plain, reads past, both past, us: 42 MB of rows 47.6, 45.4, 46.3; 57 MB 59.4, 58.8, 58.6; 67 MB 71.5, 67.6, 68.0; 84 MB 88.3, 85.5, 84.1; 101 MB 103.5,
  // 100.8, 96.4; 135 MB 146, 130, 128; 201 MB 209, 199, 187; 403 MB 402, 406, 384.  Calls alone, inputs cold and outputs kept for one call: 42 MB 18.0, 21.3,
  // 21.2; 57 MB 28.2, 25.3, 26.0; 67 MB 33.7, 29.3, 30.5; 84 MB 45.0, 39.2, 41.3; 101 MB 49.0, 45.3, 43.8; 135 MB 62.8, 61.7, 56.8; 201 MB 89.0, 88.6, 79.0.
  const int64_t bytes = (int64_t)a.num_rows * (a.Hq + 2 * a.Hkv) * a.D * 2;
  const PastCaches past = bytes > (128ll << 20) ? kAllPast : bytes > (64ll << 20) ? kReadPast : kCached;
  if (a.D == 64) write_of_type<64>(a, past, s);
  else if (a.D == 128) write_of_type<128>(a, past, s);
  else write_of_type<256>(a, past, s);
  return hipGetLastError();
}

hipError_t launch_read_paged(ReadLaunch a, hipStream_t s) {
  const int pieces = a.Hkv * (a.D / (a.out_dtype == TRI_REAL_FP32 ? 4 : 8));
  int together = 1;
  while (together < kWave && 2 * together * pieces <= kWave) together *= 2;
  a.rows_per_wave = together * (a.num_rows >= 8192 * together ? kRowsAtOnce : 1);
  if (a.kv_dtype == TRI_KV_FP8_E4M3) read_to_type<TRI_KV_FP8_E4M3>(a, s);
  else if (a.kv_dtype == TRI_KV_FP16) read_to_type<TRI_KV_FP16>(a, s);
  else read_to_type<TRI_KV_BF16>(a, s);
  return hipGetLastError();
}

}  // namespace tri
