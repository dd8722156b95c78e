// Attention of a few query rows per sequence over the paged cache (gfx950): one decoding step, a tree of drafted
// tokens, or the blocks of a list.  Instantiated per head dimension in tri_attend_{64,128,256}.hip.
//
//   s[m][t] = scale * q[m] . k[t]   where row m sees token t, else -inf
//   out[m]  = sum_t 2^(s log2 e - M) v[t] / sum_t 2^(s log2 e - M),   M the running maximum
//
// Rows: a sequence has n new tokens, the last n of its cache; KV head h serves the M = n * G rows (token i, query head
// h * G + g), m = i * G + g.  Row m sees every token before the new ones, and of those token i and its ancestors.
//
// A wave takes 32 tokens at a time and RT tiles of 16 rows.  S^T = K Q^T on the matrix cores (16 tokens x 16 rows x 32
// elements) leaves in a lane the scores of one row (lane & 15) for tokens (lane >> 4) * 4 + r of either half: exactly
// the order in which the B operand of O^T = V^T P^T wants them, if the 32 tokens are numbered (lane >> 4) * 8 + j =
// token (j & 4) * 4 + (lane >> 4) * 4 + (j & 3).  So the weights never leave their lane, a row's maximum is two
// exchanges between lanes, and the rescaling of O is a multiplication inside a lane.  V^T comes out of LDS by the
// transposing read (16 lanes, 4 tokens x 16 elements).  The four waves of a workgroup take tiles in turn and meet once
// at the end; a sequence is cut into splits where there are few rows, joined by attend_join_kernel.
#pragma once

#include "tri_common.h"
#include "tri_mma_device.h"
#include "tri_score_device.h"

namespace tri {
namespace {

constexpr int kAttendThreads = 256;
constexpr int kAttendWaves = kAttendThreads / kWave;
constexpr int kAttendTile = 32;       // tokens a wave takes at a time

template <int T>
struct Half;                          // the type of the products
template <>
struct Half<TRI_KV_BF16> {
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    bf16x2 v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, v);
  }
  static __device__ __forceinline__ uint32_t widen_lo(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.0f, false));
  }
  static __device__ __forceinline__ uint32_t widen_hi(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.0f, true));
  }
  static __device__ __forceinline__ float value(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }
};
template <>
struct Half<TRI_KV_FP16> {
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    f16x2 v = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, v);
  }
  static __device__ __forceinline__ uint32_t widen_lo(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, false));
  }
  static __device__ __forceinline__ uint32_t widen_hi(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, true));
  }
  static __device__ __forceinline__ float value(uint16_t x) { return (float)__builtin_bit_cast(_Float16, x); }
};

// Eight fp8 codes (two dwords) as eight 16-bit numbers; exact in either type.
template <int T>
__device__ __forceinline__ uint4 widen8(uint32_t a, uint32_t b) {
  return uint4{Half<T>::widen_lo(a), Half<T>::widen_hi(a), Half<T>::widen_lo(b), Half<T>::widen_hi(b)};
}

// Whether a packed pair of 16-bit numbers holds an infinity or a NaN (all exponent bits set).
template <int T>
__device__ __forceinline__ bool not_finite2(uint32_t w) {
  constexpr uint32_t e = T == TRI_KV_FP16 ? 0x7c00u : 0x7f80u;
  return (w & e) == e || (w >> 16 & e) == e;
}

typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4* LdsI16x4;

// The transposing read: each 16 lanes read a piece of 4 rows (4 lanes of 8 bytes each, lane / 4 the row) x 16 columns
// and lane c receives column c, rows 0 to 3.
typedef __attribute__((address_space(3))) unsigned char* LdsBytes;
__device__ __forceinline__ uint2 lds_read_transposed(LdsBytes at) {
  const i16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsI16x4)at);
  return __builtin_bit_cast(uint2, v);
}

// Two 2^(x) terms of one sum: -inf - -inf is a row without tokens on either side, and a factor of 0.
__device__ __forceinline__ float rescale(float m, float top) { return m == -INFINITY ? 0.f : exp2f(m - top); }

__device__ __forceinline__ int64_t shfl64(int64_t v, int lane) {
  const int lo = __shfl((int)(uint32_t)v, lane), hi = __shfl((int)(v >> 32), lane);
  return (int64_t)(((uint64_t)(uint32_t)hi << 32) | (uint32_t)lo);
}

// Ancestors and self of new token `lane` (bit j: token j), by pointer doubling: after step k the word covers 2^k
// generations and p is the 2^k-th ancestor.  A parent outside [0, lane) hangs the token on the cache.
__device__ __forceinline__ uint64_t ancestor_mask(const int32_t* parents, int first, int n, int lane) {
  int p = -1;
  if (lane < n) p = parents ? parents[first + lane] : lane - 1;
  if (p >= lane || p < 0) p = -1;
  uint64_t m = 1ull << lane;
#pragma unroll
  for (int step = 0; step < 6; ++step) {
    const int src = p < 0 ? lane : p;
    const uint64_t up = (uint64_t)shfl64((int64_t)m, src);
    const int next = __shfl(p, src);
    if (p >= 0) {
      m |= up;
      p = next;
    }
  }
  return m;
}

struct RowRange {
  int first, n;      // first row of the sequence and their number
};
__device__ __forceinline__ RowRange rows_of(const AttendLaunch& a, int b) {
  if (!a.row_starts) return {b, 1};
  int first = a.row_starts[b], end = a.row_starts[b + 1];
  first = min(max(first, 0), a.num_rows);
  end = min(max(end, first), a.num_rows);
  return {first, min(end - first, a.max_rows)};
}

// Tokens the call reads of a sequence, in the order it reads them: its cache, or the blocks of its list one after the other.
__device__ __forceinline__ int tokens_of(const AttendLaunch& a, int b, int T) {
  if (!a.list) return T;
  return min(a.list_k, ceil_div(T, a.block_size)) * a.block_size;
}

template <int QT, bool FP8, int D, int RT>
__global__ __launch_bounds__(kAttendThreads) void attend_kernel(AttendLaunch a) {
  constexpr int PT = FP8 ? TRI_KV_BF16 : QT;              // fp8 rows with a scale of their own: the weight carries it, which fp16 has no room for
  constexpr int ES = FP8 ? 1 : 2;
  constexpr int KC = D * ES / 64;                         // 16-byte pieces of a key in a lane
  constexpr int LPR = D * ES / 16;                        // lanes that load one value row
  constexpr int NV = LPR / 2;                             // 16-byte pieces of a tile's values in a lane
  constexpr int NT = D / 16;
  constexpr int kPitch = D * 2 + 32;                      // bytes of a value row in LDS: eight rows reach all banks
  constexpr int kWaveBytes = kAttendTile * kPitch;
  __shared__ __align__(16) unsigned char s_v[kAttendWaves * kWaveBytes];
  __shared__ __align__(16) float s_scale[kAttendWaves][2][kAttendTile];
  __shared__ float s_ml[kAttendWaves][RT * 16][2];

  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int c16 = lane & 15, q4 = lane >> 4;
  int idx = blockIdx.x;
  const int h = idx % a.Hkv; idx /= a.Hkv;
  const int rb = idx % a.row_blocks; idx /= a.row_blocks;
  const int split = idx % a.nsplit;
  const int b = idx / a.nsplit;

  const int T = min(max(a.seq_lens[b], 0), a.Tmax);
  const RowRange rows = rows_of(a, b);
  const int n = rows.n, M = n * a.G, m0 = rb * RT * 16;
  if (m0 >= M) return;
  const int Tv = tokens_of(a, b, T);
  const int begin = split * a.split_tokens, end = min(begin + a.split_tokens, Tv);
  if (begin >= Tv && split > 0) return;
  const int base = T - n;                                 // first new token (negative: not all of them are in the cache)
  const int32_t* table = a.block_table ? a.block_table + (int64_t)b * a.block_table_pitch : nullptr;
  const int32_t* list = a.list ? a.list + ((int64_t)b * a.Hkv + h) * a.list_pitch : nullptr;
  const char* kb = reinterpret_cast<const char*>(a.k_layers[a.layer]) + (int64_t)h * a.stride_head * ES;
  const char* vb = reinterpret_cast<const char*>(a.v_layers[a.layer]) + (int64_t)h * a.stride_head * ES;
  const float* ksc = a.k_scale_layers ? a.k_scale_layers[a.layer] + h : nullptr;
  const float* vsc = a.v_scale_layers ? a.v_scale_layers[a.layer] + h : nullptr;

  // Queries: lane = row c16 of a tile, elements as the keys are loaded (fp8: 16 in a piece, two steps of 8).
  uint4 qf[RT][D / 32];
  uint64_t seen[RT];
  const uint64_t anc = n > 1 ? ancestor_mask(a.parents, rows.first, n, lane) : 1ull;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int m = m0 + rt * 16 + c16;
    const int i = m < M ? m / a.G : 0, g = m < M ? m % a.G : 0;
    seen[rt] = (uint64_t)shfl64((int64_t)anc, i);
    const char* qp = reinterpret_cast<const char*>(a.q) + ((int64_t)(rows.first + i) * a.q_stride_row + (int64_t)(h * a.G + g) * a.q_stride_head) * 2;
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
      const int el = FP8 ? (s / 2) * 64 + q4 * 16 + (s & 1) * 8 : s * 32 + q4 * 8;
      qf[rt][s] = m < M ? *reinterpret_cast<const uint4*>(qp + el * 2) : uint4{0, 0, 0, 0};
    }
  }

  f32x4 o[RT][NT];
  float top[RT], sum[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    top[rt] = -INFINITY;
    sum[rt] = 0.f;
#pragma unroll
    for (int t = 0; t < NT; ++t) o[rt][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // Lane l holds the place of token l & 31 of a tile: list entry, then page, then byte offset, each asked for a tile
  // ahead of the next (a wait for a young load would be a wait for every older one).
  const int mine = lane & (kAttendTile - 1);
  const int first_tile = begin + wave * kAttendTile;
  constexpr int kStep = kAttendWaves * kAttendTile;
  auto list_entry = [&](int tile) {
    const int t = tile + mine;
    return list && t < end ? list[t / a.block_size] : 0;
  };
  auto token_at = [&](int tile, int entry) {     // position in the sequence, or -1
    const int t = tile + mine;
    const int tok = list ? entry * a.block_size + t % a.block_size : t;
    return t < end && entry >= 0 && tok < T ? tok : -1;
  };
  auto page_of = [&](int tok) {
    if (tok < 0) return -1;
    return table ? table[tok / a.block_size] : b;
  };
  struct Place {
    int64_t byte, row;     // offset of the row, index of its scale
    bool ok;
  };
  auto place_of = [&](int tok, int page) {
    Place p;
    p.ok = tok >= 0 && page >= 0 && page < a.num_blocks;
    const int in = p.ok ? tok % a.block_size : 0;
    const int64_t pg = p.ok ? page : 0;
    p.byte = (pg * a.stride_block + (int64_t)in * a.stride_token) * ES;
    p.row = (pg * a.block_size + in) * a.Hkv;
    return p;
  };

  uint4 kr[2][KC], vr[NV];
  float ks_mine = 1.f, vs_mine = 1.f;
  auto load_keys = [&](const Place& p) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const char* src = kb + shfl64(p.byte, i * 16 + c16) + q4 * 16;
#pragma unroll
      for (int c = 0; c < KC; ++c) kr[i][c] = *reinterpret_cast<const uint4*>(src + c * 64);
    }
    if (FP8 && vsc) {
      ks_mine = ksc[p.row];
      vs_mine = vsc[p.row];
    }
  };
  auto load_values = [&](const Place& p) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      vr[i] = *reinterpret_cast<const uint4*>(vb + shfl64(p.byte, i * (kWave / LPR) + lane / LPR) + (lane % LPR) * 16);
  };

  unsigned char* const my_v = s_v + wave * kWaveBytes;
  const LdsBytes my_lds = (LdsBytes)my_v;
  Place now{}, next{};
  int next_tok = -1, next_page = -1, next2_entry = 0;
  if (first_tile < end) {
    const int t0 = token_at(first_tile, list_entry(first_tile));
    next_tok = token_at(first_tile + kStep, list_entry(first_tile + kStep));
    next_page = page_of(next_tok);
    next2_entry = list_entry(first_tile + 2 * kStep);
    now = place_of(t0, page_of(t0));
    load_keys(now);
    load_values(now);
  }
  for (int tile = first_tile; tile < end; tile += kStep) {
    const bool more = tile + kStep < end;
    const uint32_t okm = (uint32_t)__ballot(now.ok);
    const bool drafts = n > 1 && tile + kAttendTile > base;

    // ---- scores
    f32x4 sc[RT][2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) sc[rt][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < D / 32; ++s) {
        uint4 kf;
        if constexpr (FP8) {
          const uint4& w = kr[i][s / 2];
          kf = (s & 1) ? widen8<QT>(w.z, w.w) : widen8<QT>(w.x, w.y);
        } else {
          kf = kr[i][s];
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) sc[rt][i] = mfma_16x16x32<QT>(kf, qf[rt][s], sc[rt][i]);
      }
    }
    if (FP8 && vsc && lane < kAttendTile) {
      s_scale[wave][0][lane] = ks_mine;
      s_scale[wave][1][lane] = vs_mine;
    }
    // ---- the next tile's keys into the registers of this one's, this one's values into LDS
    if (more) {
      next = place_of(next_tok, next_page);
      next_tok = token_at(tile + 2 * kStep, next2_entry);
      next_page = page_of(next_tok);
      next2_entry = list_entry(tile + 3 * kStep);
      load_keys(next);
    }
    bool odd_values = false;                    // an infinity or a NaN among the values of new tokens
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int row = i * (kWave / LPR) + lane / LPR;
      uint4 w[2] = {vr[i], uint4{0, 0, 0, 0}};
      if constexpr (FP8) {
        w[0] = widen8<PT>(vr[i].x, vr[i].y);
        w[1] = widen8<PT>(vr[i].z, vr[i].w);
      }
      if (okm != 0xffffffffu && !(okm >> row & 1)) w[0] = w[1] = uint4{0, 0, 0, 0};      // 0 * what lies behind the end could be NaN
      if (drafts) {
#pragma unroll
        for (int j = 0; j < (FP8 ? 2 : 1); ++j)
          odd_values |= not_finite2<PT>(w[j].x) || not_finite2<PT>(w[j].y) || not_finite2<PT>(w[j].z) || not_finite2<PT>(w[j].w);
      }
      uint4* dst = reinterpret_cast<uint4*>(my_v + row * kPitch + (lane % LPR) * (FP8 ? 32 : 16));
      dst[0] = w[0];
      if (FP8) dst[1] = w[1];
    }
    if (more) load_values(next);

    // ---- softmax: a lane holds tokens i * 16 + q4 * 4 + r of row c16
    const bool masked = okm != 0xffffffffu || drafts;
    float ks[2][4], vs[2][4];
    if (FP8 && vsc) {
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          ks[i][r] = s_scale[wave][0][i * 16 + q4 * 4 + r] * a.scale_log2;
          vs[i][r] = s_scale[wave][1][i * 16 + q4 * 4 + r];
        }
    }
    uint4 pf[RT];
    float p[RT][2][4];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float best = -INFINITY;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float x = sc[rt][i][r] * (FP8 && vsc ? ks[i][r] : a.scale_log2);
          if (masked) {
            const int j = i * 16 + q4 * 4 + r;
            const int d = tile + j - base;
            const bool sees = (okm >> j & 1) && (!drafts || d < 0 || (seen[rt] >> (d & 63) & 1));
            x = sees ? x : -INFINITY;
          }
          sc[rt][i][r] = x;
          best = fmaxf(best, x);
        }
      if (a.scores) {
        const int m = m0 + rt * 16 + c16;
        if (m < M) {
          float* dst = a.scores + (((int64_t)b * a.Hkv + h) * a.max_rows * a.G + m) * a.score_pitch + tile + q4 * 4;
          *reinterpret_cast<f32x4*>(dst) = sc[rt][0];
          *reinterpret_cast<f32x4*>(dst + 16) = sc[rt][1];
        }
      }
      best = fmaxf(best, __shfl_xor(best, 16));
      best = fmaxf(best, __shfl_xor(best, 32));
      const float now_top = fmaxf(top[rt], best);
      const float safe = now_top == -INFINITY ? 0.f : now_top;
      const float alpha = rescale(top[rt], safe);
      top[rt] = now_top;
      float part = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          p[rt][i][r] = exp2f(sc[rt][i][r] - safe);
          part += p[rt][i][r];
        }
      sum[rt] = sum[rt] * alpha + part;
      if (__ballot(alpha != 1.f)) {
#pragma unroll
        for (int t = 0; t < NT; ++t) o[rt][t] *= alpha;
      }
      if (FP8 && vsc) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) p[rt][i][r] *= vs[i][r];
      }
      // The weights are rounded to 16 bits for the second product (the sum above adds them unrounded): errors of half
      // a step each and of either sign, below the one rounding of the output.
      pf[rt] = uint4{Half<PT>::pack(p[rt][0][0], p[rt][0][1]), Half<PT>::pack(p[rt][0][2], p[rt][0][3]),
                     Half<PT>::pack(p[rt][1][0], p[rt][1][1]), Half<PT>::pack(p[rt][1][2], p[rt][1][3])};
    }
    // ---- O^T += V^T P^T
    if (!__ballot(odd_values)) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const LdsBytes at = my_lds + (q4 * 4 + (c16 >> 2)) * kPitch + t * 32 + (c16 & 3) * 8;
        const uint2 lo = lds_read_transposed(at), hi = lds_read_transposed(at + 16 * kPitch);
        const uint4 vf{lo.x, lo.y, hi.x, hi.y};
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) o[rt][t] = mfma_16x16x32<PT>(vf, pf[rt], o[rt][t]);
      }
    } else {
      // An infinity or a NaN in a new token's values reaches the rows that see the token and no others (0 * inf would
      // put it into all of them): token by token on the vector unit.
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            for (int qq = 0; qq < 4; ++qq) {
              const int j = i * 16 + qq * 4 + r, d = tile + j - base;
              const float w = __shfl(p[rt][i][r], qq * 16 + c16);
              const bool sees = (okm >> j & 1) && (d < 0 || (seen[rt] >> (d & 63) & 1));
              const uint16_t* row = reinterpret_cast<const uint16_t*>(my_v + j * kPitch);
#pragma unroll
              for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float v = Half<PT>::value(row[t * 16 + q4 * 4 + e]);
                  if (sees) o[rt][t][e] += w * v;
                }
            }
    }
    __builtin_amdgcn_wave_barrier();
    now = next;
  }

  // ---- the four waves meet
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    sum[rt] += __shfl_xor(sum[rt], 16);
    sum[rt] += __shfl_xor(sum[rt], 32);
    if (q4 == 0) {
      s_ml[wave][rt * 16 + c16][0] = top[rt];
      s_ml[wave][rt * 16 + c16][1] = sum[rt];
    }
  }
  __syncthreads();
  f32x4* const box = reinterpret_cast<f32x4*>(s_v);       // [wave][NT][64]: 4 * D / 16 * 1 KB, no more than the value tiles
  static_assert(kAttendWaves * NT * kWave * 16 <= kAttendWaves * kWaveBytes, "the exchange fits the value tiles");
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    float all = -INFINITY;
#pragma unroll
    for (int w = 0; w < kAttendWaves; ++w) all = fmaxf(all, s_ml[w][rt * 16 + c16][0]);
    const float mine_f = rescale(top[rt], all);
#pragma unroll
    for (int t = 0; t < NT; ++t) box[(wave * NT + t) * kWave + lane] = o[rt][t] * mine_f;
    __syncthreads();
    for (int it = threadIdx.x; it < NT * kWave; it += kAttendThreads) {
      const int t = it / kWave, l = it % kWave, row = rt * 16 + (l & 15), m = m0 + row;
      if (m >= M) continue;
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
      float total = 0.f, big = -INFINITY;
#pragma unroll
      for (int w = 0; w < kAttendWaves; ++w) big = fmaxf(big, s_ml[w][row][0]);
#pragma unroll
      for (int w = 0; w < kAttendWaves; ++w) {
        v += box[(w * NT + t) * kWave + l];
        total += rescale(s_ml[w][row][0], big) * s_ml[w][row][1];
      }
      const int d = t * 16 + (l >> 4) * 4;
      if (a.nsplit > 1) {
        const int64_t at = (((int64_t)b * a.Hkv + h) * a.nsplit + split) * a.max_rows * a.G + m;
        *reinterpret_cast<f32x4*>(a.part_out + at * D + d) = v;
        if (d == 0) {
          a.part_ml[at * 2] = big;
          a.part_ml[at * 2 + 1] = total;
        }
      } else {
        const int64_t i = rows.first + m / a.G;
        const int hq = h * a.G + m % a.G;
        // (a row that saw nothing: zeros and -inf)
        const float inv = total == 0.f ? 0.f : a.v_scale / total;
        uint16_t* dst = reinterpret_cast<uint16_t*>(a.out) + i * a.out_stride_row + (int64_t)hq * a.out_stride_head + d;
        *reinterpret_cast<uint2*>(dst) = uint2{Half<QT>::pack(v[0] * inv, v[1] * inv), Half<QT>::pack(v[2] * inv, v[3] * inv)};
        if (d == 0) {
          const float l2 = total == 0.f ? -INFINITY : big + log2f(total);
          if (a.lse) a.lse[i * a.Hq + hq] = l2 * 0.69314718055994530942f;
          if (a.lse2) a.lse2[i * a.Hq + hq] = l2;
        }
      }
    }
    __syncthreads();
  }
}

// Row tiles of an instance: as many as the rows of a KV head need, up to what the registers hold.
template <int QT, bool FP8, int D>
hipError_t launch_attend_typed(const AttendLaunch& a, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)a.B * a.nsplit * a.row_blocks * a.Hkv));
  if (a.row_tiles == 1) hipLaunchKernelGGL((attend_kernel<QT, FP8, D, 1>), grid, dim3(kAttendThreads), 0, s, a);
  else if (a.row_tiles == 2) hipLaunchKernelGGL((attend_kernel<QT, FP8, D, 2>), grid, dim3(kAttendThreads), 0, s, a);
  else if constexpr (D <= 128) {
    if (a.row_tiles != 4) return hipErrorInvalidValue;
    hipLaunchKernelGGL((attend_kernel<QT, FP8, D, 4>), grid, dim3(kAttendThreads), 0, s, a);
  } else return hipErrorInvalidValue;
  return hipGetLastError();
}

template <int D>
hipError_t launch_attend_dim(const AttendLaunch& a, hipStream_t s) {
  const bool fp8 = a.kv_dtype == TRI_KV_FP8_E4M3;
  if (a.q_dtype == TRI_KV_BF16) return fp8 ? launch_attend_typed<TRI_KV_BF16, true, D>(a, s) : launch_attend_typed<TRI_KV_BF16, false, D>(a, s);
  return fp8 ? launch_attend_typed<TRI_KV_FP16, true, D>(a, s) : launch_attend_typed<TRI_KV_FP16, false, D>(a, s);
}

}  // namespace
}  // namespace tri
