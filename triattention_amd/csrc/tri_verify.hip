// Verification of drafted tokens against the target's logits, and the move of the accepted ones' rows (gfx950).
//
//   w(x) = exp((l(x) - max l) / T),  E = sum w,  p = w / E             (probabilities as they come: w = p)
// Chain with draft probabilities q: row i + 1, drawn from q[i + 1] behind row i, is accepted iff u q(x) E < w(x) of row i; behind
// the last accepted row the next token is drawn from p, or where a row was rejected from max(p - q, 0) over its sum.  Without
// them (chain or tree): every row's token is drawn from p (T = 0: the first largest), and the walk goes on to the child that holds it.
// A draw is the least x whose running sum exceeds u times the whole.  Which token that is must not depend on the order of a sum:
// exponentials and sums are 64-bit, off by some 2^-46 of the whole, and of 2^17 boundaries between tokens one lies that
// near a random number once in 2^29 draws.
//
//  verify_sums_kernel  : every row's pieces of 2048 logits, a wave each: largest, where, and the sum of w against that
//  verify_walk_kernel  : (no draft probabilities) a workgroup per sequence: a wave draws a row's token, then the walk
//  verify_chain_kernel : (draft probabilities) which rows are accepted, and sums of max(p - q, 0) by pieces
//  verify_draw_kernel  : the token behind them
//  accept_rows_kernel  : rows of the accepted path to consecutive slots, every layer
#include <algorithm>
#include <cfloat>

#include "tri_common.h"
#include "tri_rows_device.h"

namespace tri {
namespace {

constexpr int kPieceSteps = kVerifyPiece / (kWave * 8);
constexpr int kVerifyThreads = 256;
constexpr int kVerifyWaves = kVerifyThreads / kWave;
constexpr int kWalkThreads = 1024;

// 2^y for y <= 0 (anything below -1100, and NaN, gives 0): y = n + f, the Taylor series of 2^f up to f^11 on [-1/2, 1/2], whose next
// term is 2^-47 of the result, and the exponent n.  Sixteen 64-bit instructions; the library's exponential has about twice that.
__device__ __forceinline__ double pow2_64(double y) {
  y = fmax(y, -1100.0);
  const double n = __builtin_rint(y), f = y - n;
  double p = 4.4455382718708113e-10;
  p = __builtin_fma(p, f, 7.0549116208011234e-09);
  p = __builtin_fma(p, f, 1.0178086009239700e-07);
  p = __builtin_fma(p, f, 1.3215486790144310e-06);
  p = __builtin_fma(p, f, 1.5252733804059841e-05);
  p = __builtin_fma(p, f, 1.5403530393381610e-04);
  p = __builtin_fma(p, f, 1.3333558146428443e-03);
  p = __builtin_fma(p, f, 9.6181291076284772e-03);
  p = __builtin_fma(p, f, 5.5504108664821580e-02);
  p = __builtin_fma(p, f, 2.4022650695910072e-01);
  p = __builtin_fma(p, f, 6.9314718055994531e-01);
  p = __builtin_fma(p, f, 1.0);
  return __builtin_ldexp(p, (int)n);
}

// w of a logit against `most`, c = log2 e / T.  Infinite logits share everything, -inf has nothing.
__device__ __forceinline__ double weight_of(float x, float most, double c) {
  if (most == INFINITY) return x == INFINITY ? 1.0 : 0.0;
  return x == -INFINITY ? 0.0 : pow2_64(((double)x - (double)most) * c);
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(1))) char* GlobalRows;
typedef __attribute__((address_space(1))) u32x4* GlobalPiece;
typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(2)));

// The number a logit or probability counts as.  NaN logits are -inf; probabilities that are no positive finite number are 0.
template <bool PROBS>
__device__ __forceinline__ float counted(float x) {
  if constexpr (PROBS) return x > 0.f && x <= FLT_MAX ? x : 0.f;
  else return x == x ? x : -INFINITY;
}
template <int RT, bool PROBS>
__device__ __forceinline__ float load_one(const void* row, int64_t i) {
  if constexpr (RT == TRI_REAL_FP32) return counted<PROBS>(reinterpret_cast<const float*>(row)[i]);
  else if constexpr (RT == TRI_REAL_FP16) return counted<PROBS>((float)reinterpret_cast<const _Float16*>(row)[i]);
  else return counted<PROBS>(__uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(row)[i] << 16));
}
// Eight of them from element i on (rows lie at any element); behind the row what counts as nothing.
template <int RT, bool PROBS>
__device__ __forceinline__ void load_eight(const void* row, int i, int V, float (&x)[8]) {
  if (i + 8 <= V) {
    if constexpr (RT == TRI_REAL_FP32) {
      const u32x4u* p = reinterpret_cast<const u32x4u*>(reinterpret_cast<const float*>(row) + i);
      const u32x4u a = p[0], b = p[1];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = __uint_as_float(a[e]);
        x[4 + e] = __uint_as_float(b[e]);
      }
    } else {
      const u32x4u a = *reinterpret_cast<const u32x4u*>(reinterpret_cast<const uint16_t*>(row) + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (RT == TRI_REAL_FP16) {
          x[2 * e] = (float)__builtin_bit_cast(_Float16, (unsigned short)(a[e] & 0xffffu));
          x[2 * e + 1] = (float)__builtin_bit_cast(_Float16, (unsigned short)(a[e] >> 16));
        } else {
          x[2 * e] = __uint_as_float(a[e] << 16);
          x[2 * e + 1] = __uint_as_float(a[e] & 0xffff0000u);
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = counted<PROBS>(x[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = i + e < V ? load_one<RT, PROBS>(row, i + e) : (PROBS ? 0.f : -INFINITY);
  }
}

__device__ __forceinline__ double shfl_double(double v, int lane) { return __shfl(v, lane); }
__device__ __forceinline__ double sum_of_wave(double v) {
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) v += __shfl_xor(v, d);
  return v;
}
// Inclusive running sum over the lanes.
__device__ __forceinline__ double running_sum(double v, int lane) {
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const double below = __shfl_up(v, d);
    if (lane >= d) v += below;
  }
  return v;
}

// The rows of sequence b that are looked at: n of them from `first` on.
__device__ __forceinline__ int rows_of_sequence(const VerifyLaunch& a, int b, int& first) {
  first = a.row_starts[b];
  const int end = min(a.row_starts[b + 1], a.num_rows);
  if (first < 0 || end <= first) return 0;
  return min(end - first, a.max_rows);
}
// log2 e / T; 0 where the sequence takes the largest (T not above 0).
__device__ __forceinline__ double sharpness_of(const VerifyLaunch& a, int b, bool& greedy) {
  const float t = a.temperatures ? a.temperatures[b] : 1.f;
  greedy = !(t > 0.f);
  return greedy ? 0.0 : 1.44269504088896340736 / (double)t;
}

template <int RT, bool PROBS>
__device__ __forceinline__ const void* row_of(const VerifyLaunch& a, int row) {
  return reinterpret_cast<const char*>(a.target) + row * a.target_stride * (RT == TRI_REAL_FP32 ? 4 : 2);
}

template <int RT, bool PROBS>
__global__ __launch_bounds__(kVerifyThreads) void verify_sums_kernel(VerifyLaunch a) {
  const int lane = threadIdx.x % kWave;
  const int64_t unit = (int64_t)blockIdx.x * kVerifyWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int row = (int)(unit / a.pieces), piece = (int)(unit % a.pieces);
  if (row >= a.num_rows) return;
  const void* const src = row_of<RT, PROBS>(a, row);
  float x[kPieceSteps][8];
#pragma unroll
  for (int s = 0; s < kPieceSteps; ++s) {
    const int64_t i = (int64_t)piece * kVerifyPiece + s * kWave * 8 + lane * 8;
    load_eight<RT, PROBS>(src, (int)min(i, (int64_t)a.vocab), a.vocab, x[s]);
  }
  const int b = sequence_of_row(a.row_starts, a.B, row, lane);
  if (b < 0 || row - a.row_starts[b] >= a.max_rows) return;
  bool greedy;
  const double c = sharpness_of(a, b, greedy);
  float most = -INFINITY;
#pragma unroll
  for (int s = 0; s < kPieceSteps; ++s)
#pragma unroll
    for (int e = 0; e < 8; ++e) most = fmaxf(most, x[s][e]);
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) most = fmaxf(most, __shfl_xor(most, d));
  int where = INT32_MAX;
#pragma unroll
  for (int s = kPieceSteps - 1; s >= 0; --s)
#pragma unroll
    for (int e = 7; e >= 0; --e)
      if (x[s][e] == most) where = s * kWave * 8 + lane * 8 + e;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) where = min(where, __shfl_xor(where, d));
  double sum = 0.0;
  if constexpr (PROBS) {
#pragma unroll
    for (int s = 0; s < kPieceSteps; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += (double)x[s][e];
    sum = sum_of_wave(sum);
  } else if (!greedy && most > -INFINITY) {
#pragma unroll
    for (int s = 0; s < kPieceSteps; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += weight_of(x[s][e], most, c);
    sum = sum_of_wave(sum);
  }
  if (lane == 0) a.part[unit] = VerifyPart{sum, most, piece * kVerifyPiece + where};
}

// A row's largest number, the first place that holds it (-1: every number is -inf) and the sum of its weights.
struct RowTotal {
  double sum;
  float most;
  int where;
};

// The sum of a piece's weights against the row's largest number.
template <bool PROBS>
__device__ __forceinline__ double against(const VerifyPart& p, float most, double c) {
  if constexpr (PROBS) return p.sum;
  else return p.sum == 0.0 ? 0.0 : p.sum * weight_of(p.most, most, c);
}

template <bool PROBS>
__device__ __forceinline__ RowTotal total_of_row(const VerifyLaunch& a, int row, double c, int lane) {
  const VerifyPart* part = a.part + (int64_t)row * a.pieces;
  RowTotal t{0.0, -INFINITY, INT32_MAX};
  for (int i = lane; i < a.pieces; i += kWave)
    if (part[i].most > t.most) {
      t.most = part[i].most;
      t.where = part[i].where;
    }
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const float m = __shfl_xor(t.most, d);
    const int w = __shfl_xor(t.where, d);
    if (m > t.most || (m == t.most && w < t.where)) {
      t.most = m;
      t.where = w;
    }
  }
  if (t.most == -INFINITY) t.where = -1;
  for (int i = lane; i < a.pieces; i += kWave) t.sum += against<PROBS>(part[i], t.most, c);
  t.sum = sum_of_wave(t.sum);
  return t;
}

// The least place whose running sum exceeds u of the whole; piece_sum(i) is piece i's sum, weights(i, w) its eight weights from element i
// on.  A wave's work: the pieces' sums tell the piece, whose weights are found anew.  Where rounding leaves nothing above the
// mark, and for u >= 1, the last place of any weight; -1 if there is none.
template <class PieceSum, class Weights>
__device__ __forceinline__ int draw(const VerifyLaunch& a, double whole, float u, int lane, PieceSum piece_sum, Weights weights) {
  const double mark = (u > 0.f ? (double)u : 0.0) * whole;
  double before = 0.0, start = 0.0;
  int piece = -1, last = -1;
  for (int i0 = 0; i0 < a.pieces && piece < 0; i0 += kWave) {
    const double v = i0 + lane < a.pieces ? piece_sum(i0 + lane) : 0.0;
    const double upto = before + running_sum(v, lane);
    const uint64_t some = __ballot(v > 0.0), over = __ballot(v > 0.0 && upto > mark);
    if (over) {
      const int at = __ffsll((unsigned long long)over) - 1;
      piece = i0 + at;
      start = at ? shfl_double(upto, at - 1) : before;
    } else if (some) {
      last = i0 + 63 - __clzll((long long)some);
    }
    before = shfl_double(upto, kWave - 1);
  }
  const bool found = piece >= 0;
  if (!found) {
    piece = last;
    if (piece < 0) return -1;
  }
  int best = -1;
  for (int s = 0; s < kPieceSteps; ++s) {
    const int i = piece * kVerifyPiece + s * kWave * 8 + lane * 8;
    double w[8], sum = 0.0;
    weights(i, w);
    int final = -1;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      sum += w[e];
      if (w[e] > 0.0) final = i + e;
    }
    const double upto = running_sum(sum, lane);
    if (found) {
      double running = start + (upto - sum);
      int mine = -1;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        running += w[e];
        if (mine < 0 && w[e] > 0.0 && running > mark) mine = i + e;
      }
      const uint64_t over = __ballot(mine >= 0);
      if (over) return __shfl(mine, __ffsll((unsigned long long)over) - 1);
    }
    const uint64_t some = __ballot(final >= 0);
    if (some) best = __shfl(final, 63 - __clzll((long long)some));
    start += shfl_double(upto, kWave - 1);
  }
  return best;
}

// A token drawn from a row's weights.
template <int RT, bool PROBS>
__device__ __forceinline__ int draw_from_row(const VerifyLaunch& a, int row, const RowTotal& t, double c, float u, int lane) {
  const void* const src = row_of<RT, PROBS>(a, row);
  const VerifyPart* part = a.part + (int64_t)row * a.pieces;
  return draw(a, t.sum, u, lane, [&](int i) { return against<PROBS>(part[i], t.most, c); },
              [&](int i, double (&w)[8]) {
                float x[8];
                load_eight<RT, PROBS>(src, min(i, a.vocab), a.vocab, x);
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] = PROBS ? (double)x[e] : weight_of(x[e], t.most, c);
              });
}

__device__ __forceinline__ void write_path(const VerifyLaunch& a, int b, int lane, int row, int count, int next) {
  for (int i = lane; i < a.max_rows; i += kWave) a.rows_out[(int64_t)b * a.max_rows + i] = i < count ? row : -1;
  if (lane == 0) {
    a.counts[b] = count;
    a.next[b] = next;
  }
}

template <int RT, bool PROBS>
__global__ __launch_bounds__(kWalkThreads) void verify_walk_kernel(VerifyLaunch a) {
  __shared__ int picked[64];
  const int b = blockIdx.x, lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  int first;
  const int n = rows_of_sequence(a, b, first);
  bool greedy;
  const double c = sharpness_of(a, b, greedy);
  for (int i = wave; i < n; i += kWalkThreads / kWave) {
    const RowTotal t = total_of_row<PROBS>(a, first + i, c, lane);
    const int token = greedy ? t.where : draw_from_row<RT, PROBS>(a, first + i, t, c, a.uniforms[2 * (int64_t)(first + i) + 1], lane);
    if (lane == 0) picked[i] = token;
  }
  __syncthreads();
  if (wave) return;
  // lane i is row i
  int parent = -1, token = -1;
  if (lane < n && lane > 0) {
    parent = a.parents ? a.parents[first + lane] : lane - 1;
    if (parent < 0 || parent >= lane) parent = -1;
    token = a.tokens[first + lane];
  }
  int here = 0, count = n > 0 ? 1 : 0, path = 0;
  while (n > 0) {
    const int want = picked[here];
    const uint64_t child = __ballot(parent == here && token == want && want >= 0);
    if (!child) break;
    here = __ffsll((unsigned long long)child) - 1;
    if (lane == count) path = here;
    ++count;
  }
  write_path(a, b, lane, path, count, n > 0 ? picked[here] : -1);
}

template <int RT, bool PROBS>
__global__ __launch_bounds__(kVerifyThreads) void verify_chain_kernel(VerifyLaunch a, int groups) {
  __shared__ RowTotal totals[64];
  __shared__ int fits[64];
  const int b = blockIdx.x / groups, group = blockIdx.x % groups;
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  int first;
  const int n = rows_of_sequence(a, b, first);
  bool greedy;
  const double c = sharpness_of(a, b, greedy);
  for (int i = wave; i < n; i += kVerifyWaves) {
    const RowTotal t = total_of_row<PROBS>(a, first + i, c, lane);
    if (lane == 0) {
      totals[i] = t;
      if (i + 1 < n) {
        const int64_t next = first + i + 1;
        const int token = a.tokens[next];
        bool ok = false;
        if (greedy) {
          ok = t.where >= 0 && token == t.where;
        } else if (token >= 0 && token < a.vocab) {
          const float x = load_one<RT, PROBS>(row_of<RT, PROBS>(a, first + i), token);
          const double w = PROBS ? (double)x : weight_of(x, t.most, c);
          const float q = counted<true>(a.draft[next * a.draft_stride + token]), u = a.uniforms[2 * next];
          ok = (u > 0.f ? (double)u : 0.0) * (double)q * t.sum < w;
        }
        fits[i + 1] = ok;
      }
    }
  }
  __syncthreads();
  const uint64_t refused = __ballot(lane > 0 && lane < n && !fits[lane]);
  const int count = refused ? __ffsll((unsigned long long)refused) - 1 : n;
  const RowTotal t = n > 0 ? totals[count - 1] : RowTotal{0.0, -INFINITY, -1};
  const bool rest = refused && !greedy && t.sum > 0.0;
  if (group == 0 && threadIdx.x == 0) a.state[b] = VerifyState{t.sum, t.most, t.where, count, rest};
  const int piece = group * kVerifyWaves + wave;
  if (!rest || piece >= a.pieces) return;
  const void* const src = row_of<RT, PROBS>(a, first + count - 1);
  const float* const q = a.draft + (int64_t)(first + count) * a.draft_stride;
  double sum = 0.0;
#pragma unroll
  for (int s = 0; s < kPieceSteps; ++s) {
    const int i = (int)min((int64_t)piece * kVerifyPiece + s * kWave * 8 + lane * 8, (int64_t)a.vocab);
    float x[8], y[8];
    load_eight<RT, PROBS>(src, i, a.vocab, x);
    load_eight<TRI_REAL_FP32, true>(q, i, a.vocab, y);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const double w = PROBS ? (double)x[e] : weight_of(x[e], t.most, c);
      sum += fmax(w / t.sum - (double)y[e], 0.0);
    }
  }
  sum = sum_of_wave(sum);
  if (lane == 0) a.rest[(int64_t)b * a.pieces + piece] = sum;
}

template <int RT, bool PROBS>
__global__ __launch_bounds__(kWave) void verify_draw_kernel(VerifyLaunch a) {
  const int b = blockIdx.x, lane = threadIdx.x;
  int first;
  const int n = rows_of_sequence(a, b, first);
  if (n == 0) return write_path(a, b, lane, 0, 0, -1);
  bool greedy;
  const double c = sharpness_of(a, b, greedy);
  const VerifyState st = a.state[b];
  const int row = first + st.count - 1;
  const RowTotal t{st.sum, st.most, st.where};
  const float u = a.uniforms[2 * (int64_t)row + 1];
  int token = t.where;
  if (!greedy) {
    double whole = 0.0;
    const double* const rest = a.rest + (int64_t)b * a.pieces;
    if (st.rest) {
      for (int i = lane; i < a.pieces; i += kWave) whole += rest[i];
      whole = sum_of_wave(whole);
    }
    if (whole > 0.0) {
      const void* const src = row_of<RT, PROBS>(a, row);
      const float* const q = a.draft + (int64_t)(row + 1) * a.draft_stride;
      token = draw(a, whole, u, lane, [&](int i) { return rest[i]; },
                   [&](int i, double (&w)[8]) {
                     float x[8], y[8];
                     load_eight<RT, PROBS>(src, min(i, a.vocab), a.vocab, x);
                     load_eight<TRI_REAL_FP32, true>(q, min(i, a.vocab), a.vocab, y);
#pragma unroll
                     for (int e = 0; e < 8; ++e)
                       w[e] = fmax((PROBS ? (double)x[e] : weight_of(x[e], t.most, c)) / t.sum - (double)y[e], 0.0);
                   });
    } else {
      token = draw_from_row<RT, PROBS>(a, row, t, c, u, lane);
    }
  }
  write_path(a, b, lane, lane, st.count, token);
}

// Rows [first new token + rows[j]] to [first new token + j], j = 1 .. count - 1, of one side of one layer.  Lists ascend, so rows[j] >= j:
// a thread has one place of every row, and what it writes lies before all that it still reads.
constexpr int kAcceptAtOnce = 8;
__global__ __launch_bounds__(kVerifyThreads) void accept_rows_kernel(AcceptLaunch a) {
  __shared__ int64_t from_row[64], to_row[64];           // elements of the cache
  __shared__ int64_t from_slot[64], to_slot[64];         // slots, for what lies beside it
  const int b = blockIdx.x / (2 * a.L), l = blockIdx.x / 2 % a.L, side = blockIdx.x % 2, lane = threadIdx.x % kWave;
  const int first = a.row_starts[b], n = max(a.row_starts[b + 1] - first, 0);
  const int T = min(max(a.seq_lens[b], 0), a.Tmax), base = T - n;
  const int asked = min(min(max(a.counts[b], 0), n), a.max_rows);
  // (every wave for itself) lane j has the path's row j; a list that does not ascend within the sequence's rows ends there
  const int r = lane < asked ? a.rows[(int64_t)b * a.max_rows + lane] : -1;
  const int below = __shfl_up(r, 1);
  const uint64_t bad = __ballot(lane >= asked || r < 0 || r >= n || (lane > 0 && r <= below));
  const int count = bad ? __ffsll((unsigned long long)bad) - 1 : 64;
  if (l == 0 && side == 0 && threadIdx.x == 0 && a.lens_out) a.lens_out[b] = max(base + count, 0);
  int from = -1, to = -1;
  if (lane < count && r != lane && base + lane >= 0) {
    from = page_of_token(a.block_table, a.block_table_pitch, a.block_size, a.num_blocks, b, base + r);
    to = page_of_token(a.block_table, a.block_table_pitch, a.block_size, a.num_blocks, b, base + lane);
  }
  const uint64_t moves = __ballot(from >= 0 && to >= 0);
  const int m = __popcll(moves);
  if (m == 0) return;
  if (threadIdx.x < kWave && (moves >> lane & 1)) {
    const int at = __popcll(moves & ((1ull << lane) - 1));
    const int from_off = (base + r) % a.block_size, to_off = (base + lane) % a.block_size;
    from_row[at] = from * a.stride_block + from_off * a.stride_token;
    to_row[at] = to * a.stride_block + to_off * a.stride_token;
    from_slot[at] = (int64_t)from * a.block_size + from_off;
    to_slot[at] = (int64_t)to * a.block_size + to_off;
  }
  __syncthreads();
  const GlobalRows cache = (GlobalRows)(uintptr_t)(side ? a.v_layers : a.k_layers)[l];
  const int lanes = a.D * a.elem_bytes / 16, pieces = a.Hkv * lanes;
  for (int p = threadIdx.x; p < pieces; p += kVerifyThreads) {
    const int h = p / lanes;
    const int64_t at = (int64_t)h * a.stride_head * a.elem_bytes + (p - h * lanes) * 16;
    for (int j0 = 0; j0 < m; j0 += kAcceptAtOnce) {
      u32x4 x[kAcceptAtOnce];
#pragma unroll
      for (int u = 0; u < kAcceptAtOnce; ++u)
        x[u] = *(GlobalPiece)(cache + from_row[min(j0 + u, m - 1)] * a.elem_bytes + at);
#pragma unroll
      for (int u = 0; u < kAcceptAtOnce; ++u)
        if (j0 + u < m) *(GlobalPiece)(cache + to_row[j0 + u] * a.elem_bytes + at) = x[u];
    }
  }
  // numbers beside the rows: an fp8 row's scale, a token's weight
  float* const scales = a.v_scale_layers ? (side ? a.v_scale_layers : a.k_scale_layers)[l] : nullptr;
  float* const weights = a.weights && side ? a.weights + l * a.weights_stride_layer : nullptr;
  for (int p = threadIdx.x; p < 2 * a.Hkv; p += kVerifyThreads) {
    const int h = p % a.Hkv;
    float* const x = p < a.Hkv ? scales : weights;
    if (!x) continue;
    for (int j0 = 0; j0 < m; j0 += kAcceptAtOnce) {
      float v[kAcceptAtOnce];
#pragma unroll
      for (int u = 0; u < kAcceptAtOnce; ++u) v[u] = x[from_slot[min(j0 + u, m - 1)] * a.Hkv + h];
#pragma unroll
      for (int u = 0; u < kAcceptAtOnce; ++u)
        if (j0 + u < m) x[to_slot[j0 + u] * a.Hkv + h] = v[u];
    }
  }
}

template <int RT, bool PROBS>
hipError_t verify_of(const VerifyLaunch& a, hipStream_t s) {
  if (a.num_rows > 0)
    hipLaunchKernelGGL((verify_sums_kernel<RT, PROBS>), dim3((unsigned)ceil_div64((int64_t)a.num_rows * a.pieces, kVerifyWaves)),
                       dim3(kVerifyThreads), 0, s, a);
  if (!a.draft) {
    hipLaunchKernelGGL((verify_walk_kernel<RT, PROBS>), dim3(a.B), dim3(kWalkThreads), 0, s, a);
  } else {
    const int groups = ceil_div(a.pieces, kVerifyWaves);
    hipLaunchKernelGGL((verify_chain_kernel<RT, PROBS>), dim3((unsigned)(a.B * groups)), dim3(kVerifyThreads), 0, s, a, groups);
    hipLaunchKernelGGL((verify_draw_kernel<RT, PROBS>), dim3(a.B), dim3(kWave), 0, s, a);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_verify_drafts(const VerifyLaunch& a, hipStream_t s) {
  if (a.probs) return verify_of<TRI_REAL_FP32, true>(a, s);
  if (a.target_dtype == TRI_REAL_FP32) return verify_of<TRI_REAL_FP32, false>(a, s);
  if (a.target_dtype == TRI_REAL_FP16) return verify_of<TRI_REAL_FP16, false>(a, s);
  return verify_of<TRI_REAL_BF16, false>(a, s);
}

hipError_t launch_accept_rows(const AcceptLaunch& a, hipStream_t s) {
  hipLaunchKernelGGL(accept_rows_kernel, dim3((unsigned)(a.B * a.L * 2)), dim3(kVerifyThreads), 0, s, a);
  return hipGetLastError();
}

}  // namespace tri
