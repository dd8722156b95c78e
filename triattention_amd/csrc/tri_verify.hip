// Verification of drafted tokens against the target's logits, and the move of the accepted ones' rows (gfx950).
//
//   w(x) = exp((l(x) - max l) / T),  E = sum w,  p = w / E             (probabilities as they come: w = p)
// Chain with draft probabilities q: row i + 1, drawn from q[i + 1] behind row i, is accepted iff u q(x) E < w(x) of row i; behind
// the last accepted row the next token is drawn from p, or where a row was rejected from max(w - q E, 0) over its sum.  Without
// them (chain or tree): every row's token is drawn from p (T = 0: the first largest), and the walk goes on to the child that holds it.
// A draw is the least x whose running sum exceeds u times the whole.  Which token that is must not depend on the order of a sum:
// exponentials and sums are 64-bit, off by some 2^-44 of the whole, and of 2^17 boundaries between tokens one lies that
// near a random number once in 2^26 draws.
//
//  verify_sums_kernel  : every row's pieces of 2048 logits, a wave each: largest, where, and the sum of w against that
//  verify_walk_kernel  : (no draft probabilities) a wave draws a row's token, a sequence's last workgroup walks
//  verify_chain_kernel : (draft probabilities) which rows are accepted, sums of max(w - q E, 0) by pieces; the last workgroup draws
//  accept_rows_kernel  : rows of the accepted path to consecutive slots, every layer
//
// Two launches a call.  A third, for what the last workgroup of a sequence does, took 4 us more of the host and 3 of the GPU; one launch for
// all of it would need counters cleared before it.  One chain of six rows of 32768 logits 4.4 + 7.0 us, 60 greedy rows of 131072
// 5.8 + 4.4: launches and dependent reads; the host behind them takes 14.
#include <algorithm>
#include <cfloat>

#include "tri_common.h"
#include "tri_rows_device.h"

namespace tri {
namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kPieceSteps = kVerifyPiece / (kWave * 8);
constexpr int kVerifyThreads = 256;
constexpr int kVerifyWaves = kVerifyThreads / kWave;
constexpr int kChainThreads = 512;
constexpr int kChainWaves = kChainThreads / kWave;

// 2^(c d) of numbers d <= 0 times c >= 2^-200, never less than about 2^-1000 (which NaN gives too): c d = n + j / 256 + f, rounded by an addition; 2^f on
// [-1/512, 1/512] by 1 and f times the Chebyshev interpolation of degree 2 (off by 2^-44.7 of it), 2^(j/256) out of LDS, n into the exponent:
// ten vector instructions and an LDS read.  262 rows of 131072 logits, the sums' kernel as it then was: a Taylor series of degree 11 on
// [-1/2, 1/2] 43 us, the interpolation of degree 9 with scalar coefficients 32, degree 4 and a table of 32 numbers 27; that table's whole
// call at its best 39.5, this one's 37.  Lanes meet in the banks of 256 numbers and not in those of 32, but a place among 256 is the low
// byte of the units and needs no mask, and a product is saved.  The coefficients are kept from being constants that the compiler copies
// into vector registers before every step: they are the products' scalar operand.
constexpr double kLeastPower = -1000.0;
constexpr int kTable = 256;
static_assert(kVerifyThreads >= kTable && kChainThreads >= kTable, "a thread makes a number of the table");
struct Powers {
  const double* table;      // 2^(j/256) with j << 12 taken off its high word: what the units of 1/256, shifted as far, add to it is n alone
  double per, least;
  double c[3];
  __device__ __forceinline__ Powers(const double* in_lds, double per_number)
      : table(in_lds), per(per_number), least(kLeastPower * __builtin_amdgcn_rcp(per_number)) {
    const double exact[3] = {0.6931471805599453, 0.24022653447679007, 0.05550411247958329};
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      c[i] = exact[i];
      asm("" : "+s"(c[i]));
    }
  }
  // Factors of eight of them, one in [2^-1/512, 2^1/512]: the table's words are all asked for before the first is used.
  __device__ __forceinline__ void factors(double (&d)[8], double (&power)[8]) const {
    constexpr double kUnits = 26388279066624.0;      // 1.5 * 2^44: a sum's low bits are units of 1/256
    uint32_t units[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      d[e] = fmax(d[e], least);
      const double shifted = __builtin_fma(d[e], per, kUnits);
      units[e] = (uint32_t)__builtin_bit_cast(uint64_t, shifted);
      power[e] = table[units[e] % kTable];
      d[e] = __builtin_fma(d[e], per, kUnits - shifted);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const double p = __builtin_fma(__builtin_fma(c[2], d[e], c[1]), d[e], c[0]);
      d[e] = __builtin_fma(p, d[e], 1.0);
      u32x2 words = __builtin_bit_cast(u32x2, power[e]);
      words.y += units[e] << 12;
      power[e] = __builtin_bit_cast(double, words);
    }
  }
  __device__ __forceinline__ void operator()(double (&d)[8]) const {
    double power[8];
    factors(d, power);
#pragma unroll
    for (int e = 0; e < 8; ++e) d[e] *= power[e];
  }
  // added to two sums
  __device__ __forceinline__ void add(double (&d)[8], double (&sums)[2]) const {
    double power[8];
    factors(d, power);
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[e % 2] = __builtin_fma(d[e], power[e], sums[e % 2]);
  }
  __device__ __forceinline__ double operator()(double d) const {
    double eight[8] = {d, 0, 0, 0, 0, 0, 0, 0};
    (*this)(eight);
    return eight[0];
  }
};
// 2^(j/32) and 2^(j/256), whose products the table holds.
__device__ const double kCoarse[32] = {
    1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237,
    1.0905077326652577, 1.1143867425958924, 1.1387886347566916, 1.1637248587775775,
    1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332,
    1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832,
    1.4142135623730951, 1.4451808069770467, 1.4768261459394993, 1.5091644275934228,
    1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.645755478153965,
    1.681792830507429, 1.718619298122478, 1.7562521603732995, 1.7947090750031072,
    1.8340080864093424, 1.8741676341103, 1.9152065613971474, 1.9571441241754002};
__device__ const double kFine[8] = {1.0, 1.0027112750502025, 1.0054299011128027, 1.0081558981184175,
                                   1.0108892860517005, 1.0136300849514894, 1.016378314910953, 1.019133996077738};
// A thread's word of the table is asked for before all else and put into LDS where it has come (the counter of a wave's loads goes in
// their order: a load behind those of a piece would be waited for with them).
__device__ __forceinline__ double own_power() { return kCoarse[threadIdx.x / 8 % 32] * kFine[threadIdx.x % 8]; }
__device__ __forceinline__ void keep_power(double* table, double own) {
  u32x2 words = __builtin_bit_cast(u32x2, own);
  words.y -= threadIdx.x % kTable << 12;
  if (threadIdx.x < kTable) table[threadIdx.x] = __builtin_bit_cast(double, words);
}

// A sharpness from which on infinities, which count as the largest finite number, leave nothing to any other: the next one of 32 bits is 2^104 less.
constexpr double kAlone = 0x1p-94;
// What weighs no more than this beside the largest (-inf, NaN, and numbers that far below it) has nothing.
constexpr double kNothing = 0x1p-900;
// w of logits against the largest one; of what has nothing 2^-1000 at least.
__device__ __forceinline__ void weights_of(const Powers& powers, const float (&x)[8], double most, double (&w)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = (double)x[e] - most;
  powers(w);
}
__device__ __forceinline__ double weight_of(const Powers& powers, float x, double most) {
  const double w = powers((double)x - most);
  return w > kNothing ? w : 0.0;
}

typedef __attribute__((address_space(1))) char* GlobalRows;
typedef __attribute__((address_space(1))) u32x4* GlobalPiece;
typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(2)));

// The number a logit or probability counts as.  Logits: NaN as -inf, +inf as the largest finite number, so that infinities share
// everything.  Probabilities that are no positive finite number: 0.  Raw logits are taken as they are.
enum Numbers { kRawLogits = 0, kLogits = 1, kProbs = 2 };
template <int N>
__device__ __forceinline__ float counted(float x) {
  if constexpr (N == kProbs) return x <= FLT_MAX ? fmaxf(x, 0.f) : 0.f;
  else if constexpr (N == kLogits) return x == x ? fminf(x, FLT_MAX) : -INFINITY;
  else return x;
}
template <int RT, int N>
__device__ __forceinline__ float load_one(const void* row, int64_t i) {
  if constexpr (RT == TRI_REAL_FP32) return counted<N>(reinterpret_cast<const float*>(row)[i]);
  else if constexpr (RT == TRI_REAL_FP16) return counted<N>((float)reinterpret_cast<const _Float16*>(row)[i]);
  else return counted<N>(__uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(row)[i] << 16));
}
// Eight of them from element i on as they lie (rows begin at any element); behind the row what counts as nothing.
template <int RT>
struct Eight {
  uint32_t word[RT == TRI_REAL_FP32 ? 8 : 4];
};
template <int RT, int N>
__device__ __forceinline__ Eight<RT> load_eight(const void* row, int i, int V) {
  Eight<RT> x;
  if (i + 8 <= V) {
    const u32x4u* p = reinterpret_cast<const u32x4u*>(reinterpret_cast<const char*>(row) + (int64_t)i * (RT == TRI_REAL_FP32 ? 4 : 2));
#pragma unroll
    for (int e = 0; e < (RT == TRI_REAL_FP32 ? 8 : 4); ++e) x.word[e] = p[e / 4][e % 4];
    return x;
  }
  if constexpr (RT == TRI_REAL_FP32) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x.word[e] = i + e < V ? reinterpret_cast<const uint32_t*>(row)[i + e] : N == kProbs ? 0u : 0xff800000u;
  } else {
    const uint32_t nothing = N == kProbs ? 0u : RT == TRI_REAL_FP16 ? 0xfc00u : 0xff80u;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const uint32_t lo = i + e < V ? reinterpret_cast<const uint16_t*>(row)[i + e] : nothing;
      const uint32_t hi = i + e + 1 < V ? reinterpret_cast<const uint16_t*>(row)[i + e + 1] : nothing;
      x.word[e / 2] = lo | hi << 16;
    }
  }
  return x;
}
struct Numbers8 {
  float x[8];
};
template <int RT, int N>
__device__ __forceinline__ Numbers8 numbers_of(const Eight<RT>& eight) {
  Numbers8 n;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float x;
    if constexpr (RT == TRI_REAL_FP32) x = __uint_as_float(eight.word[e]);
    else if constexpr (RT == TRI_REAL_FP16) x = (float)__builtin_bit_cast(_Float16, (unsigned short)(eight.word[e / 2] >> e % 2 * 16));
    else x = __uint_as_float(e % 2 ? eight.word[e / 2] & 0xffff0000u : eight.word[e / 2] << 16);
    n.x[e] = counted<N>(x);
  }
  return n;
}
// A piece as a wave has it: step s is 512 numbers, eight a lane.
template <int RT>
struct Piece {
  Eight<RT> step[kPieceSteps];
};
template <int RT, int N>
__device__ __forceinline__ Piece<RT> load_piece(const VerifyLaunch& a, const void* row, int piece, int lane) {
  Piece<RT> x;
#pragma unroll
  for (int s = 0; s < kPieceSteps; ++s)
    x.step[s] = load_eight<RT, N>(row, (int)min((int64_t)piece * kVerifyPiece + s * kWave * 8 + lane * 8, (int64_t)a.vocab), a.vocab);
  return x;
}

// Exchanges inside a wave without LDS: every 16 lanes by their row's permutations, the four rows by broadcasts or scalar registers.
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ double moved(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xf, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xf, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double lane_of(double v, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, lane), hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double sum_of_wave(double v) {
  v += moved<0xB1>(v);        // quad_perm [1, 0, 3, 2]
  v += moved<0x4E>(v);        // quad_perm [2, 3, 0, 1]
  v += moved<0x141>(v);       // row_half_mirror
  v += moved<0x128>(v);       // row_ror:8
  return (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
}
template <int CTRL>
__device__ __forceinline__ int moved_int(int v) { return __builtin_amdgcn_update_dpp(v, v, CTRL, 0xf, 0xf, false); }
__device__ __forceinline__ float most_of_wave(float v) {
  v = fmaxf(v, __int_as_float(moved_int<0xB1>(__float_as_int(v))));
  v = fmaxf(v, __int_as_float(moved_int<0x4E>(__float_as_int(v))));
  v = fmaxf(v, __int_as_float(moved_int<0x141>(__float_as_int(v))));
  v = fmaxf(v, __int_as_float(moved_int<0x128>(__float_as_int(v))));
  const auto of = [&](int lane) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane)); };
  return fmaxf(fmaxf(of(0), of(16)), fmaxf(of(32), of(48)));
}
__device__ __forceinline__ int least_of_wave(int v) {
  v = min(v, moved_int<0xB1>(v));
  v = min(v, moved_int<0x4E>(v));
  v = min(v, moved_int<0x141>(v));
  v = min(v, moved_int<0x128>(v));
  const auto of = [&](int lane) { return __builtin_amdgcn_readlane(v, lane); };
  return min(min(of(0), of(16)), min(of(32), of(48)));
}
// Inclusive running sum over the lanes: within rows of 16 by shifts, then each row's last lane into the rows behind it.
__device__ __forceinline__ double running_sum(double v) {
  v += moved<0x111>(v);
  v += moved<0x112>(v);
  v += moved<0x114>(v);
  v += moved<0x118>(v);
  v += moved<0x142, 0xa>(v);  // row_bcast:15 into rows 1 and 3
  v += moved<0x143, 0xc>(v);  // row_bcast:31 into rows 2 and 3
  return v;
}

// The rows of sequence b that are looked at: n of them from `first` on.
__device__ __forceinline__ int rows_of_sequence(const VerifyLaunch& a, int b, int& first) {
  first = a.row_starts[b];
  const int end = min(a.row_starts[b + 1], a.num_rows);
  if (first < 0 || end <= first) return 0;
  return min(end - first, a.max_rows);
}
// log2 e / T (of an infinite T so little that all finite logits weigh the same); 0 where the sequence takes the largest (T not above 0).
__device__ __forceinline__ double sharpness(float temperature, bool& greedy) {
  greedy = !(temperature > 0.f);
  return greedy ? 0.0 : fmax(1.44269504088896340736 / (double)temperature, 0x1p-200);
}
__device__ __forceinline__ double sharpness_of(const VerifyLaunch& a, int b, bool& greedy) {
  return sharpness(a.temperatures ? a.temperatures[b] : 1.f, greedy);
}

template <int RT, bool PROBS>
__device__ __forceinline__ const void* row_of(const VerifyLaunch& a, int row) {
  return reinterpret_cast<const char*>(a.target) + row * a.target_stride * (RT == TRI_REAL_FP32 ? 4 : 2);
}

// A wave's 2048 numbers of a row.  Sampled rows want the sum, greedy ones the place of the largest.  Bound by vector instructions
// (16 a logit, most of them 64-bit) where rows fill the chip: 262 rows of 131072 bf16 logits, 69 MB, in 21.1 us, 83 % of whose cycles those
// take; 161 rows of 100003 fp32 ones, 64 MB, in 16.4 and 55 %, one round of waves that wait for their loads and then compute.  Pieces of fewer numbers, loads past
// the caches, two halves of 16 bytes side by side for fp32 and a shorter form for rows whose numbers lie near each other gained nothing; weights
// against the first step's largest number, while the other steps' loads are on their way, 1 us of the second and lost half of one in the first.
template <int RT, bool PROBS>
__global__ __launch_bounds__(kVerifyThreads) void verify_sums_kernel(VerifyLaunch a) {
  __shared__ double table[kTable];
  const int lane = threadIdx.x % kWave;
  for (int64_t i = (int64_t)blockIdx.x * kVerifyThreads + threadIdx.x; i < a.B; i += (int64_t)gridDim.x * kVerifyThreads) a.arrived[i] = 0;
  // (scalar numbers, and less than 2^26: a launch's threads are less than 2^32)
  const int unit = (int)blockIdx.x * kVerifyWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int row = __builtin_amdgcn_readfirstlane(unit / a.pieces), piece = unit - row * a.pieces;
  constexpr int N = PROBS ? kProbs : kRawLogits;
  // what is needed to know the row's temperature comes before the piece: of up to 64 sequences all of it at once
  const double power = own_power();
  const int mine = min(lane, a.B - 1);
  const int32_t start = a.row_starts[mine], end = a.row_starts[mine + 1];
  const float temperature = a.temperatures ? a.temperatures[mine] : 1.f;
  Piece<RT> held;
  if (row < a.num_rows) held = load_piece<RT, N>(a, row_of<RT, PROBS>(a, row), piece, lane);
  keep_power(table, power);
  __syncthreads();
  if (row >= a.num_rows) return;
  bool greedy;
  double c;
  if (a.B <= kWave) {
    const uint64_t own = __ballot(lane < a.B && start <= row && row < end && row - start < a.max_rows);
    if (!own) return;
    c = sharpness(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(temperature), __ffsll((unsigned long long)own) - 1)), greedy);
  } else {
    const int b = __builtin_amdgcn_readfirstlane(sequence_of_row(a.row_starts, a.B, row, lane));
    if (b < 0 || row - a.row_starts[b] >= a.max_rows) return;
    c = sharpness_of(a, b, greedy);
  }
  float most = -INFINITY;
#pragma unroll
  for (int s = 0; s < kPieceSteps; ++s) {
    const Numbers8 n = numbers_of<RT, N>(held.step[s]);
#pragma unroll
    for (int e = 0; e < 8; ++e) most = __builtin_elementwise_maximum(most, n.x[e]);
  }
  // NaN, which that hands on, count as -inf (fmaxf is no way past them: behind a signalling one it has lost what was before)
  if (!PROBS && __ballot(most != most)) {
    most = -INFINITY;
#pragma unroll
    for (int s = 0; s < kPieceSteps; ++s) {
      const Numbers8 n = numbers_of<RT, N>(held.step[s]);
#pragma unroll
      for (int e = 0; e < 8; ++e) most = n.x[e] > most ? n.x[e] : most;
    }
  }
  most = most_of_wave(most);
  const float top = PROBS ? most : fminf(most, FLT_MAX);      // (infinities are the largest finite number)
  double sum = 0.0;
  int where = 0;
  if (greedy) {
    where = INT32_MAX;
#pragma unroll
    for (int s = kPieceSteps - 1; s >= 0; --s) {
      const Numbers8 n = numbers_of<RT, N>(held.step[s]);
#pragma unroll
      for (int e = 7; e >= 0; --e)
        if (n.x[e] >= top) where = s * kWave * 8 + lane * 8 + e;
    }
    where = most > -INFINITY ? least_of_wave(where) : 0;
  } else if (PROBS || (most == INFINITY && c >= kAlone)) {
    // (beside infinities all else weighs nothing)
#pragma unroll
    for (int s = 0; s < kPieceSteps; ++s) {
      const Numbers8 n = numbers_of<RT, N>(held.step[s]);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += PROBS ? (double)n.x[e] : n.x[e] >= top ? 1.0 : 0.0;
    }
    sum = sum_of_wave(sum);
  } else if (most == INFINITY) {
    // (a temperature of 1e28 or more; one number at a time, so that the loop below keeps its registers)
    const Powers powers(table, c);
    const int end = min(kVerifyPiece, a.vocab - piece * kVerifyPiece);
#pragma unroll 1
    for (int i = lane; i < end; i += kWave)
      sum += powers((double)load_one<RT, kLogits>(row_of<RT, PROBS>(a, row), (int64_t)piece * kVerifyPiece + i) - (double)top);
    sum = sum_of_wave(sum);
  } else if (most > -INFINITY) {
    // (what weighs less than 2^-1000 counts as that here: the largest weighs 1)
    const Powers powers(table, c);
    const double largest = most;
    double sums[2] = {0.0, 0.0};
#pragma unroll
    for (int s = 0; s < kPieceSteps; ++s) {
      const Numbers8 n = numbers_of<RT, N>(held.step[s]);
      double d[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = (double)n.x[e] - largest;
      powers.add(d, sums);
    }
    sum = sums[0] + sums[1];
    sum = sum_of_wave(sum);
  }
  if (lane == 0) a.part[unit] = VerifyPart{sum, top, piece * kVerifyPiece + where};
}

template <bool PROBS>
__device__ __forceinline__ void weights_or_probs(const Powers& powers, const Numbers8& n, float most, double (&w)[8]) {
  if constexpr (PROBS) {
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = n.x[e];
  } else {
    weights_of(powers, n.x, most, w);
  }
}

// A row's largest number, the first place that holds it (-1: every number is -inf) and the sum of its weights.
struct RowTotal {
  double sum;
  float most;
  int where;
};

// The sum of a piece's weights against the row's largest number.
template <bool PROBS>
__device__ __forceinline__ double against(const Powers& powers, const VerifyPart& p, float most) {
  if constexpr (PROBS) return p.sum;
  else return p.sum == 0.0 ? 0.0 : p.sum * weight_of(powers, p.most, most);
}

__device__ __forceinline__ VerifyPart first_part(const VerifyLaunch& a, int row, int lane) {
  return lane < a.pieces ? a.part[(int64_t)row * a.pieces + lane] : VerifyPart{0.0, -INFINITY, INT32_MAX};
}
// (a row of up to 2^17 numbers: one piece a lane, `mine`)
template <bool PROBS>
__device__ __forceinline__ RowTotal total_of_row(const VerifyLaunch& a, const Powers& powers, int row, const VerifyPart& mine, int lane) {
  const VerifyPart* part = a.part + (int64_t)row * a.pieces;
  RowTotal t{0.0, -INFINITY, INT32_MAX};
  t.most = mine.most;
  t.where = mine.where;
  for (int i = lane + kWave; i < a.pieces; i += kWave)
    if (part[i].most > t.most) {
      t.most = part[i].most;
      t.where = part[i].where;
    }
  const float most = most_of_wave(t.most);
  t.where = least_of_wave(t.most == most ? t.where : INT32_MAX);
  t.most = most;
  if (t.most == -INFINITY) t.where = -1;
  t.sum = against<PROBS>(powers, mine, t.most);
  for (int i = lane + kWave; i < a.pieces; i += kWave) t.sum += against<PROBS>(powers, part[i], t.most);
  t.sum = sum_of_wave(t.sum);
  return t;
}

// The least place whose running sum exceeds u of the whole; piece_sum(i) is piece i's sum, weights(load(i), s, w) a lane's eight weights in
// its step s (of the first 64 pieces lane i asks for piece i's sum).  A wave's work: the pieces' sums tell the piece, whose weights are found
// anew.  Where rounding leaves nothing above the mark, and for u >= 1, the last place of any weight; -1 if there is none.
template <class PieceSum, class Load, class Weights>
__device__ __forceinline__ int draw(const VerifyLaunch& a, double whole, float u, int lane, PieceSum piece_sum, Load load, Weights weights) {
  const double mark = (u > 0.f ? (double)u : 0.0) * whole;
  double before = 0.0, start = 0.0;
  int piece = -1, last = -1;
  for (int i0 = 0; i0 < a.pieces && piece < 0; i0 += kWave) {
    const double v = i0 + lane < a.pieces ? piece_sum(i0 + lane) : 0.0;
    const double upto = before + running_sum(v);
    const uint64_t some = __ballot(v > kNothing), over = __ballot(v > kNothing && upto > mark);
    if (over) {
      const int at = __ffsll((unsigned long long)over) - 1;
      piece = i0 + at;
      start = at ? lane_of(upto, at - 1) : before;
    } else if (some) {
      last = i0 + 63 - __clzll((long long)some);
    }
    before = lane_of(upto, kWave - 1);
  }
  const bool found = piece >= 0;
  if (!found) {
    piece = last;
    if (piece < 0) return -1;
  }
  const auto held = load(piece);
  int best = -1;
#pragma unroll
  for (int s = 0; s < kPieceSteps; ++s) {
    const int i = piece * kVerifyPiece + s * kWave * 8 + lane * 8;
    double w[8], sum = 0.0;
    weights(held, s, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += w[e];
    const double upto = running_sum(sum);
    double running = start + (upto - sum);
    int mine = -1, final = -1;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      running += w[e];
      if (w[e] > kNothing) {
        if (mine < 0 && running > mark) mine = i + e;
        final = i + e;
      }
    }
    const uint64_t over = found ? __ballot(mine >= 0) : 0, some = __ballot(final >= 0);
    if (over) return __builtin_amdgcn_readlane(mine, __ffsll((unsigned long long)over) - 1);
    if (some) best = __builtin_amdgcn_readlane(final, 63 - __clzll((long long)some));
    start += lane_of(upto, kWave - 1);
  }
  return best;
}

__device__ __forceinline__ void write_path(const VerifyLaunch& a, int b, int lane, int row, int count, int next) {
  for (int i = lane; i < a.max_rows; i += kWave) a.rows_out[(int64_t)b * a.max_rows + i] = i < count ? row : -1;
  if (lane == 0) {
    a.counts[b] = count;
    a.next[b] = next;
  }
}

// Whether this workgroup is the last of `groups` of sequence b to come here: what the others wrote before is then seen by its first wave.
// Every wave waits until its own stores have left it, which the barrier does not; then one thread's write-back, which waits for its own wave's
// alone, finds the workgroup's in the cache that it writes back.  (A release of every wave made the kernel of 48 chains take 61 us.)
__device__ __forceinline__ bool last_to_arrive(const VerifyLaunch& a, int b, int groups) {
  __shared__ int count;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "agent");
    count = __hip_atomic_fetch_add(a.arrived + b, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (count != groups - 1) return false;
  if (threadIdx.x < kWave) __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
  return true;
}

// A wave a row, four to a workgroup: the rows of a sequence are drawn at once, not only those of the path, which is known one row after the
// other.  8 trees of up to 32 rows of 100003 logits 7.5 us (one workgroup of sixteen waves a sequence 26), dependent reads and one piece's weights.
template <int RT, bool PROBS>
__global__ __launch_bounds__(kVerifyThreads) void verify_walk_kernel(VerifyLaunch a, int max_groups) {
  constexpr int N = PROBS ? kProbs : kLogits;
  __shared__ double table[kTable];
  const int b = blockIdx.x / max_groups, group = blockIdx.x % max_groups;
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const double power = own_power();
  bool greedy;
  const double c = sharpness_of(a, b, greedy);
  int first;
  const int n = rows_of_sequence(a, b, first), groups = max(1, ceil_div(n, kVerifyWaves));
  if (group >= groups) return;
  const int i = group * kVerifyWaves + wave;
  int32_t* const picked = a.picked + (int64_t)b * a.max_rows;
  const VerifyPart mine = i < n ? first_part(a, first + i, lane) : VerifyPart{};
  const float u = i < n ? a.uniforms[2 * (int64_t)(first + i) + 1] : 0.f;
  keep_power(table, power);
  __syncthreads();
  const Powers powers(table, c);
  if (i < n) {
    const RowTotal t = total_of_row<PROBS>(a, powers, first + i, mine, lane);
    int token = t.where;
    if (!greedy) {
      const void* const src = row_of<RT, PROBS>(a, first + i);
      const VerifyPart* const part = a.part + (int64_t)(first + i) * a.pieces;
      token = draw(a, t.sum, u, lane, [&](int piece) { return against<PROBS>(powers, piece < kWave ? mine : part[piece], t.most); },
                   [&](int piece) { return load_piece<RT, N>(a, src, piece, lane); },
                   [&](const Piece<RT>& held, int s, double (&w)[8]) { weights_or_probs<PROBS>(powers, numbers_of<RT, N>(held.step[s]), t.most, w); });
    }
    if (lane == 0) picked[i] = token;
  }
  if (!last_to_arrive(a, b, groups) || wave) return;
  // lane i is row i
  int parent = -1, token = -1, want = -1;
  if (lane < n) {
    want = picked[lane];
    if (lane > 0) {
      parent = a.parents ? a.parents[first + lane] : lane - 1;
      if (parent < 0 || parent >= lane) parent = -1;
      token = a.tokens[first + lane];
    }
  }
  // a row that may follow its parent; of those the walk takes the first behind where it stands
  const int wanted = __shfl(want, max(parent, 0));
  const bool follows = parent >= 0 && token == wanted && wanted >= 0;
  int here = 0, count = n > 0 ? 1 : 0, path = 0;
  while (n > 0) {
    const uint64_t child = __ballot(follows && parent == here);
    if (!child) break;
    here = __ffsll((unsigned long long)child) - 1;
    if (lane == count) path = here;
    ++count;
  }
  write_path(a, b, lane, path, count, n > 0 ? __builtin_amdgcn_readlane(want, here) : -1);
}

// A piece of a row and of the draft probabilities of the row behind it, and what a rejection leaves of its tokens: max(w - q E, 0), each of them cut
// where it is nothing (the sums of a piece and of the whole are then something only where a token is).  Where the token comes from the row
// itself, q is no pointer.
template <int RT>
struct Rest {
  Piece<RT> row;
  Piece<TRI_REAL_FP32> draft;
};
template <int RT, int N>
__device__ __forceinline__ Rest<RT> load_rest(const VerifyLaunch& a, const void* row, const float* q, int piece, int lane) {
  Rest<RT> x;
  x.row = load_piece<RT, N>(a, row, piece, lane);
  if (q) {
    x.draft = load_piece<TRI_REAL_FP32, kProbs>(a, q, piece, lane);
  } else {
#pragma unroll
    for (int s = 0; s < kPieceSteps; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) x.draft.step[s].word[e] = 0;
  }
  return x;
}
template <int RT, bool PROBS>
__device__ __forceinline__ void rest_of(const Powers& powers, const Rest<RT>& held, int s, float most, double sum, double (&w)[8]) {
  const Numbers8 q = numbers_of<TRI_REAL_FP32, kProbs>(held.draft.step[s]);
  weights_or_probs<PROBS>(powers, numbers_of<RT, PROBS ? kProbs : kLogits>(held.row.step[s]), most, w);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const double rest = __builtin_fma(-(double)q.x[e], sum, w[e]);
    w[e] = rest > kNothing ? rest : 0.0;
  }
}

// Every workgroup of a sequence finds for itself which rows are accepted (a wave a row); where one is not, each takes some pieces of what
// that leaves, and the last one draws from it.  48 chains of up to eight rows of 131072 logits 16.9 us: 4 until the rows are decided, 8 for the
// 38 MB of logits and draft probabilities of the rejected ones (4.7 TB/s), 1.5 until the last has come, 4 for its draw.  Workgroups of four
// and of sixteen waves were 1 us slower.
template <int RT, bool PROBS>
__global__ __launch_bounds__(kChainThreads, 4) void verify_chain_kernel(VerifyLaunch a, int groups) {
  constexpr int N = PROBS ? kProbs : kLogits;
  __shared__ RowTotal totals[64];
  __shared__ int fits[64];
  __shared__ double table[kTable];
  const int b = blockIdx.x / groups, group = blockIdx.x % groups;
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const double power = own_power();
  int first;
  const int n = rows_of_sequence(a, b, first);
  bool greedy;
  const double c = sharpness_of(a, b, greedy);
  VerifyPart mine = wave < n ? first_part(a, first + wave, lane) : VerifyPart{};
  keep_power(table, power);
  __syncthreads();
  const Powers powers(table, c);
  for (int i = wave; i < n; i += kChainWaves) {
    if (i != wave) mine = first_part(a, first + i, lane);
    // what the decision on the next row needs is asked for before the sums are joined
    int token = -1;
    float x = -INFINITY, q = 0.f, u = 0.f;
    if (i + 1 < n) {
      const int64_t next = first + i + 1;
      token = a.tokens[next];
      u = a.uniforms[2 * next];
      if (!greedy && token >= 0 && token < a.vocab) {
        x = load_one<RT, N>(row_of<RT, PROBS>(a, first + i), token);
        q = counted<kProbs>(a.draft[next * a.draft_stride + token]);
      }
    }
    const RowTotal t = total_of_row<PROBS>(a, powers, first + i, mine, lane);
    bool ok = false;
    if (greedy) {
      ok = t.where >= 0 && token == t.where;
    } else if (token >= 0 && token < a.vocab) {
      const double w = PROBS ? (double)x : weight_of(powers, x, t.most);
      ok = (u > 0.f ? (double)u : 0.0) * (double)q * t.sum < w;
    }
    if (lane == 0) {
      totals[i] = t;
      if (i + 1 < n) fits[i + 1] = ok;
    }
  }
  __syncthreads();
  const uint64_t refused = __ballot(lane > 0 && lane < n && !fits[lane]);
  const int count = refused ? __ffsll((unsigned long long)refused) - 1 : n, row = first + count - 1;
  const RowTotal t = n > 0 ? totals[count - 1] : RowTotal{0.0, -INFINITY, -1};
  const bool partly = refused && !greedy && t.sum > 0.0;      // a row was rejected: the token comes from what that leaves
  if (!partly && (group || wave)) return;
  const void* const src = row_of<RT, PROBS>(a, row);
  const float* const q = a.draft + (int64_t)(row + 1) * a.draft_stride;
  double* const rest = a.rest + (int64_t)b * a.pieces;
  double whole = 0.0, own = 0.0;
  if (partly) {
    const int piece = group * kChainWaves + wave;
    if (piece < a.pieces) {
      const Rest<RT> held = load_rest<RT, N>(a, src, q, piece, lane);
      double sum = 0.0;
#pragma unroll
      for (int s = 0; s < kPieceSteps; ++s) {
        double w[8];
        rest_of<RT, PROBS>(powers, held, s, t.most, t.sum, w);
        sum += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
      }
      sum = sum_of_wave(sum);
      if (lane == 0) rest[piece] = sum;
    }
    if (!last_to_arrive(a, b, groups) || wave) return;
    own = lane < a.pieces ? rest[lane] : 0.0;
    whole = own;
    for (int i = lane + kWave; i < a.pieces; i += kWave) whole += rest[i];
    whole = sum_of_wave(whole);
  }
  int token = t.where;
  if (!greedy && n > 0) {
    const float u = a.uniforms[2 * (int64_t)row + 1];
    const bool left = whole > kNothing;  // (or rounding left nothing)
    const VerifyPart* const part = a.part + (int64_t)row * a.pieces;
    token = draw(a, left ? whole : t.sum, u, lane, [&](int piece) { return left ? (piece < kWave ? own : rest[piece]) : against<PROBS>(powers, part[piece], t.most); },
                 [&](int piece) { return load_rest<RT, N>(a, src, left ? q : nullptr, piece, lane); },
                 [&](const Rest<RT>& held, int s, double (&w)[8]) { rest_of<RT, PROBS>(powers, held, s, t.most, t.sum, w); });
  }
  write_path(a, b, lane, lane, count, token);
}

// Rows [first new token + rows[j]] to [first new token + j], j < count, of one side of one layer.  Lists ascend, so rows[j] >= j: a thread has one
// place of every row, and what it writes lies before all that it still reads.  32 sequences, 36 layers, 96 rows of 8 x 128 fp8 with scales
// and weights in 8.3 us, one sequence in 3.7: four dependent reads (starts, list, table, row); 15 MB moved would take 3.
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
  for (int p = threadIdx.x; p < pieces; p += blockDim.x) {
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
  for (int p = threadIdx.x; p < 2 * a.Hkv; p += blockDim.x) {
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
  const int64_t units = std::max<int64_t>((int64_t)a.num_rows * a.pieces, 1);
  hipLaunchKernelGGL((verify_sums_kernel<RT, PROBS>), dim3((unsigned)ceil_div64(units, kVerifyWaves)), dim3(kVerifyThreads), 0, s, a);
  if (!a.draft) {
    const int groups = ceil_div(a.max_rows, kVerifyWaves);
    hipLaunchKernelGGL((verify_walk_kernel<RT, PROBS>), dim3((unsigned)(a.B * groups)), dim3(kVerifyThreads), 0, s, a, groups);
  } else {
    const int groups = ceil_div(a.pieces, kChainWaves);
    hipLaunchKernelGGL((verify_chain_kernel<RT, PROBS>), dim3((unsigned)(a.B * groups)), dim3(kChainThreads), 0, s, a, groups);
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
  // (a thread for every 16 bytes of a row)
  const int threads = std::min<int>(kVerifyThreads, (int)align_up(a.Hkv * a.D * a.elem_bytes / 16, kWave));
  hipLaunchKernelGGL(accept_rows_kernel, dim3((unsigned)(a.B * a.L * 2)), dim3(threads), 0, s, a);
  return hipGetLastError();
}

}  // namespace tri
