// Attention of a few query rows per sequence over the paged cache (gfx950): one decoding step, a tree of drafted
// tokens, or the blocks of a list.  Instantiated per head dimension and type of the queries in
// tri_attend_{64,128,256}_{bf16,fp16}.hip.
//
//   s[m][t] = scale * q[m] . k[t]   where row m sees token t, else -inf
//   out[m]  = sum_t 2^(s log2 e - M) v[t] / sum_t 2^(s log2 e - M),   M the running maximum
//
// Rows: the new tokens of a sequence are the last of its cache, n of them have rows here; KV head h serves the M = n * G rows
// (token i, query head h * G + g), m = i * G + g.  Row m sees every token before the new ones, and of those token i and its ancestors.
//
// S^T = K Q^T on the matrix cores (16 tokens x 16 rows x 32 elements) leaves in a lane the scores of one row (lane & 15) for
// tokens (lane >> 4) * 4 + r: exactly the order in which the B operand of O^T = V^T P^T wants them, if the 32 tokens of that
// product are numbered (lane >> 4) * 8 + j = token (j & 4) * 4 + (lane >> 4) * 4 + (j & 3).  So the weights never leave
// their lane, and the rescaling of O is a multiplication inside a lane.
// V^T comes out of LDS by the transposing read (16 lanes, 4 tokens x 16 elements).
//
// Up to 16 rows (attend_few_kernel) the four waves of a workgroup take tiles of 32 tokens in turn, keys straight from
// memory into the operand's registers, and meet once at the end: such a call is bound by reading K and V, and what
// counts is how many bytes are asked for at a time; in long sequences they take a KV head each instead.  Beyond that
// (attend_rows_kernel) every wave has rows of its own and the workgroup shares the tiles through LDS: a tile is read from
// memory once for up to 256 rows.  A sequence is cut into
// splits, as many as the chip has room for at once, joined by attend_finish_kernel.
#pragma once

#include <type_traits>

#include "tri_common.h"
#include "tri_mma_device.h"
#include "tri_score_device.h"

namespace tri {
namespace {

constexpr int kAttendThreads = 256;
constexpr int kAttendWaves = kAttendThreads / kWave;
constexpr int kWaitLoads = 0x0f70;    // s_waitcnt vmcnt(0), the other counters left alone
constexpr int kAttendTile = 32;       // tokens of one product with V

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
__device__ __forceinline__ u32x4 widen8(uint32_t a, uint32_t b) {
  return u32x4{Half<T>::widen_lo(a), Half<T>::widen_hi(a), Half<T>::widen_lo(b), Half<T>::widen_hi(b)};
}

// The bits of the infinities and NaNs among the numbers of a word, to replace them by 0.  (16-bit types: all exponent bits set;
// e4m3 has no infinity, its NaN is all bits but the sign.)
template <int T>
__device__ __forceinline__ uint32_t odd_bits(uint32_t w) {
  constexpr int bits = T == TRI_KV_FP8_E4M3 ? 8 : 16;
  constexpr uint32_t e = T == TRI_KV_FP16 ? 0x7c00u : T == TRI_KV_BF16 ? 0x7f80u : 0x7fu;
  uint32_t drop = 0;
#pragma unroll
  for (int i = 0; i < 32; i += bits)
    if ((w >> i & e) == e) drop |= (bits == 8 ? 0xffu : 0xffffu) << i;
  return drop;
}
template <int T>
__device__ __forceinline__ bool clear_odd(u32x4& w) {
  const u32x4 drop = {odd_bits<T>(w[0]), odd_bits<T>(w[1]), odd_bits<T>(w[2]), odd_bits<T>(w[3])};
  w &= ~drop;
  return (drop[0] | drop[1] | drop[2] | drop[3]) != 0;
}

// One matrix-core step on operands as they come out of memory and LDS.
template <int T>
__device__ __forceinline__ f32x4 mfma(const u32x4& x, const u32x4& y, f32x4 c) {
  if constexpr (T == TRI_KV_FP16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, y), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
}

// The lane's number where the compiler must not compute what follows from it before a loop: rare branches would hold
// registers all the time.
__device__ __forceinline__ int here(int lane) {
  asm volatile("" : "+v"(lane));
  return lane;
}

typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4* LdsI16x4;

// The transposing read: each 16 lanes read a piece of 4 rows (4 lanes of 8 bytes each, lane / 4 the row) x 16 columns
// and lane c receives column c, rows 0 to 3.
typedef __attribute__((address_space(3))) unsigned char* LdsBytes;
__device__ __forceinline__ u32x2 lds_read_transposed(LdsBytes at) {
  const i16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsI16x4)at);
  return __builtin_bit_cast(u32x2, v);
}

// 2^x, the instruction alone: results below 2^-126 become 0, which no sum of weights that holds a 1 sees.
__device__ __forceinline__ float pow2(float x) { return __builtin_amdgcn_exp2f(x); }

// Two 2^(x) terms of one sum: -inf - -inf is a row without tokens on either side, and a factor of 0.
__device__ __forceinline__ float rescale(float m, float top) { return m == -INFINITY ? 0.f : pow2(m - top); }

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

// Rows of a sequence of T tokens: the first of them, how many are computed, and how many new tokens the sequence has, which is more where
// there are rows beyond max_rows or beyond q's.  (No row that is computed sees a new token behind the 64th, so more of
// them than T + 64 are that many.)
struct RowRange {
  int first, n, fresh;
};
__device__ __forceinline__ RowRange rows_of(const AttendLaunch& a, int b, int T) {
  if (!a.row_starts) return {b, 1, 1};
  const int64_t from = a.row_starts[b], to = a.row_starts[b + 1];
  const int first = min(max((int)from, 0), a.num_rows), end = min(max((int)to, first), a.num_rows);
  return {first, min(end - first, a.max_rows), (int)min(max(to - from, (int64_t)0), (int64_t)T + 64)};
}

// What a workgroup works on: a split of a sequence (the unit), one KV head and block of rows of it (inner).  (All blocks of rows of a
// unit on one die, where its L2 has the unit's K and V, gave nothing: 2 x 32768 tokens, 512 rows a KV head 168 us either way, 16 x
// 8192 with 320 rows 267.)
struct Work {
  int b, split, h, rb;
};
__device__ __forceinline__ Work work_of(const AttendLaunch& a) {
  const int heads = a.Hkv / a.heads_per_group, inner_n = heads * a.row_blocks;
  const int inner = blockIdx.x % inner_n, unit = blockIdx.x / inner_n;
  return {unit / a.nsplit, unit % a.nsplit, inner % heads * a.heads_per_group, inner / heads};
}

// Tokens the call reads of a sequence, in the order it reads them: its cache, or the blocks of its list one after the other.
__device__ __forceinline__ int tokens_of(const AttendLaunch& a, int b, int T) {
  if (!a.list) return T;
  return min(a.list_k, ceil_div(T, a.block_size)) * a.block_size;
}

// Where the tokens of a tile lie: list entry, then page, then row, each asked for a tile ahead of the next (a wait for a young
// load would be a wait for every older one), by loads that are never skipped (where one path has fewer of them,
// every wait behind it would be for all).
struct Seq {
  const AttendLaunch& a;
  const int32_t* table;
  const int32_t* list;
  int b, T, end, blocks;                     // blocks: that hold the sequence's tokens
  __device__ __forceinline__ Seq(const AttendLaunch& a_, int b_, int h, int T_, int end_) : a(a_), b(b_), T(T_), end(end_) {
    table = a.block_table ? a.block_table + (int64_t)b * a.block_table_pitch : a.seq_lens;      // (any readable word where there is no table)
    list = a.list ? a.list + ((int64_t)b * a.Hkv + h) * a.list_pitch : nullptr;
    blocks = div(T + a.block_size - 1);
  }
  // (t >= 0; exact below 2^31: the factor is 2^div_shift / block_size rounded up, div_shift = 31 + log2 block_size rounded up)
  __device__ __forceinline__ int div(int t) const { return (int)((uint64_t)(uint32_t)t * a.div_factor >> a.div_shift); }
  __device__ __forceinline__ int mod(int t) const { return t - div(t) * a.block_size; }
  __device__ __forceinline__ uint64_t byte(int page, int in, int es) const {
    return ((uint64_t)(uint32_t)page * (uint64_t)a.stride_block + (uint64_t)(uint32_t)in * (uint32_t)a.stride_token) * es;
  }
};

// The tile of TOK tokens that comes next, STEP tokens apart; ok: which of its tokens there are.  Here for blocks of any size: a
// lane holds one token of the tile.
template <bool UNI, int ES, int TOK, int STEP>
struct Finder {
  const Seq& q;
  int mine, page = 0, in = 0;                // of the lane's token; 0 and 0 for one that is not there
  uint64_t ok = 0;
  int next_tok = -1, next_page = -1, next2_entry = 0;
  __device__ __forceinline__ Finder(const Seq& q_, int lane) : q(q_), mine(lane & (TOK - 1)) {}
  __device__ __forceinline__ int entry(int tile) const {
    if (!q.list) return 0;
    const int t = tile + mine;
    return q.list[t < q.end ? q.div(t) : 0];
  }
  __device__ __forceinline__ int token(int tile, int entry) const {     // position in the sequence, or -1
    const int t = tile + mine;
    const int tok = q.list ? entry * q.a.block_size + q.mod(t) : t;
    return ((t < q.end) & ((uint32_t)entry < (uint32_t)q.blocks) & (tok < q.T)) ? tok : -1;
  }
  __device__ __forceinline__ int page_of(int tok) const {
    const int p = q.table[q.a.block_table ? q.div(max(tok, 0)) : 0];
    return q.a.block_table ? p : q.b;
  }
  __device__ __forceinline__ void begin(int tile) {
    next_tok = token(tile, entry(tile));
    next_page = page_of(next_tok);
    next2_entry = entry(tile + STEP);
  }
  __device__ __forceinline__ void take(int tile) {       // the places of `tile`; the next one's are asked for
    const bool there = (next_tok >= 0) & ((uint32_t)next_page < (uint32_t)q.a.num_blocks);
    page = there ? next_page : 0;
    in = there ? q.mod(next_tok) : 0;
    ok = __ballot(there);
    if (TOK < 64) ok &= 0xffffffffu;
    next_tok = token(tile + STEP, next2_entry);
    next_page = page_of(next_tok);
    next2_entry = entry(tile + 2 * STEP);
  }
  __device__ __forceinline__ GlobalBytes row(GlobalBytes base, int, int r) const {
    return base + q.byte(__shfl(page, r), __shfl(in, r), ES);
  }
  __device__ __forceinline__ int64_t scale_at(int) const { return ((int64_t)page * q.a.block_size + in) * q.a.Hkv; }
};

// Blocks of a multiple of 16 tokens: 16 tokens in a row lie behind one another, so a tile is TOK / 16 places; lane g (and every
// TOK / 16-th behind it) looks up the g-th.  A load of rows asks for the place of its own group alone, on the scalar unit, and
// which tokens there are takes one comparison where all are.  (Scalar loads of the tables do worse: every wait for LDS
// is then one for them too.)
template <int ES, int TOK, int STEP>
struct Finder<true, ES, TOK, STEP> {
  static constexpr int kGroups = TOK / 16;
  const Seq& q;
  int ahead, now = 0, page = 0;
  uint64_t ok = 0;
  int next_entry = 0, next_page = 0, next2_entry = 0;       // of the lane's group
  __device__ __forceinline__ Finder(const Seq& q_, int lane) : q(q_), ahead((lane & (kGroups - 1)) * 16) {}
  __device__ __forceinline__ int entry(int tile) const {
    if (!q.list) return 0;
    const int t = tile + ahead;
    return q.list[t < q.end ? q.div(t) : 0];
  }
  __device__ __forceinline__ int page_of(int tile, int entry) const {
    const int t = tile + ahead;
    const int p = q.table[!q.a.block_table ? 0 : q.list ? ((uint32_t)entry < (uint32_t)q.blocks ? entry : 0) : t < q.end ? q.div(t) : 0];
    return q.a.block_table ? p : q.b;
  }
  __device__ __forceinline__ void begin(int tile) {
    next_entry = entry(tile);
    next_page = page_of(tile, next_entry);
    next2_entry = entry(tile + STEP);
  }
  __device__ __forceinline__ void take(int tile) {
    now = tile;
    page = next_page;
    bool whole = (uint32_t)page < (uint32_t)q.a.num_blocks;
    if (q.list) whole &= ((uint32_t)next_entry < (uint32_t)q.blocks) & ((next_entry + 1) * q.a.block_size <= q.T);
    constexpr uint64_t all = TOK < 64 ? 0xffffffffu : ~0ull;
    ok = all;
    if (tile + TOK > q.end || ~__ballot(whole)) {
      ok = 0;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        const int t = tile + 16 * g, e = __builtin_amdgcn_readlane(next_entry, g), p = __builtin_amdgcn_readlane(page, g);
        const int left = min(q.end - t, q.T - (q.list ? e * q.a.block_size + q.mod(t) : t));        // tokens from the group's first to the end
        const bool there = (left > 0) & ((uint32_t)e < (uint32_t)q.blocks) & ((uint32_t)p < (uint32_t)q.a.num_blocks);
        ok |= (uint64_t)(there ? (left >= 16 ? 0xffffu : (1u << left) - 1) : 0) << (16 * g);
      }
    }
    next_entry = next2_entry;
    next_page = page_of(tile + STEP, next_entry);
    next2_entry = entry(tile + 2 * STEP);
  }
  // row0: the first row of the wave's load, all of whose rows lie in one group.  (A place that is not there: a row of another
  // block, or of block 0.)
  __device__ __forceinline__ GlobalBytes row(GlobalBytes base, int row0, int r) const {
    const int g = row0 / 16;
    int p = __builtin_amdgcn_readlane(page, g);
    p = (uint32_t)p < (uint32_t)q.a.num_blocks ? p : 0;
    return base + q.byte(p, q.mod(now + g * 16), ES) + (uint32_t)((r - g * 16) * (int)q.a.stride_token * ES);
  }
  __device__ __forceinline__ int64_t scale_at(int l) const {
    const int g = (l & (TOK - 1)) / 16;
    int p = __shfl(page, g);
    p = (uint32_t)p < (uint32_t)q.a.num_blocks ? p : 0;
    return ((int64_t)p * q.a.block_size + q.mod(now + g * 16) + (l & 15)) * q.a.Hkv;
  }
};

// Queries of row c16 of 16 rows from m0 on: elements as the keys are loaded (fp8: 16 in a piece, two steps of 8).
template <bool FP8, int D>
__device__ __forceinline__ void load_queries(const AttendLaunch& a, const RowRange& rows, int h, int m0, int M, int lane, u32x4 (&qf)[D / 32]) {
  const int m = m0 + (lane & 15), q4 = lane >> 4;
  const int i = m < M ? m / a.G : 0, g = m < M ? m % a.G : 0;
  const char* qp = reinterpret_cast<const char*>(a.q) + ((int64_t)(rows.first + i) * a.q_stride_row + (int64_t)(h * a.G + g) * a.q_stride_head) * 2;
#pragma unroll
  for (int s = 0; s < D / 32; ++s) {
    const int el = FP8 ? (s / 2) * 64 + q4 * 16 + (s & 1) * 8 : s * 32 + q4 * 8;
    qf[s] = m < M ? *reinterpret_cast<const u32x4*>(qp + el * 2) : u32x4{0, 0, 0, 0};
  }
}

// Infinities and NaNs among the values (and value scales, vsc) of new tokens reach the rows that see the token and no others (0 * inf in the matrix
// product would put them into all of them, so there they are 0): rare, at the end, read from memory again.  Tokens from
// first_tok to end of which every step-th piece of 32, from the piece-th on, is the caller's.
template <int PT, bool FP8, int NT, int RT>
__device__ __forceinline__ void add_odd_values(f32x4 (&o)[RT][NT], const Seq& q, GlobalBytes vb, GlobalF32 vsc, int begin, int base,
                                               const uint64_t (&seen)[RT], int lane, int piece, int step) {
  constexpr int ES = FP8 ? 1 : 2;
#pragma unroll 1
  for (int tok = max(begin, base); tok < min(q.end, base + 64); ++tok) {
    if ((tok - begin) / kAttendTile % step != piece) continue;
    const int page = q.a.block_table ? q.table[q.div(tok)] : q.b;
    if (page < 0 || page >= q.a.num_blocks) continue;
    const GlobalBytes row = vb + q.byte(page, q.mod(tok), ES);
    const float by = FP8 && vsc ? vsc[((int64_t)page * q.a.block_size + q.mod(tok)) * q.a.Hkv] : 1.f;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = t * 16 + (lane >> 4) * 4 + e;
        float v;
        if constexpr (FP8) v = __builtin_amdgcn_cvt_f32_fp8((int)(uint8_t)row[d], 0);
        else v = Half<PT>::value(*(const __attribute__((address_space(1))) uint16_t*)(row + d * ES));
        if (!(v - v == 0.f) || !(by - by == 0.f)) {
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
            if (seen[rt] >> (tok - base) & 1) o[rt][t][e] += v * by;
        }
      }
    }
  }
}

// A value's scale as it goes into the product: 0 behind the end, and where it is a new token's and no number (odd).
__device__ __forceinline__ float scale_of(float vs, bool there, bool is_new, bool& odd) {
  const bool out = is_new && there && !(vs - vs == 0.f);
  odd |= out;
  return there && !out ? vs : 0.f;
}

__device__ __forceinline__ float lse_of(float top, float total) { return total == 0.f ? -INFINITY : top + log2f(total); }

// One row's four elements d to d + 3 of a workgroup's result: its part, or the output itself.
template <int QT, int D>
__device__ __forceinline__ void put_row(const AttendLaunch& a, const RowRange& rows, int b, int h, int split, int m, int d, const f32x4& v,
                                        float top, float total) {
  if (a.nsplit > 1) {
    const int64_t at = (((int64_t)b * a.Hkv + h) * a.nsplit + split) * a.max_rows * a.G + m;
    *reinterpret_cast<f32x4*>(a.part_out + at * D + d) = v;
    if (d == 0) {
      a.part_ml[at * 2] = top;
      a.part_ml[at * 2 + 1] = total;
    }
    return;
  }
  const int64_t i = rows.first + m / a.G;
  const int hq = h * a.G + m % a.G;
  const float inv = total == 0.f ? 0.f : a.v_scale / total;       // (a row that saw nothing: zeros and -inf)
  uint16_t* dst = reinterpret_cast<uint16_t*>(a.out) + i * a.out_stride_row + (int64_t)hq * a.out_stride_head + d;
  *reinterpret_cast<uint2*>(dst) = uint2{Half<QT>::pack(v[0] * inv, v[1] * inv), Half<QT>::pack(v[2] * inv, v[3] * inv)};
  if (d == 0) {
    const float l2 = lse_of(top, total);
    if (a.lse) a.lse[i * a.Hq + hq] = l2 * 0.69314718055994530942f;
    if (a.lse2) a.lse2[i * a.Hq + hq] = l2;
  }
}

// Where the scores of a wave's rows go, where weights are wanted.
struct ScoreRows {
  float* head = nullptr;           // of the (sequence, KV head), or NULL
  int64_t pitch = 0;
  int m0 = 0, M = 0;
};
__device__ __forceinline__ ScoreRows score_rows(const AttendLaunch& a, int b, int h, int m0, int M) {
  return {a.scores ? a.scores + ((int64_t)b * a.Hkv + h) * a.max_rows * a.G * a.score_pitch : nullptr, a.score_pitch, m0, M};
}

// Running maximum (base 2, behind the true one by at most kSlack) and sum of a row, with what every 32 tokens ask of the maximum:
// the product above which it has to grow, and what is added to the exponents.
struct RowState {
  float top = -INFINITY, sum = 0.f, grow = -INFINITY, down = 0.f;
};
// How far a score may lie above the maximum that weights are taken against before O is rescaled: weights stay below 2^8, far
// inside either type, and a rescaling (a read and a write of all of O) is rare after the first tokens, where a new maximum is not.
constexpr float kSlack = 8.f;

// Which of 32 tokens a row sees (bit j: token first + j counted from the first new one): those that are there and, of the new
// ones, itself and its ancestors.
__device__ __forceinline__ uint32_t seen_of(uint32_t okm, bool drafts, int first, uint64_t seen) {
  if (!drafts) return okm;
  if (first >= 64) return 0;
  return okm & (first >= 0 ? (uint32_t)(seen >> (first & 63)) : (uint32_t)(seen << (-first & 63)) | ((1u << (-first & 31)) - 1));
}

// The softmax of 32 tokens for RT rows a lane: sc holds q . k of tokens i * 16 + (lane >> 4) * 4 + r; pf receives the weights
// 2^(x - top) packed for the product with V (vs scales them: fp8 rows with scales of their own) in PIECES numbers of the
// queries' type.  Two, the rounded weight and what that left of it, hold a bf16 weight to 2^-16 and an fp16 one to 2^-22; a single one
// to 2^-8 and 2^-11, while the sum adds them unrounded: errors of either sign, which take outputs from 0.0017 to 0.0022 of their size
// off the exact ones (fp16 0.0002 to 0.0003), most of it the rounding of the output in either case.  The second piece doubles
// the products with V.  Up to 16 rows, where reading bounds, that costs nothing (16 x 2176: 45.0 us both; fp8 16 x 16384: 155), of 17
// to 64 rows of 16-bit caches 1 to 2 % (8 x 8192 tokens, 64 rows: 66 -> 67).  With more rows, and of fp8 where
// widening takes turns with the products, it would be felt: 2 x 32768 with 240 rows 101 -> 124 us, 8 x 4096 with 256 rows 55 -> 64, fp8
// 8 x 8192 with 64 rows 53 -> 58: there weights are one number.
// fp8 rows with scales of their own: the weight of a value carries its row's scale, which fp16 has no room for.  There all weights carry
// a power of two as well, lift, that puts the largest scale so far between 1 and 2^6 (weights stay below 2^14) and that O is freed from
// at the end.  fp16 loses up to 2^-25 of a weight there, against the 1 or more of the largest scale: no more than the output's own
// rounding among scales within 2^14 of each other.  A larger scale rescales O, as a larger maximum does; lanes hold the scales
// of 8 tokens, the lanes of all 32 meet where one of them asks for it.
template <int QT, bool FP8>
inline constexpr bool kLifts = FP8 && QT == TRI_KV_FP16;
template <int RT, int NT>
__device__ __forceinline__ void lift_scales(f32x4 (&vs)[2], float& lift, f32x4 (&o)[RT][NT]) {
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) most = fmaxf(most, fabsf(vs[i][r]) < INFINITY ? fabsf(vs[i][r]) : 0.f);
  // (the first scales set it too, however small)
  if (__ballot(most * lift > 64.f || (lift == 0.f && most > 0.f))) {
    most = fmaxf(most, __shfl_xor(most, 16));
    most = fmaxf(most, __shfl_xor(most, 32));
    const float now = ldexpf(1.f, min(-ilogbf(most), 120)), by = lift == 0.f ? 1.f : now / lift;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int t = 0; t < NT; ++t) o[rt][t] *= by;
    lift = now;
  }
  // (no lift yet: scales of 0, infinities and NaN alone, which go as they are)
#pragma unroll
  for (int i = 0; i < 2; ++i) vs[i] *= lift == 0.f ? 1.f : lift;
}
template <int RT, int NT>
__device__ __forceinline__ void free_of_lift(f32x4 (&o)[RT][NT], float lift) {
  if (lift == 0.f) return;             // (no scale but 0, or none)
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int t = 0; t < NT; ++t) o[rt][t] *= 1.f / lift;
}

template <int PT, bool SCALED, bool SCORES, int RT, int NT, int PIECES>
__device__ __forceinline__ void softmax32(f32x4 (&sc)[RT][2], RowState (&st)[RT], f32x4 (&o)[RT][NT], u32x4 (&pf)[PIECES][RT], float scale,
                                          const f32x4 (&ks)[2], const f32x4 (&vs)[2], bool masked, bool drafts, uint32_t okm, int first,
                                          const uint64_t (&seen)[RT], int lane, const ScoreRows& scores, int at) {
  float best[RT];
  bool grows = false;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    if (SCALED) {
      sc[rt][0] *= ks[0];
      sc[rt][1] *= ks[1];
    }
    if (masked) {
      const uint32_t vis = seen_of(okm, drafts, first, seen[rt]) >> (here(lane) >> 4) * 4;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) sc[rt][i][r] = vis >> (i * 16 + r) & 1 ? sc[rt][i][r] : -INFINITY;
    }
    best[rt] = fmaxf(fmaxf(fmaxf(sc[rt][0][0], sc[rt][0][1]), fmaxf(sc[rt][0][2], sc[rt][0][3])),
                     fmaxf(fmaxf(sc[rt][1][0], sc[rt][1][1]), fmaxf(sc[rt][1][2], sc[rt][1][3])));
    grows |= best[rt] > st[rt].grow;
    if (SCORES && scores.head) {
      const int l = here(lane), m = scores.m0 + rt * 16 + (l & 15);
      float* dst = scores.head + m * scores.pitch + at + (l >> 4) * 4;
      if (m < scores.M) {
        *reinterpret_cast<f32x4*>(dst) = sc[rt][0] * scale;
        *reinterpret_cast<f32x4*>(dst + 16) = sc[rt][1] * scale;
      }
    }
  }
  // (the four lanes of a row only speak to each other where one of them has outgrown the maximum)
  if (__ballot(grows)) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float high = fmaxf(best[rt], __shfl_xor(best[rt], 16));
      high = fmaxf(high, __shfl_xor(high, 32));
      const float top = high > st[rt].grow ? high * scale : st[rt].top;
      const float alpha = rescale(st[rt].top, top);
      st[rt].top = top;
      st[rt].sum *= alpha;
      st[rt].grow = (top + kSlack) / scale;
      st[rt].down = top == -INFINITY ? 0.f : -top;
#pragma unroll
      for (int t = 0; t < NT; ++t) o[rt][t] *= alpha;
    }
  }
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    float part = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        sc[rt][i][r] = pow2(__builtin_fmaf(sc[rt][i][r], scale, st[rt].down));
        part += sc[rt][i][r];
      }
      if (SCALED) sc[rt][i] *= vs[i];
    }
    st[rt].sum += part;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float lo = sc[rt][i / 2][(i & 1) * 2], hi = sc[rt][i / 2][(i & 1) * 2 + 1];
#pragma unroll
      for (int p = 0; p < PIECES; ++p) {
        const uint32_t w = Half<PT>::pack(lo, hi);
        pf[p][rt][i] = w;
        lo -= Half<PT>::value((uint16_t)w);
        hi -= Half<PT>::value((uint16_t)(w >> 16));
        if (SCALED) {                  // (of an infinite scale nothing is left)
          lo = fabsf(lo) < INFINITY ? lo : 0.f;
          hi = fabsf(hi) < INFINITY ? hi : 0.f;
        }
      }
    }
  }
}

// ---- up to 16 rows of a KV head
// Bound by reading K and V.  Keys go from memory into the operand's registers (a lane's 16 bytes are a piece of it), values
// through LDS, which transposes them; the next tile's are asked for as soon as this one's registers are free, so that two
// workgroups a CU (four of 64 dimensions) have 128 KiB on their way (fp8: 64).
// 16 x 2176 tokens of 8 x 128 bf16 with four query heads each 36 us (4.0 TB/s), 16 x 16384 of fp8 with HEADS 131 us (K, V and
// the scores written for the weights: 4.4 TB/s), without weights 114 (4.7), where a copy reaches 5.1; 160 tokens 7 us.
// HEADS: a wave has a KV head to itself, four neighbours in a workgroup, and nothing is joined here.
template <int QT, bool FP8, int D, bool UNI, bool HEADS>
__global__ __launch_bounds__(kAttendThreads, D == 256 ? 1 : D == 128 ? 2 : 4) void attend_few_kernel(AttendLaunch a) {
  constexpr int PT = QT;                                  // type of the product with V
  constexpr int ES = FP8 ? 1 : 2;
  constexpr int KC = D * ES / 64;                         // 16-byte pieces of a key in a lane
  constexpr int LPR = D * ES / 16;                        // lanes that load one value row
  constexpr int RPL = kWave / LPR;                        // rows of one load
  constexpr int NV = kAttendTile / RPL;                   // 16-byte pieces of a tile's values in a lane
  constexpr int NT = D / 16;
  constexpr int kPitch = D * 2 + 32;                      // bytes of a value row in LDS: eight rows reach all banks
  constexpr int kWaveBytes = kAttendTile * kPitch;
  constexpr int kParts = HEADS ? 1 : kAttendWaves;        // waves that share a head's tokens
  constexpr int kPieces = 2;                              // of a weight (see softmax32)
  constexpr int kStep = kParts * kAttendTile;
  __shared__ __align__(16) unsigned char s_v[kAttendWaves * kWaveBytes];
  __shared__ __align__(16) float s_scale[kAttendWaves][2][kAttendTile];
  __shared__ float s_ml[kAttendWaves][16][2];

  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int c16 = lane & 15, q4 = lane >> 4;
  const Work work = work_of(a);
  const int b = work.b, split = work.split, h = work.h + (HEADS ? wave : 0), part = HEADS ? 0 : wave;

  const int T = min(max(a.seq_lens[b], 0), a.Tmax);
  const RowRange rows = rows_of(a, b, T);
  const int n = rows.n, fresh = rows.fresh, M = n * a.G;
  if (M == 0) return;
  const int Tv = tokens_of(a, b, T);
  const int begin = split * a.split_tokens, end = min(begin + a.split_tokens, Tv);
  if (begin >= Tv && split > 0) return;
  const int base = T - fresh;                             // first new token (negative: not all of them are in the cache)
  const GlobalBytes kb = (GlobalBytes)a.k_layers[a.layer] + (int64_t)h * a.stride_head * ES;
  const GlobalBytes vb = (GlobalBytes)a.v_layers[a.layer] + (int64_t)h * a.stride_head * ES;
  const bool scaled = FP8 && a.k_scale_layers;
  const GlobalF32 ksc = scaled ? (GlobalF32)a.k_scale_layers[a.layer] + h : nullptr;
  const GlobalF32 vsc = scaled ? (GlobalF32)a.v_scale_layers[a.layer] + h : nullptr;

  // (the queries first: the loop's first wait for them is then none for the keys and values behind them)
  u32x4 qf[D / 32];
  load_queries<FP8, D>(a, rows, h, 0, M, lane, qf);
  uint64_t seen[1] = {1};
  if (fresh > 1) seen[0] = (uint64_t)shfl64((int64_t)ancestor_mask(a.parents, rows.first, n, lane), min(c16, M - 1) / a.G);

  const Seq seq(a, b, h, T, end);
  Finder<UNI, ES, kAttendTile, kStep> find(seq, lane);
  const int first_tile = begin + part * kAttendTile;
  u32x4 kr[2][KC], vr[NV];
  float ks_mine = 0.f, vs_mine = 0.f;
  auto load_keys = [&] {
    if (scaled) {
      ks_mine = ksc[find.scale_at(lane)];
      vs_mine = vsc[find.scale_at(lane)];
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const GlobalBytes src = find.row(kb, i * 16, i * 16 + c16) + q4 * 16;
#pragma unroll
      for (int c = 0; c < KC; ++c) kr[i][c] = *(GlobalU4)(src + c * 64);
    }
  };
  auto load_values = [&] {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      vr[i] = *(GlobalU4)(find.row(vb, i * RPL, i * RPL + lane / LPR) + (lane % LPR) * 16);
  };

  const ScoreRows scores = score_rows(a, b, h, 0, M);

  f32x4 o[1][NT];
  bool odd = false;
  float lift = 0.f;
  RowState st[1];
#pragma unroll
  for (int t = 0; t < NT; ++t) o[0][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  unsigned char* const my_v = s_v + wave * kWaveBytes;
  const LdsBytes my_lds = (LdsBytes)my_v + (q4 * 4 + (c16 >> 2)) * kPitch + (c16 & 3) * 8;
  uint32_t ok_now = 0;
  // One tile; the last one has no next (a body of its own: see the loads above).
  auto step = [&](int tile, auto has_next) {
    constexpr bool more = decltype(has_next)::value;
    const uint32_t okm = ok_now;
    const bool drafts = fresh > 1 && tile + kAttendTile > base;

    f32x4 sc[1][2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      sc[0][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < D / 32; ++s) {
        u32x4 kf;
        if constexpr (FP8) {
          kf = widen8<QT>(kr[i][s / 2][(s & 1) * 2], kr[i][s / 2][(s & 1) * 2 + 1]);
        } else {
          kf = kr[i][s];
        }
        sc[0][i] = mfma<QT>(kf, qf[s], sc[0][i]);
      }
    }
    if (scaled && lane < kAttendTile) {
      s_scale[wave][0][lane] = ks_mine;
      // (behind the end there may be anything)
      s_scale[wave][1][lane] = scale_of(vs_mine, okm >> lane & 1, drafts && tile + lane >= base, odd);
    }
    __builtin_amdgcn_sched_barrier(0);
    // the next tile's keys into the registers of this one's, this one's values into LDS
    if constexpr (more) {
      find.take(tile + kStep);
      ok_now = (uint32_t)find.ok;
      load_keys();
    }
    if (okm != 0xffffffffu || drafts) {
      // What lies behind the end is 0 in the product (0 * what is there could be NaN), and so are a new token's infinities.
      const int l = here(lane);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int row = i * RPL + l / LPR;
        if (!(okm >> row & 1)) vr[i] = u32x4{0, 0, 0, 0};
        if (drafts && tile + row >= base) odd |= clear_odd<FP8 ? TRI_KV_FP8_E4M3 : PT>(vr[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      u32x4* dst = reinterpret_cast<u32x4*>(my_v + (i * RPL + lane / LPR) * kPitch + (lane % LPR) * (FP8 ? 32 : 16));
      if constexpr (FP8) {
        dst[0] = widen8<PT>(vr[i][0], vr[i][1]);
        dst[1] = widen8<PT>(vr[i][2], vr[i][3]);
      } else {
        dst[0] = vr[i];
      }
    }
    if constexpr (more) load_values();
    order_lds_of_wave();
    __builtin_amdgcn_sched_barrier(0);
    const bool masked = okm != 0xffffffffu || drafts;
    u32x4 pf[kPieces][1];
    f32x4 ks[2] = {}, vs[2] = {};
    if (scaled) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        ks[i] = *reinterpret_cast<const f32x4*>(&s_scale[wave][0][i * 16 + q4 * 4]);
        vs[i] = *reinterpret_cast<const f32x4*>(&s_scale[wave][1][i * 16 + q4 * 4]);
      }
      if constexpr (kLifts<QT, FP8>) lift_scales<1, NT>(vs, lift, o);
      softmax32<PT, true, true, 1, NT, kPieces>(sc, st, o, pf, a.scale_log2, ks, vs, masked, drafts, okm, tile - base, seen, lane, scores, tile);
    } else {
      softmax32<PT, false, true, 1, NT, kPieces>(sc, st, o, pf, a.scale_log2, ks, vs, masked, drafts, okm, tile - base, seen, lane, scores, tile);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const u32x2 lo = lds_read_transposed(my_lds + t * 32), hi = lds_read_transposed(my_lds + t * 32 + 16 * kPitch);
#pragma unroll
      for (int p = 0; p < kPieces; ++p) o[0][t] = mfma<PT>(u32x4{lo[0], lo[1], hi[0], hi[1]}, pf[p][0], o[0][t]);
    }
    order_lds_of_wave();             // (the next tile goes to the same places)
  };
  if (first_tile < end) {
    find.begin(first_tile);
    find.take(first_tile);
    ok_now = (uint32_t)find.ok;
    __builtin_amdgcn_sched_barrier(0);
    load_keys();
    __builtin_amdgcn_sched_barrier(0);
    load_values();
    __builtin_amdgcn_sched_barrier(0);
    int tile = first_tile;
    for (; tile + kStep < end; tile += kStep) step(tile, std::true_type{});
    if (tile < end) step(tile, std::false_type{});
  }
  if constexpr (kLifts<QT, FP8>) free_of_lift<1, NT>(o, lift);
  if (__ballot(odd)) add_odd_values<PT, FP8, NT, 1>(o, seq, vb, vsc, begin, base, seen, lane, part, kParts);

  st[0].sum += __shfl_xor(st[0].sum, 16);
  st[0].sum += __shfl_xor(st[0].sum, 32);
  if constexpr (HEADS) {
    if (c16 >= M) return;
#pragma unroll
    for (int t = 0; t < NT; ++t) put_row<QT, D>(a, rows, b, h, split, c16, t * 16 + q4 * 4, o[0][t], st[0].top, st[0].sum);
    return;
  }
  // the four waves meet
  if (q4 == 0) {
    s_ml[wave][c16][0] = st[0].top;
    s_ml[wave][c16][1] = st[0].sum;
  }
  __syncthreads();
  f32x4* const box = reinterpret_cast<f32x4*>(s_v);       // [wave][NT][64]
  static_assert(NT * kWave * 16 <= kWaveBytes, "the exchange fits the value tiles");
  float all = -INFINITY;
#pragma unroll
  for (int w = 0; w < kAttendWaves; ++w) all = fmaxf(all, s_ml[w][c16][0]);
  const float mine = rescale(st[0].top, all);
#pragma unroll
  for (int t = 0; t < NT; ++t) box[(wave * NT + t) * kWave + lane] = o[0][t] * mine;
  __syncthreads();
  for (int it = threadIdx.x; it < NT * kWave; it += kAttendThreads) {
    const int t = it / kWave, l = it % kWave, m = l & 15;
    if (m >= M) continue;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    float total = 0.f, top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kAttendWaves; ++w) top = fmaxf(top, s_ml[w][m][0]);
#pragma unroll
    for (int w = 0; w < kAttendWaves; ++w) {
      v += box[(w * NT + t) * kWave + l];
      total += rescale(s_ml[w][m][0], top) * s_ml[w][m][1];
    }
    put_row<QT, D>(a, rows, b, h, split, m, t * 16 + (l >> 4) * 4, v, top, total);
  }
}

// ---- more rows: RT tiles of 16 rows a wave, W waves, K and V of BT tokens in LDS for all of them
// Bound by turns: the matrix cores work a third of the time, the softmax's vector instructions and LDS reads about as long
// each, and two waves a SIMD overlap little of it (phases a barrier apart, so that one wave's softmax would meet the other's
// products, were slower: 137 us and more against 112).  Two row tiles to a wave halve what it reads of LDS a row, and eight
// waves what is read of memory (with the slack in rescaling, 257 -> 111 us for the call below when they came).  The next tile
// waits in registers while this one is worked on.  2 x 32768 tokens with 60 rows of 4 query heads, 8 x 128 fp16: 88 to 92 us, 700
// to 730 TFLOP/s of the 1200 a large product reaches; 8 x 4096 with up to 32 rows of 8: 48 us; 1217 tokens with 16 rows: 12 us.
template <int QT, bool FP8, int D, int RT, int W, bool UNI>
__global__ __launch_bounds__(W * kWave, 2) void attend_rows_kernel(AttendLaunch a) {
  constexpr int PT = QT;
  constexpr int ES = FP8 ? 1 : 2;
  constexpr int BT = D == 256 ? 32 : 64;                  // tokens of a tile
  constexpr int LPR = D * ES / 16;                        // lanes that load one row
  constexpr int RPL = kWave / LPR;                        // rows of a wave's load
  constexpr int NL = BT / (RPL * W) > 0 ? BT / (RPL * W) : 1;      // loads of a lane for K, and for V
  constexpr int NT = D / 16;
  constexpr int kKeyPitch = D * 2 + 16;                   // 16 rows, 16 bytes of each, reach all banks
  constexpr int kValPitch = D * 2 + 32;                   // 8 rows, 32 bytes of each
  static_assert(RPL <= 16 && BT % RPL == 0, "a wave's load stays within 16 rows");
  __shared__ __align__(16) unsigned char s_k[2][BT * kKeyPitch];
  __shared__ __align__(16) unsigned char s_v[2][BT * kValPitch];
  __shared__ __align__(16) float s_scale[2][2][BT];
  __shared__ int s_odd;

  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int c16 = lane & 15, q4 = lane >> 4;
  const Work work = work_of(a);
  const int b = work.b, split = work.split, h = work.h, rb = work.rb;

  const int T = min(max(a.seq_lens[b], 0), a.Tmax);
  const RowRange rows = rows_of(a, b, T);
  const int n = rows.n, fresh = rows.fresh, M = n * a.G;
  if (rb * RT * 16 * W >= M) return;
  const int m0 = (rb * W + wave) * RT * 16;
  const bool loads = RPL * W <= BT || wave * RPL < BT;    // (small rows: a load of every wave would be more than a tile)
  const int Tv = tokens_of(a, b, T);
  const int begin = split * a.split_tokens, end = min(begin + a.split_tokens, Tv);
  if (begin >= Tv && split > 0) return;
  const int base = T - fresh;
  const GlobalBytes kb = (GlobalBytes)a.k_layers[a.layer] + (int64_t)h * a.stride_head * ES;
  const GlobalBytes vb = (GlobalBytes)a.v_layers[a.layer] + (int64_t)h * a.stride_head * ES;
  const bool scaled = FP8 && a.k_scale_layers;
  const GlobalF32 ksc = scaled ? (GlobalF32)a.k_scale_layers[a.layer] + h : nullptr;
  const GlobalF32 vsc = scaled ? (GlobalF32)a.v_scale_layers[a.layer] + h : nullptr;

  const Seq seq(a, b, h, T, end);
  Finder<UNI, ES, BT, BT> find(seq, lane);
  u32x4 kr[NL], vr[NL];
  float ks_mine = 0.f, vs_mine = 0.f;
  uint64_t ok_now = 0;                   // tokens of the tile at work that are there
  auto load = [&] {
    if (!loads) return;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int row0 = (i * W + wave) * RPL;              // (the load's rows: all in one group of 16, the same for the whole wave)
      kr[i] = *(GlobalU4)(find.row(kb, row0, row0 + lane / LPR) + (lane % LPR) * 16);
      vr[i] = *(GlobalU4)(find.row(vb, row0, row0 + lane / LPR) + (lane % LPR) * 16);
    }
    if (scaled && wave == 0) {
      ks_mine = ksc[find.scale_at(lane)];
      vs_mine = vsc[find.scale_at(lane)];
    }
  };
  auto store = [&](int tile, int buf) {
    const uint64_t okm = find.ok;
    if (!loads) return;
    const bool all = BT == 64 ? okm == ~0ull : (uint32_t)okm == ~0u;
    const bool drafts = fresh > 1 && tile + BT > base;
    if (!all || drafts) {
      const int l = here(lane);
      bool odd = false;
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int row = (i * W + wave) * RPL + l / LPR;
        if (!(okm >> row & 1)) vr[i] = u32x4{0, 0, 0, 0};
        if (drafts && tile + row >= base) odd |= clear_odd<FP8 ? TRI_KV_FP8_E4M3 : PT>(vr[i]);
      }
      if (odd) s_odd = 1;
    }
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int row = (i * W + wave) * RPL + lane / LPR;
      u32x4* kd = reinterpret_cast<u32x4*>(s_k[buf] + row * kKeyPitch + (lane % LPR) * (FP8 ? 32 : 16));
      u32x4* vd = reinterpret_cast<u32x4*>(s_v[buf] + row * kValPitch + (lane % LPR) * (FP8 ? 32 : 16));
      if constexpr (FP8) {
        kd[0] = widen8<QT>(kr[i][0], kr[i][1]);
        kd[1] = widen8<QT>(kr[i][2], kr[i][3]);
        vd[0] = widen8<PT>(vr[i][0], vr[i][1]);
        vd[1] = widen8<PT>(vr[i][2], vr[i][3]);
      } else {
        kd[0] = kr[i];
        vd[0] = vr[i];
      }
    }
    if (scaled && wave == 0 && lane < BT) {
      s_scale[buf][0][lane] = ks_mine;
      bool odd = false;
      s_scale[buf][1][lane] = scale_of(vs_mine, okm >> lane & 1, fresh > 1 && tile + lane >= base, odd);
      if (odd) s_odd = 1;
    }
  };

  // tile t in LDS, t + 1 in registers, pages of t + 2 and list entries of t + 3 on their way
  if (threadIdx.x == 0) s_odd = 0;
  if (begin < end) {
    find.begin(begin);
    find.take(begin);
    load();
  }
  u32x4 qf[RT][D / 32];
  uint64_t seen[RT];
  constexpr bool kScores = RT * W == 4;                   // (of more rows the weights come from the keys once more)
  constexpr int kPieces = RT * W == 4 && !FP8 ? 2 : 1;    // (see softmax32)
  const ScoreRows scores = kScores ? score_rows(a, b, h, m0, M) : ScoreRows{};
  f32x4 o[RT][NT];
  float lift = 0.f;
  RowState st[RT];
  const uint64_t anc = fresh > 1 ? ancestor_mask(a.parents, rows.first, n, lane) : 1ull;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int m = m0 + rt * 16 + c16;
    load_queries<FP8, D>(a, rows, h, m0 + rt * 16, M, lane, qf[rt]);
    seen[rt] = (uint64_t)shfl64((int64_t)anc, min(m, M - 1) / a.G);
#pragma unroll
    for (int t = 0; t < NT; ++t) o[rt][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  __syncthreads();          // (s_odd)
  // The queries are waited for here: left to the loop, the wait for them would be one for the next tile's rows in every turn.
  __builtin_amdgcn_s_waitcnt(kWaitLoads);
  // (The next tile is asked for in any case, see Seq: behind the end that is some row of the pool, one tile a workgroup.)
  if (begin < end) {
    store(begin, 0);
    ok_now = find.ok;
    find.take(begin + BT);
    load();
  }
  __syncthreads();

  u32x4 kf[2][D / 32], pf[kPieces][RT];
  u32x2 vlo[NT], vhi[NT];
  f32x4 sc[RT][2];
  auto read_keys = [&](int sub, int buf) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const unsigned char* src = s_k[buf] + (sub * 32 + i * 16 + c16) * kKeyPitch;
#pragma unroll
      for (int s = 0; s < D / 32; ++s) {
        const int el = FP8 ? (s / 2) * 64 + q4 * 16 + (s & 1) * 8 : s * 32 + q4 * 8;
        kf[i][s] = *reinterpret_cast<const u32x4*>(src + el * 2);
      }
    }
  };
  auto read_values = [&](int sub, int buf, int from, int to) {
    const LdsBytes at = (LdsBytes)s_v[buf] + (sub * 32 + q4 * 4 + (c16 >> 2)) * kValPitch + (c16 & 3) * 8;
#pragma unroll
    for (int t = from; t < to; ++t) {
      vlo[t] = lds_read_transposed(at + t * 32);
      vhi[t] = lds_read_transposed(at + t * 32 + 16 * kValPitch);
    }
  };
  auto times_keys = [&] {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) sc[rt][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < D / 32; ++s)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) sc[rt][i] = mfma<QT>(kf[i][s], qf[rt][s], sc[rt][i]);
    }
  };
  auto times_values = [&] {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const u32x4 vf{vlo[t][0], vlo[t][1], vhi[t][0], vhi[t][1]};
#pragma unroll
      for (int p = 0; p < kPieces; ++p)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) o[rt][t] = mfma<PT>(vf, pf[p][rt], o[rt][t]);
    }
  };
  auto softmax = [&](int first, int sub, int buf) {
    const uint32_t okm = (uint32_t)(ok_now >> (sub * 32));
    const bool drafts = fresh > 1 && first + 32 > base;
    const bool masked = okm != 0xffffffffu || drafts;
    f32x4 ks[2] = {}, vs[2] = {};
    if (scaled) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        ks[i] = *reinterpret_cast<const f32x4*>(&s_scale[buf][0][sub * 32 + i * 16 + q4 * 4]);
        vs[i] = *reinterpret_cast<const f32x4*>(&s_scale[buf][1][sub * 32 + i * 16 + q4 * 4]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) ks[i] = vs[i] = f32x4{1.f, 1.f, 1.f, 1.f};
    }
    if (kLifts<QT, FP8> && scaled) lift_scales<RT, NT>(vs, lift, o);
    softmax32<PT, FP8, kScores, RT, NT, kPieces>(sc, st, o, pf, a.scale_log2, ks, vs, masked, drafts, okm, first - base, seen, lane, scores, first);
  };
  const bool busy = m0 < M;
  // A tile, while the next one goes from registers to LDS and the one behind it is asked for.
  auto step = [&](int tile, int buf, auto has_next) {
    constexpr bool more = decltype(has_next)::value;
    uint64_t ok_after = 0;
    if (more) {
      store(tile + BT, buf ^ 1);
      ok_after = find.ok;
      find.take(tile + 2 * BT);
      load();
    }
    if (busy) {
#pragma unroll
      for (int sub = 0; sub < BT / 32; ++sub) {
        const int first = tile + sub * 32;
        if (!more && sub > 0 && first >= end) continue;  // (nothing there, and rows of scores are whole pieces of 32 tokens)
        // (values asked for before the softmax, which hides their way out of LDS)
        constexpr int kEarly = NT * RT <= 8 ? NT : NT / 2;
        read_keys(sub, buf);
        __builtin_amdgcn_sched_barrier(0);
        times_keys();
        __builtin_amdgcn_sched_barrier(0);
        read_values(sub, buf, 0, kEarly);
        __builtin_amdgcn_sched_barrier(0);
        softmax(first, sub, buf);
        __builtin_amdgcn_sched_barrier(0);
        read_values(sub, buf, kEarly, NT);
        times_values();
      }
    }
    ok_now = ok_after;
    if (more) __syncthreads();
  };
  int tile = begin, buf = 0;
  for (; tile + BT < end; tile += BT, buf ^= 1) step(tile, buf, std::true_type{});
  if (tile < end) step(tile, buf, std::false_type{});
  if constexpr (kLifts<QT, FP8>) free_of_lift<RT, NT>(o, lift);
  if (s_odd) add_odd_values<PT, FP8, NT, RT>(o, seq, vb, vsc, begin, base, seen, lane, 0, 1);
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    st[rt].sum += __shfl_xor(st[rt].sum, 16);
    st[rt].sum += __shfl_xor(st[rt].sum, 32);
    const int m = m0 + rt * 16 + c16;
    if (m >= M) continue;
#pragma unroll
    for (int t = 0; t < NT; ++t) put_row<QT, D>(a, rows, b, h, split, m, t * 16 + q4 * 4, o[rt][t], st[rt].top, st[rt].sum);
  }
}

// ---- the weights of many rows, from their lse
// weight[token] (+)= sum over rows of 2^(scale q . k - lse): the scores a second time, where leaving them behind takes 8 bytes a row
// and token, written and read, and the keys are read once however many rows there are.  A wave has 64 tokens of a KV head, their keys in
// the operand's registers, and goes through all rows; a lane sums its rows' weights of its tokens, and the sixteen
// lanes of a token's rows meet once at the end: no order of anything to depend on.  Bound by reading the keys, of many rows by the
// exponentials: 2 x 32768 tokens of 8 x 128 bf16, 64 rows of four query heads, 98 to 104 us of the 185 that the call takes with the
// attention, 32 rows 64 of 136; 8 x 4096 with 32 rows of eight 49 of 105, 16 x 2176 of scaled fp8 with 32 of four 37 of 88.
constexpr int kWeighTokens = kWave;
template <int QT, bool FP8, int D, bool UNI>
__global__ __launch_bounds__(kAttendThreads, 2) void weigh_rows_kernel(AttendLaunch a) {
  constexpr int ES = FP8 ? 1 : 2;
  constexpr int TOK = kWeighTokens, NG = TOK / 16;        // tokens of a wave, groups of the product
  __shared__ __align__(16) float s_token[kAttendWaves][TOK];
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int c16 = lane & 15, q4 = lane >> 4;
  const int h = blockIdx.x % a.Hkv, spans = ceil_div(a.Tmax, TOK * kAttendWaves);
  const int unit = blockIdx.x / a.Hkv, b = unit / spans, t0 = (unit % spans * kAttendWaves + wave) * TOK;
  const int T = min(max(a.seq_lens[b], 0), a.Tmax);
  if (t0 >= T) return;
  const RowRange rows = rows_of(a, b, T);
  const int n = rows.n, fresh = rows.fresh, M = n * a.G, base = T - fresh;
  const GlobalBytes kb = (GlobalBytes)a.k_layers[a.layer] + (int64_t)h * a.stride_head * ES;
  const bool scaled = FP8 && a.k_scale_layers;

  const Seq seq(a, b, h, T, T);
  Finder<UNI, ES, TOK, TOK> find(seq, lane);
  find.begin(t0);
  find.take(t0);
  u32x4 kf[NG][D / 32];
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    const GlobalBytes src = find.row(kb, i * 16, i * 16 + c16) + q4 * 16;
#pragma unroll
    for (int c = 0; c < D * ES / 64; ++c) {
      const u32x4 w = *(GlobalU4)(src + c * 64);
      if constexpr (FP8) {
        kf[i][2 * c] = widen8<QT>(w[0], w[1]);
        kf[i][2 * c + 1] = widen8<QT>(w[2], w[3]);
      } else {
        kf[i][c] = w;
      }
    }
  }
  // the lane's token at the end
  const int t = min(t0 + lane, T - 1), page = seq.a.block_table ? seq.table[seq.div(t)] : b;
  const bool there = t0 + lane < T && page >= 0 && page < a.num_blocks;
  float* const w = a.weights + (there ? ((int64_t)page * a.block_size + seq.mod(t)) * a.Hkv + h : 0);
  const float before = a.weight_set || !there || t >= base ? 0.f : *w;
  f32x4 ks[NG], sum[NG];
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    ks[i] = f32x4{a.scale_log2, a.scale_log2, a.scale_log2, a.scale_log2};
    sum[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  if (scaled) {
    const GlobalF32 ksc = (GlobalF32)a.k_scale_layers[a.layer] + h;
    s_token[wave][lane] = ksc[find.scale_at(lane)];
    order_lds_of_wave();
#pragma unroll
    for (int i = 0; i < NG; ++i) ks[i] *= *reinterpret_cast<const f32x4*>(&s_token[wave][i * 16 + q4 * 4]);
    order_lds_of_wave();
  }
  const uint64_t anc = fresh > 1 ? ancestor_mask(a.parents, rows.first, n, lane) : 1ull;
  const bool drafts = fresh > 1 && t0 + TOK > base;

  // a row's queries, lse (infinite where it adds nothing) and new tokens it sees; asked for one tile of rows ahead
  u32x4 q_next[D / 32];
  float lse_next;
  uint64_t seen_next;
  auto ask = [&](int m0) {
    const int m = min(m0 + c16, M - 1), i = m / a.G;
    const int64_t row = rows.first + i;
    const int hq = h * a.G + m - i * a.G;
    const GlobalBytes qp = (GlobalBytes)a.q + (row * a.q_stride_row + hq * a.q_stride_head) * 2;
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
      const int el = FP8 ? (s / 2) * 64 + q4 * 16 + (s & 1) * 8 : s * 32 + q4 * 8;
      q_next[s] = *(GlobalU4)(qp + el * 2);
    }
    lse_next = ((GlobalF32)a.lse2)[row * a.Hq + hq];
    seen_next = (uint64_t)shfl64((int64_t)anc, i);
  };
  if (M > 0) ask(0);
  for (int m0 = 0; m0 < M; m0 += 16) {
    u32x4 qf[D / 32];
#pragma unroll
    for (int s = 0; s < D / 32; ++s) qf[s] = q_next[s];
    const float lse = m0 + c16 >= M || lse_next == -INFINITY ? INFINITY : lse_next;
    const uint64_t seen = seen_next;
    ask(m0 + 16);
    f32x4 sc[NG];
#pragma unroll
    for (int i = 0; i < NG; ++i) sc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < D / 32; ++s)
#pragma unroll
      for (int i = 0; i < NG; ++i) sc[i] = mfma<QT>(kf[i][s], qf[s], sc[i]);
#pragma unroll
    for (int i = 0; i < NG; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) sc[i][r] = __builtin_fmaf(sc[i][r], ks[i][r], -lse);
    if (drafts) {
#pragma unroll
      for (int p = 0; p < NG / 2; ++p) {
        const int first = t0 + p * 32 - base;
        const uint32_t vis = seen_of(~0u, first > -32, first, seen) >> (here(lane) >> 4) * 4;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) sc[p * 2 + i][r] = vis >> (i * 16 + r) & 1 ? sc[p * 2 + i][r] : -INFINITY;
      }
    }
#pragma unroll
    for (int i = 0; i < NG; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) sum[i][r] += pow2(sc[i][r]);
  }
#pragma unroll
  for (int i = 0; i < NG; ++i) {
#pragma unroll
    for (int step = 1; step < 16; step *= 2)
#pragma unroll
      for (int r = 0; r < 4; ++r) sum[i][r] += __shfl_xor(sum[i][r], step);
    if (c16 == 0) *reinterpret_cast<f32x4*>(&s_token[wave][i * 16 + q4 * 4]) = sum[i];
  }
  order_lds_of_wave();
  if (there) *w = before + s_token[wave][lane];
}

template <int QT, bool FP8, int D, bool UNI>
hipError_t launch_attend_typed(const AttendLaunch& a, hipStream_t s) {
  if (a.weigh) {
    const int span = kWeighTokens * kAttendWaves;
    hipLaunchKernelGGL((weigh_rows_kernel<QT, FP8, D, UNI>), dim3((unsigned)(a.B * ceil_div(a.Tmax, span) * a.Hkv)), dim3(kAttendThreads), 0, s, a);
    return hipGetLastError();
  }
  const int64_t units = (int64_t)a.B * a.nsplit;
  const dim3 grid((unsigned)(units * a.row_blocks * (a.Hkv / a.heads_per_group)));
  if (a.heads_per_group > 1) hipLaunchKernelGGL((attend_few_kernel<QT, FP8, D, UNI, true>), grid, dim3(kAttendThreads), 0, s, a);
  else if (a.row_tiles == 0) hipLaunchKernelGGL((attend_few_kernel<QT, FP8, D, UNI, false>), grid, dim3(kAttendThreads), 0, s, a);
  else if (a.row_tiles == 4) hipLaunchKernelGGL((attend_rows_kernel<QT, FP8, D, 1, 4, UNI>), grid, dim3(4 * kWave), 0, s, a);
  else if (a.row_tiles == 8) hipLaunchKernelGGL((attend_rows_kernel<QT, FP8, D, 1, 8, UNI>), grid, dim3(8 * kWave), 0, s, a);
  else if constexpr (D <= 128) {
    if (a.row_tiles != 16) return hipErrorInvalidValue;
    hipLaunchKernelGGL((attend_rows_kernel<QT, FP8, D, 2, 8, UNI>), grid, dim3(8 * kWave), 0, s, a);
  } else return hipErrorInvalidValue;
  return hipGetLastError();
}

template <int QT, int D>
hipError_t launch_attend_dim(const AttendLaunch& a, hipStream_t s) {
  const bool uni = a.block_size % 16 == 0;
  if (a.kv_dtype == TRI_KV_FP8_E4M3) return uni ? launch_attend_typed<QT, true, D, true>(a, s) : launch_attend_typed<QT, true, D, false>(a, s);
  return uni ? launch_attend_typed<QT, false, D, true>(a, s) : launch_attend_typed<QT, false, D, false>(a, s);
}

}  // namespace
}  // namespace tri
