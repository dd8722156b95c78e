// extern "C" boundary of libtriattention_hip.so: argument validation on the host,
// then kernel launches on the caller's stream.  Nothing here allocates or waits.
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <algorithm>
#include <atomic>
#include <climits>
#include <mutex>

#include "tri_common.h"

// Scratch of tri_compress_step_static: one copy per GPU, loaded with the code object.  In host
// code this name is only a handle for hipGetSymbolAddress; the address kernels are given is
// the one that call returns on the device in question.
static __device__ __align__(256) unsigned char scratch[TRI_STATIC_WORKSPACE_BYTES];

namespace {

thread_local char g_err[512] = "";

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

int launch_status(hipError_t e, const char* what) {
  if (e == hipSuccess) return TRI_OK;
  return fail(TRI_ERR_LAUNCH, "%s: %s", what, hipGetErrorString(e));
}

bool is_aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

int elem_bytes(int dt) { return dt == TRI_KV_FP8_E4M3 ? 1 : 2; }

int check_layout(const tri_kv_layout* kv, bool need_v) {
  if (!kv) return fail(TRI_ERR_INVALID_ARGUMENT, "kv layout is NULL");
  if (kv->num_layers <= 0 || kv->num_kv_heads <= 0 || kv->num_kv_heads > 256)
    return fail(TRI_ERR_INVALID_ARGUMENT, "bad layer/head count (%d, %d)", kv->num_layers, kv->num_kv_heads);
  if (kv->head_dim != 64 && kv->head_dim != 128 && kv->head_dim != 256)
    return fail(TRI_ERR_UNSUPPORTED, "head_dim %d not in {64,128,256}", kv->head_dim);
  if (kv->block_size <= 0) return fail(TRI_ERR_INVALID_ARGUMENT, "block_size %d", kv->block_size);
  if (kv->kv_dtype != TRI_KV_BF16 && kv->kv_dtype != TRI_KV_FP16 && kv->kv_dtype != TRI_KV_FP8_E4M3)
    return fail(TRI_ERR_INVALID_ARGUMENT, "kv_dtype %d", kv->kv_dtype);
  if (kv->rope_style != TRI_ROPE_HALF && kv->rope_style != TRI_ROPE_INTERLEAVED)
    return fail(TRI_ERR_INVALID_ARGUMENT, "rope_style %d", kv->rope_style);
  const int eb = elem_bytes(kv->kv_dtype);
  const int64_t per16 = 16 / eb;   // elements per 16-byte access
  if (kv->stride_block % per16 || kv->stride_token % per16 || kv->stride_head % per16)
    return fail(TRI_ERR_INVALID_ARGUMENT, "strides must be multiples of %lld elements (16 bytes)", (long long)per16);
  if (kv->stride_head < kv->head_dim && kv->num_kv_heads > 1)
    return fail(TRI_ERR_INVALID_ARGUMENT, "stride_head %lld < head_dim", (long long)kv->stride_head);
  if (!kv->k_layers) return fail(TRI_ERR_INVALID_ARGUMENT, "k_layers is NULL");
  if (need_v && !kv->v_layers) return fail(TRI_ERR_INVALID_ARGUMENT, "v_layers is NULL");
  if (kv->kv_dtype == TRI_KV_FP8_E4M3 && !kv->k_scale_layers)
    return fail(TRI_ERR_INVALID_ARGUMENT, "fp8 cache without k_scale_layers");
  // v_scale_layers may be NULL: the rows then carry no scales of their own (a cache with one
  // scale per tensor) and compaction moves rows only.
  return TRI_OK;
}

int check_batch(const tri_batch* b, bool need_budget) {
  if (!b) return fail(TRI_ERR_INVALID_ARGUMENT, "batch is NULL");
  if (b->num_seqs <= 0) return fail(TRI_ERR_INVALID_ARGUMENT, "num_seqs %d", b->num_seqs);
  if (b->max_seq_len <= 0) return fail(TRI_ERR_INVALID_ARGUMENT, "max_seq_len %d", b->max_seq_len);
  if (!b->seq_lens) return fail(TRI_ERR_INVALID_ARGUMENT, "seq_lens is NULL");
  if (b->block_table && b->block_table_pitch <= 0)
    return fail(TRI_ERR_INVALID_ARGUMENT, "block_table_pitch %d", b->block_table_pitch);
  if (b->seq_lens_host)
    for (int i = 0; i < b->num_seqs; ++i)
      if (b->seq_lens_host[i] < 0 || b->seq_lens_host[i] > b->max_seq_len)
        return fail(TRI_ERR_INVALID_ARGUMENT, "seq_lens_host[%d] = %d not in [0, max_seq_len = %d]", i,
                    b->seq_lens_host[i], b->max_seq_len);
  if (need_budget) {
    if (!b->budgets) return fail(TRI_ERR_INVALID_ARGUMENT, "budgets is NULL");
    if (b->max_budget <= 0) return fail(TRI_ERR_INVALID_ARGUMENT, "max_budget %d", b->max_budget);
  }
  return TRI_OK;
}

// The calls that read a sequence's pages by themselves: the table has an entry for every block a sequence can have, and without one
// a sequence is one block.
int check_pages(const tri_kv_layout* kv, const tri_batch* b) {
  if (!b->block_table && b->max_seq_len > kv->block_size)
    return fail(TRI_ERR_INVALID_ARGUMENT, "without a block table a sequence is one block: of %d tokens, not %d", kv->block_size, b->max_seq_len);
  if (b->block_table && (int64_t)b->block_table_pitch * kv->block_size < b->max_seq_len)
    return fail(TRI_ERR_INVALID_ARGUMENT, "block_table_pitch %d: %d blocks of %d tokens do not hold %d", b->block_table_pitch,
                b->block_table_pitch, kv->block_size, b->max_seq_len);
  return TRI_OK;
}

int check_score(const tri_kv_layout* kv, const tri_score_params* sp) {
  if (!sp) return fail(TRI_ERR_INVALID_ARGUMENT, "score params are NULL");
  if (sp->num_score_heads <= 0 || sp->num_score_heads % kv->num_kv_heads)
    return fail(TRI_ERR_INVALID_ARGUMENT, "num_score_heads %d is not a multiple of num_kv_heads %d",
                sp->num_score_heads, kv->num_kv_heads);
  if (sp->num_offsets <= 0 || sp->num_offsets > tri::kMaxOffsets)
    return fail(TRI_ERR_INVALID_ARGUMENT, "num_offsets %d not in [1, %d]", sp->num_offsets, tri::kMaxOffsets);
  if (sp->aggregation != TRI_REDUCE_MEAN && sp->aggregation != TRI_REDUCE_MAX)
    return fail(TRI_ERR_INVALID_ARGUMENT, "aggregation %d", sp->aggregation);
  if (!sp->folded || !sp->omega || !sp->offsets)
    return fail(TRI_ERR_INVALID_ARGUMENT, "folded / omega / offsets is NULL");
  if (!is_aligned(sp->folded, 16)) return fail(TRI_ERR_INVALID_ARGUMENT, "folded must be 16-byte aligned");
  return TRI_OK;
}

tri::Workspace plan(const tri_kv_layout* kv, const tri_batch* b, const tri_score_params* sp, int assume_resident = 0,
                    bool allow_resident = true) {
  // Resident kernels: two-byte and fp8 keys go to the matrix-core kernel where the shape has one,
  // and only launches that fill most of the chip take them.  TRI_TUNE_RESIDENT_KERNEL overrides
  // the choice: 1 / 2 take the matrix-core / vector-unit kernel whenever the shape has it (however
  // small the launch), 3 never takes a resident kernel.
  const int64_t force = tri::tuning(TRI_TUNE_RESIDENT_KERNEL);
  const bool f_valu = force == 2;
  const bool f_mfma = force == 1;
  const bool f_off = force == 3;
  // The matrix-core kernel addresses the 16 rows of a step with 32-bit offsets from a scalar base.
  const bool want_mfma = (kv->kv_dtype == TRI_KV_BF16 || kv->kv_dtype == TRI_KV_FP16 || kv->kv_dtype == TRI_KV_FP8_E4M3) &&
                         !f_valu &&
                         kv->stride_token > 0 && kv->stride_token < (1 << 25);
  const int G = sp->num_score_heads / kv->num_kv_heads;
  const bool paged = b->block_table != nullptr;
  // assume_resident > 0: a dry run for a device of that size (tri_describe_plan); no device is asked.
  const int resident = (f_off || !allow_resident) ? 0
                       : (assume_resident > 0 ? assume_resident : tri::fused_resident_workgroups());
  tri::FusedPlan fused{};
  // Small batches are cut by layers as well (TRI_TUNE_LAYER_SPLIT = 0 switches that off, 1 switches
  // it on where the kernel was forced, which otherwise keeps whole-model workgroups).
  const int64_t split_set = tri::tuning(TRI_TUNE_LAYER_SPLIT);
  const bool split = split_set >= 0 ? split_set != 0 : !f_mfma;
  if (want_mfma)
    fused = tri::plan_fused_mfma(b->num_seqs, kv->num_kv_heads, kv->head_dim, G, kv->block_size, paged,
                                 sp->aggregation, b->max_seq_len, resident, f_mfma, kv->kv_dtype, b->seq_lens_host,
                                 kv->num_layers, split);
  if (!fused.eligible && !f_mfma)
    fused = tri::plan_fused(b->num_seqs, kv->num_kv_heads, kv->head_dim, G, kv->block_size, paged, sp->aggregation,
                            b->max_seq_len, resident, f_valu);
  return tri::plan_workspace(b->num_seqs, kv->num_layers, sp->num_score_heads, kv->head_dim / 2, sp->num_offsets,
                             kv->num_kv_heads, b->max_seq_len, fused);
}

int check_workspace(const tri::Workspace& w, void* ws, uint64_t bytes) {
  if (!ws) return fail(TRI_ERR_WORKSPACE, "workspace is NULL");
  if (!is_aligned(ws, 256)) return fail(TRI_ERR_WORKSPACE, "workspace must be 256-byte aligned");
  if (bytes < (uint64_t)w.total)
    return fail(TRI_ERR_WORKSPACE, "workspace has %llu bytes, %lld needed", (unsigned long long)bytes, (long long)w.total);
  return TRI_OK;
}

struct ResidentGate {
  static constexpr int kMaxDevices = 64;
  std::mutex mutex;
  hipEvent_t event[kMaxDevices] = {};
};
ResidentGate& resident_gate() {
  static ResidentGate gate;
  return gate;
}

// Both with the gate's mutex held.  A stream under capture is left alone.
bool gate_applies(hipStream_t s, int& dev) {
  hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
  return hipGetDevice(&dev) == hipSuccess && dev >= 0 && dev < ResidentGate::kMaxDevices &&
         hipStreamIsCapturing(s, &cap) == hipSuccess && cap == hipStreamCaptureStatusNone;
}
int gate_enter(ResidentGate& gate, hipStream_t s) {
  int dev = 0;
  if (!gate_applies(s, dev) || !gate.event[dev]) return TRI_OK;
  return launch_status(hipStreamWaitEvent(s, gate.event[dev], 0), "resident chain wait");
}
int gate_leave(ResidentGate& gate, hipStream_t s) {
  int dev = 0;
  if (!gate_applies(s, dev)) return TRI_OK;
  if (!gate.event[dev]) {
    const hipError_t e = hipEventCreateWithFlags(&gate.event[dev], hipEventDisableTiming);
    if (e != hipSuccess) return launch_status(e, "resident chain event");
  }
  return launch_status(hipEventRecord(gate.event[dev], s), "resident chain record");
}

// Process-wide settings (tri_set_tuning).
constexpr int kTunings = 5;
std::atomic<int64_t> g_tuning[kTunings] = {{0}, {0}, {-1}, {0}, {2000000}};

// Device address of `scratch` on the current device, looked up once per device.
struct StaticScratch {
  static constexpr int kMaxDevices = 64;
  std::mutex mutex;
  void* ptr[kMaxDevices] = {};
};
int static_scratch(void** out) {
  static StaticScratch st;
  int dev = -1;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return launch_status(e, "hipGetDevice");
  if (dev < 0 || dev >= StaticScratch::kMaxDevices) return fail(TRI_ERR_UNSUPPORTED, "device %d out of range", dev);
  std::lock_guard<std::mutex> lock(st.mutex);
  if (!st.ptr[dev]) {
    void* p = nullptr;
    e = hipGetSymbolAddress(&p, HIP_SYMBOL(scratch));
    if (e != hipSuccess) return launch_status(e, "hipGetSymbolAddress(scratch)");
    if (!p || !is_aligned(p, 256)) return fail(TRI_ERR_WORKSPACE, "static scratch at %p is not 256-byte aligned", p);
    st.ptr[dev] = p;
  }
  *out = st.ptr[dev];
  return TRI_OK;
}

template <typename T>
T* at(void* ws, int64_t off) { return reinterpret_cast<T*>(reinterpret_cast<char*>(ws) + off); }

int do_score(const tri_kv_layout* kv, const tri_batch* batch, const tri_score_params* sp, float* raw,
             int64_t rs_layer, int64_t rs_token, int64_t rs_head, void* ws, const tri::Workspace& w,
             hipStream_t s, int fine, float* partial, uint32_t* status) {
  const int F = kv->head_dim / 2;
  hipError_t e = tri::launch_prepare(sp->folded, sp->omega, sp->offsets, sp->num_offsets, batch->round_start,
                                     batch->num_seqs, kv->num_layers, sp->num_score_heads, F, sp->aggregation,
                                     at<float>(ws, w.coef), at<float>(ws, w.trig), status, s);
  if (e != hipSuccess) return launch_status(e, "prepare");
  tri::ScoreLaunch a{};
  a.B = batch->num_seqs; a.L = kv->num_layers; a.Hkv = kv->num_kv_heads; a.D = kv->head_dim;
  a.block_size = kv->block_size; a.kv_dtype = kv->kv_dtype; a.rope_style = kv->rope_style;
  a.A = sp->num_score_heads; a.G = sp->num_score_heads / kv->num_kv_heads; a.NO = sp->num_offsets;
  a.aggregation = sp->aggregation;
  a.Tmax = batch->max_seq_len; a.fine = fine;
  a.stride_block = kv->stride_block; a.stride_token = kv->stride_token; a.stride_head = kv->stride_head;
  a.k_layers = kv->k_layers; a.k_scale_layers = kv->k_scale_layers;
  a.block_table = batch->block_table; a.block_table_pitch = batch->block_table_pitch;
  a.seq_lens = batch->seq_lens;
  a.coef = at<float>(ws, w.coef); a.trig = at<float>(ws, w.trig); a.partial = partial;
  a.raw = raw; a.raw_stride_layer = rs_layer; a.raw_stride_token = rs_token; a.raw_stride_head = rs_head;
  return launch_status(tri::launch_score(a, s), "score");
}

int check_select(const tri_select_params* sel) {
  if (!sel) return fail(TRI_ERR_INVALID_ARGUMENT, "select params are NULL");
  if (sel->group_reduce != TRI_REDUCE_MEAN && sel->group_reduce != TRI_REDUCE_MAX)
    return fail(TRI_ERR_INVALID_ARGUMENT, "group_reduce %d", sel->group_reduce);
  if (sel->layer_reduce != TRI_REDUCE_MEAN && sel->layer_reduce != TRI_REDUCE_MAX && sel->layer_reduce != -1)
    return fail(TRI_ERR_INVALID_ARGUMENT, "layer_reduce %d", sel->layer_reduce);
  if (sel->window_size < 0) return fail(TRI_ERR_INVALID_ARGUMENT, "window_size %d", sel->window_size);
  if (sel->normalize < 0 || sel->normalize > 2) return fail(TRI_ERR_INVALID_ARGUMENT, "normalize %d", sel->normalize);
  if (sel->normalize == 2 && sel->group_first)
    return fail(TRI_ERR_UNSUPPORTED, "the population-std normalisation is built for the normalise-then-reduce order only");
  return TRI_OK;
}

int do_select(const tri_kv_layout* kv, const tri_batch* batch, const tri_score_params* sp,
              const tri_select_params* sel, const float* raw, int64_t rs_layer, int64_t rs_token,
              int64_t rs_head, float* fin, int32_t* keep, void* ws, const tri::Workspace& w, hipStream_t s,
              int fine, const float* partial, int pass_nan) {
  tri::SelectLaunch a{};
  a.B = batch->num_seqs; a.L = kv->num_layers; a.Hkv = kv->num_kv_heads; a.A = sp->num_score_heads;
  a.G = sp->num_score_heads / kv->num_kv_heads; a.Tmax = batch->max_seq_len; a.fine = fine;
  a.max_budget = batch->max_budget;
  a.normalize = sel->normalize; a.window_size = sel->window_size; a.protect_prefill = sel->protect_prefill;
  a.group_reduce = sel->group_reduce; a.layer_reduce = sel->layer_reduce; a.shared = sel->shared;
  a.group_first = sel->group_first ? 1 : 0;
  a.pass_nan = pass_nan;
  a.seq_lens = batch->seq_lens; a.prefill_lens = batch->prefill_lens; a.budgets = batch->budgets;
  a.partial = partial; a.mustd = at<float>(ws, w.mustd);
  a.raw = raw; a.raw_stride_layer = rs_layer; a.raw_stride_token = rs_token; a.raw_stride_head = rs_head;
  a.fin = fin ? fin : at<float>(ws, w.fin);
  a.keep = keep;
  // Scratch of the chunked statistics: the coefficients (the scorer is done with them) or, where one score per KV head
  // needs no sums of the scorer's tiles, the room planned for those.
  a.group_scratch = at<double>(ws, pass_nan ? w.partial : w.coef);
  a.group_scratch_bytes = pass_nan ? w.mustd - w.partial : w.trig - w.coef;
  return launch_status(tri::launch_select(a, s), "select");
}

// A keep set per layer (layer_reduce -1) of a single layer is the mean over that one layer: same
// rows, same scores (x / 1).  The reference's per-layer modes call their selector once per layer
// (runtime/selector_hf.py:473-747 from the layer loop), so those calls may take a resident kernel.
int layer_reduce_of(const tri_kv_layout* kv, const tri_select_params* sel) {
  return (sel->layer_reduce < 0 && kv->num_layers == 1) ? TRI_REDUCE_MEAN : sel->layer_reduce;
}

bool takes_resident(const tri::Workspace& w, const tri_kv_layout* kv, const tri_select_params* sel) {
  return w.fused.eligible && layer_reduce_of(kv, sel) >= 0 && !sel->shared && !sel->group_first && !sel->no_resident;
}

// Quarter tiles of the two-pass scorer.  Their sums take more room than the workspace plans; they go where the
// selection scores are written later (the statistics are finished by then).
bool takes_quarter_tiles(const tri_kv_layout* kv, int B, int Tmax, int A, int aggregation) {
  const int64_t sums = (int64_t)B * kv->num_layers * A * tri::ceil_div(Tmax, tri::kScoreFineTokens) * 4 * 4;
  const int64_t room = tri::align_up((int64_t)B * kv->num_layers * kv->num_kv_heads * Tmax * 4, 256);   // Workspace::fin
  return sums <= room && tri::score_takes_fine(B, kv->num_layers, kv->num_kv_heads, kv->head_dim, A / kv->num_kv_heads,
                                               Tmax, aggregation);
}

// A few layers of a few requests, where the resident kernel would be taken for them, go through
// tri_score_small.hip: a wave per step of 16 tokens, statistics in the selection's workgroups.  Which of the two is faster goes by
//  - the scorer's workgroups (128 tokens of a KV head of a layer), each of which evaluates the phases again: one round
//    of the chip is 1024 of them, 512 at a head dimension of 256;
//  - the layers, which the selection walks one after the other, the longer the more tokens a thread holds of a row: up to
//    4096 tokens four (one query head per KV head 8192, eight), beyond that twice as many;
//  - what the resident kernel costs: with at most four KV heads its workgroups have four waves and it is about 5 us faster.
// Score + select, called eagerly (the event that chains resident launches is 3 us of theirs; a captured launch has none), us,
// resident / small, `layers x requests x tokens, KV heads x head dimension, workgroups`.  Two to four query heads per KV
// head: 1 x 8 x 1987, 8 x 128, 1024: 31.0 / 24.9; 1 x 4 x 3923, 8 x 256, 992: 41.5 / 34.9; 2 x 1 x 3771, 16 x 128, 960:
// 33.9 / 27.3; 3 x 3 x 1663, 8 x 64, 936: 29.6 / 25.1; 4 x 8 x 415, 8 x 128, 1024: 33.7 / 33.0.  Four KV heads: 2 x 4 x 3495, 4 x 64, 896:
// 27.3 / 22.2; 3 x 8 x 1057, 4 x 128, 864: 28.0 / 26.4, but 3 x 8 x 1075, 4 x 256, 864: 32.1 / 36.4 and 4 x 3 x 2596, 4 x 64, 1008:
// 27.0 / 28.2.  Long rows: 1 x 4 x 7782, 4 x 64, 976: 31.0 / 25.8; 2 x 1 x 7139, 8 x 128, 896: 36.7 / 32.2, but 2 x 3 x 5038, 4 x 128, 960:
// 31.1 / 32.7, 3 x 1 x 5052, 8 x 128, 960: 35.7 / 37.7, 3 x 2 x 5036, 4 x 128, 960: 31.5 / 37.8, 4 x 1 x 4170, 1 x 64, 132: 27.9 / 30.9 and
// 4 x 1 x 7652, 4 x 256, 960: 39.5 / 51.0.  One query head: 4 x 1 x 7964, 4 x 64, 1008: 33.2 / 28.7; 2 x 1 x 14202, 4 x 128, 888:
// 38.7 / 35.4, but 3 x 1 x 8914, 4 x 128, 840: 36.4 / 37.3, 4 x 1 x 14881, 2 x 128, 936: 40.4 / 42.7.  Eight: 1 x 4 x 3821, 8 x 128, 960:
// 32.7 / 30.4; 2 x 2 x 3534, 4 x 128, 448: 27.4 / 25.6, but 1 x 8 x 3770, 4 x 128, 960: 26.7 / 29.9.  Of 830 shapes drawn over 1 to
// 4 layers, 1 to 8 query heads, 1 to 16 KV heads of 64 to 256 and 64 to 1024 workgroups 760 go this way, two of them more than
// 2 % slower (1.04 x), and seven of the others would be more than 2 % faster.
int64_t small_workgroups(int L, int G, int D, int Tmax, bool four_waves) {
  const bool wide = D == 256, long_rows = Tmax > (G == 1 ? 8192 : 4096);
  if (L > (G > 4 ? 2 : 4)) return 0;
  if (G > 4) return std::min(1024 / L, four_waves ? (wide ? 512 : 768) : 1024);
  if (long_rows) return L == 1 ? 1024 : L == 2 ? (four_waves && G > 1 ? 768 : 1024) : L == 3 ? (four_waves ? 512 : 768) : G == 1 ? 512 : 0;
  if (four_waves && G > 1 && L >= 3) return wide ? 512 : L == 4 ? 704 : 1024;
  return 1024;
}
bool takes_small(const tri::Workspace& w, const tri_kv_layout* kv, const tri_batch* batch, const tri_score_params* sp,
                 const tri_select_params* sel) {
  const int G = sp->num_score_heads / kv->num_kv_heads, L = kv->num_layers;
  const int64_t wgs = (int64_t)batch->num_seqs * L * kv->num_kv_heads * tri::ceil_div(batch->max_seq_len, 128);
  return tri::tuning(TRI_TUNE_RESIDENT_KERNEL) == 0 && takes_resident(w, kv, sel) && w.fused.eligible == 2 &&
         kv->kv_dtype != TRI_KV_FP8_E4M3 && tri::select_small_takes(batch->max_seq_len, G) &&
         (int64_t)batch->num_seqs * kv->num_kv_heads <= 256 &&
         wgs <= small_workgroups(L, G, kv->head_dim, batch->max_seq_len, w.fused.waves == 4);
}

// Selection straight from the paged keys: the resident kernel when the shape has one,
// else score into the workspace and select from there.
int do_select_paged(const tri_kv_layout* kv, const tri_batch* batch, const tri_score_params* sp,
                    const tri_select_params* sel, float* fin, int32_t* keep, void* ws, const tri::Workspace& w,
                    hipStream_t s, int pass_nan = 0) {
  if (takes_small(w, kv, batch, sp, sel)) {
    tri::SmallScore c{};
    c.k_layers = kv->k_layers; c.block_table = batch->block_table; c.block_table_pitch = batch->block_table_pitch;
    c.seq_lens = batch->seq_lens; c.round_start = batch->round_start;
    c.folded = sp->folded; c.omega = sp->omega; c.offsets = sp->offsets; c.NO = sp->num_offsets;
    c.raw = at<float>(ws, w.raw); c.raw_pitch = batch->max_seq_len; c.status = at<uint32_t>(ws, w.status);
    c.stride_block = kv->stride_block; c.stride_token = kv->stride_token; c.stride_head = kv->stride_head;
    c.L = kv->num_layers; c.A = sp->num_score_heads; c.G = sp->num_score_heads / kv->num_kv_heads;
    c.Tmax = batch->max_seq_len; c.block_size = kv->block_size;
    hipError_t e = tri::launch_score_small(c, batch->num_seqs, kv->num_kv_heads, kv->head_dim, kv->kv_dtype, kv->rope_style, s);
    if (e != hipSuccess) return launch_status(e, "score_small");
    tri::SmallSelect a{};
    a.raw = c.raw; a.raw_pitch = c.raw_pitch; a.seq_lens = batch->seq_lens; a.prefill_lens = batch->prefill_lens;
    a.budgets = batch->budgets; a.fin = fin; a.keep = keep; a.keep_pitch = batch->max_budget; a.status = c.status;
    a.L = c.L; a.Hkv = kv->num_kv_heads; a.A = c.A; a.G = c.G; a.Tmax = c.Tmax;
    a.normalize = sel->normalize; a.window_size = sel->window_size; a.protect_prefill = sel->protect_prefill;
    a.group_reduce = sel->group_reduce; a.layer_reduce = layer_reduce_of(kv, sel); a.pass_nan = 0;
    return launch_status(tri::launch_select_small(a, batch->num_seqs, s), "select_small");
  }
  const bool fused = takes_resident(w, kv, sel);
  if (!fused) {
    float* raw = at<float>(ws, w.raw);
    const int64_t A = sp->num_score_heads;
    const int64_t rs_layer = (int64_t)batch->max_seq_len * A;
    const int fine = takes_quarter_tiles(kv, batch->num_seqs, batch->max_seq_len, (int)A, sp->aggregation);
    float* partial = at<float>(ws, fine ? w.fin : w.partial);
    // The status word belongs to the resident kernel; on this path it just reads "fine".
    const int rc = do_score(kv, batch, sp, raw, rs_layer, A, 1, ws, w, s, fine, partial, at<uint32_t>(ws, w.status));
    if (rc) return rc;
    return do_select(kv, batch, sp, sel, raw, rs_layer, A, 1, fin, keep, ws, w, s, fine, partial, pass_nan);
  }
  const int F = kv->head_dim / 2;
  hipError_t e = hipSuccess;
  if (w.fused.eligible != 2) {   // the matrix-core kernel has a preparation launch of its own
    e = tri::launch_prepare(sp->folded, sp->omega, sp->offsets, sp->num_offsets, batch->round_start,
                            batch->num_seqs, kv->num_layers, sp->num_score_heads, F, sp->aggregation,
                            at<float>(ws, w.coef), at<float>(ws, w.trig), nullptr, s);
    if (e != hipSuccess) return launch_status(e, "prepare");
  }
  tri::FusedLaunch a{};
  a.B = batch->num_seqs; a.L = kv->num_layers; a.Hkv = kv->num_kv_heads; a.D = kv->head_dim;
  a.block_size = kv->block_size; a.kv_dtype = kv->kv_dtype; a.rope_style = kv->rope_style;
  a.A = sp->num_score_heads; a.G = sp->num_score_heads / kv->num_kv_heads; a.Tmax = batch->max_seq_len;
  a.normalize = sel->normalize; a.window_size = sel->window_size; a.protect_prefill = sel->protect_prefill;
  a.group_reduce = sel->group_reduce; a.layer_reduce = layer_reduce_of(kv, sel);
  a.stride_block = kv->stride_block; a.stride_token = kv->stride_token; a.stride_head = kv->stride_head;
  a.k_layers = kv->k_layers; a.k_scale_layers = kv->k_scale_layers;
  a.block_table = batch->block_table; a.block_table_pitch = batch->block_table_pitch;
  a.seq_lens = batch->seq_lens; a.prefill_lens = batch->prefill_lens;
  a.coef = at<float>(ws, w.coef);
  a.folded = sp->folded; a.omega = sp->omega; a.offsets = sp->offsets; a.NO = sp->num_offsets;
  a.round_start = batch->round_start;
  a.xchg = at<unsigned long long>(ws, w.xchg);
  a.status = at<uint32_t>(ws, w.status);
  a.pack = at<int32_t>(ws, w.pack);
  a.fin = fin ? fin : at<float>(ws, w.fin);
  // Partial results of a layer-split launch live where the two-pass path keeps its raw scores
  // ([B][L][Tmax][A] floats, never smaller than [groups][B][Hkv][Tmax]).
  a.fin_part = at<float>(ws, w.raw);
  a.plan = w.fused;
  // Nobody asked for the selection scores themselves: the groups' partial rows go straight to the
  // top-k, which adds them while it loads (one launch less).
  const bool split = w.fused.eligible == 2 && w.fused.layer_groups > 1;
  a.skip_layer_reduce = split && !fin && keep && batch->max_seq_len <= tri::topk_register_row_limit();
  a.bmat = at<char>(ws, w.bmat);
  if (w.fused.eligible == 2) {
    // The preparation launch writes one 16-byte entry per (sequence, layer, KV head, operand, lane); the region planned for them must hold that.
    const int64_t need = (int64_t)a.B * a.L * a.Hkv * tri::mfma_operands(F, a.G) * 64 * 16;
    if (need > w.total - w.bmat)
      return fail(TRI_ERR_WORKSPACE, "coefficient slabs need %lld bytes, %lld planned", (long long)need,
                  (long long)(w.total - w.bmat));
  }
  {
    // Two resident launches that run at the same time on one device would each hold part of
    // the CUs and wait for the other's workgroups until their waits expire.  Launches of this
    // process are therefore chained: each waits (on the device, not on the host) for the
    // previous one on whatever stream that was.  Streams under graph capture are left alone
    // (whoever replays the graph brackets the replay with tri_resident_gate_enter / _leave).
    ResidentGate& gate = resident_gate();
    std::lock_guard<std::mutex> lock(gate.mutex);
    int rc = gate_enter(gate, s);
    if (rc) return rc;
    e = w.fused.eligible == 2 ? tri::launch_fused_mfma(a, s) : tri::launch_fused_select(a, s);
    if (e != hipSuccess) return launch_status(e, "fused_select");
    rc = gate_leave(gate, s);
    if (rc) return rc;
  }
  if (!keep) return TRI_OK;   // selection scores only
  if (a.skip_layer_reduce)
    return launch_status(tri::launch_topk_rows(a.fin_part, a.Tmax, a.B * a.Hkv, a.seq_lens, batch->budgets, a.Hkv, a.Tmax,
                                               keep, batch->max_budget, s, w.fused.layer_groups,
                                               (int64_t)a.B * a.Hkv * a.Tmax, a.layer_reduce == TRI_REDUCE_MAX),
                         "topk_rows");
  return launch_status(tri::launch_topk_rows(a.fin, a.Tmax, a.B * a.Hkv, a.seq_lens, batch->budgets, a.Hkv, a.Tmax, keep,
                                             batch->max_budget, s),
                       "topk_rows");
}

int fill_compact(const tri_kv_layout* kv, const tri_batch* batch, const int32_t* keep, int keep_per_layer,
                 int shared, tri::CompactLaunch& a) {
  int rc = check_layout(kv, true);
  if (rc) return rc;
  rc = check_batch(batch, true);
  if (rc) return rc;
  if (!batch->block_table) return fail(TRI_ERR_INVALID_ARGUMENT, "compaction needs a block table");
  if (!keep) return fail(TRI_ERR_INVALID_ARGUMENT, "keep is NULL");
  const int eb = elem_bytes(kv->kv_dtype);
  a.B = batch->num_seqs; a.L = kv->num_layers; a.Hkv = kv->num_kv_heads; a.D = kv->head_dim;
  a.block_size = kv->block_size; a.elem_bytes = eb; a.max_budget = batch->max_budget;
  a.keep_per_layer = keep_per_layer ? 1 : 0; a.shared = shared ? 1 : 0;
  a.has_scales = kv->kv_dtype == TRI_KV_FP8_E4M3 && kv->v_scale_layers != nullptr;
  a.stride_block = kv->stride_block; a.stride_token = kv->stride_token; a.stride_head = kv->stride_head;
  a.k_layers = kv->k_layers; a.v_layers = kv->v_layers;
  a.k_scale_layers = kv->k_scale_layers; a.v_scale_layers = kv->v_scale_layers;
  a.block_table = batch->block_table; a.block_table_pitch = batch->block_table_pitch;
  a.seq_lens = batch->seq_lens; a.budgets = batch->budgets; a.keep = keep; a.Tmax = batch->max_seq_len;
  a.staging = nullptr;
  return TRI_OK;
}

}  // namespace

namespace tri {
int64_t tuning(int key) { return key >= 0 && key < kTunings ? g_tuning[key].load(std::memory_order_relaxed) : 0; }
}  // namespace tri

extern "C" {

int tri_abi_version(void) { return TRI_ABI_VERSION; }

const char* tri_last_error(void) { return g_err; }

#ifndef TRI_SOURCE_DIGEST
#define TRI_SOURCE_DIGEST "unknown"
#endif
const char* tri_source_digest(void) {
  static const char digest[] = "TRI_SOURCE_DIGEST=" TRI_SOURCE_DIGEST;
  return digest + sizeof("TRI_SOURCE_DIGEST=") - 1;
}

int tri_set_tuning(int32_t key, int64_t value) {
  switch (key) {
    case TRI_TUNE_RESIDENT_KERNEL:
      if (value < 0 || value > 3) return fail(TRI_ERR_INVALID_ARGUMENT, "TRI_TUNE_RESIDENT_KERNEL takes 0..3, got %lld", (long long)value);
      break;
    case TRI_TUNE_RESIDENT_WORKGROUPS:
      if (value < 0 || value > INT_MAX) return fail(TRI_ERR_INVALID_ARGUMENT, "TRI_TUNE_RESIDENT_WORKGROUPS %lld", (long long)value);
      break;
    case TRI_TUNE_LAYER_SPLIT:
      if (value < -1 || value > 1) return fail(TRI_ERR_INVALID_ARGUMENT, "TRI_TUNE_LAYER_SPLIT takes -1, 0 or 1, got %lld", (long long)value);
      break;
    case TRI_TUNE_MAX_KERNEL:
      if (value < 0 || value > 1) return fail(TRI_ERR_INVALID_ARGUMENT, "TRI_TUNE_MAX_KERNEL takes 0 or 1, got %lld", (long long)value);
      break;
    case TRI_TUNE_RESIDENT_WAIT_US:
      // (the kernels count ticks of a 100 MHz clock in 64 bits)
      if (value > (int64_t)3600 * 1000000) return fail(TRI_ERR_INVALID_ARGUMENT, "TRI_TUNE_RESIDENT_WAIT_US beyond one hour");
      break;
    default:
      return fail(TRI_ERR_INVALID_ARGUMENT, "unknown tuning key %d", key);
  }
  g_tuning[key].store(value, std::memory_order_relaxed);
  return TRI_OK;
}

int64_t tri_get_tuning(int32_t key) {
  if (key < 0 || key >= kTunings) return INT64_MIN;
  return g_tuning[key].load(std::memory_order_relaxed);
}

int tri_resident_gate_enter(void* stream) {
  ResidentGate& gate = resident_gate();
  std::lock_guard<std::mutex> lock(gate.mutex);
  return gate_enter(gate, (hipStream_t)stream);
}

int tri_resident_gate_leave(void* stream) {
  ResidentGate& gate = resident_gate();
  std::lock_guard<std::mutex> lock(gate.mutex);
  return gate_leave(gate, (hipStream_t)stream);
}

int tri_fold_stats(const float* q_mean_real, const float* q_mean_imag, const float* q_abs_mean,
                   const float* freq_scale_sq, int32_t num_layers, int32_t num_score_heads,
                   int32_t num_pairs, int32_t disable_mlr, int32_t disable_trig, float* folded,
                   void* stream) {
  if (!q_mean_real || !q_mean_imag || !q_abs_mean || !freq_scale_sq || !folded)
    return fail(TRI_ERR_INVALID_ARGUMENT, "tri_fold_stats: NULL pointer");
  if (num_layers <= 0 || num_score_heads <= 0 || num_pairs <= 0)
    return fail(TRI_ERR_INVALID_ARGUMENT, "tri_fold_stats: bad sizes (%d, %d, %d)", num_layers, num_score_heads, num_pairs);
  return launch_status(tri::launch_fold_stats(q_mean_real, q_mean_imag, q_abs_mean, freq_scale_sq, num_layers,
                                              num_score_heads, num_pairs, disable_mlr, disable_trig, folded,
                                              (hipStream_t)stream),
                       "fold_stats");
}

uint64_t tri_workspace_bytes(const tri_kv_layout* kv, const tri_batch* batch, const tri_score_params* sp) {
  if (check_layout(kv, false) || check_batch(batch, false) || !sp || sp->num_score_heads <= 0 ||
      sp->num_offsets <= 0)
    return 0;
  return (uint64_t)plan(kv, batch, sp).total;
}

uint64_t tri_workspace_status_offset(const tri_kv_layout* kv, const tri_batch* batch,
                                     const tri_score_params* sp) {
  if (check_layout(kv, false) || check_batch(batch, false) || !sp || sp->num_score_heads <= 0 ||
      sp->num_offsets <= 0)
    return 0;
  return (uint64_t)plan(kv, batch, sp).status;
}

int tri_score_paged(const tri_kv_layout* kv, const tri_batch* batch, const tri_score_params* sp,
                    float* raw, int64_t raw_stride_layer, int64_t raw_stride_token,
                    int64_t raw_stride_head, void* workspace, uint64_t workspace_bytes, void* stream) {
  int rc = check_layout(kv, false);
  if (rc) return rc;
  rc = check_batch(batch, false);
  if (rc) return rc;
  rc = check_score(kv, sp);
  if (rc) return rc;
  if (!batch->round_start) return fail(TRI_ERR_INVALID_ARGUMENT, "round_start is NULL");
  if (!raw) return fail(TRI_ERR_INVALID_ARGUMENT, "raw is NULL");
  const tri::Workspace w = plan(kv, batch, sp);
  rc = check_workspace(w, workspace, workspace_bytes);
  if (rc) return rc;
  return do_score(kv, batch, sp, raw, raw_stride_layer, raw_stride_token, raw_stride_head, workspace, w,
                  (hipStream_t)stream, 0, at<float>(workspace, w.partial), nullptr);
}

int tri_select(const tri_kv_layout* kv, const tri_batch* batch, const tri_score_params* sp,
               const tri_select_params* sel, const float* raw, int64_t raw_stride_layer,
               int64_t raw_stride_token, int64_t raw_stride_head, float* final_scores, int32_t* keep,
               void* workspace, uint64_t workspace_bytes, void* stream) {
  int rc = check_layout(kv, false);
  if (rc) return rc;
  rc = check_batch(batch, true);
  if (rc) return rc;
  if (!sp || sp->num_score_heads <= 0 || sp->num_score_heads % kv->num_kv_heads || sp->num_offsets <= 0)
    return fail(TRI_ERR_INVALID_ARGUMENT, "tri_select: bad score params");
  rc = check_select(sel);
  if (rc) return rc;
  if (!raw || !keep) return fail(TRI_ERR_INVALID_ARGUMENT, "raw / keep is NULL");
  const tri::Workspace w = plan(kv, batch, sp);
  rc = check_workspace(w, workspace, workspace_bytes);
  if (rc) return rc;
  return do_select(kv, batch, sp, sel, raw, raw_stride_layer, raw_stride_token, raw_stride_head, final_scores,
                   keep, workspace, w, (hipStream_t)stream, 0, at<float>(workspace, w.partial), 0);
}

int tri_select_paged(const tri_kv_layout* kv, const tri_batch* batch, const tri_score_params* sp,
                     const tri_select_params* sel, float* final_scores, int32_t* keep, void* workspace,
                     uint64_t workspace_bytes, void* stream) {
  int rc = check_layout(kv, false);
  if (rc) return rc;
  rc = check_batch(batch, true);
  if (rc) return rc;
  rc = check_score(kv, sp);
  if (rc) return rc;
  rc = check_select(sel);
  if (rc) return rc;
  if (!batch->round_start) return fail(TRI_ERR_INVALID_ARGUMENT, "round_start is NULL");
  if (!keep && !final_scores) return fail(TRI_ERR_INVALID_ARGUMENT, "keep and final_scores are both NULL");
  const tri::Workspace w = plan(kv, batch, sp);
  rc = check_workspace(w, workspace, workspace_bytes);
  if (rc) return rc;
  return do_select_paged(kv, batch, sp, sel, final_scores, keep, workspace, w, (hipStream_t)stream);
}

int tri_select_path(const tri_kv_layout* kv, const tri_batch* batch, const tri_score_params* sp,
                    const tri_select_params* sel) {
  if (check_layout(kv, false) || check_batch(batch, false) || check_score(kv, sp) || check_select(sel)) return -1;
  const tri::Workspace w = plan(kv, batch, sp);
  return takes_resident(w, kv, sel) ? w.fused.eligible : 0;
}

int tri_describe_plan(const tri_kv_layout* kv, const tri_batch* batch, const tri_score_params* sp,
                      const tri_select_params* sel, int32_t assume_resident_workgroups, tri_plan_info* out) {
  if (!out) return fail(TRI_ERR_INVALID_ARGUMENT, "tri_describe_plan: out is NULL");
  if (assume_resident_workgroups < 0)
    return fail(TRI_ERR_INVALID_ARGUMENT, "assume_resident_workgroups %d", assume_resident_workgroups);
  int rc = check_layout(kv, false);
  if (!rc) rc = check_batch(batch, false);
  if (!rc) rc = check_score(kv, sp);
  if (!rc) rc = check_select(sel);
  if (rc) return rc;
  const tri::Workspace w = plan(kv, batch, sp, assume_resident_workgroups);
  *out = tri_plan_info{};
  out->workspace_bytes = w.total;
  out->layer_groups = 1;
  out->layers_per_group = kv->num_layers;
  if (!takes_resident(w, kv, sel)) return TRI_OK;
  const tri::FusedPlan& f = w.fused;
  out->path = f.eligible;
  out->tile_tokens = f.tile_tokens;
  out->tiles_per_seq = f.tiles_per_seq;
  out->resident_workgroups = (f.eligible == 2 && f.waves == 4) ? f.resident / 2 : f.resident;
  out->waves_per_workgroup = f.eligible == 2 ? f.waves : 8;
  if (f.eligible == 2 && f.layer_groups > 1) {
    out->layer_groups = f.layer_groups;
    out->layers_per_group = f.layers_per_group;
  }
  if (batch->num_seqs <= f.seqs_per_launch) out->launches = 1;
  else out->launches = f.launches;      // > 0: the planner replayed the packing of the host's lengths
  return TRI_OK;
}

int tri_small_launches(const tri_kv_layout* kv, const tri_batch* batch, const tri_score_params* sp,
                       const tri_select_params* sel, int32_t assume_resident_workgroups) {
  if (check_layout(kv, false) || check_batch(batch, false) || check_score(kv, sp) || check_select(sel)) return -1;
  if (assume_resident_workgroups < 0) {
    fail(TRI_ERR_INVALID_ARGUMENT, "assume_resident_workgroups %d", assume_resident_workgroups);
    return -1;
  }
  return takes_small(plan(kv, batch, sp, assume_resident_workgroups), kv, batch, sp, sel) ? 1 : 0;
}

int32_t tri_score_tile_tokens(const tri_kv_layout* kv, int32_t num_seqs, int32_t max_seq_len, int32_t num_score_heads,
                              int32_t aggregation) {
  if (check_layout(kv, false) || num_seqs <= 0 || max_seq_len <= 0 || num_score_heads <= 0 ||
      num_score_heads % kv->num_kv_heads)
    return 0;
  return takes_quarter_tiles(kv, num_seqs, max_seq_len, num_score_heads, aggregation) ? tri::kScoreFineTokens
                                                                                      : tri::kScoreTileTokens;
}

int tri_topk_rows(const float* scores, int64_t row_pitch, int32_t num_rows, const int32_t* row_lens,
                  const int32_t* row_ks, int32_t rows_per_entry, int32_t max_len, int32_t* keep,
                  int32_t keep_pitch, void* stream) {
  if (!scores || !row_lens || !row_ks || !keep) return fail(TRI_ERR_INVALID_ARGUMENT, "tri_topk_rows: NULL pointer");
  if (num_rows < 0 || rows_per_entry <= 0 || row_pitch < max_len || keep_pitch <= 0 || max_len <= 0)
    return fail(TRI_ERR_INVALID_ARGUMENT, "tri_topk_rows: bad sizes");
  return launch_status(tri::launch_topk_rows(scores, row_pitch, num_rows, row_lens, row_ks, rows_per_entry, max_len, keep,
                                             keep_pitch, (hipStream_t)stream),
                       "topk_rows");
}

namespace {

// Workgroups of 128 tokens and a head up to which a dense call goes through the small launch's kernels (8 heads: 600 tokens
// 38 -> 21 us, 4096 44 -> 21, 9000 56 -> 35, 16384 52 -> 37, of 256 elements 57 -> 49; 128 heads of 256 x 2048 tokens 100 -> 98; longer rows
// do not fit the selection's registers).
constexpr int64_t kDenseSmallWorkgroups = 2048;

// A dense call as the general layout, batch and parameters, on a workspace whose last part holds what those
// point to.
struct DensePlan {
  tri_kv_layout kv{};
  tri_batch batch{};
  tri_score_params sp{};
  tri_select_params sel{};
  tri::Workspace w{};
  int64_t arg_key, arg_words, folded, keep32, total;
};

int plan_dense(const tri_dense_params* p, DensePlan& d) {
  if (!p) return fail(TRI_ERR_INVALID_ARGUMENT, "dense params are NULL");
  if (p->kv_dtype != TRI_KV_BF16 && p->kv_dtype != TRI_KV_FP16)
    return fail(TRI_ERR_UNSUPPORTED, "tri_dense_compress takes two-byte keys, got kv_dtype %d", p->kv_dtype);
  if (p->num_tokens <= 0 || p->budget <= 0 || p->budget > p->num_tokens)
    return fail(TRI_ERR_INVALID_ARGUMENT, "budget %d of %d tokens", p->budget, p->num_tokens);
  if (p->k_stride_head % 2 || p->k_stride_token % 2)
    return fail(TRI_ERR_INVALID_ARGUMENT, "key strides must be whole elements");
  d.kv.num_layers = 1; d.kv.num_kv_heads = p->num_heads; d.kv.head_dim = p->head_dim; d.kv.block_size = p->num_tokens;
  d.kv.kv_dtype = p->kv_dtype; d.kv.rope_style = p->rope_style;
  d.kv.stride_block = p->k_stride_head / 2 * p->num_heads;          // one sequence: never used as a distance
  d.kv.stride_token = p->k_stride_token / 2; d.kv.stride_head = p->k_stride_head / 2;
  d.batch.num_seqs = 1; d.batch.max_seq_len = p->num_tokens; d.batch.max_budget = p->budget;
  d.sp.num_score_heads = p->num_heads; d.sp.num_offsets = p->num_offsets; d.sp.aggregation = p->aggregation;
  d.sel.normalize = p->normalize ? 1 : 0; d.sel.window_size = p->window_size;
  d.sel.group_reduce = TRI_REDUCE_MAX; d.sel.layer_reduce = TRI_REDUCE_MEAN;
  d.sel.group_first = 1; d.sel.no_resident = 1;
  if (p->num_heads <= 0 || p->num_heads > 256 ||
      (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256) || p->num_offsets <= 0)
    return fail(TRI_ERR_UNSUPPORTED, "%d heads of %d, %d offsets", p->num_heads, p->head_dim, p->num_offsets);
  d.w = plan(&d.kv, &d.batch, &d.sp, 0, false);
  int64_t off = d.w.total;
  auto take = [&](int64_t bytes) { const int64_t o = off; off = tri::align_up(off + bytes, 256); return o; };
  d.arg_key = take(8);
  d.arg_words = take(12);
  d.folded = take((int64_t)p->num_heads * 3 * (p->head_dim / 2) * 4);
  d.keep32 = take((int64_t)p->num_heads * p->budget * 4);
  d.total = off;
  return TRI_OK;
}

}  // namespace

uint64_t tri_dense_workspace_bytes(const tri_dense_params* params) {
  DensePlan d;
  return plan_dense(params, d) ? 0 : (uint64_t)d.total;
}

int tri_dense_compress(const tri_dense_params* p, void* ws, uint64_t ws_bytes, void* stream) {
  DensePlan d;
  int rc = plan_dense(p, d);
  if (rc) return rc;
  tri::Workspace need = d.w;
  need.total = d.total;
  rc = check_workspace(need, ws, ws_bytes);
  if (rc) return rc;
  if (!p->k || !p->v || !p->q_mean_complex || !p->q_abs_mean || !p->freq_scale_sq || !p->out_k || !p->out_v || !p->out_keep)
    return fail(TRI_ERR_INVALID_ARGUMENT, "tri_dense_compress: NULL pointer");
  if (!is_aligned(p->k, 16) || !is_aligned(p->v, 16) || !is_aligned(p->out_k, 16) || !is_aligned(p->out_v, 16))
    return fail(TRI_ERR_INVALID_ARGUMENT, "tri_dense_compress: bases must be 16-byte aligned");
  if (p->v_row_bytes <= 0 || p->v_row_bytes % 16 || p->v_stride_head % 16 || p->v_stride_token % 16 ||
      p->k_stride_head % 16 || p->k_stride_token % 16)
    return fail(TRI_ERR_INVALID_ARGUMENT, "tri_dense_compress: rows and strides must be multiples of 16 bytes");
  d.kv.k_layers = at<const void*>(ws, d.arg_key);
  int32_t* words = at<int32_t>(ws, d.arg_words);
  d.batch.seq_lens = words; d.batch.round_start = words + 1; d.batch.budgets = words + 2;
  d.sp.folded = at<float>(ws, d.folded); d.sp.omega = p->omega; d.sp.offsets = p->offsets;
  rc = check_layout(&d.kv, false);
  if (!rc) rc = check_batch(&d.batch, true);
  if (!rc) rc = check_score(&d.kv, &d.sp);
  if (!rc) rc = check_select(&d.sel);
  if (rc) return rc;
  tri::DenseLaunch l{};
  l.k = p->k; l.v = p->v;
  l.k_stride_head = p->k_stride_head; l.k_stride_token = p->k_stride_token;
  l.v_stride_head = p->v_stride_head; l.v_stride_token = p->v_stride_token;
  l.k_row_bytes = p->head_dim * 2; l.v_row_bytes = p->v_row_bytes;
  l.H = p->num_heads; l.T = p->num_tokens; l.D = p->head_dim; l.budget = p->budget; l.round_start = p->round_start;
  l.disable_mlr = p->disable_mlr; l.disable_trig = p->disable_trig;
  l.q_mean = p->q_mean_complex; l.q_abs = p->q_abs_mean; l.freq_scale = p->freq_scale_sq;
  l.out_k = p->out_k; l.out_v = p->out_v; l.out_keep = p->out_keep;
  l.folded = at<float>(ws, d.folded); l.arg_key = at<const void*>(ws, d.arg_key); l.arg_words = words;
  l.keep32 = at<int32_t>(ws, d.keep32);
  hipStream_t s = (hipStream_t)stream;
  // (NaN scores stay NaN, the largest of a row or, with the sign set, the smallest: torch's normalisation and
  // tri_topk_rows, which this call stands for, treat them so)
  if (p->aggregation == TRI_REDUCE_MEAN && tri::select_small_takes(p->num_tokens, 1) &&
      (int64_t)p->num_heads * tri::ceil_div(p->num_tokens, 128) <= kDenseSmallWorkgroups) {
    // Three launches: the scorer takes the call's arguments by value and folds the statistics itself.
    tri::SmallScore c{};
    c.k = p->k; c.round = p->round_start;
    c.q_mean = p->q_mean_complex; c.q_abs = p->q_abs_mean; c.freq_scale = p->freq_scale_sq;
    c.disable_mlr = p->disable_mlr; c.disable_trig = p->disable_trig;
    c.omega = p->omega; c.offsets = p->offsets; c.NO = p->num_offsets;
    c.raw = at<float>(ws, d.w.raw); c.raw_pitch = p->num_tokens;
    c.stride_token = d.kv.stride_token; c.stride_head = d.kv.stride_head;
    c.L = 1; c.A = p->num_heads; c.G = 1; c.Tmax = p->num_tokens; c.block_size = p->num_tokens;
    rc = launch_status(tri::launch_score_small(c, 1, p->num_heads, p->head_dim, p->kv_dtype, p->rope_style, s), "score_small");
    if (rc) return rc;
    tri::SmallSelect a{};
    a.raw = c.raw; a.raw_pitch = c.raw_pitch; a.keep = at<int32_t>(ws, d.keep32); a.keep_pitch = p->budget;
    a.L = 1; a.Hkv = p->num_heads; a.A = p->num_heads; a.G = 1; a.Tmax = p->num_tokens;
    a.normalize = d.sel.normalize; a.window_size = d.sel.window_size;
    a.group_reduce = TRI_REDUCE_MAX; a.layer_reduce = TRI_REDUCE_MEAN; a.pass_nan = 1;
    rc = launch_status(tri::launch_select_small(a, 1, s), "select_small");
    if (rc) return rc;
    return launch_status(tri::launch_dense_gather(l, s), "dense gather");
  }
  rc = launch_status(tri::launch_dense_prologue(l, s), "dense prologue");
  if (rc) return rc;
  rc = do_select_paged(&d.kv, &d.batch, &d.sp, &d.sel, nullptr, at<int32_t>(ws, d.keep32), ws, d.w, s, 1);
  if (rc) return rc;
  return launch_status(tri::launch_dense_gather(l, s), "dense gather");
}

int tri_compact_paged(const tri_kv_layout* kv, const tri_batch* batch, const int32_t* keep,
                      int32_t keep_per_layer, int32_t shared, void* stream) {
  tri::CompactLaunch a{};
  const int rc = fill_compact(kv, batch, keep, keep_per_layer, shared, a);
  if (rc) return rc;
  return launch_status(tri::launch_compact(a, (hipStream_t)stream), "compact");
}

uint64_t tri_compact_full_staging_bytes(const tri_kv_layout* kv, const tri_batch* batch) {
  if (check_layout(kv, true) || check_batch(batch, false)) return 0;
  // one layer: K and V of every head row of every logical slot of every sequence
  return (uint64_t)batch->num_seqs * 2 * kv->num_kv_heads * (uint64_t)batch->max_seq_len * kv->head_dim *
         elem_bytes(kv->kv_dtype);
}

int tri_compact_paged_full(const tri_kv_layout* kv, const tri_batch* batch, const int32_t* keep,
                           int32_t keep_per_layer, int32_t shared, void* staging, uint64_t staging_bytes,
                           void* stream) {
  tri::CompactLaunch a{};
  const int rc = fill_compact(kv, batch, keep, keep_per_layer, shared, a);
  if (rc) return rc;
  if (a.has_scales) return fail(TRI_ERR_UNSUPPORTED, "full-permutation compaction of fp8 caches is not built");
  if (!staging || !is_aligned(staging, 16)) return fail(TRI_ERR_WORKSPACE, "staging is NULL or unaligned");
  if (staging_bytes < tri_compact_full_staging_bytes(kv, batch))
    return fail(TRI_ERR_WORKSPACE, "staging has %llu bytes, %llu needed", (unsigned long long)staging_bytes,
                (unsigned long long)tri_compact_full_staging_bytes(kv, batch));
  a.staging = staging;
  return launch_status(tri::launch_compact_full(a, (hipStream_t)stream), "compact_full");
}

int tri_compress_step(const tri_kv_layout* kv, const tri_batch* batch, const tri_score_params* sp,
                      const tri_select_params* sel, int32_t* keep, void* workspace,
                      uint64_t workspace_bytes, void* stream) {
  int rc = check_layout(kv, true);
  if (rc) return rc;
  rc = check_batch(batch, true);
  if (rc) return rc;
  rc = check_score(kv, sp);
  if (rc) return rc;
  rc = check_select(sel);
  if (rc) return rc;
  if (!batch->round_start) return fail(TRI_ERR_INVALID_ARGUMENT, "round_start is NULL");
  if (!batch->block_table) return fail(TRI_ERR_INVALID_ARGUMENT, "tri_compress_step needs a block table");
  if (!keep) return fail(TRI_ERR_INVALID_ARGUMENT, "keep is NULL");
  const tri::Workspace w = plan(kv, batch, sp);
  rc = check_workspace(w, workspace, workspace_bytes);
  if (rc) return rc;
  hipStream_t s = (hipStream_t)stream;
  rc = do_select_paged(kv, batch, sp, sel, nullptr, keep, workspace, w, s);
  if (rc) return rc;
  tri::CompactLaunch c{};
  rc = fill_compact(kv, batch, keep, sel->layer_reduce < 0, sel->shared, c);
  if (rc) return rc;
  // A resident kernel whose bounded wait expired leaves meaningless keep lists and a raised
  // status word: the compaction kernels look at that word and then leave the cache alone.
  c.guard = at<uint32_t>(workspace, w.status);
  return launch_status(tri::launch_compact(c, s), "compact");
}

int tri_compress_step_static(const tri_kv_layout* kv, const tri_batch* batch, const tri_score_params* sp,
                             const tri_select_params* sel, int32_t* keep, const uint32_t** status_out,
                             void* stream) {
  int rc = check_layout(kv, true);
  if (rc) return rc;
  rc = check_batch(batch, true);
  if (rc) return rc;
  rc = check_score(kv, sp);
  if (rc) return rc;
  rc = check_select(sel);
  if (rc) return rc;
  if (!batch->round_start) return fail(TRI_ERR_INVALID_ARGUMENT, "round_start is NULL");
  if (!batch->block_table) return fail(TRI_ERR_INVALID_ARGUMENT, "tri_compress_step_static needs a block table");
  if (!keep) return fail(TRI_ERR_INVALID_ARGUMENT, "keep is NULL");
  // Always the score-then-select kernels, so the scratch is sized for them alone (a resident plan
  // would add its coefficient slabs and exchange words; the status word sits at the same offset).
  const tri::Workspace w = plan(kv, batch, sp, 0, false);
  if ((uint64_t)w.total > (uint64_t)TRI_STATIC_WORKSPACE_BYTES)
    return fail(TRI_ERR_WORKSPACE, "this step needs %lld bytes of scratch, the library's static array holds %llu; "
                "use tri_compress_step with a workspace of the caller's", (long long)w.total,
                (unsigned long long)TRI_STATIC_WORKSPACE_BYTES);
  void* ws = nullptr;
  rc = static_scratch(&ws);
  if (rc) return rc;
  if (status_out) *status_out = at<uint32_t>(ws, w.status);
  tri_select_params two_pass = *sel;
  two_pass.no_resident = 1;   // the resident path chains its launches with an event it creates
  hipStream_t s = (hipStream_t)stream;
  rc = do_select_paged(kv, batch, sp, &two_pass, nullptr, keep, ws, w, s);
  if (rc) return rc;
  tri::CompactLaunch c{};
  rc = fill_compact(kv, batch, keep, sel->layer_reduce < 0, sel->shared, c);
  if (rc) return rc;
  c.guard = at<uint32_t>(ws, w.status);
  c.no_side_stream = 1;
  return launch_status(tri::launch_compact(c, s), "compact");
}

namespace {

// How a call of attend_kernel is cut, and what it needs of the workspace.
struct AttendPlan {
  tri::AttendLaunch a{};
  int64_t part_out, part_ml, lse2, scores, q_copy, total;
  // block selection
  int64_t block_scores, counts;
  int max_count;
  bool weigh_again, copies_q;
};

constexpr int kMaxNewTokens = 64;          // a word of ancestors
// Workgroups of an attention kernel that a CU holds, by its registers.
int attend_workgroups_per_cu(int row_tiles, int D) {
  if (row_tiles == 0) return D == 64 ? 4 : D == 128 ? 2 : 1;
  if (row_tiles == 4) return D == 64 ? 4 : 2;
  return 1;
}

// The bytes that rows of heads span.
struct Span {
  intptr_t from, to;
};
Span span_of(const void* p, int64_t rows, int64_t stride_row, int64_t heads, int64_t stride_head, int D) {
  const int64_t r = (rows - 1) * stride_row, h = (heads - 1) * stride_head;
  const intptr_t at = reinterpret_cast<intptr_t>(p);
  return {at + (std::min<int64_t>(r, 0) + std::min<int64_t>(h, 0)) * 2, at + (std::max<int64_t>(r, 0) + std::max<int64_t>(h, 0) + D) * 2};
}

bool is_finite(float x) { return x - x == 0.f; }

int plan_attend(const tri_kv_layout* kv, const tri_batch* batch, const tri_attend_params* p, const tri_block_params* bp,
                AttendPlan& d) {
  int rc = check_layout(kv, true);
  if (!rc) rc = check_batch(batch, false);
  if (rc) return rc;
  if (!p) return fail(TRI_ERR_INVALID_ARGUMENT, "attention params are NULL");
  if (p->layer < 0 || p->layer >= kv->num_layers) return fail(TRI_ERR_INVALID_ARGUMENT, "layer %d of %d", p->layer, kv->num_layers);
  if (p->num_q_heads <= 0 || p->num_q_heads % kv->num_kv_heads)
    return fail(TRI_ERR_INVALID_ARGUMENT, "num_q_heads %d is not a multiple of num_kv_heads %d", p->num_q_heads, kv->num_kv_heads);
  if (p->q_dtype != TRI_KV_BF16 && p->q_dtype != TRI_KV_FP16)
    return fail(TRI_ERR_UNSUPPORTED, "q_dtype %d (bf16 or fp16 queries)", p->q_dtype);
  if (kv->kv_dtype != TRI_KV_FP8_E4M3 && p->q_dtype != kv->kv_dtype)
    return fail(TRI_ERR_UNSUPPORTED, "queries of type %d over a cache of type %d", p->q_dtype, kv->kv_dtype);
  if (p->num_blocks <= 0) return fail(TRI_ERR_INVALID_ARGUMENT, "num_blocks %d", p->num_blocks);
  if (p->max_rows < 1 || p->max_rows > kMaxNewTokens)
    return fail(TRI_ERR_UNSUPPORTED, "max_rows %d not in [1, %d]", p->max_rows, kMaxNewTokens);
  if (p->num_rows < 0 || p->num_rows > INT_MAX / p->num_q_heads) return fail(TRI_ERR_INVALID_ARGUMENT, "num_rows %d", p->num_rows);
  if (!p->row_starts && (p->num_rows != batch->num_seqs || p->max_rows != 1 || p->parents))
    return fail(TRI_ERR_INVALID_ARGUMENT, "without row_starts there is one row per sequence (%d rows of at most %d, %d sequences) and no parents",
                p->num_rows, p->max_rows, batch->num_seqs);
  if (p->q_stride_row % 8 || p->q_stride_head % 8 || p->out_stride_row % 8 || p->out_stride_head % 8)
    return fail(TRI_ERR_INVALID_ARGUMENT, "strides of q and out must be multiples of 8 elements (16 bytes)");
  if (p->num_q_heads > 1 && p->out_stride_head < kv->head_dim)
    return fail(TRI_ERR_INVALID_ARGUMENT, "out_stride_head %lld < head_dim", (long long)p->out_stride_head);
  if (p->num_rows > 1 && p->out_stride_row < kv->head_dim)
    return fail(TRI_ERR_INVALID_ARGUMENT, "out_stride_row %lld < head_dim", (long long)p->out_stride_row);
  if (!is_finite(p->scale) || !is_finite(p->k_scale) || !is_finite(p->v_scale) || !is_finite(p->scale * p->k_scale * 1.44269504f))
    return fail(TRI_ERR_INVALID_ARGUMENT, "scale, k_scale and v_scale must be finite");
  if (!(p->scale * p->k_scale > 0.f)) return fail(TRI_ERR_INVALID_ARGUMENT, "scale * k_scale must be positive");
  // (in-block offsets of the rows a wave reads together are 32-bit)
  if (kv->stride_token < 0 || kv->stride_token >= (1 << 25))
    return fail(TRI_ERR_UNSUPPORTED, "stride_token %lld", (long long)kv->stride_token);
  if (p->weight_mode != 0 && p->weight_mode != 1) return fail(TRI_ERR_INVALID_ARGUMENT, "weight_mode %d", p->weight_mode);
  if (bp) {
    if (p->row_starts || p->parents || p->weights)
      return fail(TRI_ERR_UNSUPPORTED, "attention over chosen blocks takes one row per sequence and adds up no weights");
    if (bp->top_blocks <= 0 || bp->sink_blocks < 0 || bp->recent_blocks < 0 ||
        (int64_t)bp->sink_blocks + bp->recent_blocks > bp->top_blocks)
      return fail(TRI_ERR_INVALID_ARGUMENT, "%d sink and %d recent blocks of %d", bp->sink_blocks, bp->recent_blocks, bp->top_blocks);
    if (bp->group_reduce != TRI_REDUCE_MEAN && bp->group_reduce != TRI_REDUCE_MAX)
      return fail(TRI_ERR_INVALID_ARGUMENT, "group_reduce %d", bp->group_reduce);
  }
  tri::AttendLaunch& a = d.a;
  a.B = batch->num_seqs; a.Hkv = kv->num_kv_heads; a.Hq = p->num_q_heads; a.G = a.Hq / a.Hkv; a.D = kv->head_dim;
  a.block_size = kv->block_size; a.kv_dtype = kv->kv_dtype; a.q_dtype = p->q_dtype; a.layer = p->layer;
  a.Tmax = batch->max_seq_len; a.num_blocks = p->num_blocks;
  a.stride_block = kv->stride_block; a.stride_token = kv->stride_token; a.stride_head = kv->stride_head;
  a.k_layers = kv->k_layers; a.v_layers = kv->v_layers;
  if (kv->kv_dtype == TRI_KV_FP8_E4M3 && kv->v_scale_layers) {
    a.k_scale_layers = kv->k_scale_layers;
    a.v_scale_layers = kv->v_scale_layers;
  }
  a.div_shift = 31;
  while ((1ll << (a.div_shift - 31)) < a.block_size) ++a.div_shift;
  a.div_factor = (uint32_t)(((1ull << a.div_shift) + a.block_size - 1) / a.block_size);
  a.block_table = batch->block_table; a.block_table_pitch = batch->block_table_pitch; a.seq_lens = batch->seq_lens;
  a.q = p->q; a.q_stride_row = p->q_stride_row; a.q_stride_head = p->q_stride_head;
  a.out = p->out; a.out_stride_row = p->out_stride_row; a.out_stride_head = p->out_stride_head; a.lse = p->lse;
  a.row_starts = p->row_starts; a.parents = p->parents; a.num_rows = p->num_rows; a.max_rows = p->max_rows;
  a.scale_log2 = p->scale * p->k_scale * 1.44269504088896340736f;
  a.v_scale = p->v_scale;
  // Blocks and tokens a sequence has at most, and tokens of the batch.
  d.max_count = tri::ceil_div(a.Tmax, a.block_size);
  const int64_t chosen = bp ? (int64_t)std::min(bp->top_blocks, d.max_count) * a.block_size : INT_MAX;
  if (bp && chosen > INT_MAX / 2) return fail(TRI_ERR_UNSUPPORTED, "%d blocks of %d tokens", bp->top_blocks, a.block_size);
  const int64_t longest = std::min<int64_t>(bp ? chosen : a.Tmax, bp ? (int64_t)d.max_count * a.block_size : a.Tmax);
  int64_t total = 0;
  for (int b = 0; b < a.B; ++b) total += std::min<int64_t>(batch->seq_lens_host ? batch->seq_lens_host[b] : a.Tmax, longest);
  const int rows = a.max_rows * a.G;
  // Tiles of 16 rows a workgroup has room for: 8 x 4096 tokens of 8 x 128 bf16, a call with four, eight and sixteen of them: 80 rows
  // 53, 41, 42 us; 128 rows 57, 46, 45; 160 rows 89, 70, 52; 256 rows 94, 74, 61; of 64 dimensions 128 rows 38, 30, 33, 256 rows
  // 59, 47, 41.  Of up to 64 rows four leave the scores that weights come from and hold weights as two numbers (softmax32); calls that
  // want neither would gain from eight, of which waves without rows still load (64 rows 42, 37, 41).  (256 dimensions have no sixteen:
  // registers.)
  a.row_tiles = rows <= 16 ? 0 : rows <= 64 ? 4 : rows <= 128 || a.D == 256 ? 8 : 16;
  a.row_blocks = a.row_tiles ? tri::ceil_div(rows, 16 * a.row_tiles) : 1;
  // A split is as long as lets every workgroup run at once (each sequence's last one is short); with more sequences than that
  // allows, what a workgroup has to do on the mean, so that a long one among short ones is still cut.
  const int64_t holds = 256 * attend_workgroups_per_cu(a.row_tiles, a.D);
  auto length = [&](int64_t inner, int step) {
    const int64_t most = tri::align_up(longest, step), cap = holds / inner;
    int64_t lo = std::min<int64_t>(tri::align_up(std::max<int64_t>(tri::ceil_div64(total * inner, holds), 1), step), most);
    if (cap <= a.B) return (int)lo;
    int64_t hi = std::min(tri::align_up(std::max<int64_t>(tri::ceil_div64(total, cap - a.B), 1), step), most);      // (surely fits)
    while (lo < hi) {
      const int64_t mid = lo + (hi - lo) / step / 2 * step;
      int64_t count = 0;
      for (int b = 0; b < a.B; ++b)
        count += std::max<int64_t>(1, tri::ceil_div64(std::min<int64_t>(batch->seq_lens_host ? batch->seq_lens_host[b] : a.Tmax, longest), mid));
      if (count <= cap) hi = mid;
      else lo = mid + step;
    }
    return (int)hi;
  };
  // Few rows of long sequences: a workgroup takes four KV heads, a wave each.  Its waves then read neighbouring rows, a token's
  // heads lie side by side, and have nothing to join: 16 x 16384 tokens of fp8 114 us against 125 with four waves to a head, 24
  // ragged ones of up to 8192 with 64 dimensions 48 against 55.  The splits are a quarter as long, which has to leave a wave
  // enough to do: at 128 tokens a split 1 x 32768 of 128 dimensions take 42 us against 37, at 256 the two are level (rows of up
  // to 128 bytes gain from 128 tokens on: 41 us against 45 for 64 x 1024).
  a.heads_per_group = 1;
  const int row_bytes = a.D * (a.kv_dtype == TRI_KV_FP8_E4M3 ? 1 : 2);
  if (a.row_tiles == 0 && a.Hkv % 4 == 0 && a.block_size % 16 == 0) {
    a.split_tokens = length(a.Hkv / 4, 32);
    if (a.split_tokens >= (row_bytes <= 128 ? 128 : 256)) a.heads_per_group = 4;
  }
  // (128: whole tiles of every kernel; a single tile a workgroup saves the attention nothing and costs the join)
  if (a.heads_per_group == 1) a.split_tokens = length((int64_t)a.Hkv * a.row_blocks, 128);
  // (the partial results of all splits: at most 512 MiB, of one split where that alone is more)
  const int64_t part_bytes = (int64_t)a.B * a.Hkv * rows * (a.D + 2) * 4, parts_most = std::max<int64_t>((512ll << 20) / part_bytes, 1);
  if (tri::ceil_div64(longest, a.split_tokens) > parts_most) a.split_tokens = (int)tri::align_up(tri::ceil_div64(longest, parts_most), 128);
  a.nsplit = (int)tri::ceil_div64(longest, a.split_tokens);
  int64_t off = 0;
  auto take = [&](int64_t bytes) { const int64_t o = off; off = tri::align_up(off + bytes, 256); return o; };
  const int64_t parts = a.nsplit > 1 ? (int64_t)a.B * a.Hkv * a.nsplit * rows : 0;
  if ((int64_t)a.B * a.nsplit * a.row_blocks * a.Hkv > INT_MAX || (int64_t)a.B * tri::ceil_div(a.Tmax, 64) * a.Hkv > INT_MAX ||
      (int64_t)a.B * a.Hkv * rows > INT_MAX)
    return fail(TRI_ERR_UNSUPPORTED, "%d sequences of %d rows and %d KV heads in one call", a.B, a.max_rows, a.Hkv);
  a.score_pitch = tri::align_up(a.Tmax, 32);
  d.part_out = take(parts * a.D * 4);
  d.part_ml = take(parts * 8);
  // Weights of few rows come from their scores, which the attention leaves (8 bytes a row and token, written and read), of many
  // from the keys once more.  Calls on 2 x 32768 tokens of eight KV heads, from scores and from keys, us: 128 dimensions bf16, 16 rows
  // a KV head 84 and 100, 24 rows 97 and 103, 32 rows 105 and 104, 64 rows 152 and 115; fp8 16 rows 59 and 69, 32 rows 76 and 78,
  // 64 rows 111 and 91; 64 dimensions 16 rows 59 and 65, 24 rows 71 and 71, 32 rows 78 and 72 (fp8 with scales 76 and 76), 64 rows 103 and
  // 79; 256 dimensions 32 rows 161 and 171, 48 rows 181 and 182, 64 rows 208 and 193.
  // Scores of all sequences lie as far apart as the longest one's, so a long one among many short ones would take scratch without
  // end: beyond 2 GiB and all of the batch's K and V in this layer, which sequences of one length never need, the keys are read again
  // too.  One of 60000 tokens among 299 of 300, 64 query heads over 8 of 128: 4.6 GB of scores for 0.6 GB of K and V, 255 us; from
  // the keys 467.
  const int64_t score_bytes = (int64_t)a.B * a.Hkv * rows * a.score_pitch * 4;
  const int64_t cache_bytes = total * a.Hkv * a.D * 2 * elem_bytes(a.kv_dtype);
  d.weigh_again = p->weights && (rows > (a.D == 256 ? 64 : 32) || score_bytes > std::max<int64_t>(2ll << 30, cache_bytes));
  // (they read the queries again when out is written: out in q's memory is read from a copy)
  const Span of_q = span_of(p->q, a.num_rows, a.q_stride_row, a.Hq, a.q_stride_head, a.D);
  const Span of_out = span_of(p->out, a.num_rows, a.out_stride_row, a.Hq, a.out_stride_head, a.D);
  d.copies_q = d.weigh_again && a.num_rows > 0 && of_q.from < of_out.to && of_out.from < of_q.to;
  d.q_copy = take(d.copies_q ? (int64_t)a.num_rows * a.Hq * a.D * 2 : 0);
  d.lse2 = take(p->weights ? (int64_t)a.num_rows * a.Hq * 4 : 0);
  d.scores = take(p->weights && !d.weigh_again ? score_bytes : 0);
  d.block_scores = take(bp ? (int64_t)a.B * a.Hkv * d.max_count * 4 : 0);
  d.counts = take(bp ? (int64_t)a.B * 8 : 0);
  d.total = std::max<int64_t>(off, 256);
  return TRI_OK;
}

int check_attend_pointers(const tri_attend_params* p, const AttendPlan& d, void* ws, uint64_t ws_bytes) {
  if (p->num_rows > 0 && (!p->q || !p->out)) return fail(TRI_ERR_INVALID_ARGUMENT, "q / out is NULL");
  if (!is_aligned(p->q, 16) || !is_aligned(p->out, 16)) return fail(TRI_ERR_INVALID_ARGUMENT, "q and out must be 16-byte aligned");
  tri::Workspace need{};
  need.total = d.total;
  return check_workspace(need, ws, ws_bytes);
}

int do_attend(AttendPlan& d, void* ws, float* weights, int weight_mode, hipStream_t s) {
  tri::AttendLaunch& a = d.a;
  if (a.nsplit > 1) {
    a.part_out = at<float>(ws, d.part_out);
    a.part_ml = at<float>(ws, d.part_ml);
  }
  const bool again = d.weigh_again;
  if (again || (weights && a.nsplit == 1)) a.lse2 = at<float>(ws, d.lse2);
  if (weights && !again) a.scores = at<float>(ws, d.scores);
  int rc = TRI_OK;
  if (d.copies_q) rc = launch_status(tri::launch_copy_queries(a, at<void>(ws, d.q_copy), s), "copy_queries");
  if (!rc) rc = launch_status(tri::launch_attend(a, s), "attend");
  if (!rc) rc = launch_status(tri::launch_attend_finish(a, again ? nullptr : weights, weight_mode, s), "attend_finish");
  if (rc || !again) return rc;
  if (d.copies_q) {
    a.q = at<void>(ws, d.q_copy);
    a.q_stride_row = (int64_t)a.Hq * a.D;
    a.q_stride_head = a.D;
  }
  a.weigh = 1;
  a.weights = weights;
  a.weight_set = weight_mode;
  return launch_status(tri::launch_attend(a, s), "weigh_rows");
}

int fill_evict(const tri_kv_layout* kv, const tri_batch* batch, const tri_evict_params* p, int32_t* keep, tri::EvictLaunch& a) {
  int rc = check_layout(kv, false);
  if (!rc) rc = check_batch(batch, true);
  if (!rc) rc = check_pages(kv, batch);
  if (rc) return rc;
  if (!p) return fail(TRI_ERR_INVALID_ARGUMENT, "evict params are NULL");
  if (p->num_blocks <= 0) return fail(TRI_ERR_INVALID_ARGUMENT, "num_blocks %d", p->num_blocks);
  if (p->window_size < 0) return fail(TRI_ERR_INVALID_ARGUMENT, "window_size %d", p->window_size);
  if (p->layer_reduce != TRI_REDUCE_MEAN && p->layer_reduce != TRI_REDUCE_MAX && p->layer_reduce != -1)
    return fail(TRI_ERR_INVALID_ARGUMENT, "layer_reduce %d", p->layer_reduce);
  if (p->protect_prefill && !batch->prefill_lens) return fail(TRI_ERR_INVALID_ARGUMENT, "protect_prefill without prefill_lens");
  if (kv->num_layers > 1 && p->weights_stride_layer < (int64_t)p->num_blocks * kv->block_size * kv->num_kv_heads)
    return fail(TRI_ERR_INVALID_ARGUMENT, "weights_stride_layer %lld is less than a layer", (long long)p->weights_stride_layer);
  const int64_t width = std::max(batch->max_seq_len, batch->max_budget);
  if (tri::ceil_div64(width, 256) * tri::ceil_div(kv->num_kv_heads, 4) * batch->num_seqs * kv->num_layers > INT_MAX)
    return fail(TRI_ERR_UNSUPPORTED, "%d sequences of %d tokens and %d layers in one call", batch->num_seqs, batch->max_seq_len, kv->num_layers);
  a.B = batch->num_seqs; a.L = kv->num_layers; a.Hkv = kv->num_kv_heads; a.block_size = kv->block_size;
  a.Tmax = batch->max_seq_len; a.max_budget = batch->max_budget; a.num_blocks = p->num_blocks;
  a.window_size = p->window_size; a.protect_prefill = p->protect_prefill; a.layer_reduce = p->layer_reduce; a.shared = p->shared ? 1 : 0;
  a.block_table = batch->block_table; a.block_table_pitch = batch->block_table_pitch; a.seq_lens = batch->seq_lens;
  a.prefill_lens = batch->prefill_lens; a.budgets = batch->budgets;
  a.weights = p->weights; a.weights_stride_layer = p->weights_stride_layer; a.keep = keep;
  return TRI_OK;
}

int64_t evict_rows(const tri::EvictLaunch& a) { return (int64_t)a.B * (a.layer_reduce < 0 ? a.L : 1) * (a.shared ? 1 : a.Hkv); }

int do_select_by_weight(tri::EvictLaunch& a, const tri_evict_params* p, float* final_scores, void* ws, uint64_t ws_bytes, hipStream_t s) {
  if (!p->weights || !a.keep) return fail(TRI_ERR_INVALID_ARGUMENT, "weights / keep is NULL");
  tri::Workspace need{};
  need.total = tri::align_up(evict_rows(a) * a.Tmax * 4, 256);
  if (!final_scores) {
    const int rc = check_workspace(need, ws, ws_bytes);
    if (rc) return rc;
  }
  a.fin = final_scores ? final_scores : at<float>(ws, 0);
  int rc = launch_status(tri::launch_weight_rows(a, s), "weight_rows");
  if (rc) return rc;
  const int rows = (int)evict_rows(a);
  return launch_status(tri::launch_topk_rows(a.fin, a.Tmax, rows, a.seq_lens, a.budgets, rows / a.B, a.Tmax, a.keep, a.max_budget, s),
                       "topk_rows");
}

}  // namespace

uint64_t tri_attend_workspace_bytes(const tri_kv_layout* kv, const tri_batch* batch, const tri_attend_params* p) {
  AttendPlan d;
  return plan_attend(kv, batch, p, nullptr, d) ? 0 : (uint64_t)d.total;
}

int tri_attend_paged(const tri_kv_layout* kv, const tri_batch* batch, const tri_attend_params* p, void* ws, uint64_t ws_bytes,
                     void* stream) {
  AttendPlan d;
  int rc = plan_attend(kv, batch, p, nullptr, d);
  if (!rc) rc = check_attend_pointers(p, d, ws, ws_bytes);
  if (!rc) rc = check_pages(kv, batch);
  if (rc) return rc;
  if (p->num_rows == 0 && !p->weights) return TRI_OK;
  return do_attend(d, ws, p->weights, p->weight_mode, (hipStream_t)stream);
}

int tri_block_bounds(const tri_kv_layout* kv, const tri_batch* batch, int32_t num_blocks, int32_t new_tokens, void* bounds,
                     int64_t bounds_stride_layer, void* stream) {
  int rc = check_layout(kv, false);
  if (!rc) rc = check_batch(batch, false);
  if (!rc) rc = check_pages(kv, batch);
  if (rc) return rc;
  if (num_blocks <= 0 || new_tokens < 0) return fail(TRI_ERR_INVALID_ARGUMENT, "num_blocks %d, new_tokens %d", num_blocks, new_tokens);
  if (!bounds || !is_aligned(bounds, 16) || bounds_stride_layer % 8)
    return fail(TRI_ERR_INVALID_ARGUMENT, "bounds must be 16-byte aligned, layer by layer");
  if (kv->num_layers > 1 && bounds_stride_layer < (int64_t)num_blocks * kv->num_kv_heads * 2 * kv->head_dim)
    return fail(TRI_ERR_INVALID_ARGUMENT, "bounds_stride_layer %lld is less than a layer", (long long)bounds_stride_layer);
  const int64_t waves = tri::ceil_div(kv->num_kv_heads * (kv->head_dim / 8), 64);
  if ((int64_t)batch->num_seqs * kv->num_layers * tri::ceil_div(batch->max_seq_len, kv->block_size) * waves > INT_MAX)
    return fail(TRI_ERR_UNSUPPORTED, "%d sequences of %d tokens and %d layers in one call", batch->num_seqs, batch->max_seq_len, kv->num_layers);
  tri::BoundsLaunch a{};
  a.B = batch->num_seqs; a.L = kv->num_layers; a.Hkv = kv->num_kv_heads; a.D = kv->head_dim; a.block_size = kv->block_size;
  a.kv_dtype = kv->kv_dtype; a.Tmax = batch->max_seq_len; a.num_blocks = num_blocks; a.new_tokens = std::min(new_tokens, batch->max_seq_len);
  a.stride_block = kv->stride_block; a.stride_token = kv->stride_token; a.stride_head = kv->stride_head;
  a.k_layers = kv->k_layers;
  if (kv->kv_dtype == TRI_KV_FP8_E4M3 && kv->v_scale_layers) a.k_scale_layers = kv->k_scale_layers;
  a.block_table = batch->block_table; a.block_table_pitch = batch->block_table_pitch; a.seq_lens = batch->seq_lens;
  a.bounds = bounds; a.bounds_stride_layer = bounds_stride_layer;
  return launch_status(tri::launch_block_bounds(a, (hipStream_t)stream), "block_bounds");
}

uint64_t tri_attend_blocks_workspace_bytes(const tri_kv_layout* kv, const tri_batch* batch, const tri_attend_params* p,
                                           const tri_block_params* bp) {
  AttendPlan d;
  if (!bp) {
    fail(TRI_ERR_INVALID_ARGUMENT, "block params are NULL");
    return 0;
  }
  return plan_attend(kv, batch, p, bp, d) ? 0 : (uint64_t)d.total;
}

int tri_attend_blocks(const tri_kv_layout* kv, const tri_batch* batch, const tri_attend_params* p, const tri_block_params* bp,
                      void* ws, uint64_t ws_bytes, void* stream) {
  if (!bp) return fail(TRI_ERR_INVALID_ARGUMENT, "block params are NULL");
  AttendPlan d;
  int rc = plan_attend(kv, batch, p, bp, d);
  if (!rc) rc = check_attend_pointers(p, d, ws, ws_bytes);
  if (!rc) rc = check_pages(kv, batch);
  if (rc) return rc;
  if (!bp->bounds || !bp->blocks || !is_aligned(bp->bounds, 16))
    return fail(TRI_ERR_INVALID_ARGUMENT, "bounds / blocks is NULL or bounds not 16-byte aligned");
  if ((int64_t)d.a.B * d.a.Hkv > INT_MAX / std::max(bp->top_blocks, 1))
    return fail(TRI_ERR_UNSUPPORTED, "%d sequences of %d blocks", d.a.B, bp->top_blocks);
  hipStream_t s = (hipStream_t)stream;
  tri::BlockScoreLaunch c{};
  c.B = d.a.B; c.Hkv = d.a.Hkv; c.G = d.a.G; c.D = d.a.D; c.block_size = d.a.block_size;
  c.bounds_dtype = kv->kv_dtype == TRI_KV_FP8_E4M3 ? TRI_KV_BF16 : kv->kv_dtype; c.q_dtype = p->q_dtype;
  c.Tmax = d.a.Tmax; c.num_blocks = d.a.num_blocks; c.max_count = d.max_count;
  c.top = bp->top_blocks; c.sinks = bp->sink_blocks; c.recent = bp->recent_blocks; c.group_max = bp->group_reduce == TRI_REDUCE_MAX;
  c.block_table = d.a.block_table; c.block_table_pitch = d.a.block_table_pitch; c.seq_lens = d.a.seq_lens;
  c.q = p->q; c.q_stride_row = p->q_stride_row; c.q_stride_head = p->q_stride_head; c.bounds = bp->bounds;
  c.scores = at<float>(ws, d.block_scores); c.counts = at<int32_t>(ws, d.counts); c.blocks = bp->blocks;
  rc = launch_status(tri::launch_block_scores(c, s), "block_scores");
  if (rc) return rc;
  rc = launch_status(tri::launch_topk_rows(c.scores, d.max_count, c.B * c.Hkv, c.counts, c.counts + c.B, c.Hkv, d.max_count, bp->blocks,
                                           bp->top_blocks, s),
                     "topk_rows");
  if (rc) return rc;
  d.a.list = bp->blocks; d.a.list_k = bp->top_blocks; d.a.list_pitch = bp->top_blocks;
  return do_attend(d, ws, nullptr, 0, s);
}

uint64_t tri_evict_workspace_bytes(const tri_kv_layout* kv, const tri_batch* batch, const tri_evict_params* p) {
  tri::EvictLaunch a{};
  if (fill_evict(kv, batch, p, nullptr, a)) return 0;
  return (uint64_t)tri::align_up(evict_rows(a) * a.Tmax * 4, 256);
}

int tri_select_by_weight(const tri_kv_layout* kv, const tri_batch* batch, const tri_evict_params* p, float* final_scores,
                         int32_t* keep, void* ws, uint64_t ws_bytes, void* stream) {
  tri::EvictLaunch a{};
  const int rc = fill_evict(kv, batch, p, keep, a);
  if (rc) return rc;
  return do_select_by_weight(a, p, final_scores, ws, ws_bytes, (hipStream_t)stream);
}

int tri_evict_step(const tri_kv_layout* kv, const tri_batch* batch, const tri_evict_params* p, int32_t* keep, void* ws,
                   uint64_t ws_bytes, void* stream) {
  tri::EvictLaunch a{};
  int rc = fill_evict(kv, batch, p, keep, a);
  if (rc) return rc;
  tri::CompactLaunch c{};
  rc = fill_compact(kv, batch, keep, p->layer_reduce < 0, p->shared, c);
  if (rc) return rc;
  hipStream_t s = (hipStream_t)stream;
  rc = do_select_by_weight(a, p, nullptr, ws, ws_bytes, s);
  if (rc) return rc;
  rc = launch_status(tri::launch_compact(c, s), "compact");
  if (rc) return rc;
  return launch_status(tri::launch_move_weights(a, s), "move_weights");
}

uint64_t tri_qstats_workspace_bytes(int32_t num_heads, int32_t num_tokens, int32_t head_dim) {
  if (num_heads <= 0 || num_tokens <= 0 || (head_dim != 64 && head_dim != 128 && head_dim != 256)) return 0;
  return (uint64_t)tri::qstats_workspace_bytes(num_heads, num_tokens, head_dim);
}

int tri_qstats(const void* q_rot, int64_t stride_head, int64_t stride_token, const void* cos, const void* sin,
               int32_t num_heads, int32_t num_tokens, int32_t head_dim, int32_t dtype, int32_t rope_style,
               float scale, float* out_real, float* out_imag, float* out_abs, void* workspace,
               uint64_t workspace_bytes, void* stream) {
  if (!q_rot || !cos || !sin || !out_real || !out_imag || !out_abs)
    return fail(TRI_ERR_INVALID_ARGUMENT, "tri_qstats: NULL pointer");
  if (num_heads <= 0 || num_tokens <= 0) return fail(TRI_ERR_INVALID_ARGUMENT, "tri_qstats: bad sizes");
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return fail(TRI_ERR_UNSUPPORTED, "head_dim %d not in {64,128,256}", head_dim);
  if (dtype != TRI_KV_BF16 && dtype != TRI_KV_FP16)
    return fail(TRI_ERR_UNSUPPORTED, "tri_qstats: dtype %d (bf16 or fp16 query states)", dtype);
  if (rope_style != TRI_ROPE_HALF && rope_style != TRI_ROPE_INTERLEAVED)
    return fail(TRI_ERR_INVALID_ARGUMENT, "rope_style %d", rope_style);
  if (scale == 0.f) return fail(TRI_ERR_INVALID_ARGUMENT, "attention scaling factor must be non-zero");
  if (stride_token < head_dim || stride_token % 2 || stride_head % 2 || !is_aligned(q_rot, 4) || !is_aligned(cos, 4) ||
      !is_aligned(sin, 4))
    return fail(TRI_ERR_INVALID_ARGUMENT, "tri_qstats: rows must be 4-byte aligned and head_dim contiguous");
  const uint64_t need = tri_qstats_workspace_bytes(num_heads, num_tokens, head_dim);
  if (!workspace || workspace_bytes < need || !is_aligned(workspace, 16))
    return fail(TRI_ERR_WORKSPACE, "tri_qstats: workspace of %llu bytes needed", (unsigned long long)need);
  tri::QStatsLaunch q{};
  q.q_rot = q_rot; q.cos = cos; q.sin = sin;
  q.stride_head = stride_head; q.stride_token = stride_token;
  q.H = num_heads; q.T = num_tokens; q.D = head_dim; q.dtype = dtype; q.rope_style = rope_style;
  q.scale = scale;
  q.out_real = out_real; q.out_imag = out_imag; q.out_abs = out_abs;
  q.workspace = workspace;
  return launch_status(tri::launch_qstats(q, (hipStream_t)stream), "qstats");
}

}  // extern "C"
