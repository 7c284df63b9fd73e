// The C ABI of libpthdec.so (include/pth_dec.h): the reference's argument checks and error
// messages (kernels/pth_dec/pth_dec.cpp:16-91, kernels/fa_pth/pth_fa.cpp:41-85), the validation of
// the tensor descriptors, and the calls into the kernel files. The library is built with hidden
// visibility; only the entry points declared in pth_dec.h are exported.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>

#pragma GCC visibility push(default)
#include "pth_dec.h"
#pragma GCC visibility pop

#include "pd_kernels.hpp"
#include "pd_plan.hpp"

namespace pd {
namespace {

LaunchArgs make_args(const void* q, int64_t q_st, const void* kc, int64_t k_sb, int64_t k_ss, int64_t k_sh,
                     const int* block_table, int64_t bt_stride, const int* seq_lens, const int* qsl, int num_seqs,
                     int num_tokens, int heads_q, int heads_kv, int block_size, float scale, int qmax,
                     float* part_o, float* part_m, float* part_l, int nseg, int nsplit, void* out, int64_t o_st,
                     int64_t o_sh, int window, int causal) {
    LaunchArgs x;
    x.q = q;
    x.q_st = q_st;
    x.kc = kc;
    x.k_sb = k_sb;
    x.k_ss = k_ss;
    x.k_sh = k_sh;
    x.block_table = block_table;
    x.bt_stride = bt_stride;
    x.seq_lens = seq_lens;
    x.qsl = qsl;
    x.num_seqs = num_seqs;
    x.num_tokens = num_tokens;
    x.heads_q = heads_q;
    x.heads_kv = heads_kv;
    x.block_size = block_size;
    x.scale = scale;
    x.qmax = qmax;
    x.part_o = part_o;
    x.part_m = part_m;
    x.part_l = part_l;
    x.nseg = nseg;
    x.nsplit = nsplit;
    x.out = out;
    x.o_st = o_st;
    x.o_sh = o_sh;
    x.window = window;
    x.causal = causal;
    x.lse = nullptr;
    x.sinks = 0;
    return x;
}

// ---- descriptor checks (pth_dec.cpp:16-80) ----

bool is_dtype(const pd_tensor* t, int dt) { return t && t->dtype == dt; }

bool same_rows(const pd_tensor* scale, const pd_tensor* cache, int64_t byte_off) {
    // f32 scale view [blocks, block_size, Hkv] sitting byte_off bytes into each cache row
    const uintptr_t base = reinterpret_cast<uintptr_t>(cache->data);
    return scale->ndim == 3 && scale->dtype == PD_DTYPE_FP32 &&
           reinterpret_cast<uintptr_t>(scale->data) == base + (uintptr_t)byte_off &&
           scale->strides[0] * 4 == cache->strides[0] && scale->strides[1] * 4 == cache->strides[1] &&
           scale->strides[2] * 4 == cache->strides[2];
}

bool layout_ok(const pd_tensor* kc, const pd_tensor* vc, const pd_tensor* ks, const pd_tensor* vs) {
    if (!kc || !vc || !ks || !vs) return false;
    if (kc->dtype != PD_DTYPE_INT8 || vc->dtype != PD_DTYPE_INT8 || kc->ndim != 4 || vc->ndim != 4 ||
        kc->sizes[3] != 260 || vc->sizes[3] != 260 || kc->strides[3] != 1 || vc->strides[3] != 1)
        return false;
    for (int i = 0; i < 3; ++i)
        if (kc->strides[i] != vc->strides[i] || kc->sizes[i] != vc->sizes[i]) return false;
    const uintptr_t kb = reinterpret_cast<uintptr_t>(kc->data);
    if (reinterpret_cast<uintptr_t>(vc->data) != kb + 260) return false;
    if (kb % 8 || kc->strides[0] % 8 || kc->strides[1] % 8 || kc->strides[2] % 8) return false;
    if (kc->strides[0] > INT32_MAX || kc->strides[1] > INT32_MAX || kc->strides[2] > INT32_MAX) return false;
    return same_rows(ks, kc, 256) && same_rows(vs, kc, 516);
}

bool is_contig(const pd_tensor* t) {
    for (int i = 0; i < t->ndim; ++i)
        if (t->sizes[i] == 0) return true;  // an empty tensor is contiguous whatever its strides
    int64_t expect = 1;
    for (int i = t->ndim - 1; i >= 0; --i) {
        if (t->sizes[i] != 1 && t->strides[i] != expect) return false;
        expect *= t->sizes[i];
    }
    return true;
}

int fail(char* err, int errlen, const char* msg) {
    if (err && errlen > 0) {
        strncpy(err, msg, (size_t)errlen - 1);
        err[errlen - 1] = '\0';
    }
    return 1;
}

}  // namespace
}  // namespace pd

using namespace pd;

#pragma GCC visibility push(default)

extern "C" {

hipError_t pth_dec_launch(const void* q, int q_st, const void* kc, int k_sb, int k_ss, int k_sh,
                          const int* block_table, int bt_stride, const int* seq_lens, const int* qsl,
                          int num_seqs, int num_tokens, int heads_q, int heads_kv, int block_size,
                          float scale, int qmax, float* part_o, float* part_m, float* part_l, int nseg,
                          int nsplit, void* out, long o_st, long o_sh, hipStream_t stream) {
    const LaunchArgs x = make_args(q, q_st, kc, k_sb, k_ss, k_sh, block_table, bt_stride, seq_lens, qsl, num_seqs,
                                   num_tokens, heads_q, heads_kv, block_size, scale, qmax, part_o, part_m, part_l,
                                   nseg, nsplit, out, o_st, o_sh, -1, 1);
    return launch_all(x, stream, true);
}

hipError_t pth_dec_launch_window(const void* q, int q_st, const void* kc, int k_sb, int k_ss, int k_sh,
                                 const int* block_table, int bt_stride, const int* seq_lens,
                                 const int* qsl, int num_seqs, int num_tokens, int heads_q, int heads_kv,
                                 int block_size, float scale, int qmax, float* part_o, float* part_m,
                                 float* part_l, int nseg, int nsplit, void* out, long o_st, long o_sh,
                                 hipStream_t stream, int window, int causal) {
    const LaunchArgs x = make_args(q, q_st, kc, k_sb, k_ss, k_sh, block_table, bt_stride, seq_lens, qsl, num_seqs,
                                   num_tokens, heads_q, heads_kv, block_size, scale, qmax, part_o, part_m, part_l,
                                   nseg, nsplit, out, o_st, o_sh, window, causal);
    return launch_all(x, stream, false);
}

hipError_t pth_dec_launch_noalloc(const void* q, int q_st, const void* kc, int k_sb, int k_ss, int k_sh,
                                  const int* block_table, int bt_stride, const int* seq_lens,
                                  const int* qsl, int num_seqs, int num_tokens, int heads_q,
                                  int heads_kv, int block_size, float scale, int qmax, int nsplit,
                                  void* out, long o_st, long o_sh, hipStream_t stream, int window,
                                  int causal) {
    LaunchArgs x = make_args(q, q_st, kc, k_sb, k_ss, k_sh, block_table, bt_stride, seq_lens, qsl, num_seqs,
                             num_tokens, heads_q, heads_kv, block_size, scale, qmax, nullptr, nullptr, nullptr,
                             nsplit, nsplit, out, o_st, o_sh, window, causal);
    hipError_t e = check_args(x, false);
    if (e != hipSuccess) return e;
    if (num_tokens == 0) return hipSuccess;
    // partial rows the array holds; the product is bounded in two steps so that it cannot wrap
    const uint64_t max_rows = kScratchBytes / ((kDim + 2) * sizeof(float));
    const uint64_t th = (uint64_t)num_tokens * (uint64_t)heads_q;  // both below 2^31
    if (th > max_rows || th * (uint64_t)nsplit > max_rows) return hipErrorOutOfMemory;
    const size_t rows = (size_t)(th * (uint64_t)nsplit);
    void* base = nullptr;
    e = scratch_address(&base);
    if (e != hipSuccess) return e;
    x.part_o = static_cast<float*>(base);
    x.part_m = x.part_o + rows * kDim;
    x.part_l = x.part_m + rows;
    return launch_both(x, stream);
}

hipError_t pth_dec_launch_partial(const void* q, int q_st, const void* kc, int k_sb, int k_ss, int k_sh,
                                  const int* block_table, int bt_stride, const int* seq_lens,
                                  const int* qsl, int num_seqs, int num_tokens, int heads_q,
                                  int heads_kv, int block_size, float scale, int qmax, float* part_o,
                                  float* part_m, float* part_l, int nseg, int nsplit,
                                  hipStream_t stream, int window, int causal) {
    const LaunchArgs x = make_args(q, q_st, kc, k_sb, k_ss, k_sh, block_table, bt_stride, seq_lens, qsl, num_seqs,
                                   num_tokens, heads_q, heads_kv, block_size, scale, qmax, part_o, part_m, part_l,
                                   nseg, nsplit, nullptr, 0, 0, window, causal);
    hipError_t e = check_args(x, false);
    if (e != hipSuccess) return e;
    if (num_tokens == 0) return hipSuccess;
    return launch_partial(x, stream);
}

hipError_t pth_dec_launch_combine(const int* seq_lens, const int* qsl, int num_seqs, int num_tokens,
                                  int heads_q, int qmax, const float* part_o, const float* part_m,
                                  const float* part_l, int nseg, int nsplit, void* out, long o_st,
                                  long o_sh, hipStream_t stream) {
    if (num_seqs < 1 || heads_q < 1 || qmax < 1 || nsplit < 1 || nsplit > nseg || num_tokens < 0)
        return hipErrorInvalidValue;
    if (num_tokens == 0) return hipSuccess;
    const LaunchArgs x = make_args(nullptr, 0, nullptr, 0, 0, 0, nullptr, 0, seq_lens, qsl, num_seqs, num_tokens,
                                   heads_q, 1, 1, 1.f, qmax, const_cast<float*>(part_o), const_cast<float*>(part_m),
                                   const_cast<float*>(part_l), nseg, nsplit, out, o_st, o_sh, -1, 1);
    return launch_combine(x, stream);
}

int pth_dec_supported_layout(const pd_tensor* key_cache, const pd_tensor* value_cache, const pd_tensor* k_scale,
                             const pd_tensor* v_scale) {
    return layout_ok(key_cache, value_cache, k_scale, v_scale) ? 1 : 0;
}

// null if lse (may be null) can take the rows' logarithms, else why not
static const char* lse_refused(const pd_tensor* lse, int64_t T, int64_t Hq) {
    if (!lse) return nullptr;
    const bool ok = lse->dtype == PD_DTYPE_FP32 && lse->ndim == 2 && lse->sizes[0] >= T && lse->sizes[1] == Hq && is_contig(lse);
    return ok ? nullptr : "lse must be contiguous fp32 [T, Hq]";
}

static int64_t cache_span(const pd_tensor* kc);
static bool int_rows(const pd_tensor* t, int64_t n);
static bool int_table(const pd_tensor* t, int64_t n);
static bool rows_apart(const pd_tensor* t, int64_t n0, int64_t len);

// The decode entries' body; prefix >= 0: the shared-prefix decode (nsplit is not looked at beyond its check).
static int decode_entry(const pd_tensor* q, const pd_tensor* key_cache, const pd_tensor* value_cache,
                        const pd_tensor* k_scale, const pd_tensor* v_scale, const pd_tensor* block_table,
                        const pd_tensor* seq_lens, const pd_tensor* query_start_loc, const pd_tensor* out, double scale,
                        const pd_tensor* part_o, const pd_tensor* part_m, const pd_tensor* part_l, const pd_tensor* lse,
                        int64_t num_seqs, int64_t qmax, int64_t nsplit, int64_t window, int64_t causal,
                        hipStream_t stream, char* err, int errlen, int64_t prefix = -1, int64_t sinks = 0) {
    if (!q || !key_cache || !value_cache || !k_scale || !v_scale || !block_table || !seq_lens ||
        !query_start_loc || !out || !part_o || !part_m || !part_l)
        return fail(err, errlen, "null tensor descriptor");
    if (!(q->dtype == PD_DTYPE_FP16 && q->ndim == 3 && q->sizes[2] == 256 && q->strides[2] == 1 &&
          q->strides[1] == 256 && q->strides[0] % 2 == 0 && q->strides[0] <= INT32_MAX &&
          (reinterpret_cast<uintptr_t>(q->data) % 4) == 0))
        return fail(err, errlen, "q must be fp16 [T, Hq, 256] with contiguous heads");
    if (!(out->dtype == PD_DTYPE_FP16 && out->ndim == 3 && out->sizes[0] == q->sizes[0] &&
          out->sizes[1] == q->sizes[1] && out->sizes[2] == 256 && out->strides[2] == 1))
        return fail(err, errlen, "out must be fp16 [T, Hq, 256] with unit dim stride");
    if (!(q->sizes[0] <= INT32_MAX && q->sizes[1] <= INT32_MAX && num_seqs <= INT32_MAX && qmax <= INT32_MAX &&
          nsplit <= INT32_MAX && window >= INT32_MIN && window <= INT32_MAX))
        return fail(err, errlen, "sizes, num_seqs, qmax, nsplit and window must fit in 32 bits");
    if (!layout_ok(key_cache, value_cache, k_scale, v_scale))
        return fail(err, errlen, "KV cache views do not have the int8 per-token-head row layout");
    if (!(block_table->dtype == PD_DTYPE_INT32 && seq_lens->dtype == PD_DTYPE_INT32 &&
          query_start_loc->dtype == PD_DTYPE_INT32 && block_table->ndim == 2 && block_table->strides[1] == 1 &&
          block_table->strides[0] <= INT32_MAX && is_contig(seq_lens) && is_contig(query_start_loc)))
        return fail(err, errlen, "block_table / seq_lens / query_start_loc must be int32");
    if (!(part_o->dtype == PD_DTYPE_FP32 && is_contig(part_o) && part_o->ndim == 4 && part_o->sizes[3] == 256 &&
          part_m->dtype == PD_DTYPE_FP32 && part_l->dtype == PD_DTYPE_FP32 && is_contig(part_m) &&
          is_contig(part_l) && part_m->ndim == 3 && part_l->ndim == 3))
        return fail(err, errlen, "partial buffers must be contiguous fp32");
    const int64_t T = q->sizes[0], Hq = q->sizes[1], Hkv = key_cache->sizes[2];
    const int64_t nseg = part_o->sizes[2];
    if (!(part_o->sizes[0] >= T && part_o->sizes[1] == Hq && part_m->sizes[0] >= T && part_m->sizes[1] == Hq &&
          part_m->sizes[2] == nseg && part_l->sizes[0] >= T && part_l->sizes[1] == Hq && part_l->sizes[2] == nseg &&
          nseg <= INT32_MAX))
        return fail(err, errlen, "partial buffers too small");
    if (!(Hkv > 0 && Hq % Hkv == 0)) return fail(err, errlen, "heads_q must be a multiple of heads_kv");
    if (!(qmax >= 1 && qmax * (Hq / Hkv) <= 16 * kMaxRowBlocks))
        return fail(err, errlen, "qmax * (Hq / Hkv) must be in [1, 48]");
    if (!(nsplit >= 1 && nsplit <= nseg)) return fail(err, errlen, "nsplit must be in [1, NSEG]");
    if (!(num_seqs >= 1 && seq_lens->sizes[0] >= num_seqs && query_start_loc->sizes[0] >= num_seqs + 1 &&
          block_table->sizes[0] >= num_seqs))
        return fail(err, errlen, "per-sequence tensors too small");
    if (const char* why = lse_refused(lse, T, Hq)) return fail(err, errlen, why);
    if (prefix >= 0) {
        const int64_t bs = key_cache->sizes[1], cols = block_table->sizes[1];
        if (nseg < kSharedMinSegments) return fail(err, errlen, "a shared-prefix decode needs at least 4 segments");
        if (!(prefix <= INT32_MAX && bs > 0 && cols <= INT32_MAX && prefix <= cols * bs))
            return fail(err, errlen, "prefix_len must be within the block table");
        // 32 bits number the rows and the line of own key tiles
        const int64_t tiles = cols * bs / 32 + 16;
        if (!(Hq >= 1 && T <= ((int64_t)1 << 25) / Hq && tiles <= INT32_MAX / 2 && tiles * num_seqs <= INT32_MAX / (2 * Hkv)))
            return fail(err, errlen, "a shared-prefix decode takes at most 2^25 (token, head) rows and 2^30 key tiles");
    }
    if (!(sinks >= 0 && sinks <= INT32_MAX)) return fail(err, errlen, "sinks must be at least 0 and fit in 32 bits");
    if (T == 0) return 0;
    LaunchArgs x = make_args(
        q->data, q->strides[0], key_cache->data, key_cache->strides[0], key_cache->strides[1],
        key_cache->strides[2], static_cast<const int*>(block_table->data), block_table->strides[0],
        static_cast<const int*>(seq_lens->data), static_cast<const int*>(query_start_loc->data), (int)num_seqs,
        (int)T, (int)Hq, (int)Hkv, (int)key_cache->sizes[1], (float)scale, (int)qmax,
        static_cast<float*>(const_cast<void*>(part_o->data)), static_cast<float*>(const_cast<void*>(part_m->data)),
        static_cast<float*>(const_cast<void*>(part_l->data)), (int)nseg, (int)nsplit, const_cast<void*>(out->data),
        out->strides[0], out->strides[1], (int)window, (int)causal);
    x.lse = lse ? static_cast<float*>(const_cast<void*>(lse->data)) : nullptr;
    x.sinks = window > 0 ? (int)sinks : 0;
    // (16-key block offsets fit a 32-bit LDS table in 8-byte units when the cache spans less than 2^35 bytes)
    const hipError_t e = prefix < 0 ? launch_all(x, stream, false)
                                    : launch_shared(x, (int)prefix, cache_span(key_cache) < ((int64_t)1 << 35), stream);
    if (e != hipSuccess) {
        char msg[256];
        snprintf(msg, sizeof msg, "pth_dec launch failed: %s", hipGetErrorString(e));
        fail(err, errlen, msg);
        return 2;
    }
    return 0;
}

int pth_dec_decode(const pd_tensor* q, const pd_tensor* key_cache, const pd_tensor* value_cache,
                   const pd_tensor* k_scale, const pd_tensor* v_scale, const pd_tensor* block_table,
                   const pd_tensor* seq_lens, const pd_tensor* query_start_loc, const pd_tensor* out, double scale,
                   const pd_tensor* part_o, const pd_tensor* part_m, const pd_tensor* part_l, int64_t num_seqs,
                   int64_t qmax, int64_t nsplit, int64_t window, int64_t causal, hipStream_t stream, char* err,
                   int errlen) {
    return decode_entry(q, key_cache, value_cache, k_scale, v_scale, block_table, seq_lens, query_start_loc, out, scale,
                        part_o, part_m, part_l, nullptr, num_seqs, qmax, nsplit, window, causal, stream, err, errlen);
}

int pth_dec_decode_lse(const pd_tensor* q, const pd_tensor* key_cache, const pd_tensor* value_cache,
                       const pd_tensor* k_scale, const pd_tensor* v_scale, const pd_tensor* block_table,
                       const pd_tensor* seq_lens, const pd_tensor* query_start_loc, const pd_tensor* out, double scale,
                       const pd_tensor* part_o, const pd_tensor* part_m, const pd_tensor* part_l, const pd_tensor* lse,
                       int64_t num_seqs, int64_t qmax, int64_t nsplit, int64_t window, int64_t causal,
                       hipStream_t stream, char* err, int errlen) {
    if (!lse) return fail(err, errlen, "null tensor descriptor");
    return decode_entry(q, key_cache, value_cache, k_scale, v_scale, block_table, seq_lens, query_start_loc, out, scale,
                        part_o, part_m, part_l, lse, num_seqs, qmax, nsplit, window, causal, stream, err, errlen);
}

int pth_dec_decode_sinks(const pd_tensor* q, const pd_tensor* key_cache, const pd_tensor* value_cache,
                         const pd_tensor* k_scale, const pd_tensor* v_scale, const pd_tensor* block_table,
                         const pd_tensor* seq_lens, const pd_tensor* query_start_loc, const pd_tensor* out, double scale,
                         const pd_tensor* part_o, const pd_tensor* part_m, const pd_tensor* part_l, const pd_tensor* lse,
                         int64_t num_seqs, int64_t qmax, int64_t nsplit, int64_t window, int64_t sinks, int64_t causal,
                         hipStream_t stream, char* err, int errlen) {
    return decode_entry(q, key_cache, value_cache, k_scale, v_scale, block_table, seq_lens, query_start_loc, out, scale,
                        part_o, part_m, part_l, lse, num_seqs, qmax, nsplit, window, causal, stream, err, errlen, -1, sinks);
}

int pth_dec_decode_shared(const pd_tensor* q, const pd_tensor* key_cache, const pd_tensor* value_cache,
                          const pd_tensor* k_scale, const pd_tensor* v_scale, const pd_tensor* block_table,
                          const pd_tensor* seq_lens, const pd_tensor* query_start_loc, const pd_tensor* out, double scale,
                          const pd_tensor* part_o, const pd_tensor* part_m, const pd_tensor* part_l, const pd_tensor* lse,
                          int64_t num_seqs, int64_t qmax, int64_t prefix_len, hipStream_t stream, char* err, int errlen) {
    if (prefix_len < 0) return fail(err, errlen, "prefix_len must be within the block table");
    return decode_entry(q, key_cache, value_cache, k_scale, v_scale, block_table, seq_lens, query_start_loc, out, scale,
                        part_o, part_m, part_l, lse, num_seqs, qmax, 1, -1, 1, stream, err, errlen, prefix_len);
}

static int fa_result(hipError_t e, char* err, int errlen) {
    if (e == hipSuccess) return 0;
    char msg[256];
    snprintf(msg, sizeof msg, "pth_fa launch failed: %s", hipGetErrorString(e));
    fail(err, errlen, msg);
    return 2;
}

// bytes from the cache base to the last K row's scale
static int64_t cache_span(const pd_tensor* kc) {
    return (kc->sizes[0] - 1) * kc->strides[0] + (kc->sizes[1] - 1) * kc->strides[1] + (kc->sizes[2] - 1) * kc->strides[2] + 8;
}

// Whether 32 bits number the line of a balanced prefill: items x the key tiles that a block table can hold.
static bool balanced_ok(int64_t items, int64_t table_keys) {
    const int64_t tiles = table_keys / 32 + 64;
    return items <= INT32_MAX / 2 && tiles <= INT32_MAX / 2 && items * tiles <= INT32_MAX;
}
static const char* balanced_workspace(FaParams& p, FaRowsParams& r, const pd_tensor* ws, int64_t items, int64_t max_keys,
                                      hipStream_t stream) {
    if (!(ws && ws->dtype == PD_DTYPE_FP32 && ws->ndim == 1 && is_contig(ws) &&
          reinterpret_cast<uintptr_t>(ws->data) % 16 == 0 && ws->sizes[0] >= 2 * kFaSlotFloats))
        return "workspace must be contiguous 16-byte aligned fp32 of pth_fa_balanced_workspace";
    const int cus = compute_units(stream);
    r.nwg = (int)std::min(ws->sizes[0] / (2 * kFaSlotFloats),
                          balanced_prefill_workgroups(items, std::max<int64_t>(0, max_keys), cus > 0 ? cus : 256));
    float* f = static_cast<float*>(const_cast<void*>(ws->data));
    const int64_t rows = 2ll * r.nwg * kFaRows;
    p.part_o = f;
    p.part_m = f + rows * kDim;
    p.part_l = p.part_m + rows;
    return nullptr;
}

static int fa_forward(const pd_tensor* q, const pd_tensor* key_cache, const pd_tensor* value_cache,
                      const pd_tensor* block_table, const pd_tensor* seq_lens, double scale,
                      const pd_tensor* q_abs_offset, const pd_tensor* out, hipStream_t stream, char* err, int errlen,
                      bool exact, int64_t nsplit = 1, const pd_tensor* workspace = nullptr,
                      const int64_t* balanced_keys = nullptr) {
    if (!q || !key_cache || !value_cache || !block_table || !seq_lens || !q_abs_offset || !out)
        return fail(err, errlen, "null tensor descriptor");
    if (!(q->dtype == PD_DTYPE_FP32 && q->ndim == 4 && is_contig(q)))
        return fail(err, errlen, "q must be contiguous fp32 [B, Hq, Sq, D]");
    if (!(key_cache->dtype == PD_DTYPE_INT8 && value_cache->dtype == PD_DTYPE_INT8))
        return fail(err, errlen, "key/value cache views must be int8");
    if (!(key_cache->ndim == 4 && value_cache->ndim == 4)) return fail(err, errlen, "cache views must be 4D");
    if (!(key_cache->strides[3] == 1 && value_cache->strides[3] == 1))
        return fail(err, errlen, "cache rows must be contiguous");
    if (!(block_table->dtype == PD_DTYPE_INT32 && seq_lens->dtype == PD_DTYPE_INT32 &&
          q_abs_offset->dtype == PD_DTYPE_INT32))
        return fail(err, errlen, "block_table/seq_lens/q_abs_offset must be int32");
    const int64_t B = q->sizes[0], Hq = q->sizes[1], Sq = q->sizes[2], D = q->sizes[3];
    const int64_t bs = key_cache->sizes[1], Hkv = key_cache->sizes[2];
    if (!(B <= INT32_MAX && Hq <= INT32_MAX && Sq <= INT32_MAX))
        return fail(err, errlen, "B, Hq and Sq must be below 2^31");
    if (D != 256) return fail(err, errlen, "head_dim must be 256 (only instantiation built)");
    if (!(key_cache->sizes[3] >= D + 4 && value_cache->sizes[3] >= D + 4))
        return fail(err, errlen, "cache rows must hold D int8 values and a fp32 scale");
    if (!(Hkv > 0 && Hq % Hkv == 0)) return fail(err, errlen, "heads_q must be a multiple of heads_kv");
    if (!(block_table->ndim == 2 && block_table->sizes[0] == B && block_table->strides[1] == 1 &&
          seq_lens->sizes[0] == B && q_abs_offset->sizes[0] == B && is_contig(seq_lens) && is_contig(q_abs_offset)))
        return fail(err, errlen, "per-sequence tensors must have B rows");
    const uintptr_t kb = reinterpret_cast<uintptr_t>(key_cache->data);
    if (!(kb % 8 == 0 && (reinterpret_cast<uintptr_t>(value_cache->data) % 4) == 0 && key_cache->strides[1] % 8 == 0 &&
          key_cache->strides[2] % 8 == 0 && key_cache->strides[0] % 8 == 0))
        return fail(err, errlen, "K rows must be 8-byte aligned and V rows 4-byte aligned");
    // the kernel reads K and V from one 520-byte row: V must be the same rows, 260 bytes in
    bool same = reinterpret_cast<uintptr_t>(value_cache->data) == kb + 260;
    for (int i = 0; i < 3; ++i)
        same = same && value_cache->strides[i] == key_cache->strides[i] && value_cache->sizes[i] == key_cache->sizes[i];
    if (!same) return fail(err, errlen, "value_cache must view the same cache rows as key_cache, 260 bytes in");
    if (!(key_cache->strides[0] <= INT32_MAX && key_cache->strides[1] <= INT32_MAX && key_cache->strides[2] <= INT32_MAX))
        return fail(err, errlen, "cache strides must be below 2^31");
    const int64_t G = Hq / Hkv;
    if (G > kFaRows) return fail(err, errlen, "heads_q / heads_kv must be at most 192");
    if (!(out->dtype == PD_DTYPE_FP32 && out->ndim == 4 && out->sizes[0] == B && out->sizes[1] == Sq &&
          out->sizes[2] == Hq && out->sizes[3] == D && out->strides[3] == 1))
        return fail(err, errlen, "out must be fp32 [B, Sq, Hq, D] with unit dim stride");
    // q rows are read and out rows written as 16-byte vectors
    if (!((reinterpret_cast<uintptr_t>(q->data) % 16) == 0 && (reinterpret_cast<uintptr_t>(out->data) % 16) == 0 &&
          out->strides[0] % 4 == 0 && out->strides[1] % 4 == 0 && out->strides[2] % 4 == 0))
        return fail(err, errlen, "q and out rows must be 16-byte aligned");
    if (!(nsplit >= 1 && nsplit <= 64)) return fail(err, errlen, "nsplit must be in [1, 64]");
    // the merge numbers rows (b, token, head) in 32 bits; B, Sq < 2^31 keep B * Sq within int64
    if (nsplit > 1 && Hq > 0 && B * Sq > INT32_MAX / Hq)
        return fail(err, errlen, "a split prefill takes at most 2^31 - 1 (token, head) rows");
    if (nsplit > 1) {
        if (!(workspace && workspace->dtype == PD_DTYPE_FP32 && workspace->ndim == 1 && is_contig(workspace) &&
              workspace->sizes[0] >= prefill_workspace_floats(B, Sq, Hq, nsplit) &&
              (reinterpret_cast<uintptr_t>(workspace->data) % 16) == 0))
            return fail(err, errlen, "workspace must be contiguous 16-byte aligned fp32 of B * Sq * Hq * nsplit * 258");
    }
    if (B == 0 || Sq == 0) return 0;
    FaParams p;
    p.q = q->data;
    p.q_sb = q->strides[0];
    p.q_sh = q->strides[1];
    p.q_st = q->strides[2];
    p.kc = static_cast<const int8_t*>(key_cache->data);
    p.k_sb = key_cache->strides[0];
    p.k_ss = key_cache->strides[1];
    p.k_sh = key_cache->strides[2];
    p.block_table = static_cast<const int*>(block_table->data);
    p.bt_stride = block_table->strides[0];
    p.seq_lens = static_cast<const int*>(seq_lens->data);
    p.q_abs = static_cast<const int*>(q_abs_offset->data);
    p.out = const_cast<void*>(out->data);
    p.o_sb = out->strides[0];
    p.o_st = out->strides[1];
    p.o_sh = out->strides[2];
    p.Sq = (int)Sq;
    p.Hq = (int)Hq;
    p.G = (int)G;
    p.tok_per_wg = (int)(kFaRows / G);
    p.block_size = (int)bs;
    p.bs_shift = (bs & (bs - 1)) == 0 ? __builtin_ctz((unsigned)bs) : -1;
    p.scale_log2 = (float)scale * 1.4426950408889634f;
    // 16-key block offsets fit the LDS table's 32 bits (in 8-byte units) when the cache spans
    // less than 2^35 bytes
    p.bt32 = cache_span(key_cache) < ((int64_t)1 << 35);
    p.nsplit = (int)nsplit;
    p.part_o = nullptr;
    p.part_m = nullptr;
    p.part_l = nullptr;
    if (nsplit > 1) {
        float* ws = static_cast<float*>(const_cast<void*>(workspace->data));
        const int64_t prow = B * Sq * Hq * nsplit;
        p.part_o = ws;
        p.part_m = ws + prow * kDim;
        p.part_l = p.part_m + prow;
    }
    if (balanced_keys) {
        FaRowsParams r = {};
        const int64_t qtiles = (Sq + p.tok_per_wg - 1) / p.tok_per_wg;
        r.first_tile[0] = (int)B;
        r.tiles = (int)(B * qtiles);
        const char* why = nullptr;
        if (!balanced_ok(B * qtiles * Hkv, block_table->sizes[1] * bs) || Hq == 0)
            why = "a balanced prefill takes at most 2^31 key tiles";
        else
            why = balanced_workspace(p, r, workspace, r.tiles * Hkv, *balanced_keys, stream);
        if (why) return fail(err, errlen, why);
        return fa_result(launch_prefill_balanced(p, r, (int)Hkv, PD_DTYPE_FP32, stream, exact), err, errlen);
    }
    return fa_result(launch_prefill(p, (int)B, (int)Hkv, PD_DTYPE_FP32, stream, exact), err, errlen);
}

// The rows form: sequence i has rows [query_start[i], query_start[i + 1]) of q and out [T, Hq, 256], the last
// tokens of its seq_lens[i] keys. nsplit 0: balanced; else one sequence with its keys in nsplit splits.
static int fa_forward_rows(const pd_tensor* q, const pd_tensor* kc, const pd_tensor* vc, const pd_tensor* bt,
                           const pd_tensor* seq_lens, double scale, const int* query_start, int64_t num_seqs,
                           const pd_tensor* out, const pd_tensor* workspace, int64_t max_keys, int64_t nsplit,
                           bool exact, hipStream_t stream, char* err, int errlen) {
    if (!(q->ndim == 3 && q->dtype == PD_DTYPE_FP16 && q->sizes[2] == kDim &&
          q->strides[2] == 1 && q->sizes[0] <= INT32_MAX && q->sizes[1] <= INT32_MAX))
        return fail(err, errlen, "q must be fp16 [T, Hq, 256] with unit dim stride");
    if (!(out->ndim == 3 && out->dtype == q->dtype && out->sizes[1] == q->sizes[1] && out->sizes[2] == kDim &&
          out->strides[2] == 1))
        return fail(err, errlen, "out must be fp16 [T, Hq, 256] with unit dim stride");
    if (!(reinterpret_cast<uintptr_t>(q->data) % 16 == 0 && q->strides[0] % 8 == 0 && q->strides[1] % 8 == 0 &&
          reinterpret_cast<uintptr_t>(out->data) % 8 == 0 && out->strides[0] % 4 == 0 && out->strides[1] % 4 == 0))
        return fail(err, errlen, "q rows must be 16-byte aligned and out rows 8-byte aligned");
    if (!(kc->dtype == PD_DTYPE_INT8 && vc->dtype == PD_DTYPE_INT8 && kc->ndim == 4 && vc->ndim == 4 &&
          kc->strides[3] == 1 && vc->strides[3] == 1 && kc->sizes[3] >= kDim + 4 && vc->sizes[3] >= kDim + 4))
        return fail(err, errlen, "key/value cache views must be 4D int8 rows of D values and a fp32 scale");
    const uintptr_t kb = reinterpret_cast<uintptr_t>(kc->data);
    bool rows_ok = kb % 8 == 0 && reinterpret_cast<uintptr_t>(vc->data) == kb + 260;
    for (int i = 0; i < 3; ++i)
        rows_ok = rows_ok && kc->strides[i] == vc->strides[i] && kc->sizes[i] == vc->sizes[i] && kc->strides[i] % 8 == 0 &&
                  kc->strides[i] <= INT32_MAX;
    if (!rows_ok) return fail(err, errlen, "value_cache must view the same 8-byte aligned cache rows as key_cache, 260 bytes in");
    const int64_t T = q->sizes[0], Hq = q->sizes[1], bs = kc->sizes[1], Hkv = kc->sizes[2];
    if (!(Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && Hq / Hkv <= kFaRows))
        return fail(err, errlen, "heads_q must be a multiple of heads_kv, at most 192 times");
    if (!(num_seqs >= 1 && num_seqs <= kFaMaxSeqs && query_start[0] >= 0 && query_start[num_seqs] <= T &&
          query_start[num_seqs] <= out->sizes[0]))
        return fail(err, errlen, "1 to 32 sequences within the rows of q and out");
    for (int64_t i = 0; i < num_seqs; ++i)
        if (query_start[i] > query_start[i + 1]) return fail(err, errlen, "query_start must not decrease");
    if (!(bt->dtype == PD_DTYPE_INT32 && bt->ndim == 2 && bt->sizes[0] >= num_seqs && bt->strides[1] == 1 &&
          seq_lens->dtype == PD_DTYPE_INT32 && seq_lens->ndim == 1 && seq_lens->sizes[0] >= num_seqs && is_contig(seq_lens)))
        return fail(err, errlen, "block_table / seq_lens must be int32 with a row per sequence");
    FaParams p = {};
    p.q = q->data;
    p.q_sh = q->strides[1];
    p.q_st = q->strides[0];
    p.kc = static_cast<const int8_t*>(kc->data);
    p.k_sb = kc->strides[0];
    p.k_ss = kc->strides[1];
    p.k_sh = kc->strides[2];
    p.block_table = static_cast<const int*>(bt->data);
    p.bt_stride = bt->strides[0];
    p.seq_lens = static_cast<const int*>(seq_lens->data);
    p.out = const_cast<void*>(out->data);
    p.o_st = out->strides[0];
    p.o_sh = out->strides[1];
    p.Hq = (int)Hq;
    p.G = (int)(Hq / Hkv);
    p.tok_per_wg = kFaRows / p.G;
    p.block_size = (int)bs;
    p.bs_shift = (bs & (bs - 1)) == 0 ? __builtin_ctz((unsigned)bs) : -1;
    p.scale_log2 = (float)scale * 1.4426950408889634f;
    p.bt32 = cache_span(kc) < ((int64_t)1 << 35);
    p.nsplit = 1;
    if (nsplit != 0) {
        const int64_t n = query_start[1] - query_start[0];
        if (!(num_seqs == 1 && nsplit >= 1 && nsplit <= 64 && (nsplit == 1 || n * Hq * nsplit <= INT32_MAX)))
            return fail(err, errlen, "nsplit must be 0, or in [1, 64] for one sequence");
        if (n == 0) return 0;
        if (nsplit > 1) {
            const int64_t rows = n * Hq * nsplit;
            if (!(workspace && workspace->dtype == PD_DTYPE_FP32 && workspace->ndim == 1 && is_contig(workspace) &&
                  workspace->sizes[0] >= prefill_workspace_floats(1, n, Hq, nsplit) &&
                  reinterpret_cast<uintptr_t>(workspace->data) % 16 == 0))
                return fail(err, errlen, "workspace must be contiguous 16-byte aligned fp32 of rows * Hq * nsplit * 258");
            p.part_o = static_cast<float*>(const_cast<void*>(workspace->data));
            p.part_m = p.part_o + rows * kDim;
            p.part_l = p.part_m + rows;
        }
        p.q = static_cast<const _Float16*>(p.q) + query_start[0] * p.q_st;
        p.out = static_cast<_Float16*>(p.out) + query_start[0] * p.o_st;
        p.Sq = (int)n;
        p.nsplit = (int)nsplit;
        return fa_result(launch_prefill(p, 1, (int)Hkv, PD_DTYPE_FP16, stream, exact), err, errlen);
    }
    FaRowsParams r = {};
    r.n = (int)num_seqs;
    int64_t tiles = 0;
    for (int64_t i = 0; i < num_seqs; ++i) {
        r.first_tok[i] = query_start[i];
        r.first_tile[i] = (int)tiles;
        tiles += (query_start[i + 1] - query_start[i] + p.tok_per_wg - 1) / p.tok_per_wg;
    }
    r.first_tok[num_seqs] = query_start[num_seqs];
    r.first_tile[num_seqs] = r.tiles = (int)tiles;
    if (tiles == 0) return 0;
    if (!balanced_ok(tiles * Hkv, bt->sizes[1] * bs)) return fail(err, errlen, "a balanced prefill takes at most 2^31 key tiles");
    if (const char* why = balanced_workspace(p, r, workspace, tiles * Hkv, max_keys, stream)) return fail(err, errlen, why);
    return fa_result(launch_prefill_balanced(p, r, (int)Hkv, q->dtype, stream, exact), err, errlen);
}

static bool window_tensors_apart(const pd_tensor* q, const pd_tensor* kc, const pd_tensor* block_table, const pd_tensor* seq_lens,
                                 const pd_tensor* query_start, const pd_tensor* out, const pd_tensor* workspace, int64_t num_seqs,
                                 int64_t ws_floats);

int64_t pth_fa_window_splits(int64_t tokens, int64_t num_seqs, int64_t heads_q, int64_t heads_kv, int64_t window, int64_t sinks,
                             int64_t table_keys, int64_t exact) {
    if (tokens < 1 || tokens > INT32_MAX || num_seqs < 1 || num_seqs > INT32_MAX || heads_kv < 1 || heads_q < heads_kv ||
        heads_q % heads_kv != 0 || heads_q > (1 << 20) || window < 1 || window > INT32_MAX || sinks < 0 || sinks > INT32_MAX)
        return 1;
    int dev = 0, cus = 0;
    if (hipGetDevice(&dev) != hipSuccess ||
        hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus < 1)
        cus = 256;
    return fw_splits({tokens, num_seqs, heads_q, heads_kv, window, sinks, std::max<int64_t>(0, table_keys), cus, exact != 0});
}

int pth_fa_forward_window(const pd_tensor* q, const pd_tensor* key_cache, const pd_tensor* value_cache,
                          const pd_tensor* block_table, const pd_tensor* seq_lens, double scale,
                          const pd_tensor* query_start_loc, const pd_tensor* out, const pd_tensor* workspace, int64_t num_seqs,
                          int64_t window, int64_t sinks, int64_t nsplit, int64_t exact, hipStream_t stream, char* err, int errlen) {
    if (!q || !key_cache || !value_cache || !block_table || !seq_lens || !query_start_loc || !out)
        return fail(err, errlen, "null tensor descriptor");
    if (!(q->ndim == 3 && q->dtype == PD_DTYPE_FP16 && q->sizes[2] == kDim && q->strides[2] == 1 && q->sizes[0] <= INT32_MAX &&
          q->sizes[1] <= (1 << 20)))
        return fail(err, errlen, "q must be fp16 [T, Hq, 256] with unit dim stride");
    if (!(out->ndim == 3 && out->dtype == PD_DTYPE_FP16 && out->sizes[0] == q->sizes[0] && out->sizes[1] == q->sizes[1] &&
          out->sizes[2] == kDim && out->strides[2] == 1))
        return fail(err, errlen, "out must be fp16 [T, Hq, 256] with unit dim stride");
    if (!(reinterpret_cast<uintptr_t>(q->data) % 16 == 0 && q->strides[0] % 8 == 0 && q->strides[1] % 8 == 0 &&
          reinterpret_cast<uintptr_t>(out->data) % 8 == 0 && out->strides[0] % 4 == 0 && out->strides[1] % 4 == 0))
        return fail(err, errlen, "q rows must be 16-byte aligned and out rows 8-byte aligned");
    if (!(key_cache->dtype == PD_DTYPE_INT8 && value_cache->dtype == PD_DTYPE_INT8 && key_cache->ndim == 4 && value_cache->ndim == 4 &&
          key_cache->strides[3] == 1 && value_cache->strides[3] == 1 && key_cache->sizes[3] >= kDim + 4 && value_cache->sizes[3] >= kDim + 4))
        return fail(err, errlen, "key/value cache views must be 4D int8 rows of D values and a fp32 scale");
    const uintptr_t kb = reinterpret_cast<uintptr_t>(key_cache->data);
    bool rows_ok = kb % 8 == 0 && reinterpret_cast<uintptr_t>(value_cache->data) == kb + 260;
    for (int i = 0; i < 3; ++i)
        rows_ok = rows_ok && key_cache->strides[i] == value_cache->strides[i] && key_cache->sizes[i] == value_cache->sizes[i] &&
                  key_cache->strides[i] % 8 == 0 && key_cache->strides[i] <= INT32_MAX;
    if (!rows_ok) return fail(err, errlen, "value_cache must view the same 8-byte aligned cache rows as key_cache, 260 bytes in");
    const int64_t T = q->sizes[0], Hq = q->sizes[1], bs = key_cache->sizes[1], Hkv = key_cache->sizes[2];
    if (!(Hkv > 0 && Hkv <= 65535 && Hq > 0 && Hq % Hkv == 0 && Hq <= 65535 && Hq / Hkv <= kFwRows && bs > 0 && bs <= INT32_MAX))
        return fail(err, errlen, "heads_q must be a multiple of heads_kv, at most 256 times and 65535");
    if (!(num_seqs >= 1 && num_seqs <= INT32_MAX && int_table(block_table, num_seqs) && int_rows(seq_lens, num_seqs) &&
          int_rows(query_start_loc, num_seqs + 1)))
        return fail(err, errlen, "block_table / seq_lens / query_start_loc must be int32 with a row for each of at least one sequence");
    if (!(window >= 1 && window <= INT32_MAX && sinks >= 0 && sinks <= INT32_MAX))
        return fail(err, errlen, "window must be at least 1, sinks at least 0, and both fit in 32 bits");
    if (!(nsplit >= 1 && nsplit <= 64)) return fail(err, errlen, "nsplit must be in [1, 64]");
    // a launch's workgroups, and the 32 bits that number query tiles and rows
    const int64_t G = Hq / Hkv, tiles = window_tiles(T, num_seqs, G, kFwNarrowRows);
    // (the merge of splits takes four tokens a workgroup)
    if (!(T * Hq <= ((int64_t)1 << 30) && tiles * nsplit <= (1 << 24) / Hkv - 1 && (nsplit == 1 || T <= ((int64_t)1 << 26) - 4)))
        return fail(err, errlen, "at most 2^30 (token, head) rows and 2^24 workgroups per call");
    if (!rows_apart(out, T, kDim)) return fail(err, errlen, "out rows must not overlap");
    if (nsplit > 1 && !(workspace && workspace->dtype == PD_DTYPE_FP32 && workspace->ndim == 1 && is_contig(workspace) &&
                        workspace->sizes[0] >= prefill_workspace_floats(1, T, Hq, nsplit) &&
                        reinterpret_cast<uintptr_t>(workspace->data) % 16 == 0))
        return fail(err, errlen, "workspace must be contiguous 16-byte aligned fp32 of T * Hq * nsplit * 258");
    if (!window_tensors_apart(q, key_cache, block_table, seq_lens, query_start_loc, out, nsplit > 1 ? workspace : nullptr, num_seqs,
                              prefill_workspace_floats(1, T, Hq, nsplit)))
        return fail(err, errlen, "out and the workspace must not overlap each other or what the call reads");
    if (T == 0) return 0;
    FaParams p = {};
    p.q = q->data;
    p.q_sh = q->strides[1];
    p.q_st = q->strides[0];
    p.kc = static_cast<const int8_t*>(key_cache->data);
    p.k_sb = key_cache->strides[0];
    p.k_ss = key_cache->strides[1];
    p.k_sh = key_cache->strides[2];
    p.block_table = static_cast<const int*>(block_table->data);
    p.bt_stride = block_table->strides[0];
    p.seq_lens = static_cast<const int*>(seq_lens->data);
    p.out = const_cast<void*>(out->data);
    p.o_st = out->strides[0];
    p.o_sh = out->strides[1];
    p.Hq = (int)Hq;
    p.G = (int)G;
    p.block_size = (int)bs;
    p.bs_shift = (bs & (bs - 1)) == 0 ? __builtin_ctz((unsigned)bs) : -1;
    p.bt32 = cache_span(key_cache) < ((int64_t)1 << 35);
    p.scale_log2 = (float)scale * 1.4426950408889634f;
    p.nsplit = (int)nsplit;
    if (nsplit > 1) {
        const int64_t rows = T * Hq * nsplit;
        p.part_o = static_cast<float*>(const_cast<void*>(workspace->data));
        p.part_m = p.part_o + rows * kDim;
        p.part_l = p.part_m + rows;
    }
    const FaWindow w = {static_cast<const int*>(query_start_loc->data), (int)num_seqs, (int)T,
                         (int)std::min<int64_t>(window, 1 << 30), (int)sinks};  // (no sequence is longer; see launch_partial)
    const int cus = compute_units(stream);
    const FwCall call = {T, num_seqs, Hq, Hkv, window, sinks, block_table->sizes[1] * bs, cus > 0 ? cus : 256, exact != 0};
    return fa_result(launch_window(p, w, fw_narrow(call, nsplit) ? kFwNarrowRows : kFwRows, (int)Hkv, stream, exact != 0), err, errlen);
}

int pth_fa_forward(const pd_tensor* q, const pd_tensor* key_cache, const pd_tensor* value_cache,
                   const pd_tensor* block_table, const pd_tensor* seq_lens, double scale, const pd_tensor* q_abs_offset,
                   const pd_tensor* out, hipStream_t stream, char* err, int errlen) {
    return fa_forward(q, key_cache, value_cache, block_table, seq_lens, scale, q_abs_offset, out, stream, err, errlen,
                      false);
}

int pth_fa_forward_exact(const pd_tensor* q, const pd_tensor* key_cache, const pd_tensor* value_cache,
                         const pd_tensor* block_table, const pd_tensor* seq_lens, double scale,
                         const pd_tensor* q_abs_offset, const pd_tensor* out, hipStream_t stream, char* err,
                         int errlen) {
    return fa_forward(q, key_cache, value_cache, block_table, seq_lens, scale, q_abs_offset, out, stream, err, errlen,
                      true);
}

int pth_fa_forward_split(const pd_tensor* q, const pd_tensor* key_cache, const pd_tensor* value_cache,
                         const pd_tensor* block_table, const pd_tensor* seq_lens, double scale,
                         const pd_tensor* q_abs_offset, const pd_tensor* out, const pd_tensor* workspace,
                         int64_t nsplit, int64_t exact, hipStream_t stream, char* err, int errlen) {
    return fa_forward(q, key_cache, value_cache, block_table, seq_lens, scale, q_abs_offset, out, stream, err, errlen,
                      exact != 0, nsplit, workspace);
}

int64_t pth_fa_balanced_workspace(int64_t num_seqs, const int* query_start, int64_t sq, int64_t heads_q, int64_t heads_kv,
                                  int64_t max_keys, int64_t table_keys) {
    if (num_seqs < 1 || heads_kv < 1 || heads_q < 1 || heads_q % heads_kv != 0 || heads_q / heads_kv > kFaRows) return 0;
    const int64_t tok = kFaRows / (heads_q / heads_kv);
    int64_t tiles = 0;
    if (query_start) {
        if (num_seqs > kFaMaxSeqs) return 0;
        for (int64_t i = 0; i < num_seqs; ++i) tiles += (query_start[i + 1] - query_start[i] + tok - 1) / tok;
    } else {
        if (sq < 0 || sq > INT32_MAX || num_seqs > INT32_MAX) return 0;
        tiles = num_seqs * ((sq + tok - 1) / tok);
    }
    if (tiles < 1 || tiles > INT32_MAX / heads_kv || !balanced_ok(tiles * heads_kv, std::max<int64_t>(0, table_keys))) return 0;
    int dev = 0, cus = 0;
    if (hipGetDevice(&dev) != hipSuccess ||
        hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus < 1)
        cus = 256;
    return 2 * kFaSlotFloats * balanced_prefill_workgroups(tiles * heads_kv, std::max<int64_t>(0, max_keys), cus);
}

int pth_fa_forward_balanced(const pd_tensor* q, const pd_tensor* key_cache, const pd_tensor* value_cache,
                            const pd_tensor* block_table, const pd_tensor* seq_lens, double scale,
                            const pd_tensor* q_abs_offset, const int* query_start, int64_t num_seqs, const pd_tensor* out,
                            const pd_tensor* workspace, int64_t max_keys, int64_t nsplit, int64_t exact, hipStream_t stream,
                            char* err, int errlen) {
    if (query_start) {
        if (!q || !key_cache || !value_cache || !block_table || !seq_lens || !out)
            return fail(err, errlen, "null tensor descriptor");
        return fa_forward_rows(q, key_cache, value_cache, block_table, seq_lens, scale, query_start, num_seqs, out, workspace,
                               max_keys, nsplit, exact != 0, stream, err, errlen);
    }
    if (nsplit != 0) return fail(err, errlen, "nsplit must be 0 in the batch form");
    return fa_forward(q, key_cache, value_cache, block_table, seq_lens, scale, q_abs_offset, out, stream, err, errlen,
                      exact != 0, 1, workspace, &max_keys);
}

int pth_cache_write(const pd_tensor* key, const pd_tensor* value, const pd_tensor* key_cache,
                    const pd_tensor* value_cache, const pd_tensor* k_scale, const pd_tensor* v_scale,
                    const pd_tensor* slot_mapping, hipStream_t stream, char* err, int errlen) {
    if (!key || !value || !key_cache || !value_cache || !k_scale || !v_scale || !slot_mapping)
        return fail(err, errlen, "null tensor descriptor");
    if (!layout_ok(key_cache, value_cache, k_scale, v_scale))
        return fail(err, errlen, "KV cache views do not have the int8 per-token-head row layout");
    const int dt = key->dtype;
    if (!((dt == PD_DTYPE_FP16 || dt == PD_DTYPE_BF16 || dt == PD_DTYPE_FP32) && value->dtype == dt))
        return fail(err, errlen, "key and value must be fp16, bf16 or fp32 of the same dtype");
    const int64_t T = key->sizes[0], Hkv = key_cache->sizes[2];
    if (!(key->ndim == 3 && value->ndim == 3 && key->sizes[1] == Hkv && value->sizes[1] == Hkv &&
          key->sizes[2] == 256 && value->sizes[2] == 256 && value->sizes[0] == T && key->strides[2] == 1 &&
          value->strides[2] == 1))
        return fail(err, errlen, "key and value must be [T, Hkv, 256] with unit dim stride");
    if (T * Hkv > ((int64_t)1 << 30)) return fail(err, errlen, "at most 2^30 (token, kv head) rows per call");
    const int64_t esz = dt == PD_DTYPE_FP32 ? 4 : 2;
    const int64_t vec = 4 * esz;  // each lane loads 4 elements
    if (!((reinterpret_cast<uintptr_t>(key->data) % vec) == 0 && (reinterpret_cast<uintptr_t>(value->data) % vec) == 0 &&
          key->strides[0] % 4 == 0 && key->strides[1] % 4 == 0 && value->strides[0] % 4 == 0 &&
          value->strides[1] % 4 == 0))
        return fail(err, errlen, "key and value rows must be aligned to 4 elements");
    if (!(slot_mapping->dtype == PD_DTYPE_INT64 && slot_mapping->ndim == 1 && slot_mapping->sizes[0] >= T &&
          (slot_mapping->strides[0] == 1 || slot_mapping->sizes[0] <= 1)))
        return fail(err, errlen, "slot_mapping must be a contiguous int64 [T]");
    if (T == 0) return 0;
    CacheWriteParams p;
    p.key = key->data;
    p.value = value->data;
    p.k_st = key->strides[0];
    p.k_sh = key->strides[1];
    p.v_st = value->strides[0];
    p.v_sh = value->strides[1];
    p.kc = static_cast<int8_t*>(const_cast<void*>(key_cache->data));
    p.k_sb = key_cache->strides[0];
    p.k_ss = key_cache->strides[1];
    p.k_sh_c = key_cache->strides[2];
    p.slots = static_cast<const int64_t*>(slot_mapping->data);
    p.block_size = (int)key_cache->sizes[1];
    p.num_slots = key_cache->sizes[0] * key_cache->sizes[1];
    p.T = (int)T;
    p.Hkv = (int)Hkv;
    const hipError_t e = pd::launch_cache_write(p, dt, stream);
    if (e != hipSuccess) {
        char msg[256];
        snprintf(msg, sizeof msg, "cache write launch failed: %s", hipGetErrorString(e));
        fail(err, errlen, msg);
        return 2;
    }
    return 0;
}

static int op_result(hipError_t e, const char* what, char* err, int errlen) {
    if (e == hipSuccess) return 0;
    char msg[256];
    snprintf(msg, sizeof msg, "%s launch failed: %s", what, hipGetErrorString(e));
    fail(err, errlen, msg);
    return 2;
}

// Heads of 256 values that can be loaded four at a time: data and strides aligned to four elements.
static bool heads_of_4(const pd_tensor* t, int64_t esz) {
    return reinterpret_cast<uintptr_t>(t->data) % (uintptr_t)(4 * esz) == 0 && t->strides[0] % 4 == 0 && t->strides[1] % 4 == 0;
}

// Whether the rows of `len` elements of an output's first n0 x sizes[1] (dims 0 and 1) are apart: no element has two writers.
static bool rows_apart(const pd_tensor* t, int64_t n0, int64_t len) {
    int64_t n[2] = {n0, t->sizes[1]}, st[2] = {t->strides[0], t->strides[1]};
    if (n[1] <= 1 || (n[0] > 1 && st[0] < st[1])) std::swap(n[0], n[1]), std::swap(st[0], st[1]);  // the smaller stride second
    if (n[1] <= 1 || len == 0) return true;
    return st[1] >= len && (n[0] <= 1 || (st[0] - len) / st[1] >= n[1] - 1);
}

// Rows of `len` bytes that a call reads or writes: n[0] x n[1] of them, st bytes apart.
struct ByteRows {
    uintptr_t at;
    int64_t n[2], st[2], len;
};
static ByteRows byte_rows(const pd_tensor* t, int64_t n0, int64_t len, int64_t esz) {
    const bool two = t->ndim == 3;
    return {reinterpret_cast<uintptr_t>(t->data), {n0, two ? t->sizes[1] : 1}, {t->strides[0] * esz, two ? t->strides[1] * esz : 0}, len * esz};
}
// The first n0 elements or rows of a tensor of one or two dims, its last dim contiguous.
static ByteRows byte_span(const pd_tensor* t, int64_t n0, int64_t esz) {
    if (t->ndim == 1) return {reinterpret_cast<uintptr_t>(t->data), {1, 1}, {0, 0}, n0 * esz};
    return byte_rows(t, n0, t->sizes[1], esz);
}

// Whether two tensors' rows surely share no byte: their extents are apart, or both repeat with one stride and lie apart in a period
// of it (heads of one fused buffer, say). Rows of other strides within one another's extent count as overlapping.
static bool apart(const ByteRows& a, const ByteRows& b) {
    if (a.n[0] <= 0 || a.n[1] <= 0 || a.len <= 0 || b.n[0] <= 0 || b.n[1] <= 0 || b.len <= 0) return true;
    auto extent = [](const ByteRows& r) { return (uint64_t)((r.n[0] - 1) * r.st[0] + (r.n[1] - 1) * r.st[1] + r.len); };
    if (a.at + extent(a) <= b.at || b.at + extent(b) <= a.at) return true;
    for (int d = 0; d < 2; ++d) {
        const int o = 1 - d;
        const int64_t s = a.n[d] > 1 ? a.st[d] : b.st[d];
        if (s <= 0 || (a.n[d] <= 1 && b.n[d] <= 1) || (a.n[d] > 1 && b.n[d] > 1 && a.st[d] != b.st[d])) continue;
        // bytes of a period that the rows of the other dim take (those a whole number of periods on fall together)
        auto width = [&](const ByteRows& r) { return r.n[o] <= 1 || r.st[o] % s == 0 ? r.len : (r.n[o] - 1) * r.st[o] + r.len; };
        const uint64_t gap = b.at >= a.at ? (b.at - a.at) % (uint64_t)s : ((uint64_t)s - (a.at - b.at) % (uint64_t)s) % (uint64_t)s;
        if (gap >= (uint64_t)width(a) && gap + (uint64_t)width(b) <= (uint64_t)s) return true;
    }
    return false;
}

// What a windowed prefill writes against all that it touches (workspace: null if the call has none).
static bool window_tensors_apart(const pd_tensor* q, const pd_tensor* kc, const pd_tensor* block_table, const pd_tensor* seq_lens,
                                 const pd_tensor* query_start, const pd_tensor* out, const pd_tensor* workspace, int64_t num_seqs,
                                 int64_t ws_floats) {
    const ByteRows cache = {reinterpret_cast<uintptr_t>(kc->data), {1, 1}, {0, 0}, kc->sizes[0] > 0 ? cache_span(kc) - 8 + kRowBytes : 0};
    const ByteRows reads[] = {byte_rows(q, q->sizes[0], kDim, 2), cache, byte_span(block_table, num_seqs, 4), byte_span(seq_lens, num_seqs, 4),
                              byte_span(query_start, num_seqs + 1, 4)};
    const ByteRows rows = byte_rows(out, out->sizes[0], kDim, 2);
    for (const ByteRows& r : reads)
        if (!apart(rows, r)) return false;
    if (!workspace) return true;
    const ByteRows ws = byte_span(workspace, ws_floats, 4);
    for (const ByteRows& r : reads)
        if (!apart(ws, r)) return false;
    return apart(rows, ws);
}

// The norms of a rotary write's query and key heads.
struct HeadNorms {
    const pd_tensor *q_weight, *k_weight;
    double eps, offset;
};

static int rotary_entry(const pd_tensor* query, const pd_tensor* query_out, const pd_tensor* key, const pd_tensor* value,
                        const pd_tensor* positions, const pd_tensor* cos_sin, const pd_tensor* key_cache,
                        const pd_tensor* value_cache, const pd_tensor* k_scale, const pd_tensor* v_scale,
                        const pd_tensor* slot_mapping, int64_t interleaved, hipStream_t stream, char* err, int errlen,
                        const HeadNorms* norms = nullptr) {
    if (!query || !query_out || !key || !value || !positions || !cos_sin || !key_cache || !value_cache || !k_scale ||
        !v_scale || !slot_mapping)
        return fail(err, errlen, "null tensor descriptor");
    if (!layout_ok(key_cache, value_cache, k_scale, v_scale))
        return fail(err, errlen, "KV cache views do not have the int8 per-token-head row layout");
    const int dt = query->dtype;
    if (!((dt == PD_DTYPE_FP16 || dt == PD_DTYPE_BF16 || dt == PD_DTYPE_FP32) && key->dtype == dt && value->dtype == dt))
        return fail(err, errlen, "query, key and value must be fp16, bf16 or fp32 of the same dtype");
    if (!(query->ndim == 3 && query->sizes[1] > 0 && query->sizes[2] == kDim && query->strides[2] == 1))
        return fail(err, errlen, "query must be [T, Hq, 256] with unit dim stride");
    const int64_t T = query->sizes[0], Hq = query->sizes[1], Hkv = key_cache->sizes[2];
    if (!(key->ndim == 3 && value->ndim == 3 && key->sizes[0] == T && value->sizes[0] == T && key->sizes[1] == Hkv &&
          value->sizes[1] == Hkv && key->sizes[2] == kDim && value->sizes[2] == kDim && key->strides[2] == 1 &&
          value->strides[2] == 1))
        return fail(err, errlen, "key and value must be [T, Hkv, 256] with unit dim stride");
    const int out_dt = query_out->dtype;
    if (!((out_dt == dt || out_dt == PD_DTYPE_FP16) && query_out->ndim == 3 && query_out->sizes[0] == T &&
          query_out->sizes[1] == Hq && query_out->sizes[2] == kDim && query_out->strides[2] == 1))
        return fail(err, errlen, "query_out must be [T, Hq, 256] with unit dim stride, of the query's dtype or fp16");
    if (Hq > (1 << 20) || Hkv > (1 << 20) || T > ((int64_t)1 << 30) || T * Hq > ((int64_t)1 << 30) || T * Hkv > ((int64_t)1 << 30))
        return fail(err, errlen, "at most 2^30 (token, head) rows per call");
    const int64_t esz = dt == PD_DTYPE_FP32 ? 4 : 2, osz = out_dt == PD_DTYPE_FP32 ? 4 : 2;
    if (!(heads_of_4(query, esz) && heads_of_4(key, esz) && heads_of_4(value, esz) && heads_of_4(query_out, osz)))
        return fail(err, errlen, "query, query_out, key and value rows must be aligned to 4 elements");
    if (!rows_apart(query_out, T, kDim)) return fail(err, errlen, "query_out rows must not overlap");
    const bool in_place = T > 0 && query_out->data == query->data;  // (all empty tensors are at null)
    if (in_place && !(out_dt == dt && query_out->strides[0] == query->strides[0] && query_out->strides[1] == query->strides[1]))
        return fail(err, errlen, "query_out must be the query itself or not overlap it");
    const ByteRows written = byte_rows(query_out, T, kDim, osz);
    if (!in_place && !apart(written, byte_rows(query, T, kDim, esz)))
        return fail(err, errlen, "query_out must be the query itself or not overlap it");
    if (!apart(written, byte_rows(key, T, kDim, esz)) || !apart(written, byte_rows(value, T, kDim, esz)))
        return fail(err, errlen, "query_out must not overlap key or value");
    if (!(positions->dtype == PD_DTYPE_INT64 && positions->ndim == 1 && positions->sizes[0] >= T &&
          (positions->strides[0] == 1 || positions->sizes[0] <= 1)))
        return fail(err, errlen, "positions must be a contiguous int64 [T]");
    if (!(slot_mapping->dtype == PD_DTYPE_INT64 && slot_mapping->ndim == 1 && slot_mapping->sizes[0] >= T &&
          (slot_mapping->strides[0] == 1 || slot_mapping->sizes[0] <= 1)))
        return fail(err, errlen, "slot_mapping must be a contiguous int64 [T]");
    if (norms) {
        for (const pd_tensor* w : {norms->q_weight, norms->k_weight}) {
            if (!((w->dtype == dt || w->dtype == PD_DTYPE_FP32) && w->dtype == norms->q_weight->dtype && w->ndim == 1 &&
                  w->sizes[0] == kDim && w->strides[0] == 1 &&
                  reinterpret_cast<uintptr_t>(w->data) % (w->dtype == PD_DTYPE_FP32 ? 16 : 8) == 0))
                return fail(err, errlen, "query_weight and key_weight must be contiguous [256] of one dtype, the query's or fp32, aligned to 4 elements");
            if (!apart(written, byte_span(w, kDim, w->dtype == PD_DTYPE_FP32 ? 4 : 2)))
                return fail(err, errlen, "query_out must not overlap the weights");
        }
        if (!(norms->eps >= 0 && norms->eps < 1e30 && norms->offset > -1e30 && norms->offset < 1e30))
            return fail(err, errlen, "eps must be at least 0 and finite, weight_offset finite");
    }
    const int64_t rd = cos_sin->ndim == 2 ? cos_sin->sizes[1] : 0;
    if (!(cos_sin->dtype == PD_DTYPE_FP32 && cos_sin->ndim == 2 && rd >= 8 && rd <= kDim && rd % 8 == 0 &&
          cos_sin->strides[1] == 1 && cos_sin->strides[0] % 4 == 0 && reinterpret_cast<uintptr_t>(cos_sin->data) % 16 == 0))
        return fail(err, errlen, "cos_sin must be fp32 [positions, rotary_dim], 16-byte aligned rows, rotary_dim a multiple of 8 up to 256");
    if (T == 0) return 0;
    RotaryWriteParams p = {};
    p.query = query->data;
    p.query_out = const_cast<void*>(query_out->data);
    p.key = key->data;
    p.value = value->data;
    p.q_st = query->strides[0];
    p.q_sh = query->strides[1];
    p.o_st = query_out->strides[0];
    p.o_sh = query_out->strides[1];
    p.k_st = key->strides[0];
    p.k_sh = key->strides[1];
    p.v_st = value->strides[0];
    p.v_sh = value->strides[1];
    p.positions = static_cast<const int64_t*>(positions->data);
    p.cos_sin = static_cast<const float*>(cos_sin->data);
    p.cs_st = cos_sin->strides[0];
    p.max_positions = cos_sin->sizes[0];
    p.kc = static_cast<int8_t*>(const_cast<void*>(key_cache->data));
    p.c_sb = key_cache->strides[0];
    p.c_ss = key_cache->strides[1];
    p.c_sh = key_cache->strides[2];
    p.slots = static_cast<const int64_t*>(slot_mapping->data);
    p.num_slots = key_cache->sizes[0] * key_cache->sizes[1];
    p.T = (int)T;
    p.Hq = (int)Hq;
    p.Hkv = (int)Hkv;
    p.block_size = (int)key_cache->sizes[1];
    p.rotary_dim = (int)rd;
    p.interleaved = interleaved != 0;
    p.in_place = in_place;
    if (norms) {
        p.q_weight = norms->q_weight->data;
        p.k_weight = norms->k_weight->data;
        p.weight_fp32 = norms->q_weight->dtype == PD_DTYPE_FP32;
        p.eps = (float)norms->eps;
        p.weight_offset = (float)norms->offset;
    }
    return op_result(launch_rotary_write(p, dt, out_dt, stream), "rotary cache write", err, errlen);
}

int pth_cache_write_rotary(const pd_tensor* query, const pd_tensor* query_out, const pd_tensor* key, const pd_tensor* value,
                           const pd_tensor* positions, const pd_tensor* cos_sin, const pd_tensor* key_cache,
                           const pd_tensor* value_cache, const pd_tensor* k_scale, const pd_tensor* v_scale,
                           const pd_tensor* slot_mapping, int64_t interleaved, hipStream_t stream, char* err, int errlen) {
    return rotary_entry(query, query_out, key, value, positions, cos_sin, key_cache, value_cache, k_scale, v_scale, slot_mapping,
                        interleaved, stream, err, errlen);
}

int pth_cache_write_norm_rotary(const pd_tensor* query, const pd_tensor* query_out, const pd_tensor* key, const pd_tensor* value,
                                const pd_tensor* query_weight, const pd_tensor* key_weight, double eps, double weight_offset,
                                const pd_tensor* positions, const pd_tensor* cos_sin, const pd_tensor* key_cache,
                                const pd_tensor* value_cache, const pd_tensor* k_scale, const pd_tensor* v_scale,
                                const pd_tensor* slot_mapping, int64_t interleaved, hipStream_t stream, char* err, int errlen) {
    if (!query_weight || !key_weight) return fail(err, errlen, "null tensor descriptor");
    const HeadNorms norms = {query_weight, key_weight, eps, weight_offset};
    return rotary_entry(query, query_out, key, value, positions, cos_sin, key_cache, value_cache, k_scale, v_scale, slot_mapping,
                        interleaved, stream, err, errlen, &norms);
}

// The batch of a decode step as the weights and the eviction take it.
static bool int_rows(const pd_tensor* t, int64_t n) { return t->dtype == PD_DTYPE_INT32 && t->ndim == 1 && is_contig(t) && t->sizes[0] >= n; }
static bool int_table(const pd_tensor* t, int64_t n) {
    return t->dtype == PD_DTYPE_INT32 && t->ndim == 2 && t->strides[1] == 1 && t->sizes[0] >= n && t->sizes[1] <= INT32_MAX;
}
// Keys of a row of weights, and that stay: the kernels step over them in 32 bits, and a launch copies 32 to a workgroup.
constexpr int64_t kMaxWeightKeys = (int64_t)1 << 28;
// fp32 [>= num_seqs, Hkv, keys] with its keys side by side
static bool weight_rows(const pd_tensor* t, int64_t n, int64_t hkv) {
    return t->dtype == PD_DTYPE_FP32 && t->ndim == 3 && t->sizes[0] >= n && t->sizes[1] == hkv && t->sizes[2] <= kMaxWeightKeys &&
           (t->strides[2] == 1 || t->sizes[2] <= 1);
}

int pth_cache_key_weights(const pd_tensor* q, const pd_tensor* key_cache, const pd_tensor* value_cache, const pd_tensor* k_scale,
                    const pd_tensor* v_scale, const pd_tensor* block_table, const pd_tensor* seq_lens,
                    const pd_tensor* query_start_loc, const pd_tensor* lse, const pd_tensor* weights, double scale,
                    int64_t num_seqs, int64_t qmax, hipStream_t stream, char* err, int errlen) {
    if (!q || !key_cache || !value_cache || !k_scale || !v_scale || !block_table || !seq_lens || !query_start_loc || !lse ||
        !weights)
        return fail(err, errlen, "null tensor descriptor");
    if (!(q->dtype == PD_DTYPE_FP16 && q->ndim == 3 && q->sizes[2] == 256 && q->strides[2] == 1 &&
          q->strides[1] == 256 && q->strides[0] % 2 == 0 && (reinterpret_cast<uintptr_t>(q->data) % 4) == 0))
        return fail(err, errlen, "q must be fp16 [T, Hq, 256] with contiguous heads");
    if (!layout_ok(key_cache, value_cache, k_scale, v_scale))
        return fail(err, errlen, "KV cache views do not have the int8 per-token-head row layout");
    const int64_t T = q->sizes[0], Hq = q->sizes[1], Hkv = key_cache->sizes[2], bs = key_cache->sizes[1];
    if (!(Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && T <= INT32_MAX && Hq <= INT32_MAX && Hkv <= 65535))
        return fail(err, errlen, "heads_q must be a multiple of heads_kv");
    if (!(qmax >= 1 && qmax <= INT32_MAX && qmax * (Hq / Hkv) <= 16 * kMaxRowBlocks))
        return fail(err, errlen, "qmax * (Hq / Hkv) must be in [1, 48]");
    if (!(num_seqs >= 1 && num_seqs <= 65535 && int_table(block_table, num_seqs) && int_rows(seq_lens, num_seqs) &&
          int_rows(query_start_loc, num_seqs + 1)))
        return fail(err, errlen, "block_table / seq_lens / query_start_loc must be int32 with a row for each of 1 to 65535 sequences");
    if (const char* why = lse_refused(lse, T, Hq)) return fail(err, errlen, why);
    if (!(weight_rows(weights, num_seqs, Hkv) && rows_apart(weights, num_seqs, weights->sizes[2])))
        return fail(err, errlen, "weights must be fp32 [num_seqs, Hkv, keys] of at most 2^28 keys with unit key stride, its rows apart");
    if (T == 0 || weights->sizes[2] == 0) return 0;
    KeyWeightsParams p = {};
    p.q = static_cast<const _Float16*>(q->data);
    p.q_st = q->strides[0];
    p.kc = static_cast<const int8_t*>(key_cache->data);
    p.k_sb = key_cache->strides[0];
    p.k_ss = key_cache->strides[1];
    p.k_sh = key_cache->strides[2];
    p.block_table = static_cast<const int*>(block_table->data);
    p.bt_stride = block_table->strides[0];
    p.seq_lens = static_cast<const int*>(seq_lens->data);
    p.qsl = static_cast<const int*>(query_start_loc->data);
    p.lse = static_cast<const float*>(lse->data);
    p.weights = static_cast<float*>(const_cast<void*>(weights->data));
    p.w_sb = weights->strides[0];
    p.w_sh = weights->strides[1];
    p.max_keys = (int)weights->sizes[2];
    p.block_size = (int)bs;
    p.bs_shift = (bs & (bs - 1)) == 0 ? __builtin_ctz((unsigned)bs) : -1;
    p.G = (int)(Hq / Hkv);
    p.Hq = (int)Hq;
    p.qmax = (int)qmax;
    p.table_keys = block_table->sizes[1] * bs;
    p.scale_log2 = (float)scale * 1.4426950408889634f;
    return op_result(launch_key_weights(p, (int)num_seqs, (int)Hkv, stream), "key weights", err, errlen);
}

int pth_cache_evict(const pd_tensor* weights, const pd_tensor* key_cache, const pd_tensor* value_cache, const pd_tensor* k_scale,
              const pd_tensor* v_scale, const pd_tensor* block_table, const pd_tensor* seq_lens,
              const pd_tensor* new_block_table, const pd_tensor* new_seq_lens, const pd_tensor* new_weights,
              const pd_tensor* kept, int64_t num_seqs, int64_t keep, int64_t recent, hipStream_t stream, char* err, int errlen) {
    if (!weights || !key_cache || !value_cache || !k_scale || !v_scale || !block_table || !seq_lens || !new_block_table ||
        !new_seq_lens || !new_weights || !kept)
        return fail(err, errlen, "null tensor descriptor");
    if (!layout_ok(key_cache, value_cache, k_scale, v_scale))
        return fail(err, errlen, "KV cache views do not have the int8 per-token-head row layout");
    const int64_t Hkv = key_cache->sizes[2], bs = key_cache->sizes[1];
    if (!(keep >= 1 && keep <= kMaxWeightKeys && recent >= 0 && recent <= keep))
        return fail(err, errlen, "keep must be in [1, 2^28] and recent in [0, keep]");
    if (!(num_seqs >= 1 && num_seqs <= 65535 && Hkv >= 1 && Hkv <= 65535 && int_table(block_table, num_seqs) &&
          int_rows(seq_lens, num_seqs) && int_table(new_block_table, num_seqs) && int_rows(new_seq_lens, num_seqs)))
        return fail(err, errlen, "block tables and sequence lengths must be int32 with a row for each of 1 to 65535 sequences");
    if (new_block_table->sizes[1] * bs < keep) return fail(err, errlen, "new_block_table must hold keep keys");
    if (!(weight_rows(weights, num_seqs, Hkv) && weight_rows(new_weights, num_seqs, Hkv) && new_weights->sizes[2] >= keep &&
          rows_apart(new_weights, num_seqs, new_weights->sizes[2])))
        return fail(err, errlen, "weights and new_weights must be fp32 [num_seqs, Hkv, keys] of at most 2^28 keys with unit key stride, new_weights of at least keep keys, its rows apart");
    if (!(kept->dtype == PD_DTYPE_INT32 && kept->ndim == 3 && kept->sizes[0] >= num_seqs && kept->sizes[1] == Hkv &&
          kept->sizes[2] == keep && is_contig(kept)))
        return fail(err, errlen, "kept must be contiguous int32 [num_seqs, Hkv, keep]");
    if (new_weights->data == weights->data || new_seq_lens->data == seq_lens->data || new_block_table->data == block_table->data)
        return fail(err, errlen, "the new tensors must not be the old ones: eviction copies to other blocks");
    const ByteRows outs[] = {byte_rows(new_weights, num_seqs, new_weights->sizes[2], 4), byte_rows(kept, num_seqs, keep, 4),
                             byte_span(new_seq_lens, num_seqs, 4)};
    const ByteRows ins[] = {byte_rows(weights, num_seqs, weights->sizes[2], 4), byte_span(seq_lens, num_seqs, 4),
                            byte_span(block_table, num_seqs, 4), byte_span(new_block_table, num_seqs, 4)};
    for (const ByteRows& x : outs) {
        for (const ByteRows& y : ins)
            if (!apart(x, y)) return fail(err, errlen, "the tensors that eviction writes must not overlap those that it reads");
        for (const ByteRows& y : outs)
            if (&x != &y && !apart(x, y)) return fail(err, errlen, "the tensors that eviction writes must not overlap");
    }
    EvictParams p = {};
    p.weights = static_cast<const float*>(weights->data);
    p.w_sb = weights->strides[0];
    p.w_sh = weights->strides[1];
    p.new_weights = static_cast<float*>(const_cast<void*>(new_weights->data));
    p.n_sb = new_weights->strides[0];
    p.n_sh = new_weights->strides[1];
    p.max_keys = (int)std::min(weights->sizes[2], block_table->sizes[1] * bs);
    p.new_keys = (int)new_weights->sizes[2];
    p.kept = static_cast<int*>(const_cast<void*>(kept->data));
    p.seq_lens = static_cast<const int*>(seq_lens->data);
    p.new_lens = static_cast<int*>(const_cast<void*>(new_seq_lens->data));
    p.kc = static_cast<int8_t*>(const_cast<void*>(key_cache->data));
    p.k_sb = key_cache->strides[0];
    p.k_ss = key_cache->strides[1];
    p.k_sh = key_cache->strides[2];
    p.block_table = static_cast<const int*>(block_table->data);
    p.bt_stride = block_table->strides[0];
    p.new_table = static_cast<const int*>(new_block_table->data);
    p.nt_stride = new_block_table->strides[0];
    p.block_size = (int)bs;
    p.Hkv = (int)Hkv;
    p.keep = (int)keep;
    p.recent = (int)recent;
    return op_result(launch_evict(p, (int)num_seqs, stream), "evict", err, errlen);
}

// Whether the rows of a raw cache [pages, Hkv, keys, 520] are apart: in the order of the strides, each spans the dims below it.
static bool cache_rows_apart(const pd_tensor* kv) {
    int order[3] = {0, 1, 2};
    std::sort(order, order + 3, [&](int a, int b) {
        return kv->strides[a] != kv->strides[b] ? kv->strides[a] < kv->strides[b] : kv->sizes[a] < kv->sizes[b];
    });
    int64_t span = kRowBytes;
    for (int d : order) {
        if (kv->sizes[d] <= 1) continue;
        if (kv->strides[d] < span || kv->strides[d] > INT64_MAX / 4 / kv->sizes[d]) return false;
        span = kv->strides[d] * (kv->sizes[d] - 1) + span;
    }
    return true;
}

namespace {
// Where the rows of caches of one geometry lie: strides that fall, how often each is taken, and how far it and those below reach. Below a
// stride the others reach less far than it (cache_rows_apart).
struct RowLattice {
    int64_t st[3], most[3], reach[4];
    explicit RowLattice(const pd_tensor* kv) {
        int order[3] = {0, 1, 2};
        std::sort(order, order + 3, [&](int a, int b) { return (kv->sizes[a] > 1 ? kv->strides[a] : 0) > (kv->sizes[b] > 1 ? kv->strides[b] : 0); });
        reach[3] = kRowBytes;
        for (int i = 2; i >= 0; --i) {
            st[i] = kv->strides[order[i]], most[i] = kv->sizes[order[i]] - 1;
            reach[i] = reach[i + 1] + most[i] * st[i];
        }
    }
    // Whether rows of two caches that begin d bytes apart share a byte: some sum of a[i] st[i] with |a[i]| <= most[i] is less than a row
    // from d. Only the two multiples of a stride beside d can be.
    bool meet(int64_t d, int i = 0) const {
        if (std::abs(d) >= reach[i]) return false;
        if (i == 3) return true;
        if (most[i] == 0) return meet(d, i + 1);
        const int64_t a = d / st[i] - (d % st[i] < 0);
        return (std::abs(a) <= most[i] && meet(d - a * st[i], i + 1)) || (std::abs(a + 1) <= most[i] && meet(d - (a + 1) * st[i], i + 1));
    }
};
}  // namespace
// Whether rows of different caches (sorted) share a byte.
static bool caches_meet(const PageCaches& k, const RowLattice& rows) {
    bool near = false;
    for (int i = 1; i < k.layers; ++i) near = near || k.kv[i] - k.kv[i - 1] < rows.reach[0];
    if (!near) return false;
    if (rows.most[0] > 0) {  // interleaved layers: apart in every period of the largest stride
        int64_t at[kMaxPageLayers];
        for (int i = 0; i < k.layers; ++i) at[i] = (k.kv[i] - k.kv[0]) % rows.st[0];
        std::sort(at, at + k.layers, [](int64_t a, int64_t b) { return a < b; });
        bool clear = at[0] + rows.st[0] - at[k.layers - 1] >= rows.reach[1];
        for (int i = 1; i < k.layers; ++i) clear = clear && at[i] - at[i - 1] >= rows.reach[1];
        if (clear) return false;
    }
    for (int i = 0; i < k.layers; ++i)
        for (int j = i + 1; j < k.layers && k.kv[j] - k.kv[i] < rows.reach[0]; ++j)
            if (rows.meet(k.kv[j] - k.kv[i])) return true;
    return false;
}
// Whether a tensor lies clear of all caches (sorted, `extent` bytes each).
static bool clear_of_caches(const PageCaches& k, int64_t extent, const ByteRows& r) {
    if (r.n[0] <= 0 || r.n[1] <= 0 || r.len <= 0) return true;
    const uintptr_t end = r.at + (uint64_t)((r.n[0] - 1) * r.st[0] + (r.n[1] - 1) * r.st[1] + r.len);
    // of the caches that begin before its end the last one ends last
    int8_t* const* past = std::lower_bound(k.kv, k.kv + k.layers, reinterpret_cast<int8_t*>(end));
    return past == k.kv || reinterpret_cast<uintptr_t>(past[-1]) + (uint64_t)extent <= r.at;
}

// The caches and the table rows that a page operator takes; null, or why not. A cache that is given twice (layers that share one) is
// taken once.
static const char* page_caches(const pd_tensor* caches, int64_t layers, PageCaches& k) {
    if (!(layers >= 1 && layers <= kMaxPageLayers)) return "1 to 128 caches per call";
    for (int64_t i = 0; i < layers; ++i) {
        const pd_tensor& c = caches[i];
        if (!(c.dtype == PD_DTYPE_INT8 && c.ndim == 4 && c.sizes[3] == kRowBytes && c.strides[3] == 1 &&
              reinterpret_cast<uintptr_t>(c.data) % 8 == 0))
            return "caches must be int8 [pages, Hkv, block_size, 520] with contiguous, 8-byte aligned rows";
        for (int d = 0; d < 3; ++d) {
            if (c.strides[d] % 8 != 0) return "caches must be int8 [pages, Hkv, block_size, 520] with contiguous, 8-byte aligned rows";
            if (c.sizes[d] != caches[0].sizes[d] || c.strides[d] != caches[0].strides[d])
                return "the caches of a call must have the same sizes and strides";
        }
        k.kv[i] = static_cast<int8_t*>(const_cast<void*>(c.data));
    }
    const pd_tensor& c = caches[0];
    if (!(c.sizes[0] >= 1 && c.sizes[0] <= kMaxPages && c.sizes[1] >= 1 && c.sizes[1] <= (1 << 20) && c.sizes[2] >= 1 &&
          c.sizes[2] <= (1 << 20) && c.sizes[1] * c.sizes[2] <= (1 << 20)))
        return "caches of 1 to 2^22 pages of 1 to 2^20 rows";
    if (!cache_rows_apart(&c)) return "cache rows must not overlap";
    std::sort(k.kv, k.kv + layers, [](const int8_t* a, const int8_t* b) { return a < b; });
    k.layers = (int)(std::unique(k.kv, k.kv + layers) - k.kv);
    if (caches_meet(k, RowLattice(&c))) return "the caches' rows must not overlap";
    k.sb = c.strides[0];
    k.sh = c.strides[1];
    k.ss = c.strides[2];
    k.Hkv = (int)c.sizes[1];
    k.block_size = (int)c.sizes[2];
    return nullptr;
}
static bool page_table_rows(const pd_tensor* t, int64_t most) {
    return t->dtype == PD_DTYPE_INT32 && t->ndim == 2 && (t->strides[1] == 1 || t->sizes[1] <= 1) && t->sizes[0] <= most &&
           t->sizes[1] <= INT32_MAX / 2;
}
static bool table_rows_apart(const pd_tensor* t) { return t->sizes[0] <= 1 || t->strides[0] >= t->sizes[1]; }
// Workspace ints: both masks, the counts, and for a fork the rows' plans.
static int64_t page_work_ints(int64_t pages, int64_t rows, int64_t new_rows) {
    const int64_t chunks = (pages + 1023) / 1024;
    return chunks * (2 * 32 + 1) + rows + 4 * new_rows + 1;
}
static const char* page_work(const pd_tensor* ws, int64_t pages, int64_t ints, PageWork& w) {
    if (!(ws->dtype == PD_DTYPE_INT32 && ws->ndim == 1 && is_contig(ws) && ws->sizes[0] >= ints &&
          reinterpret_cast<uintptr_t>(ws->data) % 16 == 0))
        return "workspace must be contiguous 16-byte aligned int32 of pth_cache_pages_workspace";
    w.pages = (int)pages;
    w.chunks = (int)((pages + 1023) / 1024);
    w.free_mask = static_cast<unsigned long long*>(const_cast<void*>(ws->data));
    w.alone_mask = w.free_mask + 16 * w.chunks;
    w.counts = reinterpret_cast<int*>(w.alone_mask + 16 * w.chunks);
    return nullptr;
}
// Whether an output is the input itself (data and strides) or apart from it.
static bool same_or_apart(const pd_tensor* out, const pd_tensor* in, int64_t n_out, int64_t n_in, bool may_be_same) {
    const bool same = out->data == in->data && out->ndim == in->ndim && (out->ndim == 1 || (out->strides[0] == in->strides[0] &&
                      out->sizes[1] == in->sizes[1]));
    return (same && may_be_same) || apart(byte_span(out, n_out, 4), byte_span(in, n_in, 4));
}

int64_t pth_cache_pages_workspace(int64_t pages, int64_t rows, int64_t new_rows) {
    if (pages < 1 || pages > kMaxPages || rows < 0 || rows > INT32_MAX || new_rows < 0 || new_rows > INT32_MAX) return 0;
    return page_work_ints(pages, rows, new_rows);
}

int pth_cache_fork_pages(const pd_tensor* caches, int64_t layers, const pd_tensor* refs, const pd_tensor* block_table,
                         const pd_tensor* seq_lens, const pd_tensor* parents, const pd_tensor* new_refs,
                         const pd_tensor* new_block_table, const pd_tensor* new_seq_lens, const pd_tensor* needed,
                         const pd_tensor* workspace, int64_t grow, int64_t window, int64_t sinks, hipStream_t stream, char* err,
                         int errlen) {
    if (!caches || !refs || !block_table || !seq_lens || !new_refs || !new_block_table || !new_seq_lens || !needed || !workspace)
        return fail(err, errlen, "null tensor descriptor");
    ForkParams p = {};
    PageCaches k = {};
    if (const char* why = page_caches(caches, layers, k)) return fail(err, errlen, why);
    const int64_t pages = caches[0].sizes[0];
    if (!(int_rows(refs, pages) && refs->sizes[0] == pages && int_rows(new_refs, pages) && new_refs->sizes[0] == pages))
        return fail(err, errlen, "refs and new_refs must be contiguous int32 with an entry for each page");
    if (!(page_table_rows(block_table, kMaxForkRows) && page_table_rows(new_block_table, kMaxForkRows) &&
          new_block_table->sizes[1] == block_table->sizes[1]))
        return fail(err, errlen, "block tables must be int32 of at most 8192 rows, with the same columns");
    const int64_t B = block_table->sizes[0], N = new_block_table->sizes[0];
    // (the pages that all rows want are counted in 32 bits)
    if (N * new_block_table->sizes[1] > INT32_MAX) return fail(err, errlen, "at most 2^31 - 1 entries in the new block table");
    if (!(int_rows(seq_lens, B) && int_rows(new_seq_lens, N))) return fail(err, errlen, "sequence lengths must be contiguous int32 with an entry for each row");
    if (parents ? !int_rows(parents, N) : N != B)
        return fail(err, errlen, "parents must be contiguous int32 with an entry for each new row (none: as many new rows as old)");
    if (!int_rows(needed, 1)) return fail(err, errlen, "needed must be int32 [1]");
    if (!(grow >= 0 && grow <= INT32_MAX && window >= INT32_MIN && window <= INT32_MAX && sinks >= 0 && sinks <= INT32_MAX))
        return fail(err, errlen, "grow and sinks must be at least 0 and, like window, fit in 32 bits");
    if (!table_rows_apart(new_block_table)) return fail(err, errlen, "new_block_table rows must not overlap");
    const bool keeps = parents == nullptr;  // a row's entry then depends on nothing but itself
    if (!(same_or_apart(new_refs, refs, pages, pages, true) && same_or_apart(new_block_table, block_table, N, B, keeps) &&
          same_or_apart(new_seq_lens, seq_lens, N, B, keeps)))
        return fail(err, errlen, keeps ? "the new tensors must be the old ones or not overlap them"
                                       : "new_refs must be refs or not overlap it; with parents the other new tensors must not overlap the old ones");
    if (const char* why = page_work(workspace, pages, page_work_ints(pages, B, N), p.w)) return fail(err, errlen, why);
    {
        const ByteRows outs[] = {byte_span(new_refs, pages, 4), byte_span(new_block_table, N, 4), byte_span(new_seq_lens, N, 4),
                                 byte_span(needed, 1, 4), byte_span(workspace, workspace->sizes[0], 4)};
        const ByteRows ins[] = {byte_span(refs, pages, 4), byte_span(block_table, B, 4), byte_span(seq_lens, B, 4)};
        for (int i = 0; i < 5; ++i) {
            for (int j = 0; j < 5; ++j)
                if (i != j && !apart(outs[i], outs[j])) return fail(err, errlen, "the tensors that are written must not overlap");
            for (int j = 0; j < 3; ++j)
                if (i != j && !apart(outs[i], ins[j])) return fail(err, errlen, "the tensors that are written must not overlap those that are read");
            if (parents && !apart(outs[i], byte_span(parents, N, 4)))
                return fail(err, errlen, "the tensors that are written must not overlap those that are read");
        }
        const int64_t extent = RowLattice(caches).reach[0];
        bool clear = !parents || clear_of_caches(k, extent, byte_span(parents, N, 4));
        for (const ByteRows& r : outs) clear = clear && clear_of_caches(k, extent, r);
        for (const ByteRows& r : ins) clear = clear && clear_of_caches(k, extent, r);
        if (!clear) return fail(err, errlen, "the caches must not overlap the other tensors");
    }
    p.refs = static_cast<const int*>(refs->data);
    p.new_refs = static_cast<int*>(const_cast<void*>(new_refs->data));
    p.table = static_cast<const int*>(block_table->data);
    p.t_st = block_table->strides[0];
    p.new_table = static_cast<int*>(const_cast<void*>(new_block_table->data));
    p.n_st = new_block_table->strides[0];
    p.seq_lens = static_cast<const int*>(seq_lens->data);
    p.new_lens = static_cast<int*>(const_cast<void*>(new_seq_lens->data));
    // (no new rows: an empty tensor has no data, but that all old rows end is said by its not being null)
    p.parents = parents ? static_cast<const int*>(N > 0 ? parents->data : refs->data) : nullptr;
    p.needed = static_cast<int*>(const_cast<void*>(needed->data));
    p.rows = (int)B;
    p.new_rows = (int)N;
    p.cols = (int)block_table->sizes[1];
    p.block_size = k.block_size;
    p.grow = grow;
    p.window = window;
    p.sinks = sinks;
    p.eldest = p.w.counts + p.w.chunks;
    p.first_taken = p.eldest + B;
    p.copies = p.first_taken + N;
    p.copy_list = reinterpret_cast<PageCopy*>(p.copies + 1);
    return op_result(launch_fork(p, k, stream), "fork pages", err, errlen);
}

int pth_cache_compact_pages(const pd_tensor* caches, int64_t layers, const pd_tensor* refs, const pd_tensor* block_table,
                            const pd_tensor* new_refs, const pd_tensor* new_block_table, const pd_tensor* places,
                            const pd_tensor* used, const pd_tensor* workspace, hipStream_t stream, char* err, int errlen) {
    if (!caches || !refs || !block_table || !new_refs || !new_block_table || !places || !used || !workspace)
        return fail(err, errlen, "null tensor descriptor");
    CompactParams p = {};
    PageCaches k = {};
    if (const char* why = page_caches(caches, layers, k)) return fail(err, errlen, why);
    const int64_t pages = caches[0].sizes[0];
    if (!(int_rows(refs, pages) && refs->sizes[0] == pages && int_rows(new_refs, pages) && new_refs->sizes[0] == pages &&
          int_rows(places, pages) && places->sizes[0] == pages))
        return fail(err, errlen, "refs, new_refs and places must be contiguous int32 with an entry for each page");
    const int64_t B = block_table->sizes[0];
    if (!(page_table_rows(block_table, 1 << 20) && page_table_rows(new_block_table, 1 << 20) && new_block_table->sizes[0] == B &&
          new_block_table->sizes[1] == block_table->sizes[1]))
        return fail(err, errlen, "block tables must be int32 of at most 2^20 rows, with the same rows and columns");
    if (!int_rows(used, 1)) return fail(err, errlen, "used must be int32 [1]");
    if (!table_rows_apart(new_block_table)) return fail(err, errlen, "new_block_table rows must not overlap");
    if (!(same_or_apart(new_refs, refs, pages, pages, true) && same_or_apart(new_block_table, block_table, B, B, true)))
        return fail(err, errlen, "the new tensors must be the old ones or not overlap them");
    if (const char* why = page_work(workspace, pages, page_work_ints(pages, 0, 0), p.w)) return fail(err, errlen, why);
    {
        const ByteRows outs[] = {byte_span(new_refs, pages, 4), byte_span(new_block_table, B, 4), byte_span(places, pages, 4),
                                 byte_span(used, 1, 4), byte_span(workspace, workspace->sizes[0], 4)};
        const ByteRows ins[] = {byte_span(refs, pages, 4), byte_span(block_table, B, 4)};
        for (int i = 0; i < 5; ++i) {
            for (int j = 0; j < 5; ++j)
                if (i != j && !apart(outs[i], outs[j])) return fail(err, errlen, "the tensors that are written must not overlap");
            for (int j = 0; j < 2; ++j)
                if (i != j && !apart(outs[i], ins[j])) return fail(err, errlen, "the tensors that are written must not overlap those that are read");
        }
        const int64_t extent = RowLattice(caches).reach[0];
        bool clear = true;
        for (const ByteRows& r : outs) clear = clear && clear_of_caches(k, extent, r);
        for (const ByteRows& r : ins) clear = clear && clear_of_caches(k, extent, r);
        if (!clear) return fail(err, errlen, "the caches must not overlap the other tensors");
    }
    p.refs = static_cast<const int*>(refs->data);
    p.new_refs = static_cast<int*>(const_cast<void*>(new_refs->data));
    p.table = static_cast<const int*>(block_table->data);
    p.t_st = block_table->strides[0];
    p.new_table = static_cast<int*>(const_cast<void*>(new_block_table->data));
    p.n_st = new_block_table->strides[0];
    p.places = static_cast<int*>(const_cast<void*>(places->data));
    p.used = static_cast<int*>(const_cast<void*>(used->data));
    p.rows = (int)B;
    p.cols = (int)block_table->sizes[1];
    p.block_size = k.block_size;
    return op_result(launch_compact(p, k, stream), "compact pages", err, errlen);
}

const char* pth_dec_version(void) { return "pth_dec-gfx950 0.2"; }

}  // extern "C"

#pragma GCC visibility pop
