// Host side of the C ABI declared in include/vfa.h: argument checks, window/causal folding,
// kernel-parameter set-up and dispatch.  The counterpart of csrc/flash_attn/flash_api.cpp in the
// reference, minus everything that needs torch (that part lives in torch_binding.cpp).
#include <hip/hip_runtime.h>

#include <atomic>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <string>
#include <vector>

#include "../../include/vfa.h"
#include "vfa_kernel_params.h"
#include "vfa_dispatch.h"
#include "vfa_kv8.h"
#include "vfa_qk_norm.h"

namespace vfa {
hipError_t run_fwd_prefill(const KParams &p, hipStream_t stream);
hipError_t run_fwd_splitkv(const KParams &p, hipStream_t stream);
hipError_t run_append_kv(const KParams &p, hipStream_t stream);
hipError_t run_bwd(const KParams &p, hipStream_t stream, hipEvent_t *stage_events);
hipError_t run_fwd_prefill_dropout(const KParams &p, hipStream_t stream);
hipError_t run_fwd_prefill_split(const KParams &p, hipStream_t stream);
bool fwd_prefill_pack_ok(const KParams &p);                                  // fwd_prefill_pack.hip
hipError_t run_fwd_prefill_pack(const KParams &p, hipStream_t stream);
bool fwd_prefill_split_ok(const KParams &p);
hipError_t run_fwd_combine(const KParams &p, hipStream_t stream);
hipError_t run_bwd_dropout(const KParams &p, hipStream_t stream, hipEvent_t *stage_events);
hipError_t run_kv8_quantize(const KV8Params &a, hipStream_t stream);             // kv8_cache.hip
hipError_t run_kv8_dequantize(const KV8Params &a, hipStream_t stream);
hipError_t run_fwd_kv8(const KV8Params &a, hipStream_t stream);                  // fwd_kv8.hip
int kv8_heads_per_wg(int d, int h_k, bool pairs);
bool kv8_pairs(int d, int h_k, int rows, int64_t k_hs, int64_t v_hs);
int kv8_decode_rows(int d, int rows);
int kv8_decode_wgs_per_cu(int d, int rows, bool pairs);
hipError_t run_kv8_merge(const KParams &p, hipStream_t stream);
hipError_t run_fwd_kv8_prefill(const KV8Params &a, hipStream_t stream);          // fwd_prefill_kv8.hip
hipError_t run_fwd_kv8_prefill_rows(const KV8Params &a, hipStream_t stream);     // fwd_prefill_kv8_rows.hip
bool kv8_read_back_ok(int64_t seqlen_k, int h_k, int d);
hipError_t run_fwd_kv8_wide(const KParams &p, hipStream_t stream);               // fwd_prefill_wide_kv8.hip
hipError_t run_qk_norm_rotary(const QKNormParams &p, bool bwd, hipStream_t stream);   // qk_norm_rotary.hip
void qk_norm_blocks(QKNormParams &p, int cus, bool bwd);
}  // namespace vfa

using vfa::KParams;

#ifdef VFA_DEV
// Development build only (not part of include/vfa.h, absent from libvfa_hip.so): kernel-variant
// switches for A/B timing and for the tests that check a shipped kernel against its alternative.
namespace vfa { int g_tuning[8] = {0, 0, 0, 0, 0, 0, 0, 0}; }
extern "C" __attribute__((visibility("default"))) void vfa_debug_set_tuning(int idx, int value) {
    if (idx >= 0 && idx < 8) vfa::g_tuning[idx] = value;
}
#endif

static thread_local std::string g_err;

#define VFA_CHECK(cond, msg)      \
    do {                          \
        if (!(cond)) {            \
            g_err = (msg);        \
            return VFA_ERR_INVALID; \
        }                         \
    } while (0)

static int hip_fail(hipError_t e, const char *what) {
    g_err = std::string(what) + ": " + hipGetErrorString(e);
    return VFA_ERR_HIP;
}

// The reference gates on sm8x/sm90 (flash_api.cpp:254-258); here the gate is gfx950.
static int check_arch() {
    static thread_local int cached_dev = -1;
    static thread_local int cached_ok = 0;
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return hip_fail(e, "hipGetDevice");
    if (dev != cached_dev) {
        hipDeviceProp_t prop;
        e = hipGetDeviceProperties(&prop, dev);
        if (e != hipSuccess) return hip_fail(e, "hipGetDeviceProperties");
        cached_ok = std::strncmp(prop.gcnArchName, "gfx950", 6) == 0;
        cached_dev = dev;
    }
    if (!cached_ok) {
        g_err = "FlashAttention (MI355X build) only supports gfx950 GPUs.";
        return VFA_ERR_ARCH;
    }
    return VFA_OK;
}

static int num_cus() { return vfa::device_num_cus(); }

// Checks shared by the three forward entry points (flash_api.cpp:262-287 and siblings).
static int common_checks(const vfa_params *p) {
    VFA_CHECK(p != nullptr, "null params");
    VFA_CHECK(p->dtype == VFA_FP16 || p->dtype == VFA_BF16,
              "FlashAttention only support fp16 and bf16 data type");
    VFA_CHECK(p->q && p->k && p->v && p->out && p->softmax_lse, "null tensor pointer");
    VFA_CHECK(p->b > 0, "batch size must be postive");
    VFA_CHECK(p->d > 0 && p->d <= 256,
              "FlashAttention forward only supports head dimension at most 256");
    VFA_CHECK(p->d % 8 == 0, "head dimension must be a multiple of 8 (pad before calling)");
    VFA_CHECK(p->h_k > 0 && p->h % p->h_k == 0,
              "Number of heads in key/value must divide number of heads in query");
    VFA_CHECK(p->p_dropout >= 0.f && p->p_dropout < 1.f, "p_dropout must be in [0, 1)");  // flash_api.cpp:114
    VFA_CHECK(!p->s_dmask || p->p_dropout > 0.f, "return_softmax is only supported when p_dropout > 0.0");
    return VFA_OK;
}

// set_params_fprop (flash_api.cpp:21-138) + the folding rules in front of it (:289-294).
static void fill_common(const vfa_params *p, KParams &k, int seqlen_q_for_fold, int seqlen_k_for_fold) {
    std::memset(&k, 0, sizeof(k));
    k.is_bf16 = p->dtype == VFA_BF16;
    k.q = p->q; k.k = p->k; k.v = p->v; k.o = p->out; k.lse = p->softmax_lse;
    k.q_bs = p->q_batch_stride; k.q_rs = p->q_row_stride; k.q_hs = p->q_head_stride;
    k.k_bs = p->k_batch_stride; k.k_rs = p->k_row_stride; k.k_hs = p->k_head_stride;
    k.v_bs = p->v_batch_stride; k.v_rs = p->v_row_stride; k.v_hs = p->v_head_stride;
    k.o_bs = p->o_batch_stride; k.o_rs = p->o_row_stride; k.o_hs = p->o_head_stride;
    k.b = p->b; k.h = p->h; k.h_k = p->h_k; k.h_ratio = p->h / p->h_k; k.d = p->d;
    k.seqlen_q = p->seqlen_q; k.seqlen_k = p->seqlen_k;
    k.cu_seqlens_q = p->cu_seqlens_q; k.cu_seqlens_k = p->cu_seqlens_k;
    k.seqused_k = p->seqused_k;
    k.k_cumulative = p->cu_seqlens_k ? p->is_seqlens_k_cumulative : 1;
    k.block_table = p->block_table; k.bt_bs = p->block_table_batch_stride;
    k.page_size = p->block_table ? p->page_block_size : 1;
    k.page_shift = -1;
    if (k.page_size > 0 && (k.page_size & (k.page_size - 1)) == 0) {
        k.page_shift = 0;
        while ((1 << k.page_shift) < k.page_size) k.page_shift++;
    }
    k.cache_batch_idx = p->cache_batch_idx;
    k.alibi_slopes = p->alibi_slopes; k.alibi_bs = (int)p->alibi_slopes_batch_stride;
    k.scale = p->softmax_scale;
    k.scale_log2 = p->softmax_scale * (float)M_LOG2E;  // flash_api.cpp:103

    int wl = p->window_size_left, wr = p->window_size_right, causal = p->is_causal;
    if (wl >= seqlen_k_for_fold) wl = -1;              // flash_api.cpp:289-290
    if (wr >= seqlen_k_for_fold) wr = -1;
    if (seqlen_q_for_fold == 1 && !p->alibi_slopes) causal = 0;  // :293
    if (causal) wr = 0;                                // :294
    k.is_causal = (wl < 0 && wr == 0);                 // :121
    if (wl < 0 && wr >= 0) wl = seqlen_k_for_fold;     // :123-124
    if (wl >= 0 && wr < 0) wr = seqlen_k_for_fold;
    k.wl = wl; k.wr = wr;
    k.is_local = (wl >= 0 || wr >= 0) && !k.is_causal;
    k.dbg_flags = vfa::g_tuning[2];
    k.pack_gqa = 0;
    k.num_splits = 1;
    // flash_api.cpp:105-113: keep probability, its 8-bit threshold (rounded down: the test is <=)
    k.p_keep = 1.f - p->p_dropout;
    k.drop_keep_u8 = (int)(uint8_t)std::floor(k.p_keep * 255.0);
    k.rp_dropout = 1.f / k.p_keep;
    k.scale_rp = p->p_dropout > 0.f ? k.rp_dropout * k.scale : k.scale;
    k.philox_seed = p->philox_seed; k.philox_offset = p->philox_offset;
    k.seed_ptr = (const long long *)p->philox_seed_ptr; k.offset_ptr = (const long long *)p->philox_offset_ptr;
    k.offset_intragraph = p->philox_offset_intragraph;
    k.rng_state = (unsigned long long *)p->rng_state;
}

extern "C" int vfa_num_splits_heuristic(int batch_nheads_mblocks, int num_sms, int num_n_blocks,
                                        int max_splits) {
    // flash_api.cpp:158-192
    if (batch_nheads_mblocks >= 0.8f * num_sms) return 1;
    max_splits = std::min(std::min(max_splits, num_sms), num_n_blocks);
    float max_eff = 0.f;
    std::vector<float> eff;
    eff.reserve(max_splits > 0 ? max_splits : 1);
    auto cdiv = [](int a, int b) { return (a + b - 1) / b; };
    auto eligible = [&](int s) { return s == 1 || cdiv(num_n_blocks, s) != cdiv(num_n_blocks, s - 1); };
    for (int s = 1; s <= max_splits; s++) {
        if (!eligible(s)) { eff.push_back(0.f); continue; }
        float n_waves = float(batch_nheads_mblocks * s) / num_sms;
        float e = n_waves / std::ceil(n_waves);
        if (e > max_eff) max_eff = e;
        eff.push_back(e);
    }
    for (int s = 1; s <= max_splits; s++) {
        if (!eligible(s)) continue;
        if (eff[s - 1] >= 0.85f * max_eff) return s;
    }
    return 1;
}

extern "C" int vfa_splitkv_num_splits(int batch, int num_heads, int head_size, int max_seqlen_k,
                                      int max_seqlen_q, int num_cus_) {
    // flash_api.cpp:199-210.  Up to 64 query rows (decode) the block sizes follow the reference,
    // so the split count is the same function of the shapes as the reference's.
    if (max_seqlen_q > 64) {
        // Beyond 64 query rows the split work items are the prefill kernel's 128-row blocks.  Their
        // fp32 partial results cost HBM traffic in proportion to rows x splits, so splitting is
        // kept for launches that would otherwise fill at most a quarter of the resident-workgroup
        // slots, and every split gets at least 16 tiles (1024 keys).  Measured on MI355X (h32/8
        // d128): 512 rows against 8192 keys, batch 1: 195 -> 116 us; 1024 x 1024: 30 -> 77 us (not
        // split under this rule).
        const int blocks = batch * num_heads * ((max_seqlen_q + 127) / 128);
        const int chunks = ((max_seqlen_k + 63) / 64) / 16;
        if (blocks * 4 > num_cus_ * 2 || chunks < 2) return 1;
        return vfa_num_splits_heuristic(blocks, num_cus_ * 2, chunks, 128);
    }
    const int block_n = head_size <= 64 ? 256 : (head_size <= 128 ? 128 : 64);
    const int num_n_blocks = (max_seqlen_k + block_n - 1) / block_n;
    const int num_m_blocks = (max_seqlen_q + 64 - 1) / 64;
    // The decode kernel cuts the keys in 128-key tiles whatever the head dim: a split count beyond
    // the number of tiles (possible above d = 128, where the reference's block is 64 keys) would
    // only add workgroups that write empty partials.
    const int tiles = std::max(1, (max_seqlen_k + 127) / 128);
    return std::min(tiles, vfa_num_splits_heuristic(batch * num_heads * num_m_blocks, num_cus_ * 2, num_n_blocks, 128));
}

// Grouped query heads with a few query positions per sequence -- more rows than one 32-row decode
// block holds, fewer positions than fill a 128-row prefill block per head: the prefill kernel with
// the group packed into the rows of its KV head (fwd_prefill_pack.hip) sweeps the keys once per KV
// head.  Measured (b64 kv4096 h32/8 d128 fp16, query positions 16 / 32 / 64): 260 / 456 / 597 us with
// 32-row decode blocks or one 128-row block per query head, 201 / 208 / 414 us packed.
static bool pack_rows_shape(int ratio, int seqlen_q) {
    if (vfa::g_tuning[2] & 4) return false;   // development switch 2, bit 2: never
    return ratio > 1 && seqlen_q * ratio > 32 && seqlen_q < 128;
}

extern "C" int vfa_decode_num_splits(int batch, int num_heads, int num_heads_k, int head_size, int max_seqlen_k,
                                     int max_seqlen_q, int num_cus_) {
    const int ratio = (num_heads_k > 0 && num_heads % num_heads_k == 0) ? num_heads / num_heads_k : 1;
    if (pack_rows_shape(ratio, max_seqlen_q)) {
        // work items: 128-row blocks of packed rows per (batch, KV head); the rule of the prefill
        // kernel's split variants (vfa_splitkv_num_splits above)
        const int blocks = batch * num_heads_k * ((max_seqlen_q * ratio + 127) / 128);
        const int chunks = ((max_seqlen_k + 63) / 64) / 4;   // at least 4 tiles (256 keys) per split
        if (blocks * 4 > num_cus_ * 2 || chunks < 2) return 1;
        return vfa_num_splits_heuristic(blocks, num_cus_ * 2, chunks, 128);
    }
    if (ratio <= 1 || max_seqlen_q > 64)
        return vfa_splitkv_num_splits(batch, num_heads, head_size, max_seqlen_k, max_seqlen_q, num_cus_);
    // run_fwd_splitkv / launch_decode_hpb: rows = seqlen_q * ratio in 32-row blocks, one (pair of)
    // KV head(s) per workgroup; a two-head workgroup fills a CU like two one-head workgroups, so the
    // count against 2 * CUs is per head either way
    const int m_blocks = (max_seqlen_q * ratio + 31) / 32;
    const int block_n = head_size <= 64 ? 256 : (head_size <= 128 ? 128 : 64);
    const int num_n_blocks = (max_seqlen_k + block_n - 1) / block_n;
    const int tiles = std::max(1, (max_seqlen_k + 127) / 128);
    return std::min(tiles, vfa_num_splits_heuristic(batch * num_heads_k * m_blocks, num_cus_ * 2, num_n_blocks, 128));
}

static int launch_fwd(const vfa_params *p, KParams &k, bool force_split) {
    hipStream_t stream = (hipStream_t)p->stream;
    hipError_t e;
    if (k.knew) {
        e = vfa::run_append_kv(k, stream);
        if (e != hipSuccess) return hip_fail(e, "append_kv launch");
        // the cache now holds the new rows; the attention kernels read it as a longer cache
    }
    if (p->p_dropout > 0.f) {
        // flash_api.cpp:206 (no split with dropout), :296 / :919 (no decode fold, no kv-cache path)
        VFA_CHECK(p->num_splits <= 1 && !force_split && !k.knew,
                  "dropout is not supported with split-KV, paged KV or KV-cache append");
        if (p->s_dmask) {
            VFA_CHECK(p->seqlen_q_rounded % 128 == 0 && p->seqlen_q_rounded >= k.seqlen_q &&
                      p->seqlen_k_rounded % 128 == 0 && p->seqlen_k_rounded >= k.seqlen_k,
                      "s_dmask needs seqlen_q_rounded / seqlen_k_rounded (multiples of 128)");
            k.s_dmask = p->s_dmask;
            k.sq_rounded_p = p->seqlen_q_rounded; k.sk_rounded_p = p->seqlen_k_rounded;
        }
        e = vfa::run_fwd_prefill_dropout(k, stream);
        if (e != hipSuccess) return hip_fail(e, "prefill (dropout) launch");
        return VFA_OK;
    }
    if (p->num_splits > 1) {
        VFA_CHECK(p->num_splits <= 128, "num_splits > 128 not supported");
        VFA_CHECK(p->oaccum && p->softmax_lseaccum, "split-KV needs oaccum / softmax_lseaccum scratch");
        k.num_splits = p->num_splits;
        k.oaccum = p->oaccum;
        k.lseaccum = p->softmax_lseaccum;
        // Few query rows: the decode kernel (waves split the keys of a 32-row block).  More: the
        // prefill kernel's split variants (128-row blocks), when they can load this K/V layout
        // (they do not rotate the query: rotary tables keep the decode kernel).
        const bool q_rotary = k.knew && k.rotary_dim > 0;
        if (pack_rows_shape(k.h_ratio, k.seqlen_q) && !q_rotary && vfa::fwd_prefill_pack_ok(k)) {
            e = vfa::run_fwd_prefill_pack(k, stream);
            if (e == hipSuccess) e = vfa::run_fwd_combine(k, stream);
        } else if (k.seqlen_q > 64 && !q_rotary && vfa::fwd_prefill_split_ok(k)) {
            e = vfa::run_fwd_prefill_split(k, stream);
            if (e == hipSuccess) e = vfa::run_fwd_combine(k, stream);
        } else {
            e = vfa::run_fwd_splitkv(k, stream);
        }
        if (e != hipSuccess) return hip_fail(e, "splitkv launch");
        return VFA_OK;
    }
    // A few query positions of grouped heads: the group packed into the rows of its KV head (the
    // prefill kernel does not rotate the query: rotary tables keep the decode kernel).
    // ... and ragged batches whose sequences are short on average (decode sequences and short chunks
    // batched with a few long ones: a sequence of one query position then costs one workgroup per KV
    // head instead of one per query head) or that attend through a sliding window (a packed block
    // spans a quarter of the positions, so fewer of its tiles lie on the diagonal and on the
    // window's edge).  Measured on MI355X, h32/8 d128, one ragged call (tools/perf_mixed.py and a
    // batch of 8192 ... 127 tokens): 60 x 1 + 4 x 512 positions 722 -> 347 us; 80 x 300 causal 198 ->
    // 181; window 1024 + ALiBi 610 -> 537, without ALiBi 497 -> 478; window 4096 1022 -> 1002; 24 x 1024
    // causal level; long causal sequences 1.6 % behind (they keep one block per query head).
    // (Above d = 128 the unpacked rows have the hand-pipelined kernel, the packed ones the general
    // one: there only batches of mostly one-block sequences are packed.)
    const long long avg_lim = k.d <= 128 ? 512 : 128;
    const bool short_ragged = k.h_ratio > 1 && !(vfa::g_tuning[2] & 4) && p->cu_seqlens_q && k.seqlen_q >= 128 &&
                              ((p->total_q > 0 && (long long)p->total_q < avg_lim * k.b) || (k.is_local && k.d <= 128) ||
                               (vfa::g_tuning[2] & 8));
    if ((pack_rows_shape(k.h_ratio, k.seqlen_q) || short_ragged) && !(k.knew && k.rotary_dim > 0) &&
        vfa::fwd_prefill_pack_ok(k)) {
        e = vfa::run_fwd_prefill_pack(k, stream);
        if (e != hipSuccess) return hip_fail(e, "prefill (packed heads) launch");
        return VFA_OK;
    }
    // Small query blocks against long keys (decode): the split kernel's tiling (few query rows,
    // many waves along the keys) is the right one even with a single split.  The reference sends
    // every call that appends, pages or indexes the cache to its split kernel (flash_api.cpp:919)
    // because only that kernel can; here the prefill kernels read paged and indexed caches too and
    // the new keys are in the cache before the attention kernel starts, so only a query that is
    // still to be rotated (the decode kernel does that on the fly) keeps long query blocks there
    // (measured b64 kv4096 h32/8 d128 paged, 64 query positions: 1049 us in 32-row decode blocks).
    const bool q_rotary = k.knew && k.rotary_dim > 0;
    (void)force_split;
    if (q_rotary || k.seqlen_q <= 32) {
        e = vfa::run_fwd_splitkv(k, stream);
        if (e != hipSuccess) return hip_fail(e, "decode launch");
        return VFA_OK;
    }
    e = vfa::run_fwd_prefill(k, stream);
    if (e != hipSuccess) return hip_fail(e, "prefill launch");
    return VFA_OK;
}

extern "C" int vfa_mha_fwd(const vfa_params *p) {
    g_err.clear();
    int rc = common_checks(p);
    if (rc) return rc;
    if ((rc = check_arch())) return rc;
    VFA_CHECK(!p->cu_seqlens_q && !p->cu_seqlens_k, "vfa_mha_fwd takes dense batches");
    VFA_CHECK(p->seqlen_q > 0, "seqlen_q must be positive");
    KParams k;
    fill_common(p, k, p->seqlen_q, p->seqlen_k);
    return launch_fwd(p, k, false);
}

extern "C" int vfa_mha_varlen_fwd(const vfa_params *p) {
    g_err.clear();
    int rc = common_checks(p);
    if (rc) return rc;
    if ((rc = check_arch())) return rc;
    // cu_seqlens_q may be NULL for a dense query batch (single-token GQA decode folded into rows,
    // flash_api.cpp:500-507)
    VFA_CHECK(p->cu_seqlens_k, "cu_seqlens_k is required");
    VFA_CHECK(!p->block_table || p->page_block_size % 16 == 0,
              "Paged KV cache block size must be divisible by 16");
    KParams k;
    // flash_api.cpp:493-494,515-516: the varlen entry folds with the MAX lengths
    fill_common(p, k, p->seqlen_q, p->seqlen_k);
    k.k_cumulative = 1;
    return launch_fwd(p, k, p->p_dropout > 0.f && p->block_table);
}

extern "C" int vfa_mha_fwd_kvcache(const vfa_params *p) {
    g_err.clear();
    int rc = common_checks(p);
    if (rc) return rc;
    if ((rc = check_arch())) return rc;
    VFA_CHECK(!p->cu_seqlens_q, "fwd_kvcache takes a dense query batch");
    VFA_CHECK(p->p_dropout == 0.f, "fwd_kvcache has no dropout");
    VFA_CHECK(!(p->block_table && p->cache_batch_idx), "Paged KVcache does not support cache_batch_idx");
    VFA_CHECK(!p->block_table || p->page_block_size % 16 == 0,
              "Paged KV cache block size must be divisible by 16");
    KParams k;
    fill_common(p, k, p->seqlen_q, p->seqlen_k);
    k.k_cumulative = p->cu_seqlens_k ? 0 : 1;  // flash_api.cpp:859-867: lengths, not offsets
    if (p->knew) {
        VFA_CHECK(p->vnew, "If key is supplied, value must also be passed in");
        VFA_CHECK(p->cu_seqlens_k, "If key is supplied, seqlens_k must also be passed in");
        VFA_CHECK(p->seqlen_q <= p->seqlen_k,
                  "If key is supplied, it must have seqlen <= the seqlen of the KV cache");
        k.knew = p->knew; k.vnew = p->vnew; k.seqlen_knew = p->seqlen_knew;
        k.knew_bs = p->knew_batch_stride; k.knew_rs = p->knew_row_stride; k.knew_hs = p->knew_head_stride;
        k.vnew_bs = p->vnew_batch_stride; k.vnew_rs = p->vnew_row_stride; k.vnew_hs = p->vnew_head_stride;
    }
    if (p->rotary_cos) {
        VFA_CHECK(p->knew, "If rotary cos/sin are provided, new key / value to be appended to KV cache must also be provided");
        VFA_CHECK(p->rotary_sin, "If rotary cos is provided, rotary sin must also be provided");
        VFA_CHECK(p->rotary_dim <= p->d, "rotary_dim must be <= headdim");
        VFA_CHECK(p->rotary_dim % 16 == 0, "Only rotary dimensions divisible by 16 are currently supported");
        k.rotary_cos = p->rotary_cos; k.rotary_sin = p->rotary_sin;
        k.rotary_dim = p->rotary_dim; k.rotary_interleaved = p->is_rotary_interleaved;
        VFA_CHECK(p->seqlen_ro == 0 || p->seqlen_ro >= p->seqlen_k, "cos/sin seqlen must be at least the seqlen of KV cache");
        k.seqlen_ro = p->seqlen_ro;
    }
    // flash_api.cpp:919: appending, cache_batch_idx and paged caches take the split kernel
    const bool force = p->knew || p->cache_batch_idx || p->block_table;
    return launch_fwd(p, k, force);
}

// ---------------------------------------------------------------------------------------------
// vfa_mha_fwd_kvcache_noalloc: the split-KV partial results live in a file-scope device array
// instead of caller-provided workspace, for callers that cannot allocate (HIP graph capture, tight
// serving loops).  Every GPU the library runs on holds its own copy of the array at its own
// address until the process ends; in host code the array's NAME is only a handle for
// hipGetSymbolAddress -- the address kernels and copies use is the per-device pointer below.
static __device__ __align__(256) float scratch[VFA_NOALLOC_SCRATCH_BYTES / sizeof(float)];

static constexpr int kMaxDevices = 64;
static std::atomic<float *> g_scratch_ptr[kMaxDevices];

// Device address of `scratch` on the current device, resolved once per device (with that device
// current, as it is for the caller's launch).
static int scratch_on_current_device(float **out) {
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return hip_fail(e, "hipGetDevice");
    if (dev < 0 || dev >= kMaxDevices) {
        g_err = "vfa_mha_fwd_kvcache_noalloc: device index beyond the per-device scratch table";
        return VFA_ERR_UNSUPPORTED;
    }
    float *ptr = g_scratch_ptr[dev].load(std::memory_order_acquire);
    if (!ptr) {
        e = hipGetSymbolAddress((void **)&ptr, HIP_SYMBOL(scratch));
        if (e != hipSuccess) return hip_fail(e, "hipGetSymbolAddress(scratch)");
        if (!ptr) {
            g_err = "hipGetSymbolAddress(scratch) returned a null address";
            return VFA_ERR_HIP;
        }
        g_scratch_ptr[dev].store(ptr, std::memory_order_release);
    }
    *out = ptr;
    return VFA_OK;
}

static size_t split_scratch_floats(const vfa_params *p, int splits, size_t *lse_floats) {
    const size_t rows = (size_t)p->b * (size_t)p->h * (size_t)p->seqlen_q;
    const size_t lse = ((size_t)splits * rows + 63) / 64 * 64;  // keeps the O partials 256-byte aligned
    if (lse_floats) *lse_floats = lse;
    return lse + (size_t)splits * rows * (size_t)p->d;
}

extern "C" int vfa_mha_fwd_kvcache_noalloc(const vfa_params *p) {
    g_err.clear();
    int rc = common_checks(p);
    if (rc) return rc;
    VFA_CHECK(p->seqlen_q > 0, "seqlen_q must be positive");
    vfa_params q = *p;
    q.oaccum = nullptr;
    q.softmax_lseaccum = nullptr;
    constexpr size_t cap = VFA_NOALLOC_SCRATCH_BYTES / sizeof(float);
    if (q.num_splits == 0) {
        // the count the allocating path's caller would pick (set_params_splitkv), lowered until the
        // partial results fit the static array
        q.num_splits = vfa_decode_num_splits(p->b, p->h, p->h_k, p->d, p->seqlen_k, p->seqlen_q, num_cus());
        while (q.num_splits > 1 && split_scratch_floats(p, q.num_splits, nullptr) > cap) q.num_splits--;
    }
    if (q.num_splits > 1) {
        VFA_CHECK(q.num_splits <= 128, "num_splits > 128 not supported");
        size_t lse_floats = 0;
        const size_t need = split_scratch_floats(p, q.num_splits, &lse_floats);
        if (need > cap) {
            g_err = "vfa_mha_fwd_kvcache_noalloc: num_splits * b * h * seqlen_q * (d + 1) floats = " +
                    std::to_string(need * sizeof(float)) + " bytes exceed the static scratch of " +
                    std::to_string((size_t)VFA_NOALLOC_SCRATCH_BYTES) +
                    " bytes; lower num_splits or call vfa_mha_fwd_kvcache with caller-provided scratch";
            return VFA_ERR_INVALID;
        }
        float *ptr = nullptr;
        if ((rc = scratch_on_current_device(&ptr))) return rc;
        // Every split of every row is written by the kernels before the combine kernel reads it
        // (empty splits store 0 / -inf), so nothing has to start at zero; the previous call's
        // contents are simply overwritten.  Two calls that overlap on one GPU would race here.
        q.softmax_lseaccum = ptr;
        q.oaccum = ptr + lse_floats;
    }
    return vfa_mha_fwd_kvcache(&q);
}

extern "C" size_t vfa_bwd_dq_accum_elems(int b, int seqlen_q, int h, int d, int total_q_or_0) {
    const size_t rows = total_q_or_0 > 0 ? (size_t)total_q_or_0 : (size_t)b * seqlen_q;
    return rows * (size_t)h * (size_t)d;
}

extern "C" int vfa_bwd_head_splits(int batch, int num_heads, int num_heads_k, int max_seqlen_k, int num_cus_) {
    // The dK/dV kernel's work items are (batch, kv head, 256-key block); aim at two per CU.
    if (num_heads_k <= 0 || num_heads % num_heads_k != 0) return 1;
    const int g = num_heads / num_heads_k;
    const long long blocks = (long long)((max_seqlen_k + 255) / 256) * batch * num_heads_k;
    const long long target = 2LL * num_cus_;
    if (g == 1 || blocks <= 0 || blocks >= target) return 1;
    return (int)std::min<long long>(g, (target + blocks - 1) / blocks);
}

static int bwd_common(const vfa_params *p, bool varlen) {
    g_err.clear();
    int rc = common_checks(p);
    if (rc) return rc;
    if ((rc = check_arch())) return rc;
    VFA_CHECK(p->dout && p->dq && p->dk && p->dv, "null gradient pointer");
    VFA_CHECK(p->dsoftmax_sum, "backward needs the dsoftmax_sum buffer");
    VFA_CHECK(varlen == (p->cu_seqlens_q != nullptr), "cu_seqlens mismatch for this entry point");
    KParams k;
    fill_common(p, k, p->seqlen_q, p->seqlen_k);
    k.k_cumulative = 1;
    k.dout = p->dout; k.dq = p->dq; k.dk = p->dk; k.dv = p->dv;
    k.do_bs = p->do_batch_stride; k.do_rs = p->do_row_stride; k.do_hs = p->do_head_stride;
    k.dq_bs = p->dq_batch_stride; k.dq_rs = p->dq_row_stride; k.dq_hs = p->dq_head_stride;
    k.dk_bs = p->dk_batch_stride; k.dk_rs = p->dk_row_stride; k.dk_hs = p->dk_head_stride;
    k.dv_bs = p->dv_batch_stride; k.dv_rs = p->dv_row_stride; k.dv_hs = p->dv_head_stride;
    k.dsoftmax_sum = p->dsoftmax_sum;
    k.dq_accum = p->dq_accum;
    k.deterministic = p->deterministic;
    k.seqlen_q_rounded = (p->seqlen_q + 127) / 128 * 128;
    k.rng_read = p->rng_state != nullptr;
    if (p->bwd_head_splits > 1) {
        VFA_CHECK(p->dk_accum && p->dv_accum && p->bwd_part_rows > 0,
                  "bwd_head_splits > 1 needs dk_accum / dv_accum slabs and bwd_part_rows");
        VFA_CHECK(p->bwd_head_splits <= p->h / p->h_k, "bwd_head_splits exceeds the heads per KV head");
        k.hsplit = p->bwd_head_splits;
        k.dk_part = p->dk_accum; k.dv_part = p->dv_accum;
        k.part_rows = p->bwd_part_rows;
        k.part_stride = p->bwd_part_rows * p->h_k * p->d;
    }
    hipError_t e = p->p_dropout > 0.f
                       ? vfa::run_bwd_dropout(k, (hipStream_t)p->stream, (hipEvent_t *)p->stage_events)
                       : vfa::run_bwd(k, (hipStream_t)p->stream, (hipEvent_t *)p->stage_events);
    if (e != hipSuccess) return hip_fail(e, "backward launch");
    return VFA_OK;
}

extern "C" int vfa_mha_bwd(const vfa_params *p) { return bwd_common(p, false); }
extern "C" int vfa_mha_varlen_bwd(const vfa_params *p) { return bwd_common(p, true); }

extern "C" int vfa_dispatch_geometry(const vfa_params *p, int kernel) {
    g_err.clear();
    int rc = common_checks(p);
    if (rc) return rc;
    VFA_CHECK(kernel >= 0 && kernel <= 2, "kernel: 0 = forward, 1 = dK/dV, 2 = dQ");
    KParams k;
    fill_common(p, k, p->seqlen_q, p->seqlen_k);
    k.k_cumulative = 1;
    k.dout = p->dout;
    k.do_rs = p->do_row_stride;
    k.hsplit = p->bwd_head_splits > 1 ? p->bwd_head_splits : 0;
    const int cus = num_cus();
    return kernel == 0 ? vfa::fwd_geometry(k, cus) : kernel == 1 ? vfa::dkdv_geometry(k, cus) : vfa::dq_geometry(k, cus);
}

// ---------------------------------------------------------------------------------------------
// 8-bit KV cache
static bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// The window as it is given: a negative side has no end.  (fill_common ends it at the capacity, and takes a side of the
// capacity or more for endless: with more queries than keys neither is the same.)
static void kv8_window(const vfa_params &a, KParams &k) {
    constexpr int far = 1 << 30;
    // (a single query is the last: nothing is behind it)
    const int wl = a.window_size_left, wr = a.seqlen_q == 1 ? -1 : a.is_causal ? 0 : a.window_size_right;
    k.is_causal = wl < 0 && wr == 0;
    k.is_local = (wl >= 0 || wr >= 0) && !k.is_causal;
    k.wl = wl < 0 ? far : std::min(wl, far);
    k.wr = wr < 0 ? far : std::min(wr, far);
}

static int kv8_fill(const vfa_kv8_params *p, vfa::KV8Params &k) {
    VFA_CHECK(p != nullptr, "null params");
    const vfa_params &a = p->a;
    VFA_CHECK(a.dtype == VFA_FP16 || a.dtype == VFA_BF16, "FlashAttention only support fp16 and bf16 data type");
    VFA_CHECK(a.k && a.v && p->k_scale && p->v_scale, "null cache or scale pointer");
    VFA_CHECK(a.b > 0, "batch size must be postive");
    VFA_CHECK(a.h_k > 0, "number of heads must be positive");
    VFA_CHECK(a.d > 0 && a.d <= 256 && a.d % 16 == 0, "8-bit KV cache: head dimension must be a multiple of 16, at most 256");
    VFA_CHECK(!(a.block_table && a.cache_batch_idx), "Paged KVcache does not support cache_batch_idx");
    const int rows = a.block_table ? a.page_block_size : a.seqlen_k;
    VFA_CHECK(p->num_pages > 0 && rows > 0 && a.seqlen_k > 0, "8-bit KV cache: empty cache");
    VFA_CHECK(a.seqlen_k <= 1 << 30 && rows <= 1 << 30 && a.seqlen_knew <= 1 << 30, "8-bit KV cache: more than 2^30 tokens of a sequence");
    VFA_CHECK(p->scale_block > 0 && p->scale_block % 16 == 0 && rows % p->scale_block == 0,
              "8-bit KV cache: the tokens per scale must be a multiple of 16 that divides the rows of a page");
    VFA_CHECK(a.block_table || a.cache_batch_idx || a.b <= p->num_pages, "8-bit KV cache: batch size exceeds the cache's");
    VFA_CHECK(aligned16(a.k) && aligned16(a.v) && a.k_batch_stride % 16 == 0 && a.k_row_stride % 16 == 0 && a.k_head_stride % 16 == 0 &&
                  a.v_batch_stride % 16 == 0 && a.v_row_stride % 16 == 0 && a.v_head_stride % 16 == 0,
              "8-bit KV cache: codes must be 16-byte aligned, strides multiples of 16 bytes");
    for (int64_t r : {a.k_row_stride, a.v_row_stride, p->k_scale_row_stride, p->v_scale_row_stride})
        VFA_CHECK(r >= 0 && r < (int64_t)1 << 27, "8-bit KV cache: row strides must be under 128 MiB");
    fill_common(&a, k.p, a.seqlen_q, a.seqlen_k);
    kv8_window(a, k.p);
    k.p.k_cumulative = 0;
    k.ks = (unsigned char *)p->k_scale; k.vs = (unsigned char *)p->v_scale;
    k.ks_bs = p->k_scale_batch_stride; k.ks_rs = p->k_scale_row_stride; k.ks_hs = p->k_scale_head_stride;
    k.vs_bs = p->v_scale_batch_stride; k.vs_rs = p->v_scale_row_stride; k.vs_hs = p->v_scale_head_stride;
    k.blk = p->scale_block;
    k.page_rows = rows;
    k.num_pages = p->num_pages;
    k.cap = a.seqlen_k;
    vfa::kv8_div_magic(rows / 16, k.page_mul, k.page_sh);
    vfa::kv8_div_magic(k.blk / 16, k.blk_mul, k.blk_sh);
    if (a.knew) {
        VFA_CHECK(a.vnew, "If key is supplied, value must also be passed in");
        VFA_CHECK(aligned16(a.knew) && aligned16(a.vnew) && a.knew_batch_stride % 8 == 0 && a.knew_row_stride % 8 == 0 &&
                      a.knew_head_stride % 8 == 0 && a.vnew_batch_stride % 8 == 0 && a.vnew_row_stride % 8 == 0 && a.vnew_head_stride % 8 == 0,
                  "new keys and values must be 16-byte aligned, strides multiples of 8 elements");
        k.p.knew = a.knew; k.p.vnew = a.vnew; k.p.seqlen_knew = a.seqlen_knew;
        k.p.knew_bs = a.knew_batch_stride; k.p.knew_rs = a.knew_row_stride; k.p.knew_hs = a.knew_head_stride;
        k.p.vnew_bs = a.vnew_batch_stride; k.p.vnew_rs = a.vnew_row_stride; k.p.vnew_hs = a.vnew_head_stride;
        VFA_CHECK(a.seqlen_knew >= 0, "negative number of new tokens");
    }
    k.cu_new = p->cu_seqlens_new;
    return VFA_OK;
}

extern "C" int vfa_kv8_quantize(const vfa_kv8_params *p) {
    g_err.clear();
    vfa::KV8Params k;
    std::memset(&k, 0, sizeof(k));
    int rc = kv8_fill(p, k);
    if (rc) return rc;
    VFA_CHECK(p->a.knew, "no new tokens");
    if ((rc = check_arch())) return rc;
    hipError_t e = vfa::run_kv8_quantize(k, (hipStream_t)p->a.stream);
    if (e != hipSuccess) return hip_fail(e, "kv8 quantize launch");
    return VFA_OK;
}

extern "C" int vfa_kv8_dequantize(const vfa_kv8_params *p) {
    g_err.clear();
    vfa::KV8Params k;
    std::memset(&k, 0, sizeof(k));
    int rc = kv8_fill(p, k);
    if (rc) return rc;
    if (p->rows_out == 0) return VFA_OK;
    VFA_CHECK(p->k_out && p->v_out, "null output pointer");
    VFA_CHECK(p->rows_out > 0 && (p->cu_seqlens_out || p->seqlen_out > 0), "8-bit KV cache: no shape for the output");
    VFA_CHECK(aligned16(p->k_out) && aligned16(p->v_out) && p->ko_batch_stride % 8 == 0 && p->ko_row_stride % 8 == 0 &&
                  p->ko_head_stride % 8 == 0 && p->vo_batch_stride % 8 == 0 && p->vo_row_stride % 8 == 0 && p->vo_head_stride % 8 == 0,
              "outputs must be 16-byte aligned, strides multiples of 8 elements");
    if ((rc = check_arch())) return rc;
    k.k_out = p->k_out; k.v_out = p->v_out;
    k.ko_bs = p->ko_batch_stride; k.ko_rs = p->ko_row_stride; k.ko_hs = p->ko_head_stride;
    k.vo_bs = p->vo_batch_stride; k.vo_rs = p->vo_row_stride; k.vo_hs = p->vo_head_stride;
    k.cu_out = p->cu_seqlens_out; k.rows_out = p->rows_out; k.seqlen_out = p->seqlen_out;
    hipError_t e = vfa::run_kv8_dequantize(k, (hipStream_t)p->a.stream);
    if (e != hipSuccess) return hip_fail(e, "kv8 dequantize launch");
    return VFA_OK;
}

// Most (query position, head) rows of a KV head that the decode kernel takes, and the rows from which reading the
// cache back into 16 bits first is ahead of the prefill kernel over the codes, at head dims up to 128 and above: the codes'
// conversion is then done once, not once for every 128 rows (and above 128 the hand-pipelined kernel takes the rows).
// us by the decode / by the prefill kernel: h32/8 d128 b32 kv4096, 36 rows 83 / 93, 64 rows 97 / 96, 96 rows 142 / 106; b2 kv32768,
// 36 rows 48 / 51, 64 rows 53 / 54, 96 rows 66 / 58; h8/2 d256 b16 kv4096, 36 rows 34 / 68, 64 rows 40 / 72; h16/4 d64 b32
// kv4096, 36 rows 38 / 36, 64 rows 45 / 37.
// us over the codes / over the cache read back: h32/8 d128 b8 kv2048, 640 rows 85 / 78, 1024 rows 88 / 89, 1536 rows 131 / 117,
// 4096 rows 254 / 222; b4 kv8192, 384 rows 86 / 101, 1024 rows 178 / 175, 2048 rows 317 / 283; h32/8 d64 b8 kv2048, 1024 rows
// 53 / 57, 2048 rows 90 / 87; h8/4 d256 b8 kv2048, 96 rows 46 / 53, 192 rows 81 / 59, 512 rows 123 / 81.  Under a window, b4
// kv16384 h32/8 d128: 127 keys, 4096 rows 37 / 49; 1023 keys, 1024 rows 46 / 54, 4096 rows 104 / 98; 4095 keys 1024 rows 103 / 104,
// 4096 rows 334 / 288.
constexpr int VFA_KV8_DECODE_ROWS = 64, VFA_KV8_READ_BACK_ROWS = 1024, VFA_KV8_READ_BACK_ROWS_WIDE = 192;

// How a call is carried out: sequences of few (query position, head) rows by the decode kernel, the others by the
// prefill kernel -- over the codes, or over the cache read back into 16 bits first.
struct Kv8Plan {
    bool decode, prefill, read_back, wide;
    int dec_sq, dec_rows;        // most query positions and rows of a sequence of the decode kernel's
    int dec_splits, pre_splits;
    int hpw;                     // decode: KV heads, or pairs of them, of a workgroup
    bool pairs;
    int goal, grid;              // decode: parts of all sequences to aim at per head group and row block, the most there can be
    size_t o, lse, n_split;      // decode: offsets into the workspace
    size_t pre_o, pre_lse;       // prefill
    size_t k16, v16, lens;       // read back
    size_t bytes;
};

static int kv8_plan(const vfa_kv8_params *p, Kv8Plan &w) {
    const vfa_params &a = p->a;
    std::memset(&w, 0, sizeof(w));
    const int ratio = a.h / a.h_k, cus = num_cus();
    const long long rows = (long long)a.seqlen_q * ratio;
    w.prefill = rows > VFA_KV8_DECODE_ROWS;
    // Beside longer ones only sequences of one 16-row block (of one query position, if that is more rows).  us with 16 / 32 /
    // 64 as the limit, seven of eight sequences short: h32/8 d128 b16 kv8192 beside 512 positions, 16 rows each 308 / 312 / 339,
    // 20 rows 567 / 311 / 339, 64 rows 577 / 590 / 339; beside 64 positions, 16 rows 341 / 346 / 380, 20 rows 271 / 359 / 393;
    // h8/2 d256 b16 kv4096 beside 128 positions 152 / 154 / 165 and 156 / 154 / 166.
    w.dec_rows = !w.prefill ? VFA_KV8_DECODE_ROWS : ratio <= 16 ? 16 : ratio <= 32 ? 32 : VFA_KV8_DECODE_ROWS;
    // a dense batch is all one kind; of a ragged one with long members only the lengths on the device know
    w.decode = !w.prefill || (a.cu_seqlens_q && ratio <= w.dec_rows);
    w.dec_sq = w.prefill ? std::max(1, w.dec_rows / ratio) : a.seqlen_q;
    if (!w.decode) w.dec_rows = 0;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t o = at; at += (bytes + 255) / 256 * 256; return o; };
    if (w.decode) {
        w.pairs = vfa::kv8_pairs(a.d, a.h_k, w.dec_sq * ratio, a.k_head_stride, a.v_head_stride);
        const int per = vfa::kv8_decode_rows(a.d, w.dec_sq * ratio), mblocks = (w.dec_sq * ratio + per - 1) / per;
        const long long heads = w.pairs ? a.h_k / 2 : a.h_k, codes = 2LL * a.b * a.seqlen_k * a.h_k * a.d;
        w.hpw = vfa::kv8_heads_per_wg(a.d, a.h_k, w.pairs);
        // A few short sequences wait for the steps of a wave, not for bytes: their heads go apart, where that gives more
        // CUs work (h16/8 d128, 512 keys, b8: 18.3 -> 10.5 us, b24: 19.2 -> 11.8; 2048 keys, b8: 18.2 against 19.6)
        while (w.hpw > 1 && a.b * heads / w.hpw * mblocks < cus && a.seqlen_k <= 1024 && codes <= 64LL << 20) w.hpw /= 2;
        const int parts = 8 / w.hpw;
        const long long items = a.b * heads / w.hpw * mblocks;
        // Parts of all sequences together: one workgroup each fills the device once.  A sequence may take up to four
        // times the average (their lengths can differ), as many as its keys allow.
        const int groups = (int)std::max(1LL, items / a.b);
        const long long most = std::max(1LL, (long long)a.seqlen_k / (32LL * 3 * parts));
        w.goal = std::max(1, cus * vfa::kv8_decode_wgs_per_cu(a.d, w.dec_sq * ratio, w.pairs) / groups);
        const long long s = a.num_splits > 1 ? a.num_splits + 1LL   // (cuts at its average length: one part more than cuts)
                            : a.num_splits == 1 || w.goal * 4 <= a.b ? 1 : a.b == 1 ? w.goal : 4LL * ((w.goal + a.b - 1) / a.b);
        w.dec_splits = (int)std::max(1LL, std::min({s, most, 128LL}));
        if (a.num_splits > 1) w.goal = (int)std::min<long long>(1 << 24, (long long)a.b * a.num_splits);
        if (a.b * (16LL * (a.seqlen_k / 32 + 5)) > 1 << 30) w.dec_splits = 1;   // (the device adds the steps up in 32 bits)
        w.grid = std::max(w.goal, a.b);
        if (w.dec_splits > 1) {
            const size_t n = (size_t)w.dec_splits * a.b * a.h * w.dec_sq;
            w.o = take(n * a.d * sizeof(float));
            w.lse = take(n * sizeof(float));
            w.n_split = take((size_t)a.b * mblocks * sizeof(int));
        }
    }
    if (w.prefill) {
        const size_t codes = (size_t)a.b * a.seqlen_k * a.h_k * a.d;
        w.read_back = rows >= (a.d <= 128 ? VFA_KV8_READ_BACK_ROWS : VFA_KV8_READ_BACK_ROWS_WIDE) && codes * 4 <= (size_t)2 << 30 &&
                      vfa::kv8_read_back_ok(a.seqlen_k, a.h_k, a.d);
        w.pre_splits = 1;
        if (!a.cu_seqlens_q) {
            // 128-row blocks, two workgroups per CU (over the cache read back above head dim 128: one); split only what
            // would fill less than half of them (a part's fp32 results cost HBM traffic in proportion to its rows), at
            // least four 64-key tiles each
            const long long slots = (w.read_back && a.d > 128 ? 1LL : 2LL) * cus;
            const long long blocks = (long long)a.b * a.h_k * ((rows + 127) / 128);
            const long long chunks = ((long long)a.seqlen_k + 255) / 256;
            long long s = a.num_splits > 0 ? a.num_splits : blocks * 2 > slots ? 1 : slots / blocks;
            w.pre_splits = (int)std::max(1LL, std::min({s, chunks, 128LL}));
        }
        if (w.read_back) {
            w.wide = a.d > 128 && !a.alibi_slopes && w.pre_splits == 1;
            w.k16 = take(codes * 2);
            w.v16 = take(codes * 2);
            w.lens = take((size_t)a.b * sizeof(int));
        }
        if (w.pre_splits > 1) {
            const size_t n = (size_t)w.pre_splits * a.b * a.h * a.seqlen_q;
            w.pre_o = take(n * a.d * sizeof(float));
            w.pre_lse = take(n * sizeof(float));
        }
    }
    w.bytes = at;
    return VFA_OK;
}

static int kv8_fwd_checks(const vfa_kv8_params *p, vfa::KV8Params &k) {
    std::memset(&k, 0, sizeof(k));
    int rc = kv8_fill(p, k);
    if (rc) return rc;
    const vfa_params &a = p->a;
    VFA_CHECK(a.h > 0 && a.h % a.h_k == 0, "Number of heads in key/value must divide number of heads in query");
    VFA_CHECK(a.seqlen_q >= 0 && a.num_splits >= 0, "negative size");
    VFA_CHECK(a.num_splits <= 128, "num_splits > 128 not supported");
    VFA_CHECK((long long)a.seqlen_q * a.h <= 1 << 30, "seqlen_q out of range");
    return VFA_OK;
}

extern "C" size_t vfa_kv8_workspace(const vfa_kv8_params *p) {
    g_err.clear();
    vfa::KV8Params k;
    if (kv8_fwd_checks(p, k)) return 0;
    Kv8Plan w;
    kv8_plan(p, w);
    return w.bytes;
}

extern "C" int vfa_kv8_mha_fwd(const vfa_kv8_params *p) {
    g_err.clear();
    vfa::KV8Params k;
    int rc = kv8_fwd_checks(p, k);
    if (rc) return rc;
    const vfa_params &a = p->a;
    if ((rc = common_checks(&a))) return rc;
    VFA_CHECK(a.p_dropout == 0.f, "fwd_kvcache has no dropout");
    VFA_CHECK(a.softmax_scale > 0.f, "softmax_scale must be positive");
    VFA_CHECK(!(a.knew && (a.cu_seqlens_q || p->cu_seqlens_new)), "8-bit KV cache: new tokens go with a dense query batch");
    VFA_CHECK(aligned16(a.q) && aligned16(a.out) && a.q_batch_stride % 8 == 0 && a.q_row_stride % 8 == 0 && a.q_head_stride % 8 == 0 &&
                  a.o_batch_stride % 8 == 0 && a.o_row_stride % 8 == 0 && a.o_head_stride % 8 == 0,
              "q and out must be 16-byte aligned, strides multiples of 8 elements");
    if ((rc = check_arch())) return rc;
    Kv8Plan w;
    kv8_plan(p, w);
    VFA_CHECK(w.bytes == 0 || (p->workspace && p->workspace_bytes >= w.bytes && ((uintptr_t)p->workspace & 255) == 0),
              "8-bit KV cache: workspace missing, too small (vfa_kv8_workspace) or not 256-byte aligned");
    hipStream_t stream = (hipStream_t)a.stream;
    hipError_t e;
    if (a.knew) {
        e = vfa::run_kv8_quantize(k, stream);
        if (e != hipSuccess) return hip_fail(e, "kv8 quantize launch");
    }
    if (a.seqlen_q == 0) return VFA_OK;
    char *ws = (char *)p->workspace;
    k.min_rows = w.dec_rows;
    if (w.prefill) {
        vfa::KV8Params f = k;
        if (w.pre_splits > 1) {
            f.p.num_splits = w.pre_splits;
            f.p.oaccum = (float *)(ws + w.pre_o);
            f.p.lseaccum = (float *)(ws + w.pre_lse);
        }
        if (w.read_back) {
            f.k_out = ws + w.k16; f.v_out = ws + w.v16;
            f.lens_out = (int *)(ws + w.lens);
            f.ko_hs = f.vo_hs = a.d; f.ko_rs = f.vo_rs = (int64_t)a.h_k * a.d; f.ko_bs = f.vo_bs = f.ko_rs * a.seqlen_k;
            f.rows_out = (int64_t)a.b * a.seqlen_k; f.seqlen_out = a.seqlen_k;
            e = vfa::run_kv8_dequantize(f, stream);
            if (e != hipSuccess) return hip_fail(e, "kv8 dequantize launch");
        }
        if (w.wide) {
            vfa_params q = a;
            q.k = f.k_out; q.v = f.v_out;
            q.k_batch_stride = q.v_batch_stride = f.ko_bs; q.k_row_stride = q.v_row_stride = f.ko_rs; q.k_head_stride = q.v_head_stride = a.d;
            q.cu_seqlens_k = f.lens_out; q.is_seqlens_k_cumulative = 0;
            q.block_table = nullptr; q.cache_batch_idx = nullptr; q.knew = q.vnew = nullptr;
            KParams k16;
            fill_common(&q, k16, q.seqlen_q, q.seqlen_k);
            kv8_window(a, k16);
            k16.k_cumulative = 0;
            e = vfa::run_fwd_kv8_wide(k16, stream);
        } else {
            e = w.read_back ? vfa::run_fwd_kv8_prefill_rows(f, stream) : vfa::run_fwd_kv8_prefill(f, stream);
        }
        if (e == hipSuccess && w.pre_splits > 1) e = vfa::run_kv8_merge(f.p, stream);
        if (e != hipSuccess) return hip_fail(e, "kv8 prefill launch");
    }
    if (w.decode) {   // (after the kernel of head dims above 128, which writes zeros for the sequences that are not its own)
        k.heads_per_wg = w.hpw;
        k.pairs = w.pairs;
        k.max_rows = w.prefill ? w.dec_rows : 0;
        k.acc_sq = w.dec_sq;
        k.p.num_splits = w.dec_splits;
        if (w.dec_splits > 1) {
            k.p.oaccum = (float *)(ws + w.o);
            k.p.lseaccum = (float *)(ws + w.lse);
            k.n_split = (int *)(ws + w.n_split);
            k.split_goal = w.goal;
            k.split_grid = w.grid;
        }
        e = vfa::run_fwd_kv8(k, stream);
        if (e != hipSuccess) return hip_fail(e, "kv8 attention launch");
    }
    return VFA_OK;
}

// ---------------------------------------------------------------------------------------------
// q / k norm + rotation
static int qk_norm_fill(const vfa_qk_norm_rotary_params *p, vfa::QKNormParams &k, bool bwd) {
    VFA_CHECK(p != nullptr, "null params");
    VFA_CHECK(p->dtype == VFA_FP16 || p->dtype == VFA_BF16, "qk_norm_rotary only supports fp16 and bf16 data type");
    VFA_CHECK(p->b >= 0 && p->s >= 0 && p->h > 0 && p->h_k > 0, "negative size, or no heads");
    VFA_CHECK(p->d > 0 && p->d <= 256 && p->d % 8 == 0, "qk_norm_rotary: head dimension must be a multiple of 8, at most 256");
    VFA_CHECK(p->rotary_dim > 0 && p->rotary_dim % 16 == 0, "Only rotary dimensions divisible by 16 are currently supported");
    VFA_CHECK(p->rotary_dim <= p->d, "rotary_dim must be <= headdim");
    VFA_CHECK(p->table_rows > 0 && p->rotary_cos && p->rotary_sin, "rotary tables are required");
    VFA_CHECK(p->positions || p->s <= p->table_rows, "cos/sin seqlen must be at least the seqlen of q");
    VFA_CHECK(p->q_weight && p->k_weight, "null weight pointer");
    const bool tokens = (int64_t)p->b * p->s > 0;
    VFA_CHECK(!tokens || (p->q && p->k), "null tensor pointer");
    std::memset(&k, 0, sizeof(k));
    auto side = [&](int i, const void *x, int64_t bs, int64_t rs, int64_t hs, const void *w, int h, void *y, int64_t ybs, int64_t yrs,
                    int64_t yhs, const void *dy, int64_t dbs, int64_t drs, int64_t dhs, void *dw) {
        vfa::QKNormTensor &t = k.t[i];
        t.x = x; t.x_bs = bs; t.x_rs = rs; t.x_hs = hs; t.w = w; t.h = h;
        t.y = y; t.y_bs = ybs; t.y_rs = yrs; t.y_hs = yhs;
        t.dy = dy; t.dy_bs = dbs; t.dy_rs = drs; t.dy_hs = dhs; t.dw = dw;
        return aligned16(x) && aligned16(y) && aligned16(dy) && bs % 8 == 0 && rs % 8 == 0 && hs % 8 == 0 && ybs % 8 == 0 &&
               yrs % 8 == 0 && yhs % 8 == 0 && dbs % 8 == 0 && drs % 8 == 0 && dhs % 8 == 0;
    };
    const bool ok_q = side(0, p->q, p->q_batch_stride, p->q_row_stride, p->q_head_stride, p->q_weight, p->h, p->q_out, p->qo_batch_stride,
                           p->qo_row_stride, p->qo_head_stride, p->dq_out, p->dqo_batch_stride, p->dqo_row_stride, p->dqo_head_stride,
                           p->dq_weight);
    const bool ok_k = side(1, p->k, p->k_batch_stride, p->k_row_stride, p->k_head_stride, p->k_weight, p->h_k, p->k_out, p->ko_batch_stride,
                           p->ko_row_stride, p->ko_head_stride, p->dk_out, p->dko_batch_stride, p->dko_row_stride, p->dko_head_stride,
                           p->dk_weight);
    VFA_CHECK(ok_q && ok_k, "tensors must be 16-byte aligned, strides multiples of 8 elements");
    VFA_CHECK(aligned16(p->q_weight) && aligned16(p->k_weight) && aligned16(p->rotary_cos) && aligned16(p->rotary_sin),
              "weights and tables must be 16-byte aligned");
    if (!bwd) VFA_CHECK(!tokens || (p->q_out && p->k_out), "null output pointer");
    else VFA_CHECK(!tokens || (p->dq_out && p->dk_out), "null gradient pointer");
    k.b = p->b; k.s = p->s; k.d = p->d;
    k.positions = p->positions; k.pos_bs = p->positions_batch_stride;
    k.cos = p->rotary_cos; k.sin = p->rotary_sin;
    k.table_rows = p->table_rows; k.rd = p->rotary_dim; k.interleaved = p->is_rotary_interleaved;
    k.eps = p->eps;
    k.is_bf16 = p->dtype == VFA_BF16; k.table_f32 = p->table_fp32; k.w_f32 = p->weight_fp32;
    return VFA_OK;
}

extern "C" int vfa_qk_norm_rotary_fwd(const vfa_qk_norm_rotary_params *p) {
    g_err.clear();
    vfa::QKNormParams k;
    int rc = qk_norm_fill(p, k, false);
    if (rc) return rc;
    if ((rc = check_arch())) return rc;
    vfa::qk_norm_blocks(k, num_cus(), false);
    hipError_t e = vfa::run_qk_norm_rotary(k, false, (hipStream_t)p->stream);
    if (e != hipSuccess) return hip_fail(e, "qk_norm_rotary launch");
    return VFA_OK;
}

extern "C" size_t vfa_qk_norm_rotary_bwd_workspace(const vfa_qk_norm_rotary_params *p) {
    if (!p || p->d <= 0 || p->h <= 0 || p->h_k <= 0) return 0;
    vfa::QKNormParams k;
    std::memset(&k, 0, sizeof(k));
    k.t[0].h = p->h; k.t[1].h = p->h_k;
    k.b = p->b; k.s = p->s; k.d = p->d;
    vfa::qk_norm_blocks(k, num_cus(), true);
    return (size_t)(k.blocks_q + k.blocks_k) * (size_t)p->d;
}

extern "C" int vfa_qk_norm_rotary_bwd(const vfa_qk_norm_rotary_params *p) {
    g_err.clear();
    vfa::QKNormParams k;
    int rc = qk_norm_fill(p, k, true);
    if (rc) return rc;
    VFA_CHECK(!(p->dq_weight || p->dk_weight) || p->workspace, "qk_norm_rotary: the weights' gradients need the workspace");
    if ((rc = check_arch())) return rc;
    k.dw_part = p->workspace;
    vfa::qk_norm_blocks(k, num_cus(), true);
    hipError_t e = vfa::run_qk_norm_rotary(k, true, (hipStream_t)p->stream);
    if (e != hipSuccess) return hip_fail(e, "qk_norm_rotary backward launch");
    return VFA_OK;
}

extern "C" size_t vfa_params_sizeof(void) { return sizeof(vfa_params); }
extern "C" size_t vfa_kv8_params_sizeof(void) { return sizeof(vfa_kv8_params); }
extern "C" size_t vfa_qk_norm_rotary_params_sizeof(void) { return sizeof(vfa_qk_norm_rotary_params); }
extern "C" const char *vfa_last_error(void) { return g_err.c_str(); }
extern "C" const char *vfa_version(void) { return "vfa-mi355x 0.1.0 (api of vllm_flash_attn 2.5.8.post3)"; }
