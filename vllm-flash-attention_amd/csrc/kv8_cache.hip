// Writing tokens to an 8-bit KV cache and reading it back (see vfa_kv8.h for the format).
//
// Both are copies: 2 bytes in and 1 out per element, or 1 in and 2 out, bound by HBM (by the launch for a
// decode step's few tokens).  Measured, h8 d128: prompts of 16 100 tokens written 20.9 us (99 MB, 4.75 TB/s), 139 000
// tokens read back 176 us (855 MB, 4.85 TB/s), where a 2 GiB copy runs at 4.9 TB/s; one token of 128 sequences written
// 4.9 us, of which an empty launch is 3.6.
#include "vfa_kv8.h"
#include <algorithm>

namespace vfa {

constexpr int Q_NT = 256, Q_NW = Q_NT / 64;
constexpr int Q_KEEP = 8;        // rows a wave keeps in registers between the maximum and the encoding

// exponent of the least power-of-two scale that brings `amax` to at most 448 = 1.75 * 2^8
__device__ __forceinline__ int kv8_exponent(float amax) {
    const unsigned u = __float_as_uint(amax);
    const int x = (int)(u >> 23) - 127;
    return max(KV8_EMIN, x - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0));
}
__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }

// 8 values of 16 bits times `inv` -> 8 codes, rounded to nearest even once (the product is exact).  NaN and
// the infinities become NaN codes (e4m3 has no infinity).  `lim`: 448, or 240 where the next code would
// stand for 2^16 (fp16) or 2^128 (bf16) and could not be read back as a finite value.
template <bool BF16>
__device__ __forceinline__ i32x2 kv8_encode(i32x4 x, float inv, float lim) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const unsigned short h = (unsigned short)((unsigned)x[i >> 1] >> (16 * (i & 1)));
        const float v = to_f32<BF16>(h) * inv;
        const float m = fabsf(v);
        y[i] = (m > lim && m < INFINITY) ? copysignf(lim, v) : v;
    }
    i32x2 c;
#pragma unroll
    for (int w = 0; w < 2; w++) {
        int t = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * w], y[4 * w + 1], 0, false);
        c[w] = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * w + 2], y[4 * w + 3], t, true);
    }
    return c;
}

// 8 codes times `f` (a power of two <= 1): the block's scale has grown
__device__ __forceinline__ i32x2 kv8_recode(i32x2 c, float f) {
    i32x2 o;
#pragma unroll
    for (int w = 0; w < 2; w++) {
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(c[w], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(c[w], true);
        int t = __builtin_amdgcn_cvt_pk_fp8_f32(lo[0] * f, lo[1] * f, 0, false);
        o[w] = __builtin_amdgcn_cvt_pk_fp8_f32(hi[0] * f, hi[1] * f, t, true);
    }
    return o;
}

// largest finite magnitude of 8 values, as a bit pattern (16-bit floats order like their bits)
template <bool BF16>
__device__ __forceinline__ int amax_bits(i32x4 x, int m) {
    constexpr int INF = BF16 ? 0x7f80 : 0x7c00;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int a = x[i] & 0x7fff, b = (x[i] >> 16) & 0x7fff;
        m = max(m, a < INF ? a : 0);
        m = max(m, b < INF ? b : 0);
    }
    return m;
}

// The arguments of the two copies, in order of use: they lie in host memory, and the cache lines of a decode step's
// launch are most of its time (KV8Params whole: 5.3 us, b128 of one token).
struct KV8CacheArgs {                    // names as in KV8Params
    struct Base {
        const int *cu_seqlens_k, *block_table, *cache_batch_idx;
        int64_t bt_bs;
        void *k, *v;
        int64_t k_bs, k_rs, k_hs, v_bs, v_rs, v_hs;
        int seqlen_k, h_k, d, b;
    } p;
    unsigned char *ks, *vs;
    int64_t ks_bs, ks_rs, ks_hs, vs_bs, vs_rs, vs_hs;
    int cap, blk, page_rows, num_pages;
    unsigned page_mul, blk_mul;
    int page_sh, blk_sh;
    explicit KV8CacheArgs(const KV8Params &a)
        : p{a.p.cu_seqlens_k, a.p.block_table, a.p.cache_batch_idx, a.p.bt_bs, (void *)a.p.k, (void *)a.p.v,
            a.p.k_bs, a.p.k_rs, a.p.k_hs, a.p.v_bs, a.p.v_rs, a.p.v_hs, a.p.seqlen_k, a.p.h_k, a.p.d, a.p.b},
          ks(a.ks), vs(a.vs), ks_bs(a.ks_bs), ks_rs(a.ks_rs), ks_hs(a.ks_hs), vs_bs(a.vs_bs), vs_rs(a.vs_rs), vs_hs(a.vs_hs),
          cap(a.cap), blk(a.blk), page_rows(a.page_rows), num_pages(a.num_pages), page_mul(a.page_mul), blk_mul(a.blk_mul),
          page_sh(a.page_sh), blk_sh(a.blk_sh) {}
};
struct KV8New {
    const int *cu;                       // ragged: (b + 1)
    const void *k, *v;
    int64_t k_bs, k_rs, k_hs, v_bs, v_rs, v_hs;
    int seqlen, n_blocks, n_hgroups;
};

// One workgroup per (sequence, touched block of tokens, group of heads, K or V).  LPR lanes hold one head's
// row (8 elements each), so a wave covers 64 / LPR adjacent heads of a token, whose rows are adjacent in
// memory; the four waves take the block's rows in turn.  The block belongs to this workgroup alone, so its
// scale is found (maximum over lanes, then over waves through LDS) and its codes are written without
// atomics, and nothing depends on the order of workgroups.
template <bool BF16, int LPR>
__global__ void __launch_bounds__(Q_NT)
kv8_quantize_kernel(const KV8New x_new, const KV8CacheArgs a) {
    const auto &p = a.p;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    unsigned L = blockIdx.x;
    const bool is_v = L & 1; L >>= 1;
    const int hg = (int)(L % x_new.n_hgroups); L /= x_new.n_hgroups;
    const int j = (int)(L % x_new.n_blocks);
    const int bidb = (int)(L / x_new.n_blocks);

    const int start = kv8_cached(a, bidb);
    int64_t src0;                        // first new token's row
    int n_new;
    if (x_new.cu) { src0 = x_new.cu[bidb]; n_new = x_new.cu[bidb + 1] - x_new.cu[bidb]; }
    else { src0 = 0; n_new = x_new.seqlen; }
    const int end = (int)min((int64_t)start + max(n_new, 0), (int64_t)a.cap);
    const int64_t block0 = kv8_div(start >> 4, a.blk_mul, a.blk_sh) * a.blk + (int64_t)j * a.blk;
    if (block0 >= end || end <= start) return;
    const int lo = (int)block0;
    const int r0 = max(start, lo), r1 = min(end, lo + a.blk);
    const int page = kv8_page(a, bidb, lo);
    if (page < 0) return;                // the table names no page of the pool: nothing is written

    const int head = hg * (64 / LPR) + lane / LPR, ch = lane % LPR;
    const bool ok = ch * 8 < p.d && head < p.h_k;
    const int hsafe = min(head, p.h_k - 1), csafe = ch * 8 < p.d ? ch * 8 : 0;
    const int in_page = kv8_row_in_page(a, lo);
    const int64_t rs = is_v ? p.v_rs : p.k_rs;
    unsigned char *codes = (unsigned char *)(is_v ? p.v : p.k) + (int64_t)page * (is_v ? p.v_bs : p.k_bs) +
                           (int64_t)in_page * rs + (int64_t)hsafe * (is_v ? p.v_hs : p.k_hs) + csafe;   // row lo
    unsigned char *scale = (is_v ? a.vs : a.ks) + (int64_t)page * (is_v ? a.vs_bs : a.ks_bs) +
                           (int64_t)kv8_div(in_page >> 4, a.blk_mul, a.blk_sh) * (is_v ? a.vs_rs : a.ks_rs) +
                           (int64_t)hsafe * (is_v ? a.vs_hs : a.ks_hs);
    const int64_t nrs = is_v ? x_new.v_rs : x_new.k_rs;
    const unsigned short *src = (const unsigned short *)(is_v ? x_new.v : x_new.k) +
                                (x_new.cu ? src0 * nrs : (int64_t)bidb * (is_v ? x_new.v_bs : x_new.k_bs)) -
                                (int64_t)start * nrs + (int64_t)hsafe * (is_v ? x_new.v_hs : x_new.k_hs) + csafe;   // row of token 0

    const bool holds = start > lo;       // the block has tokens already: its scale only grows
    const int e_old = holds ? (int)*scale - 127 : KV8_EMIN;

    i32x4 x[Q_KEEP];
    int m = 0;
#pragma unroll
    for (int i = 0; i < Q_KEEP; i++) {
        const int row = r0 + wave + Q_NW * i;
        x[i] = (ok && row < r1) ? *(const i32x4 *)(src + row * nrs) : i32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int i = 0; i < Q_KEEP; i++) m = amax_bits<BF16>(x[i], m);
    for (int row = r0 + wave + Q_NW * Q_KEEP; row < r1; row += Q_NW)
        m = amax_bits<BF16>(ok ? *(const i32x4 *)(src + row * nrs) : i32x4{0, 0, 0, 0}, m);
#pragma unroll
    for (int off = LPR / 2; off > 0; off >>= 1) m = max(m, __shfl_xor(m, off));
    __shared__ int s_m[Q_NW][64 / LPR];
    if (ch == 0) s_m[wave][lane / LPR] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < Q_NW; w++) m = max(m, s_m[w][lane / LPR]);
    if (!ok) return;

    int e = kv8_exponent(to_f32<BF16>((unsigned short)m));
    if (holds) e = max(e, e_old);
    // past this exponent the largest code would stand for a value the 16-bit type does not have
    constexpr int E_TOP = BF16 ? 120 : 8;
    // (a scale of 2^127 and one that is NaN are never written here, but can stand in a cache made elsewhere)
    const float inv = e < 127 ? exp2_int(-e) : __uint_as_float(0x400000u), lim = e >= E_TOP ? 240.f : 448.f;
    if (holds && e > e_old) {
        const float f = e - e_old > 126 ? 0.f : exp2_int(e_old - e);
        for (int row = wave; row < start - lo; row += Q_NW) {
            i32x2 *c = (i32x2 *)(codes + row * rs);
            *c = kv8_recode(*c, f);
        }
    }
#pragma unroll
    for (int i = 0; i < Q_KEEP; i++) {
        const int row = r0 + wave + Q_NW * i;
        if (row < r1) *(i32x2 *)(codes + (row - lo) * rs) = kv8_encode<BF16>(x[i], inv, lim);
    }
    for (int row = r0 + wave + Q_NW * Q_KEEP; row < r1; row += Q_NW)
        *(i32x2 *)(codes + (row - lo) * rs) = kv8_encode<BF16>(*(const i32x4 *)(src + row * nrs), inv, lim);
    if (wave == 0 && ch == 0) *scale = (unsigned char)(e + 127);
}

hipError_t run_kv8_quantize(const KV8Params &a, hipStream_t stream) {
    const KParams &p = a.p;
    if (p.seqlen_knew <= 0) return hipSuccess;
    const int lpr = p.d <= 64 ? 8 : p.d <= 128 ? 16 : 32;
    const int n_hgroups = (p.h_k + 64 / lpr - 1) / (64 / lpr);
    const int n_blocks = (p.seqlen_knew + a.blk - 2) / a.blk + 1;   // a run of n tokens touches at most so many
    const long long blocks = 2LL * p.b * n_blocks * n_hgroups;
    if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
    const dim3 grid((unsigned)blocks), wg(Q_NT);
    const KV8New x{a.cu_new, p.knew, p.vnew, p.knew_bs, p.knew_rs, p.knew_hs, p.vnew_bs, p.vnew_rs, p.vnew_hs,
                   p.seqlen_knew, n_blocks, n_hgroups};
    const KV8CacheArgs c(a);
#define VFA_Q(LPR)                                                                                          \
    if (p.is_bf16) hipLaunchKernelGGL((kv8_quantize_kernel<true, LPR>), grid, wg, 0, stream, x, c);         \
    else hipLaunchKernelGGL((kv8_quantize_kernel<false, LPR>), grid, wg, 0, stream, x, c)
    if (lpr == 8) { VFA_Q(8); } else if (lpr == 16) { VFA_Q(16); } else { VFA_Q(32); }
#undef VFA_Q
    return hipGetLastError();
}

constexpr int D_NT = 256;
constexpr int D_CU = 1024;       // offsets of a ragged output that are bisected in LDS

struct KV8Out {                          // what is read back goes here
    const int *cu;                       // ragged: (b + 1)
    int64_t rows;                        // in all
    void *k, *v;
    int64_t k_bs, k_rs, k_hs, v_bs, v_rs, v_hs;
    int seqlen, n_new;                   // dense: rows a sequence; tokens that the call has appended
    int tpw, cph;                        // rows a workgroup, 8-element chunks of a head's row
    // for the attention kernels over what is read back: the lengths they are to see, and the window on the left (-1: none)
    int *lens;
    const int *cu_q;
    int seqlen_q, ratio, min_rows, wl;
};
constexpr int D_TILE = 64;               // keys of a tile of those kernels

// A workgroup takes `tpw` output rows (tokens): its first threads find each row's sequence (ragged: by bisection of the
// offsets), page and scale row, then all threads copy 8 codes at a time, so that a wave's store is 1 KiB without gaps
// (16 codes and two stores each: 188 us against 176 for b32, 500..8192 tokens, h8 d128).  Rows behind a sequence's tokens
// are zeros.  What is written is twice what is read, so the streams go through the caches (past them: 240 us).
struct RowOf {
    int64_t k, v, ks, vs, out_k, out_v;   // k < 0: no token here
};

template <bool BF16>
__global__ void __launch_bounds__(D_NT)
kv8_dequantize_kernel(const KV8Out o, const KV8CacheArgs a) {
    __shared__ RowOf s_row[64];
    __shared__ int s_cu[D_CU];
    const auto &p = a.p;
    const int tpw = o.tpw, cph = o.cph;
    const int tid = threadIdx.x;
    const int64_t first = (int64_t)blockIdx.x * tpw;
    // Read back for the attention kernels: sequences that are the decode kernel's have length 0 there, and
    // rows behind a sequence are not read, so not written.  Neither are keys in front of the window of the sequence's
    // first query, but for those in the first tile of a visible one: they are zeros, whatever the cache has there (a
    // released page, a NaN code), because their weight 0 is multiplied with them.
    auto queries = [&](int i) -> int { return o.cu_q ? o.cu_q[i + 1] - o.cu_q[i] : o.seqlen_q; };
    auto length = [&](int i) -> int {
        const int n = kv8_total(a, i, o.n_new);
        if (!o.lens) return n;
        return min(queries(i), o.seqlen_q) * o.ratio <= o.min_rows ? 0 : n;
    };
    if (o.lens && blockIdx.x == 0)
        for (int i = tid; i < p.b; i += D_NT) o.lens[i] = length(i);
    const bool near = o.cu && p.b < D_CU;
    if (near) {
        for (int i = tid; i <= p.b; i += D_NT) s_cu[i] = o.cu[i];
        __syncthreads();
    }
    if (tid < tpw && first + tid < o.rows) {
        const int64_t t = first + tid;
        int seq;
        int64_t tok;
        RowOf r;
        if (o.cu) {
            int lo = 0, hi = p.b;          // last sequence that starts at or before t
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if ((near ? s_cu[mid] : o.cu[mid]) <= t) lo = mid; else hi = mid;
            }
            seq = lo;
            tok = t - (near ? s_cu[seq] : o.cu[seq]);
            if (t >= (near ? s_cu[p.b] : o.cu[p.b])) tok = a.cap;   // behind the last sequence
            r.out_k = t * o.k_rs; r.out_v = t * o.v_rs;
        } else {
            seq = o.rows <= 0x7fffffff ? (int)((unsigned)t / (unsigned)o.seqlen) : (int)(t / o.seqlen);
            tok = t - (int64_t)seq * o.seqlen;
            r.out_k = seq * o.k_bs + tok * o.k_rs; r.out_v = seq * o.v_bs + tok * o.v_rs;
        }
        r.k = o.lens ? -3 : -1; r.v = r.ks = r.vs = 0;
        const int len = tok >= 0 && tok < a.cap ? length(seq) : 0;
        const int first_key = o.lens && o.wl >= 0 ? max(0, (len - queries(seq)) - o.wl) : 0;
        if (tok >= 0 && tok < len && tok < first_key) {
            if (tok >= first_key / D_TILE * D_TILE) r.k = -1;
        } else if (tok >= 0 && tok < len) {
            const int page = kv8_page(a, seq, (int)tok);
            if (page >= 0) {
                const int row = kv8_row_in_page(a, (int)tok), blk = kv8_div(row >> 4, a.blk_mul, a.blk_sh);
                r.k = page * p.k_bs + row * p.k_rs;   r.v = page * p.v_bs + row * p.v_rs;
                r.ks = page * a.ks_bs + blk * a.ks_rs; r.vs = page * a.vs_bs + blk * a.vs_rs;
            } else {
                r.k = -2;                             // a page outside the pool: NaN
            }
        }
        s_row[tid] = r;
    }
    __syncthreads();
    const int per = p.h_k * cph;                      // chunks of a token
    const int rows = (int)min((int64_t)tpw, o.rows - first);
    int t = tid / per, c = tid - t * per;
    const int t_step = D_NT / per, c_step = D_NT - t_step * per;
#pragma unroll 2
    for (; t < rows; t += t_step, c += c_step) {
        if (c >= per) {
            c -= per;
            if (++t >= rows) break;
        }
        const int head = c / cph, col = (c - head * cph) * 8;
        const RowOf &r = s_row[t];
        if (r.k == -3) continue;
        i32x2 k = {0, 0}, v = k;
        float ks = 1.f, vs = 1.f;
        if (r.k >= 0) {
            k = *(const i32x2 *)((const unsigned char *)p.k + r.k + head * p.k_hs + col);
            v = *(const i32x2 *)((const unsigned char *)p.v + r.v + head * p.v_hs + col);
            ks = e8m0_to_f32(a.ks[r.ks + head * a.ks_hs]);
            vs = e8m0_to_f32(a.vs[r.vs + head * a.vs_hs]);
        } else if (r.k == -2) {
            k = i32x2{0x7f7f7f7f, 0x7f7f7f7f};
            v = k;
        }
        *(i32x4 *)((unsigned short *)o.k + r.out_k + head * o.k_hs + col) = kv8_to16<BF16>(k, ks);
        *(i32x4 *)((unsigned short *)o.v + r.out_v + head * o.v_hs + col) = kv8_to16<BF16>(v, vs);
    }
}

hipError_t run_kv8_dequantize(const KV8Params &a, hipStream_t stream) {
    const KParams &p = a.p;
    if (a.rows_out <= 0) return hipSuccess;
    const int cph = p.d / 8, per = p.h_k * cph;
    // rows enough for eight chunks a thread (finding the rows is a chain of loads), down to one where that leaves fewer
    // than 1024 workgroups; at most the 64 whose places fit in LDS
    const long long least = std::max(1, D_NT / per), most = std::max(1, 8 * D_NT / per);
    const int tpw = (int)std::min(64LL, std::max(least, std::min(most, (long long)a.rows_out / 1024)));
    const long long blocks = (a.rows_out + tpw - 1) / tpw;
    if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
    const KV8Out o{a.cu_out, a.rows_out, a.k_out, a.v_out, a.ko_bs, a.ko_rs, a.ko_hs, a.vo_bs, a.vo_rs, a.vo_hs, a.seqlen_out,
                   p.knew ? p.seqlen_knew : 0, tpw, cph, a.lens_out, p.cu_seqlens_q, p.seqlen_q, p.h_ratio, a.min_rows, p.is_local ? p.wl : -1};
    const KV8CacheArgs c(a);
    if (p.is_bf16) hipLaunchKernelGGL(kv8_dequantize_kernel<true>, dim3((unsigned)blocks), dim3(D_NT), 0, stream, o, c);
    else hipLaunchKernelGGL(kv8_dequantize_kernel<false>, dim3((unsigned)blocks), dim3(D_NT), 0, stream, o, c);
    return hipGetLastError();
}

}  // namespace vfa
