// A KV cache held in 8 bits: e4m3 codes with one power-of-two scale per (block of tokens, KV head), in
// E8M0 bytes (value 2^(byte - 127), 255 = NaN).  Parameter block and device helpers shared by the kernels
// that write such a cache, read it back and attend over it.
//
// Why a power of two.  e4m3 is a floating format: a block's scale only has to bring the block's largest
// magnitude under 448; within the format's normal range a value keeps its 3 mantissa bits whatever the
// scale.  With 2^e every product with the scale is exact, so the value a code stands for is exact in
// bf16 / fp16, the conversion instructions apply it (v_cvt_scalef32_pk_{bf16,f16}_fp8 take the exponent of
// a float), and re-encoding a block whose scale has grown rounds only what falls among the subnormals.
#pragma once
#include "vfa_kernel_params.h"

namespace vfa {

constexpr int KV8_EMIN = -126;   // smallest exponent of a scale (2^126 is still a normal float)

struct KV8Params {
    KParams p;                   // k / v: the codes (strides in bytes); lengths, pages, masks, q, out as elsewhere
    unsigned char *ks, *vs;      // scales
    int64_t ks_bs, ks_rs, ks_hs; // page (batch row), block of tokens, head
    int64_t vs_bs, vs_rs, vs_hs;
    int blk;                     // tokens per scale: a multiple of 16 that divides page_rows
    int page_rows;               // rows of a page; of a contiguous cache: its capacity
    int num_pages;               // pages; batch rows of a contiguous cache
    int cap;                     // most tokens a sequence can have
    int heads_per_wg;            // attention: adjacent KV heads, or pairs of them, per workgroup (1, 2, 4, 8)
    int pairs;                   // decode kernel: KV heads in pairs
    int max_rows;                // decode kernel: sequences with more (query, head) rows than this are another kernel's; 0: none are
    int min_rows;                // prefill kernel, reading back for it: the sequences with at most so many rows are the decode kernel's
    int split_goal;              // decode kernel: parts of the keys to aim at per head group and row block, over all sequences
    int split_grid;              // and the most there can be
    int acc_sq;                  // query positions of a sequence in the partial results
    int *n_split;                // (b, row blocks): parts that a sequence's keys were cut into
    int *lens_out;               // reading back: the lengths, or null
    unsigned page_mul, blk_mul;  // exact division by page_rows / 16 and blk / 16 (kv8_div)
    int page_sh, blk_sh;
    // writing: new tokens are p.knew / p.vnew, dense (b, seqlen_knew) or ragged
    const int *cu_new;
    // reading back
    void *k_out, *v_out;
    int64_t ko_bs, ko_rs, ko_hs, vo_bs, vo_rs, vo_hs;
    const int *cu_out;           // ragged: (b + 1); else (b, seqlen_out)
    int64_t rows_out;            // output rows in all
    int seqlen_out;
};

// Exact division of n < 2^27 by d < 2^27 in one high product: M = ceil(2^(31 + s) / d), s = floor(log2 d), is off by
// less than d 2^-(31 + s) of its value's unit, so n M / 2^(31 + s) is over n / d by less than 2^-3 / d.
inline void kv8_div_magic(int d, unsigned &mul, int &shift) {
    shift = 0;
    while ((2 << shift) <= d) shift++;
    mul = (unsigned)(((1ull << (31 + shift)) + d - 1) / (unsigned)d);
}
__device__ __forceinline__ int kv8_div(int n, unsigned mul, int shift) {
    return (int)(__umulhi((unsigned)n << 1, mul) >> shift);
}

// (the helpers take a KV8Params, or a kernel's shorter argument block with the same names)
// tokens in the cache of sequence bidb before the call
template <class A>
__device__ __forceinline__ int kv8_cached(const A &a, int bidb) {
    const int n = a.p.cu_seqlens_k ? a.p.cu_seqlens_k[bidb] : a.p.seqlen_k;
    return min(max(n, 0), a.cap);
}

// ... and with the call's own (both up to 2^30)
template <class A>
__device__ __forceinline__ int kv8_total(const A &a, int bidb, int n_new) {
    const int n = kv8_cached(a, bidb);
    return n + min(n_new, a.cap - n);
}
// The keys [lo, hi) that a query position sees, aligned at the last query and the last key.  (Positions, lengths and
// windows go up to 2^30: no sum of two of them is formed that could be more.)
struct Kv8Seen {
    int sk, shift, wl, wr;             // shift: sk - sq
    bool left, right;
    __device__ __forceinline__ Kv8Seen(const KParams &p, int sq, int sk_)
        : sk(sk_), shift(sk_ - sq), wl(p.wl), wr(p.wr), left(p.is_local), right(p.is_causal || p.is_local) {}
    __device__ __forceinline__ int lo(int pos) const { return left ? max(0, shift + pos - wl) : 0; }
    __device__ __forceinline__ int hi(int pos) const {
        const int next = shift + pos + 1;
        return right ? next + min(wr, sk - next) : sk;
    }
};

// Page that holds token `tok` of sequence bidb (a contiguous cache: its batch row); -1 if the table names
// none of the pool.  tok < cap.
template <class A>
__device__ __forceinline__ int kv8_page(const A &a, int bidb, int tok) {
    int page;
    if (a.p.block_table) page = a.p.block_table[(int64_t)bidb * a.p.bt_bs + kv8_div(tok >> 4, a.page_mul, a.page_sh)];
    else page = a.p.cache_batch_idx ? a.p.cache_batch_idx[bidb] : bidb;
    return (unsigned)page < (unsigned)a.num_pages ? page : -1;
}
template <class A>
__device__ __forceinline__ int kv8_row_in_page(const A &a, int tok) {
    return a.p.block_table ? tok - kv8_div(tok >> 4, a.page_mul, a.page_sh) * a.page_rows : tok;
}

// Requests every cache line of the kernel's arguments (a KV8Params first) at once.  They lie in host memory: left to
// their first uses, the lines of a large argument block arrive one after the other, a microsecond or two each.
__device__ __forceinline__ void touch_kv8_args() {
    static_assert(sizeof(KV8Params) > 14 * 64 && sizeof(KV8Params) <= 15 * 64, "a load per line");
    int x[15];
    asm volatile("s_load_dword %0, %15, 0x0\n\ts_load_dword %1, %15, 0x40\n\ts_load_dword %2, %15, 0x80\n\t"
                 "s_load_dword %3, %15, 0xc0\n\ts_load_dword %4, %15, 0x100\n\ts_load_dword %5, %15, 0x140\n\t"
                 "s_load_dword %6, %15, 0x180\n\ts_load_dword %7, %15, 0x1c0\n\ts_load_dword %8, %15, 0x200\n\t"
                 "s_load_dword %9, %15, 0x240\n\ts_load_dword %10, %15, 0x280\n\ts_load_dword %11, %15, 0x2c0\n\t"
                 "s_load_dword %12, %15, 0x300\n\ts_load_dword %13, %15, 0x340\n\ts_load_dword %14, %15, 0x380\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&s"(x[0]), "=&s"(x[1]), "=&s"(x[2]), "=&s"(x[3]), "=&s"(x[4]), "=&s"(x[5]), "=&s"(x[6]), "=&s"(x[7]),
                   "=&s"(x[8]), "=&s"(x[9]), "=&s"(x[10]), "=&s"(x[11]), "=&s"(x[12]), "=&s"(x[13]), "=&s"(x[14])
                 : "s"(__builtin_amdgcn_kernarg_segment_ptr()));
}

__device__ __forceinline__ float e8m0_to_f32(unsigned byte) {
    return __uint_as_float(byte == 255u ? 0x7fc00000u : byte << 23);
}

// 8 codes -> 8 values of 16 bits, times 2^e
template <bool BF16>
__device__ __forceinline__ i32x4 kv8_to16(i32x2 c, float scale) {
    i32x4 w;
    if constexpr (BF16) {
        w[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[0], scale, false));
        w[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[0], scale, true));
        w[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[1], scale, false));
        w[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[1], scale, true));
    } else {
        w[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[0], scale, false));
        w[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[0], scale, true));
        w[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[1], scale, false));
        w[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[1], scale, true));
    }
    return w;
}

}  // namespace vfa
