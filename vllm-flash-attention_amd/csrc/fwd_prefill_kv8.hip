// Attention over an 8-bit KV cache (format: vfa_kv8.h) for more query rows than the decode kernel takes: chunks of prompts,
// drafted tokens of many heads.
//
// The query heads of a KV head are packed into the rows of one workgroup (row i = query position i / group, head i % group),
// so that the keys are swept once per KV head.  4 waves own 32 rows each; wave64, MFMA 32x32x16:
//   * S^T = K Q^T: the query row is on the lane and the keys in registers, so the softmax is in-lane arithmetic and one
//     half-wave exchange, and P^T is directly the B operand of O^T += V^T P^T;
//   * tiles of 64 keys, double buffered in LDS as 16-bit rows, one barrier a tile.  The codes go through staging registers,
//     16 of a row per load, one tile ahead, and are converted once per workgroup on their way to LDS; page ids are requested
//     another tile ahead.  The rows of a wave's load lie in one group of 16, so in one page and one block of the scales;
//   * V^T fragments by ds_read_b64_tr_b16 on the row-major tile.
//
// Sums, the running maximum and O are fp32; P is rounded to 16 bits once in front of the second product, whose MFMA takes
// 16-bit operands (with V exact in 16 bits a relative error of half a step per key, averaged by the sum).
//
// CODES = false: over the cache read back into contiguous 16-bit rows (args.k_out / v_out), which go straight into LDS
// (buffer_load ... lds).  For long queries the conversions are then done once, not once for every 128 rows.
//
// MFMA-bound, in the shadow of it the conversions (one per two elements of K and V and 128 rows).  The whole call, h32/8
// d128: over the codes b8 kv2048 640 rows 85 us, b4 kv8192 384 rows 86 us; read back b8 kv2048 4096 rows 222 us, b4 kv4096
// 16384 rows 571 us.
#include "vfa_kv8.h"
#include <algorithm>
#include <type_traits>

namespace vfa {

namespace kv8p {
constexpr int BN = 64, NW = 4, NT = NW * 64, BM = NW * 32;
template <int DP>
struct Cfg {
    static constexpr int CPR = DP / 8;                    // 16-byte chunks of a 16-bit row
    static constexpr int TILE_BYTES = BN * DP * 2;
    static constexpr int O_ROWB = DP * 2 + 16;            // padded row of the O staging
    static constexpr int KV_LDS = 4 * TILE_BYTES;         // K0 K1 V0 V1
    static constexpr int O_LDS = BM * O_ROWB;
    static constexpr int LDS_BYTES = KV_LDS > O_LDS ? KV_LDS : O_LDS;
};
}  // namespace kv8p

// The grid walks (sequence, KV head, row block), with p.h = p.h_k, p.pack_gqa = the group's size and p.h_ratio = the row
// blocks of a (sequence, KV head) that stand next to each other in the launch (n_mblocks: such runs of them).
// SPLIT: blockIdx.y is a part of the keys, whose result goes to the fp32 partials.
// DV <= DP: the products stop at column DV (the tiles keep the layout of DP columns, zero beyond the head dim).
template <int DP, bool BF16, bool SPLIT, bool CODES, int DV = DP>
__global__ void __launch_bounds__(kv8p::NT, DP == 256 ? 1 : 2)
kv8_prefill_kernel(const KV8Params args, const int n_mblocks) {
    using namespace kv8p;
    using Cfg = kv8p::Cfg<DP>;
    const KParams &p = args.p;
    static_assert(DV % 32 == 0 && DV <= DP && 2 * DV > DP, "DV");
    constexpr int CPR = Cfg::CPR, KS = DV / 16, NDB = DV / 32;   // k-steps of QK^T, 32-column blocks of O
    extern __shared__ __attribute__((aligned(16))) char smem[];

    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, hh = lane >> 5;

    int bidb, hk, m_block;
    map_block(p, n_mblocks, 32 * (DP == 256 ? 1 : 2), bidb, hk, m_block);
    m_block = m_block * p.h_ratio + p.h_ratio - 1 - hk % p.h_ratio;
    hk /= p.h_ratio;
    const int ratio = p.pack_gqa;

    const BlockInfo bi(p, bidb);
    const int sq = bi.sq, sk = kv8_total(args, bidb, p.knew ? p.seqlen_knew : 0);
    const int rows = min(sq, p.seqlen_q) * ratio;
    if (rows <= args.min_rows || m_block * BM >= rows) return;   // the decode kernel's, or none

    // ---- key tiles of the block: query positions [pos_lo_b, pos_hi_b) ----
    const int pos_lo_b = m_block * BM / ratio, pos_hi_b = min(sq, ((m_block + 1) * BM - 1) / ratio + 1);
    const Kv8Seen seen(p, sq, sk);
    const int vis_lo = seen.lo(pos_lo_b), vis_hi = seen.hi(pos_hi_b - 1);   // keys that some row of the block sees
    int n_min = vis_lo / BN, n_max = (vis_hi + BN - 1) / BN;

    const int h_all = p.h * ratio, head0 = hk * ratio;           // query heads of the tensors, the group's first
    const unsigned short *qg = (const unsigned short *)p.q + bi.q_off(p.q_bs, p.q_rs, bidb) + (int64_t)head0 * p.q_hs;
    unsigned short *og = (unsigned short *)p.o + bi.q_off(p.o_bs, p.o_rs, bidb) + (int64_t)head0 * p.o_hs;
    float *lse_g = p.lse + ((int64_t)bidb * h_all + head0) * p.seqlen_q, *oacc_g = nullptr;
    if constexpr (SPLIT) {   // the keys this block sees, in equal parts
        const int split = blockIdx.y, per = (max(n_max - n_min, 0) + p.num_splits - 1) / p.num_splits;
        n_min += split * per;
        n_max = min(n_max, n_min + per);
        const int64_t acc_row0 = (((int64_t)split * p.b + bidb) * h_all + head0) * p.seqlen_q;
        lse_g = p.lseaccum + acc_row0;
        oacc_g = p.oaccum + acc_row0 * p.d;
    }
    const int q0w = m_block * BM + wave * 32;                    // first row of this wave
    auto q_row_off = [&](const int row) __attribute__((always_inline)) -> int64_t {
        return (int64_t)(row / ratio) * p.q_rs + (int64_t)(row % ratio) * p.q_hs;
    };
    auto o_row_off = [&](const int row) __attribute__((always_inline)) -> int64_t {
        return (int64_t)(row / ratio) * p.o_rs + (int64_t)(row % ratio) * p.o_hs;
    };
    auto stat_off = [&](const int row) __attribute__((always_inline)) -> int64_t {   // lse_g[...], oacc_g[... * d]
        return (int64_t)(row % ratio) * p.seqlen_q + row / ratio;
    };
    const int pos_l = (q0w + r) / ratio;                                  // this lane's query position
    // keys that some row of the wave sees, and that all of them see
    const int pos_lo_w = q0w / ratio, pos_hi_w = (q0w + 31) / ratio;
    const int some_lo = seen.lo(pos_lo_w), some_hi = q0w >= rows ? 0 : seen.hi(pos_hi_w);
    const int all_lo = seen.lo(pos_hi_w), all_hi = seen.hi(pos_lo_w);

    if (n_max <= n_min) {
        // no visible key: O = 0, LSE = +inf; in a part: O = 0, LSE = -inf
        for (int c = tid; c < BM * CPR; c += NT) {
            const int row = m_block * BM + c / CPR, ch = c % CPR;
            if (row < rows && ch * 8 < p.d) {
                if constexpr (SPLIT) {
                    *(f32x4 *)(oacc_g + stat_off(row) * p.d + ch * 8) = f32x4{0, 0, 0, 0};
                    *(f32x4 *)(oacc_g + stat_off(row) * p.d + ch * 8 + 4) = f32x4{0, 0, 0, 0};
                } else {
                    *(i32x4 *)(og + o_row_off(row) + ch * 8) = i32x4{0, 0, 0, 0};
                }
            }
        }
        for (int c = tid; c < BM; c += NT)
            if (m_block * BM + c < rows) lse_g[stat_off(m_block * BM + c)] = SPLIT ? -INFINITY : INFINITY;
        return;
    }

    // ---- read back: a wave instruction fills 1 KiB of LDS in lane order, RPI rows, so a lane fetches the chunk that the XOR
    // swizzle places at its slot; the rows of a wave's instructions are RPI * NW apart, which leaves a lane's swizzle as it
    // is, or (8 apart, d256) alternates between two.  Chunks past the head dim and rows past the sequence are out of the
    // buffer's range: zeros. ----
    constexpr int RPI = 64 / CPR, NI = BN / (RPI * NW), NVAR = (RPI * NW) % 16 == 0 ? 1 : 2;
    static_assert((RPI * NW) % 8 == 0, "swizzle of a lane's rows");
    const unsigned k_rs2 = (unsigned)args.ko_rs * 2, v_rs2 = (unsigned)args.vo_rs * 2;
    const auto k16 = __builtin_amdgcn_make_buffer_rsrc((unsigned short *)args.k_out + bidb * args.ko_bs + hk * args.ko_hs, 0,
                                                       CODES ? 0u : (unsigned)(sk - 1) * k_rs2 + p.d * 2, 0x00020000);
    const auto v16 = __builtin_amdgcn_make_buffer_rsrc((unsigned short *)args.v_out + bidb * args.vo_bs + hk * args.vo_hs, 0,
                                                       CODES ? 0u : (unsigned)(sk - 1) * v_rs2 + p.d * 2, 0x00020000);
    unsigned k_voff[NVAR], v_voff[NVAR];
#pragma unroll
    for (int e = 0; e < NVAR; e++) {
        const int row0 = RPI * wave + lane / CPR, ch = (lane % CPR) ^ swz<DP>(row0 + RPI * NW * e);
        k_voff[e] = ch * 8 < p.d ? (unsigned)row0 * k_rs2 + ch * 16 : 0x80000000u;
        v_voff[e] = ch * 8 < p.d ? (unsigned)row0 * v_rs2 + ch * 16 : 0x80000000u;
    }

    // ---- the tile's codes: 16-byte pieces per thread, and the scales of the wave's rows ----
    const int bidb_cache = p.cache_batch_idx ? p.cache_batch_idx[bidb] : bidb;
    const int *bt = p.block_table ? p.block_table + (int64_t)bidb * p.bt_bs : nullptr;
    constexpr int PPR = DP / 16, NP = BN * PPR / NT;              // pieces of a row, of a thread
    static_assert(NP >= 1 && 64 / PPR <= 16 && NT / PPR % 16 == 0, "pieces of a wave lie in one group of 16 rows");
    i32x4 kc8[NP], vc8[NP];
    unsigned ks8[NP], vs8[NP], bad8[NP];
    int pg8[NP];
    const unsigned char *k_base = (const unsigned char *)p.k + (int64_t)hk * p.k_hs, *v_base = (const unsigned char *)p.v + (int64_t)hk * p.v_hs;
    const unsigned char *ks_base = args.ks + (int64_t)hk * args.ks_hs, *vs_base = args.vs + (int64_t)hk * args.vs_hs;
    // (a thread's row in its group of 16 and its columns are the same in every piece; columns past the head dim
    // read column 0: they meet zero columns of Q, or columns of O that are not stored)
    const int col8 = tid % PPR * 16 < p.d ? tid % PPR * 16 : 0;
    const unsigned koff8 = (unsigned)(((tid / PPR) & 15) * (int)p.k_rs + col8), voff8 = (unsigned)(((tid / PPR) & 15) * (int)p.v_rs + col8);
    auto group16 = [&](const int n, const int i) __attribute__((always_inline)) -> int {   // the wave's rows in piece i of tile n
        return min(n * BN + (((wave * 64 + i * NT) / PPR) & ~15), (sk - 1) & ~15);
    };
    auto load_pages = [&](const int n) __attribute__((always_inline)) {
        if constexpr (!CODES) return;
#pragma unroll
        for (int i = 0; i < NP; i++) {
            if (bt) pg8[i] = bt[kv8_div(group16(n, i) >> 4, args.page_mul, args.page_sh)];
            else pg8[i] = bidb_cache;
        }
    };
    auto load_tile = [&](const int n, auto BUFC) __attribute__((always_inline)) {
        if constexpr (!CODES) {
#ifdef __HIP_DEVICE_COMPILE__   // (loads of 16 bytes to LDS are this target's: the host pass does not take them)
            constexpr int BUF = decltype(BUFC)::value;
#pragma unroll
            for (int i = 0; i < NI; i++) {
                typedef __attribute__((address_space(3))) void *lds_ptr;
                const unsigned at = (unsigned)(n * BN + RPI * NW * i);
                char *to = smem + BUF * Cfg::TILE_BYTES + (wave + NW * i) * 1024;
                __builtin_amdgcn_raw_ptr_buffer_load_lds(k16, (lds_ptr)to, 16, k_voff[i % NVAR] + at * k_rs2, 0, 0, 0);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(v16, (lds_ptr)(to + 2 * Cfg::TILE_BYTES), 16, v_voff[i % NVAR] + at * v_rs2, 0, 0, 0);
            }
#endif
            return;
        }
#pragma unroll
        for (int i = 0; i < NP; i++) {
            const int g16 = group16(n, i);
            const int page = __builtin_amdgcn_readfirstlane(pg8[i]);
            const bool bad = (unsigned)page >= (unsigned)args.num_pages;   // outside the pool: NaN, from the scale
            const int row = bt ? g16 - kv8_div(g16 >> 4, args.page_mul, args.page_sh) * args.page_rows : g16;
            const int64_t pg = bad ? 0 : page, blk = kv8_div(row >> 4, args.blk_mul, args.blk_sh);
            bad8[i] = bad ? 255u : 0u;
            ks8[i] = ks_base[pg * args.ks_bs + blk * args.ks_rs];
            vs8[i] = vs_base[pg * args.vs_bs + blk * args.vs_rs];
            kc8[i] = *(const i32x4 *)(k_base + pg * p.k_bs + (int64_t)row * p.k_rs + koff8);
            vc8[i] = *(const i32x4 *)(v_base + pg * p.v_bs + (int64_t)row * p.v_rs + voff8);
        }
    };
    auto store_tile = [&](const int n, auto BUFC) __attribute__((always_inline)) {
        constexpr int BUF = decltype(BUFC)::value;
        if constexpr (!CODES) {
            __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0): this wave's part of the tile is in LDS
            return;
        }
#pragma unroll
        for (int i = 0; i < NP; i++) vs8[i] |= bad8[i];
        if (n * BN < vis_lo || (n + 1) * BN > vis_hi) {   // V of keys that no row sees must not count, whatever stands there
#pragma unroll
            for (int i = 0; i < NP; i++) {
                const int key = n * BN + (tid + i * NT) / PPR;
                if (key < vis_lo || key >= vis_hi) { vc8[i] = i32x4{0, 0, 0, 0}; vs8[i] = 127u; }   // (the scale may be a NaN)
            }
        }
#pragma unroll
        for (int i = 0; i < NP; i++) {
            const int tr = (tid + i * NT) / PPR, ch = (tid + i * NT) % PPR * 2;
            const float ks = e8m0_to_f32(ks8[i] | bad8[i]), vs = e8m0_to_f32(vs8[i]);
            char *kd = smem + BUF * Cfg::TILE_BYTES, *vd = smem + (2 + BUF) * Cfg::TILE_BYTES;
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int off = lds_off<DP>(tr, ch + e);
                *(i32x4 *)(kd + off) = kv8_to16<BF16>(i32x2{kc8[i][2 * e], kc8[i][2 * e + 1]}, ks);
                *(i32x4 *)(vd + off) = kv8_to16<BF16>(i32x2{vc8[i][2 * e], vc8[i][2 * e + 1]}, vs);
            }
        }
    };

    // ---- Q fragments (B operand of S^T = K Q^T): lane (r, hh) holds row q0w + r, columns 16 s + 8 hh .. ----
    i32x4 qf[KS];
    {
        const bool rok = q0w + r < rows;
        const unsigned short *qr = qg + (rok ? q_row_off(q0w + r) : 0);
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const int col = 16 * s + 8 * hh;
            qf[s] = (rok && col < p.d) ? *(const i32x4 *)(qr + col) : i32x4{0, 0, 0, 0};
        }
    }
    f32x16 o[NDB];
#pragma unroll
    for (int i = 0; i < NDB; i++)
#pragma unroll
        for (int j = 0; j < 16; j++) o[i][j] = 0.f;
    float m_run = -INFINITY;  // reference point of the exponentials: the running maximum, followed lazily
    float l_run = 0.f;        // running sum, partial per lane half

    // ALiBi in linear form where every visible key has col <= row + sk - sq: the bias -slope |row + sk - sq - col| is then
    // slope * (col - cref) plus a constant of the row, which cancels in the softmax and returns in the LSE; cref, the block's
    // first diagonal column, keeps magnitudes small.
    float alibi = 0.f;
    const bool has_alibi = p.alibi_slopes != nullptr;
    if (has_alibi) alibi = p.alibi_slopes[(int64_t)bidb * p.alibi_bs + head0 + (q0w + r) % ratio] / p.scale;
    const bool alibi_lin = has_alibi && (p.is_causal || (p.is_local && p.wr <= 0));
    const int cref = seen.shift + pos_lo_b;
    const float c2 = p.scale_log2;

    // per-lane LDS read offsets; buffer, k-step and key block are compile-time constants on top
    const int tr_q = (lane & 15) >> 2, tr_p = lane & 3, tr_g = (lane >> 4) & 1;
    int k_rd[KS];        // K row read of k-step ks: row r (+32 per key block), chunk 2 ks + hh
    int v_rd[NDB][2];    // V transposed read of block db: rows 4 hh + tr_q (+8), +16 per k-step
#pragma unroll
    for (int ks = 0; ks < KS; ks++) k_rd[ks] = lds_off<DP>(r, 2 * ks + hh);
#pragma unroll
    for (int db = 0; db < NDB; db++)
#pragma unroll
        for (int e = 0; e < 2; e++)
            v_rd[db][e] = lds_off<DP>(4 * hh + tr_q + 8 * e, 4 * db + 2 * tr_g + (tr_p >> 1)) + 8 * (tr_p & 1);
    constexpr int ROWB = DP * 2;

    load_pages(n_max - 1);
    load_tile(n_max - 1, std::integral_constant<int, 0>{});
    if (n_max - 2 >= n_min) load_pages(n_max - 2);
    store_tile(n_max - 1, std::integral_constant<int, 0>{});
    __syncthreads();

    // one tile of keys; BUF (compile time) is the LDS buffer it sits in
    auto tile_step = [&](const int n, auto BUFC) {
        constexpr int BUF = decltype(BUFC)::value;
        const bool has_next = n > n_min;
        if (has_next) {
            load_tile(n - 1, std::integral_constant<int, BUF ^ 1>{});
            if (n - 2 >= n_min) load_pages(n - 2);
        }
        const char *kb = smem + BUF * Cfg::TILE_BYTES;
        const char *vb = smem + (2 + BUF) * Cfg::TILE_BYTES;
        const int c0 = n * BN;
        // a wave whose 32 rows see none of this tile's keys only helps with the staging
        if (c0 < some_hi && c0 + BN > some_lo) {
        // ---- S^T = K Q^T: s[kb2][reg] = score(key = c0 + 32 kb2 + (reg & 3) + 8 (reg >> 2) + 4 hh, row q0w + r) ----
        // Vector instructions of a wave run in the shadow of its own MFMAs, so the maximum of the first 32 keys and the
        // exponentials of the first 16, against the current reference point, go with the MFMAs of the second 32 keys.
        // They stand unless the tile needs a mask or moves the reference point (both rare), which redoes them.
        const bool need_mask = c0 + BN > all_hi || c0 < all_lo;
        const bool need = need_mask || has_alibi;
        f32x16 s[2];
        i32x4 pf[4];
        float ps[4] = {0.f, 0.f, 0.f, 0.f};  // four short chains of the row sum
        auto exp_step = [&](const int ks, const float mc_) __attribute__((always_inline)) {
            const int b8 = 8 * (ks & 1);   // k-step ks = 16 keys = registers 8 (ks & 1) .. of s[ks >> 1]
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[ks >> 1][b8 + 2 * w], c2, -mc_));
                const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[ks >> 1][b8 + 2 * w + 1], c2, -mc_));
                ps[w] += e0 + e1;
                pf[ks][w] = pack2<BF16>(e0, e1);
            }
        };
        const f32x16 zero = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int ks = 0; ks < KS; ks++) s[0] = mma32<BF16>(*(const i32x4 *)(kb + k_rd[ks]), qf[ks], ks == 0 ? zero : s[0]);
        constexpr bool SPEC = DP >= 128;   // (at 64 columns the MFMAs are too few to hide anything: 2.5 % behind)
        const float mc_old = (m_run == -INFINITY ? 0.f : m_run) * c2;
        float mx = -INFINITY;
        if (!SPEC || need) {
#pragma unroll
            for (int ks = 0; ks < KS; ks++) s[1] = mma32<BF16>(*(const i32x4 *)(kb + k_rd[ks] + 32 * ROWB), qf[ks], ks == 0 ? zero : s[1]);
        } else {
            // MFMA ks, then a slice of the vector work, fenced so that it stays there; K fragments two steps ahead
            i32x4 kf2[3];
            kf2[0] = *(const i32x4 *)(kb + k_rd[0] + 32 * ROWB);
            kf2[1] = *(const i32x4 *)(kb + k_rd[1] + 32 * ROWB);
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                if (ks + 2 < KS) kf2[(ks + 2) % 3] = *(const i32x4 *)(kb + k_rd[ks + 2] + 32 * ROWB);
                s[1] = mma32<BF16>(kf2[ks % 3], qf[ks], ks == 0 ? zero : s[1]);
                if constexpr (!SPEC) continue;
#pragma unroll
                for (int j = ks * 16 / KS; j < (ks + 1) * 16 / KS; j++) mx = fmaxf(mx, s[0][j]);
#pragma unroll
                for (int pr = 0; pr < 8; pr++) {  // pair pr: k-step pr >> 2, dword pr & 3 of its P fragment
                    if (pr * KS / 8 != ks) continue;
                    const int st = pr >> 2, w = pr & 3, b8 = 8 * (st & 1);
                    const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][b8 + 2 * w], c2, -mc_old));
                    const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][b8 + 2 * w + 1], c2, -mc_old));
                    ps[w] += e0 + e1;
                    pf[st][w] = pack2<BF16>(e0, e1);
                    asm volatile("" : "+v"(pf[st][w]), "+v"(ps[w]));   // (or the compiler moves the slice to its first use)
                }
                asm volatile("" : "+v"(mx));
                __builtin_amdgcn_sched_barrier(0);
            }
        }

        // ---- masks and ALiBi, each form behind a branch of its own that the usual tile walks around ----
        if (alibi_lin && !need_mask) {
            const float t = alibi * (float)(c0 + 4 * hh - cref);
#pragma unroll
            for (int kb2 = 0; kb2 < 2; kb2++)
#pragma unroll
                for (int j = 0; j < 16; j++)
                    s[kb2][j] = __builtin_fmaf(alibi, (float)(32 * kb2 + (j & 3) + 8 * (j >> 2)), s[kb2][j] + t);
        }
        if (need_mask && !has_alibi && !p.is_local) {
            const int lim = seen.hi(pos_l) - c0 - 4 * hh;
#pragma unroll
            for (int kb2 = 0; kb2 < 2; kb2++)
#pragma unroll
                for (int j = 0; j < 16; j++)
                    s[kb2][j] = (32 * kb2 + (j & 3) + 8 * (j >> 2) < lim) ? s[kb2][j] : -INFINITY;
        }
        if ((need_mask && (has_alibi || p.is_local)) || (has_alibi && !alibi_lin && !need_mask)) {
            const int lo = seen.lo(pos_l), hi = seen.hi(pos_l);
#pragma unroll
            for (int kb2 = 0; kb2 < 2; kb2++)
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    const int col = c0 + 32 * kb2 + (j & 3) + 8 * (j >> 2) + 4 * hh;
                    float x = s[kb2][j];
                    if (has_alibi)
                        x = alibi_lin ? x + alibi * (float)(col - cref)
                                      : x - alibi * fabsf((float)(seen.shift + pos_l - col));
                    s[kb2][j] = (col >= lo && col < hi) ? x : -INFINITY;
                }
        }
        if (!SPEC || need) {   // (the early maximum was taken on scores without mask or bias)
            mx = s[0][0];
#pragma unroll
            for (int j = 1; j < 16; j++) mx = fmaxf(mx, s[0][j]);
        }

        // ---- online softmax, one row per lane ----
#pragma unroll
        for (int j = 0; j < 16; j++) mx = fmaxf(mx, s[1][j]);
        mx = half_swap_max(mx);
        // The reference point follows the maximum lazily: it moves, for every row of the wave at once, only when some
        // row's maximum outgrew it by more than 2^4.  Any reference point gives the same O and LSE up to rounding.
        const bool upd = __any((mx - m_run) * c2 > 4.f);
        const float m_new = upd ? fmaxf(m_run, mx) : m_run;
        const float m_cur = (m_new == -INFINITY) ? 0.f : m_new;
        if (upd) {
            const float alpha = __builtin_amdgcn_exp2f((m_run - m_cur) * c2);
            l_run *= alpha;
#pragma unroll
            for (int i = 0; i < NDB; i++)
#pragma unroll
                for (int j = 0; j < 16; j++) o[i][j] *= alpha;
        }
        m_run = m_new;
        const float mc = m_cur * c2;
        if constexpr (SPEC) {
            if (need || upd) {  // the early exponentials were taken on unmasked scores or an old reference
#pragma unroll
                for (int w = 0; w < 4; w++) ps[w] = 0.f;
                exp_step(0, mc);
                exp_step(1, mc);
            }
        } else {
            exp_step(0, mc);
        }
        // ---- O^T += V^T P^T; element j of lane half hh in k-step ks is key 16 ks + 8 (j >> 2) + 4 hh + (j & 3) ----
#pragma unroll
        for (int ks = 0; ks < 4; ks++) {
            if constexpr (SPEC) { if (ks < 2) exp_step(ks + 2, mc); }  // next to the MFMAs of k-step ks
            else { if (ks < 3) exp_step(ks + 1, mc); }
#pragma unroll
            for (int db = 0; db < NDB; db++) {
                const i32x2 a0 = __builtin_bit_cast(i32x2, lds_read_tr16(vb + v_rd[db][0] + 16 * ks * ROWB));
                const i32x2 a1 = __builtin_bit_cast(i32x2, lds_read_tr16(vb + v_rd[db][1] + 16 * ks * ROWB));
                o[db] = mma32<BF16>(i32x4{a0[0], a0[1], a1[0], a1[1]}, pf[ks], o[db]);
            }
        }
        l_run += (ps[0] + ps[1]) + (ps[2] + ps[3]);
        }
        if (has_next) store_tile(n - 1, std::integral_constant<int, BUF ^ 1>{});
        __syncthreads();
    };
    for (int n = n_max - 1;;) {
        tile_step(n, std::integral_constant<int, 0>{});
        if (--n < n_min) break;
        tile_step(n, std::integral_constant<int, 1>{});
        if (--n < n_min) break;
    }

    // ---- normalise, LSE, store O through LDS as whole rows ----
    const float l_tot = half_swap_sum(l_run);
    const bool bad = (l_tot == 0.f) || (l_tot != l_tot);
    const float inv = bad ? 1.f : 1.f / l_tot;
    // (a row that sees no key is zero; its O is a sum of zero weights times V, NaN if V is)
    auto result = [&](const float x) __attribute__((always_inline)) -> float { return l_tot == 0.f ? 0.f : x * inv; };
    float lse = bad ? (SPLIT ? -INFINITY : INFINITY) : m_run * p.scale + __logf(l_tot);
    if (alibi_lin && !bad) lse -= alibi * p.scale * (float)(seen.shift + pos_l - cref);   // the row constant left out of the linear form
    if (hh == 0 && q0w + r < rows) lse_g[stat_off(q0w + r)] = lse;

    if constexpr (SPLIT) {
        // straight from the accumulators: lane (r, hh) holds, per block db and group g4, four columns of row q0w + r
        if (q0w + r < rows) {
            float *dst = oacc_g + stat_off(q0w + r) * p.d;
#pragma unroll
            for (int db = 0; db < NDB; db++)
#pragma unroll
                for (int g4 = 0; g4 < 4; g4++) {
                    const int col = 32 * db + 8 * g4 + 4 * hh;
                    if (col < p.d)
                        *(f32x4 *)(dst + col) = f32x4{result(o[db][4 * g4]), result(o[db][4 * g4 + 1]),
                                                      result(o[db][4 * g4 + 2]), result(o[db][4 * g4 + 3])};
                }
        }
        return;
    }
    // (the loop's last barrier fenced all reads of the tiles)
    char *ob = smem + wave * 32 * Cfg::O_ROWB;
#pragma unroll
    for (int db = 0; db < NDB; db++)
#pragma unroll
        for (int g4 = 0; g4 < 4; g4++) {
            i32x2 w;
            w[0] = pack2<BF16>(result(o[db][4 * g4 + 0]), result(o[db][4 * g4 + 1]));
            w[1] = pack2<BF16>(result(o[db][4 * g4 + 2]), result(o[db][4 * g4 + 3]));
            *(i32x2 *)(ob + r * Cfg::O_ROWB + (32 * db + 8 * g4 + 4 * hh) * 2) = w;
        }
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): this wave's own LDS writes
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < (32 * CPR) / 64; i++) {
        const int c = lane + 64 * i;
        const int row = c / CPR, ch = c % CPR;
        const i32x4 w = *(const i32x4 *)(ob + row * Cfg::O_ROWB + ch * 16);
        if (q0w + row < rows && ch * 8 < p.d) *(i32x4 *)(og + o_row_off(q0w + row) + ch * 8) = w;
    }
}

// Of a ragged batch the short sequences' workgroups leave at once.  With the row blocks of different sequences in turn the
// workgroups that stay are a fixed number apart, and the dispatcher, which goes round the chip's parts, gives them to the
// same few; all blocks of a sequence next to each other reach every part.  (h32/8 d128 b16 kv8192, a quarter of the
// sequences up to 1024 queries: in turn 631 us, runs of 2 / 4 / 8 370 / 365 / 363, all 364; prompts b16 up to 4096 795, 795 /
// 607 / 606, 616; h16/16 b16 up to 2048 177, 176 / 181 / 183, 176; d64 b32 up to 2048 232, 233 / 197 / 195, 195.)
static int row_block_run(const KParams &p, int n_mblocks) { return p.cu_seqlens_q ? std::max(1, n_mblocks) : 1; }
template <int DP, bool BF16, bool SPLIT, bool CODES, int DV>
static hipError_t launch_kv8_prefill(KV8Params a, hipStream_t stream) {
    KParams &p = a.p;
    const int all = (p.seqlen_q * p.pack_gqa + kv8p::BM - 1) / kv8p::BM;
    p.h_ratio = row_block_run(p, all);
    const int n_mblocks = (all + p.h_ratio - 1) / p.h_ratio;
    const long long blocks = (long long)n_mblocks * p.h_ratio * p.b * p.h;   // (p.h: KV heads)
    if (blocks <= 0) return hipSuccess;
    if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
    auto kern = kv8_prefill_kernel<DP, BF16, SPLIT, CODES, DV>;
    static std::atomic<uint64_t> lds_set{0};
    if (hipError_t e = set_dyn_lds_once((const void *)kern, kv8p::Cfg<DP>::LDS_BYTES, lds_set); e != hipSuccess) return e;
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks, SPLIT ? (unsigned)p.num_splits : 1u), dim3(kv8p::NT), kv8p::Cfg<DP>::LDS_BYTES, stream, a, n_mblocks);
    return hipGetLastError();
}
template <int DP, bool CODES, int DV = DP>
static hipError_t launch_kv8_prefill_type(const KV8Params &a, hipStream_t stream) {
    if (a.p.num_splits > 1) return a.p.is_bf16 ? launch_kv8_prefill<DP, true, true, CODES, DV>(a, stream) : launch_kv8_prefill<DP, false, true, CODES, DV>(a, stream);
    return a.p.is_bf16 ? launch_kv8_prefill<DP, true, false, CODES, DV>(a, stream) : launch_kv8_prefill<DP, false, false, CODES, DV>(a, stream);
}
static KV8Params packed(KV8Params a) {   // the grid walks the KV heads
    a.p.pack_gqa = a.p.h_ratio;
    a.p.h = a.p.h_k;
    return a;
}
#ifdef VFA_KV8_ROWS_TU
// over what was read back, whose rows a 32-bit offset reaches (kv8_read_back_ok)
hipError_t run_fwd_kv8_prefill_rows(const KV8Params &a, hipStream_t stream) {
    if (a.p.d <= 64) return launch_kv8_prefill_type<64, false>(packed(a), stream);
    if (a.p.d <= 96) return launch_kv8_prefill_type<128, false, 96>(packed(a), stream);
    return a.p.d <= 128 ? launch_kv8_prefill_type<128, false>(packed(a), stream) : launch_kv8_prefill_type<256, false>(packed(a), stream);
}
bool kv8_read_back_ok(int64_t seqlen_k, int h_k, int d) { return (seqlen_k + 256) * h_k * d * 2 < (int64_t)1 << 30; }
#else
hipError_t run_fwd_kv8_prefill(const KV8Params &a, hipStream_t stream) {
    if (a.p.d <= 64) return launch_kv8_prefill_type<64, true>(packed(a), stream);
    return a.p.d <= 128 ? launch_kv8_prefill_type<128, true>(packed(a), stream) : launch_kv8_prefill_type<256, true>(packed(a), stream);
}
#endif

}  // namespace vfa
