// Attention over an 8-bit KV cache (format: vfa_kv8.h): a few query rows per KV head against a long key
// range -- decode, drafted tokens, short chunks.
//
// The keys and values are the exact 16-bit values that the codes stand for (the conversion instruction
// applies the power-of-two scale), so the result is that of the 16-bit cache path on the cache read back,
// up to the order of sums.
//
// Measured (reads alone reach 6.1 to 6.3 TB/s on this card): b128 kv8192 h32/8 d128 fp16 353 us (6.1 TB/s); b48 kv16384 h16
// d64 274 us (5.9 TB/s); b1 kv65536 h32/8 d128 36 us, of which the loop over the keys is 20 (6.5 TB/s) and the rest the
// launch, 4.5 us of dependent loads to the first key (arguments, lengths, page ids) and 5.5 us for the merge.
//
// HBM-bound: 2 d bytes per key and KV head against 4 d rows flops.  A workgroup is 8 waves; each wave owns
// one KV head (of heads_per_wg adjacent ones, whose rows are adjacent in memory) and every parts-th step of
// 32 keys, with a running maximum, sum and output of its own.  Waves share nothing until the end, so the key
// loop has no barrier:
//   * the 16 NR rows of a workgroup are (query position, query head of the group) pairs: the heads that share
//     a KV head read it once;
//   * S^T = K Q^T by 16x16x32 MFMAs with the key on the accumulator's rows and the query row on the lane.  A
//     lane's K operand is 16 consecutive codes of one key: two k-steps, loaded straight from memory to
//     registers (which columns a k-step takes is free as long as Q agrees);
//   * P is rounded to 16 bits in front of the second product, whose MFMA takes 16-bit operands (V is exact in them): at most
//     half a step per key, 2^-8 in bf16 and 2^-11 in fp16 of the weight, which the sum over keys averages out; its sum l
//     is taken in fp32 before that.  Against 64 bits the error is up to 6 % above that of a P kept in fp32.
//   * P^T of 32 keys is, in the registers it is computed in, the B operand of O^T += V^T P^T if V^T takes its
//     keys in the order {4g .. 4g+3, 16+4g .. 16+4g+3} for lane group g: ds_read_b64_tr_b8 reads any 8 rows,
//     so V goes through a wave-private LDS image as codes and comes back transposed, to be converted there.
#include "vfa_kv8.h"
#include <algorithm>

namespace vfa {

constexpr int A_NW = 8, A_NT = A_NW * 64;
constexpr int A_STEP = 32;                   // keys of a step
constexpr long long VFA_KV8_LONG = 512LL << 20;   // bytes of codes of a launch that streams for long
constexpr int A_MIN_STEPS = 3;               // least steps of a wave in a part of the keys

template <int DP, int NR>
struct Kv8Cfg {
    static constexpr int VB = A_STEP * DP;               // V image of a wave
    static constexpr int O_ROWB = DP * 4 + 16;
    static constexpr int O_BYTES = A_NW * 16 * O_ROWB;   // merge area: 16 rows of every wave
    static constexpr int MAIN = A_NW * VB > O_BYTES ? A_NW * VB : O_BYTES;
    static constexpr int ML = A_NW * 16 * NR * 2 * 4;    // maxima and sums
    static constexpr int LDS_BYTES = MAIN + ML;
};

template <bool BF16>
__device__ __forceinline__ f32x4 mma16(i32x4 a, i32x4 b, f32x4 c) {
    if constexpr (BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// combined over the four lanes that hold one row (l, l ^ 16, l ^ 32, l ^ 48)
__device__ __forceinline__ float quad_max(float x) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return half_swap_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float quad_sum(float x) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return half_swap_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}
// Inclusive scan over the wave's lanes (sum or maximum) by lane shifts inside the vector unit; lane 63 ends up with
// the total.
template <bool MAX>
__device__ __forceinline__ int wave_scan(int x) {
    auto join = [](int a, int b) { return MAX ? max(a, b) : a + b; };
    x = join(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));   // row_shr:1
    x = join(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));
    x = join(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));
    x = join(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));
    x = join(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));   // row_bcast:15
    x = join(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));   // row_bcast:31
    return x;
}
// (values of at least 0: what a shift brings in from outside is 0)
__device__ __forceinline__ int wave_total(int x) { return __builtin_amdgcn_readlane(wave_scan<false>(x), 63); }
__device__ __forceinline__ int wave_top(int x) { return __builtin_amdgcn_readlane(wave_scan<true>(x), 63); }

// 16-byte chunk of row `row` of the V image: the 16 rows that 32 lanes of a transposed read touch lie in
// different banks
template <int DP>
__host__ __device__ constexpr int kv8_swz(int row) {
    if constexpr (DP == 64) return ((row >> 2) & 1) | ((row >> 4) & 1) << 1;
    else if constexpr (DP == 128) return ((row >> 1) & 3) | ((row >> 4) & 1) << 2;
    else return (row & 7) | ((row >> 4) & 1) << 3;
}

// Steps of 32 keys of sequence i that the rows from q0 on see, about; -1: it has no such rows, or is not this launch's.
template <int NR>
__device__ __forceinline__ int kv8_steps(const KV8Params &a, int i, int q0) {
    const KParams &p = a.p;
    if (i >= p.b) return -1;
    const int span = p.is_local ? (int)(((int64_t)min(p.wl, a.cap) + min(p.wr, a.cap) + 16 * NR) >> 5) + 2 : 1 << 30;
    static_assert(A_STEP == 32, "");
    const int len = kv8_total(a, i, p.knew ? p.seqlen_knew : 0);
    const int rows = (p.cu_seqlens_q ? p.cu_seqlens_q[i + 1] - p.cu_seqlens_q[i] : p.seqlen_q) * p.h_ratio;
    return rows > q0 && !(a.max_rows > 0 && rows > a.max_rows) ? min((len + A_STEP - 1) / A_STEP, span) : -1;
}

// PAIR: two adjacent heads of at most 64 columns and 8 rows share a wave.  They take the 16 columns of Q^T between
// them and each a half of the 128 columns of K and V, whose rows then are whole 128-byte lines: as head dim 64 alone,
// waves that request half a line each, the kernel reaches 4.6 TB/s.  A column's scores come from its own head's product
// (the other one's is dropped, not added as zeros: a NaN of one head stays out of the other).
//
// Columns from p.d to DP are zero in Q; a lane whose columns lie there reads column 0 of its key instead (a
// finite code times zero, or a NaN that the key has anyway), its O is never stored.
//
// The loop is free of branches on the usual path, loads run NBUF steps ahead of their use, and the page ids
// another step ahead of the loads.
// NT: the codes are loaded past the caches.  For streams that the 256 MiB last-level cache cannot hold anyway
// (b128 kv8192 h32/8 d128: 5.85 -> 6.23 TB/s); shorter ones find part of it there (b1 kv65536: 37 against 50 us).
//
// A launch of too few (sequence, head group, row block) items to fill the chip evenly is cut along the keys, by the
// lengths of all sequences, which only the device knows.
template <int DP, bool BF16, int NR, bool PAGED, bool NT, bool RUNS, bool PAIR>
__global__ void __launch_bounds__(A_NT, (DP == 64 && NR == 1) ? 4 : 2)
fwd_kv8_kernel(const KV8Params args, const int n_mblocks) {
    using Cfg = Kv8Cfg<DP, NR>;
    constexpr int NBUF = DP == 64 || (DP == 128 && NR == 1) ? 2 : 1;   // (more do not leave the registers: d 128, 32 rows 166 -> 163 us)
    touch_kv8_args();
    constexpr int NJ = DP / 64;              // 64-column groups of K: one 16-byte load per lane and key tile
    constexpr int NDB = DP / 16;             // 16-column blocks of O
    constexpr int HD = PAIR ? DP / 2 : DP;   // columns of a head
    constexpr int HR = PAIR ? 8 : 16 * NR;   // its rows in a workgroup
    static_assert(!PAIR || (DP == 128 && NR == 1), "");
    constexpr int CPR = DP / 16;             // 16-byte chunks of a V row
    constexpr int NV = A_STEP * CPR / 64;    // V loads per lane and step
    extern __shared__ __attribute__((aligned(16))) char smem[];

    // row blocks of the same keys on one XCD, whose L2 they share
    int L = blockIdx.x;
    if (n_mblocks > 1) {
        const int group = 8 * n_mblocks;
        if (L < (int)gridDim.x / group * group) {
            const int k = L / 8;
            L = k / n_mblocks * group + L % 8 * n_mblocks + k % n_mblocks;
        }
    }
    const int hpw = args.heads_per_wg, hpw_sh = __builtin_ctz(hpw), parts = A_NW >> hpw_sh;   // (powers of two)
    const int n_hblocks = (PAIR ? args.p.h_k >> 1 : args.p.h_k) >> hpw_sh;
    const int m_block = L % n_mblocks; L /= n_mblocks;
    const int hblock = L % n_hblocks; L /= n_hblocks;
    const int q0 = m_block * 16 * NR;

    // ---- L -> its sequence; or, where keys are cut into parts, what it has of them ----
    // Every wave works this out for itself, a lane a sequence (64 at a time): no barrier.
    // Usually a workgroup has one part, and a sequence's parts are of equal length.  Steps of a part: the total over the
    // goal, less about half a part that every sequence leaves over; if the parts then are more than the goal after all
    // (a second round of workgroups), less a whole one each.
    // RUNS: where that leaves much of the chip idle (65 sequences to 128 workgroups: one each), a workgroup has an equal
    // run of all sequences' steps instead, across their ends: their weights (steps, and what a piece of work costs beside
    // them) stand in a row, cut at every multiple of `run`.  A cut within `edge` of a sequence's end moves there.  All in
    // 1/16 steps.
    constexpr int U = 16;
    const bool cut = args.p.num_splits > 1;
    const int few = A_MIN_STEPS * parts, edge = U * few / 2;
    int bidb0 = L, split0 = 0, nsplit0 = 1;
    bool runs = false;
    int run = 1, chunk = 0, before = 0, at_w = 0, at_s = 0;
    uint64_t hits = 0;                       // sequences of this chunk that the workgroup has a piece of
    auto weight_of = [&](int st) -> int { return st < 0 ? 0 : U * (st + few / 2); };
    // the cuts inside a sequence (weight w, at s in the row) are numbers first .. last; its parts are their workgroups'
    // and the one's before
    auto first_cut = [&](int s) -> int { return (s + edge + run - 1) / run; };
    auto last_cut = [&](int s, int w) -> int { return w < 2 * edge ? first_cut(s) - 1 : (s + w - edge) / run; };
    auto place = [&]() __attribute__((always_inline)) {
        const int upto = wave_scan<false>(at_w);
        at_s = before + upto - at_w;
        before += __builtin_amdgcn_readlane(upto, 63);
        const int lo = first_cut(at_s), hi = last_cut(at_s, at_w), whole = (at_s + at_w / 2) / run;
        hits = __ballot(at_w > 0 && (hi < lo ? L == whole : L >= lo - 1 && L <= hi));
    };
    if (cut) {
        const int lane = threadIdx.x & 63;
        auto parts_of = [](int st, int part_steps) -> int { return st < 0 ? 0 : max(1, (st + part_steps - 1) / part_steps); };
        const int st0 = kv8_steps<NR>(args, lane, q0);
        int sum = max(st0, 0), top = sum, some = st0 >= 0;
        for (int i = lane + 64; i < args.p.b; i += 64) {
            const int st = kv8_steps<NR>(args, i, q0);
            sum += max(st, 0);
            top = max(top, st);
            some += st >= 0;
        }
        sum = wave_total(sum);
        some = wave_total(some);
        top = wave_top(top);
        // (no more parts of one sequence than there is scratch for)
        const int least = max((top + args.p.num_splits - 1) / args.p.num_splits, few);
        int part_steps = max((sum - 1) / max(args.split_goal - some / 2, 1) + 1, least);
        if (some > 1) {
            int n = parts_of(st0, part_steps);
            for (int i = lane + 64; i < args.p.b; i += 64) n += parts_of(kv8_steps<NR>(args, i, q0), part_steps);
            if (wave_total(n) > args.split_goal)
                part_steps = args.split_goal > some ? max((sum - 1) / (args.split_goal - some) + 1, least) : max(top, 1);
        }
        if constexpr (RUNS) {
            const int sum_w = U * (sum + some * (few / 2));
            run = max((int)((float)sum_w / (float)args.split_goal) + (sum_w >> 20) + 1, U * few);   // (no less than exact)
            if (args.p.num_splits < args.split_goal) run = max(run, (weight_of(top) - 2 * edge) / (args.p.num_splits - 1) + 1);
            // (a second piece of work costs about as much as `few` steps; more sequences than workgroups: rounds of them)
            const int rounds = some <= args.split_goal ? 1 : (some + args.split_goal - 1) / args.split_goal;
            runs = U * (rounds * min(part_steps, top) - few) > run;
            if (runs) {
                if ((int64_t)L * run >= sum_w) return;   // fewer runs than workgroups
                at_w = weight_of(st0);
                place();
            }
        }
        if (!runs) {
            // the sequence in whose row of parts L falls
            int first = 0;
            bidb0 = -1;
            for (int i = lane; i - lane < args.p.b && bidb0 < 0; i += 64) {
                const int mine = parts_of(i == lane ? st0 : kv8_steps<NR>(args, i, q0), part_steps);
                const int upto = wave_scan<false>(mine);
                const uint64_t hit = __ballot(first + upto > L);
                if (hit) {
                    const int at = __builtin_ctzll(hit);
                    bidb0 = i - lane + at;
                    nsplit0 = __builtin_amdgcn_readlane(mine, at);
                    split0 = L - first - (__builtin_amdgcn_readlane(upto, at) - nsplit0);
                }
                first += __builtin_amdgcn_readlane(upto, 63);
            }
            if (bidb0 < 0) return;                        // fewer parts than workgroups
        }
    }

  for (;;) {
    int tid = threadIdx.x;
    const KV8Params *args_at = &args;
    if constexpr (RUNS) {
        // (nothing but the plan stays in registers from one piece to the next: the arguments and the lane's place are
        // new to the compiler here, or it would keep all that depends on them, and spill)
        const auto *at = (const __attribute__((address_space(4))) KV8Params *)__builtin_amdgcn_kernarg_segment_ptr();
        asm volatile("" : "+s"(at), "+v"(tid));
        args_at = (const KV8Params *)at;
    }
    const KV8Params &a = *args_at;
    const KParams &p = a.p;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int whead = wave & (hpw - 1), part = wave >> hpw_sh;
    const int hk = (hblock * hpw + whead) * (PAIR ? 2 : 1);
    const int ratio = p.h_ratio;

    int bidb = bidb0, split = split0, nsplit = nsplit0;
    int r_lo = split, r_hi = split + 1, weight = nsplit;      // the part's ends inside its sequence, of `weight`
    if (runs) {
        while (hits == 0) {
            chunk += 64;
            if (chunk >= p.b || before - edge > (L + 1) * run) return;
            at_w = weight_of(kv8_steps<NR>(a, chunk + lane, q0));
            place();
        }
        const int at = __builtin_ctzll(hits);
        hits &= hits - 1;
        bidb = chunk + at;
        weight = __builtin_amdgcn_readlane(at_w, at);
        const int s = __builtin_amdgcn_readlane(at_s, at), lo = first_cut(s), hi = last_cut(s, weight);
        nsplit = hi < lo ? 1 : hi - lo + 2;
        split = hi < lo ? 0 : L - lo + 1;
        r_lo = split == 0 ? 0 : L * run - s;
        r_hi = split == nsplit - 1 ? weight : (L + 1) * run - s;
    }
    if (cut && tid == 0 && split == 0 && hblock == 0) a.n_split[bidb * n_mblocks + m_block] = nsplit;
    bidb = __builtin_amdgcn_readfirstlane(bidb);
    split = __builtin_amdgcn_readfirstlane(split);
    nsplit = __builtin_amdgcn_readfirstlane(nsplit);
    const bool is_split = nsplit > 1;

    const BlockInfo bi(p, bidb);
    const int sq = bi.sq;
    const int sk = kv8_total(a, bidb, p.knew ? p.seqlen_knew : 0);
    const int rows = min(sq, p.seqlen_q) * ratio;    // (results have places for seqlen_q positions)
    if (q0 >= rows || (a.max_rows > 0 && rows > a.max_rows)) {
        if (runs) continue;
        return;
    }
    const int pos_lo = q0 / ratio, pos_hi = min(rows - 1, q0 + 16 * NR - 1) / ratio;

    // keys that some row of the block sees, and this part of them
    const Kv8Seen seen(p, sq, sk);
    const int vis_lo = seen.lo(pos_lo), vis_hi = seen.hi(pos_hi);
    const int all_lo = seen.lo(pos_hi), all_hi = seen.hi(pos_lo);     // ... and that all of them see
    int n0 = vis_lo / A_STEP, n1 = vis_hi > vis_lo ? (vis_hi + A_STEP - 1) / A_STEP : n0;
    if (is_split) {
        const float per = (float)(n1 - n0) / (float)weight;
        const int n_all = n1 - n0, lo = min(n_all, (int)((float)r_lo * per));
        if (split < nsplit - 1) n1 = n0 + min(n_all, (int)((float)r_hi * per));
        n0 += lo;
    }

    const unsigned short *qg = (const unsigned short *)p.q + bi.q_off(p.q_bs, p.q_rs, bidb);
    unsigned short *og = (unsigned short *)p.o + bi.q_off(p.o_bs, p.o_rs, bidb);
    // row i of KV head `head`: query position i / ratio, query head head * ratio + i % ratio
    auto stat_at = [&](int head, int i) -> int64_t {
        const int64_t bh = (int64_t)bidb * p.h + head * ratio + i % ratio;
        return is_split ? ((int64_t)split * p.b * p.h + bh) * a.acc_sq + i / ratio : bh * p.seqlen_q + i / ratio;
    };
    float *lse = is_split ? p.lseaccum : p.lse;

    if (n1 <= n0) {
        for (int i = tid; i < hpw * 16 * NR * (HD / 8); i += A_NT) {
            const int ch = i % (HD / 8), rr = i / (HD / 8) % HR, head = hblock * hpw * (PAIR ? 2 : 1) + i / (HD / 8) / HR;
            const int row = q0 + rr;
            if (row >= rows || ch * 8 >= p.d) continue;
            if (is_split) {
                float *dst = p.oaccum + stat_at(head, row) * p.d + ch * 8;
                *(f32x4 *)dst = f32x4{0, 0, 0, 0};
                *(f32x4 *)(dst + 4) = f32x4{0, 0, 0, 0};
            } else {
                *(i32x4 *)(og + (int64_t)(row / ratio) * p.o_rs + (int64_t)(head * ratio + row % ratio) * p.o_hs + ch * 8) = i32x4{0, 0, 0, 0};
            }
            if (ch == 0) lse[stat_at(head, row)] = is_split ? -INFINITY : INFINITY;
        }
        if (runs) continue;
        return;
    }

    const int tl = lane & 1;                         // the tile of a step that this lane works out addresses for
    const int last_tile = (sk - 1) & ~15;
    // Page id of the lane's tile.  A tile of 16 keys lies in one page and in one block of the scales (both
    // are multiples of 16 rows); one that starts past the sequence's end takes its last tile (masked keys).
    const int *table = PAGED ? p.block_table + (int64_t)bidb * p.bt_bs : nullptr;
    int pid = PAGED ? 0 : p.cache_batch_idx ? p.cache_batch_idx[bidb] : bidb;
    auto load_pages = [&](int n) __attribute__((always_inline)) {
        if constexpr (PAGED) pid = table[kv8_div(min(n * A_STEP + 16 * tl, last_tile) >> 4, a.page_mul, a.page_sh)];
    };
    const int first = n0 + part;
    load_pages(min(first, n1 - 1));      // (in front of Q: the first rows wait for these)

    // Q operand: columns 64 j + 16 g + 8 s .. of k-step 2 j + s (PAIR: of both heads' k-steps s)
    constexpr int NQ = PAIR ? 2 : 2 * NJ;
    i32x4 qf[NR][NQ];
    int pos[NR];
    float slope[NR];
#pragma unroll
    for (int r = 0; r < NR; r++) {
        const int row = min(PAIR ? c & 7 : q0 + 16 * r + c, rows - 1);
        pos[r] = row / ratio;
        const int head = (hk + (PAIR ? c >> 3 : 0)) * ratio + row % ratio;
        slope[r] = p.alibi_slopes ? p.alibi_slopes[(int64_t)bidb * p.alibi_bs + head] / p.scale : 0.f;
        const unsigned short *qr = qg + (int64_t)pos[r] * p.q_rs + (int64_t)head * p.q_hs;
#pragma unroll
        for (int s = 0; s < NQ; s++) {
            const int col = 64 * (s >> 1) + 16 * g + 8 * (s & 1);
            qf[r][s] = col < p.d ? *(const i32x4 *)(qr + col) : i32x4{0, 0, 0, 0};
        }
    }

    const unsigned k_rs = (unsigned)p.k_rs, v_rs = (unsigned)p.v_rs;   // (under 2^27: sixteen rows and a head stay under 2^32)
    // lane offsets inside a tile of 16 keys: K 16 columns of key c, V chunk lane + 64 i
    unsigned koff[NJ], voff[NV / 2];
#pragma unroll
    for (int j = 0; j < NJ; j++) {
        const int col = (PAIR ? 0 : 64 * j) + 16 * g;
        koff[j] = (unsigned)c * k_rs + (PAIR ? j * (unsigned)p.k_hs : 0u) + (unsigned)(col < p.d ? col : 0);
    }
#pragma unroll
    for (int i = 0; i < NV / 2; i++) {
        const int ci = lane + 64 * i, vc = ci % CPR * 16 % HD;
        voff[i] = (unsigned)(ci / CPR) * v_rs + (PAIR ? (unsigned)(ci % CPR * 16 / HD) * (unsigned)p.v_hs : 0u) + (unsigned)(vc < p.d ? vc : 0);
    }

    // A step needs eight addresses: of K, V and their scales, for its two tiles.  Lane i of every eight works out
    // address i (tile i & 1 of K, V, K scale, V scale); the rows' are then read into scalar registers and the
    // scales fetched by the lanes that hold theirs.  (As scalar arithmetic this was a third of the step's
    // instructions, and few-wave launches are bound by those.)
    const int sel = (lane >> 1) & 3;
    const int sc_head = hk + (PAIR ? (lane >> 3) & 1 : 0);   // (PAIR: the second eight fetch the second head's scales)
    const unsigned char *lbase = sel == 0 ? (const unsigned char *)p.k + (int64_t)hk * p.k_hs
                               : sel == 1 ? (const unsigned char *)p.v + (int64_t)hk * p.v_hs
                               : sel == 2 ? a.ks + (int64_t)sc_head * a.ks_hs : a.vs + (int64_t)sc_head * a.vs_hs;
    const int64_t lps = sel == 0 ? p.k_bs : sel == 1 ? p.v_bs : sel == 2 ? a.ks_bs : a.vs_bs;
    const unsigned lrs = (unsigned)(sel == 0 ? p.k_rs : sel == 1 ? p.v_rs : sel == 2 ? a.ks_rs : a.vs_rs);

    struct Set {                 // one step's loads
        i32x4 k[2][NJ], v[NV];
        unsigned sc, bad;        // lanes 4..7 (mod 8): K scales of the two tiles, V scales; 255 for a page outside the pool
    };
    Set set[NBUF];
    // (the ids of the step after `n`, in `after`, are requested in front of n's rows: loads return in order, so
    // what waits for those ids later does not wait for the rows)
    auto load_step = [&](int n, Set &w, int after) __attribute__((always_inline)) {
        const unsigned bytes = n < n1 ? 0xffffffffu : 0u;           // past the last step: zeros, and no access
        const int key = min(n * A_STEP + 16 * tl, last_tile);
        const bool bad = (unsigned)pid >= (unsigned)a.num_pages;   // outside the pool: NaN, from the scale
        const unsigned pg = bad ? 0u : (unsigned)pid;
        const int row = PAGED ? key - kv8_div(key >> 4, a.page_mul, a.page_sh) * a.page_rows : key;
        const unsigned idx = (unsigned)(sel < 2 ? row : kv8_div(row >> 4, a.blk_mul, a.blk_sh));
        const unsigned char *at = lbase + (int64_t)pg * lps + (uint64_t)idx * lrs;
        load_pages(after);
        w.sc = *at;
        w.bad = bad ? 255u : 0u;
        const unsigned alo = (unsigned)(uintptr_t)at, ahi = (unsigned)((uintptr_t)at >> 32);
        auto rows_at = [&](int i) __attribute__((always_inline)) {   // address i of the eight, as a buffer's base
            const uint64_t base = (uint64_t)(unsigned)__builtin_amdgcn_readlane((int)alo, i) |
                                  (uint64_t)(unsigned)__builtin_amdgcn_readlane((int)ahi, i) << 32;
            return __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, bytes, 0x00020000);
        };
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const auto kr = rows_at(t);
#pragma unroll
            for (int j = 0; j < NJ; j++) w.k[t][j] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(kr, koff[j], 0, NT ? 2 : 0));
        }
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const auto vr = rows_at(2 + t);
#pragma unroll
            for (int i = 0; i < NV / 2; i++)
                w.v[t * (NV / 2) + i] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(vr, voff[i], 0, NT ? 2 : 0));
        }
        __builtin_amdgcn_sched_barrier(0);   // (steps' loads stay in order: the waits count them)
    };

    f32x4 o[NR][NDB];
    float m_run[NR], l_run[NR];
#pragma unroll
    for (int r = 0; r < NR; r++) {
        m_run[r] = -INFINITY;
        l_run[r] = 0.f;
#pragma unroll
        for (int db = 0; db < NDB; db++) o[r][db] = f32x4{0, 0, 0, 0};
    }
    const float c2 = p.scale_log2;
    char *vimg = smem + wave * Cfg::VB;
    // transposed read: lane i of group g names row {4g + j, 16 + 4g + j - 4}[j = (i >> 1)], half i & 1 of a chunk
    const int tj = c >> 1, trow = (tj < 4 ? 4 * g + tj : 12 + 4 * g + tj);
    const char *tr_base = vimg + trow * DP + (c & 1) * 8;
    const int tr_swz = kv8_swz<DP>(trow) << 4;
    int vwr[NV / 2];             // where a lane's V chunks go (the second tile: 16 rows on, chunks turned by a constant)
#pragma unroll
    for (int i = 0; i < NV / 2; i++) {
        const int ci = lane + 64 * i;
        vwr[i] = (ci / CPR) * DP + ((ci % CPR ^ kv8_swz<DP>(ci / CPR)) << 4);
    }
    constexpr int SWZ16 = kv8_swz<DP>(16) << 4;
    const bool has_alibi = p.alibi_slopes != nullptr;

    auto step = [&](const int n, Set &w, const int next) __attribute__((always_inline)) {
        const int k0 = n * A_STEP;
        float sc[PAIR ? 2 : 1][4];
        const int scl = (int)(w.sc | w.bad);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int e = 0; e < (PAIR ? 2 : 1); e++) sc[e][i] = e8m0_to_f32((unsigned)__builtin_amdgcn_readlane(scl, 4 + i + 8 * e));
        f32x4 s[NR][2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
#pragma unroll
            for (int r = 0; r < NR; r++) s[r][t] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                const float ks = sc[PAIR ? j : 0][t];
                const i32x4 k_lo = kv8_to16<BF16>(i32x2{w.k[t][j][0], w.k[t][j][1]}, ks);
                const i32x4 k_hi = kv8_to16<BF16>(i32x2{w.k[t][j][2], w.k[t][j][3]}, ks);
                if constexpr (PAIR) {    // each head's keys against all 16 columns; a column takes its own head's
                    f32x4 x = {0, 0, 0, 0};
                    x = mma16<BF16>(k_lo, qf[0][0], x);
                    x = mma16<BF16>(k_hi, qf[0][1], x);
#pragma unroll
                    for (int i = 0; i < 4; i++) s[0][t][i] = j == 0 ? x[i] : c < 8 ? s[0][t][i] : x[i];
                } else {
#pragma unroll
                    for (int r = 0; r < NR; r++) {
                        s[r][t] = mma16<BF16>(k_lo, qf[r][2 * j], s[r][t]);
                        s[r][t] = mma16<BF16>(k_hi, qf[r][2 * j + 1], s[r][t]);
                    }
                }
            }
        }
        if (k0 < vis_lo || k0 + A_STEP > vis_hi) {    // V of keys that no row sees must not count, whatever stands there
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const int key = k0 + (lane + 64 * (i % (NV / 2))) / CPR + 16 * (i / (NV / 2));
                if (key < vis_lo || key >= vis_hi) w.v[i] = i32x4{0, 0, 0, 0};
            }
#pragma unroll
            for (int t = 0; t < 2; t++)               // nor the scale of a tile of such keys (a NaN, a page outside the pool)
                if (k0 + 16 * t + 16 <= vis_lo || k0 + 16 * t >= vis_hi)
#pragma unroll
                    for (int e = 0; e < (PAIR ? 2 : 1); e++) sc[e][2 + t] = 1.f;
        }
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int at = i < NV / 2 ? vwr[i] : (vwr[i - NV / 2] ^ SWZ16) + 16 * DP;
            *(i32x4 *)(vimg + at) = w.v[i];
        }
        load_step(next, w, next + parts);

        const bool need = k0 + A_STEP > all_hi || k0 < all_lo;
        if (has_alibi) {
#pragma unroll
            for (int r = 0; r < NR; r++) {
                // (by the distance, in the causal case too: slope * key, equal up to a constant of the row, is large over
                // a long cache, and with it the rounding of every score)
                const int at = seen.shift + pos[r] - (k0 + 4 * g);
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) s[r][t][i] -= slope[r] * fabsf((float)(at - 16 * t - i));
            }
        }
        if (need) {
#pragma unroll
            for (int r = 0; r < NR; r++) {
                const int lo = seen.lo(pos[r]) - k0 - 4 * g;
                const int hi = seen.hi(pos[r]) - k0 - 4 * g;
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        s[r][t][i] = (16 * t + i >= lo && 16 * t + i < hi) ? s[r][t][i] : -INFINITY;
            }
        }
        i32x4 pf[NR];
#pragma unroll
        for (int r = 0; r < NR; r++) {
            float mx = fmaxf(fmaxf(fmaxf(s[r][0][0], s[r][0][1]), fmaxf(s[r][0][2], s[r][0][3])),
                             fmaxf(fmaxf(s[r][1][0], s[r][1][1]), fmaxf(s[r][1][2], s[r][1][3])));
            mx = quad_max(mx);
            // the reference point of the exponentials follows the maximum lazily (P stays under 2^4)
            if (__any((mx - m_run[r]) * c2 > 4.f)) {
                const float m_new = fmaxf(m_run[r], mx);
                const float alpha = __builtin_amdgcn_exp2f((m_run[r] - (m_new == -INFINITY ? 0.f : m_new)) * c2);
                l_run[r] *= alpha;
#pragma unroll
                for (int db = 0; db < NDB; db++) o[r][db] *= alpha;
                m_run[r] = m_new;
            }
            const float mc = (m_run[r] == -INFINITY ? 0.f : m_run[r]) * c2;
            float sum = 0.f;
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r][t][i], c2, -mc));
                    s[r][t][i] = e;
                    sum += e;
                }
            l_run[r] += sum;
#pragma unroll
            for (int t = 0; t < 2; t++) {
                pf[r][2 * t] = pack2<BF16>(s[r][t][0], s[r][t][1]);
                pf[r][2 * t + 1] = pack2<BF16>(s[r][t][2], s[r][t][3]);
            }
        }
#pragma unroll
        for (int db = 0; db < NDB; db++) {
            const i32x2 vt = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                (__attribute__((address_space(3))) i32x2 *)(tr_base + ((db << 4) ^ tr_swz)));
            i32x4 vf;
            const float *vs = sc[PAIR ? db * 16 / HD : 0] + 2;
            const i32x4 lo = kv8_to16<BF16>(i32x2{vt[0], 0}, vs[0]), hi = kv8_to16<BF16>(i32x2{vt[1], 0}, vs[1]);
            vf[0] = lo[0]; vf[1] = lo[1]; vf[2] = hi[0]; vf[3] = hi[1];
#pragma unroll
            for (int r = 0; r < NR; r++) o[r][db] = mma16<BF16>(vf, pf[r], o[r][db]);
        }
    };

    if (first < n1) {
#pragma unroll
        for (int i = 0; i < NBUF; i++) load_step(first + i * parts, set[i], first + (i + 1) * parts);
        // (one way out of the loop: with another in the middle the compiler's wait counts take the path
        // around it for one that leads back, and every step waits for the loads of the next)
        int n = first;
        if constexpr (NBUF == 2) {
            for (; n + parts < n1; n += 2 * parts) {
                step(n, set[0], n + 2 * parts);
                step(n + parts, set[1], n + 3 * parts);
            }
            if (n < n1) step(n, set[0], n + 2 * parts);
        } else {
            for (; n < n1; n += parts) step(n, set[0], n + parts);
        }
    }

    // ---- merge the waves of a head: weights from the maxima and sums, then 16 rows at a time ----
    float *ml = (float *)(smem + Cfg::MAIN);     // [wave][row][2]
#pragma unroll
    for (int r = 0; r < NR; r++) {
        const float l = quad_sum(l_run[r]);
        if (g == 0) {
            ml[((wave * NR + r) * 16 + c) * 2] = m_run[r];
            ml[((wave * NR + r) * 16 + c) * 2 + 1] = l;
        }
    }
#pragma unroll
    for (int r = 0; r < NR; r++) {
        __syncthreads();                          // statistics written; V images and the rows before are done with
        float m_all = -INFINITY, l_all = 0.f;
        for (int w = 0; w < parts; w++) m_all = fmaxf(m_all, ml[(((w * hpw + whead) * NR + r) * 16 + c) * 2]);
        const float m_fin = m_all == -INFINITY ? 0.f : m_all;
        for (int w = 0; w < parts; w++) {
            const float *e = ml + (((w * hpw + whead) * NR + r) * 16 + c) * 2;
            l_all += e[1] * __builtin_amdgcn_exp2f((e[0] - m_fin) * c2);
        }
        const bool none = m_all == -INFINITY && l_all == 0.f;
        const float f = none ? 0.f : __builtin_amdgcn_exp2f((m_run[r] - m_fin) * c2) / l_all;
        // (a wave that saw no key of this row has nothing to add: its O is a sum of zero weights times V, NaN if V is)
        const bool saw = ml[((wave * NR + r) * 16 + c) * 2 + 1] != 0.f;
        char *ob = smem + wave * 16 * Cfg::O_ROWB + c * Cfg::O_ROWB + g * 16;
#pragma unroll
        for (int db = 0; db < NDB; db++) {
            f32x4 x = o[r][db] * f;
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = saw ? x[i] : 0.f;
            *(f32x4 *)(ob + db * 64) = x;
        }
        const int row = PAIR ? c & 7 : q0 + 16 * r + c;
        if (part == 0 && g == 0 && row < rows)
            lse[stat_at(hk + (PAIR ? c >> 3 : 0), row)] = none ? (is_split ? -INFINITY : INFINITY) : m_all * p.scale + __logf(l_all);
        __syncthreads();
        const int live = PAIR ? 16 : min(16, rows - (q0 + 16 * r));           // rows of this 16 that exist
        for (int i = tid; i < hpw * live * (HD / 8); i += A_NT) {
            const int ch = i % (HD / 8), j = i / (HD / 8), hs = j & (hpw - 1), rr = j >> hpw_sh;
            const int orow = PAIR ? rr & 7 : q0 + 16 * r + rr, head = PAIR ? 2 * (hblock * hpw + hs) + (rr >> 3) : hblock * hpw + hs;
            if (ch * 8 >= p.d || (PAIR && orow >= rows)) continue;
            f32x4 a0 = {0, 0, 0, 0}, a1 = {0, 0, 0, 0};
            for (int w = 0; w < parts; w++) {
                const char *src = smem + ((w * hpw + hs) * 16 + rr) * Cfg::O_ROWB + (PAIR ? (rr >> 3) * HD * 4 : 0) + ch * 32;
                a0 += *(const f32x4 *)src;
                a1 += *(const f32x4 *)(src + 16);
            }
            const int opos = orow / ratio, ohead = head * ratio + orow - opos * ratio;
            if (is_split) {
                float *dst = p.oaccum + ((((int64_t)split * p.b + bidb) * p.h + ohead) * a.acc_sq + opos) * p.d + ch * 8;
                *(f32x4 *)dst = a0;
                *(f32x4 *)(dst + 4) = a1;
            } else {
                i32x4 w;
                w[0] = pack2<BF16>(a0[0], a0[1]); w[1] = pack2<BF16>(a0[2], a0[3]);
                w[2] = pack2<BF16>(a1[0], a1[1]); w[3] = pack2<BF16>(a1[2], a1[3]);
                *(i32x4 *)(og + (int64_t)opos * p.o_rs + (int64_t)ohead * p.o_hs + ch * 8) = w;
            }
        }
    }
    if (!runs) return;
    __syncthreads();                              // the next part's V images overwrite these rows
  }
}

// Merge of the parts of a row: LSE-weighted sum, in part order.  Its arguments in two cache lines: they lie in host
// memory, and the kernel is little else than its latency.
struct Kv8Merge {
    const float *o, *lse;
    float *out_lse;
    unsigned short *out;
    const int *n_split, *cu_q;     // n_split: parts of a row's keys; null: num_splits each (prefill kernel)
    int64_t out_bs, out_rs, out_hs;
    int b, h, d, acc_sq, num_splits, seqlen_q, max_rows, ratio, n_mblocks, rows_per_block;
};

struct Kv8MergeRow {
    int bidb, head, pos, n;        // n: parts, 0 where there is nothing to merge (one part is written in place)
    int64_t rows, at;              // rows of a part, the row in it
    __device__ __forceinline__ Kv8MergeRow(const Kv8Merge &a, int row) {
        pos = row % a.acc_sq;
        const int bh = row / a.acc_sq;
        bidb = bh / a.h;
        head = bh - bidb * a.h;
        rows = (int64_t)a.b * a.h * a.acc_sq;
        at = row;
        n = a.n_split ? a.n_split[bidb * a.n_mblocks + (pos * a.ratio + head % a.ratio) / a.rows_per_block] : a.num_splits;
        const int sq = a.cu_q ? a.cu_q[bidb + 1] - a.cu_q[bidb] : a.seqlen_q;
        if (pos >= sq || (a.max_rows > 0 && sq * a.ratio > a.max_rows) || n <= 1) n = 0;
    }
    __device__ __forceinline__ unsigned short *out(const Kv8Merge &a) const {
        return a.out + (a.cu_q ? (int64_t)a.cu_q[bidb] * a.out_rs : bidb * a.out_bs) + (int64_t)head * a.out_hs + (int64_t)pos * a.out_rs;
    }
    __device__ __forceinline__ float *lse(const Kv8Merge &a) const { return a.out_lse + ((int64_t)bidb * a.h + head) * a.seqlen_q + pos; }
};
template <bool BF16>
__device__ __forceinline__ void kv8_store8(unsigned short *to, f32x4 a0, f32x4 a1) {
    i32x4 w;
    w[0] = pack2<BF16>(a0[0], a0[1]); w[1] = pack2<BF16>(a0[2], a0[3]);
    w[2] = pack2<BF16>(a1[0], a1[1]); w[3] = pack2<BF16>(a1[2], a1[3]);
    *(i32x4 *)to = w;
}

// Up to 16 parts: a wave a row.  Lanes are (16-byte output chunk) x (lane over the parts); everything is requested before
// the number of parts is known.
constexpr int A_FEW_PARTS = 16;
template <bool BF16>
__global__ void __launch_bounds__(256)
kv8_combine_few_kernel(const Kv8Merge a) {
    const int lane = threadIdx.x & 63, row = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    if (row >= a.b * a.h * a.acc_sq) return;
    const Kv8MergeRow r(a, row);
    const int cpr = a.d / 8, nlane = min(4, 64 / cpr), ch = lane % cpr, sl = lane / cpr;   // (lanes past nlane * cpr idle)
    const int top = a.num_splits - 1;
    const float my_lse = a.lse[min(lane, top) * r.rows + r.at];
    constexpr int PRE = A_FEW_PARTS / 2;     // (at head dim 256 two lanes share the parts, else three or four)
    f32x4 x0[PRE], x1[PRE];
#pragma unroll
    for (int i = 0; i < PRE; i++) {
        if (i * nlane > top) break;
        const float *src = a.o + (min(sl + i * nlane, top) * r.rows + r.at) * a.d + ch * 8;
        x0[i] = *(const f32x4 *)src;
        x1[i] = *(const f32x4 *)(src + 4);
    }
    if (r.n == 0) return;
    const float my = lane < r.n ? my_lse : -INFINITY;
    float m = my;
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));   // (16 lanes hold them all)
    m = __shfl(m, 0);
    const float ref = m == -INFINITY ? 0.f : m;
    const float e = lane < r.n ? expf(my - ref) : 0.f;
    float sum = e;
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
    sum = __shfl(sum, 0);
    const bool none = sum == 0.f;                             // no part saw a key of this row
    const float w = none ? 0.f : e / sum;
    if (lane == 0) *r.lse(a) = none ? INFINITY : logf(sum) + ref;
    f32x4 a0 = {0, 0, 0, 0}, a1 = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < PRE; i++) {
        if (i * nlane >= r.n) break;
        const int sp = sl + i * nlane;
        const float f = __shfl(w, sp & 63);
        if (sl < nlane && sp < r.n) { a0 += x0[i] * f; a1 += x1[i] * f; }
    }
    for (int k = 1; k < nlane; k++) {
        const int from = (lane + k * cpr) & 63;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float y0 = __shfl(a0[i], from), y1 = __shfl(a1[i], from);
            if (sl == 0) { a0[i] += y0; a1[i] += y1; }
        }
    }
    if (sl == 0) kv8_store8<BF16>(r.out(a) + ch * 8, a0, a1);
}

// More: a workgroup a row, 256 threads on the same plan.
template <bool BF16>
__global__ void __launch_bounds__(256)
kv8_combine_kernel(const Kv8Merge a) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    __shared__ float s_w[128], s_red[2][2], s_part[256 * 8];
    const int cpr = a.d / 8, nlane = 256 / cpr, ch = tid % cpr, sl = tid / cpr;
    const Kv8MergeRow r(a, blockIdx.x);
    float my = a.lse[min(tid, a.num_splits - 1) * r.rows + r.at];
    constexpr int PRE = 4;
    f32x4 r0[PRE], r1[PRE];
#pragma unroll
    for (int i = 0; i < PRE; i++) {
        const float *src = a.o + (min(sl + i * nlane, a.num_splits - 1) * r.rows + r.at) * a.d + ch * 8;
        r0[i] = *(const f32x4 *)src;
        r1[i] = *(const f32x4 *)(src + 4);
    }
    const int ns = r.n;
    if (ns == 0) return;
    my = tid < ns ? my : -INFINITY;
    float m = my;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
    if (wave < 2 && lane == 0) s_red[0][wave] = m;           // (at most 128 parts: waves 0 and 1)
    __syncthreads();
    m = fmaxf(s_red[0][0], s_red[0][1]);
    const float ref = m == -INFINITY ? 0.f : m;
    float e = tid < ns ? expf(my - ref) : 0.f;
    float sum = e;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
    if (wave < 2 && lane == 0) s_red[1][wave] = sum;
    __syncthreads();
    sum = s_red[1][0] + s_red[1][1];
    const bool none = sum == 0.f;                             // no part saw a key of this row
    if (tid < 128) s_w[tid] = none ? 0.f : e / sum;
    if (tid == 0) *r.lse(a) = none ? INFINITY : logf(sum) + ref;
    __syncthreads();
    f32x4 a0 = {0, 0, 0, 0}, a1 = {0, 0, 0, 0};
    if (sl < nlane) {
#pragma unroll
        for (int i = 0; i < PRE; i++) {
            const int sp = sl + i * nlane;
            if (sp < ns) { a0 += r0[i] * s_w[sp]; a1 += r1[i] * s_w[sp]; }
        }
        for (int sp = sl + PRE * nlane; sp < ns; sp += nlane) {
            const float *src = a.o + (sp * r.rows + r.at) * a.d + ch * 8;
            a0 += *(const f32x4 *)src * s_w[sp];
            a1 += *(const f32x4 *)(src + 4) * s_w[sp];
        }
    }
    *(f32x4 *)(s_part + tid * 8) = a0;
    *(f32x4 *)(s_part + tid * 8 + 4) = a1;
    __syncthreads();
    if (tid < cpr) {
        for (int l = 1; l < min(nlane, ns); l++) {
            a0 += *(const f32x4 *)(s_part + (l * cpr + tid) * 8);
            a1 += *(const f32x4 *)(s_part + (l * cpr + tid) * 8 + 4);
        }
        kv8_store8<BF16>(r.out(a) + tid * 8, a0, a1);
    }
}

template <bool BF16>
static hipError_t launch_merge(const Kv8Merge &m, hipStream_t stream) {
    const long long rows = (long long)m.b * m.h * m.acc_sq;
    if (rows > 0x7fffffffLL) return hipErrorInvalidValue;
    if (m.num_splits <= A_FEW_PARTS) hipLaunchKernelGGL(kv8_combine_few_kernel<BF16>, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream, m);
    else hipLaunchKernelGGL(kv8_combine_kernel<BF16>, dim3((unsigned)rows), dim3(256), 0, stream, m);
    return hipGetLastError();
}

// The prefill kernel's parts, up to 8: many rows, so the bytes count and not the latency of a row.  A thread takes 8 columns
// of a row through all parts, in part order.  (The whole call, wave a row / this: 32768 rows of 2 parts, d128 88.3 / 68.8 us;
// 8192 of 8 107.4 / 102.7; but 2048 rows of 32 45.1 / 57.4, 1536 of 32 at d256 80.1 / 94.0: those go by the wave or workgroup.)
template <bool BF16>
__global__ void __launch_bounds__(256)
kv8_combine_rows_kernel(const Kv8Merge a) {
    const int cpr = a.d / 8;
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, rows = (int64_t)a.b * a.h * a.seqlen_q, row = at / cpr;
    const int ch = (int)(at - row * cpr);
    if (row >= rows) return;
    const float *lse = a.lse + row, *o = a.o + row * a.d + ch * 8;
    float m = -INFINITY;
    for (int i = 0; i < a.num_splits; i++) m = fmaxf(m, lse[i * rows]);
    const float ref = m == -INFINITY ? 0.f : m;
    float sum = 0.f;
    f32x4 a0 = {0, 0, 0, 0}, a1 = {0, 0, 0, 0};
#pragma unroll 4
    for (int i = 0; i < a.num_splits; i++) {
        const float w = expf(lse[i * rows] - ref);            // (a part that saw no key of this row: 0, and zeros)
        const float *src = o + i * rows * a.d;
        sum += w;
        a0 += *(const f32x4 *)src * w;
        a1 += *(const f32x4 *)(src + 4) * w;
    }
    const bool none = sum == 0.f;                             // no part saw a key of this row
    const float f = none ? 0.f : 1.f / sum;
    const int bh = (int)(row / a.seqlen_q), pos = (int)(row - (int64_t)bh * a.seqlen_q), bidb = bh / a.h, head = bh - bidb * a.h;
    if (ch == 0) a.out_lse[row] = none ? INFINITY : logf(sum) + ref;
    kv8_store8<BF16>(a.out + bidb * a.out_bs + (int64_t)head * a.out_hs + (int64_t)pos * a.out_rs + ch * 8, a0 * f, a1 * f);
}
hipError_t run_kv8_merge(const KParams &p, hipStream_t stream) {   // (dense queries)
    const Kv8Merge m{p.oaccum, p.lseaccum, p.lse, (unsigned short *)p.o, nullptr, nullptr, p.o_bs, p.o_rs, p.o_hs,
                     p.b, p.h, p.d, p.seqlen_q, p.num_splits, p.seqlen_q, 0, p.h_ratio, 1, 1};
    if (p.num_splits > 8) return p.is_bf16 ? launch_merge<true>(m, stream) : launch_merge<false>(m, stream);
    const long long blocks = ((long long)p.b * p.h * p.seqlen_q * (p.d / 8) + 255) / 256;
    if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
    if (p.is_bf16) hipLaunchKernelGGL(kv8_combine_rows_kernel<true>, dim3((unsigned)blocks), dim3(256), 0, stream, m);
    else hipLaunchKernelGGL(kv8_combine_rows_kernel<false>, dim3((unsigned)blocks), dim3(256), 0, stream, m);
    return hipGetLastError();
}

// Rows of a decode workgroup (above head dim 128 the accumulators of 32 rows do not fit beside the loads) and
// row blocks of the launch.
int kv8_decode_rows(int d, int rows) { return d <= 128 && rows > 16 ? 32 : 16; }

// Resident workgroups of 8 waves per CU: two where the kernel needs at most 128 registers, else one.
int kv8_decode_wgs_per_cu(int d, int rows, bool pairs) { return d <= 64 && rows <= 16 && !pairs ? 2 : 1; }

template <int DP, bool BF16, int NR, bool PAGED, bool NT, bool PAIR, bool RUNS = false>
static hipError_t launch_kv8(const KV8Params &a, hipStream_t stream) {
    const KParams &p = a.p;
    const int n_mblocks = (a.acc_sq * p.h_ratio + 16 * NR - 1) / (16 * NR);
    const long long blocks = (long long)n_mblocks * ((PAIR ? p.h_k / 2 : p.h_k) / a.heads_per_wg) * (p.num_splits > 1 ? a.split_grid : p.b);
    if (blocks <= 0) return hipSuccess;
    if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
    auto kern = fwd_kv8_kernel<DP, BF16, NR, PAGED, NT, RUNS, PAIR>;
    constexpr int lds = Kv8Cfg<DP, NR>::LDS_BYTES;
    static std::atomic<uint64_t> lds_set{0};
    if (hipError_t e = set_dyn_lds_once((const void *)kern, lds, lds_set); e != hipSuccess) return e;
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(A_NT), lds, stream, a, n_mblocks);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.num_splits <= 1) return e;
    const Kv8Merge m{p.oaccum, p.lseaccum, p.lse, (unsigned short *)p.o, a.n_split, p.cu_seqlens_q, p.o_bs, p.o_rs, p.o_hs,
                     p.b, p.h, p.d, a.acc_sq, p.num_splits, p.seqlen_q, a.max_rows, p.h_ratio, n_mblocks, 16 * NR};
    return launch_merge<BF16>(m, stream);
}

template <int DP, bool BF16, int NR, bool NT, bool PAIR = false>
static hipError_t launch_kv8_layout(const KV8Params &a, long long codes, hipStream_t stream) {
    const bool paged = a.p.block_table != nullptr;
    // Runs of steps (see the kernel) cost 2 us more before the first key; worth it where parts of equal length can leave
    // a good part of the chip idle: two parts a sequence at most, or up to eight of long ones.  kv4096 h32/8 d128, 64-row
    // pages: b129 311 -> 196 us, b65 154 -> 107; b48 kv16384 320 -> 274; b20 42.5 (44 with runs).
    // (In the 128 registers of head dim 64 the loop over pieces spills.)
    if constexpr (DP > 64 || NR > 1)
        if (a.p.num_splits > 1 && (a.p.b * 2 > a.split_goal || (a.p.b * 8 > a.split_goal && codes > VFA_KV8_LONG)))
            return paged ? launch_kv8<DP, BF16, NR, true, NT, PAIR, true>(a, stream) : launch_kv8<DP, BF16, NR, false, NT, PAIR, true>(a, stream);
    return paged ? launch_kv8<DP, BF16, NR, true, NT, PAIR>(a, stream) : launch_kv8<DP, BF16, NR, false, NT, PAIR>(a, stream);
}
template <int DP, bool BF16, int NR, bool PAIR = false>
static hipError_t launch_kv8_stream(const KV8Params &a, hipStream_t stream) {
    // codes that the calls of a program can name at all: what the sequences may hold, or the pool
    const long long codes = std::min((long long)a.p.b * a.cap, (long long)a.num_pages * a.page_rows) * a.p.h_k * a.p.d * 2;
    if constexpr (DP == 128)
        if (codes > VFA_KV8_LONG) return launch_kv8_layout<DP, BF16, NR, true, PAIR>(a, codes, stream);
    return launch_kv8_layout<DP, BF16, NR, false, PAIR>(a, codes, stream);
}
template <int DP, bool BF16>
static hipError_t launch_kv8_rows(const KV8Params &a, hipStream_t stream) {
    if constexpr (DP <= 128)
        if (kv8_decode_rows(a.p.d, a.acc_sq * a.p.h_ratio) == 32) return launch_kv8_stream<DP, BF16, 2>(a, stream);
    return launch_kv8_stream<DP, BF16, 1>(a, stream);
}

// Whether adjacent KV heads of `rows` (query, head) rows each go in pairs (their codes in one buffer's 32-bit offsets).
bool kv8_pairs(int d, int h_k, int rows, int64_t k_hs, int64_t v_hs) {
    return d <= 64 && h_k % 2 == 0 && rows <= 8 && std::min(k_hs, v_hs) >= 0 && std::max(k_hs, v_hs) <= 1 << 30;
}

// Adjacent KV heads of a workgroup: a key's codes of one head are d bytes, and reads of 512 contiguous bytes
// are what keeps HBM busy (b128 kv8192 h32/8 d128, heads 1 / 2 / 4: 465 / 391 / 374 us).
int kv8_heads_per_wg(int d, int h_k, bool pairs) {   // (in pairs: of those)
    if (pairs) d *= 2, h_k /= 2;
    int n = 1;
    while (n < 8 && n * d < 512 && h_k % (2 * n) == 0) n *= 2;
    return n;
}

hipError_t run_fwd_kv8(const KV8Params &a, hipStream_t stream) {
    const bool bf = a.p.is_bf16;
    if (a.pairs)
        return bf ? launch_kv8_stream<128, true, 1, true>(a, stream) : launch_kv8_stream<128, false, 1, true>(a, stream);
    if (a.p.d <= 64) return bf ? launch_kv8_rows<64, true>(a, stream) : launch_kv8_rows<64, false>(a, stream);
    if (a.p.d <= 128) return bf ? launch_kv8_rows<128, true>(a, stream) : launch_kv8_rows<128, false>(a, stream);
    return bf ? launch_kv8_rows<256, true>(a, stream) : launch_kv8_rows<256, false>(a, stream);
}

}  // namespace vfa
