// RMS norm of every query / key head and the position rotation in one pass, forward and backward.
//
//   forward   r = 1 / sqrt(mean(x^2) + eps),  n = x r w,  y = R n
//   backward  g = R^T dy,  dx = r (g w - x r^2 mean(g w x)),  dw = sum over rows of g x r
//
// R turns the pairs (2i, 2i + 1) (interleaved) or (i, i + rd / 2) by the token's angles and leaves the
// columns from rd on alone.  Everything is fp32 from the 16-bit inputs to the one rounding of the result:
// the normalised value is not rounded in front of the rotation.
//
// HBM-bound: the forward reads and writes q and k once; the backward reads x and dy and writes dx, and
// needs nothing else from the forward (r is recomputed from the x it reads anyway).  A head row is held by
// LPR lanes, 8 elements (16 bytes) each, so that sums over the row are log2(LPR) lane exchanges and the
// partner of a rotation pair (rd / 16 lanes away, as rd is a multiple of 16) is one exchange of the packed
// 16-bit words.  A wave stays with one token while it walks that token's heads: angles and weights are
// loaded once per wave and the rows of adjacent heads are adjacent in memory.
//
// Measured, b4 s4096 h32/8 d128 bf16: forward 74 us (336 MB, 4.5 TB/s), backward 115 us (503 MB, 4.4 TB/s) and 4.6 us for
// the sum of the weights' partials, where a 2 GiB copy runs at 4.9 TB/s.  One token of 64 sequences: 4.5 us, of which an
// empty launch is 3.6.
#include "vfa_qk_norm.h"
#include <algorithm>
#include <type_traits>

namespace vfa {

constexpr int N_NT = 256, N_NW = N_NT / 64;

template <bool BF16>
__device__ __forceinline__ void unpack8(i32x4 x, float f[8]) {
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = to_f32<BF16>((unsigned short)((unsigned)x[i >> 1] >> (16 * (i & 1))));
}
template <bool BF16>
__device__ __forceinline__ i32x4 pack8(const float f[8]) {
    i32x4 w;
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = pack2<BF16>(f[2 * i], f[2 * i + 1]);
    return w;
}
// N (4 or 8) consecutive elements of a table or weight held in fp32 or in the tensors' type, from element i
// on (a multiple of N)
template <bool BF16, int N>
__device__ __forceinline__ void ld_f(const void *p, int64_t i, int f32, float out[N]) {
    if (f32) {
#pragma unroll
        for (int j = 0; j < N / 4; j++) {
            const f32x4 v = *(const f32x4 *)((const float *)p + i + 4 * j);
#pragma unroll
            for (int t = 0; t < 4; t++) out[4 * j + t] = v[t];
        }
    } else {
#pragma unroll
        for (int j = 0; j < N / 4; j++) {
            const i32x2 v = *(const i32x2 *)((const unsigned short *)p + i + 4 * j);
#pragma unroll
            for (int t = 0; t < 4; t++) out[4 * j + t] = to_f32<BF16>((unsigned short)((unsigned)v[t >> 1] >> (16 * (t & 1))));
        }
    }
}
template <int LPR>
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
    for (int off = LPR / 2; off > 0; off >>= 1) x += __shfl_xor(x, off);
    return x;
}

// What a lane needs of the rotation for its 8 columns of a token.
struct Turn {
    float c[8], s[8];            // interleaved: the first 4 of each; outside rd: 1 and 0
    int partner;                 // lane that holds the other half's columns (pairs (i, i + rd / 2)), or own
};

template <bool BF16>
__device__ __forceinline__ void load_turn(const QKNormParams &p, int pos, int ch, int lane, Turn &t) {
    const int col = ch * 8, half = p.rd / 2;
    t.partner = lane;
#pragma unroll
    for (int i = 0; i < 8; i++) { t.c[i] = 1.f; t.s[i] = 0.f; }
    if (col >= p.rd) return;
    if (pos >= p.table_rows) {                 // no such row: loud, and nothing is read
#pragma unroll
        for (int i = 0; i < 8; i++) t.c[i] = t.s[i] = __uint_as_float(0x7fc00000u);
    }
    const int64_t row = (int64_t)pos * half;
    if (p.interleaved) {
        if (pos < p.table_rows) {
            ld_f<BF16, 4>(p.cos, row + col / 2, p.table_f32, t.c);
            ld_f<BF16, 4>(p.sin, row + col / 2, p.table_f32, t.s);
        }
    } else {
        const bool left = col < half;
        t.partner = left ? lane + half / 8 : lane - half / 8;
        if (pos < p.table_rows) {
            ld_f<BF16, 8>(p.cos, row + (left ? col : col - half), p.table_f32, t.c);
            ld_f<BF16, 8>(p.sin, row + (left ? col : col - half), p.table_f32, t.s);
        }
        if (left)
#pragma unroll
            for (int i = 0; i < 8; i++) t.s[i] = -t.s[i];   // y = n c + partner s
    }
}

// f turned (fwd) or turned back, with `o` the partner columns' values (pairs (i, i + rd / 2) only)
__device__ __forceinline__ void turn8(const QKNormParams &p, const Turn &t, bool inside, float f[8], const float o[8], float sign) {
    if (!inside) return;
    if (p.interleaved) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float a = f[2 * i], b = f[2 * i + 1], s = sign * t.s[i];
            f[2 * i] = a * t.c[i] - b * s;
            f[2 * i + 1] = a * s + b * t.c[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = f[i] * t.c[i] + o[i] * (sign * t.s[i]);
    }
}

__device__ __forceinline__ i32x4 from_lane(i32x4 x, int src) {
    i32x4 o;
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = __shfl(x[i], src);
    return o;
}

// What a wave works on.  An item is U passes over 64 / LPR head rows each of one token of q or of k (head0: the first
// pass's first); where a token has half as many heads as a pass has rows, or fewer, it is one pass over several tokens,
// and all of this is the lane's own (head0: its head; t.h if there is none).
struct Item {
    int bi, si, head0, pos;
};
__device__ __forceinline__ Item at_token(const QKNormParams &p, int64_t tok, int head0) {
    Item it;
    it.head0 = head0;
    it.bi = (int64_t)p.b * p.s <= 0x7fffffff ? (int)((unsigned)tok / (unsigned)p.s) : (int)(tok / p.s);
    it.si = (int)(tok - (int64_t)it.bi * p.s);
    it.pos = p.positions ? p.positions[it.bi * p.pos_bs + it.si] : it.si;
    return it;
}
__device__ __forceinline__ Item find_item(const QKNormParams &p, int64_t item, int parts, int rows) {
    const int64_t tok = parts == 1 ? item : item / parts;
    return at_token(p, tok, (int)(item - tok * parts) * rows);
}
// row `j` of an item of 1 << t.toks_sh tokens with `rows` rows
__device__ __forceinline__ Item find_row(const QKNormParams &p, const QKNormTensor &t, int64_t item, int j, int rows) {
    const int heads = rows >> t.toks_sh;                      // (a power of two)
    const int64_t tok = (item << t.toks_sh) + j / heads, all = (int64_t)p.b * p.s;
    return at_token(p, min(tok, all - 1), tok < all ? j % heads : t.h);
}

// The first blocks_q workgroups walk q's items, the others k's.
template <bool BF16, int LPR, int U>
__global__ void __launch_bounds__(N_NT)
qk_norm_fwd_kernel(const QKNormParams p, const int64_t items_q, const int64_t items_k, const int parts_q, const int parts_k) {
    constexpr int RPW = 64 / LPR;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool is_k = (int)blockIdx.x >= p.blocks_q;
    const QKNormTensor t = is_k ? p.t[1] : p.t[0];   // (selected field by field: an index would put both in scratch)
    const int blk = is_k ? blockIdx.x - p.blocks_q : blockIdx.x, n_blk = is_k ? p.blocks_k : p.blocks_q;
    const int64_t items = is_k ? items_k : items_q;
    const int parts = is_k ? parts_k : parts_q;
    const int sub = lane / LPR, ch = lane % LPR, col = ch * 8;
    const bool col_ok = col < p.d, inside = col < p.rd, pairs = inside && !p.interleaved;
    float w[8], wo[8];
    const int pcol = (col < p.rd / 2 ? col + p.rd / 2 : col - p.rd / 2);   // the partner's columns
#pragma unroll
    for (int i = 0; i < 8; i++) w[i] = wo[i] = 0.f;
    if (col_ok) ld_f<BF16, 8>(t.w, col, p.w_f32, w);
    if (pairs) ld_f<BF16, 8>(t.w, pcol, p.w_f32, wo);
    auto walk = [&](auto several) __attribute__((always_inline)) {
        constexpr bool MULTI = decltype(several)::value;
        constexpr int NU = MULTI ? 1 : U;
        for (int64_t item = (int64_t)blk * N_NW + wave; item < items; item += (int64_t)n_blk * N_NW) {
            const Item it = MULTI ? find_row(p, t, item, sub, RPW) : find_item(p, item, parts, RPW * U);
            auto head_of = [&](int u) __attribute__((always_inline)) { return MULTI ? it.head0 : it.head0 + u * RPW + sub; };
            const bool pad = it.pos < 0;               // zeros, whatever stands there
            i32x4 x[NU];
#pragma unroll
            for (int u = 0; u < NU; u++) {
                const unsigned short *xp = (const unsigned short *)t.x + it.bi * t.x_bs + it.si * t.x_rs + (col_ok ? col : 0);
                x[u] = (col_ok && head_of(u) < t.h) ? *(const i32x4 *)(xp + head_of(u) * t.x_hs) : i32x4{0, 0, 0, 0};
            }
            Turn tr;
            load_turn<BF16>(p, pad ? 0 : it.pos, ch, lane, tr);
#pragma unroll
            for (int u = 0; u < NU; u++) {
                float f[8], o[8], ss = 0.f;
                unpack8<BF16>(x[u], f);
#pragma unroll
                for (int j = 0; j < 8; j++) ss += f[j] * f[j];
                const float r = 1.f / sqrtf(row_sum<LPR>(ss) / (float)p.d + p.eps);
                unpack8<BF16>(from_lane(x[u], tr.partner), o);
#pragma unroll
                for (int j = 0; j < 8; j++) { f[j] *= r * w[j]; o[j] *= r * wo[j]; }
                turn8(p, tr, inside, f, o, 1.f);
                unsigned short *yp = (unsigned short *)t.y + it.bi * t.y_bs + it.si * t.y_rs + col;
                if (col_ok && head_of(u) < t.h) *(i32x4 *)(yp + head_of(u) * t.y_hs) = pad ? i32x4{0, 0, 0, 0} : pack8<BF16>(f);
            }
        }
    };
    if (t.toks_sh > 0) walk(std::true_type{}); else walk(std::false_type{});
}

// Backward.  The first blocks_q workgroups walk q's items, the others k's, so that a workgroup's partial dw
// (registers over its items, then lanes and waves in a fixed order) is one side's; a second kernel adds the
// partials in workgroup order: the same bits on every run.
template <bool BF16, int LPR, int U>
__global__ void __launch_bounds__(N_NT)
qk_norm_bwd_kernel(const QKNormParams p, const int64_t items_q, const int64_t items_k, const int parts_q, const int parts_k) {
    constexpr int RPW = 64 / LPR;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool is_k = (int)blockIdx.x >= p.blocks_q;
    const QKNormTensor t = is_k ? p.t[1] : p.t[0];
    const int blk = is_k ? blockIdx.x - p.blocks_q : blockIdx.x, n_blk = is_k ? p.blocks_k : p.blocks_q;
    const int64_t items = is_k ? items_k : items_q;
    const int parts = is_k ? parts_k : parts_q;
    const int sub = lane / LPR, ch = lane % LPR, col = ch * 8;
    const bool col_ok = col < p.d, inside = col < p.rd;
    float w[8], acc[8];
#pragma unroll
    for (int i = 0; i < 8; i++) w[i] = acc[i] = 0.f;
    if (col_ok) ld_f<BF16, 8>(t.w, col, p.w_f32, w);
    auto walk = [&](auto several) __attribute__((always_inline)) {
        constexpr bool MULTI = decltype(several)::value;
        constexpr int NU = MULTI ? 1 : U;
        for (int64_t item = (int64_t)blk * N_NW + wave; item < items; item += (int64_t)n_blk * N_NW) {
            const Item it = MULTI ? find_row(p, t, item, sub, RPW) : find_item(p, item, parts, RPW * U);
            auto head_of = [&](int u) __attribute__((always_inline)) { return MULTI ? it.head0 : it.head0 + u * RPW + sub; };
            const bool pad = it.pos < 0;               // zeros, whatever stands there
            i32x4 x[NU], g[NU];
#pragma unroll
            for (int u = 0; u < NU; u++) {
                const unsigned short *xp = (const unsigned short *)t.x + it.bi * t.x_bs + it.si * t.x_rs + (col_ok ? col : 0);
                const unsigned short *gp = (const unsigned short *)t.dy + it.bi * t.dy_bs + it.si * t.dy_rs + (col_ok ? col : 0);
                const bool ok = col_ok && head_of(u) < t.h && !pad;
                x[u] = ok ? *(const i32x4 *)(xp + head_of(u) * t.x_hs) : i32x4{0, 0, 0, 0};
                g[u] = ok ? *(const i32x4 *)(gp + head_of(u) * t.dy_hs) : i32x4{0, 0, 0, 0};
            }
            Turn tr;
            load_turn<BF16>(p, pad ? 0 : it.pos, ch, lane, tr);
#pragma unroll
            for (int u = 0; u < NU; u++) {
                const bool live = col_ok && head_of(u) < t.h;
                float f[8], q[8], o[8];
                unpack8<BF16>(x[u], f);
                unpack8<BF16>(g[u], q);
                unpack8<BF16>(from_lane(g[u], tr.partner), o);
                turn8(p, tr, inside, q, o, -1.f);             // g = R^T dy
                float ss = 0.f, sg = 0.f;
#pragma unroll
                for (int j = 0; j < 8; j++) { ss += f[j] * f[j]; sg += q[j] * w[j] * f[j]; }
                const float r = 1.f / sqrtf(row_sum<LPR>(ss) / (float)p.d + p.eps);
                const float m = row_sum<LPR>(sg) / (float)p.d * r * r;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    if (live && !pad) acc[j] += q[j] * f[j] * r;
                    f[j] = r * (q[j] * w[j] - f[j] * m);
                }
                unsigned short *yp = (unsigned short *)t.y + it.bi * t.y_bs + it.si * t.y_rs + col;
                if (t.y && live) *(i32x4 *)(yp + head_of(u) * t.y_hs) = pad ? i32x4{0, 0, 0, 0} : pack8<BF16>(f);
            }
        }
    };
    if (t.toks_sh > 0) walk(std::true_type{}); else walk(std::false_type{});
    if (!t.dw) return;
    __shared__ float s_acc[N_NW][LPR * 8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
#pragma unroll
        for (int off = 32; off >= LPR; off >>= 1) acc[i] += __shfl_xor(acc[i], off);
        if (sub == 0) s_acc[wave][col + i] = acc[i];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < p.d; c += N_NT) {
        float sum = 0.f;
#pragma unroll
        for (int v = 0; v < N_NW; v++) sum += s_acc[v][c];
        p.dw_part[(int64_t)blockIdx.x * p.d + c] = sum;
    }
}

// dw of q (blockIdx.y 0) and of k (1): 8 columns per workgroup, 32 threads a column, partials in a fixed order
template <bool BF16>
__global__ void __launch_bounds__(N_NT)
qk_norm_dw_kernel(const QKNormParams p) {
    const QKNormTensor t = blockIdx.y ? p.t[1] : p.t[0];
    if (!t.dw) return;
    const int c = blockIdx.x * 8 + (threadIdx.x & 7), part = threadIdx.x >> 3;
    const int first = blockIdx.y ? p.blocks_q : 0, n = blockIdx.y ? p.blocks_k : p.blocks_q;
    float sum = 0.f;
    constexpr int AHEAD = 8;       // loads in flight: the loop is latency
    const float *src = p.dw_part + (int64_t)first * p.d + c;
    for (int i = part; i < n; i += AHEAD * (N_NT / 8)) {
        float v[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; j++) {
            const int at = i + j * (N_NT / 8);
            v[j] = src[(int64_t)min(at, n - 1) * p.d];
        }
#pragma unroll
        for (int j = 0; j < AHEAD; j++) sum += i + j * (N_NT / 8) < n ? v[j] : 0.f;
    }
    __shared__ float s[N_NT];
    s[threadIdx.x] = sum;
    __syncthreads();
    if (threadIdx.x < 8) {
        for (int i = 1; i < N_NT / 8; i++) sum += s[i * 8 + threadIdx.x];
        if (p.w_f32) ((float *)t.dw)[c] = sum;
        else ((unsigned short *)t.dw)[c] = (unsigned short)(pack2<BF16>(sum, 0.f) & 0xffff);
    }
}

static int lanes_per_row(int d) { return d <= 64 ? 8 : d <= 128 ? 16 : 32; }
constexpr int N_U = 2;           // passes of a wave over a token's heads

// Parts of a token's heads, and a wave's items on one side.  (b19 s2517 h1/1 d128 forward: one token a pass 57 us, four 16.)
static int head_parts(const QKNormParams &p, int side) {
    const int rows = 64 / lanes_per_row(p.d) * N_U;
    return (p.t[side].h + rows - 1) / rows;
}
static int tokens_shift(const QKNormParams &p, int side) {
    const int rows = 64 / lanes_per_row(p.d);
    int sh = 0;
    while (p.t[side].h << (sh + 1) <= rows) sh++;
    return sh;
}
static int64_t side_items(const QKNormParams &p, int side) {
    const int sh = tokens_shift(p, side);
    return (((int64_t)p.b * p.s + (1 << sh) - 1) >> sh) * head_parts(p, side);
}

// Workgroups, shared out between the sides by their items: enough that every CU has work, few enough that the
// weights are loaded (and, backward, the partial sums of dw written) seldom.
void qk_norm_blocks(QKNormParams &p, int cus, bool bwd) {
    const long long iq = side_items(p, 0), ik = side_items(p, 1);
    const long long most = (bwd ? 6LL : 8LL) * cus, all = std::max(1LL, iq + ik);
    auto share = [&](long long items) {
        const long long want = (items + N_NW - 1) / N_NW, part = (most * items + all - 1) / all;
        return (int)std::max(1LL, std::min(want, part));
    };
    p.blocks_q = share(iq);
    p.blocks_k = share(ik);
    for (int side = 0; side < 2; side++) p.t[side].toks_sh = tokens_shift(p, side);
}

template <bool BF16, int LPR>
static hipError_t launch(const QKNormParams &p, bool bwd, hipStream_t stream) {
    const int parts_q = head_parts(p, 0), parts_k = head_parts(p, 1);
    const int64_t items_q = side_items(p, 0), items_k = side_items(p, 1);
    if (!bwd) {
        hipLaunchKernelGGL((qk_norm_fwd_kernel<BF16, LPR, N_U>), dim3((unsigned)(p.blocks_q + p.blocks_k)), dim3(N_NT), 0, stream, p,
                           items_q, items_k, parts_q, parts_k);
        return hipGetLastError();
    }
    hipLaunchKernelGGL((qk_norm_bwd_kernel<BF16, LPR, N_U>), dim3((unsigned)(p.blocks_q + p.blocks_k)), dim3(N_NT), 0, stream, p,
                       items_q, items_k, parts_q, parts_k);
    if (p.t[0].dw || p.t[1].dw) {
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        hipLaunchKernelGGL(qk_norm_dw_kernel<BF16>, dim3((unsigned)(p.d / 8), 2), dim3(N_NT), 0, stream, p);
    }
    return hipGetLastError();
}

hipError_t run_qk_norm_rotary(const QKNormParams &p, bool bwd, hipStream_t stream) {
    if ((int64_t)p.b * p.s <= 0) {
        // no token: the weights' gradients are zero, and the backward's kernels write that
        if (!bwd) return hipSuccess;
    }
    const int lpr = lanes_per_row(p.d);
    if (p.is_bf16) return lpr == 8 ? launch<true, 8>(p, bwd, stream) : lpr == 16 ? launch<true, 16>(p, bwd, stream) : launch<true, 32>(p, bwd, stream);
    return lpr == 8 ? launch<false, 8>(p, bwd, stream) : lpr == 16 ? launch<false, 16>(p, bwd, stream) : launch<false, 32>(p, bwd, stream);
}

}  // namespace vfa
