// PyTorch extension module `vllm_flash_attn_2_cuda` for MI355X: the tensor-level boundary the
// reference exposes through pybind (csrc/flash_attn/flash_api.cpp:939-946), re-implemented as a
// shim over the C ABI of libvfa_hip.so (include/vfa.h).  Same function names, argument order,
// return lists and error strings; `bwd` / `varlen_bwd` follow the call sites in
// vllm_flash_attn/flash_attn_interface.py:135-154 and :183-207 (the fork exports no backward).
#include <torch/python.h>
#include <torch/nn/functional.h>
#include <ATen/hip/HIPGeneratorImpl.h>
#include <ATen/hip/HIPContext.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/hip/HIPGraphsC10Utils.h>

#include <ATen/Parallel.h>

#include <algorithm>
#include <cmath>
#include <limits>
#include <optional>
#include <vector>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/variable.h>

#include "vfa.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<at::Tensor>;

void expect_shape(const Tensor &t, const char *name, std::initializer_list<int64_t> want) {
    TORCH_CHECK(t.sizes() == at::IntArrayRef(want.begin(), want.size()), name, " must have shape ",
                at::IntArrayRef(want.begin(), want.size()), ", got ", t.sizes());
}
void expect_gpu(const Tensor &t, const char *name) { TORCH_CHECK(t.is_cuda(), name, " must be on CUDA"); }
void expect_contig(const Tensor &t, const char *name) { TORCH_CHECK(t.is_contiguous(), name, " must be contiguous"); }

int dtype_code(const Tensor &q) {
    auto dt = q.scalar_type();
    TORCH_CHECK(dt == at::kHalf || dt == at::kBFloat16, "FlashAttention only support fp16 and bf16 data type");
    return dt == at::kBFloat16 ? VFA_BF16 : VFA_FP16;
}

void run(int rc) { TORCH_CHECK(rc == 0, vfa_last_error()); }

void *current_stream() { return (void *)at::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }

int cu_count() { return at::cuda::getCurrentDeviceProperties()->multiProcessorCount; }

Tensor pad_head(const Tensor &t, int64_t d) {
    if (d % 8 == 0) return t;
    namespace F = torch::nn::functional;
    return F::pad(t, F::PadFuncOptions({0, 8 - d % 8}));
}

void set_alibi(vfa_params &P, const OptTensor &slopes, int64_t b, int64_t h) {
    if (!slopes.has_value()) return;
    const Tensor &a = slopes.value();
    TORCH_CHECK(a.scalar_type() == at::kFloat, "ALiBi slopes must have dtype fp32");
    expect_gpu(a, "alibi_slopes");
    TORCH_CHECK(a.stride(-1) == 1, "ALiBi slopes tensor must have contiguous last dimension");
    TORCH_CHECK(a.sizes() == at::IntArrayRef({h}) || a.sizes() == at::IntArrayRef({b, h}),
                "alibi_slopes must have shape (num_heads) or (batch_size, num_heads)");
    P.alibi_slopes = a.data_ptr<float>();
    P.alibi_slopes_batch_stride = a.dim() == 2 ? a.stride(0) : 0;
}

// q/k/v/out pointers + strides (set_params_fprop, flash_api.cpp:53-77)
void set_qkvo(vfa_params &P, const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &out,
              bool batched) {
    P.q = q.data_ptr(); P.k = k.data_ptr(); P.v = v.data_ptr(); P.out = out.data_ptr();
    P.q_row_stride = q.stride(-3); P.q_head_stride = q.stride(-2);
    P.k_row_stride = k.stride(-3); P.k_head_stride = k.stride(-2);
    P.v_row_stride = v.stride(-3); P.v_head_stride = v.stride(-2);
    P.o_row_stride = out.stride(-3); P.o_head_stride = out.stride(-2);
    if (batched) {
        P.q_batch_stride = q.stride(0); P.k_batch_stride = k.stride(0);
        P.v_batch_stride = v.stride(0); P.o_batch_stride = out.stride(0);
    }
}

// Split scratch is held by the caller until the launches are enqueued (the reference lets it go
// back to the caching allocator before the launch, flash_api.cpp:212-215).
struct SplitScratch { Tensor lse, out; };
void plan_splits(vfa_params &P, SplitScratch &S, int num_splits, int64_t b, int64_t h, int64_t d,
                 int64_t sk, int64_t sq, const at::TensorOptions &opts) {
    if (num_splits < 1) {
        // Grouped query heads over few query tokens run packed into the rows of their KV head: the
        // library counts the work items the way its decode kernel is launched.
        num_splits = vfa_decode_num_splits(b, h, P.h_k > 0 ? P.h_k : h, d, sk, sq, cu_count());
    }
    TORCH_CHECK(num_splits <= 128, "num_splits > 128 not supported");
    P.num_splits = num_splits;
    if (num_splits > 1) {
        S.lse = torch::empty({num_splits, b, h, sq}, opts.dtype(at::kFloat));
        S.out = torch::empty({num_splits, b, h, sq, d}, opts.dtype(at::kFloat));
        P.softmax_lseaccum = S.lse.data_ptr<float>();
        P.oaccum = S.out.data_ptr<float>();
    }
}

int64_t round128(int64_t x) { return (x + 127) / 128 * 128; }

// Dropout set-up shared by fwd / varlen_fwd (flash_api.cpp:349-354,379-394): the optional
// Return_softmax tensor and the Philox state.  The generator's offset advances by b * h * 32, the
// number of draws the kernels index per (batch, head) (dropout.h:21).
Tensor plan_dropout(vfa_params &P, double p_dropout, bool return_softmax, int64_t b, int64_t h,
                    int64_t sq, int64_t sk, const at::TensorOptions &opts, Tensor &rng_state,
                    std::optional<at::Generator> &gen_) {
    TORCH_CHECK(p_dropout >= 0.0 && p_dropout < 1.0, "p_dropout must be in [0, 1)");
    Tensor p = torch::empty({0}, opts);  // flash_api.cpp:355-357: an empty tensor, not None
    if (return_softmax) {
        TORCH_CHECK(p_dropout > 0.0, "return_softmax is only supported when p_dropout > 0.0");
        // zero-filled (the reference leaves tiles its kernel never visits uninitialised)
        p = torch::zeros({b, h, round128(sq), round128(sk)}, opts);
        P.s_dmask = p.data_ptr();
        P.seqlen_q_rounded = (int)round128(sq);
        P.seqlen_k_rounded = (int)round128(sk);
    }
    P.p_dropout = (float)p_dropout;
    P.rng_state = (uint64_t *)rng_state.data_ptr<int64_t>();
    if (p_dropout > 0.0) {
        auto gen = at::get_generator_or_default<at::CUDAGeneratorImpl>(
            gen_, at::cuda::detail::getDefaultCUDAGenerator());
        std::lock_guard<std::mutex> lock(gen->mutex_);
        // flash_api.cpp:388-394: under graph capture the state is a pair of device pointers plus an
        // offset inside the graph, read by the kernel at replay time; otherwise plain values
        const at::PhiloxCudaState st = gen->philox_cuda_state((uint64_t)(b * h * 32));
        if (st.captured_) {
            P.philox_seed_ptr = st.seed_.ptr;
            P.philox_offset_ptr = st.offset_.ptr;
            P.philox_offset_intragraph = st.offset_intragraph_;
        } else {
            P.philox_seed = st.seed_.val;
            P.philox_offset = st.offset_.val;
        }
    }
    return p;
}


// ---------------------------------------------------------------------------------------------
// fp32 tensors in HOST memory: a plain C++ evaluation of the same function, so that
// flash_attn_func(q, k, v) on CPU fp32 inputs can be checked against torch's
// scaled_dot_product_attention without a GPU (the reference itself rejects such input,
// flash_api.cpp:263-271).  It is taken ONLY for CPU fp32 tensors -- nothing a GPU call could reach:
// CUDA tensors always run the HIP kernels, 16-bit CPU tensors are rejected as in the reference --
// and it is forward-only.  Same conventions as the kernels: bottom-right aligned causal / window
// mask (mask.h:171-172), ALiBi -slope * |i + sk - sq - j|, GQA head i -> i / (h / h_k), empty rows
// -> 0 with LSE = +inf, LSE = max * scale + ln(sum).
std::vector<Tensor> fwd_cpu_fp32(const Tensor &q_, const Tensor &k_, const Tensor &v_, OptTensor &out_,
                                 OptTensor &alibi_slopes_, double p_dropout, double softmax_scale, bool is_causal,
                                 int64_t wl, int64_t wr) {
    TORCH_CHECK(k_.scalar_type() == at::kFloat && v_.scalar_type() == at::kFloat && !k_.is_cuda() && !v_.is_cuda(),
                "q, k, v must all be fp32 CPU tensors for the host path");
    TORCH_CHECK(p_dropout == 0.0, "the host fp32 path has no dropout");
    TORCH_CHECK(q_.dim() == 4 && k_.dim() == 4 && v_.dim() == 4, "q, k, v must be 4-dimensional");
    const Tensor q = q_.contiguous(), k = k_.contiguous(), v = v_.contiguous();
    const int64_t b = q.size(0), sq = q.size(1), h = q.size(2), d = q.size(3);
    const int64_t sk = k.size(1), hk = k.size(2);
    TORCH_CHECK(b > 0, "batch size must be postive");
    TORCH_CHECK(hk > 0 && h % hk == 0, "Number of heads in key/value must divide number of heads in query");
    expect_shape(k, "k", {b, sk, hk, d});
    expect_shape(v, "v", {b, sk, hk, d});
    if (wl >= sk) wl = -1;                       // flash_api.cpp:289-294
    if (wr >= sk) wr = -1;
    if (is_causal) wr = 0;
    const float *slopes = nullptr;
    int64_t slope_bs = 0;
    Tensor sl;
    if (alibi_slopes_.has_value()) {
        sl = alibi_slopes_.value().contiguous();
        TORCH_CHECK(sl.scalar_type() == at::kFloat && !sl.is_cuda(), "ALiBi slopes must be fp32 on the CPU here");
        TORCH_CHECK(sl.sizes() == at::IntArrayRef({h}) || sl.sizes() == at::IntArrayRef({b, h}),
                    "alibi_slopes must have shape (num_heads) or (batch_size, num_heads)");
        slopes = sl.data_ptr<float>();
        slope_bs = sl.dim() == 2 ? h : 0;
    }
    Tensor out = torch::empty_like(q);
    Tensor lse = torch::empty({b, h, sq}, q.options());
    const float *Q = q.data_ptr<float>(), *K = k.data_ptr<float>(), *V = v.data_ptr<float>();
    float *O = out.data_ptr<float>(), *L = lse.data_ptr<float>();
    const float scale = (float)softmax_scale;
    const int64_t g = h / hk;
    at::parallel_for(0, b * h, 1, [&](int64_t lo, int64_t hi) {
        std::vector<float> s((size_t)sk);
        std::vector<double> acc((size_t)d);
        for (int64_t bh = lo; bh < hi; bh++) {
            const int64_t bi = bh / h, hi_ = bh % h, kh = hi_ / g;
            const float slope = slopes ? slopes[bi * slope_bs + hi_] : 0.f;
            for (int64_t i = 0; i < sq; i++) {
                const float *qr = Q + ((bi * sq + i) * h + hi_) * d;
                const int64_t j_lo = wl < 0 ? 0 : std::max<int64_t>(0, i + sk - sq - wl);
                const int64_t j_hi = wr < 0 ? sk : std::min<int64_t>(sk, i + 1 + sk - sq + wr);
                float m = -std::numeric_limits<float>::infinity();
                for (int64_t j = j_lo; j < j_hi; j++) {
                    const float *kr = K + ((bi * sk + j) * hk + kh) * d;
                    float dot = 0.f;
                    for (int64_t c = 0; c < d; c++) dot += qr[c] * kr[c];
                    dot = dot * scale - slope * std::fabs((float)(i + sk - sq - j));
                    s[(size_t)j] = dot;
                    m = std::max(m, dot);
                }
                float *orow = O + ((bi * sq + i) * h + hi_) * d;
                if (j_hi <= j_lo) {  // fully masked row (softmax.h:178-179)
                    std::fill(orow, orow + d, 0.f);
                    L[bh * sq + i] = std::numeric_limits<float>::infinity();
                    continue;
                }
                double sum = 0.0;
                std::fill(acc.begin(), acc.end(), 0.0);
                for (int64_t j = j_lo; j < j_hi; j++) {
                    const float pj = std::exp(s[(size_t)j] - m);
                    sum += pj;
                    const float *vr = V + ((bi * sk + j) * hk + kh) * d;
                    for (int64_t c = 0; c < d; c++) acc[(size_t)c] += (double)pj * vr[c];
                }
                for (int64_t c = 0; c < d; c++) orow[c] = (float)(acc[(size_t)c] / sum);
                L[bh * sq + i] = m + (float)std::log(sum);
            }
        }
    });
    if (out_.has_value()) {
        TORCH_CHECK(out_.value().sizes() == out.sizes() && out_.value().scalar_type() == at::kFloat,
                    "out must have the shape and dtype of q");
        out_.value().copy_(out);
        out = out_.value();
    }
    Tensor rng_state = torch::zeros({2}, q.options().dtype(at::kLong));
    return {out, q, k, v, out, lse, torch::empty({0}, q.options()), rng_state};
}

// ---------------------------------------------------------------------------------------------
// fwd  (flash_api.cpp:240-420)
std::vector<Tensor> fwd(Tensor &q, const Tensor &k, const Tensor &v, OptTensor &out_,
                        OptTensor &alibi_slopes_, const double p_dropout, const double softmax_scale,
                        bool is_causal, int64_t window_size_left, int64_t window_size_right,
                        const bool return_softmax, std::optional<at::Generator> gen_) {
    // (fp32 CPU tensors are rejected here like any other non-CUDA input, as the reference does
    //  (flash_api.cpp:263-271); the host evaluation is the separate entry `fwd_cpu_fp32`)
    const int dt = dtype_code(q);
    TORCH_CHECK(k.scalar_type() == q.scalar_type(), "query and key must have the same dtype");
    TORCH_CHECK(v.scalar_type() == q.scalar_type(), "query and value must have the same dtype");
    expect_gpu(q, "q"); expect_gpu(k, "k"); expect_gpu(v, "v");
    TORCH_CHECK(q.stride(-1) == 1 && k.stride(-1) == 1 && v.stride(-1) == 1,
                "Input tensor must have contiguous last dimension");
    TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, "q, k, v must be 4-dimensional");
    const auto in_sizes = q.sizes().vec();
    const int64_t b = in_sizes[0], d_og = in_sizes[3];
    int64_t sq = in_sizes[1], h = in_sizes[2];
    const int64_t sk = k.size(1), hk = k.size(2);
    TORCH_CHECK(b > 0, "batch size must be postive");
    TORCH_CHECK(d_og <= 256, "FlashAttention forward only supports head dimension at most 256");
    TORCH_CHECK(hk > 0 && h % hk == 0, "Number of heads in key/value must divide number of heads in query");

    // Single-token GQA decode: fold the query heads of a KV group into the row dimension
    // (flash_api.cpp:296-304) so one K/V stream serves the whole group.
    int64_t wl = window_size_left, wr = window_size_right;
    if (wl >= sk) wl = -1;
    if (wr >= sk) wr = -1;
    const bool causal_eff = is_causal && !(sq == 1 && !alibi_slopes_.has_value());
    const bool fold = sq == 1 && h > hk && wl < 0 && wr < 0 && !causal_eff && d_og % 8 == 0 &&
                      !alibi_slopes_.has_value() && p_dropout == 0.0;
    const int64_t g = h / hk;
    if (fold) {
        q = q.reshape({b, hk, g, d_og}).transpose(1, 2);
        sq = g;
        h = hk;
    }
    expect_shape(q, "q", {b, sq, h, d_og});
    expect_shape(k, "k", {b, sk, hk, d_og});
    expect_shape(v, "v", {b, sk, hk, d_og});

    Tensor qp = pad_head(q, d_og), kp = pad_head(k, d_og), vp = pad_head(v, d_og);
    Tensor out;
    if (out_.has_value()) {
        out = out_.value();
        TORCH_CHECK(out.scalar_type() == q.scalar_type(), "Output must have the same dtype as inputs");
        expect_gpu(out, "out");
        TORCH_CHECK(out.stride(-1) == 1, "Output tensor must have contiguous last dimension");
        expect_shape(out, "out", {b, in_sizes[1], in_sizes[2], d_og});
        if (fold) out = out.reshape({b, hk, g, d_og}).transpose(1, 2);
        if (d_og % 8 != 0) out = torch::empty_like(qp);
    } else {
        out = torch::empty_like(qp);
    }
    const int64_t d = qp.size(3);

    at::hip::HIPGuardMasqueradingAsCUDA device_guard{(c10::DeviceIndex)q.get_device()};
    auto opts = q.options();
    Tensor lse = torch::empty({b, h, sq}, opts.dtype(at::kFloat));
    Tensor rng_state = torch::empty({2}, opts.dtype(at::kLong));

    vfa_params P{};
    Tensor p_unused = plan_dropout(P, p_dropout, return_softmax, b, h, sq, sk, opts, rng_state, gen_);
    P.dtype = dt;
    set_qkvo(P, qp, kp, vp, out, true);
    P.softmax_lse = lse.data_ptr<float>();
    P.b = b; P.seqlen_q = sq; P.seqlen_k = sk; P.h = h; P.h_k = hk; P.d = d;
    P.softmax_scale = (float)softmax_scale;
    // after folding the call is never causal/local, so the raw flags can be passed through
    P.is_causal = is_causal; P.window_size_left = window_size_left; P.window_size_right = window_size_right;
    if (fold) { P.is_causal = 0; P.window_size_left = -1; P.window_size_right = -1; }
    set_alibi(P, alibi_slopes_, b, h);
    SplitScratch scratch;
    if (sk > 0) {
        if (p_dropout == 0.0) plan_splits(P, scratch, 0, b, h, d, sk, sq, opts);  // flash_api.cpp:206
        P.stream = current_stream();
        run(vfa_mha_fwd(&P));
    } else {  // flash_api.cpp:401-405
        out.zero_();
        lse.fill_(std::numeric_limits<float>::infinity());
    }

    Tensor out_padded = out;
    if (d_og % 8 != 0) {
        out = out.index({"...", torch::indexing::Slice(torch::indexing::None, d_og)});
        if (out_.has_value()) out_.value().copy_(out);
    }
    if (fold) {
        out = out.transpose(1, 2).reshape({b, 1, hk * sq, d_og});
        out_padded = out_padded.transpose(1, 2).reshape({b, 1, hk * sq, d_og});
        qp = qp.transpose(1, 2).reshape({b, 1, hk * sq, d_og});
        lse = lse.reshape({b, hk * sq, 1});
    }
    return {out, qp, kp, vp, out_padded, lse, p_unused, rng_state};
}

// ---------------------------------------------------------------------------------------------
// varlen_fwd  (flash_api.cpp:422-669)
std::vector<Tensor> varlen_fwd(Tensor &q, const Tensor &k, const Tensor &v, OptTensor &out_,
                               const Tensor &cu_seqlens_q, const Tensor &cu_seqlens_k,
                               OptTensor &seqused_k, OptTensor &block_table_, OptTensor &alibi_slopes_,
                               int64_t max_seqlen_q, const int64_t max_seqlen_k, const double p_dropout,
                               const double softmax_scale, const bool zero_tensors, bool is_causal,
                               int64_t window_size_left, int64_t window_size_right,
                               const bool return_softmax, std::optional<at::Generator> gen_) {
    const int dt = dtype_code(q);
    TORCH_CHECK(k.scalar_type() == q.scalar_type(), "query and key must have the same dtype");
    TORCH_CHECK(v.scalar_type() == q.scalar_type(), "query and value must have the same dtype");
    TORCH_CHECK(cu_seqlens_q.scalar_type() == at::kInt, "cu_seqlens_q must have dtype int32");
    TORCH_CHECK(cu_seqlens_k.scalar_type() == at::kInt, "cu_seqlens_k must have dtype int32");
    expect_gpu(q, "q"); expect_gpu(k, "k"); expect_gpu(v, "v");
    expect_gpu(cu_seqlens_q, "cu_seqlens_q"); expect_gpu(cu_seqlens_k, "cu_seqlens_k");
    const bool paged = block_table_.has_value();
    Tensor block_table;
    if (paged) {
        block_table = block_table_.value();
        expect_gpu(block_table, "block_table");
        TORCH_CHECK(block_table.scalar_type() == at::kInt, "block_table must have dtype torch.int32");
        TORCH_CHECK(block_table.stride(-1) == 1, "block_table must have contiguous last dimension");
    }
    TORCH_CHECK(q.stride(-1) == 1 && k.stride(-1) == 1 && v.stride(-1) == 1,
                "Input tensor must have contiguous last dimension");
    expect_contig(cu_seqlens_q, "cu_seqlens_q"); expect_contig(cu_seqlens_k, "cu_seqlens_k");
    TORCH_CHECK(q.dim() == 3, "q must be (total_q, num_heads, head_size)");

    const auto in_sizes = q.sizes().vec();
    const int64_t b = cu_seqlens_q.numel() - 1;
    int64_t h = in_sizes[1];
    const int64_t d_og = in_sizes[2];
    const int64_t hk = paged ? k.size(2) : k.size(1);
    const int64_t max_blocks = paged ? block_table.size(1) : 0;
    const int64_t num_blocks = paged ? k.size(0) : 0;
    const int64_t page = paged ? k.size(1) : 1;
    TORCH_CHECK(!paged || page % 16 == 0, "Paged KV cache block size must be divisible by 16");
    TORCH_CHECK(!(paged && p_dropout > 0.0), "dropout is not supported with a paged KV cache");

    int64_t wl = window_size_left, wr = window_size_right;
    if (wl >= max_seqlen_k) wl = -1;
    if (wr >= max_seqlen_k) wr = -1;
    const bool causal_eff = is_causal && !(max_seqlen_q == 1 && !alibi_slopes_.has_value());
    const bool fold = max_seqlen_q == 1 && h > hk && wl < 0 && wr < 0 && !causal_eff &&
                      d_og % 8 == 0 && !alibi_slopes_.has_value() && p_dropout == 0.0;
    const int64_t g = h / std::max<int64_t>(hk, 1);
    bool dense_q = false;
    if (fold) {  // flash_api.cpp:500-507: every sequence has exactly one query token
        q = q.reshape({b, hk, g, d_og}).transpose(1, 2).reshape({b * g, hk, d_og});
        max_seqlen_q = g;
        h = hk;
        dense_q = true;
    }
    const int64_t total_q = q.size(0);
    TORCH_CHECK(b > 0, "batch size must be positive");
    TORCH_CHECK(d_og <= 256, "FlashAttention forward only supports head dimension at most 256");
    TORCH_CHECK(hk > 0 && h % hk == 0, "Number of heads in key/value must divide number of heads in query");
    expect_shape(q, "q", {total_q, h, d_og});
    if (!paged) {
        const int64_t total_k = k.size(0);
        expect_shape(k, "k", {total_k, hk, d_og});
        expect_shape(v, "v", {total_k, hk, d_og});
    } else {
        expect_shape(k, "k", {num_blocks, page, hk, d_og});
        expect_shape(v, "v", {num_blocks, page, hk, d_og});
        expect_shape(block_table, "block_table", {b, max_blocks});
    }
    expect_shape(cu_seqlens_q, "cu_seqlens_q", {b + 1});
    expect_shape(cu_seqlens_k, "cu_seqlens_k", {b + 1});
    if (seqused_k.has_value()) {
        const Tensor &s = seqused_k.value();
        TORCH_CHECK(s.scalar_type() == at::kInt, "seqused_k must have dtype int32");
        TORCH_CHECK(s.is_cuda(), "seqused_k must be on CUDA device");
        TORCH_CHECK(s.is_contiguous(), "seqused_k must be contiguous");
        expect_shape(s, "seqused_k", {b});
    }

    Tensor qp = pad_head(q, d_og), kp = pad_head(k, d_og), vp = pad_head(v, d_og);
    Tensor out;
    if (out_.has_value()) {
        out = out_.value();
        TORCH_CHECK(out.scalar_type() == q.scalar_type(), "Output must have the same dtype as inputs");
        expect_gpu(out, "out");
        TORCH_CHECK(out.stride(-1) == 1, "Output tensor must have contiguous last dimension");
        expect_shape(out, "out", {in_sizes[0], in_sizes[1], d_og});
        if (fold) out = out.reshape({b, hk, g, d_og}).transpose(1, 2).reshape({b * g, hk, d_og});
        if (d_og % 8 != 0) out = torch::empty_like(qp);
    } else {
        out = torch::empty_like(qp);
    }
    const int64_t d = qp.size(2);

    at::hip::HIPGuardMasqueradingAsCUDA device_guard{(c10::DeviceIndex)q.get_device()};
    auto opts = q.options();
    Tensor lse = torch::empty({b, h, max_seqlen_q}, opts.dtype(at::kFloat));
    Tensor rng_state = torch::empty({2}, opts.dtype(at::kLong));
    if (zero_tensors) {
        out.zero_();
        lse.fill_(-std::numeric_limits<float>::infinity());
    }

    vfa_params P{};
    Tensor p_unused = plan_dropout(P, p_dropout, return_softmax, b, h, max_seqlen_q, max_seqlen_k, opts,
                                   rng_state, gen_);
    P.dtype = dt;
    set_qkvo(P, qp, kp, vp, out, false);
    P.softmax_lse = lse.data_ptr<float>();
    P.b = b; P.seqlen_q = max_seqlen_q; P.seqlen_k = max_seqlen_k; P.h = h; P.h_k = hk; P.d = d;
    P.total_q = (int)total_q;
    P.cu_seqlens_k = cu_seqlens_k.data_ptr<int32_t>();
    P.is_seqlens_k_cumulative = 1;
    if (seqused_k.has_value()) P.seqused_k = seqused_k.value().data_ptr<int32_t>();
    if (paged) {
        P.block_table = block_table.data_ptr<int32_t>();
        P.block_table_batch_stride = block_table.stride(0);
        P.k_batch_stride = kp.stride(0);
        P.v_batch_stride = vp.stride(0);
        P.page_block_size = page;
    }
    P.softmax_scale = (float)softmax_scale;
    P.is_causal = is_causal; P.window_size_left = window_size_left; P.window_size_right = window_size_right;
    set_alibi(P, alibi_slopes_, b, h);
    P.stream = current_stream();
    SplitScratch scratch;
    if (max_seqlen_k > 0) {
        if (dense_q) {
            // one query token per sequence, heads folded into rows: a dense (b, g, hk, d) query
            // against the ragged keys; this is the decode path (split-KV allowed)
            P.is_causal = 0; P.window_size_left = -1; P.window_size_right = -1;
            P.q_batch_stride = g * qp.stride(0); P.o_batch_stride = g * out.stride(0);
            plan_splits(P, scratch, 0, b, h, d, max_seqlen_k, max_seqlen_q, opts);
            P.cu_seqlens_q = nullptr;
            // ragged keys with a dense query go through the kv-cache entry semantics
            run(vfa_mha_varlen_fwd(&P));
        } else {
            P.cu_seqlens_q = cu_seqlens_q.data_ptr<int32_t>();
            run(vfa_mha_varlen_fwd(&P));
        }
    } else {
        out.zero_();
        lse.fill_(std::numeric_limits<float>::infinity());
    }

    Tensor out_padded = out;
    if (d_og % 8 != 0) {
        out = out.index({"...", torch::indexing::Slice(torch::indexing::None, d_og)});
        if (out_.has_value()) out_.value().copy_(out);
    }
    if (fold) {
        std::vector<int64_t> before = {b, max_seqlen_q, hk, d_og}, after = {b, hk * max_seqlen_q, d_og};
        out = out.reshape(before).transpose(1, 2).reshape(after);
        out_padded = out_padded.reshape(before).transpose(1, 2).reshape(after);
        qp = qp.reshape(before).transpose(1, 2).reshape(after);
        lse = lse.reshape({b, hk * max_seqlen_q, 1});
    }
    return {out, qp, kp, vp, out_padded, lse, p_unused, rng_state};
}

// ---------------------------------------------------------------------------------------------
// fwd_kvcache  (flash_api.cpp:671-937)
std::vector<Tensor> fwd_kvcache(Tensor &q, const Tensor &kcache, const Tensor &vcache,
                                std::optional<const Tensor> &k_, std::optional<const Tensor> &v_,
                                std::optional<const Tensor> &seqlens_k_,
                                std::optional<const Tensor> &rotary_cos_,
                                std::optional<const Tensor> &rotary_sin_,
                                std::optional<const Tensor> &cache_batch_idx_, OptTensor &block_table_,
                                OptTensor &alibi_slopes_, OptTensor &out_, const double softmax_scale,
                                bool is_causal, int64_t window_size_left, int64_t window_size_right,
                                bool is_rotary_interleaved, int64_t num_splits) {
    const int dt = dtype_code(q);
    TORCH_CHECK(kcache.scalar_type() == q.scalar_type(), "query and key must have the same dtype");
    TORCH_CHECK(vcache.scalar_type() == q.scalar_type(), "query and value must have the same dtype");
    expect_gpu(q, "q"); expect_gpu(kcache, "kcache"); expect_gpu(vcache, "vcache");
    TORCH_CHECK(q.stride(-1) == 1 && kcache.stride(-1) == 1 && vcache.stride(-1) == 1,
                "Input tensor must have contiguous last dimension");
    const bool paged = block_table_.has_value();
    Tensor block_table;
    if (paged) {
        TORCH_CHECK(!cache_batch_idx_.has_value(), "Paged KVcache does not support cache_batch_idx");
        block_table = block_table_.value();
        expect_gpu(block_table, "block_table");
        TORCH_CHECK(block_table.scalar_type() == at::kInt, "block_table must have dtype torch.int32");
        TORCH_CHECK(block_table.stride(-1) == 1, "block_table must have contiguous last dimension");
    }
    TORCH_CHECK(q.dim() == 4, "q must be (batch, seqlen_q, num_heads, head_size)");
    const auto in_sizes = q.sizes().vec();
    const int64_t b = in_sizes[0], d_og = in_sizes[3];
    int64_t sq = in_sizes[1], h = in_sizes[2];
    const int64_t max_blocks = paged ? block_table.size(1) : 0;
    const int64_t num_blocks = paged ? kcache.size(0) : 0;
    const int64_t page = paged ? kcache.size(1) : 1;
    TORCH_CHECK(!paged || page % 16 == 0, "Paged KV cache block size must be divisible by 16");
    const int64_t sk = paged ? max_blocks * page : kcache.size(1);
    const int64_t hk = kcache.size(2);
    const int64_t b_c = paged ? b : kcache.size(0);
    TORCH_CHECK(b > 0, "batch size must be postive");
    TORCH_CHECK(d_og <= 256, "FlashAttention forward only supports head dimension at most 256");
    TORCH_CHECK(hk > 0 && h % hk == 0, "Number of heads in key/value must divide number of heads in query");

    const bool causal_eff = is_causal && !(sq == 1 && !alibi_slopes_.has_value());
    const bool fold = sq == 1 && h > hk && window_size_left < 0 && window_size_right < 0 &&
                      !causal_eff && d_og % 8 == 0 && !alibi_slopes_.has_value();
    const int64_t g = h / hk;
    if (fold) {  // flash_api.cpp:747-755
        q = q.reshape({b, hk, g, d_og}).transpose(1, 2);
        sq = g;
        h = hk;
    }
    expect_shape(q, "q", {b, sq, h, d_og});
    if (!paged) {
        expect_shape(kcache, "kcache", {b_c, sk, hk, d_og});
        expect_shape(vcache, "vcache", {b_c, sk, hk, d_og});
    } else {
        expect_shape(kcache, "kcache", {num_blocks, page, hk, d_og});
        expect_shape(vcache, "vcache", {num_blocks, page, hk, d_og});
        expect_shape(block_table, "block_table", {b, max_blocks});
    }

    Tensor qp = pad_head(q, d_og), kcp = pad_head(kcache, d_og), vcp = pad_head(vcache, d_og);
    Tensor out;
    if (out_.has_value()) {
        out = out_.value();
        TORCH_CHECK(out.scalar_type() == q.scalar_type(), "Output must have the same dtype as inputs");
        expect_gpu(out, "out");
        TORCH_CHECK(out.stride(-1) == 1, "Output tensor must have contiguous last dimension");
        // The reference checks `out` against the FOLDED query shape here (flash_api.cpp:787), so a
        // caller-shaped (b, 1, h, d) output is rejected whenever the GQA decode fold applies, while
        // mha_fwd re-views it (flash_api.cpp:327-330).  Accept both: the caller's shape is viewed
        // like the query, the folded shape is taken as is.
        if (fold && out.dim() == 4 && out.size(1) == 1 && out.size(2) == hk * g) {
            expect_shape(out, "out", {b, 1, hk * g, d_og});
            out = out.reshape({b, hk, g, d_og}).transpose(1, 2);
        } else {
            expect_shape(out, "out", {b, sq, h, d_og});
        }
        if (d_og % 8 != 0) out = torch::empty_like(qp);
    } else {
        out = torch::empty_like(qp);
    }
    const int64_t d = qp.size(3);

    at::hip::HIPGuardMasqueradingAsCUDA device_guard{(c10::DeviceIndex)q.get_device()};
    auto opts = q.options();
    Tensor lse = torch::empty({b, h, sq}, opts.dtype(at::kFloat));

    vfa_params P{};
    P.dtype = dt;
    set_qkvo(P, qp, kcp, vcp, out, true);
    P.softmax_lse = lse.data_ptr<float>();
    P.b = b; P.seqlen_q = sq; P.seqlen_k = sk; P.h = h; P.h_k = hk; P.d = d;
    P.softmax_scale = (float)softmax_scale;
    P.is_causal = is_causal; P.window_size_left = window_size_left; P.window_size_right = window_size_right;
    if (fold) { P.is_causal = 0; P.window_size_left = -1; P.window_size_right = -1; }

    Tensor knew, vnew;
    if (k_.has_value()) {
        TORCH_CHECK(v_.has_value(), "If key is supplied, value must also be passed in");
        TORCH_CHECK(seqlens_k_.has_value(), "If key is supplied, seqlens_k must also be passed in");
        TORCH_CHECK(sq <= sk, "If key is supplied, it must have seqlen <= the seqlen of the KV cache");
        const Tensor &kk = k_.value(), &vv = v_.value();
        TORCH_CHECK(kk.scalar_type() == q.scalar_type(), "Key must have the same dtype as query");
        TORCH_CHECK(vv.scalar_type() == q.scalar_type(), "Value must have the same dtype as query");
        expect_gpu(kk, "k"); expect_gpu(vv, "v");
        TORCH_CHECK(kk.stride(-1) == 1, "Key tensor must have contiguous last dimension");
        TORCH_CHECK(vv.stride(-1) == 1, "Value tensor must have contiguous last dimension");
        const int64_t s_new = kk.size(1);
        expect_shape(kk, "k", {b, s_new, hk, d_og});
        expect_shape(vv, "v", {b, s_new, hk, d_og});
        knew = pad_head(kk, d_og); vnew = pad_head(vv, d_og);
        P.knew = knew.data_ptr(); P.vnew = vnew.data_ptr(); P.seqlen_knew = s_new;
        P.knew_batch_stride = knew.stride(0); P.knew_row_stride = knew.stride(-3); P.knew_head_stride = knew.stride(-2);
        P.vnew_batch_stride = vnew.stride(0); P.vnew_row_stride = vnew.stride(-3); P.vnew_head_stride = vnew.stride(-2);
    }
    if (seqlens_k_.has_value()) {
        const Tensor &s = seqlens_k_.value();
        TORCH_CHECK(s.scalar_type() == at::kInt, "seqlens_k must have dtype int32");
        expect_gpu(s, "seqlens_k"); expect_contig(s, "seqlens_k");
        expect_shape(s, "seqlens_k", {b});
        P.cu_seqlens_k = s.data_ptr<int32_t>();
    }
    P.is_seqlens_k_cumulative = !seqlens_k_.has_value();
    if (rotary_cos_.has_value()) {
        TORCH_CHECK(k_.has_value(), "If rotary cos/sin are provided, new key / value to be appended to KV cache must also be provided");
        const Tensor &rc = rotary_cos_.value();
        expect_gpu(rc, "rotary_cos");
        P.rotary_dim = rc.size(1) * 2;
        TORCH_CHECK(P.rotary_dim <= d, "rotary_dim must be <= headdim");
        TORCH_CHECK(P.rotary_dim % 16 == 0, "Only rotary dimensions divisible by 16 are currently supported");
        const int64_t s_ro = rc.size(0);
        TORCH_CHECK(s_ro >= sk, "cos/sin seqlen must be at least the seqlen of KV cache");
        expect_shape(rc, "rotary_cos", {s_ro, P.rotary_dim / 2});
        expect_contig(rc, "rotary_cos");
        TORCH_CHECK(rc.scalar_type() == q.scalar_type(), "rotary_cos must have the same dtype as query");
        TORCH_CHECK(rotary_sin_.has_value(), "If rotary cos is provided, rotary sin must also be provided");
        const Tensor &rs = rotary_sin_.value();
        expect_gpu(rs, "rotary_sin");
        expect_shape(rs, "rotary_sin", {s_ro, P.rotary_dim / 2});
        expect_contig(rs, "rotary_sin");
        TORCH_CHECK(rs.scalar_type() == q.scalar_type(), "rotary_cos must have the same dtype as query");
        P.rotary_cos = rc.data_ptr(); P.rotary_sin = rs.data_ptr();
        P.is_rotary_interleaved = is_rotary_interleaved;
        P.seqlen_ro = (int)s_ro;
    }
    if (cache_batch_idx_.has_value()) {
        const Tensor &c = cache_batch_idx_.value();
        expect_gpu(c, "cache_batch_idx"); expect_contig(c, "cache_batch_idx");
        TORCH_CHECK(c.scalar_type() == at::kInt, "cache_batch_idx must have dtype int32");
        P.cache_batch_idx = c.data_ptr<int32_t>();
    }
    if (paged) {
        P.block_table = block_table.data_ptr<int32_t>();
        P.block_table_batch_stride = block_table.stride(0);
        P.page_block_size = page;
    }
    set_alibi(P, alibi_slopes_, b, h);
    SplitScratch scratch;
    plan_splits(P, scratch, (int)num_splits, b, h, d, sk, sq, opts);
    P.stream = current_stream();
    run(vfa_mha_fwd_kvcache(&P));

    if (d_og % 8 != 0) {
        out = out.index({"...", torch::indexing::Slice(torch::indexing::None, d_og)});
        if (out_.has_value()) out_.value().copy_(out);
        if (k_.has_value()) {  // flash_api.cpp:924-929
            kcache.copy_(kcp.index({"...", torch::indexing::Slice(torch::indexing::None, d_og)}));
            vcache.copy_(vcp.index({"...", torch::indexing::Slice(torch::indexing::None, d_og)}));
        }
    }
    if (fold) {
        out = out.transpose(1, 2).reshape({b, 1, hk * sq, d_og});
        lse = lse.reshape({b, hk * sq, 1});
    }
    return {out, lse};
}

// ---------------------------------------------------------------------------------------------
// bwd / varlen_bwd  (call sites flash_attn_interface.py:135-154, :183-207; Flash_bwd_params,
// csrc/flash_attn/src/flash.h:145-183)
std::vector<Tensor> bwd_impl(const Tensor &dout_in, const Tensor &q_in, const Tensor &k_in, const Tensor &v_in,
                             const Tensor &out_in, const Tensor &softmax_lse, OptTensor &dq_, OptTensor &dk_,
                             OptTensor &dv_, const Tensor *cu_seqlens_q, const Tensor *cu_seqlens_k,
                             OptTensor &alibi_slopes_, int64_t max_seqlen_q, int64_t max_seqlen_k,
                             const double p_dropout, const double softmax_scale, const bool zero_tensors,
                             const bool is_causal, int64_t window_size_left, int64_t window_size_right,
                             const bool deterministic, std::optional<at::Generator> gen_,
                             OptTensor &rng_state_) {
    const bool varlen = cu_seqlens_q != nullptr;
    const int dt = dtype_code(q_in);
    for (const Tensor *t : {&k_in, &v_in, &out_in, &dout_in})
        TORCH_CHECK(t->scalar_type() == q_in.scalar_type(), "query, key, value, out and dout must have the same dtype");
    for (const Tensor *t : {&q_in, &k_in, &v_in, &out_in, &dout_in, &softmax_lse}) expect_gpu(*t, "input");
    for (const Tensor *t : {&q_in, &k_in, &v_in, &out_in, &dout_in})
        TORCH_CHECK(t->stride(-1) == 1, "Input tensor must have contiguous last dimension");
    // Head dims that are not a multiple of 8: the forward returned q, k, v, out zero-padded to the
    // next multiple (flash_api.cpp:310-319) and autograd saved those, while dout arrives with the
    // caller's head dim; upstream's mha_bwd pads dout (and slices dq, dk, dv back at the end).
    // Unpadded q / k / v / out are accepted too and padded here the same way.
    const int64_t d_og = dout_in.size(-1);
    const int64_t d_in = q_in.size(-1);
    const int64_t d_pad = (std::max(d_og, d_in) + 7) / 8 * 8;
    TORCH_CHECK(d_og <= d_in && d_pad - d_og < 8 && (d_in == d_og || d_in == d_pad),
                "dout must have the head size of q, or the head size q had before it was padded to a multiple of 8");
    auto pad_to = [&](const Tensor &t) {
        TORCH_CHECK(t.size(-1) == d_og || t.size(-1) == d_pad, "q, k, v, out must share one head size");
        if (t.size(-1) == d_pad) return t;
        namespace F = torch::nn::functional;
        return F::pad(t, F::PadFuncOptions({0, d_pad - t.size(-1)}));
    };
    const Tensor q = pad_to(q_in), k = pad_to(k_in), v = pad_to(v_in), out = pad_to(out_in), dout = pad_to(dout_in);
    TORCH_CHECK(p_dropout >= 0.0 && p_dropout < 1.0, "p_dropout must be in [0, 1)");
    TORCH_CHECK(softmax_lse.scalar_type() == at::kFloat, "softmax_lse must be fp32");

    int64_t b, sq, sk, h, hk, d, total_q = 0, total_k = 0;
    if (varlen) {
        TORCH_CHECK(cu_seqlens_q->scalar_type() == at::kInt && cu_seqlens_k->scalar_type() == at::kInt,
                    "cu_seqlens must have dtype int32");
        expect_gpu(*cu_seqlens_q, "cu_seqlens_q"); expect_gpu(*cu_seqlens_k, "cu_seqlens_k");
        expect_contig(*cu_seqlens_q, "cu_seqlens_q"); expect_contig(*cu_seqlens_k, "cu_seqlens_k");
        b = cu_seqlens_q->numel() - 1;
        total_q = q.size(0); h = q.size(1); d = q.size(2);
        total_k = k.size(0); hk = k.size(1);
        sq = max_seqlen_q; sk = max_seqlen_k;
        expect_shape(k, "k", {total_k, hk, d}); expect_shape(v, "v", {total_k, hk, d});
        expect_shape(out, "out", {total_q, h, d}); expect_shape(dout, "dout", {total_q, h, d});
    } else {
        b = q.size(0); sq = q.size(1); h = q.size(2); d = q.size(3);
        sk = k.size(1); hk = k.size(2);
        expect_shape(k, "k", {b, sk, hk, d}); expect_shape(v, "v", {b, sk, hk, d});
        expect_shape(out, "out", {b, sq, h, d}); expect_shape(dout, "dout", {b, sq, h, d});
    }
    TORCH_CHECK(b > 0, "batch size must be positive");
    TORCH_CHECK(d % 8 == 0, "head_size should be a multiple of 8");
    TORCH_CHECK(d <= 256, "FlashAttention backward only supports head dimension at most 256");
    TORCH_CHECK(hk > 0 && h % hk == 0, "Number of heads in key/value must divide number of heads in query");

    // Caller-provided gradients have the shape of the q / k / v that were passed in; when those were
    // not padded the kernels write padded temporaries and the head-dim prefix is copied back.
    auto grad_buf = [&](OptTensor &g_, const Tensor &like_in, const Tensor &like_pad) {
        if (!g_.has_value()) return torch::empty_like(like_pad);
        const Tensor &g = g_.value();
        TORCH_CHECK(g.scalar_type() == q.scalar_type(), "dq, dk, dv must have the same dtype as q");
        expect_gpu(g, "gradient");
        TORCH_CHECK(g.stride(-1) == 1, "gradient must have contiguous last dimension");
        TORCH_CHECK(g.sizes() == like_in.sizes(), "dq, dk, dv must have the shapes of q, k, v");
        return g.size(-1) == d_pad ? g : torch::empty_like(like_pad);
    };
    Tensor dq = grad_buf(dq_, q_in, q), dk = grad_buf(dk_, k_in, k), dv = grad_buf(dv_, v_in, v);

    at::hip::HIPGuardMasqueradingAsCUDA device_guard{(c10::DeviceIndex)q.get_device()};
    auto opts = q.options();
    const int64_t sq_rounded = (sq + 127) / 128 * 128;
    Tensor softmax_d = torch::empty({b, h, sq_rounded}, opts.dtype(at::kFloat));
    // No fp32 dq accumulator (the kernels accumulate in registers, flash.h:153-156); fp32 dK / dV
    // slabs only when the heads of a KV group are split over workgroups to fill the chip.
    const int head_splits = vfa_bwd_head_splits((int)b, (int)h, (int)hk, (int)sk, cu_count());
    const int64_t part_rows = varlen ? total_k : b * sk;
    Tensor dk_accum, dv_accum;
    if (head_splits > 1) {
        dk_accum = torch::empty({head_splits, part_rows, hk, d}, opts.dtype(at::kFloat));
        dv_accum = torch::empty({head_splits, part_rows, hk, d}, opts.dtype(at::kFloat));
    }
    if (zero_tensors) { dq.zero_(); dk.zero_(); dv.zero_(); softmax_d.zero_(); }

    vfa_params P{};
    P.dtype = dt;
    set_qkvo(P, q, k, v, out, !varlen);
    P.softmax_lse = softmax_lse.data_ptr<float>();
    P.b = b; P.seqlen_q = sq; P.seqlen_k = sk; P.h = h; P.h_k = hk; P.d = d;
    if (varlen) {
        P.cu_seqlens_q = cu_seqlens_q->data_ptr<int32_t>();
        P.cu_seqlens_k = cu_seqlens_k->data_ptr<int32_t>();
        P.is_seqlens_k_cumulative = 1;
    }
    P.softmax_scale = (float)softmax_scale;
    P.is_causal = is_causal; P.window_size_left = window_size_left; P.window_size_right = window_size_right;
    set_alibi(P, alibi_slopes_, b, h);
    P.dout = dout.data_ptr(); P.dq = dq.data_ptr(); P.dk = dk.data_ptr(); P.dv = dv.data_ptr();
    P.do_row_stride = dout.stride(-3); P.do_head_stride = dout.stride(-2);
    P.dq_row_stride = dq.stride(-3); P.dq_head_stride = dq.stride(-2);
    P.dk_row_stride = dk.stride(-3); P.dk_head_stride = dk.stride(-2);
    P.dv_row_stride = dv.stride(-3); P.dv_head_stride = dv.stride(-2);
    if (!varlen) {
        P.do_batch_stride = dout.stride(0); P.dq_batch_stride = dq.stride(0);
        P.dk_batch_stride = dk.stride(0); P.dv_batch_stride = dv.stride(0);
    }
    P.dsoftmax_sum = softmax_d.data_ptr<float>();
    P.deterministic = deterministic;
    P.stream = current_stream();
    if (head_splits > 1) {
        P.bwd_head_splits = head_splits;
        P.bwd_part_rows = part_rows;
        P.dk_accum = dk_accum.data_ptr<float>();
        P.dv_accum = dv_accum.data_ptr<float>();
    }
    // The forward's Philox state: the rng_state tensor it returned (read on the device), else a
    // fresh draw from the generator like the upstream backward does when none is passed.
    P.p_dropout = (float)p_dropout;
    if (p_dropout > 0.0) {
        if (rng_state_.has_value()) {
            const Tensor &rs = rng_state_.value();
            TORCH_CHECK(rs.is_cuda() && rs.scalar_type() == at::kLong && rs.numel() == 2 && rs.is_contiguous(),
                        "rng_state must be a CUDA int64 tensor with 2 elements");
            P.rng_state = (uint64_t *)rs.data_ptr<int64_t>();
        } else {
            auto gen = at::get_generator_or_default<at::CUDAGeneratorImpl>(
                gen_, at::cuda::detail::getDefaultCUDAGenerator());
            std::lock_guard<std::mutex> lock(gen->mutex_);
            const auto seed_offset = gen->philox_engine_inputs((uint64_t)(b * h * 32));
            P.philox_seed = seed_offset.first;
            P.philox_offset = seed_offset.second;
        }
    }
    if (sk > 0 && sq > 0) {
        run(varlen ? vfa_mha_varlen_bwd(&P) : vfa_mha_bwd(&P));
    } else {
        dq.zero_(); dk.zero_(); dv.zero_(); softmax_d.zero_();
    }
    if (d_og != d_pad) {  // upstream mha_bwd: slice the padding off (and fill the caller's buffers)
        auto unpad = [&](Tensor &g, OptTensor &g_) {
            if (g_.has_value() && g_.value().size(-1) != d_pad) g_.value().copy_(g.narrow(-1, 0, g_.value().size(-1)));
            g = g.narrow(-1, 0, d_og);
        };
        unpad(dq, dq_); unpad(dk, dk_); unpad(dv, dv_);
    }
    return {dq, dk, dv, softmax_d};
}

std::vector<Tensor> bwd(const Tensor &dout, const Tensor &q, const Tensor &k, const Tensor &v,
                        const Tensor &out, const Tensor &softmax_lse, OptTensor &dq_, OptTensor &dk_,
                        OptTensor &dv_, OptTensor &alibi_slopes_, const double p_dropout,
                        const double softmax_scale, const bool is_causal, int64_t window_size_left,
                        int64_t window_size_right, const bool deterministic,
                        std::optional<at::Generator> gen_, OptTensor &rng_state) {
    return bwd_impl(dout, q, k, v, out, softmax_lse, dq_, dk_, dv_, nullptr, nullptr, alibi_slopes_, 0, 0,
                    p_dropout, softmax_scale, false, is_causal, window_size_left, window_size_right,
                    deterministic, gen_, rng_state);
}

std::vector<Tensor> varlen_bwd(const Tensor &dout, const Tensor &q, const Tensor &k, const Tensor &v,
                               const Tensor &out, const Tensor &softmax_lse, OptTensor &dq_, OptTensor &dk_,
                               OptTensor &dv_, const Tensor &cu_seqlens_q, const Tensor &cu_seqlens_k,
                               OptTensor &alibi_slopes_, const int64_t max_seqlen_q,
                               const int64_t max_seqlen_k, const double p_dropout,
                               const double softmax_scale, const bool zero_tensors, const bool is_causal,
                               int64_t window_size_left, int64_t window_size_right,
                               const bool deterministic, std::optional<at::Generator> gen_,
                               OptTensor &rng_state) {
    return bwd_impl(dout, q, k, v, out, softmax_lse, dq_, dk_, dv_, &cu_seqlens_q, &cu_seqlens_k,
                    alibi_slopes_, max_seqlen_q, max_seqlen_k, p_dropout, softmax_scale, zero_tensors,
                    is_causal, window_size_left, window_size_right, deterministic, gen_, rng_state);
}

// ---------------------------------------------------------------------------------------------
// 8-bit KV cache (vfa_kv8_params) and the q / k norm + rotation: no counterpart in the reference

// Strides of dims that hold one index mean nothing and need not be aligned.
int64_t stride_of(const Tensor &t, int64_t dim) { return t.size(dim) > 1 ? t.stride(dim) : 0; }

// A 16-bit tensor as the kernels read it: last dim contiguous, 16-byte aligned rows; copied if it is not.
Tensor aligned_rows(const Tensor &t) {
    bool ok = ((uintptr_t)t.data_ptr() & 15) == 0 && (t.size(-1) <= 1 || t.stride(-1) == 1);
    for (int64_t i = 0; i + 1 < t.dim(); i++) ok = ok && stride_of(t, i) % 8 == 0;
    return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

void expect_with(const Tensor &t, const char *name, const Tensor &other) {
    expect_gpu(t, name);
    TORCH_CHECK(t.device() == other.device(), name, " must be on the device of the other tensors, ", other.device(), ", got ", t.device());
}
void expect_int32(const Tensor &t, const char *name, const Tensor &other) {
    TORCH_CHECK(t.scalar_type() == at::kInt, name, " must have dtype int32");
    expect_with(t, name, other);
    expect_contig(t, name);
}

// Cache, scales, lengths and pages; returns the batch size.
int64_t set_kv8_cache(vfa_kv8_params &P, const Tensor &kc, const Tensor &vc, const Tensor &ks, const Tensor &vs, int64_t b,
                      const OptTensor &seqlens_, const OptTensor &cache_batch_idx_, const OptTensor &block_table_) {
    for (const Tensor *t : {&kc, &vc}) {
        TORCH_CHECK(t->scalar_type() == at::kFloat8_e4m3fn, "k_cache and v_cache must have dtype float8_e4m3fn");
        TORCH_CHECK(t->dim() == 4, "k_cache and v_cache must be 4-dimensional");
        TORCH_CHECK(t->size(-1) <= 1 || t->stride(-1) == 1, "k_cache and v_cache must have contiguous last dimension");
    }
    expect_gpu(kc, "k_cache");
    expect_with(vc, "v_cache", kc);
    const bool paged = block_table_.has_value();
    const int64_t pages = kc.size(0), rows = kc.size(1), hk = kc.size(2), d = kc.size(3);
    TORCH_CHECK(pages > 0 && rows > 0 && hk > 0 && d > 0, "k_cache must not be empty");
    TORCH_CHECK(vc.sizes() == kc.sizes(), "v_cache must have the shape of k_cache, ", kc.sizes(), ", got ", vc.sizes());
    TORCH_CHECK(d <= 256 && d % 16 == 0, "8-bit KV cache: head dimension must be a multiple of 16, at most 256");
    for (const Tensor *t : {&ks, &vs}) {
        TORCH_CHECK(t->scalar_type() == at::kFloat8_e8m0fnu, "k_scale and v_scale must have dtype float8_e8m0fnu");
        expect_with(*t, "k_scale / v_scale", kc);
        TORCH_CHECK(t->dim() == 3 && t->size(0) == pages && t->size(2) == hk && t->sizes() == ks.sizes(),
                    "k_scale and v_scale must have shape (", pages, ", blocks of tokens, ", hk, "), got ", t->sizes());
    }
    const int64_t nblk = ks.size(1);
    TORCH_CHECK(nblk > 0 && rows % nblk == 0 && (rows / nblk) % 16 == 0,
                "8-bit KV cache: the tokens per scale must be a multiple of 16 that divides the rows of a page (", rows, " rows, ", nblk, " scales)");
    TORCH_CHECK(rows <= (1 << 30) && pages <= (1 << 30), "8-bit KV cache: too large");
    P.a.k = kc.data_ptr(); P.a.v = vc.data_ptr();
    P.a.k_batch_stride = stride_of(kc, 0); P.a.k_row_stride = stride_of(kc, 1); P.a.k_head_stride = stride_of(kc, 2);
    P.a.v_batch_stride = stride_of(vc, 0); P.a.v_row_stride = stride_of(vc, 1); P.a.v_head_stride = stride_of(vc, 2);
    P.k_scale = ks.data_ptr(); P.v_scale = vs.data_ptr();
    P.k_scale_batch_stride = stride_of(ks, 0); P.k_scale_row_stride = stride_of(ks, 1); P.k_scale_head_stride = stride_of(ks, 2);
    P.v_scale_batch_stride = stride_of(vs, 0); P.v_scale_row_stride = stride_of(vs, 1); P.v_scale_head_stride = stride_of(vs, 2);
    P.scale_block = (int)(rows / nblk);
    P.num_pages = (int)pages;
    if (b < 0) {
        TORCH_CHECK(seqlens_.has_value(), "cache_seqlens must be passed in");
        b = seqlens_.value().numel();
    }
    TORCH_CHECK(b > 0, "batch size must be postive");
    P.a.b = (int)b; P.a.h_k = (int)hk; P.a.d = (int)d;
    if (seqlens_.has_value()) {
        const Tensor &s = seqlens_.value();
        expect_int32(s, "cache_seqlens", kc);
        expect_shape(s, "cache_seqlens", {b});
        P.a.cu_seqlens_k = s.data_ptr<int32_t>();
    }
    if (cache_batch_idx_.has_value()) {
        TORCH_CHECK(!paged, "Paged KVcache does not support cache_batch_idx");
        expect_int32(cache_batch_idx_.value(), "cache_batch_idx", kc);
        expect_shape(cache_batch_idx_.value(), "cache_batch_idx", {b});
        P.a.cache_batch_idx = cache_batch_idx_.value().data_ptr<int32_t>();
    }
    if (paged) {
        const Tensor &bt = block_table_.value();
        TORCH_CHECK(bt.scalar_type() == at::kInt, "block_table must have dtype torch.int32");
        expect_with(bt, "block_table", kc);
        TORCH_CHECK(bt.dim() == 2 && bt.size(0) == b && bt.size(1) > 0, "block_table must have shape (batch_size, max_blocks)");
        TORCH_CHECK(bt.size(1) <= 1 || bt.stride(-1) == 1, "block_table must have contiguous last dimension");
        TORCH_CHECK(bt.size(1) * rows <= (1 << 30), "8-bit KV cache: too large");
        P.a.block_table = bt.data_ptr<int32_t>();
        P.a.block_table_batch_stride = stride_of(bt, 0);
        P.a.page_block_size = (int)rows;
        P.a.seqlen_k = (int)(bt.size(1) * rows);
    } else {
        TORCH_CHECK(cache_batch_idx_.has_value() || b <= pages, "batch size exceeds the cache's");
        P.a.seqlen_k = (int)rows;
    }
    return b;
}

// New tokens (dense or ragged); the returned pair keeps copies alive until the launch.
std::pair<Tensor, Tensor> set_kv8_new(vfa_kv8_params &P, const Tensor &k_, const Tensor &v_, const Tensor &kc, const OptTensor &cu_, int64_t max_seqlen) {
    const int dt = dtype_code(k_);
    TORCH_CHECK(v_.scalar_type() == k_.scalar_type(), "k and v must have the same dtype");
    expect_with(k_, "k", kc);
    expect_with(v_, "v", kc);
    TORCH_CHECK(k_.dim() == (cu_.has_value() ? 3 : 4), cu_.has_value() ? "k and v must be (total, nheads_k, headdim) with cu_seqlens"
                                                                       : "k and v must be (batch_size, seqlen, nheads_k, headdim), or ragged with cu_seqlens");
    TORCH_CHECK(k_.sizes() == v_.sizes(), "k and v must have the same shape");
    TORCH_CHECK(k_.size(-2) == P.a.h_k && k_.size(-1) == P.a.d, "k and v must have the heads and the head size of the cache, (", P.a.h_k, ", ", P.a.d, "), got ", k_.sizes());
    Tensor k = aligned_rows(k_), v = aligned_rows(v_);
    P.a.dtype = dt;
    P.a.knew = k.data_ptr(); P.a.vnew = v.data_ptr();
    P.a.knew_row_stride = stride_of(k, -3); P.a.knew_head_stride = stride_of(k, -2);
    P.a.vnew_row_stride = stride_of(v, -3); P.a.vnew_head_stride = stride_of(v, -2);
    if (cu_.has_value()) {
        expect_int32(cu_.value(), "cu_seqlens", kc);
        expect_shape(cu_.value(), "cu_seqlens", {(int64_t)P.a.b + 1});
        TORCH_CHECK(max_seqlen >= 0 && max_seqlen <= (1 << 30), "max_seqlen out of range");
        P.cu_seqlens_new = cu_.value().data_ptr<int32_t>();
        P.a.seqlen_knew = (int)std::min<int64_t>(max_seqlen, k.size(0));
    } else {
        TORCH_CHECK(k.size(0) == P.a.b, "k and v must have the batch size ", P.a.b, ", got ", k.size(0));
        TORCH_CHECK(k.size(1) <= (1 << 30), "too many new tokens");
        P.a.knew_batch_stride = stride_of(k, 0); P.a.vnew_batch_stride = stride_of(v, 0);
        P.a.seqlen_knew = (int)k.size(1);
    }
    return {k, v};
}

void kv8_quantize(const Tensor &k, const Tensor &v, const Tensor &kc, const Tensor &vc, const Tensor &ks, const Tensor &vs,
                  const Tensor &seqlens, const OptTensor &cache_batch_idx, const OptTensor &block_table, const OptTensor &cu_seqlens,
                  int64_t max_seqlen) {
    at::NoGradGuard no_grad;   // a cache is not trained through
    vfa_kv8_params P{};
    set_kv8_cache(P, kc, vc, ks, vs, -1, seqlens, cache_batch_idx, block_table);
    at::hip::HIPGuardMasqueradingAsCUDA device_guard{(c10::DeviceIndex)kc.get_device()};
    const auto keep = set_kv8_new(P, k, v, kc, cu_seqlens, max_seqlen);
    if (keep.first.numel() == 0) return;
    P.a.stream = current_stream();
    run(vfa_kv8_quantize(&P));
}

std::vector<Tensor> kv8_dequantize(const Tensor &kc, const Tensor &vc, const Tensor &ks, const Tensor &vs, const Tensor &seqlens,
                                   const OptTensor &cache_batch_idx, const OptTensor &block_table, const OptTensor &cu_seqlens,
                                   int64_t rows, at::ScalarType dtype) {
    at::NoGradGuard no_grad;   // a cache is not trained through
    vfa_kv8_params P{};
    const int64_t b = set_kv8_cache(P, kc, vc, ks, vs, -1, seqlens, cache_batch_idx, block_table);
    TORCH_CHECK(dtype == at::kHalf || dtype == at::kBFloat16, "FlashAttention only support fp16 and bf16 data type");
    TORCH_CHECK(rows >= 0 && rows <= (1 << 30), "max_seqlen / total_seqlen out of range");
    at::hip::HIPGuardMasqueradingAsCUDA device_guard{(c10::DeviceIndex)kc.get_device()};
    const int64_t hk = P.a.h_k, d = P.a.d;
    Tensor k, v;
    if (cu_seqlens.has_value()) {
        expect_int32(cu_seqlens.value(), "cu_seqlens", kc);
        expect_shape(cu_seqlens.value(), "cu_seqlens", {b + 1});
        P.cu_seqlens_out = cu_seqlens.value().data_ptr<int32_t>();
        P.rows_out = rows;
        k = torch::empty({rows, hk, d}, kc.options().dtype(dtype));
    } else {
        P.seqlen_out = (int)rows;
        P.rows_out = b * rows;
        k = torch::empty({b, rows, hk, d}, kc.options().dtype(dtype));
    }
    v = torch::empty_like(k);
    if (k.numel() == 0) return {k, v};
    P.a.dtype = dtype == at::kBFloat16 ? VFA_BF16 : VFA_FP16;
    P.k_out = k.data_ptr(); P.v_out = v.data_ptr();
    P.ko_batch_stride = P.vo_batch_stride = rows * hk * d;
    P.ko_row_stride = P.vo_row_stride = hk * d;
    P.ko_head_stride = P.vo_head_stride = d;
    P.a.stream = current_stream();
    run(vfa_kv8_dequantize(&P));
    return {k, v};
}

std::vector<Tensor> fwd_kv8(const Tensor &q_, const Tensor &kc, const Tensor &vc, const Tensor &ks, const Tensor &vs, OptTensor &k_,
                            OptTensor &v_, OptTensor &seqlens, OptTensor &cache_batch_idx, OptTensor &block_table, OptTensor &alibi_slopes,
                            OptTensor &out_, OptTensor &cu_seqlens_q, int64_t max_seqlen_q, const double softmax_scale, bool is_causal,
                            int64_t window_size_left, int64_t window_size_right, int64_t num_splits) {
    at::NoGradGuard no_grad;   // a cache is not trained through
    const int dt = dtype_code(q_);
    const bool ragged = cu_seqlens_q.has_value();
    TORCH_CHECK(q_.dim() == (ragged ? 3 : 4), ragged ? "q must be (total_q, nheads, headdim) with cu_seqlens_q"
                                                     : "q must be (batch_size, seqlen_q, nheads, headdim), or ragged with cu_seqlens_q");
    if (ragged) TORCH_CHECK(cu_seqlens_q.value().dim() == 1 && cu_seqlens_q.value().numel() > 1, "cu_seqlens_q must have shape (batch_size + 1)");
    const int64_t b = ragged ? cu_seqlens_q.value().numel() - 1 : q_.size(0);
    vfa_kv8_params P{};
    TORCH_CHECK(b > 0, "batch size must be postive");
    set_kv8_cache(P, kc, vc, ks, vs, b, seqlens, cache_batch_idx, block_table);
    expect_with(q_, "q", kc);
    at::hip::HIPGuardMasqueradingAsCUDA device_guard{(c10::DeviceIndex)kc.get_device()};
    const int64_t h = q_.size(-2), d = P.a.d, hk = P.a.h_k, sq = ragged ? max_seqlen_q : q_.size(1);
    TORCH_CHECK(q_.size(-1) == d, "q must have the head size of the cache, ", d, ", got ", q_.size(-1));
    TORCH_CHECK(h > 0 && h % hk == 0, "Number of heads in key/value must divide number of heads in query");
    TORCH_CHECK(sq >= 0 && sq * h <= (1 << 30), "max_seqlen_q out of range");
    std::pair<Tensor, Tensor> keep;
    if (k_.has_value() || v_.has_value()) {
        TORCH_CHECK(k_.has_value() && v_.has_value(), "If key is supplied, value must also be passed in");
        TORCH_CHECK(seqlens.has_value(), "If key is supplied, seqlens_k must also be passed in");
        TORCH_CHECK(!ragged, "new keys and values go with a dense query batch: write them with quantize_kvcache first");
        TORCH_CHECK(k_.value().scalar_type() == q_.scalar_type(), "Key must have the same dtype as query");
        keep = set_kv8_new(P, k_.value(), v_.value(), kc, std::nullopt, 0);
    }
    const Tensor q = aligned_rows(q_);
    Tensor out;
    if (out_.has_value()) {
        const Tensor &o = out_.value();
        TORCH_CHECK(o.scalar_type() == q.scalar_type(), "Output must have the same dtype as inputs");
        expect_with(o, "out", kc);
        TORCH_CHECK(o.sizes() == q.sizes(), "out must have the shape of q, ", q.sizes(), ", got ", o.sizes());
        TORCH_CHECK(o.size(-1) <= 1 || o.stride(-1) == 1, "Output tensor must have contiguous last dimension");
        bool fits = ((uintptr_t)o.data_ptr() & 15) == 0;
        for (int64_t i = 0; i + 1 < o.dim(); i++) fits = fits && stride_of(o, i) % 8 == 0;
        // (rows behind the last sequence of a ragged batch stay as they are: they come back with the copy)
        out = fits ? o : ragged ? o.clone(at::MemoryFormat::Contiguous) : torch::empty(q.sizes(), q.options());
    } else {
        out = torch::empty(q.sizes(), q.options());
    }
    auto opts = q.options();
    Tensor lse = torch::empty({b, h, sq}, opts.dtype(at::kFloat));
    if (q.numel() == 0 || sq == 0) {
        // no query: the new tokens still enter the cache
        if (k_.has_value() && keep.first.numel() > 0) { P.a.stream = current_stream(); run(vfa_kv8_quantize(&P)); }
        return {out_.has_value() ? out_.value() : out, lse};
    }
    P.a.dtype = dt;
    P.a.q = q.data_ptr(); P.a.out = out.data_ptr(); P.a.softmax_lse = lse.data_ptr<float>();
    P.a.q_row_stride = stride_of(q, -3); P.a.q_head_stride = stride_of(q, -2);
    P.a.o_row_stride = stride_of(out, -3); P.a.o_head_stride = stride_of(out, -2);
    P.a.h = (int)h; P.a.seqlen_q = (int)sq;
    if (ragged) {
        expect_int32(cu_seqlens_q.value(), "cu_seqlens_q", kc);
        P.a.cu_seqlens_q = cu_seqlens_q.value().data_ptr<int32_t>();
        P.a.total_q = (int)q.size(0);
    } else {
        P.a.q_batch_stride = stride_of(q, 0); P.a.o_batch_stride = stride_of(out, 0);
    }
    if (keep.first.defined() && keep.first.numel() == 0) P.a.knew = P.a.vnew = nullptr;
    P.a.softmax_scale = (float)softmax_scale;
    P.a.is_causal = is_causal;
    P.a.window_size_left = (int)std::clamp<int64_t>(window_size_left, -1, 1 << 30);
    P.a.window_size_right = (int)std::clamp<int64_t>(window_size_right, -1, 1 << 30);
    if (alibi_slopes.has_value()) expect_with(alibi_slopes.value(), "alibi_slopes", kc);
    set_alibi(P.a, alibi_slopes, b, h);
    TORCH_CHECK(num_splits <= 128, "num_splits > 128 not supported");
    P.a.num_splits = (int)std::max<int64_t>(num_splits, 0);
    Tensor work;
    P.workspace_bytes = vfa_kv8_workspace(&P);
    if (P.workspace_bytes > 0) {
        work = torch::empty({(int64_t)P.workspace_bytes}, opts.dtype(at::kByte));
        P.workspace = work.data_ptr();
    }
    P.a.stream = current_stream();
    run(vfa_kv8_mha_fwd(&P));
    if (out_.has_value() && out.data_ptr() != out_.value().data_ptr()) {
        out_.value().copy_(out);
        out = out_.value();
    }
    return {out, lse};
}

struct QKNormHeld { std::vector<Tensor> t; };

void set_qk_norm(vfa_qk_norm_rotary_params &P, QKNormHeld &held, const Tensor &q_, const Tensor &k_, const Tensor &wq, const Tensor &wk,
                 const Tensor &cos, const Tensor &sin, const OptTensor &positions, double eps, bool interleaved) {
    P.dtype = dtype_code(q_);
    TORCH_CHECK(k_.scalar_type() == q_.scalar_type(), "q and k must have the same dtype");
    expect_gpu(q_, "q");
    expect_with(k_, "k", q_);
    TORCH_CHECK(q_.dim() == 4 && k_.dim() == 4 && q_.size(0) == k_.size(0) && q_.size(1) == k_.size(1) && q_.size(3) == k_.size(3),
                "q and k must have the same tokens and head size, got ", q_.sizes(), " and ", k_.sizes());
    const int64_t b = q_.size(0), s = q_.size(1), h = q_.size(2), hk = k_.size(2), d = q_.size(3);
    TORCH_CHECK(h > 0 && hk > 0, "q and k must have heads");
    TORCH_CHECK(d > 0 && d <= 256 && d % 8 == 0, "qk_norm_rotary: head dimension must be a multiple of 8, at most 256");
    TORCH_CHECK(b <= (1 << 30) && s <= (1 << 30) && h <= (1 << 20) && hk <= (1 << 20), "qk_norm_rotary: too large");
    for (const Tensor *w : {&wq, &wk}) {
        expect_with(*w, "weight", q_);
        TORCH_CHECK(w->scalar_type() == q_.scalar_type() || w->scalar_type() == at::kFloat, "q_weight and k_weight must have the dtype of q or fp32");
        TORCH_CHECK(w->scalar_type() == wq.scalar_type(), "q_weight and k_weight must have the same dtype");
        expect_shape(*w, "q_weight / k_weight", {d});
        expect_contig(*w, "q_weight / k_weight");
    }
    TORCH_CHECK(cos.dim() == 2, "rotary_cos must be 2-dimensional");
    for (const Tensor *c : {&cos, &sin}) {
        expect_with(*c, "rotary_cos / rotary_sin", q_);
        TORCH_CHECK(c->scalar_type() == q_.scalar_type() || c->scalar_type() == at::kFloat, "rotary_cos and rotary_sin must have the dtype of q or fp32");
        TORCH_CHECK(c->scalar_type() == cos.scalar_type(), "rotary_cos and rotary_sin must have the same dtype");
        expect_shape(*c, "rotary_cos / rotary_sin", {cos.size(0), cos.size(1)});
        expect_contig(*c, "rotary_cos / rotary_sin");
    }
    const int64_t rd = 2 * cos.size(1);
    TORCH_CHECK(cos.size(0) > 0 && cos.size(0) <= (1 << 30), "rotary_cos must have rows");
    TORCH_CHECK(rd > 0 && rd % 16 == 0, "Only rotary dimensions divisible by 16 are currently supported");
    TORCH_CHECK(rd <= d, "rotary_dim must be <= headdim");
    if (positions.has_value()) {
        const Tensor &p = positions.value();
        TORCH_CHECK(p.scalar_type() == at::kInt, "positions must have dtype int32");
        expect_with(p, "positions", q_);
        expect_shape(p, "positions", {b, s});
        TORCH_CHECK(s <= 1 || p.stride(1) == 1, "positions must have contiguous last dimension");
        P.positions = p.data_ptr<int32_t>();
        P.positions_batch_stride = stride_of(p, 0);
    } else {
        TORCH_CHECK(s <= cos.size(0), "cos/sin seqlen must be at least the seqlen of q");
    }
    P.weight_fp32 = wq.scalar_type() == at::kFloat;
    P.table_fp32 = cos.scalar_type() == at::kFloat;
    P.b = (int)b; P.s = (int)s; P.h = (int)h; P.h_k = (int)hk; P.d = (int)d;
    const Tensor q = aligned_rows(q_), k = aligned_rows(k_);
    held.t.push_back(q); held.t.push_back(k);
    P.q = q.data_ptr(); P.k = k.data_ptr();
    P.q_batch_stride = stride_of(q, 0); P.q_row_stride = stride_of(q, 1); P.q_head_stride = stride_of(q, 2);
    P.k_batch_stride = stride_of(k, 0); P.k_row_stride = stride_of(k, 1); P.k_head_stride = stride_of(k, 2);
    const void *aligned[4];
    int n = 0;
    for (const Tensor *t : {&wq, &wk, &cos, &sin}) {   // (contiguous; a view can still start off a 16-byte boundary)
        held.t.push_back(((uintptr_t)t->data_ptr() & 15) == 0 ? *t : t->clone());
        aligned[n++] = held.t.back().data_ptr();
    }
    P.q_weight = aligned[0]; P.k_weight = aligned[1];
    P.rotary_cos = aligned[2]; P.rotary_sin = aligned[3];
    P.table_rows = (int)cos.size(0); P.rotary_dim = (int)rd; P.is_rotary_interleaved = interleaved;
    P.eps = (float)eps;
}

void set_qk_out(vfa_qk_norm_rotary_params &P, const Tensor &q, const Tensor &k) {   // contiguous (b, s, heads, d)
    P.q_out = q.defined() ? q.data_ptr() : nullptr;
    P.k_out = k.defined() ? k.data_ptr() : nullptr;
    const int64_t s = P.s, d = P.d;
    P.qo_batch_stride = s * P.h * d; P.qo_row_stride = P.h * d; P.qo_head_stride = d;
    P.ko_batch_stride = s * P.h_k * d; P.ko_row_stride = P.h_k * d; P.ko_head_stride = d;
}

std::vector<Tensor> qk_norm_rotary_fwd(const Tensor &q, const Tensor &k, const Tensor &wq, const Tensor &wk, const Tensor &cos,
                                       const Tensor &sin, const OptTensor &positions, double eps, bool interleaved) {
    vfa_qk_norm_rotary_params P{};
    QKNormHeld held;
    expect_gpu(q, "q");
    at::hip::HIPGuardMasqueradingAsCUDA device_guard{(c10::DeviceIndex)q.get_device()};
    set_qk_norm(P, held, q, k, wq, wk, cos, sin, positions, eps, interleaved);
    Tensor qo = torch::empty(q.sizes(), q.options()), ko = torch::empty(k.sizes(), k.options());
    if (q.size(0) * q.size(1) == 0) return {qo, ko};
    set_qk_out(P, qo, ko);
    P.stream = current_stream();
    run(vfa_qk_norm_rotary_fwd(&P));
    return {qo, ko};
}

std::vector<Tensor> qk_norm_rotary_bwd(const Tensor &dqo_, const Tensor &dko_, const Tensor &q, const Tensor &k, const Tensor &wq,
                                       const Tensor &wk, const Tensor &cos, const Tensor &sin, const OptTensor &positions, double eps,
                                       bool interleaved, bool need_q, bool need_k, bool need_wq, bool need_wk) {
    vfa_qk_norm_rotary_params P{};
    QKNormHeld held;
    expect_gpu(q, "q");
    at::hip::HIPGuardMasqueradingAsCUDA device_guard{(c10::DeviceIndex)q.get_device()};
    set_qk_norm(P, held, q, k, wq, wk, cos, sin, positions, eps, interleaved);
    expect_with(dqo_, "dq_out", q);
    expect_with(dko_, "dk_out", q);
    TORCH_CHECK(dqo_.sizes() == q.sizes() && dko_.sizes() == k.sizes(), "gradients must have the shapes of the outputs");
    TORCH_CHECK(dqo_.scalar_type() == q.scalar_type() && dko_.scalar_type() == q.scalar_type(), "gradients must have the dtype of the outputs");
    const Tensor dqo = aligned_rows(dqo_), dko = aligned_rows(dko_);
    P.dq_out = dqo.data_ptr(); P.dk_out = dko.data_ptr();
    P.dqo_batch_stride = stride_of(dqo, 0); P.dqo_row_stride = stride_of(dqo, 1); P.dqo_head_stride = stride_of(dqo, 2);
    P.dko_batch_stride = stride_of(dko, 0); P.dko_row_stride = stride_of(dko, 1); P.dko_head_stride = stride_of(dko, 2);
    Tensor dq, dk, dwq, dwk, work;
    if (need_q) dq = torch::empty(q.sizes(), q.options());
    if (need_k) dk = torch::empty(k.sizes(), k.options());
    if (need_wq) dwq = torch::empty_like(wq);
    if (need_wk) dwk = torch::empty_like(wk);
    set_qk_out(P, dq, dk);
    if (need_wq) P.dq_weight = dwq.data_ptr();
    if (need_wk) P.dk_weight = dwk.data_ptr();
    if (need_wq || need_wk) {
        work = torch::empty({(int64_t)vfa_qk_norm_rotary_bwd_workspace(&P)}, q.options().dtype(at::kFloat));
        P.workspace = work.data_ptr<float>();
    }
    P.stream = current_stream();
    run(vfa_qk_norm_rotary_bwd(&P));
    return {dq, dk, dwq, dwk};
}

// qk_norm_rotary as a node of the autograd graph.  In C++ rather than Python: forward and backward of a short
// sequence are a few microseconds of kernels, and a Python node's backward costs the engine's thread several times
// that (b1 s2731 h12/12 d96: 97 -> 78 us a forward and backward).
struct QKNormRotary : torch::autograd::Function<QKNormRotary> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &wq,
                                                  const Tensor &wk, const Tensor &cos, const Tensor &sin, const OptTensor &positions,
                                                  double eps, bool interleaved) {
        ctx->save_for_backward({q, k, wq, wk, cos, sin, positions.has_value() ? positions.value() : Tensor()});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["interleaved"] = interleaved;
        return qk_norm_rotary_fwd(q, k, wq, wk, cos, sin, positions, eps, interleaved);
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "qk_norm_rotary_func: its gradients have no gradient (create_graph=True)");
        const auto saved = ctx->get_saved_variables();
        const Tensor &q = saved[0], &k = saved[1];
        OptTensor positions;
        if (saved[6].defined()) positions = saved[6];
        // an output that nothing was asked of
        const Tensor dq_out = grads[0].defined() ? grads[0] : torch::zeros_like(q), dk_out = grads[1].defined() ? grads[1] : torch::zeros_like(k);
        auto out = qk_norm_rotary_bwd(dq_out, dk_out, q, k, saved[2], saved[3], saved[4], saved[5], positions,
                                      ctx->saved_data["eps"].toDouble(), ctx->saved_data["interleaved"].toBool(), ctx->needs_input_grad(0),
                                      ctx->needs_input_grad(1), ctx->needs_input_grad(2), ctx->needs_input_grad(3));
        out.resize(9);
        return out;
    }
};

// A node of a graph keeps the stream that it was recorded on (a leaf: that of the first live graph it is part of), and a
// backward pass hands its gradient over to that stream.  The default stream cannot take part in a capture: the backward
// pass would end the process.
void expect_capturable(const Tensor &x) {
    if (!x.requires_grad()) return;
    const auto refuse_default = [](const std::shared_ptr<torch::autograd::Node> &node) {
        const auto stream = node ? node->stream() : std::nullopt;
        TORCH_CHECK(!stream || stream->id() != 0,
                    "qk_norm_rotary_func: a graph recorded on the default stream still holds an input; drop it before capturing a pass with gradients");
    };
    refuse_default(x.grad_fn());
    const Tensor base = x.is_view() ? Tensor(x._base()) : x;   // (a ragged or packed input is a view)
    if (!base.requires_grad()) return;
    refuse_default(base.is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(base) : base.grad_fn());
}

std::vector<Tensor> qk_norm_rotary(const Tensor &q, const Tensor &k, const Tensor &wq, const Tensor &wk, const Tensor &cos, const Tensor &sin,
                                   const OptTensor &positions, double eps, bool interleaved) {
    for (const Tensor *x : {&q, &k, &wq, &wk, &cos, &sin})   // (a tensor with a tangent need not require a gradient)
        TORCH_CHECK(!x->_fw_grad(0).defined(), "qk_norm_rotary_func has no forward-mode derivative");
    // a serving step is a few microseconds: it is not recorded for a backward that cannot come
    if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || wq.requires_grad() || wk.requires_grad())) {
        if (q.is_cuda()) {
            at::hip::HIPGuardMasqueradingAsCUDA device_guard{(c10::DeviceIndex)q.get_device()};
            if (c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None)
                for (const Tensor *x : {&q, &k, &wq, &wk}) expect_capturable(*x);
        }
        return QKNormRotary::apply(q, k, wq, wk, cos, sin, positions, eps, interleaved);
    }
    return qk_norm_rotary_fwd(q, k, wq, wk, cos, sin, positions, eps, interleaved);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.doc() = "FlashAttention (MI355X / gfx950)";
    m.def("fwd", &fwd, "Forward pass");
    // No counterpart in the reference (which accepts fp16 / bf16 CUDA tensors only): a plain host
    // loop for fp32 CPU tensors, forward only, for the one configuration of the benchmark list that
    // runs without a GPU (batch 2, seqlen 128, 4 heads, head dim 64 against torch SDPA).  The Python
    // package routes to it only when asked (vllm_flash_attn.enable_cpu_fp32).
    m.def("fwd_cpu_fp32",
          [](const Tensor &q, const Tensor &k, const Tensor &v, OptTensor out_, OptTensor alibi_slopes_, double p_dropout,
             double softmax_scale, bool is_causal, int64_t wl, int64_t wr) {
              TORCH_CHECK(!q.is_cuda() && q.scalar_type() == at::kFloat, "fwd_cpu_fp32 takes fp32 CPU tensors");
              return fwd_cpu_fp32(q, k, v, out_, alibi_slopes_, p_dropout, softmax_scale, is_causal, wl, wr);
          },
          "Forward pass on fp32 CPU tensors (host loop, forward only)");
    m.def("varlen_fwd", &varlen_fwd, "Forward pass (variable length)");
    m.def("bwd", &bwd, "Backward pass");
    m.def("varlen_bwd", &varlen_bwd, "Backward pass (variable length)");
    m.def("fwd_kvcache", &fwd_kvcache, "Forward pass, with KV-cache");
    // No counterpart in the reference: a KV cache in 8 bits, and the norm and rotation of q and k heads.
    m.def("kv8_quantize", &kv8_quantize, "Write tokens to an 8-bit KV cache");
    m.def("kv8_dequantize", [](const Tensor &kc, const Tensor &vc, const Tensor &ks, const Tensor &vs, const Tensor &seqlens,
                               const OptTensor &cache_batch_idx, const OptTensor &block_table, const OptTensor &cu_seqlens, int64_t rows,
                               const py::object &dtype) {
        return kv8_dequantize(kc, vc, ks, vs, seqlens, cache_batch_idx, block_table, cu_seqlens, rows,
                              torch::python::detail::py_object_to_dtype(dtype));
    }, "Read an 8-bit KV cache in 16 bits");
    m.def("fwd_kv8", &fwd_kv8, "Forward pass, with an 8-bit KV cache");
    m.def("qk_norm_rotary", &qk_norm_rotary, "RMS norm and rotation of query and key heads, differentiable");
}
