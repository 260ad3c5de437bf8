"""CPU tests of the refusals of the 8-bit KV cache and q / k norm entry points: the C ABI's argument checks run before
any HIP call, the Python functions' and the extension's before any launch."""
import ctypes

import pytest
import torch

import cabi_kv8
import vllm_flash_attn as fa


def test_struct_mirrors_match():
    lib = cabi_kv8.lib()
    assert lib.vfa_kv8_params_sizeof() == ctypes.sizeof(cabi_kv8.VfaKv8Params)
    assert lib.vfa_qk_norm_rotary_params_sizeof() == ctypes.sizeof(cabi_kv8.VfaQkNormRotaryParams)


CACHE = [
    (dict(dtype=7), b"only support fp16 and bf16"),
    (dict(k=0), b"null cache or scale pointer"),
    (dict(k_scale=0), b"null cache or scale pointer"),
    (dict(b=0), b"batch size must be postive"),
    (dict(d=72), b"multiple of 16"),
    (dict(d=272), b"at most 256"),
    (dict(num_pages=0), b"empty cache"),
    (dict(seqlen_k=0), b"empty cache"),
    (dict(scale_block=24), b"multiple of 16 that divides"),
    (dict(scale_block=48), b"multiple of 16 that divides"),
    (dict(b=3), b"batch size exceeds the cache's"),
    (dict(k=4100), b"16-byte aligned"),
    (dict(v_row_stride=264), b"16-byte aligned"),
    (dict(k_row_stride=1 << 30), b"row strides must be under"),
    (dict(block_table=4096, cache_batch_idx=4096, page_block_size=64), b"does not support cache_batch_idx"),
    (dict(knew=4096), b"value must also be passed in"),
    (dict(knew=4096, vnew=4100), b"must be 16-byte aligned"),
    (dict(knew=4096, vnew=4096, seqlen_knew=-1), b"negative number of new tokens"),
]


@pytest.mark.parametrize("over,message", CACHE, ids=[str(c[0]) for c in CACHE])
@pytest.mark.parametrize("entry", ["vfa_kv8_quantize", "vfa_kv8_dequantize", "vfa_kv8_mha_fwd"])
def test_cache_arguments(entry, over, message):
    lib = cabi_kv8.lib()
    P = cabi_kv8.kv8(**over)
    assert getattr(lib, entry)(ctypes.byref(P)) == -1
    assert message in lib.vfa_last_error()
    assert getattr(lib, entry)(None) == -1


ATTENTION = [
    (dict(h=7), b"must divide number of heads in query"),
    (dict(num_splits=129), b"num_splits > 128"),
    (dict(q=0), b"null tensor pointer"),
    (dict(softmax_lse=0), b"null tensor pointer"),
    (dict(softmax_scale=0.0), b"softmax_scale must be positive"),
    (dict(softmax_scale=-1.0), b"softmax_scale must be positive"),
    (dict(p_dropout=0.1), b"no dropout"),
    (dict(q=4104), b"16-byte aligned"),
    (dict(o_row_stride=12), b"strides multiples of 8"),
    (dict(knew=4096, vnew=4096, seqlen_knew=1, cu_seqlens_q=4096), b"dense query batch"),
    (dict(seqlen_q=-1), b"negative size"),
]


@pytest.mark.parametrize("over,message", ATTENTION, ids=[str(c[0]) for c in ATTENTION])
def test_attention_arguments(over, message):
    lib = cabi_kv8.lib()
    P = cabi_kv8.kv8(**over)
    assert lib.vfa_kv8_mha_fwd(ctypes.byref(P)) == -1
    assert message in lib.vfa_last_error()


def test_workspace_plan():
    """Enough for the partial results of what the launch can do; none where one workgroup per item fills the chip."""
    lib = cabi_kv8.lib()
    size = lambda **kw: lib.vfa_kv8_workspace(ctypes.byref(cabi_kv8.kv8(**kw)))
    assert size(cu_seqlens_k=4096, b=1, seqlen_k=65536, num_pages=1) >= 128 * 8 * 129 * 4
    assert size(num_splits=1) == 0
    assert size(b=512, num_pages=512, h_k=8) == 0
    assert size(num_splits=3, seqlen_k=65536) >= 3 * 2 * 8 * 129 * 4
    assert size(seqlen_k=64) == 0                              # nothing to cut
    # long queries: the cache in 16 bits, K and V
    assert size(seqlen_q=512) >= 2 * 1024 * 2 * 128 * 2 * 2
    assert size(h=7) == 0 and b"must divide" in lib.vfa_last_error()


QK = [
    (dict(dtype=3), b"only supports fp16 and bf16"),
    (dict(d=100), b"multiple of 8"),
    (dict(d=264, rotary_dim=64), b"at most 256"),
    (dict(h=0), b"no heads"),
    (dict(b=-1), b"negative size"),
    (dict(rotary_dim=24), b"divisible by 16"),
    (dict(rotary_dim=0), b"divisible by 16"),
    (dict(rotary_dim=144), b"rotary_dim must be <= headdim"),
    (dict(rotary_cos=0), b"rotary tables are required"),
    (dict(s=17), b"at least the seqlen of q"),
    (dict(q_weight=0), b"null weight pointer"),
    (dict(k_weight=4100), b"weights and tables must be 16-byte aligned"),
    (dict(k=0), b"null tensor pointer"),
    (dict(q=4100), b"16-byte aligned"),
    (dict(k_head_stride=4), b"strides multiples of 8"),
]


@pytest.mark.parametrize("over,message", QK, ids=[str(c[0]) for c in QK])
@pytest.mark.parametrize("entry", ["vfa_qk_norm_rotary_fwd", "vfa_qk_norm_rotary_bwd"])
def test_qk_norm_arguments(entry, over, message):
    lib = cabi_kv8.lib()
    P = cabi_kv8.qk(**over)
    assert getattr(lib, entry)(ctypes.byref(P)) == -1
    assert message in lib.vfa_last_error()
    assert getattr(lib, entry)(None) == -1


def test_qk_norm_backward_needs_its_workspace_for_the_weights():
    lib = cabi_kv8.lib()
    P = cabi_kv8.qk(dq_weight=4096)
    assert lib.vfa_qk_norm_rotary_bwd(ctypes.byref(P)) == -1 and b"workspace" in lib.vfa_last_error()
    P = cabi_kv8.qk(dq_out=0)
    assert lib.vfa_qk_norm_rotary_bwd(ctypes.byref(P)) == -1 and b"null gradient" in lib.vfa_last_error()
    assert lib.vfa_qk_norm_rotary_bwd_workspace(ctypes.byref(cabi_kv8.qk())) >= 2 * 128


def test_cpu_tensors_and_wrong_combinations_are_refused():
    cache = [torch.zeros(2, 64, 1, 64).to(torch.float8_e4m3fn) for _ in range(2)] + [torch.zeros(2, 4, 1, dtype=torch.float8_e8m0fnu) for _ in range(2)]
    lens = torch.zeros(2, dtype=torch.int32)
    x = torch.zeros(2, 1, 1, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="must be on CUDA"):
        fa.quantize_kvcache(x, x, *cache, lens)
    with pytest.raises(RuntimeError, match="must be on CUDA"):
        fa.dequantize_kvcache(*cache, lens, max_seqlen=4)
    with pytest.raises(RuntimeError, match="must be on CUDA"):
        fa.flash_attn_with_quantized_kvcache(x, *cache, cache_seqlens=lens)
    w, c = torch.ones(64), torch.zeros(4, 16)
    with pytest.raises(RuntimeError, match="must be on CUDA"):
        fa.qk_norm_rotary_func(x, x, w, w, c, c)
    with pytest.raises(RuntimeError, match="float8_e4m3fn"):
        fa.quantize_kvcache(x, x, cache[0].float(), cache[1], *cache[2:], lens)
    with pytest.raises(ValueError, match="max_seqlen is required"):
        fa.quantize_kvcache(x[0], x[0], *cache, lens, cu_seqlens=lens)
    with pytest.raises(ValueError, match="goes with cu_seqlens"):
        fa.quantize_kvcache(x, x, *cache, lens, max_seqlen=3)
    for kw in ({}, dict(max_seqlen=3, cu_seqlens=lens, total_seqlen=4), dict(cu_seqlens=lens), dict(max_seqlen=3, total_seqlen=3)):
        with pytest.raises(ValueError, match="either max_seqlen"):
            fa.dequantize_kvcache(*cache, lens, **kw)
    with pytest.raises(ValueError, match="go together"):
        fa.flash_attn_with_quantized_kvcache(x, *cache, cu_seqlens_q=lens)
    with pytest.raises(ValueError, match="positions are required"):
        fa.qk_norm_rotary_func(x[0], x[0], w, w, c, c)
    with pytest.raises(ValueError, match="no gradient"):
        fa.qk_norm_rotary_func(x, x, w, w, c.clone().requires_grad_(), c)
