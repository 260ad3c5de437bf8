"""CPU tests: lengths past 2^30 are refused by the C ABI of the 8-bit KV cache, whose kernels add two of them in 32 bits."""
import ctypes

import pytest

import cabi_kv8


@pytest.mark.parametrize("entry", ["vfa_kv8_quantize", "vfa_kv8_dequantize", "vfa_kv8_mha_fwd"])
@pytest.mark.parametrize("over", [dict(seqlen_k=2 ** 30 + 64), dict(block_table=4096, page_block_size=64, seqlen_k=2 ** 30 + 64),
                                  dict(knew=4096, vnew=4096, seqlen_knew=2 ** 30 + 1)], ids=str)
def test_more_than_2_to_the_30_tokens(entry, over):
    lib = cabi_kv8.lib()
    P = cabi_kv8.kv8(**over)
    assert getattr(lib, entry)(ctypes.byref(P)) == -1
    assert b"2^30 tokens" in lib.vfa_last_error()
    assert lib.vfa_kv8_workspace(ctypes.byref(P)) == 0
