// The forward prefill kernel over an 8-bit KV cache (template instantiations of fwd_prefill.hip; see
// run_fwd_kv8_prefill there), compiled as their own translation unit.
#define VFA_DROPOUT_TU 1
#define VFA_KV8_TU 1
#include "fwd_prefill.hip"
