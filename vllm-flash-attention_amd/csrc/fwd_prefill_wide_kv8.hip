// The forward kernel for head dims above 128 (fwd_prefill_wide.hip) over an 8-bit KV cache read back into 16 bits: a
// translation unit of its own, built without packed fp32 instructions as all that the 8-bit cache's operators launch, and
// with zeros for a row that sees no key.
#define VFA_KV8_TU 1
#define fwd_prefill_wide_kernel kv8_prefill_wide_kernel
#include "fwd_prefill_wide.hip"
