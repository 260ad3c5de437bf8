// The instantiations of fwd_prefill_kv8.hip over the cache read back into 16-bit rows, a translation unit of their own: the
// two halves compile side by side.
#define VFA_KV8_ROWS_TU 1
#include "fwd_prefill_kv8.hip"
