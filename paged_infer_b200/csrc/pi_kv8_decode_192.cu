// Decode attention over the 8-bit cache: the instantiations of these pitches.
#include "pi_kv8_decode.cuh"

namespace pi_kv8 {
template pi_status launch_decode_pitch<192>(pi_ctx*, int, int, int, const pi_kv8_attn_params&, dim3, int, int);
}  // namespace pi_kv8
