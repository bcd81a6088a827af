#include "kv_attention_kernels.hpp"

void icx::launch_attention_bf16(int bits, unsigned few, unsigned many, hipStream_t s, const AttnArgs& a) {
    if (bits == 4) launch_bits<4, 1, __bf16>(few, many, s, a);
    else launch_bits<8, 1, __bf16>(few, many, s, a);
}
