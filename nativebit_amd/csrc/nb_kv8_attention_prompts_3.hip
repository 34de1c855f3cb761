// nb_kv8_attention's kernel with 3 digits, for steps of prompts too.
#include "nb_kv8_attention.h"

namespace nb {

void launch_kv8_prompts_3(const Kv8AttentionArgs& a, dim3 grid, bool rules, hipStream_t stream) {
    launch_kv8_digits<3, true>(a, grid, rules, stream);
}

}  // namespace nb
