// nb_kv8_attention's kernel with 2 digits, for steps of single tokens.
#include "nb_kv8_attention.h"

namespace nb {

void launch_kv8_tokens_2(const Kv8AttentionArgs& a, dim3 grid, bool rules, hipStream_t stream) {
    launch_kv8_digits<2, false>(a, grid, rules, stream);
}

}  // namespace nb
