// nb_kv8_attention's kernel with 3 digits (see nb_kv8_attention.h).
#include "nb_kv8_attention.h"

namespace nb {

void launch_kv8_attention_3(const Kv8AttentionArgs& a, dim3 grid, bool rules, hipStream_t stream) {
    launch_kv8_digits<3>(a, grid, rules, stream);
}

}  // namespace nb
