// What a call of the attention over whole prompts consists of.
#pragma once

#include "common.hpp"

namespace uniql {

struct PromptArgs {
    const half_t *q, *k, *v;  // [rows][heads][k_dim], [k_rows][heads / group][k_dim], [k_rows][heads / group][v_dim]
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head;
    const int32_t *cu_q, *cu_k;
    half_t* out;
    int rows, k_rows, sequences, heads, group, k_dim, v_dim, causal;
    float scale;
    // set by the launch: the scale's sign, blocks of rows in all sequences at most, factor and shift for quotients by `group`
    int q_sign, blocks, group_shift;
    unsigned group_factor;
};

}  // namespace uniql
