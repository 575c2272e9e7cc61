// What a call of the attention over the 4-bit cache consists of.
#pragma once

#include "kv_cache.hpp"

namespace uniql {

struct KvAttentionArgs {
    const half_t* q;        // [rows][heads][k_dim]
    int64_t q_row, q_head;  // elements between rows and heads
    KvCache cache;
    const int32_t *table, *lengths, *cu_q;
    half_t* out;            // [rows][heads][v_dim]
    int64_t out_row, out_head;
    void* accum;
    float* temp;
    int rows, requests, columns, group;  // group: query heads of a key / value head
    int shares;                          // runs of positions that a head's work is shared out to
    float scale;
    int group_shift;                     // for quotients by `group`, set by the launch, as `shares` is
    unsigned group_factor;
};

}  // namespace uniql
