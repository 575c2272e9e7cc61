// The layout of the paged 4-bit key / value cache.
#pragma once

#include "common.hpp"

namespace uniql {

// eight fp16 values at any address that holds fp16 values: the hardware takes a 16-byte access at any alignment
typedef _Float16 h8u __attribute__((ext_vector_type(8), aligned(2)));

// Eight values of a vector from column j on; those past the vector's width count as zeros.
__device__ __forceinline__ h8 load_eight_of(const half_t* x, int j, int width) {
    if (j + 8 <= width) {
        const h8u v = *reinterpret_cast<const h8u*>(x + j);
        return h8{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]};
    }
    h8 v = {};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (j + i < width) v[i] = x[j + i];
    return v;
}

// bit position of value i of eight in a word: the order of the embedding's words, in which the pairs (0, 1), (2, 3), (4, 5),
// (6, 7) lie 16 bits apart and come out with a mask and at most one shift each
__device__ __host__ constexpr int kNibble(int i) { return 4 * (i >> 1) + 16 * (i & 1); }

// Keys: a token's words lie together, [page][head][token][words]: 16 tokens x 4 S words are contiguous, and a lane of a matrix
// instruction that takes 32 channels at a time reads the S words of its token in one access.
// Values: [page][head][token / 4][word][token % 4]: a lane of the second product holds one group of eight channels for four and
// four tokens, which is one 16-byte access each, while every word still belongs to one token, so that tokens are written without
// touching each other's.
// Scales: [page][head][token].
struct KvCache {
    uint32_t *k_codes, *v_codes;
    half_t *k_scales, *v_scales;
    int pages, page_shift, heads;
    int k_dim, v_dim, k_words, v_words;  // words of eight values, multiples of four

    __device__ __forceinline__ int64_t scale_at(int64_t slot, int head) const {
        const int64_t page = slot >> page_shift;
        return ((page * heads + head) << page_shift) + (slot & ((1 << page_shift) - 1));
    }
    __device__ __forceinline__ int64_t k_word(int64_t slot, int head, int word) const { return scale_at(slot, head) * k_words + word; }
    __device__ __forceinline__ int64_t v_word(int64_t slot, int head, int word) const {
        const int64_t at = scale_at(slot, head);
        return (at & ~(int64_t)3) * v_words + 4 * word + (at & 3);
    }
};

}  // namespace uniql
