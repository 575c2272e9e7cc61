// Causal attention over the prompts of several sequences that lie behind each other: o = sum_j p_j v_j / sum_j p_j,
// p_j = exp(scale q . k_j - m), row i of a sequence with t queries and n keys over the keys j <= i + n - t.
//
// A workgroup takes 32 rows of a head for each of its waves and goes through the keys 64 at a time, in LDS, the next 64 on their way
// meanwhile (two buffers, straight from memory to LDS).  Matrix instructions of 32 x 32 x 16: the scores come transposed, keys along
// the rows, K q^T, because a lane then holds scores of one query and of just those keys that the second product, V^T P^T, wants
// from it: the weights never leave its registers.  That product takes V transposed, four keys of one channel at a time, which the
// transposing LDS read gives.  Rows of K and V lie in LDS with their 16-byte pieces exchanged by the row's number, so that neither
// kind of read meets itself in a bank.
// The maximum follows the scores only when a weight would pass 2^8 (weights are fp16, sums and outputs fp32): mostly once.
// The rounding of the weights to fp16 (2^-11) is what a matrix instruction on fp16 asks for; their sum takes the rounded ones.
#include "prompt_attention.hpp"

namespace uniql {

constexpr int kKeys = 64;               // keys of a step
constexpr int kQueries = 32;            // rows of a wave
constexpr float kLowest = -3.0e38f;
constexpr float kRoom = 8.0f;           // weights may grow to 2^8 before the maximum follows
typedef __attribute__((address_space(3))) void* lds_ptr;
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s4* lds_s4_ptr;
typedef _Float16 h4u __attribute__((ext_vector_type(4), aligned(2)));

#define UNIQL_WAIT_ALL_LOADS() __builtin_amdgcn_s_waitcnt(0x0F70)  // vmcnt(0), the other counters left alone (gfx9 encoding)

__device__ __forceinline__ int clamp_to(int v, int low, int high) { return v < low ? low : (v > high ? high : v); }

struct Rows {
    int q_first, q_count, k_first, k_count;
};
__device__ __forceinline__ Rows rows_of(const PromptArgs& a, int s) {
    Rows r;
    r.q_first = clamp_to(a.cu_q[s], 0, a.rows);
    r.q_count = clamp_to(a.cu_q[s + 1], r.q_first, a.rows) - r.q_first;
    r.k_first = clamp_to(a.cu_k[s], 0, a.k_rows);
    r.k_count = clamp_to(a.cu_k[s + 1], r.k_first, a.k_rows) - r.k_first;
    return r;
}
// The sequence and the block of rows in it that block `index` of all is; every wave finds it for itself.
__device__ __forceinline__ bool find_block(const PromptArgs& a, int index, int block_rows, int& sequence, int& block) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base < a.sequences; base += 64) {
        const int s = base + lane;
        int mine = 0;
        if (s < a.sequences) mine = (rows_of(a, s).q_count + block_rows - 1) / block_rows;
        int upto = mine;
        for (int d = 1; d < 64; d <<= 1) {
            const int other = __shfl_up(upto, d, 64);
            if (lane >= d) upto += other;
        }
        const unsigned long long above = __ballot(before + upto > index);
        if (above) {
            const int owner = __builtin_ctzll(above);
            sequence = __builtin_amdgcn_readfirstlane(base + owner);
            block = __builtin_amdgcn_readfirstlane(index - before - __shfl(upto - mine, owner, 64));
            return true;
        }
        before += __shfl(upto, 63, 64);
    }
    return false;
}

// Eight values of a row from column j on; those past its width count as zeros.
__device__ __forceinline__ h8 row_piece(const half_t* x, int j, int width) {
    typedef _Float16 h8u __attribute__((ext_vector_type(8), aligned(2)));
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

// D: the wider of the two head widths in units of 32, 2 to 4.  PIECES: rows of 16-byte pieces at multiples of 16 bytes, which go to LDS by
// themselves; otherwise they pass through registers.
template <int D, int WAVES, bool PIECES>
__global__ __launch_bounds__(64 * WAVES, WAVES == 8 ? 1 : 2) void prompt_attention_kernel(const PromptArgs a) {
    constexpr int kSteps = 2 * D;                      // of 16 channels, of the first product
    constexpr int kPieces = D == 2 ? 8 : 16;           // 16-byte pieces of a row in LDS
    constexpr int kRowBytes = kPieces * 16;
    constexpr int kTileBytes = kKeys * kRowBytes;
    constexpr int kRowsAtOnce = 64 / kPieces;          // rows that a wave's access covers
    constexpr int kAccesses = kKeys / (kRowsAtOnce * WAVES);
    // Two K tiles and two V tiles: variables of their own, which tells the compiler that reading one does not wait for what is on its way
    // into another.
    __shared__ __attribute__((aligned(16))) char k_even[kTileBytes], k_odd[kTileBytes], v_even[kTileBytes], v_odd[kTileBytes];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5, col = lane & 31;
    // neighbouring workgroups have different key / value heads: those of one head stay on an XCD and share its L2
    const unsigned kv_heads = (unsigned)(a.heads / a.group), kv_head = blockIdx.x % kv_heads, rest = blockIdx.x / kv_heads;
    const int head = (int)(kv_head * a.group + rest % a.group);
    // later blocks see more keys: they come first
    int sequence, block;
    if (!find_block(a, (int)(a.blocks - 1 - rest / a.group), kQueries * WAVES, sequence, block)) return;
    const Rows r = rows_of(a, sequence);
    const int offset = r.k_count - r.q_count;
    const int row0 = block * kQueries * WAVES + wave * kQueries, row = row0 + col;
    const bool row_exists = row < r.q_count;
    const int seen = a.causal ? clamp_to(row + offset + 1, 0, r.k_count) : r.k_count;  // keys of the lane's row
    // of the wave's first row and of its last, and of the workgroup's last
    const int last_row = clamp_to(row0 + kQueries - 1, 0, r.q_count - 1), block_last = clamp_to((block + 1) * kQueries * WAVES - 1, 0, r.q_count - 1);
    const int fewest = a.causal ? clamp_to(row0 + offset + 1, 0, r.k_count) : r.k_count;
    const int most = row0 < r.q_count ? (a.causal ? clamp_to(last_row + offset + 1, 0, r.k_count) : r.k_count) : 0;
    const int block_most = a.causal ? clamp_to(block_last + offset + 1, 0, r.k_count) : r.k_count;
    const int block_fewest = a.causal ? clamp_to(block * kQueries * WAVES + offset + 1, 0, r.k_count) : r.k_count;
    const int tiles = (block_most + kKeys - 1) / kKeys;

    h8 q[kSteps];
    {
        const half_t* from = a.q + (int64_t)(r.q_first + (row_exists ? row : 0)) * a.q_row + (int64_t)head * a.q_head;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            q[i] = h8{};
            if (row_exists && a.q_sign != 0) q[i] = row_piece(from, 16 * i + 8 * half, a.k_dim);
            if (a.q_sign < 0) q[i] = -q[i];
        }
    }
    f16 out[D];
#pragma unroll
    for (int i = 0; i < D; ++i) out[i] = f16{};
    float m = kLowest, l = 0.f;
    const float unit = a.scale * 1.4426950408889634f;  // positive: a negative scale has turned q

    const half_t* const k_base = a.k + (int64_t)r.k_first * a.k_row + (int64_t)kv_head * a.k_head;
    const half_t* const v_base = a.v + (int64_t)r.k_first * a.v_row + (int64_t)kv_head * a.v_head;
    // this lane's part of an access: a row of the tile and a piece of it
    const int part_row = wave * kRowsAtOnce + lane / kPieces, part = lane % kPieces;
    const int k_piece = part ^ (part_row & (kPieces - 1)), v_piece = part ^ (2 * (part_row & 3));
    // Rows behind the sequence lie beyond the descriptor and come as zeros, and so do pieces behind the width.
    auto fetch = [&](const half_t* base, int64_t stride, int width, int piece, int tile, char* to) __attribute__((always_inline)) {
        const int key0 = tile * kKeys, left = r.k_count - key0 < kKeys ? r.k_count - key0 : kKeys;
        if constexpr (PIECES) {
            const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<half_t*>(base + (int64_t)key0 * stride), 0,
                                                                                  (unsigned)(((int64_t)(left - 1) * stride + width) * 2), 0x00020000);
#pragma unroll
            for (int i = 0; i < kAccesses; ++i) {
                const int at = i * kRowsAtOnce * WAVES;  // a multiple of 16 rows: the exchange of pieces is the same
                const unsigned off = piece * 8 < width ? 2u * ((unsigned)(at + part_row) * (unsigned)stride) + 16u * piece : 0xfffffff0u;
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr)(to + (at + wave * kRowsAtOnce) * kRowBytes), 16, off, 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kAccesses; ++i) {
                const int at = i * kRowsAtOnce * WAVES + part_row;
                h8 v = {};
                if (at < left) v = row_piece(base + (int64_t)(key0 + at) * stride, 8 * piece, width);
                *reinterpret_cast<h8*>(to + at * kRowBytes + part * 16) = v;
            }
        }
    };
    auto fetch_k = [&](int tile, char* to) __attribute__((always_inline)) { fetch(k_base, a.k_row, a.k_dim, k_piece, tile, to); };
    auto fetch_v = [&](int tile, char* to) __attribute__((always_inline)) { fetch(v_base, a.v_row, a.v_dim, v_piece, tile, to); };
    // where the lane reads: K rows col and 32 + col, piece 2 step + half; V rows 4 half + j (+ 8), j = (lane / 4) % 4, four channels
    const int k_read = col * kRowBytes, k_swap = col & (kPieces - 1);
    const int v_j = (lane >> 2) & 3, v_read = (4 * half + v_j) * kRowBytes + (lane & 1) * 8;
    const int v_sub = 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
    auto keys_of = [&](const char* tile, int k, int i) __attribute__((always_inline)) {
        return *reinterpret_cast<const h8*>(tile + k_read + k * 32 * kRowBytes + (((2 * i + half) ^ k_swap) * 16));
    };
    // A step: the weights of tile t from its scores, which the step before has computed, the next tile's scores, the second product.
    auto step = [&](int t, char* k_lds, char* v_lds, char* next_k_lds, char* next_v_lds, f16 (&score)[2], f16 (&next)[2]) __attribute__((always_inline)) {
        const int key0 = t * kKeys;
        UNIQL_WAIT_ALL_LOADS();
        __syncthreads();
        if (t + 2 < tiles) fetch_k(t + 2, k_lds);
        if (t + 1 < tiles) fetch_v(t + 1, next_v_lds);
        const bool masked = key0 + kKeys > fewest;
        // A key that some rows of the tile see and others do not: its weight is zero for those, but zero times an infinity is not.  Keys
        // with such values are found first and taken out of the product, see below; each lane looks at one key.
        unsigned long long odd_keys = 0;
        if (a.causal && key0 + kKeys > block_fewest) {
            uint32_t any = 0;
#pragma unroll 4
            for (int i = 0; i < kPieces; ++i) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(v_lds + lane * kRowBytes + ((i + lane) & (kPieces - 1)) * 16);
#pragma unroll
                for (int j = 0; j < 4; ++j) any |= ((w[j] & 0x7c007c00u) + 0x04000400u) & 0x80008000u;  // an exponent of all ones runs over
            }
            odd_keys = __ballot(any != 0);
        }
        const bool active = key0 < most;  // the wave's rows see some of the keys (all waves take part in the barriers)
        if (active) {
            if (masked) {
                asm volatile("");  // keeps the comparisons out of the other tiles' way
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (key0 + 32 * k + 8 * (i / 4) + 4 * half + i % 4 >= seen) score[k][i] = -INFINITY;
            }
            float top = score[0][0];
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int i = 0; i < 16; ++i) top = fmaxf(top, score[k][i]);
            if (__any(top * unit > m + kRoom)) {
                const float higher = fmaxf(m, fmaxf(top, __shfl_xor(top, 32, 64)) * unit);
                const float fade = __builtin_amdgcn_exp2f(m - higher);
                m = higher;
                l *= fade;
#pragma unroll
                for (int i = 0; i < D; ++i) out[i] *= fade;
            }
        }
        if (odd_keys) {  // the same for all waves
            // one key at a time, in the rows that see it; then zeros take the keys' place in LDS
            if (active) {
                for (unsigned long long left = odd_keys; left; left &= left - 1) {
                    const int key = __builtin_ctzll(left);
                    const int index = 4 * (key >> 3) + (key & 3);  // of the scores, in the half (key >> 2) & 1
                    float value = 0.f;
#pragma unroll
                    for (int i = 0; i < 32; ++i) value = i == index ? score[i >> 4][i & 15] : value;
                    value = __shfl(value, col + 32 * ((key >> 2) & 1), 64);
                    const float p = (float)(half_t)__builtin_amdgcn_exp2f(__builtin_fmaf(value, unit, -m));
                    if (key0 + key < seen && row_exists) {
#pragma unroll
                        for (int i = 0; i < D; ++i)
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                const int channel = 32 * i + 8 * (j / 4) + 4 * half + j % 4;
                                const half_t v = *reinterpret_cast<const half_t*>(v_lds + key * kRowBytes +
                                                                                  ((channel >> 3) ^ (2 * (key & 3))) * 16 + (channel & 7) * 2);
                                out[i][j] += p * (float)v;
                            }
                    }
                }
            }
            __syncthreads();
            if (wave == 0 && ((odd_keys >> lane) & 1))
                for (int i = 0; i < kPieces; ++i) *reinterpret_cast<u32x4*>(v_lds + lane * kRowBytes + i * 16) = u32x4{0u, 0u, 0u, 0u};
            __syncthreads();
        }
        if (!active) return;
        // Slots of one matrix instruction each, closed by scheduling barriers.  First the next tile's scores, operands four slots ahead,
        // beside them this tile's weights, a pair or two a slot; then the second product, operands kAhead slots ahead.
        constexpr int kFirst = 2 * kSteps, kSecond = 4 * D, kAhead = 3;
        h8 keys[4];
        s4 values[kAhead][2];
        auto read_keys = [&](int i) __attribute__((always_inline)) { keys[i & 3] = keys_of(next_k_lds, i & 1, i >> 1); };
        auto read_values = [&](int i) __attribute__((always_inline)) {
            const int piece = ((4 * (i % D) + v_sub) ^ (2 * v_j)) * 16, at = (i / D) * 16;
            values[i % kAhead][0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_ptr)(v_lds + v_read + piece + at * kRowBytes));
            values[i % kAhead][1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_ptr)(v_lds + v_read + piece + (at + 8) * kRowBytes));
        };
        f2 power[2];
        h2 pair[16];
        auto raise = [&](int i) __attribute__((always_inline)) {
            power[i & 1] = f2{__builtin_amdgcn_exp2f(__builtin_fmaf(score[i >> 3][2 * (i & 7)], unit, -m)),
                              __builtin_amdgcn_exp2f(__builtin_fmaf(score[i >> 3][2 * (i & 7) + 1], unit, -m))};
        };
        auto round_pair = [&](int i) __attribute__((always_inline)) {
            pair[i] = __builtin_convertvector(power[i & 1], h2);
            l = __builtin_amdgcn_fdot2(pair[i], h2{(half_t)1.f, (half_t)1.f}, l, false);
        };
        next[0] = next[1] = f16{};
#pragma unroll
        for (int i = 0; i < 4; ++i) read_keys(i);
        __builtin_amdgcn_sched_barrier(0);
        int raised = 0;
#pragma unroll
        for (int i = 0; i < kFirst; ++i) {
            next[i & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(keys[i & 3], q[i >> 1], next[i & 1], 0, 0, 0);
            if (i + 4 < kFirst) read_keys(i + 4);
            else if (i + 4 - kFirst < kAhead) read_values(i + 4 - kFirst);
#pragma unroll
            for (; raised < 16 * (i + 1) / kFirst; ++raised) {
                if (raised > 0) round_pair(raised - 1);
                raise(raised);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        round_pair(15);
#pragma unroll
        for (int i = 0; i < kSecond; ++i) {
            const int s = i / D;
            const s4 lo = values[i % kAhead][0], hi = values[i % kAhead][1];
            const h8 weight = {pair[4 * s][0], pair[4 * s][1], pair[4 * s + 1][0], pair[4 * s + 1][1],
                               pair[4 * s + 2][0], pair[4 * s + 2][1], pair[4 * s + 3][0], pair[4 * s + 3][1]};
            out[i % D] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, s8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}),
                                                                weight, out[i % D], 0, 0, 0);
            if (i + kAhead < kSecond) read_values(i + kAhead);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    if (tiles > 0) {
        f16 even[2], odd[2];
        fetch_k(0, k_even);
        fetch_v(0, v_even);
        if (tiles > 1) fetch_k(1, k_odd);
        UNIQL_WAIT_ALL_LOADS();
        __syncthreads();
        even[0] = even[1] = f16{};
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
            for (int k = 0; k < 2; ++k) even[k] = __builtin_amdgcn_mfma_f32_32x32x16_f16(keys_of(k_even, k, i), q[i], even[k], 0, 0, 0);
        for (int t = 0; t < tiles; t += 2) {
            step(t, k_even, v_even, k_odd, v_odd, even, odd);
            if (t + 1 < tiles) step(t + 1, k_odd, v_odd, k_even, v_even, odd, even);
        }
    }
    l += __shfl_xor(l, 32, 64);
    if (!row_exists) return;
    half_t* to = a.out + (int64_t)(r.q_first + row) * a.out_row + (int64_t)head * a.out_head;
    const float inverse = seen > 0 ? 1.0f / l : 0.f;
#pragma unroll
    for (int i = 0; i < D; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int channel = 32 * i + 8 * j + 4 * half;
            half_t v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = seen > 0 ? (half_t)(out[i][4 * j + e] * inverse) : (half_t)0.f;
            if (channel + 4 <= a.v_dim) {
                *reinterpret_cast<h4u*>(to + channel) = h4u{v[0], v[1], v[2], v[3]};
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (channel + e < a.v_dim) to[channel + e] = v[e];
            }
        }
}

template <int D, int WAVES, bool PIECES>
static void go(const PromptArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL((prompt_attention_kernel<D, WAVES, PIECES>), dim3((unsigned)(a.blocks * a.heads)), dim3(64 * WAVES), 0, stream, a);
}
template <int D>
static void go(const PromptArgs& a, bool pieces, hipStream_t stream) {
    if (pieces) go<D, 4, true>(a, stream);
    else go<D, 4, false>(a, stream);
}

int prompt_attention_launch(const PromptArgs& args, hipStream_t stream) {
    PromptArgs a = args;
    a.q_sign = a.scale == 0.f ? 0 : (a.scale < 0.f ? -1 : 1);
    a.scale = a.q_sign == 0 ? 1.0f : (a.scale < 0.f ? -a.scale : a.scale);
    const int waves = 4;
    const int64_t blocks = (int64_t)a.rows / (kQueries * waves) + (a.sequences < a.rows ? a.sequences : a.rows);
    if (blocks * a.heads > 0x7fffffffLL) return UNIQL_E_SHAPE;
    a.blocks = (int)blocks;
    // 64 rows of K or V stay below 2^32 bytes
    const int64_t far = 1LL << 25;
    const uintptr_t bases = reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v);
    const bool pieces = ((a.k_row | a.k_head | a.v_row | a.v_head | a.k_dim | a.v_dim) & 7) == 0 && (bases & 15) == 0 && a.k_row >= 0 &&
                        a.v_row >= 0 && a.k_row <= far && a.v_row <= far;
    const int width = ((a.k_dim > a.v_dim ? a.k_dim : a.v_dim) + 31) / 32;
    if (width <= 2) go<2>(a, pieces, stream);
    else if (width == 3) go<3>(a, pieces, stream);
    else go<4>(a, pieces, stream);
    return hipGetLastError() == hipSuccess ? UNIQL_OK : UNIQL_E_LAUNCH;
}

}  // namespace uniql
