// Causal attention over the prompts of several sequences that lie behind each other: o = sum_j p_j v_j / sum_j p_j,
// p_j = exp(scale q . k_j - m), row i of a sequence with t queries and n keys over the keys j <= i + n - t.
//
// A workgroup takes 32 rows for each of its four waves (a query's heads that share keys side by side) and goes through the keys 64 at a
// time, in LDS, the next 64 on their way meanwhile (two buffers, straight from memory to LDS).  Matrix instructions of 32 x 32 x 16: the scores come transposed, keys along
// the rows, K q^T, because a lane then holds scores of one query and of just those keys that the second product, V^T P^T, wants
// from it: the weights never leave its registers.  That product takes V transposed, four keys of one channel at a time, which the
// transposing LDS read gives.  Rows of K and V lie in LDS with their 16-byte pieces exchanged by the row's number, so that neither
// kind of read meets itself in a bank.
// The maximum follows the scores only when a weight would pass 2^14 (weights are fp16, sums and outputs fp32): mostly once.  Weights are
// 2^6 times as large as they need be, so that many small ones beside a large one are not lost (16384 tokens 2.095 -> 2.108 ms).
// Scores beyond 2^22 (in powers of two), whose rounding alone is more than that room, are taken relative to the largest in a second pass,
// as infinities and NaN behind the causal border have a pass of their own (16384 tokens 2.138 -> 2.154 ms; as a branch of every step instead
// 2.121 -> 2.156).
// The rounding of the weights to fp16 (2^-11) is what a matrix instruction on fp16 asks for; their sum takes the rounded ones.
//
// Bound by the matrix and vector instructions together, and by power: 32 + 8 heads of 128, 16384 tokens 2.11 to 2.19 ms, 1.00 to 1.04
// PFLOP/s, where the library's product of 16384 x 16384 reaches 1.26 at the clock that the GPU holds; 8 prompts of 2048 0.82, 1 of 2048
// 0.66, 24 of 1 to 1850 tokens 0.60 to 0.65.  A step of 64 keys is 32 matrix instructions of 32 clocks for a wave, and beside the next tile's
// scores 32 exponentials, as many products, 16 conversions and 16 sums; two workgroups a compute unit fill each other's gaps.  Short
// prompts are bound by latency (1 token 6.8 us, 333 12): offsets, queries and the first tile follow each other, then 1.2 us a step.
// Tried and taken out: two sets of four waves that share the keys out (333 tokens 14.3 -> 13.9, 24 prompts 81 -> 107 us: a compute unit
// then holds one workgroup), blocks of all sequences in order of their length (24 prompts 75 -> 74, 64 of 512 276 -> 299 us), V's pieces
// exchanged so that no read meets another in a bank (a third of the LDS cycles less, 333 tokens 12.7 -> 12.55, 16384 2.115 -> 2.135 ms).
#include "prompt_attention.hpp"

namespace uniql {

constexpr int kKeys = 64;               // keys of a step
constexpr int kQueries = 32;            // rows of a wave
constexpr int kWaves = 4;
constexpr int kBlockRows = kWaves * kQueries;
constexpr float kLowest = -3.0e38f;
constexpr float kLift = 6.0f;           // the largest weight is 2^6: ones 2^-24 as large are many among long rows of keys and keep five bits
constexpr float kRoom = 8.0f;           // weights may grow to 2^14 before the maximum follows
constexpr float kFar = 4194304.0f;      // 2^22: below it a product of a score and the scale is rounded by a quarter at most
typedef __attribute__((address_space(3))) void* lds_ptr;
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) s4* lds_s4_ptr;
typedef _Float16 h8u __attribute__((ext_vector_type(8), aligned(2)));

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
// Sums over the lanes up to and including each.
template <int CTRL, int ROWS>
__device__ __forceinline__ int add_from(int v) { return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false); }
__device__ __forceinline__ int sums_upto(int v) {
    v = add_from<0x111, 0xf>(v);  // one, two, four, eight lanes below, within sixteen
    v = add_from<0x112, 0xf>(v);
    v = add_from<0x114, 0xf>(v);
    v = add_from<0x118, 0xf>(v);
    v = add_from<0x142, 0xa>(v);  // the last of the sixteen below, for the second and fourth sixteen
    return add_from<0x143, 0xc>(v);  // lane 31, for the upper half
}

// row / a.group for rows below 2^30 (see the launch)
__device__ __forceinline__ int query_of(const PromptArgs& a, int row) { return (int)(((uint64_t)(unsigned)row * a.group_factor) >> a.group_shift); }

// The sequence and the block of rows (of its queries times the heads of a key / value head) that block `index` of all is; every wave
// finds it for itself.
__device__ __forceinline__ bool find_block(const PromptArgs& a, int index, int block_rows, Rows& rows, int& block) {
    if (a.sequences == 1) {
        rows = rows_of(a, 0);
        block = index;
        return (int64_t)index * block_rows < (int64_t)rows.q_count * a.group;
    }
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base < a.sequences; base += 64) {
        const int s = base + lane;
        Rows r = {0, 0, 0, 0};
        if (s < a.sequences) r = rows_of(a, s);
        const int mine = (int)(((int64_t)r.q_count * a.group + block_rows - 1) / block_rows);
        const int upto = sums_upto(mine);
        const unsigned long long above = __ballot(before + upto > index);
        if (above) {
            const int owner = __builtin_ctzll(above);
            rows.q_first = __builtin_amdgcn_readlane(r.q_first, owner);
            rows.q_count = __builtin_amdgcn_readlane(r.q_count, owner);
            rows.k_first = __builtin_amdgcn_readlane(r.k_first, owner);
            rows.k_count = __builtin_amdgcn_readlane(r.k_count, owner);
            block = index - before - __builtin_amdgcn_readlane(upto - mine, owner);
            return true;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
        if (before > 0x3fffffff) return false;  // (offsets that fall and rise again)
    }
    return false;
}

// Eight values at any address that holds fp16 values.
__device__ __forceinline__ h8 whole_piece(const half_t* x) {
    const h8u v = *reinterpret_cast<const h8u*>(x);
    return h8{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]};
}

// How K and V come to LDS: straight, rows in whole 16-byte pieces at multiples of 16 bytes; straight, rows of any even width at
// multiples of 4 bytes, the last piece of K masked where it is read; or through registers.
enum { kWhole = 0, kTail = 1, kThrough = 2 };

// D: the wider of the two head widths in units of 32, 2 to 4.
template <int D, int LOAD>
__global__ __launch_bounds__(64 * kWaves, LOAD == kThrough ? 1 : 2) void prompt_attention_kernel(const PromptArgs a) {
    constexpr int kSteps = 2 * D;                      // of 16 channels, of the first product
    constexpr int kPieces = D == 2 ? 8 : 16;           // 16-byte pieces of a row in LDS
    constexpr int kRowBytes = kPieces * 16;
    constexpr int kTileBytes = kKeys * kRowBytes;
    constexpr int kRowsAtOnce = 64 / kPieces;          // rows that a wave's access covers
    constexpr int kAccesses = kKeys / (kRowsAtOnce * kWaves);
    // Two K tiles and two V tiles: variables of their own, which tells the compiler that reading one does not wait for what is on its way
    // into another.
    __shared__ __attribute__((aligned(16))) char k_even[kTileBytes], k_odd[kTileBytes], v_even[kTileBytes], v_odd[kTileBytes];
    __shared__ int spoilt[kWaves];
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, col = lane & 31, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // neighbouring workgroups have different key / value heads: those of one head stay on an XCD and share its L2
    const unsigned kv_heads = (unsigned)(a.heads / a.group);
    const int kv_head = (int)(blockIdx.x % kv_heads);
    // later blocks see more keys: they come first
    Rows r;
    int block;
    if (!find_block(a, (int)(a.blocks - 1 - blockIdx.x / kv_heads), kBlockRows, r, block)) return;
    // Rows are a sequence's queries times the query heads that share the key / value head, one query's heads side by side: short
    // sequences fill a tile of rows, and the rows of a tile see almost the same keys.
    const int offset = r.k_count - r.q_count, rows = r.q_count * a.group;
    auto seen_by = [&](int row) __attribute__((always_inline)) { return a.causal ? clamp_to(query_of(a, row) + offset + 1, 0, r.k_count) : r.k_count; };
    const int row0 = block * kBlockRows + wave * kQueries, row = row0 + col;
    const int seen = seen_by(row);  // keys of the lane's row
    // of the wave's first row and of its last, and of the workgroup's
    const int last_row = rows - 1;
    int fewest = seen_by(row0);
    const int most = row0 < rows ? seen_by(row0 + kQueries - 1 < last_row ? row0 + kQueries - 1 : last_row) : 0;
    const int block_end = (block + 1) * kBlockRows - 1, block_most = seen_by(block_end < last_row ? block_end : last_row);
    const int block_fewest = seen_by(block * kBlockRows);
    const int tiles = (block_most + kKeys - 1) / kKeys;

    // With a width that is no multiple of eight the last two pieces that K has change places with the last two that LDS has, so that the
    // last step reads them.
    const int tail_pair = LOAD == kTail && (a.k_dim >> 4) < kSteps ? a.k_dim >> 4 : kSteps - 1;
    auto moved = [&](int pair) __attribute__((always_inline)) {
        return LOAD == kTail ? (pair == kSteps - 1 ? tail_pair : (pair == tail_pair ? kSteps - 1 : pair)) : pair;
    };
    bool careful = false;
    const float unit = a.scale * 1.4426950408889634f;  // positive: a negative scale has turned q

    const half_t* const k_base = a.k + (int64_t)r.k_first * a.k_row + (int64_t)kv_head * a.k_head;
    const half_t* const v_base = a.v + (int64_t)r.k_first * a.v_row + (int64_t)kv_head * a.v_head;
    // this lane's part of an access: a row of the tile and a piece of it
    const int part_row = wave * kRowsAtOnce + lane / kPieces, part = lane % kPieces;
    // Rows behind the sequence lie beyond the descriptor and come as zeros, and so do pieces behind the width.
    auto fetch = [&](const half_t* tile, unsigned stride, int width, bool keys, int left, char* to) __attribute__((always_inline)) {
        auto piece_of = [&](int row) __attribute__((always_inline)) {
            if (!keys) return part ^ (2 * (row & 3));
            const int piece = part ^ (row & (kPieces - 1));
            return 2 * moved(piece >> 1) + (piece & 1);
        };
        if constexpr (LOAD == kThrough) {
            // (value by value in the last piece of a row; these layouts are for other callers than the fused projection)
#pragma unroll 1
            for (int row = part_row; row < kKeys; row += kRowsAtOnce * kWaves) {
                const int piece = piece_of(row);
                h8 v = {};
                if (row < left) {
                    const half_t* const from = tile + (int64_t)row * (keys ? a.k_row : a.v_row) + 8 * piece;
                    if (8 * piece + 8 <= width) v = whole_piece(from);
                    else
                        for (int j = 0; 8 * piece + j < width; ++j) {
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                if (e == j) v[e] = from[j];
                        }
                }
                *reinterpret_cast<h8*>(to + row * kRowBytes + part * 16) = v;
            }
        } else {
            const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
                const_cast<half_t*>(tile), 0, 2u * ((unsigned)((left < kKeys ? left : kKeys) - 1) * stride + (unsigned)width), 0x00020000);
            // (at is a multiple of the rows over which pieces change places)
            const int piece = piece_of(part_row);
            const unsigned first = piece * 8 < width ? 2u * ((unsigned)part_row * stride) + 16u * piece : 0x80000000u;
#pragma unroll
            for (int i = 0; i < kAccesses; ++i) {
                const int at = i * kRowsAtOnce * kWaves;
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr)(to + (at + wave * kRowsAtOnce) * kRowBytes), 16,
                                                         first + 2u * (unsigned)at * stride, 0, 0, 0);
            }
        }
    };
    // The tiles come one after the other, K and V each.
    const half_t *k_tile = k_base, *v_tile = v_base;
    auto fetch_k = [&](int t, char* to) __attribute__((always_inline)) {
        if (t >= tiles) return;
        fetch(k_tile, (unsigned)a.k_row, a.k_dim, true, r.k_count - t * kKeys, to);
        k_tile += kKeys * a.k_row;
    };
    auto fetch_v = [&](int t, char* to) __attribute__((always_inline)) {
        if (t >= tiles) return;
        fetch(v_tile, (unsigned)a.v_row, a.v_dim, false, r.k_count - t * kKeys, to);
        v_tile += kKeys * a.v_row;
    };
    auto fetch_first = [&]() __attribute__((always_inline)) {
        fetch_k(0, k_even);
        fetch_v(0, v_even);
        fetch_k(1, k_odd);
    };
    fetch_first();

    h8 q[kSteps];
    const bool row_exists = row < rows;
    {
        const int token = row_exists ? query_of(a, row) : 0, head = kv_head * a.group + (row_exists ? row - token * a.group : 0);
        const half_t* from = a.q + (int64_t)(r.q_first + token) * a.q_row + (int64_t)head * a.q_head;
        // whole pieces, then the one that is not whole
        const int partial = a.k_dim >> 3;
        h8 rest = {};
        if (row_exists && (partial & 1) == half)
            for (int j = 0; j < (a.k_dim & 7); ++j) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (e == j) rest[e] = from[8 * partial + j];
            }
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int piece = 2 * moved(i) + half;
            q[i] = h8{};
            if (row_exists && piece < partial) q[i] = whole_piece(from + 8 * piece);
            if (piece == partial) q[i] = rest;
            if (a.q_sign <= 0) q[i] = a.q_sign < 0 ? -q[i] : h8{};
        }
    }
    f16 out[D];
    float m = kLowest, l, shift = 0.f;  // shift: taken off the row's scores in a careful pass
    bool searching = false;             // the pass looks for the row's maximum
    // where the lane reads: K rows col and 32 + col, piece 2 step + half; V rows 4 half + j (+ 8), j = (lane / 4) % 4, four channels
    const int k_read = col * kRowBytes, k_swap = col & (kPieces - 1);
    const int v_j = (lane >> 2) & 3, v_read = (4 * half + v_j) * kRowBytes + (lane & 1) * 8;
    const int v_sub = 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
    auto keys_of = [&](const char* tile, int k, int i) __attribute__((always_inline)) {
        return *reinterpret_cast<const h8*>(tile + k_read + k * 32 * kRowBytes + (((2 * i + half) ^ k_swap) * 16));
    };
    // what the last step's piece holds of the width, two values a word; the rest of it is another head's
    uint32_t inside[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) inside[j] = 16 * tail_pair + 8 * half + 2 * j < a.k_dim ? 0xffffffffu : 0u;
    auto product = [&](h8 keys, int i, const f16& sum) __attribute__((always_inline)) {
        if (LOAD == kTail && i == kSteps - 1) {
            const u32x4 w = __builtin_bit_cast(u32x4, keys);
            keys = __builtin_bit_cast(h8, u32x4{w[0] & inside[0], w[1] & inside[1], w[2] & inside[2], w[3] & inside[3]});
        }
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(keys, q[i], sum, 0, 0, 0);
    };
    // A step: the weights of tile t from its scores, which the step before has computed, the next tile's scores, the second product.
    auto step = [&](int t, char* k_lds, char* v_lds, char* next_k_lds, char* next_v_lds, f16 (&score)[2], f16 (&next)[2]) __attribute__((always_inline)) {
        const int key0 = t * kKeys;
        UNIQL_WAIT_ALL_LOADS();
        __syncthreads();
        fetch_k(t + 2, k_lds);
        fetch_v(t + 1, next_v_lds);
        const bool masked = key0 + kKeys > fewest;
        // A key that some rows of the tile see and others do not: its weight is zero for those, but zero times an infinity is not.  In the
        // careful pass each lane looks at one such key; those with such values become zeros in LDS, and what they give to the rows that see
        // them is added on its own, below.
        unsigned long long odd_keys = 0;
        if (careful && key0 + kKeys > block_fewest) {  // the same for all waves
            uint32_t any = 0;
            for (int i = 0; i < kPieces; ++i) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(v_lds + lane * kRowBytes + i * 16);
#pragma unroll
                for (int j = 0; j < 4; ++j) any |= ((w[j] & 0x7c007c00u) + 0x04000400u) & 0x80008000u;  // an exponent of all ones runs over
            }
            odd_keys = __ballot(any != 0);
            __syncthreads();
            if ((odd_keys >> lane) & 1)
                for (int i = 0; i < kPieces; ++i) *reinterpret_cast<u32x4*>(v_lds + lane * kRowBytes + i * 16) = u32x4{0u, 0u, 0u, 0u};
        }
        const bool active = key0 < most;  // the wave's rows see some of the keys (all waves take part in the barriers)
        if (active) {
            if (masked) {
                if (careful) {
                    float by = shift;
                    asm volatile("" : "+v"(by));  // (not the scores and then the scale in one go: the difference is rounded first)
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int i = 0; i < 16; ++i) score[k][i] -= by;
                }
                int seen_here = seen - key0 - 4 * half;
                asm volatile("" : "+v"(seen_here));  // keeps the comparisons out of the other tiles' way
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (32 * k + 8 * (i / 4) + i % 4 >= seen_here) score[k][i] = -INFINITY;
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
                if (t > 0) {  // (all zeros so far)
                    l *= fade;
#pragma unroll
                    for (int i = 0; i < D; ++i) out[i] *= fade;
                }
            }
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
        const float base = m - kLift;
        f2 power[2];
        u32x16 pair = {};
        auto raise = [&](int i) __attribute__((always_inline)) {
            power[i & 1] = f2{__builtin_amdgcn_exp2f(__builtin_fmaf(score[i >> 3][2 * (i & 7)], unit, -base)),
                              __builtin_amdgcn_exp2f(__builtin_fmaf(score[i >> 3][2 * (i & 7) + 1], unit, -base))};
        };
        auto round_pair = [&](int i) __attribute__((always_inline)) {
            const h2 both = __builtin_convertvector(power[i & 1], h2);
            pair[i] = h2_to_bits(both);
            l = __builtin_amdgcn_fdot2(both, h2{(half_t)1.f, (half_t)1.f}, l, false);
        };
        next[0] = next[1] = f16{};
#pragma unroll
        for (int i = 0; i < 4; ++i) read_keys(i);
        __builtin_amdgcn_sched_barrier(0);
        int raised = 0;
#pragma unroll
        for (int i = 0; i < kFirst; ++i) {
            next[i & 1] = product(keys[i & 3], i >> 1, next[i & 1]);
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
            const h8 weight = __builtin_bit_cast(h8, u32x4{pair[4 * s], pair[4 * s + 1], pair[4 * s + 2], pair[4 * s + 3]});
            out[i % D] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, s8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}),
                                                                weight, out[i % D], 0, 0, 0);
            if (i + kAhead < kSecond) read_values(i + kAhead);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (odd_keys) {
            for (unsigned long long left = odd_keys; left; left &= left - 1) {
                const int key = __builtin_ctzll(left);
                const int index = 4 * (key >> 4) + 2 * ((key >> 3) & 1) + ((key >> 1) & 1);  // of the pair of weights, in the half (key >> 2) & 1
                uint32_t both = 0;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const uint32_t other = pair[i];
                    both = i == index ? other : both;
                    asm volatile("" : "+v"(both));  // or the weights become an array in memory
                }
                both = (uint32_t)__shfl((int)both, col + 32 * ((key >> 2) & 1), 64);
                const float p = (float)bits_to_h2(both)[key & 1];
                // (columns behind the width are beyond the descriptor)
                const __amdgpu_buffer_rsrc_t v = __builtin_amdgcn_make_buffer_rsrc(const_cast<half_t*>(v_base + (int64_t)(key0 + key) * a.v_row), 0,
                                                                                   2u * (unsigned)a.v_dim, 0x00020000);
                if (key0 + key < seen) {
#pragma unroll
                    for (int i = 0; i < D; ++i)
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            out[i][j] += p * (float)__builtin_bit_cast(half_t, (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(
                                                                                   v, 8 * half, 2 * (32 * i + 8 * (j / 4) + j % 4), 0));
                }
            }
        }
    };
    for (int pass = 0;; ++pass) {
        careful = pass > 0;
#pragma unroll
        for (int i = 0; i < D; ++i) out[i] = f16{};
        l = 0.f;
        if (tiles > 0) {
            f16 even[2], odd[2];
            UNIQL_WAIT_ALL_LOADS();
            __syncthreads();
            h8 keys[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) keys[i] = keys_of(k_even, i & 1, i >> 1);
            even[0] = even[1] = f16{};
#pragma unroll
            for (int i = 0; i < 2 * kSteps; ++i) {
                even[i & 1] = product(keys[i & 3], i >> 1, even[i & 1]);
                if (i + 4 < 2 * kSteps) keys[i & 3] = keys_of(k_even, i & 1, (i + 4) >> 1);
                __builtin_amdgcn_sched_barrier(0);
            }
            for (int t = 0; t < tiles; t += 2) {
                step(t, k_even, v_even, k_odd, v_odd, even, odd);
                if (t + 1 < tiles) step(t + 1, k_odd, v_odd, k_even, v_even, odd, even);
            }
        }
        // Two things ask for all to be done again, with care.  Infinities and NaN, which are rare and show in a result.  And maxima so
        // large that the products of the scores and the scale, exact in the exponentials, differ from the rounded maximum by more
        // than the room that weights have: such a row's scores are taken relative to their largest, of which a pass leaves 2^-23,
        // until the maximum is a near one; a last pass starts from it, as it does for the other rows.
        const bool row_far = m != kLowest && fabsf(m) >= kFar;
        bool bad = row_far || searching;
        searching = row_far;
        if (row_far) {
            shift += m / unit;
            m = kLowest;
        }
        if (pass == 0) {
            float zero = 0.f;
#pragma unroll
            for (int i = 0; i < D; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) zero = __builtin_fmaf(out[i][j], 0.f, zero);
            bad |= row < rows && zero != 0.f;
        }
        bad = __any(bad);
        if (lane == 0) spoilt[wave] = bad;
        __syncthreads();
        int any = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) any |= spoilt[w];
        if (__builtin_amdgcn_readfirstlane(any) == 0 || pass == 3) break;
        fewest = 0;  // a careful pass treats every tile as one that not all rows see
        k_tile = k_base, v_tile = v_base;
        fetch_first();
    }
    l += __shfl_xor(l, 32, 64);
    int my_row = row;
    asm volatile("" : "+v"(my_row));  // the quotient is not kept over the loop
    if (my_row >= rows) return;
    const int token = query_of(a, my_row), head = kv_head * a.group + my_row - token * a.group;
    half_t* to = a.out + (int64_t)(r.q_first + token) * a.out_row + (int64_t)head * a.out_head;
    // A lane has four values of every eight, the lane 32 from it the others: exchanged so that each has whole eights.
    const float inverse = seen > 0 ? 1.0f / l : 0.f;
#pragma unroll
    for (int i = 0; i < D; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            uint32_t w[2][2];
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int f = 0; f < 2; ++f) {
                    const f2 v = {out[i][8 * j + 4 * e + 2 * f] * inverse, out[i][8 * j + 4 * e + 2 * f + 1] * inverse};
                    w[e][f] = seen > 0 ? h2_to_bits(__builtin_convertvector(v, h2)) : 0u;
                }
            const auto x = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
            const auto y = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
            const h8 v = __builtin_bit_cast(h8, u32x4{x[0], y[0], x[1], y[1]});
            const int channel = 32 * i + 16 * j + 8 * half;
            if (channel + 8 <= a.v_dim) {
                *reinterpret_cast<h8u*>(to + channel) = h8u{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]};
            } else {
                for (int e = 0; channel + e < a.v_dim; ++e) {
                    half_t one = v[0];
#pragma unroll
                    for (int f = 1; f < 8; ++f) one = e == f ? v[f] : one;
                    to[channel + e] = one;
                }
            }
        }
}

template <int D>
static void go(const PromptArgs& a, int load, hipStream_t stream) {
    const dim3 grid((unsigned)(a.blocks * (a.heads / a.group))), block(64 * kWaves);
    if (load == kWhole) hipLaunchKernelGGL((prompt_attention_kernel<D, kWhole>), grid, block, 0, stream, a);
    else if (load == kTail) hipLaunchKernelGGL((prompt_attention_kernel<D, kTail>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((prompt_attention_kernel<D, kThrough>), grid, block, 0, stream, a);
}

int prompt_attention_launch(const PromptArgs& args, hipStream_t stream) {
    PromptArgs a = args;
    a.q_sign = a.scale == 0.f ? 0 : (a.scale < 0.f ? -1 : 1);
    a.scale = a.q_sign == 0 ? 1.0f : (a.scale < 0.f ? -a.scale : a.scale);
    // 64 rows of K or V stay below 2^31 bytes
    const int64_t far = 1LL << 24, strides = a.k_row | a.k_head | a.v_row | a.v_head | a.k_dim | a.v_dim;
    const uintptr_t bases = reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v);
    const bool near = a.k_row >= a.k_dim && a.v_row >= a.v_dim && a.k_row <= far && a.v_row <= far;
    const int load = near && (strides & 7) == 0 && (bases & 15) == 0 ? kWhole
                     : near && (strides & 1) == 0 && (bases & 3) == 0 && a.k_row >= 8 && a.v_row >= 8 ? kTail : kThrough;
    const int64_t rows = (int64_t)a.rows * a.group, blocks = rows / kBlockRows + (a.sequences < a.rows ? a.sequences : a.rows);
    if (rows > (1LL << 30) || blocks * (a.heads / a.group) >= (1LL << 32) / (64 * kWaves)) return UNIQL_E_SHAPE;
    a.blocks = (int)blocks;
    // floor(row / d) = row f >> (31 + s) with f = 2^(31 + s) / d rounded up and s so that d <= 2^s < 2 d: f d - 2^(31 + s) < 2^s, so the
    // excess stays below 1 / d for rows below 2^31
    int s = 0;
    while ((1 << s) < a.group) ++s;
    a.group_shift = 31 + s;
    a.group_factor = (unsigned)(((1ULL << a.group_shift) + a.group - 1) / a.group);
    const int width = ((a.k_dim > a.v_dim ? a.k_dim : a.v_dim) + 31) / 32;
    if (width <= 2) go<2>(a, load, stream);
    else if (width == 3) go<3>(a, load, stream);
    else go<4>(a, load, stream);
    return hipGetLastError() == hipSuccess ? UNIQL_OK : UNIQL_E_LAUNCH;
}

}  // namespace uniql
