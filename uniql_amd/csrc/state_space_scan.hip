// Linear attention with a decay for each head over packed prompts: S_t = exp(l_t) S_{t-1} + s_t x_t b_t^T, y_t = S_t c_t + d x_t,
// with the time step s_t = softplus(dt_t + bias) and l_t = s_t a, for each head's matrix S [head_dim][states].
//
// Chunks of 64 rows: with L_i the sum of l up to row i of the chunk,
//   y_i = exp(L_i) S c_i + sum_{j <= i} exp(L_i - L_j) s_j (b_j . c_i) x_j + d x_i,      S' = exp(L_63) S + sum_j exp(L_63 - L_j) s_j x_j b_j^T,
// all four products on matrix instructions (16 x 16 x 32).  A workgroup walks through the chunks of one head with S in registers, b and x in
// LDS, the next chunk's on their way meanwhile.  Each of its four waves has sixteen rows i for the outputs - their c stays in registers, and
// the weights of the third product come out of the first one where the matrix instruction wants them (the scores transposed, as
// b c^T) - and sixteen channels for the state, of which it leaves a rounded copy in LDS for the next chunk's second product.
//
// Sequences of any lengths are cut into segments of equally many chunks, from the offsets on the device.  Where there are several, a
// first launch walks through what lies in front of the last segment for the state alone: what each segment adds to the state of the sequence
// that goes on behind it, and the decay over it.  The second launch puts them together where a segment begins within a sequence.
//
// S, all sums and the decays are fp32, L is summed up in 64 bits and kept as two floats (its differences matter, also behind a
// token that wipes the state).  Rounded to fp16 are the weights and S for the outputs, which are fp16 themselves, each relative to the largest
// of its row, so that no finite value overflows or vanishes; what goes into S is split into two fp16 numbers, 22 bits.  An infinity or
// NaN in x must not reach rows in front of it, also as zero times it: a chunk with one is done again row by row.
#include "state_space.hpp"

namespace uniql {

constexpr int kChunk = 64;
constexpr int kScanThreads = 256;
typedef __attribute__((address_space(3))) void* lds_ptr;
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s4* lds_s4_ptr;

#define UNIQL_WAIT_ALL_LOADS() __builtin_amdgcn_s_waitcnt(0x0F70)  // vmcnt(0), the other counters left alone (gfx9 encoding)

__device__ __forceinline__ h8 join(s4 lo, s4 hi) { return __builtin_bit_cast(h8, s8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}); }
__device__ __forceinline__ float power_of_two(int e) { return __builtin_bit_cast(float, (127 + e) << 23); }  // -126 <= e <= 127
__device__ __forceinline__ int exponent_of(float v) { return (int)((__builtin_bit_cast(uint32_t, v) >> 23) & 255u) - 127; }
__device__ __forceinline__ int clamp_to(int v, int low, int high) { return v < low ? low : (v > high ? high : v); }
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// What is known of a chunk's rows before its products: the logarithms (base 2) of the decay up to each row as a sum of two floats, the time
// steps, what a row adds to the state, and the decays themselves.
struct RowValues {
    float log_hi[kChunk], log_lo[kChunk], step[kChunk], into[kChunk], decay[kChunk];
};

// Rows row .. end of a sequence that a workgroup goes through.
struct Walk {
    Sequence q;
    int index, row, end;  // end: of the sequence's rows within the segment
};

// Chunks in all sequences.
__device__ __forceinline__ int count_chunks(const Sequences& all) {
    const int lane = threadIdx.x & 63;
    int total = 0;
    for (int base = 0; base < all.count; base += 64) {
        const int s = base + lane;
        const int mine = s < all.count ? (sequence_of(all, s).rows + kChunk - 1) / kChunk : 0;
        total += __builtin_amdgcn_readlane(sums_upto(mine), 63);
        if (total > 0x3fffffff) return 0;  // (offsets that fall and rise again)
    }
    return total;
}
// The sequence that chunk `index` of all belongs to, and how many of its chunks come before.
__device__ __forceinline__ int find_chunk(const Sequences& all, int index, int& before_in_sequence) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base < all.count; base += 64) {
        const int s = base + lane;
        const int mine = s < all.count ? (sequence_of(all, s).rows + kChunk - 1) / kChunk : 0;
        const int upto = sums_upto(mine);
        const unsigned long long above = __ballot(before + upto > index);
        if (above) {
            const int owner = __builtin_ctzll(above);
            before_in_sequence = index - before - __builtin_amdgcn_readlane(upto - mine, owner);
            return base + owner;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    before_in_sequence = 0;
    return all.count;
}
__device__ __forceinline__ int border(int segment, int segments, int chunks) { return (int)((int64_t)segment * chunks / segments); }

// N32: the states in units of 32; THROUGH: rows that cannot go straight to LDS; LAST: the second launch, or the only one.
template <int N32, bool THROUGH, bool LAST>
__global__ __launch_bounds__(kScanThreads, N32 <= 4 ? 2 : 1) void state_space_scan_kernel(const ScanArgs a) {
    constexpr int kPieces = N32 <= 2 ? 8 : (N32 <= 4 ? 16 : 32);  // 16-byte pieces of a row of b in LDS
    constexpr int kRowBytes = kPieces * 16;
    constexpr int kTiles = 2 * N32;                               // of sixteen states
    __shared__ __attribute__((aligned(16))) char b_even[kChunk * kRowBytes], b_odd[kChunk * kRowBytes];
    __shared__ __attribute__((aligned(16))) char x_even[kChunk * 128], x_odd[kChunk * 128];
    __shared__ __attribute__((aligned(16))) char s_lds[LAST ? kChunk * kRowBytes : 16];
    __shared__ __attribute__((aligned(16))) float s_unit[kChunk];
    __shared__ RowValues values[2];
    __shared__ int odd_x;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), low = lane & 15, high = lane >> 4;

    // neighbouring workgroups, which are on different XCDs, have heads of different groups: those of one group share an L2
    const int units = a.heads * a.head_blocks;
    const int unit = units % 8 == 0 ? (int)(blockIdx.x % 8) * (units / 8) + (int)(blockIdx.x / 8) : (int)blockIdx.x;
    const int head = unit / a.head_blocks, p0 = unit % a.head_blocks * 64;
    const int segment = blockIdx.y;
    const int chunks = uniform(count_chunks(a.sequences));
    const int begin = border(segment, a.segments, chunks), end = border(segment + 1, a.segments, chunks);
    if (begin >= end) return;

    const int head_dim = a.head_dim - p0;  // (from p0 on; a head may be wider than the block's 64)
    const float rate = a.a[head], bias = a.dt_bias ? a.dt_bias[head] : 0.f, skip = a.d ? a.d[head] : 0.f;
    const int group = head / a.share;
    const half_t* const x_base = a.x + (int64_t)head * a.x_head + p0;
    const half_t* const b_base = a.b + (int64_t)group * a.b_group;
    const half_t* const c_base = a.c + (int64_t)group * a.c_group;
    const half_t* const dt_base = a.dt + head;
    half_t* const y_base = a.y + (int64_t)head * a.y_head + p0;

    // what the first launch leaves: for each segment but the last and each workgroup's head, in the registers' order
    constexpr int kHeld = kTiles * kScanThreads;  // vectors of four
    const int64_t place = (int64_t)segment * units + unit;
    const int64_t added_all = (int64_t)(a.segments - 1) * units * kHeld;
    f4* const added = reinterpret_cast<f4*>(a.temp);
    f4* const kept_first = added + added_all;                                 // states that sequences begin with, likewise
    float* const faded = reinterpret_cast<float*>(kept_first + added_all);    // decays over segments

    int offset;
    Walk now;
    int budget = end - begin;  // chunks
    if constexpr (LAST) {
        now.index = uniform(find_chunk(a.sequences, begin, offset));
    } else {
        // what goes on behind the segment's last chunk
        int last_offset;
        now.index = uniform(find_chunk(a.sequences, end - 1, last_offset));
        last_offset = uniform(last_offset);
        const Sequence q = sequence_of(a.sequences, now.index);
        if ((last_offset + 1) * kChunk >= q.rows) return;  // nothing
        offset = last_offset + 1 < budget ? 0 : last_offset + 1 - budget;
        budget = last_offset + 1 - offset;
    }
    offset = uniform(offset);
    auto enter = [&](Walk& w, int from_chunk) __attribute__((always_inline)) {
        w.q = sequence_of(a.sequences, w.index);
        w.row = w.q.first + from_chunk * kChunk;
        const int left = w.q.rows - from_chunk * kChunk, room = budget < (1 << 24) ? budget * kChunk : 0x7fffffff;
        const int rows = left < room ? left : room;
        w.end = w.row + rows;
        budget -= (rows + kChunk - 1) / kChunk;
    };
    enter(now, offset);

    // ---- loads ----------------------------------------------------------------------------------------------------------
    // LDS holds a row's pieces exchanged by its number, so that neither kind of read meets itself in a bank.
    auto swap_of = [&](int row) __attribute__((always_inline)) { return kPieces == 8 ? (row >> 1) & 7 : row & 15; };
    auto fetch_tile = [&](const half_t* tile, int64_t stride, int width, int rows, bool is_x, char* to) __attribute__((always_inline)) {
        const int pieces = is_x ? 8 : kPieces, rows_at_once = 64 / pieces;
        const int part_row = wave * rows_at_once + lane / pieces, part = lane % pieces;
        const int accesses = kChunk / (rows_at_once * 4);
        if constexpr (THROUGH) {
#pragma unroll 1
            for (int row = part_row; row < kChunk; row += rows_at_once * 4) {
                const int piece = part ^ (is_x ? (row >> 1) & 7 : swap_of(row));
                h8 v = {};
                if (row < rows && piece * 8 < width) v = load_halves(tile + row * stride + piece * 8, width - piece * 8);
                *reinterpret_cast<h8*>(to + row * (pieces * 16) + part * 16) = v;
            }
        } else {
            // rows behind the chunk and pieces behind the width are beyond the descriptor and come as zeros
            const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
                const_cast<half_t*>(tile), 0, 2u * ((unsigned)(rows - 1) * (unsigned)stride + (unsigned)width), 0x00020000);
#pragma unroll
            for (int i = 0; i < accesses; ++i) {
                const int row = i * rows_at_once * 4 + part_row;
                const int piece = part ^ (is_x ? (row >> 1) & 7 : swap_of(row));
                const unsigned at = piece * 8 < width ? 2u * (unsigned)row * (unsigned)stride + 16u * piece : 0x80000000u;
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr)(to + (i * rows_at_once * 4 + wave * rows_at_once) * (pieces * 16)), 16,
                                                         at, 0, 0, 0);
            }
        }
    };
    const int x_width = head_dim < 64 ? head_dim : 64;
    auto fetch = [&](int row, int rows, char* b_to, char* x_to) __attribute__((always_inline)) {
        fetch_tile(b_base + (int64_t)row * a.b_row, a.b_row, a.states, rows, false, b_to);
        fetch_tile(x_base + (int64_t)row * a.x_row, a.x_row, x_width, rows, true, x_to);
    };
    h8 c[N32];
    auto fetch_c = [&](int row, int rows) __attribute__((always_inline)) {
        const int i = 16 * wave + low;
        const half_t* const from = c_base + (int64_t)(row + i) * a.c_row;
#pragma unroll
        for (int k = 0; k < N32; ++k) {
            const int n = 32 * k + 8 * high;
            c[k] = h8{};
            if (i < rows && n < a.states) c[k] = load_halves(from + n, THROUGH ? a.states - n : 8);
        }
    };
    // The first wave works out a chunk's row values, a row a lane.
    auto row_values = [&](float dt, int rows, RowValues& to) __attribute__((always_inline)) {
        const float step = lane < rows ? time_step(a, dt, bias) : 0.f;
        const double mine = lane < rows ? (double)step * (double)rate * 1.4426950408889634 : 0.0;
        const double log = sums_upto(mine);
        const double all = __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(log), 63), __builtin_amdgcn_readlane(__double2loint(log), 63));
        const float hi = (float)log;
        to.log_hi[lane] = hi;
        to.log_lo[lane] = (float)(log - (double)hi);
        to.step[lane] = step;
        to.into[lane] = lane < rows ? __builtin_amdgcn_exp2f((float)(all - log)) * step : 0.f;
        to.decay[lane] = __builtin_amdgcn_exp2f(hi) * (1.0f + (float)(log - (double)hi) * 0.6931471805599453f);
    };
    auto load_dt = [&](int row, int rows) __attribute__((always_inline)) {
        return wave == 0 && lane < rows ? (float)dt_base[(int64_t)(row + lane) * a.dt_row] : 0.f;
    };

    // ---- the state ------------------------------------------------------------------------------------------------------
    // Lane: channel 16 wave + low, states 16 t + 4 high + r, in units of `unit_s` (a power of two of the channel's own).
    f4 S[kTiles];
    float unit_s = 1.f;
    const int my_p = 16 * wave + low;
    const bool p_there = my_p < head_dim;
    const int64_t pool_size = (int64_t)a.head_dim * a.states;
    const bool quads = a.states % 4 == 0;
    auto pool_at = [&](int place_of) __attribute__((always_inline)) { return ((int64_t)place_of * a.heads + head) * pool_size + (int64_t)(p0 + my_p) * a.states + 4 * high; };
    auto load_state = [&](int place_of) __attribute__((always_inline)) {
        const float* const from = a.state + pool_at(place_of);
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            const int n = 16 * t + 4 * high;
            S[t] = f4{};
            if (p_there && n < a.states) {
                if (quads) S[t] = *reinterpret_cast<const f4*>(from + 16 * t);
                else
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (n + r < a.states) S[t][r] = from[16 * t + r];
            }
        }
    };
    auto store_state = [&](int place_of) __attribute__((always_inline)) {
        float* const to = a.state_out + pool_at(place_of);
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            const int n = 16 * t + 4 * high;
            if (p_there && n < a.states) {
                const f4 v = S[t] * unit_s;
                if (quads) *reinterpret_cast<f4*>(to + 16 * t) = v;
                else
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (n + r < a.states) to[16 * t + r] = v[r];
            }
        }
    };
    // The copy for the next chunk's outputs.
    auto leave_copy = [&]() __attribute__((always_inline)) {
        float top = 0.f;
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) top = fmaxf(top, fabsf(S[t][r]));
        top = max_of_sixteenths(top);
        const int e = clamp_to(exponent_of(top), -100, 127);
        const float up = power_of_two(14 - e);
        if (high == 0) s_unit[my_p] = power_of_two(e - 14) * unit_s;
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            const int piece = 2 * t + (high >> 1);
            const h4 v = {(half_t)(S[t][0] * up), (half_t)(S[t][1] * up), (half_t)(S[t][2] * up), (half_t)(S[t][3] * up)};
            *reinterpret_cast<h4*>(s_lds + my_p * kRowBytes + ((piece ^ swap_of(my_p)) * 16) + (high & 1) * 8) = v;
        }
    };
    // A sequence's state where the workgroup comes upon it: from earlier segments, from the pool, or empty.
    auto first_state = [&](const Walk& w, bool from_earlier) __attribute__((always_inline)) {
        unit_s = 1.f;
        if constexpr (LAST) {
            if (from_earlier) {
                const int first_chunk = begin - offset;
                const int from = (int)((((int64_t)first_chunk + 1) * a.segments - 1) / chunks);
#pragma unroll
                for (int t = 0; t < kTiles; ++t) S[t] = f4{};
                for (int g = from; g < segment; ++g) {
                    const int64_t at = (int64_t)g * units + unit;
                    const float fade = faded[at];
#pragma unroll
                    for (int t = 0; t < kTiles; ++t) {
                        const f4 v = added[at * kHeld + t * kScanThreads + tid];
                        S[t] = g == from ? v : S[t] * fade + v;
                    }
                }
                return;
            }
            if (a.state && w.q.continued && w.end < w.q.first + w.q.rows) {
                // goes on behind this segment, where the pool's may be replaced at any time
#pragma unroll
                for (int t = 0; t < kTiles; ++t) S[t] = kept_first[place * kHeld + t * kScanThreads + tid];
                return;
            }
        }
        if (!from_earlier && a.state && w.q.continued) {
            load_state(w.q.place);
        } else {
#pragma unroll
            for (int t = 0; t < kTiles; ++t) S[t] = f4{};
        }
        if constexpr (!LAST) {
            if (!from_earlier && a.state && w.q.continued) {
#pragma unroll
                for (int t = 0; t < kTiles; ++t) kept_first[place * kHeld + t * kScanThreads + tid] = S[t];
            }
        }
    };

    // ---- reads of LDS ---------------------------------------------------------------------------------------------------
    // rows 16 t + low, states 32 k + 8 high .. + 7
    auto rows_of = [&](const char* tile, int t, int k) __attribute__((always_inline)) {
        const int row = 16 * t + low;
        return *reinterpret_cast<const h8*>(tile + row * kRowBytes + (((4 * k + high) ^ swap_of(row)) * 16));
    };
    // column 16 t + low of rows 32 k + 4 high .. + 3 and 32 k + 16 + 4 high .. + 3: a lane reads four columns of one row, and sixteen lanes
    // exchange them
    const int tr_row = 4 * high + (low >> 2);
    auto columns_of = [&](const char* tile, int t, int k, bool is_x) __attribute__((always_inline)) {
        const int bytes = is_x ? 128 : kRowBytes;
        s4 v[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int row = 32 * k + 16 * h + tr_row, piece = 2 * t + ((low >> 1) & 1);
            const int swap = is_x ? (row >> 1) & 7 : swap_of(row);
            v[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_ptr)(const_cast<char*>(tile) + row * bytes + ((piece ^ swap) * 16) + (low & 1) * 8));
        }
        return join(v[0], v[1]);
    };

    // ---- the walk -------------------------------------------------------------------------------------------------------
    int careful_until = now.row;  // rows in front of it are done one by one
    auto rows_at = [&](const Walk& w) __attribute__((always_inline)) {
        const int most = w.row < careful_until ? 1 : kChunk;
        return w.end - w.row < most ? w.end - w.row : most;
    };
    int rows = rows_at(now);
    fetch(now.row, rows, b_even, x_even);
    if constexpr (LAST) fetch_c(now.row, rows);
    {
        const float dt = load_dt(now.row, rows);
        if (tid == 0) odd_x = 0;
        if (wave == 0) row_values(dt, rows, values[0]);
    }
    first_state(now, offset > 0);
    if constexpr (LAST) leave_copy();
    double segment_log = 0.0;

    // One chunk, with its tile in b_now and x_now; false when it was the last.
    auto chunk = [&](char* b_now, char* x_now, char* b_next, char* x_next, RowValues& now_values, RowValues& next_values) __attribute__((always_inline)) {
        UNIQL_WAIT_ALL_LOADS();
        __syncthreads();
        // what comes next
        Walk next = now;
        next.row = now.row + rows;
        bool new_sequence = false, more = true;
        if (next.row >= now.end) {
            more = false;
            if constexpr (LAST) {
                while (budget > 0 && !more) {
                    ++next.index;
                    if (next.index >= a.sequences.count) break;
                    if (sequence_of(a.sequences, next.index).rows == 0) continue;
                    enter(next, 0);
                    new_sequence = more = true;
                }
            }
        }
        if (new_sequence) careful_until = next.row;
        int next_rows = more ? rows_at(next) : 0;
        float next_dt = 0.f;
        if (more) {
            fetch(next.row, next_rows, b_next, x_next);
            next_dt = load_dt(next.row, next_rows);
        }

        // What a row adds to the state, x scaled by its time step and the decay behind it, in units of the channel's largest.
        h8 into_hi[2], into_lo[2];
        float unit_x;
        {
            float v[2][8], top = 0.f;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const h8 x = columns_of(x_now, wave, k, true);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const f4 w = *reinterpret_cast<const f4*>(&now_values.into[32 * k + 16 * h + 4 * high]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float u = (float)x[4 * h + r];
                        v[k][4 * h + r] = u * w[r];
                        // (a NaN is larger than all numbers here, as whole numbers are compared)
                        const uint32_t size = __builtin_bit_cast(uint32_t, u) & 0x7fffffffu;
                        if (rows > 1 && size >= 0x7f800000u && p_there) odd_x = 1;
                        top = fmaxf(top, fabsf(v[k][4 * h + r]));
                    }
                }
            }
            top = max_of_sixteenths(top);
            const int e = clamp_to(exponent_of(top), -60, 60);
            const float up = power_of_two(14 - e);
            unit_x = power_of_two(e - 14);
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float u = v[k][j] * up;
                    const half_t hi = (half_t)u;
                    into_hi[k][j] = hi;
                    // an infinity has no rest
                    const float rest = u - (float)hi;
                    into_lo[k][j] = (half_t)(fabsf(u) < INFINITY ? rest : 0.f);
                }
        }

        f4 y[4];
        float row_unit = 1.f, row_decay = 1.f;
        if constexpr (LAST) {
            const int i = 16 * wave + low;
            const float log_hi = now_values.log_hi[i], log_lo = now_values.log_lo[i];
            row_decay = now_values.decay[i];
            // weights of rows j (16 t + 4 high + r) for row i
            f4 m[4];
            float top = 0.f;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                m[t] = f4{};
                if (t <= wave && 16 * t < rows) {
#pragma unroll
                    for (int k = 0; k < N32; ++k) m[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(rows_of(b_now, t, k), c[k], m[t], 0, 0, 0);
                    const int j = 16 * t + 4 * high;
                    const f4 hi = *reinterpret_cast<const f4*>(&now_values.log_hi[j]), lo = *reinterpret_cast<const f4*>(&now_values.log_lo[j]);
                    const f4 step = *reinterpret_cast<const f4*>(&now_values.step[j]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float apart = (log_hi - hi[r]) + (log_lo - lo[r]);
                        const float w = m[t][r] * (__builtin_amdgcn_exp2f(apart) * step[r]);
                        m[t][r] = j + r <= i && j + r < rows ? w : 0.f;
                        top = fmaxf(top, fabsf(m[t][r]));
                    }
                }
            }
            top = max_of_sixteenths(top);
            const int e = clamp_to(exponent_of(top), -100, 127);
            const float up = power_of_two(14 - e);
            row_unit = power_of_two(e - 14);
            h8 weight[2];
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) weight[t >> 1][4 * (t & 1) + r] = (half_t)(m[t][r] * up);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                f4 within = {}, before = {};
                within = __builtin_amdgcn_mfma_f32_16x16x32_f16(columns_of(x_now, t, 0, true), weight[0], within, 0, 0, 0);
                if (wave >= 2) within = __builtin_amdgcn_mfma_f32_16x16x32_f16(columns_of(x_now, t, 1, true), weight[1], within, 0, 0, 0);
#pragma unroll
                for (int k = 0; k < N32; ++k) before = __builtin_amdgcn_mfma_f32_16x16x32_f16(rows_of(s_lds, t, k), c[k], before, 0, 0, 0);
                const f4 unit = *reinterpret_cast<const f4*>(&s_unit[16 * t + 4 * high]);
                // channels 16 t + 4 high + r of row i
                const int piece = 2 * t + (high >> 1);
                const h4 x = *reinterpret_cast<const h4*>(x_now + i * 128 + ((piece ^ ((i >> 1) & 7)) * 16) + (high & 1) * 8);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float v = __builtin_fmaf(before[r], unit[r] * row_decay, within[r] * row_unit);
                    if (a.d) v = __builtin_fmaf(skip, (float)x[r], v);
                    y[t][r] = v;
                }
            }
        }
        __syncthreads();
        if (rows > 1 && uniform(odd_x)) {
            // again, row by row; S is as it was
            __syncthreads();
            careful_until = now.row + rows;
            if (new_sequence) {
                // (its chunks are counted again when it is entered again)
                budget += (next.end - next.row + kChunk - 1) / kChunk;
            }
            rows = 1;
            if (tid == 0) odd_x = 0;
            UNIQL_WAIT_ALL_LOADS();  // the next chunk's tile, which is not the next one any more
            fetch(now.row, 1, b_next, x_next);
            if constexpr (LAST) fetch_c(now.row, 1);
            const float dt = load_dt(now.row, 1);
            if (wave == 0) row_values(dt, 1, next_values);
            return true;
        }
        if constexpr (LAST) {
            const int i = 16 * wave + low;
            if (i < rows) {
                half_t* const to = y_base + (int64_t)(now.row + i) * a.y_row;
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const int p = 16 * t + 4 * high;
                    const h4 v = {(half_t)y[t][0], (half_t)y[t][1], (half_t)y[t][2], (half_t)y[t][3]};
                    if (p + 4 <= head_dim) *reinterpret_cast<h4_any*>(to + p) = h4_any{v[0], v[1], v[2], v[3]};
                    else
#pragma unroll
                        for (int r = 0; r < 3; ++r)
                            if (p + r < head_dim) to[p + r] = v[r];
                }
            }
            if (more) fetch_c(next.row, next_rows);
        }
        // the state behind the chunk
        {
            const float decay = now_values.decay[kChunk - 1];
            const float keep = decay * (unit_s * (1.0f / unit_x));
            if constexpr (!LAST) segment_log += (double)now_values.log_hi[kChunk - 1] + (double)now_values.log_lo[kChunk - 1];
            unit_s = unit_x;
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
                S[t] *= keep;
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const h8 b = columns_of(b_now, t, k, false);
                    S[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b, into_hi[k], S[t], 0, 0, 0);
                    S[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b, into_lo[k], S[t], 0, 0, 0);
                }
            }
        }
        if constexpr (LAST) {
            if (now.row + rows == now.q.first + now.q.rows && a.state_out) store_state(now.q.place);
        }
        if (!more) return false;
        if (new_sequence) first_state(next, false);
        if constexpr (LAST) leave_copy();
        if (wave == 0) row_values(next_dt, next_rows, next_values);
        now = next;
        rows = next_rows;
        return true;
    };
    while (true) {
        if (!chunk(b_even, x_even, b_odd, x_odd, values[0], values[1])) break;
        if (!chunk(b_odd, x_odd, b_even, x_even, values[1], values[0])) break;
    }
    if constexpr (!LAST) {
#pragma unroll
        for (int t = 0; t < kTiles; ++t) added[place * kHeld + t * kScanThreads + tid] = S[t] * unit_s;
        if (tid == 0) faded[place] = (float)exp2(segment_log);
    }
}

// 512 workgroups keep the chip's 256 compute units busy, two each.
static int segments_of(int rows, int count, int units) {
    const int64_t chunks = rows / kChunk + (count < rows ? count : rows);
    int64_t n = 512 / units;
    if (n > chunks / 4) n = chunks / 4;
    return n < 1 ? 1 : (int)n;
}
static int tiles_of(int states) { return states <= 64 ? 4 : (states <= 96 ? 6 : (states <= 128 ? 8 : (states <= 192 ? 12 : 16))); }

size_t state_space_scan_needs(int rows, int count, int heads, int head_dim, int states) {
    const int units = heads * ((head_dim + 63) / 64), segments = segments_of(rows, count, units);
    return (size_t)(segments - 1) * units * ((size_t)2 * tiles_of(states) * kScanThreads * sizeof(f4) + sizeof(float));
}

template <int N32>
static int go(const ScanArgs& a, bool through, hipStream_t stream) {
    const dim3 block(kScanThreads), first((unsigned)(a.heads * a.head_blocks), (unsigned)(a.segments - 1)),
        last((unsigned)(a.heads * a.head_blocks), (unsigned)a.segments);
    if (a.segments > 1) {
        if (through) hipLaunchKernelGGL((state_space_scan_kernel<N32, true, false>), first, block, 0, stream, a);
        else hipLaunchKernelGGL((state_space_scan_kernel<N32, false, false>), first, block, 0, stream, a);
    }
    if (through) hipLaunchKernelGGL((state_space_scan_kernel<N32, true, true>), last, block, 0, stream, a);
    else hipLaunchKernelGGL((state_space_scan_kernel<N32, false, true>), last, block, 0, stream, a);
    return hipGetLastError() == hipSuccess ? UNIQL_OK : UNIQL_E_LAUNCH;
}

int state_space_scan_launch(const ScanArgs& args, hipStream_t stream) {
    ScanArgs a = args;
    a.head_blocks = (a.head_dim + 63) / 64;
    a.segments = segments_of(a.sequences.rows, a.sequences.count, a.heads * a.head_blocks);
    // straight to LDS: pieces at multiples of 4 bytes, whole ones of b, 64 rows below 2^31 bytes
    const int64_t far = 1LL << 23, strides = a.x_row | a.x_head | a.b_row | a.b_group;
    const uintptr_t bases = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.b);
    const bool near = a.x_row >= 8 && a.b_row >= a.states && a.x_row <= far && a.b_row <= far;
    const bool through = !(near && (strides & 1) == 0 && (bases & 3) == 0 && a.states % 8 == 0);
    switch (tiles_of(a.states)) {
        case 4: return go<2>(a, through, stream);
        case 6: return go<3>(a, through, stream);
        case 8: return go<4>(a, through, stream);
        case 12: return go<6>(a, through, stream);
        default: return go<8>(a, through, stream);
    }
}

}  // namespace uniql
