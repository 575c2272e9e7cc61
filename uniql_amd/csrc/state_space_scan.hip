// Linear attention with a decay for each head over packed prompts: S_t = exp(l_t) S_{t-1} + s_t x_t b_t^T, y_t = S_t c_t + d x_t,
// with the time step s_t = softplus(dt_t + bias) and l_t = s_t a, for each head's matrix S [head_dim][states].
//
// Chunks of 64 rows: with L_i the sum of l up to row i of the chunk,
//   y_i = exp(L_i) S c_i + sum_{j <= i} exp(L_i - L_j) s_j (b_j . c_i) x_j + d x_i,      S' = exp(L_63) S + sum_j exp(L_63 - L_j) s_j x_j b_j^T,
// all four products on matrix instructions (16 x 16 x 32).  A workgroup walks through the chunks of one head with b and x in LDS, the next chunk's
// on their way meanwhile.  Nine waves: one loads, four have the outputs, sixteen rows i each
// - their c stays in registers, and the weights of the third product come out of the first one where the matrix instruction wants them
// (the scores transposed, as b c^T) - and four have the state, sixteen channels each, in registers; these leave a rounded copy in LDS for the
// next chunk's second product.  All work at a chunk side by side and meet once a chunk.
//
// Sequences of any lengths are cut into segments of equally many chunks, from the offsets on the device.  Where there are several, a
// first launch walks through what lies in front of the last segment for the state alone, in smaller pieces: what each adds to
// the state of the sequence that goes on behind it, and the decay over it.  The second launch puts them together where a segment begins
// within a sequence.
//
// Bound by latency within a chunk.  Of its 5900 clocks (counters of the second launch, 16384 tokens of 128 heads of 64, 8 groups of 128 states) a SIMD
// has 2400 of vector instructions and 1000 of matrix instructions, LDS 2000 (320 of them bank conflicts); a request to L2 takes 560, and waves
// wait in 54 % of their cycles, for each other, for LDS and for loads.  397 us in two launches (the first one 78), 1.6 TB/s and 0.4 PFLOP/s of
// matrix instructions.  Rows of 20480 bytes share few sets of the first cache: 256 bytes longer the call takes 390 us on a card where it takes 443.
// 4096 tokens of 256 states 207 us (9200 clocks a chunk: 3400, 2000 and 3400); 333 tokens 18.8, six chunks of 2.4 us each behind a launch.
// Tried and taken out, against 390 us: two heads that share b and c in a workgroup of sixteen waves (128 registers each: operands cannot be asked
// for ahead, 430 to 460), one set of four waves for everything with two workgroups a compute unit (530), more segments (530).
//
// S, all sums and the decays are fp32, L is summed up in 64 bits (its differences matter, also behind a token that wipes the state).
// Rounded to fp16 are the weights and S for the outputs, which are fp16 themselves (distance from 64 bits 2.2e-4 to 2.5e-4 of the outputs, 2.1e-4
// where only they are rounded; two fp16 numbers for each would double the second and third products and their reads).  Both are relative to the
// largest of their row: none overflows, and what is below 2^-28 of that one loses digits, below 2^-39 itself, which shows only where x or c is zero
// at the largest.  What goes into S is split into two fp16 numbers, 22 bits.  An infinity or NaN in x must not reach rows in front of it, also as
// zero times it: where a result shows one, such values are taken out of the product and added on their own.
#include <type_traits>

#include "state_space.hpp"

namespace uniql {

constexpr int kChunk = 64;
typedef __attribute__((address_space(3))) void* lds_ptr;
typedef __attribute__((address_space(3))) char* lds_bytes;
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s4* lds_s4_ptr;

#define UNIQL_WAIT_ALL_LOADS() __builtin_amdgcn_s_waitcnt(0x0F70)  // vmcnt(0), the other counters left alone (gfx9 encoding)

__device__ __forceinline__ h8 join(s4 lo, s4 hi) { return __builtin_bit_cast(h8, s8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}); }
__device__ __forceinline__ h4 round_four(float a, float b, float c, float d) {
    const h2 lo = __builtin_convertvector((f2{a, b}), h2), hi = __builtin_convertvector((f2{c, d}), h2);
    return h4{lo[0], lo[1], hi[0], hi[1]};
}
__device__ __forceinline__ float power_of_two(int e) { return __builtin_bit_cast(float, (127 + e) << 23); }  // -126 <= e <= 127
__device__ __forceinline__ int exponent_of(float v) { return (int)((__builtin_bit_cast(uint32_t, v) >> 23) & 255u) - 127; }
__device__ __forceinline__ int clamp_to(int v, int low, int high) { return v < low ? low : (v > high ? high : v); }
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
template <typename T>
__device__ __forceinline__ T* uniform(T* p) {
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    return reinterpret_cast<T*>((uint64_t)(unsigned)uniform((int)(v >> 32)) << 32 | (unsigned)uniform((int)v));
}
// The largest size among eight values (NaN counts as nothing).
__device__ __forceinline__ float largest_of(h8 v) {
    const u32x4 w = __builtin_bit_cast(u32x4, v) & 0x7fff7fffu;
    h2 a = bits_to_h2(w[0]), b = bits_to_h2(w[1]);
    a = __builtin_elementwise_max(a, bits_to_h2(w[2]));
    b = __builtin_elementwise_max(b, bits_to_h2(w[3]));
    a = __builtin_elementwise_max(a, b);
    return fmaxf((float)a[0], (float)a[1]);
}
// Of values that are zero or NaN.
__device__ __forceinline__ bool all_zero(h8 v) {
    const h2 s = (h2{v[0], v[1]} + h2{v[2], v[3]}) + (h2{v[4], v[5]} + h2{v[6], v[7]});
    return (float)s[0] + (float)s[1] == 0.f;
}
__device__ __forceinline__ bool finite(half_t v) { return __builtin_fabsf16(v) < (half_t)INFINITY; }

// What is known of a chunk's rows before its products: the logarithms L (base 2) of the decay up to each row, rounded to floats; their
// rests r as factors, 2^r, and the time steps with the same taken off, s 2^-r: exp2(L_i - L_j) of the rounded ones times both is off by
// the roundings of the difference (2^-24 of it) and of the three exponentials alone; what a row adds to the state (its time step, faded), and
// the decays.
struct RowValues {
    float log[kChunk], rest[kChunk], step[kChunk], into[kChunk], decay[kChunk];
    float unit, per_unit;  // of `into`, a power of two, and its inverse
    double all;            // the last row's logarithm
};

// Chunks in all sequences.  Rows that belong to one sequence at most make no more than a chunk each 64 and one a sequence: more come of offsets
// that fall and rise again, whose walk would take as long as they like.  Such a call does nothing.
__device__ __forceinline__ int count_chunks(const Sequences& all) {
    const int lane = threadIdx.x & 63;
    int total = 0;
    for (int base = 0; base < all.count; base += 64) {
        const int s = base + lane;
        const int mine = s < all.count ? (sequence_of(all, s).rows + kChunk - 1) / kChunk : 0;
        total += __builtin_amdgcn_readlane(sums_upto(mine), 63);
        if (total > all.rows / kChunk + all.count) return 0;
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
// The first chunk of a piece, and the piece that a chunk belongs to.
__device__ __forceinline__ int border(int piece, int pieces, int chunks) { return (int)((int64_t)piece * chunks / pieces); }
__device__ __forceinline__ int piece_of(int chunk, int pieces, int chunks) { return (int)((((int64_t)chunk + 1) * pieces - 1) / chunks); }

// LDS holds a row's 16-byte pieces exchanged by its number, so that neither kind of read meets itself in a bank: the transposing ones take two
// neighbouring pieces of eight rows at once, the others a piece of the rows 0 to 3 and 12 to 15 with the next piece of the rows 4 to 11.
template <int PIECES>
__device__ __forceinline__ int exchange(int row) {
    if (PIECES == 8) return 2 * (((row >> 1) & 3) ^ ((row >> 2) & 2)) | ((row >> 3) & 1);
    return 2 * ((row & 7) ^ ((row >> 1) & 4)) | ((row >> 3) & 1);
}
// 16 bytes a lane from a buffer, at a lane's and a common offset, straight to the KiB at `to`; zeros where they lie beyond it.
__device__ __forceinline__ void buffer_to_lds(const half_t* buffer, unsigned bytes, lds_bytes to, unsigned lane_at, unsigned at) {
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<half_t*>(buffer), 0, bytes, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr)to, 16, lane_at, at, 0, 0);
}
// A tile of 64 rows to LDS, rows of PIECES pieces there, by OF waves; rows behind the chunk and pieces behind the width come as zeros.
template <bool THROUGH, int PIECES, int OF>
__device__ __forceinline__ void fetch_tile(const half_t* tile, int64_t stride, int width, int rows, int wave, lds_bytes to) {
    constexpr int kAtOnce = 64 / PIECES, kSet = kAtOnce * OF;  // rows of a wave's access, and of all
    const int lane = threadIdx.x & 63, part_row = wave * kAtOnce + lane / PIECES, part = lane % PIECES;
    if constexpr (THROUGH) {
#pragma unroll 1
        for (int row = part_row; row < kChunk; row += kSet) {
            const int piece = part ^ exchange<PIECES>(row);
            h8 v = {};
            if (row < rows && piece * 8 < width) v = load_halves(tile + row * stride + piece * 8, width - piece * 8);
            *(__attribute__((address_space(3))) h8*)(to + row * (PIECES * 16) + part * 16) = v;
        }
    } else {
        // (rows and pieces that are not there lie beyond the buffer)
        const unsigned bytes = 2u * ((unsigned)(rows - 1) * (unsigned)stride + (unsigned)width);
        // (pieces are exchanged over 16 rows: alike in accesses that lie so far apart)
        constexpr int kCycle = kSet < 16 ? 16 / kSet : 1;
        const unsigned step = (unsigned)uniform((int)stride);
        unsigned at[kCycle];
#pragma unroll
        for (int i = 0; i < kCycle; ++i) {
            const int row = i * kSet + part_row, piece = part ^ exchange<PIECES>(row);
            at[i] = piece * 8 < width ? 2u * (unsigned)row * step + 16u * piece : 0x80000000u;
        }
#pragma unroll
        for (int i = 0; i < kChunk / kSet; ++i)
            buffer_to_lds(tile, bytes, to + (i * kSet + wave * kAtOnce) * (PIECES * 16), at[i % kCycle],
                          (unsigned)(i / kCycle * kCycle * kSet * 2) * step);
    }
}

// Where a lane reads of the tiles, in bytes from their first one.
struct Reads {
    int rows, b_columns, x_columns;
};

// The call's arguments anew from memory, for code that is rarely run: kept over the walk they would be written to lanes of vector registers
// and read back in every chunk.
typedef const ScanArgs __attribute__((address_space(4)))* ArgsAgain;
__device__ __forceinline__ ArgsAgain args_again() {
    ArgsAgain p = (ArgsAgain)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return p;
}
__device__ __forceinline__ Sequences sequences_again(ArgsAgain p) {
    return {p->sequences.cu, p->sequences.starts, p->sequences.places, p->sequences.count, p->sequences.pool, p->sequences.rows,
            p->sequences.only};
}

// Who asks for the tiles.  For outputs over up to 128 states waves of their own, one, or four where the values pass through their registers: asking
// takes some 2400 clocks a chunk, in which a wave of the others would not do its work (16384 tokens 430 -> 375 us).  Otherwise those three
// waves of the state that do not work out row values: a ninth wave would leave 168 registers to each, too few for more states (4096 tokens with
// 256 states 141 -> 171 us), and the first launch has more workgroups a compute unit without it (16384 tokens 130 -> 85 us).
constexpr int loading_waves(int n32, bool through, bool last) { return last && n32 <= 4 ? (through ? 4 : 1) : 0; }
constexpr int scan_waves(int n32, bool through, bool last) { return (last ? 8 : 4) + loading_waves(n32, through, last); }

// N32: the states in units of 32; THROUGH: rows that cannot go straight to LDS; LAST: the second launch, or the only one.
template <int N32, bool THROUGH, bool LAST>
__global__ __launch_bounds__(64 * scan_waves(N32, THROUGH, LAST), !LAST && N32 <= 4 ? 3 : 1) void state_space_scan_kernel(const ScanArgs a) {
    constexpr int kPieces = N32 <= 2 ? 8 : (N32 <= 4 ? 16 : 32);  // 16-byte pieces of a row of b in LDS
    constexpr int kRowBytes = kPieces * 16, kTileBytes = kChunk * kRowBytes, kXBytes = kChunk * 128;
    constexpr int kTiles = 2 * N32;                               // of sixteen states
    constexpr int kLoading = loading_waves(N32, THROUGH, LAST);
    constexpr int kCopyBytes = LAST ? kTileBytes : 16;
    // Each in variables of its own, which tells the compiler that reading one does not wait for what is on its way into another.
    __shared__ __attribute__((aligned(16))) char b_even[kTileBytes], b_odd[kTileBytes];
    __shared__ __attribute__((aligned(16))) char x_even[kXBytes], x_odd[kXBytes];
    __shared__ __attribute__((aligned(16))) char s_even[kCopyBytes], s_odd[kCopyBytes];
    __shared__ __attribute__((aligned(16))) float s_unit[2][kChunk];
    __shared__ __attribute__((aligned(16))) RowValues values[2];
    const int tid = threadIdx.x, lane = tid & 63, low = lane & 15, high = lane >> 4, all_wave = uniform(tid >> 6);
    const int wave = all_wave % 4, role = all_wave / 4;
    const bool has_state = role == 0, loads = role == 2;

    // neighbouring workgroups, which are on different XCDs, have heads of different groups: those of one group share an L2
    const int units = a.heads * a.head_blocks;
    const int unit = units % 8 == 0 ? (int)(blockIdx.x % 8) * (units / 8) + (int)(blockIdx.x / 8) : (int)blockIdx.x, head = unit / a.head_blocks, p0 = unit % a.head_blocks * 64;
    // a segment is one piece in the first launch, several in the second
    const int all_pieces = a.segments * a.pieces, piece0 = LAST ? (int)blockIdx.y * a.pieces : (int)blockIdx.y;
    const int chunks = uniform(count_chunks(a.sequences));
    const int begin = border(piece0, all_pieces, chunks), end = border(piece0 + (LAST ? a.pieces : 1), all_pieces, chunks);
    if (begin >= end) return;

    const int head_dim = a.head_dim - p0;  // (from p0 on; a head may be wider than the 64 of a set of waves)
    const int group = head / a.share, states = a.states;

    // what the first launch leaves: for each piece and each unit, in the registers' order - what it adds, and the states that
    // sequences begin with; then the decays over pieces
    constexpr int kHeld = kTiles * 256;  // vectors of four
    auto held_all = [&](ArgsAgain k) __attribute__((always_inline)) { return (int64_t)(k->segments - 1) * k->pieces * units * kHeld; };
    auto held_at = [&](int piece) __attribute__((always_inline)) { return ((int64_t)piece * units + unit) * kHeld + wave * 64 + lane; };

    // The sequence, its chunks in front of this segment, and how many chunks are left.
    int index, offset, budget = end - begin;
    if constexpr (LAST) {
        index = uniform(find_chunk(a.sequences, begin, offset));
    } else {
        // what goes on behind the piece's last chunk
        int last_offset;
        index = uniform(find_chunk(a.sequences, end - 1, last_offset));
        last_offset = uniform(last_offset);
        if ((last_offset + 1) * kChunk >= sequence_of(a.sequences, index).rows) return;  // nothing
        offset = last_offset + 1 < budget ? 0 : last_offset + 1 - budget;
        budget = last_offset + 1 - offset;
    }
    offset = uniform(offset);

    // ---- loads ----------------------------------------------------------------------------------------------------------
    auto swap_of = [&](int row) __attribute__((always_inline)) { return exchange<kPieces>(row); };
    const int x_width = uniform(head_dim < 64 ? head_dim : 64);
    // Where the next tile is.
    struct Tiles {
        const half_t *b, *x;
        int64_t b_stride, x_stride;
    };
    auto tiles_at = [&](int row) __attribute__((always_inline)) {
        const ArgsAgain k = args_again();
        return Tiles{k->b + (int64_t)row * k->b_row + group * k->b_group, k->x + (int64_t)row * k->x_row + head * k->x_head + p0, k->b_row, k->x_row};
    };
    auto fetch = [&](Tiles& tiles, int rows, lds_bytes b_to, lds_bytes x_to) __attribute__((always_inline)) {
        // (a buffer that the compiler does not take for the same in all lanes costs a loop over the lanes for each access)
        rows = uniform(rows);
        if constexpr (kLoading > 0) {
            fetch_tile<THROUGH, 8, kLoading>(uniform(tiles.x), tiles.x_stride, x_width, rows, wave, x_to);
            fetch_tile<THROUGH, kPieces, kLoading>(uniform(tiles.b), tiles.b_stride, states, rows, wave, b_to);
        } else {
            if (wave == 1) fetch_tile<THROUGH, 8, 1>(uniform(tiles.x), tiles.x_stride, x_width, rows, 0, x_to);
            if (wave >= 2) fetch_tile<THROUGH, kPieces, 2>(uniform(tiles.b), tiles.b_stride, states, rows, wave - 2, b_to);
        }
        tiles.b += rows * tiles.b_stride;
        tiles.x += rows * tiles.x_stride;
    };
    // Chunks of the rows row .. last, by the loading waves, always one ahead.
    auto walk_loads = [&](int row, int last) __attribute__((always_inline)) {
        Tiles tiles = tiles_at(row);
        bool odd = false;
        while (true) {
            const int rows = last - row < kChunk ? last - row : kChunk;
            if (odd) fetch(tiles, rows, (lds_bytes)b_odd, (lds_bytes)x_odd);
            else fetch(tiles, rows, (lds_bytes)b_even, (lds_bytes)x_even);
            row += rows;
            odd = !odd;
            UNIQL_WAIT_ALL_LOADS();
            __syncthreads();
            if (row >= last) break;
        }
    };

    // ---- reads of LDS ---------------------------------------------------------------------------------------------------
    // Pieces are numbers of four (rows) or two (columns) more bits than what a lane has of its own, and exchanging them is an exclusive or
    // with the row's number: the next piece's address is the first one's, exclusive or the piece.  The first ones are worked out in each chunk.
    auto reads = [&]() __attribute__((always_inline)) {
        const int tr_row = 4 * high + (low >> 2), part = (low >> 1) & 1;
        Reads r = {low * kRowBytes + (high ^ swap_of(low)) * 16, tr_row * kRowBytes + (part ^ swap_of(tr_row)) * 16 + (low & 1) * 8,
                   tr_row * 128 + (part ^ exchange<8>(tr_row)) * 16 + (low & 1) * 8};
        asm volatile("" : "+v"(r.rows), "+v"(r.b_columns), "+v"(r.x_columns));
        return r;
    };
    // rows 16 t + low, states 32 k + 8 high .. + 7
    auto rows_of = [&](const char* tile, const Reads& r, int t, int k) __attribute__((always_inline)) {
        return *reinterpret_cast<const h8*>(tile + (r.rows ^ (64 * k)) + t * 16 * kRowBytes);
    };
    // column 16 t + low of rows 32 k + 4 high .. + 3 and 32 k + 16 + 4 high .. + 3: a lane reads four columns of one row, and sixteen lanes
    // exchange them
    auto columns_of = [&](const char* tile, const Reads& r, int t, int k, auto is_x) __attribute__((always_inline)) {
        constexpr bool kIsX = decltype(is_x)::value;
        constexpr int bytes = kIsX ? 128 : kRowBytes;
        const char* const at = tile + ((kIsX ? r.x_columns : r.b_columns) ^ (32 * t)) + 32 * k * bytes;
        return join(__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_ptr)(const_cast<char*>(at))),
                    __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_ptr)(const_cast<char*>(at) + 16 * bytes)));
    };
    constexpr std::true_type of_x{};
    constexpr std::false_type of_b{};

    // ---- outputs --------------------------------------------------------------------------------------------------------
    // Chunks of the rows row .. last, by a wave for its rows 16 W .. + 15 of each, which see the rows of the tiles up to W.  The walk's barriers
    // are those of the waves for the state.
    auto walk_outputs = [&](auto slice, int row, int last) __attribute__((always_inline)) {
        constexpr int W = decltype(slice)::value;
        const ArgsAgain k0 = args_again();
        const int64_t c_stride = k0->c_row, y_stride = k0->y_row;
        // Four neighbouring lanes have a row of c or y in memory; the products want c of row low and give y of row low, so both change lanes.
        // (With a row for each of sixteen neighbouring lanes instead, each lane's piece is an access of its own: 2710 a chunk and head, with
        // all that stands behind waiting, and now 960.)
        const int my_row = lane >> 2, my_part = lane & 3;
        // (a common address and a lane's distance from it, 32 bits of it where rows are near each other)
        auto distance = [&](int rows, int64_t stride, int more) __attribute__((always_inline)) {
            if constexpr (THROUGH) return rows * stride + more;
            else return (unsigned)(rows * (int)stride + more);
        };
        const half_t* c_tile = k0->c + (int64_t)(row + 16 * W) * c_stride + group * k0->c_group;
        half_t* y_tile = k0->y + (int64_t)(row + 16 * W) * y_stride + head * k0->y_head + p0;
        auto from_lane = [&](uint32_t v, int from) __attribute__((always_inline)) { return (uint32_t)__builtin_amdgcn_ds_bpermute(4 * from, (int)v); };
        const bool has_skip = k0->d != nullptr;
        const float skip = has_skip ? k0->d[head] : 0.f;
        h8 c[N32];
        // (rows behind the chunk read its last one: their results are not stored)
        auto fetch_c = [&](int rows) __attribute__((always_inline)) {
            // (W's rows may all lie behind the chunk: its last row then)
            const int last_row = rows - 1 - 16 * W;
            const half_t* const from = uniform(c_tile + (last_row < 0 ? last_row * c_stride : 0)) +
                                       distance(my_row < last_row ? my_row : (last_row < 0 ? 0 : last_row), c_stride, 8 * my_part);
            if (!THROUGH && states == 32 * N32) {
#pragma unroll
                for (int k = 0; k < N32; ++k) c[k] = load_halves(from + 32 * k, 8);
            } else {
                int n0 = 8 * my_part;
                asm volatile("" : "+v"(n0));  // (comparisons are not kept over the walk, where their masks would fill the scalar registers)
#pragma unroll
                for (int k = 0; k < N32; ++k) {
                    const int n = 32 * k + n0;
                    if constexpr (THROUGH) {
                        c[k] = load_halves(from + 32 * k, states - n);
                    } else {
                        const h8 v = load_halves(from + (n < states ? 32 * k : -n0), 8);  // (behind the states: the row's first ones, unused)
                        c[k] = n < states ? v : h8{};
                    }
                }
            }
            c_tile += rows * c_stride;
        };
        auto place_c = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int k = 0; k < N32; ++k) {
                u32x4 w = __builtin_bit_cast(u32x4, c[k]);
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = from_lane(w[e], 4 * low + high);
                c[k] = __builtin_bit_cast(h8, w);
            }
        };
        // A chunk's outputs are stored while the next one is under way: a store that has just been issued is not waited for.
        h4 held[4];
        int held_rows = 0;
        auto store_outputs = [&]() __attribute__((always_inline)) {
            half_t* const to = uniform(y_tile) + distance(my_row, y_stride, 4 * my_part);
            const bool there = 16 * W + my_row < held_rows;
            if (there && head_dim >= 64) {
#pragma unroll
                for (int t = 0; t < 4; ++t) *reinterpret_cast<h4_any*>(to + 16 * t) = h4_any{held[t][0], held[t][1], held[t][2], held[t][3]};
            } else if (there) {
                int first = 4 * my_part;
                asm volatile("" : "+v"(first));
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const int p = 16 * t + first;
                    const h4 v = held[t];
                    if (p + 4 <= head_dim) *reinterpret_cast<h4_any*>(to + 16 * t) = h4_any{v[0], v[1], v[2], v[3]};
                    else
#pragma unroll
                        for (int r = 0; r < 3; ++r)
                            if (p + r < head_dim) to[16 * t + r] = v[r];
                }
            }
            y_tile += held_rows * y_stride;
        };
        auto place_outputs = [&]() __attribute__((always_inline)) {
            typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const u32x2 w = __builtin_bit_cast(u32x2, held[t]);
                held[t] = __builtin_bit_cast(h4, u32x2{from_lane(w[0], 16 * my_part + (lane >> 2)), from_lane(w[1], 16 * my_part + (lane >> 2))});
            }
        };
        auto chunk = [&](const char* b_now, const char* x_now, const char* s_now, const float* unit, const RowValues& now) __attribute__((always_inline)) {
            __syncthreads();
            store_outputs();
            const int rows = last - row < kChunk ? last - row : kChunk, next_rows = last - row - rows < kChunk ? last - row - rows : kChunk;
            const Reads at = reads();
            int i = 16 * W + low;
            asm volatile("" : "+v"(i));
            // weights of rows j (16 t + 4 high + r) for row i
            f4 m[W + 1];
#pragma unroll
            for (int t = 0; t <= W; ++t) m[t] = f4{};
            // The products' operands are asked for kAhead steps of four instructions in front of them: N32 steps of the first one, N32 of the
            // second, kSteps of the third.
            constexpr int kSteps = W / 2 + 1, kAhead = 2, kAll = 2 * N32 + kSteps;
            h8 operand[kAhead + 1][4];
            auto ask = [&](int step) __attribute__((always_inline)) {
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    if (step < N32 && t <= W) operand[step % (kAhead + 1)][t] = rows_of(b_now, at, t, step);
                    if (step >= N32 && step < 2 * N32) operand[step % (kAhead + 1)][t] = rows_of(s_now, at, t, step - N32);
                    if (step >= 2 * N32 && step < kAll) operand[step % (kAhead + 1)][t] = columns_of(x_now, at, t, step - 2 * N32, of_x);
                }
                __builtin_amdgcn_sched_barrier(0);
            };
#pragma unroll
            for (int step = 0; step < kAhead; ++step) ask(step);
#pragma unroll
            for (int k = 0; k < N32; ++k) {
                ask(k + kAhead);
#pragma unroll
                for (int t = 0; t <= W; ++t) m[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(operand[k % (kAhead + 1)][t], c[k], m[t], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
            f4 before[4], within[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) before[t] = within[t] = f4{};
#pragma unroll
            for (int k = 0; k < N32; ++k) {
                ask(N32 + k + kAhead);
#pragma unroll
                for (int t = 0; t < 4; ++t) before[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(operand[(N32 + k) % (kAhead + 1)][t], c[k], before[t], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (next_rows > 0) fetch_c(next_rows);
            const float log = now.log[i], row_decay = now.decay[i];
            float top = 0.f;
#pragma unroll
            for (int t = 0; t <= W; ++t) {
                const int j = 16 * t + 4 * high;
                const f4 from = *reinterpret_cast<const f4*>(&now.log[j]), step = *reinterpret_cast<const f4*>(&now.step[j]);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float w = m[t][r] * (__builtin_amdgcn_exp2f(log - from[r]) * step[r]);
                    if (t == W) w = j + r <= i ? w : 0.f;
                    m[t][r] = w;
                    top = fmaxf(top, fabsf(w));
                }
            }
            const int e = clamp_to(exponent_of(max_of_sixteenths(top)), -100, 127);
            const float up = power_of_two(14 - e), row_unit = power_of_two(e - 14) * now.rest[i];
            h8 weight[kSteps];  // of 32 rows j each
#pragma unroll
            for (int t = 0; t < 2 * kSteps; ++t) {
                const h4 v = t <= W ? round_four(m[t <= W ? t : 0][0] * up, m[t <= W ? t : 0][1] * up, m[t <= W ? t : 0][2] * up, m[t <= W ? t : 0][3] * up) : h4{};
#pragma unroll
                for (int r = 0; r < 4; ++r) weight[t >> 1][4 * (t & 1) + r] = v[r];
            }
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
#pragma unroll
                for (int t = 0; t < 4; ++t) within[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(operand[(2 * N32 + k) % (kAhead + 1)][t], weight[k], within[t], 0, 0, 0);
            }
            // channels 16 t + 4 high + r of row i
            auto finish = [&](int t, f4 sum) __attribute__((always_inline)) {
                const f4 of_s = *reinterpret_cast<const f4*>(&unit[16 * t + 4 * high]);
#pragma unroll
                for (int r = 0; r < 4; ++r) sum[r] = __builtin_fmaf(before[t][r], of_s[r] * row_decay, sum[r] * row_unit);
                return sum;
            };
            auto x_of = [&](int t, int row) __attribute__((always_inline)) {
                const int piece = 2 * t + (high >> 1);
                return *reinterpret_cast<const h4*>(x_now + row * 128 + ((piece ^ exchange<8>(row)) * 16) + (high & 1) * 8);
            };
            f4 y[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) y[t] = finish(t, within[t]);
            if (has_skip) {
                asm volatile("");  // (a branch for all, not a choice for each)
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const h4 x = x_of(t, i);
#pragma unroll
                    for (int r = 0; r < 4; ++r) y[t][r] = __builtin_fmaf(skip, (float)x[r], y[t][r]);
                }
            }
#pragma unroll
            for (int t = 0; t < 4; ++t) held[t] = round_four(y[t][0], y[t][1], y[t][2], y[t][3]);
            h8 zero = {};
#pragma unroll
            for (int t = 0; t < 4; t += 2) zero = __builtin_elementwise_fma(h8{held[t][0], held[t][1], held[t][2], held[t][3], held[t + 1][0], held[t + 1][1], held[t + 1][2], held[t + 1][3]}, h8{}, zero);
            if (__any(!all_zero(zero))) {
                // again, without values that are no numbers, which are then added to the rows that see them
                asm volatile("");
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    f4 sum = {};
#pragma unroll
                    for (int k = 0; k < kSteps; ++k) {
                        h8 x = columns_of(x_now, at, t, k, of_x);
#pragma unroll
                        for (int j = 0; j < 8; ++j) x[j] = finite(x[j]) ? x[j] : (half_t)0.f;
                        sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, weight[k], sum, 0, 0, 0);
                    }
#pragma unroll 1
                    for (int j = 0; j < 16 * (W + 1); ++j) {
                        // row j's weight for each row i: element 4 (j / 16 % 2) + j % 4 of step j / 32, of the lane j / 4 % 4 sixteens on
                        half_t w = weight[0][0];
#pragma unroll
                        for (int q = 0; q < 8 * kSteps; ++q) w = (j >> 5) * 8 + ((j >> 4) & 1) * 4 + (j & 3) == q ? weight[q >> 3][q & 7] : w;
                        const float of_j = __shfl((float)w, low + 16 * ((j >> 2) & 3), 64);
                        const h4 x = x_of(t, j);
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (j <= i && !finite(x[r])) sum[r] += of_j * (float)x[r];
                    }
                    sum = finish(t, sum);
                    const h4 x = x_of(t, i);
                    if (has_skip)
#pragma unroll
                        for (int r = 0; r < 4; ++r) sum[r] = __builtin_fmaf(skip, (float)x[r], sum[r]);
                    held[t] = round_four(sum[0], sum[1], sum[2], sum[3]);
                }
            }
            place_outputs();
            if (next_rows > 0) place_c();
            held_rows = rows;
            row += rows;
        };
        fetch_c(last - row < kChunk ? last - row : kChunk);
        place_c();
        while (true) {
            chunk(b_even, x_even, s_even, s_unit[0], values[0]);
            if (row >= last) break;
            chunk(b_odd, x_odd, s_odd, s_unit[1], values[1]);
            if (row >= last) break;
        }
        store_outputs();
    };

    // ---- the state ------------------------------------------------------------------------------------------------------
    auto walk_state = [&](const Sequence& q, int row, int last) __attribute__((always_inline)) {
        const ArgsAgain k0 = args_again();
        const int64_t dt_stride = k0->dt_row;
        const half_t* dt_row = k0->dt + (int64_t)(row + lane) * dt_stride + head;
        const float rate = k0->a[head], bias = k0->dt_bias ? k0->dt_bias[head] : 0.f, dt_min = k0->dt_min, dt_max = k0->dt_max;
        const int softplus = k0->softplus;
        const bool has_rows = wave == 0;
        auto load_dt = [&](int rows) __attribute__((always_inline)) {
            const half_t dt = dt_row[-(lane < rows ? 0 : lane - rows + 1) * dt_stride];
            dt_row += rows * dt_stride;
            return dt;
        };
        // One wave works out a chunk's row values, a row a lane.
        auto row_values = [&](half_t dt, int rows, RowValues& to) __attribute__((always_inline)) {
            const float step = lane < rows ? time_step((float)dt, bias, softplus, dt_min, dt_max) : 0.f;
            // (A row that fades by 2^-300 leaves nothing of any fp32 state, as one that fades by more: L of a chunk stays below 2^15, and its rest small.)
            double row_log = (double)step * (double)rate * 1.4426950408889634;
            row_log = row_log < -300.0 ? -300.0 : row_log;
            const double log = sums_upto(lane < rows ? row_log : 0.0);
            const double all = __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(log), 63), __builtin_amdgcn_readlane(__double2loint(log), 63));
            const float hi = (float)log, rest = (float)(log - (double)hi);
            const float into = lane < rows ? __builtin_amdgcn_exp2f((float)(all - log)) * step : 0.f;
            float most = max_of_sixteenths(into);
            most = fmaxf(most, dpp_from<0x140>(most));
            most = fmaxf(most, dpp_from<0x141>(most));
            most = fmaxf(most, dpp_from<0x4E>(most));
            most = fmaxf(most, dpp_from<0xB1>(most));
            const int e = clamp_to(exponent_of(most), -95, 100);
            to.log[lane] = hi;
            const float factor = __builtin_amdgcn_exp2f(rest);
            to.rest[lane] = factor;
            to.step[lane] = step * __builtin_amdgcn_exp2f(-rest);
            to.into[lane] = into * power_of_two(-1 - e);
            to.decay[lane] = __builtin_amdgcn_exp2f(hi) * factor;
            if (lane == 0) to.unit = power_of_two(e + 1), to.per_unit = power_of_two(-1 - e), to.all = all;
        };
        // Lane: channel 16 wave + low, states 16 t + 4 high + r, in units of `unit_s` (a power of two of the channel's own).
        f4 S[kTiles];
        float unit_s = 1.f;
        const int my_p = 16 * wave + low;
        const bool p_there = my_p < head_dim, quads = states % 4 == 0;
        auto pool_at = [&](ArgsAgain k) __attribute__((always_inline)) {
            return (((int64_t)q.place * k->heads + head) * k->head_dim + p0 + my_p) * states + 4 * high;
        };
        auto load_state = [&](ArgsAgain k) __attribute__((always_inline)) {
            const float* const from = k->state + pool_at(k);
            int n0 = 4 * high;
            asm volatile("" : "+v"(n0));
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
                const int n = 16 * t + n0;
                if (p_there && n < states) {
                    if (quads) S[t] = *reinterpret_cast<const f4*>(from + 16 * t);
                    else
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (n + r < states) S[t][r] = from[16 * t + r];
                }
            }
        };
        auto store_state = [&](ArgsAgain k) __attribute__((always_inline)) {
            float* const to = k->state_out + pool_at(k);
            int n0 = 4 * high;
            asm volatile("" : "+v"(n0));
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
                const int n = 16 * t + n0;
                if (p_there && n < states) {
                    const f4 v = S[t] * unit_s;
                    if (quads) *reinterpret_cast<f4*>(to + 16 * t) = v;
                    else
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (n + r < states) to[16 * t + r] = v[r];
                }
            }
        };
        // The copy for the next chunk's outputs.
        auto leave_copy = [&](char* s_next, float* unit) __attribute__((always_inline)) {
            float top = 0.f;
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) top = fmaxf(top, fabsf(S[t][r]));
            const int e = clamp_to(exponent_of(max_of_sixteenths(top)), -100, 127);
            const float up = power_of_two(14 - e);
            if (high == 0) unit[my_p] = power_of_two(e - 14) * unit_s;
            int to = my_p * kRowBytes + (((high >> 1) ^ swap_of(my_p)) * 16) + (high & 1) * 8;
            asm volatile("" : "+v"(to));
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
                *reinterpret_cast<h4*>(s_next + (to ^ (32 * t))) = round_four(S[t][0] * up, S[t][1] * up, S[t][2] * up, S[t][3] * up);
        };
        // The state where the workgroup comes upon the sequence: from earlier pieces, from the pool, or empty.
        {
            f4* const added = reinterpret_cast<f4*>(k0->temp);
            f4* const kept_first = added + held_all(k0);
#pragma unroll
            for (int t = 0; t < kTiles; ++t) S[t] = f4{};
            if (LAST && offset > 0) {
                const float* const faded = reinterpret_cast<const float*>(kept_first + held_all(k0));
                const int from = piece_of(begin - offset, all_pieces, chunks);
#pragma unroll 1
                for (int g = from; g < piece0; ++g) {
                    if (border(g, all_pieces, chunks) == border(g + 1, all_pieces, chunks)) continue;
                    const float fade = g == from ? 0.f : faded[(int64_t)g * units + unit];
#pragma unroll
                    for (int t = 0; t < kTiles; ++t) {
                        const f4 v = added[held_at(g) + t * 256];
                        S[t] = g == from ? v : S[t] * fade + v;
                    }
                }
            } else if (offset == 0 && k0->state && q.continued) {
                if (LAST && last < q.first + q.rows) {
                    // it goes on behind this segment, and the workgroup that comes to its end may have replaced the pool's
                    const int64_t at = held_at(piece_of(end - budget, all_pieces, chunks));
#pragma unroll
                    for (int t = 0; t < kTiles; ++t) S[t] = kept_first[at + t * 256];
                } else {
                    load_state(k0);
                    if constexpr (!LAST) {
#pragma unroll
                        for (int t = 0; t < kTiles; ++t) kept_first[held_at(piece0) + t * 256] = S[t];
                    }
                }
            }
        }
        // The largest finite size among a lane's channel's states, in their units.
        auto largest_state = [&]() __attribute__((always_inline)) {
            float top = 0.f;
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) top = fmaxf(top, fabsf(S[t][r]) < INFINITY ? fabsf(S[t][r]) : 0.f);
            return max_of_sixteenths(top);
        };
        // What the inverse of a chunk's units stays below as long as no finite state can pass fp32: one that the walk begins with, or one that it adds
        // up to (64 rows a chunk, time steps up to the longest, values of x and b below 2^16, 2^21 chunks).
        float room;
        {
            int most = exponent_of(fmaxf(fminf(65505.f + fabsf(bias), dt_max), dt_min)) + 61;
            if (offset > 0 || (k0->state && q.continued)) {
                float top = largest_state();
                top = fmaxf(top, dpp_from<0x140>(top));
                top = fmaxf(top, dpp_from<0x141>(top));
                top = fmaxf(top, dpp_from<0x4E>(top));
                top = fmaxf(top, dpp_from<0xB1>(top));
                const int e = uniform(exponent_of(top));
                most = e > most ? e : most;
            }
            room = power_of_two(125 - clamp_to(most, 0, 125));
        }
        double walk_log = 0.0;
        Tiles tiles = tiles_at(row);
        if constexpr (kLoading == 0) fetch(tiles, last - row < kChunk ? last - row : kChunk, (lds_bytes)b_even, (lds_bytes)x_even);
        auto chunk = [&](const char* b_now, const char* x_now, char* s_next, lds_bytes b_next, lds_bytes x_next, float* unit, const RowValues& now, RowValues& next) __attribute__((always_inline)) {
            if constexpr (kLoading == 0) UNIQL_WAIT_ALL_LOADS();
            __syncthreads();
            const int rows = last - row < kChunk ? last - row : kChunk, next_rows = last - row - rows < kChunk ? last - row - rows : kChunk;
            if constexpr (kLoading == 0)
                if (next_rows > 0) fetch(tiles, next_rows, b_next, x_next);
            half_t next_dt = (half_t)0.f;
            if (has_rows && next_rows > 0) next_dt = load_dt(next_rows);
            const Reads at = reads();
            // What a row adds: x times what is left of its time step, in units of the channel's largest x and of the chunk's largest step
            // (`into` is at most 1), so that no product passes fp16 and none that matters is too small for it.
            h8 into_hi[2], into_lo[2], zero = {};
            h8 x[2] = {columns_of(x_now, at, wave, 0, of_x), columns_of(x_now, at, wave, 1, of_x)};
            // The product's operands are asked for a step of eight instructions in front of them.
            constexpr int kSteps = 2 * ((kTiles + 3) / 4);
            constexpr int kAhead = 1;
            h8 operand[kAhead + 1][4];
            auto ask = [&](int step) __attribute__((always_inline)) {
#pragma unroll
                for (int t = step / 2 * 4; t < step / 2 * 4 + 4 && t < kTiles; ++t) operand[step % (kAhead + 1)][t % 4] = columns_of(b_now, at, t, step % 2, of_b);
                __builtin_amdgcn_sched_barrier(0);
            };
            ask(0);
            float top = 0.f;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                zero = __builtin_elementwise_fma(x[k], h8{}, zero);   // a NaN where one is no number
                top = fmaxf(top, largest_of(x[k]));
            }
            const int e = clamp_to(exponent_of(max_of_sixteenths(top)), -16, 15);
            // (exact: no x becomes larger than 2^15, and smaller only where the largest is 2^15 and more)
            const int up = 14 - e < 15 ? 14 - e : 15;
            const half_t by = (half_t)power_of_two(up);
            float unit_x = power_of_two(e - 14) * now.unit, per_unit_x = power_of_two(14 - e) * now.per_unit;
#pragma unroll
            for (int k = 0; k < 2; ++k) x[k] *= by;
            if (__any(14 - e > 15 || per_unit_x >= room)) {
                asm volatile("");
#pragma unroll
                for (int k = 0; k < 2; ++k) x[k] *= (half_t)power_of_two(14 - e - up);
                if (__any(per_unit_x >= room)) {
                    // The state might pass fp32 in units of what the chunk adds, which is little: larger ones where it would, in which that little keeps the
                    // digits that matter beside such a state.
#pragma unroll
                    for (int t = 0; t < kTiles; ++t) S[t] *= unit_s;
                    unit_s = 1.f;
                    const int more = clamp_to(exponent_of(largest_state()) + exponent_of(per_unit_x) - 120, 0, 126);
                    unit_x *= power_of_two(more), per_unit_x *= power_of_two(-more);
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int j = 0; j < 8; ++j) x[k][j] = (half_t)((float)x[k][j] * power_of_two(-more));
                }
            }
            float one = 1.f;
            asm volatile("" : "+s"(one));  // (v - one hi is one instruction for an fp16 hi, v - hi two)
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const f4 w = *reinterpret_cast<const f4*>(&now.into[32 * k + 16 * h + 4 * high]);
#pragma unroll
                    for (int r = 0; r < 4; r += 2) {
                        const f2 v = {__builtin_fmaf((float)x[k][4 * h + r], w[r], 0.f), __builtin_fmaf((float)x[k][4 * h + r + 1], w[r + 1], 0.f)};
                        const h2 hi = __builtin_convertvector(v, h2);
                        const h2 lo = __builtin_convertvector((f2{__builtin_fmaf((float)hi[0], -one, v[0]), __builtin_fmaf((float)hi[1], -one, v[1])}), h2);
                        into_hi[k][4 * h + r] = hi[0], into_hi[k][4 * h + r + 1] = hi[1];
                        into_lo[k][4 * h + r] = lo[0], into_lo[k][4 * h + r + 1] = lo[1];
                    }
                }
            const bool infinities = __any(!all_zero(zero));
            if (infinities) {
                asm volatile("");  // infinities have no rest
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int j = 0; j < 8; ++j) into_lo[k][j] = finite(into_hi[k][j]) ? into_lo[k][j] : (half_t)0.f;
            }
            const float keep = now.decay[kChunk - 1] * (unit_s * per_unit_x);
            if constexpr (!LAST) walk_log += now.all;
            unit_s = unit_x;
#pragma unroll
            for (int t = 0; t < kTiles; ++t) S[t] *= keep;
#pragma unroll
            for (int step = 0; step < kSteps; ++step) {
                ask(step + kAhead);
                const int k = step % 2, t0 = step / 2 * 4;
#pragma unroll
                for (int t = t0; t < t0 + 4 && t < kTiles; ++t) S[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(operand[step % (kAhead + 1)][t - t0], into_hi[k], S[t], 0, 0, 0);
#pragma unroll
                for (int t = t0; t < t0 + 4 && t < kTiles; ++t) S[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(operand[step % (kAhead + 1)][t - t0], into_lo[k], S[t], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (infinities && states < 32 * N32) {
                // b is zero behind the states, and zero times an infinity would stay there for the outputs' products
                int n0 = 4 * high;
                asm volatile("" : "+v"(n0));
#pragma unroll
                for (int t = 0; t < kTiles; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) S[t][r] = 16 * t + n0 + r < states ? S[t][r] : 0.f;
            }
            if (next_rows > 0) {
                if constexpr (LAST) leave_copy(s_next, unit);
                if (has_rows) row_values(next_dt, next_rows, next);
            }
            row += rows;
        };
        {
            const int rows = last - row < kChunk ? last - row : kChunk;
            const half_t dt = has_rows ? load_dt(rows) : (half_t)0.f;
            if constexpr (LAST) leave_copy(s_even, s_unit[0]);
            if (has_rows) row_values(dt, rows, values[0]);
        }
        while (true) {
            chunk(b_even, x_even, s_odd, (lds_bytes)b_odd, (lds_bytes)x_odd, s_unit[1], values[0], values[1]);
            if (row >= last) break;
            chunk(b_odd, x_odd, s_even, (lds_bytes)b_even, (lds_bytes)x_even, s_unit[0], values[1], values[0]);
            if (row >= last) break;
        }
        const ArgsAgain k = args_again();
        if constexpr (LAST) {
            if (last == q.first + q.rows && k->state_out) store_state(k);
        } else {
            f4* const added = reinterpret_cast<f4*>(k->temp);
#pragma unroll
            for (int t = 0; t < kTiles; ++t) added[held_at(piece0) + t * 256] = S[t] * unit_s;
            if (wave == 0 && lane == 0) reinterpret_cast<float*>(added + 2 * held_all(k))[(int64_t)piece0 * units + unit] = (float)exp2(walk_log);
        }
    };

    while (index < a.sequences.count) {
        const ArgsAgain k = args_again();
        const Sequences all = sequences_again(k);
        Sequence q = sequence_of(all, index);
        q.first = uniform(q.first), q.rows = uniform(q.rows), q.place = uniform(q.place);
        const int row = q.first + offset * kChunk;
        const int behind = q.rows - offset * kChunk, room = budget < (1 << 24) ? budget * kChunk : 0x7fffffff;
        const int last = row + (behind < room ? behind : room);  // the end of the sequence's rows within the segment
        __syncthreads();  // (all have done with the tiles, the copies and the row values)
        if (kLoading > 0 && loads) walk_loads(row, last);
        else if (has_state) walk_state(q, row, last);
        else
            switch (wave) {
                case 0: walk_outputs(std::integral_constant<int, 0>{}, row, last); break;
                case 1: walk_outputs(std::integral_constant<int, 1>{}, row, last); break;
                case 2: walk_outputs(std::integral_constant<int, 2>{}, row, last); break;
                default: walk_outputs(std::integral_constant<int, 3>{}, row, last);
            }
        if constexpr (!LAST) break;
        budget -= (last - row + kChunk - 1) / kChunk;
        offset = 0;
        if (budget <= 0) break;
        do ++index;
        while (index < all.count && sequence_of(all, index).rows == 0);
    }
}

// One workgroup a compute unit in the second launch, three in the first: as much as their LDS allows.  (16384 tokens of 128 heads when 2 segments took
// 460 us: 4 of them, whose second launch holds half of its workgroups back, 530; 6 pieces in the first launch 77, 4 as much.)
constexpr int kWorkgroups = 256, kFirstWorkgroups = 768;

// How a call is shared out: segments, and pieces of a segment in the first launch.
struct Shares {
    int segments, pieces;
};
static Shares shares_of(int rows, int count, int units) {
    const int64_t chunks = rows / kChunk + (count < rows ? count : rows), most = chunks / 4 < 1 ? 1 : chunks / 4;
    Shares s;
    int64_t n = kWorkgroups / units;
    if (n > most) n = most;
    s.segments = n < 1 ? 1 : (int)n;
    s.pieces = 1;
    if (s.segments > 1) {
        int64_t m = kFirstWorkgroups / (units * (s.segments - 1));
        if (m > chunks / (2 * s.segments)) m = chunks / (2 * s.segments);
        s.pieces = m < 1 ? 1 : (int)m;
    }
    return s;
}
static int tiles_of(int states) { return states <= 64 ? 4 : (states <= 96 ? 6 : (states <= 128 ? 8 : (states <= 192 ? 12 : 16))); }

size_t state_space_scan_needs(int rows, int count, int heads, int head_dim, int states) {
    const int units = heads * ((head_dim + 63) / 64);
    const Shares s = shares_of(rows, count, units);
    return (size_t)(s.segments - 1) * s.pieces * units * ((size_t)2 * tiles_of(states) * 256 * sizeof(f4) + sizeof(float));
}

template <int N32, bool THROUGH>
static void launch(const ScanArgs& a, hipStream_t stream) {
    const unsigned units = (unsigned)(a.heads * a.head_blocks);
    if (a.segments > 1)
        hipLaunchKernelGGL((state_space_scan_kernel<N32, THROUGH, false>), dim3(units, (unsigned)((a.segments - 1) * a.pieces)),
                           dim3(64 * scan_waves(N32, THROUGH, false)), 0, stream, a);
    hipLaunchKernelGGL((state_space_scan_kernel<N32, THROUGH, true>), dim3(units, (unsigned)a.segments), dim3(64 * scan_waves(N32, THROUGH, true)), 0,
                       stream, a);
}
template <int N32>
static void go(const ScanArgs& a, bool through, hipStream_t stream) {
    if (through) launch<N32, true>(a, stream);
    else launch<N32, false>(a, stream);
}

int state_space_scan_launch(const ScanArgs& args, hipStream_t stream) {
    ScanArgs a = args;
    a.head_blocks = (a.head_dim + 63) / 64;
    const Shares s = shares_of(a.sequences.rows, a.sequences.count, a.heads * a.head_blocks);
    a.segments = s.segments, a.pieces = s.pieces;
    // straight to LDS: pieces at multiples of 4 bytes, whole ones of b and whole words of x (a buffer that ends within a word: its last value
    // would be lost, or the next one read); rows that do not overlap (what lies behind a chunk's rows then lies behind the buffer), 64 of them below
    // 2^31 bytes
    const int64_t far = 1LL << 23, strides = a.x_row | a.x_head | a.b_row | a.b_group;
    const uintptr_t bases = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.b);
    const bool near = a.x_row >= (a.head_dim < 64 ? a.head_dim : 64) && a.b_row >= a.states && a.c_row >= 0 && a.y_row >= 0 && a.x_row <= far && a.b_row <= far && a.c_row <= far &&
                      a.y_row <= far;
    const bool through = !(near && (strides & 1) == 0 && (bases & 3) == 0 && a.head_dim % 2 == 0 && a.states % 8 == 0);
    switch (tiles_of(a.states)) {
        case 4: go<2>(a, through, stream); break;
        case 6: go<3>(a, through, stream); break;
        case 8: go<4>(a, through, stream); break;
        case 12: go<6>(a, through, stream); break;
        default: go<8>(a, through, stream);
    }
    return hipGetLastError() == hipSuccess ? UNIQL_OK : UNIQL_E_LAUNCH;
}

}  // namespace uniql
