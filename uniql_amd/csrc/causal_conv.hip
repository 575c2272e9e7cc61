// The causal convolution of a state-space layer: y[t, c] = f(bias[c] + sum_k w[c, k] x[t - W + 1 + k, c]), f SiLU or nothing, inputs in front
// of a sequence's first row from its state (the last W - 1 inputs of before) or zeros.
//
// A thread takes eight channels and a run of rows, of which it reads each once: the last W - 1 stay in registers.  The first W - 1
// rows of a sequence, and its new state, belong to a workgroup of their own: it has read the state before it writes it, which makes
// a state that is replaced in place safe, and a batch of single tokens is these workgroups alone.
//
// Bound by HBM: 16384 rows of 10240 channels 136 to 147 us, 4.6 to 4.9 TB/s, what a copy reaches.  48 single tokens 4.5 to 4.8 us: offsets, then state and
// rows, then the store, each a round trip.
#include "row_mask.hpp"
#include "state_space.hpp"

namespace uniql {

constexpr int kConvThreads = 256;
constexpr int kMostRows = 32;  // of a run: a bit each

template <int W>
struct Taps {
    float w[W][8], bias[8];
    __device__ __forceinline__ void load(const ConvArgs& a, int c0, int left) {
        h8 v[W];
#pragma unroll
        for (int k = 0; k < W; ++k) v[k] = load_halves(a.weight + (int64_t)c0 * W + 8 * k, left * W - 8 * k);
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int k = 0; k < W; ++k) w[k][e] = (float)v[(e * W + k) / 8][(e * W + k) % 8];
        const h8 b = a.bias ? load_halves(a.bias + c0, left) : h8{};
#pragma unroll
        for (int e = 0; e < 8; ++e) bias[e] = (float)b[e];
    }
    // x[0 .. W-1]: the inputs of a row, the oldest first
    __device__ __forceinline__ h8 apply(const h8 (&x)[W], bool activation) const {
        h8 y;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float u = bias[e];
#pragma unroll
            for (int k = 0; k < W; ++k) u = __builtin_fmaf((float)x[k][e], w[k][e], u);
            y[e] = (half_t)(activation ? silu_fast(u) : u);
        }
        return y;
    }
};

// The largest s in -1 .. count - 1 with cu[s] <= row, for offsets that ascend; all lanes of a wave ask for the same row.
__device__ __forceinline__ int last_not_behind(const int32_t* cu, int count, int row) {
    const int lane = threadIdx.x & 63;
    int below = -1, above = count;  // cu[below] <= row < cu[above]
    while (above - below > 1) {
        const int span = above - below - 1, step = (span + 63) / 64;
        const int at = below + (lane + 1) * step;
        const bool fits = at < above && cu[at] <= row;
        const int n = __builtin_popcountll(__ballot(fits));
        const int upper = below + (n + 1) * step;
        below += n * step;
        above = upper < above ? upper : above;
    }
    return below;
}

// The rows of any lane's mask, in each lane.
__device__ __forceinline__ uint32_t rows_of_all(uint32_t mask) {
    int v = (int)mask;
    auto join = [&](int other) __attribute__((always_inline)) { v = (int)rows_of_either((uint32_t)v, (uint32_t)other); };
    join(dpp_or_zero<0x111, 0xf>(v));  // one, two, four, eight lanes below, within sixteen
    join(dpp_or_zero<0x112, 0xf>(v));
    join(dpp_or_zero<0x114, 0xf>(v));
    join(dpp_or_zero<0x118, 0xf>(v));
    join(dpp_or_zero<0x142, 0xa>(v));  // the last of the sixteen below, for the second and fourth sixteen
    join(dpp_or_zero<0x143, 0xc>(v));  // lane 31, for the upper half
    return (uint32_t)__builtin_amdgcn_readlane(v, 63);
}

template <int W>
__global__ __launch_bounds__(kConvThreads) void causal_conv_kernel(const ConvArgs a) {
    const int c0 = (blockIdx.y * kConvThreads + threadIdx.x) * 8, left = a.channels - c0;
    Taps<W> taps;
    const bool active = left > 0;
    const int index = (int)blockIdx.x + a.begin;
    if (index >= a.tiles) {
        // a sequence's first rows and its state
        const Sequence q = sequence_of(a.sequences, index - a.tiles);
        if (q.rows == 0 || !active) return;
        h8 x[2 * (W - 1)];  // the state, the first rows
        const int64_t at = ((int64_t)q.place * (W - 1)) * a.channels + c0;
        const half_t* from = a.x + (int64_t)q.first * a.x_row + c0;
#pragma unroll
        for (int k = 0; k < W - 1; ++k) {
            x[k] = a.state && q.continued ? load_halves(a.state + at + (int64_t)k * a.channels, left) : h8{};
            x[W - 1 + k] = k < q.rows ? load_halves(from + k * a.x_row, left) : h8{};
        }
        taps.load(a, c0, left);
        if (a.state_out) {
#pragma unroll
            for (int k = 0; k < W - 1; ++k) {
                h8 v = x[W - 2 + 1 + k];
                if (q.rows >= W - 1) {
                    v = load_halves(from + (int64_t)(q.rows - (W - 1) + k) * a.x_row, left);
                } else {
#pragma unroll
                    for (int r = 1; r < W - 1; ++r)
                        if (q.rows == r) v = x[r + k];
                }
                store_halves(a.state_out + at + (int64_t)k * a.channels, v, left);
            }
        }
        half_t* to = a.out + (int64_t)q.first * a.out_row + c0;
#pragma unroll
        for (int r = 0; r < W - 1; ++r)
            if (r < q.rows) {
                h8 row[W];
#pragma unroll
                for (int k = 0; k < W; ++k) row[k] = x[r + k];
                store_halves(to + r * a.out_row, taps.apply(row, a.activation), left);
            }
        return;
    }
    const int row0 = index * a.run, rows = a.sequences.rows - row0 < a.run ? a.sequences.rows - row0 : a.run;
    // Rows that have W - 1 others of their sequence in front of them, a bit each: 64 sequences at a time.
    const int lane = threadIdx.x & 63;
    uint32_t allowed = 0;
    for (int base = __builtin_amdgcn_readfirstlane(last_not_behind(a.sequences.cu, a.sequences.count, row0)); base < a.sequences.count; base += 64) {
        const int s = base + lane;
        uint32_t mine = 0;
        if (s >= 0 && s < a.sequences.count) {
            const Sequence q = sequence_of(a.sequences, s);
            mine = rows_between(q.first + (W - 1) - row0, q.first + q.rows - row0, rows);
        }
        allowed = rows_of_either(allowed, rows_of_all(mine));
        const int next = base + 64;
        if (next >= a.sequences.count || a.sequences.cu[next] >= row0 + rows) break;
    }
    if (!active || allowed == 0) return;
    taps.load(a, c0, left);
    h8 x[W];
#pragma unroll
    for (int k = 1; k < W; ++k) {
        const int row = row0 - W + k;
        x[k] = row >= 0 ? load_halves(a.x + (int64_t)row * a.x_row + c0, left) : h8{};
    }
    const half_t* from = a.x + (int64_t)row0 * a.x_row + c0;
    half_t* to = a.out + (int64_t)row0 * a.out_row + c0;
    // eight rows on their way at once
    for (int r0 = 0; r0 < rows; r0 += 8) {
        h8 next[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) next[r] = r0 + r < rows ? load_halves(from + (int64_t)(r0 + r) * a.x_row, left) : h8{};
#pragma unroll
        for (int r = 0; r < 8; ++r) {
#pragma unroll
            for (int k = 0; k < W - 1; ++k) x[k] = x[k + 1];
            x[W - 1] = next[r];
            if ((allowed >> (r0 + r)) & 1) store_halves(to + (int64_t)(r0 + r) * a.out_row, taps.apply(x, a.activation), left);
        }
    }
}

int causal_conv_launch(const ConvArgs& args, int width, hipStream_t stream) {
    ConvArgs a = args;
    const int64_t down = (a.channels + 8 * kConvThreads - 1) / (8 * kConvThreads);
    // Long runs read little twice (35 rows for 32); short ones make workgroups enough where there are few rows (9 pieces of 333 rows at most
    // 15.4 -> 12.4 us with runs of 8; 16384 rows 147 with runs of 32, 142 of 16).
    a.run = kMostRows;
    while (a.run > 8 && a.sequences.rows / a.run * down < 1024) a.run /= 2;
    a.tiles = a.sequences.cu ? (a.sequences.rows + a.run - 1) / a.run : 0;
    const int64_t across = (int64_t)a.tiles + a.sequences.count;
    if (down > 65535) return UNIQL_E_SHAPE;
    for (int64_t begin = 0; begin < across; begin += kMostWorkgroups) {
        a.begin = (int)begin;
        const dim3 grid((unsigned)(across - begin < kMostWorkgroups ? across - begin : kMostWorkgroups), (unsigned)down), block(kConvThreads);
        if (width == 2) hipLaunchKernelGGL(causal_conv_kernel<2>, grid, block, 0, stream, a);
        else if (width == 3) hipLaunchKernelGGL(causal_conv_kernel<3>, grid, block, 0, stream, a);
        else hipLaunchKernelGGL(causal_conv_kernel<4>, grid, block, 0, stream, a);
    }
    return hipGetLastError() == hipSuccess ? UNIQL_OK : UNIQL_E_LAUNCH;
}

}  // namespace uniql
