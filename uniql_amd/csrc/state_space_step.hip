// One more token of every request, or of those of a batch that have one, through a state-space layer: S' = exp(s a) S + s x b^T,
// y = S' c + d x, with the time step s = softplus(dt + bias), for each head's matrix S [head_dim][states] of fp32.
//
// Lanes lie along the states, four to a lane, so that rows of S come and go in whole lines; a wave takes 64 / LANES rows of the head at
// once, and a thread ROWS of them, all on their way before the first is used.  The products with c are summed over the lanes.
//
// Bound by HBM: the state is read and written once.  256 requests of 128 heads of 64 x 128 400 us, 5.4 TB/s; 48 of 54 x 96 67 us where the
// states come from memory, 54 where the last-level cache holds some.
#include "state_space.hpp"

namespace uniql {

constexpr int kStepThreads = 256;

// LANES: of a row; EACH: neighbouring states of a lane, PARTS: how often the lanes go over the row.
template <int LANES, int EACH, int PARTS, int ROWS>
__global__ __launch_bounds__(kStepThreads) void state_space_step_kernel(const ScanArgs a) {
    constexpr int kAtOnce = kStepThreads / LANES;  // rows that the workgroup covers in one go
    const unsigned per_sequence = (unsigned)(a.heads * a.head_blocks);
    const unsigned s = blockIdx.x / per_sequence, rest = blockIdx.x % per_sequence;
    const int head = rest / a.head_blocks, block = rest % a.head_blocks;
    const Sequence q = sequence_of(a.sequences, a.begin + (int)s);
    if (q.rows == 0) return;
    const int lane = threadIdx.x % LANES, p0 = block * kAtOnce * ROWS + threadIdx.x / LANES;
    const int64_t size = (int64_t)a.head_dim * a.states;
    const int64_t at = ((int64_t)q.place * a.heads + head) * size;
    float S[ROWS][PARTS][EACH];
    typedef float vec __attribute__((ext_vector_type(EACH)));
    const bool from_state = a.state && q.continued;
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
            const int p = p0 + r * kAtOnce, n = (i * LANES + lane) * EACH;
            vec v = {};
            if (from_state && p < a.head_dim && n < a.states) v = *reinterpret_cast<const vec*>(a.state + at + (int64_t)p * a.states + n);
#pragma unroll
            for (int e = 0; e < EACH; ++e) S[r][i][e] = v[e];
        }
    const int group = head / a.share;
    const half_t* const b_from = a.b + (int64_t)q.first * a.b_row + group * a.b_group;
    const half_t* const c_from = a.c + (int64_t)q.first * a.c_row + group * a.c_group;
    const half_t* const x_from = a.x + (int64_t)q.first * a.x_row + head * a.x_head;
    float b[PARTS][EACH], c[PARTS][EACH], x[ROWS];
#pragma unroll
    for (int i = 0; i < PARTS; ++i)
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            const int n = (i * LANES + lane) * EACH;
            b[i][e] = n < a.states ? (float)b_from[n + e] : 0.f;
            c[i][e] = n < a.states ? (float)c_from[n + e] : 0.f;
        }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const int p = p0 + r * kAtOnce;
        x[r] = p < a.head_dim ? (float)x_from[p] : 0.f;
    }
    const float step = time_step((float)a.dt[(int64_t)q.first * a.dt_row + head], a.dt_bias ? a.dt_bias[head] : 0.f, a.softplus,
                                 a.dt_min, a.dt_max);
    const float decay = expf(step * a.a[head]), skip = a.d ? a.d[head] : 0.f;
    float y[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const float in = step * x[r];
        y[r] = 0.f;
#pragma unroll
        for (int i = 0; i < PARTS; ++i)
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                // (an empty state is not multiplied: a decay that is no number would not leave it empty)
                S[r][i][e] = from_state ? __builtin_fmaf(S[r][i][e], decay, in * b[i][e]) : in * b[i][e];
                y[r] = __builtin_fmaf(S[r][i][e], c[i][e], y[r]);
            }
    }
    if (a.state_out) {
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
#pragma unroll
            for (int i = 0; i < PARTS; ++i) {
                const int p = p0 + r * kAtOnce, n = (i * LANES + lane) * EACH;
                vec v;
#pragma unroll
                for (int e = 0; e < EACH; ++e) v[e] = S[r][i][e];
                if (p < a.head_dim && n < a.states) *reinterpret_cast<vec*>(a.state_out + at + (int64_t)p * a.states + n) = v;
            }
    }
    half_t* const to = a.y + (int64_t)q.first * a.y_row + head * a.y_head;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const int p = p0 + r * kAtOnce;
        const float sum = sum_over<LANES>(y[r]);
        if (lane == 0 && p < a.head_dim) to[p] = (half_t)(a.d ? __builtin_fmaf(skip, x[r], sum) : sum);
    }
}

template <int LANES, int EACH, int PARTS, int ROWS>
static int go(ScanArgs& a, hipStream_t stream) {
    constexpr int rows = kStepThreads / LANES * ROWS;
    a.head_blocks = (a.head_dim + rows - 1) / rows;
    const int each = a.heads * a.head_blocks, most = (int)(kMostWorkgroups / each);  // (sequences of a launch)
    for (int64_t begin = 0; begin < a.sequences.count; begin += most) {
        a.begin = (int)begin;
        const int64_t count = a.sequences.count - begin < most ? a.sequences.count - begin : most;
        hipLaunchKernelGGL((state_space_step_kernel<LANES, EACH, PARTS, ROWS>), dim3((unsigned)(count * each)), dim3(kStepThreads), 0, stream, a);
    }
    return hipGetLastError() == hipSuccess ? UNIQL_OK : UNIQL_E_LAUNCH;
}

// A row of `states` by 8 lanes, PARTS vectors of four each: whole lines of 128 bytes a row in each access, no lane without work where the states
// are a multiple of 32, and three steps to sum a row up.  Eight vectors of a thread on their way at once, fewer where there are few states or
// few heads (`spread`: one user's 128 heads 5.8 -> 5.4 us).
template <int PARTS>
static int by_eight(ScanArgs& a, bool spread, hipStream_t stream) {
    if (spread) return go<8, 4, PARTS, 1>(a, stream);
    return go<8, 4, PARTS, (PARTS > 4 ? 1 : (PARTS > 2 ? 2 : 4))>(a, stream);
}

int state_space_step_launch(const ScanArgs& args, hipStream_t stream) {
    ScanArgs a = args;
    if (a.states % 4 != 0) return go<64, 1, 4, 2>(a, stream);
    const bool spread = (int64_t)a.sequences.count * a.heads < 2048;
    // 128 and 256 states fill 32 and 64 lanes, which then read a row in one piece (256 requests of 128 heads 410 -> 400 us)
    if (a.states == 128 && !spread) return go<32, 4, 1, 8>(a, stream);
    if (a.states == 256 && !spread) return go<64, 4, 1, 8>(a, stream);
    switch ((a.states + 31) / 32) {
        case 1: return by_eight<1>(a, spread, stream);
        case 2: return by_eight<2>(a, spread, stream);
        case 3: return by_eight<3>(a, spread, stream);
        case 4: return by_eight<4>(a, spread, stream);
        case 5: return by_eight<5>(a, spread, stream);
        case 6: return by_eight<6>(a, spread, stream);
        case 7: return by_eight<7>(a, spread, stream);
        default: return by_eight<8>(a, spread, stream);
    }
}

}  // namespace uniql
