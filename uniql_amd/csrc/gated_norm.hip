// The gate and the norm behind a state-space layer's scan: u = x z / (1 + exp(-z)), y = u / sqrt(mean(u^2) + eps) w, the mean over
// each group of neighbouring channels.  The reference's order: the gate first, the sum of squares in fp32, one rounding at the end.
//
// A wave takes a group of up to 1024 channels, a workgroup a wider one; the gated values stay in registers.
//
// Bound by HBM: 16384 rows of 8 groups of 1024 147 us, 5.5 TB/s (two streams in, one out); one row 3.0 us, a round trip each way.
#include "state_space.hpp"

namespace uniql {

// WAVES: of a group; a thread holds PIECES pieces of eight values, REREAD: wider groups than that are read a second time.
template <int WAVES, int PIECES, bool REREAD>
__global__ __launch_bounds__(256) void gated_group_norm_kernel(const NormArgs a) {
    constexpr int kThreads = 64 * WAVES;
    __shared__ float sums[4];
    const int tid = threadIdx.x % kThreads;
    const int64_t index = (a.begin + blockIdx.x) * (256 / kThreads) + threadIdx.x / kThreads;
    const int64_t all = (int64_t)a.rows * a.groups;
    const bool there = index < all;
    const int64_t row = there ? index / a.groups : 0;
    const int group = there ? (int)(index % a.groups) : 0;
    const int c0 = group * a.width;
    const half_t *const x = a.x + row * a.x_row + c0, *const z = a.z + row * a.z_row + c0;
    auto gated = [&](int at, float (&u)[8]) __attribute__((always_inline)) {
        const h8 xv = load_halves(x + at, a.width - at), zv = load_halves(z + at, a.width - at);
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = (float)xv[e] * silu_fast((float)zv[e]);
    };
    float u[PIECES][8], sum = 0.f;
    const int passes = REREAD ? (a.width + kThreads * PIECES * 8 - 1) / (kThreads * PIECES * 8) : 1;
    for (int pass = 0; pass < passes; ++pass)
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int at = ((pass * PIECES + i) * kThreads + tid) * 8;
#pragma unroll
            for (int e = 0; e < 8; ++e) u[i][e] = 0.f;
            if (at < a.width) {
                gated(at, u[i]);
#pragma unroll
                for (int e = 0; e < 8; ++e) sum += u[i][e] * u[i][e];
            }
        }
    sum = sum_over<64>(sum);
    if (WAVES > 1) {
        if ((tid & 63) == 0) sums[tid >> 6] = sum;
        __syncthreads();
        sum = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) sum += sums[w];
    }
    if (!there) return;
    const float factor = rsqrtf(sum / (float)a.width + a.eps);
    for (int pass = 0; pass < passes; ++pass)
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int at = ((pass * PIECES + i) * kThreads + tid) * 8, left = a.width - at;
            if (left <= 0) continue;
            if (REREAD) gated(at, u[i]);
            const h8 w = load_halves(a.weight + c0 + at, left);
            h8 y;
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = (half_t)(u[i][e] * factor * (float)w[e]);
            store_halves(a.out + row * a.out_row + c0 + at, y, left);
        }
}

template <int WAVES, int PIECES, bool REREAD>
static int go(NormArgs a, hipStream_t stream) {
    const int64_t each = 4 / WAVES, blocks = ((int64_t)a.rows * a.groups + each - 1) / each;
    for (a.begin = 0; a.begin < blocks; a.begin += kMostWorkgroups) {
        const int64_t count = blocks - a.begin < kMostWorkgroups ? blocks - a.begin : kMostWorkgroups;
        hipLaunchKernelGGL((gated_group_norm_kernel<WAVES, PIECES, REREAD>), dim3((unsigned)count), dim3(256), 0, stream, a);
    }
    return hipGetLastError() == hipSuccess ? UNIQL_OK : UNIQL_E_LAUNCH;
}

int gated_group_norm_launch(const NormArgs& a, hipStream_t stream) {
    if (a.width <= 512) return go<1, 1, false>(a, stream);
    if (a.width <= 1024) return go<1, 2, false>(a, stream);
    if (a.width <= 2048) return go<4, 1, false>(a, stream);
    if (a.width <= 4096) return go<4, 2, false>(a, stream);
    if (a.width <= 8192) return go<4, 4, false>(a, stream);
    return go<4, 4, true>(a, stream);
}

}  // namespace uniql
