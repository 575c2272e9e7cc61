// What the calls of a state-space layer consist of, and how a kernel finds the sequences of a batch.
#pragma once

#include "common.hpp"

namespace uniql {

// Which rows belong to which sequence, and where their states lie.
struct Sequences {
    const int32_t *cu, *starts, *places;  // any may be null: a row each; all continued; place s
    int count, pool, rows;
    int only;  // 0: sequences of any length have rows; kSingle: those of one row; kLonger: the others
};
constexpr int kSingle = 1, kLonger = 2;
struct Sequence {
    int first, rows, place;
    bool continued;
};

struct ConvArgs {
    const half_t *x, *weight, *bias, *state;  // [rows][channels], [channels][width], [channels] or null, [pool][width - 1][channels] or null
    half_t *state_out, *out;
    int64_t x_row, out_row;
    Sequences sequences;
    int channels, activation;
    int run, tiles, begin;  // set by the launch: rows of a run, and the runs; the launch's first workgroup
};

struct ScanArgs {
    const half_t *x, *dt, *b, *c;  // [rows][heads][head_dim], [rows][heads], [rows][groups][states] twice
    const float *a, *d, *dt_bias;  // [heads], the last two may be null
    const float* state;            // [pool][heads][head_dim][states] or null
    float* state_out;
    half_t* y;
    int64_t x_row, x_head, dt_row, b_row, b_group, c_row, c_group, y_row, y_head;
    float dt_min, dt_max;
    Sequences sequences;
    int heads, share, head_dim, states, softplus;  // share: heads of a group
    // set by the launch
    int segments, pieces, head_blocks, begin;  // pieces: of a segment, in the first launch; begin: a step's first sequence
    float* temp;
};

struct NormArgs {
    const half_t *x, *z, *weight;
    half_t* out;
    int64_t x_row, z_row, out_row;
    int rows, groups, width;
    float eps;
    int64_t begin;  // set by the launch: its first workgroup
};

// Workgroups of 256 threads that a launch takes (fewer than 2^32 threads); calls of more are several launches.
constexpr int64_t kMostWorkgroups = (1 << 24) - 1;

// ---- sequences ---------------------------------------------------------------------------------------------------------
// Whatever the arrays hold, rows and places lie within the call's; sequences without a place have no rows.
__device__ __forceinline__ Sequence sequence_of(const Sequences& all, int s) {
    Sequence q;
    q.first = s;
    q.rows = 1;
    if (all.cu) {
        const int a = all.cu[s], b = all.cu[s + 1];
        q.first = a < 0 ? 0 : (a > all.rows ? all.rows : a);
        const int last = b < q.first ? q.first : (b > all.rows ? all.rows : b);
        q.rows = last - q.first;
    }
    q.place = all.places ? all.places[s] : s;
    if ((unsigned)q.place >= (unsigned)all.pool) q.rows = 0;
    if (all.only && (q.rows == 1) != (all.only == kSingle)) q.rows = 0;
    q.continued = !all.starts || all.starts[s] > 0;
    return q;
}

// ---- across lanes ------------------------------------------------------------------------------------------------------
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_or_zero(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false); }
// Sums over the lanes up to and including each.
__device__ __forceinline__ int sums_upto(int v) {
    v += dpp_or_zero<0x111, 0xf>(v);  // one, two, four, eight lanes below, within sixteen
    v += dpp_or_zero<0x112, 0xf>(v);
    v += dpp_or_zero<0x114, 0xf>(v);
    v += dpp_or_zero<0x118, 0xf>(v);
    v += dpp_or_zero<0x142, 0xa>(v);  // the last of the sixteen below, for the second and fourth sixteen
    return v + dpp_or_zero<0x143, 0xc>(v);  // lane 31, for the upper half
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_or_zero(double v) {
    const int lo = dpp_or_zero<CTRL, ROWS>(__double2loint(v)), hi = dpp_or_zero<CTRL, ROWS>(__double2hiint(v));
    return __hiloint2double(hi, lo);
}
__device__ __forceinline__ double sums_upto(double v) {
    v += dpp_or_zero<0x111, 0xf>(v);
    v += dpp_or_zero<0x112, 0xf>(v);
    v += dpp_or_zero<0x114, 0xf>(v);
    v += dpp_or_zero<0x118, 0xf>(v);
    v += dpp_or_zero<0x142, 0xa>(v);
    return v + dpp_or_zero<0x143, 0xc>(v);
}
// The sum over LANES neighbouring lanes (a power of two), in each of them.
template <int CTRL>
__device__ __forceinline__ float dpp_from(float v) {
    const int i = __builtin_bit_cast(int, v);
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float other_sixteen(float v, float& mine) {
    const auto x = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    mine = __builtin_bit_cast(float, (unsigned)x[0]);
    return __builtin_bit_cast(float, (unsigned)x[1]);
}
__device__ __forceinline__ float other_half(float v, float& mine) {
    const auto x = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    mine = __builtin_bit_cast(float, (unsigned)x[0]);
    return __builtin_bit_cast(float, (unsigned)x[1]);
}
template <int LANES>
__device__ __forceinline__ float sum_over(float v) {
    if (LANES > 1) v += dpp_from<0xB1>(v);   // lane ^ 1
    if (LANES > 2) v += dpp_from<0x4E>(v);   // lane ^ 2
    if (LANES > 4) v += dpp_from<0x141>(v);  // mirrored within eight
    if (LANES > 8) v += dpp_from<0x140>(v);  // mirrored within sixteen
    float mine;
    if (LANES > 16) {
        const float other = other_sixteen(v, mine);
        v = mine + other;
    }
    if (LANES > 32) {
        const float other = other_half(v, mine);
        v = mine + other;
    }
    return v;
}
// The largest of the lanes that differ by 16, 32 or 48, in each of them (NaN counts as nothing).
__device__ __forceinline__ float max_of_sixteenths(float v) {
    float mine, other = other_sixteen(v, mine);
    v = fmaxf(mine, other);
    other = other_half(v, mine);
    return fmaxf(mine, other);
}

// ---- values ------------------------------------------------------------------------------------------------------------
typedef _Float16 h8_any __attribute__((ext_vector_type(8), aligned(2)));
typedef _Float16 h4_any __attribute__((ext_vector_type(4), aligned(2)));
// Eight values at any address that holds fp16 values, the first `left` of which exist; the others are zeros.
__device__ __forceinline__ h8 load_halves(const half_t* p, int left) {
    if (left >= 8) {
        const h8_any v = *reinterpret_cast<const h8_any*>(p);
        return h8{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]};
    }
    h8 v = {};
#pragma unroll
    for (int i = 0; i < 7; ++i)
        if (i < left) v[i] = p[i];
    return v;
}
__device__ __forceinline__ void store_halves(half_t* p, h8 v, int left) {
    if (left >= 8) {
        *reinterpret_cast<h8_any*>(p) = h8_any{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]};
        return;
    }
#pragma unroll
    for (int i = 0; i < 7; ++i)
        if (i < left) p[i] = v[i];
}
// u / (1 + exp(-u)) with the hardware's exponential and reciprocal (1 ulp each; the result is rounded to fp16)
__device__ __forceinline__ float silu_fast(float u) {
    return u * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * u));
}
// The length of a token's time step, log(1 + exp(u)) = max(u, 0) + log(1 + t) with t = exp(-|u|).  The logarithm by its series
// 2 (r + r^3 / 3 + ..), r = t / (2 + t) <= 1/3, whose next term is below 2^-32 of it: the logarithm of a rounded 1 + t would be off by
// 2^-24 / t, which the states, summed up in fp32, would show.  The exponential's argument is kept in two parts for the same reason.
__device__ __forceinline__ float time_step(float dt, float bias, int softplus, float dt_min, float dt_max) {
    float u = dt + bias;
    if (softplus) {
        const float size = -fabsf(u), hi = size * 1.4426950408889634f;
        const float lo = __builtin_fmaf(size, 1.4426950408889634f, -hi) + size * 1.925963033500e-8f;
        const float e = __builtin_amdgcn_exp2f(hi), t = hi > -126.f ? __builtin_fmaf(e, lo * 0.6931471805599453f, e) : e;
        const float sum = 2.0f + t, about = __builtin_amdgcn_rcpf(sum), per = __builtin_fmaf(__builtin_fmaf(-sum, about, 1.0f), about, about);
        const float r = t * per, q = r * r;
        float v = 1.0f / 17.0f;
        v = __builtin_fmaf(v, q, 1.0f / 15.0f);
        v = __builtin_fmaf(v, q, 1.0f / 13.0f);
        v = __builtin_fmaf(v, q, 1.0f / 11.0f);
        v = __builtin_fmaf(v, q, 1.0f / 9.0f);
        v = __builtin_fmaf(v, q, 1.0f / 7.0f);
        v = __builtin_fmaf(v, q, 1.0f / 5.0f);
        v = __builtin_fmaf(v, q, 1.0f / 3.0f);
        v = __builtin_fmaf(v * q, r, r);
        u = fmaxf(u, 0.f) + 2.0f * v;
    }
    // (comparisons, which let a NaN pass)
    u = u < dt_min ? dt_min : u;
    return u > dt_max ? dt_max : u;
}

}  // namespace uniql
