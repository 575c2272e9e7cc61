// Attention of each request's newest tokens over its pages of the 4-bit cache: o = sum_j p_j v_j / sum_j p_j,
// p_j = exp(scale q . k_j - m), over the positions j that the row sees; k_j = s_j (c_j - 8), v_j = s'_j (c'_j - 8).
//
// A workgroup takes 16 rows (query heads of one key / value head, of one or several tokens) of a request over a run of positions;
// its four waves take 64 positions in turn.  Both products are matrix instructions of 16 x 16 x 32 on fp16 with the codes as they are: a code
// c in an fp16 number's low bits is the subnormal c 2^-24 (c 2^-20 four bits higher), which the instruction multiplies exactly, so that a
// pair of codes costs one mask.  Scales and, of the keys, the 8 that belongs off the codes come in around the products:
//   scores   scale s_j (2^24 (q . c_j 2^-24) - 8 sum q)      positions along the rows of the first product, so that
//   output   2^24 sum_j w_j ((c'_j - 8) 2^-24)               its results are the second one's operand in the lanes where they are
// (The values' 8 is taken off in front of the product, one more instruction a pair: behind it, over 65536 positions, the difference of two sums
// 80 times as large as itself was four times as far from the exact result.)
// with w_j = fp16(p_j s'_j).  For w_j to use fp16's range whatever the values' sizes, m is the running maximum of each
// position's score with the exponent of its s'_j, less 6: w_j is 2^5 to 2^6 at the maximum, and it moves only when some w_j might pass 2^14.  (Largest score
// and largest exponent apart save 1 % of the time, but lose small values that have the weight beside large ones that have none.)
// Beyond 2^22 (in powers of two), where such sums are rounded by as much as the room that weights have, m is the largest score alone.
// The rounding of w_j (2^-11) is what a matrix instruction on fp16 asks for; sums, maxima and the output stay in fp32.
//
// Bound by HBM: 132 bytes for a position of 128 + 128 channels (16 requests of 65536 tokens, 8 heads of 128: 198 us, 5.6 TB/s; a kernel
// that sums up 2 GB reads 6.1).  Fewer bytes are bound by latency: share, page numbers, positions, sums, exchange follow each other (1 x 4096
// 10.9 us, 48 requests of 1 to 8192 16.9: finding the share 1 us, the first positions 1.5, 1.5 for each further 64 a wave takes, the
// waves' sums 0.4, exchange and adding up 2).  The lengths are on the device, so every workgroup finds its share from them
// (tiles of 64 positions x tiles of 16 rows, shared out evenly): requests of any lengths fill the GPU alike.  Where several workgroups share a
// request's rows they leave (m, sum p, o) in scratch memory and the last to arrive adds them up in their order.
#include <algorithm>

#include "kv_attention.hpp"

namespace uniql {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x3 __attribute__((ext_vector_type(3)));

constexpr int kTile = 64;              // positions a wave takes at a time
constexpr int kRows = 16;              // rows of a workgroup
constexpr int kWaves = 4;
constexpr int kSlotFloats = 16 * 130;  // a workgroup's partial result: 16 rows of 128 channels, then (m, sum p) of each
constexpr int kDeviceScope = 16;       // cache policy bit sc1: as relaxed device-scope loads and stores compile to
constexpr int kOutStride = 132;
constexpr float kNoMaximum = -3.0e38f;
constexpr float kLift = 6.0f;          // weights at the maximum are 2^5 to 2^6: ones 2^-24 as large are many in a long cache and keep five bits
constexpr float kSlack = kLift + 8.0f; // they may grow by 2^8 before the maximum follows
constexpr float kFar = 4194304.0f;     // 2^22: below it a score's sum with an exponent is off by a quarter at most
// Workgroups that a call is shared out to, two a compute unit, as many as its registers allow to run at once: what does not fit waits for a
// whole one to end (us with 512 / 768 / 1024: 9 x 5 pruned 15 / 21 / 21, 48 requests 17 / 19 / 19, 16 x 65536 198 / 199 / 202, 1 x 4096 10.9
// for all).
constexpr int kWorkgroups = 512;

template <int S>
struct Words;
template <>
struct Words<1> { typedef uint32_t type; };
template <>
struct Words<2> { typedef u32x2 type; };
template <>
struct Words<3> { typedef u32x3 type __attribute__((aligned(4))); };
template <>
struct Words<4> { typedef u32x4 type; };
template <int S>
__device__ __forceinline__ uint32_t word_of(const typename Words<S>::type& v, int i) {
    if constexpr (S == 1) return v;
    else return v[i];
}

__device__ __forceinline__ float quad_max(float v) {  // over the lanes l, l ^ 16, l ^ 32, l ^ 48
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float quad_sum(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}
// Codes of two positions a word, less eight: exact, subnormal numbers and sums of them.
__device__ __forceinline__ uint32_t less_eight(uint32_t codes, uint32_t eight) { return h2_to_bits(bits_to_h2(codes) + bits_to_h2(eight)); }
__device__ __forceinline__ h8 halves(uint32_t a, uint32_t b, uint32_t c, uint32_t d) { return __builtin_bit_cast(h8, u32x4{a, b, c, d}); }
__device__ __forceinline__ h8 values_of(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t mask, uint32_t eight) {
    return halves(less_eight(a & mask, eight), less_eight(b & mask, eight), less_eight(c & mask, eight), less_eight(d & mask, eight));
}

// What a request asks for: its rows [first, first + count) and the positions in the cache.
struct Request {
    int first, count;
    int length;
};
// row / a.group for rows below 2^31 (see the launch)
__device__ __forceinline__ int query_of(const KvAttentionArgs& a, int row) { return (int)(((uint64_t)(unsigned)row * a.group_factor) >> a.group_shift); }
__device__ __forceinline__ int row_tiles(const KvAttentionArgs& a, const Request& q) { return (int)(((int64_t)q.count * a.group + kRows - 1) / kRows); }
__device__ __forceinline__ int position_tiles(const Request& q) { return (q.length + kTile - 1) / kTile; }

// Sums over the lanes up to and including each.
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned from_below(unsigned v) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false); }
template <typename Add>
__device__ __forceinline__ unsigned sums_upto(unsigned v, Add add) {
    v = add(v, from_below<0x111, 0xf>(v));  // one, two, four, eight lanes below, within sixteen
    v = add(v, from_below<0x112, 0xf>(v));
    v = add(v, from_below<0x114, 0xf>(v));
    v = add(v, from_below<0x118, 0xf>(v));
    v = add(v, from_below<0x142, 0xa>(v));  // the last of the sixteen below, for the second and fourth sixteen
    return add(v, from_below<0x143, 0xc>(v));  // lane 31, for the upper half
}
__device__ __forceinline__ unsigned lane_value(unsigned v, int lane) { return (unsigned)__builtin_amdgcn_readlane((int)v, lane); }

// The requests from `base` on, one a lane.  `end`: where the rows of those before end; offsets that fall count as ones that stay, so
// that all requests together have no more rows than there are, and no more workgroups than are launched: were some of those that
// share a request's rows missing, the others' count of arrivals would stay behind in `accum`.
__device__ __forceinline__ Request requests_of(const KvAttentionArgs& a, int base, unsigned& end) {
    const int lane = threadIdx.x & 63, r = base + lane;
    Request q = {0, 0, 0};
    if (a.cu_q) {
        int first = 0, last = 0;
        if (r < a.requests) {
            first = a.cu_q[r];
            last = a.cu_q[r + 1];
        }
        first = first < 0 ? 0 : (first > a.rows ? a.rows : first);
        last = last < 0 ? 0 : (last > a.rows ? a.rows : last);
        const auto larger = [](unsigned x, unsigned y) { return x > y ? x : y; };
        const unsigned begin = larger(sums_upto((unsigned)first, larger), end);
        const unsigned stop = larger(begin, (unsigned)last);
        q.first = (int)begin;
        q.count = r < a.requests ? (int)(stop - begin) : 0;
        end = lane_value(stop, 63);
    } else {
        q.first = r;
        q.count = r < a.requests ? 1 : 0;
    }
    if (r < a.requests) {
        const int64_t room = (int64_t)a.columns << a.cache.page_shift;
        const int n = a.lengths[r];
        q.length = n < 0 ? 0 : (n > room ? (int)room : n);
    }
    return q;
}

// A workgroup's share of a request's row tile `rows`.  Either the position tiles from `run * chunk` on, `run` of them, for one key /
// value head, a tile a wave in turn; `chunks` workgroups share these rows, and their partial results lie in the places `place - chunk`
// and on (rows of one workgroup need none: places are counted over those with whole runs, so there are at most twice as many as shares).
// Or, `alone`, all of its positions, a head a wave: requests too short to keep four waves busy.
struct Share {
    Request what;
    int request, rows, chunk, chunks, run, place, head;
    bool alone;
};
// How a request is taken apart: whole runs, and a rest or not; or alone.
struct Parts {
    int runs, rest, alone;
};
__device__ __forceinline__ Parts parts_of(int positions, int run, float by_run) {
    Parts p = {0, 0, 0};
    if (positions * kWaves <= run) {  // (rows that see nothing are among them)
        p.alone = 1;
        return p;
    }
    // positions / run from the quotient in fp32, which is off by one at most
    p.runs = (int)((float)positions * by_run);
    while ((int64_t)(p.runs + 1) * run <= positions) ++p.runs;
    while ((int64_t)p.runs * run > positions) --p.runs;
    p.rest = p.runs * run < positions;
    return p;
}
// Every wave finds it for itself.  Position tiles times row tiles of all requests, over the workgroups there are, give the run's
// length.  Whole runs come first, request after request, then the rests, then what is done alone: what takes longest starts first.
__device__ __forceinline__ bool find_share(const KvAttentionArgs& a, Share& s) {
    const int heads = a.cache.heads;
    const auto add_f = [](unsigned x, unsigned y) { return __builtin_bit_cast(unsigned, __builtin_bit_cast(float, x) + __builtin_bit_cast(float, y)); };
    const auto add_u = [](unsigned x, unsigned y) { return x + y; };
    Request q = {0, 0, 0};
    float total = 0.f;
    unsigned rows_end = 0;
    for (int base = 0; base < a.requests; base += 64) {
        q = requests_of(a, base, rows_end);
        const float mine = (float)row_tiles(a, q) * (float)position_tiles(q);
        total += __builtin_bit_cast(float, lane_value(sums_upto(__builtin_bit_cast(unsigned, mine), add_f), 63));
    }
    // (a little more than the quotient: sums in fp32 must not make more runs than there are workgroups for)
    const float run_f = total * 1.0001f / (float)a.shares;
    int run = run_f < 1.0e9f ? (int)run_f + 1 : 1 << 30;
    run = __builtin_amdgcn_readfirstlane((run + kWaves - 1) / kWaves * kWaves);
    const float by_run = 1.0f / (float)run;
    const unsigned index = blockIdx.x / (unsigned)heads;
    s.run = run;
    s.head = (int)(blockIdx.x - index * (unsigned)heads);
    // The first round over the requests looks for `index` among the whole runs, the second among the rests and what is done alone; the
    // sums up to a request tell where its places begin.
    // Whole runs, of which there are no more than shares, and the rests beside them go through one sum, sixteen bits each.
    unsigned all_runs = 0, all_rests = 0, alone_index = 0;
    bool alone = false;
    for (int round = 0; round < 2; ++round) {
        unsigned shared = 0, rests = 0, alones = 0;
        rows_end = 0;
        for (int base = 0; base < a.requests; base += 64) {
            if (a.requests > 64) q = requests_of(a, base, rows_end);
            const int tiles = row_tiles(a, q);
            const Parts p = parts_of(position_tiles(q), run, by_run);
            const int64_t want = (int64_t)tiles * p.runs;
            const unsigned some = tiles < (1 << 24) ? (unsigned)tiles : 1u << 24;  // (more than any grid has)
            const unsigned my_runs = want < 0x7fff ? (unsigned)want : 0x7fffu, my_rests = some * (unsigned)p.rest, my_alones = some * (unsigned)p.alone;
            const unsigned my_shared = my_runs | (p.runs > 0 ? my_rests << 16 : 0u);
            const unsigned upto_shared = shared + sums_upto(my_shared, add_u), upto_rests = rests + sums_upto(my_rests, add_u);
            const unsigned upto_runs = upto_shared & 0xffffu;
            unsigned upto = upto_runs, looked_for = index;
            if (round == 1) {
                const unsigned upto_alones = alones + sums_upto(my_alones, add_u);
                upto = alone ? upto_alones : all_runs + upto_rests;
                looked_for = alone ? alone_index : index;
                alones = lane_value(upto_alones, 63);
            }
            const unsigned long long above = __ballot(upto > looked_for);
            if (above) {
                const int owner = __builtin_ctzll(above);
                s.what = Request{(int)lane_value((unsigned)q.first, owner), (int)lane_value((unsigned)q.count, owner),
                                 (int)lane_value((unsigned)q.length, owner)};
                s.request = base + owner;
                s.alone = alone;
                const int r = (int)lane_value((unsigned)p.runs, owner);
                s.chunks = alone ? 1 : r + (int)lane_value((unsigned)p.rest, owner);
                const unsigned before = lane_value(upto_shared - my_shared, owner);
                if (round == 0) {
                    const int at = (int)(index - (before & 0xffffu));
                    s.rows = r == 1 ? at : at / r;
                    s.chunk = at - s.rows * r;
                } else {
                    s.rows = (int)(looked_for - lane_value(upto - (alone ? my_alones : my_rests), owner));
                    s.chunk = alone ? 0 : r;
                }
                s.place = (int)((before & 0xffffu) + (before >> 16)) + s.rows * s.chunks + s.chunk;
                return true;
            }
            shared = lane_value(upto_shared, 63);
            rests = lane_value(upto_rests, 63);
            if ((rests | alones) > 0x1fffffffu) return false;
        }
        all_runs = shared & 0xffffu;
        all_rests = rests;
        if (round == 0 && index >= all_runs + all_rests) {
            alone = true;
            const unsigned groups = (unsigned)(heads + kWaves - 1) / kWaves, at = blockIdx.x - (all_runs + all_rests) * (unsigned)heads;
            alone_index = at / groups;
            s.head = (int)(at - alone_index * groups) * kWaves + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
        }
    }
    return false;
}

// What a wave reads for 64 positions.
template <int S>
struct Positions {
    typename Words<S>::type k[4];
    u32x4 v[4];
    uint64_t k_scales[4], v_scales[4];
};

template <int S>
__global__ __launch_bounds__(256, 2) void kv4_attention_kernel(const KvAttentionArgs a) {
    __shared__ __attribute__((aligned(16))) float merge[kWaves * 16 * kOutStride];
    __shared__ float merge_m[kWaves * 16], merge_l[kWaves * 16];
    __shared__ int last_flag;
    const KvCache& c = a.cache;
    const int heads = c.heads;
    Share s;
    if (!find_share(a, s)) return;
    const bool head_exists = s.head < heads;  // (of four heads that are done alone some may not)
    const int kv_head = head_exists ? s.head : heads - 1;
    const Request rq = s.what;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, quad = lane >> 4;
    const int rows_total = rq.count * a.group, flat = s.rows * kRows + col;
    const bool row_exists = flat < rows_total && head_exists;
    const int token = row_exists ? query_of(a, flat) : 0, sub_head = row_exists ? flat - token * a.group : 0;
    // positions that the lane's row sees; the first and the last row of the tile have the fewest and the most
    const int limit = row_exists ? rq.length - rq.count + token + 1 : 0;
    const int last_flat = rows_total - 1 < s.rows * kRows + kRows - 1 ? rows_total - 1 : s.rows * kRows + kRows - 1;
    const int seen_by_all = rq.length - rq.count + query_of(a, s.rows * kRows) + 1, seen_by_any = rq.length - rq.count + query_of(a, last_flat) + 1;
    const int tiles = (seen_by_any + kTile - 1) / kTile;
    const int end = s.alone ? (head_exists ? tiles : 0) : ((s.chunk + 1) * s.run < tiles ? (s.chunk + 1) * s.run : tiles);
    const int step = s.alone ? 1 : kWaves;

    const int32_t* table = a.table + (int64_t)s.request * a.columns;
    const int last_column = rq.length > 0 ? (rq.length - 1) >> c.page_shift : 0;
    const int n_word = col < c.v_words ? col : 0;
    const uint32_t mask_low = 0x000f000fu, mask_high = 0x00f000f0u;
    const uint32_t eight_low = 0x80088008u, eight_high = 0x80808080u;  // -8 2^-24 and -8 2^-20, twice
    struct Pages {
        int page[4];
    };
    auto pages_of = [&](int t) __attribute__((always_inline)) {
        Pages p;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int column = (t * kTile + 16 * u) >> c.page_shift;
            p.page[u] = table[column < last_column ? column : last_column];
        }
        return p;
    };
    auto load = [&](int t, const Pages& p) __attribute__((always_inline)) {
        Positions<S> x;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const bool there = (unsigned)p.page[u] < (unsigned)c.pages;
            const int64_t at = (((int64_t)(there ? p.page[u] : 0) * heads + kv_head) << c.page_shift) + ((t * kTile + 16 * u) & ((1 << c.page_shift) - 1));
            x.k[u] = *reinterpret_cast<const typename Words<S>::type*>(c.k_codes + at * (4 * S) + col * (4 * S) + quad * S);
            x.k_scales[u] = *reinterpret_cast<const uint64_t*>(c.k_scales + at + 4 * quad);
            x.v_scales[u] = *reinterpret_cast<const uint64_t*>(c.v_scales + at + 4 * quad);
            x.v[u] = *reinterpret_cast<const u32x4*>(c.v_codes + at * c.v_words + quad * (4 * c.v_words) + 4 * n_word);
        }
        return x;
    };
    int t = s.alone ? 0 : s.chunk * s.run + wave;
    Pages pages = pages_of(t);
    h8 q[S];
    {
        const half_t* row = a.q + (int64_t)(rq.first + token) * a.q_row + (int64_t)(kv_head * a.group + sub_head) * a.q_head;
#pragma unroll
        for (int i = 0; i < S; ++i) {
            q[i] = h8{};
            if (row_exists) q[i] = load_eight_of(row, 8 * (S * quad + i), c.k_dim);
        }
    }
    Positions<S> next = {};
    if (t < end) next = load(t, pages);
    Pages next_pages = pages_of(t + step);

    float q_sum = 0.f;
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) q_sum += (float)q[i][j];
    q_sum = quad_sum(q_sum);
    const float log2e = 1.4426950408889634f;
    const float by_code = a.scale * log2e * 16777216.0f, by_sum = -8.0f * q_sum * a.scale * log2e;

    f4 out[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = f4{0.f, 0.f, 0.f, 0.f};
    float m = kNoMaximum, l = 0.f;

    for (; t < end; t += step) {
        const int j0 = t * kTile;
        typename Words<S>::type kw[4];
        u32x4 vw[4];
        uint64_t ks[4], vs[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            kw[u] = next.k[u], vw[u] = next.v[u], ks[u] = next.k_scales[u], vs[u] = next.v_scales[u];
            if ((unsigned)pages.page[u] >= (unsigned)c.pages) ks[u] = 0x7e007e007e007e00ull;  // no such page: NaN
        }
        pages = next_pages;
        if (t + step < end) next = load(t + step, pages);
        next_pages = pages_of(t + 2 * step);
        float score[16];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            f4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < S; ++i) {
                const uint32_t w = word_of<S>(kw[u], i);
                acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                    halves(w & mask_low, (w >> 4) & mask_low, (w >> 8) & mask_low, (w >> 12) & mask_low), q[i], acc, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const half_t scale = __builtin_bit_cast(half_t, (uint16_t)(ks[u] >> (16 * i)));
                score[4 * u + i] = (acc[i] * by_code + by_sum) * (float)scale;
            }
        }
        const bool masked = j0 + kTile > seen_by_all;
        if (masked) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                uint64_t keep = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int j = j0 + 16 * u + 4 * quad + i;
                    if (j < limit) keep |= 0xffffull << (16 * i);
                    else score[4 * u + i] = -INFINITY;
                }
                vs[u] &= keep;
            }
        }
        // the largest score with its value's exponent, 14 too large: the scale's bits are its exponent, and 0 for zero and what is masked
        float top = -INFINITY;
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                top = fmaxf(top, score[4 * u + i] + (float)(unsigned)((uint32_t)(vs[u] >> (16 * i + 10)) & 31u));
        top -= 14.f;
        if (__any(top - m > kSlack)) {
            const float row_top = quad_max(top);
            const bool far = fabsf(row_top) > kFar;
            float wanted = row_top - kLift;
            if (__any(far)) {
                // Sums of scores that large and exponents are rounded by more than the room: the scores alone, which are exact
                // beside each other; weights then reach the scales themselves, 2^14 at most.
                float highest = -INFINITY;
#pragma unroll
                for (int i = 0; i < 16; ++i) highest = fmaxf(highest, score[i]);
                highest = quad_max(highest);
                wanted = far ? highest : wanted;
            }
            const float next = fmaxf(m, wanted);
            const float fade = __builtin_amdgcn_exp2f(m - next);
            m = next;
            l *= fade;
#pragma unroll
            for (int i = 0; i < 8; ++i) out[i] *= fade;
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            h8 weight;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int u = 2 * k + h;
                    const float p = __builtin_amdgcn_exp2f(score[4 * u + i] - m);
                    l += p;
                    weight[4 * h + i] = (half_t)(p * (float)__builtin_bit_cast(half_t, (uint16_t)(vs[u] >> (16 * i))));
                }
            const u32x4 first = vw[2 * k], second = vw[2 * k + 1];
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                // byte b of four and four tokens' words, two tokens a register: value 2 (b & 1) .. in its low nibble, the next but one above
                const uint32_t pick = 0x0c000c00u + ((uint32_t)(4 + b) << 16) + (uint32_t)b;
                const uint32_t x0 = __builtin_amdgcn_perm(first[1], first[0], pick), x1 = __builtin_amdgcn_perm(first[3], first[2], pick);
                const uint32_t x2 = __builtin_amdgcn_perm(second[1], second[0], pick), x3 = __builtin_amdgcn_perm(second[3], second[2], pick);
                const int low = 4 * (b & 1) + (b >> 1), high = low + 2;
                out[low] = __builtin_amdgcn_mfma_f32_16x16x32_f16(values_of(x0, x1, x2, x3, mask_low, eight_low), weight, out[low], 0, 0, 0);
                out[high] = __builtin_amdgcn_mfma_f32_16x16x32_f16(values_of(x0, x1, x2, x3, mask_high, eight_high), weight, out[high], 0, 0, 0);
            }
        }
    }
    l = quad_sum(l);
    // the lane's row: channels 32 quad + 8 i + (0 .. 7); value index 2, 3, 6, 7 came from the high nibbles
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float* to = merge + (wave * 16 + col) * kOutStride + 32 * quad + 8 * i;
        f4 lo, hi;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float unit = (j & 2) ? 1048576.0f : 16777216.0f;
            lo[j] = out[j][i] * unit;
            hi[j] = out[4 + j][i] * unit;
        }
        *reinterpret_cast<f4*>(to) = lo;
        *reinterpret_cast<f4*>(to + 4) = hi;
    }
    if (quad == 0) {
        merge_m[wave * 16 + col] = m;
        merge_l[wave * 16 + col] = l;
    }
    __syncthreads();
    // eight channels of a row
    auto finish = [&](int row, int head, int channel, const float (&o)[8], float sum) __attribute__((always_inline)) {
        const int of_token = query_of(a, row), q_head = head * a.group + row - of_token * a.group;
        const bool empty = rq.length - rq.count + of_token + 1 <= 0;
        half_t* to = a.out + (int64_t)(rq.first + of_token) * a.out_row + (int64_t)q_head * a.out_head + channel;
        h8u result;
#pragma unroll
        for (int i = 0; i < 8; ++i) result[i] = empty ? (half_t)0.f : (half_t)(o[i] / sum);
        if (channel + 8 <= c.v_dim) {
            *reinterpret_cast<h8u*>(to) = result;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (channel + i < c.v_dim) to[i] = result[i];
        }
    };
    if (s.alone) {
        for (int i = 0; i < 4; ++i) {
            const int row = 4 * i + quad, flat_row = s.rows * kRows + row;
            if (flat_row >= rows_total || !head_exists) break;
            const float* from = merge + (wave * 16 + row) * kOutStride + 8 * col;
            const float mine[8] = {from[0], from[1], from[2], from[3], from[4], from[5], from[6], from[7]};
            finish(flat_row, kv_head, 8 * col, mine, merge_l[wave * 16 + row]);
        }
        return;
    }
    // a thread: eight channels of a row, of all four waves' positions
    int my_row = tid >> 4;
    const int my_channel = 8 * (tid & 15);
    float top = kNoMaximum, sum = 0.f, o[8] = {};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, merge_m[w * 16 + my_row]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        const float part = __builtin_amdgcn_exp2f(merge_m[w * 16 + my_row] - top);
        sum += merge_l[w * 16 + my_row] * part;
        const float* from = merge + (w * 16 + my_row) * kOutStride + my_channel;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] += from[i] * part;
    }
    int my_flat = s.rows * kRows + my_row;
    const bool mine = my_flat < rows_total;
    if (s.chunks > 1) {
        // The exchange: relaxed stores at device scope, which pass the local L2; a wait until they have been acknowledged; the
        // barrier; the count.  The last to arrive reads with relaxed loads at device scope.
        const __amdgpu_buffer_rsrc_t slot =
            __builtin_amdgcn_make_buffer_rsrc(a.temp + ((int64_t)s.place * heads + kv_head) * kSlotFloats, 0, (unsigned)kSlotFloats * 4u, 0x00020000);
        if (mine) {
            const uint32_t at = 4u * (uint32_t)(my_row * 128 + my_channel);
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, f4{o[0], o[1], o[2], o[3]}), slot, at, 0, kDeviceScope);
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, f4{o[4], o[5], o[6], o[7]}), slot, at + 16u, 0, kDeviceScope);
            if ((tid & 15) == 0)
                __builtin_amdgcn_raw_buffer_store_b64(u32x2{__builtin_bit_cast(uint32_t, top), __builtin_bit_cast(uint32_t, sum)}, slot,
                                                      8192u + 8u * (uint32_t)my_row, 0, kDeviceScope);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        unsigned* count = reinterpret_cast<unsigned*>(a.accum) + (int64_t)(s.place - s.chunk) * heads + kv_head;
        if (tid == 0) last_flag = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)s.chunks - 1;
        __syncthreads();
        if (!last_flag) return;
        if (tid == 0) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        asm volatile("" ::: "memory");
        // Rows of the tile that exist, times slices of the partial results: all threads read, four results on their way at a time.
        const int rows_here = rows_total - s.rows * kRows < kRows ? rows_total - s.rows * kRows : kRows;
        int shift = 0;
        while ((1 << shift) < rows_here) ++shift;
        const int slices = kRows >> shift, slice = (tid >> 4) >> shift;
        my_row = (tid >> 4) & ((1 << shift) - 1);
        top = kNoMaximum, sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = 0.f;
        for (int first = slice; first < s.chunks; first += 4 * slices) {
            u32x4 lo[4], hi[4];
            u32x2 ml[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int from = first + k * slices < s.chunks ? first + k * slices : first;
                const __amdgpu_buffer_rsrc_t part = __builtin_amdgcn_make_buffer_rsrc(a.temp + ((int64_t)(s.place - s.chunk) * heads + kv_head) * kSlotFloats, 0,
                                                                                      0xffffffffu, 0x00020000);
                const uint32_t at = 4u * (uint32_t)from * (uint32_t)(heads * kSlotFloats);
                lo[k] = __builtin_amdgcn_raw_buffer_load_b128(part, at + 4u * (uint32_t)(my_row * 128 + my_channel), 0, kDeviceScope);
                hi[k] = __builtin_amdgcn_raw_buffer_load_b128(part, at + 4u * (uint32_t)(my_row * 128 + my_channel) + 16u, 0, kDeviceScope);
                ml[k] = __builtin_amdgcn_raw_buffer_load_b64(part, at + 8192u + 8u * (uint32_t)my_row, 0, kDeviceScope);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (first + k * slices >= s.chunks) break;
                const uint32_t m_bits = ml[k][0], l_bits = ml[k][1];  // (a bit cast of an element takes the vector's first one)
                const float other = __builtin_bit_cast(float, m_bits), other_sum = __builtin_bit_cast(float, l_bits);
                const float higher = fmaxf(top, other), keep = __builtin_amdgcn_exp2f(top - higher), add = __builtin_amdgcn_exp2f(other - higher);
                top = higher;
                sum = sum * keep + other_sum * add;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    o[i] = o[i] * keep + __builtin_bit_cast(f4, lo[k])[i] * add;
                    o[4 + i] = o[4 + i] * keep + __builtin_bit_cast(f4, hi[k])[i] * add;
                }
            }
        }
        if (slices > 1) {
            float* const to = merge + (tid >> 4) * kOutStride + my_channel;
            *reinterpret_cast<f4*>(to) = f4{o[0], o[1], o[2], o[3]};
            *reinterpret_cast<f4*>(to + 4) = f4{o[4], o[5], o[6], o[7]};
            merge_m[tid >> 4] = top;
            merge_l[tid >> 4] = sum;
            __syncthreads();
            if (slice > 0) return;
            for (int k = 1; k < slices; ++k) {
                const int at = my_row + (k << shift);
                const float other = merge_m[at], higher = fmaxf(top, other);
                const float keep = __builtin_amdgcn_exp2f(top - higher), add = __builtin_amdgcn_exp2f(other - higher);
                top = higher;
                sum = sum * keep + merge_l[at] * add;
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] = o[i] * keep + merge[at * kOutStride + my_channel + i] * add;
            }
        }
        my_flat = s.rows * kRows + my_row;
        if (my_row >= rows_here) return;
    } else if (!mine) {
        return;
    }
    finish(my_flat, kv_head, my_channel, o, sum);
}

// Workgroups for each key / value head: one for each run, and one more for each row tile whose last run is not whole.
static int64_t shares_of(int heads) { return heads < kWorkgroups ? (kWorkgroups + heads - 1) / heads : 1; }
static int64_t workgroups_of(int rows, int requests, int group, int heads, bool single) {
    const int64_t tiles = single ? (int64_t)rows * ((group + kRows - 1) / kRows)
                                 : (int64_t)rows * group / kRows + (requests < rows ? requests : rows);
    return shares_of(heads) + tiles;
}

void kv4_attention_needs(int rows, int requests, int q_heads, const KvCache& cache, size_t* accum_bytes, size_t* temp_bytes) {
    // (with and without cu_q alike: the larger of the two)
    const int group = q_heads / cache.heads;
    const int64_t one = workgroups_of(rows, requests, group, cache.heads, true), many = workgroups_of(rows, requests, group, cache.heads, false);
    const int64_t workgroups = rows == requests && one > many ? one : many;
    // rows that several workgroups share have a whole run at least, and one rest: two places for a share
    const int64_t places = std::min(workgroups, 2 * shares_of(cache.heads)) * cache.heads;
    *accum_bytes = (size_t)(places * 4 + 7) / 8 * 8;
    *temp_bytes = (size_t)places * kSlotFloats * 4;
}

int kv4_attention_launch(const KvAttentionArgs& args, hipStream_t stream) {
    KvAttentionArgs a = args;
    a.shares = (int)shares_of(a.cache.heads);
    // floor(row / d) = row f >> (31 + s) with f = 2^(31 + s) / d rounded up and s so that d <= 2^s < 2 d
    int shift = 0;
    while ((1 << shift) < a.group) ++shift;
    a.group_shift = 31 + shift;
    a.group_factor = (unsigned)(((1ULL << a.group_shift) + a.group - 1) / a.group);
    const int64_t workgroups = workgroups_of(a.rows, a.requests, a.group, a.cache.heads, a.cu_q == nullptr) * a.cache.heads;
    if (workgroups >= (1LL << 32) / (64 * kWaves)) return UNIQL_E_SHAPE;  // (threads of a grid)
    const dim3 grid((unsigned)workgroups), block(64 * kWaves);
    switch (a.cache.k_words / 4) {
        case 1: hipLaunchKernelGGL(kv4_attention_kernel<1>, grid, block, 0, stream, a); break;
        case 2: hipLaunchKernelGGL(kv4_attention_kernel<2>, grid, block, 0, stream, a); break;
        case 3: hipLaunchKernelGGL(kv4_attention_kernel<3>, grid, block, 0, stream, a); break;
        default: hipLaunchKernelGGL(kv4_attention_kernel<4>, grid, block, 0, stream, a); break;
    }
    return hipGetLastError() == hipSuccess ? UNIQL_OK : UNIQL_E_LAUNCH;
}

}  // namespace uniql
