// The paged 4-bit key / value cache: which pages a request holds and where its new tokens go (assign), writing keys and
// values into it (store), reading them back as fp16 (load).
//
// A vector x of one token and one key / value head is held as s (c - 8), s = fp16(max|x| 2/15), c = clamp(round(x / s) + 8, 0, 15),
// the arithmetic of the 4-bit projections with one scale for the vector.  Layout: see KvCache in kv_cache.hpp.
#include "kv_cache.hpp"

namespace uniql {

// ---- pages and slots ---------------------------------------------------------------------------------------------
struct AssignArgs {
    const int32_t *new_tokens, *lengths;
    int32_t *table, *free_pages;
    const int32_t* free_count;
    int32_t *lengths_out, *free_count_out;
    int64_t* slots;
    int32_t *positions, *cu, *refused;
    int rows, columns, pool, page_shift, max_tokens;
};
constexpr int kAssignThreads = 1024;

// Sums over the workgroup's threads up to and including each, and the whole sum; within a wave in 32 bits.  wave_sums is the scan's own:
// between two uses of it all threads have met.
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned add_from(unsigned v) {
    return v + (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int64_t scan_inclusive(unsigned v, unsigned* wave_sums, int64_t& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    v = add_from<0x111, 0xf>(v);  // one, two, four, eight lanes below, within sixteen
    v = add_from<0x112, 0xf>(v);
    v = add_from<0x114, 0xf>(v);
    v = add_from<0x118, 0xf>(v);
    v = add_from<0x142, 0xa>(v);  // the last of the sixteen below, for the second and fourth sixteen
    v = add_from<0x143, 0xc>(v);  // lane 31, for the upper half
    if (lane == 63) wave_sums[wave] = v;
    __syncthreads();
    int64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kAssignThreads / 64; ++w) {
        const unsigned s = wave_sums[w];
        if (w < wave) before += s;
        total += s;
    }
    return v + before;
}

// The first of `count` ascending values that is greater than `v`.
template <typename P>
__device__ __forceinline__ int first_above(const P* ascending, int count, int v) {
    int low = 0, high = count;
    while (low < high) {
        const int mid = (low + high) >> 1;
        if (ascending[mid] > v) high = mid;
        else low = mid + 1;
    }
    return low;
}

// Where token t of the batch goes.  `old`: tokens the request held before, or -1 where it was refused.
__device__ __forceinline__ void place_token(const AssignArgs& a, int t, int request, int first, int old) {
    const int position = old < 0 ? 0 : old + (t - first);
    int64_t slot = -1;
    if (old >= 0) {
        const int64_t page = a.table[(int64_t)request * a.columns + (position >> a.page_shift)];
        slot = (page << a.page_shift) + (position & ((1 << a.page_shift) - 1));
    }
    a.slots[t] = slot;
    a.positions[t] = position;
}

// Bound by latency (64 requests 5 us with the launch; 500 requests with 37386 tokens 8 us and 4 for the tokens' kernel).
// One workgroup: releases, then requests in order, both by prefix sums over the rows; pages are moved by a flat loop over pages,
// each of which finds its row among the sums, so that one request with thousands of pages takes no longer than many with a few.
// PLACE: it also places the tokens (a small batch: no second launch).
template <bool PLACE>
__global__ __launch_bounds__(kAssignThreads) void kv_assign_kernel(const AssignArgs a) {
    __shared__ unsigned sums[3][kAssignThreads / 64];
    __shared__ int upto[kAssignThreads], upto_tokens[kAssignThreads], held_by[kAssignThreads], used;
    const int tid = threadIdx.x;
    const int page = 1 << a.page_shift;
    const int64_t capacity = (int64_t)a.columns << a.page_shift;
    if (tid == 0) used = 0;
    // what the first rows ask for and hold is read once, with the count
    const int first_asked = tid < a.rows ? a.new_tokens[tid] : 0, first_held = tid < a.rows ? a.lengths[tid] : 0;
    int count = *a.free_count;
    count = count < 0 ? 0 : (count > a.pool ? a.pool : count);
    for (int base = 0; base < a.rows; base += kAssignThreads) {
        const int r = base + tid;
        int pages = 0;
        if (r < a.rows && (base == 0 ? first_asked : a.new_tokens[r]) < 0) {
            int64_t n = base == 0 ? first_held : a.lengths[r];
            n = n < 0 ? 0 : (n > capacity ? capacity : n);
            pages = (int)((n + page - 1) >> a.page_shift);
        }
        int64_t released;
        const int sum = (int)scan_inclusive((unsigned)pages, sums[0], released);
        const int total = (int)released;  // at most 2^30
        if (total > 0) {
            upto[tid] = sum;
            held_by[tid] = pages;
            __syncthreads();
            for (int i = tid; i < total; i += kAssignThreads) {
                const int row = first_above(upto, kAssignThreads, i), j = i - (upto[row] - held_by[row]);
                if (i < a.pool - count) a.free_pages[count + i] = a.table[(int64_t)(base + row) * a.columns + j];
            }
            count = total > a.pool - count ? a.pool : count + total;
        }
        __syncthreads();  // (the sums have been read; released pages are on the list)
    }
    int64_t tokens_before = 0;
    int64_t pages_before = 0;
    for (int base = 0; base < a.rows; base += kAssignThreads) {
        const int r = base + tid;
        const bool exists = r < a.rows;
        const int asked = base == 0 ? first_asked : (exists ? a.new_tokens[r] : 0), n = asked > 0 ? asked : 0;
        const int64_t old = base == 0 ? first_held : (exists ? a.lengths[r] : 0);
        int64_t tokens, pages_total;
        // (more than max_tokens count as one more)
        const int64_t sum_tokens = tokens_before + scan_inclusive((unsigned)(n <= a.max_tokens ? n : a.max_tokens + 1), sums[1], tokens);
        const bool fits = n > 0 && old >= 0 && old + n <= capacity && sum_tokens <= a.max_tokens;
        const int held = (int)((old + page - 1) >> a.page_shift);
        const int need = fits ? (int)((old + n + page - 1) >> a.page_shift) - held : 0;
        const int64_t sum_pages = pages_before + scan_inclusive((unsigned)need, sums[2], pages_total);
        const bool served = fits && (need == 0 || sum_pages <= count);
        const int end = sum_tokens < a.max_tokens ? (int)sum_tokens : a.max_tokens;
        if (PLACE) upto_tokens[tid] = end;
        if (exists) {
            a.cu[r + 1] = end;
            a.refused[r] = n > 0 && !served;
            a.lengths_out[r] = asked < 0 ? 0 : (int)(served ? old + n : old);
        }
        // those that are served and need pages come before all that are refused for want of them
        const int64_t mine = sum_pages - pages_before;
        upto[tid] = (int)(mine < 0x7fffffff ? mine : 0x7fffffff);
        held_by[tid] = need;
        __shared__ int first_page[kAssignThreads], old_or_none[kAssignThreads];
        first_page[tid] = held;
        old_or_none[tid] = served ? (int)old : -1;
        if (served && need) atomicMax(&used, (int)sum_pages);
        __syncthreads();
        const int64_t give64 = (int64_t)used - pages_before;
        const int give = give64 > 0 ? (int)give64 : 0;
        for (int i = tid; i < give; i += kAssignThreads) {
            const int row = first_above(upto, kAssignThreads, i), j = i - (upto[row] - held_by[row]);
            a.table[(int64_t)(base + row) * a.columns + first_page[row] + j] = a.free_pages[count - 1 - (pages_before + i)];
        }
        if (PLACE) {
            __syncthreads();
            for (int t = tid; t < a.max_tokens; t += kAssignThreads) {
                const int row = first_above(upto_tokens, a.rows, t);
                const bool there = row < a.rows;
                place_token(a, t, row, there && row > 0 ? upto_tokens[row - 1] : 0, there ? old_or_none[row] : -1);
            }
        }
        tokens_before += tokens;
        pages_before += pages_total;
        __syncthreads();
    }
    if (PLACE && a.rows == 0)
        for (int t = tid; t < a.max_tokens; t += kAssignThreads) place_token(a, t, 0, 0, -1);
    __syncthreads();
    if (tid == 0) {
        a.cu[0] = 0;
        *a.free_count_out = count - used;
    }
}

// Larger batches: a token a thread, behind the kernel above.
__global__ __launch_bounds__(256) void kv_place_kernel(const AssignArgs a) {
    const int t = (int)blockIdx.x * 256 + (int)threadIdx.x;
    if (t >= a.max_tokens) return;
    const int request = first_above(a.cu + 1, a.rows, t);
    const bool served = request < a.rows && a.refused[request] == 0;
    place_token(a, t, request, served ? a.cu[request] : 0, served ? a.lengths_out[request] - a.new_tokens[request] : -1);
}

int kv_assign_launch(const int32_t* new_tokens, const int32_t* lengths, int32_t* table, int32_t* free_pages, const int32_t* free_count,
                     int32_t* lengths_out, int32_t* free_count_out, int64_t* slots, int32_t* positions, int32_t* cu, int32_t* refused,
                     int rows, int columns, int pool, int page_size, int max_tokens, hipStream_t stream) {
    const AssignArgs a = {new_tokens, lengths, table, free_pages, free_count, lengths_out, free_count_out, slots, positions, cu, refused,
                          rows, columns, pool, __builtin_ctz((unsigned)page_size), max_tokens};
    // Up to four tokens a thread the one workgroup places them itself, beyond that the whole GPU in a second launch (2.8 us and more).
    const bool place = rows <= kAssignThreads && max_tokens <= 4096;
    if (place) {
        hipLaunchKernelGGL(kv_assign_kernel<true>, dim3(1), dim3(kAssignThreads), 0, stream, a);
    } else {
        hipLaunchKernelGGL(kv_assign_kernel<false>, dim3(1), dim3(kAssignThreads), 0, stream, a);
        if (max_tokens > 0)
            hipLaunchKernelGGL(kv_place_kernel, dim3(((unsigned)max_tokens + 255u) / 256u), dim3(256), 0, stream, a);
    }
    return hipGetLastError() == hipSuccess ? UNIQL_OK : UNIQL_E_LAUNCH;
}

// ---- store ---------------------------------------------------------------------------------------------------------
// Bound by HBM: 16384 tokens of 8 heads of 128 stored in 20 us (4.3 TB/s of fp16 read and codes written), loaded in 17 (5.0).
// Both kernels below: sixteen lanes take a token's key and value of one head, eight values of each a lane, consecutive tokens beside
// each other, so that the words of four tokens that lie together in the cache are written and read together.
struct StoreArgs {
    const half_t *k, *v;
    int64_t k_row, k_head, v_row, v_head;
    const int64_t* slots;
    KvCache cache;
    int tokens;
};

// The scale and the word of codes of this lane's eight values of a vector.
__device__ __forceinline__ half_t quantise(h8 v, uint32_t& word) {
    uint32_t top = 0;  // the largest magnitude's bits: they order as the magnitudes do, infinities and NaN above all
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const half_t value = v[i];  // (a bit cast of the element itself takes the vector's first one)
        const uint32_t bits = __builtin_bit_cast(uint16_t, value) & 0x7fffu;
        top = bits > top ? bits : top;
    }
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) {
        const uint32_t other = (uint32_t)__shfl_xor((int)top, d, 64);
        top = other > top ? other : top;
    }
    const bool finite = top < 0x7c00u;
    // fp16(max 2/15): twice an 11-bit number over 15 stays 2^-16 of itself away from the midpoints between fp16 numbers, so
    // the products' and the constant's errors in fp32 (2^-23) do not show
    const half_t scale = finite ? scaled_to_half((float)__builtin_bit_cast(half_t, (uint16_t)top), 2.0f / 15.0f)
                                : __builtin_bit_cast(half_t, (uint16_t)0x7e00);
    const float s = (float)scale;
    const bool usable = finite && s > 0.f;
    const float by_scale = usable ? 1.0f / s : 0.f;
    // x / s is a midpoint between whole numbers or at least 2^-12 away from one (both have 11 bits, and their quotient is below 8);
    // x (1/s) is 2^-20 away from it at most.  Rounded to multiples of 2^-13 first, which adding and taking off 1536 does, a midpoint is
    // one again and nothing else becomes one: no division for each value (with one: 33.8 us where this and keys and values
    // in one workgroup take 19.7).
    word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float x = (float)v[i] * by_scale + 1536.0f;
        asm volatile("" : "+v"(x));
        const float c = usable ? fminf(fmaxf(rintf(x - 1536.0f), -8.f), 7.f) : 0.f;
        word |= (uint32_t)((int)c + 8) << kNibble(i);
    }
    return scale;
}

__global__ __launch_bounds__(256) void kv4_store_kernel(const StoreArgs a) {
    const int token = (int)(blockIdx.x * 16 + (threadIdx.x >> 4)), head = blockIdx.y, part = threadIdx.x & 15;
    if (token >= a.tokens) return;
    const KvCache& c = a.cache;
    const int64_t slot = a.slots[token];
    const h8 k = load_eight_of(a.k + token * a.k_row + head * a.k_head, part * 8, c.k_dim);
    const h8 v = load_eight_of(a.v + token * a.v_row + head * a.v_head, part * 8, c.v_dim);
    if (slot < 0 || slot >= ((int64_t)c.pages << c.page_shift)) return;
    uint32_t k_word, v_word;
    const half_t k_scale = quantise(k, k_word), v_scale = quantise(v, v_word);
    if (part < c.k_words) c.k_codes[c.k_word(slot, head, part)] = k_word;
    if (part < c.v_words) c.v_codes[c.v_word(slot, head, part)] = v_word;
    if (part == 0) {
        c.k_scales[c.scale_at(slot, head)] = k_scale;
        c.v_scales[c.scale_at(slot, head)] = v_scale;
    }
}

int kv4_store_launch(const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head, const int64_t* slots,
                     const KvCache& cache, int tokens, hipStream_t stream) {
    const StoreArgs a = {reinterpret_cast<const half_t*>(k), reinterpret_cast<const half_t*>(v), k_row, k_head, v_row, v_head, slots, cache,
                         tokens};
    hipLaunchKernelGGL(kv4_store_kernel, dim3(((unsigned)tokens + 15u) / 16u, (unsigned)cache.heads), dim3(256), 0, stream, a);
    return hipGetLastError() == hipSuccess ? UNIQL_OK : UNIQL_E_LAUNCH;
}

// ---- load ----------------------------------------------------------------------------------------------------------
struct LoadArgs {
    KvCache cache;
    const int32_t *table, *cu, *starts;
    half_t *k, *v;
    int64_t k_row, k_head, v_row, v_head;
    int requests, columns, rows;
};

// Eight values of a vector from column j on, as far as the vector goes: a product of a code and a scale is rounded once.
__device__ __forceinline__ void put_eight(half_t* x, int j, int width, uint32_t word, half_t s) {
    const h2 s2 = {s, s};
    const h2 p0 = code_pair_low(word) * s2, p1 = code_pair_high(word) * s2, p2 = code_pair_low(word >> 8) * s2,
             p3 = code_pair_high(word >> 8) * s2;
    const h8u out = {p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
    if (j + 8 <= width) {
        *reinterpret_cast<h8u*>(x + j) = out;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (j + i < width) x[j + i] = out[i];
    }
}

__global__ __launch_bounds__(256) void kv4_load_kernel(const LoadArgs a) {
    const int row = (int)(blockIdx.x * 16 + (threadIdx.x >> 4)), head = blockIdx.y, part = threadIdx.x & 15;
    const KvCache& c = a.cache;
    if (row >= a.rows || row < a.cu[0]) return;
    const int request = first_above(a.cu + 1, a.requests, row);
    if (request >= a.requests) return;   // behind the last request
    const int64_t position = (int64_t)row - a.cu[request] + (a.starts ? a.starts[request] : 0);
    const int64_t column = position >> c.page_shift;
    int64_t page = -1;
    if (position >= 0 && column < a.columns) page = a.table[(int64_t)request * a.columns + column];
    uint32_t k_word = 0, v_word = 0;
    half_t k_scale = __builtin_bit_cast(half_t, (uint16_t)0x7e00), v_scale = k_scale;   // no such page: NaN
    if (page >= 0 && page < c.pages) {
        const int64_t slot = (page << c.page_shift) + (position & ((1 << c.page_shift) - 1));
        if (part < c.k_words) k_word = c.k_codes[c.k_word(slot, head, part)];
        if (part < c.v_words) v_word = c.v_codes[c.v_word(slot, head, part)];
        k_scale = c.k_scales[c.scale_at(slot, head)];
        v_scale = c.v_scales[c.scale_at(slot, head)];
    }
    put_eight(a.k + row * a.k_row + head * a.k_head, part * 8, c.k_dim, k_word, k_scale);
    put_eight(a.v + row * a.v_row + head * a.v_head, part * 8, c.v_dim, v_word, v_scale);
}

int kv4_load_launch(const KvCache& cache, const int32_t* table, const int32_t* cu, const int32_t* starts, void* k, int64_t k_row,
                    int64_t k_head, void* v, int64_t v_row, int64_t v_head, int requests, int columns, int rows, hipStream_t stream) {
    const LoadArgs a = {cache, table, cu, starts, reinterpret_cast<half_t*>(k), reinterpret_cast<half_t*>(v), k_row, k_head, v_row, v_head,
                        requests, columns, rows};
    hipLaunchKernelGGL(kv4_load_kernel, dim3(((unsigned)rows + 15u) / 16u, (unsigned)cache.heads), dim3(256), 0, stream, a);
    return hipGetLastError() == hipSuccess ? UNIQL_OK : UNIQL_E_LAUNCH;
}

}  // namespace uniql
