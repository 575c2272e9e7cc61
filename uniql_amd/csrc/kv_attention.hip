// Attention of each request's newest tokens over its pages of the 4-bit cache: o = sum_j p_j v_j / sum_j p_j,
// p_j = exp(scale q . k_j - m), over the positions j that the row sees.
#include "kv_attention.hpp"

namespace uniql {

// One wave per row and head; 64 positions at a time, a lane each.
__global__ __launch_bounds__(64) void kv4_attention_kernel(const KvAttentionArgs a) {
    const int lane = threadIdx.x, row = blockIdx.x, head = blockIdx.y, kv_head = head / a.group;
    __shared__ float q[128];
    int request = row, first = 0, last = 1;
    if (a.cu_q) {
        if (row < a.cu_q[0]) return;
        int low = 0, high = a.requests;
        while (low < high) {
            const int mid = (low + high) >> 1;
            if (a.cu_q[mid + 1] > row) high = mid;
            else low = mid + 1;
        }
        request = low;
        if (request >= a.requests) return;
        first = a.cu_q[request];
        last = a.cu_q[request + 1];
    } else {
        first = row;
        last = row + 1;
    }
    const KvCache& c = a.cache;
    const int64_t capacity = (int64_t)a.columns << c.page_shift;
    int64_t length = a.lengths[request];
    length = length > capacity ? capacity : length;
    const int64_t limit = length - (last - first) + (row - first) + 1;
    const half_t* q_row = a.q + row * a.q_row + head * a.q_head;
    for (int i = lane; i < 128; i += 64) q[i] = i < c.k_dim ? (float)q_row[i] : 0.f;
    __syncthreads();
    float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
    const float nan = __builtin_nanf("");
    for (int64_t base = 0; base < limit; base += 64) {
        const int64_t j = base + lane;
        float score = -INFINITY, vs = 0.f;
        int64_t slot = -1;
        if (j < limit) {
            const int64_t page = a.table[(int64_t)request * a.columns + (j >> c.page_shift)];
            if (page >= 0 && page < c.pages) {
                slot = (page << c.page_shift) + (j & ((1 << c.page_shift) - 1));
                float dot = 0.f;
                for (int w = 0; w < c.k_words; ++w) {
                    const uint32_t word = c.k_codes[c.k_word(slot, kv_head, w)];
#pragma unroll
                    for (int i = 0; i < 8; ++i) dot += q[8 * w + i] * ((float)((word >> kNibble(i)) & 15u) - 8.f);
                }
                score = dot * (float)c.k_scales[c.scale_at(slot, kv_head)] * a.scale;
                vs = (float)c.v_scales[c.scale_at(slot, kv_head)];
            } else {
                score = nan;
            }
        }
        float top = score;
        for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
        const float next = fmaxf(m, top);
        const float p = j < limit ? (next == -INFINITY ? (score != score ? nan : 0.f) : expf(score - next)) : 0.f;
        const float keep = m == -INFINITY ? 0.f : expf(m - next);
        m = next;
        l = l * keep + p;
        o0 *= keep;
        o1 *= keep;
        const float w = j < limit ? p * vs : 0.f;
        for (int t = 0; t < 64; ++t) {
            if (base + t >= limit) break;
            const float wt = __shfl(w, t, 64);
            const int64_t st = __shfl(slot, t, 64);
            if (st < 0) {
                o0 = o1 = nan;
                continue;
            }
            const int w0 = lane >> 3, w1 = 8 + (lane >> 3), n = kNibble(lane & 7);
            if (w0 < c.v_words) o0 += wt * ((float)((c.v_codes[c.v_word(st, kv_head, w0)] >> n) & 15u) - 8.f);
            if (w1 < c.v_words) o1 += wt * ((float)((c.v_codes[c.v_word(st, kv_head, w1)] >> n) & 15u) - 8.f);
        }
    }
    for (int d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d, 64);
    half_t* out = a.out + row * a.out_row + head * a.out_head;
    const bool empty = limit <= 0;
    if (lane < c.v_dim) out[lane] = empty ? (half_t)0.f : (half_t)(o0 / l);
    if (lane + 64 < c.v_dim) out[lane + 64] = empty ? (half_t)0.f : (half_t)(o1 / l);
}

void kv4_attention_needs(int rows, int requests, int q_heads, const KvCache& cache, size_t* accum_bytes, size_t* temp_bytes) {
    *accum_bytes = *temp_bytes = 0;
}

int kv4_attention_launch(const KvAttentionArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL(kv4_attention_kernel, dim3((unsigned)a.rows, (unsigned)(a.group * a.cache.heads)), dim3(64), 0, stream, a);
    return hipGetLastError() == hipSuccess ? UNIQL_OK : UNIQL_E_LAUNCH;
}

}  // namespace uniql
