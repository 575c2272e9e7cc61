// Causal attention over the prompts of several sequences that lie behind each other: o = sum_j p_j v_j / sum_j p_j,
// p_j = exp(scale q . k_j - m), row i of a sequence with t queries and n keys over the keys j <= i + n - t.
#include "prompt_attention.hpp"

namespace uniql {

__device__ __forceinline__ int clamp_to(int v, int low, int high) { return v < low ? low : (v > high ? high : v); }

// One wave per row and head; 64 keys at a time, a lane each.
__global__ __launch_bounds__(64) void prompt_attention_kernel(const PromptArgs a) {
    const int lane = threadIdx.x, row = blockIdx.x, head = blockIdx.y, kv_head = head / a.group;
    __shared__ float q[128];
    if (row < a.cu_q[0]) return;
    int low = 0, high = a.sequences;
    while (low < high) {
        const int mid = (low + high) >> 1;
        if (a.cu_q[mid + 1] > row) high = mid;
        else low = mid + 1;
    }
    if (low >= a.sequences) return;
    const int first = a.cu_q[low], last = a.cu_q[low + 1];
    const int k_first = clamp_to(a.cu_k[low], 0, a.k_rows), k_last = clamp_to(a.cu_k[low + 1], k_first, a.k_rows);
    const int length = k_last - k_first;
    const int64_t seen = a.causal ? (int64_t)length - (last - first) + (row - first) + 1 : length;
    const int limit = seen < 0 ? 0 : (seen > length ? length : (int)seen);
    const half_t* q_row = a.q + row * a.q_row + head * a.q_head;
    for (int i = lane; i < 128; i += 64) q[i] = i < a.k_dim ? (float)q_row[i] : 0.f;
    __syncthreads();
    float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
    for (int base = 0; base < limit; base += 64) {
        const int j = base + lane;
        float score = -INFINITY;
        if (j < limit) {
            const half_t* k = a.k + (int64_t)(k_first + j) * a.k_row + kv_head * a.k_head;
            float dot = 0.f;
            for (int i = 0; i < a.k_dim; ++i) dot += q[i] * (float)k[i];
            score = dot * a.scale;
        }
        float top = score;
        for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
        const float next = fmaxf(m, top);
        const float p = j < limit ? (next == -INFINITY ? (score != score ? score : 0.f) : expf(score - next)) : 0.f;
        const float keep = m == -INFINITY ? 0.f : expf(m - next);
        m = next;
        l = l * keep + p;
        o0 *= keep;
        o1 *= keep;
        for (int t = 0; t < 64 && base + t < limit; ++t) {
            const float pt = __shfl(p, t, 64);
            const half_t* v = a.v + (int64_t)(k_first + base + t) * a.v_row + kv_head * a.v_head;
            if (lane < a.v_dim) o0 += pt * (float)v[lane];
            if (lane + 64 < a.v_dim) o1 += pt * (float)v[lane + 64];
        }
    }
    for (int d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d, 64);
    half_t* out = a.out + row * a.out_row + head * a.out_head;
    if (lane < a.v_dim) out[lane] = limit == 0 ? (half_t)0.f : (half_t)(o0 / l);
    if (lane + 64 < a.v_dim) out[lane + 64] = limit == 0 ? (half_t)0.f : (half_t)(o1 / l);
}

int prompt_attention_launch(const PromptArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL(prompt_attention_kernel, dim3((unsigned)a.rows, (unsigned)a.heads), dim3(64), 0, stream, a);
    return hipGetLastError() == hipSuccess ? UNIQL_OK : UNIQL_E_LAUNCH;
}

}  // namespace uniql
