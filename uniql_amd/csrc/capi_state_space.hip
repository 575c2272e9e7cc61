// extern "C" surface of what stands between the projections of a state-space layer: argument checks and dispatch.  Nothing here
// allocates, synchronises or throws.
#include "state_space.hpp"

namespace uniql {
int causal_conv_launch(const ConvArgs& a, int width, hipStream_t stream);
int state_space_step_launch(const ScanArgs& a, hipStream_t stream);
int state_space_scan_launch(const ScanArgs& a, hipStream_t stream);
size_t state_space_scan_needs(int rows, int count, int heads, int head_dim, int states);
int gated_group_norm_launch(const NormArgs& a, hipStream_t stream);
}  // namespace uniql

using namespace uniql;

static constexpr int kMaxRows = 1 << 27, kMaxSequences = 1 << 24, kMaxChannels = 1 << 24, kMaxScanHeads = 1 << 15;
static constexpr int kMaxHeadDim = 128, kMaxStates = 256;

static int sequences_of(const uniql_sequences* s, int rows, bool any_state, Sequences& out) {
    if (!s) return UNIQL_E_NULL;
    if (rows < 0 || rows > kMaxRows || s->count < 0 || s->count > kMaxSequences || s->pool < 0) return UNIQL_E_SHAPE;
    if (!s->cu && s->count != rows) return UNIQL_E_SHAPE;
    out.cu = s->cu;
    out.starts = s->starts;
    out.places = s->places;
    out.count = s->count;
    out.pool = any_state ? s->pool : 0x7fffffff;
    out.rows = rows;
    return UNIQL_OK;
}

extern "C" {

int uniql_causal_conv(const void* x, int64_t x_row, const void* weight, const void* bias, const void* state, void* state_out,
                      const uniql_sequences* sequences, void* out, int64_t out_row, int rows, int channels, int width, int activation,
                      void* stream) {
    ConvArgs a = {};
    if (const int code = sequences_of(sequences, rows, state || state_out, a.sequences)) return code;
    if (channels <= 0 || channels > kMaxChannels) return UNIQL_E_SHAPE;
    if (width < 2 || width > 4) return UNIQL_E_UNSUPPORTED;
    if (rows == 0 || a.sequences.count == 0) return UNIQL_OK;
    if (!x || !weight || !out) return UNIQL_E_NULL;
    a.x = reinterpret_cast<const half_t*>(x);
    a.weight = reinterpret_cast<const half_t*>(weight);
    a.bias = reinterpret_cast<const half_t*>(bias);
    a.state = reinterpret_cast<const half_t*>(state);
    a.state_out = reinterpret_cast<half_t*>(state_out);
    a.out = reinterpret_cast<half_t*>(out);
    a.x_row = x_row, a.out_row = out_row;
    a.channels = channels;
    a.activation = activation != 0;
    return causal_conv_launch(a, width, reinterpret_cast<hipStream_t>(stream));
}

static int scan_sizes(int rows, int count, int heads, int groups, int head_dim, int states) {
    if (rows < 0 || rows > kMaxRows || count < 0 || count > kMaxSequences) return UNIQL_E_SHAPE;
    if (heads <= 0 || heads > kMaxScanHeads || groups <= 0 || heads % groups != 0 || head_dim <= 0 || states <= 0) return UNIQL_E_SHAPE;
    if (head_dim > kMaxHeadDim || states > kMaxStates) return UNIQL_E_UNSUPPORTED;
    return UNIQL_OK;
}

int uniql_state_space_scan_workspace(int rows, int count, int heads, int groups, int head_dim, int states, size_t* temp_bytes) {
    if (!temp_bytes) return UNIQL_E_NULL;
    if (const int code = scan_sizes(rows, count, heads, groups, head_dim, states)) return code;
    *temp_bytes = rows == 0 || count == 0 ? 0 : state_space_scan_needs(rows, count, heads, head_dim, states);
    return UNIQL_OK;
}

int uniql_state_space_scan(const void* x, int64_t x_row, int64_t x_head, const void* dt, int64_t dt_row, const float* decay, const void* b,
                           int64_t b_row, int64_t b_group, const void* c, int64_t c_row, int64_t c_group, const float* skip,
                           const float* dt_bias, int softplus, float dt_min, float dt_max, const float* state, float* state_out,
                           const uniql_sequences* sequences, void* y, int64_t y_row, int64_t y_head, void* temp, size_t temp_bytes,
                           int rows, int heads, int groups, int head_dim, int states, void* stream) {
    ScanArgs a = {};
    if (const int code = sequences_of(sequences, rows, state || state_out, a.sequences)) return code;
    if (const int code = scan_sizes(rows, a.sequences.count, heads, groups, head_dim, states)) return code;
    if (!(dt_min >= 0.f && dt_min <= dt_max)) return UNIQL_E_UNSUPPORTED;
    if (rows == 0 || a.sequences.count == 0) return UNIQL_OK;
    if (!x || !dt || !decay || !b || !c || !y) return UNIQL_E_NULL;
    if ((reinterpret_cast<uintptr_t>(state) | reinterpret_cast<uintptr_t>(state_out)) & 15u) return UNIQL_E_ALIGN;
    a.x = reinterpret_cast<const half_t*>(x);
    a.dt = reinterpret_cast<const half_t*>(dt);
    a.b = reinterpret_cast<const half_t*>(b);
    a.c = reinterpret_cast<const half_t*>(c);
    a.a = decay, a.d = skip, a.dt_bias = dt_bias;
    a.state = state;
    a.state_out = state_out;
    a.y = reinterpret_cast<half_t*>(y);
    a.x_row = x_row, a.x_head = x_head, a.dt_row = dt_row, a.b_row = b_row, a.b_group = b_group, a.c_row = c_row, a.c_group = c_group;
    a.y_row = y_row, a.y_head = y_head;
    a.softplus = softplus != 0;
    a.dt_min = dt_min, a.dt_max = dt_max;
    a.heads = heads, a.share = heads / groups, a.head_dim = head_dim, a.states = states;
    if (!a.sequences.cu) return state_space_step_launch(a, reinterpret_cast<hipStream_t>(stream));
    const size_t need = state_space_scan_needs(rows, a.sequences.count, heads, head_dim, states);
    if (temp_bytes < need) return UNIQL_E_WORKSPACE;
    if (need && !temp) return UNIQL_E_NULL;
    if (reinterpret_cast<uintptr_t>(temp) & 15u) return UNIQL_E_ALIGN;
    a.temp = reinterpret_cast<float*>(temp);
    // Single tokens among prompts are steps, which take less than a chunk of 64 rows for each (128 heads: 256 tokens 735 -> 420 us, 48 tokens
    // 138 -> 78, 255 tokens and 2048 of a prompt 816 -> 495).  How many there are is not known here: where there are none that launch finds
    // nothing to do (24 prompts 250 to 256 us with and without).  Fewer than four are as fast beside the prompts.
    if (a.sequences.count >= 4 && (int64_t)a.sequences.count * heads < (1 << 20)) {
        ScanArgs step = a;
        step.sequences.only = kSingle;
        if (const int code = state_space_step_launch(step, reinterpret_cast<hipStream_t>(stream))) return code;
        a.sequences.only = kLonger;
    }
    return state_space_scan_launch(a, reinterpret_cast<hipStream_t>(stream));
}

int uniql_gated_group_norm(const void* x, int64_t x_row, const void* z, int64_t z_row, const void* weight, void* out, int64_t out_row,
                           int rows, int channels, int groups, float eps, void* stream) {
    if (rows < 0 || rows > kMaxRows || channels <= 0 || channels > kMaxChannels || groups <= 0 || channels % groups != 0)
        return UNIQL_E_SHAPE;
    if (!(eps >= 0.f)) return UNIQL_E_UNSUPPORTED;
    if (rows == 0) return UNIQL_OK;
    if (!x || !z || !weight || !out) return UNIQL_E_NULL;
    NormArgs a;
    a.x = reinterpret_cast<const half_t*>(x);
    a.z = reinterpret_cast<const half_t*>(z);
    a.weight = reinterpret_cast<const half_t*>(weight);
    a.out = reinterpret_cast<half_t*>(out);
    a.x_row = x_row, a.z_row = z_row, a.out_row = out_row;
    a.rows = rows, a.groups = groups, a.width = channels / groups;
    a.eps = eps;
    return gated_group_norm_launch(a, reinterpret_cast<hipStream_t>(stream));
}

}  // extern "C"
