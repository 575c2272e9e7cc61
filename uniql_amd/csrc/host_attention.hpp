// The host side of the 4-bit key / value cache and of attention, part of host.cpp (inside its anonymous namespace): argument
// checks, the outputs' allocation and the launch in one native step, as for the calls there.

decltype(&uniql_kv_assign_pages) p_assign = nullptr;
decltype(&uniql_kv4_store) p_store = nullptr;
decltype(&uniql_kv4_load) p_load = nullptr;
decltype(&uniql_kv4_attention_workspace) p_attention_workspace = nullptr;
decltype(&uniql_kv4_attention) p_attention = nullptr;
decltype(&uniql_prompt_attention) p_prompt = nullptr;
decltype(&uniql_stream_capture_id) p_capture_id = nullptr;

void bind_attention(uintptr_t assign, uintptr_t store, uintptr_t load, uintptr_t workspace, uintptr_t attention, uintptr_t prompt,
                    uintptr_t capture_id) {
    p_assign = reinterpret_cast<decltype(p_assign)>(assign);
    p_store = reinterpret_cast<decltype(p_store)>(store);
    p_load = reinterpret_cast<decltype(p_load)>(load);
    p_attention_workspace = reinterpret_cast<decltype(p_attention_workspace)>(workspace);
    p_attention = reinterpret_cast<decltype(p_attention)>(attention);
    p_prompt = reinterpret_cast<decltype(p_prompt)>(prompt);
    p_capture_id = reinterpret_cast<decltype(p_capture_id)>(capture_id);
}

void require_device(const Tensor& t, const char* name, const Tensor& like) {
    require_gpu(t, name);
    if (t.device() != like.device()) fail(std::string(name) + " is on another device");
}
// a contiguous tensor of one axis (or `dims` axes) of `type` on like's device
void require_plain(const Tensor& t, const char* name, at::ScalarType type, int64_t dims, const Tensor& like) {
    require_device(t, name, like);
    if (t.scalar_type() != type || t.dim() != dims || !t.is_contiguous())
        fail(std::string(name) + " must be contiguous " + c10::toString(type) + " with " + std::to_string(dims) +
             (dims == 1 ? " axis" : " axes"));
}
// fp16 [rows, heads, width] with unit inner stride
void require_heads(const Tensor& t, const char* name) {
    if (t.scalar_type() != at::kHalf || t.dim() != 3 || (t.size(2) > 1 && t.stride(2) != 1))
        fail(std::string(name) + " must be float16 [rows, heads, width] with unit stride along the width");
    if (t.size(0) > 0x7fffffff || t.size(1) > 0x7fffffff || t.size(2) > 0x7fffffff) fail(std::string(name) + " is larger than a call can take");
    if (t.size(1) == 0 || t.size(2) == 0) fail(std::string(name) + " has no heads or no width");
}
// The caller's scale, or that of the heads' width.
float scale_of(const std::optional<double>& scale, const Tensor& q) { return (float)(scale ? *scale : 1.0 / std::sqrt((double)q.size(2))); }
// Where the elements of [rows, heads, width] with unit inner stride lie, in elements; heads and rows that follow each other count as
// one wider head.
struct Lattice {
    int64_t first, rows, row, heads, head, width;
    int64_t span() const { return (rows - 1) * row + (heads - 1) * head + width; }
};
Lattice lattice_of(const Tensor& t) {
    Lattice l = {(int64_t)(reinterpret_cast<uintptr_t>(t.data_ptr()) / t.element_size()), t.size(0), t.stride(0), t.size(1), t.stride(1), t.size(2)};
    if (l.heads == 1 || l.head == l.width) l.width *= l.heads, l.heads = 1, l.head = 0;
    if (l.heads == 1 && (l.rows == 1 || l.row == l.width)) l.width *= l.rows, l.rows = 1, l.row = 0;
    return l;
}
int64_t quotient_down(int64_t a, int64_t b) { return a / b - (a % b < 0); }  // b > 0
// Whether t step lies strictly between `low` and `high` for a whole t from `least` to `most`.
bool hits(int64_t step, int64_t least, int64_t most, int64_t low, int64_t high) {
    if (step == 0) return low < 0 && 0 < high;
    const int64_t t = std::max(least, quotient_down(low, step) + 1);
    return t <= most && t * step < high && t * step > low;
}
// Whether two tensors of heads have an element in common.  Mostly they lie apart; otherwise each pair of heads is looked at, for all
// rows at once where both have the same distance between rows.
bool share_memory(const Tensor& x, const Tensor& y) {
    if (x.numel() == 0 || y.numel() == 0) return false;
    Lattice a = lattice_of(x), b = lattice_of(y);
    if (a.first + a.span() <= b.first || b.first + b.span() <= a.first) return false;
    if (a.rows == 1) a.row = b.row;
    if (b.rows == 1) b.row = a.row;
    if (a.row != b.row && a.rows > b.rows) std::swap(a, b);
    for (int64_t i = 0; i < a.heads; ++i)
        for (int64_t j = 0; j < b.heads; ++j) {
            const int64_t apart = a.first + i * a.head - b.first - j * b.head;
            if (a.row == b.row) {
                if (hits(a.row, 1 - b.rows, a.rows - 1, -a.width - apart, b.width - apart)) return true;
                continue;
            }
            for (int64_t r = 0; r < a.rows; ++r) {
                const int64_t at = apart + r * a.row;   // less a row of b
                if (hits(b.row, 0, b.rows - 1, at - b.width, at + a.width)) return true;
            }
        }
    return false;
}
bool overlaps_itself(const Tensor& t) {
    if (t.numel() == 0) return false;
    const Lattice l = lattice_of(t);
    if (l.head >= l.width && l.row >= (l.heads - 1) * l.head + l.width) return false;
    if (l.rows > 1 && l.row < l.width) return true;
    for (int64_t i = 1; i < l.heads; ++i)
        if (hits(l.row, 1 - l.rows, l.rows - 1, -l.width - i * l.head, l.width - i * l.head)) return true;
    return false;
}
// The tensor that a call writes: the caller's, of exactly this shape, or a new one.
Tensor heads_output(const std::optional<Tensor>& out, const char* name, int64_t rows, int64_t heads, int64_t width, const Tensor& like) {
    if (!out) return new_output({rows, heads, width}, at::kHalf, like);
    require_device(*out, name, like);
    require_heads(*out, name);
    if (out->size(0) != rows || out->size(1) != heads || out->size(2) != width)
        fail(std::string(name) + " must be [" + std::to_string(rows) + ", " + std::to_string(heads) + ", " + std::to_string(width) + "]");
    if (overlaps_itself(*out)) fail(std::string(name) + " overlaps itself");
    return *out;
}
// Row r of a table of requests, entry p: the page of positions p page_size ..
void require_table(const Tensor& table, const Tensor& like) {
    require_plain(table, "table", at::kInt, 2, like);
    if (table.size(0) > 0x7fffffff || table.size(1) > 0x7fffffff) fail("table is larger than a call can take");
    if (table.size(1) == 0) fail("table must have at least one column");
}

// The pool of a cache: codes and scales of keys and values, [pages, heads, ..].
uniql_kv4_cache cache_of(const Tensor& k_codes, const Tensor& k_scales, const Tensor& v_codes, const Tensor& v_scales, int64_t k_dim,
                         int64_t v_dim) {
    require_gpu(k_codes, "k_codes");
    require_plain(k_codes, "k_codes", at::kInt, 4, k_codes);
    require_plain(k_scales, "k_scales", at::kHalf, 3, k_codes);
    require_plain(v_codes, "v_codes", at::kInt, 5, k_codes);
    require_plain(v_scales, "v_scales", at::kHalf, 3, k_codes);
    const int64_t pages = k_codes.size(0), heads = k_codes.size(1), page_size = k_codes.size(2);
    if (pages < 1 || pages > 0x7fffffff || heads < 1 || heads > 0x7fffffff) fail("the cache must have at least one page and one head");
    if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128 && page_size != 256)
        fail("pages must hold 16, 32, 64, 128 or 256 tokens");
    if (k_dim < 1 || k_dim > 128 || v_dim < 1 || v_dim > 128) fail("heads must be 1 to 128 wide");
    if (k_codes.size(3) != (k_dim + 31) / 32 * 4 || v_codes.size(3) != (v_dim + 31) / 32 * 4)
        fail("heads of " + std::to_string(k_dim) + " and " + std::to_string(v_dim) + " do not belong to this cache");
    const auto same = [&](const Tensor& t) { return t.size(0) == pages && t.size(1) == heads; };
    if (!same(k_scales) || k_scales.size(2) != page_size || !same(v_scales) || v_scales.size(2) != page_size || !same(v_codes) ||
        v_codes.size(2) != page_size / 4 || v_codes.size(4) != 4)
        fail("codes and scales of the cache do not belong together");
    return {k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(), v_scales.data_ptr(), (int)pages, (int)page_size, (int)heads,
            (int)k_dim, (int)v_dim};
}

// `count` numbers of `type` from byte `offset` of a buffer on, as a tensor that shares its memory.
Tensor part_of(const Tensor& buffer, int64_t offset, int64_t count, at::ScalarType type) {
    const auto meta = c10::scalarTypeToTypeMeta(type);
    auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(buffer.storage()), buffer.key_set(), meta);
    impl->set_storage_offset(offset / (int64_t)meta.itemsize());
    impl->set_sizes_contiguous({count});
    return Tensor(std::move(impl));
}

std::tuple<Tensor, Tensor, Tensor, Tensor> kv_assign_pages(const Tensor& new_tokens, const Tensor& lengths, const Tensor& table,
                                                           const Tensor& free_pages, const Tensor& free_count, int64_t page_size,
                                                           int64_t max_tokens, const std::optional<Tensor>& lengths_out,
                                                           const std::optional<Tensor>& count_out, uintptr_t stream) {
    const py::gil_scoped_release release;
    const at::NoGradGuard no_grad;
    require_gpu(new_tokens, "new_tokens");
    require_plain(new_tokens, "new_tokens", at::kInt, 1, new_tokens);
    require_plain(lengths, "lengths", at::kInt, 1, new_tokens);
    require_table(table, new_tokens);
    require_plain(free_pages, "free_pages", at::kInt, 1, new_tokens);
    require_plain(free_count, "free_count", at::kInt, 1, new_tokens);
    const int64_t rows = new_tokens.size(0), columns = table.size(1);
    if (lengths.size(0) != rows || table.size(0) != rows) fail("new_tokens, lengths and table must have one entry per request");
    if (free_count.size(0) != 1) fail("free_count must have one entry");
    if (free_pages.size(0) > 0x7fffffff) fail("free_pages is larger than a call can take");
    if (lengths_out) {
        require_plain(*lengths_out, "lengths_out", at::kInt, 1, new_tokens);
        if (lengths_out->size(0) != rows) fail("lengths_out must have one entry per request");
    }
    if (count_out) {
        require_plain(*count_out, "count_out", at::kInt, 1, new_tokens);
        if (count_out->size(0) != 1) fail("count_out must have one entry");
    }
    // what is written is read by other threads of the call at other times
    const Tensor &new_lengths = lengths_out ? *lengths_out : lengths, &new_count = count_out ? *count_out : free_count;
    const auto apart = [](const Tensor& x, const char* x_name, const Tensor& y, const char* y_name, bool may_be_one) {
        const char *a = static_cast<const char*>(x.data_ptr()), *b = static_cast<const char*>(y.data_ptr());
        if (x.numel() == 0 || y.numel() == 0 || a + x.nbytes() <= b || b + y.nbytes() <= a || (may_be_one && a == b)) return;
        fail(std::string(x_name) + " must not be " + y_name + " or share memory with it");
    };
    apart(new_lengths, "lengths_out", new_tokens, "new_tokens", false);
    apart(new_lengths, "lengths_out", lengths, "lengths", true);
    apart(new_lengths, "lengths_out", free_count, "free_count", false);
    apart(new_count, "count_out", new_tokens, "new_tokens", false);
    apart(new_count, "count_out", lengths, "lengths", false);
    apart(new_count, "count_out", new_lengths, "lengths_out", false);
    apart(new_count, "count_out", free_count, "free_count", true);
    for (const auto& [x, name] : {std::pair<const Tensor&, const char*>{table, "table"}, {free_pages, "free_pages"}}) {
        apart(x, name, new_tokens, "new_tokens", false);
        apart(x, name, lengths, "lengths", false);
        apart(x, name, new_lengths, "lengths_out", false);
        apart(x, name, free_count, "free_count", false);
        apart(x, name, new_count, "count_out", false);
    }
    apart(table, "table", free_pages, "free_pages", false);
    if (max_tokens < 0 || max_tokens > (1 << 24)) fail("max_tokens must be between 0 and 2^24");
    if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128 && page_size != 256)
        fail("pages must hold 16, 32, 64, 128 or 256 tokens");
    const c10::DeviceGuard guard(new_tokens.device());
    // one allocation for the four (0.7 us each)
    const Tensor buffer = new_output({8 * max_tokens + 4 * (max_tokens + 2 * rows + 1)}, at::kByte, new_tokens);
    Tensor slots = part_of(buffer, 0, max_tokens, at::kLong), positions = part_of(buffer, 8 * max_tokens, max_tokens, at::kInt);
    Tensor cu = part_of(buffer, 12 * max_tokens, rows + 1, at::kInt), refused = part_of(buffer, 12 * max_tokens + 4 * (rows + 1), rows, at::kInt);
    check(p_assign(new_tokens.data_ptr<int>(), lengths.data_ptr<int>(), table.data_ptr<int>(), free_pages.data_ptr<int>(),
                   free_count.data_ptr<int>(), new_lengths.data_ptr<int>(), new_count.data_ptr<int>(), slots.data_ptr<int64_t>(), positions.data_ptr<int>(),
                   cu.data_ptr<int>(), refused.data_ptr<int>(), (int)rows, (int)columns, (int)free_pages.size(0), (int)page_size,
                   (int)max_tokens, reinterpret_cast<void*>(stream)),
          "uniql_kv_assign_pages");
    return {slots, positions, cu, refused};
}

void kv4_store(const Tensor& k, const Tensor& v, const Tensor& slots, const Tensor& k_codes, const Tensor& k_scales, const Tensor& v_codes,
               const Tensor& v_scales, uintptr_t stream) {
    const py::gil_scoped_release release;
    const at::NoGradGuard no_grad;
    require_gpu(k, "k");
    require_device(v, "v", k);
    require_heads(k, "k");
    require_heads(v, "v");
    require_plain(slots, "slots", at::kLong, 1, k);
    require_device(k_codes, "k_codes", k);
    const uniql_kv4_cache cache = cache_of(k_codes, k_scales, v_codes, v_scales, k.size(2), v.size(2));
    const int64_t tokens = k.size(0);
    if (k.size(1) != cache.heads || v.size(1) != cache.heads) fail("k and v must have the cache's " + std::to_string(cache.heads) + " heads");
    if (v.size(0) != tokens || slots.size(0) != tokens) fail("k, v and slots must have one entry per token");
    const c10::DeviceGuard guard(k.device());
    check(p_store(k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), slots.data_ptr<int64_t>(), &cache,
                  (int)tokens, reinterpret_cast<void*>(stream)),
          "uniql_kv4_store");
}

std::pair<Tensor, Tensor> kv4_load(const Tensor& k_codes, const Tensor& k_scales, const Tensor& v_codes, const Tensor& v_scales,
                                   const Tensor& table, const Tensor& cu, int64_t rows, int64_t k_dim, int64_t v_dim,
                                   const std::optional<Tensor>& starts, const std::optional<Tensor>& k_out,
                                   const std::optional<Tensor>& v_out, uintptr_t stream) {
    const py::gil_scoped_release release;
    const at::NoGradGuard no_grad;
    const uniql_kv4_cache cache = cache_of(k_codes, k_scales, v_codes, v_scales, k_dim, v_dim);
    require_table(table, k_codes);
    require_plain(cu, "cu", at::kInt, 1, k_codes);
    const int64_t requests = table.size(0);
    if (cu.size(0) != requests + 1) fail("cu must have one entry more than table has rows");
    if (starts) {
        require_plain(*starts, "starts", at::kInt, 1, k_codes);
        if (starts->size(0) != requests) fail("starts must have one entry per request");
    }
    if (rows < 0 || rows > 0x7fffffff) fail("rows must be between 0 and 2^31 - 1");
    const c10::DeviceGuard guard(k_codes.device());
    Tensor k = heads_output(k_out, "k_out", rows, cache.heads, k_dim, k_codes), v = heads_output(v_out, "v_out", rows, cache.heads, v_dim, k_codes);
    if (k_out && v_out && share_memory(k, v)) fail("k_out and v_out must not share memory");
    check(p_load(&cache, table.data_ptr<int>(), cu.data_ptr<int>(), starts ? starts->data_ptr<int>() : nullptr, k.data_ptr(), k.stride(0),
                 k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), (int)requests, (int)table.size(1), (int)rows,
                 reinterpret_cast<void*>(stream)),
          "uniql_kv4_load");
    return {k, v};
}

Tensor kv4_attention(const Tensor& q, const Tensor& k_codes, const Tensor& k_scales, const Tensor& v_codes, const Tensor& v_scales,
                     const Tensor& table, const Tensor& lengths, int64_t v_dim, const std::optional<Tensor>& cu_q, std::optional<double> scale,
                     const std::optional<Tensor>& out_in, uintptr_t stream, const py::object& accumulator) {
    const py::gil_scoped_release release;
    const at::NoGradGuard no_grad;
    require_gpu(q, "q");
    require_heads(q, "q");
    require_device(k_codes, "k_codes", q);
    const uniql_kv4_cache cache = cache_of(k_codes, k_scales, v_codes, v_scales, q.size(2), v_dim);
    require_table(table, q);
    require_plain(lengths, "lengths", at::kInt, 1, q);
    const int64_t rows = q.size(0), heads = q.size(1), requests = table.size(0);
    if (lengths.size(0) != requests) fail("lengths must have one entry per request");
    if (heads % cache.heads) fail("q's heads must be a multiple of the cache's " + std::to_string(cache.heads));
    if (cu_q) {
        require_plain(*cu_q, "cu_q", at::kInt, 1, q);
        if (cu_q->size(0) != requests + 1) fail("cu_q must have one entry more than table has rows");
    } else if (rows != requests) {
        fail("without cu_q, q must have one row per request");
    }
    const c10::DeviceGuard guard(q.device());
    Tensor out = heads_output(out_in, "out", rows, heads, v_dim, q);
    if (out_in && share_memory(out, q)) fail("out must not be q or share memory with it: workgroups that share a row read it at different times");
    size_t need_accum = 0, need_temp = 0;
    check(p_attention_workspace(&cache, (int)rows, (int)requests, (int)table.size(1), (int)heads, &need_accum, &need_temp),
          "uniql_kv4_attention_workspace");
    Tensor accum, temp;
    if (need_accum) {
        // a capture has counts of its own: its graph may be replayed on any stream, beside eager calls and other graphs
        unsigned long long capture = 0;
        check(p_capture_id(reinterpret_cast<void*>(stream), &capture), "uniql_stream_capture_id");
        const py::gil_scoped_acquire lock;
        accum = accumulator(py::cast(q.device()), need_accum, stream, capture != 0).cast<Tensor>();
    }
    if (need_temp) temp = new_output({(int64_t)need_temp}, at::kByte, q);
    check(p_attention(q.data_ptr(), q.stride(0), q.stride(1), &cache, table.data_ptr<int>(), lengths.data_ptr<int>(),
                      cu_q ? cu_q->data_ptr<int>() : nullptr, out.data_ptr(), out.stride(0), out.stride(1),
                      need_accum ? accum.data_ptr() : nullptr, need_accum ? (size_t)accum.numel() * 8 : 0,
                      need_temp ? temp.data_ptr() : nullptr, need_temp, (int)rows, (int)requests, (int)table.size(1), (int)heads,
                      scale_of(scale, q), reinterpret_cast<void*>(stream)),
          "uniql_kv4_attention");
    return out;
}

Tensor prompt_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu_q, const std::optional<Tensor>& cu_k_in,
                        bool causal, std::optional<double> scale, const std::optional<Tensor>& out_in, uintptr_t stream) {
    const py::gil_scoped_release release;
    const at::NoGradGuard no_grad;
    require_gpu(q, "q");
    require_device(k, "k", q);
    require_device(v, "v", q);
    require_heads(q, "q");
    require_heads(k, "k");
    require_heads(v, "v");
    const int64_t rows = q.size(0), heads = q.size(1), k_rows = k.size(0), kv_heads = k.size(1);
    if (k.size(2) != q.size(2)) fail("q and k must have heads of one width");
    if (v.size(0) != k_rows || v.size(1) != kv_heads) fail("k and v must have the same rows and heads");
    if (heads % kv_heads) fail("q's heads must be a multiple of k's");
    if (q.size(2) > 128 || v.size(2) > 128) fail("heads must be 1 to 128 wide");
    require_plain(cu_q, "cu_q", at::kInt, 1, q);
    if (cu_q.size(0) < 1) fail("cu_q must have at least one entry");
    if (cu_q.size(0) > 0x7fffffff) fail("cu_q is larger than a call can take");
    const Tensor& cu_k = cu_k_in ? *cu_k_in : cu_q;
    if (cu_k_in) {
        require_plain(cu_k, "cu_k", at::kInt, 1, q);
        if (cu_k.size(0) != cu_q.size(0)) fail("cu_q and cu_k must have the same number of entries");
    }
    const c10::DeviceGuard guard(q.device());
    Tensor out = heads_output(out_in, "out", rows, heads, v.size(2), q);
    if (out_in && (share_memory(out, q) || share_memory(out, k) || share_memory(out, v)))
        fail("out must not be q, k or v or share memory with them");
    check(p_prompt(q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
                   cu_q.data_ptr<int>(), cu_k.data_ptr<int>(), out.data_ptr(), out.stride(0), out.stride(1), (int)rows, (int)k_rows,
                   (int)(cu_q.size(0) - 1), (int)heads, (int)kv_heads, (int)q.size(2), (int)v.size(2), causal, scale_of(scale, q),
                   reinterpret_cast<void*>(stream)),
          "uniql_prompt_attention");
    return out;
}

// The tensors of a module's cache, so that a call does not hand them over one by one (1 us for the four and 1.2 for a module to look
// its buffers up); every call checks them as it would the caller's.
struct KvPool {
    Tensor k_codes, k_scales, v_codes, v_scales;
    int64_t k_dim, v_dim;
};
void require_width(const Tensor& t, const char* name, int64_t width) {
    if (t.dim() == 3 && t.size(2) != width) fail(std::string(name) + " must be " + std::to_string(width) + " wide");
}
void pool_store(const KvPool& p, const Tensor& k, const Tensor& v, const Tensor& slots, uintptr_t stream) {
    require_width(k, "k", p.k_dim);
    require_width(v, "v", p.v_dim);
    kv4_store(k, v, slots, p.k_codes, p.k_scales, p.v_codes, p.v_scales, stream);
}
std::pair<Tensor, Tensor> pool_load(const KvPool& p, const Tensor& table, const Tensor& cu, int64_t rows, const std::optional<Tensor>& starts,
                                    const std::optional<Tensor>& k_out, const std::optional<Tensor>& v_out, uintptr_t stream) {
    return kv4_load(p.k_codes, p.k_scales, p.v_codes, p.v_scales, table, cu, rows, p.k_dim, p.v_dim, starts, k_out, v_out, stream);
}
Tensor pool_attend(const KvPool& p, const Tensor& q, const Tensor& table, const Tensor& lengths, const std::optional<Tensor>& cu_q,
                   std::optional<double> scale, const std::optional<Tensor>& out, uintptr_t stream, const py::object& accumulator) {
    require_width(q, "q", p.k_dim);
    return kv4_attention(q, p.k_codes, p.k_scales, p.v_codes, p.v_scales, table, lengths, p.v_dim, cu_q, scale, out, stream, accumulator);
}
