// paged_ops.cu — the kernel value objects of the paged serving step
// (validation + routing) and their half of the C ABI. The arithmetic lives
// in paged.cu, paged_attention*.cu and sample.cu.
#include <memory>

#include "common.cuh"
#include "launch.hpp"
#include "popcorn.hpp"

namespace popcorn {
void set_last_error(const std::string& m);
int make_kernel(std::unique_ptr<Kernel> k, pc_kernel** out);

namespace {

bool is_float(int dt) { return dt == PC_F32 || dt == PC_F16 || dt == PC_BF16; }
const char* tag(int dt) { return dt == PC_F32 ? "" : dt == PC_F16 ? "_f16" : "_bf16"; }

void want(bool ok, int code, const std::string& message) {
    if (!ok) fail(code, message);
}

// An int32 tensor of exactly n elements (any rank).
const Tensor& ints(const Tensor& t, int64_t n, const char* what) {
    want(t.dtype() == PC_I32, PC_ERR_UNSUPPORTED_DATA_TYPE_COMBINATION,
         std::string(what) + " must be i32; got " + dtype_name(t.dtype()) + ".");
    want(t.element_count() == n, PC_ERR_TENSOR_SHAPE_MISMATCH,
         std::string(what) + " must hold " + std::to_string(n) + " elements; got " + t.shape_string() + ".");
    return t;
}

const Tensor& floats(const Tensor& t, int64_t n, const char* what) {
    want(t.dtype() == PC_F32, PC_ERR_UNSUPPORTED_DATA_TYPE_COMBINATION,
         std::string(what) + " must be f32; got " + dtype_name(t.dtype()) + ".");
    want(t.element_count() == n, PC_ERR_TENSOR_SHAPE_MISMATCH,
         std::string(what) + " must hold " + std::to_string(n) + " elements; got " + t.shape_string() + ".");
    return t;
}

template <class P>
P* ptr(const Tensor& t) { return static_cast<P*>(t.data()); }

// The memory of two tensors overlaps.
bool overlap(const Tensor& a, const Tensor& b) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.data()), y = reinterpret_cast<uintptr_t>(b.data());
    const uintptr_t nx = uintptr_t(a.element_count()) * dtype_stride(a.dtype()),
                    ny = uintptr_t(b.element_count()) * dtype_stride(b.dtype());
    return nx && ny && x < y + ny && y < x + nx;
}

// Every tensor at an address of its type's alignment; every output apart
// from every other tensor, except the pairs in `same` (which may be one
// buffer, whole).
void apart(const std::vector<Binding>& bindings, const char* what, const std::vector<std::pair<size_t, size_t>>& same = {}) {
    for (const Binding& b : bindings) {
        const uintptr_t at = reinterpret_cast<uintptr_t>(b.tensor.data());
        want(b.tensor.element_count() == 0 || (at && at % uintptr_t(dtype_stride(b.tensor.dtype())) == 0),
             PC_ERR_TENSOR_SHAPE_MISMATCH, std::string(what) + " has a tensor without memory, or not aligned to its type.");
    }
    for (size_t i = 0; i < bindings.size(); ++i)
        for (size_t j = 0; j < bindings.size(); ++j) {
            if (i == j || !(bindings[i].access & PC_ACCESS_WRITE) || !overlap(bindings[i].tensor, bindings[j].tensor)) continue;
            bool ok = false;
            for (const auto& s : same)
                ok = ok || (((s.first == i && s.second == j) || (s.first == j && s.second == i)) &&
                            bindings[i].tensor.data() == bindings[j].tensor.data());
            want(ok, PC_ERR_TENSOR_SHAPE_MISMATCH, std::string(what) + " output overlaps another of its tensors.");
        }
}

constexpr int64_t kIntMax = 0x7fffffff;

// ---------------------------------------------------------------------------
// PagedBatchBuild
// ---------------------------------------------------------------------------
class PagedBatchKernel : public Kernel {
public:
    PagedBatchKernel(const Tensor& cached, const Tensor& added, const Tensor& free_pages, const Tensor& free_head,
                     const Tensor& table, int64_t ps, const Tensor& seq_lens, const Tensor& query_start,
                     const Tensor& positions, const Tensor& slots, const Tensor& last_rows,
                     const Tensor& free_head_out, const Tensor& admitted) {
        want(table.rank() == 2, PC_ERR_TENSOR_INVALID_RANK, "PagedBatchBuild block_table must be [requests, pages].");
        const int64_t R = table[0], W = table[1];
        want(R <= launch::kMaxRequests, PC_ERR_TENSOR_SHAPE_MISMATCH,
             "PagedBatchBuild takes at most " + std::to_string(launch::kMaxRequests) + " requests; got " + std::to_string(R) + ".");
        want(ps >= 1 && ps <= kIntMax, PC_ERR_TENSOR_SHAPE_MISMATCH, "page size must be >= 1; got " + std::to_string(ps) + ".");
        ints(table, R * W, "block_table");
        ints(cached, R, "cached");
        ints(added, R, "added");
        ints(free_pages, free_pages.element_count(), "free_pages");
        ints(free_head, 1, "free_head");
        ints(seq_lens, R, "seq_lens");
        ints(query_start, R + 1, "query_start");
        const int64_t T = positions.element_count();
        ints(positions, T, "positions");
        ints(slots, T, "slots");
        ints(last_rows, R, "last_rows");
        ints(free_head_out, 1, "free_head_out");
        ints(admitted, 1, "admitted");
        want(T <= kIntMax && free_pages.element_count() <= kIntMax && W <= kIntMax, PC_ERR_TENSOR_SHAPE_MISMATCH,
             "PagedBatchBuild tensors are longer than int32 indices.");
        b_ = {{cached, PC_ACCESS_READ}, {added, PC_ACCESS_READ}, {free_pages, PC_ACCESS_READ}, {free_head, PC_ACCESS_READ},
              {table, PC_ACCESS_READ_WRITE}, {seq_lens, PC_ACCESS_WRITE}, {query_start, PC_ACCESS_WRITE},
              {positions, PC_ACCESS_WRITE}, {slots, PC_ACCESS_WRITE}, {last_rows, PC_ACCESS_WRITE},
              {free_head_out, PC_ACCESS_WRITE}, {admitted, PC_ACCESS_WRITE}};
        apart(b_, "PagedBatchBuild", {{0, 5}, {3, 10}});  // seq_lens may be cached, free_head_out free_head
        p_ = launch::PagedBatch{ptr<int32_t>(cached), ptr<int32_t>(added), ptr<int32_t>(free_pages), ptr<int32_t>(free_head),
                                ptr<int32_t>(table), ptr<int32_t>(seq_lens), ptr<int32_t>(query_start),
                                ptr<int32_t>(positions), ptr<int32_t>(slots), ptr<int32_t>(last_rows),
                                ptr<int32_t>(free_head_out), ptr<int32_t>(admitted), int(R), W,
                                free_pages.element_count(), T, ps, 1};
        function_names_ = "paged_batch_build";
    }
    const char* name() const override { return "PagedBatchBuild"; }
    std::vector<Binding> tensors() const override { return b_; }
    void encode(KernelCommandEncoder& enc) const override {
        launch::PagedBatch p = p_;
        enc.dispatch(function_names_, b_, [p](cudaStream_t s) { return launch::paged_batch_build(p, s); });
    }

private:
    std::vector<Binding> b_;
    launch::PagedBatch p_{};
};

// ---------------------------------------------------------------------------
// PagedQKVScatter
// ---------------------------------------------------------------------------
class PagedScatterKernel : public Kernel {
public:
    PagedScatterKernel(const Tensor& qkv, const Tensor& slots, const Tensor& q, const Tensor& k, const Tensor& v,
                       const Tensor* cos, const Tensor* sin, bool qk_norm, const Tensor* q_norm, const Tensor* k_norm,
                       bool norm_v, float eps, bool add_one) {
        const int dt = qkv.dtype();
        want(is_float(dt) && q.dtype() == dt && k.dtype() == dt && v.dtype() == dt, PC_ERR_UNSUPPORTED_DATA_TYPE_COMBINATION,
             "PagedQKVScatter needs one float data type for qkv, q and the pages; got " + dtype_name(dt) + ", " +
                 dtype_name(q.dtype()) + ", " + dtype_name(k.dtype()) + ", " + dtype_name(v.dtype()) + ".");
        want(qkv.rank() == 2 && q.rank() == 3 && k.rank() == 4 && v.rank() == 4, PC_ERR_TENSOR_INVALID_RANK,
             "PagedQKVScatter wants qkv [T,(Nq+2Nkv)*Hd], q [T,Nq,Hd], pages [P,Nkv,ps,Hd].");
        const int64_t T = q[0], Nq = q[1], Hd = q[2], P = k[0], Nkv = k[1], ps = k[2];
        want(k.same_shape(v) && k[3] == Hd && Hd >= 1 && Nq >= 1 && Nkv >= 1 && ps >= 1 && qkv[0] == T &&
                 qkv[1] == (Nq + 2 * Nkv) * Hd,
             PC_ERR_TENSOR_SHAPE_MISMATCH, "PagedQKVScatter shapes disagree: qkv " + qkv.shape_string() + ", q " +
                                               q.shape_string() + ", pages " + k.shape_string() + ", " + v.shape_string() + ".");
        want(Nq + 2 * Nkv <= 65535 && Hd <= 65536 && T <= kIntMax && P * ps <= kIntMax, PC_ERR_TENSOR_SHAPE_MISMATCH,
             "PagedQKVScatter takes at most 65535 heads, 65536 elements a head and 2^31 - 1 slots.");
        ints(slots, T, "slots");
        want((cos == nullptr) == (sin == nullptr), PC_ERR_TENSOR_SHAPE_MISMATCH, "RoPE needs both cos and sin.");
        if (cos) {
            want(Hd % 2 == 0, PC_ERR_TENSOR_SHAPE_MISMATCH, "RoPE needs an even head dim; got " + std::to_string(Hd) + ".");
            floats(*cos, T * (Hd / 2), "cos");
            floats(*sin, T * (Hd / 2), "sin");
        }
        if (q_norm || k_norm)
            want(qk_norm, PC_ERR_TENSOR_SHAPE_MISMATCH, "q_norm / k_norm weights need qk_norm.");
        if (q_norm) floats(*q_norm, Hd, "q_norm");
        if (k_norm) floats(*k_norm, Hd, "k_norm");
        b_ = {{qkv, PC_ACCESS_READ}, {slots, PC_ACCESS_READ}, {q, PC_ACCESS_WRITE}, {k, PC_ACCESS_WRITE}, {v, PC_ACCESS_WRITE}};
        for (const Tensor* t : {cos, sin, q_norm, k_norm})
            if (t) b_.push_back({*t, PC_ACCESS_READ});
        apart(b_, "PagedQKVScatter");
        p_ = launch::PagedScatter{qkv.data(), ptr<int32_t>(slots), q.data(), k.data(), v.data(),
                                  cos ? ptr<float>(*cos) : nullptr, sin ? ptr<float>(*sin) : nullptr,
                                  q_norm ? ptr<float>(*q_norm) : nullptr, k_norm ? ptr<float>(*k_norm) : nullptr, dt, T, P,
                                  ps, Hd, int(Nq), int(Nkv), qk_norm ? 1 : 0, norm_v ? 1 : 0, add_one ? 1 : 0, eps};
        function_names_ = std::string("paged_qkv_scatter") + tag(dt);
    }
    const char* name() const override { return "PagedQKVScatter"; }
    std::vector<Binding> tensors() const override { return b_; }
    void encode(KernelCommandEncoder& enc) const override {
        launch::PagedScatter p = p_;
        enc.dispatch(function_names_, b_, [p](cudaStream_t s) { return launch::paged_qkv_scatter(p, s); });
    }

private:
    std::vector<Binding> b_;
    launch::PagedScatter p_{};
};

// ---------------------------------------------------------------------------
// PagedAttention
// ---------------------------------------------------------------------------
class PagedAttentionKernel : public Kernel {
public:
    PagedAttentionKernel(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& seq_lens,
                         const Tensor& query_start, const Tensor& out, float scale, pc_attention_mask mask, int32_t sinks) {
        const int dt = q.dtype();
        want(is_float(dt) && k.dtype() == dt && v.dtype() == dt && out.dtype() == dt, PC_ERR_UNSUPPORTED_DATA_TYPE_COMBINATION,
             "PagedAttention needs one float data type for q, the pages and the output; got " + dtype_name(dt) + ", " +
                 dtype_name(k.dtype()) + ", " + dtype_name(v.dtype()) + ", " + dtype_name(out.dtype()) + ".");
        want(q.rank() == 3 && k.rank() == 4 && v.rank() == 4 && table.rank() == 2, PC_ERR_TENSOR_INVALID_RANK,
             "PagedAttention wants q [T,Nq,Hd], pages [P,Nkv,ps,Hd], block_table [R,W].");
        const int64_t T = q[0], Nq = q[1], Hd = q[2], P = k[0], Nkv = k[1], ps = k[2], R = table[0], W = table[1];
        want(Nkv > 0 && Nq > 0 && Nq % Nkv == 0, PC_ERR_TENSOR_SHAPE_MISMATCH,
             "PagedAttention query heads must be divisible by KV heads; got " + std::to_string(Nq) + " and " +
                 std::to_string(Nkv) + ".");
        want(Hd >= 1 && Hd <= 512, PC_ERR_TENSOR_SHAPE_MISMATCH,
             "PagedAttention head dim must be 1..512; got " + std::to_string(Hd) + ".");
        want(k.same_shape(v) && k[3] == Hd && ps >= 1 && out.same_shape(q), PC_ERR_TENSOR_SHAPE_MISMATCH,
             "PagedAttention shapes disagree: q " + q.shape_string() + ", pages " + k.shape_string() + ", " +
                 v.shape_string() + ", output " + out.shape_string() + ".");
        want(R <= launch::kMaxRequests, PC_ERR_TENSOR_SHAPE_MISMATCH,
             "PagedAttention takes at most " + std::to_string(launch::kMaxRequests) + " requests; got " + std::to_string(R) + ".");
        want(T * Nq <= kIntMax && W <= kIntMax && ps <= kIntMax && W * ps <= (int64_t(1) << 30) && P * ps <= kIntMax,
             PC_ERR_TENSOR_SHAPE_MISMATCH, "PagedAttention takes at most 2^31 - 1 query rows and slots and 2^30 keys a request.");
        ints(table, R * W, "block_table");
        ints(seq_lens, R, "seq_lens");
        ints(query_start, R + 1, "query_start");
        want(mask.kind >= 0 && mask.kind <= 2, PC_ERR_TENSOR_SHAPE_MISMATCH,
             "unknown attention mask kind " + std::to_string(mask.kind) + ".");
        want(mask.kind != PC_MASK_CAUSAL_SLIDING_WINDOW || mask.window >= 1, PC_ERR_TENSOR_SHAPE_MISMATCH,
             "sliding-window length must be >= 1.");
        want(sinks >= 0 && (sinks == 0 || mask.kind == PC_MASK_CAUSAL_SLIDING_WINDOW), PC_ERR_TENSOR_SHAPE_MISMATCH,
             "sinks (first tokens that stay visible) need the sliding-window mask, and a count >= 0.");
        b_ = {{q, PC_ACCESS_READ}, {k, PC_ACCESS_READ}, {v, PC_ACCESS_READ}, {table, PC_ACCESS_READ},
              {seq_lens, PC_ACCESS_READ}, {query_start, PC_ACCESS_READ}, {out, PC_ACCESS_WRITE}};
        apart(b_, "PagedAttention");
        p_ = launch::PagedAttention{q.data(), k.data(), v.data(), ptr<int32_t>(table), ptr<int32_t>(seq_lens),
                                    ptr<int32_t>(query_start), out.data(), dt, T, P, ps, Hd, W, int(R), int(Nq), int(Nkv),
                                    scale, mask.kind, mask.window, sinks};
        tc_ = launch::paged_attention_tc_supports(p_);
        function_names_ = std::string("paged_attention") + (tc_ ? "_tc" : "") + tag(dt);
        if (tc_) function_names_ += std::string(";paged_attention_join") + tag(dt);
    }
    const char* name() const override { return "PagedAttention"; }
    std::vector<Binding> tensors() const override { return b_; }
    void encode(KernelCommandEncoder& enc) const override {
        launch::PagedAttention p = p_;
        if (p.T == 0 || p.R == 0) return;
        if (!tc_) {
            enc.dispatch(function_names_, b_, [p](cudaStream_t s) { return launch::paged_attention_any(p, s); });
            return;
        }
        const int ctas = enc.sm_count();
        const int64_t words = int64_t((launch::paged_attention_scratch_bytes(p, ctas) + 3) / 4);
        enc.with_temporaries({{{words}, PC_F32}}, [&](const std::vector<Tensor>& t) {
            want(launch::aligned16(t[0].data()), PC_ERR_TENSOR_ALLOCATION_FAILED,
                 "PagedAttention needs scratch memory that is aligned to 16 bytes.");
            const launch::PagedScratch sc{t[0].data(), ctas};
            std::vector<Binding> first = b_;
            first.push_back({t[0], PC_ACCESS_WRITE});
            enc.dispatch(std::string("paged_attention_tc") + tag(p.dtype), first,
                         [p, sc](cudaStream_t s) { return launch::paged_attention_tc(p, sc, s); });
            enc.dispatch(std::string("paged_attention_join") + tag(p.dtype), {{t[0], PC_ACCESS_READ}, {b_.back().tensor, PC_ACCESS_WRITE}},
                         [p, sc](cudaStream_t s) { return launch::paged_attention_join(p, sc, s); });
        });
    }

private:
    std::vector<Binding> b_;
    launch::PagedAttention p_{};
    bool tc_ = false;
};

// ---------------------------------------------------------------------------
// Sample
// ---------------------------------------------------------------------------
class SampleKernel : public Kernel {
public:
    SampleKernel(const Tensor& logits, const Tensor& uniform, const Tensor& tokens, const Tensor* temperature,
                 const Tensor* top_k, const Tensor* top_p, const Tensor* min_p) {
        want(logits.rank() >= 1, PC_ERR_TENSOR_INVALID_RANK, "Sample logits must have a vocabulary axis.");
        want(is_float(logits.dtype()), PC_ERR_UNSUPPORTED_DATA_TYPE_COMBINATION,
             "Sample logits must be f32, f16 or bf16; got " + dtype_name(logits.dtype()) + ".");
        const int64_t V = logits[logits.rank() - 1];
        want(V >= 1 && V <= (int64_t(1) << 21), PC_ERR_TENSOR_SHAPE_MISMATCH,  // (42-bit weights: 63-bit sums)
             "Sample vocabulary must be 1..2^21; got " + std::to_string(V) + ".");
        const int64_t rows = logits.element_count() / V;
        want(rows <= (int64_t(1) << 27), PC_ERR_TENSOR_SHAPE_MISMATCH, "Sample takes at most 2^27 rows.");
        ints(tokens, rows, "tokens");
        floats(uniform, rows, "uniform");
        if (temperature) floats(*temperature, rows, "temperature");
        if (top_k) ints(*top_k, rows, "top_k");
        if (top_p) floats(*top_p, rows, "top_p");
        if (min_p) floats(*min_p, rows, "min_p");
        b_ = {{logits, PC_ACCESS_READ}, {uniform, PC_ACCESS_READ}, {tokens, PC_ACCESS_WRITE}};
        for (const Tensor* t : {temperature, top_k, top_p, min_p})
            if (t) b_.push_back({*t, PC_ACCESS_READ});
        apart(b_, "Sample");
        p_ = launch::Sample{logits.data(), logits.dtype(), ptr<float>(uniform), temperature ? ptr<float>(*temperature) : nullptr,
                            top_k ? ptr<int32_t>(*top_k) : nullptr, top_p ? ptr<float>(*top_p) : nullptr,
                            min_p ? ptr<float>(*min_p) : nullptr, ptr<int32_t>(tokens), rows, V};
        function_names_ = std::string("sample") + tag(logits.dtype());
    }
    const char* name() const override { return "Sample"; }
    std::vector<Binding> tensors() const override { return b_; }
    void encode(KernelCommandEncoder& enc) const override {
        launch::Sample p = p_;
        if (p.rows == 0) return;
        enc.dispatch(function_names_, b_, [p](cudaStream_t s) { return launch::sample(p, s); });
    }

private:
    std::vector<Binding> b_;
    launch::Sample p_{};
};

// A tensor argument that may be NULL.
struct Optional {
    Tensor t;
    bool given = false;
    Optional(const pc_tensor* p, const char* what) {
        if (p) {
            t = tensor_arg(p, what);
            given = true;
        }
    }
    const Tensor* get() const { return given ? &t : nullptr; }
};

template <class F>
int guarded(pc_kernel** kernel, F make) {
    try {
        if (!kernel) fail(PC_ERR_TENSOR_SHAPE_MISMATCH, "kernel result pointer is null.");
        *kernel = nullptr;
        return make_kernel(make(), kernel);
    } catch (const PopcornError& e) {
        set_last_error(e.message);
        return e.code;
    } catch (const std::exception& e) {
        set_last_error(e.what());
        return PC_ERR_GPU_INTERNAL;
    }
}

}  // namespace
}  // namespace popcorn

using namespace popcorn;

extern "C" {

int pc_kernel_paged_batch_build(const pc_tensor* cached, const pc_tensor* added, const pc_tensor* free_pages,
                                const pc_tensor* free_head, const pc_tensor* block_table, int64_t page_size,
                                const pc_tensor* seq_lens, const pc_tensor* query_start, const pc_tensor* positions,
                                const pc_tensor* slots, const pc_tensor* last_rows, const pc_tensor* free_head_out,
                                const pc_tensor* admitted, pc_kernel** kernel) {
    return guarded(kernel, [&] {
        return std::make_unique<PagedBatchKernel>(
            tensor_arg(cached, "cached"), tensor_arg(added, "added"), tensor_arg(free_pages, "free_pages"),
            tensor_arg(free_head, "free_head"), tensor_arg(block_table, "block_table"), page_size,
            tensor_arg(seq_lens, "seq_lens"), tensor_arg(query_start, "query_start"), tensor_arg(positions, "positions"),
            tensor_arg(slots, "slots"), tensor_arg(last_rows, "last_rows"), tensor_arg(free_head_out, "free_head_out"),
            tensor_arg(admitted, "admitted"));
    });
}

int pc_kernel_paged_qkv_scatter(const pc_tensor* qkv, const pc_tensor* slots, const pc_tensor* q_out,
                                const pc_tensor* k_pages, const pc_tensor* v_pages, const pc_tensor* cos_t,
                                const pc_tensor* sin_t, int32_t qk_norm, const pc_tensor* q_norm, const pc_tensor* k_norm,
                                int32_t norm_v, float eps, int32_t add_one_to_weight, pc_kernel** kernel) {
    return guarded(kernel, [&] {
        const Optional c(cos_t, "cos"), s(sin_t, "sin"), qn(q_norm, "q_norm"), kn(k_norm, "k_norm");
        return std::make_unique<PagedScatterKernel>(tensor_arg(qkv, "qkv"), tensor_arg(slots, "slots"),
                                                    tensor_arg(q_out, "q_out"), tensor_arg(k_pages, "k_pages"),
                                                    tensor_arg(v_pages, "v_pages"), c.get(), s.get(), qk_norm != 0, qn.get(),
                                                    kn.get(), norm_v != 0, eps, add_one_to_weight != 0);
    });
}

int pc_kernel_paged_attention(const pc_tensor* q, const pc_tensor* k_pages, const pc_tensor* v_pages,
                              const pc_tensor* block_table, const pc_tensor* seq_lens, const pc_tensor* query_start,
                              const pc_tensor* out, float scale, pc_attention_mask mask, int32_t sinks,
                              pc_kernel** kernel) {
    return guarded(kernel, [&] {
        return std::make_unique<PagedAttentionKernel>(tensor_arg(q, "q"), tensor_arg(k_pages, "k_pages"),
                                                      tensor_arg(v_pages, "v_pages"), tensor_arg(block_table, "block_table"),
                                                      tensor_arg(seq_lens, "seq_lens"),
                                                      tensor_arg(query_start, "query_start"), tensor_arg(out, "out"), scale,
                                                      mask, sinks);
    });
}

int pc_kernel_sample(const pc_tensor* logits, const pc_tensor* uniform, const pc_tensor* tokens,
                     const pc_tensor* temperature, const pc_tensor* top_k, const pc_tensor* top_p, const pc_tensor* min_p,
                     pc_kernel** kernel) {
    return guarded(kernel, [&] {
        const Optional t(temperature, "temperature"), k(top_k, "top_k"), p(top_p, "top_p"), m(min_p, "min_p");
        return std::make_unique<SampleKernel>(tensor_arg(logits, "logits"), tensor_arg(uniform, "uniform"),
                                              tensor_arg(tokens, "tokens"), t.get(), k.get(), p.get(), m.get());
    });
}

}  // extern "C"
