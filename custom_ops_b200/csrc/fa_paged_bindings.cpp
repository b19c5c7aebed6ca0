// Torch operator boundary of the paged key/value cache group (the reference has no such group):
//
//   recsys_ops::paged_extend, paged_extend_, paged_shrink_   block tables, slots, positions
//   recsys_ops::rotary                                       rotary positions in the attention's layout
//   recsys_ops::rotary_append, paged_append                  new tokens into the pages
//   recsys_ops::paged_attention, paged_attention_lse         one new token per request over the pages
//
// Same namespace, dispatch key and style of checks as the masked-attention group (fa_bindings.cpp): arguments
// are checked, outputs and scratch come from torch's caching allocator on the operands' device, and plain
// pointers go to the C ABI (include/fa_paged_sm100.h) on the current stream.  Nothing is copied or cast.

#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <limits>

#include "../../include/fa_paged_sm100.h"

namespace {

using torch::Tensor;

int32_t as_i32(int64_t v, const char* what) {
    TORCH_CHECK(v >= 0 && v <= std::numeric_limits<int32_t>::max(), what, " is out of range: ", v);
    return static_cast<int32_t>(v);
}

void check_rc(int rc, const char* op) { TORCH_CHECK(rc == FA_PAGED_OK, op, ": ", fa_paged_sm100_strerror(rc)); }

void* stream_of(const Tensor& t) {
    return static_cast<void*>(at::cuda::getCurrentCUDAStream(t.get_device()).stream());
}

// torch::empty without the dispatcher's way to it: these calls last a few microseconds.
Tensor empty(at::IntArrayRef sizes, at::ScalarType dtype, const Tensor& like) {
    return at::detail::empty_cuda(sizes, dtype, like.device(), c10::nullopt);
}

void check_cuda(const char* op, std::initializer_list<const Tensor*> tensors) {
    const Tensor& first = **tensors.begin();
    for (const Tensor* t : tensors) TORCH_CHECK(t->is_cuda(), op, " is only supported on CUDA");
    for (const Tensor* t : tensors)
        TORCH_CHECK(t->device() == first.device(), op, ": all tensors must be on the same device");
}

int32_t dtype_code(const Tensor& q, const char* op) {
    TORCH_CHECK(q.dtype() == torch::kHalf || q.dtype() == torch::kBFloat16, op, ": q, k, v must be float16 or bfloat16");
    return q.dtype() == torch::kBFloat16 ? FA_PAGED_BF16 : FA_PAGED_FP16;
}

// Stride of a dimension; that of a dimension of one element says nothing, nor do those of a tensor without any.
int64_t step(const Tensor& t, int64_t dim) { return t.size(dim) > 1 && t.numel() > 0 ? t.stride(dim) : 0; }

void check_rows(const Tensor& t, const char* op, const char* name) {
    if (t.numel() == 0) return;
    TORCH_CHECK(t.size(-1) <= 1 || t.stride(-1) == 1, op, ": the last dimension of ", name, " must be contiguous");
    TORCH_CHECK(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, op, ": ", name, " must be 16-byte aligned");
    for (int64_t i = 0; i + 1 < t.dim(); ++i)
        TORCH_CHECK(step(t, i) % 8 == 0, op, ": the strides of ", name, " must be multiples of 8 elements");
}

void check_head_dim(int64_t d, const char* op) {
    TORCH_CHECK(d == 64 || d == 128, op, ": Only head_dim=64 or head_dim=128 is supported");
}

void check_int(const Tensor& t, int64_t dim, bool allow_64, const char* op, const char* name) {
    TORCH_CHECK(t.dtype() == torch::kInt || (allow_64 && t.dtype() == torch::kLong), op, ": ", name, " must be int32",
                allow_64 ? " or int64" : "");
    TORCH_CHECK(t.dim() == dim, op, ": ", name, " must be ", dim, "D");
}

void check_list(const Tensor& t, int64_t n, bool allow_64, const char* op, const char* name) {
    check_int(t, 1, allow_64, op, name);
    TORCH_CHECK(t.size(0) == n, op, ": ", name, " must hold ", n, " values");
    TORCH_CHECK(t.is_contiguous(), op, ": ", name, " must be contiguous");
}

FaPagedCache cache_of(const Tensor& k, const Tensor& v, const char* op) {
    TORCH_CHECK(k.dim() == 4 && v.dim() == 4, op, ": k_cache and v_cache must be 4D (pages, Hk, page_size, d)");
    TORCH_CHECK(k.sizes() == v.sizes(), op, ": k_cache and v_cache must have one shape");
    TORCH_CHECK(k.dtype() == v.dtype(), op, ": k_cache and v_cache dtype must match");
    check_head_dim(k.size(3), op);
    TORCH_CHECK(k.size(1) > 0 && k.size(2) > 0, op, ": the cache must have heads and a page size");
    check_rows(k, op, "k_cache");
    check_rows(v, op, "v_cache");
    FaPagedCache c{};
    c.k = k.data_ptr();
    c.v = v.data_ptr();
    c.k_page_stride = step(k, 0), c.k_head_stride = step(k, 1), c.k_row_stride = step(k, 2);
    c.v_page_stride = step(v, 0), c.v_head_stride = step(v, 1), c.v_row_stride = step(v, 2);
    c.num_pages = as_i32(k.size(0), "the number of pages");
    c.heads_k = as_i32(k.size(1), "the number of key heads");
    c.page_size = as_i32(k.size(2), "page_size");
    c.head_dim = static_cast<int32_t>(k.size(3));
    return c;
}

FaRotarySpec rotary_of(const Tensor& positions, const Tensor& freqs, bool interleaved, double mscale, bool adjoint,
                       int64_t d, const char* op) {
    TORCH_CHECK(freqs.dtype() == torch::kDouble && freqs.dim() == 1 && freqs.is_contiguous(), op,
                ": freqs must be a contiguous 1D float64 tensor");
    TORCH_CHECK(freqs.size(0) >= 1 && 2 * freqs.size(0) <= d, op, ": freqs must hold 1 to head_dim / 2 values");
    TORCH_CHECK(std::isfinite(mscale), op, ": mscale must be finite");
    FaRotarySpec r{};
    r.freqs = freqs.data_ptr<double>();
    r.positions = positions.data_ptr();
    r.positions_64 = positions.dtype() == torch::kLong;
    r.rot_dim = static_cast<int32_t>(2 * freqs.size(0));
    r.interleaved = interleaved;
    r.adjoint = adjoint;
    r.mscale = static_cast<float>(mscale);
    return r;
}

// ------------------------------------------------------------------ tables
// Two contiguous tensors must not share memory.
void check_apart(const Tensor& a, const Tensor& b, const char* op) {
    const char *x = static_cast<const char*>(a.data_ptr()), *y = static_cast<const char*>(b.data_ptr());
    TORCH_CHECK(x + a.nbytes() <= y || y + b.nbytes() <= x, op, ": a tensor that is written shares a memory location with another");
}

// What a call updates in place, or reads while it does.  (The lengths to add or to keep are read before anything is
// written; they may be the lengths themselves.)
void check_in_place(const Tensor& seq_lens, const Tensor& free_pages, const Tensor& free_head, const char* op) {
    check_apart(seq_lens, free_pages, op);
    check_apart(seq_lens, free_head, op);
    check_apart(free_pages, free_head, op);
}

void check_table(const Tensor& block_table, const Tensor& seq_lens, const Tensor& other, const Tensor& free_pages,
                 const Tensor& free_head, int64_t page_size, const char* op) {
    check_cuda(op, {&block_table, &seq_lens, &other, &free_pages, &free_head});
    check_int(block_table, 2, false, op, "block_table");
    TORCH_CHECK(block_table.size(1) <= 1 || block_table.stride(1) == 1, op, ": the rows of block_table must be contiguous");
    const int64_t B = block_table.size(0);
    TORCH_CHECK(B <= FA_PAGED_MAX_REQUESTS, op, ": at most ", FA_PAGED_MAX_REQUESTS, " requests are supported");
    check_list(seq_lens, B, false, op, "seq_lens");
    check_list(other, B, false, op, "new_lens or keep_lens");
    check_list(free_pages, free_pages.numel(), false, op, "free_pages");
    check_list(free_head, 1, false, op, "free_head");
    if (block_table.is_contiguous())
        for (const Tensor* t : {&seq_lens, &other, &free_pages, &free_head}) check_apart(block_table, *t, op);
    TORCH_CHECK(page_size > 0, op, ": page_size must be positive");
    TORCH_CHECK(page_size <= std::numeric_limits<int32_t>::max() &&
                    block_table.size(1) <= std::numeric_limits<int32_t>::max() / page_size,
                op, ": a request's tokens must be countable in 32 bits (columns * page_size)");
}

struct Extended { Tensor slots, positions, cu; };

Extended extend(const Tensor& block_table, const Tensor& seq_lens, const Tensor& new_lens, const Tensor& free_pages,
                const Tensor& free_head, int64_t page_size, int64_t num_tokens, const Tensor& lens_out,
                const Tensor& head_out, const char* op) {
    at::assert_no_internal_overlap(block_table);
    const int64_t B = block_table.size(0);
    Extended r{empty({num_tokens}, torch::kLong, seq_lens), empty({num_tokens}, torch::kInt, seq_lens),
               empty({B + 1}, torch::kInt, seq_lens)};
    FaPagedExtendArgs a{};
    a.struct_size = sizeof(a);
    a.device = block_table.get_device();
    a.block_table = block_table.data_ptr<int32_t>();
    a.table_stride = step(block_table, 0);
    a.lens = seq_lens.data_ptr<int32_t>();
    a.new_lens = new_lens.data_ptr<int32_t>();
    a.free_pages = free_pages.data_ptr<int32_t>();
    a.free_head = free_head.data_ptr<int32_t>();
    a.lens_out = lens_out.data_ptr<int32_t>();
    a.head_out = head_out.data_ptr<int32_t>();
    a.slots = r.slots.data_ptr<int64_t>();
    a.positions = r.positions.data_ptr<int32_t>();
    a.cu = r.cu.data_ptr<int32_t>();
    a.batch = static_cast<int32_t>(B);
    a.table_width = as_i32(block_table.size(1), "the width of block_table");
    a.page_size = static_cast<int32_t>(page_size);
    a.num_free_pages = as_i32(free_pages.numel(), "the number of free pages");
    a.num_tokens = num_tokens;
    check_rc(fa_paged_extend_sm100(&a, stream_of(block_table)), op);
    return r;
}

void check_num_tokens(int64_t n, const char* op) {
    TORCH_CHECK(n >= 0 && n <= std::numeric_limits<int32_t>::max(), op, ": num_tokens is out of range: ", n);
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> paged_extend(const Tensor& block_table, const Tensor& seq_lens,
                                                                const Tensor& new_lens, const Tensor& free_pages,
                                                                const Tensor& free_head, int64_t page_size,
                                                                int64_t num_tokens) {
    const char* op = "paged_extend";
    check_table(block_table, seq_lens, new_lens, free_pages, free_head, page_size, op);
    check_num_tokens(num_tokens, op);
    const c10::cuda::CUDAGuard guard(block_table.device());
    auto lens = empty({seq_lens.size(0)}, torch::kInt, seq_lens), head = empty({1}, torch::kInt, seq_lens);
    auto r = extend(block_table, seq_lens, new_lens, free_pages, free_head, page_size, num_tokens, lens, head, op);
    return {lens, head, r.slots, r.positions, r.cu};
}

std::tuple<Tensor, Tensor, Tensor> paged_extend_(const Tensor& block_table, const Tensor& seq_lens, const Tensor& new_lens,
                                                 const Tensor& free_pages, const Tensor& free_head, int64_t page_size,
                                                 int64_t num_tokens) {
    const char* op = "paged_extend_";
    check_table(block_table, seq_lens, new_lens, free_pages, free_head, page_size, op);
    check_num_tokens(num_tokens, op);
    check_in_place(seq_lens, free_pages, free_head, op);
    const c10::cuda::CUDAGuard guard(block_table.device());
    auto r = extend(block_table, seq_lens, new_lens, free_pages, free_head, page_size, num_tokens, seq_lens, free_head, op);
    return {r.slots, r.positions, r.cu};
}

void paged_shrink_(const Tensor& block_table, const Tensor& seq_lens, const Tensor& keep_lens, const Tensor& free_pages,
                   const Tensor& free_head, int64_t page_size) {
    const char* op = "paged_shrink_";
    check_table(block_table, seq_lens, keep_lens, free_pages, free_head, page_size, op);
    at::assert_no_partial_overlap(seq_lens, keep_lens);
    check_in_place(seq_lens, free_pages, free_head, op);
    const c10::cuda::CUDAGuard guard(block_table.device());
    FaPagedShrinkArgs a{};
    a.struct_size = sizeof(a);
    a.device = block_table.get_device();
    a.block_table = block_table.data_ptr<int32_t>();
    a.table_stride = step(block_table, 0);
    a.lens = seq_lens.data_ptr<int32_t>();
    a.keep_lens = keep_lens.data_ptr<int32_t>();
    a.free_pages = free_pages.data_ptr<int32_t>();
    a.free_head = free_head.data_ptr<int32_t>();
    a.batch = static_cast<int32_t>(block_table.size(0));
    a.table_width = as_i32(block_table.size(1), "the width of block_table");
    a.page_size = static_cast<int32_t>(page_size);
    a.num_free_pages = as_i32(free_pages.numel(), "the number of free pages");
    check_rc(fa_paged_shrink_sm100(&a, stream_of(block_table)), op);
}

// ------------------------------------------------------------------ rotary positions, append
std::tuple<Tensor, Tensor> rotary(const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& freqs,
                                  bool interleaved, double mscale, bool adjoint) {
    const char* op = "rotary";
    check_cuda(op, {&q, &k, &positions, &freqs});
    FaRotaryArgs a{};
    a.dtype = dtype_code(q, op);
    TORCH_CHECK(k.dtype() == q.dtype(), op, ": k dtype must match q");
    TORCH_CHECK(q.dim() == 4 && k.dim() == 4, op, ": q must be 4D (B, H, S, d) and k 4D (B, Hk, S, d)");
    const int64_t B = q.size(0), H = q.size(1), S = q.size(2), d = q.size(3), Hk = k.size(1);
    TORCH_CHECK(k.size(0) == B && k.size(2) == S && k.size(3) == d, op, ": shape mismatch between q and k");
    check_head_dim(d, op);
    check_rows(q, op, "q");
    check_rows(k, op, "k");
    check_int(positions, positions.dim() == 1 ? 1 : 2, true, op, "positions");
    TORCH_CHECK(positions.size(-1) == S && (positions.dim() == 1 || positions.size(0) == B), op,
                ": positions must be (S) or (B, S)");
    TORCH_CHECK(S <= 1 || positions.stride(-1) == 1, op, ": the rows of positions must be contiguous");
    a.rotary = rotary_of(positions, freqs, interleaved, mscale, adjoint, d, op);
    const c10::cuda::CUDAGuard guard(q.device());
    auto q_out = empty({B, H, S, d}, q.scalar_type(), q), k_out = empty({B, Hk, S, d}, q.scalar_type(), q);
    a.struct_size = sizeof(a);
    a.device = q.get_device();
    a.q_batch_stride = step(q, 0), a.q_head_stride = step(q, 1), a.q_row_stride = step(q, 2);
    a.k_batch_stride = step(k, 0), a.k_head_stride = step(k, 1), a.k_row_stride = step(k, 2);
    a.position_batch_stride = positions.dim() == 2 ? step(positions, 0) : 0;
    a.heads = as_i32(H, "the number of heads");
    a.heads_k = as_i32(Hk, "the number of key heads"), a.seqlen = as_i32(S, "the length");
    a.head_dim = static_cast<int32_t>(d);
    const auto at = [](const Tensor& t, int64_t elements) { return static_cast<char*>(t.data_ptr()) + elements * t.element_size(); };
    for (int64_t b = 0; b < B; b += FA_ROTARY_MAX_BATCH) {
        a.batch = static_cast<int32_t>(std::min<int64_t>(B - b, FA_ROTARY_MAX_BATCH));
        a.q = at(q, b * a.q_batch_stride);
        a.k = at(k, b * a.k_batch_stride);
        a.q_out = at(q_out, b * H * S * d);
        a.k_out = at(k_out, b * Hk * S * d);
        a.rotary.positions = at(positions, b * a.position_batch_stride);
        check_rc(fa_rotary_sm100(&a, stream_of(q)), op);
    }
    return {q_out, k_out};
}

// Recorded gradients: the rotation is linear, so the gradient is one call of the operator, turning the other way.
using RotaryCall = std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&, bool, double, bool);

const c10::TypedOperatorHandle<RotaryCall>& rotary_op() {
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("recsys_ops::rotary", "").typed<RotaryCall>();
    return op;
}

// A gradient may come in any layout; the operator wants whole rows, 16-byte aligned.
Tensor as_rows(const Tensor& t) {
    const Tensor c = t.contiguous();
    return c.sym_storage_offset() % 8 == 0 ? c : c.clone();
}

struct RotaryFunction : torch::autograd::Function<RotaryFunction> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Tensor& k,
                                                  const Tensor& positions, const Tensor& freqs, bool interleaved, double mscale,
                                                  bool adjoint) {
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({positions, freqs});
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["mscale"] = mscale;
        ctx->saved_data["adjoint"] = adjoint;
        auto [q_out, k_out] = rotary_op().call(q, k, positions, freqs, interleaved, mscale, adjoint);
        return {q_out, k_out};
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        // heads whose gradient nobody wants are left out
        const bool for_q = ctx->needs_input_grad(0), for_k = ctx->needs_input_grad(1);
        const Tensor dq = as_rows(for_q ? grads[0] : grads[0].narrow(1, 0, 0));
        const Tensor dk = as_rows(for_k ? grads[1] : grads[1].narrow(1, 0, 0));
        auto [gq, gk] = rotary_op().call(dq, dk, saved[0], saved[1], ctx->saved_data["interleaved"].toBool(),
                                         ctx->saved_data["mscale"].toDouble(), !ctx->saved_data["adjoint"].toBool());
        return {for_q ? gq : Tensor(), for_k ? gk : Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

std::tuple<Tensor, Tensor> rotary_autograd(c10::DispatchKeySet keys, const Tensor& q, const Tensor& k, const Tensor& positions,
                                           const Tensor& freqs, bool interleaved, double mscale, bool adjoint) {
    if (c10::GradMode::is_enabled()) {
        TORCH_CHECK(!freqs.requires_grad(), "rotary: no gradient is recorded for freqs");
        if (q.requires_grad() || k.requires_grad()) {
            auto out = RotaryFunction::apply(q, k, positions, freqs, interleaved, mscale, adjoint);
            return {out[0], out[1]};
        }
    }
    return rotary_op().redispatch(keys & c10::after_ADInplaceOrView_keyset, q, k, positions, freqs, interleaved, mscale, adjoint);
}

FaPagedAppendArgs append_args(const Tensor& k, const Tensor& v, const Tensor& slots, const Tensor& k_cache,
                              const Tensor& v_cache, const char* op) {
    FaPagedAppendArgs a{};
    a.dtype = dtype_code(k, op);
    TORCH_CHECK(v.dtype() == k.dtype() && k_cache.dtype() == k.dtype() && v_cache.dtype() == k.dtype(), op,
                ": v and cache dtype must match k");
    a.cache = cache_of(k_cache, v_cache, op);
    at::assert_no_internal_overlap(k_cache);
    at::assert_no_internal_overlap(v_cache);
    at::assert_no_overlap(k_cache, v_cache);
    TORCH_CHECK(k.dim() == 3 && k.sizes() == v.sizes(), op, ": k and v must be 3D (T, Hk, d)");
    TORCH_CHECK(k.size(1) == a.cache.heads_k && k.size(2) == a.cache.head_dim, op, ": k and v must have the cache's heads and head_dim");
    check_rows(k, op, "k");
    check_rows(v, op, "v");
    check_list(slots, k.size(0), true, op, "slots");
    for (const Tensor* t : {&k, &v}) {        // rows would be read while others are written
        at::assert_no_overlap(k_cache, *t);
        at::assert_no_overlap(v_cache, *t);
    }
    a.struct_size = sizeof(a);
    a.device = k.get_device();
    a.k = k.data_ptr();
    a.v = v.data_ptr();
    a.slots = slots.data_ptr();
    a.slots_64 = slots.dtype() == torch::kLong;
    a.k_token_stride = step(k, 0), a.k_head_stride = step(k, 1);
    a.v_token_stride = step(v, 0), a.v_head_stride = step(v, 1);
    a.num_tokens = k.size(0);
    return a;
}

Tensor rotary_append(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& positions, const Tensor& slots,
                     const Tensor& k_cache, const Tensor& v_cache, const Tensor& freqs, bool interleaved, double mscale) {
    const char* op = "rotary_append";
    check_cuda(op, {&q, &k, &v, &positions, &slots, &k_cache, &v_cache, &freqs});
    FaPagedAppendArgs a = append_args(k, v, slots, k_cache, v_cache, op);
    TORCH_CHECK(q.dtype() == k.dtype(), op, ": q dtype must match k");
    TORCH_CHECK(q.dim() == 3 && q.size(0) == k.size(0) && q.size(2) == k.size(2), op, ": q must be 3D (T, H, d)");
    check_rows(q, op, "q");
    at::assert_no_overlap(k_cache, q);
    at::assert_no_overlap(v_cache, q);
    check_list(positions, k.size(0), true, op, "positions");
    a.rotary = rotary_of(positions, freqs, interleaved, mscale, false, q.size(2), op);
    const c10::cuda::CUDAGuard guard(q.device());
    auto out = empty({q.size(0), q.size(1), q.size(2)}, q.scalar_type(), q);
    a.q = q.data_ptr();
    a.q_out = out.data_ptr();
    a.q_token_stride = step(q, 0), a.q_head_stride = step(q, 1);
    a.heads = as_i32(q.size(1), "the number of heads");
    check_rc(fa_paged_append_sm100(&a, stream_of(q)), op);
    return out;
}

void paged_append(const Tensor& k, const Tensor& v, const Tensor& slots, const Tensor& k_cache, const Tensor& v_cache) {
    const char* op = "paged_append";
    check_cuda(op, {&k, &v, &slots, &k_cache, &v_cache});
    const FaPagedAppendArgs a = append_args(k, v, slots, k_cache, v_cache, op);
    const c10::cuda::CUDAGuard guard(k.device());
    check_rc(fa_paged_append_sm100(&a, stream_of(k)), op);
}

// ------------------------------------------------------------------ attention
std::tuple<Tensor, Tensor> attention(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache,
                                     const Tensor& block_table, const Tensor& seq_lens, c10::optional<double> scale,
                                     int64_t window, double softcap, const c10::optional<Tensor>& slopes, bool want_lse,
                                     const char* op) {
    check_cuda(op, {&q, &k_cache, &v_cache, &block_table, &seq_lens});
    FaPagedAttentionArgs a{};
    a.dtype = dtype_code(q, op);
    TORCH_CHECK(k_cache.dtype() == q.dtype() && v_cache.dtype() == q.dtype(), op, ": cache dtype must match q");
    a.cache = cache_of(k_cache, v_cache, op);
    TORCH_CHECK(q.dim() == 3, op, ": q must be 3D (B, H, d)");
    const int64_t B = q.size(0), H = q.size(1), d = q.size(2);
    TORCH_CHECK(d == a.cache.head_dim, op, ": head_dim mismatch between q and the cache");
    TORCH_CHECK(H % a.cache.heads_k == 0, op, ": n_heads must be divisible by n_kv_heads (GQA)");
    check_rows(q, op, "q");
    check_int(block_table, 2, false, op, "block_table");
    TORCH_CHECK(block_table.size(0) == B, op, ": block_table must hold one row per request");
    TORCH_CHECK(block_table.size(1) <= 1 || block_table.stride(1) == 1, op, ": the rows of block_table must be contiguous");
    check_list(seq_lens, B, false, op, "seq_lens");
    TORCH_CHECK(window >= 0, op, ": window must be >= 0");
    const double s = scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(d));
    TORCH_CHECK(std::isfinite(s) && s >= 0.0, op, ": scale must be finite and >= 0");
    TORCH_CHECK(std::isfinite(softcap) && softcap >= 0.0, op, ": softcap must be finite and >= 0");
    const bool biased = slopes.has_value() && slopes->defined();
    if (biased) {
        check_cuda(op, {&q, &*slopes});
        TORCH_CHECK(slopes->dtype() == torch::kFloat && slopes->dim() == 1 && slopes->size(0) == H && slopes->is_contiguous(), op,
                    ": slopes must be a contiguous float32 tensor with one value per head");
    }
    const c10::cuda::CUDAGuard guard(q.device());
    auto out = empty({B, H, d}, q.scalar_type(), q);
    Tensor lse;
    if (want_lse) lse = empty({B, H}, torch::kFloat, q);
    a.struct_size = sizeof(a);
    a.device = q.get_device();
    a.q = q.data_ptr();
    a.out = out.data_ptr();
    a.lse = want_lse ? lse.data_ptr<float>() : nullptr;
    a.block_table = block_table.data_ptr<int32_t>();
    a.lens = seq_lens.data_ptr<int32_t>();
    a.slopes = biased ? slopes->data_ptr<float>() : nullptr;
    a.q_batch_stride = step(q, 0), a.q_head_stride = step(q, 1);
    a.table_stride = step(block_table, 0);
    a.batch = as_i32(B, "the batch"), a.heads = as_i32(H, "the number of heads");
    a.table_width = as_i32(block_table.size(1), "the width of block_table");
    // a window beyond every length is no window
    a.window = static_cast<int32_t>(std::min<int64_t>(window, std::numeric_limits<int32_t>::max()));
    a.scale = static_cast<float>(s);
    a.softcap = static_cast<float>(softcap);
    size_t bytes = 0;
    check_rc(fa_paged_attention_sm100_workspace_bytes(&a, &bytes), op);
    Tensor ws;
    if (bytes > 0) ws = empty({static_cast<int64_t>(bytes)}, torch::kByte, q);
    check_rc(fa_paged_attention_sm100(&a, bytes > 0 ? ws.data_ptr() : nullptr, bytes, stream_of(q)), op);
    return {out, lse};
}

Tensor paged_attention(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& block_table,
                       const Tensor& seq_lens, c10::optional<double> scale, int64_t window, double softcap,
                       const c10::optional<Tensor>& slopes) {
    return std::get<0>(attention(q, k_cache, v_cache, block_table, seq_lens, scale, window, softcap, slopes, false,
                                 "paged_attention"));
}

std::tuple<Tensor, Tensor> paged_attention_lse(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache,
                                               const Tensor& block_table, const Tensor& seq_lens,
                                               c10::optional<double> scale, int64_t window, double softcap,
                                               const c10::optional<Tensor>& slopes) {
    return attention(q, k_cache, v_cache, block_table, seq_lens, scale, window, softcap, slopes, true, "paged_attention_lse");
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(recsys_ops, m) {
    m.def("paged_extend(Tensor(a!) block_table, Tensor seq_lens, Tensor new_lens, Tensor free_pages, Tensor free_head, "
          "int page_size, int num_tokens) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
    m.def("paged_extend_(Tensor(a!) block_table, Tensor(b!) seq_lens, Tensor new_lens, Tensor free_pages, "
          "Tensor(c!) free_head, int page_size, int num_tokens) -> (Tensor, Tensor, Tensor)");
    m.def("paged_shrink_(Tensor block_table, Tensor(a!) seq_lens, Tensor keep_lens, Tensor(b!) free_pages, "
          "Tensor(c!) free_head, int page_size) -> ()");
    m.def("rotary(Tensor q, Tensor k, Tensor positions, Tensor freqs, bool interleaved=False, float mscale=1.0, "
          "bool adjoint=False) -> (Tensor, Tensor)");
    m.def("rotary_append(Tensor q, Tensor k, Tensor v, Tensor positions, Tensor slots, Tensor(a!) k_cache, "
          "Tensor(b!) v_cache, Tensor freqs, bool interleaved=False, float mscale=1.0) -> Tensor");
    m.def("paged_append(Tensor k, Tensor v, Tensor slots, Tensor(a!) k_cache, Tensor(b!) v_cache) -> ()");
    m.def("paged_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, Tensor seq_lens, "
          "float? scale=None, int window=0, float softcap=0.0, Tensor? slopes=None) -> Tensor");
    m.def("paged_attention_lse(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, Tensor seq_lens, "
          "float? scale=None, int window=0, float softcap=0.0, Tensor? slopes=None) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(recsys_ops, CompositeExplicitAutograd, m) {
    m.impl("paged_extend", &paged_extend);
    m.impl("paged_extend_", &paged_extend_);
    m.impl("paged_shrink_", &paged_shrink_);
    m.impl("rotary", &rotary);
    m.impl("rotary_append", &rotary_append);
    m.impl("paged_append", &paged_append);
    m.impl("paged_attention", &paged_attention);
    m.impl("paged_attention_lse", &paged_attention_lse);
}

TORCH_LIBRARY_IMPL(recsys_ops, Autograd, m) { m.impl("rotary", &rotary_autograd); }

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) { m.doc() = "recsys_ops / paged group: paged key/value cache for sm_100a"; }
