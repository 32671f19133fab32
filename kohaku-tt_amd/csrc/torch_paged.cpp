// torch ops of the rotation and the paged cache (ktt::_rotary, ktt::_paged_append,
// ktt::_paged_read, ktt::_sdpa_paged) over the C ABI.  The Python entry points and what they
// accept are in kohakutt_amd/paged.py.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/autograd.h>
#include <torch/library.h>

#include <cmath>
#include <string>

#include "../../include/kohakutt_amd.h"

namespace kta {
namespace {

using at::Tensor;
using std::optional;

void check(int status, const char* what) {
    TORCH_CHECK(status == KMI_OK, "kohakutt_amd: ", what, " failed (", status, "): ", kmi_last_error());
}

int code_of(at::ScalarType t) {
    switch (t) {
        case at::kBFloat16: return KMI_BF16;
        case at::kHalf: return KMI_F16;
        case at::kFloat: return KMI_F32;
        default: return 0;
    }
}

void* stream_of(const Tensor& t) {
    return static_cast<void*>(c10::hip::getCurrentHIPStream(t.get_device()).stream());
}

bool given(const optional<Tensor>& t) { return t.has_value() && t->defined(); }

// Rows as the kernels read them: last-dim stride 1, 16-byte aligned, other strides multiples of
// 8 elements; anything else is copied once.
Tensor rows_operand(const Tensor& t) {
    bool ok = t.stride(-1) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    for (int64_t i = 0; ok && i + 1 < t.dim(); ++i) ok = t.stride(i) % 8 == 0 && t.stride(i) >= 0;
    if (ok) return t;
    const Tensor c = t.contiguous();
    return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone(at::MemoryFormat::Contiguous);
}

// ---------------------------------------------------------------- rotary

// One of the rotated tensors: [B, H, S, D], or packed [T, H, D].
void rotary_slot(kmi_rotary_args& a, int w, const Tensor& x, const Tensor& y) {
    const bool packed = x.dim() == 3;
    a.x[w] = x.data_ptr();
    a.y[w] = y.data_ptr();
    a.heads[w] = x.size(1);
    const Tensor* ts[2] = {&x, &y};
    int64_t* ss[2] = {a.x_stride[w], a.y_stride[w]};
    for (int i = 0; i < 2; ++i) {
        ss[i][0] = packed ? 0 : ts[i]->stride(0);
        ss[i][1] = ts[i]->stride(1);
        ss[i][2] = packed ? ts[i]->stride(0) : ts[i]->stride(2);
    }
}

std::tuple<Tensor, Tensor> rotary(const Tensor& x_in, const optional<Tensor>& second, const Tensor& positions,
                                  const Tensor& inv_freq, bool interleaved, double scale, bool inverse) {
    const char* op = "kohakutt_amd.rotary: ";
    const auto st = x_in.scalar_type();
    TORCH_CHECK_VALUE(st == at::kBFloat16 || st == at::kHalf || st == at::kFloat, op,
                      "tensors must be bf16, fp16 or fp32, got ", st);
    TORCH_CHECK_VALUE(x_in.dim() == 3 || x_in.dim() == 4, op, "tensors must be [B, H, S, D] or packed [T, H, D], got ",
                      x_in.sizes());
    const bool packed = x_in.dim() == 3;
    const int64_t batch = packed ? 1 : x_in.size(0), seq = packed ? x_in.size(0) : x_in.size(2), d = x_in.size(-1);
    if (given(second)) {
        const Tensor& k = *second;
        TORCH_CHECK_VALUE(k.scalar_type() == st && k.device() == x_in.device() && k.dim() == x_in.dim() &&
                              k.size(-1) == d && k.size(0) == x_in.size(0) && (packed || k.size(2) == seq),
                          op, "k must match the first tensor but for its heads, got ", k.sizes(), " ", k.scalar_type(),
                          " beside ", x_in.sizes(), " ", st);
    }
    TORCH_CHECK_VALUE(d >= 2 && d <= 256, op, "head dims must lie in [2, 256], got ", d);
    TORCH_CHECK_VALUE(inv_freq.scalar_type() == at::kFloat && inv_freq.dim() == 1 && inv_freq.numel() >= 1 &&
                          2 * inv_freq.numel() <= d && inv_freq.device() == x_in.device(),
                      op, "inv_freq must be fp32 [rotated dims / 2], at most ", d / 2, ", on the tensors' device, got ",
                      inv_freq.sizes(), " ", inv_freq.scalar_type());
    TORCH_CHECK_VALUE((positions.scalar_type() == at::kLong || positions.scalar_type() == at::kInt) &&
                          positions.device() == x_in.device(),
                      op, "positions must be int32 or int64 on the tensors' device, got ", positions.scalar_type());
    const bool shared = positions.dim() == 1 && positions.size(0) == seq;
    TORCH_CHECK_VALUE(shared || (!packed && positions.dim() == 2 && positions.size(1) == seq &&
                                 (positions.size(0) == batch || positions.size(0) == 1)),
                      op, "positions must be [", seq, "]", packed ? "" : " or [B or 1, S]", ", got ", positions.sizes());
    c10::DeviceGuard guard(x_in.device());
    const auto unit_rows = [](const Tensor& t) { return t.stride(-1) == 1 ? t : t.contiguous(); };
    const Tensor x = unit_rows(x_in);
    Tensor y = at::empty_like(x);
    if (y.stride(-1) != 1) y = at::empty(x.sizes(), x.options());
    const Tensor freq = inv_freq.contiguous();
    kmi_rotary_args a{};
    rotary_slot(a, 0, x, y);
    Tensor k, ky;  // (undefined without a second tensor)
    if (given(second)) {
        k = unit_rows(*second);
        ky = at::empty_like(k);
        if (ky.stride(-1) != 1) ky = at::empty(k.sizes(), k.options());
        rotary_slot(a, 1, k, ky);
    }
    if (x.numel() == 0 && (!k.defined() || k.numel() == 0)) return {y, ky};
    TORCH_CHECK_VALUE(x.size(1) > 0 && (!k.defined() || k.size(1) > 0), op, "tensors without heads");
    a.dtype = code_of(st);
    a.interleaved = interleaved;
    a.inverse = inverse;
    a.position_bits = positions.scalar_type() == at::kLong ? 64 : 32;
    a.batch = batch;
    a.seq = seq;
    a.head_dim = d;
    a.rotary_dim = 2 * freq.numel();
    a.positions = positions.data_ptr();
    a.position_stride[0] = positions.dim() == 2 && positions.size(0) > 1 ? positions.stride(0) : 0;
    a.position_stride[1] = positions.stride(-1);
    a.inv_freq = freq.data_ptr<float>();
    a.scale = scale;
    check(kmi_rotary(&a, stream_of(x)), "kmi_rotary");
    return {y, ky};
}

using RotaryOp = std::tuple<Tensor, Tensor>(const Tensor&, const optional<Tensor>&, const Tensor&, const Tensor&, bool,
                                            double, bool);

// The op through the dispatcher: the gradient's own gradient is the rotation again.
const c10::TypedOperatorHandle<RotaryOp>& rotary_op() {
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("ktt::_rotary", "").typed<RotaryOp>();
    return op;
}

// Rotary positions with gradients: the rotation back of whichever gradients there are.
struct RotaryFn : public torch::autograd::Function<RotaryFn> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& x,
                                                  const optional<Tensor>& second, const Tensor& positions,
                                                  const Tensor& inv_freq, bool interleaved, double scale, bool inverse) {
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({positions, inv_freq});
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["inverse"] = inverse;
        ctx->set_materialize_grads(false);
        auto [y, ky] = rotary_op().call(x, second, positions, inv_freq, interleaved, scale, inverse);
        if (!ky.defined()) return {y};
        return {y, ky};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                   torch::autograd::variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor first = grads[0], second = grads.size() > 1 ? grads[1] : Tensor();
        Tensor gx, gk;
        if (first.defined() || second.defined()) {
            const bool both = first.defined() && second.defined();
            auto [a, b] = rotary_op().call(first.defined() ? first : second, both ? optional<Tensor>(second) : std::nullopt,
                                           saved[0], saved[1], ctx->saved_data["interleaved"].toBool(),
                                           ctx->saved_data["scale"].toDouble(), !ctx->saved_data["inverse"].toBool());
            (first.defined() ? gx : gk) = a;
            if (both) gk = b;
        }
        return {gx, gk, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

// ktt::_rotary at AutogradCUDA.
std::tuple<Tensor, Tensor> rotary_autograd(const Tensor& x, const optional<Tensor>& second, const Tensor& positions,
                                           const Tensor& inv_freq, bool interleaved, double scale, bool inverse) {
    TORCH_CHECK_VALUE(!at::GradMode::is_enabled() || !inv_freq.requires_grad(),
                      "kohakutt_amd.rotary: inv_freq takes no gradient");
    if (at::GradMode::is_enabled() && (x.requires_grad() || (given(second) && second->requires_grad()))) {
        auto out = RotaryFn::apply(x, second, positions, inv_freq, interleaved, scale, inverse);
        return {out[0], out.size() > 1 ? out[1] : Tensor()};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    // (Traced tensors have no data: the dispatcher finds them their shapes.)
    constexpr c10::DispatchKeySet traced({c10::DispatchKey::Python, c10::DispatchKey::PythonTLSSnapshot,
                                          c10::DispatchKey::Functionalize});
    if (!(x.key_set() & traced).empty()) return rotary_op().call(x, second, positions, inv_freq, interleaved, scale, inverse);
    return rotary(x, second, positions, inv_freq, interleaved, scale, inverse);
}

// ---------------------------------------------------------------- the cache

int64_t stride_of(const Tensor& t, int64_t i) { return t.size(i) > 1 ? t.stride(i) : 0; }

// The cache of a call, checked.  `dtype`: what a 4-bit cache's values come out in.
kmi_paged_cache cache_of(const char* op, const Tensor& k, const Tensor& v, const optional<Tensor>& k_scale,
                         const optional<Tensor>& v_scale, const Tensor& table, const Tensor& lengths,
                         const optional<Tensor>& cu, int64_t tokens, at::ScalarType dtype) {
    kmi_paged_cache c{};
    const bool four = given(k_scale) || given(v_scale);
    TORCH_CHECK_VALUE(k.dim() == 4 && v.dim() == 4 && k.size(0) == v.size(0) && k.size(1) == v.size(1) &&
                          k.size(2) == v.size(2),
                      op, "k_cache and v_cache must be [pages, heads, page size, D], got ", k.sizes(), " and ", v.sizes());
    const int64_t pages = k.size(0), heads = k.size(1), page = k.size(2);
    TORCH_CHECK_VALUE(pages > 0 && heads > 0 && page > 0 && page % 16 == 0, op,
                      "a cache needs pages, heads and pages of a multiple of 16 keys, got ", k.sizes());
    const auto dev = k.device();
    TORCH_CHECK_VALUE(v.device() == dev && table.device() == dev && lengths.device() == dev, op,
                      "the cache, block_table and key_lengths must be on one device");
    TORCH_CHECK_VALUE(table.scalar_type() == at::kInt && table.dim() == 2, op, "block_table must be int32 [B, pages of a "
                      "sequence], got ", table.sizes(), " ", table.scalar_type());
    TORCH_CHECK_VALUE(lengths.scalar_type() == at::kInt && lengths.dim() == 1 && lengths.size(0) == table.size(0), op,
                      "key_lengths must be int32 [", table.size(0), "], got ", lengths.sizes(), " ", lengths.scalar_type());
    TORCH_CHECK_VALUE(table.size(1) == 0 || table.stride(1) == 1 || table.size(1) == 1, op,
                      "block_table rows must be contiguous");
    TORCH_CHECK_VALUE(lengths.size(0) <= 1 || lengths.stride(0) == 1, op, "key_lengths must be contiguous");
    TORCH_CHECK_VALUE(k.stride(3) == 1 && v.stride(3) == 1, op, "cache rows must be contiguous");
    if (four) {
        TORCH_CHECK_VALUE(given(k_scale) && given(v_scale) && k.scalar_type() == at::kByte &&
                              v.scalar_type() == at::kByte && k_scale->scalar_type() == at::kByte &&
                              v_scale->scalar_type() == at::kByte,
                          op, "a 4-bit cache is four uint8 tensors: k_cache, v_cache, k_scale and v_scale");
        const Tensor* vals[2] = {&k, &v};
        const Tensor* scs[2] = {&*k_scale, &*v_scale};
        for (int i = 0; i < 2; ++i)
            TORCH_CHECK_VALUE(scs[i]->dim() == 4 && scs[i]->device() == dev && scs[i]->size(0) == pages &&
                                  scs[i]->size(1) == heads && scs[i]->size(2) == page &&
                                  scs[i]->size(3) * 16 == vals[i]->size(3) && (scs[i]->size(3) == 1 || scs[i]->stride(3) == 1),
                              op, "scales must be [pages, heads, page size, D / 32] with contiguous rows, got ",
                              scs[i]->sizes(), " beside codes ", vals[i]->sizes());
        TORCH_CHECK_VALUE(dtype == at::kBFloat16 || dtype == at::kHalf, op, "values must be bf16 or fp16, got ", dtype);
        c.k_scale = k_scale->data_ptr();
        c.v_scale = v_scale->data_ptr();
        for (int i = 0; i < 3; ++i) {
            c.k_scale_stride[i] = stride_of(*k_scale, i);
            c.v_scale_stride[i] = stride_of(*v_scale, i);
        }
    } else {
        TORCH_CHECK_VALUE((k.scalar_type() == at::kBFloat16 || k.scalar_type() == at::kHalf) &&
                              v.scalar_type() == k.scalar_type(),
                          op, "k_cache and v_cache must be bf16 or fp16 (or uint8 codes with scales), got ",
                          k.scalar_type(), " and ", v.scalar_type());
        TORCH_CHECK_VALUE(dtype == k.scalar_type(), op, "the cache is ", k.scalar_type(), ", not ", dtype);
    }
    c.k = k.data_ptr();
    c.v = v.data_ptr();
    for (int i = 0; i < 3; ++i) {
        c.k_stride[i] = stride_of(k, i);
        c.v_stride[i] = stride_of(v, i);
    }
    c.dtype = code_of(dtype);
    c.bits = four ? 4 : 16;
    c.pages = pages;
    c.page_size = page;
    c.heads_kv = heads;
    c.head_dim = k.size(3) * (four ? 2 : 1);
    c.head_dim_v = v.size(3) * (four ? 2 : 1);
    c.block_table = table.data_ptr<int32_t>();
    c.table_stride = table.size(0) > 1 ? table.stride(0) : 0;
    c.table_width = table.size(1);
    c.key_lengths = lengths.data_ptr<int32_t>();
    c.batch = table.size(0);
    c.tokens = tokens;
    if (given(cu)) {
        TORCH_CHECK_VALUE(cu->scalar_type() == at::kInt && cu->dim() == 1 && cu->size(0) == c.batch + 1 &&
                              cu->device() == dev && (cu->size(0) == 1 || cu->stride(0) == 1),
                          op, "offsets must be contiguous int32 [", c.batch + 1, "] on the cache's device, got ",
                          cu->sizes(), " ", cu->scalar_type());
        c.cu_seqlens = cu->data_ptr<int32_t>();
    }
    return c;
}

optional<Tensor> paged_append(const Tensor& k_in, const Tensor& v_in, const Tensor& k_cache, const Tensor& v_cache,
                              const Tensor& table, const Tensor& lengths, const optional<Tensor>& cu,
                              const optional<Tensor>& q_in, const optional<Tensor>& inv_freq, bool interleaved,
                              double rotary_scale, const optional<Tensor>& k_scale, const optional<Tensor>& v_scale) {
    const char* op = "kohakutt_amd.paged_append: ";
    TORCH_CHECK_VALUE(k_in.dim() == 3 && v_in.dim() == 3 && k_in.size(0) == v_in.size(0) && k_in.size(1) == v_in.size(1),
                      op, "k and v must be [T, heads, D], got ", k_in.sizes(), " and ", v_in.sizes());
    TORCH_CHECK_VALUE(k_in.scalar_type() == v_in.scalar_type() && k_in.device() == v_in.device() &&
                          k_in.device() == k_cache.device(),
                      op, "k and v must have one type and be on the cache's device");
    const auto st = k_in.scalar_type();
    kmi_paged_append_args a{};
    a.cache = cache_of(op, k_cache, v_cache, k_scale, v_scale, table, lengths, cu, k_in.size(0), st);
    TORCH_CHECK_VALUE(k_in.size(1) == a.cache.heads_kv && k_in.size(2) == a.cache.head_dim &&
                          v_in.size(2) == a.cache.head_dim_v,
                      op, "k and v are [T, ", k_in.size(1), ", ", k_in.size(2), " / ", v_in.size(2), "], the cache holds [",
                      a.cache.heads_kv, ", ", a.cache.head_dim, " / ", a.cache.head_dim_v, "]");
    TORCH_CHECK_VALUE(!at::GradMode::is_enabled() || !(k_in.requires_grad() || v_in.requires_grad()), op,
                      "a cache takes no gradients: call it under torch.no_grad()");
    TORCH_CHECK_VALUE(given(cu) || a.cache.tokens == a.cache.batch, op, "without offsets there is one token per sequence (",
                      a.cache.batch, "), got ", a.cache.tokens);
    c10::DeviceGuard guard(k_in.device());
    const Tensor k = rows_operand(k_in), v = rows_operand(v_in);
    Tensor q, q_out, freq;
    if (given(inv_freq)) {
        TORCH_CHECK_VALUE(!at::GradMode::is_enabled() || !inv_freq->requires_grad(), op,
                          "a cache takes no gradients: call it under torch.no_grad()");
        TORCH_CHECK_VALUE(inv_freq->scalar_type() == at::kFloat && inv_freq->dim() == 1 && inv_freq->numel() >= 1 &&
                              2 * inv_freq->numel() <= a.cache.head_dim && inv_freq->device() == k.device(),
                          op, "inv_freq must be fp32 [rotated dims / 2], at most ", a.cache.head_dim / 2,
                          ", on the cache's device, got ", inv_freq->sizes(), " ", inv_freq->scalar_type());
        freq = inv_freq->contiguous();
        a.inv_freq = freq.data_ptr<float>();
        a.rotary_dim = 2 * freq.numel();
    }
    if (given(q_in)) {
        TORCH_CHECK_VALUE(given(inv_freq), op, "q is taken to be rotated: it needs inv_freq");
        TORCH_CHECK_VALUE(q_in->dim() == 3 && q_in->size(0) == k.size(0) && q_in->size(1) > 0 &&
                              q_in->size(2) == a.cache.head_dim && q_in->scalar_type() == st &&
                              q_in->device() == k.device(),
                          op, "q must be [", k.size(0), ", heads, ", a.cache.head_dim, "] of k's type and device, got ",
                          q_in->sizes(), " ", q_in->scalar_type());
        TORCH_CHECK_VALUE(!at::GradMode::is_enabled() || !q_in->requires_grad(), op,
                          "a cache takes no gradients: call it under torch.no_grad()");
        q = rows_operand(*q_in);
        q_out = at::empty(q.sizes(), q.options());
        a.q = q.data_ptr();
        a.q_out = q_out.data_ptr();
        a.heads_q = q.size(1);
        for (int i = 0; i < 2; ++i) {
            a.q_stride[i] = q.stride(i);
            a.q_out_stride[i] = q_out.stride(i);
        }
    }
    if (a.cache.tokens > 0) {
        a.k = k.data_ptr();
        a.v = v.data_ptr();
        for (int i = 0; i < 2; ++i) {
            a.k_stride[i] = k.stride(i);
            a.v_stride[i] = v.stride(i);
        }
        a.interleaved = interleaved;
        a.rotary_scale = rotary_scale;
        check(kmi_paged_append(&a, stream_of(k)), "kmi_paged_append");
    }
    if (!q_out.defined()) return std::nullopt;
    return q_out;
}

std::tuple<Tensor, Tensor> paged_read(const Tensor& k_cache, const Tensor& v_cache, const Tensor& table,
                                      const Tensor& lengths, int64_t max_k, at::ScalarType dtype,
                                      const optional<Tensor>& k_scale, const optional<Tensor>& v_scale) {
    const char* op = "kohakutt_amd.paged_read: ";
    const kmi_paged_cache c = cache_of(op, k_cache, v_cache, k_scale, v_scale, table, lengths, std::nullopt, 0, dtype);
    TORCH_CHECK_VALUE(max_k >= 0, op, "max_k must not be negative, got ", max_k);
    c10::DeviceGuard guard(k_cache.device());
    const auto opts = k_cache.options().dtype(dtype);
    Tensor k = at::empty({c.batch, c.heads_kv, max_k, c.head_dim}, opts);
    Tensor v = at::empty({c.batch, c.heads_kv, max_k, c.head_dim_v}, opts);
    if (k.numel() > 0)
        check(kmi_paged_read(&c, k.data_ptr(), v.data_ptr(), max_k, stream_of(k)), "kmi_paged_read");
    return {k, v};
}

// (out [T, H, Dv], lse [H, T] when `stats`, else none.)
std::tuple<Tensor, Tensor> sdpa_paged(const Tensor& q_in, const Tensor& k_cache, const Tensor& v_cache,
                                      const Tensor& table, const Tensor& lengths, const optional<Tensor>& cu,
                                      optional<int64_t> max_q, optional<int64_t> max_k, bool is_causal,
                                      optional<double> scale, bool stats, const optional<Tensor>& k_scale,
                                      const optional<Tensor>& v_scale) {
    const char* op = "kohakutt_amd.sdpa_paged: ";
    TORCH_CHECK_VALUE(q_in.dim() == 3, op, "q must be [T, heads, D], got ", q_in.sizes());
    TORCH_CHECK_VALUE(q_in.device() == k_cache.device(), op, "q must be on the cache's device");
    TORCH_CHECK_VALUE(q_in.scalar_type() == at::kBFloat16 || q_in.scalar_type() == at::kHalf, op,
                      "q must be bf16 or fp16, got ", q_in.scalar_type());
    TORCH_CHECK_VALUE(!at::GradMode::is_enabled() || !q_in.requires_grad(), op,
                      "attention over a cache has no gradient: call it under torch.no_grad()");
    kmi_paged_attn_args a{};
    a.cache = cache_of(op, k_cache, v_cache, k_scale, v_scale, table, lengths, cu, q_in.size(0), q_in.scalar_type());
    const kmi_paged_cache& c = a.cache;
    TORCH_CHECK_VALUE(q_in.size(2) == c.head_dim && q_in.size(1) > 0 && q_in.size(1) % c.heads_kv == 0, op, "q is [T, ",
                      q_in.size(1), ", ", q_in.size(2), "]; the cache holds ", c.heads_kv, " heads (which must divide q's) of ",
                      c.head_dim);
    TORCH_CHECK_VALUE(given(cu) || c.tokens == c.batch, op, "without offsets there is one token per sequence (", c.batch,
                      "), got ", c.tokens);
    a.max_q = max_q.value_or(given(cu) ? c.tokens : 1);
    a.max_k = max_k.value_or(c.table_width * c.page_size);
    TORCH_CHECK_VALUE(a.max_q >= 0 && a.max_k >= 0, op, "max_q and max_k must not be negative, got ", a.max_q, " and ",
                      a.max_k);
    a.max_q = std::min(a.max_q, c.tokens);
    c10::DeviceGuard guard(q_in.device());
    const Tensor q = rows_operand(q_in);
    Tensor out = at::empty({c.tokens, q.size(1), c.head_dim_v}, q.options());
    Tensor lse;  // (undefined without statistics)
    if (stats) lse = at::empty({q.size(1), c.tokens}, q.options().dtype(at::kFloat));
    if (c.tokens == 0) return {out, lse};
    if (c.batch == 0) {
        if (stats) lse.fill_(-INFINITY);
        return {out.zero_(), lse};
    }
    a.q = q.data_ptr();
    a.out = out.data_ptr();
    if (stats) a.lse = lse.data_ptr<float>();
    for (int i = 0; i < 2; ++i) {
        a.q_stride[i] = q.stride(i);
        a.o_stride[i] = out.stride(i);
        if (stats) a.lse_stride[i] = lse.stride(i);
    }
    a.heads_q = q.size(1);
    a.causal = is_causal;
    a.scale = scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(c.head_dim));
    size_t ws = 0;
    check(kmi_paged_attn_workspace_bytes(&a, &ws), "kmi_paged_attn_workspace_bytes");
    Tensor work;
    if (ws) work = at::empty({static_cast<int64_t>(ws)}, q.options().dtype(at::kByte));
    check(kmi_paged_attn(&a, ws ? work.data_ptr() : nullptr, ws, stream_of(q)), "kmi_paged_attn");
    return {out, lse};
}

}  // namespace
}  // namespace kta

TORCH_LIBRARY_FRAGMENT(ktt, m) {
    m.def("_rotary(Tensor x, Tensor? second, Tensor positions, Tensor inv_freq, bool interleaved=False, "
          "float scale=1.0, bool inverse=False) -> (Tensor, Tensor)");
    m.def("_paged_append(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor block_table, "
          "Tensor key_lengths, Tensor? cu_seq=None, Tensor? q=None, Tensor? inv_freq=None, bool interleaved=False, "
          "float rotary_scale=1.0, Tensor(c!)? k_scale=None, Tensor(d!)? v_scale=None) -> Tensor?");
    m.def("_paged_read(Tensor k_cache, Tensor v_cache, Tensor block_table, Tensor key_lengths, int max_k, "
          "ScalarType dtype, Tensor? k_scale=None, Tensor? v_scale=None) -> (Tensor, Tensor)");
    m.def("_sdpa_paged(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, Tensor key_lengths, "
          "Tensor? cu_seq_q=None, int? max_q=None, int? max_k=None, bool is_causal=True, float? scale=None, "
          "bool stats=False, Tensor? k_scale=None, Tensor? v_scale=None) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(ktt, CUDA, m) {
    m.impl("_rotary", TORCH_FN(kta::rotary));
    m.impl("_paged_append", TORCH_FN(kta::paged_append));
    m.impl("_paged_read", TORCH_FN(kta::paged_read));
    m.impl("_sdpa_paged", TORCH_FN(kta::sdpa_paged));
}

TORCH_LIBRARY_IMPL(ktt, AutogradCUDA, m) {
    m.impl("_rotary", TORCH_FN(kta::rotary_autograd));
}
