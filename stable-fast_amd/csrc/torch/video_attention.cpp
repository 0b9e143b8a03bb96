// torch.ops.sfast.rotary_embedding_nd and torch.ops.sfast_xformers.block_* on the C ABI of libsfast_hip.so, with their gradients.
//
// Native because these calls are small where they are made once a token: argument checks, allocation and launch cost 6 - 11 us here against
// 15 - 32 us through ctypes, a call with its gradient 66 - 81 us against 230 - 250 (45 of them are what torch's engine takes for any backward).
// The rules are those of the Python operators: outputs are fresh tensors, inputs are never written, work goes to the current stream of the
// input's device, operands a kernel cannot read in place are copied, everything else is refused.
#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <ATen/ops/zeros_like.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <atomic>
#include <cmath>
#include <limits>

#include "../../../include/sfast_hip.h"

namespace {

using at::Tensor;
using c10::optional;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

#define SFAST_RUN(call, what)                                                                    \
    do {                                                                                         \
        const int rc_ = (call);                                                                  \
        TORCH_CHECK(rc_ == SFAST_OK, what, " failed (", rc_, "): ", sfast_hip_last_error());     \
    } while (0)

// Selects the first tensor's device for the call (launches, kernel attributes and allocations follow it) and sets its kernels up once.
struct Call {
    c10::DeviceGuard guard;
    sfast_stream_t stream;
    explicit Call(const char *who, const Tensor &t) : guard(checked(who, t)) {
        static std::atomic<bool> ready[64];
        const auto index = t.device().index();
        TORCH_CHECK(index >= 0 && index < 64, who, ": device ", t.device());
        if (!ready[index].load(std::memory_order_acquire)) {
            TORCH_CHECK(sfast_hip_abi_version() == SFAST_HIP_ABI_VERSION, who, ": libsfast_hip.so ABI version mismatch; rebuild");
            SFAST_RUN(sfast_hip_init(), "sfast_hip_init");
            ready[index].store(true, std::memory_order_release);
        }
        stream = (sfast_stream_t)c10::hip::getCurrentHIPStream(index).stream();
    }
    static c10::Device checked(const char *who, const Tensor &t) {
        TORCH_CHECK(t.is_cuda(), who, ": needs tensors on a ROCm device (got ", t.device(), "); there is no CPU path");
        return t.device();
    }
};

void same_device(const char *who, const Tensor &first, const Tensor &other) {
    TORCH_CHECK(!other.defined() || other.device() == first.device(), who, ": tensors on ", first.device(), " and ", other.device());
}

int dtype_of(const char *who, const Tensor &t) {
    if (t.scalar_type() == at::kHalf) return SFAST_F16;
    if (t.scalar_type() == at::kBFloat16) return SFAST_BF16;
    TORCH_CHECK(t.scalar_type() == at::kFloat, who, ": f16 / bf16 / f32 only, got ", t.scalar_type());
    return SFAST_F32;
}

int32_t i32(const char *who, int64_t n) {
    TORCH_CHECK(n >= 0 && n <= std::numeric_limits<int32_t>::max(), who, ": a dimension of ", n, " is too long");
    return (int32_t)n;
}

void strides(const Tensor &t, int64_t *out) {
    for (int i = 0; i < 3; ++i) out[i] = t.stride(i);
}

Tensor contiguous_copy(const Tensor &t) { return t.clone(at::MemoryFormat::Contiguous); }

// [B] sequence lengths as int32 (undefined: every sequence is full). Their values stay on the device; the kernels clip them.
Tensor lengths_of(const char *who, const char *name, const optional<Tensor> &lengths, int64_t B, int64_t S, const Tensor &like) {
    if (!lengths || !lengths->defined()) return Tensor();
    const Tensor &t = *lengths;
    same_device(who, like, t);
    TORCH_CHECK((t.scalar_type() == at::kInt || t.scalar_type() == at::kLong) && t.dim() == 1 && t.size(0) == B, who, ": ", name, " must be ", B,
                " int32 or int64 values, got ", t.scalar_type(), " ", t.sizes());
    return t.scalar_type() == at::kLong ? t.clamp(0, S).to(at::kInt).contiguous() : t.contiguous();
}

const int32_t *ints(const Tensor &t) { return t.defined() ? t.const_data_ptr<int32_t>() : nullptr; }

Tensor workspace(size_t bytes, const Tensor &like) {
    return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}
void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

// ---- rotary positions -------------------------------------------------------------------------------------------------------------------
std::tuple<Tensor, Tensor> rotary(const Tensor &query, const optional<Tensor> &key, const Tensor &positions, at::IntArrayRef sections, double theta,
                                  bool interleaved, bool inverse) {
    const char *who = "rotary_embedding_nd";
    const Call call(who, query);
    Tensor q = query, k = key ? *key : Tensor(), pos = positions;
    same_device(who, q, k);
    same_device(who, q, pos);
    TORCH_CHECK(q.dim() == 4 && (!k.defined() || (k.dim() == 4 && k.size(0) == q.size(0) && k.size(1) == q.size(1) && k.size(3) == q.size(3) &&
                                                  k.scalar_type() == q.scalar_type())),
                who, ": expected query [B, S, H, D] and key [B, S, Hk, D] of one type");
    sfast_rope_params p{};
    const int64_t B = q.size(0), S = q.size(1), H = q.size(2), D = q.size(3), Hk = k.defined() ? k.size(2) : 0, A = (int64_t)sections.size();
    p.dtype = dtype_of(who, q);
    p.B = i32(who, B), p.S = i32(who, S), p.H = i32(who, H), p.Hk = i32(who, Hk), p.D = i32(who, D);
    TORCH_CHECK(A >= 1 && A <= SFAST_ROPE_MAX_AXES, who, ": 1 to ", SFAST_ROPE_MAX_AXES, " axes, got ", A);
    int64_t used = 0;
    for (int64_t a = 0; a < A; ++a) {
        TORCH_CHECK(sections[a] > 0 && sections[a] % 2 == 0 && sections[a] <= D - used, who, ": sections ", sections,
                    " must be even, positive and fit the head dim ", D);
        p.sections[a] = (int32_t)sections[a];
        used += sections[a];
    }
    TORCH_CHECK(theta > 0.0 && std::isfinite(theta), who, ": theta must be positive and finite, got ", theta);
    p.n_axes = (int32_t)A, p.interleaved = interleaved, p.inverse = inverse, p.theta = theta;
    switch (pos.scalar_type()) {
    case at::kInt: p.pos_type = SFAST_POS_I32; break;
    case at::kLong: p.pos_type = SFAST_POS_I64; break;
    case at::kFloat: p.pos_type = SFAST_POS_F32; break;
    case at::kDouble: p.pos_type = SFAST_POS_F64; break;
    default: TORCH_CHECK(false, who, ": positions must be int32, int64, float32 or float64, got ", pos.scalar_type());
    }
    const int64_t pd = pos.dim();
    TORCH_CHECK((pd == 2 || (pd == 3 && (pos.size(0) == 1 || pos.size(0) == B))) && pos.size(pd - 2) == S && pos.size(pd - 1) == A, who,
                ": positions must be [S, ", A, "] or [B, S, ", A, "], got ", pos.sizes());
    if (pos.stride(pd - 1) != 1) pos = pos.contiguous();
    p.ps[0] = pd == 3 && pos.size(0) > 1 ? pos.stride(0) : 0;
    p.ps[1] = pos.stride(pd - 2);
    // neighbouring pairs are read whole: rows start at even elements and pair-aligned addresses
    const auto fit = [&](Tensor &t) {
        bool ok = t.stride(3) == 1;
        if (ok && interleaved)
            ok = t.stride(0) % 2 == 0 && t.stride(1) % 2 == 0 && t.stride(2) % 2 == 0 && (uintptr_t)t.const_data_ptr() % (2 * t.element_size()) == 0;
        if (!ok) t = contiguous_copy(t);
    };
    Tensor qo = at::empty(q.sizes(), q.options()), ko = k.defined() ? at::empty(k.sizes(), k.options()) : Tensor();
    if (qo.numel() == 0) {
        if (ko.defined() && ko.numel()) ko = std::get<0>(rotary(k, c10::nullopt, positions, sections, theta, interleaved, inverse));
        return {qo, ko};
    }
    TORCH_CHECK(D % 2 == 0 && D <= 256, who, ": head dim ", D, " (even, up to 256)");
    fit(q);
    strides(q, p.qs), strides(qo, p.qos);
    if (k.defined() && k.numel() == 0) p.Hk = 0;
    if (p.Hk) fit(k), strides(k, p.ks), strides(ko, p.kos);
    SFAST_RUN(sfast_hip_rope_nd(q.const_data_ptr(), p.Hk ? k.const_data_ptr() : nullptr, pos.const_data_ptr(), qo.data_ptr(),
                                p.Hk ? ko.data_ptr() : nullptr, &p, call.stream),
              "sfast_hip_rope_nd");
    return {qo, ko};
}

struct Rotary : torch::autograd::Function<Rotary> {
    static variable_list forward(AutogradContext *ctx, const Variable &q, const optional<Variable> &k, const Variable &positions, std::vector<int64_t> sections,
                                 double theta, bool interleaved, bool inverse) {
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({positions});
        ctx->saved_data["sections"] = sections;
        ctx->saved_data["theta"] = theta;
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["inverse"] = inverse;
        ctx->set_materialize_grads(false);
        auto [qo, ko] = rotary(q, k, positions, sections, theta, interleaved, inverse);
        if (!ko.defined()) return {qo};
        return {qo, ko};
    }
    // a turn is orthogonal: its gradient is the turn back (positions take no gradient)
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const auto positions = ctx->get_saved_variables()[0];
        const auto sections = ctx->saved_data["sections"].toIntVector();
        const bool inverse = ctx->saved_data["inverse"].toBool();
        static const auto op = c10::Dispatcher::singleton()
                                   .findSchemaOrThrow("sfast::rotary_embedding_nd", "")
                                   .typed<std::tuple<Tensor, Tensor>(const Tensor &, const optional<Tensor> &, const Tensor &, at::IntArrayRef, double, bool, bool)>();
        variable_list out(7);
        const bool q = grads[0].defined(), k = grads.size() > 1 && grads[1].defined();
        if (q || k) {
            auto [x, y] = op.call(q ? grads[0] : grads[1], q && k ? optional<Tensor>(grads[1]) : c10::nullopt, positions, sections, ctx->saved_data["theta"].toDouble(),
                                  ctx->saved_data["interleaved"].toBool(), !inverse);
            if (q) out[0] = x;
            if (k) out[1] = q ? y : x;
        }
        return out;
    }
};

bool wants_grad(std::initializer_list<const Tensor *> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor *t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// There are no derivatives in forward mode; a tangent that was left behind would count as zero.
void no_tangents(const char *who, std::initializer_list<const Tensor *> ts) {
    for (const Tensor *t : ts)
        TORCH_CHECK(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), who, ": there are no derivatives in forward mode (a tensor carries a tangent)");
}

std::tuple<Tensor, Tensor> rotary_autograd(const Tensor &q, const optional<Tensor> &key, const Tensor &positions, at::IntArrayRef sections, double theta,
                                           bool interleaved, bool inverse) {
    const Tensor k = key ? *key : Tensor();
    no_tangents("rotary_embedding_nd", {&q, &k, &positions});
    if (!wants_grad({&q, &k})) {
        at::AutoDispatchBelowADInplaceOrView below;
        return rotary(q, key, positions, sections, theta, interleaved, inverse);
    }
    auto r = Rotary::apply(q, key, positions, sections.vec(), theta, interleaved, inverse);
    return {r[0], r.size() > 1 ? r[1] : Tensor()};
}

// ---- block means and choice ---------------------------------------------------------------------------------------------------------------
Tensor block_means(const Tensor &input, int64_t block, const optional<Tensor> &lengths) {
    const char *who = "block_means";
    const Call call(who, input);
    Tensor x = input;
    TORCH_CHECK(x.dim() == 4, who, ": expected [B, S, H, D]");
    TORCH_CHECK(block >= 1 && block <= 1024, who, ": blocks of ", block, " rows (1 to 1024)");
    sfast_block_means_params p{};
    p.dtype = dtype_of(who, x);
    p.B = i32(who, x.size(0)), p.S = i32(who, x.size(1)), p.H = i32(who, x.size(2)), p.D = i32(who, x.size(3)), p.block = (int32_t)block;
    i32(who, x.size(2) * x.size(3));
    const Tensor len = lengths_of(who, "lengths", lengths, p.B, p.S, x);
    Tensor out = at::empty({p.B, (p.S + block - 1) / block, p.H, p.D}, x.options().dtype(at::kFloat));
    if (out.numel() == 0) return out;
    if (x.stride(3) != 1) x = contiguous_copy(x);
    strides(x, p.xs);
    SFAST_RUN(sfast_hip_block_means(x.const_data_ptr(), ints(len), out.data_ptr<float>(), &p, call.stream), "sfast_hip_block_means");
    return out;
}

Tensor block_topk(const Tensor &query_means, const Tensor &key_means, int64_t topk, int64_t block_k, const optional<Tensor> &key_lengths) {
    const char *who = "block_topk";
    const Call call(who, query_means);
    Tensor qm = query_means, km = key_means;
    same_device(who, qm, km);
    TORCH_CHECK(qm.dim() == 4 && km.dim() == 4 && qm.scalar_type() == at::kFloat && km.scalar_type() == at::kFloat, who,
                ": expected fp32 means [B, nQ, H, D] and [B, nK, Hk, D]");
    TORCH_CHECK(km.size(0) == qm.size(0) && km.size(3) == qm.size(3) && km.size(2) > 0 && qm.size(2) % km.size(2) == 0, who, ": means ", qm.sizes(), " and ",
                km.sizes(), " do not fit");
    TORCH_CHECK(topk >= 1 && block_k >= 1, who, ": topk ", topk, " and block_k ", block_k, " must be positive");
    sfast_block_topk_params p{};
    p.B = i32(who, qm.size(0)), p.nQ = i32(who, qm.size(1)), p.nK = i32(who, km.size(1)), p.H = i32(who, qm.size(2)), p.Hk = i32(who, km.size(2));
    p.D = i32(who, qm.size(3)), p.topk = i32(who, topk), p.block_k = i32(who, block_k);
    const int64_t reach = std::min<int64_t>((int64_t)p.nK * block_k, std::numeric_limits<int32_t>::max());
    const Tensor len = lengths_of(who, "key_lengths", key_lengths, p.B, reach, qm);
    Tensor out = at::empty({p.B, p.Hk, p.nQ, topk}, qm.options().dtype(at::kInt));
    if (out.numel() == 0) return out;
    if (p.nK == 0) return out.fill_(-1);
    for (Tensor *t : {&qm, &km})
        if (!t->is_contiguous() || (uintptr_t)t->const_data_ptr() % 16) *t = contiguous_copy(*t);
    const size_t nb = sfast_hip_block_topk_workspace_bytes(&p);
    const Tensor ws = workspace(nb, qm);
    SFAST_RUN(sfast_hip_block_topk(qm.const_data_ptr<float>(), km.const_data_ptr<float>(), ints(len), out.data_ptr<int32_t>(), &p, ptr(ws), nb, call.stream),
              "sfast_hip_block_topk");
    return out;
}

// ---- attention over chosen blocks ---------------------------------------------------------------------------------------------------------
struct Attention {
    sfast_block_attn_params p{};
    Tensor blocks, klen, qlen;
    Attention(const char *who, const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &lists, int64_t block_q, int64_t block_k,
              const optional<Tensor> &key_lengths, const optional<Tensor> &query_lengths, optional<double> scale) {
        same_device(who, q, k);
        same_device(who, q, v);
        same_device(who, q, lists);
        TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, who, ": expected [B, S, H, D] tensors");
        TORCH_CHECK(k.size(0) == q.size(0) && k.size(3) == q.size(3) && v.sizes() == k.sizes() && k.size(2) > 0 && q.size(2) % k.size(2) == 0 &&
                        k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
                    who, ": query ", q.sizes(), " ", q.scalar_type(), ", key ", k.sizes(), " ", k.scalar_type(), ", value ", v.sizes(), " ", v.scalar_type(),
                    " do not fit");
        p.dtype = dtype_of(who, q);
        TORCH_CHECK(p.dtype != SFAST_F32, who, ": f16 / bf16 only");
        const int64_t D = q.size(3);
        TORCH_CHECK(D % 8 == 0 && D >= 8 && D <= 128, who, ": head dim ", D, " (a multiple of 8 up to 128)");
        TORCH_CHECK((block_q == 64 || block_q == 128) && (block_k == 64 || block_k == 128), who, ": blocks of 64 or 128 rows, got ", block_q, " and ", block_k);
        p.B = i32(who, q.size(0)), p.Sq = i32(who, q.size(1)), p.H = i32(who, q.size(2)), p.D = (int32_t)D;
        p.Sk = i32(who, k.size(1)), p.Hk = i32(who, k.size(2)), p.block_q = (int32_t)block_q, p.block_k = (int32_t)block_k;
        TORCH_CHECK(lists.scalar_type() == at::kInt && lists.dim() == 4 && lists.size(0) == p.B && lists.size(1) == p.Hk &&
                        lists.size(2) == (p.Sq + block_q - 1) / block_q,
                    who, ": blocks must be int32 [", p.B, ", ", p.Hk, ", ", (p.Sq + block_q - 1) / block_q, ", topk], got ", lists.scalar_type(), " ", lists.sizes());
        p.topk = i32(who, lists.size(3));
        p.scale = (float)(scale ? *scale : 1.0 / std::sqrt((double)D));
        TORCH_CHECK(p.scale >= 0x1p-100f && std::isfinite(p.scale), who, ": the scale must be positive (2^-100 and more) and finite, got ", p.scale);
        blocks = lists.contiguous();
        klen = lengths_of(who, "key_lengths", key_lengths, p.B, p.Sk, q);
        qlen = lengths_of(who, "query_lengths", query_lengths, p.B, p.Sq, q);
    }
};

// The kernels read 16-byte runs of a row: head-dim stride 1, other strides multiples of 8, an aligned address, rows that do not overlap and
// are less than 2^23 elements apart. Anything else is copied.
Tensor rows16(const Tensor &t) {
    const bool ok = t.stride(3) == 1 && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 && t.stride(2) % 8 == 0 && (uintptr_t)t.const_data_ptr() % 16 == 0 &&
                    t.stride(1) >= t.size(3) && t.stride(1) < (1 << 23);
    return ok ? t : contiguous_copy(t);
}

// out, lse and, where asked for, what the rounding of out left behind (backward sums out * dout without that rounding's error)
std::tuple<Tensor, Tensor, Tensor> attend(const Tensor &query, const Tensor &key, const Tensor &value, const Tensor &lists, int64_t block_q, int64_t block_k,
                                          const optional<Tensor> &key_lengths, const optional<Tensor> &query_lengths, optional<double> scale, bool want_rest) {
    const char *who = "block_sparse_attention";
    const Call call(who, query);
    Attention a(who, query, key, value, lists, block_q, block_k, key_lengths, query_lengths, scale);
    Tensor out = at::empty(query.sizes(), query.options()), lse = at::empty({a.p.B, a.p.H, a.p.Sq}, query.options().dtype(at::kFloat)), rest;
    if (want_rest) rest = at::empty(query.sizes(), query.options());
    if (out.numel() == 0) return {out, lse, rest};
    if (a.p.Sk == 0 || a.p.topk == 0) {
        if (want_rest) rest.zero_();
        return {out.zero_(), lse.fill_(-std::numeric_limits<double>::infinity()), rest};
    }
    const Tensor q = rows16(query), k = rows16(key), v = rows16(value);
    strides(q, a.p.qs), strides(k, a.p.ks), strides(v, a.p.vs), strides(out, a.p.os);
    const size_t nb = sfast_hip_block_attention_workspace_bytes(&a.p);
    const Tensor ws = workspace(nb, q);
    SFAST_RUN(sfast_hip_block_attention(q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), a.blocks.const_data_ptr<int32_t>(), ints(a.klen),
                                        ints(a.qlen), out.data_ptr(), lse.data_ptr<float>(), ptr(rest), &a.p, ptr(ws), nb, call.stream),
              "sfast_hip_block_attention");
    return {out, lse, rest};
}

std::tuple<Tensor, Tensor> block_sparse_attention(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &blocks, int64_t block_q, int64_t block_k,
                                                  const optional<Tensor> &key_lengths, const optional<Tensor> &query_lengths, optional<double> scale) {
    auto [out, lse, rest] = attend(q, k, v, blocks, block_q, block_k, key_lengths, query_lengths, scale, false);
    return {out, lse};
}

std::tuple<Tensor, Tensor, Tensor> block_sparse_attention_backward(const Tensor &grad_out, const optional<Tensor> &grad_lse_, const Tensor &query,
                                                                   const Tensor &key, const Tensor &value, const Tensor &lists, const Tensor &out_,
                                                                   const Tensor &lse_, int64_t block_q, int64_t block_k, const optional<Tensor> &key_lengths,
                                                                   const optional<Tensor> &query_lengths, optional<double> scale,
                                                                   const optional<Tensor> &out_rest) {
    const char *who = "block_sparse_attention_backward";
    const Call call(who, query);
    Attention a(who, query, key, value, lists, block_q, block_k, key_lengths, query_lengths, scale);
    Tensor grad_lse = grad_lse_ ? *grad_lse_ : Tensor(), rest = out_rest ? *out_rest : Tensor();
    for (const Tensor *t : std::initializer_list<const Tensor *>{&grad_out, &out_, &rest}) {
        same_device(who, query, *t);
        TORCH_CHECK(!t->defined() || (t->sizes() == query.sizes() && t->scalar_type() == query.scalar_type()), who,
                    ": out, what its rounding left and its gradient must be like the query");
    }
    for (const Tensor *t : std::initializer_list<const Tensor *>{&lse_, &grad_lse}) {
        same_device(who, query, *t);
        TORCH_CHECK(!t->defined() || (t->scalar_type() == at::kFloat && t->dim() == 3 && t->size(0) == a.p.B && t->size(1) == a.p.H && t->size(2) == a.p.Sq), who,
                    ": lse and its gradient must be fp32 [", a.p.B, ", ", a.p.H, ", ", a.p.Sq, "]");
    }
    Tensor dq = at::empty(query.sizes(), query.options()), dk = at::empty(key.sizes(), key.options()), dv = at::empty(value.sizes(), value.options());
    if (dq.numel() == 0 || dk.numel() == 0 || a.p.topk == 0) return {dq.zero_(), dk.zero_(), dv.zero_()};
    const Tensor q = rows16(query), k = rows16(key), v = rows16(value), go = rows16(grad_out), lse = lse_.contiguous();
    // out and its rest share their strides
    Tensor out = rows16(out_);
    if (rest.defined() && (rest.strides() != out.strides() || (uintptr_t)rest.const_data_ptr() % 16)) out = contiguous_copy(out_), rest = contiguous_copy(rest);
    if (grad_lse.defined()) grad_lse = grad_lse.contiguous();
    strides(q, a.p.qs), strides(k, a.p.ks), strides(v, a.p.vs), strides(out, a.p.os), strides(go, a.p.dos);
    strides(dq, a.p.dqs), strides(dk, a.p.dks), strides(dv, a.p.dvs);
    const size_t nb = sfast_hip_block_attention_backward_workspace_bytes(&a.p);
    const Tensor ws = workspace(nb, q);
    SFAST_RUN(sfast_hip_block_attention_backward(q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), a.blocks.const_data_ptr<int32_t>(), ints(a.klen),
                                                 ints(a.qlen), out.const_data_ptr(), ptr(rest), lse.const_data_ptr<float>(), go.const_data_ptr(),
                                                 grad_lse.defined() ? grad_lse.const_data_ptr<float>() : nullptr, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                                                 &a.p, ptr(ws), nb, call.stream),
              "sfast_hip_block_attention_backward");
    return {dq, dk, dv};
}

struct BlockSparse : torch::autograd::Function<BlockSparse> {
    static variable_list forward(AutogradContext *ctx, const Variable &q, const Variable &k, const Variable &v, const Variable &blocks, int64_t block_q,
                                 int64_t block_k, const optional<Variable> &key_lengths, const optional<Variable> &query_lengths, optional<double> scale) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto [out, lse, rest] = attend(q, k, v, blocks, block_q, block_k, key_lengths, query_lengths, scale, true);
        ctx->save_for_backward({q, k, v, blocks, key_lengths ? *key_lengths : Tensor(), query_lengths ? *query_lengths : Tensor(), out, lse, rest});
        ctx->saved_data["block_q"] = block_q;
        ctx->saved_data["block_k"] = block_k;
        ctx->saved_data["scale"] = scale;
        ctx->set_materialize_grads(false);
        return {out, lse};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list result(9);
        if (!grads[0].defined() && !grads[1].defined()) return result;
        TORCH_CHECK(!at::GradMode::is_enabled(), "block_sparse_attention: there is no second derivative (create_graph)");
        const auto s = ctx->get_saved_variables();
        const auto some = [](const Tensor &t) { return t.defined() ? optional<Tensor>(t) : c10::nullopt; };
        const auto scale = ctx->saved_data["scale"];
        auto [dq, dk, dv] = block_sparse_attention_backward(grads[0].defined() ? grads[0] : at::zeros_like(s[6]), some(grads[1]), s[0], s[1], s[2], s[3], s[6],
                                                            s[7], ctx->saved_data["block_q"].toInt(), ctx->saved_data["block_k"].toInt(), some(s[4]), some(s[5]),
                                                            scale.isNone() ? c10::nullopt : optional<double>(scale.toDouble()), some(s[8]));
        result[0] = dq, result[1] = dk, result[2] = dv;
        return result;
    }
};

std::tuple<Tensor, Tensor> block_sparse_attention_autograd(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &blocks, int64_t block_q,
                                                           int64_t block_k, const optional<Tensor> &key_lengths, const optional<Tensor> &query_lengths,
                                                           optional<double> scale) {
    no_tangents("block_sparse_attention", {&q, &k, &v});
    if (!wants_grad({&q, &k, &v})) {
        at::AutoDispatchBelowADInplaceOrView below;
        return block_sparse_attention(q, k, v, blocks, block_q, block_k, key_lengths, query_lengths, scale);
    }
    auto r = BlockSparse::apply(q, k, v, blocks, block_q, block_k, key_lengths, query_lengths, scale);
    return {r[0], r[1]};
}

// gradients computed by the call itself: whoever differentiates them is told
struct BlockSparseBackward : torch::autograd::Function<BlockSparseBackward> {
    static variable_list forward(AutogradContext *, const Variable &grad_out, const optional<Variable> &grad_lse, const Variable &q, const Variable &k,
                                 const Variable &v, const Variable &blocks, const Variable &out, const Variable &lse, int64_t block_q, int64_t block_k,
                                 const optional<Variable> &key_lengths, const optional<Variable> &query_lengths, optional<double> scale,
                                 const optional<Variable> &out_rest) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto [dq, dk, dv] = block_sparse_attention_backward(grad_out, grad_lse, q, k, v, blocks, out, lse, block_q, block_k, key_lengths, query_lengths, scale, out_rest);
        return {dq, dk, dv};
    }
    static variable_list backward(AutogradContext *, variable_list) {
        TORCH_CHECK(false, "block_sparse_attention_backward: there is no second derivative");
    }
};

std::tuple<Tensor, Tensor, Tensor> block_sparse_attention_backward_autograd(const Tensor &grad_out, const optional<Tensor> &grad_lse, const Tensor &q,
                                                                            const Tensor &k, const Tensor &v, const Tensor &blocks, const Tensor &out,
                                                                            const Tensor &lse, int64_t block_q, int64_t block_k,
                                                                            const optional<Tensor> &key_lengths, const optional<Tensor> &query_lengths,
                                                                            optional<double> scale, const optional<Tensor> &out_rest) {
    const Tensor gl = grad_lse ? *grad_lse : Tensor(), rest = out_rest ? *out_rest : Tensor();
    no_tangents("block_sparse_attention_backward", {&grad_out, &gl, &q, &k, &v, &out, &lse, &rest});
    if (!wants_grad({&grad_out, &gl, &q, &k, &v, &out, &lse, &rest})) {
        at::AutoDispatchBelowADInplaceOrView below;
        return block_sparse_attention_backward(grad_out, grad_lse, q, k, v, blocks, out, lse, block_q, block_k, key_lengths, query_lengths, scale, out_rest);
    }
    auto r = BlockSparseBackward::apply(grad_out, grad_lse, q, k, v, blocks, out, lse, block_q, block_k, key_lengths, query_lengths, scale, out_rest);
    return {r[0], r[1], r[2]};
}

// the choice takes no gradient: its means are those of the values
Tensor block_means_autograd(const Tensor &input, int64_t block, const optional<Tensor> &lengths) {
    no_tangents("block_means", {&input});
    at::AutoDispatchBelowADInplaceOrView below;
    return block_means(input.detach(), block, lengths);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(sfast, m) {
    m.def("rotary_embedding_nd(Tensor query, Tensor? key, Tensor positions, int[] sections, float theta=10000.0, bool interleaved=True, bool inverse=False) "
          "-> (Tensor, Tensor)");
}
TORCH_LIBRARY_IMPL(sfast, CUDA, m) { m.impl("rotary_embedding_nd", rotary); }
TORCH_LIBRARY_IMPL(sfast, AutogradCUDA, m) { m.impl("rotary_embedding_nd", rotary_autograd); }

TORCH_LIBRARY_FRAGMENT(sfast_xformers, m) {
    m.def("block_means(Tensor input, int block, Tensor? lengths=None) -> Tensor");
    m.def("block_topk(Tensor query_means, Tensor key_means, int topk, int block_k=64, Tensor? key_lengths=None) -> Tensor");
    m.def("block_sparse_attention(Tensor query, Tensor key, Tensor value, Tensor blocks, int block_q=128, int block_k=64, Tensor? key_lengths=None, "
          "Tensor? query_lengths=None, float? scale=None) -> (Tensor, Tensor)");
    m.def("block_sparse_attention_backward(Tensor grad_out, Tensor? grad_lse, Tensor query, Tensor key, Tensor value, Tensor blocks, Tensor out, Tensor lse, "
          "int block_q=128, int block_k=64, Tensor? key_lengths=None, Tensor? query_lengths=None, float? scale=None, Tensor? out_rest=None) "
          "-> (Tensor, Tensor, Tensor)");
}
TORCH_LIBRARY_IMPL(sfast_xformers, CUDA, m) {
    m.impl("block_means", block_means);
    m.impl("block_topk", block_topk);
    m.impl("block_sparse_attention", block_sparse_attention);
    m.impl("block_sparse_attention_backward", block_sparse_attention_backward);
}
TORCH_LIBRARY_IMPL(sfast_xformers, AutogradCUDA, m) {
    m.impl("block_means", block_means_autograd);
    m.impl("block_sparse_attention", block_sparse_attention_autograd);
    m.impl("block_sparse_attention_backward", block_sparse_attention_backward_autograd);
}
