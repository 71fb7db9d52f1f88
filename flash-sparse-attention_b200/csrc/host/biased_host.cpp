// Attention with changed scores (capped, biased by distance) and masks: checks, workspaces, launches and the autograd function.
#include "host_common.h"

#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>

#include <cmath>
#include <optional>

namespace fsa_host {

using MaybeTensor = std::optional<Tensor>;

// A tensor [N, H, D] as the kernels take it: rows of D in one piece, strides that tensor maps can hold.  (The stride of a dimension of one
// entry means nothing and may be any number.)
struct Rows3 {
    Tensor t;
    int64_t sn, sh;
    Rows3(const Tensor& x, bool packed) : t(x) {
        const int64_t H = x.size(1), D = x.size(2);
        auto strides = [&] {
            sh = t.size(1) == 1 ? D : t.stride(1);
            sn = t.size(0) <= 1 ? sh * H : t.stride(0);
        };
        strides();
        const bool ok = x.stride(2) == 1 && sn % 8 == 0 && sh % 8 == 0 && sn >= D && sh >= D && ((uintptr_t)x.data_ptr() & 15) == 0 &&
                        (!packed || (sh == D && sn >= H * D));
        if (!ok) {
            t = x.contiguous();
            if (((uintptr_t)t.data_ptr() & 15) != 0) t = t.clone(at::MemoryFormat::Contiguous);
            strides();
        }
    }
};

struct BiasedArgs {
    Tensor cu_q, cu_k, slopes, docs, prefix;
    double scale, cap;
    int64_t window;         // -1: none
};

static void check_biased_status(const char* what) {
    if (!checking_status()) return;
    int st = 0;
    check(fsa_biased_read_status(&st), what);
    check(st == 0 ? FSA_OK : FSA_ERR_DEVICE_STATUS, what);
}

// Gradients of a leaf are added up on the stream that its first live graph was made on.  Where that is another than the capturing one, torch ends the capture, and the
// process with it, in the backward pass: refused here, before anything is captured.
static void check_capture(const Tensor& q, const Tensor& k, const Tensor& v) {
    const auto stream = c10::cuda::getCurrentCUDAStream(q.device().index());
    cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(stream.stream(), &capturing) != cudaSuccess || capturing == cudaStreamCaptureStatusNone) return;
    for (const Tensor* t : {&q, &k, &v}) {
        if (!t->requires_grad() || !t->is_leaf()) continue;
        const auto sum = torch::autograd::impl::try_get_grad_accumulator(*t);
        const auto on = sum ? sum->stream() : std::nullopt;
        TORCH_CHECK(!on || *on == stream.unwrap(), "biased_attention: a graph made on another stream still holds a leaf of this capture: release what depends on it first");
    }
}

static void check_lengths(const Tensor& t, const Tensor& q, int64_t n, const char* name) {
    TORCH_CHECK_TYPE(t.scalar_type() == at::kInt, name, " has to be int32, got ", t.scalar_type());
    TORCH_CHECK_VALUE(t.dim() == 1 && (n < 0 || t.size(0) == n), name, " has to have ", n, " entries, got a tensor of shape ", t.sizes());
    TORCH_CHECK_VALUE(t.device() == q.device(), name, " is on ", t.device(), ", q on ", q.device());
}

// Forward-mode tangents would be lost where no gradient is asked for (autograd refuses them itself where one is).
static void check_no_tangents(const char* what, std::initializer_list<const Tensor*> ts) {
    for (const Tensor* t : ts)
        TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), what, " has no forward-mode derivative: give tensors without tangents");
}

static Tensor check_slopes(const MaybeTensor& s, const Tensor& q) {
    if (!s) return Tensor();
    TORCH_CHECK_TYPE(s->scalar_type() == at::kFloat, "alibi_slopes has to be float32, got ", s->scalar_type());
    TORCH_CHECK_VALUE(s->dim() == 1 && s->size(0) == q.size(1), "alibi_slopes has to have one entry for each of the ", q.size(1), " query heads, got ", s->sizes());
    TORCH_CHECK_VALUE(s->device() == q.device(), "alibi_slopes is on ", s->device(), ", q on ", q.device());
    TORCH_CHECK_VALUE(!s->requires_grad(), "alibi_slopes has no gradient here: give slopes that need none");
    check_no_tangents("alibi_slopes", {&*s});
    return s->contiguous();
}

static void check_scores(const Tensor& q, double scale, double cap) {
    const float log2 = (float)scale * 1.44269504f;         // (as the kernels take it)
    TORCH_CHECK_VALUE(scale > 0 && std::isfinite(scale) && std::isnormal(log2), "sm_scale has to be above 0 and finite, in 32 bits too, got ", scale);
    TORCH_CHECK_VALUE(cap >= 0 && std::isfinite(cap), "softcap has to be above 0 and finite (or None), got ", cap);
    TORCH_CHECK_VALUE(cap == 0 || (cap > 1e-30 && cap < 1e30 && scale / cap > 1e-30 && scale / cap < 1e30),
                      "softcap and sm_scale / softcap have to be between 1e-30 and 1e30, got ", cap, " and ", scale / cap);
    TORCH_CHECK_VALUE(q.is_cuda(), "the sm_100a kernels need CUDA tensors (no CPU fallback)");
}

static void check_qkv(const Tensor& q, const Tensor& k, const Tensor& v) {
    dtype_code(q);
    TORCH_CHECK_TYPE(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), "q, k and v have to be of one type");
    TORCH_CHECK_VALUE(q.dim() == 3 && k.dim() == 3 && v.dim() == 3, "q, k and v have to have three dimensions (rows, heads, head size)");
    TORCH_CHECK_VALUE(k.sizes() == v.sizes(), "k and v have to be of one shape, got ", k.sizes(), " and ", v.sizes());
    TORCH_CHECK_VALUE(k.size(2) == q.size(2) && k.size(1) > 0 && q.size(1) % k.size(1) == 0 && q.size(1) > 0,
                      "q heads have to be a multiple of the k heads, of one head size: got ", q.sizes(), " and ", k.sizes());
    TORCH_CHECK_VALUE(k.device() == q.device() && v.device() == q.device(), "q, k and v have to be on one device");
    TORCH_CHECK_VALUE(q.size(2) == 64 || q.size(2) == 128, "head size 64 or 128 expected, got ", q.size(2));
    TORCH_CHECK_VALUE(q.size(1) / k.size(1) <= 32, "up to 32 query heads a k head, got ", q.size(1) / k.size(1));
}

static std::tuple<Tensor, Tensor, Tensor> biased_fwd(const Tensor& q_, const Tensor& k_, const Tensor& v_, const BiasedArgs& a) {
    c10::cuda::CUDAGuard guard(q_.device());
    const int64_t N = q_.size(0), Hq = q_.size(1), D = q_.size(2), Nk = k_.size(0), Hk = k_.size(1);
    int64_t nb = 0;
    check(fsa_biased_attn_limits_bytes(N, &nb), "fsa_biased_attn_limits_bytes");
    Tensor limits = bytes(nb, q_);
    if (N == 0 || Nk == 0)          // nobody sees anything
        return {at::zeros({N, Hq, D}, q_.options().requires_grad(false)),
                at::full({Hq, N}, -INFINITY, q_.options().dtype(at::kFloat).requires_grad(false)), limits};
    const Rows3 q(q_, false), k(k_, true), v(v_, true);
    Tensor o = fresh({N, Hq, D}, q_), lse = f32({Hq, N}, q_), scratch;
    const int B = (int)a.cu_q.size(0) - 1;
    check(fsa_biased_attn_fwd_bytes(N, Nk, B, (int)Hq, (int)Hk, (int)D, (int)a.window, &nb), "fsa_biased_attn_fwd_bytes");
    if (nb > 0) scratch = bytes(nb, q_);
    check(fsa_biased_attn_fwd(ptr(q.t), ptr(k.t), ptr(v.t), iptr(a.cu_q), iptr(a.cu_k), iptr(a.docs), iptr(a.prefix),
                              a.slopes.defined() ? a.slopes.data_ptr<float>() : nullptr, N, Nk, B, (int)Hq, (int)Hk, (int)D,
                              dtype_code(q_), q.sn, q.sh, k.sn, v.sn, (float)a.scale, (float)a.cap, (int)a.window, ptr(o), lse.data_ptr<float>(), ptr(limits),
                              limits.numel(), ptr(scratch), nb, stream_of(q_)),
          "fsa_biased_attn_fwd");
    check_biased_status("fsa_biased_attn_fwd status");
    return {o, lse, limits};
}

static std::tuple<Tensor, Tensor, Tensor> biased_bwd(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& o, const Tensor& lse, const Tensor& do_,
                                                     const Tensor& limits, const BiasedArgs& a) {
    c10::cuda::CUDAGuard guard(q_.device());
    const int64_t N = q_.size(0), Hq = q_.size(1), D = q_.size(2), Nk = k_.size(0), Hk = k_.size(1);
    if (N == 0 || Nk == 0) {
        auto zeros = [](const Tensor& x) { return at::zeros(x.sizes(), x.options().requires_grad(false)); };
        return {zeros(q_), zeros(k_), zeros(v_)};
    }
    const Rows3 q(q_, false), k(k_, true), v(v_, true), dout(do_, false);
    int64_t nb = 0;
    const int B = (int)a.cu_q.size(0) - 1;
    check(fsa_biased_attn_bwd_bytes(N, Nk, B, (int)Hq, (int)Hk, (int)D, (int)a.window, &nb), "fsa_biased_attn_bwd_bytes");
    const Tensor scratch = bytes(nb, q_);
    Tensor dq = fresh({N, Hq, D}, q_), dk = fresh({Nk, Hk, D}, q_), dv = fresh_like(dk);
    check(fsa_biased_attn_bwd(ptr(q.t), ptr(k.t), ptr(v.t), ptr(o), lse.data_ptr<float>(), ptr(dout.t), iptr(a.cu_q), iptr(a.cu_k), iptr(a.docs),
                              iptr(a.prefix), a.slopes.defined() ? a.slopes.data_ptr<float>() : nullptr, N, Nk, B, (int)Hq, (int)Hk, (int)D,
                              dtype_code(q_), q.sn, q.sh, k.sn, v.sn, dout.sn, dout.sh, (float)a.scale, (float)a.cap, (int)a.window, ptr(dq), ptr(dk), ptr(dv), ptr(limits),
                              limits.numel(), ptr(scratch), scratch.numel(), stream_of(q_)),
          "fsa_biased_attn_bwd");
    check_biased_status("fsa_biased_attn_bwd status");
    return {dq, dk, dv};
}

struct BiasedAttention : torch::autograd::Function<BiasedAttention> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const BiasedArgs& a) {
        auto [o, lse, limits] = biased_fwd(q, k, v, a);
        ctx->save_for_backward({q, k, v, o, lse, limits, a.cu_q, a.cu_k, a.slopes, a.docs, a.prefix});
        ctx->saved_data["scale"] = a.scale;
        ctx->saved_data["cap"] = a.cap;
        ctx->saved_data["window"] = a.window;
        ctx->mark_non_differentiable({lse});
        return {o, lse};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
        const auto t = ctx->get_saved_variables();
        const bool again = at::GradMode::is_enabled();          // (create_graph)
        at::NoGradGuard plain;
        auto [dq, dk, dv] = biased_bwd(t[0], t[1], t[2], t[3], t[4], g[0], t[5],
                                       {t[6], t[7], t[8], t[9], t[10], ctx->saved_data["scale"].toDouble(), ctx->saved_data["cap"].toDouble(),
                                        ctx->saved_data["window"].toInt()});
        if (!again) return {dq, dk, dv, Tensor()};
        // Their own derivative is not there: whoever asks for it, on the way to what they are made of, is told so instead of getting a gradient that lacks it.
        const auto none = std::make_shared<torch::autograd::Error>("biased_attention has no second derivative",
                                                                   torch::autograd::collect_next_edges(t[0], t[1], t[2], g[0]));
        for (const Tensor& x : {dq, dk, dv}) torch::autograd::set_history(x, none);
        return {dq, dk, dv, Tensor()};
    }
};

std::tuple<Tensor, Tensor> biased_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu_q, const MaybeTensor& cu_k_, const MaybeTensor& slopes_,
                                            const MaybeTensor& docs_, const MaybeTensor& prefix_, double scale, double cap, int64_t window) {
    check_qkv(q, k, v);
    check_no_tangents("biased_attention", {&q, &k, &v});
    TORCH_CHECK_VALUE(cu_q.dim() == 1 && cu_q.size(0) >= 2, "cu_seqlens has to have an entry more than there are sequences, and there is one at least");
    const int64_t B = cu_q.size(0) - 1;
    check_lengths(cu_q, q, -1, "cu_seqlens");
    if (cu_k_) check_lengths(*cu_k_, q, B + 1, "cu_seqlens_k");
    else TORCH_CHECK_VALUE(q.size(0) == k.size(0), "q and k have to have as many rows (or give cu_seqlens_k), got ", q.size(0), " and ", k.size(0));
    if (docs_) check_lengths(*docs_, q, k.size(0), "doc_ids");
    if (prefix_) check_lengths(*prefix_, q, B, "prefix_lens");
    TORCH_CHECK_VALUE(!(prefix_ && (docs_ || window >= 0)), "prefix_lens cannot be given with doc_ids or window_size");
    TORCH_CHECK_VALUE(window >= -1 && window <= INT32_MAX, "window_size has to be 0 or more (or None)");
    const Tensor slopes = check_slopes(slopes_, q);
    check_scores(q, scale, cap);
    auto plain = [](const MaybeTensor& t) { return t ? t->contiguous() : Tensor(); };
    const Tensor cu = cu_q.contiguous(), cu_k = cu_k_ ? cu_k_->contiguous() : cu, docs = plain(docs_), prefix = plain(prefix_);
    if (wants_grad({&q, &k, &v})) {
        check_capture(q, k, v);
        const auto r = BiasedAttention::apply(q, k, v, BiasedArgs{cu, cu_k, slopes, docs, prefix, scale, cap, window});
        return {r[0], r[1]};
    }
    auto [o, lse, limits] = biased_fwd(q, k, v, {cu, cu_k, slopes, docs, prefix, scale, cap, window});
    return {o, lse};
}

// A cache of rows [rows, Hk, D] as it is read in place.  (None is copied: a copy of the cache at every step would be slower than all the rest.)
static void check_cache(const Tensor& t, const char* name) {
    TORCH_CHECK_VALUE(t.stride(2) == 1 && (t.size(1) == 1 || t.stride(1) == t.size(2)) && (t.size(0) <= 1 || (t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1) * t.size(2))) &&
                          ((uintptr_t)t.data_ptr() & 15) == 0,
                      name, ": the heads of a row have to be adjacent, rows and memory aligned to 16 bytes; got strides ", t.strides());
}
static int64_t row_stride(const Tensor& t) { return t.size(0) <= 1 ? t.size(1) * t.size(2) : t.stride(0); }

std::tuple<Tensor, Tensor> biased_decode(const Tensor& q_, const Tensor& k, const Tensor& v, const Tensor& seq_len, const Tensor& row0, const MaybeTensor& pk,
                                         const MaybeTensor& pv, const MaybeTensor& cu_prefix, const MaybeTensor& cu_group, const MaybeTensor& slopes_, double scale,
                                         double cap, int64_t window, int64_t max_len, int64_t max_prefix) {
    check_qkv(q_, k, v);
    check_no_tangents("decode", {&q_, &k, &v});
    const int64_t B = q_.size(0), Hq = q_.size(1), D = q_.size(2), Hk = k.size(1);
    check_lengths(seq_len, q_, B, "seq_len");
    check_lengths(row0, q_, B, "seq_row0");
    int64_t groups = 0, prefix_rows = 0;
    if (pk) {
        check_qkv(q_, *pk, *pv);
        check_no_tangents("decode", {&*pk, &*pv});
        TORCH_CHECK_VALUE(pk->size(1) == Hk, "prefix_k has ", pk->size(1), " heads, k ", Hk);
        TORCH_CHECK_VALUE(cu_prefix->dim() == 1 && cu_prefix->size(0) >= 2, "cu_prefix has to have an entry more than there are prefixes, and there is one at least");
        groups = cu_prefix->size(0) - 1;
        check_lengths(*cu_prefix, q_, groups + 1, "cu_prefix");
        check_lengths(*cu_group, q_, groups + 1, "cu_group");
        prefix_rows = pk->size(0);
    }
    TORCH_CHECK_VALUE(window >= -1 && window <= INT32_MAX, "window_size has to be 0 or more (or None)");
    TORCH_CHECK_VALUE(max_len >= 0 && max_prefix >= 0, "max_len and max_prefix have to be 0 or more");
    const Tensor slopes = check_slopes(slopes_, q_);
    check_scores(q_, scale, cap);
    check_cache(k, "k");
    check_cache(v, "v");
    if (pk) {
        check_cache(*pk, "prefix_k");
        check_cache(*pv, "prefix_v");
    }
    c10::cuda::CUDAGuard guard(q_.device());
    Tensor q = q_.contiguous();
    if (((uintptr_t)q.data_ptr() & 15) != 0) q = q.clone(at::MemoryFormat::Contiguous);
    if (B == 0) return {fresh({B, Hq, D}, q), f32({B, Hq}, q)};
    TORCH_CHECK_VALUE(k.size(0) > 0, "the cache has no rows");
    int64_t nb = 0;
    check(fsa_biased_decode_bytes((int)B, (int)Hq, (int)Hk, (int)D, (int)groups, max_len, max_prefix, (int)window, &nb), "fsa_biased_decode_bytes");
    const Tensor scratch = bytes(nb, q), lens = seq_len.contiguous(), rows = row0.contiguous(), cp = cu_prefix ? cu_prefix->contiguous() : Tensor(),
                 cg = cu_group ? cu_group->contiguous() : Tensor();
    Tensor o = fresh({B, Hq, D}, q), lse = f32({B, Hq}, q);
    check(fsa_biased_decode(ptr(q), ptr(k), ptr(v), k.size(0), row_stride(k), row_stride(v), iptr(lens), iptr(rows), pk ? ptr(*pk) : nullptr, pk ? ptr(*pv) : nullptr,
                            prefix_rows, pk ? row_stride(*pk) : 0, pk ? row_stride(*pv) : 0, iptr(cp), iptr(cg), (int)groups,
                            slopes.defined() ? slopes.data_ptr<float>() : nullptr, (int)B, (int)Hq, (int)Hk, (int)D, dtype_code(q), (float)scale, (float)cap,
                            (int)window, max_len, max_prefix, ptr(o), lse.data_ptr<float>(), ptr(scratch), scratch.numel(), stream_of(q)),
          "fsa_biased_decode");
    check_biased_status("fsa_biased_decode status");
    return {o, lse};
}

void bind_biased(pybind11::module& m) {
    m.def("biased_attention", &biased_attention);
    m.def("biased_decode", &biased_decode);
}

}  // namespace fsa_host
