// Torch bindings of attention_ext.hip and gated_norm.hip: every shape, type, stride, device and size that the kernels assume
// is checked here (a faulting kernel can take the whole node down), outputs and workspaces come from the caching allocator,
// launches go to the current stream of the operands' device.
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <cmath>
#include <initializer_list>
#include <limits>
#include <unordered_set>

#include "../kernels/attention_ext.h"
#include "../kernels/gated_norm.h"
#include "binding.h"

namespace pdt {
namespace {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;

hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream(); }
bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

// The operators are differentiable calls with their nodes in C++: with Python functions a backward spent 20 to 50 us more on the
// interpreter (lock, unpacking of saved tensors), more than its kernels take on small inputs.  A call whose operands the kernels
// do not take (or that nobody should make) returns nothing: the Python side has the words for why.

// `t` with the numbers in memory that the tensor stands for (autograd hands out views that are negated when they are read, and zeros
// without memory)
Tensor written_out(const Tensor& t) {
    if (t._is_zerotensor()) return at::zeros(t.sizes(), t.options());
    return t.is_neg() ? t.resolve_neg() : t;
}
Tensor dense16(const Tensor& t) {  // contiguous and 16-B aligned, by a copy where it is not
    if (!t.defined()) return t;
    Tensor c = written_out(t).contiguous();
    return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone();
}
Tensor param32(const Tensor& t) { return t.defined() ? dense16(t.scalar_type() == at::kFloat ? t : t.to(at::kFloat)) : t; }
Tensor int32(const Tensor& t) {
    if (!t.defined() || t.scalar_type() == at::kInt) return dense16(t);
    return written_out(t).clamp(std::numeric_limits<int32_t>::min(), std::numeric_limits<int32_t>::max()).to(at::kInt);
}
bool is_index(const Tensor& t) { return t.scalar_type() == at::kInt || t.scalar_type() == at::kLong; }
OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
bool wants_grad(std::initializer_list<const Tensor*> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}
// The gradients of a node's backward pass under create_graph: constants whose own derivative raises.  (Only then: a model may have
// another term that does need second derivatives.)  The raising node hangs on all that the gradients depend on, the node's inputs
// and the gradients that came in, so that no way to ask for the derivative finds nothing to differentiate.
template <typename F>
torch::autograd::variable_list first_order(const char* op, const torch::autograd::variable_list& g, F&& backward) {
    if (!at::GradMode::is_enabled()) return backward();
    torch::autograd::variable_list r;
    {
        at::NoGradGuard no_grad;
        r = backward();
    }
    torch::autograd::edge_list edges;
    if (const auto node = torch::autograd::get_current_node())
        for (const auto& e : node->next_edges())
            if (e.is_valid()) edges.push_back(e);
    for (const Tensor& t : g)
        if (t.defined() && t.requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(t));
    const auto raise = std::make_shared<torch::autograd::Error>(std::string(op) + ": the backward pass cannot be differentiated again",
                                                                std::move(edges));
    for (Tensor& t : r) {
        if (!t.defined()) continue;
        if (t.is_view()) t = t.clone();  // (a history of its own)
        torch::autograd::set_history(t, raise);
    }
    return r;
}

// A tracer, and a mode whose tensors are proxies, fakes or wrappers, sees only the allocation of the outputs: what it records
// would return memory that nobody has written.  Other modes (counters of operations and the like) may be on.
bool is_recording() {
    using Mode = c10::impl::TorchDispatchModeKey;
    if (torch::jit::tracer::isTracing() || c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch)) return true;
    if (!c10::impl::TorchDispatchModeTLS::any_modes_set()) return false;
    for (Mode m : {Mode::FAKE, Mode::PROXY, Mode::FUNCTIONAL})
        if (c10::impl::TorchDispatchModeTLS::get_mode(m).has_value()) return true;
    return false;
}
// The kernels are called at once, outside the dispatcher: what autograd and the transforms have beyond a backward pass would be
// lost without a word.  A tensor with a tangent (forward-mode derivatives) does not require a gradient, so that a node alone would
// not see it; a tensor of a transform or a wrapper may say that it is on the GPU and have no memory there.
void check_plain(const char* op, std::initializer_list<const Tensor*> ts) {
    TORCH_CHECK(!is_recording(), op, ": cannot be traced, exported or run on fake tensors (its kernels are called outside the dispatcher)");
    for (const Tensor* t : ts) {
        if (!t->defined()) continue;
        TORCH_CHECK(!t->_fw_grad(/*level=*/0).defined(), op, ": no forward-mode derivative, only a backward pass");
        TORCH_CHECK(t->has_storage() && (t->numel() == 0 || t->_is_zerotensor() || t->const_data_ptr()), op,
                    ": expected tensors with memory of their own (no vmap, no torch.func, no wrappers)");
    }
}

// The engine hands a gradient to the stream on which the tensor's own node was made.  Where that is a node of an eager graph (an
// input computed before the capture, or a leaf of a graph that lives), a captured backward pass would leave the capture, and the
// process ends.  Refused at the forward, for the inputs and for all that they were computed from within the capture.
bool outside_capture(torch::autograd::Node& node) {
    const auto stream = node.stream();
    if (!stream) return false;
    const hipStream_t s = c10::hip::HIPStreamMasqueradingAsCUDA(c10::hip::HIPStreamMasqueradingAsCUDA::UNCHECKED, *stream).stream();
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (s) (void)hipStreamIsCapturing(s, &status);
    return status != hipStreamCaptureStatusActive;
}
void check_capture(std::initializer_list<const Tensor*> inputs) {
    using torch::autograd::Node;
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    std::vector<std::shared_ptr<Node>> todo;
    std::unordered_set<const Node*> seen;
    auto visit = [&](std::shared_ptr<Node> n) {
        if (n && seen.insert(n.get()).second) todo.push_back(std::move(n));
    };
    for (const Tensor* t : inputs)
        if (t->defined() && t->requires_grad()) visit(t->is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(*t) : t->grad_fn());
    while (!todo.empty()) {
        const std::shared_ptr<Node> n = std::move(todo.back());
        todo.pop_back();
        TORCH_CHECK(!outside_capture(*n),
                    "a forward pass with gradients is being captured while an eager graph of the same parameters or inputs lives on "
                    "another stream: release that graph's outputs first, or detach the inputs from it");
        for (const auto& e : n->next_edges()) visit(e.function);
    }
}

void check_same_device(const Tensor& t, const Tensor& like, const char* name) {
    TORCH_CHECK(t.device() == like.device(), name, ": expected on ", like.device(), ", got ", t.device());
}
// [B, rows, width] bf16 with contiguous, 16-B aligned, non-overlapping rows
void check_rows(const Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kBFloat16 && t.dim() == 3, name, ": expected a bf16 GPU tensor [B, rows, width]");
    TORCH_CHECK(t.numel() == 0 || (t.stride(2) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0), name,
                ": expected contiguous rows, 16-B aligned");
    TORCH_CHECK(t.size(1) < 2 || (t.stride(1) % 8 == 0 && t.stride(1) >= t.size(2) && t.stride(1) < (1L << 23)), name,
                ": row stride ", t.stride(1));
    TORCH_CHECK(t.size(0) < 2 || (t.stride(0) % 8 == 0 && t.stride(0) >= 0), name, ": batch stride ", t.stride(0));
}
// `t` where its rows are as check_rows wants them, else a copy
Tensor rows3(const Tensor& given) {
    const Tensor t = written_out(given);
    const bool ok = t.stride(2) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 &&
                    (t.size(1) < 2 || (t.stride(1) % 8 == 0 && t.stride(1) >= t.size(2) && t.stride(1) < (1L << 23))) &&
                    (t.size(0) < 2 || t.stride(0) % 8 == 0);
    return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}
bool lengths_fit(const OptTensor& lens, const Tensor& like) {
    return !given(lens) || (lens->dim() == 1 && lens->size(0) == like.size(0) && is_index(*lens) && lens->device() == like.device());
}
bool attention_dim_ok(int64_t width, int64_t parts) {
    if (parts < 1 || width % parts) return false;
    const int64_t hd = width / parts;
    return hd == 32 || hd == 64 || hd == 128;
}
void check_dense(const Tensor& t, at::IntArrayRef shape, at::ScalarType type, const Tensor& like, const char* name) {
    TORCH_CHECK(t.scalar_type() == type && t.is_contiguous() && t.sizes() == shape, name, ": expected contiguous ", type, " ", shape,
                ", got ", t.scalar_type(), " ", t.sizes());
    TORCH_CHECK(t.numel() == 0 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, name, ": data pointer must be 16-B aligned");
    check_same_device(t, like, name);
}
void check_codes(const Tensor& t, long S, const Tensor& like, const char* name) {
    TORCH_CHECK(is_index(t) && t.is_contiguous() && t.dim() == 1 && t.size(0) == S, name, ": expected ", S, " contiguous integers, got ",
                t.scalar_type(), " ", t.sizes());
    check_same_device(t, like, name);
}
ExtView view_of(const Tensor& t, int G) {
    return {t.size(0) < 2 ? 0 : (long)t.stride(0), t.size(1) < 2 ? (long)t.size(2) : (long)t.stride(1), make_fastdiv((uint32_t)G)};
}
const __bf16* bf16_ptr(const Tensor& t) { return static_cast<const __bf16*>(t.data_ptr()); }

// operands that forward and backward share; q [B,Sq,H*hd], k and v [B,Sk,Hkv*hd] with equal strides
ExtArgs ext_args(const Tensor& q, const Tensor& k, const Tensor& v, int64_t heads, int64_t kv_heads, const OptTensor& lens, int64_t hd,
                 bool self) {
    TORCH_CHECK(hd == 32 || hd == 64 || hd == 128, "attention: head_dim ", hd, " not supported (32, 64 or 128)");
    const long B = q.size(0), G = heads / kv_heads, M = q.size(1) * G;
    TORCH_CHECK(M < (1L << 30) && k.size(1) < (1L << 30) && B < (1L << 30), "attention: lengths below 2^30");
    ExtArgs a{};
    a.q = bf16_ptr(q); a.k = bf16_ptr(k); a.v = bf16_ptr(v);
    a.qv = view_of(q, (int)G); a.kv = view_of(k, 1);
    a.o = {(long)(q.size(1) * heads * hd), (long)(heads * hd), make_fastdiv((uint32_t)G)};
    TORCH_CHECK(a.o.rs < (1L << 23), "attention: width ", a.o.rs);
    if (given(lens)) {
        check_dense(*lens, {B}, at::kInt, q, "lengths");
        a.lens = lens->data_ptr<int>();
    }
    a.self = self;
    a.B = (int)B; a.Hkv = (int)kv_heads; a.G = (int)G; a.Sq = (int)q.size(1); a.Sk = (int)k.size(1);
    a.M = (int)M; a.Mp = (int)((M + 63) / 64 * 64);
    a.stat_n = B * kv_heads * a.Mp;
    a.scale = (float)(1.0 / std::sqrt((double)hd));
    a.c = (float)(1.4426950408889634 / std::sqrt((double)hd));
    return a;
}
// a launch has fewer than 2^32 threads: 2^24 workgroups of 256
void check_grid(const ExtArgs& a, const ExtPlan& p) {
    TORCH_CHECK((long)a.B * a.Hkv < (1L << 24) / std::max(1, p.tiles * p.splits), "attention: ", a.B, " sequences of ", a.Hkv,
                " key heads are more workgroups than a launch has (2^24)");
}
void set_tables(ExtArgs& a, const Tensor& tab, const Tensor& codes, int64_t R) {
    const long Sp = (a.Sk + 127) / 128 * 128, Rp = (R + 3) / 4 * 4;
    TORCH_CHECK(R >= 1 && R <= kExtMaxEntries, "rel_bias_attention: ", R, " entries (1 to ", kExtMaxEntries, ")");
    TORCH_CHECK(tab.sizes() == at::IntArrayRef({(long)a.Hkv, Rp}) && codes.sizes() == at::IntArrayRef({2 * Sp + Sp / 8}), "bias tables: shape");
    a.tab = tab.data_ptr<float>();
    a.q_codes4 = codes.data_ptr<int>();
    a.k_codes4 = codes.data_ptr<int>() + Sp;
    a.q_range = reinterpret_cast<const int2*>(codes.data_ptr<int>() + 2 * Sp);
    a.k_range = a.q_range + Sp / 32;
    a.R = (int)R; a.Rp = (int)Rp;
}

// -> out, stat (with `grad`)
std::tuple<Tensor, Tensor> ext_fwd(ExtArgs& a, const Tensor& q, int64_t heads, int64_t hd, bool grad) {
    Tensor out = at::empty({a.B, a.Sq, heads * hd}, q.options().memory_format(at::MemoryFormat::Contiguous)), stat;
    const auto f32 = q.options().dtype(at::kFloat);
    if (grad) stat = at::empty({2, (long)a.B * a.Hkv, a.Mp}, f32);
    if (out.numel() == 0) return {out, stat};
    const long BH = (long)a.B * a.Hkv;
    const ExtPlan p = ext_plan_fwd(BH, a.M, a.Sk, a.tab != nullptr);
    check_grid(a, p);
    Tensor part, ml;
    if (p.splits > 1) {
        part = at::empty({BH * p.splits * a.M * hd}, f32);
        ml = at::empty({BH * p.splits * a.M * 2}, f32);
    }
    launch_ext_fwd(a, p, (int)hd, out.data_ptr(), grad ? stat.data_ptr<float>() : nullptr,
                   part.defined() ? part.data_ptr<float>() : nullptr, ml.defined() ? ml.data_ptr<float>() : nullptr, stream_of(q));
    return {out, stat};
}

// dq / dk / dv: views to fill; -> dtable [NB, H] when bucket_of is given
Tensor ext_bwd(ExtArgs& a, const Tensor& q, int64_t heads, int64_t hd, const Tensor& dout, const Tensor& out, const Tensor& stat,
               Tensor dq, Tensor dk, Tensor dv, const OptTensor& bucket_of, int64_t NB) {
    const long width = heads * hd, BH = (long)a.B * a.Hkv;
    check_dense(dout, {a.B, a.Sq, width}, at::kBFloat16, q, "dout");
    check_dense(out, {a.B, a.Sq, width}, at::kBFloat16, q, "out");
    check_dense(stat, {2, BH, a.Mp}, at::kFloat, q, "stat");
    const auto f32 = q.options().dtype(at::kFloat);
    Tensor dtable;
    if (given(bucket_of)) {
        check_dense(*bucket_of, {a.R}, at::kInt, q, "bucket_of");
        dtable = at::empty({NB, heads}, f32);
    }
    if (BH == 0 || a.M == 0 || a.Sk == 0) {
        dq.zero_(); dk.zero_(); dv.zero_();
        if (dtable.defined()) dtable.zero_();
        return dtable;
    }
    ExtBwd w{};
    w.out = out.data_ptr(); w.dout = dout.data_ptr();
    w.stat = stat.data_ptr<float>();
    w.dq = dq.data_ptr(); w.dk = dk.data_ptr(); w.dv = dv.data_ptr();
    a.dqv = view_of(dq, a.G); a.dkv = view_of(dk, 1);
    ext_plan_bwd(BH, a.M, a.Sk, a.tab != nullptr, w.q, w.kv);
    check_grid(a, w.q); check_grid(a, w.kv);
    Tensor dsum = at::empty({w.q.few ? 1 : w.q.splits, BH, a.Mp}, f32), ends, pq, pk, pv;
    w.dsum = dsum.data_ptr<float>();
    const long n_ends = dtable.defined() && NB > 0 ? ext_ends(a, w.q) : 0;
    if (n_ends) {
        ends = at::empty({n_ends}, f32);
        w.ends = ends.data_ptr<float>();
    }
    if (w.q.splits > 1) {
        pq = at::empty({BH * w.q.splits * a.M * hd}, f32);
        w.part_q = pq.data_ptr<float>();
    }
    if (w.kv.splits > 1) {
        pk = at::empty({BH * w.kv.splits * a.Sk * hd}, f32);
        pv = at::empty_like(pk);
        w.part_k = pk.data_ptr<float>();
        w.part_v = pv.data_ptr<float>();
    }
    launch_ext_bwd(a, w, (int)hd, stream_of(q));
    if (dtable.defined() && NB > 0) {
        const RelPlan p = rel_plan(a.B, a.Hkv, a.Sk, (int)hd);
        Tensor dense = at::empty({p.dense}, f32), slab = at::empty({(long)heads * p.rows, a.Rp}, f32),
               mid = at::empty({(long)heads, a.Rp}, f32);
        launch_rel_bias_grad(a, w, (int)hd, p, dense.data_ptr<float>(), slab.data_ptr<float>(), mid.data_ptr<float>(),
                             bucket_of->data_ptr<int>(), dtable.data_ptr<float>(), (int)NB, stream_of(q));
    }
    return dtable;
}

// ------------------------------------------------------------------------------------ relative-position bias
long packed_head_dim(const Tensor& qkv, int64_t heads) {
    check_rows(qkv, "qkv");
    TORCH_CHECK(heads > 0 && qkv.size(2) % (3 * heads) == 0, "rel_bias_attention: width ", qkv.size(2), " is not 3 * heads * head_dim");
    return qkv.size(2) / (3 * heads);
}

// -> out, stat (with `grad`), tab [H, Rp], codes
std::tuple<Tensor, Tensor, Tensor, Tensor> rel_bias_attention_fwd(const Tensor& qkv, const Tensor& table, const Tensor& q_codes,
                                                                  const Tensor& k_codes, const Tensor& bucket_of, int64_t heads,
                                                                  const OptTensor& lens, bool grad) {
    const long hd = packed_head_dim(qkv, heads), D = heads * hd, S = qkv.size(1), R = bucket_of.size(0), NB = table.size(0);
    TORCH_CHECK(R >= 1 && R <= kExtMaxEntries, "rel_bias_attention: ", R, " entries (1 to ", kExtMaxEntries, ")");
    TORCH_CHECK(NB < (1L << 24) && S < (1L << 29) && heads < 65536, "rel_bias_attention: ", NB, " buckets, ", S, " positions, ", heads,
                " heads (below 2^24, 2^29 and 2^16)");
    check_dense(table, {NB, heads}, at::kFloat, qkv, "table");
    check_codes(q_codes, S, qkv, "q_codes");
    check_codes(k_codes, S, qkv, "k_codes");
    check_dense(bucket_of, {R}, at::kInt, qkv, "bucket_of");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(qkv.device());
    const long Rp = (R + 3) / 4 * 4, Sp = (S + 127) / 128 * 128;
    Tensor tab = at::empty({heads, Rp}, table.options()), codes = at::empty({2 * Sp + Sp / 8}, q_codes.options().dtype(at::kInt));
    launch_bias_tables(table.data_ptr<float>(), bucket_of.data_ptr<int>(), q_codes.data_ptr(), q_codes.scalar_type() == at::kLong,
                       k_codes.data_ptr(), k_codes.scalar_type() == at::kLong, tab.data_ptr<float>(), codes.data_ptr<int>(), (int)R, (int)Rp, (int)NB, (int)heads,
                       (int)S, (int)Sp, (float)std::sqrt((double)hd), stream_of(qkv));
    const Tensor q = qkv.narrow(2, 0, D), k = qkv.narrow(2, D, D), v = qkv.narrow(2, 2 * D, D);
    ExtArgs a = ext_args(q, k, v, heads, heads, lens, hd, true);
    set_tables(a, tab, codes, R);
    auto [out, stat] = ext_fwd(a, q, heads, hd, grad);
    return {out, stat, tab, codes};
}

// -> dqkv [B, S, 3 H hd], dtable [NB, H] fp32 (undefined without `want_table`)
std::tuple<Tensor, Tensor> rel_bias_attention_bwd(const Tensor& dout, const Tensor& qkv, const Tensor& out, const Tensor& stat,
                                                  const Tensor& tab, const Tensor& codes, const Tensor& bucket_of,
                                                  int64_t NB, int64_t heads, const OptTensor& lens, bool want_table) {
    const long hd = packed_head_dim(qkv, heads), D = heads * hd;
    TORCH_CHECK(NB >= 0 && NB < (1L << 24) && heads < 65536, "rel_bias_attention: ", NB, " buckets, ", heads, " heads");
    check_same_device(tab, qkv, "tab"); check_same_device(codes, qkv, "codes");
    TORCH_CHECK(tab.scalar_type() == at::kFloat && tab.is_contiguous() && codes.scalar_type() == at::kInt && codes.is_contiguous(),
                "bias tables: as the forward made them");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(qkv.device());
    const Tensor q = qkv.narrow(2, 0, D), k = qkv.narrow(2, D, D), v = qkv.narrow(2, 2 * D, D);
    ExtArgs a = ext_args(q, k, v, heads, heads, lens, hd, true);
    set_tables(a, tab, codes, bucket_of.size(0));
    Tensor dqkv = at::empty({qkv.size(0), qkv.size(1), 3 * D}, qkv.options().memory_format(at::MemoryFormat::Contiguous));
    Tensor dtable = ext_bwd(a, q, heads, hd, dout, out, stat, dqkv.narrow(2, 0, D), dqkv.narrow(2, D, D), dqkv.narrow(2, 2 * D, D),
                            want_table ? OptTensor(bucket_of) : OptTensor(), NB);
    return {dqkv, dtable};
}

struct RelBiasFn : torch::autograd::Function<RelBiasFn> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& qkv_, const Tensor& table_, const Tensor& q_codes,
                          const Tensor& k_codes, const Tensor& bucket_of_, const OptTensor& lens_, int64_t heads) {
        const Tensor qkv = rows3(qkv_), bucket_of = int32(bucket_of_), lens = given(lens_) ? int32(*lens_) : Tensor();
        auto [out, stat, tab, codes] = rel_bias_attention_fwd(qkv, param32(table_), written_out(q_codes).contiguous(), written_out(k_codes).contiguous(), bucket_of, heads, opt(lens), true);
        ctx->save_for_backward({qkv, out, stat, tab, codes, bucket_of, lens});
        ctx->set_materialize_grads(false);
        ctx->saved_data["heads"] = heads;
        ctx->saved_data["buckets"] = table_.size(0);
        ctx->saved_data["type"] = (int64_t)table_.scalar_type();
        return out;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
        return first_order("rel_bias_attention", g, [&] { return gradients(ctx, g); });
    }
    static torch::autograd::variable_list gradients(torch::autograd::AutogradContext* ctx, const torch::autograd::variable_list& g) {
        torch::autograd::variable_list r(7);
        if (!g[0].defined()) return r;
        check_plain("rel_bias_attention", {&g[0]});
        const auto s = ctx->get_saved_variables();
        auto [dqkv, dtable] = rel_bias_attention_bwd(dense16(g[0]), s[0], s[1], s[2], s[3], s[4], s[5], ctx->saved_data["buckets"].toInt(),
                                                     ctx->saved_data["heads"].toInt(), opt(s[6]), ctx->needs_input_grad(1));
        r[0] = dqkv;
        if (dtable.defined()) r[1] = dtable.to((at::ScalarType)ctx->saved_data["type"].toInt());
        return r;
    }
};
OptTensor rel_bias_attention(const Tensor& qkv, const Tensor& table, const Tensor& q_codes, const Tensor& k_codes, const Tensor& bucket_of,
                             int64_t heads, const OptTensor& lens) {
    if (!qkv.is_cuda() || qkv.scalar_type() != at::kBFloat16 || qkv.dim() != 3 || heads < 1 || !attention_dim_ok(qkv.size(2), 3 * heads) ||
        table.dim() != 2 || table.size(1) != heads || !at::isFloatingType(table.scalar_type()) || bucket_of.dim() != 1 ||
        bucket_of.size(0) < 1 || bucket_of.size(0) > kExtMaxEntries || !lengths_fit(lens, qkv))
        return {};
    for (const Tensor* t : {&q_codes, &k_codes})
        if (t->dim() != 1 || t->size(0) != qkv.size(1)) return {};
    for (const Tensor* t : {&q_codes, &k_codes, &bucket_of})
        if (!is_index(*t) || t->device() != qkv.device()) return {};
    if (table.device() != qkv.device()) return {};
    check_plain("rel_bias_attention", {&qkv, &table, &q_codes, &k_codes, &bucket_of, given(lens) ? &*lens : &qkv});
    if (!wants_grad({&qkv, &table}))
        return std::get<0>(rel_bias_attention_fwd(rows3(qkv), param32(table), written_out(q_codes).contiguous(), written_out(k_codes).contiguous(), int32(bucket_of), heads,
                                                  given(lens) ? opt(int32(*lens)) : lens, false));
    check_capture({&qkv, &table});
    return RelBiasFn::apply(qkv, table, q_codes, k_codes, bucket_of, lens, heads);
}

// ------------------------------------------------------------------------------------------- cross attention
long cross_head_dim(const Tensor& q, const Tensor& kv, int64_t heads, int64_t kv_heads) {
    check_rows(q, "q"); check_rows(kv, "kv");
    check_same_device(kv, q, "kv");
    TORCH_CHECK(heads > 0 && kv_heads > 0 && heads % kv_heads == 0, "cross_attention: ", heads, " heads over ", kv_heads, " key heads");
    TORCH_CHECK(q.size(2) % heads == 0 && kv.size(2) == 2 * kv_heads * (q.size(2) / heads), "cross_attention: widths ", q.size(2), " and ",
                kv.size(2), " for ", heads, " heads and ", kv_heads, " key heads");
    TORCH_CHECK(q.size(0) == kv.size(0), "cross_attention: batches ", q.size(0), " and ", kv.size(0));
    return q.size(2) / heads;
}
// q [B, Sq, H hd], kv [B, Sk, 2 Hkv hd] (keys | values) -> out [B, Sq, H hd], stat (with `grad`)
std::tuple<Tensor, Tensor> cross_attention_fwd(const Tensor& q, const Tensor& kv, int64_t heads, int64_t kv_heads, const OptTensor& lens,
                                               bool grad) {
    const long hd = cross_head_dim(q, kv, heads, kv_heads), W = kv_heads * hd;
    c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
    ExtArgs a = ext_args(q, kv.narrow(2, 0, W), kv.narrow(2, W, W), heads, kv_heads, lens, hd, false);
    return ext_fwd(a, q, heads, hd, grad);
}
std::tuple<Tensor, Tensor> cross_attention_bwd(const Tensor& dout, const Tensor& q, const Tensor& kv, const Tensor& out, const Tensor& stat,
                                               int64_t heads, int64_t kv_heads, const OptTensor& lens) {
    const long hd = cross_head_dim(q, kv, heads, kv_heads), W = kv_heads * hd;
    c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
    ExtArgs a = ext_args(q, kv.narrow(2, 0, W), kv.narrow(2, W, W), heads, kv_heads, lens, hd, false);
    Tensor dq = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
    Tensor dkv = at::empty(kv.sizes(), kv.options().memory_format(at::MemoryFormat::Contiguous));
    ext_bwd(a, q, heads, hd, dout, out, stat, dq, dkv.narrow(2, 0, W), dkv.narrow(2, W, W), OptTensor(), 0);
    return {dq, dkv};
}

struct CrossFn : torch::autograd::Function<CrossFn> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& q_, const Tensor& kv_, const OptTensor& lens_, int64_t heads,
                          int64_t kv_heads) {
        const Tensor q = rows3(q_), kv = rows3(kv_), lens = given(lens_) ? int32(*lens_) : Tensor();
        auto [out, stat] = cross_attention_fwd(q, kv, heads, kv_heads, opt(lens), true);
        ctx->save_for_backward({q, kv, out, stat, lens});
        ctx->set_materialize_grads(false);
        ctx->saved_data["heads"] = heads;
        ctx->saved_data["kv_heads"] = kv_heads;
        return out;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
        return first_order("cross_attention", g, [&] { return gradients(ctx, g); });
    }
    static torch::autograd::variable_list gradients(torch::autograd::AutogradContext* ctx, const torch::autograd::variable_list& g) {
        torch::autograd::variable_list r(5);
        if (!g[0].defined()) return r;
        check_plain("cross_attention", {&g[0]});
        const auto s = ctx->get_saved_variables();
        auto [dq, dkv] = cross_attention_bwd(dense16(g[0]), s[0], s[1], s[2], s[3], ctx->saved_data["heads"].toInt(),
                                             ctx->saved_data["kv_heads"].toInt(), opt(s[4]));
        r[0] = dq;
        r[1] = dkv;
        return r;
    }
};
OptTensor cross_attention(const Tensor& q, const Tensor& kv, int64_t heads, int64_t kv_heads, const OptTensor& lens) {
    if (!q.is_cuda() || q.scalar_type() != at::kBFloat16 || kv.scalar_type() != at::kBFloat16 || q.dim() != 3 || kv.dim() != 3 || heads < 1 ||
        kv_heads < 1 || heads % kv_heads || !attention_dim_ok(q.size(2), heads) || kv.size(2) != 2 * kv_heads * (q.size(2) / heads) ||
        q.size(0) != kv.size(0) || q.device() != kv.device() || !lengths_fit(lens, q))
        return {};
    check_plain("cross_attention", {&q, &kv, given(lens) ? &*lens : &q});
    if (!wants_grad({&q, &kv}))
        return std::get<0>(cross_attention_fwd(rows3(q), rows3(kv), heads, kv_heads, given(lens) ? opt(int32(*lens)) : lens, false));
    check_capture({&q, &kv});
    return CrossFn::apply(q, kv, lens, heads, kv_heads);
}

// ---------------------------------------------------------------------------------------- gated residual norm
// x, y [..., D] contiguous; gate [D], or [B, D] for x [B, ..., D]
GatedNorm gated_norm_args(const Tensor& x, const Tensor& y, const Tensor& gate, const Tensor& w, const Tensor& b, const OptTensor& pw,
                          const OptTensor& pb, double eps, double scale) {
    TORCH_CHECK(x.is_cuda() && x.scalar_type() == at::kBFloat16 && x.dim() >= 2, "gated_residual_norm: expected a bf16 GPU tensor [..., D]");
    check_dense(x, x.sizes(), at::kBFloat16, x, "x");
    check_dense(y, x.sizes(), at::kBFloat16, x, "branch");
    const long D = x.size(-1);
    TORCH_CHECK(gated_norm_dim_ok(D), "gated_residual_norm: unsupported width ", D);
    GatedNorm p{};
    p.D = (int)D;
    p.M = x.numel() / D;
    p.per_sample = gate.dim() == 2;
    if (p.per_sample) {
        check_dense(gate, {x.size(0), D}, at::kFloat, x, "gate");
        p.T = x.size(0) ? p.M / x.size(0) : 0;
    } else {
        check_dense(gate, {D}, at::kFloat, x, "gate");
        p.T = p.M;
    }
    TORCH_CHECK(p.M < (1L << 32), "gated_residual_norm: ", p.M, " rows");
    check_dense(w, {D}, at::kFloat, x, "weight"); check_dense(b, {D}, at::kFloat, x, "bias");
    TORCH_CHECK(given(pw) == given(pb), "gated_residual_norm: post_weight and post_bias come together");
    if (given(pw)) {
        check_dense(*pw, {D}, at::kFloat, x, "post_weight"); check_dense(*pb, {D}, at::kFloat, x, "post_bias");
        p.pw = pw->data_ptr<float>(); p.pb = pb->data_ptr<float>();
    }
    p.x = bf16_ptr(x); p.y = bf16_ptr(y);
    p.gate = gate.data_ptr<float>(); p.w = w.data_ptr<float>(); p.b = b.data_ptr<float>();
    p.a = (float)scale; p.eps = (float)eps;
    p.stream = p.M * D * 2 >= 64L << 20;
    return p;
}
// -> u, n, stats [2 or 4, M] (with `grad`)
std::tuple<Tensor, Tensor, Tensor> gated_norm_fwd(const Tensor& x, const Tensor& y, const Tensor& gate, const Tensor& w, const Tensor& b,
                                                  const OptTensor& pw, const OptTensor& pb, double eps, double scale, bool grad) {
    const GatedNorm p = gated_norm_args(x, y, gate, w, b, pw, pb, eps, scale);
    c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    Tensor u = at::empty_like(x), n = at::empty_like(x), stats;
    if (grad) stats = at::empty({p.pw ? 4 : 2, p.M}, w.options());
    if (p.M > 0) launch_gated_norm_fwd(p, u.data_ptr(), n.data_ptr(), grad ? stats.data_ptr<float>() : nullptr, stream_of(x));
    return {u, n, stats};
}
// -> dx, dy, dgate, dw, db[, dpw, dpb]
std::vector<Tensor> gated_norm_bwd(const OptTensor& du, const OptTensor& dn, const Tensor& x, const Tensor& y, const Tensor& gate,
                                   const Tensor& w, const Tensor& b, const OptTensor& pw, const OptTensor& pb, const Tensor& stats,
                                   double eps, double scale) {
    const GatedNorm p = gated_norm_args(x, y, gate, w, b, pw, pb, eps, scale);
    if (given(du)) check_dense(*du, x.sizes(), at::kBFloat16, x, "gradient of the stream");
    if (given(dn)) check_dense(*dn, x.sizes(), at::kBFloat16, x, "gradient of the normalised");
    const bool post = p.pw != nullptr;
    check_dense(stats, {post ? 4 : 2, p.M}, at::kFloat, x, "stats");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    const long D = p.D;
    Tensor dx = at::empty_like(x), dy = at::empty_like(x);
    const int cols = post ? 4 : 2;
    if (p.M == 0) {
        Tensor z = at::zeros({cols, D}, w.options());
        std::vector<Tensor> r = {dx, dy, at::zeros(gate.sizes(), gate.options()), z[1], z[0]};
        if (post) { r.push_back(z[3]); r.push_back(z[2]); }
        return r;
    }
    const GatedNormPlan q = gated_norm_plan(x.size(0), p.T, p.M, p.per_sample);
    // without a gate per sample a workgroup has one unit: its gate sums are one more column block of the slab
    const int groups = cols + (p.per_sample ? 0 : 1), srow = (int)(groups * D);
    const bool parts = p.per_sample && q.chunks > 1;  // (with fewer than 512 samples: the grid that sums the parts is small)
    Tensor work = at::empty({(long)q.blocks * srow + (parts ? q.units * D : 0)}, w.options());
    float* slab = work.data_ptr<float>();
    Tensor sums = q.blocks == 1 ? work.narrow(0, 0, srow).view({groups, D}) : at::empty({groups, D}, w.options());
    Tensor dgate = p.per_sample ? at::empty(gate.sizes(), gate.options()) : Tensor();
    float* gp = !p.per_sample ? slab + cols * D : parts ? slab + (long)q.blocks * srow : dgate.data_ptr<float>();
    launch_gated_norm_bwd(p, q, given(du) ? du->data_ptr() : nullptr, given(dn) ? dn->data_ptr() : nullptr, stats.data_ptr<float>(),
                          dx.data_ptr(), dy.data_ptr(), gp, p.per_sample ? D : srow, slab, srow, stream_of(x));
    launch_gated_norm_sums(slab, q.blocks > 1 ? sums.data_ptr<float>() : nullptr, q.blocks, srow, gp, parts ? dgate.data_ptr<float>() : nullptr,
                           x.size(0), p.D, q.chunks, stream_of(x));
    const std::vector<Tensor> c = sums.unbind(0);  // db, dw[, dpb, dpw][, dgate]
    std::vector<Tensor> r = {dx, dy, p.per_sample ? dgate : c[cols], c[1], c[0]};
    if (post) {
        r.push_back(c[3]);
        r.push_back(c[2]);
    }
    return r;
}

struct GatedNormFn : torch::autograd::Function<GatedNormFn> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& x_, const Tensor& y_, const Tensor& gate_,
                                                  const Tensor& w_, const Tensor& b_, const OptTensor& pw_, const OptTensor& pb_, double eps,
                                                  double scale) {
        const Tensor x = dense16(x_), y = dense16(y_), gate = param32(gate_), w = param32(w_), b = param32(b_);
        const Tensor pw = given(pw_) ? param32(*pw_) : Tensor(), pb = given(pb_) ? param32(*pb_) : Tensor();
        auto [u, n, stats] = gated_norm_fwd(x, y, gate, w, b, opt(pw), opt(pb), eps, scale, true);
        ctx->save_for_backward({x, y, gate, w, b, pw, pb, stats});
        ctx->set_materialize_grads(false);
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["scale"] = scale;
        std::vector<int64_t> types;
        for (const Tensor& t : {gate_, w_, b_, given(pw_) ? *pw_ : w_, given(pb_) ? *pb_ : b_}) types.push_back((int64_t)t.scalar_type());
        ctx->saved_data["types"] = types;
        return {u, n};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
        return first_order("gated_residual_norm", g, [&] { return gradients(ctx, g); });
    }
    static torch::autograd::variable_list gradients(torch::autograd::AutogradContext* ctx, const torch::autograd::variable_list& g) {
        torch::autograd::variable_list r(9);
        if (!g[0].defined() && !g[1].defined()) return r;
        check_plain("gated_residual_norm", {&g[0], &g[1]});
        const auto s = ctx->get_saved_variables();
        const auto types = ctx->saved_data["types"].toIntVector();
        const auto d = gated_norm_bwd(opt(dense16(g[0])), opt(dense16(g[1])), s[0], s[1], s[2], s[3], s[4], opt(s[5]), opt(s[6]), s[7],
                                      ctx->saved_data["eps"].toDouble(), ctx->saved_data["scale"].toDouble());
        for (size_t i = 0; i < d.size(); ++i) {
            const bool typed = i < 2 || types[i - 2] == (int64_t)at::kFloat;
            r[i] = typed ? d[i] : d[i].to((at::ScalarType)types[i - 2]);
        }
        return r;
    }
};
c10::optional<std::tuple<Tensor, Tensor>> gated_residual_norm(const Tensor& x, const Tensor& y, const Tensor& gate, const Tensor& w,
                                                              const Tensor& b, const OptTensor& pw_, const OptTensor& pb_, double eps,
                                                              double scale) {
    const Tensor pw = given(pw_) ? *pw_ : Tensor(), pb = given(pb_) ? *pb_ : Tensor();
    if (!x.is_cuda() || x.scalar_type() != at::kBFloat16 || x.dim() < 2 || !gated_norm_dim_ok(x.size(-1)) || y.scalar_type() != x.scalar_type() ||
        y.sizes() != x.sizes() || y.device() != x.device() || pw.defined() != pb.defined())
        return {};
    const int64_t D = x.size(-1);
    if (gate.sizes() != at::IntArrayRef({D}) && gate.sizes() != at::IntArrayRef({x.size(0), D})) return {};
    for (const Tensor* t : {&gate, &w, &b, &pw, &pb}) {
        if (!t->defined()) continue;
        if (t->device() != x.device() || !at::isFloatingType(t->scalar_type()) || (t != &gate && t->sizes() != at::IntArrayRef({D}))) return {};
    }
    check_plain("gated_residual_norm", {&x, &y, &gate, &w, &b, &pw, &pb});
    if (!wants_grad({&x, &y, &gate, &w, &b, &pw, &pb})) {
        auto [u, n, stats] = gated_norm_fwd(dense16(x), dense16(y), param32(gate), param32(w), param32(b), opt(param32(pw)),
                                            opt(param32(pb)), eps, scale, false);
        return std::make_tuple(u, n);
    }
    check_capture({&x, &y, &gate, &w, &b, &pw, &pb});
    const auto r = GatedNormFn::apply(x, y, gate, w, b, pw_, pb_, eps, scale);
    return std::make_tuple(r[0], r[1]);
}

}  // namespace

void bind_transformer_ops(pybind11::module& m) {
    using release = pybind11::call_guard<pybind11::gil_scoped_release>;
    m.def("rel_bias_attention", &rel_bias_attention, release());
    m.def("cross_attention", &cross_attention, release());
    m.def("gated_residual_norm", &gated_residual_norm, release());
    m.attr("rel_bias_max_entries") = kExtMaxEntries;
}

}  // namespace pdt
