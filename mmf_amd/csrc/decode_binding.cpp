// mmf_amd :: torch.ops.mmf_amd_decode.* — the operators of mmf_amd/decoding.py over the C ABI of include/mmf_amd.h (libmmf_amd_decode.so; host code only).
// Every argument check of these operators is here, so that a call costs the host a few microseconds: a decoding step is a handful of kernels of about as many.
// The library loads without a GPU as well; the operators then refuse (no CPU path).
#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <initializer_list>
#include <optional>
#include <tuple>

#include "mmf_amd.h"

namespace {

using at::Tensor;
using std::optional;

#define NEED(cond, ...) TORCH_CHECK(cond, "mmf_amd decoding: ", __VA_ARGS__)

void check(const Tensor& t, const char* name, at::ScalarType dt) {
    NEED(t.scalar_type() == dt, name, " must be ", dt, ", got ", t.scalar_type());
    NEED(!(t.requires_grad() && at::GradMode::is_enabled()), name, " requires a gradient: decoding is forward only (torch.no_grad)");
    NEED(!(c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined()), name, " carries a tangent: decoding has no derivative in forward mode");
    NEED(!t.is_neg(), name, " is a negated view, whose memory holds other values (resolve_neg)");
}
void check_float(const Tensor& t, const char* name) {
    NEED(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat, name, " must be bfloat16 or float32, got ", t.scalar_type());
    check(t, name, t.scalar_type());
}
// shape: -1 takes any size
void check_dense(const Tensor& t, const char* name, at::ScalarType dt, std::initializer_list<int64_t> shape) {
    check(t, name, dt);
    bool same = t.dim() == (int64_t)shape.size();
    int64_t a = 0;
    for (int64_t n : shape) { same = same && (n < 0 || t.size(a) == n); ++a; }
    NEED(same, name, " must be ", at::IntArrayRef(shape.begin(), shape.size()), " (-1: any), got ", t.sizes());
    NEED(t.is_contiguous(), name, " must be contiguous");
}
void check_page(int64_t n) { NEED(n >= 1 && n <= MMF_PAGE_MAX && (n & (n - 1)) == 0, "page_size must be a power of two up to ", MMF_PAGE_MAX, ", got ", n); }
void check_beams(int64_t n) { NEED(n >= 1 && n <= MMF_BEAMS_MAX, "beams must be 1 .. ", MMF_BEAMS_MAX, ", got ", n); }

void check_pools(const Tensor& k, const Tensor& v) {
    check_float(k, "key_cache");
    check(v, "value_cache", k.scalar_type());
    NEED(k.dim() == 4 && k.stride(3) == 1 && k.numel() > 0, "key_cache must be [pages, kv_heads, page_size, head_dim] with contiguous head_dim, got ", k.sizes());
    check_page(k.size(2));
    NEED(v.sizes() == k.sizes() && v.strides() == k.strides(), "key_cache and value_cache must have one shape and one layout");
    NEED(k.size(0) <= 0x7fffffff, "too many pages");
}
bool on16(const Tensor& t, int64_t dims) {
    const int64_t unit = 16 / t.element_size();
    bool ok = reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    for (int64_t a = 0; a < dims; ++a) ok = ok && (t.size(a) == 1 || t.stride(a) % unit == 0);
    return ok;
}
// a stride that no element is reached by (size 1) may be anything: the kernels only want it on 16 bytes
int64_t step_of(const Tensor& t, int64_t a) { return t.size(a) == 1 ? 0 : t.stride(a); }

// the device of the tensors for the duration of a call; its current stream takes the work
struct On {
    c10::hip::OptionalHIPGuard guard;
    void* stream;
    On(std::initializer_list<const Tensor*> ts) : stream(nullptr) {
        const at::Device d = (*ts.begin())->device();
        for (const Tensor* t : ts) NEED(!t->defined() || t->device() == d, "tensors on different devices: ", d, " and ", t->device());
        NEED(d.is_cuda(), "tensors must live in HBM (cuda/hip tensors), got ", d, "; there is no CPU path");
        guard.set_index(d.index());
        stream = reinterpret_cast<void*>(c10::hip::getCurrentHIPStream(d.index()).stream());
    }
};

void done(int rc, const char* what) { TORCH_CHECK(rc == 0, what, " failed: ", mmf_amd_last_error()); }

// several small results in one allocation: an allocation costs as much time as a small plan
struct Carver {
    Tensor base;
    int64_t at = 0;
    Carver(int64_t bytes, const Tensor& like) : base(at::empty({bytes}, like.options().dtype(at::kByte))) {}
    static int64_t room(int64_t bytes) { return (bytes + 15) / 16 * 16; }
    Tensor take(at::IntArrayRef shape, at::ScalarType dt) {
        Tensor t = at::detail::make_tensor<at::TensorImpl>(c10::Storage(base.storage()), base.key_set(), c10::scalarTypeToTypeMeta(dt));
        t.unsafeGetTensorImpl()->set_storage_offset(at / (int64_t)c10::elementSize(dt));
        t.unsafeGetTensorImpl()->set_sizes_contiguous(shape);
        at += room(t.numel() * (int64_t)c10::elementSize(dt));
        return t;
    }
};
Tensor workspace(int64_t bytes, const Tensor& like) { return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor(); }
void* P(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
template <typename T> T* PT(const Tensor& t) { return static_cast<T*>(P(t)); }

using Plan = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor>;

// out: where the results go, all or (null) none of them
Plan plan_into(const Tensor& q_lens, const Tensor& kv_lens, const Tensor& tables, const Tensor& owned, const Tensor& free_pages, const Tensor& free_top, int64_t page_size,
               int64_t rows, int64_t beams, bool shared, const Plan* out) {
    check_page(page_size);
    check_beams(beams);
    check_dense(q_lens, "q_lens", at::kInt, {-1});
    const int64_t G = q_lens.numel(), R = G * beams, n = shared ? G : R;
    NEED(G > 0 && rows > 0 && rows <= (1 << 30), "a plan needs groups and 1 .. 2**30 rows, got ", G, " and ", rows);
    check_dense(kv_lens, "kv_lens", at::kInt, {G});
    check_dense(tables, "tables", at::kInt, {R, -1});
    check_dense(owned, "owned", at::kInt, {R, tables.size(1)});
    check_dense(free_pages, "free_pages", at::kInt, {-1});
    check_dense(free_top, "free_top", at::kInt, {1});
    NEED(tables.size(1) > 0 && free_pages.numel() > 0, "tables and free_pages must not be empty");
    NEED(tables.size(1) * page_size <= (1 << 30) && R <= 0x0fffffff && free_pages.numel() <= 0x7fffffff, "a table row names more than 2**30 tokens");
    Plan p;
    if (out) {
        p = *out;
        check_dense(std::get<0>(p), "out.q_start", at::kInt, {n});
        check_dense(std::get<1>(p), "out.q_lens", at::kInt, {G});
        check_dense(std::get<2>(p), "out.kv_lens", at::kInt, {G});
        check_dense(std::get<3>(p), "out.slots", at::kLong, {rows});
        check_dense(std::get<4>(p), "out.positions", at::kInt, {rows});
        check_dense(std::get<5>(p), "out.copies", at::kInt, {R, 3});
        check_dense(std::get<6>(p), "out.free_top", at::kInt, {1});
        check_dense(std::get<7>(p), "out.refused", at::kInt, {1});
    }
    On on({&q_lens, &kv_lens, &tables, &owned, &free_pages, &free_top, &std::get<0>(p), &std::get<1>(p), &std::get<2>(p), &std::get<3>(p), &std::get<4>(p), &std::get<5>(p),
           &std::get<6>(p), &std::get<7>(p)});
    const int64_t ws_bytes = mmf_paged_plan_ws_bytes((int)G, (int)beams);
    void* ws;                                                     // (small: next to the results it costs no allocation of its own)
    Tensor ws_owner;
    if (!out) {
        Carver c(Carver::room(ws_bytes) + Carver::room(8 * rows) + Carver::room(4 * n) + 2 * Carver::room(4 * G) + Carver::room(4 * rows) + Carver::room(12 * R) + 32, q_lens);
        ws = c.base.data_ptr();
        c.at = Carver::room(ws_bytes);
        const Tensor slots = c.take({rows}, at::kLong), start = c.take({n}, at::kInt), granted = c.take({G}, at::kInt), kv = c.take({G}, at::kInt),
                     pos = c.take({rows}, at::kInt), copies = c.take({R, 3}, at::kInt), top = c.take({1}, at::kInt), refused = c.take({1}, at::kInt);
        p = {start, granted, kv, slots, pos, copies, top, refused};
    } else {
        ws_owner = workspace(ws_bytes, q_lens);
        ws = P(ws_owner);
    }
    mmf_paged_plan_desc d = {};
    d.q_lens = PT<int32_t>(q_lens); d.kv_lens = PT<int32_t>(kv_lens); d.tables = PT<int32_t>(tables); d.owned = PT<int32_t>(owned);
    d.free_pages = PT<int32_t>(free_pages); d.free_top = PT<int32_t>(free_top);
    d.q_start = PT<int32_t>(std::get<0>(p)); d.granted = PT<int32_t>(std::get<1>(p)); d.kv_out = PT<int32_t>(std::get<2>(p)); d.slots = PT<int64_t>(std::get<3>(p));
    d.positions = PT<int32_t>(std::get<4>(p)); d.copies = PT<int32_t>(std::get<5>(p)); d.top_out = PT<int32_t>(std::get<6>(p)); d.refused = PT<int32_t>(std::get<7>(p));
    d.ws = ws;
    d.groups = (int)G; d.beams = (int)beams; d.blocks = (int)tables.size(1); d.page_size = (int)page_size; d.rows = (int)rows; d.shared = shared;
    d.free_capacity = (int)free_pages.numel();
    done(mmf_paged_plan(&d, on.stream), "mmf_paged_plan");
    return p;
}
Plan plan_pages(const Tensor& q_lens, const Tensor& kv_lens, const Tensor& tables, const Tensor& owned, const Tensor& free_pages, const Tensor& free_top, int64_t page_size,
                int64_t rows, int64_t beams, bool shared) {
    return plan_into(q_lens, kv_lens, tables, owned, free_pages, free_top, page_size, rows, beams, shared, nullptr);
}
void plan_pages_out(const Tensor& q_lens, const Tensor& kv_lens, const Tensor& tables, const Tensor& owned, const Tensor& free_pages, const Tensor& free_top, int64_t page_size,
                    int64_t rows, int64_t beams, bool shared, const Tensor& q_start, const Tensor& granted, const Tensor& kv_out, const Tensor& slots, const Tensor& positions,
                    const Tensor& copies, const Tensor& top_out, const Tensor& refused) {
    const Plan out(q_start, granted, kv_out, slots, positions, copies, top_out, refused);
    plan_into(q_lens, kv_lens, tables, owned, free_pages, free_top, page_size, rows, beams, shared, &out);
}

void write_pages(const Tensor& k, const Tensor& v, const Tensor& key_cache, const Tensor& value_cache, const Tensor& slots) {
    check_pools(key_cache, value_cache);
    check_dense(slots, "slots", at::kLong, {-1});
    const int64_t T = slots.numel(), H = key_cache.size(1), D = key_cache.size(3);
    NEED(T <= 0x7fffffff, "too many rows");
    const Tensor* ts[2] = {&k, &v};
    const char* names[2] = {"k", "v"};
    for (int i = 0; i < 2; ++i) {
        const Tensor& t = *ts[i];
        check(t, names[i], key_cache.scalar_type());
        NEED(t.dim() == 3 && t.size(0) == T && t.size(1) == H && t.size(2) == D, names[i], " must be [", T, ", ", H, ", ", D, "], got ", t.sizes());
        NEED(t.stride(2) == 1 || D == 1, names[i], " must have contiguous head_dim");
    }
    On on({&k, &v, &key_cache, &value_cache, &slots});
    mmf_paged_write_desc d = {};
    d.k = P(k); d.v = P(v);
    d.k_row = step_of(k, 0); d.k_head = step_of(k, 1); d.v_row = step_of(v, 0); d.v_head = step_of(v, 1);
    d.k_cache = P(key_cache); d.v_cache = P(value_cache);
    d.page_stride = step_of(key_cache, 0); d.head_stride = step_of(key_cache, 1); d.pos_stride = step_of(key_cache, 2);
    d.slots = PT<int64_t>(slots);
    d.tokens = (int)T; d.pages = (int)key_cache.size(0); d.page_size = (int)key_cache.size(2); d.kv_heads = (int)H; d.head_dim = (int)D;
    d.is_f32 = k.scalar_type() == at::kFloat;
    if (T) done(mmf_paged_write(&d, on.stream), "mmf_paged_write");
}

Tensor attend_into(const Tensor& q, const Tensor& key_cache, const Tensor& value_cache, const Tensor& tables, const Tensor& kv_lens, const Tensor& q_start,
                   const Tensor& q_lens, int64_t max_q, int64_t beams, bool causal, optional<double> scale, Tensor out) {
    check_pools(key_cache, value_cache);
    const int64_t D = key_cache.size(3), Hk = key_cache.size(1);
    NEED(D == 64 || D == 128, "head_dim must be 64 or 128, got ", D);
    check_beams(beams);
    check(tables, "tables", at::kInt);
    NEED(tables.dim() == 2 && tables.numel() > 0 && (tables.stride(1) == 1 || tables.size(1) == 1), "tables must be [requests, blocks] with contiguous rows");
    const int64_t R = tables.size(0);
    NEED(R % beams == 0 && R <= 0x7fffffff, R, " table rows are no groups of ", beams, " beams");
    NEED(tables.size(1) * key_cache.size(2) <= (1 << 30), "a table row names more than 2**30 tokens");
    check_dense(kv_lens, "kv_lens", at::kInt, {R / beams});
    check_dense(q_lens, "q_lens", at::kInt, {R / beams});
    check_dense(q_start, "q_start", at::kInt, {R});
    check(q, "q", key_cache.scalar_type());
    NEED(q.dim() == 3 && q.size(2) == D && q.stride(2) == 1 && q.size(1) > 0 && q.size(1) % Hk == 0, "q must be [rows, heads, ", D,
         "], contiguous head_dim, heads a multiple of ", Hk, "; got ", q.sizes());
    NEED(max_q >= 1, "max_q must be at least 1, got ", max_q);
    NEED(on16(q, 2) && on16(key_cache, 3) && on16(value_cache, 3), "q, key_cache and value_cache must start and stride on 16 bytes");
    if (out.defined()) {
        check(out, "out", q.scalar_type());
        NEED(out.sizes() == q.sizes() && out.stride(2) == 1 && on16(out, 2), "out must be shaped as q, with contiguous head_dim, and start and stride on 16 bytes");
    }
    On on({&q, &key_cache, &value_cache, &tables, &kv_lens, &q_start, &q_lens, &out});
    if (!out.defined()) out = at::empty(q.sizes(), q.options());
    const int64_t T = q.size(0);
    if (T == 0) return out;
    NEED(T <= 0x7fffffff && q.size(1) <= 0xffff, "too many rows or heads");
    mmf_paged_attn_desc d = {};
    d.q = P(q); d.q_row = step_of(q, 0); d.q_head = step_of(q, 1);
    d.k_cache = P(key_cache); d.v_cache = P(value_cache);
    d.page_stride = step_of(key_cache, 0); d.head_stride = step_of(key_cache, 1); d.pos_stride = step_of(key_cache, 2);
    d.tables = PT<int32_t>(tables); d.table_row = step_of(tables, 0);
    d.kv_lens = PT<int32_t>(kv_lens); d.q_start = PT<int32_t>(q_start); d.q_lens = PT<int32_t>(q_lens);
    d.out = P(out); d.out_row = step_of(out, 0); d.out_head = step_of(out, 1);
    d.tokens = (int)T; d.requests = (int)R; d.beams = (int)beams; d.blocks = (int)tables.size(1); d.pages = (int)key_cache.size(0); d.page_size = (int)key_cache.size(2);
    d.heads = (int)q.size(1); d.kv_heads = (int)Hk; d.head_dim = (int)D; d.max_q = (int)std::min(max_q, T); d.causal = causal; d.is_f32 = q.scalar_type() == at::kFloat;
    d.scale = (float)(scale.has_value() ? *scale : 1.0 / std::sqrt((double)D));
    const Tensor ws = workspace(mmf_paged_attention_ws_bytes(&d), q);
    d.ws = P(ws);
    done(mmf_paged_attention(&d, on.stream), "mmf_paged_attention");
    return out;
}
Tensor attend_pages(const Tensor& q, const Tensor& key_cache, const Tensor& value_cache, const Tensor& tables, const Tensor& kv_lens, const Tensor& q_start,
                    const Tensor& q_lens, int64_t max_q, int64_t beams, bool causal, optional<double> scale) {
    return attend_into(q, key_cache, value_cache, tables, kv_lens, q_start, q_lens, max_q, beams, causal, scale, Tensor());
}
void attend_pages_out(const Tensor& q, const Tensor& key_cache, const Tensor& value_cache, const Tensor& tables, const Tensor& kv_lens, const Tensor& q_start,
                      const Tensor& q_lens, int64_t max_q, int64_t beams, bool causal, optional<double> scale, const Tensor& out) {
    attend_into(q, key_cache, value_cache, tables, kv_lens, q_start, q_lens, max_q, beams, causal, scale, out);
}

using Beams = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>;

// out: where the results go, all (the history where there is one) or (null) none of them
Beams select_into(const Tensor& logits, const Tensor& scores, const Tensor& finished, int64_t eos, const optional<Tensor>& history_, int64_t step,
                  const optional<Tensor>& step_at_, const Tensor* const* out) {
    check_dense(scores, "scores", at::kFloat, {-1, -1});
    const int64_t G = scores.size(0), W = scores.size(1);
    check_beams(W);
    NEED(G > 0 && G * W <= 65535, "select_beams needs 1 .. 65535 rows in groups, got ", G * W);
    check_float(logits, "logits");
    NEED(logits.dim() == 2 && logits.size(0) == G * W, "logits must be [", G * W, ", vocab], got ", logits.sizes());
    const int64_t V = logits.size(1);
    NEED(V <= (1 << 22), "a vocabulary of up to 2**22 tokens, got ", V);
    NEED(V > 0 && (logits.stride(1) == 1 || V == 1) && (logits.stride(0) >= V || G * W == 1), "logits must have contiguous rows that do not overlap");
    check_dense(finished, "finished", at::kBool, {G, W});
    NEED(eos >= 0 && eos < V, "eos ", eos, " is not in the vocabulary of ", V);
    const Tensor history = history_.has_value() ? *history_ : Tensor();
    const Tensor step_at = step_at_.has_value() ? *step_at_ : Tensor();
    if (step_at.defined()) check_dense(step_at, "step", at::kInt, {1});
    if (history.defined()) {
        check_dense(history, "history", at::kLong, {G, W, -1});
        NEED(step_at.defined() || (step >= 0 && step < history.size(2)), "step ", step, " is not a column of the history of length ", history.size(2));
    }
    Tensor o[5];
    if (out) {
        NEED(out[4]->defined() == history.defined(), "out is a BeamStep; its history goes with history");
        const char* names[4] = {"out.scores", "out.parents", "out.tokens", "out.finished"};
        const at::ScalarType types[4] = {at::kFloat, at::kLong, at::kLong, at::kBool};
        for (int i = 0; i < 4; ++i) check_dense(o[i] = *out[i], names[i], types[i], {G, W});
        if (history.defined()) check_dense(o[4] = *out[4], "out.history", at::kLong, {G, W, history.size(2)});
    }
    On on({&logits, &scores, &finished, &history, &step_at, &o[0], &o[1], &o[2], &o[3], &o[4]});
    if (!out) {
        Carver c(Carver::room(4 * G * W) + 2 * Carver::room(8 * G * W) + Carver::room(G * W), logits);
        o[0] = c.take({G, W}, at::kFloat);
        o[1] = c.take({G, W}, at::kLong);
        o[2] = c.take({G, W}, at::kLong);
        o[3] = c.take({G, W}, at::kBool);
        if (history.defined()) o[4] = at::empty(history.sizes(), history.options());
    }
    const Tensor ws = workspace(mmf_beam_select_ws_bytes((int)G, (int)W, V, logits.scalar_type() == at::kFloat), logits);
    mmf_beam_select_desc d = {};
    d.logits = P(logits); d.ld = G * W == 1 ? V : logits.stride(0);
    d.scores = PT<float>(scores); d.finished = PT<uint8_t>(finished); d.history = PT<int64_t>(history);
    d.scores_out = PT<float>(o[0]); d.parents = PT<int64_t>(o[1]); d.tokens = PT<int64_t>(o[2]); d.finished_out = PT<uint8_t>(o[3]); d.history_out = PT<int64_t>(o[4]);
    d.ws = P(ws);
    d.vocab = V; d.eos = eos; d.length = history.defined() ? history.size(2) : 0; d.step = step;
    d.groups = (int)G; d.beams = (int)W; d.is_f32 = logits.scalar_type() == at::kFloat;
    done(step_at.defined() ? mmf_beam_select_at(&d, PT<int32_t>(step_at), on.stream) : mmf_beam_select(&d, on.stream), "mmf_beam_select");
    if (!o[4].defined()) o[4] = at::empty({0}, o[1].options());
    return {o[0], o[1], o[2], o[3], o[4]};
}
Beams select_beams(const Tensor& logits, const Tensor& scores, const Tensor& finished, int64_t eos, const optional<Tensor>& history, int64_t step,
                   const optional<Tensor>& step_at) {
    return select_into(logits, scores, finished, eos, history, step, step_at, nullptr);
}
void select_beams_out(const Tensor& logits, const Tensor& scores, const Tensor& finished, int64_t eos, const optional<Tensor>& history, int64_t step,
                      const optional<Tensor>& step_at, const Tensor& scores_out, const Tensor& parents, const Tensor& tokens, const Tensor& finished_out,
                      const optional<Tensor>& history_out) {
    const Tensor none;
    const Tensor* out[5] = {&scores_out, &parents, &tokens, &finished_out, history_out.has_value() ? &*history_out : &none};
    select_into(logits, scores, finished, eos, history, step, step_at, out);
}

// The planes of a cache are one run: a leading dimension steps over all planes of the dimension behind it, and of the next one that has several (what stands between,
// of size 1, may have any stride).
int64_t inner_plane_dim(const Tensor& c, int64_t a) {             // the next leading dimension behind a of a size other than 1; -1: none
    for (++a; a <= c.dim() - 5; ++a)
        if (c.size(a) != 1) return a;
    return -1;
}
void check_planes(const Tensor& c) {
    check_float(c, "cache");
    NEED(c.dim() >= 4 && c.numel() > 0 && c.stride(-1) == 1, "cache must be [..., pages, kv_heads, page_size, head_dim] with contiguous head_dim, got ", c.sizes());
    for (int64_t a = 0; a < c.dim() - 5; ++a) {
        const int64_t in = inner_plane_dim(c, a);
        NEED(c.size(a) == 1 || (c.stride(a) == c.stride(a + 1) * c.size(a + 1) && (in < 0 || c.stride(a) == c.stride(in) * c.size(in))),
             "the leading dimensions of cache must be one run of planes");
    }
    check_page(c.size(-2));
}
int64_t plane_step(const Tensor& c) {                             // from a plane to the next; 0: there is one
    for (int64_t a = c.dim() - 5; a >= 0; --a)
        if (c.size(a) != 1) return c.stride(a);
    return 0;
}
void copy(const int32_t* copies, int64_t n, const Tensor& c, void* stream) {
    mmf_paged_copy_desc d = {};
    int64_t planes = 1;
    for (int64_t a = 0; a < c.dim() - 4; ++a) planes *= c.size(a);
    d.copies = copies; d.cache = P(c);
    d.plane_stride = plane_step(c);
    d.page_stride = step_of(c, c.dim() - 4); d.head_stride = step_of(c, c.dim() - 3); d.pos_stride = step_of(c, c.dim() - 2);
    NEED(n <= 0x7fffffff && planes <= 65535 && c.size(-4) <= 0x7fffffff, "too many rows or planes");
    d.rows = (int)n; d.planes = (int)planes; d.pages = (int)c.size(-4); d.page_size = (int)c.size(-2); d.kv_heads = (int)c.size(-3); d.head_dim = (int)c.size(-1);
    d.is_f32 = c.scalar_type() == at::kFloat;
    done(mmf_paged_copy(&d, stream), "mmf_paged_copy");
}

Tensor reorder_into(const Tensor& parents, const Tensor& kv_lens, const Tensor& tables, const Tensor& cache, Tensor out) {
    check_dense(parents, "parents", at::kLong, {-1, -1});
    const int64_t G = parents.size(0), W = parents.size(1);
    check_beams(W);
    NEED(G > 0 && G * W <= 0x3fffffff, "reorder_pages needs a group");
    check_dense(kv_lens, "kv_lens", at::kInt, {G});
    check_dense(tables, "tables", at::kInt, {G * W, -1});
    NEED(tables.size(1) > 0 && tables.size(1) <= 0x3fffffff, "tables must not be empty");
    check_planes(cache);
    if (out.defined()) check_dense(out, "out", at::kInt, {G * W, tables.size(1)});
    On on({&parents, &kv_lens, &tables, &cache, &out});
    if (!out.defined()) out = at::empty(tables.sizes(), tables.options());
    const Tensor copies = at::empty({G * W, 3}, tables.options());
    mmf_paged_reorder_desc d = {};
    d.parents = PT<int64_t>(parents); d.kv_lens = PT<int32_t>(kv_lens); d.tables = PT<int32_t>(tables); d.tables_out = PT<int32_t>(out); d.copies = PT<int32_t>(copies);
    d.groups = (int)G; d.beams = (int)W; d.blocks = (int)tables.size(1); d.page_size = (int)cache.size(-2);
    done(mmf_paged_reorder(&d, on.stream), "mmf_paged_reorder");
    copy(d.copies, G * W, cache, on.stream);
    return out;
}
Tensor reorder_pages(const Tensor& parents, const Tensor& kv_lens, const Tensor& tables, const Tensor& cache) {
    return reorder_into(parents, kv_lens, tables, cache, Tensor());
}
void reorder_pages_out(const Tensor& parents, const Tensor& kv_lens, const Tensor& tables, const Tensor& cache, const Tensor& out) {
    reorder_into(parents, kv_lens, tables, cache, out);
}

void copy_pages(const Tensor& copies, const Tensor& cache) {
    check_dense(copies, "copies", at::kInt, {-1, 3});
    check_planes(cache);
    On on({&copies, &cache});
    if (copies.size(0)) copy(PT<int32_t>(copies), copies.size(0), cache, on.stream);
}

}  // namespace

// A schema marks every tensor that its call writes: the state that plans and copies change, and in the forms with `out` the results, which may be the inputs of their kind.
// The results that a call makes itself are tensors of their own (several in one allocation, apart from each other).
#define PLAN_ARGS "Tensor q_lens, Tensor kv_lens, Tensor(a!) tables, Tensor(b!) owned, Tensor(c!) free_pages, Tensor free_top, int page_size, int rows, int beams, bool shared"
#define ATTEND_ARGS "Tensor q, Tensor key_cache, Tensor value_cache, Tensor tables, Tensor kv_lens, Tensor q_start, Tensor q_lens, int max_q, int beams, bool causal, float? scale"
#define SELECT_ARGS "Tensor logits, Tensor scores, Tensor finished, int eos, Tensor? history, int step, Tensor? step_at"
TORCH_LIBRARY(mmf_amd_decode, m) {
    m.def("plan_pages(" PLAN_ARGS ") -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
    m.def("plan_pages.out(" PLAN_ARGS ", *, Tensor(d!) out_q_start, Tensor(e!) out_q_lens, Tensor(f!) out_kv_lens, Tensor(g!) out_slots, Tensor(h!) out_positions, "
          "Tensor(i!) out_copies, Tensor(j!) out_free_top, Tensor(k!) out_refused) -> ()");
    m.def("write_pages(Tensor k, Tensor v, Tensor(a!) key_cache, Tensor(b!) value_cache, Tensor slots) -> ()");
    m.def("attend_pages(" ATTEND_ARGS ") -> Tensor");
    m.def("attend_pages.out(" ATTEND_ARGS ", *, Tensor(a!) out) -> ()");
    m.def("select_beams(" SELECT_ARGS ") -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
    m.def("select_beams.out(" SELECT_ARGS ", *, Tensor(a!) out_scores, Tensor(b!) out_parents, Tensor(c!) out_tokens, Tensor(d!) out_finished, "
          "Tensor(e!)? out_history) -> ()");
    m.def("reorder_pages(Tensor parents, Tensor kv_lens, Tensor tables, Tensor(a!) cache) -> Tensor");
    m.def("reorder_pages.out(Tensor parents, Tensor kv_lens, Tensor tables, Tensor(a!) cache, *, Tensor(b!) out) -> ()");
    m.def("copy_pages(Tensor copies, Tensor(a!) cache) -> ()");
}

TORCH_LIBRARY_IMPL(mmf_amd_decode, CompositeImplicitAutograd, m) {
    m.impl("plan_pages", plan_pages);
    m.impl("plan_pages.out", plan_pages_out);
    m.impl("write_pages", write_pages);
    m.impl("attend_pages", attend_pages);
    m.impl("attend_pages.out", attend_pages_out);
    m.impl("select_beams", select_beams);
    m.impl("select_beams.out", select_beams_out);
    m.impl("reorder_pages", reorder_pages);
    m.impl("reorder_pages.out", reorder_pages_out);
    m.impl("copy_pages", copy_pages);
}
