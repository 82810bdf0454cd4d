// Host side of the batched calls: argument checks, outputs, workspace and the call of the C ABI (include/trb_kv.h), for
// tokenrush_b200/fused.py.  The calls are made once per layer and step with a dozen tensors each; checked and packed in Python they
// took 14 to 22 us, several times what a small step's kernels do.  Knows torch tensors; the CUDA library itself does not,
// and is reached through the function addresses that bind() is given.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <optional>
#include <unordered_map>

#include "../../include/trb_kv.h"

namespace py = pybind11;
using at::Tensor;
using Maybe = std::optional<Tensor>;

namespace {

decltype(&trb_paged_append) p_append;
decltype(&trb_attn_paged_workspace_bytes) p_workspace;
decltype(&trb_attn_paged) p_attn;
decltype(&trb_spec_verify) p_verify;
PyObject *on_error;                      // called with (code, function name), raises

inline void need(bool ok, const char *what) { if (!ok) throw py::value_error(what); }
inline void call(int code, const char *name) {
    if (code) py::reinterpret_borrow<py::object>(on_error)(code, name);
}

struct Device {
    int index;
    explicit Device(const Tensor &first) : index(first.is_cuda() ? first.get_device() : -1) { check(first); }
    void check(const Tensor &t) const {
        if (!t.is_cuda()) throw std::runtime_error("tokenrush_b200 runs on CUDA tensors only (there is no CPU path)");
        if (t.get_device() != index) throw std::runtime_error("the tensors of a call have to be on one device");
    }
    void check(const Maybe &t) const { if (t) check(*t); }
    template <typename... T> void all(const T &...t) const {
        (check(t), ...);
        if (c10::cuda::current_device() != index) throw std::runtime_error("the tensors are not on the current CUDA device");
    }
    void *stream() const { return (void *)c10::cuda::getCurrentCUDAStream(index).stream(); }
};

inline void *ptr(const Tensor &t) { return t.data_ptr(); }
inline void *ptr(const Maybe &t) { return t ? t->data_ptr() : nullptr; }
inline int width(const Tensor &t) { return t.scalar_type() == at::kInt ? 4 : 8; }
inline bool is_int(const Tensor &t) { return t.scalar_type() == at::kInt || t.scalar_type() == at::kLong; }

trb_paged_t make_pool(const Tensor &k, const Tensor &v, const Maybe &ks, const Maybe &vs) {
    need(k.dim() == 4 && v.sizes() == k.sizes() && k.is_contiguous() && v.is_contiguous(), "pools must be contiguous [PAGES, HKV, PAGE, D] of one shape");
    const bool fp8 = k.scalar_type() == at::kFloat8_e4m3fn;
    if (v.scalar_type() != k.scalar_type() || !(fp8 || k.scalar_type() == at::kBFloat16)) throw py::type_error("pools must be float8_e4m3fn or bfloat16");
    trb_paged_t p = {};
    p.k = ptr(k); p.v = ptr(v);
    p.hkv = (int32_t)k.size(1); p.d = (int32_t)k.size(3); p.page_size = (int32_t)k.size(2); p.num_pages = k.size(0);
    p.kv_dtype = fp8 ? TRB_KV_FP8 : TRB_KV_BF16;
    if (fp8) {
        for (const Maybe *s : {&ks, &vs})
            need(*s && (*s)->scalar_type() == at::kFloat && (*s)->sizes() == k.sizes().slice(0, 3) && (*s)->is_contiguous(),
                 "an fp8 pool needs contiguous float32 k_scale and v_scale [PAGES, HKV, PAGE]");
        p.k_scale = (float *)ptr(*ks); p.v_scale = (float *)ptr(*vs);
    }
    return p;
}

trb_batch_t make_batch(const Tensor &table, const Tensor &lens) {
    need(table.scalar_type() == at::kInt && table.dim() == 2 && table.stride(1) == 1, "table must be int32 [B, PAGES] with contiguous rows");
    need(is_int(lens) && lens.dim() == 1 && lens.size(0) == table.size(0) && lens.is_contiguous(), "lens must be contiguous int32 or int64 [B]");
    trb_batch_t b = {};
    b.table = (const int32_t *)ptr(table); b.table_stride = table.stride(0); b.table_pages = (int32_t)table.size(1);
    b.lens = ptr(lens); b.lens_width = width(lens); b.n_seqs = (int32_t)table.size(0);
    return b;
}

// A python int, or a device tensor of one int32 / int64.
trb_cursor_t make_length(const py::handle &x, const Device &dev) {
    trb_cursor_t c = {nullptr, 8, 0, 0};
    if (!THPVariable_Check(x.ptr())) {
        c.host = py::cast<int64_t>(x);
        return c;
    }
    const Tensor &t = THPVariable_Unpack(x.ptr());
    if (!is_int(t) || t.numel() != 1) throw py::type_error("a length on the device is an int32 or int64 tensor of one element");
    dev.check(t);
    c.dev = ptr(t); c.width = width(t);
    return c;
}

void check_weight(const Maybe &w, int64_t d) {
    if (w) need(w->scalar_type() == at::kBFloat16 && w->dim() == 1 && w->size(0) == d && w->is_contiguous(), "norm weights must be bfloat16 [D]");
}

Maybe paged_append(const Tensor &k, const Tensor &v, const Tensor &k_pages, const Tensor &v_pages, const Tensor &table, const Tensor &lens, const Maybe &k_scale,
                   const Maybe &v_scale, const Maybe &q, const Maybe &cu, py::handle base, const Maybe &q_norm_w, const Maybe &k_norm_w, double eps,
                   const Maybe &inv_freq, bool interleaved, double amplitude) {
    const Device dev(k);
    dev.all(v, k_pages, v_pages, k_scale, v_scale, table, lens, q, cu, q_norm_w, k_norm_w, inv_freq);
    const trb_paged_t pool = make_pool(k_pages, v_pages, k_scale, v_scale);
    const trb_batch_t batch = make_batch(table, lens);
    need(k.dim() == 3 && k.size(1) == pool.hkv && k.size(2) == pool.d && v.sizes() == k.sizes(), "k and v must be [T, HKV, D] of the pool's heads");
    for (const Tensor *t : {&k, &v}) need(t->scalar_type() == at::kBFloat16 && t->stride(2) == 1, "k and v must be bfloat16 with a contiguous last dim");
    check_weight(q_norm_w, pool.d);
    check_weight(k_norm_w, pool.d);
    trb_paged_append_args_t a = {};
    a.k = ptr(k); a.v = ptr(v);
    a.k_row_stride = k.stride(0); a.k_head_stride = k.stride(1); a.v_row_stride = v.stride(0); a.v_head_stride = v.stride(1);
    need(k.size(0) <= 0x7fffffff, "too many rows");
    a.n_rows = (int32_t)k.size(0);
    if (!cu) {
        need(batch.n_seqs > 0 && a.n_rows % batch.n_seqs == 0, "without cu every sequence has the same number of rows");
        a.rows_per_seq = a.n_rows / batch.n_seqs;
    } else {
        need(cu->scalar_type() == at::kInt && cu->dim() == 1 && cu->size(0) == batch.n_seqs + 1 && cu->is_contiguous(), "cu must be int32 [B + 1]");
        a.cu = (const int32_t *)ptr(cu);
    }
    if (inv_freq) {
        need(inv_freq->scalar_type() == at::kDouble && inv_freq->dim() == 1 && inv_freq->is_contiguous() && inv_freq->size(0) <= pool.d,
             "inv_freq must be float64 [rotary_dim / 2]");
        a.rotary_dim = 2 * (int32_t)inv_freq->size(0);
        a.inv_freq = (const double *)ptr(inv_freq);
    }
    Maybe out;
    if (q) {
        need(q->dim() == 3 && q->size(0) == a.n_rows && q->size(2) == pool.d && q->scalar_type() == at::kBFloat16 && q->stride(2) == 1,
             "q must be bfloat16 [T, HQ, D] with a contiguous last dim");
        a.hq = (int32_t)q->size(1);
        a.q_row_stride = q->stride(0); a.q_head_stride = q->stride(1);
        out = at::empty(q->sizes(), q->options());
        a.q = ptr(q); a.q_out = ptr(out);
    }
    a.base = make_length(base, dev);
    if (a.n_rows == 0) return out;
    a.q_norm_w = ptr(q_norm_w); a.k_norm_w = ptr(k_norm_w); a.eps = (float)eps; a.interleaved = interleaved; a.amplitude = (float)amplitude;
    call(p_append(&pool, &batch, &a, dev.stream()), "trb_paged_append");
    return out;
}

Tensor attn_paged(const Tensor &q, const Tensor &k_pages, const Tensor &v_pages, const Tensor &table, const Tensor &lens, const Maybe &k_scale, const Maybe &v_scale,
                  const Maybe &prefix_table, py::handle prefix_len, const Maybe &gate, std::optional<double> scale, const Maybe &out_given) {
    const Device dev(q);
    dev.all(k_pages, v_pages, k_scale, v_scale, table, lens, prefix_table, gate, out_given);
    const trb_paged_t pool = make_pool(k_pages, v_pages, k_scale, v_scale);
    const trb_batch_t batch = make_batch(table, lens);
    need(q.dim() == 4 && q.size(0) == batch.n_seqs && q.size(3) == pool.d && q.scalar_type() == at::kBFloat16 && q.is_contiguous(),
         "q must be contiguous bf16 [B, M, HQ, D]");
    need(q.size(1) <= 1024 && q.size(2) <= 65536, "q has too many rows or heads");
    trb_attn_paged_args_t a = {};
    a.m = (int32_t)q.size(1); a.hq = (int32_t)q.size(2);
    a.prefix_len = make_length(prefix_len, dev);
    if (prefix_table) {
        need(prefix_table->scalar_type() == at::kInt && prefix_table->dim() == 1 && prefix_table->is_contiguous() && prefix_table->size(0) <= 0x7fffffff,
             "prefix_table must be contiguous int32 [P]");
        a.prefix_pages = (int32_t)prefix_table->size(0);
        if (!a.prefix_len.dev)
            need(a.prefix_len.host >= 0 && a.prefix_len.host <= (int64_t)a.prefix_pages * pool.page_size, "prefix_len exceeds the pages of prefix_table");
        if (!a.prefix_len.dev && pool.page_size > 0) a.prefix_pages = (int32_t)((a.prefix_len.host + pool.page_size - 1) / pool.page_size);      // the pages in use
        if (a.prefix_pages) a.prefix_table = (const int32_t *)ptr(prefix_table);
    } else {
        need(!a.prefix_len.dev && a.prefix_len.host == 0, "a prefix needs its prefix_table");
    }
    if (gate) {
        need(gate->sizes() == q.sizes() && gate->scalar_type() == at::kBFloat16 && gate->stride(3) == 1 &&
                 (batch.n_seqs == 1 || a.m == 1 || gate->stride(0) == a.m * gate->stride(1)),
             "gate must be a bf16 [B, M, HQ, D] view with equally spaced rows");
        // (the stride of a dim of size 1 means nothing)
        a.gate = ptr(gate); a.gate_row_stride = gate->stride(a.m == 1 ? 0 : 1); a.gate_head_stride = gate->stride(2);
    }
    Tensor out;
    if (out_given) {
        out = *out_given;
        need(out.sizes() == q.sizes() && out.scalar_type() == at::kBFloat16 && out.is_contiguous(), "out must be contiguous bf16 [B, M, HQ, D]");
    } else {
        out = at::empty(q.sizes(), q.options());
    }
    if (q.numel() == 0) return out;
    a.workspace_bytes = p_workspace(&pool, batch.n_seqs, a.m, a.hq, a.prefix_pages);
    need(a.workspace_bytes > 0, "unsupported geometry (heads, head dim, page size, rows or batch)");
    // a fresh buffer for every call: calls on other streams and in other captured graphs never share one
    const Tensor ws = at::empty({(int64_t)a.workspace_bytes}, q.options().dtype(at::kByte));
    a.q = ptr(q); a.out = ptr(out); a.workspace = ptr(ws);
    a.scale = (float)(scale ? *scale : 1.0 / std::sqrt((double)pool.d));
    call(p_attn(&pool, &batch, &a, dev.stream()), "trb_attn_paged");
    return out;
}

std::pair<Tensor, Tensor> spec_verify(const Tensor &probs, const Tensor &drafts, const Tensor &u, const Maybe &draft_probs, const Maybe &n_drafts, const Maybe &lens) {
    const Device dev(probs);
    dev.all(drafts, u, draft_probs, n_drafts, lens);
    trb_spec_verify_args_t a = {};
    const auto kind = probs.scalar_type();
    a.dtype = kind == at::kFloat ? TRB_DT_F32 : kind == at::kBFloat16 ? TRB_DT_BF16 : kind == at::kHalf ? TRB_DT_F16 : -1;
    need(probs.dim() == 3 && a.dtype >= 0 && probs.stride(2) == 1 && probs.size(1) >= 1, "probs must be fp32, bf16 or fp16 [B, K + 1, V] with a contiguous last dim");
    const int64_t b = probs.size(0), k = probs.size(1) - 1, v = probs.size(2);
    need(b <= 0x7fffffff && k <= 0x7fffffff && v <= 0x7fffffff, "probs is too large");
    need(drafts.dim() == 2 && drafts.size(0) == b && drafts.size(1) == k && drafts.scalar_type() == at::kLong && drafts.is_contiguous(), "drafts must be contiguous int64 [B, K]");
    need(u.dim() == 2 && u.size(0) == b && u.size(1) == k + 1 && u.scalar_type() == at::kFloat && u.is_contiguous(), "u must be contiguous float32 [B, K + 1]");
    if (draft_probs) {
        const Tensor &q = *draft_probs;
        need(q.dim() == 3 && q.size(0) == b && q.size(1) == k && q.size(2) == v && q.scalar_type() == kind && q.stride(2) == 1,
             "draft_probs must be [B, K, V] of the type of probs with a contiguous last dim");
        a.draft_probs = ptr(q); a.draft_seq_stride = q.stride(0); a.draft_row_stride = q.stride(1);
    }
    if (n_drafts)
        need(n_drafts->dim() == 1 && n_drafts->size(0) == b && n_drafts->scalar_type() == at::kInt && n_drafts->is_contiguous(), "n_drafts must be contiguous int32 [B]");
    if (lens) {
        need(lens->dim() == 1 && lens->size(0) == b && is_int(*lens) && lens->is_contiguous(), "lens must be contiguous int32 or int64 [B]");
        a.lens = ptr(lens); a.lens_width = width(*lens);
    }
    const Tensor tokens = at::empty({b, k + 1}, drafts.options()), n = at::empty({b}, drafts.options());
    if (b == 0) return {tokens, n};
    a.probs = ptr(probs); a.probs_seq_stride = probs.stride(0); a.probs_row_stride = probs.stride(1);
    a.drafts = (const int64_t *)ptr(drafts); a.u = (const float *)ptr(u); a.n_drafts = (const int32_t *)ptr(n_drafts);
    a.tokens = (int64_t *)ptr(tokens); a.n_accepted = (int64_t *)ptr(n);
    a.n_seqs = (int32_t)b; a.k = (int32_t)k; a.vocab = (int32_t)v;
    call(p_verify(&a, dev.stream()), "trb_spec_verify");
    return {tokens, n};
}

}  // namespace

PYBIND11_MODULE(_binding, m) {
    m.def("bind", [](uintptr_t append, uintptr_t workspace, uintptr_t attn, uintptr_t verify, py::object error) {
        p_append = (decltype(p_append))append; p_workspace = (decltype(p_workspace))workspace;
        p_attn = (decltype(p_attn))attn; p_verify = (decltype(p_verify))verify;
        on_error = error.release().ptr();
    });
    m.def("paged_append", &paged_append);
    m.def("attn_paged", &attn_paged);
    m.def("spec_verify", &spec_verify);
}
