// The launches of a prompt step's longest stretches, issued from native code: a norm; queries, keys and values, attention and output
// projection; gate, up and down; three recurrent mixers whole; and the launches for several continuations of one prompt (ops/branches.py) and for a
// cache in 8 bits (ops/cache_e4m3.py). The kernels and the library products are those that the Python entries of
// ops/kernels.py launch one by one, where a layer of few microseconds a kernel waits for its arguments to be made (a launch 4 to 5
// microseconds of host time beside 2 to 3 of the driver's own, a buffer 3 to 5; here 3 and 1).
// Every function looks at its tensors as those entries do and answers None, having done nothing, for what it does not take: the caller then
// goes their way, where the same condition is reported or another kernel chosen. Nothing is kept between calls but the entries' addresses.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <vector>

namespace {

typedef cudaStream_t Stream;
struct QkvArgs {   // TcQkvArgs of tc_gemm.cu
    const void* bias;
    const void* angles;
    const int *tok_pos, *tok_seq, *slots;
    void *q_out, *kv_base;
    const int* table;
    long long page_elems;
    int table_stride, n_heads, kv_heads, head_dim, write_cache;
    const float* inv_freq;
};

int (*add_rms_norm)(int, float*, const void*, const void*, void*, int, int, float, int, Stream);
int (*qkv_pairs_pays)(int, int, int, int);
int (*qkv_pairs)(const void*, int, const void*, int, int, int, const QkvArgs*, int*, Stream);
int (*prefill_tc)(const void*, void*, const int*, const int*, const int*, void*, const int*, long long, int, int, int, int, int, int, int, int,
                  float, int, int*, const float*, int, Stream);
int (*tc_is_persistent)(int, int, int);
int (*tc_gemm)(int, const void*, int, const void*, int, void*, int, int, int, int, int*, Stream);
int (*tc_gemm_tail)(const void*, int, const void*, int, void*, int, float*, int, int, int, int, int*, Stream);
int (*stabilized_gates)(const float*, int, const float*, float, const int*, const int*, int, float*, long long, long long, int, float*, float*,
                        float*, Stream);
int (*state_chunks)(const void*, int, const void*, int, const void*, int, const float*, const float*, const float*, const float*, int, const int*,
                    const int*, int, int, float*, long long, long long, long long, int, int, int, int, float, float*, long long, int, float*,
                    float*, Stream);
int (*gated_group_norm)(int, const float*, const void*, int, const void*, float, void*, int, int, int, int, int, int, const float*, const float*,
                        float, const float*, const void*, int, Stream);
int (*rope_cache_write)(int, const void*, const void*, int, const int*, const int*, const int*, const float*, int, int, void*, void*, const int*, long long, int,
                        int, int, int, int, int*, Stream);
int (*swiglu)(int, const void*, void*, int, int, Stream);
int (*causal_conv)(int, const void*, int, const float*, const float*, const int*, const int*, const int*, int, float*, long long, long long, int, int, int,
                   void*, int, int, Stream);
int (*row_chunks)(const void*, int, const void*, int, const void*, int, const float*, const float*, int, float, const float*, const int*, const int*, int, int,
                  float*, long long, long long, int, int, int, float, float*, long long, int, float*, Stream);
int (*attention_shared)(int, const void*, void*, const int*, const int*, const int*, const int*, const int*, const int*, const int*, int, int, int, int, int,
                        void*, const int*, long long, int, int, int, int, int, float, float*, float*, int*, const float*, int*, Stream);
int (*copy_pages)(void*, int, int, int, long long, long long, int, long long, long long, int, const int*, int, Stream);
int (*verify_drafts)(const float*, int, int, long long, const float*, long long, const int*, int, const int*, int, const float*, float, unsigned long long,
                     unsigned long long, const long long*, const int*, int*, int*, int, double*, void*, void*, int*, Stream);
int (*write_e4m3)(int, const void*, const void*, long long, const int*, const int*, const int*, const int*, const float*, int, int, void*, void*, float*,
                  const int*, long long, long long, int, int, int, int, int, int, int, int, int, int, int*, Stream);
int (*read_e4m3)(int, void*, long long, const int*, const int*, const int*, void*, float*, const int*, long long, long long, int, int, int, int, int, int, int,
                 int, int*, Stream);
int (*attention_e4m3_slots)(int, int, int);
int (*attention_e4m3)(int, const void*, void*, const int*, const int*, const int*, void*, float*, const int*, long long, long long, int, int, int, int, int, int,
                      int, int, int, int, int, int, int, int, float, int, int, float*, float*, int*, int*, Stream);
PyObject* kernel_error = nullptr;

const struct {
    const char* name;
    void** to;
} entries[] = {{"qf_add_rms_norm", (void**)&add_rms_norm}, {"qf_tc_gemm_qkv_pairs_pays", (void**)&qkv_pairs_pays},
               {"qf_tc_gemm_qkv_pairs", (void**)&qkv_pairs}, {"qf_attention_prefill_tc_ex", (void**)&prefill_tc},
               {"qf_tc_gemm_is_persistent", (void**)&tc_is_persistent}, {"qf_tc_gemm", (void**)&tc_gemm}, {"qf_tc_gemm_tail", (void**)&tc_gemm_tail},
               {"qf_stabilized_gates", (void**)&stabilized_gates}, {"qf_state_chunks", (void**)&state_chunks},
               {"qf_gated_group_norm", (void**)&gated_group_norm}, {"qf_rope_cache_write", (void**)&rope_cache_write}, {"qf_swiglu", (void**)&swiglu},
               {"qf_causal_conv", (void**)&causal_conv}, {"qf_row_chunks", (void**)&row_chunks},
               {"qf_attention_shared", (void**)&attention_shared}, {"qf_copy_pages", (void**)&copy_pages}, {"qf_verify_drafts", (void**)&verify_drafts},
               {"qf_rope_cache_write_e4m3", (void**)&write_e4m3}, {"qf_cache_read_e4m3", (void**)&read_e4m3}, {"qf_attention_e4m3", (void**)&attention_e4m3},
               {"qf_attention_e4m3_slots", (void**)&attention_e4m3_slots}};

// setup(KernelError, {name: address}): some of the entries, or more of them later.
PyObject* setup(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 2 || !PyDict_Check(args[1])) return PyErr_Format(PyExc_TypeError, "setup(error, addresses)");
    Py_INCREF(args[0]);
    Py_XDECREF(kernel_error);
    kernel_error = args[0];
    for (const auto& e : entries)
        if (PyObject* at = PyDict_GetItemString(args[1], e.name)) *e.to = PyLong_AsVoidPtr(at);
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
}

// ---- arguments
const at::Tensor* tensor(PyObject* o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }
long long number(PyObject* o) { return PyLong_AsLongLong(o); }

bool whole(const at::Tensor* t, at::ScalarType type) { return t && t->is_cuda() && t->scalar_type() == type && t->is_contiguous(); }
const int* ints(const at::Tensor* t) { return t->const_data_ptr<int>(); }
template <typename T = void> T* at_ptr(const at::Tensor& t) { return static_cast<T*>(t.data_ptr()); }
bool on16(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
// What `tc_gemm_takes` asks of a matrix: rows on 16-byte boundaries.
bool rows16(const at::Tensor* t) {
    return t && t->is_cuda() && t->scalar_type() == at::kBFloat16 && t->dim() == 2 && t->stride(1) == 1 && t->size(1) % 8 == 0 && t->stride(0) % 8 == 0 && on16(*t);
}
// Floats of a buffer, up to whole 256 bytes, where small buffers share an allocation. The large ones, rows in float32 and the chunks' records,
// have allocations of their own: a state space of 28 heads, microseconds of a pass, one allocation of parts on 16 bytes / on 256 / apart: 5,003
// tokens 203.5 / 196.8 / 195.5, 2,501 and 2,500 202.4 / 194.7 / 193.6 (a warp's loads meet a fifth line, its stores straddle sectors).
long long whole_lines(long long floats) { return (floats + 63) / 64 * 64; }
Stream stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

// What a launch was refused with; said once the interpreter's lock is held again.
struct Refusal {
    int code = 0;
    const char* what = nullptr;
    bool ok(int answer, const char* name) {
        if (answer == 0) return true;
        code = answer, what = name;
        return false;
    }
};
struct Unlocked {   // without the interpreter's lock, however the block is left
    PyThreadState* state = PyEval_SaveThread();
    ~Unlocked() { PyEval_RestoreThread(state); }
};
// What `launch` returns, run without the interpreter's lock, as the calls that it stands for are: a launch into a full queue and an allocation that
// asks the driver may block, and a server's other threads go on meanwhile. (The caller's frame holds the tensors.)
template <typename Launch> PyObject* unlocked(Launch launch) {
    Refusal refused;
    at::Tensor out;
    {
        Unlocked without;
        out = launch(refused);
    }
    if (!refused.what) return THPVariable_Wrap(std::move(out));
    if (refused.code == 801) return PyErr_Format(kernel_error, "%s: the driver offers no tensor-map encoder (cuTensorMapEncodeTiled)", refused.what);
    return PyErr_Format(kernel_error, "%s: CUDA error %d at launch", refused.what, refused.code);
}

// rms_norm(hidden, delta or None, weight, eps) -> out: `add_rms_norm` into a new tensor.
PyObject* rms_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 4) return PyErr_Format(PyExc_TypeError, "rms_norm: 4 arguments");
    const at::Tensor *hidden = tensor(args[0]), *delta = tensor(args[1]), *weight = tensor(args[2]);
    if (!add_rms_norm || !whole(hidden, at::kFloat) || hidden->dim() != 2 || (!delta && args[1] != Py_None) || !weight ||
        (weight->scalar_type() != at::kBFloat16 && weight->scalar_type() != at::kFloat) || !whole(weight, weight->scalar_type()) ||
        weight->dim() != 1 || weight->size(0) != hidden->size(1) || (delta && (!whole(delta, weight->scalar_type()) || delta->sizes() != hidden->sizes())))
        Py_RETURN_NONE;
    const double eps = PyFloat_AsDouble(args[3]);
    if (PyErr_Occurred()) return nullptr;
    return unlocked([&](Refusal& refused) {
        at::Tensor out = at::empty(hidden->sizes(), weight->options());
        if (!refused.ok(add_rms_norm(weight->scalar_type() == at::kBFloat16, at_ptr<float>(*hidden), delta ? delta->data_ptr() : nullptr, weight->data_ptr(),
                             out.data_ptr(), (int)hidden->size(0), (int)hidden->size(1), (float)eps, 0, stream()), "add_rms_norm"))
            return at::Tensor();
        return out;
    });
    END_HANDLE_TH_ERRORS
}

// prompt_attention(x, qkv_weight, bias, inv_freq, o_weight, tok_seq, tok_pos, slots, cu_q, storage, table, err,
//                  n_heads, kv_heads, head_dim, n_seqs, max_q_len, max_kv_len, scale, window, write_cache) -> out
// `qkv_product` where it is the faster way, else the library's product and `rope_cache_write`; `attention_prefill_tc`; the output projection by the library.
PyObject* prompt_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 21) return PyErr_Format(PyExc_TypeError, "prompt_attention: 21 arguments");
    const at::Tensor *x = tensor(args[0]), *w = tensor(args[1]), *bias = tensor(args[2]), *freq = tensor(args[3]), *o = tensor(args[4]);
    const at::Tensor *seq = tensor(args[5]), *pos = tensor(args[6]), *slots = tensor(args[7]), *cu = tensor(args[8]), *storage = tensor(args[9]);
    const at::Tensor *table = tensor(args[10]), *err = tensor(args[11]);
    const long long heads = number(args[12]), kv = number(args[13]), d = number(args[14]), n_seqs = number(args[15]), longest = number(args[16]);
    const long long keys = number(args[17]), window = number(args[19]), write = number(args[20]);
    const double scale = PyFloat_AsDouble(args[18]);
    if (PyErr_Occurred()) return nullptr;
    if (!qkv_pairs_pays || !qkv_pairs || !rope_cache_write || !prefill_tc || !rows16(x) || !rows16(w) || (!bias && args[2] != Py_None) || (!freq && args[3] != Py_None) ||
        !o || !o->is_cuda() || o->scalar_type() != at::kBFloat16 || o->dim() != 2 || o->size(1) != heads * d || !whole(seq, at::kInt) ||
        !whole(pos, at::kInt) || !whole(slots, at::kInt) || !whole(cu, at::kInt) || !whole(storage, at::kBFloat16) || !table || !table->is_cuda() ||
        table->scalar_type() != at::kInt || !whole(err, at::kInt))
        Py_RETURN_NONE;
    const long long m = x->size(0), k = x->size(1), page = storage->stride(0);
    if ((d != 64 && d != 128) || heads <= 0 || kv <= 0 || heads % kv || w->size(0) != (heads + 2 * kv) * d || w->size(1) != k ||
        (bias && (!whole(bias, at::kBFloat16) || bias->numel() != w->size(0) || !on16(*bias))) ||
        (freq && (!whole(freq, at::kFloat) || 2 * freq->numel() > d)) || storage->dim() < 2 || !on16(*storage) || page % 8 ||
        page != 2 * kv * storage->size(-2) * d || seq->numel() != m || pos->numel() != m || slots->numel() < n_seqs || cu->numel() < n_seqs + 1)
        Py_RETURN_NONE;
    return unlocked([&](Refusal& refused) {
        at::Tensor q = at::empty({m, heads * d}, x->options()), attended = at::empty({m, heads * d}, x->options());
        const Stream s = stream();
        const float* angles = freq ? freq->const_data_ptr<float>() : nullptr;
        if ((!freq || 2 * freq->numel() == d) && qkv_pairs_pays((int)m, (int)w->size(0), (int)k, (int)d)) {
            const QkvArgs a = {bias ? bias->data_ptr() : nullptr, nullptr, ints(pos), ints(seq), ints(slots), q.data_ptr(), storage->data_ptr(), ints(table), page,
                               (int)table->stride(0), (int)heads, (int)kv, (int)d, write != 0, angles};
            if (!refused.ok(qkv_pairs(x->data_ptr(), (int)x->stride(0), w->data_ptr(), (int)w->stride(0), (int)m, (int)k, &a, at_ptr<int>(*err), s), "qkv_product")) return at::Tensor();
        } else {
            at::Tensor qkv = at::linear(*x, *w);
            if (!refused.ok(rope_cache_write(1, qkv.data_ptr(), bias ? bias->data_ptr() : nullptr, (int)qkv.stride(0), ints(seq), ints(pos), ints(slots), angles,
                                     freq ? (int)(2 * freq->numel()) : 0, (int)heads, q.data_ptr(), storage->data_ptr(), ints(table), page, (int)table->stride(0),
                                     (int)kv, (int)d, write != 0, (int)m, at_ptr<int>(*err), s), "rope_cache_write"))
                return at::Tensor();
        }
        if (!refused.ok(prefill_tc(q.data_ptr(), attended.data_ptr(), ints(cu), ints(pos), ints(slots), storage->data_ptr(), ints(table), page, (int)table->stride(0),
                           (int)kv, (int)d, (int)heads, (int)n_seqs, (int)m, (int)longest, (int)keys, (float)scale, (int)window, at_ptr<int>(*err), nullptr,
                           0, s), "attention_prefill_tc"))
            return at::Tensor();
        return at::linear(attended, *o);
    });
    END_HANDLE_TH_ERRORS
}

// gated_feed_forward(x, gate_up, down, err) -> out: `tc_gemm` with the gate in its epilogue where it has tiles for every pair of SMs, else the
// library's product and `swiglu`; down by the library.
PyObject* gated_feed_forward(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 4) return PyErr_Format(PyExc_TypeError, "gated_feed_forward: 4 arguments");
    const at::Tensor *x = tensor(args[0]), *gate_up = tensor(args[1]), *down = tensor(args[2]), *err = tensor(args[3]);
    if (!tc_gemm || !tc_is_persistent || !swiglu || !rows16(x) || !rows16(gate_up) || !down || !down->is_cuda() || down->scalar_type() != at::kBFloat16 || down->dim() != 2 ||
        !whole(err, at::kInt))
        Py_RETURN_NONE;
    const long long m = x->size(0), k = x->size(1), inter = gate_up->size(0) / 2;
    if (gate_up->size(0) != 2 * inter || inter % 8 || gate_up->size(1) != k || down->size(1) != inter) Py_RETURN_NONE;
    return unlocked([&](Refusal& refused) {
        at::Tensor act = at::empty({m, inter}, x->options());
        if (tc_is_persistent(1, (int)m, (int)(2 * inter))) {
            if (!refused.ok(tc_gemm(1, x->data_ptr(), (int)x->stride(0), gate_up->data_ptr(), (int)gate_up->stride(0), act.data_ptr(), (int)inter, (int)m, (int)(2 * inter),
                            (int)k, at_ptr<int>(*err), stream()), "tc_gemm"))
                return at::Tensor();
        } else {
            at::Tensor both = at::linear(*x, *gate_up);
            if (!refused.ok(swiglu(1, both.data_ptr(), act.data_ptr(), (int)m, (int)inter, stream()), "swiglu")) return at::Tensor();
        }
        return at::linear(act, *down);
    });
    END_HANDLE_TH_ERRORS
}

// matrix_memory(x, joint, gate_bias, norm, o_weight, state, cu_q, slots, err, heads, dim, vdim, max_q_len, records, each, s_offset, n_offset,
//               m_offset, cap, eps, floor) -> out: `tc_gemm_tail`, `stabilized_gates`, `state_chunks`, `gated_group_norm` and the output
// projection by the library. The caller has found the tail and the chunks to be the ways to go; joint is [q | k | v | gate | i | f].
PyObject* matrix_memory(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 21) return PyErr_Format(PyExc_TypeError, "matrix_memory: 21 arguments");
    const at::Tensor *x = tensor(args[0]), *joint = tensor(args[1]), *gate_bias = tensor(args[2]), *norm = tensor(args[3]), *o = tensor(args[4]);
    const at::Tensor *state = tensor(args[5]), *cu = tensor(args[6]), *slots = tensor(args[7]), *err = tensor(args[8]);
    long long v[9];
    for (int i = 0; i < 9; ++i) v[i] = number(args[9 + i]);
    const long long h = v[0], d = v[1], vd = v[2], longest = v[3], records = v[4], each = v[5], s_at = v[6], n_at = v[7], m_at = v[8];
    const double cap = PyFloat_AsDouble(args[18]), eps = PyFloat_AsDouble(args[19]), floor_add = PyFloat_AsDouble(args[20]);
    if (PyErr_Occurred()) return nullptr;
    if (!tc_gemm_tail || !stabilized_gates || !state_chunks || !gated_group_norm || !rows16(x) || !rows16(joint) || !whole(gate_bias, at::kFloat) ||
        !whole(norm, at::kBFloat16) || !o || !o->is_cuda() || o->scalar_type() != at::kBFloat16 || o->dim() != 2 || !whole(state, at::kFloat) || state->dim() != 2 ||
        !whole(cu, at::kInt) || !whole(slots, at::kInt) || !whole(err, at::kInt))
        Py_RETURN_NONE;
    const long long t = x->size(0), main = 2 * h * (d + vd), inner = h * vd, seqs = cu->numel() - 1, floats = state->size(1);
    if (h <= 0 || (d != 64 && d != 128) || vd <= 0 || vd % 64 || seqs <= 0 || seqs > 65535 || inner / 64 > 65535 || joint->size(0) != main + 2 * h ||
        joint->size(1) != x->size(1) || gate_bias->numel() != 2 * h || norm->numel() != inner || o->size(1) != inner || slots->numel() < seqs ||
        s_at < 0 || s_at + h * d * vd > floats || n_at < 0 || n_at + h * d > floats || m_at < 0 || m_at + h > floats || records <= 0 || each < 0)
        Py_RETURN_NONE;
    return unlocked([&](Refusal& refused) {
        at::Tensor proj = at::empty({t, main}, x->options()), out = at::empty({t, inner}, x->options());
        const long long gates = whole_lines(t * h);
        at::Tensor room = at::empty({6 * gates}, state->options()), made = at::empty({t * inner}, state->options());
        at::Tensor kept = at::empty({records * h * (d * vd + d + 1) + (each ? seqs * h * (d * vd + d) : 0)}, state->options());
        float* decay = at_ptr<float>(room);
        float *take = decay + gates, *floor = take + gates, *nq = floor + gates, *pre = nq + gates, *y = at_ptr<float>(made), *scratch = at_ptr<float>(kept);
        unsigned char* p = at_ptr<unsigned char>(proj);
        const unsigned char *q = p, *k = p + 2 * h * d, *vals = p + 4 * h * d, *gate = vals + 2 * inner;
        const Stream s = stream();
        const long long slot = state->stride(0);
        if (!refused.ok(tc_gemm_tail(x->data_ptr(), (int)x->stride(0), joint->data_ptr(), (int)joint->stride(0), p, (int)main, pre, (int)t, (int)main, (int)(2 * h),
                             (int)x->size(1), at_ptr<int>(*err), s), "tc_gemm_tail") ||
            !refused.ok(stabilized_gates(pre, (int)(2 * h), gate_bias->const_data_ptr<float>(), (float)cap, ints(cu), ints(slots), (int)seqs, at_ptr<float>(*state), slot,
                                 m_at, (int)h, decay, take, floor, s), "stabilized_gates") ||
            !refused.ok(state_chunks(q, (int)main, k, (int)main, vals, (int)main, decay, take, nullptr, nullptr, (int)h, ints(cu), ints(slots), (int)seqs, (int)longest,
                             at_ptr<float>(*state), slot, s_at, n_at, (int)h, (int)h, (int)d, (int)vd, (float)std::pow((double)d, -0.5), scratch, records,
                             (int)each, y, nq, s), "state_chunks") ||
            !refused.ok(gated_group_norm(1, y, gate, (int)main, norm->data_ptr(), (float)eps, out.data_ptr(), (int)t, (int)inner, (int)h, (int)h, 0, 0, nq, floor,
                                 (float)floor_add, nullptr, nullptr, 0, s), "gated_group_norm"))
            return at::Tensor();
        return at::linear(out, *o);
    });
    END_HANDLE_TH_ERRORS
}

// state_space(x, joint, conv_weight, conv_bias, dt_bias, rate_log, skip, norm, o_weight, state, cu_q, tok_seq, slots, err, heads, vdim, state_size,
//             groups, norm_parts, max_q_len, records, each, s_offset, conv_offset, eps) -> out: `tc_gemm_tail`, `causal_conv_silu`,
// `state_chunks` with the gates formed inside, `gated_group_norm` and the output projection by the library; joint is [z | x | B | C | dt].
PyObject* state_space(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 25) return PyErr_Format(PyExc_TypeError, "state_space: 25 arguments");
    const at::Tensor* t[14];
    for (int i = 0; i < 14; ++i) t[i] = tensor(args[i]);
    const at::Tensor *x = t[0], *joint = t[1], *conv_w = t[2], *conv_b = t[3], *dt_bias = t[4], *rate = t[5], *skip = t[6], *norm = t[7], *o = t[8], *state = t[9];
    const at::Tensor *cu = t[10], *seq = t[11], *slots = t[12], *err = t[13];
    long long v[10];
    for (int i = 0; i < 10; ++i) v[i] = number(args[14 + i]);
    const long long h = v[0], vd = v[1], d = v[2], groups = v[3], parts = v[4], longest = v[5], records = v[6], each = v[7], s_at = v[8], conv_at = v[9];
    const double eps = PyFloat_AsDouble(args[24]);
    if (PyErr_Occurred()) return nullptr;
    if (!tc_gemm_tail || !causal_conv || !state_chunks || !gated_group_norm || !rows16(x) || !rows16(joint) || !whole(conv_w, at::kFloat) || conv_w->dim() != 2 ||
        !whole(conv_b, at::kFloat) || !whole(dt_bias, at::kFloat) || !whole(rate, at::kFloat) || !whole(skip, at::kFloat) || !whole(norm, at::kBFloat16) || !o ||
        !o->is_cuda() || o->scalar_type() != at::kBFloat16 || o->dim() != 2 || !whole(state, at::kFloat) || state->dim() != 2 || !whole(cu, at::kInt) ||
        !whole(seq, at::kInt) || !whole(slots, at::kInt) || !whole(err, at::kInt))
        Py_RETURN_NONE;
    const long long m = x->size(0), inner = h * vd, channels = inner + 2 * groups * d, main = inner + channels, seqs = cu->numel() - 1, taps = conv_w->size(1);
    if (h <= 0 || (d != 64 && d != 128) || vd <= 0 || vd % 64 || groups <= 0 || h % groups || parts <= 0 || inner % parts || seqs <= 0 || seqs > 65535 ||
        inner / 64 > 65535 || joint->size(0) != main + h || joint->size(1) != x->size(1) || conv_w->size(0) != channels || taps < 1 || taps > 16 ||
        conv_b->numel() != channels || dt_bias->numel() != h || rate->numel() != h || skip->numel() != h || norm->numel() != inner || o->size(1) != inner ||
        seq->numel() != m || slots->numel() < seqs || s_at < 0 || s_at + h * d * vd > state->size(1) || conv_at < 0 ||
        conv_at + (taps - 1) * channels > state->size(1) || records <= 0 || each < 0)
        Py_RETURN_NONE;
    return unlocked([&](Refusal& refused) {
        at::Tensor made = at::empty({m, main}, x->options()), mixed = at::empty({m, channels}, x->options()), out = at::empty({m, inner}, x->options());
        at::Tensor pre = at::empty({m * h}, state->options()), sums = at::empty({m * inner}, state->options());
        at::Tensor kept = at::empty({records * h * (d * vd + d + 1) + (each ? seqs * h * (d * vd + d) : 0)}, state->options());
        float *dt = at_ptr<float>(pre), *y = at_ptr<float>(sums), *scratch = at_ptr<float>(kept);
        const unsigned char *z = at_ptr<unsigned char>(made), *vals = at_ptr<unsigned char>(mixed), *k = vals + 2 * inner, *q = k + 2 * groups * d;
        const Stream s = stream();
        const long long slot = state->stride(0);
        if (!refused.ok(tc_gemm_tail(x->data_ptr(), (int)x->stride(0), joint->data_ptr(), (int)joint->stride(0), made.data_ptr(), (int)main, dt, (int)m, (int)main, (int)h,
                             (int)x->size(1), at_ptr<int>(*err), s), "tc_gemm_tail") ||
            !refused.ok(causal_conv(1, z + 2 * inner, (int)main, conv_w->const_data_ptr<float>(), conv_b->const_data_ptr<float>(), ints(cu), ints(seq), ints(slots), (int)seqs,
                            at_ptr<float>(*state), slot, conv_at, (int)taps, (int)m, (int)channels, mixed.data_ptr(), 0, 0, s), "causal_conv_silu") ||
            !refused.ok(state_chunks(q, (int)channels, k, (int)channels, vals, (int)channels, dt, nullptr, dt_bias->const_data_ptr<float>(), rate->const_data_ptr<float>(),
                             (int)h, ints(cu), ints(slots), (int)seqs, (int)longest, at_ptr<float>(*state), slot, s_at, -1, (int)h, (int)groups, (int)d, (int)vd, 1.f,
                             scratch, records, (int)each, y, nullptr, s), "state_chunks") ||
            !refused.ok(gated_group_norm(1, y, z, (int)main, norm->data_ptr(), (float)eps, out.data_ptr(), (int)m, (int)inner, (int)parts, (int)h, 1, 1, nullptr, nullptr, 0.f,
                                 skip->const_data_ptr<float>(), vals, (int)channels, s), "gated_group_norm"))
            return at::Tensor();
        return at::linear(out, *o);
    });
    END_HANDLE_TH_ERRORS
}

// gated_linear_attention(x, joint, a2, a2_bias, norm, o_weight, state, cu_q, slots, heads, dim, vdim, max_q_len, records, each, inv_tau, eps) -> out:
// the library's product of [q | k | v | gate | middle] and of the middle in float32, `row_chunks`, `gated_group_norm` and the output projection.
PyObject* gated_linear_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 17) return PyErr_Format(PyExc_TypeError, "gated_linear_attention: 17 arguments");
    const at::Tensor* t[9];
    for (int i = 0; i < 9; ++i) t[i] = tensor(args[i]);
    const at::Tensor *x = t[0], *joint = t[1], *a2 = t[2], *bias = t[3], *norm = t[4], *o = t[5], *state = t[6], *cu = t[7], *slots = t[8];
    long long v[6];
    for (int i = 0; i < 6; ++i) v[i] = number(args[9 + i]);
    const long long h = v[0], d = v[1], vd = v[2], longest = v[3], records = v[4], each = v[5];
    const double inv_tau = PyFloat_AsDouble(args[15]), eps = PyFloat_AsDouble(args[16]);
    if (PyErr_Occurred()) return nullptr;
    if (!row_chunks || !gated_group_norm || !rows16(x) || !rows16(joint) || !rows16(a2) || !whole(bias, at::kFloat) || !whole(norm, at::kBFloat16) || !o ||
        !o->is_cuda() || o->scalar_type() != at::kBFloat16 || o->dim() != 2 || !whole(state, at::kFloat) || state->dim() != 2 || !whole(cu, at::kInt) ||
        !whole(slots, at::kInt))
        Py_RETURN_NONE;
    const long long m = x->size(0), inner = h * vd, main = 2 * h * d + 2 * inner, rank = a2->size(1), seqs = cu->numel() - 1, wide = main + rank;
    if (h <= 0 || d != 64 || vd <= 0 || vd % 64 || vd > 512 || seqs <= 0 || seqs > 65535 || inner / 64 > 65535 || joint->size(0) != wide ||
        joint->size(1) != x->size(1) || a2->size(0) != h * d || bias->numel() != h * d || norm->numel() != inner || o->size(1) != inner ||
        slots->numel() < seqs || h * d * vd > state->size(1) || records <= 0 || each < 0)
        Py_RETURN_NONE;
    return unlocked([&](Refusal& refused) {
        at::Tensor all = at::linear(*x, *joint), pre = at::mm(all.narrow(1, main, rank), a2->t(), at::kFloat), out = at::empty({m, inner}, x->options());
        TORCH_CHECK(on16(all) && on16(pre) && pre.is_contiguous(), "gated_linear_attention: the allocator's rows begin on no 16-byte boundary");
        at::Tensor sums = at::empty({m * inner}, state->options());
        at::Tensor kept = at::empty({records * h * (d * vd + d) + (each ? seqs * h * d * vd : 0) + m * h * d}, state->options());
        float *y = at_ptr<float>(sums), *scratch = at_ptr<float>(kept);
        const unsigned char *q = at_ptr<unsigned char>(all), *k = q + 2 * h * d, *vals = k + 2 * h * d, *gate = vals + 2 * inner;
        const Stream s = stream();
        if (!refused.ok(row_chunks(q, (int)wide, k, (int)wide, vals, (int)wide, pre.const_data_ptr<float>(), bias->const_data_ptr<float>(), 2, (float)inv_tau, nullptr, ints(cu),
                           ints(slots), (int)seqs, (int)longest, at_ptr<float>(*state), state->stride(0), 0, (int)h, (int)d, (int)vd, (float)std::pow((double)d, -0.5),
                           scratch, records, (int)each, y, s), "row_chunks") ||
            !refused.ok(gated_group_norm(1, y, gate, (int)wide, norm->data_ptr(), (float)eps, out.data_ptr(), (int)m, (int)inner, (int)h, (int)h, 1, 0, nullptr, nullptr, 0.f,
                                 nullptr, nullptr, 0, s), "gated_group_norm"))
            return at::Tensor();
        return at::linear(out, *o);
    });
    END_HANDLE_TH_ERRORS
}

// ---- several continuations of one prompt: the launches of ops/branches.py, whose checks stand there. These answer the entry's code, None for what they do
// not take (the caller then checks and launches itself). Host time of a call, microseconds, there / here: attention of two sequences 17 / 7.8, four
// drafts of one 16 / 6.3, a page forked seven times 10 / 4.1.
bool on(const at::Tensor* t, at::ScalarType type, int device) { return t && t->is_cuda() && t->scalar_type() == type && t->get_device() == device; }
bool dense(const at::Tensor* t, at::ScalarType type, int device) { return on(t, type, device) && t->is_contiguous(); }
template <typename Launch> PyObject* code_of(Launch launch) {
    int code;
    {
        Unlocked without;
        code = launch();
    }
    return PyLong_FromLong(code);
}

// attention_shared(q, out, cu_q, tok_pos, slots, storage, table, share (five tensors), part_o, part_ml, part_n, sinks or None, err, page_elems, kv_heads,
//                  head_dim, n_heads, n_seqs, scale, groups, most_pages, units, tiles, most_shared, most_own)
PyObject* shared_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 29) return PyErr_Format(PyExc_TypeError, "attention_shared: 29 arguments");
    const at::Tensor* t[17];
    for (int i = 0; i < 17; ++i) t[i] = tensor(args[i]);
    const at::Tensor *q = t[0], *out = t[1], *cu = t[2], *pos = t[3], *slots = t[4], *storage = t[5], *table = t[6], *sinks = t[15], *err = t[16];
    const long long page = number(args[17]), kv = number(args[18]), d = number(args[19]), heads = number(args[20]), seqs = number(args[21]);
    const double scale = PyFloat_AsDouble(args[22]);
    const long long groups = number(args[23]), most_pages = number(args[24]), units = number(args[25]), tiles = number(args[26]);
    const long long shared = number(args[27]), own = number(args[28]);
    if (PyErr_Occurred()) return nullptr;
    const int device = c10::cuda::current_device();
    const at::ScalarType type = q ? q->scalar_type() : at::kInt;
    bool takes = attention_shared && (type == at::kBFloat16 || type == at::kFloat) && dense(q, type, device) && dense(out, type, device) &&
                 dense(cu, at::kInt, device) && dense(pos, at::kInt, device) && dense(slots, at::kInt, device) && on(storage, type, device) &&
                 on(table, at::kInt, device) && dense(err, at::kInt, device) && (args[15] == Py_None || dense(sinks, at::kFloat, device)) &&
                 on(t[12], at::kFloat, device) && on(t[13], at::kFloat, device) && on(t[14], at::kInt, device);
    for (int i = 7; takes && i < 12; ++i) takes = on(t[i], at::kInt, device);
    if (!takes || d <= 0 || d > 256 || kv <= 0 || heads <= 0 || heads % kv || seqs <= 0 || seqs > 2048 || t[7]->numel() != seqs || slots->numel() != seqs ||
        cu->numel() != seqs + 1 || pos->numel() != seqs || q->dim() != 2 || q->size(0) != seqs || q->size(1) != heads * d || out->sizes() != q->sizes() ||
        storage->dim() != 5 || storage->size(1) != 2 || storage->size(2) != kv || storage->size(3) != 64 || storage->size(4) != d || page < 2 * kv * 64 * d ||
        storage->stride(1) != kv * 64 * d || storage->stride(2) != 64 * d || storage->stride(3) != d || storage->stride(4) != 1 || table->dim() != 2 ||
        table->stride(1) != 1 || most_pages > table->size(1) || (sinks && sinks->numel() != heads) || shared < 0 || own <= 0 || units <= 0 || tiles < 0 ||
        t[12]->numel() < seqs * heads * (shared + own) * d || t[13]->numel() < seqs * heads * (shared + own) * 2 || t[14]->numel() < seqs ||
        (type == at::kBFloat16 && (!on16(*q) || !on16(*storage) || page % d)))
        Py_RETURN_NONE;
    return code_of([&] {
        return attention_shared(type == at::kBFloat16, q->data_ptr(), out->data_ptr(), ints(pos), ints(slots), ints(t[7]), ints(t[8]), ints(t[9]), ints(t[10]),
                                ints(t[11]), (int)groups, (int)units, (int)tiles, (int)shared, (int)own, storage->data_ptr(), ints(table), page,
                                (int)table->stride(0), (int)kv, (int)d, (int)heads, (int)seqs, (float)scale, at_ptr<float>(*t[12]), at_ptr<float>(*t[13]),
                                at_ptr<int>(*t[14]), sinks ? sinks->const_data_ptr<float>() : nullptr, at_ptr<int>(*err), stream());
    });
    END_HANDLE_TH_ERRORS
}

// verify_drafts(target, draft or None, drafted, first, uniforms, seq_ids, steps, accepted, tokens, held, counters, temperature, seed, redraw_seed,
//               row_chunk, race_chunk): draws, and the greedy choice at a temperature of 0 or less. Chunks: those of a row's statistics, and of a row's race.
PyObject* drafts_verified(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 16) return PyErr_Format(PyExc_TypeError, "verify_drafts: 16 arguments");
    const at::Tensor* t[11];
    for (int i = 0; i < 11; ++i) t[i] = tensor(args[i]);
    const at::Tensor *target = t[0], *draft = t[1], *drafted = t[2], *first = t[3], *uniforms = t[4], *ids = t[5], *steps = t[6], *accepted = t[7], *tokens = t[8];
    const double temperature = PyFloat_AsDouble(args[11]);
    const unsigned long long seed = PyLong_AsUnsignedLongLongMask(args[12]), redraw_seed = PyLong_AsUnsignedLongLongMask(args[13]);
    const long long row_chunk = number(args[14]), race_chunk = number(args[15]);
    if (PyErr_Occurred()) return nullptr;
    const int device = c10::cuda::current_device();
    const bool draws = temperature > 0;
    if (!verify_drafts || !on(target, at::kFloat, device) || (!draft && args[1] != Py_None) || !dense(drafted, at::kInt, device) || !dense(first, at::kInt, device) ||
        !dense(uniforms, at::kFloat, device) || !dense(accepted, at::kInt, device) || !dense(tokens, at::kInt, device) || !on(t[9], at::kDouble, device) ||
        !on(t[10], at::kInt, device) || target->dim() != 2 || target->stride(1) != 1 || target->size(1) <= 0 || tokens->dim() != 2 || row_chunk <= 0 || race_chunk <= 0 ||
        (draws && (!dense(ids, at::kLong, device) || !dense(steps, at::kInt, device))))
        Py_RETURN_NONE;
    const long long rows = target->size(0), vocab = target->size(1), entries = accepted->numel(), total = drafted->numel();
    const bool used = draws && draft && total > 0;
    if (rows <= 0 || entries <= 0 || first->numel() != entries + 1 || tokens->size(0) != entries || tokens->size(1) < 1 || total < rows - entries ||
        entries > 65535 || rows + total > 65535 || (draws && (uniforms->numel() != total || ids->numel() != entries || steps->numel() != entries)) ||
        (draws && draft && (!on(draft, at::kFloat, device) || draft->dim() != 2 || draft->size(0) != total || draft->size(1) != vocab)) ||
        (used && draft->stride(1) != 1))
        Py_RETURN_NONE;
    const long long row_chunks = (rows + (used ? total : 0)) * ((vocab + row_chunk - 1) / row_chunk), races = entries * ((vocab + race_chunk - 1) / race_chunk);
    if (t[9]->numel() < 2 * (row_chunks + races) || t[10]->numel() < entries) Py_RETURN_NONE;
    double* held = at_ptr<double>(*t[9]);
    return code_of([&] {
        return verify_drafts(target->const_data_ptr<float>(), (int)rows, (int)vocab, target->stride(0), used ? draft->const_data_ptr<float>() : nullptr,
                             used ? draft->stride(0) : 0, ints(drafted), (int)total, ints(first), (int)entries, uniforms->const_data_ptr<float>(),
                             draws ? (float)temperature : 0.f, seed, redraw_seed, draws ? reinterpret_cast<const long long*>(ids->const_data_ptr<int64_t>()) : nullptr,
                             draws ? ints(steps) : nullptr, at_ptr<int>(*accepted), at_ptr<int>(*tokens), (int)tokens->size(1) - 1, held, held + row_chunks,
                             held + 2 * row_chunks, at_ptr<int>(*t[10]), stream());
    });
    END_HANDLE_TH_ERRORS
}

// copy_pages(storage, moves): a list of tuples of three or two whole numbers.
PyObject* pages_copied(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 2) return PyErr_Format(PyExc_TypeError, "copy_pages: 2 arguments");
    const at::Tensor* storage = tensor(args[0]);
    if (!copy_pages || !storage || !storage->is_cuda() || storage->get_device() != c10::cuda::current_device() || !PyList_CheckExact(args[1])) Py_RETURN_NONE;
    const int dims = (int)storage->dim();
    if (dims < 2) Py_RETURN_NONE;
    const long long entries = storage->size(0), pages = storage->size(1), item = (long long)storage->element_size();
    const long long rows = dims >= 4 ? storage->size(dims - 2) : 1, width = dims >= 4 ? storage->size(dims - 1) : dims == 3 ? storage->size(2) : 1;
    long long page = 1, segments = 1;
    for (int i = dims - 1; i >= 2; --i) {
        if (storage->size(i) != 1 && storage->stride(i) != page) Py_RETURN_NONE;
        page *= storage->size(i);
        if (i < dims - 2) segments *= storage->size(i);
    }
    const long long apart = entries > 1 ? storage->stride(0) : 0, step = pages > 1 ? storage->stride(1) : 0;
    if (page <= 0 || entries <= 0 || entries > 65535 || pages <= 0 || pages > INT_MAX || rows > INT_MAX || segments > INT_MAX || (pages > 1 && step < page) ||
        (entries > 1 && apart < page) || (entries > 1 && pages > 1 && apart < (pages - 1) * step + page && step < (entries - 1) * apart + page))
        Py_RETURN_NONE;
    const Py_ssize_t count = PyList_GET_SIZE(args[1]);
    if (count <= 0 || count > 1 << 20) Py_RETURN_NONE;
    std::vector<int> moves((size_t)count * 3);
    for (Py_ssize_t i = 0; i < count; ++i) {
        PyObject* move = PyList_GET_ITEM(args[1], i);
        if (!PyTuple_CheckExact(move)) Py_RETURN_NONE;
        const Py_ssize_t size = PyTuple_GET_SIZE(move);
        if ((size != 2 && size != 3) || size != PyTuple_GET_SIZE(PyList_GET_ITEM(args[1], 0))) Py_RETURN_NONE;
        for (int e = 0; e < 3; ++e) {
            long long v = rows;
            int over = 0;
            if (e < size) {
                PyObject* o = PyTuple_GET_ITEM(move, e);
                if (!PyLong_CheckExact(o)) Py_RETURN_NONE;
                v = PyLong_AsLongLongAndOverflow(o, &over);
            }
            if (over || v < INT_MIN || v > INT_MAX) Py_RETURN_NONE;
            moves[i * 3 + e] = (int)v;
        }
    }
    unsigned char* base = at_ptr<unsigned char>(*storage);
    const long long row = width * item, low = (long long)reinterpret_cast<uintptr_t>(base) | row | apart * item | step * item;
    const int unit = !(low & 15) ? 16 : !(low & 3) ? 4 : !(low & 1) ? 2 : 1;
    return code_of([&] {
        return copy_pages(base, (int)entries, (int)pages, (int)rows, apart * item, step * item, (int)segments, rows * row, row, unit, moves.data(), (int)count, stream());
    });
    END_HANDLE_TH_ERRORS
}

// ---- a cache in 8 bits: the launches of ops/cache_e4m3.py, in the same manner (a call on one sequence, back to back, microseconds, there / here: a token written 13.4 / 4.2, pages read 14.3 / 3.9).
// A site's place: the tuple (codes, scales, table, page_bytes, page_scales, table_stride, columns, n_slots, kv_heads, head_dim) of its checked tensors.
struct Place {
    void* codes;
    float* scales;
    const int* table;
    long long page_bytes, page_scales;
    int table_stride, columns, n_slots, kv_heads, head_dim;
};
bool placed(PyObject* o, Place& p) {
    if (!PyTuple_CheckExact(o) || PyTuple_GET_SIZE(o) != 10) return false;
    long long v[10];
    for (int i = 0; i < 10; ++i) v[i] = number(PyTuple_GET_ITEM(o, i));
    p = Place{(void*)v[0], (float*)v[1], (const int*)v[2], v[3], v[4], (int)v[5], (int)v[6], (int)v[7], (int)v[8], (int)v[9]};
    return true;
}

// rope_cache_write_e4m3(qkv, bias or None, cu_q, tok_seq, tok_pos, slots, inv_freq or None, q_out, err, storage, place, rot_dim, n_heads, write_cache, max_q_len, constants)
PyObject* e4m3_written(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 16) return PyErr_Format(PyExc_TypeError, "rope_cache_write_e4m3: 16 arguments");
    const at::Tensor* t[10];
    for (int i = 0; i < 10; ++i) t[i] = tensor(args[i]);
    const at::Tensor *qkv = t[0], *bias = t[1], *cu = t[2], *seq = t[3], *pos = t[4], *slots = t[5], *freq = t[6], *q = t[7], *err = t[8], *storage = t[9];
    Place p;
    const bool known = placed(args[10], p);
    const long long rot = number(args[11]), heads = number(args[12]), writes = number(args[13]), most = number(args[14]), constants = number(args[15]);
    if (PyErr_Occurred()) return nullptr;
    const int device = c10::cuda::current_device();
    const at::ScalarType type = qkv ? qkv->scalar_type() : at::kInt;
    if (!known || !write_e4m3 || (type != at::kBFloat16 && type != at::kFloat) || !on(qkv, type, device) || !dense(q, type, device) || !dense(cu, at::kInt, device) ||
        !dense(seq, at::kInt, device) || !dense(pos, at::kInt, device) || !dense(slots, at::kInt, device) || !dense(err, at::kInt, device) || !storage ||
        !storage->is_cuda() || storage->get_device() != device || (args[1] != Py_None && !dense(bias, type, device)) ||
        (args[6] != Py_None && !dense(freq, at::kFloat, device)) || heads <= 0 || most <= 0 || most > INT_MAX || qkv->dim() != 2 || qkv->stride(1) != 1)
        Py_RETURN_NONE;
    const long long rows = qkv->size(0), width = (heads + 2 * p.kv_heads) * p.head_dim;
    if (rows <= 0 || qkv->size(1) < width || q->dim() != 2 || q->size(0) != rows || q->size(1) != heads * p.head_dim || seq->numel() != rows || pos->numel() != rows ||
        cu->numel() != slots->numel() + 1 || (bias && bias->numel() != width) || (freq && (rot < 0 || rot > p.head_dim || freq->numel() * 2 != rot)))
        Py_RETURN_NONE;
    return code_of([&] {
        return write_e4m3(type == at::kBFloat16, qkv->data_ptr(), bias ? bias->data_ptr() : nullptr, qkv->stride(0), ints(cu), ints(seq), ints(pos), ints(slots),
                          freq ? freq->const_data_ptr<float>() : nullptr, (int)rot, (int)heads, q->data_ptr(), p.codes, p.scales, p.table, p.page_bytes, p.page_scales,
                          p.table_stride, p.columns, p.n_slots, p.kv_heads, p.head_dim, writes != 0, (int)rows, (int)slots->numel(), (int)most, constants != 0, at_ptr<int>(*err), stream());
    });
    END_HANDLE_TH_ERRORS
}

// cache_read_e4m3(out, cu_q, tok_pos, slots, err, storage, place, n_seqs, max_kv_len, window)
PyObject* e4m3_read(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 10) return PyErr_Format(PyExc_TypeError, "cache_read_e4m3: 10 arguments");
    const at::Tensor* t[6];
    for (int i = 0; i < 6; ++i) t[i] = tensor(args[i]);
    const at::Tensor *out = t[0], *cu = t[1], *pos = t[2], *slots = t[3], *err = t[4], *storage = t[5];
    Place p;
    const bool known = placed(args[6], p);
    const long long seqs = number(args[7]), longest = number(args[8]), window = number(args[9]);
    if (PyErr_Occurred()) return nullptr;
    const int device = c10::cuda::current_device();
    const at::ScalarType type = out ? out->scalar_type() : at::kInt;
    if (!known || !read_e4m3 || (type != at::kBFloat16 && type != at::kFloat) || !on(out, type, device) || !dense(cu, at::kInt, device) || !dense(pos, at::kInt, device) ||
        !dense(slots, at::kInt, device) || !dense(err, at::kInt, device) || !storage || !storage->is_cuda() || storage->get_device() != device || seqs <= 0 ||
        slots->numel() != seqs || cu->numel() != seqs + 1 || longest <= 0 || window < 0 || window > INT_MAX || out->sizes() != storage->sizes() || !on16(*out))
        Py_RETURN_NONE;
    const long long d = p.head_dim, page = 2ll * p.kv_heads * 64 * d, step = out->size(0) == 1 ? page : out->stride(0);
    if (out->stride(4) != 1 || out->stride(3) != d || out->stride(2) != 64 * d || out->stride(1) != p.kv_heads * 64 * d || step < page || step % 8) Py_RETURN_NONE;
    const long long pages = (longest + 63) / 64;
    return code_of([&] {
        return read_e4m3(type == at::kBFloat16, out->data_ptr(), step, ints(cu), ints(pos), ints(slots), p.codes, p.scales, p.table, p.page_bytes, p.page_scales,
                         p.table_stride, p.columns, p.n_slots, p.kv_heads, p.head_dim, (int)seqs, (int)(pages < p.columns ? pages : p.columns), (int)window,
                         at_ptr<int>(*err), stream());
    });
    END_HANDLE_TH_ERRORS
}

// attention_e4m3(q, out, cu_q, tok_pos, slots, err, storage, place, part_o, part_ml, tickets, n_heads, n_seqs, max_q_len, scale, window, max_kv_len, constants)
PyObject* e4m3_attended(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 18) return PyErr_Format(PyExc_TypeError, "attention_e4m3: 18 arguments");
    const at::Tensor *q = tensor(args[0]), *out = tensor(args[1]), *cu = tensor(args[2]), *pos = tensor(args[3]), *slots = tensor(args[4]), *err = tensor(args[5]),
                     *storage = tensor(args[6]), *part_o = tensor(args[8]), *part_ml = tensor(args[9]), *tickets = tensor(args[10]);
    Place p;
    const bool known = placed(args[7], p);
    const long long heads = number(args[11]), seqs = number(args[12]), most_q = number(args[13]);
    const double scale = PyFloat_AsDouble(args[14]);
    const long long window = number(args[15]), longest = number(args[16]), constants = number(args[17]);
    if (PyErr_Occurred()) return nullptr;
    const int device = c10::cuda::current_device();
    const at::ScalarType type = q ? q->scalar_type() : at::kInt;
    if (!known || !attention_e4m3 || !attention_e4m3_slots || (type != at::kBFloat16 && type != at::kFloat) || !dense(q, type, device) || !dense(out, type, device) ||
        !dense(cu, at::kInt, device) || !dense(pos, at::kInt, device) || !dense(slots, at::kInt, device) || !dense(err, at::kInt, device) || !storage ||
        !storage->is_cuda() || storage->get_device() != device || !on(part_o, at::kFloat, device) || !on(part_ml, at::kFloat, device) || !on(tickets, at::kInt, device) ||
        seqs <= 0 || slots->numel() != seqs || cu->numel() != seqs + 1 || heads <= 0 || heads % p.kv_heads || most_q <= 0 || window < 0 || window > INT_MAX ||
        q->dim() != 2 || q->size(0) <= 0 || q->size(1) != heads * p.head_dim || out->sizes() != q->sizes() || pos->numel() != q->size(0) || !on16(*q) || !on16(*out))
        Py_RETURN_NONE;
    const long long tokens = q->size(0), rows = (most_q < tokens ? most_q : tokens) * (heads / p.kv_heads), block_rows = rows <= 8 ? 8 : 16;
    const long long chunks = (rows + block_rows - 1) / block_rows;
    long long most = (longest + 63) / 64 > p.columns ? p.columns : (longest + 63) / 64;
    if (window > 0 && (window + most_q + 62) / 64 + 1 < most) most = (window + most_q + 62) / 64 + 1;
    const long long block_slots = attention_e4m3_slots(type == at::kBFloat16, p.head_dim, (int)block_rows);
    const long long need = seqs * p.kv_heads * chunks * ((most + 3) / 4), blocks = need < block_slots ? need : block_slots;
    if (most <= 0 || block_slots <= 0 || chunks > INT_MAX || part_o->numel() < 2 * blocks * block_rows * ((p.head_dim + 31) / 32 * 32) ||
        part_ml->numel() < 4 * blocks * block_rows || tickets->numel() < 4 * blocks)
        Py_RETURN_NONE;
    return code_of([&] {
        return attention_e4m3(type == at::kBFloat16, q->data_ptr(), out->data_ptr(), ints(cu), ints(pos), ints(slots), p.codes, p.scales, p.table, p.page_bytes,
                              p.page_scales, p.table_stride, p.columns, p.n_slots, p.kv_heads, p.head_dim, (int)heads, (int)seqs, (int)tokens, most_q == 1 && tokens == seqs,
                              (int)block_rows, (int)chunks, (int)most, (int)blocks, (int)block_slots, (float)scale, (int)window, constants != 0, at_ptr<float>(*part_o),
                              at_ptr<float>(*part_ml), at_ptr<int>(*tickets), at_ptr<int>(*err), stream());
    });
    END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {{"setup", (PyCFunction)(void (*)())setup, METH_FASTCALL, nullptr},
                         {"rms_norm", (PyCFunction)(void (*)())rms_norm, METH_FASTCALL, nullptr},
                         {"prompt_attention", (PyCFunction)(void (*)())prompt_attention, METH_FASTCALL, nullptr},
                         {"gated_feed_forward", (PyCFunction)(void (*)())gated_feed_forward, METH_FASTCALL, nullptr},
                         {"matrix_memory", (PyCFunction)(void (*)())matrix_memory, METH_FASTCALL, nullptr},
                         {"state_space", (PyCFunction)(void (*)())state_space, METH_FASTCALL, nullptr},
                         {"gated_linear_attention", (PyCFunction)(void (*)())gated_linear_attention, METH_FASTCALL, nullptr},
                         {"attention_shared", (PyCFunction)(void (*)())shared_attention, METH_FASTCALL, nullptr},
                         {"verify_drafts", (PyCFunction)(void (*)())drafts_verified, METH_FASTCALL, nullptr},
                         {"copy_pages", (PyCFunction)(void (*)())pages_copied, METH_FASTCALL, nullptr},
                         {"rope_cache_write_e4m3", (PyCFunction)(void (*)())e4m3_written, METH_FASTCALL, nullptr},
                         {"cache_read_e4m3", (PyCFunction)(void (*)())e4m3_read, METH_FASTCALL, nullptr},
                         {"attention_e4m3", (PyCFunction)(void (*)())e4m3_attended, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "qf_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_qf_host() { return PyModule_Create(&module); }
