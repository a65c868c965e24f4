// host_bind.cpp - localstack_b200/_host.so: the bounded-cache wrappers (bounded.py, evict.py) as one
// compiled call each.
//
// Their smallest calls take about 8 us on the device, and the ctypes wrappers of this package cost 12
// to 20 us of host time: 21 arguments through ctypes 2 us, two outputs from torch.empty 5 us, checks
// and pointers of ten tensors 5 us, next to the C entry point's own 7 us (pointer query, tensor maps,
// launches). Here the checks, the outputs and the call are C++ over the same C ABI
// (include/lstk_cuda_attn.h); nothing is kept between calls.
//
// Every function returns the entry point's status first (the Python side raises LstkError for it)
// and raises ValueError for tensors that do not fit. Outputs and scratch are allocated on the stream that
// the kernels run on, so a call on another stream than the current one takes no memory that work
// on the current one may still use; the current device is left as it was. The C call itself runs
// without the interpreter lock, as one through ctypes does: a launch waits while the stream's queue
// is full, and the first call loads the kernels.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <initializer_list>
#include <optional>

#include "lstk_cuda_attn.h"

namespace {

constexpr int64_t kD = 128;
using Tensors = std::initializer_list<const at::Tensor *>;

struct BadValue {
    const char *what;
};

void require(bool ok, const char *what) {
    if (!ok) throw BadValue{what};
}

// A tensor argument (undefined for None).
at::Tensor tensor(PyObject *o, const char *what) {
    if (o == Py_None) return at::Tensor();
    require(THPVariable_Check(o), what);
    return THPVariable_Unpack(o);
}

int64_t integer(PyObject *o) {
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
}

// An integer argument of 32 bits, as the C ABI takes it.
int32_t int32(PyObject *o, const char *what) {
    const int64_t v = integer(o);
    require(v >= INT32_MIN && v <= INT32_MAX, what);
    return (int32_t) v;
}

float scale_of(PyObject *o) {
    if (o == Py_None) return 0.08838834764831845f;  // 1 / sqrt(128)
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return (float) v;
}

int32_t dtype_of(const at::Tensor &t) {
    return t.scalar_type() == at::kFloat ? LSTK_DTYPE_F32 : t.scalar_type() == at::kHalf ? LSTK_DTYPE_F16 : LSTK_DTYPE_BF16;
}

bool is_out_type(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16; }

at::ScalarType out_type(PyObject *o) {
    require(THPDtype_Check(o) && is_out_type(reinterpret_cast<THPDtype *>(o)->scalar_type),
            "out_dtype must be float32 or bfloat16");
    return reinterpret_cast<THPDtype *>(o)->scalar_type;
}

void require_i32(const at::Tensor &t, const char *what) {
    require(t.defined() && t.scalar_type() == at::kInt && t.is_contiguous(), what);
}

// A layer's K and V: f16 tensors, or the planes of q8_0 caches (kd, vd defined).
struct Cache {
    at::Tensor k, kd, v, vd;
    lstk_kv_layout layout;
    bool q8() const { return kd.defined(); }
};

Cache cache_of(PyObject *k, PyObject *kd, PyObject *v, PyObject *vd) {
    Cache c = {tensor(k, "the caches must be tensors"), tensor(kd, "the caches must be tensors"),
               tensor(v, "the caches must be tensors"), tensor(vd, "the caches must be tensors"), {}};
    require(c.k.defined() && c.v.defined() && c.k.dim() == 3 && c.k.sizes() == c.v.sizes() && c.k.is_contiguous() &&
                c.v.is_contiguous() && c.kd.defined() == c.vd.defined(),
            "the K and V caches must be contiguous tensors of the same shape");
    if (c.q8()) {
        require(c.k.scalar_type() == at::kChar && c.v.scalar_type() == at::kChar, "q8_0 planes must be int8");
        require(c.kd.scalar_type() == at::kHalf && c.kd.sizes() == c.vd.sizes() && c.vd.scalar_type() == at::kHalf &&
                    c.kd.dim() == 3 && c.kd.size(0) == c.k.size(0) && c.kd.size(1) == c.k.size(1) &&
                    c.kd.size(2) == kD / 32 && c.kd.is_contiguous() && c.vd.is_contiguous(),
                "q8_0 scales must be f16 [n_cells][n_head_kv][4]");
    } else {
        require(c.k.scalar_type() == at::kHalf && c.v.scalar_type() == at::kHalf,
                "cache must be a contiguous f16 [n_cells, n_head_kv, head_dim] tensor");
    }
    require(c.k.size(1) <= INT32_MAX && c.k.size(2) <= INT32_MAX, "cache dimensions out of range");
    c.layout = {c.k.size(0), (int32_t) c.k.size(1), (int32_t) c.k.size(2), 32};
    return c;
}

// The stream argument (None: the current stream of the tensors' device), made current for the scope
// with its device, so that what the scope allocates belongs to it.
struct OnStream {
    std::optional<c10::cuda::CUDAStreamGuard> guard;
    std::optional<c10::cuda::CUDAGuard> device;
    void *handle = nullptr;
    OnStream(PyObject *stream, const at::Device &dev) {
        require(dev.is_cuda(), "the tensors must be on a CUDA device");
        if (stream == Py_None) {
            device.emplace(dev.index());
            handle = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
            return;
        }
        PyObject *h = PyObject_GetAttrString(stream, "cuda_stream");
        if (!h) throw python_error();
        handle = PyLong_AsVoidPtr(h);
        Py_DECREF(h);
        if (PyErr_Occurred()) throw python_error();
        guard.emplace(c10::cuda::getStreamFromExternal(static_cast<cudaStream_t>(handle), dev.index()));
    }
};

// Other Python threads may run while the object lives; nothing of Python may be touched meanwhile.
struct Unlocked {
    PyThreadState *state = PyEval_SaveThread();
    ~Unlocked() { PyEval_RestoreThread(state); }
    Unlocked() = default;
    Unlocked(const Unlocked &) = delete;
};

void same_device(const at::Tensor &a, const at::Tensor &b) {
    require(!b.defined() || a.device() == b.device(), "the tensors must be on one device");
}

void *ptr(const at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
size_t bytes(const at::Tensor &t) { return t.defined() ? (size_t) t.nbytes() : 0; }

// A workspace argument: its bytes are its own (an expanded tensor has fewer than it counts).
at::Tensor space(PyObject *o, const char *what) {
    at::Tensor t = tensor(o, what);
    require(!t.defined() || t.is_contiguous(), what);
    return t;
}

// An uninitialised tensor on the device of `like`, from torch's allocator (without the dispatcher's
// way there, which costs as much again).
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor &like) {
    return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}

at::Tensor scratch(size_t n, const at::Tensor &like) { return fresh({(int64_t) n}, at::kByte, like); }

PyObject *wrap(const at::Tensor &t) {
    if (t.defined()) return THPVariable_Wrap(t);
    Py_RETURN_NONE;
}

// (status, tensors...)
template <typename... T>
PyObject *result(int rc, const T &...t) {
    constexpr int n = 1 + (int) sizeof...(t);
    PyObject *items[n] = {PyLong_FromLong(rc), wrap(t)...};
    PyObject *out = PyTuple_New(n);
    for (int i = 0; i < n; i++) PyTuple_SET_ITEM(out, i, items[i]);
    return out;
}

// What both decodes share: q, tables and lengths, outputs.
struct Decode {
    at::Tensor q, tables, lens, out, lse;
    int32_t B, Hq, max_blocks;
    at::ScalarType type;
    bool want_lse;
    Decode(PyObject *const *a, PyObject *out_, PyObject *out_dtype, PyObject *lse_, PyObject *want) {
        q = tensor(a[0], "q must be a tensor");
        tables = tensor(a[1], "block_tables must be a tensor");
        lens = tensor(a[2], "seq_lens must be a tensor");
        require(q.defined() && q.dim() == 3 && q.size(2) == kD && (q.scalar_type() == at::kHalf || q.scalar_type() == at::kFloat),
                "q must be f16 or f32 [B][Hq][128]");
        require(q.is_contiguous(), "q, block_tables and seq_lens must be contiguous");
        require_i32(tables, "block_tables must be a contiguous int32 tensor");
        require_i32(lens, "seq_lens must be a contiguous int32 tensor");
        require(tables.dim() == 2 && tables.size(0) == q.size(0) && lens.numel() == q.size(0),
                "block_tables must be [B][max_blocks] and seq_lens [B]");
        require(q.size(0) <= INT32_MAX && q.size(1) <= INT32_MAX && tables.size(1) <= INT32_MAX, "sizes out of range");
        B = (int32_t) q.size(0), Hq = (int32_t) q.size(1), max_blocks = (int32_t) tables.size(1);
        out = tensor(out_, "out must be a tensor");
        if (out.defined())
            require(is_out_type(out.scalar_type()) && out.sizes() == q.sizes() && out.is_contiguous(),
                    "out must be a contiguous f32 or bf16 tensor of q's shape");
        else type = out_type(out_dtype);
        lse = tensor(lse_, "lse_out must be a tensor");
        if (lse.defined())
            require(lse.scalar_type() == at::kFloat && lse.dim() == 2 && lse.size(0) == B && lse.size(1) == Hq && lse.is_contiguous(),
                    "lse_out must be a contiguous f32 [B][Hq] tensor");
        const int truth = PyObject_IsTrue(want);
        if (truth < 0) throw python_error();
        want_lse = truth == 1;
    }
    void check_devices(const Cache &c) const {
        for (const at::Tensor *t : Tensors{&c.kd, &c.v, &c.vd, &q, &tables, &lens, &out, &lse}) same_device(c.k, *t);
    }
    void allocate() {
        if (!out.defined()) out = fresh(q.sizes(), type, q);
        if (want_lse && !lse.defined()) lse = fresh({B, Hq}, at::kFloat, q);
    }
};

// (k, kd, v, vd, q, block_tables, seq_lens, window, n_sink, scale, max_seq_len, out, out_dtype, lse_out,
//  want_lse, workspace, n_ctas, stream) -> (status, out, lse)
PyObject *window(PyObject *const *a) {
    const Cache c = cache_of(a[0], a[1], a[2], a[3]);
    Decode d(a + 4, a[11], a[12], a[13], a[14]);
    const int32_t win = int32(a[7], "window out of range"), sink = int32(a[8], "n_sink out of range");
    const int32_t max_len = int32(a[10], "max_seq_len out of range"), n_ctas = int32(a[16], "n_ctas out of range");
    const float scale = scale_of(a[9]);
    at::Tensor ws = space(a[15], "workspace must be a contiguous tensor");
    d.check_devices(c);
    same_device(c.k, ws);
    OnStream s(a[17], c.k.device());
    d.allocate();
    if (d.B == 0) return result(LSTK_OK, d.out, d.lse);
    const size_t need = lstk_cuda_attn_decode_workspace_size(d.B, d.Hq, c.layout.n_head_kv, (int32_t) kD);
    if (bytes(ws) < need) ws = scratch(need, d.q);
    int rc;
    {
        const Unlocked u;
        rc = c.q8()
                 ? lstk_cuda_attn_decode_window_q8(&c.layout, static_cast<const int8_t *>(ptr(c.k)), ptr(c.kd),
                                                     static_cast<const int8_t *>(ptr(c.v)), ptr(c.vd), ptr(d.q), dtype_of(d.q),
                                                     d.B, d.Hq, static_cast<int32_t *>(ptr(d.tables)), d.max_blocks,
                                                     static_cast<int32_t *>(ptr(d.lens)), max_len, win, sink, scale, ptr(d.out),
                                                     dtype_of(d.out), static_cast<float *>(ptr(d.lse)), ptr(ws), bytes(ws),
                                                     n_ctas, s.handle)
                   : lstk_cuda_attn_decode_window(&c.layout, ptr(c.k), ptr(c.v), ptr(d.q), dtype_of(d.q), d.B, d.Hq,
                                                  static_cast<int32_t *>(ptr(d.tables)), d.max_blocks,
                                                  static_cast<int32_t *>(ptr(d.lens)), max_len, win, sink, scale, ptr(d.out),
                                                  dtype_of(d.out), static_cast<float *>(ptr(d.lse)), ptr(ws), bytes(ws), n_ctas,
                                                  s.handle);
    }
    return result(rc, d.out, d.lse);
}

// (k, kd, v, vd, q, block_tables, seq_lens, acc, scale, max_seq_len, out, out_dtype, lse_out, want_lse,
//  workspace, n_ctas, stream) -> (status, out, lse)
PyObject *weights(PyObject *const *a) {
    const Cache c = cache_of(a[0], a[1], a[2], a[3]);
    Decode d(a + 4, a[10], a[11], a[12], a[13]);
    const at::Tensor acc = tensor(a[7], "acc must be a tensor");
    require(acc.defined() && acc.scalar_type() == at::kFloat && acc.dim() == 2 && acc.size(0) == d.B && acc.stride(1) == 1,
            "acc must be f32 [B][cells] with contiguous rows");
    require(d.B <= 1 || acc.stride(0) >= acc.size(1), "the rows of acc must not overlap");
    int64_t max_len = integer(a[9]);
    const int64_t cells = (int64_t) d.max_blocks * 32;
    if (max_len <= 0 || max_len > cells) max_len = cells;
    require(max_len <= INT32_MAX, "max_seq_len out of range");
    require(acc.size(1) >= max_len, "a row of acc must hold max_seq_len keys (0: every key of a block table)");
    const int32_t n_ctas = int32(a[15], "n_ctas out of range");
    const float scale = scale_of(a[8]);
    at::Tensor ws = space(a[14], "workspace must be a contiguous tensor");
    d.check_devices(c);
    same_device(c.k, acc);
    same_device(c.k, ws);
    OnStream s(a[16], c.k.device());
    d.allocate();
    if (d.B == 0) return result(LSTK_OK, d.out, d.lse);
    if (!ws.defined())
        ws = scratch(lstk_cuda_attn_decode_weights_workspace_size(d.B, d.Hq, c.layout.n_head_kv, (int32_t) kD, (int32_t) max_len),
                     d.q);
    const int64_t stride = d.B > 1 ? acc.stride(0) : acc.size(1);
    int rc;
    {
        const Unlocked u;
        rc = c.q8()
                 ? lstk_cuda_attn_decode_weights_q8(&c.layout, static_cast<const int8_t *>(ptr(c.k)), ptr(c.kd),
                                                      static_cast<const int8_t *>(ptr(c.v)), ptr(c.vd), ptr(d.q),
                                                      dtype_of(d.q), d.B, d.Hq, static_cast<int32_t *>(ptr(d.tables)),
                                                      d.max_blocks, static_cast<int32_t *>(ptr(d.lens)), (int32_t) max_len,
                                                      scale, static_cast<float *>(ptr(acc)), stride, ptr(d.out), dtype_of(d.out),
                                                      static_cast<float *>(ptr(d.lse)), ptr(ws), bytes(ws), n_ctas, s.handle)
                   : lstk_cuda_attn_decode_weights(&c.layout, ptr(c.k), ptr(c.v), ptr(d.q), dtype_of(d.q), d.B, d.Hq,
                                                   static_cast<int32_t *>(ptr(d.tables)), d.max_blocks,
                                                   static_cast<int32_t *>(ptr(d.lens)), (int32_t) max_len, scale,
                                                   static_cast<float *>(ptr(acc)), stride, ptr(d.out), dtype_of(d.out),
                                                   static_cast<float *>(ptr(d.lse)), ptr(ws), bytes(ws), n_ctas, s.handle);
    }
    return result(rc, d.out, d.lse);
}

// (k, kd, v, vd, q, q_seq_start, q_pos0, kv_lens, block_tables, max_q_len, window, n_sink, scale, out,
//  out_dtype, workspace, scratch, stream) -> (status, out)
PyObject *prefill(PyObject *const *a) {
    const Cache c = cache_of(a[0], a[1], a[2], a[3]);
    const at::Tensor q = tensor(a[4], "q must be a tensor");
    require(q.defined() && q.dim() == 3 && q.size(2) == kD && q.is_contiguous() &&
                (q.scalar_type() == at::kHalf || q.scalar_type() == at::kFloat),
            "q must be a contiguous f16 or f32 tensor [total_tokens][Hq][128]");
    at::Tensor i[4];  // q_seq_start, q_pos0, kv_lens, block_tables
    for (int k = 0; k < 4; k++) {
        i[k] = tensor(a[5 + k], "q_seq_start, q_pos0, kv_lens and block_tables must be tensors");
        require_i32(i[k], "q_seq_start, q_pos0, kv_lens and block_tables must be contiguous int32 tensors");
    }
    const int64_t B = i[1].numel();
    require(i[0].numel() == B + 1 && i[2].numel() == B && i[3].dim() == 2 && i[3].size(0) == B,
            "q_seq_start [B+1], q_pos0 / kv_lens [B] and block_tables [B][max_blocks] must agree");
    require(B <= INT32_MAX && q.size(0) <= INT32_MAX && q.size(1) <= INT32_MAX && i[3].size(1) <= INT32_MAX,
            "sizes out of range");
    const int32_t max_q = int32(a[9], "max_q_len out of range"), win = int32(a[10], "window out of range");
    const int32_t sink = int32(a[11], "n_sink out of range"), max_blocks = (int32_t) i[3].size(1);
    const float scale = scale_of(a[12]);
    at::Tensor out = tensor(a[13], "out must be a tensor"), ws = space(a[15], "workspace must be a contiguous tensor");
    at::Tensor sc = space(a[16], "scratch must be a contiguous tensor");
    at::ScalarType type = at::kFloat;
    if (out.defined())
        require(is_out_type(out.scalar_type()) && out.sizes() == q.sizes() && out.is_contiguous(),
                "out must be a contiguous f32 or bf16 tensor of q's shape");
    else type = out_type(a[14]);
    for (const at::Tensor *t : Tensors{&c.kd, &c.v, &c.vd, &q, &i[0], &i[1], &i[2], &i[3], &out, &ws, &sc}) same_device(c.k, *t);
    OnStream s(a[17], c.k.device());
    if (!out.defined()) out = fresh(q.sizes(), type, q);
    if (B == 0 || q.size(0) == 0) return result(LSTK_OK, out);
    const int32_t Hq = (int32_t) q.size(1), hkv = c.layout.n_head_kv;
    // A workspace of the caller's that holds the f16 queries is used as it is (it may be too small to split
    // the keys); otherwise one that allows the split.
    if (!ws.defined() || bytes(ws) < lstk_cuda_attn_prefill_workspace_size((int32_t) B, Hq, hkv, (int32_t) kD, max_q,
                                                                           max_blocks, q.size(0), dtype_of(q))) {
        const size_t need = lstk_cuda_attn_prefill_window_workspace_size((int32_t) B, Hq, hkv, (int32_t) kD, max_q, max_blocks,
                                                                         q.size(0), dtype_of(q), win, sink);
        if (need) ws = scratch(need, q);
    }
    const int32_t *start = static_cast<int32_t *>(ptr(i[0])), *pos0 = static_cast<int32_t *>(ptr(i[1]));
    const int32_t *lens = static_cast<int32_t *>(ptr(i[2])), *tables = static_cast<int32_t *>(ptr(i[3]));
    if (c.q8()) {
        const size_t room = lstk_cuda_q8_prefill_scratch_size((int32_t) B, max_blocks, hkv);
        if (bytes(sc) < room) sc = scratch(room, q);
    }
    int rc;
    {
        const Unlocked u;
        rc = c.q8() ? lstk_cuda_attn_prefill_window_q8(&c.layout, static_cast<const int8_t *>(ptr(c.k)), ptr(c.kd),
                                                       static_cast<const int8_t *>(ptr(c.v)), ptr(c.vd), ptr(q),
                                                       dtype_of(q), (int32_t) B, Hq, start, max_q, q.size(0), pos0, lens,
                                                       tables, max_blocks, win, sink, scale, ptr(out), dtype_of(out),
                                                       ptr(ws), bytes(ws), ptr(sc), bytes(sc), s.handle)
                    : lstk_cuda_attn_prefill_window(&c.layout, ptr(c.k), ptr(c.v), ptr(q), dtype_of(q), (int32_t) B, Hq,
                                                    start, max_q, q.size(0), pos0, lens, tables, max_blocks, win, sink,
                                                    scale, ptr(out), dtype_of(out), ptr(ws), bytes(ws), s.handle);
    }
    return result(rc, out);
}

// (acc, pos, held, shift, seq_lens, budget, n_sink, n_recent, n, src, dst, stream) -> (status, n, src, dst);
// n, src and dst None: allocated. The state's tensors were checked when it was made.
PyObject *select(PyObject *const *a) {
    const at::Tensor acc = tensor(a[0], "acc must be a tensor"), pos = tensor(a[1], "pos must be a tensor");
    const at::Tensor held = tensor(a[2], "held must be a tensor"), shift = tensor(a[3], "shift must be a tensor");
    const at::Tensor lens = tensor(a[4], "seq_lens must be a tensor");
    const int64_t rows = acc.size(0), cells = acc.size(1);
    require_i32(lens, "seq_lens must be a contiguous int32 tensor, one per row");
    require(lens.numel() == rows, "seq_lens must be a contiguous int32 tensor, one per row");
    require(rows <= INT32_MAX && cells <= INT32_MAX, "sizes out of range");
    const int32_t budget = int32(a[5], "budget out of range"), sink = int32(a[6], "n_sink out of range");
    const int32_t recent = int32(a[7], "n_recent out of range");
    const int64_t most = std::max<int64_t>(0, std::min<int64_t>(budget, cells - budget));
    at::Tensor n = tensor(a[8], "moves must be tensors"), src = tensor(a[9], "moves must be tensors");
    at::Tensor dst = tensor(a[10], "moves must be tensors");
    if (n.defined()) {
        for (const at::Tensor *t : Tensors{&n, &src, &dst})
            require_i32(*t, "moves must hold min(budget, cells - budget) moves for every row");
        require(n.numel() == rows && src.dim() == 2 && src.sizes() == dst.sizes() && src.size(0) == rows &&
                    src.size(1) >= most && src.size(1) <= INT32_MAX,
                "moves must hold min(budget, cells - budget) moves for every row");
    }
    for (const at::Tensor *t : Tensors{&lens, &n, &src, &dst}) same_device(acc, *t);
    OnStream s(a[11], acc.device());
    if (!n.defined()) {
        n = fresh({rows}, at::kInt, acc);
        src = fresh({rows, most}, at::kInt, acc);
        dst = fresh({rows, most}, at::kInt, acc);
    }
    if (rows == 0) return result(LSTK_OK, n, src, dst);
    const lstk_kv_weights w = {static_cast<float *>(ptr(acc)), static_cast<int32_t *>(ptr(pos)),
                               static_cast<int32_t *>(ptr(held)), static_cast<int32_t *>(ptr(shift)), (int32_t) rows,
                               (int32_t) cells};
    int rc;
    {
        const Unlocked u;
        rc = lstk_cuda_kv_evict_select(&w, static_cast<int32_t *>(ptr(lens)), budget, sink, recent, (int32_t) src.size(1),
                                       static_cast<int32_t *>(ptr(n)), static_cast<int32_t *>(ptr(src)),
                                       static_cast<int32_t *>(ptr(dst)), s.handle);
    }
    return result(rc, n, src, dst);
}

// (k, kd, v, vd, block_tables, n, src, dst, stream) -> (status,)
PyObject *move(PyObject *const *a) {
    const Cache c = cache_of(a[0], a[1], a[2], a[3]);
    const at::Tensor tables = tensor(a[4], "block_tables must be a tensor"), n = tensor(a[5], "moves must be tensors");
    const at::Tensor src = tensor(a[6], "moves must be tensors"), dst = tensor(a[7], "moves must be tensors");
    for (const at::Tensor *t : Tensors{&n, &src, &dst}) require_i32(*t, "moves must be contiguous int32 tensors");
    require_i32(tables, "block_tables must be a contiguous int32 [rows][max_blocks] tensor");
    require(src.dim() == 2 && src.sizes() == dst.sizes() && n.numel() == src.size(0), "moves must be [rows] and [rows][max_moves]");
    require(tables.dim() == 2 && tables.size(0) == src.size(0), "block_tables must be a contiguous int32 [rows][max_blocks] tensor");
    require(src.size(0) <= INT32_MAX && src.size(1) <= INT32_MAX && tables.size(1) <= INT32_MAX, "sizes out of range");
    for (const at::Tensor *t : Tensors{&c.kd, &c.v, &c.vd, &tables, &n, &src, &dst}) same_device(c.k, *t);
    OnStream s(a[8], c.k.device());
    if (src.size(0) == 0 || src.size(1) == 0) return result(LSTK_OK);
    const int32_t rows = (int32_t) src.size(0), cap = (int32_t) src.size(1), max_blocks = (int32_t) tables.size(1);
    const int32_t *bt = static_cast<int32_t *>(ptr(tables)), *np = static_cast<int32_t *>(ptr(n));
    const int32_t *sp = static_cast<int32_t *>(ptr(src)), *dp = static_cast<int32_t *>(ptr(dst));
    int rc;
    {
        const Unlocked u;
        rc = c.q8() ? lstk_cuda_kv_move_q8(&c.layout, static_cast<int8_t *>(ptr(c.k)), ptr(c.kd),
                                           static_cast<int8_t *>(ptr(c.v)), ptr(c.vd), bt, rows, max_blocks, np, sp, dp, cap,
                                           s.handle)
                    : lstk_cuda_kv_move(&c.layout, ptr(c.k), ptr(c.v), bt, rows, max_blocks, np, sp, dp, cap, s.handle);
    }
    return result(rc);
}

template <PyObject *(*F)(PyObject *const *), int N>
PyObject *call(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != N) {
        PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", N, n);
        return nullptr;
    }
    try {
        return F(args);
    } catch (const BadValue &e) {
        PyErr_SetString(PyExc_ValueError, e.what);
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

#define LSTK_METHOD(name, n) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(call<name, n>)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {LSTK_METHOD(window, 18), LSTK_METHOD(weights, 17), LSTK_METHOD(prefill, 18),
                          LSTK_METHOD(select, 12), LSTK_METHOD(move, 9),     {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_host", "Compiled calls of the bounded-cache wrappers.", -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) { return PyModule_Create(&kModule); }
