// CPython side of the Python mirror's calls: argument checks, output and workspace allocation and the launch, in one call
// into native code.  A decode forward runs a few microseconds on the GPU; through ctypes its host side took 17 us (dtype
// queries, a device context manager, torch.empty, a dictionary of workspaces, a dozen ctypes conversions), and a half-
// precision forward 35 us with its two conversion kernels.
//
// `Storage` is the native half of QCudaStorage.  Its methods return a tensor, or None when the arguments do not fit -- the
// Python side then runs its own checks to say why -- and raise through the registered error function when the library
// reports a status.
//
// Launch overlap, unless lloom_b200_set_launch_overlap has settled the matter for all calls: a storage's first forward waits for everything before it on its stream like any kernel.  From then on
// the blocks are known to be in place (nothing writes them after the upload), and later forwards may stream them while the
// stream's previous kernel is still finishing.  A storage whose device pointer has been handed out, or that was made over a
// caller's tensor, stays with the first kind: the holder may write through it.
#include <torch/csrc/Device.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/extension.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <atomic>
#include <map>
#include <mutex>
#include <utility>
#include <vector>

#include "../forward.h"

namespace {

using lloom::FwdIo;

PyObject *g_error = nullptr;  // callable(status, where): raises

PyObject *fail(int status, const char *where) {
    PyObject *r = PyObject_CallFunction(g_error, "is", status, where);
    if (r) {  // it should have raised
        Py_DECREF(r);
        PyErr_Format(PyExc_RuntimeError, "%s: status %d", where, status);
    }
    return nullptr;
}

// Grow-only scratch per (device, stream): launches on different streams never share a buffer.  A buffer that has been outgrown stays alive: kernels
// in flight may still use it.
// A call that is being captured gets scratch of its own, because graphs captured on one stream may be replayed side by side on others.  In torch's
// captures it comes from the graph's pool, and stays there.  In a capture by the runtime's own calls the allocator would give it to others as soon as
// the call has returned: there it is kept, per capture and stream, and a user object ties it to the graph and all that is instantiated from it.  (Not
// in torch's captures too: a replay of a graph with a user object takes 2.6 us longer.)
struct Workspaces {
    struct Captured {
        std::pair<unsigned long long, cudaStream_t> key;
        at::Tensor buf;
        std::vector<at::Tensor> outgrown;
    };
    std::mutex mu;
    std::map<std::pair<int, cudaStream_t>, at::Tensor> bufs;
    std::vector<at::Tensor> retired;
    std::map<std::pair<unsigned long long, cudaStream_t>, Captured *> captured;
    unsigned long long last_pooled = ~0ull;  // capture, by torch
    std::mutex released_mu;
    std::vector<Captured *> released;  // of graphs that are gone; freed by the next call
    std::atomic<bool> any_released{false};

    at::Tensor get(c10::Device dev, cudaStream_t stream, int64_t bytes);
    at::Tensor get_captured(c10::Device dev, cudaStream_t stream, int64_t bytes);
    bool pooled(unsigned long long capture, const at::Tensor &t);
    void drop_released() {
        if (!any_released.load(std::memory_order_relaxed)) return;
        std::vector<Captured *> gone;
        {
            std::lock_guard<std::mutex> lock(released_mu);
            gone.swap(released);
            any_released = false;
        }
        for (Captured *c : gone) {
            captured.erase(c->key);
            delete c;
        }
    }
};
Workspaces &workspaces() {
    static Workspaces *w = new Workspaces;  // never destroyed: the CUDA context may be gone by then
    return *w;
}

// The last graph that holds this scratch is gone.  A thread of the driver may call this: no CUDA call, no lock that is held over one.
void release_captured(void *p) {
    std::lock_guard<std::mutex> lock(workspaces().released_mu);
    workspaces().released.push_back(static_cast<Workspaces::Captured *>(p));
    workspaces().any_released = true;
}

// Whether what the allocator gives to this capture belongs to its graph: a pool of torch's, or an allocator whose memory is part of the graph.  The
// allocator's list of segments is all that says so, which is why a capture asks once.
bool Workspaces::pooled(unsigned long long capture, const at::Tensor &t) {
    namespace alloc = c10::cuda::CUDACachingAllocator;
    if (capture == last_pooled) return true;
    bool yes = alloc::name() != "native";
    if (!yes) {
        const size_t at = reinterpret_cast<size_t>(t.const_data_ptr());
        for (const auto &seg : alloc::snapshot({0, 0}, false).segments)
            if (seg.device == t.device().index() && at - static_cast<size_t>(seg.address) < static_cast<size_t>(seg.total_size))
                yes = seg.owner_private_pool_id != c10::MempoolId_t{0, 0};
    }
    if (yes) last_pooled = capture;
    return yes;
}

at::Tensor Workspaces::get_captured(c10::Device dev, cudaStream_t stream, int64_t bytes) {
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    unsigned long long id = 0;
    cudaGraph_t graph = nullptr;
    C10_CUDA_CHECK(cudaStreamGetCaptureInfo(stream, &status, &id, &graph));
    const auto known = captured.find({id, stream});
    if (known != captured.end() && known->second->buf.numel() >= bytes) return known->second->buf;
    const at::Tensor fresh = at::detail::empty_cuda({std::max<int64_t>(bytes, 512)}, at::kByte, dev, std::nullopt);
    if (known != captured.end()) {
        known->second->outgrown.push_back(known->second->buf);
        return known->second->buf = fresh;
    }
    if (pooled(id, fresh)) return fresh;
    Captured *c = new Captured{{id, stream}, fresh, {}};
    cudaUserObject_t object;
    cudaError_t e = cudaUserObjectCreate(&object, c, release_captured, 1, cudaUserObjectNoDestructorSync);
    if (e != cudaSuccess) delete c;
    C10_CUDA_CHECK(e);
    captured[c->key] = c;  // the object owns it
    e = cudaGraphRetainUserObject(graph, object, 1, cudaGraphUserObjectMove);
    if (e != cudaSuccess) cudaUserObjectRelease(object, 1);
    C10_CUDA_CHECK(e);
    return fresh;
}

at::Tensor Workspaces::get(c10::Device dev, cudaStream_t stream, int64_t bytes) {
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    const bool capturing = cudaStreamIsCapturing(stream, &capture) == cudaSuccess && capture == cudaStreamCaptureStatusActive;
    std::lock_guard<std::mutex> lock(mu);
    drop_released();
    if (capturing) return get_captured(dev, stream, bytes);
    at::Tensor &buf = bufs[{dev.index(), stream}];
    if (!buf.defined() || buf.numel() < bytes) {
        if (buf.defined()) retired.push_back(buf);
        buf = at::detail::empty_cuda({std::max<int64_t>(bytes, 1 << 20)}, at::kByte, dev, std::nullopt);
    }
    return buf;
}

struct Storage {
    PyObject_HEAD
    at::Tensor *data;   // packed blocks
    at::Tensor *image;  // prefill image, or null
    int64_t image_off;
    int64_t bytes;      // of the blocks, without the padding
    int dtype;
    bool settled, exposed;
};

PyTypeObject StorageType = {PyVarObject_HEAD_INIT(nullptr, 0)};  // filled in by the module's init

bool elem_type(at::ScalarType t, int &out) {
    switch (t) {
    case at::kFloat: out = LLOOM_F32; return true;
    case at::kHalf: out = LLOOM_F16; return true;
    case at::kBFloat16: out = LLOOM_BF16; return true;
    default: return false;
    }
}

int Storage_init(PyObject *o, PyObject *args, PyObject *) {
    Storage *self = reinterpret_cast<Storage *>(o);
    PyObject *t;
    int dtype;
    long long bytes;
    if (!PyArg_ParseTuple(args, "OiL", &t, &dtype, &bytes)) return -1;
    if (!THPVariable_Check(t)) {
        PyErr_SetString(PyExc_TypeError, "a tensor of packed blocks is wanted");
        return -1;
    }
    delete self->data;
    self->data = new at::Tensor(THPVariable_Unpack(t));
    self->dtype = dtype;
    self->bytes = bytes;
    self->settled = self->exposed = false;
    return 0;
}

void Storage_dealloc(PyObject *o) {
    Storage *self = reinterpret_cast<Storage *>(o);
    delete self->data;
    delete self->image;
    Py_TYPE(o)->tp_free(o);
}

PyObject *Storage_set_image(PyObject *o, PyObject *args) {
    Storage *self = reinterpret_cast<Storage *>(o);
    PyObject *t;
    long long off = 0;
    if (!PyArg_ParseTuple(args, "O|L", &t, &off)) return nullptr;
    delete self->image;
    self->image = nullptr;
    if (t != Py_None) {
        if (!THPVariable_Check(t)) {
            PyErr_SetString(PyExc_TypeError, "a tensor or None is wanted");
            return nullptr;
        }
        self->image = new at::Tensor(THPVariable_Unpack(t));
        self->image_off = off;
    }
    Py_RETURN_NONE;
}

PyObject *Storage_expose(PyObject *o, PyObject *) {
    reinterpret_cast<Storage *>(o)->exposed = true;
    Py_RETURN_NONE;
}

// Whether this storage's next forward may start before its stream predecessor has finished
bool overlaps(const Storage *self) {
    const int mode = lloom::launch_overlap();
    return mode > 0 || (mode < 0 && self->settled && !self->exposed);
}

PyObject *Storage_exposed(PyObject *o, PyObject *) { return PyBool_FromLong(reinterpret_cast<Storage *>(o)->exposed); }
PyObject *Storage_overlaps(PyObject *o, PyObject *) { return PyBool_FromLong(overlaps(reinterpret_cast<Storage *>(o))); }

bool shape2(PyObject *t, int64_t &n, int64_t &k) {
    if (!PyTuple_Check(t) || PyTuple_GET_SIZE(t) != 2) return false;
    n = PyLong_AsLongLong(PyTuple_GET_ITEM(t, 0));
    k = PyLong_AsLongLong(PyTuple_GET_ITEM(t, 1));
    return !PyErr_Occurred() && n > 0 && k > 0;
}

// An activation tensor of this storage's device, [.., k], contiguous, of a type the kernels read
bool acts_ok(const Storage *self, const at::Tensor &x, int64_t k, int &x_type) {
    return x.defined() && x.device() == self->data->device() && x.layout() == at::kStrided && elem_type(x.scalar_type(), x_type) &&
           x.dim() >= 2 && x.size(-1) == k && x.numel() > 0 && x.is_contiguous();
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

PyObject *none_or_error() {
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
}

// forward(x, (n, k)[, out, column, store]) -> [.., n] of x's type, or f32 into columns of `out` [m, ld]
PyObject *Storage_forward(PyObject *o, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    Storage *self = reinterpret_cast<Storage *>(o);
    int64_t n, k;
    int store = LLOOM_STORE_PLAIN, x_type;
    if (nargs < 2 || !THPVariable_Check(args[0]) || !shape2(args[1], n, k)) return none_or_error();
    at::Tensor x = THPVariable_Unpack(args[0]);
    if (!acts_ok(self, x, k, x_type)) Py_RETURN_NONE;
    int64_t column = 0;
    at::Tensor y;
    if (nargs == 5) {
        column = PyLong_AsLongLong(args[3]);
        store = (int)PyLong_AsLong(args[4]);
        if (PyErr_Occurred()) return nullptr;
        if (args[2] != Py_None) {
            if (!THPVariable_Check(args[2])) Py_RETURN_NONE;
            y = THPVariable_Unpack(args[2]);
        }
    }
    const c10::Device dev = self->data->device();
    c10::cuda::CUDAGuard guard(dev);
    const int64_t m = x.numel() / k;
    FwdIo io;
    io.overlap = overlaps(self);
    if (x_type != LLOOM_F32 && !aligned16(x.const_data_ptr())) x = x.clone();
    io.x_type = x_type;
    int64_t ldy = n;
    char *yp;
    const bool fresh = !y.defined();
    if (!fresh) {
        ldy = y.dim() >= 2 ? y.stride(-2) : y.numel();
        yp = static_cast<char *>(y.data_ptr()) + 4 * column;
    } else {
        c10::SmallVector<int64_t, 5> sizes(x.sizes().begin(), x.sizes().end());
        sizes.back() = n;
        const bool plain = store == LLOOM_STORE_PLAIN;
        y = at::detail::empty_cuda(sizes, plain ? x.scalar_type() : at::kFloat, dev, std::nullopt);
        io.y_type = plain ? x_type : LLOOM_F32;
        yp = static_cast<char *>(y.data_ptr());
    }
    const bool image = self->image && m > 8 && store == LLOOM_STORE_PLAIN;
    const int64_t need = image ? lloom_b200_workspace_bytes_with_image(self->dtype, m, n, k)
                               : lloom_b200_workspace_bytes(self->dtype, m, n, k);
    if (need <= 0) Py_RETURN_NONE;
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
    const at::Tensor ws = workspaces().get(dev, stream, need);
    const int rc = lloom::qmatmul_forward(self->dtype, self->data->const_data_ptr(),
                                          image ? static_cast<char *>(self->image->data_ptr()) + self->image_off : nullptr,
                                          x.const_data_ptr(), yp, m, n, k, ldy, store, ws.data_ptr(), ws.numel(), stream, io);
    if (rc != LLOOM_OK) return fail(rc, "qmatmul_fwd");
    self->settled = true;
    if (fresh && y.scalar_type() != x.scalar_type()) y = y.to(x.scalar_type());  // a store block's outputs are f32
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// Contiguous canonical activation blocks [.., row bytes] of this storage's device, for rows of k elements
bool blocks_ok(const Storage *self, const at::Tensor &a, int64_t k) {
    const int64_t row = lloom_b200_act_row_bytes(self->dtype, k);
    return a.defined() && a.device() == self->data->device() && a.layout() == at::kStrided && a.scalar_type() == at::kByte && row > 0 &&
           a.dim() >= 2 && a.size(-1) == row && a.numel() > 0 && a.is_contiguous();
}

at::ScalarType scalar_of(int type) { return type == LLOOM_F16 ? at::kHalf : type == LLOOM_BF16 ? at::kBFloat16 : at::kFloat; }

// forward_acts(blocks, (n, k), element type of the result) -> [.., n]
PyObject *Storage_forward_acts(PyObject *o, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    Storage *self = reinterpret_cast<Storage *>(o);
    int64_t n, k;
    if (nargs != 3 || !THPVariable_Check(args[0]) || !shape2(args[1], n, k)) return none_or_error();
    const int y_type = (int)PyLong_AsLong(args[2]);
    if (PyErr_Occurred()) return nullptr;
    const at::Tensor &a = THPVariable_Unpack(args[0]);
    if (!blocks_ok(self, a, k)) Py_RETURN_NONE;
    const c10::Device dev = self->data->device();
    c10::cuda::CUDAGuard guard(dev);
    const int64_t m = a.numel() / a.size(-1);
    const bool image = self->image && m > 8;
    const int64_t need = image ? lloom_b200_workspace_bytes_with_image(self->dtype, m, n, k)
                               : lloom_b200_workspace_bytes(self->dtype, m, n, k);
    if (need <= 0) Py_RETURN_NONE;
    c10::SmallVector<int64_t, 5> sizes(a.sizes().begin(), a.sizes().end());
    sizes.back() = n;
    at::Tensor y = at::detail::empty_cuda(sizes, scalar_of(y_type), dev, std::nullopt);
    FwdIo io;
    io.overlap = overlaps(self);
    io.y_type = y_type;
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
    const at::Tensor ws = workspaces().get(dev, stream, need);
    const int rc = lloom::qmatmul_forward_acts(self->dtype, self->data->const_data_ptr(),
                                               image ? static_cast<char *>(self->image->data_ptr()) + self->image_off : nullptr,
                                               a.const_data_ptr(), y.data_ptr(), m, n, k, n, ws.data_ptr(), ws.numel(), stream, io);
    if (rc != LLOOM_OK) return fail(rc, "qmatmul_fwd_acts");
    self->settled = true;
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// embedding(ids, (rows, hidden)) -> f32 ids.shape + [hidden]
PyObject *Storage_embedding(PyObject *o, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    Storage *self = reinterpret_cast<Storage *>(o);
    int64_t rows, hidden;
    if (nargs != 2 || !THPVariable_Check(args[0]) || !shape2(args[1], rows, hidden)) return none_or_error();
    const int64_t be = lloom_b200_block_elems(self->dtype), bb = lloom_b200_block_bytes(self->dtype);
    if (hidden % be != 0 || self->bytes != rows * (hidden / be) * bb) Py_RETURN_NONE;
    const c10::Device dev = self->data->device();
    c10::cuda::CUDAGuard guard(dev);
    at::Tensor ids = THPVariable_Unpack(args[0]);
    c10::SmallVector<int64_t, 5> sizes(ids.sizes().begin(), ids.sizes().end());
    sizes.push_back(hidden);
    if (ids.device() != dev || (ids.scalar_type() != at::kLong && ids.scalar_type() != at::kInt)) ids = ids.to(dev, at::kLong);
    ids = ids.contiguous();
    at::Tensor out = at::detail::empty_cuda(sizes, at::kFloat, dev, std::nullopt);
    if (ids.numel() > 0) {
        const int rc = lloom::get_rows(self->dtype, self->data->const_data_ptr(), rows, hidden, ids.const_data_ptr(),
                                       ids.scalar_type() == at::kLong, ids.numel(), out.data_ptr<float>(),
                                       c10::cuda::getCurrentCUDAStream(dev.index()).stream(), lloom::launch_overlap() != 0);
        if (rc != LLOOM_OK) return fail(rc, "get_rows");
    }
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// experts(x, ids, n_experts, n, k) -> f32 [batch, topk, n]
PyObject *Storage_experts(PyObject *o, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    Storage *self = reinterpret_cast<Storage *>(o);
    if (nargs != 5 || !THPVariable_Check(args[0]) || !THPVariable_Check(args[1])) Py_RETURN_NONE;
    const int64_t n_experts = PyLong_AsLongLong(args[2]), n = PyLong_AsLongLong(args[3]), k = PyLong_AsLongLong(args[4]);
    if (PyErr_Occurred()) return nullptr;
    at::Tensor x = THPVariable_Unpack(args[0]), ids = THPVariable_Unpack(args[1]);
    const c10::Device dev = self->data->device();
    if (x.dim() != 3 || ids.dim() != 2 || x.device() != dev || ids.device() != dev || x.size(2) != k || x.size(0) != ids.size(0) ||
        (x.size(1) != 1 && x.size(1) != ids.size(1)) || x.numel() == 0 || ids.numel() == 0)
        Py_RETURN_NONE;
    c10::cuda::CUDAGuard guard(dev);
    if (x.scalar_type() != at::kFloat) x = x.to(at::kFloat);
    x = x.contiguous();
    if (ids.scalar_type() != at::kLong && ids.scalar_type() != at::kInt) ids = ids.to(at::kLong);
    ids = ids.contiguous();
    at::Tensor out = at::detail::empty_cuda({x.size(0), ids.size(1), n}, at::kFloat, dev, std::nullopt);
    const int64_t need = lloom_b200_workspace_bytes(self->dtype, 1, n, k);
    if (need <= 0) Py_RETURN_NONE;
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
    const at::Tensor ws = workspaces().get(dev, stream, need);
    FwdIo io;
    io.overlap = overlaps(self);
    const int rc = lloom::indexed_moe_forward(self->dtype, self->data->const_data_ptr(), n_experts, n, k, x.const_data_ptr<float>(),
                                              x.size(0), x.size(1), ids.const_data_ptr(), ids.scalar_type() == at::kLong, ids.size(1),
                                              out.data_ptr<float>(), ws.data_ptr(), ws.numel(), stream, io);
    if (rc != LLOOM_OK) return fail(rc, "indexed_moe_forward");
    self->settled = true;
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}


// A destination of m rows of n f32 values, `ld` apart
bool out_ok(const at::Tensor &t, c10::Device dev, int64_t m, int64_t n, int64_t &ld) {
    if (!t.defined() || t.device() != dev || t.layout() != at::kStrided || t.scalar_type() != at::kFloat || t.dim() < 1 || t.size(-1) != n ||
        t.numel() != m * n || (n > 1 && t.stride(-1) != 1))
        return false;
    ld = t.dim() == 2 && m > 1 ? t.stride(0) : n;  // (the stride of an extent of 1 says nothing)
    return m == 1 || (t.dim() == 2 ? ld >= n : t.is_contiguous());
}

// group(storages, [(n, k), ..], x, stores or None, outs or None, whether x is activation blocks) -> list of f32 [.., n_g]
PyObject *module_group(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    if (nargs != 6 || !PyList_Check(args[0]) || !PyList_Check(args[1]) || !THPVariable_Check(args[2])) Py_RETURN_NONE;
    const Py_ssize_t G = PyList_GET_SIZE(args[0]);
    if (G < 1 || G > LLOOM_B200_MAX_GROUP || PyList_GET_SIZE(args[1]) != G) Py_RETURN_NONE;
    const at::Tensor &x = THPVariable_Unpack(args[2]);
    PyObject *stores = args[3] == Py_None ? nullptr : args[3], *outs = args[4] == Py_None ? nullptr : args[4];
    if ((stores && (!PyList_Check(stores) || PyList_GET_SIZE(stores) != G)) || (outs && (!PyList_Check(outs) || PyList_GET_SIZE(outs) != G)))
        Py_RETURN_NONE;
    Storage *st[LLOOM_B200_MAX_GROUP];
    const void *w[LLOOM_B200_MAX_GROUP];
    float *y[LLOOM_B200_MAX_GROUP];
    int64_t n[LLOOM_B200_MAX_GROUP], ld[LLOOM_B200_MAX_GROUP], n_max = 0, k = 0;
    int store[LLOOM_B200_MAX_GROUP];
    FwdIo io;
    io.overlap = true;
    for (Py_ssize_t g = 0; g < G; ++g) {
        PyObject *s = PyList_GET_ITEM(args[0], g);
        if (Py_TYPE(s) != &StorageType) Py_RETURN_NONE;
        st[g] = reinterpret_cast<Storage *>(s);
        if (st[g]->dtype != st[0]->dtype || st[g]->data->device() != st[0]->data->device()) Py_RETURN_NONE;
        w[g] = st[g]->data->const_data_ptr();
        int64_t k_g;  // (of a stack of experts the first two extents would pass for n and k: shape2 refuses one)
        if (!shape2(PyList_GET_ITEM(args[1], g), n[g], k_g) || (g > 0 && k_g != k)) return none_or_error();
        k = k_g;
        store[g] = stores ? (int)PyLong_AsLong(PyList_GET_ITEM(stores, g)) : LLOOM_STORE_PLAIN;
        if (PyErr_Occurred()) return nullptr;
        if (store[g] == LLOOM_STORE_MUL_INTO && !outs) Py_RETURN_NONE;  // nothing to multiply into
        n_max = std::max(n_max, n[g]);
        io.overlap = io.overlap && overlaps(st[g]);
    }
    int x_type;
    const bool blocks = args[5] == Py_True;
    if (blocks ? !blocks_ok(st[0], x, k) : !acts_ok(st[0], x, k, x_type) || x_type != LLOOM_F32) Py_RETURN_NONE;
    const c10::Device dev = st[0]->data->device();
    const int64_t m = x.numel() / x.size(-1);
    for (Py_ssize_t g = 0; outs && g < G; ++g) {
        PyObject *item = PyList_GET_ITEM(outs, g);
        if (!THPVariable_Check(item) || !out_ok(THPVariable_Unpack(item), dev, m, n[g], ld[g])) Py_RETURN_NONE;
    }
    c10::cuda::CUDAGuard guard(dev);
    const int64_t need = lloom_b200_workspace_bytes(st[0]->dtype, m, n_max, k);
    if (need <= 0) Py_RETURN_NONE;
    THPObjectPtr list(PyList_New(G));
    if (!list) return nullptr;
    for (Py_ssize_t g = 0; g < G; ++g) {
        PyObject *item;
        if (outs) {
            item = PyList_GET_ITEM(outs, g);
            Py_INCREF(item);
            y[g] = static_cast<float *>(THPVariable_Unpack(item).data_ptr());
        } else {
            c10::SmallVector<int64_t, 5> sizes(x.sizes().begin(), x.sizes().end());
            sizes.back() = n[g];
            at::Tensor t = at::detail::empty_cuda(sizes, at::kFloat, dev, std::nullopt);
            y[g] = static_cast<float *>(t.data_ptr());
            ld[g] = n[g];
            item = THPVariable_Wrap(std::move(t));
            if (!item) return nullptr;
        }
        PyList_SET_ITEM(list.get(), g, item);
    }
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
    const at::Tensor ws = workspaces().get(dev, stream, need);
    const int rc = lloom::qmatmul_forward_group(st[0]->dtype, (int)G, w, blocks ? x.const_data_ptr() : nullptr,
                                                blocks ? nullptr : x.const_data_ptr(), y, n, ld, store, m, k, ws.data_ptr(),
                                                ws.numel(), stream, io);
    if (rc != LLOOM_OK) return fail(rc, "qmatmul_fwd_group");
    for (Py_ssize_t g = 0; g < G; ++g) st[g]->settled = true;
    return list.release();
    END_HANDLE_TH_ERRORS
}

// Native half of MxTensor: the image of an [n, k] matrix of microscaled 4-bit values, which nobody else holds.
struct MxStorage {
    PyObject_HEAD
    at::Tensor *image;
    int64_t n, k;
    bool settled;
    cudaStream_t home, last;  // where the image was allocated, and the stream of its last use
};
PyTypeObject MxStorageType = {PyVarObject_HEAD_INIT(nullptr, 0)};

void MxStorage_dealloc(PyObject *o) {
    delete reinterpret_cast<MxStorage *>(o)->image;
    Py_TYPE(o)->tp_free(o);
}

cudaStream_t stream_of(c10::Device dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

// An image of its own for [n, k], not yet written; null with an exception
MxStorage *mx_new(int64_t n, int64_t k, c10::Device dev) {
    PyObject *o = MxStorageType.tp_alloc(&MxStorageType, 0);
    if (!o) return nullptr;
    MxStorage *st = reinterpret_cast<MxStorage *>(o);
    st->n = n;
    st->k = k;
    st->settled = false;
    st->home = st->last = stream_of(dev);
    try {
        st->image = new at::Tensor(at::detail::empty_cuda({lloom_b200_mx_image_bytes(n, k)}, at::kByte, dev, std::nullopt));
    } catch (...) {
        Py_DECREF(o);
        throw;
    }
    return st;
}

// The current stream, which is about to read the image.  Nobody but this storage holds that, so it tells the allocator of streams other than the
// image's own: the memory may go to others only when they have finished with it.
cudaStream_t stream_to_read(MxStorage *self) {
    const c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream(self->image->device().index());
    if (stream.stream() != self->home && stream.stream() != self->last) c10::cuda::CUDACachingAllocator::recordStream(self->image->storage().data_ptr(), stream);
    self->last = stream.stream();
    return stream.stream();
}

// mx_quantize(x [.., k]) -> storage of [rows, k]
PyObject *module_mx_quantize(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    int x_type;
    if (nargs != 1 || !THPVariable_Check(args[0])) Py_RETURN_NONE;
    at::Tensor x = THPVariable_Unpack(args[0]);
    if (!x.defined() || !x.is_cuda() || x.layout() != at::kStrided || !elem_type(x.scalar_type(), x_type) || x.dim() < 2 || x.numel() == 0 ||
        !x.is_contiguous())
        Py_RETURN_NONE;
    const int64_t k = x.size(-1), n = x.numel() / k;
    if (lloom_b200_mx_image_bytes(n, k) <= 0) Py_RETURN_NONE;
    const c10::Device dev = x.device();
    c10::cuda::CUDAGuard guard(dev);
    if (!aligned16(x.const_data_ptr())) x = x.clone();
    MxStorage *st = mx_new(n, k, dev);
    if (!st) return nullptr;
    THPObjectPtr own(reinterpret_cast<PyObject *>(st));
    const int rc = lloom::mx_quantize(x.const_data_ptr(), x_type, n, k, st->image->data_ptr(), st->image->numel(), stream_of(dev),
                                      lloom::launch_overlap() != 0);
    if (rc != LLOOM_OK) return fail(rc, "mx_quantize");
    return own.release();
    END_HANDLE_TH_ERRORS
}

// mx_from_blocks(blocks uint8 on the GPU, (n, k)) -> storage
PyObject *module_mx_from_blocks(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    int64_t n, k;
    if (nargs != 2 || !THPVariable_Check(args[0]) || !shape2(args[1], n, k)) return none_or_error();
    const at::Tensor &b = THPVariable_Unpack(args[0]);
    if (!b.defined() || !b.is_cuda() || b.scalar_type() != at::kByte || !b.is_contiguous() || lloom_b200_mx_image_bytes(n, k) <= 0 ||
        b.numel() != n * (k / 32) * 17)
        Py_RETURN_NONE;
    c10::cuda::CUDAGuard guard(b.device());
    MxStorage *st = mx_new(n, k, b.device());
    if (!st) return nullptr;
    THPObjectPtr own(reinterpret_cast<PyObject *>(st));
    const int rc = lloom_b200_mx_from_blocks(b.const_data_ptr(), n, k, st->image->data_ptr(), st->image->numel(), stream_of(b.device()));
    if (rc != LLOOM_OK) return fail(rc, "mx_from_blocks");
    return own.release();
    END_HANDLE_TH_ERRORS
}

// shape() -> (n, k)
PyObject *MxStorage_shape(PyObject *o, PyObject *) {
    return Py_BuildValue("LL", (long long)reinterpret_cast<MxStorage *>(o)->n, (long long)reinterpret_cast<MxStorage *>(o)->k);
}
// device() -> torch.device
PyObject *MxStorage_device(PyObject *o, PyObject *) { return THPDevice_New(reinterpret_cast<MxStorage *>(o)->image->device()); }

// to_blocks() -> uint8 [n, k / 32 * 17] on the GPU
PyObject *MxStorage_to_blocks(PyObject *o, PyObject *) {
    HANDLE_TH_ERRORS
    MxStorage *self = reinterpret_cast<MxStorage *>(o);
    const c10::Device dev = self->image->device();
    c10::cuda::CUDAGuard guard(dev);
    at::Tensor out = at::detail::empty_cuda({self->n, self->k / 32 * 17}, at::kByte, dev, std::nullopt);
    const int rc = lloom_b200_mx_to_blocks(self->image->const_data_ptr(), self->n, self->k, out.data_ptr(), stream_to_read(self));
    if (rc != LLOOM_OK) return fail(rc, "mx_to_blocks");
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// dequantize(f16) -> [n, k]
PyObject *MxStorage_dequantize(PyObject *o, PyObject *f16) {
    HANDLE_TH_ERRORS
    MxStorage *self = reinterpret_cast<MxStorage *>(o);
    const c10::Device dev = self->image->device();
    c10::cuda::CUDAGuard guard(dev);
    at::Tensor out = at::detail::empty_cuda({self->n, self->k}, f16 == Py_True ? at::kHalf : at::kFloat, dev, std::nullopt);
    const int rc = lloom::mx_dequantize(self->image->const_data_ptr(), self->n, self->k, out.data_ptr(), f16 == Py_True, stream_to_read(self),
                                        lloom::launch_overlap() != 0);
    if (rc != LLOOM_OK) return fail(rc, "mx_dequantize");
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// As for Storage, but the first forward always waits: the kernel in front may be the one that writes the image, which is this package's own
bool overlaps(const MxStorage *self) { return lloom::launch_overlap() != 0 && self->settled; }
PyObject *MxStorage_overlaps(PyObject *o, PyObject *) { return PyBool_FromLong(overlaps(reinterpret_cast<MxStorage *>(o))); }

// forward(x [.., k]) -> [.., n] of x's type
PyObject *MxStorage_forward(PyObject *o, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    MxStorage *self = reinterpret_cast<MxStorage *>(o);
    int x_type;
    if (nargs != 1 || !THPVariable_Check(args[0])) Py_RETURN_NONE;
    at::Tensor x = THPVariable_Unpack(args[0]);
    const c10::Device dev = self->image->device();
    if (!x.defined() || x.device() != dev || x.layout() != at::kStrided || !elem_type(x.scalar_type(), x_type) || x.dim() < 2 ||
        x.size(-1) != self->k || x.numel() == 0 || !x.is_contiguous())
        Py_RETURN_NONE;
    c10::cuda::CUDAGuard guard(dev);
    if (!aligned16(x.const_data_ptr())) x = x.clone();
    const int64_t m = x.numel() / self->k, need = lloom_b200_mx_workspace_bytes(m, self->n, self->k);
    if (need <= 0) Py_RETURN_NONE;
    c10::SmallVector<int64_t, 5> sizes(x.sizes().begin(), x.sizes().end());
    sizes.back() = self->n;
    at::Tensor y = at::detail::empty_cuda(sizes, x.scalar_type(), dev, std::nullopt);
    const cudaStream_t stream = stream_to_read(self);
    const at::Tensor ws = workspaces().get(dev, stream, need);
    const int rc = lloom::mx_forward(self->image->const_data_ptr(), x.const_data_ptr(), x_type, y.data_ptr(), x_type, m, self->n, self->k,
                                     self->n, ws.data_ptr(), ws.numel(), stream, overlaps(self));
    if (rc != LLOOM_OK) return fail(rc, "mx_fwd");
    self->settled = true;
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// The rows of [.., k] and how far apart they are: a contiguous tensor, or a matrix whose rows are
bool row_layout(const at::Tensor &t, int64_t &rows, int64_t &k, int64_t &ld) {
    if (!t.defined() || t.layout() != at::kStrided || !t.is_cuda() || t.dim() < 1) return false;
    k = t.size(-1);
    if (k == 0) return false;
    rows = t.numel() / k;
    ld = k;
    if (t.is_contiguous()) return true;
    if (t.dim() != 2 || t.stride(1) != 1 || t.stride(0) < k) return false;
    ld = t.stride(0);
    return true;
}

// rms_norm(x, weight, eps, residual or None, -1 or the block type) -> y, or (y, h) with a residual
PyObject *module_rms_norm(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    if (nargs != 5 || !THPVariable_Check(args[0]) || !THPVariable_Check(args[1]) || (args[3] != Py_None && !THPVariable_Check(args[3])))
        Py_RETURN_NONE;
    const at::Tensor &x = THPVariable_Unpack(args[0]), &w = THPVariable_Unpack(args[1]);
    const double eps = PyFloat_AsDouble(args[2]);
    const int blocks = (int)PyLong_AsLong(args[4]);
    if (PyErr_Occurred()) return nullptr;
    int64_t m, k, ldx, rm, rk, ldr = 0;
    int x_type, w_type;
    if (!row_layout(x, m, k, ldx) || !elem_type(x.scalar_type(), x_type)) Py_RETURN_NONE;
    if (!w.defined() || w.device() != x.device() || w.dim() != 1 || w.size(0) != k || !w.is_contiguous() || !elem_type(w.scalar_type(), w_type))
        Py_RETURN_NONE;
    at::Tensor r;
    if (args[3] != Py_None) {
        r = THPVariable_Unpack(args[3]);
        if (!row_layout(r, rm, rk, ldr) || r.scalar_type() != x.scalar_type() || r.device() != x.device() || r.sizes() != x.sizes()) Py_RETURN_NONE;
    }
    const int64_t be = blocks >= 0 ? lloom_b200_block_elems(blocks) : 1;
    if (be <= 0 || k % be != 0) Py_RETURN_NONE;
    const c10::Device dev = x.device();
    c10::cuda::CUDAGuard guard(dev);
    c10::SmallVector<int64_t, 5> sizes(x.sizes().begin(), x.sizes().end());
    at::Tensor h, y;
    if (r.defined()) h = at::detail::empty_cuda(sizes, x.scalar_type(), dev, std::nullopt);
    if (blocks >= 0) sizes.back() = k / be * lloom_b200_block_bytes(blocks);
    y = at::detail::empty_cuda(sizes, blocks >= 0 ? at::kByte : x.scalar_type(), dev, std::nullopt);
    if (m > 0) {
        const int rc = lloom::rms_norm(x.const_data_ptr(), r.defined() ? r.const_data_ptr() : nullptr, w.const_data_ptr(), x_type, w_type, eps,
                                       m, k, ldx, ldr, r.defined() ? h.data_ptr() : nullptr, y.data_ptr(), blocks >= 0 ? blocks : x_type,
                                       c10::cuda::getCurrentCUDAStream(dev.index()).stream(), lloom::launch_overlap() != 0);
        if (rc != LLOOM_OK) return fail(rc, "rms_norm");
    }
    if (!r.defined()) return THPVariable_Wrap(y);
    THPObjectPtr yo(THPVariable_Wrap(y)), ho(THPVariable_Wrap(h));
    return yo && ho ? PyTuple_Pack(2, yo.get(), ho.get()) : nullptr;
    END_HANDLE_TH_ERRORS
}

// dequantize_act(blocks [.., row bytes], block type) -> f32 [.., k]
PyObject *module_dequantize_act(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    if (nargs != 2 || !THPVariable_Check(args[0])) Py_RETURN_NONE;
    const at::Tensor &a = THPVariable_Unpack(args[0]);
    const int type = (int)PyLong_AsLong(args[1]);
    if (PyErr_Occurred()) return nullptr;
    const int64_t be = lloom_b200_block_elems(type), bb = lloom_b200_block_bytes(type);
    if (!a.defined() || !a.is_cuda() || a.scalar_type() != at::kByte || !a.is_contiguous() || a.dim() < 1 || be <= 0 || a.size(-1) % bb != 0)
        Py_RETURN_NONE;
    c10::cuda::CUDAGuard guard(a.device());
    c10::SmallVector<int64_t, 5> sizes(a.sizes().begin(), a.sizes().end());
    sizes.back() = sizes.back() / bb * be;
    at::Tensor out = at::detail::empty_cuda(sizes, at::kFloat, a.device(), std::nullopt);
    if (out.numel() > 0) {
        const int rc = lloom::dequantize_act(type, a.const_data_ptr(), out.numel(), out.data_ptr<float>(),
                                             c10::cuda::getCurrentCUDAStream(a.device().index()).stream(), lloom::launch_overlap() != 0);
        if (rc != LLOOM_OK) return fail(rc, "dequantize_act");
    }
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// A setting of the sampler: one number, or a contiguous tensor with a value per row.  False with or without an exception
bool setting(PyObject *o, const at::Tensor &like, int64_t rows, at::ScalarType type, const void *&per_row, double &all) {
    per_row = nullptr;
    all = 0.0;
    if (!THPVariable_Check(o)) {
        all = PyFloat_AsDouble(o);
        return !PyErr_Occurred();
    }
    const at::Tensor &t = THPVariable_Unpack(o);
    if (!t.defined() || t.device() != like.device() || t.scalar_type() != type || t.numel() != rows || !t.is_contiguous()) return false;
    per_row = t.const_data_ptr();
    return true;
}

// sample(logits [.., vocab], u, temperature, top_k, top_p, min_p) -> (ids, probs)
PyObject *module_sample(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    if (nargs != 6 || !THPVariable_Check(args[0]) || !THPVariable_Check(args[1])) Py_RETURN_NONE;
    const at::Tensor &x = THPVariable_Unpack(args[0]), &u = THPVariable_Unpack(args[1]);
    int64_t rows, vocab, ld;
    int type;
    if (!row_layout(x, rows, vocab, ld) || !elem_type(x.scalar_type(), type)) Py_RETURN_NONE;
    if (!u.defined() || u.device() != x.device() || u.scalar_type() != at::kFloat || u.sizes() != x.sizes().slice(0, x.dim() - 1) || !u.is_contiguous())
        Py_RETURN_NONE;
    const void *t, *k, *p, *mp;
    double t_all, k_all, p_all, mp_all;
    if (!setting(args[2], x, rows, at::kFloat, t, t_all) || !setting(args[3], x, rows, at::kInt, k, k_all) ||
        !setting(args[4], x, rows, at::kFloat, p, p_all) || !setting(args[5], x, rows, at::kFloat, mp, mp_all))
        return none_or_error();
    const c10::Device dev = x.device();
    c10::cuda::CUDAGuard guard(dev);
    at::Tensor ids = at::detail::empty_cuda(u.sizes(), at::kLong, dev, std::nullopt), probs = at::detail::empty_cuda(u.sizes(), at::kFloat, dev, std::nullopt);
    if (rows > 0) {
        const int64_t k_int = k_all >= 0 ? (int64_t)std::min(k_all, 9.0e15) : -1;
        const int rc = lloom::sample(x.const_data_ptr(), type, rows, vocab, ld, u.const_data_ptr<float>(), (const float *)t, t_all, (const int *)k,
                                     k_int, (const float *)p, p_all, (const float *)mp, mp_all, ids.data_ptr<int64_t>(), probs.data_ptr<float>(),
                                     stream_of(dev), lloom::launch_overlap() != 0);
        if (rc != LLOOM_OK) return fail(rc, "sample");
    }
    THPObjectPtr a(THPVariable_Wrap(ids)), b(THPVariable_Wrap(probs));
    return a && b ? PyTuple_Pack(2, a.get(), b.get()) : nullptr;
    END_HANDLE_TH_ERRORS
}

// workspace(device index, stream, bytes) -> uint8 tensor of at least that size, kept for later calls
PyObject *module_workspace(PyObject *, PyObject *args) {
    HANDLE_TH_ERRORS
    int index;
    unsigned long long stream;
    long long bytes;
    if (!PyArg_ParseTuple(args, "iKL", &index, &stream, &bytes)) return nullptr;
    const c10::Device dev(c10::kCUDA, (c10::DeviceIndex)index);
    c10::cuda::CUDAGuard guard(dev);
    return THPVariable_Wrap(workspaces().get(dev, reinterpret_cast<cudaStream_t>(stream), bytes));
    END_HANDLE_TH_ERRORS
}

PyObject *module_set_error(PyObject *, PyObject *fn) {
    Py_INCREF(fn);
    Py_XDECREF(g_error);
    g_error = fn;
    Py_RETURN_NONE;
}

#define FAST(fn) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(fn))
PyMethodDef storage_methods[] = {{"forward", FAST(Storage_forward), METH_FASTCALL, nullptr},
                                 {"forward_acts", FAST(Storage_forward_acts), METH_FASTCALL, nullptr},
                                 {"embedding", FAST(Storage_embedding), METH_FASTCALL, nullptr},
                                 {"experts", FAST(Storage_experts), METH_FASTCALL, nullptr},
                                 {"set_image", Storage_set_image, METH_VARARGS, nullptr},
                                 {"expose", Storage_expose, METH_NOARGS, nullptr},
                                 {"exposed", Storage_exposed, METH_NOARGS, nullptr},
                                 {"overlaps", Storage_overlaps, METH_NOARGS, nullptr},
                                 {nullptr, nullptr, 0, nullptr}};

PyMethodDef mx_methods[] = {{"forward", FAST(MxStorage_forward), METH_FASTCALL, nullptr},
                            {"dequantize", MxStorage_dequantize, METH_O, nullptr},
                            {"to_blocks", MxStorage_to_blocks, METH_NOARGS, nullptr},
                            {"shape", MxStorage_shape, METH_NOARGS, nullptr},
                            {"device", MxStorage_device, METH_NOARGS, nullptr},
                            {"overlaps", MxStorage_overlaps, METH_NOARGS, nullptr},
                            {nullptr, nullptr, 0, nullptr}};

PyMethodDef module_methods[] = {{"group", FAST(module_group), METH_FASTCALL, nullptr},
                                {"rms_norm", FAST(module_rms_norm), METH_FASTCALL, nullptr},
                                {"dequantize_act", FAST(module_dequantize_act), METH_FASTCALL, nullptr},
                                {"mx_quantize", FAST(module_mx_quantize), METH_FASTCALL, nullptr},
                                {"mx_from_blocks", FAST(module_mx_from_blocks), METH_FASTCALL, nullptr},
                                {"sample", FAST(module_sample), METH_FASTCALL, nullptr},
                                {"workspace", module_workspace, METH_VARARGS, nullptr},
                                {"set_error", module_set_error, METH_O, nullptr},
                                {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, module_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) {
    StorageType.tp_name = "lloom_b200._native.Storage";
    StorageType.tp_basicsize = sizeof(Storage);
    StorageType.tp_flags = Py_TPFLAGS_DEFAULT;
    StorageType.tp_new = PyType_GenericNew;
    StorageType.tp_init = Storage_init;
    StorageType.tp_dealloc = Storage_dealloc;
    StorageType.tp_methods = storage_methods;
    if (PyType_Ready(&StorageType) < 0) return nullptr;
    MxStorageType.tp_name = "lloom_b200._native.MxStorage";
    MxStorageType.tp_basicsize = sizeof(MxStorage);
    MxStorageType.tp_flags = Py_TPFLAGS_DEFAULT;
    MxStorageType.tp_dealloc = MxStorage_dealloc;
    MxStorageType.tp_methods = mx_methods;
    if (PyType_Ready(&MxStorageType) < 0) return nullptr;
    PyObject *m = PyModule_Create(&module_def);
    if (!m) return nullptr;
    Py_INCREF(&StorageType);
    if (PyModule_AddObject(m, "Storage", reinterpret_cast<PyObject *>(&StorageType)) < 0) return nullptr;
    return m;
}
