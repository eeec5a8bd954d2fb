// The Python calls of the 8-bit key/value cache and the token log probabilities over torch tensors (the module
// mimizuku_b200._serving): each checks its tensors, fills the structs of mimizuku_b200.h and calls the library. Compiled,
// because a decoding step outside a CUDA graph is bound by the host: the checks and the packing take 5 us a call when
// interpreted, as long as the launch of one or two kernels.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>
#include <stdexcept>
#include <string>

#include "mimizuku_b200.h"

namespace {

PyObject* mmz_error = nullptr;  // mimizuku_b200.MmzError

struct Refused : std::runtime_error {  // becomes an MmzError
    using std::runtime_error::runtime_error;
};
struct Raised {};  // a Python exception is set already

template <typename... A>
[[noreturn]] void refuse(const char* what, A... parts) {
    std::string m = std::string(what) + ": ";
    for (const std::string& p : {std::string(parts)...}) m += p;
    throw Refused(m);
}

// ---------------------------------------------------------------- arguments

// the values of a call's parameters in the order of `names`, null where not given
template <int N>
struct Params {
    PyObject* v[N] = {};
    Params(const char* what, PyObject* const (&names)[N], int required, PyObject* const* args, Py_ssize_t nargs, PyObject* kw) {
        if (nargs > N) {
            PyErr_Format(PyExc_TypeError, "%s() takes at most %d arguments (%zd given)", what, N, nargs);
            throw Raised();
        }
        for (Py_ssize_t i = 0; i < nargs; i++) v[i] = args[i];
        const Py_ssize_t nkw = kw ? PyTuple_GET_SIZE(kw) : 0;
        for (Py_ssize_t k = 0; k < nkw; k++) {
            PyObject* name = PyTuple_GET_ITEM(kw, k);
            int at = -1;
            for (int i = 0; i < N && at < 0; i++)
                if (names[i] == name) at = i;  // both interned, as a rule
            for (int i = 0; i < N && at < 0; i++)
                if (PyUnicode_Compare(names[i], name) == 0) at = i;
            if (at < 0 || v[at]) {
                PyErr_Format(PyExc_TypeError, at < 0 ? "%s() got an unexpected keyword argument '%U'"
                                                     : "%s() got multiple values for argument '%U'", what, name);
                throw Raised();
            }
            v[at] = args[nargs + k];
        }
        for (int i = 0; i < N; i++) {
            if (i < required && !v[i]) {
                PyErr_Format(PyExc_TypeError, "%s() missing required argument '%U'", what, names[i]);
                throw Raised();
            }
            if (i >= required && v[i] == Py_None) v[i] = nullptr;
        }
    }
};

long long integer(PyObject* o, long long otherwise) {
    if (!o) return otherwise;
    const long long x = PyLong_AsLongLong(o);
    if (x == -1 && PyErr_Occurred()) throw Raised();
    return x;
}

std::string dims_text(at::IntArrayRef s) {
    std::string t = "(";
    for (size_t i = 0; i < s.size(); i++) t += (i ? ", " : "") + std::to_string(s[i]);
    return t + (s.size() == 1 ? ",)" : ")");
}

const at::Tensor* tensor(PyObject* o) { return o && THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

const at::Tensor& cuda_tensor(const char* what, const char* name, PyObject* o) {
    const at::Tensor* t = tensor(o);
    if (!t || !t->is_cuda()) refuse(what, name, " is not a CUDA tensor");
    return *t;
}

// the current device, which has to be that of the tensor
int device_of(const char* what, const char* name, PyObject* o) {
    const int dev = cuda_tensor(what, name, o).get_device(), current = c10::cuda::current_device();
    if (dev != current)
        refuse(what, name, " is on cuda:" + std::to_string(dev) + ", the current device is cuda:" + std::to_string(current));
    return dev;
}

// a tensor of that type, of that shape (one without dimensions of its own: any) and on device dev
const at::Tensor& typed(const char* what, const char* name, PyObject* o, at::ScalarType type, int dev) {
    const at::Tensor& t = cuda_tensor(what, name, o);
    if (t.scalar_type() != type)
        refuse(what, name, std::string(" is ") + at::toString(t.scalar_type()) + ", not " + at::toString(type));
    if (t.get_device() != dev)
        refuse(what, name, " is on cuda:" + std::to_string(t.get_device()) + ", the current device is cuda:" + std::to_string(dev));
    return t;
}
const at::Tensor& shaped(const char* what, const char* name, PyObject* o, at::ScalarType type, at::IntArrayRef shape, int dev) {
    const at::Tensor& t = typed(what, name, o, type, dev);
    if (t.sizes() != shape) refuse(what, name, " is " + dims_text(t.sizes()) + ", not " + dims_text(shape));
    return t;
}
// the address of such a contiguous tensor; null for one that was not given
void* dense(const char* what, const char* name, PyObject* o, at::ScalarType type, at::IntArrayRef shape, int dev) {
    if (!o) return nullptr;
    const at::Tensor& t = shaped(what, name, o, type, shape, dev);
    if (!t.is_contiguous()) refuse(what, name, " is not contiguous");
    return t.data_ptr();
}

int narrow(const char* what, const char* name, int64_t x) {
    if (x < 0 || x > 0x7fffffff) refuse(what, name, " of " + std::to_string(x));
    return (int)x;
}

// a stride of a dimension of `count` (that of a dimension of one may be anything)
long long step(int64_t count, int64_t stride) { return count > 1 ? (long long)stride : 0; }

bool alike(const at::Tensor& a, const at::Tensor& b) {  // strides, of tensors of one shape
    for (int64_t i = 0; i < a.dim(); i++)
        if (a.size(i) > 1 && a.stride(i) != b.stride(i)) return false;
    return true;
}

struct Stream {
    cudaStream_t raw;
    bool given;  // not the current one, or not known to be
    Stream(PyObject* o, int dev) : given(o != nullptr) {
        if (!o) {
            raw = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
        } else if (PyLong_Check(o)) {
            raw = (cudaStream_t)PyLong_AsVoidPtr(o);
        } else {
            PyObject* p = PyObject_GetAttrString(o, "cuda_stream");
            if (!p) throw Raised();
            raw = (cudaStream_t)PyLong_AsVoidPtr(p);
            Py_DECREF(p);
        }
        if (PyErr_Occurred()) throw Raised();
    }
};

// Scratch of one call, from the memory of the call's own stream: whoever had the block before used it on that stream, and
// so will whoever has it next. (A block of the current stream's memory may still be read or written there.)
at::Tensor own_scratch(size_t bytes, const Stream& st, int dev) {
    c10::cuda::OptionalCUDAStreamGuard on;
    if (st.given) on.reset_stream(c10::cuda::getStreamFromExternal(st.raw, (c10::DeviceIndex)dev));
    return at::empty({(int64_t)bytes}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA, (c10::DeviceIndex)dev));
}
// a given one
void* their_scratch(const char* what, PyObject* o, int dev, unsigned long long* bytes) {
    const at::Tensor& t = typed(what, "scratch", o, at::kByte, dev);
    if (!t.is_contiguous()) refuse(what, "scratch is not contiguous");
    *bytes = (unsigned long long)t.numel();
    return t.data_ptr();
}

template <typename F>
PyObject* launch(const char* what, F call) {
    int rc;
    Py_BEGIN_ALLOW_THREADS rc = call();
    Py_END_ALLOW_THREADS
    if (rc) refuse(what, mmz_last_error());
    Py_RETURN_NONE;
}

// a call's body with its exceptions as Python's
template <typename F>
PyObject* guarded(F body) {
    try {
        return body();
    } catch (const Raised&) {
    } catch (const Refused& e) {
        PyErr_SetString(mmz_error, e.what());
    } catch (const std::exception& e) {
        PyErr_SetString(mmz_error, e.what());
    }
    return nullptr;
}

// ---------------------------------------------------------------- the 8-bit cache

struct Cache {
    mmz_kv8 c;
    int64_t batch, heads, cap;
};
Cache cache_of(const char* what, PyObject* const* four, long long block, int dev) {
    const at::Tensor& k8 = cuda_tensor(what, "k8", four[0]);
    const at::ScalarType type = k8.scalar_type();
    if ((type != at::kChar && type != at::kFloat8_e4m3fn) || k8.dim() != 4 || k8.size(3) != 64)
        refuse(what, "k8 is an int8 or float8_e4m3fn tensor [batch][heads][cap][64]");
    if (block != 16 && block != 32 && block != 64 && block != 128) refuse(what, "block is 16, 32, 64 or 128");
    const int64_t b = k8.size(0), h = k8.size(1), cap = k8.size(2), blocks[3] = {b, h, (cap + block - 1) / block};
    const at::Tensor& v8 = shaped(what, "v8", four[1], type, k8.sizes(), dev);
    const at::Tensor& ks = shaped(what, "ks", four[2], at::kFloat, blocks, dev);
    const at::Tensor& vs = shaped(what, "vs", four[3], at::kFloat, blocks, dev);
    const at::IntArrayRef cs = k8.strides(), ss = ks.strides();
    if (!alike(k8, v8) || !alike(ks, vs)) refuse(what, "keys and values of the cache have the same strides");
    if (cs[3] != 1 || (cap > 1 && cs[2] != 64) || (blocks[2] > 1 && ss[2] != 1))
        refuse(what, "a head's rows of the cache, and its scales, lie one after another");
    mmz_kv8 c{k8.data_ptr(), v8.data_ptr(), (float*)ks.data_ptr(), (float*)vs.data_ptr(), step(b, cs[0]), step(h, cs[1]),
              step(b, ss[0]), step(h, ss[1]), narrow(what, "heads", h), narrow(what, "cap", cap), (int)block,
              type == at::kFloat8_e4m3fn};
    return {c, narrow(what, "batch", b), h, cap};
}

struct Tokens {  // k and v [batch][n][heads][64] fp16
    void *k, *v;
    long long seq, tok, head;
    int n;
};
Tokens tokens_of(const char* what, PyObject* ko, PyObject* vo, const Cache& c, int dev) {
    const at::Tensor* given = tensor(ko);
    if (!given || given->dim() != 4) refuse(what, "k is a tensor [batch][n][heads][64]");
    const int64_t n = given->size(1), shape[4] = {c.batch, n, c.heads, 64};
    const at::Tensor& k = shaped(what, "k", ko, at::kHalf, shape, dev);
    const at::Tensor& v = shaped(what, "v", vo, at::kHalf, shape, dev);
    const at::IntArrayRef s = k.strides();
    if (!alike(k, v) || s[3] != 1) refuse(what, "k and v have the same strides, the last dimension dense");
    return {k.data_ptr(), v.data_ptr(), step(c.batch, s[0]), step(n, s[1]), step(c.heads, s[2]), narrow(what, "n", n)};
}

#define NAME(x) PyUnicode_InternFromString(x)

PyObject* kv8_write(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kw) {
    static PyObject* const names[] = {NAME("k"), NAME("v"), NAME("k8"), NAME("v8"), NAME("ks"), NAME("vs"), NAME("block"),
                                      NAME("pos"), NAME("stream")};
    return guarded([&] {
        const char* what = "kv8_write";
        const Params<9> p(what, names, 6, args, nargs, kw);
        const int dev = device_of(what, "k8", p.v[2]);
        const Cache c = cache_of(what, p.v + 2, integer(p.v[6], 64), dev);
        const Tokens x = tokens_of(what, p.v[0], p.v[1], c, dev);
        const int* pos = (const int*)dense(what, "pos", p.v[7], at::kInt, c.batch, dev);
        const Stream st(p.v[8], dev);
        return launch(what, [&] {
            return mmz_kv8_write(&c.c, x.k, x.v, x.seq, x.tok, x.head, pos, (int)c.batch, x.n, st.raw);
        });
    });
}

PyObject* kv8_read(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kw) {
    static PyObject* const names[] = {NAME("k8"), NAME("v8"), NAME("ks"), NAME("vs"), NAME("k"), NAME("v"), NAME("block"),
                                      NAME("pos"), NAME("lens"), NAME("stream")};
    return guarded([&] {
        const char* what = "kv8_read";
        const Params<10> p(what, names, 6, args, nargs, kw);
        const int dev = device_of(what, "k8", p.v[0]);
        const Cache c = cache_of(what, p.v, integer(p.v[6], 64), dev);
        const Tokens x = tokens_of(what, p.v[4], p.v[5], c, dev);
        const int* pos = (const int*)dense(what, "pos", p.v[7], at::kInt, c.batch, dev);
        const int* lens = (const int*)dense(what, "lens", p.v[8], at::kInt, c.batch, dev);
        const Stream st(p.v[9], dev);
        return launch(what, [&] {
            return mmz_kv8_read(&c.c, x.k, x.v, x.seq, x.tok, x.head, pos, lens, (int)c.batch, x.n, st.raw);
        });
    });
}

PyObject* attn8(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kw) {
    static PyObject* const names[] = {NAME("q"), NAME("k8"), NAME("v8"), NAME("ks"), NAME("vs"), NAME("out"), NAME("block"),
                                      NAME("lens"), NAME("causal"), NAME("scale"), NAME("probs"), NAME("pslot"),
                                      NAME("scratch"), NAME("stream")};
    return guarded([&] {
        const char* what = "attn8";
        const Params<14> p(what, names, 6, args, nargs, kw);
        const int dev = device_of(what, "k8", p.v[1]);
        const Cache c = cache_of(what, p.v + 1, integer(p.v[6], 64), dev);
        const at::Tensor* given = tensor(p.v[0]);
        if (!given || given->dim() != 4) refuse(what, "q is a tensor [batch][rows][q_heads][64]");
        const int64_t rows = given->size(1), hq = given->size(2), shape[4] = {c.batch, rows, hq, 64};
        const at::Tensor& q = shaped(what, "q", p.v[0], at::kHalf, shape, dev);
        const at::Tensor& out = shaped(what, "out", p.v[5], at::kHalf, shape, dev);
        const at::IntArrayRef s = q.strides(), o = out.strides();
        if (s[3] != 1 || o[3] != 1) refuse(what, "the last dimension of q and out is dense");
        mmz_attn8_args a{};
        a.q = q.data_ptr(), a.q_seq = step(c.batch, s[0]), a.q_row = step(rows, s[1]), a.q_head = step(hq, s[2]);
        a.out = out.data_ptr(), a.o_seq = step(c.batch, o[0]), a.o_row = step(rows, o[1]), a.o_head = step(hq, o[2]);
        a.batch = (int)c.batch, a.rows = narrow(what, "rows", rows), a.q_heads = narrow(what, "q_heads", hq);
        a.lens = (const int*)dense(what, "lens", p.v[7], at::kInt, c.batch, dev);
        a.causal = p.v[8] ? PyObject_IsTrue(p.v[8]) : 0;
        a.scale = p.v[9] ? (float)PyFloat_AsDouble(p.v[9]) : 0.125f;
        if (PyErr_Occurred()) throw Raised();
        if (p.v[10]) {
            const at::Tensor* probs = tensor(p.v[10]);
            const int64_t slots = probs && probs->dim() == 4 ? probs->size(1) : 1, there[4] = {c.batch, slots, rows, c.cap};
            a.probs = dense(what, "probs", p.v[10], at::kHalf, there, dev);
            a.pslot = (const int*)dense(what, "pslot", p.v[11], at::kInt, hq, dev);
            a.slots = narrow(what, "slots", slots);
        }
        const Stream st(p.v[13], dev);
        at::Tensor own;
        if (p.v[12]) {
            a.scratch = their_scratch(what, p.v[12], dev, &a.scratch_bytes);
        } else if ((a.scratch_bytes = mmz_attn8_scratch_bytes(a.batch, a.rows, a.q_heads, c.c.heads, c.c.cap, a.slots))) {
            own = own_scratch(a.scratch_bytes, st, dev);
            a.scratch = own.data_ptr();
        }
        return launch(what, [&] { return mmz_attn8(&c.c, &a, st.raw); });
    });
}

// ---------------------------------------------------------------- token log probabilities

// the outputs, [rows] each or [rows][steps] with a column counter; v: target, logp, entropy, lse, top_id, top_logp, sup, col
mmz_logprobs outputs_of(const char* what, int64_t rows, PyObject* const* v, int dev) {
    const at::Tensor* logp = tensor(v[1]);
    PyObject* col = v[7];
    if (!logp || logp->dim() != (col ? 2 : 1)) refuse(what, "logp is a tensor [rows], or [rows][steps] with col");
    const int64_t ld = col ? logp->size(1) : 1;
    const at::Tensor* one = tensor(v[4] ? v[4] : v[5]);
    const int64_t top = one && one->dim() ? one->size(-1) : 0, there[3] = {rows, col ? ld : top, top};
    const at::IntArrayRef row(there, col ? 2 : 1), list(there, col ? 3 : 2);
    mmz_logprobs o{};
    o.target = (const int*)dense(what, "target", v[0] == Py_None ? nullptr : v[0], at::kInt, row, dev);
    o.logp = (float*)dense(what, "logp", v[1], at::kFloat, row, dev);
    o.entropy = (float*)dense(what, "entropy", v[2], at::kFloat, row, dev);
    o.lse = (float*)dense(what, "lse", v[3], at::kFloat, row, dev);
    o.top_id = (int*)dense(what, "top_id", v[4], at::kInt, list, dev);
    o.top_logp = (float*)dense(what, "top_logp", v[5], at::kFloat, list, dev);
    o.ld = ld;
    o.top = narrow(what, "top", top);
    if (col) {
        const at::Tensor& t = typed(what, "col", col, at::kInt, dev);
        if (!t.numel()) refuse(what, "col is an int32 tensor of one number");
        o.col = (const int*)t.data_ptr();
    }
    return o;
}

PyObject* token_logprobs(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kw) {
    static PyObject* const names[] = {NAME("logits"), NAME("target"), NAME("logp"), NAME("entropy"), NAME("lse"),
                                      NAME("top_id"), NAME("top_logp"), NAME("sup"), NAME("col"), NAME("stream")};
    return guarded([&] {
        const char* what = "token_logprobs";
        const Params<10> p(what, names, 3, args, nargs, kw);
        const at::Tensor* given = tensor(p.v[0]);
        if (!given || (given->scalar_type() != at::kHalf && given->scalar_type() != at::kFloat) || given->dim() != 2)
            refuse(what, "logits is an fp16 or fp32 tensor [rows][vocab]");
        const int dev = device_of(what, "logits", p.v[0]);
        const at::Tensor& x = *given;
        const int64_t rows = x.size(0), vocab = x.size(1);
        if (x.stride(1) != 1 && vocab > 1) refuse(what, "the last dimension of logits is dense");
        const mmz_logprobs o = outputs_of(what, rows, p.v + 1, dev);
        const unsigned char* sup = (const unsigned char*)dense(what, "sup", p.v[7], at::kByte, vocab, dev);
        const int r = narrow(what, "rows", rows), n = narrow(what, "vocab", vocab), type = x.scalar_type() == at::kFloat;
        const long long ldx = rows > 1 ? x.stride(0) : vocab;
        const void* px = x.data_ptr();
        const Stream st(p.v[9], dev);
        return launch(what, [&] { return mmz_token_logprobs(px, ldx, type, r, n, sup, &o, st.raw); });
    });
}

PyObject* linear_logprobs(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kw) {
    static PyObject* const names[] = {NAME("x"), NAME("emb"), NAME("target"), NAME("logp"), NAME("entropy"), NAME("lse"),
                                      NAME("top_id"), NAME("top_logp"), NAME("sup"), NAME("col"), NAME("scratch"),
                                      NAME("stream")};
    return guarded([&] {
        const char* what = "linear_logprobs";
        const Params<12> p(what, names, 4, args, nargs, kw);
        const at::Tensor *xt = tensor(p.v[0]), *et = tensor(p.v[1]);
        if (!xt || !et || xt->dim() != 2 || et->dim() != 2) refuse(what, "x [rows][d] and emb [vocab][d] are tensors");
        const int dev = device_of(what, "x", p.v[0]);
        const at::Tensor& x = typed(what, "x", p.v[0], at::kHalf, dev);
        const int64_t rows = x.size(0), d = x.size(1), vocab = et->size(0), table[2] = {vocab, d};
        const void* emb = dense(what, "emb", p.v[1], at::kHalf, table, dev);
        if (x.stride(1) != 1) refuse(what, "the last dimension of x is dense");
        const mmz_logprobs o = outputs_of(what, rows, p.v + 2, dev);
        const unsigned char* sup = (const unsigned char*)dense(what, "sup", p.v[8], at::kByte, vocab, dev);
        const int r = narrow(what, "rows", rows), n = narrow(what, "vocab", vocab), w = narrow(what, "width", d);
        const long long ldx = rows > 1 ? x.stride(0) : d;
        const void* px = x.data_ptr();
        const Stream st(p.v[11], dev);
        at::Tensor own;
        void* scratch = nullptr;
        unsigned long long bytes = 0;
        if (p.v[10]) {
            scratch = their_scratch(what, p.v[10], dev, &bytes);
        } else if ((bytes = mmz_linear_logprobs_scratch_bytes(r, n, w))) {
            own = own_scratch(bytes, st, dev);
            scratch = own.data_ptr();
        }
        return launch(what, [&] { return mmz_linear_logprobs(px, ldx, emb, r, n, w, sup, &o, scratch, bytes, st.raw); });
    });
}

#define CALL(f) (PyCFunction)(void (*)(void)) f, METH_FASTCALL | METH_KEYWORDS

PyMethodDef methods[] = {
    {"kv8_write", CALL(kv8_write),
     "kv8_write(k, v, k8, v8, ks, vs, block=64, pos=None, stream=None)\n--\n\n"
     "Quantises the tokens k, v [b][n][heads][64] fp16 into the cache k8, v8 [b][heads][cap][64] (int8 or\n"
     "float8_e4m3fn) with the scales ks, vs [b][heads][ceil(cap / block)] float32, at positions pos[b].. (int32 [b]; None:\n"
     "from 0). A block that already has tokens keeps at least its scale; its codes are rounded again when it grows."},
    {"kv8_read", CALL(kv8_read),
     "kv8_read(k8, v8, ks, vs, k, v, block=64, pos=None, lens=None, stream=None)\n--\n\n"
     "The cache's values at positions pos[b].. (None: from 0) into k, v [b][n][heads][64] fp16, zeros from position\n"
     "min(lens[b], cap) on (lens None: cap)."},
    {"attn8", CALL(attn8),
     "attn8(q, k8, v8, ks, vs, out, block=64, lens=None, causal=False, scale=0.125, probs=None, pslot=None, scratch=None, "
     "stream=None)\n--\n\n"
     "Attention of q [b][rows][q_heads][64] fp16 over the cache's first lens[b] positions (int32 [b]; None: all of\n"
     "them), into out of the same shape (q itself, or apart from it); causal: the rows are the sequence's last ones, row i\n"
     "sees lens - rows + i + 1 positions. A row that sees nothing gives zeros. probs [b][slots][rows][cap] fp16 receives\n"
     "the probabilities of the heads with pslot[head] >= 0 (int32 [q_heads]). scratch: a uint8 tensor of\n"
     "attn8_scratch_bytes(...) (allocated here when None and needed)."},
    {"token_logprobs", CALL(token_logprobs),
     "token_logprobs(logits, target, logp, entropy=None, lse=None, top_id=None, top_logp=None, sup=None, col=None, "
     "stream=None)\n--\n\n"
     "Per row of logits [rows][vocab] (fp16 or fp32): logp[r] = log p(target[r]), the entropy, log sum e^x, and the\n"
     "ids and log probabilities of the largest logits (top_id int32, top_logp float32 [rows][top <= 8]; ties to the lower\n"
     "id). sup [vocab] uint8: ids left out. With col (an int32 device scalar) target and outputs are [rows][steps] and\n"
     "column col[0] is read and written. A target outside the vocabulary has logp 0."},
    {"linear_logprobs", CALL(linear_logprobs),
     "linear_logprobs(x, emb, target, logp, entropy=None, lse=None, top_id=None, top_logp=None, sup=None, col=None, "
     "scratch=None, stream=None)\n--\n\n"
     "token_logprobs of the logits x . emb^T (x [rows][d], emb [vocab][d] fp16), in fp32 from the product on. scratch:\n"
     "a uint8 tensor of linear_logprobs_scratch_bytes(rows, vocab, d) (allocated here when None)."},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "mimizuku_b200._serving", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__serving() {
    PyObject* package = PyImport_ImportModule("mimizuku_b200");
    if (!package) return nullptr;
    mmz_error = PyObject_GetAttrString(package, "MmzError");
    Py_DECREF(package);
    return mmz_error ? PyModule_Create(&module) : nullptr;
}
