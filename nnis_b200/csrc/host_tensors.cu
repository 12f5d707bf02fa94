// Tensors of a call looked at together, on the host.  An operator over the 8-bit cache takes ten tensors; their types, shapes, devices,
// strides and addresses read one attribute at a time in Python take 4 us, more than the launch, here 0.9.  Tensors are read through the
// exchange interface that torch.Tensor publishes for native code (DLPack 1.3: a table of functions in a capsule, one of which describes a
// tensor without owning it), so the library needs neither torch's headers nor its libraries.  The interpreter's functions are looked up
// when the first check is made; the library itself does not depend on one.
#include <dlfcn.h>
#include <string.h>

#include "common.cuh"

namespace {

// ---- the exchange interface, as its standard lays it out
struct ExchangedTensor {
    void* data;
    int32_t device_type, device_id;  // 2: CUDA
    int32_t ndim;
    uint8_t type, bits;  // 0 whole numbers, 2 floating point, 4 bfloat16
    uint16_t lanes;
    int64_t *shape, *strides;
    uint64_t byte_offset;
};
struct Exchange {
    uint32_t major, minor;
    void* older;
    void *allocate, *own, *give;
    int (*describe)(void* object, ExchangedTensor* out);  // 0, or -1 and an exception
    int (*stream)(int32_t device_type, int32_t device_id, void** out);
};

struct Method {  // of the interpreter's stable interface
    const char* name;
    void* function;
    int flags;
    const char* doc;
};
constexpr int kFastCall = 0x0080;

struct Interpreter {
    int (*is_instance)(void*, void*);
    long long (*as_long)(void*);
    void* (*from_long)(long long);
    double (*as_double)(void*);
    void* (*new_tuple)(long);
    int (*set_item)(void*, long, void*);  // takes the reference
    void* (*error)();
    void (*clear)();
    char* (*bytes)(void*);
    void* (*new_function)(Method*, void* self, void* module);
    void* (*leave)();
    void (*enter)(void*);
    void (*hold)(void*);
    void (*release)(void*);
    void* none;
    bool found;
};

template <typename F>
bool look_up(F& f, const char* name) {
    f = reinterpret_cast<F>(dlsym(RTLD_DEFAULT, name));
    return f != nullptr;
}
Interpreter interpreter() {
    Interpreter p;
    p.found = look_up(p.is_instance, "PyObject_IsInstance") && look_up(p.as_long, "PyLong_AsLongLong") &&
              look_up(p.from_long, "PyLong_FromLongLong") && look_up(p.as_double, "PyFloat_AsDouble") && look_up(p.new_tuple, "PyTuple_New") &&
              look_up(p.set_item, "PyTuple_SetItem") && look_up(p.error, "PyErr_Occurred") && look_up(p.clear, "PyErr_Clear") &&
              look_up(p.bytes, "PyBytes_AsString") && look_up(p.new_function, "PyCFunction_NewEx") && look_up(p.leave, "PyEval_SaveThread") &&
              look_up(p.enter, "PyEval_RestoreThread") && look_up(p.hold, "Py_IncRef") && look_up(p.release, "Py_DecRef") &&
              look_up(p.none, "_Py_NoneStruct");
    return p;
}
const Interpreter& py() {
    static const Interpreter p = interpreter();
    return p;
}
const Exchange* exchange = nullptr;  // set once, under the interpreter's lock
void* tensor_class = nullptr;

void* none() {
    py().hold(py().none);
    return py().none;
}

constexpr int kSymbols = 32, kTensors = 16;
constexpr long long kUnbound = -0x7fffffffffffffffLL - 1;
enum { PACKED = 0, AT_LEAST = 1, ROWS = 2 };  // how a tensor lies; as many elements as a symbol says, in any shape; rows at a distance
enum { ANY_FLOAT = 0, FLOAT32 = 1, INT8 = 2, INT32 = 3 };

// The places of the tensors of a call, or false where something is not as its description says.  `what`: for every tensor its type, how it
// lies, whether it may be None, how many sizes, a symbol for each (AT_LEAST: the one), and for ROWS one for the distance of rows.
// A symbol stands for one value in all of a call's tensors.
bool places(const unsigned char* what, int device_type, int tensors, void* const* args, long long* symbols, long long* at, long long& device, long long& dtype) {
    device = dtype = -1;
    auto is = [&](int symbol, long long value) {
        if (symbols[symbol] == kUnbound) symbols[symbol] = value;
        return symbols[symbol] == value;
    };
    for (int i = 0; i < tensors; ++i) {
        const int type = what[0], lies = what[1], optional = what[2], sizes = what[3];
        const unsigned char* names = what + 4;
        what = names + sizes + (lies == ROWS ? 1 : 0);
        at[i] = 0;
        if (optional && args[i] == py().none) continue;
        ExchangedTensor t;
        if (py().is_instance(args[i], tensor_class) != 1 || exchange->describe(args[i], &t) != 0) return false;
        if (t.device_type != device_type || t.lanes != 1 || (device >= 0 && t.device_id != device)) return false;
        device = t.device_id;
        at[i] = reinterpret_cast<long long>(t.data) + (long long)t.byte_offset;
        const bool f32 = t.type == 2 && t.bits == 32, bf16 = t.type == 4 && t.bits == 16;
        if (type == ANY_FLOAT) {
            const long long code = f32 ? NNIS_DTYPE_F32 : NNIS_DTYPE_BF16;
            if (!(f32 || bf16) || (dtype >= 0 && dtype != code)) return false;
            dtype = code;
        } else if (type == FLOAT32 ? !f32 : t.type != 0 || t.bits != (type == INT8 ? 8 : 32)) {
            return false;
        }
        long long count = 1;  // elements behind the size that is looked at, and in the end all
        bool packed = true, empty = false;
        for (int s = t.ndim - 1; s >= 0; --s) {
            empty = empty || t.shape[s] == 0;
            packed = packed && (t.shape[s] == 1 || !t.strides || t.strides[s] == count);
            count *= t.shape[s];
        }
        if (lies == AT_LEAST) {
            if (!(packed || empty) || symbols[names[0]] == kUnbound || count < symbols[names[0]]) return false;
            continue;
        }
        if (t.ndim != sizes) return false;
        for (int s = 0; s < sizes; ++s)
            if (!is(names[s], t.shape[s])) return false;
        if (lies == PACKED) {
            if (!(packed || empty)) return false;
        } else {  // (rows of one value, and a single row, lie anyhow)
            if (sizes != 2 || (t.strides && t.strides[1] != 1 && t.shape[1] > 1)) return false;
            if (!is(names[2], t.shape[0] > 1 && t.strides ? t.strides[0] : t.shape[1])) return false;
        }
    }
    return true;
}

// self: bytes, the numbers of symbols that are given, of all symbols and of tensors, the type of device, then the tensors' descriptions.  Called with the given
// symbols' values and the tensors.  None where something does not fit, else (device, torch's current stream there or -1 where another device is the
// current one, float type or -1, the other symbols' values, the tensors' addresses).  One that is None counts for nothing but an address of 0.
void* check(void* self, void* const* args, long count) {
    const unsigned char* what = reinterpret_cast<const unsigned char*>(py().bytes(self));
    const int given = what[0], all = what[1], tensors = what[2];
    if (count != given + tensors || all > kSymbols || tensors > kTensors) return none();
    long long symbols[kSymbols], at[kTensors], device, dtype;
    for (int i = 0; i < all; ++i) {
        symbols[i] = i < given ? py().as_long(args[i]) : kUnbound;
        if (i < given && symbols[i] == -1 && py().error()) {
            py().clear();
            return none();
        }
    }
    if (!places(what + 4, what[3], tensors, args + given, symbols, at, device, dtype)) {
        if (py().error()) py().clear();
        return none();
    }
    void* stream = nullptr;
    int current = (int)device;
    const bool here = what[3] != 2 || (cudaGetDevice(&current) == cudaSuccess && current == (int)device);
    if (what[3] == 2 && here && exchange->stream(2, (int32_t)device, &stream) != 0) {
        py().clear();
        return none();
    }
    void* facts = py().new_tuple(3 + all - given + tensors);
    if (!facts) return nullptr;
    long n = 0;
    auto put = [&](long long v) {
        void* number = py().from_long(v);
        if (number) py().set_item(facts, n++, number);
        return number != nullptr;
    };
    bool whole = put(device) && put(here ? reinterpret_cast<long long>(stream) : -1) && put(dtype);
    for (int i = given; whole && i < all; ++i) whole = put(symbols[i] == kUnbound ? -1 : symbols[i]);
    for (int i = 0; whole && i < tensors; ++i) whole = put(at[i]);
    if (whole) return facts;
    py().release(facts);
    return nullptr;
}

// self: bytes, the address of an entry that takes a record, then the record's fields (p: an address or another whole number of 64 bits, i: an int, f: a
// float), ended by a zero.
// Called with their values: the entry's code, NNIS_ERR_ARGUMENT where a value is not one of its field.  The interpreter's lock is not held
// meanwhile: a launch may have to wait for the launches ahead of it.
void* call(void* self, void* const* args, long count) {
    const char* what = py().bytes(self);
    int (*entry)(const void*);
    memcpy(&entry, what, sizeof entry);
    const char* fields = what + sizeof entry;
    alignas(8) unsigned char record[320];
    size_t at = 0;
    bool fits = true;
    long i = 0;
    for (; fits && fields[i] && i < count; ++i) {
        if (fields[i] == 'f') {
            const float v = (float)py().as_double(args[i]);
            fits = !py().error();
            memcpy(record + at, &v, 4);
            at += 4;
            continue;
        }
        const long long v = py().as_long(args[i]);
        if (v == -1 && py().error()) {
            fits = false;
        } else if (fields[i] == 'p') {
            at = (at + 7) / 8 * 8;
            memcpy(record + at, &v, 8);
            at += 8;
        } else {
            const int32_t w = (int32_t)v;
            fits = w == v;
            memcpy(record + at, &w, 4);
            at += 4;
        }
        fits = fits && at + 8 <= sizeof record;
    }
    fits = fits && !fields[i] && i == count;
    if (py().error()) {
        py().clear();
        fits = false;
    }
    if (!fits) return py().from_long(NNIS_ERR_ARGUMENT);
    void* thread = py().leave();
    const int code = entry(record);
    py().enter(thread);
    return py().from_long(code);
}

}  // namespace

// Once, before the others, with the interpreter's lock held: the address of the exchange interface and the class of tensors.
NNIS_API int nnis_tensors_begin(void* interface, void* tensors) {
    const Exchange* e = static_cast<const Exchange*>(interface);
    if (!py().found || !e || e->major != 1 || e->minor < 3 || !e->describe || !e->stream || !tensors) return NNIS_ERR_UNSUPPORTED;
    py().hold(tensors);
    exchange = e;
    tensor_class = tensors;
    return NNIS_OK;
}

// A function of the interpreter: 0 checks the tensors that the bytes describe, 1 calls the entry that they name.
NNIS_API void* nnis_host_function(int which, void* description) {
    static Method methods[2] = {{"tensors_of_a_call", reinterpret_cast<void*>(check), kFastCall, nullptr},
                                {"call_of_a_record", reinterpret_cast<void*>(call), kFastCall, nullptr}};
    return py().new_function(&methods[which ? 1 : 0], description, nullptr);
}
