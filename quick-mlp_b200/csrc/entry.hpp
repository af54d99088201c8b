// What the extern "C" entry points share: argument checks in the style of the reference's CHECK_* macros
// (src_cpp/include/qmlp/errors.h:78-90), exception -> status-code translation, per-kernel timing.
#pragma once
#include "host.hpp"

#include <cuda_runtime.h>

namespace qmlp {

#define QMLP_TRY try {
#define QMLP_CATCH                                                                                              \
    }                                                                                                           \
    catch (const qmlp::configuration_error& e) { return qmlp::reportError(QMLP_ERROR_CONFIGURATION, e.what()); } \
    catch (const qmlp::cuda_error& e) { return qmlp::reportError(QMLP_ERROR_CUDA, e.what()); }                  \
    catch (const qmlp::compile_error& e) { return qmlp::reportError(QMLP_ERROR_COMPILE, e.what()); }            \
    catch (const std::exception& e) { return qmlp::reportError(QMLP_ERROR_RUNTIME, e.what()); }                 \
    catch (...) { return qmlp::reportError(QMLP_ERROR_RUNTIME, "unknown error"); }                              \
    return QMLP_OK;

inline void checkCuda(cudaError_t e, const char* what)
{
    if (e == cudaSuccess) return;
    (void)cudaGetLastError();   // reported here: the check after the next launch must not find it again
    throw cuda_error(std::string(what) + ": " + cudaGetErrorString(e));
}
inline void checkLaunch(int e, const char* what)
{
    if (e != 0) throw cuda_error(std::string(what) + ": " + cudaGetErrorString(static_cast<cudaError_t>(e)));
}

inline void checkDefined(const qmlp_tensor_t* t, const char* name)
{
    if (t == nullptr || t->ndim <= 0) throw std::runtime_error(std::string(name) + " is undefined");
    bool empty = false;
    for (int i = 0; i < t->ndim && i < 2; ++i) empty = empty || t->sizes[i] == 0;
    if (t->data == nullptr && !empty) throw std::runtime_error(std::string(name) + " is undefined");
}
inline void checkDim(const qmlp_tensor_t* t, int dim, const char* name)
{
    checkDefined(t, name);
    if (t->ndim != dim) throw std::runtime_error(format("%s has the wrong dimension, expected %d but got %d", name, dim, t->ndim));
}
inline void checkSize(const qmlp_tensor_t* t, int d, int64_t size, const char* name)
{
    if (t->sizes[d] != size)
        throw std::runtime_error(format("%s has the wrong size at dimension %d, expected %lld but got %lld", name, d,
                                        static_cast<long long>(size), static_cast<long long>(t->sizes[d])));
}
inline const char* precisionName(int precision)
{
    static const char* names[] = {"float", "half", "double", "bfloat16", "int32", "int64"};
    return precision >= 0 && precision < 6 ? names[precision] : "unknown";
}
inline void checkDtype(const qmlp_tensor_t* t, int precision, const char* name)
{
    if (t->precision != precision)
        throw std::runtime_error(format("%s has the wrong data type, expected %s", name, precisionName(precision)));
}

// Optional per-kernel device timing (qmlp_set_kernel_timing): an event pair around every launch the library makes,
// read back and summed per kernel by qmlp_read_kernel_timing. Off by default: the events cost a little.
struct KernelTimer {
    struct Record { int id; cudaEvent_t begin, end; };
    std::mutex mutex;
    bool enabled = false;
    std::vector<Record> records;
};
extern KernelTimer g_timer;

struct TimedLaunch {
    int id;
    cudaStream_t stream;
    cudaEvent_t begin = nullptr, end = nullptr;
    TimedLaunch(int kernelId, cudaStream_t s) : id(kernelId), stream(s)
    {
        if (!g_timer.enabled) return;
        if (cudaEventCreate(&begin) != cudaSuccess || cudaEventCreate(&end) != cudaSuccess) { begin = end = nullptr; return; }
        cudaEventRecord(begin, stream);
    }
    ~TimedLaunch()
    {
        if (!begin) return;
        cudaEventRecord(end, stream);
        std::lock_guard<std::mutex> lock(g_timer.mutex);
        g_timer.records.push_back({id, begin, end});
    }
};

} // namespace qmlp
