// Host side of what the operators' kernels share.
#include "common.cuh"

#include <mutex>
#include <set>
#include <utility>

namespace qmlp {
namespace kernel {
namespace ops {

cudaError_t allowShared(const void* kernel, int bytes)
{
    static std::mutex mutex;
    static std::set<std::pair<int, const void*>> allowed;
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    std::lock_guard<std::mutex> lock(mutex);
    if (allowed.count({device, kernel}) != 0) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e == cudaSuccess) allowed.insert({device, kernel});
    return e;
}

} // namespace ops
} // namespace kernel
} // namespace qmlp
