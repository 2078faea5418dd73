// What the files of the C ABI share: errors, the per-device context, tensor maps.  Nothing here is exported.
#pragma once
#include "../../include/nvfp4_b200.h"

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <cstring>
#include <string>

#define NVFP4_HIDDEN __attribute__((visibility("hidden")))

namespace nvfp4 {
namespace host {

extern NVFP4_HIDDEN thread_local const char* t_last_kernel;
extern NVFP4_HIDDEN std::atomic<uint64_t> g_launches;
extern NVFP4_HIDDEN std::atomic<uint64_t> g_timeout_ns;

// Notes the message for nvfp4_last_error() and returns `code`.
NVFP4_HIDDEN int fail(int code, const char* fmt, ...);

#define CUDA_TRY(expr)                                                                             \
    do {                                                                                           \
        cudaError_t e__ = (expr);                                                                  \
        if (e__ != cudaSuccess) return fail(NVFP4_ERR_CUDA, "%s failed: %s", #expr, cudaGetErrorString(e__)); \
    } while (0)

// What a tensor map is encoded from.
struct MapKey {
    const void* ptr;
    uint64_t dims[4];
    uint64_t strides[3];
    uint32_t box[4];
    int dtype;
    int rank;
    int swizzle;
};

constexpr int kStreamSets = 8;   // scratch sets of a device (see nvfp4_api.cu)

struct DeviceCtx {
    int device = -1;
    int num_sms = 0;
    bool sm100 = false;
    float* scratch = nullptr;    // kStreamSets sets of partial-tile slots
    int* counters = nullptr;     // kStreamSets sets of tile counters
    cudaStream_t set_stream[kStreamSets] = {};
    bool set_used[kStreamSets] = {};
    bool set_in_graph[kStreamSets] = {};   // a launch with this set was recorded into a CUDA graph
    int* status_host = nullptr;
    int* status_dev = nullptr;
    size_t scratch_bytes = 0;
    std::atomic<bool> scratch_ready{false};   // scratch and counters are allocated and cleared
    std::atomic<int> max_pairs{-1};      // CTA pairs that can be co-resident (cluster occupancy), queried by the first thread that needs it
    std::atomic<int> expert_pairs{-1};   // the same for the experts' kernel
    std::atomic<bool> smem_attr_set[96] = {};   // by kernel variant: 0..26 the tiled kernels, 32.. the decode kernels, 72.. the experts' kernels
};

// The context of the current device.
NVFP4_HIDDEN int get_ctx(DeviceCtx** out);
// Encodes a tensor map into caller storage.
NVFP4_HIDDEN int encode_map(const MapKey& key, CUtensorMap* out);
// Operand / output tiles: {inner extent, rows, batches}, 128-byte swizzle.
NVFP4_HIDDEN MapKey make_key(const void* ptr, uint64_t d0, uint64_t d1, uint64_t d2, uint64_t s0, uint64_t s1, uint32_t b0, uint32_t b1, int dtype);
// Permuted scale factors of `rows` rows, boxes of the four atoms of a 256-wide k-tile for `blocks` row blocks.
NVFP4_HIDDEN MapKey make_sf_key(const void* ptr, int rows, int k, int l, uint64_t batch_stride, uint32_t blocks);

inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

}  // namespace host
}  // namespace nvfp4
