// What the host sides of this library share: a context (device, stream, resident weights), growing device and pinned
// buffers, error reporting, kernel launches and the TMA tensor maps. Included by each .cu file that implements entry
// points of include/ktmoe.h.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <mutex>
#include <string>
#include <unordered_map>
#include <utility>

#include "digit_gemm.cuh"
#include "fixed_point.cuh"
#include "host_prep.h"
#include "ktmoe.h"

using kt::Scale;

namespace ktc {

inline int64_t round_up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }
inline Scale S(ktmoe_scale s) { return Scale{s.mant, s.shift}; }
inline ktmoe_scale C(Scale s) { return ktmoe_scale{s.mant, s.shift}; }
inline Scale S(hp::HScale s) { return Scale{s.mant, s.shift}; }

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = (EncodeTiledFn)p;
    });
    return fn;
}

// A device buffer that only grows.
struct DevBuf {
    void* p = nullptr;
    size_t bytes = 0;
    cudaError_t ensure(size_t want) {
        if (want <= bytes) return cudaSuccess;
        if (p) cudaFree(p);
        p = nullptr;
        bytes = 0;
        cudaError_t e = cudaMalloc(&p, want);
        if (e == cudaSuccess) bytes = want;
        return e;
    }
    void release() {
        if (p) cudaFree(p);
        p = nullptr;
        bytes = 0;
    }
    template <class T>
    T* as() const {
        return (T*)p;
    }
};

// Pinned host memory, grown on demand (the staging of small LinearBackend transfers).
struct HostBuf {
    void* p = nullptr;
    size_t bytes = 0;
    cudaError_t ensure(size_t want) {
        if (want <= bytes) return cudaSuccess;
        if (p) cudaFreeHost(p);
        p = nullptr;
        bytes = 0;
        cudaError_t e = cudaHostAlloc(&p, want, cudaHostAllocDefault);
        if (e == cudaSuccess) bytes = want;
        return e;
    }
    void release() {
        if (p) cudaFreeHost(p);
        p = nullptr;
        bytes = 0;
    }
};

// Digit planes: [groups][3][rows_pad][k_pad] int8.
struct Planes {
    int8_t* ptr = nullptr;
    int64_t groups = 1, rows_pad = 0, k = 0, k_pad = 0;
};

struct Resident {
    DevBuf buf;
    int64_t out = 0, k = 0, out_pad = 0, k_pad = 0;
    bool small = false;  // every code within ±3280: planes 0 and 1 hold it, plane 2 is zero
    uint64_t last_use = 0;
};

}  // namespace ktc

using ktc::DevBuf;
using ktc::HostBuf;
using ktc::Planes;
using ktc::Resident;

struct ktmoe_ctx {
    int device = 0;
    int num_sms = 148;
    int pair_clusters = 0;  // co-resident clusters of the pair GEMM on this device (0: not yet queried)
    cudaStream_t stream = nullptr;
    cudaStream_t side = nullptr;  // the shared expert runs here, beside the routed experts
    cudaEvent_t ev_fork = nullptr, ev_join = nullptr;
    cudaEvent_t ev_g0 = nullptr, ev_g1 = nullptr;  // around the last linear call's GEMM (ktmoe_linear_last_gemm)
    int last_gemm_planes = 0;                      // 0: no GEMM timed yet; 3: nine-plane kernel; 1: (1, 2) kernel
    int* d_err = nullptr;  // [2]
    // pinned host words for the status a linear call reads back with its result: [0..2] the packing counters, [3]
    // the error word (one synchronisation for both, instead of a blocking copy each)
    unsigned long long* h_status = nullptr;
    std::string last_error = "";
    uint64_t launches = 0;
    std::mutex mu;
    // LinearBackend scratch
    DevBuf lin_xi, lin_wi, lin_xp, lin_xr, lin_wp, lin_y, lin_bad;
    // pinned staging of a call's activations and result up to LIN_STAGE_MAX bytes each: a copy through pageable
    // memory costs the driver's own staging and a blocking wait per transfer, which dominate decode-sized calls
    HostBuf lin_hx, lin_hy;
    // resident weights (linear_weights)
    std::unordered_map<uint64_t, Resident*> cache;
    uint64_t budget = 0, resident = 0, tick = 0;
};

namespace ktc {

inline int fail(ktmoe_ctx* ctx, int status, const std::string& what) {
    if (ctx) ctx->last_error = what;
    return status;
}

inline int fail_cuda(ktmoe_ctx* ctx, cudaError_t e, const char* what) {
    return fail(ctx, KTMOE_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

#define CK(expr)                                                        \
    do {                                                                \
        cudaError_t e__ = (expr);                                       \
        if (e__ != cudaSuccess) return fail_cuda(ctx, e__, #expr);      \
    } while (0)

#define CKL(ctx)                                                        \
    do {                                                                \
        ++(ctx)->launches;                                              \
        cudaError_t e__ = cudaGetLastError();                           \
        if (e__ != cudaSuccess) return fail_cuda(ctx, e__, "kernel launch"); \
    } while (0)

// Programmatic dependent launch of this library's kernels (every one begins with kt::pdl_enter(), which waits for
// the kernel before it on the stream): a kernel is scheduled while its predecessor finishes, which hides most of the
// gap between two dependent launches. KTMOE_PDL=0, read once, launches them plainly.
inline bool pdl_on() {
    static const bool on = [] {
        const char* e = getenv("KTMOE_PDL");
        return !(e && e[0] == '0');
    }();
    return on;
}

// One launch of `kernel` on clusters of `cluster` CTAs along x (1: no cluster attribute).
template <typename... KArgs, typename... Args>
int launch_kc(ktmoe_ctx* ctx, cudaStream_t st, dim3 grid, dim3 block, size_t smem, unsigned cluster,
              void (*kernel)(KArgs...), Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    int na = 0;
    if (pdl_on()) {
        at[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[na].val.programmaticStreamSerializationAllowed = 1;
        ++na;
    }
    if (cluster > 1) {
        at[na].id = cudaLaunchAttributeClusterDimension;
        at[na].val.clusterDim.x = cluster;
        at[na].val.clusterDim.y = 1;
        at[na].val.clusterDim.z = 1;
        ++na;
    }
    cfg.attrs = at;
    cfg.numAttrs = na;
    CK(cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...));
    CKL(ctx);
    return KTMOE_OK;
}

template <typename... KArgs, typename... Args>
int launch_k(ktmoe_ctx* ctx, cudaStream_t st, dim3 grid, dim3 block, size_t smem, void (*kernel)(KArgs...),
             Args&&... args) {
    return launch_kc(ctx, st, grid, block, smem, 1u, kernel, std::forward<Args>(args)...);
}

// KLAUNCH(stream, grid, block, shared bytes, (kernel), args...): launch_k, returning its status on failure; one
// statement (safe under an unbraced if / else).
#define KLAUNCH(...)                                                   \
    do {                                                               \
        if (int r_kl__ = launch_k(ctx, __VA_ARGS__)) return r_kl__;    \
    } while (0)
// KLAUNCHC(stream, grid, block, shared bytes, cluster size, (kernel), args...): the same through launch_kc.
#define KLAUNCHC(...)                                                  \
    do {                                                               \
        if (int r_kl__ = launch_kc(ctx, __VA_ARGS__)) return r_kl__;   \
    } while (0)

inline int make_map(ktmoe_ctx* ctx, CUtensorMap* map, const void* base, int64_t k_pad, int64_t rows_total, int box_rows) {
    EncodeTiledFn enc = encode_fn();
    if (!enc) return fail(ctx, KTMOE_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
    cuuint64_t gdim[2] = {(cuuint64_t)k_pad, (cuuint64_t)rows_total};
    cuuint64_t gstride[1] = {(cuuint64_t)k_pad};
    cuuint32_t box[2] = {(cuuint32_t)dg::BK, (cuuint32_t)box_rows};
    cuuint32_t estride[2] = {1, 1};
    CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), gdim, gstride, box, estride,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(ctx, KTMOE_ERR_CUDA, "cuTensorMapEncodeTiled failed (" + std::to_string((int)r) + ")");
    return KTMOE_OK;
}

inline int set_device(ktmoe_ctx* ctx) {
    CK(cudaSetDevice(ctx->device));
    return KTMOE_OK;
}

// What a kernel leaves in the second error word: something wrong in a batch description that only the device could see
// (kv_kernels.cuh). The first word has the code of a bounded wait that expired, and ends the other waits of the context.
enum : int { ERR_BAD_PAGE = 1, ERR_BAD_LENGTH = 2, ERR_BAD_POSITION = 3 };

inline int fail_err_word(ktmoe_ctx* ctx, int code) {
    return fail(ctx, KTMOE_ERR_KERNEL, "a kernel's bounded wait expired (code " + std::to_string(code) + ")");
}

// The first error word; with `batches` the second one too.
inline int check_err_word(ktmoe_ctx* ctx, bool batches = false) {
    int h[2] = {0, 0};
    CK(cudaMemcpy(h, ctx->d_err, batches ? sizeof(h) : sizeof(int), cudaMemcpyDeviceToHost));
    if (h[0] == 0 && h[1] == 0) return KTMOE_OK;
    CK(cudaMemset(ctx->d_err, 0, batches ? sizeof(h) : sizeof(int)));
    if (h[0] != 0) return fail_err_word(ctx, h[0]);
    return fail(ctx, KTMOE_ERR_ARG,
                h[1] == ERR_BAD_PAGE     ? "a page table entry lies outside the cache's pages"
                : h[1] == ERR_BAD_LENGTH ? "a batch's row offsets or lengths do not fit its rows and page table"
                                         : "a position lies beyond the rotation table");
}

}  // namespace ktc

using namespace ktc;
