// What the serving operators of b200serve.h share: the layout of a 4-bit page, division by a page size that is only known
// at run time, launches with clusters and programmatic order.
#pragma once

#include "stream.cuh"
#include "../../include/b200serve.h"

namespace b200 {

// n / d for 0 <= n < 2^31 by one high product, d >= 1: m = floor(2^32 (2^s - d) / d) + 1 with 2^s >= d, n / d =
// (hi(m n) + n) >> s (Granlund and Montgomery's round-up method).
struct FastDiv {
    uint32_t d = 1, m = 1, s = 0;
    FastDiv() = default;
    explicit FastDiv(uint32_t by) : d(by) {
        while (((uint64_t)1 << s) < by) ++s;
        m = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << s) - by)) / by) + 1;
    }
#ifdef __CUDACC__
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(m, n) + n) >> s; }
#endif
};

// Parts of a page, in bytes from its start (the K codes stand first).
struct Kv4Page {
    int64_t k_scale = 0, v_code = 0, v_scale = 0, bytes = 0;
    Kv4Page() = default;
    Kv4Page(int page, int KV, int hd, int kind) {
        auto up = [](int64_t n) { return (n + 127) / 128 * 128; };
        const int64_t codes = up((int64_t)KV * page * (hd / 2)), scales = up((int64_t)KV * page * (hd / 32) * (kind == 1 ? 4 : 2));
        k_scale = codes;
        v_code = codes + scales;
        v_scale = 2 * codes + scales;
        bytes = 2 * (codes + scales);
    }
};
int kv4_check(const char* who, int num_pages, int page, int KV, int hd, int kind);

#ifdef __CUDACC__
// Two fp32 numbers in a register pair: one instruction for both.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 two(float a, float b) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 each(f32x2 x) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
    return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
#endif

static inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// cluster > 1: that many blocks along x form a cluster; early: the kernel is set up while the one before it ends (it waits by itself, in
// its first statement: pdl_wait() or short_begin()).  Grids of short_grid() take it; larger ones would hold SMs that the kernel before
// them still has use for.
template <typename Kern, typename Args>
static int launch_serve(const char* name, Kern kern, dim3 grid, dim3 block, size_t smem, int cluster, bool early, const Args& a) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream();
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = cluster;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        ++n;
    }
    if (early) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return cuda_status(e, name);
    }
    ++g_kernel_launches;
    return B200_OK;
}

}  // namespace b200
