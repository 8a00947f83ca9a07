// Shared host-side helpers of the C-ABI launchers: error reporting and launch checks.
#pragma once

#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdio>

#include "../../include/sfnx_b200.h"

namespace fnxk {

// the calling thread's last error text (fnx_last_error)
char* err_buf();
int fail(const char* fmt, ...);
// cudaGetLastError after a launch: 0, or the failure recorded under `what`
int launch_ok(const char* what);
// kernels launched by this library so far (every launch is checked by one launch_ok()); reset: read and zero
long launch_count(bool reset);

inline cudaStream_t strm(void* st) { return (cudaStream_t) st; }

// ---- programmatic dependent launch.  A kernel launched through launch() may be scheduled while the kernel before
// it in the stream still runs: its blocks do what does not depend on that kernel (index arithmetic, the first loads
// of weights) and then call pdl_wait(), which returns once the kernel before has finished and its writes are visible.
// Rules every such kernel keeps: before pdl_wait() it reads nothing the kernel directly before it writes and writes
// no global memory; it calls pdl_go() only after pdl_wait(), so the kernel after it overlaps with this one and with
// nothing older.  Off (plain stream order) while a window is traced, since the trace times single kernels, and with
// FNX_NO_PDL set.
bool pdl_on(int kind);   // kind: a launch site's class, for FNX_PDL_MASK (a tuning knob: bit k switches class k)
void pdl_hold(bool hold);   // the trace's switch

template <typename... KArgs, typename... Args>
inline void launch(int kind, void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid, cfg.blockDim = block, cfg.dynamicSmemBytes = smem, cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at, cfg.numAttrs = pdl_on(kind) ? 1 : 0;
    cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...);   // a failure shows in launch_ok()
}

#ifdef __CUDACC__
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_go() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
// two 32-bit operations an instruction, each rounded by itself
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n\t.reg .b64 x, y, w, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 w, {%6, %7};\n\tfma.rn.f32x2 z, x, y, w;\n\tmov.b64 {%0, %1}, "
        "z;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
// 2^x by the special-function unit (2^-22 relative), denormal results zero
__device__ __forceinline__ float ex2_ftz(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// brings a line into L2, for what may be written until pdl_wait() returns and so must not be read before it
__device__ __forceinline__ void l2_ask(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
#endif

#define FNX_REQUIRE(cond, ...) \
    do {                       \
        if (!(cond)) return fnxk::fail(__VA_ARGS__); \
    } while (0)

}  // namespace fnxk
