// vxc_kv8.cuh — device helpers of the paged 8-bit KV cache (vxc_kv8,
// include/veltrix_cuda.h), shared by its writer and its readers.
#pragma once
#include "vxc_common.cuh"
#include "vxc_internal.h"
#include "vxc_ptx.cuh"

#define KV8_MAX_BS 256               // tokens per block at most
#define KV8_MAX_TOKENS (1ll << 30)   // tokens of a table row at most (positions and splits are ints)

// Largest code of a type.
__host__ __device__ constexpr float kv8_qmax(int type) { return type == VXC_KV8_INT8 ? 127.0f : 448.0f; }

// Exponent of the smallest power of two s with amax <= qmax * s, at least
// -126 (amax > 0 finite).  qmax is 1.984375 * 2^6 or 1.75 * 2^8, so the
// comparison is one of significand bits.
__device__ __forceinline__ int kv8_scale_exp(float amax, int type) {
    const uint32_t u = __float_as_uint(amax);
    const int k = (int)(u >> 23) - 127;
    const uint32_t f = u & 0x7FFFFFu;
    const int e = type == VXC_KV8_INT8 ? k - 6 + (f > 0x7E0000u) : k - 8 + (f > 0x600000u);
    return e < -126 ? -126 : e;
}

// Four integer codes of x * inv, inv a power of two, |x * inv| <= 127: the sum
// with 1.5 * 2^23 is rounded to an integer (once: the product is exact), which
// its low byte holds.
__device__ __forceinline__ uint32_t kv8_pack4_int8(float a, float b, float c, float d, float inv) {
    const float big = 12582912.0f;
    const uint32_t x = __float_as_uint(__fmaf_rn(a, inv, big)), y = __float_as_uint(__fmaf_rn(b, inv, big));
    const uint32_t z = __float_as_uint(__fmaf_rn(c, inv, big)), w = __float_as_uint(__fmaf_rn(d, inv, big));
    return __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, w, 0x0040), 0x5410);
}

// Four codes of x[] (already in units of the scale) as one word, to nearest,
// ties to even.
template <int TYPE>
__device__ __forceinline__ uint32_t kv8_pack4(float a, float b, float c, float d) {
    if (TYPE == VXC_KV8_INT8) return kv8_pack4_int8(a, b, c, d, 1.0f);
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return (uint32_t)lo | ((uint32_t)hi << 16);
}

// Two codes (bytes 0 and 1 of w) as half2: exact for both types.
__device__ __forceinline__ uint32_t kv8_e4m3x2_h2(uint16_t w) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(w));
    return r;
}

// One code as a float.
template <int TYPE>
__device__ __forceinline__ float kv8_value(uint8_t c) {
    if (TYPE == VXC_KV8_INT8) return (float)(int8_t)c;
    const uint32_t h = kv8_e4m3x2_h2(c);
    return vxc_h2f((uint16_t)(h & 0xFFFFu));
}

// A launch with programmatic dependent launch; every kernel of this file's
// users begins with griddepcontrol.wait.
template <typename... KArgs, typename... Args>
static cudaError_t kv8_launch(void (*k)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, int cluster,
                              Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = 1;
    at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, k, ((KArgs)args)...);
    if (e == cudaSuccess) vxc_count_launches(1);
    return e;
}

// Lets `kernel` be launched with `bytes` of dynamic shared memory on the current device.
cudaError_t kv8_allow_smem(const void *kernel, size_t bytes);
// Whether an address can be that of ints or floats (a misaligned one would fault on the device).
template <typename... P>
static inline bool kv8_words(const P *...p) { return ((((uintptr_t)p % 4) == 0) && ...); }
// 0, or -4 with the error set: the fields of a cache (host side).
int vxc_kv8_check(const vxc_kv8 *kv, const char *who);
