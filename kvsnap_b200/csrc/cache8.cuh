// What the translation units of the 8-bit paged cache share: elements, scales, and the checks and
// device handling of their C entries.
//
// A block (page) of one side (keys or values) and KV head is block_size tokens
// of head_dim e4m3 codes with one scale s, a power of two: the smallest with
// amax <= 448 s. e4m3 is a floating format, so a power of two costs no
// precision, and it buys three things: a page whose scale grows by 2^k re-rounds
// only codes that fall among e4m3's subnormals; code * s is exact in bf16; and
// an amax that rounds to either side of a border gives the same values.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <mutex>
#include <set>
#include <utility>

#include "kvsnap_cuda.h"
#include "kvsnap_internal.h"

namespace {

using Cache = kvsnap_c8_cache;
using Batch = kvsnap_c8_batch;

// ---- elements ---------------------------------------------------------------------

struct Bf16 {
    static __device__ float2 wide(uint32_t v) {
        return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
    }
    static __device__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return reinterpret_cast<const uint32_t&>(v);
    }
    // The larger of a (not negative) and |b|, of each half.
    static __device__ uint32_t max_size(uint32_t a, uint32_t b) {
        uint32_t d;
        asm("max.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b & 0x7FFF7FFFu));
        return d;
    }
};

struct Fp16 {
    static __device__ float2 wide(uint32_t v) { return __half22float2(reinterpret_cast<const __half2&>(v)); }
    static __device__ uint32_t pack(float a, float b) {
        const __half2 v = __floats2half2_rn(a, b);
        return reinterpret_cast<const uint32_t&>(v);
    }
    static __device__ uint32_t max_size(uint32_t a, uint32_t b) {
        uint32_t d;
        asm("max.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b & 0x7FFF7FFFu));
        return d;
    }
};

constexpr int kGranule = 16;               // tokens that always lie in one page

// 16 bytes, or zeros, predicated: where a branch around a load joins, the load is waited for.
__device__ __forceinline__ uint4 fetch16(const char* at, bool there) {
    uint4 v;
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %5, 0;\nmov.u32 %0, 0;\nmov.u32 %1, 0;\nmov.u32 %2, 0;\nmov.u32 %3, 0;\n"
                 "@p ld.global.v4.u32 {%0,%1,%2,%3}, [%4];\n}"
                 : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w) : "l"(at), "r"(uint32_t(there)));
    return v;
}

__device__ __forceinline__ uint2 fetch8(const char* at, bool there) {
    uint2 v;
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %3, 0;\nmov.u32 %0, 0;\nmov.u32 %1, 0;\n"
                 "@p ld.global.v2.u32 {%0,%1}, [%2];\n}"
                 : "=&r"(v.x), "=&r"(v.y) : "l"(at), "r"(uint32_t(there)));
    return v;
}

// 8 consecutive 16-bit elements.
template <typename T>
__device__ __forceinline__ void widen8(const uint4& x, float (&v)[8]) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 p = T::wide(w[i]);
        v[2 * i] = p.x, v[2 * i + 1] = p.y;
    }
}

template <typename T>
__device__ __forceinline__ void load8(const char* at, float (&v)[8]) {
    widen8<T>(*reinterpret_cast<const uint4*>(at), v);
}

__device__ __forceinline__ float2 from_e4m3x2(uint32_t v) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(v), __NV_E4M3);
    return __half22float2(__half2(h));
}

// 8 codes, times `by`.
__device__ __forceinline__ void widen_codes(uint2 x, float by, float (&v)[8]) {
    const uint32_t w[4] = {x.x & 0xFFFFu, x.x >> 16, x.y & 0xFFFFu, x.y >> 16};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 p = from_e4m3x2(w[i]);
        v[2 * i] = p.x * by, v[2 * i + 1] = p.y * by;
    }
}

__device__ __forceinline__ void load_codes(const char* at, float by, float (&v)[8]) {
    widen_codes(*reinterpret_cast<const uint2*>(at), by, v);
}

// Nearest codes of v * by (ties to even); beyond +-448, infinities included, +-448.
__device__ __forceinline__ uint2 codes_of(const float (&v)[8], float by) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * i] * by, v[2 * i + 1] * by), __NV_SATFINITE, __NV_E4M3);
    return make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
}

__device__ __forceinline__ void store_codes(char* at, const float (&v)[8], float by) {
    *reinterpret_cast<uint2*>(at) = codes_of(v, by);
}

// ---- scales ------------------------------------------------------------------------

// The smallest 2^e >= 2^-126 with amax <= 448 * 2^e = 1.75 * 2^(e + 8), from amax's bits; 0 for 0.
__device__ __forceinline__ float needed_scale(float amax) {
    const uint32_t bits = __float_as_uint(amax);
    if (!bits) return 0.0f;
    const int e = int(bits >> 23) - 8 + ((bits & 0x7FFFFFu) > 0x600000u);     // biased
    return __uint_as_float(uint32_t(e < 1 ? 1 : e) << 23);
}

// 1 / s of a scale. A block of zeros (s = 0) takes any factor: its codes stand for 0 whatever they are.
__device__ __forceinline__ float inverse(float s) { return s > 0.0f ? 1.0f / s : 1.0f; }

__device__ __forceinline__ float finite_size(float x) {
    const float a = fabsf(x);
    return a <= 3.402823466e38f ? a : 0.0f;      // neither infinities nor NaN set a scale
}

__device__ __forceinline__ float max8(const float (&v)[8], float m) {
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, finite_size(v[i]));
    return m;
}

__device__ __forceinline__ float warp_max(float m) {
#pragma unroll
    for (int k = 16; k; k >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, k));
    return m;
}

struct Rows {                 // 16-bit rows [token][head][dim]
    const char* at;
    int64_t token, head;
};

__device__ __forceinline__ const int32_t* ints(int64_t p) { return reinterpret_cast<const int32_t*>(p); }

// ---- host side --------------------------------------------------------------------------

struct Fail {
    const char* what;
};

// A call's error is its own: it is not left behind as the thread's last one, which later launches would take for theirs.
void check(cudaError_t rc) {
    if (rc == cudaSuccess) return;
    cudaGetLastError();
    throw Fail{cudaGetErrorString(rc)};
}

void require(bool ok, const char* what) {
    if (!ok) throw Fail{what};
}

// Checks the arguments, then runs `body` with `device` current if `checks` says that there is
// something to do, and puts the caller's device back.
template <typename C, typename F>
int on_device(int device, C&& checks, F&& body) {
    int before = -1;
    int rc = -1;
    try {
        if (!checks()) return 0;
        check(cudaGetDevice(&before));
        if (device != before) check(cudaSetDevice(device));
        body();
        rc = 0;
    } catch (const Fail& f) {
        kvsnap_internal_set_error(f.what);
    } catch (...) {
        kvsnap_internal_set_error("the 8-bit cache's host side failed");
    }
    if (before >= 0 && device != before) cudaSetDevice(before);
    return rc;
}

// Raise a kernel's shared memory limit on the current device, once per kernel and device.
void allow_shared(const void* kernel, int bytes) {
    static std::mutex mu;
    static std::set<std::pair<const void*, int>> done;
    int device = 0;
    check(cudaGetDevice(&device));
    std::lock_guard<std::mutex> hold(mu);
    if (done.count({kernel, device})) return;
    check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done.insert({kernel, device});
}

// `after`: the kernel may start while the one before it in the stream ends (and waits for it itself).
template <typename K, typename... A>
void launch(K kernel, dim3 grid, int threads, size_t shared, cudaStream_t stream, bool after, const A&... args) {
    if (shared > 48 << 10) allow_shared(reinterpret_cast<const void*>(kernel), int(shared));
    cudaLaunchConfig_t config{};
    config.gridDim = grid, config.blockDim = dim3(unsigned(threads));
    config.dynamicSmemBytes = shared, config.stream = stream;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attribute, config.numAttrs = after ? 1 : 0;
    check(cudaLaunchKernelEx(&config, kernel, args...));
}

bool aligned(int64_t v) { return v % 16 == 0; }

void check_cache(const Cache* c) {
    require(c && c->codes && c->scales, "the 8-bit cache has no storage");
    require(c->head_dim == 64 || c->head_dim == 128, "head_dim must be 64 or 128");
    require(c->block_size > 0 && c->block_size % 16 == 0, "block_size must be a multiple of 16");
    require(c->kv_heads > 0 && c->blocks > 0, "the 8-bit cache is empty");
    require(aligned(c->codes) && aligned(c->side_pitch) && aligned(c->block_pitch) && aligned(c->token_pitch) &&
                aligned(c->head_pitch),
            "the 8-bit cache's codes must be 16-byte aligned");
}

void check_batch(const Batch* b, const Cache* c) {
    require(b && (!b->seqs || (b->start && b->lengths && (b->table || !b->width))), "the batch has no tables");
    require(b->seqs >= 0 && b->rows >= 0 && b->width >= 0 && b->max_query >= 0, "invalid batch");
    // the kernels count a sequence's tokens in 32 bits, some of them past its end
    require(int64_t(b->width) * c->block_size <= 1LL << 30, "the block table holds more than 2^30 tokens a sequence");
}

void check_rows(const void* at, int64_t token, int64_t head) {
    require(at && aligned(reinterpret_cast<intptr_t>(at)) && aligned(token) && aligned(head),
            "rows must be 16-byte aligned");
}

void check_type(int type) {
    require(type == KVSNAP_C8_BF16 || type == KVSNAP_C8_FP16, "the element type must be bf16 or fp16");
}

template <typename F>
void by_type(int type, int head_dim, F&& launch) {
    if (type == KVSNAP_C8_BF16) {
        if (head_dim == 64) launch(Bf16{}, std::integral_constant<int, 64>{});
        else launch(Bf16{}, std::integral_constant<int, 128>{});
    } else {
        if (head_dim == 64) launch(Fp16{}, std::integral_constant<int, 64>{});
        else launch(Fp16{}, std::integral_constant<int, 128>{});
    }
}

}  // namespace
