// dropout_add.hip -- dropout from a counter-based generator with the residual
// add behind it: y = residual + keep * x * 65536 / (65536 - border), and its
// gradient, which draws the same bits again instead of reading a stored mask.
//
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy
// as 1, 2, 3", 2011): ten rounds turn a 128-bit counter and a 64-bit key into
// four 32-bit words.  One counter serves eight elements with 16 bits each, so a
// thread with eight elements (16 or 32 bytes, whole vector loads) needs one call:
// twenty 32 x 32 -> 64 multiplications, which memory hides.
//
// Bound by memory: 98304 x 1024 bfloat16 with a residual 120 us (604 MB at 5.0
// TB/s), the gradient 68 us (403 MB at 5.9 TB/s); a large copy reaches 4.7.  6144 x
// 256 float32: 4.6 us each way, out of the caches.
#include <hip/hip_runtime.h>

#include "float_types.h"
#include "trx_internal.h"

namespace trx {
namespace {

struct Words {
    uint32_t w[4];
};

__device__ __forceinline__ Words philox(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1) {
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return {{c0, c1, c2, c3}};
}

constexpr int kThreads = 256;

template <typename T, bool RES>
__global__ void __launch_bounds__(kThreads)
    dropout_add_kernel(int64_t n, const T* __restrict__ x, const T* __restrict__ residual,
                       const int64_t* __restrict__ rng, int border, uint32_t site, float scale, T* __restrict__ y,
                       int64_t* __restrict__ rng_used) {
    const int64_t seed = rng[0], step = rng[1];
    if (rng_used && blockIdx.x == 0 && threadIdx.x == 0) {
        rng_used[0] = seed;
        rng_used[1] = step;
    }
    const int64_t groups = (n + 7) / 8, stride = (int64_t)gridDim.x * kThreads;
    for (int64_t g = (int64_t)blockIdx.x * kThreads + threadIdx.x; g < groups; g += stride) {
        const Words r = philox((uint32_t)g, (uint32_t)(g >> 32), (uint32_t)step, site, (uint32_t)seed,
                               (uint32_t)((uint64_t)seed >> 32));
        const int64_t e0 = 8 * g;
        const int here = n - e0 < 8 ? (int)(n - e0) : 8;
        Eight<T> a, b, o;
        if (here == 8) {
            a = load8(x + e0);
            if (RES) b = load8(residual + e0);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                a.e[e] = e < here ? x[e0 + e] : (T)0.0f;
                if (RES) b.e[e] = e < here ? residual[e0 + e] : (T)0.0f;
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t bits = (r.w[e / 2] >> (16 * (e & 1))) & 0xffffu;
            // a dropped element is a zero whatever x holds there
            float v = (int)bits >= border ? (float)a.e[e] * scale : 0.0f;
            if (RES) v = v + (float)b.e[e];
            o.e[e] = (T)v;
        }
        if (here == 8) {
            store8(y + e0, o);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < here) y[e0 + e] = o.e[e];
        }
    }
}

}  // namespace

hipError_t launch_dropout_add(int64_t n, int dtype, const void* x, const void* residual, const int64_t* rng, int border,
                              uint32_t site, void* y, int64_t* rng_used, hipStream_t stream) {
    const int64_t blocks = ((n + 7) / 8 + kThreads - 1) / kThreads;
    const dim3 grid((unsigned)(blocks < 8192 ? blocks : 8192));
    const float scale = (float)(65536.0 / (65536 - border));
    return by_dtype(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if (residual)
            hipLaunchKernelGGL((dropout_add_kernel<T, true>), grid, dim3(kThreads), 0, stream, n,
                               static_cast<const T*>(x), static_cast<const T*>(residual), rng, border, site, scale,
                               static_cast<T*>(y), rng_used);
        else
            hipLaunchKernelGGL((dropout_add_kernel<T, false>), grid, dim3(kThreads), 0, stream, n,
                               static_cast<const T*>(x), static_cast<const T*>(nullptr), rng, border, site, scale,
                               static_cast<T*>(y), rng_used);
        return hipGetLastError();
    });
}

}  // namespace trx
