// enc_dropout.cu -- y = residual + x keep / (1 - p), keep from a counter-based
// generator and never stored: the backward pass draws it again from the same
// seed and offset.
//
// Generator: Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", SC 2011).  Element e takes word e % 4 of the
// block with counter (e / 4, offset) and the seed as its key, and is kept where
// the word is at least floor(p 2^32).  A dropped element is selected away, not
// multiplied by zero, so infinities and NaN in dropped places do not reach y.
#include "enc_common.cuh"

namespace d2pb {
namespace enc {

__device__ __forceinline__ uint4 philox(uint64_t block, uint64_t seed, uint64_t offset) {
    uint32_t a = (uint32_t)block, b = (uint32_t)(block >> 32), x = (uint32_t)offset, y = (uint32_t)(offset >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t p = (uint64_t)a * 0xD2511F53u, q = (uint64_t)x * 0xCD9E8D57u;
        a = (uint32_t)(q >> 32) ^ b ^ k0;
        b = (uint32_t)q;
        x = (uint32_t)(p >> 32) ^ y ^ k1;
        y = (uint32_t)p;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(a, b, x, y);
}

// eight elements a thread and step; RES: add the residual
template <class T, bool RES>
__global__ void __launch_bounds__(256) dropout_kernel(const T* __restrict__ x, const T* __restrict__ res,
                                                      T* __restrict__ y, size_t n, uint32_t thr, float scale,
                                                      uint64_t seed, uint64_t offset, int vec) {
    const size_t step = (size_t)gridDim.x * blockDim.x * 8;
    for (size_t e = ((size_t)blockIdx.x * blockDim.x + threadIdx.x) * 8; e < n; e += step) {
        float v[8], r[8];
        const bool whole = vec && e + 8 <= n;
        if (whole) {
            load8<T>(x + e, v);
            if (RES) load8<T>(res + e, r);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[i] = e + i < n ? to_f<T>(x[e + i]) : 0.f;
                if (RES) r[i] = e + i < n ? to_f<T>(res[e + i]) : 0.f;
            }
        }
        const uint4 w0 = philox(e / 4, seed, offset), w1 = philox(e / 4 + 1, seed, offset);
        const uint32_t w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float d = w[i] >= thr ? v[i] * scale : 0.f;
            v[i] = RES ? r[i] + d : d;
        }
        if (whole) {
            store8<T>(y + e, v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (e + i < n) y[e + i] = from_f<T>(v[i]);
        }
    }
}

template <class T>
int launch_dropout(const void* x, const void* res, void* y, size_t n, uint32_t thr, float scale, uint64_t seed,
                   uint64_t offset, int sms, cudaStream_t st) {
    const int vec = ((((uintptr_t)x | (uintptr_t)res | (uintptr_t)y) & 15) == 0);
    const size_t want = (n + 8 * 256 - 1) / (8 * 256);
    const unsigned blocks = (unsigned)(want < (size_t)sms * 32 ? want : (size_t)sms * 32);
    if (res)
        dropout_kernel<T, true><<<blocks, 256, 0, st>>>((const T*)x, (const T*)res, (T*)y, n, thr, scale, seed, offset, vec);
    else
        dropout_kernel<T, false><<<blocks, 256, 0, st>>>((const T*)x, nullptr, (T*)y, n, thr, scale, seed, offset, vec);
    return (int)cudaGetLastError();
}

}  // namespace enc
}  // namespace d2pb

using namespace d2pb;

extern "C" int d2p_dropout_add(const void* x, const void* residual, int dtype, unsigned long long n, double p,
                               unsigned long long seed, unsigned long long offset, void* y, void* stream) {
    if (!(p >= 0.0 && p < 1.0)) return D2P_ERR_INVALID_ARGUMENT;
    if (n == 0) return D2P_OK;
    if (!x || !y) return D2P_ERR_INVALID_ARGUMENT;
    static DeviceSetup setup;
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    int rc = device_setup(setup, dev, [] { return 0; }, &sms);
    if (rc) return rc;
    const uint32_t thr = (uint32_t)(uint64_t)(p * 4294967296.0);
    const float scale = (float)(1.0 / (1.0 - p));
    cudaStream_t st = (cudaStream_t)stream;
    switch (dtype) {
        case D2P_DTYPE_F32: return enc::launch_dropout<float>(x, residual, y, n, thr, scale, seed, offset, sms, st);
        case D2P_DTYPE_BF16:
            return enc::launch_dropout<__nv_bfloat16>(x, residual, y, n, thr, scale, seed, offset, sms, st);
        case D2P_DTYPE_F16: return enc::launch_dropout<__half>(x, residual, y, n, thr, scale, seed, offset, sms, st);
        default: return D2P_ERR_INVALID_ARGUMENT;
    }
}
