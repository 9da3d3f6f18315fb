// enc_dropout.cu -- y = residual + x keep / (1 - p), keep from a counter-based
// generator and never stored: the backward pass draws it again from the same
// seed and offset.
//
// Generator: Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", SC 2011).  Element e takes word e % 4 of the
// block with counter (e / 4, offset) and the seed as its key, and is kept where
// the word is at least floor(p 2^32).  A dropped element is selected away, not
// multiplied by zero, so infinities and NaN in dropped places do not reach y.
//
// Measured, 131072 x 256 bf16: with a residual 42 us (201 MB: 4.8 TB/s), without 39
// us (134 MB: 3.4 TB/s).  So not the bytes bound it but the generator's arithmetic:
// the integer pipe is 60 % busy, the multiplies' 54, and issue waits on both.
#include "enc_common.cuh"

namespace d2pb {
namespace enc {

// a M in two words.  The same product from 16-bit halves on the plain multiply and
// the logic pipes costs more (three of a block's products that way, when this was
// tried: 51 us against 46).
template <uint32_t M>
__device__ __forceinline__ uint2 wide(uint32_t a) {
    const uint64_t p = (uint64_t)a * M;
    return make_uint2((uint32_t)p, (uint32_t)(p >> 32));
}
constexpr uint32_t kM0 = 0xD2511F53u, kM1 = 0xCD9E8D57u, kW0 = 0x9E3779B9u, kW1 = 0xBB67AE85u;

// what every block of a call shares: the key, and the first rounds' products of the offset (the block's high word is
// zero below 2^34 elements, which leaves round 1's first word the same for all too)
struct Stream {
    uint32_t k0, k1, off1;      // key, offset's high word
    uint2 q0;                   // round 0: offset's low word by M1
    uint2 p1;                   // round 1: the word above by M0, where the block's high word is zero
};
// the block with counter (block, offset); p0 = block M0, which a caller steps by additions
__device__ __forceinline__ uint4 philox(uint64_t block, uint64_t p0, const Stream& s) {
    uint32_t k0 = s.k0, k1 = s.k1;
    uint32_t a = s.q0.y ^ (uint32_t)(block >> 32) ^ k0, b = s.q0.x;
    uint32_t x = (uint32_t)(p0 >> 32) ^ s.off1 ^ k1, y = (uint32_t)p0;
#pragma unroll
    for (int r = 1; r < 10; ++r) {
        k0 += kW0, k1 += kW1;
        uint2 p = s.p1;
        if (r > 1 || (block >> 32)) p = wide<kM0>(a);
        const uint2 q = wide<kM1>(x);
        a = q.y ^ b ^ k0, b = q.x;
        x = p.y ^ y ^ k1, y = p.x;
    }
    return make_uint4(a, b, x, y);
}

// eight elements a thread and step; RES: add the residual
template <class T, bool RES>
__global__ void __launch_bounds__(256) dropout_kernel(const T* __restrict__ x, const T* __restrict__ res,
                                                      T* __restrict__ y, size_t n, uint32_t thr, float scale,
                                                      const Stream s, int vec) {
    const size_t step = (size_t)gridDim.x * blockDim.x * 8;
    size_t e = ((size_t)blockIdx.x * blockDim.x + threadIdx.x) * 8;
    // M0 times the low word of the block's counter, stepped with it (exact while the high word is zero; past that, anew)
    uint64_t p0 = (uint64_t)(uint32_t)(e / 4) * kM0;
    for (; e < n; e += step) {
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
        const uint64_t block = e / 4;   // even, so that block + 1 has the same high word
        if (block >> 32) p0 = (uint64_t)(uint32_t)block * kM0;
        const uint4 w0 = philox(block, p0, s), w1 = philox(block + 1, p0 + kM0, s);
        p0 += (uint64_t)(step / 4) * kM0;
        const uint32_t w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float d = w[i] >= thr ? v[i] : 0.f;
            v[i] = RES ? fmaf(d, scale, r[i]) : d * scale;
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
    const uint64_t q0 = (uint64_t)(uint32_t)offset * kM1;
    const uint64_t p1 = (uint64_t)((uint32_t)(q0 >> 32) ^ (uint32_t)seed) * kM0;
    const Stream s = {(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)(offset >> 32), {(uint32_t)q0, (uint32_t)(q0 >> 32)},
                      {(uint32_t)p1, (uint32_t)(p1 >> 32)}};
    if (res)
        dropout_kernel<T, true><<<blocks, 256, 0, st>>>((const T*)x, (const T*)res, (T*)y, n, thr, scale, s, vec);
    else
        dropout_kernel<T, false><<<blocks, 256, 0, st>>>((const T*)x, nullptr, (T*)y, n, thr, scale, s, vec);
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
    if (((uintptr_t)x | (uintptr_t)residual | (uintptr_t)y) & (dtype == D2P_DTYPE_F32 ? 3 : 1)) return D2P_ERR_INVALID_ARGUMENT;
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
