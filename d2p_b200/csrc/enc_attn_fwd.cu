// enc_attn_fwd.cu -- attention forward on the fifth-generation tensor cores.
//
// One CTA takes 128 query rows of a head and runs over the keys in tiles of
// 128.  S = Q K^T (tcgen05, both operands in shared memory, K-major) lands in
// 128 TMEM columns; a warpgroup reads it, one row a thread, adds the bias, and
// takes the softmax in base 2 with a running reference m: p = 2^(s - m), l =
// sum p.  P goes back to TMEM in 16 bits and is operand A
// of O += P V (V from shared memory, contraction down its rows).  m is raised,
// and O and l rescaled, only when a row's maximum passes it by more than
// kSlack (2^kSlack stays in range of the 16-bit types), which after the first
// tiles is rare.  In the last tile the rows of V past the keys are zeroed in
// shared memory, since 0 x NaN would reach the sums.
#include "enc_tc.cuh"

namespace d2pb {
namespace enc {

namespace fwd {

constexpr int kThreads = 160;   // a softmax warpgroup and the warp that copies and multiplies
constexpr int kRows = 128;
constexpr int kColumns = 256;   // TMEM: S / P 128, O up to 128; two CTAs a SM
constexpr int kChunk = kRows * 128;

template <int DP>
struct Shape {
    static constexpr int kChunks = DP / 64;
    static constexpr int kTile = kChunks * kChunk;
    // K and V tiles in flight: one of each for 128 elements (two CTAs an SM); kApart needs two, since it asks for V
    // tile j only after P j - 1
    static constexpr int kStages = DP == 64 ? 2 : 1;
    static constexpr int kBars = 5 + 2 * kStages;
    // P has TMEM columns of its own, so that the next S is formed while this one's exponentials are taken; for 128
    // elements there is no room and P overwrites S (that shape is bound by its products as it is)
    static constexpr bool kApart = DP == 64;
    static constexpr size_t smem(int lut) { return 1024 + (size_t)kTile * (1 + 2 * kStages) + kBars * 8 + 16 + (size_t)lut * 4; }
};

template <class T, int DP, bool BIAS>
__global__ void __launch_bounds__(kThreads, 2)
    attn_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                    const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmO,
                    const __grid_constant__ AttnArgs a, T* __restrict__ out, float* __restrict__ lse) {
    using Sh = Shape<DP>;
    constexpr int NST = Sh::kStages;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // causal: the rows with the most keys first
    const int q0 = (a.causal ? gridDim.x - 1 - blockIdx.x : blockIdx.x) * kRows, h = blockIdx.y, b = blockIdx.z;
    int lq, lk;
    problem_lengths(a, b, &lq, &lk);
    const int off = a.causal ? lk - lq : 0;
    const int last = min(q0 + kRows, lq) - 1;   // the tile's last live row
    const int keys = q0 < lq ? (a.causal ? min(lk, last + off + 1) : lk) : 0;
    const int tiles = keys > 0 ? (keys + kRows - 1) / kRows : 0;
    if (tiles == 0) {   // no row of the tile has a key
        const int rows = min(kRows, a.Lq - q0), units = a.D / 8;
        for (int e = tid; e < rows * units; e += kThreads) {
            const size_t at = (((size_t)b * a.Lq + q0 + e / units) * a.H + h) * a.D + (e % units) * 8;
            *reinterpret_cast<uint4*>(out + at) = make_uint4(0, 0, 0, 0);
        }
        if (lse)
            for (int e = tid; e < rows; e += kThreads) lse[((size_t)b * a.H + h) * a.Lq + q0 + e] = INFINITY;
        return;
    }

    extern __shared__ uint8_t raw[];
    const uint32_t r0 = smem_addr(raw), base = (r0 + 1023u) & ~1023u;
    uint8_t* const gbase = raw + (base - r0);
    const uint32_t sQ = base, sK = base + Sh::kTile, sV = sK + NST * Sh::kTile;
    uint64_t* const bars = reinterpret_cast<uint64_t*>(gbase + (size_t)Sh::kTile * (1 + 2 * NST));
    const uint32_t barQ = smem_addr(bars), barS = barQ + 8, barP = barQ + 16, barO = barQ + 24, barR = barQ + 32,
                   barK = barQ + 40, barV = barK + 8 * NST;
    volatile int* const dead = reinterpret_cast<volatile int*>(bars + Sh::kBars);
    uint32_t* const slot = reinterpret_cast<uint32_t*>(bars + Sh::kBars) + 1;
    float* const lut = reinterpret_cast<float*>(bars + Sh::kBars + 2);
    const int reach = BIAS ? reach_of(a.edges) : 0;

    const int kh = h / (a.H / a.Hkv);
    auto load = [&](uint32_t dst, const CUtensorMap* tm, int row, int head, uint32_t bar) {
        bar_expect(bar, Sh::kTile);
#pragma unroll
        for (int c = 0; c < Sh::kChunks; ++c) tma_load(dst + c * kChunk, tm, 64 * c, row, head, b, bar);
    };
    auto load_k = [&](int j) { load(sK + (j % NST) * Sh::kTile, &tmK, j * kRows, kh, barK + 8 * (j % NST)); };
    auto load_v = [&](int j) { load(sV + (j % NST) * Sh::kTile, &tmV, j * kRows, kh, barV + 8 * (j % NST)); };
    if (warp == 4) {   // barriers, and the first copies before the CTA meets
        if (lane == 0) {
            bar_init(barQ, 1), bar_init(barS, 1), bar_init(barP, 4), bar_init(barO, 1), bar_init(barR, 4);
            for (int s = 0; s < NST; ++s) bar_init(barK + 8 * s, 1), bar_init(barV + 8 * s, 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            fence_async_smem();
            *dead = 0;
            load(sQ, &tmQ, q0, h, barQ);
            for (int j = 0; j < NST && j < tiles; ++j) load_k(j), load_v(j);
        }
        __syncwarp();
        tmem_alloc(smem_addr(slot), kColumns);
    } else if (BIAS) {
        fill_lut<T>(lut, a, h, reach, warp, 4);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *slot, tO = tmem + 128, tP = tmem + (Sh::kApart ? 192 : 0);

    if (warp == 4) {
        // the whole warp runs this, so that the operands' words stay in uniform registers; one lane issues
        const bool lead = elect_one();
        const int nu = __shfl_sync(0xffffffffu, tiles, 0);
        const uint32_t uS = __shfl_sync(0xffffffffu, tmem, 0), uO = uS + 128, uP = uS + (Sh::kApart ? 192 : 0);
        constexpr uint32_t idS = mma_desc<T>(128, 128, false), idO = mma_desc<T>(128, DP, true);
        auto scores = [&](int j) {
            const int s = j % NST;
            if (!bar_wait_warp(barK + 8 * s, (j / NST) & 1, dead)) return false;
            tc_fence_after();
            const uint32_t dQ = desc_along(sQ), dK = desc_along(sK + s * Sh::kTile);
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) {
                const uint32_t o = ((k / 4) * kChunk + (k % 4) * 32) / 16;
                if (lead) mma_ss(uS, dQ + o, dK + o, idS, k != 0);
            }
            if (lead) tc_commit(barS);
            return true;
        };
        bool ok = bar_wait_warp(barQ, 0, dead) && scores(0);
        int j = 0;
        for (; ok && j < nu; ++j) {
            const int s = j % NST;
            // S done, and read into registers where P has columns of its own: K's tile is free, and the next S can begin
            if (!(ok = bar_wait_warp(Sh::kApart ? barR : barS, j & 1, dead))) break;
            if (j + NST < nu && lead) load_k(j + NST);
            // (S j was issued after the product before: that one is over too, and its V tile free)
            if (!Sh::kApart && j > 0 && j - 1 + NST < nu && lead) load_v(j - 1 + NST);
            if (Sh::kApart && j + 1 < nu && !(ok = scores(j + 1))) break;
            if (!(ok = bar_wait_warp(barV + 8 * s, (j / NST) & 1, dead) && bar_wait_warp(barP, j & 1, dead))) break;
            // (P j was written after the product before was over: its V tile is free)
            if (Sh::kApart && j > 0 && j - 1 + NST < nu && lead) load_v(j - 1 + NST);
            tc_fence_after();
            const uint32_t dV = desc_down(sV + s * Sh::kTile, kChunk);
#pragma unroll
            for (int k = 0; k < kRows / 16; ++k)
                if (lead) mma_ts(uO, uP + 8 * k, dV + k * (2048 / 16), idO, (j | k) != 0);
            if (lead) tc_commit(barO);
            if (!Sh::kApart && j + 1 < nu) ok = scores(j + 1);
        }
        if (!ok) {   // a wait gave up: what is in flight ends (bounded) before the CTA does
            volatile int none = 0;
            for (int t = max(j - 1, 0); t < min(j + 1 + NST, nu); ++t) {
                bar_wait(barK + 8 * (t % NST), (t / NST) & 1, &none);
                bar_wait(barV + 8 * (t % NST), (t / NST) & 1, &none);
            }
            bar_wait(barQ, 0, &none);
            if (lead) atomicAdd(&g_gave_up, 1ull);
        }
        __syncwarp();
    } else {
        const int i = q0 + tid, pos = i + off;
        const uint32_t trow = (uint32_t)(32 * warp) << 16;
        const float c = a.scale * kLog2e;
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        for (int j = 0; j < tiles; ++j) {
            const int k0 = j * kRows;
            if (!(ok = bar_wait_warp(barS, j & 1, dead))) break;
            tc_fence_after();
            uint32_t v[128];
#pragma unroll
            for (int x = 0; x < 4; ++x) tmem_ld32(tmem + trow + 32 * x, v + 32 * x);
            tmem_wait_ld();
#pragma unroll
            for (int x = 0; x < 4; ++x) tmem_tie32(v + 32 * x);
            if (Sh::kApart) {
                tc_fence_before();
                bar_arrive_warp(barR);
            }
            float* const t = reinterpret_cast<float*>(v);
            if (BIAS) {   // scores in base 2; blocks of 32 x 32 that lie past the last edge take one value
                const float* const lp = lut + (k0 - pos + reach + kPad);
                const int dmin = k0 - (q0 + 32 * warp + 31 + off);
#pragma unroll
                for (int x = 0; x < 128; x += 32) {
                    if (dmin + x < reach && dmin + x + 62 > -reach) {
#pragma unroll
                        for (int y = x; y < x + 32; ++y) t[y] = fmaf(t[y], c, lp[y]);
                    } else {
                        const float far = dmin + x >= reach ? lut[lut_size(reach) - 1] : lut[0];
#pragma unroll
                        for (int y = x; y < x + 32; ++y) t[y] = fmaf(t[y], c, far);
                    }
                }
            }
            if (k0 + kRows > lk || (a.causal && k0 + kRows - 1 > q0 + off)) {
                const int lim = (a.causal ? min(lk - 1, pos) : lk - 1) - k0;
#pragma unroll
                for (int x = 0; x < 128; ++x) t[x] = x <= lim ? t[x] : -INFINITY;
            }
            float mx[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) mx[x] = t[x];
#pragma unroll
            for (int x = 4; x < 128; ++x) mx[x & 3] = fmaxf(mx[x & 3], t[x]);
            float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
            if (!BIAS) top *= c;
            float f = 1.f;
            const bool raise = top > m + Softmax<T>::kSlack || (m == -INFINITY && top > -INFINITY);
            if (raise) {
                f = m == -INFINITY ? 0.f : ex2(m - top);
                m = top;
                l *= f;
            }
            const bool rescale = __any_sync(0xffffffffu, raise) && j > 0;
            // the product before reads P's columns and adds to O
            if (j > 0 && (Sh::kApart || rescale)) {
                if (!(ok = bar_wait_warp(barO, (j - 1) & 1, dead))) break;
                tc_fence_after();
            }
            if (rescale) {   // O's rows of this warp
#pragma unroll 1
                for (int x = 0; x < DP; x += 32) {
                    uint32_t o[32];
                    tmem_ld32(tO + trow + x, o);
                    tmem_wait_ld();
                    tmem_tie32(o);
#pragma unroll
                    for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * f);
                    tmem_st32(tO + trow + x, o);
                }
                tmem_wait_st();
            }
            const float ref = (m == -INFINITY ? 0.f : m) - Softmax<T>::kShift;
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int x = 0; x < 128; x += 32) {
                uint32_t p[16];
#pragma unroll
                for (int y = 0; y < 32; y += 2) {
                    const float e0 = ex2(BIAS ? t[x + y] - ref : fmaf(t[x + y], c, -ref));
                    const float e1 = ex2(BIAS ? t[x + y + 1] - ref : fmaf(t[x + y + 1], c, -ref));
                    sum[y & 2] += e0;
                    sum[(y & 2) + 1] += e1;
                    p[y / 2] = pack2<T>(e0, e1);
                }
                tmem_st16(tP + trow + x / 2, p);
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            const int live = lk - k0;
            if (live < kRows) {   // the keys' last tile: rows of V past them to zero
                if (!(ok = bar_wait_warp(barV + 8 * (j % NST), (j / NST) & 1, dead))) break;
                for (int e = tid; e < (kRows - live) * 8 * Sh::kChunks; e += 128) {
                    const int ch = e / ((kRows - live) * 8), r = e % ((kRows - live) * 8);
                    *reinterpret_cast<uint4*>(gbase + (sV - base) + (j % NST) * Sh::kTile + ch * kChunk + live * 128 + r * 16) =
                        make_uint4(0, 0, 0, 0);
                }
                fence_async_smem();
            }
            tmem_wait_st();
            tc_fence_before();
            bar_arrive_warp(barP);
        }
        ok = ok && bar_wait_warp(barO, (tiles - 1) & 1, dead);
        tc_fence_after();
        const bool row = i < lq;
        const bool some = l > 0.f || l != l;
        const float w = !ok ? NAN : (row && some ? 1.f / l : 0.f);
        // O / l into Q's tile (its last use was the last S), swizzled as the copy out reads it
#pragma unroll 1
        for (int x = 0; x < DP; x += 32) {
            uint32_t o[32];
            tmem_ld32(tO + trow + x, o);
            tmem_wait_ld();
            tmem_tie32(o);
            uint8_t* const rp = gbase + (x / 64) * kChunk + tid * 128;
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                uint32_t p[4];
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                    const float u0 = __uint_as_float(o[8 * y + 2 * z]), u1 = __uint_as_float(o[8 * y + 2 * z + 1]);
                    p[z] = w == 0.f ? 0u : pack2<T>(u0 * w, u1 * w);   // a dead row is zero whatever it held
                }
                *reinterpret_cast<uint4*>(rp + ((((x % 64) / 8 + y) ^ (tid & 7)) << 4)) = make_uint4(p[0], p[1], p[2], p[3]);
            }
        }
        if (lse && i < a.Lq)
            lse[((size_t)b * a.H + h) * a.Lq + i] = row && some ? m - Softmax<T>::kShift + log2f(l) : INFINITY;
        fence_async_smem();
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (tid == 0) {
#pragma unroll
            for (int ch = 0; ch < Sh::kChunks; ++ch)
                if (64 * ch < a.D) tma_store(&tmO, 64 * ch, q0, h, b, sQ + ch * kChunk);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 4) tmem_free(tmem, kColumns);
}

template <class T, int DP, bool BIAS>
int launch(const AttnArgs& a, int dtype, void* out, float* lse, cudaStream_t st) {
    using Sh = Shape<DP>;
    static DeviceSetup setup;
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    int rc = device_setup(setup, dev, [] {
        return (int)cudaFuncSetAttribute(attn_fwd_kernel<T, DP, BIAS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)Sh::smem(lut_size(kMaxReach)));
    }, &sms);
    if (rc) return rc;
    CUtensorMap q, k, v, o;
    const long long os[3] = {(long long)a.Lq * a.H * a.D, (long long)a.H * a.D, a.D};
    if (!rows_map(&q, dtype, a.q, a.B, a.Lq, a.H, a.D, a.qs, kRows) || !rows_map(&o, dtype, out, a.B, a.Lq, a.H, a.D, os, kRows))
        return D2P_ERR_INVALID_ARGUMENT;
    if (a.Lk == 0) k = v = q;   // never read
    else if (!rows_map(&k, dtype, a.k, a.B, a.Lk, a.Hkv, a.D, a.ks, kRows) ||
             !rows_map(&v, dtype, a.v, a.B, a.Lk, a.Hkv, a.D, a.vs, kRows))
        return D2P_ERR_INVALID_ARGUMENT;
    const int lut = BIAS ? lut_size(reach_of(a.edges)) : 0;
    // at least a third of the SM's shared memory: no more than two CTAs (2 x 256 TMEM columns), so no allocation waits
    size_t smem = Sh::smem(lut);
    if (smem < 80 * 1024) smem = 80 * 1024;
    attn_fwd_kernel<T, DP, BIAS><<<dim3((a.Lq + kRows - 1) / kRows, a.H, a.B), kThreads, smem, st>>>(q, k, v, o, a, (T*)out, lse);
    return (int)cudaGetLastError();
}

template <class T>
int pick(const AttnArgs& a, int dtype, void* out, float* lse, cudaStream_t st) {
    if (a.D <= 64) return a.bias ? launch<T, 64, true>(a, dtype, out, lse, st) : launch<T, 64, false>(a, dtype, out, lse, st);
    return a.bias ? launch<T, 128, true>(a, dtype, out, lse, st) : launch<T, 128, false>(a, dtype, out, lse, st);
}

}  // namespace fwd

namespace {
PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
    }();
    return fn;
}
}  // namespace

bool rows_map(CUtensorMap* tm, int dtype, const void* base, int B, int L, int heads, int D, const long long* s, int rows) {
    auto fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)L, (cuuint64_t)heads, (cuuint64_t)B};
    const cuuint64_t strides[3] = {(cuuint64_t)s[1] * 2, (cuuint64_t)s[2] * 2, (cuuint64_t)s[0] * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1};
    const cuuint32_t es[4] = {1, 1, 1, 1};
    return fn(tm, dtype == D2P_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
              const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int attn_forward_gave_up(unsigned long long* n) { return (int)cudaMemcpyFromSymbol(n, g_gave_up, sizeof(*n)); }

int attn_forward_tiles(const AttnArgs& a, int dtype, void* out, float* lse, cudaStream_t st) {
    return dtype == D2P_DTYPE_BF16 ? fwd::pick<__nv_bfloat16>(a, dtype, out, lse, st) : fwd::pick<__half>(a, dtype, out, lse, st);
}

}  // namespace enc
}  // namespace d2pb
