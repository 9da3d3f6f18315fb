// enc_tc.cuh -- the pieces the attention kernels on the fifth-generation tensor
// cores share: bounded mbarrier waits, TMA tile copies, tcgen05 products with
// their descriptors, and TMEM loads and stores.
//
// Shared tiles are rows of 64 16-bit elements (128 bytes, 128-byte swizzle); a
// head of up to 128 elements is one or two such chunks.  Columns past the
// head's size and rows past the tensor are zero-filled by the copy.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>

#include "enc_attn.cuh"

namespace d2pb {
namespace enc {

static __device__ unsigned long long g_gave_up;   // CTAs one of whose waits gave up (rows whose results did not come are NaN)

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void bar_init(uint32_t bar, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// one arrival for a warp, after all its lanes (one for each lane would queue up on the barrier's word)
__device__ __forceinline__ void bar_arrive_warp(uint32_t bar) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) bar_arrive(bar);
}
// the CTA's flag that some wait gave up (then every other wait ends as well), and the polls before one does
struct Dead {
    volatile int* flag;
    int polls;
};
// waits for the phase of the given parity
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, const Dead& dead) {
    for (int it = 0; it < dead.polls; ++it) {
        uint32_t done;
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
            : "=r"(done)
            : "r"(bar), "r"(parity)
            : "memory");
        if (done) return true;
        if ((it & 255) == 255 && *dead.flag) return false;
    }
    *dead.flag = 1;
    return false;
}

// the same for a whole warp, one answer for its lanes
__device__ __forceinline__ bool bar_wait_warp(uint32_t bar, uint32_t parity, const Dead& dead) {
    return __all_sync(0xffffffffu, bar_wait(bar, parity, dead));
}

// a value that all lanes of the warp share, by a reduction, whose result lives in a uniform register
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __reduce_or_sync(0xffffffffu, v); }

// true in one lane of a converged warp
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n selp.u32 %0, 1, 0, q;\n}\n" : "=r"(p));
    return p != 0;
}

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* tm, int x, int row, int head, int b, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(dst),
        "l"((unsigned long long)tm), "r"(x), "r"(row), "r"(head), "r"(b), "r"(bar)
        : "memory");
}

__device__ __forceinline__ void tmem_alloc(uint32_t slot, int columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t tmem, int columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// after a wait that gave up, by the warp that issued products (its elected lane): those under way end (bounded) before TMEM is freed
__device__ __forceinline__ void tc_drain(uint32_t bar) {
    int none = 0;
    if (elect_one()) {
        tc_commit(bar);
        bar_wait(bar, 0, Dead{&none, kWaitLimit});
    }
    __syncwarp();
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Shared-memory operands, 128-byte rows and swizzle, 8-row groups 1024 bytes
// apart.  The low words differ by address only, so a step along a tile is one
// addition (in 16-byte units: addresses stay below 2^18); the high word is constant.
// along: the contraction runs along the rows.  down: it runs down the rows, and
// the next 64 elements of the other extent lie one chunk further.
constexpr uint32_t kDescHigh = (1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_along(uint32_t saddr) { return (saddr >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_down(uint32_t saddr, uint32_t chunk_bytes) { return (saddr >> 4) | ((chunk_bytes >> 4) << 16); }
// fp32 accumulator, both operands of type T; b_rows: operand B's contraction runs down its rows
template <class T>
__host__ __device__ constexpr uint32_t mma_desc(int m, int n, bool b_rows);
template <>
__host__ __device__ constexpr uint32_t mma_desc<__nv_bfloat16>(int m, int n, bool b_rows) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (b_rows ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
template <>
__host__ __device__ constexpr uint32_t mma_desc<__half>(int m, int n, bool b_rows) {
    return (1u << 4) | (b_rows ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// d (+)= A B: A from shared memory (ss) or TMEM (ts), B from shared memory, K = 16
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 x, y;\n setp.ne.b32 p, %4, 0;\n mov.b64 x, {%1, %5};\n mov.b64 y, {%2, %5};\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)acc), "n"(kDescHigh)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 y;\n setp.ne.b32 p, %4, 0;\n mov.b64 y, {%2, %5};\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)acc), "n"(kDescHigh)
        : "memory");
}

#define ENC_R8(v, o) "r"(v[o]), "r"(v[o + 1]), "r"(v[o + 2]), "r"(v[o + 3]), "r"(v[o + 4]), "r"(v[o + 5]), "r"(v[o + 6]), "r"(v[o + 7])
#define ENC_W8(v, o) "=r"(v[o]), "=r"(v[o + 1]), "=r"(v[o + 2]), "=r"(v[o + 3]), "=r"(v[o + 4]), "=r"(v[o + 5]), "=r"(v[o + 6]), "=r"(v[o + 7])
// 32 columns of this warp's 32 TMEM lanes, one lane a thread
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : ENC_W8(v, 0), ENC_W8(v, 8), ENC_W8(v, 16), ENC_W8(v, 24)
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : ENC_W8(v, 0), ENC_W8(v, 8)
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::ENC_R8(v, 0),
        ENC_R8(v, 8), ENC_R8(v, 16), ENC_R8(v, 24), "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15};" ::ENC_R8(v, 0),
        ENC_R8(v, 8), "r"(addr)
        : "memory");
}
// the values of a load are used after its wait, not before (no instruction of its own)
#define ENC_T8(v, o) "+r"(v[o]), "+r"(v[o + 1]), "+r"(v[o + 2]), "+r"(v[o + 3]), "+r"(v[o + 4]), "+r"(v[o + 5]), "+r"(v[o + 6]), "+r"(v[o + 7])
__device__ __forceinline__ void tmem_tie32(uint32_t* v) {
    asm volatile("" : ENC_T8(v, 0), ENC_T8(v, 8), ENC_T8(v, 16), ENC_T8(v, 24));
}
__device__ __forceinline__ void tmem_tie16(uint32_t* v) { asm volatile("" : ENC_T8(v, 0), ENC_T8(v, 8)); }
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// sixteen 16-bit elements, of which the first `n` (8 or 16) are stored; whole: at a 32-byte boundary, one store a sector
__device__ __forceinline__ void store16(void* to, const uint32_t* p, int n, bool whole) {
    if (whole) {
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), ENC_R8(p, 0) : "memory");
    } else {
        reinterpret_cast<uint4*>(to)[0] = make_uint4(p[0], p[1], p[2], p[3]);
        if (n > 8) reinterpret_cast<uint4*>(to)[1] = make_uint4(p[4], p[5], p[6], p[7]);
    }
}

// two fp32 operations in one instruction
struct Two {
    uint64_t v;
    __device__ __forceinline__ Two() {}
    __device__ __forceinline__ Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
    __device__ __forceinline__ void get(float* a, float* b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(*a), "=f"(*b) : "l"(v)); }
};
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
    Two d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return d;
}
__device__ __forceinline__ Two add2(Two a, Two b) {
    Two d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
    return d;
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
    Two d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
    return d;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The bias by relative position of one head, in shared memory: entry d + reach +
// kPad for d in [-(reach + kPad), reach + kPad], reach the largest edge, so that a
// 32 x 32 block that touches |d| < reach reads it without clamping.  Four copies,
// copy k shifted by k entries, give a thread the entries of four columns in one
// aligned load whatever its row (one load a column made the biased kernel half as
// slow again); copies are 8 words apart modulo the 32 banks, so that the rows of a
// load meet no bank twice.
constexpr int kPad = 64;
__host__ __device__ inline int reach_of(const Edges& e) { return e.n ? e.e[e.n - 1] : 1; }
__host__ __device__ inline int lut_entries(int reach) { return 2 * (reach + kPad) + 1; }
__host__ __device__ inline int lut_pitch(int reach) { return ((lut_entries(reach) + 3 - 8 + 31) & ~31) + 8; }   // of a copy
__host__ __device__ inline int lut_size(int reach) { return 4 * lut_pitch(reach); }
// the four entries from `at` on are at lut_row(..)[0 .. 3]
__device__ __forceinline__ const float* lut_row(const float* lut, int reach, int at) {
    return lut + (at & 3) * lut_pitch(reach) + (at & ~3);
}

// fills lut for head h by `warps` warps, a bucket each in turn: its value is
// fetched once, its positions are consecutive.  Returns whether any is large, so that rows have bases
template <class T>
__device__ __forceinline__ bool fill_lut(float* lut, const AttnArgs& a, int h, int reach, int warp, int warps) {
    const int lane = threadIdx.x & 31, nb = n_buckets(a.edges), far = reach + kPad;
    float mine[(kMaxEdges + 1) / 16];
#pragma unroll
    for (int i = 0; i < (kMaxEdges + 1) / 16; ++i) mine[i] = lane + 32 * i < nb ? bias_log2<T>(a, lane + 32 * i, h) : 0.f;
    bool large = false;
#pragma unroll
    for (int i = 0; i < (kMaxEdges + 1) / 16; ++i) large |= large_bias(mine[i]);
    for (int t = warp; t < nb; t += warps) {
        float v = mine[0];
#pragma unroll
        for (int i = 1; i < (kMaxEdges + 1) / 16; ++i) v = t >> 5 == i ? mine[i] : v;
        v = __shfl_sync(0xffffffffu, v, t & 31);
        const int2 r = bucket_range(a.edges, t, far);
        for (int d = r.x + lane; d <= r.y; d += 32)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (d + far >= k) lut[k * lut_pitch(reach) + d + far - k] = v;
    }
    return __any_sync(0xffffffffu, large);
}

// Launches that begin before the one ahead has ended (programmatic): what that one writes is read after the wait, which
// does nothing in an ordinary launch
__device__ __forceinline__ void wait_ahead() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
template <class... P, class... A>
int launch_early(bool early, void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid, cfg.blockDim = dim3(threads), cfg.dynamicSmemBytes = smem, cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr, cfg.numAttrs = early ? 1 : 0;
    return (int)cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

// Items in order of falling work, for CTAs that take several each: a stable
// counting sort by one CTA of 1024 threads, so that which CTA takes an item never
// changes from run to run.  bin(i): the item's work, at most kBins - 1
constexpr int kBins = 1024, kMaxOrder = 1 << 14;
template <class Bin>
__device__ __forceinline__ void order_items(int items, Bin bin, int* order) {
    __shared__ int first[kBins], warp_sum[32];
    const int t = threadIdx.x, lane = t & 31;
    first[t] = 0;
    __syncthreads();
    for (int i = t; i < items; i += 1024) atomicAdd(&first[kBins - 1 - bin(i)], 1);
    __syncthreads();
    const int n = first[t];
    int sum = n;   // inclusive scan over the bins
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
    }
    if (lane == 31) warp_sum[t >> 5] = sum;
    __syncthreads();
    for (int w = 0; w < (t >> 5); ++w) sum += warp_sum[w];
    first[t] = sum - n;
    __syncthreads();
    for (int base = 0; base < items; base += 1024) {
        const int i = base + t, k = i < items ? kBins - 1 - bin(i) : -1;
        const uint32_t same = __match_any_sync(0xffffffffu, k);
        const int rank = __popc(same & ((1u << lane) - 1));
        for (int w = 0; w < 32; ++w) {   // warps in turn
            if (t >> 5 == w) {
                const int at = k >= 0 ? first[k] : 0;
                __syncwarp();
                if (k >= 0) {
                    order[at + rank] = i;
                    if (rank == 0) first[k] = at + __popc(same);
                }
            }
            __syncthreads();
        }
    }
}
// the e-th item of CTA y of n: rows of n items, every other one backwards, so that shares of falling work come out even
__device__ __forceinline__ int item_index(int e, int y, int n) { return e * n + (e & 1 ? n - 1 - y : y); }
__device__ __forceinline__ int item_count(int items, int y, int n) {
    const int rows = items / n;
    return rows + (item_index(rows, y, n) < items);
}

// [B, L, heads, D] rows with element strides s (batch, position, head) as a 4-D
// tensor (D, position, head, batch) in boxes of 64 elements x rows
bool rows_map(CUtensorMap* tm, int dtype, const void* base, int B, int L, int heads, int D, const long long* s, int rows);

}  // namespace enc
}  // namespace d2pb
