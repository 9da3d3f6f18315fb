// enc_attn_token.cu -- attention of a few query rows over a long cache: single
// tokens when serving.
//
// The query rows of one key head (queries x the heads that share it, at most 16)
// are one 16-row operand of the warp-level matrix instructions, so that each key
// and value is read once for all of them: the cache's bytes are what bounds
// this, and 16 rows are too few to gain from the larger tensor-core tiles.  The
// keys are split over the CTAs of a cluster and over a CTA's warps; a warp takes
// 16 keys at a time through its own ring of shared memory (cp.async, so no
// barrier in the loop) with a running maximum and sum, and the partial results
// join in shared memory, then through the cluster's (one launch, no workspace) or,
// where there are more splits than a cluster holds, by a second launch; always in
// a fixed order.
//
// P in 16 bits is the operand, as in the tiles' kernel.
//
// Measured: one token, 32 x 16 heads of 64, 4096 keys each: 86 us, 6.2 TB/s of keys
// and values (0.95 of a copy's rate); 8 x 8 key heads of 128, 8192 keys: 48 us, 5.6
// TB/s; with 32 buckets of bias 98 us, and 74 us over ragged caches of up to 4096
// (4.1 TB/s: the last CTAs' share).  One short cache (513 keys): 6 us, with the bias
// 12, latency.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "enc_attn.cuh"

namespace d2pb {
namespace enc {
namespace tok {

namespace cg = cooperative_groups;

constexpr int kWarps = 4, kKeys = 16, kRowsM = 16;
constexpr int kMaxSplits = 16;  // CTAs of a cluster: past 8 is allowed on this device on request
constexpr int kMinRounds = 2;   // of a CTA's warps: the least keys worth a CTA of their own

template <int DP>
struct Shape {
    static constexpr int kStages = 3;
    static constexpr int kResident = DP == 64 ? 4 : 2;            // CTAs an SM holds
    static constexpr int kTile = kKeys * DP * 2;                  // bytes of a warp's keys (or values)
    static constexpr int kRing = kWarps * kStages * 2 * kTile;    // 48 KB / 96 KB
    // in the ring's place: the warps' partial results, the CTA's, and the weights of the cluster's
    static constexpr int kPitch = DP + 4;
    static constexpr int kJoin = 4 * ((kWarps + 1) * kRowsM * (kPitch + 2) + kRowsM * kMaxSplits);
};

template <class T>
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool TRANS>
__device__ __forceinline__ void ldmatrix4(uint32_t* r, uint32_t addr) {
    if (TRANS)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// one side's bucket of each position by search: only the few blocks near the queries come here
__device__ __forceinline__ int bucket_of(const Edges& e, int d) {
    const int n = e.two ? abs(d) : max(-d, 0);
    int lo = 0, hi = e.n;         // the number of edges <= n
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (e.e[mid] <= n) lo = mid + 1;
        else hi = mid;
    }
    return lo + ((e.two && d > 0) ? e.n + 1 : 0);
}

template <class T, int DP, bool BIAS, bool REST>
__global__ void __launch_bounds__(32 * kWarps) attn_token_kernel(const __grid_constant__ AttnArgs a, T* __restrict__ out,
                                                                float* __restrict__ lse, T* __restrict__ rest, const __grid_constant__ Parts part) {
    using Sh = Shape<DP>;
    constexpr int NST = Sh::kStages, CH = DP / 8;   // 16-byte units of a row
    extern __shared__ __align__(128) uint8_t sm[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int split = blockIdx.x, splits = gridDim.x, kh = blockIdx.y, b = blockIdx.z;
    const int G = a.H / a.Hkv, rows = a.Lq * G;
    // an entry of these heads' bias a thread, asked for ahead of all else: whether any is large, and rows have bases (every
    // row's own maximum in its place: a short cache 2 us longer)
    float entry = 0.f;
    if (BIAS && tid < G * n_buckets(a.edges)) entry = bias_log2<T>(a, tid / G, kh * G + tid % G);
    int lq, lk;
    problem_lengths(a, b, &lq, &lk);
    const int off = a.causal ? lk - lq : 0;
    // keys any row meets, and this CTA's share in whole rounds of its warps
    const int most = lq > 0 ? (a.causal ? min(lk, lq + off) : lk) : 0;
    const int round = kWarps * kKeys;
    const int share = max(((most + splits - 1) / splits + round - 1) / round, kMinRounds) * round;
    const int k0 = min(most, split * share), k1 = min(most, k0 + share);

    // rows g and g + 8 of the operand: query i = row / G, head kh G + row % G
    int qi[2], head[2], lim[2];
    bool live[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const int r = g + 8 * w;
        qi[w] = r / G, head[w] = kh * G + r % G;
        live[w] = r < rows && qi[w] < lq;
        lim[w] = live[w] ? (a.causal ? min(lk, qi[w] + off + 1) : lk) : 0;   // keys of the row: [0, lim)
    }
    uint32_t qa[DP / 16][4];
#pragma unroll
    for (int k = 0; k < DP / 16; ++k)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int w = x & 1, d = 16 * k + 2 * t + 8 * (x >> 1);
            qa[k][x] = 0;
            if (live[w] && d < a.D)
                qa[k][x] = *reinterpret_cast<const uint32_t*>((const T*)a.q + b * a.qs[0] + qi[w] * a.qs[1] + head[w] * a.qs[2] + d);
        }
    const int reach = a.edges.n ? a.edges.e[a.edges.n - 1] : 1;
    float before[2] = {0.f, 0.f}, after[2] = {0.f, 0.f};   // the bias past the last edge, on either side
    if (BIAS) {
#pragma unroll
        for (int w = 0; w < 2; ++w)
            if (live[w]) {
                before[w] = bias_log2<T>(a, a.edges.n, head[w]);
                if (a.edges.two) after[w] = bias_log2<T>(a, 2 * a.edges.n + 1, head[w]);
            }
    }

    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(sm) + warp * NST * 2 * Sh::kTile;
    const int first = k0 + warp * kKeys, n = first < k1 ? (k1 - first + round - 1) / round : 0;
    // a lane copies unit fc of rows fr, fr + kStep, ..; zeros past k1 and past the head's size
    constexpr int kStep = 32 / CH;
    const int fr = lane / CH, fc = lane % CH;
    const bool fin = 8 * fc < a.D;
    const T* kp = (const T*)a.k + b * a.ks[0] + kh * a.ks[2] + (long long)(first + fr) * a.ks[1] + 8 * fc;
    const T* vp = (const T*)a.v + b * a.vs[0] + kh * a.vs[2] + (long long)(first + fr) * a.vs[1] + 8 * fc;
    int fat = first + fr;
    auto fetch = [&](int stage) {
        const uint32_t dst = ring + stage * 2 * Sh::kTile + fr * (DP * 2);
#pragma unroll
        for (int i = 0; i < kKeys / kStep; ++i) {
            const bool in = fin && fat + i * kStep < k1;
            const uint32_t d = dst + i * kStep * (DP * 2) + ((fc ^ ((fr + i * kStep) & 7)) << 4);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(in ? kp + i * kStep * a.ks[1] : (const T*)a.k), "r"(in ? 16 : 0) : "memory");
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d + Sh::kTile), "l"(in ? vp + i * kStep * a.vs[1] : (const T*)a.v), "r"(in ? 16 : 0) : "memory");
        }
        kp += round * a.ks[1], vp += round * a.vs[1], fat += round;
    };
#pragma unroll
    for (int s = 0; s < NST - 1; ++s) {
        if (s < n) fetch(s);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }

    const float c2 = a.scale * kLog2e;
    float rb[2] = {0.f, 0.f}, rc[2] = {c2, c2};   // the rows' bases, what multiplies their scores
    if (BIAS) {
        bool large = large_bias(entry);
        for (int x = tid + 32 * kWarps; x < G * n_buckets(a.edges); x += 32 * kWarps) large |= large_bias(bias_log2<T>(a, x / G, kh * G + x % G));
        if (__builtin_expect(__syncthreads_or(large), 0)) {
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                if (live[w]) rb[w] = base_of(row_top<T>(a, head[w], qi[w] + off, lim[w]));
                rc[w] = score_factor(rb[w], c2);
                before[w] -= rb[w], after[w] -= rb[w];
            }
        }
    }

    float o[DP / 8][4];
#pragma unroll
    for (int x = 0; x < DP / 8; ++x) o[x][0] = o[x][1] = o[x][2] = o[x][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    for (int it = 0; it < n; ++it) {
        asm volatile("cp.async.wait_group %0;" ::"n"(NST - 2) : "memory");
        __syncwarp();
        if (it + NST - 1 < n) fetch((it + NST - 1) % NST);
        asm volatile("cp.async.commit_group;" ::: "memory");
        const uint32_t ks = ring + (it % NST) * 2 * Sh::kTile, vs = ks + Sh::kTile;
        const int at = first + it * round;
        float s[kKeys / 8][4] = {};
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)   // matrices: keys 0-7 / 8-15 (lane >> 4) by elements 0-7 / 8-15 (lane >> 3 & 1)
#pragma unroll
            for (int y = 0; y < kKeys / 16; ++y) {
                const int r = 16 * y + (lane & 7) + ((lane >> 4) << 3), c = 2 * k + ((lane >> 3) & 1);
                uint32_t f[4];
                ldmatrix4<false>(f, ks + r * (DP * 2) + ((c ^ (r & 7)) << 4));
                mma16816<T>(s[2 * y], qa[k], f[0], f[1]);
                mma16816<T>(s[2 * y + 1], qa[k], f[2], f[3]);
            }
        // element (w, j): row g + 8 w, key at + 8 (j >> 1) + 2 t + (j & 1)
        float p[2][kKeys / 4];
        bool raised = false;
        float f[2];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const int pos = qi[w] + off;
            float top = -INFINITY;
            // past the last edge on one side the bias is one value
            const bool one = !BIAS || at + kKeys - 1 - pos <= -reach || (a.edges.two && at - pos >= reach);
            const float flat = !BIAS ? 0.f : at + kKeys - 1 - pos <= -reach ? before[w] : after[w];
#pragma unroll
            for (int j = 0; j < kKeys / 4; ++j) {
                const int key = at + 8 * (j >> 1) + 2 * t + (j & 1);
                float v = s[j >> 1][2 * w + (j & 1)] * rc[w];
                if (one) v += flat;
                else if (live[w]) v += bias_log2<T>(a, bucket_of(a.edges, key - pos), head[w]) - rb[w];
                p[w][j] = key < lim[w] ? v : -INFINITY;
                top = fmaxf(top, p[w][j]);
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const bool raise = top > m[w] + Softmax<T>::kSlack || (m[w] == -INFINITY && top > -INFINITY);
            f[w] = raise ? (m[w] == -INFINITY ? 0.f : exp2_fast(m[w] - top)) : 1.f;
            m[w] = raise ? top : m[w];
            raised |= raise;
            const float ref = (m[w] == -INFINITY ? 0.f : m[w]) - Softmax<T>::kShift;
            l[w] *= f[w];
#pragma unroll
            for (int j = 0; j < kKeys / 4; ++j) {
                p[w][j] = exp2_fast(p[w][j] - ref);
                l[w] += p[w][j];
            }
        }
        if (__any_sync(0xffffffffu, raised)) {
#pragma unroll
            for (int x = 0; x < DP / 8; ++x) o[x][0] *= f[0], o[x][1] *= f[0], o[x][2] *= f[1], o[x][3] *= f[1];
        }
#pragma unroll
        for (int y = 0; y < kKeys / 16; ++y) {
            const uint32_t pa[4] = {pack2<T>(p[0][4 * y], p[0][4 * y + 1]), pack2<T>(p[1][4 * y], p[1][4 * y + 1]),
                                    pack2<T>(p[0][4 * y + 2], p[0][4 * y + 3]), pack2<T>(p[1][4 * y + 2], p[1][4 * y + 3])};
            uint32_t pl[4];   // what rounding took from them, where out's rest is wanted
            if (REST)
#pragma unroll
                for (int x = 0; x < 4; ++x) pl[x] = rest2<T>(p[x & 1][4 * y + 2 * (x >> 1)], p[x & 1][4 * y + 2 * (x >> 1) + 1], pa[x]);
#pragma unroll
            for (int x = 0; x < DP / 16; ++x) {   // matrices: keys 0-7 / 8-15 (lane >> 3 & 1) by elements 0-7 / 8-15 (lane >> 4)
                const int r = 16 * y + (lane & 7) + (((lane >> 3) & 1) << 3), c = 2 * x + (lane >> 4);
                uint32_t e[4];
                ldmatrix4<true>(e, vs + r * (DP * 2) + ((c ^ (r & 7)) << 4));
                mma16816<T>(o[2 * x], pa, e[0], e[1]);
                mma16816<T>(o[2 * x + 1], pa, e[2], e[3]);
                if (REST) mma16816<T>(o[2 * x], pl, e[0], e[1]), mma16816<T>(o[2 * x + 1], pl, e[2], e[3]);
            }
        }
        __syncwarp();
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        l[w] += __shfl_xor_sync(0xffffffffu, l[w], 1);
        l[w] += __shfl_xor_sync(0xffffffffu, l[w], 2);
    }

    // join in the ring's place: o [set][16][pitch], m and l [set][16]; sets 0 .. kWarps - 1 the warps', set kWarps the CTA's
    constexpr int kPitch = Sh::kPitch;
    float* const jo = reinterpret_cast<float*>(sm);
    float* const jm = jo + (kWarps + 1) * kRowsM * kPitch;
    float* const jl = jm + (kWarps + 1) * kRowsM;
    float* const jw = jl + (kWarps + 1) * kRowsM;   // [16][kMaxSplits] weights of the cluster's sets
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const int r = warp * kRowsM + g + 8 * w;
        if (g + 8 * w < rows) {
#pragma unroll
            for (int x = 0; x < DP / 8; ++x)
                *reinterpret_cast<float2*>(jo + r * kPitch + 8 * x + 2 * t) = make_float2(o[x][2 * w], o[x][2 * w + 1]);
            if (t == 0) jm[r] = m[w], jl[r] = l[w];
        }
    }
    __syncthreads();
    const int units = a.D / 2;
    auto finish = [&](int r, int d, float x, float y, float top, float sum) {
        const int i = r / G, h = kh * G + r % G;
        const bool some = (sum > 0.f || sum != sum) && i < lq;
        const float w = some ? 1.f / sum : 0.f;
        const size_t at = (((size_t)b * a.Lq + i) * a.H + h) * a.D + d;
        const uint32_t p = some ? pack2<T>(x * w, y * w) : 0u;
        *reinterpret_cast<uint32_t*>(out + at) = p;
        if (REST) *reinterpret_cast<uint32_t*>(rest + at) = some ? rest2<T>(x * w, y * w, p) : 0u;
        if (lse && d == 0) lse[((size_t)b * a.H + h) * a.Lq + i] = some ? top - Softmax<T>::kShift + log2f(sum) : INFINITY;
    };
    for (int e = tid; e < rows * units; e += 32 * kWarps) {
        const int r = e / units, d = 2 * (e % units);
        float top = jm[r], sum = 0.f, x = 0.f, y = 0.f;
#pragma unroll
        for (int p = 1; p < kWarps; ++p) top = fmaxf(top, jm[p * kRowsM + r]);
#pragma unroll
        for (int p = 0; p < kWarps; ++p) {
            const float pm = jm[p * kRowsM + r], f = pm == -INFINITY ? 0.f : exp2_fast(pm - top);
            const float2 v = *reinterpret_cast<const float2*>(jo + (p * kRowsM + r) * kPitch + d);
            sum = fmaf(f, jl[p * kRowsM + r], sum), x = fmaf(f, v.x, x), y = fmaf(f, v.y, y);
        }
        if (splits == 1) {
            finish(r, d, x, y, top, sum);
        } else if (part.o) {
            const int i = r / G;
            const size_t set = part.set(a, b, kh * G + r % G, split, i);
            *reinterpret_cast<float2*>(part.o + set * a.D + d) = make_float2(x, y);
            if (d == 0) part.ml[set] = make_float2(top, sum);
        } else {
            *reinterpret_cast<float2*>(jo + (kWarps * kRowsM + r) * kPitch + d) = make_float2(x, y);
            if (d == 0) jm[kWarps * kRowsM + r] = top, jl[kWarps * kRowsM + r] = sum;
        }
    }
    if (splits == 1 || part.o) return;
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    // every CTA finishes its part of the rows from all the cluster's sets: their weights first, then the sums
    for (int e = tid; e < rows * splits; e += 32 * kWarps)
        jw[(e / splits) * kMaxSplits + e % splits] = cluster.map_shared_rank(jm, e % splits)[kWarps * kRowsM + e / splits];
    __syncthreads();
    for (int e = split * 32 * kWarps + tid; e < rows * units; e += splits * 32 * kWarps) {
        const int r = e / units, d = 2 * (e % units), at = kWarps * kRowsM + r;
        float top = -INFINITY, sum = 0.f, x = 0.f, y = 0.f;
        for (int p = 0; p < splits; ++p) top = fmaxf(top, jw[r * kMaxSplits + p]);
#pragma unroll 8
        for (int p = 0; p < splits; ++p) {
            const float pm = jw[r * kMaxSplits + p], f = pm == -INFINITY ? 0.f : exp2_fast(pm - top);
            const float2 v = *reinterpret_cast<const float2*>(cluster.map_shared_rank(jo, p) + at * kPitch + d);
            sum = fmaf(f, cluster.map_shared_rank(jl, p)[at], sum), x = fmaf(f, v.x, x), y = fmaf(f, v.y, y);
        }
        finish(r, d, x, y, top, sum);
    }
    cluster.sync();   // the sets are read from other CTAs
}

int resident(const AttnArgs& a) { return a.D <= 64 ? Shape<64>::kResident : Shape<128>::kResident; }
// CTAs of a cluster that share a problem's keys: for every place there is, as far as the keys go round.  When this was chosen:
// 32 x 16 heads of 64, 4096 keys: 105 us with two CTAs a problem, 119 with one of larger steps; 8 x 8 heads of 128, 8192
// keys: 63 us with places for all, 84 with twice as many
int cluster_of(const AttnArgs& a, int sms) {
    int splits = 1;
    while (splits < kMaxSplits && (long long)a.B * a.Hkv * splits < (long long)resident(a) * sms && (long long)a.Lk > (long long)splits * kMinRounds * kWarps * kKeys)
        splits *= 2;
    return splits;
}
// more splits than a cluster holds, joined by a second launch: for long caches of few heads.  Clusters of 16 also find no
// place for all at once.  One token, us by a cluster / by parts: 2 x 8 heads of 128, 27248 keys 71 / 42; 1 x 4 of 128, 32768
// keys 38 / 18, 4096 keys 9.5 / 9.0; 11 x 2 of 64, 17687 keys 27.6 / 21.6; 1 x 2 of 64, 2900 keys 6.7 / 8.1
int parts_of(const AttnArgs& a, int sms) {
    if (a.Lk < 4096 || cluster_of(a, sms) < kMaxSplits) return 1;
    const long long places = (long long)resident(a) * sms / ((long long)a.B * a.Hkv), most = a.Lk / (kMinRounds * kWarps * kKeys);
    const long long n = std::min(std::min(places, most), (long long)kMaxParts);
    return n > kMaxSplits ? (int)n : 1;
}

template <class T, int DP, bool BIAS, bool REST>
int launch(const AttnArgs& a, void* out, float* lse, void* rest, void* ws, cudaStream_t st) {
    using Sh = Shape<DP>;
    constexpr int smem = Sh::kRing > Sh::kJoin ? Sh::kRing : Sh::kJoin;
    static DeviceSetup setup;
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    int rc = device_setup(setup, dev, [] {
        cudaError_t e = cudaFuncSetAttribute(attn_token_kernel<T, DP, BIAS, REST>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(attn_token_kernel<T, DP, BIAS, REST>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        return (int)e;
    }, &sms);
    if (rc) return rc;
    const Parts part = parts_at(a, parts_of(a, sms), parts_of(a, sms) > 1 ? ws : nullptr);
    const int splits = part.splits > 1 ? part.splits : cluster_of(a, sms);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(splits, a.Hkv, a.B), cfg.blockDim = dim3(32 * kWarps), cfg.dynamicSmemBytes = smem, cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = splits, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr, cfg.numAttrs = part.splits > 1 ? 0 : 1;
    e = cudaLaunchKernelEx(&cfg, attn_token_kernel<T, DP, BIAS, REST>, a, (T*)out, lse, (T*)rest, part);
    if (e != cudaSuccess || part.splits == 1) return (int)e;
    return attn_join(a, std::is_same<T, __half>::value ? D2P_DTYPE_F16 : D2P_DTYPE_BF16, part, out, lse, rest, st);
}

}  // namespace tok

template <class T, int DP>
static int pick_token(const AttnArgs& a, void* out, float* lse, void* rest, void* ws, cudaStream_t st) {
    if (a.bias) return rest ? tok::launch<T, DP, true, true>(a, out, lse, rest, ws, st) : tok::launch<T, DP, true, false>(a, out, lse, rest, ws, st);
    return rest ? tok::launch<T, DP, false, true>(a, out, lse, rest, ws, st) : tok::launch<T, DP, false, false>(a, out, lse, rest, ws, st);
}
template <class T>
static int pick_token(const AttnArgs& a, void* out, float* lse, void* rest, void* ws, cudaStream_t st) {
    return a.D <= 64 ? pick_token<T, 64>(a, out, lse, rest, ws, st) : pick_token<T, 128>(a, out, lse, rest, ws, st);
}
int attn_forward_tokens(const AttnArgs& a, int dtype, void* out, float* lse, void* rest, void* ws, cudaStream_t st) {
    return dtype == D2P_DTYPE_BF16 ? pick_token<__nv_bfloat16>(a, out, lse, rest, ws, st) : pick_token<__half>(a, out, lse, rest, ws, st);
}
size_t attn_tokens_bytes(const AttnArgs& a) {
    int sms = 0;
    if (attn_sms(&sms)) return (size_t)-1;
    return parts_bytes(a, tok::parts_of(a, sms));
}

}  // namespace enc
}  // namespace d2pb
