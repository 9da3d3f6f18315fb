// enc_attn_bwd.cu -- attention's gradients on the fifth-generation tensor cores,
// the probabilities recomputed from the forward's lse:
//   P = 2^(s - lse),  dP = dO V^T,  dS = P (dP - delta),  delta = rowsum(dO O),
//   dV = P^T dO,  dK = scale dS^T Q,  dQ = scale dS K,  dbias = buckets' sums of dS.
//
// Two passes in one launch, a CTA taking 128 rows that it owns at a time, so that
// every sum stays in the CTA's accumulators and none is atomic: the key pass
// (DKV) owns 128 keys and streams 64 queries at a time of every head that shares
// them, the query pass owns 128 queries and streams 64 keys.  The queries pass's
// CTAs come after the keys pass's in the grid and so take the SMs that these leave
// free; neither reads what the other writes.  With X1, X2 the
// owned and Y1, Y2 the streamed rows (keys pass: K, V / Q, dO; query pass: Q, dO
// / K, V) both are
//   S = X1 Y1^T,  dP = X2 Y2^T  (two 64-column products into TMEM),
//   P, dS in 16 bits over S's and dP's own columns (TMEM operands A; each half
//   of the columns over its own, so that no warp writes what another still reads),
//   acc1 += P Y2 (keys pass: dV),  acc2 += dS Y1 (dK or dQ).
// S and dP have three buffers (two where the accumulators leave no third): two
// warpgroups work on even tiles (32 columns each), two on odd, and find the next
// S and dP ready.  A round from P to the next S takes ~1300 cycles of waits and
// latencies besides the products, so with two buffers the tensor cores wait.  The scores are formed
// twice (7 products a tile pair rather than 5); in exchange dQ needs no
// cross-CTA sums, whose order would change results from run to run.
//
// Setting up a CTA, its first copies and its last products cost 5 to 7 us, as much
// as 512 streamed rows: where there are many owned tiles a CTA stays and takes one
// after the other, in order of their work, and the next one's copies and scores
// begin while this one's results leave.
//
// In fp16 the operand dS is held 2^k times as large, k by problem and key head so that it fits: |dS| is at most 2 |dO| |V|
// (largest norms of a row), and 2^k of that lies in [2^14, 2^15).  As it is, a small gradient's dS lies
// among fp16's subnormals, whose spacing then shows in dQ and dK (dO around 2^-16: 7591 of 128000 entries of dQ past what
// the results' own rounding explains), and a large one's may pass 65504.
//
// The bias's gradient sums dS over many rows, and a row's dS sum to nothing: what
// delta is off by would show there whole where one bucket holds most of a row's
// weight (1 % of the sum with delta from the plain output).  For it the forward
// forms O from P in twice 16 bits and keeps what rounding O took.  Without a bias
// it keeps the latter alone: short rows' dQ and dK are off by a sixth less.
//
// P and dS in 16 bits are the tensor cores' operands, of the type of the rows they
// multiply: an entry is off by as much as one of those is; all sums are fp32.
//
// Measured: 2 x 4096 causal, 16/4 heads of 128: 463 us (statistics and order 26
// more), 740 TFLOP/s counted as the gradients' 5 products, 1040 as the 7 taken;
// 64 x 512, 8 heads of 64: 193 us and 18, in fp16 210 and 30.  No pipe is full: at 1 x 4096 the
// products' unit is busy 71 % of the time, its tensor pipe 53 (S and dP, 64 columns
// wide, take both operands from shared memory), the exponentials' 30.
//
// The query pass also sums dS by relative position.  Along a diagonal of a
// warp's 32 x 32 block the sum moves one lane per column (one shuffle each), the
// 63 sums are scanned within the buckets they belong to, and each lane takes its
// buckets' last entries, in a fixed order.  (Differences of one scan over all carry
// the rounding of the buckets before: one of no weight got 2^-20 rather than nothing.)
#include <limits.h>

#include <algorithm>
#include <type_traits>

#include "enc_tc.cuh"

namespace d2pb {
namespace enc {

namespace bwd {

constexpr int kWork = 512;              // four warpgroups: two for a tile, half of its columns each
constexpr int kThreads = kWork + 96;    // and the warps of the scores, of the sums' products and of the copies
constexpr int kOwn = 128, kStep = 64;
constexpr int kColumns = 512;   // TMEM: buffers of 64 columns of S and 64 of dP, then the accumulators
constexpr int kChunkX = kOwn * 128, kChunkY = kStep * 128;
constexpr int kBuckets = 2 * (kMaxEdges + 1);
constexpr int kMaxItems = 64;   // owned tiles a CTA takes at most
constexpr int kStartWords = (2 * (kMaxReach + kPad) + 1 + 31) / 32 + 2;   // a bit for each position that begins a bucket, read 64 at a time

template <int DP, bool DKV>
__host__ __device__ constexpr int buffers() { return DKV && DP == 128 ? 2 : 3; }
// barriers of the scores: a warpgroup pair waits for every other tile, and of each barrier it has to have seen the phase
// before, or the parity would not tell the two apart; with three buffers that takes one for each buffer and pair
__host__ __device__ constexpr int score_bars(int nb) { return nb == 2 ? 2 : 6; }

// 2^k and 2^-k for what dS is at most; nothing is scaled where that is zero or not finite
__device__ __forceinline__ float2 ds_scale(float grad_top, float v_top) {
    const float most = 2.f * grad_top * v_top;
    if (!(most > 0.f && most < INFINITY)) return make_float2(1.f, 1.f);
    const int k = min(max(14 - ilogbf(most), -100), 60);
    return make_float2(ldexpf(1.f, k), ldexpf(1.f, -k));
}

template <int DP, bool BIAS>
struct Shape {
    static constexpr int kChunks = DP / 64;
    static constexpr int kX = kChunks * kChunkX, kY = kChunks * kChunkY;
    static constexpr int kRowStats = 2 * kStep * 4;               // lse and delta of a streamed tile's queries
    static constexpr int kStage = 2 * kY + 1024;                  // keeps the tiles at 1024-byte boundaries
    static constexpr int kOwned = DP == 64 ? 2 : 1;                          // owned tiles in shared memory: the next one's copies early
    static constexpr int kStages = DP == 64 ? 6 : BIAS ? 3 : 4;              // (the bias by position takes up to 35 KB)
    static constexpr int kBars = 2 * kOwned + 4 + 2 * kStages + 12;
    static constexpr size_t kTiles = 2 * (size_t)kOwned * kX + (size_t)kStages * kStage;
    static constexpr size_t fixed() { return 1024 + kTiles + kBars * 8 + 32 + kMaxItems * 24; }
};
// after the tiles: the bias by position, then (query pass) the diagonals' stage of each warp and the buckets' ranges
__host__ __device__ inline size_t extra(bool bias, int reach) {
    return bias ? 4 * (size_t)(lut_size(reach) + 16 * 144 + 16 * kBuckets + 2 * kBuckets + kStartWords) : 0;
}
// at least 116 KB: one CTA an SM, since it takes the whole TMEM (no allocation waits)
template <int DP, bool BIAS>
size_t smem_bytes(int reach) {
    const size_t n = Shape<DP, BIAS>::fixed() + extra(BIAS, reach);
    return n < 116 * 1024 ? 116 * 1024 : n;
}

struct Args {
    AttnArgs a;
    const float* lse;      // [B, H, Lp] padded copies, negated: kShift - lse and -delta kDown; -inf and 0 in dead rows
    const float* delta;
    const float* base;     // of the rows, where there is a bias: 0 in dead rows
    int Lp;
    void *dv, *dk, *dq;
    float* part;           // query pass: [H][buckets][CTAs of a head] sums of dS, or null
    const float *grad_top, *v_top;  // fp16: [B][Hkv] largest norms of dO's (of the heads that share a key head) and V's rows
    const int *order_k, *order_q;   // the passes' items in order of their work, or null
    int ctas_k, ctas_q;    // CTAs of a head (0: no such pass)
};
struct Maps {              // 128 rows for those a CTA owns, 64 for those it streams
    CUtensorMap q, grad, k, v;
};

// one owned tile: its rows [x0, x0 + 128) of problem b, and the streamed rows [y0, ..) in `per` tiles that any of them meets
struct Item {
    int b, x0, lq, lk, y0, per;
};
template <bool DKV>
__device__ __forceinline__ Item item_at(const AttnArgs& a, const int* order, int index) {
    Item w;
    const int row_tiles = ((DKV ? a.Lk : a.Lq) + kOwn - 1) / kOwn;
    if (order) index = order[index];
    // causal: the first keys and the last queries have the most to do, over all problems
    w.b = a.causal ? index % a.B : index / row_tiles;
    int t = a.causal ? index / a.B : index % row_tiles;
    if (a.causal && !DKV) t = row_tiles - 1 - t;
    w.x0 = t * kOwn;
    problem_lengths(a, w.b, &w.lq, &w.lk);
    const int off = a.causal ? w.lk - w.lq : 0;
    w.y0 = 0;
    int y1 = w.x0 < (DKV ? w.lk : w.lq) ? (DKV ? w.lq : w.lk) : 0;
    if (a.causal) {
        if (DKV) w.y0 = max(0, w.x0 - off) / kStep * kStep;
        else y1 = min(y1, min(w.x0 + kOwn, w.lq) + off);
    }
    w.per = y1 > w.y0 ? (y1 - w.y0 + kStep - 1) / kStep : 0;
    return w;
}

// rows of X past the lengths never reach a sum of another row; rows of Y do (0 x NaN), and are zeroed in shared memory
// CTA y of the `ys` of head hx
template <class T, int DP, bool BIAS, bool DKV>
__device__ __forceinline__ void attn_bwd_pass(const CUtensorMap& tmX1, const CUtensorMap& tmX2, const CUtensorMap& tmY1,
                                              const CUtensorMap& tmY2, const Args& g, const int hx, const int y_cta, const int y_ctas) {
    using Sh = Shape<DP, BIAS>;
    constexpr int NST = Sh::kStages, NB = buffers<DP, DKV>(), NS = score_bars(NB), NX = Sh::kOwned;
    const AttnArgs& a = g.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int group = a.H / a.Hkv;
    const int* const order = DKV ? g.order_k : g.order_q;
    void *const dx1 = g.dv, *const dx2 = DKV ? g.dk : g.dq;   // (the query pass has one result)
    const int Lx = DKV ? a.Lk : a.Lq, heads = DKV ? a.Hkv : a.H, row_tiles = (Lx + kOwn - 1) / kOwn, items = a.B * row_tiles;
    const int count = item_count(items, y_cta, y_ctas);   // of this CTA

    extern __shared__ uint8_t raw[];
    const uint32_t r0 = smem_addr(raw), base = (r0 + 1023u) & ~1023u;
    uint8_t* const gb = raw + (base - r0);
    const uint32_t sY = base + 2 * NX * Sh::kX;
    uint64_t* const bars = reinterpret_cast<uint64_t*>(gb + Sh::kTiles);
    const uint32_t barX = smem_addr(bars), barXE = barX + 8 * NX, barF = barXE + 8 * NX, barA = barF + 8, barY = barA + 8,
                   barE = barY + 8 * NST, barS = barE + 8 * NST, barP = barS + 8 * NS, barPE = barP + 24, barD = barPE + 24;   // (D: the products' end, after a wait that gave up)
    uint8_t* const after = gb + (Sh::kTiles + Sh::kBars * 8 + 15) / 16 * 16;
    const Dead dead = {reinterpret_cast<volatile int*>(after), a.polls};
    uint32_t* const slot = reinterpret_cast<uint32_t*>(after) + 1;
    int* const asked = reinterpret_cast<int*>(after) + 2;                    // items (with work) and streamed tiles whose copies were issued
    int4* const entry = reinterpret_cast<int4*>(after + 16);                 // b, x0, lq, lk of an item
    int2* const span = reinterpret_cast<int2*>(entry + kMaxItems);           // and y0, per
    float* const lut = reinterpret_cast<float*>(span + kMaxItems);
    const int reach = BIAS ? reach_of(a.edges) : 0;
    float* const diag = lut + lut_size(reach);                        // [16][144] a warp's diagonals, and their scan
    float* const red = diag + 16 * 144;                               // [16][kBuckets]
    int* const range = reinterpret_cast<int*>(red + 16 * kBuckets);   // [kBuckets][2] positions of a bucket
    uint32_t* const starts = reinterpret_cast<uint32_t*>(range + 2 * kBuckets);   // [kStartWords] bit d + reach + kPad: a bucket begins at d
    const bool sums = !DKV && BIAS && g.part;

    auto copy = [&](uint32_t dst, const CUtensorMap* tm, int row, int head, int b, uint32_t bar, int chunk) {
#pragma unroll
        for (int c = 0; c < Sh::kChunks; ++c) tma_load(dst + c * chunk, tm, 64 * c, row, head, b, bar);
    };
    auto own = [&](int i, int b, int x0) {   // item i (of those with work): its X1 and X2
        const uint32_t dst = base + (i % NX) * 2 * Sh::kX, bar = barX + 8 * (i % NX);
        bar_expect(bar, 2 * Sh::kX);
        copy(dst, &tmX1, x0, hx, b, bar, kChunkX);
        copy(dst + Sh::kX, &tmX2, x0, hx, b, bar, kChunkX);
    };
    auto stream = [&](int t, int b, int row, int head) {   // streamed tile t: its Y1, Y2 and row statistics
        const uint32_t dst = sY + (t % NST) * Sh::kStage, bar = barY + 8 * (t % NST);
        bar_expect(bar, 2 * Sh::kY + (DKV ? Sh::kRowStats : 0));
        copy(dst, &tmY1, row, head, b, bar, kChunkY);
        copy(dst + Sh::kY, &tmY2, row, head, b, bar, kChunkY);
        if (DKV) {
            const size_t at = ((size_t)b * a.H + head) * g.Lp + row;
#pragma unroll
            for (int w = 0; w < 2; ++w)
                asm volatile(
                    "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                        dst + 2 * Sh::kY + w * kStep * 4),
                    "l"((w ? g.delta : g.lse) + at), "r"(kStep * 4), "r"(bar)
                    : "memory");
        }
    };
    bool large = false;   // whether rows of these heads have bases
    if (warp == kWork / 32 + 2) {   // barriers, and the first item's copies before the CTA meets
        if (lane == 0) {
            for (int s = 0; s < NX; ++s) bar_init(barX + 8 * s, 1), bar_init(barXE + 8 * s, 1);
            bar_init(barF, 1), bar_init(barA, kWork / 32), bar_init(barD, 1), bar_init(barD + 8, 1);
            for (int s = 0; s < NST; ++s) bar_init(barY + 8 * s, 1), bar_init(barE + 8 * s, 1);
            for (int s = 0; s < NS; ++s) bar_init(barS + 8 * s, 1);
            for (int s = 0; s < NB; ++s) bar_init(barP + 8 * s, 8), bar_init(barPE + 8 * s, 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            fence_async_smem();
            *dead.flag = 0;
            const Item w = item_at<DKV>(a, order, item_index(0, y_cta, y_ctas));
            if (w.per) {
                own(0, w.b, w.x0);
                stream(0, w.b, w.y0, DKV ? hx * group : hx / group);
            }
        }
        __syncwarp();
    } else if (warp == kWork / 32) {
        tmem_alloc(smem_addr(slot), kColumns);
    } else if (warp < kWork / 32) {
        for (int e = tid; e < count; e += kWork) {
            const Item w = item_at<DKV>(a, order, item_index(e, y_cta, y_ctas));
            entry[e] = make_int4(w.b, w.x0, w.lq, w.lk);
            span[e] = make_int2(w.y0, w.per);
        }
        __syncwarp();
        if (BIAS && (!DKV || group == 1)) large = fill_lut<T>(lut, a, hx, reach, warp, kWork / 32);
        if (BIAS && DKV && group > 1)
            for (int t = tid; t < group * n_buckets(a.edges); t += kWork) large |= large_bias(bias_log2<T>(a, t / group, hx * group + t % group));
        if (sums)
            for (int t = tid; t < n_buckets(a.edges); t += kWork) {
                const int2 v = bucket_range(a.edges, t, 1 << 29);
                range[2 * t] = v.x, range[2 * t + 1] = v.y;
            }
        if (sums && warp == 0) {
            for (int t = lane; t < kStartWords; t += 32) starts[t] = 0u;
            __syncwarp();
            for (int t = lane; t < n_buckets(a.edges); t += 32) {
                const int at = bucket_range(a.edges, t, 1 << 29).x + reach + kPad;
                if (at >= 0) atomicOr(starts + (at >> 5), 1u << (at & 31));
            }
        }
    }
    tc_fence_before();
    large = __syncthreads_or(large);
    tc_fence_after();
    const uint32_t tmem = *slot, tA1 = tmem + 128 * NB, tA2 = DKV ? tA1 + DP : tA1;

    if (warp == kWork / 32 + 2) {   // copies
        if (lane == 0) {
            bool ok = true;
            int t = 0, i = 0;   // streamed tiles and items (with work) asked for
            for (int e = 0; ok && e < count; ++e) {
                const int per = span[e].y, y0 = span[e].x;
                if (per == 0) continue;
                const int b = entry[e].x;
                if (i >= NX && !(ok = bar_wait(barXE + 8 * (i % NX), (i / NX - 1) & 1, dead))) break;
                if (e > 0) own(i, b, entry[e].y);   // (the first item's are under way)
                ++i;
                for (int k = 0; ok && k < (DKV ? group : 1); ++k)
                    for (int step = 0; step < per; ++step, ++t) {
                        if (t >= NST && !(ok = bar_wait(barE + 8 * (t % NST), (t / NST - 1) & 1, dead))) break;
                        if (e + t > 0) stream(t, b, y0 + step * kStep, DKV ? hx * group + k : hx / group);
                    }
            }
            asked[0] = i, asked[1] = t;
        }
        __syncwarp();
    } else if (warp >= kWork / 32) {
        // Products: one warp forms the scores, one the sums, so that neither's waits and issues stand before the other's;
        // with two buffers only, one warp does both, since there the scores should follow the sums' products at once (keys
        // pass, heads of 128: 1830 clocks a tile together, 2325 apart; query pass: 1677 together, 1428 apart).
        // A whole warp runs this, its operands' words in uniform registers; one lane issues
        constexpr bool kApart = NB > 2;
        const bool lead = elect_one();
        const uint32_t tm = uniform(tmem), uA1 = tm + 128 * NB, uA2 = DKV ? uA1 + DP : uA1;
        bool ok = true;
        int t = 0, i = 0;   // tiles and items (with work) so far
        // (steps past the head's size are left out)
        const int steps = (a.D + 15) / 16;
        const uint32_t idS = mma_desc<T>(128, kStep, false), idA = mma_desc<T>(128, 16 * steps, true);
        auto scores = [&](int t, uint32_t dX) {
            const int s = t % NST, buf = t % NB;
            if (!bar_wait_warp(barY + 8 * s, (t / NST) & 1, dead)) return false;
            if (kApart && t >= NB && !bar_wait_warp(barPE + 8 * buf, (t / NB - 1) & 1, dead)) return false;
            tc_fence_after();
            const uint32_t d = tm + buf * 128, dY = desc_along(sY + s * Sh::kStage);
#pragma unroll
            for (int w = 0; w < 2; ++w)
#pragma unroll
                for (int k = 0; k < DP / 16; ++k)
                    if (lead && k < steps) mma_ss(d + 64 * w, dX + (w * Sh::kX + (k / 4) * kChunkX + (k % 4) * 32) / 16,
                                     dY + (w * Sh::kY + (k / 4) * kChunkY + (k % 4) * 32) / 16, idS, k != 0);
            if (lead) tc_commit(barS + 8 * (t % NS));
            return true;
        };
        if (kApart && warp == kWork / 32) {
            for (int e = 0; ok && e < count; ++e) {
                const int n = (int)uniform(span[e].y * (DKV ? group : 1));
                if (n == 0) continue;
                const int xs = i % NX;
                if (!(ok = bar_wait_warp(barX + 8 * xs, (i / NX) & 1, dead))) break;
                const uint32_t dX = desc_along(base + xs * 2 * Sh::kX);
                for (int it = 0; it < n; ++it, ++t)
                    if (!(ok = scores(t, dX))) break;
                if (lead) tc_commit(barXE + 8 * xs);   // the owned tile's last use
                ++i;
            }
        } else if (warp == kWork / 32 + 1) {
            for (int e = 0; ok && e < count; ++e) {
                const int n = (int)uniform(span[e].y * (DKV ? group : 1));
                if (n == 0) continue;
                const int xs = i % NX;
                const uint32_t dX = desc_along(base + xs * 2 * Sh::kX);
                if (!kApart) {
                    ok = bar_wait_warp(barX + 8 * xs, (i / NX) & 1, dead);
                    for (int it = 0; ok && it < NB && it < n; ++it) ok = scores(t + it, dX);
                    if (!ok) break;
                }
                for (int it = 0; it < n; ++it, ++t) {
                    const int s = t % NST, buf = t % NB;
                    if (!(ok = bar_wait_warp(barP + 8 * buf, (t / NB) & 1, dead))) break;
                    if (it == 0 && i > 0 && !(ok = bar_wait_warp(barA, (i - 1) & 1, dead))) break;   // the results before are read
                    tc_fence_after();
                    const uint32_t p = tm + buf * 128, dY = desc_down(sY + s * Sh::kStage, kChunkY);
                    if (DKV) {
#pragma unroll
                        for (int k = 0; k < kStep / 16; ++k)
                            if (lead) mma_ts(uA1, p + 32 * (k / 2) + 8 * (k % 2), dY + (Sh::kY + k * 2048) / 16, idA, (it | k) != 0);
                    }
#pragma unroll
                    for (int k = 0; k < kStep / 16; ++k)
                        if (lead) mma_ts(uA2, p + 64 + 32 * (k / 2) + 8 * (k % 2), dY + k * (2048 / 16), idA, (it | k) != 0);
                    if (lead) tc_commit(barE + 8 * s);
                    if (kApart) {
                        if (lead) tc_commit(barPE + 8 * buf);
                    } else {
                        if (it + NB < n && !(ok = scores(t + NB, dX))) break;
                        if (it + NB == max(n, NB) && lead) tc_commit(barXE + 8 * xs);   // the owned tile's last use
                    }
                }
                if (!ok) break;   // (sums without their last products must not pass for whole ones)
                if (lead) tc_commit(barF);
                ++i;
            }
        }
        __syncwarp();
    } else {   // P and dS of a tile
        const int pair = warp >> 3, half = (warp >> 2) & 1, w4 = warp & 3, r = tid & 127;
        const uint32_t trow = (uint32_t)(32 * w4) << 16;
        const float c = a.scale * kLog2e;
        bool ok = true;
        float* const dw = diag + warp * 144;
        int t0 = 0, done = 0;   // tiles and items (with work) so far
        float far0 = 0.f, far1 = 0.f, bsum[kBuckets / 32];   // dS by position, over all the CTA's items
#pragma unroll
        for (int i = 0; i < kBuckets / 32; ++i) bsum[i] = 0.f;

        // An item's results are stored after this warp's first tile of the next one, whose work covers the wait for the
        // last products.  keys pass: half of dV's or dK's columns a warpgroup; query pass: a quarter of dQ's.  A row a
        // thread, whole 32-byte sectors
        constexpr bool kScaled = std::is_same<T, __half>::value;   // (bf16 has fp32's range)
        int kept_b = -1, kept_x = 0, kept_l = 0;   // problem, this thread's row, rows there are
        float kept_down = 1.f;                     // and 2^-k of its dS
        auto store = [&]() {
            ok = ok && bar_wait_warp(barF, (done - 1) & 1, dead);
            tc_fence_after();
            const bool row = kept_x < kept_l, first = DKV && pair == 0;
            const float w = first ? Softmax<T>::kDown : kScaled ? a.scale * kept_down : a.scale;
            const int f0 = DKV ? half * (DP / 2) : (warp >> 2) * (DP / 4);
            constexpr int kCols = DKV ? DP / 2 : DP / 4;
            const uint32_t acc = (first ? tA1 : tA2) + trow;
            uint32_t o[kCols];
#pragma unroll
            for (int f = 0; f < kCols; f += 16) tmem_ld16(acc + f0 + f, o + f);
            tmem_wait_ld();
#pragma unroll
            for (int f = 0; f < kCols; f += 16) tmem_tie16(o + f);
            tc_fence_before();
            bar_arrive_warp(barA);   // the next item's products may overwrite them
            const bool whole = a.D % 16 == 0 && (((uintptr_t)dx1 | (uintptr_t)dx2) & 31) == 0;
            if (kept_x < Lx) {
                T* const rp = (T*)(first ? dx1 : dx2) + (((size_t)kept_b * Lx + kept_x) * heads + hx) * a.D + f0;
#pragma unroll
                for (int y = 0; y < kCols; y += 16) {
                    uint32_t p[8];
#pragma unroll
                    for (int z = 0; z < 8; ++z) {
                        const float u0 = __uint_as_float(o[y + 2 * z]) * w, u1 = __uint_as_float(o[y + 2 * z + 1]) * w;
                        p[z] = !row ? 0u : ok ? pack2<T>(u0, u1) : pack2<T>(NAN, NAN);
                    }
                    if (f0 + y < a.D) store16(rp + y, p, a.D - f0 - y, whole);
                }
            }
            kept_b = -1;
        };
        // the row statistics of the next item, asked for one ahead (query pass)
        float nl = 0.f, nd = 0.f;
        auto ask = [&](int e) {
            if (!DKV && e < count) {
                const int4 en = entry[e];
                const size_t at = ((size_t)en.x * a.H + hx) * g.Lp + en.y + r;   // Lp covers the tile
                nl = g.lse[at], nd = g.delta[at];
            }
        };
        // LARGE: rows have bases.  A loop of its own (in the same one the others took a tenth longer)
        auto items = [&](auto large_c) {
        constexpr bool LARGE = decltype(large_c)::value;
        ask(0);
        for (int e = 0; e < count; ++e) {
            const int4 en = entry[e];
            const float rl = nl, rd = nd;   // -lse, -delta
            ask(e + 1);
            // (from one lane for all, so that the branches on them are known to be the warp's)
            const int x0 = __shfl_sync(0xffffffffu, en.y, 0), lq = __shfl_sync(0xffffffffu, en.z, 0), lk = __shfl_sync(0xffffffffu, en.w, 0);
            const int y0 = __shfl_sync(0xffffffffu, span[e].x, 0), per = __shfl_sync(0xffffffffu, span[e].y, 0);
            const int b = en.x, off = a.causal ? lk - lq : 0, lx = DKV ? lk : lq, ly = DKV ? lq : lk, x = x0 + r;
            if (per == 0) {   // nothing meets these rows
                const int rows = min(kOwn, Lx - x0), units = a.D / 8;
                for (int v = tid; v < rows * units; v += kWork) {
                    const size_t at = (((size_t)b * Lx + x0 + v / units) * heads + hx) * a.D + (v % units) * 8;
                    *reinterpret_cast<uint4*>((T*)dx2 + at) = make_uint4(0, 0, 0, 0);
                    if (DKV) *reinterpret_cast<uint4*>((T*)dx1 + at) = make_uint4(0, 0, 0, 0);
                }
                continue;
            }
            float up = 1.f, down = 1.f;
            if (kScaled) {
                const size_t at = (size_t)b * a.Hkv + (DKV ? hx : hx / group);
                const float2 s = ds_scale(g.grad_top[at], g.v_top[at]);
                up = s.x, down = s.y;
            }
            for (int head = 0; head < (DKV ? group : 1); ++head) {
                if (BIAS && DKV && group > 1) {   // keys pass: the bias of the group's next head, once every warp is past the one before
                    asm volatile("bar.sync 1, 512;" ::: "memory");
                    fill_lut<T>(lut, a, hx * group + head, reach, warp, kWork / 32);
                    asm volatile("bar.sync 1, 512;" ::: "memory");
                }
                for (int step = (pair ^ (t0 + head * per)) & 1; step < per; step += 2) {   // this pair's tiles of the head
                    const int t = t0 + head * per + step, s = t % NST, buf = t % NB, yb = y0 + step * kStep;
                    // (after a wait that gave up a warp still meets its partners at the barriers above)
                    // (the streamed tile's own barrier: the keys pass reads the row statistics that came with it.  After the scores',
                    // which were formed behind it: a pair sees a stage's phases two apart where there are three stages, and the
                    // parity alone would not tell this one from the last but one)
                    ok = ok && bar_wait_warp(barS + 8 * (t % NS), (t / NS) & 1, dead) &&
                         (!DKV || bar_wait_warp(barY + 8 * s, (t / NST) & 1, dead));
                    if (!ok) continue;
                    tc_fence_after();
                    const int col0 = 32 * half, yc = yb + col0;
                    const uint32_t tS = tmem + trow + buf * 128, tD = tS + 64;
                    const float* const st = reinterpret_cast<const float*>(gb + 2 * NX * Sh::kX + s * Sh::kStage + 2 * Sh::kY) + col0;
                    // d = key position - query position of this row and the block's first column; a column is one less or one more
                    const int d0 = DKV ? x - (yc + off) : yc - (x + off);
                    // the range of d in the warp's block of 32 x 32
                    const int lo = DKV ? x0 + 32 * w4 - (yc + 31 + off) : yc - (x0 + 32 * w4 + 31 + off), hi = lo + 62;
                    const bool near = BIAS && lo < reach && hi > -reach;
                    // columns this row meets: [c0, c1)
                    int c0 = 0, c1 = x < lx ? min(32, ly - yc) : 0;
                    if (a.causal) {
                        if (DKV) c0 = max(0, d0);
                        else c1 = min(c1, 1 - d0);
                    }
                    const bool edge = __any_sync(0xffffffffu, c0 > 0 || c1 < 32);
                    bool live_block = true;
                    float run = 0.f, all = 0.f;   // the diagonals under way; the sum of a block in one bucket
                    // (forms without the masks and without the bias by position: a block needs them rarely)
                    auto block = [&](auto edge_c, auto near_c) {
                        constexpr bool EDGE = decltype(edge_c)::value, NEAR = decltype(near_c)::value;
                        // four columns' entries at lp +- y: the keys pass meets them in falling order
                        const float* const lp = lut_row(lut, reach, d0 + reach + kPad - (DKV ? 3 : 0));
                        const float flat = BIAS && !NEAR ? (lo >= reach ? lut[lut_entries(reach) - 1] : lut[0]) : 0.f;
                        const float* const bases = LARGE ? g.base + ((size_t)b * a.H + (DKV ? hx * group + head : hx)) * g.Lp + (DKV ? yc : x) : nullptr;
                        uint32_t sv[32], dv[32];
                        tmem_ld32(tS + col0, sv);
                        tmem_ld32(tD + col0, dv);
                        tmem_wait_ld();
                        tmem_tie32(sv), tmem_tie32(dv);
#pragma unroll
                        for (int y = 0; y < 32; y += 4) {
                            float4 L = make_float4(rl, rl, rl, rl), E = make_float4(rd, rd, rd, rd);   // -lse and -delta
                            if (DKV) {
                                L = *reinterpret_cast<const float4*>(st + y);
                                E = *reinterpret_cast<const float4*>(st + kStep + y);
                            }
                            float pv[4], gv[4];
                            Two t0(__uint_as_float(sv[y]), __uint_as_float(sv[y + 1])), t1(__uint_as_float(sv[y + 2]), __uint_as_float(sv[y + 3]));
                            const Two L0(L.x, L.y), L1(L.z, L.w);
                            if (LARGE) {
                                const float4 R = DKV ? *reinterpret_cast<const float4*>(bases + y) : make_float4(*bases, *bases, *bases, *bases);
                                float4 e = make_float4(flat, flat, flat, flat);
                                if (NEAR) {
                                    e = *reinterpret_cast<const float4*>(DKV ? lp - y : lp + y);
                                    if (DKV) e = make_float4(e.w, e.z, e.y, e.x);
                                }
                                t0 = add2(fma2(t0, Two(score_factor(R.x, c), score_factor(R.y, c)), Two(e.x - R.x, e.y - R.y)), L0);
                                t1 = add2(fma2(t1, Two(score_factor(R.z, c), score_factor(R.w, c)), Two(e.z - R.z, e.w - R.w)), L1);
                            } else if (BIAS && NEAR) {
                                const float4 e = *reinterpret_cast<const float4*>(DKV ? lp - y : lp + y);
                                t0 = add2(fma2(t0, Two(c, c), DKV ? Two(e.w, e.z) : Two(e.x, e.y)), L0);
                                t1 = add2(fma2(t1, Two(c, c), DKV ? Two(e.y, e.x) : Two(e.z, e.w)), L1);
                            } else {
                                const Two m(c, c), f(flat, flat);
                                t0 = fma2(t0, m, BIAS ? add2(f, L0) : L0), t1 = fma2(t1, m, BIAS ? add2(f, L1) : L1);
                            }
                            t0.get(pv, pv + 1), t1.get(pv + 2, pv + 3);
#pragma unroll
                            for (int z = 0; z < 4; ++z) pv[z] = ex2(pv[z]);
                            const Two d0(__uint_as_float(dv[y]), __uint_as_float(dv[y + 1])), d1(__uint_as_float(dv[y + 2]), __uint_as_float(dv[y + 3]));
                            // (fp16: P is 2^kShift times as large here, delta that much less, and dS 2^k times as large)
                            const float w = Softmax<T>::kDown * up;
                            Two E0(E.x, E.y), E1(E.z, E.w);
                            if (kScaled) E0 = mul2(E0, Two(up, up)), E1 = mul2(E1, Two(up, up));
                            mul2(Two(pv[0], pv[1]), kScaled ? fma2(d0, Two(w, w), E0) : add2(d0, E0)).get(gv, gv + 1);
                            mul2(Two(pv[2], pv[3]), kScaled ? fma2(d1, Two(w, w), E1) : add2(d1, E1)).get(gv + 2, gv + 3);
#pragma unroll
                            for (int z = 0; z < 4; ++z) {
                                const int col = y + z;
                                if (EDGE) {
                                    const bool in = col >= c0 && col < c1;
                                    pv[z] = in ? pv[z] : 0.f;
                                    gv[z] = in ? gv[z] : 0.f;
                                }
                                if (BIAS && !DKV) {
                                    if (NEAR) {
                                        run = __shfl_up_sync(0xffffffffu, run, 1);
                                        run = (lane ? run : 0.f) + gv[z];
                                        if (lane == 31) dw[col] = run;
                                    } else {
                                        all += gv[z];
                                    }
                                }
                            }
                            sv[y / 2] = pack2<T>(pv[0], pv[1]), sv[y / 2 + 1] = pack2<T>(pv[2], pv[3]);
                            dv[y / 2] = pack2<T>(gv[0], gv[1]), dv[y / 2 + 1] = pack2<T>(gv[2], gv[3]);
                        }
                        if (DKV) tmem_st16(tS + col0, sv);
                        tmem_st16(tD + col0, dv);
                    };
                    if (!__any_sync(0xffffffffu, c0 < c1)) {   // the whole block masked: zeros, whatever S holds
                        uint32_t zero[16];
#pragma unroll
                        for (int y = 0; y < 16; ++y) zero[y] = 0u;
                        if (DKV) tmem_st16(tS + col0, zero);
                        tmem_st16(tD + col0, zero);
                        live_block = false;
                    } else if (BIAS && near) {
                        if (LARGE || edge) block(std::true_type{}, std::true_type{});
                        else block(std::integral_constant<bool, LARGE>{}, std::true_type{});
                    } else {
                        if (LARGE || edge) block(std::true_type{}, std::false_type{});
                        else block(std::integral_constant<bool, LARGE>{}, std::false_type{});
                    }
                    const int live = ly - yb;
                    if (live < kStep) {   // rows of Y past the length to zero, for the products that sum over them
                        uint8_t* const y = gb + 2 * NX * Sh::kX + s * Sh::kStage;
                        const int dead_units = (kStep - live) * 8;
                        for (int e = tid & 255; e < dead_units * Sh::kChunks * (DKV ? 2 : 1); e += 256) {
                            const int ch = e / dead_units, o = e % dead_units;
                            *reinterpret_cast<uint4*>(y + ch * kChunkY + live * 128 + o * 16) = make_uint4(0, 0, 0, 0);
                        }
                        fence_async_smem();
                    }
                    tmem_wait_st();
                    tc_fence_before();
                    bar_arrive_warp(barP + 8 * buf);
                    if (kept_b >= 0) store();   // the item before
                    if (sums && live_block) {
                        if (near) {
                            dw[62 - lane] = run;   // the diagonals still under way; lane 31's is in place
                            __syncwarp();
                            // the 63 sums (and a zero): lane l takes 2 l and 2 l + 1, and scans from where their buckets begin
                            const float s0 = dw[2 * lane], s1 = lane < 31 ? dw[2 * lane + 1] : 0.f;
                            const int at = lo + reach + kPad + (lane < 16 ? 0 : 32);
                            const uint32_t begin = __funnelshift_r(starts[at >> 5], starts[(at >> 5) + 1], at & 31) >> ((2 * lane) & 31);
                            const uint32_t from = (__ballot_sync(0xffffffffu, (begin & 3u) != 0) | 1u) & (0xffffffffu >> (31 - lane));
                            const int first = 31 - __clz(from);   // the lane in which this one's last bucket begins
                            float t = begin & 2u ? s1 : s0 + s1;
#pragma unroll
                            for (int o = 1; o < 32; o <<= 1) {
                                const float u = __shfl_up_sync(0xffffffffu, t, o);
                                if (lane - o >= first) t += u;
                            }
                            const float u = __shfl_up_sync(0xffffffffu, t, 1);
                            // sum[e]: of the diagonals up to lo + e that lie in its bucket
                            float* const sum = dw + 72;
                            sum[2 * lane] = begin & 1u || lane == 0 ? s0 : u + s0, sum[2 * lane + 1] = t;
                            __syncwarp();
                            const int nb = n_buckets(a.edges);
#pragma unroll
                            for (int i = 0; i < kBuckets / 32; ++i) {
                                const int t2 = lane + 32 * i;
                                if (t2 < nb) {
                                    const int e0 = max(range[2 * t2] - lo, 0), e1 = min(range[2 * t2 + 1] - lo + 1, 63);
                                    if (e0 < e1) bsum[i] += down * sum[e1 - 1];
                                }
                            }
                            __syncwarp();
                        } else if (lo >= reach) {
                            far1 += down * all;
                        } else {
                            far0 += down * all;
                        }
                    }
                }
            }
            if (kept_b >= 0) store();   // (this warp had no tile of the item)
            kept_b = b, kept_x = x, kept_l = lx, kept_down = down;
            t0 += per * (DKV ? group : 1), ++done;
        }
        };
        if (!BIAS || __builtin_expect(!large, 1)) items(std::false_type{});
        else items(std::integral_constant<bool, BIAS>{});
        if (kept_b >= 0) store();
        if (sums) {   // the CTA's sums, warp by warp in order
            const int nb = n_buckets(a.edges);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                far0 += __shfl_xor_sync(0xffffffffu, far0, o);
                far1 += __shfl_xor_sync(0xffffffffu, far1, o);
            }
#pragma unroll
            for (int i = 0; i < kBuckets / 32; ++i) {
                const int t = lane + 32 * i;
                if (t < nb) red[warp * kBuckets + t] = !ok ? NAN : bsum[i] + (t == a.edges.n ? far0 : 0.f) + (a.edges.two && t == nb - 1 ? far1 : 0.f);
            }
            asm volatile("bar.sync 1, 512;" ::: "memory");
            for (int t = tid; t < nb; t += kWork) {
                float v = 0.f;
#pragma unroll
                for (int k = 0; k < kWork / 32; ++k) v += red[k * kBuckets + t];
                g.part[((size_t)hx * nb + t) * y_ctas + y_cta] = v;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (*dead.flag) {   // a wait gave up: what is in flight ends (bounded) before the CTA does
        if (warp < kWork / 32) tmem_wait_st();
        if (warp == kWork / 32 || warp == kWork / 32 + 1) tc_drain(barD + 8 * (warp - kWork / 32));
        if (warp == kWork / 32 + 2 && lane == 0) {
            int none = 0;
            const Dead end = {&none, kWaitLimit};
            for (int x = max(0, asked[0] - NX); x < asked[0]; ++x) bar_wait(barX + 8 * (x % NX), (x / NX) & 1, end);
            for (int x = max(0, asked[1] - NST); x < asked[1]; ++x) bar_wait(barY + 8 * (x % NST), (x / NST) & 1, end);
            atomicAdd(&g_gave_up, 1ull);
        }
        __syncthreads();
    }
    if (warp == kWork / 32) tmem_free(tmem, kColumns);
}

// Both passes wait for the statistics and the order at their start: what these wrote is theirs to read only after that wait.
// 1 x 4096 causal, 16/4 heads of 128, whose 128 items of keys leave SMs free: 285 us, 370 as two launches one after the other
template <class T, int DP, bool BIAS>
__global__ void __launch_bounds__(kThreads, 1)
    attn_bwd_kernel(const __grid_constant__ Maps own, const __grid_constant__ Maps str, const __grid_constant__ Args g) {
    wait_ahead();   // (the statistics and the order)
    const int keys = g.ctas_k * g.a.Hkv;
    if ((int)blockIdx.x < keys) {
        attn_bwd_pass<T, DP, BIAS, true>(own.k, own.v, str.q, str.grad, g, blockIdx.x % g.a.Hkv, blockIdx.x / g.a.Hkv, g.ctas_k);
    } else {
        const int at = blockIdx.x - keys;
        attn_bwd_pass<T, DP, BIAS, false>(own.q, own.grad, str.k, str.v, g, at % g.a.H, at / g.a.H, g.ctas_q);
    }
}

// -delta = -rowsum(dO O) (times kDown) and kShift - lse in rows padded to whole tiles: 0 and -inf where no key is met; and the
// rows' bases, where there is a bias.  O with what its
// rounding took, where it is there.  A block takes 16
// positions of up to 8 heads: rows are read as they lie, heads of a position together, and the sums leave by head, 16
// positions together.  LANES threads a row
constexpr int kStatRows = 16, kStatHeads = 8;
template <class T, int LANES>
__global__ void __launch_bounds__(256) attn_stats_kernel(const __grid_constant__ AttnArgs a, const T* __restrict__ out, const T* __restrict__ rest,
                                                         const float* __restrict__ lse, const T* __restrict__ grad, int Lp,
                                                         float* __restrict__ lp, float* __restrict__ dp, float* __restrict__ bp,
                                                         unsigned* __restrict__ grad_top) {
    let_next();
    constexpr bool kScaled = std::is_same<T, __half>::value;
    __shared__ float sum[kStatHeads][kStatRows + 1], norm[kScaled ? kStatHeads : 1][kStatRows + 1];
    const int lane = threadIdx.x % LANES, i0 = blockIdx.x * kStatRows, h0 = blockIdx.y * kStatHeads, b = blockIdx.z;
    const int heads = min(kStatHeads, a.H - h0);
    int lq, lk;
    problem_lengths(a, b, &lq, &lk);
    constexpr int kStride = 256 / LANES;
#pragma unroll
    for (int k = 0; k < kStatRows * kStatHeads / kStride; ++k) {
        const int row = k * kStride + threadIdx.x / LANES, i = i0 + row / kStatHeads, h = row % kStatHeads;
        float d = 0.f, n = 0.f;
        if (i < lq && h < heads && 8 * lane < a.D) {
            const size_t at = (((size_t)b * a.Lq + i) * a.H + h0 + h) * a.D + 8 * lane;
            float o[8], g[8];
            load8<T>(out + at, o);
            load8<T>(grad + at, g);
#pragma unroll
            for (int x = 0; x < 8; ++x) d = fmaf(o[x], g[x], d), n = fmaf(g[x], g[x], n);
            if (rest) {
                load8<T>(rest + at, o);
#pragma unroll
                for (int x = 0; x < 8; ++x) d = fmaf(o[x], g[x], d);
            }
        }
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) {
            d += __shfl_xor_sync(0xffffffffu, d, o);
            if (kScaled) n += __shfl_xor_sync(0xffffffffu, n, o);
        }
        if (lane == 0) sum[h][row / kStatHeads] = d;
        if (kScaled && lane == 0) norm[h][row / kStatHeads] = n;
    }
    bool large = false;
    if (bp)
        for (int x = threadIdx.x; x < heads * n_buckets(a.edges); x += 256) large |= large_bias(bias_log2<T>(a, x / heads, h0 + x % heads));
    large = __syncthreads_or(large);
    if (kScaled && threadIdx.x < heads) {   // (NaN is above every number here)
        unsigned top = 0;
#pragma unroll
        for (int x = 0; x < kStatRows; ++x) top = max(top, __float_as_uint(sqrtf(norm[threadIdx.x][x])));
        atomicMax(grad_top + (size_t)b * a.Hkv + (h0 + threadIdx.x) / (a.H / a.Hkv), top);
    }
    const int h = threadIdx.x / kStatRows, i = i0 + threadIdx.x % kStatRows;
    if (h < heads && h < kStatHeads) {
        const size_t at = ((size_t)b * a.H + h0 + h) * Lp + i;
        dp[at] = -sum[h][threadIdx.x % kStatRows] * Softmax<T>::kDown;
        if (bp) {
            const int pos = i + (a.causal ? lk - lq : 0);
            bp[at] = large && i < lq ? base_of(row_top<T>(a, h0 + h, pos, a.causal ? min(lk, pos + 1) : lk)) : 0.f;
        }
        lp[at] = i < lq ? Softmax<T>::kShift - lse[((size_t)b * a.H + h0 + h) * a.Lq + i] : -INFINITY;
    }
    // (the order is not read here, but by the passes, which wait for this launch alone: one block ends after it)
    if (blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1 && blockIdx.z == gridDim.z - 1) wait_ahead();
}

// the largest norm of V's live rows of each problem and key head, LANES threads a row (fp16)
template <int LANES>
__global__ void __launch_bounds__(256) attn_v_top_kernel(const __grid_constant__ AttnArgs a, unsigned* __restrict__ v_top) {
    const int lane = threadIdx.x % LANES, kh = blockIdx.y, b = blockIdx.z;
    int lq, lk;
    problem_lengths(a, b, &lq, &lk);
    const __half* const v = (const __half*)a.v + b * a.vs[0] + kh * a.vs[2] + 8 * lane;
    constexpr int kStride = 256 / LANES;
    unsigned top = 0;
    for (int j0 = blockIdx.x * kStride; j0 < lk; j0 += gridDim.x * kStride) {
        const int j = j0 + threadIdx.x / LANES;
        float n = 0.f;
        if (j < lk && 8 * lane < a.D) {
            float x[8];
            load8<__half>(v + (long long)j * a.vs[1], x);
#pragma unroll
            for (int i = 0; i < 8; ++i) n = fmaf(x[i], x[i], n);
        }
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
        top = max(top, __float_as_uint(sqrtf(n)));
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0 && top) atomicMax(v_top + (size_t)b * a.Hkv + kh, top);
}

// dbias[t][h]: one warp each, the CTAs' sums in a fixed order
template <class T>
__global__ void __launch_bounds__(128) attn_dbias_kernel(const float* part, int nb, int H, int n, T* dbias) {
    const int lane = threadIdx.x & 31, at = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (at >= nb * H) return;
    const int h = at / nb, t = at % nb;
    float s = 0.f;
    for (int k = lane; k < n; k += 32) s += part[(size_t)at * n + k];
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    if (lane == 0) dbias[(size_t)t * H + h] = from_f<T>(s);
}

__global__ void __launch_bounds__(1024) attn_order_kernel(const __grid_constant__ AttnArgs a, int* keys, int* queries) {
    let_next();
    if (blockIdx.x == 0) {
        if (keys) order_items(a.B * ((a.Lk + kOwn - 1) / kOwn), [&](int i) { return min(item_at<true>(a, nullptr, i).per, kBins - 1); }, keys);
    } else if (queries) {
        order_items(a.B * ((a.Lq + kOwn - 1) / kOwn), [&](int i) { return min(item_at<false>(a, nullptr, i).per, kBins - 1); }, queries);
    }
}

int tiles_of(int L) { return (L + kOwn - 1) / kOwn; }
size_t stats_floats(const AttnArgs& a) { return (size_t)a.B * a.H * tiles_of(a.Lq) * kOwn; }
// CTAs of a head: one for each owned tile, or, where each SM would see four or more of them, its share of the SMs
long long ctas_of(const AttnArgs& a, bool dkv, int sms) {
    const long long items = (long long)a.B * tiles_of(dkv ? a.Lk : a.Lq), heads = dkv ? a.Hkv : a.H;
    if (items * heads < 4LL * sms) return items;
    return std::max<long long>(sms > heads ? sms / heads : 1, (items + kMaxItems - 1) / kMaxItems);
}
size_t part_floats(const AttnArgs& a, int sms) {
    return ((size_t)((a.edges.n + 1) << a.edges.two) * a.H * ctas_of(a, false, sms) + 3) & ~(size_t)3;
}
size_t top_floats(const AttnArgs& a) { return ((size_t)2 * a.B * a.Hkv + 3) & ~(size_t)3; }
// ints of its items' order, where lengths differ and CTAs take several
size_t order_ints(const AttnArgs& a, bool dkv, int sms) {
    const long long items = (long long)a.B * tiles_of(dkv ? a.Lk : a.Lq);
    return (a.lengths || a.causal) && ctas_of(a, dkv, sms) < items && items <= kMaxOrder ? (size_t)(items + 3) & ~(size_t)3 : 0;
}

template <class T, int DP, bool BIAS>
int launch_passes(const Args& g, const Maps& own, const Maps& str, cudaStream_t st) {
    static DeviceSetup setup;
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    int rc = device_setup(setup, dev, [] {
        return (int)cudaFuncSetAttribute(attn_bwd_kernel<T, DP, BIAS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes<DP, BIAS>(kMaxReach));
    }, &sms);
    if (rc) return rc;
    const long long ctas = (long long)g.ctas_k * g.a.Hkv + (long long)g.ctas_q * g.a.H;
    if (ctas > INT_MAX) return D2P_ERR_TOO_LARGE;
    return launch_early(true, attn_bwd_kernel<T, DP, BIAS>, dim3((unsigned)ctas), kThreads, smem_bytes<DP, BIAS>(BIAS ? reach_of(g.a.edges) : 0), st, own,
                        str, g);
}

template <class T>
int run(const AttnArgs& a, int dtype, const void* out, const void* rest, const float* lse, const void* grad, void* dq, void* dk, void* dv,
        void* dbias, void* ws, int sms, cudaStream_t st) {
    const int Lp = tiles_of(a.Lq) * kOwn;
    float* const lp = (float*)ws;
    float* const dp = lp + stats_floats(a);
    float* const bp = a.bias ? dp + stats_floats(a) : nullptr;
    float* const part = dp + (a.bias ? 2 : 1) * stats_floats(a);
    float* const top = part + (dbias ? part_floats(a, sms) : 0);
    int* const order = (int*)(top + top_floats(a));
    const size_t ok = order_ints(a, true, sms), oq = order_ints(a, false, sms);
    int* const order_k = ok ? order : nullptr;
    int* const order_q = oq ? order + ok : nullptr;
    int rc = 0;
    if (std::is_same<T, __half>::value && a.B) {
        if ((rc = (int)cudaMemsetAsync(top, 0, top_floats(a) * sizeof(float), st))) return rc;
        if (a.Lk) {
            const dim3 grid((unsigned)std::min(std::max(8LL * sms / ((long long)a.B * a.Hkv), 1LL), (a.Lk + 31LL) / 32), a.Hkv, a.B);
            if (a.D <= 64) attn_v_top_kernel<8><<<grid, 256, 0, st>>>(a, (unsigned*)top + (size_t)a.B * a.Hkv);
            else attn_v_top_kernel<16><<<grid, 256, 0, st>>>(a, (unsigned*)top + (size_t)a.B * a.Hkv);
            if ((rc = (int)cudaGetLastError())) return rc;
        }
    }
    if (ok || oq) {
        attn_order_kernel<<<2, 1024, 0, st>>>(a, order_k, order_q);
        if ((rc = (int)cudaGetLastError())) return rc;
    }
    if (a.B && a.Lq) {
        const dim3 grid(Lp / kStatRows, (a.H + kStatHeads - 1) / kStatHeads, a.B);
        // (beside the order: what it reads was there before that launch)
        rc = launch_early(ok || oq, a.D <= 64 ? attn_stats_kernel<T, 8> : attn_stats_kernel<T, 16>, grid, 256, 0, st, a, (const T*)out, (const T*)rest,
                          lse, (const T*)grad, Lp, lp, dp, bp, (unsigned*)top);
        if (rc) return rc;
    }
    if (a.B && (a.Lq || a.Lk)) {
        // maps of the rows there are; an axis without rows is never read
        const long long gs[3] = {(long long)a.Lq * a.H * a.D, (long long)a.H * a.D, a.D};
        Maps own = {}, str = {};
        bool fine = true;
        for (int w = 0; w < 2; ++w) {
            Maps& m = w ? str : own;
            const int rows = w ? kStep : kOwn;
            if (a.Lq)
                fine = fine && rows_map(&m.q, dtype, a.q, a.B, a.Lq, a.H, a.D, a.qs, rows) && rows_map(&m.grad, dtype, grad, a.B, a.Lq, a.H, a.D, gs, rows);
            if (a.Lk)
                fine = fine && rows_map(&m.k, dtype, a.k, a.B, a.Lk, a.Hkv, a.D, a.ks, rows) && rows_map(&m.v, dtype, a.v, a.B, a.Lk, a.Hkv, a.D, a.vs, rows);
        }
        if (!fine) return D2P_ERR_INVALID_ARGUMENT;
        const long long nk = a.Lk ? ctas_of(a, true, sms) : 0, nq = a.Lq ? ctas_of(a, false, sms) : 0;
        if (nk > INT_MAX || nq > INT_MAX) return D2P_ERR_TOO_LARGE;
        const Args g = {a, lp, dp, bp, Lp, dv, dk, dq, dbias ? part : nullptr, top, top + (size_t)a.B * a.Hkv, order_k, order_q, (int)nk, (int)nq};
        if (a.D <= 64) rc = a.bias ? launch_passes<T, 64, true>(g, own, str, st) : launch_passes<T, 64, false>(g, own, str, st);
        else rc = a.bias ? launch_passes<T, 128, true>(g, own, str, st) : launch_passes<T, 128, false>(g, own, str, st);
        if (rc) return rc;
    }
    if (dbias) {
        const int nb = (a.edges.n + 1) << a.edges.two, n = a.B * tiles_of(a.Lq) ? (int)ctas_of(a, false, sms) : 0;
        if (a.bias_f32)
            attn_dbias_kernel<float><<<(nb * a.H + 3) / 4, 128, 0, st>>>(part, nb, a.H, n, (float*)dbias);
        else
            attn_dbias_kernel<T><<<(nb * a.H + 3) / 4, 128, 0, st>>>(part, nb, a.H, n, (T*)dbias);
        rc = (int)cudaGetLastError();
    }
    return rc;
}

}  // namespace bwd

int attn_backward_gave_up(unsigned long long* n) { return (int)cudaMemcpyFromSymbol(n, g_gave_up, sizeof(*n)); }

size_t attn_backward_bytes(const AttnArgs& a, bool dbias) {
    int sms = 0;
    if (attn_sms(&sms)) return (size_t)-1;
    return ((a.bias ? 3 : 2) * bwd::stats_floats(a) + (dbias ? bwd::part_floats(a, sms) : 0) + bwd::top_floats(a) + bwd::order_ints(a, true, sms) +
            bwd::order_ints(a, false, sms)) * sizeof(float);
}
int attn_backward_tiles(const AttnArgs& a, int dtype, const void* out, const void* rest, const float* lse, const void* grad, void* dq,
                        void* dk, void* dv, void* dbias, void* ws, cudaStream_t st) {
    int sms = 0;
    const int rc = attn_sms(&sms);
    if (rc) return rc;
    return dtype == D2P_DTYPE_BF16 ? bwd::run<__nv_bfloat16>(a, dtype, out, rest, lse, grad, dq, dk, dv, dbias, ws, sms, st)
                                   : bwd::run<__half>(a, dtype, out, rest, lse, grad, dq, dk, dv, dbias, ws, sms, st);
}

}  // namespace enc
}  // namespace d2pb
