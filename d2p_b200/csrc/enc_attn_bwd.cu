// enc_attn_bwd.cu -- attention's gradients on the fifth-generation tensor cores,
// the probabilities recomputed from the forward's lse:
//   P = 2^(s - lse),  dP = dO V^T,  dS = P (dP - delta),  delta = rowsum(dO O),
//   dV = P^T dO,  dK = scale dS^T Q,  dQ = scale dS K,  dbias = buckets' sums of dS.
//
// Two passes of one kernel, each a CTA per 128 rows that it owns, so that every
// sum stays in the CTA's accumulators and no atomics are needed: the key pass
// (DKV) owns 128 keys and streams 64 queries at a time of every head that shares
// them, the query pass owns 128 queries and streams 64 keys.  With X1, X2 the
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
// The query pass also sums dS by relative position.  Along a diagonal of a
// warp's 32 x 32 block the sum moves one lane per column (one shuffle each), the
// 63 sums are scanned, and each lane takes its buckets as differences of the
// scan: registers only, in a fixed order.
#include <type_traits>

#include "enc_tc.cuh"

namespace d2pb {
namespace enc {

namespace bwd {

constexpr int kWork = 512;              // four warpgroups: two for a tile, half of its columns each
constexpr int kThreads = kWork + 64;    // and the products' warp and the copies' warp
constexpr int kOwn = 128, kStep = 64;
constexpr int kColumns = 512;   // TMEM: buffers of 64 columns of S and 64 of dP, then the accumulators
constexpr int kChunkX = kOwn * 128, kChunkY = kStep * 128;
constexpr int kBuckets = 2 * (kMaxEdges + 1);

template <int DP, bool DKV>
__host__ __device__ constexpr int buffers() { return DKV && DP == 128 ? 2 : 3; }

template <int DP, bool BIAS>
struct Shape {
    static constexpr int kChunks = DP / 64;
    static constexpr int kX = kChunks * kChunkX, kY = kChunks * kChunkY;
    static constexpr int kRowStats = 2 * kStep * 4;               // lse and delta of a streamed tile's queries
    static constexpr int kStage = 2 * kY + 1024;                  // keeps the tiles at 1024-byte boundaries
    static constexpr int kStages = DP == 64 ? 8 : BIAS ? 3 : 4;   // (the bias by position takes up to 35 KB)
    static constexpr int kBars = 2 + 2 * kStages + 6;
    static constexpr size_t fixed() { return 1024 + 2 * (size_t)kX + (size_t)kStages * kStage + kBars * 8 + 16; }
};
// after the tiles: the bias by position, then (query pass) the diagonals' stage of each warp and the buckets' ranges
__host__ __device__ inline size_t extra(bool bias, bool dkv, int reach) {
    if (!bias) return 0;
    return 4 * (size_t)lut_size(reach) + (dkv ? 0 : 4 * (size_t)(16 * 72 + 16 * kBuckets + 2 * kBuckets));
}
// at least 116 KB: one CTA an SM, since it takes the whole TMEM (no allocation waits)
template <int DP, bool BIAS>
size_t smem_bytes(bool dkv, int reach) {
    const size_t n = Shape<DP, BIAS>::fixed() + extra(BIAS, dkv, reach);
    return n < 116 * 1024 ? 116 * 1024 : n;
}

struct Args {
    AttnArgs a;
    const float* lse;      // [B, H, Lp] padded copies: +inf and 0 in dead rows
    const float* delta;
    int Lp;
    void* dx1;             // keys pass: dv; query pass: unused
    void* dx2;             // dk or dq
    float* part;           // query pass: [H][buckets][B][gridDim.x] sums of dS, or null
};

// rows of X past the lengths never reach a sum of another row; rows of Y do (0 x NaN), and are zeroed in shared memory
template <class T, int DP, bool BIAS, bool DKV>
__global__ void __launch_bounds__(kThreads, 1)
    attn_bwd_kernel(const __grid_constant__ CUtensorMap tmX1, const __grid_constant__ CUtensorMap tmX2,
                    const __grid_constant__ CUtensorMap tmY1, const __grid_constant__ CUtensorMap tmY2,
                    const __grid_constant__ CUtensorMap tmD1, const __grid_constant__ CUtensorMap tmD2,
                    const __grid_constant__ Args g) {
    using Sh = Shape<DP, BIAS>;
    constexpr int NST = Sh::kStages, NB = buffers<DP, DKV>();
    const AttnArgs& a = g.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // causal: the first keys and the last queries have the most to do
    const int x0 = (a.causal && !DKV ? gridDim.x - 1 - blockIdx.x : blockIdx.x) * kOwn, hx = blockIdx.y, b = blockIdx.z;
    int lq, lk;
    problem_lengths(a, b, &lq, &lk);
    const int off = a.causal ? lk - lq : 0, group = a.H / a.Hkv;
    const int lx = DKV ? lk : lq, ly = DKV ? lq : lk, Lx = DKV ? a.Lk : a.Lq, heads = DKV ? a.Hkv : a.H;
    // the streamed rows [y0, y1) that any owned row meets, in tiles of kStep
    int y0 = 0, y1 = x0 < lx ? ly : 0;
    if (a.causal) {
        if (DKV) y0 = max(0, x0 - off) / kStep * kStep;
        else y1 = min(y1, min(x0 + kOwn, lq) + off);
    }
    const int per = y1 > y0 ? (y1 - y0 + kStep - 1) / kStep : 0, n = DKV ? per * group : per;
    if (n == 0) {   // nothing meets these rows
        const int rows = min(kOwn, Lx - x0), units = a.D / 8;
        for (int e = tid; e < rows * units; e += kThreads) {
            const size_t at = (((size_t)b * Lx + x0 + e / units) * heads + hx) * a.D + (e % units) * 8;
            *reinterpret_cast<uint4*>((T*)g.dx2 + at) = make_uint4(0, 0, 0, 0);
            if (DKV) *reinterpret_cast<uint4*>((T*)g.dx1 + at) = make_uint4(0, 0, 0, 0);
        }
        if (!DKV && BIAS && g.part) {
            const int nb = n_buckets(a.edges);
            for (int t = tid; t < nb; t += kThreads)
                g.part[(((size_t)hx * nb + t) * a.B + b) * gridDim.x + blockIdx.x] = 0.f;
        }
        return;
    }

    extern __shared__ uint8_t raw[];
    const uint32_t r0 = smem_addr(raw), base = (r0 + 1023u) & ~1023u;
    uint8_t* const gb = raw + (base - r0);
    const uint32_t sX1 = base, sX2 = base + Sh::kX, sY = base + 2 * Sh::kX;
    constexpr size_t kTiles = 2 * (size_t)Sh::kX + (size_t)NST * Sh::kStage;
    uint64_t* const bars = reinterpret_cast<uint64_t*>(gb + kTiles);
    const uint32_t barX = smem_addr(bars), barF = barX + 8, barY = barX + 16, barE = barY + 8 * NST, barS = barE + 8 * NST,
                   barP = barS + 24;
    volatile int* const dead = reinterpret_cast<volatile int*>(bars + Sh::kBars);
    uint32_t* const slot = reinterpret_cast<uint32_t*>(bars + Sh::kBars) + 1;
    float* const lut = reinterpret_cast<float*>(bars + Sh::kBars + 2);
    const int reach = BIAS ? reach_of(a.edges) : 0;
    float* const diag = lut + lut_size(reach);                        // [16][72] a warp's diagonals, scanned in place
    float* const red = diag + 16 * 72;                                // [16][kBuckets]
    int* const range = reinterpret_cast<int*>(red + 16 * kBuckets);   // [kBuckets][2] positions of a bucket
    const bool sums = !DKV && BIAS && g.part;

    auto copy = [&](uint32_t dst, const CUtensorMap* tm, int row, int head, uint32_t bar, int chunk) {
#pragma unroll
        for (int c = 0; c < Sh::kChunks; ++c) tma_load(dst + c * chunk, tm, 64 * c, row, head, b, bar);
    };
    auto stream = [&](int it) {
        const int s = it % NST, head = DKV ? hx * group + it / per : hx / group, row = y0 + (it % per) * kStep;
        const uint32_t dst = sY + s * Sh::kStage, bar = barY + 8 * s;
        bar_expect(bar, 2 * Sh::kY + (DKV ? Sh::kRowStats : 0));
        copy(dst, &tmY1, row, head, bar, kChunkY);
        copy(dst + Sh::kY, &tmY2, row, head, bar, kChunkY);
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
    if (warp == kWork / 32 + 1) {   // barriers, and the first copies before the CTA meets
        if (lane == 0) {
            bar_init(barX, 1), bar_init(barF, 1);
            for (int s = 0; s < NST; ++s) bar_init(barY + 8 * s, 1), bar_init(barE + 8 * s, 1);
            for (int s = 0; s < NB; ++s) bar_init(barS + 8 * s, 1), bar_init(barP + 8 * s, 8);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            fence_async_smem();
            *dead = 0;
            bar_expect(barX, 2 * Sh::kX);
            copy(sX1, &tmX1, x0, hx, barX, kChunkX);
            copy(sX2, &tmX2, x0, hx, barX, kChunkX);
            for (int it = 0; it < NST && it < n; ++it) stream(it);
        }
        __syncwarp();
    } else if (warp == kWork / 32) {
        tmem_alloc(smem_addr(slot), kColumns);
    } else if (BIAS && !DKV) {
        fill_lut<T>(lut, a, hx, reach, warp, kWork / 32);
        if (sums)
            for (int t = tid; t < n_buckets(a.edges); t += kWork) {
                const int2 v = bucket_range(a.edges, t, 1 << 29);
                range[2 * t] = v.x, range[2 * t + 1] = v.y;
            }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *slot, tA1 = tmem + 128 * NB, tA2 = DKV ? tA1 + DP : tA1;

    if (warp == kWork / 32 + 1) {   // copies
        if (lane == 0) {
            bool ok = true;
            int it = min(n, NST);
            for (; it < n; ++it) {
                if (!(ok = bar_wait(barE + 8 * (it % NST), (it / NST - 1) & 1, dead))) break;
                stream(it);
            }
            if (!ok || *dead) {   // what is in flight ends (bounded) before the CTA does
                volatile int none = 0;
                bar_wait(barX, 0, &none);
                for (int t = max(0, it - NST); t < it; ++t) bar_wait(barY + 8 * (t % NST), (t / NST) & 1, &none);
            }
        }
        __syncwarp();
    } else if (warp == kWork / 32) {   // products
        {
            // the whole warp runs this, so that the operands' words stay in uniform registers; one lane issues
            const bool lead = elect_one();
            const int nu = __shfl_sync(0xffffffffu, n, 0);
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0), uA1 = tm + 128 * NB, uA2 = DKV ? uA1 + DP : uA1;
            constexpr uint32_t idS = mma_desc<T>(128, kStep, false), idA = mma_desc<T>(128, DP, true);
            auto scores = [&](int it) {
                const int s = it % NST;
                if (!bar_wait_warp(barY + 8 * s, (it / NST) & 1, dead)) return false;
                tc_fence_after();
                const uint32_t d = tm + (it % NB) * 128, dX = desc_along(sX1), dY = desc_along(sY + s * Sh::kStage);
#pragma unroll
                for (int w = 0; w < 2; ++w)
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k)
                        if (lead) mma_ss(d + 64 * w, dX + (w * Sh::kX + (k / 4) * kChunkX + (k % 4) * 32) / 16,
                               dY + (w * Sh::kY + (k / 4) * kChunkY + (k % 4) * 32) / 16, idS, k != 0);
                if (lead) tc_commit(barS + 8 * (it % NB));
                return true;
            };
            bool ok = bar_wait_warp(barX, 0, dead);
            for (int it = 0; ok && it < NB && it < nu; ++it) ok = scores(it);
            for (int it = 0; ok && it < nu; ++it) {
                const int s = it % NST;
                if (!(ok = bar_wait_warp(barP + 8 * (it % NB), (it / NB) & 1, dead))) break;
                tc_fence_after();
                const uint32_t p = tm + (it % NB) * 128, dY = desc_down(sY + s * Sh::kStage, kChunkY);
                if (DKV) {
#pragma unroll
                    for (int k = 0; k < kStep / 16; ++k)
                        if (lead) mma_ts(uA1, p + 32 * (k / 2) + 8 * (k % 2), dY + (Sh::kY + k * 2048) / 16, idA, (it | k) != 0);
                }
#pragma unroll
                for (int k = 0; k < kStep / 16; ++k)
                    if (lead) mma_ts(uA2, p + 64 + 32 * (k / 2) + 8 * (k % 2), dY + k * (2048 / 16), idA, (it | k) != 0);
                if (lead) tc_commit(barE + 8 * s);
                if (it + NB < nu) ok = scores(it + NB);
            }
            if (lead) tc_commit(barF);
            if (!ok && lead) atomicAdd(&g_gave_up, 1ull);
        }
        __syncwarp();
    } else {   // P and dS of a tile
        const int pair = warp >> 3, half = (warp >> 2) & 1, w4 = warp & 3, r = tid & 127, x = x0 + r;
        const uint32_t trow = (uint32_t)(32 * w4) << 16;
        const float c = a.scale * kLog2e;
        float rl = 0.f, rd = 0.f;
        if (!DKV) {
            const size_t at = ((size_t)b * a.H + hx) * g.Lp + x;   // Lp covers the tile
            rl = g.lse[at], rd = g.delta[at];
        }
        float far0 = 0.f, far1 = 0.f, bsum[kBuckets / 32];
#pragma unroll
        for (int i = 0; i < kBuckets / 32; ++i) bsum[i] = 0.f;
        bool ok = true;
        float* const dw = diag + warp * 72;
        for (int head = 0; head < (DKV ? group : 1); ++head) {
        if (BIAS && DKV) {   // keys pass: the bias of the group's next head, once every warp is past the one before
            asm volatile("bar.sync 1, 512;" ::: "memory");
            fill_lut<T>(lut, a, hx * group + head, reach, warp, kWork / 32);
            asm volatile("bar.sync 1, 512;" ::: "memory");
        }
        for (int step = (pair ^ (head * per)) & 1; step < per; step += 2) {   // this pair's tiles of the head
            const int it = head * per + step, s = it % NST, buf = it % NB, yb = y0 + step * kStep;
            // (after a wait that gave up a warp still meets its partners at the barriers above)
            // (the streamed tile's own barrier: the keys pass reads the row statistics that came with it)
            ok = ok && (!DKV || bar_wait_warp(barY + 8 * s, (it / NST) & 1, dead)) &&
                 bar_wait_warp(barS + 8 * buf, (it / NB) & 1, dead);
            if (!ok) continue;
            tc_fence_after();
            const int col0 = 32 * half, yc = yb + col0;
            const uint32_t tS = tmem + trow + buf * 128, tD = tS + 64;
            const float* const st = reinterpret_cast<const float*>(gb + 2 * Sh::kX + s * Sh::kStage + 2 * Sh::kY) + col0;
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
            float run = 0.f, all = 0.f;   // the diagonals under way; the sum of a block in one bucket
            // (forms without the masks and without the bias by position: a block needs them rarely)
            auto block = [&](auto edge_c, auto near_c) {
                constexpr bool EDGE = decltype(edge_c)::value, NEAR = decltype(near_c)::value;
                // four columns' entries at lp +- y: the keys pass meets them in falling order
                const float* const lp = lut_row(lut, reach, d0 + reach + kPad - (DKV ? 3 : 0));
                const float flat = BIAS && !NEAR ? (lo >= reach ? lut[lut_entries(reach) - 1] : lut[0]) : 0.f;
                uint32_t sv[32], dv[32];
                tmem_ld32(tS + col0, sv);
                tmem_ld32(tD + col0, dv);
                tmem_wait_ld();
                tmem_tie32(sv), tmem_tie32(dv);
#pragma unroll
                for (int y = 0; y < 32; y += 4) {
                    float4 L, E;
                    if (DKV) {
                        L = *reinterpret_cast<const float4*>(st + y);
                        E = *reinterpret_cast<const float4*>(st + kStep + y);
                    } else {
                        L = make_float4(rl, rl, rl, rl), E = make_float4(rd, rd, rd, rd);
                    }
                    const float Lv[4] = {L.x, L.y, L.z, L.w}, Ev[4] = {E.x, E.y, E.z, E.w};
                    float4 e = make_float4(flat, flat, flat, flat);
                    if (BIAS && NEAR) e = *reinterpret_cast<const float4*>(DKV ? lp - y : lp + y);
                    const float Bv[4] = {DKV ? e.w : e.x, DKV ? e.z : e.y, DKV ? e.y : e.z, DKV ? e.x : e.w};
                    float pv[4], gv[4];
#pragma unroll
                    for (int z = 0; z < 4; ++z) {
                        const int col = y + z;
                        const float raw_s = __uint_as_float(sv[col]);
                        const float t = BIAS ? fmaf(raw_s, c, Bv[z]) - Lv[z] : fmaf(raw_s, c, -Lv[z]);
                        pv[z] = ex2(t);
                        gv[z] = pv[z] * (__uint_as_float(dv[col]) - Ev[z]);
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
            if (BIAS && near) {
                if (edge) block(std::true_type{}, std::true_type{});
                else block(std::false_type{}, std::true_type{});
            } else {
                if (edge) block(std::true_type{}, std::false_type{});
                else block(std::false_type{}, std::false_type{});
            }
            const int live = ly - yb;
            if (live < kStep) {   // rows of Y past the length to zero, for the products that sum over them
                uint8_t* const y = gb + 2 * Sh::kX + s * Sh::kStage;
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
            if (sums) {
                if (near) {
                    dw[62 - lane] = run;   // the diagonals still under way; lane 31's is in place
                    __syncwarp();
                    // the 63 sums (and a zero) scanned: lane l takes 2 l and 2 l + 1
                    const float s0 = dw[2 * lane], s1 = s0 + (lane < 31 ? dw[2 * lane + 1] : 0.f);
                    float t = s1;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const float u = __shfl_up_sync(0xffffffffu, t, o);
                        if (lane >= o) t += u;
                    }
                    __syncwarp();
                    dw[2 * lane + 1] = t - s1 + s0, dw[2 * lane + 2] = t;
                    if (lane == 0) dw[0] = 0.f;
                    __syncwarp();
                    // entry e now holds the sum of the diagonals d in [lo, lo + e)
                    const int nb = n_buckets(a.edges);
#pragma unroll
                    for (int i = 0; i < kBuckets / 32; ++i) {
                        const int t2 = lane + 32 * i;
                        if (t2 < nb) {
                            const int e0 = max(range[2 * t2] - lo, 0), e1 = min(range[2 * t2 + 1] - lo + 1, 63);
                            if (e0 < e1) bsum[i] += dw[e1] - dw[e0];
                        }
                    }
                    __syncwarp();
                } else if (lo >= reach) {
                    far1 += all;
                } else {
                    far0 += all;
                }
            }
        }
        }
        ok = ok && bar_wait_warp(barF, 0, dead);
        tc_fence_after();
        // accumulators to the owned tiles' shared memory (their last use is over), swizzled as the copy out reads them:
        // keys pass: half of dV's or dK's columns a warpgroup; query pass: a quarter of dQ's
        const bool row = x < lx;
        const bool first = DKV && pair == 0;
        const float w = !ok ? NAN : (first ? 1.f : a.scale);
        const int f0 = DKV ? half * (DP / 2) : (warp >> 2) * (DP / 4), f1 = f0 + (DKV ? DP / 2 : DP / 4);
        const uint32_t acc = (first ? tA1 : tA2) + trow;
        uint8_t* const stage = gb + (first ? 0 : Sh::kX);
#pragma unroll 1
        for (int f = f0; f < f1; f += 16) {
            uint32_t o[16];
            tmem_ld16(acc + f, o);
            tmem_wait_ld();
            tmem_tie16(o);
            uint8_t* const rp = stage + (f / 64) * kChunkX + r * 128;
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                uint32_t p[4];
#pragma unroll
                for (int z = 0; z < 4; ++z)
                    p[z] = row ? pack2<T>(__uint_as_float(o[8 * y + 2 * z]) * w, __uint_as_float(o[8 * y + 2 * z + 1]) * w) : 0u;
                *reinterpret_cast<uint4*>(rp + ((((f % 64) / 8 + y) ^ (r & 7)) << 4)) = make_uint4(p[0], p[1], p[2], p[3]);
            }
        }
        if (sums) {
            const int nb = n_buckets(a.edges);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                far0 += __shfl_xor_sync(0xffffffffu, far0, o);
                far1 += __shfl_xor_sync(0xffffffffu, far1, o);
            }
#pragma unroll
            for (int i = 0; i < kBuckets / 32; ++i) {
                const int t = lane + 32 * i;
                if (t < nb) red[warp * kBuckets + t] = bsum[i] + (t == a.edges.n ? far0 : 0.f) + (a.edges.two && t == nb - 1 ? far1 : 0.f);
            }
        }
        fence_async_smem();
        asm volatile("bar.sync 1, 512;" ::: "memory");
        if (tid == 0) {
#pragma unroll
            for (int ch = 0; ch < Sh::kChunks; ++ch) {
                if (DKV) tma_store(&tmD1, 64 * ch, x0, hx, b, sX1 + ch * kChunkX);
                tma_store(&tmD2, 64 * ch, x0, hx, b, sX2 + ch * kChunkX);
            }
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        }
        if (sums) {
            const int nb = n_buckets(a.edges);
            for (int t = tid; t < nb; t += kWork) {
                float v = 0.f;
#pragma unroll
                for (int k = 0; k < kWork / 32; ++k) v += red[k * kBuckets + t];
                g.part[(((size_t)hx * nb + t) * a.B + b) * gridDim.x + blockIdx.x] = v;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kWork / 32) tmem_free(tmem, kColumns);
}

// delta = rowsum(dO O) and lse in rows padded to whole tiles: +inf and 0 where no key is met.  16 lanes a row
template <class T>
__global__ void __launch_bounds__(256) attn_stats_kernel(const __grid_constant__ AttnArgs a, const T* __restrict__ out,
                                                         const float* __restrict__ lse, const T* __restrict__ grad, int Lp,
                                                         float* __restrict__ lp, float* __restrict__ dp) {
    const int lane = threadIdx.x & 15, h = blockIdx.y, b = blockIdx.z, i = blockIdx.x * 16 + (threadIdx.x >> 4);
    int lq, lk;
    problem_lengths(a, b, &lq, &lk);
    float d = 0.f;
    if (i < lq && 8 * lane < a.D) {
        const size_t at = (((size_t)b * a.Lq + i) * a.H + h) * a.D + 8 * lane;
        float o[8], g[8];
        load8<T>(out + at, o);
        load8<T>(grad + at, g);
#pragma unroll
        for (int x = 0; x < 8; ++x) d = fmaf(o[x], g[x], d);
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    if (lane == 0) {
        const size_t at = ((size_t)b * a.H + h) * Lp + i;
        dp[at] = d;
        lp[at] = i < lq ? lse[((size_t)b * a.H + h) * a.Lq + i] : INFINITY;
    }
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

int tiles_of(int L) { return (L + kOwn - 1) / kOwn; }
size_t stats_floats(const AttnArgs& a) { return (size_t)a.B * a.H * tiles_of(a.Lq) * kOwn; }
size_t part_floats(const AttnArgs& a) { return (size_t)((a.edges.n + 1) << a.edges.two) * a.H * a.B * tiles_of(a.Lq); }

template <class T, int DP, bool BIAS, bool DKV>
int launch_pass(const Args& g, const CUtensorMap* tm, cudaStream_t st) {
    static DeviceSetup setup;
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    int rc = device_setup(setup, dev, [] {
        return (int)cudaFuncSetAttribute(attn_bwd_kernel<T, DP, BIAS, DKV>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)smem_bytes<DP, BIAS>(DKV, kMaxReach));
    }, &sms);
    if (rc) return rc;
    const int reach = BIAS ? reach_of(g.a.edges) : 0;
    const size_t smem = smem_bytes<DP, BIAS>(DKV, reach);
    const dim3 grid(tiles_of(DKV ? g.a.Lk : g.a.Lq), DKV ? g.a.Hkv : g.a.H, g.a.B);
    attn_bwd_kernel<T, DP, BIAS, DKV><<<grid, kThreads, smem, st>>>(tm[0], tm[1], tm[2], tm[3], tm[4], tm[5], g);
    return (int)cudaGetLastError();
}
template <class T, int DP>
int launch_pass(const Args& g, bool dkv, const CUtensorMap* tm, cudaStream_t st) {
    if (g.a.bias) return dkv ? launch_pass<T, DP, true, true>(g, tm, st) : launch_pass<T, DP, true, false>(g, tm, st);
    return dkv ? launch_pass<T, DP, false, true>(g, tm, st) : launch_pass<T, DP, false, false>(g, tm, st);
}

template <class T>
int run(const AttnArgs& a, int dtype, const void* out, const float* lse, const void* grad, void* dq, void* dk, void* dv,
        void* dbias, void* ws, cudaStream_t st) {
    const int Lp = tiles_of(a.Lq) * kOwn;
    float* const lp = (float*)ws;
    float* const dp = lp + stats_floats(a);
    float* const part = dp + stats_floats(a);
    int rc = 0;
    if (a.B && a.Lq) {
        attn_stats_kernel<T><<<dim3(Lp / 16, a.H, a.B), 256, 0, st>>>(a, (const T*)out, lse, (const T*)grad, Lp, lp, dp);
        if ((rc = (int)cudaGetLastError())) return rc;
    }
    if (a.B && (a.Lq || a.Lk)) {
        // maps of the rows there are; an axis without rows is never read
        const long long gs[3] = {(long long)a.Lq * a.H * a.D, (long long)a.H * a.D, a.D};
        const long long os[3] = {(long long)a.Lk * a.Hkv * a.D, (long long)a.Hkv * a.D, a.D};
        CUtensorMap own[4] = {}, str[4] = {}, res[3] = {};   // q, dO, k, v; dq, dk, dv
        bool ok = true;
        if (a.Lq) {
            for (int w = 0; w < 2; ++w) {
                CUtensorMap* const m = w ? str : own;
                ok = ok && rows_map(m, dtype, a.q, a.B, a.Lq, a.H, a.D, a.qs, w ? kStep : kOwn) &&
                     rows_map(m + 1, dtype, grad, a.B, a.Lq, a.H, a.D, gs, w ? kStep : kOwn);
            }
            ok = ok && rows_map(res, dtype, dq, a.B, a.Lq, a.H, a.D, gs, kOwn);
        }
        if (a.Lk) {
            for (int w = 0; w < 2; ++w) {
                CUtensorMap* const m = w ? str : own;
                ok = ok && rows_map(m + 2, dtype, a.k, a.B, a.Lk, a.Hkv, a.D, a.ks, w ? kStep : kOwn) &&
                     rows_map(m + 3, dtype, a.v, a.B, a.Lk, a.Hkv, a.D, a.vs, w ? kStep : kOwn);
            }
            ok = ok && rows_map(res + 1, dtype, dk, a.B, a.Lk, a.Hkv, a.D, os, kOwn) &&
                 rows_map(res + 2, dtype, dv, a.B, a.Lk, a.Hkv, a.D, os, kOwn);
        }
        if (!ok) return D2P_ERR_INVALID_ARGUMENT;
        Args g = {a, lp, dp, Lp, nullptr, nullptr, nullptr};
        if (a.Lk) {
            g.dx1 = dv, g.dx2 = dk;
            const CUtensorMap tm[6] = {own[2], own[3], str[0], str[1], res[2], res[1]};
            rc = a.D <= 64 ? launch_pass<T, 64>(g, true, tm, st) : launch_pass<T, 128>(g, true, tm, st);
            if (rc) return rc;
        }
        if (a.Lq) {
            g.dx1 = nullptr, g.dx2 = dq, g.part = dbias ? part : nullptr;
            const CUtensorMap tm[6] = {own[0], own[1], str[2], str[3], res[0], res[0]};
            rc = a.D <= 64 ? launch_pass<T, 64>(g, false, tm, st) : launch_pass<T, 128>(g, false, tm, st);
            if (rc) return rc;
        }
    }
    if (dbias) {
        const int nb = (a.edges.n + 1) << a.edges.two, n = a.B * tiles_of(a.Lq);
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
    return (2 * bwd::stats_floats(a) + (dbias ? bwd::part_floats(a) : 0)) * sizeof(float);
}
int attn_backward_tiles(const AttnArgs& a, int dtype, const void* out, const float* lse, const void* grad, void* dq,
                        void* dk, void* dv, void* dbias, void* ws, cudaStream_t st) {
    return dtype == D2P_DTYPE_BF16 ? bwd::run<__nv_bfloat16>(a, dtype, out, lse, grad, dq, dk, dv, dbias, ws, st)
                                   : bwd::run<__half>(a, dtype, out, lse, grad, dq, dk, dv, dbias, ws, st);
}

}  // namespace enc
}  // namespace d2pb
