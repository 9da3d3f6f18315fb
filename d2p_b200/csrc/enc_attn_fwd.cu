// enc_attn_fwd.cu -- attention forward on the fifth-generation tensor cores.
//
// A CTA takes 128 query rows of a head and runs over the keys in tiles of 128 (64
// for heads above 64).  S = Q K^T (tcgen05, both operands in shared memory,
// K-major) lands in TMEM; a warpgroup reads it, one row a thread, adds the bias, and takes the
// softmax in base 2 with a running reference m: p = 2^(s - m), l = sum p.  P goes
// back to TMEM in 16 bits and is operand A of O += P V (V from shared memory,
// contraction down its rows).  m is raised, and O and l rescaled, only when a
// row's maximum passes it by more than kSlack, which after the first tiles is
// rare.  In the last tile the rows of V past the keys are zeroed in shared
// memory, since 0 x NaN would reach the sums.
//
// Setting up a CTA, its first copies and its last product cost about 5 us beside
// 1.7 us a tile, so where there are many row tiles a CTA stays and takes one
// after the other of its head: the copies and scores of the next begin while this
// one's results leave, and the bias by position is laid out once.
//
// P in 16 bits is the tensor cores' operand, of V's own type: an entry is off by as
// much as one of V is; l sums what it was rounded from, in fp32.
//
// Measured: 4 x 4096, 8 heads of 128: 259 us, 1060 TFLOP/s (two thirds of what a
// large library product reaches).  No pipe is full there: the products' unit is
// busy 64 % of the time and its tensor pipe 50 (S takes both operands from shared
// memory), the exponentials' pipe 50.  8 x 4096, 8 heads of 64: 404 us, 680
// TFLOP/s, with the bias 447: the softmax warps' own chain of waits (a quarter of
// the exponentials moved to the fp32 pipes gained 5 % without the bias, nothing
// with it).  256 x 512, 8 heads of 64: 229 us, with the bias 281: an item's end
// costs as much as one more tile.
#include <algorithm>
#include <type_traits>

#include "enc_tc.cuh"

namespace d2pb {
namespace enc {

namespace fwd {

constexpr int kThreads = 256;   // a softmax warpgroup; the warps of S, of O, of the copies and of the empty row tiles
constexpr int kRows = 128;
constexpr int kColumns = 256;   // TMEM of a CTA; two CTAs a SM
constexpr int kChunk = kRows * 128;
constexpr int kMaxItems = 128;  // row tiles a CTA takes at most
// registers: a softmax thread holds a row's 128 scores.  The two warpgroups' shares must fit what the CTA is launched with
constexpr int kRegs = 128, kRegsSoftmax = 208, kRegsOther = 48;
static_assert(kRegsSoftmax + kRegsOther <= 2 * kRegs, "register split");

// Heads of up to 64: S 128 columns, O 64, P 64 of its own, so that the next S is formed while this one's exponentials
// are taken.  Above, O takes 128: two buffers of 64 keys' S, each overwritten by its own P, do the same (tiles of 128 keys
// with one buffer: 2015 clocks a tile and SM where the products need 1024).  REST: P in twice 16 bits, the second half
// behind the first in the buffer, for an O as exact as fp32 sums give it, and what rounding O took kept: for the
// gradient of the bias, whose sums cancel
template <int DP, bool REST>
struct Shape {
    static constexpr bool kApart = DP == 64 && !REST;
    static constexpr int kKeys = kApart ? 128 : 64, kBuffers = kApart ? 1 : 2;
    static constexpr int kColO = 128, kColP = kApart ? 192 : 0;
    static constexpr int kChunks = DP / 64;
    static constexpr int kTile = kChunks * kChunk;                                // Q
    static constexpr int kChunkKV = kKeys * 128, kTileKV = kChunks * kChunkKV;    // a K or V tile
    static constexpr int kStages = 2;                                             // K and V tiles in flight
    static constexpr int kBars = 5 + 3 * kBuffers + 4 * kStages;
    static constexpr size_t kTiles = kTile + 2 * (size_t)kStages * kTileKV;
    static constexpr size_t smem(int lut) { return 1024 + kTiles + kBars * 8 + 48 + kMaxItems * 20 + (size_t)lut * 4; }
};

// one row tile of a problem: its rows and the key tiles that any of them meets
struct Item {
    int b, q0, lq, lk, off, tiles;
};
template <int KEYS>
__device__ __forceinline__ Item item_at(const AttnArgs& a, const int* order, int index, int row_tiles) {
    Item w;
    if (order) index = order[index];
    // causal: the rows with the most keys first, over all problems
    const int t = a.causal ? row_tiles - 1 - index / a.B : index % row_tiles;
    w.b = a.causal ? index % a.B : index / row_tiles;
    w.q0 = t * kRows;
    problem_lengths(a, w.b, &w.lq, &w.lk);
    w.off = a.causal ? w.lk - w.lq : 0;
    const int last = min(w.q0 + kRows, w.lq) - 1;   // the tile's last live row
    const int keys = w.q0 < w.lq ? (a.causal ? min(w.lk, last + w.off + 1) : w.lk) : 0;
    w.tiles = keys > 0 ? (keys + KEYS - 1) / KEYS : 0;
    return w;
}
// KEEP: what rounding O took is kept, for the gradients.  SPLIT: the keys split over blockIdx.z, the sums for the join (a form
// of its own: as branches these cost heads of 128 4 %)
template <class T, int DP, bool BIAS, bool REST, bool KEEP, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 2)
    attn_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                    const __grid_constant__ CUtensorMap tmV, const __grid_constant__ AttnArgs a, T* __restrict__ out,
                    float* __restrict__ lse, T* __restrict__ rest, const int* __restrict__ order, const __grid_constant__ Parts part) {
    using Sh = Shape<DP, REST>;
    constexpr int NST = Sh::kStages, NB = Sh::kBuffers, KT = Sh::kKeys;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int h = blockIdx.x, row_tiles = (a.Lq + kRows - 1) / kRows, items = a.B * row_tiles;
    const int count = item_count(items, blockIdx.y, gridDim.y);   // of this CTA

    extern __shared__ uint8_t raw[];
    const uint32_t r0 = smem_addr(raw), base = (r0 + 1023u) & ~1023u;
    uint8_t* const gbase = raw + (base - r0);
    const uint32_t sQ = base, sK = base + Sh::kTile, sV = sK + NST * Sh::kTileKV;
    uint64_t* const bars = reinterpret_cast<uint64_t*>(gbase + Sh::kTiles);
    // Q there, Q free; S read (S and P apart); of a buffer S there, P there, its product done; K, V there, free
    const uint32_t barQ = smem_addr(bars), barQE = barQ + 8, barR = barQ + 16, barS = barQ + 24,
                   barP = barS + 8 * NB, barPE = barP + 8 * NB, barK = barPE + 8 * NB, barV = barK + 8 * NST,
                   barKE = barV + 8 * NST, barVE = barKE + 8 * NST, barD = barVE + 8 * NST;   // (D: the products' end, after a wait that gave up)
    uint8_t* const after_bars = gbase + (Sh::kTiles + Sh::kBars * 8 + 15) / 16 * 16;
    const Dead dead = {reinterpret_cast<volatile int*>(after_bars), a.polls};
    uint32_t* const slot = reinterpret_cast<uint32_t*>(after_bars) + 1;
    int* const from = reinterpret_cast<int*>(after_bars) + 2;                // this split's first key tile
    int* const asked = reinterpret_cast<int*>(after_bars) + 4;               // copies issued: Q, K, V
    int4* const entry = reinterpret_cast<int4*>(after_bars + 32);            // b, q0, lq, lk of an item
    int* const tiles = reinterpret_cast<int*>(entry + kMaxItems);            // and the key tiles that its rows meet
    float* const lut = reinterpret_cast<float*>(tiles + kMaxItems);
    const int reach = BIAS ? reach_of(a.edges) : 0;

    const int kh = h / (a.H / a.Hkv);
    auto load = [&](uint32_t dst, const CUtensorMap* tm, int row, int head, int b, uint32_t bar, int chunk) {
        bar_expect(bar, Sh::kChunks * chunk);
#pragma unroll
        for (int c = 0; c < Sh::kChunks; ++c) tma_load(dst + c * chunk, tm, 64 * c, row, head, b, bar);
    };
    // this split's part of an item's key tiles: the first, how many (a CTA of a split takes one item)
    auto share = [&](int n) {
        if (!SPLIT) return make_int2(0, n);
        const int per = (n + part.splits - 1) / part.splits, t = min(n, (int)blockIdx.z * per);
        return make_int2(t, min(per, n - t));
    };
    bool large = false;   // whether rows of this head have bases
    if (warp == 5) {
        if (lane == 0) {
            bar_init(barQ, 1), bar_init(barQE, 1), bar_init(barR, 4), bar_init(barD, 1), bar_init(barD + 8, 1);
            for (int s = 0; s < NB; ++s) bar_init(barS + 8 * s, 1), bar_init(barP + 8 * s, 4), bar_init(barPE + 8 * s, 1);
            for (int s = 0; s < NST; ++s)
                bar_init(barK + 8 * s, 1), bar_init(barV + 8 * s, 1), bar_init(barKE + 8 * s, 1), bar_init(barVE + 8 * s, 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            fence_async_smem();
            *dead.flag = 0;
            wait_ahead();   // (the items' order)
            const Item w = item_at<KT>(a, order, item_index(0, blockIdx.y, gridDim.y), row_tiles);   // the first item's Q and first tile before the CTA meets
            const int2 r = share(w.tiles);
            if (SPLIT) *from = r.x;
            if (r.y) {
                load(sQ, &tmQ, w.q0, h, w.b, barQ, kChunk);
                load(sK, &tmK, r.x * KT, kh, w.b, barK, Sh::kChunkKV);
                load(sV, &tmV, r.x * KT, kh, w.b, barV, Sh::kChunkKV);
            }
        }
        __syncwarp();
    } else if (warp == 4) {
        tmem_alloc(smem_addr(slot), kColumns);
    } else {
        if (BIAS) large = fill_lut<T>(lut, a, h, reach, warp < 4 ? warp : warp - 2, 6);
        wait_ahead();
        for (int e = warp < 4 ? tid : tid - 64; e < count; e += 192) {
            const Item w = item_at<KT>(a, order, item_index(e, blockIdx.y, gridDim.y), row_tiles);
            entry[e] = make_int4(w.b, w.q0, w.lq, w.lk);
            tiles[e] = share(w.tiles).y;
        }
    }
    tc_fence_before();
    large = __syncthreads_or(large);
    tc_fence_after();
    const uint32_t tmem = *slot, tO = tmem + Sh::kColO;

    if (warp >= 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    if (warp == 6) {   // items no row of which has a key
        for (int e = 0; e < count; ++e) {
            if (tiles[e]) continue;
            const int4 w = entry[e];
            const int rows = min(kRows, a.Lq - w.y), units = a.D / 8;
            if (SPLIT) {
                for (int x = lane; x < rows; x += 32) part.ml[part.set(a, w.x, h, blockIdx.z, w.y + x)] = make_float2(-INFINITY, 0.f);
                continue;
            }
            for (int x = lane; x < rows * units; x += 32) {
                const size_t at = (((size_t)w.x * a.Lq + w.y + x / units) * a.H + h) * a.D + (x % units) * 8;
                *reinterpret_cast<uint4*>(out + at) = make_uint4(0, 0, 0, 0);
                if (KEEP) *reinterpret_cast<uint4*>(rest + at) = make_uint4(0, 0, 0, 0);
            }
            if (lse)
                for (int x = lane; x < rows; x += 32) lse[((size_t)w.x * a.H + h) * a.Lq + w.y + x] = INFINITY;
        }
    } else if (warp == 5) {   // copies
        if (lane == 0) {
            bool ok = true;
            const int j0 = SPLIT ? *from : 0;
            int t = 0, q = 0, asked_k = 0, asked_v = 0;   // tiles and items asked for
            for (int i = 0; ok && i < count; ++i) {
                const int n = tiles[i];
                if (n == 0) continue;
                const int4 e = entry[i];
                if (q > 0 && !(ok = bar_wait(barQE, (q - 1) & 1, dead))) break;
                if (i > 0) load(sQ, &tmQ, e.y, h, e.x, barQ, kChunk);   // (the first one's is under way)
                ++q;
                for (int j = 0; j < n; ++j, ++t) {
                    const int s = t % NST;
                    if (t >= NST && !(ok = bar_wait(barKE + 8 * s, (t / NST - 1) & 1, dead))) break;
                    if (i + j > 0) load(sK + s * Sh::kTileKV, &tmK, (j0 + j) * KT, kh, e.x, barK + 8 * s, Sh::kChunkKV);
                    asked_k = t + 1;
                    if (t >= NST && !(ok = bar_wait(barVE + 8 * s, (t / NST - 1) & 1, dead))) break;
                    if (i + j > 0) load(sV + s * Sh::kTileKV, &tmV, (j0 + j) * KT, kh, e.x, barV + 8 * s, Sh::kChunkKV);
                    asked_v = t + 1;
                }
            }
            asked[0] = q, asked[1] = asked_k, asked[2] = asked_v;
        }
        __syncwarp();
    } else {
        // Products: one warp forms S and one O, so that neither's waits and issues stand before the other's.  A whole warp
        // runs this, its operands' words in uniform registers; one lane issues.  Steps past the head's size are left out
        const bool lead = elect_one();
        const uint32_t uS = uniform(tmem), uO = uS + Sh::kColO, uP = uS + Sh::kColP;
        const int steps = (a.D + 15) / 16;
        bool ok = true;
        int t = 0, q = 0;   // tiles and items begun
        if (warp == 4) {
            constexpr uint32_t idS = mma_desc<T>(128, KT, false);
            const uint32_t dQ = desc_along(sQ);
            for (int e = 0; ok && e < count; ++e) {
                const int n = (int)uniform(tiles[e]);
                if (n == 0) continue;
                if (!(ok = bar_wait_warp(barQ, q++ & 1, dead))) break;
                for (int j = 0; j < n; ++j, ++t) {
                    const int s = t % NST, buf = t % NB;
                    if (!(ok = bar_wait_warp(barK + 8 * s, (t / NST) & 1, dead))) break;
                    // S's columns are free once the one before is in registers, or its P has been multiplied
                    if (Sh::kApart && t > 0 && !(ok = bar_wait_warp(barR, (t - 1) & 1, dead))) break;
                    if (!Sh::kApart && t >= NB && !(ok = bar_wait_warp(barPE + 8 * buf, (t / NB - 1) & 1, dead))) break;
                    tc_fence_after();
                    const uint32_t dK = desc_along(sK + s * Sh::kTileKV), d = uS + buf * KT;
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k)
                        if (lead && k < steps)
                            mma_ss(d, dQ + ((k / 4) * kChunk + (k % 4) * 32) / 16, dK + ((k / 4) * Sh::kChunkKV + (k % 4) * 32) / 16, idS, k != 0);
                    if (lead) tc_commit(barS + 8 * buf), tc_commit(barKE + 8 * s);
                }
                if (lead) tc_commit(barQE);
            }
        } else if (warp == 7) {
            const uint32_t idO = mma_desc<T>(128, 16 * steps, true);
            for (int e = 0; ok && e < count; ++e) {
                const int n = (int)uniform(tiles[e]), lk = (int)uniform(entry[e].w) - (SPLIT ? (int)uniform(*from) * KT : 0);
                if (n == 0) continue;
                for (int j = 0; j < n; ++j, ++t) {
                    const int s = t % NST, buf = t % NB, ks = lk - j * KT <= KT / 2 ? KT / 32 : KT / 16;   // steps with keys
                    if (!(ok = bar_wait_warp(barV + 8 * s, (t / NST) & 1, dead) && bar_wait_warp(barP + 8 * buf, (t / NB) & 1, dead))) break;
                    tc_fence_after();
                    const uint32_t dV = desc_down(sV + s * Sh::kTileKV, Sh::kChunkKV), p = uP + buf * KT;
#pragma unroll
                    for (int k = 0; k < KT / 16; ++k)
                        if (lead && k < ks) mma_ts(uO, p + 8 * k, dV + k * (2048 / 16), idO, (j | k) != 0);
                    if (REST) {
#pragma unroll
                        for (int k = 0; k < KT / 16; ++k)
                            if (lead && k < ks) mma_ts(uO, p + KT / 2 + 8 * k, dV + k * (2048 / 16), idO, true);
                    }
                    if (lead) tc_commit(barPE + 8 * buf), tc_commit(barVE + 8 * s);
                }
            }
        }
        __syncwarp();
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
        const uint32_t trow = (uint32_t)(32 * warp) << 16;
        const float c = a.scale * kLog2e;
        bool ok = true;
        int tt = 0;   // tiles so far
        const int j0 = SPLIT ? __shfl_sync(0xffffffffu, *from, 0) : 0;
        float before = 0.f, after = 0.f;   // the bias past the last edge on either side
        if (BIAS) before = lut[0], after = lut[lut_entries(reach) - 1];
        // An item's rows are finished behind the next one's first maximum, which covers the wait for its last product: O /
        // l, a row a thread, whole 32-byte sectors
        // tile t's product done, by its buffer's barrier: of that one the phase before is always over (S t was formed after
        // it), while a barrier for all products could be two phases behind, which its parity does not tell
        auto product = [&](int t) { return bar_wait_warp(barPE + 8 * (t % NB), (t / NB) & 1, dead); };
        int kept = -1, item = 0;   // the item that waits for it, and the one begun
        float kept_m = 0.f, kept_l = 0.f;
        auto finish = [&]() {
            if (!(ok = product(tt - 1))) return;
            tc_fence_after();
            const int4 w = entry[kept];   // b, q0, lq, lk
            const int i = w.y + tid;
            const bool some = i < w.z && (kept_l > 0.f || kept_l != kept_l);
            if (SPLIT) {   // sums as they are, for the join
                const size_t set = part.set(a, w.x, h, blockIdx.z, min(i, a.Lq - 1));
#pragma unroll 1
                for (int x = 0; x < a.D; x += 16) {
                    uint32_t o[16];
                    tmem_ld16(tO + trow + x, o);
                    tmem_wait_ld();
                    tmem_tie16(o);
                    if (i < a.Lq) {
#pragma unroll
                        for (int y = 0; y < 16; y += 4)
                            if (x + y < a.D) *reinterpret_cast<uint4*>(part.o + set * a.D + x + y) = make_uint4(o[y], o[y + 1], o[y + 2], o[y + 3]);
                    }
                }
                if (i < a.Lq) part.ml[set] = some ? make_float2(kept_m, kept_l) : make_float2(-INFINITY, 0.f);
                tc_fence_before();
                kept = -1;
                return;
            }
            const float s = some ? 1.f / kept_l : 0.f;
            const bool whole = a.D % 16 == 0 && (((uintptr_t)out | (uintptr_t)rest) & 31) == 0;
            const size_t at = (((size_t)w.x * a.Lq + i) * a.H + h) * a.D;
#pragma unroll 1
            for (int x = 0; x < a.D; x += 16) {
                uint32_t o[16];
                tmem_ld16(tO + trow + x, o);
                tmem_wait_ld();
                tmem_tie16(o);
                if (i < a.Lq) {
                    uint32_t p[8], q[8];
#pragma unroll
                    for (int z = 0; z < 8; ++z) {
                        const float u0 = __uint_as_float(o[2 * z]) * s, u1 = __uint_as_float(o[2 * z + 1]) * s;
                        p[z] = s == 0.f ? 0u : pack2<T>(u0, u1);   // a dead row is zero whatever it held
                        q[z] = KEEP && s != 0.f ? rest2<T>(u0, u1, p[z]) : 0u;
                    }
                    store16(out + at + x, p, a.D - x, whole);
                    if (KEEP) store16(rest + at + x, q, a.D - x, whole);
                }
            }
            if (lse && i < a.Lq)
                lse[((size_t)w.x * a.H + h) * a.Lq + i] = some ? kept_m - Softmax<T>::kShift + log2f(kept_l) : INFINITY;
            tc_fence_before();   // the next item's first product overwrites O after this warp's first P of it
            kept = -1;
        };
        // LARGE: rows have bases.  A loop of its own (in the same one the others took a tenth longer)
        auto items = [&](auto large_c) {
        constexpr bool LARGE = decltype(large_c)::value;
        for (; item < count; ++item) {
            const int4 en = entry[item];
            // (from one lane for all, so that the branches on them are known to be the warp's)
            const int lku = __shfl_sync(0xffffffffu, en.w, 0), offu = __shfl_sync(0xffffffffu, a.causal ? en.w - en.z : 0, 0);
            const Item w = {en.x, __shfl_sync(0xffffffffu, en.y, 0), en.z, lku, offu, __shfl_sync(0xffffffffu, tiles[item], 0)};
            if (w.tiles == 0) continue;
            const int pos = w.q0 + tid + w.off, lk = w.lk;
            float rb = 0.f, rc = c;   // this row's base, what multiplies its scores
            if (LARGE && w.q0 + tid < w.lq) {
                rb = base_of(row_top<T>(a, h, pos, a.causal ? min(lk, pos + 1) : lk));
                rc = score_factor(rb, c);
            }
            float m = -INFINITY, l = 0.f;
            for (int j = 0; j < w.tiles && ok; ++j, ++tt) {
                const int k0 = (j0 + j) * KT, buf = tt % NB;
                const uint32_t tS = tmem + trow + buf * KT, tP = tmem + trow + Sh::kColP + buf * KT;
                if (!(ok = bar_wait_warp(barS + 8 * buf, (tt / NB) & 1, dead))) break;
                tc_fence_after();
                constexpr int kBlocks = KT / 32;
                const bool half = lk - k0 <= KT / 2;   // no key in the tile's second half: left out, here and in the product
                uint32_t v[KT];
#pragma unroll
                for (int x = 0; x < kBlocks; ++x) tmem_ld32(tS + 32 * x, v + 32 * x);
                tmem_wait_ld();
#pragma unroll
                for (int x = 0; x < kBlocks; ++x) tmem_tie32(v + 32 * x);
                if (Sh::kApart) {
                    tc_fence_before();
                    bar_arrive_warp(barR);
                }
                float* const t = reinterpret_cast<float*>(v);
                // a block's scores in base 2 are mul t + add: with the bias past the last edge (one value) or without any
                // they stay as they are until the exponential; near the diagonal the bias is added here
                float mul[kBlocks], add[kBlocks];
#pragma unroll
                for (int x = 0; x < kBlocks; ++x) mul[x] = c, add[x] = 0.f;
                if (BIAS) {
                    const float* const lp = lut_row(lut, reach, k0 - pos + reach + kPad);
                    // (from one lane for all, so that the branches are known to be the warp's)
                    const int dmin = __shfl_sync(0xffffffffu, k0 - (w.q0 + 32 * warp + 31 + w.off), 0);   // of the warp's 32 rows and the first 32 keys
#pragma unroll
                    for (int x = 0; x < kBlocks; ++x) {
                        if (2 * x >= kBlocks && half) break;
                        const int lo = dmin + 32 * x;
                        add[x] = (lo >= reach ? after : before) - rb;
                        const bool near = lo < reach && lo + 62 > -reach;
                        if (LARGE && near) {   // (the scores themselves, so that their maximum is one of them and no exponent is above 0)
#pragma unroll
                            for (int y = 32 * x; y < 32 * x + 32; ++y) t[y] = fmaf(t[y], rc, lp[y] - rb);
                        } else if (LARGE) {
#pragma unroll
                            for (int y = 32 * x; y < 32 * x + 32; ++y) t[y] = fmaf(t[y], rc, add[x]);
                        } else if (near) {
#pragma unroll
                            for (int y = 32 * x; y < 32 * x + 32; y += 4) {
                                const float4 e = *reinterpret_cast<const float4*>(lp + y);
                                fma2(Two(t[y], t[y + 1]), Two(c, c), Two(e.x, e.y)).get(t + y, t + y + 1);
                                fma2(Two(t[y + 2], t[y + 3]), Two(c, c), Two(e.z, e.w)).get(t + y + 2, t + y + 3);
                            }
                        }
                        if (LARGE || near) mul[x] = 1.f, add[x] = 0.f;
                    }
                }
                if (k0 + KT > lk || (a.causal && k0 + KT - 1 > w.q0 + w.off)) {
                    const int lim = (a.causal ? min(lk - 1, pos) : lk - 1) - k0;
#pragma unroll
                    for (int x = 0; x < KT; ++x) t[x] = x <= lim ? t[x] : -INFINITY;
                }
                float top = -INFINITY;
#pragma unroll
                for (int x = 0; x < kBlocks; ++x) {
                    if (2 * x >= kBlocks && half) break;
                    float mx = fmaxf(t[32 * x], t[32 * x + 1]), my = fmaxf(t[32 * x + 2], t[32 * x + 3]);
#pragma unroll
                    for (int y = 32 * x + 4; y < 32 * x + 32; y += 4)
                        mx = fmaxf(mx, fmaxf(t[y], t[y + 1])), my = fmaxf(my, fmaxf(t[y + 2], t[y + 3]));
                    top = fmaxf(top, BIAS ? fmaf(fmaxf(mx, my), mul[x], add[x]) : fmaxf(mx, my));
                }
                if (!BIAS) top *= c;
                float f = 1.f;
                const bool raise = top > m + Softmax<T>::kSlack || (m == -INFINITY && top > -INFINITY);
                if (raise) {
                    f = m == -INFINITY ? 0.f : ex2(m - top);
                    m = top;
                    l *= f;
                }
                const bool rescale = __any_sync(0xffffffffu, raise) && j > 0;
                if (kept >= 0) finish();   // (the item before)
                if (!ok) break;
                // the product before reads P's columns and adds to O
                if (j > 0 && (Sh::kApart || rescale)) {
                    if (!(ok = product(tt - 1))) break;
                    tc_fence_after();
                }
                if (rescale) {   // O's rows of this warp
#pragma unroll 1
                    for (int x = 0; x < a.D; x += 32) {
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
                Two sum[2] = {Two(0.f, 0.f), Two(0.f, 0.f)};
#pragma unroll
                for (int x = 0; x < KT; x += 32) {
                    if (2 * x >= KT && half) break;
                    uint32_t p[16], p2[16];
                    const Two u(mul[x / 32], mul[x / 32]), v0(add[x / 32] - ref, add[x / 32] - ref);
#pragma unroll
                    for (int y = 0; y < 32; y += 2) {
                        float e0, e1;
                        fma2(Two(t[x + y], t[x + y + 1]), u, v0).get(&e0, &e1);
                        e0 = ex2(e0), e1 = ex2(e1);
                        sum[(y / 2) & 1] = add2(sum[(y / 2) & 1], Two(e0, e1));
                        p[y / 2] = pack2<T>(e0, e1);
                        if (REST) p2[y / 2] = rest2<T>(e0, e1, p[y / 2]);
                    }
                    tmem_st16(tP + x / 2, p);
                    if (REST) tmem_st16(tP + KT / 2 + x / 2, p2);
                }
                {
                    float s0, s1;
                    add2(sum[0], sum[1]).get(&s0, &s1);
                    l += s0 + s1;
                }
                const int live = lk - k0;
                if (live < KT) {   // the keys' last tile: rows of V past them to zero
                    if (!(ok = bar_wait_warp(barV + 8 * (tt % NST), (tt / NST) & 1, dead))) break;
                    const int units = (KT - live) * 8;
                    for (int e = tid; e < units * Sh::kChunks; e += 128)
                        *reinterpret_cast<uint4*>(gbase + (sV - base) + (tt % NST) * Sh::kTileKV + (e / units) * Sh::kChunkKV + live * 128 +
                                                  (e % units) * 16) = make_uint4(0, 0, 0, 0);
                    fence_async_smem();
                }
                tmem_wait_st();
                tc_fence_before();
                bar_arrive_warp(barP + 8 * buf);
            }
            if (!ok) break;
            kept = item, kept_m = m, kept_l = l;
        }
        };
        if (!BIAS || __builtin_expect(!large, 1)) items(std::false_type{});
        else items(std::integral_constant<bool, BIAS>{});
        if (ok && kept >= 0) finish();
        if (!ok) {   // a wait gave up: NaN in this warp's rows of the items from there on
            for (int e = kept >= 0 ? kept : item; e < count; ++e) {
                const int4 w = entry[e];
                const int i = w.y + tid;
                if (tiles[e] == 0 || i >= a.Lq) continue;
                if (SPLIT) {
                    part.ml[part.set(a, w.x, h, blockIdx.z, i)] = make_float2(0.f, NAN);
                    continue;
                }
                const size_t at = (((size_t)w.x * a.Lq + i) * a.H + h) * a.D;
                for (int x = 0; x < a.D; ++x) {
                    out[at + x] = from_f<T>(NAN);
                    if (KEEP) rest[at + x] = from_f<T>(NAN);
                }
                if (lse) lse[((size_t)w.x * a.H + h) * a.Lq + i] = NAN;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (*dead.flag) {   // a wait gave up: what is in flight ends (bounded) before the CTA does
        if (warp < 4) tmem_wait_st();
        if (warp == 4 || warp == 7) tc_drain(barD + (warp == 7 ? 8 : 0));
        if (warp == 5 && lane == 0) {
            int none = 0;
            const Dead end = {&none, kWaitLimit};
            if (asked[0]) bar_wait(barQ, (asked[0] - 1) & 1, end);
            for (int x = max(asked[1] - NST, 0); x < asked[1]; ++x) bar_wait(barK + 8 * (x % NST), (x / NST) & 1, end);
            for (int x = max(asked[2] - NST, 0); x < asked[2]; ++x) bar_wait(barV + 8 * (x % NST), (x / NST) & 1, end);
            atomicAdd(&g_gave_up, 1ull);
        }
        __syncthreads();
    }
    if (warp == 4) tmem_free(tmem, kColumns);
}

__global__ void __launch_bounds__(1024) attn_order_kernel(const __grid_constant__ AttnArgs a, int* __restrict__ order) {
    let_next();
    const int row_tiles = (a.Lq + kRows - 1) / kRows;
    order_items(a.B * row_tiles, [&](int i) { return min(item_at<128>(a, nullptr, i, row_tiles).tiles, kBins - 1); }, order);
}

// a CTA for each item, or, where each place on the device (two CTAs an SM) would see four or more of them, a CTA for
// each place, which takes its share: 256 x 512, 8 heads of 64 when this was chosen: 243 us against 277
long long stays(const AttnArgs& a, int sms) {
    const long long items = (long long)a.B * ((a.Lq + kRows - 1) / kRows), places = 2LL * sms;
    if (items * a.H < 4 * places) return 0;
    return std::max<long long>(places > a.H ? places / a.H : 1, (items + kMaxItems - 1) / kMaxItems);
}
// splits of the keys where the row tiles leave half the places free or more, each at least 256 keys.  Below 1024 the
// join costs what they save (2 x 512 x 512, 8 heads: 12.8 us whole, 15.9 split); 11 x 17 x 3766, 2 heads of 80: 54 us
// whole, 14.6 split; 3 x 689 x 3951, 4 heads of 80: 57 and 31
int splits_of(const AttnArgs& a, int sms) {
    const long long ctas = (long long)a.B * ((a.Lq + kRows - 1) / kRows) * a.H, places = 2LL * sms;
    return 2 * ctas > places || a.Lk < 1024 ? 1 : (int)std::min<long long>(std::min<long long>(places / ctas, a.Lk / 256), kMaxParts);
}
// whether its items are put in order first (a launch of 5 us): lengths differ, and the shares with them.  256 ragged problems
// of up to 512 with the bias: 174 us with the order, 180 without it when this was chosen
bool ordered(const AttnArgs& a, int sms) {
    return (a.lengths || a.causal) && stays(a, sms) && (long long)a.B * ((a.Lq + kRows - 1) / kRows) <= kMaxOrder;
}

template <class T, int DP, bool BIAS, bool REST, bool KEEP, bool SPLIT>
int launch(const AttnArgs& a, int dtype, void* out, float* lse, void* rest, void* ws, cudaStream_t st) {
    using Sh = Shape<DP, REST>;
    static DeviceSetup setup;
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    int rc = device_setup(setup, dev, [] {
        cudaFuncAttributes at;   // the register split above counts on the launch's share
        cudaError_t e = cudaFuncGetAttributes(&at, attn_fwd_kernel<T, DP, BIAS, REST, KEEP, SPLIT>);
        if (e == cudaSuccess && at.numRegs < (kRegsSoftmax + kRegsOther + 1) / 2) e = cudaErrorLaunchOutOfResources;
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(attn_fwd_kernel<T, DP, BIAS, REST, KEEP, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     (int)Sh::smem(lut_size(kMaxReach)));
        return (int)e;
    }, &sms);
    if (rc) return rc;
    CUtensorMap q, k, v;
    if (!rows_map(&q, dtype, a.q, a.B, a.Lq, a.H, a.D, a.qs, kRows)) return D2P_ERR_INVALID_ARGUMENT;
    if (a.Lk == 0) k = v = q;   // never read
    else if (!rows_map(&k, dtype, a.k, a.B, a.Lk, a.Hkv, a.D, a.ks, Sh::kKeys) ||
             !rows_map(&v, dtype, a.v, a.B, a.Lk, a.Hkv, a.D, a.vs, Sh::kKeys))
        return D2P_ERR_INVALID_ARGUMENT;
    const int lut = BIAS ? lut_size(reach_of(a.edges)) : 0;
    // at least a third of the SM's shared memory: no more than two CTAs (2 x 256 TMEM columns), so no allocation waits
    size_t smem = Sh::smem(lut);
    if (smem < 80 * 1024) smem = 80 * 1024;
    const long long stay = stays(a, sms), ctas = stay ? stay : (long long)a.B * ((a.Lq + kRows - 1) / kRows);
    if (ctas > 65535) return D2P_ERR_TOO_LARGE;
    int* order = nullptr;
    if (ordered(a, sms)) {
        order = (int*)ws;
        attn_order_kernel<<<1, 1024, 0, st>>>(a, order);
    }
    const Parts part = parts_at(a, splits_of(a, sms), ws);
    rc = launch_early(order != nullptr, attn_fwd_kernel<T, DP, BIAS, REST, KEEP, SPLIT>, dim3(a.H, (unsigned)ctas, part.splits), kThreads, smem, st, q,
                      k, v, a, (T*)out, lse, (T*)rest, (const int*)order, part);
    return rc || part.splits == 1 ? rc : attn_join(a, dtype, part, out, lse, rest, st);
}

template <class T, int DP, bool BIAS, bool REST, bool KEEP>
int launch(const AttnArgs& a, int dtype, void* out, float* lse, void* rest, void* ws, int sms, cudaStream_t st) {
    return splits_of(a, sms) > 1 ? launch<T, DP, BIAS, REST, false, true>(a, dtype, out, lse, rest, ws, st)
                                 : launch<T, DP, BIAS, REST, KEEP, false>(a, dtype, out, lse, rest, ws, st);
}
template <class T, int DP>
int pick(const AttnArgs& a, int dtype, void* out, float* lse, void* rest, void* ws, int sms, cudaStream_t st) {
    if (a.bias)
        return rest ? launch<T, DP, true, true, true>(a, dtype, out, lse, rest, ws, sms, st) : launch<T, DP, true, false, false>(a, dtype, out, lse, rest, ws, sms, st);
    return rest ? launch<T, DP, false, false, true>(a, dtype, out, lse, rest, ws, sms, st) : launch<T, DP, false, false, false>(a, dtype, out, lse, rest, ws, sms, st);
}
template <class T>
int pick(const AttnArgs& a, int dtype, void* out, float* lse, void* rest, void* ws, int sms, cudaStream_t st) {
    return a.D <= 64 ? pick<T, 64>(a, dtype, out, lse, rest, ws, sms, st) : pick<T, 128>(a, dtype, out, lse, rest, ws, sms, st);
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

size_t attn_forward_bytes(const AttnArgs& a) {
    int sms = 0;
    if (attn_sms(&sms)) return (size_t)-1;
    if (fwd::splits_of(a, sms) > 1) return parts_bytes(a, fwd::splits_of(a, sms));
    return fwd::ordered(a, sms) ? (size_t)a.B * ((a.Lq + fwd::kRows - 1) / fwd::kRows) * sizeof(int) : 0;
}
int attn_forward_tiles(const AttnArgs& a, int dtype, void* out, float* lse, void* rest, void* ws, cudaStream_t st) {
    int sms = 0;
    const int rc = attn_sms(&sms);
    if (rc) return rc;
    return dtype == D2P_DTYPE_BF16 ? fwd::pick<__nv_bfloat16>(a, dtype, out, lse, rest, ws, sms, st) : fwd::pick<__half>(a, dtype, out, lse, rest, ws, sms, st);
}

}  // namespace enc
}  // namespace d2pb
