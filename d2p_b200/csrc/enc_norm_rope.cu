// enc_norm_rope.cu -- RMS norms of queries and keys for each head with the
// position rotation in the same pass, and its backward pass.
//
// A row x[D] (one token, one head) becomes y = x r w, r = 1 / sqrt(mean x^2 +
// eps); its first R elements are rotated in pairs (d, d + R / 2) by the angle
// of the token's position (cos, sin: [P, R / 2] fp32 tables), the rest pass.
// With g the gradient of the rotated row, u = g rotated back, t = u w:
//   dx = r (t - xh mean(t xh)),  xh = x r,   dw = sum over rows of u xh.
// Both passes move each element once and recompute r.  A thread holds 16 elements of a row as two 8-element units that are
// each other's rotation partners, so the rotation needs no exchange, and D / 16
// threads (rounded up to a power of two) share the row's sums by shuffles.
//
// Measured, 64 x 512 tokens, 8 + 8 heads of 64, bf16: forward 34 us (142 MB: 4.1
// TB/s), backward 56 us (210 MB: 3.7 TB/s) and 4 us for the weights' sums; a
// token of 32 sequences 5 us, latency.  Memory is not full (0.6 of a copy's rate),
// nor are the issue slots (69 and 63 %): too few rows are asked for ahead, and the
// forward reads the token's cosines and sines again for every head.
#include "enc_common.cuh"

namespace d2pb {
namespace enc {

struct NormRopeArgs {
    const void* x[2];            // q, k
    long long xs[2][3];          // element strides of batch, token, head
    const void* g[2];            // backward: gradients of the outputs, [B, L, heads, D]
    const void* w[2];            // [D]
    void* y[2];                  // outputs (forward) or dx (backward), [B, L, heads, D]
    const float* cosv;
    const float* sinv;
    const void* pos;             // [B, L] or [L] int32 / int64, or null (0 .. L - 1)
    int pos64;
    long long pos_bs;            // batch stride of pos (0: shared)
    int P, B, L, heads[2], D, R;
    float eps;
    int span;                    // backward: heads of a token that a group takes together
    float* part;                 // backward: [2][gridDim.x][D] partial sums of dw
};

constexpr int kThreadsNR = 256;

// the two 8-element units of pair p: rotation partners, or two units past the rotated part
__device__ __forceinline__ void units(int p, int R, int* a, int* b) {
    const int h = R >> 4;
    *a = p < h ? 8 * p : R + 16 * (p - h);
    *b = p < h ? 8 * p + (R >> 1) : *a + 8;
}

template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// a row a group of G threads and step
template <class T, class W, int G>
__global__ void __launch_bounds__(kThreadsNR) norm_rope_fwd_kernel(const NormRopeArgs a) {
    constexpr int kRows = kThreadsNR / G;                 // rows a block takes per step
    const int lane = threadIdx.x & (G - 1), grp = threadIdx.x / G;
    const int pairs = a.D >> 4;
    const bool on = lane < pairs;
    int ea, eb;
    units(on ? lane : 0, a.R, &ea, &eb);
    const bool turn = on && lane < (a.R >> 4);
    const float invD = 1.f / (float)a.D;
    const long long tokens = (long long)a.B * a.L;

#pragma unroll 1
    for (int part = 0; part < 2; ++part) {
        const int H = a.heads[part];
        const T* X = (const T*)a.x[part];
        float w[16];
        if (on) {
            load8<W>((const W*)a.w[part] + ea, w);
            load8<W>((const W*)a.w[part] + eb, w + 8);
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = 0.f;
        }
        const long long rows = tokens * H;
        // the loop's bound is the same for a warp's groups: shuffles stay converged
        for (long long r0 = (long long)blockIdx.x * kRows; r0 < rows; r0 += (long long)gridDim.x * kRows) {
            const long long row = r0 + grp;
            const bool live = on && row < rows;
            const long long rr = row < rows ? row : rows - 1;
            long long tok, b;
            if (rows < (1ll << 31)) tok = (unsigned)rr / (unsigned)H, b = (unsigned)tok / (unsigned)a.L;   // (64-bit division is several times as long)
            else tok = rr / H, b = tok / a.L;
            const int h = (int)(rr - tok * H), l = (int)(tok - b * a.L);
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = 0.f;
            if (live) {
                const T* px = X + b * a.xs[part][0] + l * a.xs[part][1] + h * a.xs[part][2];
                load8<T>(px + ea, x);
                load8<T>(px + eb, x + 8);
            }
            float c[8], s[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) c[i] = 1.f, s[i] = 0.f;
            if (turn) {
                long long p = l;
                if (a.pos) {
                    const long long at = b * a.pos_bs + l;
                    p = a.pos64 ? ((const long long*)a.pos)[at] : (long long)((const int*)a.pos)[at];
                    p = p < 0 ? 0 : (p >= a.P ? a.P - 1 : p);   // a position past the table reads its last row
                }
                load8<float>(a.cosv + p * (a.R >> 1) + ea, c);
                load8<float>(a.sinv + p * (a.R >> 1) + ea, s);
            }
            float q = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) q = fmaf(x[i], x[i], q);
            const float r = rsqrtf(group_sum<G>(q) * invD + a.eps);
            float o[16];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float u = x[i] * r * w[i], v = x[8 + i] * r * w[8 + i];
                o[i] = u * c[i] - v * s[i];
                o[8 + i] = v * c[i] + u * s[i];
            }
            if (live) {
                T* py = (T*)a.y[part] + rr * a.D;
                store8<T>(py + ea, o);
                store8<T>(py + eb, o + 8);
            }
        }
    }
}

// a row's two units as they lie in memory
template <class T>
struct Units {
    uint4 v[sizeof(T)];
    __device__ __forceinline__ void load(const T* p, int ea, int eb) {
        constexpr int n = sizeof(T) / 2;
#pragma unroll
        for (int i = 0; i < n; ++i) {
            v[i] = reinterpret_cast<const uint4*>(p + ea)[i];
            v[n + i] = reinterpret_cast<const uint4*>(p + eb)[i];
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T); ++i) v[i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void get(float* f) const {
        const T* h = reinterpret_cast<const T*>(v);
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i] = to_f<T>(h[i]);
    }
};

// A group of G threads takes `span` heads of one token at a time, which share the
// token's cosines and sines (as many bytes as a row of 16 bits itself).  The next
// row is asked for before this one is used, across tokens too.
template <class T, class W, int G>
__global__ void __launch_bounds__(kThreadsNR, sizeof(T) == 4 ? 1 : 2) norm_rope_bwd_kernel(const NormRopeArgs a) {
    constexpr int kGroups = kThreadsNR / G;
    const int lane = threadIdx.x & (G - 1), grp = threadIdx.x / G;
    const int pairs = a.D >> 4;
    const bool on = lane < pairs;
    int ea, eb;
    units(on ? lane : 0, a.R, &ea, &eb);
    const bool turn = on && lane < (a.R >> 4);
    const float invD = 1.f / (float)a.D;
    const long long tokens = (long long)a.B * a.L;
    __shared__ float red[(kThreadsNR / 32) * 256];

#pragma unroll 1
    for (int part = 0; part < 2; ++part) {
        const int H = a.heads[part], span = min(a.span, H), sets = span ? (H + span - 1) / span : 0;
        const long long work = tokens * sets, step = (long long)gridDim.x * kGroups;
        float w[16];
        if (on) {
            load8<W>((const W*)a.w[part] + ea, w);
            load8<W>((const W*)a.w[part] + eb, w + 8);
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = 0.f;
        }
        float dw[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) dw[i] = 0.f;
        if (work > 0) {
            // a unit (set of heads, position, batch) is stepped with carries rather than divided out
            const long long u0 = (long long)blockIdx.x * kGroups + grp, t0 = u0 / sets, dtok = step / sets;
            int set = (int)(u0 - t0 * sets), l = (int)(t0 % a.L);
            long long b = t0 / a.L;
            const int dset = (int)(step - dtok * sets), dl = (int)(dtok % a.L);
            const long long db = dtok / a.L;
            const long long hs = a.xs[part][2];
            const T *px, *pg;   // the row asked for next
            bool live, ahead, there;   // whether this unit, and the one asked for, is one there is; this lane's, and any
            auto seek = [&]() {
                ahead = on && b < a.B;
                const long long tok = b * a.L + l;
                px = (const T*)a.x[part] + b * a.xs[part][0] + l * a.xs[part][1] + set * span * hs;
                pg = (const T*)a.g[part] + (tok * H + set * span) * a.D;
            };
            auto ask = [&](Units<T>& x, Units<T>& g, int h) {   // row h of the token
                if (ahead && h < H) {
                    x.load(px, ea, eb);
                    g.load(pg, ea, eb);
                } else {
                    x.zero();
                    g.zero();
                }
                px += hs;
                pg += a.D;
            };
            auto place = [&]() -> long long {   // the unit's position in the tables
                if (!turn || b >= a.B) return 0;
                if (!a.pos) return l;
                const long long at = b * a.pos_bs + l;
                return a.pos64 ? ((const long long*)a.pos)[at] : (long long)((const int*)a.pos)[at];
            };
            Units<T> xs, gs, nx, ng;
            seek();
            ask(nx, ng, set * span);
            long long at = place();
            // the loops' bounds are the same for a warp's groups: shuffles stay converged
            for (long long base = (long long)blockIdx.x * kGroups; base < work; base += step) {
                float c[8], s[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) c[i] = 1.f, s[i] = 0.f;
                if (turn) {
                    const long long p = at < 0 ? 0 : (at >= a.P ? a.P - 1 : at);   // past the table: its last row
                    load8<float>(a.cosv + p * (a.R >> 1) + ea, c);
                    load8<float>(a.sinv + p * (a.R >> 1) + ea, s);
                }
                const int h0 = set * span;
                T* py = (T*)a.y[part] + ((b * a.L + l) * H + h0) * a.D;
                live = ahead, there = b < a.B;
                for (int k = 0; k < span; ++k, py += a.D) {
                    xs = nx;
                    gs = ng;
                    if (k + 1 < span) {
                        ask(nx, ng, h0 + k + 1);
                    } else {
                        set += dset, l += dl, b += db;
                        if (set >= sets) set -= sets, ++l;
                        if (l >= a.L) l -= a.L, ++b;
                        seek();
                        ask(nx, ng, set * span);
                        at = place();
                    }
                    float x[16], o[16];
                    xs.get(x);
                    float q = 0.f;
#pragma unroll
                    for (int i = 0; i < 16; ++i) q = fmaf(x[i], x[i], q);
                    // (a place without a row adds nothing to dw, with eps = 0 too)
                    const float sq = group_sum<G>(q), r = there && h0 + k < H ? rsqrtf(sq * invD + a.eps) : 0.f;
                    float g[16];
                    gs.get(g);
                    float dot = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float u = g[i] * c[i] + g[8 + i] * s[i], v = g[8 + i] * c[i] - g[i] * s[i];
                        x[i] *= r;
                        x[8 + i] *= r;
                        dw[i] = fmaf(u, x[i], dw[i]);
                        dw[8 + i] = fmaf(v, x[8 + i], dw[8 + i]);
                        o[i] = u * w[i];
                        o[8 + i] = v * w[8 + i];
                        dot = fmaf(o[i], x[i], dot);
                        dot = fmaf(o[8 + i], x[8 + i], dot);
                    }
                    dot = group_sum<G>(dot) * invD;
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] = r * (o[i] - x[i] * dot);
                    if (live && h0 + k < H) {
                        store8<T>(py + ea, o);
                        store8<T>(py + eb, o + 8);
                    }
                }
            }
        }
        {   // the block's dw: groups of a warp by shuffles, warps in order
#pragma unroll
            for (int i = 0; i < 16; ++i) {
#pragma unroll
                for (int o = 16; o >= G; o >>= 1) dw[i] += __shfl_xor_sync(0xffffffffu, dw[i], o);
            }
            const int warp = threadIdx.x >> 5;
            __syncthreads();
            if ((threadIdx.x & 31) < G && on) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    red[warp * 256 + ea + i] = dw[i];
                    red[warp * 256 + eb + i] = dw[8 + i];
                }
            }
            __syncthreads();
            if (threadIdx.x < a.D) {
                float t = 0.f;
                for (int k = 0; k < kThreadsNR / 32; ++k) t += red[k * 256 + threadIdx.x];
                a.part[((size_t)part * gridDim.x + blockIdx.x) * a.D + threadIdx.x] = t;
            }
        }
    }
}

// dw[part][d] = sum of the blocks' partial sums, in a fixed order
template <class W>
__global__ void __launch_bounds__(1024) norm_rope_dw_kernel(const float* __restrict__ part, int blocks, int D, W* dq,
                                                            W* dk) {
    __shared__ float red[32][32];
    const int d = blockIdx.x * 32 + (threadIdx.x & 31), k = threadIdx.x >> 5, which = blockIdx.y;
    float t = 0.f;
    if (d < D) {
#pragma unroll 8
        for (int i = k; i < blocks; i += 32) t += part[((size_t)which * blocks + i) * D + d];
    }
    red[k][threadIdx.x & 31] = t;
    __syncthreads();
    if (k == 0 && d < D) {
#pragma unroll
        for (int i = 1; i < 32; ++i) t += red[i][threadIdx.x & 31];
        (which ? dk : dq)[d] = from_f<W>(t);
    }
}

int norm_rope_group(int D) {
    int g = 1;
    while (g < D / 16) g *= 2;
    return g;
}
// backward: two blocks a SM (each leaves a row of partial sums), and as many heads of a token at a time as leave every
// group eight units
int norm_rope_blocks(const NormRopeArgs& a, int sms, bool bwd) {
    const long long heads = a.heads[0] > a.heads[1] ? a.heads[0] : a.heads[1];
    const long long rows = (long long)a.B * a.L * heads, per = kThreadsNR / norm_rope_group(a.D);
    const long long want = (rows + per - 1) / per, most = (long long)sms * (bwd ? 2 : 16);
    return (int)(want < most ? (want > 0 ? want : 1) : most);
}
int norm_rope_span(const NormRopeArgs& a, int blocks) {
    const int heads = a.heads[0] > a.heads[1] ? a.heads[0] : a.heads[1];
    const long long groups = (long long)blocks * (kThreadsNR / norm_rope_group(a.D)), tokens = (long long)a.B * a.L;
    int span = 1;
    while (2 * span <= heads && tokens * (heads / (2 * span)) >= 8 * groups) span *= 2;
    return span;
}

template <class T, class W, int G>
void launch_group(const NormRopeArgs& a, int blocks, cudaStream_t st) {
    if (a.part) norm_rope_bwd_kernel<T, W, G><<<blocks, kThreadsNR, 0, st>>>(a);
    else norm_rope_fwd_kernel<T, W, G><<<blocks, kThreadsNR, 0, st>>>(a);
}
template <class T, class W>
int launch_norm_rope(const NormRopeArgs& a, int blocks, void* dqw, void* dkw, cudaStream_t st) {
    switch (norm_rope_group(a.D)) {
        case 1: launch_group<T, W, 1>(a, blocks, st); break;
        case 2: launch_group<T, W, 2>(a, blocks, st); break;
        case 4: launch_group<T, W, 4>(a, blocks, st); break;
        case 8: launch_group<T, W, 8>(a, blocks, st); break;
        default: launch_group<T, W, 16>(a, blocks, st); break;
    }
    const int rc = (int)cudaGetLastError();
    if (rc || !a.part) return rc;
    norm_rope_dw_kernel<W><<<dim3((a.D + 31) / 32, 2), 1024, 0, st>>>(a.part, blocks, a.D, (W*)dqw, (W*)dkw);
    return (int)cudaGetLastError();
}
template <class T>
int launch_norm_rope(const NormRopeArgs& a, int blocks, int wdtype, int dtype, void* dqw, void* dkw, cudaStream_t st) {
    if (wdtype == D2P_DTYPE_F32) return launch_norm_rope<T, float>(a, blocks, dqw, dkw, st);
    if (wdtype != dtype) return D2P_ERR_INVALID_ARGUMENT;
    return launch_norm_rope<T, T>(a, blocks, dqw, dkw, st);
}

}  // namespace enc
}  // namespace d2pb

using namespace d2pb;

static int norm_rope_check(const d2p_norm_rope_args* p) {
    if (!p || p->B < 0 || p->L < 0 || p->H < 0 || p->Hkv < 0) return D2P_ERR_INVALID_ARGUMENT;
    if (p->D < 16 || p->D > 256 || p->D % 16 || p->R < 0 || p->R > p->D || p->R % 16) return D2P_ERR_INVALID_ARGUMENT;
    if (p->R > 0 && (!p->cos || !p->sin || p->P <= 0)) return D2P_ERR_INVALID_ARGUMENT;
    if (!p->positions && p->R > 0 && p->L > p->P) return D2P_ERR_INVALID_ARGUMENT;
    if (!(p->eps >= 0.f)) return D2P_ERR_INVALID_ARGUMENT;
    if (((uintptr_t)p->q | (uintptr_t)p->k | (uintptr_t)p->q_weight | (uintptr_t)p->k_weight | (uintptr_t)p->cos | (uintptr_t)p->sin) & 15)
        return D2P_ERR_INVALID_ARGUMENT;
    if ((uintptr_t)p->positions & (p->positions_int64 ? 7 : 3)) return D2P_ERR_INVALID_ARGUMENT;
    const int unit = p->dtype == D2P_DTYPE_F32 ? 4 : 8;
    for (int i = 0; i < 3; ++i)
        if (p->q_stride[i] % unit || p->k_stride[i] % unit) return D2P_ERR_INVALID_ARGUMENT;
    return D2P_OK;
}
static enc::NormRopeArgs norm_rope_args(const d2p_norm_rope_args* p) {
    enc::NormRopeArgs a = {};
    a.x[0] = p->q, a.x[1] = p->k, a.w[0] = p->q_weight, a.w[1] = p->k_weight;
    for (int i = 0; i < 3; ++i) a.xs[0][i] = p->q_stride[i], a.xs[1][i] = p->k_stride[i];
    a.cosv = p->cos, a.sinv = p->sin, a.pos = p->positions, a.pos64 = p->positions_int64, a.pos_bs = p->position_batch_stride;
    a.P = p->P, a.B = p->B, a.L = p->L, a.heads[0] = p->H, a.heads[1] = p->Hkv, a.D = p->D, a.R = p->R, a.eps = p->eps;
    return a;
}
static int norm_rope_sms(int* sms) {
    static DeviceSetup setup;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    return device_setup(setup, dev, [] { return 0; }, sms);
}
static int norm_rope_run(const enc::NormRopeArgs& a, const d2p_norm_rope_args* p, int blocks, void* dqw, void* dkw,
                         cudaStream_t st) {
    switch (p->dtype) {
        case D2P_DTYPE_F32: return enc::launch_norm_rope<float>(a, blocks, p->weight_dtype, p->dtype, dqw, dkw, st);
        case D2P_DTYPE_BF16:
            return enc::launch_norm_rope<__nv_bfloat16>(a, blocks, p->weight_dtype, p->dtype, dqw, dkw, st);
        case D2P_DTYPE_F16: return enc::launch_norm_rope<__half>(a, blocks, p->weight_dtype, p->dtype, dqw, dkw, st);
        default: return D2P_ERR_INVALID_ARGUMENT;
    }
}

extern "C" {

int d2p_norm_rope_forward(const d2p_norm_rope_args* p, void* q_out, void* k_out, void* stream) {
    int rc = norm_rope_check(p);
    if (rc) return rc;
    if (p->B == 0 || p->L == 0 || (p->H == 0 && p->Hkv == 0)) return D2P_OK;
    if ((p->H && (!p->q || !q_out)) || (p->Hkv && (!p->k || !k_out)) || !p->q_weight || !p->k_weight)
        return D2P_ERR_INVALID_ARGUMENT;
    if (((uintptr_t)q_out | (uintptr_t)k_out) & 15) return D2P_ERR_INVALID_ARGUMENT;
    int sms = 0;
    if ((rc = norm_rope_sms(&sms))) return rc;
    enc::NormRopeArgs a = norm_rope_args(p);
    a.y[0] = q_out, a.y[1] = k_out;
    return norm_rope_run(a, p, enc::norm_rope_blocks(a, sms, false), nullptr, nullptr, (cudaStream_t)stream);
}

size_t d2p_norm_rope_workspace_bytes(const d2p_norm_rope_args* p) {
    int sms = 0;
    if (norm_rope_check(p) || norm_rope_sms(&sms)) return (size_t)-1;
    return (size_t)2 * enc::norm_rope_blocks(norm_rope_args(p), sms, true) * p->D * sizeof(float);
}

int d2p_norm_rope_backward(const d2p_norm_rope_args* p, const void* dq_out, const void* dk_out, void* dq, void* dk,
                           void* dq_weight, void* dk_weight, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = norm_rope_check(p);
    if (rc) return rc;
    if (!p->q_weight || !p->k_weight || !dq_weight || !dk_weight || !workspace) return D2P_ERR_INVALID_ARGUMENT;
    if (p->B && p->L && ((p->H && (!p->q || !dq_out || !dq)) || (p->Hkv && (!p->k || !dk_out || !dk))))
        return D2P_ERR_INVALID_ARGUMENT;
    if (((uintptr_t)dq_out | (uintptr_t)dk_out | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)workspace) & 15) return D2P_ERR_INVALID_ARGUMENT;
    int sms = 0;
    if ((rc = norm_rope_sms(&sms))) return rc;
    enc::NormRopeArgs a = norm_rope_args(p);
    const int blocks = enc::norm_rope_blocks(a, sms, true);
    a.span = enc::norm_rope_span(a, blocks);
    if (workspace_bytes < (size_t)2 * blocks * p->D * sizeof(float)) return D2P_ERR_WORKSPACE_TOO_SMALL;
    a.y[0] = dq, a.y[1] = dk, a.g[0] = dq_out, a.g[1] = dk_out, a.part = (float*)workspace;
    return norm_rope_run(a, p, blocks, dq_weight, dk_weight, (cudaStream_t)stream);
}

}  // extern "C"
