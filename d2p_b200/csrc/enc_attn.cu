// enc_attn.cu -- attention over a ragged batch with a learned relative position
// bias by buckets, and its gradients: the C entry points and the general
// kernels, one warp per row on the CUDA cores, the head's elements over the
// lanes.
//
// Forward, a warp per query row, keys in order with a running maximum m and sum
// l in base 2: s = scale log2(e) q.k + b; m' = max(m, s); acc = acc 2^(m - m') +
// 2^(s - m') v; out = acc / l and lse = m + log2 l.
// Backward, P = 2^(s - lse): dP = dO.v, delta = dO.O, dS = P (dP - delta);
// a warp per query row sums dq = scale dS k and the buckets' dS, a warp per key
// row sums dk = scale dS q and dv = P dO over its queries and heads.
#include "enc_attn.cuh"

namespace d2pb {
namespace enc {

constexpr int kRowWarps = 4;

template <class T>
struct Row {                       // D / 32 rounded up elements a lane: d = lane + 32 i
    float v[4];
    __device__ void load(const T* p, int D, int lane) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = lane + 32 * i < D ? to_f<T>(p[lane + 32 * i]) : 0.f;
    }
    __device__ float dot(const Row& o) const {
        float s = v[0] * o.v[0];
#pragma unroll
        for (int i = 1; i < 4; ++i) s = fmaf(v[i], o.v[i], s);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        return s;
    }
    __device__ void zero() { v[0] = v[1] = v[2] = v[3] = 0.f; }
    __device__ void add(float w, const Row& o) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = fmaf(w, o.v[i], v[i]);
    }
    __device__ void store(T* p, int D, int lane, float w) const {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (lane + 32 * i < D) p[lane + 32 * i] = from_f<T>(v[i] * w);
    }
};

template <class T>
__device__ const T* row_at(const void* p, const long long* s, int b, int l, int h) {
    return (const T*)p + b * s[0] + l * s[1] + h * s[2];
}

// dq, delta and the row block's bucket sums
template <class T>
__global__ void __launch_bounds__(32 * kRowWarps) attn_dq_rows_kernel(const __grid_constant__ AttnArgs a, const T* out,
                                                                      const float* lse, const T* grad, T* dq,
                                                                      float* delta, float* part) {
    __shared__ float sums[kRowWarps][2 * (kMaxEdges + 1)];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, i = blockIdx.x * kRowWarps + w, h = blockIdx.y, b = blockIdx.z;
    const int nb = n_buckets(a.edges);
    for (int t = lane; t < nb; t += 32) sums[w][t] = 0.f;
    __syncwarp();
    if (i < a.Lq) {
        int lq, lk;
        problem_lengths(a, b, &lq, &lk);
        const int off = a.causal ? lk - lq : 0, kh = h / (a.H / a.Hkv);
        const int end = i < lq ? (a.causal ? min(lk, i + off + 1) : lk) : 0;
        const size_t at = (((size_t)b * a.Lq + i) * a.H + h) * a.D, st = ((size_t)b * a.H + h) * a.Lq + i;
        Row<T> q, g, o, acc, k, v;
        acc.zero();
        float del = 0.f, L = INFINITY;
        if (end > 0) {
            q.load(row_at<T>(a.q, a.qs, b, i, h), a.D, lane);
            g.load(grad + at, a.D, lane);
            o.load(out + at, a.D, lane);
            del = g.dot(o);
            L = lse[st];
        }
        if (lane == 0) delta[st] = del;
        for (int j = 0; j < end; ++j) {
            k.load(row_at<T>(a.k, a.ks, b, j, kh), a.D, lane);
            v.load(row_at<T>(a.v, a.vs, b, j, kh), a.D, lane);
            float s = q.dot(k) * (a.scale * kLog2e);
            const int bu = a.bias ? bucket_of(a.edges, j - i - off) : 0;
            if (a.bias) s += bias_log2<T>(a, bu, h);
            const float ds = exp2f(s - L) * (g.dot(v) - del);
            acc.add(ds, k);
            if (part && lane == 0) sums[w][bu] += ds;
        }
        acc.store(dq + at, a.D, lane, a.scale);
    }
    __syncthreads();
    if (part)
        for (int t = threadIdx.x; t < nb; t += blockDim.x) {
            float s = 0.f;
            for (int k = 0; k < kRowWarps; ++k) s += sums[k][t];
            part[(((size_t)h * nb + t) * a.B + b) * gridDim.x + blockIdx.x] = s;
        }
}

template <class T>
__global__ void __launch_bounds__(32 * kRowWarps) attn_dkv_rows_kernel(const __grid_constant__ AttnArgs a,
                                                                       const float* lse, const float* delta,
                                                                       const T* grad, T* dk, T* dv) {
    const int lane = threadIdx.x & 31, j = blockIdx.x * kRowWarps + (threadIdx.x >> 5), kh = blockIdx.y, b = blockIdx.z;
    if (j >= a.Lk) return;
    int lq, lk;
    problem_lengths(a, b, &lq, &lk);
    const int off = a.causal ? lk - lq : 0, group = a.H / a.Hkv;
    const int from = a.causal ? max(0, j - off) : 0, to = j < lk ? lq : 0;
    Row<T> k, v, q, g, ak, av;
    k.zero(), v.zero(), ak.zero(), av.zero();
    if (from < to) {
        k.load(row_at<T>(a.k, a.ks, b, j, kh), a.D, lane);
        v.load(row_at<T>(a.v, a.vs, b, j, kh), a.D, lane);
    }
    for (int h = kh * group; h < (kh + 1) * group; ++h)
        for (int i = from; i < to; ++i) {
            q.load(row_at<T>(a.q, a.qs, b, i, h), a.D, lane);
            g.load(grad + (((size_t)b * a.Lq + i) * a.H + h) * a.D, a.D, lane);
            float s = q.dot(k) * (a.scale * kLog2e);
            if (a.bias) s += bias_log2<T>(a, bucket_of(a.edges, j - i - off), h);
            const size_t st = ((size_t)b * a.H + h) * a.Lq + i;
            const float p = exp2f(s - lse[st]);
            av.add(p, g);
            ak.add(p * (g.dot(v) - delta[st]), q);
        }
    const size_t at = (((size_t)b * a.Lk + j) * a.Hkv + kh) * a.D;
    ak.store(dk + at, a.D, lane, a.scale);
    av.store(dv + at, a.D, lane, 1.f);
}

// dbias[t][h]: one warp each, the blocks' sums in a fixed order
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

int attn_args(const d2p_attention_args* p, AttnArgs* a) {
    if (!p || p->B < 0 || p->Lq < 0 || p->Lk < 0 || p->H <= 0 || p->Hkv <= 0 || p->H % p->Hkv) return D2P_ERR_INVALID_ARGUMENT;
    if (p->D < 8 || p->D > 128 || p->D % 8) return D2P_ERR_INVALID_ARGUMENT;
    if (p->dtype != D2P_DTYPE_BF16 && p->dtype != D2P_DTYPE_F16) return D2P_ERR_INVALID_ARGUMENT;
    if (!(p->scale > 0.f) || p->scale > 1e30f) return D2P_ERR_INVALID_ARGUMENT;
    if (p->B > 65535 || p->H > 65535 || p->Lq > (1 << 30) || p->Lk > (1 << 30)) return D2P_ERR_TOO_LARGE;
    *a = AttnArgs{};
    if (p->bias) {
        if (p->bias_dtype != D2P_DTYPE_F32 && p->bias_dtype != p->dtype) return D2P_ERR_INVALID_ARGUMENT;
        if (p->n_edges < 0 || p->n_edges > kMaxEdges || (p->n_edges && !p->bucket_edges)) return D2P_ERR_INVALID_ARGUMENT;
        for (int i = 0; i < p->n_edges; ++i) {
            const int e = p->bucket_edges[i];
            if (e < 1 || e > kMaxReach || (i && e < p->bucket_edges[i - 1])) return D2P_ERR_INVALID_ARGUMENT;
            a->edges.e[i] = e;
        }
        a->edges.n = p->n_edges;
        a->edges.two = !p->causal;
    }
    const bool rows = p->B && p->Lq, keys = p->B && p->Lk;
    if ((rows && !p->q) || (keys && (!p->k || !p->v))) return D2P_ERR_INVALID_ARGUMENT;
    if (((uintptr_t)p->q | (uintptr_t)p->k | (uintptr_t)p->v) & 15) return D2P_ERR_INVALID_ARGUMENT;
    a->q = p->q, a->k = p->k, a->v = p->v, a->bias = p->bias, a->bias_f32 = p->bias_dtype == D2P_DTYPE_F32;
    for (int i = 0; i < 3; ++i) {
        if (p->q_stride[i] % 8 || p->k_stride[i] % 8 || p->v_stride[i] % 8) return D2P_ERR_INVALID_ARGUMENT;
        a->qs[i] = p->q_stride[i], a->ks[i] = p->k_stride[i], a->vs[i] = p->v_stride[i];
    }
    a->lengths = p->lengths;
    a->B = p->B, a->Lq = p->Lq, a->Lk = p->Lk, a->H = p->H, a->Hkv = p->Hkv, a->D = p->D, a->causal = p->causal != 0;
    a->scale = p->scale;
    return D2P_OK;
}

int row_blocks(int n) { return (n + kRowWarps - 1) / kRowWarps; }

size_t delta_bytes(const AttnArgs& a) { return (((size_t)a.B * a.H * a.Lq * sizeof(float)) + 255) & ~(size_t)255; }
size_t part_bytes(const AttnArgs& a) {
    return (size_t)((a.edges.n + 1) << a.edges.two) * a.H * a.B * row_blocks(a.Lq) * sizeof(float);
}

template <class T>
int launch_backward(const AttnArgs& a, const void* out, const float* lse, const void* grad, void* dq, void* dk, void* dv,
                    void* dbias, void* ws, cudaStream_t st) {
    float* delta = (float*)ws;
    float* part = dbias ? (float*)((char*)ws + delta_bytes(a)) : nullptr;
    if (a.Lq)
        attn_dq_rows_kernel<T><<<dim3(row_blocks(a.Lq), a.H, a.B), 32 * kRowWarps, 0, st>>>(
            a, (const T*)out, lse, (const T*)grad, (T*)dq, delta, part);
    if (a.Lk)
        attn_dkv_rows_kernel<T><<<dim3(row_blocks(a.Lk), a.Hkv, a.B), 32 * kRowWarps, 0, st>>>(a, lse, delta, (const T*)grad,
                                                                                            (T*)dk, (T*)dv);
    if (dbias) {
        const int nb = (a.edges.n + 1) << a.edges.two, n = a.Lq ? a.B * row_blocks(a.Lq) : 0;
        if (a.bias_f32)
            attn_dbias_kernel<float><<<(nb * a.H + 3) / 4, 128, 0, st>>>(part, nb, a.H, n, (float*)dbias);
        else
            attn_dbias_kernel<T><<<(nb * a.H + 3) / 4, 128, 0, st>>>(part, nb, a.H, n, (T*)dbias);
    }
    return (int)cudaGetLastError();
}

}  // namespace enc
}  // namespace d2pb

using namespace d2pb;

extern "C" {

int d2p_attention_forward(const d2p_attention_args* p, void* out, float* lse, void* stream) {
    enc::AttnArgs a;
    const int rc = enc::attn_args(p, &a);
    if (rc) return rc;
    if (a.B == 0 || a.Lq == 0) return D2P_OK;
    if (!out) return D2P_ERR_INVALID_ARGUMENT;
    if ((uintptr_t)out & 15) return D2P_ERR_INVALID_ARGUMENT;
    return enc::attn_forward_tiles(a, p->dtype, out, lse, (cudaStream_t)stream);
}

size_t d2p_attention_backward_workspace_bytes(const d2p_attention_args* p, int want_dbias) {
    enc::AttnArgs a;
    if (enc::attn_args(p, &a) || (want_dbias && !a.bias)) return (size_t)-1;
    return enc::delta_bytes(a) + (want_dbias ? enc::part_bytes(a) : 0);
}

int d2p_attention_backward(const d2p_attention_args* p, const void* out, const float* lse, const void* grad, void* dq,
                           void* dk, void* dv, void* dbias, void* workspace, size_t workspace_bytes, void* stream) {
    enc::AttnArgs a;
    const int rc = enc::attn_args(p, &a);
    if (rc) return rc;
    if (dbias && !a.bias) return D2P_ERR_INVALID_ARGUMENT;
    if (a.B == 0 && !dbias) return D2P_OK;
    const bool rows = a.B && a.Lq, keys = a.B && a.Lk;
    if ((rows && (!out || !lse || !grad || !dq)) || (keys && (!dk || !dv))) return D2P_ERR_INVALID_ARGUMENT;
    const size_t need = enc::delta_bytes(a) + (dbias ? enc::part_bytes(a) : 0);
    if (need && (!workspace || workspace_bytes < need)) return D2P_ERR_WORKSPACE_TOO_SMALL;
    if (a.B == 0) a.Lq = a.Lk = 0;
    return p->dtype == D2P_DTYPE_BF16
               ? enc::launch_backward<__nv_bfloat16>(a, out, lse, grad, dq, dk, dv, dbias, workspace, (cudaStream_t)stream)
               : enc::launch_backward<__half>(a, out, lse, grad, dq, dk, dv, dbias, workspace, (cudaStream_t)stream);
}

}  // extern "C"
