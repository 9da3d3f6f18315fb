// enc_attn.cu -- the C entry points of attention over a ragged batch: checks of
// the arguments, and which kernels take them.
#include <atomic>

#include "enc_attn.cuh"

namespace d2pb {
namespace enc {

static std::atomic<int> wait_polls{kWaitLimit};

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
    if (((uintptr_t)p->lengths & 3) || ((uintptr_t)p->bias & (a->bias_f32 ? 3 : 1))) return D2P_ERR_INVALID_ARGUMENT;
    a->lengths = p->lengths;
    a->B = p->B, a->Lq = p->Lq, a->Lk = p->Lk, a->H = p->H, a->Hkv = p->Hkv, a->D = p->D, a->causal = p->causal != 0;
    a->scale = p->scale, a->polls = wait_polls.load(std::memory_order_relaxed);
    return D2P_OK;
}

int attn_sms(int* sms) {
    static DeviceSetup setup;
    int dev = 0;
    const cudaError_t e = cudaGetDevice(&dev);
    return e != cudaSuccess ? (int)e : device_setup(setup, dev, [] { return 0; }, sms);
}

// The splits' sums in a fixed order, each in the frame of the largest reference: WARPS warps a row, each every WARPS-th
// split, four elements a lane.  Eight where there are many splits, whose loads would follow one another
template <class T, int WARPS>
__global__ void __launch_bounds__(256) attn_join_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ Parts p, T* __restrict__ out,
                                                        float* __restrict__ lse, T* __restrict__ rest) {
    __shared__ float4 accs[WARPS == 1 ? 1 : 8][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, first = WARPS == 1 ? 0 : warp;
    const long long rows = (long long)a.B * a.H * a.Lq, row = WARPS == 1 ? (long long)blockIdx.x * 8 + warp : blockIdx.x;   // ((b, h), i)
    if (row >= rows) return;
    const long long bh = row / a.Lq;
    const int i = (int)(row - bh * a.Lq), b = (int)(bh / a.H), h = (int)(bh - (long long)b * a.H);
    const size_t set = p.set(a, b, h, 0, i);
    float2 ml[kMaxParts / 32];   // of splits lane, lane + 32
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < kMaxParts / 32; ++k) {
        ml[k] = lane + 32 * k < p.splits ? p.ml[set + (size_t)(lane + 32 * k) * a.Lq] : make_float2(-INFINITY, 0.f);
        top = fmaxf(top, ml[k].x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float weight[kMaxParts / 32], part = 0.f;
    bool some_of[kMaxParts / 32];   // a split without a key of the row left its sums unwritten
#pragma unroll
    for (int k = 0; k < kMaxParts / 32; ++k) {
        some_of[k] = !(ml[k].x == -INFINITY && ml[k].y == 0.f);
        weight[k] = ml[k].x == -INFINITY ? 0.f : exp2f(ml[k].x - top);
        part = fmaf(weight[k], ml[k].y, part);
    }
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    const bool on = 4 * lane < a.D;
#pragma unroll 8
    for (int s = first; s < p.splits; s += WARPS) {
        const float f = __shfl_sync(0xffffffffu, s < 32 ? weight[0] : weight[1], s & 31);
        const bool there = __shfl_sync(0xffffffffu, s < 32 ? some_of[0] : some_of[1], s & 31);
        const float4 v = on ? *reinterpret_cast<const float4*>(p.o + (set + (size_t)s * a.Lq) * a.D + 4 * lane) : make_float4(0.f, 0.f, 0.f, 0.f);
        if (there) acc.x = fmaf(f, v.x, acc.x), acc.y = fmaf(f, v.y, acc.y), acc.z = fmaf(f, v.z, acc.z), acc.w = fmaf(f, v.w, acc.w);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
    if (WARPS > 1) {
        accs[warp][lane] = acc;
        __syncthreads();
        if (warp) return;
#pragma unroll
        for (int w = 1; w < WARPS; ++w) {
            const float4 v = accs[w][lane];
            acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
        }
    }
    const bool some = part > 0.f || part != part;
    const float w = some ? 1.f / part : 0.f;
    const size_t at = (((size_t)b * a.Lq + i) * a.H + h) * a.D + 4 * lane;
    const uint2 r = some ? make_uint2(pack2<T>(acc.x * w, acc.y * w), pack2<T>(acc.z * w, acc.w * w)) : make_uint2(0u, 0u);
    if (on) *reinterpret_cast<uint2*>(out + at) = r;
    if (on && rest)
        *reinterpret_cast<uint2*>(rest + at) = some ? make_uint2(rest2<T>(acc.x * w, acc.y * w, r.x), rest2<T>(acc.z * w, acc.w * w, r.y)) : make_uint2(0u, 0u);
    if (lse && lane == 0) lse[row] = some ? top - Softmax<T>::kShift + log2f(part) : INFINITY;
}
template <class T>
static void launch_join(const AttnArgs& a, const Parts& p, void* out, float* lse, void* rest, cudaStream_t st) {
    const long long rows = (long long)a.B * a.H * a.Lq;
    if (p.splits > 8) attn_join_kernel<T, 8><<<(unsigned)rows, 256, 0, st>>>(a, p, (T*)out, lse, (T*)rest);
    else attn_join_kernel<T, 1><<<(unsigned)((rows + 7) / 8), 256, 0, st>>>(a, p, (T*)out, lse, (T*)rest);
}
int attn_join(const AttnArgs& a, int dtype, const Parts& p, void* out, float* lse, void* rest, cudaStream_t st) {
    if (dtype == D2P_DTYPE_BF16) launch_join<__nv_bfloat16>(a, p, out, lse, rest, st);
    else launch_join<__half>(a, p, out, lse, rest, st);
    return (int)cudaGetLastError();
}

}  // namespace enc
}  // namespace d2pb

using namespace d2pb;

extern "C" {

// few query rows of a key head: tiles of 128 rows would be mostly empty, and read the keys once for each query head.  One
// token, 32 x 4096 keys, us by tiles / by tokens: 16/16 heads of 64, ragged, 119 / 74; 16 query heads to a key head of 64 124 /
// 24, of 128 144 / 45; 4 x 16384, 16/1 of 128 83 / 26.  The tokens' operand holds 16 rows: past that tiles it is (17
// heads to one 124, 32 to one 210)
static bool few_rows(const enc::AttnArgs& a) { return (long long)a.Lq * (a.H / a.Hkv) <= 16; }

size_t d2p_attention_forward_workspace_bytes(const d2p_attention_args* p) {
    enc::AttnArgs a;
    if (enc::attn_args(p, &a)) return (size_t)-1;
    return a.B == 0 || a.Lq == 0 ? 0 : few_rows(a) ? enc::attn_tokens_bytes(a) : enc::attn_forward_bytes(a);
}

int d2p_attention_forward(const d2p_attention_args* p, void* out, float* lse, void* rest, void* workspace, size_t workspace_bytes,
                          void* stream) {
    enc::AttnArgs a;
    const int rc = enc::attn_args(p, &a);
    if (rc) return rc;
    if (a.B == 0 || a.Lq == 0) return D2P_OK;
    if (!out || (((uintptr_t)out | (uintptr_t)rest | (uintptr_t)workspace) & 15) || ((uintptr_t)lse & 3)) return D2P_ERR_INVALID_ARGUMENT;
    const size_t need = few_rows(a) ? enc::attn_tokens_bytes(a) : enc::attn_forward_bytes(a);
    if (need && (!workspace || workspace_bytes < need)) return D2P_ERR_WORKSPACE_TOO_SMALL;
    if (few_rows(a)) return enc::attn_forward_tokens(a, p->dtype, out, lse, rest, workspace, (cudaStream_t)stream);
    return enc::attn_forward_tiles(a, p->dtype, out, lse, rest, workspace, (cudaStream_t)stream);
}

size_t d2p_attention_backward_workspace_bytes(const d2p_attention_args* p, int want_dbias) {
    enc::AttnArgs a;
    if (enc::attn_args(p, &a) || (want_dbias && !a.bias)) return (size_t)-1;
    return enc::attn_backward_bytes(a, want_dbias != 0);
}

int d2p_attention_backward(const d2p_attention_args* p, const void* out, const void* rest, const float* lse,
                           const void* grad, void* dq, void* dk, void* dv, void* dbias, void* workspace, size_t workspace_bytes, void* stream) {
    enc::AttnArgs a;
    const int rc = enc::attn_args(p, &a);
    if (rc) return rc;
    if (dbias && !a.bias) return D2P_ERR_INVALID_ARGUMENT;
    const bool rows = a.B && a.Lq, keys = a.B && a.Lk;
    if ((rows && (!out || !lse || !grad || !dq)) || (keys && (!dk || !dv))) return D2P_ERR_INVALID_ARGUMENT;
    if (((uintptr_t)out | (uintptr_t)rest | (uintptr_t)grad | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv | (uintptr_t)workspace) & 15)
        return D2P_ERR_INVALID_ARGUMENT;
    if (((uintptr_t)lse & 3) || ((uintptr_t)dbias & (a.bias_f32 ? 3 : 1))) return D2P_ERR_INVALID_ARGUMENT;
    const size_t need = enc::attn_backward_bytes(a, dbias != nullptr);
    if (need && (!workspace || workspace_bytes < need)) return D2P_ERR_WORKSPACE_TOO_SMALL;
    return enc::attn_backward_tiles(a, p->dtype, out, rest, lse, grad, dq, dk, dv, dbias, workspace, (cudaStream_t)stream);
}

int d2p_attention_wait_limit(int polls) { return enc::wait_polls.exchange(polls < 0 ? enc::kWaitLimit : polls); }

int d2p_attention_gave_up(unsigned long long* n) {
    if (!n) return D2P_ERR_INVALID_ARGUMENT;
    unsigned long long f = 0, b = 0;
    int rc = enc::attn_forward_gave_up(&f);
    if (rc == D2P_OK) rc = enc::attn_backward_gave_up(&b);
    if (rc == D2P_OK) *n = f + b;
    return rc;
}

}  // extern "C"
