// enc_attn.cu -- the C entry points of attention over a ragged batch: checks of
// the arguments, and which kernels take them.
#include "enc_attn.cuh"

namespace d2pb {
namespace enc {

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
    a->scale = p->scale;
    return D2P_OK;
}

}  // namespace enc
}  // namespace d2pb

using namespace d2pb;

extern "C" {

// few query rows of a key head: tiles of 128 rows would be mostly empty, and the keys of one problem stay with one CTA;
// 32 x 16 heads over ragged caches of up to 4096: 119 us by tiles against 72
static bool few_rows(const enc::AttnArgs& a) { return (long long)a.Lq * (a.H / a.Hkv) <= 16; }

size_t d2p_attention_forward_workspace_bytes(const d2p_attention_args* p) {
    enc::AttnArgs a;
    if (enc::attn_args(p, &a)) return (size_t)-1;
    return a.B == 0 || a.Lq == 0 || few_rows(a) ? 0 : enc::attn_forward_bytes(a);
}

int d2p_attention_forward(const d2p_attention_args* p, void* out, float* lse, void* rest, void* workspace, size_t workspace_bytes,
                          void* stream) {
    enc::AttnArgs a;
    const int rc = enc::attn_args(p, &a);
    if (rc) return rc;
    if (a.B == 0 || a.Lq == 0) return D2P_OK;
    if (!out || (((uintptr_t)out | (uintptr_t)rest | (uintptr_t)workspace) & 15) || ((uintptr_t)lse & 3)) return D2P_ERR_INVALID_ARGUMENT;
    if (rest && !a.bias) return D2P_ERR_INVALID_ARGUMENT;
    if (few_rows(a)) return enc::attn_forward_tokens(a, p->dtype, out, lse, rest, (cudaStream_t)stream);
    const size_t need = enc::attn_forward_bytes(a);
    if (need && (!workspace || workspace_bytes < need)) return D2P_ERR_WORKSPACE_TOO_SMALL;
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

int d2p_attention_gave_up(unsigned long long* n) {
    if (!n) return D2P_ERR_INVALID_ARGUMENT;
    unsigned long long f = 0, b = 0;
    int rc = enc::attn_forward_gave_up(&f);
    if (rc == D2P_OK) rc = enc::attn_backward_gave_up(&b);
    if (rc == D2P_OK) *n = f + b;
    return rc;
}

}  // extern "C"
