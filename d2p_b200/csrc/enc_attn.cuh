// enc_attn.cuh -- the arguments of an attention call as the kernels take them,
// and the bucket of a relative position.
#pragma once
#include "enc_common.cuh"

namespace d2pb {
namespace enc {

constexpr int kMaxEdges = 63;
constexpr int kMaxReach = 1024;   // largest bucket edge: past it a side's last bucket is one constant

struct Edges {
    int n;                        // edges of one side; that side has n + 1 buckets
    int two;                      // keys after the query take the second half of the buckets
    int e[kMaxEdges];
};

struct AttnArgs {
    const void *q, *k, *v;
    long long qs[3], ks[3], vs[3];
    const void* bias;
    int bias_f32;
    Edges edges;
    const int* lengths;
    int B, Lq, Lk, H, Hkv, D, causal;
    float scale;                  // of the natural scores
    int polls;                    // of a wait before it gives up
};
constexpr int kWaitLimit = 1 << 21;

__device__ __forceinline__ int n_buckets(const Edges& e) { return (e.n + 1) << e.two; }

// bias of a bucket in base-2 units.  Finite values are held within 1e30 so that
// a row of lowest values stays a row of equal finite scores
template <class T>
__device__ __forceinline__ float bias_log2(const AttnArgs& a, int bucket, int h) {
    const size_t at = (size_t)bucket * a.H + h;
    const float b = a.bias_f32 ? ((const float*)a.bias)[at] : to_f<T>(((const T*)a.bias)[at]);
    return fabsf(b) < INFINITY ? fminf(fmaxf(b, -1e30f), 1e30f) * kLog2e : b;
}

// positions d of bucket t, clipped to +-far
__device__ __forceinline__ int2 bucket_range(const Edges& e, int t, int far) {
    const int side = e.n + 1, u = t < side ? t : t - side;
    const int lo = u ? e.e[u - 1] : 0, hi = u < e.n ? e.e[u] - 1 : far;
    if (t >= side) return make_int2(max(lo, 1), min(hi, far));
    return make_int2(-min(hi, far), !e.two && u == 0 ? far : -lo);
}
// A row's scores are formed in fp32 less its base, the largest bias of its keys where that is kLargeBias or more in base 2
// (else zero): beside a bias of 1e9 the scores, and beside a reference of 1e9 the logarithm of the sum, would be lost, in
// one kernel here and in another there.  Every kernel takes the same base, and lse is less it too
constexpr float kLargeBias = 256.f;
__device__ __forceinline__ bool large_bias(float b) { return fabsf(b) >= kLargeBias && fabsf(b) < INFINITY; }
// of query position `pos` whose keys are those before `keys`
template <class T>
__device__ __forceinline__ float row_top(const AttnArgs& a, int h, int pos, int keys) {
    float top = -INFINITY;
    for (int t = 0; t < n_buckets(a.edges); ++t) {
        const int2 r = bucket_range(a.edges, t, 1 << 30);
        if (r.y >= -pos && r.x < keys - pos) top = fmaxf(top, bias_log2<T>(a, t, h));
    }
    return top;
}
__device__ __forceinline__ float base_of(float top) { return large_bias(top) ? top : 0.f; }
// what multiplies a row's scores: a base of 2^56 and more swallows them (in 64 bits too), which leaves its keys equal (the
// factor leaves a masked -inf what it is)
__device__ __forceinline__ float score_factor(float base, float c) { return fabsf(base) < 72057594037927936.f ? c : 1e-30f; }

__device__ __forceinline__ void problem_lengths(const AttnArgs& a, int b, int* lq, int* lk) {
    *lq = a.Lq, *lk = a.Lk;
    if (a.lengths) {
        *lq = min(max(a.lengths[2 * b], 0), a.Lq);
        *lk = min(max(a.lengths[2 * b + 1], 0), a.Lk);
    }
}

// the softmax's running reference is raised when a row's maximum passes it by
// more than kSlack (2^kSlack stays in range of the 16-bit types)
template <class T>
struct Softmax {   // fp16: probabilities are held 2^8 times as large, so that small ones stay above its subnormals
    static constexpr float kShift = 0.f, kSlack = 8.f, kDown = 1.f;   // kDown: 2^-kShift
};
template <>
struct Softmax<__half> {
    static constexpr float kShift = 8.f, kSlack = 7.f, kDown = 1.f / 256.f;
};

// SMs of the current device
int attn_sms(int* sms);
// checks of the C entry points; fills *a
int attn_args(const d2p_attention_args* p, AttnArgs* a);
// Where rows are few and keys many, the keys are split and the splits' results joined by a second launch.  Of split s,
// row i of head h: sum of p v at o + set D, with set = ((b H + h) splits + s) Lq + i, its reference and sum of p in ml[set]
constexpr int kMaxParts = 64;
struct Parts {
    float* o;
    float2* ml;
    int splits;                   // 1: no splits, results written at once
    __host__ __device__ size_t set(const AttnArgs& a, int b, int h, int s, int i) const {
        return (((size_t)b * a.H + h) * splits + s) * a.Lq + i;
    }
};
inline size_t parts_bytes(const AttnArgs& a, int splits) {   // (rows of o stay at 16-byte boundaries)
    return splits > 1 ? (size_t)a.B * a.H * splits * a.Lq * (a.D * sizeof(float) + sizeof(float2)) : 0;
}
inline Parts parts_at(const AttnArgs& a, int splits, void* ws) {
    Parts p = {(float*)ws, nullptr, splits};
    if (splits > 1) p.ml = (float2*)(p.o + (size_t)a.B * a.H * splits * a.Lq * a.D);
    return p;
}
int attn_join(const AttnArgs& a, int dtype, const Parts& p, void* out, float* lse, void* rest, cudaStream_t st);
// out, and lse and rest (what rounding took from out; null: not wanted) by tiles of 128 query rows (enc_attn_fwd.cu)
int attn_forward_tiles(const AttnArgs& a, int dtype, void* out, float* lse, void* rest, void* ws, cudaStream_t st);
size_t attn_forward_bytes(const AttnArgs& a);
// the same for at most 16 query rows of a key head, split over the keys (enc_attn_token.cu)
int attn_forward_tokens(const AttnArgs& a, int dtype, void* out, float* lse, void* rest, void* ws, cudaStream_t st);
size_t attn_tokens_bytes(const AttnArgs& a);
// the gradients (enc_attn_bwd.cu) and their workspace
size_t attn_backward_bytes(const AttnArgs& a, bool dbias);
int attn_backward_tiles(const AttnArgs& a, int dtype, const void* out, const void* rest, const float* lse, const void* grad, void* dq,
                        void* dk, void* dv, void* dbias, void* ws, cudaStream_t st);
// CTAs of the current device one of whose bounded waits gave up, since the library was loaded
int attn_forward_gave_up(unsigned long long* n);
int attn_backward_gave_up(unsigned long long* n);

}  // namespace enc
}  // namespace d2pb
