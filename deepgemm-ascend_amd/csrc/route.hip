// Routing of tokens to experts: scores, selection and weights of a token's row of logits, and the gradient.
//
//   s = softmax(l) or 1 / (1 + exp(-l)), b = s + bias; the groups whose best b sum up highest stay; the topk largest b there.
//   w = scale s[id] / (sum s[id] + 1e-20):
//   d s[id_c] = scale (d_w_c - sum_j d_w_j s[id_j] / S) / S with S the sum and its 1e-20, then through softmax or sigmoid.
//
// LPT lanes hold a token's row, P experts each.  A key carries its expert's index in its low ten bits, so that all keys differ and
// comparing them alone gives the order, equal numbers to the lowest index.  The lanes sort their keys and join lists of the KP largest
// pairwise: max(a[i], b[KP - 1 - i]) of two descending lists are the KP largest of both, in an order that one bitonic merge sorts.
#include "op_launch.hpp"

namespace dg {
namespace {

typedef unsigned int u32;
typedef unsigned long long u64;

constexpr int kThreads = 256;
constexpr int kMaxExperts = 1024;
constexpr int kMaxTopk = 16;
constexpr float kTiny = 1e-20f;

struct RouteParams {
    const void* logits;
    int64_t ld;
    int bf16, softmax;
    int tokens, experts, topk;
    int groups, per_group, keep, group_top;
    u32 per_group_inv;         // ceil(2^21 / per_group): e / per_group = e * inv >> 21 for e < 1024
    int by_logit;              // the order of b is the logits' own
    int renormalize;
    float scale;
    const float* bias;
    int32_t* ids;
    float* weights;
    const float* d_weights;    // gradient
    void* d_logits;
    int64_t d_ld;
    uint32_t* status;
    int vbase;
};

typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short u16x4_any __attribute__((ext_vector_type(4), aligned(2)));

// A lane's expert i: runs of four, so that a token's lanes read side by side.
template <int LPT>
__device__ __forceinline__ int expert_of(int sub, int i) { return (i >> 2) * (4 * LPT) + sub * 4 + (i & 3); }

template <int LPT, int P>
__device__ __forceinline__ void load_row(const RouteParams& p, int64_t t, int sub, float (&l)[P]) {
    const float* const f = reinterpret_cast<const float*>(p.logits) + t * p.ld;
    const uint16_t* const h = reinterpret_cast<const uint16_t*>(p.logits) + t * p.ld;
#pragma unroll
    for (int q = 0; q < P / 4; ++q) {
        const int e = expert_of<LPT>(sub, q * 4);
        if (e + 4 <= p.experts) {
            if (p.bf16) {
                const u16x4_any v = *reinterpret_cast<const u16x4_any*>(h + e);
#pragma unroll
                for (int i = 0; i < 4; ++i) l[q * 4 + i] = bf16_to_f32(v[i]);
            } else {
                const f32x4_any v = *reinterpret_cast<const f32x4_any*>(f + e);
#pragma unroll
                for (int i = 0; i < 4; ++i) l[q * 4 + i] = v[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) l[q * 4 + i] = e + i >= p.experts ? -__builtin_inff() : p.bf16 ? bf16_to_f32(h[e + i]) : f[e + i];
        }
    }
}

__device__ __forceinline__ float logit_at(const RouteParams& p, int64_t t, int e) {
    return p.bf16 ? bf16_to_f32(reinterpret_cast<const uint16_t*>(p.logits)[t * p.ld + e]) : reinterpret_cast<const float*>(p.logits)[t * p.ld + e];
}

// Values of other lanes of a token: within rows of 16 lanes by their exchange (xor 1, xor 2, and the mirrors, which are xor 4 and
// xor 8 for what four and eight lanes share).
template <int M>
__device__ __forceinline__ u32 other(u32 v) {
    if constexpr (M == 1) return (u32)__builtin_amdgcn_mov_dpp((int)v, 0xb1, 0xf, 0xf, true);
    else if constexpr (M == 2) return (u32)__builtin_amdgcn_mov_dpp((int)v, 0x4e, 0xf, 0xf, true);
    else if constexpr (M == 4) return (u32)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xf, 0xf, true);
    else if constexpr (M == 8) return (u32)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xf, 0xf, true);
    else return (u32)__shfl_xor((int)v, M);
}
template <int M>
__device__ __forceinline__ float other(float v) { return __builtin_bit_cast(float, other<M>(__builtin_bit_cast(u32, v))); }
template <int M>
__device__ __forceinline__ double other(double v) {
    const u64 b = __builtin_bit_cast(u64, v);
    return __builtin_bit_cast(double, (u64)other<M>((u32)(b >> 32)) << 32 | other<M>((u32)b));
}

template <int LPT, typename T>
__device__ __forceinline__ T lanes_sum(T v) {
    v += other<1>(v); v += other<2>(v); v += other<4>(v); v += other<8>(v);
    if constexpr (LPT > 16) v += other<16>(v);
    if constexpr (LPT > 32) v += other<32>(v);
    return v;
}
template <int LPT>
__device__ __forceinline__ float lanes_max(float v) {
    v = fmaxf(v, other<1>(v)); v = fmaxf(v, other<2>(v)); v = fmaxf(v, other<4>(v)); v = fmaxf(v, other<8>(v));
    if constexpr (LPT > 16) v = fmaxf(v, other<16>(v));
    if constexpr (LPT > 32) v = fmaxf(v, other<32>(v));
    return v;
}

// ------------------------------------------------------------------------------------------------ lists of the largest keys
template <typename T>
__device__ __forceinline__ void swap_desc(T& a, T& b) {
    const T hi = __builtin_elementwise_max(a, b), lo = __builtin_elementwise_min(a, b);
    a = hi;
    b = lo;
}

// A bitonic list in descending order.
template <int N, typename T>
__device__ __forceinline__ void merge_desc(T (&v)[N]) {
#pragma unroll
    for (int d = N / 2; d > 0; d >>= 1)
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (!(i & d)) swap_desc(v[i], v[i + d]);
}

template <int N, typename T>
__device__ __forceinline__ void sort_desc(T (&v)[N]) {
#pragma unroll
    for (int k = 2; k <= N; k <<= 1)
#pragma unroll
        for (int d = k / 2; d > 0; d >>= 1)
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (!(i & d)) {
                    if (i & k) swap_desc(v[i + d], v[i]);
                    else swap_desc(v[i], v[i + d]);
                }
}

// The KP largest of a (descending) and b (descending) into a.
template <int KP, typename T>
__device__ __forceinline__ void join_desc(T (&a)[KP], const T (&b)[KP]) {
#pragma unroll
    for (int i = 0; i < KP; ++i) a[i] = __builtin_elementwise_max(a[i], b[KP - 1 - i]);
    merge_desc(a);
}

template <int M, int KP, typename T>
__device__ __forceinline__ void join_lanes(T (&a)[KP]) {
    T b[KP];
#pragma unroll
    for (int i = 0; i < KP; ++i) b[i] = other<M>(a[i]);
    join_desc(a, b);
}

// The KP largest keys of a token's lanes, in every one of them.
template <int LPT, int P, int KP, typename T>
__device__ __forceinline__ void largest(const T (&key)[P], T (&top)[KP], T none) {
    constexpr int N = P < KP ? P : KP;
    T part[N];
#pragma unroll
    for (int i = 0; i < N; ++i) part[i] = key[i];
    sort_desc(part);
#pragma unroll
    for (int i = 0; i < KP; ++i) top[i] = i < N ? part[i < N ? i : 0] : none;
    if constexpr (N == KP) {
#pragma unroll
        for (int q = 1; q < P / N; ++q) {
#pragma unroll
            for (int i = 0; i < N; ++i) part[i] = key[q * N + i];
            sort_desc(part);
            join_desc(top, part);
        }
    }
    join_lanes<1>(top); join_lanes<2>(top); join_lanes<4>(top); join_lanes<8>(top);
    if constexpr (LPT > 16) join_lanes<16>(top);
    if constexpr (LPT > 32) join_lanes<32>(top);
}

// A number as a key: its low ten bits give way to the expert's index (the lower, the larger).  Finite numbers here are far from a
// double's largest, where experts that are out, infinity and NaN (the largest) have their places.
constexpr double kOut = -0x1p1023, kInf = 0x1p1022, kNan = 0x1p1023;
__device__ __forceinline__ double key_of(double b, int e) {
    if (b != b) b = kNan;
    else if (b == -__builtin_inf()) b = kOut;
    else if (b == __builtin_inf()) b = kInf;
    const u64 v = __builtin_bit_cast(u64, b);
    return __builtin_bit_cast(double, (v & ~1023ull) | (u32)((int)(v >> 32) < 0 ? e : 1023 - e));
}
__device__ __forceinline__ int expert_of_key(double k) {
    const u64 v = __builtin_bit_cast(u64, k);
    if (k <= kOut) return -1;
    return (int)(v >> 32) < 0 ? (int)(v & 1023) : 1023 - (int)(v & 1023);
}

// s of a token's experts, in 64 bits.
template <int LPT, int P>
__device__ __forceinline__ void scores64(const RouteParams& p, const float (&l)[P], float top, double (&s)[P]) {
    if (p.softmax) {
        double sum = 0;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            s[i] = exp((double)l[i] - (double)top);
            sum += s[i];
        }
        sum = lanes_sum<LPT>(sum);
#pragma unroll
        for (int i = 0; i < P; ++i) s[i] /= sum;
    } else {
#pragma unroll
        for (int i = 0; i < P; ++i) s[i] = 1.0 / (1.0 + exp(-(double)l[i]));
    }
}

template <int LPT, int P, int KP>
__global__ __launch_bounds__(kThreads) void route_kernel(const RouteParams p) {
    // b of the workgroup's tokens, and the scores of their groups (at most one an expert)
    __shared__ double b_of[kThreads * P];
    __shared__ double group_of[kThreads * P];
    const int tid = threadIdx.x, sub = tid % LPT, mine = tid / LPT;
    const int64_t t = (int64_t)(blockIdx.x + p.vbase) * (kThreads / LPT) + mine;
    const int64_t row = t < p.tokens ? t : p.tokens - 1;   // (lanes past the last token keep the others company)
    float l[P];
    load_row<LPT>(p, row, sub, l);
    float top = l[0];
#pragma unroll
    for (int i = 1; i < P; ++i) top = fmaxf(top, l[i]);
    top = lanes_max<LPT>(top);
    top = top == -__builtin_inff() ? 0.f : top;   // (every expert out)

    double b[P];
    if (p.by_logit) {
#pragma unroll
        for (int i = 0; i < P; ++i) b[i] = l[i];
    } else {
        scores64<LPT>(p, l, top, b);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int e = expert_of<LPT>(sub, i);
            if (l[i] == -__builtin_inff()) b[i] = -__builtin_inf();
            else if (p.bias != nullptr) b[i] += (double)p.bias[min(e, p.experts - 1)];
        }
    }
    if (p.groups > 1) {
        double* const rows = b_of + mine * (LPT * P);
        double* const sums = group_of + mine * (LPT * P);
#pragma unroll
        for (int i = 0; i < P; ++i) rows[expert_of<LPT>(sub, i)] = b[i];
        __syncthreads();
        for (int g = sub; g < p.groups; g += LPT) {
            double first = -__builtin_inf(), second = first;
            bool nan = false;
            for (int j = 0; j < p.per_group; ++j) {
                const double v = rows[g * p.per_group + j];
                nan = nan || v != v;
                second = fmax(second, fmin(first, v));
                first = fmax(first, v);
            }
            // (a group of one expert, or with one left, has that one's b; NaN is the largest here too)
            double sum = first;
            if (p.group_top > 1 && second != -__builtin_inf()) sum += second;
            sums[g] = nan || sum != sum ? kNan : sum == __builtin_inf() ? kInf : sum;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int e = expert_of<LPT>(sub, i);
            if (e >= p.experts) continue;
            const int g = (int)((u32)e * p.per_group_inv >> 21);
            const double mine_sum = sums[g];
            int before = 0;
            for (int o = 0; o < p.groups; ++o) before += sums[o] > mine_sum || (sums[o] == mine_sum && o < g);
            if (before >= p.keep) b[i] = -__builtin_inf();
        }
    }
    double list[KP];
#pragma unroll
    for (int i = 0; i < P; ++i) b[i] = key_of(b[i], expert_of<LPT>(sub, i));
    largest<LPT, P, KP>(b, list, kOut * 1.5);

    int id = -1;
#pragma unroll
    for (int c = 0; c < KP; ++c)
        if (sub == c) id = expert_of_key(list[c]);
    if (sub >= p.topk || sub >= KP) id = -1;
    float w = 0.f, sum = 1.f;
    if (p.softmax) {
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < P; ++i) sum += expf(l[i] - top);
        sum = lanes_sum<LPT>(sum);
    }
    if (id >= 0) {
        const float v = logit_at(p, row, id);
        w = p.softmax ? expf(v - top) / sum : 1.f / (1.f + expf(-v));
    }
    if (p.renormalize) w /= lanes_sum<16>(w) + kTiny;   // (the choices lie in a token's first 16 lanes)
    if (t < p.tokens && sub < p.topk) {
        p.ids[t * p.topk + sub] = id;
        p.weights[t * p.topk + sub] = id >= 0 ? w * p.scale : 0.f;
    }
}

template <int LPT, int P>
__global__ __launch_bounds__(kThreads) void route_backward_kernel(const RouteParams p) {
    __shared__ float d_of[kThreads * P];   // the gradients of s
    const int tid = threadIdx.x, sub = tid % LPT, mine = tid / LPT;
    const int64_t t = (int64_t)(blockIdx.x + p.vbase) * (kThreads / LPT) + mine;
    const int64_t row = t < p.tokens ? t : p.tokens - 1;
    float l[P];
    load_row<LPT>(p, row, sub, l);
    float* const d = d_of + mine * (LPT * P);
#pragma unroll
    for (int i = 0; i < P; ++i) d[expert_of<LPT>(sub, i)] = 0.f;

    int id = -1;
    float s = 0.f, dw = 0.f, top = 0.f, sum = 1.f;
    if (p.softmax) {
        top = l[0];
#pragma unroll
        for (int i = 1; i < P; ++i) top = fmaxf(top, l[i]);
        top = lanes_max<LPT>(top);
        top = top == -__builtin_inff() ? 0.f : top;
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            l[i] = expf(l[i] - top);
            sum += l[i];
        }
        sum = lanes_sum<LPT>(sum);
    }
    if (sub < p.topk) {
        id = p.ids[row * p.topk + sub];
        if (id >= p.experts) {
            if (p.status != nullptr) p.status[2] = 1u;
            id = -1;
        }
        if (id >= 0) {
            dw = p.d_weights[row * p.topk + sub];
            const float v = logit_at(p, row, id);
            s = p.softmax ? expf(v - top) / sum : 1.f / (1.f + expf(-v));
        }
    }
    float ds = dw;
    if (p.renormalize) {
        const float total = lanes_sum<16>(s) + kTiny;
        ds = (dw - lanes_sum<16>(dw * s) / total) / total;
    }
    ds = id >= 0 ? ds * p.scale : 0.f;
    const float inner = p.softmax ? __shfl(lanes_sum<16>(ds * s), (tid & 63) / LPT * LPT) : 0.f;
    // an expert that repeats: its choices' sum, by the first of them
    float all = 0.f;
    bool first = true;
    for (int c = 0; c < p.topk; ++c) {
        const int from = (tid & 63) / LPT * LPT + c;
        const int o = __shfl(id, from);
        const float v = __shfl(ds, from);
        if (o == id) {
            all += v;
            first = first && c >= sub;
        }
    }
    __syncthreads();
    if (id >= 0 && first) d[id] = all;
    __syncthreads();
    if (t >= p.tokens) return;
    float* const f = reinterpret_cast<float*>(p.d_logits) + t * p.d_ld;
    uint16_t* const h = reinterpret_cast<uint16_t*>(p.d_logits) + t * p.d_ld;
#pragma unroll
    for (int q = 0; q < P / 4; ++q) {
        const int e = expert_of<LPT>(sub, q * 4);
        float g[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float v = d[e + i], x = l[q * 4 + i];
            if (p.softmax) {
                g[i] = x / sum * (v - inner);
                if (x == 0.f) g[i] = 0.f;   // (out, or too small to count: also where every expert is out)
            } else {
                const float y = expf(-fabsf(x));   // s (1 - s), without a difference
                g[i] = v == 0.f ? 0.f : v * (y / ((1.f + y) * (1.f + y)));
            }
        }
        if (e + 4 <= p.experts) {
            if (p.bf16) {
                typedef u32 u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
                *reinterpret_cast<u32x2_any*>(h + e) = u32x2_any{pack_bf16x2(g[0], g[1]), pack_bf16x2(g[2], g[3])};
            } else {
                *reinterpret_cast<f32x4_any*>(f + e) = f32x4_any{g[0], g[1], g[2], g[3]};
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (e + i < p.experts) {
                    if (p.bf16) h[e + i] = f32_to_bf16_rne(g[i]);
                    else f[e + i] = g[i];
                }
        }
    }
}

typedef void (*RouteKernel)(const RouteParams);

// Lanes to a token and experts to a lane: 16 lanes are a row whose exchanges are single instructions; past 256 experts more lanes.
template <bool BACKWARD, int LPT, int P>
RouteKernel pick_topk(int topk) {
    if constexpr (BACKWARD) return &route_backward_kernel<LPT, P>;
    else return topk <= 4 ? &route_kernel<LPT, P, 4> : topk <= 8 ? &route_kernel<LPT, P, 8> : &route_kernel<LPT, P, 16>;
}

template <bool BACKWARD>
RouteKernel pick(int experts, int topk, int& lanes) {
    lanes = experts <= 256 ? 16 : experts <= 512 ? 32 : 64;
    if (experts <= 64) return pick_topk<BACKWARD, 16, 4>(topk);
    if (experts <= 128) return pick_topk<BACKWARD, 16, 8>(topk);
    if (experts <= 256) return pick_topk<BACKWARD, 16, 16>(topk);
    return experts <= 512 ? pick_topk<BACKWARD, 32, 16>(topk) : pick_topk<BACKWARD, 64, 16>(topk);
}

template <bool BACKWARD>
int route_run(const dg_moe_route_args* a, void* stream) {
    if (a == nullptr) return dg_set_error("dg_moe_route: null args");
    if (a->scores != DG_SCORES_SOFTMAX && a->scores != DG_SCORES_SIGMOID) return dg_set_error("dg_moe_route: unknown scores");
    if (a->dtype != DG_DTYPE_BF16 && a->dtype != DG_DTYPE_F32) return dg_set_error("dg_moe_route: logits are bf16 or fp32");
    if (a->tokens < 0 || a->tokens > kMaxExtent) return dg_set_error("dg_moe_route: at most 2^30 tokens");
    if (a->experts < 1 || a->experts > kMaxExperts) return dg_set_error("dg_moe_route: between 1 and 1024 experts");
    if (a->topk < 0 || a->topk > kMaxTopk || a->topk > a->experts) return dg_set_error("dg_moe_route: topk is at most 16 and at most the experts");
    if (a->logits_ld < a->experts || (BACKWARD && a->d_logits_ld < a->experts)) return dg_set_error("dg_moe_route: leading dimension smaller than the row");
    if (!BACKWARD) {
        if (a->num_groups < 1 || a->experts % a->num_groups != 0) return dg_set_error("dg_moe_route: the groups must divide the experts");
        if (a->topk_groups < 1 || a->topk_groups > a->num_groups) return dg_set_error("dg_moe_route: topk_groups must be between 1 and num_groups");
        if (a->group_top != 1 && a->group_top != 2) return dg_set_error("dg_moe_route: group_top is 1 or 2");
        if (a->topk > a->topk_groups * (a->experts / a->num_groups)) return dg_set_error("dg_moe_route: topk is more than the kept groups' experts");
    }
    if (a->tokens == 0 || (!BACKWARD && a->topk == 0)) return DG_OK;
    if (a->logits == nullptr || (a->topk > 0 && a->ids == nullptr) || (!BACKWARD && a->weights == nullptr) ||
        (BACKWARD && ((a->topk > 0 && a->d_weights == nullptr) || a->d_logits == nullptr)))
        return dg_set_error("dg_moe_route: null tensor");
    const int64_t size = a->dtype == DG_DTYPE_BF16 ? 2 : 4;
    if (!aligned_to(a->logits, size) || !aligned_to(a->d_logits, size) || !aligned_to(a->ids, 4) || !aligned_to(a->weights, 4) ||
        !aligned_to(a->d_weights, 4) || !aligned_to(a->bias, 4))
        return dg_set_error("dg_moe_route: tensors must be aligned");
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    RouteParams p = {};
    p.logits = a->logits;
    p.ld = a->logits_ld;
    p.bf16 = a->dtype == DG_DTYPE_BF16;
    p.softmax = a->scores == DG_SCORES_SOFTMAX;
    p.tokens = a->tokens;
    p.experts = a->experts;
    p.topk = a->topk;
    p.renormalize = a->renormalize;
    p.scale = a->scale;
    p.ids = a->ids;
    if constexpr (BACKWARD) {
        p.d_weights = a->d_weights;
        p.d_logits = a->d_logits;
        p.d_ld = a->d_logits_ld;
        p.status = status_words_for(st);
    } else {
        p.groups = a->topk_groups == a->num_groups ? 1 : a->num_groups;   // (all groups stay: none to choose)
        p.per_group = a->experts / a->num_groups;
        p.per_group_inv = ((1u << 21) + p.per_group - 1) / p.per_group;
        p.keep = a->topk_groups;
        p.group_top = a->group_top;
        p.bias = a->bias;
        p.by_logit = a->bias == nullptr && (p.groups == 1 || a->group_top == 1);
        p.weights = a->weights;
    }
    int lanes = 0;
    const RouteKernel kernel = pick<BACKWARD>(a->experts, a->topk, lanes);
    return launch_op(kernel, ceil_div64(a->tokens, kThreads / lanes), kThreads, p, st, a->num_cus);
}

}  // namespace
}  // namespace dg

extern "C" int dg_moe_route(const dg_moe_route_args* args, void* stream) { return dg::route_run<false>(args, stream); }
extern "C" int dg_moe_route_backward(const dg_moe_route_args* args, void* stream) { return dg::route_run<true>(args, stream); }
