// Routing of tokens to experts: scores, selection and weights of a token's row of logits, and the gradient.
//
//   s = softmax(l) or 1 / (1 + exp(-l)), b = s + bias; the groups whose best b sum up highest stay; the topk largest b there.
//   w = scale s[id] / (sum s[id] + 1e-20):
//   d s[id_c] = scale (d_w_c - sum_j d_w_j s[id_j] / S) / S with S the sum and its 1e-20, then through softmax or sigmoid.
//
// LPT lanes hold a token's row, P experts each.  A key is a number whose low bits gave way to its expert's index, so that all keys
// differ and comparing them alone gives the order, equal numbers to the lowest index.  The lanes sort their keys and join lists of the KP
// largest pairwise: max(a[i], b[KP - 1 - i]) of two descending lists are the KP largest of both, in an order that one bitonic merge sorts.
//
// Keys of 32 bits select quickly but not surely: 22 to 26 bits of a score in fp32.  The choice is then checked against the scores
// themselves: every chosen one above the next, and the last above all others, by more than fp32 can be off.  A token that fails
// (about one in a hundred, and rows with infinities or NaN) is done again in 64 bits, whose keys' choice is checked likewise, exactly.
#include "op_launch.hpp"

#include <utility>

namespace dg {
namespace {

typedef unsigned int u32;
typedef unsigned long long u64;

constexpr int kThreads = 256;
constexpr int kMaxExperts = 1024;
constexpr int kMaxTopk = 16;
constexpr int kMaxGroups = 64;
constexpr float kTiny = 1e-20f;

struct RouteParams {
    const void* logits;
    int64_t ld;
    int bf16, softmax;
    int tokens, experts, topk;
    int groups, per_group, keep, group_top;
    u32 per_group_inv;         // ceil(2^21 / per_group): e / per_group = e * inv >> 21 for e < 1024
    int by_logit;              // the order of b is the logits' own
    int exact_keys;            // keys of 32 bits hold all of b
    int group_lanes;           // 1 + log2 of a group's lanes, where these are a power of two, at most 16; 0 otherwise
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

// f of 0 ... N - 1 as constants: the arrays that they index are registers from the start (loops, unrolled later, leave the compiler
// moving an array as a whole: 211 registers, and 36 us in place of 25 for 32768 tokens over 256 experts).
template <int N, typename F>
__device__ __forceinline__ void each(F&& f) {
    [&]<int... I>(std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>()), ...); }(std::make_integer_sequence<int, N>());
}

// A lane's expert i: runs of four, so that a token's lanes read side by side.
template <int LPT>
__device__ __forceinline__ int expert_of(int sub, int i) { return (i >> 2) * (4 * LPT) + sub * 4 + (i & 3); }

template <int LPT, int P>
__device__ __forceinline__ void load_row(const RouteParams& p, int64_t t, int sub, float (&l)[P]) {
    const float* const f = reinterpret_cast<const float*>(p.logits) + t * p.ld;
    const uint16_t* const h = reinterpret_cast<const uint16_t*>(p.logits) + t * p.ld;
    each<P / 4>([&](auto q) {
        const int e = expert_of<LPT>(sub, q * 4);
        u32 v[4];
        if (p.experts == LPT * P || e + 4 <= p.experts) {
            if (p.bf16) {
                const u16x4_any w = *reinterpret_cast<const u16x4_any*>(h + e);
                each<4>([&](auto i) { v[i] = (u32)w[i.value] << 16; });
            } else {
                const f32x4_any w = *reinterpret_cast<const f32x4_any*>(f + e);
                each<4>([&](auto i) { v[i] = __builtin_bit_cast(u32, (float)w[i.value]); });
            }
        } else {
            each<4>([&](auto i) {
                v[i] = 0xff800000u;
                if (e + i < p.experts) v[i] = p.bf16 ? (u32)h[e + i] << 16 : __builtin_bit_cast(u32, f[e + i]);
            });
        }
        each<4>([&](auto i) { l[q * 4 + i] = __builtin_bit_cast(float, v[i]); });
    });
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
__device__ __forceinline__ int other(int v) { return (int)other<M>((u32)v); }
template <int M>
__device__ __forceinline__ double other(double v) {
    const u64 b = __builtin_bit_cast(u64, v);
    return __builtin_bit_cast(double, (u64)other<M>((u32)(b >> 32)) << 32 | other<M>((u32)b));
}

// The next lane's value, within a row of 16 lanes.
__device__ __forceinline__ int after(int v) { return __builtin_amdgcn_mov_dpp(v, 0x101, 0xf, 0xf, true); }   // row_shl:1
__device__ __forceinline__ double after(double v) {
    const u64 b = __builtin_bit_cast(u64, v);
    return __builtin_bit_cast(double, (u64)(u32)after((int)(b >> 32)) << 32 | (u32)after((int)b));
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

// Finite numbers here are far from a double's largest, where experts that are out, infinity and NaN (the largest) have their places.
constexpr double kOut = -0x1p1023, kInf = 0x1p1022, kNan = 0x1p1023;
__device__ __forceinline__ double placed(double b) {
    return b != b ? kNan : b == -__builtin_inf() ? kOut : b == __builtin_inf() ? kInf : b;
}
__device__ __forceinline__ double key_bits(double b, u32 low) { return __builtin_bit_cast(double, (__builtin_bit_cast(u64, b) & ~1023ull) | low); }
// A number as a key: its low ten bits give way to the expert's index (the lower, the larger).
__device__ __forceinline__ double key_of(double b, int e) {
    const u64 v = __builtin_bit_cast(u64, b);
    return key_bits(b, (int)(v >> 32) < 0 ? e : 1023 - e);
}
__device__ __forceinline__ int expert_of_key(double k) {
    const u64 v = __builtin_bit_cast(u64, k);
    if (k <= kOut) return -1;
    return (int)(v >> 32) < 0 ? (int)(v & 1023) : 1023 - (int)(v & 1023);
}

// What a token's lanes, all of one wave, wrote to LDS before is there for the others after.
__device__ __forceinline__ void lanes_wait() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The choices of one token in 64 bits, by the whole wave: lane c has the id of choice c, -1 for none.  logits, rows [N]: its logits, and
// room for b; sums [kMaxGroups].
template <int N, int KP, bool SOFTMAX>
__device__ __forceinline__ int choose64(const RouteParams& p, const float* logits, double* rows, double* sums) {
    constexpr int P = N / 64;
    const int lane = threadIdx.x & 63;
    double b[P];
#pragma unroll
    for (int i = 0; i < P; ++i) b[i] = (double)logits[i * 64 + lane] + 0.0;   // (-inf past the last expert; -0 becomes +0)
    if (!p.by_logit) {
        if constexpr (SOFTMAX) {
            double top = b[0], sum = 0;
#pragma unroll
            for (int i = 1; i < P; ++i) top = fmax(top, b[i]);
            top = fmax(top, other<1>(top)); top = fmax(top, other<2>(top)); top = fmax(top, other<4>(top));
            top = fmax(top, other<8>(top)); top = fmax(top, other<16>(top)); top = fmax(top, other<32>(top));
#pragma unroll
            for (int i = 0; i < P; ++i) {
                b[i] = b[i] == -__builtin_inf() ? b[i] : exp(b[i] - top);
                if (b[i] != -__builtin_inf()) sum += b[i];
            }
            sum = lanes_sum<64>(sum);
#pragma unroll
            for (int i = 0; i < P; ++i)
                if (b[i] != -__builtin_inf()) b[i] /= sum;
        } else {
#pragma unroll
            for (int i = 0; i < P; ++i)
                if (b[i] != -__builtin_inf()) b[i] = 1.0 / (1.0 + exp(-b[i]));
        }
        if (p.bias != nullptr) {
#pragma unroll
            for (int i = 0; i < P; ++i) {
                // (an expert that is out by its logit or its bias stays out, whatever the other is and beside NaN)
                const float bias = p.bias[min(i * 64 + lane, p.experts - 1)];
                b[i] += (double)bias;
                if (logits[i * 64 + lane] == -__builtin_inff() || bias == -__builtin_inff()) b[i] = -__builtin_inf();
            }
        }
    }
    if (p.groups > 1) {
#pragma unroll
        for (int i = 0; i < P; ++i) rows[i * 64 + lane] = b[i];
        lanes_wait();
        if (lane < p.groups) {
            double first = -__builtin_inf(), second = first;
            bool nan = false;
            for (int j = 0; j < p.per_group; ++j) {
                const double v = rows[lane * p.per_group + j];
                nan = nan || v != v;
                second = fmax(second, fmin(first, v));
                first = fmax(first, v);
            }
            // (a group of one expert, or with one left, has that one's b; NaN is the largest here too)
            double sum = first;
            if (p.group_top > 1 && second != -__builtin_inf()) sum += second;
            sums[lane] = nan || sum != sum ? kNan : sum == __builtin_inf() ? kInf : sum;
        }
        lanes_wait();
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int e = i * 64 + lane;
            if (e >= p.experts) continue;
            const int g = (int)((u32)e * p.per_group_inv >> 21);
            const double mine = sums[g];
            int before = 0;
            for (int o = 0; o < p.groups; ++o) before += sums[o] > mine || (sums[o] == mine && o < g);
            if (before >= p.keep) b[i] = -__builtin_inf();
        }
    }
    double list[KP];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        b[i] = placed(b[i]);
        rows[i * 64 + lane] = b[i];
        b[i] = key_of(b[i], i * 64 + lane);
    }
    largest<64, P, KP>(b, list, kOut * 1.5);
    double key = kOut, last_key = kOut;
#pragma unroll
    for (int c = 0; c < KP; ++c) {
        if (lane == c) key = list[c];
        if (c == p.topk - 1) last_key = list[c];
    }
    int id = expert_of_key(key);
    if (p.by_logit) return id;
    // Keys are numbers without their last bits (those of logits end before).  The choice is held against the numbers: each above the next,
    // or equal to it by a lower index; and where experts beside the choices share the last one's bits, as many at or above it as choices.
    lanes_wait();
    const double at = id >= 0 ? rows[id] : kOut, next = after(at);
    const int next_id = after(id);
    bool wrong = lane + 1 < p.topk && next_id >= 0 && !(at > next || (at == next && id < next_id));
    if (last_key > kOut) {
        const double from = fmin(key_bits(last_key, 0), key_bits(last_key, 1023));
        int near = 0;
#pragma unroll
        for (int i = 0; i < P; ++i) near += __popcll(__ballot(b[i] >= from));
        if (near > p.topk) {
            const u64 bits = __builtin_bit_cast(u64, at);
            const u32 high = (u32)__builtin_amdgcn_readlane((int)(bits >> 32), p.topk - 1), low = (u32)__builtin_amdgcn_readlane((int)bits, p.topk - 1);
            const double last = __builtin_bit_cast(double, (u64)high << 32 | low);
            const int last_id = expert_of_key(last_key);
            near = 0;
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const double v = rows[i * 64 + lane];
                near += __popcll(__ballot(v > last || (v == last && i * 64 + lane <= last_id)));
            }
            wrong = wrong || near != p.topk;
        }
    }
    if (__ballot(wrong) != 0) {   // (numbers nearer than 2^-42 of their size and not equal, such as sigmoids near 1)
#pragma unroll 1
        for (int c = 0; c < p.topk; ++c) {
            double best = kOut;
            int who = N;
#pragma unroll 1
            for (int e = lane; e < N; e += 64)
                if (rows[e] > best) {
                    best = rows[e];
                    who = e;
                }
            auto join = [&](double o, int w) {
                if (o > best || (o == best && w < who)) {
                    best = o;
                    who = w;
                }
            };
            join(other<1>(best), other<1>(who)); join(other<2>(best), other<2>(who)); join(other<4>(best), other<4>(who));
            join(other<8>(best), other<8>(who)); join(other<16>(best), other<16>(who)); join(other<32>(best), other<32>(who));
            if (lane == c) id = who < N ? who : -1;
            if (who < N && (who & 63) == lane) rows[who] = kOut;   // (which this lane alone reads)
        }
    }
    return id;
}

// In fp32: a number that stands for "out", far below all others but finite.
constexpr float kLow = -0x1.8p127f;
constexpr float kHuge = 0x1p126f;   // (a group's sum of numbers past this may have left fp32)

// s of a logit; softmax: `top` and the inverse of the sum.  For the choice, with an error that grows with the exponent (32768 tokens over
// 256 experts 27 us, with that of weight32 31); what is near is looked at again.
template <bool SOFTMAX>
__device__ __forceinline__ float score32(float l, float top, float inv) {
    if constexpr (SOFTMAX) return __expf(l - top) * inv;
    else return __builtin_amdgcn_rcpf(1.f + __expf(-l));
}
// The same for the weights.
template <bool SOFTMAX>
__device__ __forceinline__ float weight32(float l, float top, float inv) {
    if constexpr (SOFTMAX) return expf(l - top) * inv;
    else return 1.f / (1.f + expf(-l));
}

template <int LPT, int P, int KP, bool SOFTMAX>
__global__ __launch_bounds__(kThreads) void route_kernel(const RouteParams p) {
    // for the tokens that need 64 bits, one of a wave at a time; and, of every token, the groups' scores
    __shared__ double rows64[kThreads / 64][LPT * P], sums64[kThreads / 64][kMaxGroups];
    __shared__ f32x2 sums_of[kThreads / LPT][kMaxGroups];
    __shared__ float rows_of[kThreads / LPT][LPT * P];   // b, for groups that are no run of lanes; then the logits, for 64 bits
    const int tid = threadIdx.x, sub = tid % LPT, mine = tid / LPT, wave = tid >> 6;
    const int64_t t = (int64_t)(blockIdx.x + p.vbase) * (kThreads / LPT) + mine;
    const int64_t row = t < p.tokens ? t : p.tokens - 1;   // (lanes past the last token keep the others company)
    float l[P], b[P];
    load_row<LPT>(p, row, sub, l);
    if (p.bias != nullptr) {
        RouteParams as_row = p;
        as_row.logits = p.bias;
        as_row.ld = as_row.bf16 = 0;
        load_row<LPT>(as_row, 0, sub, b);
    } else {
        each<P>([&](auto i) {
            b[i] = 0.f;
        });
    }
    float top = 0.f, inv = 1.f;
    if constexpr (SOFTMAX) {
        top = l[0];
        each<P - 1>([&](auto from_1) {
            constexpr int i = from_1 + 1;
            top = fmaxf(top, l[i]);
        });
        top = lanes_max<LPT>(top);
        top = top == -__builtin_inff() ? 0.f : top;   // (every expert out)
        float sum = 0.f;
        each<P>([&](auto i) {
            sum += __expf(l[i] - top);
        });
        inv = 1.f / lanes_sum<LPT>(sum);
    }
    // b in fp32, and whether the row has a NaN, +inf or a finite number as low as kLow (then odd is NaN)
    float odd = 0.f;
    if (p.by_logit) {
        each<P>([&](auto i) {
            b[i] = l[i] + 0.f;   // (-0 becomes +0: keys tell them apart, numbers do not)
        });
    } else {
        each<P>([&](auto i) {
            b[i] += score32<SOFTMAX>(l[i], top, inv);
        });
    }
    each<P>([&](auto i) {
        if (l[i] == -__builtin_inff() || b[i] == -__builtin_inff()) b[i] = kLow;
        else if (b[i] <= kLow) b[i] = __builtin_inff();
        odd = __builtin_fmaf(b[i], 0.f, odd);
    });
    if (SOFTMAX && !p.by_logit) odd = __builtin_fmaf(top, 0.f, odd);
    bool sure = lanes_sum<LPT>(odd) == 0.f;
    // How far a difference of two b can be off, beside 2^-21 of their size (score32's steps are within 2^-22 of s, and softmax's sum
    // within 2^-19 of itself; twice that and more).
    const float slack = p.by_logit ? 0.f : SOFTMAX ? __builtin_fmaf(0x1p-17f, inv, 0x1p-21f) : 0x1p-20f;
    const float relative = p.by_logit ? 0.f : 0x1p-21f;

    if (p.groups > 1) {
        // A group's sum, as the least and the most that it can be.  Its terms may cancel, so the size of these counts, not of the sum.
        f32x2* const sums = sums_of[mine];
        auto put = [&](int g, float first, float second) {
            const bool two = p.group_top > 1 && second > kLow;
            const float sum = two ? first + second : first, size = fabsf(first) + (two ? fabsf(second) : 0.f);
            const float off = slack + relative * size;
            sums[g] = f32x2{sum - off, sum + off};
            if (first != kLow && !(size < kHuge)) sure = false;
        };
        const int lanes = p.per_group >> 2;   // of a group, where it lies in a run of them
        const int shift = p.group_lanes - 1, in_run = LPT >> shift;   // log2 of these; groups side by side in a token's lanes
        if (p.group_lanes) {
            each<P / 4>([&](auto q) {
                float first = fmaxf(b[4 * q], b[4 * q + 1]), second = fminf(b[4 * q], b[4 * q + 1]);
                each<4 - 2>([&](auto from_2) {
                    constexpr int i = from_2 + 2;
                    second = fmaxf(second, fminf(first, b[4 * q + i]));
                    first = fmaxf(first, b[4 * q + i]);
                });
                auto join = [&](float f, float s) {
                    second = fmaxf(fminf(first, f), fmaxf(second, s));
                    first = fmaxf(first, f);
                };
                if (lanes > 1) join(other<1>(first), other<1>(second));
                if (lanes > 2) join(other<2>(first), other<2>(second));
                if (lanes > 4) join(other<4>(first), other<4>(second));
                if (lanes > 8) join(other<8>(first), other<8>(second));
                const int g = q * in_run + (sub >> shift);
                if ((sub & (lanes - 1)) == 0 && g < p.groups) put(g, first, second);
            });
        } else {
            float* const rows = rows_of[mine];
            each<P>([&](auto i) { rows[expert_of<LPT>(sub, i)] = b[i]; });
            lanes_wait();
            for (int g = sub; g < p.groups; g += LPT) {
                float first = kLow, second = kLow;
                for (int j = 0; j < p.per_group; ++j) {
                    const float v = rows[g * p.per_group + j];
                    second = fmaxf(second, fminf(first, v));
                    first = fmaxf(first, v);
                }
                put(g, first, second);
            }
        }
        lanes_wait();
        if (!p.group_lanes) {
            // a group's place, by the lane that has its score; then what becomes of it, in the place of the score
            float state[kMaxGroups / LPT];
            each<kMaxGroups / LPT>([&](auto q) {
                const int g = q * LPT + sub;
                state[q] = 0.f;
                if (g >= p.groups) return;
                const f32x2 own = sums[g];
                int better = 0, near = 0;
                for (int o = 0; o < p.groups; ++o) {
                    better += sums[o][0] > own[1];
                    near += sums[o][1] >= own[0];   // (itself among them)
                }
                if (better < p.keep && near > p.keep) sure = false;
                state[q] = better >= p.keep ? 1.f : 0.f;
            });
            lanes_wait();
            each<kMaxGroups / LPT>([&](auto q) {
                if (q * LPT + sub < p.groups) sums[q * LPT + sub][0] = state[q];
            });
            lanes_wait();
            each<P>([&](auto i) {
                const u32 e = (u32)min(expert_of<LPT>(sub, i), p.experts - 1);
                if (sums[e * p.per_group_inv >> 21][0] != 0.f) b[i] = kLow;
            });
        }
        if (p.group_lanes) {
            int better[P / 4], near[P / 4];
            f32x2 own[P / 4];
            each<P / 4>([&](auto q) {
                own[q] = sums[min(q * in_run + (sub >> shift), p.groups - 1)];
                better[q] = near[q] = 0;
            });
#pragma unroll 4
            for (int o = 0; o < p.groups; ++o) {
                const f32x2 v = sums[o];
                each<P / 4>([&](auto q) {
                    better[q] += v[0] > own[q][1];
                    near[q] += v[1] >= own[q][0];   // (itself among them)
                });
            }
            each<P / 4>([&](auto q) {
                const bool gone = better[q] >= p.keep;
                if (!gone && near[q] > p.keep && q * in_run + (sub >> shift) < p.groups) sure = false;
                each<4>([&](auto i) {
                    b[4 * q + i] = gone ? kLow : b[4 * q + i];
                });
            });
        }
    }

    constexpr u32 kIndex = LPT * P - 1;
    u32 key[P], list[KP];
    each<P>([&](auto i) {
        const u32 f = __builtin_bit_cast(u32, b[i]);
        const u32 order = f ^ ((u32)((int)f >> 31) | 0x80000000u);   // (as whole numbers compare)
        key[i] = (b[i] == kLow ? 0u : order & ~kIndex) | (kIndex - (u32)expert_of<LPT>(sub, i));
    });
    largest<LPT, P, KP>(key, list, 0u);
    int id = -1;
    each<KP>([&](auto c) {
        if (sub == c && list[c] > kIndex) id = (int)(kIndex - (list[c] & kIndex));
    });
    if (sub >= p.topk) id = -1;
    float s = 0.f, at = kLow;
    if (id >= 0) {
        const float v = logit_at(p, row, id);
        s = weight32<SOFTMAX>(v, top, inv);
        at = p.by_logit ? v : s + (p.bias != nullptr ? p.bias[id] : 0.f);
    }
    if (!p.exact_keys) {
        const int base = (tid & 63) - sub;
        const float after = __shfl(at, min(base + sub + 1, 63)), last = __shfl(at, base + p.topk - 1);
        const float off = slack + relative * fabsf(at), off_last = slack + relative * fabsf(last);
        if (sub + 1 < p.topk && after != kLow && !(at - after > off)) sure = false;
        if (last != kLow) {
            int from = 0;
            each<P>([&](auto i) {
                from += b[i] >= last - off_last;
            });
            if (lanes_sum<LPT>(from) != p.topk) sure = false;
        }
    }
    // (a token's lanes agree)
    const u64 unsure = __ballot(!sure);
    if (unsure != 0) {
        constexpr u64 kLanes = LPT == 64 ? ~0ull : (1ull << (LPT & 63)) - 1;
        each<P>([&](auto i) { rows_of[mine][expert_of<LPT>(sub, i)] = l[i]; });
        lanes_wait();
#pragma unroll 1
        for (int o = 0; o < 64 / LPT; ++o) {
            if (!(unsure >> (o * LPT) & kLanes)) continue;
            const bool its = (tid & 63) / LPT == o;
            const int found = __shfl(choose64<LPT * P, KP, SOFTMAX>(p, rows_of[wave * (64 / LPT) + o], rows64[wave], sums64[wave]), sub);
            lanes_wait();
            if (!its) continue;
            id = sub < p.topk ? found : -1;
            s = id >= 0 ? weight32<SOFTMAX>(logit_at(p, row, id), top, inv) : 0.f;
        }
    }
    float w = s;
    if (p.renormalize) w /= lanes_sum<16>(s) + kTiny;   // (the choices lie in a token's first 16 lanes)
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

// 32768 tokens over 256 experts in 8 groups: 27 us (36 MB; the bytes take 7), 16 of them or more VALU instructions (74 a logit: the
// exponentials, the sorting of 16 keys a lane and the joining of four times eight are most), the rest the loads of two rounds of workgroups
// at four waves a SIMD; 16 tokens 5.7, a chain of loads, sums and exchanges.  Logits in bf16 with a bias of zeros have many equal scores,
// which go through 64 bits: 61.  Gradient: 8191 tokens over 160 experts 7.2.
typedef void (*RouteKernel)(const RouteParams);

// Lanes to a token and experts to a lane: 16 lanes are a row whose exchanges are single instructions; past 256 experts more lanes.
template <bool BACKWARD, int LPT, int P>
RouteKernel pick_topk(int topk, bool softmax) {
    if constexpr (BACKWARD) return &route_backward_kernel<LPT, P>;
    else if (softmax) return topk <= 4 ? &route_kernel<LPT, P, 4, true> : topk <= 8 ? &route_kernel<LPT, P, 8, true> : &route_kernel<LPT, P, 16, true>;
    else return topk <= 4 ? &route_kernel<LPT, P, 4, false> : topk <= 8 ? &route_kernel<LPT, P, 8, false> : &route_kernel<LPT, P, 16, false>;
}

template <bool BACKWARD>
RouteKernel pick(int experts, int topk, bool softmax, int& lanes) {
    lanes = experts <= 256 ? 16 : experts <= 512 ? 32 : 64;
    if (experts <= 64) return pick_topk<BACKWARD, 16, 4>(topk, softmax);
    if (experts <= 128) return pick_topk<BACKWARD, 16, 8>(topk, softmax);
    if (experts <= 256) return pick_topk<BACKWARD, 16, 16>(topk, softmax);
    return experts <= 512 ? pick_topk<BACKWARD, 32, 16>(topk, softmax) : pick_topk<BACKWARD, 64, 16>(topk, softmax);
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
        if (a->num_groups > kMaxGroups) return dg_set_error("dg_moe_route: at most 64 groups");
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
        p.exact_keys = p.by_logit && p.bf16;
        const int in_group = p.per_group >> 2;
        if (p.per_group % 4 == 0 && (in_group & (in_group - 1)) == 0 && in_group <= 16) p.group_lanes = 1 + __builtin_ctz(in_group);
        p.weights = a->weights;
    }
    int lanes = 0;
    const RouteKernel kernel = pick<BACKWARD>(a->experts, a->topk, p.softmax, lanes);
    return launch_op(kernel, ceil_div64(a->tokens, kThreads / lanes), kThreads, p, st, a->num_cus);
}

}  // namespace
}  // namespace dg

extern "C" int dg_moe_route(const dg_moe_route_args* args, void* stream) { return dg::route_run<false>(args, stream); }
extern "C" int dg_moe_route_backward(const dg_moe_route_args* args, void* stream) { return dg::route_run<true>(args, stream); }
