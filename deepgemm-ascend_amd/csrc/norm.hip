// Root-mean-square norm with the residual's addition before it, its output in the rows' type or quantised, and the gradient.
//
//   h = round(x + r), rstd = (mean h^2 + eps)^(-1/2), y = h rstd w
//   d_x = rstd (w d_y - h rstd^2 mean(w d_y h)) + d_h,  d_w = sum_t d_y h rstd
//
// A row lies in registers from its loads to its stores, eight values a lane and step, held by a wave or by a workgroup.  Sums in fp32.
#include "mx_eight.hpp"
#include "op_launch.hpp"

#include <type_traits>

namespace dg {
namespace {

constexpr int kMaxWidth = 32768;
constexpr int kMaxPartials = 256;   // workgroups of the gradient, each of which leaves a partial d_weight

struct NormParams {
    const void *x, *residual, *weight;
    int64_t x_ld, r_ld;
    void* h;
    int64_t h_ld;
    float* rstd;
    void* y;
    int64_t y_ld;
    int16_t* sf;
    int64_t sf_ld;
    const void *d_y, *d_h;
    int64_t dy_ld, dh_ld;
    void* d_x;
    int64_t dx_ld;
    float* partial;            // [groups][partial_ld] (gradient)
    int partial_ld;
    float* d_weight;
    int tokens, width, weight_f32;
    int groups;
    float eps, inv_width;
    int vbase;
};

// The sum over a wave, the same in every lane: within rows of 16 lanes, then lane 15 to the next row and lane 31 to the upper half.
__device__ __forceinline__ float wave_sum(float v) {
    auto moved = [](float x, auto ctrl, auto rows) {
        return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, decltype(rows)::value, 0xf, false));
    };
    using std::integral_constant;
    v += moved(v, integral_constant<int, kXor1>(), integral_constant<int, 0xf>());
    v += moved(v, integral_constant<int, kXor2>(), integral_constant<int, 0xf>());
    v += moved(v, integral_constant<int, kMirror8>(), integral_constant<int, 0xf>());
    v += moved(v, integral_constant<int, 0x140>(), integral_constant<int, 0xf>());   // row_mirror
    v += moved(v, integral_constant<int, 0x142>(), integral_constant<int, 0xa>());   // row_bcast15 to rows 1 and 3
    v += moved(v, integral_constant<int, 0x143>(), integral_constant<int, 0xc>());   // row_bcast31 to rows 2 and 3
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

// The sum over the THREADS that hold a row, of TEAMS in a workgroup; `turn` alternates between two halves of `part`, so that one
// barrier does.
template <int THREADS, int TEAMS>
__device__ __forceinline__ float row_sum(float v, float (&part)[2][16], int turn) {
    v = wave_sum(v);
    if constexpr (THREADS > 64) {
        constexpr int WAVES = THREADS / 64;
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) part[turn][wave] = v;
        __syncthreads();
        v = 0.f;
        const float* const mine = part[turn] + wave / WAVES * WAVES;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) v += mine[i];
    }
    return v;
}

__device__ __forceinline__ void load_weight(Eight<float>& w, const NormParams& p, int col, int n) {
    if (p.weight_f32) load_eight(w, reinterpret_cast<const float*>(p.weight) + col, n);
    else load_eight(w, reinterpret_cast<const uint16_t*>(p.weight) + col, n);
}

// FMT: -1 values, DG_MX_*.  THREADS hold a row (64: the workgroup's four waves hold one each), V steps of eight values a thread.
// ROWS rows to a workgroup, so that exponent bytes leave as runs of rows.  Bound by the bytes: 8192 x 4096 bf16 with residual 44 us (6.1
// TB/s), 4096 x 7168 to e4m3 40 (5.1); 16 x 7168 to e4m3 3.9, one chain of loads, sum and stores.
template <typename E, int FMT, int THREADS, int V, int ROWS>
__global__ __launch_bounds__(THREADS < 256 ? 256 : THREADS) void norm_kernel(const NormParams p) {
    constexpr int WG = THREADS < 256 ? 256 : THREADS, AT_ONCE = WG / THREADS;
    __shared__ float part[2][16];
    __shared__ uint16_t pairs[FMT >= 0 ? THREADS * V / 8 : 1][ROWS + 2];
    const int at = threadIdx.x % THREADS, which = threadIdx.x / THREADS;
    const int64_t row0 = (int64_t)(blockIdx.x + p.vbase) * ROWS;
    Eight<float> w[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int col = (j * THREADS + at) * 8;
        load_weight(w[j], p, col, p.width - col);
    }
#pragma unroll 1
    for (int r = 0; r < ROWS; r += AT_ONCE) {
        const int64_t t = row0 + r + which;
        if (THREADS > 64 && t >= p.tokens) break;   // (the whole workgroup)
        const bool on = t < p.tokens;
        Eight<float> v[V];
        float squares = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int col = (j * THREADS + at) * 8, n = on ? p.width - col : 0;
            load_eight(v[j], reinterpret_cast<const E*>(p.x) + t * p.x_ld + col, n);
            if (p.residual != nullptr) {
                Eight<float> a;
                load_eight(a, reinterpret_cast<const E*>(p.residual) + t * p.r_ld + col, n);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    v[j].v[i] += a.v[i];
                    if constexpr (sizeof(E) == 2) v[j].v[i] = bf16_to_f32(f32_to_bf16_rne(v[j].v[i]));   // (what the residual stream holds)
                }
                store_eight(reinterpret_cast<E*>(p.h) + t * p.h_ld + col, v[j], n);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) squares += v[j].v[i] * v[j].v[i];
        }
        const float rstd = rsqrtf(row_sum<THREADS, AT_ONCE>(squares, part, r & 1) * p.inv_width + p.eps);
        if (on && at == 0) p.rstd[t] = rstd;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int col = (j * THREADS + at) * 8, n = on ? p.width - col : 0;
            Eight<float> y;
#pragma unroll
            for (int i = 0; i < 8; ++i) y.v[i] = v[j].v[i] * rstd * w[j].v[i];
            if constexpr (FMT < 0) {
                store_eight(reinterpret_cast<E*>(p.y) + t * p.y_ld + col, y, n);
            } else {
                // (a width that is a multiple of 32: a lane has eight values or none, and so have a block's others)
                constexpr bool FP4 = FMT == DG_MX_E2M1;
                const u32 s = block_scale<FP4>(y.top()), next = dpp<kMirror8>(s);
                if ((at & 7) == 0) pairs[(j * THREADS + at) >> 3][r + which] = (uint16_t)(s | (col + 32 < p.width ? next << 8 : 0u));
                if (n > 0) {
                    uint8_t* const to = reinterpret_cast<uint8_t*>(p.y) + t * p.y_ld + (FP4 ? col / 2 : col);
                    if constexpr (FP4) *reinterpret_cast<u32*>(to) = codes_e2m1(y, s);
                    else *reinterpret_cast<i32x2*>(to) = codes_e4m3(y, s);
                }
            }
        }
    }
    if constexpr (FMT >= 0) {
        __syncthreads();
        // two rows a thread: the leading dimension is even, and an odd last row's partner is written 0
        const int k64 = ceil_div(p.width, 64);
        if constexpr (ROWS == 1) {
            for (int j = threadIdx.x; j < k64; j += WG) {
                int16_t* const to = p.sf + (int64_t)j * p.sf_ld + row0;
                if (row0 % 2 == 0 && row0 + 1 == p.tokens) *reinterpret_cast<u32*>(to) = pairs[j][0];
                else *to = (int16_t)pairs[j][0];
            }
            return;
        }
        constexpr int TWO = ROWS > 1 ? ROWS / 2 : 1;
        for (int e = threadIdx.x; e < k64 * TWO; e += WG) {
            const int j = e / TWO, r = e % TWO * 2;
            if (row0 + r >= p.tokens) continue;
            const u32 two = pairs[j][r] | (row0 + r + 1 < p.tokens ? (u32)pairs[j][r + 1] << 16 : 0u);
            *reinterpret_cast<u32*>(p.sf + (int64_t)j * p.sf_ld + row0 + r) = two;
        }
    }
}

// What a thread holds of a token's h and d_y.
template <typename E, int V>
struct BackwardRow {
    Raw<E> h[V], d[V];
    float rstd;
    template <int THREADS>
    __device__ __forceinline__ void load(const NormParams& p, int64_t t, int at) {
        const bool on = t < p.tokens;
        rstd = on ? p.rstd[t] : 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int col = (j * THREADS + at) * 8, n = on ? p.width - col : 0;
            h[j].load(reinterpret_cast<const E*>(p.h) + t * p.h_ld + col, n);
            d[j].load(reinterpret_cast<const E*>(p.d_y) + t * p.dy_ld + col, n);
        }
    }
};

// TEAMS of THREADS hold a row each and step through the tokens together; the next rows (bf16) are in flight while a row is summed.
// d_weight is summed over a team's rows in registers, over the teams in LDS, in order.  8192 x 4096 bf16 51 us (5.2 TB/s, 32 bytes a lane
// in scratch at the 128 registers that 1024 threads leave; 82 with two workgroups of one row a CU that read a row when they are done with
// the one before), and 5 for the partial sums.
template <typename E, int THREADS, int TEAMS, int V>
__global__ __launch_bounds__(THREADS * TEAMS) void norm_backward_kernel(const NormParams p) {
    constexpr bool AHEAD = sizeof(E) == 2 && V <= 2;
    __shared__ float part[2][16];
    __shared__ float joined[TEAMS > 1 ? THREADS * V * 8 : 1];
    const int at = threadIdx.x % THREADS, team = threadIdx.x / THREADS, group = blockIdx.x + p.vbase;
    Eight<float> sum[V];
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[j].v[i] = 0.f;
    const int64_t step = (int64_t)p.groups * TEAMS;
    int64_t t = (int64_t)group * TEAMS + team;
    BackwardRow<E, V> row, next;
    row.template load<THREADS>(p, t, at);
    int turn = 0;
    // (a workgroup's teams take as many steps: that of the first team, whose tokens come first)
#pragma unroll 1
    for (int64_t first = (int64_t)group * TEAMS; first < p.tokens; first += step, t += step) {
        Raw<E> a[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int col = (j * THREADS + at) * 8;
            a[j].load(reinterpret_cast<const E*>(p.d_h) + t * p.dh_ld + col, p.d_h != nullptr && t < p.tokens ? p.width - col : 0);
        }
        if constexpr (AHEAD) next.template load<THREADS>(p, t + step, at);
        const float rstd = row.rstd;
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int col = (j * THREADS + at) * 8;
            Eight<float> w, h, d;
            load_weight(w, p, col, p.width - col);
            row.h[j].values(h);
            row.d[j].values(d);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                h.v[i] *= rstd;
                sum[j].v[i] += d.v[i] * h.v[i];
                dot += d.v[i] * w.v[i] * h.v[i];
            }
        }
        const float mean = row_sum<THREADS, TEAMS>(dot, part, turn) * p.inv_width;
        turn ^= 1;
        if (t < p.tokens) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int col = (j * THREADS + at) * 8, n = p.width - col;
                Eight<float> w, h, d, g;
                load_weight(w, p, col, n);
                row.h[j].values(h);
                row.d[j].values(d);
                a[j].values(g);
#pragma unroll
                for (int i = 0; i < 8; ++i) g.v[i] += rstd * (d.v[i] * w.v[i] - h.v[i] * rstd * mean);
                store_eight(reinterpret_cast<E*>(p.d_x) + t * p.dx_ld + col, g, n);
            }
        }
        if constexpr (AHEAD) row = next;
        else row.template load<THREADS>(p, t + step, at);
    }
    if constexpr (TEAMS > 1) {
        for (int o = 0; o < TEAMS; ++o) {
            if (team == o)
#pragma unroll
                for (int j = 0; j < V; ++j)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        float& to = joined[(j * 8 + i) * THREADS + at];
                        to = o == 0 ? sum[j].v[i] : to + sum[j].v[i];
                    }
            __syncthreads();
        }
        if (team != 0) return;
#pragma unroll
        for (int j = 0; j < V; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[j].v[i] = joined[(j * 8 + i) * THREADS + at];
    }
    float* const to = p.partial + (int64_t)group * p.partial_ld;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int col = (j * THREADS + at) * 8;
        store_eight(to + col, sum[j], p.width - col);
    }
}

// d_weight from the partial sums, in order: 32 columns a workgroup, four a thread, 32 threads to a column.
__global__ __launch_bounds__(256) void norm_weight_kernel(const NormParams p) {
    __shared__ f32x4 part[32][8];
    const int c = threadIdx.x & 7, r = threadIdx.x >> 3, col = (blockIdx.x + p.vbase) * 32 + c * 4;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    if (col < p.width) {
#pragma unroll 8
        for (int g = r; g < p.groups; g += 32) {
            const f32x4 o = *reinterpret_cast<const f32x4*>(p.partial + (int64_t)g * p.partial_ld + col);   // (rows of whole fours)
#pragma unroll
            for (int q = 0; q < 4; ++q) sum[q] += o[q];
        }
    }
    part[r][c] = sum;
    __syncthreads();
    const int one = threadIdx.x, mine = (blockIdx.x + p.vbase) * 32 + one;
    if (one >= 32 || mine >= p.width) return;
    float all = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) all += part[i][one >> 2][one & 3];
    p.d_weight[mine] = all;
}

typedef void (*NormKernel)(const NormParams);

// A workgroup to a row, as wide as the row allows; many short rows go to a wave each, four side by side (8192 x 1024 12.7 -> 11.1 us, to
// e4m3 13.9 -> 11.8).  Rows that follow each other in a workgroup of 256 threads, whose exponent bytes then leave as runs of eight rows, wait
// for each other's sums: 1024 x 7168 to e4m3 34.6 us in place of 11.3, 4096 x 7168 62 in place of 42.
template <typename E, int FMT>
NormKernel pick_forward(int tokens, int width, unsigned& threads, int& rows) {
    if (width <= 1024 && tokens > 2048) {
        rows = FMT >= 0 ? 8 : 4;
        threads = 256;
        if (width <= 512) return &norm_kernel<E, FMT, 64, 1, FMT >= 0 ? 8 : 4>;
        return &norm_kernel<E, FMT, 64, 2, FMT >= 0 ? 8 : 4>;
    }
    rows = 1;
    threads = width <= 2048 ? 256 : width <= 4096 ? 512 : 1024;
    if (width <= 2048) return &norm_kernel<E, FMT, 256, 1, 1>;
    if (width <= 4096) return &norm_kernel<E, FMT, 512, 1, 1>;
    if (width <= 8192) return &norm_kernel<E, FMT, 1024, 1, 1>;
    if (width <= 16384) return &norm_kernel<E, FMT, 1024, 2, 1>;
    return &norm_kernel<E, FMT, 1024, 4, 1>;
}

// Rows that a workgroup of the gradient holds at once.
int teams(int width) { return width <= 1024 ? 16 : width <= 2048 ? 8 : width <= 4096 ? 4 : width <= 8192 ? 2 : 1; }

// Few tokens: 512 threads to a workgroup where a row leaves that choice, so that more CUs have rows.
bool few(int tokens, int width) { return width <= 4096 && tokens < kMaxPartials * teams(width); }

template <typename E>
NormKernel pick_backward(int tokens, int width) {
    if (few(tokens, width)) {
        if (width <= 512) return &norm_backward_kernel<E, 64, 8, 1>;
        if (width <= 1024) return &norm_backward_kernel<E, 64, 8, 2>;
        if (width <= 2048) return &norm_backward_kernel<E, 128, 4, 2>;
        return &norm_backward_kernel<E, 256, 2, 2>;
    }
    if (width <= 512) return &norm_backward_kernel<E, 64, 16, 1>;
    if (width <= 1024) return &norm_backward_kernel<E, 64, 16, 2>;
    if (width <= 2048) return &norm_backward_kernel<E, 128, 8, 2>;
    if (width <= 4096) return &norm_backward_kernel<E, 256, 4, 2>;
    if (width <= 8192) return &norm_backward_kernel<E, 512, 2, 2>;
    if (width <= 16384) return &norm_backward_kernel<E, 1024, 1, 2>;
    return &norm_backward_kernel<E, 1024, 1, 4>;
}

// Workgroups of the gradient: one to a CU, whose partial sums cost little.
int partials(int tokens, int width) {
    return std::max(1, std::min(ceil_div(tokens, few(tokens, width) ? teams(width) / 2 : teams(width)), kMaxPartials));
}

int check(const dg_rms_norm_args* a, NormParams& p) {
    if (a == nullptr) return dg_set_error("dg_rms_norm: null args");
    if ((a->dtype != DG_DTYPE_BF16 && a->dtype != DG_DTYPE_F32) || (a->weight_dtype != DG_DTYPE_BF16 && a->weight_dtype != DG_DTYPE_F32))
        return dg_set_error("dg_rms_norm: values and weight are bf16 or fp32");
    if (a->tokens < 0 || a->tokens > kMaxExtent) return dg_set_error("dg_rms_norm: at most 2^30 tokens");
    if (a->width < 1 || a->width > kMaxWidth) return dg_set_error("dg_rms_norm: width must be between 1 and 32768");
    p = {};
    p.tokens = a->tokens;
    p.width = a->width;
    p.inv_width = 1.f / a->width;
    p.eps = a->eps;
    p.weight = a->weight;
    p.weight_f32 = a->weight_dtype == DG_DTYPE_F32;
    p.h = a->h;
    p.h_ld = a->h_ld;
    p.rstd = a->rstd;
    return DG_OK;
}

int forward(const dg_rms_norm_args* a, void* stream) {
    NormParams p;
    if (const int rc = check(a, p); rc != DG_OK) return rc;
    const int64_t size = a->dtype == DG_DTYPE_BF16 ? 2 : 4;
    const bool quant = a->format != -1;
    if (quant && a->format != DG_MX_E2M1 && a->format != DG_MX_E4M3) return dg_set_error("dg_rms_norm: unknown format");
    if (quant && a->width % 32 != 0) return dg_set_error("dg_rms_norm: a quantised width must be a multiple of the block of 32 values");
    if (a->tokens == 0) return DG_OK;
    if (a->x == nullptr || a->weight == nullptr || a->rstd == nullptr || a->y == nullptr || (a->residual != nullptr && a->h == nullptr) ||
        (quant && a->sf == nullptr))
        return dg_set_error("dg_rms_norm: null tensor");
    const int64_t row = a->format == DG_MX_E2M1 ? a->width / 2 : a->width;
    if (a->x_ld < a->width || a->y_ld < row || (a->residual != nullptr && (a->residual_ld < a->width || a->h_ld < a->width)) ||
        (quant && a->sf_ld < a->tokens))
        return dg_set_error("dg_rms_norm: leading dimension smaller than the row");
    if (quant && (a->sf_ld % 2 != 0 || !aligned_to(a->sf, 4))) return dg_set_error("dg_rms_norm: scale factors need an even leading dimension and 4-byte alignment");
    if (quant && (a->y_ld % 8 != 0 || !aligned_to(a->y, 8))) return dg_set_error("dg_rms_norm: rows of codes must be 8-byte aligned");
    if (!aligned_to(a->x, size) || !aligned_to(a->residual, size) || !aligned_to(a->h, size) || !aligned_to(a->rstd, 4) ||
        (!quant && !aligned_to(a->y, size)) || !aligned_to(a->weight, p.weight_f32 ? 4 : 2))
        return dg_set_error("dg_rms_norm: tensors must be aligned");
    p.x = a->x;
    p.x_ld = a->x_ld;
    p.residual = a->residual;
    p.r_ld = a->residual_ld;
    p.y = a->y;
    p.y_ld = a->y_ld;
    p.sf = a->sf;
    p.sf_ld = a->sf_ld;
    unsigned threads = 0;
    int rows = 0;
    NormKernel kernel;
    if (a->dtype == DG_DTYPE_F32)
        kernel = !quant ? pick_forward<float, -1>(a->tokens, a->width, threads, rows)
                        : a->format == DG_MX_E2M1 ? pick_forward<float, DG_MX_E2M1>(a->tokens, a->width, threads, rows) : pick_forward<float, DG_MX_E4M3>(a->tokens, a->width, threads, rows);
    else
        kernel = !quant ? pick_forward<uint16_t, -1>(a->tokens, a->width, threads, rows)
                        : a->format == DG_MX_E2M1 ? pick_forward<uint16_t, DG_MX_E2M1>(a->tokens, a->width, threads, rows) : pick_forward<uint16_t, DG_MX_E4M3>(a->tokens, a->width, threads, rows);
    return launch_op(kernel, ceil_div64(a->tokens, rows), threads, p, reinterpret_cast<hipStream_t>(stream), a->num_cus);
}

int workspace_size(const dg_rms_norm_args* a, int64_t* bytes) {
    NormParams p;
    if (bytes == nullptr) return dg_set_error("dg_rms_norm: null result");
    if (const int rc = check(a, p); rc != DG_OK) return rc;
    *bytes = (int64_t)partials(a->tokens, a->width) * align_up(a->width, 4) * 4;
    return DG_OK;
}

int backward(const dg_rms_norm_args* a, void* stream) {
    NormParams p;
    if (const int rc = check(a, p); rc != DG_OK) return rc;
    const int64_t size = a->dtype == DG_DTYPE_BF16 ? 2 : 4;
    const bool some = a->tokens > 0;
    if (a->d_weight == nullptr || a->weight == nullptr || (some && (a->h == nullptr || a->rstd == nullptr || a->d_y == nullptr || a->d_x == nullptr)))
        return dg_set_error("dg_rms_norm: null tensor");
    if (some && (a->h_ld < a->width || a->d_y_ld < a->width || a->d_x_ld < a->width || (a->d_h != nullptr && a->d_h_ld < a->width)))
        return dg_set_error("dg_rms_norm: leading dimension smaller than the row");
    if (!aligned_to(a->h, size) || !aligned_to(a->d_y, size) || !aligned_to(a->d_h, size) || !aligned_to(a->d_x, size) || !aligned_to(a->rstd, 4) ||
        !aligned_to(a->d_weight, 4) || !aligned_to(a->workspace, 16) || !aligned_to(a->weight, p.weight_f32 ? 4 : 2))
        return dg_set_error("dg_rms_norm: tensors must be aligned");
    p.groups = partials(a->tokens, a->width);
    if (a->workspace == nullptr || a->workspace_bytes < (int64_t)p.groups * align_up(a->width, 4) * 4) return dg_set_error("dg_rms_norm: workspace too small");
    p.d_y = a->d_y;
    p.dy_ld = a->d_y_ld;
    p.d_h = a->d_h;
    p.dh_ld = a->d_h_ld;
    p.d_x = a->d_x;
    p.dx_ld = a->d_x_ld;
    p.partial = static_cast<float*>(a->workspace);
    p.partial_ld = align_up(a->width, 4);
    p.d_weight = a->d_weight;
    const NormKernel kernel = a->dtype == DG_DTYPE_F32 ? pick_backward<float>(a->tokens, a->width) : pick_backward<uint16_t>(a->tokens, a->width);
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (const int rc = launch_op(kernel, p.groups, few(a->tokens, a->width) ? 512 : 1024, p, st, a->num_cus); rc != DG_OK) return rc;
    return launch_op(&norm_weight_kernel, ceil_div(a->width, 32), 256, p, st, a->num_cus);
}

}  // namespace
}  // namespace dg

extern "C" int dg_rms_norm_workspace_size(const dg_rms_norm_args* args, int64_t* bytes) { return dg::workspace_size(args, bytes); }
extern "C" int dg_rms_norm_forward(const dg_rms_norm_args* args, void* stream) { return dg::forward(args, stream); }
extern "C" int dg_rms_norm_backward(const dg_rms_norm_args* args, void* stream) { return dg::backward(args, stream); }
