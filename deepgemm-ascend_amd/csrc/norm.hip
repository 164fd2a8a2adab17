// Root-mean-square norm with the residual's addition before it, its output in the rows' type or quantised, and the gradient.
//
//   h = round(x + r), rstd = (mean h^2 + eps)^(-1/2), y = h rstd w
//   d_x = rstd (w d_y - h rstd^2 mean(w d_y h)) + d_h,  d_w = sum_t d_y h rstd
//
// A row lies in registers from its loads to its stores, eight values a lane and step, held by a wave or by a workgroup.  Sums in fp32.
#include "mx_eight.hpp"
#include "op_launch.hpp"

namespace dg {
namespace {

constexpr int kMaxWidth = 32768;
constexpr int kMaxPartials = 512;   // workgroups of the gradient, each of which leaves a partial d_weight

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
    float* partial;            // [groups][width] (gradient)
    float* d_weight;
    int tokens, width, weight_f32;
    int groups;
    float eps, inv_width;
    int vbase;
};

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m);
    return v;
}

// The sum over the threads that hold a row; `turn` alternates between the two halves of `part`, so that one barrier does.
template <int THREADS>
__device__ __forceinline__ float row_sum(float v, float (*part)[16], int turn) {
    v = wave_sum(v);
    if constexpr (THREADS > 64) {
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) part[turn][wave] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < THREADS / 64; ++i) v += part[turn][i];
    }
    return v;
}

__device__ __forceinline__ void load_weight(Eight<float>& w, const NormParams& p, int col, int n) {
    if (p.weight_f32) load_eight(w, reinterpret_cast<const float*>(p.weight) + col, n);
    else load_eight(w, reinterpret_cast<const uint16_t*>(p.weight) + col, n);
}

// FMT: -1 values, DG_MX_*.  THREADS hold a row (64: the workgroup's four waves hold one each), V steps of eight values a thread.
// ROWS rows to a workgroup, so that exponent bytes leave as runs of rows.
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
        const float rstd = rsqrtf(row_sum<THREADS>(squares, part, r & 1) * p.inv_width + p.eps);
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
        for (int e = threadIdx.x; e < k64 * (ROWS / 2); e += WG) {
            const int j = e / (ROWS / 2), r = e % (ROWS / 2) * 2;
            if (row0 + r >= p.tokens) continue;
            const u32 two = pairs[j][r] | (row0 + r + 1 < p.tokens ? (u32)pairs[j][r + 1] << 16 : 0u);
            *reinterpret_cast<u32*>(p.sf + (int64_t)j * p.sf_ld + row0 + r) = two;
        }
    }
}

// Rows t, t + step, ...: d_x as they come, d_weight summed over them in registers.
template <typename E, int THREADS, int V>
__global__ __launch_bounds__(THREADS < 256 ? 256 : THREADS) void norm_backward_kernel(const NormParams p) {
    constexpr int WG = THREADS < 256 ? 256 : THREADS, AT_ONCE = WG / THREADS;
    __shared__ float part[2][16];
    __shared__ float joined[AT_ONCE > 1 ? THREADS * V * 8 : 1];
    const int at = threadIdx.x % THREADS, which = threadIdx.x / THREADS, group = blockIdx.x + p.vbase;
    Eight<float> w[V], sum[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int col = (j * THREADS + at) * 8;
        load_weight(w[j], p, col, p.width - col);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[j].v[i] = 0.f;
    }
    int turn = 0;
#pragma unroll 1
    for (int64_t t = (int64_t)group * AT_ONCE + which; t < p.tokens; t += (int64_t)p.groups * AT_ONCE) {
        Eight<float> h[V], d[V];
        const float rstd = p.rstd[t];
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int col = (j * THREADS + at) * 8, n = p.width - col;
            load_eight(h[j], reinterpret_cast<const E*>(p.h) + t * p.h_ld + col, n);
            load_eight(d[j], reinterpret_cast<const E*>(p.d_y) + t * p.dy_ld + col, n);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                h[j].v[i] *= rstd;
                sum[j].v[i] += d[j].v[i] * h[j].v[i];
                d[j].v[i] *= w[j].v[i];
                dot += d[j].v[i] * h[j].v[i];
            }
        }
        const float mean = row_sum<THREADS>(dot, part, turn) * p.inv_width;
        turn ^= 1;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int col = (j * THREADS + at) * 8, n = p.width - col;
            Eight<float> g;
#pragma unroll
            for (int i = 0; i < 8; ++i) g.v[i] = rstd * (d[j].v[i] - h[j].v[i] * mean);
            if (p.d_h != nullptr) {
                Eight<float> a;
                load_eight(a, reinterpret_cast<const E*>(p.d_h) + t * p.dh_ld + col, n);
#pragma unroll
                for (int i = 0; i < 8; ++i) g.v[i] += a.v[i];
            }
            store_eight(reinterpret_cast<E*>(p.d_x) + t * p.dx_ld + col, g, n);
        }
    }
    // the waves of a workgroup one after another, in order
    if constexpr (AT_ONCE > 1) {
        for (int o = 0; o < AT_ONCE; ++o) {
            if (which == o)
#pragma unroll
                for (int j = 0; j < V; ++j)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        float& to = joined[(j * 8 + i) * THREADS + at];
                        to = o == 0 ? sum[j].v[i] : to + sum[j].v[i];
                    }
            __syncthreads();
        }
        if (which != 0) return;
#pragma unroll
        for (int j = 0; j < V; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[j].v[i] = joined[(j * 8 + i) * THREADS + at];
    }
    float* const to = p.partial + (int64_t)group * p.width;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int col = (j * THREADS + at) * 8;
        store_eight(to + col, sum[j], p.width - col);
    }
}

// d_weight from the partial sums, in order: 16 columns a workgroup, 16 threads to a column.
__global__ __launch_bounds__(256) void norm_weight_kernel(const NormParams p) {
    __shared__ float part[16][17];
    const int c = threadIdx.x & 15, r = threadIdx.x >> 4, col = (blockIdx.x + p.vbase) * 16 + c;
    float sum = 0.f;
    if (col < p.width)
        for (int g = r; g < p.groups; g += 16) sum += p.partial[(int64_t)g * p.width + col];
    part[r][c] = sum;
    __syncthreads();
    if (r != 0 || col >= p.width) return;
#pragma unroll
    for (int i = 1; i < 16; ++i) sum += part[i][c];
    p.d_weight[col] = sum;
}

typedef void (*NormKernel)(const NormParams);

// A wave to a row up to 2048 values, a workgroup of 256 threads up to 16384, of 512 up to 32768.
template <typename E, int FMT>
NormKernel pick_forward(int width, unsigned& threads, int& rows) {
    constexpr int ROWS = FMT >= 0 ? 8 : 4;
    rows = ROWS;
    threads = width <= 16384 ? 256 : 512;
    if (width <= 512) return &norm_kernel<E, FMT, 64, 1, ROWS>;
    if (width <= 1024) return &norm_kernel<E, FMT, 64, 2, ROWS>;
    if (width <= 2048) return &norm_kernel<E, FMT, 64, 4, ROWS>;
    if (width <= 4096) return &norm_kernel<E, FMT, 256, 2, ROWS>;
    if (width <= 8192) return &norm_kernel<E, FMT, 256, 4, ROWS>;
    if (width <= 16384) return &norm_kernel<E, FMT, 256, 8, ROWS>;
    return &norm_kernel<E, FMT, 512, 8, ROWS>;
}
template <typename E>
NormKernel pick_backward(int width, unsigned& threads, int& at_once) {
    at_once = width <= 2048 ? 4 : 1;
    threads = width <= 16384 ? 256 : 512;
    if (width <= 512) return &norm_backward_kernel<E, 64, 1>;
    if (width <= 1024) return &norm_backward_kernel<E, 64, 2>;
    if (width <= 2048) return &norm_backward_kernel<E, 64, 4>;
    if (width <= 4096) return &norm_backward_kernel<E, 256, 2>;
    if (width <= 8192) return &norm_backward_kernel<E, 256, 4>;
    if (width <= 16384) return &norm_backward_kernel<E, 256, 8>;
    return &norm_backward_kernel<E, 512, 8>;
}

// Workgroups of the gradient: enough for every CU, few enough that their partial sums cost little.
int partials(int tokens, int width) {
    const int at_once = width <= 2048 ? 4 : 1;
    return std::max(1, std::min(ceil_div(tokens, at_once), kMaxPartials));
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
        kernel = !quant ? pick_forward<float, -1>(a->width, threads, rows)
                        : a->format == DG_MX_E2M1 ? pick_forward<float, DG_MX_E2M1>(a->width, threads, rows) : pick_forward<float, DG_MX_E4M3>(a->width, threads, rows);
    else
        kernel = !quant ? pick_forward<uint16_t, -1>(a->width, threads, rows)
                        : a->format == DG_MX_E2M1 ? pick_forward<uint16_t, DG_MX_E2M1>(a->width, threads, rows) : pick_forward<uint16_t, DG_MX_E4M3>(a->width, threads, rows);
    return launch_op(kernel, ceil_div64(a->tokens, rows), threads, p, reinterpret_cast<hipStream_t>(stream), a->num_cus);
}

int workspace_size(const dg_rms_norm_args* a, int64_t* bytes) {
    NormParams p;
    if (bytes == nullptr) return dg_set_error("dg_rms_norm: null result");
    if (const int rc = check(a, p); rc != DG_OK) return rc;
    *bytes = (int64_t)partials(a->tokens, a->width) * a->width * 4;
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
        !aligned_to(a->d_weight, 4) || !aligned_to(a->workspace, 4) || !aligned_to(a->weight, p.weight_f32 ? 4 : 2))
        return dg_set_error("dg_rms_norm: tensors must be aligned");
    p.groups = partials(a->tokens, a->width);
    if (a->workspace == nullptr || a->workspace_bytes < (int64_t)p.groups * a->width * 4) return dg_set_error("dg_rms_norm: workspace too small");
    p.d_y = a->d_y;
    p.dy_ld = a->d_y_ld;
    p.d_h = a->d_h;
    p.dh_ld = a->d_h_ld;
    p.d_x = a->d_x;
    p.dx_ld = a->d_x_ld;
    p.partial = static_cast<float*>(a->workspace);
    p.d_weight = a->d_weight;
    unsigned threads = 0;
    int at_once = 0;
    const NormKernel kernel = a->dtype == DG_DTYPE_F32 ? pick_backward<float>(a->width, threads, at_once) : pick_backward<uint16_t>(a->width, threads, at_once);
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (const int rc = launch_op(kernel, p.groups, threads, p, st, a->num_cus); rc != DG_OK) return rc;
    return launch_op(&norm_weight_kernel, ceil_div(a->width, 16), 256, p, st, a->num_cus);
}

}  // namespace
}  // namespace dg

extern "C" int dg_rms_norm_workspace_size(const dg_rms_norm_args* args, int64_t* bytes) { return dg::workspace_size(args, bytes); }
extern "C" int dg_rms_norm_forward(const dg_rms_norm_args* args, void* stream) { return dg::forward(args, stream); }
extern "C" int dg_rms_norm_backward(const dg_rms_norm_args* args, void* stream) { return dg::backward(args, stream); }
