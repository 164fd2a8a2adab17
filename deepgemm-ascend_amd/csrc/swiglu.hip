// The gated activation between two products, its output in the rows' type or quantised, its input kept in 8 bits for the backward
// pass, and the gradient from there.
//
//   act = g s u, s = 1 / (1 + exp(-g)), of rows (g | u)
//   d_g = d u s (1 + g (1 - s)), d_u = d g s
//
// A workgroup takes ROWS rows x 512 columns of either half, a wave a row at a time, eight values of each a lane; exponent bytes pass
// through LDS, so that they are read and written as runs of rows.  Bound by the bytes: 32768 x 2048 bf16 with checkpoint 105 to 114 us
// (540 MB, 4.7 to 5.1 TB/s), its gradient and the activation again from there 142 (674 MB, 4.7); 1248 rows, a fifth of them live, to e4m3 4.9.
#include "mx_eight.hpp"
#include "op_launch.hpp"

namespace dg {
namespace {

constexpr int kThreads = 256;

struct GateParams {
    const void* h;
    int64_t h_ld;
    void* act;
    int64_t act_ld;
    int16_t* act_sf;
    int64_t act_sf_ld;
    uint8_t* saved;
    int64_t saved_ld;
    int16_t* saved_sf;
    int64_t saved_sf_ld;
    const void* d_act;
    int64_t da_ld;
    void* d_h;
    int64_t dh_ld;
    const int32_t* m_indices;
    int zero_padding;
    int rows, width;
    int col_tiles;
    int vbase;
};

// By the hardware's exponential of x / ln 2, whose argument's rounding costs up to |x| units of 2^-24 where x is negative (9 for x between -8
// and -2, 30 down to -30); 0 below 2^-126.  With a full exponential 3 units, but few rows take 5.2 us in place of 4.5 (1248 x 2048 bf16)
// and many to e4m3 70.3 in place of 67.4 (fp32 rows the same 152).  Rows of both types have the same fp32 values before they are rounded.
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.f + __expf(-x)); }

// Exponent bytes of a tile, [block][row], to scale factors whose pairs start at any block (`block0`: the tile's first): as runs of two
// rows where pairs do not straddle the halves, byte by byte otherwise.  `blocks`: how many of the 16 exist.
template <int ROWS>
__device__ __forceinline__ void store_scales(const uint8_t (*bytes)[ROWS + 4], int16_t* sf, int64_t ld, int block0, int blocks, int row0, int rows) {
    if (block0 % 2 == 0 && blocks % 2 == 0) {
        for (int e = threadIdx.x; e < blocks / 2 * (ROWS / 2); e += kThreads) {
            const int j = e / (ROWS / 2), r = e % (ROWS / 2) * 2;
            if (row0 + r >= rows) continue;
            // (the leading dimension is even; an odd last row's partner is written 0)
            const u32 one = bytes[2 * j][r] | (u32)bytes[2 * j + 1][r] << 8, two = bytes[2 * j][r + 1] | (u32)bytes[2 * j + 1][r + 1] << 8;
            *reinterpret_cast<u32*>(sf + (int64_t)(block0 / 2 + j) * ld + row0 + r) = one | (row0 + r + 1 < rows ? two << 16 : 0u);
        }
    } else {
        for (int e = threadIdx.x; e < blocks * ROWS; e += kThreads) {
            const int j = e / ROWS, r = e % ROWS, b = block0 + j;
            const int past = rows % 2;   // (the partner of an odd last row)
            if (row0 + r >= rows + past) continue;
            reinterpret_cast<uint8_t*>(sf + (int64_t)(b >> 1) * ld + row0 + r)[b & 1] = row0 + r < rows ? bytes[j][r] : 0;
        }
        // (an odd row count's partner row opens a tile of its own only where rows % ROWS is 0, and then rows is even)
    }
}

template <typename E, int FMT, bool SAVE, int ROWS>
__global__ __launch_bounds__(kThreads) void gate_kernel(const GateParams p) {
    __shared__ uint8_t act_bytes[FMT >= 0 ? 16 : 1][ROWS + 4], gate_bytes[SAVE ? 16 : 1][ROWS + 4], up_bytes[SAVE ? 16 : 1][ROWS + 4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tile = blockIdx.x + p.vbase;
    const int ct = tile % p.col_tiles, row0 = tile / p.col_tiles * ROWS, col = ct * 512 + lane * 8, n = p.width - col;
    constexpr int PER = ROWS / 4, U = PER < 2 ? PER : 2;
#pragma unroll 1
    for (int r0 = 0; r0 < PER; r0 += U) {
        Eight<float> g[U], u[U];
        bool on[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int row = row0 + (r0 + k) * 4 + wave;
            on[k] = row < p.rows && (p.m_indices == nullptr || p.m_indices[row] >= 0);
            const E* const h = reinterpret_cast<const E*>(p.h) + (int64_t)row * p.h_ld + col;
            load_eight(g[k], h, on[k] ? n : 0);
            load_eight(u[k], h + p.width, on[k] ? n : 0);
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int at = (r0 + k) * 4 + wave, row = row0 + at;
            const bool write = row < p.rows && n > 0 && (on[k] || p.zero_padding);
            Eight<float> a;
#pragma unroll
            for (int i = 0; i < 8; ++i) a.v[i] = g[k].v[i] * sigmoid(g[k].v[i]) * u[k].v[i];
            if constexpr (FMT < 0) {
                if (write) store_eight(reinterpret_cast<E*>(p.act) + (int64_t)row * p.act_ld + col, a, n);
            } else {
                // (a width that is a multiple of 32: a lane has eight values or none, and so have a block's others)
                constexpr bool FP4 = FMT == DG_MX_E2M1;
                const u32 s = block_scale<FP4>(a.top());
                if ((lane & 3) == 0) act_bytes[lane >> 2][at] = (uint8_t)(on[k] && n > 0 ? s : 0u);
                if (write) {
                    uint8_t* const to = reinterpret_cast<uint8_t*>(p.act) + (int64_t)row * p.act_ld + (FP4 ? col / 2 : col);
                    if constexpr (FP4) *reinterpret_cast<u32*>(to) = codes_e2m1(a, s);
                    else *reinterpret_cast<i32x2*>(to) = codes_e4m3(a, s);
                }
            }
            if constexpr (SAVE) {
                const u32 sg = block_scale<false>(g[k].top()), su = block_scale<false>(u[k].top());
                if ((lane & 3) == 0) {
                    gate_bytes[lane >> 2][at] = (uint8_t)(on[k] && n > 0 ? sg : 0u);
                    up_bytes[lane >> 2][at] = (uint8_t)(on[k] && n > 0 ? su : 0u);
                }
                if (write) {
                    uint8_t* const to = p.saved + (int64_t)row * p.saved_ld + col;
                    *reinterpret_cast<i32x2*>(to) = codes_e4m3(g[k], sg);
                    *reinterpret_cast<i32x2*>(to + p.width) = codes_e4m3(u[k], su);
                }
            }
        }
    }
    if constexpr (FMT >= 0 || SAVE) {
        __syncthreads();
        const int blocks = min(16, p.width / 32 - ct * 16);
        if constexpr (FMT >= 0) store_scales<ROWS>(act_bytes, p.act_sf, p.act_sf_ld, ct * 16, blocks + blocks % 2, row0, p.rows);
        if constexpr (SAVE) {
            store_scales<ROWS>(gate_bytes, p.saved_sf, p.saved_sf_ld, ct * 16, blocks, row0, p.rows);
            store_scales<ROWS>(up_bytes, p.saved_sf, p.saved_sf_ld, p.width / 32 + ct * 16, blocks, row0, p.rows);
        }
    }
}

template <typename E, bool SAVED, int ROWS>
__global__ __launch_bounds__(kThreads) void gate_backward_kernel(const GateParams p) {
    __shared__ uint16_t gate_pairs[SAVED ? 9 : 1][ROWS + 2], up_pairs[SAVED ? 9 : 1][ROWS + 2];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tile = blockIdx.x + p.vbase;
    const int ct = tile % p.col_tiles, row0 = tile / p.col_tiles * ROWS, col = ct * 512 + lane * 8, n = p.width - col;
    const int up_block = SAVED ? p.width / 32 + ct * 16 : 0;   // the tile's first block of the upper half; its pair may begin in the lower
    if constexpr (SAVED) {
        const int k64 = p.width / 32;   // (2 width / 64)
        for (int e = threadIdx.x; e < 9 * ROWS; e += kThreads) {
            const int j = e / ROWS, r = e % ROWS, gp = ct * 8 + j, up = up_block / 2 + j;
            const bool in = row0 + r < p.rows;
            gate_pairs[j][r] = in && gp < k64 ? (uint16_t)p.saved_sf[(int64_t)gp * p.saved_sf_ld + row0 + r] : 0;
            up_pairs[j][r] = in && up < k64 ? (uint16_t)p.saved_sf[(int64_t)up * p.saved_sf_ld + row0 + r] : 0;
        }
        __syncthreads();
    }
    constexpr int PER = ROWS / 4, U = PER < 2 ? PER : 2;
#pragma unroll 1
    for (int r0 = 0; r0 < PER; r0 += U) {
        Eight<float> g[U], u[U], d[U];
        bool on[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int at = (r0 + k) * 4 + wave, row = row0 + at;
            on[k] = row < p.rows && (p.m_indices == nullptr || p.m_indices[row] >= 0);
            load_eight(d[k], reinterpret_cast<const E*>(p.d_act) + (int64_t)row * p.da_ld + col, on[k] ? n : 0);
            if constexpr (SAVED) {
                i32x2 cg = {0, 0}, cu = {0, 0};
                if (on[k] && n > 0) {
                    const uint8_t* const from = p.saved + (int64_t)row * p.saved_ld + col;
                    cg = *reinterpret_cast<const i32x2*>(from);
                    cu = *reinterpret_cast<const i32x2*>(from + p.width);
                }
                const int bg = lane >> 2, bu = (up_block & 1) + (lane >> 2);
                const float sg = scale_value((gate_pairs[bg >> 1][at] >> (bg & 1 ? 8 : 0)) & 255u);
                const float su = scale_value((up_pairs[bu >> 1][at] >> (bu & 1 ? 8 : 0)) & 255u);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    g[k].v[4 * i] = __builtin_amdgcn_cvt_f32_fp8(cg[i], 0) * sg;
                    g[k].v[4 * i + 1] = __builtin_amdgcn_cvt_f32_fp8(cg[i], 1) * sg;
                    g[k].v[4 * i + 2] = __builtin_amdgcn_cvt_f32_fp8(cg[i], 2) * sg;
                    g[k].v[4 * i + 3] = __builtin_amdgcn_cvt_f32_fp8(cg[i], 3) * sg;
                    u[k].v[4 * i] = __builtin_amdgcn_cvt_f32_fp8(cu[i], 0) * su;
                    u[k].v[4 * i + 1] = __builtin_amdgcn_cvt_f32_fp8(cu[i], 1) * su;
                    u[k].v[4 * i + 2] = __builtin_amdgcn_cvt_f32_fp8(cu[i], 2) * su;
                    u[k].v[4 * i + 3] = __builtin_amdgcn_cvt_f32_fp8(cu[i], 3) * su;
                }
            } else {
                const E* const h = reinterpret_cast<const E*>(p.h) + (int64_t)row * p.h_ld + col;
                load_eight(g[k], h, on[k] ? n : 0);
                load_eight(u[k], h + p.width, on[k] ? n : 0);
            }
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int row = row0 + (r0 + k) * 4 + wave;
            if (!(row < p.rows && n > 0 && (on[k] || p.zero_padding))) continue;
            Eight<float> dg, du, a;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = g[k].v[i], y = u[k].v[i], s = sigmoid(x), xs = x * s;
                du.v[i] = on[k] ? d[k].v[i] * xs : 0.f;
                dg.v[i] = on[k] ? d[k].v[i] * y * (s * (1.f + x * (1.f - s))) : 0.f;
                a.v[i] = on[k] ? xs * y : 0.f;
            }
            E* const to = reinterpret_cast<E*>(p.d_h) + (int64_t)row * p.dh_ld + col;
            store_eight(to, dg, n);
            store_eight(to + p.width, du, n);
            if (p.act != nullptr) store_eight(reinterpret_cast<E*>(p.act) + (int64_t)row * p.act_ld + col, a, n);
        }
    }
}

typedef void (*GateKernel)(const GateParams);

template <typename E, int ROWS>
GateKernel pick_forward(int fmt, bool save) {
    if (fmt == DG_MX_E2M1) return save ? &gate_kernel<E, DG_MX_E2M1, true, ROWS> : &gate_kernel<E, DG_MX_E2M1, false, ROWS>;
    if (fmt == DG_MX_E4M3) return save ? &gate_kernel<E, DG_MX_E4M3, true, ROWS> : &gate_kernel<E, DG_MX_E4M3, false, ROWS>;
    return save ? &gate_kernel<E, -1, true, ROWS> : &gate_kernel<E, -1, false, ROWS>;
}
template <typename E, int ROWS>
GateKernel pick_backward(bool saved) { return saved ? &gate_backward_kernel<E, true, ROWS> : &gate_backward_kernel<E, false, ROWS>; }

template <bool BACKWARD>
int gate_run(const dg_swiglu_args* a, void* stream) {
    if (a == nullptr) return dg_set_error("dg_swiglu: null args");
    if (a->dtype != DG_DTYPE_BF16 && a->dtype != DG_DTYPE_F32) return dg_set_error("dg_swiglu: values are bf16 or fp32");
    if (a->format != -1 && (BACKWARD || (a->format != DG_MX_E2M1 && a->format != DG_MX_E4M3))) return dg_set_error("dg_swiglu: unknown format");
    if (a->rows < 0 || a->width < 0) return dg_set_error("dg_swiglu: negative size");
    if (a->rows > kMaxExtent || a->width > kMaxExtent / 2) return dg_set_error("dg_swiglu: at most 2^30 rows and 2^29 values of a half row");
    const bool quant = a->format != -1, kept = BACKWARD ? a->h == nullptr : a->saved != nullptr, f32 = a->dtype == DG_DTYPE_F32;
    if ((quant || kept) && a->width % 32 != 0) return dg_set_error("dg_swiglu: a quantised width must be a multiple of the block of 32 values");
    if (a->rows == 0 || a->width == 0) return DG_OK;
    if ((!BACKWARD && (a->h == nullptr || a->act == nullptr)) || (quant && a->act_sf == nullptr) || (kept && (a->saved == nullptr || a->saved_sf == nullptr)) ||
        (BACKWARD && (a->d_act == nullptr || a->d_h == nullptr)))
        return dg_set_error("dg_swiglu: null tensor");
    const int64_t act_row = a->format == DG_MX_E2M1 ? a->width / 2 : a->width, full = 2 * (int64_t)a->width;
    if ((a->h != nullptr && a->h_ld < full) || (a->act != nullptr && a->act_ld < act_row) || (quant && a->act_sf_ld < a->rows) ||
        (kept && (a->saved_ld < full || a->saved_sf_ld < a->rows)) || (BACKWARD && (a->d_act_ld < a->width || a->d_h_ld < full)))
        return dg_set_error("dg_swiglu: leading dimension smaller than the row");
    if ((quant && (a->act_sf_ld % 2 != 0 || !aligned_to(a->act_sf, 4))) || (kept && (a->saved_sf_ld % 2 != 0 || !aligned_to(a->saved_sf, 4))))
        return dg_set_error("dg_swiglu: scale factors need an even leading dimension and 4-byte alignment");
    if ((quant && (a->act_ld % 8 != 0 || !aligned_to(a->act, 8))) || (kept && (a->saved_ld % 8 != 0 || !aligned_to(a->saved, 8))))
        return dg_set_error("dg_swiglu: rows of codes must be 8-byte aligned");
    const int64_t size = f32 ? 4 : 2;
    if (!aligned_to(a->h, size) || (!quant && !aligned_to(a->act, size)) || !aligned_to(a->d_act, size) || !aligned_to(a->d_h, size) ||
        !aligned_to(a->m_indices, 4))
        return dg_set_error("dg_swiglu: tensors must be aligned");
    GateParams p = {};
    p.h = a->h; p.h_ld = a->h_ld;
    p.act = a->act; p.act_ld = a->act_ld;
    p.act_sf = a->act_sf; p.act_sf_ld = a->act_sf_ld;
    p.saved = static_cast<uint8_t*>(a->saved); p.saved_ld = a->saved_ld;
    p.saved_sf = a->saved_sf; p.saved_sf_ld = a->saved_sf_ld;
    p.d_act = a->d_act; p.da_ld = a->d_act_ld;
    p.d_h = a->d_h; p.dh_ld = a->d_h_ld;
    p.m_indices = a->m_indices;
    p.zero_padding = a->zero_padding;
    p.rows = a->rows; p.width = a->width;
    p.col_tiles = ceil_div(a->width, 512);
    // tall tiles where they alone give every CU several workgroups
    const bool tall = (int64_t)ceil_div(a->rows, 64) * p.col_tiles >= 1024;
    GateKernel kernel;
    if constexpr (BACKWARD)
        kernel = f32 ? (tall ? pick_backward<float, 64>(kept) : pick_backward<float, 8>(kept)) : (tall ? pick_backward<uint16_t, 64>(kept) : pick_backward<uint16_t, 8>(kept));
    else
        kernel = f32 ? (tall ? pick_forward<float, 64>(a->format, kept) : pick_forward<float, 8>(a->format, kept))
                     : (tall ? pick_forward<uint16_t, 64>(a->format, kept) : pick_forward<uint16_t, 8>(a->format, kept));
    return launch_op(kernel, ceil_div64(a->rows, tall ? 64 : 8) * p.col_tiles, kThreads, p, reinterpret_cast<hipStream_t>(stream), a->num_cus);
}

}  // namespace
}  // namespace dg

extern "C" int dg_swiglu_forward(const dg_swiglu_args* args, void* stream) { return dg::gate_run<false>(args, stream); }
extern "C" int dg_swiglu_backward(const dg_swiglu_args* args, void* stream) { return dg::gate_run<true>(args, stream); }
