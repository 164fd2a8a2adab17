// Microscaled quantisation: blocks of 32 values of a row share a power of two, kept as its exponent byte.
//
//   s = the smallest power of two with max |x| <= L s (L = 6 for e2m1, 448 for e4m3), at least 2^-126,
//   code = x / s rounded to the nearest value of the format, ties to even.
// No value passes the format's largest, so nothing saturates.  With max |x| = m 2^e (1 <= m < 2) and L = l 2^p, s is
// 2^(e - p), or 2^(e - p + 1) where m > l: exact in integers (6 = 1.5 * 2^2, 448 = 1.75 * 2^8).  A maximum too
// small for that (subnormal numbers among them) has s = 2^-126.  A block with an infinity or a NaN gets the exponent byte 255
// (NaN in E8M0), and every product that reads it is NaN.
//
// Scale factors come out as the GEMMs read them: int16 pairs of exponent bytes (even block low), [k64][ld], rows
// contiguous.
#include "op_launch.hpp"
#include "mx_eight.hpp"

namespace dg {
namespace {

constexpr int kThreads = 256;

struct MxParams {
    const void* x;             // [batches][rows][ld] bf16 or fp32 (quantise: input, dequantise: output)
    void* codes;               // [batches][rows][codes_ld bytes]
    int16_t* sf;               // [batches][k64][sf_ld]
    int64_t x_ld, x_bs;        // elements
    int64_t codes_ld, codes_bs;   // bytes
    int64_t sf_ld, sf_bs;
    int batches, rows, k;
    int row_tiles, col_tiles;
    int vbase;
};

// A workgroup quantises ROWS rows x 512 values, a wave a row at a time: eight values a lane (1 KB of bf16 a wave), the
// block's maximum over four lanes, and the exponent bytes of the tile collected in LDS so that they leave as runs
// of rows.  Bound by the bytes of x; four rows of a wave are in flight.  7168 x 16384 bf16 to e2m1 61 to 73 us (298 MB: 4.1 to 4.9
// TB/s; a copy of as many bytes 58), 777 x 1440 fp32 to e4m3 3.4.
template <typename E, bool FP4, int ROWS>
__global__ __launch_bounds__(kThreads) void mx_quantize_kernel(const MxParams p) {
    __shared__ uint16_t pairs[8][ROWS + 2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int t = blockIdx.x + p.vbase;
    const int ct = t % p.col_tiles;
    t /= p.col_tiles;
    const int rt = t % p.row_tiles, batch = t / p.row_tiles;
    const int row0 = rt * ROWS, col = ct * 512 + lane * 8;
    const bool on = col < p.k, paired = col + 32 < p.k;
    const E* const x = reinterpret_cast<const E*>(p.x) + batch * p.x_bs + col;
    uint8_t* const codes = reinterpret_cast<uint8_t*>(p.codes) + batch * p.codes_bs + (FP4 ? col / 2 : col);
    constexpr int PER = ROWS / 4, U = PER < 4 ? PER : 4;
#pragma unroll 1
    for (int r0 = 0; r0 < PER; r0 += U) {
        Eight<E> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int row = row0 + (r0 + u) * 4 + wave;
            v[u].zero();
            if (on && row < p.rows) v[u].load(x + (int64_t)row * p.x_ld);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = (r0 + u) * 4 + wave, row = row0 + at;
            u32 a = v[u].top();
            a = max(a, dpp<kXor1>(a));
            a = max(a, dpp<kXor2>(a));
            const u32 s = scale_byte<FP4>(a), other = dpp<kMirror8>(s);
            if ((lane & 7) == 0) pairs[lane >> 3][at] = (uint16_t)(s | (paired ? other << 8 : 0u));
            if (!on || row >= p.rows) continue;
            uint8_t* const d = codes + (int64_t)row * p.codes_ld;
            // (s lies in [1, 254 - p] for finite blocks: 2^(s - 127) and its reciprocal are normal numbers)
            if constexpr (FP4) {
                const u32 c = v[u].e2m1(__builtin_bit_cast(float, s << 23));
                *reinterpret_cast<u32*>(d) = s == 255u ? 0u : c;
            } else {
                const i32x2 c = v[u].e4m3(__builtin_bit_cast(float, (254u - s) << 23));
                *reinterpret_cast<i32x2*>(d) = s == 255u ? i32x2{0, 0} : c;
            }
        }
    }
    __syncthreads();
    // two rows a thread: the leading dimension is even, and an odd last row's partner is written 0
    const int k64 = ceil_div(p.k, 64);
    int16_t* const sf = p.sf + batch * p.sf_bs;
    for (int e = tid; e < 8 * (ROWS / 2); e += kThreads) {
        const int j = e / (ROWS / 2), r = e % (ROWS / 2) * 2, kj = ct * 8 + j;
        if (kj >= k64 || row0 + r >= p.rows) continue;
        const u32 w = pairs[j][r] | (row0 + r + 1 < p.rows ? (u32)pairs[j][r + 1] << 16 : 0u);
        *reinterpret_cast<u32*>(sf + (int64_t)kj * p.sf_ld + row0 + r) = w;
    }
}

// The values of codes under their scale factors; the same tiles, with the exponent pairs read into LDS first.  Bound by the bytes
// written: 7168 x 16384 e2m1 to bf16 53 to 68 us, 777 x 1440 e4m3 to bf16 4.
template <typename E, bool FP4, int ROWS>
__global__ __launch_bounds__(kThreads) void mx_dequantize_kernel(const MxParams p) {
    __shared__ uint16_t pairs[8][ROWS + 2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int t = blockIdx.x + p.vbase;
    const int ct = t % p.col_tiles;
    t /= p.col_tiles;
    const int rt = t % p.row_tiles, batch = t / p.row_tiles;
    // A lane's eight values: side by side, or (fp32) four in either half of the tile, so that the wave's stores are whole runs of
    // 1 KB (7168 x 16384 e2m1: 128 us, side by side 155).
    constexpr bool SPLIT = sizeof(E) == 4;
    const int row0 = rt * ROWS, col = ct * 512 + lane * (SPLIT ? 4 : 8), k64 = ceil_div(p.k, 64);
    const int16_t* const sf = p.sf + batch * p.sf_bs;
    for (int e = tid; e < 8 * ROWS; e += kThreads) {
        const int j = e / ROWS, r = e % ROWS, kj = ct * 8 + j;
        pairs[j][r] = kj < k64 && row0 + r < p.rows ? (uint16_t)sf[(int64_t)kj * p.sf_ld + row0 + r] : 0;
    }
    const uint8_t* const codes = reinterpret_cast<const uint8_t*>(p.codes) + batch * p.codes_bs;
    E* const x = reinterpret_cast<E*>(const_cast<void*>(p.x)) + batch * p.x_bs;
    constexpr int PER = ROWS / 4, U = PER < 4 ? PER : 4;
    typedef typename std::conditional<FP4, u32, i32x2>::type code_t;
    const bool on = col < p.k, on2 = SPLIT && col + 256 < p.k;
    __syncthreads();
#pragma unroll 1
    for (int r0 = 0; r0 < PER; r0 += U) {
        code_t c[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int row = row0 + (r0 + u) * 4 + wave;
            c[u] = code_t{};
            if (!on || row >= p.rows) continue;
            const uint8_t* const at = codes + (int64_t)row * p.codes_ld + (FP4 ? col / 2 : col);
            if constexpr (!SPLIT) {
                c[u] = *reinterpret_cast<const code_t*>(at);
            } else if constexpr (FP4) {
                c[u] = *reinterpret_cast<const uint16_t*>(at) | (on2 ? (u32)*reinterpret_cast<const uint16_t*>(at + 128) << 16 : 0u);
            } else {
                c[u] = i32x2{*reinterpret_cast<const int*>(at), on2 ? *reinterpret_cast<const int*>(at + 256) : 0};
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = (r0 + u) * 4 + wave, row = row0 + at;
            if (!on || row >= p.rows) continue;
            // 2^(s - 127); exponent byte 0 is 2^-127, 255 is NaN
            auto scale_of = [&](int block) {
                const u32 s = (pairs[block >> 1][at] >> (block & 1 ? 8 : 0)) & 255u;
                return __builtin_bit_cast(float, s == 255u ? 0x7fc00000u : s == 0u ? 0x00400000u : s << 23);
            };
            const float scale = scale_of(SPLIT ? lane >> 3 : lane >> 2), scale2 = SPLIT ? scale_of(8 + (lane >> 3)) : scale;
            float v[8];
            if constexpr (FP4) {
                typedef float f2 __attribute__((ext_vector_type(2)));
                const f2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u], 1.f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u], 1.f, 1);
                const f2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u], 1.f, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u], 1.f, 3);
                v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1]; v[4] = d[0]; v[5] = d[1]; v[6] = e[0]; v[7] = e[1];
            } else {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    v[4 * h] = __builtin_amdgcn_cvt_f32_fp8(c[u][h], 0);
                    v[4 * h + 1] = __builtin_amdgcn_cvt_f32_fp8(c[u][h], 1);
                    v[4 * h + 2] = __builtin_amdgcn_cvt_f32_fp8(c[u][h], 2);
                    v[4 * h + 3] = __builtin_amdgcn_cvt_f32_fp8(c[u][h], 3);
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] *= i < 4 ? scale : scale2;
            E* const to = x + (int64_t)row * p.x_ld + col;
            if constexpr (SPLIT) {
                *reinterpret_cast<f32x4_any*>(to) = f32x4{v[0], v[1], v[2], v[3]};
                if (on2) *reinterpret_cast<f32x4_any*>(to + 256) = f32x4{v[4], v[5], v[6], v[7]};
            } else {
                *reinterpret_cast<i32x4_half*>(to) = i32x4{(int)pack_bf16x2(v[0], v[1]), (int)pack_bf16x2(v[2], v[3]),
                                                           (int)pack_bf16x2(v[4], v[5]), (int)pack_bf16x2(v[6], v[7])};
            }
        }
    }
}

typedef void (*MxKernel)(const MxParams);

template <bool QUANT, typename E>
MxKernel pick(bool fp4, bool tall) {
    if constexpr (QUANT) {
        if (fp4) return tall ? &mx_quantize_kernel<E, true, 64> : &mx_quantize_kernel<E, true, 8>;
        return tall ? &mx_quantize_kernel<E, false, 64> : &mx_quantize_kernel<E, false, 8>;
    } else {
        if (fp4) return tall ? &mx_dequantize_kernel<E, true, 64> : &mx_dequantize_kernel<E, true, 8>;
        return tall ? &mx_dequantize_kernel<E, false, 64> : &mx_dequantize_kernel<E, false, 8>;
    }
}

template <bool QUANT>
int mx_run(const dg_mx_args* a, void* stream) {
    if (a == nullptr) return dg_set_error("dg_mx: null args");
    if (a->format != DG_MX_E2M1 && a->format != DG_MX_E4M3) return dg_set_error("dg_mx: unknown format");
    if (a->x_dtype != DG_DTYPE_BF16 && a->x_dtype != DG_DTYPE_F32) return dg_set_error("dg_mx: values are bf16 or fp32");
    if (a->batches < 0 || a->rows < 0 || a->k < 0) return dg_set_error("dg_mx: negative size");
    if (a->rows > kMaxExtent || a->k > kMaxExtent) return dg_set_error("dg_mx: at most 2^30 rows and values of a row");
    if (a->k % 32 != 0) return dg_set_error("dg_mx: K must be a multiple of the block of 32 values");
    if (a->batches == 0 || a->rows == 0 || a->k == 0) return DG_OK;
    const bool fp4 = a->format == DG_MX_E2M1, f32 = a->x_dtype == DG_DTYPE_F32;
    const int64_t code_bytes = fp4 ? a->k / 2 : a->k;
    if (a->x == nullptr || a->codes == nullptr || a->sf == nullptr) return dg_set_error("dg_mx: null tensor");
    if (a->x_ld < a->k || a->codes_ld < code_bytes || a->sf_ld < a->rows) return dg_set_error("dg_mx: leading dimension smaller than the row");
    if (a->sf_ld % 2 != 0 || a->sf_batch_stride % 2 != 0 || !aligned_to(a->sf, 4))
        return dg_set_error("dg_mx: scale factors need an even leading dimension and 4-byte alignment");
    if (a->codes_ld % 8 != 0 || a->codes_batch_stride % 8 != 0 || !aligned_to(a->codes, 8))
        return dg_set_error("dg_mx: rows of codes must be 8-byte aligned");
    if (!aligned_to(a->x, f32 ? 4 : 2)) return dg_set_error("dg_mx: values must be aligned");
    MxParams p = {};
    p.x = a->x; p.codes = a->codes; p.sf = a->sf;
    p.x_ld = a->x_ld; p.x_bs = a->x_batch_stride;
    p.codes_ld = a->codes_ld; p.codes_bs = a->codes_batch_stride;
    p.sf_ld = a->sf_ld; p.sf_bs = a->sf_batch_stride;
    p.batches = a->batches; p.rows = a->rows; p.k = a->k;
    p.col_tiles = ceil_div(a->k, 512);
    // tall tiles where they alone give every CU several workgroups
    const bool tall = (int64_t)ceil_div(a->rows, 64) * p.col_tiles * a->batches >= 1024;
    p.row_tiles = ceil_div(a->rows, tall ? 64 : 8);
    const int64_t grid = (int64_t)p.row_tiles * p.col_tiles * a->batches;
    return launch_op(f32 ? pick<QUANT, float>(fp4, tall) : pick<QUANT, uint16_t>(fp4, tall), grid, kThreads, p,
                     reinterpret_cast<hipStream_t>(stream), a->num_cus);
}

}  // namespace
}  // namespace dg

extern "C" int dg_mx_quantize(const dg_mx_args* args, void* stream) { return dg::mx_run<true>(args, stream); }
extern "C" int dg_mx_dequantize(const dg_mx_args* args, void* stream) { return dg::mx_run<false>(args, stream); }
