// Products of few rows with e2m1 weights: a token, or an expert's few tokens, against all rows of w.
//
//   D[m][n] = sum over blocks b of 2^(sa[m][b] + sw[n][b] - 254) sum_{k in b} a[m][k] w[n][k]
// Bound by the bytes of w, which is read once, straight into registers: a lane of v_mfma_scale_f32_16x16x128_f8f6f4 holds the
// 16 bytes of one block of 32 codes of one row, so a wave's load is 16 rows x 64 bytes as they lie in memory, no two lanes
// need the same bytes, and neither LDS nor a barrier stands between memory and the matrix unit.  A wave owns 32 rows of w and
// a range of K, two to eight steps of 128 ahead in registers; the waves of a workgroup that share rows join their sums in LDS, in
// order.  The few rows of a come the same way (from the caches).  One row of 4096 values against 7168: 6 to 7 us where the 15.6 MB
// alone would take 3, a launch whose steps wait for each other: one round of loads (a wave's four steps of w and behind them x, which
// is there when all of them are), the quantisation, a barrier, the products and the join of eight waves' sums.  32 x 8 pairs over 32 experts, N = 2048 K = 4096: 30 to
// 33 us (143 MB: 4.3 to 4.8 TB/s).
//
// The rows of a are e2m1 codes (an M-grouped layout: each expert's rows with its weights), or a few rows of bf16 / fp32 values
// that every workgroup quantises into LDS, a block of 32 a thread, once its first weights have arrived too (loads return in order, and
// the values are asked for last).
#include "gemm_kernel.hpp"
#include "op_launch.hpp"
#include "mx_scale.hpp"

namespace dg {
namespace {

struct MxProductParams {
    const uint8_t* a;          // codes [rows][lda], or values
    const uint8_t* w;          // codes [groups][n][ldw]
    uint8_t* d;
    const uint16_t *sfa, *sfw; // [k64][ld]; sfa: codes only
    const int* psum;           // M-grouped layout (codes); values are one group of m rows
    int m, n, k, groups, alignment;
    int64_t lda, ldw, ldd;     // bytes, bytes, elements
    int64_t w_bs, sfw_bs;      // bytes, int16 elements
    int64_t sfa_ld, sfw_ld;
    int f32, accumulate;       // of D
    int strips;
    int vbase;
};

enum Rows : int { kCodes = 0, kBf16Rows = 1, kF32Rows = 2 };

// Quantised rows in LDS: codes [row][kPad + K / 2], then exponent bytes [row][K / 32].  (The pad sets the rows that a read of 16
// rows x 16 bytes touches 16 bytes apart.)
constexpr int kPad = 16;
__host__ __device__ __forceinline__ int row_pitch(int k) { return k / 2 + kPad; }
__host__ __device__ __forceinline__ int rows_lds(int m, int k) { return align_up(m * (row_pitch(k) + k / 32), 16); }
// Values quantised inside, at most (17.6 KB of LDS).  Every workgroup quantises all of them; beyond, the quantiser's own launch
// costs less (with the quantiser's launch in brackets, us: 1x7168x4096 7.3 (9.5), 4x7168x4096 8.3 (9.6), 4x2112x7168 9.4
// (10.6), 8x2112x7168 10.5 (10.7), 16x7168x4096 10.4 (10.0), 4x7168x16384 21.6 (21.1)).
constexpr int kInside = 32768;

template <typename E, int THREADS>
__device__ __forceinline__ void quantise_rows(const MxProductParams& p, uint8_t* lds) {
    typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
    typedef int i32x4_any __attribute__((ext_vector_type(4), aligned(4)));
    const int blocks = p.k / 32;
    for (int b = threadIdx.x; b < p.m * blocks; b += THREADS) {
        const int row = b / blocks, block = b - row * blocks;
        const uint8_t* const x = p.a + row * p.lda + block * 32 * (int)sizeof(E);
        float v[32];
        uint32_t top = 0;
        if constexpr (sizeof(E) == 2) {
            i32x4 w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = reinterpret_cast<const i32x4_any*>(x)[i];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const uint32_t u = (uint32_t)w[i / 4][i % 4];
                v[2 * i] = __builtin_bit_cast(float, u << 16);
                v[2 * i + 1] = __builtin_bit_cast(float, u & 0xffff0000u);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const f32x4 w = reinterpret_cast<const f32x4_any*>(x)[i];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[4 * i + e] = w[e];
            }
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) top = max(top, __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu);
        const uint32_t s = scale_byte<true>(top);
        const float f = __builtin_bit_cast(float, s << 23);
        i32x4 codes;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t c = 0;
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[8 * j], v[8 * j + 1], f, 0);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[8 * j + 2], v[8 * j + 3], f, 1);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[8 * j + 4], v[8 * j + 5], f, 2);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[8 * j + 6], v[8 * j + 7], f, 3);
            codes[j] = s == 255u ? 0 : (int)c;
        }
        *reinterpret_cast<i32x4*>(lds + row * row_pitch(p.k) + block * 16) = codes;
        lds[p.m * row_pitch(p.k) + row * blocks + block] = (uint8_t)s;
    }
}

constexpr int kNB = 2;         // 16-row blocks of w of a wave
constexpr int kStrip = 16 * kNB;

// MT: 16-row blocks of a in flight together; DEPTH: steps of 128 values of K ahead.
template <int ROWS, int MT, int DEPTH, int KS>
__device__ __forceinline__ void product_rows(const MxProductParams& p, const uint8_t* a, const uint16_t* sfa, const uint8_t* w,
                                             const uint16_t* sfw, uint8_t* d, int rows, int n0, float* red, uint8_t* lds) {
    constexpr bool kLoaded = ROWS == kCodes;                                 // (else in LDS)
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int part = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);       // of K (KS waves share the strip)
    const int blocks = p.k / 32, steps = ceil_div(blocks, 4), per = ceil_div(steps, KS);
    const int s0 = part * per, s1 = min(steps, s0 + per);
    const int cols = min(kStrip, p.n - n0);
    const __amdgpu_buffer_rsrc_t rs_w = make_rsrc(w, (int64_t)cols * p.ldw);
    const __amdgpu_buffer_rsrc_t rs_a = make_rsrc(a, kLoaded ? (int64_t)rows * p.lda : 0);
    const int k64 = ceil_div(p.k, 64);
    // Scales: one load holds the dwords (a row pair's exponents of 64 K) of all the wave's rows for several steps, lane l the pair
    // l % P of the (l / P)-th 64 K, and every lane fetches its own from there.  (With a load for each 16 rows and step, 32 x 8
    // pairs over 32 experts, N = 2048 K = 4096, took 40 us in place of 37; without scales 33, without rows of a too 28.)
    constexpr int kPairsW = kStrip / 2, kStepsW = 64 / kPairsW / 2, kPairsA = 8 * MT, kStepsA = 64 / kPairsA / 2;
    static_assert(DEPTH % kStepsW == 0 && DEPTH % kStepsA == 0, "steps in flight");
    const __amdgpu_buffer_rsrc_t rs_sw = make_rsrc(sfw, ((int64_t)(k64 - 1) * p.sfw_ld + align_up(cols, 2)) * 2);
    const __amdgpu_buffer_rsrc_t rs_sa = make_rsrc(sfa, kLoaded ? ((int64_t)(k64 - 1) * p.sfa_ld + align_up(rows, 2)) * 2 : 0);
    const int shift = 8 * ((r & 1) * 2 + (g & 1));
    const uint32_t vsw = lane % kPairsW * 2 < cols ? (uint32_t)((lane / kPairsW * p.sfw_ld + lane % kPairsW * 2) * 2) : kOOBOffset;
    const uint32_t vsa = lane % kPairsA * 2 < rows ? (uint32_t)((lane / kPairsA * p.sfa_ld + lane % kPairsA * 2) * 2) : kOOBOffset;
    uint32_t vw[kNB], va[MT];                       // (rows past the end: out of range, zeros)
#pragma unroll
    for (int j = 0; j < kNB; ++j) {
        const bool on = 16 * j + r < cols;
        vw[j] = on ? (uint32_t)((16 * j + r) * p.ldw + 16 * g) : kOOBOffset;
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const bool on = 16 * i + r < rows;
        va[i] = on ? (uint32_t)((16 * i + r) * p.lda + 16 * g) : kOOBOffset;
    }
    i32x4 fw[DEPTH][kNB], fa[DEPTH][MT];
    int sw[DEPTH / kStepsW], sa[DEPTH / kStepsA];
    auto load = [&](auto slot, int s) {
        constexpr int S = decltype(slot)::value;
        const bool on = s < s1 && 4 * s + g < blocks;   // (past K: zeros)
        const int step_w = __builtin_amdgcn_readfirstlane(s * 64);
#pragma unroll
        for (int j = 0; j < kNB; ++j)
            fw[S][j] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rs_w, on ? vw[j] : kOOBOffset, step_w, 0));
        if constexpr (kLoaded) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
                fa[S][i] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rs_a, on ? va[i] : kOOBOffset, step_w, 0));
        }
    };
    // the scales that slot S is the last to need (s: its next step), or, at the start, those that it is the first to need
    auto load_scales = [&](auto slot, int s, auto start) {
        constexpr int S = decltype(slot)::value;
        constexpr bool kStart = decltype(start)::value != 0;
        if constexpr ((S + (kStart ? 0 : 1)) % kStepsW == 0) {
            const int first = s - (kStart ? 0 : kStepsW - 1);
            sw[S / kStepsW] = (int)__builtin_amdgcn_raw_buffer_load_b32(rs_sw, vsw, __builtin_amdgcn_readfirstlane((int)(first * 4 * p.sfw_ld)), 0);
        }
        if constexpr (kLoaded && (S + (kStart ? 0 : 1)) % kStepsA == 0) {
            const int first = s - (kStart ? 0 : kStepsA - 1);
            sa[S / kStepsA] = (int)__builtin_amdgcn_raw_buffer_load_b32(rs_sa, vsa, __builtin_amdgcn_readfirstlane((int)(first * 4 * p.sfa_ld)), 0);
        }
    };
    // Exponent byte of block g of row 16 `blk` + r in the step-th step of a load (0 past K, where the codes are zeros too)
    auto scale_of = [&](int held, int pairs, int step, int blk, bool on) -> int {
        const int from = (2 * step + (g >> 1)) * pairs + 8 * blk + (r >> 1);
        const int v = __builtin_amdgcn_ds_bpermute(from * 4, held);
        return on ? (v >> shift) & 255 : 0;
    };
    f32x4 acc[kNB][MT];
#pragma unroll
    for (int j = 0; j < kNB; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](auto slot, int s) {
        constexpr int S = decltype(slot)::value;
        const bool on = 4 * s + g < blocks;
        int scale_w[kNB];
#pragma unroll
        for (int j = 0; j < kNB; ++j) scale_w[j] = scale_of(sw[S / kStepsW], kPairsW, S % kStepsW, j, on);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            i32x4 c = {0, 0, 0, 0};
            int scale = 0;
            if constexpr (kLoaded) {
                c = fa[S][i];
                scale = scale_of(sa[S / kStepsA], kPairsA, S % kStepsA, i, on);
            } else if (r < rows && on) {
                c = *reinterpret_cast<const i32x4*>(lds + r * row_pitch(p.k) + s * 64 + g * 16);
                scale = lds[rows * row_pitch(p.k) + r * blocks + 4 * s + g];
            }
            const i32x8 fa8 = {c[0], c[1], c[2], c[3], 0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < kNB; ++j) {
                const i32x4 b = fw[S][j];
                const i32x8 fb8 = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
                acc[j][i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb8, fa8, acc[j][i], kFmtE2M1, kFmtE2M1, 0, scale_w[j], 0, scale);
            }
        }
    };
    static_for<DEPTH>([&](auto s) {
        load_scales(s, s0 + decltype(s)::value, Int<1>{});
        load(s, s0 + decltype(s)::value);
        __builtin_amdgcn_sched_barrier(0);
    });
    if constexpr (!kLoaded) {
        if constexpr (ROWS == kBf16Rows) quantise_rows<uint16_t, 64 * KS>(p, lds);
        else quantise_rows<float, 64 * KS>(p, lds);
        __syncthreads();
    }
    for (int s = s0; s < s1; s += DEPTH) {
        static_for<DEPTH>([&](auto x) {
            multiply(x, s + decltype(x)::value);   // (a step past the range holds zero weights and adds nothing)
            __builtin_amdgcn_sched_barrier(0);
            load(x, s + DEPTH + decltype(x)::value);
            load_scales(x, s + DEPTH + decltype(x)::value, Int<0>{});
            __builtin_amdgcn_sched_barrier(0);
        });
    }
    // sums of the K ranges, in order: red[part][block][lane]
    if constexpr (KS > 1) {
#pragma unroll
        for (int j = 0; j < kNB; ++j)
#pragma unroll
            for (int i = 0; i < MT; ++i) *reinterpret_cast<f32x4*>(red + ((part * kNB * MT + j * MT + i) * 64 + lane) * 4) = acc[j][i];
        __syncthreads();
        if (part != 0) return;
        for (int w2 = 1; w2 < KS; ++w2)
#pragma unroll
            for (int j = 0; j < kNB; ++j)
#pragma unroll
                for (int i = 0; i < MT; ++i) acc[j][i] += *reinterpret_cast<const f32x4*>(red + ((w2 * kNB * MT + j * MT + i) * 64 + lane) * 4);
    }
    // lane (r, g): columns 4 g .. + 3 of block j, row 16 i + r of a
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int row = 16 * i + r;
        if (row >= rows) continue;
#pragma unroll
        for (int j = 0; j < kNB; ++j) {
            const int n = n0 + 16 * j + 4 * g, live = min(4, p.n - n);
            const int64_t at = row * p.ldd + n;
            f32x4 v = acc[j][i];
            if (p.f32) {
                float* const out = reinterpret_cast<float*>(d) + at;
                for (int x = 0; x < live; ++x) out[x] = p.accumulate ? out[x] + v[x] : v[x];
            } else {
                uint16_t* const out = reinterpret_cast<uint16_t*>(d) + at;
                if (!p.accumulate && live == 4 && (reinterpret_cast<uintptr_t>(out) & 7) == 0) {
                    *reinterpret_cast<i32x2*>(out) = i32x2{(int)pack_bf16x2(v[0], v[1]), (int)pack_bf16x2(v[2], v[3])};
                } else {
                    for (int x = 0; x < live; ++x) out[x] = f32_to_bf16_rne(p.accumulate ? v[x] + bf16_to_f32(out[x]) : v[x]);
                }
            }
        }
    }
}

// Zeros in columns [n0, n0 + cols) of rows first, first + step, ... below end, by a workgroup: four columns a thread.
template <int THREADS, int COLS>
__device__ __forceinline__ void clear_rows(const MxProductParams& p, int64_t first, int64_t end, int step, int n0, int cols) {
    constexpr int PER = COLS / 4;
    const int c = threadIdx.x % PER * 4, live = min(4, cols - c);
    for (int64_t row = first + (int64_t)(threadIdx.x / PER) * step; row < end; row += (int64_t)(THREADS / PER) * step) {
        const int64_t at = row * p.ldd + n0 + c;
        if (p.f32) {
            float* const d = reinterpret_cast<float*>(p.d) + at;
            if (live == 4 && (reinterpret_cast<uintptr_t>(d) & 15) == 0) *reinterpret_cast<f32x4*>(d) = f32x4{0.f, 0.f, 0.f, 0.f};
            else for (int x = 0; x < live; ++x) d[x] = 0.f;
        } else {
            uint16_t* const d = reinterpret_cast<uint16_t*>(p.d) + at;
            if (live == 4 && (reinterpret_cast<uintptr_t>(d) & 7) == 0) *reinterpret_cast<i32x2*>(d) = i32x2{0, 0};
            else for (int x = 0; x < live; ++x) d[x] = 0;
        }
    }
}

// Chunk `x` of 64 rows among those past their group's first, groups in order: its group and number (0: there is none).  A lane
// takes four groups, so that up to 256 are read at once (most launches have no such chunk, and their workgroups only look).
__device__ __forceinline__ int later_chunk(const MxProductParams& p, int x, int& group) {
    const int lane = threadIdx.x & 63;
    for (int base = 0; base < p.groups; base += 256) {
        const int e = base + 4 * lane;
        int start = e > 0 && e < p.groups ? max(0, align_up(p.psum[e - 1], p.alignment)) : 0, later[4], sum = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int end = e + j < p.groups ? p.psum[e + j] : start;
            later[j] = max(0, ceil_div(min(p.m, end) - start, 64) - 1);
            start = max(0, align_up(end, p.alignment));
            sum += later[j];
        }
        int incl = sum;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int v = __shfl_up(incl, off, 64);
            if (lane >= off) incl += v;
        }
        const uint64_t hit = __ballot(x < incl);
        if (hit != 0) {
            const int src = __builtin_ctzll(hit);
            x -= __shfl(incl - sum, src, 64);
            for (int j = 0; j < 4; ++j) {
                const int n = __shfl(later[j], src, 64);
                if (x < n) {
                    group = base + 4 * src + j;
                    break;
                }
                x -= n;
            }
            return x + 1;
        }
        x -= __shfl(incl, 63, 64);
    }
    return 0;
}

template <int ROWS, int KS>
__global__ __launch_bounds__(64 * KS) void mx_product_kernel(const MxProductParams p) {
    __shared__ __attribute__((aligned(16))) float red[KS > 1 ? KS * kNB * (ROWS == kCodes ? 4 : 1) * 256 : 4];
    // (strips dealt over the XCDs one by one: an expert without rows, or with many, is then spread over all of them; with an
    // expert's strips on one XCD 16 x 8 pairs over 64 experts took 49 us in place of 41.  Four strips to a workgroup, whose
    // waves would share their rows of a in the CU's cache, were no faster, and 128 x 8 pairs over 32 77 us in place of 64.)
    const int t = blockIdx.x + p.vbase;
    int e = t / p.strips, chunk = 0;
    const int n0 = (t - e * p.strips) * kStrip;
    if (ROWS == kCodes && e >= p.groups) {
        // (workgroups of their own, behind the others: 256 rows of one of 32 experts, 16 of the others, N = 2048 K = 4096 50 us where a
        // strip's one workgroup took its chunks in turn for 77; 2048 rows in one 51 and 467)
        chunk = __builtin_amdgcn_readfirstlane(later_chunk(p, e - p.groups, e));
        e = __builtin_amdgcn_readfirstlane(e);
        if (chunk == 0) return;
    }
    const uint8_t* const w = p.w + (int64_t)e * p.w_bs + (int64_t)n0 * p.ldw;
    const uint16_t* const sfw = p.sfw + (int64_t)e * p.sfw_bs + n0;
    extern __shared__ __attribute__((aligned(16))) uint8_t rows_in_lds[];
    if constexpr (ROWS != kCodes) {
        product_rows<ROWS, 1, KS == 8 ? 8 : 4, KS>(p, nullptr, nullptr, w, sfw, p.d, p.m, n0, red, rows_in_lds);
    } else {
        const int first = __builtin_amdgcn_readfirstlane(e == 0 ? 0 : max(0, align_up(p.psum[e - 1], p.alignment)));
        const int rows = __builtin_amdgcn_readfirstlane(min(p.m, p.psum[e]) - first), end = min(p.m, align_up(p.psum[e], p.alignment));
        const int esize = p.f32 ? 4 : 2;
        // (every 64 rows of an expert read its weights, the later ones from the caches; with 32 at a time, 128 x 8 pairs over 32
        // experts took 64 us in place of 56)
        const int m0 = 64 * chunk, live = min(64, rows - m0);
        if (live > 0) {
            const uint8_t* const a = p.a + (int64_t)(first + m0) * p.lda;
            const uint16_t* const sfa = p.sfa + first + m0;
            uint8_t* const d = p.d + (int64_t)(first + m0) * p.ldd * esize;
            if (live <= 16) product_rows<ROWS, 1, 8, KS>(p, a, sfa, w, sfw, d, live, n0, red, nullptr);
            else if (live <= 32) product_rows<ROWS, 2, 4, KS>(p, a, sfa, w, sfw, d, live, n0, red, nullptr);
            else product_rows<ROWS, 4, 2, KS>(p, a, sfa, w, sfw, d, live, n0, red, nullptr);
        }
        if (chunk > 0) return;
        // padding rows of the group, and every groups-th row past the last group, are zeros
        const int cols = min(kStrip, p.n - n0);
        clear_rows<64 * KS, kStrip>(p, first + max(rows, 0), end, 1, n0, cols);
        clear_rows<64 * KS, kStrip>(p, (int64_t)max(0, align_up(p.psum[p.groups - 1], p.alignment)) + e, p.m, p.groups, n0, cols);
    }
}

// Waves that share a strip: as many as give the card about eight waves a CU, while each keeps four steps.  (Codes: at most four,
// eight would share a SIMD's registers by twos and spill.)
int k_waves(int64_t strips, int k, bool codes) {
    int ks = 1;
    while (ks < (codes ? 4 : 8) && strips * ks < 2048 && ceil_div(k, 128) >= 4 * ks) ks *= 2;
    return ks;
}

template <int ROWS>
int launch_product(MxProductParams p, hipStream_t st, int cus) {
    p.strips = ceil_div(p.n, kStrip);
    // (chunks of 64 rows past a group's first: m / 64 at most)
    const int64_t grid = (int64_t)p.strips * (p.groups + (ROWS == kCodes ? p.m / 64 : 0));
    if (grid > 0x7fffffffLL) return dg_set_error("dg_mx_gemm: too many workgroups");
    const unsigned lds = ROWS == kCodes ? 0 : (unsigned)rows_lds(p.m, p.k);
    const int ks = k_waves((int64_t)p.strips * p.groups, p.k, ROWS == kCodes);
    if (ks == 1) return launch_op(mx_product_kernel<ROWS, 1>, grid, 64, p, st, cus, lds);
    if (ks == 2) return launch_op(mx_product_kernel<ROWS, 2>, grid, 128, p, st, cus, lds);
    if constexpr (ROWS != kCodes)
        if (ks == 8) return launch_op(mx_product_kernel<ROWS, 8>, grid, 512, p, st, cus, lds);
    return launch_op(mx_product_kernel<ROWS, 4>, grid, 256, p, st, cus, lds);
}

bool span32(int64_t rows, int64_t ld_bytes) { return rows * ld_bytes < 0x40000000LL; }

}  // namespace

// csrc/gemm.hip: an M-grouped psum GEMM of e2m1 rows, a few to an expert.  Whether this kernel serves it.
bool mx_experts_fit(const dg_gemm_args& a) {
    return a.gemm_type == kMGroupedPsum && a.kind == kFP4FP4 && a.k > 0 && a.k % 32 == 0 && a.m <= (int64_t)64 * a.num_groups &&
           (a.d_dtype == DG_DTYPE_BF16 || a.d_dtype == DG_DTYPE_F32) && a.epilogue == DG_EPI_DEFAULT && !a.accumulate &&
           a.bias == nullptr && a.alpha == 1.0f && a.block_m == 0 && a.block_n == 0 && a.split_k <= 1 && !a.jit && span32(64, a.lda) &&
           span32(kStrip, a.ldb) && span32(ceil_div(a.k, 64), a.sfa_ld * 2) && span32(ceil_div(a.k, 64), a.sfb_ld * 2);
}

int mx_experts(const dg_gemm_args& a, hipStream_t st, dg_launch_info* info) {
    MxProductParams p = {};
    p.a = reinterpret_cast<const uint8_t*>(a.a); p.w = reinterpret_cast<const uint8_t*>(a.b); p.d = reinterpret_cast<uint8_t*>(a.d);
    p.sfa = reinterpret_cast<const uint16_t*>(a.sfa); p.sfw = reinterpret_cast<const uint16_t*>(a.sfb);
    p.psum = a.grouped_layout;
    p.m = a.m; p.n = a.n; p.k = a.k; p.groups = a.num_groups; p.alignment = a.alignment;
    p.lda = a.lda; p.ldw = a.ldb; p.ldd = a.ldd;
    p.w_bs = a.batch_stride_b; p.sfw_bs = a.sfb_batch_stride;
    p.sfa_ld = a.sfa_ld; p.sfw_ld = a.sfb_ld;
    p.f32 = a.d_dtype == DG_DTYPE_F32;
    if (info != nullptr) {
        const int64_t strips = ceil_div(a.n, kStrip), grid = strips * (a.num_groups + a.m / 64);
        info->block_m = 64;
        info->block_n = kStrip;
        info->plan_workgroups = info->tiles = info->grid = grid;
        info->threads = 64 * k_waves(strips * a.num_groups, a.k, true);
        info->split_k = 1;
        info->skinny = 4;
        return DG_OK;
    }
    return launch_product<kCodes>(p, st, 0);
}

}  // namespace dg

extern "C" int dg_mx_gemm(const void* x, int32_t x_dtype, int64_t x_ld, const void* w, int64_t w_ld, const int16_t* sfw, int64_t sfw_ld,
                          void* d, int32_t d_dtype, int64_t ldd, int32_t m, int32_t n, int32_t k, int32_t accumulate, int32_t num_cus,
                          void* stream) {
    using namespace dg;
    if (m < 0 || n < 0 || k < 0) return dg_set_error("dg_mx_gemm: negative size");
    if (n > kMaxExtent) return dg_set_error("dg_mx_gemm: at most 2^30 columns");
    if (x_dtype != DG_DTYPE_BF16 && x_dtype != DG_DTYPE_F32) return dg_set_error("dg_mx_gemm: x is bf16 or fp32");
    if (d_dtype != DG_DTYPE_BF16 && d_dtype != DG_DTYPE_F32) return dg_set_error("dg_mx_gemm: D is bf16 or fp32");
    if (m > 16 || (int64_t)m * k > kInside) {
        dg_set_error("dg_mx_gemm: more than 16 rows or 32768 values (quantise them with dg_mx_quantize, then dg_gemm)");
        return DG_ENOKERNEL;
    }
    if (k % 32 != 0 || k == 0) return dg_set_error("dg_mx_gemm: K must be a multiple of the block of 32 values");
    if (m == 0 || n == 0) return DG_OK;
    const int64_t e = x_dtype == DG_DTYPE_F32 ? 4 : 2;
    if (x == nullptr || w == nullptr || sfw == nullptr || d == nullptr) return dg_set_error("dg_mx_gemm: null tensor");
    if ((m > 1 && x_ld < k) || w_ld < k / 2 || sfw_ld < n || (m > 1 && ldd < n)) return dg_set_error("dg_mx_gemm: leading dimension smaller than the row");
    if (x_ld * e % 4 != 0 || !aligned_to(x, 4) || w_ld % 4 != 0 || !aligned_to(w, 4) || !aligned_to(d, d_dtype == DG_DTYPE_F32 ? 4 : 2))
        return dg_set_error("dg_mx_gemm: rows of x and w must be 4-byte aligned");
    if (sfw_ld % 2 != 0 || !aligned_to(sfw, 4)) return dg_set_error("dg_mx_gemm: scale factors need an even leading dimension and 4-byte alignment");
    if (!span32(16, x_ld * e) || !span32(kStrip, w_ld) || !span32(ceil_div(k, 64), sfw_ld * 2)) return dg_set_error("dg_mx_gemm: row stride too large");
    MxProductParams p = {};
    p.a = reinterpret_cast<const uint8_t*>(x); p.w = reinterpret_cast<const uint8_t*>(w); p.d = reinterpret_cast<uint8_t*>(d);
    p.sfw = reinterpret_cast<const uint16_t*>(sfw);
    p.m = m; p.n = n; p.k = k; p.groups = 1; p.alignment = 1;
    p.lda = x_ld * e; p.ldw = w_ld; p.ldd = ldd; p.sfw_ld = sfw_ld;
    p.f32 = d_dtype == DG_DTYPE_F32;
    p.accumulate = accumulate != 0;
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    return x_dtype == DG_DTYPE_F32 ? launch_product<kF32Rows>(p, st, num_cus) : launch_product<kBf16Rows>(p, st, num_cus);
}
