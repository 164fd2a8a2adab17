// Cross entropy of a linear layer over a large vocabulary, without keeping the logits.
//
//   z[t][v] = <x[t], w[v]>,  lse[t] = log sum_v exp z[t][v],  loss[t] = lse[t] - z[t][target[t]]
//   d[t][v] = (exp(z[t][v] - lse[t]) - [v = target[t]]) d_loss[t],  d_x = d w,  d_w = d^T x
//
// Forward: the bf16 tile kernel (quad_kernel.hpp) computes a tile of logits, and instead of storing it each row leaves its
// maximum, the sum of its exponentials under that maximum and, in the one tile that has it, the target's logit; a second
// kernel joins a row's tiles.  Nothing of tokens x vocabulary is written.
// Backward, a piece of the vocabulary at a time: the logits are computed again, d leaves the tile in bf16, and two products take
// it on.  d is rounded to bf16 because the matrix unit takes it so; that error is as large as that of the bf16 inputs and
// outputs beside it.  It is rounded in units of the largest |d_loss|, which both products multiply their fp32 sums by: with
// the equal weights of a mean the targets' entries are then p - 1, nearly exact, where 1 / tokens rounded to 8 bits put the
// same error of up to 0.4 % into all of them (777 tokens: gradients 0.25 % off against 0.17 % of the outputs' rounding alone).
// With unequal weights d_x gets what rounding took from the target's entry (one row of w a token); d_w, whose sums run over
// the tokens, would need it inside the product, and keeps that error.
// Logits, maxima, sums, losses and the sum of d_x over the pieces are fp32.
#include "op_launch.hpp"
#include "quad_kernel.hpp"

namespace dg {

int gemm_k_rows(const dg_gemm_args* args, int k_rows, void* stream);
void bf16_tile_plan(int m, int n, int k, bool mn, bool stats, int most, int cus, int& bm, int& bn, int& split, int64_t& partial_bytes);
int device_cus();

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct XentParams {
    const void* target;        // [tokens] int32 or int64
    int wide;
    int tokens;
    int first, vocab;          // first word of the piece, words in all
    int64_t ignore;
    float* target_logit;       // [tokens]
    f32x2* stats;              // forward: [tile columns][tokens] (maximum, sum)
    const float *lse, *d_loss; // backward
    float* unit;               // backward: 1 / u and u, the unit of d
    int own_unit;              // found by every tile itself (else ahead of them)
    float* left;               // backward: [tokens] what rounding took from d at the target, in units of d
    uint16_t* d;               // backward: [tokens][d_ld] bf16, whole tiles wide
    int64_t d_ld;
};

// Target of token t, or -1 where it counts for nothing (ignored, or outside the vocabulary).
__device__ __forceinline__ int target_of(const void* target, int wide, int64_t ignore, int vocab, int t) {
    const int64_t v = wide ? reinterpret_cast<const int64_t*>(target)[t] : reinterpret_cast<const int32_t*>(target)[t];
    return v == ignore || v < 0 || v >= vocab ? -1 : (int)v;
}

// u = the largest |d_loss| of a token with a target (1 where that, or its reciprocal, is no normal number), as (1 / u, u).
__device__ __forceinline__ f32x2 unit_of(float top) {
    return top >= 0x1p-100f && top <= 0x1p100f ? f32x2{1.f / top, top} : f32x2{1.f, 1.f};
}

// Tokens whose d_loss a tile's 256 threads take one each: past that a launch of one workgroup finds u.
constexpr int kOwnUnit = 256;

// Columns of a lane within its row of a tile: four runs of four to a 32-column block.
__device__ __forceinline__ int run_col(int block_col, int q, int e) { return block_col + 4 * q + 8 * (e >> 2) + (e & 3); }

// The logits of one row block that a lane holds: NB blocks of 16, with their first columns within the tile.
template <typename T, typename TAKE, typename COL, typename HA, typename I, int NB>
__device__ __forceinline__ void take_row(TAKE& take, COL& col_of, HA ha, I i, f32x16 (&z)[NB], int (&col)[NB]) {
    using SB = typename T::SB;
    static_for<NB>([&](auto b_c) {
        constexpr int b = decltype(b_c)::value, hb = b >= SB::NB0, j = hb ? b - SB::NB0 : b;
        z[b] = take(ha, Int<hb>{}, i, Int<j>{});
        col[b] = col_of(Int<hb>{}) + j * 32;
    });
}

// Forward.  The tile's product bounds it: 8192 tokens, 131072 words of width 4096 6.2 ms (1.41 PFLOP/s; the library's bf16 product
// of 8192^3 reaches 1.34), 777 tokens, 32003 words of width 1536 84 to 92 us (two rounds of tiles over the CUs of 24
// stages each, where fill and tail weigh most), 131 tokens, 32000 words of width 2048 30 us (w at 4.4 TB/s).
struct StatsTail {
    static constexpr bool kOn = true;
    XentParams x;

    __device__ __forceinline__ void begin() {}

    template <typename T, typename TAKE, typename ROW, typename COL>
    __device__ __forceinline__ void run(TAKE& take, ROW& row_of, COL& col_of, const TileLoc& tl, uint8_t* smem) const {
        using SA = typename T::SA;
        using SB = typename T::SB;
        constexpr int BM = SA::H0 + SA::H1, BN = SB::H0 + SB::H1, NB = SB::NB0 + SB::NB1;
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave & 1, wn = wave >> 1, r = lane & 31, q = lane >> 5;
        const int cols = x.vocab - x.first - tl.n0;          // columns of the tile that are words
        f32x2* const st = reinterpret_cast<f32x2*>(smem);    // [2][BM]: of each wave column
        __syncthreads();                                     // (every wave has read its last fragments)
        static_for<2>([&](auto ha_c) {
            static_for<SA::nb(decltype(ha_c)::value)>([&](auto i_c) {
                const int m = row_of(ha_c, i_c, wm, r);
                f32x16 z[NB];
                int col[NB];
                take_row<T>(take, col_of, ha_c, i_c, z, col);
                const int tc = m < x.tokens ? target_of(x.target, x.wide, x.ignore, x.vocab, m) - x.first - tl.n0 : -1;
                if (cols < BN) {                     // (the last tile: columns past the vocabulary)
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            if (run_col(col[b], q, e) >= cols) z[b][e] = -__builtin_inff();
                }
                // (few row blocks have a target among their columns: the search is a branch of the wave)
                if (__ballot((unsigned)tc < (unsigned)BN) != 0) {
                    float hit = 0.f;
                    bool mine = false;
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const bool here = run_col(col[b], q, e) == tc;
                            hit = here ? z[b][e] : hit;
                            mine = mine || here;
                        }
                    if (mine) x.target_logit[m] = hit;
                }
                float top[4] = {z[0][0], z[0][1], z[0][2], z[0][3]};
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int e = 0; e < 16; ++e) top[e & 3] = fmaxf(top[e & 3], z[b][e]);
                float row_top = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                row_top = fmaxf(row_top, __shfl_xor(row_top, 32, 64));
                // exponents in units of log 2: one multiply-add each (a row of nothing but -inf: exponentials of zero)
                const float shift = row_top == -__builtin_inff() ? 0.f : row_top * kLog2e;
                float sum[4] = {};
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int e = 0; e < 16; ++e) sum[e & 3] += __builtin_amdgcn_exp2f(__builtin_fmaf(z[b][e], kLog2e, -shift));
                float s = (sum[0] + sum[1]) + (sum[2] + sum[3]);
                s += __shfl_xor(s, 32, 64);
                if (q == 0) st[wn * BM + m - tl.m0] = f32x2{row_top, s};
            });
        });
        __syncthreads();
        const int m = tl.m0 + (int)threadIdx.x;
        if ((int)threadIdx.x < BM && m < x.tokens) {
            const f32x2 a = st[threadIdx.x], b = st[BM + threadIdx.x];
            const float top = fmaxf(a[0], b[0]), shift = top == -__builtin_inff() ? 0.f : top;
            const float s = a[1] * __builtin_amdgcn_exp2f((a[0] - shift) * kLog2e) + b[1] * __builtin_amdgcn_exp2f((b[0] - shift) * kLog2e);
            x.stats[(int64_t)(tl.n0 / BN) * x.tokens + m] = f32x2{top, s};
        }
    }
};

// Runs of four columns of a lane (and its partner in the wave's other half) -> 16 columns in a row, as two pieces of 16 bytes.
__device__ __forceinline__ void runs_of_16(const i32x2 (&pk)[4], i32x4 (&w)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const auto s02 = __builtin_amdgcn_permlane32_swap(pk[2][h], pk[0][h], false, false);
        const auto s13 = __builtin_amdgcn_permlane32_swap(pk[3][h], pk[1][h], false, false);
        w[0][h] = (int)s02[0]; w[0][2 + h] = (int)s02[1];
        w[1][h] = (int)s13[0]; w[1][2 + h] = (int)s13[1];
    }
}

// Backward: d of the tile.  The same product, and 2 bytes an element on top: 8192 tokens, 43776 words of width 4096 2.2 ms (1.34
// PFLOP/s, 717 MB of d); the products behind it take 2.06 each.
struct GradTail {
    static constexpr bool kOn = true;
    XentParams x;
    float top;                 // own_unit: |d_loss| of this thread's token

    // (loaded ahead of the tile's stages.  The backward pass with it and with the unit's own launch, us: 1 token, 4000 words of width
    // 512 22.9 and 25.1, 90, 11000 of 704 34.5 and 36.9, 256, 1000 of 4096 52.4 and 54.5, 128, 131072 of 4096 906 and 909, but 16,
    // 131072 of 4096 737 and 735.)
    __device__ __forceinline__ void begin() {
        const int t = threadIdx.x;
        top = 0.f;
        if (x.own_unit && t < x.tokens) {
            const float g = fabsf(x.d_loss[t]);
            top = target_of(x.target, x.wide, x.ignore, x.vocab, t) >= 0 ? fmaxf(g, 0.f) : 0.f;
        }
    }

    __device__ __forceinline__ float own_unit(const TileLoc& tl, uint8_t* smem) const {
        float* const part = reinterpret_cast<float*>(smem);
        float all = top;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) all = fmaxf(all, __shfl_xor(all, off, 64));
        __syncthreads();                             // (every wave has read its last fragments)
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = all;
        __syncthreads();
        const f32x2 u = unit_of(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])));
        if (threadIdx.x == 0 && tl.m0 == 0 && tl.n0 == 0) {   // (for the kernels behind)
            x.unit[0] = u[0];
            x.unit[1] = u[1];
        }
        return u[0];
    }

    template <typename T, typename TAKE, typename ROW, typename COL>
    __device__ __forceinline__ void run(TAKE& take, ROW& row_of, COL& col_of, const TileLoc& tl, uint8_t* smem) const {
        using SA = typename T::SA;
        using SB = typename T::SB;
        constexpr int BN = SB::H0 + SB::H1, NB = SB::NB0 + SB::NB1;
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave & 1, r = lane & 31, q = lane >> 5;
        const int cols = x.vocab - x.first - tl.n0;
        const float per_unit = x.own_unit ? own_unit(tl, smem) : x.unit[0];
        static_for<2>([&](auto ha_c) {
            static_for<SA::nb(decltype(ha_c)::value)>([&](auto i_c) {
                const int m = row_of(ha_c, i_c, wm, r);
                f32x16 z[NB];
                int col[NB];
                take_row<T>(take, col_of, ha_c, i_c, z, col);
                const int target = m < x.tokens ? target_of(x.target, x.wide, x.ignore, x.vocab, m) : -1;
                const float lse = target >= 0 ? x.lse[m] * kLog2e : 0.f, g = target >= 0 ? x.d_loss[m] * per_unit : 0.f;
                const int tc = target - x.first - tl.n0;
                const bool some = __ballot(target >= 0 && (unsigned)tc < (unsigned)BN) != 0;   // (a target among the columns)
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    float d[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) d[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(z[b][e], kLog2e, -lse));
                    if (some) {
                        // (columns of the block that this lane holds: bit 2 of their number is the lane's half)
                        const bool mine = (unsigned)(tc - col[b]) < 32u && (tc - col[b] >> 2 & 1) == q;
                        float v = 0.f;
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const bool here = run_col(col[b], q, e) == tc;
                            d[e] -= here ? 1.f : 0.f;
                            v = here ? d[e] * g : v;
                        }
                        if (mine) x.left[m] = v - bf16_to_f32(f32_to_bf16_rne(v));   // (m has a target: a token's row)
                    }
                    if (cols < BN) {                 // (the last tile: columns past the vocabulary)
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            if (run_col(col[b], q, e) >= cols) d[e] = 0.f;
                    }
                    i32x2 pk[4];
#pragma unroll
                    for (int t = 0; t < 4; ++t)
                        pk[t] = i32x2{(int)pack_bf16x2(d[4 * t] * g, d[4 * t + 1] * g), (int)pack_bf16x2(d[4 * t + 2] * g, d[4 * t + 3] * g)};
                    if (target < 0) {                // (zeros whatever the logits)
#pragma unroll
                        for (int t = 0; t < 4; ++t) pk[t] = i32x2{0, 0};
                    }
                    i32x4 w[2];
                    runs_of_16(pk, w);
                    if (m < x.tokens) {
                        uint16_t* const d = x.d + (int64_t)m * x.d_ld + tl.n0 + col[b] + (q ? 0 : 16);
                        *reinterpret_cast<i32x4*>(d) = w[0];
                        *reinterpret_cast<i32x4*>(d + 8) = w[1];
                    }
                }
            });
        });
    }
};

// d_w's tile: the sums in units of d, as bf16 (1.42 PFLOP/s at 8192 tokens, 43776 words of width 4096; 80 to 87 us at 777 tokens,
// 32003 words of width 1536: K is only 13 stages there, and D 98 MB).
struct WeightTail {
    static constexpr bool kOn = true;
    XentParams x;
    uint16_t* d_w;             // [words][ld]
    int64_t ld;
    int words, width;

    template <typename T, typename TAKE, typename ROW, typename COL>
    __device__ __forceinline__ void run(TAKE& take, ROW& row_of, COL& col_of, const TileLoc& tl, uint8_t*) const {
        using SA = typename T::SA;
        using SB = typename T::SB;
        constexpr int NB = SB::NB0 + SB::NB1;
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave & 1, r = lane & 31, q = lane >> 5;
        const float unit = x.unit[1];
        static_for<2>([&](auto ha_c) {
            static_for<SA::nb(decltype(ha_c)::value)>([&](auto i_c) {
                const int m = row_of(ha_c, i_c, wm, r);
                f32x16 z[NB];
                int col[NB];
                take_row<T>(take, col_of, ha_c, i_c, z, col);
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    i32x2 pk[4];
#pragma unroll
                    for (int t = 0; t < 4; ++t)
                        pk[t] = i32x2{(int)pack_bf16x2(z[b][4 * t] * unit, z[b][4 * t + 1] * unit),
                                      (int)pack_bf16x2(z[b][4 * t + 2] * unit, z[b][4 * t + 3] * unit)};
                    i32x4 w[2];
                    runs_of_16(pk, w);
                    const int n = tl.n0 + col[b] + (q ? 0 : 16);
                    uint16_t* const d = d_w + (int64_t)m * ld + n;
                    // (a row ends after a multiple of 8 values)
                    if (m < words && n < width) *reinterpret_cast<i32x4*>(d) = w[0];
                    if (m < words && n + 8 < width) *reinterpret_cast<i32x4*>(d + 8) = w[1];
                }
            });
        });
    }
};

template <int BM, int BN, typename TAIL>
__global__ __launch_bounds__(256, (quad_occupancy<BM, BN, kBF16, false, false>())) void xent_tile_kernel(const KParams p, const XentParams x) {
    TAIL tail = {x};
    tail.begin();
    quad_body<BM, BN, kBF16, kEpiBf16, kNormal, 1, 0, 0, 0, false, false, TAIL>(p, blockIdx.x + p.vbase, tail);
}

template <int BM, int BN>
__global__ __launch_bounds__(256, (quad_occupancy<BM, BN, kBF16, true, true>())) void xent_weight_kernel(const KParams p, const WeightTail tail) {
    quad_body<BM, BN, kBF16, kEpiBf16, kNormal, 1, 0, 0, 0, true, true, WeightTail>(p, blockIdx.x + p.vbase, tail);
}

struct CastParams {
    const float* src;          // [rows][width], whole rows together, in units of d
    const float* unit;
    uint16_t* dst;             // [rows][ld]
    int64_t ld;
    int rows, chunks;          // eight values each
    int vbase;
    const uint16_t* w;         // d_x: what rounding left of d at the targets times their words' rows (else nullptr)
    int64_t w_ld;
    const float* left;
    const void* target;
    int wide, vocab;
    int64_t ignore;
};

// d_x: the fp32 sums over the pieces as bf16, a chunk a thread (8192 x 4096: 43 us, 268 MB).  The target's entry of d, most of
// its row, is joined by what its rounding left, so that it counts in fp32 whatever the weights of the losses.  In the launch of few tokens' d_w it
// saves its own: the backward pass of 1 token, 4000 words of width 512 1.6 us, of 90, 11000 of 704 1.6, of 256, 1000 of 4096 1.9.
__device__ __forceinline__ void cast_chunks(const CastParams& p, int block) {
    const int64_t e = (int64_t)block * 256 + threadIdx.x;
    const int64_t row = e / p.chunks;
    if (row >= p.rows) return;
    const int c = (int)(e - row * p.chunks) * 8;
    const float* const s = p.src + row * p.chunks * 8 + c;
    const float unit = p.unit[1];
    f32x4 a = *reinterpret_cast<const f32x4*>(s), b = *reinterpret_cast<const f32x4*>(s + 4);
    const int target = p.w != nullptr ? target_of(p.target, p.wide, p.ignore, p.vocab, (int)row) : -1;
    if (target >= 0) {
        const float left = p.left[row];
        const i32x4 w = *reinterpret_cast<const i32x4*>(p.w + (int64_t)target * p.w_ld + c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f32x4& v = i < 2 ? a : b;
            v[2 * (i & 1)] += left * __builtin_bit_cast(float, (uint32_t)w[i] << 16);
            v[2 * (i & 1) + 1] += left * __builtin_bit_cast(float, (uint32_t)w[i] & 0xffff0000u);
        }
    }
    a *= unit;
    b *= unit;
    *reinterpret_cast<i32x4*>(p.dst + row * p.ld + c) = i32x4{(int)pack_bf16x2(a[0], a[1]), (int)pack_bf16x2(a[2], a[3]),
                                                             (int)pack_bf16x2(b[0], b[1]), (int)pack_bf16x2(b[2], b[3])};
}

// d_w of few tokens: a product of short K, where a tile's fill and stores are more than its stages, so that several workgroups share
// a CU and run them beside each other: 128 words x 128 values, four waves of 64 x 64, 32 tokens a stage in two slots of LDS (32 KB a
// workgroup, four to a CU).  Both operands are MN-major: 16-byte pieces of a token's row go to LDS as they are (swizzled so that a
// transposing read of four rows meets every bank once), and the reads hand each lane consecutive tokens of a word.
// Bound by the bytes of d_w, or by its LDS reads where there are more tokens.  The whole backward pass with it and with the four-wave
// tiles, us: 16 tokens, 131072 words of width 4096 757 and 799, 50257 of 1024 73 and 87, 100000 of 512 82 and 97, 32000 of 2048 85 and
// 97; 128 tokens 930 and 937, 100 and 114, 117 and 131, 107 and 119; 200 tokens, 50257 of 1024 124 and 141; 300 tokens 1365 and
// 1340, 170 and 189, 188 and 205, 182 and 189; 512 tokens 1665 and 1575, 209 and 220, 271 and 278, 221 and 223; 777 tokens 2581 and 2410.
// The limit is where the widest d_w turns: past it, to about 500 tokens, narrow ones give up 1 to 10 % that the short tiles would still gain.
constexpr int kShortTile = 128, kShortK = 32, kShortTokens = 256;

struct ShortParams {
    const uint16_t *d, *x;
    int64_t d_ld, x_ld, ld;
    const float* unit;
    uint16_t* d_w;
    int tokens, words, width;
    int col_tiles, tiles;
    CastParams cast;           // d_x, by the workgroups past the tiles (the last piece's launch: d_x is complete there)
    int vbase;
};

__global__ __launch_bounds__(256, 4) void xent_weight_short_kernel(const ShortParams p) {
    constexpr int PITCH = kShortTile * 2, SIDE = kShortK * PITCH, SLOT = 2 * SIDE, LOADS = SIDE / (256 * 16);
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * SLOT];
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, q = lane >> 5;
    if ((int)blockIdx.x + p.vbase >= p.tiles) {
        cast_chunks(p.cast, blockIdx.x + p.vbase - p.tiles);
        return;
    }
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave & 1, wn = wave >> 1;
    // (neighbours in a row of tiles share their d, on one XCD)
    const int t = xcd_remap(blockIdx.x + p.vbase, p.tiles);
    const int m0 = t / p.col_tiles * kShortTile, n0 = t % p.col_tiles * kShortTile;
    // tokens past the last, and values past the width in the last row, lie past the ranges and read zeros
    const __amdgpu_buffer_rsrc_t rs_d = make_rsrc(p.d + m0, (p.tokens * p.d_ld - m0) * 2);
    const __amdgpu_buffer_rsrc_t rs_x = make_rsrc(p.x + n0, ((p.tokens - 1) * p.x_ld + p.width - n0) * 2);
    const int k_of = tid / (PITCH / 16), piece = (tid % (PITCH / 16)) ^ ((k_of & 3) << 2);
    const uint32_t at_d = (uint32_t)(k_of * p.d_ld * 2 + piece * 16), at_x = (uint32_t)(k_of * p.x_ld * 2 + piece * 16);
    const int row_d = __builtin_amdgcn_readfirstlane((int)(p.d_ld * 2)), row_x = __builtin_amdgcn_readfirstlane((int)(p.x_ld * 2));
    constexpr int KSTEP = 256 / (PITCH / 16);          // tokens of one load of the workgroup
    static_assert(KSTEP % 4 == 0, "a thread's piece of the swizzle is the same in each of its loads");
    auto issue = [&](int s, int slot) {
        uint8_t* const to = lds + slot * SLOT + wave * 1024;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int k = s * kShortK + i * KSTEP;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs_d, (lds_void*)(to + i * 4096), 16, at_d, k * row_d, 0, 0);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs_x, (lds_void*)(to + SIDE + i * 4096), 16, at_x, k * row_x, 0, 0);
        }
    };
    // K [8 q, + 8) of 16 tokens from `k0` of MN row R0 + (lane & 31): two transposing reads
    typedef short v4s __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) v4s lds_v4s;
    const int s16 = lane & 15, h = (lane >> 4) & 1;
    auto fragment = [&](const uint8_t* side, int R0, int k0) {
        const int col = R0 + 16 * h + 4 * (s16 & 3), k = k0 + 8 * q + (s16 >> 2);
        const uint8_t* const at = side + k * PITCH + (((col >> 3) ^ ((k & 3) << 2)) << 4) + ((col >> 2) & 1) * 8;
        const i32x2 a = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)at));
        const i32x2 b = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(at + 4 * PITCH)));
        const i32x4 both = {a[0], a[1], b[0], b[1]};
        return __builtin_bit_cast(bf16x8, both);
    };
    f32x16 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = f32x16{};
    const int ns = ceil_div(p.tokens, kShortK);
    issue(0, 0);
    if (ns > 1) issue(1, 1);
    for (int s = 0; s < ns; ++s) {
        if (s + 1 < ns) wait_vmcnt<2 * LOADS>();
        else wait_vmcnt<0>();
        stage_barrier();
        const uint8_t* const side = lds + (s & 1) * SLOT;
#pragma unroll
        for (int k0 = 0; k0 < kShortK; k0 += 16) {
            bf16x8 a[2], b[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                a[i] = fragment(side, wm * 64 + 32 * i, k0);
                b[i] = fragment(side + SIDE, wn * 64 + 32 * i, k0);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(b[j], a[i], acc[i][j], 0, 0, 0);
        }
        if (s + 2 < ns) {
            __builtin_amdgcn_s_waitcnt(0xc07f);        // (lgkmcnt 0: this wave's reads of the slot have returned)
            stage_barrier();
            issue(s + 2, s & 1);
        }
    }
    // through LDS, so that 16 lanes store a row's 256 bytes (16-byte pieces, each row's in an order of its own)
    const float unit = p.unit[1];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int row = wm * 64 + 32 * i + r;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            i32x2 pk[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                pk[e] = i32x2{(int)pack_bf16x2(acc[i][j][4 * e] * unit, acc[i][j][4 * e + 1] * unit),
                              (int)pack_bf16x2(acc[i][j][4 * e + 2] * unit, acc[i][j][4 * e + 3] * unit)};
            i32x4 w[2];
            runs_of_16(pk, w);
            const int at = wn * 8 + 4 * j + (q ? 0 : 2);
#pragma unroll
            for (int x = 0; x < 2; ++x) *reinterpret_cast<i32x4*>(lds + row * PITCH + (((at + x) ^ (row & 15)) << 4)) = w[x];
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kShortTile / 16; ++i) {
        const int row = i * 16 + tid / 16, n = n0 + ((tid % 16) ^ (row & 15)) * 8;
        // (a row ends after a multiple of 8 values)
        if (m0 + row < p.words && n < p.width)
            *reinterpret_cast<i32x4*>(p.d_w + (int64_t)(m0 + row) * p.ld + n) = *reinterpret_cast<const i32x4*>(lds + row * PITCH + (tid % 16) * 16);
    }
}

struct UnitParams {
    const float* d_loss;
    const void* target;
    int wide, tokens, vocab;
    int64_t ignore;
    float* unit;               // 1 / u, u
    int vbase;
};

// u by one workgroup: 3 to 8 us up to 8192 tokens, next to at least a hundred of products.
__global__ __launch_bounds__(1024) void xent_unit_kernel(const UnitParams p) {
    __shared__ float part[16];
    float top = 0.f;
#pragma unroll 8
    for (int t = threadIdx.x; t < p.tokens; t += 1024)
        if (target_of(p.target, p.wide, p.ignore, p.vocab, t) >= 0) top = fmaxf(top, fabsf(p.d_loss[t]));
    for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int w = 1; w < 16; ++w) top = fmaxf(top, part[w]);
    const f32x2 u = unit_of(top);
    p.unit[0] = u[0];
    p.unit[1] = u[1];
}

struct JoinParams {
    const f32x2* stats;
    const float* target_logit;
    const void* target;
    int wide, tokens, vocab, tiles;
    int64_t ignore;
    float *loss, *lse;
    uint32_t* status;
    int vbase;
};

// A row's tiles joined: TOK rows of a workgroup, 256 / TOK threads a row; their results meet lane by lane, then wave by wave.
// Bound by the latency of its loads: 4.4 us at 131 tokens of 250 tiles, 9.7 at 8192 tokens of 512 (34 MB).
template <int TOK>
__global__ __launch_bounds__(256) void xent_join_kernel(const JoinParams p) {
    constexpr int PARTS = 256 / TOK;
    __shared__ f32x2 part[4][TOK];
    const int tid = threadIdx.x, tok = tid % TOK, slice = tid / TOK, t = (blockIdx.x + p.vbase) * TOK + tok;
    float top = -__builtin_inff(), sum = 0.f;
    auto join = [&](f32x2 v) {
        const float both = fmaxf(top, v[0]), shift = both == -__builtin_inff() ? 0.f : both;
        sum = sum * __builtin_amdgcn_exp2f((top - shift) * kLog2e) + v[1] * __builtin_amdgcn_exp2f((v[0] - shift) * kLog2e);
        top = both;
    };
    if (t < p.tokens) {
        for (int i = slice; i < p.tiles; i += 8 * PARTS) {
            f32x2 v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u)
                v[u] = i + u * PARTS < p.tiles ? p.stats[(int64_t)(i + u * PARTS) * p.tokens + t] : f32x2{-__builtin_inff(), 0.f};
#pragma unroll
            for (int u = 0; u < 8; ++u) join(v[u]);
        }
    }
#pragma unroll
    for (int off = TOK; off < 64; off <<= 1) join(f32x2{__shfl_xor(top, off, 64), __shfl_xor(sum, off, 64)});
    if ((tid & 63) < TOK) part[tid >> 6][tok] = f32x2{top, sum};
    __syncthreads();
    if (slice != 0 || t >= p.tokens) return;
    for (int i = 1; i < 4; ++i) join(part[i][tok]);
    const float lse = top + kLn2 * __builtin_amdgcn_logf(sum);
    const int64_t raw = p.wide ? reinterpret_cast<const int64_t*>(p.target)[t] : reinterpret_cast<const int32_t*>(p.target)[t];
    const int target = target_of(p.target, p.wide, p.ignore, p.vocab, t);
    if (raw != p.ignore && target < 0 && p.status != nullptr) p.status[4] = 1u;
    p.lse[t] = lse;
    p.loss[t] = target < 0 ? 0.f : lse - p.target_logit[t];
}

// d_x by itself, behind more tokens than the short kernel takes.
__global__ __launch_bounds__(256) void xent_cast_kernel(const CastParams p) { cast_chunks(p, blockIdx.x + p.vbase); }

// ------------------------------------------------------------------------------------------------ host
// Tokens of one call: the gradient's product reads d MN-major, whose K rows (tokens) times a tile's words stay below 1 GiB.
constexpr int kMaxTokens = 1 << 20;

// Whether d_w's tiles read x, MN-major, through one range of 32-bit offsets.  Where its rows span more, the tokens go in pieces
// whose products are summed in fp32 (a range of 2^31 - 1 bytes would end inside x, and the tokens past it read as zeros).
bool x_in_one_range(const dg_linear_xent_args& a) { return (int64_t)a.tokens * a.x_ld * 2 <= 0x7fffffffLL; }

// Tokens of such a piece: below 1 GiB of x and of d, as dg_gemm takes MN-major operands; whole stages.  (The backward pass of width 4096
// and 32000 words: 262143 tokens, the most in one range, 186 ms, 262144 in three pieces 194.)
int piece_tokens(const dg_linear_xent_args& a, int words) {
    const int64_t row = 2 * std::max<int64_t>(a.x_ld, words);
    return (int)std::min<int64_t>(0x3fffffffLL / row / 64 * 64, a.tokens);
}

// Words of a piece: whole tiles; d and the piece of w stay below 1 GiB each (they are read MN-major).
int piece_words(const dg_linear_xent_args& a) {
    // (and 256 rows of d below 2 GiB, a tile's; d_w's fp32 sums below 1 GiB)
    const int64_t most = (int64_t(1) << 29) - 1, sums = x_in_one_range(a) ? most : (int64_t(1) << 28) / a.width;
    const int64_t fit = std::min({most / a.tokens, most / a.w_ld, int64_t(1) << 21, sums}) / 256 * 256;
    const int64_t pieces = ceil_div64(a.vocab, std::max<int64_t>(256, fit));
    return (int)align_up64(ceil_div64(a.vocab, pieces), 256);
}

struct Space {   // the workspace, cut up
    int64_t bytes = 0;
    int64_t take(int64_t n) {
        const int64_t at = bytes;
        bytes += align_up64(n, 256);
        return at;
    }
};

struct Plan {
    int bm, bn;                // the logits' tile
    int words, pieces;
    int xbm, xbn, xsplit, wbm, wbn;
    int64_t stats, logit, d, d_x, d_w, unit, left, partial, partial_bytes, bytes;
};

int cus_of(const dg_linear_xent_args& a) { return a.num_cus > 0 ? a.num_cus : device_cus(); }

Plan plan_of(const dg_linear_xent_args& a, bool backward) {
    Plan p = {};
    Space s;
    int one = 1;
    int64_t none = 0;
    const int cus = cus_of(a);
    if (!backward) {
        bf16_tile_plan(a.tokens, a.vocab, a.width, false, true, 1, cus, p.bm, p.bn, one, none);
        p.stats = s.take((int64_t)ceil_div(a.vocab, p.bn) * a.tokens * 8);
        p.logit = s.take((int64_t)a.tokens * 4);
    } else {
        p.words = piece_words(a);
        p.pieces = ceil_div(a.vocab, p.words);
        bf16_tile_plan(a.tokens, std::min(p.words, a.vocab), a.width, false, false, 1, cus, p.bm, p.bn, one, none);
        p.d = s.take((int64_t)a.tokens * p.words * 2);
        p.d_x = s.take((int64_t)a.tokens * a.width * 4);
        p.d_w = s.take(x_in_one_range(a) ? 0 : (int64_t)p.words * a.width * 4);
        p.unit = s.take(8);
        p.left = s.take((int64_t)a.tokens * 4);
        bf16_tile_plan(a.tokens, a.width, p.words, true, false, 32, cus, p.xbm, p.xbn, p.xsplit, p.partial_bytes);
        bf16_tile_plan(std::min(p.words, a.vocab), a.width, a.tokens, true, false, 1, cus, p.wbm, p.wbn, one, none);
        p.partial = s.take(p.partial_bytes);
    }
    p.bytes = s.bytes;
    return p;
}

int check(const dg_linear_xent_args* a) {
    if (a == nullptr) return dg_set_error("dg_linear_xent: null args");
    if (a->tokens < 0 || a->width < 1 || a->vocab < 1) return dg_set_error("dg_linear_xent: invalid size");
    if (a->vocab > kMaxExtent || a->width > kMaxExtent) return dg_set_error("dg_linear_xent: at most 2^30 words and values of a row");
    if (a->tokens > kMaxTokens) return dg_set_error("dg_linear_xent: at most 2^20 tokens");
    if (a->width % 8 != 0) return dg_set_error("dg_linear_xent: the width must be a multiple of 8");
    if (a->target_bytes != 4 && a->target_bytes != 8) return dg_set_error("dg_linear_xent: targets are int32 or int64");
    if (a->x_ld < a->width || a->w_ld < a->width || a->x_ld % 8 != 0 || a->w_ld % 8 != 0 || !aligned_to(a->x, 16) || !aligned_to(a->w, 16))
        return dg_set_error("dg_linear_xent: rows of x and w must be 16-byte aligned and hold the width");
    if (256 * a->x_ld * 2 > 0x7fffffffLL || 256 * a->w_ld * 2 > 0x3fffffffLL)
        return dg_set_error("dg_linear_xent: row stride too large");
    return DG_OK;
}

// The workgroups of a tile kernel over m x n outputs: fn(grid) launches with p, whose vbase is the first one.
template <typename F>
int launch_grid(KParams& p, int m, int n, int bm, int bn, int num_cus, F&& fn) {
    p.num_m_blocks = ceil_div(m, bm);
    p.num_n_blocks = ceil_div(n, bn);
    const int64_t grid = (int64_t)p.num_m_blocks * p.num_n_blocks;
    if (grid > 0x7fffffffLL) return dg_set_error("dg_linear_xent: too many tiles");
    p.num_tiles = p.vgrid = (int)grid;
    const int64_t most = num_cus > 0 ? (num_cus >= 8 ? num_cus / 8 * 8 : num_cus) : grid;
    for (int64_t base = 0; base < grid; base += most) {
        p.vbase = (int)base;
        fn(dim3((unsigned)std::min(most, grid - base)));
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) {
            dg_set_error(hipGetErrorString(e));
            return DG_ELAUNCH;
        }
    }
    return DG_OK;
}

KParams tile_params() {
    KParams p = {};
    p.num_groups = 1;
    p.out_esize = 2;
    p.alpha = 1.f;
    p.group_m = 4;
    p.split_k = 1;
    return p;
}

// Logits of all tokens and `words` words from x.first on.
int launch_logits(const Plan& pl, const dg_linear_xent_args& a, const XentParams& x, int words, bool backward, hipStream_t st) {
    KParams p = tile_params();
    p.a = reinterpret_cast<const uint8_t*>(a.x);
    p.b = reinterpret_cast<const uint8_t*>(a.w) + (int64_t)x.first * a.w_ld * 2;
    p.m = a.tokens; p.n = words; p.k = a.width;
    p.lda = a.x_ld * 2; p.ldb = a.w_ld * 2;
    p.kbytes_a = p.kbytes_b = a.width * 2;
    return launch_grid(p, a.tokens, words, pl.bm, pl.bn, a.num_cus, [&](dim3 grid) {
        auto go = [&](auto tail, auto bm, auto bn) {
            hipLaunchKernelGGL((xent_tile_kernel<decltype(bm)::value, decltype(bn)::value, decltype(tail)>), grid, dim3(256), 0, st, p, x);
        };
        auto tile = [&](auto tail) {
            if (pl.bm == 256 && pl.bn == 256) go(tail, Int<256>{}, Int<256>{});
            else if (pl.bm == 256) go(tail, Int<256>{}, Int<128>{});
            else go(tail, Int<128>{}, Int<128>{});
        };
        if (backward) tile(GradTail{});
        else tile(StatsTail{});
    });
}

int64_t cast_blocks(const CastParams& c) { return ceil_div64((int64_t)c.rows * c.chunks, 256); }

// d_w rows of the piece = d^T x (both read MN-major): K rows past the tokens are not read.  Behind the last piece, d_x from
// its sums: for few tokens in the same launch.
// `sums`: fp32 [words][width], used only where x spans more than one range.
int launch_weight(const Plan& pl, const dg_linear_xent_args& a, const XentParams& x, int words, float* sums, const CastParams& cast, hipStream_t st) {
    const bool last = x.first + words == a.vocab;
    if (a.tokens <= kShortTokens && (int64_t)(a.tokens + kShortK) * a.x_ld * 2 <= 0x7fffffffLL) {   // (32-bit offsets into x)
        ShortParams s = {};
        s.d = x.d; s.d_ld = x.d_ld; s.x = reinterpret_cast<const uint16_t*>(a.x); s.x_ld = a.x_ld;
        s.unit = x.unit; s.d_w = reinterpret_cast<uint16_t*>(a.d_w) + (int64_t)x.first * a.d_w_ld; s.ld = a.d_w_ld;
        s.tokens = a.tokens; s.words = words; s.width = a.width;
        s.col_tiles = ceil_div(a.width, kShortTile);
        const int64_t tiles = (int64_t)ceil_div(words, kShortTile) * s.col_tiles, grid = tiles + (last ? cast_blocks(cast) : 0);
        if (grid > 0x7fffffffLL) return dg_set_error("dg_linear_xent: too many tiles");
        s.tiles = (int)tiles;
        s.cast = cast;
        return launch_op(xent_weight_short_kernel, grid, 256, s, st, a.num_cus);
    }
    uint16_t* const d_w = reinterpret_cast<uint16_t*>(a.d_w) + (int64_t)x.first * a.d_w_ld;
    if (!x_in_one_range(a)) {
        const int step = piece_tokens(a, pl.words);
        for (int t = 0; t < a.tokens; t += step) {
            const int tokens = std::min(step, a.tokens - t);
            dg_gemm_args g = {};
            g.kind = DG_KIND_BF16; g.gemm_type = DG_GEMM_NORMAL; g.num_groups = 1; g.alpha = 1.f; g.num_cus = a.num_cus;
            g.a = x.d + (int64_t)t * x.d_ld; g.lda = x.d_ld; g.a_mn_major = 1;
            g.b = reinterpret_cast<const uint16_t*>(a.x) + (int64_t)t * a.x_ld; g.ldb = a.x_ld; g.b_mn_major = 1;
            g.d = sums; g.ldd = a.width; g.d_dtype = DG_DTYPE_F32;
            g.accumulate = t > 0;
            g.m = words; g.n = a.width; g.k = (int)align_up64(tokens, 8);
            g.block_m = pl.wbm; g.block_n = pl.wbn; g.split_k = 1;
            if (const int rc = gemm_k_rows(&g, tokens, reinterpret_cast<void*>(st))) return rc;
        }
        const CastParams rounded = {sums, x.unit, d_w, a.d_w_ld, words, a.width / 8};
        if (const int rc = launch_op(xent_cast_kernel, cast_blocks(rounded), 256, rounded, st, a.num_cus)) return rc;
        return last ? launch_op(xent_cast_kernel, cast_blocks(cast), 256, cast, st, a.num_cus) : DG_OK;
    }
    KParams p = tile_params();
    p.a = reinterpret_cast<const uint8_t*>(x.d);
    p.b = reinterpret_cast<const uint8_t*>(a.x);
    p.m = words; p.n = a.width; p.k = a.tokens;
    p.lda = x.d_ld * 2; p.ldb = a.x_ld * 2;
    const WeightTail tail = {x, d_w, a.d_w_ld, words, a.width};
    const int rc = launch_grid(p, words, a.width, pl.wbm, pl.wbn, a.num_cus, [&](dim3 grid) {
        if (pl.wbm == 256 && pl.wbn == 256) hipLaunchKernelGGL((xent_weight_kernel<256, 256>), grid, dim3(256), 0, st, p, tail);
        else if (pl.wbm == 256) hipLaunchKernelGGL((xent_weight_kernel<256, 128>), grid, dim3(256), 0, st, p, tail);
        else hipLaunchKernelGGL((xent_weight_kernel<128, 128>), grid, dim3(256), 0, st, p, tail);
    });
    return rc != DG_OK || !last ? rc : launch_op(xent_cast_kernel, cast_blocks(cast), 256, cast, st, a.num_cus);
}

XentParams xent_params(const dg_linear_xent_args& a) {
    XentParams x = {};
    x.target = a.target;
    x.wide = a.target_bytes == 8;
    x.tokens = a.tokens;
    x.vocab = a.vocab;
    x.ignore = a.ignore_index;
    return x;
}

}  // namespace
}  // namespace dg

extern "C" int dg_linear_xent_workspace_size(const dg_linear_xent_args* args, int32_t backward, int64_t* bytes) {
    if (bytes == nullptr) return dg_set_error("dg_linear_xent: null bytes");
    if (const int rc = dg::check(args)) return rc;
    *bytes = args->tokens == 0 ? 0 : dg::plan_of(*args, backward != 0).bytes;
    return DG_OK;
}

extern "C" int dg_linear_xent_forward(const dg_linear_xent_args* args, void* stream) {
    using namespace dg;
    if (const int rc = check(args)) return rc;
    const dg_linear_xent_args& a = *args;
    if (a.tokens == 0) return DG_OK;
    if (a.x == nullptr || a.w == nullptr || a.target == nullptr || a.loss == nullptr || a.lse == nullptr)
        return dg_set_error("dg_linear_xent: null tensor");
    const Plan pl = plan_of(a, false);
    if (a.workspace == nullptr || a.workspace_bytes < pl.bytes)
        return dg_set_error("dg_linear_xent: workspace smaller than dg_linear_xent_workspace_size() reports");
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    uint8_t* const ws = reinterpret_cast<uint8_t*>(a.workspace);
    XentParams x = xent_params(a);
    x.stats = reinterpret_cast<f32x2*>(ws + pl.stats);
    x.target_logit = reinterpret_cast<float*>(ws + pl.logit);
    if (const int rc = launch_logits(pl, a, x, a.vocab, false, st)) return rc;
    JoinParams j = {};
    j.stats = x.stats; j.target_logit = x.target_logit; j.target = a.target; j.wide = x.wide;
    j.tokens = a.tokens; j.vocab = a.vocab; j.tiles = ceil_div(a.vocab, pl.bn); j.ignore = a.ignore_index;
    j.loss = a.loss; j.lse = const_cast<float*>(a.lse);
    j.status = status_words_for(st);
    // (few tokens: more threads to each)
    if (a.tokens <= 256) return launch_op(xent_join_kernel<2>, ceil_div(a.tokens, 2), 256, j, st, a.num_cus);
    return launch_op(xent_join_kernel<16>, ceil_div(a.tokens, 16), 256, j, st, a.num_cus);
}

extern "C" int dg_linear_xent_backward(const dg_linear_xent_args* args, void* stream) {
    using namespace dg;
    if (const int rc = check(args)) return rc;
    const dg_linear_xent_args& a = *args;
    if (a.d_x_ld < a.width || a.d_w_ld < a.width || a.d_x_ld % 8 != 0 || a.d_w_ld % 8 != 0 || !aligned_to(a.d_x, 16) || !aligned_to(a.d_w, 16))
        return dg_set_error("dg_linear_xent: rows of the gradients must be 16-byte aligned and hold the width");
    if (a.d_w == nullptr) return dg_set_error("dg_linear_xent: null tensor");
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (a.tokens == 0) return dg_set_error("dg_linear_xent: no tokens (the gradient of w is zero)");
    if (a.x == nullptr || a.w == nullptr || a.target == nullptr || a.lse == nullptr || a.d_loss == nullptr || a.d_x == nullptr)
        return dg_set_error("dg_linear_xent: null tensor");
    const Plan pl = plan_of(a, true);
    if (a.workspace == nullptr || a.workspace_bytes < pl.bytes)
        return dg_set_error("dg_linear_xent: workspace smaller than dg_linear_xent_workspace_size() reports");
    uint8_t* const ws = reinterpret_cast<uint8_t*>(a.workspace);
    XentParams x = xent_params(a);
    x.lse = a.lse;
    x.d_loss = a.d_loss;
    x.d = reinterpret_cast<uint16_t*>(ws + pl.d);
    x.d_ld = pl.words;
    float* const unit = reinterpret_cast<float*>(ws + pl.unit);
    x.unit = unit;
    x.left = reinterpret_cast<float*>(ws + pl.left);
    const CastParams cast = {reinterpret_cast<const float*>(ws + pl.d_x), unit, reinterpret_cast<uint16_t*>(a.d_x), a.d_x_ld, a.tokens,
                             a.width / 8, 0, reinterpret_cast<const uint16_t*>(a.w), a.w_ld, x.left, a.target, x.wide, a.vocab,
                             a.ignore_index};
    x.own_unit = a.tokens <= kOwnUnit;
    const UnitParams u = {a.d_loss, a.target, x.wide, a.tokens, a.vocab, a.ignore_index, unit, 0};
    if (!x.own_unit)
        if (const int rc = launch_op(xent_unit_kernel, 1, 1024, u, st, 0)) return rc;
    for (int first = 0; first < a.vocab; first += pl.words) {
        const int words = std::min(pl.words, a.vocab - first);
        x.first = first;
        if (const int rc = launch_logits(pl, a, x, words, true, st)) return rc;
        // d_x (+)= d w: d's rows are zeros past the words, up to a whole tile; w's rows end with the vocabulary
        dg_gemm_args g = {};
        g.kind = DG_KIND_BF16; g.gemm_type = DG_GEMM_NORMAL; g.num_groups = 1; g.alpha = 1.f; g.num_cus = a.num_cus;
        g.a = x.d; g.lda = x.d_ld;
        g.b = reinterpret_cast<const uint16_t*>(a.w) + (int64_t)first * a.w_ld; g.ldb = a.w_ld; g.b_mn_major = 1;
        g.d = ws + pl.d_x; g.ldd = a.width; g.d_dtype = DG_DTYPE_F32;
        g.accumulate = first > 0;
        g.m = a.tokens; g.n = a.width; g.k = (int)align_up64(words, 8);
        g.block_m = pl.xbm; g.block_n = pl.xbn; g.split_k = pl.xsplit;
        if (pl.xsplit > 1) {
            g.workspace = ws + pl.partial;
            g.workspace_bytes = pl.partial_bytes;
        }
        if (const int rc = gemm_k_rows(&g, words, stream)) return rc;
        if (const int rc = launch_weight(pl, a, x, words, reinterpret_cast<float*>(ws + pl.d_w), cast, st)) return rc;
    }
    return DG_OK;
}
