// Low-rank adapters of many requests beside a shared projection: d[t] = c[t] + s_i (x[t] a_i^T) b_i^T for the adapter i of token t.
//
// Tokens lie sorted by adapter in the rows of an M-grouped layout, whose groups start at multiples of 32, so that 16 rows belong to
// one adapter.  A first launch leaves the inner products v = x a^T of 16 rows and a range of k in fp32 (ranges are summed in order by
// their readers), a second one multiplies them by b.  Both put the adapter's matrix on the side of the matrix instruction whose
// results a lane holds four of, and the tokens on the other: a lane has consecutive values of one token.
//
// v enters the second product as the sum of two bf16 numbers, 2^-17 of it lost: an instruction of depth 32 takes 16 of them twice, the
// high parts in its first half and the low parts in its second, against the same 16 columns of b.
#include "dg_common.hpp"
#include "op_launch.hpp"

namespace dg {
namespace {

typedef unsigned int u32;

constexpr int kThreads = 256;
constexpr int kRows = 16;      // of a tile
constexpr int kCols = 256;     // of d to a workgroup
constexpr int kMaxRank = 256;

struct LoraParams {
    const uint16_t *x, *a, *b;
    int64_t x_ld, a_ld, a_stride, b_ld, b_stride;
    const float* scales;
    const void* c;
    int64_t c_ld;
    void* d;
    int64_t d_ld;
    const int32_t *slots, *source, *m_indices;
    float* v;                  // [splits][rows][padded rank]
    uint32_t* status;
    int tokens, adapters, rank, n, k;
    int rows, splits, k_range, strips, tile_groups;
    int vbase;
};

typedef i32x4 i32x4_any __attribute__((aligned(2)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));

__device__ __forceinline__ bf16x8 eight_or_zero(const uint16_t* at, bool on) {
    i32x4 v = {0, 0, 0, 0};
    if (on) v = *reinterpret_cast<const i32x4*>(at);
    return __builtin_bit_cast(bf16x8, v);
}

// The token of a row, -1 for padding.
__device__ __forceinline__ int token_of(const LoraParams& p, int row) {
    const int t = p.source[row];
    return (u32)t < (u32)p.tokens ? t : -1;
}

// v of a tile's 16 rows over a range of k: the four waves take steps of 32 in turn and join through LDS.
template <int NT>
__global__ __launch_bounds__(kThreads) void lora_inner_kernel(const LoraParams p) {
    __shared__ f32x4 part[4][NT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, index = blockIdx.x + p.vbase;
    const int tile = index / p.splits, split = index % p.splits, row0 = tile * kRows;
    const int i = p.m_indices[row0];
    if (i < 0 || i >= p.adapters) return;
    const int t = token_of(p, row0 + (lane & 15)), deep = (lane >> 4) * 8;
    const uint16_t* const x = p.x + (int64_t)max(t, 0) * p.x_ld + deep;
    const uint16_t* const a = p.a + i * p.a_stride + (int64_t)(lane & 15) * p.a_ld + deep;
    const int end = min(p.k, (split + 1) * p.k_range);
    f32x4 acc[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int k = split * p.k_range + wave * 32; k < end; k += 128) {
        const bool in = k + deep < end;
        const bf16x8 xs = eight_or_zero(x + k, in && t >= 0);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const bf16x8 as = eight_or_zero(a + (int64_t)j * 16 * p.a_ld + k, in && j * 16 + (lane & 15) < p.rank);
            acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as, xs, acc[j], 0, 0, 0);
        }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) part[wave][j][lane] = acc[j];
    __syncthreads();
    float* const v = p.v + ((int64_t)split * p.rows + row0 + (lane & 15)) * (NT * 16) + (lane >> 4) * 4;
    for (int j = wave; j < NT; j += 4) {
        f32x4 sum = part[0][j][lane];
#pragma unroll
        for (int w = 1; w < 4; ++w) {
            const f32x4 o = part[w][j][lane];
#pragma unroll
            for (int q = 0; q < 4; ++q) sum[q] += o[q];
        }
        *reinterpret_cast<f32x4*>(v + j * 16) = sum;
    }
}

template <typename E>
__device__ __forceinline__ float value(const E* at) {
    if constexpr (sizeof(E) == 4) return *at;
    else return bf16_to_f32(*at);
}

// d of a tile's rows and 256 columns; past the tiles, workgroups that copy c to 16 tokens' d where these have no adapter.
template <int NT, typename E>
__global__ __launch_bounds__(kThreads) void lora_outer_kernel(const LoraParams p) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int index = blockIdx.x + p.vbase;
    const int tile = index / p.strips, strip = index % p.strips, row0 = tile * kRows;
    if (tile >= p.tile_groups) {
        index -= p.tile_groups * p.strips;
        for (int t = index * 16; t < min(p.tokens, index * 16 + 16); ++t) {
            if (p.slots[t] >= 0) continue;
            E* const d = reinterpret_cast<E*>(p.d) + t * p.d_ld;
            const E* const c = reinterpret_cast<const E*>(p.c) + t * p.c_ld;
            for (int n = threadIdx.x; n < p.n; n += kThreads) d[n] = p.c != nullptr ? c[n] : E(0);
        }
        return;
    }
    const int i = p.m_indices[row0];
    if (i < 0) return;
    const bool some = i < p.adapters;
    if (!some && p.status != nullptr) p.status[2] = 1u;
    const int t = token_of(p, row0 + (lane & 15)), part = lane >> 4, n0 = strip * kCols + wave * 64;
    bf16x8 vs[NT];
    const float scale = some ? (p.scales != nullptr ? p.scales[i] : 1.f) : 0.f;
    const float* const v = p.v + (int64_t)(row0 + (lane & 15)) * (NT * 16) + (part & 1) * 8;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        float s[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) s[q] = 0.f;
        if (some)
            for (int k = 0; k < p.splits; ++k) {
                const f32x4* const from = reinterpret_cast<const f32x4*>(v + (int64_t)k * p.rows * (NT * 16) + j * 16);
                const f32x4 lo = from[0], hi = from[1];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    s[q] += lo[q];
                    s[4 + q] += hi[q];
                }
            }
        u32 w[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float a = s[2 * q] * scale, b = s[2 * q + 1] * scale;
            u32 h = pack_bf16x2(a, b);
            if (part >= 2) {
                a -= __builtin_bit_cast(float, h << 16);
                b -= __builtin_bit_cast(float, h & 0xffff0000u);
                // (the low part beside an infinity is 0, not NaN)
                h = pack_bf16x2(fabsf(a) < __builtin_inff() ? a : 0.f, fabsf(b) < __builtin_inff() ? b : 0.f);
            }
            w[q] = h;
        }
        vs[j] = __builtin_bit_cast(bf16x8, i32x4{(int)w[0], (int)w[1], (int)w[2], (int)w[3]});
    }
    // Row m of the matrix operand of instruction h holds column n0 + (m / 4) * 8 + h * 4 + m % 4, so that two of them leave a lane with
    // eight columns side by side.
    const int m = lane & 15, deep = (part & 1) * 8;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        f32x4 acc[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            acc[h] = f32x4{0.f, 0.f, 0.f, 0.f};
            const int n = n0 + g * 32 + (m >> 2) * 8 + h * 4 + (m & 3);
            const uint16_t* const b = p.b + i * p.b_stride + (int64_t)n * p.b_ld + deep;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const bf16x8 bs = eight_or_zero(b + j * 16, some && n < p.n && j * 16 + deep < p.rank);
                acc[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bs, vs[j], acc[h], 0, 0, 0);
            }
        }
        const int n = n0 + g * 32 + part * 8;
        if (t < 0 || n >= p.n) continue;
        E* const d = reinterpret_cast<E*>(p.d) + t * p.d_ld + n;
        const E* const c = reinterpret_cast<const E*>(p.c) + t * p.c_ld + n;
        float out[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) out[q] = acc[q >> 2][q & 3];
        if (n + 8 <= p.n) {
            if constexpr (sizeof(E) == 4) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    f32x4 o = {out[4 * h], out[4 * h + 1], out[4 * h + 2], out[4 * h + 3]};
                    if (p.c != nullptr) {
                        const f32x4 was = *reinterpret_cast<const f32x4_any*>(c + 4 * h);
#pragma unroll
                        for (int q = 0; q < 4; ++q) o[q] += was[q];
                    }
                    *reinterpret_cast<f32x4_any*>(d + 4 * h) = o;
                }
            } else {
                if (p.c != nullptr) {
                    const i32x4 was = *reinterpret_cast<const i32x4_any*>(c);
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        out[2 * q] += __builtin_bit_cast(float, (u32)was[q] << 16);
                        out[2 * q + 1] += __builtin_bit_cast(float, (u32)was[q] & 0xffff0000u);
                    }
                }
                *reinterpret_cast<i32x4_any*>(d) = i32x4{(int)pack_bf16x2(out[0], out[1]), (int)pack_bf16x2(out[2], out[3]),
                                                         (int)pack_bf16x2(out[4], out[5]), (int)pack_bf16x2(out[6], out[7])};
            }
        } else {
#pragma unroll
            for (int q = 0; q < 8; ++q)
                if (n + q < p.n) {
                    const float o = out[q] + (p.c != nullptr ? value(c + q) : 0.f);
                    if constexpr (sizeof(E) == 4) d[q] = o;
                    else d[q] = f32_to_bf16_rne(o);
                }
        }
    }
}

typedef void (*LoraKernel)(const LoraParams);

int padded_rank(int rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : rank <= 64 ? 64 : rank <= 128 ? 128 : 256; }

LoraKernel pick_inner(int rank) {
    switch (padded_rank(rank)) {
        case 16: return &lora_inner_kernel<1>;
        case 32: return &lora_inner_kernel<2>;
        case 64: return &lora_inner_kernel<4>;
        case 128: return &lora_inner_kernel<8>;
        default: return &lora_inner_kernel<16>;
    }
}
template <typename E>
LoraKernel pick_outer(int rank) {
    switch (padded_rank(rank)) {
        case 16: return &lora_outer_kernel<1, E>;
        case 32: return &lora_outer_kernel<2, E>;
        case 64: return &lora_outer_kernel<4, E>;
        case 128: return &lora_outer_kernel<8, E>;
        default: return &lora_outer_kernel<16, E>;
    }
}

// Ranges of k: enough that the tiles which hold tokens fill the card, at least 512 of k each.
int splits_of(const dg_lora_args* a) {
    const int64_t groups = std::min(a->tokens, a->adapters);
    const int64_t tiles = std::max<int64_t>(1, std::min<int64_t>(a->layout->rows / kRows, ceil_div(a->tokens, kRows) + groups));
    return (int)std::max<int64_t>(1, std::min<int64_t>(512 / tiles, a->k / 512));
}

int check(const dg_lora_args* a) {
    if (a == nullptr || a->layout == nullptr) return dg_set_error("dg_lora: null args");
    if (a->tokens < 0 || a->adapters < 0 || a->n < 0 || a->k < 0 || a->rank < 0) return dg_set_error("dg_lora: negative size");
    if (a->tokens > kMaxExtent || a->n > kMaxExtent || a->k > kMaxExtent || a->adapters > kMaxExtent) return dg_set_error("dg_lora: every extent must be at most 2^30");
    if (a->rank < 8 || a->rank % 8 != 0 || a->rank > kMaxRank) return dg_set_error("dg_lora: rank must be a multiple of 8, at most 256");
    if (a->k < 8 || a->k % 8 != 0) return dg_set_error("dg_lora: K must be a multiple of 8");
    if (a->d_dtype != DG_DTYPE_BF16 && a->d_dtype != DG_DTYPE_F32) return dg_set_error("dg_lora: D is bf16 or fp32");
    if (a->layout->tokens != a->tokens || a->layout->topk != 1) return dg_set_error("dg_lora: the layout must be of one choice a token");
    if (a->layout->rows < 0 || a->layout->rows > kMaxExtent || a->layout->rows % 32 != 0) return dg_set_error("dg_lora: the layout's rows must be a multiple of 32");
    return DG_OK;
}

int workspace_size(const dg_lora_args* a, int64_t* bytes) {
    if (bytes == nullptr) return dg_set_error("dg_lora: null result");
    if (const int rc = check(a); rc != DG_OK) return rc;
    *bytes = (int64_t)splits_of(a) * a->layout->rows * padded_rank(a->rank) * 4;
    return DG_OK;
}

int run(const dg_lora_args* a, void* stream) {
    if (const int rc = check(a); rc != DG_OK) return rc;
    if (a->tokens == 0 || a->n == 0) return DG_OK;
    const int64_t size = a->d_dtype == DG_DTYPE_BF16 ? 2 : 4;
    const dg_moe_layout& l = *a->layout;
    if (a->x == nullptr || (a->adapters > 0 && (a->a == nullptr || a->b == nullptr)) || a->d == nullptr || l.slots == nullptr ||
        (l.rows > 0 && (l.source == nullptr || l.m_indices == nullptr)))
        return dg_set_error("dg_lora: null tensor");
    if (a->x_ld < a->k || a->a_ld < a->k || a->b_ld < a->rank || a->d_ld < a->n || (a->c != nullptr && a->c_ld < a->n) || a->a_stride < 0 || a->b_stride < 0)
        return dg_set_error("dg_lora: leading dimension smaller than the row");
    if (!aligned_to(a->x, 16) || !aligned_to(a->a, 16) || !aligned_to(a->b, 16) || a->x_ld % 8 != 0 || a->a_ld % 8 != 0 || a->b_ld % 8 != 0 ||
        a->a_stride % 8 != 0 || a->b_stride % 8 != 0)
        return dg_set_error("dg_lora: rows of x, a and b must be 16-byte aligned");
    if (!aligned_to(a->d, size) || !aligned_to(a->c, size) || !aligned_to(a->scales, 4)) return dg_set_error("dg_lora: tensors must be aligned");
    if (a->c == a->d && a->c_ld != a->d_ld) return dg_set_error("dg_lora: c in place of d must have its leading dimension");
    int64_t need = 0;
    if (const int rc = workspace_size(a, &need); rc != DG_OK) return rc;
    if (need > 0 && (a->workspace == nullptr || a->workspace_bytes < need || !aligned_to(a->workspace, 16))) return dg_set_error("dg_lora: workspace too small");
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    LoraParams p = {};
    p.x = static_cast<const uint16_t*>(a->x); p.x_ld = a->x_ld;
    p.a = static_cast<const uint16_t*>(a->a); p.a_ld = a->a_ld; p.a_stride = a->a_stride;
    p.b = static_cast<const uint16_t*>(a->b); p.b_ld = a->b_ld; p.b_stride = a->b_stride;
    p.scales = a->scales;
    p.c = a->c; p.c_ld = a->c_ld;
    p.d = a->d; p.d_ld = a->d_ld;
    p.slots = l.slots; p.source = l.source; p.m_indices = l.m_indices;
    p.v = static_cast<float*>(a->workspace);
    p.status = status_words_for(st);
    p.tokens = a->tokens; p.adapters = a->adapters; p.rank = a->rank; p.n = a->n; p.k = a->k;
    p.rows = l.rows;
    p.splits = splits_of(a);
    p.k_range = align_up(ceil_div(a->k, p.splits), 128);
    p.strips = ceil_div(a->n, kCols);
    p.tile_groups = l.rows / kRows;
    if (p.tile_groups > 0)
        if (const int rc = launch_op(pick_inner(a->rank), (int64_t)p.tile_groups * p.splits, kThreads, p, st, a->num_cus); rc != DG_OK) return rc;
    const int64_t copies = a->c == a->d ? 0 : ceil_div(a->tokens, 16);   // (in place, other tokens' rows are as they have to be)
    return launch_op(size == 4 ? pick_outer<float>(a->rank) : pick_outer<uint16_t>(a->rank), (int64_t)p.tile_groups * p.strips + copies, kThreads, p, st,
                     a->num_cus);
}

}  // namespace
}  // namespace dg

extern "C" int dg_lora_workspace_size(const dg_lora_args* args, int64_t* bytes) { return dg::workspace_size(args, bytes); }
extern "C" int dg_lora_gemm(const dg_lora_args* args, void* stream) { return dg::run(args, stream); }
