// Low-rank adapters of many requests beside a shared projection: d[t] = c[t] + s_i (x[t] a_i^T) b_i^T for the adapter i of token t.
//
// Tokens lie sorted by adapter in the rows of an M-grouped layout, whose groups start at multiples of 32, so that 16 rows belong to
// one adapter.  A first launch leaves the inner products v = x a^T of 16 rows and a range of k in fp32 (ranges are summed in order by
// their readers), a second one multiplies them by b.  Both put the adapter's matrix on the side of the matrix instruction whose
// results a lane holds four of, and the tokens on the other: a lane has consecutive values of one token.
//
// v enters the second product as a sum of bf16 numbers: an instruction of depth 32 takes 16 of the rank twice, the high parts in its
// first half and the low parts in its second, against the same 16 columns of b.  Two parts lose 2^-17, which the rounding of a bf16 d
// hides; for an fp32 d the rest of v, which a third part holds whole, takes further instructions.
#include "dg_common.hpp"
#include "op_launch.hpp"

namespace dg {
namespace {

typedef unsigned int u32;

constexpr int kThreads = 256;
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
    int rows, splits, k_range, strips, strip_cols, copies;
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

// Inner products of TT times 16 rows (ts: a lane's tokens, -1 for none) with the adapter's NT * 16, over k from k0 to `end`: a wave's
// range lies in one piece, so that it reads whole lines of the rows.
template <int NT, int TT>
__device__ __forceinline__ void inner_products(const LoraParams& p, int i, const int (&ts)[TT], int lane, int k0, int end, f32x4 (&acc)[TT][NT]) {
    // (rows without a token and past the rank repeat another: what comes of them is not used)
    const int deep = (lane >> 4) * 8;
    const uint16_t *x[TT], *a[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) a[j] = p.a + i * p.a_stride + (int64_t)min(j * 16 + (lane & 15), p.rank - 1) * p.a_ld + deep;
#pragma unroll
    for (int s = 0; s < TT; ++s) {
        x[s] = p.x + (int64_t)max(ts[s], 0) * p.x_ld + deep;
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[s][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    constexpr int U = NT + TT <= 2 ? 8 : NT + TT <= 6 ? 4 : 2;   // (steps whose loads are in flight together)
    int k = k0;
    for (; k + U * 32 <= end; k += U * 32) {
        bf16x8 xs[U][TT], as[U][NT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int s = 0; s < TT; ++s) xs[u][s] = *reinterpret_cast<const bf16x8*>(x[s] + k + u * 32);
#pragma unroll
            for (int j = 0; j < NT; ++j) as[u][j] = *reinterpret_cast<const bf16x8*>(a[j] + k + u * 32);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int s = 0; s < TT; ++s)
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[s][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as[u][j], xs[u][s], acc[s][j], 0, 0, 0);
    }
#pragma unroll 2
    for (; k < end; k += 32) {
        const bool in = k + deep < end;
        bf16x8 xs[TT], as[NT];
#pragma unroll
        for (int s = 0; s < TT; ++s) xs[s] = eight_or_zero(x[s] + k, in);
#pragma unroll
        for (int j = 0; j < NT; ++j) as[j] = eight_or_zero(a[j] + k, in);
#pragma unroll
        for (int s = 0; s < TT; ++s)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[s][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as[j], xs[s], acc[s][j], 0, 0, 0);
    }
}

// v of TT times 16 rows of one adapter over a range of k: the four waves take a quarter each and join through LDS.  4099 tokens, rank 32,
// K=2048 9.4 us (17 MB of x); 48 tokens over 20 adapters, rank 16, K=7168 4.6.
template <int NT, int TT>
__global__ __launch_bounds__(kThreads) void lora_inner_kernel(const LoraParams p) {
    __shared__ f32x4 part[4][TT * NT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, index = blockIdx.x + p.vbase;
    const int split = index % p.splits, row0 = index / p.splits * (TT * 16);
    const int i = p.m_indices[row0];
    int ts[TT];
#pragma unroll
    for (int s = 0; s < TT; ++s) ts[s] = token_of(p, row0 + s * 16 + (lane & 15));
    if (i < 0 || i >= p.adapters) return;
    f32x4 acc[TT][NT];
    const int from = split * p.k_range + wave * (p.k_range / 4);   // (a range is a multiple of 128)
    inner_products<NT, TT>(p, i, ts, lane, from, min(p.k, from + p.k_range / 4), acc);
#pragma unroll
    for (int s = 0; s < TT; ++s)
#pragma unroll
        for (int j = 0; j < NT; ++j) part[wave][s * NT + j][lane] = acc[s][j];
    __syncthreads();
    for (int e = wave; e < TT * NT; e += 4) {
        const int s = e / NT, j = e % NT;
        f32x4 sum = part[0][e][lane];
#pragma unroll
        for (int w = 1; w < 4; ++w) {
            const f32x4 o = part[w][e][lane];
#pragma unroll
            for (int q = 0; q < 4; ++q) sum[q] += o[q];
        }
        float* const v = p.v + ((int64_t)split * p.rows + row0 + s * 16 + (lane & 15)) * (NT * 16) + (lane >> 4) * 4;
        *reinterpret_cast<f32x4*>(v + j * 16) = sum;
    }
}

// The operand of the second product in LDS: the parts of 16 rows' v, [part][16 of the rank][token][16], two for a d of bf16, three for
// fp32.
template <int NT, typename E>
struct Operand {
    static constexpr int PARTS = sizeof(E) == 4 ? 3 : 2;
    alignas(16) uint16_t v[PARTS][NT][16][16];

    // Four values of token lane & 15, from (lane >> 4) * 4 of the j-th sixteen on; zeros past the rank.
    __device__ __forceinline__ void put(int j, int lane, f32x4 s, float scale, int rank) {
        if (j * 16 + (lane >> 4) * 4 >= rank) s = f32x4{0.f, 0.f, 0.f, 0.f};
        float rest[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) rest[q] = s[q] * scale;
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
            u32 w[2];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                float &a = rest[2 * q], &b = rest[2 * q + 1];
                w[q] = pack_bf16x2(a, b);
                a -= __builtin_bit_cast(float, w[q] << 16);
                b -= __builtin_bit_cast(float, w[q] & 0xffff0000u);
                // (the other parts beside an infinity are 0, not NaN)
                a = fabsf(a) < __builtin_inff() ? a : 0.f;
                b = fabsf(b) < __builtin_inff() ? b : 0.f;
            }
            *reinterpret_cast<i32x2*>(&v[part][j][lane & 15][(lane >> 4) * 4]) = i32x2{(int)w[0], (int)w[1]};
        }
    }
    __device__ __forceinline__ bf16x8 get(int j, int lane) const {
        return __builtin_bit_cast(bf16x8, *reinterpret_cast<const i32x4*>(&v[lane >> 5][j][lane & 15][((lane >> 4) & 1) * 8]));
    }
    // The third parts: of one sixteen of the rank, with zeros for the instruction's second half, or of two, one to each half.
    static constexpr int THIRDS = NT >= 8 ? 2 : 1;
    __device__ __forceinline__ bf16x8 third(int j, int lane) const {
        const i32x4 w = *reinterpret_cast<const i32x4*>(&v[PARTS - 1][THIRDS > 1 ? j + (lane >> 5) : j][lane & 15][((lane >> 4) & 1) * 8]);
        return __builtin_bit_cast(bf16x8, THIRDS > 1 || lane < 32 ? w : i32x4{0, 0, 0, 0});
    }
};

// Eight columns of a row of c, as they lie in memory.
template <typename E> struct Before;
template <>
struct Before<float> {
    f32x4 lo, hi;
    __device__ __forceinline__ void load(const float* c) {
        lo = reinterpret_cast<const f32x4_any*>(c)[0];
        hi = reinterpret_cast<const f32x4_any*>(c)[1];
    }
    __device__ __forceinline__ void load(const float* c, int n) {
        lo = hi = f32x4{0.f, 0.f, 0.f, 0.f};
        if (n >= 8) {
            load(c);
        } else {
#pragma unroll
            for (int q = 0; q < 7; ++q)
                if (q < n) (q < 4 ? lo : hi)[q & 3] = c[q];
        }
    }
    __device__ __forceinline__ float value(int q) const { return q < 4 ? lo[q & 3] : hi[q & 3]; }
};
template <>
struct Before<uint16_t> {
    i32x4 w;
    __device__ __forceinline__ void load(const uint16_t* c) { w = *reinterpret_cast<const i32x4_any*>(c); }
    __device__ __forceinline__ void load(const uint16_t* c, int n) {
        w = i32x4{0, 0, 0, 0};
        if (n >= 8) {
            load(c);
        } else {
#pragma unroll
            for (int q = 0; q < 7; ++q)
                if (q < n) w[q >> 1] |= (int)((u32)c[q] << (q & 1 ? 16 : 0));
        }
    }
    __device__ __forceinline__ float value(int q) const { return __builtin_bit_cast(float, q & 1 ? (u32)w[q >> 1] & 0xffff0000u : (u32)w[q >> 1] << 16); }
};

__device__ __forceinline__ void store_columns(float* d, const float (&o)[8]) {
    reinterpret_cast<f32x4_any*>(d)[0] = f32x4{o[0], o[1], o[2], o[3]};
    reinterpret_cast<f32x4_any*>(d)[1] = f32x4{o[4], o[5], o[6], o[7]};
}
__device__ __forceinline__ void store_columns(uint16_t* d, const float (&o)[8]) {
    *reinterpret_cast<i32x4_any*>(d) = i32x4{(int)pack_bf16x2(o[0], o[1]), (int)pack_bf16x2(o[2], o[3]),
                                             (int)pack_bf16x2(o[4], o[5]), (int)pack_bf16x2(o[6], o[7])};
}
template <typename E>
__device__ __forceinline__ void store_columns(E* d, const float (&o)[8], int n) {
    if (n >= 8) {
        store_columns(d, o);
    } else {
#pragma unroll
        for (int q = 0; q < 7; ++q)
            if (q < n) {
                if constexpr (sizeof(E) == 4) d[q] = o[q];
                else d[q] = f32_to_bf16_rne(o[q]);
            }
    }
}

// The matrix operand of 32 columns from n0 on.  Row m of instruction h's holds column (m / 4) * 8 + h * 4 + m % 4, so that two
// instructions leave a lane with eight columns side by side.  Whole columns (uniform over a wave) need no comparison.
template <int NT>
__device__ __forceinline__ void load_columns(const LoraParams& p, int i, bool some, int lane, int n0, bf16x8 (&b)[2][NT]) {
    const int m = lane & 15, deep = ((lane >> 4) & 1) * 8;
    const bool whole = some && n0 + 32 <= p.n && p.rank == NT * 16;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int n = n0 + (m >> 2) * 8 + h * 4 + (m & 3);
        const uint16_t* const from = p.b + i * p.b_stride + (int64_t)n * p.b_ld + deep;
        if (whole) {
#pragma unroll
            for (int j = 0; j < NT; ++j) b[h][j] = *reinterpret_cast<const bf16x8*>(from + j * 16);
        } else {
#pragma unroll
            for (int j = 0; j < NT; ++j) b[h][j] = eight_or_zero(from + j * 16, some && n < p.n && j * 16 + deep < p.rank);
        }
    }
}

// Third parts come from LDS as they are needed (held beside the others they cost waves: 4096 tokens, K=N=4096, fp32 d, rank 64 62 us in place
// of 73, rank 128 106 of 120, and two sixteens to an instruction there: 106 of 108, rank 256 215 of 227; without third parts 72, 104 and 202).
template <int NT, typename E>
__device__ __forceinline__ void outer_products(const bf16x8 (&b)[2][NT], const bf16x8 (&vs)[NT], const Operand<NT, E>& operand, int lane, float (&out)[8]) {
    f32x4 acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[h][j], vs[j], acc[h], 0, 0, 0);
    if constexpr (Operand<NT, E>::PARTS == 3) {
        if constexpr (NT >= 4) __builtin_amdgcn_sched_barrier(0);
        constexpr int AT_ONCE = Operand<NT, E>::THIRDS;
        const bool upper = AT_ONCE > 1 && lane >= 32;
#pragma unroll
        for (int j = 0; j < NT; j += AT_ONCE) {
            const bf16x8 rest = operand.third(j, lane);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const i32x4 b0 = __builtin_bit_cast(i32x4, b[h][j]), b1 = __builtin_bit_cast(i32x4, b[h][j + AT_ONCE - 1]);
                acc[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, upper ? b1 : b0), rest, acc[h], 0, 0, 0);
            }
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int q = 0; q < 4; ++q) out[h * 4 + q] = acc[h][q];
}

// Those columns of 16 rows, straight from and to memory (t: the token of row lane & 15): for few tokens.
template <int NT, typename E>
struct Columns {
    bf16x8 b[2][NT];
    Before<E> c;

    // (rows without a token read another's)
    __device__ __forceinline__ void load(const LoraParams& p, int i, bool some, int t, int lane, int n0) {
        const int at = n0 + (lane >> 4) * 8;
        load_columns<NT>(p, i, some, lane, n0, b);
        const E* const from = reinterpret_cast<const E*>(p.c) + max(t, 0) * p.c_ld + at;
        if (p.c != nullptr && n0 + 32 <= p.n) c.load(from);
        else c.load(from, p.c != nullptr ? p.n - at : 0);
    }
    __device__ __forceinline__ void finish(const LoraParams& p, int t, int lane, int n0, const bf16x8 (&vs)[NT], const Operand<NT, E>& operand) const {
        const int n = n0 + (lane >> 4) * 8;
        float out[8];
        outer_products<NT, E>(b, vs, operand, lane, out);
#pragma unroll
        for (int q = 0; q < 8; ++q) out[q] += c.value(q);
        if (t >= 0) store_columns(reinterpret_cast<E*>(p.d) + t * p.d_ld + n, out, p.n - n);
    }
};

// Tokens without an adapter, a wave each: d = c.
template <typename E>
__device__ __forceinline__ void copy_rows(const LoraParams& p, int64_t t) {
    if (t >= p.tokens || p.slots[t] >= 0) return;
    const int lane = threadIdx.x & 63;
    const E* const c = reinterpret_cast<const E*>(p.c) + t * p.c_ld;
    E* const d = reinterpret_cast<E*>(p.d) + t * p.d_ld;
    constexpr int U = 4;
    for (int n0 = lane * 8; n0 < p.n; n0 += U * 512) {
        Before<E> was[U];
#pragma unroll
        for (int u = 0; u < U; ++u) was[u].load(c + n0 + u * 512, p.c != nullptr ? p.n - n0 - u * 512 : 0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float o[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) o[q] = was[u].value(q);
            store_columns(d + n0 + u * 512, o, p.n - n0 - u * 512);
        }
    }
}

// The operands of TT times 16 rows of adapter i from the ranges' inner products, in order.
template <int NT, int TT, typename E>
__device__ __forceinline__ void gather_operand(const LoraParams& p, int i, bool some, int row0, Operand<NT, E> (&operand)[TT]) {
    const int lane = threadIdx.x & 63;
    const float scale = !some ? 0.f : p.scales != nullptr ? p.scales[i] : 1.f;
    for (int e = threadIdx.x; e < TT * NT * 64; e += kThreads) {
        const int s = e / (NT * 64), j = (e >> 6) % NT, row = row0 + s * 16 + (lane & 15);
        const float* const v = p.v + (int64_t)row * (NT * 16) + j * 16 + (lane >> 4) * 4;
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
        if (some) {
#pragma unroll 8
            for (int k = 0; k < p.splits; ++k) {
                const f32x4 o = *reinterpret_cast<const f32x4*>(v + (int64_t)k * p.rows * (NT * 16));
#pragma unroll
                for (int q = 0; q < 4; ++q) sum[q] += o[q];
            }
        }
        operand[s].put(j, lane, sum, scale, p.rank);
    }
}

// d of 16 rows and a strip of columns, 32 of them a wave at a time; before the tiles, workgroups that copy c to the d of four tokens
// where these have no adapter.
template <int NT, typename E>
__global__ __launch_bounds__(kThreads) void lora_outer_kernel(const LoraParams p) {
    __shared__ Operand<NT, E> operand[1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, index = blockIdx.x + p.vbase - p.copies;
    if (index < 0) {
        copy_rows<E>(p, (int64_t)(blockIdx.x + p.vbase) * 4 + wave);
        return;
    }
    const int strip = index % p.strips, row0 = index / p.strips * 16;
    const int i = p.m_indices[row0];
    const int t = token_of(p, row0 + (lane & 15));
    if (i < 0) return;
    const bool some = i < p.adapters;
    if (!some && p.status != nullptr) p.status[2] = 1u;
    // the next columns are read before these are written
    constexpr bool AHEAD = NT <= 4;
    const int end = min(p.n, (strip + 1) * p.strip_cols);
    int n0 = strip * p.strip_cols + wave * 32;
    Columns<NT, E> now, next;
    if (n0 < end) now.load(p, i, some, t, lane, n0);
    gather_operand<NT, 1, E>(p, i, some, row0, operand);
    __syncthreads();
    bf16x8 vs[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) vs[j] = operand[0].get(j, lane);
    for (; n0 < end; n0 += 128) {
        if (AHEAD && n0 + 128 < end) next.load(p, i, some, t, lane, n0 + 128);
        now.finish(p, t, lane, n0, vs, operand[0]);
        if constexpr (AHEAD) now = next;
        else if (n0 + 128 < end) now.load(p, i, some, t, lane, n0 + 128);
    }
}

// Many tokens: d of 32 rows (one adapter's) in pieces of 256 columns, which pass through LDS so that half a wave reads and writes 256
// columns of a token; the next piece of c is on its way meanwhile.  4099 tokens over 8 adapters, rank 32, N=7168: 33 us (117 MB, 3.5 TB/s;
// straight to memory in runs of 32 columns by 16 rows 43, by 64 rows 51, in LDS pieces of 512 columns without the next one 40).
template <int NT, typename E>
__global__ __launch_bounds__(kThreads) void lora_rows_kernel(const LoraParams p) {
    __shared__ Operand<NT, E> operand[2];
    __shared__ float delta[32][256 + 8];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, index = blockIdx.x + p.vbase - p.copies;
    if (index < 0) {
        copy_rows<E>(p, (int64_t)(blockIdx.x + p.vbase) * 4 + wave);
        return;
    }
    const int strip = index % p.strips, row0 = index / p.strips * 32;
    const int i = p.m_indices[row0];
    // this lane's rows when it reads and writes: 8 wave + 2 r + its half
    int ts[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) ts[r] = token_of(p, row0 + wave * 8 + r * 2 + (lane >> 5));
    if (i < 0) return;
    const bool some = i < p.adapters;
    if (!some && p.status != nullptr) p.status[2] = 1u;
    const int end = min(p.n, (strip + 1) * p.strip_cols), mine = (lane & 31) * 8;
    Before<E> c[4], next[4];
    auto load = [&](Before<E> (&to)[4], int n0) {
        const int n = n0 + mine;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const E* const from = reinterpret_cast<const E*>(p.c) + max(ts[r], 0) * p.c_ld + n;
            if (p.c != nullptr && n0 + 256 <= p.n) to[r].load(from);
            else to[r].load(from, p.c != nullptr ? p.n - n : 0);
        }
    };
    int n0 = strip * p.strip_cols;
    load(c, n0);
    gather_operand<NT, 2, E>(p, i, some, row0, operand);
    __syncthreads();
    for (; n0 < end; n0 += 256) {
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const int at = wave * 64 + g * 32;
            bf16x8 b[2][NT];
            load_columns<NT>(p, i, some, lane, n0 + at, b);
            if (g == 1 && n0 + 256 < end) load(next, n0 + 256);
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                bf16x8 vs[NT];
#pragma unroll
                for (int j = 0; j < NT; ++j) vs[j] = operand[s].get(j, lane);
                float out[8];
                outer_products<NT, E>(b, vs, operand[s], lane, out);
                f32x4* const to = reinterpret_cast<f32x4*>(&delta[s * 16 + (lane & 15)][at + (lane >> 4) * 8]);
                to[0] = f32x4{out[0], out[1], out[2], out[3]};
                to[1] = f32x4{out[4], out[5], out[6], out[7]};
            }
        }
        __syncthreads();
        const int n = n0 + mine;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const f32x4* const from = reinterpret_cast<const f32x4*>(&delta[wave * 8 + r * 2 + (lane >> 5)][mine]);
            const f32x4 lo = from[0], hi = from[1];
            float out[8];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                out[q] = c[r].value(q) + lo[q];
                out[4 + q] = c[r].value(4 + q) + hi[q];
            }
            E* const to = reinterpret_cast<E*>(p.d) + ts[r] * p.d_ld + n;
            if (n0 + 256 <= p.n) {
                if (ts[r] >= 0) store_columns(to, out);
            } else if (ts[r] >= 0) {
                store_columns(to, out, p.n - n);
            }
            c[r] = next[r];
        }
        __syncthreads();
    }
}

// Few tokens: both products in one launch.  Every strip of 512 columns computes its tile's inner products for itself (sixteen waves, a
// sixteenth of k each, from the XCD's L2), which costs less than a second launch that waits for the first: one token, rank 16, K=2048
// N=7168 5.5 us, by two launches 7.8.
template <int NT, typename E>
__global__ __launch_bounds__(1024) void lora_kernel(const LoraParams p) {
    __shared__ f32x4 part[16][NT][64];
    __shared__ Operand<NT, E> operand;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, index = blockIdx.x + p.vbase - p.copies;
    if (index < 0) {
        copy_rows<E>(p, (int64_t)(blockIdx.x + p.vbase) * 16 + wave);
        return;
    }
    // Workgroups go round the eight XCDs: the strips of 32 rows to one of them, whose L2 then holds the adapter's matrix.
    const int turn = index >> 3, unit = (turn / (2 * p.strips)) * 8 + (index & 7), tile = unit * 2 + turn / p.strips % 2, strip = turn % p.strips;
    const int row0 = tile * 16;
    if (row0 >= p.rows) return;
    const int i = p.m_indices[row0];
    const int t = token_of(p, row0 + (lane & 15)), ts[1] = {t};
    if (i < 0) return;
    const bool some = i < p.adapters;
    if (!some && p.status != nullptr) p.status[2] = 1u;
    const float scale = !some ? 0.f : p.scales != nullptr ? p.scales[i] : 1.f;
    const int n0 = strip * 512 + wave * 32;
    f32x4 acc[1][NT];
    inner_products<NT, 1>(p, some ? i : 0, ts, lane, wave * p.k_range, some ? min(p.k, (wave + 1) * p.k_range) : 0, acc);
#pragma unroll
    for (int j = 0; j < NT; ++j) part[wave][j][lane] = acc[0][j];
    Columns<NT, E> columns;   // (on their way while the products are joined)
    if (n0 < p.n) columns.load(p, i, some, t, lane, n0);
    __syncthreads();
    if (wave < NT) {
        f32x4 s = part[0][wave][lane];
#pragma unroll
        for (int w = 1; w < 16; ++w) {
            const f32x4 o = part[w][wave][lane];
#pragma unroll
            for (int q = 0; q < 4; ++q) s[q] += o[q];
        }
        operand.put(wave, lane, s, scale, p.rank);
    }
    __syncthreads();
    if (n0 >= p.n) return;
    bf16x8 vs[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) vs[j] = operand.get(j, lane);
    columns.finish(p, t, lane, n0, vs, operand);
}

typedef void (*LoraKernel)(const LoraParams);

int padded_rank(int rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : rank <= 64 ? 64 : rank <= 128 ? 128 : 256; }

// Rows of a tile.
int tile_rows(const dg_lora_args* a) { return a->tokens >= 512 && a->tokens >= 16 * (int64_t)a->adapters ? 32 : 16; }

template <int NT>
LoraKernel inner_of(int rows) { return rows == 16 ? &lora_inner_kernel<NT, 1> : &lora_inner_kernel<NT, 2>; }
LoraKernel pick_inner(int rank, int rows) {
    switch (padded_rank(rank)) {
        case 16: return inner_of<1>(rows);
        case 32: return inner_of<2>(rows);
        case 64: return inner_of<4>(rows);
        case 128: return inner_of<8>(rows);
        default: return inner_of<16>(rows);
    }
}
template <typename E, int NT>
LoraKernel outer_of(int rows) { return rows == 16 ? &lora_outer_kernel<NT, E> : &lora_rows_kernel<NT, E>; }
template <typename E>
LoraKernel pick_outer(int rank, int rows) {
    switch (padded_rank(rank)) {
        case 16: return outer_of<E, 1>(rows);
        case 32: return outer_of<E, 2>(rows);
        case 64: return outer_of<E, 4>(rows);
        case 128: return outer_of<E, 8>(rows);
        default: return outer_of<E, 16>(rows);
    }
}
template <typename E>
LoraKernel pick_one(int rank) {
    switch (padded_rank(rank)) {
        case 16: return &lora_kernel<1, E>;
        case 32: return &lora_kernel<2, E>;
        default: return &lora_kernel<4, E>;
    }
}

// Tiles of `rows` rows that hold tokens, at most.
int64_t live_tiles(const dg_lora_args* a, int rows) {
    return std::max<int64_t>(1, std::min<int64_t>(ceil_div(a->layout->rows, rows), ceil_div(a->tokens, rows) + std::min(a->tokens, a->adapters)));
}

// One launch where every strip has a CU to itself and reads little there for its inner products: the adapter's matrix, once a strip.  By its
// size, one launch and two in us on the device (adapters from HBM): 1 token, rank 16, N=7168 64 KB 5.5 and 7.8, 112 KB 7.1 and 8.6, 128 KB 7.8
// and 7.3, 160 KB 9.1 and 7.7, 224 KB 11.2 and 8.6; 16 tokens, rank 32, N=4096 112 KB 9.1 and 10.0, 160 KB 11.4 and 10.3.  The second launch
// costs the host 3 us (one token, 128 KB, calls behind each other from Python 7.9 and 11.2), so the limit lies past where the device
// would have it.  511 tokens over 8 adapters, rank 16, K=N=4096, 320 strips: 21.5 and 11.4.
bool one_launch(const dg_lora_args* a) {
    const int64_t bytes = (int64_t)padded_rank(a->rank) * a->k * 2;
    return padded_rank(a->rank) <= 64 && bytes <= (160 << 10) && live_tiles(a, 16) * ceil_div(a->n, 512) <= 256;
}

// Ranges of k: enough that the tiles which hold tokens fill the card, at least 512 of k each.
int splits_of(const dg_lora_args* a) {
    return (int)std::max<int64_t>(1, std::min<int64_t>(512 / live_tiles(a, tile_rows(a)), a->k / 512));
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
    if (a->layout->alignment % 32 != 0) return dg_set_error("dg_lora: the layout's alignment must be a multiple of 32");
    return DG_OK;
}

int workspace_size(const dg_lora_args* a, int64_t* bytes) {
    if (bytes == nullptr) return dg_set_error("dg_lora: null result");
    if (const int rc = check(a); rc != DG_OK) return rc;
    *bytes = one_launch(a) ? 0 : (int64_t)splits_of(a) * a->layout->rows * padded_rank(a->rank) * 4;
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
    const int64_t tiles = l.rows / 16;
    const bool copy = a->c != a->d;   // (in place, other tokens' rows are as they have to be)
    if (one_launch(a)) {
        p.strips = ceil_div(a->n, 512);
        p.k_range = align_up(ceil_div(a->k, 16), 32);
        p.copies = copy ? ceil_div(a->tokens, 16) : 0;
        // (whole rounds of the XCDs, also of the copying workgroups before the tiles')
        p.copies = align_up(p.copies, 8);
        return launch_op(size == 4 ? pick_one<float>(a->rank) : pick_one<uint16_t>(a->rank), align_up64(tiles / 2, 8) * 2 * p.strips + p.copies, 1024, p, st,
                         a->num_cus);
    }
    p.splits = splits_of(a);
    p.k_range = align_up(ceil_div(a->k, p.splits), 128);
    const int height = tile_rows(a);
    const int64_t many = l.rows / height, live = live_tiles(a, height);
    if (many > 0)
        if (const int rc = launch_op(pick_inner(a->rank, height), many * p.splits, kThreads, p, st, a->num_cus); rc != DG_OK) return rc;
    // as many strips of at least 256 columns as give every CU a few workgroups
    const int units = ceil_div(a->n, 256);
    p.strip_cols = ceil_div(units, (int)std::max<int64_t>(1, std::min<int64_t>(units, 1024 / live))) * 256;
    p.strips = ceil_div(a->n, p.strip_cols);
    p.copies = copy ? ceil_div(a->tokens, 4) : 0;
    return launch_op(size == 4 ? pick_outer<float>(a->rank, height) : pick_outer<uint16_t>(a->rank, height), many * p.strips + p.copies, kThreads, p, st,
                     a->num_cus);
}

}  // namespace
}  // namespace dg

extern "C" int dg_lora_workspace_size(const dg_lora_args* args, int64_t* bytes) { return dg::workspace_size(args, bytes); }
extern "C" int dg_lora_gemm(const dg_lora_args* args, void* stream) { return dg::run(args, stream); }
