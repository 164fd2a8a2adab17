// Tokens sorted by expert, moved into the rows of an M-grouped layout and back, with the gradients.
//
// A pair is (token t, choice c) with p = t * topk + c and an expert id[p]; negative ids are dropped.  Pairs of one expert
// keep their order, expert e's rows start at a multiple of the alignment:
//   start[e] = sum_{f < e} align(count[f]),   slot[p] = start[id[p]] + #{p' < p : id[p'] = id[p]}.
// Everything is integer and ordered, so the layout is the same on every run.
#include "op_launch.hpp"

namespace dg {
namespace {

typedef unsigned int u32;

// ------------------------------------------------------------------------------------------------ sorting
constexpr int kSortThreads = 512, kSortWaves = kSortThreads / 64;   // (1024 threads: 32768 x 8 pairs 20.7 us in place of 17.2)
constexpr int kMaxGroups = 1024;
// Up to kSortOnePass pairs every workgroup counts all of them itself (one launch; us, and with a counting launch: 4096 pairs over 64
// groups 6.0 and 9.5, 6126 over 40 7.5 and 9.3, 8000 over 256 8.0 and 11.2, 8192 over 8 7.7 and 9.1); past that a first launch counts
// blocks of pairs, and past kSortMaxBlocks blocks, whose counts each workgroup would read for itself, another one sums them
// (256 groups, 2^23 pairs 156 us in place of 185, 2^26 1.19 ms in place of 3.9).
constexpr int kSortOnePass = 8192;
constexpr int kSortMaxBlocks = 256;
// Pairs of a block past that (32768 x 8 pairs over 256 groups: 18.7 us with 1024, 17.3 with 2048, 18.7 with 4096, 28 with 8192).
constexpr int kSortPairs = 2048;
constexpr int kSortBlock = 8192;   // pairs of a workgroup, at most

struct SortParams {
    const void* ids;
    int wide;                  // 64-bit ids
    int pairs, groups, alignment, rows;
    int per_block, blocks;     // pairs of a block, blocks
    int32_t *slots, *source, *indices, *psum;
    int32_t* counts;           // [blocks][groups] (two launches) or nullptr; summed: of the blocks before, and [groups] of all
    int summed;
    u32* status;
    int vbase;
};

// Expert of pair i, or `groups` for a dropped one (an id past the last expert is reported too).
__device__ __forceinline__ int key_of(const SortParams& p, int i) {
    const int64_t id = p.wide ? reinterpret_cast<const int64_t*>(p.ids)[i] : reinterpret_cast<const int32_t*>(p.ids)[i];
    if (id >= p.groups && p.status != nullptr) p.status[2] = 1u;
    return id >= 0 && id < p.groups ? (int)id : p.groups;
}

__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(const SortParams p) {
    __shared__ int hist[kMaxGroups + 1];
    const int b = blockIdx.x + p.vbase, tid = threadIdx.x;
    for (int g = tid; g <= p.groups; g += kSortThreads) hist[g] = 0;
    __syncthreads();
    const int first = b * p.per_block, last = min(p.pairs, first + p.per_block);
    for (int i = first + tid; i < last; i += kSortThreads) atomicAdd(&hist[key_of(p, i)], 1);
    __syncthreads();
    for (int g = tid; g < p.groups; g += kSortThreads) p.counts[(int64_t)b * p.groups + g] = hist[g];
}

// Counts of many blocks -> counts of the blocks before, in place, and of all blocks behind them.  A lane takes a group, a wave a run of
// blocks, twice: its sum, then its rows under what the waves before have.
constexpr int kSumThreads = 1024;
__global__ __launch_bounds__(kSumThreads) void sort_sum_kernel(const SortParams p) {
    __shared__ int part[kSumThreads / 64][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = kSumThreads / 64;
    const int g = (blockIdx.x + p.vbase) * 64 + lane, per = ceil_div(p.blocks, waves);
    const int b0 = min(p.blocks, wave * per), b1 = min(p.blocks, b0 + per);
    const bool on = g < p.groups;
    int sum = 0;
#pragma unroll 8
    for (int b = b0; b < b1; ++b) sum += on ? p.counts[(int64_t)b * p.groups + g] : 0;
    part[wave][lane] = sum;
    __syncthreads();
    int next = 0;
    for (int w = 0; w < wave; ++w) next += part[w][lane];
    if (!on) return;
#pragma unroll 8
    for (int b = b0; b < b1; ++b) {
        int32_t* const c = p.counts + (int64_t)b * p.groups + g;
        const int n = *c;
        *c = next;
        next += n;
    }
    if (wave == waves - 1) p.counts[(int64_t)p.blocks * p.groups + g] = next;
}

// Lanes of the wave with this lane's key (keys of `bits` bits).
__device__ __forceinline__ uint64_t same_key(int key, int bits) {
    uint64_t m = ~0ull;
    for (int i = 0; i < bits; ++i) {
        const uint64_t set = __ballot(key >> i & 1);
        m &= key >> i & 1 ? set : ~set;
    }
    return m;
}

// Workgroup b places its pairs [b * per_block, ...), writes the padding rows of every blocks-th group and its share of
// the rows past the last group.  What it needs of the other pairs is how many of each expert there are, and how many
// before its own: from `counts`, or counted here.  Bound by its chain of dependent steps (ids, counts, scan, ranks, slots), not by
// bytes: 16 x 8 pairs over 256 groups 4.8 us, 32768 x 8 pairs 11 us (4.5 MB) behind 3.5 us of counting.
__global__ __launch_bounds__(kSortThreads) void sort_place_kernel(const SortParams p) {
    __shared__ int wave_next[kSortWaves][kMaxGroups + 1];   // counts of a wave's pairs, then its next row of each expert
    __shared__ int total[kMaxGroups], before[kMaxGroups], start[kMaxGroups + 1], wave_sum[kSortWaves];
    __shared__ uint16_t keys[kSortBlock];                   // of this workgroup's pairs (read from memory once)
    const int b = blockIdx.x + p.vbase, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int G = p.groups;
    const int first = b * p.per_block, last = min(p.pairs, first + p.per_block);
    for (int g = tid; g < G; g += kSortThreads) total[g] = before[g] = 0;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w)
        for (int g = tid; g <= G; g += kSortThreads) wave_next[w][g] = 0;
    __syncthreads();
    if (p.summed) {
        for (int g = tid; g < G; g += kSortThreads) {
            total[g] = p.counts[(int64_t)p.blocks * G + g];
            before[g] = p.counts[(int64_t)b * G + g];
        }
        for (int i = first + tid; i < last; i += kSortThreads) keys[i - first] = (uint16_t)key_of(p, i);
    } else if (p.counts != nullptr) {
        // a part of the blocks each, so that the loads of all parts are in flight
        const int parts = max(1, kSortThreads / G), part = tid / G;
        if (G >= kSortThreads) {
            for (int g = tid; g < G; g += kSortThreads) {
                int all = 0, mine = 0;
#pragma unroll 32
                for (int i = 0; i < p.blocks; ++i) {
                    const int c = p.counts[(int64_t)i * G + g];
                    all += c;
                    mine += i < b ? c : 0;
                }
                total[g] = all;
                before[g] = mine;
            }
        } else if (part < parts) {
            const int g = tid - part * G;
            int all = 0, mine = 0;
#pragma unroll 32
            for (int i = part; i < p.blocks; i += parts) {
                const int c = p.counts[(int64_t)i * G + g];
                all += c;
                mine += i < b ? c : 0;
            }
            atomicAdd(&total[g], all);
            atomicAdd(&before[g], mine);
        }
        for (int i = first + tid; i < last; i += kSortThreads) keys[i - first] = (uint16_t)key_of(p, i);
    } else {
#pragma unroll 4
        for (int i = tid; i < p.pairs; i += kSortThreads) {
            const int k = key_of(p, i);
            if (k < G) {
                atomicAdd(&total[k], 1);
                if (i < first) atomicAdd(&before[k], 1);
            }
            if (i >= first && i < last) keys[i - first] = (uint16_t)k;
        }
    }
    __syncthreads();
    // this wave's pairs: a run of whole batches of 64
    const int batches = ceil_div(max(0, last - first), 64), per_wave = ceil_div(batches, kSortWaves);
    const int w0 = first + wave * per_wave * 64, w1 = min(last, w0 + per_wave * 64);
    for (int i = w0 + lane; i < w1; i += 64) atomicAdd(&wave_next[wave][keys[i - first]], 1);
    __syncthreads();
    // first rows of the groups: scan over two groups a thread
    const int g0 = 2 * tid;
    const int n0 = g0 < G ? align_up(total[g0], p.alignment) : 0, n1 = g0 + 1 < G ? align_up(total[g0 + 1], p.alignment) : 0;
    int incl = n0 + n1;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int v = __shfl_up(incl, off, 64);
        if (lane >= off) incl += v;
    }
    if (lane == 63) wave_sum[wave] = incl;
    __syncthreads();
    int base = incl - n0 - n1;
    for (int w = 0; w < wave; ++w) base += wave_sum[w];
    if (g0 <= G) start[g0] = base;                  // (start[G]: the rows of all groups)
    if (g0 + 1 <= G) start[g0 + 1] = base + n0;
    if (G == kMaxGroups && g0 == G - 2) start[G] = base + n0 + n1;
    __syncthreads();
    for (int g = tid; g < G; g += kSortThreads) {
        int at = start[g] + before[g];
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) {
            const int n = wave_next[w][g];
            wave_next[w][g] = at;
            at += n;
        }
        if (b == 0) p.psum[g] = min(p.rows, start[g] + total[g]);
    }
    if (b == 0 && tid == 0 && start[G] > p.rows && p.status != nullptr) p.status[3] = 1u;
    __syncthreads();
    const int bits = 32 - __clz(G);
    for (int base_i = w0; base_i < w1; base_i += 64) {
        const int i = base_i + lane;
        const bool on = i < w1;
        const int key = on ? keys[i - first] : G;
        const uint64_t same = same_key(key, bits);
        const int rank = __popcll(same & ((1ull << lane) - 1));
        const int row = key < G ? wave_next[wave][key] + rank : -1;
        __builtin_amdgcn_wave_barrier();            // (every lane has read before a first lane moves the counter on)
        if (key < G && rank == 0) wave_next[wave][key] = row + __popcll(same);
        __builtin_amdgcn_wave_barrier();
        const bool fits = row >= 0 && row < p.rows;
        if (on) p.slots[i] = fits ? row : -1;
        if (on && fits) {
            p.source[row] = i;
            p.indices[row] = key;
        }
    }
    // padding rows: of every blocks-th group (16 lanes each: a group has few of them), then the rows past the last group
    const int sub = tid / 16, subs = kSortThreads / 16;
    for (int g = b + sub * p.blocks; g < G; g += subs * p.blocks) {
        const int end = min(p.rows, start[g + 1]);
        for (int r = start[g] + total[g] + (tid & 15); r < end; r += 16) p.source[r] = p.indices[r] = -1;
    }
    for (int64_t r = (int64_t)start[G] + b * kSortThreads + tid; r < p.rows; r += p.blocks * kSortThreads)
        p.source[r] = p.indices[r] = -1;
}

int sort_blocks(int pairs, int rows) {
    // One pass: blocks share out the placing (a batch for every wave) and the padding (16 x 8 pairs over 256 groups,
    // 4096 rows: 7.8 us on one block, 5.3 on eight).
    if (pairs <= kSortOnePass) return std::max({1, std::min(32, ceil_div(pairs, 512)), std::min(32, ceil_div(rows, 512))});
    // (every block reads the counts of all, so that more of them cost more than they share out)
    return std::max(std::min(kSortMaxBlocks, ceil_div(pairs, kSortPairs)), ceil_div(pairs, kSortBlock));
}

// ------------------------------------------------------------------------------------------------ rows
// A row is cut into chunks of 16 bytes; `lanes` threads (a power of two up to the workgroup) walk the chunks of one row
// and a workgroup holds 256 / lanes rows, so that short rows leave no lane idle and every access of a wave is one run
// of bytes of a row.  The last chunk ends with the row: where the row is no whole number of chunks it overlaps the one
// before, and both write the same values there.  Rows need no alignment (global memory takes 16 bytes at any address:
// 1021 x 6 pairs of 1407 fp32 values there and back with gradients: sums 9 us against 19 in single values).  Rows below 16 bytes go
// value by value.
constexpr int kRowThreads = 256;

int row_lanes(int64_t chunks) {
    int l = 8;
    while (l < kRowThreads && l < chunks) l <<= 1;
    return l;
}

// Workgroups that share the rows of `blocks` ones: for few tokens a row's chunks go beside each other rather than after each other
// (sums of 16 x 8 pairs of 7168 bf16 values 4.2 us, 9.5 with one workgroup a token; 256 x 8 7.0 and 14.2, 512 x 8 12.5 and 17.6), up to
// `most` workgroups in all: moving keeps four chunks of a thread in flight already (16 x 8 of 7168 fp32 values 4.5 and 6.9, but 256 x 8
// of bf16 8.4 and 7.8 with 1024 workgroups).
int row_parts(int64_t blocks, int chunks, int lanes, int most) {
    return (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(chunks, lanes), most / std::max<int64_t>(blocks, 1)));
}

typedef int i32x4_any __attribute__((ext_vector_type(4), aligned(1)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef int i32x4_half __attribute__((ext_vector_type(4), aligned(2)));

template <int V> struct Chunk;
template <> struct Chunk<16> { typedef i32x4 type; typedef i32x4_any mem; };
template <> struct Chunk<1> { typedef int8_t type; typedef int8_t mem; };

constexpr int kPadRows = 32;    // rows of a workgroup that clears padding: at the layout's end they come in thousands

// Rows of a layout that hold no pair are cleared by workgroups of kPadRows rows.
template <int V>
__device__ __forceinline__ void clear_padding(const int32_t* source, int rows, int first, uint8_t* dst, int64_t dst_ld,
                                              int64_t row_bytes) {
    typedef typename Chunk<V>::mem M;
    const int n = min(kPadRows, rows - first);
    const int mine = (int)(threadIdx.x & 63);
    uint64_t live = __ballot(mine < n && source[first + mine] < 0);
    while (live != 0) {
        const int r = __builtin_ctzll(live);
        live &= live - 1;
        uint8_t* const d = dst + (int64_t)(first + r) * dst_ld;
        for (int64_t at = (int64_t)threadIdx.x * V; at < row_bytes; at += kRowThreads * V)
            *reinterpret_cast<M*>(d + min(at, row_bytes - V)) = typename Chunk<V>::type{};
    }
}

struct DispatchParams {
    const uint8_t* src;
    uint8_t* dst;
    int64_t src_ld, dst_ld, row_bytes;
    const int32_t *slots, *source;
    int tokens, topk, rows, chunks, lanes;
    int parts;                 // workgroups that share a token's row
    int pad_blocks;            // first workgroups: padding rows (0: left as they are)
    int sf_blocks;             // next workgroups: scale factors (0: none)
    const int16_t* sf;         // [k64][sf_ld]
    int16_t* sf_out;           // [k64][sf_out_ld]
    int64_t sf_ld, sf_out_ld;
    int k64;
    int vbase;
};

constexpr int kSfRows = 512;    // rows of a workgroup that moves scale factors, two a thread

// Token rows to all their slots: each is read once and written topk times.  Bound by the bytes written: 8192 x 8 pairs of 4096
// bf16 values 104 us with the stores left in the last-level cache, 134 among other work (670 MB: 5.0 TB/s).
template <int V>
__global__ __launch_bounds__(kRowThreads) void dispatch_kernel(const DispatchParams p) {
    typedef typename Chunk<V>::type T;
    typedef typename Chunk<V>::mem M;
    int b = blockIdx.x + p.vbase;
    const int tid = threadIdx.x;
    if (b < p.pad_blocks) {
        clear_padding<V>(p.source, p.rows, b * kPadRows, p.dst, p.dst_ld, p.row_bytes);
        return;
    }
    b -= p.pad_blocks;
    if (b < p.sf_blocks) {
        // out[j][r] = sf[j][token of r]: two rows a thread, so that a store is a whole dword; zeros in padding rows
        const int per = ceil_div(p.rows, kSfRows), j = b / per, r = (b - j * per) * kSfRows + 2 * tid;
        if (r >= p.rows) return;
        const int16_t* const in = p.sf + (int64_t)j * p.sf_ld;
        u32 pair = 0;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int s = r + x < p.rows ? p.source[r + x] : -1, t = s < 0 || p.topk == 0 ? p.tokens : s / p.topk;
            if (t < p.tokens) pair |= (u32)(uint16_t)in[t] << (16 * x);
        }
        *reinterpret_cast<u32*>(p.sf_out + (int64_t)j * p.sf_out_ld + r) = pair;   // (an even leading dimension)
        return;
    }
    b -= p.sf_blocks;
    const int part = b % p.parts, step = p.lanes * p.parts;
    const int t = b / p.parts * (kRowThreads / p.lanes) + tid / p.lanes, c0 = part * p.lanes + tid % p.lanes;
    if (t >= p.tokens) return;
    const uint8_t* const in = p.src + (int64_t)t * p.src_ld;
    const int32_t* const slots = p.slots + (int64_t)t * p.topk;
    constexpr int U = 4;
    for (int c = c0; c < p.chunks; c += U * step) {
        T v[U];
        int64_t at[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            at[u] = min((int64_t)(c + u * step) * V, p.row_bytes - V);
            if (c + u * step < p.chunks) v[u] = *reinterpret_cast<const M*>(in + at[u]);
        }
        for (int k = 0; k < p.topk; ++k) {
            const int s = slots[k];
            if ((u32)s >= (u32)p.rows) continue;    // (dropped: -1)
            uint8_t* const d = p.dst + (int64_t)s * p.dst_ld;
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (c + u * step < p.chunks) *reinterpret_cast<M*>(d + at[u]) = v[u];
        }
    }
}

// N values of type E as they are loaded (16 bytes, or one value) and in fp32.  They stay as loaded until they are used:
// unpacked on arrival, the rows in flight took 94 registers of a thread (157 with the gradients) in place of 62 (128), and
// 8192 x 8 pairs of 4096 bf16 values 288 us with the gradients in place of 226.
template <typename E, int N> struct Raw;
template <> struct Raw<float, 4> { typedef f32x4 type; typedef f32x4_any mem; };
template <> struct Raw<uint16_t, 8> { typedef i32x4 type; typedef i32x4_half mem; };
template <> struct Raw<float, 1> { typedef float type; typedef float mem; };
template <> struct Raw<uint16_t, 1> { typedef uint16_t type; typedef uint16_t mem; };

template <typename E, int N>
__device__ __forceinline__ typename Raw<E, N>::type load_raw(const E* s) {
    return *reinterpret_cast<const typename Raw<E, N>::mem*>(s);
}

template <typename E, int N>
__device__ __forceinline__ void unpack(const typename Raw<E, N>::type w, float (&v)[N]) {
    if constexpr (sizeof(E) == 4 && N == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = w[i];
    } else if constexpr (N == 8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __builtin_bit_cast(float, (u32)w[i] << 16);
            v[2 * i + 1] = __builtin_bit_cast(float, (u32)w[i] & 0xffff0000u);
        }
    } else if constexpr (sizeof(E) == 4) {
        v[0] = w;
    } else {
        v[0] = bf16_to_f32(w);
    }
}

template <typename E, int N>
__device__ __forceinline__ void store_values(E* d, const float (&v)[N]) {
    if constexpr (sizeof(E) == 4 && N == 4) {
        *reinterpret_cast<f32x4_any*>(d) = f32x4{v[0], v[1], v[2], v[3]};
    } else if constexpr (sizeof(E) == 2 && N == 8) {
        *reinterpret_cast<i32x4_half*>(d) = i32x4{(int)pack_bf16x2(v[0], v[1]), (int)pack_bf16x2(v[2], v[3]),
                                            (int)pack_bf16x2(v[4], v[5]), (int)pack_bf16x2(v[6], v[7])};
    } else if constexpr (sizeof(E) == 4) {
        *d = v[0];
    } else {
        *d = f32_to_bf16_rne(v[0]);
    }
}

struct CombineParams {
    const void* rows_in;       // [rows][ld] of E
    const void* d_out;         // backward: [tokens][d_out_ld]
    void* out;                 // forward: [tokens][out_ld]; backward: gradient rows [rows][out_ld]
    float* d_weights;          // backward: [tokens][topk]
    const float* weights;      // [tokens][topk] or nullptr (ones)
    const int32_t *slots, *source;
    int64_t in_ld, out_ld, d_out_ld;   // elements
    int tokens, topk, rows, width, chunks, lanes, pad_blocks;
    int parts;                 // forward: workgroups that share a token's row
    int vbase;
};

constexpr int kChoices = 8;     // choices whose rows are in flight together

// out[t] = sum_c weight[t][c] * row[slot[t][c]], added in order in fp32 and rounded once.  Bound by the rows'
// bytes: 8192 x 8 pairs of 4096 bf16 values 124 us (604 MB: 4.9 TB/s), 140 to 160 behind a kernel whose stores are still going out.
template <typename E, int N>
__global__ __launch_bounds__(kRowThreads) void combine_kernel(const CombineParams p) {
    const int b = (blockIdx.x + p.vbase) / p.parts, part = (blockIdx.x + p.vbase) % p.parts, tid = threadIdx.x;
    const int t = b * (kRowThreads / p.lanes) + tid / p.lanes;
    if (t >= p.tokens) return;
    const int32_t* const slots = p.slots + (int64_t)t * p.topk;
    const float* const weights = p.weights + (int64_t)t * p.topk;
    E* const out = reinterpret_cast<E*>(p.out) + (int64_t)t * p.out_ld;
    const E* const in = reinterpret_cast<const E*>(p.rows_in);
    for (int c = part * p.lanes + tid % p.lanes; c < p.chunks; c += p.parts * p.lanes) {
        const int at = min(c * N, p.width - N);
        float sum[N] = {};
        for (int k0 = 0; k0 < p.topk; k0 += kChoices) {
            typename Raw<E, N>::type v[kChoices];
            float w[kChoices];
#pragma unroll
            for (int k = 0; k < kChoices; ++k) {
                const int s = k0 + k < p.topk ? slots[k0 + k] : -1;
                const bool live = (u32)s < (u32)p.rows;
                // (a dropped pair's weight is not used: whatever it is, it adds nothing)
                w[k] = !live ? 0.f : p.weights != nullptr ? weights[k0 + k] : 1.f;
                v[k] = typename Raw<E, N>::type{};
                if (live) v[k] = load_raw<E, N>(in + (int64_t)s * p.in_ld + at);
            }
#pragma unroll
            for (int k = 0; k < kChoices; ++k) {
                float x[N];
                unpack<E, N>(v[k], x);
#pragma unroll
                for (int i = 0; i < N; ++i) sum[i] = __builtin_fmaf(w[k], x[i], sum[i]);
            }
        }
        store_values<E, N>(out + at, sum);
    }
}

// d_row[slot[t][c]] = weight[t][c] * d_out[t], d_weight[t][c] = <d_out[t], row[slot[t][c]]>; padding rows get zeros.
// One pass: d_out once, the rows once, their gradients once.  The products are summed in fp32 along a thread's chunks,
// then over the row's threads in a fixed order.  Bound by those bytes: 8192 x 8 pairs of 4096 bf16 values 227 to 249 us (1.2 GB:
// 4.9 to 5.3 TB/s).
template <typename E, int N>
__global__ __launch_bounds__(kRowThreads) void combine_backward_kernel(const CombineParams p) {
    __shared__ float part[kRowThreads / 64][kChoices];
    int b = blockIdx.x + p.vbase;
    const int tid = threadIdx.x;
    if (b < p.pad_blocks) {
        clear_padding<(N == 1 ? 1 : 16)>(p.source, p.rows, b * kPadRows, reinterpret_cast<uint8_t*>(p.out), p.out_ld * (int)sizeof(E),
                                          (int64_t)p.width * (int)sizeof(E));
        return;
    }
    b -= p.pad_blocks;
    const int t = b * (kRowThreads / p.lanes) + tid / p.lanes, c0 = tid % p.lanes;
    const bool on = t < p.tokens;                   // (every thread takes part in the sums)
    const int32_t* const slots = p.slots + (int64_t)(on ? t : 0) * p.topk;
    const float* const weights = p.weights + (int64_t)(on ? t : 0) * p.topk;
    const E* const d_out = reinterpret_cast<const E*>(p.d_out) + (int64_t)(on ? t : 0) * p.d_out_ld;
    const E* const in = reinterpret_cast<const E*>(p.rows_in);
    E* const out = reinterpret_cast<E*>(p.out);
    for (int k0 = 0; k0 < p.topk; k0 += kChoices) {
        int s[kChoices];
        float w[kChoices], dot[kChoices];
#pragma unroll
        for (int k = 0; k < kChoices; ++k) {
            s[k] = on && k0 + k < p.topk ? slots[k0 + k] : -1;
            if ((u32)s[k] >= (u32)p.rows) s[k] = -1;
            w[k] = s[k] >= 0 ? weights[k0 + k] : 0.f;
            dot[k] = 0.f;
        }
        for (int c = c0; on && c < p.chunks; c += p.lanes) {
            const int at = min(c * N, p.width - N), counted = c * N - at;   // (values that the chunk before has counted)
            float g[N];
            typename Raw<E, N>::type v[kChoices];
            unpack<E, N>(load_raw<E, N>(d_out + at), g);
#pragma unroll
            for (int k = 0; k < kChoices; ++k)
                if (s[k] >= 0) v[k] = load_raw<E, N>(in + (int64_t)s[k] * p.in_ld + at);
#pragma unroll
            for (int k = 0; k < kChoices; ++k) {
                if (s[k] < 0) continue;
                float x[N], d[N];
                unpack<E, N>(v[k], x);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    if (i >= counted) dot[k] = __builtin_fmaf(g[i], x[i], dot[k]);
                    d[i] = w[k] * g[i];
                }
                store_values<E, N>(out + (int64_t)s[k] * p.out_ld + at, d);
            }
        }
#pragma unroll
        for (int k = 0; k < kChoices; ++k)
            for (int off = k0 + k < p.topk ? min(p.lanes, 64) / 2 : 0; off > 0; off >>= 1) dot[k] += __shfl_xor(dot[k], off, 64);
        if (p.lanes > 64) {
            if (k0 > 0) __syncthreads();            // (the last group's sums have been read)
            if ((tid & 63) == 0) {
#pragma unroll
                for (int k = 0; k < kChoices; ++k) part[tid >> 6][k] = dot[k];
            }
            __syncthreads();
            if (c0 == 0) {
#pragma unroll
                for (int k = 0; k < kChoices; ++k) {
                    dot[k] = 0.f;
                    for (int x = 0; x < p.lanes / 64; ++x) dot[k] += part[tid / 64 + x][k];
                }
            }
        }
        if (on && c0 == 0) {
#pragma unroll
            for (int k = 0; k < kChoices; ++k)
                if (k0 + k < p.topk) p.d_weights[(int64_t)t * p.topk + k0 + k] = dot[k];
        }
    }
}

int layout_ok(const dg_moe_layout* l, const char* who) {
    if (l == nullptr) return dg_set_error("dg_moe: null layout");
    if (l->tokens < 0 || l->topk < 0 || l->rows < 0 || l->tokens > kMaxExtent || l->rows > kMaxExtent ||
        (int64_t)l->tokens * l->topk > kMaxExtent)
        return dg_set_error(who);
    return DG_OK;
}

}  // namespace
}  // namespace dg

extern "C" int dg_moe_sort_workspace_size(int32_t num_pairs, int32_t num_groups, int64_t* bytes) {
    if (bytes == nullptr || num_pairs < 0 || num_groups < 1) return dg_set_error("dg_moe_sort: invalid size");
    const int64_t blocks = dg::sort_blocks(num_pairs, 0);
    *bytes = num_pairs <= dg::kSortOnePass ? 0 : (blocks + (blocks > dg::kSortMaxBlocks ? 1 : 0)) * num_groups * 4;
    return DG_OK;
}

extern "C" int dg_moe_sort(const void* ids, int32_t id_bytes, const dg_moe_layout* l, void* workspace, int64_t workspace_bytes,
                           int32_t num_cus, void* stream) {
    using namespace dg;
    if (const int rc = layout_ok(l, "dg_moe_sort: invalid size")) return rc;
    if (id_bytes != 4 && id_bytes != 8) return dg_set_error("dg_moe_sort: ids are int32 or int64");
    if (l->num_groups < 1 || l->num_groups > kMaxGroups) return dg_set_error("dg_moe_sort: 1 to 1024 groups");
    if (l->alignment < 1 || l->rows % l->alignment != 0) return dg_set_error("dg_moe_sort: rows must be a multiple of the alignment");
    const int64_t pairs = (int64_t)l->tokens * l->topk;
    // (first rows of the groups are 32-bit even where they pass the rows given)
    if (pairs + (int64_t)std::min<int64_t>(pairs, l->num_groups) * (l->alignment - 1) > 0x7fffffffLL)
        return dg_set_error("dg_moe_sort: too many rows");
    if ((pairs > 0 && (ids == nullptr || l->slots == nullptr)) || l->psum == nullptr ||
        (l->rows > 0 && (l->source == nullptr || l->m_indices == nullptr)))
        return dg_set_error("dg_moe_sort: null tensor");
    int64_t need = 0;
    (void)dg_moe_sort_workspace_size((int32_t)pairs, l->num_groups, &need);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need))
        return dg_set_error("dg_moe_sort: workspace smaller than dg_moe_sort_workspace_size() reports");
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    SortParams p = {};
    p.ids = ids;
    p.wide = id_bytes == 8;
    p.pairs = (int)pairs; p.groups = l->num_groups; p.alignment = l->alignment; p.rows = l->rows;
    p.blocks = sort_blocks(p.pairs, p.rows);
    p.per_block = ceil_div(std::max(1, p.pairs), p.blocks);
    p.slots = l->slots; p.source = l->source; p.indices = l->m_indices; p.psum = l->psum;
    p.counts = need > 0 ? reinterpret_cast<int32_t*>(workspace) : nullptr;
    p.status = status_words_for(st);
    p.summed = need > 0 && p.blocks > kSortMaxBlocks;
    if (need > 0)
        if (const int rc = launch_op(sort_count_kernel, p.blocks, kSortThreads, p, st, num_cus)) return rc;
    if (p.summed)
        if (const int rc = launch_op(sort_sum_kernel, ceil_div(p.groups, 64), kSumThreads, p, st, num_cus)) return rc;
    return launch_op(sort_place_kernel, p.blocks, kSortThreads, p, st, num_cus);
}

extern "C" int dg_moe_dispatch(const void* src, int64_t src_ld, int64_t row_bytes, const dg_moe_layout* l, void* dst, int64_t dst_ld,
                               const int16_t* sf, int64_t sf_ld, int32_t k64, int16_t* sf_out, int64_t sf_out_ld, int32_t zero_padding,
                               int32_t num_cus, void* stream) {
    using namespace dg;
    if (const int rc = layout_ok(l, "dg_moe_dispatch: invalid size")) return rc;
    if (row_bytes < 0 || (l->tokens > 1 && src_ld < row_bytes) || (l->rows > 1 && dst_ld < row_bytes))
        return dg_set_error("dg_moe_dispatch: leading dimension smaller than the row");
    if (sf != nullptr && (k64 < 0 || sf_ld < l->tokens || sf_out_ld < l->rows || sf_out_ld % 2 != 0 || sf_out == nullptr || !aligned_to(sf_out, 4)))
        return dg_set_error("dg_moe_dispatch: scale factors are [k64][ld], ld at least the rows and (out) even");
    if (l->rows == 0 || row_bytes == 0) return DG_OK;
    if (dst == nullptr || l->source == nullptr || (l->tokens > 0 && (src == nullptr || (l->topk > 0 && l->slots == nullptr))))
        return dg_set_error("dg_moe_dispatch: null tensor");
    const int v = row_bytes >= 16 ? 16 : 1;
    if (row_bytes > 0x7fffffffLL) return dg_set_error("dg_moe_dispatch: row too long");
    DispatchParams p = {};
    p.src = reinterpret_cast<const uint8_t*>(src); p.dst = reinterpret_cast<uint8_t*>(dst);
    p.src_ld = src_ld; p.dst_ld = dst_ld;
    p.slots = l->slots; p.source = l->source;
    p.tokens = l->tokens; p.topk = l->topk; p.rows = l->rows;
    p.row_bytes = row_bytes;
    p.chunks = (int)ceil_div64(row_bytes, v);
    p.lanes = row_lanes(p.chunks);
    p.pad_blocks = zero_padding ? ceil_div(l->rows, kPadRows) : 0;
    if (sf != nullptr && k64 > 0) {
        p.sf = sf; p.sf_out = sf_out; p.sf_ld = sf_ld; p.sf_out_ld = sf_out_ld; p.k64 = k64;
        const int64_t n = (int64_t)ceil_div(l->rows, kSfRows) * k64;
        if (n > 0x3fffffffLL) return dg_set_error("dg_moe_dispatch: too many scale factors");
        p.sf_blocks = (int)n;
    }
    const int64_t blocks = l->topk > 0 ? ceil_div(l->tokens, kRowThreads / p.lanes) : 0;
    p.parts = row_parts(blocks, p.chunks, p.lanes, 256);
    const int64_t grid = p.pad_blocks + (int64_t)p.sf_blocks + blocks * p.parts;
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    return launch_op(v == 16 ? dispatch_kernel<16> : dispatch_kernel<1>, grid, kRowThreads, p, st, num_cus);
}

namespace dg {
namespace {

// Threads of a token in the gradient, at most: eight chunks of its rows to each, where there are tokens enough, so that the sums
// over the threads stay small beside them (us with 64 and 256 threads: 8192 x 2 pairs of 2048 bf16 values 36 and 49, 8192 x 1 of
// 4096 48 and 57, 32768 x 4 of 1024 127 and 138; 8192 x 8 of 4096 261 and 250, 16 x 8 of 7168 39 and 27).
int backward_lanes(int tokens, int topk, int chunks) {
    int lanes = kRowThreads;
    while (tokens >= 1024 && lanes > 64 && (int64_t)chunks * topk < 8 * (int64_t)lanes) lanes /= 2;
    return lanes;
}

// n: values of a chunk
int combine_params(const dg_moe_layout* l, int64_t width, int n, CombineParams& p) {
    p.slots = l->slots; p.source = l->source;
    p.tokens = l->tokens; p.topk = l->topk; p.rows = l->rows;
    if (width > 0x3fffffffLL) return dg_set_error("dg_moe_combine: row too long");
    p.width = (int)width;
    p.chunks = ceil_div(p.width, n);
    p.lanes = row_lanes(p.chunks);
    return DG_OK;
}

}  // namespace
}  // namespace dg

extern "C" int dg_moe_combine(const void* rows, int64_t rows_ld, int32_t dtype, int64_t width, const dg_moe_layout* l,
                              const float* weights, void* out, int64_t out_ld, int32_t num_cus, void* stream) {
    using namespace dg;
    if (const int rc = layout_ok(l, "dg_moe_combine: invalid size")) return rc;
    if (dtype != DG_DTYPE_BF16 && dtype != DG_DTYPE_F32) return dg_set_error("dg_moe_combine: rows are bf16 or fp32");
    if (width < 0 || (l->rows > 1 && rows_ld < width) || (l->tokens > 1 && out_ld < width))
        return dg_set_error("dg_moe_combine: leading dimension smaller than the row");
    if (l->tokens == 0 || width == 0) return DG_OK;
    if (out == nullptr || (l->topk > 0 && l->slots == nullptr) || (l->rows > 0 && rows == nullptr)) return dg_set_error("dg_moe_combine: null tensor");
    const int64_t e = dtype == DG_DTYPE_F32 ? 4 : 2;
    if (!aligned_to(rows, e) || !aligned_to(out, e)) return dg_set_error("dg_moe_combine: values must be aligned");
    CombineParams p = {};
    p.rows_in = rows; p.out = out; p.weights = weights; p.in_ld = rows_ld; p.out_ld = out_ld;
    const bool f32 = dtype == DG_DTYPE_F32;
    const bool vec = width >= (f32 ? 4 : 8);
    if (const int rc = combine_params(l, width, !vec ? 1 : f32 ? 4 : 8, p)) return rc;
    const int64_t blocks = ceil_div(l->tokens, kRowThreads / p.lanes);
    p.parts = row_parts(blocks, p.chunks, p.lanes, 1024);
    const int64_t grid = blocks * p.parts;
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (f32) return launch_op(vec ? combine_kernel<float, 4> : combine_kernel<float, 1>, grid, kRowThreads, p, st, num_cus);
    return launch_op(vec ? combine_kernel<uint16_t, 8> : combine_kernel<uint16_t, 1>, grid, kRowThreads, p, st, num_cus);
}

extern "C" int dg_moe_combine_backward(const void* d_out, int64_t d_out_ld, const void* rows, int64_t rows_ld, int32_t dtype,
                                       int64_t width, const dg_moe_layout* l, const float* weights, void* d_rows, int64_t d_rows_ld,
                                       float* d_weights, int32_t num_cus, void* stream) {
    using namespace dg;
    if (const int rc = layout_ok(l, "dg_moe_combine_backward: invalid size")) return rc;
    if (dtype != DG_DTYPE_BF16 && dtype != DG_DTYPE_F32) return dg_set_error("dg_moe_combine_backward: rows are bf16 or fp32");
    if (width < 0 || (l->rows > 1 && (rows_ld < width || d_rows_ld < width)) || (l->tokens > 1 && d_out_ld < width))
        return dg_set_error("dg_moe_combine_backward: leading dimension smaller than the row");
    const int64_t pairs = (int64_t)l->tokens * l->topk;
    if ((pairs > 0 && (d_out == nullptr || l->slots == nullptr || weights == nullptr || d_weights == nullptr)) ||
        (l->rows > 0 && width > 0 && (rows == nullptr || d_rows == nullptr || l->source == nullptr)))
        return dg_set_error("dg_moe_combine_backward: null tensor");
    const int64_t e = dtype == DG_DTYPE_F32 ? 4 : 2;
    if (!aligned_to(rows, e) || !aligned_to(d_rows, e) || !aligned_to(d_out, e)) return dg_set_error("dg_moe_combine_backward: values must be aligned");
    CombineParams p = {};
    p.rows_in = rows; p.d_out = d_out; p.out = d_rows; p.weights = weights; p.d_weights = d_weights;
    p.in_ld = rows_ld; p.out_ld = d_rows_ld; p.d_out_ld = d_out_ld;
    const bool f32 = dtype == DG_DTYPE_F32;
    const bool vec = width >= (f32 ? 4 : 8);
    if (const int rc = combine_params(l, width, !vec ? 1 : f32 ? 4 : 8, p)) return rc;
    p.lanes = std::min(p.lanes, backward_lanes(l->tokens, l->topk, p.chunks));
    p.pad_blocks = width > 0 ? ceil_div(l->rows, kPadRows) : 0;
    const int64_t grid = p.pad_blocks + (int64_t)(l->topk > 0 ? ceil_div(l->tokens, kRowThreads / p.lanes) : 0);
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (f32) return launch_op(vec ? combine_backward_kernel<float, 4> : combine_backward_kernel<float, 1>, grid, kRowThreads, p, st, num_cus);
    return launch_op(vec ? combine_backward_kernel<uint16_t, 8> : combine_backward_kernel<uint16_t, 1>, grid, kRowThreads, p, st, num_cus);
}
