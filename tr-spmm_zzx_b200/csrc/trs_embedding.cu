// Embedding lookup with scaling, and its gradient.
//
//   out[i, :]  = scale * table[id_i, :]                 (product with the selection matrix of the ids)
//   grad[v, :] = scale * sum over i with id_i = v of dout[i, :]     (product with its transpose)
//
// An id equal to the padding id reads a row of zeros and gives no gradient.  An id outside the table reads a row of NaN
// (as sddmm answers a column outside its range) and gives no gradient: nothing is read or written out of bounds.
// Sums are in fp32 and in an order that the ids alone fix, so that results do not change from run to run; each result is
// rounded once.
#include "trs_types.cuh"

namespace trs {
namespace {

// Ids are 32 or 64 bits wide; the branch is the same for all threads.
__device__ __forceinline__ long long load_id(const void* __restrict__ ids, int ids64, long long i) {
    return ids64 ? __ldg((const long long*)ids + i) : (long long)__ldg((const int*)ids + i);
}

// ----------------------------------------------------------------------------------------------
// Lookup
// ----------------------------------------------------------------------------------------------
// A group of G lanes copies kLookupRows rows at a time, piece by piece, so that a thread has as many loads in flight.
constexpr int kThreads = 256, kLookupRows = 4;

template <class TI, class TO, int VEC, int G>
__global__ void __launch_bounds__(kThreads) k_lookup(const TI* __restrict__ table, long long rows, long long stride,
                                                     const void* __restrict__ ids, int ids64, long long n, int pieces, float scale,
                                                     long long padding, TO* __restrict__ out, long long out_stride) {
    const long long group = ((long long)blockIdx.x * kThreads + threadIdx.x) / G;
    const int lane = threadIdx.x % G;
    const long long i0 = group * kLookupRows;
    if (i0 >= n) return;
    const TI* from[kLookupRows];
    float mul[kLookupRows];
#pragma unroll
    for (int u = 0; u < kLookupRows; ++u) {
        const long long id = i0 + u < n ? load_id(ids, ids64, i0 + u) : -1;
        const bool pad = id == padding && padding != TRS_NO_PADDING, bad = (unsigned long long)id >= (unsigned long long)rows;
        from[u] = pad || bad ? nullptr : table + id * stride + lane * VEC;
        mul[u] = pad ? 0.f : bad ? __int_as_float(0x7fffffff) : scale;   // what zeros are multiplied by where there is no row
    }
    TO* to = out + i0 * out_stride + lane * VEC;
    for (int c = lane; c < pieces; c += G) {
        Piece<TI, VEC> p[kLookupRows];
#pragma unroll
        for (int u = 0; u < kLookupRows; ++u) {
            p[u] = Piece<TI, VEC>{};
            if (from[u]) p[u] = *(const Piece<TI, VEC>*)(from[u] + (c - lane) * VEC);
        }
#pragma unroll
        for (int u = 0; u < kLookupRows; ++u)
            if (i0 + u < n) *(Piece<TO, VEC>*)(to + u * out_stride + (c - lane) * VEC) = scaled<TO>(p[u], mul[u]);
    }
}

// ----------------------------------------------------------------------------------------------
// Positions sorted by id
// ----------------------------------------------------------------------------------------------
// Stable, so that a row's positions ascend.  Positions without a row (padding, outside the table) get the key `rows` and come last.
// The keys have bits(rows) bits, sorted by up to 11 at a time: two passes for tables of up to 4 M rows.  Pass: the counts of
// each digit in each tile, their prefix sums over the tiles, then every key to its place.
constexpr int kSortThreads = 512, kSortWarps = kSortThreads / 32, kSortItems = 16, kTile = kSortThreads * kSortItems, kMaxDigit = 11;

__device__ __forceinline__ unsigned key_of(long long id, long long rows, long long padding) {
    return id == padding || id < 0 || id >= rows ? (unsigned)rows : (unsigned)id;
}

// FIRST: keys are made from the ids (and the segments of all rows are emptied); otherwise they are the last pass's.
template <bool FIRST>
__global__ void __launch_bounds__(kSortThreads) k_digit_counts(const void* __restrict__ ids, int ids64, long long rows, long long padding,
                                                               const unsigned* __restrict__ keys, int n, int shift, int digit_bits,
                                                               int* __restrict__ counts, int2* __restrict__ segment) {
    extern __shared__ int s_count[];
    if (!FIRST) wait_for_kernel_before();
    const int bins = 1 << digit_bits, tiles = gridDim.x;
    for (int b = threadIdx.x; b < bins; b += kSortThreads) s_count[b] = 0;
    __syncthreads();
    const int base = blockIdx.x * kTile;
    unsigned key[kSortItems];
#pragma unroll
    for (int k = 0; k < kSortItems; ++k) {
        const int i = base + k * kSortThreads + threadIdx.x;
        if (i < n && i >= 0) key[k] = FIRST ? key_of(load_id(ids, ids64, i), rows, padding) : keys[i];
    }
#pragma unroll
    for (int k = 0; k < kSortItems; ++k) {
        const int i = base + k * kSortThreads + threadIdx.x;
        if (i < n && i >= 0) atomicAdd(&s_count[(key[k] >> shift) & (bins - 1)], 1);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += kSortThreads) counts[(size_t)b * tiles + blockIdx.x] = s_count[b];
    if (FIRST)
        for (long long v = (long long)blockIdx.x * kSortThreads + threadIdx.x; v < rows; v += (long long)tiles * kSortThreads)
            segment[v] = make_int2(0, 0);
}

// counts[bin, tile] -> the number of keys with that digit in earlier tiles; total[bin].  One warp a bin.
__global__ void __launch_bounds__(256) k_digit_prefix(int* __restrict__ counts, int tiles, int bins, int* __restrict__ total) {
    const int bin = (blockIdx.x * 256 + threadIdx.x) / 32, lane = threadIdx.x % 32;
    wait_for_kernel_before();
    if (bin >= bins) return;
    int* c = counts + (size_t)bin * tiles;
    int sum = 0;
    for (int t0 = 0; t0 < tiles; t0 += 32) {
        const int x = t0 + lane < tiles ? c[t0 + lane] : 0;
        int incl = x;
        for (int o = 1; o < 32; o *= 2) {
            const int y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        if (t0 + lane < tiles) c[t0 + lane] = sum + incl - x;
        sum += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) total[bin] = sum;
}

// A warp has 16 x 32 neighbouring keys of the tile and ranks them by its own counters, 32 at a time: lanes with one digit find each
// other, the first of them counts for all.
template <bool FIRST>
__global__ void __launch_bounds__(kSortThreads) k_digit_scatter(const void* __restrict__ ids, int ids64, long long rows, long long padding,
                                                                const unsigned* __restrict__ keys, const int* __restrict__ pos, int n,
                                                                int shift, int digit_bits, const int* __restrict__ counts,
                                                                const int* __restrict__ total, unsigned* __restrict__ keys_out,
                                                                int* __restrict__ pos_out) {
    extern __shared__ int s_mem[];
    const int bins = 1 << digit_bits, tiles = gridDim.x, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    int* s_base = s_mem;                                            // [bins] place of the tile's first key of a digit
    unsigned short* s_rank = (unsigned short*)(s_mem + bins);       // [warps][bins]
    __shared__ int s_sum[kSortWarps];
    for (int k = threadIdx.x; k < bins * kSortWarps / 2; k += kSortThreads) ((int*)s_rank)[k] = 0;
    wait_for_kernel_before();
    // prefix sums of the digits' totals: each thread has bins / threads neighbouring ones
    const int per = (bins + kSortThreads - 1) / kSortThreads, b0 = threadIdx.x * per;
    int mine = 0;
    for (int b = b0; b < b0 + per && b < bins; ++b) mine += total[b];
    int incl = mine;
    for (int o = 1; o < 32; o *= 2) {
        const int y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
    }
    if (lane == 31) s_sum[warp] = incl;
    __syncthreads();
    int at = incl - mine;
    for (int w = 0; w < warp; ++w) at += s_sum[w];
    for (int b = b0; b < b0 + per && b < bins; ++b) {
        s_base[b] = at + counts[(size_t)b * tiles + blockIdx.x];
        at += total[b];
    }
    const int first = blockIdx.x * kTile + warp * (kSortItems * 32) + lane;
    unsigned key[kSortItems];
    unsigned short rank[kSortItems];
    unsigned short* my = s_rank + warp * bins;
#pragma unroll
    for (int k = 0; k < kSortItems; ++k) {
        const int i = first + k * 32;
        key[k] = i < n && i >= 0 ? (FIRST ? key_of(load_id(ids, ids64, i), rows, padding) : keys[i]) : 0u;
    }
    for (int k = 0; k < kSortItems; ++k) {
        const int i = first + k * 32;
        const bool in = i < n && i >= 0;
        const unsigned digit = in ? (key[k] >> shift) & (bins - 1) : (unsigned)bins;   // lanes past the end match each other only
        const unsigned same = __match_any_sync(0xffffffffu, digit);
        const int before = __popc(same & ((1u << lane) - 1));
        int r = 0;
        if (in) r = my[digit] + before;
        __syncwarp();
        if (in && before == 0) my[digit] += (unsigned short)__popc(same);
        __syncwarp();
        rank[k] = (unsigned short)r;
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += kSortThreads) {   // counters of a digit -> keys of it in the warps before
        int sum = 0;
        for (int w = 0; w < kSortWarps; ++w) {
            const int x = s_rank[w * bins + b];
            s_rank[w * bins + b] = (unsigned short)sum;
            sum += x;
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSortItems; ++k) {
        const int i = first + k * 32;
        if (i >= n || i < 0) continue;
        const unsigned digit = (key[k] >> shift) & (bins - 1);
        const int to = s_base[digit] + my[digit] + rank[k];
        keys_out[to] = key[k];
        pos_out[to] = FIRST ? i : pos[i];
    }
}

// Up to kFewIds ids: one CTA sorts (key, position) words in shared memory by a bitonic network, the other CTAs empty the segments.
// (4 K ids of a 16 K row table by the digit passes: six launches, 25 us of them; this one 5 us.)
constexpr int kFewIds = 4096, kFewThreads = 1024;

__global__ void __launch_bounds__(kFewThreads) k_sort_few(const void* __restrict__ ids, int ids64, long long rows, long long padding, int n,
                                                          int size, unsigned* __restrict__ keys_out, int* __restrict__ pos_out,
                                                          int2* __restrict__ segment) {
    const int threads = blockDim.x;   // up to half of `size`, the power of two from 64 on that holds n
    if (blockIdx.x) {
        for (long long v = (long long)(blockIdx.x - 1) * threads + threadIdx.x; v < rows; v += (long long)(gridDim.x - 1) * threads)
            segment[v] = make_int2(0, 0);
        return;
    }
    __shared__ unsigned long long s_word[kFewIds];
    for (int i = threadIdx.x; i < size; i += threads)
        s_word[i] = i < n ? (unsigned long long)key_of(load_id(ids, ids64, i), rows, padding) << 32 | (unsigned)i : ~0ull;
    __syncthreads();
    for (int run = 2; run <= size; run *= 2) {
        for (int o = run / 2; o; o /= 2) {
            for (int i = threadIdx.x; i < size / 2; i += threads) {
                const int lo = 2 * i - (i & (o - 1)), hi = lo + o;
                const unsigned long long a = s_word[lo], b = s_word[hi];
                if ((a > b) == ((lo & run) == 0)) {
                    s_word[lo] = b;
                    s_word[hi] = a;
                }
            }
            // 32 neighbouring pairs of a distance up to 32 are 64 words of their own
            if (o > 32 || (o == 1 && run >= 64)) __syncthreads();
            else __syncwarp();
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += threads) {
        keys_out[i] = (unsigned)(s_word[i] >> 32);
        pos_out[i] = (int)(unsigned)s_word[i];
    }
}

// ----------------------------------------------------------------------------------------------
// Sums of equal ids
// ----------------------------------------------------------------------------------------------
// The sorted positions are cut into blocks of 64 and spans of several blocks.  A block whose positions all name one row is summed
// ahead (a span of one row as a whole), all of them in parallel, so that a row with a hundred thousand positions is not one
// group's work; k_sums then walks a row's segment and takes a span's or a block's sum where the segment holds all of it.
constexpr int kBlock = 64, kSpanWarps = kThreads / 32;

template <class T, int VEC>
__device__ __forceinline__ void add_row(float (&acc)[VEC], const T* __restrict__ row, int c) {
    add_piece(acc, *(const Piece<T, VEC>*)(row + (size_t)c * VEC));
}

// The sum of the 64 rows whose positions the warp's lanes hold (pa: the first 32), at piece c of a group of G lanes; the groups of the warp
// take the positions in turn, and their sums are added in a fixed order.  All lanes come along.
template <class T, int VEC, int G>
__device__ __forceinline__ void sum_block(float (&acc)[VEC], const T* __restrict__ g, long long stride, int pa, int pb, int c, int pieces) {
    constexpr int GROUPS = 32 / G;
    const int group = threadIdx.x % 32 / G;
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
#pragma unroll 8
    for (int i = 0; i < kBlock / GROUPS; ++i) {
        const int j = i * GROUPS + group, p = __shfl_sync(0xffffffffu, i < kBlock / GROUPS / 2 ? pa : pb, j % 32);
        if (c < pieces) add_row<T, VEC>(acc, g + (size_t)p * stride, c);
    }
#pragma unroll
    for (int o = G; o < 32; o *= 2)
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] += __shfl_xor_sync(0xffffffffu, acc[k], o);
}

// One CTA a span: notes where segments begin and end, and sums its uniform blocks.
template <class T, int VEC, int G>
__global__ void __launch_bounds__(kThreads) k_block_sums(const T* __restrict__ g, long long stride, const unsigned* __restrict__ keys,
                                                         const int* __restrict__ pos, int n, unsigned rows, int F, int span,
                                                         int2* __restrict__ segment, float* __restrict__ block_sum,
                                                         float* __restrict__ span_sum) {
    wait_for_kernel_before();
    const int p0 = blockIdx.x * span, p1 = min(n - p0, span) + p0;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, pieces = F / VEC;
    const bool whole = p1 - p0 == span && keys[p0] == keys[p1 - 1] && keys[p0] < rows;
    for (int b = p0 + warp * kBlock; b < p1; b += kSpanWarps * kBlock) {
        const int i0 = b + lane, i1 = i0 + 32;
        const unsigned none = ~0u, k0 = i0 < n ? keys[i0] : none, k1 = i1 < n ? keys[i1] : none;
        unsigned edge = none;   // the keys around the block
        if (lane == 0 && b > 0) edge = keys[b - 1];
        if (lane == 31 && b + kBlock < n) edge = keys[b + kBlock];
        const unsigned k0_up = __shfl_up_sync(none, k0, 1), k1_up = __shfl_up_sync(none, k1, 1), k0_down = __shfl_down_sync(none, k0, 1),
                       k1_down = __shfl_down_sync(none, k1, 1), k0_last = __shfl_sync(none, k0, 31), k1_first = __shfl_sync(none, k1, 0);
        auto note = [&](int i, unsigned k, unsigned before, unsigned after) {
            if (k >= rows) return;
            if (before != k && after != k) segment[k] = make_int2(i, i + 1);
            else if (before != k) segment[k].x = i;
            else if (after != k) segment[k].y = i + 1;
        };
        note(i0, k0, lane ? k0_up : edge, lane < 31 ? k0_down : k1_first);
        note(i1, k1, lane ? k1_up : k0_last, lane < 31 ? k1_down : edge);
        if (whole) continue;
        const unsigned key = __shfl_sync(none, k0, 0);
        if (!__all_sync(none, k0 == key && k1 == key) || key >= rows) continue;   // (the end of the list is not: none)
        const int pa = pos[i0], pb = pos[i1];
        for (int c0 = 0; c0 < pieces; c0 += G) {
            const int c = c0 + lane % G;
            float acc[VEC];
            sum_block<T, VEC, G>(acc, g, stride, pa, pb, c, pieces);
            if (c < pieces && lane < G)
#pragma unroll
                for (int k = 0; k < VEC; ++k) block_sum[(size_t)(b / kBlock) * F + c * VEC + k] = acc[k];
        }
    }
    if (!whole) return;   // the same for all threads of the CTA
    __shared__ float s_part[kSpanWarps][G * VEC];
    for (int c0 = 0; c0 < pieces; c0 += G) {
        const int c = c0 + lane % G;
        float sum[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) sum[k] = 0.f;
        for (int b = p0 + warp * kBlock; b < p1; b += kSpanWarps * kBlock) {
            float acc[VEC];
            sum_block<T, VEC, G>(acc, g, stride, pos[b + lane], pos[b + 32 + lane], c, pieces);
#pragma unroll
            for (int k = 0; k < VEC; ++k) sum[k] += acc[k];
        }
        __syncthreads();
        if (lane < G)
#pragma unroll
            for (int k = 0; k < VEC; ++k) s_part[warp][lane * VEC + k] = sum[k];
        __syncthreads();
        for (int f = threadIdx.x; f < G * VEC; f += kThreads) {
            float s = 0.f;
            for (int w = 0; w < kSpanWarps; ++w) s += s_part[w][f];
            if (c0 * VEC + f < F) span_sum[(size_t)blockIdx.x * F + c0 * VEC + f] = s;
        }
    }
}

// A group of G lanes writes kSumRows neighbouring rows, G pieces of each.  Their positions are neighbours too: where no row has a block's
// worth of them, the group streams through them, kSumBatch at a time, and writes a row when the key changes; otherwise it goes
// row by row and takes the blocks' and spans' sums.
constexpr int kSumRows = 8, kSumBatch = 8, kPartBatch = 4;

template <class TO, int VEC>
__device__ __forceinline__ void write_sum(TO* __restrict__ o, const float (&acc)[VEC], float scale, int accumulate) {
    Piece<TO, VEC> q;
    if (accumulate) q = *(Piece<TO, VEC>*)o;
#pragma unroll
    for (int k = 0; k < VEC; ++k) q.v[k] = from_float<TO>(accumulate ? fmaf(scale, acc[k], as_float(q.v[k])) : scale * acc[k]);
    *(Piece<TO, VEC>*)o = q;
}

template <class TI, class TO, int VEC, int G>
__global__ void __launch_bounds__(kThreads) k_sums(const TI* __restrict__ g, long long stride, const unsigned* __restrict__ keys,
                                                   const int* __restrict__ pos, int n, long long rows, int F, int slabs, int span,
                                                   const int2* __restrict__ segment, const float* __restrict__ block_sum,
                                                   const float* __restrict__ span_sum, float scale, TO* __restrict__ out,
                                                   long long out_stride, int accumulate) {
    wait_for_kernel_before();
    const long long item = ((long long)blockIdx.x * kThreads + threadIdx.x) / G, set = slabs == 1 ? item : item / slabs;
    const long long v0 = set * kSumRows;
    const int c = (slabs == 1 ? 0 : (int)(item - set * slabs) * G) + threadIdx.x % G;
    if (v0 >= rows || c >= F / VEC) return;
    g += (size_t)c * VEC;
    out += v0 * out_stride + (size_t)c * VEC;
    int begin = n, end_all = 0;
    bool blocks = false;
    {
        int2 s[kSumRows];
#pragma unroll
        for (int u = 0; u < kSumRows; ++u) s[u] = n > 0 && v0 + u < rows ? segment[v0 + u] : make_int2(0, 0);
#pragma unroll
        for (int u = 0; u < kSumRows; ++u) {
            if (s[u].x < s[u].y) {
                begin = min(begin, s[u].x);
                end_all = max(end_all, s[u].y);
                blocks |= s[u].y - s[u].x >= kBlock;
            } else if (!accumulate && v0 + u < rows) {
                *(Piece<TO, VEC>*)(out + u * out_stride) = Piece<TO, VEC>{};
            }
        }
    }
    if (!blocks) {
        float acc[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
        for (int p = begin; p < end_all; p += kSumBatch) {
            int at[kSumBatch];
            unsigned key[kSumBatch + 1];
#pragma unroll
            for (int k = 0; k < kSumBatch; ++k) at[k] = p + k < end_all ? pos[p + k] : -1;
#pragma unroll
            for (int k = 0; k <= kSumBatch; ++k) key[k] = p + k < end_all ? keys[p + k] : ~0u;
            Piece<TI, VEC> row[kSumBatch];
#pragma unroll
            for (int k = 0; k < kSumBatch; ++k)
                if (at[k] >= 0) row[k] = *(const Piece<TI, VEC>*)(g + (size_t)at[k] * stride);
#pragma unroll
            for (int k = 0; k < kSumBatch; ++k) {
                if (at[k] < 0) break;
                add_piece(acc, row[k]);
                if (key[k] == key[k + 1]) continue;
                write_sum<TO, VEC>(out + (long long)(key[k] - (unsigned)v0) * out_stride, acc, scale, accumulate);
#pragma unroll
                for (int q = 0; q < VEC; ++q) acc[q] = 0.f;
            }
        }
        return;
    }
#pragma unroll 1
    for (int u = 0; u < kSumRows; ++u) {
        if (v0 + u >= rows) break;
        const int2 s = segment[v0 + u];
        int p = s.x;
        const int end = s.y;
        if (p == end) continue;
        float acc[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
        while (p < end) {
            // whole blocks and spans from their sums, single positions otherwise
            if ((p & (kBlock - 1)) == 0 && p + kBlock <= end) {
                const bool spans = p % span == 0 && p + span <= end;
                const int step = spans ? span : kBlock;
                const float* from = (spans ? span_sum + (size_t)(p / span) * F : block_sum + (size_t)(p / kBlock) * F) + c * VEC;
                // blocks up to the next span (which is taken as one) or the segment's end
                const int stop = spans ? end : min(end, p - p % span + span), count = min((stop - p) / step, kPartBatch);
                Piece<float, VEC> part[kPartBatch];
#pragma unroll
                for (int k = 0; k < kPartBatch; ++k)
#pragma unroll
                    for (int q = 0; q < VEC; ++q) part[k].v[q] = k < count ? from[(size_t)k * F + q] : 0.f;
#pragma unroll
                for (int k = 0; k < kPartBatch; ++k)
#pragma unroll
                    for (int q = 0; q < VEC; ++q) acc[q] += part[k].v[q];
                p += count * step;
            } else {
                const int stop = min(end, (p & ~(kBlock - 1)) + kBlock);
                Piece<TI, VEC> row[kSumBatch];
                int at[kSumBatch];
#pragma unroll
                for (int k = 0; k < kSumBatch; ++k) at[k] = p + k < stop ? pos[p + k] : -1;
#pragma unroll
                for (int k = 0; k < kSumBatch; ++k) {
                    row[k] = Piece<TI, VEC>{};
                    if (at[k] >= 0) row[k] = *(const Piece<TI, VEC>*)(g + (size_t)at[k] * stride);
                }
#pragma unroll
                for (int k = 0; k < kSumBatch; ++k) add_piece(acc, row[k]);
                p = min(p + kSumBatch, stop);
            }
        }
        write_sum<TO, VEC>(out + u * out_stride, acc, scale, accumulate);
    }
}

// ----------------------------------------------------------------------------------------------
// Host side
// ----------------------------------------------------------------------------------------------

// Elements per load and store: as many as 16 bytes hold of the wider type, fewer where rows do not begin on such boundaries.
int elements_per_piece(int F, const void* a, int type_a, long long stride_a, const void* b, int type_b, long long stride_b) {
    const int wide = type_bytes(type_a) > type_bytes(type_b) ? type_bytes(type_a) : type_bytes(type_b);
    for (int vec = 16 / wide; vec > 1; vec /= 2) {
        const size_t in = (size_t)vec * type_bytes(type_a), out = (size_t)vec * type_bytes(type_b);
        if (F % vec == 0 && (uintptr_t)a % in == 0 && stride_a % vec == 0 && (uintptr_t)b % out == 0 && stride_b % vec == 0) return vec;
    }
    return 1;
}

template <class Fn>
int with_vec(int vec, Fn fn) {
    if (vec == 8) return fn(std::integral_constant<int, 8>());
    if (vec == 4) return fn(std::integral_constant<int, 4>());
    if (vec == 2) return fn(std::integral_constant<int, 2>());
    return fn(std::integral_constant<int, 1>());
}

// Lanes per row: a power of two that covers the row's pieces, 4 to 32.
template <class Fn>
int with_group(int pieces, Fn fn) {
    if (pieces <= 4) return fn(std::integral_constant<int, 4>());
    if (pieces <= 8) return fn(std::integral_constant<int, 8>());
    if (pieces <= 16) return fn(std::integral_constant<int, 16>());
    return fn(std::integral_constant<int, 32>());
}

constexpr long long kMaxIds = (1ll << 31) - (1 << 16), kMaxRows = (1ll << 31) - 2;
constexpr int kMaxFeatures = 1 << 20;

struct GradPlan {
    int digits = 0, digit_bits = 0, tiles = 0, span = 0, spans = 0;
    size_t keys[2] = {}, pos[2] = {}, counts = 0, total = 0, segment = 0, block_sum = 0, span_sum = 0, bytes = 0;
};

GradPlan grad_plan(long long n, long long rows, int F) {
    GradPlan p;
    int bits = 1;
    while (bits < 32 && (rows >> bits)) ++bits;   // keys 0 .. rows
    p.digits = (bits + kMaxDigit - 1) / kMaxDigit;
    p.digit_bits = (bits + p.digits - 1) / p.digits;
    p.tiles = (int)ceil_div64(n, kTile);
    // spans: up to about a thousand of them, of 512 positions or more
    p.span = kBlock * kSpanWarps;
    while (p.span < (1 << 20) && (long long)p.span * 1024 < n) p.span *= 2;
    p.spans = (int)ceil_div64(n, p.span);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) & ~(size_t)255;
        return here;
    };
    for (int k = 0; k < 2; ++k) {
        p.keys[k] = take((size_t)n * 4);
        p.pos[k] = take((size_t)n * 4);
    }
    p.counts = take(((size_t)p.tiles << p.digit_bits) * 4);
    p.total = take((size_t)4 << p.digit_bits);
    p.segment = take((size_t)rows * 8);
    p.block_sum = take((size_t)(n / kBlock) * F * 4);
    p.span_sum = take((size_t)p.spans * F * 4);
    p.bytes = at;
    return p;
}

int check_sizes(long long rows, long long n, int F) {
    if (rows < 1 || n < 0 || F < 1) return TRS_E_ARG;
    if (rows > kMaxRows || n > kMaxIds || F > kMaxFeatures) return TRS_E_LIMIT;
    return TRS_OK;
}

std::atomic<unsigned long long> g_scatter_done[2];

template <bool FIRST>
int sort_pass(const void* ids, int ids64, long long rows, long long padding, unsigned char* ws, const GradPlan& p, int n, int pass,
              cudaStream_t st) {
    const int from = (pass + 1) & 1, to = pass & 1, shift = pass * p.digit_bits, bins = 1 << p.digit_bits;
    const unsigned* keys = (const unsigned*)(ws + p.keys[from]);
    const int* pos = (const int*)(ws + p.pos[from]);
    int *counts = (int*)(ws + p.counts), *total = (int*)(ws + p.total);
    int rc = launch_behind(k_digit_counts<FIRST>, dim3(p.tiles), kSortThreads, (size_t)bins * 4, st, !FIRST, ids, ids64, rows, padding, keys, n, shift,
                    p.digit_bits, counts, (int2*)(ws + p.segment));
    if (rc) return rc;
    rc = launch_behind(k_digit_prefix, dim3(ceil_div(bins, 8)), 256, 0, st, true, counts, p.tiles, bins, total);
    if (rc) return rc;
    const size_t smem = (size_t)bins * (4 + 2 * kSortWarps);
    rc = allow_smem(k_digit_scatter<FIRST>, (1 << kMaxDigit) * (4 + 2 * kSortWarps), false, g_scatter_done[FIRST]);
    if (rc) return rc;
    return launch_behind(k_digit_scatter<FIRST>, dim3(p.tiles), kSortThreads, smem, st, true, ids, ids64, rows, padding, keys, pos, n, shift, p.digit_bits,
                  (const int*)counts, (const int*)total, (unsigned*)(ws + p.keys[to]), (int*)(ws + p.pos[to]));
}

}  // namespace
}  // namespace trs

using namespace trs;

extern "C" int trs_embedding(const void* table, int table_type, long long rows, long long table_stride, const void* ids, int ids64,
                             long long n, int F, float scale, long long padding_id, void* out, int out_type, long long out_stride,
                             void* stream) try {
    const int rc = check_sizes(rows, n, F);
    if (rc) return rc;
    if (!type_known(table_type) || !type_known(out_type) || table_stride < F || out_stride < F) return TRS_E_ARG;
    if (n == 0) return TRS_OK;
    if (!table || !ids || !out) return TRS_E_ARG;
    const int vec = elements_per_piece(F, table, table_type, table_stride, out, out_type, out_stride), pieces = F / vec;
    return with_type(table_type, [&](auto ti) {
        return with_type(out_type, [&](auto to) {
            using TI = decltype(ti);
            using TO = decltype(to);
            return with_vec(vec, [&](auto v) {
                constexpr int VEC = decltype(v)::value;
                if constexpr (VEC * (sizeof(TI) > sizeof(TO) ? sizeof(TI) : sizeof(TO)) > 16) {
                    return (int)TRS_E_ARG;   // not reached: elements_per_piece
                } else {
                    return with_group(pieces, [&](auto gr) {
                        constexpr int G = decltype(gr)::value;
                        const long long groups = ceil_div64(n, kLookupRows);
                        return launch(k_lookup<TI, TO, VEC, G>, dim3((unsigned)ceil_div64(groups * G, kThreads)), kThreads, 0,
                                      (cudaStream_t)stream, (const TI*)table, rows, table_stride, ids, ids64, n, pieces, scale, padding_id,
                                      (TO*)out, out_stride);
                    });
                }
            });
        });
    });
}
TRS_CATCH

extern "C" int trs_embedding_grad_workspace_bytes(long long n, long long rows, int F, size_t* bytes) try {
    if (!bytes) return TRS_E_ARG;
    const int rc = check_sizes(rows, n, F);
    if (rc) return rc;
    *bytes = n ? grad_plan(n, rows, F).bytes : 0;
    return TRS_OK;
}
TRS_CATCH

extern "C" int trs_embedding_grad(const void* grad, int grad_type, long long grad_stride, const void* ids, int ids64, long long n,
                                  long long rows, int F, float scale, long long padding_id, void* out, int out_type, long long out_stride,
                                  int accumulate, void* workspace, size_t workspace_bytes, void* stream) try {
    int rc = check_sizes(rows, n, F);
    if (rc) return rc;
    if (!type_known(grad_type) || !type_known(out_type) || grad_stride < F || out_stride < F || !out) return TRS_E_ARG;
    if (n && (!grad || !ids)) return TRS_E_ARG;
    if (n == 0 && accumulate) return TRS_OK;
    const cudaStream_t st = (cudaStream_t)stream;
    GradPlan p;
    unsigned char* ws = (unsigned char*)workspace;
    if (n) {
        p = grad_plan(n, rows, F);
        if (!ws || workspace_bytes < p.bytes || (uintptr_t)ws % 16) return TRS_E_WORKSPACE;
        if (n <= kFewIds) {
            p.digits = 1;   // (the result is where a first pass leaves it)
            int size = 64;
            while (size < n) size *= 2;
            const int threads = size / 2 < kFewThreads ? size / 2 : kFewThreads;
            const long long zero = ceil_div64(rows, 4 * threads);
            rc = launch(k_sort_few, dim3(1 + (unsigned)(zero < 2 * 148 ? zero : 2 * 148)), threads, 0, st, ids, ids64, rows, padding_id, (int)n, size, (unsigned*)(ws + p.keys[0]),
                        (int*)(ws + p.pos[0]), (int2*)(ws + p.segment));
            if (rc) return rc;
        } else for (int pass = 0; pass < p.digits; ++pass) {
            rc = pass == 0 ? sort_pass<true>(ids, ids64, rows, padding_id, ws, p, (int)n, pass, st)
                           : sort_pass<false>(ids, ids64, rows, padding_id, ws, p, (int)n, pass, st);
            if (rc) return rc;
        }
    }
    const int last = (p.digits + 1) & 1;
    const unsigned* keys = (const unsigned*)(ws + p.keys[last]);
    const int* pos = (const int*)(ws + p.pos[last]);
    int2* segment = (int2*)(ws + p.segment);
    float *block_sum = (float*)(ws + p.block_sum), *span_sum = (float*)(ws + p.span_sum);
    const int vec = elements_per_piece(F, grad, grad_type, grad_stride, out, out_type, out_stride), pieces = F / vec;
    return with_type(grad_type, [&](auto ti) {
        using TI = decltype(ti);
        return with_vec(vec, [&](auto v) {
            constexpr int VEC = decltype(v)::value;
            if constexpr (VEC * sizeof(TI) > 16) {
                return (int)TRS_E_ARG;   // not reached: elements_per_piece
            } else {
                return with_group(pieces, [&](auto gr) {
                    constexpr int G = decltype(gr)::value;
                    if (n) {
                        const int e = launch_behind(k_block_sums<TI, VEC, G>, dim3(p.spans), kThreads, 0, st, true, (const TI*)grad, grad_stride, keys, pos,
                                                    (int)n, (unsigned)rows, F, p.span, segment, block_sum, span_sum);
                        if (e) return e;
                    }
                    return with_type(out_type, [&](auto to) {
                        using TO = decltype(to);
                        if constexpr (VEC * sizeof(TO) > 16) {
                            return (int)TRS_E_ARG;   // not reached: elements_per_piece
                        } else {
                            const int slabs = ceil_div(pieces, G);
                            const long long threads = ceil_div64(rows, kSumRows) * slabs * G;
                            if (ceil_div64(threads, kThreads) > 0x7fffffffll) return (int)TRS_E_LIMIT;
                            return launch_behind(k_sums<TI, TO, VEC, G>, dim3((unsigned)ceil_div64(threads, kThreads)), kThreads, 0, st, n > 0,
                                                 (const TI*)grad, grad_stride, keys, pos, (int)n, rows, F, slabs, p.span, (const int2*)segment,
                                                 (const float*)block_sum, (const float*)span_sum, scale, (TO*)out, out_stride, accumulate);
                        }
                    });
                });
            }
        });
    });
}
TRS_CATCH
