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
// A group of G lanes copies ROWS rows at a time, PER pieces a lane, so that a thread has ROWS x PER loads in flight, with no branch around
// them.  COPY: the result has the table's type and the factor is 1, so the bits are moved as they are.  Bound by DRAM: 2^20
// popular rows of 128 fp16 features 66 us, 5.1 TB/s of the rows that are named, the ids and the result.
constexpr int kThreads = 256, kLookupThreads = 128;

template <class TI, class TO, int VEC, int G, int ROWS, int PER, bool COPY>
__global__ void __launch_bounds__(kLookupThreads, 8) k_lookup(const TI* __restrict__ table, unsigned rows, unsigned stride,
                                                           const void* __restrict__ ids, int ids64, unsigned n, int pieces, float scale,
                                                           long long padding, TO* __restrict__ out, unsigned out_stride) {
    const unsigned i0 = (blockIdx.x * (kLookupThreads / G) + threadIdx.x / G) * ROWS;   // below 2^32 wherever a CTA is
    int c = threadIdx.x % G;
    if (i0 >= n) return;
    const TI* from[ROWS];
    bool none[ROWS];   // no row to read: the result is zeros times `mul`
    float mul[ROWS];
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
        const long long id = load_id(ids, ids64, min(i0 + u, n - 1));
        const bool pad = id == padding && padding != TRS_NO_PADDING;
        none[u] = pad || (unsigned long long)id >= rows;
        mul[u] = pad ? 0.f : none[u] ? __int_as_float(0x7fffffff) : scale;
        from[u] = table + (size_t)(none[u] ? 0u : (unsigned)id) * stride;   // (row 0 in its place: no branch around the load)
    }
    TO* to = out + (size_t)i0 * out_stride;
    for (; c < pieces; c += PER * G) {
        Piece<TI, VEC> p[ROWS][PER];
#pragma unroll
        for (int u = 0; u < ROWS; ++u)
#pragma unroll
            for (int i = 0; i < PER; ++i) p[u][i] = *(const Piece<TI, VEC>*)(from[u] + min(c + i * G, pieces - 1) * VEC);
#pragma unroll
        for (int u = 0; u < ROWS; ++u) {
            if (i0 + u >= n) break;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                if (i && c + i * G >= pieces) break;
                if (none[u]) {
#pragma unroll
                    for (int k = 0; k < VEC; ++k) p[u][i].v[k] = from_float<TI>(COPY ? mul[u] : 0.f);
                }
                Piece<TO, VEC>* o = (Piece<TO, VEC>*)(to + (size_t)u * out_stride + (c + i * G) * VEC);
                if constexpr (COPY) *o = *(const Piece<TO, VEC>*)&p[u][i];
                else *o = scaled<TO>(p[u][i], mul[u]);
            }
        }
    }
}

// ----------------------------------------------------------------------------------------------
// Positions sorted by id
// ----------------------------------------------------------------------------------------------
// Stable, so that a row's positions ascend.  Positions without a row (padding, outside the table) get the key `rows` and come last.
// The keys have bits(rows) bits, sorted by up to 11 (from 2^19 ids on: 8) at a time: two (three) passes for tables of up to 4 M rows.
// Pass: the counts of each digit in each tile, their prefix sums over the tiles, then every key to its place.
constexpr int kSortThreads = 512, kSortWarps = kSortThreads / 32, kSortItems = 8, kTile = kSortThreads * kSortItems, kMaxDigit = 11;

__device__ __forceinline__ unsigned key_of(long long id, long long rows, long long padding) {
    return id == padding || id < 0 || id >= rows ? (unsigned)rows : (unsigned)id;
}

// All segments empty, and no row popular, by `threads` threads; two at a time (the array begins on a 16-byte boundary and has room for an even number).
__device__ __forceinline__ void empty_segments(int2* __restrict__ segment, int* __restrict__ popular, long long rows, long long me,
                                               long long threads) {
    if (me == 0) *popular = 0;
    for (long long v = me; v < (rows + 1) / 2; v += threads) ((int4*)segment)[v] = make_int4(0, 0, 0, 0);
}

// FIRST: keys are made from the ids (and the segments of all rows are emptied); otherwise they are the last pass's.
template <bool FIRST>
__global__ void __launch_bounds__(kSortThreads) k_digit_counts(const void* __restrict__ ids, int ids64, long long rows, long long padding,
                                                               const uint2* __restrict__ words, int n, int shift, int digit_bits,
                                                               int* __restrict__ counts, int2* __restrict__ segment, int* __restrict__ popular) {
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
        if (i < n && i >= 0) key[k] = FIRST ? key_of(load_id(ids, ids64, i), rows, padding) : words[i].x;
    }
#pragma unroll
    for (int k = 0; k < kSortItems; ++k) {
        const int i = base + k * kSortThreads + threadIdx.x;
        if (i < n && i >= 0) atomicAdd(&s_count[(key[k] >> shift) & (bins - 1)], 1);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += kSortThreads) counts[(size_t)b * tiles + blockIdx.x] = s_count[b];
    if (FIRST)
        empty_segments(segment, popular, rows, (long long)blockIdx.x * kSortThreads + threadIdx.x, (long long)tiles * kSortThreads);
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

// A warp has kSortItems x 32 neighbouring words of the tile and ranks them by its own counters, 32 at a time: lanes with one digit find
// each other by a vote on each bit, the first of them counts for all.  The tile is put in order in shared memory first: a store
// of 32 scattered words takes an SM 32 cycles, and a tile's words of one digit go to neighbouring places.
template <bool FIRST>
__global__ void __launch_bounds__(kSortThreads, 2) k_digit_scatter(const void* __restrict__ ids, int ids64, long long rows, long long padding,
                                                                const uint2* __restrict__ words, int n, int shift, int digit_bits,
                                                                const int* __restrict__ counts, const int* __restrict__ total,
                                                                uint2* __restrict__ words_out) {
    extern __shared__ __align__(16) unsigned char s_mem[];
    const int bins = 1 << digit_bits, tiles = gridDim.x, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    uint2* s_word = (uint2*)s_mem;                                              // [kTile]
    int* s_to = (int*)(s_word + kTile);                                         // [bins] a digit's first place, less its first place in the tile
    unsigned short* s_rank = (unsigned short*)(s_to + bins);                    // [warps][bins]
    unsigned short* s_start = s_rank + kSortWarps * bins;                       // [bins] a digit's first place in the tile
    __shared__ int s_sum[kSortWarps], s_sum_tile[kSortWarps];
    for (int k = threadIdx.x; k < bins * kSortWarps / 2; k += kSortThreads) ((int*)s_rank)[k] = 0;
    wait_for_kernel_before();
    const int base = blockIdx.x * kTile, first = base + warp * (kSortItems * 32) + lane;
    uint2 word[kSortItems];
    unsigned short rank[kSortItems];
    unsigned short* my = s_rank + warp * bins;
#pragma unroll
    for (int k = 0; k < kSortItems; ++k) {
        const int i = first + k * 32;
        word[k] = make_uint2(0, 0);
        if (i < n && i >= 0) word[k] = FIRST ? make_uint2(key_of(load_id(ids, ids64, i), rows, padding), i) : words[i];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSortItems; ++k) {
        const int i = first + k * 32;
        const bool in = i < n && i >= 0;
        const unsigned digit = (word[k].x >> shift) & (bins - 1);
        unsigned same = __ballot_sync(0xffffffffu, in);
#pragma unroll
        for (int b = 0; b < kMaxDigit; ++b) {
            if (b >= digit_bits) break;
            const unsigned vote = __ballot_sync(0xffffffffu, digit >> b & 1);
            same &= digit >> b & 1 ? vote : ~vote;
        }
        const int before = __popc(same & ((1u << lane) - 1));
        int r = 0;
        if (in) r = my[digit] + before;
        __syncwarp();
        if (in && before == 0) my[digit] += (unsigned short)__popc(same);
        __syncwarp();
        rank[k] = (unsigned short)r;
    }
    __syncthreads();
    // Prefix sums over the digits, of all keys and of the tile's: each thread has bins / threads neighbouring pairs of digits (16 bits
    // hold a tile's counts, so two digits are added in one word).  A digit's counters become the number of its keys in the warps before.
    const int pairs = bins / 2, per = (pairs + kSortThreads - 1) / kSortThreads, b0 = threadIdx.x * per;
    int all = 0, here = 0;
    for (int b = b0; b < b0 + per && b < pairs; ++b) {
        all += total[2 * b] + total[2 * b + 1];
        unsigned sum = 0;
#pragma unroll
        for (int w = 0; w < kSortWarps; ++w) {
            const unsigned x = ((unsigned*)s_rank)[w * pairs + b];
            ((unsigned*)s_rank)[w * pairs + b] = sum;
            sum += x;
        }
        ((unsigned*)s_start)[b] = sum;   // for the second round
        here += (sum & 0xffff) + (sum >> 16);
    }
    int incl = all, incl_tile = here;
    for (int o = 1; o < 32; o *= 2) {
        const int y = __shfl_up_sync(0xffffffffu, incl, o), z = __shfl_up_sync(0xffffffffu, incl_tile, o);
        if (lane >= o) incl += y, incl_tile += z;
    }
    if (lane == 31) s_sum[warp] = incl, s_sum_tile[warp] = incl_tile;
    __syncthreads();
    int at = incl - all, at_tile = incl_tile - here;
    for (int w = 0; w < warp; ++w) at += s_sum[w], at_tile += s_sum_tile[w];
    for (int b = 2 * b0; b < 2 * (b0 + per) && b < bins; ++b) {
        const int sum = s_start[b];
        s_to[b] = at + counts[(size_t)b * tiles + blockIdx.x] - at_tile;
        s_start[b] = (unsigned short)at_tile;
        at += total[b];
        at_tile += sum;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSortItems; ++k) {
        const int i = first + k * 32;
        const unsigned digit = (word[k].x >> shift) & (bins - 1);
        if (i < n && i >= 0) s_word[s_start[digit] + my[digit] + rank[k]] = word[k];
    }
    __syncthreads();
    const int count = min(n - base, kTile);
#pragma unroll
    for (int k = 0; k < kSortItems; ++k) {
        const int i = k * kSortThreads + threadIdx.x;
        if (i >= count) break;
        const uint2 w = s_word[i];
        words_out[s_to[(w.x >> shift) & (bins - 1)] + i] = w;
    }
}

// Up to a tile of ids: one CTA does all passes in shared memory, the other CTAs empty the segments.
// (4 096 ids of a table of 16 384 rows: 11 us; one id more, six launches, 24 us and as much again on the host.  A bitonic network: 36 us.)
constexpr int kFewIds = kTile, kFewDigit = 8, kFewBins = 1 << kFewDigit;

__global__ void __launch_bounds__(kSortThreads) k_sort_few(const void* __restrict__ ids, int ids64, long long rows, long long padding, int n,
                                                           int bits, uint2* __restrict__ words_out, int2* __restrict__ segment,
                                                           int* __restrict__ popular) {
    if (blockIdx.x) {
        empty_segments(segment, popular, rows, (long long)(blockIdx.x - 1) * kSortThreads + threadIdx.x, (long long)(gridDim.x - 1) * kSortThreads);
        return;
    }
    __shared__ uint2 s_word[kFewIds];
    __shared__ unsigned short s_rank[kSortWarps][kFewBins], s_start[kFewBins];
    __shared__ int s_sum[kFewBins / 64];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int rounds = (n + kSortThreads - 1) / kSortThreads, first = warp * (rounds * 32) + lane;   // a warp has neighbouring words
    uint2 word[kSortItems];
    unsigned short rank[kSortItems];
#pragma unroll
    for (int k = 0; k < kSortItems; ++k) {
        const int i = first + k * 32;
        word[k] = make_uint2(0, 0);
        if (k < rounds && i < n) word[k] = make_uint2(key_of(load_id(ids, ids64, i), rows, padding), i);
    }
    for (int shift = 0; shift < bits; shift += kFewDigit) {
        for (int k = threadIdx.x; k < kSortWarps * kFewBins / 2; k += kSortThreads) ((unsigned*)s_rank)[k] = 0;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kSortItems; ++k) {
            if (k >= rounds) break;
            const bool in = first + k * 32 < n;
            const unsigned digit = (word[k].x >> shift) & (kFewBins - 1);
            unsigned same = __ballot_sync(0xffffffffu, in);
#pragma unroll
            for (int b = 0; b < kFewDigit; ++b) {
                const unsigned vote = __ballot_sync(0xffffffffu, digit >> b & 1);
                same &= digit >> b & 1 ? vote : ~vote;
            }
            const int before = __popc(same & ((1u << lane) - 1));
            int r = 0;
            if (in) r = s_rank[warp][digit] + before;
            __syncwarp();
            if (in && before == 0) s_rank[warp][digit] += (unsigned short)__popc(same);
            __syncwarp();
            rank[k] = (unsigned short)r;
        }
        __syncthreads();
        // a pair of digits a thread: counters become the words of the digit in the warps before; then places of the digits
        unsigned sum = 0;
        int here = 0, incl = 0;
        if (threadIdx.x < kFewBins / 2) {
#pragma unroll
            for (int w = 0; w < kSortWarps; ++w) {
                unsigned* c = (unsigned*)&s_rank[w][2 * threadIdx.x];
                const unsigned x = *c;
                *c = sum;
                sum += x;
            }
            here = incl = (int)(sum & 0xffff) + (int)(sum >> 16);
            for (int o = 1; o < 32; o *= 2) {
                const int y = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += y;
            }
            if (lane == 31) s_sum[warp] = incl;
        }
        __syncthreads();
        if (threadIdx.x < kFewBins / 2) {
            int at = incl - here;
            for (int w = 0; w < warp; ++w) at += s_sum[w];
            s_start[2 * threadIdx.x] = (unsigned short)at;
            s_start[2 * threadIdx.x + 1] = (unsigned short)(at + (sum & 0xffff));
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kSortItems; ++k) {
            const unsigned digit = (word[k].x >> shift) & (kFewBins - 1);
            if (k < rounds && first + k * 32 < n) s_word[s_start[digit] + s_rank[warp][digit] + rank[k]] = word[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kSortItems; ++k)
            if (k < rounds && first + k * 32 < n) word[k] = s_word[first + k * 32];
    }
    for (int i = threadIdx.x; i < n; i += kSortThreads) words_out[i] = s_word[i];
}

// ----------------------------------------------------------------------------------------------
// Sums of equal ids
// ----------------------------------------------------------------------------------------------
// The sorted positions are cut into blocks of 64 and spans of several blocks.  A block whose positions all name one row is summed
// ahead (a span of one row as a whole), all of them in parallel, so that a row with a hundred thousand positions is not one
// group's work.  Rows with kPopular positions or more are noted in a list (popular[0] of them, in any order) and get a CTA each, the
// first ones of k_sums: as part of their neighbours' work a hub was its last 60 us where others were done, and 2^20 popular ids of a table
// whose rows are in the order of their popularity took 336 us where the same ids spread over it took 196 (now 197 and 195; from 16 positions
// on 184, but 600 k ids of 50 k rows 99 us for 77).
constexpr int kBlock = 64, kSpanWarps = kThreads / 32, kPopular = 24;

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
    constexpr int BATCH = 8;
    for (int i0 = 0; i0 < kBlock / GROUPS; i0 += BATCH) {
        Piece<T, VEC> row[BATCH];
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            const int j = (i0 + k) * GROUPS + group, p = __shfl_sync(0xffffffffu, j < 32 ? pa : pb, j % 32);
            row[k] = Piece<T, VEC>{};
            if (c < pieces) row[k] = *(const Piece<T, VEC>*)(g + (size_t)p * stride + (size_t)c * VEC);
        }
#pragma unroll
        for (int k = 0; k < BATCH; ++k) add_piece(acc, row[k]);
    }
#pragma unroll
    for (int o = G; o < 32; o *= 2)
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] += __shfl_xor_sync(0xffffffffu, acc[k], o);
}

// One CTA a span: notes where segments begin and end, and sums its uniform blocks.  (Four CTAs an SM leave 64 registers, and what the
// compiler wants beyond them lies in local memory: 64 to 80 bytes a thread for fp16 in pieces of eight, about 250 for bf16, 728 for single
// fp32 elements by 32 lanes.  The bound was chosen on fp16; the whole gradient of 2^20 bf16 rows of 128 takes 195 us as that of fp16 does.)
template <class T, int VEC, int G>
__global__ void __launch_bounds__(kThreads, 4) k_block_sums(const T* __restrict__ g, long long stride, const uint2* __restrict__ words, int n, unsigned rows, int F, int span,
                                                         int2* __restrict__ segment, float* __restrict__ block_sum,
                                                         float* __restrict__ span_sum, int* __restrict__ popular) {
    wait_for_kernel_before();
    const int p0 = blockIdx.x * span, p1 = min(n - p0, span) + p0;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, pieces = F / VEC;
    const bool whole = p1 - p0 == span && words[p0].x == words[p1 - 1].x && words[p0].x < rows;
    for (int b = p0 + warp * kBlock; b < p1; b += kSpanWarps * kBlock) {
        const int i0 = b + lane, i1 = i0 + 32;
        const unsigned none = ~0u;
        const uint2 w0 = i0 < n ? words[i0] : make_uint2(none, 0), w1 = i1 < n ? words[i1] : make_uint2(none, 0);
        const unsigned k0 = w0.x, k1 = w1.x;
        unsigned edge = none;   // the keys around the block
        if (lane == 0 && b > 0) edge = words[b - 1].x;
        if (lane == 31 && b + kBlock < n) edge = words[b + kBlock].x;
        const unsigned k0_up = __shfl_up_sync(none, k0, 1), k1_up = __shfl_up_sync(none, k1, 1), k0_down = __shfl_down_sync(none, k0, 1),
                       k1_down = __shfl_down_sync(none, k1, 1), k0_last = __shfl_sync(none, k0, 31), k1_first = __shfl_sync(none, k1, 0);
        auto note = [&](int i, unsigned k, unsigned before, unsigned after) {
            if (k >= rows) return;
            if (before != k && after == k && i < n - (kPopular - 1) && words[i + kPopular - 1].x == k)
                popular[1 + atomicAdd(popular, 1)] = (int)k;
            if (before != k && after != k) segment[k] = make_int2(i, i + 1);
            else if (before != k) segment[k].x = i;
            else if (after != k) segment[k].y = i + 1;
        };
        note(i0, k0, lane ? k0_up : edge, lane < 31 ? k0_down : k1_first);
        note(i1, k1, lane ? k1_up : k0_last, lane < 31 ? k1_down : edge);
        const unsigned key = __shfl_sync(none, k0, 0);
        if (!__all_sync(none, k0 == key && k1 == key) || key >= rows) continue;   // (the end of the list is not: none)
        if (whole) continue;
        const int pa = (int)w0.y, pb = (int)w1.y;
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
            sum_block<T, VEC, G>(acc, g, stride, (int)words[b + lane].y, (int)words[b + 32 + lane].y, c, pieces);
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

// A group of G lanes writes ROWS neighbouring rows, G pieces of each.  Their positions are neighbours too: where none of the rows is
// popular, the group streams through them, kSumBatch at a time, and writes a row when the key changes; otherwise it goes row by row.
constexpr int kSumThreads = 128, kSumBatch = 4;

__device__ __forceinline__ bool is_popular(int2 s) { return s.y - s.x >= kPopular; }

template <class TO, int VEC>
__device__ __forceinline__ void write_sum(TO* __restrict__ o, const float (&acc)[VEC], float scale, int accumulate) {
    Piece<TO, VEC> q;
    if (accumulate) q = *(Piece<TO, VEC>*)o;
#pragma unroll
    for (int k = 0; k < VEC; ++k) q.v[k] = from_float<TO>(accumulate ? fmaf(scale, acc[k], as_float(q.v[k])) : scale * acc[k]);
    *(Piece<TO, VEC>*)o = q;
}

// What k_sums gets.
template <class TI, class TO>
struct SumArgs {
    const TI* g;
    long long stride;
    const uint2* words;
    int n;
    long long rows;
    int F, slabs, span;
    const int2* segment;
    const float *block_sum, *span_sum;
    const int* popular;
    int popular_ctas;
    float scale;
    TO* out;
    long long out_stride;
    int accumulate;
};

// A popular row by a CTA: its groups of lanes take the positions outside whole blocks, the blocks outside whole spans and the
// spans in turn, and their sums are added in order.
template <class TI, class TO, int VEC, int G>
__device__ __forceinline__ void sum_popular(const SumArgs<TI, TO>& a, long long v, float (*s_part)[G * VEC]) {
    constexpr int GROUPS = kSumThreads / G;
    const int group = threadIdx.x / G, lane = threadIdx.x % G, pieces = a.F / VEC;
    const int2 s = a.segment[v];
    int b0 = (s.x + kBlock - 1) & ~(kBlock - 1), b1 = s.y & ~(kBlock - 1);                // whole blocks
    if (b0 > b1) b0 = b1 = s.y;
    const int t0 = (int)min(((long long)b0 + a.span - 1) / a.span * a.span, (long long)b1), t1 = max(b1 / a.span * a.span, t0);   // whole spans
    const int head = b0 - s.x, singles = head + s.y - b1;
    const int before = (t0 - b0) / kBlock, spans = (t1 - t0) / a.span, parts = before + spans + (b1 - t1) / kBlock;
    for (int c0 = 0; c0 < pieces; c0 += G) {
        const int c = c0 + lane;
        float acc[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
        if (c < pieces) {
#pragma unroll 4
            for (int i = group; i < singles; i += GROUPS)
                add_row<TI, VEC>(acc, a.g + (size_t)a.words[i < head ? s.x + i : b1 + i - head].y * a.stride, c);
#pragma unroll 4
            for (int i = group; i < parts; i += GROUPS) {
                const float* from = i < before           ? a.block_sum + (size_t)(b0 / kBlock + i) * a.F
                                    : i < before + spans ? a.span_sum + (size_t)(t0 / a.span + i - before) * a.F
                                                         : a.block_sum + (size_t)(t1 / kBlock + i - before - spans) * a.F;
#pragma unroll
                for (int k = 0; k < VEC; ++k) acc[k] += from[c * VEC + k];
            }
        }
#pragma unroll
        for (int k = 0; k < VEC; ++k) s_part[group][lane * VEC + k] = acc[k];
        __syncthreads();
        if (group == 0 && c < pieces) {
            for (int w = 1; w < GROUPS; ++w)
#pragma unroll
                for (int k = 0; k < VEC; ++k) acc[k] += s_part[w][lane * VEC + k];
            write_sum<TO, VEC>(a.out + v * a.out_stride + (size_t)c * VEC, acc, a.scale, a.accumulate);
        }
        __syncthreads();
    }
}

template <class TI, class TO, int VEC, int G, int ROWS>
__global__ void __launch_bounds__(kSumThreads) k_sums(const SumArgs<TI, TO> a) {
    __shared__ float s_part[kSumThreads / G][G * VEC];
    wait_for_kernel_before();
    if ((int)blockIdx.x < a.popular_ctas) {
        for (int i = blockIdx.x; i < a.popular[0]; i += a.popular_ctas) sum_popular<TI, TO, VEC, G>(a, a.popular[1 + i], s_part);
        return;
    }
    const long long item = ((long long)(blockIdx.x - a.popular_ctas) * kSumThreads + threadIdx.x) / G;
    const long long set = a.slabs == 1 ? item : item / a.slabs, v0 = set * ROWS;
    const int c = (a.slabs == 1 ? 0 : (int)(item - set * a.slabs) * G) + threadIdx.x % G;
    if (v0 >= a.rows || c >= a.F / VEC) return;
    const TI* __restrict__ g = a.g + (size_t)c * VEC;
    TO* __restrict__ out = a.out + v0 * a.out_stride + (size_t)c * VEC;
    int begin = a.n, end_all = 0;
    bool popular = false;
    {
        int2 s[ROWS];
#pragma unroll
        for (int u = 0; u < ROWS; ++u) s[u] = a.n > 0 ? a.segment[min(v0 + u, a.rows - 1)] : make_int2(0, 0);
#pragma unroll
        for (int u = 0; u < ROWS; ++u) {
            if (s[u].x < s[u].y && v0 + u < a.rows) {
                begin = min(begin, s[u].x);
                end_all = max(end_all, s[u].y);
                popular |= is_popular(s[u]);
            } else if (!a.accumulate && v0 + u < a.rows) {
                *(Piece<TO, VEC>*)(out + u * a.out_stride) = Piece<TO, VEC>{};
            }
        }
    }
    // the rows of positions [p, end), written when the key changes
    auto stream = [&](int p, int end) {
        float acc[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
        for (; p < end; p += kSumBatch) {
            uint2 w[kSumBatch + 1];
#pragma unroll
            for (int k = 0; k <= kSumBatch; ++k) w[k] = p + k < end ? a.words[p + k] : make_uint2(~0u, 0);
            Piece<TI, VEC> row[kSumBatch];
#pragma unroll
            for (int k = 0; k < kSumBatch; ++k)
                if (p + k < end) row[k] = *(const Piece<TI, VEC>*)(g + (size_t)w[k].y * a.stride);
#pragma unroll
            for (int k = 0; k < kSumBatch; ++k) {
                if (p + k >= end) break;
                add_piece(acc, row[k]);
                if (w[k].x == w[k + 1].x) continue;
                write_sum<TO, VEC>(out + (long long)(w[k].x - (unsigned)v0) * a.out_stride, acc, a.scale, a.accumulate);
#pragma unroll
                for (int q = 0; q < VEC; ++q) acc[q] = 0.f;
            }
        }
    };
    const int runs = popular ? ROWS : 1;
    for (int u = 0; u < runs; ++u) {
        int2 s = make_int2(begin, end_all);
        if (popular) {
            s = v0 + u < a.rows ? a.segment[v0 + u] : make_int2(0, 0);
            if (is_popular(s)) continue;
        }
        stream(s.x, s.y);
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

// Lookup: lanes, rows and pieces in flight.  Few lanes a row spare instructions (what a lane spends on a row's id and address is as much
// as it spends on three pieces): F = 47 of fp32 rows, single elements as in all odd widths, 27 us with 32 lanes x 4 rows, 17 us with
// 16 lanes x 2 rows x 3 pieces.  That fits 33 to 48 pieces; longer rows take further turns of 48, in the last of which lanes without a piece load the
// row's last one again.  The kernel keeps to 64 registers: 2^20 rows of 128 fp16 features 77 us with 66 of them, 66 with 64, 79 with 40.
template <class Fn>
int with_lookup(int pieces, Fn fn) {
    using std::integral_constant;
    if (pieces <= 4) return fn(integral_constant<int, 4>(), integral_constant<int, 4>(), integral_constant<int, 1>());
    if (pieces <= 8) return fn(integral_constant<int, 4>(), integral_constant<int, 4>(), integral_constant<int, 2>());
    if (pieces <= 16) return fn(integral_constant<int, 8>(), integral_constant<int, 4>(), integral_constant<int, 2>());
    if (pieces <= 32) return fn(integral_constant<int, 16>(), integral_constant<int, 2>(), integral_constant<int, 2>());
    return fn(integral_constant<int, 16>(), integral_constant<int, 2>(), integral_constant<int, 3>());
}

constexpr long long kManyIds = 1 << 19;
constexpr long long kMaxIds = (1ll << 31) - (1 << 16), kMaxRows = (1ll << 31) - 2;
constexpr long long kMaxStride = (1ll << 31) - 1;
constexpr int kMaxFeatures = 1 << 20;

struct GradPlan {
    int bits = 0, digits = 0, digit_bits = 0, tiles = 0, span = 0, spans = 0;
    size_t words[2] = {}, counts = 0, total = 0, segment = 0, block_sum = 0, span_sum = 0, popular = 0, bytes = 0;
};

GradPlan grad_plan(long long n, long long rows, int F) {
    GradPlan p;
    int bits = 1;
    while (bits < 32 && (rows >> bits)) ++bits;   // keys 0 .. rows
    p.bits = bits;
    // Narrow digits cost a pass more and far less per pass (2^20 ids: two passes of 11 bits 67 us, three of 7 bits 55); the launches
    // decide where ids are few.
    const int widest = n >= kManyIds ? 8 : kMaxDigit;
    p.digits = (bits + widest - 1) / widest;
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
    for (int k = 0; k < 2; ++k) p.words[k] = take((size_t)n * 8);
    p.counts = take(((size_t)p.tiles << p.digit_bits) * 4);
    p.total = take((size_t)4 << p.digit_bits);
    p.segment = take((size_t)(rows + 1) * 8);
    p.block_sum = take((size_t)(n / kBlock) * F * 4);
    p.span_sum = take((size_t)p.spans * F * 4);
    p.popular = take((size_t)(n / kPopular + 1) * 4);
    p.bytes = at;
    return p;
}

bool aligned(const void* p, int bytes) { return (uintptr_t)p % bytes == 0; }

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
    const uint2* words = (const uint2*)(ws + p.words[from]);
    int *counts = (int*)(ws + p.counts), *total = (int*)(ws + p.total);
    int rc = launch_behind(k_digit_counts<FIRST>, dim3(p.tiles), kSortThreads, (size_t)bins * 4, st, !FIRST, ids, ids64, rows, padding, words, n, shift,
                    p.digit_bits, counts, (int2*)(ws + p.segment), (int*)(ws + p.popular));
    if (rc) return rc;
    rc = launch_behind(k_digit_prefix, dim3(ceil_div(bins, 8)), 256, 0, st, true, counts, p.tiles, bins, total);
    if (rc) return rc;
    auto smem = [](int bins) { return kTile * 8 + bins * (6 + 2 * kSortWarps); };
    rc = allow_smem(k_digit_scatter<FIRST>, smem(1 << kMaxDigit), false, g_scatter_done[FIRST]);
    if (rc) return rc;
    return launch_behind(k_digit_scatter<FIRST>, dim3(p.tiles), kSortThreads, (size_t)smem(bins), st, true, ids, ids64, rows, padding, words, n, shift, p.digit_bits,
                  (const int*)counts, (const int*)total, (uint2*)(ws + p.words[to]));
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
    if (table_stride > kMaxStride || out_stride > kMaxStride) return TRS_E_LIMIT;
    if (n == 0) return TRS_OK;
    if (!table || !ids || !out) return TRS_E_ARG;
    if (!aligned(table, type_bytes(table_type)) || !aligned(ids, ids64 ? 8 : 4) || !aligned(out, type_bytes(out_type))) return TRS_E_ARG;
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
                    return with_lookup(pieces, [&](auto gr, auto ro, auto pe) {
                        constexpr int G = decltype(gr)::value, ROWS = decltype(ro)::value, PER = decltype(pe)::value;
                        const dim3 grid((unsigned)ceil_div64(ceil_div64(n, ROWS) * G, kLookupThreads));
                        auto run = [&](auto copy) {
                            return launch(k_lookup<TI, TO, VEC, G, ROWS, PER, decltype(copy)::value>, grid, kLookupThreads, 0, (cudaStream_t)stream,
                                          (const TI*)table, (unsigned)rows, (unsigned)table_stride, ids, ids64, (unsigned)n, pieces, scale, padding_id,
                                          (TO*)out, (unsigned)out_stride);
                        };
                        if constexpr (std::is_same<TI, TO>::value)
                            if (scale == 1.f) return run(std::true_type());
                        return run(std::false_type());
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
    if ((n && (!aligned(grad, type_bytes(grad_type)) || !aligned(ids, ids64 ? 8 : 4))) || !aligned(out, type_bytes(out_type))) return TRS_E_ARG;
    if (n == 0 && accumulate) return TRS_OK;
    const cudaStream_t st = (cudaStream_t)stream;
    GradPlan p;
    unsigned char* ws = (unsigned char*)workspace;
    if (n) {
        p = grad_plan(n, rows, F);
        if (!ws || workspace_bytes < p.bytes || (uintptr_t)ws % 16) return TRS_E_WORKSPACE;
        if (n <= kFewIds) {
            p.digits = 1;   // (the result is where a first pass leaves it)
            const long long zero = ceil_div64(rows, 4 * kSortThreads);
            rc = launch(k_sort_few, dim3(1 + (unsigned)(zero < 2 * 148 ? zero : 2 * 148)), kSortThreads, 0, st, ids, ids64, rows, padding_id, (int)n,
                        p.bits, (uint2*)(ws + p.words[0]), (int2*)(ws + p.segment), (int*)(ws + p.popular));
            if (rc) return rc;
        } else for (int pass = 0; pass < p.digits; ++pass) {
            rc = pass == 0 ? sort_pass<true>(ids, ids64, rows, padding_id, ws, p, (int)n, pass, st)
                           : sort_pass<false>(ids, ids64, rows, padding_id, ws, p, (int)n, pass, st);
            if (rc) return rc;
        }
    }
    const int last = (p.digits + 1) & 1;
    const uint2* words = (const uint2*)(ws + p.words[last]);
    int2* segment = (int2*)(ws + p.segment);
    float *block_sum = (float*)(ws + p.block_sum), *span_sum = (float*)(ws + p.span_sum);
    int* popular = (int*)(ws + p.popular);
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
                        const int e = launch_behind(k_block_sums<TI, VEC, G>, dim3(p.spans), kThreads, 0, st, true, (const TI*)grad, grad_stride, words,
                                                    (int)n, (unsigned)rows, F, p.span, segment, block_sum, span_sum, popular);
                        if (e) return e;
                    }
                    return with_type(out_type, [&](auto to) {
                        using TO = decltype(to);
                        if constexpr (VEC * sizeof(TO) > 16) {
                            return (int)TRS_E_ARG;   // not reached: elements_per_piece
                        } else {
                            const int slabs = ceil_div(pieces, G);
                            const int popular_ctas = (int)(n / kPopular < 8 * 148 ? n / kPopular : 8 * 148);
                            const SumArgs<TI, TO> args{(const TI*)grad, grad_stride, words, (int)n, rows, F, slabs, p.span, segment, block_sum, span_sum,
                                                       popular, popular_ctas, scale, (TO*)out, out_stride, accumulate};
                            auto run = [&](auto rows_a_group) {
                                constexpr int ROWS = decltype(rows_a_group)::value;
                                const long long ctas = ceil_div64(ceil_div64(rows, ROWS) * slabs * G, kSumThreads);
                                if (ctas > 0x7fff0000ll) return (int)TRS_E_LIMIT;
                                return launch_behind(k_sums<TI, TO, VEC, G, ROWS>, dim3((unsigned)(popular_ctas + ctas)), kSumThreads, 0, st, n > 0, args);
                            };
                            // eight rows where most have no more than a position or two, otherwise their positions are a long chain
                            return n > 2 * rows ? run(std::integral_constant<int, 2>()) : run(std::integral_constant<int, 8>());
                        }
                    });
                });
            }
        });
    });
}
TRS_CATCH
