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
        const long long id = i0 + u < n ? load_id(ids, ids64, i0 + u) : 0;
        const bool pad = id == padding && padding != TRS_NO_PADDING, bad = id < 0 || id >= rows;
        // no row to read: the result is the constant
        from[u] = pad || bad || i0 + u >= n ? nullptr : table + id * stride;
        mul[u] = pad ? 0.f : bad ? __int_as_float(0x7fffffff) : scale;
    }
    for (int c = lane; c < pieces; c += G) {
        Piece<TI, VEC> p[kLookupRows];
#pragma unroll
        for (int u = 0; u < kLookupRows; ++u)
            if (from[u]) p[u] = *(const Piece<TI, VEC>*)(from[u] + (size_t)c * VEC);
#pragma unroll
        for (int u = 0; u < kLookupRows; ++u) {
            if (i0 + u >= n) break;
            Piece<TO, VEC> q;
#pragma unroll
            for (int k = 0; k < VEC; ++k) q.v[k] = from_float<TO>(from[u] ? as_float(p[u].v[k]) * mul[u] : mul[u]);
            *(Piece<TO, VEC>*)(out + (i0 + u) * out_stride + (size_t)c * VEC) = q;
        }
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
    const int bins = 1 << digit_bits, tiles = gridDim.x;
    for (int b = threadIdx.x; b < bins; b += kSortThreads) s_count[b] = 0;
    __syncthreads();
    const int base = blockIdx.x * kTile;
    for (int k = 0; k < kSortItems; ++k) {
        const int i = base + k * kSortThreads + threadIdx.x;
        if (i >= n || i < base) break;
        const unsigned key = FIRST ? key_of(load_id(ids, ids64, i), rows, padding) : keys[i];
        atomicAdd(&s_count[(key >> shift) & (bins - 1)], 1);
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

// ----------------------------------------------------------------------------------------------
// Sums of equal ids
// ----------------------------------------------------------------------------------------------
// The sorted positions are cut into blocks of 64 and spans of several blocks.  A block whose positions all name one row is summed
// ahead (a span of one row as a whole), all of them in parallel, so that a row with a hundred thousand positions is not one
// group's work; k_sums then walks a row's segment and takes a span's or a block's sum where the segment holds all of it.
constexpr int kBlock = 64, kSpanWarps = kThreads / 32;

template <class T, int VEC>
__device__ __forceinline__ void add_row(float (&acc)[VEC], const T* __restrict__ row, int c) {
    const Piece<T, VEC> p = *(const Piece<T, VEC>*)(row + (size_t)c * VEC);
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] += as_float(p.v[k]);
}

// One CTA a span: notes where segments begin and end, and sums its uniform blocks.
template <class T, int VEC>
__global__ void __launch_bounds__(kThreads) k_block_sums(const T* __restrict__ g, long long stride, const unsigned* __restrict__ keys,
                                                         const int* __restrict__ pos, int n, unsigned rows, int F, int span,
                                                         int2* __restrict__ segment, float* __restrict__ block_sum,
                                                         float* __restrict__ span_sum) {
    const int p0 = blockIdx.x * span, p1 = min(n - p0, span) + p0;
    for (int p = p0 + threadIdx.x; p < p1; p += kThreads) {
        const unsigned k = keys[p];
        if (k >= rows) continue;
        if (p == 0 || keys[p - 1] != k) segment[k].x = p;
        if (p == n - 1 || keys[p + 1] != k) segment[k].y = p + 1;
    }
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, pieces = F / VEC;
    const bool whole = p1 - p0 == span && keys[p0] == keys[p1 - 1] && keys[p0] < rows;
    __shared__ float s_part[kSpanWarps][32 * VEC];
    for (int c0 = 0; c0 < pieces; c0 += 32) {
        const int c = c0 + lane;
        float sum[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) sum[k] = 0.f;
        for (int b = p0 + warp * kBlock; b + kBlock <= p1; b += kSpanWarps * kBlock) {
            if (!whole && (keys[b] != keys[b + kBlock - 1] || keys[b] >= rows)) continue;
            float acc[VEC];
#pragma unroll
            for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
            if (c < pieces) {
#pragma unroll 8
                for (int p = b; p < b + kBlock; ++p) add_row<T, VEC>(acc, g + (size_t)pos[p] * stride, c);
                if (!whole)
#pragma unroll
                    for (int k = 0; k < VEC; ++k) block_sum[(size_t)(b / kBlock) * F + c * VEC + k] = acc[k];
            }
#pragma unroll
            for (int k = 0; k < VEC; ++k) sum[k] += acc[k];
        }
        if (whole) {   // the same for all threads of the CTA
            __syncthreads();
#pragma unroll
            for (int k = 0; k < VEC; ++k) s_part[warp][lane * VEC + k] = sum[k];
            __syncthreads();
            for (int f = threadIdx.x; f < 32 * VEC; f += kThreads) {
                float s = 0.f;
                for (int w = 0; w < kSpanWarps; ++w) s += s_part[w][f];
                if (c0 * VEC + f < F) span_sum[(size_t)blockIdx.x * F + c0 * VEC + f] = s;
            }
        }
    }
}

// A group of G lanes sums one row's segment for G pieces of the row.
template <class TI, class TO, int VEC, int G>
__global__ void __launch_bounds__(kThreads) k_sums(const TI* __restrict__ g, long long stride, const int* __restrict__ pos, int n,
                                                   long long rows, int F, int slabs, int span, const int2* __restrict__ segment,
                                                   const float* __restrict__ block_sum, const float* __restrict__ span_sum, float scale,
                                                   TO* __restrict__ out, long long out_stride, int accumulate) {
    const long long item = ((long long)blockIdx.x * kThreads + threadIdx.x) / G;
    const long long v = slabs == 1 ? item : item / slabs;
    const int c = (slabs == 1 ? 0 : (int)(item - v * slabs) * G) + threadIdx.x % G;
    if (v >= rows || c >= F / VEC) return;
    int p = 0, end = 0;
    if (n > 0) {
        const int2 s = segment[v];
        p = s.x;
        end = s.y;
    }
    if (accumulate && p == end) return;
    float acc[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
    while (p < end) {
        if ((p & (kBlock - 1)) == 0 && p + kBlock <= end) {
            const bool whole = p % span == 0 && p + span <= end;
            const float* from = whole ? span_sum + (size_t)(p / span) * F : block_sum + (size_t)(p / kBlock) * F;
#pragma unroll
            for (int k = 0; k < VEC; ++k) acc[k] += from[c * VEC + k];
            p += whole ? span : kBlock;
        } else {
            const int stop = min(end, (p & ~(kBlock - 1)) + kBlock);
#pragma unroll 4
            for (; p < stop; ++p) add_row<TI, VEC>(acc, g + (size_t)pos[p] * stride, c);
        }
    }
    TO* o = out + v * out_stride + (size_t)c * VEC;
    Piece<TO, VEC> q;
    if (accumulate) q = *(Piece<TO, VEC>*)o;
#pragma unroll
    for (int k = 0; k < VEC; ++k) q.v[k] = from_float<TO>(accumulate ? as_float(q.v[k]) + scale * acc[k] : scale * acc[k]);
    *(Piece<TO, VEC>*)o = q;
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
    // spans: some 600 of them, of 512 to 8192 positions
    p.span = kBlock * kSpanWarps;
    while (p.span < 8192 && (long long)p.span * 592 < n) p.span *= 2;
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
    int rc = launch(k_digit_counts<FIRST>, dim3(p.tiles), kSortThreads, (size_t)bins * 4, st, ids, ids64, rows, padding, keys, n, shift,
                    p.digit_bits, counts, (int2*)(ws + p.segment));
    if (rc) return rc;
    rc = launch(k_digit_prefix, dim3(ceil_div(bins, 8)), 256, 0, st, counts, p.tiles, bins, total);
    if (rc) return rc;
    const size_t smem = (size_t)bins * (4 + 2 * kSortWarps);
    rc = allow_smem(k_digit_scatter<FIRST>, (1 << kMaxDigit) * (4 + 2 * kSortWarps), false, g_scatter_done[FIRST]);
    if (rc) return rc;
    return launch(k_digit_scatter<FIRST>, dim3(p.tiles), kSortThreads, smem, st, ids, ids64, rows, padding, keys, pos, n, shift, p.digit_bits,
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
        for (int pass = 0; pass < p.digits; ++pass) {
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
                if (n) {
                    const int e = launch(k_block_sums<TI, VEC>, dim3(p.spans), kThreads, 0, st, (const TI*)grad, grad_stride, keys, pos, (int)n,
                                         (unsigned)rows, F, p.span, segment, block_sum, span_sum);
                    if (e) return e;
                }
                return with_type(out_type, [&](auto to) {
                    using TO = decltype(to);
                    if constexpr (VEC * sizeof(TO) > 16) {
                        return (int)TRS_E_ARG;   // not reached: elements_per_piece
                    } else {
                        return with_group(pieces, [&](auto gr) {
                            constexpr int G = decltype(gr)::value;
                            const int slabs = ceil_div(pieces, G);
                            const long long threads = rows * slabs * G;
                            if (ceil_div64(threads, kThreads) > 0x7fffffffll) return (int)TRS_E_LIMIT;
                            return launch(k_sums<TI, TO, VEC, G>, dim3((unsigned)ceil_div64(threads, kThreads)), kThreads, 0, st,
                                          (const TI*)grad, grad_stride, pos, (int)n, rows, F, slabs, p.span, (const int2*)segment,
                                          (const float*)block_sum, (const float*)span_sum, scale, (TO*)out, out_stride, accumulate);
                        });
                    }
                });
            }
        });
    });
}
TRS_CATCH
