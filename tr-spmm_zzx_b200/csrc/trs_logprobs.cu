// Log probabilities of given classes, entropy and the best alternatives of every row of scores, and their gradient.
//
// With the classes j that may be chosen (not masked, score above -inf), m = max x_j, d_j = scale (x_j - m), S = sum e^(d_j),
// T = sum e^(d_j) d_j:
//   log p_j = d_j - log S,   entropy = log S - T / S,   alternatives: the largest x_j, the lowest class first among equal ones.
// A row is read once; m, S and T are carried along it and rescaled when m grows.  Differences to m are taken before the scale, so
// rows of the type's lowest value stay exact.  Everything is held in fp32.
//   no class left:        log probability -inf, entropy 0, alternatives -1 with -inf, gradient 0
//   NaN or +inf left:     NaN (alternatives -1), gradient NaN
//   target = ignore id:   log probability 0, no gradient of it;   target outside [0, classes): NaN, no gradient of it
//
// Gradient with weights a (target), b (entropy), t_k (alternatives c_k), A = a + sum t_k:
//   dx_j = scale ( a [j = target] + sum t_k [j = c_k] - p_j (A + b (log p_j + entropy)) ),  0 where masked.
#include <cooperative_groups.h>

#include "trs_types.cuh"

namespace trs {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kFar = -200.f;   // 2^-200 is 0 in fp32: scores further below the maximum (-inf too) count as this far
constexpr int kMaxTop = 32;

typedef unsigned long long Key;   // (score, class): larger scores first, then lower classes; 0: none

__device__ __forceinline__ Key key_of(float x, int j) {
    const unsigned b = __float_as_uint(x + 0.f);   // -0 as 0
    const unsigned up = b & 0x80000000u ? ~b : b | 0x80000000u;
    return (Key)up << 32 | (unsigned)~j;
}
__device__ __forceinline__ float key_score(Key k) {
    const unsigned up = (unsigned)(k >> 32);
    return __uint_as_float(up & 0x80000000u ? up & 0x7fffffffu : ~up);
}
__device__ __forceinline__ int key_class(Key k) { return (int)~(unsigned)k; }

__device__ __forceinline__ float max_nan(float a, float b) {   // NaN where one is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float exp_2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ long long load_target(const void* __restrict__ t, int t64, long long i) {
    return t64 ? __ldg((const long long*)t + i) : (long long)__ldg((const int*)t + i);
}

// m, S, T of a part of a row, d in log2 units.  m = -inf: nothing yet; NaN stays.
struct Sums {
    float m, S, T;
};
__device__ __forceinline__ void rescale(Sums& s, float m, float c) {
    const float d = fmaxf((s.m - m) * c, kFar), f = exp_2(d);   // (-inf - -inf: kFar)
    s.T = f * fmaf(s.S, d, s.T);
    s.S *= f;
    s.m = m;
}
__device__ __forceinline__ Sums merge(Sums a, Sums b, float c) {
    const float m = max_nan(a.m, b.m);
    rescale(a, m, c);
    rescale(b, m, c);
    return {m, a.S + b.S, a.T + b.T};
}

// The memory that a matrix of scores or a mask takes: an aligned piece inside may be read whole, whatever row its ends belong to.
struct Extent {
    uintptr_t begin, end;
    __device__ __forceinline__ bool holds(const void* p, int bytes) const { return (uintptr_t)p >= begin && (uintptr_t)p + bytes <= end; }
};

// A row in pieces of 16 bytes on 16-byte boundaries; `head` elements of the first piece lie before the row.
template <class T>
struct Row {
    static constexpr int VEC = 16 / sizeof(T);
    const T* x;
    const unsigned char* mask;   // null: none
    int head, pieces, classes;
    Extent x_in, mask_in;
    template <class Args>
    __device__ __forceinline__ Row(const Args& a, long long r) : classes(a.classes), x_in(a.x_in), mask_in(a.mask_in) {
        x = (const T*)a.x + r * a.stride;
        mask = a.mask ? a.mask + r * a.mask_stride : nullptr;
        head = (int)((uintptr_t)x % 16 / sizeof(T));
        pieces = (head + classes + VEC - 1) / VEC;
    }
    __device__ __forceinline__ int first(int piece) const { return piece * VEC - head; }
    __device__ __forceinline__ bool inside(int j) const { return j >= 0 && j + VEC <= classes; }
    // scores as floats, -inf where there is none or it is masked
    __device__ __forceinline__ void load(int piece, float (&v)[VEC]) const {
        const int j = first(piece);
        if (x_in.holds(x + j, 16)) {
            const Piece<T, VEC> p = *(const Piece<T, VEC>*)(x + j);
#pragma unroll
            for (int k = 0; k < VEC; ++k) v[k] = as_float(p.v[k]);
        } else {   // the first piece of the matrix and its last
#pragma unroll
            for (int k = 0; k < VEC; ++k) v[k] = (unsigned)(j + k) < (unsigned)classes ? as_float(x[j + k]) : -INFINITY;
        }
        if (!inside(j)) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) v[k] = (unsigned)(j + k) < (unsigned)classes ? v[k] : -INFINITY;
        }
        if (mask) apply_mask(j, v);
    }
    __device__ __forceinline__ void apply_mask(int j, float (&v)[VEC]) const {
        const unsigned char* at = mask + j;
        const unsigned* word = (const unsigned*)((uintptr_t)at & ~(uintptr_t)3);
        const unsigned shift = ((uintptr_t)at & 3) * 8;
        constexpr int WORDS = VEC / 4 + 1;
        if (mask_in.holds(word, 4 * WORDS)) {   // the bytes out of the aligned words around them
            unsigned w[WORDS];
#pragma unroll
            for (int k = 0; k < WORDS; ++k) w[k] = __ldg(word + k);
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const unsigned four = __funnelshift_r(w[k / 4], w[k / 4 + 1], shift);
                if (!(four >> (k % 4 * 8) & 0xff)) v[k] = -INFINITY;
            }
        } else {
#pragma unroll
            for (int k = 0; k < VEC; ++k)
                if ((unsigned)(j + k) < (unsigned)classes && !at[k]) v[k] = -INFINITY;
        }
    }
};

struct Forward {
    const void* x;
    long long n, stride;
    int classes;
    const void* target;
    int target64;
    long long ignore;
    const unsigned char* mask;
    long long mask_stride;
    Extent x_in, mask_in;
    float scale, c;   // c = scale log2(e)
    int top;
    float *logprobs, *entropy, *top_logprobs;
    int* top_ids;
    float2* stats;
};

// What a row's sums say: thread 0 writes the log probability and the entropy.
template <class T>
__device__ __forceinline__ void write_row(const Forward& a, long long r, const T* x, const unsigned char* mask, Sums s) {
    const bool none = s.m == -INFINITY, broken = !(s.m < INFINITY);
    const float log_S = none || broken ? 0.f : logf(s.S);
    if (a.stats) a.stats[r] = make_float2(s.m, s.S);
    if (a.entropy) a.entropy[r] = broken ? NAN : none ? 0.f : fmaxf(log_S - s.T * kLn2 / s.S, 0.f);
    if (a.logprobs) {
        const long long t = load_target(a.target, a.target64, r);
        float lp;
        if (t == a.ignore && a.ignore != TRS_NO_IGNORE) lp = 0.f;
        else if (t < 0 || t >= a.classes || broken) lp = NAN;
        else if (none || (mask && !mask[t])) lp = -INFINITY;
        else lp = (as_float(x[t]) - s.m) * a.scale - log_S;
        a.logprobs[r] = lp;
    }
}
__device__ __forceinline__ void write_top(const Forward& a, long long r, int k, Key key, Sums s) {
    const bool broken = !(s.m < INFINITY), has = key != 0 && !broken;
    a.top_ids[r * a.top + k] = has ? key_class(key) : -1;
    a.top_logprobs[r * a.top + k] = broken ? NAN : has ? (key_score(key) - s.m) * a.scale - logf(s.S) : -INFINITY;
}

__device__ __forceinline__ Key warp_max(Key k) {
    const unsigned hi = (unsigned)(k >> 32), best = __reduce_max_sync(0xffffffffu, hi);
    const unsigned lo = __reduce_max_sync(0xffffffffu, hi == best ? (unsigned)k : 0u);
    return (Key)best << 32 | lo;
}

// The `top` largest of n different keys (0: none), in order, by one warp.
__device__ __forceinline__ void warp_top(const Key* keys, int n, int top, Key* out) {
    const int lane = threadIdx.x % 32;
    Key last = ~0ull;
    for (int k = 0; k < top; ++k) {
        Key best = 0;
        for (int i = lane; i < n; i += 32)
            if (keys[i] < last && keys[i] > best) best = keys[i];
        last = warp_max(best);
        if (lane == 0) out[k] = last;
        if (last == 0) {   // the same for the warp
            for (int q = k + 1 + lane; q < top; q += 32) out[q] = 0;
            break;
        }
    }
    __syncwarp();
}

// ----------------------------------------------------------------------------------------------
// One CTA a row
// ----------------------------------------------------------------------------------------------
// The maximum of each thread's part and where it is first come with the sums for nothing.  The top-th largest of those maxima, K, bounds the
// row's top-th score from below, and only the `top` threads with maxima from K on can hold scores from K on: their parts are
// read again (from L2), and the few scores that reach K are sorted out by one warp.
constexpr int kCandidates = 1024;

template <class T, int THREADS>
__global__ void __launch_bounds__(THREADS) k_row(const Forward a) {
    constexpr int WARPS = THREADS / 32, VEC = Row<T>::VEC;
    const long long r = blockIdx.x;
    const Row<T> row(a, r);
    Sums s{-INFINITY, 0.f, 0.f};
    int at = 0;   // where m is first
    for (int piece = threadIdx.x; piece < row.pieces; piece += THREADS) {
        float v[VEC];
        row.load(piece, v);
        float m = s.m;
#pragma unroll
        for (int k = 0; k < VEC; ++k) m = max_nan(m, v[k]);
        if (!(m <= s.m)) {
            rescale(s, m, a.c);
#pragma unroll
            for (int k = VEC; k-- > 0;)
                if (v[k] == m) at = row.first(piece) + k;
        }
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            const float d = fmaxf((v[k] - m) * a.c, kFar), e = exp_2(d);
            s.S += e;
            s.T = fmaf(e, d, s.T);
        }
    }
    __shared__ Sums s_part[WARPS];
    __shared__ Key s_key[THREADS], s_found[kCandidates], s_best[kMaxTop];
    __shared__ int s_sel[kMaxTop], s_count[2];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const Key mine = s.m > -INFINITY ? key_of(s.m, at) : 0;
    Sums w = s;
#pragma unroll
    for (int o = 16; o; o /= 2) {
        const Sums other{__shfl_xor_sync(0xffffffffu, w.m, o), __shfl_xor_sync(0xffffffffu, w.S, o), __shfl_xor_sync(0xffffffffu, w.T, o)};
        w = merge(w, other, a.c);
    }
    if (lane == 0) s_part[warp] = w;
    if (a.top) s_key[threadIdx.x] = mine;
    if (threadIdx.x < 2) s_count[threadIdx.x] = 0;
    __syncthreads();
    Sums all = s_part[0];
    for (int k = 1; k < WARPS; ++k) all = merge(all, s_part[k], a.c);
    if (threadIdx.x == 0) write_row<T>(a, r, row.x, row.mask, all);
    if (!a.top) return;

    if (warp == 0) warp_top(s_key, THREADS, a.top, s_best);
    __syncthreads();
    const Key bound = s_best[a.top - 1];
    if (mine != 0 && mine >= bound) s_sel[atomicAdd(&s_count[0], 1)] = threadIdx.x;   // at most `top`: keys differ
    __syncthreads();
    const int turns = (row.pieces + THREADS - 1) / THREADS, items = s_count[0] * turns;
    for (int i = threadIdx.x; i < items; i += THREADS) {
        const int piece = s_sel[i / turns] + i % turns * THREADS;
        if (piece >= row.pieces) continue;
        float v[VEC];
        row.load(piece, v);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            if (!(v[k] > -INFINITY)) continue;
            const Key key = key_of(v[k], row.first(piece) + k);
            if (key < bound) continue;
            const int to = atomicAdd(&s_count[1], 1);
            if (to < kCandidates) s_found[to] = key;
        }
    }
    __syncthreads();
    if (s_count[1] <= kCandidates) {
        if (warp == 0) warp_top(s_found, s_count[1], a.top, s_best);
    } else {
        // more scores than the list holds (rows in which a few threads' parts have nearly all of the largest ones): one round
        // over the row for each alternative
        Key last = ~0ull;
        for (int k = 0; k < a.top; ++k) {
            Key best = 0;
            for (int piece = threadIdx.x; piece < row.pieces; piece += THREADS) {
                float v[VEC];
                row.load(piece, v);
#pragma unroll
                for (int q = 0; q < VEC; ++q) {
                    const Key key = v[q] > -INFINITY ? key_of(v[q], row.first(piece) + q) : 0;
                    if (key < last && key > best) best = key;
                }
            }
            best = warp_max(best);
            __syncthreads();
            if (lane == 0) s_key[warp] = best;
            __syncthreads();
            last = 0;
            for (int q = 0; q < WARPS; ++q) last = s_key[q] > last ? s_key[q] : last;
            if (threadIdx.x == 0) s_best[k] = last;
        }
    }
    __syncthreads();
    for (int k = threadIdx.x; k < a.top; k += THREADS) write_top(a, r, k, s_best[k], all);
}

// ----------------------------------------------------------------------------------------------
// Short rows: a group of G lanes a row
// ----------------------------------------------------------------------------------------------
// The whole row is held in registers, PER pieces a lane (16 scores, or 32 for the longest), so the maximum comes first and the sums
// after it.  An alternative is the group's maximum, then the lowest class that has it, taken out for the next one.
constexpr int kShortThreads = 256;

template <int G>
__device__ __forceinline__ Sums group_sum(Sums s) {   // m is common
#pragma unroll
    for (int o = G / 2; o; o /= 2) {
        s.S += __shfl_xor_sync(0xffffffffu, s.S, o);
        s.T += __shfl_xor_sync(0xffffffffu, s.T, o);
    }
    return s;
}

template <class T, int G, int PER>
__global__ void __launch_bounds__(kShortThreads) k_short_rows(const Forward a) {
    constexpr int VEC = Row<T>::VEC;
    const int g = threadIdx.x % G;
    const long long r0 = ((long long)blockIdx.x * kShortThreads + threadIdx.x) / G, r = r0 < a.n ? r0 : a.n - 1;   // lanes stay together
    const Row<T> row(a, r);
    float v[PER][VEC];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if (g + i * G < row.pieces) {
            row.load(g + i * G, v[i]);
        } else {
#pragma unroll
            for (int k = 0; k < VEC; ++k) v[i][k] = -INFINITY;
        }
    }
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < PER; ++i)
#pragma unroll
        for (int k = 0; k < VEC; ++k) m = max_nan(m, v[i][k]);
#pragma unroll
    for (int o = G / 2; o; o /= 2) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    Sums s{m, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < PER; ++i)
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            const float d = fmaxf((v[i][k] - m) * a.c, kFar), e = exp_2(d);
            s.S += e;
            s.T = fmaf(e, d, s.T);
        }
    s = group_sum<G>(s);
    if (g == 0 && r == r0) write_row<T>(a, r, row.x, row.mask, s);
    const bool broken = !(m < INFINITY);
    for (int k = 0; k < a.top; ++k) {
        if (k) {
            m = -INFINITY;
#pragma unroll
            for (int i = 0; i < PER; ++i)
#pragma unroll
                for (int q = 0; q < VEC; ++q) m = fmaxf(m, v[i][q]);
#pragma unroll
            for (int o = G / 2; o; o /= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        }
        int at = 0x7fffffff;
#pragma unroll
        for (int i = PER; i-- > 0;)
#pragma unroll
            for (int q = VEC; q-- > 0;)
                if (v[i][q] == m) at = row.first(g + i * G) + q;
#pragma unroll
        for (int o = G / 2; o; o /= 2) at = min(at, __shfl_xor_sync(0xffffffffu, at, o));
#pragma unroll
        for (int i = 0; i < PER; ++i)
#pragma unroll
            for (int q = 0; q < VEC; ++q)
                if (row.first(g + i * G) + q == at) v[i][q] = -INFINITY;
        if (k % G == g && r == r0) write_top(a, r, k, broken || m == -INFINITY ? 0 : key_of(m, at), s);
    }
}

// ----------------------------------------------------------------------------------------------
// Gradient
// ----------------------------------------------------------------------------------------------
struct Backward {
    const void* x;
    long long n, stride;
    int classes;
    const void* target;
    int target64;
    long long ignore;
    const unsigned char* mask;
    long long mask_stride;
    Extent x_in, mask_in;
    float scale, c;
    int top;
    const int* top_ids;
    const float2* stats;
    const float *entropy, *g_logprobs, *g_entropy, *g_top;
    void* dx;
    long long dx_stride;
};

// What the gradient of a row needs beside its scores.
struct RowGrad {
    float m, inv_S, A, B, c;   // -p (A + B d) scale is what a class without a weight of its own gets, d in log2 units
    bool zero;
};

__device__ __forceinline__ bool target_counts(const Backward& a, long long t) {
    return t >= 0 && t < a.classes && !(t == a.ignore && a.ignore != TRS_NO_IGNORE);
}

__device__ __forceinline__ RowGrad row_grad(const Backward& a, long long r) {
    const float2 st = a.stats[r];
    float A = 0.f;
    if (a.g_logprobs && target_counts(a, load_target(a.target, a.target64, r))) A = a.g_logprobs[r];
    if (a.g_top)
        for (int k = 0; k < a.top; ++k)
            if (a.top_ids[r * a.top + k] >= 0) A += a.g_top[r * a.top + k];
    const float b = a.g_entropy ? a.g_entropy[r] : 0.f;
    RowGrad g;
    g.m = st.x;
    g.c = a.c;
    g.zero = st.x == -INFINITY || (A == 0.f && b == 0.f);
    // log p + entropy = d ln 2 - log S + entropy
    g.inv_S = st.x < INFINITY ? 1.f / st.y : NAN;
    g.A = b == 0.f ? A : A + b * (a.entropy[r] - logf(st.y));
    g.B = b * kLn2;
    return g;
}
__device__ __forceinline__ float without_own(const RowGrad& g, float x) {
    const float d = fmaxf((x - g.m) * g.c, kFar);
    return -exp_2(d) * g.inv_S * fmaf(g.B, d, g.A);
}

// Class j with weights of its own (the target, an alternative): all of them, and the rest as any class.
template <class T>
__device__ __forceinline__ void write_own(const Backward& a, long long r, const RowGrad& g, const Row<T>& row, T* dx, long long j) {
    float own = 0.f;
    if (a.g_logprobs && load_target(a.target, a.target64, r) == j && target_counts(a, j)) own += a.g_logprobs[r];
    if (a.g_top)
        for (int k = 0; k < a.top; ++k)
            if (a.top_ids[r * a.top + k] == j) own += a.g_top[r * a.top + k];
    const float x = as_float(row.x[j]);
    if ((row.mask && !row.mask[j]) || x == -INFINITY) return;   // stays 0
    dx[j] = from_float<T>(a.scale * (own + without_own(g, x)));
}
template <class T>
__device__ __forceinline__ void write_piece(const Backward& a, const RowGrad& g, const Row<T>& row, T* dx, int piece) {
    constexpr int VEC = Row<T>::VEC;
    const int j = row.first(piece);
    Piece<T, VEC> q;
    if (g.zero) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) q.v[k] = from_float<T>(0.f);
    } else {
        float v[VEC];
        row.load(piece, v);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            const bool out = v[k] == -INFINITY;   // masked, or as good as
            q.v[k] = from_float<T>(out ? 0.f : a.scale * without_own(g, v[k]));
        }
    }
    if (row.inside(j) && (uintptr_t)(dx + j) % 16 == 0) {
        *(Piece<T, VEC>*)(dx + j) = q;
    } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k)
            if (j + k >= 0 && j + k < row.classes) dx[j + k] = q.v[k];
    }
}

constexpr int kGradThreads = 256, kGradPieces = 8;   // pieces per thread

template <class T>
__global__ void __launch_bounds__(kGradThreads) k_row_grad(const Backward a, int parts) {
    const long long r = blockIdx.x / parts;
    const int part = (int)(blockIdx.x - r * parts);
    const Row<T> row(a, r);
    T* dx = (T*)a.dx + r * a.dx_stride;
    const RowGrad g = row_grad(a, r);
    const int p0 = part * kGradThreads * kGradPieces, p1 = min(row.pieces, p0 + kGradThreads * kGradPieces);
    for (int piece = p0 + threadIdx.x; piece < p1; piece += kGradThreads) write_piece<T>(a, g, row, dx, piece);
    if (g.zero) return;
    __syncthreads();   // classes with weights of their own are written once more, by one thread each (equal values where they coincide)
    for (int k = threadIdx.x; k < 1 + (a.g_top ? a.top : 0); k += kGradThreads) {
        const long long j = k ? a.top_ids[r * a.top + k - 1] : a.g_logprobs ? load_target(a.target, a.target64, r) : -1;
        if (j < 0 || j >= a.classes || (k == 0 && !target_counts(a, j))) continue;
        const int piece = (int)((j + row.head) / Row<T>::VEC);
        if (piece >= p0 && piece < p1) write_own<T>(a, r, g, row, dx, j);
    }
}

template <class T, int G, int PER>
__global__ void __launch_bounds__(kShortThreads) k_short_rows_grad(const Backward a) {
    const int g = threadIdx.x % G;
    const long long r = ((long long)blockIdx.x * kShortThreads + threadIdx.x) / G;
    const bool in = r < a.n;
    const Row<T> row(a, in ? r : 0);
    T* dx = (T*)a.dx + (in ? r : 0) * a.dx_stride;
    const RowGrad w = row_grad(a, in ? r : 0);
#pragma unroll
    for (int i = 0; i < PER; ++i)
        if (in && g + i * G < row.pieces) write_piece<T>(a, w, row, dx, g + i * G);
    __syncwarp();   // behind the lanes of the row, as in k_row_grad
    if (!in || w.zero) return;
    for (int k = g; k < 1 + (a.g_top ? a.top : 0); k += G) {
        const long long j = k ? a.top_ids[r * a.top + k - 1] : a.g_logprobs ? load_target(a.target, a.target64, r) : -1;
        if (j < 0 || j >= a.classes || (k == 0 && !target_counts(a, j))) continue;
        write_own<T>(a, r, w, row, dx, j);
    }
}

// Lanes and pieces per lane that hold a row of so many pieces; beyond 32 x 2 x (16 scores) a row is a CTA's.
constexpr int kShortScores = 16;
template <class T, class Fn>
int with_short(int pieces, Fn fn) {
    constexpr int PER = kShortScores / Row<T>::VEC;
    if (pieces <= PER) return fn(std::integral_constant<int, 1>(), std::integral_constant<int, PER>());
    if (pieces <= 2 * PER) return fn(std::integral_constant<int, 2>(), std::integral_constant<int, PER>());
    if (pieces <= 4 * PER) return fn(std::integral_constant<int, 4>(), std::integral_constant<int, PER>());
    if (pieces <= 8 * PER) return fn(std::integral_constant<int, 8>(), std::integral_constant<int, PER>());
    if (pieces <= 16 * PER) return fn(std::integral_constant<int, 16>(), std::integral_constant<int, PER>());
    if (pieces <= 32 * PER) return fn(std::integral_constant<int, 32>(), std::integral_constant<int, PER>());
    return fn(std::integral_constant<int, 32>(), std::integral_constant<int, 2 * PER>());
}
template <class T>
constexpr int kShortPieces = 64 * kShortScores / Row<T>::VEC;
// Pieces of a row, wherever it begins.
template <class T>
int most_pieces(int classes) { return (int)ceil_div64((long long)classes + Row<T>::VEC - 1, Row<T>::VEC); }

Extent extent(const void* p, long long rows, long long stride, long long width, int size) {
    return {(uintptr_t)p, (uintptr_t)p + (size_t)((rows - 1) * stride + width) * size};
}

int check(const void* x, int type, long long n, int classes, long long stride, const void* mask, long long mask_stride, float scale,
          int top) {
    if (!type_known(type) || n < 0 || classes < 1 || stride < classes || top < 0 || !(scale > 0.f) || !(scale < INFINITY)) return TRS_E_ARG;
    if (mask && mask_stride != 0 && mask_stride < classes) return TRS_E_ARG;
    if (n > 0x7fffffffll || classes > (1 << 30) || top > kMaxTop) return TRS_E_LIMIT;
    if (n && (!x || (uintptr_t)x % type_bytes(type))) return TRS_E_ARG;
    return TRS_OK;
}

}  // namespace
}  // namespace trs

using namespace trs;

extern "C" int trs_logprobs(const void* x, int type, long long n, int classes, long long stride, const void* targets, int targets64,
                            long long ignore_id, const unsigned char* mask, long long mask_stride, float scale, int top, float* logprobs,
                            float* entropy, float* top_logprobs, int32_t* top_ids, float* stats, void* stream) try {
    const int rc = check(x, type, n, classes, stride, mask, mask_stride, scale, top);
    if (rc) return rc;
    if (n == 0) return TRS_OK;
    if ((logprobs && !targets) || (top && (!top_logprobs || !top_ids)) || (uintptr_t)stats % 8) return TRS_E_ARG;
    const Forward a{x, n, stride, classes, targets, targets64, ignore_id, mask, mask_stride, extent(x, n, stride, classes, type_bytes(type)), extent(mask, n, mask_stride, classes, 1), scale, scale * kLog2e, top, logprobs, entropy,
                    top_logprobs, top_ids, (float2*)stats};
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        const int pieces = most_pieces<T>(classes);
        if (pieces <= kShortPieces<T>)
            return with_short<T>(pieces, [&](auto g, auto per) {
                constexpr int G = decltype(g)::value;
                return launch(k_short_rows<T, G, decltype(per)::value>, dim3((unsigned)ceil_div64(n * G, kShortThreads)), kShortThreads, 0,
                              (cudaStream_t)stream, a);
            });
        if (pieces <= 256) return launch(k_row<T, 128>, dim3((unsigned)n), 128, 0, (cudaStream_t)stream, a);
        return launch(k_row<T, 512>, dim3((unsigned)n), 512, 0, (cudaStream_t)stream, a);
    });
}
TRS_CATCH

extern "C" int trs_logprobs_grad(const void* x, int type, long long n, int classes, long long stride, const void* targets, int targets64,
                                 long long ignore_id, const unsigned char* mask, long long mask_stride, float scale, int top,
                                 const int32_t* top_ids, const float* stats, const float* entropy, const float* g_logprobs,
                                 const float* g_entropy, const float* g_top_logprobs, void* dx, long long dx_stride, void* stream) try {
    const int rc = check(x, type, n, classes, stride, mask, mask_stride, scale, top);
    if (rc) return rc;
    if (dx_stride < classes) return TRS_E_ARG;
    if (n == 0) return TRS_OK;
    if (!dx || (uintptr_t)dx % type_bytes(type) || !stats || (uintptr_t)stats % 8) return TRS_E_ARG;
    if ((g_logprobs && !targets) || (g_entropy && !entropy) || (g_top_logprobs && (!top_ids || !top))) return TRS_E_ARG;
    const Backward a{x, n, stride, classes, targets, targets64, ignore_id, mask, mask_stride, extent(x, n, stride, classes, type_bytes(type)), extent(mask, n, mask_stride, classes, 1), scale, scale * kLog2e, top, top_ids,
                     (const float2*)stats, entropy, g_logprobs, g_entropy, g_top_logprobs, dx, dx_stride};
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        const int pieces = most_pieces<T>(classes);
        if (pieces <= kShortPieces<T>)
            return with_short<T>(pieces, [&](auto g, auto per) {
                constexpr int G = decltype(g)::value;
                return launch(k_short_rows_grad<T, G, decltype(per)::value>, dim3((unsigned)ceil_div64(n * G, kShortThreads)), kShortThreads,
                              0, (cudaStream_t)stream, a);
            });
        const long long parts = ceil_div64((long long)classes + Row<T>::VEC - 1, (long long)Row<T>::VEC * kGradThreads * kGradPieces);
        if (n * parts > 0x7fffffffll) return (int)TRS_E_LIMIT;
        return launch(k_row_grad<T>, dim3((unsigned)(n * parts)), kGradThreads, 0, (cudaStream_t)stream, a, (int)parts);
    });
}
TRS_CATCH
