// Log probabilities of given classes, entropy and the best alternatives of every row of scores, and their gradient.
//
// With the classes j that may be chosen (not masked, score above -inf), m = max x_j, d_j = scale (x_j - m), S = sum e^(d_j),
// T = sum e^(d_j) d_j:
//   log p_j = d_j - log S,   entropy = log S - T / S,   alternatives: the largest x_j, the lowest class first among equal ones.
// A row is read once; m, S and T are carried along it and rescaled when m grows.  Differences to m are taken before the scale, so
// rows of the type's lowest value stay exact; a score whose distance to m leaves fp32's range (3.4e38) counts as infinitely far.  Everything is
// held in fp32.
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

// Unsigned numbers in the order of the scores; -0 as 0.
__device__ __forceinline__ unsigned order_of(float x) {
    const unsigned b = __float_as_uint(x + 0.f);
    return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}
template <class T>
__device__ __forceinline__ unsigned order_of_16(T x) {
    unsigned b = *(const unsigned short*)&x;
    if (b == 0x8000u) b = 0;
    return b & 0x8000u ? b ^ 0xffffu : b | 0x8000u;
}
__device__ __forceinline__ Key key_of(float x, int j) { return (Key)order_of(x) << 32 | (unsigned)~j; }
__device__ __forceinline__ float key_score(Key k) {
    const unsigned up = (unsigned)(k >> 32);
    return __uint_as_float(up & 0x80000000u ? up & 0x7fffffffu : ~up);
}
__device__ __forceinline__ int key_class(Key k) { return (int)~(unsigned)k; }

// e^(d) as 2^(d log2 e) by the special-function unit: two instructions a score, where the library's function takes several and the
// forward pass is bound by them.  The argument is rounded once after its factor, so a class |z| below the best has a probability off by up to
// |z| 2^-24 of itself beside the unit's 2^-22; what is that far down hardly counts in the sums.
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
        at((const T*)a.x + r * a.stride, a.mask ? a.mask + r * a.mask_stride : nullptr);
    }
    __device__ __forceinline__ void at(const T* x_, const unsigned char* mask_) {
        x = x_;
        mask = mask_;
        head = (int)((unsigned)(uintptr_t)x % 16 / sizeof(T));
        pieces = (head + classes + VEC - 1) / VEC;
    }
    __device__ __forceinline__ int first(int piece) const { return piece * VEC - head; }
    __device__ __forceinline__ bool inside(int j) const { return j >= 0 && j + VEC <= classes; }
    // scores as floats, -inf where there is none or it is masked
    __device__ __forceinline__ void load(int piece, float (&v)[VEC]) const {
        const int j = first(piece);
        if (x_in.holds(x + j, 16)) {
            as_floats(*(const Piece<T, VEC>*)(x + j), v);
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

// The mask's bytes of whole pieces, out of the aligned words that hold them.
template <int VEC>
struct MaskWords {
    static constexpr int WORDS = VEC / 4 + 1;
    const unsigned char* word;   // of piece 0
    unsigned shift;
    int last;                    // the last word with a byte of the piece
    bool even;                   // a piece's bytes in one load
    __device__ __forceinline__ MaskWords(const unsigned char* mask, int head) {
        const uintptr_t at = (uintptr_t)(mask - head);
        word = (const unsigned char*)(at & ~(uintptr_t)3);
        shift = ((unsigned)at & 3) * 8;
        last = shift ? VEC : VEC - 4;
        even = at % VEC == 0;
    }
    __device__ __forceinline__ void fetch(unsigned (&bits)[WORDS], int piece) const {
        const unsigned char* w = word + (size_t)piece * VEC;
        if (even) {
            const Piece<unsigned, VEC / 4> b = *(const Piece<unsigned, VEC / 4>*)w;
#pragma unroll
            for (int k = 0; k < VEC / 4; ++k) bits[k] = b.v[k];
            bits[VEC / 4] = 0;
        } else {
#pragma unroll
            for (int k = 0; k < WORDS; ++k) bits[k] = __ldg((const unsigned*)(w + (k < WORDS - 1 ? 4 * k : last)));
        }
    }
    template <class T>
    __device__ __forceinline__ void apply(Piece<T, VEC>& x, const unsigned (&bits)[WORDS]) const {   // -inf where masked
#pragma unroll
        for (int k = 0; k < VEC / 4; ++k) mask_four(x, 4 * k, __funnelshift_r(bits[k], bits[k + 1], shift));
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
__device__ __forceinline__ void write_top(const Forward& a, long long r, int k, bool has, int id, float score, float m, float log_S) {
    const bool broken = !(m < INFINITY);
    has = has && !broken;
    a.top_ids[r * a.top + k] = has ? id : -1;
    a.top_logprobs[r * a.top + k] = broken ? NAN : has ? (score - m) * a.scale - log_S : -INFINITY;
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

// The same by all threads of a CTA or a warp (`me` of `threads`), each key to the place that its rank gives it; out is 0 before.  For short lists.
__device__ __forceinline__ void rank_top(const Key* keys, int n, int top, Key* out, int me, int threads) {
    for (int i = me; i < n; i += threads) {
        const Key k = keys[i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) rank += keys[j] > k;
        if (k != 0 && rank < top) out[rank] = k;
    }
}

// The warp's keys in descending order over the lanes.
__device__ __forceinline__ Key warp_sort(Key k) {
    const int lane = threadIdx.x % 32;
#pragma unroll
    for (int size = 2; size <= 32; size *= 2)
#pragma unroll
        for (int o = size / 2; o; o /= 2) {
            const Key other = __shfl_xor_sync(0xffffffffu, k, o);
            const bool larger = ((lane & o) == 0) == ((lane & size) == 0);   // (lane & 32 is 0: the last merge descends)
            if ((other > k) == larger) k = other;
        }
    return k;
}

// ----------------------------------------------------------------------------------------------
// One CTA a row
// ----------------------------------------------------------------------------------------------
// A thread takes TURN pieces, THREADS apart, at a time: their loads are under way together, their maximum is compared once with the
// part's, and the sums go two scores an instruction.  The pieces that the row's ends cut come last.
//
// Alternatives: each thread's largest score and the piece it is first in come with the sums for nothing.  The key (score, last class of that
// piece) is at most the key of a score of the row, so the top-th largest of the threads' keys - of 32 groups of threads, which
// one sort of a warp gives - is at most the row's top-th largest: K.  Only threads whose key (score, first class of the piece)
// reaches K can hold scores from K on, little more than `top` of them.  That piece is read again - all pieces of the thread where the
// second largest of its pieces' maxima reaches K too - and the few scores that reach K are put in order by their ranks.
//
// Few rows are split over the CTAs of a cluster (`parts`), which hand their sums and alternatives to the first one.
constexpr int kTurn = 4, kMaxParts = 8;
constexpr int candidates(int threads) { return threads >= 128 ? 1024 : 256; }   // (the alternatives of 8 parts fit)

// A thread's sums with two accumulators, relative to `ref`: a maximum up to 2^kSlack below the present one (e^(d) stays far from
// overflow, and sums are rescaled once or twice in a row instead of at every new maximum); and where the maximum is first.
constexpr float kSlack = 16.f;
struct Running {
    float m = -INFINITY, ref = -INFINITY;
    float second = -INFINITY;   // largest of the other pieces' maxima
    float2 S = {0.f, 0.f}, T = {0.f, 0.f};
    int at = 0x7fffffff;   // a piece
    __device__ __forceinline__ Sums sums(float c) const {
        Sums s{ref, S.x + S.y, T.x + T.y};
        rescale(s, m, c);
        return s;
    }
    // before scores up to `top` are added
    __device__ __forceinline__ void make_room(float top, float c) {
        if ((top - ref) * c <= kSlack) return;
        Sums s{ref, S.x + S.y, T.x + T.y};
        rescale(s, top, c);
        ref = top;
        S = make_float2(s.S, 0.f);
        T = make_float2(s.T, 0.f);
    }
    // NEAR: no score is -inf, or so far below m that d is; otherwise T is NaN afterwards
    template <bool NEAR, class E, int N>
    __device__ __forceinline__ void add(const Piece<E, N>& x, float2 minus, float2 c2) {
        float v[N];
        as_floats(x, v);
#pragma unroll
        for (int k = 0; k < N; k += 2) {
            float2 d = __fmul2_rn(__fadd2_rn(make_float2(v[k], v[k + 1]), minus), c2);
            if (!NEAR) {
                d.x = fmaxf(d.x, kFar);
                d.y = fmaxf(d.y, kFar);
            }
            const float2 e = make_float2(exp_2(d.x), exp_2(d.y));
            S = __fadd2_rn(S, e);
            T = __ffma2_rn(e, d, T);
        }
    }
};
template <class T, int THREADS, bool MASKED>
__global__ void __launch_bounds__(THREADS, THREADS == 32 ? 24 : (MASKED ? 1024 : 1280) / THREADS) k_row(const Forward a, int parts) {
    constexpr int WARPS = THREADS / 32, VEC = Row<T>::VEC, TURN = kTurn, WORDS = VEC / 4 + 1;
    const long long r = blockIdx.x / parts;
    const int part = (int)(blockIdx.x - r * parts);
    const Row<T> row(a, r);
    const int per = (row.pieces + parts - 1) / parts, p0 = min(row.pieces, part * per), p1 = min(row.pieces, p0 + per);
    // pieces [q0, q1) lie inside the row
    int q0 = max(p0, row.head ? 1 : 0);
    int q1 = min(p1, (row.head + row.classes) / VEC);
    q0 = min(q0, p1);
    q1 = max(q1, q0);
    const MaskWords<VEC> mask(row.mask, row.head);
    const float2 c2 = make_float2(a.c, a.c);
    Running s;
    struct Raw {
        Piece<T, VEC> x;
        unsigned bits[WORDS];
    };
    auto fetch = [&](int piece) {
        Raw w;
        w.x = *(const Piece<T, VEC>*)(row.x + row.first(piece));
        if (MASKED) mask.fetch(w.bits, piece);
        return w;
    };
    auto masked = [&](Raw& w) {
        if (MASKED) mask.apply(w.x, w.bits);
    };
    // one turn; `near`: no difference is bounded, and the answer is whether none needed to be (otherwise nothing is added)
    auto take = [&](auto near, int base) {
        constexpr bool NEAR = decltype(near)::value;
        Raw w[TURN];
#pragma unroll
        for (int u = 0; u < TURN; ++u) w[u] = fetch(base + u * THREADS);
        float pm[TURN], m = s.m;
#pragma unroll
        for (int u = 0; u < TURN; ++u) {
            masked(w[u]);
            pm[u] = max_of(w[u].x);
            m = max_nan(m, pm[u]);
        }
        if (a.top) {
            float first = s.m;
#pragma unroll
            for (int u = 0; u < TURN; ++u) {
                s.second = fmaxf(s.second, fminf(first, pm[u]));
                first = fmaxf(first, pm[u]);
            }
            if (m > s.m) {
#pragma unroll
                for (int u = TURN; u-- > 0;)
                    if (pm[u] == m) s.at = base + u * THREADS;
            }
        }
        s.m = m;
        s.make_room(m, a.c);
        const float2 minus = make_float2(-s.ref, -s.ref), S0 = s.S, T0 = s.T;
#pragma unroll
        for (int u = 0; u < TURN; ++u) s.template add<NEAR>(w[u].x, minus, c2);
        const float sum = s.T.x + s.T.y;
        if (NEAR && !(sum == sum)) {
            s.S = S0;
            s.T = T0;
            return false;
        }
        return true;
    };
    auto take_one = [&](int piece) {
        Raw w = fetch(piece);
        masked(w);
        const float pm = max_of(w.x);
        s.second = fmaxf(s.second, fminf(s.m, pm));
        if (pm > s.m) s.at = piece;
        s.m = max_nan(s.m, pm);
        s.make_room(s.m, a.c);
        s.template add<false>(w.x, make_float2(-s.ref, -s.ref), c2);
    };
    int base = q0 + threadIdx.x;
    const int last = q1 - (TURN - 1) * THREADS;
    bool near = !MASKED;
    while (near && base < last) {
        near = take(std::true_type(), base);
        if (near) base += TURN * THREADS;
    }
    for (; base < last; base += TURN * THREADS) take(std::false_type(), base);
    for (; base < q1; base += THREADS) take_one(base);
    const int cut = q0 - p0 + p1 - q1;   // pieces that are not whole
    auto cut_piece = [&](int i) { return i < q0 - p0 ? p0 + i : q1 + i - (q0 - p0); };
    if (THREADS - 1 - (int)threadIdx.x < cut) {
        float v[VEC];
        const int piece = cut_piece(THREADS - 1 - threadIdx.x);
        row.load(piece, v);
        Piece<T, VEC> x;
#pragma unroll
        for (int k = 0; k < VEC; ++k) x.v[k] = from_float<T>(v[k]);   // what it was
        const float pm = max_of(x);
        s.second = fmaxf(s.second, fminf(s.m, pm));
        if (pm > s.m || (pm == s.m && piece < s.at)) s.at = piece;
        s.m = max_nan(s.m, pm);
        s.make_room(s.m, a.c);
        s.template add<false>(x, make_float2(-s.ref, -s.ref), c2);
    }
    __shared__ Sums s_part[WARPS], s_all;
    __shared__ Key s_key[THREADS], s_found[candidates(THREADS)], s_best[kMaxTop];
    __shared__ Key s_bound;
    __shared__ int s_sel[THREADS], s_count[2];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    auto warp_sum = [&](Sums w, int lanes) {
        for (int o = lanes / 2; o; o /= 2) {
            const Sums other{__shfl_xor_sync(0xffffffffu, w.m, o), __shfl_xor_sync(0xffffffffu, w.S, o), __shfl_xor_sync(0xffffffffu, w.T, o)};
            w = merge(w, other, a.c);
        }
        return w;
    };
    const Sums w = warp_sum(s.sums(a.c), 32);
    if (lane == 0) s_part[warp] = w;
    const bool some = s.m > -INFINITY;
    if (a.top) s_key[threadIdx.x] = some ? key_of(s.m, row.first(s.at) + VEC - 1) : 0;
    if (threadIdx.x < 2) s_count[threadIdx.x] = 0;
    if (threadIdx.x < a.top) s_best[threadIdx.x] = 0;
    __syncthreads();
    if (warp == WARPS - 1) {
        const Sums all = warp_sum(s_part[lane % WARPS], WARPS);
        if (lane == 0) {
            s_all = all;
            if (parts == 1) write_row<T>(a, r, row.x, row.mask, all);
        }
    }
    if (a.top) {
        if (warp == 0) {
            Key best = 0;
#pragma unroll
            for (int i = 0; i < WARPS; ++i) best = s_key[i * 32 + lane] > best ? s_key[i * 32 + lane] : best;
            best = __shfl_sync(0xffffffffu, warp_sort(best), a.top - 1);
            if (best == 0) {   // fewer groups have a score: the threads' own keys
                warp_top(s_key, THREADS, a.top, s_found);
                best = s_found[a.top - 1];
            }
            if (lane == 0) s_bound = best;
        }
        __syncthreads();
        const Key bound = s_bound;
        const float least = bound ? key_score(bound) : -INFINITY;
        auto keep = [&](const float (&v)[VEC], int piece) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                if (!(v[k] > -INFINITY)) continue;
                const Key key = key_of(v[k], row.first(piece) + k);
                if (key < bound) continue;
                const int to = atomicAdd(&s_count[1], 1);
                if (to < candidates(THREADS)) s_found[to] = key;
            }
        };
        if (some && key_of(s.m, max(row.first(s.at), 0)) >= bound) {
            if (s.second >= least) {
                s_sel[atomicAdd(&s_count[0], 1)] = threadIdx.x;
            } else if (s.at >= q0 && s.at < q1) {   // no other piece of the thread's reaches K
                Raw w = fetch(s.at);
                masked(w);
                float v[VEC];
                as_floats(w.x, v);
                keep(v, s.at);
            }
        }
        __syncthreads();
        const int turns = (q1 - q0 + THREADS - 1) / THREADS, items = s_count[0] * turns;
        for (int i0 = threadIdx.x; i0 < items; i0 += kTurn * THREADS) {
            Raw w[kTurn];
            int at[kTurn];
#pragma unroll
            for (int u = 0; u < kTurn; ++u) {
                const int i = i0 + u * THREADS, sel = i / turns;
                at[u] = i < items ? q0 + s_sel[sel] + (i - sel * turns) * THREADS : q1;
                if (at[u] < q1) w[u] = fetch(at[u]);
            }
#pragma unroll
            for (int u = 0; u < kTurn; ++u) {
                if (at[u] >= q1) continue;
                masked(w[u]);
                if (max_of(w[u].x) < least) continue;
                float v[VEC];
                as_floats(w[u].x, v);
                keep(v, at[u]);
            }
        }
        if (THREADS - 1 - (int)threadIdx.x < cut) {   // the cut pieces too, whoever had them
            float v[VEC];
            const int piece = cut_piece(THREADS - 1 - threadIdx.x);
            row.load(piece, v);
            keep(v, piece);
        }
        __syncthreads();
        if (s_count[1] <= 256) {
            rank_top(s_found, s_count[1], a.top, s_best, threadIdx.x, THREADS);
        } else if (s_count[1] <= candidates(THREADS)) {
            if (warp == 0) warp_top(s_found, s_count[1], a.top, s_best);
        } else {
            // more scores than the list holds (rows in which a few threads' parts have nearly all of the largest ones): one round
            // over the row for each alternative
            Key last = ~0ull;
            for (int k = 0; k < a.top; ++k) {
                Key best = 0;
                for (int piece = p0 + threadIdx.x; piece < p1; piece += THREADS) {
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
    }
    if (parts > 1) {
        const auto cluster = cooperative_groups::this_cluster();
        cluster.sync();
        if (part == 0 && warp == 0) {
            const Sums all = warp_sum(*cluster.map_shared_rank(&s_all, lane % parts), parts);
            for (int i = lane; i < parts * a.top; i += 32) s_found[i] = cluster.map_shared_rank(s_best, i / a.top)[i % a.top];
            __syncwarp();
            if (lane < a.top) s_best[lane] = 0;
            __syncwarp();
            if (a.top) rank_top(s_found, parts * a.top, a.top, s_best, lane, 32);
            if (lane == 0) {
                s_all = all;
                write_row<T>(a, r, row.x, row.mask, all);
            }
        }
        cluster.sync();   // nobody leaves while its shared memory is read
        if (part) return;
    } else if (a.top) {
        __syncthreads();
    }
    for (int k = threadIdx.x; k < a.top; k += THREADS)
        write_top(a, r, k, s_best[k] != 0, key_class(s_best[k]), key_score(s_best[k]), s_all.m, logf(s_all.S));
}

// ----------------------------------------------------------------------------------------------
// Short rows: a group of G lanes a row
// ----------------------------------------------------------------------------------------------
// The whole row is held in registers, PER pieces a lane (16 scores, or 32 for the longest), so the maximum comes first and the sums
// after it.
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

// The alternatives of a row that a group of lanes holds.
template <class T, int G, int PER>
__device__ __forceinline__ void short_top(const Forward& a, long long r, const Row<T>& row, float (&v)[PER][Row<T>::VEC], const Sums& s) {
    constexpr int VEC = Row<T>::VEC;
    const int g = threadIdx.x % G;
    const float log_S = logf(s.S);
    // One word a score: as much of its order as fits above its class, so that a maximum of words is a maximum of scores with the lowest
    // class first among equal ones.  16-bit scores fit; fp32 scores lose their lowest bits, and where two of the best (or the
    // last and the next) agree in what is left, the warp takes the exact rounds below instead.
    int bits = 16;
    if constexpr (sizeof(T) == 4) bits = 32 - __clz(a.classes - 1 | 1);
    const unsigned low = (1u << bits) - 1;
    unsigned word[PER][VEC];
#pragma unroll
    for (int i = 0; i < PER; ++i)
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            const unsigned up = sizeof(T) == 4 ? order_of(v[i][k]) : order_of_16(from_float<T>(v[i][k])) << 16;
            word[i][k] = v[i][k] > -INFINITY ? (up & ~low) | (low - (unsigned)(row.first(g + i * G) + k)) : 0u;
        }
    bool close = false;
    unsigned last = ~0u, mine = 0;   // `mine`: the group's lanes take the found ones in turn, and write them together
    for (int k = 0; k < a.top + (sizeof(T) == 4 ? 1 : 0); ++k) {
        unsigned best = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i)
#pragma unroll
            for (int q = 0; q < VEC; ++q) best = max(best, word[i][q] - last);   // (words below `last` wrap around to above the others)
#pragma unroll
        for (int o = G / 2; o; o /= 2) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        const unsigned next = best + last;
        const unsigned found = last == 0 || next >= last ? 0u : next;
        if (sizeof(T) == 4 && k && found) close |= ((found ^ last) & ~low) == 0;
        last = found;
        if (k >= a.top) break;
        if (k % G == g) mine = found;
        if (k % G == G - 1 || k == a.top - 1) {
            if (g <= k % G && r < a.n) {
                const int id = (int)(low - (mine & low));
                write_top(a, r, k - k % G + g, mine != 0, id, mine ? as_float(row.x[id]) : 0.f, s.m, log_S);
            }
        }
    }
    if constexpr (sizeof(T) == 4) {
        if (!__any_sync(0xffffffffu, close)) return;
        for (int k = 0; k < a.top; ++k) {
            float m = s.m;
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
            if (k % G == g && r < a.n) write_top(a, r, k, m > -INFINITY, at, m, s.m, log_S);
        }
    }
}

// A group does ROWS rows one after the other, and a lane each of what is to be done once a row (ROWS = 1 where rows are few).
template <class T, int G, int PER, int ROWS>
__global__ void __launch_bounds__(kShortThreads) k_short_rows(const Forward a) {
    static_assert(ROWS == 1 || ROWS <= G, "a lane a row");
    constexpr int VEC = Row<T>::VEC;
    const int g = threadIdx.x % G;
    const long long r0 = ((long long)blockIdx.x * (kShortThreads / G) + threadIdx.x / G) * ROWS;
    Row<T> row(a, min(r0, a.n - 1));   // (groups past the end do the last row once more, and write nothing: lanes stay together)
    Sums own{};                        // of row r0 + g
    const float2 c2 = make_float2(a.c, a.c);
#pragma unroll 1
    for (int u = 0; u < ROWS; ++u) {
        const long long r = r0 + u;
        if (u && r < a.n) row.at(row.x + a.stride, row.mask ? row.mask + a.mask_stride : nullptr);
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
            for (int k = 0; k < VEC; k += 2) m = max_nan(m, v[i][k], v[i][k + 1]);
#pragma unroll
        for (int o = G / 2; o; o /= 2) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float2 minus = make_float2(-m, -m);
        float2 S = make_float2(0.f, 0.f), Q = S;
#pragma unroll
        for (int i = 0; i < PER; ++i)
#pragma unroll
            for (int k = 0; k < VEC; k += 2) {
                float2 d = __fmul2_rn(__fadd2_rn(make_float2(v[i][k], v[i][k + 1]), minus), c2);
                d.x = fmaxf(d.x, kFar);
                d.y = fmaxf(d.y, kFar);
                const float2 e = make_float2(exp_2(d.x), exp_2(d.y));
                S = __fadd2_rn(S, e);
                Q = __ffma2_rn(e, d, Q);
            }
        const Sums s = group_sum<G>(Sums{m, S.x + S.y, Q.x + Q.y});
        if (u == g) own = s;
        if (a.top) short_top<T, G, PER>(a, r, row, v, s);
    }
    if (g < ROWS && r0 + g < a.n) {
        row.at((const T*)a.x + (r0 + g) * a.stride, a.mask ? a.mask + (r0 + g) * a.mask_stride : nullptr);
        write_row<T>(a, r0 + g, row.x, row.mask, own);
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
    bool weights = A != 0.f;   // any: their sum may be 0 where they are not (a margin of two classes)
    const bool broken = !(st.x < INFINITY);   // no alternatives there, and NaN for their log probabilities
    if (a.g_top)
        for (int k = 0; k < a.top; ++k) {
            const bool has = a.top_ids[r * a.top + k] >= 0;
            if (!has && !broken) continue;
            const float t = a.g_top[r * a.top + k];
            weights |= t != 0.f;
            if (has) A += t;
        }
    const float b = a.g_entropy ? a.g_entropy[r] : 0.f;
    RowGrad g;
    g.m = st.x;
    g.c = a.c;
    g.zero = st.x == -INFINITY || (!weights && b == 0.f);
    // log p + entropy = d ln 2 - log S + entropy
    g.inv_S = broken ? NAN : 1.f / st.y;
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
    if ((row.mask && !row.mask[j]) || x == -INFINITY) return;   // as it is
    dx[j] = from_float<T>(a.scale * (own + without_own(g, x)));
}
// The k-th of the classes with weights: the target, then the alternatives.
template <class T>
__device__ __forceinline__ void write_own_of(const Backward& a, long long r, const RowGrad& g, const Row<T>& row, int k) {
    const long long j = k ? a.top_ids[r * a.top + k - 1] : a.g_logprobs ? load_target(a.target, a.target64, r) : -1;
    if (j < 0 || j >= a.classes || (k == 0 && !target_counts(a, j))) return;
    write_own<T>(a, r, g, row, (T*)a.dx + r * a.dx_stride, j);
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
            bool out = v[k] == -INFINITY;   // masked, or as good as
            if (out && g.inv_S != g.inv_S)   // in a row without a distribution what is not masked is NaN
                out = (unsigned)(j + k) >= (unsigned)row.classes || (row.mask && !row.mask[j + k]);
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

constexpr int kGradTurn = 4, kGradPieces = 2 * kGradTurn;   // pieces per thread: turns of four whose loads are under way together

template <class T, int THREADS, bool MASKED>
__global__ void __launch_bounds__(THREADS) k_row_grad(const Backward a, int parts) {
    constexpr int VEC = Row<T>::VEC;
    const long long r = blockIdx.x / parts;
    const int part = (int)(blockIdx.x - r * parts);
    const Row<T> row(a, r);
    T* dx = (T*)a.dx + r * a.dx_stride;
    const RowGrad g = row_grad(a, r);
    const int per = (row.pieces + parts - 1) / parts, p0 = min(row.pieces, part * per), p1 = min(row.pieces, p0 + per);
    // Whole pieces whose places in dx are aligned as in x.  Where they are not (scores cut from a padded product, and a dx without gaps) the
    // row goes by write_piece, its stores element by element: 4096 rows of 50021 bf16 scores, 50024 apart, 533 us; into a dx with the same
    // gaps 134, as without gaps on both sides.
    const bool straight = (uintptr_t)(dx - row.head) % 16 == 0;
    const bool broken = MASKED && g.inv_S != g.inv_S;   // what is masked is 0 even there: piece by piece
    const int q0 = straight && !broken ? max(p0, row.head ? 1 : 0) : p1, q1 = min(p1, (row.head + row.classes) / VEC);
    if (g.zero) {
        for (int piece = p0 + threadIdx.x; piece < p1; piece += THREADS) write_piece<T>(a, g, row, dx, piece);
        return;
    }
    const float2 minus = make_float2(-g.m, -g.m), c2 = make_float2(g.c, g.c), A2 = make_float2(g.A, g.A), B2 = make_float2(g.B, g.B);
    const float f = -a.scale * g.inv_S * (g.B != 0.f ? 1.f : g.A);
    const float2 f2 = make_float2(f, f);
    const MaskWords<VEC> mask(row.mask, row.head);
    auto whole = [&](auto with_d) {
        for (int base = q0 + threadIdx.x; base < q1; base += kGradTurn * THREADS) {
            Piece<T, VEC> w[kGradTurn];
            unsigned bits[kGradTurn][MaskWords<VEC>::WORDS];
#pragma unroll
            for (int u = 0; u < kGradTurn; ++u)
                if (base + u * THREADS < q1) {
                    w[u] = *(const Piece<T, VEC>*)(row.x + row.first(base + u * THREADS));
                    if (MASKED) mask.fetch(bits[u], base + u * THREADS);
                }
#pragma unroll
            for (int u = 0; u < kGradTurn; ++u) {
                if (base + u * THREADS >= q1) break;
                if (MASKED) mask.apply(w[u], bits[u]);
                float v[VEC];
                as_floats(w[u], v);
                Piece<T, VEC> q;
#pragma unroll
                for (int k = 0; k < VEC; k += 2) {
                    float2 d = __fmul2_rn(__fadd2_rn(make_float2(v[k], v[k + 1]), minus), c2);
                    if (with_d) {
                        d.x = fmaxf(d.x, kFar);
                        d.y = fmaxf(d.y, kFar);
                    }
                    const float2 p = __fmul2_rn(make_float2(exp_2(d.x), exp_2(d.y)), f2);
                    const float2 y = with_d ? __fmul2_rn(p, __ffma2_rn(B2, d, A2)) : p;
                    q.v[k] = from_float<T>(y.x);
                    q.v[k + 1] = from_float<T>(y.y);
                }
                *(Piece<T, VEC>*)(dx + row.first(base + u * THREADS)) = q;
            }
        }
    };
    if (g.B != 0.f) whole(std::true_type());
    else whole(std::false_type());   // the weight is A for all
    // the others: those that the row's ends cut, or all
    for (int piece = p0 + threadIdx.x; piece < min(q0, p1); piece += THREADS) write_piece<T>(a, g, row, dx, piece);
    for (int piece = max(q0, q1) + threadIdx.x; piece < p1; piece += THREADS) write_piece<T>(a, g, row, dx, piece);
    __syncthreads();   // classes with weights of their own are written once more, by one thread each (equal values where they coincide)
    for (int k = threadIdx.x; k < 1 + (a.g_top ? a.top : 0); k += THREADS) {
        const long long j = k ? a.top_ids[r * a.top + k - 1] : a.g_logprobs ? load_target(a.target, a.target64, r) : -1;
        if (j < 0 || j >= a.classes || (k == 0 && !target_counts(a, j))) continue;
        const int piece = (int)((j + row.head) / VEC);
        if (piece >= p0 && piece < p1) write_own<T>(a, r, g, row, dx, j);
    }
}

// A group does ROWS rows one after the other; what a row needs beside its scores is a lane's to fetch, and to write what has weights of its own.
template <class T, int G, int PER, int ROWS>
__global__ void __launch_bounds__(kShortThreads) k_short_rows_grad(const Backward a) {
    static_assert(ROWS == 1 || ROWS <= G, "a lane a row");
    const int g = threadIdx.x % G;
    const long long r0 = ((long long)blockIdx.x * (kShortThreads / G) + threadIdx.x / G) * ROWS;
    const long long mine = min(r0 + (ROWS == 1 ? 0 : g % ROWS), a.n - 1);
    const RowGrad own = row_grad(a, mine);
    Row<T> row(a, min(r0, a.n - 1));
    T* dx = (T*)a.dx + min(r0, a.n - 1) * a.dx_stride;
#pragma unroll 1
    for (int u = 0; u < ROWS; ++u) {
        RowGrad w = own;
        if (ROWS > 1) {
            w.m = __shfl_sync(0xffffffffu, own.m, u, G);
            w.inv_S = __shfl_sync(0xffffffffu, own.inv_S, u, G);
            w.A = __shfl_sync(0xffffffffu, own.A, u, G);
            w.B = __shfl_sync(0xffffffffu, own.B, u, G);
            w.zero = __shfl_sync(0xffffffffu, (int)own.zero, u, G);
        }
        if (r0 + u < a.n) {
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (g + i * G < row.pieces) write_piece<T>(a, w, row, dx, g + i * G);
            row.at(row.x + a.stride, row.mask ? row.mask + a.mask_stride : nullptr);   // (only looked at where there is a next row)
            dx += a.dx_stride;
        }
    }
    __syncwarp();   // behind the lanes of the row, as in k_row_grad
    if (ROWS > 1) {
        if (g >= ROWS || r0 + g >= a.n || own.zero) return;
        const Row<T> its(a, mine);
        for (int k = 0; k < 1 + (a.g_top ? a.top : 0); ++k) write_own_of<T>(a, mine, own, its, k);
    } else {
        if (r0 >= a.n || own.zero) return;
        const Row<T> its(a, mine);
        for (int k = g; k < 1 + (a.g_top ? a.top : 0); k += G) write_own_of<T>(a, mine, own, its, k);
    }
}

// Lanes and pieces per lane that hold a row of so many pieces, and rows a group.  Longer ones are a CTA's: forward from 128 pieces on, the
// gradient from 64 (2^27 fp16 scores, us: 1000 classes 136 by groups, 148 by CTAs; their gradient 194, 119; of 300 classes 379, 392).
constexpr int kShortScores = 16, kShortPieces = 128, kShortPiecesGrad = 64;
template <class T, int MOST, class Fn>   // MOST: pieces of the longest row
int with_short(int pieces, long long n, Fn fn) {
    constexpr int PER = kShortScores / Row<T>::VEC;
    auto rows = [&](auto g, auto per) {
        constexpr int G = decltype(g)::value, ROWS = G < 8 ? G : 8;
        if (ROWS > 1 && n * G / ROWS >= 4 * 148 * 1024) return fn(g, per, std::integral_constant<int, ROWS>());   // otherwise more lanes are worth more
        return fn(g, per, std::integral_constant<int, 1>());
    };
    const std::integral_constant<int, PER> per;
    if (pieces <= PER) return rows(std::integral_constant<int, 1>(), per);
    if (pieces <= 2 * PER) return rows(std::integral_constant<int, 2>(), per);
    if (pieces <= 4 * PER) return rows(std::integral_constant<int, 4>(), per);
    if (pieces <= 8 * PER) return rows(std::integral_constant<int, 8>(), per);
    if constexpr (MOST > 16 * PER) {
        if constexpr (MOST > 32 * PER) {
            if (pieces > 32 * PER) return rows(std::integral_constant<int, 32>(), std::integral_constant<int, 2 * PER>());
        }
        if (pieces > 16 * PER) return rows(std::integral_constant<int, 32>(), per);
    }
    return rows(std::integral_constant<int, 16>(), per);
}
// Pieces of a row, wherever it begins.
template <class T>
int most_pieces(int classes) { return (int)ceil_div64((long long)classes + Row<T>::VEC - 1, Row<T>::VEC); }

template <class T, int THREADS, bool MASKED>
int launch_rows(long long n, int parts, cudaStream_t st, const Forward& a) {
    if (n * parts > 0x7fffffffll) return TRS_E_LIMIT;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)parts;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(n * parts));
    cfg.blockDim = dim3(THREADS);
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = parts > 1 ? 1 : 0;
    TRS_CUDA(cudaLaunchKernelEx(&cfg, k_row<T, THREADS, MASKED>, a, parts));
    return TRS_OK;
}

Extent extent(const void* p, long long rows, long long stride, long long width, int size) {
    return {(uintptr_t)p, (uintptr_t)p + (size_t)((rows - 1) * stride + width) * size};
}

int check(const void* x, int type, long long n, int classes, long long stride, const void* mask, long long mask_stride, float scale,
          int top) {
    if (!type_known(type) || n < 0 || classes < 1 || stride < classes || top < 0 || !(scale > 0.f) || !(scale * kLog2e < INFINITY)) return TRS_E_ARG;
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
    if ((logprobs && (!targets || (uintptr_t)targets % (targets64 ? 8 : 4))) || ((uintptr_t)logprobs | (uintptr_t)entropy) % 4 ||
        ((uintptr_t)top_logprobs | (uintptr_t)top_ids) % 4)
        return TRS_E_ARG;
    if ((top && (!top_logprobs || !top_ids)) || (uintptr_t)stats % 8) return TRS_E_ARG;
    const Forward a{x, n, stride, classes, targets, targets64, ignore_id, mask, mask_stride, extent(x, n, stride, classes, type_bytes(type)), extent(mask, n, mask_stride, classes, 1), scale, scale * kLog2e, top, logprobs, entropy,
                    top_logprobs, top_ids, (float2*)stats};
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        const int pieces = most_pieces<T>(classes);
        if (pieces <= kShortPieces)
            return with_short<T, kShortPieces>(pieces, n, [&](auto g, auto per, auto rows) {
                constexpr int G = decltype(g)::value, ROWS = decltype(rows)::value;
                return launch(k_short_rows<T, G, decltype(per)::value, ROWS>, dim3((unsigned)ceil_div64(ceil_div64(n, ROWS) * G, kShortThreads)),
                              kShortThreads, 0, (cudaStream_t)stream, a);
            });
        auto run = [&](auto threads, int parts) {
            constexpr int THREADS = decltype(threads)::value;
            return a.mask ? launch_rows<T, THREADS, true>(n, parts, (cudaStream_t)stream, a)
                          : launch_rows<T, THREADS, false>(n, parts, (cudaStream_t)stream, a);
        };
        // As few threads a row as keep it going, many rows at a time: what a row costs beside its scores grows with its threads.  2^27 fp16
        // scores by 32 / 64 / 128 / 256 threads, us: 2000 classes 99 / 122 / 146 / 247, 9000: 67 / 56 / 62 / 87, 33000:
        // 70 / 54 / 52 / 56; 2^27 fp32 scores in rows of 33000: 89 / 99 / 93 / 97.
        int threads = sizeof(T) == 4 ? (pieces <= 8192 ? 32 : 256) : pieces <= 640 ? 32 : pieces <= 2400 ? 64 : pieces <= 8192 ? 128 : 256;
        while (threads < 256 && n * threads < 148 * 1024 && pieces > threads * kTurn) threads *= 2;   // unless rows are few
        if (threads == 32) return run(std::integral_constant<int, 32>(), 1);
        if (threads == 64) return run(std::integral_constant<int, 64>(), 1);
        if (threads == 128) return run(std::integral_constant<int, 128>(), 1);
        // Very few rows: parts until there are two CTAs an SM (or a part has one turn).  More of them only add ends: 512 rows of 2^18 masked
        // fp16 scores, ten alternatives: 87 us whole, 92 / 96 / 125 us in 2 / 4 / 8 parts.
        int parts = 1;
        while (parts < kMaxParts && n * parts < 2 * 148 && pieces > parts * 256 * kTurn) parts *= 2;
        if (n * parts < 2 * 148) return run(std::integral_constant<int, 512>(), parts);
        return run(std::integral_constant<int, 256>(), parts);
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
    if (((uintptr_t)entropy | (uintptr_t)g_logprobs | (uintptr_t)g_entropy | (uintptr_t)g_top_logprobs | (uintptr_t)top_ids) % 4) return TRS_E_ARG;
    if ((g_logprobs && (!targets || (uintptr_t)targets % (targets64 ? 8 : 4))) || (g_entropy && !entropy) || (g_top_logprobs && (!top_ids || !top))) return TRS_E_ARG;
    const Backward a{x, n, stride, classes, targets, targets64, ignore_id, mask, mask_stride, extent(x, n, stride, classes, type_bytes(type)), extent(mask, n, mask_stride, classes, 1), scale, scale * kLog2e, top, top_ids,
                     (const float2*)stats, entropy, g_logprobs, g_entropy, g_top_logprobs, dx, dx_stride};
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        const int pieces = most_pieces<T>(classes);
        if (pieces <= kShortPiecesGrad)
            return with_short<T, kShortPiecesGrad>(pieces, n, [&](auto g, auto per, auto rows) {
                constexpr int G = decltype(g)::value, ROWS = decltype(rows)::value;
                return launch(k_short_rows_grad<T, G, decltype(per)::value, ROWS>,
                              dim3((unsigned)ceil_div64(ceil_div64(n, ROWS) * G, kShortThreads)), kShortThreads, 0, (cudaStream_t)stream, a);
            });
        auto run = [&](auto threads) {
            constexpr int THREADS = decltype(threads)::value;
            const long long parts = ceil_div64(pieces, THREADS * kGradPieces);
            if (n * parts > 0x7fffffffll) return (int)TRS_E_LIMIT;
            return launch(a.mask ? k_row_grad<T, THREADS, true> : k_row_grad<T, THREADS, false>, dim3((unsigned)(n * parts)), THREADS, 0,
                          (cudaStream_t)stream, a, (int)parts);
        };
        // (2^27 fp16 scores by 32 / 64 / 256 threads, us: 1100 classes 144 / 195 / 525, 9000: 98 / 93 / 107, 33000: 94 / 88 / 99)
        if (pieces <= 32 * kGradPieces) return run(std::integral_constant<int, 32>());
        return run(std::integral_constant<int, 64>());
    });
}
TRS_CATCH
