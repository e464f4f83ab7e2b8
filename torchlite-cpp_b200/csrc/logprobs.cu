// Log-probabilities of given tokens under logits [..., V], with the entropy
// and the most likely alternatives, and the gradient to the logits, fp32.
//
//   z_j = scale (x_j - max x),  l = sum e^z_j,  log p_j = z_j - log l
//   out = log p_t,  H = -sum p_j log p_j = log l - sum e^z_j z_j / l
//   dx_j = scale (g (1[j = t] - p_j) - h p_j (log p_j + H)),   g, h: the gradients of out and H
//
// Everything goes by differences to the row's maximum, so large logits lose
// nothing; the maximum and log l are what the backward needs (`stats`).
// One pass over the logits: the lanes of a warp share a running maximum m, and
// each keeps l = sum e^(scale (x - m)) and w = sum e^(.) log2 e^(.) of its own
// values, rescaled when m grows.  Bound by HBM: 4 bytes a logit forward, 8 backward.  Measured (GPU
// time): 4095 x 50001 with 5 alternatives 140 us (5.8 TB/s), 1200 x 262143 203
// us (6.2 TB/s), 8192 x 2001 17 us (3.8 TB/s); the gradient 4096 x 50001 267 us
// (6.1 TB/s).
//
// Short rows are read by a warp each, others by a block, or by a cluster of
// blocks when the rows alone would leave SMs idle.
//
// The alternatives need no second pass over the row: every thread knows the
// largest of its own values, so what k of the maxima of disjoint sets of values
// reach is a bound that the k largest values all reach, and only the few
// threads whose maximum reaches it look at their values again.  Where that bound
// leaves more values than the list holds (many equal logits, or fewer above -inf
// than alternatives, so that the bound is -inf) the row is read again: by a block
// nine times, a digit of the k-th key each, by a warp once for each alternative.
// With 3 logits above -inf 4095 x 50001 with 5 alternatives takes 7.2 ms (137 us
// ordinarily), 8192 x 2001 with 20 takes 444 us (48), 1 x 131072 with 20 176 us (12).
//
// Cases without a distribution: a row of -inf alone has log p = -inf,
// entropy 0 and no gradient; a NaN or +inf in a row makes its results NaN.
// Token -1: no token is asked for (log p = 0, no gradient from it); any other
// token outside [0, V) gives NaN.
#include <algorithm>
#include <cmath>
#include <utility>

#include "rows.cuh"
#include "tcgen05.cuh"

namespace tlc {
namespace {

constexpr const char* kFwd = "token_logprobs";
constexpr const char* kBwd = "token_logprobs_backward";
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kMaxTop = 32;

// 2^x to 2 ulp, 0 below 2^-126: the probabilities' own rounding is what the sums see.
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The larger, NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
// The largest of three, NaN if one is; the smallest of three numbers.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float y;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
    float y;
    asm("min.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
// Exponents below this give 0; the bound keeps 0 * exponent from being NaN.
constexpr float kFloor = -160.0f;

// ---- running sums ---------------------------------------------------------------------

// m: maximum (-inf: nothing yet), l = sum 2^y, w = sum 2^y y with y = a (x - m), a = scale log2 e.
struct Run {
    float m = -INFINITY, l = 0.0f, w = 0.0f;
    __device__ __forceinline__ void raise(float to, float a) {
        if (m == -INFINITY) {
            m = to;
            return;
        }
        const float y = max_nan((m - to) * a, kFloor);
        const float c = ex2(y);
        w = c * fmaf(y, l, w);
        l *= c;
        m = to;
    }
};

// Adds values to a run, two at a time: 8 instructions for two values.  The lanes
// of a warp add together and share the running maximum, so that it moves a few
// times a row (each lane's own moves in some lane in nearly every batch).
struct PairRun {
    float m = -INFINITY;  // the warp's
    // for the alternatives, of this lane alone: batch `where` has the largest value `most`, batch
    // `where2` the second largest of the batches' maxima, `rest` is the largest of the others'
    float most = -INFINITY, second = -INFINITY, rest = -INFINITY;
    int where = 0, where2 = 0;
    Pair l, w, a2;
    float a;
    __device__ __forceinline__ explicit PairRun(float scale2) : l(0), w(0), a2(pair(scale2, scale2)), a(scale2) {}
    template <int N>
    __device__ __forceinline__ void add(const float (&v)[N], int batch) {
        float top = v[0], low = v[0];
#pragma unroll
        for (int i = 1; i < N; i += 2) {
            const float other = i + 1 < N ? v[i + 1] : v[i];
            top = max3_nan(top, v[i], other);
            low = min3(low, v[i], other);
        }
        if (__any_sync(0xffffffffu, !(top <= m))) {  // also when top is NaN
            float to = max_nan(top, m);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) to = max_nan(to, __shfl_xor_sync(0xffffffffu, to, o));
            if (m != -INFINITY) {
                const float y = max_nan((m - to) * a, kFloor), c = ex2(y);
                w = mul2(pair(c, c), fma2(pair(y, y), l, w));
                l = mul2(pair(c, c), l);
            }
            m = to;
        }
        // a new largest value pushes the old one to second place, a new second the old second out
        const bool first = top > most, one_of_two = top > second;
        rest = fmaxf(rest, one_of_two ? second : top);
        second = fmaxf(second, fminf(top, most));
        where2 = first ? where : one_of_two ? batch : where2;
        most = fmaxf(most, top);
        where = first ? batch : where;
        const float base = m == -INFINITY ? 0.0f : -m;
        const Pair shift = pair(base, base);
        // masked values need the bound on their exponent; without any it is left out
        if ((low + base) * a >= kFloor)
            exponentials<N, false>(v, shift);
        else
            exponentials<N, true>(v, shift);
    }
    template <int N, bool BOUND>
    __device__ __forceinline__ void exponentials(const float (&v)[N], Pair shift) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            Pair y2 = mul2(add2(pair(v[i], i + 1 < N ? v[i + 1] : -INFINITY), shift), a2);
            float y0, y1;
            unpair(y2, y0, y1);
            if (BOUND || i + 1 == N) {
                y0 = max_nan(y0, kFloor), y1 = max_nan(y1, kFloor);
                y2 = pair(y0, y1);
            }
            const Pair e = pair(ex2(y0), ex2(y1));
            l = add2(l, e);
            w = fma2(e, y2, w);
        }
    }
    __device__ __forceinline__ Run sum() const {
        Run r;
        float x, y;
        r.m = m;
        unpair(l, x, y);
        r.l = x + y;
        unpair(w, x, y);
        r.w = x + y;
        return r;
    }
};

// The runs of a warp's lanes as one, in every lane: all are raised to the common
// maximum first, then only sums are left.
__device__ __forceinline__ Run warp_run(Run r, float a) {
    float to = r.m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) to = max_nan(to, __shfl_xor_sync(0xffffffffu, to, o));
    if (r.m != to) r.raise(to, a);
    float s[2] = {r.l, r.w};
    warp_sum(s);
    r.m = to, r.l = s[0], r.w = s[1];
    return r;
}
// The same where the lanes have one maximum already.
__device__ __forceinline__ Run warp_run(const PairRun& own) {
    Run r = own.sum();
    float s[2] = {r.l, r.w};
    warp_sum(s);
    r.l = s[0], r.w = s[1];
    return r;
}

// ---- order of the alternatives --------------------------------------------------------

// Larger value first, NaN before all, then the lower index: one unsigned key.
__device__ __forceinline__ uint32_t order_of(float v) {
    if (v != v) return 0xffffffffu;
    const uint32_t u = __float_as_uint(v + 0.0f);  // -0 as +0
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ uint64_t key_of(float v, uint32_t index) {
    return ((uint64_t)order_of(v) << 32) | (uint32_t)~index;
}
__device__ __forceinline__ uint32_t index_of(uint64_t key) { return ~(uint32_t)key; }
__device__ __forceinline__ float value_of(uint64_t key) {
    const uint32_t u = (uint32_t)(key >> 32);
    return u == 0xffffffffu ? __int_as_float(0x7fc00000) : __uint_as_float((u & 0x80000000u) ? u ^ 0x80000000u : ~u);
}

// The highest bound that k of a warp's values (some a lane) reach, to its first
// 16 bits: sign, exponent, 7 of the mantissa.
template <class... V>
__device__ __forceinline__ uint32_t highest_bound(int k, V... v) {
    uint32_t bound = 0;
#pragma unroll
    for (int bit = 31; bit >= 16; --bit) {
        const uint32_t to = bound | (1u << bit);
        const int reach = (__popc(__ballot_sync(0xffffffffu, v >= to)) + ...);
        if (reach >= k) bound = to;
    }
    return bound;
}

struct LpFwd {
    const float* x;
    Rows xm;
    TokenRef tok;
    int64_t rows;
    int V;
    float scale, a;  // a = scale * log2 e
    float *logp, *entropy, *stats;
    int top;
    float* top_logp;
    void* top_tok;
    int top_wide;
};

// The token of a row and its logit.
struct Asked {
    int64_t t = -1;
    float x = 0.0f;
    Asked() = default;
    __device__ __forceinline__ Asked(const LpFwd& p, int64_t r, const float* row) {
        if (!p.logp) return;
        t = p.tok.get(r);
        if (t >= 0 && t < p.V) x = row[t];
    }
};

// What the row's results are, from its sums.
__device__ __forceinline__ void row_results(const LpFwd& p, int64_t r, const Asked& q, const Run& s) {
    const bool none = s.m == -INFINITY;
    const float log_l = none ? 0.0f : logf(s.l);
    if (p.stats) {
        p.stats[2 * r] = s.m;
        p.stats[2 * r + 1] = log_l;
    }
    if (p.entropy) p.entropy[r] = none ? 0.0f : fmaxf(log_l - kLn2 * (s.w / s.l), 0.0f) + (s.l != s.l ? s.l : 0.0f);
    if (p.logp) {
        float lp = 0.0f;
        if (q.t != -1) {
            if (q.t < 0 || q.t >= p.V)
                lp = __int_as_float(0x7fc00000);
            else
                lp = none ? -INFINITY : (q.x - s.m) * p.scale - log_l;
        }
        p.logp[r] = lp;
    }
}

__device__ __forceinline__ void top_result(const LpFwd& p, int64_t r, int i, uint64_t key, float m, float log_l) {
    const uint32_t j = index_of(key);
    p.top_logp[r * p.top + i] = m == -INFINITY ? -INFINITY : (value_of(key) - m) * p.scale - log_l;
    if (p.top_wide)
        static_cast<int64_t*>(p.top_tok)[r * p.top + i] = j;
    else
        static_cast<int32_t*>(p.top_tok)[r * p.top + i] = (int32_t)j;
}

// ---- the copies ahead -------------------------------------------------------------------

constexpr int BATCH = 4;   // float4 that a thread takes at once
constexpr int STAGES = 3;  // batches in shared memory or on their way to it

// A block's (or warp's) part of a row: the first `head` values singly up to a 16-byte
// boundary, then `vecs` float4, then `tail` values.
struct Part {
    const float* x;  // the part's first value
    int first, n;    // its index in the row, and how many
    int head, vecs, tail;
    __device__ __forceinline__ Part(const float* row, int lo, int hi) {
        x = row + lo;
        first = lo;
        n = hi - lo;
        head = min(n, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) >> 2);
        vecs = (n - head) >> 2;
        tail = n - head - 4 * vecs;
    }
    __device__ __forceinline__ float4 vec(int i) const {
        return __ldcs(reinterpret_cast<const float4*>(x + head) + i);
    }
    // the single value of thread t < 6, if it has one: its position in the part, or -1
    __device__ __forceinline__ int single(int t) const {
        if (t < 3) return t < head ? t : -1;
        if (t < 6) return t - 3 < tail ? head + 4 * vecs + t - 3 : -1;
        return -1;
    }
};

// The values of a thread's rows, batch by batch, through a ring of asynchronous
// copies that runs across the rows' ends, so that the memory stays busy while a
// row's results are put together.  T threads of a 256-thread block share a row;
// a thread copies what it reads itself, which needs no barrier.  Whole batches,
// nearly all of them, go without tests of single vectors.
template <int T>
struct Feed {
    static constexpr int STEP = BATCH * T;  // vectors of a batch
    float4* ring;                           // [STAGES][BATCH][256], this thread's
    int t;
    const LpFwd& p;
    int lo, hi;
    int64_t row, step;
    const float4* src = nullptr;  // this thread's next vector of the row being copied
    int left = 0;                 // vectors of that row, from thread 0's next one on
    int stage = 0;
    __device__ __forceinline__ Feed(float4* ring_, int t_, const LpFwd& p_, int lo_, int hi_, int64_t first, int64_t step_)
        : ring(ring_), t(t_), p(p_), lo(lo_), hi(hi_), row(first), step(step_) {
        open();
#pragma unroll
        for (int q = 0; q < STAGES; ++q) fetch(q);
    }
    template <int... U>
    __device__ __forceinline__ void copy_batch(uint32_t to, const float4* from, std::integer_sequence<int, U...>) {
        (copy_at<U * 256 * 16, U * T * 16>(to, from), ...);
    }
    template <int TO, int FROM>
    __device__ __forceinline__ void copy_at(uint32_t to, const float4* from) {
        asm volatile("cp.async.cg.shared.global [%0+%2], [%1+%3], 16;" ::"r"(to), "l"(from), "n"(TO), "n"(FROM) : "memory");
    }
    __device__ __forceinline__ void open() {
        if (row >= p.rows) return;
        const Part part(p.x + p.xm.offset(row), lo, hi);
        src = reinterpret_cast<const float4*>(part.x + part.head) + t;
        left = part.vecs;
    }
    __device__ __forceinline__ void fetch(int to) {
        if (row < p.rows) {
            const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(ring + to * BATCH * 256));
            if (left >= STEP) {
                copy_batch(at, src, std::make_integer_sequence<int, BATCH>());
            } else {
#pragma unroll
                for (int u = 0; u < BATCH; ++u)
                    if (t + u * T < left)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at + u * 256 * 16), "l"(src + u * T)
                                     : "memory");
            }
            src += STEP;
            left -= STEP;
            if (left <= 0) {  // every row has one batch at least
                row += step;
                open();
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    // all of one row's batches, then its single value
    __device__ __forceinline__ void add_row(const Part& now, PairRun& own) {
        const int alone_at = now.single(t);
        const float alone = alone_at >= 0 ? now.x[alone_at] : -INFINITY;
        int batch = 0, rest = now.vecs;
        do {
            asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
            float v[4 * BATCH];
            const float4* from = ring + stage * BATCH * 256;
            if (rest >= STEP) {
#pragma unroll
                for (int u = 0; u < BATCH; ++u) {
                    const float4 f = from[u * 256];
                    v[4 * u] = f.x, v[4 * u + 1] = f.y, v[4 * u + 2] = f.z, v[4 * u + 3] = f.w;
                }
            } else {
#pragma unroll
                for (int u = 0; u < BATCH; ++u) {
                    float4 f = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                    if (t + u * T < rest) f = from[u * 256];
                    v[4 * u] = f.x, v[4 * u + 1] = f.y, v[4 * u + 2] = f.z, v[4 * u + 3] = f.w;
                }
            }
            fetch(stage);  // into what was just read
            stage = stage + 1 == STAGES ? 0 : stage + 1;
            own.add(v, batch);
            ++batch;
            rest -= STEP;
        } while (rest > 0);
        if (__any_sync(0xffffffffu, alone_at >= 0)) {
            const float v[1] = {alone};
            own.add(v, -1);
        }
    }
    __device__ __forceinline__ void end() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }
};

// One batch of thread t's values, seen again by that thread (-1: its single value).
template <int T, class F>
__device__ __forceinline__ void look_at_batch(const Part& part, int t, int batch, F&& take) {
    if (batch < 0) {
        const int at = part.single(t);
        take(part.x[at], at);
        return;
    }
    float4 f[BATCH];
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
        const int i = (batch * BATCH + u) * T + t;
        if (i < part.vecs) f[u] = part.vec(i);
    }
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
        const int i = (batch * BATCH + u) * T + t, at = part.head + 4 * i;
        if (i < part.vecs) {
            take(f[u].x, at);
            take(f[u].y, at + 1);
            take(f[u].z, at + 2);
            take(f[u].w, at + 3);
        }
    }
}
// The float4 [begin, end) of thread t's values, and its single one if asked,
// seen again by a warp together.
template <int T, class F>
__device__ __forceinline__ void look_together(const Part& part, int t, int begin, int end, bool alone, int lane, F&& take) {
    for (int i = begin + t + T * lane; i < end; i += T * 32) {
        const float4 f = part.vec(i);
        const int at = part.head + 4 * i;
        take(f.x, at);
        take(f.y, at + 1);
        take(f.z, at + 2);
        take(f.w, at + 3);
    }
    if (alone && lane == 0) {
        const int at = part.single(t);
        if (at >= 0) take(part.x[at], at);
    }
}

// ---- a row for a warp -------------------------------------------------------------------

constexpr int WARP_CAP = 128;  // candidates for the alternatives that a warp keeps

// A warp a row, 8 rows a block at once.
template <bool TOP>
__global__ void __launch_bounds__(256, 3) lp_warp_kernel(LpFwd p) {
    extern __shared__ __align__(16) float4 ring[];  // [STAGES][BATCH][256]
    __shared__ uint64_t cands[TOP ? 8 : 1][TOP ? WARP_CAP : 1];
    __shared__ int founds[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t first = blockIdx.x + (int64_t)gridDim.x * warp, step = (int64_t)gridDim.x * 8;
    Feed<32> feed(ring + threadIdx.x, lane, p, 0, p.V, first, step);
    for (int64_t r = first; r < p.rows; r += step) {
        const float* x = p.x + p.xm.offset(r);
        const Part part(x, 0, p.V);
        const Asked asked = lane == 0 ? Asked(p, r, x) : Asked();
        PairRun own(p.a);
        feed.add_row(part, own);
        const Run s = warp_run(own);
        if (lane == 0) row_results(p, r, asked, s);
        if constexpr (TOP) {
            uint64_t* cand = cands[warp];
            const float log_l = s.m == -INFINITY ? 0.0f : logf(s.l);
            int found = WARP_CAP + 1;
            if (s.m == s.m) {
                // Each lane has three maxima of disjoint sets of its values.  What `top` of
                // these 96 reach, `top` values reach.
                const uint32_t most = order_of(own.most), second = order_of(own.second), rest = order_of(own.rest);
                const uint32_t bound = highest_bound(p.top, most, second, rest);
                if (lane == 0) founds[warp] = 0;
                __syncwarp();
                auto take = [&](float v, int at) {
                    if (order_of(v) >= bound) {
                        const int c = atomicAdd(&founds[warp], 1);
                        if (c < WARP_CAP) cand[c] = key_of(v, (uint32_t)at);
                    }
                };
                // a lane looks at its one or two batches itself, at more with the others' help
                const bool many = rest >= bound;
                if (most >= bound && !many) look_at_batch<32>(part, lane, own.where, take);
                if (second >= bound && !many) look_at_batch<32>(part, lane, own.where2, take);
                __syncwarp();
                for (uint32_t left = __ballot_sync(0xffffffffu, many); left; left &= left - 1)
                    look_together<32>(part, __ffs(left) - 1, 0, part.vecs, true, lane, take);
                __syncwarp();
                found = founds[warp];
            }
            if (found <= WARP_CAP) {
                for (int c = lane; c < found; c += 32) {
                    const uint64_t key = cand[c];
                    int before = 0;
#pragma unroll 4
                    for (int o = 0; o < found; ++o) before += cand[o] > key;
                    if (before < p.top) top_result(p, r, before, key, s.m, log_l);
                }
            } else {
                // NaN, or too many equal values: one alternative a round, the largest key below the last
                uint64_t last = ~0ull;
                for (int i = 0; i < p.top; ++i) {
                    uint64_t best = 0;
                    for (int j = lane; j < p.V; j += 32) {
                        const uint64_t k = key_of(x[j], (uint32_t)j);
                        if (k < last && k > best) best = k;
                    }
                    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(best >> 32));
                    const uint32_t lo =
                        __reduce_max_sync(0xffffffffu, (uint32_t)(best >> 32) == hi ? (uint32_t)best : 0u);
                    last = ((uint64_t)hi << 32) | lo;
                    if (lane == 0) top_result(p, r, i, last, s.m, log_l);
                }
            }
            __syncwarp();  // the list is written again
        }
    }
    feed.end();
}

// ---- a row for a block or a cluster of blocks ----------------------------------------------

constexpr int CAP = 512;  // candidates for the alternatives that a block keeps

template <int T>
struct LpSmem {
    float m[T / 32], l[T / 32], w[T / 32];
    float row_m, row_l, row_w;         // the block's sums, read by the cluster's first block
    uint32_t group[64];
    uint32_t bound;
    int threads, found;
    uint16_t look[T];                  // threads whose values reach the bound
    int batch[T];                      // and in which batch: a number, -1 (the single value), -2 (any)
    uint64_t cand[CAP];
    uint64_t best[kMaxTop];            // the block's alternatives, in order
    uint64_t all[8 * kMaxTop];         // the cluster's, in its first block
    uint32_t hist[256];
    int bin, need;
};

// The part's `k` largest keys in order, into sm.best (k <= part.n values; the
// rest of sm.best is 0).  top: the largest number of this thread (-inf: none),
// which its batch `where` has (-1: its single value), rest: that of the others.
// sm.row_m, written by warp 0 before, is NaN if the part has one.
template <int T>
__device__ void part_top(LpSmem<T>& sm, const Part& part, int k, float top, float rest, int where) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int G = T / 64;  // neighbouring lanes a group
    uint32_t g = order_of(top);
#pragma unroll
    for (int o = 1; o < G; o <<= 1) g = max(g, __shfl_xor_sync(0xffffffffu, g, o));
    if (tid % G == 0) sm.group[tid / G] = g;
    if (tid == 0) sm.threads = sm.found = 0;
    if (tid < kMaxTop) sm.best[tid] = 0;
    __syncthreads();
    if (warp == 0) {
        const uint32_t reach = highest_bound(k, sm.group[lane], sm.group[lane + 32]);
        if (lane == 0) sm.bound = reach;
    }
    __syncthreads();
    const uint32_t bound = sm.bound;
    auto take = [&](float v, int at) {
        if (order_of(v) >= bound) {
            const int c = atomicAdd(&sm.found, 1);
            if (c < CAP) sm.cand[c] = key_of(v, (uint32_t)(part.first + at));
        }
    };
    // mostly no other batch of the thread reaches the bound: then one is looked at, else all
    if (order_of(top) >= bound) {
        const int c = atomicAdd(&sm.threads, 1);
        sm.look[c] = (uint16_t)tid;
        sm.batch[c] = order_of(rest) >= bound ? -2 : where;
    }
    __syncthreads();
    const int threads = sm.threads;
    for (int q = warp; q < threads; q += T / 32) {
        const int batch = sm.batch[q], begin = batch >= 0 ? batch * BATCH * T : 0;
        const int end = batch >= 0 ? min(part.vecs, begin + BATCH * T) : batch == -1 ? 0 : part.vecs;
        look_together<T>(part, sm.look[q], begin, end, batch < 0, lane, take);
    }
    __syncthreads();
    int found = sm.found;
    if (found > CAP || sm.row_m != sm.row_m) {
        // NaN, or too many values that reach the bound (equal logits, or few
        // that are not masked): find the k-th largest key digit by digit, reading the part
        // once for each of the 8 digits, then take the k keys from it up.
        uint64_t prefix = 0;
        if (tid == 0) sm.need = k;
        for (int shift = 56; shift >= 0; shift -= 8) {
            for (int b = tid; b < 256; b += T) sm.hist[b] = 0;
            __syncthreads();
            for (int i0 = 0; i0 < part.n; i0 += T) {
                const int i = i0 + tid;
                const uint64_t key = i < part.n ? key_of(part.x[i], (uint32_t)(part.first + i)) : 0;
                const bool in = i < part.n && (shift == 56 || (key >> (shift + 8)) == (prefix >> (shift + 8)));
                const uint32_t bin = (uint32_t)(key >> shift) & 255u;
                const uint32_t act = __ballot_sync(0xffffffffu, in);
                if (act) {
                    // equal digits are the rule here: one add for the lanes that share the first one's
                    const uint32_t b0 = __shfl_sync(0xffffffffu, bin, __ffs(act) - 1);
                    const uint32_t same = __ballot_sync(0xffffffffu, in && bin == b0);
                    if (lane == __ffs(act) - 1) atomicAdd(&sm.hist[b0], (uint32_t)__popc(same));
                    if (in && bin != b0) atomicAdd(&sm.hist[bin], 1u);
                }
            }
            __syncthreads();
            if (tid == 0) {
                int need = sm.need, b = 255;
                while (b > 0 && (int)sm.hist[b] < need) need -= (int)sm.hist[b--];
                sm.bin = b;
                sm.need = need;
            }
            __syncthreads();
            prefix |= (uint64_t)(uint32_t)sm.bin << shift;
            __syncthreads();
        }
        if (tid == 0) sm.found = 0;
        __syncthreads();
        for (int i = tid; i < part.n; i += T) {
            const uint64_t key = key_of(part.x[i], (uint32_t)(part.first + i));
            if (key >= prefix) sm.cand[min(atomicAdd(&sm.found, 1), CAP - 1)] = key;
        }
        __syncthreads();
        found = min(sm.found, CAP);
    }
    for (int c = tid; c < found; c += T) {
        const uint64_t key = sm.cand[c];
        int above = 0;
        for (int o = 0; o < found; ++o) above += sm.cand[o] > key;
        if (above < k) sm.best[above] = key;
    }
    __syncthreads();
}

// C blocks a row (1, or the cluster's size), T threads a block.  A block takes several
// rows in turn where there are more than blocks; a cluster has one (see launch_row).
template <int T>
__global__ void __launch_bounds__(T) lp_row_kernel(LpFwd p, int C) {
    extern __shared__ __align__(16) float4 ring[];  // [STAGES][BATCH][T]
    __shared__ LpSmem<T> sm;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = C > 1 ? (int)cluster_ctarank() : 0;
    const int64_t first = blockIdx.x / C, step = gridDim.x / C;
    const int per = ((p.V + C - 1) / C + 31) & ~31;
    const int lo = (int)min((int64_t)p.V, (int64_t)rank * per), hi = (int)min((int64_t)p.V, (int64_t)lo + per);

    static_assert(T == 256, "the ring's layout");
    Feed<T> feed(ring + tid, tid, p, lo, hi, first, step);
    for (int64_t r = first; r < p.rows; r += step) {
        const float* x = p.x + p.xm.offset(r);
        const Part part(x, lo, hi);
        const Asked asked = tid == 0 && rank == 0 ? Asked(p, r, x) : Asked();
        PairRun own(p.a);
        feed.add_row(part, own);
        const Run s = warp_run(own);
        if (lane == 0) sm.m[warp] = s.m, sm.l[warp] = s.l, sm.w[warp] = s.w;
        __syncthreads();
        if (warp == 0) {
            Run q;
            if (lane < T / 32) q.m = sm.m[lane], q.l = sm.l[lane], q.w = sm.w[lane];
            q = warp_run(q, p.a);
            if (lane == 0) sm.row_m = q.m, sm.row_l = q.l, sm.row_w = q.w;
        }
        const int k = min(p.top, part.n);
        if (k > 0)
            part_top(sm, part, k, own.most, fmaxf(own.second, own.rest), own.where);
        else if (p.top > 0 && tid < kMaxTop)
            sm.best[tid] = 0;
        __syncthreads();
        if (C == 1) {
            if (tid == 0) {
                Run q;
                q.m = sm.row_m, q.l = sm.row_l, q.w = sm.row_w;
                row_results(p, r, asked, q);
            }
            if (tid < p.top) {
                const float log_l = sm.row_m == -INFINITY ? 0.0f : logf(sm.row_l);
                top_result(p, r, tid, sm.best[tid], sm.row_m, log_l);
            }
            continue;  // what the next row writes first, nobody reads here
        }
        cluster_sync();
        if (rank == 0) {
            if (warp == 0) {
                Run q;
                if (lane < C) {
                    auto get = [&](const float* f) {
                        float v;
                        const uint32_t a = mapa(static_cast<uint32_t>(__cvta_generic_to_shared(f)), (uint32_t)lane);
                        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
                        return v;
                    };
                    q.m = get(&sm.row_m), q.l = get(&sm.row_l), q.w = get(&sm.row_w);
                }
                q = warp_run(q, p.a);
                if (lane == 0) {
                    row_results(p, r, asked, q);
                    sm.m[0] = q.m, sm.l[0] = q.l;
                }
            }
            for (int c = tid; c < C * p.top; c += T) {
                const int from = c / p.top;
                const uint32_t a =
                    mapa(static_cast<uint32_t>(__cvta_generic_to_shared(&sm.best[c - from * p.top])), (uint32_t)from);
                asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(sm.all[c]) : "r"(a) : "memory");
            }
            __syncthreads();
            const float log_l = sm.m[0] == -INFINITY ? 0.0f : logf(sm.l[0]);
            for (int c = tid; c < C * p.top; c += T) {
                const uint64_t key = sm.all[c];
                if (key == 0) continue;  // a block with fewer values
                int above = 0;
                for (int o = 0; o < C * p.top; ++o) above += sm.all[o] > key;
                if (above < p.top) top_result(p, r, above, key, sm.m[0], log_l);
            }
        }
        cluster_sync();  // the first block has read the others' shared memory
    }
    feed.end();
}

// ---- the gradient ---------------------------------------------------------------------------

struct LpBwd {
    const float *x, *stats, *entropy, *g, *h;
    Rows xm, sm, em, gm, hm;
    TokenRef tok;
    float* dx;  // may be x itself: each value is read and written by one thread
    int64_t rows;
    int V;
    float scale;
};

// A row's constants: with d = x - m,
//   p = 2^(d a - log2 l),  log p + H = d scale + (H - log l),
//   dx = p (g' + h' (log p + H)) and g scale more at the token, g' = -g scale, h' = -h scale.
// Two roundings of an exponent of size y cost y 2^-24 relative to p each.
struct RowGrad {
    float m, a, scale, log2_l, offset, g, h;
    int64_t t;
    bool none;
    __device__ __forceinline__ RowGrad(const LpBwd& p, int64_t r) {
        const float* st = p.stats + p.sm.offset(r);
        m = st[0];
        const float log_l = st[1];
        t = p.tok.get(r);
        g = p.g && t != -1 ? -p.scale * p.g[p.gm.offset(r)] : 0.0f;
        if (p.g && (t < -1 || t >= p.V)) g = __int_as_float(0x7fc00000);
        h = p.h ? -p.scale * p.h[p.hm.offset(r)] : 0.0f;
        offset = p.h ? p.entropy[p.em.offset(r)] - log_l : 0.0f;
        none = m == -INFINITY;
        scale = p.scale;
        a = p.scale * kLog2e;
        log2_l = log_l * kLog2e;
    }
    template <bool ENT>
    __device__ __forceinline__ float at(float x) const {
        const float d = x - m;
        const float pr = ex2(fmaf(d, a, -log2_l));
        if constexpr (!ENT) return pr * g;
        // where p is 0 the exponent may be -inf; p is 0 from -104 on
        return pr * fmaf(h, max_nan(fmaf(d, scale, offset), -1000.0f), g);
    }
};

// T threads take a run of at most 64 T values of one row, all of them asked for
// before the row's constants (which take as long to come) and before the first
// result is written; nobody waits for anybody.
constexpr int BWD_RUN = 64;
template <bool VEC, bool ENT, int T>
__global__ void __launch_bounds__(256) lp_bwd_kernel(LpBwd p, int pieces) {
    constexpr int BW = BWD_RUN * T;
    const int t = threadIdx.x & (T - 1);
    const int64_t unit = (int64_t)blockIdx.x * (256 / T) + threadIdx.x / T, r = unit / pieces;
    if (r >= p.rows) return;
    const int lo = (int)(unit - r * pieces) * BW, hi = min(p.V, lo + BW);
    const float* x = p.x + p.xm.offset(r);
    float* d = p.dx + r * p.V + lo;
    if constexpr (VEC) {
        const Part part(x, lo, hi);
        const float4* from = reinterpret_cast<const float4*>(part.x + part.head);
        float4* to = reinterpret_cast<float4*>(d + part.head);
        constexpr int U = BWD_RUN / 4;
        float4 f[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (t + u * T < part.vecs) f[u] = __ldcs(from + t + u * T);
        const int at = part.single(t);
        const float alone = at >= 0 ? part.x[at] : 0.0f;
        const RowGrad q(p, r);
        const int tok = q.t >= lo && q.t < hi ? (int)(q.t - lo) : -1;  // the token's place here
        if (at >= 0) d[at] = q.none ? 0.0f : q.at<ENT>(alone) - (at == tok ? q.g : 0.0f);
        const int tv = tok < part.head ? -1 : (tok - part.head) >> 2;  // the token's vector
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = t + u * T;
            if (i < part.vecs) {
                float4 y;
                y.x = q.at<ENT>(f[u].x), y.y = q.at<ENT>(f[u].y), y.z = q.at<ENT>(f[u].z), y.w = q.at<ENT>(f[u].w);
                if (i == tv) {
                    const int c = (tok - part.head) & 3;
                    if (c == 0) y.x -= q.g;
                    if (c == 1) y.y -= q.g;
                    if (c == 2) y.z -= q.g;
                    if (c == 3) y.w -= q.g;
                }
                if (q.none) y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);  // no distribution, no gradient
                __stcs(to + i, y);
            }
        }
    } else {
        const int n = hi - lo;
        constexpr int U = BWD_RUN;
        float f[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (t + u * T < n) f[u] = __ldcs(x + lo + t + u * T);
        const RowGrad q(p, r);
        const int tok = q.t >= lo && q.t < hi ? (int)(q.t - lo) : -1;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = t + u * T;
            if (j < n) __stcs(d + j, q.none ? 0.0f : q.at<ENT>(f[u]) - (j == tok ? q.g : 0.0f));
        }
    }
}

template <int T>
int launch_bwd(const LpBwd& p, bool vec, cudaStream_t s) {
    const int pieces = (p.V + BWD_RUN * T - 1) / (BWD_RUN * T);
    const int64_t blocks = (p.rows * pieces + 256 / T - 1) / (256 / T);
    if (blocks > INT32_MAX) return set_error(TLC_ERR_UNSUPPORTED, "token_logprobs_backward: too many rows");
    const unsigned grid = (unsigned)blocks;
    if (vec && p.h)
        lp_bwd_kernel<true, true, T><<<grid, 256, 0, s>>>(p, pieces);
    else if (vec)
        lp_bwd_kernel<true, false, T><<<grid, 256, 0, s>>>(p, pieces);
    else if (p.h)
        lp_bwd_kernel<false, true, T><<<grid, 256, 0, s>>>(p, pieces);
    else
        lp_bwd_kernel<false, false, T><<<grid, 256, 0, s>>>(p, pieces);
    count_launch();
    return check_launch(kBwd);
}

// 256 threads and a ring of 48 KB a block: three blocks an SM, as the registers allow (512
// threads: 188 us for 143, 128: 151; four stages: no gain).
constexpr int ROW_T = 256;
constexpr int ROW_BLOCKS = 3;
constexpr size_t kRing = sizeof(float4) * STAGES * BATCH * ROW_T;

int launch_warp(const LpFwd& p, cudaStream_t s) {
    static DeviceOnce once[2];
    TLC_TRY(smem_limit_once(once[0], lp_warp_kernel<false>, (int)kRing));
    TLC_TRY(smem_limit_once(once[1], lp_warp_kernel<true>, (int)kRing));
    const int64_t grid = std::min<int64_t>(p.rows, (int64_t)sm_count() * ROW_BLOCKS);
    if (p.top)
        lp_warp_kernel<true><<<(unsigned)grid, 256, kRing, s>>>(p);
    else
        lp_warp_kernel<false><<<(unsigned)grid, 256, kRing, s>>>(p);
    count_launch();
    return check_launch(kFwd);
}

int launch_row(const LpFwd& p, cudaStream_t s) {
    static DeviceOnce once;
    TLC_TRY(smem_limit_once(once, lp_row_kernel<ROW_T>, (int)kRing));
    const int64_t slots = (int64_t)sm_count() * ROW_BLOCKS;
    // a cluster a row while the rows alone leave more than half the slots empty, down to 4096
    // logits a block (one row of 131072: 11 us by eight blocks; with 4095 rows, two blocks a row
    // took 217 us for 143: each row then costs two cluster barriers)
    int C = 1;
    while (C < 8 && p.rows * C * 2 <= slots && p.V / (2 * C) >= 4096) C *= 2;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(std::min<int64_t>(p.rows, std::max<int64_t>(1, slots / C)) * C));
    cfg.blockDim = dim3(ROW_T);
    cfg.dynamicSmemBytes = kRing;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)C;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = C > 1 ? 1 : 0;
    TLC_CUDA_TRY(cudaLaunchKernelEx(&cfg, lp_row_kernel<ROW_T>, p, C));
    count_launch();
    return check_launch(kFwd);
}

// Above 2^127 scale * log2 e is infinite and the row's maximum gave 0 * inf; the gradient's
// constants, scale times the gradients times up to 1000, leave float32 before that.
int check_scale(float scale, const char* op) {
    if (scale > 0.0f && scale <= 0x1p100f) return TLC_OK;
    return set_error(TLC_ERR_INVALID_ARGUMENT, std::string(op) + ": scale must be positive and at most 2^100");
}

// tokens (and others) have the shape of the logits without their last dim
int same_lead(const tlc_tensor* logits, int nd, const int64_t* sizes, const char* op, const char* name) {
    bool same = nd == logits->ndim - 1;
    for (int i = 0; same && i < nd; ++i) same = sizes[i] == logits->sizes[i];
    if (same) return TLC_OK;
    return set_error(TLC_ERR_INVALID_ARGUMENT, std::string(op) + ": " + name + ": wrong shape");
}

}  // namespace
}  // namespace tlc

using namespace tlc;

extern "C" int tlc_token_logprobs(const tlc_tensor* logits, const tlc_index* tokens, float scale,
                                  tlc_tensor* logprobs, tlc_tensor* entropy, tlc_tensor* stats, int top,
                                  tlc_tensor* top_logprobs, tlc_index* top_tokens, void* stream) {
    clear_error();
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    RowView vx;
    LpFwd p{};
    int64_t n = 0, sz[TLC_MAX_DIMS];
    Extent et, eo[5];
    TLC_TRY(row_view(logits, kFwd, "logits", vx));
    TLC_TRY(check_scale(scale, kFwd));
    if (vx.cols > (1 << 30)) return set_error(TLC_ERR_UNSUPPORTED, "token_logprobs: vocabulary too large");
    const int nd = logits->ndim - 1;
    if (logprobs) {
        TLC_TRY(index_view(tokens, kFwd, "tokens", p.tok, &n, &et));
        TLC_TRY(same_lead(logits, tokens->ndim, tokens->sizes, kFwd, "tokens"));
    }
    if (top < 0 || top > vx.cols)
        return set_error(TLC_ERR_INVALID_ARGUMENT, "token_logprobs: top must be 0 to the vocabulary's size");
    if (top > kMaxTop)
        return set_error(TLC_ERR_UNSUPPORTED, "token_logprobs: top is at most " + std::to_string(kMaxTop));
    if (vx.rows > 0 && vx.cols == 0)
        return set_error(TLC_ERR_INVALID_ARGUMENT, "token_logprobs: rows without logits");
    const char* names[5] = {"logprobs", "entropy", "stats", "top_logprobs", "top_tokens"};
    if (logprobs) TLC_TRY(shaped(logprobs, kFwd, names[0], nd, logits->sizes, true, &eo[0]));
    if (entropy) TLC_TRY(shaped(entropy, kFwd, names[1], nd, logits->sizes, true, &eo[1]));
    std::copy(logits->sizes, logits->sizes + nd, sz);
    sz[nd] = 2;
    if (stats) TLC_TRY(shaped(stats, kFwd, names[2], nd + 1, sz, true, &eo[2]));
    if (top) {
        sz[nd] = top;
        TLC_TRY(shaped(top_logprobs, kFwd, names[3], nd + 1, sz, true, &eo[3]));
        TokenRef ref;
        int64_t cnt;
        TLC_TRY(index_view(top_tokens, kFwd, names[4], ref, &cnt, &eo[4]));
        bool same = top_tokens->ndim == nd + 1;
        for (int i = 0; same && i <= nd; ++i) same = top_tokens->sizes[i] == sz[i];
        if (!same) return set_error(TLC_ERR_INVALID_ARGUMENT, "token_logprobs: top_tokens: wrong shape");
        if (!dense_strides(nd + 1, top_tokens->sizes, top_tokens->strides))
            return set_error(TLC_ERR_INVALID_ARGUMENT, "token_logprobs: top_tokens must be contiguous");
    }
    for (int i = 0; i < 5; ++i) {
        TLC_TRY(no_overlap(kFwd, names[i], eo[i], "logits", vx.ext));
        TLC_TRY(no_overlap(kFwd, names[i], eo[i], "tokens", et));
        for (int j = 0; j < i; ++j) TLC_TRY(no_overlap(kFwd, names[i], eo[i], names[j], eo[j]));
    }
    if (vx.rows == 0) return TLC_OK;
    RowScratch cx(s);
    TLC_TRY(unit_rows(logits, vx, cx));
    p.x = vx.data;
    p.xm = vx.map;
    p.rows = vx.rows;
    p.V = (int)vx.cols;
    p.scale = scale;
    p.a = scale * kLog2e;
    p.logp = logprobs ? logprobs->data : nullptr;
    p.entropy = entropy ? entropy->data : nullptr;
    p.stats = stats ? stats->data : nullptr;
    p.top = top;
    if (top) {
        p.top_logp = top_logprobs->data;
        p.top_tok = top_tokens->data;
        p.top_wide = top_tokens->bits == 64;
    }
    // a warp a row where a block's finish would cost more than its reading (8192 x 2001: 17 us by
    // warps, 48 by blocks) and the rows keep every SM's warps busy
    if (p.V <= 1024 || (p.V <= 16384 && p.rows >= (int64_t)sm_count() * 8)) return launch_warp(p, s);
    return launch_row(p, s);
}

extern "C" int tlc_token_logprobs_backward(const tlc_tensor* logits, const tlc_index* tokens,
                                           const tlc_tensor* stats, const tlc_tensor* entropy,
                                           const tlc_tensor* grad_logprobs, const tlc_tensor* grad_entropy,
                                           float scale, tlc_tensor* dlogits, void* stream) {
    clear_error();
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    RowView vx, vs;
    LpBwd p{};
    int64_t n = 0, sz[TLC_MAX_DIMS];
    Extent et, es, ee, eg, eh, ed;
    TLC_TRY(row_view(logits, kBwd, "logits", vx));
    TLC_TRY(check_scale(scale, kBwd));
    if (vx.cols > (1 << 30)) return set_error(TLC_ERR_UNSUPPORTED, "token_logprobs_backward: vocabulary too large");
    const int nd = logits->ndim - 1;
    TLC_TRY(index_view(tokens, kBwd, "tokens", p.tok, &n, &et));
    TLC_TRY(same_lead(logits, tokens->ndim, tokens->sizes, kBwd, "tokens"));
    std::copy(logits->sizes, logits->sizes + nd, sz);
    sz[nd] = 2;
    TLC_TRY(shaped(stats, kBwd, "stats", nd + 1, sz, false, &es));
    TLC_TRY(row_view(stats, kBwd, "stats", vs));
    if (grad_logprobs) {
        TLC_TRY(shaped(grad_logprobs, kBwd, "grad_logprobs", nd, logits->sizes, false, &eg));
        p.g = grad_logprobs->data;
        p.gm = merge_rows(nd, grad_logprobs->sizes, grad_logprobs->strides);
    }
    if (grad_entropy) {
        TLC_TRY(shaped(grad_entropy, kBwd, "grad_entropy", nd, logits->sizes, false, &eh));
        TLC_TRY(shaped(entropy, kBwd, "entropy", nd, logits->sizes, false, &ee));
        p.h = grad_entropy->data;
        p.hm = merge_rows(nd, grad_entropy->sizes, grad_entropy->strides);
        p.entropy = entropy->data;
        p.em = merge_rows(nd, entropy->sizes, entropy->strides);
    }
    TLC_TRY(shaped(dlogits, kBwd, "dlogits", logits->ndim, logits->sizes, true, &ed));
    const bool in_place = dlogits->data == logits->data && dense_strides(logits->ndim, logits->sizes, logits->strides);
    if (!in_place) TLC_TRY(no_overlap(kBwd, "dlogits", ed, "logits", vx.ext));
    TLC_TRY(no_overlap(kBwd, "dlogits", ed, "tokens", et));
    TLC_TRY(no_overlap(kBwd, "dlogits", ed, "stats", es));
    TLC_TRY(no_overlap(kBwd, "dlogits", ed, "entropy", ee));
    TLC_TRY(no_overlap(kBwd, "dlogits", ed, "grad_logprobs", eg));
    TLC_TRY(no_overlap(kBwd, "dlogits", ed, "grad_entropy", eh));
    if (vx.numel == 0) return TLC_OK;
    RowScratch cx(s), cs(s);
    TLC_TRY(unit_rows(logits, vx, cx));
    TLC_TRY(unit_rows(stats, vs, cs));
    p.x = vx.data;
    p.xm = vx.map;
    p.stats = vs.data;
    p.sm = vs.map;
    p.dx = dlogits->data;
    p.rows = vx.rows;
    p.V = (int)vx.cols;
    p.scale = scale;
    // float4 where each row of x and dx starts at the same place within 16 bytes
    const bool vec = (reinterpret_cast<uintptr_t>(p.x) - reinterpret_cast<uintptr_t>(p.dx)) % 16 == 0 &&
                     (p.rows == 1 || (p.xm.nd == 1 && (p.xm.st[0] - p.V) % 4 == 0) ||
                      (p.V % 4 == 0 && p.xm.multiple_of(4)));
    // a block a run of a long row (4096 x 50001: 265 us, 296 by warps), a warp a run of a
    // short one (8192 x 999: 17 us, 46 by blocks)
    return p.V > 8192 ? launch_bwd<256>(p, vec, s) : launch_bwd<32>(p, vec, s);
}
