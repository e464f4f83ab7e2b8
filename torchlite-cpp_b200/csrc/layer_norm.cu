// Layer norm over the last dim of [..., D] and its gradients, fp32.
//
//   mean = sum_D x / D,  var = sum_D (x - mean)^2 / D,  rstd = 1 / sqrt(var + eps)
//   xhat = (x - mean) rstd,  y = xhat w + b
//   dx = rstd (gw - (sum_D gw + xhat sum_D gw xhat) / D)   with gw = g w
//   dw = sum_rows g xhat,  db = sum_rows g
//
// Bound by HBM: the forward moves 8 bytes an element (x in, y out), the
// backward 12 (x and g in, dx out).  So a row is read once, into registers,
// and both statistics come from there: a first mean, then the sums of the
// differences to it and of their squares.  A sum of D values is off by some
// roundings of its size, which a row whose mean is many times its spread would
// feel in every result (of a row of 1000.1 alone xhat was 0.06), so the
// differences' own mean is taken off them and off the variance.
// Measured (GPU time): forward 8192 x 768 10.4 us (4.8 TB/s), 4096 x 16384
// 88 us (6.1 TB/s), unaligned 4099 x 5001 34.8 us (4.7 TB/s); backward 8192 x
// 768 19.8 us (3.8 TB/s), 8192 x 8192 144 us (5.6 TB/s), unaligned 16000 x 1001
// 43 us (4.5 TB/s).
#include <algorithm>
#include <cmath>

#include "rows.cuh"

namespace tlc {
namespace {

// What a first mean lacks, and 1 / sqrt(var + eps), from the sums of the differences to it and of
// their squares; xhat of a difference d is d * rstd + shift.
struct Spread {
    float off, rstd, shift;
    __device__ __forceinline__ Spread(const float (&s)[2], int D, float eps) {
        off = __fdiv_rn(s[0], (float)D);
        const float var = fmaf(-off, off, __fdiv_rn(s[1], (float)D));
        rstd = __frsqrt_rn((var < 0.0f ? 0.0f : var) + eps);  // a NaN stays one
        shift = -off * rstd;
    }
    // the corrected mean; an infinite one, whose differences are infinite too, stays
    __device__ __forceinline__ float mean(float first) const {
        const float m = first + off;
        return m == m ? m : first;
    }
};

struct LnFwd {
    const float *x, *w, *b;
    float *out, *stats;
    Rows xm;
    int64_t rows;
    int D;
    float eps;
};

// THREADS threads a row (a block, or up to 32 neighbouring lanes of 4 warps), VPT
// vectors of VEC floats a thread: D <= THREADS * VPT * VEC.  Blocks that share a row
// have 64 registers a thread, so that 1024 threads are on an SM; the lane groups, whose
// blocks hold several rows, are not bounded (62 to 85).
template <int VEC, int VPT, int THREADS>
__global__ void __launch_bounds__(THREADS <= 32 ? 128 : THREADS, THREADS <= 32 ? 1 : 1024 / THREADS)
    ln_fwd_kernel(LnFwd p) {
    constexpr int RPB = THREADS <= 32 ? 128 / THREADS : 1;
    constexpr bool FEW = VEC * VPT < 32;  // 32 values spill with it (4096 x 16384: 90.6 us for 87.8)
    __shared__ float red[32], red2[64];
    const int t = threadIdx.x % THREADS, sub = threadIdx.x / THREADS;
    const int n = p.D / VEC;
    const int whole = n / THREADS + (t < n % THREADS ? 1 : 0);  // this thread's vectors of a row
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < p.rows; r0 += (int64_t)gridDim.x * RPB) {
        const int64_t r = r0 + sub;
        const bool live = RPB == 1 || r < p.rows;  // lanes without a row take part in the sums
        const int mine = live ? whole : 0;
        const float* xr = p.x + (live ? p.xm.offset(r) : 0) + t * VEC;
        float v[VPT][VEC];
#pragma unroll
        for (int i = 0; i < VPT; ++i)
            if (i < mine) load_once<VEC>(xr + i * THREADS * VEC, v[i]);
        float s[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < VPT; ++i)
            if (i < mine)
#pragma unroll
                for (int k = 0; k < VEC; ++k) s[0] += v[i][k];
        group_sum<THREADS, FEW>(s, red);
        const float mean = __fdiv_rn(s[0], (float)p.D);
        float d[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < VPT; ++i)
            if (i < mine)
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    v[i][k] -= mean;
                    d[0] += v[i][k];
                    d[1] = fmaf(v[i][k], v[i][k], d[1]);
                }
        group_sum<THREADS, FEW>(d, red2);
        const Spread sp(d, p.D, p.eps);
        if (p.stats && t == 0 && live) {
            p.stats[2 * r] = sp.mean(mean);
            p.stats[2 * r + 1] = sp.rstd;
        }
        float* yr = p.out + r * p.D + t * VEC;
        const float* w = p.w + t * VEC;
        const float* b = p.b + t * VEC;
        if (p.w && p.b) {
#pragma unroll
            for (int i = 0; i < VPT; ++i)
                if (i < mine) {
                    float wv[VEC], bv[VEC];
                    load_vec<VEC>(w + i * THREADS * VEC, wv);
                    load_vec<VEC>(b + i * THREADS * VEC, bv);
#pragma unroll
                    for (int k = 0; k < VEC; ++k) v[i][k] = fmaf(fmaf(v[i][k], sp.rstd, sp.shift), wv[k], bv[k]);
                    store_once<VEC>(yr + i * THREADS * VEC, v[i]);
                }
        } else {
#pragma unroll
            for (int i = 0; i < VPT; ++i)
                if (i < mine) {
#pragma unroll
                    for (int k = 0; k < VEC; ++k) {
                        v[i][k] = fmaf(v[i][k], sp.rstd, sp.shift);
                        if (p.w) v[i][k] *= w[i * THREADS * VEC + k];
                        if (p.b) v[i][k] += b[i * THREADS * VEC + k];
                    }
                    store_once<VEC>(yr + i * THREADS * VEC, v[i]);
                }
        }
    }
}

// Rows too long for the registers of a block (above 32768 columns, 16384
// unaligned): the row is read three times (from L2 after the first).  Two blocks
// an SM read while one another's sums meet (4096 x 40000 445 us, one block 482).
__global__ void __launch_bounds__(1024, 2) ln_fwd_long_kernel(LnFwd p) {
    __shared__ float red[32], red2[64];
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const float* xr = p.x + p.xm.offset(r);
        float s[1] = {0.0f};
        for (int64_t j = threadIdx.x; j < p.D; j += 1024) s[0] += xr[j];
        group_sum<1024>(s, red);
        const float mean = __fdiv_rn(s[0], (float)p.D);
        float d[2] = {0.0f, 0.0f};
        for (int64_t j = threadIdx.x; j < p.D; j += 1024) {
            const float v = xr[j] - mean;
            d[0] += v;
            d[1] = fmaf(v, v, d[1]);
        }
        group_sum<1024>(d, red2);
        const Spread sp(d, p.D, p.eps);
        float* yr = p.out + r * p.D;
        for (int64_t j = threadIdx.x; j < p.D; j += 1024) {
            float y = fmaf(xr[j] - mean, sp.rstd, sp.shift);
            if (p.w) y *= p.w[j];
            if (p.b) y += p.b[j];
            yr[j] = y;
        }
        if (p.stats && threadIdx.x == 0) {
            p.stats[2 * r] = sp.mean(mean);
            p.stats[2 * r + 1] = sp.rstd;
        }
    }
}

struct LnBwd {
    const float *g, *x, *w, *stats;
    float *dx, *part;  // part: [gridDim.x][2][D], the blocks' sums for dw and db, or NULL
    Rows gm, xm, sm;   // sm: the rows of stats
    int64_t rows;
    int D;
    int accumulate;
};

__device__ __forceinline__ void copy16(float* dst, const float* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
                 "l"(src)
                 : "memory");
}
__device__ __forceinline__ void copy4(float* dst, const float* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
                 "l"(src)
                 : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// One block an SM, 16 warps; THREADS threads a row (8 lanes to the whole block),
// 512 / THREADS rows at a time.  Each thread keeps the same columns for every
// row, so the sums for dw and db stay in its registers until the end; up to 16
// columns a thread, two an instruction (with 8 warps of 32 columns the loop's
// code was fetched more slowly than it ran: half of all stalls), and 24 or 32,
// with spills, only for rows that a block could not hold otherwise.
//
// The rows come through a ring of rows of x and g in shared memory, filled by
// asynchronous copies, so that rows far enough ahead are always in flight
// although the registers allow only 16 warps.  Where all rows start on 16 bytes
// (VEC 4) a thread copies just what it reads itself, which needs no barrier.
// Otherwise (VEC 1) the row's threads copy its aligned 16-byte pieces together,
// single values at its ends, and meet before they read and before they refill.
constexpr int BT = 512;

template <int VEC, int VPT, int THREADS>
struct LnRing {
    static constexpr int ROW = THREADS * VPT * VEC + (VEC == 1 ? 8 : 0);  // floats a row
    static constexpr int SLOT = 2 * (BT / THREADS) * ROW;                 // x and g of the rows at a time
    static constexpr int FIT = 200 * 1024 / (SLOT * 4);
    static constexpr int STAGES = FIT < 8 ? FIT : 8;
    static constexpr int BYTES = STAGES * SLOT * 4;
};

// The VPT * VEC values of a thread as pairs: value q is (vector q / VEC, element q % VEC).
template <int VEC, int VPT, int THREADS>
__global__ void __launch_bounds__(BT, 1) ln_bwd_kernel(LnBwd p) {
    using R = LnRing<VEC, VPT, THREADS>;
    constexpr int S = R::STAGES, GROUPS = BT / THREADS, W = THREADS > 32 ? THREADS / 32 : 1, N = VEC * VPT;
    extern __shared__ __align__(16) float ring[];  // [S][GROUPS][2][ROW], then [GROUPS][2][D]
    __shared__ float red[2][GROUPS][2 * W];
    const int group = threadIdx.x / THREADS, t = threadIdx.x % THREADS, lane = threadIdx.x & 31;
    const float inv = 1.0f / (float)p.D;
    next_may_launch();
    const int vecs = p.D / VEC;
    const int whole = vecs / THREADS + (t < vecs % THREADS ? 1 : 0);  // this thread's vectors of a row
    Pair aw[N / 2], ab[N / 2], w[N / 2];
    auto load_w = [&]() {
        float one[VPT][VEC];
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            if (p.w && i < whole) load_vec<VEC>(p.w + (t + i * THREADS) * VEC, one[i]);
#pragma unroll
            for (int k = 0; k < VEC; ++k)
                if (!p.w || i >= whole) one[i][k] = 1.0f;
        }
#pragma unroll
        for (int q = 0; q < N / 2; ++q)
            w[q] = pair(one[2 * q / VEC][2 * q % VEC], one[(2 * q + 1) / VEC][(2 * q + 1) % VEC]);
    };
    constexpr bool KEEP_W = N <= 16;  // else the registers have no room for it
    if (KEEP_W) load_w();
#pragma unroll
    for (int q = 0; q < N / 2; ++q) aw[q] = ab[q] = 0;
    // Rows go to the blocks first, then to a block's warps; the lane groups of a warp take
    // neighbouring rows and run out together.
    constexpr int PER_WARP = THREADS < 32 ? 32 / THREADS : 1;
    const int unit = group / PER_WARP, sub = group % PER_WARP;
    const int64_t blocks = gridDim.x, step = blocks * GROUPS;
    const int64_t u0 = (blockIdx.x + blocks * unit) * PER_WARP;  // first row of the warp (or group)
    auto slot = [&](int stage, int which) { return ring + ((stage * GROUPS + group) * 2 + which) * R::ROW; };
    auto fetch_row = [&](const float* from, float* to) {
        if constexpr (VEC == 4) {
#pragma unroll
            for (int i = 0; i < VPT; ++i) {
                const int j = (t + i * THREADS) * 4;
                if (i < whole) copy16(to + j, from + j);
            }
        } else {
            const int phase = (int)(reinterpret_cast<uintptr_t>(from) >> 2) & 3;
            const int pieces = (phase + p.D + 3) >> 2;
#pragma unroll
            for (int i = 0; i <= (VPT + 3) / 4; ++i) {
                const int q = t + i * THREADS, j = 4 * q - phase;
                if (j >= 0 && j + 4 <= p.D) copy16(to + 4 * q, from + j);
            }
            // the ends, a value a thread: before the first whole piece and behind the last
            if (phase && t < 4 - phase && t < p.D) copy4(to + phase + t, from + t);
            const int last = 4 * (pieces - 1) - phase;  // begin of the last piece
            if (last + 4 > p.D && (last > 0 || !phase) && last + t < p.D && t < 4) copy4(to + phase + last + t, from + last + t);
        }
    };
    auto fetch = [&](int64_t r, int stage) {
        if (r < p.rows) {
            fetch_row(p.x + p.xm.offset(r), slot(stage, 0));
            fetch_row(p.g + p.gm.offset(r), slot(stage, 1));
        }
        copies_commit();
    };
    // where the row's values are within their slot
    auto placed = [&](const float* from, float* at) {
        return VEC == 4 ? at : at + ((reinterpret_cast<uintptr_t>(from) >> 2) & 3);
    };
    auto meet = [&]() {
        if constexpr (THREADS <= 32)
            __syncwarp();
        else
            asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(THREADS) : "memory");
    };
#pragma unroll
    for (int s = 0; s < S; ++s) fetch(u0 + s * step + sub, s);
    int stage = 0, turn = 0;
    float next[2] = {0.0f, 0.0f};
    auto fetch_stats = [&](int64_t r) {
        if (r < p.rows) {
            const float* st = p.stats + p.sm.offset(r);
            next[0] = st[0], next[1] = st[1];
        }
    };
    fetch_stats(u0 + sub);
    for (int64_t u = u0; u < p.rows; u += step) {
        const int64_t r = u + sub;
        const bool live = PER_WARP == 1 || r < p.rows;
        const int mine = live ? whole : 0;
        const float mean = next[0], rstd = next[1];
        fetch_stats(r + step);
        copies_wait<S - 1>();
        if constexpr (VEC == 1) meet();
        Pair x[N / 2], g[N / 2];
        {
            const float* xs = placed(p.x + (live ? p.xm.offset(r) : 0), slot(stage, 0)) + t * VEC;
            const float* gs = placed(p.g + (live ? p.gm.offset(r) : 0), slot(stage, 1)) + t * VEC;
            float xv[VPT][VEC], gv[VPT][VEC];
#pragma unroll
            for (int i = 0; i < VPT; ++i) {
                if (i < mine) {
                    load_vec<VEC>(xs + i * THREADS * VEC, xv[i]);
                    load_vec<VEC>(gs + i * THREADS * VEC, gv[i]);
                } else {  // adds nothing
#pragma unroll
                    for (int k = 0; k < VEC; ++k) xv[i][k] = mean, gv[i][k] = 0.0f;
                }
            }
#pragma unroll
            for (int q = 0; q < N / 2; ++q) {
                x[q] = pair(xv[2 * q / VEC][2 * q % VEC], xv[(2 * q + 1) / VEC][(2 * q + 1) % VEC]);
                g[q] = pair(gv[2 * q / VEC][2 * q % VEC], gv[(2 * q + 1) / VEC][(2 * q + 1) % VEC]);
            }
        }
        if (!KEEP_W) load_w();
        const Pair shift = pair(-mean, -mean), scale = pair(rstd, rstd);
        Pair s0 = 0, s1 = 0;
#pragma unroll
        for (int q = 0; q < N / 2; ++q) {
            x[q] = mul2(add2(x[q], shift), scale);
            aw[q] = fma2(g[q], x[q], aw[q]);
            ab[q] = add2(ab[q], g[q]);
            g[q] = mul2(g[q], w[q]);
            s0 = add2(s0, g[q]);
            s1 = fma2(g[q], x[q], s1);
        }
        if constexpr (VEC == 1) meet();
        fetch(r + S * step, stage);  // into the row just read
        stage = stage + 1 == S ? 0 : stage + 1;
        if (!p.dx) continue;
        float s[2], other[2];
        unpair(s0, s[0], other[0]);
        unpair(s1, s[1], other[1]);
        s[0] += other[0], s[1] += other[1];
        warp_sum<(THREADS < 32 ? THREADS : 32)>(s);
        if constexpr (W > 1) {
            float* sums = red[turn][group];
            if (lane == 0) sums[2 * (t >> 5)] = s[0], sums[2 * (t >> 5) + 1] = s[1];
            meet();
            s[0] = s[1] = 0.0f;
#pragma unroll
            for (int q = 0; q < W; ++q) s[0] += sums[2 * q], s[1] += sums[2 * q + 1];
            turn ^= 1;
        }
        s[0] *= -inv, s[1] *= -inv;
        const Pair c0 = pair(s[0], s[0]), c1 = pair(s[1], s[1]);
        float* dr = p.dx + r * p.D + t * VEC;
#pragma unroll
        for (int q = 0; q < N / 2; ++q) x[q] = mul2(scale, add2(g[q], fma2(x[q], c1, c0)));
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            if (i < mine) {
                float y[VEC], old[VEC];
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    float lo, hi;
                    unpair(x[(i * VEC + k) / 2], lo, hi);
                    y[k] = (i * VEC + k) % 2 ? hi : lo;
                }
                if (p.accumulate) {
                    load_vec<VEC>(dr + i * THREADS * VEC, old);
#pragma unroll
                    for (int k = 0; k < VEC; ++k) y[k] = __fadd_rn(y[k], old[k]);  // the gradient rounded, then added
                }
                store_once<VEC>(dr + i * THREADS * VEC, y);
            }
        }
    }
    copies_wait<0>();
    if (!p.part) return;
    float* part = p.part + (int64_t)blockIdx.x * 2 * p.D;
    float* sums = GROUPS > 1 ? ring + (int64_t)group * 2 * p.D : part;
    __syncthreads();  // nobody reads the ring any more
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int j = (t + i * THREADS) * VEC;
        if (i < whole) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                float lo, hi;
                unpair(aw[(i * VEC + k) / 2], lo, hi);
                sums[j + k] = (i * VEC + k) % 2 ? hi : lo;
                unpair(ab[(i * VEC + k) / 2], lo, hi);
                sums[p.D + j + k] = (i * VEC + k) % 2 ? hi : lo;
            }
        }
    }
    if constexpr (GROUPS > 1) {
        __syncthreads();
        for (int j = threadIdx.x; j < 2 * p.D; j += BT) {
            float a = 0.0f;
#pragma unroll 8
            for (int q = 0; q < GROUPS; ++q) a += ring[q * 2 * p.D + j];
            part[j] = a;
        }
    }
}

// Rows too long for that (above 16384 columns): dx alone, the row read twice ...
__global__ void __launch_bounds__(1024) ln_bwd_long_kernel(LnBwd p) {
    __shared__ float red[2][64];
    const float inv = 1.0f / (float)p.D;
    int turn = 0;
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const float* xr = p.x + p.xm.offset(r);
        const float* gr = p.g + p.gm.offset(r);
        const float* st = p.stats + p.sm.offset(r);
        const float mean = st[0], rstd = st[1];
        float s[2] = {0.0f, 0.0f};
        for (int64_t j = threadIdx.x; j < p.D; j += 1024) {
            const float gw = p.w ? gr[j] * p.w[j] : gr[j];
            s[0] += gw;
            s[1] = fmaf(gw, (xr[j] - mean) * rstd, s[1]);
        }
        group_sum<1024>(s, red[turn]);
        turn ^= 1;
        const float c0 = s[0] * inv, c1 = s[1] * inv;
        float* dr = p.dx + r * p.D;
        for (int64_t j = threadIdx.x; j < p.D; j += 1024) {
            const float gw = p.w ? gr[j] * p.w[j] : gr[j];
            float y = __fmul_rn(rstd, gw - fmaf((xr[j] - mean) * rstd, c1, c0));
            if (p.accumulate) y = __fadd_rn(y, dr[j]);
            dr[j] = y;
        }
    }
}

// ... and the columns' sums over a run of rows for each block row.
__global__ void __launch_bounds__(256) ln_bwd_cols_kernel(LnBwd p, int64_t rows_per) {
    const int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (j >= p.D) return;
    const int64_t r0 = blockIdx.y * rows_per, r1 = min(p.rows, r0 + rows_per);
    float a = 0.0f, b = 0.0f;
    for (int64_t r = r0; r < r1; ++r) {
        const float* st = p.stats + p.sm.offset(r);
        const float g = p.g[p.gm.offset(r) + j];
        a = fmaf(g, (p.x[p.xm.offset(r) + j] - st[0]) * st[1], a);
        b += g;
    }
    float* part = p.part + (int64_t)blockIdx.y * 2 * p.D;
    part[j] = a;
    part[p.D + j] = b;
}

// dw = sum of the blocks' sums in their order: 32 columns a block, 16 warps
// over the parts.  Columns [0, D) are dw's, [D, 2D) db's.  `part` is still being
// written when this kernel's blocks are set up: not __restrict__.
__global__ void __launch_bounds__(512)
    ln_bwd_finish_kernel(const float* part, int parts, int D, float* dw, float* db, int accumulate) {
    __shared__ float red[16][33];
    after_previous();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t j = (int64_t)blockIdx.x * 32 + lane;
    float a = 0.0f;
    if (j < 2 * (int64_t)D)
#pragma unroll 5
        for (int q = warp; q < parts; q += 16) a += part[(int64_t)q * 2 * D + j];
    red[warp][lane] = a;
    __syncthreads();
    if (warp == 0 && j < 2 * (int64_t)D) {
        a = 0.0f;
#pragma unroll
        for (int q = 0; q < 16; ++q) a += red[q][lane];
        float* out = j < D ? (dw ? dw + j : nullptr) : (db ? db + (j - D) : nullptr);
        if (out) *out = accumulate ? *out + a : a;
    }
}

constexpr const char* kFwd = "layer_norm";
constexpr const char* kBwd = "layer_norm_backward";

template <int VEC, int VPT, int THREADS>
int launch_fwd(const LnFwd& p, cudaStream_t s) {
    constexpr int RPB = THREADS <= 32 ? 128 / THREADS : 1;
    const int64_t want = (p.rows + RPB - 1) / RPB;
    const unsigned grid = (unsigned)std::min<int64_t>(want, INT32_MAX);
    ln_fwd_kernel<VEC, VPT, THREADS><<<grid, THREADS <= 32 ? 128 : THREADS, 0, s>>>(p);
    count_launch();
    return check_launch(kFwd);
}

// 16 to 32 values a thread: many small blocks keep more rows in flight than few large ones
// (4099 x 5001: 35 us by 256 threads, 46 by 512, 75 by 1024) and than rings of copies ahead
// (8192 x 768: 10.6 us, 14 through a ring).
template <int VEC>
int pick_fwd(const LnFwd& p, cudaStream_t s) {
    const int n = (p.D + VEC - 1) / VEC;  // vectors a row
    if (p.D <= 128) return launch_fwd<VEC, 16 / VEC, 8>(p, s);
    if (p.D <= 256) return launch_fwd<VEC, 16 / VEC, 16>(p, s);
    if (p.D <= 512) return launch_fwd<VEC, 16 / VEC, 32>(p, s);
    if (p.D <= 768) return launch_fwd<VEC, 24 / VEC, 32>(p, s);
    if (p.D <= 1024) return launch_fwd<VEC, 32 / VEC, 32>(p, s);
    if constexpr (VEC == 4) {
        if (n <= 128 * 4) return launch_fwd<4, 4, 128>(p, s);
        if (n <= 256 * 4) return launch_fwd<4, 4, 256>(p, s);
        if (n <= 256 * 8) return launch_fwd<4, 8, 256>(p, s);
        if (n <= 512 * 8) return launch_fwd<4, 8, 512>(p, s);
        if (n <= 1024 * 8) return launch_fwd<4, 8, 1024>(p, s);
    } else {
        if (n <= 128 * 16) return launch_fwd<1, 16, 128>(p, s);
        if (n <= 256 * 16) return launch_fwd<1, 16, 256>(p, s);
        if (n <= 256 * 24) return launch_fwd<1, 24, 256>(p, s);
        if (n <= 512 * 16) return launch_fwd<1, 16, 512>(p, s);
        if (n <= 512 * 24) return launch_fwd<1, 24, 512>(p, s);
        if (n <= 1024 * 16) return launch_fwd<1, 16, 1024>(p, s);
    }
    ln_fwd_long_kernel<<<(unsigned)std::min<int64_t>(p.rows, INT32_MAX), 1024, 0, s>>>(p);
    count_launch();
    return check_launch(kFwd);
}

constexpr int kRingMax = 16384;  // 32 columns a thread

template <int VEC, int VPT, int THREADS>
int launch_bwd(const LnBwd& p, int blocks, cudaStream_t s) {
    using R = LnRing<VEC, VPT, THREADS>;
    static DeviceOnce once;
    TLC_TRY(smem_limit_once(once, ln_bwd_kernel<VEC, VPT, THREADS>, R::BYTES));
    ln_bwd_kernel<VEC, VPT, THREADS><<<blocks, BT, R::BYTES, s>>>(p);
    count_launch();
    return check_launch(kBwd);
}

// 8 lanes a row up to 128 columns, the whole block from 4097 on.
template <int VEC>
int pick_bwd(const LnBwd& p, int blocks, cudaStream_t s) {
    if (p.D <= 128) return launch_bwd<VEC, 16 / VEC, 8>(p, blocks, s);
    if (p.D <= 256) return launch_bwd<VEC, 16 / VEC, 16>(p, blocks, s);
    if (p.D <= 512) return launch_bwd<VEC, 16 / VEC, 32>(p, blocks, s);
    if (p.D <= 768) return launch_bwd<VEC, 12 / VEC, 64>(p, blocks, s);
    if (p.D <= 1024) return launch_bwd<VEC, 16 / VEC, 64>(p, blocks, s);
    if (p.D <= 1536) return launch_bwd<VEC, 12 / VEC, 128>(p, blocks, s);
    if (p.D <= 2048) return launch_bwd<VEC, 16 / VEC, 128>(p, blocks, s);
    if (p.D <= 4096) return launch_bwd<VEC, 16 / VEC, 256>(p, blocks, s);
    if (p.D <= 6144) return launch_bwd<VEC, 12 / VEC, 512>(p, blocks, s);
    if (p.D <= 8192) return launch_bwd<VEC, 16 / VEC, 512>(p, blocks, s);
    if (p.D <= 12288) return launch_bwd<VEC, 24 / VEC, 512>(p, blocks, s);
    return launch_bwd<VEC, 32 / VEC, 512>(p, blocks, s);
}

// A weight or bias: NULL, or a 1-D tensor of length D with stride 1 (a copy in `sc` otherwise).
int column_vector(const tlc_tensor* t, const char* op, const char* name, int64_t D, RowScratch& sc, const float** out,
                  Extent* ext) {
    *out = nullptr;
    if (!t) return TLC_OK;
    TLC_TRY(shaped(t, op, name, 1, &D, false, ext));
    RowView v;
    TLC_TRY(row_view(t, op, name, v));
    TLC_TRY(unit_rows(t, v, sc));
    *out = v.data;
    return TLC_OK;
}

}  // namespace
}  // namespace tlc

using namespace tlc;

extern "C" int tlc_layer_norm(const tlc_tensor* x, const tlc_tensor* weight, const tlc_tensor* bias, float eps,
                              tlc_tensor* out, tlc_tensor* stats, void* stream) {
    clear_error();
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    RowView vx;
    TLC_TRY(row_view(x, kFwd, "x", vx));
    if (!(eps >= 0.0f) || std::isinf(eps))
        return set_error(TLC_ERR_INVALID_ARGUMENT, "layer_norm: eps must be finite and not negative");
    if (vx.cols > INT32_MAX / 4) return set_error(TLC_ERR_UNSUPPORTED, "layer_norm: last dim too large");
    Extent eo, es, ew, eb;
    TLC_TRY(shaped(out, kFwd, "out", x->ndim, x->sizes, true, &eo));
    TLC_TRY(no_overlap(kFwd, "out", eo, "x", vx.ext));
    if (stats) {
        int64_t sz[TLC_MAX_DIMS];
        std::copy(x->sizes, x->sizes + x->ndim, sz);
        sz[x->ndim - 1] = 2;
        TLC_TRY(shaped(stats, kFwd, "stats", x->ndim, sz, true, &es));
        TLC_TRY(no_overlap(kFwd, "stats", es, "x", vx.ext));
        TLC_TRY(no_overlap(kFwd, "stats", es, "out", eo));
    }
    if (weight) {
        TLC_TRY(shaped(weight, kFwd, "weight", 1, &vx.cols, false, &ew));
        TLC_TRY(no_overlap(kFwd, "out", eo, "weight", ew));
        TLC_TRY(no_overlap(kFwd, "stats", es, "weight", ew));
    }
    if (bias) {
        TLC_TRY(shaped(bias, kFwd, "bias", 1, &vx.cols, false, &eb));
        TLC_TRY(no_overlap(kFwd, "out", eo, "bias", eb));
        TLC_TRY(no_overlap(kFwd, "stats", es, "bias", eb));
    }
    if (vx.cols == 0 && vx.rows > 0 && stats)
        return set_error(TLC_ERR_INVALID_ARGUMENT, "layer_norm: no statistics of rows without elements");
    if (vx.numel == 0) return TLC_OK;
    RowScratch cx(s), cw(s), cb(s);
    TLC_TRY(unit_rows(x, vx, cx));
    LnFwd p{};
    TLC_TRY(column_vector(weight, kFwd, "weight", vx.cols, cw, &p.w, &ew));
    TLC_TRY(column_vector(bias, kFwd, "bias", vx.cols, cb, &p.b, &eb));
    p.x = vx.data;
    p.xm = vx.map;
    p.out = out->data;
    p.stats = stats ? stats->data : nullptr;
    p.rows = vx.rows;
    p.D = (int)vx.cols;
    p.eps = eps;
    // float4 where every row of x, out, weight and bias starts on 16 bytes
    const bool vec = p.D % 4 == 0 && vx.map.multiple_of(4) && aligned_to(p.x, 16) && aligned_to(p.out, 16) &&
                     aligned_to(p.w, 16) && aligned_to(p.b, 16);
    return vec ? pick_fwd<4>(p, s) : pick_fwd<1>(p, s);
}

extern "C" int tlc_layer_norm_backward(const tlc_tensor* grad, const tlc_tensor* x, const tlc_tensor* stats,
                                       const tlc_tensor* weight, tlc_tensor* dx, tlc_tensor* dweight,
                                       tlc_tensor* dbias, int accumulate, void* stream) {
    clear_error();
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    RowView vx, vg, vs;
    TLC_TRY(row_view(x, kBwd, "x", vx));
    if (vx.cols > INT32_MAX / 4) return set_error(TLC_ERR_UNSUPPORTED, "layer_norm_backward: last dim too large");
    Extent eg, est, ew;
    TLC_TRY(shaped(grad, kBwd, "grad", x->ndim, x->sizes, false, &eg));
    TLC_TRY(row_view(grad, kBwd, "grad", vg));
    int64_t sz[TLC_MAX_DIMS];
    std::copy(x->sizes, x->sizes + x->ndim, sz);
    sz[x->ndim - 1] = 2;
    TLC_TRY(shaped(stats, kBwd, "stats", x->ndim, sz, false, &est));
    TLC_TRY(row_view(stats, kBwd, "stats", vs));
    if (weight) TLC_TRY(shaped(weight, kBwd, "weight", 1, &vx.cols, false, &ew));
    tlc_tensor* outs[3] = {dx, dweight, dbias};
    const char* names[3] = {"dx", "dweight", "dbias"};
    Extent eo[3];
    for (int i = 0; i < 3; ++i) {
        if (!outs[i]) continue;
        TLC_TRY(i == 0 ? shaped(dx, kBwd, "dx", x->ndim, x->sizes, true, &eo[0])
                       : shaped(outs[i], kBwd, names[i], 1, &vx.cols, true, &eo[i]));
        TLC_TRY(no_overlap(kBwd, names[i], eo[i], "x", vx.ext));
        TLC_TRY(no_overlap(kBwd, names[i], eo[i], "grad", eg));
        TLC_TRY(no_overlap(kBwd, names[i], eo[i], "stats", est));
        TLC_TRY(no_overlap(kBwd, names[i], eo[i], "weight", ew));
        for (int j = 0; j < i; ++j) TLC_TRY(no_overlap(kBwd, names[i], eo[i], names[j], eo[j]));
    }
    if (vx.cols == 0) return TLC_OK;
    if (vx.rows == 0) {  // a sum over no rows
        for (int i = 1; i < 3; ++i)
            if (outs[i] && !accumulate) TLC_TRY(launch_fill_zero(outs[i]->data, vx.cols, s));
        return TLC_OK;
    }
    if (!dx && !dweight && !dbias) return TLC_OK;
    RowScratch cx(s), cg(s), cs(s), cw(s), cp(s);
    TLC_TRY(unit_rows(x, vx, cx));
    TLC_TRY(unit_rows(grad, vg, cg));
    TLC_TRY(unit_rows(stats, vs, cs));
    LnBwd p{};
    TLC_TRY(column_vector(weight, kBwd, "weight", vx.cols, cw, &p.w, &ew));
    p.g = vg.data;
    p.x = vx.data;
    p.stats = vs.data;
    p.gm = vg.map;
    p.xm = vx.map;
    p.sm = vs.map;
    p.dx = dx ? dx->data : nullptr;
    p.rows = vx.rows;
    p.D = (int)vx.cols;
    p.accumulate = accumulate != 0;
    const bool sums = dweight || dbias;
    const bool vec = p.D % 4 == 0 && vx.map.multiple_of(4) && vg.map.multiple_of(4) && aligned_to(p.x, 16) &&
                     aligned_to(p.g, 16) && aligned_to(p.dx, 16) && aligned_to(p.w, 16);
    const int sms = sm_count();
    int parts = 0;
    if (p.D <= kRingMax) {
        const int rows_a_warp = p.D <= 128 ? 4 : p.D <= 256 ? 2 : 1;
        parts = (int)std::min<int64_t>((p.rows + rows_a_warp - 1) / rows_a_warp, sms);
        if (sums) {
            TLC_TRY(scratch_alloc(&cp.p, sizeof(float) * 2 * (size_t)p.D * (size_t)parts, s));
            p.part = cp.f();
        }
        TLC_TRY(vec ? pick_bwd<4>(p, parts, s) : pick_bwd<1>(p, parts, s));
    } else {
        if (dx) {
            ln_bwd_long_kernel<<<(unsigned)std::min<int64_t>(p.rows, INT32_MAX), 1024, 0, s>>>(p);
            count_launch();
            TLC_TRY(check_launch(kBwd));
        }
        if (sums) {
            const int64_t cols = ((int64_t)p.D + 255) / 256;
            // eight blocks an SM, but at most 128 rows in one running sum, which loses a rounding of
            // its size with each row (as many more where the grid's 65535 block rows ask for it)
            const int64_t even = (p.rows * cols + 8 * sms - 1) / (8 * sms);
            const int64_t rows_per = std::max(std::clamp<int64_t>(even, 8, 128), (p.rows + 65534) / 65535);
            parts = (int)((p.rows + rows_per - 1) / rows_per);
            TLC_TRY(scratch_alloc(&cp.p, sizeof(float) * 2 * (size_t)p.D * (size_t)parts, s));
            p.part = cp.f();
            ln_bwd_cols_kernel<<<dim3((unsigned)cols, (unsigned)parts), 256, 0, s>>>(p, rows_per);
            count_launch();
            TLC_TRY(check_launch(kBwd));
        }
    }
    if (sums) {
        const int64_t blocks = (2 * (int64_t)p.D + 31) / 32;
        TLC_TRY(launch_after(ln_bwd_finish_kernel, (unsigned)blocks, 512, s, kBwd, (const float*)p.part, parts, p.D,
                             dweight ? dweight->data : nullptr, dbias ? dbias->data : nullptr, p.accumulate));
    }
    return TLC_OK;
}
