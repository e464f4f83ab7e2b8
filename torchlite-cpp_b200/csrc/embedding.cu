// Embedding lookup with scaling, and its gradient, fp32.
//
//   out[i] = scale * W[t_i]
//   dW[v]  = scale * sum of g[i] over the positions i with t_i = v, 0 for the others
//
// A token of -1 is padding: a row of zeros, and no gradient.  Any other token
// outside [0, rows) is never used as an address: its output row is NaN and the
// gradient leaves it out.
//
// The gradient sorts the positions by token (stable, so each row's sum runs
// over ascending positions and every call gives the same bits), cuts the
// sorted list into chunks of equal length whatever the tokens are, sums runs
// of one token inside a chunk, and joins the runs that cross chunks in order.
//
// Both are bound by HBM: the lookup reads and writes 4 bytes an element, the
// gradient reads 4 an element of g and writes 4 an element of the table.
// Measured (GPU time): lookup 32768 x 4096 of 131072 rows 117 us (6.0 TB/s),
// 131072 x 64 9.3 us; gradient 65536 x 2048 into 100003 rows 244 us (5.5
// TB/s), 8192 x 768 into 32000 33 us (3.5 TB/s: three dependent kernels).  Many
// short rows are bound by the sort on eight SMs: 131072 x 64 into 1000 rows 64 us,
// 1048576 x 64 into 32000 471 us; so is accumulation (8192 x 768 27 us, 65536 x
// 2048 228 us), where no zeros are written beside it.
#include <algorithm>
#include <cmath>

#include "rows.cuh"
#include "tcgen05.cuh"

namespace tlc {
namespace {

constexpr const char* kFwd = "embedding";
constexpr const char* kBwd = "embedding_backward";

struct EmbFwd {
    const float* w;
    float* out;
    TokenRef tok;
    int64_t w_rs, rows, n;
    int D;
    float scale;
};

// A warp copies EV vectors a lane of one row: 2 KB, whatever the vector.  Rows
// and results are read and written once: streaming loads and stores leave the
// L2 to the other tensors.
template <int VEC, int EV = 16 / VEC>
__global__ void __launch_bounds__(256) embed_kernel(EmbFwd p, int pieces) {
    const int lane = threadIdx.x & 31;
    const int64_t warps = (int64_t)gridDim.x * 8;
    for (int64_t u = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); u < p.n * pieces; u += warps) {
        const int64_t i = u / pieces;
        const int j0 = (int)(u - i * pieces) * (32 * EV * VEC) + lane * VEC;
        const int64_t t = p.tok.get(i);
        const bool ok = t >= 0 && t < p.rows;
        const float fill = t == -1 ? 0.0f : __int_as_float(0x7fc00000);
        const float* src = p.w + (ok ? t : 0) * p.w_rs + j0;
        float v[EV][VEC];
#pragma unroll
        for (int k = 0; k < EV; ++k)
            if (ok && j0 + k * 32 * VEC < p.D) load_once<VEC>(src + k * 32 * VEC, v[k]);
        float* dst = p.out + i * p.D + j0;
#pragma unroll
        for (int k = 0; k < EV; ++k) {
            if (j0 + k * 32 * VEC < p.D) {
#pragma unroll
                for (int c = 0; c < VEC; ++c) v[k][c] = ok ? v[k][c] * p.scale : fill;
                store_once<VEC>(dst + k * 32 * VEC, v[k]);
            }
        }
    }
}

// Short rows: a warp copies `tokens` neighbouring rows of the result, which are
// one run of tokens * units vectors (at most 32 * EV), the k-th of a lane in row
// (32 k + lane) / units.  inv = 2^20 / units rounded up gives that quotient for
// any place below 2^20 / units, here 512 at most.
template <int VEC, int EV = 16 / VEC>
__global__ void __launch_bounds__(256) embed_short_kernel(EmbFwd p, int units, int tokens, uint32_t inv) {
    const int lane = threadIdx.x & 31;
    const int64_t warps = (int64_t)gridDim.x * 8, groups = (p.n + tokens - 1) / tokens;
    for (int64_t u = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); u < groups; u += warps) {
        const int64_t i0 = u * tokens;
        const int count = (int)min((int64_t)tokens, p.n - i0) * units;
        int col[EV];
        int64_t i[EV], t[EV];
        bool in[EV];
#pragma unroll
        for (int k = 0; k < EV; ++k) {
            const uint32_t e = k * 32 + lane;
            const int row = (int)((e * inv) >> 20);
            col[k] = ((int)e - row * units) * VEC;
            i[k] = i0 + row;
            in[k] = (int)e < count;
        }
        p.tok.get(i, in, t);
        float v[EV][VEC];
#pragma unroll
        for (int k = 0; k < EV; ++k) {
            if (t[k] >= 0 && t[k] < p.rows) load_vec<VEC>(p.w + t[k] * p.w_rs + col[k], v[k]);
        }
        float* dst = p.out + i0 * p.D;
#pragma unroll
        for (int k = 0; k < EV; ++k) {
            if (in[k]) {
                const bool ok = t[k] >= 0 && t[k] < p.rows;
                const float fill = t[k] == -1 ? 0.0f : __int_as_float(0x7fc00000);
#pragma unroll
                for (int c = 0; c < VEC; ++c) v[k][c] = ok ? v[k][c] * p.scale : fill;
                store_once<VEC>(dst + (k * 32 + lane) * VEC, v[k]);
            }
        }
    }
}

// ---- the positions sorted by token, and the rows that stay zero ----------------------------
//
// One launch does both, so that the zeros of the table are written while eight
// SMs sort.  Cluster 0 of CL blocks runs a radix sort, least digit first.  In
// each pass a warp ranks its 32 * items consecutive keys by matching digits
// across lanes, the warps' counts are scanned digit by digit, the cluster
// exchanges the blocks' counts through distributed shared memory, and each key
// goes to its place.  Stable at every level, and the result does not depend on
// timing.  Up to CL * TILE positions the list stays in the blocks' shared
// memory between passes; longer lists go through global memory tile by tile.
// The other clusters share the rows: a cluster's blocks look through the
// positions (each an eighth), mark its rows that occur in one another's shared
// memory, and write zeros to the rest.

constexpr int CL = 8;
constexpr int SORT_T = 1024;
constexpr int WARPS = SORT_T / 32;
constexpr int ITEMS = 8;
constexpr int MAX_BITS = 9;
constexpr int BINS = 1 << MAX_BITS;
constexpr int TILE = SORT_T * ITEMS;
constexpr int ZROWS = 65536;  // rows whose marks a block holds at once

struct SortArgs {
    TokenRef tok;
    int64_t rows;     // tokens outside [0, rows) get the key `rows`: behind all others
    int n;
    int bits, passes;  // digits of `bits` bits
    uint2* a;          // [n] (key, position), where even passes write
    uint2* b;          // [n], odd passes
    int* crossing;     // set to 0 here: the count of runs that cross chunks
    float* dw;         // rows to fill with zeros (NULL: none)
    int D;
    int group_shift;   // rows are dealt to the blocks in groups of 2^group_shift, at least 2 KB each
};

struct SortSmem {
    uint32_t hist[BINS];           // this block's counts, read by the cluster
    uint32_t base[BINS];           // where this block's next key of a digit goes
    uint32_t warp[WARPS][BINS];    // a warp's counts, then where its keys go within the block's
    uint32_t wsum[WARPS];
    uint2 keys[TILE];              // the block's part of the list between passes
};
struct FillSmem {
    uint32_t marks[ZROWS / 32];
};

__device__ __forceinline__ uint32_t cluster_addr(const void* local, uint32_t rank) {
    return mapa(static_cast<uint32_t>(__cvta_generic_to_shared(local)), rank);
}
__device__ __forceinline__ uint32_t ld_cluster_u32(const uint32_t* local, uint32_t rank) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(cluster_addr(local, rank)) : "memory");
    return v;
}

__device__ void sort_positions(const SortArgs& p, SortSmem& sm) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = (int)cluster_ctarank();
    const int per = (p.n + CL - 1) / CL;
    const int i0 = min(p.n, rank * per), i1 = min(p.n, i0 + per);
    const int bins = 1 << p.bits;
    const bool one = per <= TILE;  // the block's part is one tile
    const int items = min(ITEMS, (per + SORT_T - 1) / SORT_T);
    if (rank == 0 && tid == 0) *p.crossing = 0;
    uint2 kv[ITEMS];
    uint32_t at[ITEMS];
    for (int pass = 0; pass < p.passes; ++pass) {
        const uint2* src = (pass & 1) ? p.a : p.b;  // pass 0 reads the tokens
        uint2* dst = (pass & 1) ? p.b : p.a;
        const bool last = pass + 1 == p.passes;
        const int shift = pass * p.bits;
        auto digit = [&](uint2 k) { return (k.x >> shift) & (uint32_t)(bins - 1); };
        // keys first, first + step, ... below i1 (all loads before the first use)
        auto load = [&](int first, int step, uint2 (&to)[ITEMS]) {
            if (pass == 0) {
                int64_t t[ITEMS];
                p.tok.get(first, step, i1, t);
#pragma unroll
                for (int k = 0; k < ITEMS; ++k)
                    to[k] = make_uint2((uint32_t)(t[k] >= 0 && t[k] < p.rows ? t[k] : p.rows),
                                       (uint32_t)(first + k * step));
            } else if (one) {
#pragma unroll
                for (int k = 0; k < ITEMS; ++k)
                    if (first + k * step < i1) to[k] = sm.keys[first + k * step - i0];
            } else {
#pragma unroll
                for (int k = 0; k < ITEMS; ++k)
                    if (first + k * step < i1) to[k] = __ldcg(src + first + k * step);
            }
        };
        // a tile's keys, and each key's place among its warp's of the same digit
        auto rank_tile = [&](int t0) {
            for (int d = lane; d < bins; d += 32) sm.warp[warp][d] = 0;
            const int w0 = t0 + warp * 32 * items + lane;
            load(w0, 32, kv);  // with fewer items a warp also reads its neighbours' keys, and leaves them
            __syncwarp();
#pragma unroll
            for (int k = 0; k < ITEMS; ++k) {
                if (k >= items) break;
                const bool in = w0 + k * 32 < i1;
                const uint32_t d = in ? digit(kv[k]) : 0u;
                // the lanes with the same digit, by a vote for each of its bits
                uint32_t peers = __ballot_sync(0xffffffffu, in);
                for (int b = 0; b < p.bits; ++b) {
                    const uint32_t vote = __ballot_sync(0xffffffffu, (d >> b) & 1u);
                    peers &= (d >> b) & 1u ? vote : ~vote;
                }
                const uint32_t old = in ? sm.warp[warp][d] : 0u;
                __syncwarp();
                if (in && lane == 31 - __clz(peers)) sm.warp[warp][d] = old + __popc(peers);
                __syncwarp();
                at[k] = old + __popc(peers & ((1u << lane) - 1u));
            }
            __syncthreads();
        };
        // the warps' counts of a digit -> the places of each warp's first; returns the block's count
        auto scan_warps = [&](int d) -> uint32_t {
            uint32_t c[WARPS], run = 0;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) c[w] = sm.warp[w][d];
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                sm.warp[w][d] = run;
                run += c[w];
            }
            return run;
        };
        auto place_tile = [&](int t0) {
            const int w0 = t0 + warp * 32 * items + lane;
#pragma unroll
            for (int k = 0; k < ITEMS; ++k) {
                if (k < items && w0 + k * 32 < i1) {
                    const uint32_t d = digit(kv[k]);
                    const uint32_t to = sm.base[d] + sm.warp[warp][d] + at[k];
                    if (one && !last) {
                        const uint32_t owner = to / (uint32_t)per;
                        asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(
                                         cluster_addr(&sm.keys[to - owner * (uint32_t)per], owner)),
                                     "r"(kv[k].x), "r"(kv[k].y)
                                     : "memory");
                    } else {
                        dst[to] = kv[k];
                    }
                }
            }
        };
        if (one) {
            rank_tile(i0);
            if (tid < bins) sm.hist[tid] = scan_warps(tid);
        } else {
            for (int d = tid; d < bins; d += SORT_T) sm.hist[d] = 0;
            __syncthreads();
            for (int i = i0 + tid; i < i1; i += TILE) {
                load(i, SORT_T, kv);
#pragma unroll
                for (int k = 0; k < ITEMS; ++k)
                    if (i + k * SORT_T < i1) atomicAdd(&sm.hist[digit(kv[k])], 1u);
            }
        }
        cluster_sync();  // counts in place; with one tile all keys are in registers as well
        // base[d] = keys of lower digits in the cluster + keys of d in lower blocks
        uint32_t total = 0, below = 0;
        if (tid < bins) {
            uint32_t c[CL];
#pragma unroll
            for (int q = 0; q < CL; ++q) c[q] = ld_cluster_u32(&sm.hist[tid], (uint32_t)q);
#pragma unroll
            for (int q = 0; q < CL; ++q) {
                total += c[q];
                if (q < rank) below += c[q];
            }
        }
        uint32_t incl = total;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) sm.wsum[warp] = incl;
        __syncthreads();
        if (tid < bins) {
            uint32_t before = 0;
#pragma unroll
            for (int w = 0; w < BINS / 32; ++w) before += w < warp ? sm.wsum[w] : 0u;
            sm.base[tid] = before + incl - total + below;
        }
        __syncthreads();
        if (one) {
            place_tile(i0);
        } else {
            for (int t0 = i0; t0 < i1; t0 += TILE) {
                rank_tile(t0);
                const uint32_t count = tid < bins ? scan_warps(tid) : 0u;
                __syncthreads();
                place_tile(t0);
                __syncthreads();
                if (tid < bins) sm.base[tid] += count;
            }
        }
        cluster_sync();  // the pass's list is complete, and the counts have been read
    }
}

__device__ void fill_absent(const SortArgs& p, FillSmem& sm, uint32_t cluster, uint32_t clusters) {
    const int tid = threadIdx.x, lane = tid & 31;
    const uint32_t rank = cluster_ctarank(), blocks = clusters * CL, me = cluster * CL + rank;
    // Rows in groups of 2^gs, dealt to the blocks in turn: frequent tokens have
    // low numbers, so ranges of neighbouring rows would leave some blocks
    // without work (600 MB of zeros in 140 us instead of 100).
    const int gs = p.group_shift;
    const int64_t span = (int64_t)blocks * ZROWS;  // rows whose marks fit at once
    // the lanes that share a row
    int g = 1;
    while (g < 32 && g * 4 < p.D) g <<= 1;
    for (int64_t lo = 0; lo < p.rows; lo += span) {
        const uint32_t rows = (uint32_t)min(span, p.rows - lo);
        const uint32_t groups = (rows + (1u << gs) - 1) >> gs;
        const uint32_t per = ((groups + blocks - 1) / blocks) << gs;  // marks a block
        for (uint32_t w = tid; w * 32 < per; w += SORT_T) sm.marks[w] = 0;
        cluster_sync();
        for (int64_t i0 = (int64_t)rank * SORT_T + tid; i0 < p.n; i0 += CL * SORT_T * 4) {
            int64_t t[4];
            p.tok.get(i0, CL * SORT_T, p.n, t);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                t[k] -= lo;
                if (t[k] < 0 || t[k] >= (int64_t)rows) continue;
                const uint32_t group = (uint32_t)t[k] >> gs, turn = group / blocks, owner = group - turn * blocks;
                if (owner / CL != cluster) continue;
                const uint32_t at = (turn << gs) | ((uint32_t)t[k] & ((1u << gs) - 1u));
                asm volatile("red.relaxed.cluster.shared::cluster.or.b32 [%0], %1;" ::"r"(
                                 cluster_addr(&sm.marks[at >> 5], owner % CL)),
                             "r"(1u << (at & 31))
                             : "memory");
            }
        }
        cluster_sync();
        for (uint32_t q = tid / g; q < per; q += SORT_T / g) {
            if ((sm.marks[q >> 5] >> (q & 31)) & 1u) continue;
            const uint32_t v = ((((q >> gs) * blocks) + me) << gs) | (q & ((1u << gs) - 1u));
            if (v >= rows) continue;
            float* row = p.dw + (lo + v) * p.D;
            // single values up to a 16-byte boundary and behind the last one, float4 between
            const int head = min(p.D, (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) >> 2);
            const int vecs = (p.D - head) >> 2;
            for (int j = lane & (g - 1); j < vecs; j += g)
                __stcs(reinterpret_cast<float4*>(row + head) + j, make_float4(0.0f, 0.0f, 0.0f, 0.0f));
            for (int j = lane & (g - 1); j < head; j += g) __stcs(row + j, 0.0f);
            for (int j = head + 4 * vecs + (lane & (g - 1)); j < p.D; j += g) __stcs(row + j, 0.0f);
        }
        cluster_sync();  // before the marks are cleared again
    }
}

__global__ void __cluster_dims__(CL, 1, 1) __launch_bounds__(SORT_T) embed_sort_kernel(SortArgs p) {
    extern __shared__ __align__(16) unsigned char raw[];
    next_may_launch();
    const int cluster = (int)blockIdx.x / CL, clusters = (int)gridDim.x / CL;
    if (cluster == 0)
        sort_positions(p, *reinterpret_cast<SortSmem*>(raw));
    else
        fill_absent(p, *reinterpret_cast<FillSmem*>(raw), (uint32_t)(cluster - 1), (uint32_t)(clusters - 1));
}

// ---- the sums of runs -------------------------------------------------------------------

constexpr int AHEAD = 8;  // rows whose loads a warp has in flight

struct SumArgs {
    const uint2* list;  // (token, position) by token
    const float* g;
    Rows gm;
    float* dw;
    float* part;    // [chunks][2][D]: 0: a run that began before the chunk, 1: one that goes on behind it
    int* crossing;  // count, then the chunks whose last run begins there and goes on
    int64_t rows;
    int n, D;
    int ch;  // sorted positions a chunk, at most 32
    int accumulate;
    float scale;
};

template <int VEC>
__device__ __forceinline__ void write_row(const SumArgs& p, int64_t row, int j, float (&a)[VEC]) {
    float* o = p.dw + row * p.D + j;
    float old[VEC];
    if (p.accumulate) load_vec<VEC>(o, old);
#pragma unroll
    for (int c = 0; c < VEC; ++c) {
        a[c] = __fmul_rn(p.scale, a[c]);
        if (p.accumulate) a[c] = __fadd_rn(a[c], old[c]);  // the gradient rounded, then added
    }
    store_vec<VEC>(o, a);
}

// A warp takes one chunk and 32 * VEC * VPT columns.  Lane i holds the i-th
// position's key and row; where runs end is one mask.
template <int VEC, int VPT>
__global__ void __launch_bounds__(256) embed_sum_kernel(SumArgs p, int64_t units, int slices) {
    next_may_launch();
    after_previous();
    const int lane = threadIdx.x & 31;
    const int64_t u = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (u >= units) return;
    const int chunk = (int)(u / slices), slice = (int)(u - (int64_t)chunk * slices);
    const int j0 = slice * (32 * VEC * VPT) + lane * VEC;
    const int p0 = chunk * p.ch, cnt = min(p.ch, p.n - p0);
    const uint32_t none = (uint32_t)p.rows;
    const uint2 mine = lane < cnt ? p.list[p0 + lane] : make_uint2(none, 0u);
    const uint32_t prev = p0 > 0 ? p.list[p0 - 1].x : none, next = p0 + cnt < p.n ? p.list[p0 + cnt].x : none;
    const int valid = __popc(__ballot_sync(0xffffffffu, mine.x != none));  // keys that are none come last
    if (valid == 0) return;
    const int64_t row = p.gm.offset(mine.y);
    const uint32_t after = __shfl_down_sync(0xffffffffu, mine.x, 1);
    const uint32_t ends = __ballot_sync(0xffffffffu, lane < valid && (lane == valid - 1 || after != mine.x));
    const bool on = valid == cnt && __shfl_sync(0xffffffffu, mine.x, valid - 1) == next;
    bool before = __shfl_sync(0xffffffffu, mine.x, 0) == prev;
    float a[VPT][VEC];
#pragma unroll
    for (int q = 0; q < VPT; ++q)
#pragma unroll
        for (int c = 0; c < VEC; ++c) a[q][c] = 0.0f;
    for (int i0 = 0; i0 < valid; i0 += AHEAD) {
        float v[AHEAD][VPT][VEC];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const float* g = p.g + __shfl_sync(0xffffffffu, row, (i0 + k) & 31) + j0;
            if (i0 + k < valid) {
#pragma unroll
                for (int q = 0; q < VPT; ++q)
                    if (j0 + q * 32 * VEC < p.D) load_once<VEC>(g + q * 32 * VEC, v[k][q]);
            }
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const int i = i0 + k;
            if (i >= valid) break;
#pragma unroll
            for (int q = 0; q < VPT; ++q)
#pragma unroll
                for (int c = 0; c < VEC; ++c) a[q][c] += v[k][q][c];
            if (!((ends >> i) & 1u)) continue;
            const uint32_t key = __shfl_sync(0xffffffffu, mine.x, i);
            const bool goes_on = on && i == valid - 1;
#pragma unroll
            for (int q = 0; q < VPT; ++q) {
                const int j = j0 + q * 32 * VEC;
                if (j < p.D) {
                    if (!before && !goes_on)
                        write_row<VEC>(p, key, j, a[q]);
                    else
                        store_vec<VEC>(p.part + ((int64_t)chunk * 2 + (before ? 0 : 1)) * p.D + j, a[q]);
                }
#pragma unroll
                for (int c = 0; c < VEC; ++c) a[q][c] = 0.0f;
            }
            // the order of this list does not matter: each entry is summed by itself
            if (goes_on && !before && slice == 0 && lane == 0) p.crossing[1 + atomicAdd(p.crossing, 1)] = chunk;
            before = false;
        }
    }
}

// The sums of `count` parts 0 from chunk `c` on, in their order.
template <int VEC, int VPT>
__device__ __forceinline__ void add_parts(const SumArgs& p, int c, int count, int j, float (&a)[VPT][VEC]) {
    constexpr int U = 4;
    for (int q = 0; q < count; q += U) {
        float v[U][VPT][VEC];
#pragma unroll
        for (int k = 0; k < U; ++k)
#pragma unroll
            for (int i = 0; i < VPT; ++i)
                if (q + k < count && j + i * 32 * VEC < p.D)
                    load_vec<VEC>(p.part + (int64_t)(c + q + k) * 2 * p.D + j + i * 32 * VEC, v[k][i]);
#pragma unroll
        for (int k = 0; k < U; ++k)
            if (q + k < count)
#pragma unroll
                for (int i = 0; i < VPT; ++i)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) a[i][e] += v[k][i][e];
    }
}

// A run that crosses chunks: its first chunk's part 1, then part 0 of the
// chunks behind it, in their order.  A warp takes a run and 32 * VEC * VPT
// columns (a run is found by five loads one after the other, so a warp finds
// few and sums much); runs of more than LONG chunks (one token in hundreds of
// positions) are shared by the block's warps, an eighth of the chunks each.
constexpr int LONG = 16;
template <int VEC, int VPT>
__global__ void __launch_bounds__(256) embed_join_kernel(SumArgs p, int slices) {
    __shared__ int long_chunk[8], long_slice[8], long_count[8];
    __shared__ __align__(16) float eighth[8][VPT][32 * VEC];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    after_previous();
    const int runs = *p.crossing;
    const int64_t units = (int64_t)runs * slices;
    // the block's warps take units far apart: frequent tokens, neighbours in the list, have long runs
    for (int64_t u0 = blockIdx.x; u0 < units; u0 += (int64_t)gridDim.x * 8) {
        const int64_t u = u0 + (int64_t)gridDim.x * warp;
        int count = 0;  // chunks behind the first
        float a[VPT][VEC];
        auto first_part = [&](int chunk, int j) {
#pragma unroll
            for (int i = 0; i < VPT; ++i)
                if (j + i * 32 * VEC < p.D)
                    load_vec<VEC>(p.part + ((int64_t)chunk * 2 + 1) * p.D + j + i * 32 * VEC, a[i]);
        };
        auto write = [&](uint32_t key, int j) {
#pragma unroll
            for (int i = 0; i < VPT; ++i)
                if (j + i * 32 * VEC < p.D) write_row<VEC>(p, key, j + i * 32 * VEC, a[i]);
        };
        if (u < units) {
            // neighbouring warps take different runs: the slices of a long one go to different blocks
            const int slice = (int)(u / runs), chunk = p.crossing[1 + (int)(u - (int64_t)slice * runs)];
            const int j = slice * (32 * VEC * VPT) + lane * VEC;
            const uint32_t key = p.list[(int64_t)(chunk + 1) * p.ch - 1].x;
            for (;;) {  // does the run reach into chunk + 1 + count + lane?
                const int64_t begin = (int64_t)(chunk + 1 + count + lane) * p.ch;
                const uint32_t go = __ballot_sync(0xffffffffu, begin < p.n && p.list[begin < p.n ? begin : 0].x == key);
                const int full = go == 0xffffffffu ? 32 : __ffs(~go) - 1;
                count += full;
                if (full < 32) break;
            }
            if (count <= LONG) {
                first_part(chunk, j);
                add_parts<VEC, VPT>(p, chunk + 1, count, j, a);
                write(key, j);
            }
            if (lane == 0) long_chunk[warp] = chunk, long_slice[warp] = slice;
        }
        if (lane == 0) long_count[warp] = count > LONG ? count : 0;
        __syncthreads();
        for (int q = 0; q < 8; ++q) {
            const int n = long_count[q];
            if (n == 0) continue;
            const int chunk = long_chunk[q], j = long_slice[q] * (32 * VEC * VPT) + lane * VEC;
            const int per = (n + 7) / 8, c0 = min(n, warp * per), c1 = min(n, c0 + per);
#pragma unroll
            for (int i = 0; i < VPT; ++i)
#pragma unroll
                for (int e = 0; e < VEC; ++e) a[i][e] = 0.0f;
            if (warp == 0) first_part(chunk, j);
            add_parts<VEC, VPT>(p, chunk + 1 + c0, c1 - c0, j, a);
#pragma unroll
            for (int i = 0; i < VPT; ++i) store_vec<VEC>(&eighth[warp][i][lane * VEC], a[i]);
            __syncthreads();
            if (warp == 0) {
#pragma unroll
                for (int w = 1; w < 8; ++w)
#pragma unroll
                    for (int i = 0; i < VPT; ++i) {
                        float v[VEC];
                        load_vec<VEC>(&eighth[w][i][lane * VEC], v);
#pragma unroll
                        for (int e = 0; e < VEC; ++e) a[i][e] += v[e];
                    }
                write(p.list[(int64_t)(chunk + 1) * p.ch - 1].x, j);
            }
            __syncthreads();
        }
        __syncthreads();  // the lists are written again
    }
}

int table_view(const tlc_tensor* w, const char* op, const char* name, RowView& v) {
    TLC_TRY(row_view(w, op, name, v));
    if (w->ndim != 2) return set_error(TLC_ERR_INVALID_ARGUMENT, std::string(op) + ": " + name + " must be 2-D");
    if (v.rows > INT32_MAX - 1 || v.cols > INT32_MAX / 4)
        return set_error(TLC_ERR_UNSUPPORTED, std::string(op) + ": " + name + " too large");
    return TLC_OK;
}

// [tokens' shape, D]
int hidden_shape(const tlc_index* t, int64_t D, const char* op, int* nd, int64_t* sz) {
    if (t->ndim + 1 > TLC_MAX_DIMS)
        return set_error(TLC_ERR_INVALID_ARGUMENT, std::string(op) + ": tokens have too many dims");
    std::copy(t->sizes, t->sizes + t->ndim, sz);
    sz[t->ndim] = D;
    *nd = t->ndim + 1;
    return TLC_OK;
}

int check_scale(float scale, const char* op) {
    if (std::isfinite(scale)) return TLC_OK;
    return set_error(TLC_ERR_INVALID_ARGUMENT, std::string(op) + ": scale must be finite");
}

template <int VEC>
int launch_embed(const EmbFwd& p, cudaStream_t s) {
    const int units = p.D / VEC, tokens = 512 / VEC / units;
    if (tokens >= 2) {
        const uint32_t inv = ((1u << 20) + units - 1) / units;
        const int64_t want = ((p.n + tokens - 1) / tokens + 7) / 8;
        embed_short_kernel<VEC><<<(unsigned)std::min<int64_t>(want, INT32_MAX), 256, 0, s>>>(p, units, tokens, inv);
        count_launch();
        return check_launch(kFwd);
    }
    const int pieces = (p.D + 511) / 512;
    const int64_t want = (p.n * pieces + 7) / 8;
    embed_kernel<VEC><<<(unsigned)std::min<int64_t>(want, INT32_MAX), 256, 0, s>>>(p, pieces);
    count_launch();
    return check_launch(kFwd);
}

template <int VEC, int VPT>
int launch_sums(const SumArgs& p, cudaStream_t s) {
    const int64_t chunks = (p.n + p.ch - 1) / p.ch;
    const int slices = (p.D + 32 * VEC * VPT - 1) / (32 * VEC * VPT);
    const int64_t blocks = (chunks * slices + 7) / 8;
    if (blocks > INT32_MAX) return set_error(TLC_ERR_UNSUPPORTED, "embedding_backward: too many tokens");
    TLC_TRY(launch_after(embed_sum_kernel<VEC, VPT>, (unsigned)blocks, 256, s, kBwd, p, chunks * slices, slices));
    if (chunks == 1) return TLC_OK;  // no run crosses
    // the number of crossing runs is on the device: enough blocks to keep every SM busy
    constexpr int WIDE = 2;
    const int wide = (p.D + 32 * VEC * WIDE - 1) / (32 * VEC * WIDE);
    const unsigned grid = (unsigned)std::min<int64_t>((chunks * wide + 7) / 8, (int64_t)sm_count() * 4);
    return launch_after(embed_join_kernel<VEC, WIDE>, grid, 256, s, kBwd, p, wide);
}

// The most clusters of the sort kernel that run at once on the current device.
int max_clusters(int* out) {
    static DeviceOnce once;
    static int clusters[64];
    int dev = 0;
    TLC_TRY(device_once(
        once,
        [](int d) -> int {
            SetupDuringCapture relaxed;
            const int smem = (int)std::max(sizeof(SortSmem), sizeof(FillSmem));
            TLC_CUDA_TRY(cudaFuncSetAttribute(embed_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
            cudaLaunchConfig_t cfg{};
            cfg.gridDim = dim3(CL);
            cfg.blockDim = dim3(SORT_T);
            cfg.dynamicSmemBytes = (size_t)smem;
            int n = 0;
            TLC_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, embed_sort_kernel, &cfg));
            clusters[d] = std::max(n, 2);
            return TLC_OK;
        },
        &dev));
    *out = clusters[dev];
    return TLC_OK;
}

}  // namespace
}  // namespace tlc

using namespace tlc;

extern "C" int tlc_embedding(const tlc_tensor* weight, const tlc_index* tokens, float scale, tlc_tensor* out,
                             void* stream) {
    clear_error();
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    RowView vw;
    EmbFwd p{};
    Extent et, eo;
    int64_t sz[TLC_MAX_DIMS];
    int nd;
    TLC_TRY(table_view(weight, kFwd, "weight", vw));
    TLC_TRY(index_view(tokens, kFwd, "tokens", p.tok, &p.n, &et));
    TLC_TRY(check_scale(scale, kFwd));
    TLC_TRY(hidden_shape(tokens, vw.cols, kFwd, &nd, sz));
    TLC_TRY(shaped(out, kFwd, "out", nd, sz, true, &eo));
    TLC_TRY(no_overlap(kFwd, "out", eo, "weight", vw.ext));
    TLC_TRY(no_overlap(kFwd, "out", eo, "tokens", et));
    if (p.n == 0 || vw.cols == 0) return TLC_OK;
    RowScratch cw(s);
    TLC_TRY(unit_rows(weight, vw, cw));
    p.w = vw.data;
    p.w_rs = vw.map.nd ? vw.map.st[0] : 0;
    p.out = out->data;
    p.rows = vw.rows;
    p.D = (int)vw.cols;
    p.scale = scale;
    const bool vec = p.D % 4 == 0 && p.w_rs % 4 == 0 && aligned_to(p.w, 16) && aligned_to(p.out, 16);
    return vec ? launch_embed<4>(p, s) : launch_embed<1>(p, s);
}

extern "C" int tlc_embedding_backward(const tlc_tensor* grad, const tlc_index* tokens, float scale,
                                      tlc_tensor* dweight, int accumulate, void* stream) {
    clear_error();
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    RowView vd, vg;
    TokenRef tok;
    Extent et, ed, eg;
    int64_t sz[TLC_MAX_DIMS], n;
    int nd;
    TLC_TRY(table_view(dweight, kBwd, "dweight", vd));
    TLC_TRY(shaped(dweight, kBwd, "dweight", 2, dweight->sizes, true, &ed));
    TLC_TRY(index_view(tokens, kBwd, "tokens", tok, &n, &et));
    TLC_TRY(check_scale(scale, kBwd));
    TLC_TRY(hidden_shape(tokens, vd.cols, kBwd, &nd, sz));
    TLC_TRY(shaped(grad, kBwd, "grad", nd, sz, false, &eg));
    TLC_TRY(row_view(grad, kBwd, "grad", vg));
    TLC_TRY(no_overlap(kBwd, "dweight", ed, "grad", eg));
    TLC_TRY(no_overlap(kBwd, "dweight", ed, "tokens", et));
    if (n > INT32_MAX - TILE) return set_error(TLC_ERR_UNSUPPORTED, "embedding_backward: too many tokens");
    if (vd.numel == 0) return TLC_OK;
    if (n == 0) return accumulate ? TLC_OK : launch_fill_zero(dweight->data, vd.numel, s);
    RowScratch cg(s), cw(s);
    TLC_TRY(unit_rows(grad, vg, cg));
    const int D = (int)vd.cols;
    const bool vec = D % 4 == 0 && vg.map.multiple_of(4) && aligned_to(vg.data, 16) && aligned_to(dweight->data, 16);
    // 32 positions a chunk; 16 where that would leave an SM fewer than 16 warps
    const int64_t slices = (D + 255) / 256;
    const int ch = (n / 32) * slices >= (int64_t)sm_count() * 16 ? 32 : 16;
    const int64_t chunks = (n + ch - 1) / ch;
    // one workspace: the parts, the two lists, the crossing runs
    const size_t part_bytes = sizeof(float) * 2 * (size_t)chunks * (size_t)D;
    const size_t list_at = (part_bytes + 15) & ~size_t(15), list_bytes = sizeof(uint2) * (size_t)n;
    TLC_TRY(scratch_alloc(&cw.p, list_at + 2 * list_bytes + sizeof(int) * (size_t)(chunks + 1), s));
    char* ws = static_cast<char*>(cw.p);
    SortArgs q{};
    q.tok = tok;
    q.rows = vd.rows;
    q.n = (int)n;
    int width = 1;  // bits of the largest key, vd.rows
    while ((vd.rows >> width) != 0) ++width;
    q.passes = (width + MAX_BITS - 1) / MAX_BITS;
    q.bits = (width + q.passes - 1) / q.passes;
    q.a = reinterpret_cast<uint2*>(ws + list_at);
    q.b = q.a + n;
    q.crossing = reinterpret_cast<int*>(q.b + n);
    int clusters = 1;
    if (!accumulate) {
        TLC_TRY(max_clusters(&clusters));
        q.dw = dweight->data;
        q.D = D;
        while (q.group_shift < 5 && ((int64_t)D * 4 << q.group_shift) < 2048) ++q.group_shift;
    } else {
        int unused;
        TLC_TRY(max_clusters(&unused));  // sets the kernel's shared-memory limit
    }
    embed_sort_kernel<<<CL * clusters, SORT_T, std::max(sizeof(SortSmem), sizeof(FillSmem)), s>>>(q);
    count_launch();
    TLC_TRY(check_launch(kBwd));
    SumArgs p{};
    p.list = (q.passes & 1) ? q.a : q.b;
    p.g = vg.data;
    p.gm = vg.map;
    p.dw = dweight->data;
    p.part = reinterpret_cast<float*>(ws);
    p.crossing = q.crossing;
    p.rows = vd.rows;
    p.n = (int)n;
    p.D = D;
    p.accumulate = accumulate != 0;
    p.scale = scale;
    p.ch = ch;
    return vec ? launch_sums<4, 2>(p, s) : launch_sums<1, 4>(p, s);
}
