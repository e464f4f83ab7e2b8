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

// A warp copies 4 vectors a lane of one row.
template <int VEC>
__global__ void __launch_bounds__(256) embed_kernel(EmbFwd p, int pieces) {
    const int lane = threadIdx.x & 31;
    const int64_t warps = (int64_t)gridDim.x * 8;
    for (int64_t u = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); u < p.n * pieces; u += warps) {
        const int64_t i = u / pieces;
        const int j0 = (int)(u - i * pieces) * (128 * VEC) + lane * VEC;
        const int64_t t = p.tok.get(i);
        const bool ok = t >= 0 && t < p.rows;
        const float fill = t == -1 ? 0.0f : __int_as_float(0x7fc00000);
        const float* src = p.w + (ok ? t : 0) * p.w_rs;
        float v[4][VEC];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int j = j0 + k * 32 * VEC;
            if (ok && j < p.D) load_vec<VEC>(src + j, v[k]);
        }
        float* dst = p.out + i * p.D;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int j = j0 + k * 32 * VEC;
            if (j < p.D) {
#pragma unroll
                for (int c = 0; c < VEC; ++c) v[k][c] = ok ? v[k][c] * p.scale : fill;
                store_vec<VEC>(dst + j, v[k]);
            }
        }
    }
}

// ---- the positions sorted by token ------------------------------------------------------
//
// A radix sort by one cluster of CL blocks, least digit first.  In each pass a
// block counts the digits of its part of the list, the cluster exchanges the
// counts through distributed shared memory, and the block scatters its part
// tile by tile: a warp ranks its 32 * ITEMS consecutive keys by matching
// digits across lanes, then the warps' counts are scanned digit by digit.
// Stable at every level, and the result does not depend on timing.

constexpr int CL = 8;
constexpr int SORT_T = 1024;
constexpr int ITEMS = 8;
constexpr int MAX_BITS = 9;
constexpr int BINS = 1 << MAX_BITS;
constexpr int TILE = SORT_T * ITEMS;

struct SortArgs {
    TokenRef tok;
    int64_t rows;     // tokens outside [0, rows) get the key `rows`: behind all others
    int n;
    int bits, passes;  // digits of `bits` bits
    uint2* a;          // [n] (key, position): even passes write here
    uint2* b;          // [n]: odd passes
};

struct SortSmem {
    uint32_t hist[BINS];           // this block's counts, read by the cluster
    uint32_t base[BINS];           // where this block's next key of a digit goes
    uint32_t scan[BINS];
    uint32_t warp[SORT_T / 32][BINS];
    uint32_t wsum[32];
};

__device__ __forceinline__ uint32_t ld_cluster_u32(const uint32_t* local, uint32_t rank) {
    uint32_t v;
    const uint32_t addr = mapa(static_cast<uint32_t>(__cvta_generic_to_shared(local)), rank);
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}

__global__ void __cluster_dims__(CL, 1, 1) __launch_bounds__(SORT_T) embed_sort_kernel(SortArgs p) {
    extern __shared__ __align__(16) unsigned char raw[];
    SortSmem& sm = *reinterpret_cast<SortSmem*>(raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = (int)cluster_ctarank();
    const int per = (p.n + CL - 1) / CL;
    const int i0 = min(p.n, rank * per), i1 = min(p.n, i0 + per);
    const int bins = 1 << p.bits;
    for (int pass = 0; pass < p.passes; ++pass) {
        const uint2* src = (pass & 1) ? p.a : p.b;  // pass 0 reads the tokens
        uint2* dst = (pass & 1) ? p.b : p.a;
        const int shift = pass * p.bits;
        auto load = [&](int i) -> uint2 {
            if (pass > 0) return __ldcg(src + i);
            const int64_t t = p.tok.get(i);
            return make_uint2((uint32_t)(t >= 0 && t < p.rows ? t : p.rows), (uint32_t)i);
        };
        for (int d = tid; d < BINS; d += SORT_T) sm.hist[d] = 0;
        __syncthreads();
        for (int i = i0 + tid; i < i1; i += SORT_T) atomicAdd(&sm.hist[(load(i).x >> shift) & (bins - 1)], 1u);
        cluster_sync();
        // base[d] = keys of lower digits in the cluster + keys of d in lower blocks
        uint32_t total = 0, below = 0;
        if (tid < bins) {
            for (int c = 0; c < CL; ++c) {
                const uint32_t v = ld_cluster_u32(&sm.hist[tid], (uint32_t)c);
                total += v;
                if (c < rank) below += v;
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
            for (int w = 0; w < warp; ++w) before += sm.wsum[w];
            sm.base[tid] = before + incl - total + below;
        }
        __syncthreads();
        for (int t0 = i0; t0 < i1; t0 += TILE) {
            for (int d = lane; d < bins; d += 32) sm.warp[warp][d] = 0;
            __syncwarp();
            uint2 kv[ITEMS];
            uint32_t at[ITEMS];
            const int w0 = t0 + warp * 32 * ITEMS;
#pragma unroll
            for (int k = 0; k < ITEMS; ++k) {
                const int i = w0 + k * 32 + lane;
                kv[k] = i < i1 ? load(i) : make_uint2(0u, 0u);
            }
#pragma unroll
            for (int k = 0; k < ITEMS; ++k) {
                const bool in = w0 + k * 32 + lane < i1;
                // lanes past the end match nobody's digit
                const uint32_t d = in ? (kv[k].x >> shift) & (uint32_t)(bins - 1) : (uint32_t)(BINS + lane);
                const uint32_t peers = __match_any_sync(0xffffffffu, d);
                const uint32_t old = in ? sm.warp[warp][d] : 0u;
                __syncwarp();
                if (in && lane == 31 - __clz(peers)) sm.warp[warp][d] = old + __popc(peers);
                __syncwarp();
                at[k] = old + __popc(peers & ((1u << lane) - 1u));
            }
            __syncthreads();
            if (tid < bins) {  // the warps' counts -> where each warp's keys of this digit go
                uint32_t run = sm.base[tid];
                for (int w = 0; w < SORT_T / 32; ++w) {
                    const uint32_t c = sm.warp[w][tid];
                    sm.warp[w][tid] = run;
                    run += c;
                }
                sm.base[tid] = run;
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < ITEMS; ++k)
                if (w0 + k * 32 + lane < i1)
                    dst[sm.warp[warp][(kv[k].x >> shift) & (uint32_t)(bins - 1)] + at[k]] = kv[k];
            __syncthreads();
        }
        cluster_sync();  // the pass's list is complete, and the counts have been read
    }
}

// ---- the sums of runs -------------------------------------------------------------------

constexpr int CH = 32;  // sorted positions a chunk
constexpr int AHEAD = 8;

struct SumArgs {
    const uint2* list;  // (token, position) by token
    const float* g;
    Rows gm;
    float* dw;
    float* part;  // [chunks][2][D]: 0: a run that began before the chunk, 1: one that goes on behind it
    int64_t rows;
    int n, D;
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

// A warp takes one chunk and 32 * VEC columns.
template <int VEC>
__global__ void __launch_bounds__(256) embed_sum_kernel(SumArgs p, int64_t units, int slices) {
    const int lane = threadIdx.x & 31;
    const int64_t u = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (u >= units) return;
    const int chunk = (int)(u / slices);
    const int j = (int)(u - (int64_t)chunk * slices) * (32 * VEC) + lane * VEC;
    const int p0 = chunk * CH, cnt = min(CH, p.n - p0);
    const uint32_t none = (uint32_t)p.rows;
    const uint2 mine = lane < cnt ? p.list[p0 + lane] : make_uint2(none, 0u);
    const uint32_t prev = p0 > 0 ? p.list[p0 - 1].x : none, next = p0 + cnt < p.n ? p.list[p0 + cnt].x : none;
    const bool in = j < p.D;
    float a[VEC];
#pragma unroll
    for (int c = 0; c < VEC; ++c) a[c] = 0.0f;
    bool first = true;  // the run being summed is the chunk's first
    for (int i0 = 0; i0 < cnt; i0 += AHEAD) {
        float v[AHEAD][VEC];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const uint32_t key = __shfl_sync(0xffffffffu, mine.x, (i0 + k) & 31);
            const uint32_t pos = __shfl_sync(0xffffffffu, mine.y, (i0 + k) & 31);
            if (in && i0 + k < cnt && key != none) {
                load_once<VEC>(p.g + p.gm.offset(pos) + j, v[k]);
            } else {
#pragma unroll
                for (int c = 0; c < VEC; ++c) v[k][c] = 0.0f;
            }
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const int i = i0 + k;
            const uint32_t key = __shfl_sync(0xffffffffu, mine.x, i & 31);
            const uint32_t after = i + 1 < cnt ? __shfl_sync(0xffffffffu, mine.x, (i + 1) & 31) : next;
            if (i >= cnt || key == none) return;  // only keys that are none follow
#pragma unroll
            for (int c = 0; c < VEC; ++c) a[c] += v[k][c];
            if (after == key && i + 1 < cnt) continue;
            const bool before = first && prev == key, on = after == key;
            if (in) {
                if (!before && !on) {
                    write_row<VEC>(p, key, j, a);
                } else {
                    store_vec<VEC>(p.part + ((int64_t)chunk * 2 + (before ? 0 : 1)) * p.D + j, a);
                }
            }
#pragma unroll
            for (int c = 0; c < VEC; ++c) a[c] = 0.0f;
            first = false;
        }
    }
}

// A run that crosses chunks: its first chunk's part 1, then part 0 of the
// chunks behind it, in their order.
template <int VEC>
__global__ void __launch_bounds__(256) embed_join_kernel(SumArgs p, int64_t units, int slices) {
    const int lane = threadIdx.x & 31;
    const int64_t u = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (u >= units) return;
    const int chunk = (int)(u / slices);
    const int j = (int)(u - (int64_t)chunk * slices) * (32 * VEC) + lane * VEC;
    const int end = (chunk + 1) * CH;  // first position behind the chunk
    if (end >= p.n) return;
    const uint32_t key = p.list[end - 1].x;
    if (key == (uint32_t)p.rows || p.list[end].x != key) return;
    // does the run begin in this chunk?
    if (p.list[chunk * CH].x == key && chunk > 0 && p.list[chunk * CH - 1].x == key) return;
    float a[VEC];
    if (j < p.D) load_vec<VEC>(p.part + ((int64_t)chunk * 2 + 1) * p.D + j, a);
    for (int c = chunk + 1;; ++c) {
        float v[VEC];
        if (j < p.D) {
            load_vec<VEC>(p.part + (int64_t)c * 2 * p.D + j, v);
#pragma unroll
            for (int q = 0; q < VEC; ++q) a[q] += v[q];
        }
        const int64_t behind = (int64_t)(c + 1) * CH;
        if (behind >= p.n || p.list[behind].x != key) break;
    }
    if (j < p.D) write_row<VEC>(p, key, j, a);
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
    const int pieces = (p.D + 128 * VEC - 1) / (128 * VEC);
    const int64_t want = (p.n * pieces + 7) / 8;
    embed_kernel<VEC><<<(unsigned)std::min<int64_t>(want, INT32_MAX), 256, 0, s>>>(p, pieces);
    count_launch();
    return check_launch(kFwd);
}

template <int VEC>
int launch_sums(const SumArgs& p, cudaStream_t s) {
    const int slices = (p.D + 32 * VEC - 1) / (32 * VEC);
    const int64_t units = (int64_t)((p.n + CH - 1) / CH) * slices;
    const int64_t blocks = (units + 7) / 8;
    if (blocks > INT32_MAX) return set_error(TLC_ERR_UNSUPPORTED, "embedding_backward: too many tokens");
    embed_sum_kernel<VEC><<<(unsigned)blocks, 256, 0, s>>>(p, units, slices);
    count_launch();
    TLC_TRY(check_launch(kBwd));
    embed_join_kernel<VEC><<<(unsigned)blocks, 256, 0, s>>>(p, units, slices);
    count_launch();
    return check_launch(kBwd);
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
    if (!accumulate) TLC_TRY(launch_fill_zero(dweight->data, vd.numel, s));
    if (n == 0) return TLC_OK;
    RowScratch cg(s), cl(s), cp(s);
    TLC_TRY(unit_rows(grad, vg, cg));
    TLC_TRY(scratch_alloc(&cl.p, sizeof(uint2) * 2 * (size_t)n, s));
    SortArgs q{};
    q.tok = tok;
    q.rows = vd.rows;
    q.n = (int)n;
    int width = 1;  // bits of the largest key, vd.rows
    while ((vd.rows >> width) != 0) ++width;
    q.passes = (width + MAX_BITS - 1) / MAX_BITS;
    q.bits = (width + q.passes - 1) / q.passes;
    q.a = static_cast<uint2*>(cl.p);
    q.b = q.a + n;
    static DeviceOnce once;
    TLC_TRY(smem_limit_once(once, embed_sort_kernel, (int)sizeof(SortSmem)));
    embed_sort_kernel<<<CL, SORT_T, sizeof(SortSmem), s>>>(q);
    count_launch();
    TLC_TRY(check_launch(kBwd));
    SumArgs p{};
    p.list = (q.passes & 1) ? q.a : q.b;
    p.g = vg.data;
    p.gm = vg.map;
    p.dw = dweight->data;
    p.rows = vd.rows;
    p.n = (int)n;
    p.D = (int)vd.cols;
    p.accumulate = accumulate != 0;
    p.scale = scale;
    const int64_t chunks = (n + CH - 1) / CH;
    TLC_TRY(scratch_alloc(&cp.p, sizeof(float) * 2 * (size_t)chunks * (size_t)p.D, s));
    p.part = cp.f();
    const bool vec = p.D % 4 == 0 && vg.map.multiple_of(4) && aligned_to(p.g, 16) && aligned_to(p.dw, 16);
    return vec ? launch_sums<4>(p, s) : launch_sums<1>(p, s);
}
