// Shared by the row operators (layer norm, embedding, token log-probabilities):
// tensors [..., D] seen as rows, with any strides over the leading dims, their
// argument checks, and sums over a warp or a block.
#pragma once

#include <string>

#include "common.cuh"

namespace tlc {

// Row (or element) number -> element offset: the leading dims of a view,
// those that walk as one merged into one (almost always one is left).
struct Rows {
    int nd = 0;
    int64_t sz[TLC_MAX_DIMS] = {};
    int64_t st[TLC_MAX_DIMS] = {};
    __host__ __device__ __forceinline__ int64_t offset(int64_t r) const {
        if (nd <= 1) return r * st[0];
        int64_t o = 0;
        for (int d = nd - 1; d > 0; --d) {
            const int64_t q = r / sz[d];
            o += (r - q * sz[d]) * st[d];
            r = q;
        }
        return o + r * st[0];
    }
    // Whether every row starts at a multiple of `m` elements from the first.
    bool multiple_of(int64_t m) const {
        for (int d = 0; d < nd; ++d)
            if (sz[d] > 1 && st[d] % m != 0) return false;
        return true;
    }
};

inline Rows merge_rows(int nd, const int64_t* sz, const int64_t* st) {
    Rows m;
    for (int d = 0; d < nd; ++d) {
        if (sz[d] == 1) continue;
        if (m.nd > 0 && m.st[m.nd - 1] == st[d] * sz[d]) {
            m.sz[m.nd - 1] *= sz[d];
            m.st[m.nd - 1] = st[d];
            continue;
        }
        m.sz[m.nd] = sz[d];
        m.st[m.nd] = st[d];
        ++m.nd;
    }
    return m;
}

inline bool aligned_to(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// Token numbers on the device, 32 or 64 bits each.
struct TokenRef {
    const void* data = nullptr;
    int wide = 0;  // 64 bits
    Rows map;
    __device__ __forceinline__ int64_t get(int64_t i) const {
        const int64_t o = map.offset(i);
        return wide ? static_cast<const int64_t*>(data)[o] : static_cast<int64_t>(static_cast<const int32_t*>(data)[o]);
    }
    // N tokens, those with in[k] (-1 for the others).  All loads are issued before the first is
    // waited for, which a loop over get() with its branches does not get from the compiler.
    template <int N>
    __device__ __forceinline__ void get(const int64_t (&i)[N], const bool (&in)[N], int64_t (&t)[N]) const {
        int64_t o[N];
        if (map.nd <= 1) {
#pragma unroll
            for (int k = 0; k < N; ++k) o[k] = i[k] * map.st[0];
        } else {
#pragma unroll
            for (int k = 0; k < N; ++k) o[k] = in[k] ? map.offset(i[k]) : 0;
        }
        if (wide) {
#pragma unroll
            for (int k = 0; k < N; ++k) t[k] = in[k] ? static_cast<const int64_t*>(data)[o[k]] : -1;
        } else {
#pragma unroll
            for (int k = 0; k < N; ++k) t[k] = in[k] ? static_cast<const int32_t*>(data)[o[k]] : -1;
        }
    }
    // The tokens first + k * step below end.
    template <int N>
    __device__ __forceinline__ void get(int64_t first, int64_t step, int64_t end, int64_t (&t)[N]) const {
        int64_t i[N];
        bool in[N];
#pragma unroll
        for (int k = 0; k < N; ++k) i[k] = first + k * step, in[k] = i[k] < end;
        get(i, in, t);
    }
};

// ---- argument checks (host) ----------------------------------------------------------

// Scratch that is given back to the stream's pool on every return path.
struct RowScratch {
    void* p = nullptr;
    cudaStream_t s;
    explicit RowScratch(cudaStream_t st) : s(st) {}
    ~RowScratch() { scratch_free(p, s); }
    RowScratch(const RowScratch&) = delete;
    RowScratch& operator=(const RowScratch&) = delete;
    float* f() const { return static_cast<float*>(p); }
};

// The memory that a view touches, to refuse outputs that lie over inputs.
struct Extent {
    uintptr_t lo = 0, hi = 0;  // [lo, hi); empty: lo == hi
    bool overlaps(const Extent& o) const { return lo < hi && o.lo < o.hi && lo < o.hi && o.lo < hi; }
};

// A refusal, and its message "op: name<what>" (built only then: small calls are bound by the host).
inline int bad(const char* op, const char* name, const char* what) {
    return set_error(TLC_ERR_INVALID_ARGUMENT, std::string(op) + ": " + name + what);
}

// Checks of one view (`bytes` an element): rank 1..8 (or 0), sizes and strides
// not negative, a size that fits, an address that is aligned and not NULL.
inline int check_view(const char* op, const char* name, const void* data, int ndim, const int64_t* sizes,
                      const int64_t* strides, int min_nd, int bytes, int64_t* numel, Extent* ext) {
    if (ndim < min_nd || ndim > TLC_MAX_DIMS)
        return bad(op, name, (": ndim must be " + std::to_string(min_nd) + ".." + std::to_string(TLC_MAX_DIMS)).c_str());
    int64_t n = 1;
    bool empty = false;
    for (int i = 0; i < ndim; ++i) {
        if (sizes[i] < 0) return bad(op, name, ": negative size");
        if (strides[i] < 0) return bad(op, name, ": negative stride");
        empty = empty || sizes[i] == 0;
    }
    int64_t last = 0;
    for (int i = 0; i < ndim && !empty; ++i) {
        int64_t step;
        if (__builtin_mul_overflow(n, sizes[i], &n) || __builtin_mul_overflow(sizes[i] - 1, strides[i], &step) ||
            __builtin_add_overflow(last, step, &last) || n > INT64_MAX / 16 || last > INT64_MAX / 16)
            return bad(op, name, ": too large");
    }
    *numel = empty ? 0 : n;
    if (!empty) {
        if (!data) return bad(op, name, ": NULL data");
        if (!aligned_to(data, (size_t)bytes)) return bad(op, name, ": misaligned data");
    }
    ext->lo = reinterpret_cast<uintptr_t>(data);
    ext->hi = empty ? ext->lo : ext->lo + (uintptr_t)(last + 1) * (uintptr_t)bytes;
    return TLC_OK;
}

inline bool dense_strides(int nd, const int64_t* sz, const int64_t* st) {
    int64_t e = 1;
    for (int i = 0; i < nd; ++i)
        if (sz[i] == 0) return true;
    for (int i = nd - 1; i >= 0; --i) {
        if (sz[i] != 1 && st[i] != e) return false;
        e *= sz[i];
    }
    return true;
}

// A float input [..., cols] as rows.
struct RowView {
    const float* data = nullptr;
    int64_t rows = 0, cols = 0, numel = 0;
    Rows map;
    Extent ext;
};

inline int row_view(const tlc_tensor* t, const char* op, const char* name, RowView& v) {
    if (!t) return bad(op, name, " is NULL");
    TLC_TRY(check_view(op, name, t->data, t->ndim, t->sizes, t->strides, 1, 4, &v.numel, &v.ext));
    v.data = t->data;
    v.cols = t->sizes[t->ndim - 1];
    v.rows = 1;
    for (int i = 0; i + 1 < t->ndim; ++i) v.rows = v.numel ? v.rows * t->sizes[i] : v.rows;
    if (!v.numel) {  // an empty view still has rows when only its last dim is 0
        v.rows = 1;
        for (int i = 0; i + 1 < t->ndim; ++i)
            if (__builtin_mul_overflow(v.rows, t->sizes[i], &v.rows))
                return bad(op, name, ": too large");
    }
    v.map = merge_rows(t->ndim - 1, t->sizes, t->strides);
    return TLC_OK;
}

// Gives the view's rows a last dim of stride 1, by a dense copy in `sc` where
// it has another (as the other operators of the library do).
inline int unit_rows(const tlc_tensor* t, RowView& v, RowScratch& sc) {
    if (v.numel == 0 || v.cols <= 1 || t->strides[t->ndim - 1] == 1) return TLC_OK;
    TLC_TRY(scratch_alloc(&sc.p, sizeof(float) * (size_t)v.numel, sc.s));
    TLC_TRY(launch_strided_copy(v.data, t->ndim, t->sizes, t->strides, sc.f(), sc.s));
    v.data = sc.f();
    v.map = Rows{};
    if (v.rows > 1) {
        v.map.nd = 1;
        v.map.sz[0] = v.rows;
        v.map.st[0] = v.cols;
    }
    return TLC_OK;
}

// A float input or output of exactly this shape; `contiguous` for outputs.
inline int shaped(const tlc_tensor* t, const char* op, const char* name, int nd, const int64_t* sizes,
                  bool contiguous, Extent* ext) {
    if (!t) return bad(op, name, " is NULL");
    bool same = t->ndim == nd;
    for (int i = 0; same && i < nd; ++i) same = t->sizes[i] == sizes[i];
    if (!same) return bad(op, name, ": wrong shape");
    int64_t n;
    TLC_TRY(check_view(op, name, t->data, t->ndim, t->sizes, t->strides, 0, 4, &n, ext));
    if (contiguous && !dense_strides(nd, t->sizes, t->strides))
        return bad(op, name, " must be contiguous");
    return TLC_OK;
}

inline int index_view(const tlc_index* t, const char* op, const char* name, TokenRef& r, int64_t* numel, Extent* ext) {
    if (!t) return bad(op, name, " is NULL");
    if (t->bits != 32 && t->bits != 64) return bad(op, name, ": bits must be 32 or 64");
    TLC_TRY(check_view(op, name, t->data, t->ndim, t->sizes, t->strides, 0, t->bits / 8, numel, ext));
    r.data = t->data;
    r.wide = t->bits == 64;
    r.map = merge_rows(t->ndim, t->sizes, t->strides);
    return TLC_OK;
}

// Refuses an output that lies over an input (or another output).
inline int no_overlap(const char* op, const char* out_name, const Extent& out, const char* in_name, const Extent& in) {
    if (!out.overlaps(in)) return TLC_OK;
    return set_error(TLC_ERR_INVALID_ARGUMENT, std::string(op) + ": " + out_name + " overlaps " + in_name);
}

inline int sm_count() {
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0)
        return 148;
    return sms;
}

// A launch whose blocks may be set up while the kernel before it on the stream
// still runs; the kernel begins with after_previous().
template <class K, class... A>
int launch_after(K kernel, unsigned grid, unsigned block, cudaStream_t s, const char* what, A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    TLC_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, args...));
    count_launch();
    return check_launch(what);
}

// ---- device helpers --------------------------------------------------------------------

// Waits until the kernel before this one has ended and its writes are visible
// (see launch_after; nothing of that kernel's may be touched before).
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// Lets the next kernel's blocks be set up from here on.
__device__ __forceinline__ void next_may_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// VEC floats at p (16-byte aligned where VEC is 4).  load_once, store_once: streaming.
template <int VEC>
__device__ __forceinline__ void load_vec(const float* p, float (&v)[VEC]) {
    if constexpr (VEC == 4) {
        const float4 t = *reinterpret_cast<const float4*>(p);
        v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
    } else {
        v[0] = *p;
    }
}
template <int VEC>
__device__ __forceinline__ void load_once(const float* p, float (&v)[VEC]) {
    if constexpr (VEC == 4) {
        const float4 t = __ldcs(reinterpret_cast<const float4*>(p));
        v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
    } else {
        v[0] = __ldcs(p);
    }
}
template <int VEC>
__device__ __forceinline__ void store_vec(float* p, const float (&v)[VEC]) {
    if constexpr (VEC == 4)
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    else
        *p = v[0];
}

template <int VEC>
__device__ __forceinline__ void store_once(float* p, const float (&v)[VEC]) {
    if constexpr (VEC == 4)
        __stcs(reinterpret_cast<float4*>(p), make_float4(v[0], v[1], v[2], v[3]));
    else
        __stcs(p, v[0]);
}

// Two floats in one 64-bit register pair: one instruction for both.
using Pair = unsigned long long;
__device__ __forceinline__ Pair pair(float lo, float hi) {
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(lo), "f"(hi));
    return p;
}
__device__ __forceinline__ void unpair(Pair p, float& lo, float& hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(p));
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    Pair d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    Pair d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}

// Sums of N values over LANES neighbouring lanes, in each of them.
template <int LANES = 32, int N>
__device__ __forceinline__ void warp_sum(float (&v)[N]) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1)
#pragma unroll
        for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
}

// Sums of N values over THREADS threads (at most 32: neighbouring lanes; else
// the whole block), in every thread.  `red` holds THREADS / 32 * N floats that
// nobody else uses until all threads have passed one more block barrier.  FEW:
// only as many lanes as there are warps meet at the end: fewer shuffles, some registers.
template <int THREADS, bool FEW = false, int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float* red) {
    if constexpr (THREADS <= 32) {
        warp_sum<THREADS>(v);
    } else {
        warp_sum(v);
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        if (lane == 0)
#pragma unroll
            for (int n = 0; n < N; ++n) red[warp * N + n] = v[n];
        __syncthreads();
#pragma unroll
        for (int n = 0; n < N; ++n)
            v[n] = FEW ? red[lane % (THREADS / 32) * N + n] : lane < THREADS / 32 ? red[lane * N + n] : 0.0f;
        warp_sum<FEW ? THREADS / 32 : 32>(v);
    }
}

}  // namespace tlc
