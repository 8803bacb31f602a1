// Global gradient norm over many tensors, and clipping by it or by value.
//
//   norm = sqrt(sum over all tensors of g^2),  factor = min(1, max_norm / (norm + 1e-6)),  out = factor g
//
// The tensors are cut into tiles of CL_VECS 16-byte vectors; a launch takes up to CL_MOST tensors, their addresses and sizes by
// value in the kernel's arguments (no table in memory that would have to outlive the call or be copied into a captured
// graph).  Squares are summed in fp64: exact products, no overflow, and at 6 TB/s still far below the fp64 rate.  Every tile leaves
// its sum in the workspace; norm_final_kernel adds them in tile order, so the result does not depend on the order of execution.
#include "common.h"

#include <algorithm>
#include <new>
#include <type_traits>

namespace {

constexpr int CL_MOST = 128;           // tensors of a launch (28 bytes each of the 4 KiB of kernel arguments)
constexpr int CL_VECS = 4096;          // 16-byte vectors of a tile (64 KiB)
constexpr int CL_THREADS = 256;
constexpr int CL_DEEP = 8;             // vectors a thread has in flight
// Tiles at the list's end that the norm reads into the caches for the scaling, which begins there (192 MiB of the 256 MiB that the
// memory-side cache holds).  The tiles in front of them, and what scaling reads last and writes into other tensors, go past
// the caches: 365M fp32 values 821 -> 763 us.  64M bf16 values, 134 MB, take 82 us in place where lists come in turn (norm 37, scaling 40),
// 69 into other tensors, 64 where the list is still in the caches.
constexpr int CL_KEEP = (192 << 20) / (CL_VECS * 16);

struct ClipArgs {
    const void* in[CL_MOST];
    void* out[CL_MOST];
    long long n[CL_MOST];
    int first[CL_MOST];  // the tensor's first tile, counted from the launch's first
    int count;
    double* partial;     // the launch's first tile's
    int keep;            // the launch's first tile that the norm reads into the caches
    const float* factor; // NULL: every workgroup adds the `tiles` sums itself
    const double* sums;
    int tiles;
    float* norm;
    float limit;         // scaling: max_norm; by value: clamp to [-limit, limit]
};

template <typename T> struct Vec;
template <> struct Vec<float> {
    static constexpr int N = 4;
    typedef f32x4 __attribute__((aligned(4))) V;
    static __device__ __forceinline__ float get(const float* p) { return *p; }
    static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
    static __device__ __forceinline__ void unpack(const f32x4& v, float* f) { f[0] = v[0]; f[1] = v[1]; f[2] = v[2]; f[3] = v[3]; }
    static __device__ __forceinline__ f32x4 pack(const float* f) { return f32x4{f[0], f[1], f[2], f[3]}; }
    typedef f32x4 R;
};
template <> struct Vec<unsigned short> {
    static constexpr int N = 8;
    typedef u32x4 __attribute__((aligned(2))) V;
    static __device__ __forceinline__ float get(const unsigned short* p) { return bf16_bits_to_f32(*p); }
    static __device__ __forceinline__ void put(unsigned short* p, float v) { *p = f32_to_bf16_bits(v); }
    static __device__ __forceinline__ void unpack(const u32x4& v, float* f) { unpack8(v, f); }
    static __device__ __forceinline__ u32x4 pack(const float* f) { return pack8(f); }
    typedef u32x4 R;
};

// elements in front of the first 16-byte boundary of a tensor, and its whole vectors behind it
template <typename T>
__host__ __device__ __forceinline__ long long head_of(const void* p, long long n) {
    const long long h = (long long)((16 - ((uintptr_t)p & 15)) & 15) / (long long)sizeof(T);
    return h < n ? h : n;
}
template <typename T>
__host__ __device__ __forceinline__ long long tiles_of(const void* p, long long n) {
    const long long vecs = (n - head_of<T>(p, n)) / (16 / (long long)sizeof(T));
    const long long t = (vecs + CL_VECS - 1) / CL_VECS;
    return n == 0 ? 0 : t > 0 ? t : 1;
}

// the tensor of tile `tile` of the launch: the last one whose first tile is not behind it (tensors without elements have none)
__device__ __forceinline__ int tensor_of(const ClipArgs& a, int tile) {
    int lo = 0, hi = a.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.first[mid] <= tile) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Sum of squares of a tile: CL_DEEP 16-byte loads in flight a thread, an fp64 sum for each of a vector's elements, one write a workgroup.
// Bound by memory: 365M fp32 values in three launches 221 us = 6.6 TB/s; 40 small tensors 3.7 us, the launch.
template <typename T>
__global__ __launch_bounds__(CL_THREADS) void norm_tile_kernel(const ClipArgs a) {
    typedef Vec<T> X;
    const int k = tensor_of(a, blockIdx.x), tile = blockIdx.x - a.first[k];
    const T* p = (const T*)a.in[k];
    const long long n = a.n[k], head = head_of<T>(p, n), vecs = (n - head) / X::N;
    const long long v0 = (long long)tile * CL_VECS, v1 = min(vecs, v0 + CL_VECS);
    const typename X::R* body = (const typename X::R*)(p + head);
    double s[X::N] = {};
    auto add = [&](const typename X::R& r) {
        float f[X::N];
        X::unpack(r, f);
#pragma unroll
        for (int e = 0; e < X::N; ++e) s[e] = fma((double)f[e], (double)f[e], s[e]);
    };
    auto walk = [&](auto past_c) {  // (a loop each: merged accesses lose their cache hint)
        constexpr bool PAST = decltype(past_c)::value;
        long long v = v0 + threadIdx.x;
        for (; v + (CL_DEEP - 1) * CL_THREADS < v1; v += CL_DEEP * CL_THREADS) {
            typename X::R r[CL_DEEP];
#pragma unroll
            for (int u = 0; u < CL_DEEP; ++u) r[u] = PAST ? __builtin_nontemporal_load(body + v + u * CL_THREADS) : body[v + u * CL_THREADS];
#pragma unroll
            for (int u = 0; u < CL_DEEP; ++u) add(r[u]);
        }
        for (; v < v1; v += CL_THREADS) add(body[v]);
    };
    if ((int)blockIdx.x >= a.keep) walk(std::false_type{});
    else walk(std::true_type{});
    if (tile == 0) {  // what lies outside the whole vectors: at most N - 1 elements on either side
        const long long tail = head + vecs * X::N;
        const long long i = threadIdx.x < head ? (long long)threadIdx.x : tail + ((long long)threadIdx.x - head);
        if (i < n) {
            const double f = X::get(p + i);
            s[0] = fma(f, f, s[0]);
        }
    }
    double t = 0;
#pragma unroll
    for (int e = 0; e < X::N; ++e) t += s[e];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o);
    __shared__ double red[CL_THREADS / 64];
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = t;
    __syncthreads();
    if (threadIdx.x == 0) a.partial[blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// the sum of the tiles' sums in a fixed order, in every thread (blockDim.x a multiple of 64, at most 1024)
__device__ __forceinline__ double all_sum(const double* sums, int n) {
    double t = 0;
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += blockDim.x) t += sums[i];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o);
    __shared__ double red[16];
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = t;
    __syncthreads();
    double s = 0;
    for (int i = 0; i < (int)blockDim.x / 64; ++i) s += red[i];
    return s;
}
// a norm that is not finite scales nothing: the caller sees it and skips its step
__device__ __forceinline__ float factor_of(double norm, float max_norm) {
    const float f = (float)((double)max_norm / (norm + 1e-6));
    return (float)norm <= 3.4028235e38f && f < 1.0f ? f : 1.0f;
}

// One workgroup, the tiles' sums in their order (22468 of them: 8.8 us, the latency of 22 loads a thread and the reduction).
__global__ __launch_bounds__(1024) void norm_final_kernel(const double* sums, int n, float max_norm, float* norm, float* factor) {
    const double r = sqrt(all_sum(sums, n));
    if (threadIdx.x == 0) {
        *norm = (float)r;
        if (factor) *factor = factor_of(r, max_norm);
    }
}

// out = factor g, a tile a workgroup.  Bound by memory: 365M fp32 values into other tensors 528 us for 2.9 GB = 5.5 TB/s (a copy of
// 2 GiB 4.9), from the list's end, which the norm has left in the cache; 40 small tensors 3.5 us.
template <typename T, bool VALUE>
__global__ __launch_bounds__(CL_THREADS) void clip_tile_kernel(const ClipArgs a) {
    typedef Vec<T> X;
    const int at = gridDim.x - 1 - blockIdx.x;  // the tiles that the norm read last, and the cache may still hold, first
    const int k = tensor_of(a, at), tile = at - a.first[k];
    const T* p = (const T*)a.in[k];
    T* q = (T*)a.out[k];
    const float lim = a.limit;
    float f = 1.0f;
    if constexpr (!VALUE) {
        if (a.factor) {
            f = *a.factor;
        } else {
            const double r = sqrt(all_sum(a.sums, a.tiles));
            f = factor_of(r, lim);
            if (a.norm && blockIdx.x == 0 && threadIdx.x == 0) *a.norm = (float)r;
        }
    }
    if (!VALUE && f == 1.0f && p == q) return;
    // (a NaN stays one: it compares with neither limit)
    auto one = [&](float v) { return VALUE ? (v > lim ? lim : v < -lim ? -lim : v) : v * f; };
    const long long n = a.n[k], head = head_of<T>(p, n), vecs = (n - head) / X::N;
    const long long v0 = (long long)tile * CL_VECS, v1 = min(vecs, v0 + CL_VECS);
    const typename X::R* body = (const typename X::R*)(p + head);
    auto walk = [&](auto apart_c, auto past_c) {
        constexpr bool APART = decltype(apart_c)::value, PAST = decltype(past_c)::value;
        auto put = [&](long long v, const typename X::R& r) {
            float x[X::N];
            X::unpack(r, x);
#pragma unroll
            for (int e = 0; e < X::N; ++e) x[e] = one(x[e]);
            typename X::V* to = (typename X::V*)(q + head + v * X::N);  // (the output may be aligned to its elements only)
            if constexpr (APART) __builtin_nontemporal_store(X::pack(x), to);
            else *to = X::pack(x);
        };
        long long v = v0 + threadIdx.x;
        for (; v + (CL_DEEP - 1) * CL_THREADS < v1; v += CL_DEEP * CL_THREADS) {
            typename X::R r[CL_DEEP];
#pragma unroll
            for (int u = 0; u < CL_DEEP; ++u) r[u] = PAST ? __builtin_nontemporal_load(body + v + u * CL_THREADS) : body[v + u * CL_THREADS];
#pragma unroll
            for (int u = 0; u < CL_DEEP; ++u) put(v + u * CL_THREADS, r[u]);
        }
        for (; v < v1; v += CL_THREADS) put(v, body[v]);
    };
    if (p == q) walk(std::false_type{}, std::false_type{});
    else if (at >= a.keep) walk(std::true_type{}, std::false_type{});
    else walk(std::true_type{}, std::true_type{});
    if (tile == 0) {
        const long long tail = head + vecs * X::N;
        const long long i = threadIdx.x < head ? (long long)threadIdx.x : tail + ((long long)threadIdx.x - head);
        if (i < n) X::put(q + i, one(X::get(p + i)));
    }
}

// fills the launches of the tensors [i, count) in turn: launch(args, first tile of all, tiles)
template <typename T, typename F>
int each_launch(const void* const* in, void* const* out, const int64_t* numel, int i, int count, F launch) {
    long long before = 0;
    while (i < count) {
        ClipArgs a{};
        long long tiles = 0;
        while (i < count && a.count < CL_MOST) {
            const long long t = tiles_of<T>(in[i], numel[i]);
            if (t == 0) { ++i; continue; }
            if (tiles + t > 0x7fffffffLL) {
                if (a.count == 0) return CCNET_EUNSUP;
                break;
            }
            a.in[a.count] = in[i];
            a.out[a.count] = out ? out[i] : nullptr;
            a.n[a.count] = numel[i];
            a.first[a.count] = (int)tiles;
            ++a.count;
            tiles += t;
            ++i;
        }
        if (a.count == 0) break;
        launch(a, before, (unsigned)tiles);
        CCNET_LAUNCH_CHECK();
        before += tiles;
    }
    return CCNET_OK;
}

bool list_ok(const void* const* p, const int64_t* numel, int count, int esz) {
    if (count < 0 || (count > 0 && (!p || !numel))) return false;
    for (int i = 0; i < count; ++i)
        if (numel[i] < 0 || (numel[i] > 0 && (!p[i] || (uintptr_t)p[i] % esz))) return false;
    return true;
}

template <typename T>
int norm_launches(const void* const* g, const int64_t* numel, int count, long long tiles_all, double* ws, hipStream_t st) {
    return each_launch<T>(g, nullptr, numel, 0, count, [&](ClipArgs& a, long long before, unsigned tiles) {
        a.partial = ws + 1 + before;
        const long long keep = tiles_all - CL_KEEP - before;
        a.keep = keep > 0 ? (int)std::min<long long>(keep, 0x7fffffff) : 0;
        hipLaunchKernelGGL(norm_tile_kernel<T>, dim3(tiles), dim3(CL_THREADS), 0, st, a);
    });
}
template <typename T, bool VALUE>
int clip_launches(const void* const* g, void* const* out, const int64_t* numel, int count, const float* factor, const double* sums, int tiles_all,
                  float* norm, float limit, hipStream_t st) {
    long long left = tiles_all;
    for (int end = count; end > 0;) {  // the list from its end, as the tiles of a launch
        const int begin = end > CL_MOST ? end - CL_MOST : 0;
        for (int i = begin; i < end; ++i) left -= tiles_of<T>(g[i], numel[i]);
        const int rc = each_launch<T>(g, out, numel, begin, end, [&](ClipArgs& a, long long before, unsigned tiles) {
            const long long keep = VALUE ? 0 : tiles_all - CL_KEEP - left - before;
            a.keep = keep > 0 ? (int)keep : 0;
            a.factor = factor;
            a.sums = sums;
            a.tiles = tiles_all;
            a.norm = norm;
            a.limit = limit;
            norm = nullptr;  // (one launch writes it)
            hipLaunchKernelGGL((clip_tile_kernel<T, VALUE>), dim3(tiles), dim3(CL_THREADS), 0, st, a);
        });
        if (rc != CCNET_OK) return rc;
        end = begin;
    }
    return CCNET_OK;
}

// Whether no two of the tensors written overlap, and none of them a tensor read other than its own whole.
struct Span { uintptr_t lo, hi; int i; };
int aliases_ok(const void* const* in, void* const* out, const int64_t* numel, int count, int esz) {
    if (count == 0) return CCNET_OK;
    Span* s = new (std::nothrow) Span[2 * (size_t)count];
    if (!s) return CCNET_EWS;
    Span* r = s + count;
    int n = 0;
    bool apart = false;
    for (int i = 0; i < count; ++i) {
        if (numel[i] == 0) continue;
        s[n] = Span{(uintptr_t)out[i], (uintptr_t)out[i] + (uintptr_t)numel[i] * esz, i};
        r[n++] = Span{(uintptr_t)in[i], (uintptr_t)in[i] + (uintptr_t)numel[i] * esz, i};
        apart |= out[i] != in[i];
    }
    auto less = [](const Span& a, const Span& b) { return a.lo < b.lo; };
    std::sort(s, s + n, less);
    bool ok = true;
    for (int i = 0; i + 1 < n; ++i) ok &= s[i].hi <= s[i + 1].lo;
    for (int i = 0; ok && apart && i < n; ++i) {  // the written spans are disjoint: the ones that touch r[i] are neighbours
        Span* w = std::lower_bound(s, s + n, r[i], [](const Span& a, const Span& b) { return a.hi <= b.lo; });
        for (; w != s + n && w->lo < r[i].hi; ++w) ok &= w->i == r[i].i && w->lo == r[i].lo;
    }
    delete[] s;
    return ok ? CCNET_OK : CCNET_EINVAL;
}

// Whether the norm and the workspace (its `bytes` in use) lie apart from each other and from every tensor of the lists.
bool norm_apart(const void* const* in, void* const* out, const int64_t* numel, int count, int esz, const void* workspace, size_t bytes, const float* norm) {
    auto range = [](const void* p, long long n) { return RowSpan{p, n, n, n > 0}; };
    const RowSpan ws = range(workspace, (long long)bytes), to = range(norm, 4);
    bool ok = spans_apart(ws, to);
    for (int i = 0; i < count; ++i)
        for (const void* p : {in[i], out ? (const void*)out[i] : in[i]}) {
            const RowSpan t = range(p, numel[i] * esz);
            ok &= spans_apart(ws, t) && spans_apart(to, t);
        }
    return ok;
}

long long all_tiles(const void* const* g, const int64_t* numel, int count, int dtype) {
    long long t = 0;
    for (int i = 0; i < count; ++i) t += dtype == 0 ? tiles_of<float>(g[i], numel[i]) : tiles_of<unsigned short>(g[i], numel[i]);
    return t;
}

}  // namespace

extern "C" size_t ccnet_grad_norm_workspace_bytes(const void* const* grads, const int64_t* numel, int count, int dtype) {
    if ((dtype != 0 && dtype != 1) || !list_ok(grads, numel, count, dtype == 0 ? 4 : 2)) return 0;
    return 8 * (size_t)(1 + all_tiles(grads, numel, count, dtype));
}

extern "C" int ccnet_grad_norm(const void* const* grads, const int64_t* numel, int count, int dtype, void* workspace,
                               size_t workspace_bytes, float* norm, void* stream) {
    if ((dtype != 0 && dtype != 1) || !norm || !list_ok(grads, numel, count, dtype == 0 ? 4 : 2)) return CCNET_EINVAL;
    const long long tiles = all_tiles(grads, numel, count, dtype);
    if (tiles > 0x7fffffffLL) return CCNET_EUNSUP;
    if (!workspace || ((uintptr_t)workspace & 7) || ((uintptr_t)norm & 3)) return CCNET_EINVAL;
    if (workspace_bytes < 8 * (size_t)(1 + tiles)) return CCNET_EWS;
    if (!norm_apart(grads, nullptr, numel, count, dtype == 0 ? 4 : 2, workspace, 8 * (size_t)(1 + tiles), norm)) return CCNET_EINVAL;
    hipStream_t st = (hipStream_t)stream;
    double* ws = (double*)workspace;
    const int rc = dtype == 0 ? norm_launches<float>(grads, numel, count, tiles, ws, st) : norm_launches<unsigned short>(grads, numel, count, tiles, ws, st);
    if (rc != CCNET_OK) return rc;
    hipLaunchKernelGGL(norm_final_kernel, dim3(1), dim3(1024), 0, st, ws + 1, (int)tiles, 0.f, norm, (float*)nullptr);
    CCNET_LAUNCH_CHECK();
    return CCNET_OK;
}

extern "C" int ccnet_clip_grad_norm(const void* const* grads, void* const* out, const int64_t* numel, int count, int dtype,
                                    float max_norm, void* workspace, size_t workspace_bytes, float* norm, void* stream) {
    const int esz = dtype == 0 ? 4 : 2;
    if ((dtype != 0 && dtype != 1) || !norm || !(max_norm >= 0.f) || !list_ok(grads, numel, count, esz) ||
        !list_ok((const void* const*)out, numel, count, esz))
        return CCNET_EINVAL;
    int rc = aliases_ok(grads, out, numel, count, esz);
    if (rc != CCNET_OK) return rc;
    const long long tiles = all_tiles(grads, numel, count, dtype);
    if (tiles > 0x7fffffffLL) return CCNET_EUNSUP;
    if (!workspace || ((uintptr_t)workspace & 7) || ((uintptr_t)norm & 3)) return CCNET_EINVAL;
    if (workspace_bytes < 8 * (size_t)(1 + tiles)) return CCNET_EWS;
    if (!norm_apart(grads, out, numel, count, esz, workspace, 8 * (size_t)(1 + tiles), norm)) return CCNET_EINVAL;
    hipStream_t st = (hipStream_t)stream;
    double* ws = (double*)workspace;
    float* factor = (float*)workspace;  // the workspace's first 8 bytes
    rc = dtype == 0 ? norm_launches<float>(grads, numel, count, tiles, ws, st) : norm_launches<unsigned short>(grads, numel, count, tiles, ws, st);
    if (rc != CCNET_OK) return rc;
    // few tiles: the scaling workgroups add their sums themselves, a launch less (40 tensors of up to 1280 values: 8.0 -> 5.9 us); many:
    // one workgroup adds them for all
    const bool own_sum = tiles > 0 && tiles <= 1024;
    if (!own_sum) {
        hipLaunchKernelGGL(norm_final_kernel, dim3(1), dim3(1024), 0, st, ws + 1, (int)tiles, max_norm, norm, factor);
        CCNET_LAUNCH_CHECK();
    }
    const float* fp = own_sum ? nullptr : factor;
    return dtype == 0 ? clip_launches<float, false>(grads, out, numel, count, fp, ws + 1, (int)tiles, norm, max_norm, st)
                      : clip_launches<unsigned short, false>(grads, out, numel, count, fp, ws + 1, (int)tiles, norm, max_norm, st);
}

extern "C" int ccnet_clip_grad_value(const void* const* grads, void* const* out, const int64_t* numel, int count, int dtype,
                                     float limit, void* stream) {
    const int esz = dtype == 0 ? 4 : 2;
    if ((dtype != 0 && dtype != 1) || !(limit >= 0.f) || !list_ok(grads, numel, count, esz) ||
        !list_ok((const void* const*)out, numel, count, esz))
        return CCNET_EINVAL;
    const int rc = aliases_ok(grads, out, numel, count, esz);
    if (rc != CCNET_OK) return rc;
    hipStream_t st = (hipStream_t)stream;
    return dtype == 0 ? clip_launches<float, true>(grads, out, numel, count, nullptr, nullptr, 0, nullptr, limit, st)
                      : clip_launches<unsigned short, true>(grads, out, numel, count, nullptr, nullptr, 0, nullptr, limit, st);
}
