// One norm over all gradients of a step, and their scaling by it:
//     norm = (sum over all tensors and elements of |g|^p)^(1/p), p in {1, 2, inf}
//     coef = min(1, max_norm / (norm + 1e-6)),   g <- round(g * coef)
// Bound by memory: the norm reads every gradient once, the scaling reads and writes it once more.
//
// The list of tensors travels in the kernel arguments (128 per launch): nothing is copied to the device, so a captured
// launch carries its own list.  A tile is 16 KiB of one tensor.  For the norm, workgroups walk over the tiles of all tensors, each
// keeps one running sum and leaves one partial.  Sums are held in 64 bits: a dictionary's gradient has 10^8 elements, and
// squares of fp32 values leave the range of fp32; squaring in fp32 instead measured no faster (60 us for 340 MB either
// way).  The partials are added in a fixed order (no atomics: the same bits on every run).
//
// Scaling.  Up to SMALL_TILES tiles every workgroup adds up the partials for itself, which saves a launch and its wait (61
// tensors of 5 KiB 11 against 15 us, 75 MB 38 against 39); beyond, one workgroup does it once and each tile gets a
// workgroup of its own (1.36 GB 672 against 731 us: neighbouring workgroups then share DRAM pages).  It walks from the
// last tile to the first, because the norm's pass has left the last ones in the Infinity Cache.  Stores are
// non-temporal (340 MB 156 against 190 us; an Adam update right behind is no slower for it), loads only when the list is
// well beyond that cache (1.36 GB 648 against 672 us; 340 MB 161 against 156).
#include <algorithm>
#include <new>
#include "common.hpp"

namespace mtc {

constexpr int CLIP_BATCH = 128;            // tensors per launch (kernel arguments are limited to 4 KiB)
constexpr int TILE_UNITS = 1024;           // 16-byte units per tile: 4 per thread
constexpr int PER_THREAD = TILE_UNITS / 256;
constexpr int CLIP_GRID = 2048;            // workgroups of one launch that walk over tiles
constexpr int LARGE_GRID = 1 << 22;        // a workgroup per tile up to 64 GiB (a launch has at most 2^32 threads)
constexpr int SMALL_TILES = 8192;          // 128 MiB
constexpr uint64_t STREAM_TILES = 32768;   // 512 MiB: twice the Infinity Cache
constexpr float CLIP_EPS = 1e-6f;

enum { POW_1 = 1, POW_2 = 2, POW_INF = 3 };

struct ClipBatch {
    int n, tiles;
    uint32_t first[CLIP_BATCH];            // first tile of each tensor
    const void* src[CLIP_BATCH];
    void* dst[CLIP_BATCH];
    uint64_t elems[CLIP_BATCH];            // bit 63: bf16, bit 62: every address a multiple of 16 bytes
};
static_assert(sizeof(ClipBatch) <= 3800, "the tensor list has to fit the kernel arguments");
constexpr uint64_t ELEM_MASK = (1ull << 62) - 1;

// the tensor a tile belongs to: last t with first[t] <= tile (empty tensors have no tile and are not in the list)
__device__ __forceinline__ int tensor_of(const ClipBatch& b, uint32_t tile) {
    int lo = 0, hi = b.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (b.first[mid] <= tile) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// running sum of one thread; for p = inf the largest |g| by its bits (a NaN's are above every number's)
template <int POW> struct Acc {
    double s = 0.0;
    uint32_t m = 0;
    __device__ __forceinline__ void add(float x) {
        if (POW == POW_INF) m = max(m, __float_as_uint(x) & 0x7fffffffu);
        else if (POW == POW_1) s += (double)fabsf(x);
        else { const double d = (double)x; s = fma(d, d, s); }
    }
    __device__ __forceinline__ double value() const { return POW == POW_INF ? (double)__uint_as_float(m) : s; }
};
template <int POW> __device__ __forceinline__ double join(double a, double b) {
    if (POW == POW_INF) return a != a ? a : b != b ? b : fmax(a, b);
    return a + b;
}

// sum over 256 threads, the same value in all of them
template <int POW> __device__ __forceinline__ double block_join(double v, double* sm) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = join<POW>(v, __shfl_xor(v, o, 64));
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = v;
    __syncthreads();
    return join<POW>(join<POW>(sm[0], sm[1]), join<POW>(sm[2], sm[3]));
}
template <int POW> __device__ __forceinline__ double join_partials(const double* __restrict__ partial, int parts, double* sm) {
    double v = 0.0;
#pragma unroll 8
    for (int i = threadIdx.x; i < parts; i += 256) v = join<POW>(v, partial[i]);
    return block_join<POW>(v, sm);
}
template <int POW> __device__ __forceinline__ float root(double total) { return (float)(POW == POW_2 ? sqrt(total) : total); }
__device__ __forceinline__ float clip_coef(float norm, float max_norm) {
    const float c = max_norm / (norm + CLIP_EPS);
    return c > 1.f ? 1.f : c;              // a NaN norm gives NaN
}

template <int DT> __device__ __forceinline__ void unit_values(u32x4 r, float (&v)[DType<DT>::kVec]) {
    if constexpr (DT == MTC_BF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(r[i] << 16);
            v[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(r[i]);
    }
}
template <int DT> __device__ __forceinline__ u32x4 unit_pack(const float (&v)[DType<DT>::kVec]) {
    u32x4 r;
    if constexpr (DT == MTC_BF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = pack2_bf16(v[2 * i], v[2 * i + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = __float_as_uint(v[i]);
    }
    return r;
}

template <bool STREAM> __device__ __forceinline__ u32x4 load_unit(const u32x4* p) {
    if constexpr (STREAM) return __builtin_nontemporal_load(p);
    else return *p;
}

template <int DT, int POW, bool STREAM>
__device__ __forceinline__ void sum_tile(const void* src, uint64_t n, bool aligned, uint64_t local, Acc<POW>& acc) {
    typedef typename DType<DT>::T T;
    constexpr int E = DType<DT>::kVec;
    const T* p = reinterpret_cast<const T*>(src);
    const uint64_t e0 = local * (uint64_t)(TILE_UNITS * E);
    if (aligned && e0 + TILE_UNITS * E <= n) {
        const u32x4* q = reinterpret_cast<const u32x4*>(p + e0) + threadIdx.x;
        u32x4 r[PER_THREAD];
#pragma unroll
        for (int k = 0; k < PER_THREAD; ++k) r[k] = load_unit<STREAM>(q + k * 256);
#pragma unroll
        for (int k = 0; k < PER_THREAD; ++k) {
            float v[E];
            unit_values<DT>(r[k], v);
#pragma unroll
            for (int i = 0; i < E; ++i) acc.add(v[i]);
        }
        return;
    }
    const uint64_t end = min(n, e0 + TILE_UNITS * E);
    uint64_t i = e0;
    if (aligned) {
        const uint64_t units = (end - e0) / E;
        for (uint64_t u = threadIdx.x; u < units; u += 256) {
            float v[E];
            unit_values<DT>(reinterpret_cast<const u32x4*>(p + e0)[u], v);
#pragma unroll
            for (int k = 0; k < E; ++k) acc.add(v[k]);
        }
        i = e0 + units * E;
    }
    for (i += threadIdx.x; i < end; i += 256) acc.add(DType<DT>::ld(p + i));
}

template <int POW, bool STREAM>
__global__ __launch_bounds__(256) void power_sum_kernel(ClipBatch b, double* __restrict__ partial) {
    __shared__ double sm[4];
    Acc<POW> acc;
    for (uint32_t tile = blockIdx.x; tile < (uint32_t)b.tiles; tile += gridDim.x) {
        const int t = tensor_of(b, tile);
        const uint64_t n = b.elems[t] & ELEM_MASK;
        const bool aligned = (b.elems[t] >> 62) & 1;
        if (b.elems[t] >> 63) sum_tile<MTC_BF16, POW, STREAM>(b.src[t], n, aligned, tile - b.first[t], acc);
        else sum_tile<MTC_F32, POW, STREAM>(b.src[t], n, aligned, tile - b.first[t], acc);
    }
    const double v = block_join<POW>(acc.value(), sm);
    if (threadIdx.x == 0) partial[blockIdx.x] = v;
}

// the partials' total: as it is (to be added up over ranks), as {norm, coef}, as the norm
template <int POW>
__global__ __launch_bounds__(256) void norm_finish_kernel(const double* __restrict__ partial, int parts, float max_norm,
                                                          double* __restrict__ total, float* __restrict__ norm_coef,
                                                          float* __restrict__ norm_out) {
    __shared__ double sm[4];
    const double v = join_partials<POW>(partial, parts, sm);
    if (threadIdx.x) return;
    const float norm = root<POW>(v);
    if (total) *total = v;
    if (norm_coef) {
        norm_coef[0] = norm;
        norm_coef[1] = clip_coef(norm, max_norm);
    }
    if (norm_out) *norm_out = norm;
}

template <int DT, bool STREAM>
__device__ __forceinline__ void scale_tile(const void* src, void* dst, uint64_t n, bool aligned, uint64_t local, float coef) {
    typedef typename DType<DT>::T T;
    constexpr int E = DType<DT>::kVec;
    const T* p = reinterpret_cast<const T*>(src);
    T* o = reinterpret_cast<T*>(dst);
    const uint64_t e0 = local * (uint64_t)(TILE_UNITS * E);
    if (aligned && e0 + TILE_UNITS * E <= n) {
        const u32x4* q = reinterpret_cast<const u32x4*>(p + e0) + threadIdx.x;
        u32x4* w = reinterpret_cast<u32x4*>(o + e0) + threadIdx.x;
        u32x4 r[PER_THREAD];
#pragma unroll
        for (int k = 0; k < PER_THREAD; ++k) r[k] = load_unit<STREAM>(q + k * 256);
#pragma unroll
        for (int k = 0; k < PER_THREAD; ++k) {
            float v[E];
            unit_values<DT>(r[k], v);
#pragma unroll
            for (int i = 0; i < E; ++i) v[i] *= coef;
            __builtin_nontemporal_store(unit_pack<DT>(v), w + k * 256);
        }
        return;
    }
    const uint64_t end = min(n, e0 + TILE_UNITS * E);
    uint64_t i = e0;
    if (aligned) {
        const uint64_t units = (end - e0) / E;
        for (uint64_t u = threadIdx.x; u < units; u += 256) {
            float v[E];
            unit_values<DT>(reinterpret_cast<const u32x4*>(p + e0)[u], v);
#pragma unroll
            for (int k = 0; k < E; ++k) v[k] *= coef;
            reinterpret_cast<u32x4*>(o + e0)[u] = unit_pack<DT>(v);
        }
        i = e0 + units * E;
    }
    for (i += threadIdx.x; i < end; i += 256) DType<DT>::st(o + i, DType<DT>::ld(p + i) * coef);
}

template <bool STREAM>
__device__ __forceinline__ void scale_tiles(const ClipBatch& b, uint32_t k, uint32_t step, float coef) {
    for (; k < (uint32_t)b.tiles; k += step) {
        const uint32_t tile = b.tiles - 1 - k;           // last tiles first
        const int t = tensor_of(b, tile);
        const uint64_t n = b.elems[t] & ELEM_MASK;
        const bool aligned = (b.elems[t] >> 62) & 1;
        if (b.elems[t] >> 63) scale_tile<MTC_BF16, STREAM>(b.src[t], b.dst[t], n, aligned, tile - b.first[t], coef);
        else scale_tile<MTC_F32, STREAM>(b.src[t], b.dst[t], n, aligned, tile - b.first[t], coef);
    }
}

// in place and coef 1: nothing would change, g * 1 is g bit for bit
template <int POW>
__global__ __launch_bounds__(256) void clip_small_kernel(ClipBatch b, const double* __restrict__ partial, int parts, float max_norm,
                                                         int in_place, float* __restrict__ norm_out) {
    __shared__ double sm[4];
    const float norm = root<POW>(join_partials<POW>(partial, parts, sm));
    const float coef = clip_coef(norm, max_norm);
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
    if (in_place && coef == 1.f) return;
    scale_tiles<false>(b, blockIdx.x, gridDim.x, coef);
}

template <bool STREAM>
__global__ __launch_bounds__(256) void clip_large_kernel(ClipBatch b, const float* __restrict__ norm_coef, int in_place) {
    const float coef = norm_coef[1];
    if (in_place && coef == 1.f) return;
    scale_tiles<STREAM>(b, blockIdx.x, gridDim.x, coef);
}

template <int POW> __global__ void norm_coef_kernel(const double* __restrict__ total, float max_norm, float* __restrict__ norm_coef) {
    const float norm = root<POW>(*total);
    norm_coef[0] = norm;
    norm_coef[1] = clip_coef(norm, max_norm);
}

}  // namespace mtc

using namespace mtc;

struct ClipList {
    int32_t n;
    const void* const* src;
    void* const* dst;                      // NULL: norm only
    const uint64_t* elems;
    const int32_t* dtype;
};

static int clip_pow(float p) { return p == 1.f ? POW_1 : p == 2.f ? POW_2 : p == __builtin_inff() ? POW_INF : 0; }

static int clip_check(const ClipList& l, float p, const char* who) {
    MTC_REQUIRE(l.n >= 0 && (l.n == 0 || (l.src && l.elems && l.dtype)), "%s: bad tensor list", who);
    MTC_REQUIRE(clip_pow(p), "%s: the norm's order must be 1, 2 or inf (got %g)", who, (double)p);
    for (int i = 0; i < l.n; ++i) {
        MTC_REQUIRE(l.dtype[i] == MTC_F32 || l.dtype[i] == MTC_BF16, "%s: tensor %d: bad dtype %d", who, i, l.dtype[i]);
        MTC_REQUIRE(l.elems[i] < (1ull << 40), "%s: tensor %d: too many elements", who, i);
        const uintptr_t align = l.dtype[i] == MTC_BF16 ? 1 : 3;
        MTC_REQUIRE(l.elems[i] == 0 || (l.src[i] && !((uintptr_t)l.src[i] & align)), "%s: tensor %d: null or misaligned", who, i);
        if (l.dst) MTC_REQUIRE(l.elems[i] == 0 || (l.dst[i] && !((uintptr_t)l.dst[i] & align)), "%s: output %d: null or misaligned", who, i);
    }
    return 0;
}

// what is written must not be read or written under another index: two workgroups would race on it
static int clip_check_overlap(const ClipList& l, const char* who) {
    struct Span { uintptr_t a, b; int32_t i, out; };
    if (l.n == 0) return 0;
    Span* s = new (std::nothrow) Span[2 * (size_t)l.n];
    MTC_REQUIRE(s, "%s: out of host memory", who);
    int m = 0;
    for (int i = 0; i < l.n; ++i) {
        if (!l.elems[i]) continue;
        const uintptr_t bytes = l.elems[i] * (l.dtype[i] == MTC_BF16 ? 2 : 4);
        s[m++] = {(uintptr_t)l.dst[i], (uintptr_t)l.dst[i] + bytes, i, 1};
        if (l.dst[i] != l.src[i]) s[m++] = {(uintptr_t)l.src[i], (uintptr_t)l.src[i] + bytes, i, 0};
    }
    std::sort(s, s + m, [](const Span& x, const Span& y) { return x.a < y.a; });
    // sweep by start: the furthest end among the outputs, and among all, seen so far
    uintptr_t out_end = 0, any_end = 0;
    int bad = -1;
    for (int k = 0; k < m && bad < 0; ++k) {
        if (s[k].a < out_end || (s[k].out && s[k].a < any_end)) bad = s[k].i;
        if (s[k].out) out_end = std::max(out_end, s[k].b);
        any_end = std::max(any_end, s[k].b);
    }
    delete[] s;
    MTC_REQUIRE(bad < 0, "%s: tensor %d shares memory with another tensor or output of the list", who, bad);
    return 0;
}

// the next batch of the list from index i on; returns the index behind it
static int clip_batch(const ClipList& l, int i, ClipBatch& b) {
    b.n = b.tiles = 0;
    for (; i < l.n && b.n < CLIP_BATCH; ++i) {
        if (!l.elems[i]) continue;
        const bool bf = l.dtype[i] == MTC_BF16;
        const uint64_t per = (uint64_t)TILE_UNITS * (bf ? 8 : 4);
        const uint64_t tiles = (l.elems[i] + per - 1) / per;
        if (b.n && b.tiles + tiles > 0x7fffffffull) break;
        const bool aligned = (((uintptr_t)l.src[i] | (l.dst ? (uintptr_t)l.dst[i] : 0)) & 15) == 0;
        b.first[b.n] = (uint32_t)b.tiles;
        b.src[b.n] = l.src[i];
        b.dst[b.n] = l.dst ? l.dst[i] : nullptr;
        b.elems[b.n] = l.elems[i] | (bf ? 1ull << 63 : 0) | (aligned ? 1ull << 62 : 0);
        b.tiles += (int)tiles;
        ++b.n;
    }
    return i;
}

static int clip_parts(const ClipList& l) {
    int parts = 0;
    ClipBatch b;
    for (int i = 0; i < l.n;) {
        i = clip_batch(l, i, b);
        parts += std::min(b.tiles, CLIP_GRID);
    }
    return parts;
}

static uint64_t clip_tiles(const ClipList& l) {
    uint64_t tiles = 0;
    for (int i = 0; i < l.n; ++i) {
        const uint64_t per = (uint64_t)TILE_UNITS * (l.dtype[i] == MTC_BF16 ? 8 : 4);
        tiles += (l.elems[i] + per - 1) / per;
    }
    return tiles;
}

extern "C" size_t mtc_grad_norm_workspace_bytes(int32_t n, const uint64_t* elems, const int32_t* dtype) {
    if (n < 0 || (n && (!elems || !dtype))) return 0;
    // one partial per workgroup of the norm's launches (each at most its tiles, and CLIP_GRID), then {norm, coef}
    const uint64_t tiles = clip_tiles({n, nullptr, nullptr, elems, dtype});
    const uint64_t cap = (uint64_t)CLIP_GRID * ((n + CLIP_BATCH - 1) / CLIP_BATCH + 1);
    return (size_t)(std::min(tiles, cap) + 1) * sizeof(double);
}

template <int POW> static int sum_launch(const ClipList& l, double* partial, bool streaming, hipStream_t s) {
    int parts = 0;
    ClipBatch b;
    for (int i = 0; i < l.n;) {
        i = clip_batch(l, i, b);
        if (!b.tiles) continue;
        const int grid = std::min(b.tiles, CLIP_GRID);
        if (streaming) hipLaunchKernelGGL((power_sum_kernel<POW, true>), dim3(grid), dim3(256), 0, s, b, partial + parts);
        else hipLaunchKernelGGL((power_sum_kernel<POW, false>), dim3(grid), dim3(256), 0, s, b, partial + parts);
        parts += grid;
    }
    return parts;
}

template <int POW>
static void norm_launch(const ClipList& l, double* ws, double* total, float max_norm, float* norm_coef, hipStream_t s) {
    const int parts = sum_launch<POW>(l, ws, clip_tiles(l) > STREAM_TILES, s);
    hipLaunchKernelGGL(norm_finish_kernel<POW>, dim3(1), dim3(256), 0, s, ws, parts, max_norm, total, norm_coef, (float*)nullptr);
}

template <int POW> static void clip_launch(const ClipList& l, double* ws, float max_norm, float* norm_out, hipStream_t s) {
    const uint64_t tiles = clip_tiles(l);
    const bool streaming = tiles > STREAM_TILES, small = tiles <= SMALL_TILES;
    const int parts = sum_launch<POW>(l, ws, streaming, s);
    float* norm_coef = reinterpret_cast<float*>(ws + parts);
    if (!small || !tiles)
        hipLaunchKernelGGL(norm_finish_kernel<POW>, dim3(1), dim3(256), 0, s, ws, parts, max_norm, (double*)nullptr, norm_coef, norm_out);
    ClipBatch b;
    for (int i = 0; i < l.n;) {
        i = clip_batch(l, i, b);
        if (!b.tiles) continue;
        int in_place = 1;
        for (int t = 0; t < b.n; ++t) in_place &= b.src[t] == b.dst[t];
        if (small) {
            hipLaunchKernelGGL(clip_small_kernel<POW>, dim3(std::min(b.tiles, CLIP_GRID)), dim3(256), 0, s, b, ws, parts, max_norm, in_place,
                               norm_out);
            norm_out = nullptr;                          // the first launch has written it
        } else if (streaming) {
            hipLaunchKernelGGL(clip_large_kernel<true>, dim3(std::min(b.tiles, LARGE_GRID)), dim3(256), 0, s, b, norm_coef, in_place);
        } else {
            hipLaunchKernelGGL(clip_large_kernel<false>, dim3(std::min(b.tiles, LARGE_GRID)), dim3(256), 0, s, b, norm_coef, in_place);
        }
    }
}

extern "C" int mtc_grad_norm(int32_t n, const void* const* grads, const uint64_t* elems, const int32_t* dtype, float p,
                             void* workspace, size_t workspace_bytes, double* total, float max_norm, float* norm_coef,
                             void* stream) {
    static const char* who = "mtc_grad_norm";
    const ClipList l = {n, grads, nullptr, elems, dtype};
    if (clip_check(l, p, who)) return -1;
    MTC_REQUIRE(total || norm_coef, "%s: no output", who);
    MTC_REQUIRE(max_norm >= 0.f, "%s: max_norm must not be negative or NaN", who);
    MTC_REQUIRE(workspace && ((uintptr_t)workspace & 7) == 0 && workspace_bytes >= (size_t)(clip_parts(l) + 1) * sizeof(double),
                "%s: workspace missing, misaligned or too small", who);
    double* ws = reinterpret_cast<double*>(workspace);
    hipStream_t s = as_stream(stream);
    switch (clip_pow(p)) {
        case POW_1: norm_launch<POW_1>(l, ws, total, max_norm, norm_coef, s); break;
        case POW_2: norm_launch<POW_2>(l, ws, total, max_norm, norm_coef, s); break;
        default: norm_launch<POW_INF>(l, ws, total, max_norm, norm_coef, s);
    }
    return check_launch(who);
}

extern "C" int mtc_grad_norm_coef(const double* total, float p, float max_norm, float* norm_coef, void* stream) {
    static const char* who = "mtc_grad_norm_coef";
    MTC_REQUIRE(total && norm_coef, "%s: null pointer", who);
    MTC_REQUIRE(clip_pow(p), "%s: the norm's order must be 1, 2 or inf (got %g)", who, (double)p);
    MTC_REQUIRE(max_norm >= 0.f, "%s: max_norm must not be negative or NaN", who);
    hipStream_t s = as_stream(stream);
    if (clip_pow(p) == POW_2) hipLaunchKernelGGL(norm_coef_kernel<POW_2>, dim3(1), dim3(1), 0, s, total, max_norm, norm_coef);
    else hipLaunchKernelGGL(norm_coef_kernel<POW_1>, dim3(1), dim3(1), 0, s, total, max_norm, norm_coef);
    return check_launch(who);
}

extern "C" int mtc_grad_clip(int32_t n, const void* const* grads, void* const* out, const uint64_t* elems, const int32_t* dtype,
                             float p, float max_norm, void* workspace, size_t workspace_bytes, float* norm_out, void* stream) {
    static const char* who = "mtc_grad_clip";
    const ClipList l = {n, grads, out, elems, dtype};
    MTC_REQUIRE(n <= 0 || out, "%s: null output list", who);
    if (clip_check(l, p, who) || clip_check_overlap(l, who)) return -1;
    MTC_REQUIRE(max_norm >= 0.f, "%s: max_norm must not be negative or NaN", who);
    MTC_REQUIRE(workspace && ((uintptr_t)workspace & 7) == 0 && workspace_bytes >= (size_t)(clip_parts(l) + 1) * sizeof(double),
                "%s: workspace missing, misaligned or too small", who);
    double* ws = reinterpret_cast<double*>(workspace);
    hipStream_t s = as_stream(stream);
    switch (clip_pow(p)) {
        case POW_1: clip_launch<POW_1>(l, ws, max_norm, norm_out, s); break;
        case POW_2: clip_launch<POW_2>(l, ws, max_norm, norm_out, s); break;
        default: clip_launch<POW_INF>(l, ws, max_norm, norm_out, s);
    }
    return check_launch(who);
}
