// The global norm of a model's gradients and their clipping to a bound on it
// (train.py's clip_grad_norm_ before the optimizer's step):
//
//     norm = sqrt(sum over all tensors of g^2)  or  max |g|
//     out  = g min(1, max_norm / (norm + 1e-6))
//
// The tensors travel as a table in the kernel's arguments, cut into chunks of equal length
// that a fixed number of workgroups share; every workgroup leaves one partial norm and the
// scaling kernel adds those up by itself. Squares are exact in double and summed in it:
// no gradient of the three types over- or underflows there. Fixed order, no atomics.
#include <math.h>
#include <type_traits>

#include "ulm_common.h"

namespace ulm {
namespace gr {

constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr int kPer = 32;                                    // a thread's elements of a chunk
constexpr int kChunk = kThreads * kPer;                     // 8192 elements
constexpr int kBlocks = 1024;                               // workgroups of a norm launch at most
constexpr int kTable = 112;                                 // tensors a launch takes: the arguments stay under 4 KB
constexpr float kEps = 1e-6f;

typedef uint32_t u32x4_any __attribute__((vector_size(16), aligned(2)));   // views start anywhere
typedef uint32_t u32x2_any __attribute__((vector_size(8), aligned(2)));

struct Table {
    const char *src[kTable];
    char *dst[kTable];
    long long numel[kTable];
    uint32_t first[kTable + 1];   // the tensors' first chunks, and their number
    uint8_t src_dt[kTable], dst_dt[kTable];
    int n;
};

// the tensor of chunk c
__device__ __forceinline__ int tensor_of(const Table &t, uint32_t c) {
    int lo = 0, hi = t.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (t.first[mid] <= c) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// V consecutive elements, 4 or 8: 16 bytes, or 8 of a 16-bit type where the other side has 32
template <bool ONCE, class T> __device__ __forceinline__ T fetch(const char *p) {
    if constexpr (ONCE) return __builtin_nontemporal_load(reinterpret_cast<const T *>(p));
    else return *reinterpret_cast<const T *>(p);
}
template <int DT, int V, bool ONCE> __device__ __forceinline__ void load_vec(const char *p, long long i, float (&x)[V]) {
    if constexpr (DT == ULM_F32) {
        static_assert(V == 4, "16 bytes");
        const u32x4_any w = fetch<ONCE, u32x4_any>(p + 4 * i);
#pragma unroll
        for (int k = 0; k < V; ++k) x[k] = __uint_as_float(w[k]);
    } else {
        const auto w = fetch<ONCE, std::conditional_t<V == 8, u32x4_any, u32x2_any>>(p + 2 * i);
#pragma unroll
        for (int k = 0; k < V / 2; ++k) {
            if constexpr (DT == ULM_BF16) {
                x[2 * k] = __uint_as_float(w[k] << 16);
                x[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
            } else {
                x[2 * k] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[k])));
                x[2 * k + 1] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[k] >> 16)));
            }
        }
    }
}

template <int DT, int V> __device__ __forceinline__ void store_vec(char *p, long long i, const float (&x)[V]) {
    if constexpr (DT == ULM_F32) {
        u32x4_any w;
#pragma unroll
        for (int k = 0; k < V; ++k) w[k] = __float_as_uint(x[k]);
        __builtin_nontemporal_store(w, reinterpret_cast<u32x4_any *>(p + 4 * i));
    } else {
        using T = std::conditional_t<V == 8, u32x4_any, u32x2_any>;
        T w;
#pragma unroll
        for (int k = 0; k < V / 2; ++k) {
            if constexpr (DT == ULM_BF16)
                w[k] = f32_to_bf16_bits(x[2 * k]) | (static_cast<uint32_t>(f32_to_bf16_bits(x[2 * k + 1])) << 16);
            else
                w[k] = __builtin_bit_cast(uint16_t, static_cast<_Float16>(x[2 * k])) |
                       (static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<_Float16>(x[2 * k + 1]))) << 16);
        }
        __builtin_nontemporal_store(w, reinterpret_cast<T *>(p + 2 * i));
    }
}

// a chunk's elements of a thread: vectors of V, zeros past the tensor's end
template <int DT, int V, bool ONCE>
__device__ __forceinline__ void load_chunk(const char *p, long long base, long long numel, int tid, float (&x)[kPer / V][V]) {
    if (base + kChunk <= numel) {
#pragma unroll
        for (int j = 0; j < kPer / V; ++j) load_vec<DT, V, ONCE>(p, base + (j * kThreads + tid) * V, x[j]);
    } else {
#pragma unroll
        for (int j = 0; j < kPer / V; ++j) {
            const long long i = base + (j * kThreads + tid) * V;
            if (i + V <= numel) {
                load_vec<DT, V, ONCE>(p, i, x[j]);
            } else {
#pragma unroll
                for (int k = 0; k < V; ++k) x[j][k] = i + k < numel ? load_as_f32(p, i + k, DT) : 0.f;
            }
        }
    }
}

// The norms' two measures: an accumulator as a double (the sum of squares) or as the bits
// of the largest |g| (a NaN's are above infinity's, so it stays).
template <bool MAX> struct Acc {
    using T = std::conditional_t<MAX, unsigned long long, double>;
    static __device__ __forceinline__ T add(T a, T b) {
        if constexpr (MAX) return a > b ? a : b;
        else return a + b;
    }
    static __device__ __forceinline__ T take(T a, float x) {
        if constexpr (MAX) {
            const unsigned long long b = __float_as_uint(x) & 0x7fffffffu;
            return a > b ? a : b;
        } else {
            const double d = x;
            return __builtin_fma(d, d, a);
        }
    }
    static __device__ __forceinline__ float norm(T a) {
        if constexpr (MAX) return __uint_as_float(static_cast<uint32_t>(a));
        else return static_cast<float>(sqrt(a));
    }
};

// the workgroup's accumulators joined; every thread gets the result
template <bool MAX> __device__ typename Acc<MAX>::T join(typename Acc<MAX>::T v) {
    __shared__ typename Acc<MAX>::T part[kWaves];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = Acc<MAX>::add(v, __shfl_xor(v, off, kWave));
    if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v = Acc<MAX>::add(v, part[w]);
    return v;
}

template <bool MAX, int DT>
__device__ __forceinline__ typename Acc<MAX>::T take_chunk(typename Acc<MAX>::T acc, const char *p, long long base,
                                                           long long numel) {
    constexpr int V = DT == ULM_F32 ? 4 : 8;
    float x[kPer / V][V];
    load_chunk<DT, V, false>(p, base, numel, threadIdx.x, x);   // the caches keep what they can for the scaling
#pragma unroll
    for (int j = 0; j < kPer / V; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) acc = Acc<MAX>::take(acc, x[j][i]);
    return acc;
}

// Bound by the reading: 88M fp32 gradients 63 us, 5.6 TB/s; 88M bf16 41. Squares added in fp32 eight at a time,
// two chunks' loads on their way, shares of consecutive chunks, 512 and 2048 workgroups: all within 5% of it.
template <bool MAX>
__global__ __launch_bounds__(kThreads) void norm_kernel(Table t, typename Acc<MAX>::T *partial) {
    typename Acc<MAX>::T acc{};
    for (uint32_t c = blockIdx.x; c < t.first[t.n]; c += gridDim.x) {
        const int k = tensor_of(t, c);
        const long long base = static_cast<long long>(c - t.first[k]) * kChunk;
        if (t.src_dt[k] == ULM_F32) acc = take_chunk<MAX, ULM_F32>(acc, t.src[k], base, t.numel[k]);
        else if (t.src_dt[k] == ULM_BF16) acc = take_chunk<MAX, ULM_BF16>(acc, t.src[k], base, t.numel[k]);
        else acc = take_chunk<MAX, ULM_F16>(acc, t.src[k], base, t.numel[k]);
    }
    acc = join<MAX>(acc);
    if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

// the norm of all partials, the same bits in every workgroup
template <bool MAX> __device__ float total(const typename Acc<MAX>::T *partial, int n) {
    typename Acc<MAX>::T acc{};
    for (int i = threadIdx.x; i < n; i += kThreads) acc = Acc<MAX>::add(acc, partial[i]);
    return Acc<MAX>::norm(join<MAX>(acc));
}

template <bool MAX>
__global__ __launch_bounds__(kThreads) void finish_kernel(const typename Acc<MAX>::T *partial, int n, float *norm) {
    const float v = total<MAX>(partial, n);
    if (threadIdx.x == 0) *norm = v;
}

template <int S, int D>
__device__ __forceinline__ void scale_chunk(const char *src, char *dst, long long base, long long numel, float coef) {
    constexpr int V = S == ULM_F32 || D == ULM_F32 ? 4 : 8;
    const int tid = threadIdx.x;
    float x[kPer / V][V];
    load_chunk<S, V, true>(src, base, numel, tid, x);
#pragma unroll
    for (int j = 0; j < kPer / V; ++j) {
        const long long i = base + (j * kThreads + tid) * V;
#pragma unroll
        for (int k = 0; k < V; ++k) x[j][k] *= coef;
        if (i + V <= numel) {
            store_vec<D, V>(dst, i, x[j]);
        } else {
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (i + k < numel) store_from_f32(dst, i + k, D, x[j][k]);
        }
    }
}

// The chunks scaled, last first: what the norm kernel read last is what the caches still hold. 88M fp32
// gradients into other buffers 113 us, 6.2 TB/s; 150 with ordinary loads and stores, which keep the
// results in the caches instead, and with each thread's 32 bytes in two stores.
template <bool MAX>
__global__ __launch_bounds__(kThreads) void scale_kernel(Table t, const typename Acc<MAX>::T *partial, int n, float max_norm,
                                                         float *norm) {
    const float v = total<MAX>(partial, n);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = v;
    float coef = max_norm / (v + kEps);
    if (coef > 1.f) coef = 1.f;   // a NaN stays
    for (uint32_t b = blockIdx.x; b < t.first[t.n]; b += gridDim.x) {
        const uint32_t c = t.first[t.n] - 1 - b;
        const int k = tensor_of(t, c);
        if (coef == 1.f && t.src[k] == t.dst[k]) continue;   // in place and nothing to change
        const long long base = static_cast<long long>(c - t.first[k]) * kChunk;
        const char *src = t.src[k];
        char *dst = t.dst[k];
        switch (t.src_dt[k] * 3 + t.dst_dt[k]) {
#define ULM_GR_CASE(S, D) case S * 3 + D: scale_chunk<S, D>(src, dst, base, t.numel[k], coef); break;
            ULM_GR_CASE(ULM_F32, ULM_F32) ULM_GR_CASE(ULM_F32, ULM_BF16) ULM_GR_CASE(ULM_F32, ULM_F16)
            ULM_GR_CASE(ULM_BF16, ULM_F32) ULM_GR_CASE(ULM_BF16, ULM_BF16) ULM_GR_CASE(ULM_BF16, ULM_F16)
            ULM_GR_CASE(ULM_F16, ULM_F32) ULM_GR_CASE(ULM_F16, ULM_BF16) ULM_GR_CASE(ULM_F16, ULM_F16)
#undef ULM_GR_CASE
        }
    }
}

static_assert(sizeof(Table) <= 4000, "kernel arguments");

// the tables of up to kTable non-empty tensors each, in order; f(table, chunks)
template <class F> void tables(const ulm_grad *g, int n, F f) {
    Table t;
    t.n = 0;
    t.first[0] = 0;
    for (int i = 0; i < n; ++i) {
        if (g[i].numel <= 0) continue;
        const long long chunks = (g[i].numel + kChunk - 1) / kChunk;
        if (t.n == kTable || t.first[t.n] + chunks > UINT32_MAX / 2) {
            f(t);
            t.n = 0;
        }
        t.src[t.n] = static_cast<const char *>(g[i].src);
        t.dst[t.n] = static_cast<char *>(g[i].dst);
        t.numel[t.n] = g[i].numel;
        t.src_dt[t.n] = static_cast<uint8_t>(g[i].src_dtype);
        t.dst_dt[t.n] = static_cast<uint8_t>(g[i].dst_dtype);
        t.first[t.n + 1] = t.first[t.n] + static_cast<uint32_t>(chunks);
        ++t.n;
    }
    if (t.n) f(t);
}

inline int blocks_of(const Table &t) {
    const uint32_t chunks = t.first[t.n];
    return chunks < static_cast<uint32_t>(kBlocks) ? static_cast<int>(chunks) : kBlocks;
}

template <bool MAX>
int run(const char *fn, const ulm_grad *g, int n, bool scale, float max_norm, float *norm, void *ws, hipStream_t s) {
    using T = typename Acc<MAX>::T;
    T *partial = static_cast<T *>(ws);
    int used = 0;
    tables(g, n, [&](const Table &t) {
        const int blocks = blocks_of(t);
        norm_kernel<MAX><<<dim3(blocks), dim3(kThreads), 0, s>>>(t, partial + used);
        used += blocks;
    });
    if (!scale || used == 0) {
        finish_kernel<MAX><<<dim3(1), dim3(kThreads), 0, s>>>(partial, used, norm);
    } else {
        float *out = norm;
        tables(g, n, [&](const Table &t) {
            scale_kernel<MAX><<<dim3(blocks_of(t)), dim3(kThreads), 0, s>>>(t, partial, used, max_norm, out);
            out = nullptr;
        });
    }
    return check_launch(fn);
}

int check(const char *fn, const ulm_grad *g, int n, int norm_type, bool scale, float max_norm, const float *norm, const void *ws,
          size_t bytes) {
    if (n < 0 || (n > 0 && !g) || !norm || !ws) return fail(ULM_ERR_INVALID, "%s: null pointer or n=%d", fn, n);
    if (norm_type != ULM_NORM_2 && norm_type != ULM_NORM_INF) return fail(ULM_ERR_INVALID, "%s: bad norm type %d", fn, norm_type);
    if (scale && !(max_norm >= 0.f)) return fail(ULM_ERR_INVALID, "%s: max_norm must not be negative", fn);
    for (int i = 0; i < n; ++i) {
        const ulm_grad &t = g[i];
        if (t.numel < 0 || t.numel > (1LL << 40))
            return fail(ULM_ERR_INVALID, "%s: tensor %d has %lld elements", fn, i, t.numel);
        if (!valid_dtype(t.src_dtype) || (scale && !valid_dtype(t.dst_dtype)))
            return fail(ULM_ERR_INVALID, "%s: bad dtype of tensor %d", fn, i);
        if (t.numel && (!t.src || (scale && !t.dst))) return fail(ULM_ERR_INVALID, "%s: null pointer in tensor %d", fn, i);
        if (scale && t.numel && t.src == t.dst && t.src_dtype != t.dst_dtype)
            return fail(ULM_ERR_INVALID, "%s: tensor %d in place in another dtype", fn, i);
    }
    const size_t need = ulm_grad_norm_workspace_bytes(g, n);
    if (bytes < need) return fail(ULM_ERR_INVALID, "%s: workspace %zu < %zu", fn, bytes, need);
    return ULM_OK;
}

}  // namespace gr
}  // namespace ulm

using namespace ulm;

extern "C" size_t ulm_grad_norm_workspace_bytes(const ulm_grad *grads, int n) {
    size_t blocks = 0;
    if (grads && n > 0) gr::tables(grads, n, [&](const gr::Table &t) { blocks += gr::blocks_of(t); });
    return (blocks ? blocks : 1) * sizeof(double);
}

extern "C" int ulm_grad_norm(const ulm_grad *grads, int n, int norm_type, float *norm, void *workspace, size_t workspace_bytes,
                             void *stream) {
    ULM_TRY(gr::check("ulm_grad_norm", grads, n, norm_type, false, 0.f, norm, workspace, workspace_bytes));
    hipStream_t s = static_cast<hipStream_t>(stream);
    return norm_type == ULM_NORM_INF ? gr::run<true>("ulm_grad_norm", grads, n, false, 0.f, norm, workspace, s)
                                     : gr::run<false>("ulm_grad_norm", grads, n, false, 0.f, norm, workspace, s);
}

extern "C" int ulm_clip_grads(const ulm_grad *grads, int n, int norm_type, float max_norm, float *norm, void *workspace,
                              size_t workspace_bytes, void *stream) {
    ULM_TRY(gr::check("ulm_clip_grads", grads, n, norm_type, true, max_norm, norm, workspace, workspace_bytes));
    hipStream_t s = static_cast<hipStream_t>(stream);
    return norm_type == ULM_NORM_INF ? gr::run<true>("ulm_clip_grads", grads, n, true, max_norm, norm, workspace, s)
                                     : gr::run<false>("ulm_clip_grads", grads, n, true, max_norm, norm, workspace, s);
}
