// Rows of logits (..., V) as the kernels at the classifier's end read and write them: token log probabilities,
// distillation, drawing of tokens.
#pragma once

#include "ulm_common.h"

namespace ulm {
namespace rows {

constexpr float kLog2e = 1.44269504088896341f;

typedef uint32_t u32x4_any __attribute__((vector_size(16), aligned(2)));   // rows may start anywhere

// 16 bytes of a stream that the caches need not keep (bf16 rows of 32000: 6.7 TB/s, 5.9 with ordinary loads)
__device__ __forceinline__ u32x4_any load_once(const char *p) {
    return __builtin_nontemporal_load(reinterpret_cast<const u32x4_any *>(p));
}

template <int DT> struct Elem { static constexpr int vec = DT == ULM_F32 ? 4 : 8, bytes = DT == ULM_F32 ? 4 : 2; };

template <int DT> __device__ __forceinline__ void unpack(const u32x4_any &w, float (&x)[Elem<DT>::vec]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if constexpr (DT == ULM_F32) {
            x[k] = __uint_as_float(w[k]);
        } else if constexpr (DT == ULM_BF16) {
            x[2 * k] = __uint_as_float(w[k] << 16);
            x[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
        } else {
            x[2 * k] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[k])));
            x[2 * k + 1] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[k] >> 16)));
        }
    }
}

template <int DT> __device__ __forceinline__ uint32_t pack_word(float a, float b) {
    if constexpr (DT == ULM_BF16) {
        return f32_to_bf16_bits(a) | (static_cast<uint32_t>(f32_to_bf16_bits(b)) << 16);
    } else {
        return __builtin_bit_cast(uint16_t, static_cast<_Float16>(a)) |
               (static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<_Float16>(b))) << 16);
    }
}

// x's elements [i, i + vec) of a row that ends at `end`, -inf past it; ONCE: as a stream (load_once)
template <int DT, bool ONCE = true>
__device__ __forceinline__ void load_vec(const char *row, int i, int end, float (&x)[Elem<DT>::vec]) {
    constexpr int V = Elem<DT>::vec;
    if (i + V <= end) {
        const char *p = row + static_cast<size_t>(i) * Elem<DT>::bytes;
        unpack<DT>(ONCE ? load_once(p) : *reinterpret_cast<const u32x4_any *>(p), x);
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) x[k] = i + k < end ? load_as_f32(row, i + k, DT) : -INFINITY;
    }
}

// Unique keys in the order of the alternatives: by value (a NaN above all), then by the lower index.
__device__ __forceinline__ uint64_t key_of(float x, int i) {
    uint32_t b = __float_as_uint(x + 0.f);   // -0 and 0 are one value
    b = x != x ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return static_cast<uint64_t>(b) << 32 | (0xffffffffu - static_cast<uint32_t>(i));
}
__device__ __forceinline__ int index_of(uint64_t key) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(key)); }
__device__ __forceinline__ float value_of(uint64_t key) {
    const uint32_t b = key >> 32;
    return __uint_as_float((b & 0x80000000u) ? b & 0x7fffffffu : ~b);
}

// The larger one of numbers; three at a time, and without the quieting of a signalling NaN that fmaxf adds
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// Workgroup b of n: the grid's second dimension takes what the first cannot count.
constexpr long long kGridX = 1 << 20;
inline dim3 grid_of(long long n) {
    return n <= kGridX ? dim3(static_cast<unsigned>(n)) : dim3(kGridX, static_cast<unsigned>((n + kGridX - 1) / kGridX));
}
__device__ __forceinline__ long long block_id() { return static_cast<long long>(blockIdx.y) * gridDim.x + blockIdx.x; }

// Row r starts at (r / inner) outer_stride + (r % inner) row_stride elements.
struct View {
    const char *x;
    long long inner, outer_stride, row_stride, rows;
    int V;
    __device__ __forceinline__ const char *row(long long r, int bytes) const {
        const long long outer = r < inner ? 0 : r / inner;   // mostly one stride: no division
        return x + (outer * outer_stride + (r - outer * inner) * row_stride) * bytes;
    }
};

}  // namespace rows
}  // namespace ulm
