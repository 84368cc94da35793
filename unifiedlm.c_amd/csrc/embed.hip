// Embedding lookup with scaling and the weight's gradient (nn.Embedding in
// UnifiedLM, model.py:117, 150):
//
//     out[n] = scale W[t_n]      dW[v] = scale sum over n with t_n = v of dout[n]
//
// The gradient's rows are summed in an order that the tokens fix: the tokens are sorted with their
// positions by a stable radix sort, the rows of dout are summed along the sorted order in
// chunks of equal length, one wave each, and sums that go over a chunk's end are
// joined afterwards. No atomics on numbers: equal inputs give equal bits.
#include <algorithm>
#include <type_traits>

#include "ulm_common.h"

namespace ulm {
namespace emb {

constexpr int kThreads = 256;
typedef uint32_t u32x4_any __attribute__((vector_size(16), aligned(2)));   // rows may start anywhere

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

template <int DT> __device__ __forceinline__ u32x4_any pack(const float (&x)[Elem<DT>::vec]) {
    u32x4_any w;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if constexpr (DT == ULM_F32) {
            w[k] = __float_as_uint(x[k]);
        } else if constexpr (DT == ULM_BF16) {
            w[k] = f32_to_bf16_bits(x[2 * k]) | (static_cast<uint32_t>(f32_to_bf16_bits(x[2 * k + 1])) << 16);
        } else {
            w[k] = __builtin_bit_cast(uint16_t, static_cast<_Float16>(x[2 * k])) |
                   (static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<_Float16>(x[2 * k + 1]))) << 16);
        }
    }
    return w;
}

// Vector p of a row of D elements: the row's last vector ends with it and overlaps the one before,
// whose elements it computes as well, to the same bits. Rows shorter than a vector are one
// vector, read and written by elements.
template <int E> __device__ __forceinline__ int column(int p, int D) { return D < E ? 0 : min(p * E, D - E); }

template <int DT> __device__ __forceinline__ void load_vec(const char *row, int i, int D, float (&x)[Elem<DT>::vec]) {
    constexpr int E = Elem<DT>::vec;
    if (D >= E) {
        unpack<DT>(*reinterpret_cast<const u32x4_any *>(row + static_cast<size_t>(i) * Elem<DT>::bytes), x);
    } else {
#pragma unroll
        for (int k = 0; k < E; ++k) x[k] = k < D ? load_as_f32(row, k, DT) : 0.f;
    }
}

// the vector as it lies in memory, of a stream that the caches need not keep
template <int DT> __device__ __forceinline__ u32x4_any load_raw(const char *row, int i, int D) {
    constexpr int E = Elem<DT>::vec;
    const char *p = row + static_cast<size_t>(i) * Elem<DT>::bytes;
    if (D >= E) return __builtin_nontemporal_load(reinterpret_cast<const u32x4_any *>(p));
    float x[E];
    load_vec<DT>(row, i, D, x);
    return pack<DT>(x);
}

template <int DT, bool STREAM = false>
__device__ __forceinline__ void store_vec(char *row, int i, int D, const float (&x)[Elem<DT>::vec]) {
    constexpr int E = Elem<DT>::vec;
    if (D >= E) {
        u32x4_any *to = reinterpret_cast<u32x4_any *>(row + static_cast<size_t>(i) * Elem<DT>::bytes);
        if constexpr (STREAM) __builtin_nontemporal_store(pack<DT>(x), to);
        else *to = pack<DT>(x);
    } else {
#pragma unroll
        for (int k = 0; k < E; ++k)
            if (k < D) store_from_f32(row, k, DT, x[k]);
    }
}

// the same of fp32 sums
template <int E> __device__ __forceinline__ void load_sums(const float *row, int i, int D, float (&x)[E]) {
    if (D >= E) {
#pragma unroll
        for (int k = 0; k < E; k += 4) {
            const u32x4_any w = *reinterpret_cast<const u32x4_any *>(row + i + k);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[k + j] = __uint_as_float(w[j]);
        }
    } else {
#pragma unroll
        for (int k = 0; k < E; ++k) x[k] = k < D ? row[k] : 0.f;
    }
}
template <int E> __device__ __forceinline__ void store_sums(float *row, int i, int D, const float (&x)[E]) {
    if (D >= E) {
#pragma unroll
        for (int k = 0; k < E; k += 4) {
            u32x4_any w;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = __float_as_uint(x[k + j]);
            *reinterpret_cast<u32x4_any *>(row + i + k) = w;
        }
    } else {
#pragma unroll
        for (int k = 0; k < E; ++k)
            if (k < D) row[k] = x[k];
    }
}

// ---- lookup: each thread one vector of a row, vectors in order over the grid

template <int DT>
__global__ __launch_bounds__(kThreads) void fwd_kernel(const char *__restrict__ weight, const long long *__restrict__ tokens,
                                                       char *__restrict__ out, long long N, int V, int D, uint32_t pieces,
                                                       float scale) {
    constexpr int E = Elem<DT>::vec, B = Elem<DT>::bytes;
    const long long total = N * pieces, step = static_cast<long long>(gridDim.x) * kThreads;
    for (long long p = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x; p < total; p += step) {
        // 32-bit division where it will do
        const long long n = total <= UINT32_MAX ? static_cast<uint32_t>(p) / pieces : p / pieces;
        const int i = column<E>(static_cast<int>(p - n * pieces), D);
        const long long t = tokens[n];
        float x[E];
        if (t >= 0 && t < V) {
            load_vec<DT>(weight + t * D * B, i, D, x);
#pragma unroll
            for (int k = 0; k < E; ++k) x[k] *= scale;
        } else {
#pragma unroll
            for (int k = 0; k < E; ++k) x[k] = __uint_as_float(0x7fc00000u);
        }
        store_vec<DT>(out + n * D * B, i, D, x);
    }
}

// ---- the stable radix sort of (token, position) by token, kBits bits a pass

constexpr int kBits = 10, kBins = 1 << kBits;
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / kWave;
constexpr int kTile = 4096;   // entries per workgroup of a long sequence's pass
constexpr int kShort = 32768;   // tokens up to which a pass is one launch (at 65536 as long as three); half a counter holds them

struct Entry {
    uint32_t token, pos;
};

// where a pass reads its entries: the caller's tokens (the first), or the last pass's output.
// A token outside [0, V) takes part as V, behind all others.
struct Source {
    const long long *tokens;
    const Entry *entries;
    int V;
    __device__ __forceinline__ Entry at(int i) const {
        if (!tokens) return entries[i];
        const long long t = tokens[i];
        return {t >= 0 && t < V ? static_cast<uint32_t>(t) : static_cast<uint32_t>(V), static_cast<uint32_t>(i)};
    }
};

__device__ __forceinline__ uint32_t digit_of(uint32_t token, int shift) { return (token >> shift) & (kBins - 1); }

__device__ __forceinline__ uint32_t wave_scan(uint32_t v, int lane) {   // inclusive
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
        const uint32_t o = __shfl_up(v, off, kWave);
        if (lane >= off) v += o;
    }
    return v;
}

// How many lanes, this one first, hold `value` one after the other; 0 on a lane that follows another of its
// run or is not live. Live lanes come first. What counts equal values adds a run at once: additions to
// one counter go one by one, and a frequent token's entries come together (padding, or an earlier pass).
__device__ __forceinline__ uint32_t run_length(uint32_t value, bool live, int lane) {
    const uint32_t left = __shfl_up(value, 1, kWave);
    const uint64_t in = __ballot(live), first = __ballot(lane == 0 || left != value) & in;
    const uint64_t ends = (first | ~in) & ~((2ull << lane) - 1);   // the lanes above that end the run
    const int end = ends ? __ffsll(static_cast<unsigned long long>(ends)) - 1 : kWave;
    return first >> lane & 1 ? end - lane : 0;
}

// counts[bin][tile]: the entries of each tile by their digit
__global__ __launch_bounds__(kSortThreads) void count_kernel(Source src, int N, int shift, uint32_t *counts, int tiles) {
    __shared__ uint32_t hist[kBins];
    for (int b = threadIdx.x; b < kBins; b += kSortThreads) hist[b] = 0;
    __syncthreads();
    const int tile = blockIdx.x, end = min(N, (tile + 1) * kTile);
    for (int i = tile * kTile; i < end; i += kSortThreads) {
        const int at = i + threadIdx.x;
        const uint32_t digit = digit_of(src.at(min(at, end - 1)).token, shift);
        const uint32_t run = run_length(digit, at < end, threadIdx.x % kWave);
        if (run) atomicAdd(&hist[digit], run);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < kBins; b += kSortThreads) counts[static_cast<size_t>(b) * tiles + tile] = hist[b];
}

// Each bin's counts turned into the entries of that bin in earlier tiles, in place; totals[bin].
__global__ __launch_bounds__(kWave) void scan_kernel(uint32_t *counts, int tiles, uint32_t *totals) {
    uint32_t *c = counts + static_cast<size_t>(blockIdx.x) * tiles;
    const int lane = threadIdx.x;
    uint32_t before = 0;
    for (int t0 = 0; t0 < tiles; t0 += kWave) {
        const int t = t0 + lane;
        const uint32_t v = t < tiles ? c[t] : 0, inc = wave_scan(v, lane);
        if (t < tiles) c[t] = before + inc - v;
        before += __shfl(inc, kWave - 1, kWave);
    }
    if (lane == 0) totals[blockIdx.x] = before;
}

// dW as zeros, by the workgroups behind a short sequence's first sorting launch: the sort leaves most of the
// device idle, and the rows that occur are written over by their sums. 16384 x 768 fp32 rows into 32000: the
// gradient 38 us, 46 with only the absent rows zeroed, beside the sums; of one token 19 and 26. Ordinary stores
// take 40, more of them a thread 40 (four, eight).
struct Zero {
    static constexpr int kStores = 2, kBytes = kStores * kSortThreads * 16;   // a workgroup's at a time
    char *dw;
    size_t bytes;
    int from;   // the first workgroup
    __device__ __forceinline__ bool take(int tid) const {
        if (static_cast<int>(blockIdx.x) < from) return false;
        const size_t step = static_cast<size_t>(gridDim.x - from) * kBytes;
        for (size_t at = static_cast<size_t>(blockIdx.x - from) * kBytes; at < bytes; at += step) {
#pragma unroll
            for (int j = 0; j < kStores; ++j) {
                const size_t b = at + (j * kSortThreads + tid) * 16;
                if (b + 16 <= bytes) __builtin_nontemporal_store(u32x4_any{0, 0, 0, 0}, reinterpret_cast<u32x4_any *>(dw + b));
                else
                    for (size_t k = b; k < bytes; k += 2) *reinterpret_cast<uint16_t *>(dw + k) = 0;
            }
        }
        return true;
    }
    unsigned blocks() const { return static_cast<unsigned>(std::min<size_t>((bytes + kBytes - 1) / kBytes, 1 << 16)); }
};

// Every entry of a tile of PER x kSortThreads to its place: the smaller digits' total, the same
// digit's entries in earlier tiles, in earlier waves of this tile, and among the lanes before.
// COUNT: the first two are counted here, by every workgroup, over the whole sequence, which for
// a short one takes less time than two more launches (counts and totals are not used then).
template <int PER, bool COUNT>
__global__ __launch_bounds__(kSortThreads) void place_kernel(Source src, int N, int shift, const uint32_t *counts, int tiles,
                                                             const uint32_t *totals, Entry *out, Zero zero) {
    static_assert(kBins == kSortThreads, "one bin per thread");
    __shared__ uint32_t base[kBins], all[COUNT ? kBins : 1];
    __shared__ uint16_t seen[kSortWaves][kBins];   // a wave's entries of each digit, then those of the waves before it
    __shared__ uint32_t sums[kSortWaves];
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave, tile = blockIdx.x, start = tile * PER * kSortThreads;
    if (COUNT && zero.take(tid)) return;

    Entry e[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int i = start + (wave * PER + k) * kWave + lane;
        e[k] = i < N ? src.at(i) : Entry{0, 0};
    }
    uint32_t *clear = reinterpret_cast<uint32_t *>(seen);
    for (int i = tid; i < kSortWaves * kBins / 2; i += kSortThreads) clear[i] = 0;
    static_assert(!COUNT || PER == 1, "tiles of one entry a thread");
    if constexpr (COUNT) {
        base[tid] = all[tid] = 0;
        __syncthreads();
        constexpr int kRead = 16;
        for (int i = 0; i < N; i += kRead * kSortThreads) {
            uint32_t digit[kRead];
#pragma unroll
            for (int k = 0; k < kRead; ++k) digit[k] = digit_of(src.at(min(i + k * kSortThreads + tid, N - 1)).token, shift);
#pragma unroll
            for (int k = 0; k < kRead; ++k) {
                const int at = i + k * kSortThreads;   // of the whole workgroup: a tile of one entry a thread
                if (at >= N) break;
                const uint32_t run = run_length(digit[k], at + tid < N, lane);
                if (run) atomicAdd(&(at < start ? base : all)[digit[k]], run);
            }
        }
    }
    __syncthreads();
    const uint32_t total = COUNT ? all[tid] + base[tid] : totals[tid], inc = wave_scan(total, lane);
    if (lane == kWave - 1) sums[wave] = inc;
    __syncthreads();
    uint32_t below = lane < wave ? sums[lane] : 0;   // the waves' totals before this one's
#pragma unroll
    for (int off = kSortWaves / 2; off > 0; off >>= 1) below += __shfl_xor(below, off, kWave);
    below = __builtin_amdgcn_readfirstlane(below) + inc - total;
    if constexpr (COUNT) base[tid] += below;
    else base[tid] = below + counts[static_cast<size_t>(tid) * tiles + tile];

    uint32_t rank[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int i = start + (wave * PER + k) * kWave + lane;
        const bool live = i < N;
        const uint32_t digit = digit_of(e[k].token, shift);
        uint64_t same = __ballot(live);   // the lanes with this digit
#pragma unroll
        for (int b = 0; b < kBits; ++b) {
            const uint64_t m = __ballot(digit >> b & 1);
            same &= (digit >> b & 1) ? m : ~m;
        }
        rank[k] = seen[wave][digit] + __popcll(same & ((1ull << lane) - 1));
        // the wave's own counters: every lane has read them before the last lane of each digit writes
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (live && (same >> lane) == 1) seen[wave][digit] = static_cast<uint16_t>(rank[k] + 1);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    uint16_t c[kSortWaves];
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) c[w] = seen[w][tid];
    uint32_t before = 0;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
        seen[w][tid] = static_cast<uint16_t>(before);
        before += c[w];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int i = start + (wave * PER + k) * kWave + lane;
        if (i >= N) continue;
        const uint32_t digit = digit_of(e[k].token, shift);
        out[base[digit] + seen[wave][digit] + rank[k]] = e[k];
    }
}

// The whole sort of a short sequence of tokens below kSmallV in one launch: every workgroup
// counts all tokens, those of earlier tiles in the counter's upper half, turns the counts
// into the places where its tile's entries begin, and its tile's waves take theirs in turn. At 16384
// tokens 13 us, where the two digits' launches take 20; with tiles of 1024 entries, 16 turns, 1 us more, of
// 128 as long as with 256.
constexpr int kSmallTile = 256;
constexpr int kSmallV = (1 << 15) - 1;   // tokens 0 .. kSmallV, the last one for those outside
__global__ __launch_bounds__(kSortThreads) void place_small_kernel(Source src, int N, Entry *out, Zero zero) {
    constexpr int kSmallBins = kSmallV + 1, kPer = kSmallBins / kSortThreads, kRead = 16;
    alignas(16) __shared__ uint32_t bins[kSmallBins + kSortThreads];   // a word between threads' shares, off the same bank
    __shared__ uint32_t sums[kSortWaves];
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave, start = blockIdx.x * kSmallTile;
    auto bin = [&](uint32_t token) -> uint32_t & { return bins[token + token / kPer]; };

    if (zero.take(tid)) return;
    const int i = start + tid;
    const bool live = tid < kSmallTile && i < N;
    const Entry mine = live ? src.at(i) : Entry{0, 0};
    for (int k = 4 * tid; k < kSmallBins + kSortThreads; k += 4 * kSortThreads)
        *reinterpret_cast<uint4 *>(&bins[k]) = uint4{0, 0, 0, 0};
    __syncthreads();
    for (int k = 0; k < N; k += kRead * kSortThreads) {
        uint32_t token[kRead];
#pragma unroll
        for (int j = 0; j < kRead; ++j) token[j] = src.at(min(k + j * kSortThreads + tid, N - 1)).token;
#pragma unroll
        for (int j = 0; j < kRead; ++j) {
            const int at = k + j * kSortThreads;
            if (at >= N) break;
            const bool in = at + tid < N;
            const uint32_t one = at + wave * kWave < start ? 0x10001u : 1u;   // the wave's: in one tile
            // 64 alike (padding) at once: additions to one counter go one by one
            if (__all(in && token[j] == __builtin_amdgcn_readfirstlane(token[j]))) {
                if (lane == 0) atomicAdd(&bin(token[j]), kWave * one);
            } else if (in) {
                atomicAdd(&bin(token[j]), one);
            }
        }
    }
    __syncthreads();
    uint32_t total = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) total += bins[tid * (kPer + 1) + j] & 0xffffu;
    const uint32_t inc = wave_scan(total, lane);
    if (lane == kWave - 1) sums[wave] = inc;
    __syncthreads();
    uint32_t below = lane < wave ? sums[lane] : 0;   // the waves' totals before this one's
#pragma unroll
    for (int off = kSortWaves / 2; off > 0; off >>= 1) below += __shfl_xor(below, off, kWave);
    below = __builtin_amdgcn_readfirstlane(below) + inc - total;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const uint32_t c = bins[tid * (kPer + 1) + j];
        bins[tid * (kPer + 1) + j] = below + (c >> 16);
        below += c & 0xffffu;
    }
    uint64_t same = __ballot(live);   // the wave's lanes with this token
#pragma unroll
    for (int b = 0; b < 15; ++b) {
        const uint64_t m = __ballot(mine.token >> b & 1);
        same &= (mine.token >> b & 1) ? m : ~m;
    }
    for (int w = 0; w < kSmallTile / kWave; ++w) {
        __syncthreads();
        if (wave != w || !live) continue;
        const uint32_t base = bin(mine.token);
        out[base + __popcll(same & ((1ull << lane) - 1))] = mine;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();   // every lane has read before the last of each token writes
        if ((same >> lane) == 1) bin(mine.token) = base + __popcll(same);
    }
}

// ---- the sums along the sorted order

constexpr int kAhead = 8;   // rows of dout, or partial sums, in flight per wave

// The first of the sorted entries lo .. N - 1 whose token is no less than t (N: none); the wave searches
// together, 65 ways a step.
__device__ __forceinline__ int lower_bound(const Entry *e, int lo, int N, uint32_t t, int lane) {
    int hi = N;   // the answer is in [lo, hi]
    while (hi > lo) {
        const int len = hi - lo, step = (len + kWave) / (kWave + 1);
        const int at = lo + (lane + 1) * step - 1;   // lane's probe
        const bool less = at < hi && e[at].token < t;
        const int n = __popcll(__ballot(less));      // probes are ordered: the first n are less
        lo += n * step;
        if (n < kWave) hi = min(hi, lo + step - 1);   // past the last probe: up to hi itself
    }
    return lo;
}

struct Sort {
    const Entry *entries;
    int N, V, D, chunk, chunks, pieces;   // chunk entries a wave, pieces vectors a row
};

// One wave per (chunk, strip of 64 vectors of columns); bound by the rows read and written: 16384 x 768
// fp32 rows into 32000 13 us, 5.6 TB/s; streaming loads and stores take a tenth less than ordinary ones. Runs of
// one token inside the chunk are written; a run that began before the chunk goes to partial[2 chunk],
// one that begins in it and goes on behind it to partial[2 chunk + 1], both fp32.
template <int DT>
__device__ __forceinline__ void sum_chunk(const Sort &s, const char *dout, char *dw, float *partial, float scale, int chunk,
                                          int strip, int lane) {
    constexpr int E = Elem<DT>::vec, B = Elem<DT>::bytes;
    const int i0 = chunk * s.chunk, i1 = min(s.N, i0 + s.chunk), piece = strip * kWave + lane;
    const bool live = piece < s.pieces;
    const int col = column<E>(live ? piece : s.pieces - 1, s.D);   // the others' loads: in the row, and dropped
    uint32_t token = s.entries[i0].token;
    const uint32_t last = s.entries[i1 - 1].token;
    bool open = i0 > 0 && s.entries[i0 - 1].token == token;      // the run began before
    const bool goes_on = i1 < s.N && s.entries[i1].token == last;
    float acc[E];
#pragma unroll
    for (int k = 0; k < E; ++k) acc[k] = 0.f;
    auto put_partial = [&](int slot) {
        if (live) store_sums(partial + (2 * static_cast<size_t>(chunk) + slot) * s.D, col, s.D, acc);
    };
    auto put_row = [&]() {
        if (token >= static_cast<uint32_t>(s.V) || !live) return;
        float x[E];
#pragma unroll
        for (int k = 0; k < E; ++k) x[k] = acc[k] * scale;
        store_vec<DT, true>(dw + static_cast<size_t>(token) * s.D * B, col, s.D, x);
    };
    constexpr int A = kAhead;
    u32x4_any w[A];
    uint32_t tok[A], next_tok[A];
    Entry mine{};   // 64 entries at once, lane by lane
    auto load = [&](int i, u32x4_any (&to)[A], uint32_t (&t)[A]) {
        if ((i - i0) % kWave == 0) mine = s.entries[min(i + lane, i1 - 1)];
#pragma unroll
        for (int j = 0; j < A; ++j) {
            const int from = (i - i0) % kWave + j;
            t[j] = __builtin_amdgcn_readlane(mine.token, from);
            to[j] = load_raw<DT>(dout + static_cast<size_t>(__builtin_amdgcn_readlane(mine.pos, from)) * s.D * B, col, s.D);
        }
    };
    load(i0, w, tok);
    for (int i = i0; i < i1; i += A) {
        u32x4_any next[A];
        if (i + A < i1) load(i + A, next, next_tok);   // on their way while these are summed
#pragma unroll
        for (int j = 0; j < A; ++j) {
            const bool in = i + j < i1;
            if (in && tok[j] != token) {
                if (open) put_partial(0);
                else put_row();
                open = false;
                token = tok[j];
#pragma unroll
                for (int k = 0; k < E; ++k) acc[k] = 0.f;
            }
            float x[E];
            unpack<DT>(w[j], x);
#pragma unroll
            for (int k = 0; k < E; ++k) acc[k] += in ? x[k] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < A; ++j) {
            w[j] = next[j];
            tok[j] = next_tok[j];
        }
    }
    if (open) put_partial(0);
    else if (goes_on) put_partial(1);
    else put_row();
}

constexpr int kZeroRows = 8;   // rows of dW a wave looks after behind a long sequence's sums: the absent ones are zeroed

template <int DT>
__global__ __launch_bounds__(kThreads) void sum_kernel(Sort s, const char *dout, char *dw, float *partial, float scale,
                                                       int strips, int sum_blocks) {
    constexpr int E = Elem<DT>::vec, B = Elem<DT>::bytes;
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    if (static_cast<int>(blockIdx.x) < sum_blocks) {
        const int id = blockIdx.x * (kThreads / kWave) + wave;
        if (id < s.chunks * strips) sum_chunk<DT>(s, dout, dw, partial, scale, id / strips, id % strips, lane);
        return;
    }
    // absent rows: 0
    const long long v0 = (static_cast<long long>(blockIdx.x - sum_blocks) * (kThreads / kWave) + wave) * kZeroRows;
    if (v0 >= s.V) return;
    const int rows = static_cast<int>(min(static_cast<long long>(kZeroRows), s.V - v0));
    uint32_t present = 0;
    int i = lower_bound(s.entries, 0, s.N, static_cast<uint32_t>(v0), lane);
    for (;;) {   // 64 entries, then on behind the last one's run: at most one turn a row
        uint32_t t = i + lane < s.N ? s.entries[i + lane].token - static_cast<uint32_t>(v0) : kZeroRows;
        uint32_t bits = t < kZeroRows ? 1u << t : 0;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) bits |= __shfl_xor(bits, off, kWave);
        present |= bits;
        t = __shfl(t, kWave - 1, kWave);
        if (t >= kZeroRows) break;
        i = lower_bound(s.entries, i + kWave, s.N, static_cast<uint32_t>(v0) + t + 1, lane);
    }
    float zero[E];
#pragma unroll
    for (int k = 0; k < E; ++k) zero[k] = 0.f;
    for (int r = 0; r < rows; ++r) {
        if (present >> r & 1) continue;
        for (int p = lane; p < s.pieces; p += kWave)
            store_vec<DT, true>(dw + static_cast<size_t>(v0 + r) * s.D * B, column<E>(p, s.D), s.D, zero);
    }
}

// Runs that go over chunks: a run's parts are added up where it begins. Each wave looks after one
// (strip, chunk) and joins what its run left in up to kAlone chunks; a longer run's are joined by all
// waves of the workgroup, each a contiguous share of them, and the waves' sums in order.
// The workgroup's chunks follow each other, so that hardly more than one long run begins in them.
constexpr int kJoinThreads = 512, kAlone = kAhead;

template <int E>
__device__ __forceinline__ void add_parts(const float *partial, int first, int from, int to, int col, int D, float (&acc)[E]) {
    for (int c = from; c < to; c += kAhead) {
        float x[kAhead][E];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int cc = min(c + j, to - 1);
            load_sums(partial + (2 * static_cast<size_t>(cc) + (cc == first)) * D, col, D, x[j]);
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
#pragma unroll
            for (int k = 0; k < E; ++k) acc[k] += c + j < to ? x[j][k] : 0.f;
    }
}

template <int DT>
__global__ __launch_bounds__(kJoinThreads) void join_kernel(Sort s, char *dw, const float *partial, float scale, int strips) {
    constexpr int E = Elem<DT>::vec, B = Elem<DT>::bytes, W = kJoinThreads / kWave;
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    __shared__ int runs[W][2];   // each wave's run: its first and last chunk, where it is for all to join
    __shared__ uint32_t tokens[W];
    __shared__ float part[W][kWave][E];

    auto put = [&](uint32_t token, int col, float (&acc)[E]) {
#pragma unroll
        for (int k = 0; k < E; ++k) acc[k] *= scale;
        store_vec<DT, true>(dw + static_cast<size_t>(token) * s.D * B, col, s.D, acc);
    };
    // the run that begins in `chunk` and goes on behind it, if there is one: its token and last chunk
    auto run_of = [&](int chunk, uint32_t &token, int &last) {
        const int i0 = chunk * s.chunk, i1 = i0 + s.chunk;
        if (i1 >= s.N) return false;
        const uint32_t before = i0 > 0 ? s.entries[i0 - 1].token : ~0u, first = s.entries[i0].token;
        const uint32_t after = s.entries[i1].token;
        token = s.entries[i1 - 1].token;
        if (token >= static_cast<uint32_t>(s.V) || after != token || (first == token && before == token)) return false;
        for (last = chunk;;) {   // the last chunk that begins with it
            const int c = last + 1 + lane;
            const uint64_t same = __ballot(c < s.chunks && s.entries[min(c, s.chunks - 1) * s.chunk].token == token);
            last += __popcll(same);
            if (~same) return true;
        }
    };
    const int id = blockIdx.x * W + wave, chunk = id % s.chunks;
    uint32_t token = 0;
    int last = 0;
    const bool found = id < s.chunks * strips && run_of(chunk, token, last), alone = found && last - chunk < kAlone;
    if (lane == 0) {
        runs[wave][0] = found && !alone ? chunk : -1;
        runs[wave][1] = last;
        tokens[wave] = token;
    }
    if (alone) {
        const int piece = id / s.chunks * kWave + lane, col = column<E>(min(piece, s.pieces - 1), s.D);
        float acc[E] = {};
        add_parts(partial, chunk, chunk, last + 1, col, s.D, acc);
        if (piece < s.pieces) put(token, col, acc);
    }
    __syncthreads();
    for (int w = 0; w < W; ++w) {
        const int first = runs[w][0];
        if (first < 0) continue;
        const int parts = runs[w][1] - first + 1, each = (parts + W - 1) / W, from = first + wave * each;
        const int piece = (blockIdx.x * W + w) / s.chunks * kWave + lane, col = column<E>(min(piece, s.pieces - 1), s.D);
        float acc[E] = {};
        add_parts(partial, first, from, min(first + parts, from + each), col, s.D, acc);
#pragma unroll
        for (int k = 0; k < E; ++k) part[wave][lane][k] = acc[k];
        __syncthreads();
        if (wave == 0 && piece < s.pieces) {
#pragma unroll
            for (int v = 1; v < W; ++v)
#pragma unroll
                for (int k = 0; k < E; ++k) acc[k] += part[v][lane][k];
            put(tokens[w], col, acc);
        }
        __syncthreads();
    }
}

constexpr int kMaxV = 1 << 28, kMaxD = 1 << 20;
constexpr long long kMaxN = 1LL << 30;

inline int passes_of(int V) {   // the digits of 0 .. V
    int bits = 1;
    while (bits < 31 && (static_cast<long long>(V) >> bits)) ++bits;
    return (bits + kBits - 1) / kBits;
}
// About 1024 chunks, of at least 16 entries: shorter ones fill the device, longer ones leave less to join
// (16384 x 768 fp32 rows of 32000 tokens 60, 62 and 80 us with 16, 64 and 128; 131072 240 with 8, 160 with 64).
inline int chunk_of(long long N) {
    int c = 16;
    while (c < 512 && c * 1024LL < N) c *= 2;
    return c;
}

struct Plan {
    Entry *a, *b;
    uint32_t *counts, *totals;
    float *partial;
    int tiles, chunks;
    size_t bytes;
};
inline Plan plan(void *ws, long long N, int D) {
    Plan p;
    Carver c(ws);
    p.tiles = static_cast<int>((N + kTile - 1) / kTile);
    p.chunks = static_cast<int>((N + chunk_of(N) - 1) / chunk_of(N));
    p.a = c.take<Entry>(N);
    p.b = c.take<Entry>(N);
    p.counts = c.take<uint32_t>(static_cast<size_t>(kBins) * p.tiles);
    p.totals = c.take<uint32_t>(kBins);
    p.partial = c.take<float>(2 * static_cast<size_t>(p.chunks) * D);
    p.bytes = c.off;
    return p;
}

int check(const char *fn, int dtype, long long N, int V, int D) {
    if (!valid_dtype(dtype)) return fail(ULM_ERR_INVALID, "%s: bad dtype %d", fn, dtype);
    if (N < 1 || N > kMaxN || V < 1 || V > kMaxV || D < 1 || D > kMaxD)
        return fail(ULM_ERR_INVALID, "%s: bad sizes N=%lld V=%d D=%d", fn, N, V, D);
    return ULM_OK;
}

template <class F> void by_dtype(int dtype, F f) {
    if (dtype == ULM_F32) f(std::integral_constant<int, ULM_F32>{});
    else if (dtype == ULM_BF16) f(std::integral_constant<int, ULM_BF16>{});
    else f(std::integral_constant<int, ULM_F16>{});
}

}  // namespace emb
}  // namespace ulm

using namespace ulm;

extern "C" int ulm_embed_fwd(const void *weight, int dtype, const long long *tokens, long long N, int V, int D, float scale,
                             void *out, void *stream) {
    ULM_TRY(emb::check("ulm_embed_fwd", dtype, N, V, D));
    ULM_REQUIRE(weight && tokens && out, "ulm_embed_fwd: null pointer");
    const int vec = dtype == ULM_F32 ? 4 : 8, pieces = (D + vec - 1) / vec;
    hipStream_t st = static_cast<hipStream_t>(stream);
    long long blocks = (N * pieces + emb::kThreads - 1) / emb::kThreads;
    if (blocks > 65536) blocks = 65536;
    emb::by_dtype(dtype, [&](auto dt) {
        emb::fwd_kernel<decltype(dt)::value><<<dim3(static_cast<unsigned>(blocks)), dim3(emb::kThreads), 0, st>>>(
            static_cast<const char *>(weight), tokens, static_cast<char *>(out), N, V, D, pieces, scale);
    });
    return check_launch("ulm_embed_fwd");
}

extern "C" size_t ulm_embed_bwd_workspace_bytes(long long N, int V, int D) {
    if (N < 1 || N > emb::kMaxN || V < 1 || V > emb::kMaxV || D < 1 || D > emb::kMaxD) return 0;
    return emb::plan(nullptr, N, D).bytes;
}

extern "C" int ulm_embed_bwd(const void *dout, int dtype, const long long *tokens, long long N, int V, int D, float scale,
                             void *dweight, void *workspace, size_t workspace_bytes, void *stream) {
    ULM_TRY(emb::check("ulm_embed_bwd", dtype, N, V, D));
    ULM_REQUIRE(dout && tokens && dweight && workspace, "ulm_embed_bwd: null pointer");
    const size_t need = ulm_embed_bwd_workspace_bytes(N, V, D);
    ULM_REQUIRE(workspace_bytes >= need, "ulm_embed_bwd: workspace %zu < %zu", workspace_bytes, need);
    const int chunks = emb::plan(nullptr, N, D).chunks;
    constexpr int W = emb::kThreads / kWave;
    const int vec = dtype == ULM_F32 ? 4 : 8, pieces = (D + vec - 1) / vec, strips = (pieces + kWave - 1) / kWave;
    const long long sum_blocks = (static_cast<long long>(chunks) * strips + W - 1) / W;
    const bool few = N <= emb::kShort;
    const long long zero_blocks = few ? 0 : (static_cast<long long>(V) + W * emb::kZeroRows - 1) / (W * emb::kZeroRows);
    constexpr int JW = emb::kJoinThreads / kWave;
    const long long join_blocks = (static_cast<long long>(chunks) * strips + JW - 1) / JW;
    ULM_REQUIRE(sum_blocks + zero_blocks < (1 << 24) && join_blocks < (1 << 23),
                "ulm_embed_bwd: N=%lld V=%d D=%d is too large", N, V, D);
    const emb::Plan p = emb::plan(workspace, N, D);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int n = static_cast<int>(N);
    emb::Source src{tokens, nullptr, V};
    int passes = emb::passes_of(V);
    emb::Zero zero{static_cast<char *>(dweight), static_cast<size_t>(V) * D * (dtype == ULM_F32 ? 4 : 2), 0};
    if (few && V <= emb::kSmallV && passes > 1) {
        zero.from = (n + emb::kSmallTile - 1) / emb::kSmallTile;
        const dim3 grid(zero.from + zero.blocks());
        emb::place_small_kernel<<<grid, dim3(emb::kSortThreads), 0, st>>>(src, n, p.a, zero);
        src = {nullptr, p.a, V};
        passes = 0;
    }
    for (int k = 0; k < passes; ++k) {
        emb::Entry *to = k % 2 ? p.b : p.a;
        const int shift = k * emb::kBits;
        if (few) {
            zero.from = (n + emb::kSortThreads - 1) / emb::kSortThreads;
            const dim3 grid(zero.from + (k ? 0 : zero.blocks()));
            emb::place_kernel<1, true><<<grid, dim3(emb::kSortThreads), 0, st>>>(src, n, shift, nullptr, 0, nullptr, to, zero);
        } else {
            emb::count_kernel<<<dim3(p.tiles), dim3(emb::kSortThreads), 0, st>>>(src, n, shift, p.counts, p.tiles);
            emb::scan_kernel<<<dim3(emb::kBins), dim3(kWave), 0, st>>>(p.counts, p.tiles, p.totals);
            emb::place_kernel<emb::kTile / emb::kSortThreads, false><<<dim3(p.tiles), dim3(emb::kSortThreads), 0, st>>>(
                src, n, shift, p.counts, p.tiles, p.totals, to, zero);
        }
        src = {nullptr, to, V};
    }
    const emb::Sort s{src.entries, n, V, D, emb::chunk_of(N), p.chunks, pieces};
    emb::by_dtype(dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        emb::sum_kernel<DT><<<dim3(static_cast<unsigned>(sum_blocks + zero_blocks)), dim3(emb::kThreads), 0, st>>>(
            s, static_cast<const char *>(dout), static_cast<char *>(dweight), p.partial, scale, strips,
            static_cast<int>(sum_blocks));
        if (p.chunks > 1)
            emb::join_kernel<DT><<<dim3(static_cast<unsigned>(join_blocks)), dim3(emb::kJoinThreads), 0, st>>>(
                s, static_cast<char *>(dweight), p.partial, scale, strips);
    });
    return check_launch("ulm_embed_bwd");
}
