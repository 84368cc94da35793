// Embedding lookup with scaling and the weight's gradient (nn.Embedding in
// UnifiedLM, model.py:117, 150):
//
//     out[n] = scale W[t_n]      dW[v] = scale sum over n with t_n = v of dout[n]
//
// The gradient's rows are summed in the order of n: the tokens are sorted with their
// positions by a stable radix sort, the rows of dout are summed along the sorted order in
// chunks of equal length, one wave each, and sums that go over a chunk's end are
// joined afterwards. No atomics on numbers: equal inputs give equal bits.
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

// elements [i, i + vec) of a row of D, zeros past its end
template <int DT> __device__ __forceinline__ void load_vec(const char *row, int i, int D, float (&x)[Elem<DT>::vec]) {
    constexpr int V = Elem<DT>::vec;
    if (i + V <= D) {
        unpack<DT>(*reinterpret_cast<const u32x4_any *>(row + static_cast<size_t>(i) * Elem<DT>::bytes), x);
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) x[k] = i + k < D ? load_as_f32(row, i + k, DT) : 0.f;
    }
}

template <int DT> __device__ __forceinline__ void store_vec(char *row, int i, int D, const float (&x)[Elem<DT>::vec]) {
    constexpr int V = Elem<DT>::vec;
    if (i + V <= D) {
        *reinterpret_cast<u32x4_any *>(row + static_cast<size_t>(i) * Elem<DT>::bytes) = pack<DT>(x);
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (i + k < D) store_from_f32(row, i + k, DT, x[k]);
    }
}

// ---- lookup: each thread one 16-byte piece of a row, pieces in order over the grid

template <int DT>
__global__ __launch_bounds__(kThreads) void fwd_kernel(const char *__restrict__ weight, const long long *__restrict__ tokens,
                                                       char *__restrict__ out, long long N, int V, int D, int pieces,
                                                       float scale) {
    constexpr int E = Elem<DT>::vec, B = Elem<DT>::bytes;
    const long long total = N * pieces, step = static_cast<long long>(gridDim.x) * kThreads;
    for (long long p = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x; p < total; p += step) {
        const long long n = p / pieces;
        const int i = static_cast<int>(p % pieces) * E;
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
constexpr int kTile = 4096;   // entries per workgroup of a pass

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

// counts[bin][tile]: the entries of each tile by their digit
__global__ __launch_bounds__(kSortThreads) void count_kernel(Source src, int N, int shift, uint32_t *counts, int tiles) {
    __shared__ uint32_t hist[kBins];
    for (int b = threadIdx.x; b < kBins; b += kSortThreads) hist[b] = 0;
    __syncthreads();
    const int tile = blockIdx.x, end = min(N, (tile + 1) * kTile);
    for (int i = tile * kTile + threadIdx.x; i < end; i += kSortThreads)
        atomicAdd(&hist[(src.at(i).token >> shift) & (kBins - 1)], 1u);
    __syncthreads();
    for (int b = threadIdx.x; b < kBins; b += kSortThreads) counts[static_cast<size_t>(b) * tiles + tile] = hist[b];
}

__device__ __forceinline__ uint32_t wave_scan(uint32_t v, int lane) {   // inclusive
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
        const uint32_t o = __shfl_up(v, off, kWave);
        if (lane >= off) v += o;
    }
    return v;
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

// Every entry of a tile to its place: the smaller digits' total, the same digit's entries in
// earlier tiles, in earlier waves of this tile, and among the lanes before.
__global__ __launch_bounds__(kSortThreads) void place_kernel(Source src, int N, int shift, const uint32_t *counts, int tiles,
                                                             const uint32_t *totals, Entry *out) {
    static_assert(kBins == kSortThreads, "one bin per thread");
    constexpr int kPer = kTile / kSortThreads;   // 64-entry rows of a wave
    __shared__ uint32_t base[kBins];
    __shared__ uint16_t seen[kSortWaves][kBins];   // a wave's entries of each digit, then those of the waves before it
    __shared__ uint32_t sums[kSortWaves];
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave, tile = blockIdx.x;

    const uint32_t total = totals[tid], inc = wave_scan(total, lane);
    if (lane == kWave - 1) sums[wave] = inc;
    for (int w = 0; w < kSortWaves; ++w) seen[w][tid] = 0;
    __syncthreads();
    uint32_t below = inc - total;
    for (int w = 0; w < wave; ++w) below += sums[w];
    base[tid] = below + counts[static_cast<size_t>(tid) * tiles + tile];

    Entry e[kPer];
    uint32_t rank[kPer];
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        const int i = tile * kTile + (wave * kPer + k) * kWave + lane;
        const bool live = i < N;
        e[k] = live ? src.at(i) : Entry{0, 0};
        const uint32_t digit = (e[k].token >> shift) & (kBins - 1);
        uint64_t same = __ballot(live);   // the lanes with this digit
        if (!live) same = ~same;
#pragma unroll
        for (int b = 0; b < kBits; ++b) {
            const uint64_t m = __ballot(digit >> b & 1);
            same &= (digit >> b & 1) ? m : ~m;
        }
        const uint32_t ahead = __popcll(same & ((1ull << lane) - 1));
        rank[k] = seen[wave][digit] + ahead;
        // the wave's own counters: every lane has read them before the last lane of each digit writes
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (live && (same >> lane) == 1) seen[wave][digit] = static_cast<uint16_t>(rank[k] + 1);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    uint32_t before = 0;
    for (int w = 0; w < kSortWaves; ++w) {
        const uint32_t c = seen[w][tid];
        seen[w][tid] = static_cast<uint16_t>(before);
        before += c;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        const int i = tile * kTile + (wave * kPer + k) * kWave + lane;
        if (i >= N) continue;
        const uint32_t digit = (e[k].token >> shift) & (kBins - 1);
        out[base[digit] + seen[wave][digit] + rank[k]] = e[k];
    }
}

// ---- the sums along the sorted order

constexpr int kAhead = 8;   // rows of dout in flight per wave

// The first of the sorted entries lo .. N - 1 whose token is no less than t (N: none); the wave searches together, 65 ways a step.
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
    int N, V, D, chunk, chunks;   // chunk entries a wave
};

// One wave per (chunk, strip of 64 vectors of columns). Runs of one token inside the chunk are
// written; a run that began before the chunk goes to partial[2 chunk], one that begins in it and
// goes on behind it to partial[2 chunk + 1], both fp32.
template <int DT>
__device__ __forceinline__ void sum_chunk(const Sort &s, const char *dout, char *dw, float *partial, float scale, int chunk,
                                          int strip, int lane) {
    constexpr int E = Elem<DT>::vec, B = Elem<DT>::bytes;
    const int i0 = chunk * s.chunk, i1 = min(s.N, i0 + s.chunk), col = (strip * kWave + lane) * E;
    uint32_t token = s.entries[i0].token;
    const uint32_t last = s.entries[i1 - 1].token;
    bool open = i0 > 0 && s.entries[i0 - 1].token == token;      // the run began before
    const bool goes_on = i1 < s.N && s.entries[i1].token == last;
    float acc[E];
#pragma unroll
    for (int k = 0; k < E; ++k) acc[k] = 0.f;
    auto put_partial = [&](int slot) {
#pragma unroll
        for (int k = 0; k < E; ++k)
            if (col + k < s.D) partial[(2 * static_cast<size_t>(chunk) + slot) * s.D + col + k] = acc[k];
    };
    auto put_row = [&]() {
        if (token >= static_cast<uint32_t>(s.V) || col >= s.D) return;
        float x[E];
#pragma unroll
        for (int k = 0; k < E; ++k) x[k] = acc[k] * scale;
        store_vec<DT>(dw + static_cast<size_t>(token) * s.D * B, col, s.D, x);
    };
    for (int i = i0; i < i1; i += kAhead) {
        float x[kAhead][E];
        uint32_t tok[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const Entry e = s.entries[min(i + j, i1 - 1)];
            tok[j] = e.token;
            if (col < s.D) load_vec<DT>(dout + static_cast<size_t>(e.pos) * s.D * B, col, s.D, x[j]);
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            if (i + j >= i1) break;
            if (tok[j] != token) {
                if (open) put_partial(0);
                else put_row();
                open = false;
                token = tok[j];
#pragma unroll
                for (int k = 0; k < E; ++k) acc[k] = 0.f;
            }
#pragma unroll
            for (int k = 0; k < E; ++k) acc[k] += x[j][k];
        }
    }
    if (open) put_partial(0);
    else if (goes_on) put_partial(1);
    else put_row();
}

constexpr int kZeroRows = 32;   // rows of dW a wave looks after: the absent ones are zeroed

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
        for (int c = lane * E; c < s.D; c += kWave * E) store_vec<DT>(dw + static_cast<size_t>(v0 + r) * s.D * B, c, s.D, zero);
    }
}

// Runs that go over chunks: the workgroup of the chunk in which one begins adds up its parts, each wave a
// contiguous share of them and the waves' sums in order.
template <int DT>
__global__ __launch_bounds__(kThreads) void join_kernel(Sort s, char *dw, const float *partial, float scale, int strips) {
    constexpr int E = Elem<DT>::vec, B = Elem<DT>::bytes, W = kThreads / kWave;
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int chunk = blockIdx.x / strips, strip = blockIdx.x % strips, col = (strip * kWave + lane) * E;
    const int i0 = chunk * s.chunk, i1 = i0 + s.chunk;
    if (i1 >= s.N) return;
    const uint32_t token = s.entries[i1 - 1].token;
    if (token >= static_cast<uint32_t>(s.V) || s.entries[i1].token != token) return;   // no run goes on from here
    if (s.entries[i0].token == token && i0 > 0 && s.entries[i0 - 1].token == token) return;   // it began earlier
    const int end = lower_bound(s.entries, i1, s.N, token + 1, lane);
    const int last = (end - 1) / s.chunk, parts = last - chunk + 1, each = (parts + W - 1) / W;
    const int from = chunk + wave * each, to = min(last + 1, from + each);
    float acc[E];
#pragma unroll
    for (int k = 0; k < E; ++k) acc[k] = 0.f;
    for (int c = from; c < to; c += kAhead) {
        float x[kAhead][E];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int cc = min(c + j, to - 1);
            const float *p = partial + (2 * static_cast<size_t>(cc) + (cc == chunk)) * s.D;
#pragma unroll
            for (int k = 0; k < E; ++k) x[j][k] = col + k < s.D ? p[col + k] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (c + j < to)
#pragma unroll
                for (int k = 0; k < E; ++k) acc[k] += x[j][k];
    }
    __shared__ float part[W][kWave][E];
#pragma unroll
    for (int k = 0; k < E; ++k) part[wave][lane][k] = acc[k];
    __syncthreads();
    if (wave || col >= s.D) return;
#pragma unroll
    for (int w = 1; w < W; ++w)
#pragma unroll
        for (int k = 0; k < E; ++k) acc[k] += part[w][lane][k];
#pragma unroll
    for (int k = 0; k < E; ++k) acc[k] *= scale;
    store_vec<DT>(dw + static_cast<size_t>(token) * s.D * B, col, s.D, acc);
}

constexpr int kMaxV = 1 << 30;
constexpr long long kMaxN = 1LL << 30;

inline int passes_of(int V) {   // the digits of 0 .. V
    int bits = 1;
    while (bits < 31 && (static_cast<long long>(V) >> bits)) ++bits;
    return (bits + kBits - 1) / kBits;
}
inline int chunk_of(long long N) { return N <= 65536 ? 32 : 128; }

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
    if (N < 1 || N > kMaxN || V < 1 || V > kMaxV || D < 1 || D > (1 << 24))
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
    long long blocks = (N * pieces + emb::kThreads - 1) / emb::kThreads;
    if (blocks > 65536) blocks = 65536;
    emb::by_dtype(dtype, [&](auto dt) {
        emb::fwd_kernel<decltype(dt)::value><<<dim3(static_cast<unsigned>(blocks)), dim3(emb::kThreads), 0, static_cast<hipStream_t>(stream)>>>(
            static_cast<const char *>(weight), tokens, static_cast<char *>(out), N, V, D, pieces, scale);
    });
    return check_launch("ulm_embed_fwd");
}

extern "C" size_t ulm_embed_bwd_workspace_bytes(long long N, int V, int D) {
    if (N < 1 || N > emb::kMaxN || V < 1 || V > emb::kMaxV || D < 1 || D > (1 << 24)) return 0;
    return emb::plan(nullptr, N, D).bytes;
}

extern "C" int ulm_embed_bwd(const void *dout, int dtype, const long long *tokens, long long N, int V, int D, float scale,
                             void *dweight, void *workspace, size_t workspace_bytes, void *stream) {
    ULM_TRY(emb::check("ulm_embed_bwd", dtype, N, V, D));
    ULM_REQUIRE(dout && tokens && dweight && workspace, "ulm_embed_bwd: null pointer");
    const size_t need = ulm_embed_bwd_workspace_bytes(N, V, D);
    ULM_REQUIRE(workspace_bytes >= need, "ulm_embed_bwd: workspace %zu < %zu", workspace_bytes, need);
    const int chunks = emb::plan(nullptr, N, D).chunks;
    const int vec = dtype == ULM_F32 ? 4 : 8, strips = (D + vec * kWave - 1) / (vec * kWave), W = emb::kThreads / kWave;
    const long long sum_blocks = (static_cast<long long>(chunks) * strips + W - 1) / W;
    const long long zero_blocks = (static_cast<long long>(V) + W * emb::kZeroRows - 1) / (W * emb::kZeroRows);
    const long long join_blocks = static_cast<long long>(chunks) * strips;
    ULM_REQUIRE(sum_blocks + zero_blocks < (1 << 24) && join_blocks < (1 << 24), "ulm_embed_bwd: N=%lld V=%d D=%d is too large", N, V, D);
    const emb::Plan p = emb::plan(workspace, N, D);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int n = static_cast<int>(N), passes = emb::passes_of(V);
    emb::Source src{tokens, nullptr, V};
    for (int k = 0; k < passes; ++k) {
        emb::Entry *to = k % 2 ? p.b : p.a;
        const int shift = k * emb::kBits;
        emb::count_kernel<<<dim3(p.tiles), dim3(emb::kSortThreads), 0, st>>>(src, n, shift, p.counts, p.tiles);
        emb::scan_kernel<<<dim3(emb::kBins), dim3(kWave), 0, st>>>(p.counts, p.tiles, p.totals);
        emb::place_kernel<<<dim3(p.tiles), dim3(emb::kSortThreads), 0, st>>>(src, n, shift, p.counts, p.tiles, p.totals, to);
        src = {nullptr, to, V};
    }
    const emb::Sort s{src.entries, n, V, D, emb::chunk_of(N), p.chunks};
    emb::by_dtype(dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        emb::sum_kernel<DT><<<dim3(static_cast<unsigned>(sum_blocks + zero_blocks)), dim3(emb::kThreads), 0, st>>>(
            s, static_cast<const char *>(dout), static_cast<char *>(dweight), p.partial, scale, strips, static_cast<int>(sum_blocks));
        if (p.chunks > 1)
            emb::join_kernel<DT><<<dim3(static_cast<unsigned>(join_blocks)), dim3(emb::kThreads), 0, st>>>(
                s, static_cast<char *>(dweight), p.partial, scale, strips);
    });
    return check_launch("ulm_embed_bwd");
}
