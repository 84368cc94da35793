// Log probabilities of given tokens, with each row's entropy and its largest
// entries, and the logits' gradient: the classifier's end of a training step
// (F.cross_entropy over the logits, model.py:160-161), of scoring and of a
// decode position.
//
// For a row x of V logits, m = max x, d_i = x_i - m, s = sum e^d_i:
//
//     logprob = d_t - ln s      entropy = ln s - (sum e^d_i d_i) / s      p_i = e^d_i / s
//     dx_i    = a [i = t] + sum_j c_j [i = top_j] - p_i (G + h (ln p_i + H)),  G = a + sum_j c_j
//
// with a, h, c_j the gradients of logprob, entropy and the top log probabilities.
#include <type_traits>

#include "logit_rows.h"

namespace ulm {
namespace lp {

using namespace rows;

constexpr int kUnroll = 4;            // 16-byte loads in flight per thread
constexpr int kMaxTop = 64;           // one lane of a wave each
constexpr int kMaxParts = 64;          // a row's, one lane of a wave each
constexpr int kMaxTopV = 1 << 22;      // columns with alternatives: kMaxParts parts of 65536
constexpr float kLn2 = 0.693147180559945309f;
constexpr float kFloor = -1e4f;       // 2^t and e^d are 0 from here on: keeps 0 x (-inf) out of the sums
constexpr float kHuge = 0x1p24f;      // maxima from which on m log2(e) is not formed: its rounding is at most 1 below

__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }

// The sums of a set of logits about their maximum m: s = sum e^(x - m), u = sum e^(x - m) (x - m).
struct Sums {
    float m, s, u;
    __device__ __forceinline__ void rebase(float to) {   // to >= m
        const float d = m == to ? 0.f : fmaxf(m - to, kFloor), f = exp_of(d);
        u = f * __builtin_fmaf(s, d, u);
        s *= f;
        m = to;
    }
};

// over groups of W lanes
template <int W> __device__ __forceinline__ Sums group_add(Sums v) {
    float to = v.m;
#pragma unroll
    for (int off = W / 2; off > 0; off >>= 1) to = fmaxf(to, __shfl_xor(to, off, kWave));
    v.rebase(to);
#pragma unroll
    for (int off = W / 2; off > 0; off >>= 1) {
        v.s += __shfl_xor(v.s, off, kWave);
        v.u += __shfl_xor(v.u, off, kWave);
    }
    return v;
}

// A thread's running sums in powers of two about ref = m log2(e), rounded: s = sum 2^t_i,
// u = sum 2^t_i t_i with t_i = x_i log2(e) - ref in one fused operation (5.5 instructions an
// element, conversion and maximum included, where differences from m itself and a guard for
// masked ones take 8: at 16384 rows of 32000 bf16 the ALUs were busy 83% of 204 us). The largest t is
// what ref lacks of m log2(e), half a step of ref: at most 1 below kHuge, and put right at the
// end. From kHuge on (rows masked with a large negative number, say) the powers
// 2^t would leave fp32's range: there t_i = (x_i - m) log2(e).
struct Running {
    float m = -INFINITY, s = 0.f, u = 0.f, lacks = 0.f;
    static __device__ __forceinline__ float ref(float m) { return m * kLog2e; }
    __device__ __forceinline__ bool plain() const { return fabsf(m) < kHuge; }
    __device__ __forceinline__ void rebase(float to) {   // to > m
        const float lacked = fabsf(to) < kHuge ? __builtin_fmaf(to, kLog2e, -ref(to)) : 0.f;
        // not ref(m) - ref(to): fused into one operation it takes m log2(e) for ref(m), unrounded, and the sums of a
        // row about 6e4 come out off by 1e-4
        const float d = __builtin_fmaf(m - to, kLog2e, lacked - lacks);
        const float t = fmaxf(d, kFloor), f = __builtin_amdgcn_exp2f(t);   // m = -inf: s and u are 0
        u = f * __builtin_fmaf(s, t, u);
        s *= f;
        m = to;
        lacks = lacked;
    }
    __device__ __forceinline__ Sums sums() const {
        const float f = __builtin_amdgcn_exp2f(-lacks);
        return {m, s * f, kLn2 * f * __builtin_fmaf(-lacks, s, u)};
    }
};

struct Rows {
    const char *x;
    const long long *tokens;
    long long inner, outer_stride, row_stride;   // row r starts at (r / inner) outer_stride + (r % inner) row_stride elements
    long long ignore, rows;
    int V, top, parts, part_len;
    __device__ __forceinline__ const char *row(long long r, int bytes) const {
        const long long outer = r < inner ? 0 : r / inner;   // mostly one stride: no division
        return x + (outer * outer_stride + (r - outer * inner) * row_stride) * bytes;
    }
};

struct Outs {
    float *logprob, *entropy, *top_logprobs, *stats;
    long long *top_tokens;
};

// what every row ends with, on one thread: its log probability, entropy and (m, ln s). The token t and,
// where there is one, its logit x were read ahead.
struct Target {
    long long t;
    float x;
};
template <int DT> __device__ __forceinline__ Target target_of(const Rows &a, const char *row, long long r) {
    const long long t = a.tokens[r];
    return {t, t >= 0 && t < a.V ? load_as_f32(row, t, DT) : 0.f};
}
__device__ __forceinline__ void finish_row(const Rows &a, const Outs &o, long long r, Target to, Sums v, float &m, float &logs) {
    logs = v.s > 0.f ? logf(v.s) : v.s == 0.f ? -INFINITY : v.s;   // an empty row: -inf; a NaN stays
    m = v.m;
    float lp = 0.f;
    if (to.t != a.ignore) {
        lp = __uint_as_float(0x7fc00000u);
        if (to.t >= 0 && to.t < a.V) lp = v.s == 0.f ? -INFINITY : (to.x - m) - logs;
    }
    o.logprob[r] = lp;
    o.entropy[r] = v.s == 0.f ? 0.f : logs - v.u / v.s;
    if (o.stats) {
        o.stats[2 * r] = m;
        o.stats[2 * r + 1] = logs;
    }
}

__device__ __forceinline__ void put_top(const Rows &a, const Outs &o, long long r, int rank, uint64_t key, float m, float logs) {
    const float x = value_of(key);
    o.top_logprobs[r * a.top + rank] = logs == -INFINITY ? -INFINITY : (x - m) - logs;
    o.top_tokens[r * a.top + rank] = index_of(key);
}

// The workgroup's batches: batch k of a thread is its kUnroll vectors of tile k.
template <int DT, int NT> struct Tile {
    static constexpr int vec = Elem<DT>::vec, size = NT * vec * kUnroll;
    static __device__ __forceinline__ int at(int e0, int k, int j, int tid) { return e0 + k * size + (j * NT + tid) * vec; }
};

// Room for the alternatives of a unit, by the workgroup's size, so that small ones fill a CU.
constexpr int batches_of(int NT) { return NT <= 256 ? 16 : 8; }
template <int NT> struct TopScratch {
    static constexpr int cap = NT < 256 ? 4 * NT : 1024;     // candidates held at once
    static constexpr int most_hits = NT < 256 ? 2 * NT : 512;   // batches read again at once
    static constexpr int tie_lanes = NT < 256 ? 16 : kWave;  // that look for equal ones, 8 elements each
    uint64_t list[cap + 8 * tie_lanes + kMaxTop];
    float table[batches_of(NT) * NT];   // the batches' maxima
    int hits[most_hits];
    int rank[kWave];
    int count, hit_count;
    uint64_t bound;
};

// The keys of elements [e0, e1) among which the `top` largest are, in sc.list; returns their number.
//
// sc.table holds every thread's largest element of each batch (NaN where the batch has one) and
// `mine` is the thread's largest of all. The top-th largest of 64 groups' maxima (a lane's
// across the waves), `low`, is no more than the top-th largest element; the few batches
// whose maximum is no less are read again, all of them at once. Where that is too many for
// the lists:
//   - many elements equal to `low` (a masked row, say): those above it, and in the order
//     of the row as many equal ones as are wanted;
//   - many above it (they lie in a few groups): every element is looked at in turns, each
//     with a higher bound, the top-th largest of the kCap keys that the turn before kept, so
//     that a turn leaves out kCap - top elements or more.
template <int DT, int NT>
__device__ int candidates(const char *row, int e0, int e1, int top, float mine, TopScratch<NT> &sc) {
    using T = Tile<DT, NT>;
    constexpr int V = T::vec, W = NT / kWave, kCap = TopScratch<NT>::cap, kHits = TopScratch<NT>::most_hits;
    constexpr int kTieLanes = TopScratch<NT>::tie_lanes;
    static_assert(W <= kWave && kWave % W == 0, "a share of the groups for every wave");
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    const int batches = (e1 - e0 + T::size - 1) / T::size;
    float *maxima = reinterpret_cast<float *>(sc.list);   // not in use yet
    static_assert(NT * sizeof(float) <= sizeof(sc.list), "scratch");
    maxima[tid] = mine;
    if (tid < kWave) sc.rank[tid] = 0;
    __syncthreads();
    float group = maxima[lane];
#pragma unroll
    for (int w = 1; w < W; ++w) group = fmaxf(group, maxima[lane + w * kWave]);
    int rank = 0;
#pragma unroll
    for (int i = 0; i < kWave / W; ++i) {
        const int j = wave * (kWave / W) + i;
        const float o = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(group), j));
        rank += o > group || (o == group && j < lane);
    }
    atomicAdd(&sc.rank[lane], rank);
    if (tid == 0) sc.count = sc.hit_count = 0;
    __syncthreads();
    const uint64_t which = __ballot(sc.rank[lane] == top - 1);   // one lane
    const float low = __shfl(group, __ffsll(static_cast<unsigned long long>(which)) - 1, kWave);

    auto push = [&](uint64_t key) {
        const int at = atomicAdd(&sc.count, 1);
        if (at < static_cast<int>(sizeof(sc.list) / sizeof(key))) sc.list[at] = key;
    };
    auto gather = [&](auto wanted) {   // the wanted elements, or more than kCap; counts are 0 before
        for (int k = 0; k < batches; ++k)
            if (wanted(sc.table[k * NT + tid])) {
                const int at = atomicAdd(&sc.hit_count, 1);
                if (at < kHits) sc.hits[at] = k * NT + tid;
            }
        __syncthreads();
        const int hits = sc.hit_count;
        if (hits > kHits) return kCap + 1;
        for (int h = tid / kUnroll; h < hits; h += NT / kUnroll) {
            const int i = T::at(e0, sc.hits[h] / NT, tid % kUnroll, sc.hits[h] % NT);
            if (i >= e1) continue;
            float x[V];
            load_vec<DT>(row, i, e1, x);
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (i + k < e1 && wanted(x[k])) push(key_of(x[k], i + k));
        }
        __syncthreads();
        return sc.count;
    };
    int n = gather([low](float x) { return !(x < low); });
    if (n <= kCap) return n;
    __syncthreads();
    if (tid == 0) sc.count = sc.hit_count = 0;
    __syncthreads();
    n = gather([low](float x) { return x > low || x != x; });
    if (n <= kCap) {
        if (wave == 0) {
            for (int i = e0 + lane * V; __any(i < e1); i += kTieLanes * V) {
                if (i < e1 && lane < kTieLanes) {
                    float x[V];
                    load_vec<DT>(row, i, e1, x);
#pragma unroll
                    for (int k = 0; k < V; ++k)
                        if (i + k < e1 && x[k] == low) push(key_of(x[k], i + k));
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
                if (__builtin_amdgcn_readfirstlane(*const_cast<volatile int *>(&sc.count)) >= n + top) break;
            }
        }
        __syncthreads();
        return sc.count;
    }
    if (tid == 0) sc.bound = 0;   // every key
    for (;;) {
        __syncthreads();
        if (tid == 0) sc.count = 0;
        __syncthreads();
        const uint64_t bound = sc.bound;
        for (int i = e0 + tid * V; i < e1; i += NT * V) {
            float x[V];
            load_vec<DT>(row, i, e1, x);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const uint64_t key = key_of(x[k], i + k);
                if (i + k < e1 && !(x[k] < low) && key >= bound) push(key);
            }
        }
        __syncthreads();
        n = sc.count;
        if (n <= kCap) return n;
        for (int i = tid; i < kCap; i += NT) {
            const uint64_t k = sc.list[i];
            int above = 0;
            for (int j = 0; j < kCap; ++j) above += sc.list[j] > k;
            if (above == top - 1) sc.bound = k;
        }
    }
}

// One batch of a thread added to its running sums; returns the batch's largest element.
template <int N> __device__ __forceinline__ float take(const float (&x)[N], bool guard, bool &masked, Running &v) {
    float most = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; i += 2) most = max3(most, x[i], x[i + 1]);
    if (most > v.m) v.rebase(most);
    if (v.m == -INFINITY) {   // nothing but masked elements so far (or NaN)
#pragma unroll
        for (int i = 0; i < N; ++i) v.s += x[i] != x[i] ? x[i] : 0.f;
    } else if (v.plain()) {
        const float ref = -Running::ref(v.m);
        float s = v.s, u = v.u;
        guard |= masked;
        if (!guard) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float t = __builtin_fmaf(x[i], kLog2e, ref), e = __builtin_amdgcn_exp2f(t);
                s += e;
                u = __builtin_fmaf(e, t, u);
            }
            guard = masked = u != u;   // 0 x (-inf), or a NaN among the elements
        }
        if (guard) {
            s = v.s;
            u = v.u;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float t = __builtin_fmaf(x[i], kLog2e, ref), e = __builtin_amdgcn_exp2f(t);
                s += e;
                u = __builtin_fmaf(e, fmaxf(t, kFloor), u);
            }
        }
        v.s = s;
        v.u = u;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float t = (x[i] - v.m) * kLog2e, e = __builtin_amdgcn_exp2f(t);
            v.s += e;
            v.u = __builtin_fmaf(e, fmaxf(t, kFloor), v.u);
        }
    }
    return most;
}

// One workgroup of NT threads per (row, part). With one part, as always without alternatives, it writes the
// row's outputs, with more the part's sums and its `top` best keys in order (0 where it has fewer). One pass over the
// row, which bounds it: 16384 rows of 32000 bf16 157 us, 6.7 TB/s. Workgroups that go from row to row with the
// next loads ahead took 197 (118 registers leave half the waves), the alternatives 30 more.
template <int DT, bool TOP, int NT>
__global__ __launch_bounds__(NT) void fwd_kernel(Rows a, Outs o, Sums *part_sums, uint64_t *part_keys) {
    using T = Tile<DT, NT>;
    constexpr int V = T::vec, W = NT / kWave;
    // Without alternatives r is id, e0 0 and e1 V, but with those constants the compiler settles on 64 registers
    // instead of 80, and 16 x 1023 rows of 32000 bf16 take 158.4 us instead of 157.2.
    const long long id = block_id(), r = a.parts == 1 ? id : id / a.parts;
    if (r >= a.rows) return;
    const int tid = threadIdx.x, part = static_cast<int>(id - r * a.parts);
    const char *row = a.row(r, Elem<DT>::bytes);
    const int e0 = part * a.part_len, e1 = min(a.V, e0 + a.part_len);
    const bool whole_row = !TOP || a.parts == 1;
    __shared__ std::conditional_t<TOP, TopScratch<NT>, int> scratch;

    const Target to = whole_row && tid == 0 ? target_of<DT>(a, row, r) : Target{};
    Running v;
    bool masked = false;   // -inf was met: its t is kept finite from then on
    for (int k = 0; e0 + k * T::size < e1; ++k) {
        float x[kUnroll * V];
        const bool whole = e0 + (k + 1) * T::size <= e1;
        if (e1 - e0 >= V) {   // every load inside the row: the last tile's overhang reads its last elements and drops them
            u32x4_any w[kUnroll];
#pragma unroll
            for (int j = 0; j < kUnroll; ++j)
                w[j] = load_once(row + static_cast<size_t>(min(T::at(e0, k, j, tid), e1 - V)) * Elem<DT>::bytes);
#pragma unroll
            for (int j = 0; j < kUnroll; ++j) unpack<DT>(w[j], *reinterpret_cast<float(*)[V]>(&x[j * V]));
            if (!whole) {
                asm volatile("");   // a branch: 64 selects in every tile otherwise
#pragma unroll
                for (int j = 0; j < kUnroll; ++j) {
                    const int over = T::at(e0, k, j, tid) - (e1 - V);   // the first `over` elements are others'
#pragma unroll
                    for (int i = 0; i < V; ++i) x[j * V + i] = i < over ? -INFINITY : x[j * V + i];
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < kUnroll; ++j)
                load_vec<DT>(row, T::at(e0, k, j, tid), e1, *reinterpret_cast<float(*)[V]>(&x[j * V]));
        }
        const float most = take(x, !whole, masked, v);
        if constexpr (TOP) scratch.table[k * NT + tid] = v.s == v.s ? most : __uint_as_float(0x7fc00000u);
    }

    __shared__ Sums waves[W];
    __shared__ float ml[2];
    const Sums w = group_add<kWave>(v.sums());
    if (tid % kWave == 0) waves[tid / kWave] = w;
    __syncthreads();
    if (tid < kWave) {
        const Sums all = group_add<W>(waves[tid % W]);
        if (tid == 0) {
            if (whole_row) finish_row(a, o, r, to, all, ml[0], ml[1]);
            else part_sums[id] = all;
        }
    }
    if constexpr (TOP) {
        const int n = candidates<DT, NT>(row, e0, e1, a.top, v.m, scratch);
        const float m = ml[0], logs = ml[1];
        for (int i = tid; i < n; i += NT) {
            const uint64_t k = scratch.list[i];
            int rank = 0;
            for (int j = 0; j < n; ++j) rank += scratch.list[j] > k;
            if (rank >= a.top) continue;
            if (whole_row) put_top(a, o, r, rank, k, m, logs);
            else part_keys[id * a.top + rank] = k;
        }
        if (!whole_row)
            for (int i = n + tid; i < a.top; i += NT) part_keys[id * a.top + i] = 0;
    }
}

constexpr int kThreads = 256;   // of the kernels below

// The parts of a row with alternatives joined: one workgroup per row.
template <int DT>
__global__ __launch_bounds__(kThreads) void join_kernel(Rows a, Outs o, const Sums *part_sums, const uint64_t *part_keys) {
    const long long r = block_id();
    if (r >= a.rows) return;
    const int tid = threadIdx.x;
    __shared__ float ml[2];
    __shared__ uint64_t list[kMaxParts * kMaxTop];
    const int n = a.parts * a.top;
    for (int i = tid; i < n; i += kThreads) list[i] = part_keys[r * n + i];
    if (tid < kWave) {   // at most a wave's lanes of parts
        const Sums all = group_add<kWave>(tid < a.parts ? part_sums[r * a.parts + tid] : Sums{-INFINITY, 0.f, 0.f});
        if (tid == 0) finish_row(a, o, r, target_of<DT>(a, a.row(r, Elem<DT>::bytes), r), all, ml[0], ml[1]);
    }
    __syncthreads();
    const float m = ml[0], logs = ml[1];
    for (int i = tid; i < n; i += kThreads) {
        const uint64_t k = list[i];
        if (k == 0) continue;
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += list[j] > k;
        if (rank < a.top) put_top(a, o, r, rank, k, m, logs);
    }
}

struct Grads {
    const float *stats, *entropy, *dlogprob, *dentropy, *dtop;
    const long long *top_tokens;
    char *dx;   // (rows, V), dense
};

// One workgroup per (row, tile of U vectors a thread). At 16384 x 32000 in bf16 340 us, 6.2 TB/s, with one
// vector a thread and stores that leave the caches to others; 404 with ordinary stores, 357 and 360
// with two and four vectors. With alternatives a workgroup has more to do besides (their gradients' sum,
// their elements), and two vectors share it: 16384 x 32000 in bf16 with 5 of them and the entropy 381 us,
// 464 with one (364 with four, but 90 instead of 85 at 2048 x 32000 in fp32 with 20). From the last row
// back: the caches still hold what the forward read last (1% of the pair from 2048 to 16384 rows).
template <int DT, bool ENT, int U>
__global__ __launch_bounds__(kThreads) void bwd_kernel(Rows a, Grads g, int tiles) {
    constexpr int V = Elem<DT>::vec, kTile = kThreads * V * U, B = Elem<DT>::bytes;
    const long long id = a.rows * tiles - 1 - block_id();
    if (id < 0) return;
    const long long r = id / tiles;
    const int tid = threadIdx.x, lane = tid % kWave;
    const int e0 = static_cast<int>(id - r * tiles) * kTile, e1 = min(a.V, e0 + kTile);
    const char *row = a.row(r, B);
    char *out = g.dx + static_cast<size_t>(r) * a.V * B;
    // the row's numbers first: they arrive while its elements are under way
    const float m = g.stats[2 * r], logs = g.stats[2 * r + 1];
    const float h = ENT ? g.dentropy[r] : 0.f, H = ENT ? g.entropy[r] : 0.f;
    const long long t = a.tokens[r];
    const float dl = g.dlogprob ? g.dlogprob[r] : 0.f;
    float x[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int i = e0 + (u * kThreads + tid) * V;
        if (i < e1) load_vec<DT>(row, i, e1, x[u]);
    }

    float da = t != a.ignore ? dl : 0.f;
    if (t != a.ignore && (t < 0 || t >= a.V)) da = __uint_as_float(0x7fc00000u);
    float G = da, dc = 0.f;
    long long which = -1;   // lane's alternative, and its gradient
    if (g.dtop) {
        if (lane < a.top) {
            dc = g.dtop[r * a.top + lane];
            which = g.top_tokens[r * a.top + lane];
        }
        G += wave_sum(dc);
    }
    const bool empty = m == -INFINITY && logs == -INFINITY;
    auto grad = [&](float x) {   // without the tokens' own terms
        const float d = x - m, p = exp_of(d - logs);
        const float f = ENT ? __builtin_fmaf(h, (fmaxf(d, kFloor) - logs) + H, G) : G;
        return empty ? 0.f : -p * f;
    };
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int i = e0 + (u * kThreads + tid) * V;
        if (i >= e1) continue;
        const long long own = t - i;   // the token's place among these
#pragma unroll
        for (int k = 0; k < V; ++k) {
            x[u][k] = grad(x[u][k]);
            if (own == k && !empty) x[u][k] += da;
        }
        if (i + V <= e1) {
            u32x4_any w;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if constexpr (DT == ULM_F32) w[k] = __float_as_uint(x[u][k]);
                else w[k] = pack_word<DT>(x[u][2 * k], x[u][2 * k + 1]);
            }
            __builtin_nontemporal_store(w, reinterpret_cast<u32x4_any *>(out + static_cast<size_t>(i) * B));
        } else {
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (i + k < e1) store_from_f32(out, i + k, DT, x[u][k]);
        }
    }
    if (!g.dtop || empty) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the streaming stores are done
    __syncthreads();   // the alternatives' elements are written again, with their own terms
    if (tid < a.top && which >= e0 && which < e1)
        store_from_f32(out, which, DT, grad(load_as_f32(row, which, DT)) + dc + (which == t ? da : 0.f));
}

// How the rows are spread: a function of the sizes, the same for the workspace and the launch. A
// workgroup as large as leaves a row two tiles, at most 256 threads: at 16384 rows of 200 bf16 16 us
// with 64 threads (39 with 256); of 8000 48 with 128 (56); of 32000 178 with 256 (183 with 128, 179 with
// 512; ordinary loads). Up to 512 rows do not fill the device: twice as many threads a row
// (256 rows of 32000 fp32 and 20 alternatives 10.7 us, 13.1 with 256; one row 7.3 and 9.4).
struct Plan {
    int threads, parts, part_len;
};
inline Plan plan_of(long long rows, int V, int top, int dtype) {
    Plan p{64, 1, V};
    const int vec = dtype == ULM_F32 ? 4 : 8;
    while (p.threads < 256 && V >= 2 * p.threads * vec * kUnroll) p.threads *= 2;
    if (rows <= 512 && V >= p.threads * vec * kUnroll / 4) p.threads *= 2;
    // the alternatives' table holds so many tiles
    const long long most = static_cast<long long>(batches_of(p.threads)) * p.threads * vec * kUnroll;
    const long long parts = top ? (V + most - 1) / most : 1;
    if (parts > 1) {
        p.parts = static_cast<int>(parts);
        p.part_len = static_cast<int>((V + parts * 8 - 1) / (parts * 8) * 8);   // whole 8-element vectors
    }
    return p;
}

}  // namespace lp
}  // namespace ulm

using namespace ulm;

static int check_rows(const char *fn, long long rows, long long inner, int V, int top, int dtype) {
    if (rows < 1 || rows > (1LL << 34) || inner < 1 || V < 1 || V > (1 << 30))
        return fail(ULM_ERR_INVALID, "%s: bad sizes rows=%lld inner=%lld V=%d", fn, rows, inner, V);
    if (top < 0 || top > lp::kMaxTop || top > V)
        return fail(ULM_ERR_INVALID, "%s: top=%d outside 0 .. min(V, %d)", fn, top, lp::kMaxTop);
    if (top && V > lp::kMaxTopV) return fail(ULM_ERR_INVALID, "%s: top=%d with V=%d", fn, top, V);
    if (!valid_dtype(dtype)) return fail(ULM_ERR_INVALID, "%s: bad dtype %d", fn, dtype);
    return ULM_OK;
}

extern "C" int ulm_token_logprobs_max_top(void) { return lp::kMaxTop; }

extern "C" size_t ulm_token_logprobs_workspace_bytes(long long rows, int V, int top, int dtype) {
    if (rows < 1 || V < 1 || top < 0 || top > lp::kMaxTop || !valid_dtype(dtype)) return 0;
    const int parts = lp::plan_of(rows, V, top, dtype).parts;
    if (parts == 1) return 0;
    Carver c(nullptr);
    c.take<lp::Sums>(static_cast<size_t>(rows) * parts);
    c.take<uint64_t>(static_cast<size_t>(rows) * parts * top);
    return c.off;
}

extern "C" int ulm_token_logprobs(const void *logits, int dtype, const long long *tokens, long long rows, long long inner,
                                  long long outer_stride, long long row_stride, int V, int top, long long ignore_index,
                                  float *logprob, float *entropy, float *top_logprobs, long long *top_tokens, float *stats,
                                  void *workspace, size_t workspace_bytes, void *stream) {
    ULM_TRY(check_rows("ulm_token_logprobs", rows, inner, V, top, dtype));
    ULM_REQUIRE(logits && tokens && logprob && entropy && (top == 0 || (top_logprobs && top_tokens)),
                "ulm_token_logprobs: null pointer");
    const lp::Plan plan = lp::plan_of(rows, V, top, dtype);
    const int parts = plan.parts;
    const size_t need = ulm_token_logprobs_workspace_bytes(rows, V, top, dtype);
    ULM_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), "ulm_token_logprobs: workspace %zu < %zu",
                workspace_bytes, need);
    Carver c(workspace);
    lp::Sums *sums = parts > 1 ? c.take<lp::Sums>(static_cast<size_t>(rows) * parts) : nullptr;
    uint64_t *keys = parts > 1 ? c.take<uint64_t>(static_cast<size_t>(rows) * parts * top) : nullptr;
    const lp::Rows a{static_cast<const char *>(logits), tokens, inner, outer_stride, row_stride, ignore_index, rows, V, top,
                     parts, plan.part_len};
    const lp::Outs o{logprob, entropy, top_logprobs, stats, top_tokens};
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto launch = [&](auto dt, auto with_top) {
        constexpr int DT = decltype(dt)::value;
        constexpr bool TOP = decltype(with_top)::value;
        const dim3 grid = lp::grid_of(rows * parts);
        if (plan.threads == 64) lp::fwd_kernel<DT, TOP, 64><<<grid, dim3(64), 0, s>>>(a, o, sums, keys);
        else if (plan.threads == 128) lp::fwd_kernel<DT, TOP, 128><<<grid, dim3(128), 0, s>>>(a, o, sums, keys);
        else if (plan.threads == 256) lp::fwd_kernel<DT, TOP, 256><<<grid, dim3(256), 0, s>>>(a, o, sums, keys);
        else lp::fwd_kernel<DT, TOP, 512><<<grid, dim3(512), 0, s>>>(a, o, sums, keys);
        if constexpr (TOP)
            if (parts > 1) lp::join_kernel<DT><<<lp::grid_of(rows), dim3(lp::kThreads), 0, s>>>(a, o, sums, keys);
    };
    auto by_top = [&](auto dt) {
        if (top) launch(dt, std::true_type{});
        else launch(dt, std::false_type{});
    };
    if (dtype == ULM_F32) by_top(std::integral_constant<int, ULM_F32>{});
    else if (dtype == ULM_BF16) by_top(std::integral_constant<int, ULM_BF16>{});
    else by_top(std::integral_constant<int, ULM_F16>{});
    return check_launch("ulm_token_logprobs");
}

extern "C" int ulm_token_logprobs_bwd(const void *logits, int dtype, const long long *tokens, long long rows, long long inner,
                                      long long outer_stride, long long row_stride, int V, int top, long long ignore_index,
                                      const float *stats, const float *entropy, const long long *top_tokens,
                                      const float *dlogprob, const float *dentropy, const float *dtop, void *dlogits,
                                      void *stream) {
    ULM_TRY(check_rows("ulm_token_logprobs_bwd", rows, inner, V, top, dtype));
    ULM_REQUIRE(logits && tokens && stats && dlogits && (!dentropy || entropy) && (!dtop || (top_tokens && top)),
                "ulm_token_logprobs_bwd: null pointer");
    ULM_REQUIRE(dlogits != logits, "ulm_token_logprobs_bwd: dlogits must not alias logits");
    const int each = dtop ? 2 : 1;   // vectors a thread
    const int tile = lp::kThreads * each * (dtype == ULM_F32 ? 4 : 8), tiles = (V + tile - 1) / tile;
    const lp::Rows a{static_cast<const char *>(logits), tokens, inner, outer_stride, row_stride, ignore_index, rows, V, top,
                     1, V};
    const lp::Grads g{stats, entropy, dlogprob, dentropy, dtop, top_tokens, static_cast<char *>(dlogits)};
    hipStream_t s = static_cast<hipStream_t>(stream);
    const dim3 grid = lp::grid_of(rows * tiles), block(lp::kThreads);
    auto launch = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        if (each == 2) {
            if (dentropy) lp::bwd_kernel<DT, true, 2><<<grid, block, 0, s>>>(a, g, tiles);
            else lp::bwd_kernel<DT, false, 2><<<grid, block, 0, s>>>(a, g, tiles);
        } else {
            if (dentropy) lp::bwd_kernel<DT, true, 1><<<grid, block, 0, s>>>(a, g, tiles);
            else lp::bwd_kernel<DT, false, 1><<<grid, block, 0, s>>>(a, g, tiles);
        }
    };
    if (dtype == ULM_F32) launch(std::integral_constant<int, ULM_F32>{});
    else if (dtype == ULM_BF16) launch(std::integral_constant<int, ULM_BF16>{});
    else launch(std::integral_constant<int, ULM_F16>{});
    return check_launch("ulm_token_logprobs_bwd");
}
