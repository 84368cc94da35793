// Drawing tokens: one a row from its logits, with temperature, top-k, top-p and
// min-p, from given random numbers (what the reference's generate and run.c's
// sampler do on the host's side of the logits: model.py:205-222, sample.py:61).
//
// For a row x at temperature T, w_i = e^((x_i - max x) / T). In the order of the
// keys (by value down, the lower index first) the kept entries are a prefix:
//
//     rank j is kept iff j = 0, or j < k and sum_(ranks < j) w < p sum_(ranks < k) w and w_j >= min_p
//
// so that one key, the last kept one's, says what is kept. The token is the first kept index at
// which the running sum of kept w exceeds u times their sum.
//
// A token is right or wrong: where the sum is within its rounding of a border another token comes
// out. Sums in fp32 (2^-24 of the whole, with 32000 borders in a row) would draw another token once in
// some hundred rows. So w is formed in double (fp64 operations run at fp32's rate on this card)
// and rounded to an integer multiple of 2^-47 or, in rows past 2^15 columns, of so much that all of
// them add up in 62 bits: sums that depend on no order, whatever the waves and atomics do.
#include <atomic>
#include <type_traits>

#include "logit_rows.h"

namespace ulm {
namespace smp {

using namespace rows;

constexpr int kMaxV = 1 << 22;
constexpr int kBins = 1024;             // of the exact search
constexpr int kFine = 2048;             // of the estimate
constexpr float kBinsPerNat = 32.f, kFinePerNat = 96.f;   // 32 and 21 nats
constexpr int kList = 512;              // entries that the estimate's way holds
constexpr int kShort = 256;             // and the short way
constexpr int kGroups = 128;            // groups of threads whose maxima bound the k-th largest entry

constexpr int kMostHeld = 142 << 10;    // bytes of a row, or of its table, in LDS

typedef unsigned long long u64;

struct Setting {
    double one;
    const float *each;
    __device__ __forceinline__ double at(long long r) const { return each ? static_cast<double>(each[r]) : one; }
};

struct Args {
    View v;
    const void *u;
    Setting temperature, top_p, min_p;
    long long top_k;
    const long long *top_ks;
    long long *token, *kept;
    float *logprob;
    int u_double, bits;   // w in units of 2^-bits
    int tabled;           // LDS holds the largest of every vector of a row that is read again
};

// w = e^((x - m) / T) = 2^t: with t = n + f, |f| <= 1/2, as 2^n (1 + f g(f)), g of degree 8 through (2^f - 1) / f at
// Chebyshev's nodes (off by 4e-14 of w). Additions of large powers of two round t to n and w to its units,
// which they leave in the low bits of the sums: 21 instructions an entry.
struct Mass {
    double m, c, least, magic;   // c = log2(e) / T, least: (x - m) c = -1000, magic = 2^(52 - bits)
    __device__ __forceinline__ Mass(float max, double inv, int bits)
        : m(static_cast<double>(max)), c(1.4426950408889634074 * inv), least(-1000. / c), magic(__builtin_ldexp(1., 52 - bits)) {}
    __device__ __forceinline__ double real(float x) const {
        constexpr double shift = 6755399441055744.;   // 1.5 2^52
        const double d = fmax(static_cast<double>(x) - m, least);
        const double k = __builtin_fma(d, c, shift), n = k - shift, f = __builtin_fma(d, c, -n);
        double g = 1.0203121063391729e-07;
        g = __builtin_fma(g, f, 1.3255224878668817e-06);
        g = __builtin_fma(g, f, 1.525268684626772e-05);
        g = __builtin_fma(g, f, 0.00015403455852453838);
        g = __builtin_fma(g, f, 0.0013333558179043112);
        g = __builtin_fma(g, f, 0.009618129159402558);
        g = __builtin_fma(g, f, 0.055504108664760424);
        g = __builtin_fma(g, f, 0.2402265069581299);
        g = __builtin_fma(g, f, 0.6931471805599453);
        g = __builtin_fma(g, f, 1.);
        const u64 e = __builtin_bit_cast(u64, g) + (__builtin_bit_cast(u64, k) << 52);
        return __builtin_bit_cast(double, e);
    }
    __device__ __forceinline__ u64 units(double e) const { return __builtin_bit_cast(u64, e + magic) & ((1ull << 52) - 1); }
    __device__ __forceinline__ u64 operator()(float x) const { return units(real(x)); }
};

// A wave's inclusive scan: within rows of 16 lanes, then from row to row; 4 instructions a step and word where a
// shuffle through LDS takes some 60 cycles.
template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t moved(uint32_t v) {   // 0 where nothing comes in
    return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS> __device__ __forceinline__ u64 moved(u64 v) {
    return static_cast<u64>(moved<CTRL, ROWS>(static_cast<uint32_t>(v >> 32))) << 32 | moved<CTRL, ROWS>(static_cast<uint32_t>(v));
}
template <class T, class Op> __device__ __forceinline__ T wave_scan(T v, Op op) {   // 0 is the operation's neutral element
    v = op(v, moved<0x111, 0xf>(v));   // from 1, 2, 4 and 8 lanes below in the row
    v = op(v, moved<0x112, 0xf>(v));
    v = op(v, moved<0x114, 0xf>(v));
    v = op(v, moved<0x118, 0xf>(v));
    v = op(v, moved<0x142, 0xa>(v));   // the last lane of the row below, into rows 1 and 3
    v = op(v, moved<0x143, 0xc>(v));   // lane 31, into rows 2 and 3
    return v;
}
struct Plus {
    template <class T> __device__ __forceinline__ T operator()(T a, T b) const { return a + b; }
};
struct Larger {
    __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const { return max(a, b); }
};
__device__ __forceinline__ u64 wave_scan(u64 v) { return wave_scan(v, Plus()); }
__device__ __forceinline__ u64 lane_of(u64 v, int lane) {   // lane uniform
    return static_cast<u64>(__builtin_amdgcn_readlane(static_cast<uint32_t>(v >> 32), lane)) << 32 |
           static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<uint32_t>(v), lane));
}

__device__ __forceinline__ u64 wave_add(u64 v) { return lane_of(wave_scan(v), kWave - 1); }
// the largest of floats, as order-keeping whole numbers; none is NaN
__device__ __forceinline__ float wave_max(float x) {
    const uint32_t top = wave_scan(static_cast<uint32_t>(key_of(x, 0) >> 32), Larger());
    return value_of(static_cast<u64>(__builtin_amdgcn_readlane(top, kWave - 1)) << 32);
}

// The workgroup's row. A wave has a run of `count` tiles, 64 vectors each, from element `from` on. HELD: read once, into LDS
// (what lies past the row's end is -inf); otherwise read again by every pass, but for those that look for large
// entries where LDS holds every vector's largest (tabled). Held in registers, 64 a thread for 32000 fp32, the row
// left the passes too few.
template <int DT, int NT, bool HELD> struct Row {
    static constexpr int vec = Elem<DT>::vec, tile = kWave * vec, W = NT / kWave, kBatch = HELD ? 8 : 4;
    const char *row;
    u32x4_any *held;
    float *table;
    int n, run, from, count, lane;   // run: elements of a wave's run

    __device__ __forceinline__ Row(const Args &a, long long r, int tid, u32x4_any *lds)
        : row(a.v.row(r, Elem<DT>::bytes)), held(lds), table(!HELD && a.tabled ? reinterpret_cast<float *>(lds) : nullptr),
          n(a.v.V), lane(tid % kWave) {
        const int tiles = (n + tile - 1) / tile, per_wave = (tiles + W - 1) / W, wave = tid / kWave;
        run = per_wave * tile;
        from = wave * run;
        count = max(0, min(per_wave, tiles - wave * per_wave));
    }
    __device__ __forceinline__ int at(int t) const { return from + t * tile + lane * vec; }
    __device__ __forceinline__ u32x4_any read(int i) const {
        const uint32_t none = DT == ULM_F32 ? 0xff800000u : DT == ULM_BF16 ? 0xff80ff80u : 0xfc00fc00u;
        u32x4_any v = {none, none, none, none};
        const char *p = row + static_cast<size_t>(i) * Elem<DT>::bytes;
        if (i + vec <= n) {
            v = HELD ? load_once(p) : *reinterpret_cast<const u32x4_any *>(p);
        } else if constexpr (DT == ULM_F32) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (i + k < n) v[k] = reinterpret_cast<const uint32_t *>(p)[k];
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (i + k < n) {
                    const uint32_t b = reinterpret_cast<const uint16_t *>(p)[k];
                    v[k / 2] = k % 2 ? (v[k / 2] & 0xffffu) | b << 16 : (v[k / 2] & 0xffff0000u) | b;
                }
        }
        return v;
    }
    __device__ __forceinline__ void vector(int i, float (&x)[vec]) const { unpack<DT>(HELD ? held[i / vec] : read(i), x); }
    // f(elements, index of the first, tile) with a batch of loads under way
    template <class F> __device__ __forceinline__ void batches(F f) const {
        for (int t0 = 0; t0 < count; t0 += kBatch) {
            u32x4_any w[kBatch];
#pragma unroll
            for (int t = 0; t < kBatch; ++t) w[t] = read(t0 + t < count ? at(t0 + t) : n);
#pragma unroll
            for (int t = 0; t < kBatch; ++t)
                if (t0 + t < count) f(w[t], at(t0 + t));
        }
    }
    // the first pass over the row: f(elements) returns their largest
    template <class F> __device__ __forceinline__ void start(F f) const {
        batches([&](const u32x4_any &w, int i) {
            float x[vec];
            unpack<DT>(w, x);
            const float most = f(x);
            if constexpr (HELD) held[i / vec] = w;
            else if (table) table[i / vec] = most;
        });
    }
    // f(elements, index of the first)
    template <class F> __device__ __forceinline__ void tiles(F f) const {
        if constexpr (HELD) {
            for (int t = 0; t < count; ++t) {
                float x[vec];
                vector(at(t), x);
                f(x, at(t));
            }
        } else {
            batches([&](const u32x4_any &w, int i) {
                float x[vec];
                unpack<DT>(w, x);
                f(x, i);
            });
        }
    }
    // the same without tiles in which none is `low` (above -inf) or more
    template <class F> __device__ __forceinline__ void large_tiles(float low, F f) const {
        if (!HELD && table) {
            for (int t = 0; t < count; ++t) {
                if (!__any(table[at(t) / vec] >= low)) continue;
                float x[vec];
                vector(at(t), x);
                f(x, at(t));
            }
        } else {
            tiles([&](const float (&x)[vec], int i) {
                float most = x[0];
#pragma unroll
                for (int k = 1; k < vec; ++k) most = fmaxf(most, x[k]);
                if (__any(most >= low)) f(x, i);
            });
        }
    }
    // f(element, index) of those that are not masked and at least `low`
    template <class F> __device__ __forceinline__ void each(float low, F f) const {
        low = fmaxf(low, -__FLT_MAX__);
        large_tiles(low, [&](const float (&x)[vec], int i) {
#pragma unroll
            for (int k = 0; k < vec; ++k)
                if (x[k] >= low) f(x[k], i + k);
        });
    }
};

struct __attribute__((aligned(16))) Entry {
    u64 key, weight;
};

template <int NT> struct Scratch {
    union {
        u64 mass[kBins];
        u64 estimate[kFine];
        float top[NT];
        struct {
            Entry list[kList];
            u64 before_of[kList];
        };
        struct {
            u64 key[kShort], sorted[kWave];
            int rank[kShort];
        };
    };
    u64 few[kWave];
    u64 wave_mass[NT / kWave];
    int wave_count[NT / kWave];
    float wave_top[NT / kWave];
    u64 lo, hi, before, found;
    float low;
    int held, bin, first, odd;
};

// The sum over the workgroup, on every thread.
template <int NT> __device__ __forceinline__ u64 group_sum(u64 v, Scratch<NT> &sc) {
    v = wave_add(v);
    if (threadIdx.x % kWave == 0) sc.wave_mass[threadIdx.x / kWave] = v;
    __syncthreads();
    u64 all = 0;
#pragma unroll
    for (int i = 0; i < NT / kWave; ++i) all += sc.wave_mass[i];
    __syncthreads();
    return all;
}

// The last kept key where the first `k` ranks are kept (MASS false), or those before which lies less than `goal` of mass
// (MASS true). Only keys of `least` and above exist.
//
// The entries are sorted into bins by an order-keeping function: at first by their distance from the
// largest, 1/32 nat a bin, then by the bits of their keys, which are unique, until the
// bin in which the last kept one lies holds no more than a wave can rank. (LDS adds whole numbers of 64 bits in 3 us
// for a row of 32000, floats in 41.)
template <bool MASS, int DT, int NT, bool HELD>
__device__ __forceinline__ u64 last_key(const Row<DT, NT, HELD> &row, const Mass &mass, float m, float scale, u64 least, int k,
                                        double goal, Scratch<NT> &sc) {
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    const float low = least ? value_of(least) : -INFINITY;
    u64 lo = 0, hi = 0, above = 0;   // the window of keys, and what lies above it: mass, or entries
    bool first = true;
    int shift = 0;
    auto falls_short = [&](u64 before) { return MASS ? static_cast<double>(before) < goal : before < static_cast<u64>(k); };
    for (;;) {
        for (int i = tid; i < kBins; i += NT) sc.mass[i] = 0;
        if (tid == 0) {
            sc.lo = ~0ull;
            sc.hi = 0;
            sc.held = 0;
        }
        __syncthreads();
        auto bin_of = [&](float x, u64 key) {
            if (first) return static_cast<int>(fminf((m - x) * scale, static_cast<float>(kBins - 1)));
            return static_cast<int>((hi - key) >> shift);
        };
        auto inside = [&](u64 key) { return key >= least && (first || (key >= lo && key <= hi)); };
        row.each(low, [&](float x, int i) {
            const u64 key = key_of(x, i);
            if (inside(key)) atomicAdd(&sc.mass[bin_of(x, key)], MASS ? mass(x) : 1ull);
        });
        __syncthreads();
        // the bin in which the last kept one lies: a thread adds up consecutive bins
        constexpr int each = kBins / NT;
        u64 own = 0;
        for (int i = 0; i < each; ++i) own += sc.mass[tid * each + i];
        const u64 to = wave_scan(own);
        if (lane == kWave - 1) sc.wave_mass[wave] = to;
        __syncthreads();
        u64 before = above + to - own;
        for (int i = 0; i < wave; ++i) before += sc.wave_mass[i];
        for (int i = 0; i < each; ++i) {
            const u64 o = sc.mass[tid * each + i];
            if (falls_short(before) && !falls_short(before + o)) {
                sc.bin = tid * each + i;
                sc.before = before;
            }
            before += o;
        }
        __syncthreads();
        const int bin = sc.bin;
        above = sc.before;
        // its entries' keys, and the range of those
        row.each(low, [&](float x, int i) {
            const u64 key = key_of(x, i);
            if (!inside(key) || bin_of(x, key) != bin) return;
            const int at = atomicAdd(&sc.held, 1);
            if (at < kWave) sc.few[at] = key;
            atomicMin(&sc.lo, key);
            atomicMax(&sc.hi, key);
        });
        __syncthreads();
        if (sc.held <= kWave) break;
        lo = sc.lo;
        hi = sc.hi;
        first = false;
        shift = max(0, 64 - __clzll(hi - lo) - 10);   // (hi - lo) >> shift below kBins
        static_assert(kBins == 1 << 10);
        __syncthreads();
    }
    if (wave == 0) {
        const int held = sc.held;
        const u64 key = lane < held ? sc.few[lane] : 0, own = lane < held ? MASS ? mass(value_of(key)) : 1ull : 0;
        u64 before = above;
        int rank = 0;
        for (int j = 0; j < held; ++j) {
            const bool higher = lane_of(key, j) > key;
            before += higher ? lane_of(own, j) : 0;
            rank += higher;
        }
        // kept ones are a prefix: the last is the one that as many others precede as are kept but one
        const u64 keep = __ballot(lane < held && falls_short(before));
        if (lane < held && rank == __popcll(keep) - 1) sc.found = key;
    }
    __syncthreads();
    const u64 found = sc.found;
    __syncthreads();
    return found;
}

// What a row's draw needs, on every thread.
struct Draw {
    double T, inv, p, mp, u;
    int k;
    __device__ __forceinline__ u64 goal(u64 Z) const {   // running sums above it, in whole units
        const double v = u >= 0. ? fmin(u, 1.) : 0.;
        return min(static_cast<u64>(v * static_cast<double>(Z)), Z - 1);
    }
};
__device__ __forceinline__ void put(const Args &a, long long r, const Draw &d, const Mass &mass, int token, float x, u64 Z, int kept) {
    a.token[r] = token;
    a.logprob[r] = static_cast<float>((static_cast<double>(x) - mass.m) * d.inv - log(__builtin_ldexp(static_cast<double>(Z), -a.bits)));
    a.kept[r] = kept;
}

// The draw from the d.k <= 64 largest; false, with nothing written, where too many entries are as large as the bound.
//
// The k-th largest of 128 groups' maxima is no more than the k-th largest entry; the entries that are no less
// (90 at k = 64 of a random row) are ranked, and one wave ends the draw with an entry a lane.
template <int DT, int NT, bool HELD>
__device__ __forceinline__ bool draw_short(const Args &a, long long r, const Row<DT, NT, HELD> &row, const Draw &d, const Mass &mass,
                                           float own_max, Scratch<NT> &sc) {
    constexpr int W = NT / kWave, kShare = kGroups / W, kParts = NT / kShort;
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    sc.top[tid] = own_max;
    __syncthreads();
    float g[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < W; ++i) g[i % 2] = fmaxf(g[i % 2], sc.top[i * kWave + lane]);
    __syncthreads();
    if (tid < kShort) sc.rank[tid] = 0;
    if (tid == 0) sc.held = 0;
    __syncthreads();
    int rank[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < kShare; ++i) {
        const int j = wave * kShare + i;   // a share lies in one half
        const float o = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(j < kWave ? g[0] : g[1]), j % kWave));
#pragma unroll
        for (int h = 0; h < 2; ++h) rank[h] += o > g[h] || (o == g[h] && j < h * kWave + lane);
    }
    atomicAdd(&sc.rank[lane], rank[0]);
    atomicAdd(&sc.rank[kWave + lane], rank[1]);
    __syncthreads();
    if (tid < kGroups && sc.rank[tid] == d.k - 1) sc.low = wave == 0 ? g[0] : g[1];
    __syncthreads();
    if (tid < kShort) sc.rank[tid] = 0;
    row.each(sc.low, [&](float x, int i) {
        const int at = atomicAdd(&sc.held, 1);
        if (at < kShort) sc.key[at] = key_of(x, i);
    });
    __syncthreads();
    const int n = sc.held;
    if (n > kShort) {
        __syncthreads();
        return false;
    }
    const int i = tid % kShort, part = tid / kShort;
    const u64 key = i < n ? sc.key[i] : 0;
    int above = 0;
    for (int j = part; j < n; j += kParts) above += sc.key[j] > key;
    if (kParts > 1) {
        if (i < n) atomicAdd(&sc.rank[i], above);
        __syncthreads();
        above = sc.rank[i];
    }
    if (tid < n && above < d.k) sc.sorted[above] = key;   // in order
    __syncthreads();
    if (wave) return true;
    const u64 own_key = lane < d.k ? sc.sorted[lane] : 0;
    const float x = value_of(own_key);
    const double e = lane < d.k ? mass.real(x) : 0.;
    const u64 w = lane < d.k ? mass.units(e) : 0, to = wave_scan(w);
    const u64 all = lane_of(to, d.k - 1);
    const bool keep = lane == 0 || (lane < d.k && (d.p >= 1. || static_cast<double>(to - w) < d.p * static_cast<double>(all)) && e >= d.mp);
    const int kept = __popcll(__ballot(keep));
    const u64 Z = lane_of(to, kept - 1), goal = d.goal(Z);
    const int token = index_of(own_key);
    u64 run = 0;   // up to and with this one, in the order of the indices
    for (int j = 0; j < kept; ++j) run += __builtin_amdgcn_readlane(token, j) <= token ? lane_of(w, j) : 0;
    if (lane < kept && run - w <= goal && goal < run) put(a, r, d, mass, token, x, Z, kept);
    return true;
}

// The last key of the top-p set of a whole row, and in sc.wave_mass and sc.wave_count what is kept of each wave's run;
// 0 where the estimate did not hold.
//
// Sums of fp32 exponentials in bins of 1/96 nat say in which bin the last kept one lies. One pass in whole units then
// adds up what lies above that bin, per wave, and everything, and holds the bin's own entries, among
// which the border is found. The estimate may be wrong, the bin's entries too many: what the units say is
// looked at, and nothing is kept of it then.
template <int DT, int NT, bool HELD>
__device__ __forceinline__ u64 last_key_by_estimate(const Row<DT, NT, HELD> &row, const Draw &d, const Mass &mass, float m,
                                                    Scratch<NT> &sc) {
    constexpr int W = NT / kWave, V = Row<DT, NT, HELD>::vec, each = kFine / NT, kCols = kList / 2, kParts = NT / kCols;
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    for (int i = tid; i < kFine; i += NT) sc.estimate[i] = 0;
    if (tid == 0) {
        sc.held = 0;
        sc.bin = kFine - 1;
        sc.found = ~0ull;
    }
    __syncthreads();
    const float scale = static_cast<float>(fmin(kFinePerNat * d.inv, 3e38)), c = static_cast<float>(fmin(mass.c, 3e38));
    row.tiles([&](const float (&x)[V], int) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float away = m - x[i];
            const uint32_t e = static_cast<uint32_t>(fminf(__builtin_amdgcn_exp2f(__builtin_fmaf(-away, c, 32.f)), 0x1.fffffep31f));
            const int bin = static_cast<int>(fminf(away * scale, static_cast<float>(kFine - 1)));
            if (e) atomicAdd(&sc.estimate[bin], static_cast<u64>(e));
        }
    });
    __syncthreads();
    u64 own = 0;
#pragma unroll
    for (int i = 0; i < each; ++i) own += sc.estimate[tid * each + i];
    const u64 to = wave_scan(own);
    if (lane == kWave - 1) sc.wave_mass[wave] = to;
    __syncthreads();
    u64 before = to - own, all = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        before += i < wave ? sc.wave_mass[i] : 0;
        all += sc.wave_mass[i];
    }
    const u64 border = static_cast<u64>(d.p * static_cast<double>(all));
    for (int i = 0; i < each; ++i) {
        const u64 after = before + sc.estimate[tid * each + i];
        if (before <= border && border < after) sc.bin = tid * each + i;
        before = after;
    }
    __syncthreads();
    if (sc.bin == kFine - 1) {
        __syncthreads();
        return 0;
    }
    const double bin = sc.bin, width = d.T / kFinePerNat;
    const float slack = (fabsf(m) + static_cast<float>(32. * fmin(d.T, 1e30))) * 0x1p-22f;   // of the bins' own roundings
    const float high = static_cast<float>(mass.m - bin * width) + slack;
    const float low = fmaxf(static_cast<float>(mass.m - (bin + 1.) * width) - slack, -__FLT_MAX__);
    u64 above = 0;
    int count = 0;
    all = 0;
    row.tiles([&](const float (&x)[V], int first) {
        u64 w[V];   // 0 of a masked one
#pragma unroll
        for (int i = 0; i < V; ++i) w[i] = mass(x[i]);
        bool listed = false;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const bool over = x[i] > high;
            all += w[i];
            above += over ? w[i] : 0;
            count += over;
            listed |= !over && x[i] >= low;
        }
        if (listed) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (x[i] <= high && x[i] >= low) {
                    const int at = atomicAdd(&sc.held, 1);
                    if (at < kList) sc.list[at] = Entry{key_of(x[i], first + i), w[i]};
                }
        }
    });
    all = wave_add(all);
    above = wave_add(above);
    count = wave_scan(static_cast<uint32_t>(count), Plus());
    if (lane == kWave - 1) {
        sc.wave_mass[wave] = above;
        sc.few[wave] = all;
        sc.wave_count[wave] = count;
    }
    for (int i = tid; i < kList; i += NT) sc.before_of[i] = 0;
    __syncthreads();
    above = all = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        above += sc.wave_mass[i];
        all += sc.few[i];
    }
    const int held = sc.held;
    const double goal = d.p * static_cast<double>(all);
    if (held > kList || !(static_cast<double>(above) < goal)) {   // uniform
        __syncthreads();
        return 0;
    }
    // what lies before an entry: kParts threads each take a share of the others
    for (int i = tid % kCols; i < held; i += kCols) {
        const u64 key = sc.list[i].key;
        u64 part = 0;
        for (int j = tid / kCols; j < held; j += kParts) {
            const Entry o = sc.list[j];
            part += o.key > key ? o.weight : 0;
        }
        atomicAdd(&sc.before_of[i], part);
    }
    __syncthreads();
    for (int i = tid; i < held; i += NT)
        if (static_cast<double>(above + sc.before_of[i]) < goal) {   // kept
            const Entry e = sc.list[i];
            atomicMin(&sc.found, e.key);
            const int owner = index_of(e.key) / row.run;
            atomicAdd(&sc.wave_mass[owner], e.weight);
            atomicAdd(&sc.wave_count[owner], 1);
        }
    __syncthreads();
    // the border lies among them if what is kept reaches it
    const u64 found = sc.found;
    u64 kept = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) kept += sc.wave_mass[i];
    __syncthreads();
    return found != ~0ull && !(static_cast<double>(kept) < goal) ? found : 0;
}

// One workgroup a row. What is kept comes from one of
//   - the short way: top_k up to 64 (draw_short);
//   - the estimate: top_p alone (last_key_by_estimate);
//   - the exact search (last_key), which serves all, for larger top_k and where the others give up;
//   - nothing to search for: min_p, or no setting.
// Every wave then knows what is kept of its run; the run in which the token lies is read once more by the whole workgroup.
template <int DT, int NT, bool HELD>
__global__ __launch_bounds__(NT, 4) void sample_kernel(Args a) {
    using Mine = Row<DT, NT, HELD>;
    constexpr int V = Mine::vec, W = NT / kWave;
    const long long r = block_id();
    if (r >= a.v.rows) return;
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave, n = a.v.V;
    __shared__ Scratch<NT> sc;
    extern __shared__ u32x4_any held[];
    const Mine row(a, r, tid, held);
    Draw d;
    d.T = a.temperature.at(r);
    d.p = a.top_p.at(r);
    d.mp = a.min_p.at(r);
    d.u = a.u_double ? static_cast<const double *>(a.u)[r] : static_cast<double>(static_cast<const float *>(a.u)[r]);
    const long long k = a.top_ks ? a.top_ks[r] : a.top_k;
    if (tid == 0) {
        sc.first = n;
        sc.odd = 0;
    }

    // the largest entry, how many are not masked, and whether one is no number
    float own_max = -INFINITY;
    int there = 0;
    bool odd = false;
    row.start([&](const float (&x)[V]) {
        float most = x[0];
#pragma unroll
        for (int i = 1; i < V; i += 2) most = max3(most, x[i], x[i + 1 < V ? i + 1 : i]);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            there += __popcll(__ballot(x[i] > -INFINITY));   // the wave's
            odd |= !(x[i] < INFINITY);
        }
        own_max = fmaxf(own_max, most);
        return most;
    });
    float m = wave_max(own_max);
    odd = __any(odd);
    if (lane == 0) {
        sc.wave_top[wave] = m;
        sc.wave_count[wave] = there;
    }
    __syncthreads();
    if (lane == 0 && odd) sc.odd = 1;
    there = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        m = fmaxf(m, sc.wave_top[i]);
        there += sc.wave_count[i];
    }
    __syncthreads();
    if (sc.odd || there == 0 || !(d.T >= 0. && d.T < static_cast<double>(INFINITY)) || d.p != d.p || d.mp != d.mp) {
        if (tid == 0) {
            a.token[r] = -1;
            a.logprob[r] = __builtin_nanf("");
            a.kept[r] = 0;
        }
        return;
    }
    if (d.T == 0. || k == 1 || d.p <= 0. || d.mp > 1.) {   // the first of the largest
        row.each(m, [&](float, int i) { atomicMin(&sc.first, i); });
        __syncthreads();
        if (tid == 0) {
            a.token[r] = sc.first;
            a.logprob[r] = 0.f;
            a.kept[r] = 1;
        }
        return;
    }

    d.T = fmin(d.T, 1e60);   // from there on all are alike
    d.inv = 1. / d.T;
    const Mass mass(m, d.inv, a.bits);
    const float scale = static_cast<float>(fmin(kBinsPerNat * d.inv, 3e38));
    const bool by_k = k > 1 && k < there, by_p = d.p < 1.;
    d.k = by_k ? static_cast<int>(k) : there;
    if (by_k && k <= kWave && draw_short(a, r, row, d, mass, own_max, sc)) return;
    u64 least = 0;
    bool counted = false;
    if (by_k) least = last_key<false>(row, mass, m, scale, 0, d.k, 0., sc);
    if (by_p) {
        u64 found = 0;
        if (!by_k) found = last_key_by_estimate(row, d, mass, m, sc);
        if (found) {
            counted = d.mp <= 0.;
        } else {
            u64 own = 0;
            row.each(least ? value_of(least) : -INFINITY, [&](float x, int i) { own += key_of(x, i) >= least ? mass(x) : 0; });
            const u64 total = group_sum(own, sc);
            found = last_key<true>(row, mass, m, scale, least, 0, d.p * static_cast<double>(total), sc);
        }
        least = found;
    }

    // what is kept of each wave's run: the values above the last kept one's, and of its equals the lower indices; and
    // what min_p lets through (low: a little less than that, by more than fp32's roundings)
    const float last = least ? value_of(least) : -INFINITY;
    const int last_at = least ? index_of(least) : n;
    float low = fmaxf(last, -__FLT_MAX__);
    if (d.mp > 0.) {
        const double x = mass.m + d.T * log(d.mp);
        low = fmaxf(low, static_cast<float>(x - (fabs(x) + fabs(mass.m)) * 1e-6 - 1e-30));
    }
    const bool by_mp = d.mp > 0.;
    auto kept = [&](float x, int i, u64 &w) {
        const double e = mass.real(x);
        const bool keep = x >= low && (x > last || i <= last_at) && (!by_mp || e >= d.mp);
        w = keep ? mass.units(e) : 0;
        return keep;
    };
    if (!counted) {
        u64 own = 0;
        int count = 0;
        if (least || by_mp) {
            row.large_tiles(low, [&](const float (&x)[V], int first) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    u64 w;
                    count += kept(x[i], first + i, w);
                    own += w;
                }
            });
            count = wave_scan(static_cast<uint32_t>(count), Plus());
        } else {   // all of it
            row.tiles([&](const float (&x)[V], int) {
#pragma unroll
                for (int i = 0; i < V; ++i) own += mass(x[i]);
            });
            count = wave == 0 ? there : 0;
        }
        own = wave_add(own);
        if (lane == kWave - 1) {
            sc.wave_mass[wave] = own;
            sc.wave_count[wave] = count;
        }
        __syncthreads();
    }
    u64 Z = 0, before = 0;
    int count = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        Z += sc.wave_mass[i];
        count += sc.wave_count[i];
    }
    const u64 goal = d.goal(Z);
    int owner = 0;
    while (before + sc.wave_mass[owner] <= goal) before += sc.wave_mass[owner++];   // ends: goal < Z
    __syncthreads();

    // the owner's run once more, consecutive vectors a thread
    const int vectors = (row.run / V + NT - 1) / NT, end = min(n, (owner + 1) * row.run);
    auto vector = [&](int j, float (&x)[V]) {   // of this thread, and its first index
        const int i = owner * row.run + (tid * vectors + j) * V;
        if (i < end) {
            row.vector(i, x);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) x[e] = -INFINITY;
        }
        return i;
    };
    u64 own = 0;
    for (int j = 0; j < vectors; ++j) {
        float x[V];
        const int i = vector(j, x);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            u64 w;
            kept(x[e], i + e, w);
            own += w;
        }
    }
    const u64 to = wave_scan(own);
    if (lane == kWave - 1) sc.wave_mass[wave] = to;
    __syncthreads();
    before += to - own;
#pragma unroll
    for (int i = 0; i < W; ++i) before += i < wave ? sc.wave_mass[i] : 0;
    if (before > goal || goal >= before + own) return;   // another thread's
    for (int j = 0; j < vectors; ++j) {
        float x[V];
        const int i = vector(j, x);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            u64 w;
            kept(x[e], i + e, w);
            if (before <= goal && goal < before + w) put(a, r, d, mass, i + e, x[e], Z, count);
            before += w;
        }
    }
}

}  // namespace smp
}  // namespace ulm

using namespace ulm;

extern "C" int ulm_sample_tokens(const void *logits, int dtype, long long rows, long long inner, long long outer_stride,
                                 long long row_stride, int V, const void *u, int u_double, const ulm_sampling *how,
                                 long long *token, float *logprob, long long *kept, void *stream) {
    ULM_REQUIRE(rows >= 1 && rows <= (1LL << 34) && inner >= 1 && V >= 1 && V <= smp::kMaxV,
                "ulm_sample_tokens: bad sizes rows=%lld inner=%lld V=%d", rows, inner, V);
    ULM_REQUIRE(valid_dtype(dtype), "ulm_sample_tokens: bad dtype %d", dtype);
    ULM_REQUIRE(logits && u && how && token && logprob && kept, "ulm_sample_tokens: null pointer");
    int log_v = 0;
    while ((1 << log_v) < V) ++log_v;
    smp::Args a{{static_cast<const char *>(logits), inner, outer_stride, row_stride, rows, V},
                      u,
                      {how->temperature, how->temperatures},
                      {how->top_p, how->top_ps},
                      {how->min_p, how->min_ps},
                      how->top_k,
                      how->top_ks,
                      token,
                      kept,
                      logprob,
                      u_double,
                      log_v <= 15 ? 47 : 62 - log_v,
                      0};
    hipStream_t s = static_cast<hipStream_t>(stream);
    // The row in LDS: four workgroups of 256 threads a CU, two of 512, or one of 1024. Past that rows are read again, with a
    // table beside two workgroups of 512 threads or one of 1024, or without one.
    auto launch = [&](auto dt) {
        constexpr int DT = decltype(dt)::value, kTile = smp::Row<DT, 256, true>::tile;
        const size_t tiles = (V + kTile - 1) / kTile, row = tiles * 1024, table = tiles * kWave * sizeof(float);
        auto run = [&](auto threads, auto held, size_t lds) {
            constexpr int NT = decltype(threads)::value;
            constexpr bool H = decltype(held)::value;
            const void *fn = reinterpret_cast<const void *>(&smp::sample_kernel<DT, NT, H>);
            if (lds > 48 << 10) {
                static std::atomic<unsigned> ready{0};   // a bit a device
                int dev = 0;
                if (hipGetDevice(&dev) != hipSuccess) return check_launch("hipGetDevice");
                if (dev >= 32 || !(ready.load() >> dev & 1)) {
                    if (hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, smp::kMostHeld) != hipSuccess)
                        return check_launch("hipFuncSetAttribute(sample_kernel)");
                    if (dev < 32) ready.fetch_or(1u << dev);
                }
            }
            smp::sample_kernel<DT, NT, H><<<smp::grid_of(rows), dim3(NT), lds, s>>>(a);
            return check_launch("ulm_sample_tokens");
        };
        using std::integral_constant;
        a.tabled = table <= smp::kMostHeld;
        if (row <= 16 << 10) return run(integral_constant<int, 256>{}, std::true_type{}, row);
        if (row <= 63 << 10) return run(integral_constant<int, 512>{}, std::true_type{}, row);
        if (row <= smp::kMostHeld) return run(integral_constant<int, 1024>{}, std::true_type{}, row);
        if (table <= 64 << 10) return run(integral_constant<int, 512>{}, std::false_type{}, table);
        return run(integral_constant<int, 1024>{}, std::false_type{}, a.tabled ? table : 0);
    };
    if (dtype == ULM_F32) return launch(std::integral_constant<int, ULM_F32>{});
    if (dtype == ULM_BF16) return launch(std::integral_constant<int, ULM_BF16>{});
    return launch(std::integral_constant<int, ULM_F16>{});
}
