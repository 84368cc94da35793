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
#pragma once

#include <atomic>
#include <type_traits>

#include "logit_rows.h"

namespace ulm {
namespace smp {

using namespace rows;

constexpr int kMaxV = 1 << 22;
constexpr int kBins = 2048;
constexpr float kBinsPerNat = 96.f;     // 21 nats at first
constexpr int kHeld = 1024;             // entries of one bin that are held by key, the same number for every wave
constexpr int kSplit = 256;             // parts into which these are cut
constexpr int kMostShort = 128;         // top_k of the short way,
constexpr int kShort = 512;             // and the entries that it ranks
constexpr int kGroups = 256;            // groups of threads whose maxima bound the k-th largest entry
constexpr int kTable = 140 << 10, kTableOfTwo = 62 << 10;   // bytes of a row's table in LDS, alone on a CU or with another

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
// Chebyshev's nodes (off by 4e-14 of w). The addition of a large power of two rounds t to n and leaves it in the low bits
// of the sum; that of 2^(52 - bits) rounds w to its units. Its last bit set, w never lies half way
// between two, so that adding several to one such power rounds each alike, whatever came before: a
// sum of an entry's w takes 18 instructions.
//
// -inf is formed as `floor`, which weighs nothing but where the lowest float lies within some units of t of the maximum:
// rows of masked entries of that value only, or of such low ones at temperatures past 1e29. There (low) the -inf entries, and what lies past
// a row's end, are left out by comparison.
struct Mass {
    double m, c, magic;   // c = log2(e) / T, magic = 2^(52 - bits)
    float floor;          // entries below are formed as this one, whose t is within 32 bits
    bool low;             // and may have mass

    __device__ __forceinline__ Mass(float max, double inv, int bits)
        : m(static_cast<double>(max)), magic(__builtin_ldexp(1., 52 - bits)) {
        // where neighbouring floats are past 2^28 apart in t, only the largest have mass, and they keep it with less
        const double step = fmax(fabs(m) * 0x1p-23, 0x1p-149);
        c = fmin(1.4426950408889634074 * inv, 0x1p29 / step);
        const uint32_t b = __float_as_uint(max);
        const float below = max > 0.f ? __uint_as_float(b - 1) : max < 0.f ? __uint_as_float(b + 1) : -0x1p-149f;
        floor = fmaxf(fminf(static_cast<float>(m - 0x1p29 / c), below), -__FLT_MAX__);
        low = (static_cast<double>(floor) - m) * c > -2. - bits;   // half a unit is 2^(-1 - bits)
    }
    __device__ __forceinline__ double real(float x) const {
        constexpr double shift = 6755399441055744.;   // 1.5 2^52
        const double d = static_cast<double>(fmaxf(x, floor)) - m;
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
        g = __builtin_ldexp(g, static_cast<int>(__builtin_bit_cast(u64, k)));
        return __builtin_bit_cast(double, __builtin_bit_cast(u64, g) | 1);
    }
    __device__ __forceinline__ u64 units(double e) const { return __builtin_bit_cast(u64, e + magic) & ((1ull << 52) - 1); }
    __device__ __forceinline__ u64 operator()(float x) const { return units(real(x)); }
};

// The sum of some entries' w, a tile's (at most 8, no more than magic) at a time.
struct Total {
    double part;
    u64 raw;
    int parts;
    __device__ __forceinline__ Total() : part(0.), raw(0), parts(0) {}
    __device__ __forceinline__ void begin(const Mass &mass) { part = mass.magic; }
    __device__ __forceinline__ void end() {
        raw += __builtin_bit_cast(u64, part);
        ++parts;
    }
    __device__ __forceinline__ u64 units(const Mass &mass) const {
        return raw - static_cast<u64>(parts) * __builtin_bit_cast(u64, mass.magic);
    }
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
    template <class T> __device__ __forceinline__ T operator()(T a, T b) const { return a > b ? a : b; }
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

// The workgroup's row. A wave has `count` tiles of it, 64 vectors each, from element `from` on: its run. Every pass reads
// the row again, from the caches, but those that look for large entries where LDS holds every vector's largest (table).
// Held in LDS, one workgroup a CU, a row left the CU idle at its barriers and while it was loaded: 4096 rows of 32000
// fp32 with top_p, 300 us now, took 515 instead of 364 then. Held in registers it left the passes too few.
template <int DT, int NT> struct Row {
    static constexpr int vec = Elem<DT>::vec, tile = kWave * vec, W = NT / kWave, kBatch = 4;
    const char *row;
    float *table;   // the wave's: of every two tiles, a lane's largest
    int n, run, from, count, whole, lane;   // run: a wave's elements; whole: tiles that end inside the row

    __device__ __forceinline__ Row(const Args &a, long long r, int tid, float *lds)
        : row(a.v.row(r, Elem<DT>::bytes)), n(a.v.V), lane(tid % kWave) {
        const int tiles = (n + tile - 1) / tile, per_wave = (tiles + W - 1) / W, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
        run = per_wave * tile;
        from = wave * run;
        count = max(0, min(per_wave, tiles - wave * per_wave));
        whole = max(0, min(count, (n - from) / tile));
        table = a.tabled ? lds + wave * table_of(n) / W + lane : nullptr;
    }
    // entries of all waves' tables
    static __host__ __device__ __forceinline__ int table_of(int n) {
        const int tiles = (n + tile - 1) / tile, per_wave = (tiles + W - 1) / W;
        return W * ((per_wave + 1) / 2) * kWave;
    }
    __device__ __forceinline__ void note(int at, float most) const {   // of the tile at whose vector `at` the lane is
        const int t = (at - from) / tile;
        float &e = table[t / 2 * kWave];
        e = t % 2 ? fmaxf(e, most) : most;
    }
    __device__ __forceinline__ int at(int t) const { return from + t * tile + lane * vec; }
    __device__ __forceinline__ void vector(int i, float (&x)[vec]) const { load_vec<DT, false>(row, i, n, x); }
    // f(elements, index of the first) with a batch of loads under way; what lies past the row's end is -inf
    template <class F> __device__ __forceinline__ void tiles(F f) const {
        int t0 = 0;
        for (; t0 + kBatch <= whole; t0 += kBatch) {
            u32x4_any w[kBatch];
            const char *p = row + static_cast<size_t>(at(t0)) * Elem<DT>::bytes;
#pragma unroll
            for (int t = 0; t < kBatch; ++t) w[t] = *reinterpret_cast<const u32x4_any *>(p + t * 1024);
#pragma unroll
            for (int t = 0; t < kBatch; ++t) {
                float x[vec];
                unpack<DT>(w[t], x);
                f(x, at(t0 + t));
            }
        }
        for (; t0 < count; ++t0) {
            float x[vec];
            vector(at(t0), x);
            f(x, at(t0));
        }
    }
    // the same without tiles in which none is `low` (above -inf) or more
    template <class F> __device__ __forceinline__ void large_tiles(float low, F f) const {
        int pairs = count;   // with such an entry
        if (table) {
            pairs = 0;
            for (int t = 0; t < count; t += 2) pairs += __any(table[t / 2 * kWave] >= low);
        }
        if (pairs * 8 <= count) {   // few: not worth batches of all
            for (int t = 0; t < count; t += 2) {
                if (!__any(table[t / 2 * kWave] >= low)) continue;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (t + h >= count) continue;
                    float x[vec];
                    vector(at(t + h), x);
                    f(x, at(t + h));
                }
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
};

// A wave's own list in LDS: lanes push by their place among the lanes that do, without an atomic's round trip (that of
// one a vector made a pass over a row of 32000 4 us longer).
template <class T> struct WaveList {
    T *at;
    int room, count;   // count: of pushes, which may be more than there is room for
    __device__ __forceinline__ void push(bool does, T v) {
        const u64 who = __ballot(does);
        if (who == 0) return;
        const int place = count + __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(who >> 32),
                                                            __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(who), 0));
        if (does && place < room) at[place] = v;
        count += __popcll(who);
    }
    static __device__ __forceinline__ void settle() {   // before other lanes' entries are read
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
};

template <int NT> struct Scratch {
    static constexpr int W = NT / kWave;
    union {
        u64 mass[kBins];
        float top[NT];
        struct {
            u64 list[kHeld];
            u64 split[kSplit], few[kWave], few_mass[kWave];
            int vectors[kHeld];
        };
        struct {
            u64 own[W][kHeld / W];
            union {
                u64 key[kShort];
                int hits[W][kWave];
            };
            u64 sorted[kMostShort];
            int rank[kShort];
        };
    };
    u64 wave_mass[W], wave_all[W];
    int wave_count[W];
    float wave_top[W];
    u64 lo, hi, before, found;
    float low;
    int held, bin, from, to, first, odd, crowded;
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

// The bin of sc.mass in which the last kept one lies, and in `above`, what lies above the bins, what lies above it;
// of all bins' sum comes the goal, where there is none yet (less than 0). ABOUT: sc.from .. sc.to are the bins in which
// it may lie, each of `entries` entries being off by a unit, and all sums by 2^-16 of the whole.
template <bool ABOUT, int NT>
__device__ __forceinline__ int border_bin(u64 &above, double &goal, double share, Scratch<NT> &sc, int entries = 0) {
    constexpr int W = NT / kWave, n = kBins / NT;
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    u64 own[n], sum = 0;
#pragma unroll
    for (int i = 0; i < n; ++i) sum += own[i] = sc.mass[tid * n + i];
    const u64 to = wave_scan(sum);
    if (lane == kWave - 1) sc.wave_mass[wave] = to;
    if (tid == 0) {
        sc.bin = sc.to = kBins - 1;
        sc.from = 0;
    }
    __syncthreads();
    u64 before = above + to - sum, all = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        before += i < wave ? sc.wave_mass[i] : 0;
        all += sc.wave_mass[i];
    }
    if (goal < 0.) goal = share * static_cast<double>(all);
    const double off = static_cast<double>(all) * 0x1p-16 + entries;
#pragma unroll
    for (int i = 0; i < n; ++i) {
        auto lies_in = [&](double goal) {   // one bin
            return static_cast<double>(before) < goal && !(static_cast<double>(before + own[i]) < goal);
        };
        if (lies_in(goal)) {
            sc.bin = tid * n + i;
            sc.before = before;
        }
        if (ABOUT && lies_in(goal - off)) sc.from = tid * n + i;
        if (ABOUT && lies_in(goal + off)) sc.to = tid * n + i;
        before += own[i];
    }
    __syncthreads();
    above = sc.before;
    return sc.bin;
}

// The last kept key among those that the waves hold, each in its list: the first of the order before which lies no less
// than `goal` is not kept. `above`: what lies before all of them, in mass or, MASS false, in numbers. They are cut
// into parts by their keys, which are unique, until a wave can rank one part's. 0 where all are kept.
template <bool MASS, int NT>
__device__ __forceinline__ u64 last_held(const WaveList<u64> &list, const Mass &mass, u64 above, double goal, Scratch<NT> &sc) {
    constexpr int W = NT / kWave, kRoom = kHeld / W, kOwn = kRoom / kWave;
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    auto falls_short = [&](u64 before) { return static_cast<double>(before) < goal; };
    u64 key[kOwn], weight[kOwn];
    int part[kOwn];   // -1: none, or not among the border's
#pragma unroll
    for (int h = 0; h < kOwn; ++h) {
        const int i = h * kWave + lane;
        part[h] = i < list.count ? 0 : -1;
        key[h] = i < list.count ? list.at[i] : 0;
        weight[h] = i < list.count ? MASS ? mass(value_of(key[h])) : 1 : 0;
    }
    for (;;) {
        __syncthreads();   // every wave has read its list and, later, the border's part
        if (tid < kSplit) sc.split[tid] = 0;
        if (tid == 0) {
            sc.held = 0;
            sc.hi = sc.lo = 0;
            sc.bin = -1;
        }
        __syncthreads();
        u64 top = 0, bottom = 0;   // the largest key, and the largest of their complements
#pragma unroll
        for (int h = 0; h < kOwn; ++h)
            if (part[h] >= 0) {
                top = key[h] > top ? key[h] : top;
                bottom = ~key[h] > bottom ? ~key[h] : bottom;
            }
        top = lane_of(wave_scan(top, Larger()), kWave - 1);
        bottom = lane_of(wave_scan(bottom, Larger()), kWave - 1);
        if (lane == 0 && top) {
            atomicMax(&sc.hi, top);
            atomicMax(&sc.lo, bottom);
        }
        __syncthreads();
        const u64 hi = sc.hi;
        const int shift = max(0, 64 - __clzll(hi - ~sc.lo) - 8);   // (hi - lo) >> shift below kSplit
        static_assert(kSplit == 1 << 8);
#pragma unroll
        for (int h = 0; h < kOwn; ++h)
            if (part[h] >= 0) {
                part[h] = static_cast<int>((hi - key[h]) >> shift);
                atomicAdd(&sc.split[part[h]], weight[h]);
            }
        __syncthreads();
        if (wave == 0) {
            constexpr int n = kSplit / kWave;
            u64 o[n], sum = 0;
#pragma unroll
            for (int i = 0; i < n; ++i) sum += o[i] = sc.split[lane * n + i];
            u64 before = above + wave_scan(sum) - sum;
#pragma unroll
            for (int i = 0; i < n; ++i) {
                if (falls_short(before) && !falls_short(before + o[i])) {   // one
                    sc.bin = lane * n + i;
                    sc.before = before;
                }
                before += o[i];
            }
        }
        __syncthreads();
        const int border = sc.bin;
        if (border < 0) return 0;   // uniform
        above = sc.before;
#pragma unroll
        for (int h = 0; h < kOwn; ++h) {
            if (part[h] != border) part[h] = -1;
            if (part[h] >= 0) {
                const int at = atomicAdd(&sc.held, 1);
                if (at < kWave) {
                    sc.few[at] = key[h];
                    sc.few_mass[at] = weight[h];
                }
            }
        }
        __syncthreads();
        if (sc.held <= kWave) break;
    }
    if (wave == 0) {
        const int few = sc.held;
        const u64 own = lane < few ? sc.few[lane] : 0, w = lane < few ? sc.few_mass[lane] : 0;
        u64 before = above;
        int rank = 0;
        for (int j = 0; j < few; ++j) {
            const bool higher = lane_of(own, j) > own;
            before += higher ? lane_of(w, j) : 0;
            rank += higher;
        }
        // kept ones are a prefix: the last is the one that as many others precede as are kept but one
        const u64 keep = __ballot(lane < few && falls_short(before));
        if (lane < few && rank == __popcll(keep) - 1) sc.found = own;
    }
    __syncthreads();
    return sc.found;
}

// The last kept key where the first d.k ranks are kept (MASS false), or the fewest that hold d.p of the mass (MASS
// true). Only keys of `least` and above exist.
//
// The entries' masses, or numbers, are added up in bins of an order-keeping function: at first of the distance from
// the largest, 1/96 nat a bin, then of the bits of their keys, until the waves can hold the entries of the bin
// in which the last kept one lies. (LDS adds whole numbers of 64 bits in 3 us for a row of 32000, floats in 41; with a
// quarter of the bins, so that lanes meet in them, in 15.)
template <bool MASS, int DT, int NT>
__device__ __forceinline__ u64 last_key(const Row<DT, NT> &row, const Draw &d, const Mass &mass, float m, u64 least,
                                        Scratch<NT> &sc) {
    constexpr int W = NT / kWave, V = Row<DT, NT>::vec, kRoom = kHeld / W;
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    const float last = least ? value_of(least) : -INFINITY, low = fmaxf(last, -__FLT_MAX__);
    const int last_at = least ? index_of(least) : row.n;
    double goal = MASS ? -1. : static_cast<double>(d.k);
    const float scale = static_cast<float>(fmin(kBinsPerNat * d.inv, 3e38));
    constexpr float kLast = static_cast<float>(kBins - 1);
    u64 lo = 0, hi = 0, above = 0;   // the window of keys, and what lies above it
    int shift = 0;
    bool first = true;
    // the bin of an entry in the window, -1 of others
    auto bin_of = [&](float x, int i) {
        if (!(x >= low) || (x == last && i > last_at)) return -1;
        if (first) return static_cast<int>(fminf((m - x) * scale, kLast));
        const u64 key = key_of(x, i);
        return key >= lo && key <= hi ? static_cast<int>((hi - key) >> shift) : -1;
    };
    WaveList<u64> list;
    for (;; first = false) {
        for (int i = tid; i < kBins; i += NT) sc.mass[i] = 0;
        __syncthreads();
        u64 tail = 0;   // of the last bin, which may hold most of a row
        row.large_tiles(low, [&](const float (&x)[V], int at) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int b = bin_of(x[i], at + i);
                const u64 w = MASS ? mass(x[i]) : 1;
                if (b >= 0 && b < kBins - 1) atomicAdd(&sc.mass[b], w);
                tail += b == kBins - 1 ? w : 0;
            }
        });
        tail = wave_add(tail);
        if (lane == 0 && tail) atomicAdd(&sc.mass[kBins - 1], tail);
        __syncthreads();
        const int bin = border_bin<false>(above, goal, d.p, sc);
        if (tid == 0) {
            sc.crowded = 0;
            sc.hi = sc.lo = 0;
        }
        __syncthreads();   // the bins' room is for the list now
        list = {sc.list + wave * kRoom, kRoom, 0};
        u64 top = 0, bottom = 0;   // its entries' range
        row.large_tiles(low, [&](const float (&x)[V], int at) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const bool in = bin_of(x[i], at + i) == bin;
                const u64 key = key_of(x[i], at + i);
                list.push(in, key);
                top = in && key > top ? key : top;
                bottom = in && ~key > bottom ? ~key : bottom;
            }
        });
        if (list.count > list.room && lane == 0) sc.crowded = 1;
        __syncthreads();
        if (!sc.crowded) break;
        top = lane_of(wave_scan(top, Larger()), kWave - 1);
        bottom = lane_of(wave_scan(bottom, Larger()), kWave - 1);
        if (lane == 0 && top) {
            atomicMax(&sc.hi, top);
            atomicMax(&sc.lo, bottom);
        }
        __syncthreads();
        hi = sc.hi;
        lo = ~sc.lo;
        shift = max(0, 64 - __clzll(hi - lo) - 11);   // (hi - lo) >> shift below kBins
        static_assert(kBins == 1 << 11);
        __syncthreads();
    }
    const u64 found = last_held<MASS>(list, mass, above, goal, sc);
    __syncthreads();
    return found;
}

// The last key of the top-p set of a row, or of its entries down to key `least` where that is not 0, and in sc.wave_mass and sc.wave_count what is kept of each wave's run;
// 0 where the estimate did not hold.
//
// Sums of fp32 exponentials in bins of 1/96 nat say in which bin, or few bins, the last kept one lies. One pass in whole
// units then adds up what lies above them, per wave, and everything, and holds their entries, among
// which the border is found. The estimate may be wrong, the entries too many: what the units say is
// looked at, and nothing is kept of it then. idle: min_p leaves less than top_p would, by more than the estimate may be
// off. (4096 rows of 32000 bf16 with top_k 1000 and top_p: 532 us, and 703 with an exact search behind top_k.)
template <int DT, int NT>
__device__ __forceinline__ u64 last_key_by_estimate(const Row<DT, NT> &row, const Draw &d, const Mass &mass, float m,
                                                    u64 least, Scratch<NT> &sc, bool &idle) {
    constexpr int W = NT / kWave, V = Row<DT, NT>::vec, kRoom = kHeld / W;
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    const float last = least ? value_of(least) : -INFINITY;
    const int last_at = index_of(least);
    // the entries that count of a vector, -inf for the others; false where the wave has none
    auto counting = [&](const float (&all)[V], int at, float (&x)[V]) {
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = all[i];
        if (!least) return true;   // uniform
        bool any = false;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const bool in = x[i] > last || (x[i] == last && at + i <= last_at);
            x[i] = in ? x[i] : -INFINITY;
            any |= in;
        }
        return __any(any) != 0;
    };
    for (int i = tid; i < kBins; i += NT) sc.mass[i] = 0;
    __syncthreads();
    const float scale = static_cast<float>(fmin(kBinsPerNat * d.inv, 3e38)), c = static_cast<float>(fmin(mass.c, 3e38));
    row.tiles([&](const float (&all)[V], int at) {
        float x[V];
        if (!counting(all, at, x)) return;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float away = m - x[i];
            const uint32_t e = static_cast<uint32_t>(__builtin_amdgcn_exp2f(__builtin_fmaf(-away, c, 31.f)));
            const int bin = static_cast<int>(fminf(away * scale, static_cast<float>(kBins - 1)));
            if (e) atomicAdd(&sc.mass[bin], static_cast<u64>(e));
        }
    });
    __syncthreads();
    u64 above = 0;
    double goal = -1.;
    const int bin = border_bin<true>(above, goal, d.p, sc, row.n);
    if (d.mp > 0.) {   // uniform
        // what min_p keeps lies above this bin; each of the sums is off by a unit an entry and, an exponent being rounded to
        // 2^-19 and the distances to 2^-24 of themselves, 2^-17 of itself at most
        const int after = static_cast<int>(fmin(-log(d.mp) * kBinsPerNat, kBins - 1.)) + 2;
        u64 own = 0;
        for (int i = tid; i < min(after, kBins); i += NT) own += sc.mass[i];
        const u64 most = group_sum(own, sc);
        idle = after <= bin && static_cast<double>(most) * (1. + 0x1p-15) + 2. * row.n < goal * (1. - 0x1p-15);
    }
    if (idle || bin == kBins - 1) {   // uniform
        __syncthreads();
        return 0;
    }
    const double width = d.T / kBinsPerNat, from = max(sc.from, bin - 64), to = min(sc.to, bin + 64) + 1;
    const float slack = (fabsf(m) + static_cast<float>(32. * fmin(d.T, 1e30))) * 0x1p-22f;   // of the bins' own roundings
    const float high = static_cast<float>(mass.m - from * width) + slack;
    const float low = fmaxf(static_cast<float>(mass.m - to * width) - slack, -__FLT_MAX__);
    Total everything, over;
    int count = 0;   // the wave's
    WaveList<int> vectors{sc.vectors + wave * kRoom, kRoom, 0};   // with an entry of the bin
    __syncthreads();   // the bins' room is for the lists now
    row.tiles([&](const float (&all)[V], int at) {
        float x[V];
        if (!counting(all, at, x)) return;
        everything.begin(mass);
        over.begin(mass);
        bool listed = false;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const double e = mass.real(x[i]);
            const bool higher = x[i] > high;
            everything.part += e;
            over.part = __builtin_fma(e, higher ? 1. : 0., over.part);
            count += __popcll(__ballot(higher));
            listed |= !higher && x[i] >= low;
        }
        everything.end();
        over.end();
        vectors.push(listed, at);
    });
    vectors.settle();
    WaveList<u64> list{sc.list + wave * kRoom, kRoom, 0};
    for (int h = lane; h - lane < min(vectors.count, kRoom); h += kWave) {
        float held[V], x[V];
#pragma unroll
        for (int i = 0; i < V; ++i) held[i] = -INFINITY;
        const int at = h < min(vectors.count, kRoom) ? vectors.at[h] : 0;
        if (h < min(vectors.count, kRoom)) row.vector(at, held);
        if (!counting(held, at, x)) continue;
#pragma unroll
        for (int i = 0; i < V; ++i) list.push(x[i] <= high && x[i] >= low, key_of(x[i], at + i));
    }
    above = wave_add(over.units(mass));
    u64 all = wave_add(everything.units(mass));
    if (tid == 0) sc.crowded = 0;
    __syncthreads();
    if (lane == 0) {
        sc.wave_mass[wave] = above;
        sc.wave_all[wave] = all;
        sc.wave_count[wave] = count;
        if (list.count > kRoom || vectors.count > kRoom) sc.crowded = 1;
    }
    __syncthreads();
    above = all = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        above += sc.wave_mass[i];
        all += sc.wave_all[i];
    }
    goal = d.p * static_cast<double>(all);
    if (sc.crowded || !(static_cast<double>(above) < goal)) {   // uniform
        __syncthreads();
        return 0;
    }
    const u64 found = last_held<true>(list, mass, above, goal, sc);
    if (found) {   // uniform
        u64 kept = 0;
        int more = 0;
        for (int i = lane; i - lane < list.count; i += kWave) {
            const u64 key = i < list.count ? list.at[i] : 0;
            kept += key >= found ? mass(value_of(key)) : 0;
            more += __popcll(__ballot(key >= found));
        }
        kept = wave_add(kept);
        if (lane == 0) {
            sc.wave_mass[wave] += kept;
            sc.wave_count[wave] += more;
        }
    }
    __syncthreads();
    return found;
}

// The draw from the d.k <= 128 largest; false, with nothing written, where too many entries are as large as the bound.
//
// The k-th largest of 256 groups' maxima is no more than the k-th largest entry; the entries that are no less
// (180 at k = 128 of a random row, 74 at 64) are ranked, and one wave ends the draw with two entries a lane.
template <int DT, int NT>
__device__ __forceinline__ bool draw_short(const Args &a, long long r, const Row<DT, NT> &row, const Draw &d, const Mass &mass,
                                           float own_max, Scratch<NT> &sc) {
    constexpr int W = NT / kWave, V = Row<DT, NT>::vec, kG = kGroups / kWave, kShare = kGroups / W, kRoom = kHeld / W;
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    sc.top[tid] = own_max;
    __syncthreads();
    float g[kG];   // group i * 64 + lane: the lane's in waves i, i + 4 ..
#pragma unroll
    for (int i = 0; i < kG; ++i) g[i] = sc.top[i * kWave + lane];
#pragma unroll
    for (int i = kG; i < W; ++i) g[i % kG] = fmaxf(g[i % kG], sc.top[i * kWave + lane]);
    __syncthreads();
    for (int i = tid; i < kShort; i += NT) sc.rank[i] = 0;
    if (tid == 0) sc.held = sc.crowded = 0;
    __syncthreads();
    int rank[kG] = {};
    const int first = wave * kShare / kWave;   // the row of groups in which this wave's share lies
    static_assert(kG == 4 && kWave % kShare == 0);
    u64 group[kG];
#pragma unroll
    for (int h = 0; h < kG; ++h) group[h] = key_of(g[h], h * kWave + lane);
    const u64 share = first == 0 ? group[0] : first == 1 ? group[1] : first == 2 ? group[2] : group[3];
#pragma clang loop unroll(disable)
    for (int i = 0; i < kShare; ++i) {
        const u64 o = lane_of(share, (wave * kShare + i) % kWave);
#pragma unroll
        for (int h = 0; h < kG; ++h) rank[h] += o > group[h];
    }
#pragma unroll
    for (int h = 0; h < kG; ++h) atomicAdd(&sc.rank[h * kWave + lane], rank[h]);
    __syncthreads();
    if (wave == 0) {
#pragma unroll
        for (int h = 0; h < kG; ++h)
            if (sc.rank[h * kWave + lane] == d.k - 1) sc.low = g[h];
    }
    __syncthreads();
    for (int i = tid; i < kShort; i += NT) sc.rank[i] = 0;
    const float low = fmaxf(sc.low, -__FLT_MAX__);
    WaveList<u64> own{sc.own[wave], kRoom, 0};
    // the vectors with such an entry first, so that they come all at once
    WaveList<int> hits{sc.hits[wave], kWave, 0};
    if (row.table) {
        for (int t = 0; t < row.count; t += 2) hits.push(row.table[t / 2 * kWave] >= low, row.at(t));
    } else {
        row.tiles([&](const float (&x)[V], int at) {
            float most = x[0];
#pragma unroll
            for (int i = 1; i < V; ++i) most = fmaxf(most, x[i]);
            hits.push(most >= low, at);
        });
    }
    hits.settle();
    const int at = lane < min(hits.count, kWave) ? sc.hits[wave][lane] : -1;
    const int next = at + Row<DT, NT>::tile;   // an entry of the table is of two tiles
    float x[2][V];
#pragma unroll
    for (int i = 0; i < V; ++i) x[0][i] = x[1][i] = -INFINITY;
    if (at >= 0) row.vector(at, x[0]);
    if (at >= 0 && row.table && next < row.from + row.count * Row<DT, NT>::tile) row.vector(next, x[1]);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < V; ++i) own.push(x[h][i] >= low, key_of(x[h][i], (h ? next : at) + i));
    own.count += hits.count > kWave ? kRoom + 1 : 0;
    own.settle();
    int base = 0;
    if (lane == 0) {
        base = atomicAdd(&sc.held, own.count);
        if (own.count > kRoom) sc.crowded = 1;
    }
    base = __builtin_amdgcn_readfirstlane(base);
    __syncthreads();   // the vectors' places are the keys' now
    for (int i = lane; i < min(own.count, kRoom); i += kWave)
        if (base + i < kShort) sc.key[base + i] = sc.own[wave][i];
    __syncthreads();
    const int n = sc.held;
    if (n > kShort || sc.crowded) {   // uniform
        __syncthreads();
        return false;
    }
    constexpr int kCols = NT < kShort ? NT : kShort, kParts = NT / kCols;
    for (int i = tid % kCols; i < n; i += kCols) {
        const u64 key = sc.key[i];
        int above = 0;
        for (int j = tid / kCols; j < n; j += kParts) above += sc.key[j] > key;
        if (kParts > 1) atomicAdd(&sc.rank[i], above);
        else sc.rank[i] = above;
    }
    __syncthreads();
    for (int i = tid; i < n; i += NT)
        if (sc.rank[i] < d.k) sc.sorted[sc.rank[i]] = sc.key[i];
    __syncthreads();
    if (wave) return true;
    u64 w[2], to[2];   // ranks 2 lane and 2 lane + 1
    float own_x[2];
    double e[2];
    int token[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const u64 key = 2 * lane + h < d.k ? sc.sorted[2 * lane + h] : 0;
        own_x[h] = value_of(key);
        token[h] = index_of(key);
        e[h] = mass.real(own_x[h]);
        w[h] = key ? mass.units(e[h]) : 0;
    }
    to[1] = wave_scan(w[0] + w[1]);
    to[0] = to[1] - w[1];
    const double goal_p = d.p * static_cast<double>(lane_of(to[1], kWave - 1));   // what lies past the k-th weighs 0
    int kept = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int rank = 2 * lane + h;
        const bool keep = rank == 0 || (rank < d.k && (d.p >= 1. || static_cast<double>(to[h] - w[h]) < goal_p) && e[h] >= d.mp);
        kept += __popcll(__ballot(keep));
    }
    const u64 Z = lane_of(kept % 2 ? to[0] : to[1], (kept - 1) / 2), goal = d.goal(Z);
    u64 before[2] = {0, 0};   // up to and with this one, in the order of the indices
    for (int j = 0; j < kept; ++j) {
        const int other = __builtin_amdgcn_readlane(j % 2 ? token[1] : token[0], j / 2);
        const u64 weight = lane_of(j % 2 ? w[1] : w[0], j / 2);
#pragma unroll
        for (int h = 0; h < 2; ++h) before[h] += other <= token[h] ? weight : 0;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
        if (2 * lane + h < kept && before[h] - w[h] <= goal && goal < before[h])
            put(a, r, d, mass, token[h], own_x[h], Z, kept);
    return true;
}

// One workgroup a row. What is kept comes from one of
//   - the short way: top_k up to 128 (draw_short);
//   - the estimate: top_p, alone or behind a larger top_k (last_key_by_estimate);
//   - the exact search, which serves all: larger top_k, and where the others give up (last_key);
//   - nothing to search for: min_p, or no setting.
// The kept mass of every wave's run is then known; the run in which the token lies is looked through once more.
template <int DT, int NT>
__global__ __launch_bounds__(NT, 4) void sample_kernel(Args a) {
    using Mine = Row<DT, NT>;
    constexpr int V = Mine::vec, W = NT / kWave;
    const long long r = block_id();
    if (r >= a.v.rows) return;
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave, n = a.v.V;
    __shared__ Scratch<NT> sc;
    extern __shared__ float table[];
    const Mine row(a, r, tid, table);
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
    u64 no_numbers = 0;
    row.tiles([&](const float (&x)[V], int at) {
        float most = x[0];
#pragma unroll
        for (int i = 1; i < V; i += 2) most = max3(most, x[i], x[i + 1 < V ? i + 1 : i]);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            there += __popcll(__ballot(x[i] > -INFINITY));   // the wave's
            no_numbers |= __ballot(!(x[i] < INFINITY));
        }
        if (row.table) row.note(at, most);
        own_max = fmaxf(own_max, most);
    });
    const bool odd = no_numbers != 0;
    float m = wave_max(own_max);
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
        row.large_tiles(m, [&](const float (&x)[V], int at) {
#pragma unroll
            for (int i = V - 1; i >= 0; --i)
                if (x[i] == m) atomicMin(&sc.first, at + i);
        });
        __syncthreads();
        if (tid == 0) {
            a.token[r] = sc.first;
            a.logprob[r] = 0.f;
            a.kept[r] = 1;
        }
        return;
    }

    d.T = fmin(fmax(d.T, 1e-300), 1e60);   // past these nothing changes any more, and 1 / T is a number
    d.inv = 1. / d.T;
    const Mass mass(m, d.inv, a.bits);
    const bool by_k = k > 1 && k < there, by_p = d.p < 1.;
    d.k = by_k ? static_cast<int>(k) : there;
    if (by_k && k <= kMostShort && draw_short(a, r, row, d, mass, own_max, sc)) return;
    u64 least = 0;
    bool counted = false;
    if (by_k) least = last_key<false>(row, d, mass, m, 0, sc);
    if (by_p) {
        bool idle = false;
        const u64 found = mass.low ? 0 : last_key_by_estimate(row, d, mass, m, least, sc, idle);
        // min_p takes nothing more away, nor from larger entries, whose mass as formed may be 4e-14 less
        counted = found && (d.mp <= 0. || mass.real(value_of(found)) >= d.mp * (1. + 0x1p-40));
        if (found) least = found;
        else if (!idle) least = last_key<true>(row, d, mass, m, least, sc);
    }

    // what is kept of each run: the values above the last kept one's, and of its equals the lower indices; and
    // what min_p lets through (low: a little less than that, by more than fp32's roundings)
    const float last = least ? value_of(least) : -INFINITY;
    const int last_at = least ? index_of(least) : n;
    float low = fmaxf(last, -__FLT_MAX__);
    if (d.mp > 0.) {
        const double x = mass.m + d.T * log(d.mp);
        low = fmaxf(low, static_cast<float>(x - (fabs(x) + fabs(mass.m)) * 1e-6 - 1e-30));
    }
    const bool by_mp = d.mp > 0.;
    auto kept = [&](float x, int i, double e) {
        return x >= low && (x > last || i <= last_at) && (!by_mp || e >= d.mp);
    };
    if (!counted) {
        Total own;
        int count = 0;   // the wave's
        auto add = [&](const float (&x)[V], auto keep) {
            own.begin(mass);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const double e = mass.real(x[i]);
                const bool k = keep(x[i], i, e);
                own.part = __builtin_fma(e, k ? 1. : 0., own.part);
                count += __popcll(__ballot(k));
            }
            own.end();
        };
        if (least) {
            row.large_tiles(low, [&](const float (&x)[V], int at) {
                add(x, [&](float x, int i, double e) { return kept(x, at + i, e); });
            });
        } else if (by_mp || mass.low) {
            row.large_tiles(low, [&](const float (&x)[V], int) {
                add(x, [&](float x, int, double e) { return x >= low && e >= d.mp; });
            });
        } else {   // all of it
            row.tiles([&](const float (&x)[V], int) {
                own.begin(mass);
#pragma unroll
                for (int i = 0; i < V; ++i) own.part += mass.real(x[i]);
                own.end();
            });
            count = wave == 0 ? there : 0;
        }
        const u64 all = wave_add(own.units(mass));
        if (lane == 0) {
            sc.wave_mass[wave] = all;
            sc.wave_count[wave] = count;
        }
        __syncthreads();
    }
    u64 Z = 0, before = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) Z += sc.wave_mass[i];
    const u64 goal = d.goal(Z);
    int owner = 0, count = 0;
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
            const double w = mass.real(x[e]);
            own += kept(x[e], i + e, w) ? mass.units(w) : 0;
        }
    }
    const u64 to = wave_scan(own);
    if (lane == kWave - 1) sc.wave_mass[wave] = to;
    __syncthreads();
    before += to - own;
#pragma unroll
    for (int i = 0; i < W; ++i) before += i < wave ? sc.wave_mass[i] : 0;
    if (before > goal || goal >= before + own) return;   // another thread's
    for (int i = 0; i < W; ++i) count += sc.wave_count[i];
    for (int j = 0; j < vectors; ++j) {
        float x[V];
        const int i = vector(j, x);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const double share = mass.real(x[e]);
            const u64 w = kept(x[e], i + e, share) ? mass.units(share) : 0;
            if (before <= goal && goal < before + w) put(a, r, d, mass, i + e, x[e], Z, count);
            before += w;
        }
    }
}

// Threads a row: as many as it has use for; where there are more rows than CUs, no more than two workgroups a CU allow.
// 4096 rows of 32000 fp32 with top_p: 360 us with 256, 348 with 512, 452 with 1024. One row of 8192 fp32 with top_p 13.8
// with 512 and 16.8 with 1024, without 7.4 and 9.0; of 32000 24.4 and 24.8, 13.5 and 12.7; 64 rows of 128256 bf16 74 and
// 67, 46 and 37. (Launches one after another.) The table where it fits.
template <int DT> int launch(Args a, hipStream_t s) {
    constexpr int kTile = Row<DT, 256>::tile;
    const int V = a.v.V;
    const long long rows = a.v.rows;
    const bool many = rows > 256;
    auto run = [&](auto threads) {
        constexpr int NT = decltype(threads)::value;
        const size_t table = Row<DT, NT>::table_of(V) * sizeof(float);
        a.tabled = table <= (many ? kTableOfTwo : kTable);
        const size_t lds = a.tabled ? table : 0;
        if (lds > 40 << 10) {
            static std::atomic<unsigned> ready{0};   // a bit a device
            int dev = 0;
            if (hipGetDevice(&dev) != hipSuccess) return check_launch("hipGetDevice");
            if (dev >= 32 || !(ready.load() >> dev & 1)) {
                if (hipFuncSetAttribute(reinterpret_cast<const void *>(&sample_kernel<DT, NT>),
                                        hipFuncAttributeMaxDynamicSharedMemorySize, kTable) != hipSuccess)
                    return check_launch("hipFuncSetAttribute(sample_kernel)");
                if (dev < 32) ready.fetch_or(1u << dev);
            }
        }
        sample_kernel<DT, NT><<<grid_of(rows), dim3(NT), lds, s>>>(a);
        return check_launch("ulm_sample_tokens");
    };
    if (V <= 16 * kTile) return run(std::integral_constant<int, 256>{});
    if (many || V <= 64 * kTile) return run(std::integral_constant<int, 512>{});
    return run(std::integral_constant<int, 1024>{});
}
extern template int launch<ULM_F32>(Args, hipStream_t);
extern template int launch<ULM_BF16>(Args, hipStream_t);
extern template int launch<ULM_F16>(Args, hipStream_t);

}  // namespace smp
}  // namespace ulm
