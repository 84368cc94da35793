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
#include <type_traits>

#include "logit_rows.h"

namespace ulm {
namespace smp {

using namespace rows;

constexpr int kMaxV = 1 << 22;
constexpr int kBins = 2048;
constexpr float kBinsPerNat = 64.f;   // of the first search: 32 nats
constexpr int kList = kWave;          // entries that one wave ranks, a lane each

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
};

// w = e^((x - m) / T) in units of 2^-bits, rounded to the nearest: 2^t with t = n + f, |f| <= 1/2, the series
// of e^(f ln 2) to the tenth power (off by 2e-13 of itself), and an addition that leaves the integer in
// the low bits of the sum.
struct Mass {
    double m, c, magic;   // c = log2(e) / T, magic = 2^(52 - bits)
    __device__ __forceinline__ double real(float x) const {
        const double t = fmax((static_cast<double>(x) - m) * c, -1000.);
        const double n = __builtin_rint(t), f = (t - n) * 0.69314718055994530942;
        double p = 1. / 3628800;
        p = __builtin_fma(p, f, 1. / 362880);
        p = __builtin_fma(p, f, 1. / 40320);
        p = __builtin_fma(p, f, 1. / 5040);
        p = __builtin_fma(p, f, 1. / 720);
        p = __builtin_fma(p, f, 1. / 120);
        p = __builtin_fma(p, f, 1. / 24);
        p = __builtin_fma(p, f, 1. / 6);
        p = __builtin_fma(p, f, 0.5);
        p = __builtin_fma(p, f, 1.);
        p = __builtin_fma(p, f, 1.);
        return __builtin_ldexp(p, static_cast<int>(n));
    }
    __device__ __forceinline__ u64 units(double e) const {
        return __builtin_bit_cast(u64, e + magic) - __builtin_bit_cast(u64, magic);
    }
    __device__ __forceinline__ u64 operator()(float x) const { return units(real(x)); }
};

__device__ __forceinline__ u64 wave_add(u64 v) {
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
    return v;
}
__device__ __forceinline__ u64 wave_scan(u64 v, int lane) {   // inclusive
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
        const u64 o = __shfl_up(v, off, kWave);
        v += lane >= off ? o : 0;
    }
    return v;
}

// A wave's run of the row: `count` tiles of 64 vectors each, from element `from` on.
template <int DT> struct Run {
    static constexpr int vec = Elem<DT>::vec, tile = kWave * vec;
    const char *row;
    int n, from, count, lane;
    // f(elements, index of the first): false ends the run
    template <class F> __device__ __forceinline__ void each_tile(F f) const {
        for (int t = 0; t < count; ++t) {
            const int i = from + t * tile + lane * vec;
            float x[vec];
            load_vec<DT, false>(row, i, n, x);
            if (!f(x, i)) return;
        }
    }
    // f(element, index), masked ones (and what lies past the end) left out
    template <class F> __device__ __forceinline__ void each(F f) const {
        each_tile([&](const float (&x)[vec], int i) {
#pragma unroll
            for (int k = 0; k < vec; ++k)
                if (x[k] > -INFINITY) f(x[k], i + k);
            return true;
        });
    }
};

template <int NT> struct Scratch {
    u64 mass[kBins];
    int count[kBins];
    u64 wave_mass[NT / kWave];
    int wave_count[NT / kWave];
    float wave_top[NT / kWave];
    int wave_odd[NT / kWave];
    u64 key[kList], weight[kList];
    u64 lo, hi, before_mass, found;
    int held, bin, before_count, bin_count, first;
};

// Entries of the row with keys in [lo, hi], sorted into bins from the top down, and what lies above them.
struct Window {
    u64 lo, hi;         // keys
    u64 above_mass;
    int above_count;
};

// The last kept key where the first `k` ranks are kept (MASS false), or those before which lies less than `goal` of mass
// (MASS true). Only keys of `least` and above exist. Also the mass down to that key.
//
// The entries are sorted into bins by an order-keeping function: at first by their distance from the
// largest, 1/64 nat a bin, then by the bits of their keys, which are unique, until the
// bin in which the last kept one lies holds no more than a wave can rank.
template <bool MASS, int DT, int NT>
__device__ u64 last_key(const Run<DT> &run, const Mass &mass, float m, float scale, u64 least, int k, double goal,
                        u64 &mass_down_to, Scratch<NT> &sc) {
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    Window w{0, 0, 0, 0};
    bool first = true;
    int shift = 0;
    for (;;) {
        for (int i = tid; i < kBins; i += NT) sc.mass[i] = sc.count[i] = 0;
        if (tid == 0) {
            sc.lo = ~0ull;
            sc.hi = 0;
            sc.held = 0;
        }
        __syncthreads();
        auto bin_of = [&](float x, u64 key) {
            if (first) return static_cast<int>(fminf((m - x) * scale, static_cast<float>(kBins - 1)));
            return static_cast<int>((w.hi - key) >> shift);
        };
        auto inside = [&](u64 key) { return key >= least && (first || (key >= w.lo && key <= w.hi)); };
        run.each([&](float x, int i) {
            const u64 key = key_of(x, i);
            if (!inside(key)) return;
            const int b = bin_of(x, key);
            atomicAdd(&sc.count[b], 1);
            atomicAdd(&sc.mass[b], mass(x));
        });
        __syncthreads();
        // the bin in which the last kept one lies: a thread adds up consecutive bins
        constexpr int each = kBins / NT;
        u64 own = 0;
        int own_count = 0;
        for (int i = 0; i < each; ++i) {
            own += sc.mass[tid * each + i];
            own_count += sc.count[tid * each + i];
        }
        const u64 to = wave_scan(own, lane);
        const int to_count = static_cast<int>(wave_scan(static_cast<u64>(own_count), lane));
        if (lane == kWave - 1) {
            sc.wave_mass[wave] = to;
            sc.wave_count[wave] = to_count;
        }
        __syncthreads();
        u64 before = w.above_mass + to - own;
        int before_count = w.above_count + to_count - own_count;
        for (int i = 0; i < wave; ++i) {
            before += sc.wave_mass[i];
            before_count += sc.wave_count[i];
        }
        for (int i = 0; i < each; ++i) {
            const int b = tid * each + i, c = sc.count[b];
            const u64 o = sc.mass[b];
            const bool starts = MASS ? static_cast<double>(before) < goal : before_count < k;
            const bool ends = MASS ? !(static_cast<double>(before + o) < goal) : before_count + c >= k;
            if (c && starts && ends) {
                sc.bin = b;
                sc.before_mass = before;
                sc.before_count = before_count;
                sc.bin_count = c;
            }
            before += o;
            before_count += c;
        }
        __syncthreads();
        const int bin = sc.bin, held = sc.bin_count;
        w.above_mass = sc.before_mass;
        w.above_count = sc.before_count;
        // its entries: their keys, or the range of those
        run.each([&](float x, int i) {
            const u64 key = key_of(x, i);
            if (!inside(key) || bin_of(x, key) != bin) return;
            if (held <= kList) {
                sc.key[atomicAdd(&sc.held, 1)] = key;
            } else {
                atomicMin(&sc.lo, key);
                atomicMax(&sc.hi, key);
            }
        });
        __syncthreads();
        if (held <= kList) break;
        w.lo = sc.lo;
        w.hi = sc.hi;
        first = false;
        shift = max(0, 64 - __clzll(w.hi - w.lo) - 11);   // (hi - lo) >> shift below 2048
        __syncthreads();
    }
    if (wave == 0) {
        const int held = sc.bin_count;
        const u64 key = lane < held ? sc.key[lane] : 0, own = lane < held ? mass(value_of(key)) : 0;
        u64 before = w.above_mass;
        int rank = w.above_count;
        for (int j = 0; j < held; ++j) {
            const u64 o = __shfl(key, j, kWave), om = __shfl(own, j, kWave);
            if (o > key) {
                before += om;
                ++rank;
            }
        }
        const bool keep = lane < held && (MASS ? static_cast<double>(before) < goal : rank < k);
        const int last = __popcll(__ballot(keep)) - 1;   // kept ones are a prefix: ranks 0 .. last of the bin
        if (keep && rank - w.above_count == last) {
            sc.found = key;
            sc.before_mass = before + own;
        }
    }
    __syncthreads();
    mass_down_to = sc.before_mass;
    const u64 found = sc.found;
    __syncthreads();
    return found;
}

template <int DT, int NT>
__global__ __launch_bounds__(NT) void sample_kernel(Args a) {
    using R = Run<DT>;
    constexpr int V = R::vec, W = NT / kWave;
    const long long r = block_id();
    if (r >= a.v.rows) return;
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave, n = a.v.V;
    __shared__ Scratch<NT> sc;
    const int tiles = (n + R::tile - 1) / R::tile, per_wave = (tiles + W - 1) / W;
    R run;
    run.row = a.v.row(r, Elem<DT>::bytes);
    run.n = n;
    run.from = wave * per_wave * R::tile;
    run.count = max(0, min(per_wave, tiles - wave * per_wave));
    run.lane = lane;
    const double T = a.temperature.at(r), p = a.top_p.at(r), mp = a.min_p.at(r);
    const long long k = a.top_ks ? a.top_ks[r] : a.top_k;
    double u = a.u_double ? static_cast<const double *>(a.u)[r] : static_cast<double>(static_cast<const float *>(a.u)[r]);

    // the largest entry, the number of those that are not masked, and whether one is no number
    float m = -INFINITY;
    int finite = 0, odd = 0;
    run.each_tile([&](const float (&x)[V], int) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            m = fmaxf(m, x[i]);
            finite += x[i] > -INFINITY;
            odd |= !(x[i] < INFINITY);
        }
        return true;
    });
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) {
        m = fmaxf(m, __shfl_xor(m, off, kWave));
        finite += __shfl_xor(finite, off, kWave);
        odd |= __shfl_xor(odd, off, kWave);
    }
    if (lane == 0) {
        sc.wave_top[wave] = m;
        sc.wave_count[wave] = finite;
        sc.wave_odd[wave] = odd;
    }
    if (tid == 0) sc.first = n;
    __syncthreads();
    finite = 0;
    for (int i = 0; i < W; ++i) {
        m = fmaxf(m, sc.wave_top[i]);
        finite += sc.wave_count[i];
        odd |= sc.wave_odd[i];
    }
    if (odd || finite == 0 || !(T >= 0. && T < static_cast<double>(INFINITY)) || p != p || mp != mp) {
        if (tid == 0) {
            a.token[r] = -1;
            a.logprob[r] = __builtin_nanf("");
            a.kept[r] = 0;
        }
        return;
    }
    if (T == 0. || k == 1 || p <= 0. || mp > 1.) {   // the first of the largest
        run.each([&](float x, int i) {
            if (x == m) atomicMin(&sc.first, i);
        });
        __syncthreads();
        if (tid == 0) {
            a.token[r] = sc.first;
            a.logprob[r] = 0.f;
            a.kept[r] = 1;
        }
        return;
    }
    __syncthreads();

    const double inv = 1. / T;
    const Mass mass{static_cast<double>(m), 1.4426950408889634074 * inv, __builtin_ldexp(1., 52 - a.bits)};
    const float scale = static_cast<float>(fmin(kBinsPerNat * inv, 3e38));
    u64 least = 0, total = 0;
    const bool by_k = k > 1 && k < finite;
    if (by_k) least = last_key<false>(run, mass, m, scale, 0, static_cast<int>(k), 0., total, sc);
    if (p < 1.) {
        if (!by_k) {
            u64 own = 0;
            run.each([&](float x, int) { own += mass(x); });
            own = wave_add(own);
            if (lane == 0) sc.wave_mass[wave] = own;
            __syncthreads();
            for (int i = 0; i < W; ++i) total += sc.wave_mass[i];
            __syncthreads();
        }
        u64 down;
        least = last_key<true>(run, mass, m, scale, least, 0, p * static_cast<double>(total), down, sc);
    }

    // what is kept of each wave's run
    auto kept = [&](float x, int i, u64 &w) {
        if (key_of(x, i) < least) return false;
        const double e = mass.real(x);
        w = mass.units(e);
        return e >= mp;
    };
    u64 own = 0;
    int count = 0;
    run.each([&](float x, int i) {
        u64 w;
        if (kept(x, i, w)) {
            own += w;
            ++count;
        }
    });
    own = wave_add(own);
    count = static_cast<int>(wave_add(static_cast<u64>(count)));
    if (lane == 0) {
        sc.wave_mass[wave] = own;
        sc.wave_count[wave] = count;
    }
    __syncthreads();
    u64 Z = 0;
    count = 0;
    for (int i = 0; i < W; ++i) {
        Z += sc.wave_mass[i];
        count += sc.wave_count[i];
    }
    u = u >= 0. ? fmin(u, 1.) : 0.;
    const u64 goal = min(static_cast<u64>(u * static_cast<double>(Z)), Z - 1);   // running sums above it, in whole units
    u64 before = 0;
    for (int i = 0; i < wave; ++i) before += sc.wave_mass[i];
    if (!(before <= goal && goal < before + own)) return;   // another wave's
    run.each_tile([&](const float (&x)[V], int i) {
        u64 w[V], lane_sum = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            w[j] = 0;
            u64 o;
            if (x[j] > -INFINITY && kept(x[j], i + j, o)) w[j] = o;
            lane_sum += w[j];
        }
        const u64 to = wave_scan(lane_sum, lane);
        const u64 tile_sum = __shfl(to, kWave - 1, kWave);
        if (before + tile_sum <= goal) {
            before += tile_sum;
            return true;
        }
        u64 run_to = before + to - lane_sum;
        if (run_to <= goal && goal < run_to + lane_sum) {   // one lane
            bool done = false;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                run_to += w[j];
                if (!done && goal < run_to) {
                    done = true;
                    a.token[r] = i + j;
                    a.logprob[r] = static_cast<float>((static_cast<double>(x[j]) - mass.m) * inv -
                                                      log(__builtin_ldexp(static_cast<double>(Z), -a.bits)));
                    a.kept[r] = count;
                }
            }
        }
        return false;
    });
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
    const smp::Args a{{static_cast<const char *>(logits), inner, outer_stride, row_stride, rows, V},
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
                      log_v <= 15 ? 47 : 62 - log_v};
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto launch = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        const dim3 grid = smp::grid_of(rows);
        if (V <= 4096) smp::sample_kernel<DT, 256><<<grid, dim3(256), 0, s>>>(a);
        else smp::sample_kernel<DT, 1024><<<grid, dim3(1024), 0, s>>>(a);
    };
    if (dtype == ULM_F32) launch(std::integral_constant<int, ULM_F32>{});
    else if (dtype == ULM_BF16) launch(std::integral_constant<int, ULM_BF16>{});
    else launch(std::integral_constant<int, ULM_F16>{});
    return check_launch("ulm_sample_tokens");
}
