// Distillation from a teacher's top logits: how far a row's distribution is from
// the teacher's over the tokens that the teacher lists, and the logits' gradient.
// Beside it, in the same passes, the log probability of the row's own token (the
// text's loss, F.cross_entropy's, model.py:160-161).
//
// For a row x of V logits and entries (i_k, t_k), k < K, at temperature T:
//
//     p_j = softmax(x / T)_j      q_k = softmax_k(t / T)          loss = sum_k q_k (ln q_k - ln p_(i_k))
//     dloss/dx_j = (Q p_j - sum_(k: i_k = j) q_k) / T,            Q = sum_k q_k (1, or 0 without entries)
//
// or, with the rest, q_k = e^t_k, q_r = max(0, 1 - sum_k q_k) and p_r the mass of the tokens not
// listed, which share it as h_j = p_j / p_r:
//
//     loss += q_r (ln q_r - ln p_r)      dloss/dx_j = (Q p_j - sum_(k: i_k = j) q_k) / T   j listed, Q = sum_k q_k + q_r
//                                                    = h_j (Q p_r - q_r) / T               j not listed
//
// p_r is a sum of its own: 1 less the listed tokens' mass has no digits left where the student knows
// the teacher's tokens.
#include <type_traits>

#include "logit_rows.h"

namespace ulm {
namespace ds {

using namespace rows;

constexpr int kUnroll = 4;               // 16-byte loads in flight per thread
constexpr int kMaxEntries = 1024;
constexpr int kMaxRestV = 1 << 18;       // one bit a column in LDS
constexpr long long kHeld = 256ll << 20;   // bytes that the last-level cache holds, from the forward to the backward
constexpr int kStats = 8;                // floats a row kept for the backward
constexpr float kNaN = __builtin_nanf("");

__device__ __forceinline__ float exp2_of(float t) { return __builtin_amdgcn_exp2f(t); }

struct Teacher {
    const long long *ids;
    const void *values;
    int dtype, K;
};

struct Args {
    View v;
    Teacher t;
    const long long *tokens;
    long long ignore;
    float inv_tau, c;   // 1 / T and log2(e) / T
};

// An entry of a row: -1 is none.
struct Entry {
    long long id;
    float t, x;   // the teacher's value and the student's logit; -inf where there is none
    bool there, bad;
};
template <int DT> __device__ __forceinline__ Entry entry_of(const Args &a, const char *row, long long r, int k) {
    Entry e{-1, -INFINITY, -INFINITY, false, false};
    if (k >= a.t.K) return e;
    e.id = a.t.ids[r * a.t.K + k];
    e.there = e.id >= 0 && e.id < a.v.V;
    e.bad = !e.there && e.id != -1;
    if (e.there) {
        e.t = load_as_f32(a.t.values, r * a.t.K + k, a.t.dtype);
        e.x = load_as_f32(row, e.id, DT);
    }
    return e;
}

// The tokens' own log probabilities beside a loss at another temperature take exponentials of their own, but at twice
// theirs, the usual one: there e^(x - m) is the square of e^((x - m) / 2) (the forward of 16384 rows of 32000 bf16
// 156 us, bound by the reading, and 183 with exponentials of their own).
enum Second { ONE = 0, TWO = 1, SQUARE = 2 };

// Sums of e^((x - m) / T), and of e^(x - m) but with ONE, about their maximum m.
template <Second S> struct Sums {
    float m, s, s1;
    static __device__ __forceinline__ Sums none() { return {-INFINITY, 0.f, 0.f}; }
    __device__ __forceinline__ void rebase(float to, float c) {   // to > m, or to = m
        const float d = m == to ? 0.f : m - to;
        s *= exp2_of(d * c);
        if constexpr (S != ONE) s1 *= exp2_of(d * kLog2e);
        m = to;
    }
    template <int N> __device__ __forceinline__ void take(const float (&x)[N], float c) {
        float most = m;
#pragma unroll
        for (int i = 0; i < N; i += 2) most = max3(most, x[i], x[i + 1]);
        if (most > m) rebase(most, c);
        if (m == -INFINITY) {   // nothing but masked elements so far (or NaN)
#pragma unroll
            for (int i = 0; i < N; ++i) s += x[i] != x[i] ? x[i] : 0.f;
            s1 = s;
            return;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float d = x[i] - m, e = exp2_of(d * c);
            s += e;
            if constexpr (S == TWO) s1 += exp2_of(d * kLog2e);
            if constexpr (S == SQUARE) s1 = __builtin_fmaf(e, e, s1);
        }
    }
    // over groups of W lanes
    template <int W> __device__ __forceinline__ void join(float c) {
        float to = m;
#pragma unroll
        for (int off = W / 2; off > 0; off >>= 1) to = fmaxf(to, __shfl_xor(to, off, kWave));
        rebase(to, c);
#pragma unroll
        for (int off = W / 2; off > 0; off >>= 1) {
            s += __shfl_xor(s, off, kWave);
            if constexpr (S != ONE) s1 += __shfl_xor(s1, off, kWave);
        }
    }
};

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, kWave));
    return v;
}

// 32 bits of a mask from bit i on
__device__ __forceinline__ uint32_t bits_at(const uint32_t *mask, int i) {
    return __builtin_amdgcn_alignbit(mask[i / 32 + 1], mask[i / 32], i % 32);
}

// KEEP, where the cache holds them all: the logits are read as what will be read again. Forward and backward with 32 entries,
// one batch after another, of 4096 rows of 32000 bf16 (250 MiB) 137 us, and 144 with loads that stream in both; of 2048 rows fp32
// 125 and 130; of 6400 rows bf16 (390 MiB) 216 and 218, of 8192 (500 MiB) 282 and 280; of 1 GB 561 and 551. A forward alone,
// which nothing follows, is the slower for it: of 4096 rows bf16 49 us and 44, of 2048 rows fp32 47 and 42.
//
// One workgroup of NT threads per row, one pass over it, which bounds it: 8192 rows of 32000 bf16 82 us, 6.4 TB/s; 2048
// rows of 32000 fp32 with the rest 42 us, 6.2 TB/s. The teacher's entries, the token and their logits are read ahead
// and end the row on one wave.
template <int DT, bool REST, Second S, bool KEEP, int NT>
__global__ __launch_bounds__(NT) void fwd_kernel(Args a, float *loss_out, float *logprob_out, float *stats) {
    constexpr int V = Elem<DT>::vec, B = Elem<DT>::bytes, W = NT / kWave, kTile = NT * V * kUnroll;
    const long long r = block_id();
    if (r >= a.v.rows) return;
    const int tid = threadIdx.x, lane = tid % kWave, n = a.v.V, K = a.t.K;
    const char *row = a.v.row(r, B);
    extern __shared__ uint32_t mask[];   // REST: the listed columns
    __shared__ Sums<S> waves[W];
    __shared__ int twice;                // a token is listed more than once
    if constexpr (REST) {
        if (tid == 0) twice = 0;
        for (int i = tid; i < n / 32 + 2; i += NT) mask[i] = 0;
        __syncthreads();
        for (int k = tid; k < K; k += NT) {
            const long long id = a.t.ids[r * K + k];
            if (id >= 0 && id < n && (atomicOr(&mask[id / 32], 1u << (id % 32)) >> (id % 32) & 1)) twice = 1;
        }
        __syncthreads();
    }
    // what the row ends with arrives while its elements are under way
    Entry first{};
    long long label = -1;
    float label_x = 0.f;
    if (tid < kWave) {
        first = entry_of<DT>(a, row, r, lane);
        if (a.tokens) {
            label = a.tokens[r];
            if (label >= 0 && label < n) label_x = load_as_f32(row, label, DT);
        }
    }

    Sums<S> v = Sums<S>::none();
    for (int e0 = 0; e0 < n; e0 += kTile) {
        float x[kUnroll * V];
        const bool whole = e0 + kTile <= n;
        auto at = [&](int j) { return e0 + (j * NT + tid) * V; };
        if (n >= V) {   // every load inside the row: the last tile's overhang reads its last elements and drops them
            u32x4_any w[kUnroll];
#pragma unroll
            for (int j = 0; j < kUnroll; ++j) {
                const char *p = row + static_cast<size_t>(min(at(j), n - V)) * B;
                w[j] = KEEP ? *reinterpret_cast<const u32x4_any *>(p) : load_once(p);
            }
#pragma unroll
            for (int j = 0; j < kUnroll; ++j) unpack<DT>(w[j], *reinterpret_cast<float(*)[V]>(&x[j * V]));
            if (!whole) {
                asm volatile("");   // a branch: 64 selects in every tile otherwise
#pragma unroll
                for (int j = 0; j < kUnroll; ++j) {
                    const int over = at(j) - (n - V);   // the first `over` elements are others'
#pragma unroll
                    for (int i = 0; i < V; ++i) x[j * V + i] = i < over ? -INFINITY : x[j * V + i];
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < kUnroll; ++j) load_vec<DT>(row, at(j), n, *reinterpret_cast<float(*)[V]>(&x[j * V]));
        }
        if constexpr (REST) {
#pragma unroll
            for (int j = 0; j < kUnroll; ++j) {
                const uint32_t bits = bits_at(mask, max(0, min(at(j), n - V)));
                if (bits & ((1u << V) - 1)) {
#pragma unroll
                    for (int i = 0; i < V; ++i) x[j * V + i] = bits >> i & 1 ? -INFINITY : x[j * V + i];
                }
            }
        }
        v.take(x, a.c);
    }
    v.template join<kWave>(a.c);
    if (lane == 0) waves[tid / kWave] = v;
    __syncthreads();
    if (tid >= kWave) return;
    Sums<S> all = waves[lane % W];
    all.template join<W>(a.c);

    // one wave ends the row, a lane per entry at a time
    auto each = [&](auto f) {
        for (int k = lane; k - lane < K; k += kWave) f(k < kWave ? first : entry_of<DT>(a, row, r, k), k);
    };
    const Sums<S> rest = all;
    bool bad = false;
    float tm = -INFINITY, Q = 0.f, qr = 0.f, tl = 0.f;
    if constexpr (REST) {
        Sums<S> listed = Sums<S>::none();
        double q = 0.;
        bool any = false;
        each([&](const Entry &e, int k) {
            bad |= e.bad;
            any |= e.there;
            if (e.there) q += exp(static_cast<double>(e.t));
            bool counts = e.there;
            if (counts && twice)
                for (int j = 0; j < k; ++j) counts &= a.t.ids[r * K + j] != e.id;
            const float x[2] = {counts ? e.x : -INFINITY, -INFINITY};
            listed.take(x, a.c);
        });
        q = wave_sum(q);
        qr = __any(any) ? static_cast<float>(fmax(0., 1. - q)) : 0.f;   // without entries nothing is known of the rest
        Q = static_cast<float>(q) + qr;
        listed.template join<kWave>(a.c);
        const float to = fmaxf(all.m, listed.m);
        listed.rebase(to, a.c);
        all.rebase(to, a.c);
        all.s += listed.s;
        all.s1 += listed.s1;
    } else {
        each([&](const Entry &e, int) {
            bad |= e.bad;
            tm = fmaxf(tm, e.t);
        });
        tm = wave_max(tm);
        float s = 0.f;
        each([&](const Entry &e, int) { s += e.there && tm != -INFINITY ? exp2_of((e.t - tm) * a.c) : e.t != e.t ? e.t : 0.f; });
        s = wave_sum(s);
        tl = logf(s);
        Q = s > 0.f ? 1.f : s;
    }
    bad = __any(bad);
    const bool empty = all.s == 0.f;
    const float ls = logf(all.s), M = all.m;
    float loss = 0.f;
    each([&](const Entry &e, int) {
        const float lq = REST ? e.t : (e.t - tm) * a.inv_tau - tl;
        const float lp = empty ? -INFINITY : (e.x - M) * a.inv_tau - ls;
        const bool nothing = !e.there || (!REST && tm == -INFINITY && e.t == e.t);
        const float q = nothing ? 0.f : exp2_of(lq * kLog2e);
        loss += q == 0.f ? 0.f : q * (lq - lp);
    });
    loss = wave_sum(loss);
    if (lane) return;
    float mu = M, lu = ls, Cu = Q;   // the tokens not listed: e^((x - mu) / T - lu) Cu
    if constexpr (REST) {
        const bool none = rest.s == 0.f;
        const float lr = logf(rest.s), lpr = none ? -INFINITY : (rest.m - M) * a.inv_tau + (lr - ls);
        loss += qr == 0.f ? 0.f : qr * (logf(qr) - lpr);
        mu = none ? 0.f : rest.m;
        lu = none ? 0.f : lr;
        Cu = none ? 0.f : Q * exp2_of(lpr * kLog2e) - qr;
    }
    if (bad) loss = Q = Cu = kNaN;
    loss_out[r] = loss;
    const float l1 = S != ONE ? logf(all.s1) : ls;
    if (logprob_out) {
        float lp = 0.f;
        if (label != a.ignore) {
            lp = kNaN;
            if (label >= 0 && label < n) lp = empty ? -INFINITY : (label_x - M) - l1;
        }
        logprob_out[r] = lp;
    }
    if (stats) {
        float *o = stats + r * kStats;
        o[0] = mu;
        o[1] = lu * kLog2e;
        o[2] = Cu;
        o[3] = Q;
        o[4] = REST ? M : tm;
        o[5] = (REST ? ls : tl) * kLog2e;
        o[6] = l1 * kLog2e;
        o[7] = empty ? 1.f : 0.f;
    }
}

struct Grads {
    const float *stats, *dloss, *dlogprob;
    char *dx;   // (rows, V), dense
};

constexpr int kThreads = 256;    // of the backward
constexpr int kBwdVectors = 3;   // a thread

// One workgroup per (row, tile of three vectors a thread). The tile's entries are found first, while its elements are
// under way: a bit and a value a column. Vectors without an entry or the token, nearly all, take
// their elements alike. Forward and backward of 16384 rows of 32000 bf16 with 64 entries, at twice the temperature and with
// the text's tokens, 548 us; of 2048 rows fp32 with 32 entries, the rest and the text's tokens 129. (With one vector a thread
// 674 and 159, so many workgroups look for their entries; with two 550 and 138, with four 537 and 132.)
template <int DT, bool REST, Second S, bool KEEP>
__global__ __launch_bounds__(kThreads) void bwd_kernel(Args a, Grads g, int tiles) {
    constexpr int V = Elem<DT>::vec, B = Elem<DT>::bytes, U = kBwdVectors, kTile = kThreads * V * U;
    const long long id = a.v.rows * tiles - 1 - block_id();   // from the last row back: the caches hold what was read last
    if (id < 0) return;
    const long long r = id / tiles;
    const int tid = threadIdx.x, K = a.t.K, n = a.v.V;
    const int e0 = static_cast<int>(id - r * tiles) * kTile, e1 = min(n, e0 + kTile);
    const char *row = a.v.row(r, B);
    char *out = g.dx + static_cast<size_t>(r) * n * B;
    __shared__ uint32_t mask[kTile / 32 + 1];
    __shared__ uint16_t entry[kTile];       // of the listed columns,
    __shared__ float value[kMaxEntries];    // and each one's -q / T times the loss's gradient
    __shared__ int twice;
    const float *st = g.stats + r * kStats;
    const float mu = st[0], lu = st[1], s4 = st[4], s5 = st[5], l1 = st[6];
    const bool empty = st[7] != 0.f;
    const float A = g.dloss ? g.dloss[r] * a.inv_tau : 0.f;
    const bool learns = A != 0.f;   // a row that pads takes nothing from its entries, NaN among them neither
    const float Cu = learns ? st[2] : 0.f, Q = learns ? st[3] : 0.f;
    const bool own = g.dlogprob != nullptr;   // the row's own token has a gradient
    const long long t = own ? a.tokens[r] : a.ignore;
    float da = t != a.ignore ? g.dlogprob[r] : 0.f;
    if (t != a.ignore && (t < 0 || t >= n)) da = kNaN;
    float x[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int i = e0 + (u * kThreads + tid) * V;
        if (i < e1) load_vec<DT, !KEEP>(row, i, e1, x[u]);
    }
    if (tid == 0) twice = 0;
    for (int i = tid; i < kTile / 32 + 1; i += kThreads) mask[i] = 0;
    __syncthreads();
    auto q_of = [&](float v) {
        if (REST) return exp2_of(v * kLog2e);
        return s4 == -INFINITY && v == v ? 0.f : exp2_of((v - s4) * a.c - s5);
    };
    auto part_of = [&](float q) { return learns ? -A * q : 0.f; };
    auto value_at = [&](int k) { return load_as_f32(a.t.values, r * K + k, a.t.dtype); };
    for (int k = tid; k < K; k += kThreads) {
        const long long j = a.t.ids[r * K + k];
        const float v = value_at(k);   // with the token: not after it
        if (j < e0 || j >= e1) continue;
        const int at = static_cast<int>(j) - e0;
        if (atomicOr(&mask[at / 32], 1u << (at % 32)) >> (at % 32) & 1) twice = 1;
        entry[at] = static_cast<uint16_t>(k);
        value[k] = part_of(q_of(v));
    }
    __syncthreads();
    if (twice) {   // the same token again: its entries' sum, in their order, for each of them
        for (int k = tid; k < K; k += kThreads) {
            const long long j = a.t.ids[r * K + k];
            if (j < e0 || j >= e1) continue;
            float q = 0.f;
            for (int i = 0; i < K; ++i)
                if (a.t.ids[r * K + i] == j) q += q_of(value_at(i));
            value[k] = part_of(q);
        }
        __syncthreads();
    }
    const float M = REST ? s4 : mu, ls = REST ? s5 : lu;
    const bool plain = S == ONE && !REST;   // one exponential serves both
    const float cu = plain ? A * Cu - da : A * Cu;
    const float square = S == SQUARE && !REST ? -da * exp2_of(2.f * lu - l1) : 0.f;   // of p at twice the temperature
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int i = e0 + (u * kThreads + tid) * V;
        if (i >= e1) continue;
        auto own_part = [&](float x) { return -da * exp2_of(__builtin_fmaf(x - M, kLog2e, -l1)); };
        float y[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const float h = exp2_of(__builtin_fmaf(x[u][k] - mu, a.c, -lu));
            y[k] = S == SQUARE && !REST ? h * __builtin_fmaf(h, square, cu) : cu * h;
            if (!plain && !(S == SQUARE && !REST) && own) y[k] += own_part(x[u][k]);
        }
        const uint32_t bits = bits_at(mask, i - e0) & ((1u << V) - 1);
        const bool here = t >= i && t < i + V;
        if (bits || here) {
            const int place = here ? static_cast<int>(t - i) : -1;
#pragma unroll
            for (int k = 0; k < V; ++k) {
                if (bits >> k & 1) {
                    const float q = value[entry[i - e0 + k]];
                    if (REST) {
                        y[k] = __builtin_fmaf(A * Q, exp2_of(__builtin_fmaf(x[u][k] - M, a.c, -ls)), q);
                        if (own) y[k] += own_part(x[u][k]);
                    } else {
                        y[k] += q;
                    }
                }
                if (place == k) y[k] += da;
            }
        }
#pragma unroll
        for (int k = 0; k < V; ++k) x[u][k] = empty ? 0.f : y[k];
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
}

}  // namespace ds
}  // namespace ulm

using namespace ulm;

static int check_distill(const char *fn, const ulm_distillation *d) {
    if (!d) return fail(ULM_ERR_INVALID, "%s: null pointer", fn);
    if (d->rows < 1 || d->rows > (1LL << 34) || d->inner < 1 || d->V < 1 || d->V > (1 << 30))
        return fail(ULM_ERR_INVALID, "%s: bad sizes rows=%lld inner=%lld V=%d", fn, d->rows, d->inner, d->V);
    if (d->K < 1 || d->K > ds::kMaxEntries)
        return fail(ULM_ERR_INVALID, "%s: K=%d outside 1 .. %d", fn, d->K, ds::kMaxEntries);
    if (d->rest && d->V > ds::kMaxRestV) return fail(ULM_ERR_INVALID, "%s: the rest with V=%d", fn, d->V);
    if (!valid_dtype(d->dtype) || !valid_dtype(d->teacher_dtype))
        return fail(ULM_ERR_INVALID, "%s: bad dtype %d or %d", fn, d->dtype, d->teacher_dtype);
    if (!(d->temperature >= 1e-6f && d->temperature <= 1e6f))
        return fail(ULM_ERR_INVALID, "%s: temperature %g", fn, d->temperature);
    if (!d->logits || !d->teacher_tokens || !d->teacher_logits) return fail(ULM_ERR_INVALID, "%s: null pointer", fn);
    return ULM_OK;
}

static ds::Args distill_args(const ulm_distillation *d) {
    return {{static_cast<const char *>(d->logits), d->inner, d->outer_stride, d->row_stride, d->rows, d->V},
            {d->teacher_tokens, d->teacher_logits, d->teacher_dtype, d->K},
            d->tokens, d->ignore_index, 1.f / d->temperature, ds::kLog2e / d->temperature};
}

template <class F> static void by_kind(const ulm_distillation *d, bool own, F f) {
    using ds::Second;
    const Second second = !own || d->temperature == 1.f ? ds::ONE : d->temperature == 2.f ? ds::SQUARE : ds::TWO;
    const bool keep = d->rows <= ds::kHeld / d->V / (d->dtype == ULM_F32 ? 4 : 2);
    auto by_keep = [&](auto dt, auto r, auto s) {
        if (keep) f(dt, r, s, std::true_type{});
        else f(dt, r, s, std::false_type{});
    };
    auto by_second = [&](auto dt, auto r) {
        if (second == ds::ONE) by_keep(dt, r, std::integral_constant<Second, ds::ONE>{});
        else if (second == ds::TWO) by_keep(dt, r, std::integral_constant<Second, ds::TWO>{});
        else by_keep(dt, r, std::integral_constant<Second, ds::SQUARE>{});
    };
    auto by_rest = [&](auto dt) {
        if (d->rest) by_second(dt, std::true_type{});
        else by_second(dt, std::false_type{});
    };
    if (d->dtype == ULM_F32) by_rest(std::integral_constant<int, ULM_F32>{});
    else if (d->dtype == ULM_BF16) by_rest(std::integral_constant<int, ULM_BF16>{});
    else by_rest(std::integral_constant<int, ULM_F16>{});
}

extern "C" int ulm_distill_max_entries(void) { return ds::kMaxEntries; }
extern "C" int ulm_distill_stats(void) { return ds::kStats; }

extern "C" int ulm_distill(const ulm_distillation *d, float *loss, float *logprob, float *stats, void *stream) {
    ULM_TRY(check_distill("ulm_distill", d));
    ULM_REQUIRE(loss && (!logprob || d->tokens), "ulm_distill: null pointer");
    const ds::Args a = distill_args(d);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int vec = d->dtype == ULM_F32 ? 4 : 8;
    int nt = 64;
    while (nt < 256 && d->V >= 2 * nt * vec * ds::kUnroll) nt *= 2;
    const size_t lds = d->rest ? (static_cast<size_t>(d->V) / 32 + 2) * 4 : 0;
    by_kind(d, logprob != nullptr, [&](auto dt, auto rest, auto second, auto keep) {
        constexpr int DT = decltype(dt)::value;
        constexpr bool R = decltype(rest)::value;
        constexpr ds::Second T = decltype(second)::value;
        constexpr bool H = decltype(keep)::value;
        const dim3 grid = ds::grid_of(d->rows);
        if (nt == 64) ds::fwd_kernel<DT, R, T, H, 64><<<grid, dim3(64), lds, s>>>(a, loss, logprob, stats);
        else if (nt == 128) ds::fwd_kernel<DT, R, T, H, 128><<<grid, dim3(128), lds, s>>>(a, loss, logprob, stats);
        else ds::fwd_kernel<DT, R, T, H, 256><<<grid, dim3(256), lds, s>>>(a, loss, logprob, stats);
    });
    return check_launch("ulm_distill");
}

extern "C" int ulm_distill_bwd(const ulm_distillation *d, const float *stats, const float *dloss, const float *dlogprob,
                               void *dlogits, void *stream) {
    ULM_TRY(check_distill("ulm_distill_bwd", d));
    ULM_REQUIRE(stats && dlogits && (!dlogprob || d->tokens), "ulm_distill_bwd: null pointer");
    ULM_REQUIRE(dlogits != d->logits, "ulm_distill_bwd: dlogits must not alias logits");
    const ds::Args a = distill_args(d);
    const ds::Grads g{stats, dloss, dlogprob, static_cast<char *>(dlogits)};
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int tile = ds::kThreads * ds::kBwdVectors * (d->dtype == ULM_F32 ? 4 : 8), tiles = (d->V + tile - 1) / tile;
    by_kind(d, dlogprob != nullptr, [&](auto dt, auto rest, auto second, auto keep) {
        ds::bwd_kernel<decltype(dt)::value, decltype(rest)::value, decltype(second)::value, decltype(keep)::value>
            <<<ds::grid_of(d->rows * tiles), dim3(ds::kThreads), 0, s>>>(a, g, tiles);
    });
    return check_launch("ulm_distill_bwd");
}
