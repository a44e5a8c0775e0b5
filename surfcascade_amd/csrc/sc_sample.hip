// sc_sample.hip -- draws from rows of scores by given random numbers, on
// gfx950 (the roulette wheel of GentleAdaboost::Train, GentleAdaboost.cpp:
// 11-231, over log-weights, with the usual ways to trim it).
//
//   w_i  = exp((s_i - max) / temperature), absent where s_i is -inf or NaN
//   kept = the first L of the scores in descending order, ties in ascending
//          place: L = min(top_k, the shortest prefix with top_p of the top_k's
//          mass, the weights >= min_p)
//   draw = the smallest place i with sum_{j <= i, kept} w_j > u * sum_kept w
//
// All three trims keep a prefix of one order, so the kept set is a threshold
// on an order-preserving key plus a quota of the places that tie with it:
// no sort.  Weights are doubles and masses integers (sample_shift), so a sum
// is the same in any order and a draw never depends on how the row was split.
//
// The threshold comes from a descent: bins hold counts for top_k, masses for
// top_p, and the bin where the sum from the top crosses is split again, by 11
// bits of the key a level, over many workgroups; in one workgroup the first
// level's bins are even steps of the score and the crossing bin's few members are
// ranked.  Cumulated masses then need one pass in place order, and a draw is a
// search through them.
//
// Short rows, and longer ones of which top_k keeps few: one workgroup each, one
// launch; a thread holds its keys and masses in registers through all passes.
// Other rows: many workgroups, one launch per pass.  Scores are few bytes (1 M of
// them: 4 MB, 1 us): what bounds the first form is one CU's issue (a weight is
// some 40 instructions, half of them in 64 bits) and a pass' barriers, the second
// its launches, 4 to 13 us each, of which most is waiting for the bins of the one
// before.  Measured (one MI355X):
//   960 scores, 960 draws                                 7 us, top_k and top_p 13
//   32 rows x 20011, top_k 2000, top_p, min_p, 128 draws  30 us (split: 60)
//   1000003 scores, top_k 500000, top_p, 16384 draws      65 us
//   64 rows x 128256, one draw, no trim 50 us, top_p 121 us
#include <hip/hip_runtime.h>

#include "sc_train.hpp"
#include "surfcascade.h"

namespace sc {

namespace {

typedef unsigned long long u64;
constexpr int kBinBits = 11, kBins = 1 << kBinBits;

// Order-preserving key of a score; 0: absent (-inf or NaN).
__device__ __forceinline__ unsigned key_of(float s) {
    if (!(s > -__builtin_inff())) return 0;
    const unsigned u = __float_as_uint(s + 0.0f);  // -0 ties with +0
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float score_of(unsigned key) {
    return __uint_as_float((key & 0x80000000u) ? key ^ 0x80000000u : ~key);
}

// The scores of K places of a row of n scores as they lie: only loads, so that
// other loads can be issued behind them before the first is waited for.  Slots
// from `used` on (the same number in every thread) lie past the row's end.
template <int K, class Place>
__device__ __forceinline__ void load_raw(const SampleArgs &a, long long base, int n, unsigned (&raw)[K], Place place,
                                         int used = K) {
    if (n <= 0) {  // nothing to read (there may be no buffer at all)
#pragma unroll
        for (int j = 0; j < K; j++) raw[j] = 0;
        return;
    }
    const int last = n - 1;
    if (a.dtype == SC_F32) {
        const unsigned *p = static_cast<const unsigned *>(a.scores) + base;
#pragma unroll
        for (int j = 0; j < K; j++) raw[j] = j < used ? p[place(j) < n ? place(j) : last] : 0;
    } else {
        const unsigned short *p = static_cast<const unsigned short *>(a.scores) + base;
#pragma unroll
        for (int j = 0; j < K; j++) raw[j] = j < used ? p[place(j) < n ? place(j) : last] : 0;
    }
}
// ... and their keys (0 past the row's end)
template <int K, class Place>
__device__ __forceinline__ void to_keys(const SampleArgs &a, int n, unsigned (&raw)[K], Place place) {
#pragma unroll
    for (int j = 0; j < K; j++) {
        const float f = a.dtype == SC_F32   ? __uint_as_float(raw[j])
                        : a.dtype == SC_F16 ? (float)__builtin_bit_cast(_Float16, (unsigned short)raw[j])
                                            : __uint_as_float(raw[j] << 16);
        raw[j] = place(j) < n ? key_of(f) : 0;
    }
}
template <int K, class Place>
__device__ __forceinline__ void load_keys(const SampleArgs &a, long long base, int n, unsigned (&key)[K], Place place,
                                          int used = K) {
    load_raw<K>(a, base, n, key, place, used);
    to_keys<K>(a, n, key, place);
}

// e^x for x <= 0 to 7e-16: x = n ln 2 + r with |r| <= ln 2 / 2, e^r by its
// Chebyshev interpolation of degree 10 there (5.9e-16), times 2^n.
__device__ __forceinline__ double exp_neg(double x) {
    x = x < -800.0 ? -800.0 : x;  // (2^-1154: 0)
    const double n = rint(x * 1.44269504088896340736);
    double r = __builtin_fma(n, -0.693147180559945286227, x);
    r = __builtin_fma(n, -2.319046813846299558e-17, r);
    double p = 2.7519707534693554e-07;
    p = __builtin_fma(p, r, 2.7642139218631665e-06);
    p = __builtin_fma(p, r, 2.4801790688999252e-05);
    p = __builtin_fma(p, r, 0.00019841165565505855);
    p = __builtin_fma(p, r, 0.00138888886671899);
    p = __builtin_fma(p, r, 0.008333333389376566);
    p = __builtin_fma(p, r, 0.04166666666755826);
    p = __builtin_fma(p, r, 0.166666666665438);
    p = __builtin_fma(p, r, 0.49999999999998807);
    p = __builtin_fma(p, r, 1.0000000000000075);
    p = __builtin_fma(p, r, 1.0);
    return ldexp(p, (int)n);
}

struct Weigh {
    float top;
    double rate;  // 1 / temperature (0: infinite, every weight but the best's is 0)
    double unit;  // 2^shift
    __device__ __forceinline__ double weight(unsigned key) const {
        const float s = score_of(key);
        return s == top ? 1.0 : exp_neg(((double)s - (double)top) * rate);  // (also +inf against +inf)
    }
    // rint(w * unit), at most 2^51: the mantissa of its sum with 2^52
    __device__ __forceinline__ u64 mass(double w) const {
        return (u64)__double_as_longlong(__builtin_fma(w, unit, 4503599627370496.0)) & 0xfffffffffffffull;
    }
};

// Inclusive sum over the lanes of a wave: DPP shifts by 1, 2, 4 and 8 inside
// the rows of 16, then the last lanes of rows broadcast into the rows behind
// (a shuffle through LDS takes several times as long a step).
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned dpp_or_0(unsigned v) {
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS, class V>
__device__ __forceinline__ V scan_step(V x) {
    if constexpr (sizeof(V) == 8) {
        const unsigned lo = dpp_or_0<CTRL, ROWS>((unsigned)x), hi = dpp_or_0<CTRL, ROWS>((unsigned)(x >> 32));
        return x + (((u64)hi << 32) | lo);
    } else {
        return x + dpp_or_0<CTRL, ROWS>(x);
    }
}
template <class V>
__device__ __forceinline__ V wave_scan(V x) {
    x = scan_step<0x111, 0xf>(x);
    x = scan_step<0x112, 0xf>(x);
    x = scan_step<0x114, 0xf>(x);
    x = scan_step<0x118, 0xf>(x);
    x = scan_step<0x142, 0xa>(x);
    return scan_step<0x143, 0xc>(x);
}
__device__ __forceinline__ unsigned lane_of(unsigned v, int lane) {
    return (unsigned)__builtin_amdgcn_readlane((int)v, lane);
}
__device__ __forceinline__ u64 lane_of(u64 v, int lane) {
    return ((u64)lane_of((unsigned)(v >> 32), lane) << 32) | lane_of((unsigned)v, lane);
}
template <class V>
__device__ __forceinline__ V wave_sum(V x) {
    return lane_of(wave_scan(x), 63);
}

// inclusive sum over the N threads of a workgroup; total in every thread
template <int N, class V>
__device__ __forceinline__ V block_scan(V x, V *s_wave, V &total) {
    const int wv = threadIdx.x >> 6;
    x = wave_scan(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) s_wave[wv] = x;
    __syncthreads();
    V before = 0;
    total = 0;
#pragma unroll
    for (int k = 0; k < N / 64; k++) {
        const V v = s_wave[k];
        before += k < wv ? v : 0;
        total += v;
    }
    return before + x;
}

// two of them at once
template <int N, class V, class W>
__device__ __forceinline__ void block_scan2(V &x, W &y, V *s_x, W *s_y, V &total_x, W &total_y) {
    const int wv = threadIdx.x >> 6;
    x = wave_scan(x);
    y = wave_scan(y);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) {
        s_x[wv] = x;
        s_y[wv] = y;
    }
    __syncthreads();
    V bx = 0;
    W by = 0;
    total_x = 0;
    total_y = 0;
#pragma unroll
    for (int k = 0; k < N / 64; k++) {
        const V vx = s_x[k];
        const W vy = s_y[k];
        bx += k < wv ? vx : 0;
        by += k < wv ? vy : 0;
        total_x += vx;
        total_y += vy;
    }
    x += bx;
    y += by;
}

__device__ __forceinline__ void extend(unsigned k, unsigned &lo, unsigned &hi, unsigned &c) {
    if (!k) return;
    lo = k < lo ? k : lo;
    hi = k > hi ? k : hi;
    c++;
}

// smallest and largest key and the count over a workgroup of N threads
template <int N>
__device__ __forceinline__ void block_extent(unsigned &lo, unsigned &hi, unsigned &c, unsigned *s_x) {
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        const unsigned l = __shfl_xor(lo, d, 64), h = __shfl_xor(hi, d, 64);
        lo = l < lo ? l : lo;
        hi = h > hi ? h : hi;
    }
    c = wave_sum(c);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        s_x[3 * (threadIdx.x >> 6)] = lo;
        s_x[3 * (threadIdx.x >> 6) + 1] = hi;
        s_x[3 * (threadIdx.x >> 6) + 2] = c;
    }
    __syncthreads();
    c = 0;
#pragma unroll
    for (int k = 0; k < N / 64; k++) {
        lo = s_x[3 * k] < lo ? s_x[3 * k] : lo;
        hi = s_x[3 * k + 1] > hi ? s_x[3 * k + 1] : hi;
        c += s_x[3 * k + 2];
    }
}

// floor(u * mass) for u clamped to [0, 1): below the mass
__device__ __forceinline__ u64 target_of(double u, u64 mass) {
    const u64 r = u > 0.0 ? (u < 1.0 ? (u64)(u * 18446744073709551616.0) : ~0ull) : 0;
    return __umul64hi(r, mass);
}

__device__ __forceinline__ u64 need_of(double share, u64 total) {  // at least 1, at most all
    const u64 need = (u64)ceil(share * (double)total);
    return need < 1 ? 1 : need > total ? total : need;
}

// ---- rows for one workgroup -----------------------------------------------------

constexpr int kRanked = 128;  // as many keys are ranked at once

template <int N>
struct RowShared {
    u64 bins[kBins];   // (later: cumulated masses of the threads' places)
    unsigned ties[N];  // ties before each thread's places
    u64 wave[N / 64];
    unsigned x[3 * (N / 64)];
    u64 list_v[N];  // the members of one bin
    unsigned list_k[N], listed;
    unsigned key;      // what a descent found
    u64 left;
};

// One level of a descent: the bin where the sum of each()'s members from the top
// reaches need (need = 0: share of the whole) -> `at`, and what is still needed
// from it.  each(f) calls f(k, v) for every member's key and what it counts for;
// bin_of(k) >= kBins: not in this level (all of them sum to less than need: so `at`).
template <int N, class Bin, class Each, class Map>
__device__ __forceinline__ void level(RowShared<N> &s, u64 &need, double share, unsigned &at, Each each, Map bin_of) {
    constexpr int kPer = kBins / N;
    Bin *bin = reinterpret_cast<Bin *>(s.bins);
    for (int i = threadIdx.x; i < kBins; i += N) bin[i] = 0;
    __syncthreads();
    if (threadIdx.x == 0) {  // (behind the barrier: what was found and listed last has been read)
        s.listed = 0;
        s.key = kBins;
    }
    each([&](unsigned k, Bin v) {
        const unsigned b = bin_of(k);
        if (b < kBins) atomicAdd(&bin[b], v);
    });
    __syncthreads();
    const int top = kBins - 1 - kPer * (int)threadIdx.x;  // this thread: bins top, top-1, ...
    Bin v[kPer], sum = 0, total;
#pragma unroll
    for (int j = 0; j < kPer; j++) sum += v[j] = bin[top - j];
    u64 before = block_scan<N, Bin>(sum, reinterpret_cast<Bin *>(s.wave), total) - sum;
    if (need == 0) need = need_of(share, total);
    if (before < need && need <= before + sum) {
#pragma unroll
        for (int j = 0; j < kPer; j++) {
            if (before < need && need <= before + v[j]) {
                s.key = top - j;
                s.left = need - before;
            }
            before += v[j];
        }
    }
    __syncthreads();
    at = s.key;
    need = s.left;
}

// The members in bin `at`, one per thread if they fit -> their number (more than
// N: they do not)
template <int N, class Bin, class Each, class Map>
__device__ __forceinline__ unsigned list(RowShared<N> &s, unsigned at, unsigned &mine, u64 &value, Each each, Map bin_of) {
    each([&](unsigned k, Bin v) {
        if (bin_of(k) != at) return;
        const unsigned to = atomicAdd(&s.listed, 1u);
        if (to >= N) return;
        s.list_k[to] = k;
        s.list_v[to] = v;
    });
    __syncthreads();
    const unsigned listed = s.listed;
    if (listed <= N && threadIdx.x < listed) {
        mine = s.list_k[threadIdx.x];
        value = s.list_v[threadIdx.x];
    }
    return listed;
}

// up to kRanked listed members: each one's sum of larger keys against need
template <int N>
__device__ __forceinline__ void rank(RowShared<N> &s, unsigned listed, unsigned mine, u64 need, unsigned &key, u64 &left) {
    if (mine) {
        u64 above = 0, with = 0;
        for (unsigned i = 0; i < listed; i++) {
            const unsigned k = s.list_k[i];
            const u64 w = s.list_v[i];
            above += k > mine ? w : 0;
            with += k >= mine ? w : 0;
        }
        if (above < need && need <= with) {  // (one key; its ties say the same)
            s.key = mine;
            s.left = need - above;
        }
    }
    __syncthreads();
    key = s.key;
    left = s.left;
}

// Descent: the largest key at which the pool's sum from the top reaches need
// (need = 0: share of the whole), and what its ties still have to bring.
// The first level's bins are even steps of the score, `window` down from the best
// at most: that spreads most pools over all of them, while the keys' own leading
// bits put a normal distribution into some twenty, and masks into one, where the
// atomics wait for each other (20011 scores: 6 us).  The bin where the sum crosses
// is listed, and ranked if it has at most kRanked members.  Without such a bin, or
// if it does not fit, the levels are 11 bits of the key each, until one does.
template <int N, class Bin, class Each>
__device__ __forceinline__ void descend(RowShared<N> &s, unsigned kmin, unsigned kmax, float window, u64 need, double share,
                                        Each each, unsigned &key, u64 &left) {
    unsigned listed = N + 1, mine = 0, at;
    u64 value = 0;
    const float top = score_of(kmax), range = top - score_of(kmin), width = fminf(range, window), per = kBins / width;
    const float low = range < window ? score_of(kmin) : top - width;  // (the whole range loses no score to a rounding)
    if (kmax - kmin >= kBins && per > 0.0f && per < __builtin_inff()) {
        auto even = [&](unsigned k) {
            const float b = (score_of(k) - low) * per;
            return b >= 0.0f ? b < kBins - 1 ? (unsigned)b : kBins - 1u : (unsigned)kBins;
        };
        u64 rest = need;
        level<N, Bin>(s, rest, share, at, each, even);
        if (at < kBins) listed = list<N, Bin>(s, at, mine, value, each, even);
        if (listed <= kRanked) return rank(s, listed, mine, rest, key, left);
        if (listed <= N) {
            need = rest;
            kmin = mine ? mine : 0xffffffffu;
            kmax = mine;
            unsigned some = 0;
            block_extent<N>(kmin, kmax, some, s.x);
        }
    }
    int shift = 0;
    while (((kmax - kmin) >> shift) >= kBins) shift++;
    unsigned lo = kmin, bins = kBins;
    auto listed_ones = [&](auto f) {
        if (mine) f(mine, (Bin)value);
    };
    for (;;) {
        auto bits = [&](unsigned k) { return k < lo || ((k - lo) >> shift) >= bins ? (unsigned)kBins : (k - lo) >> shift; };
        if (listed > N) level<N, Bin>(s, need, share, at, each, bits);
        else level<N, Bin>(s, need, share, at, listed_ones, bits);
        if (shift && listed > N) {
            listed = list<N, Bin>(s, at, mine, value, each, bits);
            if (listed <= kRanked) return rank(s, listed, mine, need, key, left);
        }
        lo += at << shift;
        if (shift == 0) break;
        bins = shift > kBinBits ? kBins : 1u << shift;
        shift = shift > kBinBits ? shift - kBinBits : 0;
    }
    key = lo;
    left = need;
}

// Scores that a descent of counts sets apart: those whose weights are above e^-128,
// mostly all.  (What masks leave lies far below.)
__device__ __forceinline__ float count_window(const SampleArgs &a) { return (float)(128.0 * a.temperature); }

// A row's kept places from its n keys in s_key (N K of them in place order, 0:
// absent), and the draws.  Thread t has the `own` <= K neighbouring ones from
// t own on (as few as hold them all), keys and masses in registers.  top_k: still to be applied (0: no).  s_place: the
// keys' places, where the keys are not all of the row's (NULL: their order).
template <int N, int K>
__device__ __forceinline__ void finish_row(const SampleArgs &a, int row, RowShared<N> &s, const unsigned *s_key,
                                           const unsigned short *s_place, int own, unsigned kmin, unsigned kmax,
                                           unsigned count, int top_k) {
    const int tid = threadIdx.x;
    unsigned key[K];
#pragma unroll
    for (int j = 0; j < K; j++) key[j] = j < own ? s_key[tid * own + j] : 0;
    const Weigh wg{score_of(kmax), 1.0 / a.temperature, ldexp(1.0, a.shift)};
    u64 mass[K];
    unsigned low = 0;  // places under min_p
#pragma unroll
    for (int j = 0; j < K; j++) {
        mass[j] = 0;
        if (j >= own) continue;
        const double w = key[j] ? wg.weight(key[j]) : 0.0;
        mass[j] = wg.mass(w);
        low |= (unsigned)(w < a.min_p) << j;
    }
    unsigned thr = 0;   // places with a larger key are kept,
    u64 quota = ~0ull;  // and this many of those with this key
    if (top_k == 1) {
        thr = kmax;
        quota = 1;
    } else if (top_k > 0 && (unsigned)top_k < count)
        descend<N, unsigned>(s, kmin, kmax, count_window(a), (u64)top_k, 0.0,
            [&](auto f) {
#pragma unroll
                for (int j = 0; j < K; j++)
                    if (key[j]) f(key[j], 1u);
            },
            thr, quota);
    if (a.top_p < 1.0) {
        const unsigned thr_k = thr;
        const u64 quota_k = quota;
        u64 left;
        // (a mass is a multiple of 2^-51 at most: a place 37 temperatures below the best has none)
        descend<N, u64>(s, kmin, kmax, (float)(37.0 * a.temperature), 0, a.top_p,
            [&](auto f) {
#pragma unroll
                for (int j = 0; j < K; j++)
                    if (key[j] > thr_k) f(key[j], mass[j]);
                if (tid == 0 && thr_k) f(thr_k, quota_k * wg.mass(wg.weight(thr_k)));  // the ties top_k keeps
            },
            thr, left);
        const u64 each = wg.mass(wg.weight(thr));
        quota = (left + each - 1) / (each ? each : 1);
    }

    // what is kept, in place order
    unsigned ties = 0;
    if (thr) {
#pragma unroll
        for (int j = 0; j < K; j++) ties += key[j] == thr;
        unsigned every;
        ties = block_scan<N, unsigned>(ties, s.x, every) - ties;
    }
    const unsigned ties_before = ties;
    u64 sum = 0;
    unsigned kept = 0;
#pragma unroll
    for (int j = 0; j < K; j++) {
        const bool tie = key[j] == thr;
        const bool in = key[j] && key[j] >= thr && !(tie && ties >= quota) && !(low >> j & 1);
        ties += tie;
        kept += in;
        sum += in ? mass[j] : 0;
    }
    unsigned kept_all;
    u64 all;
    block_scan2<N, u64, unsigned>(sum, kept, s.wave, s.x, all, kept_all);
    s.bins[tid] = sum;
    s.ties[tid] = ties_before;
    __syncthreads();
    if (a.kept && tid == 0) a.kept[row] = (int)kept_all;
    for (int j = tid; j < a.S; j += N) {
        const u64 target = target_of(a.u[row * a.u_ld + j], all);
        int at = 0;  // the first thread whose cumulated mass passes the target
#pragma unroll
        for (int d = N / 2; d; d >>= 1) at += s.bins[at + d - 1] > target ? 0 : d;
        u64 c = at ? s.bins[at - 1] : 0;
        unsigned tie = s.ties[at];
        int found = -1;
#pragma unroll
        for (int i = 0; i < K; i++) {
            if (i >= own) break;
            const unsigned k = s_key[at * own + i];
            if (found >= 0 || !k || k < thr || (k == thr && tie++ >= quota)) continue;
            const double w = wg.weight(k);
            if (w < a.min_p) continue;
            c += wg.mass(w);
            if (c > target) found = at * own + i;
        }
        a.index[row * a.index_ld + j] = found >= 0 && s_place ? s_place[found] : found;
    }
}

// nothing to draw from
template <int N>
__device__ __forceinline__ void empty_row(const SampleArgs &a, int row) {
    for (int j = threadIdx.x; j < a.S; j += N) a.index[row * a.index_ld + j] = -1;
    if (a.kept && threadIdx.x == 0) a.kept[row] = 0;
}

__device__ __forceinline__ int row_length(const SampleArgs &a, int row) {
    const int n = a.lens ? a.lens[row] : a.V;
    return n < 0 ? 0 : n > a.V ? a.V : n;
}

template <int N, int K>
__global__ __launch_bounds__(N) void sample_row_kernel(SampleArgs a) {
    __shared__ RowShared<N> s;
    __shared__ unsigned s_key[N * K];
    const int row = blockIdx.x, tid = threadIdx.x, n = row_length(a, row);
    // neighbouring lanes load neighbouring places; the keys change owners in LDS
    unsigned key[K];
    unsigned kmin = 0xffffffffu, kmax = 0, count = 0;
    const int own = (n + N - 1) / N;
    load_keys<K>(a, row * a.ld, n, key, [&](int j) { return j * N + tid; }, own);
#pragma unroll
    for (int j = 0; j < K; j++) {
        s_key[j * N + tid] = key[j];
        extend(key[j], kmin, kmax, count);
    }
    block_extent<N>(kmin, kmax, count, s.x);
    if (count == 0) return empty_row<N>(a, row);
    finish_row<N, K>(a, row, s, s_key, nullptr, own, kmin, kmax, count, a.temperature == 0.0 ? 1 : a.top_k);
}

// ---- longer rows of which top_k keeps few ----------------------------------------
//
// One workgroup: the row's keys in registers, K a thread, for top_k's descent;
// what it keeps, at most kTrimKept, moves into LDS in place order, and all that
// needs weights runs on that.

constexpr int kTrimThreads = 1024, kTrimOwn = 8, kTrimKept = kTrimThreads * kTrimOwn;

__device__ __forceinline__ unsigned below(u64 lanes) {  // how many of them lie below this one
    return __builtin_amdgcn_mbcnt_hi((unsigned)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)lanes, 0));
}

template <int K>
__global__ __launch_bounds__(kTrimThreads) void sample_trim_kernel(SampleArgs a) {
    constexpr int N = kTrimThreads, kWaves = N / 64;
    __shared__ RowShared<N> s;
    __shared__ unsigned s_key[kTrimKept];
    __shared__ unsigned short s_place[kTrimKept];
    __shared__ unsigned s_above[K * kWaves], s_tied[K * kWaves];  // of 64 neighbouring places, then before them
    const int row = blockIdx.x, tid = threadIdx.x, n = row_length(a, row);
    unsigned key[K];
    unsigned kmin = 0xffffffffu, kmax = 0, count = 0;
    const int steps = (n + N - 1) / N;
    load_keys<K>(a, row * a.ld, n, key, [&](int j) { return j * N + tid; }, steps);
#pragma unroll
    for (int j = 0; j < K; j++) extend(key[j], kmin, kmax, count);
    block_extent<N>(kmin, kmax, count, s.x);
    if (count == 0) return empty_row<N>(a, row);
    const int top_k = a.temperature == 0.0 ? 1 : a.top_k;  // 1 .. kTrimKept
    unsigned thr = 0;
    u64 quota = 0;
    if (top_k == 1) {
        thr = kmax;
        quota = 1;
    } else if ((unsigned)top_k < count)
        descend<N, unsigned>(s, kmin, kmax, count_window(a), (u64)top_k, 0.0,
            [&](auto f) {
#pragma unroll
                for (int j = 0; j < K; j++)
                    if (j < steps && key[j]) f(key[j], 1u);
            },
            thr, quota);
    // 64 neighbouring places are a wave's j-th: lane j has their counts, then
    // what lies before them
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    unsigned above = 0, tied = 0;
#pragma unroll
    for (int j = 0; j < K; j++) {
        if (j >= steps) break;
        const unsigned more = __popcll(__ballot(key[j] > thr)), same = thr ? __popcll(__ballot(key[j] == thr)) : 0;
        above = lane == j ? more : above;
        tied = lane == j ? same : tied;
    }
    if (lane < K) {
        s_above[lane * kWaves + wave] = above;
        s_tied[lane * kWaves + wave] = tied;
    }
    for (int i = tid; i < kTrimKept; i += N) s_key[i] = 0;
    __syncthreads();
    const bool mine = tid < K * kWaves;
    above = mine ? s_above[tid] : 0;
    tied = mine ? s_tied[tid] : 0;
    unsigned past_above = above, past_tied = tied, every, ties;
    block_scan2<N, unsigned, unsigned>(past_above, past_tied, s.x, s.x + kWaves, every, ties);
    if (mine) {
        s_above[tid] = past_above - above;
        s_tied[tid] = past_tied - tied;
    }
    __syncthreads();
    above = s_above[(lane & (K - 1)) * kWaves + wave];
    tied = s_tied[(lane & (K - 1)) * kWaves + wave];
    const unsigned some = (unsigned)quota;  // of the ties (at most top_k)
#pragma unroll
    for (int j = 0; j < K; j++) {
        if (j >= steps) break;
        u64 in = __ballot(key[j] > thr);
        const unsigned before = lane_of(tied, j), first = before < some ? before : some;
        if (before < some) {
            const u64 here = __ballot(key[j] == thr);
            in |= (unsigned)__popcll(here) <= some - before ? here : __ballot(key[j] == thr && below(here) < some - before);
        }
        if (in >> lane & 1) {
            const unsigned to = lane_of(above, j) + first + below(in);
            s_key[to] = key[j];
            s_place[to] = (unsigned short)(j * N + tid);
        }
    }
    __syncthreads();
    const int kept = (unsigned)top_k < count ? top_k : (int)count;
    finish_row<N, kTrimOwn>(a, row, s, s_key, s_place, (kept + N - 1) / N, thr ? thr : kmin, kmax, count, 0);
}

// ---- long rows: many workgroups per row ------------------------------------
//
// A row is cut into parts of 64 x 64 x f places, one workgroup each, and the
// same steps run as one launch each; what a step finds is read by the next:
//   extent  : each part's smallest and largest key, its count and its weights' sum
//   level 1 : bins over the row's key range: counts (top_k), masses (top_p)
//   level 2, 3 of top_k, level 2, 3 of top_p : bins over the one bin the
//             descent is in; every workgroup finds that bin itself from the
//             bins of the launch before
//   sums    : mass, places and ties above the threshold, per part and per
//             group of 64 f places
//   draw    : one wave per draw: part, group and place by three searches
// Bins are shared by atomics on integers, so their order does not matter.
//
// The unit of mass is chosen from the row's own sum of weights (to 4 digits, in 32
// bits), not from what its length could bring: a long row of one heavy place and
// many light ones would have units in which the light ones are 0, all of them
// together 2^-12 of the best at 2^26 places.  (1000003 scores, top_k and top_p:
// 63.3 us with the unit from the length, 64.7 with this.)

constexpr int kPartThreads = 512;  // (256: 10 to 30 % slower to 200 parts; 1024: 50 % slower from 2000)
constexpr int kDrawThreads = 256;
constexpr int kGroups = 64;  // groups of 64 f places per part, one per lane of a draw's wave
constexpr int kMostParts = 1024;    // (a draw's workgroup holds their sums in LDS)

enum BinArray { kC1, kM1, kC2, kK2, kC3, kK3, kM2, kM3, kBinArrays };  // K: masses of top_k's levels

// where a descent is: its window of keys [lo, lo + (bins << shift))
struct Descent {
    unsigned lo, bins;
    int shift;
    int on;     // 0: this trim is off
    int done;   // lo is the threshold's key, need what its ties bring
    u64 need;   // still needed from the window
    u64 above;  // mass of the keys above the window (top_k's descent)
};

struct RowState {
    unsigned kmin, kmax, count;
    int shift;     // a weight of 1 is 2^shift units of mass
    unsigned thr;  // set by the sums, as quota
    u64 quota;
    Descent k, p;
};

// (member by member: a copy of the whole struct would go through scratch memory)
__device__ __forceinline__ void copy(Descent &to, const Descent &from) {
    to.lo = from.lo;
    to.bins = from.bins;
    to.shift = from.shift;
    to.on = from.on;
    to.done = from.done;
    to.need = from.need;
    to.above = from.above;
}
__device__ __forceinline__ void copy(RowState &to, const RowState &from) {
    to.kmin = from.kmin;
    to.kmax = from.kmax;
    to.count = from.count;
    to.shift = from.shift;
    to.thr = from.thr;
    to.quota = from.quota;
    copy(to.k, from.k);
    copy(to.p, from.p);
}

struct Split {  // workspace of one row
    int parts, f;
    RowState *state;  // one per launch step
    unsigned *extent;  // [parts][4]: keys, count, sum of weights beside the part's largest (float)
    u64 *bins;         // [kBinArrays][kBins]
    u64 *group_mass;   // [parts][kGroups], places above the threshold
    unsigned *group_ties;
    u64 *part_mass;
    unsigned *part_kept, *part_ties;
};

// A weight beside another to 4 digits, or more than it is where the difference of
// the scores or their `rate` (finite) passes 32 bits.
__device__ __forceinline__ float weight_beside(float score, float best, float rate) {
    return score == best ? 1.0f : __expf(fmaxf(score - best, -3.4028235e38f) * rate);
}

// the unit with which weights of this sum (1 or more; 0: none) stay below 2^62
__device__ __forceinline__ int mass_shift(float sum) {
    const int lg = ((int)(__float_as_uint(sum) >> 23) & 255) - 126;  // sum < 2^lg
    return 62 - lg < 51 ? 62 - lg : 51;
}

enum Step { kExtent, kLevel1, kK2Step, kK3Step, kP2Step, kP3Step, kSums, kSteps };

__host__ __device__ inline int split_f(int V) {
    const int per = kGroups * 64;
    return (V + per * kMostParts - 1) / (per * kMostParts);
}
__host__ __device__ inline int split_parts(int V) { return (V + kGroups * 64 * split_f(V) - 1) / (kGroups * 64 * split_f(V)); }

__host__ __device__ inline size_t split_row_bytes(int parts) {
    size_t n = kSteps * sizeof(RowState) + (size_t)kBinArrays * kBins * 8 + (size_t)parts * (kGroups * 12 + 8 + 24);
    return (n + 255) & ~(size_t)255;
}

__host__ __device__ inline Split split_of(void *ws, int V, int row) {
    Split w;
    w.f = split_f(V);
    w.parts = split_parts(V);
    char *p = static_cast<char *>(ws) + split_row_bytes(w.parts) * row;
    w.bins = reinterpret_cast<u64 *>(p);
    p += (size_t)kBinArrays * kBins * 8;
    w.state = reinterpret_cast<RowState *>(p);
    p += kSteps * sizeof(RowState);
    w.group_mass = reinterpret_cast<u64 *>(p);
    p += (size_t)w.parts * kGroups * 8;
    w.part_mass = reinterpret_cast<u64 *>(p);
    p += (size_t)w.parts * 8;
    w.group_ties = reinterpret_cast<unsigned *>(p);
    p += (size_t)w.parts * kGroups * 4;
    w.part_kept = reinterpret_cast<unsigned *>(p);
    p += (size_t)w.parts * 4;
    w.part_ties = reinterpret_cast<unsigned *>(p);
    p += (size_t)w.parts * 4;
    w.extent = reinterpret_cast<unsigned *>(p);
    return w;
}

struct SplitShared {
    u64 bins[2 * kBins];
    u64 wave[2][kPartThreads / 64];
    u64 found_before, found_other;
    int found_bin;
};

// A thread's share of the bins of a level, loaded before the row's state is
// known: counts or masses `v`, and the masses `o` beside top_k's counts.
constexpr int kPer = kBins / kPartThreads;
struct Bins {
    u64 v[kPer], o[kPer];
    __device__ __forceinline__ void load(const u64 *bin, const u64 *other) {
        const int top = kBins - 1 - (int)threadIdx.x * kPer;  // bins top, top-1, ... (unused ones are 0)
#pragma unroll
        for (int j = 0; j < kPer; j++) {
            v[j] = bin[top - j];
            o[j] = other ? other[top - j] : 0;
        }
    }
};

// The bin, from the top, where the running sum of b.v reaches need (share >= 0:
// that share of the whole sum), and the sums of b.v and b.o before it.
__device__ __forceinline__ void find_bin(SplitShared &s, const Bins &b, double share, int &at, u64 &need, u64 &before_out,
                                         u64 &other_before) {
    u64 sum = 0, osum = 0;
#pragma unroll
    for (int j = 0; j < kPer; j++) {
        sum += b.v[j];
        osum += b.o[j];
    }
    u64 upto = sum, oupto = osum, total, ototal;
    block_scan2<kPartThreads, u64, u64>(upto, oupto, s.wave[0], s.wave[1], total, ototal);
    u64 before = upto - sum, obefore = oupto - osum;
    if (share >= 0.0) need = need_of(share, total);
    if (before < need && need <= upto) {
#pragma unroll
        for (int j = 0; j < kPer; j++) {
            if (before < need && need <= before + b.v[j]) {
                s.found_bin = kBins - 1 - (int)threadIdx.x * kPer - j;
                s.found_before = before;
                s.found_other = obefore;
            }
            before += b.v[j];
            obefore += b.o[j];
        }
    }
    __syncthreads();
    at = s.found_bin;
    before_out = s.found_before;
    other_before = s.found_other;
}

// one level down, into bin `at`
__device__ __forceinline__ void into_bin(Descent &d, int at, u64 before, u64 above) {
    d.lo += (unsigned)at << d.shift;
    d.need -= before;
    d.above += above;
    d.done = d.shift == 0;
    d.bins = d.shift > kBinBits ? kBins : 1u << d.shift;
    d.shift = d.shift > kBinBits ? d.shift - kBinBits : 0;
}

// A thread's places of a part: wave w has the groups w, w + 8, ... (64 f
// places each), one place of 64 neighbouring ones per lane.  All loads of a round are
// issued before the first is used.
constexpr int kPartKeys = kGroups * 64 / kPartThreads;
struct PartKeys {
    const SampleArgs &a;
    long long base;
    int i0, n, f;
    unsigned key[kPartKeys];
    __device__ __forceinline__ int place(int j, int jj) const {
        return i0 + ((j * (kPartThreads / 64) + ((int)threadIdx.x >> 6)) * f + jj) * 64 + ((int)threadIdx.x & 63);
    }
    __device__ __forceinline__ void start(int jj) {
        load_raw<kPartKeys>(a, base, n, key, [&](int j) { return place(j, jj); });
    }
    __device__ __forceinline__ void finish(int jj) {
        to_keys<kPartKeys>(a, n, key, [&](int j) { return place(j, jj); });
    }
    __device__ __forceinline__ void load(int jj) {  // every round after the first
        start(jj);
        finish(jj);
    }
};

// The part's keys inside a descent's window -> the row's bins, through LDS:
// counts and / or masses.
__device__ __forceinline__ void fill_bins(SplitShared &s, PartKeys &keys, int f, const Weigh &wg, unsigned lo,
                                          int shift, unsigned bins, u64 *counts, u64 *masses) {
    u64 *s_c = s.bins, *s_m = s.bins + kBins;
    for (int i = threadIdx.x; i < (int)bins; i += kPartThreads) s_c[i] = s_m[i] = 0;
    __syncthreads();
    for (int jj = 0; jj < f; jj++) {
        if (jj) keys.load(jj);
#pragma unroll
        for (int j = 0; j < kPartKeys; j++) {
            const unsigned k = keys.key[j];
            if (!k || k < lo || ((k - lo) >> shift) >= bins) continue;
            const unsigned b = (k - lo) >> shift;
            if (counts) atomicAdd(&s_c[b], 1ull);
            if (masses) atomicAdd(&s_m[b], wg.mass(wg.weight(k)));
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < (int)bins; i += kPartThreads) {
        if (counts && s_c[i]) atomicAdd(&counts[i], s_c[i]);
        if (masses && s_m[i]) atomicAdd(&masses[i], s_m[i]);
    }
}

// sum over a workgroup's threads, in each of them, always in the same order
__device__ __forceinline__ float block_sum(float v, float *s_wave) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s_wave[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int k = 0; k < kPartThreads / 64; k++) v += s_wave[k];
    return v;
}

template <int STEP>
__global__ __launch_bounds__(kPartThreads) void sample_step_kernel(SampleArgs a) {
    __shared__ SplitShared s;
    const int all = split_parts(a.V);
    const int row = blockIdx.x / all, part = blockIdx.x - row * all, tid = threadIdx.x;
    const Split w = split_of(a.ws, a.V, row);
    const int n = row_length(a, row);
    const int size = kGroups * 64 * w.f;
    const long long base = row * a.ld;
    const bool use_k = a.top_k > 0 || a.temperature == 0.0, use_p = a.top_p < 1.0;  // (the launches that run)
    const float rate32 = (float)fmin(1.0 / a.temperature, 3.4028235e38);
    PartKeys keys{a, base, part * size, n, w.f, {}};
    keys.start(0);

    if constexpr (STEP == kExtent) {
        keys.finish(0);
        const int words = kBinArrays * kBins;
        if (use_k || use_p)
            for (int i = part * kPartThreads + tid; i < words; i += w.parts * kPartThreads) w.bins[i] = 0;
        unsigned lo = 0xffffffffu, hi = 0, c = 0;
        float best = 0.0f, sum = 0.0f;  // of this thread's weights, beside the best so far
        for (int jj = 0; jj < w.f; jj++) {
            if (jj) keys.load(jj);
#pragma unroll
            for (int j = 0; j < kPartKeys; j++) extend(keys.key[j], lo, hi, c);
            if (!hi) continue;
            if (sum > 0.0f) sum *= weight_beside(best, score_of(hi), rate32);
            best = score_of(hi);
#pragma unroll
            for (int j = 0; j < kPartKeys; j++)
                sum += keys.key[j] ? weight_beside(score_of(keys.key[j]), best, rate32) : 0.0f;
        }
        block_extent<kPartThreads>(lo, hi, c, reinterpret_cast<unsigned *>(s.bins));
        if (sum > 0.0f) sum *= weight_beside(best, score_of(hi), rate32);
        sum = block_sum(sum, reinterpret_cast<float *>(s.wave));
        if (tid == 0) {
            w.extent[part * 4] = lo;
            w.extent[part * 4 + 1] = hi;
            w.extent[part * 4 + 2] = c;
            w.extent[part * 4 + 3] = __float_as_uint(sum);
        }
        return;
    }

    u64 *C1 = w.bins + kC1 * kBins, *M1 = w.bins + kM1 * kBins, *C2 = w.bins + kC2 * kBins, *K2 = w.bins + kK2 * kBins;
    u64 *C3 = w.bins + kC3 * kBins, *K3 = w.bins + kK3 * kBins, *M2 = w.bins + kM2 * kBins, *M3 = w.bins + kM3 * kBins;
    Bins bins, bins3;  // of the level before; top_k's last one
    if (STEP == kK2Step) bins.load(C1, use_p ? M1 : nullptr);
    if (STEP == kK3Step) bins.load(C2, use_p ? K2 : nullptr);
    if (STEP == kP2Step) bins.load(M1, nullptr);
    if (STEP == kP3Step) bins.load(M2, nullptr);
    if (STEP == kSums && use_p) bins.load(M3, nullptr);
    if ((STEP == kP2Step || (STEP == kSums && !use_p)) && use_k) bins3.load(C3, use_p ? K3 : nullptr);
    RowState st;
    const int before_sums = use_p ? kP3Step : use_k ? kK3Step : kLevel1;
    if (STEP == kLevel1 || (STEP == kSums && before_sums == kLevel1)) {  // no trim: the sums are the second step
        unsigned lo = 0xffffffffu, hi = 0, c = 0;
        constexpr int kShare = kMostParts / kPartThreads;
        unsigned top[kShare];
        float sums[kShare], sum = 0.0f;
#pragma unroll
        for (int i = 0; i < kShare; i++) {
            const int k = i * kPartThreads + tid;
            const bool in = k < w.parts;
            const unsigned l = in ? w.extent[k * 4] : 0xffffffffu;
            top[i] = in ? w.extent[k * 4 + 1] : 0;
            sums[i] = in ? __uint_as_float(w.extent[k * 4 + 3]) : 0.0f;
            lo = l < lo ? l : lo;
            hi = top[i] > hi ? top[i] : hi;
            c += in ? w.extent[k * 4 + 2] : 0;
        }
        block_extent<kPartThreads>(lo, hi, c, reinterpret_cast<unsigned *>(s.bins));
#pragma unroll
        for (int i = 0; i < kShare; i++)
            if (top[i]) sum += sums[i] * weight_beside(score_of(top[i]), score_of(hi), rate32);
        sum = block_sum(sum, reinterpret_cast<float *>(s.wave));
        __syncthreads();
        st.shift = mass_shift(sum);
        st.thr = 0;
        st.quota = 0;
        st.k.done = st.p.done = 0;
        st.k.above = st.p.above = st.p.need = 0;
        st.kmin = lo;
        st.kmax = hi;
        st.count = c;
        const int top_k = a.temperature == 0.0 ? 1 : a.top_k;
        st.k.on = use_k && (unsigned)top_k < c;
        st.k.need = top_k;
        st.p.on = use_p && c > 0;
        int shift = 0;
        while (c && ((hi - lo) >> shift) >= kBins) shift++;
        st.k.lo = st.p.lo = lo;
        st.k.bins = st.p.bins = kBins;
        st.k.shift = st.p.shift = shift;
    } else {
        constexpr int kBefore = STEP == kK2Step ? kLevel1 : STEP == kK3Step ? kK2Step : STEP == kP3Step ? kP2Step : -1;
        copy(st, w.state[STEP == kP2Step ? (use_k ? kK3Step : kLevel1) : STEP == kSums ? before_sums : kBefore]);
    }
    const Weigh wg{score_of(st.kmax), 1.0 / a.temperature, ldexp(1.0, st.shift)};
    auto down = [&](Descent &d, const Bins &b, double share) {
        int at;
        u64 before, above;
        find_bin(s, b, share, at, d.need, before, above);
        into_bin(d, at, before, above);
    };
    u64 *counts = nullptr, *masses = nullptr;  // of the window of st.k (of st.p: P2 and P3)
    if (STEP == kLevel1) {
        counts = st.k.on ? C1 : nullptr;
        masses = st.p.on ? M1 : nullptr;
    }
    if (STEP == kK2Step && st.k.on) {
        down(st.k, bins, -1.0);
        counts = C2;
        masses = st.p.on ? K2 : nullptr;
    }
    if (STEP == kK3Step && st.k.on && !st.k.done) {
        down(st.k, bins, -1.0);
        counts = C3;
        masses = st.p.on ? K3 : nullptr;
    }
    if ((STEP == kP2Step || (STEP == kSums && !use_p)) && st.k.on && !st.k.done)
        down(st.k, bins3, -1.0);
    if (STEP == kP2Step && st.p.on) {
        double share = a.top_p;
        if (st.k.on) {  // of what top_k keeps: every key above its threshold, and its share of the ties
            const u64 total = st.k.above + st.k.need * wg.mass(wg.weight(st.k.lo));
            st.p.need = need_of(a.top_p, total);
            share = -1.0;
        }
        down(st.p, bins, share);
        masses = M2;
    }
    if (STEP == kP3Step && st.p.on && !st.p.done) {
        down(st.p, bins, -1.0);
        masses = M3;
    }
    if (STEP == kSums && st.p.on && !st.p.done) down(st.p, bins, -1.0);
    keys.finish(0);
    if constexpr (STEP != kSums) {
        if (part == 0 && tid == 0) copy(w.state[STEP], st);
        constexpr bool kOfP = STEP == kP2Step || STEP == kP3Step;
        if ((counts || masses) && !(kOfP ? st.p.done : st.k.done))
            fill_bins(s, keys, w.f, wg, kOfP ? st.p.lo : st.k.lo, kOfP ? st.p.shift : st.k.shift,
                      kOfP ? st.p.bins : st.k.bins, counts, masses);
    } else {
        st.thr = 0;
        st.quota = ~0ull;
        u64 each = 0;
        if (st.p.on || st.k.on) {
            st.thr = st.p.on ? st.p.lo : st.k.lo;
            const double wt = wg.weight(st.thr);
            each = wg.mass(wt);
            st.quota = st.p.on ? (st.p.need + each - 1) / (each ? each : 1) : st.k.need;
            if (wt < a.min_p) st.quota = 0;
        }
        if (part == 0 && tid == 0) copy(w.state[STEP], st);
        const int lane = tid & 63, wave = tid >> 6;
        u64 mass[kPartKeys], part_mass = 0;
        unsigned ties[kPartKeys], part_kept = 0, part_ties = 0;
#pragma unroll
        for (int j = 0; j < kPartKeys; j++) mass[j] = ties[j] = 0;
        for (int jj = 0; jj < w.f; jj++) {
            if (jj) keys.load(jj);
#pragma unroll
            for (int j = 0; j < kPartKeys; j++) {
                const unsigned k = keys.key[j];
                ties[j] += __popcll(__ballot(k && k == st.thr));
                const double wt = wg.weight(k);
                const bool in = k > st.thr && wt >= a.min_p;
                mass[j] += in ? wg.mass(wt) : 0;
                part_kept += __popcll(__ballot(in));
            }
        }
#pragma unroll
        for (int j = 0; j < kPartKeys; j++) {
            const u64 m = wave_sum(mass[j]);
            if (lane == 0) {
                w.group_mass[part * kGroups + j * (kPartThreads / 64) + wave] = m;
                w.group_ties[part * kGroups + j * (kPartThreads / 64) + wave] = ties[j];
            }
            part_mass += m;
            part_ties += ties[j];
        }
        unsigned *x = reinterpret_cast<unsigned *>(s.bins);
        constexpr int kWaves = kPartThreads / 64;
        if (lane == 0) {
            s.wave[0][wave] = part_mass;
            x[wave] = part_kept;
            x[kWaves + wave] = part_ties;
        }
        __syncthreads();
        if (tid == 0) {
            for (int k = 1; k < kWaves; k++) {
                part_mass += s.wave[0][k];
                part_kept += x[k];
                part_ties += x[kWaves + k];
            }
            w.part_mass[part] = part_mass;
            w.part_kept[part] = part_kept;
            w.part_ties[part] = part_ties;
        }
    }
}

// One wave's draw inside a group: its lane's key, the ties and the mass before
// the group -> the lane of the place, -1 if the target lies behind; `sum` and
// `before` move past the group.
__device__ __forceinline__ int draw_lane(unsigned k, unsigned thr, u64 quota, const Weigh &wg, double min_p, u64 target,
                                         u64 &sum, u64 &before) {
    const bool tie = k && k == thr;
    const u64 tied = __ballot(tie);
    u64 q = 0;
    if (k > thr || (tie && before + __popcll(tied & ((1ull << (threadIdx.x & 63)) - 1)) < quota)) {
        const double w = wg.weight(k);
        if (w >= min_p) q = wg.mass(w);
    }
    before += __popcll(tied);
    const u64 c = sum + wave_scan(q);
    const u64 hit = __ballot(c > target);
    sum = lane_of(c, 63);
    return __ffsll((long long)hit) - 1;
}

__global__ __launch_bounds__(kDrawThreads) void sample_draw_kernel(SampleArgs a, int chunks, int draws) {
    __shared__ u64 s_mass[kMostParts];       // cumulated kept mass, by part
    __shared__ unsigned s_ties[kMostParts];  // ties before each part
    __shared__ u64 s_wave[2][kDrawThreads / 64];
    const int row = blockIdx.x / chunks, chunk = blockIdx.x - row * chunks, tid = threadIdx.x;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Split w = split_of(a.ws, a.V, row);
    const RowState &st = w.state[kSums];
    const unsigned thr = st.thr, count = st.count;
    const u64 quota = st.quota;
    const Weigh wg{score_of(st.kmax), 1.0 / a.temperature, ldexp(1.0, st.shift)};
    const u64 each = thr ? wg.mass(wg.weight(thr)) : 0;
    const int n = row_length(a, row);
    // cumulated by part: mass above the threshold, and ties, of which the first
    // `quota` are kept
    u64 total;
    {
        constexpr int kPer = kMostParts / kDrawThreads;  // parts tid*kPer ..
        u64 mass[kPer], sum = 0, counts = 0;
        unsigned ties[kPer];
#pragma unroll
        for (int j = 0; j < kPer; j++) {
            const int p = tid * kPer + j;
            const bool in = p < w.parts;
            mass[j] = in ? w.part_mass[p] : 0;
            ties[j] = in ? w.part_ties[p] : 0;
            sum += mass[j];
            counts += ((u64)ties[j] << 32) + (in ? w.part_kept[p] : 0);  // (both below 2^27)
        }
        u64 upto = sum, cupto = counts, every;
        block_scan2<kDrawThreads, u64, u64>(upto, cupto, s_wave[0], s_wave[1], total, every);
        upto -= sum;
        u64 before = (cupto - counts) >> 32;
#pragma unroll
        for (int j = 0; j < kPer; j++) {
            s_ties[tid * kPer + j] = (unsigned)before;
            upto += mass[j];
            before += ties[j];
            s_mass[tid * kPer + j] = upto + (before < quota ? before : quota) * each;
        }
        const u64 kept = (every >> 32) < quota ? every >> 32 : quota;
        total += kept * each;
        if (a.kept && chunk == 0 && tid == 0) a.kept[row] = (int)((every & 0xffffffffu) + kept);
    }
    __syncthreads();
    const long long base = row * a.ld;
    const int size = kGroups * 64 * w.f;
    for (int d = 0; d < draws; d++) {
        const long long j = ((long long)chunk * draws + d) * (kDrawThreads / 64) + wave;
        if (j >= a.S) break;
        int found = -1;
        if (count) {
            const double u = a.u[row * a.u_ld + j];
            const u64 target = target_of(u, total);
            // part: 16 of them per lane, then one of those
            const int l16 = __ffsll((long long)__ballot(s_mass[lane * 16 + 15] > target)) - 1;
            const int part = l16 * 16 + __ffsll((long long)__ballot(lane < 16 && s_mass[l16 * 16 + (lane & 15)] > target)) - 1;
            u64 sum = part ? s_mass[part - 1] : 0;
            // group
            const unsigned ties = w.group_ties[part * kGroups + lane], ties0 = s_ties[part];
            const u64 mass = wave_scan(w.group_mass[part * kGroups + lane]), past = ties0 + wave_scan(ties);
            const u64 upto = sum + mass + ((past < quota ? past : quota) - (ties0 < quota ? ties0 : quota)) * each;
            const int g = __builtin_amdgcn_readfirstlane(__ffsll((long long)__ballot(upto > target)) - 1);
            if (g > 0) sum = lane_of(upto, g - 1);
            u64 before = lane_of(past - ties, g);
            // place
            for (int f = 0; f < w.f && found < 0; f++) {
                const int i = part * size + (g * w.f + f) * 64 + lane;
                unsigned key[1];
                load_keys<1>(a, base, n, key, [&](int) { return i; });
                const unsigned k = key[0];
                const int at = draw_lane(k, thr, quota, wg, a.min_p, target, sum, before);
                if (at >= 0) found = part * size + (g * w.f + f) * 64 + at;
            }
        }
        if (lane == 0) a.index[row * a.index_ld + j] = found;
    }
}

template <int STEP>
void launch_step(const SampleArgs &a, hipStream_t s) {
    hipLaunchKernelGGL((sample_step_kernel<STEP>), dim3((unsigned)a.B * split_parts(a.V)), dim3(kPartThreads), 0, s, a);
}

}  // namespace

// Rows of up to kRowScores scores have one workgroup, whose registers hold them
// all the way; up to kTrimScores, if top_k keeps few, one that trims them first.
// The rest are cut over many, at most kSplitRows rows at a time (their workspace);
// a grid of 1024 threads a row has at most kGridRows (fewer than 2^32 threads).
constexpr int kRowScores = 8192, kTrimScores = 32768, kSplitRows = 512, kGridRows = 1 << 21;

// (one row of 20011, top_k 2001 alone: 128 draws 25 us trimmed and 32 split, 4096
// draws 31 and 34, with top_k 6670 43 and 34, with top_p too 35 and 50; 16 rows of
// 32768, 4096 draws, top_k 3276: 42 and 64)
// (Rows of one workgroup make all their draws there, however many: 2^20 of them take
// 1.4 ms from 960 scores and 4.3 ms from 8192, where 8193 scores, split, take 0.4.)
static bool trim(const SampleArgs &a) {
    const bool few = a.temperature == 0.0 || (a.top_k > 0 && a.top_k <= kTrimKept);
    const bool light = a.V <= kTrimScores / 2 || a.S <= 1024 || a.B >= 8 || a.top_p < 1.0 || a.temperature == 0.0;
    return few && light && a.V <= kTrimScores;
}
static bool split(const SampleArgs &a) { return a.V > kRowScores && !trim(a); }

SamplePlan sample_plan(const SampleArgs &a) {
    SamplePlan p{0};
    if (split(a)) p.ws_bytes = split_row_bytes(split_parts(a.V)) * (a.B < kSplitRows ? a.B : kSplitRows);
    return p;
}

template <int N, int K>
static void launch_row(const SampleArgs &a, hipStream_t s) {
    hipLaunchKernelGGL((sample_row_kernel<N, K>), dim3((unsigned)a.B), dim3(N), 0, s, a);
}

static void launch_split(const SampleArgs &a, hipStream_t s) {
    const bool use_k = a.top_k > 0 || a.temperature == 0.0, use_p = a.top_p < 1.0;
    launch_step<kExtent>(a, s);
    if (use_k || use_p) launch_step<kLevel1>(a, s);
    if (use_k) {
        launch_step<kK2Step>(a, s);
        launch_step<kK3Step>(a, s);
    }
    if (use_p) {
        launch_step<kP2Step>(a, s);
        launch_step<kP3Step>(a, s);
    }
    launch_step<kSums>(a, s);
    // draws per wave: one until half of the chip's 8192 waves are taken, 16 at most
    const long long waves = (long long)a.B * a.S;
    // (a grid has fewer than 2^32 threads, so past 2^28 draws more again)
    const int draws = waves <= 4096           ? 1
                      : waves < 16 * 4096     ? (int)((waves + 4095) / 4096)
                      : waves <= 16ll << 24   ? 16
                                              : (int)((waves >> 24) + 1);
    const int per = draws * kDrawThreads / 64, chunks = a.S > per ? (a.S + per - 1) / per : 1;
    hipLaunchKernelGGL(sample_draw_kernel, dim3((unsigned)((long long)a.B * chunks)), dim3(kDrawThreads), 0, s, a,
                       chunks, draws);
}

static void launch_rows(const SampleArgs &a, bool cut, hipStream_t s) {
    if (cut) launch_split(a, s);
    else if (a.V <= 256) launch_row<256, 1>(a, s);
    else if (a.V <= 1024) launch_row<1024, 1>(a, s);
    else if (a.V <= 4096) launch_row<1024, 4>(a, s);
    else if (a.V <= kRowScores) launch_row<1024, 8>(a, s);
    else if (a.V <= kTrimScores / 2) hipLaunchKernelGGL(sample_trim_kernel<16>, dim3((unsigned)a.B), dim3(kTrimThreads), 0, s, a);
    else hipLaunchKernelGGL(sample_trim_kernel<32>, dim3((unsigned)a.B), dim3(kTrimThreads), 0, s, a);
}

void launch_sample(const SampleArgs &a, hipStream_t s) {
    const bool cut = split(a);
    const int most = cut ? kSplitRows : kGridRows;
    const int elem = a.dtype == SC_F32 ? 4 : 2;
    for (int r = 0; r < a.B; r += most) {
        SampleArgs b = a;
        b.B = a.B - r < most ? a.B - r : most;
        b.scores = static_cast<const char *>(a.scores) + r * a.ld * elem;
        if (a.lens) b.lens = a.lens + r;
        b.u = a.u + r * a.u_ld;
        b.index = a.index + r * a.index_ld;
        if (a.kept) b.kept = a.kept + r;
        launch_rows(b, cut, s);
    }
}

}  // namespace sc
