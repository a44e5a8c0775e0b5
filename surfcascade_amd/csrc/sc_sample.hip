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
// One workgroup per row.  The threshold comes from a radix descent of 11 bits
// a pass over the row's own key range (bins hold counts for top_k, masses for
// top_p), then each thread owns a contiguous part of the row, one block scan
// gives every part's first cumulated mass, and a draw is a binary search over
// the parts and a walk through one.
#include <hip/hip_runtime.h>

#include "sc_train.hpp"
#include "surfcascade.h"

namespace sc {

namespace {

typedef unsigned long long u64;
constexpr int kThreads = 1024;
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

__device__ __forceinline__ unsigned load_key(const SampleArgs &a, long long base, int i) {
    if (a.dtype == SC_F32) return key_of(static_cast<const float *>(a.scores)[base + i]);
    if (a.dtype == SC_F16) return key_of((float)static_cast<const _Float16 *>(a.scores)[base + i]);
    return key_of(__uint_as_float((unsigned)static_cast<const unsigned short *>(a.scores)[base + i] << 16));
}

struct Weigh {
    float top;
    double rate;  // 1 / temperature
    double unit;  // 2^shift
    __device__ __forceinline__ double weight(unsigned key) const {
        const float s = score_of(key);
        return s == top ? 1.0 : exp(((double)s - (double)top) * rate);  // (also +inf against +inf)
    }
    __device__ __forceinline__ u64 mass(double w) const { return (u64)rint(w * unit); }
};

template <class V>
__device__ __forceinline__ V wave_scan(V x, int lane) {  // inclusive
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const V o = __shfl_up(x, d, 64);
        if (lane >= d) x += o;
    }
    return x;
}

// inclusive block scan; total in every thread
template <class V>
__device__ __forceinline__ V block_scan(V x, V *s_wave, V &total) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    x = wave_scan(x, lane);
    __syncthreads();
    if (lane == 63) s_wave[wv] = x;
    __syncthreads();
    V before = 0;
    total = 0;
    for (int k = 0; k < kThreads / 64; k++) {
        before += k < wv ? s_wave[k] : 0;
        total += s_wave[k];
    }
    return before + x;
}

struct Found {
    unsigned key;  // the key where the descending sum first reaches `need`
    u64 left;      // what is still needed from the places with that key
};

// Radix descent: the largest key whose descending sum over the pool's bins
// reaches `need`.  fill(lo, shift, bins) adds every pool member whose key lies
// in [lo, lo + (bins << shift)) to s_bin[(key - lo) >> shift]: the whole pool
// first, then the one bin where the sum crosses.
template <class Fill, class Need>
__device__ Found descend(unsigned kmin, unsigned kmax, u64 *s_bin, u64 *s_wave, Found *s_found, Fill fill, Need need_of) {
    int shift = 0;
    while (((kmax - kmin) >> shift) >= kBins) shift++;
    unsigned lo = kmin, bins = kBins;
    u64 need = 0;
    for (bool first = true;; first = false) {
        __syncthreads();
        for (int i = threadIdx.x; i < kBins; i += kThreads) s_bin[i] = 0;
        __syncthreads();
        fill(lo, shift, bins);
        __syncthreads();
        // bins from the top: thread t has bins kBins-1-2t and kBins-2-2t
        const int hi_bin = kBins - 1 - 2 * (int)threadIdx.x;
        const u64 v1 = s_bin[hi_bin], v0 = s_bin[hi_bin - 1];
        u64 total;
        const u64 upto = block_scan<u64>(v1 + v0, s_wave, total);
        if (first) need = need_of(total);
        const u64 before = upto - v1 - v0;
        if (before < need && need <= upto) {
            const bool in_hi = need <= before + v1;
            s_found->key = lo + ((unsigned)(in_hi ? hi_bin : hi_bin - 1) << shift);
            s_found->left = need - before - (in_hi ? 0 : v1);
        }
        __syncthreads();
        const Found f = *s_found;
        if (shift == 0) return f;
        lo = f.key;
        need = f.left;
        bins = shift > kBinBits ? kBins : 1u << shift;
        shift = shift > kBinBits ? shift - kBinBits : 0;
    }
}

__global__ __launch_bounds__(kThreads) void sample_row_kernel(SampleArgs a) {
    __shared__ u64 s_bin[kBins];  // (later: the parts' cumulated masses)
    __shared__ u64 s_wave[kThreads / 64];
    __shared__ unsigned s_min, s_max, s_count;
    __shared__ Found s_found;
    const int row = blockIdx.x, tid = threadIdx.x;
    int n = a.lens ? a.lens[row] : a.V;
    n = n < 0 ? 0 : n > a.V ? a.V : n;
    const long long base = row * a.ld;
    int *index = a.index + row * a.index_ld;

    if (tid == 0) {
        s_min = 0xffffffffu;
        s_max = 0;
        s_count = 0;
    }
    __syncthreads();
    {
        unsigned lo = 0xffffffffu, hi = 0, c = 0;
        for (int i = tid; i < n; i += kThreads) {
            const unsigned k = load_key(a, base, i);
            if (!k) continue;
            lo = k < lo ? k : lo;
            hi = k > hi ? k : hi;
            c++;
        }
        if (c) {
            atomicMin(&s_min, lo);
            atomicMax(&s_max, hi);
            atomicAdd(&s_count, c);
        }
    }
    __syncthreads();
    const unsigned kmin = s_min, kmax = s_max, count = s_count;
    if (count == 0) {  // nothing to draw from
        for (int j = tid; j < a.S; j += kThreads) index[j] = -1;
        if (a.kept && tid == 0) a.kept[row] = 0;
        return;
    }
    const int top_k = a.temperature == 0.0 ? 1 : a.top_k;  // temperature 0: the best place
    const Weigh wg{score_of(kmax), a.temperature == 0.0 ? 0.0 : 1.0 / a.temperature, ldexp(1.0, a.shift)};

    unsigned thr = 0;         // places with a larger key are kept,
    u64 quota = ~0ull;        // and this many of those with this key
    if (top_k > 0 && (unsigned)top_k < count) {
        const Found f = descend(kmin, kmax, s_bin, s_wave, &s_found,
            [&](unsigned lo, int shift, unsigned bins) {
                for (int i = tid; i < n; i += kThreads) {
                    const unsigned k = load_key(a, base, i);
                    if (k && k >= lo && ((k - lo) >> shift) < bins) atomicAdd(&s_bin[(k - lo) >> shift], 1ull);
                }
            },
            [&](u64) { return (u64)top_k; });
        thr = f.key;
        quota = f.left;
    }
    if (a.top_p < 1.0) {
        const unsigned thr_k = thr;
        const u64 quota_k = quota;
        const Found f = descend(kmin, kmax, s_bin, s_wave, &s_found,
            [&](unsigned lo, int shift, unsigned bins) {
                for (int i = tid; i < n; i += kThreads) {
                    const unsigned k = load_key(a, base, i);
                    if (k > thr_k && k >= lo && ((k - lo) >> shift) < bins)
                        atomicAdd(&s_bin[(k - lo) >> shift], wg.mass(wg.weight(k)));
                }
                if (tid == 0 && thr_k && thr_k >= lo && ((thr_k - lo) >> shift) < bins)  // the ties top_k keeps
                    atomicAdd(&s_bin[(thr_k - lo) >> shift], quota_k * wg.mass(wg.weight(thr_k)));
            },
            [&](u64 total) {
                const u64 need = (u64)ceil(a.top_p * (double)total);
                return need < 1 ? 1 : need > total ? total : need;
            });
        const u64 each = wg.mass(wg.weight(f.key));
        thr = f.key;
        quota = (f.left + each - 1) / each;
    }

    // each thread owns places [i0, i1): ties in place order, then masses
    const int per = (n + kThreads - 1) / kThreads;
    const long long first = (long long)tid * per;
    const int i0 = (int)(first < n ? first : n), i1 = (int)(first + per < n ? first + per : n);
    u64 ties = 0;
    if (thr)
        for (int i = i0; i < i1; i++) ties += load_key(a, base, i) == thr;
    u64 total;
    const u64 ties_before = block_scan<u64>(ties, s_wave, total) - ties;
    auto walk = [&](u64 tie, int from, int to, auto visit) {
        for (int i = from; i < to; i++) {
            const unsigned k = load_key(a, base, i);
            if (!k || k < thr || (k == thr && tie++ >= quota)) continue;
            const double w = wg.weight(k);
            if (w < a.min_p) continue;
            if (visit(i, wg.mass(w))) return;
        }
    };
    u64 mass = 0, kept = 0;
    walk(ties_before, i0, i1, [&](int, u64 q) {
        mass += q;
        kept++;
        return false;
    });
    u64 kept_all, mass_all;
    block_scan<u64>(kept, s_wave, kept_all);
    const u64 upto = block_scan<u64>(mass, s_wave, mass_all);
    __syncthreads();
    s_bin[tid] = upto;
    s_bin[kThreads + tid] = ties_before;
    __syncthreads();
    if (a.kept && tid == 0) a.kept[row] = (int)kept_all;
    for (int j = tid; j < a.S; j += kThreads) {
        const double u = a.u[row * a.u_ld + j];
        const u64 r = u > 0.0 ? (u < 1.0 ? (u64)(u * 18446744073709551616.0) : ~0ull) : 0;
        const u64 target = __umul64hi(r, mass_all);  // floor(u * mass), below the mass
        int lo = 0, hi = kThreads - 1;  // the first part whose cumulated mass passes the target
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (s_bin[mid] > target) hi = mid;
            else lo = mid + 1;
        }
        u64 sum = lo ? s_bin[lo - 1] : 0;
        const long long b = (long long)lo * per;
        int found = -1;
        walk(s_bin[kThreads + lo], (int)(b < n ? b : n), (int)(b + per < n ? b + per : n), [&](int i, u64 q) {
            sum += q;
            found = i;
            return sum > target;
        });
        index[j] = found;
    }
}

}  // namespace

SamplePlan sample_plan(const SampleArgs &) { return SamplePlan{0}; }

void launch_sample(const SampleArgs &a, hipStream_t s) {
    if (a.B == 0) return;
    hipLaunchKernelGGL(sample_row_kernel, dim3((unsigned)a.B), dim3(kThreads), 0, s, a);
}

}  // namespace sc
