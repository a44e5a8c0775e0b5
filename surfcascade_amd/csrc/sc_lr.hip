// sc_lr.hip -- gfx950 kernels of the weak learners over a sample matrix
// (LogisticRegression::Predict and its training sums, LogisticRegression.cpp:
// 35-68, over the descriptors ExtractFeatures leaves,
// DenseSURFFeatureExtractor.cpp:88-93), for R rows x M learners x H parameter
// sets:
//   z[r,m,h]   = x[row r, patch m] . w[m,h] + b[m,h]
//   response   : y = alpha * act(z) + beta * residual
//   gradient   : g = alpha * dy * act'(z); dw = sum_r g x, db = sum_r g
//   loss       : L = sum_r c (softplus(z) - t z), g = c (sigmoid(z) - t)
// A (row, patch) descriptor is 128 B (64 B in 16 bits) that feeds 64 flops per
// parameter set (128 with its gradient), so up to 16 sets the matrix' own bytes
// are the bound: each descriptor is read once from memory and everything is done
// on it in registers.  Sums over rows are in 32 bits within a chunk of them (2048
// of a wave at most); the chunks are joined in 64 bits in a fixed order (no
// atomics: the same call gives the same bits).
//
// Up to kNarrowSets sets, the narrow form: one descriptor on LPI = 8 lanes (4 in
// 16 bits), 16 B each, so a wave's load is 8 (16) neighbouring descriptors of one
// row = 1 KB in one piece.  A wave keeps its learners' weights in registers and
// walks rows, LPI of them at a time: the LPI x LPI partial dots are summed by a
// butterfly that also transposes, leaving lane q with row q's dot, so the sigmoid
// runs once per result on full lanes; a gradient spreads g back over the lanes.
// More sets: the matrix cores (below), whose time hardly depends on their number
// up to 16.  The borders, on 8191 x 608: responses of f32 with 5 sets 153 us
// narrow and 205 wide (with 7 275: its stores are not whole 16-B pieces), with 8
// sets 191 and 182; the gradient with 4 sets 150 us narrow, with 5 241 and 206
// wide; the loss with 5 sets 184 and 208 in f32, 155 and 105 in bf16.  (One border
// serves gradients and losses of every type: it costs the f32 loss of 5 sets 24 us.)
//
// Measured (one MI355X; a 2 GiB copy moves 4.9 TB/s there, reads and writes):
//   responses, 16384 x 608, f32, 1 set          221 us, 5.9 TB/s
//   loss and gradient, 16384 x 608, f32, 1 set  219 us, 5.8 TB/s
//   responses, 2001 x 608, f16, 16 sets          60 us, 3.5 TB/s
//   loss and gradient, 8191 x 608, bf16, 16 sets 131 us, 2.5 TB/s (the VALU, 68 %
//     of the cycles: the sigmoid, its loss and the operand splits of 80 M results)
//   gradient, 480 x 11870, bf16, 8 sets, dres   171 us, 4.4 TB/s
#include <hip/hip_runtime.h>

#include <type_traits>

#include "sc_train.hpp"
#include "surfcascade.h"

namespace sc {

namespace {

constexpr int kWaves = 4;  // waves per workgroup
constexpr int kWideWaves = 8;   // ... of the wide form (4: 20 % slower on 16 sets of 608 patches)
// parameter sets per learner up to which the narrow form runs
constexpr int kNarrowSets = 4, kNarrowResponse = 7;
// ... and up to which the wide form of 16-bit samples takes two learners per wave
constexpr int kPairSets = 8;

struct F32 {
    static constexpr int kSize = 4;
};
struct F16 {
    static constexpr int kSize = 2;
};
struct BF16 {
    static constexpr int kSize = 2;
};

// 16 B with the alignment of an element (the sample matrix may start, and its
// rows may lie, at any element)
typedef unsigned uint4_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned uint4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned uint4_v __attribute__((ext_vector_type(4)));
typedef _Float16 half2_v __attribute__((ext_vector_type(2)));

typedef float float4_v __attribute__((ext_vector_type(4)));
typedef float float4_a4 __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ void load4(const float *p, bool on, float *to) {  // (0 where not on)
    float4_v v = {0, 0, 0, 0};
    if (on) v = *reinterpret_cast<const float4_a4 *>(p);
#pragma unroll
    for (int k = 0; k < 4; k++) to[k] = v[k];
}

template <class T>
__device__ __forceinline__ uint4_v load16(const char *p) {
    if constexpr (T::kSize == 4) return *reinterpret_cast<const uint4_a4 *>(p);
    else return *reinterpret_cast<const uint4_a2 *>(p);
}

// the 16 / kSize values of a 16-B piece
template <class T>
__device__ __forceinline__ void unpack(uint4_v v, float *f) {
    if constexpr (T::kSize == 4) {
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = __uint_as_float(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const unsigned u = v[i];
            if constexpr (__is_same(T, BF16)) {
                f[2 * i] = __uint_as_float(u << 16);
                f[2 * i + 1] = __uint_as_float(u & 0xffff0000u);
            } else {
                const half2_v h = __builtin_bit_cast(half2_v, u);
                f[2 * i] = (float)h[0];
                f[2 * i + 1] = (float)h[1];
            }
        }
    }
}

constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kReverse4 = 0x1B, kMirror8 = 0x141;  // DPP controls

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}

// v[u] = this lane's part of row u's sum, over the LPI lanes of an item ->
// lane q's return value is row q's sum.
template <int LPI>
__device__ __forceinline__ float sum_rows(float *v, int q) {
    if constexpr (LPI == 8) {
        const bool hi = q & 4;
#pragma unroll
        for (int i = 0; i < 4; i++) {  // partner 7 - q
            const float send = hi ? v[i] : v[i + 4];
            v[i] = (hi ? v[i + 4] : v[i]) + dpp<kMirror8>(send);
        }
    }
    const bool mid = q & 2, odd = q & 1;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const float send = mid ? v[i] : v[i + 2];
        v[i] = (mid ? v[i + 2] : v[i]) + dpp<kXor2>(send);
    }
    const float send = odd ? v[0] : v[1];
    return (odd ? v[1] : v[0]) + dpp<kXor1>(send);
}

// lane q holds row q's value -> all[u] = row u's, in every lane of the item
template <int LPI>
__device__ __forceinline__ void spread_rows(float v, int q, float *all) {
    float low = v;
    if constexpr (LPI == 8) {
        const float other = dpp<kReverse4>(dpp<kMirror8>(v));  // lane q ^ 4's
        low = (q & 4) ? other : v;
        const float high = (q & 4) ? v : other;
        all[4] = dpp<0x00>(high);
        all[5] = dpp<0x55>(high);
        all[6] = dpp<0xAA>(high);
        all[7] = dpp<0xFF>(high);
    }
    all[0] = dpp<0x00>(low);
    all[1] = dpp<0x55>(low);
    all[2] = dpp<0xAA>(low);
    all[3] = dpp<0xFF>(low);
}

// sum over the LPI lanes of an item, in each of them
template <int LPI>
__device__ __forceinline__ float sum_lanes(float v) {
    v += dpp<kXor1>(v);
    v += dpp<kXor2>(v);
    if constexpr (LPI == 8) v += dpp<kMirror8>(v);
    return v;
}

// (the hardware's reciprocal, good to one unit in the last place: the IEEE
// division is ten instructions)
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __expf(-z)); }

enum Mode { kResponse = 0, kGrad = 1, kLoss = 2 };

// log(1 + e) / e for e in [0, 1]: a polynomial of degree 8 fitted for the least
// relative error (3.0e-8; 3 roundings of 2^-24 as evaluated)
__device__ __forceinline__ float log1p_over(float e) {
    float p = 0.005232677f;
    p = __builtin_fmaf(p, e, -0.029505169f);
    p = __builtin_fmaf(p, e, 0.078225836f);
    p = __builtin_fmaf(p, e, -0.13663235f);
    p = __builtin_fmaf(p, e, 0.19106002f);
    p = __builtin_fmaf(p, e, -0.24842981f);
    p = __builtin_fmaf(p, e, 0.33319098f);
    p = __builtin_fmaf(p, e, -0.49999493f);
    return __builtin_fmaf(p, e, 0.99999994f);
}

// What a row brings to its results' gradients: for the loss its weight on
// either side, pos = c (1 - t) and neg = c t; for a response pos = alpha dy.
// With e = exp(-|z|) and d = 1 / (1 + e) the loss and its slope are
//   c (softplus(z) - t z) = c log(1 + e) + (z >= 0 ? pos : -neg) z
//   c (sigmoid(z) - t)    = d (z >= 0 ? pos - neg e : pos e - neg)
// neither of which takes a difference of nearly equal numbers.  A NaN z is a
// NaN e, and stays one.
template <int MODE>
__device__ __forceinline__ float grad_of(int act, float z, float pos, float neg, float &loss) {
    const float e = __expf(-fabsf(z)), d = __builtin_amdgcn_rcpf(1.0f + e);
    if constexpr (MODE == kLoss) {
        const bool up = z >= 0.0f;
        const float near = up ? pos : -neg, far = up ? -neg : pos;
        loss = __builtin_fmaf((pos + neg) * e, log1p_over(e), __builtin_fmaf(near, z, loss));
        return d * __builtin_fmaf(far, e, near);
    } else {
        return act == SC_ACT_SIGMOID ? pos * e * d * d : pos;
    }
}

template <class T, int H, int MODE>
__global__ __launch_bounds__(64 * kWaves) void lr_kernel(LrArgs a) {
    constexpr int LPI = kDesc * T::kSize / 16;  // lanes per item
    constexpr int EPL = 16 / T::kSize;          // descriptor values per lane
    constexpr int IPW = 64 / LPI;               // items per wave
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int q = lane & (LPI - 1), item = lane / LPI;
    // waves of a workgroup: neighbouring learners of one row range for a
    // response (their stores meet in one line), row ranges of the same
    // learners for a gradient (joined in LDS below)
    const int mt = MODE == kResponse ? blockIdx.x * kWaves + wave : blockIdx.x;
    const int range = MODE == kResponse ? blockIdx.y : blockIdx.y * kWaves + wave;
    const int m = mt * IPW + item;
    const bool learner = m < a.M;
    int p = 0;
    bool present = false;
    if (learner) {
        p = a.patch ? a.patch[m] : m;
        present = (unsigned)p < (unsigned)a.n_patches;
        if (!present) p = 0;
    }
    const unsigned off = (unsigned)(p * kDesc * T::kSize + q * 16);
    float w[H][EPL], bias[H];
#pragma unroll
    for (int h = 0; h < H; h++) {
        const bool on = learner && h < a.H;
        const long long mh = (long long)m * a.H + h;
#pragma unroll
        for (int e = 0; e < EPL; e += 4) load4(a.w + mh * kDesc + q * EPL + e, on, w[h] + e);
        bias[h] = on && a.b ? a.b[mh] : 0.0f;
    }
    float acc[H][EPL], sum_g[H], sum_l[H];
#pragma unroll
    for (int h = 0; h < H; h++) {
        sum_g[h] = sum_l[h] = 0.0f;
#pragma unroll
        for (int e = 0; e < EPL; e++) acc[h][e] = 0.0f;
    }
    const long long r_lo = a.row0 + (long long)range * a.rows_per_wave;
    const int r0 = (int)(r_lo < a.R ? r_lo : a.R);
    const int r1 = (int)(r_lo + a.rows_per_wave < a.R ? r_lo + a.rows_per_wave : a.R);
    const char *x = static_cast<const char *>(a.x);
    for (int r = r0; r < r1; r += LPI) {
        const int rq = r + q;  // the row whose dot this lane will hold
        int idx = -1;
        if (rq < r1) {
            idx = a.rows ? a.rows[rq] : rq;
            if ((unsigned)idx >= (unsigned)a.n) idx = -1;
        }
        float pos = 0.0f, neg = 0.0f;
        if constexpr (MODE == kLoss) {
            if (idx >= 0) {
                const float c = a.weight ? a.weight[idx] : 1.0f, t = a.target[idx];
                pos = c * (1.0f - t);
                neg = c * t;
                if (c == 0.0f) idx = -1;  // a row without weight is not looked at, whatever it holds
            }
        }
        uint4_v xv[LPI];
#pragma unroll
        for (int u = 0; u < LPI; u++) {
            const int iu = __builtin_amdgcn_readlane(idx, u);
            xv[u] = uint4_v{0, 0, 0, 0};
            if (iu >= 0) xv[u] = load16<T>(x + (long long)iu * a.ld * T::kSize + off);
        }
        float g_all[H][LPI];
        float z[H];
        {
            float part[H][LPI];
#pragma unroll
            for (int u = 0; u < LPI; u++) {
                float f[EPL];
                unpack<T>(xv[u], f);
#pragma unroll
                for (int h = 0; h < H; h++) {
                    float s = f[0] * w[h][0];
#pragma unroll
                    for (int e = 1; e < EPL; e++) s = __builtin_fmaf(f[e], w[h][e], s);
                    part[h][u] = s;
                }
            }
#pragma unroll
            for (int h = 0; h < H; h++) z[h] = sum_rows<LPI>(part[h], q) + bias[h];
        }
        if constexpr (MODE == kResponse) {
            if (learner && rq < r1) {
#pragma unroll
                for (int h = 0; h < H; h++) {
                    if (h >= a.H) break;
                    const long long col = (long long)m * a.H + h;
                    float v = 0.0f;  // an absent row or patch has no response
                    if (idx >= 0 && present) v = a.alpha * (a.act == SC_ACT_SIGMOID ? sigmoid(z[h]) : z[h]);
                    if (a.res_kind == SC_RES_ROW) v += a.beta * a.res[(long long)rq * a.res_ld];
                    else if (a.res_kind == SC_RES_FULL) v += a.beta * a.res[(long long)rq * a.res_ld + col];
                    a.y[(long long)rq * a.y_ld + col] = v;
                }
            }
        } else {
#pragma unroll
            for (int h = 0; h < H; h++) {
                float g = 0.0f;
                if constexpr (MODE == kGrad) {
                    if (learner && rq < r1 && h < a.H) {
                        const long long col = (long long)m * a.H + h;
                        const float dy = a.dy[(long long)rq * a.dy_ld + col];
                        pos = a.alpha * dy;
                        if (a.res_kind == SC_RES_FULL) a.dres[(long long)rq * a.dres_ld + col] = a.beta * dy;
                    }
                }
                if (idx >= 0 && present && h < a.H) g = grad_of<MODE>(a.act, z[h], pos, neg, sum_l[h]);
                sum_g[h] += g;
                spread_rows<LPI>(g, q, g_all[h]);
            }
#pragma unroll
            for (int u = 0; u < LPI; u++) {
                float f[EPL];
                unpack<T>(xv[u], f);
#pragma unroll
                for (int h = 0; h < H; h++)
#pragma unroll
                    for (int e = 0; e < EPL; e++) acc[h][e] = __builtin_fmaf(g_all[h][u], f[e], acc[h][e]);
            }
        }
    }
    if constexpr (MODE != kResponse) {
        constexpr int kVals = H * (EPL + 2);
        __shared__ float s_acc[kWaves][kVals][64];
#pragma unroll
        for (int h = 0; h < H; h++) {
#pragma unroll
            for (int e = 0; e < EPL; e++) s_acc[wave][h * (EPL + 2) + e][lane] = acc[h][e];
            s_acc[wave][h * (EPL + 2) + EPL][lane] = sum_lanes<LPI>(sum_g[h]);
            s_acc[wave][h * (EPL + 2) + EPL + 1][lane] = sum_lanes<LPI>(sum_l[h]);
        }
        __syncthreads();
        if (!learner) return;
        for (int v = wave; v < kVals; v += kWaves) {
            float s = s_acc[0][v][lane];
#pragma unroll
            for (int k = 1; k < kWaves; k++) s += s_acc[k][v][lane];
            const int h = v / (EPL + 2), e = v - h * (EPL + 2);
            if (h >= a.H || (e >= EPL && q != 0)) continue;
            if (e < EPL && !present) s = 0.0f;  // (0 * NaN of the patch read in its place)
            const long long mh = (long long)m * a.H + h;
            const int word = e < EPL ? q * EPL + e : kDesc + (e - EPL);
            if (a.part) a.part[((long long)blockIdx.y * a.M * a.H + mh) * kPartWords + word] = s;
            else if (word < kDesc) a.dw[mh * kDesc + word] = s;
            else if (word == kDesc) a.db[mh] = s;
            else if (MODE == kLoss) a.loss[mh] = s;
        }
    }
}

// Wide form, for many parameter sets: a wave owns one learner and 16 of its
// sets and multiplies 16 rows at a time on the matrix cores.  Neighbouring
// waves have the sets of a learner, then the next learner, whose descriptors
// lie in the same lines.
//   z = X W^T : lane (i = lane % 16, q = lane / 16) holds 8 values of row i's
//               descriptor and the same 8 places of set i's weights; any order
//               of the places will do, so each lane keeps what one 16-B load
//               brings.
//   dW = G^T X: z's result is already the operand layout of the second
//               product; X is read again with lane i = descriptor place (its
//               lines are in the vector L1 from the first read).
template <class T>
struct WideRow {  // the 8 values of a lane's row: places 8q..8q+7
    uint4_v a;
    __device__ __forceinline__ void load(const char *p) { a = load16<T>(p); }
    __device__ __forceinline__ void values(float *f) const { unpack<T>(a, f); }
    static __device__ __forceinline__ int place(int q, int four) { return q * 8 + four * 4; }  // the first of four
};
template <>
struct WideRow<F32> {  // places 4q..4q+3 and 16+4q..: each load covers half a line of 16 rows
    uint4_v a, b;
    __device__ __forceinline__ void load(const char *p) {
        a = load16<F32>(p);
        b = load16<F32>(p + 64);
    }
    __device__ __forceinline__ void values(float *f) const {
        unpack<F32>(a, f);
        unpack<F32>(b, f + 4);
    }
    static __device__ __forceinline__ int place(int q, int four) { return four * 16 + q * 4; }
};

// what a wave of the wide form works on
struct WideUnit {
    int m, h0, r0, r1;  // learner, first set, rows
    bool present;       // its patch exists
    const char *x;      // that patch of sample 0 (patch 0 in an absent one's place)
    long long step;     // bytes from sample to sample
    // samples in order, 16 of them within 2^31 bytes: one base per tile and
    // per-lane offsets that stay the same
    bool in_order;
    bool dense;  // ... of dy and dres within 2^31 elements
};

template <class T>
__device__ __forceinline__ void wide_rows(const LrArgs &a, WideUnit &u) {
    u.step = a.ld * T::kSize;
    u.in_order = !a.rows && u.step < (1 << 26);
    u.dense = a.dy_ld < (1 << 26) && a.dres_ld < (1 << 26);
    const long long lo = a.row0 + (long long)blockIdx.y * a.rows_per_wave;
    u.r0 = (int)(lo < a.R ? lo : a.R);
    u.r1 = (int)(lo + a.rows_per_wave < a.R ? lo + a.rows_per_wave : a.R);
}
template <class T>
__device__ __forceinline__ bool wide_unit(const LrArgs &a, int wave, WideUnit &u) {
    const int sets = (a.H + 15) / 16, unit = blockIdx.x * (blockDim.x >> 6) + wave;
    u.m = unit / sets;
    u.h0 = (unit - u.m * sets) * 16;
    if (u.m >= a.M) return false;
    const int p = a.patch ? a.patch[u.m] : u.m;
    u.present = (unsigned)p < (unsigned)a.n_patches;
    u.x = static_cast<const char *>(a.x) + (long long)(u.present ? p : 0) * kDesc * T::kSize;
    wide_rows<T>(a, u);
    return true;
}

// Responses: z^T = W X^T, so that lane i has row i and four neighbouring sets
// (one 16-B store).
template <class T>
__global__ __launch_bounds__(64 * kWideWaves) void lr_wide_response_kernel(LrArgs a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, q = lane >> 4;
    WideUnit u;
    if (!wide_unit<T>(a, wave, u)) return;
    float w[8];
    float4_v bias = {0, 0, 0, 0};
    const long long first = (long long)u.m * a.H + u.h0;  // column of the first set
    const int left = a.H - u.h0 - 4 * q;                  // sets from this lane's first on
#pragma unroll
    for (int k = 0; k < 2; k++)
        load4(a.w + (first + i) * kDesc + WideRow<T>::place(q, k), u.h0 + i < a.H, w + 4 * k);
#pragma unroll
    for (int k = 0; k < 4; k++)
        if (a.b && k < left) bias[k] = a.b[first + 4 * q + k];
    struct Tile {
        WideRow<T> x;
        float4_v res;
        int idx;
    };
    auto row_of = [&](int r) {  // the sample row r + i reads; -1: absent, or past the end
        int idx = -1;
        if (r + i < u.r1) {
            idx = a.rows ? a.rows[r + i] : r + i;
            if ((unsigned)idx >= (unsigned)a.n) idx = -1;
        }
        return idx;
    };
    const unsigned lane_off = (unsigned)(i * u.step) + q * 16;
    auto load = [&](int r, int idx) {
        Tile t;
        t.idx = idx;
        if (u.in_order && r + 16 <= u.r1) t.x.load(u.x + r * u.step + lane_off);
        else t.x.load(u.x + (idx < 0 ? 0 : idx) * u.step + q * 16);
        t.res = float4_v{0, 0, 0, 0};
        const int row = r + i;
        if (row < u.r1) {
            if (a.res_kind == SC_RES_ROW) {
                const float v = a.res[(long long)row * a.res_ld];
                t.res = float4_v{v, v, v, v};
            } else if (a.res_kind == SC_RES_FULL) {
                const float *p = a.res + (long long)row * a.res_ld + first + 4 * q;
                if (left >= 4) {
                    t.res = *reinterpret_cast<const float4_a4 *>(p);
                } else {
#pragma unroll
                    for (int k = 0; k < 3; k++)
                        if (k < left) t.res[k] = p[k];
                }
            }
        }
        return t;
    };
    auto finish = [&](int r, const Tile &t) {
        float f[8];
        t.x.values(f);
        float4_v z = bias;
#pragma unroll
        for (int k = 0; k < 8; k++) z = __builtin_amdgcn_mfma_f32_16x16x4f32(w[k], f[k], z, 0, 0, 0);
        float4_v y;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            y[k] = a.alpha * (a.act == SC_ACT_SIGMOID ? sigmoid(z[k]) : z[k]);
            if (t.idx < 0 || !u.present) y[k] = 0.0f;  // an absent row or patch has no response
            if (a.res_kind != SC_RES_NONE) y[k] += a.beta * t.res[k];
        }
        const int row = r + i;
        if (row < u.r1) {
            float *p = a.y + (long long)row * a.y_ld + first + 4 * q;
            if (left >= 4) {
                *reinterpret_cast<float4_a4 *>(p) = y;
            } else {
#pragma unroll
                for (int k = 0; k < 3; k++)
                    if (k < left) p[k] = y[k];
            }
        }
    };
    // two tiles in turn: the next one's loads are issued before a tile's
    // products, its rows' numbers a tile earlier still
    int ahead = row_of(u.r0 + 16);
    Tile one = load(u.r0, row_of(u.r0)), two;
    for (int r = u.r0; r < u.r1; r += 32) {
        two = load(r + 16, ahead);
        ahead = row_of(r + 32);
        finish(r, one);
        if (r + 16 >= u.r1) break;
        one = load(r + 32, ahead);
        ahead = row_of(r + 48);
        finish(r + 16, two);
    }
}

// What the gradient kernels of the wide form know of a lane's row r + i ...
struct WideMeta {
    int idx;         // its sample; -1: absent, or past the end
    float pos, neg;  // (loss)
};
template <int MODE>
__device__ __forceinline__ WideMeta wide_meta(const LrArgs &a, const WideUnit &u, int r, int i) {
    WideMeta v{-1, 0.0f, 0.0f};
    if (r + i < u.r1) {
        v.idx = a.rows ? a.rows[r + i] : r + i;
        if ((unsigned)v.idx >= (unsigned)a.n) v.idx = -1;
    }
    if constexpr (MODE == kLoss) {
        if (v.idx >= 0) {
            const float c = a.weight ? a.weight[v.idx] : 1.0f, t = a.target[v.idx];
            v.pos = c * (1.0f - t);
            v.neg = c * t;
            if (c == 0.0f) v.idx = -1;  // a row without weight is not looked at, whatever it holds
        }
    }
    return v;
}

// two neighbouring values as they are loaded
typedef float float2_a4 __attribute__((ext_vector_type(2), aligned(4)));
typedef unsigned uint_a2 __attribute__((aligned(2)));
template <class T>
using PlacePair = std::conditional_t<T::kSize == 4, float __attribute__((ext_vector_type(2))), unsigned>;
template <class T>
__device__ __forceinline__ PlacePair<T> load_pair(const char *p) {
    if constexpr (T::kSize == 4) return *reinterpret_cast<const float2_a4 *>(p);
    else return *reinterpret_cast<const uint_a2 *>(p);
}

// ... and what they load of 16 rows.  Absent rows load some sample's values
// instead, which are cleared where they are used: a tile without any (every
// tile but the last, mostly) has no branches.
template <class T>
struct WideTile {
    WideMeta v;
    WideRow<T> x;        // row i
    PlacePair<T> xc[4];  // rows 4q .. 4q+3, places 2i and 2i+1
    float dy[4];         // of those rows, set i
    bool whole;          // no row of it is absent
};
// (a lane's own offsets; everything else of an address is the same in a wave)
struct WideOffsets {
    unsigned row, place, dy, dres;
};
template <class T>
__device__ __forceinline__ WideOffsets wide_offsets(const LrArgs &a, const WideUnit &u, int i, int q, long long col) {
    WideOffsets o;
    o.row = (unsigned)(i * u.step) + q * 16;
    o.place = (unsigned)(4 * q * u.step) + 2 * i * T::kSize;
    o.dy = (unsigned)(4 * q * a.dy_ld + col);
    o.dres = (unsigned)(4 * q * a.dres_ld + col);
    return o;
}
__device__ __forceinline__ void load_dy(const LrArgs &a, const WideUnit &u, const WideOffsets &o, int r, int q,
                                        long long col, float (&dy)[4]) {
    if (u.dense && r + 16 <= u.r1) {
#pragma unroll
        for (int k = 0; k < 4; k++) dy[k] = (a.dy + (long long)(r + k) * a.dy_ld)[o.dy];
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int row = r + q * 4 + k < u.r1 ? r + q * 4 + k : u.r0;
            dy[k] = a.dy[(long long)row * a.dy_ld + col];
        }
    }
}
__device__ __forceinline__ void store_dres(const LrArgs &a, const WideUnit &u, const WideOffsets &o, int r, int q,
                                           long long col, const float (&dy)[4]) {
    if (u.dense && r + 16 <= u.r1) {
#pragma unroll
        for (int k = 0; k < 4; k++) (a.dres + (long long)(r + k) * a.dres_ld)[o.dres] = a.beta * dy[k];
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (r + q * 4 + k < u.r1) a.dres[(long long)(r + q * 4 + k) * a.dres_ld + col] = a.beta * dy[k];
    }
}
template <class T, int MODE>
__device__ __forceinline__ void wide_load(const LrArgs &a, const WideUnit &u, const WideOffsets &o, int r, WideMeta v,
                                          int i, int q, long long col, WideTile<T> &t) {
    t.v = v;
    t.whole = u.present && __ballot(v.idx < 0) == 0;
    if (u.in_order && r + 16 <= u.r1) {
        const char *base = u.x + r * u.step;
        t.x.load(base + o.row);
#pragma unroll
        for (int k = 0; k < 4; k++) t.xc[k] = load_pair<T>(base + k * u.step + o.place);
    } else {
        const int j = v.idx < 0 ? 0 : v.idx;
        t.x.load(u.x + j * u.step + q * 16);
#pragma unroll
        for (int k = 0; k < 4; k++)
            t.xc[k] = load_pair<T>(u.x + __shfl(j, q * 4 + k, 64) * u.step + 2 * i * T::kSize);
    }
    if constexpr (MODE == kGrad) load_dy(a, u, o, r, q, col, t.dy);
}

// g of this lane's four results; clears what an absent row loaded
template <class T, int MODE>
__device__ __forceinline__ void wide_grad(const LrArgs &a, const WideUnit &u, const WideOffsets &o, WideTile<T> &t, float4_v z,
                                          int r, int q, bool on, long long col, float (&g)[4], float &sum_g, float &sum_l) {
    float pos[4], neg[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        if constexpr (MODE == kLoss) {
            pos[k] = __shfl(t.v.pos, q * 4 + k, 64);
            neg[k] = __shfl(t.v.neg, q * 4 + k, 64);
        } else {
            pos[k] = a.alpha * t.dy[k];
            neg[k] = 0.0f;
        }
    }
    if (MODE == kGrad && a.res_kind == SC_RES_FULL && on) store_dres(a, u, o, r, q, col, t.dy);
    if (t.whole) {
#pragma unroll
        for (int k = 0; k < 4; k++) g[k] = grad_of<MODE>(a.act, z[k], pos[k], neg[k], sum_l);
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const bool there = u.present && __shfl(t.v.idx, q * 4 + k, 64) >= 0;
            float l = sum_l;
            const float gk = grad_of<MODE>(a.act, z[k], pos[k], neg[k], l);
            g[k] = there ? gk : 0.0f;
            sum_l = there ? l : sum_l;
            if (!there) t.xc[k] = PlacePair<T>{};
        }
    }
    sum_g += (g[0] + g[1]) + (g[2] + g[3]);
}

// a wave's sums -> the partial sums of its chunk, or the results: of a lane's
// places 2i and 2i+1, of `left` sets from `first` on; of its own set `col`
template <int MODE>
__device__ __forceinline__ void wide_store(const LrArgs &a, const float4_v *acc, float sum_g, float sum_l, int i, int q,
                                           long long first, int left, bool on, long long col) {
    sum_g += __shfl_xor(sum_g, 16, 64);
    sum_g += __shfl_xor(sum_g, 32, 64);
    sum_l += __shfl_xor(sum_l, 16, 64);
    sum_l += __shfl_xor(sum_l, 32, 64);
    float *part = a.part ? a.part + (long long)blockIdx.y * a.M * a.H * kPartWords : nullptr;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        if (k >= left) continue;
        const long long mh = first + k;
        float *to = part ? part + mh * kPartWords : a.dw + mh * kDesc;
        to[2 * i] = acc[0][k];
        to[2 * i + 1] = acc[1][k];
    }
    if (on && q == 0) {
        if (part) {
            part[col * kPartWords + kDesc] = sum_g;
            part[col * kPartWords + kDesc + 1] = sum_l;
        } else {
            a.db[col] = sum_g;
            if (MODE == kLoss) a.loss[col] = sum_l;
        }
    }
}

template <class T>
__device__ __forceinline__ float place_value(PlacePair<T> v, int half) {
    if constexpr (__is_same(T, F32)) return v[half];
    else return (float)__builtin_bit_cast(half2_v, v)[half];
}

// Gradient and loss, f32 products (16x16x4: nothing is rounded that the narrow
// form does not round).
template <class T, int MODE>
__global__ __launch_bounds__(64 * kWideWaves, 4) void lr_wide_kernel(LrArgs a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, q = lane >> 4;
    WideUnit u;
    if (!wide_unit<T>(a, wave, u)) return;
    const bool on = u.h0 + i < a.H;
    const long long col = (long long)u.m * a.H + (on ? u.h0 + i : 0);  // (lanes past the sets read the first one's)
    float w[8];
#pragma unroll
    for (int k = 0; k < 2; k++) load4(a.w + col * kDesc + WideRow<T>::place(q, k), on, w + 4 * k);
    const float bias = on && a.b ? a.b[col] : 0.0f;
    const WideOffsets o = wide_offsets<T>(a, u, i, q, col);
    float4_v acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    float sum_g = 0.0f, sum_l = 0.0f;
    auto products = [&](int r, WideTile<T> &t) {
        float f[8], g[4];
        t.x.values(f);
        float4_v z = {bias, bias, bias, bias};
#pragma unroll
        for (int k = 0; k < 8; k++) z = __builtin_amdgcn_mfma_f32_16x16x4f32(f[k], w[k], z, 0, 0, 0);
        wide_grad<T, MODE>(a, u, o, t, z, r, q, on, col, g, sum_g, sum_l);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            acc[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(g[k], place_value<T>(t.xc[k], 0), acc[0], 0, 0, 0);
            acc[1] = __builtin_amdgcn_mfma_f32_16x16x4f32(g[k], place_value<T>(t.xc[k], 1), acc[1], 0, 0, 0);
        }
    };
    WideMeta ahead = wide_meta<MODE>(a, u, u.r0 + 16, i);
    WideTile<T> one, two;
    wide_load<T, MODE>(a, u, o, u.r0, wide_meta<MODE>(a, u, u.r0, i), i, q, col, one);
    for (int r = u.r0; r < u.r1; r += 32) {
        wide_load<T, MODE>(a, u, o, r + 16, ahead, i, q, col, two);
        ahead = wide_meta<MODE>(a, u, r + 32, i);
        products(r, one);
        if (r + 16 >= u.r1) break;
        wide_load<T, MODE>(a, u, o, r + 32, ahead, i, q, col, one);
        ahead = wide_meta<MODE>(a, u, r + 48, i);
        products(r + 16, two);
    }
    wide_store<MODE>(a, acc, sum_g, sum_l, i, q, (long long)u.m * a.H + u.h0 + 4 * q, a.H - u.h0 - 4 * q, on, col);
}

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// v = a + b + c, each a bfloat16 (8 + 8 + 8 bits of 24): the high halves (an
// infinite v: a, and NaN for what is left of it).  The products of an infinite
// sample with the parts are NaN where a part is 0, and of a small g the bits
// below a bfloat16's least, 2^-133, are in no part.  A chunk whose sums come out
// not finite or that small is therefore summed again, `exact`: only the first
// part meets infinite samples, the others 0 in their place, and small sums' g are
// split 2^16 times as large (the other sets' sums get the bits they had).
__device__ __forceinline__ void split3(float v, unsigned &a, unsigned &b, unsigned &c) {
    a = __float_as_uint(v) & 0xffff0000u;
    const float r = v - __uint_as_float(a);
    b = __float_as_uint(r) & 0xffff0000u;
    c = __float_as_uint(r - __uint_as_float(b)) & 0xffff0000u;
}
// two high halves -> one register, `lo` first
__device__ __forceinline__ unsigned pack(unsigned lo, unsigned hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302u); }

// two samples a register, 0 where they are infinite or NaN
__device__ __forceinline__ unsigned finite_pair(unsigned v) {
    if ((v & 0x7f80u) == 0x7f80u) v &= 0xffff0000u;
    if ((v & 0x7f800000u) == 0x7f800000u) v &= 0xffffu;
    return v;
}
template <class V>
__device__ __forceinline__ V finite_pairs(V v) {
#pragma unroll
    for (unsigned k = 0; k < sizeof(V) / 4; k++) v[k] = finite_pair(v[k]);
    return v;
}

// g's parts of two results
template <bool EXACT>
__device__ __forceinline__ void split_grads(float g0, float g1, float scale, float &most, unsigned &p0, unsigned &p1,
                                            unsigned &p2) {
    unsigned lo[3], hi[3];
    if constexpr (EXACT) {
        most = fmaxf(most, fmaxf(fabsf(g0), fabsf(g1)));
        g0 *= scale;
        g1 *= scale;
    }
    split3(g0, lo[0], lo[1], lo[2]);
    split3(g1, hi[0], hi[1], hi[2]);
    if constexpr (EXACT) {
        if (__builtin_isinf(g0)) lo[1] = lo[2] = 0;
        if (__builtin_isinf(g1)) hi[1] = hi[2] = 0;
    }
    p0 = pack(lo[0], hi[0]);
    p1 = pack(lo[1], hi[1]);
    p2 = pack(lo[2], hi[2]);
}

// Whether a wave has to sum again; `scale` of its lane's set then.  (Of 2^11 rows
// the bits below 2^-133 are one in 2^24 of sums below 2^-98.)
template <int N>
__device__ __forceinline__ bool again(const float4_v (&acc)[N], float sum_g, float &scale) {
    float t = 0.0f * sum_g;
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
        for (int k = 0; k < 4; k++) t = __builtin_fmaf(acc[n][k], 0.0f, t);
    sum_g += __shfl_xor(sum_g, 16, 64);
    sum_g += __shfl_xor(sum_g, 32, 64);
    scale = sum_g != 0.0f && fabsf(sum_g) < 3.1554436e-30f ? 65536.0f : 1.0f;
    return __any(t != t || scale != 1.0f);
}
// Large g that cancel leave a small sum as well, but do not bear the scale (`most`
// of them; their sums' bits are far above): whether a set has to go without
__device__ __forceinline__ bool without(float most, float &scale) {
    most = fmaxf(most, __shfl_xor(most, 16, 64));
    most = fmaxf(most, __shfl_xor(most, 32, 64));
    const bool large = scale != 1.0f && most > 1.0f;
    if (large) scale = 1.0f;
    return __any(large);
}
// the sums of the sets 4q .. as they are
template <int N>
__device__ __forceinline__ void unscale(float4_v (&acc)[N], float scale, int q) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const float by = 1.0f / __shfl(scale, q * 4 + k, 64);  // (a power of two)
#pragma unroll
        for (int n = 0; n < N; n++) acc[n][k] *= by;
    }
}

// a lane's 8 weights (as they are: times log 2's inverse, for an exponential with
// a product less, the largest would be infinite)
__device__ __forceinline__ void split_weights(const float (&wf)[8], uint4_v (&w)[3]) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
        unsigned lo[3], hi[3];
        const float a = wf[2 * k], b = wf[2 * k + 1];
        split3(a, lo[0], lo[1], lo[2]);
        split3(b, hi[0], hi[1], hi[2]);
        if (__builtin_isinf(a)) lo[1] = lo[2] = 0;  // (an infinite weight's response is no NaN)
        if (__builtin_isinf(b)) hi[1] = hi[2] = 0;
#pragma unroll
        for (int e = 0; e < 3; e++) w[e][k] = pack(lo[e], hi[e]);
    }
}

// Gradient and loss of bfloat16 samples on the bfloat16 matrix cores (16x16x32,
// a fifth of the f32 ones' time for these products): the samples are exact
// there, and the weights and g go in as sums of three bfloat16 each, their 24
// bits whole (but for what lies below 2^-133 of a g beside large ones or in a sum
// of 0), so every product is exact and the sums are f32 as before.
template <int MODE>
__global__ __launch_bounds__(64 * kWideWaves) void lr_wide_bf16_kernel(LrArgs a) {
    using T = BF16;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, q = lane >> 4;
    WideUnit u;
    if (!wide_unit<T>(a, wave, u)) return;
    const bool on = u.h0 + i < a.H;
    const long long col = (long long)u.m * a.H + (on ? u.h0 + i : 0);
    uint4_v w[3];
    float wf[8];
    load4(a.w + col * kDesc + 8 * q, on, wf);
    load4(a.w + col * kDesc + 8 * q + 4, on, wf + 4);
    split_weights(wf, w);
    const float bias = on && a.b ? a.b[col] : 0.0f;
    const WideOffsets o = wide_offsets<T>(a, u, i, q, col);
    float4_v acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    float sum_g = 0.0f, sum_l = 0.0f, scale, most;
    auto dot = [&](const WideTile<T> &t, auto exact) {
        const uint4_v rest = exact ? finite_pairs(t.x.a) : t.x.a;
        float4_v z = {bias, bias, bias, bias};
#pragma unroll
        for (int e = 2; e >= 0; e--)
            z = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, e ? rest : t.x.a),
                                                        __builtin_bit_cast(bf16x8, w[e]), z, 0, 0, 0);
        return z;
    };
    // the 32 rows of two tiles: k of the second product = (tile, row 4q + k)
    auto products = [&](int r, WideTile<T> &one, WideTile<T> &two, auto exact) {
        const float4_v z1 = dot(one, exact), z2 = dot(two, exact);
        float g[2][4];
        wide_grad<T, MODE>(a, u, o, one, z1, r, q, on, col, g[0], sum_g, sum_l);
        wide_grad<T, MODE>(a, u, o, two, z2, r + 16, q, on, col, g[1], sum_g, sum_l);
        uint4_v gs[3], xs[2];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int tile = k >> 1, e = 2 * (k & 1);
            unsigned p0, p1, p2;
            split_grads<exact>(g[tile][e], g[tile][e + 1], scale, most, p0, p1, p2);
            gs[0][k] = p0;
            gs[1][k] = p1;
            gs[2][k] = p2;
            const WideTile<T> &t = tile ? two : one;
            xs[0][k] = __builtin_amdgcn_perm(t.xc[e + 1], t.xc[e], 0x05040100u);  // the low halves
            xs[1][k] = pack(t.xc[e], t.xc[e + 1]);
        }
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const uint4_v rest = exact ? finite_pairs(xs[half]) : xs[half];
#pragma unroll
            for (int p = 2; p >= 0; p--)
                acc[half] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, gs[p]),
                                                                    __builtin_bit_cast(bf16x8, p ? rest : xs[half]),
                                                                    acc[half], 0, 0, 0);
        }
    };
    WideTile<T> t[4];
    auto load = [&](int r, int k, const WideMeta &m0, const WideMeta &m1) {
        wide_load<T, MODE>(a, u, o, r, m0, i, q, col, t[k]);
        wide_load<T, MODE>(a, u, o, r + 16, m1, i, q, col, t[k + 1]);
    };
    WideMeta m0 = wide_meta<MODE>(a, u, u.r0 + 32, i), m1 = wide_meta<MODE>(a, u, u.r0 + 48, i);
    load(u.r0, 0, wide_meta<MODE>(a, u, u.r0, i), wide_meta<MODE>(a, u, u.r0 + 16, i));
    for (int r = u.r0; r < u.r1; r += 64) {
        load(r + 32, 2, m0, m1);
        m0 = wide_meta<MODE>(a, u, r + 64, i);
        m1 = wide_meta<MODE>(a, u, r + 80, i);
        products(r, t[0], t[1], std::false_type{});
        if (r + 32 >= u.r1) break;
        load(r + 64, 0, m0, m1);
        m0 = wide_meta<MODE>(a, u, r + 96, i);
        m1 = wide_meta<MODE>(a, u, r + 112, i);
        products(r + 32, t[2], t[3], std::false_type{});
    }
    for (bool more = again(acc, sum_g, scale); more; more = without(most, scale)) {
        acc[0] = acc[1] = float4_v{0, 0, 0, 0};
        sum_g = sum_l = most = 0.0f;
        for (int r = u.r0; r < u.r1; r += 32) {
            load(r, 0, wide_meta<MODE>(a, u, r, i), wide_meta<MODE>(a, u, r + 16, i));
            products(r, t[0], t[1], std::true_type{});
        }
        unscale(acc, scale, q);
    }
    wide_store<MODE>(a, acc, sum_g, sum_l, i, q, (long long)u.m * a.H + u.h0 + 4 * q, a.H - u.h0 - 4 * q, on, col);
}

// Up to 8 sets of 16-bit samples, a wave owns two neighbouring learners, lane i's
// results being those of set i % 8 of learner i / 8: every learner has its own
// products, half of which is left (a descriptor's NaN stays its learner's), but
// dy, dres and the arithmetic of g fill the wave.  8191 x 608 x 8, alone and in
// pairs: loss 127 and 106 us in bf16, 189 and 159 in f16, gradient 143 and 103,
// 168 and 146; f32 206 and 253, 197 and 196 (it has no registers for two).  480 x
// 11870 x 8 with dres: 205 and 171.
template <class T>
struct PairTile {
    WideMeta v;
    WideRow<T> x[2];
    PlacePair<T> xc[2][4];
    float dy[4];
    bool whole;
};

typedef unsigned uint2_v __attribute__((ext_vector_type(2)));
typedef short short4_v __attribute__((ext_vector_type(4)));

template <class T, int MODE>
__global__ __launch_bounds__(64 * kWideWaves, 4) void lr_pair_kernel(LrArgs a) {
    constexpr bool kBf16 = __is_same(T, BF16);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, q = lane >> 4;
    WideUnit u;
    u.m = 2 * (blockIdx.x * kWideWaves + wave);
    if (u.m >= a.M) return;
    const char *x[2];
    bool present[2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const int m = u.m + k < a.M ? u.m + k : u.m;
        const int p = a.patch ? a.patch[m] : m;
        present[k] = (unsigned)p < (unsigned)a.n_patches;
        x[k] = static_cast<const char *>(a.x) + (long long)(present[k] ? p : 0) * kDesc * T::kSize;
    }
    u.h0 = 0;
    u.present = present[0] && present[1];
    wide_rows<T>(a, u);
    const int mine = i >> 3;
    const bool on = (i & 7) < a.H && u.m + mine < a.M;
    const bool here = mine ? present[1] : present[0];
    const long long col = on ? (long long)(u.m + mine) * a.H + (i & 7) : (long long)u.m * a.H;
    float wf[8];
    uint4_v w[3];
#pragma unroll
    for (int k = 0; k < 2; k++) load4(a.w + col * kDesc + WideRow<T>::place(q, k), on, wf + 4 * k);
    const float bias = on && a.b ? a.b[col] : 0.0f;
    if constexpr (kBf16) split_weights(wf, w);
    const WideOffsets o = wide_offsets<T>(a, u, i, q, col);
    float4_v acc[2][2] = {};
    float sum_g = 0.0f, sum_l = 0.0f, scale, most;
    auto load = [&](int r, const WideMeta &v, PairTile<T> &t) {
        t.v = v;
        t.whole = u.present && __ballot(v.idx < 0) == 0;
        if (u.in_order && r + 16 <= u.r1) {
#pragma unroll
            for (int l = 0; l < 2; l++) {
                const char *base = x[l] + r * u.step;
                t.x[l].load(base + o.row);
#pragma unroll
                for (int k = 0; k < 4; k++) t.xc[l][k] = load_pair<T>(base + k * u.step + o.place);
            }
        } else {
            const int j = v.idx < 0 ? 0 : v.idx;
#pragma unroll
            for (int l = 0; l < 2; l++) t.x[l].load(x[l] + j * u.step + q * 16);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const long long at = __shfl(j, q * 4 + k, 64) * u.step + 2 * i * T::kSize;
                t.xc[0][k] = load_pair<T>(x[0] + at);
                t.xc[1][k] = load_pair<T>(x[1] + at);
            }
        }
        if constexpr (MODE == kGrad) load_dy(a, u, o, r, q, col, t.dy);
    };
    auto products = [&](int r, PairTile<T> &t, auto exact) {
        float4_v z[2];
#pragma unroll
        for (int l = 0; l < 2; l++) {
            z[l] = float4_v{bias, bias, bias, bias};
            if constexpr (kBf16) {
                const uint4_v rest = exact ? finite_pairs(t.x[l].a) : t.x[l].a;
#pragma unroll
                for (int e = 2; e >= 0; e--)
                    z[l] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, e ? rest : t.x[l].a),
                                                                   __builtin_bit_cast(bf16x8, w[e]), z[l], 0, 0, 0);
            } else {
                float f[8];
                t.x[l].values(f);
#pragma unroll
                for (int k = 0; k < 8; k++) z[l] = __builtin_amdgcn_mfma_f32_16x16x4f32(f[k], wf[k], z[l], 0, 0, 0);
            }
        }
        if (MODE == kGrad && a.res_kind == SC_RES_FULL && on) store_dres(a, u, o, r, q, col, t.dy);
        float g[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float zk = mine ? z[1][k] : z[0][k];
            float pos, neg = 0.0f;
            if constexpr (MODE == kLoss) {
                pos = __shfl(t.v.pos, q * 4 + k, 64);
                neg = __shfl(t.v.neg, q * 4 + k, 64);
            } else {
                pos = a.alpha * t.dy[k];
            }
            if (t.whole) {
                g[k] = grad_of<MODE>(a.act, zk, pos, neg, sum_l);
            } else {
                const bool row = __shfl(t.v.idx, q * 4 + k, 64) >= 0;
                float l = sum_l;
                const float gk = grad_of<MODE>(a.act, zk, pos, neg, l);
                g[k] = row && here ? gk : 0.0f;
                sum_l = row && here ? l : sum_l;
                if (!(row && present[0])) t.xc[0][k] = PlacePair<T>{};
                if (!(row && present[1])) t.xc[1][k] = PlacePair<T>{};
            }
        }
        sum_g += (g[0] + g[1]) + (g[2] + g[3]);
        if constexpr (kBf16) {
            uint2_v gs[3];
#pragma unroll
            for (int k = 0; k < 2; k++) {
                unsigned p0, p1, p2;
                split_grads<exact>(g[2 * k], g[2 * k + 1], scale, most, p0, p1, p2);
                gs[0][k] = p0;
                gs[1][k] = p1;
                gs[2][k] = p2;
            }
#pragma unroll
            for (int l = 0; l < 2; l++) {
                uint2_v xs[2];
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    xs[0][k] = __builtin_amdgcn_perm(t.xc[l][2 * k + 1], t.xc[l][2 * k], 0x05040100u);  // the low halves
                    xs[1][k] = pack(t.xc[l][2 * k], t.xc[l][2 * k + 1]);
                }
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    const uint2_v rest = exact ? finite_pairs(xs[half]) : xs[half];
#pragma unroll
                    for (int p = 2; p >= 0; p--)
                        acc[l][half] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(
                            __builtin_bit_cast(short4_v, gs[p]), __builtin_bit_cast(short4_v, p ? rest : xs[half]),
                            acc[l][half], 0, 0, 0);
                }
            }
        } else {
#pragma unroll
            for (int l = 0; l < 2; l++)
#pragma unroll
                for (int k = 0; k < 4; k++)
#pragma unroll
                    for (int half = 0; half < 2; half++)
                        acc[l][half] = __builtin_amdgcn_mfma_f32_16x16x4f32(g[k], place_value<T>(t.xc[l][k], half),
                                                                            acc[l][half], 0, 0, 0);
        }
    };
    WideMeta ahead = wide_meta<MODE>(a, u, u.r0 + 16, i);
    PairTile<T> one, two;
    load(u.r0, wide_meta<MODE>(a, u, u.r0, i), one);
    for (int r = u.r0; r < u.r1; r += 32) {
        load(r + 16, ahead, two);
        ahead = wide_meta<MODE>(a, u, r + 32, i);
        products(r, one, std::false_type{});
        if (r + 16 >= u.r1) break;
        load(r + 32, ahead, one);
        ahead = wide_meta<MODE>(a, u, r + 48, i);
        products(r + 16, two, std::false_type{});
    }
    if constexpr (kBf16) {
        for (bool more = again(acc[0], sum_g, scale) | again(acc[1], sum_g, scale); more; more = without(most, scale)) {
            for (int k = 0; k < 4; k++) acc[k >> 1][k & 1] = float4_v{0, 0, 0, 0};
            sum_g = sum_l = most = 0.0f;
            for (int r = u.r0; r < u.r1; r += 16) {
                PairTile<T> t;
                load(r, wide_meta<MODE>(a, u, r, i), t);
                products(r, t, std::true_type{});
            }
            unscale(acc[0], scale, q);
            unscale(acc[1], scale, q);
        }
    }
#pragma unroll
    for (int half = 0; half < 2; half++) acc[0][half] = q >> 1 ? acc[1][half] : acc[0][half];
    // lane (i, q): places 2i and 2i+1 of the sets 4 (q % 2) .. of learner q / 2; sums: of its own set
    wide_store<MODE>(a, acc[0], sum_g, sum_l, i, q, (long long)(u.m + (q >> 1)) * a.H + 4 * (q & 1),
                     u.m + (q >> 1) < a.M ? a.H - 4 * (q & 1) : 0, on, col);
}

// What follows the row chunks, in one launch.  The first `joins` workgroups join
// their partial sums: WORDS neighbouring ones each, every one of SUBS rows of
// threads walks every SUBS-th chunk, in 64 bits; where the rows take several
// launches, acc carries the sums from one's join to the next's.  The others, in
// the last launch, write the gradient of a residual of one value per row, beta *
// the sum of the row's dy: `lanes` of a wave a row, in 64 bits.  (Loss of 8191 x 608 x 16: 13 chunks, 17 MB of
// partial sums, 7.2 us; with 8 rows of 32 threads 8.5.)
template <int SUBS, int WORDS>
__global__ __launch_bounds__(WORDS * SUBS) void lr_tail_kernel(LrArgs a, int loss, int joins, int lanes, int last) {
    if ((int)blockIdx.x >= joins) {
        const long long cols = (long long)a.M * a.H, rows = WORDS * SUBS / lanes;
        const int at = threadIdx.x & (lanes - 1);
        const long long step = (gridDim.x - joins) * rows;
        for (long long r0 = (blockIdx.x - joins) * rows; r0 < a.R; r0 += step) {
            const long long r = r0 + threadIdx.x / lanes;
            double s = 0.0;
            if (r < a.R) {
#pragma unroll 4
                for (long long c = at; c < cols; c += lanes) s += (double)a.dy[r * a.dy_ld + c];
            }
            for (int d = lanes / 2; d; d >>= 1) s += __shfl_xor(s, d, 64);
            if (r < a.R && at == 0) a.dres[r * a.dres_ld] = (float)((double)a.beta * s);
        }
        return;
    }
    __shared__ double s_sum[SUBS][WORDS];
    const long long words = (long long)a.M * a.H * kPartWords;
    const long long i = (long long)blockIdx.x * WORDS + threadIdx.x % WORDS;
    const int sub = threadIdx.x / WORDS;
    double s = 0.0;
    if (i < words) {
#pragma unroll 8
        for (int k = sub; k < a.chunks; k += SUBS) s += (double)a.part[k * words + i];
    }
    s_sum[sub][threadIdx.x % WORDS] = s;
    __syncthreads();
    if (sub != 0 || i >= words) return;
#pragma unroll
    for (int k = 1; k < SUBS; k++) s += s_sum[k][threadIdx.x];
    if (a.acc) {
        if (a.row0) s += a.acc[i];
        if (!last) {
            a.acc[i] = s;
            return;
        }
    }
    const long long mh = i / kPartWords;
    const int word = (int)(i - mh * kPartWords);
    if (word < kDesc) a.dw[mh * kDesc + word] = (float)s;
    else if (word == kDesc) a.db[mh] = (float)s;
    else if (loss) a.loss[mh] = (float)s;
}

// the sums of no rows
__global__ __launch_bounds__(256) void lr_zero_kernel(LrArgs a, int loss) {
    const long long sets = (long long)a.M * a.H, step = (long long)gridDim.x * 256;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < sets * kDesc; i += step) {
        a.dw[i] = 0.0f;
        if (i >= sets) continue;
        a.db[i] = 0.0f;
        if (loss) a.loss[i] = 0.0f;
    }
}

int items_per_wave(const LrArgs &a) { return a.dtype == SC_F32 ? 8 : 16; }
int lanes_per_item(const LrArgs &a) { return a.dtype == SC_F32 ? 8 : 4; }

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

bool wide(const LrArgs &a) { return a.H > kNarrowSets; }
bool pair(const LrArgs &a) { return wide(a) && a.H <= kPairSets && a.dtype != SC_F32; }
bool wide_response(const LrArgs &a) { return a.H > kNarrowResponse; }

template <class T, int MODE>
void launch_form(const LrArgs &a, dim3 grid, hipStream_t s) {
    if (MODE == kResponse ? wide_response(a) : wide(a)) {
        constexpr dim3 block(64 * kWideWaves);
        if constexpr (MODE == kResponse) hipLaunchKernelGGL((lr_wide_response_kernel<T>), grid, block, 0, s, a);
        else if (pair(a)) {
            if constexpr (T::kSize == 2) hipLaunchKernelGGL((lr_pair_kernel<T, MODE>), grid, block, 0, s, a);
        } else if constexpr (__is_same(T, BF16)) hipLaunchKernelGGL((lr_wide_bf16_kernel<MODE>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((lr_wide_kernel<T, MODE>), grid, block, 0, s, a);
        return;
    }
    const dim3 block(64 * kWaves);
    if (a.H == 1) hipLaunchKernelGGL((lr_kernel<T, 1, MODE>), grid, block, 0, s, a);
    else if (a.H == 2) hipLaunchKernelGGL((lr_kernel<T, 2, MODE>), grid, block, 0, s, a);
    else if (a.H <= 4) hipLaunchKernelGGL((lr_kernel<T, 4, MODE>), grid, block, 0, s, a);
    else if constexpr (MODE == kResponse) {
        if (a.H <= 6) hipLaunchKernelGGL((lr_kernel<T, 6, MODE>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((lr_kernel<T, 8, MODE>), grid, block, 0, s, a);
    }
}

template <int MODE>
void launch_mode(const LrArgs &a, dim3 grid, hipStream_t s) {
    switch (a.dtype) {
        case SC_F32: launch_form<F32, MODE>(a, grid, s); break;
        case SC_F16: launch_form<F16, MODE>(a, grid, s); break;
        default: launch_form<BF16, MODE>(a, grid, s); break;
    }
}

}  // namespace

// Gradient and loss: rows are cut into chunks, of `ranges` waves' rows each.
// Time goes in steps of as many waves as the registers of 256 CUs hold (room),
// each of a wave's rows and what its start and end cost (some 48 rows' time), and
// an eighth of one for the last waves; `join` is what a wave's partial sums cost,
// written and read again, beside a row, and 24 rows the launch that does it.  The
// best of 1 to 4 full rounds of waves.
static int rows_per_wave(long long R, long long waves, int ranges, int step, long long room, int join) {
    if (R <= 16 * ranges) return (int)(ceil_div(ceil_div(R, ranges), step) * step);  // one chunk: nothing to join
    const long long most = ceil_div(R, (long long)ranges * step);
    long long best = -1;
    int found = step;
    for (int rounds = 1; rounds <= 4; rounds++) {
        long long chunks = rounds * room / waves;
        chunks = chunks < 1 ? 1 : chunks > most ? most : chunks;
        const long long rows = ceil_div(ceil_div(R, chunks * ranges), step) * step;
        const long long all = waves * ceil_div(R, rows * ranges);
        long long cost = ((all > room ? all : room) + room / 8) * (rows + 48);
        if (join && all > waves) cost += join * all + 24 * room;
        if (best >= 0 && cost >= best) continue;
        best = cost;
        found = (int)rows;
    }
    return found;
}

// waves over the learners (and sets, which the narrow form has all in one)
static long long narrow_waves(const LrArgs &a) { return ceil_div(a.M, items_per_wave(a)); }
static long long wide_waves(const LrArgs &a) { return a.M * ceil_div(a.H, 16); }
static long long wide_grad_waves(const LrArgs &a) { return pair(a) ? ceil_div(a.M, 2) : wide_waves(a); }

// The rows of a wave's sums in 32 bits, whatever the occupancy would have: some
// 2^11 roundings.  (w = 0 and equal weights, 600000 rows x 5000 x 16 of bf16: with
// 200000 rows a wave, which fill the chip, loss and dw are off by 5e-4 and 1e-3 of
// their values in 59 ms, with 2048 by 3e-6 and 7e-6 in 55; 400000 x 32768 of f32:
// dw 1.5e-3 in 61 ms and 3e-5 in 56.)
constexpr int kSumRows = 2048;
// partial sums of one launch, where rows are cut for that reason alone
constexpr size_t kPartBytes = (size_t)1 << 28;

LrPlan lr_plan(const LrArgs &a) {
    LrPlan p{0, 0, 0, 0, 0};
    if (a.R == 0 || a.M == 0 || a.H == 0) return p;
    // (a chunk of the narrow form is one range of rows per wave of a workgroup)
    const int ranges = wide(a) ? 1 : kWaves;
    p.rows_per_wave = wide(a) ? rows_per_wave(a.R, wide_grad_waves(a), 1, 16, 4096, 20)
                              : rows_per_wave(a.R, narrow_waves(a) * kWaves, kWaves, lanes_per_item(a),
                                              1024 * (a.H == 1 ? 6 : a.H == 2 ? 4 : 3), 0);
    const long long fill = ceil_div(a.R, (long long)p.rows_per_wave * ranges);
    if (p.rows_per_wave > kSumRows) p.rows_per_wave = kSumRows;
    const long long chunks = ceil_div(a.R, (long long)p.rows_per_wave * ranges);
    const size_t words = (size_t)a.M * a.H * kPartWords;
    long long at_once = chunks;
    if (chunks > fill) {  // as many as fill the chip, or as the memory above holds (grid y: 65535), evenly
        at_once = (long long)(kPartBytes / (words * sizeof(float)));
        at_once = at_once < fill ? fill : at_once > 65535 ? 65535 : at_once;
        at_once = ceil_div(chunks, ceil_div(chunks, at_once));
    }
    p.chunks = (int)chunks;
    p.at_once = (int)at_once;
    if (chunks > 1) p.part_bytes = at_once * words * sizeof(float);
    if (chunks > at_once) p.acc_bytes = words * sizeof(double);
    return p;
}

void launch_lr_response(const LrArgs &a0, hipStream_t s) {
    LrArgs a = a0;
    const long long waves = wide_response(a) ? wide_waves(a) : narrow_waves(a);
    // As few rows as a wave can take: one pass, its loads issued at once (16384 x
    // 608 f32: 222 us with 8 rows, 235 with 16, 259 with 64).  The wide form
    // takes 32, for its prefetch, once there are waves enough (2001 x 608 x 16
    // f16: 59.5 us with 32, 63 with 16, 61 with 160).
    const long long rows = !wide_response(a) ? 8 : waves * ceil_div(a.R, 32) < 2048 ? 16 : 32;
    const long long least = ceil_div(ceil_div(a.R, 65535), wide_response(a) ? 16 : 8) * (wide_response(a) ? 16 : 8);  // (grid y)
    a.rows_per_wave = (int)(rows > least ? rows : least);
    const dim3 grid = wide_response(a) ? dim3((unsigned)ceil_div(waves, kWideWaves), (unsigned)ceil_div(a.R, a.rows_per_wave))
                              : dim3((unsigned)ceil_div(waves, kWaves), (unsigned)ceil_div(a.R, a.rows_per_wave));
    launch_mode<kResponse>(a, grid, s);
}

// the sums of one launch's chunks, their join and, behind the last, dres
static void launch_chunks(const LrArgs &a, bool loss, bool last, hipStream_t s) {
    if (a.chunks > 0) {
        const dim3 grid = wide(a) ? dim3((unsigned)ceil_div(wide_grad_waves(a), kWideWaves), (unsigned)a.chunks)
                                  : dim3((unsigned)narrow_waves(a), (unsigned)a.chunks);
        if (loss) launch_mode<kLoss>(a, grid, s);
        else launch_mode<kGrad>(a, grid, s);
    } else if (a.M && a.H) {
        const long long blocks = ceil_div((long long)a.M * a.H * kDesc, 256);
        hipLaunchKernelGGL(lr_zero_kernel, dim3((unsigned)(blocks < 8192 ? blocks : 8192)), dim3(256), 0, s, a, loss ? 1 : 0);
    }
    // threads over the chunks of a word: 32 of many chunks, 4, or 1 of a few (2 chunks
    // of 480 x 11870 x 8: 28 us with 4, 15 with 1)
    const int subs = a.chunks > 32 ? 32 : a.chunks > 4 ? 4 : 1, block = subs == 32 ? 1024 : 256;
    const int joins = a.part ? (int)ceil_div((long long)a.M * a.H * kPartWords, block / subs) : 0;
    // a wave per row, or 16 lanes where rows are short
    const int lanes = (long long)a.M * a.H > 64 ? 64 : 16;
    long long sums = last && !loss && a.res_kind == SC_RES_ROW ? ceil_div(a.R, block / lanes) : 0;
    if (sums > 4096) sums = 4096;
    if (joins + sums == 0) return;
    const dim3 grid((unsigned)(joins + sums));
    if (subs == 32) hipLaunchKernelGGL((lr_tail_kernel<32, 32>), grid, dim3(block), 0, s, a, loss ? 1 : 0, joins, lanes, last);
    else if (subs == 4) hipLaunchKernelGGL((lr_tail_kernel<4, 64>), grid, dim3(block), 0, s, a, loss ? 1 : 0, joins, lanes, last);
    else hipLaunchKernelGGL((lr_tail_kernel<1, 256>), grid, dim3(block), 0, s, a, loss ? 1 : 0, joins, lanes, last);
}

void launch_lr_grad(const LrArgs &a0, const LrPlan &p, void *ws, bool loss, hipStream_t s) {
    LrArgs a = a0;
    a.rows_per_wave = p.rows_per_wave;
    a.acc = p.acc_bytes ? static_cast<double *>(ws) : nullptr;
    a.part = p.part_bytes ? reinterpret_cast<float *>(static_cast<char *>(ws) + p.acc_bytes) : nullptr;
    int from = 0;
    do {
        a.chunks = p.chunks - from < p.at_once ? p.chunks - from : p.at_once;
        a.row0 = (int)((long long)from * p.rows_per_wave * (wide(a) ? 1 : kWaves));
        from += a.chunks;
        launch_chunks(a, loss, from == p.chunks, s);
    } while (from < p.chunks);
}

}  // namespace sc
