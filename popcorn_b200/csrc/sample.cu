// sample.cu — Kernels.Sample: the next token of each row of logits [rows, V]
// by temperature, top-k, top-p, min-p and one given random number per row.
//
// With l_max the row's largest logit, w_i = exp((l_i - l_max) / T). The
// tokens are ordered by (logit descending, index ascending). top-k keeps the
// first k of them, top-p the shortest prefix of those whose weight reaches p
// times theirs, min-p those with w_i >= min_p. The token is the first index i
// (in index order) with sum_{j <= i, kept} w_j > u * sum_{kept} w_j.
// T <= 0 (or NaN): the largest logit, lowest index. NaN logits count as -inf.
//
// A border between two tokens decides the result, so the weights are 42-bit
// fixed point (2^42 for the largest; exp in double by a 64-entry table and a
// degree-4 series) and every sum of them is an exact whole number (in 64
// bits, or in a double where a thread's share fits 2^53): no order of
// additions and no atomic changes a token. Tokens below 2^-43 of the largest
// weigh zero and are never drawn.
//
// One cluster of up to eight CTAs per row: the row is read from HBM once and
// stays in the CTAs' shared memory if it fits (else it is read again from
// L2). Nothing is sorted but a few candidates:
//  * top-k up to 512: a logit that is not above the k-th largest is the k-th
//    largest of the maxima of many groups of tokens (the warps', or, by a
//    histogram, the threads'). The tokens from it on, hardly more than k, go
//    to one CTA, which does all the rest.
//  * top-p: a histogram of all tokens' counts, 2048 bins linear in l_max - l.
//    A bin's weights lie within 1.5 % of one another (29.9 T / 2048), so the
//    counts tell to a few bins where the prefix ends; one pass sums all
//    weights and those before these bins exactly and lists their tokens,
//    which one CTA orders. (Where the guess fails or the list overflows: bins
//    that hold the end for certain, cut into 2048 each with their weights.)
//  * a larger top-k: the histogram; the last bin's tokens are ordered
//    directly when they are few, split again by key when many, and counted
//    off by index when their logits are equal.
// The draw is a scan in index order: per warp's segment, then inside one.
//
// Bound by instructions and, with few rows, by the chain of cluster barriers
// (some 0.6 us each) and cold code; the HBM floor is far. One row of 256000
// bf16, top-k 64: 11 us (all sorting and histogramming in full: 58). 131 rows
// of 50257 f16, top-k 200: 17 us. 48 rows of 256000 f32, top-p 0.9: 75 us, 94
// when the 49 MB come from HBM (a pass of weights more: 120; weights by exp():
// 250); without a filter 48 and 62 us, greedy 30 and 45.
#include <cooperative_groups.h>

#include "common.cuh"
#include "dtype.cuh"
#include "launch.hpp"
#include "popcorn.hpp"

namespace popcorn {
namespace launch {

namespace {

namespace cg = cooperative_groups;
using u64 = unsigned long long;

constexpr int kSampleThreads = 1024;
constexpr int kBins = 2048;
constexpr int kCap = 256;     // tokens of a bin that are ordered directly
constexpr int kList = 2048;   // candidates of a small top-k
// The largest such k: 131 rows of 50257 f16, one of 256000 bf16, 64 of 32000 f32 take 24, 23 and 21 us with the list at k =
// 400 and 30, 38 and 26 us at 1000; by the histogram of all tokens 32, 29 and 20 us whatever k is.
constexpr int kListK = 512;
// Candidates that are drawn by looking at each pair; more are sorted (k = 100, so hardly more candidates: 12.1, 15.9 and
// 14.2 us against 15.2, 18.9 and 16.9; k = 200: 18.3, 20.3 and 18.9 against 17.5, 20.3 and 18.7).
constexpr int kFew = 192;
constexpr int kOneBits = 42;
constexpr int64_t kMostTokens = (1 << 21) - 32768;  // of a CTA: sums of a thread's weights are exact in a double (see of_live)
constexpr double kOne = 4398046511104.0;  // 2^42

struct Pick {
    u64 before_cnt, before_mass;  // of the tokens above the picked bin (of everything the histogram saw, if none is)
    uint32_t n;                   // tokens in the bin
    int bin;                      // -1: the prefix takes everything
};

struct alignas(16) Shared {
    u64 mass[kBins], mass_all[kBins];  // (the second: sums over the cluster, in rank 0)
    alignas(16) uint32_t cnt[kBins];
    uint32_t cnt_all[kBins];
    // 2^(42 + j / 64) with j / 64 taken off the exponent's field, which n / 64 then adds; a copy a lane of a half-warp: no
    // bank conflicts
    double tab[64 * 16];
    u64 wsum[32], wsum2[32];
    u64 ctot[8], ctot2[8];
    u64 extra[32];  // of a warp's segment: the kept weight of the listed tokens
    uint32_t ckmin[8], ckmax[8];
    alignas(16) float maxima[8 * 32];
    float minima[8 * 32];  // of all warps of the cluster
    float border;
    Pick pick;
    u64 cut, cut_mass;  // the last token of the prefix, and the prefix's weight
    int lo_bin, hi_bin;
    uint32_t list_n, local_n;
    int32_t found;
    // (lists of candidates lie over the masses: 2048 keys, 2048 weights)
    __device__ u64* list() { return mass; }
    __device__ u64* list_w() { return mass_all; }
    // (and a CTA's own ones over the counts)
    __device__ u64* local() { return reinterpret_cast<u64*>(cnt); }
};

// NaN counts as -inf, and -0 becomes +0: equal logits have equal keys.
__device__ __forceinline__ float tidy(float f) { return f == f ? f + 0.0f : -INFINITY; }

template <class T>
__device__ __forceinline__ float logit(const char* src, int i) {
    return tidy(Elem<T>::load(src, i));
}

// f(i, l) for the n elements at src, by thread `t` of `nt`: l, an array, holds the logits (as they are) from the i-th on,
// four at a time where alignment allows, so that their arithmetic overlaps. Loads run two rounds ahead of it: a row that does not stay in
// shared memory comes from L2.
template <class T, class F>
__device__ __forceinline__ void each4(const char* src, int n, int t, int nt, F f) {
    constexpr int es = Elem<T>::bytes, V = 16 / es;
    int head = int((16u - (uint32_t(reinterpret_cast<uintptr_t>(src)) & 15u)) & 15u) / es;
    head = head < n ? head : n;
    const int nv = (n - head) / V;
    auto one = [&](int i) {
        const float l[1] = {Elem<T>::load(src, i)};
        f(i, l);
    };
    for (int i = t; i < head; i += nt) one(i);
    const uint4* v = reinterpret_cast<const uint4*>(src + head * es);
    uint4 x = t < nv ? v[t] : uint4{}, y = t + nt < nv ? v[t + nt] : uint4{};
#pragma unroll 1
    for (int c = t; c < nv; c += nt) {
        const uint4 z = c + 2 * nt < nv ? v[c + 2 * nt] : uint4{};
        const int i = head + c * V;
        if constexpr (es == 4) {
            const float l[4] = {__uint_as_float(x.x), __uint_as_float(x.y), __uint_as_float(x.z), __uint_as_float(x.w)};
            f(i, l);
        } else {
            float g[8];
            unpack8<T>(x, g);
            const float l[4] = {g[0], g[1], g[2], g[3]};
            f(i, l);
            const float r[4] = {g[4], g[5], g[6], g[7]};
            f(i + 4, r);
        }
        x = y;
        y = z;
    }
    for (int i = head + nv * V + t; i < n; i += nt) one(i);
}

// f(i, logit), one at a time and tidy.
template <class T, class F>
__device__ __forceinline__ void each(const char* src, int n, int t, int nt, F f) {
    each4<T>(src, n, t, nt, [&](int i, const auto& l) {
        constexpr int N = sizeof(l) / sizeof(float);
#pragma unroll
        for (int e = 0; e < N; ++e) f(i + e, tidy(l[e]));
    });
}

__device__ __forceinline__ uint32_t key_of(float f) {
    const uint32_t b = __float_as_uint(f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float logit_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
// A token by its place in the order: logit first, then the earlier index; larger comes first.
__device__ __forceinline__ u64 token_of(float l, int32_t index) {
    return (u64(key_of(l)) << 32) | (0xffffffffu - uint32_t(index));
}

// The weight and the bin of a logit; l_max is finite. NaN compares false: it is not live.
struct Weight {
    float half_max, half_live;  // l_max / 2; half of what l_max - l may be (halves: their difference cannot overflow)
    float scale;                // bins a unit of that half
    double top, c64;            // l_max; 64 log2(e) / T
    const double* tab;          // this lane's copy

    __device__ __forceinline__ float half_below(float l) const { return fmaf(l, -0.5f, half_max); }
    __device__ __forceinline__ bool is_live(float l) const { return half_below(l) <= half_live; }
    // (2^23 is added: the nearest whole number, 0 .. kBins - 1 of a live token, is in the low bits)
    __device__ __forceinline__ float raw_bin(float l) const { return fmaf(half_below(l), scale, 8388608.f); }
    __device__ __forceinline__ int bin(float l) const {
        return is_live(l) ? __float_as_int(raw_bin(l)) - 0x4b000000 : -1;
    }
    // 2^42 exp((l - l_max) / T) of a live token, to the nearest whole number. With k = 64 log2 of the exponential and n the
    // integer next to it: 2^(n / 64), from a table and an exponent, times 2^((k - n) / 64), |k - n| <= 1/2, by its series
    // to the fourth power (the fifth is below 2^-44). Adding 1.5 2^52 or 2^52 rounds a double to a whole number. (A
    // thread's share of a row, up to 2^11 of them, still sums exactly in a double: of kMostTokens, at whatever alignment, a
    // warp has 64512 and a lane at most 2018.)
    __device__ __forceinline__ double of_live(float l) const {
        const double d = double(l) - top;
        const double r = fma(d, c64, 6755399441055744.0);
        const int n = __double2loint(r);
        const double x = fma(d, c64, 6755399441055744.0 - r);
        double e = fma(x, 5.732851688640402e-10, 2.1173137155464774e-07);  // (ln 2 / 64)^i / i!
        e = fma(e, x, 5.864904955056169e-05);
        e = fma(e, x, 1.0830424696249145e-02);
        e = fma(e, x, 1.0);
        const double t = tab[(n & 63) * 16];
        const double s = __hiloint2double(__double2hiint(t) + int(unsigned(n) * 16384u), __double2loint(t));
        return fma(e, s, 4503599627370496.0) - 4503599627370496.0;
    }
    __device__ __forceinline__ u64 operator()(float l) const { return is_live(l) ? u64(of_live(l)) : 0; }
};

__device__ __forceinline__ u64 warp_sum64(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ u64 warp_scan64(u64 v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 a = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += a;
    }
    return v;
}

// The cluster's view: barriers and the CTAs' shared memory.
struct Cluster {
    Shared* sh;
    int C, rank;
    __device__ __forceinline__ void sync() const {
        if (C == 1) __syncthreads();
        else cg::this_cluster().sync();
    }
    __device__ __forceinline__ Shared* of(int r) const {
        return C == 1 ? sh : cg::this_cluster().map_shared_rank(sh, r);
    }
};

// The tokens [s0, s1) of a CTA's (or of a part of them) that belong to a warp.
__device__ __forceinline__ void segment(int n, int warp, int& s0, int& s1) {
    const int seg = ((n + 31) / 32 + 31) / 32 * 32;
    s0 = warp * seg < n ? warp * seg : n;
    s1 = s0 + seg < n ? s0 + seg : n;
}

// First index (in index order, over the cluster) whose running sum of
// value(i, logit) exceeds target(total), given `acc`, the sum over this warp's
// segment; every thread of the cluster calls it and learns the index (-1:
// none). The CTA that holds it looks at one warp's segment with all of its
// warps, and one of these at a 32nd of that.
template <class T, class V, class G>
__device__ int32_t find(const Cluster& cl, const char* src, int n, int32_t base, u64 acc, V value, G target) {
    Shared* sh = cl.sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (lane == 0) sh->wsum[warp] = acc;
    if (tid == 0) sh->found = -1;
    __syncthreads();
    if (warp == 0) {
        const u64 mine = warp_sum64(sh->wsum[lane]);
        if (lane < cl.C) cl.of(lane)->ctot[cl.rank] = mine;
    }
    cl.sync();
    u64 total = 0, run = 0, mine = 0;
    for (int r = 0; r < cl.C; ++r) {
        if (r == cl.rank) {
            run = total;
            mine = sh->ctot[r];
        }
        total += sh->ctot[r];
    }
    const double goal = target(total);
    if (mine > 0 && double(run) <= goal && goal < double(run + mine)) {  // (the same for the whole CTA)
        // the warp's segment that holds it
        const u64 in1 = run + warp_scan64(sh->wsum[lane], lane);
        const int w1 = __ffs(int(__ballot_sync(0xffffffffu, double(in1) > goal))) - 1;
        run = w1 > 0 ? __shfl_sync(0xffffffffu, in1, (w1 - 1) & 31) : run;
        int b0, b1, s0, s1;
        segment(n, w1 < 0 ? 31 : w1, b0, b1);
        segment(b1 - b0, warp, s0, s1);
        s0 += b0;
        s1 += b0;
        u64 part = 0;
        for (int i = s0 + lane; i < s1; i += 32) part += value(i, logit<T>(src, i));
        part = warp_sum64(part);
        if (lane == 0) sh->wsum2[warp] = part;
        __syncthreads();
        const u64 in2 = run + warp_scan64(sh->wsum2[lane], lane);
        const int w2 = __ffs(int(__ballot_sync(0xffffffffu, double(in2) > goal))) - 1;
        run = warp > 0 ? __shfl_sync(0xffffffffu, in2, (warp - 1) & 31) : run;
        if (warp == w2) {
            for (int i0 = s0; i0 < s1; i0 += 32) {
                const u64 v = i0 + lane < s1 ? value(i0 + lane, logit<T>(src, i0 + lane)) : 0;
                const u64 incl = warp_scan64(v, lane);
                const unsigned hit = __ballot_sync(0xffffffffu, double(run + incl) > goal);
                if (hit) {
                    const int32_t at = base + i0 + (__ffs(int(hit)) - 1);
                    if (lane < cl.C) cl.of(lane)->found = at;
                    break;
                }
                run += __shfl_sync(0xffffffffu, incl, 31);
            }
        }
    }
    cl.sync();
    const int32_t at = sh->found;
    __syncthreads();
    return at;
}

template <class T, class V, class G>
__device__ int32_t locate(const Cluster& cl, const char* src, int n, int32_t base, V value, G target) {
    int s0, s1;
    segment(n, threadIdx.x >> 5, s0, s1);
    u64 acc = 0;
    each<T>(src + int64_t(s0) * Elem<T>::bytes, s1 - s0, threadIdx.x & 31, 32, [&](int i, float l) { acc += value(s0 + i, l); });
    return find<T>(cl, src, n, base, warp_sum64(acc), value, target);
}

// The sum over the cluster's threads.
__device__ u64 cluster_sum(const Cluster& cl, u64 acc) {
    Shared* sh = cl.sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    acc = warp_sum64(acc);
    if (lane == 0) sh->wsum[warp] = acc;
    __syncthreads();
    if (warp == 0) {
        const u64 mine = warp_sum64(sh->wsum[lane]);
        if (lane < cl.C) cl.of(lane)->ctot[cl.rank] = mine;
    }
    cl.sync();
    u64 total = 0;
    for (int r = 0; r < cl.C; ++r) total += sh->ctot[r];
    cl.sync();
    return total;
}

// The sums of two, each thread's a whole number in a double.
__device__ void cluster_sums(const Cluster& cl, double a, double b, u64& sum_a, u64& sum_b) {
    Shared* sh = cl.sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    u64 x = warp_sum64(u64(a)), y = warp_sum64(u64(b));
    if (lane == 0) {
        sh->wsum[warp] = x;
        sh->wsum2[warp] = y;
    }
    __syncthreads();
    if (warp == 0) {
        x = warp_sum64(sh->wsum[lane]);
        y = warp_sum64(sh->wsum2[lane]);
        if (lane < cl.C) {
            cl.of(lane)->ctot[cl.rank] = x;
            cl.of(lane)->ctot2[cl.rank] = y;
        }
    }
    cl.sync();
    sum_a = sum_b = 0;
    for (int r = 0; r < cl.C; ++r) {
        sum_a += sh->ctot[r];
        sum_b += sh->ctot2[r];
    }
    cl.sync();
}

// value summed over the cluster's tokens, exactly.
template <class T, class V>
__device__ u64 total_of(const Cluster& cl, const char* src, int n, V value) {
    u64 acc = 0;
    each<T>(src, n, threadIdx.x, kSampleThreads, [&](int, float l) { acc += value(l); });
    return cluster_sum(cl, acc);
}

__device__ void clear_bins(const Cluster& cl, bool masses) {
    for (int b = threadIdx.x; b < kBins; b += kSampleThreads) {
        cl.sh->cnt[b] = 0;
        if (masses) cl.sh->mass[b] = 0;
    }
    __syncthreads();
}

// The cluster's bins summed into rank 0.
__device__ void gather_bins(const Cluster& cl, bool masses) {
    cl.sync();
    Shared* lead = cl.of(0);
    for (int b = cl.rank + cl.C * int(threadIdx.x); b < kBins; b += cl.C * kSampleThreads) {
        u64 m = 0;
        uint32_t c = 0;
#pragma unroll 4
        for (int r = 0; r < cl.C; ++r) {
            const Shared* o = cl.of(r);
            c += o->cnt[b];
            if (masses) m += o->mass[b];
        }
        lead->cnt_all[b] = c;
        lead->mass_all[b] = m;
    }
    cl.sync();
}

// Histogram of the tokens that bin(l) >= 0 places (their weights too), summed over the cluster into rank 0.
template <class T, class B>
__device__ void histogram(const Cluster& cl, const char* src, int n, const Weight& w, bool masses, B bin) {
    Shared* sh = cl.sh;
    clear_bins(cl, masses);
    each<T>(src, n, threadIdx.x, kSampleThreads, [&](int, float l) {
        const int b = bin(l);
        if (b < 0) return;
        atomicAdd(&sh->cnt[b], 1u);
        if (masses) {
            const u64 v = w(l);
            if (v) atomicAdd(&sh->mass[b], v);
        }
    });
    gather_bins(cl, masses);
}

// That of all tokens' counts.
template <class T>
__device__ void count_bins(const Cluster& cl, const char* src, int n, const Weight& w) {
    Shared* sh = cl.sh;
    clear_bins(cl, false);
    each4<T>(src, n, threadIdx.x, kSampleThreads, [&](int, const auto& l) {
        constexpr int N = sizeof(l) / sizeof(float);
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (w.is_live(l[e])) atomicAdd(&sh->cnt[__float_as_int(w.raw_bin(l[e])) - 0x4b000000], 1u);
    });
    gather_bins(cl, false);
}

// The bin in which the prefix of `goal` ends: by count (the goal-th token) or by weight (the first token with which the
// weight reaches goal), `before` of either already above it.
__device__ Pick pick_bin(const Cluster& cl, bool by_mass, double goal, u64 before_cnt, u64 before_mass) {
    Shared* sh = cl.sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (cl.rank == 0) {
        static_assert(kBins == 2 * kSampleThreads, "two bins a thread");
        const u64 c0 = sh->cnt_all[2 * tid], c1 = sh->cnt_all[2 * tid + 1];
        const u64 m0 = sh->mass_all[2 * tid], m1 = sh->mass_all[2 * tid + 1];
        u64 c = warp_scan64(c0 + c1, lane), m = warp_scan64(m0 + m1, lane);
        if (lane == 31) {
            sh->wsum[warp] = c;
            sh->wsum2[warp] = m;
        }
        __syncthreads();
        if (warp == 0) {
            const u64 a = warp_scan64(sh->wsum[lane], lane), b = warp_scan64(sh->wsum2[lane], lane);
            sh->wsum[lane] = a;
            sh->wsum2[lane] = b;
        }
        __syncthreads();
        const u64 tc = before_cnt + sh->wsum[31], tm = before_mass + sh->wsum2[31];
        c += before_cnt + (warp ? sh->wsum[warp - 1] : 0);   // inclusive of this thread's bins
        m += before_mass + (warp ? sh->wsum2[warp - 1] : 0);
        if (tid == 0) sh->pick = Pick{tc, tm, 0, -1};
        __syncthreads();
        const u64 ec = c - c0 - c1, em = m - m0 - m1;  // before the first bin
        const double p0 = by_mass ? double(em) : double(ec), p1 = by_mass ? double(em + m0) : double(ec + c0),
                     p2 = by_mass ? double(m) : double(c);
        if (p0 < goal && goal <= p1) sh->pick = Pick{ec, em, uint32_t(c0), 2 * tid};
        else if (p1 < goal && goal <= p2) sh->pick = Pick{ec + c0, em + m0, uint32_t(c1), 2 * tid + 1};
        __syncthreads();
        const Pick got = sh->pick;
        if (tid < cl.C && tid > 0) cl.of(tid)->pick = got;
    }
    cl.sync();
    const Pick p = sh->pick;
    cl.sync();
    return p;
}

// The prefix's last token among the p.n listed ones of its bin; sets sh->cut (a token's key and index, larger =
// earlier) and sh->cut_mass (the prefix's weight).
__device__ void order_list(const Cluster& cl, const Weight& w, bool by_mass, double goal, bool masses, const Pick& p) {
    Shared* sh = cl.sh;
    const int tid = threadIdx.x;
    cl.sync();
    if (cl.rank == 0) {
        const int cnt = int(p.n);
        u64 me = 0, wm = 0, above = 0;
        int place = 0;
        if (tid < cnt) {
            me = sh->list()[tid];
            wm = masses ? w(logit_of(uint32_t(me >> 32))) : 0;
            sh->list_w()[tid] = wm;
        }
        __syncthreads();
        if (tid < cnt) {
            for (int j = 0; j < cnt; ++j)
                if (sh->list()[j] > me) {
                    ++place;
                    above += sh->list_w()[j];
                }
            const u64 ec = p.before_cnt + u64(place), em = p.before_mass + above;
            const bool last =
                by_mass ? double(em) < goal && goal <= double(em + wm) : double(ec) < goal && goal <= double(ec + 1);
            if (last) {
                sh->cut = me;
                sh->cut_mass = em + wm;
            }
        }
        __syncthreads();
        const u64 cut = sh->cut, mass = sh->cut_mass;
        if (tid < cl.C && tid > 0) {
            Shared* o = cl.of(tid);
            o->cut = cut;
            o->cut_mass = mass;
        }
    }
    cl.sync();
}

// As order_list, from the tokens that in_bin(logit) tells.
template <class T, class B>
__device__ void resolve(const Cluster& cl, const char* src, int n, int32_t base, const Weight& w, bool by_mass, double goal,
                        bool masses, Pick p, B in_bin) {
    Shared* sh = cl.sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // members: the picked bin first, then a range of keys
    bool by_key = false;
    uint32_t klo = 0, khi = 0;
    auto member = [&](float l) {
        if (by_key) {
            const uint32_t k = key_of(l);
            return k >= klo && k <= khi;
        }
        return bool(in_bin(l));
    };
    for (;;) {
        if (p.n <= kCap) {
            if (tid == 0) sh->list_n = 0;
            cl.sync();
            Shared* lead = cl.of(0);
            each<T>(src, n, tid, kSampleThreads, [&](int i, float l) {
                if (member(l)) {
                    const uint32_t at = atomicAdd(&lead->list_n, 1u);
                    if (at < kCap) lead->list()[at] = token_of(l, base + i);
                }
            });
            order_list(cl, w, by_mass, goal, masses, p);
            return;
        }
        // the members' smallest and largest keys
        uint32_t kmin = 0xffffffffu, kmax = 0;
        each<T>(src, n, tid, kSampleThreads, [&](int, float l) {
            if (member(l)) {
                const uint32_t k = key_of(l);
                kmin = k < kmin ? k : kmin;
                kmax = k > kmax ? k : kmax;
            }
        });
        kmin = __reduce_min_sync(0xffffffffu, kmin);
        kmax = __reduce_max_sync(0xffffffffu, kmax);
        if (lane == 0) {
            sh->wsum[warp] = kmin;
            sh->wsum2[warp] = kmax;
        }
        __syncthreads();
        if (warp == 0) {
            kmin = __reduce_min_sync(0xffffffffu, uint32_t(sh->wsum[lane]));
            kmax = __reduce_max_sync(0xffffffffu, uint32_t(sh->wsum2[lane]));
            if (lane < cl.C) {
                Shared* o = cl.of(lane);
                o->ckmin[cl.rank] = kmin;
                o->ckmax[cl.rank] = kmax;
            }
        }
        cl.sync();
        kmin = 0xffffffffu;
        kmax = 0;
        for (int r = 0; r < cl.C; ++r) {
            kmin = sh->ckmin[r] < kmin ? sh->ckmin[r] : kmin;
            kmax = sh->ckmax[r] > kmax ? sh->ckmax[r] : kmax;
        }
        if (kmin == kmax) {
            // equal logits: the q-th of them in index order ends the prefix
            const u64 wk = masses ? w(logit_of(kmin)) : 0;
            u64 q;
            if (by_mass) {
                q = wk ? u64((goal - double(p.before_mass)) / double(wk)) : 1;
                q = q > 2 ? q - 2 : 1;
                while (q < p.n && double(p.before_mass + q * wk) < goal) ++q;
            } else {
                q = u64(goal) - p.before_cnt;
            }
            q = q < 1 ? 1 : (q > p.n ? p.n : q);
            const int32_t at = locate<T>(
                cl, src, n, base, [&](int, float l) { return u64(key_of(l) == kmin ? 1 : 0); },
                [&](u64) { return double(q - 1); });
            if (tid == 0) {
                sh->cut = (u64(kmin) << 32) | (0xffffffffu - uint32_t(at));
                sh->cut_mass = p.before_mass + q * wk;
            }
            __syncthreads();
            return;
        }
        int shift = 0;
        while (((kmax - kmin) >> shift) >= uint32_t(kBins)) ++shift;
        histogram<T>(cl, src, n, w, masses, [&](float l) {
            if (!member(l)) return -1;
            return int((kmax - key_of(l)) >> shift);
        });
        p = pick_bin(cl, by_mass, goal, p.before_cnt, p.before_mass);
        if (p.bin < 0) {  // (the goal was inside the set: not reached)
            p.bin = 0;
        }
        by_key = true;
        khi = kmax - (uint32_t(p.bin) << shift);
        const u64 span = (u64(p.bin) + 1) << shift;
        klo = u64(kmax) + 1 > span ? uint32_t(u64(kmax) + 1 - span) : 0u;
        if (klo < kmin) klo = kmin;
    }
}

// Descending bitonic sort of m (a power of two, 64 .. kList) keys, two neighbours a thread: pairs up to 32 apart are a
// thread's own or change lanes by shuffles, the others go through shared memory.
__device__ void sort_down(u64* a, int m) {
    const int tid = threadIdx.x;
    const bool on = 2 * tid < m;  // (whole warps)
    u64 v0 = 0, v1 = 0;
    __syncthreads();
    if (on) {
        v0 = a[2 * tid];
        v1 = a[2 * tid + 1];
    }
#pragma unroll 1
    for (int k = 2; k <= m; k <<= 1) {
        const bool down = (2 * tid & k) == 0;
#pragma unroll 1
        for (int j = k >> 1; j >= 64; j >>= 1) {
            __syncthreads();
            if (on) {
                a[2 * tid] = v0;
                a[2 * tid + 1] = v1;
            }
            __syncthreads();
            if (on) {
                const u64 o0 = a[(2 * tid) ^ j], o1 = a[(2 * tid + 1) ^ j];
                const bool large = ((2 * tid & j) == 0) == down;  // this one keeps the larger
                v0 = (v0 < o0) == large ? o0 : v0;
                v1 = (v1 < o1) == large ? o1 : v1;
            }
        }
        if (on) {
#pragma unroll 1
            for (int j = k >> 1 < 32 ? k >> 1 : 32; j >= 2; j >>= 1) {
                const u64 o0 = __shfl_xor_sync(0xffffffffu, v0, j >> 1), o1 = __shfl_xor_sync(0xffffffffu, v1, j >> 1);
                const bool large = ((2 * tid & j) == 0) == down;
                v0 = (v0 < o0) == large ? o0 : v0;
                v1 = (v1 < o1) == large ? o1 : v1;
            }
            if ((v0 < v1) == down) {
                const u64 t = v0;
                v0 = v1;
                v1 = t;
            }
        }
    }
    __syncthreads();
    if (on) {
        a[2 * tid] = v0;
        a[2 * tid + 1] = v1;
    }
    __syncthreads();
}

// Inclusive sums of v over the CTA's threads, and the total.
__device__ u64 scan_cta(u64 v, u64& total, u64* wsum) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    u64 incl = warp_scan64(v, lane);
    __syncthreads();
    if (lane == 31) wsum[warp] = incl;
    __syncthreads();
    if (warp == 0) wsum[lane] = warp_scan64(wsum[lane], lane);
    __syncthreads();
    total = wsum[31];
    return incl + (warp ? wsum[warp - 1] : 0);
}

// The bins sh->lo_bin .. hi_bin in which the prefix of weight `goal` may end (or that of top_p times all weight, if goal is
// negative), from the counts alone. A bin's tokens weigh between its borders' weights, half a unit each way for the weights'
// own rounding (2^-16 of slack: of an exponent of at most 29.9, l_max - l, the scale, their product and the border's exponent
// are each off by 2^-24 of it, exp2f by a little). A guess instead takes the mean of the two, and a bin more on both sides: a
// handful of bins where the safe ones hold 1.5 % of the weight.
__device__ void end_bins(const Cluster& cl, double temp, const Weight& w, double goal, double top_p, bool guess) {
    Shared* sh = cl.sh;
    const int tid = threadIdx.x;
    if (cl.rank == 0) {
        const float scale = w.scale;
        const double step = scale > 0.f ? 2.0 * 1.4426950408889634 / (temp * double(scale)) : 0.0;  // log2 a bin
        u64 hi[2], lo[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int b = 2 * tid + e;
            const double c = double(sh->cnt_all[b]);
            hi[e] = u64(c * (kOne * double(exp2f(float(-step * fmax(b - 0.5, 0.0)))) * (1.0 + 0x1p-16) + 0.5)) + 1;
            lo[e] = scale > 0.f ? u64(c * fmax(kOne * double(exp2f(float(-step * (b + 0.5)))) * (1.0 - 0x1p-16) - 0.5, 0.0)) : 0;
            if (guess) hi[e] = lo[e] = hi[e] / 2 + lo[e] / 2;
        }
        if (tid == 0) sh->lo_bin = sh->hi_bin = kBins - 1;
        u64 total;
        // the first bin with which the sum reaches the goal
        auto first = [&](u64 x0, u64 x1, int* out) {
            const u64 t = scan_cta(x0 + x1, total, sh->wsum);
            const double g = goal < 0.0 ? top_p * double(total) : goal;
            if (double(t) >= g) atomicMin(out, double(t - x1) >= g ? 2 * tid : 2 * tid + 1);
        };
        first(hi[0], hi[1], &sh->lo_bin);
        if (!guess) first(lo[0], lo[1], &sh->hi_bin);
        __syncthreads();
        int a = sh->lo_bin, b = sh->hi_bin;
        if (guess) {
            b = a < kBins - 1 ? a + 1 : a;
            a = a > 0 ? a - 1 : 0;
        }
        __syncthreads();
        if (tid < cl.C) {
            Shared* o = cl.of(tid);
            o->lo_bin = a;
            o->hi_bin = b;
        }
    }
    cl.sync();
}

// The prefix's last token among n listed ones, `before` above them; one CTA. Sets sh->cut, or leaves it 0 if the goal lies
// elsewhere.
__device__ void cut_of_list(Shared* sh, int n, const Weight& w, u64 before, double goal) {
    const int tid = threadIdx.x;
    u64* list = sh->list();
    int m = 64;
    while (m < n) m <<= 1;
    for (int i = n + tid; i < m; i += kSampleThreads) list[i] = 0;
    if (tid == 0) sh->cut = 0;
    sort_down(list, m);
    u64 v[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) v[e] = 2 * tid + e < n ? w(logit_of(uint32_t(list[2 * tid + e] >> 32))) : 0;
    u64 total;
    const u64 incl = before + scan_cta(v[0] + v[1], total, sh->wsum);
    const double p0 = double(incl - v[1] - v[0]), p1 = double(incl - v[1]), p2 = double(incl);
    if (p0 < goal && goal <= p1) sh->cut = list[2 * tid];
    if (p1 < goal && goal <= p2) sh->cut = list[2 * tid + 1];
    __syncthreads();
}

// The token from a list of at most kFew candidates that holds the k first ones; one CTA. Four lanes a candidate, which
// look at every other one twice: those before it in the order tell the cut, the kept ones of lower index the draw.
__device__ int32_t draw_from_few(Shared* sh, int n, int k, const Weight& w, float top_p, u64 floor_w, float u) {
    static_assert(4 * kFew <= kSampleThreads, "four lanes a candidate");
    const int tid = threadIdx.x, i = tid >> 2, part = tid & 3;
    const u64* list = sh->list();
    u64* lw = sh->list_w();
    const u64 me = i < n ? list[i] : 0;
    const u64 v = i < n ? w(logit_of(uint32_t(me >> 32))) : 0;
    if (part == 0) lw[i] = v;
    if (tid == 0) sh->found = -1;
    __syncthreads();
    u64 above = 0;
    int place = 0;
    if (i - (i & 7) < n) {  // (whole warps)
        for (int j = part; j < n; j += 4) {
            const bool is = list[j] > me;
            place += is;
            above += is ? lw[j] : 0;
        }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            place += __shfl_xor_sync(0xffffffffu, place, o);
            above += __shfl_xor_sync(0xffffffffu, above, o);
        }
    }
    // (the last of the k knows the whole weight)
    const bool in_k = i < n && place < k;
    if (part == 0 && i < n && place == (n < k ? n : k) - 1) sh->cut_mass = above + v;
    __syncthreads();
    const double goal = top_p < 1.f ? fmax(double(top_p) * double(sh->cut_mass), 1.0) : 1e300;
    const bool keep = in_k && double(above) < goal && v >= floor_w && v > 0;
    if (part == 0) lw[i] = keep ? v : 0;
    __syncthreads();
    if (i - (i & 7) < n) {
        u64 kept = 0, before = 0;
        for (int j = part; j < n; j += 4) {
            const u64 x = lw[j];
            kept += x;
            before += uint32_t(list[j]) > uint32_t(me) ? x : 0;  // (low words fall with the index)
        }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            kept += __shfl_xor_sync(0xffffffffu, kept, o);
            before += __shfl_xor_sync(0xffffffffu, before, o);
        }
        const double at = double(u) * double(kept);
        if (keep && part == 0 && double(before) <= at && at < double(before + v)) sh->found = int32_t(0xffffffffu - uint32_t(me));
    }
    __syncthreads();
    return sh->found;
}

// As draw_from_few, from up to kList candidates: sorted by the order, cut, sorted by index, drawn.
__device__ int32_t draw_from_list(Shared* sh, int n, int k, const Weight& w, float top_p, u64 floor_w, float u) {
    const int tid = threadIdx.x;
    u64* list = sh->list();
    u64* lw = sh->list_w();
    int m = 64;
    while (m < n) m <<= 1;
    for (int i = n + tid; i < m; i += kSampleThreads) list[i] = 0;
    sort_down(list, m);
    n = n < k ? n : k;
    // two neighbours a thread
    u64 v[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int i = 2 * tid + e;
        const uint32_t key = i < n ? uint32_t(list[i] >> 32) : 0;
        v[e] = i < n ? w(logit_of(key)) : 0;
    }
    u64 total;
    const u64 incl = scan_cta(v[0] + v[1], total, sh->wsum);
    const double goal = top_p < 1.f ? fmax(double(top_p) * double(total), 1.0) : 1e300;
    // kept: before it the weight has not reached the goal, and it weighs enough; then in index order
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int i = 2 * tid + e;
        const u64 before = incl - v[1] - (e ? 0 : v[0]);
        const bool keep = i < n && double(before) < goal && v[e] >= floor_w && v[e] > 0;
        // (the list's low words hold 2^32 - 1 - index: a larger one is an earlier token)
        const u64 id = keep ? (list[i] << 32) | uint32_t(i) : 0;
        lw[i] = keep ? v[e] : 0;
        v[e] = id;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 2; ++e)
        if (2 * tid + e < m) list[2 * tid + e] = v[e];
    sort_down(list, m);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int i = 2 * tid + e;
        v[e] = i < m && list[i] ? lw[uint32_t(list[i])] : 0;
    }
    u64 kept;
    const u64 sum = scan_cta(v[0] + v[1], kept, sh->wsum);
    const double at = double(u) * double(kept);
    if (tid == 0) sh->found = -1;
    __syncthreads();
    const u64 b0 = sum - v[0] - v[1], b1 = sum - v[1];
    if (v[0] && double(b0) <= at && at < double(b1)) sh->found = int32_t(0xffffffffu - uint32_t(list[2 * tid] >> 32));
    if (v[1] && double(b1) <= at && at < double(sum)) sh->found = int32_t(0xffffffffu - uint32_t(list[2 * tid + 1] >> 32));
    __syncthreads();
    return sh->found;
}

template <class T>
__global__ void __launch_bounds__(kSampleThreads, 1) sample_kernel(const Sample p, int C, int chunk, int resident) {
    extern __shared__ __align__(16) char smem[];
    Shared* sh = reinterpret_cast<Shared*>(smem);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    Cluster cl{sh, C, int(blockIdx.x % unsigned(C))};
    const int64_t row = blockIdx.x / unsigned(C);
    if (tid == 0) sh->list_n = 0;
    static_assert(kSampleThreads == 64 * 16, "an entry a thread");
    {
        const double t = exp2(double(tid >> 4) / 64.0);
        sh->tab[tid] = __hiloint2double(__double2hiint(t) + (kOneBits << 20) - (tid >> 4) * 16384, __double2loint(t));
    }
    if (C > 1) asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");  // (this CTA runs)
    pdl_launch_dependents();
    pdl_wait();
    constexpr int es = Elem<T>::bytes, V = 16 / es;
    const int32_t base = cl.rank * chunk;
    const int n = p.V - base < chunk ? (p.V > base ? int(p.V - base) : 0) : chunk;
    const char* global = static_cast<const char*>(p.logits) + (row * p.V + base) * es;
    // (in shared memory at the same distance from a 16-byte border)
    char* data = smem + sizeof(Shared) + (reinterpret_cast<uintptr_t>(global) & 15u);
    const char* src = resident ? data : global;

    const float temp = p.temperature ? p.temperature[row] : 1.f;
    const int32_t k = p.top_k ? p.top_k[row] : 0;
    const float tp = p.top_p ? p.top_p[row] : 1.f;
    const float mp = p.min_p ? p.min_p[row] : 0.f;
    const float u = fminf(fmaxf(p.uniform[row], 0.f), 0.99999994f);
    // the row's largest (and, for the histogram's range, smallest) logit
    // (fmaxf and fminf pass over NaN)
    float mx = -INFINITY, mn = INFINITY;
    auto look = [&](float l) {
        mx = fmaxf(mx, l);
        mn = fminf(mn, l);
    };
    if (resident) {
        int head = int((16u - (uint32_t(reinterpret_cast<uintptr_t>(global)) & 15u)) & 15u) / es;
        head = head < n ? head : n;
        const int nv = (n - head) / V;
        using S = typename T::storage;
        auto one = [&](int i) {
            reinterpret_cast<S*>(data)[i] = reinterpret_cast<const S*>(global)[i];
            look(Elem<T>::load(global, i));
        };
        if (tid < head) one(tid);
        const uint4* g = reinterpret_cast<const uint4*>(global + head * es);
        uint4* d = reinterpret_cast<uint4*>(data + head * es);
#pragma unroll 4
        for (int c = tid; c < nv; c += kSampleThreads) {
            const uint4 x = g[c];
            d[c] = x;
            if constexpr (es == 4) {
                look(__uint_as_float(x.x));
                look(__uint_as_float(x.y));
                look(__uint_as_float(x.z));
                look(__uint_as_float(x.w));
            } else {
                float f[8];
                unpack8<T>(x, f);
#pragma unroll
                for (int e = 0; e < 8; ++e) look(f[e]);
            }
        }
        if (tid < n - head - nv * V) one(head + nv * V + tid);
    } else {
        each4<T>(global, n, tid, kSampleThreads, [&](int, const auto& l) {
            constexpr int N = sizeof(l) / sizeof(float);
#pragma unroll
            for (int e = 0; e < N; ++e) look(l[e]);
        });
    }
    const float own = mx;  // this thread's largest
    auto reduce = [&] {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
        }
    };
    reduce();
    // every CTA of the cluster is running before its memory is written
    if (C > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (lane < C) {
        Shared* o = cl.of(lane);
        o->maxima[cl.rank * 32 + warp] = mx;
        o->minima[cl.rank * 32 + warp] = mn;
    }
    cl.sync();
    mx = -INFINITY;
    mn = INFINITY;
    for (int r = 0; r < C; ++r) {
        mx = fmaxf(mx, sh->maxima[r * 32 + lane]);
        mn = fminf(mn, sh->minima[r * 32 + lane]);
    }
    reduce();
    mx += 0.f;  // (not -0)
    if (!(temp > 0.f) || mx == -INFINITY) {  // (the same for the whole cluster)
        const int32_t first = mx == -INFINITY ? -1
                                              : locate<T>(cl, src, n, base, [&](int, float l) { return u64(l == mx ? 1 : 0); },
                                                          [](u64) { return 0.0; });
        if (cl.rank == 0 && tid == 0) p.tokens[row] = first;
        return;
    }
    if (mx == INFINITY) {
        // infinite logits weigh one each, the others nothing: the first k, the first p of them, all reach min-p
        const int32_t token = locate<T>(
            cl, src, n, base, [&](int, float l) { return u64(l == INFINITY ? 1 : 0); },
            [&](u64 total) {
                double take = k > 0 && double(k) < double(total) ? double(k) : double(total);
                if (tp < 1.f) take = fmax(ceil(double(tp) * take), 1.0);
                return double(u) * take;
            });
        if (cl.rank == 0 && tid == 0) p.tokens[row] = token;
        return;
    }
    const float half_live = fminf(14.95f * temp, 3.402823466e38f);
    const float half_range = fminf(fmaf(mn, -0.5f, 0.5f * mx), half_live);  // (with -inf: half_live)
    const float bins = float(kBins - 1) / half_range;  // (a range too small for it: one bin)
    const Weight w{0.5f * mx, half_live, bins <= 1e30f ? bins : 0.f,
                   double(mx), 64.0 * 1.4426950408889634 / double(temp), sh->tab + (lane & 15)};
    const double min_w = mp > 0.f ? double(fminf(mp, 1.f)) * kOne : 0.0;
    const u64 floor_w = u64(ceil(min_w));  // (v >= it as v >= min_w)
    const bool use_k = k > 0 && k < p.V, use_p = tp < 1.f;  // (NaN: off)
    u64 cut = 0;  // every token
    u64 acc = 0;  // the kept weight of this warp's segment
    bool summed = false;
    if (use_k || use_p) {
        auto d_bin = [&](float l) { return w.bin(l); };
        if (use_k && k <= kListK) {
            // a border that is not above the k-th largest logit: the k-th largest of the warps' maxima where there are
            // four times as many (64 of 8 CTAs: 2 us against the histogram's 6), or the end of its bin among the
            // threads' maxima, or among all tokens
            float border = -INFINITY;
            const int groups = 32 * C;
            const bool own_ones = 4 * k <= kSampleThreads * C;
            if (4 * k <= groups) {
                // (four lanes a maximum, each with a fourth of the others; tid / 4 beyond them only helps its warp)
                const int i = tid >> 2;
                const float me = i < groups ? sh->maxima[i] : INFINITY;
                int place = 0;
                if (i - (i & 7) < groups)
#pragma unroll 2
                    for (int j = 4 * (tid & 3); j < groups; j += 16) {
                        const float4 o = *reinterpret_cast<const float4*>(sh->maxima + j);
                        place += o.x > me || (o.x == me && j < i);
                        place += o.y > me || (o.y == me && j + 1 < i);
                        place += o.z > me || (o.z == me && j + 2 < i);
                        place += o.w > me || (o.w == me && j + 3 < i);
                    }
                place += __shfl_xor_sync(0xffffffffu, place, 1);
                place += __shfl_xor_sync(0xffffffffu, place, 2);
                if (i < groups && place == k - 1) sh->border = me;
                __syncthreads();
                border = sh->border;
            } else {
                Pick b;
                b.bin = -1;
                if (own_ones) {
                    clear_bins(cl, false);
                    const int at = d_bin(own);
                    if (at >= 0) atomicAdd(&sh->cnt[at], 1u);
                    gather_bins(cl, false);
                    b = pick_bin(cl, false, double(k), 0, 0);
                }
                if (b.bin < 0) {
                    count_bins<T>(cl, src, n, w);
                    b = pick_bin(cl, false, double(k), 0, 0);
                }
                // (in logits: a little lower than the bin's end, whatever the roundings)
                if (b.bin >= 0 && w.scale > 0.f)
                    border = mx - 2.f * ((float(b.bin) + 0.5f) / w.scale) * 1.000001f - fabsf(mx) * 1e-6f;
            }
            Shared* lead = cl.of(0);
            if (own >= border)  // (a thread's tokens are the same ones as when it took its maximum)
                each4<T>(src, n, tid, kSampleThreads, [&](int i, const auto& l) {
                    constexpr int N = sizeof(l) / sizeof(float);
                    float most = l[0];
#pragma unroll
                    for (int e = 1; e < N; ++e) most = fmaxf(most, l[e]);
                    if (!(most >= border)) return;
#pragma unroll
                    for (int e = 0; e < N; ++e)
                        if (l[e] >= border && w.is_live(l[e])) {
                            const uint32_t to = atomicAdd(&lead->list_n, 1u);
                            if (to < kList) lead->list()[to] = token_of(tidy(l[e]), base + i + e);
                        }
                });
            cl.sync();
            const uint32_t found = lead->list_n;
            cl.sync();  // (the last look at another CTA's memory, if the list is complete)
            if (found <= kList) {
                if (cl.rank == 0) {
                    const int32_t token = found <= kFew ? draw_from_few(sh, int(found), k, w, tp, floor_w, u)
                                                        : draw_from_list(sh, int(found), k, w, tp, floor_w, u);
                    if (tid == 0) p.tokens[row] = token;
                }
                return;
            }
        }
        // by the counts of all tokens
        double mass = 0.0;
        bool whole = true;  // top-k takes every token that weighs
        if (use_k) {
            count_bins<T>(cl, src, n, w);
            Pick pk = pick_bin(cl, false, double(k), 0, 0);
            if (pk.bin >= 0) {
                whole = false;
                if (use_p) {
                    pk.before_mass = total_of<T>(cl, src, n, [&](float l) {
                        const int b = d_bin(l);
                        return b >= 0 && b < pk.bin ? w(l) : u64(0);
                    });
                }
                resolve<T>(cl, src, n, base, w, false, double(k), use_p, pk, [&](float l) { return d_bin(l) == pk.bin; });
                cut = sh->cut;
                mass = double(sh->cut_mass);
            }
        }
        if (use_p) {
            count_bins<T>(cl, src, n, w);
            double goal = whole ? -1.0 : fmax(double(tp) * mass, 1.0);  // (p <= 0: the first token alone)
            int s0, s1;
            segment(n, warp, s0, s1);
            const char* part = src + int64_t(s0) * es;
            // a guess of the bins that the prefix ends in; all weight and that before them exactly, and their tokens listed
            if (tid < 32) sh->extra[tid] = 0;
            if (tid == 0) sh->list_n = sh->local_n = 0;
            end_bins(cl, double(temp), w, goal, double(tp), true);
            int b0 = sh->lo_bin, b1 = sh->hi_bin;
            float f0 = 8388608.f + float(b0), f1 = 8388608.f + float(b1);
            Shared* lead = cl.of(0);
            double all = 0.0, first = 0.0, kept = 0.0;
            const double min_weight = double(floor_w);
            each4<T>(part, s1 - s0, lane, 32, [&](int i, const auto& l) {
                constexpr int N = sizeof(l) / sizeof(float);
                bool in[N], any = false;
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const float f = w.raw_bin(l[e]);
                    const bool live = w.is_live(l[e]), early = f < f0;  // (an early one is live)
                    in[e] = live && f >= f0 && f <= f1;
                    any = any || in[e];
                    const double v = w.of_live(l[e]);
                    if (live) all += v;
                    if (early) first += v;
                    if (floor_w && early && v >= min_weight) kept += v;
                }
                if (!any) return;
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (in[e]) {
                        const u64 t = token_of(tidy(l[e]), base + s0 + i + e);
                        const uint32_t at = atomicAdd(&sh->local_n, 1u);
                        if (at < kList) {
                            sh->local()[at] = t;
                            const uint32_t to = atomicAdd(&lead->list_n, 1u);
                            if (to < kList) lead->list()[to] = t;
                        } else if (at == kList) {
                            atomicAdd(&lead->list_n, uint32_t(kList));  // (too many)
                        }
                    }
            });
            if (!floor_w) kept = first;
            u64 total, before;
            cluster_sums(cl, all, first, total, before);
            if (whole) goal = fmax(double(tp) * double(total), 1.0);
            bool done = false;
            if (lead->list_n <= kList) {  // (the same for the whole cluster)
                if (cl.rank == 0) {
                    cut_of_list(sh, int(sh->list_n), w, before, goal);
                    const u64 c = sh->cut;
                    if (tid < C && tid > 0) cl.of(tid)->cut = c;
                }
                cl.sync();
                done = sh->cut != 0;
            }
            if (done) {
                cut = sh->cut;
                for (int i = tid; i < int(sh->local_n); i += kSampleThreads) {
                    const u64 t = sh->local()[i];
                    const u64 v = t >= cut ? w(logit_of(uint32_t(t >> 32))) : 0;
                    if (v >= floor_w && v) {
                        const int seg = ((n + 31) / 32 + 31) / 32 * 32;
                        atomicAdd(&sh->extra[(int32_t(0xffffffffu - uint32_t(t)) - base) / seg], v);
                    }
                }
                __syncthreads();
                summed = true;
                acc = warp_sum64(u64(kept)) + sh->extra[warp];
            } else {
                // the safe bins; the weights of a 2048th of them each
                cl.sync();
                count_bins<T>(cl, src, n, w);
                end_bins(cl, double(temp), w, goal, double(tp), false);
                b0 = sh->lo_bin, b1 = sh->hi_bin;
                const float start = float(b0) - 0.5f, fine = float(kBins) / float(b1 + 1 - b0);
                auto f_bin = [&](float l) {  // of a token in b0 .. b1: rises with l_max - l
                    const int b = d_bin(l);
                    if (b < b0 || b > b1) return -1;
                    const int f = int(fmaf(w.half_below(l), w.scale, -start) * fine);
                    return f < 0 ? 0 : (f >= kBins ? kBins - 1 : f);
                };
                before = total_of<T>(cl, src, n, [&](float l) {
                    const int b = d_bin(l);
                    return b >= 0 && b < b0 ? w(l) : u64(0);
                });
                histogram<T>(cl, src, n, w, true, f_bin);
                const Pick pp = pick_bin(cl, true, goal, 0, before);
                if (pp.bin >= 0) {
                    resolve<T>(cl, src, n, base, w, true, goal, true, pp, [&](float l) { return f_bin(l) == pp.bin; });
                    cut = sh->cut;
                }
            }
        }
    }
    const uint32_t cut_key = uint32_t(cut >> 32);
    auto value = [&](int i, float l) -> u64 {
        const uint32_t key = key_of(l);
        if (key < cut_key || token_of(l, base + i) < cut) return 0;
        const u64 v = w(l);
        return v >= floor_w ? v : 0;
    };
    if (!summed) {
        double sum = 0.0;
        const double min_weight = double(floor_w);
        int s0, s1;
        segment(n, warp, s0, s1);
        each4<T>(src + int64_t(s0) * es, s1 - s0, lane, 32, [&](int i, const auto& l) {
            constexpr int N = sizeof(l) / sizeof(float);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const double v = w.of_live(l[e]);
                if (w.is_live(l[e]) && v >= min_weight && (!cut || token_of(tidy(l[e]), base + s0 + i + e) >= cut)) sum += v;
            }
        });
        acc = warp_sum64(u64(sum));
    }
    const int32_t token =
        find<T>(cl, src, n, base, acc, value, [&](u64 total) { return double(u) * double(total); });
    if (cl.rank == 0 && tid == 0) p.tokens[row] = token;
}

template <class T>
cudaError_t run_sample(const Sample& p, cudaStream_t s) {
    const int sms = current_sm_count();
    const size_t room = 227 * 1024 - sizeof(Shared) - 16;  // (16: the row's own distance from a 16-byte border)
    // CTAs a row: all SMs once with few rows, at least 4096 tokens each. (48 rows of 256000 f32, top-p: 3 CTAs, which read
    // the row from L2 again, 94 us, 2 as much, 1 154; 8, which hold it but are 2.6 waves, 134; 131 rows of 50257 f16,
    // top-k: 1 CTA 18 us, 2 39; one row of 256000 bf16, top-k: 8 CTAs 11 us, 4 15, 1 20.)
    auto chunk_of = [&](int c) { return ((p.V + c - 1) / c + 7) / 8 * 8; };
    int C = 1;
    while (C < 8 && p.rows * (C + 1) <= sms && chunk_of(C) > 4096) ++C;
    // (more only for rows near 2^21; a cluster of two takes twice as many CTAs for half of the time each)
    while (chunk_of(C) > kMostTokens) ++C;
    const int64_t chunk = chunk_of(C);
    const bool resident = size_t(chunk) * Elem<T>::bytes <= room;
    const size_t smem = sizeof(Shared) + (resident ? size_t(chunk) * Elem<T>::bytes + 16 : 0);
    static DeviceOnce once;
    cudaError_t e = once.run([] { return allow_smem(sample_kernel<T>, 227 * 1024); });
    if (e != cudaSuccess) return e;
    return launch_cluster(sample_kernel<T>, dim3(unsigned(p.rows * C)), dim3(kSampleThreads), unsigned(C), smem, s, p, C,
                          int(chunk), resident ? 1 : 0);
}

}  // namespace

cudaError_t sample(const Sample& p, cudaStream_t s) {
    if (p.rows == 0) return cudaSuccess;
    switch (p.dtype) {
    case PC_F32: return run_sample<TF32>(p, s);
    case PC_F16: return run_sample<TF16>(p, s);
    case PC_BF16: return run_sample<TBF16>(p, s);
    }
    return cudaErrorInvalidValue;
}

namespace {
RegisterFunctions reg_sample({
    {"sample", reinterpret_cast<const void*>(sample_kernel<TF32>)},
    {"sample_f16", reinterpret_cast<const void*>(sample_kernel<TF16>)},
    {"sample_bf16", reinterpret_cast<const void*>(sample_kernel<TBF16>)},
});
}  // namespace

}  // namespace launch
}  // namespace popcorn
