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
// fixed point (2^42 for the largest; exp in double by a 32-entry table and a
// degree-5 polynomial) and every sum of them is an exact integer: no order
// of additions and no atomic changes a token. Tokens below 2^-43 of the
// largest weigh zero and are never drawn.
//
// One cluster of up to eight CTAs per row: the row is read from HBM once and
// stays in the CTAs' shared memory (longer rows are read again from L2).
// The cut of top-k / top-p is found by selection, not by sorting: a
// histogram of counts and weights over 2048 bins linear in l_max - l (a
// bell-shaped row spreads evenly over them, so the shared atomics rarely
// collide), the bin where the prefix ends, and the exact order of the few
// tokens inside it; a bin of many tokens is split again by key, and equal
// logits are counted off by index. The draw is a two-level scan in index
// order.
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
constexpr int kCap = 256;  // tokens of a bin that are ordered directly
constexpr int kOneBits = 42;
constexpr double kOne = 4398046511104.0;  // 2^42

struct Pick {
    u64 before_cnt, before_mass;  // of the tokens above the picked bin
    u64 total_cnt, total_mass;    // of everything the histogram saw
    uint32_t n;                   // tokens in the bin
    int bin;                      // -1: the prefix takes everything
};

struct Shared {
    u64 mass[kBins], mass_all[kBins];  // (the second: sums over the cluster, in rank 0)
    uint32_t cnt[kBins], cnt_all[kBins];
    u64 list[kCap];
    u64 list_w[kCap];
    double tab[32];
    u64 wsum[32], wsum2[32];
    u64 ctot[8];
    float cmax[8], cmin[8];
    int32_t cidx[8];
    uint32_t ckmin[8], ckmax[8];
    float fa[32], fb[32];
    int32_t ia[32];
    Pick pick;
    u64 cut, cut_mass;  // the last token of the prefix, and the prefix's weight
    uint32_t list_n;
    int32_t found;
};

template <class T>
__device__ __forceinline__ float logit(const char* src, int i) {
    float f;
    if constexpr (Elem<T>::bytes == 4) f = reinterpret_cast<const float*>(src)[i];
    else f = Elem<T>::load(src, i);
    return f == f ? f + 0.0f : -INFINITY;  // (-0 becomes +0: equal logits have equal keys)
}

__device__ __forceinline__ uint32_t key_of(float f) {
    const uint32_t b = __float_as_uint(f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct Weight {
    float lmax, live;  // live: l_max - l above it weighs zero
    double c;          // log2(e) / T
    const double* tab;

    __device__ __forceinline__ bool is_live(float l) const {
        return l == lmax || (l > -INFINITY && lmax - l <= live);
    }
    __device__ __forceinline__ u64 operator()(float l) const {
        if (l == lmax) return u64(1) << kOneBits;
        if (!(lmax - l <= live)) return 0;
        const double t = (double(l) - double(lmax)) * c;
        if (!(t >= -43.0)) return 0;
        const int n = __double2int_rn(t * 32.0);
        const double x = fma(double(n), -1.0 / 32.0, t) * 0.6931471805599453;  // |x| <= ln 2 / 64
        double e = fma(x, 1.0 / 120.0, 1.0 / 24.0);
        e = fma(e, x, 1.0 / 6.0);
        e = fma(e, x, 0.5);
        e = fma(e, x, 1.0);
        e = fma(e, x, 1.0);
        const double scale = __longlong_as_double((long long)(1023 + kOneBits + (n >> 5)) << 52);
        return __double2ull_rn(tab[n & 31] * e * scale);
    }
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

// First index (in index order, over the cluster) whose running sum of
// value(i) exceeds target(total); every thread of the cluster calls it and
// learns the index (-1: none).
template <class V, class G>
__device__ int32_t locate(const Cluster& cl, int n, int32_t base, V value, G target) {
    Shared* sh = cl.sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int seg = ((n + 31) / 32 + 31) / 32 * 32;
    const int s0 = warp * seg, s1 = s0 + seg < n ? s0 + seg : n;
    u64 acc = 0;
    for (int i = s0 + lane; i < s1; i += 32) acc += value(i);
    acc = warp_sum64(acc);
    if (lane == 0) sh->wsum[warp] = acc;
    if (tid == 0) sh->found = -1;
    __syncthreads();
    if (warp == 0) {
        const u64 mine = warp_sum64(sh->wsum[lane]);
        if (lane < cl.C) cl.of(lane)->ctot[cl.rank] = mine;
    }
    cl.sync();
    u64 total = 0, run = 0;
    for (int r = 0; r < cl.C; ++r) {
        if (r == cl.rank) run = total;
        total += sh->ctot[r];
    }
    const double goal = target(total);
    for (int w = 0; w < warp; ++w) run += sh->wsum[w];
    if (acc > 0 && double(run) <= goal && goal < double(run + acc)) {  // this warp's segment holds it
        for (int i0 = s0; i0 < s1; i0 += 32) {
            const u64 v = i0 + lane < s1 ? value(i0 + lane) : 0;
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
    cl.sync();
    const int32_t at = sh->found;
    __syncthreads();
    return at;
}

// Histogram of the tokens that bin(l) >= 0 places, summed over the cluster
// into rank 0, and the bin in which the prefix of `goal` ends: by count
// (by_mass false: the goal-th token) or by weight (the first token with
// which the weight reaches goal), `before` of either already above it.
template <class T, class B>
__device__ void histogram(const Cluster& cl, const char* src, int n, const Weight& w, bool masses, B bin) {
    Shared* sh = cl.sh;
    const int tid = threadIdx.x;
    for (int b = tid; b < kBins; b += kSampleThreads) {
        sh->cnt[b] = 0;
        sh->mass[b] = 0;
    }
    __syncthreads();
    for (int i = tid; i < n; i += kSampleThreads) {
        const float l = logit<T>(src, i);
        const int b = bin(l);
        if (b >= 0) {
            atomicAdd(&sh->cnt[b], 1u);
            if (masses) {
                const u64 v = w(l);
                if (v) atomicAdd(&sh->mass[b], v);
            }
        }
    }
    cl.sync();
    Shared* lead = cl.of(0);
    const int per = kBins / cl.C;
    for (int b = cl.rank * per + tid; b < (cl.rank + 1) * per; b += kSampleThreads) {
        u64 m = 0;
        uint32_t c = 0;
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
        if (tid == 0) sh->pick = Pick{tc, tm, tc, tm, 0, -1};
        __syncthreads();
        const u64 ec = c - c0 - c1, em = m - m0 - m1;  // before the first bin
        const double p0 = by_mass ? double(em) : double(ec), p1 = by_mass ? double(em + m0) : double(ec + c0),
                     p2 = by_mass ? double(m) : double(c);
        if (p0 < goal && goal <= p1) sh->pick = Pick{ec, em, tc, tm, uint32_t(c0), 2 * tid};
        else if (p1 < goal && goal <= p2) sh->pick = Pick{ec + c0, em + m0, tc, tm, uint32_t(c1), 2 * tid + 1};
        __syncthreads();
        const Pick got = sh->pick;
        if (tid < cl.C && tid > 0) cl.of(tid)->pick = got;
    }
    cl.sync();
    const Pick p = sh->pick;
    cl.sync();
    return p;
}

// The prefix's last token inside the picked bin; sets sh->cut (a token's key
// and index, larger = earlier) and sh->cut_mass (the prefix's weight).
template <class T>
__device__ void resolve(const Cluster& cl, const char* src, int n, int32_t base, const Weight& w, float scale,
                        bool by_mass, double goal, bool masses, Pick p) {
    Shared* sh = cl.sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // members: the d-bin `p.bin` first, then a range of keys
    bool by_key = false;
    uint32_t klo = 0, khi = 0;
    const int dbin = p.bin;
    auto d_bin = [&](float l) {
        if (!w.is_live(l)) return -1;
        const float d = l == w.lmax ? 0.f : w.lmax - l;
        const int b = int(d * scale);
        return b < 0 ? 0 : (b >= kBins ? kBins - 1 : b);
    };
    auto member = [&](float l) {
        if (by_key) {
            const uint32_t k = key_of(l);
            return k >= klo && k <= khi;
        }
        return d_bin(l) == dbin;
    };
    for (;;) {
        if (p.n <= kCap) {
            if (tid == 0) sh->list_n = 0;
            cl.sync();
            Shared* lead = cl.of(0);
            for (int i = tid; i < n; i += kSampleThreads) {
                const float l = logit<T>(src, i);
                if (member(l)) {
                    const uint32_t at = atomicAdd(&lead->list_n, 1u);
                    if (at < kCap) lead->list[at] = (u64(key_of(l)) << 32) | (0xffffffffu - uint32_t(base + i));
                }
            }
            cl.sync();
            if (cl.rank == 0) {
                const int cnt = int(p.n);
                u64 me = 0, wm = 0, above = 0;
                int place = 0;
                if (tid < cnt) {
                    me = sh->list[tid];
                    const uint32_t k = uint32_t(me >> 32);
                    wm = masses ? w(__uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k)) : 0;
                    sh->list_w[tid] = wm;
                }
                __syncthreads();
                if (tid < cnt) {
                    for (int j = 0; j < cnt; ++j)
                        if (sh->list[j] > me) {
                            ++place;
                            above += sh->list_w[j];
                        }
                    const u64 ec = p.before_cnt + u64(place), em = p.before_mass + above;
                    const bool last = by_mass ? double(em) < goal && goal <= double(em + wm)
                                              : double(ec) < goal && goal <= double(ec + 1);
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
            return;
        }
        // the members' smallest and largest keys
        uint32_t kmin = 0xffffffffu, kmax = 0;
        for (int i = tid; i < n; i += kSampleThreads) {
            const float l = logit<T>(src, i);
            if (member(l)) {
                const uint32_t k = key_of(l);
                kmin = k < kmin ? k : kmin;
                kmax = k > kmax ? k : kmax;
            }
        }
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
            const u64 wk = masses ? w(__uint_as_float(kmin & 0x80000000u ? kmin & 0x7fffffffu : ~kmin)) : 0;
            u64 q;
            if (by_mass) {
                q = wk ? u64((goal - double(p.before_mass)) / double(wk)) : 1;
                q = q > 2 ? q - 2 : 1;
                while (q < p.n && double(p.before_mass + q * wk) < goal) ++q;
            } else {
                q = u64(goal) - p.before_cnt;
            }
            q = q < 1 ? 1 : (q > p.n ? p.n : q);
            const int32_t at = locate(
                cl, n, base, [&](int i) { return u64(key_of(logit<T>(src, i)) == kmin ? 1 : 0); },
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

template <class T>
__global__ void __launch_bounds__(kSampleThreads, 1) sample_kernel(const Sample p, int C, int chunk, int resident) {
    extern __shared__ __align__(16) char smem[];
    Shared* sh = reinterpret_cast<Shared*>(smem);
    char* data = smem + sizeof(Shared);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    Cluster cl{sh, C, int(blockIdx.x % unsigned(C))};
    const int64_t row = blockIdx.x / unsigned(C);
    if (tid < 32) sh->tab[tid] = exp2(double(tid) / 32.0);
    pdl_launch_dependents();
    pdl_wait();
    constexpr int es = Elem<T>::bytes;
    const int32_t base = cl.rank * chunk;
    const int n = p.V - base < chunk ? (p.V > base ? int(p.V - base) : 0) : chunk;
    const char* global = static_cast<const char*>(p.logits) + (row * p.V + base) * es;
    const char* src = resident ? data : global;

    // the row's largest (and, for the histogram's range, smallest) logit
    float mx = -INFINITY, mn = INFINITY;
    int32_t mi = 0x7fffffff;
    for (int i = tid; i < n; i += kSampleThreads) {
        using S = typename T::storage;
        if (resident) reinterpret_cast<S*>(data)[i] = reinterpret_cast<const S*>(global)[i];
        const float l = logit<T>(global, i);
        if (l > mx) {
            mx = l;
            mi = base + i;
        }
        if (l > -INFINITY) mn = fminf(mn, l);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float om = __shfl_xor_sync(0xffffffffu, mx, o);
        const int32_t oi = __shfl_xor_sync(0xffffffffu, mi, o);
        if (om > mx || (om == mx && oi < mi)) {
            mx = om;
            mi = oi;
        }
        mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    }
    if (lane == 0) {
        sh->fa[warp] = mx;
        sh->fb[warp] = mn;
        sh->ia[warp] = mi;
    }
    __syncthreads();
    if (warp == 0) {
        mx = sh->fa[lane];
        mn = sh->fb[lane];
        mi = sh->ia[lane];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float om = __shfl_xor_sync(0xffffffffu, mx, o);
            const int32_t oi = __shfl_xor_sync(0xffffffffu, mi, o);
            if (om > mx || (om == mx && oi < mi)) {
                mx = om;
                mi = oi;
            }
            mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
        }
        // every CTA of the cluster is running before its memory is written
        if (C > 1) cg::this_cluster().sync();
        if (lane < C) {
            Shared* o = cl.of(lane);
            o->cmax[cl.rank] = mx;
            o->cmin[cl.rank] = mn;
            o->cidx[cl.rank] = mi;
        }
    } else if (C > 1) {
        cg::this_cluster().sync();
    }
    cl.sync();
    mx = -INFINITY;
    mn = INFINITY;
    mi = 0x7fffffff;
    for (int r = 0; r < C; ++r) {
        if (sh->cmax[r] > mx || (sh->cmax[r] == mx && sh->cidx[r] < mi)) {
            mx = sh->cmax[r];
            mi = sh->cidx[r];
        }
        mn = fminf(mn, sh->cmin[r]);
    }
    const float temp = p.temperature ? p.temperature[row] : 1.f;
    if (!(temp > 0.f) || mx == -INFINITY) {  // (the same for the whole cluster)
        if (cl.rank == 0 && tid == 0) p.tokens[row] = mx == -INFINITY ? -1 : mi;
        return;  // no CTA touches another's memory after the barrier above
    }
    Weight w{mx, 29.9f * temp, 1.4426950408889634 / double(temp), sh->tab};
    const int32_t k = p.top_k ? p.top_k[row] : 0;
    const float tp = p.top_p ? p.top_p[row] : 1.f;
    float mp = p.min_p ? p.min_p[row] : 0.f;
    const double min_w = mp > 0.f ? double(fminf(mp, 1.f)) * kOne : 0.0;
    const bool use_k = k > 0 && k < p.V, use_p = tp < 1.f;  // (NaN: off)
    u64 cut = 0;  // every token
    if (use_k || use_p) {
        const float range = fminf(mx - mn, w.live);
        const float scale = range > 0.f ? float(kBins) / range : 0.f;
        auto d_bin = [&](float l) {
            if (!w.is_live(l)) return -1;
            const float d = l == mx ? 0.f : mx - l;
            const int b = int(d * scale);
            return b < 0 ? 0 : (b >= kBins ? kBins - 1 : b);
        };
        histogram<T>(cl, src, n, w, use_p, d_bin);
        double mass = 0.0;
        if (use_k) {
            const Pick pk = pick_bin(cl, false, double(k), 0, 0);
            mass = double(pk.total_mass);
            if (pk.bin >= 0) {
                resolve<T>(cl, src, n, base, w, scale, false, double(k), use_p, pk);
                cut = sh->cut;
                mass = double(sh->cut_mass);
                if (use_p && pk.n > kCap) histogram<T>(cl, src, n, w, true, d_bin);  // (resolve wrote over it)
            }
        }
        if (use_p) {
            if (!use_k) {
                // the whole weight: a goal beyond it picks nothing
                mass = double(pick_bin(cl, true, 1e300, 0, 0).total_mass);
            }
            const double goal = fmax(double(tp) * mass, 1.0);  // (p <= 0: the first token alone)
            const Pick pp = pick_bin(cl, true, goal, 0, 0);
            if (pp.bin >= 0) {
                resolve<T>(cl, src, n, base, w, scale, true, goal, true, pp);
                cut = sh->cut;
            }
        }
    }
    const uint32_t cut_key = uint32_t(cut >> 32);
    const float u = fminf(fmaxf(p.uniform[row], 0.f), 0.99999994f);
    const int32_t token = locate(
        cl, n, base,
        [&](int i) -> u64 {
            const float l = logit<T>(src, i);
            const uint32_t key = key_of(l);
            if (key < cut_key || ((u64(key) << 32) | (0xffffffffu - uint32_t(base + i))) < cut) return 0;
            const u64 v = w(l);
            return double(v) >= min_w ? v : 0;
        },
        [&](u64 total) { return double(u) * double(total); });
    if (cl.rank == 0 && tid == 0) p.tokens[row] = token;
}

template <class T>
cudaError_t run_sample(const Sample& p, cudaStream_t s) {
    const int sms = current_sm_count();
    const size_t room = 227 * 1024 - sizeof(Shared);
    // CTAs a row: enough to fill the GPU with few rows, at least 4096 tokens
    // each, and enough to hold the row where eight can.
    int C = 1;
    auto chunk_of = [&](int c) { return ((p.V + c - 1) / c + 7) / 8 * 8; };
    while (C < 8 && ((p.rows * C * 2 <= sms && chunk_of(C) > 8192) || size_t(chunk_of(C)) * Elem<T>::bytes > room)) C *= 2;
    const int64_t chunk = chunk_of(C);
    const bool resident = size_t(chunk) * Elem<T>::bytes <= room;
    const size_t smem = sizeof(Shared) + (resident ? size_t(chunk) * Elem<T>::bytes : 0);
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
