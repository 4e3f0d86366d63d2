// paged.cu — the bookkeeping of a paged serving step: the block table, slot
// map and token positions built on the GPU from the requests' lengths, and
// the fused QKV product scattered into q rows and K/V pages (with the
// per-head norms and RoPE applied on the way).
#include "common.cuh"
#include "dtype.cuh"
#include "launch.hpp"
#include "paged.cuh"
#include "popcorn.hpp"

namespace popcorn {
namespace launch {

namespace {

// ---- PagedBatchBuild -------------------------------------------------------
//
// need_r = ceil((c_r + n_r) / ps) - ceil(c_r / ps) pages are taken from the
// free list for request r, in request order: P_r and N_r, the exclusive
// prefix sums of need and n, place its pages in the list and its tokens in
// the step. The first request that does not fit (free list, table width or
// token capacity) waits, and all after it.
//
// One cluster: every CTA scans the lengths by itself (a few loads; R is at
// most kMaxRequests) and keeps N, P and c in shared memory; after a cluster
// barrier — the outputs may be the inputs — the cluster's threads write the
// requests' rows, the new table entries and the tokens, each finding its
// request by binary search: a token a thread where there are threads enough,
// else four neighbouring ones. Latency-bound: 3.9 us for 32 decoding requests
// (5.6 with four tokens a thread, whose look-ups follow one another), 12 us
// for 509 prompts of 178000 tokens (15 with a search a token). One CTA up to
// kOneCtaTokens tokens, eight for more (2048 tokens of a prompt: 4.0 with one
// and 4.1 with eight, 4096 of eight prompts: 4.6 and 4.4).
constexpr int kBuildThreads = 1024;
constexpr int64_t kOneCtaTokens = 4096;
constexpr int kBuildCluster = 8;

__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

// Largest r with a[r] <= x, for a[0] <= x and ascending a[0..n].
__device__ __forceinline__ int find_owner(const int32_t* a, int n, int32_t x) {
    int lo = 0, hi = n;  // a[lo] <= x < a[hi] (a[n] > x by the caller)
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Positions and slots of the step's token rows, N neighbouring ones a thread: one search for them, and one page look-up unless
// a page or a request ends among them.
template <int N>
__device__ __forceinline__ void write_tokens(const PagedBatch& p, const int32_t* start, const int32_t* pstart,
                                             const int32_t* cached, int fail, int32_t total, int64_t head, int gt, int gn) {
    const uint32_t ps = uint32_t(p.ps);
    const bool wide = N == 4 && ((reinterpret_cast<uintptr_t>(p.positions) | reinterpret_cast<uintptr_t>(p.slots)) & 15u) == 0;
    for (int64_t t0 = N * int64_t(gt); t0 < p.T; t0 += N * int64_t(gn)) {
        int32_t position[N], slot[N];
        int r = t0 < total ? find_owner(start, fail, int32_t(t0)) : 0;
        uint32_t pos = 0, pg = 0, off = 0;
        int64_t page = -1;
        bool look = true;  // (pos, pg and off are new)
#pragma unroll
        for (int j = 0; j < N; ++j) {
            position[j] = 0;
            slot[j] = -1;
            const int64_t t = t0 + j;
            if (t >= total) continue;
            if (j == 0 || t >= start[r + 1]) {
                while (j > 0 && t >= start[r + 1]) ++r;
                pos = uint32_t(cached[r]) + uint32_t(int32_t(t) - start[r]);
                pg = pos / ps;
                off = pos - pg * ps;
                look = true;
            }
            if (look) {
                const uint32_t before = (uint32_t(cached[r]) + (ps - 1)) / ps;
                page = pg < before ? p.table[int64_t(r) * p.W + pg] : p.free_pages[head + pstart[r] + (pg - before)];
            }
            const int64_t sl = page * ps + off;
            position[j] = int32_t(pos);
            slot[j] = page >= 0 && sl <= 0x7fffffffll ? int32_t(sl) : -1;
            ++pos;
            look = ++off == ps;
            if (look) {
                off = 0;
                ++pg;
            }
        }
        if constexpr (N == 4) {
            if (wide && t0 + 4 <= p.T) {
                *reinterpret_cast<int4*>(p.positions + t0) = make_int4(position[0], position[1], position[2], position[3]);
                *reinterpret_cast<int4*>(p.slots + t0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
                continue;
            }
        }
        for (int j = 0; j < N && t0 + j < p.T; ++j) {
            p.positions[t0 + j] = position[j];
            p.slots[t0 + j] = slot[j];
        }
    }
}

__global__ void __launch_bounds__(kBuildThreads) paged_batch_build_kernel(const PagedBatch p) {
    extern __shared__ int32_t sm[];
    int32_t* start = sm;                    // [R + 1] first token of each request
    int32_t* pstart = start + p.R + 1;      // [R + 1] first free-list page of each request
    int32_t* cached = pstart + p.R + 1;     // [R]
    __shared__ long long wn[32], wp[32];
    __shared__ int s_fail;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_launch_dependents();
    pdl_wait();
    long long head = *p.free_head;
    head = head < 0 ? 0 : (head > p.F ? p.F : head);
    long long base_n = 0, base_p = 0;
    int fail = -1;  // first request that does not fit
    if (tid == 0) {
        start[0] = 0;
        pstart[0] = 0;
        s_fail = 0x7fffffff;
    }
    __syncthreads();
    for (int r0 = 0; r0 < p.R; r0 += kBuildThreads) {
        const int r = r0 + tid;
        long long c = 0, n = 0, after = 0, need = 0;
        if (r < p.R) {
            c = p.cached[r];
            n = p.added[r];
            c = c < 0 ? 0 : c;
            n = n < 0 ? 0 : n;
            cached[r] = int32_t(c);
            after = (c + n + p.ps - 1) / p.ps;
            need = after - (c + p.ps - 1) / p.ps;
        }
        // inclusive scans of n and need over the block
        long long sn = n, sp = need;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long a = __shfl_up_sync(0xffffffffu, sn, o), b = __shfl_up_sync(0xffffffffu, sp, o);
            if (lane >= o) {
                sn += a;
                sp += b;
            }
        }
        if (lane == 31) {
            wn[warp] = sn;
            wp[warp] = sp;
        }
        __syncthreads();
        if (warp == 0) {
            long long a = wn[lane], b = wp[lane];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
                if (lane >= o) {
                    a += x;
                    b += y;
                }
            }
            wn[lane] = a;
            wp[lane] = b;
        }
        __syncthreads();
        sn += base_n + (warp ? wn[warp - 1] : 0);
        sp += base_p + (warp ? wp[warp - 1] : 0);
        const bool fits = sn <= p.T && head + sp <= p.F && after <= p.W && c + n <= 0x7fffffffll;
        if (r < p.R) {
            if (!fits) atomicMin(&s_fail, r);
            start[r + 1] = int32_t(sn <= p.T ? sn : 0);  // (only read below the first failure)
            pstart[r + 1] = int32_t(head + sp <= p.F ? sp : 0);
        }
        base_n += wn[31];
        base_p += wp[31];
        __syncthreads();
        if (s_fail != 0x7fffffff) {
            fail = s_fail;
            for (int i = r0 + kBuildThreads + tid; i < p.R; i += kBuildThreads) {  // (the rest of the lengths)
                const int32_t x = p.cached[i];
                cached[i] = x < 0 ? 0 : x;
            }
            break;
        }
    }
    if (p.R == 0 || fail < 0) fail = p.R;
    __syncthreads();
    const int32_t total = start[fail], pages = pstart[fail];
    // the inputs are read: seq_lens may be cached, free_head_out may be free_head
    if (p.ctas > 1) cluster_sync_all();
    const int gt = blockIdx.x * kBuildThreads + tid, gn = p.ctas * kBuildThreads;
    for (int r = gt; r < p.R; r += gn) {
        const bool in = r < fail;
        const int32_t s0 = in ? start[r] : total, s1 = in ? start[r + 1] : total;
        p.seq_lens[r] = cached[r] + (s1 - s0);
        p.query_start[r + 1] = s1;
        p.last_rows[r] = s1 > 0 ? s1 - 1 : 0;
    }
    if (gt == 0) {
        p.query_start[0] = 0;
        *p.free_head_out = int32_t(head + pages);
        *p.admitted = fail;
    }
    for (int i = gt; i < pages; i += gn) {
        const int r = find_owner(pstart, fail, i);
        const long long before = (static_cast<long long>(cached[r]) + p.ps - 1) / p.ps;
        p.table[int64_t(r) * p.W + before + (i - pstart[r])] = p.free_pages[head + i];
    }
    if (p.T <= gn) write_tokens<1>(p, start, pstart, cached, fail, total, head, gt, gn);
    else write_tokens<4>(p, start, pstart, cached, fail, total, head, gt, gn);
}

// ---- PagedQKVScatter -------------------------------------------------------
//
// Head row x of token t: x' = RMSNorm(x) (optional), then rotate-half RoPE
// (optional, q and k), in fp32 with one rounding at the store; heads without
// either are copied bit for bit. Bandwidth-bound (qkv read once, written
// once): a group of L = Hd / 16 lanes owns a row, each lane eight neighbouring
// elements of the first half and the eight they pair with, so all accesses
// are 16 bytes, the rotation needs no exchange and the norm one shuffle
// reduction. 8191 tokens of 16 heads of 256 with RoPE: 28 us, 4.8 TB/s
// (8-byte accesses and 64-bit divisions: 33.5 us). (Two or four rows a group, all loaded at the start, are no
// faster: 30.5 and 34.3 us against 30 for 8191 tokens of 16 heads of 256.)
template <class T, int L>
__global__ void __launch_bounds__(256) paged_scatter_kernel(const PagedScatter p) {
    pdl_launch_dependents();
    constexpr uint32_t G = 256 / L;  // row groups of the CTA
    const uint32_t heads = uint32_t(p.Nq + 2 * p.Nkv), rows = uint32_t(p.T) * heads;
    const uint32_t g = blockIdx.x * G + threadIdx.x / L;
    const int li = threadIdx.x % L;
    // (a group past the end repeats the last row without storing: its warp's shuffles need it)
    const uint32_t row = g < rows ? g : rows - 1, t = row / heads, h = row - t * heads;
    const bool is_q = h < uint32_t(p.Nq), is_v = h >= uint32_t(p.Nq + p.Nkv);
    const bool norm = is_v ? p.norm_v : p.qk_norm;
    const bool rope = !is_v && p.cos_t;
    const float* w = is_v || !norm ? nullptr : (is_q ? p.q_norm : p.k_norm);
    pdl_wait();
    // every load before the first use
    const uint16_t* src = static_cast<const uint16_t*>(p.qkv) + int64_t(row) * (16 * L) + 8 * li;
    uint4 a = *reinterpret_cast<const uint4*>(src), b = *reinterpret_cast<const uint4*>(src + 8 * L);
    const int32_t slot = is_q ? -1 : p.slots[t];
    float4 c[2], s[2];
    if (rope) {
        const float4* ct = reinterpret_cast<const float4*>(p.cos_t + int64_t(t) * (8 * L) + 8 * li);
        const float4* st = reinterpret_cast<const float4*>(p.sin_t + int64_t(t) * (8 * L) + 8 * li);
        c[0] = ct[0], c[1] = ct[1], s[0] = st[0], s[1] = st[1];
    }
    if (p.qk_norm || p.norm_v || p.cos_t) {  // (the same for every lane: rows of a warp may differ in `norm`)
        float x[8], y[8];
        unpack8<T>(a, x);
        unpack8<T>(b, y);
        if (p.qk_norm || p.norm_v) {
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ss += x[e] * x[e] + y[e] * y[e];
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (norm) {
                const float r = rsqrtf(ss / float(p.Hd) + p.eps);
                const float one = w && p.add_one ? 1.f : 0.f;
#pragma unroll
                for (int e = 0; e < 8; e += 4) {
                    float4 wx = make_float4(1.f, 1.f, 1.f, 1.f), wy = wx;
                    if (w) {
                        wx = *reinterpret_cast<const float4*>(w + 8 * li + e);
                        wy = *reinterpret_cast<const float4*>(w + 8 * L + 8 * li + e);
                    }
                    x[e] = x[e] * r * (wx.x + one);
                    x[e + 1] = x[e + 1] * r * (wx.y + one);
                    x[e + 2] = x[e + 2] * r * (wx.z + one);
                    x[e + 3] = x[e + 3] * r * (wx.w + one);
                    y[e] = y[e] * r * (wy.x + one);
                    y[e + 1] = y[e + 1] * r * (wy.y + one);
                    y[e + 2] = y[e + 2] * r * (wy.z + one);
                    y[e + 3] = y[e + 3] * r * (wy.w + one);
                }
            }
        }
        if (rope) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float cc = reinterpret_cast<const float*>(c)[e], sn = reinterpret_cast<const float*>(s)[e];
                const float u = x[e] * cc - y[e] * sn;
                y[e] = y[e] * cc + x[e] * sn;
                x[e] = u;
            }
        }
        if (norm || rope) {  // (others stay bit for bit)
            a = make_uint4(cvt_pair<T>(x[0], x[1]), cvt_pair<T>(x[2], x[3]), cvt_pair<T>(x[4], x[5]), cvt_pair<T>(x[6], x[7]));
            b = make_uint4(cvt_pair<T>(y[0], y[1]), cvt_pair<T>(y[2], y[3]), cvt_pair<T>(y[4], y[5]), cvt_pair<T>(y[6], y[7]));
        }
    }
    if (g >= rows) return;
    uint16_t* dst;
    if (is_q) {
        dst = static_cast<uint16_t*>(p.q_out) + (int64_t(t) * p.Nq + h) * p.Hd;
    } else {
        if (slot < 0 || slot >= p.P * p.ps) return;
        const uint32_t hk = is_v ? h - uint32_t(p.Nq + p.Nkv) : h - uint32_t(p.Nq);
        const uint32_t page = uint32_t(slot) / uint32_t(p.ps), off = uint32_t(slot) - page * uint32_t(p.ps);
        dst = static_cast<uint16_t*>(is_v ? p.v_pages : p.k_pages) + ((int64_t(page) * p.Nkv + hk) * p.ps + off) * p.Hd;
    }
    *reinterpret_cast<uint4*>(dst + 8 * li) = a;
    *reinterpret_cast<uint4*>(dst + 8 * L + 8 * li) = b;
}

// Any dtype, any even or (without RoPE) odd Hd, any alignment: a warp a row.
template <class T>
__global__ void __launch_bounds__(256) paged_scatter_any_kernel(const PagedScatter p) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int heads = p.Nq + 2 * p.Nkv;
    const int64_t rows = p.T * heads, H2 = p.Hd / 2;
    for (int64_t row = (blockIdx.x * int64_t(blockDim.x) + threadIdx.x) >> 5; row < rows;
         row += (int64_t(gridDim.x) * blockDim.x) >> 5) {
        const int64_t t = row / heads;
        const int h = int(row % heads);
        const bool is_q = h < p.Nq, is_v = h >= p.Nq + p.Nkv;
        const int64_t src = row * p.Hd;
        void* out = p.q_out;
        int64_t dst = (t * p.Nq + h) * p.Hd;
        if (!is_q) {
            const int64_t slot = p.slots[t];
            if (slot < 0 || slot >= p.P * p.ps) continue;  // (the whole warp)
            const int hk = is_v ? h - p.Nq - p.Nkv : h - p.Nq;
            out = is_v ? p.v_pages : p.k_pages;
            dst = ((slot / p.ps * p.Nkv + hk) * p.ps + slot % p.ps) * p.Hd;
        }
        const bool norm = is_v ? p.norm_v : p.qk_norm;
        const bool rope = !is_v && p.cos_t;
        if (!norm && !rope) {
            using S = typename T::storage;
            for (int64_t d = lane; d < p.Hd; d += 32)
                static_cast<S*>(out)[dst + d] = static_cast<const S*>(p.qkv)[src + d];
            continue;
        }
        float r = 1.f;
        if (norm) {
            float ss = 0.f;
            for (int64_t d = lane; d < p.Hd; d += 32) {
                const float x = Elem<T>::load(p.qkv, src + d);
                ss += x * x;
            }
            r = rsqrtf(warp_sum(ss) / float(p.Hd) + p.eps);
        }
        const float* w = is_v || !norm ? nullptr : (is_q ? p.q_norm : p.k_norm);
        auto value = [&](int64_t d) {
            float x = Elem<T>::load(p.qkv, src + d) * r;
            if (w) x *= p.add_one ? 1.f + w[d] : w[d];
            return x;
        };
        if (!rope) {
            for (int64_t d = lane; d < p.Hd; d += 32) store_one<T>(out, dst + d, value(d));
            continue;
        }
        for (int64_t d = lane; d < H2; d += 32) {
            const float c = p.cos_t[t * H2 + d], s = p.sin_t[t * H2 + d];
            const float x = value(d), y = value(H2 + d);
            store_one<T>(out, dst + d, x * c - y * s);
            store_one<T>(out, dst + H2 + d, y * c + x * s);
        }
    }
}

template <class T, int L>
cudaError_t run_scatter(const PagedScatter& p, cudaStream_t s) {
    constexpr int64_t G = 256 / L;
    const int64_t rows = p.T * (p.Nq + 2 * p.Nkv);
    return launch_k(paged_scatter_kernel<T, L>, dim3(unsigned((rows + G - 1) / G)), dim3(256), 0, s, p);
}

template <class T>
cudaError_t run_scatter_16(const PagedScatter& p, cudaStream_t s) {
    if (p.Hd == 256) return run_scatter<T, 16>(p, s);
    if (p.Hd == 128) return run_scatter<T, 8>(p, s);
    return run_scatter<T, 4>(p, s);
}

}  // namespace

cudaError_t paged_batch_build(const PagedBatch& q, cudaStream_t s) {
    PagedBatch p = q;
    const size_t smem = size_t(3 * int64_t(p.R) + 2) * 4;
    static DeviceOnce once;
    cudaError_t e = once.run([&] { return allow_smem(paged_batch_build_kernel, (3 * size_t(kMaxRequests) + 2) * 4); });
    if (e != cudaSuccess) return e;
    p.ctas = p.T > kOneCtaTokens ? kBuildCluster : 1;
    return launch_cluster(paged_batch_build_kernel, dim3(unsigned(p.ctas)), dim3(kBuildThreads), unsigned(p.ctas), smem, s, p);
}

cudaError_t paged_qkv_scatter(const PagedScatter& p, cudaStream_t s) {
    if (p.T == 0) return cudaSuccess;
    const bool vec = p.dtype != PC_F32 && (p.Hd == 64 || p.Hd == 128 || p.Hd == 256) && p.T * (p.Nq + 2 * p.Nkv) <= 0x7fffffff &&
                     aligned16(p.qkv) && aligned16(p.q_out) && aligned16(p.k_pages) && aligned16(p.v_pages) &&
                     aligned16(p.cos_t) && aligned16(p.sin_t) && aligned16(p.q_norm) && aligned16(p.k_norm);  // (or NULL)
    if (vec) return p.dtype == PC_BF16 ? run_scatter_16<TBF16>(p, s) : run_scatter_16<TF16>(p, s);
    const dim3 g(grid_for(p.T * (p.Nq + 2 * p.Nkv) * 32, 256, current_sm_count())), b(256);
    switch (p.dtype) {
    case PC_F32: return launch_k(paged_scatter_any_kernel<TF32>, g, b, 0, s, p);
    case PC_F16: return launch_k(paged_scatter_any_kernel<TF16>, g, b, 0, s, p);
    case PC_BF16: return launch_k(paged_scatter_any_kernel<TBF16>, g, b, 0, s, p);
    }
    return cudaErrorInvalidValue;
}

namespace {
RegisterFunctions reg_paged({
    {"paged_batch_build", reinterpret_cast<const void*>(paged_batch_build_kernel)},
    {"paged_qkv_scatter", reinterpret_cast<const void*>(paged_scatter_any_kernel<TF32>)},
    {"paged_qkv_scatter_bf16", reinterpret_cast<const void*>(paged_scatter_kernel<TBF16, 16>)},
    {"paged_qkv_scatter_f16", reinterpret_cast<const void*>(paged_scatter_kernel<TF16, 16>)},
});
}  // namespace

}  // namespace launch
}  // namespace popcorn
