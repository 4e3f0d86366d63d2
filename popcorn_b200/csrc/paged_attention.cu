// paged_attention.cu — attention of the step's new tokens over a paged KV
// cache: the form for every type, head dim, page size and alignment. (16-bit
// types at head dims 64, 128 and 256 over pages of a multiple of 8 rows have
// the tensor-core kernel, paged_attention_tc.cu.)
//
// Token i of request r (n_r new tokens, s_r keys with them) sits at position
// p = s_r - n_r + i and attends to the keys j of its request that its mask
// allows: causal j <= p; sliding window also p - j < window, or j < sinks
// (the first tokens stay visible); bidirectional j < s_r. Key j is row
// j % ps of page block_table[r, j / ps]. Online softmax in fp32, one rounding
// of O / l. A row without a visible key is zero. Tokens of no request keep
// their rows. A page id outside the pages is not read and sets bit 5 of the
// device error word; its request's rows then mean nothing (here its keys are
// skipped, the tensor-core kernel takes them as zeros).
#include "async.cuh"
#include "common.cuh"
#include "dtype.cuh"
#include "launch.hpp"
#include "paged.cuh"
#include "popcorn.hpp"

namespace popcorn {

__device__ unsigned int g_pa_error_word;

namespace launch {

namespace {

constexpr int kPaThreads = 128;
constexpr int kPaWarps = 4;

// One CTA per (token, query head): four warps take the visible keys in turn,
// a lane every 32nd element of the row; their states merge at the end. Only
// visible rows are read, so nothing in a masked row can reach the output.
// Simple, and far from its floor: every (token, head) reads its whole context,
// a row at a time, with no reuse over a chunk's tokens or a group's heads. f32,
// 8 / 4 heads of 256: one request of 4096 keys 2.2 to 4.3 ms, 4 prompts of 2048
// 41 ms; 32 decoding at up to 8192 keys, 16 / 8 heads: 10 ms. 16-bit: 32
// decoding, heads of 96, 3.7 ms; a windowed chunk of 2000 over pages of 100
// rows 110 ms.
template <class T>
__global__ void __launch_bounds__(kPaThreads) paged_attention_any_kernel(const PagedAttention p) {
    constexpr int MAXE = 16;
    __shared__ float mm[kPaWarps], ll[kPaWarps];
    extern __shared__ float oo[];  // [kPaWarps][Hd]
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t t = blockIdx.x / unsigned(p.Nq);
    const int hq = int(blockIdx.x % unsigned(p.Nq));
    const int hkv = hq / (p.Nq / p.Nkv);
    // the request: the last r with query_start[r] <= t, if t is before its end
    int lo = 0, hi = p.R;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (p.query_start[mid] <= t) lo = mid;
        else hi = mid;
    }
    const Request rq = request(p, lo);
    if (t < rq.t0 || t >= rq.t0 + rq.n) return;
    const Span v = visible(p, rq, rq.len - rq.n + (t - rq.t0));
    const int64_t Hd = p.Hd;
    float q[MAXE], o[MAXE];
    const int64_t qrow = (t * p.Nq + hq) * Hd;
    const float qs = p.scale * 1.4426950408889634f;
#pragma unroll
    for (int i = 0; i < MAXE; ++i) {
        const int64_t d = lane + 32 * i;
        q[i] = d < Hd ? Elem<T>::load(p.q, qrow + d) * qs : 0.f;
        o[i] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    const int64_t count = v.sink + (v.hi - v.lo);
    for (int64_t u = warp; u < count; u += kPaWarps) {
        const int64_t j = u < v.sink ? u : v.lo + (u - v.sink);
        const int32_t page = p.table[int64_t(lo) * p.W + j / p.ps];
        if (page < 0 || page >= p.P) {
            if (lane == 0) atomicOr(&g_pa_error_word, 32u);
            continue;
        }
        const int64_t row = ((int64_t(page) * p.Nkv + hkv) * p.ps + j % p.ps) * Hd;
        float acc = 0.f;
#pragma unroll
        for (int i = 0; i < MAXE; ++i) {
            const int64_t d = lane + 32 * i;
            if (d < Hd) acc = fmaf(q[i], Elem<T>::load(p.k_pages, row + d), acc);
        }
        const float s = warp_sum(acc);
        const float mn = fmaxf(m, s);
        if (mn == -INFINITY && s == s) continue;  // (a score of -inf weighs nothing; a NaN counts)
        const float so = exp2f(m - mn), pv = exp2f(s - mn);
        l = l * so + pv;
        m = mn;
#pragma unroll
        for (int i = 0; i < MAXE; ++i) {
            const int64_t d = lane + 32 * i;
            if (d < Hd) o[i] = fmaf(pv, Elem<T>::load(p.v_pages, row + d), o[i] * so);
        }
    }
    if (lane == 0) {
        mm[warp] = m;
        ll[warp] = l;
    }
#pragma unroll
    for (int i = 0; i < MAXE; ++i) {
        const int64_t d = lane + 32 * i;
        if (d < Hd) oo[warp * Hd + d] = o[i];
    }
    __syncthreads();
    float M = -INFINITY, L = 0.f, f[kPaWarps];
    for (int w = 0; w < kPaWarps; ++w) M = fmaxf(M, mm[w]);
    for (int w = 0; w < kPaWarps; ++w) {
        f[w] = mm[w] == -INFINITY ? 0.f : exp2f(mm[w] - M);
        L += f[w] * ll[w];
    }
    for (int64_t d = tid; d < Hd; d += kPaThreads) {
        float O = 0.f;
        for (int w = 0; w < kPaWarps; ++w)
            if (mm[w] != -INFINITY) O += f[w] * oo[w * Hd + d];
        // (a NaN among the visible scores makes L NaN, and the row)
        store_one<T>(p.out, qrow + d, L == 0.f ? 0.f : O / L);
    }
}

}  // namespace

cudaError_t paged_attention_any(const PagedAttention& p, cudaStream_t s) {
    if (p.T == 0 || p.R == 0) return cudaSuccess;
    const dim3 g(unsigned(p.T * p.Nq)), b(kPaThreads);
    const size_t smem = size_t(kPaWarps) * p.Hd * 4;
    switch (p.dtype) {
    case PC_F32: return launch_k(paged_attention_any_kernel<TF32>, g, b, smem, s, p);
    case PC_F16: return launch_k(paged_attention_any_kernel<TF16>, g, b, smem, s, p);
    case PC_BF16: return launch_k(paged_attention_any_kernel<TBF16>, g, b, smem, s, p);
    }
    return cudaErrorInvalidValue;
}

uint32_t read_and_clear_pa_errors() {
    unsigned int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_pa_error_word, sizeof(v)) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    if (v) cudaMemcpyToSymbol(g_pa_error_word, &zero, sizeof(zero));
    return v;
}

namespace {
RegisterFunctions reg_pa({
    {"paged_attention", reinterpret_cast<const void*>(paged_attention_any_kernel<TF32>)},
    {"paged_attention_f16", reinterpret_cast<const void*>(paged_attention_any_kernel<TF16>)},
    {"paged_attention_bf16", reinterpret_cast<const void*>(paged_attention_any_kernel<TBF16>)},
});
}  // namespace

}  // namespace launch
}  // namespace popcorn
