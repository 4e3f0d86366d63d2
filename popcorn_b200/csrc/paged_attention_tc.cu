// paged_attention_tc.cu — PagedAttention on the 5th-generation tensor cores
// (bf16 / f16, head dims 64, 128 and 256, pages of a multiple of 8 rows).
//
// The step's work is cut into items: (request, KV head, tile of up to 128
// query rows), a row being one (token, query head of the group) pair, so the
// heads that share a KV head share its K/V reads. An item's units are the
// 128-key tiles that some row of it sees: those of the sink tokens, then
// those from the first row's window start to the last row's position.
// Every CTA of one wave takes an equal run of consecutive units — ragged
// lengths, long contexts with one token and long chunks all fill the GPU —
// and cuts an item where its run ends; the pieces' (m, l, O) go to scratch
// and a second kernel joins them in order (the cut depends on the lengths
// alone, so results repeat bit for bit). The plan is computed by every CTA
// from the lengths on the device.
//
// In a CTA: warp 0 loads Q and the 64-key halves of K and V tiles by TMA
// (128-byte swizzle, one box per page run) into one ring in the order K(0),
// K(1) V(0), K(2) V(1), ...; warp 1 issues S = Q.K^T into the next of NS
// accumulators in tensor memory and O += P.V, whichever is ready; warps 4-11
// (two threads a row, 64 keys each) turn S into P = 2^(c S - m): P is packed
// into the type and written back over S, from where the second product reads
// it as its A operand, so it never passes through shared memory. A ring slot
// holds 8-key groups of [Hd/64][8 keys][128 B], so any page size that is a
// multiple of 8 gives one layout (group stride Hd/64 KB) and 128 keys in
// neighbouring slots are one operand.
//
// The running max is kept until it grows by more than 2^8 (P <= 256 then; O
// and l use the same max, so O / l is exact for any); the two threads of a
// row and all rows agree on that by one barrier vote a tile. P is rounded to
// the type once: as far from the exact weights as the output's own rounding
// is from the exact output (half a step each); sums, m, l and O are fp32.
//
// Keys that no row of the item sees are never loaded (zero-filled boxes, so
// freed pages may hold anything). In tiles that cross a mask edge V rows that
// no row sees are zeroed, and a value that is not finite, in a row that some
// see, is taken out of the product and added to their outputs alone: 0 * inf
// would be NaN for the others.
//
// Every mbarrier wait is bounded; on give-up the CTA sets the error word,
// drains, frees its tensor memory and leaves.
#include "async.cuh"
#include "common.cuh"
#include "dtype.cuh"
#include "launch.hpp"
#include "paged.cuh"
#include "popcorn.hpp"
#include "tcgen05.cuh"

namespace popcorn {

__device__ unsigned int g_pt_error_word;

namespace launch {

namespace {

using namespace tc;

constexpr int kM = 128;          // query rows of an item
constexpr int kN = 128;          // keys of a unit
constexpr int kSlotKeys = 64;    // keys of a ring slot
constexpr int kPtThreads = 384;  // warps: 0 TMA, 1 MMA, 4-11 softmax
constexpr int kSoftThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kGrow = 8.0f;  // log2 of the growth of a row's max that is let pass
constexpr uint32_t kTmem = 512;

template <int HD>
struct Shape {
    static constexpr int ATOMS = HD / 64;
    static constexpr int NS = HD == 256 ? 2 : 3;  // S accumulators: NS * 128 + HD <= 512 columns
    static constexpr int GROUP = ATOMS * 1024;    // bytes of 8 keys
    static constexpr int SLOT = 8 * GROUP;
    static constexpr int NSLOT = HD == 256 ? 5 : (HD == 128 ? 12 : 20);
    static constexpr int Q_BLOCK = kM * 128;
    static constexpr int Q_BYTES = ATOMS * Q_BLOCK;
    static constexpr uint32_t O_COL = NS * kN;
    static constexpr size_t SMEM = size_t(Q_BYTES) + size_t(NSLOT) * SLOT + 1024;
};
static_assert(Shape<64>::NSLOT * Shape<64>::SLOT >= (kMaxRequests + 1) * 8, "the plan's sums fit the ring");

// A piece of an item that was cut (written by the CTA where it begins).
struct Cut {
    int64_t tok0;
    int32_t ntok, head;
    int32_t last;    // CTA of the final piece
    int32_t begins;  // 0: no item that begins in this CTA was cut
};

struct TcArgs {
    PagedAttention p;
    int tpt;        // tokens of an item: 128 / group size
    int group;      // query heads of a KV head
    int box_groups; // 8-key groups of a TMA box
    int rows_cap;   // rows of a scratch slot
    float c;        // scale * log2(e)
    int64_t groups; // 8-row groups of the pages (past the end: zero fill)
    float* po;      // [2 * CTAs][rows_cap][HD]
    float* pml;     // [2 * CTAs][rows_cap][2]
    Cut* cuts;      // [CTAs]
};

struct Item {
    int r, h, mt;
    int64_t tok0;  // first token row
    int ntok;
    int64_t pos0;          // position of its first token
    int64_t lo, hi, sink;  // keys that some row sees: [0, sink) and [lo, hi)
    int64_t len;
    int t_lo, ns, units;  // tiles [0, ns) and from t_lo on
    int u0, u1;           // this CTA's share
    int64_t start;        // the item's first unit in the step's order
};

__device__ __forceinline__ void item_span(const TcArgs& a, const Request& rq, int mt, Item& it) {
    const PagedAttention& p = a.p;
    const int64_t i0 = int64_t(mt) * a.tpt;
    it.mt = mt;
    it.tok0 = rq.t0 + i0;
    it.ntok = int(rq.n - i0 < a.tpt ? rq.n - i0 : a.tpt);
    it.pos0 = rq.len - rq.n + i0;
    it.len = rq.len;
    const Span first = visible(p, rq, it.pos0), last = visible(p, rq, it.pos0 + it.ntok - 1);
    it.lo = first.lo;
    it.hi = last.hi;
    it.sink = last.sink;
    it.t_lo = int(it.lo / kN);
    const int t_hi = int((it.hi + kN - 1) / kN);
    int ns = int((it.sink + kN - 1) / kN);
    it.ns = ns < it.t_lo ? ns : it.t_lo;
    const int u = it.ns + (t_hi > it.t_lo ? t_hi - it.t_lo : 0);
    it.units = u > 1 ? u : 1;  // (rows without a key are written too)
}

struct Start {
    int r, h, mt, u;
    int64_t unit, left;
};

// The CTA's items in order; every role walks them by itself.
struct Walk {
    const TcArgs& a;
    Request rq;
    int r, h, mt, u, ntiles;
    int64_t unit, left;

    __device__ __forceinline__ Walk(const TcArgs& args, const Start& s)
        : a(args), r(s.r), h(s.h), mt(s.mt), u(s.u), unit(s.unit), left(s.left) {
        if (left > 0) load();
    }
    __device__ __forceinline__ void load() {
        rq = request(a.p, r);
        ntiles = int((rq.n + a.tpt - 1) / a.tpt);
    }
    __device__ __forceinline__ bool next(Item& it) {
        if (left <= 0) return false;
        item_span(a, rq, mt, it);
        it.r = r;
        it.h = h;
        it.u0 = u;
        it.u1 = it.units - u <= left ? it.units : u + int(left);
        it.start = unit - u;
        unit += it.u1 - u;
        left -= it.u1 - u;
        if (it.u1 < it.units) {
            u = it.u1;  // (left is 0)
            return true;
        }
        u = 0;
        if (++mt == ntiles) {
            mt = 0;
            if (++h == a.p.Nkv) {
                h = 0;
                if (left > 0) {
                    do ++r;
                    while (r < a.p.R && request(a.p, r).n == 0);
                    if (r < a.p.R) load();
                    else left = 0;
                }
            }
        }
        return true;
    }
};

__device__ __forceinline__ int tile_of(const Item& it, int u) { return u < it.ns ? u : it.t_lo + (u - it.ns); }

// Every row of the item sees every key of the tile at key0.
__device__ __forceinline__ bool tile_open(const TcArgs& a, const Item& it, int64_t key0) {
    const PagedAttention& p = a.p;
    const int64_t end = p.mask_kind == 2 ? it.len : (it.pos0 + 1 < it.len ? it.pos0 + 1 : it.len);
    if (key0 + kN > end) return false;
    if (p.mask_kind != 1) return true;
    return key0 >= it.pos0 + it.ntok - 1 - p.window + 1 || key0 + kN <= p.sinks;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::
            "r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
        : "memory");
}

// A from tensor memory (16-bit pairs, a row a lane), B from shared memory.
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// As smem_desc_sw128, with the 8-row groups `stride` bytes apart.
__device__ __forceinline__ uint64_t desc_k(uint32_t saddr, uint32_t stride) {
    return (smem_desc_sw128(saddr) & ~(uint64_t(0x3fff) << 32)) | (uint64_t(stride >> 4) << 32);
}
// B stored [K, N]: 8-K-row groups `stride` bytes apart, 64-element blocks of N 1024 bytes apart.
__device__ __forceinline__ uint64_t desc_mn(uint32_t saddr, uint32_t stride) {
    return (smem_desc_sw128_mn(saddr, 1024) & ~(uint64_t(0x3fff) << 32)) | (uint64_t(stride >> 4) << 32);
}

// Warp-uniform bounded wait (seconds of polling); false once any role gave up.
__device__ __forceinline__ bool wait_bar(uint64_t& bar, uint32_t parity, int lane, volatile int& abort) {
    int ok = 0;
    if (lane == 0) {
        const uint32_t b = smem_u32(&bar);
        for (uint32_t i = 0; i < (1u << 26); ++i) {
            if (mbar_test_wait(b, parity)) {
                ok = 1;
                break;
            }
            if ((i & 1023u) == 1023u && abort) break;
        }
        if (!ok && !abort) {
            atomicOr(&g_pt_error_word, 1u);
            abort = 1;
        }
    }
    return __shfl_sync(0xffffffffu, ok, 0) != 0;
}

// Barrier `id` over the softmax threads; true where any of them says so.
__device__ __forceinline__ bool soft_any(int id, bool mine) {
    uint32_t any;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.or.pred q, %2, %3, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(any)
        : "r"(uint32_t(mine)), "r"(id), "r"(kSoftThreads)
        : "memory");
    return any != 0;
}

// A half word pair that holds an infinity or a NaN.
template <class T>
__device__ __forceinline__ bool not_finite2(uint32_t w) {
    constexpr uint32_t e = T::code == TBF16::code ? 0x7f80u : 0x7c00u;
    return (w & e) == e || ((w >> 16) & e) == e;
}
template <class T>
__device__ __forceinline__ uint32_t finite_part(uint32_t w) {
    constexpr uint32_t e = T::code == TBF16::code ? 0x7f80u : 0x7c00u;
    if ((w & e) == e) w &= 0xffff0000u;
    if (((w >> 16) & e) == e) w &= 0x0000ffffu;
    return w;
}

template <int HD, class T>
__global__ void __launch_bounds__(kPtThreads, 1)
    paged_attention_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_q1,
                              const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                              const __grid_constant__ TcArgs a) {
    using S = Shape<HD>;
    constexpr int NS = S::NS, NSLOT = S::NSLOT, ATOMS = S::ATOMS;
    constexpr bool BF = T::code == TBF16::code;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t q_full, q_empty, full[NSLOT], empty[NSLOT], s_full[NS], p_full[NS], pv_done[NS], o_free;
    __shared__ uint32_t s_tmem;
    __shared__ volatile int s_abort;
    __shared__ Start s_start;
    __shared__ long long s_scan[kPtThreads / 32];
    __shared__ float s_mx[2][kM];  // a row's two maxima, at an item's end its two sums
    __shared__ uint32_t s_poison[3][4];

    pdl_launch_dependents();
    unsigned char* sq =
        reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char* ring = sq + S::Q_BYTES;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const PagedAttention& p = a.p;

    if (tid == 0) {
        mbar_init(smem_u32(&q_full), 1);
        mbar_init(smem_u32(&q_empty), 1);
        for (int i = 0; i < NSLOT; ++i) {
            mbar_init(smem_u32(&full[i]), 1);
            mbar_init(smem_u32(&empty[i]), 1);
        }
        for (int i = 0; i < NS; ++i) {
            mbar_init(smem_u32(&s_full[i]), 1);
            mbar_init(smem_u32(&pv_done[i]), 1);
            mbar_init(smem_u32(&p_full[i]), kSoftThreads / 32);
        }
        mbar_init(smem_u32(&o_free), kSoftThreads / 32);
        s_abort = 0;
        mbar_fence_init();
    }
    if (tid < 12) (&s_poison[0][0])[tid] = 0;
    if (warp == 0) tmem_alloc(smem_u32(&s_tmem), kTmem);
    pdl_wait();

    // ---- the plan: sums of the requests' units, and where this CTA begins ----
    long long* cum = reinterpret_cast<long long*>(ring);  // [R + 1], before any copy uses the ring
    auto head_units = [&](const Request& rq, int from, int step) {
        long long u = 0;
        const int nt = int((rq.n + a.tpt - 1) / a.tpt);
        Item it;
        for (int mt = from; mt < nt; mt += step) {
            item_span(a, rq, mt, it);
            u += it.units;
        }
        return u;
    };
    if (p.R <= 8 * (kPtThreads / 32)) {  // a warp a request: long chunks have many tiles
        for (int r = warp; r < p.R; r += kPtThreads / 32) {
            long long u = head_units(request(p, r), lane, 32);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) u += __shfl_xor_sync(0xffffffffu, u, o);
            if (lane == 0) cum[r + 1] = u * p.Nkv;
        }
    } else {
        for (int r = tid; r < p.R; r += kPtThreads) cum[r + 1] = head_units(request(p, r), 0, 1) * p.Nkv;
    }
    if (tid == 0) cum[0] = 0;
    __syncthreads();
    {
        const int per = (p.R + kPtThreads - 1) / kPtThreads;
        const int r0 = tid * per < p.R ? tid * per : p.R, r1 = r0 + per < p.R ? r0 + per : p.R;
        long long sum = 0;
        for (int r = r0; r < r1; ++r) sum += cum[r + 1];
        long long incl = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long x = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += x;
        }
        if (lane == 31) s_scan[warp] = incl;
        __syncthreads();
        long long run = incl - sum;
        for (int w = 0; w < warp; ++w) run += s_scan[w];
        for (int r = r0; r < r1; ++r) {
            run += cum[r + 1];
            cum[r + 1] = run;
        }
    }
    __syncthreads();
    const long long U = cum[p.R];
    const long long ctas = U < (long long)gridDim.x ? U : (long long)gridDim.x;
    if (warp == 0) {
        Start s{0, 0, 0, 0, 0, 0};
        if ((long long)blockIdx.x < ctas) {
            const long long u = blockIdx.x * U / ctas;
            s.unit = u;
            s.left = (blockIdx.x + 1) * U / ctas - u;
            int lo = 0, hi = p.R;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (cum[mid] <= u) lo = mid;
                else hi = mid;
            }
            s.r = lo;
            const long long per_head = (cum[lo + 1] - cum[lo]) / p.Nkv;
            long long rem = u - cum[lo];
            s.h = int(rem / per_head);
            rem -= s.h * per_head;
            // the item: 32 tiles at a time
            const Request rq = request(p, lo);
            const int nt = int((rq.n + a.tpt - 1) / a.tpt);
            for (int mt0 = 0; mt0 < nt; mt0 += 32) {
                Item it;
                it.units = 0;
                if (mt0 + lane < nt) item_span(a, rq, mt0 + lane, it);
                long long incl = it.units;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const long long x = __shfl_up_sync(0xffffffffu, incl, o);
                    if (lane >= o) incl += x;
                }
                const unsigned hit = __ballot_sync(0xffffffffu, incl > rem);
                if (hit) {
                    const int l = __ffs(int(hit)) - 1;
                    s.mt = mt0 + l;
                    s.u = int(rem - __shfl_sync(0xffffffffu, incl - it.units, l));
                    break;
                }
                rem -= __shfl_sync(0xffffffffu, incl, 31);
            }
        }
        if (lane == 0) s_start = s;
    }
    tc_fence_before();
    fence_async_smem();  // the sums' readers are done before copies land there
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    const Start start = s_start;

    if (warp == 0) {
        // ---- loads ----
        Walk walk(a, start);
        Item it, prev;
        const uint32_t ring_a = smem_u32(ring);
        const int boxes = 8 / a.box_groups;
        const uint32_t box_bytes = uint32_t(a.box_groups * S::GROUP);
        const uint32_t ps = uint32_t(p.ps);
        bool ok = true;
        int issued = 0;  // ring positions issued
        // This lane's box of the 64 keys at key0: its first group, or past the end for keys that no row sees.
        auto group_of = [&](const Item& t, int64_t key0) -> int {
            int64_t g = a.groups;
            const int64_t k0 = key0 + lane * a.box_groups * 8;
            if (lane < boxes && k0 < t.hi && (k0 + a.box_groups * 8 > t.lo || k0 < t.sink)) {
                const uint32_t k = uint32_t(k0);
                const int32_t page = p.table[int64_t(t.r) * p.W + k / ps];
                if (page >= 0 && page < p.P) g = ((int64_t(page) * p.Nkv + t.h) * p.ps + k % ps) / 8;
                else atomicOr(&g_pt_error_word, 32u);
            }
            return int(g);
        };
        auto put = [&](const Item& t, int u, int pos, const CUtensorMap* map) {
#pragma unroll 1
            for (int half = 0; half < 2 && ok; ++half) {
                const int64_t key0 = int64_t(tile_of(t, u)) * kN + half * kSlotKeys;
                const int g = group_of(t, key0);
                const int q = pos + half, slot = q % NSLOT;
                ok = wait_bar(empty[slot], (uint32_t(q / NSLOT) & 1u) ^ 1u, lane, s_abort);
                if (!ok) return;
                const uint32_t bar = smem_u32(&full[slot]);
                if (lane == 0) mbar_expect_tx(bar, S::SLOT);
                __syncwarp();
                if (lane < boxes) tma_load_4d(ring_a + slot * S::SLOT + lane * box_bytes, map, 0, 0, 0, g, bar);
                issued = q + 1;
            }
        };
        int j = 0, items = 0, prev_u = -1;
        bool q_pending = false;
        while (ok && walk.next(it)) {
            for (int u = it.u0; u < it.u1 && ok; ++u, ++j) {
                if (u == it.u0) {
                    if (j > 0) put(prev, prev_u, 4 * j - 2, &map_v);
                    if (!ok) break;
                    ok = wait_bar(q_empty, (uint32_t(items) & 1u) ^ 1u, lane, s_abort);
                    if (!ok) break;
                    if (lane == 0) {
                        const bool one = it.ntok == 1;
                        const uint32_t rows = uint32_t(one ? a.group : a.group * a.tpt);
                        mbar_expect_tx(smem_u32(&q_full), rows * 128 * ATOMS);
#pragma unroll
                        for (int at = 0; at < ATOMS; ++at)
                            tma_load_4d(smem_u32(sq + at * S::Q_BLOCK), one ? &map_q1 : &map_q, 0, it.h * a.group,
                                        int(it.tok0), at, smem_u32(&q_full));
                    }
                    __syncwarp();
                    q_pending = true;
                    ++items;
                    put(it, u, 4 * j, &map_k);
                } else {
                    put(it, u, 4 * j - 2, &map_k);
                    put(prev, prev_u, 4 * j, &map_v);
                }
                prev = it;
                prev_u = u;
            }
        }
        if (ok && j > 0) put(prev, prev_u, 4 * j - 2, &map_v);
        if (!ok) {
            s_abort = 1;
            // leave no copy in flight
            if (lane == 0) {
                if (q_pending) mbar_wait(smem_u32(&q_full), uint32_t(items - 1) & 1u, &g_pt_error_word);
                for (int q = issued - NSLOT < 0 ? 0 : issued - NSLOT; q < issued; ++q)
                    mbar_wait(smem_u32(&full[q % NSLOT]), uint32_t(q / NSLOT) & 1u, &g_pt_error_word);
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            // ---- MMA issue ----
            constexpr uint32_t idesc_s = make_idesc(BF, kM, kN, false), idesc_h = make_idesc(BF, kM, kSlotKeys, false);
            constexpr uint32_t idesc_o = make_idesc(BF, kM, HD, true);
            const uint32_t q_base = smem_u32(sq), ring_a = smem_u32(ring);
            auto is_full = [&](int q) {
                return mbar_test_wait(smem_u32(&full[q % NSLOT]), uint32_t(q / NSLOT) & 1u);
            };
            Walk walk_s(a, start), walk_p(a, start);
            Item is, ip;
            const int n = int(start.left);
            int ns = 0, np = 0;
            int us = 0, up = 0, items_s = 0, items_p = 0;
            bool ok = true;
            if (n > 0) {
                walk_s.next(is);
                walk_p.next(ip);
                us = is.u0;
                up = ip.u0;
            }
            uint32_t idle = 0;
            while (np < n && !s_abort) {
                bool progressed = false;
                if (ns < n && ns < np + NS) {
                    const int buf = ns % NS;
                    const bool first = us == is.u0;
                    const int q0 = first ? 4 * ns : 4 * ns - 2, q1 = q0 + 1;
                    if ((ns < NS || mbar_test_wait(smem_u32(&pv_done[buf]), uint32_t(ns / NS - 1) & 1u)) &&
                        (!first || mbar_test_wait(smem_u32(&q_full), uint32_t(items_s) & 1u)) && is_full(q0) && is_full(q1)) {
                        tc_fence_after();
                        const int s0 = q0 % NSLOT, s1 = q1 % NSLOT;
                        const uint32_t k0 = ring_a + s0 * S::SLOT, k1 = ring_a + s1 * S::SLOT;
                        const uint32_t d = tmem + uint32_t(buf * kN);
                        if (s1 == s0 + 1) {
#pragma unroll
                            for (int kk = 0; kk < HD / 16; ++kk)
                                tc_mma(d, smem_desc_sw128(q_base + (kk >> 2) * S::Q_BLOCK + (kk & 3) * 32),
                                       desc_k(k0 + (kk >> 2) * 1024 + (kk & 3) * 32, S::GROUP), idesc_s, kk > 0 ? 1u : 0u);
                        } else {  // the tile wraps round the ring: two halves
#pragma unroll
                            for (int kk = 0; kk < HD / 16; ++kk)
                                tc_mma(d, smem_desc_sw128(q_base + (kk >> 2) * S::Q_BLOCK + (kk & 3) * 32),
                                       desc_k(k0 + (kk >> 2) * 1024 + (kk & 3) * 32, S::GROUP), idesc_h, kk > 0 ? 1u : 0u);
#pragma unroll
                            for (int kk = 0; kk < HD / 16; ++kk)
                                tc_mma(d + kSlotKeys, smem_desc_sw128(q_base + (kk >> 2) * S::Q_BLOCK + (kk & 3) * 32),
                                       desc_k(k1 + (kk >> 2) * 1024 + (kk & 3) * 32, S::GROUP), idesc_h, kk > 0 ? 1u : 0u);
                        }
                        tc_commit(smem_u32(&empty[s0]));
                        tc_commit(smem_u32(&empty[s1]));
                        tc_commit(smem_u32(&s_full[buf]));
                        if (us == is.u1 - 1) tc_commit(smem_u32(&q_empty));
                        if (++us == is.u1) {
                            ++items_s;
                            if (walk_s.next(is)) us = is.u0;
                        }
                        ++ns;
                        progressed = true;
                    }
                }
                if (np < ns) {
                    const int buf = np % NS;
                    const bool first = up == ip.u0, last = up == ip.u1 - 1;
                    const int q0 = last ? 4 * np + 2 : 4 * np + 4, q1 = q0 + 1;
                    if (mbar_test_wait(smem_u32(&p_full[buf]), uint32_t(np / NS) & 1u) && is_full(q0) && is_full(q1) &&
                        (!first || items_p == 0 || mbar_test_wait(smem_u32(&o_free), uint32_t(items_p - 1) & 1u))) {
                        tc_fence_after();
                        const int s0 = q0 % NSLOT, s1 = q1 % NSLOT;
                        const uint32_t pa = tmem + uint32_t(buf * kN);
#pragma unroll
                        for (int kk = 0; kk < kN / 16; ++kk) {
                            const uint32_t v = ring_a + (kk < 4 ? s0 : s1) * S::SLOT + (kk & 3) * 2 * S::GROUP;
                            tc_mma_ts(tmem + S::O_COL, pa + kk * 8, desc_mn(v, S::GROUP), idesc_o,
                                      (!first || kk > 0) ? 1u : 0u);
                        }
                        tc_commit(smem_u32(&empty[s0]));
                        tc_commit(smem_u32(&empty[s1]));
                        tc_commit(smem_u32(&pv_done[buf]));
                        if (++up == ip.u1) {
                            ++items_p;
                            if (walk_p.next(ip)) up = ip.u0;
                        }
                        ++np;
                        progressed = true;
                    }
                }
                if (progressed) {
                    idle = 0;
                } else if (++idle > (1u << 26)) {
                    atomicOr(&g_pt_error_word, 1u);
                    ok = false;
                    break;
                }
            }
            if (!ok) s_abort = 1;
        }
    } else if (warp >= 4) {
        // ---- softmax: row (warp % 4) * 32 + lane, keys [64 w, 64 w + 64) of each tile ----
        const int w = (warp - 4) >> 2;
        const int quarter = warp & 3;
        const int row = quarter * 32 + lane;
        const int soft = (warp - 4) * 32 + lane;
        const uint32_t lane_off = uint32_t(quarter * 32) << 16;
        const int ti = row / a.group, gi = row % a.group;
        Walk walk(a, start);
        Item it;
        bool ok = true;  // (once false, the barriers below are still met, so that no warp is left at one)
        int j = 0;
        Cut cut{0, 0, 0, -1, 0};
        while (walk.next(it)) {
            const int rows = it.ntok * a.group;
            const bool valid = row < rows;
            const bool live = quarter * 32 < rows;  // some row of the warp is there
            Span v = visible(p, Request{it.tok0, it.ntok, it.len}, it.pos0 + ti);
            if (!valid) v = Span{0, 0, 0};
            float m = -INFINITY, l = 0.f;
            for (int u = it.u0; u < it.u1; ++u, ++j) {
                const int buf = j % NS;
                const int64_t key0 = int64_t(tile_of(it, u)) * kN;
                const bool open = tile_open(a, it, key0);
                if (ok) ok = wait_bar(s_full[buf], uint32_t(j / NS) & 1u, lane, s_abort);
                tc_fence_after();
                float s[64];
                float mx = -INFINITY;
                if (ok && live) {
                    tmem_ld32(tmem + uint32_t(buf * kN + w * 64) + lane_off, s);
                    tmem_ld32(tmem + uint32_t(buf * kN + w * 64 + 32) + lane_off, s + 32);
                    if (!open) {
                        const int64_t k0 = key0 + w * 64;
                        auto rel = [&](int64_t x) { return int(x - k0 < 0 ? 0 : (x - k0 > 64 ? 64 : x - k0)); };
                        const int lo = rel(v.lo), hi = rel(v.hi), sk = rel(v.sink);
#pragma unroll
                        for (int c = 0; c < 64; ++c)
                            if (!((c >= lo && c < hi) || c < sk)) s[c] = -INFINITY;
                    }
#pragma unroll
                    for (int c = 0; c < 64; ++c) mx = fmaxf(mx, s[c]);
                    mx *= a.c;
                }
                if (!open) {
                    // V rows of this tile: what is not finite leaves the product (see the file's comment). The slot's
                    // barrier is only ever one phase ahead: the product before has to be done first.
                    if (ok && u > it.u0)
                        ok = wait_bar(pv_done[(j - 1) % NS], uint32_t((j - 1) / NS) & 1u, lane, s_abort);
                    const int key = soft & 127;
                    const int q = (u == it.u1 - 1 ? 4 * j + 2 : 4 * j + 4) + (key >> 6);
                    if (ok) ok = wait_bar(full[q % NSLOT], uint32_t(q / NSLOT) & 1u, lane, s_abort);
                    if (ok) {
                        const int64_t k = key0 + key;
                        const bool seen = (k >= it.lo && k < it.hi) || k < it.sink;
                        unsigned char* base = ring + (q % NSLOT) * S::SLOT + ((key & 63) >> 3) * S::GROUP + (key & 7) * 128;
                        bool wrote = false, bad = false;
#pragma unroll 4
                        for (int i = 0; i < (ATOMS == 1 ? 4 : ATOMS * 4); ++i) {
                            const int at = ATOMS == 1 ? 0 : w * (ATOMS / 2) + (i >> 3);
                            const int ch = ATOMS == 1 ? 4 * w + ((i + key) & 3) : ((i + key) & 7);
                            uint4* x = reinterpret_cast<uint4*>(base + at * 1024 + ch * 16);
                            const uint4 y = *x;
                            if (!seen) {
                                *x = make_uint4(0, 0, 0, 0);
                                wrote = true;
                            } else if (not_finite2<T>(y.x) || not_finite2<T>(y.y) || not_finite2<T>(y.z) ||
                                       not_finite2<T>(y.w)) {
                                *x = make_uint4(finite_part<T>(y.x), finite_part<T>(y.y), finite_part<T>(y.z),
                                                finite_part<T>(y.w));
                                wrote = bad = true;
                            }
                        }
                        if (bad) atomicOr(&s_poison[j % 3][key >> 5], 1u << (key & 31));
                        if (wrote) fence_async_smem();
                    }
                }
                const bool grow = soft_any(1, ok && valid && mx > m + kGrow);
                if (soft < 4) s_poison[(j + 2) % 3][soft] = 0;  // (last read before this barrier, next set after another)
                bool poison = false;
                if (!open) {
                    const uint32_t* z = s_poison[j % 3];
                    poison = (z[0] | z[1] | z[2] | z[3]) != 0;
                }
                if (grow) {
                    s_mx[w][row] = mx;
                    soft_any(2, false);
                    const float both = fmaxf(s_mx[0][row], s_mx[1][row]);
                    float f = 1.f;
                    if (valid && both > m + kGrow) {
                        f = m == -INFINITY ? 0.f : ex2(m - both);
                        m = both;
                        l *= f;
                    }
                    if (ok && u > it.u0 && __any_sync(0xffffffffu, f != 1.f)) {
                        // O was accumulated under the old max
                        ok = wait_bar(pv_done[(j - 1) % NS], uint32_t((j - 1) / NS) & 1u, lane, s_abort);
                        tc_fence_after();
                        if (ok) {
                            // (f 0: a row whose keys so far weighed nothing; its O is zero)
                            const float g = f == 0.f ? 1.f : f;
#pragma unroll 1
                            for (int cc = 0; cc < HD / 64; ++cc) {
                                float o[32];
                                const uint32_t at = tmem + S::O_COL + uint32_t(w * (HD / 2) + cc * 32) + lane_off;
                                tmem_ld32(at, o);
#pragma unroll
                                for (int e = 0; e < 32; ++e) o[e] *= g;
                                tmem_st32(at, o);
                            }
                            tmem_wait_st();
                        }
                    }
                }
                if (ok && live) {
                    const float mu = m == -INFINITY ? 0.f : m;
                    float sum = 0.f;
#pragma unroll
                    for (int c = 0; c < 64; ++c) {
                        s[c] = ex2(fmaf(s[c], a.c, -mu));
                        sum += s[c];
                    }
                    l += sum;
                    float pk[32];
#pragma unroll
                    for (int c = 0; c < 32; ++c) pk[c] = __uint_as_float(cvt_pair<T>(s[2 * c], s[2 * c + 1]));
                    tmem_st32(tmem + uint32_t(buf * kN + w * 32) + lane_off, pk);
                    tmem_wait_st();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&p_full[buf]));
                if (poison && ok) {
                    // add what is not finite to the rows that see its key, once the product is done
                    ok = wait_bar(pv_done[buf], uint32_t(j / NS) & 1u, lane, s_abort);
                    tc_fence_after();
                    for (int key = 0; key < kN && ok; ++key) {
                        if (!((s_poison[j % 3][key >> 5] >> (key & 31)) & 1u)) continue;
                        const int64_t k = key0 + key;
                        const bool sees = (k >= v.lo && k < v.hi) || k < v.sink;
                        const int32_t page = p.table[int64_t(it.r) * p.W + k / p.ps];
                        if (page < 0 || page >= p.P) continue;
                        const int64_t vrow = ((int64_t(page) * p.Nkv + it.h) * p.ps + k % p.ps) * HD;
#pragma unroll 1
                        for (int cc = 0; cc < HD / 64; ++cc) {
                            float o[32];
                            const int col = w * (HD / 2) + cc * 32;
                            const uint32_t at = tmem + S::O_COL + uint32_t(col) + lane_off;
                            tmem_ld32(at, o);
#pragma unroll
                            for (int e = 0; e < 32; ++e) {
                                const float x = Elem<T>::load(p.v_pages, vrow + col + e);
                                if (sees && !(fabsf(x) <= 3.4e38f)) o[e] += x;
                            }
                            tmem_st32(at, o);
                        }
                        tmem_wait_st();
                    }
                    tc_fence_before();
                }
            }
            // ---- the item's share is summed: O / l, or its piece ----
            if (ok) ok = wait_bar(pv_done[(j - 1) % NS], uint32_t((j - 1) / NS) & 1u, lane, s_abort);
            s_mx[w][row] = l;  // (the last readers of the maxima arrived at p_full before that product)
            soft_any(2, false);
            tc_fence_after();
            const float L = s_mx[0][row] + s_mx[1][row];
            const bool whole = it.u0 == 0 && it.u1 == it.units;
            const float inv = L == 0.f ? 0.f : 1.0f / L;
            const int64_t slot = 2 * int64_t(blockIdx.x) + (it.u0 > 0 ? 0 : 1);
            uint16_t* dst = static_cast<uint16_t*>(p.out) +
                            ((it.tok0 + ti) * p.Nq + it.h * a.group + gi) * int64_t(HD) + w * (HD / 2);
            float* part = a.po + (slot * a.rows_cap + row) * int64_t(HD) + w * (HD / 2);
            if (ok && live) {
#pragma unroll 1
                for (int cc = 0; cc < HD / 64; ++cc) {
                    float o[32];
                    tmem_ld32(tmem + S::O_COL + uint32_t(w * (HD / 2) + cc * 32) + lane_off, o);
                    if (valid && whole) {
                        uint4* d4 = reinterpret_cast<uint4*>(dst + cc * 32);
                        if (L == 0.f) {
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = 0.f;
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            d4[e] = make_uint4(cvt_pair<T>(o[8 * e] * inv, o[8 * e + 1] * inv),
                                               cvt_pair<T>(o[8 * e + 2] * inv, o[8 * e + 3] * inv),
                                               cvt_pair<T>(o[8 * e + 4] * inv, o[8 * e + 5] * inv),
                                               cvt_pair<T>(o[8 * e + 6] * inv, o[8 * e + 7] * inv));
                    } else if (valid) {
                        float4* d4 = reinterpret_cast<float4*>(part + cc * 32);
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            d4[e] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                    }
                    __syncwarp();
                }
                if (!whole && valid && w == 0) {
                    a.pml[(slot * a.rows_cap + row) * 2] = m;
                    a.pml[(slot * a.rows_cap + row) * 2 + 1] = L;
                }
            }
            if (it.u0 == 0 && !whole && ok)
                cut = Cut{it.tok0, it.ntok, it.h, int32_t(((it.start + it.units) * ctas - 1) / U), 1};
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&o_free));
        }
        if (!ok) s_abort = 1;
        if (soft == 0) a.cuts[blockIdx.x] = cut;
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 0) tmem_dealloc(tmem, kTmem);
}

// Joins the pieces of the item that begins in CTA blockIdx.x and was cut
// there: a warp a row, pieces in CTA order.
template <int HD, class T>
__global__ void __launch_bounds__(256) paged_attention_join_kernel(const TcArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    const Cut cut = a.cuts[blockIdx.x];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row = blockIdx.y * 8 + warp;
    if (!cut.begins || row >= cut.ntok * a.group) return;
    constexpr int E = HD / 32;
    const int first = blockIdx.x, last = cut.last;
    auto slot = [&](int c) { return (2 * int64_t(c) + (c == first ? 1 : 0)) * a.rows_cap + row; };
    float M = -INFINITY;
    for (int c = first + lane; c <= last; c += 32) M = fmaxf(M, a.pml[slot(c) * 2]);
    M = warp_max(M);
    float L = 0.f;
    for (int c = first + lane; c <= last; c += 32) {
        const float m = a.pml[slot(c) * 2];
        L += (m == -INFINITY ? 0.f : ex2(m - M)) * a.pml[slot(c) * 2 + 1];
    }
    L = warp_sum(L);
    float o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
#pragma unroll 4
    for (int c = first; c <= last; ++c) {
        const float m = a.pml[slot(c) * 2];
        const float f = m == -INFINITY ? 0.f : ex2(m - M);
        const float2* src = reinterpret_cast<const float2*>(a.po + slot(c) * HD) + lane;
#pragma unroll
        for (int e = 0; e < E / 2; ++e) {
            const float2 x = src[e * 32];
            o[2 * e] = fmaf(f, x.x, o[2 * e]);
            o[2 * e + 1] = fmaf(f, x.y, o[2 * e + 1]);
        }
    }
    const int ti = row / a.group, gi = row % a.group;
    uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.p.out) +
                                                ((cut.tok0 + ti) * a.p.Nq + cut.head * a.group + gi) * int64_t(HD)) + lane;
    const float inv = L == 0.f ? 0.f : 1.0f / L;
#pragma unroll
    for (int e = 0; e < E / 2; ++e)
        dst[e * 32] = L == 0.f ? 0u : cvt_pair<T>(o[2 * e] * inv, o[2 * e + 1] * inv);
}

bool encode_map(CUtensorMap* map, const void* base, int dtype, const cuuint64_t* dims, const cuuint64_t* strides,
                const cuuint32_t* box) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    cuuint32_t estr[4] = {1, 1, 1, 1};
    return fn(map, dtype == PC_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
              const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

TcArgs tc_args(const PagedAttention& p, const PagedScratch& s) {
    TcArgs a{};
    a.p = p;
    a.group = p.Nq / p.Nkv;
    a.tpt = kM / a.group;
    int64_t g = p.ps / 8;
    a.box_groups = int(g & -g) < 8 ? int(g & -g) : 8;
    a.rows_cap = int(paged_attention_scratch_rows(p));
    a.c = p.scale * kLog2e;
    a.groups = p.P * p.Nkv * p.ps / 8;
    a.po = static_cast<float*>(s.base);
    a.pml = a.po + 2 * int64_t(s.ctas) * a.rows_cap * p.Hd;
    a.cuts = reinterpret_cast<Cut*>(a.pml + 2 * int64_t(s.ctas) * a.rows_cap * 2);
    return a;
}

template <int HD, class T>
cudaError_t run_tc(const PagedAttention& p, const PagedScratch& sc, cudaStream_t s) {
    const TcArgs a = tc_args(p, sc);
    CUtensorMap mq, mq1, mk, mv;
    {
        const cuuint64_t dims[4] = {64, cuuint64_t(p.Nq), cuuint64_t(p.T), HD / 64};
        const cuuint64_t strides[3] = {HD * 2, cuuint64_t(p.Nq) * HD * 2, 128};
        cuuint32_t box[4] = {64, cuuint32_t(a.group), cuuint32_t(a.tpt), 1};
        if (!encode_map(&mq, p.q, p.dtype, dims, strides, box)) return cudaErrorInvalidValue;
        box[2] = 1;
        if (!encode_map(&mq1, p.q, p.dtype, dims, strides, box)) return cudaErrorInvalidValue;
    }
    {
        const cuuint64_t dims[4] = {64, 8, HD / 64, cuuint64_t(a.groups)};
        const cuuint64_t strides[3] = {HD * 2, 128, 8 * HD * 2};
        const cuuint32_t box[4] = {64, 8, HD / 64, cuuint32_t(a.box_groups)};
        if (!encode_map(&mk, p.k_pages, p.dtype, dims, strides, box) ||
            !encode_map(&mv, p.v_pages, p.dtype, dims, strides, box))
            return cudaErrorInvalidValue;
    }
    static DeviceOnce once;
    cudaError_t e = once.run([] { return allow_smem(paged_attention_tc_kernel<HD, T>, Shape<HD>::SMEM); });
    if (e != cudaSuccess) return e;
    return launch_k(paged_attention_tc_kernel<HD, T>, dim3(unsigned(sc.ctas)), dim3(kPtThreads), Shape<HD>::SMEM, s, mq, mq1,
                    mk, mv, a);
}

template <int HD, class T>
cudaError_t run_join(const PagedAttention& p, const PagedScratch& sc, cudaStream_t s) {
    const TcArgs a = tc_args(p, sc);
    return launch_k(paged_attention_join_kernel<HD, T>, dim3(unsigned(sc.ctas), unsigned((a.rows_cap + 7) / 8)), dim3(256), 0,
                    s, a);
}

}  // namespace

bool paged_attention_tc_supports(const PagedAttention& p) {
    return (p.dtype == PC_BF16 || p.dtype == PC_F16) && (p.Hd == 64 || p.Hd == 128 || p.Hd == 256) && p.ps % 8 == 0 &&
           p.Nq / p.Nkv <= kM && p.P > 0 && p.scale > 0.f && p.scale < 1e30f && aligned16(p.q) && aligned16(p.k_pages) &&
           aligned16(p.v_pages) && aligned16(p.out) && p.P * p.Nkv * p.ps / 8 < (int64_t(1) << 31) && encode_fn() != nullptr;
}

int64_t paged_attention_scratch_rows(const PagedAttention& p) {
    const int64_t rows = p.T * (p.Nq / p.Nkv);
    return rows < kM ? rows : kM;
}

size_t paged_attention_scratch_bytes(const PagedAttention& p, int ctas) {
    const int64_t rows = 2 * int64_t(ctas) * paged_attention_scratch_rows(p);
    return size_t(rows * (p.Hd + 2) * 4 + int64_t(ctas) * sizeof(Cut));
}

cudaError_t paged_attention_tc(const PagedAttention& p, const PagedScratch& sc, cudaStream_t s) {
    const bool bf = p.dtype == PC_BF16;
    switch (p.Hd) {
    case 64: return bf ? run_tc<64, TBF16>(p, sc, s) : run_tc<64, TF16>(p, sc, s);
    case 128: return bf ? run_tc<128, TBF16>(p, sc, s) : run_tc<128, TF16>(p, sc, s);
    case 256: return bf ? run_tc<256, TBF16>(p, sc, s) : run_tc<256, TF16>(p, sc, s);
    }
    return cudaErrorInvalidValue;
}

cudaError_t paged_attention_join(const PagedAttention& p, const PagedScratch& sc, cudaStream_t s) {
    const bool bf = p.dtype == PC_BF16;
    switch (p.Hd) {
    case 64: return bf ? run_join<64, TBF16>(p, sc, s) : run_join<64, TF16>(p, sc, s);
    case 128: return bf ? run_join<128, TBF16>(p, sc, s) : run_join<128, TF16>(p, sc, s);
    case 256: return bf ? run_join<256, TBF16>(p, sc, s) : run_join<256, TF16>(p, sc, s);
    }
    return cudaErrorInvalidValue;
}

uint32_t read_and_clear_pt_errors() {
    unsigned int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_pt_error_word, sizeof(v)) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    if (v) cudaMemcpyToSymbol(g_pt_error_word, &zero, sizeof(zero));
    return v;
}

namespace {
RegisterFunctions reg_pa_tc({
    {"paged_attention_tc_bf16", reinterpret_cast<const void*>(paged_attention_tc_kernel<256, TBF16>)},
    {"paged_attention_tc_f16", reinterpret_cast<const void*>(paged_attention_tc_kernel<256, TF16>)},
    {"paged_attention_join_bf16", reinterpret_cast<const void*>(paged_attention_join_kernel<256, TBF16>)},
    {"paged_attention_join_f16", reinterpret_cast<const void*>(paged_attention_join_kernel<256, TF16>)},
});
}  // namespace

}  // namespace launch
}  // namespace popcorn
