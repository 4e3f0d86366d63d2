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
// In a CTA: warp 0 walks the items, looks pages up and loads Q and K by TMA
// (128-byte swizzle, a box per run of page rows); warp 2 loads V; both fill
// one ring in the order K(0), K(1), V(0), K(2), V(1), ...; warp 1 issues S = Q.K^T
// into the next of NS accumulators in tensor memory and O += P.V, whichever
// is ready; warps 4-11 (two threads a row, 64 keys each) turn S into P =
// 2^(c S - m): P is packed into the type and written back over S, from where
// the second product reads it as its A operand, so it never passes through
// shared memory. A ring slot holds 8-key groups of [Hd/64][8 keys][128 B], so
// any page size that is a multiple of 8 gives one layout (group stride Hd/64
// KB) and the two halves of a tile in neighbouring slots are one operand.
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
// would be NaN for the others (warp 3, before the product may read the slot).
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
constexpr int kPtThreads = 384;  // warps: 0 Q and K loads, 1 MMA, 2 V loads, 3 masked V, 4-11 softmax
constexpr int kSoftThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kGrow = 8.0f;  // log2 of the growth of a row's max that is let pass
constexpr uint32_t kTmem = 512;

template <int HD>
struct Shape {
    static constexpr int ATOMS = HD / 64;
    static constexpr int NS = HD == 256 ? 2 : 3;  // S accumulators: NS * 128 + HD <= 512 columns
    static constexpr int GROUP = ATOMS * 1024;    // bytes of 8 keys
    static constexpr int HALVES = HD == 256 ? 2 : 1;  // ring slots of a 128-key tile
    static constexpr int KEYS = kN / HALVES;          // keys of a slot
    static constexpr int SLOT = KEYS / 8 * GROUP;
    static constexpr int NSLOT = HD == 256 ? 5 : (HD == 128 ? 6 : 10);
    // Warp 0's notes on items and units, a ring. It writes note j with K(j - 1)
    // in the ring, so K(j - 1 - T) has been read (T tiles fit the ring), which
    // waited for the product j - 1 - T - NS: entries up to there are free
    // (Hd 256, whose odd ring mixes K and V: up to j - 4). Warp 3, idle where
    // nothing is masked, hands its entries back.
    static constexpr int NOTES = HD == 64 ? 16 : 8;
    static_assert(HD == 256 || NOTES >= NSLOT / 2 + NS + 1, "notes outlive their readers");
    static constexpr int Q_BLOCK = kM * 128;
    static constexpr int Q_BYTES = ATOMS * Q_BLOCK;
    static constexpr uint32_t O_COL = NS * kN;
    static constexpr size_t SMEM = size_t(Q_BYTES) + size_t(NSLOT) * SLOT;  // (1024-byte aligned, behind the static part)
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
    uint64_t ps_inv;  // ceil(2^64 / page size)
    int rows_cap;   // rows of a scratch slot
    float c;        // scale * log2(e)
    int64_t groups; // 8-row groups of the pages (past the end: zero fill)
    float* po;      // [2 * CTAs][rows_cap][HD]
    float* pml;     // [2 * CTAs][rows_cap][2]
    Cut* cuts;      // [CTAs]
};

// All in tokens, keys and tiles (every length is below 2^31).
struct Item {
    int r, h;
    int tok0, ntok;    // token rows
    int pos0;          // position of the first one
    int len;           // keys of the request
    int lo, hi, sink;  // keys that some row sees: [0, sink) and [lo, hi)
    int t_lo, ns, units;  // tiles [0, ns) and from t_lo on
    int u0, u1;           // this CTA's share
    int64_t start;        // the item's first unit in the step's order
};

// (Not inlined: the roles' loops are long, and the instruction cache is what they share.)
__device__ __noinline__ void item_span(const TcArgs& a, const Request& rq, int mt, Item& it) {
    const PagedAttention& p = a.p;
    const int64_t i0 = int64_t(mt) * a.tpt;
    it.tok0 = int(rq.t0 + i0);
    it.ntok = int(rq.n - i0 < a.tpt ? rq.n - i0 : a.tpt);
    const int64_t pos0 = rq.len - rq.n + i0;
    it.pos0 = int(pos0);
    it.len = int(rq.len);
    const Span first = visible(p, rq, pos0), last = visible(p, rq, pos0 + it.ntok - 1);
    it.lo = int(first.lo);
    it.hi = int(last.hi);
    it.sink = int(last.sink);
    it.t_lo = it.lo / kN;
    const int t_hi = int((last.hi + kN - 1) / kN);
    const int ns = int((last.sink + kN - 1) / kN);
    it.ns = ns < it.t_lo ? ns : it.t_lo;
    const int u = it.ns + (t_hi > it.t_lo ? t_hi - it.t_lo : 0);
    it.units = u > 1 ? u : 1;  // (rows without a key are written too)
}

struct Start {
    int r, h, mt, u;
    int64_t unit, left;
};

// The CTA's items in order (walked by the load warp, which tells the others).
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
        ntiles = int((unsigned(rq.n) + unsigned(a.tpt) - 1) / unsigned(a.tpt));
    }
    __device__ __noinline__ bool next(Item& it) {
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

// Every row of the item sees every one of the `keys` keys from key0 on.
__device__ __forceinline__ bool keys_open(const TcArgs& a, const Item& it, int64_t key0, int keys) {
    const PagedAttention& p = a.p;
    const int64_t end = p.mask_kind == 2 ? it.len : (int64_t(it.pos0) + 1 < it.len ? int64_t(it.pos0) + 1 : it.len);
    if (key0 + keys > end) return false;
    if (p.mask_kind != 1) return true;
    return key0 >= int64_t(it.pos0) + it.ntok - p.window || key0 + keys <= p.sinks;
}
// Some row of the item sees one of them.
__device__ __forceinline__ bool keys_seen(const Item& it, int64_t key0, int keys) {
    return key0 < it.hi && (key0 + keys > it.lo || key0 < it.sink);
}
// The V rows of a slot of `keys` keys need a look before the product reads them.
__device__ __forceinline__ bool guarded(const TcArgs& a, const Item& it, int64_t key0, int keys) {
    return keys_seen(it, key0, keys) && !keys_open(a, it, key0, keys);
}

// What warp 0 says of a unit.
enum : int { kFirst = 1, kLast = 2, kLook = 4 };  // first / last of its item here; kLook << h: half h is guarded
struct Unit {
    int flags;
    int group[16];  // of each box: its first 8-row group of the pages, past the last one for zeros
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 64 consecutive fp32 columns of this thread's lane.
__device__ __forceinline__ void tmem_ld64(uint32_t addr, float2* v) {
    tmem_ld32(addr, reinterpret_cast<float*>(v));
    tmem_ld32(addr + 32, reinterpret_cast<float*>(v) + 32);
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(d)
        : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)), "l"(*reinterpret_cast<uint64_t*>(&c)));
    return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(d)
        : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
    return *reinterpret_cast<float2*>(&d);
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

// Warp-uniform bounded wait (20000 suspended tries of at most 0.1 ms); false
// once any role gave up.
__device__ __noinline__ bool wait_long(uint32_t b, uint32_t parity, volatile int* abort) {
    for (int i = 0; i < 20000; ++i) {
        if (__all_sync(0xffffffffu, mbar_try_wait(b, parity))) return true;
        if (__any_sync(0xffffffffu, *abort != 0)) return false;
    }
    if ((threadIdx.x & 31) == 0) atomicOr(&g_pt_error_word, 1u);
    *abort = 1;
    return false;
}
__device__ __forceinline__ bool wait_bar(uint64_t& bar, uint32_t parity, volatile int& abort) {
    const uint32_t b = smem_u32(&bar);
    if (__all_sync(0xffffffffu, mbar_try_wait(b, parity))) return true;
    return wait_long(b, parity, &abort);
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

// Exponent fields of two 16-bit values: bit 15 of a half is set in the result where its value is not finite.
template <class T>
__device__ __forceinline__ uint32_t not_finite2(uint32_t w) {
    constexpr uint32_t e = T::code == TBF16::code ? 0x7f807f80u : 0x7c007c00u;
    constexpr uint32_t one = T::code == TBF16::code ? 0x00800080u : 0x04000400u;
    return (w & e) + one;
}
template <class T>
__device__ __forceinline__ uint32_t finite_part(uint32_t w) {
    const uint32_t bad = not_finite2<T>(w) & 0x80008000u;
    return w & ~((bad >> 15) * 0xffffu);
}

// The product left out V values that are not finite, in slots where some row does not see some key: adds them to the
// rows that see them (an infinity or a NaN outweighs any weight). O's columns [w Hd / 2, (w + 1) Hd / 2) are at `o_addr`.
template <int HD, class T>
__device__ __noinline__ void add_not_finite(const TcArgs& a, const Item& it, const Span& v, int w, uint32_t o_addr) {
    const PagedAttention& p = a.p;
    constexpr int KEYS = Shape<HD>::KEYS;
#pragma unroll 1
    for (int x = it.u0; x < it.u1; ++x) {
        const int64_t key0 = int64_t(tile_of(it, x)) * kN;
#pragma unroll 1
        for (int64_t key = key0; key < key0 + kN; ++key) {
            if (!keys_seen(it, key, 1) || !guarded(a, it, key & ~int64_t(KEYS - 1), KEYS)) continue;
            const int32_t page = p.table[int64_t(it.r) * p.W + key / p.ps];
            if (page < 0 || page >= p.P) continue;
            const bool sees = (key >= v.lo && key < v.hi) || key < v.sink;
            const int64_t vrow = ((int64_t(page) * p.Nkv + it.h) * p.ps + key % p.ps) * HD + w * (HD / 2);
#pragma unroll 1
            for (int cc = 0; cc < HD / 64; ++cc) {
                const float mine = Elem<T>::load(p.v_pages, vrow + cc * 32 + (threadIdx.x & 31));
                if (!__any_sync(0xffffffffu, !(fabsf(mine) <= 3.4e38f))) continue;
                float o[32];
                tmem_ld32(o_addr + cc * 32, o);
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    const float y = Elem<T>::load(p.v_pages, vrow + cc * 32 + e);
                    if (sees && !(fabsf(y) <= 3.4e38f)) o[e] += y;
                }
                tmem_st32(o_addr + cc * 32, o);
                tmem_wait_st();
            }
        }
    }
}

template <int HD, class T>
__global__ void __launch_bounds__(kPtThreads, 1)
    paged_attention_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_q1,
                              const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                              const __grid_constant__ TcArgs a) {
    using S = Shape<HD>;
    constexpr int NS = S::NS, NSLOT = S::NSLOT, ATOMS = S::ATOMS, kNotes = S::NOTES;
    constexpr bool BF = T::code == TBF16::code;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t item_full[kNotes], unit_full[kNotes], unit_free[kNotes], look[kNotes], q_full, q_empty,
        full[NSLOT], empty[NSLOT], s_full[NS], p_full[NS], pv_done[NS], o_free;
    __shared__ uint32_t s_tmem;
    __shared__ volatile int s_abort;
    __shared__ Start s_start;
    __shared__ long long s_scan[kPtThreads / 32];
    __shared__ float s_mx[2][kM];  // a row's two maxima, at an item's end its two sums
    __shared__ Item s_item[kNotes];
    __shared__ volatile int s_poison[kNotes];  // an item has V values that are not finite in a tile with masked keys
    __shared__ Unit s_unit[kNotes];

    pdl_launch_dependents();
    unsigned char* sq = smem_raw;
    if (smem_u32(sq) & 1023u) {  // (the swizzle's pattern repeats every 1024 bytes of address)
        if (threadIdx.x == 0) atomicOr(&g_pt_error_word, 1u);
        return;
    }
    unsigned char* ring = sq + S::Q_BYTES;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const PagedAttention& p = a.p;

    if (tid == 0) {
        mbar_init(smem_u32(&q_full), 1);
        mbar_init(smem_u32(&q_empty), 1);
        for (int i = 0; i < kNotes; ++i) {
            mbar_init(smem_u32(&item_full[i]), 1);
            mbar_init(smem_u32(&unit_full[i]), 1);
            mbar_init(smem_u32(&unit_free[i]), 1);
            mbar_init(smem_u32(&look[i]), 1);
        }
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
    if (warp == 0) tmem_alloc(smem_u32(&s_tmem), kTmem);
    pdl_wait();

    // ---- the plan: sums of the requests' units, and where this CTA begins ----
    long long* cum = reinterpret_cast<long long*>(ring);  // [R + 1], before any copy uses the ring
    auto head_units = [&](const Request& rq, int from, int step) {
        long long u = 0;
        const int nt = int((unsigned(rq.n) + unsigned(a.tpt) - 1) / unsigned(a.tpt));
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
            const int nt = int((unsigned(rq.n) + unsigned(a.tpt) - 1) / unsigned(a.tpt));
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

    const int n = int(start.left);  // units of this CTA
    constexpr int H = S::HALVES;    // ring positions of a K or V tile, from k_pos / v_pos on
    auto k_pos = [&](int j) { return j == 0 ? 0 : (2 * j - 1) * H; };
    auto v_pos = [&](int j) { return (j == n - 1 ? 2 * n - 1 : 2 * j + 2) * H; };
    // Item k of this CTA, once warp 0 has published it.
    auto item = [&](int k, Item& it) {
        if (!wait_bar(item_full[k % kNotes], uint32_t(k / kNotes) & 1u, s_abort)) return false;
        it = s_item[k % kNotes];
        return true;
    };
    const int boxes = kN / 8 / a.box_groups;  // TMA boxes of a tile
    // Box b of H-th part h, its share of the tile: issued one by one by lane 0.
    auto put = [&](const int* group, int pos, uint64_t* const* bars, const CUtensorMap* map) {
        bool ok = true;
#pragma unroll
        for (int h = 0; h < H; ++h) {
            const int q = pos + h, slot = q % NSLOT;
            ok = wait_bar(empty[slot], (uint32_t(q / NSLOT) & 1u) ^ 1u, s_abort);
            if (!ok) break;
            if (lane == 0) {
                const uint32_t bar = smem_u32(bars[h] ? bars[h] : &full[slot]);
                const uint32_t dst = smem_u32(ring) + slot * S::SLOT;
                const int per = boxes / H;
                mbar_expect_tx(bar, S::SLOT);
                for (int b = 0; b < per; ++b)
                    tma_load_4d(dst + b * a.box_groups * S::GROUP, map, 0, 0, 0, group[h * per + b], bar);
            }
        }
        __syncwarp();
        return ok;
    };

    if (warp == 0) {
        // ---- items, pages, Q and K ----
        Walk walk(a, start);
        bool ok = true;
        const int box_keys = a.box_groups * 8;
        const int per_fill = 32 / boxes;  // units whose boxes one look at the table covers
        const int my_unit = lane / boxes, my_box = lane % boxes;
        // The page of this lane's box, of unit u + my_unit (-1: no row sees a key of it). Read ahead: the table's
        // latency is longer than a tile's loads take to issue.
        auto page_of = [&](const Item& t, int u) {
            if (u + my_unit >= t.u1) return -1;
            const int64_t k0 = int64_t(tile_of(t, u + my_unit)) * kN + my_box * box_keys;
            if (!keys_seen(t, k0, box_keys)) return -1;
            const int32_t page = p.table[int64_t(t.r) * p.W + int64_t(__umul64hi(uint64_t(k0), a.ps_inv))];
            return page >= 0 ? page : 0x7fffffff;
        };
        auto group_of = [&](const Item& t, int u, int page) {
            if (page < 0) return int(a.groups);
            if (page >= p.P) {
                atomicOr(&g_pt_error_word, 32u);
                return int(a.groups);
            }
            const uint32_t k = uint32_t(tile_of(t, u + my_unit) * kN + my_box * box_keys);
            const uint32_t off = k - uint32_t(__umul64hi(uint64_t(k), a.ps_inv)) * uint32_t(p.ps);
            return int((uint32_t(page) * uint32_t(p.Nkv) + uint32_t(t.h)) * (uint32_t(p.ps) / 8) + off / 8);
        };
        Item it, nx;  // the item at hand, and the one of the next look
        int items = 0, nu = 0, page = -1, j = 0;
        bool more = n > 0 && walk.next(nx);
        if (more) {
            nu = nx.u0;
            page = page_of(nx, nu);
        }
        while (more && ok) {
            it = nx;
            const int u_first = nu;
            const int g = group_of(it, u_first, page);
            const int u_end = u_first + per_fill < it.u1 ? u_first + per_fill : it.u1;
            if (u_end < it.u1) {
                nu = u_end;
            } else {
                more = walk.next(nx);
                nu = nx.u0;
            }
            if (more) page = page_of(nx, nu);
            for (int u = u_first; u < u_end && ok; ++u, ++j) {
                Unit& note = s_unit[j % kNotes];
                ok = wait_bar(unit_free[j % kNotes], (uint32_t(j / kNotes) & 1u) ^ 1u, s_abort);
                if (!ok) break;
                if (my_unit == u - u_first) note.group[my_box] = g;
                __syncwarp();
                if (lane == 0) {
                    int flags = (u == it.u0 ? kFirst : 0) | (u == it.u1 - 1 ? kLast : 0);
#pragma unroll
                    for (int h = 0; h < H; ++h)
                        if (guarded(a, it, int64_t(tile_of(it, u)) * kN + h * S::KEYS, S::KEYS)) flags |= kLook << h;
                    note.flags = flags;
                    if (u == it.u0) {
                        s_poison[items % kNotes] = 0;
                        s_item[items % kNotes] = it;
                        mbar_arrive(smem_u32(&item_full[items % kNotes]));
                    }
                    mbar_arrive(smem_u32(&unit_full[j % kNotes]));
                }
                __syncwarp();
                if (u == it.u0) {
                    ok = wait_bar(q_empty, (uint32_t(items) & 1u) ^ 1u, s_abort);
                    if (!ok) break;
                    if (lane == 0) {
                        const bool one = it.ntok == 1;
                        mbar_expect_tx(smem_u32(&q_full), uint32_t(one ? a.group : a.group * a.tpt) * 128 * ATOMS);
                        for (int at = 0; at < ATOMS; ++at)
                            tma_load_4d(smem_u32(sq + at * S::Q_BLOCK), one ? &map_q1 : &map_q, 0, it.h * a.group, it.tok0, at,
                                        smem_u32(&q_full));
                    }
                    __syncwarp();
                    ++items;
                }
                uint64_t* const none[2] = {nullptr, nullptr};
                ok = put(note.group, k_pos(j), none, &map_k);
            }
        }
        if (!ok) s_abort = 1;
    } else if (warp == 2) {
        // ---- V ----
        bool ok = true;
        int looks = 0;
        for (int j = 0; j < n && ok; ++j) {
            ok = wait_bar(unit_full[j % kNotes], uint32_t(j / kNotes) & 1u, s_abort);
            if (!ok) break;
            const Unit& note = s_unit[j % kNotes];
            uint64_t* to[2] = {nullptr, nullptr};
#pragma unroll
            for (int h = 0; h < H; ++h)
                if (note.flags & (kLook << h)) to[h] = &look[looks++ % kNotes];
            ok = put(note.group, v_pos(j), to, &map_v);
        }
        if (!ok) s_abort = 1;
    } else if (warp == 1) {
        if (lane == 0 && n > 0) {
            // ---- MMA issue ----
            constexpr uint32_t idesc_s = make_idesc(BF, kM, kN, false), idesc_h = make_idesc(BF, kM, kN / 2, false);
            constexpr uint32_t idesc_o = make_idesc(BF, kM, HD, true);
            const uint32_t q_base = smem_u32(sq), ring_a = smem_u32(ring);
            auto is_full = [&](int q) {
                return mbar_test_wait(smem_u32(&full[q % NSLOT]), uint32_t(q / NSLOT) & 1u);
            };
            int ns = 0, np = 0;  // next tile of S, of O
            int ks = 0, kp = 0;  // their items
            int fs = 0;          // the notes on tile ns (0: not read yet)
            bool ok = true;
            uint32_t idle = 0;
            while (np < n && !s_abort) {
                bool progressed = false;
                if (ns < n && ns < np + NS) {
                    const int buf = ns % NS;
                    const int q0 = k_pos(ns), q1 = q0 + H - 1;
                    if (fs == 0 && mbar_test_wait(smem_u32(&unit_full[ns % kNotes]), uint32_t(ns / kNotes) & 1u))
                        fs = s_unit[ns % kNotes].flags | 256;
                    if (fs && (ns < NS || mbar_test_wait(smem_u32(&pv_done[buf]), uint32_t(ns / NS - 1) & 1u)) &&
                        (!(fs & kFirst) || mbar_test_wait(smem_u32(&q_full), uint32_t(ks) & 1u)) && is_full(q0) &&
                        (H == 1 || is_full(q1))) {
                        tc_fence_after();
                        const int s0 = q0 % NSLOT, s1 = q1 % NSLOT;
                        const uint32_t k0 = ring_a + s0 * S::SLOT, k1 = ring_a + s1 * S::SLOT;
                        const uint32_t d = tmem + uint32_t(buf * kN);
                        // one N = 128 product, or two of 64 where the tile wraps round the ring
                        const bool one = H == 1 || s1 == s0 + 1;
#pragma unroll 1
                        for (int h = 0; h < (one ? 1 : 2); ++h) {
                            uint64_t da = smem_desc_sw128(q_base), db = desc_k(h ? k1 : k0, S::GROUP);
                            const uint32_t to = d + uint32_t(h * (kN / 2)), idesc = one ? idesc_s : idesc_h;
#pragma unroll 1
                            for (int at = 0; at < ATOMS; ++at) {
#pragma unroll
                                for (int kk = 0; kk < 4; ++kk) tc_mma(to, da + 2 * kk, db + 2 * kk, idesc, (at | kk) ? 1u : 0u);
                                da += S::Q_BLOCK >> 4;
                                db += 1024 >> 4;
                            }
                        }
                        tc_commit(smem_u32(&empty[s0]));
                        if (H > 1) tc_commit(smem_u32(&empty[s1]));
                        tc_commit(smem_u32(&s_full[buf]));
                        if (fs & kFirst) ++ks;
                        if (fs & kLast) tc_commit(smem_u32(&q_empty));
                        fs = 0;
                        ++ns;
                        progressed = true;
                    }
                }
                if (np < ns) {
                    const int buf = np % NS;
                    const int q0 = v_pos(np), q1 = q0 + H - 1;
                    const int fp = s_unit[np % kNotes].flags;
                    const bool first = fp & kFirst;
                    if (mbar_test_wait(smem_u32(&p_full[buf]), uint32_t(np / NS) & 1u) && is_full(q0) &&
                        (H == 1 || is_full(q1)) &&
                        (!first || kp == 0 || mbar_test_wait(smem_u32(&o_free), uint32_t(kp - 1) & 1u))) {
                        tc_fence_after();
                        const int s0 = q0 % NSLOT, s1 = q1 % NSLOT;
                        const uint32_t pa = tmem + uint32_t(buf * kN);
#pragma unroll 1
                        for (int h = 0; h < 2; ++h) {  // 64 keys each
                            const uint32_t v = ring_a + (H == 1 ? s0 * S::SLOT + h * (S::SLOT / 2) : (h ? s1 : s0) * S::SLOT);
                            const uint64_t db = desc_mn(v, S::GROUP);
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk)
                                tc_mma_ts(tmem + S::O_COL, pa + (4 * h + kk) * 8, db + uint64_t(kk * (2 * S::GROUP >> 4)), idesc_o,
                                          (!first || h > 0 || kk > 0) ? 1u : 0u);
                        }
                        tc_commit(smem_u32(&empty[s0]));
                        if (H > 1) tc_commit(smem_u32(&empty[s1]));
                        tc_commit(smem_u32(&pv_done[buf]));
                        if (first) ++kp;
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
    } else if (warp == 3) {
        // ---- V of slots with masked keys ----
        Item it;
        bool ok = true;
        int looks = 0;
        for (int j = 0, k = -1; j < n && ok; ++j) {
            ok = wait_bar(unit_full[j % kNotes], uint32_t(j / kNotes) & 1u, s_abort);
            if (!ok) break;
            const int flags = s_unit[j % kNotes].flags;
            if (flags & kFirst) {
                ok = item(++k, it);
                if (!ok) break;
                it.units = it.u0;  // (here: the unit at hand)
            } else {
                ++it.units;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&unit_free[j % kNotes]));
            for (int h = 0; h < H && ok; ++h) {
                if (!(flags & (kLook << h))) continue;
                const int64_t key0 = int64_t(tile_of(it, it.units)) * kN + h * S::KEYS;
                const int slot = (v_pos(j) + h) % NSLOT;
                ok = wait_bar(look[looks % kNotes], uint32_t(looks / kNotes) & 1u, s_abort);
                ++looks;
                if (!ok) break;
                bool bad = false;
#pragma unroll 1
                for (int kk = lane; kk < S::KEYS; kk += 32) {
                    const int64_t key = key0 + kk;
                    if (keys_open(a, it, key, 1)) continue;  // (no row's product has a zero for it)
                    const bool seen = keys_seen(it, key, 1);
                    unsigned char* base = ring + slot * S::SLOT + (kk >> 3) * S::GROUP + (kk & 7) * 128;
                    uint32_t any = 0;
                    if (seen) {
#pragma unroll 8
                        for (int i = 0; i < ATOMS * 8; ++i) {
                            const uint4 y = *reinterpret_cast<const uint4*>(base + (i >> 3) * 1024 + ((i + kk) & 7) * 16);
                            any |= not_finite2<T>(y.x) | not_finite2<T>(y.y) | not_finite2<T>(y.z) | not_finite2<T>(y.w);
                        }
                    }
                    if (seen && !(any & 0x80008000u)) continue;
#pragma unroll 8
                    for (int i = 0; i < ATOMS * 8; ++i) {
                        uint4* x = reinterpret_cast<uint4*>(base + (i >> 3) * 1024 + ((i + kk) & 7) * 16);
                        uint4 y = make_uint4(0, 0, 0, 0);
                        if (seen) {
                            y = *x;
                            y = make_uint4(finite_part<T>(y.x), finite_part<T>(y.y), finite_part<T>(y.z), finite_part<T>(y.w));
                        }
                        *x = y;
                    }
                    bad = bad || seen;
                }
                if (bad) s_poison[k % kNotes] = 1;
                __threadfence_block();
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&full[slot]));
            }
        }
        if (!ok) s_abort = 1;
    } else if (warp >= 4) {
        // ---- softmax: row (warp % 4) * 32 + lane, keys [64 w, 64 w + 64) of each tile ----
        const int w = (warp - 4) >> 2;
        const int quarter = warp & 3;
        const int row = quarter * 32 + lane;
        const int soft = (warp - 4) * 32 + lane;
        const uint32_t lane_off = uint32_t(quarter * 32) << 16;
        const int ti = row / a.group, gi = row % a.group;
        Item it;
        bool ok = true;  // (once false, the barriers below are still met, so that no warp is left at one)
        int j = 0;
        Cut cut{0, 0, 0, -1, 0};
        for (int k = 0; j < n; ++k) {
            if (ok) ok = item(k, it);
            if (soft_any(2, !ok)) {  // (all leave together)
                ok = false;
                break;
            }
            const int rows = it.ntok * a.group;
            const bool valid = row < rows;
            const bool live = quarter * 32 < rows;  // some row of the warp is there
            Span v = visible(p, Request{it.tok0, it.ntok, it.len}, int64_t(it.pos0) + ti);
            if (!valid) v = Span{0, 0, 0};
            float m = -INFINITY, l = 0.f;
            for (int u = it.u0; u < it.u1; ++u, ++j) {
                const int buf = j % NS;
                const int64_t key0 = int64_t(tile_of(it, u)) * kN + w * 64;  // this thread's 64 keys
                const bool open = keys_open(a, it, key0, 64);
                if (ok) ok = wait_bar(s_full[buf], uint32_t(j / NS) & 1u, s_abort);
                tc_fence_after();
                float2 s[32];
                float mx = -INFINITY;
                if (ok && live) {
                    tmem_ld64(tmem + uint32_t(buf * kN + w * 64) + lane_off, s);
                    if (!open) {
                        // bit c: this row sees key c of the thread's 64
                        auto below = [&](int64_t x) {
                            const int64_t n = x - key0;
                            return n <= 0 ? uint64_t(0) : (n >= 64 ? ~uint64_t(0) : (uint64_t(1) << n) - 1);
                        };
                        const uint64_t sees = (below(v.hi) & ~below(v.lo)) | below(v.sink);
                        const uint32_t bits[2] = {uint32_t(sees), uint32_t(sees >> 32)};
#pragma unroll
                        for (int c = 0; c < 32; ++c) {
                            if (!(bits[c >> 4] & (1u << (2 * (c & 15))))) s[c].x = -INFINITY;
                            if (!(bits[c >> 4] & (2u << (2 * (c & 15))))) s[c].y = -INFINITY;
                        }
                    }
                    float m0 = s[0].x, m1 = s[0].y, m2 = s[1].x, m3 = s[1].y;
#pragma unroll
                    for (int c = 2; c < 32; c += 2) {
                        m0 = fmaxf(m0, s[c].x);
                        m1 = fmaxf(m1, s[c].y);
                        m2 = fmaxf(m2, s[c + 1].x);
                        m3 = fmaxf(m3, s[c + 1].y);
                    }
                    mx = fmaxf(mx, fmaxf(fmaxf(m0, m1), fmaxf(m2, m3)) * a.c);
                }
                if (soft_any(1, ok && valid && mx > m + kGrow)) {
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
                        ok = wait_bar(pv_done[(j - 1) % NS], uint32_t((j - 1) / NS) & 1u, s_abort);
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
                    const float2 c2 = make_float2(a.c, a.c), m2 = make_float2(-mu, -mu);
                    float2 sum0 = make_float2(l, 0.f), sum1 = make_float2(0.f, 0.f);
                    float pk[32];
#pragma unroll
                    for (int c = 0; c < 32; ++c) {
                        float2 x = fma2(s[c], c2, m2);
                        x.x = ex2(x.x);
                        x.y = ex2(x.y);
                        if (c & 1) sum1 = add2(sum1, x);
                        else sum0 = add2(sum0, x);
                        pk[c] = __uint_as_float(cvt_pair<T>(x.x, x.y));
                    }
                    sum0 = add2(sum0, sum1);
                    l = sum0.x + sum0.y;
                    tmem_st32(tmem + uint32_t(buf * kN + w * 32) + lane_off, pk);
                    tmem_wait_st();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&p_full[buf]));
            }
            // ---- the item's share is summed: O / l, or its piece ----
            if (ok) ok = wait_bar(pv_done[(j - 1) % NS], uint32_t((j - 1) / NS) & 1u, s_abort);
            s_mx[w][row] = l;  // (the last readers of the maxima arrived at p_full before that product)
            soft_any(2, false);
            tc_fence_after();
            if (ok && s_poison[k % kNotes])
                add_not_finite<HD, T>(a, it, v, w, tmem + S::O_COL + uint32_t(w * (HD / 2)) + lane_off);
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
    if (s_abort) {  // copies and products in flight end well within this time
        const long long t0 = clock64();
        while (clock64() - t0 < 4000000) {
        }
        __syncthreads();
    }
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
    const int64_t most = (p.Hd == 256 ? Shape<256>::KEYS : kN) / 8;  // a box stays inside a slot
    a.box_groups = int((g & -g) < most ? (g & -g) : most);
    a.ps_inv = ~uint64_t(0) / uint64_t(p.ps) + 1;  // (exact quotients for keys and sizes below 2^31)
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
