// paged_attention_tc.cu — PagedAttention on the 5th-generation tensor cores
// (bf16 / f16, head dims 64, 128 and 256, pages of a multiple of 8 rows).
//
// The step's work is cut into items: (request, KV head, tile of up to 128
// query rows), a row being one (token, query head of the group) pair, so the
// heads that share a KV head share its K/V reads. An item's units are the
// 128-key tiles that some row of it sees: those of the sink tokens, then
// those from the first row's window start to the last row's position.
// Every CTA of one wave takes an equal run of consecutive units (an item also
// counts for four, its ends' share), cutting an item where its run ends
// unless the item's own end is near: ragged lengths, long contexts with one
// token and long chunks all fill the GPU. The pieces' (m, l, O) go to scratch
// and a second kernel joins them in order (the cuts depend on the lengths
// alone, so results repeat bit for bit). The plan is computed by every CTA
// from the lengths on the device.
//
// In a CTA: warp 0 walks the items, looks pages up and loads Q and K by TMA
// (128-byte swizzle, a box per run of page rows); warp 2 loads V; both fill
// one ring in the order K(0), K(1), V(0), K(2), V(1), ...; warp 1 issues S = Q.K^T
// into the next of NS accumulators in tensor memory, warp 12 O += P.V (one
// issuer for both spent half of its time in looking at barriers, some 150
// clocks each: 2430 instead of 1700 clocks a tile at Hd 128); warps 4-7 and
// 8-11 take tiles in turn (a thread a row) and turn S into P = 2^(c S - m): P
// is packed into the type and written back over S, from where the second
// product reads it as its A operand, so it never passes through shared
// memory; one group's loads and waits pass under the other's exponentials. A
// ring slot holds 8-key groups of [Hd/64][8 keys][128 B], so any page size
// that is a multiple of 8 gives one layout (group stride Hd/64 KB). At Hd 256
// a tile takes two slots: K by columns, V by rows, the summed axis of either
// product, so neither minds where in the ring its halves lie.
//
// What bounds it. Decoding: HBM; 32 requests of up to 8192 keys, 8 KV heads
// of 256: 208 us a launch (5.55 TB/s) for the first 40 ms after a rest, at
// full clocks; 231 to 238 (4.9 TB/s) after that, where the 1000 W limit takes
// the SMs from 1965 to some 1560 MHz (a copy then goes from 6.53 to 6.3 TB/s);
// whether the inputs are the last launch's or others makes no difference. A
// single request of 4096 keys is all latency (27 us; a CTA's first product
// comes some 12 us after its start: plan 7, look-ups and loads 5; only the
// barriers' and tensor memory's set-up, 1 us, passes under the launch before).
// Chunks: neither the MUFU's 16 exponentials a clock (1024 clocks a
// tile) nor the tensor cores (as many), but the chain product, look at a
// barrier, softmax, product of a tile, some 6700 clocks, over the NS tiles in
// flight: 2250 clocks a tile at Hd 128 (32 % of the tensor cores' time; a
// window of 4096 and 4 sinks, 2000 tokens of 32 heads: 209 us, 641 TFLOP/s of
// visible pairs' work). Tiles of 64 keys, twice as many in flight, cost the
// loads' warp as much each as those of 128: 315 us. Both groups on the halves
// of one tile, which shortens the chain: 235 us, and no less at Hd 256, where
// shared memory's bandwidth (operands and copies: 320 KB a tile, 2500 clocks)
// is near. Holding a half of S in registers over the wait for the max spills:
// 250 us.
//
// The running max is kept until P would pass 2^8 (2^15 in f16; O and l use
// the same max, so O / l is exact for any); it goes from group to group with
// the tiles, warp to warp. P is rounded to the type once, as the second
// product's operand: half a step of each weight that is a normal number there
// (all of bf16's; in f16 those above 2^-25 of the row's largest, see Weights),
// so that it moves a row by half a step of sum p |v| / l at most. l adds the
// weights as they were before it; m, l and O are fp32.
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
constexpr int kPtThreads = 416;  // warps: 0 Q and K loads, 1 Q.K^T, 2 V loads, 3 masked V, 4-11 softmax, 12 P.V
constexpr int kSoftWarps = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFar = 4194304.f;  // 2^22: maxima below it are within 1/4 of their unrounded product
constexpr uint32_t kTmem = 512;

// The weights P = 2^(c S - m) that the type holds. m is set to a row's max less START (the largest weight is then
// 2^START) and kept until a weight would pass 2^TOP. bf16 has the exponents of fp32: any START does. f16 is subnormal below
// 2^-14 and ends at 2^16: START = 11 keeps weights down to 2^-25 of the largest to half a step (2^-11) of their own size,
// and smaller ones to 2^-36 of the largest. (START = 0 and TOP = 8 lost 40000 keys of 2^-25 each, 1.1e-3 of a row.)
template <class T>
struct Weights {
    static constexpr float START = T::code == TBF16::code ? 0.f : 11.f;
    static constexpr float TOP = T::code == TBF16::code ? 8.f : 15.f;
};

template <int HD>
struct Shape {
    static constexpr int ATOMS = HD / 64;
    static constexpr int NS = HD == 256 ? 2 : 3;  // S accumulators: NS * 128 + HD <= 512 columns
    static constexpr int GROUP = ATOMS * 1024;    // bytes of 8 keys
    static constexpr int HALVES = HD == 256 ? 2 : 1;  // ring slots of a 128-key tile
    static constexpr int KEYS = kN / HALVES;          // V rows of a slot: half of the tile's rows at Hd 256
    static constexpr int K_ATOMS = ATOMS / HALVES;    // K: all rows, half of their columns, so that Q.K^T has N = 128
    static constexpr int K_GROUP = K_ATOMS * 1024;
    static constexpr int SLOT = KEYS / 8 * GROUP;
    static constexpr int NSLOT = HD == 256 ? 5 : (HD == 128 ? 6 : 10);
    // Warp 0's notes on items and units, a ring. It writes note j with K(j - 1)
    // in the ring, so K(j - 1 - T) has been read (T tiles fit the ring), which
    // waited for the product j - 1 - T - NS, and both softmax groups are done
    // with the tile two before that (Hd 256, whose odd ring mixes K and V:
    // product j - 4). Warp 3, idle where nothing is masked, hands its entries
    // back.
    static constexpr int NOTES = HD == 256 ? 6 : NSLOT / 2 + NS + 3;
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
    float* po;      // [2 * CTAs][HD / 4][rows_cap][4]
    float* pml;     // [2 * CTAs][2][rows_cap]: m, l
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
    int64_t start, end;   // where the item lies in the step's order
};

// A request and a row's keys in 32 bits (every length is at most 2^30 here): [0, sink) and [lo, hi).
struct Req {
    int t0, n, len;
};
__device__ __forceinline__ Req req(const PagedAttention& p, int r) {
    int a = p.query_start[r], b = p.query_start[r + 1], len = p.seq_lens[r];
    const int T = int(p.T), most = int(p.W * p.ps);
    a = a < 0 ? 0 : (a > T ? T : a);
    b = b < a ? a : (b > T ? T : b);
    len = len < 0 ? 0 : (len > most ? most : len);
    return Req{a, b - a, len};
}
struct Keys {
    int sink, lo, hi;
};
__device__ __forceinline__ Keys keys_of(const PagedAttention& p, int len, int pos) {
    Keys v{0, 0, len};
    if (p.mask_kind != 2) v.hi = pos < 0 ? 0 : (pos < len ? pos + 1 : len);
    if (p.mask_kind == 1) {
        v.lo = pos >= p.window ? pos - p.window + 1 : 0;
        if (v.lo > v.hi) v.lo = v.hi;
        v.sink = p.sinks < v.lo ? p.sinks : v.lo;
    }
    return v;
}

// (Not inlined: the roles' loops are long, and the instruction cache is what they share.)
__device__ __noinline__ void item_span(const TcArgs& a, const Req& rq, int mt, Item& it) {
    const PagedAttention& p = a.p;
    const int i0 = mt * a.tpt;
    it.tok0 = rq.t0 + i0;
    it.ntok = rq.n - i0 < a.tpt ? rq.n - i0 : a.tpt;
    it.pos0 = rq.len - rq.n + i0;
    it.len = rq.len;
    const Keys first = keys_of(p, rq.len, it.pos0), last = keys_of(p, rq.len, it.pos0 + it.ntok - 1);
    it.lo = first.lo;
    it.hi = last.hi;
    it.sink = last.sink;
    it.t_lo = it.lo / kN;
    const int t_hi = (last.hi + kN - 1) / kN, ns = (last.sink + kN - 1) / kN;
    it.ns = ns < it.t_lo ? ns : it.t_lo;
    const int u = it.ns + (t_hi > it.t_lo ? t_hi - it.t_lo : 0);
    it.units = u > 1 ? u : 1;  // (rows without a key are written too)
}
__device__ __forceinline__ int tiles_of(const TcArgs& a, const Req& rq) {
    return int(unsigned(rq.n + a.tpt - 1) / unsigned(a.tpt));
}

// The first request from r on with new tokens (R: none), for a whole warp: 128 are looked at a round, for a step's tensors may
// hold many idle ones. (One after the other, 16382 of them between two requests: 2035 us for the step, now 220.)
__device__ __noinline__ int next_busy(const PagedAttention& p, int r) {
    const int lane = threadIdx.x & 31;
#pragma unroll 1
    for (; r < p.R; r += 128) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int x = r + 32 * i + lane;
            const unsigned busy = __ballot_sync(0xffffffffu, x < p.R && req(p, x < p.R ? x : 0).n > 0);
            if (busy) return r + 32 * i + __ffs(int(busy)) - 1;
        }
    }
    return p.R;
}

__device__ __noinline__ int64_t div64(int64_t a, int64_t b) { return a / b; }  // (one copy of a long sequence)

struct Place {
    int r, h, mt, off;
    int64_t at, cost;
};
struct Plan {
    Place begin;
    int64_t end;    // of this CTA's run
    int64_t total;  // of the step
    int ctas;       // that have a run
    int extra;      // what an item counts besides its units
};

// Where the cut at place x of an item [s, e) of `rows` rows goes: one near an end moves there. A piece costs the write
// and the read of (m, l, O) of its rows, in units about a third of one for 32 rows; runs as uneven as that cost more.
__device__ __forceinline__ int64_t moved(int64_t x, int64_t s, int64_t e, int rows, int extra) {
    const int near = extra ? rows / 40 : 0;
    return x - s <= near ? s : (e - x <= near ? e : x);
}

// The CTA's items in order (walked by warp 0, which tells the others).
struct Walk {
    const TcArgs& a;
    Req rq;
    int r, h, mt, off, ntiles, extra;
    int64_t at, end;

    __device__ __forceinline__ Walk(const TcArgs& args, const Plan& s)
        : a(args), r(s.begin.r), h(s.begin.h), mt(s.begin.mt), off(s.begin.off), extra(s.extra), at(s.begin.at), end(s.end) {
        if (at < end) load();
    }
    __device__ __forceinline__ void load() {
        rq = req(a.p, r);
        ntiles = tiles_of(a, rq);
    }
    __device__ __noinline__ bool next(Item& it) {
        while (at < end) {
            item_span(a, rq, mt, it);
            it.r = r;
            it.h = h;
            it.start = at - off;
            it.end = it.start + it.units + extra;
            const int64_t stop = it.end < end ? it.end : end;
            it.u0 = off > extra ? off - extra : 0;
            const int64_t u1 = stop - it.start - extra;
            it.u1 = u1 > 0 ? int(u1) : 0;
            at = stop;
            off = 0;
            if (++mt == ntiles) {
                mt = 0;
                if (++h == a.p.Nkv) {
                    h = 0;
                    if (at < end) {
                        r = next_busy(a.p, r + 1);
                        if (r < a.p.R) load();
                        else at = end;
                    }
                }
            }
            if (it.u1 > it.u0) return true;
        }
        return false;
    }
};

__device__ __forceinline__ int tile_of(const Item& it, int u) { return u < it.ns ? u : it.t_lo + (u - it.ns); }

// Every row of the item sees every one of the `keys` keys from key0 on.
__device__ __forceinline__ bool keys_open(const TcArgs& a, const Item& it, int key0, int keys) {
    const PagedAttention& p = a.p;
    const int end = p.mask_kind == 2 ? it.len : (it.pos0 < it.len ? it.pos0 + 1 : it.len);
    if (key0 + keys > end) return false;
    if (p.mask_kind != 1) return true;
    return key0 > it.pos0 + it.ntok - 1 - p.window || key0 + keys <= p.sinks;
}
// Some row of the item sees one of them.
__device__ __forceinline__ bool keys_seen(const Item& it, int key0, int keys) {
    return key0 < it.hi && (key0 + keys > it.lo || key0 < it.sink);
}
// The V rows of a slot of `keys` keys need a look before the product reads them.
__device__ __forceinline__ bool guarded(const TcArgs& a, const Item& it, int key0, int keys) {
    return keys_seen(it, key0, keys) && !keys_open(a, it, key0, keys);
}

// What warp 0 says of a unit.
enum : int {
    kFirst = 1, kLast = 2,  // of its item in this CTA
    kOpen = 4,              // every row sees every key of the tile
    kStop = 8,              // no unit: the CTA is done
    kNextFirst = 16, kNextLast = 32, kNextStop = 64,  // the same of the unit after it
    kLook = 128             // kLook << h: half h of V is guarded
};
struct Unit {
    int flags;
    int tile;       // its keys: from tile * 128 on
    int group[16];  // of each box: its first 8-row group of the pages, past the last one for zeros
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 64 consecutive fp32 columns of this thread's lane.
__device__ __forceinline__ void tmem_ld64(uint32_t addr, float2* v) {
    uint32_t r[64];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
        "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
        "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
        "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63"
        "}, [%64];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
          "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
          "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
          "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
          "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
        : "r"(addr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
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

// One ring slot: `n` boxes of `step` bytes.
__device__ __noinline__ void load_boxes(uint32_t dst, uint32_t bar, uint32_t bytes, const CUtensorMap* map, int atom,
                                        const int* group, int n, uint32_t step) {
    mbar_expect_tx(bar, bytes);
#pragma unroll 1
    for (int b = 0; b < n; ++b) tma_load_4d(dst + b * step, map, 0, 0, atom, group[b], bar);
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
__device__ __noinline__ bool wait_bar(uint64_t& bar, uint32_t parity, volatile int& abort) {
    const uint32_t b = smem_u32(&bar);
    if (__all_sync(0xffffffffu, mbar_try_wait(b, parity))) return true;
    return wait_long(b, parity, &abort);
}

// The same, its first look in line: for the softmax warps' turns.
__device__ __forceinline__ bool wait_fast(uint64_t& bar, uint32_t parity, volatile int& abort) {
    if (__all_sync(0xffffffffu, mbar_try_wait(smem_u32(&bar), parity))) return true;
    return wait_long(smem_u32(&bar), parity, &abort);
}

// The same for one thread.
__device__ __noinline__ bool wait_one_long(uint32_t b, uint32_t parity, volatile int* abort) {
#pragma unroll 1
    for (int i = 0; i < 20000; ++i) {
        if (mbar_try_wait(b, parity)) return true;
        if (*abort) return false;
    }
    atomicOr(&g_pt_error_word, 1u);
    *abort = 1;
    return false;
}
__device__ __forceinline__ bool wait_one(uint64_t& bar, uint32_t parity, volatile int& abort) {
    const uint32_t b = smem_u32(&bar);
    return mbar_try_wait(b, parity) || wait_one_long(b, parity, &abort);
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

// The plan: sums of the requests' units, and where this CTA's run begins and ends. cum [R + 1] and scan [2 * warps] are
// shared memory that no copy uses yet. Every thread of the CTA calls it.
__device__ __noinline__ void make_plan(const TcArgs& a, long long* cum, long long* scan, Plan& plan) {
    const PagedAttention& p = a.p;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    auto head_units = [&](const Req& rq, int from, int step) {
        long long u = 0;
        const int nt = tiles_of(a, rq);
        Item it;
#pragma unroll 1
        for (int mt = from; mt < nt; mt += step) {
            item_span(a, rq, mt, it);
            u += it.units;
        }
        return u;
    };
    // a thread a request; one of many tiles is left to a warp
    constexpr int kFewTiles = 4;
    int many = 0;
#pragma unroll 1
    for (int r = tid; r < p.R; r += kPtThreads) {
        const Req rq = req(p, r);
        const bool few = tiles_of(a, rq) <= kFewTiles;
        cum[r + 1] = few ? head_units(rq, 0, 1) * p.Nkv : -1;
        many |= !few;
    }
    if (__syncthreads_or(many)) {
#pragma unroll 1
        for (int r = warp; r < p.R; r += kPtThreads / 32) {
            if (cum[r + 1] >= 0) continue;
            long long u = head_units(req(p, r), lane, 32);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) u += __shfl_xor_sync(0xffffffffu, u, o);
            __syncwarp();
            if (lane == 0) cum[r + 1] = u * p.Nkv;
        }
    }
    if (tid == 0) cum[0] = 0;
    __syncthreads();
    {
        // each thread sums a run of requests, units and items
        const int per = (p.R + kPtThreads - 1) / kPtThreads;
        const int r0 = tid * per < p.R ? tid * per : p.R, r1 = r0 + per < p.R ? r0 + per : p.R;
        long long sum = 0, items = 0;
#pragma unroll 1
        for (int r = r0; r < r1; ++r) {
            sum += cum[r + 1];
            items += (long long)tiles_of(a, req(p, r)) * p.Nkv;
        }
        long long iu = sum, ii = items;  // inclusive over the warp
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long x = __shfl_up_sync(0xffffffffu, iu, o), y = __shfl_up_sync(0xffffffffu, ii, o);
            if (lane >= o) {
                iu += x;
                ii += y;
            }
        }
        if (lane == 31) {
            scan[warp] = iu;
            scan[kPtThreads / 32 + warp] = ii;
        }
        __syncthreads();
        long long run = iu - sum, run_items = ii - items, units = 0;
#pragma unroll 1
        for (int x = 0; x < kPtThreads / 32; ++x) {
            if (x < warp) {
                run += scan[x];
                run_items += scan[kPtThreads / 32 + x];
            }
            units += scan[x];
        }
        // With runs long enough, an item counts for its epilogue and its masked tiles too, as four units, and cuts keep
        // clear of its ends. (1, 2, 3, 4, 6: a mixed step of 13 requests 115, 110, 104, 102, 100 us, 32 decoding ones 213,
        // 209, 206, 207, 209, prompts alone 128, 133, 130, 134, 135.)
        const int extra = units >= 16ll * gridDim.x ? 4 : 0;
        run += extra * run_items;
#pragma unroll 1
        for (int r = r0; r < r1; ++r) {
            run += cum[r + 1] + extra * ((long long)tiles_of(a, req(p, r)) * p.Nkv);
            cum[r + 1] = run;
        }
        if (tid == 0) {
            plan.extra = extra;
        }
    }
    __syncthreads();
    if (warp < 2) {
        // warp 0: where the run begins, warp 1: where it ends
        const long long U = cum[p.R];
        const int ctas = U < (long long)gridDim.x ? int(U) : int(gridDim.x);
        Place b{0, 0, 0, 0, U, 0};
        const int c = int(blockIdx.x) + warp;
        if (c < ctas) {
            const long long x = div64(c * U, ctas);
            int lo = 0, hi = p.R;
#pragma unroll 1
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (cum[mid] <= x) lo = mid;
                else hi = mid;
            }
            const long long per_head = div64(cum[lo + 1] - cum[lo], p.Nkv);
            long long rem = x - cum[lo];
            b.r = lo;
            b.h = int(div64(rem, per_head));
            rem -= b.h * per_head;
            // the item: 32 tiles at a time
            const Req rq = req(p, lo);
            const int nt = tiles_of(a, rq);
#pragma unroll 1
            for (int mt0 = 0; mt0 < nt; mt0 += 32) {
                Item it;
                it.units = 0;
                if (mt0 + lane < nt) {
                    item_span(a, rq, mt0 + lane, it);
                    it.units += plan.extra;
                }
                long long incl = it.units;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const long long y = __shfl_up_sync(0xffffffffu, incl, o);
                    if (lane >= o) incl += y;
                }
                const unsigned hit = __ballot_sync(0xffffffffu, incl > rem);
                if (hit) {
                    const int l = __ffs(int(hit)) - 1;
                    b.mt = mt0 + l;
                    b.off = int(rem - __shfl_sync(0xffffffffu, incl - it.units, l));
                    b.cost = __shfl_sync(0xffffffffu, it.units, l);
                    break;
                }
                rem -= __shfl_sync(0xffffffffu, incl, 31);
            }
            const int ntok = rq.n - b.mt * a.tpt < a.tpt ? rq.n - b.mt * a.tpt : a.tpt;
            const long long s0 = x - b.off, to = moved(x, s0, s0 + b.cost, ntok * a.group, plan.extra);
            b.at = to;
            b.off = int(to - s0);
            if (to == s0 + b.cost) {  // the next item
                b.off = 0;
                if (++b.mt == nt) {
                    b.mt = 0;
                    if (++b.h == p.Nkv) {
                        b.h = 0;
                        b.r = next_busy(p, b.r + 1);
                    }
                }
            }
        }
        if (lane == 0) {
            if (warp == 0) {
                plan.begin = b;
                plan.total = U;
                plan.ctas = ctas;
            } else {
                plan.end = b.at;
            }
        }
    }
}

// The product left out V values that are not finite, in slots where some row does not see some key: adds them to the
// rows that see them (an infinity or a NaN outweighs any weight). O's columns [w Hd / 2, (w + 1) Hd / 2) are at `o_addr`.
template <int HD, class T>
__device__ __noinline__ void add_not_finite(const TcArgs& a, const Item& it, const Keys& v, int w, uint32_t o_addr) {
    const PagedAttention& p = a.p;
    constexpr int KEYS = Shape<HD>::KEYS;
#pragma unroll 1
    for (int x = it.u0; x < it.u1; ++x) {
        const int key0 = tile_of(it, x) * kN;
#pragma unroll 1
        for (int key = key0; key < key0 + kN; ++key) {
            if (!keys_seen(it, key, 1) || !guarded(a, it, key & ~(KEYS - 1), KEYS)) continue;
            const uint32_t ps = uint32_t(p.ps);
            const int32_t page = p.table[int64_t(it.r) * p.W + uint32_t(key) / ps];
            if (page < 0 || page >= p.P) continue;
            const bool sees = (key >= v.lo && key < v.hi) || key < v.sink;
            const int64_t vrow = ((int64_t(page) * p.Nkv + it.h) * p.ps + uint32_t(key) % ps) * HD + w * (HD / 2);
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

// ---- the softmax warps' rarer steps, out of their loop ----

// Scores of the keys that the row does not see: -inf, in tensor memory.
__device__ __noinline__ void hide_scores(uint32_t at, int key0, int lo, int hi, int sink) {
#pragma unroll 1
    for (int h = 0; h < kN / 32; ++h) {
        // bit c: the row sees key c of the 32 from here on
        auto below = [&](int x) {
            const int n = x - (key0 + h * 32);
            return n <= 0 ? 0u : (n >= 32 ? ~0u : (1u << n) - 1u);
        };
        const uint32_t sees = (below(hi) & ~below(lo)) | below(sink);
        float s[32];
        tmem_ld32(at + h * 32, s);
#pragma unroll
        for (int c = 0; c < 32; ++c)
            if (!(sees & (1u << c))) s[c] = -INFINITY;
        tmem_st32(at + h * 32, s);
    }
    tmem_wait_st();
}

// A tile's weights 2^(c s - m) over its scores, their sum added to l, with the product rounded as the row's maximum was: so
// far from zero (kFar) one that is not rounded lies whole powers of two above or below it.
template <class T>
__device__ __noinline__ float weigh_far(uint32_t at, float c, float m, float l) {
#pragma unroll 1
    for (int h = 0; h < kN; h += 64) {
        float pk[32];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float s[32];
            tmem_ld32(at + h + 32 * i, s);
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
                const float x = ex2(__fsub_rn(__fmul_rn(s[e], c), m)), y = ex2(__fsub_rn(__fmul_rn(s[e + 1], c), m));
                l += x + y;
                pk[16 * i + e / 2] = __uint_as_float(cvt_pair<T>(x, y));
            }
        }
        tmem_st32(at + h, pk);
    }
    tmem_wait_st();
    return l;
}

__device__ __noinline__ void scale_columns(uint32_t at, int columns, float f) {
#pragma unroll 1
    for (int c = 0; c < columns; c += 32) {
        float o[32];
        tmem_ld32(at + c, o);
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] *= f;
        tmem_st32(at + c, o);
    }
    tmem_wait_st();
}

// O times inv -> the output, `columns` columns of this thread's row from `dst` on. 16-byte chunks change places among
// four neighbouring rows, so that four lanes store 64 bytes of a row. zero: rows of no key.
template <class T>
__device__ __noinline__ void store_rows(uint32_t at, int columns, uint16_t* dst, float inv, bool zero, int row, int rows) {
    const int lane = threadIdx.x & 31, q = lane & 3;
#pragma unroll 1
    for (int cc = 0; cc < columns; cc += 32) {
        float o[32];
        tmem_ld32(at + cc, o);
        uint32_t x[4][4];
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e >> 2][e & 3] = zero ? 0u : cvt_pair<T>(o[2 * e] * inv, o[2 * e + 1] * inv);
#pragma unroll
        for (int step = 1; step <= 2; step <<= 1) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (i & step) continue;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t give = q & step ? x[i][e] : x[i | step][e];
                    const uint32_t got = __shfl_xor_sync(0xffffffffu, give, step);
                    if (q & step) x[i][e] = got;
                    else x[i | step][e] = got;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint16_t* to = reinterpret_cast<uint16_t*>(
                __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), (lane & ~3) | i));
            if (((row & ~3) | i) < rows)
                *reinterpret_cast<uint4*>(to + cc + q * 8) = make_uint4(x[i][0], x[i][1], x[i][2], x[i][3]);
        }
    }
}

// A piece's O: [column / 4][row], neighbouring rows are neighbours.
__device__ __noinline__ void store_piece(uint32_t at, int columns, float4* part, int rows_cap, bool valid) {
#pragma unroll 1
    for (int cc = 0; cc < columns; cc += 32) {
        float o[32];
        tmem_ld32(at + cc, o);
        if (valid) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                part[int64_t(cc / 4 + e) * rows_cap] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
        }
        __syncwarp();
    }
}

// The CTA of an item's last piece.
__device__ __noinline__ int last_cta(const TcArgs& a, const Item& it, const Plan& pl) {
    int64_t c = div64(it.end * pl.ctas - 1, pl.total);
    const int64_t x = div64(c * pl.total, pl.ctas);
    if (x > it.start && moved(x, it.start, it.end, it.ntok * a.group, pl.extra) == it.end) --c;
    return int(c);
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
        full[NSLOT], empty[NSLOT], s_full[NS], p_full[NS], pv_done[NS], o_free, m_ready[2][4], l_ready[2][4];
    __shared__ uint32_t s_tmem;
    __shared__ volatile int s_abort;
    __shared__ Plan s_plan;
    __shared__ float s_m[kM], s_l[kM];  // rows' running maxima (at an item's end their sums), the other group's sums
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

    if (tid < 4)
        asm volatile("prefetch.tensormap [%0];" ::"l"(tid == 0 ? &map_q : (tid == 1 ? &map_q1 : (tid == 2 ? &map_k : &map_v)))
                     : "memory");
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
            mbar_init(smem_u32(&p_full[i]), kSoftWarps / 2);
        }
        for (int i = 0; i < 8; ++i) {
            mbar_init(smem_u32(&m_ready[i >> 2][i & 3]), 1);
            mbar_init(smem_u32(&l_ready[i >> 2][i & 3]), 1);
        }
        mbar_init(smem_u32(&o_free), kSoftWarps);
        s_abort = 0;
        mbar_fence_init();
    }
    if (warp == 0) tmem_alloc(smem_u32(&s_tmem), kTmem);
    pdl_wait();

    make_plan(a, reinterpret_cast<long long*>(ring), reinterpret_cast<long long*>(sq), s_plan);
    tc_fence_before();
    fence_async_smem();  // the sums' readers are done before copies land there
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    constexpr int H = S::HALVES;    // ring positions of a K or V tile, from k_pos / v_pos on
    auto k_pos = [&](int j) { return j == 0 ? 0 : (2 * j - 1) * H; };
    auto v_pos = [&](int j) { return (2 * j + 2) * H; };
    // Item k of this CTA, once warp 0 has published it.
    auto item = [&](int k, Item& it) {
        if (!wait_bar(item_full[k % kNotes], uint32_t(k / kNotes) & 1u, s_abort)) return false;
        it = s_item[k % kNotes];
        return true;
    };
    const int boxes = kN / 8 / a.box_groups;  // TMA boxes of a tile
    // One slot's boxes, issued one by one by lane 0: `to` gets the bytes.
    auto put = [&](const int* group, int n, uint32_t step, int atom, int q, uint64_t* to, const CUtensorMap* map) {
        const int slot = q % NSLOT;
        if (!wait_bar(empty[slot], (uint32_t(q / NSLOT) & 1u) ^ 1u, s_abort)) return false;
        if (lane == 0)
            load_boxes(smem_u32(ring) + slot * S::SLOT, smem_u32(to ? to : &full[slot]), S::SLOT, map, atom, group, n, step);
        __syncwarp();
        return true;
    };

    if (warp == 0) {
        // ---- items, pages, Q and K ----
        Walk walk(a, s_plan);
        bool ok = true;
        const int box_keys = a.box_groups * 8;
        // units whose boxes one look at the table covers (fewer than there are notes: they are waited for at once)
        const int per_fill = boxes < 32 / (kNotes - 1) ? kNotes - 1 : 32 / boxes;
        const int my_unit = lane / boxes, my_box = lane % boxes;
        // The page of this lane's box, of unit u + my_unit (-1: no row sees a key of it). Read ahead: the table's
        // latency is longer than a tile's loads take to issue.
        auto page_of = [&](const Item& t, int u) {
            if (u + my_unit >= t.u1) return -1;
            const int k0 = tile_of(t, u + my_unit) * kN + my_box * box_keys;
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
        bool more = walk.next(nx);
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
            // each unit's flags, by its lanes
            const int mine = u_first + my_unit, tile = tile_of(it, mine), key0 = tile * kN;
            int flags = (mine == it.u0 ? kFirst : 0) | (mine == it.u1 - 1 ? kLast : 0) |
                        (keys_open(a, it, key0, kN) ? kOpen : 0);
            if (mine + 1 < it.u1) flags |= mine + 2 == it.u1 ? kNextLast : 0;
            else flags |= !more ? kNextStop : (kNextFirst | (nx.u0 + 1 == nx.u1 ? kNextLast : 0));
#pragma unroll
            for (int h = 0; h < H; ++h)
                if (!(flags & kOpen) && guarded(a, it, key0 + h * S::KEYS, S::KEYS)) flags |= kLook << h;
            // (warp 3 hands notes back in order and needs nothing from here for those of units before j)
            const int j_end = j + (u_end - u_first) - 1;
            ok = wait_bar(unit_free[j_end % kNotes], (uint32_t(j_end / kNotes) & 1u) ^ 1u, s_abort);
            for (int u = u_first; u < u_end && ok; ++u, ++j) {
                Unit& note = s_unit[j % kNotes];
                if (my_unit == u - u_first) {
                    note.group[my_box] = g;
                    if (my_box == 0) {
                        note.flags = flags;
                        note.tile = tile;
                    }
                }
                __syncwarp();
                if (lane == 0) {
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
                        _Pragma("unroll 1") for (int at = 0; at < ATOMS; ++at)
                            tma_load_4d(smem_u32(sq + at * S::Q_BLOCK), one ? &map_q1 : &map_q, 0, it.h * a.group, it.tok0, at,
                                        smem_u32(&q_full));
                    }
                    __syncwarp();
                    ++items;
                }
#pragma unroll 1
                for (int h = 0; h < H && ok; ++h)
                    ok = put(note.group, boxes, a.box_groups * S::K_GROUP, h * S::K_ATOMS, k_pos(j) + h, nullptr, &map_k);
            }
        }
        if (ok) ok = wait_bar(unit_free[j % kNotes], (uint32_t(j / kNotes) & 1u) ^ 1u, s_abort);
        if (ok && lane == 0) {
            s_unit[j % kNotes].flags = kStop;
            mbar_arrive(smem_u32(&unit_full[j % kNotes]));
        }
        if (!ok) s_abort = 1;
    } else if (warp == 2) {
        // ---- V ----
        bool ok = true;
        int looks = 0;
        for (int j = 0; ok; ++j) {
            ok = wait_bar(unit_full[j % kNotes], uint32_t(j / kNotes) & 1u, s_abort);
            const Unit& note = s_unit[j % kNotes];
            if (!ok || (note.flags & kStop)) break;
#pragma unroll 1
            for (int h = 0; h < H && ok; ++h)
                ok = put(note.group + h * (boxes / H), boxes / H, a.box_groups * S::GROUP, 0, v_pos(j) + h,
                         note.flags & (kLook << h) ? &look[looks++ % kNotes] : nullptr, &map_v);
        }
        if (!ok) s_abort = 1;
    } else if (warp == 1) {
        // ---- S = Q.K^T ----
        if (lane == 0) {
            constexpr uint32_t idesc_s = make_idesc(BF, kM, kN, false);
            const uint32_t q_base = smem_u32(sq), ring_a = smem_u32(ring);
            bool ok = true;
            for (int j = 0, k = 0; ok; ++j) {
                const int buf = j % NS;
                ok = wait_one(unit_full[j % kNotes], uint32_t(j / kNotes) & 1u, s_abort);
                const int flags = s_unit[j % kNotes].flags;
                if (!ok || (flags & kStop)) break;
                const int q0 = k_pos(j), q1 = q0 + H - 1;
                const int s0 = q0 % NSLOT, s1 = q1 % NSLOT;
                if (flags & kFirst) ok = wait_one(q_full, uint32_t(k++) & 1u, s_abort);
                if (ok && j >= NS) ok = wait_one(pv_done[buf], uint32_t(j / NS - 1) & 1u, s_abort);
                if (ok) ok = wait_one(full[s0], uint32_t(q0 / NSLOT) & 1u, s_abort);
                if (ok && H > 1) ok = wait_one(full[s1], uint32_t(q1 / NSLOT) & 1u, s_abort);
                if (!ok) break;
                tc_fence_after();
                const uint32_t d = tmem + uint32_t(buf * kN);
                uint64_t da = smem_desc_sw128(q_base);
#pragma unroll 1
                for (int h = 0; h < H; ++h) {
                    uint64_t db = desc_k(ring_a + (h ? s1 : s0) * S::SLOT, S::K_GROUP);
#pragma unroll 1
                    for (int at = 0; at < S::K_ATOMS; ++at) {
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk) tc_mma(d, da + 2 * kk, db + 2 * kk, idesc_s, (h | at | kk) ? 1u : 0u);
                        da += S::Q_BLOCK >> 4;
                        db += 1024 >> 4;
                    }
                }
                tc_commit(smem_u32(&s_full[buf]));
                tc_commit(smem_u32(&empty[s0]));
                if (H > 1) tc_commit(smem_u32(&empty[s1]));
                if (flags & kLast) tc_commit(smem_u32(&q_empty));
            }
            if (!ok) s_abort = 1;
        }
    } else if (warp == 12) {
        // ---- O += P.V ----
        if (lane == 0) {
            constexpr uint32_t idesc_o = make_idesc(BF, kM, HD, true);
            const uint32_t ring_a = smem_u32(ring);
            bool ok = true;
            for (int j = 0, k = 0; ok; ++j) {
                const int buf = j % NS;
                ok = wait_one(unit_full[j % kNotes], uint32_t(j / kNotes) & 1u, s_abort);
                const int flags = s_unit[j % kNotes].flags;
                if (!ok || (flags & kStop)) break;
                const int q0 = v_pos(j), q1 = q0 + H - 1;
                const int s0 = q0 % NSLOT, s1 = q1 % NSLOT;
                const bool first = flags & kFirst;
                if (first && k++ > 0) ok = wait_one(o_free, uint32_t(k - 2) & 1u, s_abort);
                // (P(j) first: with it K(j) has landed, which had V(j)'s slot before it at Hd 256)
                if (ok) ok = wait_one(p_full[buf], uint32_t(j / NS) & 1u, s_abort);
                if (ok) ok = wait_one(full[s0], uint32_t(q0 / NSLOT) & 1u, s_abort);
                if (ok && H > 1) ok = wait_one(full[s1], uint32_t(q1 / NSLOT) & 1u, s_abort);
                if (!ok) break;
                tc_fence_after();
                const uint32_t pa = tmem + uint32_t(buf * kN);
#pragma unroll 1
                for (int h = 0; h < 2; ++h) {  // 64 keys each
                    const uint32_t v = ring_a + (H == 1 ? s0 * S::SLOT + h * (S::SLOT / 2) : (h ? s1 : s0) * S::SLOT);
                    const uint64_t db = desc_mn(v, S::GROUP);
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
                        tc_mma_ts(tmem + S::O_COL, pa + h * 64 + kk * 8, db + uint64_t(kk * (2 * S::GROUP >> 4)), idesc_o,
                                  (!first || h > 0 || kk > 0) ? 1u : 0u);
                }
                tc_commit(smem_u32(&pv_done[buf]));
                tc_commit(smem_u32(&empty[s0]));
                if (H > 1) tc_commit(smem_u32(&empty[s1]));
            }
            if (!ok) s_abort = 1;
        }
    } else if (warp == 3) {
        // ---- V of slots with masked keys ----
        Item it;
        bool ok = true;
        int looks = 0;
        for (int j = 0, k = -1; ok; ++j) {
            ok = wait_bar(unit_full[j % kNotes], uint32_t(j / kNotes) & 1u, s_abort);
            const int flags = s_unit[j % kNotes].flags, tile = s_unit[j % kNotes].tile;
            if (!ok || (flags & kStop)) break;
            if (flags & kFirst) {
                ok = item(++k, it);
                if (!ok) break;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&unit_free[j % kNotes]));
            _Pragma("unroll 1") for (int h = 0; h < H && ok; ++h) {
                if (!(flags & (kLook << h))) continue;
                const int key0 = tile * kN + h * S::KEYS;
                const int slot = (v_pos(j) + h) % NSLOT;
                ok = wait_bar(look[looks % kNotes], uint32_t(looks / kNotes) & 1u, s_abort);
                ++looks;
                if (!ok) break;
                bool bad = false;
#pragma unroll 1
                for (int kk = lane; kk < S::KEYS; kk += 32) {
                    const int key = key0 + kk;
                    if (keys_open(a, it, key, 1)) continue;  // (no row's product has a zero for it)
                    const bool seen = keys_seen(it, key, 1);
                    unsigned char* base = ring + slot * S::SLOT + (kk >> 3) * S::GROUP + (kk & 7) * 128;
                    uint32_t any = 0;
                    if (seen) {
#pragma unroll 4
                        for (int i = 0; i < ATOMS * 8; ++i) {
                            const uint4 y = *reinterpret_cast<const uint4*>(base + (i >> 3) * 1024 + ((i + kk) & 7) * 16);
                            any |= not_finite2<T>(y.x) | not_finite2<T>(y.y) | not_finite2<T>(y.z) | not_finite2<T>(y.w);
                        }
                    }
                    if (seen && !(any & 0x80008000u)) continue;
#pragma unroll 2
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
    } else {
        // ---- softmax: a thread a row; group w takes the tiles with j % 2 == w ----
        const int w = (warp - 4) >> 2;
        const int quarter = warp & 3;  // TMEM lanes this warp may access
        const int row = quarter * 32 + lane;
        const uint32_t lane_off = uint32_t(quarter * 32) << 16;
        int row_lo = 0, row_hi = 0, row_sink = 0;  // keys that the row sees: [0, sink), [lo, hi)
        bool ok = true, valid = false, live = false;
        int k = -1;
        float m = -INFINITY, l = 0.f;  // l: this group's share, under m
        Cut cut{0, 0, 0, -1, 0};
        // The notes of a unit tell of the next one too, so a group reads those of its own units alone (group 1 starts
        // with the other's first).
        ok = wait_bar(unit_full[0], 0u, s_abort);
        int next = ok ? s_unit[0].flags : kStop;
        next = next & kStop ? kNextStop : ((next & kFirst ? kNextFirst : 0) | (next & kLast ? kNextLast : 0));
        for (int j = 0; ok; ++j) {
            const bool own = (j & 1) == w;
            int flags;
            if (own) {
                ok = wait_fast(unit_full[j % kNotes], uint32_t(j / kNotes) & 1u, s_abort);
                next = flags = s_unit[j % kNotes].flags;
                if (!ok || (flags & kStop)) break;
            } else {
                if (next & kNextStop) break;
                flags = (next & kNextFirst ? kFirst : 0) | (next & kNextLast ? kLast : 0);
            }
            if (flags & kFirst) {
                Item it;
                ok = item(++k, it);
                if (!ok) break;
                const int ti = row / a.group, rows = it.ntok * a.group;
                valid = row < rows;
                live = quarter * 32 < rows;  // some row of the warp is there
                const Keys v = keys_of(p, it.len, it.pos0 + ti);
                row_lo = v.lo;
                row_hi = valid ? v.hi : 0;
                row_sink = valid ? v.sink : 0;
                m = -INFINITY;
                l = 0.f;
            }
            const int buf = j % NS;
            if (own) {
                ok = wait_fast(s_full[buf], uint32_t(j / NS) & 1u, s_abort);
                if (!ok) break;
                tc_fence_after();
                float mx = -INFINITY;
                const uint32_t at_s = tmem + uint32_t(buf * kN) + lane_off;
                if (live) {
                    if (!(flags & kOpen))
                        hide_scores(at_s, s_unit[j % kNotes].tile * kN, row_lo, row_hi, row_sink);
#pragma unroll 1
                    for (int h = 0; h < 2; ++h) {
                        float2 s[32];
                        tmem_ld64(at_s + h * 64, s);
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
                }
                // the running max, from the tile before (another item's is of no use, but its turn is awaited)
                if (j > 0) {
                    ok = wait_fast(m_ready[w ^ 1][quarter], uint32_t((j - 1) >> 1) & 1u, s_abort);
                    if (!ok) break;
                }
                const bool first = flags & kFirst;
                const float before = first ? -INFINITY : s_m[row];
                float now = before;
                if (valid && mx > __fadd_rd(before, Weights<T>::TOP)) now = __fsub_ru(mx, Weights<T>::START);
                s_m[row] = now;
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&m_ready[w][quarter]));
                if (now != m) {
                    if (m != -INFINITY) l *= ex2(m - now);
                    m = now;
                }
                if (live && __any_sync(0xffffffffu, fabsf(m) >= kFar && m != -INFINITY)) {
                    l = weigh_far<T>(at_s, a.c, m == -INFINITY ? 0.f : m, l);
                } else if (live) {
                    const float mu = m == -INFINITY ? 0.f : m;
                    const float2 c2 = make_float2(a.c, a.c), m2 = make_float2(-mu, -mu);
                    float2 sum0 = make_float2(l, 0.f), sum1 = make_float2(0.f, 0.f);
#pragma unroll 1
                    for (int h = 0; h < 2; ++h) {
                        float2 s[32];
                        tmem_ld64(at_s + h * 64, s);
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
                        // over the scores that it came from
                        tmem_st32(at_s + h * 64, pk);
                    }
                    sum0 = add2(sum0, sum1);
                    l = sum0.x + sum0.y;
                    tmem_wait_st();
                }
                if (!first && __any_sync(0xffffffffu, now != before && before != -INFINITY)) {
                    // O was accumulated under the old max
                    ok = wait_bar(pv_done[(j - 1) % NS], uint32_t((j - 1) / NS) & 1u, s_abort);
                    if (!ok) break;
                    tc_fence_after();
                    scale_columns(tmem + S::O_COL + lane_off, HD,
                                  now != before && before != -INFINITY ? ex2(before - now) : 1.f);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&p_full[buf]));
            }
            if (!(flags & kLast)) continue;
            // ---- the item's share is summed: O / l, or its piece; group w has half of the columns ----
            ok = wait_bar(pv_done[buf], uint32_t(j / NS) & 1u, s_abort);
            if (ok && (j & 1) != w) ok = wait_bar(m_ready[w ^ 1][quarter], uint32_t(j >> 1) & 1u, s_abort);
            if (!ok) break;
            tc_fence_after();
            const Item it = s_item[k % kNotes];  // (kept until the next item's products have passed this point)
            const int ti = row / a.group, gi = row % a.group;
            const float last_m = s_m[row];
            if (m != last_m && m != -INFINITY) l *= ex2(m - last_m);
            // the group without the last tile gives its share, the other one the sum of both
            float L;
            if ((j & 1) != w) {
                s_l[row] = l;
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&l_ready[0][quarter]));
                ok = wait_bar(l_ready[1][quarter], uint32_t(k) & 1u, s_abort);
                L = s_m[row];
            } else {
                ok = wait_bar(l_ready[0][quarter], uint32_t(k) & 1u, s_abort);
                L = l + s_l[row];
                s_m[row] = L;
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&l_ready[1][quarter]));
            }
            if (!ok) break;
            const uint32_t o_addr = tmem + S::O_COL + uint32_t(w * (HD / 2)) + lane_off;
            if (s_poison[k % kNotes]) add_not_finite<HD, T>(a, it, Keys{row_sink, row_lo, row_hi}, w, o_addr);
            const bool whole = it.u0 == 0 && it.u1 == it.units;
            if (live && whole) {
                uint16_t* dst = static_cast<uint16_t*>(p.out) +
                                ((int64_t(it.tok0) + ti) * p.Nq + it.h * a.group + gi) * HD + w * (HD / 2);
                store_rows<T>(o_addr, HD / 2, dst, L == 0.f ? 0.f : 1.0f / L, L == 0.f, row, it.ntok * a.group);
            } else if (live) {
                const int64_t slot = 2 * int64_t(blockIdx.x) + (it.u0 > 0 ? 0 : 1);
                store_piece(o_addr, HD / 2,
                            reinterpret_cast<float4*>(a.po) + (slot * (HD / 4) + w * (HD / 8)) * a.rows_cap + row, a.rows_cap,
                            valid);
                if (valid && w == 0) {
                    a.pml[slot * 2 * a.rows_cap + row] = last_m;
                    a.pml[(slot * 2 + 1) * a.rows_cap + row] = L;
                }
            }
            if (it.u0 == 0 && !whole && warp == 4) cut = Cut{it.tok0, it.ntok, it.h, last_cta(a, it, s_plan), 1};
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&o_free));
        }
        if (!ok) s_abort = 1;
        if (warp == 4 && lane == 0) a.cuts[blockIdx.x] = cut;
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
// there, in CTA order: 32 rows (a lane each) by 32 columns (four a warp).
template <int HD, class T>
__global__ void __launch_bounds__(256) paged_attention_join_kernel(const TcArgs a) {
    __shared__ uint2 tile[32][9];
    pdl_launch_dependents();
    pdl_wait();
    const Cut cut = a.cuts[blockIdx.x];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rows = cut.ntok * a.group, row0 = blockIdx.y * 32, row = row0 + lane;
    if (!cut.begins || row0 >= rows) return;
    const int first = blockIdx.x, last = cut.last;
    auto slot = [&](int c) { return 2 * int64_t(c) + (c == first ? 1 : 0); };
    if (row < rows) {
        auto m_of = [&](int c) { return a.pml[slot(c) * 2 * a.rows_cap + row]; };
        float M = -INFINITY;
#pragma unroll 8
        for (int c = first; c <= last; ++c) M = fmaxf(M, m_of(c));
        float L = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        const int col4 = blockIdx.z * 8 + warp;
#pragma unroll 8
        for (int c = first; c <= last; ++c) {
            const float m = m_of(c), l = a.pml[(slot(c) * 2 + 1) * a.rows_cap + row];
            const float4 x = reinterpret_cast<const float4*>(a.po)[(slot(c) * (HD / 4) + col4) * a.rows_cap + row];
            const float f = m == -INFINITY ? 0.f : ex2(m - M);
            L = fmaf(f, l, L);
            o.x = fmaf(f, x.x, o.x);
            o.y = fmaf(f, x.y, o.y);
            o.z = fmaf(f, x.z, o.z);
            o.w = fmaf(f, x.w, o.w);
        }
        const float inv = L == 0.f ? 0.f : 1.0f / L;
        tile[lane][warp] = L == 0.f ? make_uint2(0u, 0u)
                                    : make_uint2(cvt_pair<T>(o.x * inv, o.y * inv), cvt_pair<T>(o.z * inv, o.w * inv));
    }
    __syncthreads();
    const int r = row0 + int(threadIdx.x >> 3), q = threadIdx.x & 7;
    if (r >= rows) return;
    uint16_t* dst = static_cast<uint16_t*>(a.p.out) +
                    ((cut.tok0 + r / a.group) * a.p.Nq + cut.head * a.group + r % a.group) * int64_t(HD) + blockIdx.z * 32;
    reinterpret_cast<uint2*>(dst)[q] = tile[r - row0][q];
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
        const cuuint32_t k_box[4] = {64, 8, Shape<HD>::K_ATOMS, cuuint32_t(a.box_groups)};
        const cuuint32_t v_box[4] = {64, 8, HD / 64, cuuint32_t(a.box_groups)};
        if (!encode_map(&mk, p.k_pages, p.dtype, dims, strides, k_box) ||
            !encode_map(&mv, p.v_pages, p.dtype, dims, strides, v_box))
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
    return launch_k(paged_attention_join_kernel<HD, T>, dim3(unsigned(sc.ctas), unsigned((a.rows_cap + 31) / 32), HD / 32), dim3(256), 0,
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
