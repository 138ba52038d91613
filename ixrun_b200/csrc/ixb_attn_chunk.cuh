// Causal attention of every request's new tokens over its pages: the form for many rows (chunks of prompts), on tcgen05.
// Formulas and packing of rows as in ixb_attn_paged.cuh.
//
//   CTA      one per SM; a range of key tiles (128 keys) out of all (KV head, request, row tile) units' in one line, equal in cost (a
//            unit's end has its own, behind its tiles), so lengths that differ cost nothing.  A unit that is cut leaves its parts in the
//            scratch, k_attn_chunk_join adds them up.
//   unit     128 or 256 packed rows (128 with heads of 256) of one request and KV head
//   step     Q K^T of 128 rows and a key tile into tensor memory (S), softmax in registers (a thread is a row), the probabilities as
//            bf16 over S in tensor memory, P V into the accumulator there.  Two steps are in flight in two slots: the two row tiles
//            of a unit; or, with one row tile, even and odd key tiles (each with an accumulator and a softmax of its own; heads of 256
//            leave room for one accumulator, there they share it).
//   warps    0 .. 3, 4 .. 7  softmax of the two slots (heads of 256: 0 .. 3); they also bring Q and write the results
//            then four       one that issues the MMAs, one that asks for K and V (TMA, a box per page and 64 dimensions, 128-byte
//                            swizzle) in a ring of [128 keys][128 dimensions] (64 with heads of 64), two that look for values that are
//                            not finite
//
// The accumulator is rescaled only when a row's maximum has grown by more than 2^8 (a running maximum that lags changes no ratio).
// Precision: scores and sums fp32, probabilities bf16 for P V (half a step, 2^-8 of each, as the result's own rounding; the tensor
// core takes no wider operand beside bf16 values), their sum from the fp32 values: results 0.0023 from 64 bits, 0.0017 of it their own
// rounding.  With the trailing bits as a second product, as the form for few rows has them, 0.0017; the chunk below then takes
// 289 us instead of 224, drafts of heads of 256 57.5 instead of 49.9, and every value has to be looked through (a trailing part of
// zero or less times infinity is NaN).
//
// Keys that no row of the unit sees are not read; the rows of V behind the last key are zeroed up to a multiple of 16 and not
// multiplied beyond.  A value that is not finite counts for the rows that see it and for no other: where a key tile is not
// seen by all rows, two warps look for such values, and the softmax warps take the tile's P V themselves if there is one.
//
// Bound: the tensor core for long chunks, with the exponentials (one per score, 16 a cycle and SM) close behind: 2048 rows of a prompt
// behind 12000 keys, 16 / 8 heads of 128: 192 us, 69 % of the measured rate of dense products; the tensor pipe and the special function
// unit are each busy 45 % of the time, the rest is the chain scores, maximum, exponentials, P V.  (In a captured graph; among
// other passes 224 us, 59 %, at the clocks that the power limit leaves.)  Fixed: 10 us for a launch, the
// first keys, the cut units' ends and the join.  Built and slower for that chunk: steps of 64 keys in slots of their own, so that
// scores wait for no P V (224 us: Q K^T of 64 columns is bound by Q's reads, and a step's overheads come twice), these with two sets
// of softmax warps that take steps in turn (228), an MMA warp per group (248: the groups then run in step and want the
// exponentials at the same time; one warp keeps them apart), a quarter of the exponentials as polynomials (214).
//
// Every wait on an mbarrier is bounded and counts this CTA's own copies and products; where one runs out the CTA's outputs
// become NaN, and it carries on to its end with nothing in flight and tensor memory released.
#pragma once
#include "ixb_attn_paged.cuh"
#include <cuda.h>

namespace ixb {

constexpr uint32_t kPcKeys = 128;
// Key tiles of a CTA, unless there are more units than that makes CTAs: parts that are joined against tiles one behind the other (64 rows
// behind 6000 keys, 16 / 8 heads of 128: 23.0 us with 2, 21.7 with 4, 21.8 with 8, 27.6 with 16; behind 2000 16.6, 17.2, 20.1, 27.3;
// 20 rows behind 4000, 12 / 2 heads of 256: 21.6, 23.7, 28.5, 39.6).
constexpr uint32_t kPcMinCost = 4;
// Cost of a unit (key tiles times row tiles), on average, up to which it is not cut (prompts from their start, 16 / 8 heads of 128: 300
// tokens 17.8 us cut, 15.7 whole; 700 tokens 19.5 cut, 21.1 whole; 64 rows behind 1200 keys 16.2 cut, 20.9 whole, behind 2000, which
// is above the limit, 17.1 cut, 26.2 whole; 300 tokens of 24 / 4 heads of 256 25.3 cut, 17.8 whole).
constexpr uint32_t kPcShortUnit = 12;

template <int D>
struct PcCfg {
    static constexpr int kTiles = D == 256 ? 1 : 2;    // row tiles of a unit at most
    static constexpr int kGroups = kTiles;             // of softmax warps
    static constexpr uint32_t kUnitRows = 128u * kTiles;
    static constexpr int kUD = D < 128 ? D : 128;      // dimensions of a ring unit
    static constexpr int kNU = D / kUD;                // ring units of a key tile's K or V
    static constexpr uint32_t kPanel = kPcKeys * 128;  // 64 dimensions of 128 rows: rows of 128 bytes
    static constexpr uint32_t kUnit = kUD / 64 * kPanel;
    static constexpr uint32_t kQTile = D / 64 * kPanel;
    static constexpr uint32_t kStages = D == 64 ? 8 : 5;
    // Cost of a unit's end and the next one's start, in steps of 128 rows and a key tile: without it CTAs with ends of two units are the last
    // (a prompt of 2048 tokens from its start, 16 / 8 heads of 128: 50.7 us with 0, 43.2 with 2, 41.2 with 4, 37.3 with 6, 37.6 with 8;
    // 32 / 8 heads of 64: 60.9, 50.1, 45.9, 45.2, 46.2; heads of 256, whose steps are longer: drafts 50.9 with 0, 47.6 with 1, 49.9 with
    // 2, but a prompt of 2048 tokens, 24 / 4 heads, 143.8, 105.6 and 91.4).
    static constexpr uint32_t kEnd = D == 256 ? 1 : 6;
    static constexpr uint32_t kRingOff = kTiles * kQTile;
    static constexpr uint32_t kBarOff = kRingOff + kStages * kUnit;
    static constexpr uint32_t kLook = 8;               // key tiles that may be looked through ahead
    static constexpr uint32_t kBars = 2 * kStages + 13 + 2 * kLook;
    static_assert(kStages / (2 * kNU) < kLook, "a barrier is not used again before its last phase was seen");
    static constexpr uint32_t kWalkOff = kBarOff + kBars * 8 + 1024 + 192;
    static constexpr uint32_t kSmem = kWalkOff + kGroups * 4 * 80;             // no static arrays: stages start on 1024 bytes
    static constexpr int kSoftWarps = 4 * kGroups, kMmaWarp = kSoftWarps, kLoadWarp = kSoftWarps + 1, kScanWarp = kSoftWarps + 2, kThreads = (kSoftWarps + 4) * 32;
    // Registers of a thread: a softmax thread keeps a row of 128 scores.  With two groups of them the launch's 168 are dealt out
    // again (256 x 216 + 128 x 72 = 384 x 168); with one 255 are left for everybody.
    static constexpr bool kDeal = kGroups == 2;
    static constexpr uint32_t kPart = kUnitRows * (D + 2);                     // floats: sums [tile][D / 4][128][4], (maximum, denominator) [rows]
    static constexpr uint32_t kO = 256;                // tensor memory: S or P of the slots at 0 and 128, accumulators from here
    static_assert(kSmem <= 227 * 1024 && kStages * kUnit >= 8 * kPaMaxRequests && kUnit % 1024 == 0, "fits");
};

// a unit that was cut, under the number of the CTA that has its first key tile; parts 0: none
struct PcCut {
    uint32_t parts, first_slot;
    uint32_t row0, m0, rows, head;                     // the request's first row; the unit's rows m0 .. m0 + rows - 1 of its packed ones, KV head
    int32_t pos0;                                      // position of the request's first new token
    uint32_t keys;                                     // that any row sees
};
__device__ __forceinline__ void pc_arrive(uint32_t mbar)
{
    asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.shared::cta.b64 st, [%0];\n\t}" ::"r"(mbar) : "memory");
}
// operand in shared memory, 128-byte swizzle, version 1.  K-major: groups of eight rows sbo bytes apart.  MN-major: 64 elements of a row
// are one swizzled line, lbo bytes to the next 64, sbo to the next eight rows.
__device__ __forceinline__ uint64_t pc_desc(uint32_t addr, uint32_t lbo, uint32_t sbo)
{
    return (uint64_t)((addr >> 4) & 0x3FFFu) | (uint64_t)(lbo >> 4) << 16 | (uint64_t)(sbo >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
// kind::f16, bf16 x bf16 -> fp32, M = 128; b_mn: B is MN-major
__device__ __forceinline__ constexpr uint32_t pc_idesc(uint32_t n, uint32_t b_mn) { return 1u << 4 | 1u << 7 | 1u << 10 | b_mn << 16 | (n >> 3) << 17 | (128u >> 4) << 24; }
__device__ __forceinline__ void pc_mma_ss(uint32_t el, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc)
{
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}"
                 :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(0u), "r"(el) : "memory");
}
__device__ __forceinline__ void pc_mma_ts(uint32_t el, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc)
{
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}"
                 :: "r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(0u), "r"(el) : "memory");
}
__device__ __forceinline__ void pc_commit(uint32_t el, uint32_t mbar)
{
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
                 "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(mbar), "r"(el) : "memory");
}
// 32 columns of this lane's row
__device__ __forceinline__ void pc_ld32(uint32_t addr, uint32_t *r)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
                   "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
                   "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(addr) : "memory");
}
__device__ __forceinline__ void pc_st32(uint32_t addr, const uint32_t *r)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
                 "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
                 :: "r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
                    "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
                    "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
                    "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void pc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// loaded registers are used behind the wait only
__device__ __forceinline__ void pc_pin(uint32_t *r)
{
#pragma unroll
    for (int i = 0; i < 32; ++i) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ float pc_max3(float a, float b, float c)
{
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// two fp32 numbers in a register pair
__device__ __forceinline__ uint64_t pc_pair(float lo, float hi)
{
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
    return v;
}
__device__ __forceinline__ float pc_lo(uint64_t v)
{
    float lo;
    asm("{\n\t.reg .f32 hi;\n\tmov.b64 {%0, hi}, %1;\n\t}" : "=f"(lo) : "l"(v));
    return lo;
}
__device__ __forceinline__ float pc_hi(uint64_t v)
{
    float hi;
    asm("{\n\t.reg .f32 lo;\n\tmov.b64 {lo, %0}, %1;\n\t}" : "=f"(hi) : "l"(v));
    return hi;
}
__device__ __forceinline__ uint64_t pc_fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t pc_add2(uint64_t a, uint64_t b)
{
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// a unit of a request: rows, keys that any of them sees, key tiles (one even if there is nothing to see: its rows become zero), cost
struct PcUnit {
    uint32_t rows, keys, tiles, weight;
};
template <int D>
__device__ __forceinline__ PcUnit pc_unit(const PagedAttn &a, const PagedReq &q, uint32_t tile)
{
    constexpr uint32_t TR = PcCfg<D>::kUnitRows;
    PcUnit u;
    const uint32_t all = q.n * a.group, m0 = tile * TR;
    u.rows = min(TR, all - m0);
    const int32_t last = q.pos0 + (int32_t)a.by_group(m0 + u.rows - 1u);
    u.keys = last < 0 ? 0u : min((uint32_t)last + 1u, q.len);
    u.tiles = max(1u, (u.keys + kPcKeys - 1u) / kPcKeys);
    u.weight = u.rows > 128u ? 2u : 1u;
    return u;
}

// the CTA's way through its units; every role walks it for itself
template <int D>
struct PcWalk {
    unsigned long long x, x_end;                       // cost before the next key tile, and where the CTA's range ends
    uint32_t h, r, tile, kt0, kt1;                     // this segment: key tiles kt0 .. kt1 - 1 of the unit
    bool by_unit;                                      // the line's parts are whole units, not key tiles
    PagedReq rq;
    PcUnit u;
    __device__ __forceinline__ static bool mine(const PagedAttn &a, const PagedReq &q) { return q.n * a.group > a.row_lo && q.n * a.group <= a.row_hi; }
    __device__ __forceinline__ void cut()
    {
        const unsigned long long left = x_end - x;     // tiles whose first cost unit lies before x_end
        kt1 = by_unit ? u.tiles : (uint32_t)min((unsigned long long)u.tiles, kt0 + (left + u.weight - 1u) / u.weight);
    }
    // Key tiles from this one on hold keys that not all of the unit's rows see, and are looked through.  (The position that its first row
    // has is the last one that all of them see.)
    __device__ __forceinline__ uint32_t looked(const PagedAttn &a) const
    {
        const int32_t low = rq.pos0 + (int32_t)a.by_group(tile * PcCfg<D>::kUnitRows);
        if ((int32_t)u.keys - 1 <= low) return u.tiles;
        return low < (int32_t)kPcKeys - 1 ? 0u : (uint32_t)(low - (int32_t)kPcKeys + 1) / kPcKeys + 1u;
    }
    // the next segment; false: there is none
    __device__ __forceinline__ bool next(const PagedAttn &a)
    {
        x += by_unit ? 1ull : (unsigned long long)(kt1 - kt0) * u.weight + (kt1 == u.tiles ? PcCfg<D>::kEnd : 0u);
        if (x >= x_end) return false;
        kt0 = 0;
        if (++tile * PcCfg<D>::kUnitRows >= rq.n * a.group) {
            tile = 0;
            do {
                if (++r == a.requests) {
                    r = 0;
                    ++h;
                }
                rq = paged_req<true>(a, r);
            } while (!mine(a, rq) && h < a.hkv);       // (there is one, unless the lengths change under the kernel)
            if (h >= a.hkv) return false;
        }
        u = pc_unit<D>(a, rq, tile);
        cut();
        return true;
    }
};

static_assert(sizeof(PcWalk<64>) <= 80, "fits");

template <int D>
__global__ void __launch_bounds__(PcCfg<D>::kThreads, 1)
k_attn_chunk(PagedAttn a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, PcCut *cuts)
{
    using CF = PcCfg<D>;
    extern __shared__ __align__(1024) unsigned char pc_smem[];
    unsigned char *smem = pc_smem;
    const uint32_t s0 = (uint32_t)__cvta_generic_to_shared(smem);
    const uint32_t tid = threadIdx.x, lane = tid & 31u;
    const int warp = __shfl_sync(0xffffffffu, (int)(tid >> 5), 0);
    const uint32_t ring = s0 + CF::kRingOff, full0 = s0 + CF::kBarOff, empty0 = full0 + 8u * CF::kStages, q_full = empty0 + 8u * CF::kStages,
                   q_free = q_full + 8u, s_full0 = q_free + 8u, p_full0 = s_full0 + 16u, p_half0 = p_full0 + 16u, o_full0 = p_half0 + 16u, pv_done0 = o_full0 + 16u,
                   done_bar = pv_done0 + 16u, w_full0 = done_bar + 8u, v_go0 = w_full0 + 8u * CF::kLook;
    float2 *sm_ml = (float2 *)(smem + CF::kBarOff + CF::kBars * 8);            // [128]
    uint32_t *tmem_slot = (uint32_t *)(sm_ml + 128), &sm_units = tmem_slot[1], &sm_two = tmem_slot[2], &sm_cost = tmem_slot[3], *sm_warp = tmem_slot + 8;
    volatile uint32_t *wild_s = tmem_slot + 4;         // [2]: the slot's P V is done by its softmax warps
    volatile uint32_t *found = tmem_slot + 24;         // [kLook][2]: what the two warps found in the values of a key tile
    asm volatile("griddepcontrol.launch_dependents;");
    if (tid == 0) {
        auto init = [&](uint32_t bar, uint32_t n, uint32_t count) {
            for (uint32_t i = 0; i < n; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar + 8u * i), "r"(count) : "memory");
        };
        init(full0, 2u * CF::kStages, 1u);
        init(q_full, 1u, CF::kSoftWarps);
        init(q_free, 1u, 1u);
        init(s_full0, 2u, 1u);
        init(p_full0, 4u, 4u);                         // (and p_half0)
        init(o_full0, 2u, 1u);
        init(pv_done0, 3u, 1u);                        // (and done_bar)
        init(w_full0, CF::kLook, 2u);
        init(v_go0, CF::kLook, 1u);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&kmap) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&vmap) : "memory");
        sm_units = sm_two = sm_cost = 0u;
    }
    if (warp == CF::kMmaWarp) {
        const uint32_t slot_addr = (uint32_t)__cvta_generic_to_shared(tmem_slot);
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot_addr), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    __syncthreads();
    // Behind k_attn_paged this does not wait for it: the two share inputs only, and the other lets this one start when its own
    // predecessors are complete.  CTAs come as the others leave (three chunks of prompts beside 29 single tokens: 64 us, 75 before);
    // the wait is at the end, for those who rely on both.
    if (!a.second) asm volatile("griddepcontrol.wait;" ::: "memory");
    // ---- every request's cost and units, of one KV head (over the ring, which is empty)
    uint32_t *first = (uint32_t *)(smem + CF::kRingOff), *units = first + kPaMaxRequests;
    const uint32_t R = a.requests, G = a.group, me = blockIdx.x;
    auto cost_of = [&](const PagedReq &q, uint32_t t) {
        if (t * CF::kUnitRows >= q.n * G) return 0u;
        const PcUnit u = pc_unit<D>(a, q, t);
        return u.tiles * u.weight + CF::kEnd;
    };
    auto note = [&](uint32_t r, const PagedReq &q, uint32_t cost) {
        const uint32_t n = cost ? (q.n * G + CF::kUnitRows - 1u) / CF::kUnitRows : 0u;
        first[r] = cost;
        units[r] = n;
        if (!n) return;
        atomicAdd(&sm_cost, cost);
        atomicAdd(&sm_units, n);
        if (CF::kTiles == 2 && q.n * G > 128u) sm_two = 1u;
    };
    const uint32_t per = (R + CF::kThreads - 1) / CF::kThreads, ra = min(R, tid * per), rb = min(R, ra + per);
    if (R <= 2u * CF::kThreads / 32u) {                // few requests, perhaps of many tiles: a warp each
        for (uint32_t r = (uint32_t)warp; r < R; r += CF::kThreads / 32) {
            const PagedReq q = paged_req<true>(a, r);
            uint32_t own = 0;
            if (PcWalk<D>::mine(a, q))
                for (uint32_t t = lane; t * CF::kUnitRows < q.n * G; t += 32u) own += cost_of(q, t);
            own = __reduce_add_sync(0xffffffffu, own);
            if (lane == 0) note(r, q, own);
        }
    } else {
        for (uint32_t r = ra; r < rb; ++r) {
            const PagedReq q = paged_req<true>(a, r);
            uint32_t own = 0;
            if (PcWalk<D>::mine(a, q))
                for (uint32_t t = 0; t * CF::kUnitRows < q.n * G; ++t) own += cost_of(q, t);
            note(r, q, own);
        }
    }
    __syncthreads();
    // What the line is cut into: key tiles; or whole units where there is room for one per CTA and they are short, so that cutting them
    // would cost more than it saves (figures at kPcShortUnit)
    const bool by_unit = (unsigned long long)sm_units * a.hkv <= gridDim.x && sm_cost <= (kPcShortUnit + CF::kEnd) * sm_units;
    const uint32_t total = by_unit ? sm_units : sm_cost;
    {
        const uint32_t *const own_of = by_unit ? units : first;
        uint32_t own = 0, before = 0;
        for (uint32_t r = ra; r < rb; ++r) own += own_of[r];
        uint32_t v = own;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t w = __shfl_up_sync(0xffffffffu, v, d);
            if (lane >= (uint32_t)d) v += w;
        }
        if (lane == 31u) sm_warp[warp] = v;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < CF::kThreads / 32; ++w)
            if (w < warp) before += sm_warp[w];
        before += v - own;
        for (uint32_t r = ra; r < rb; ++r) {
            const uint32_t c = own_of[r];
            first[r] = before;
            before += c;
        }
        __syncthreads();
    }
    const unsigned long long W = (unsigned long long)total * a.hkv;
    // CTAs: one for every four key tiles, or every unit if that is more; with units of two row tiles a range is at least as long as a
    // key tile's cost, so that every CTA between the first and the last of a unit has a key tile of it
    unsigned long long n_max = by_unit ? W : max((unsigned long long)sm_units * a.hkv, (W + kPcMinCost - 1u) / kPcMinCost);
    if (sm_two && !by_unit) n_max = min(n_max, max(W / 2u, 1ull));
    const uint32_t N = (uint32_t)min((unsigned long long)gridDim.x, n_max);
    auto part_of = [&](uint32_t c) { return W < 1u << 24 ? (unsigned long long)((uint32_t)W * c / N) : W * c / N; };      // (N at most 256)
    auto cta_of = [&](unsigned long long y) {          // the last c with part_of(c) <= y
        return W < 1u << 24 ? (((uint32_t)y + 1u) * N - 1u) / (uint32_t)W : (uint32_t)(((y + 1ull) * N - 1ull) / W);
    };
    if (me >= N) {
        if (tid == 0) cuts[me].parts = 0u;
        if (warp == CF::kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(*tmem_slot), "r"(512u) : "memory");
        if (a.second) asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }
    PcWalk<D> w;
    w.by_unit = by_unit;
    w.x = part_of(me);
    w.x_end = part_of(me + 1u);
    {
        w.h = W < 1u << 24 ? (uint32_t)w.x / total : (uint32_t)(w.x / total);
        uint32_t off = (uint32_t)(w.x - (unsigned long long)w.h * total), lo = 0, hi = R;
        while (hi - lo > 1u) {                         // the last request with first[r] <= off
            const uint32_t mid = (lo + hi) / 2u;
            if (first[mid] <= off) lo = mid;
            else hi = mid;
        }
        w.r = lo;
        off -= first[lo];
        w.rq = paged_req<true>(a, lo);
        w.tile = 0;
        if (by_unit) {
            w.tile = off;
            off = 0;
        }
        for (; !by_unit; w.tile += 32u) {              // its tile: 32 at a time (off is less than the request's cost)
            const uint32_t c = cost_of(w.rq, w.tile + lane);
            uint32_t v = c;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const uint32_t u = __shfl_up_sync(0xffffffffu, v, d);
                if (lane >= (uint32_t)d) v += u;
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, v > off);
            if (hit) {
                const int l = __ffs(hit) - 1;
                off -= __shfl_sync(0xffffffffu, v - c, l);
                w.tile += (uint32_t)l;
                break;
            }
            if ((w.tile + 32u) * CF::kUnitRows >= w.rq.n * G) break;           // (not so, unless the lengths change under the kernel)
            off -= __shfl_sync(0xffffffffu, v, 31);
        }
        w.u = pc_unit<D>(a, w.rq, w.tile);
        w.kt0 = min((off + w.u.weight - 1u) / w.u.weight, w.u.tiles);          // a tile that began before this range is its predecessor's
        w.x = w.x - off + w.kt0 * w.u.weight;
        w.kt1 = w.kt0;
        if (w.kt0 < w.u.tiles && w.x < w.x_end) w.cut();
    }
    // (an empty first segment: the range begins inside the last tile of a unit)
    bool work = w.kt1 > w.kt0 || w.next(a);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");               // (the ring held the requests' costs)
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    bool ok = true;

    if (warp == CF::kLoadWarp) {
        if (CF::kDeal) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        // ---- K and V of every key tile, in the order K0 V0 K1 V1 ..; a box is a page's (at most 128) keys and 64 dimensions
        const uint32_t bp = min(1u << a.log_page, kPcKeys), boxes = kPcKeys / bp * (CF::kUD / 64);
        const uint32_t bk = lane / (CF::kUD / 64), panel = lane % (CF::kUD / 64);      // of lane < boxes: keys bk * bp .., 64 dimensions
        uint32_t n = 0, n_look = 0;
        for (bool more = work; more && ok; more = w.next(a)) {
            const uint32_t look0 = max(w.looked(a), w.kt0);
            const int32_t *pages = a.table + (size_t)w.r * a.width;
            auto page_of = [&](uint32_t kt) {
                const uint32_t key = kt * kPcKeys + bk * bp;
                return lane < boxes && kt < w.kt1 && key < w.u.keys ? __ldcg(pages + (key >> a.log_page)) : 0;
            };
            int32_t page = page_of(w.kt0);
            for (uint32_t kt = w.kt0; kt < w.kt1 && ok; ++kt) {
                const uint32_t key = kt * kPcKeys + bk * bp, row = key & ((1u << a.log_page) - 1u);
                const bool on = lane < boxes && key < w.u.keys;
                const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, on)) * bp * 128u;
                const int32_t page_n = page_of(kt + 1u);
#pragma unroll
                for (uint32_t i = 0; i < 2u * CF::kNU; ++i, ++n) {
                    const uint32_t st = n % CF::kStages, bar = full0 + 8u * st;
                    ok = ok && pa_wait(empty0 + 8u * st, (n / CF::kStages & 1u) ^ 1u);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    if (lane == 0) asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1;\n\t}" ::"r"(bar), "r"(bytes) : "memory");
                    __syncwarp();
                    if (on)
                        asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                                     :: "r"(ring + st * CF::kUnit + panel * CF::kPanel + bk * bp * 128u), "l"(i < (uint32_t)CF::kNU ? &kmap : &vmap),
                                        "r"((i % CF::kNU) * CF::kUD + panel * 64u), "r"(w.h), "r"(row), "r"(page), "r"(bar) : "memory");
                    __syncwarp();
                }
                // (a parity of the ring's barriers alone does not tell a stage that is still to come from one two rounds before it: the
                // warp that goes through all of them says when)
                if (kt >= look0) {
                    if (lane == 0 && ok) pc_arrive(v_go0 + 8u * (n_look % CF::kLook));
                    ++n_look;
                }
                page = page_n;
            }
        }
        // the copies that may still be in flight (the tensor core's warp waits for them too, unless it gave up)
        bool landed = true;
        for (uint32_t j = n > CF::kStages ? n - CF::kStages : 0u; j < n; ++j)
            landed = pa_wait(full0 + 8u * (j % CF::kStages), j / CF::kStages & 1u) && landed;
        ok = ok && landed;
    } else if (warp == CF::kMmaWarp) {
        if (CF::kDeal) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        uint32_t el;
        asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(el));
        uint32_t n0 = 0, seg = 0, p0 = 0, p1 = 0;      // before this segment: ring units, segments, steps of the two slots
        for (bool more = work; more && ok; more = w.next(a), ++seg) {
            const bool two = w.u.weight == 2u;         // two row tiles: a key tile is two steps
            const uint32_t tiles = w.kt1 - w.kt0, steps = two ? 2u * tiles : tiles;
            auto wait = [&](uint32_t bar, uint32_t parity) {
                ok = ok && pa_wait(bar, parity);
                ok = __all_sync(0xffffffffu, ok);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            };
            auto unit = [&](uint32_t j, uint32_t i) { return n0 + (2u * j + i) * CF::kNU; };   // key tile j's K (i = 0) or V (1)
            auto qk = [&](uint32_t st) {
                const uint32_t slot = st & 1u, j = two ? st >> 1 : st, q = s0 + (two ? slot * CF::kQTile : 0u);
                const bool last_use = !two || slot;
#pragma unroll
                for (int c = 0; c < CF::kNU; ++c) {
                    const uint32_t n = unit(j, 0u) + c, rs = n % CF::kStages;
                    wait(full0 + 8u * rs, n / CF::kStages & 1u);
                    if (!ok) return;
#pragma unroll
                    for (int kk = 0; kk < CF::kUD / 16; ++kk)
                        pc_mma_ss(el, tmem + slot * 128u, pc_desc(q + (c * (CF::kUD / 64) + kk / 4) * CF::kPanel + (kk % 4) * 32u, 16u, 1024u),
                                  pc_desc(ring + rs * CF::kUnit + (kk / 4) * CF::kPanel + (kk % 4) * 32u, 16u, 1024u), pc_idesc(128u, 0u), (c || kk) ? 1u : 0u);
                    if (last_use) pc_commit(el, empty0 + 8u * rs);
                }
                pc_commit(el, s_full0 + 8u * slot);
                if (st + 1u == steps) pc_commit(el, q_free);
            };
            wait(q_full, seg & 1u);
            // Q K^T of a step two steps ahead of its P V
            for (uint32_t it = 0; it < steps + 2u && ok; ++it) {
                if (it >= 2u) {
                    const uint32_t st = it - 2u, slot = st & 1u, j = two ? st >> 1 : st, kt = w.kt0 + j;
                    const bool last_use = !two || slot;
                    const uint32_t valid = w.u.keys > kt * kPcKeys ? min(kPcKeys, w.u.keys - kt * kPcKeys) : 0u;
                    const uint32_t p_par = ((slot ? p1 : p0) + (st >> 1)) & 1u;
                    wait(p_half0 + 8u * slot, p_par);      // the first 64 keys' probabilities
                    if (!ok) break;
                    const bool wild = wild_s[slot] != 0u;
                    const uint32_t o = tmem + CF::kO + (CF::kTiles == 2 ? slot * 128u : 0u);
                    const uint32_t acc = (CF::kTiles == 2 ? st >= 2u : st >= 1u) ? 1u : 0u;
#pragma unroll
                    for (int c = 0; c < CF::kNU; ++c) {
                        const uint32_t n = unit(j, 1u) + c, rs = n % CF::kStages, base = ring + rs * CF::kUnit;
                        wait(full0 + 8u * rs, n / CF::kStages & 1u);
                        if (!ok) break;
                        if (valid & 15u) {                 // (both steps of a tile do it: the same zeros)
                            const uint32_t z0 = valid, z1 = (valid + 15u) & ~15u;
                            for (uint32_t i = lane; i < (z1 - z0) * (CF::kUD / 8); i += 32u) {
                                const uint32_t row = z0 + i / (CF::kUD / 8), p = i % (CF::kUD / 8);
                                asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(base + (p >> 3) * CF::kPanel + row * 128u + (p & 7u) * 16u), "r"(0u) : "memory");
                            }
                            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                            __syncwarp();
                        }
                        auto pv = [&](uint32_t kk) {
                            pc_mma_ts(el, o + c * CF::kUD, tmem + slot * 128u + kk * 8u, pc_desc(base + kk * 2048u, CF::kPanel, 1024u), pc_idesc(CF::kUD, 1u), kk ? 1u : acc);
                        };
                        const uint32_t steps16 = wild ? 0u : (valid + 15u) / 16u;
                        if (steps16 >= 4u) {
#pragma unroll
                            for (uint32_t kk = 0; kk < 4u; ++kk) pv(kk);
                        } else {
                            for (uint32_t kk = 0; kk < steps16; ++kk) pv(kk);
                        }
                        if (c == 0) {
                            wait(p_full0 + 8u * slot, p_par);
                            if (!ok) break;
                        }
                        if (steps16 == 8u) {
#pragma unroll
                            for (uint32_t kk = 4; kk < 8u; ++kk) pv(kk);
                        } else {
                            for (uint32_t kk = 4; kk < steps16; ++kk) pv(kk);
                        }
                        if (last_use) pc_commit(el, empty0 + 8u * rs);
                    }
                    if (!ok) break;
                    if (CF::kTiles == 1) pc_commit(el, pv_done0 + 8u * slot);
                    if (st + 1u == steps || (CF::kTiles == 2 && st + 2u == steps)) pc_commit(el, o_full0 + 8u * (CF::kTiles == 2 ? slot : 0u));
                    if (CF::kTiles == 2 && steps == 1u) pc_commit(el, o_full0 + 8u);       // (the other slot has no step)
                }
                if (it < steps) qk(it);
            }
            n0 += 2u * tiles * CF::kNU;
            p0 += (steps + 1u) >> 1;
            p1 += steps >> 1;
        }
        pc_commit(el, done_bar);
    } else if (warp >= CF::kScanWarp) {
        if (CF::kDeal) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        // ---- values that are not finite, in the key tiles that not all rows see
        const uint32_t half = (uint32_t)(warp - CF::kScanWarp);
        uint32_t n0 = 0, n_look = 0;
        for (bool more = work; more && ok; more = w.next(a)) {
            for (uint32_t kt = max(w.looked(a), w.kt0); kt < w.kt1 && ok; ++kt, ++n_look) {
                const uint32_t keys = min(kPcKeys, w.u.keys - kt * kPcKeys);
                uint32_t big = 0;
                ok = ok && pa_wait(v_go0 + 8u * (n_look % CF::kLook), n_look / CF::kLook & 1u);
#pragma unroll
                for (int c = 0; c < CF::kNU; ++c) {
                    const uint32_t n = n0 + (2u * (kt - w.kt0) + 1u) * CF::kNU + c, rs = n % CF::kStages;
                    ok = ok && pa_wait(full0 + 8u * rs, n / CF::kStages & 1u);
#pragma unroll 8
                    for (uint32_t i = half * 32u + lane; i < keys * (CF::kUD / 8); i += 64u) {
                        uint4 v;
                        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                                     : "r"(ring + rs * CF::kUnit + (i & 7u) * 16u + (i >> 3) / (CF::kUD / 64) * 128u + (i >> 3) % (CF::kUD / 64) * CF::kPanel) : "memory");
                        big = pa_larger(pa_larger(pa_larger(pa_larger(big, v.x), v.y), v.z), v.w);
                    }
                }
                ok = __all_sync(0xffffffffu, ok);
                const bool any = __any_sync(0xffffffffu, pa_wild(big));
                if (lane == 0) {
                    found[n_look % CF::kLook * 2u + half] = any;
                    pc_arrive(w_full0 + 8u * (n_look % CF::kLook));
                }
                __syncwarp();
            }
            n0 += 2u * (w.kt1 - w.kt0) * CF::kNU;
        }
    } else {
        if (CF::kDeal) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        // ---- softmax: group gr of four warps has a slot (heads of 256: both); a thread is a row
        const uint32_t gr = (uint32_t)warp >> 2, row_t = tid & 127u, lanes = ((uint32_t)warp & 3u) << 21;
        const float sl2 = a.scale * 1.4426950408889634f;
        uint32_t c0s = 0, c1s = 0, seg = 0, n0 = 0, n_look = 0;   // before this segment: steps of the slots, segments, ring units, tiles looked through
        if (tid == 0) cuts[me].parts = 0u;
        // (the way through the units lies in shared memory between segments: beside a row of scores there is no room for it)
        PcWalk<D> *const kept = (PcWalk<D> *)(smem + CF::kWalkOff) + warp;
        if (lane == 0) *kept = w;
        __syncwarp();
        for (bool more = work; more; ++seg) {
            PcWalk<D> w = *kept;
            const bool two = w.u.weight == 2u;
            const uint32_t kt0 = w.kt0, tiles = w.kt1 - kt0, steps = two ? 2u * tiles : tiles;
            // ---- Q: rows of the unit into [tile][64 dimensions][128 rows], swizzled
            if (seg) ok = ok && pa_wait(q_free, (seg - 1u) & 1u);
            const uint32_t m0 = w.tile * CF::kUnitRows, tok0 = a.by_group(m0), rem0 = m0 - tok0 * G;
            {
                constexpr uint32_t CH = D / 8, STEP = CF::kSoftWarps * 32 / CH;        // 16-byte pieces of a row, rows at a time
                const uint32_t ch = tid % CH;
                const __nv_bfloat16 *src = a.q + (size_t)(w.rq.row0 + tok0) * a.q_stride + (size_t)w.h * G * D + ch * 8u;
#pragma unroll 4
                for (uint32_t m = tid / CH; m < w.u.rows; m += STEP) {       // (what lies in rows behind the last one stays in them)
                    const uint32_t q = rem0 + m, tok = a.by_group(q), rr = m & 127u;
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                                 ::"r"(s0 + (m >> 7) * CF::kQTile + (ch >> 3) * CF::kPanel + rr * 128u + ((ch ^ rr) & 7u) * 16u),
                                 "l"(src + tok * a.q_stride + (size_t)(q - tok * G) * D) : "memory");
                }
                cp_async_commit();
                cp_async_wait<0>();
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) pc_arrive(q_full);
            // ---- this thread's row
            const uint32_t m = (two ? gr * 128u : 0u) + row_t;                 // in the unit
            const bool valid = m < w.u.rows;
            // (the last position that it sees: of those that the table holds, what lies behind them in the tile was not copied)
            const int32_t len1 = (int32_t)w.rq.len - 1, limit = valid ? min(w.rq.pos0 + (int32_t)a.by_group(m0 + m), len1) : -1;
            const bool warp_on = (m & ~31u) < w.u.rows;                        // (warp uniform) some row is there
            const int32_t low_warp = min(w.rq.pos0 + (int32_t)a.by_group(m0 + (m & ~31u)), len1);
            const uint32_t look0 = max(w.looked(a), w.kt0);
            const uint32_t o_at = tmem + lanes + CF::kO + (CF::kTiles == 2 ? gr * 128u : 0u);
            float mb = -INFINITY, l = 0.f;             // the maximum that the sums are relative to (in units of log2), the denominator
            bool any = false;                          // (group uniform) the accumulator holds something
            const uint32_t stride = CF::kTiles == 2 ? 2u : 1u;
            // One accumulator for both slots: the P V of the step before, done.  (Its slot's P V before that is: the scores that this warp
            // has seen came behind it, so the parity tells.)
            auto pv_of = [&](uint32_t of) { ok = ok && pa_wait(pv_done0 + 8u * (of & 1u), ((of & 1u ? c1s : c0s) + (of >> 1)) & 1u); };
            for (uint32_t st = CF::kTiles == 2 ? gr : 0u; st < steps; st += stride) {
                const uint32_t slot = st & 1u, j = two ? st >> 1 : st, kt = kt0 + j, s_at = tmem + lanes + slot * 128u;
                const int32_t key0 = (int32_t)(kt * kPcKeys);
                auto before = [&]() {
                    if (CF::kTiles == 2) return;
                    pv_of(st - 1u);
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                };
                ok = ok && pa_wait(s_full0 + 8u * slot, ((slot ? c1s : c0s) + (st >> 1)) & 1u);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                bool wild = false;
                ok = __all_sync(0xffffffffu, ok);
                if (warp_on && ok) {
                    uint32_t s[128];
#pragma unroll
                    for (int c = 0; c < 4; ++c) pc_ld32(s_at + 32u * c, s + 32 * c);
                    pc_wait_ld();
#pragma unroll
                    for (int c = 0; c < 4; ++c) pc_pin(s + 32 * c);
                    if (key0 + (int32_t)kPcKeys - 1 > low_warp) {              // (warp uniform)
#pragma unroll
                        for (int c = 0; c < 128; ++c)
                            if (key0 + c > limit) s[c] = 0xff800000u;
                    }
                    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int c = 0; c < 128; c += 2) mx[c / 2 & 3] = pc_max3(mx[c / 2 & 3], __uint_as_float(s[c]), __uint_as_float(s[c + 1]));
                    const float top = pc_max3(fmaxf(mx[0], mx[1]), mx[2], mx[3]) * sl2;
                    if (__any_sync(0xffffffffu, valid && top > mb + 8.f)) {    // (false for -inf; the first maximum of a row is larger than -inf)
                        const float mn = fmaxf(mb, top), f = pa_exp2(mb - (mn == -INFINITY ? 0.f : mn));
                        mb = mn;
                        l *= f;
                        if (any) {
                            before();
#pragma unroll 1
                            for (int c = 0; c < D / 32; ++c) {
                                uint32_t o[32];
                                pc_ld32(o_at + 32u * c, o);
                                pc_wait_ld();
                                pc_pin(o);
#pragma unroll
                                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                                pc_st32(o_at + 32u * c, o);
                            }
                            pc_wait_st();
                        }
                    }
                    const float nb = mb == -INFINITY ? 0.f : -mb;
                    uint64_t la = 0, lb = 0;           // pairs of sums
                    const uint64_t sl2_2 = pc_pair(sl2, sl2), nb_2 = pc_pair(nb, nb);
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
#pragma unroll
                        for (int c = 64 * half; c < 64 * half + 64; c += 2) {
                            const uint64_t x = pc_fma2(pc_pair(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), sl2_2, nb_2);
                            const float p0 = pa_exp2(pc_lo(x)), p1 = pa_exp2(pc_hi(x));
                            if (c & 2) la = pc_add2(la, pc_pair(p0, p1));
                            else lb = pc_add2(lb, pc_pair(p0, p1));
                            s[c / 2] = pa_pack(p0, p1);
                        }
                        pc_st32(s_at + 32u * half, s + 32 * half);
                        pc_wait_st();
                        if (half == 0) {
                            if (kt >= look0) {         // (group uniform)
                                const uint32_t k = n_look + kt - look0;
                                ok = ok && pa_wait(w_full0 + 8u * (k % CF::kLook), k / CF::kLook & 1u);
                                wild = found[k % CF::kLook * 2u] | found[k % CF::kLook * 2u + 1u];
                            }
                            if (row_t == 0) wild_s[slot] = wild;
                            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                            __syncwarp();
                            if (lane == 0) pc_arrive(p_half0 + 8u * slot);
                        }
                    }
                    la = pc_add2(la, lb);
                    l += pc_lo(la) + pc_hi(la);
                    if (wild) {
                        if (any) before();
                        // P V of this tile for this thread's row: what the row does not see is left out
#pragma unroll 1
                        for (int c = 0; c < D / 32; ++c) {
                            uint32_t o[32];
                            if (any) {
                                pc_ld32(o_at + 32u * c, o);
                                pc_wait_ld();
                                pc_pin(o);
                            } else {
#pragma unroll
                                for (int i = 0; i < 32; ++i) o[i] = 0u;
                            }
                            const uint32_t n = n0 + (2u * j + 1u) * CF::kNU + c / (CF::kUD / 32), rs = n % CF::kStages, cc = c % (CF::kUD / 32);
                            const uint32_t vb = ring + rs * CF::kUnit + (cc >> 1) * CF::kPanel;
#pragma unroll 1
                            for (uint32_t k = 0; k < kPcKeys; ++k) {
                                uint32_t pp;
                                asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(pp) : "r"(s_at + k / 2u) : "memory");
                                pc_wait_ld();
                                asm volatile("" : "+r"(pp));
                                const float p = __uint_as_float(k & 1u ? pp & 0xffff0000u : pp << 16);
                                if (key0 + (int32_t)k <= limit) {
#pragma unroll
                                    for (uint32_t q = 0; q < 4u; ++q) {
                                        uint32_t v[4];
                                        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                                                     : "r"(vb + k * 128u + ((((cc & 1u) * 4u + q) ^ k) & 7u) * 16u) : "memory");
#pragma unroll
                                        for (int e = 0; e < 4; ++e) {
                                            o[8 * q + 2 * e] = __float_as_uint(fmaf(p, __uint_as_float(v[e] << 16), __uint_as_float(o[8 * q + 2 * e])));
                                            o[8 * q + 2 * e + 1] = __float_as_uint(fmaf(p, __uint_as_float(v[e] & 0xffff0000u), __uint_as_float(o[8 * q + 2 * e + 1])));
                                        }
                                    }
                                }
                                __syncwarp();
                            }
                            pc_st32(o_at + 32u * c, o);
                        }
                        pc_wait_st();
                    }
                } else {
                    __syncwarp();
                    if (lane == 0) pc_arrive(p_half0 + 8u * slot);
                }
                any = true;
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) pc_arrive(p_full0 + 8u * slot);
            }
            if (CF::kTiles == 1) {
                if (steps > 1u) pv_of(steps - 2u);
                pv_of(steps - 1u);
            }
            c0s += (steps + 1u) >> 1;
            c1s += steps >> 1;
            n0 += 2u * tiles * CF::kNU;
            n_look += kt0 + tiles - min(kt0 + tiles, look0);
            // ---- the unit's sums
            asm volatile("" ::: "memory");
            w = *kept;
            ok = ok && pa_wait(o_full0 + 8u * gr, seg & 1u);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (!ok) l = __int_as_float(0x7fc00000);
            const bool whole = w.kt0 == 0u && w.kt1 == w.u.tiles;
            const bool sees = limit >= 0 && w.u.keys > 0u;                     // (of this row: anything at all, in any segment)
            const unsigned long long x0 = w.x - (unsigned long long)w.kt0 * w.u.weight;
            const uint32_t slot_n = 2u * me + (w.kt0 ? 0u : 1u);               // a unit's first part is this CTA's last segment
            float *part = a.part + (size_t)slot_n * CF::kPart;
            if (!whole && w.kt0 == 0u) {
                if (tid == 0)                          // (at most one of a CTA: its last)
                    cuts[me] = {cta_of(x0 + (unsigned long long)(w.u.tiles - 1u) * w.u.weight) - me + 1u, slot_n, w.rq.row0, m0, w.u.rows, w.h, w.rq.pos0, w.u.keys};
            }
            const bool merge = CF::kTiles == 2 && !two && steps > 1u;          // both groups have a part of the same rows
            const bool mine = two || gr == 0u;                                 // writes this row's result or part
            float other_l = 0.f, f_own = 1.f, f_other = 0.f;
            const uint32_t xbuf = s0 + CF::kQTile;                             // [columns][128 rows] floats: the second row tile's Q, unused here
            constexpr int XC = CF::kQTile / 512 < D ? (int)(CF::kQTile / 512) : D;     // columns that fit
            __nv_bfloat16 *dst = a.out;
            if (valid) {
                const uint32_t q = m0 + m, tok = a.by_group(q);
                dst = a.out + ((size_t)(w.rq.row0 + tok) * a.hq + (size_t)w.h * G + (q - tok * G)) * D;
            }
            if (merge) {
                // (Q of this unit's second tile is not there, and the next unit's is written behind this)
                if (gr == 1u) sm_ml[row_t] = make_float2(mb, l);
                asm volatile("barrier.cta.sync 3, 256;" ::: "memory");
                if (gr == 0u) {
                    const float2 o = sm_ml[row_t];
                    const float mn = fmaxf(mb, o.x), mz = mn == -INFINITY ? 0.f : mn;
                    f_own = pa_exp2(mb - mz);
                    f_other = pa_exp2(o.x - mz);
                    other_l = o.y;
                    mb = mn;
                    l = l * f_own + other_l * f_other;
                }
            }
            const float inv = 1.f / l;
#pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += merge ? XC : D) {
                const int c1 = merge ? min(D, c0 + XC) : D;
                if (merge) {
                    if (gr == 1u && warp_on) {
#pragma unroll 1
                        for (int c = c0; c < c1; c += 32) {
                            uint32_t o[32];
                            pc_ld32(o_at + c, o);
                            pc_wait_ld();
                            pc_pin(o);
#pragma unroll
                            for (int i = 0; i < 32; ++i) asm volatile("st.shared.u32 [%0], %1;" ::"r"(xbuf + ((c - c0 + i) * 128u + row_t) * 4u), "r"(o[i]) : "memory");
                        }
                    }
                    asm volatile("barrier.cta.sync 3, 256;" ::: "memory");
                }
                if (warp_on && mine) {
#pragma unroll 1
                    for (int c = c0; c < c1; c += 32) {
                        uint32_t o[32];
                        pc_ld32(o_at + c, o);
                        pc_wait_ld();
                        pc_pin(o);
                        if (merge) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) {
                                float v = __uint_as_float(o[i]) * f_own;
                                uint32_t u;
                                asm volatile("ld.shared.u32 %0, [%1];" : "=r"(u) : "r"(xbuf + ((c - c0 + i) * 128u + row_t) * 4u) : "memory");
                                v = fmaf(__uint_as_float(u), f_other, v);
                                o[i] = __float_as_uint(v);
                            }
                        }
                        if (whole) {
                            if (valid) {
#pragma unroll
                                for (int i = 0; i < 32; i += 8) {
                                    uint32_t v[4];
#pragma unroll
                                    for (int e = 0; e < 4; ++e)
                                        v[e] = sees || !ok ? pa_pack(__uint_as_float(o[i + 2 * e]) * inv, __uint_as_float(o[i + 2 * e + 1]) * inv) : 0u;
                                    *(uint4 *)(dst + c + i) = make_uint4(v[0], v[1], v[2], v[3]);
                                }
                            }
                        } else if (valid) {
#pragma unroll
                            for (int i = 0; i < 32; i += 4)
                                *(uint4 *)(part + (((m >> 7) * (D / 4) + (c + i) / 4) * 128u + (m & 127u)) * 4u) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                        }
                    }
                }
                if (merge) asm volatile("barrier.cta.sync 3, 256;" ::: "memory");
            }
            if (!whole && valid && mine) *(float2 *)(part + CF::kUnitRows * D + 2u * m) = make_float2(mb, l);
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");   // (the accumulators are read: the next unit's may be written)
            more = w.next(a);
            __syncwarp();
            if (lane == 0) *kept = w;
            __syncwarp();
        }
    }
    __syncwarp();
    ok = pa_wait(done_bar, 0u) && ok;                  // (the MMAs that were issued are done, whoever gave up)
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == CF::kMmaWarp) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
    if (a.second) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// The parts of the units that were cut.  grid (CTAs of k_attn_chunk, row tiles x groups of 16 dimensions), a thread per row; four parts
// of a row are requested at once.
template <int D>
__global__ void __launch_bounds__(128)
k_attn_chunk_join(PagedAttn a, const PcCut *cuts)
{
    using CF = PcCfg<D>;
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const PcCut cut = cuts[blockIdx.x];
    const uint32_t tile = blockIdx.y / (D / 16), c0 = blockIdx.y % (D / 16) * 4u, row = threadIdx.x, m = tile * 128u + row;
    if (cut.parts == 0u || m >= cut.rows) return;
    constexpr uint32_t UN = 4;
    auto part = [&](uint32_t p) { return a.part + (size_t)(p ? 2u * (blockIdx.x + p) : cut.first_slot) * CF::kPart; };
    float M = -INFINITY, L = 0.f;
    float4 v[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (uint32_t p0 = 0; p0 < cut.parts; p0 += UN) {
        float2 ml[UN];
        float4 s[UN][4];
#pragma unroll
        for (uint32_t i = 0; i < UN; ++i) {
            const float *src = part(min(p0 + i, cut.parts - 1u));
            ml[i] = p0 + i < cut.parts ? ((const float2 *)(src + CF::kUnitRows * D))[m] : make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int c = 0; c < 4; ++c) s[i][c] = ((const float4 *)src)[(size_t)(tile * (D / 4) + c0 + c) * 128u + row];
        }
        float mn = M;
#pragma unroll
        for (uint32_t i = 0; i < UN; ++i) mn = fmaxf(mn, ml[i].x);
        const float mz = mn == -INFINITY ? 0.f : mn, shrink = pa_exp2(M - mz);
        M = mn;
        L *= shrink;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            v[c].x *= shrink; v[c].y *= shrink; v[c].z *= shrink; v[c].w *= shrink;
        }
#pragma unroll
        for (uint32_t i = 0; i < UN; ++i) {
            if (p0 + i >= cut.parts) break;
            const float f = pa_exp2(ml[i].x - mz);
            L = fmaf(ml[i].y, f, L);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                v[c].x = fmaf(s[i][c].x, f, v[c].x); v[c].y = fmaf(s[i][c].y, f, v[c].y); v[c].z = fmaf(s[i][c].z, f, v[c].z); v[c].w = fmaf(s[i][c].w, f, v[c].w);
            }
        }
    }
    const uint32_t q = cut.m0 + m, tok = a.by_group(q);
    const bool sees = cut.pos0 + (int32_t)tok >= 0 && cut.keys > 0u;
    const float inv = 1.f / L;
    __nv_bfloat16 *dst = a.out + ((size_t)(cut.row0 + tok) * a.hq + (size_t)cut.head * a.group + (q - tok * a.group)) * D + c0 * 4u;
#pragma unroll
    for (int c = 0; c < 4; c += 2)
        *(uint4 *)(dst + c * 4) = sees ? make_uint4(pa_pack(v[c].x * inv, v[c].y * inv), pa_pack(v[c].z * inv, v[c].w * inv),
                                                    pa_pack(v[c + 1].x * inv, v[c + 1].y * inv), pa_pack(v[c + 1].z * inv, v[c + 1].w * inv))
                                       : make_uint4(0u, 0u, 0u, 0u);
}

}  // namespace ixb
