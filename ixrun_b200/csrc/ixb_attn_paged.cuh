// Causal attention of every request's new tokens over its pages: the form for few rows (single tokens, short drafts).
//
//   row (t, g) of request r and KV head h: new token t < q_len[r], query head h * G + g, position length[r] - q_len[r] + t
//   out = softmax(scale * q . K[0 .. position]) V[0 .. position]
//
// A request's rows of one KV head are packed, row t * G + g, eight or sixteen to a group, so a key is read once for all of them.
// Bound: HBM, every key and value once: 64 single tokens behind 3000 to 6000 keys, 16 / 8 heads of 128, take 184 us, 98 % of the copy rate;
// one behind 1100 takes 7.7 us, a chain of trips to memory (lengths, table, keys, ticket, parts).  mma.sync is used as an instruction that multiplies eight rows at a time: keys (or
// dimensions of values) are its M = 16, rows its N = 8, S^T = K Q^T and O^T = V^T P^T, so that a single token of a group of up to
// eight heads wastes none of it and its sums take half the registers of rows as M.
//
// Work: all (KV head, request, row group) pairs' blocks of keys in one line, cut into equal ranges, one per CTA, so lengths that differ
// cost nothing; a short pair is the CTA's that has its first block.  A block is a slice of 16 keys per warp (32 with heads of 64, where a slice's softmax would take longer than its
// bytes).  One warp asks for the blocks (TMA, a box per page and 64 dimensions, 128-byte swizzle) in a ring of stages K, V, K, .., across
// pairs; eight warps take their slices and keep a running softmax each, so they meet only where a pair ends, in shared memory.  A
// long pair that is cut leaves its parts in the scratch, and the CTA that comes last (a ticket) joins them in the order of the keys: the
// same bits every time for the same batch (where a pair is cut depends on all requests' lengths).
//
// Registers (-Xptxas -v): 188 bytes are spilled with heads of 256 and with sixteen rows of 128, 24 with sixteen rows of 64; without the
// path for values that are not finite 40, none and 40.
//
// Precision: q K^T bf16 x bf16 in fp32; probabilities as two bf16 numbers whose sum they are to 17 bits; a slice's P V starts from
// zero and joins the running sums by fp32 fused multiply-adds (the tensor core cuts low bits of what it adds to a large sum).
//
// Keys at and behind length are masked and their values taken as zeros, whatever lies there; a page number outside the pool is a
// page of zeros (the copy's fill).  A value that is not finite counts for the rows that see it and for no other: it shows in the
// sums of every row (zero times infinity is NaN), and the pair's blocks are then gone through again, straight from memory and token
// by token.
//
// Every wait on an mbarrier is bounded (kPaWaitLimit polls of 1.5 us) and counts the CTA's own copies; where one runs out the CTA's
// outputs become NaN.  Going through blocks again takes up to 105 us a block (sixteen tokens), so for a pair of two million
// positions it takes longer than a wait: the warp that asks for blocks waits on as long as the others say that they get on.
#pragma once
#include "ixb_common.cuh"
#include <cuda.h>

namespace ixb {

struct PagedAttn {
    const __nv_bfloat16 *q, *k, *v;
    __nv_bfloat16 *out;
    const int32_t *table, *length, *cu_rows;
    float *part;
    uint32_t *tickets;
    size_t k_stride, v_stride, q_stride;               // elements: page to page, row to row
    uint32_t requests, width, n_pages, log_page, rows, hq, hkv, group;
    uint32_t group_magic;                              // ceil(2^32 / group)
    uint32_t row_lo, row_hi;                           // requests with row_lo < q_len * group <= row_hi are taken
    uint32_t second;                                   // behind the form for few rows, in one call
    float scale;
    __device__ __forceinline__ uint32_t by_group(uint32_t m) const { return group == 1u ? m : __umulhi(m, group_magic); }      // m / group, m * group < 2^32
};

// what a request has: the row of its first new token, new tokens, its positions in the pages, the position of the first new token
struct PagedReq {
    uint32_t row0, n, len;
    int32_t pos0;
};
// L2: from there, for k_attn_chunk, which may begin without a wait of its own
template <bool L2 = false>
__device__ __forceinline__ PagedReq paged_req(const PagedAttn &a, uint32_t r)
{
    auto at = [](const int32_t *p) { return L2 ? __ldcg(p) : *p; };
    const int32_t c0 = min(max(at(a.cu_rows + r), 0), (int32_t)a.rows), c1 = min(max(at(a.cu_rows + r + 1), 0), (int32_t)a.rows), l = at(a.length + r);
    PagedReq q;
    q.row0 = (uint32_t)c0;
    q.n = (uint32_t)max(c1 - c0, 0);
    q.len = (uint32_t)min((unsigned long long)max(l, 0), (unsigned long long)a.width << a.log_page);
    q.pos0 = l - (int32_t)q.n;
    return q;
}

__device__ __forceinline__ void pa_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void pa_ldm(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void pa_ldmt(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// an 8 x 8 matrix of bf16 numbers transposed
__device__ __forceinline__ uint32_t pa_turn(uint32_t x)
{
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t pa_pack(float lo, float hi)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *(const uint32_t *)&h;
}
// the larger magnitudes of two pairs of bf16 numbers, as bits: 0x7f80 and above is not finite
__device__ __forceinline__ uint32_t pa_larger(uint32_t m, uint32_t x) { return __vmaxu2(m, x & 0x7fff7fffu); }
__device__ __forceinline__ bool pa_wild(uint32_t m) { return (m & 0xffffu) >= 0x7f80u || m >= 0x7f800000u; }

constexpr uint32_t kPaMaxRequests = 4096;
constexpr uint32_t kPaMaxCtas = 160;                   // one per SM

template <int D>
struct PaCfg {
    static constexpr int kWarps = 8;                   // that compute; one of four more asks for the blocks
    static constexpr int kThreads = 384, kCompute = kWarps * 32;
    static constexpr int kSub = D == 64 ? 2 : 1;       // times 16 keys of a warp's slice
    static constexpr int kSlice = 16 * kSub;
    static constexpr int kKeys = kSlice * kWarps;      // of a block
    static constexpr uint32_t kPanel = 128 * 128;      // 64 dimensions of 128 keys: rows of 128 bytes
    static constexpr uint32_t kStage = D / 64 * kSub * kPanel;     // K or V of a block: [128 keys][64 dimensions]
    static constexpr int kStages = 196608 / kStage;
    static constexpr uint32_t kRing = kStages * kStage;
    // Blocks of a pair that is not cut: 256 KB of keys and values.  A join is a CTA's 3 us and a CTA takes 64 KB in 0.45 us: 32 single
    // tokens behind 300 keys 17.2 us cut, 11.4 whole; one behind 700 (six blocks) 7.3 cut, 8.6 whole.  A limit that grows with
    // the call's size: 36.5 instead of 39 us for 64 tokens behind 700 keys, 65.4 instead of 64 for requests of unequal lengths.
    static constexpr uint32_t kWhole = 4 * 65536 / (2 * kStage);
    static constexpr int kSumD = D < 128 ? D : 128;    // dimensions that the warps' sums are joined at a time
    static constexpr int kPitch = kSumD + 4;           // floats of a row there, (maximum, denominator) at kSumD: stores without conflicts
    static constexpr uint32_t kSum = kWarps * 8 * kPitch * 4;
    static constexpr uint32_t kSmem = kRing + kSum + 2 * kStages * 8 + 64;     // (no static arrays: the ring starts on 1024 bytes)
    static constexpr uint32_t kSlot = 16 * D + 32;     // floats of a part: sums [16][D], (maximum, denominator) [16]
    static_assert(kSmem <= 227 * 1024 && kSum >= 4 * kPaMaxRequests, "fits");
};

constexpr uint32_t kPaWaitLimit = 1u << 20;            // polls
__device__ __forceinline__ bool pa_wait(uint32_t mbar, uint32_t parity)
{
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done) : "r"(mbar), "r"(parity) : "memory");
    if (done) return true;
    for (uint32_t it = 0; it < kPaWaitLimit; ++it) {
        uint32_t done;
        asm volatile("{\n\t.reg .pred p;\n\t"
                     "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                     "selp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(done) : "r"(mbar), "r"(parity) : "memory");
        if (done) return true;
    }
    return false;
}
__device__ __forceinline__ float pa_exp2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// one box of a pool's page: `keys` positions (the map's) from `row` on, 64 dimensions from d0 on, of KV head h
__device__ __forceinline__ void pa_box(uint32_t dst, const CUtensorMap *map, uint32_t d0, uint32_t h, uint32_t row, int32_t page, uint32_t mbar)
{
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 :: "r"(dst), "l"(map), "r"(d0), "r"(h), "r"(row), "r"(page), "r"(mbar) : "memory");
}

// the CTA's way through its pairs: blocks b0 .. b1 - 1 of row group rg of request r's rows of KV head h
template <int D, int NT>
struct PaWalk {
    static constexpr uint32_t kRows = 8u * NT;         // of a group
    PagedReq rq;
    uint32_t r, h, rg, kb, b0, b1;                     // kb: blocks of the pair
    unsigned long long x, x_end;                       // blocks of all pairs before block b0, and where the CTA's range ends
    __device__ __forceinline__ static bool mine(const PagedAttn &a, const PagedReq &q) { return q.n * a.group > a.row_lo && q.n * a.group <= a.row_hi; }
    __device__ __forceinline__ static uint32_t key_blocks(const PagedReq &q) { return max(1u, (q.len + PaCfg<D>::kKeys - 1) / PaCfg<D>::kKeys); }
    __device__ __forceinline__ bool whole() const { return kb <= PaCfg<D>::kWhole; }
    __device__ __forceinline__ void cut() { b1 = whole() ? kb : (uint32_t)min((unsigned long long)kb, b0 + (x_end - x)); }
    __device__ __forceinline__ uint32_t after(const PagedAttn &a) const { return r + 1u == a.requests ? 0u : r + 1u; }
    // the next pair; ahead: what the next request has (requested earlier); false: there is none
    __device__ __forceinline__ bool next(const PagedAttn &a, const PagedReq &ahead)
    {
        x += b1 - b0;
        if (x >= x_end) return false;
        if (++rg * kRows >= rq.n * a.group) {
            rg = 0;
            rq = ahead;
            if (++r == a.requests) {
                r = 0;
                ++h;
            }
            while (!mine(a, rq) && h < a.hkv) {        // (there is one, unless the lengths change under the kernel)
                if (++r == a.requests) {
                    r = 0;
                    ++h;
                }
                rq = paged_req(a, r);
            }
            if (h >= a.hkv) return false;
            kb = key_blocks(rq);
        }
        b0 = 0;
        cut();
        return true;
    }
};

// NT: times eight rows of a group
template <int D, int NT>
__global__ void __launch_bounds__(PaCfg<D>::kThreads, 1)
k_attn_paged(PagedAttn a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap)
{
    using CF = PaCfg<D>;
    constexpr int NW = CF::kWarps, ST = CF::kStages, SUB = CF::kSub;
    extern __shared__ __align__(1024) unsigned char pa_smem[];
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(pa_smem), full0 = ring + CF::kRing + CF::kSum, empty0 = full0 + 8u * ST;
    uint32_t *sm_warp = (uint32_t *)(pa_smem + CF::kRing + CF::kSum + 16 * ST), &sm_last = sm_warp[CF::kThreads / 32];
    volatile uint32_t *sm_again = sm_warp + CF::kThreads / 32 + 1;     // slices that were gone through again
    const uint32_t tid = threadIdx.x, lane = tid & 31u, wid = __shfl_sync(0xffffffffu, tid >> 5, 0), g = lane >> 2, t = lane & 3u;
    float *sum = (float *)(pa_smem + CF::kRing);       // [NW][8][kPitch]; before that the blocks before every request
    uint32_t *first = (uint32_t *)sum;
    const uint32_t R = a.requests, G = a.group, page = 1u << a.log_page;
    if (tid == 0) {
        *sm_again = 0u;
        for (int i = 0; i < ST; ++i) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(full0 + 8u * i) : "memory");
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(empty0 + 8u * i), "r"(NW) : "memory");
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&kmap) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&vmap) : "memory");
    }
    // (in this order: what starts behind this launch may rely on what came before it, see k_attn_chunk)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // ---- the blocks before every request, of one KV head
    uint32_t total = 0;
    using Walk = PaWalk<D, NT>;
    Walk s;
    auto blocks = [&](const PagedReq &q) { return Walk::mine(a, q) ? (q.n * G + Walk::kRows - 1u) / Walk::kRows * Walk::key_blocks(q) : 0u; };
    if (R == 1u) {
        s.rq = paged_req(a, 0u);
        total = blocks(s.rq);
        __syncthreads();
    } else {
        const uint32_t per = (R + CF::kThreads - 1) / CF::kThreads, ra = min(R, tid * per), rb = min(R, ra + per);
        uint32_t before = 0, own = 0;
        for (uint32_t r = ra; r < rb; ++r) {
            first[r] = own;
            own += blocks(paged_req(a, r));
        }
        uint32_t v = own;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t u = __shfl_up_sync(0xffffffffu, v, d);
            if (lane >= (uint32_t)d) v += u;
        }
        if (lane == 31u) sm_warp[wid] = v;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < CF::kThreads / 32; ++w) {
            if ((uint32_t)w < wid) before += sm_warp[w];
            total += sm_warp[w];
        }
        before += v - own;
        for (uint32_t r = ra; r < rb; ++r) first[r] += before;
        __syncthreads();
    }
    const unsigned long long W = (unsigned long long)total * a.hkv;
    const uint32_t N = (uint32_t)min((unsigned long long)gridDim.x, W), me = blockIdx.x;
    if (me >= N) return;
    auto part_of = [&](uint32_t c) { return W < 1u << 24 ? (unsigned long long)((uint32_t)W * c / N) : W * c / N; };     // (N at most 256)
    auto cta_of = [&](unsigned long long y) {          // the last c with part_of(c) <= y
        return W < 1u << 24 ? (((uint32_t)y + 1u) * N - 1u) / (uint32_t)W : (uint32_t)(((y + 1ull) * N - 1ull) / W);
    };
    s.x = part_of(me);
    s.x_end = part_of(me + 1u);
    const unsigned long long x_begin = s.x;
    {
        s.h = W < 1u << 24 ? (uint32_t)s.x / total : (uint32_t)(s.x / total);
        uint32_t off = (uint32_t)(s.x - (unsigned long long)s.h * total), lo = 0;
        if (R > 1u) {                                  // the request of the first block: the last one with first[r] <= off
            uint32_t hi = R;
            while (hi - lo > 1u) {
                const uint32_t mid = (lo + hi) / 2u;
                if (first[mid] <= off) lo = mid;
                else hi = mid;
            }
            off -= first[lo];
            s.rq = paged_req(a, lo);
        }
        s.r = lo;
        s.kb = Walk::key_blocks(s.rq);
        s.rg = off / s.kb;
        s.b0 = off - s.rg * s.kb;
        if (s.b0 && s.whole()) {                       // the CTA before has all of it
            s.b1 = s.kb;
            if (!s.next(a, paged_req(a, s.after(a)))) return;
        } else {
            s.cut();
        }
    }
    bool ok = true;
    if (wid >= (uint32_t)NW) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (wid > (uint32_t)NW) return;
        // ---- the warp that asks for K and V of every block: boxes of (at most 128) positions of a page
        const uint32_t bp = min(page, 128u), boxes = CF::kKeys / bp * (D / 64), bk = lane / (D / 64), panel = lane % (D / 64);
        // (of lane < boxes, at most 32: positions bk * bp .. of a block and 64 dimensions; with D = 256 and pages of 16 a lane has just one)
        static_assert(CF::kKeys / 16 * (D / 64) <= 32, "a box per lane");
        const uint32_t dst = (bk * bp / 128u * (D / 64) + panel) * CF::kPanel + bk * bp % 128u * 128u;
        uint32_t seen = 0;                             // of *sm_again, when a wait last ran out
        auto room = [&](uint32_t bar, uint32_t parity) {
            while (!pa_wait(bar, parity)) {
                const uint32_t now = *sm_again;
                if (now == seen) return false;
                seen = now;
            }
            return true;
        };
        uint32_t n = 0;
        bool more = true;
        while (more && ok) {
            const int32_t *pages = a.table + (size_t)s.r * a.width;
            const PagedReq ahead = paged_req(a, s.after(a));
            auto page_of = [&](uint32_t b) {
                const uint32_t key = b * CF::kKeys + bk * bp;
                return lane < boxes && b < s.b1 && key < s.rq.len ? pages[key >> a.log_page] : 0;
            };
            int32_t p = page_of(s.b0);
            for (uint32_t b = s.b0; b < s.b1 && ok; ++b) {
                const uint32_t key = b * CF::kKeys + bk * bp;
                const bool on = lane < boxes && key < s.rq.len;
                const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, on)) * bp * 128u;
                const int32_t p_next = page_of(b + 1u);
#pragma unroll
                for (int i = 0; i < 2; ++i, ++n) {
                    const uint32_t st = n % ST, bar = full0 + 8u * st;
                    ok = ok && room(empty0 + 8u * st, (n / ST & 1u) ^ 1u);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    if (lane == 0) asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1;\n\t}" ::"r"(bar), "r"(bytes) : "memory");
                    __syncwarp();
                    if (on) pa_box(ring + st * CF::kStage + dst, i ? &vmap : &kmap, panel * 64u, s.h, key & (page - 1u), p, bar);
                    __syncwarp();
                }
                p = p_next;
            }
            more = s.next(a, ahead);
        }
        for (uint32_t i = n > (uint32_t)ST ? n - ST : 0u; i < n; ++i) pa_wait(full0 + 8u * (i % ST), i / ST & 1u);        // nothing is in flight behind the end
        return;
    }
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    const float sl2 = a.scale * 1.4426950408889634f;   // scores in units of log2
    uint32_t take = 0;                                 // stages taken so far
    auto landed = [&]() {                              // the next stage's slice, as an address
        const uint32_t st = take % ST;
        ok = ok && pa_wait(full0 + 8u * st, take / ST & 1u);
        ok = __all_sync(0xffffffffu, ok);
        return ring + st * CF::kStage + wid * CF::kSlice / 128u * (D / 64) * CF::kPanel + wid * CF::kSlice % 128u * 128u;
    };
    auto taken = [&]() {
        __syncwarp();
        if (lane == 0) asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.shared::cta.b64 st, [%0];\n\t}" ::"r"(empty0 + 8u * (take % ST)) : "memory");
        ++take;
    };
    uint32_t qf[NT][D / 16][2];                        // the rows as B operands: row rg * kRows + m is token (..) / G, head (..) % G
    int32_t limit[NT][2];                              // the last position that the lane's rows 8 nt + 2 t, + 1 see
    auto rows_in = [&]() {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const uint32_t m = s.rg * Walk::kRows + nt * 8u + g, tok = a.by_group(m), gi = m - tok * G;
            const bool on = m < s.rq.n * G;
            const uint32_t *src = (const uint32_t *)(a.q + (size_t)(s.rq.row0 + (on ? tok : 0u)) * a.q_stride + ((size_t)s.h * G + (on ? gi : 0u)) * D) + t;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
                qf[nt][kk][0] = on ? src[kk * 8] : 0u;
                qf[nt][kk][1] = on ? src[kk * 8 + 4] : 0u;
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t q = s.rg * Walk::kRows + nt * 8u + 2u * t + i;
                limit[nt][i] = q < s.rq.n * G ? min(s.rq.pos0 + (int32_t)a.by_group(q), (int32_t)s.rq.len - 1) : -1;
            }
        }
    };
    rows_in();
    bool more = true;
    while (more) {
        const uint32_t rows = min(Walk::kRows, s.rq.n * G - s.rg * Walk::kRows);
        const int32_t len1 = (int32_t)s.rq.len - 1, all_see = min(s.rq.pos0 + (int32_t)a.by_group(s.rg * Walk::kRows), len1);
        const PagedReq ahead = paged_req(a, s.after(a));               // (requested here, needed where the pair ends)
        // sums: dimensions 16 d + g (+ 8 for elements 2 and 3) of rows 8 nt + 2 t (+ 1 for odd elements); maxima of the raw scores
        float o[NT][D / 16][4], m_[NT][2], l_[NT][2];
        auto zero = [&]() {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                m_[nt][0] = m_[nt][1] = -INFINITY;
                l_[nt][0] = l_[nt][1] = 0.f;
#pragma unroll
                for (int d = 0; d < D / 16; ++d) o[nt][d][0] = o[nt][d][1] = o[nt][d][2] = o[nt][d][3] = 0.f;
            }
        };
        zero();
        // scores of a slice (keys 16 u + g, + 8) into probabilities, as B operands of leading and trailing bits; corr: what the sums
        // so far shrink by
        auto softmax = [&](float (&sc)[NT][SUB][4], int32_t key0, uint32_t (&ph)[NT][SUB][2], uint32_t (&pl)[NT][SUB][2], float (&corr)[NT][2]) {
            const bool mask = key0 + CF::kSlice - 1 > all_see;         // uniform: not every row sees every key
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                if (mask) {
#pragma unroll
                    for (int u = 0; u < SUB; ++u)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (key0 + u * 16 + (int32_t)g + 8 * (i >> 1) > limit[nt][i & 1]) sc[nt][u][i] = -INFINITY;
                }
                float base[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float mx = fmaxf(sc[nt][0][i], sc[nt][0][i + 2]);
                    if (SUB == 2) mx = fmaxf(mx, fmaxf(sc[nt][SUB - 1][i], sc[nt][SUB - 1][i + 2]));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                    const float mn = fmaxf(m_[nt][i], mx);
                    base[i] = mn == -INFINITY ? 0.f : mn * sl2;        // nothing so far: sums stay zero
                    corr[nt][i] = pa_exp2(fmaf(m_[nt][i], sl2, -base[i]));
                    m_[nt][i] = mn;
                    l_[nt][i] *= corr[nt][i];
                }
#pragma unroll
                for (int u = 0; u < SUB; ++u)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {      // keys g, g + 8
                        const float p0 = pa_exp2(fmaf(sc[nt][u][2 * h], sl2, -base[0])), p1 = pa_exp2(fmaf(sc[nt][u][2 * h + 1], sl2, -base[1]));
                        l_[nt][0] += p0;
                        l_[nt][1] += p1;
                        const uint32_t hi = pa_pack(p0, p1);
                        ph[nt][u][h] = pa_turn(hi);
                        pl[nt][u][h] = pa_turn(pa_pack(p0 - __uint_as_float(hi << 16), p1 - __uint_as_float(hi & 0xffff0000u)));
                    }
            }
        };
        for (uint32_t b = s.b0; b < s.b1; ++b) {
            const int32_t key0 = (int32_t)(b * CF::kKeys + wid * CF::kSlice);
            const uint32_t sk = landed();
            if (key0 > len1) {                         // uniform: nothing for this warp
                taken();
                landed();
                taken();
                continue;
            }
            float sc[NT][SUB][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int u = 0; u < SUB; ++u) sc[nt][u][0] = sc[nt][u][1] = sc[nt][u][2] = sc[nt][u][3] = 0.f;
            const uint32_t krow = (lane & 7u) + ((lane >> 3) & 1u) * 8u, kaddr = sk + krow * 128u;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
#pragma unroll
                for (int u = 0; u < SUB; ++u) {
                    uint32_t ak[4];                    // keys 16 u .. + 15, dimensions 16 kk .. + 15
                    const uint32_t cc = 2u * kk + (lane >> 4);
                    pa_ldm(ak, kaddr + (cc >> 3) * CF::kPanel + u * 2048u + ((cc ^ krow) & 7u) * 16u);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) pa_mma(sc[nt][u], ak, qf[nt][kk][0], qf[nt][kk][1]);
                }
            }
            taken();
            uint32_t ph[NT][SUB][2], pl[NT][SUB][2];
            float corr[NT][2];
            softmax(sc, key0, ph, pl, corr);
            const uint32_t vrow = (lane & 7u) + (lane >> 4) * 8u, vaddr = landed() + vrow * 128u;
            const bool tail = key0 + CF::kSlice - 1 > len1;            // uniform: without the values behind the last key
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
                float w[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) w[nt][0] = w[nt][1] = w[nt][2] = w[nt][3] = 0.f;
#pragma unroll
                for (int u = 0; u < SUB; ++u) {
                    uint32_t av[4];                    // dimensions 16 d + g (+ 8 for odd registers), keys 16 u + 2 t, + 1 (+ 8 for the second two)
                    const uint32_t cc = 2u * d + ((lane >> 3) & 1u);
                    pa_ldmt(av, vaddr + (cc >> 3) * CF::kPanel + u * 2048u + ((cc ^ vrow) & 7u) * 16u);
                    if (tail) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int32_t key = key0 + u * 16 + 2 * (int32_t)t + 8 * (i >> 1);
                            av[i] &= key > len1 ? 0u : key == len1 ? 0xffffu : 0xffffffffu;
                        }
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        pa_mma(w[nt], av, pl[nt][u][0], pl[nt][u][1]);
                        pa_mma(w[nt], av, ph[nt][u][0], ph[nt][u][1]);
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[nt][d][i] = fmaf(o[nt][d][i], corr[nt][i & 1], w[nt][i]);
            }
            taken();
        }
        float z = 0.f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int d = 0; d < D / 16; ++d) z = fmaf(o[nt][d][0], 0.f, fmaf(o[nt][d][1], 0.f, fmaf(o[nt][d][2], 0.f, fmaf(o[nt][d][3], 0.f, z))));
        uint32_t again;
        asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                     : "=r"(again) : "r"((uint32_t)(z != 0.f)), "n"(CF::kCompute) : "memory");
        if (again) {
            // something is not finite: the same slices again, from memory, and P V for one token after the other with the values
            // that it does not see taken out
            const uint32_t tok0 = a.by_group(s.rg * Walk::kRows), tok1 = a.by_group(s.rg * Walk::kRows + rows - 1u);
            zero();
#pragma unroll 1
            for (uint32_t b = s.b0; b < s.b1; ++b) {
                const int32_t key0 = (int32_t)(b * CF::kKeys + wid * CF::kSlice);
                if (key0 > len1) break;                // uniform
                if (lane == 0) atomicAdd((uint32_t *)sm_again, 1u);
                auto at = [&](const __nv_bfloat16 *pool, size_t stride, int32_t key) -> const __nv_bfloat16 * {        // null: zeros
                    if (key > len1) return nullptr;
                    const int32_t p = a.table[(size_t)s.r * a.width + ((uint32_t)key >> a.log_page)];
                    return (uint32_t)p < a.n_pages ? pool + (size_t)p * stride + ((size_t)((uint32_t)key & (page - 1u)) * a.hkv + s.h) * D : nullptr;
                };
                float sc[NT][SUB][4];
#pragma unroll
                for (int u = 0; u < SUB; ++u) {
                    const uint32_t *k0 = (const uint32_t *)at(a.k, a.k_stride, key0 + u * 16 + (int32_t)g), *k1 = (const uint32_t *)at(a.k, a.k_stride, key0 + u * 16 + 8 + (int32_t)g);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) sc[nt][u][0] = sc[nt][u][1] = sc[nt][u][2] = sc[nt][u][3] = 0.f;
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk) {
                        const uint32_t ak[4] = {k0 ? k0[kk * 8 + t] : 0u, k1 ? k1[kk * 8 + t] : 0u, k0 ? k0[kk * 8 + 4 + t] : 0u, k1 ? k1[kk * 8 + 4 + t] : 0u};
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) pa_mma(sc[nt][u], ak, qf[nt][kk][0], qf[nt][kk][1]);
                    }
                }
                uint32_t ph[NT][SUB][2], pl[NT][SUB][2];
                float corr[NT][2];
                softmax(sc, key0, ph, pl, corr);
#pragma unroll 1
                for (uint32_t tok = tok0; tok <= tok1; ++tok) {
                    const int32_t last = min(s.rq.pos0 + (int32_t)tok, len1);
#pragma unroll
                    for (int d = 0; d < D / 16; ++d) {
                        float w[NT][4], v[NT][4];
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int i = 0; i < 4; ++i) w[nt][i] = v[nt][i] = 0.f;
#pragma unroll
                        for (int u = 0; u < SUB; ++u) {
                            uint32_t av[4];
#pragma unroll
                            for (int h = 0; h < 2; ++h) {              // keys 2 t, 2 t + 1 (+ 8)
                                const int32_t key = key0 + u * 16 + 2 * (int32_t)t + 8 * h;
                                const __nv_bfloat16 *v0 = key <= last ? at(a.v, a.v_stride, key) : nullptr, *v1 = key < last ? at(a.v, a.v_stride, key + 1) : nullptr;
#pragma unroll
                                for (int i = 0; i < 2; ++i) {          // dimension 16 d + g (+ 8)
                                    const uint32_t dim = d * 16 + i * 8 + g;
                                    av[2 * h + i] = (v0 ? (uint32_t)__bfloat16_as_ushort(v0[dim]) : 0u) | (v1 ? (uint32_t)__bfloat16_as_ushort(v1[dim]) << 16 : 0u);
                                }
                            }
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                pa_mma(w[nt], av, pl[nt][u][0], pl[nt][u][1]);
                                pa_mma(v[nt], av, ph[nt][u][0], ph[nt][u][1]);
                            }
                        }
                        // (zero times infinity in the trailing bits is no reason for a NaN)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const uint32_t m = s.rg * Walk::kRows + nt * 8u + 2u * t + (i & 1);
                                const float add = fabsf(w[nt][i]) < INFINITY ? v[nt][i] + w[nt][i] : v[nt][i];
                                if (a.by_group(m) == tok) o[nt][d][i] = fmaf(o[nt][d][i], corr[nt][i & 1], add);
                            }
                    }
                }
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                l_[nt][i] += __shfl_xor_sync(0xffffffffu, l_[nt][i], 4);
                l_[nt][i] += __shfl_xor_sync(0xffffffffu, l_[nt][i], 8);
                l_[nt][i] += __shfl_xor_sync(0xffffffffu, l_[nt][i], 16);
                if (!ok) l_[nt][i] = __int_as_float(0x7fc00000);
            }
        // ---- the next pair, whose rows come while this one's sums are joined
        const PagedReq rq = s.rq;
        const uint32_t r_h = s.h, r_rg = s.rg, r_kb = s.kb;
        const unsigned long long x0 = s.x - s.b0;      // the pair's first block
        const bool whole = s.b0 == 0u && s.b1 == s.kb; // this is all of the pair
        float *dst = a.part + (size_t)(2u * me + (s.x == x_begin ? 0u : 1u)) * CF::kSlot;
        more = s.next(a, ahead);
        if (more) rows_in();
        // ---- the warps' sums
        auto sync = [&]() { asm volatile("barrier.cta.sync 1, %0;" ::"n"(CF::kCompute) : "memory"); };
        auto write_out = [&](uint32_t m, uint32_t d4, const float4 &v, float l) {      // row m of the group
            const uint32_t q = r_rg * Walk::kRows + m, tok = a.by_group(q);
            const bool sees = rq.pos0 + (int32_t)tok >= 0 && rq.len > 0u;              // a row that sees nothing is zero
            const float inv = 1.f / l;
            *(uint2 *)(a.out + ((size_t)(rq.row0 + tok) * a.hq + r_h * G + (q - tok * G)) * D + d4 * 4) =
                sees ? make_uint2(pa_pack(v.x * inv, v.y * inv), pa_pack(v.z * inv, v.w * inv)) : make_uint2(0u, 0u);
        };
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            if (rows <= 8u * nt) break;                // uniform
#pragma unroll
            for (int d0 = 0; d0 < D; d0 += CF::kSumD) {
                if (nt || d0) sync();                  // (the first time the barrier above has been passed since the sums were read)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float *to = sum + (wid * 8u + 2u * t + i) * CF::kPitch;
                    if (8u * nt + 2u * t + i >= rows) continue;
#pragma unroll
                    for (int d = 0; d < CF::kSumD / 16; ++d) {
                        to[d * 16 + g] = o[nt][d0 / 16 + d][i];
                        to[d * 16 + 8 + g] = o[nt][d0 / 16 + d][2 + i];
                    }
                    if (g == 0) *(float2 *)(to + CF::kSumD) = make_float2(m_[nt][i], l_[nt][i]);
                }
                sync();
                for (uint32_t it = tid; it < min(8u, rows - 8u * nt) * (CF::kSumD / 4); it += CF::kCompute) {
                    const uint32_t row = it / (CF::kSumD / 4), d4 = it % (CF::kSumD / 4);
                    const float *from = sum + row * CF::kPitch;
                    float M = -INFINITY, L = 0.f;
#pragma unroll
                    for (int w = 0; w < NW; ++w) M = fmaxf(M, from[w * 8 * CF::kPitch + CF::kSumD]);
                    const float mb = M == -INFINITY ? 0.f : M * sl2;
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int w = 0; w < NW; ++w) {
                        const float2 ml = *(const float2 *)(from + w * 8 * CF::kPitch + CF::kSumD);
                        const float f = pa_exp2(fmaf(ml.x, sl2, -mb));
                        const float4 u = *(const float4 *)(from + w * 8 * CF::kPitch + d4 * 4);
                        L = fmaf(ml.y, f, L);
                        v.x = fmaf(u.x, f, v.x); v.y = fmaf(u.y, f, v.y); v.z = fmaf(u.z, f, v.z); v.w = fmaf(u.w, f, v.w);
                    }
                    const uint32_t m = row + 8u * nt;
                    if (whole) {
                        write_out(m, d0 / 4 + d4, v, L);
                    } else {
                        *(float4 *)(dst + m * D + d0 + d4 * 4) = v;
                        if (d0 == 0 && d4 == 0u) *(float2 *)(dst + 16 * D + 2 * m) = make_float2(M, L);
                    }
                }
            }
        }
        if (!whole) {
            const uint32_t c0 = cta_of(x0), parts = cta_of(x0 + r_kb - 1u) - c0 + 1u;
            sync();
            // numbers whose sum is zero, so the ticket is zero again when all have come
            if (tid == 0) {
                const uint32_t add = me == c0 ? 1u - parts : 1u;
                __threadfence();                       // the CTA's parts (behind the barrier) before the ticket
                sm_last = atomicAdd(a.tickets + c0, add) + add == 0u;
                __threadfence();
            }
            sync();
            if (sm_last) {
                const uint32_t behind = part_of(c0) != x0 ? 1u : 0u;
                auto slot_of = [&](uint32_t q) { return a.part + (size_t)(2u * q + (q == c0 ? behind : 0u)) * CF::kSlot; };
                // Few rows: up to four threads share four dimensions' parts, four of which a thread requests at once.  (Short
                // code: this is its first run in the launch, and it comes from memory.)
                const uint32_t items = rows * (D / 4), split = 4u * items <= CF::kCompute ? 2u : 2u * items <= CF::kCompute ? 1u : 0u;
#pragma unroll 1
                for (uint32_t at = tid; at >> split < items; at += CF::kCompute) {     // (a warp's threads are in or out together)
                    const uint32_t it = at >> split, m = it / (D / 4), d4 = it % (D / 4);
                    float M = -INFINITY, L = 0.f;
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
                    for (uint32_t p0 = at & ((1u << split) - 1u); p0 < parts; p0 += 4u << split) {
                        float2 e[4];
                        float4 u[4];
#pragma unroll
                        for (uint32_t i = 0; i < 4u; ++i) {
                            const uint32_t p = p0 + (i << split);
                            const float *from = slot_of(c0 + min(p, parts - 1u));
                            e[i] = __ldcg((const float2 *)(from + 16 * D) + m);
                            u[i] = __ldcg((const float4 *)(from + m * D) + d4);
                            if (p >= parts) {
                                e[i] = make_float2(-INFINITY, 0.f);
                                u[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                            }
                        }
                        const float mx = fmaxf(fmaxf(fmaxf(e[0].x, e[1].x), fmaxf(e[2].x, e[3].x)), M), mb = mx == -INFINITY ? 0.f : mx * sl2;
                        const float f0 = pa_exp2(fmaf(M, sl2, -mb));
                        M = mx;
                        L *= f0;
                        v.x *= f0; v.y *= f0; v.z *= f0; v.w *= f0;
#pragma unroll
                        for (uint32_t i = 0; i < 4u; ++i) {
                            const float f = pa_exp2(fmaf(e[i].x, sl2, -mb));
                            L = fmaf(e[i].y, f, L);
                            v.x = fmaf(u[i].x, f, v.x); v.y = fmaf(u[i].y, f, v.y); v.z = fmaf(u[i].z, f, v.z); v.w = fmaf(u[i].w, f, v.w);
                        }
                    }
#pragma unroll 1
                    for (uint32_t d = 1u; d < 1u << split; d <<= 1) {
                        const float mo = __shfl_xor_sync(0xffffffffu, M, d), mx = fmaxf(M, mo), mb = mx == -INFINITY ? 0.f : mx * sl2;
                        const float f = pa_exp2(fmaf(M, sl2, -mb));
                        M = mx;
                        auto both = [&](float x) { x *= f; return x + __shfl_xor_sync(0xffffffffu, x, d); };
                        L = both(L);
                        v.x = both(v.x); v.y = both(v.y); v.z = both(v.z); v.w = both(v.w);
                    }
                    if ((at & ((1u << split) - 1u)) == 0u) write_out(m, d4, v, L);
                }
            }
        }
    }
}

}  // namespace ixb
