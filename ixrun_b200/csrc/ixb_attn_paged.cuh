// Causal attention of every request's new tokens over its pages: the form for few rows (single tokens, short drafts).
//
//   row (t, g) of request r and KV head h: new token t < q_len[r], query head h * G + g, position length[r] - q_len[r] + t
//   out = softmax(scale * q . K[0 .. position]) V[0 .. position]
//
// A request's rows of one KV head are packed, row t * G + g, sixteen to a group (the M of mma.sync), so a key is read once for all
// of them.  Bound: HBM, every key and value once; mma.sync is used as an instruction that multiplies sixteen rows at a time, at a
// fifth of its rate.
//
// Work: all (KV head, request, row group) pairs' blocks of keys (16 per warp of a CTA) in one line, cut into equal ranges, one per
// CTA, so lengths that differ cost nothing.  A warp takes its 16 keys of every block through its own ring of TMA stages (a box is 16
// positions of a page and 64 dimensions, 128-byte swizzle) and keeps a running softmax of its own, so no barrier lies in the loop;
// the warps' sums meet in shared memory where a pair ends.  A pair that is cut leaves its parts in the scratch, and the CTA that comes
// last (a ticket) joins them in the order of the keys: the same bits every time.
//
// Precision: q K^T bf16 x bf16 in fp32; probabilities as two bf16 numbers whose sum they are to 17 bits; a slice's P V starts from
// zero and joins the running sums by fp32 fused multiply-adds (the tensor core cuts low bits of what it adds to a large sum).
//
// Keys at and behind length are masked and their values taken as zeros, whatever lies there; a page number outside the pool is a
// page of zeros (the copy's fill).  A value that is not finite counts for the rows that see it and for no other: it shows in the
// sums of every row (zero times infinity is NaN), and the pair's blocks are then gone through again, slices that hold one token by
// token.
//
// Every wait on an mbarrier is bounded and counts the warp's own copies; where one runs out the CTA's outputs become NaN.
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
    uint32_t group_magic;                              // ceil(2^32 / group): x / group = umulhi(x, magic) for x * group < 2^32, group > 1
    uint32_t row_lo, row_hi;                           // requests with row_lo < q_len * group <= row_hi are taken
    float scale;
};

// what a request has: the row of its first new token, new tokens, its positions in the pages, the position of the first new token
struct PagedReq {
    uint32_t row0, n, len;
    int32_t pos0;
};
__device__ __forceinline__ PagedReq paged_req(const PagedAttn &a, uint32_t r)
{
    const int32_t c0 = min(max(a.cu_rows[r], 0), (int32_t)a.rows), c1 = min(max(a.cu_rows[r + 1], 0), (int32_t)a.rows), l = a.length[r];
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
__device__ __forceinline__ uint32_t pa_pack(float lo, float hi)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *(const uint32_t *)&h;
}
// the larger magnitudes of two pairs of bf16 numbers, as bits: 0x7f80 and above is not finite
__device__ __forceinline__ uint32_t pa_larger(uint32_t m, uint32_t x) { return __vmaxu2(m, x & 0x7fff7fffu); }
__device__ __forceinline__ bool pa_wild(uint32_t m) { return (m & 0xffffu) >= 0x7f80u || m >= 0x7f800000u; }

template <int D>
struct PaCfg {
    static constexpr int kWarps = D == 256 ? 4 : 8, kThreads = kWarps * 32;
    static constexpr int kKeys = 16 * kWarps;          // of a block
    static constexpr uint32_t kHalf = 16 * D * 2;      // K or V of a warp's slice: [64 dimensions][16 keys] of 128 bytes
    static constexpr uint32_t kStage = 2 * kHalf;
    static constexpr int kStages = D == 64 ? 6 : 3;
    static constexpr uint32_t kRing = kWarps * kStages * kStage;
    static constexpr int kPitch = D + 8;               // floats of a row in the warps' sums, (maximum, denominator) at D: 8-byte stores without conflicts
    static constexpr uint32_t kSum = kWarps * 8 * kPitch * 4;
    static constexpr uint32_t kSmem = kRing + kSum + kWarps * kStages * 8 + kWarps * 4 + 16;       // (no static arrays: the ring starts on 1024 bytes)
    static constexpr uint32_t kSlot = 16 * D + 32;     // floats of a part: sums [16][D], (maximum, denominator) [16]
    static_assert(kSmem <= 227 * 1024 && kHalf % 1024 == 0, "fits");
};
constexpr uint32_t kPaMaxRequests = 4096;

constexpr uint32_t kPaWaitLimit = 1u << 20;            // polls
__device__ __forceinline__ bool pa_wait(uint32_t mbar, uint32_t parity)
{
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

template <int D>
__global__ void __launch_bounds__(PaCfg<D>::kThreads, 1)
k_attn_paged(PagedAttn a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap)
{
    using CF = PaCfg<D>;
    constexpr int NW = CF::kWarps, ST = CF::kStages;
    extern __shared__ __align__(1024) unsigned char pa_smem[];
    uint64_t *sm_bar = (uint64_t *)(pa_smem + CF::kRing + CF::kSum);           // [NW][ST], then:
    uint32_t *sm_warp = (uint32_t *)(sm_bar + NW * ST), &sm_last = sm_warp[NW];
    const uint32_t tid = threadIdx.x, lane = tid & 31u, wid = __shfl_sync(0xffffffffu, tid >> 5, 0), g = lane >> 2, t = lane & 3u;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(pa_smem) + wid * ST * CF::kStage;
    float *sum = (float *)(pa_smem + CF::kRing);       // [NW][8][kPitch]; before that the blocks before every request
    uint32_t *first = (uint32_t *)sum;
    static_assert(CF::kSum >= 4 * kPaMaxRequests && CF::kRing >= 256 * 16 * 8, "fits");       // (parts of a pair: at most a CTA each)
    const uint32_t R = a.requests, G = a.group, page = 1u << a.log_page;
    const uint32_t bar0 = (uint32_t)__cvta_generic_to_shared(sm_bar) + wid * ST * 8u;
    asm volatile("griddepcontrol.launch_dependents;");
    if (lane == 0) {
        for (int i = 0; i < ST; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar0 + 8u * i) : "memory");
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (tid == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&kmap) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&vmap) : "memory");
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    auto key_blocks = [&](const PagedReq &q) { return max(1u, (q.len + CF::kKeys - 1) / CF::kKeys); };
    auto mine = [&](const PagedReq &q) { return q.n * G > a.row_lo && q.n * G <= a.row_hi; };
    auto blocks = [&](const PagedReq &q) { return mine(q) ? (q.n * G + 15u) / 16u * key_blocks(q) : 0u; };
    // ---- the blocks before every request, of one KV head
    const uint32_t per = (R + CF::kThreads - 1) / CF::kThreads, ra = min(R, tid * per), rb = min(R, ra + per);
    uint32_t before = 0, total = 0;
    {
        uint32_t own = 0;
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
        for (int w = 0; w < NW; ++w) {
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
    unsigned long long x = W * me / N;
    const unsigned long long x_end = W * (me + 1ull) / N, x_begin = x;
    uint32_t h = (uint32_t)(x / total), off = (uint32_t)(x - (unsigned long long)h * total), r;
    {                                                  // the request of the first block: the last one with first[r] <= off
        uint32_t lo = 0, hi = R;
        while (hi - lo > 1u) {
            const uint32_t mid = (lo + hi) / 2u;
            if (first[mid] <= off) lo = mid;
            else hi = mid;
        }
        r = lo;
        off -= first[r];
    }
    PagedReq rq = paged_req(a, r);
    uint32_t kb = key_blocks(rq), rg = off / kb, b0 = off - rg * kb;           // key blocks, row group, first block
    const float sl2 = a.scale * 1.4426950408889634f;   // scores in units of log2
    uint32_t n = 0;                                    // stages asked for so far
    bool ok = true;
    for (;;) {
        // ---- blocks b0 .. b1 - 1 of row group rg of request r, KV head h
        const uint32_t b1 = (uint32_t)min((unsigned long long)kb, b0 + (x_end - x));
        const uint32_t rows = min(16u, rq.n * G - rg * 16u);
        const int32_t *pages = a.table + (size_t)r * a.width;
        int32_t page_l = -1;                           // lane l: the page of the warp's slice of block b0 + 32 i + l
        uint32_t page_at = 0xffffffffu;
        auto fetch = [&](uint32_t b) {                 // the warp's slice of block b into the next stage
            const uint32_t key0 = (b * NW + wid) * 16u;
            if (b >= b1 || key0 >= rq.len) return;     // uniform
            const uint32_t win = (b - b0) & ~31u;
            if (win != page_at) {
                page_at = win;
                const uint32_t key_l = ((b0 + win + lane) * NW + wid) * 16u;
                page_l = key_l < rq.len ? pages[key_l >> a.log_page] : -1;
            }
            const int32_t p = __shfl_sync(0xffffffffu, page_l, (int)((b - b0) & 31u));
            const uint32_t st = n % ST, bar = bar0 + 8u * st, dst = ring + st * CF::kStage;
            ++n;
            if (lane == 0) {
                asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1;\n\t}" ::"r"(bar), "r"(CF::kStage) : "memory");
#pragma unroll
                for (uint32_t i = 0; i < 2 * D / 64; ++i)
                    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                                 :: "r"(dst + i * 2048u), "l"(i < D / 64 ? &kmap : &vmap), "r"(i % (D / 64) * 64u), "r"(h), "r"(key0 & (page - 1u)), "r"(p), "r"(bar)
                                 : "memory");
            }
            __syncwarp();
        };
        // the rows as A operands: row rg * 16 + m is token (..) / G, head (..) % G
        uint32_t qf[D / 16][4];
        int32_t limit[2];                              // the last position that the lane's rows g and g + 8 see
        const uint32_t tok0 = rg * 16u / G, tok1 = (rg * 16u + rows - 1u) / G;         // the group's tokens
        const int32_t len1 = (int32_t)rq.len - 1, all_see = min(rq.pos0 + (int32_t)tok0, len1);
        float o[D / 8][4], m_[2], l_[2];
        for (bool careful = false;; careful = true) {
        uint32_t take = n;                             // the stage that comes next
#pragma unroll
        for (int i = 0; i < ST; ++i) fetch(b0 + i);
        if (!careful) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t m = rg * 16u + g + 8u * i, tok = m / G, gi = m - tok * G;
                const bool on = g + 8u * i < rows;
                limit[i] = on ? min(rq.pos0 + (int32_t)tok, len1) : -1;
                const uint32_t *src = (const uint32_t *)(a.q + (size_t)(rq.row0 + (on ? tok : 0u)) * a.q_stride + ((size_t)h * G + (on ? gi : 0u)) * D) + t;
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    qf[kk][i] = on ? src[kk * 8] : 0u;
                    qf[kk][i + 2] = on ? src[kk * 8 + 4] : 0u;
                }
            }
        }
        m_[0] = m_[1] = -INFINITY;                     // of the raw scores
        l_[0] = l_[1] = 0.f;
#pragma unroll
        for (int d = 0; d < D / 8; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f;
        for (uint32_t b = b0; b < b1; ++b) {
            const int32_t key0 = (int32_t)((b * NW + wid) * 16u);
            if ((uint32_t)key0 >= rq.len) break;       // uniform
            const uint32_t st = take % ST, sk = ring + st * CF::kStage, sv = sk + CF::kHalf;
            ok = ok && pa_wait(bar0 + 8u * st, take / ST & 1u);
            ok = __all_sync(0xffffffffu, ok);
            ++take;
            float s[2][4];
#pragma unroll
            for (int i = 0; i < 2; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
                uint32_t bk[4];                        // keys 0 .. 15, dimensions 16 kk .. + 15
                const uint32_t rr = (lane & 7u) + (lane >> 4) * 8u, cc = 2u * kk + ((lane >> 3) & 1u);
                pa_ldm(bk, sk + (cc >> 3) * 2048u + rr * 128u + ((cc ^ rr) & 7u) * 16u);
                pa_mma(s[0], qf[kk], bk[0], bk[1]);
                pa_mma(s[1], qf[kk], bk[2], bk[3]);
            }
            if (key0 + 15 > all_see) {                 // uniform: not every row sees every key
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (key0 + c * 8 + 2 * (int32_t)t + (i & 1) > limit[i >> 1]) s[c][i] = -INFINITY;
            }
            float corr[2], base[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float mx = fmaxf(fmaxf(s[0][2 * i], s[0][2 * i + 1]), fmaxf(s[1][2 * i], s[1][2 * i + 1]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const float mn = fmaxf(m_[i], mx);
                base[i] = mn == -INFINITY ? 0.f : mn * sl2;            // nothing so far: sums stay zero
                corr[i] = pa_exp2(fmaf(m_[i], sl2, -base[i]));
                m_[i] = mn;
                l_[i] *= corr[i];
            }
            uint32_t ph[4], pl[4];                     // probabilities as A operands, leading and trailing bits
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float p0 = pa_exp2(fmaf(s[c][2 * i], sl2, -base[i])), p1 = pa_exp2(fmaf(s[c][2 * i + 1], sl2, -base[i]));
                    l_[i] += p0 + p1;
                    const uint32_t hi = pa_pack(p0, p1);
                    ph[2 * c + i] = hi;
                    pl[2 * c + i] = pa_pack(p0 - __uint_as_float(hi << 16), p1 - __uint_as_float(hi & 0xffff0000u));
                }
            const uint32_t vrow = lane & 15u, vaddr = sv + vrow * 128u;
            auto values = [&](uint32_t (&bv)[4], int d2) {             // keys 0 .. 15, dimensions 16 d2 .. + 15
                const uint32_t cc = 2u * d2 + (lane >> 4);
                pa_ldmt(bv, vaddr + (cc >> 3) * 2048u + ((cc ^ vrow) & 7u) * 16u);
            };
            auto cut = [&](uint32_t (&bv)[4], int32_t last) {          // without the values behind position `last`
#pragma unroll
                for (int i = 0; i < 4; ++i) {          // keys 2 t, 2 t + 1 (+ 8 for odd i)
                    const int32_t key = key0 + 2 * (int32_t)t + 8 * (i & 1);
                    bv[i] &= key > last ? 0u : key + 1 > last ? 0xffffu : 0xffffffffu;
                }
            };
            const bool tail = key0 + 15 > len1;        // uniform
            bool wild = false;
            if (careful) {
                uint32_t big = 0;
#pragma unroll 1
                for (int d2 = 0; d2 < D / 16; ++d2) {
                    uint32_t bv[4];
                    values(bv, d2);
                    cut(bv, len1);
#pragma unroll
                    for (int i = 0; i < 4; ++i) big = pa_larger(big, bv[i]);
                }
                wild = __any_sync(0xffffffffu, pa_wild(big));
            }
            if (!wild) {
#pragma unroll
                for (int d2 = 0; d2 < D / 16; ++d2) {
                    uint32_t bv[4];
                    values(bv, d2);
                    if (tail) cut(bv, len1);
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float w[4] = {0.f, 0.f, 0.f, 0.f};
                        pa_mma(w, pl, bv[2 * c], bv[2 * c + 1]);
                        pa_mma(w, ph, bv[2 * c], bv[2 * c + 1]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[2 * d2 + c][i] = fmaf(o[2 * d2 + c][i], corr[i >> 1], w[i]);
                    }
                }
            } else {
                // one token after the other, with the values that it does not see taken out, into the rows of that token
#pragma unroll 1
                for (uint32_t tok = tok0; tok <= tok1; ++tok) {
                    const int32_t last = min(rq.pos0 + (int32_t)tok, len1);
#pragma unroll
                    for (int d2 = 0; d2 < D / 16; ++d2) {
                        uint32_t bv[4];
                        values(bv, d2);
                        cut(bv, last);
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            float w[4] = {0.f, 0.f, 0.f, 0.f}, u[4] = {0.f, 0.f, 0.f, 0.f};
                            pa_mma(w, pl, bv[2 * c], bv[2 * c + 1]);
                            pa_mma(u, ph, bv[2 * c], bv[2 * c + 1]);
                            // (zero times infinity in the trailing bits is no reason for a NaN)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const uint32_t m = rg * 16u + g + 8u * (i >> 1);
                                const float add = fabsf(w[i]) < INFINITY ? u[i] + w[i] : u[i];
                                if (m / G == tok) o[2 * d2 + c][i] = fmaf(o[2 * d2 + c][i], corr[i >> 1], add);
                            }
                        }
                    }
                }
            }
            __syncwarp();                              // the stage is read
            fetch(b + ST);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            l_[i] += __shfl_xor_sync(0xffffffffu, l_[i], 1);
            l_[i] += __shfl_xor_sync(0xffffffffu, l_[i], 2);
            if (!ok) l_[i] = __int_as_float(0x7fc00000);
        }
        float z = 0.f;
#pragma unroll
        for (int d = 0; d < D / 8; ++d) z = fmaf(o[d][0], 0.f, fmaf(o[d][1], 0.f, fmaf(o[d][2], 0.f, fmaf(o[d][3], 0.f, z))));
        if (careful || !__syncthreads_or(z != 0.f)) break;             // all sums are finite
        }
        // ---- the warps' sums; whole: this is all of the pair
        const bool whole = b0 == 0u && b1 == kb;
        const unsigned long long x0 = x - b0;          // the pair's first block
        float *dst = a.part + (size_t)(2u * me + (x == x_begin ? 0u : 1u)) * CF::kSlot;
        auto out_row = [&](uint32_t m) {               // row m of the group
            const uint32_t q = rg * 16u + m, tok = q / G;
            return a.out + ((size_t)(rq.row0 + tok) * a.hq + h * G + (q - tok * G)) * D;
        };
        auto write_out = [&](uint32_t m, uint32_t d4, const float4 &v, float l) {
            const uint32_t tok = (rg * 16u + m) / G;
            const bool sees = rq.pos0 + (int32_t)tok >= 0 && rq.len > 0u;      // a row that sees nothing is zero
            const float inv = sees ? 1.f / l : 0.f;
            *(uint2 *)(out_row(m) + d4 * 4) = sees ? make_uint2(pa_pack(v.x * inv, v.y * inv), pa_pack(v.z * inv, v.w * inv)) : make_uint2(0u, 0u);
        };
#pragma unroll
        for (int i = 0; i < 2; ++i) {                  // rows 0 .. 7, rows 8 .. 15
            if (rows <= 8u * i) break;                 // uniform
            __syncthreads();
            if (g + 8u * i < rows) {
                float *to = sum + (wid * 8u + g) * CF::kPitch + 2u * t;
#pragma unroll
                for (int d = 0; d < D / 8; ++d) *(float2 *)(to + d * 8) = make_float2(o[d][2 * i], o[d][2 * i + 1]);
                if (t == 0) *(float2 *)(sum + (wid * 8u + g) * CF::kPitch + D) = make_float2(m_[i], l_[i]);
            }
            __syncthreads();
            for (uint32_t it = tid; it < min(8u, rows - 8u * i) * (D / 4); it += CF::kThreads) {
                const uint32_t row = it / (D / 4), d4 = it % (D / 4);
                float M = -INFINITY, L = 0.f;
#pragma unroll
                for (int w = 0; w < NW; ++w) M = fmaxf(M, sum[(w * 8u + row) * CF::kPitch + D]);
                const float mb = M == -INFINITY ? 0.f : M * sl2;
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < NW; ++w) {
                    const float2 ml = *(const float2 *)(sum + (w * 8u + row) * CF::kPitch + D);
                    const float f = pa_exp2(fmaf(ml.x, sl2, -mb));
                    const float4 u = *(const float4 *)(sum + (w * 8u + row) * CF::kPitch + d4 * 4);
                    L = fmaf(ml.y, f, L);
                    v.x = fmaf(u.x, f, v.x); v.y = fmaf(u.y, f, v.y); v.z = fmaf(u.z, f, v.z); v.w = fmaf(u.w, f, v.w);
                }
                const uint32_t m = row + 8u * i;
                if (whole) {
                    write_out(m, d4, v, L);
                } else {
                    *(float4 *)(dst + m * D + d4 * 4) = v;
                    if (d4 == 0u) *(float2 *)(dst + 16 * D + 2 * m) = make_float2(M, L);
                }
            }
        }
        if (!whole) {
            // the CTA of block y is the last c with W c / N <= y
            const uint32_t c0 = (uint32_t)(((x0 + 1ull) * N - 1ull) / W), c1 = (uint32_t)(((x0 + kb) * N - 1ull) / W), parts = c1 - c0 + 1u;
            __syncthreads();
            // numbers whose sum is zero, so the ticket is zero again when all have come
            if (tid == 0) {
                const uint32_t add = me == c0 ? 1u - parts : 1u;
                __threadfence();                       // the CTA's parts (behind the barrier) before the ticket
                sm_last = atomicAdd(a.tickets + c0, add) + add == 0u;
                __threadfence();
            }
            __syncthreads();
            if (sm_last) {
                const uint32_t behind = W * c0 / N != x0 ? 1u : 0u;
                auto slot_of = [&](uint32_t c) { return a.part + (size_t)(2u * c + (c == c0 ? behind : 0u)) * CF::kSlot; };
                // what every part counts, for every row: all of the parts' numbers are requested at once
                float2 *ml = (float2 *)pa_smem;        // [parts][rows] (maximum, denominator): nothing is on its way into the ring
                for (uint32_t i = tid; i < parts * rows; i += CF::kThreads) ml[i] = __ldcg((const float2 *)(slot_of(c0 + i / rows) + 16 * D) + i % rows);
                __syncthreads();
                for (uint32_t it = tid; it < rows * (D / 4); it += CF::kThreads) {
                    const uint32_t m = it / (D / 4), d4 = it % (D / 4);
                    float M = -INFINITY, L = 0.f;
                    for (uint32_t p = 0; p < parts; ++p) M = fmaxf(M, ml[p * rows + m].x);
                    const float mb = M == -INFINITY ? 0.f : M * sl2;
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
                    for (uint32_t p = 0; p < parts; ++p) {
                        const float4 u = __ldcg((const float4 *)(slot_of(c0 + p) + m * D) + d4);
                        const float2 e = ml[p * rows + m];
                        const float f = pa_exp2(fmaf(e.x, sl2, -mb));
                        L = fmaf(e.y, f, L);
                        v.x = fmaf(u.x, f, v.x); v.y = fmaf(u.y, f, v.y); v.z = fmaf(u.z, f, v.z); v.w = fmaf(u.w, f, v.w);
                    }
                    write_out(m, d4, v, L);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncthreads();                       // the ring is free again
            }
        }
        x += b1 - b0;
        if (x >= x_end) break;
        // ---- the next pair: row group, request, KV head
        if (++rg * 16u >= rq.n * G) {
            rg = 0;
            do {
                if (++r == R) {
                    r = 0;
                    ++h;
                }
                rq = paged_req(a, r);
            } while (!mine(rq) && h < a.hkv);          // (there is one, unless the lengths change under the kernel)
            if (h >= a.hkv) break;
            kb = key_blocks(rq);
        }
        b0 = 0;
    }
    if (!ok)                                           // (otherwise every copy has been waited for)
        for (uint32_t i = n > (uint32_t)ST ? n - ST : 0u; i < n; ++i) pa_wait(bar0 + 8u * (i % ST), i / ST & 1u);
}

}  // namespace ixb
