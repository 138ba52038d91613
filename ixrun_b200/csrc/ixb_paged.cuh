// Paged KV cache of a batch of requests: which pages a step writes, and the write itself.
//
//   k_page_step     block tables and slot maps of a step from the requests' lengths and their numbers of new tokens
//   k_page_release  pages of finished requests back onto the free stack
//   k_rope_paged    per-head q/k norm (optional), rotary embedding, keys and values into their slots
//
// A page holds 2^log_page positions of one request; table [requests][width] has the page of every 2^log_page positions; the free
// pages are the entries below n_free of a stack.  Slot = page * 2^log_page + position % 2^log_page: the row of the pool
// [pages * 2^log_page][kv heads][D].
#pragma once
#include "ixb_common.cuh"

namespace ixb {

constexpr int kPageThreads = 512;
constexpr int kPageMaxRequests = 4096;
constexpr int kPageMaxCtas = 8;                        // of the one cluster
constexpr int kPageRelease = 4;                        // status: a release would overfill the stack
constexpr uint32_t kPageNoPages = 1, kPageNoRows = 2, kPageNoTable = 4;

// exclusive sums over the CTA of two numbers per thread; tot: the sums over all threads
__device__ __forceinline__ void page_scan(long long &a, long long &b, long long (&red)[2][kPageThreads / 32], long long (&tot)[2])
{
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    const long long a0 = a, b0 = b;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, a, d), y = __shfl_up_sync(0xffffffffu, b, d);
        if (lane >= d) {
            a += x;
            b += y;
        }
    }
    if (lane == 31) {
        red[0][wid] = a;
        red[1][wid] = b;
    }
    __syncthreads();
    long long pa = 0, pb = 0, ta = 0, tb = 0;
#pragma unroll
    for (int w = 0; w < kPageThreads / 32; ++w) {
        if (w == wid) {
            pa = ta;
            pb = tb;
        }
        ta += red[0][w];
        tb += red[1][w];
    }
    a += pa - a0;
    b += pb - b0;
    tot[0] = ta;
    tot[1] = tb;
}

// last index r in [0, n) with first[r] <= x; first is non-decreasing and first[0] <= x
__device__ __forceinline__ uint32_t page_find(const int32_t *first, uint32_t n, int32_t x)
{
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1u) {
        const uint32_t mid = (lo + hi) / 2u;
        if (first[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

struct PageStep {
    const int32_t *q_len, *length, *free_pages, *n_free;
    int32_t *table;
    int32_t *cu_rows, *new_length, *new_n_free, *slot, *pos, *owner, *status;      // new_length may be length, new_n_free n_free
    uint32_t requests, width, n_pages, log_page, rows;
};

// One cluster of up to eight CTAs.  Every CTA sums the requests up for itself (a few thousand numbers at most), a barrier of the
// cluster lies between the last read of what is updated in place and the first write, and the rows and new pages are shared out
// over all threads.  Latency is all there is: 200 KB of output for the largest steps.  3.6 us for 40 single tokens, 6.9 for 512 requests
// with 16700 new tokens (13 with one CTA).
//
// A step that does not fit (too few free pages, rows or table entries) takes nothing: cu_rows is zero, no row has a slot, lengths
// and stack stay; status says why.
__global__ void __launch_bounds__(kPageThreads)
k_page_step(PageStep s)
{
    extern __shared__ int32_t page_smem[];             // [3][requests + 1]: rows before, new pages before, length
    __shared__ long long red[2][kPageThreads / 32];
    __shared__ uint32_t sm_flags;
    const uint32_t R = s.requests, tid = threadIdx.x, ctas = gridDim.x, me = blockIdx.x;
    int32_t *cu = page_smem, *first = cu + R + 1, *len = first + R + 1;
    asm volatile("griddepcontrol.launch_dependents;");
    if (tid == 0) sm_flags = 0u;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __syncthreads();
    const long long page = 1ll << s.log_page, mask = page - 1;
    const uint32_t per = (R + kPageThreads - 1) / kPageThreads, r0 = min(R, tid * per), r1 = min(R, r0 + per);
    const int32_t n_free = min(max(*s.n_free, 0), (int32_t)s.n_pages);
    long long nq = 0, np = 0;
    bool wide = false;
    for (uint32_t r = r0; r < r1; ++r) {
        const long long q = max(s.q_len[r], 0), l = max(s.length[r], 0);
        const long long have = (l + mask) >> s.log_page, need = (l + q + mask) >> s.log_page;
        nq += q;
        np += need - have;
        wide = wide || (q > 0 && need > (long long)s.width) || l + q > 0x7fffffffll;
    }
    if (wide) atomicOr(&sm_flags, kPageNoTable);
    long long tot[2];
    page_scan(nq, np, red, tot);
    uint32_t flags = 0;
    if (tot[0] > (long long)s.rows) flags |= kPageNoRows;
    if (tot[1] > (long long)n_free) flags |= kPageNoPages;
    for (uint32_t r = r0; r < r1; ++r) {               // (of a step that fits these are small)
        const long long q = max(s.q_len[r], 0), l = max(s.length[r], 0);
        cu[r] = (int32_t)nq;
        first[r] = (int32_t)np;
        len[r] = (int32_t)l;
        nq += q;
        np += ((l + q + mask) >> s.log_page) - ((l + mask) >> s.log_page);
    }
    if (tid == 0) {
        cu[R] = (int32_t)tot[0];
        first[R] = (int32_t)tot[1];
    }
    __syncthreads();
    flags |= sm_flags;                                 // (written before page_scan's barrier)
    if (ctas > 1u) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    const uint32_t g = me * kPageThreads + tid, stride = ctas * kPageThreads;
    const bool fits = flags == 0u;
    if (g == 0) {
        *s.new_n_free = fits ? n_free - (int32_t)tot[1] : n_free;
        s.status[0] = (int32_t)flags;
        s.status[1] = (int32_t)min(tot[1], 0x7fffffffll);
    }
    for (uint32_t r = g; r <= R; r += stride) {
        s.cu_rows[r] = fits ? cu[r] : 0;
        if (r < R) s.new_length[r] = fits ? len[r] + cu[r + 1] - cu[r] : len[r];
    }
    const uint32_t n_rows = fits ? (uint32_t)tot[0] : 0u, n_new = fits ? (uint32_t)tot[1] : 0u;
    for (uint32_t i = g; i < n_new; i += stride) {
        const uint32_t r = page_find(first, R, (int32_t)i);
        const uint32_t have = (uint32_t)(((long long)len[r] + mask) >> s.log_page);
        s.table[(size_t)r * s.width + have + (i - (uint32_t)first[r])] = s.free_pages[n_free - 1 - (int32_t)i];
    }
    for (uint32_t t = g; t < s.rows; t += stride) {
        int32_t slot = -1, pos = 0, owner = -1;
        if (t < n_rows) {
            const uint32_t r = page_find(cu, R, (int32_t)t);
            owner = (int32_t)r;
            pos = len[r] + (int32_t)t - cu[r];
            const uint32_t have = (uint32_t)(((long long)len[r] + mask) >> s.log_page), b = (uint32_t)pos >> s.log_page;
            const int32_t p = b < have ? s.table[(size_t)r * s.width + b] : s.free_pages[n_free - 1 - (first[r] + (int32_t)(b - have))];
            if ((uint32_t)p < s.n_pages) slot = (int32_t)(((uint32_t)p << s.log_page) + ((uint32_t)pos & (uint32_t)mask));
        }
        s.slot[t] = slot;
        s.pos[t] = pos;
        s.owner[t] = owner;
    }
}

struct PageRelease {
    const uint8_t *done;
    const int32_t *table;
    int32_t *length, *free_pages, *n_free, *status;
    uint32_t requests, width, n_pages, log_page;
};

// One CTA: the pages of the requests with done[r] != 0 onto the stack, in the order of requests and positions; their lengths become
// zero.  If the stack cannot take them (a page would be on it twice) nothing is done.  3.1 us for 40 requests with 760 pages; 39 for 512
// with 32256, 79 for 4096 with 53248: a search per page and one CTA's threads.
__global__ void __launch_bounds__(kPageThreads)
k_page_release(PageRelease s)
{
    extern __shared__ int32_t page_smem[];             // [requests + 1] pages before
    __shared__ long long red[2][kPageThreads / 32];
    const uint32_t R = s.requests, tid = threadIdx.x;
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const long long mask = (1ll << s.log_page) - 1;
    const uint32_t per = (R + kPageThreads - 1) / kPageThreads, r0 = min(R, tid * per), r1 = min(R, r0 + per);
    const int32_t n_free = min(max(*s.n_free, 0), (int32_t)s.n_pages);
    auto pages = [&](uint32_t r) { return s.done[r] ? min(((long long)max(s.length[r], 0) + mask) >> s.log_page, (long long)s.width) : 0ll; };
    long long n = 0, zero = 0, tot[2];
    for (uint32_t r = r0; r < r1; ++r) n += pages(r);
    page_scan(n, zero, red, tot);
    const bool fits = tot[0] + n_free <= (long long)s.n_pages;
    for (uint32_t r = r0; r < r1; ++r) {
        page_smem[r] = (int32_t)n;
        n += pages(r);
    }
    if (tid == 0) page_smem[R] = (int32_t)tot[0];
    __syncthreads();
    if (tid == 0) {
        s.status[0] = fits ? 0 : kPageRelease;
        s.status[1] = (int32_t)min(tot[0], 0x7fffffffll);
        if (fits) *s.n_free = n_free + (int32_t)tot[0];
    }
    if (!fits) return;
    for (uint32_t i = tid; i < (uint32_t)tot[0]; i += kPageThreads) {
        const uint32_t r = page_find(page_smem, R, (int32_t)i);
        s.free_pages[n_free + i] = s.table[(size_t)r * s.width + (i - (uint32_t)page_smem[r])];
    }
    for (uint32_t r = tid; r < R; r += kPageThreads)
        if (s.done[r]) s.length[r] = 0;
}

// ---------------------------------------------------------------- q/k norm + RoPE + write into the pages
struct RopePaged {
    const __nv_bfloat16 *q, *k, *v;
    __nv_bfloat16 *out, *k_pages, *v_pages;            // out may be q
    const int32_t *pos, *slot;
    const __nv_bfloat16 *q_norm, *k_norm;
    const float *cos_tab, *sin_tab;                    // [max_seq][rot / 2]
    uint32_t hq, hkv, rot, max_seq, log_page;
    float eps;
    size_t q_stride, kv_stride, out_stride, k_page_stride, v_page_stride, n_slots;      // elements; rows of the pool
    uint32_t ahead;                                    // rows ahead that are asked for from L2
};

// One CTA per row: D / 16 threads take a head (two pieces of eight elements each: a rotated pair of pieces, or two that pass
// through), the CTA's HL heads at a time, so that a row's tables are read once.  Everything is held in fp32 and rounded to bf16
// once (the static cache's kernel rounds where the eager path holds bf16 tensors).  A row without a slot (-1, or outside the pool)
// is left alone; a position outside the tables is taken as the nearest one in them.  Bound: HBM, each element read once and written once:
// 7700 rows of 24 / 4 heads of 256 with norms take 48.5 us in a captured graph, 80 % of the copy rate (51 called one by one).  Five CTAs an SM, each with one row in flight, and each asks L2 for a row of a CTA to come, two rows an SM ahead (50.9
// without; one, three and five: 48.5, 48.7, 50.1; 16000 rows of 16 / 8 heads of 128 61.1 without, 56.0).  Six CTAs with fewer
// registers: 51.6 instead of 50.6.
template <int D>
__global__ void __launch_bounds__(128)
k_rope_paged(RopePaged s)
{
    constexpr int PT = D / 16, HL = 128 / PT;          // threads per head, heads at a time
    const uint32_t row = blockIdx.x, part = threadIdx.x % PT, hl = threadIdx.x / PT;
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t heads = s.hq + 2u * s.hkv, turned = s.rot / 16u;            // threads whose pieces are rotated
    const bool rot = part < turned;
    // elements a .. a + 7 and b .. b + 7 of a head
    const uint32_t a = rot ? 8u * part : s.rot + 16u * (part - turned), b = rot ? a + s.rot / 2u : a + 8u;
    constexpr int UN = 4;                              // heads of a thread in flight
    uint4 ra[UN], rb[UN];
    auto fetch = [&](uint32_t h0) {
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const uint32_t h = h0 + u * HL + hl;
            ra[u] = rb[u] = make_uint4(0, 0, 0, 0);
            if (h < heads) {
                const __nv_bfloat16 *src = h < s.hq ? s.q + (size_t)row * s.q_stride + (size_t)h * D
                                                    : (h < s.hq + s.hkv ? s.k + (size_t)(h - s.hq) * D : s.v + (size_t)(h - s.hq - s.hkv) * D) + (size_t)row * s.kv_stride;
                ra[u] = *(const uint4 *)(src + a);
                rb[u] = *(const uint4 *)(src + b);
            }
        }
    };
    if (threadIdx.x < 3u && gridDim.x - row > s.ahead) {
        const size_t r = row + s.ahead;
        const __nv_bfloat16 *src = threadIdx.x == 0 ? s.q + r * s.q_stride : (threadIdx.x == 1 ? s.k : s.v) + r * s.kv_stride;
        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(src), "r"((threadIdx.x == 0 ? s.hq : s.hkv) * (uint32_t)D * 2u) : "memory");
    }
    fetch(0u);                                         // (beside the slot and the position: one trip to memory less)
    const int32_t slot = s.slot[row];
    const uint32_t p = min((uint32_t)max(s.pos[row], 0), s.max_seq - 1u);
    if (slot < 0 || (size_t)slot >= s.n_slots) return;
    float c[8], sn[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        c[j] = 1.f;
        sn[j] = 0.f;
    }
    if (rot) {
        const float4 *ct = (const float4 *)(s.cos_tab + (size_t)p * (s.rot / 2u) + a), *st = (const float4 *)(s.sin_tab + (size_t)p * (s.rot / 2u) + a);
        const float4 c0 = ct[0], c1 = ct[1], s0 = st[0], s1 = st[1];
        c[0] = c0.x; c[1] = c0.y; c[2] = c0.z; c[3] = c0.w; c[4] = c1.x; c[5] = c1.y; c[6] = c1.z; c[7] = c1.w;
        sn[0] = s0.x; sn[1] = s0.y; sn[2] = s0.z; sn[3] = s0.w; sn[4] = s1.x; sn[5] = s1.y; sn[6] = s1.z; sn[7] = s1.w;
    }
    const size_t in_page = (uint32_t)slot & ((1u << s.log_page) - 1u), page = (uint32_t)slot >> s.log_page;
    __nv_bfloat16 *kd = s.k_pages + page * s.k_page_stride + in_page * s.hkv * D, *vd = s.v_pages + page * s.v_page_stride + in_page * s.hkv * D;
    auto f8 = [](const uint4 &r, float (&f)[8]) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f[2 * j] = __uint_as_float(w[j] << 16);
            f[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        }
    };
    auto b8 = [](const float (&f)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
            w[j] = *(const uint32_t *)&h;
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    };
    for (uint32_t h0 = 0; h0 < heads; h0 += UN * HL) { // (the bound is the same for all threads: shuffles below)
        if (h0) fetch(h0);
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const uint32_t h = h0 + u * HL + hl;
            if (h0 + u * HL >= heads) break;           // uniform
            const bool is_q = h < s.hq, is_v = h >= s.hq + s.hkv;
            __nv_bfloat16 *dst = is_q ? s.out + (size_t)row * s.out_stride + (size_t)h * D
                                      : is_v ? vd + (size_t)(h - s.hq - s.hkv) * D : kd + (size_t)(h - s.hq) * D;
            float x[8], y[8], ox[8], oy[8];
            f8(ra[u], x);
            f8(rb[u], y);
            const __nv_bfloat16 *nw = is_q ? s.q_norm : is_v ? nullptr : s.k_norm;
            if (s.q_norm || s.k_norm) {                // uniform
                float ss = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], fmaf(y[j], y[j], ss));
#pragma unroll
                for (int d = 1; d < PT; d <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
                if (nw) {
                    const float r = rsqrtf(ss / (float)D + s.eps);
                    float wx[8], wy[8];
                    f8(*(const uint4 *)(nw + a), wx);
                    f8(*(const uint4 *)(nw + b), wy);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        x[j] = x[j] * r * wx[j];
                        y[j] = y[j] * r * wy[j];
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                ox[j] = rot ? x[j] * c[j] - y[j] * sn[j] : x[j];
                oy[j] = rot ? y[j] * c[j] + x[j] * sn[j] : y[j];
            }
            if (h < heads) {
                *(uint4 *)(dst + a) = is_v ? ra[u] : b8(ox);
                *(uint4 *)(dst + b) = is_v ? rb[u] : b8(oy);
            }
        }
    }
}

// The same for any even rot and alignment: a warp per head, one pair of elements a lane at a time.
__global__ void __launch_bounds__(128)
k_rope_paged_any(RopePaged s, uint32_t D)
{
    const uint32_t row = blockIdx.x, lane = threadIdx.x & 31u, wid = threadIdx.x >> 5, half = s.rot / 2u, pairs = D / 2u;
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int32_t slot = s.slot[row];
    const uint32_t p = min((uint32_t)max(s.pos[row], 0), s.max_seq - 1u);
    if (slot < 0 || (size_t)slot >= s.n_slots) return;
    const size_t in_page = (uint32_t)slot & ((1u << s.log_page) - 1u), page = (uint32_t)slot >> s.log_page;
    for (uint32_t h = wid; h < s.hq + 2u * s.hkv; h += 4u) {
        const bool is_q = h < s.hq, is_v = h >= s.hq + s.hkv;
        const uint32_t kh = is_q ? 0u : is_v ? h - s.hq - s.hkv : h - s.hq;
        const __nv_bfloat16 *src = is_q ? s.q + (size_t)row * s.q_stride + (size_t)h * D : (is_v ? s.v : s.k) + (size_t)row * s.kv_stride + (size_t)kh * D;
        __nv_bfloat16 *dst = is_q ? s.out + (size_t)row * s.out_stride + (size_t)h * D
                           : is_v ? s.v_pages + page * s.v_page_stride + (in_page * s.hkv + kh) * D
                                  : s.k_pages + page * s.k_page_stride + (in_page * s.hkv + kh) * D;
        const __nv_bfloat16 *nw = is_q ? s.q_norm : is_v ? nullptr : s.k_norm;
        float r = 1.f;
        if (nw) {
            float ss = 0.f;
            for (uint32_t e = lane; e < D; e += 32u) {
                const float x = __bfloat162float(src[e]);
                ss = fmaf(x, x, ss);
            }
            r = rsqrtf(warp_sum(ss) / (float)D + s.eps);
        }
        auto at = [&](uint32_t e) { return nw ? __bfloat162float(src[e]) * r * __bfloat162float(nw[e]) : __bfloat162float(src[e]); };
        for (uint32_t i = lane; i < pairs; i += 32u) { // a pair is read and written by one lane: out may be q
            const bool rot = i < half;
            const uint32_t e0 = rot ? i : s.rot + 2u * (i - half), e1 = rot ? i + half : e0 + 1u;
            const float x = at(e0), y = at(e1);
            const bool turn = rot && !is_v;
            const float c = turn ? s.cos_tab[(size_t)p * half + i] : 1.f, sn = turn ? s.sin_tab[(size_t)p * half + i] : 0.f;
            dst[e0] = __float2bfloat16_rn(turn ? x * c - y * sn : x);
            dst[e1] = __float2bfloat16_rn(turn ? y * c + x * sn : y);
        }
    }
}

}  // namespace ixb
