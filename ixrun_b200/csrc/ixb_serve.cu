// C-ABI entry points of a serving step over a paged KV cache: page tables, rotary embedding and write, attention, rules on logits.
// See include/ixb200.h for the contract of each call.
#include "ixb_api.cuh"
#include "ixb_attn_chunk.cuh"
#include "ixb_attn_paged.cuh"
#include "ixb_logits.cuh"
#include "ixb_paged.cuh"

#include <algorithm>

using namespace ixb;

// a page holds 16, 32, ... 256 positions; 0: something else
static uint32_t log_page(int64_t page)
{
    for (uint32_t l = 4; l <= 8; ++l)
        if (page == 1ll << l) return l;
    return 0;
}

static int page_shape(int64_t requests, int64_t width, int64_t n_pages, int64_t page)
{
    if (requests <= 0 || requests > kPageMaxRequests) return fail(IXB_E_UNSUPPORTED, "%lld requests: 1..%d", (long long)requests, kPageMaxRequests);
    if (!log_page(page)) return fail(IXB_E_UNSUPPORTED, "pages of %lld positions: 16, 32, 64, 128 or 256", (long long)page);
    if (width <= 0 || n_pages <= 0 || n_pages > 0x7fffffffll / page || width > 0x7fffffffll / page) return fail(IXB_E_ARG, "bad shape");
    return IXB_OK;
}

extern "C" int ixb_page_step(const int32_t *q_len, const int32_t *length, int32_t *table, const int32_t *free_pages, const int32_t *n_free,
                             int64_t requests, int64_t width, int64_t n_pages, int64_t page, int64_t rows, int32_t *cu_rows, int32_t *new_length,
                             int32_t *new_n_free, int32_t *slot, int32_t *pos, int32_t *owner, int32_t *status, ixb_stream_t stream)
{
    if (!q_len || !length || !table || !free_pages || !n_free || !cu_rows || !new_length || !new_n_free || !status) return fail(IXB_E_ARG, "NULL pointer argument");
    if (rows < 0 || rows > 0x7fffffffll || (rows && (!slot || !pos || !owner))) return fail(IXB_E_ARG, "bad rows");
    const int rc = page_shape(requests, width, n_pages, page);
    if (rc) return rc;
    const PageStep s = {q_len, length, free_pages, n_free, table, cu_rows, new_length, new_n_free, slot, pos, owner, status, (uint32_t)requests,
                        (uint32_t)width, (uint32_t)n_pages, log_page(page), (uint32_t)rows};
    static bool attr_set[64] = {false};
    IXB_CUDA(opt_in_smem(k_page_step, attr_set, 3 * (kPageMaxRequests + 1) * 4));
    cudaLaunchConfig_t cfg = {};
    // two rows a thread, and one CTA as long as that takes no longer
    cfg.gridDim = dim3((unsigned)std::min<int64_t>(kPageMaxCtas, std::max<int64_t>(1, (rows + 2 * kPageThreads - 1) / (2 * kPageThreads))));
    cfg.blockDim = dim3(kPageThreads);
    cfg.dynamicSmemBytes = 3 * ((size_t)requests + 1) * 4;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cfg.gridDim.x;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_on() ? 2 : 1;
    IXB_GLUE("k_page_step", cudaLaunchKernelEx(&cfg, k_page_step, s));
}

extern "C" int ixb_page_release(const uint8_t *done, int32_t *length, const int32_t *table, int32_t *free_pages, int32_t *n_free, int64_t requests,
                                int64_t width, int64_t n_pages, int64_t page, int32_t *status, ixb_stream_t stream)
{
    if (!done || !length || !table || !free_pages || !n_free || !status) return fail(IXB_E_ARG, "NULL pointer argument");
    const int rc = page_shape(requests, width, n_pages, page);
    if (rc) return rc;
    const PageRelease s = {done, table, length, free_pages, n_free, status, (uint32_t)requests, (uint32_t)width, (uint32_t)n_pages, log_page(page)};
    IXB_GLUE("k_page_release", launch_glue_smem(k_page_release, dim3(1), dim3(kPageThreads), ((size_t)requests + 1) * 4, (cudaStream_t)stream, s));
}

extern "C" int ixb_rope_paged(const void *q, const void *k, const void *v, const int32_t *pos, const int32_t *slot, void *k_pages, void *v_pages,
                              const void *q_norm, const void *k_norm, const float *cos_tab, const float *sin_tab, void *out, int64_t rows,
                              int64_t hq, int64_t hkv, int64_t head_dim, int64_t rot_dim, float eps, int64_t q_stride, int64_t kv_stride,
                              int64_t out_stride, int64_t max_seq, int64_t n_pages, int64_t page, int64_t k_page_stride, int64_t v_page_stride,
                              ixb_stream_t stream)
{
    if (!q || !k || !v || !pos || !slot || !k_pages || !v_pages || !cos_tab || !sin_tab || !out) return fail(IXB_E_ARG, "NULL pointer argument");
    if (rows <= 0 || rows > 0x7fffffffll || hq <= 0 || hkv <= 0 || hq > 65535 || hkv > 65535 || max_seq <= 0 || max_seq > 0x7fffffffll) return fail(IXB_E_ARG, "bad shape");
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) return fail(IXB_E_UNSUPPORTED, "head_dim=%lld: 64, 128 or 256", (long long)head_dim);
    if (rot_dim <= 0 || rot_dim > head_dim || (rot_dim & 1)) return fail(IXB_E_ARG, "rot_dim must be even and at most head_dim");
    const int rc = page_shape(1, 1, n_pages, page);
    if (rc) return rc;
    if (q_stride < hq * head_dim || kv_stride < hkv * head_dim || out_stride < hq * head_dim || k_page_stride < page * hkv * head_dim ||
        v_page_stride < page * hkv * head_dim)
        return fail(IXB_E_ARG, "bad strides");
    const RopePaged s = {(const __nv_bfloat16 *)q, (const __nv_bfloat16 *)k, (const __nv_bfloat16 *)v, (__nv_bfloat16 *)out, (__nv_bfloat16 *)k_pages,
                         (__nv_bfloat16 *)v_pages, pos, slot, (const __nv_bfloat16 *)q_norm, (const __nv_bfloat16 *)k_norm, cos_tab, sin_tab,
                         (uint32_t)hq, (uint32_t)hkv, (uint32_t)rot_dim, (uint32_t)max_seq, log_page(page), eps, (size_t)q_stride, (size_t)kv_stride,
                         (size_t)out_stride, (size_t)k_page_stride, (size_t)v_page_stride, (size_t)(n_pages * page),
                         (uint32_t)(2 * num_sms())};
    const uintptr_t all = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)out | (uintptr_t)q_norm |
                          (uintptr_t)k_norm | (uintptr_t)cos_tab | (uintptr_t)sin_tab;
    const cudaStream_t st = (cudaStream_t)stream;
    // pieces of eight elements: rotated ones fill whole threads, and everything lies on 16 bytes
    if (rot_dim % 16 == 0 && (all & 15u) == 0 && ((q_stride | kv_stride | out_stride | k_page_stride | v_page_stride) & 7) == 0) {
        IXB_GLUE("k_rope_paged", head_dim == 64    ? launch_glue_smem(k_rope_paged<64>, dim3((unsigned)rows), dim3(128), 0, st, s)
                                 : head_dim == 128 ? launch_glue_smem(k_rope_paged<128>, dim3((unsigned)rows), dim3(128), 0, st, s)
                                                   : launch_glue_smem(k_rope_paged<256>, dim3((unsigned)rows), dim3(128), 0, st, s));
    }
    IXB_GLUE("k_rope_paged_any", launch_glue_smem(k_rope_paged_any, dim3((unsigned)rows), dim3(128), 0, st, s, (uint32_t)head_dim));
}

// ------------------------------------------------------------------------------------------------ attention over pages
// Requests with at most this many rows (new tokens times query heads of a KV head) go through k_attn_paged in one group of rows, the
// others through k_attn_chunk.  (Sixteen rows of 256 dimensions do not fit its registers.)
template <int D>
constexpr uint32_t few_rows() { return D == 256 ? 8 : 16; }
constexpr size_t kPaTicketBytes = 4096, kPaCutBytes = 8192;       // a word, a PcCut per CTA; the tickets are zero between launches

template <int D>
static size_t few_part_floats() { return (size_t)num_sms() * 2 * PaCfg<D>::kSlot; }
template <int D>
static size_t attn_part_bytes()                        // (the two kernels of a call overlap)
{
    return 4 * (few_part_floats<D>() + (size_t)num_sms() * 2 * PcCfg<D>::kPart);
}
extern "C" size_t ixb_attn_paged_scratch_bytes(int64_t head_dim)
{
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) return 0;
    return kPaTicketBytes + kPaCutBytes + (head_dim == 64 ? attn_part_bytes<64>() : head_dim == 128 ? attn_part_bytes<128>() : attn_part_bytes<256>());
}

// a pool as a tensor of [pages][page][kv heads][D]: boxes of 64 dimensions of one head of (at most 128) positions of a page
static CUresult pool_map(CUtensorMap *map, const __nv_bfloat16 *pool, size_t page_stride, const PagedAttn &a, uint32_t D)
{
    // (heads of 64 with 128-byte lines: of a larger piece the half would be another head's, 64 requests behind 4000 128 us instead of 100)
    const cuuint64_t dims[4] = {D, a.hkv, 1ull << a.log_page, a.n_pages}, strides[3] = {D * 2ull, (cuuint64_t)a.hkv * D * 2, (cuuint64_t)page_stride * 2};
    const cuuint32_t box[4] = {64, 1, std::min(1u << a.log_page, kPcKeys), 1}, one[4] = {1, 1, 1, 1};
    return tensor_map_encoder()(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<__nv_bfloat16 *>(pool), dims, strides, box, one,
                                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                D == 64 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

template <int D, int NT>
static int launch_attn_few(const PagedAttn &a, const CUtensorMap &kmap, const CUtensorMap &vmap, cudaStream_t st)
{
    static bool attr_set[64] = {false};
    IXB_CUDA(opt_in_smem(k_attn_paged<D, NT>, attr_set, (int)PaCfg<D>::kSmem));
    IXB_CUDA(launch_glue_smem(k_attn_paged<D, NT>, dim3((unsigned)num_sms()), dim3(PaCfg<D>::kThreads), PaCfg<D>::kSmem, st, a, kmap, vmap));
    return launch_check("k_attn_paged");
}

template <int D>
static int attn_paged_run(PagedAttn a, PcCut *cuts, int64_t max_q, cudaStream_t st)
{
    const unsigned sms = (unsigned)num_sms();
    const bool few = max_q * a.group <= few_rows<D>(), both = !few && a.requests > 1u;
    if (!tensor_map_encoder()) return fail(IXB_E_UNSUPPORTED, "the driver has no cuTensorMapEncodeTiled");
    CUtensorMap kmap, vmap;
    CUresult r = pool_map(&kmap, a.k, a.k_stride, a, D);
    if (r == CUDA_SUCCESS) r = pool_map(&vmap, a.v, a.v_stride, a, D);
    if (r != CUDA_SUCCESS) return fail(IXB_E_CUDA, "tensor map of a pool: error %d", (int)r);
    int rc;
    if (few || both) {
        if (both) a.row_hi = few_rows<D>();
        rc = D == 256 || (few && max_q * a.group <= 8) ? launch_attn_few<D, 1>(a, kmap, vmap, st) : launch_attn_few<D, D == 256 ? 1 : 2>(a, kmap, vmap, st);
        if (rc || few) return rc;
        a.row_lo = few_rows<D>();
        a.row_hi = 0xffffffffu;
        a.part += few_part_floats<D>();
        a.second = 1u;
    }
    static bool attr_set[64] = {false};
    IXB_CUDA(opt_in_smem(k_attn_chunk<D>, attr_set, (int)PcCfg<D>::kSmem));
    // (launches of one call may begin while the one before ends)
    IXB_CUDA(launch_overlapped(both || pdl_on(), k_attn_chunk<D>, dim3(sms), dim3(PcCfg<D>::kThreads), PcCfg<D>::kSmem, st, a, kmap, vmap, cuts));
    if ((rc = launch_check("k_attn_chunk"))) return rc;
    IXB_GLUE("k_attn_chunk_join", launch_overlapped(true, k_attn_chunk_join<D>, dim3(sms, PcCfg<D>::kTiles * (D / 16)), dim3(128), 0, st, a, (const PcCut *)cuts));
}

extern "C" int ixb_attn_paged(const void *q, const void *k_pages, const void *v_pages, const int32_t *table, const int32_t *length,
                              const int32_t *cu_rows, void *out, int64_t requests, int64_t width, int64_t rows, int64_t max_q, int64_t hq,
                              int64_t hkv, int64_t head_dim, int64_t n_pages, int64_t page, int64_t q_stride, int64_t k_page_stride,
                              int64_t v_page_stride, float scale, void *scratch, size_t scratch_bytes, ixb_stream_t stream)
{
    if (!q || !k_pages || !v_pages || !table || !length || !cu_rows || !out || !scratch) return fail(IXB_E_ARG, "NULL pointer argument");
    int rc = page_shape(requests, width, n_pages, page);
    if (rc) return rc;
    if (hq <= 0 || hkv <= 0 || hq > 65535 || hq % hkv) return fail(IXB_E_ARG, "query heads must be a multiple of KV heads");
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) return fail(IXB_E_UNSUPPORTED, "head_dim=%lld: 64, 128 or 256", (long long)head_dim);
    if (rows <= 0 || rows > 0x7fffffffll / hq || max_q <= 0) return fail(IXB_E_ARG, "bad rows");
    if (rows * (hq / hkv) > 0xfffffff0ll / (hq / hkv)) return fail(IXB_E_UNSUPPORTED, "%lld rows of groups of %lld heads", (long long)rows, (long long)(hq / hkv));
    // The kernels add the costs of a KV head's work up in 32 bits: groups of at least eight rows, a table's width of blocks or tiles of 128
    // positions each, twice for two row tiles, and eight more for an end.  (All factors are below 2^32: no overflow here.)
    if ((double)(rows * (hq / hkv) / 8 + requests) * (double)(2 * (width * page / 128) + 8) >= 4294967296.0)
        return fail(IXB_E_UNSUPPORTED, "%lld rows and %lld requests behind tables of %lld positions are too much for one call", (long long)rows, (long long)requests,
                    (long long)(width * page));
    if (q_stride < hq * head_dim || (q_stride & 7) || k_page_stride < page * hkv * head_dim || v_page_stride < page * hkv * head_dim ||
        ((k_page_stride | v_page_stride) & 7))
        return fail(IXB_E_ARG, "bad strides");
    if (((uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)out | (uintptr_t)scratch) & 15u)
        return fail(IXB_E_ARG, "q, pages, output or scratch are not 16-byte aligned");
    if (num_sms() > (int)kPaMaxCtas || (size_t)num_sms() * sizeof(PcCut) > kPaCutBytes)
        return fail(IXB_E_UNSUPPORTED, "a device of %d SMs", num_sms());
    if (scratch_bytes < ixb_attn_paged_scratch_bytes(head_dim)) return fail(IXB_E_SCRATCH, "attention scratch too small");
    PagedAttn a = {};
    a.q = (const __nv_bfloat16 *)q;
    a.k = (const __nv_bfloat16 *)k_pages;
    a.v = (const __nv_bfloat16 *)v_pages;
    a.out = (__nv_bfloat16 *)out;
    a.table = table;
    a.length = length;
    a.cu_rows = cu_rows;
    a.tickets = (uint32_t *)scratch;
    a.part = (float *)((unsigned char *)scratch + kPaTicketBytes + kPaCutBytes);
    a.k_stride = (size_t)k_page_stride;
    a.v_stride = (size_t)v_page_stride;
    a.q_stride = (size_t)q_stride;
    a.requests = (uint32_t)requests;
    a.width = (uint32_t)width;
    a.n_pages = (uint32_t)n_pages;
    a.log_page = log_page(page);
    a.rows = (uint32_t)rows;
    a.hq = (uint32_t)hq;
    a.hkv = (uint32_t)hkv;
    a.group = (uint32_t)(hq / hkv);
    a.group_magic = (uint32_t)(((1ull << 32) + a.group - 1) / a.group);
    a.row_lo = 0;
    a.row_hi = 0xffffffffu;
    a.scale = scale;
    if (!(scale > 0.f && scale <= 3.4e38f)) return fail(IXB_E_ARG, "the scale must be positive and finite");
    PcCut *cuts = (PcCut *)((unsigned char *)scratch + kPaTicketBytes);
    const cudaStream_t st = (cudaStream_t)stream;
    return head_dim == 64 ? attn_paged_run<64>(a, cuts, max_q, st) : head_dim == 128 ? attn_paged_run<128>(a, cuts, max_q, st) : attn_paged_run<256>(a, cuts, max_q, st);
}

// ------------------------------------------------------------------------------------------------ rules on logits
template <class C, bool F32, bool VEC, int THREADS>
static cudaError_t launch_logits(const LogitRules &s, cudaStream_t st)
{
    static bool attr_set[64] = {false};
    const cudaError_t e = opt_in_smem(k_logits<C, F32, VEC, THREADS>, attr_set, 227 * 1024 - 1024);
    if (e != cudaSuccess) return e;
    return launch_glue_smem(k_logits<C, F32, VEC, THREADS>, dim3(s.rows * kLgCtas), dim3(THREADS),
                            s.history || s.n_bias ? s.slice * sizeof(C) + s.n_slots * 8u : 0, st, s);
}
template <class C, bool F32, bool VEC>
static cudaError_t launch_logits(const LogitRules &s, cudaStream_t st)
{
    // 512 threads while the rows' CTAs fit the chip once, two an SM: fewer vectors a thread (one row of 73448: 7.1 us, 8.1 with 256)
    return s.rows * kLgCtas <= 2u * num_sms() ? launch_logits<C, F32, VEC, 512>(s, st) : launch_logits<C, F32, VEC, 256>(s, st);
}
template <class C>
static cudaError_t launch_logits(const LogitRules &s, bool f32, bool vec, cudaStream_t st)
{
    return f32 ? (vec ? launch_logits<C, true, true>(s, st) : launch_logits<C, true, false>(s, st))
               : (vec ? launch_logits<C, false, true>(s, st) : launch_logits<C, false, false>(s, st));
}

extern "C" int ixb_logits(const void *logits, int logits_f32, int64_t pitch, const int32_t *history, int64_t hist_len, int64_t hist_pitch,
                          const int32_t *n_tokens, const int32_t *n_prompt, const float *repetition, const float *presence, const float *frequency,
                          const int32_t *bias_ids, const float *bias_values, int64_t n_bias, const void *mask, int64_t n_masks, int64_t mask_pitch,
                          const int32_t *mask_row, float *out, int64_t out_pitch, int64_t *token, int64_t rows, int64_t vocab, ixb_stream_t stream)
{
    if (!logits || !out || (history && !n_tokens) || (n_bias && (!bias_ids || !bias_values))) return fail(IXB_E_ARG, "NULL pointer argument");
    if (rows <= 0 || rows > 0x7fffffffll / kLgCtas || vocab <= 0) return fail(IXB_E_ARG, "bad shape");
    if (vocab > (int64_t)kLgMaxBins * kLgCtas) return fail(IXB_E_UNSUPPORTED, "vocabulary of %lld: at most %lld", (long long)vocab, (long long)kLgMaxBins * kLgCtas);
    if (pitch < vocab || out_pitch < vocab || (history && (hist_len < 0 || hist_pitch < hist_len)) || (mask && (n_masks <= 0 || mask_pitch < (vocab + 31) / 32)))
        return fail(IXB_E_ARG, "bad pitch");
    if (hist_len > kLgMaxTokens || hist_pitch > 0x7fffffffll || n_bias < 0 || n_bias > kLgMaxBias || n_masks > 0x7fffffffll || mask_pitch > 0x7fffffffll)
        return fail(IXB_E_UNSUPPORTED, "at most %lld tokens and %lld biases a row", (long long)kLgMaxTokens, (long long)kLgMaxBias);
    LogitRules s = {logits, history, n_tokens, n_prompt, repetition, presence, frequency, bias_ids, bias_values, (const uint32_t *)mask, mask_row,
                    out, (long long *)token, (size_t)pitch, (size_t)out_pitch, (uint32_t)rows, (uint32_t)vocab, 0, 0, (uint32_t)hist_len,
                    (uint32_t)hist_pitch, (uint32_t)n_bias, 0, (uint32_t)mask_pitch, (uint32_t)n_masks};
    for (uint32_t slots = 2; n_bias && s.n_slots < 2 * n_bias; slots *= 2) s.n_slots = slots;      // the table stays at most half full
    s.slice = (uint32_t)((vocab + 32 * kLgCtas - 1) / (32 * kLgCtas) * 32);
    if (s.slice > kLgMaxBins) return fail(IXB_E_UNSUPPORTED, "vocabulary of %lld is too large", (long long)vocab);
    s.hist_vec = ((uintptr_t)history & 15u) == 0 && (rows == 1 || (hist_pitch & 3) == 0);
    const cudaStream_t st = (cudaStream_t)stream;
    const bool vec = (((uintptr_t)logits | (uintptr_t)out) & 15u) == 0 && (rows == 1 || ((pitch & (logits_f32 ? 3 : 7)) == 0 && (out_pitch & 3) == 0));
    IXB_GLUE("k_logits", hist_len > kLgShortTokens ? launch_logits<uint32_t>(s, logits_f32, vec, st) : launch_logits<uint16_t>(s, logits_f32, vec, st));
}
