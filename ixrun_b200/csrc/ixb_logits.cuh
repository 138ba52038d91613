// What stands between a decoder's logits and its token: penalties for tokens that were seen, biases, grammar masks, arg-max.
//
//   x    = logits[b][v] in fp32
//   seen = v among the row's tokens (prompt and generated);  c = how often v was generated
//   x    = x > 0 ? x / repetition : x * repetition            where seen
//   x    = x - frequency * c,  then x - presence              where c > 0
//   x    = x + bias                                           where a bias names v (of several, the last one)
//   x    = -inf                                               where the row's grammar has no bit for v
//   out[b][v] = x;  token[b] = the lowest v with the largest x (a NaN counts as the largest)
// Every step is rounded to fp32 by itself, in this order.
//
// A cluster of eight CTAs takes a row: each holds one eighth of the vocabulary as 32-bit counters in shared memory, goes through the
// row's tokens and counts those that fall into its part, then streams its part of the logits once.  So the counts never touch
// memory, the arg-max of the parts meets through distributed shared memory, and nothing has to be zero between launches.
// Bound: HBM (a bf16 logit in, an fp32 one out, a bit of mask).
#pragma once
#include "ixb_common.cuh"

namespace ixb {

constexpr int kLgThreads = 512;
constexpr int kLgCtas = 8;                             // of a cluster: one row
constexpr uint32_t kLgMaxBins = 49152;                 // of a CTA: 192 KB
// a counter: bit 31 seen in the prompt, bits 20 .. 30 one more than the index of the bias entry, bits 0 .. 19 times generated
constexpr uint32_t kLgPrompt = 1u << 31, kLgCount = (1u << 20) - 1u;
constexpr int kLgBiasShift = 20;
constexpr int64_t kLgMaxBias = 2047, kLgMaxTokens = kLgCount;

struct LogitRules {
    const void *logits;
    const int32_t *history, *n_tokens, *n_prompt;      // history null: no penalties
    const float *repetition, *presence, *frequency;    // per row; null: 1, 0, 0
    const int32_t *bias_ids;
    const float *bias_values;
    const uint32_t *mask;
    const int32_t *mask_row;                           // null: row b has mask b
    float *out;
    long long *token;                                  // null: no arg-max
    size_t pitch, out_pitch;                           // elements
    uint32_t rows, vocab, slice, hist_len, hist_pitch, n_bias, words, mask_pitch, n_masks;
};

__device__ __forceinline__ unsigned long long lg_key(float x, uint32_t v)
{
    uint32_t b = __float_as_uint(x);
    b = x != x ? 0xffffffffu : b == 0x80000000u ? 0x80000000u : b >> 31 ? ~b : b | 0x80000000u;      // ordered as the numbers; -0 is 0
    return (unsigned long long)b << 32 | (0xffffffffu - v);
}

// a counter and what hangs on it: the logit after penalties and bias
__device__ __forceinline__ float lg_apply(float x, uint32_t bin, float rep, float pres, float freq, const float *bias)
{
    const uint32_t c = bin & kLgCount;
    if (c || bin & kLgPrompt) x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
    x = __fsub_rn(x, __fmul_rn(freq, (float)c));
    if (c) x = __fsub_rn(x, pres);
    const uint32_t e = bin >> kLgBiasShift & 2047u;
    if (e) x = __fadd_rn(x, bias[e - 1u]);
    return x;
}

// grid: rows x 8, clusters of 8.  VEC: rows of logits, out and mask start on 16 bytes (mask: 4), eight logits at a time
template <bool F32, bool VEC>
__global__ void __cluster_dims__(kLgCtas, 1, 1) __launch_bounds__(kLgThreads, 2)
k_logits(LogitRules s)
{
    extern __shared__ __align__(16) uint32_t lg_bins[];
    __shared__ unsigned long long sm_key[kLgThreads / 32], sm_part[kLgCtas];
    const uint32_t tid = threadIdx.x, row = blockIdx.x / kLgCtas, me = blockIdx.x % kLgCtas;
    const uint32_t v0 = min(s.vocab, me * s.slice), v1 = min(s.vocab, v0 + s.slice), n = v1 - v0;
    asm volatile("griddepcontrol.launch_dependents;");
    if (s.token) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");      // (awaited before the first remote store)
    const bool bins = s.history || s.n_bias;           // uniform
    if (bins)
        for (uint32_t i = 4u * tid; i < n; i += 4u * kLgThreads) *(uint4 *)(lg_bins + i) = make_uint4(0, 0, 0, 0);      // (slice: a multiple of 32)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const float rep = s.repetition ? s.repetition[row] : 1.f, pres = s.presence ? s.presence[row] : 0.f,
                freq = s.frequency ? s.frequency[row] : 0.f;
    const float *bias = s.n_bias ? s.bias_values + (size_t)row * s.n_bias : nullptr;
    if (bins) __syncthreads();
    if (s.n_bias) {
        for (uint32_t i = tid; i < s.n_bias; i += kLgThreads) {
            const uint32_t id = (uint32_t)s.bias_ids[(size_t)row * s.n_bias + i] - v0;
            if (id < n) atomicMax(lg_bins + id, (i + 1u) << kLgBiasShift);     // of several entries the last
        }
        __syncthreads();
    }
    if (s.history) {
        const uint32_t len = min((uint32_t)max(s.n_tokens[row], 0), s.hist_len), np = s.n_prompt ? min((uint32_t)max(s.n_prompt[row], 0), len) : 0u;
        const int32_t *h = s.history + (size_t)row * s.hist_pitch;
        constexpr int UN = 8;                          // tokens of a thread in flight
        for (uint32_t i0 = tid; i0 < len; i0 += UN * kLgThreads) {
            uint32_t id[UN];
#pragma unroll
            for (int u = 0; u < UN; ++u) id[u] = i0 + u * kLgThreads < len ? (uint32_t)h[i0 + u * kLgThreads] - v0 : 0xffffffffu;
#pragma unroll
            for (int u = 0; u < UN; ++u)
                if (id[u] < n) {                       // (also: numbers outside the vocabulary fall into no part)
                    if (i0 + u * kLgThreads < np) atomicOr(lg_bins + id[u], kLgPrompt);
                    else atomicAdd(lg_bins + id[u], 1u);
                }
        }
    }
    if (bins) __syncthreads();
    const int32_t mr = !s.mask ? -1 : s.mask_row ? s.mask_row[row] : (int32_t)row;
    const uint32_t *mask = mr >= 0 && (uint32_t)mr < s.n_masks ? s.mask + (size_t)mr * s.mask_pitch : nullptr;
    float *out = s.out + (size_t)row * s.out_pitch;
    const float *lf = (const float *)s.logits + (size_t)row * s.pitch;
    const __nv_bfloat16 *lb = (const __nv_bfloat16 *)s.logits + (size_t)row * s.pitch;
    unsigned long long best = 0;
    float top = -INFINITY;
    uint32_t top_v = v0;                               // of this thread: the lowest of its largest
    bool nan = false, any = false;
    auto finish = [&](float x, uint32_t v, bool allowed) {
        if (bins) {
            const uint32_t bin = lg_bins[v - v0];
            if (bin) x = lg_apply(x, bin, rep, pres, freq, bias);
        }
        if (!allowed) x = -INFINITY;
        if (!nan && (x > top || x != x || !any)) {     // (a thread's indices ascend)
            top = x;
            top_v = v;
            nan = x != x;
            any = true;
        }
        return x;
    };
    const uint32_t vec_end = VEC ? v0 + (n & ~7u) : v0;
    if (VEC) {
        for (uint32_t v = v0 + 8u * tid; v < vec_end; v += 8u * kLgThreads) {
            float x[8];
            if (F32) {
                const float4 a = __ldcs((const float4 *)(lf + v)), b = __ldcs((const float4 *)(lf + v + 4));
                x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
            } else {
                const uint4 a = __ldcs((const uint4 *)(lb + v));
                const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    x[2 * j] = __uint_as_float(w[j] << 16);
                    x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
                }
            }
            const uint32_t bits = mask ? mask[v >> 5] >> (v & 31u) : 0xffu;    // (v: a multiple of 8)
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = finish(x[j], v + j, bits >> j & 1u);
            *(float4 *)(out + v) = make_float4(x[0], x[1], x[2], x[3]);
            *(float4 *)(out + v + 4) = make_float4(x[4], x[5], x[6], x[7]);
        }
    }
    for (uint32_t v = vec_end + tid; v < v1; v += kLgThreads) {
        const float x = F32 ? lf[v] : __bfloat162float(lb[v]);
        out[v] = finish(x, v, !mask || mask[v >> 5] >> (v & 31u) & 1u);
    }
    if (!s.token) return;                              // uniform
    if (any) best = lg_key(top, top_v);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, d));
    if ((tid & 31u) == 0) sm_key[tid >> 5] = best;
    __syncthreads();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");        // every CTA of the cluster has begun
    if (tid < 32u) {
        best = tid < kLgThreads / 32 ? sm_key[tid] : 0ull;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, d));
        if (tid == 0) {                                // into the first CTA's shared memory
            uint32_t there;
            const uint32_t here = (uint32_t)__cvta_generic_to_shared(sm_part + me);
            asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(there) : "r"(here));
            asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(there), "l"(best) : "memory");
        }
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (me == 0 && tid == 0) {
        best = sm_part[0];
#pragma unroll
        for (int c = 1; c < kLgCtas; ++c) best = max(best, sm_part[c]);
        s.token[row] = (long long)(0xffffffffu - (uint32_t)best);
    }
}

}  // namespace ixb
