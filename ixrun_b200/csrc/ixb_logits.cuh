// What stands between a decoder's logits and its token: penalties for tokens that were seen, biases, grammar masks, arg-max.
//
//   x    = logits[b][v] in fp32
//   seen = v among the row's tokens (prompt and generated);  c = how often v was generated
//   x    = x > 0 ? x / repetition : x * repetition            where seen
//   x    = (x - frequency * c) - presence                     where c > 0
//   x    = x + bias                                           where a bias names v (of several, the last one)
//   x    = -inf                                               where the row's grammar has no bit for v
//   out[b][v] = x;  token[b] = the lowest v with the largest x (a NaN counts as the largest)
// Every step is rounded to fp32 by itself, in this order.
//
// A cluster of eight CTAs takes a row: each holds one eighth of the vocabulary as counters in shared memory, goes through the row's
// tokens and counts those that fall into its part, then streams its part of the logits once.  So the counts never touch memory, the
// arg-max of the parts meets through distributed shared memory, and nothing has to be zero between launches.
// Bound: HBM (a bf16 logit in, an fp32 one out, a bit of mask) for large batches, the chain of lengths, tokens, counters and logits
// for small ones: a thread's first logits are requested before anything else, the tokens before their number is known.  Counters
// of 16 bits (histories of up to 16383 tokens) let all CTAs of 64 rows of 151936 be there at once: 15.7 us without a rule (9 is
// the copy rate's time for their bytes), 18 with an empty history, 23 with 4000 tokens each, and 2 more with 300 biases.
// Built and slower: the history shared out over the cluster with remote counting (32 us for tokens as skewed as text's), the counted
// tokens taken from a list behind the stream (one more pass over scattered logits, 26 to 32 us).
#pragma once
#include "ixb_common.cuh"

namespace ixb {

constexpr int kLgCtas = 8;                             // of a cluster: one row
constexpr uint32_t kLgMaxBins = 49152;                 // of a CTA: 192 KB
// A counter: the top bit for a token of the prompt, the next one for a token that a bias names, the others count how often it was
// generated.  32-bit counters are for histories that 16-bit ones cannot count.
template <class C>
struct LgBits {
    static constexpr uint32_t kPrompt = 1u << (8 * sizeof(C) - 1), kBias = kPrompt >> 1, kCount = kBias - 1u;
};
constexpr int64_t kLgMaxBias = 2047, kLgMaxTokens = (1 << 20) - 1, kLgShortTokens = 16383;

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
    uint32_t rows, vocab, slice, hist_vec, hist_len, hist_pitch, n_bias, n_slots, mask_pitch, n_masks;       // n_slots: of the biases' table, a power of two
};

__device__ __forceinline__ unsigned long long lg_key(float x, uint32_t v)
{
    uint32_t b = __float_as_uint(x);
    b = x != x ? 0xffffffffu : b == 0x80000000u ? 0x80000000u : b >> 31 ? ~b : b | 0x80000000u;      // ordered as the numbers; -0 is 0
    return (unsigned long long)b << 32 | (0xffffffffu - v);
}

// A table of the row's biases for the tokens of this CTA's part: open addressing, (token + 1, its last entry: number, then value)
__device__ __forceinline__ void lg_put(uint2 *table, uint32_t mask, uint32_t token, uint32_t entry)
{
    for (uint32_t at = token * 2654435761u >> 7 & mask;; at = (at + 1u) & mask) {          // (at most half full)
        const uint32_t was = atomicCAS(&table[at].x, 0u, token + 1u);
        if (was == 0u || was == token + 1u) {
            atomicMax(&table[at].y, entry);
            return;
        }
    }
}
__device__ __forceinline__ uint2 &lg_at(uint2 *table, uint32_t mask, uint32_t token)        // (it is there)
{
    uint32_t at = token * 2654435761u >> 7 & mask;
    for (uint32_t i = 0; i < mask && table[at].x != token + 1u; ++i) at = (at + 1u) & mask;
    return table[at];
}
// NaN if one of them is
__device__ __forceinline__ float lg_max(float a, float b)
{
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}

// grid: rows x 8, clusters of 8, of 512 threads where that fills the chip once at most, else of 256.  VEC: rows of logits and out start on 16 bytes, eight logits at a time
template <class C, bool F32, bool VEC, int kLgThreads>
__global__ void __cluster_dims__(kLgCtas, 1, 1) __launch_bounds__(kLgThreads, 1024 / kLgThreads)
k_logits(LogitRules s)
{
    using B = LgBits<C>;
    extern __shared__ __align__(16) unsigned char lg_smem[];
    C *bins = (C *)lg_smem;                            // [slice], then the biases' table
    uint2 *table = (uint2 *)(bins + s.slice);
    __shared__ unsigned long long sm_key[kLgThreads / 32], sm_part[kLgCtas];
    const uint32_t tid = threadIdx.x, row = blockIdx.x / kLgCtas, me = blockIdx.x % kLgCtas;
    const uint32_t v0 = min(s.vocab, me * s.slice), v1 = min(s.vocab, v0 + s.slice), n = v1 - v0;
    asm volatile("griddepcontrol.launch_dependents;");
    if (s.token) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");      // (awaited before the first remote store)
    const bool count = s.history || s.n_bias;          // uniform
    constexpr uint32_t PV = 16 / sizeof(C);            // counters of 16 bytes
    if (count) {
        for (uint32_t i = PV * tid; i < n; i += PV * kLgThreads) *(uint4 *)(bins + i) = make_uint4(0, 0, 0, 0);      // (slice: a multiple of 32)
        for (uint32_t i = tid; i < s.n_slots; i += kLgThreads) table[i] = make_uint2(0, 0);
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    float *out = s.out + (size_t)row * s.out_pitch;
    const float *lf = (const float *)s.logits + (size_t)row * s.pitch;
    const __nv_bfloat16 *lb = (const __nv_bfloat16 *)s.logits + (size_t)row * s.pitch;
    constexpr int UN = F32 ? 2 : 4;                    // vectors of a thread in flight
    const uint32_t vec_end = VEC ? v0 + (n & ~7u) : v0;
    uint4 raw[UN][F32 ? 2 : 1];
    auto request = [&](uint32_t v) {
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const uint32_t at = v + u * 8u * kLgThreads;
            if (at >= vec_end) continue;
            if (F32) {
                raw[u][0] = __ldcs((const uint4 *)(lf + at));
                raw[u][F32 ? 1 : 0] = __ldcs((const uint4 *)(lf + at + 4));
            } else {
                raw[u][0] = __ldcs((const uint4 *)(lb + at));
            }
        }
    };
    if (VEC) request(v0 + 8u * tid);
    constexpr int HN = 4;                              // times four tokens of a thread in flight
    int4 id[HN];
    const int32_t *hist = s.history + (size_t)row * s.hist_pitch;
    auto tokens = [&](uint32_t i0) {
#pragma unroll
        for (int u = 0; u < HN; ++u) {
            const uint32_t i = i0 + u * 4u * kLgThreads;
            if (s.hist_vec && i + 3u < s.hist_len) {
                id[u] = *(const int4 *)(hist + i);
            } else {
                id[u].x = i < s.hist_len ? hist[i] : -1;
                id[u].y = i + 1u < s.hist_len ? hist[i + 1] : -1;
                id[u].z = i + 2u < s.hist_len ? hist[i + 2] : -1;
                id[u].w = i + 3u < s.hist_len ? hist[i + 3] : -1;
            }
        }
    };
    uint32_t len = 0, np = 0;
    if (s.history) {
        tokens(4u * tid);
        len = min((uint32_t)max(s.n_tokens[row], 0), s.hist_len);
        np = s.n_prompt ? min((uint32_t)max(s.n_prompt[row], 0), len) : 0u;
    }
    const float rep = s.repetition ? s.repetition[row] : 1.f, pres = s.presence ? s.presence[row] : 0.f,
                freq = s.frequency ? s.frequency[row] : 0.f;
    constexpr int BN = 2;                              // biases of a thread that are requested ahead
    const int32_t *bias_ids = s.bias_ids + (size_t)row * s.n_bias;
    const float *bias_values = s.bias_values + (size_t)row * s.n_bias;
    uint32_t b_id[BN];
    float b_val[BN];
#pragma unroll
    for (int u = 0; u < BN; ++u) {
        const uint32_t i = tid + u * kLgThreads;
        b_id[u] = i < s.n_bias ? (uint32_t)bias_ids[i] - v0 : 0xffffffffu;
        b_val[u] = i < s.n_bias ? bias_values[i] : 0.f;
    }
    const int32_t mr = !s.mask ? -1 : s.mask_row ? s.mask_row[row] : (int32_t)row;
    const uint32_t *mask = mr >= 0 && (uint32_t)mr < s.n_masks ? s.mask + (size_t)mr * s.mask_pitch : nullptr;
    auto mark = [&](uint32_t i, uint32_t bits, bool add) {             // in the word that holds counter i
        uint32_t *word = (uint32_t *)bins + i * sizeof(C) / 4;
        const uint32_t shift = sizeof(C) == 2 ? (i & 1u) * 16u : 0u;
        if (add) atomicAdd(word, bits << shift);
        else atomicOr(word, bits << shift);
    };
    if (count) __syncthreads();
    auto biases = [&](auto &&what) {                   // this thread's biases for tokens of this part: (token, number of the thread's, entry, value)
#pragma unroll
        for (int u = 0; u < BN; ++u)
            if (b_id[u] < n) what(b_id[u], (uint32_t)u, tid + u * kLgThreads, b_val[u]);
        for (uint32_t u = BN; tid + u * kLgThreads < s.n_bias; ++u) {
            const uint32_t b = (uint32_t)bias_ids[tid + u * kLgThreads] - v0;
            if (b < n) what(b, u, tid + u * kLgThreads, bias_values[tid + u * kLgThreads]);
        }
    };
    if (s.n_bias)
        biases([&](uint32_t b, uint32_t, uint32_t i, float) {
            mark(b, B::kBias, false);
            lg_put(table, s.n_slots - 1u, b, i);
        });
    if (s.history) {
        for (uint32_t i0 = 4u * tid; i0 < len; i0 += HN * 4u * kLgThreads) {
            if (i0 != 4u * tid) tokens(i0);
#pragma unroll
            for (int u = 0; u < HN; ++u) {
                const uint32_t i = i0 + u * 4u * kLgThreads;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t at = (uint32_t)(j == 0 ? id[u].x : j == 1 ? id[u].y : j == 2 ? id[u].z : id[u].w) - v0;
                    if (at < n && i + j < len) {       // (numbers outside the vocabulary fall into no part)
                        const bool made = i + j >= np;
                        mark(at, made ? 1u : B::kPrompt, made);
                    }
                }
            }
        }
    }
    if (count) __syncthreads();
    if (s.n_bias) {                                    // the last entries' values in the place of their numbers
        uint32_t last = 0;                             // (at most eight of a thread)
        biases([&](uint32_t b, uint32_t u, uint32_t i, float) { last |= (lg_at(table, s.n_slots - 1u, b).y == i ? 1u : 0u) << u; });
        __syncthreads();
        biases([&](uint32_t b, uint32_t u, uint32_t, float value) {
            if (last >> u & 1u) lg_at(table, s.n_slots - 1u, b).y = __float_as_uint(value);
        });
        __syncthreads();
    }
    // the logit behind its counter
    auto rules = [&](float x, uint32_t v, uint32_t bin) {
        const uint32_t c = bin & B::kCount;
        if (c || bin & B::kPrompt) x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
        if (c) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, (float)c)), pres);       // (zero times an infinite penalty would be NaN)
        if (bin & B::kBias) x = __fadd_rn(x, __uint_as_float(lg_at(table, s.n_slots - 1u, v - v0).y));
        return x;
    };
    float top = -INFINITY;
    const bool any = VEC && v0 + 8u * tid < vec_end ? true : vec_end + tid < v1;
    uint32_t top_v = VEC && v0 + 8u * tid < vec_end ? v0 + 8u * tid : vec_end + tid;        // the lowest of the thread's largest (its indices ascend)
    auto keep = [&](float x, uint32_t v) {
        if (x > top || (x != x && top == top)) {
            top = x;
            top_v = v;
        }
    };
    if (VEC) {
        for (uint32_t va = v0 + 8u * tid; va < vec_end; va += UN * 8u * kLgThreads) {
            if (va != v0 + 8u * tid) request(va);
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                const uint32_t v = va + u * 8u * kLgThreads;
                if (v >= vec_end) break;
                float x[8];
                if (F32) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint4 r = raw[u][F32 ? h : 0];
                        x[4 * h] = __uint_as_float(r.x); x[4 * h + 1] = __uint_as_float(r.y); x[4 * h + 2] = __uint_as_float(r.z); x[4 * h + 3] = __uint_as_float(r.w);
                    }
                } else {
                    const uint32_t w[4] = {raw[u][0].x, raw[u][0].y, raw[u][0].z, raw[u][0].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        x[2 * j] = __uint_as_float(w[j] << 16);
                        x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
                    }
                }
                if (count) {
                    uint32_t c[4 * sizeof(C) / 2], some = 0;
#pragma unroll
                    for (int q = 0; q < (int)sizeof(C) / 2; ++q) {
                        const uint4 r = *(const uint4 *)(bins + (v - v0) + q * 4);
                        c[4 * q] = r.x; c[4 * q + 1] = r.y; c[4 * q + 2] = r.z; c[4 * q + 3] = r.w;
                        some |= r.x | r.y | r.z | r.w;
                    }
                    if (some) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const uint32_t bin = sizeof(C) == 4 ? c[j % (4 * sizeof(C) / 2)] : j & 1 ? c[j / 2] >> 16 : c[j / 2] & 0xffffu;
                            if (bin) x[j] = rules(x[j], v + j, bin);
                        }
                    }
                }
                if (mask) {
                    const uint32_t bits = mask[v >> 5] >> (v & 31u);   // (v: a multiple of 8)
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = bits >> j & 1u ? x[j] : -INFINITY;
                }
                __stcs((float4 *)(out + v), make_float4(x[0], x[1], x[2], x[3]));
                __stcs((float4 *)(out + v + 4), make_float4(x[4], x[5], x[6], x[7]));
                const float m = lg_max(lg_max(lg_max(x[0], x[1]), lg_max(x[2], x[3])), lg_max(lg_max(x[4], x[5]), lg_max(x[6], x[7])));
                if (!(m <= top)) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) keep(x[j], v + j);
                }
            }
        }
    }
    constexpr int SN = 4;                              // single logits of a thread in flight
    for (uint32_t va = vec_end + tid; va < v1; va += SN * kLgThreads) {
        float x[SN];
#pragma unroll
        for (int u = 0; u < SN; ++u) {
            const uint32_t v = min(va + u * kLgThreads, v1 - 1u);
            x[u] = F32 ? lf[v] : __bfloat162float(lb[v]);
        }
#pragma unroll
        for (int u = 0; u < SN; ++u) {
            const uint32_t v = va + u * kLgThreads;
            if (v >= v1) break;
            const uint32_t bin = count ? bins[v - v0] : 0u;
            if (bin) x[u] = rules(x[u], v, bin);
            if (mask && !(mask[v >> 5] >> (v & 31u) & 1u)) x[u] = -INFINITY;
            out[v] = x[u];
            keep(x[u], v);
        }
    }
    if (!s.token) return;                              // uniform
    unsigned long long best = any ? lg_key(top, top_v) : 0ull;
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
