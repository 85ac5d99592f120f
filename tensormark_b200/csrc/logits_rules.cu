// logits_rules.cu — what a serving program does to a batch of logits before a token is chosen: a penalty for repeated tokens,
// frequency and presence penalties, biases, a grammar's mask.
//
// Per row, with `past` = how often a token occurs in the row's list and `made` = how often behind the first n_prompt of it:
//   x = past ? (x > 0 ? x / repeat : x * repeat) : x;   x -= frequency * made;   x -= made ? presence : 0;   x += bias;   masked: -inf
//
// Bound: HBM, 8 bytes a logit and a bit of mask. A CTA takes a slice of a row's vocabulary and counts the row's list into a table of
// its slice in shared memory (integers: the order of the atomics does not show), then streams the slice once. Every CTA of a row
// reads the whole list, which is short against the slices and comes from L2.
#include "cuda_shim.h"
#include "common.cuh"
#include "kv_pages.cuh"
#include "state.h"

#include <math_constants.h>

namespace tmc {
namespace {

constexpr uint32_t kSlice = 4096;           // entries of a CTA: 16 KB of counts and as much for the biases, six CTAs per SM
constexpr uint32_t kThreads = 256;
constexpr uint32_t kPast = 1u << 31;        // occurs in the prompt; below it the number of times among the generated tokens

struct Rules {
    const int* tokens; const int* n_tokens; const int* n_prompt;
    const float* repeat; const float* presence; const float* frequency;
    const int* bias_ids; const float* bias; const int* n_bias;
    const uint32_t* mask;
    uint32_t tokens_ld, bias_ld, mask_ld;
};

__global__ void __launch_bounds__(kThreads) logits_rules_kernel(const float* x, size_t ldx, float* out, size_t ldo, uint32_t V, Rules r) {
    __shared__ uint32_t count[kSlice];
    __shared__ uint32_t bias_at[kSlice];    // 1 + the place in the row's list of biases, 0: none
    const uint32_t b = blockIdx.y, lo = blockIdx.x * kSlice, n = min(kSlice, V - lo);
    const uint32_t listed = r.tokens ? (uint32_t)min(max(r.n_tokens[b], 0), (int)r.tokens_ld) : 0u;
    const uint32_t biases = r.bias ? (uint32_t)min(max(r.n_bias ? r.n_bias[b] : (int)r.bias_ld, 0), (int)r.bias_ld) : 0u;
    const int prompt = r.n_prompt ? r.n_prompt[b] : 0;
    if (listed) for (uint32_t i = threadIdx.x; i < n; i += kThreads) count[i] = 0;
    if (biases) for (uint32_t i = threadIdx.x; i < n; i += kThreads) bias_at[i] = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < listed; i += kThreads) {
        const uint32_t at = (uint32_t)r.tokens[(size_t)b * r.tokens_ld + i] - lo;     // ids outside the vocabulary are in no slice
        if (at < n) {
            if ((int)i < prompt) atomicOr(&count[at], kPast);
            else atomicAdd(&count[at], 1u);
        }
    }
    for (uint32_t i = threadIdx.x; i < biases; i += kThreads) {
        const uint32_t at = (uint32_t)r.bias_ids[(size_t)b * r.bias_ld + i] - lo;
        if (at < n) atomicMax(&bias_at[at], i + 1);                                   // of an id that is listed twice the last one counts
    }
    __syncthreads();
    const float repeat = r.repeat ? r.repeat[b] : 1.f, presence = r.presence ? r.presence[b] : 0.f, frequency = r.frequency ? r.frequency[b] : 0.f;
    const float* xr = x + b * ldx + lo;
    float* o = out + b * ldo + lo;
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
        float v = xr[i];
        if (listed) {
            const uint32_t c = count[i];
            if (c) {
                v = v > 0.f ? v / repeat : v * repeat;
                const float made = (float)(c & ~kPast);
                if (made > 0.f) v -= fmaf(frequency, made, presence);
            }
        }
        if (biases && bias_at[i]) v += r.bias[(size_t)b * r.bias_ld + bias_at[i] - 1];
        if (r.mask && !(r.mask[(size_t)b * r.mask_ld + ((lo + i) >> 5)] >> ((lo + i) & 31u) & 1u)) v = -CUDART_INF_F;
        o[i] = v;
    }
}

}  // namespace
}  // namespace tmc

using namespace tmc;

extern "C" bool tm_cuda_logits_rules_dev(const float* x, size_t ldx, float* out, size_t ldo, unsigned B, unsigned V,
                                         const tm_cuda_logit_rules* rules, void* stream) {
    if (!x || !out || !rules) return fail("logits_rules: null pointer");
    if (!V || V > 0x7fffffffu || B > 65535u || ldx < V || ldo < V) return fail("logits_rules: %u rows of %u logits in strides of %zu and %zu", B, V, ldx, ldo);
    const tm_cuda_logit_rules& r = *rules;
    if (r.tokens && (!r.n_tokens || !r.tokens_ld || r.tokens_ld > 0x7fffffffu)) return fail("logits_rules: a token list without lengths or stride");
    if (!r.tokens && (r.repeat || r.presence || r.frequency)) return fail("logits_rules: penalties without a token list");
    if (r.bias && (!r.bias_ids || !r.bias_ld || r.bias_ld > 0x7fffffffu)) return fail("logits_rules: biases without ids or stride");
    if (r.mask && r.mask_ld < V / 32 + (V % 32 != 0)) return fail("logits_rules: a mask row of %u words for %u logits", r.mask_ld, V);
    if (!on_library_device("logits_rules")) return false;
    if (!B) return true;
    const Rules k{r.tokens, r.n_tokens, r.n_prompt, r.repeat, r.presence, r.frequency, r.bias_ids, r.bias, r.n_bias, r.mask, r.tokens_ld, r.bias_ld, r.mask_ld};
    logits_rules_kernel<<<dim3(V / kSlice + (V % kSlice != 0), B), kThreads, 0, (cudaStream_t)stream>>>(x, ldx, out, ldo, V, k);
    note_launch();
    return check_launch("logits_rules");
}
