// logits_rules.cu — what a serving program does to a batch of logits before a token is chosen: a penalty for repeated tokens,
// frequency and presence penalties, biases, a grammar's mask.
//
// Per row, with `past` = how often a token occurs in the row's list and `made` = how often behind the first n_prompt of it:
//   x = past ? (x > 0 ? x / repeat : x * repeat) : x;   x -= frequency * made;   x -= made ? presence : 0;   x += bias;   masked: -inf
//
// Bound: HBM, 8 bytes a logit and a bit of mask, and close behind it the issue of instructions. A CTA takes a slice of a row's vocabulary
// and counts the row's list into a table of its slice in shared memory (integers: the order of the atomics does not show), then a
// thread applies the rules to the logits that it has held in registers meanwhile. Every CTA of a row reads the whole list, from L2, which
// is what long lists cost: 64 rows of 128256 with masks and lists of 300 ids 10.2 us, 2500 16.4, 8000 27, 32000 67 (all of them count; 1 x 32000: 2.0
// to 14.4). 64 rows of 128256, lists of up to 2500, masks, 64 biases: 13.9 us with x and out in L2, 10.3 at the copy rate of HBM; 17.6 with an
// id compared twice, the mask taken bit by bit and every entry tested by itself.
#include "cuda_shim.h"
#include "common.cuh"
#include "kv_pages.cuh"
#include "pdl.cuh"
#include "state.h"

#include <math_constants.h>

namespace tmc {
namespace {

constexpr uint32_t kThreads = 256, kWide = 4;                // threads of a CTA, logits of a load
constexpr uint32_t kPast = 1u << 31;        // occurs in the prompt; below it the number of times among the generated tokens

struct Rules {
    const int* tokens; const int* n_tokens; const int* n_prompt;
    const float* repeat; const float* presence; const float* frequency;
    const int* bias_ids; const float* bias; const int* n_bias;
    const uint32_t* mask;
    uint32_t tokens_ld, bias_ld, mask_ld;
};

// ITEMS loads per thread: a CTA's slice is ITEMS * 1024 logits. VEC: x and out rows lie alike against 16 bytes, and slices begin on
// such a boundary; else the same places are read one by one.
template <uint32_t ITEMS, bool VEC>
__global__ void __launch_bounds__(kThreads, 5) logits_rules_kernel(const float* x, size_t ldx, float* out, size_t ldo, uint32_t V, Rules r) {
    constexpr uint32_t SLICE = ITEMS * kThreads * kWide;
    __shared__ __align__(16) uint32_t table[SLICE];         // counts; then 1 + the place in the row's list of biases, 0: none
    __shared__ uint32_t words[SLICE / 32 + 2];
    const uint32_t b = blockIdx.y, tid = threadIdx.x;
    const float* xr = x + b * ldx;
    float* o = out + b * ldo;
    // logits [lo, lo + SLICE), of which those from 0 to V exist
    const int lo = (int)(blockIdx.x * SLICE) - (VEC ? (int)((uintptr_t)xr / sizeof(float) & (kWide - 1)) : 0);
    pdl_enter();
    if (lo >= (int)V) return;                               // a last slice that only another alignment of the row would have needed
    // The logits, the mask, the rules and the first 1024 of the row's list are on their way together; how many of the list count is
    // known only when they are there.
    constexpr uint32_t AHEAD = 4;
    const int* tokens = r.tokens + (size_t)b * r.tokens_ld;
    int id[AHEAD];
    if (r.tokens) {
#pragma unroll
        for (uint32_t k = 0; k < AHEAD; ++k) id[k] = tid + k * kThreads < r.tokens_ld ? tokens[tid + k * kThreads] : -1;
    }
    float v[ITEMS][kWide];
#pragma unroll
    for (uint32_t k = 0; k < ITEMS; ++k) {
        const int i = lo + (int)((k * kThreads + tid) * kWide);
        if (VEC && i >= 0 && i + (int)kWide <= (int)V) {
            const float4 f = *reinterpret_cast<const float4*>(xr + i);
            v[k][0] = f.x; v[k][1] = f.y; v[k][2] = f.z; v[k][3] = f.w;
        } else {
#pragma unroll
            for (uint32_t e = 0; e < kWide; ++e) v[k][e] = (uint32_t)(i + (int)e) < V ? xr[i + (int)e] : 0.f;
        }
    }
    // the slice's part of the vocabulary, as a range of the table: one comparison tells whether an id is in it
    const uint32_t t0 = (uint32_t)max(lo, 0), here = min((uint32_t)(lo + (int)SLICE), V) - t0, shift = t0 - (uint32_t)lo;
    const int w0 = lo >> 5, most = (int)((V + 31) / 32);
    if (r.mask)
        for (uint32_t i = tid; i < SLICE / 32 + 2; i += kThreads) words[i] = (uint32_t)(w0 + (int)i) < (uint32_t)most ? r.mask[(size_t)b * r.mask_ld + (uint32_t)(w0 + (int)i)] : 0u;
    const uint32_t listed = r.tokens ? (uint32_t)min(max(r.n_tokens[b], 0), (int)r.tokens_ld) : 0u;
    const uint32_t biases = r.bias ? (uint32_t)min(max(r.n_bias ? r.n_bias[b] : (int)r.bias_ld, 0), (int)r.bias_ld) : 0u;
    const int prompt = r.n_prompt ? r.n_prompt[b] : 0;
    const float repeat = r.repeat ? r.repeat[b] : 1.f, presence = r.presence ? r.presence[b] : 0.f, frequency = r.frequency ? r.frequency[b] : 0.f;
    for (uint32_t i = tid; i < SLICE / 4; i += kThreads) reinterpret_cast<uint4*>(table)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    if (listed) {
        for (uint32_t i0 = tid;;) {
#pragma unroll
            for (uint32_t k = 0; k < AHEAD; ++k) {
                const uint32_t i = i0 + k * kThreads, at = (uint32_t)id[k] - t0;
                if (at < here && i < listed) {
                    if ((int)i < prompt) atomicOr(&table[at + shift], kPast);
                    else atomicAdd(&table[at + shift], 1u);
                }
            }
            i0 += AHEAD * kThreads;
            if (i0 - tid >= listed) break;
#pragma unroll
            for (uint32_t k = 0; k < AHEAD; ++k) id[k] = i0 + k * kThreads < listed ? tokens[i0 + k * kThreads] : -1;
        }
        __syncthreads();
#pragma unroll
        for (uint32_t k = 0; k < ITEMS; ++k) {              // a thread reads, and clears for the biases, the entries of its own logits
            uint4* at = reinterpret_cast<uint4*>(table + (k * kThreads + tid) * kWide);
            const uint32_t c[kWide] = {at->x, at->y, at->z, at->w};
            if (!(c[0] | c[1] | c[2] | c[3])) continue;
            if (biases) *at = make_uint4(0, 0, 0, 0);
#pragma unroll
            for (uint32_t e = 0; e < kWide; ++e)
                if (c[e]) {
                    v[k][e] = v[k][e] > 0.f ? v[k][e] / repeat : v[k][e] * repeat;
                    const float made = (float)(c[e] & ~kPast);
                    if (made > 0.f) v[k][e] -= fmaf(frequency, made, presence);
                }
        }
    }
    if (biases) {
        __syncthreads();
        for (uint32_t i = tid; i < biases; i += kThreads) {
            const uint32_t at = (uint32_t)r.bias_ids[(size_t)b * r.bias_ld + i] - t0;
            if (at < here) atomicMax(&table[at + shift], i + 1);                       // of an id that is listed twice the last one counts
        }
        __syncthreads();
#pragma unroll
        for (uint32_t k = 0; k < ITEMS; ++k) {
            const uint4 c4 = *reinterpret_cast<const uint4*>(table + (k * kThreads + tid) * kWide);
            const uint32_t c[kWide] = {c4.x, c4.y, c4.z, c4.w};
            if (!(c[0] | c[1] | c[2] | c[3])) continue;
#pragma unroll
            for (uint32_t e = 0; e < kWide; ++e)
                if (c[e]) v[k][e] += r.bias[(size_t)b * r.bias_ld + c[e] - 1];
        }
    }
#pragma unroll
    for (uint32_t k = 0; k < ITEMS; ++k) {
        const int i = lo + (int)((k * kThreads + tid) * kWide);
        if (r.mask) {
            const uint32_t bit = (uint32_t)(i - w0 * 32), bits = __funnelshift_r(words[bit >> 5], words[(bit >> 5) + 1], bit & 31u);
#pragma unroll
            for (uint32_t e = 0; e < kWide; ++e) v[k][e] = bits >> e & 1u ? v[k][e] : -CUDART_INF_F;
        }
        if (VEC && i >= 0 && i + (int)kWide <= (int)V) *reinterpret_cast<float4*>(o + i) = make_float4(v[k][0], v[k][1], v[k][2], v[k][3]);
        else {
#pragma unroll
            for (uint32_t e = 0; e < kWide; ++e)
                if ((uint32_t)(i + (int)e) < V) o[i + (int)e] = v[k][e];
        }
    }
}

// Does a row of out share memory with a row of x, other than as itself? Rows whose ranges as a whole are apart are not walked.
bool rows_meet(const float* x, size_t ldx, const float* out, size_t ldo, unsigned B, unsigned V) {
    if (x == out && (B == 1 || ldx == ldo)) return false;
    if (!overlap(x, ((B - 1) * ldx + V) * sizeof(float), out, ((B - 1) * ldo + V) * sizeof(float))) return false;
    for (unsigned i = 0, k = 0; i < B && k < B;) {
        const uintptr_t a = (uintptr_t)(x + i * ldx), b = (uintptr_t)(out + k * ldo), n = (uintptr_t)V * sizeof(float);
        if (a + n <= b) ++i;
        else if (b + n <= a) ++k;
        else return true;
    }
    return false;
}

template <uint32_t ITEMS>
void go(const float* x, size_t ldx, float* out, size_t ldo, unsigned B, unsigned V, const Rules& r, cudaStream_t st) {
    constexpr uint32_t SLICE = ITEMS * kThreads * kWide;
    const bool vec = (uintptr_t)x % 16 == (uintptr_t)out % 16 && (B == 1 || ldx % kWide == ldo % kWide);
    const dim3 grid((unsigned)(((unsigned long long)V + (vec ? kWide - 1 : 0) + SLICE - 1) / SLICE), B);
    launch_overlapped(vec ? logits_rules_kernel<ITEMS, true> : logits_rules_kernel<ITEMS, false>, grid, dim3(kThreads), 0, st, x, ldx, out, ldo, V, r);
}

}  // namespace
}  // namespace tmc

using namespace tmc;

extern "C" bool tm_cuda_logits_rules_dev(const float* x, size_t ldx, float* out, size_t ldo, unsigned B, unsigned V,
                                         const tm_cuda_logit_rules* rules, void* stream) {
    if (!B) return true;
    if (!x || !out || !rules) return fail("logits_rules: null pointer");
    if (!V || V > 0x7fff0000u || B > 65535u || ldx < V || ldo < V) return fail("logits_rules: %u rows of %u logits in strides of %zu and %zu", B, V, ldx, ldo);
    if (rows_meet(x, ldx, out, ldo, B, V)) return fail("logits_rules: a row of out overlaps one of x that it is not");
    const tm_cuda_logit_rules& r = *rules;
    if (r.tokens && (!r.n_tokens || !r.tokens_ld || r.tokens_ld > 0x7fffffffu)) return fail("logits_rules: a token list without lengths or stride");
    if (!r.tokens && (r.repeat || r.presence || r.frequency)) return fail("logits_rules: penalties without a token list");
    if (r.bias && (!r.bias_ids || !r.bias_ld || r.bias_ld > 0x7fffffffu)) return fail("logits_rules: biases without ids or stride");
    if (r.mask && r.mask_ld < V / 32 + (V % 32 != 0)) return fail("logits_rules: a mask row of %u words for %u logits", r.mask_ld, V);
    if (((uintptr_t)x | (uintptr_t)out | (uintptr_t)r.tokens | (uintptr_t)r.n_tokens | (uintptr_t)r.n_prompt | (uintptr_t)r.repeat | (uintptr_t)r.presence | (uintptr_t)r.frequency |
         (uintptr_t)r.bias_ids | (uintptr_t)r.bias | (uintptr_t)r.n_bias | (uintptr_t)r.mask) % 4) return fail("logits_rules: every array lies on a 4-byte boundary");
    if (!on_library_device("logits_rules")) return false;
    const Rules k{r.tokens, r.n_tokens, r.n_prompt, r.repeat, r.presence, r.frequency, r.bias_ids, r.bias, r.n_bias, r.mask, r.tokens_ld, r.bias_ld, r.mask_ld};
    // Slices of 4096 read the lists a quarter as often, slices of 1024 spread a small batch over the SMs: 7 x 50257 takes 2.6 us with
    // 1024, 3.6 with 4096; 64 x 128256 22.6 and 13.9.
    if ((unsigned long long)B * V >= 148ull * 4096) go<4>(x, ldx, out, ldo, B, V, k, (cudaStream_t)stream);
    else go<1>(x, ldx, out, ldo, B, V, k, (cudaStream_t)stream);
    note_launch();
    return check_launch("logits_rules");
}
