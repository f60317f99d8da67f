// Control of float32 logits [rows, vocab] ahead of a draw: penalties for repeated tokens, biases, grammar masks.
//
// The rows row_start[b] .. row_start[b + 1] - 1 belong to request b.  For the logit x of token t in a row of it
//   seen      t is in the request's history, or on the row's path down a tree of drafted tokens
//   n         how often t was generated: in the history behind its first prompt_len tokens, and on the path
//   x = seen ? (x > 0 ? x / repetition : x * repetition) : x      (src/core/sampler/LLMSampler.cpp:21-34)
//   x = x - (frequency * n + (n > 0 ? presence : 0))
//   x = x + bias[t]                                               (-infinity: the token is never drawn)
//   x = -infinity where the row's grammar mask has no bit for t
// The logits are read once and written once; what is added to that traffic is the history, and a bit a token of a mask.
//
// A CTA takes a slice of the vocabulary for all rows of one request: it counts the history's tokens of its slice in shared
// memory (integers: in any order), once for all rows, and then streams the rows' slices.  The few tokens of a row's
// path and the few biased ones are put right behind that pass, by the same CTA.
#include "common.cuh"

namespace {

constexpr int NT = 256;
constexpr int MAX_NODES = 256;                       // of a request's tree
constexpr unsigned PROMPT = 0x80000000u;             // a count's top bit: seen in the prompt

struct ControlParams {
    const float* logits; float* out;
    int rows, vocab, slice;
    const int* row_start; const float* settings;     // settings [requests, 3]: repetition, frequency, presence
    const int* history; long long history_size; const int *history_start, *history_len, *prompt_len;
    const int* bias_start; const int* bias_tokens; const float* bias_values; int biases;
    const unsigned* mask; int mask_rows, mask_words; const int* mask_row;
    const int *parents, *tokens;
};

__device__ __forceinline__ float penalised(float x, unsigned count, unsigned more, float rep, float freq, float pres) {
    const unsigned n = (count & ~PROMPT) + more;
    if (count | more) x = x > 0.f ? x / rep : x * rep;
    return n ? x - (freq * (float)n + pres) : x;
}

__global__ void __launch_bounds__(NT) control_kernel(const ControlParams p) {
    extern __shared__ unsigned counts[];             // [slice]
    __shared__ short parent[MAX_NODES];
    __shared__ int token[MAX_NODES];
    pdl_launch_dependents();
    pdl_wait();
    const int b = blockIdx.y, lo = blockIdx.x * p.slice, hi = min(p.vocab, lo + p.slice);
    const int r0 = max(0, p.row_start[b]), r1 = min(p.rows, p.row_start[b + 1]);
    if (r0 >= r1) return;
    const float rep = p.settings[3 * b], freq = p.settings[3 * b + 1], pres = p.settings[3 * b + 2];
    const bool counted = rep != 1.f || freq != 0.f || pres != 0.f;
    const int nodes = p.parents ? min(r1 - r0, MAX_NODES) : 0;
    for (int i = threadIdx.x; i < hi - lo; i += NT) counts[i] = 0u;
    for (int i = threadIdx.x; i < nodes; i += NT) {
        const int up = __ldcg(p.parents + r0 + i);
        parent[i] = (short)(up < -1 || up >= i ? -2 : up);
        token[i] = __ldcg(p.tokens + r0 + i);
    }
    __syncthreads();
    if (counted) {
        const long long first = p.history_start[b];
        const long long len = first < 0 ? 0 : min((long long)p.history_len[b], p.history_size - first);
        const int prompt = p.prompt_len[b];
        for (int i = threadIdx.x; i < len; i += NT) {
            const int t = __ldcg(p.history + first + i);
            if (t >= lo && t < hi) {
                if (i < prompt) atomicOr(&counts[t - lo], PROMPT);
                else atomicAdd(&counts[t - lo], 1u);
            }
        }
        __syncthreads();
    }
    auto mask_of = [&](int r) -> const unsigned* {
        const int m = p.mask ? (p.mask_row ? __ldcg(p.mask_row + r) : r) : -1;
        return m >= 0 && m < p.mask_rows ? p.mask + (size_t)m * p.mask_words : nullptr;
    };
    auto allowed = [&](const unsigned* mask, int t) { return mask == nullptr || (__ldcg(mask + (t >> 5)) >> (t & 31) & 1u); };
    for (int r = r0; r < r1; ++r) {
        const float* in = p.logits + (size_t)r * p.vocab;
        float* to = p.out + (size_t)r * p.vocab;
        const unsigned* mask = mask_of(r);
        for (int t = lo + threadIdx.x; t < hi; t += NT) {
            const float x = penalised(__ldcg(in + t), counts[t - lo], 0u, rep, freq, pres);
            to[t] = allowed(mask, t) ? x : -INFINITY;
        }
    }
    if (nodes > 0 && counted) {
        __syncthreads();
        // the tokens of a node's path, a thread a node; one that is there more than once is done where the path has it first
        for (int i = threadIdx.x; i < nodes; i += NT) {
            int root = i;
            while (root >= 0) root = parent[root];
            if (root != -1) continue;                // padding, or a node behind it: no path
            const float* in = p.logits + (size_t)(r0 + i) * p.vocab;
            float* to = p.out + (size_t)(r0 + i) * p.vocab;
            const unsigned* mask = mask_of(r0 + i);
            for (int a = i; a >= 0; a = parent[a]) {
                const int t = token[a];
                if (t < lo || t >= hi) continue;
                unsigned more = 1;
                bool first = true;
                for (int o = i; o > a; o = parent[o]) first = first && token[o] != t;
                for (int o = parent[a]; o >= 0; o = parent[o]) more += token[o] == t;
                if (!first) continue;
                const float x = penalised(__ldcg(in + t), counts[t - lo], more, rep, freq, pres);
                to[t] = allowed(mask, t) ? x : -INFINITY;
            }
        }
    }
    if (p.bias_start) {
        __syncthreads();
        // ascending tokens: equal ones are neighbours, whose values the first of them adds in their order
        const int e0 = max(0, p.bias_start[b]), e1 = min(p.biases, p.bias_start[b + 1]);
        for (int e = e0 + threadIdx.x; e < e1; e += NT) {
            const int t = p.bias_tokens[e];
            if (t < lo || t >= hi || (e > e0 && p.bias_tokens[e - 1] == t)) continue;
            float bias = p.bias_values[e];
            for (int o = e + 1; o < e1 && p.bias_tokens[o] == t; ++o) bias += p.bias_values[o];
            for (int r = r0; r < r1; ++r) {
                float* to = p.out + (size_t)r * p.vocab + t;
                *to = bias == -INFINITY ? bias : *to + bias;
            }
        }
    }
}

}  // namespace

TFF_API int tff_control_logits(const float* logits, float* out, int rows, int vocab, int requests, const int* row_start,
                               const float* settings, const int* history, long long history_size, const int* history_start,
                               const int* history_len, const int* prompt_len, const int* bias_start, const int* bias_tokens,
                               const float* bias_values, int biases, const void* mask, int mask_rows, int mask_words,
                               const int* mask_row, const int* parents, const int* tokens, cudaStream_t stream) {
    if (rows <= 0 || requests <= 0) return TFF_OK;
    if (vocab <= 0 || requests > 65535 || !logits || !out || !row_start || !settings || !history_start || !history_len ||
        !prompt_len || (mask && (long long)mask_words * 32 < vocab) || (parents && (!tokens || out == logits)) ||
        (bias_start && biases > 0 && (!bias_tokens || !bias_values)))
        return TFF_ERR_BAD_ARGUMENT;
    ControlParams p;
    p.logits = logits; p.out = out; p.rows = rows; p.vocab = vocab;
    p.row_start = row_start; p.settings = settings;
    p.history = history; p.history_size = history ? history_size : 0;
    p.history_start = history_start; p.history_len = history_len; p.prompt_len = prompt_len;
    p.bias_start = bias_start; p.bias_tokens = bias_tokens; p.bias_values = bias_values; p.biases = biases;
    p.mask = (const unsigned*)mask; p.mask_rows = mask_rows; p.mask_words = mask_words; p.mask_row = mask_row;
    p.parents = parents; p.tokens = tokens;
    p.slice = 4096;
    return tff_launch_pdl(control_kernel, dim3((vocab + p.slice - 1) / p.slice, requests), dim3(NT), (size_t)p.slice * 4, stream, p);
}
