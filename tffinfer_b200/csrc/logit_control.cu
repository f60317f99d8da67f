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
// memory (integers: in any order), once for all rows, and then streams the rows' slices, four logits a load and four loads a
// thread on their way, of four rows where there are as many.  The few tokens of a row's path and the few biased ones are put right behind that pass, by the
// same CTA.  Where a mask allows none of a load's four tokens nothing is read.
#include "common.cuh"
#include "tma_host.h"

namespace {

constexpr int NT = 256, CTAS_AN_SM = 4;
constexpr int MAX_NODES = 256;                       // of a request's tree
constexpr int ROWS_AT_ONCE = 256;
constexpr int MOST_TOKENS = 16384, LEAST_TOKENS = 1024;        // of a slice: 32 KB of counts leave room for four CTAs an SM
constexpr int MASK_WORDS = 2048;                     // of masks in shared memory: a part of the rows' at a time

struct ControlParams {
    const float* logits; float* out;
    int rows, vocab, slice;
    const int* row_start; const float* settings;     // settings [requests, 3]: repetition, frequency, presence
    const int* history; long long history_size; const int *history_start, *history_len, *prompt_len;
    const int* bias_start; const int* bias_tokens; const float* bias_values; int biases;
    const unsigned* mask; int mask_rows, mask_words; const int* mask_row;
    const int *parents, *tokens;
};

// The tokens of a slice as counts: 16 bits a token while no count can pass 32,767, else 32 bits, of half as many tokens.  The top
// bit: seen in the prompt.
struct Counts {
    unsigned* words;
    bool wide;
    __device__ __forceinline__ void prompt(int i) {
        if (wide) atomicOr(words + i, 0x80000000u);
        else atomicOr(words + (i >> 1), 0x8000u << (i & 1) * 16);
    }
    __device__ __forceinline__ void add(int i) {
        if (wide) atomicAdd(words + i, 1u);
        else atomicAdd(words + (i >> 1), 1u << (i & 1) * 16);
    }
    // (a count's top bit as the top bit of 32)
    __device__ __forceinline__ unsigned at(int i) const {
        if (wide) return words[i];
        const unsigned c = reinterpret_cast<const unsigned short*>(words)[i];
        return (c & 0x8000u) << 16 | (c & 0x7fffu);
    }
};

// A request's penalties.  A positive logit is multiplied by 1 / repetition, rounded once for the request: a second rounding in
// float32 (2^-24) in place of a division, which with its branches took most of the kernel's instructions.
struct Penalties {
    float rep, inverse, freq, pres;
    // ``count`` as Counts gives it; ``more`` times on the row's path.  What was not seen keeps its bits.
    __device__ __forceinline__ float operator()(float x, unsigned count, unsigned more = 0u) const {
        const unsigned n = (count & 0x7fffffffu) + more;
        const float factor = (count | more) == 0u ? 1.f : x > 0.f ? inverse : rep;
        return x * factor - (n ? fmaf(freq, (float)n, pres) : 0.f);
    }
};

// VEC: logits and outputs lie alike within 16 bytes.
template <bool VEC>
__global__ void __launch_bounds__(NT, CTAS_AN_SM) control_kernel(const ControlParams p) {
    extern __shared__ unsigned count_words[];        // [slice / 2]
    __shared__ int mask_at[ROWS_AT_ONCE];
    __shared__ unsigned masks[MASK_WORDS];           // of a part of the rows: [row][words of the slice]
    __shared__ short hits[MAX_NODES];                // nodes whose tokens lie in the slice
    __shared__ int hit_count;
    __shared__ short parent[MAX_NODES];
    __shared__ int token[MAX_NODES];
    __shared__ int bias_range[2];                    // of the slice
    pdl_launch_dependents();
    pdl_wait();
    const int b = blockIdx.y;
    const int r0 = max(0, p.row_start[b]), r1 = min(p.rows, p.row_start[b + 1]);
    if (r0 >= r1) return;
    Penalties penalised;
    penalised.rep = p.settings[3 * b]; penalised.freq = p.settings[3 * b + 1]; penalised.pres = p.settings[3 * b + 2];
    penalised.inverse = 1.f / penalised.rep;
    const bool counted = penalised.rep != 1.f || penalised.freq != 0.f || penalised.pres != 0.f;
    const long long first_token = p.history_start[b];
    const int len = first_token < 0 ? 0 : (int)max(0ll, min((long long)p.history_len[b], p.history_size - first_token));
    const int prompt = p.prompt_len[b];
    Counts counts;
    counts.words = count_words;
    counts.wide = len > 32767;
    const int e0 = p.bias_start ? max(0, p.bias_start[b]) : 0, e1 = p.bias_start ? min(p.biases, p.bias_start[b + 1]) : 0;
    const bool biased = e0 < e1;
    const int nodes = p.parents && counted ? min(r1 - r0, MAX_NODES) : 0;
    for (int i = threadIdx.x; i < nodes; i += NT) {
        const int up = __ldcg(p.parents + r0 + i);
        parent[i] = (short)(up < -1 || up >= i ? -2 : up);
        token[i] = __ldcg(p.tokens + r0 + i);
    }
    auto allowed = [&](int m, int t) { return m < 0 || (__ldcg(p.mask + (size_t)m * p.mask_words + (t >> 5)) >> (t & 31) & 1u); };
    auto mask_of = [&](int r) {
        const int m = p.mask ? (p.mask_row ? __ldcg(p.mask_row + r) : r) : -1;
        return m < p.mask_rows ? m : -1;
    };
    const int end = min(p.vocab, (int)(blockIdx.x + 1) * p.slice), width = counts.wide ? p.slice / 2 : p.slice;
    for (int lo = blockIdx.x * p.slice; lo < end; lo += width) {
        const int hi = min(end, lo + width);
        __syncthreads();                             // (the part before is through with the counts)
        if (counted) {
            for (int i = threadIdx.x; i < p.slice / 2; i += NT) count_words[i] = 0u;
            __syncthreads();
            for (int i0 = threadIdx.x; i0 < len; i0 += 8 * NT) {
                int t[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) t[u] = i0 + u * NT < len ? __ldcg(p.history + first_token + i0 + u * NT) : -1;
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    if (t[u] < lo || t[u] >= hi) continue;
                    if (i0 + u * NT < prompt) counts.prompt(t[u] - lo);
                    else counts.add(t[u] - lo);
                }
            }
        }
        // the biases of the slice: a run of the request's
        if (threadIdx.x == 0) { bias_range[0] = e1; bias_range[1] = e0; hit_count = 0; }
        __syncthreads();
        for (int e = e0 + threadIdx.x; e < e1; e += NT) {
            const int t = p.bias_tokens[e];
            if (t >= lo && t < hi) { atomicMin(&bias_range[0], e); atomicMax(&bias_range[1], e + 1); }
        }
        for (int i = threadIdx.x; i < nodes; i += NT)
            if (token[i] >= lo && token[i] < hi) hits[atomicAdd(&hit_count, 1)] = (short)i;
        const int w0 = lo >> 5, words = ((hi - 1) >> 5) - w0 + 1;
        const int at_once = p.mask ? min(ROWS_AT_ONCE, MASK_WORDS / words) : ROWS_AT_ONCE;
        for (int c0 = r0; c0 < r1; c0 += at_once) {
            const int rows = min(at_once, r1 - c0);
            if (c0 > r0) __syncthreads();
            for (int i = threadIdx.x; i < rows; i += NT) mask_at[i] = mask_of(c0 + i);
            __syncthreads();
            if (p.mask) {
                for (int i = threadIdx.x; i < rows * words; i += NT) {
                    const int m = mask_at[i / words];
                    masks[i] = m < 0 ? 0xffffffffu : __ldcg(p.mask + (size_t)m * p.mask_words + w0 + i % words);
                }
                __syncthreads();
            }
            auto allowed_here = [&](int row, int t) { return !p.mask || (masks[row * words + (t >> 5) - w0] >> (t & 31) & 1u); };
            auto one = [&](int row, int t) {
                const size_t at = (size_t)(c0 + row) * p.vocab + t;
                const float x = __ldcg(p.logits + at);
                p.out[at] = allowed_here(row, t) ? penalised(x, counted ? counts.at(t - lo) : 0u) : -INFINITY;
            };
            if (!VEC) {
                for (int row = 0; row < rows; ++row)
                    for (int t = lo + threadIdx.x; t < hi; t += NT) one(row, t);
                continue;
            }
            // tokens ahead of a row's first aligned four: the same for every fourth row, and for all where vocab is a multiple of 4
            auto skip = [&](int row) {
                return (int)((4 - (((uintptr_t)p.logits >> 2) + (size_t)(c0 + row) * p.vocab + lo)) & 3);
            };
            const int step = p.vocab & 3 ? 4 : 1;
            for (int like = 0; like < min(step, rows); ++like) {
                const int s0 = lo + skip(like), fours = (hi - s0) / 4, alike = (rows - like + step - 1) / step;
                auto from = [&](int n) { return p.logits + (size_t)(c0 + like + n * step) * p.vocab; };
                auto bits_of = [&](int n, int t) -> unsigned {
                    if (!p.mask) return 15u;
                    const unsigned* w = masks + (like + n * step) * words + (t >> 5) - w0;
                    const unsigned low = w[0], high = (t & 31) > 28 ? w[1] : 0u;
                    return __funnelshift_r(low, high, t & 31) & 15u;
                };
                auto finish = [&](float4 x, unsigned bits, int n, int t, const unsigned (&c)[4], bool any) {
                    if (any) {
                        x.x = penalised(x.x, c[0]);
                        x.y = penalised(x.y, c[1]);
                        x.z = penalised(x.z, c[2]);
                        x.w = penalised(x.w, c[3]);
                    }
                    if (bits != 15u) {
                        if (!(bits & 1u)) x.x = -INFINITY;
                        if (!(bits & 2u)) x.y = -INFINITY;
                        if (!(bits & 4u)) x.z = -INFINITY;
                        if (!(bits & 8u)) x.w = -INFINITY;
                    }
                    *reinterpret_cast<float4*>(p.out + (size_t)(c0 + like + n * step) * p.vocab + t) = x;
                };
                auto counts_of = [&](int t, unsigned (&c)[4]) -> bool {
                    if (!counted) return false;
                    const int i = t - lo;
                    if (!counts.wide && (i & 3) == 0) {
                        const uint2 w = *reinterpret_cast<const uint2*>(count_words + i / 2);
                        if ((w.x | w.y) == 0u) return false;
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) c[e] = counts.at(i + e);
                    return (c[0] | c[1] | c[2] | c[3]) != 0u;
                };
                if (alike > 1) {                     // four rows' loads of a thread's four tokens together
                    const int parts = (alike + 3) / 4;
                    for (int i = threadIdx.x; i < fours * parts; i += NT) {
                        const int part = i / fours, t = s0 + 4 * (i - part * fours), n0 = 4 * part;
                        float4 x[4];
                        unsigned bits[4];
#pragma unroll
                        for (int u = 0; u < 4; ++u) bits[u] = n0 + u < alike ? bits_of(n0 + u, t) : 0u;
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (bits[u]) x[u] = __ldcg(reinterpret_cast<const float4*>(from(n0 + u) + t));
                        }
                        unsigned c[4] = {0u, 0u, 0u, 0u};
                        const bool any = counts_of(t, c);
#pragma unroll
                        for (int u = 0; u < 4; ++u) if (n0 + u < alike) finish(x[u], bits[u], n0 + u, t, c, any);
                    }
                } else {                             // one row: a thread's loads of four fours
                    for (int k0 = threadIdx.x; k0 < fours; k0 += 4 * NT) {
                        float4 x[4];
                        unsigned bits[4];
#pragma unroll
                        for (int u = 0; u < 4; ++u) bits[u] = k0 + u * NT < fours ? bits_of(0, s0 + 4 * (k0 + u * NT)) : 0u;
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (bits[u]) x[u] = __ldcg(reinterpret_cast<const float4*>(from(0) + s0 + 4 * (k0 + u * NT)));
                        }
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            if (k0 + u * NT >= fours) continue;
                            const int t = s0 + 4 * (k0 + u * NT);
                            unsigned c[4] = {0u, 0u, 0u, 0u};
                            const bool any = counts_of(t, c);
                            finish(x[u], bits[u], 0, t, c, any);
                        }
                    }
                }
            }
            // the up to three tokens of a row ahead of its fours, and those behind
            for (int i = threadIdx.x; i < rows * 6; i += NT) {
                const int row = i / 6, e = i % 6, s = skip(row), left = (hi - lo - s) & 3;
                if (hi - lo < s) {                   // (a slice of fewer tokens than that)
                    if (e < hi - lo) one(row, lo + e);
                } else if (e < 3 ? e < s : e - 3 < left) {
                    one(row, e < 3 ? lo + e : hi - left + e - 3);
                }
            }
        }
        if (nodes > 0) {
            __syncthreads();
            // a thread a node of the slice's and a node that may have it on its path; a token that is there more than once is done where
            // the path has it first, for all of them
            for (int i = threadIdx.x; i < hit_count * nodes; i += NT) {
                const int a = hits[i / nodes], node = i % nodes, t = token[a];
                int o = node;
                bool first = true;
                while (o > a) { first = first && token[o] != t; o = parent[o]; }
                if (o != a || !first) continue;
                unsigned more = 1;
                for (o = parent[a]; o >= 0; o = parent[o]) more += token[o] == t;
                if (o != -1) continue;               // padding, or a node behind it: no path
                const size_t at = (size_t)(r0 + node) * p.vocab + t;
                const float x = penalised(__ldcg(p.logits + at), counts.at(t - lo), more);
                p.out[at] = allowed(mask_of(r0 + node), t) ? x : -INFINITY;
            }
        }
        if (biased) {
            __syncthreads();
            // ascending tokens: equal ones are neighbours, whose values the first of them adds in their order
            const int f0 = bias_range[0], f1 = bias_range[1], n = r1 - r0;
            for (long long i = threadIdx.x; i < (long long)(f1 - f0) * n; i += NT) {
                const int e = f0 + (int)(i / n), r = r0 + (int)(i % n);
                const int t = p.bias_tokens[e];
                if (t < lo || t >= hi || (e > e0 && p.bias_tokens[e - 1] == t)) continue;
                float bias = p.bias_values[e];
                for (int o = e + 1; o < e1 && p.bias_tokens[o] == t; ++o) bias += p.bias_values[o];
                float* to = p.out + (size_t)r * p.vocab + t;
                *to = bias == -INFINITY ? bias : *to + bias;
            }
        }
    }
}

// Tokens of a slice: as many slices a request as fill whole waves of four CTAs an SM, of few tokens where there are few
// requests.
int slice_tokens(int vocab, int requests, int sms) {
    const long long slots = (long long)CTAS_AN_SM * (sms > 0 ? sms : 1);
    for (int wave = 1;; ++wave) {
        const long long slices = wave * slots / requests;
        if (slices < 1) continue;
        const long long tokens = ((vocab + slices - 1) / slices + 7) / 8 * 8;
        if (tokens <= MOST_TOKENS) return (int)(tokens < LEAST_TOKENS ? LEAST_TOKENS : tokens);
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
    p.slice = slice_tokens(vocab, requests, tff_num_sms());
    const dim3 grid((vocab + p.slice - 1) / p.slice, requests);
    const size_t smem = (size_t)p.slice * 2;
    if ((((uintptr_t)logits ^ (uintptr_t)out) & 15) == 0) return tff_launch_pdl(control_kernel<true>, grid, dim3(NT), smem, stream, p);
    return tff_launch_pdl(control_kernel<false>, grid, dim3(NT), smem, stream, p);
}
