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
// thread on their way, of four rows where there are as many.  The few tokens of a row's path and the few biased ones are put right
// behind that pass.  Where a mask allows none of a load's four tokens nothing is read.
//
// What bounds it beside the traffic: instructions, and the warps that hide the way to memory.  A thread's addresses are a pointer and
// an offset, and what a count does to a logit is worked out once for four rows, and not at all where none of a thread's four tokens was
// seen (looked up and divided for every logit, 140 to 230 instructions for a warp's 128 of them, 256 rows of trees took 62 us and 64
// rows 30; as it was then).  Measured at a vocabulary of 151,936 with masks and 200 to 6,000 tokens of history: 64 rows 26.9 us (78 MB, 2.9
// TB/s; a plain pass over as many bytes 13.4: the rest is what comes ahead of the first logits, 11,000 cycles of loads that wait for
// one another, and the quotients), the 256 nodes of eight trees 62 (4.9 TB/s; 47), one row without a mask 5.3.  The comparisons below are from before the
// quotients were rounded once, with 24.9 and 56.
//   Four CTAs an SM; with three, and larger slices, 29 and 62.  Tried without gain (64 rows, 256 nodes): the next loads ahead of a
//   thread's work, 32 and 71 (registers for three CTAs an SM); a branch for each of a thread's tokens, 28 and 58; counted tokens put right behind a
//   pass that only copies, 34 and 98; parts of rows by bulk copies through shared memory, 41 and 75 (half the instructions, too few warps).
#include "common.cuh"
#include "tma_host.h"

namespace {

constexpr int NT = 256, CTAS_AN_SM = 4;
constexpr int NODES = 256;                           // of a request's tree in shared memory: a larger one's others are read where they lie
constexpr int ROWS_AT_ONCE = 256;
constexpr int MOST_TOKENS = 17408, LEAST_TOKENS = 1024;        // of a slice: 34 KB of counts beside the rest's 20 leave room for four CTAs an SM
constexpr int MASK_WORDS = 2304;                     // of masks in shared memory: a part of the rows' at a time

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
    __device__ __forceinline__ void add(int i, bool prompt) const {
        if (wide) {
            if (prompt) atomicOr(words + i, 0x80000000u);
            else atomicAdd(words + i, 1u);
        } else {
            const int shift = (i & 1) * 16;
            if (prompt) atomicOr(words + (i >> 1), 0x8000u << shift);
            else atomicAdd(words + (i >> 1), 1u << shift);
        }
    }
    // (a count's top bit as the top bit of 32)
    __device__ __forceinline__ unsigned at(int i) const {
        if (wide) return words[i];
        const unsigned c = reinterpret_cast<const unsigned short*>(words)[i];
        return (c & 0x8000u) << 16 | (c & 0x7fffu);
    }
};

// Logits that are divided without the division's own instructions: from 2^-64 to 2^64, by penalties of 2^-32 to 2^32.
constexpr unsigned LEAST_QUICK = 0x1f800000u, QUICK = 0x5f800000u - LEAST_QUICK;
__device__ __noinline__ float divided(float x, float by) { return x / by; }

// A request's penalties, with the operations of repetition_penalty_kernel (sampling.cu): a request's logits are the same, bit by bit,
// whichever of the two kernels its step takes.  A quotient rounded once, at two products more than x * (1 / repetition) takes: with the
// reciprocal y rounded to nearest, q = x y and the remainder r = x - q repetition, q + r y is x / repetition rounded to nearest (after
// P. Markstein, Computation of elementary functions on the IBM RISC System/6000, 1990; compared with the division for all 2^46 pairs of
// significands) where nothing over- or underflows.  When it was brought in: 64 rows 27.5 us, the nodes of eight trees 64.5; with a
// division for every such logit 28.1 and 72, with x y alone, a rounding more, 24.9 and 56.
struct Penalties {
    float rep, inverse, freq, pres;
    unsigned quick;                                  // QUICK, or 0: this penalty is divided by
    // What is added to the logit of a token with this count (as Counts gives it): -0, which leaves all bits, where it was not generated.
    __device__ __forceinline__ float less(unsigned count) const {
        const unsigned n = count & 0x7fffffffu;
        return n ? -fmaf(freq, (float)n, pres) : -0.f;
    }
    __device__ __forceinline__ float apply(float x, bool seen, float less_) const {
        const float q = x * inverse, quotient = fmaf(fmaf(-q, rep, x), inverse, q);
        const bool in = __float_as_uint(x) - LEAST_QUICK < quick;
        float y = in ? quotient : x * rep;
        if (!in && x > 0.f) y = divided(x, rep);
        return (seen ? y : x) + less_;
    }
    // ``more`` times on the row's path.
    __device__ __forceinline__ float operator()(float x, unsigned count, unsigned more = 0u) const {
        return apply(x, (count | more) != 0u, less((count & 0x7fffffffu) + more));
    }
};

// VEC: logits and outputs lie alike within 16 bytes.
template <bool VEC>
__global__ void __launch_bounds__(NT, CTAS_AN_SM) control_kernel(const ControlParams p) {
    extern __shared__ unsigned count_words[];        // [slice / 2]
    __shared__ int mask_at[ROWS_AT_ONCE];
    __shared__ unsigned masks[MASK_WORDS];           // of a part of the rows: [row][words of the slice]
    __shared__ short parent[NODES];
    __shared__ int token[NODES];
    __shared__ unsigned short lists[NT / 32][512];   // a warp's tokens of the slice: their places, and a bit for the prompt's
    __shared__ short hits[NODES];                    // nodes whose tokens lie in the slice, of NODES at a time
    __shared__ int hit_count, bias_range[2];
    __shared__ int own[10];                          // the request's: rows, penalties, history, biases
    pdl_launch_dependents();
    pdl_wait();
    const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
    // A lane each, once a CTA: all CTAs ask the same few lines for them (read by every warp, 64 requests' took 7,400 cycles).
    if (tid < 10) {
        const int* at = tid < 2 ? p.row_start + b + tid : tid < 5 ? reinterpret_cast<const int*>(p.settings) + 3 * b + tid - 2 : tid == 5 ? p.history_start + b
                      : tid == 6 ? p.history_len + b : tid == 7 ? p.prompt_len + b : p.bias_start ? p.bias_start + b + tid - 8 : nullptr;
        own[tid] = at ? __ldcg(at) : 0;
    }
    __syncthreads();
    const int r0 = max(0, own[0]), r1 = min(p.rows, own[1]);
    Penalties penalised;
    penalised.rep = __int_as_float(own[2]); penalised.freq = __int_as_float(own[3]); penalised.pres = __int_as_float(own[4]);
    const long long first_token = own[5], held = own[6];
    const int prompt = own[7], e0 = max(0, own[8]), e1 = min(p.biases, own[9]);
    if (r0 >= r1) return;
    penalised.inverse = 1.f / penalised.rep;
    penalised.quick = penalised.rep >= 0x1p-32f && penalised.rep <= 0x1p32f ? QUICK : 0u;
    const bool counted = penalised.rep != 1.f || penalised.freq != 0.f || penalised.pres != 0.f;
    const int len = !counted || first_token < 0 ? 0 : (int)max(0ll, min(held, p.history_size - first_token));
    Counts counts;
    counts.words = count_words;
    counts.wide = len > 32767;
    const int nodes = p.parents && counted ? r1 - r0 : 0;
    auto parent_at = [&](int i) -> int {
        const int up = __ldcg(p.parents + r0 + i);
        return up < -1 || up >= i ? -2 : up;
    };
    for (int i = tid; i < min(nodes, NODES); i += NT) {
        parent[i] = (short)parent_at(i);
        token[i] = __ldcg(p.tokens + r0 + i);
    }
    auto parent_of = [&](int i) -> int { return i < NODES ? parent[i] : parent_at(i); };
    auto token_of = [&](int i) { return i < NODES ? token[i] : __ldcg(p.tokens + r0 + i); };
    auto mask_of = [&](int r) {
        const int m = p.mask ? (p.mask_row ? __ldcg(p.mask_row + r) : r) : -1;
        return m < p.mask_rows ? m : -1;
    };
    auto allowed = [&](int r, int t) {
        const int m = mask_of(r);
        return m < 0 || (__ldcg(p.mask + (size_t)m * p.mask_words + (t >> 5)) >> (t & 31) & 1u);
    };
    const int end = min(p.vocab, (int)(blockIdx.x + 1) * p.slice), width = counts.wide ? p.slice / 2 : p.slice;
    for (int lo = blockIdx.x * p.slice; lo < end; lo += width) {
        const int hi = min(end, lo + width);
        const int w0 = lo >> 5, words = ((hi - 1) >> 5) - w0 + 1;
        // rows at a time: in equal parts, of whole fours
        const int most = p.mask ? min(ROWS_AT_ONCE, MASK_WORDS / words) : ROWS_AT_ONCE, parts = (r1 - r0 + most - 1) / most;
        const int at_once = min(most, ((r1 - r0 + parts - 1) / parts + 3) & ~3);
        __syncthreads();                             // (the part before is through with the counts)
        // The first history tokens, the masks of the first rows and the counts' zeros are on their way together.
        const int* at = p.history + first_token;
        // (without tokens nothing is loaded: their start may be any number)
        const int skew = len > 0 ? (int)((uintptr_t)at >> 2 & 3) : 0, warp0 = tid & ~31;
        int4 t4[4];
        auto tokens_of = [&](int g0) {               // four tokens a load, from the 16 bytes on in which the history begins
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int g = g0 + u * NT + tid;
                t4[u] = make_int4(-1, -1, -1, -1);
                if (g * 4 - skew < len) t4[u] = __ldcg(reinterpret_cast<const int4*>(at - skew) + g);
            }
        };
        tokens_of(0);
        // A single row is asked for while the history is counted, 32 tokens of a mask's word at a time (64 rows 26.3 -> 24.9 us; rows of trees
        // come to warps that have others to wait for: 256 of them 56 us, and 63 with this).
        const bool single = r1 - r0 == 1;
        auto ahead = [&](int word) {
            const int t = max(lo, (w0 + word) * 32);
            asm volatile("prefetch.global.L2 [%0];" ::"l"(p.logits + (size_t)r0 * p.vocab + t));
        };
        if (single && !p.mask) for (int i = tid; i < words; i += NT) ahead(i);
        int biased = e0 + tid < e1 ? __ldcg(p.bias_tokens + e0 + tid) : -1;
        bool masked = false;
        auto masks_of = [&](int c0, int rows) {      // which of rows c0 .. have one
            masked = false;
            for (int i = tid; i < rows; i += NT) { mask_at[i] = mask_of(c0 + i); masked = masked || mask_at[i] >= 0; }
        };
        auto mask_words_of = [&](int rows) {
            for (int i = tid; i < rows * words; i += NT) {
                const int m = mask_at[i / words];
                const unsigned word = m < 0 ? 0xffffffffu : __ldcg(p.mask + (size_t)m * p.mask_words + w0 + i % words);
                masks[i] = word;
                if (single && word) ahead(i);
            }
        };
        if (p.mask) masks_of(r0, min(at_once, r1 - r0));
        if (len > 0) for (int i = tid; i < p.slice / 8; i += NT) reinterpret_cast<uint4*>(count_words)[i] = make_uint4(0u, 0u, 0u, 0u);
        if (tid == 0) { hit_count = 0; bias_range[0] = e1; bias_range[1] = e0; }
        masked = __syncthreads_or(masked);
        for (int e = e0 + tid; e < e1; e += NT) {
            if (biased >= lo && biased < hi) { atomicMin(&bias_range[0], e); atomicMax(&bias_range[1], e + 1); }
            biased = e + NT < e1 ? __ldcg(p.bias_tokens + e + NT) : -1;
        }
        auto hits_of = [&](int u0) {                 // which of nodes u0 .. have a token of the slice
            for (int i = u0 + tid; i < min(nodes, u0 + NODES); i += NT)
                if (token_of(i) >= lo && token_of(i) < hi) hits[atomicAdd(&hit_count, 1)] = (short)(i - u0);
        };
        hits_of(0);
        if (masked) mask_words_of(min(at_once, r1 - r0));
        // Few tokens are the slice's: a warp lists those of its 512 and then counts them a lane each.  (With a branch for every token
        // nearly every one was taken by some lane.)
        unsigned short* list = lists[tid >> 5];
        for (int g0 = 0; (g0 + warp0) * 4 - skew < len; g0 += 4 * NT) {
            if (g0 > 0) tokens_of(g0);
            int n = 0;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int t[4] = {t4[u].x, t4[u].y, t4[u].z, t4[u].w};
                const int i0 = (g0 + u * NT + tid) * 4 - skew;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const unsigned place = (unsigned)(t[e] - lo);
                    const bool hit = place < (unsigned)(hi - lo) && (unsigned)(i0 + e) < (unsigned)len;
                    const unsigned found = __ballot_sync(0xffffffffu, hit);
                    if (hit) list[n + __popc(found & ((1u << lane) - 1))] = (unsigned short)(place | (i0 + e < prompt ? 0x8000u : 0u));
                    n += __popc(found);
                }
            }
            __syncwarp();
            for (int i = lane; i < n; i += 32) counts.add(list[i] & 0x7fff, list[i] >> 15);
            __syncwarp();
        }

        // ------------------------------------------------ the rows' slices
        for (int c0 = r0; c0 < r1; c0 += at_once) {
            const int rows = min(at_once, r1 - c0);
            if (c0 == r0) {
                __syncthreads();                     // the counts and the first rows' masks are there
            } else if (p.mask) {
                __syncthreads();
                masks_of(c0, rows);
                masked = __syncthreads_or(masked);
                if (masked) {
                    mask_words_of(rows);
                    __syncthreads();
                }
            }
            auto one = [&](int row, int t) {
                const size_t i = (size_t)(c0 + row) * p.vocab + t;
                const float x = penalised(__ldcg(p.logits + i), len > 0 ? counts.at(t - lo) : 0u);
                p.out[i] = masked && !(masks[row * words + (t >> 5) - w0] >> (t & 31) & 1u) ? -INFINITY : x;
            };
            if (!VEC) {
                for (int row = 0; row < rows; ++row)
                    for (int t = lo + tid; t < hi; t += NT) one(row, t);
                continue;
            }
            // tokens ahead of a row's first aligned four: the same for every fourth row, and for all where vocab is a multiple of 4
            auto skip = [&](int row) {
                return (int)((4 - (((uintptr_t)p.logits >> 2) + (size_t)(c0 + row) * p.vocab + lo)) & 3);
            };
            const int step = p.vocab & 3 ? 4 : 1;
            for (int like = 0; like < min(step, rows); ++like) {
                const int s0 = lo + skip(like), fours = (hi - s0) / 4, alike = (rows - like + step - 1) / step;
                const size_t row0 = (size_t)(c0 + like) * p.vocab + s0;
                const float4* from = reinterpret_cast<const float4*>(p.logits + row0);           // of the fours' first row
                float4* to = reinterpret_cast<float4*>(p.out + row0);
                const int pitch = p.vocab / 4 * step + (p.vocab & 3) * (step / 4);                // fours from a row to the next that is alike
                const unsigned* bits_at = masks + like * words;
                const int bits_pitch = step * words, bit0 = s0 - 32 * w0;
                auto bits_of = [&](int n, int k) -> unsigned {
                    const int at = bit0 + 4 * k;
                    const unsigned* w = bits_at + n * bits_pitch + (at >> 5);
                    return __funnelshift_r(w[0], (at & 31) > 28 ? w[1] : 0u, at & 31) & 15u;
                };
                // Which of the thread's four tokens were seen (a bit each), and what is added to their logits.
                const bool aligned = !counts.wide && ((s0 - lo) & 3) == 0;
                const uint2* pairs = reinterpret_cast<const uint2*>(count_words) + (s0 - lo) / 4;
                auto seen_of = [&](int k, float (&less)[4]) -> unsigned {
                    if (len == 0) return 0u;
                    unsigned c[4];
                    if (aligned) {
                        const uint2 w = pairs[k];
                        if ((w.x | w.y) == 0u) return 0u;
                        c[0] = w.x & 0xffffu; c[1] = w.x >> 16; c[2] = w.y & 0xffffu; c[3] = w.y >> 16;
#pragma unroll
                        for (int e = 0; e < 4; ++e) less[e] = penalised.less(c[e] & 0x7fffu);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) { c[e] = counts.at(s0 - lo + 4 * k + e); less[e] = penalised.less(c[e]); }
                    }
                    return (c[0] ? 1u : 0u) | (c[1] ? 2u : 0u) | (c[2] ? 4u : 0u) | (c[3] ? 8u : 0u);
                };
                auto penalise = [&](float4& x, unsigned seen, const float (&less)[4]) {
                    x.x = penalised.apply(x.x, seen & 1u, less[0]); x.y = penalised.apply(x.y, seen & 2u, less[1]);
                    x.z = penalised.apply(x.z, seen & 4u, less[2]); x.w = penalised.apply(x.w, seen & 8u, less[3]);
                };
                auto ban = [&](float4& x, unsigned bits) {
                    if (!(bits & 1u)) x.x = -INFINITY;
                    if (!(bits & 2u)) x.y = -INFINITY;
                    if (!(bits & 4u)) x.z = -INFINITY;
                    if (!(bits & 8u)) x.w = -INFINITY;
                };
                if (alike > 1) {                     // a thread's four tokens in four rows
                    const int turns = (alike + 3) / 4;
                    for (int j = tid; j < fours * turns; j += NT) {
                        const int turn = j / fours, k = j - turn * fours, n0 = 4 * turn, left = alike - n0;
                        const float4* src = from + (size_t)n0 * pitch + k;
                        float4* dst = to + (size_t)n0 * pitch + k;
                        float4 x[4];
                        unsigned bits = 0xffffu;     // of the four rows
                        if (masked) {
                            bits = 0u;
#pragma unroll
                            for (int u = 0; u < 4; ++u) if (u < left) bits |= bits_of(n0 + u, k) << (4 * u);
                        }
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (u < left && (bits >> (4 * u) & 15u)) x[u] = __ldcg(src + u * pitch);
                        }
                        float less[4];
                        const unsigned seen = seen_of(k, less);
                        if (seen) {
#pragma unroll
                            for (int u = 0; u < 4; ++u) penalise(x[u], seen, less);
                        }
                        if (bits != 0xffffu) {
#pragma unroll
                            for (int u = 0; u < 4; ++u) ban(x[u], bits >> (4 * u));
                        }
#pragma unroll
                        for (int u = 0; u < 4; ++u) if (u < left) dst[u * pitch] = x[u];
                    }
                } else {                             // 16 tokens of a row
                    for (int k0 = tid; k0 < fours; k0 += 4 * NT) {
                        float4 x[4];
                        unsigned bits = 0xffffu;
                        if (masked) {
                            bits = 0u;
#pragma unroll
                            for (int u = 0; u < 4; ++u) if (k0 + u * NT < fours) bits |= bits_of(0, k0 + u * NT) << (4 * u);
                        }
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (k0 + u * NT < fours && (bits >> (4 * u) & 15u)) x[u] = __ldcg(from + k0 + u * NT);
                        }
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            if (k0 + u * NT >= fours) continue;
                            float less[4];
                            const unsigned seen = seen_of(k0 + u * NT, less);
                            if (seen) penalise(x[u], seen, less);
                            if (bits != 0xffffu) ban(x[u], bits >> (4 * u));
                            to[k0 + u * NT] = x[u];
                        }
                    }
                }
            }
            // the up to three tokens of a row ahead of its fours, and those behind
            if (p.vocab & 3 || ((uintptr_t)p.logits & 15) || ((hi - lo) & 3)) {
                for (int i = tid; i < rows * 6; i += NT) {
                    const int row = i / 6, e = i % 6, s = skip(row), left = (hi - lo - s) & 3;
                    if (hi - lo < s) {               // (a slice of fewer tokens than that)
                        if (e < hi - lo) one(row, lo + e);
                    } else if (e < 3 ? e < s : e - 3 < left) {
                        one(row, e < 3 ? lo + e : hi - left + e - 3);
                    }
                }
            }
        }

        // ------------------------------------------------ what paths and biases change
        // a thread a node of the slice's and a node that may have it on its path; a token that is there more than once is done where
        // the path has it first, for all of them
        auto paths_of = [&](int u0, auto parent_of, auto token_of) {
            for (int i = tid; i < hit_count * nodes; i += NT) {
                const int up = u0 + hits[i / nodes], node = i % nodes, t = token_of(up);
                int o = node;
                bool first = true;
                while (o > up) { first = first && token_of(o) != t; o = parent_of(o); }
                if (o != up || !first) continue;
                unsigned more = 1;
                for (o = parent_of(up); o >= 0; o = parent_of(o)) more += token_of(o) == t;
                if (o != -1) continue;               // padding, or a node behind it: no path
                const size_t k = (size_t)(r0 + node) * p.vocab + t;
                const float x = __ldcg(p.logits + k);
                if (allowed(r0 + node, t)) p.out[k] = penalised(x, len > 0 ? counts.at(t - lo) : 0u, more);
            }
        };
        if (nodes > 0) __syncthreads();
        if (nodes <= NODES) paths_of(0, [&](int i) -> int { return parent[i]; }, [&](int i) { return token[i]; });
        else
            for (int u0 = 0; u0 < nodes; u0 += NODES) {
                if (u0 > 0) {
                    __syncthreads();
                    if (tid == 0) hit_count = 0;
                    __syncthreads();
                    hits_of(u0);
                    __syncthreads();
                }
                paths_of(u0, parent_of, token_of);
            }
        const int f0 = bias_range[0], f1 = bias_range[1], n_rows = r1 - r0;
        if (f0 < f1) {
            __syncthreads();
            // ascending tokens: equal ones are neighbours, whose values the first of them adds in their order
            for (long long i = tid; i < (long long)(f1 - f0) * n_rows; i += NT) {
                const int e = f0 + (int)(i / n_rows), r = r0 + (int)(i % n_rows);
                const int t = __ldcg(p.bias_tokens + e);
                if (t < lo || t >= hi || (e > e0 && __ldcg(p.bias_tokens + e - 1) == t)) continue;
                float* to = p.out + (size_t)r * p.vocab + t;
                const float x = *to;
                float bias = __ldcg(p.bias_values + e);
                bool banned = bias == -INFINITY;
                for (int o = e + 1; o < e1 && __ldcg(p.bias_tokens + o) == t; ++o) {
                    const float v = __ldcg(p.bias_values + o);
                    banned = banned || v == -INFINITY;
                    bias += v;
                }
                // (finite ones may add up to infinity, which frees no token that a mask or a bias bans)
                *to = banned || x == -INFINITY ? -INFINITY : x + bias;
            }
        }
    }
}

// Tokens of a slice: as many slices a request as fill whole waves, of few tokens where there are few requests.
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
    static bool configured = false;
    if (!configured) {
        if (cudaFuncSetAttribute(control_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST_TOKENS * 2) != cudaSuccess ||
            cudaFuncSetAttribute(control_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST_TOKENS * 2) != cudaSuccess)
            return TFF_ERR_LAUNCH;
        configured = true;
    }
    if ((((uintptr_t)logits ^ (uintptr_t)out) & 15) == 0) return tff_launch_pdl(control_kernel<true>, grid, dim3(NT), smem, stream, p);
    return tff_launch_pdl(control_kernel<false>, grid, dim3(NT), smem, stream, p);
}
