// Attention of trees of drafted tokens over the paged cache, in float32 arithmetic: any head size up to 512, any numbers of heads and
// groups, either type.  It is the attention of the true 32-bit path and takes every size that the tcgen05 kernel refuses.
//
// Request b has c = pos_start[b] cached tokens and brings n = q_start[b + 1] - q_start[b] nodes, node i in cache slot c + i.  Its
// parent (parents, of its row) is an earlier node or -1: it follows the cached tokens.  A node whose chain of parents does not end at
// -1 is not there: it sees nothing, nobody sees it, its output is zeros.  The others see
//   the slots below c, and those of the node's ancestors and its own
// A node's position is c + its ancestors; with a window of w it sees what is less than w positions behind it, and, with
// ``keep``, the first ``keep`` positions.  Score cap, sink and head gates as in attention_common.h:
//   s[k] = (q . k) * scale, capped;   out = gate * sum_k exp(s[k]) v[k] / (sum_k exp(s[k]) + exp(sink))
//
// A CTA takes a tile of packed rows (node, query head of the group) of one request and kv head and a share of its key blocks of
// 32, which come to shared memory once for all its rows; a warp has up to 4 rows: for the scores a lane is a key, for the values a
// lane has 4 (8, 16) columns.  What a row sees of a block is a word with a bit a key.  The shares' results (maximum, sum, weighted
// values) are joined by a second kernel.
//
// What bounds it: shared-memory reads (every warp reads the whole block) and, in small steps, chains of them: two trees of 13 nodes behind 550
// tokens (16/8 heads of 128, float32) 23 us; with 8 warps of four rows 28, and 43 with a reference that moves and a sum that is added across
// the warp with every block.
#include "common.cuh"
#include "attention_common.h"
#include "attention_tree.cuh"
#include "tma_host.h"

namespace {

constexpr float SLACK = 8.f;
constexpr int BLOCK = 32, JOIN_THREADS = 128, NODE_WORDS = TREE_MAX_NODES / 32;

struct TreeParams {
    const int *q_start, *pos_start, *parents, *block_table;
    int tokens, table_width, pages, layer, nq, nkv, d, dv, window, keep, splits, stages, vec, q_vec;
    float scale, softcap;
    int sink;
    const float *sink_val, *gate;
    float *part_o, *part_ml;
    KvLayout L;
};

__device__ __forceinline__ float4 load4(const float* p) { return __ldcg((const float4*)p); }
__device__ __forceinline__ float4 load4(const bf16* p) {
    const uint2 u = __ldcg((const uint2*)p);
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                       __uint_as_float(u.y & 0xffff0000u));
}

// RW rows a warp, ND groups of 128 value columns (4 a lane).
template <typename T, int WARPS, int RW, int ND>
__global__ void __launch_bounds__(WARPS * 32, WARPS == 8 ? 2 : 1)
attention_tree_kernel(const T* q_in, const T* cache, T* __restrict__ out, const TreeParams p) {
    extern __shared__ float4 smem4[];
    __shared__ short parent[TREE_MAX_NODES];
    __shared__ unsigned line[WARPS * RW][NODE_WORDS];         // of a row's node: itself and the ancestors it sees, a bit each
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = p.nq / p.nkv, kvh = blockIdx.y, split = blockIdx.z % p.splits, b = blockIdx.z / p.splits;
    const int k4 = (p.d + 3) / 4, v4 = (p.dv + 3) / 4;        // groups of 4 elements a row
    const int ks = k4 | 1;                                    // an odd pitch: 8 lanes read 8 rows' groups in all banks
    const int stage4 = BLOCK * (ks + v4);
    float4* sq = smem4 + p.stages * stage4;                   // [WARPS * RW][k4]
    float* sp = (float*)(sq + WARPS * RW * k4) + warp * RW * BLOCK;       // the warp's weights [RW][32]
    pdl_launch_dependents();
    pdl_wait();
    const int q0 = p.q_start[b], nodes = min(min(p.q_start[b + 1], p.tokens) - q0, TREE_MAX_NODES), rows = nodes * G, row0 = blockIdx.x * WARPS * RW;
    if (row0 >= rows) return;
    const int ctx = p.pos_start[b], hi = ctx + nodes - 1;
    const int lo_tile = p.window > 0 ? max(0, ctx - p.window + 1) : 0;    // the first position that a root sees
    const int* table = p.block_table + (size_t)b * p.table_width;
    const KeyWalk walk(p.keep, BLOCK, lo_tile / BLOCK, hi / BLOCK);
    const int per = (walk.count + p.splits - 1) / p.splits;
    const int w0 = split * per, w1 = min(walk.count, w0 + per);

    for (int i = threadIdx.x; i < nodes; i += WARPS * 32) parent[i] = tree_parent(__ldcg(p.parents + q0 + i), i);
    for (int i = threadIdx.x; i < WARPS * RW * NODE_WORDS; i += WARPS * 32) line[i / NODE_WORDS][i % NODE_WORDS] = 0u;
#pragma unroll 4
    for (int i = threadIdx.x; i < WARPS * RW * k4; i += WARPS * 32) {
        const int r = row0 + i / k4, c = (i % k4) * 4;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < rows) {
            const T* src = q_in + ((size_t)(q0 + r / G) * p.nq + (size_t)(kvh * G + r % G)) * p.d + c;
            if (p.q_vec) {
                v = load4(src);
            } else {
                v.x = ldcg_f32(src);
                if (c + 1 < p.d) v.y = ldcg_f32(src + 1);
                if (c + 2 < p.d) v.z = ldcg_f32(src + 2);
                if (c + 3 < p.d) v.w = ldcg_f32(src + 3);
            }
        }
        sq[i] = v;
    }
    __syncthreads();
    const int wrow = row0 + warp * RW;                        // the warp's first row
    int pos[RW], lo[RW];                                      // positions of the rows' nodes (-1: none), their windows' first positions
    for (int j = 0; j < RW; ++j) {
        // every lane walks the same chain; lane 0 notes it
        const int node = wrow + j < rows ? (wrow + j) / G : -1;
        const int depth = tree_depth(parent, node);
        pos[j] = depth < 0 ? -1 : ctx + depth;
        lo[j] = p.window > 0 ? max(0, pos[j] - p.window + 1) : 0;
        if (lane == 0 && depth >= 0) {
            int at = pos[j];
            for (int a = node; a >= 0; a = parent[a], --at)
                if (at >= lo[j] || at < p.keep) line[warp * RW + j][a >> 5] |= 1u << (a & 31);
        }
    }
    __syncwarp();

    // Where key n0 + lane lies: null for keys that no row sees (their slots may hold anything, and their pages may have been given
    // back) and where the table has no page; their stage rows become zeros.  Looked up a block ahead of the copies.
    auto locate = [&](int n0) -> const T* {
        const int n = n0 + lane;
        if (n > hi || !(n >= lo_tile || n < p.keep) || n / p.L.page_size >= p.table_width) return nullptr;
        const int page = table[n / p.L.page_size];
        if (page < 0 || page >= p.pages) return nullptr;
        return cache + (size_t)page * p.L.page_stride + (size_t)p.layer * p.L.layer_stride +
               (size_t)kvh * p.L.head_stride + (size_t)(n % p.L.page_size) * p.L.head_dim;
    };
    auto fetch = [&](const T* at, int stage) {
        float4* sk = smem4 + stage * stage4;
        float4* sv = sk + BLOCK * ks;
#pragma unroll 2
        for (int kr = warp; kr < BLOCK; kr += WARPS) {
            const T* kp = (const T*)__shfl_sync(0xffffffffu, (unsigned long long)at, kr);
            const bool ok = kp != nullptr;
            const T* vp = kp + p.L.kv_stride;
            auto row = [&](const T* src, int n4, int len, float4* dst) {
                for (int c = lane; c < n4; c += 32) {
                    if (!ok) dst[c] = make_float4(0.f, 0.f, 0.f, 0.f);
                    else if (p.vec) {                         // rows of whole, aligned groups
                        if constexpr (sizeof(T) == 4)
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                                         ::"r"((uint32_t)__cvta_generic_to_shared(dst + c)), "l"(src + c * 4) : "memory");
                        else dst[c] = load4(src + c * 4);
                    } else {
                        const T* from = src + c * 4;
                        float4 v = make_float4(ldcg_f32(from), 0.f, 0.f, 0.f);
                        if (c * 4 + 1 < len) v.y = ldcg_f32(from + 1);
                        if (c * 4 + 2 < len) v.z = ldcg_f32(from + 2);
                        if (c * 4 + 3 < len) v.w = ldcg_f32(from + 3);
                        dst[c] = v;
                    }
                }
            };
            row(kp, k4, p.d, sk + kr * ks);
            row(vp, v4, p.dv, sv + kr * v4);
        }
    };

    const float inv_cap = p.softcap > 0.f ? 1.f / p.softcap : 0.f;
    float m[RW], l[RW], o[RW][4 * ND];
#pragma unroll
    for (int j = 0; j < RW; ++j) {
        m[j] = -INFINITY; l[j] = 0.f;
#pragma unroll
        for (int c = 0; c < 4 * ND; ++c) o[j][c] = 0.f;
    }
    auto block_start = [&](int w) { return walk.block(w) * BLOCK; };
    const T* at = w0 < w1 ? locate(block_start(w0)) : nullptr;
    if (p.stages > 1 && w0 < w1) {
        fetch(at, 0);
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (w0 + 1 < w1) at = locate(block_start(w0 + 1));
    }
    for (int w = w0; w < w1; ++w) {
        const int n0 = block_start(w), stage = p.stages > 1 ? ((w - w0) & 1) : 0;
        if (p.stages > 1) {
            if (w + 1 < w1) fetch(at, stage ^ 1);
            asm volatile("cp.async.commit_group;" ::: "memory");
            if (w + 2 < w1) at = locate(block_start(w + 2));
            asm volatile("cp.async.wait_group 1;" ::: "memory");
        } else {
            fetch(at, 0);
            asm volatile("cp.async.wait_all;" ::: "memory");
            if (w + 1 < w1) at = locate(block_start(w + 1));
        }
        __syncthreads();
        if (wrow < rows) {
            const float4* sk = smem4 + stage * stage4 + lane * ks;
            const float4* sv = smem4 + stage * stage4 + BLOCK * ks;
            const float4* qr = sq + warp * RW * k4;
            // ------------------------------------------------ scores: key n0 + lane against the warp's rows
            float acc[RW][4];
#pragma unroll
            for (int j = 0; j < RW; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
#pragma unroll 4
            for (int c = 0; c < k4; ++c) {
                const float4 k = sk[c];
#pragma unroll
                for (int j = 0; j < RW; ++j) {
                    const float4 q = qr[j * k4 + c];
                    acc[j][0] = fmaf(q.x, k.x, acc[j][0]);
                    acc[j][1] = fmaf(q.y, k.y, acc[j][1]);
                    acc[j][2] = fmaf(q.z, k.z, acc[j][2]);
                    acc[j][3] = fmaf(q.w, k.w, acc[j][3]);
                }
            }
            const int n = n0 + lane, node = n - ctx;
            unsigned seen[RW], every = 0xffffffffu;
#pragma unroll
            for (int j = 0; j < RW; ++j) {
                float s = ((acc[j][0] + acc[j][1]) + (acc[j][2] + acc[j][3])) * p.scale;
                if (p.softcap > 0.f) s = p.softcap * tanhf(s * inv_cap);
                bool valid;
                if (node < 0) valid = pos[j] >= 0 && (n >= lo[j] || n < p.keep);
                else valid = node < nodes && (line[warp * RW + j][node >> 5] >> (node & 31) & 1u);
                seen[j] = __ballot_sync(0xffffffffu, valid);
                every &= seen[j];
                s = valid ? s : -INFINITY;
                // The reference of the exponentials is moved only when a score passes it by more than SLACK (the weights stay below e^SLACK):
                // a vote in place of five shuffles, and another five for the sum, which every lane keeps for its own keys.
                if (__any_sync(0xffffffffu, s > m[j] + SLACK || (m[j] == -INFINITY && s > -INFINITY))) {
                    const float mn = fmaxf(m[j], warp_max(s));
                    const float alpha = m[j] == -INFINITY ? 0.f : expf(m[j] - mn);
                    l[j] *= alpha;
                    m[j] = mn;
#pragma unroll
                    for (int c = 0; c < 4 * ND; ++c) o[j][c] *= alpha;
                }
                const float pr = valid && s != -INFINITY ? expf(s - m[j]) : 0.f;      // (a score of -infinity has no weight)
                l[j] += pr;
                sp[j * BLOCK + lane] = pr;
            }
            __syncwarp();
            // ------------------------------------------------ values: the lane's columns of the warp's rows
#pragma unroll 2
            for (int c = 0; c < BLOCK; c += 4) {
                float4 x4[RW];
#pragma unroll
                for (int j = 0; j < RW; ++j) x4[j] = *(const float4*)(sp + j * BLOCK + c);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float4 v[ND];
#pragma unroll
                    for (int g = 0; g < ND; ++g) {
                        const int col = lane + 32 * g;
                        v[g] = col < v4 ? sv[(c + e) * v4 + col] : make_float4(0.f, 0.f, 0.f, 0.f);
                    }
#pragma unroll
                    for (int j = 0; j < RW; ++j) {
                        // a key that the row does not see adds nothing, whatever its value is
                        if (every == 0xffffffffu || (seen[j] >> (c + e) & 1u)) {
                            const float x = e == 0 ? x4[j].x : e == 1 ? x4[j].y : e == 2 ? x4[j].z : x4[j].w;
#pragma unroll
                            for (int g = 0; g < ND; ++g) {
                                o[j][4 * g] = fmaf(x, v[g].x, o[j][4 * g]);
                                o[j][4 * g + 1] = fmaf(x, v[g].y, o[j][4 * g + 1]);
                                o[j][4 * g + 2] = fmaf(x, v[g].z, o[j][4 * g + 2]);
                                o[j][4 * g + 3] = fmaf(x, v[g].w, o[j][4 * g + 3]);
                            }
                        }
                    }
                }
            }
            __syncwarp();
        }
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < RW; ++j) l[j] = warp_sum(l[j]);
#pragma unroll
    for (int j = 0; j < RW; ++j) {
        if (wrow + j >= rows) continue;
        const int h = kvh * G + (wrow + j) % G;
        const size_t item = (size_t)(q0 + (wrow + j) / G) * p.nq + h;
        float inv = 1.f;
        if (p.splits == 1) {
            inv = tree_weight(l[j], m[j], p.sink, p.sink_val, h) * (p.gate ? __ldcg(p.gate + item) : 1.f);
        } else if (lane == 0) {
            p.part_ml[(item * p.splits + split) * 2] = m[j];
            p.part_ml[(item * p.splits + split) * 2 + 1] = l[j];
        }
#pragma unroll
        for (int c = 0; c < 4 * ND; ++c) {
            const int col = (lane + 32 * (c / 4)) * 4 + c % 4;
            if (col >= p.dv) continue;
            if (p.splits == 1) out[item * p.dv + col] = from_f32<T>(l[j] > 0.f ? o[j][c] * inv : 0.f);
            else p.part_o[(item * p.splits + split) * p.dv + col] = o[j][c];
        }
    }
}

// Joins the shares (32 at most) of a (node, head): a block each, a lane a share for the weights, a thread a column (of every JOIN_THREADS)
// for the values, eight shares' loads together.
template <typename T>
__global__ void __launch_bounds__(JOIN_THREADS)
attention_tree_join_kernel(T* __restrict__ out, const TreeParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const int b = blockIdx.y, t = blockIdx.x / p.nq, h = blockIdx.x % p.nq, q0 = p.q_start[b], lane = threadIdx.x & 31;
    if (t >= min(min(p.q_start[b + 1], p.tokens) - q0, TREE_MAX_NODES)) return;
    const size_t item = (size_t)(q0 + t) * p.nq + h;
    const float2 ml = lane < p.splits ? __ldcg((const float2*)p.part_ml + item * p.splits + lane) : make_float2(-INFINITY, 0.f);
    const float m = warp_max(ml.y > 0.f ? ml.x : -INFINITY);
    const float f = ml.y > 0.f ? expf(ml.x - m) : 0.f;       // (a share that the row sees nothing of counts for nothing)
    const float l = warp_sum(ml.y * f);
    const float inv = tree_weight(l, m, p.sink, p.sink_val, h) * (p.gate ? __ldcg(p.gate + item) : 1.f);
    for (int col0 = 0; col0 < p.dv; col0 += JOIN_THREADS) {
        const int col = col0 + threadIdx.x;
        float o = 0.f;
        for (int s0 = 0; s0 < p.splits; s0 += 8) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u)
                v[u] = s0 + u < p.splits && col < p.dv ? __ldcg(p.part_o + (item * p.splits + s0 + u) * p.dv + col) : 0.f;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const float w = __shfl_sync(0xffffffffu, f, (s0 + u) & 31);
                if (w > 0.f) o = fmaf(v[u], w, o);
            }
        }
        if (col < p.dv) out[item * p.dv + col] = from_f32<T>(l > 0.f ? o * inv : 0.f);
    }
}

template <typename T, int WARPS, int RW, int ND>
int launch(const void* q, const void* cache, void* out, TreeParams p, int requests, int max_nodes, cudaStream_t s) {
    auto kern = attention_tree_kernel<T, WARPS, RW, ND>;
    const int k4 = (p.d + 3) / 4, v4 = (p.dv + 3) / 4;
    const size_t stage = (size_t)BLOCK * ((k4 | 1) + v4) * 16;
    const size_t rest = (size_t)WARPS * RW * k4 * 16 + (size_t)WARPS * RW * BLOCK * 4;
    p.stages = 2 * stage + rest <= 200 * 1024 ? 2 : 1;
    const size_t smem = p.stages * stage + rest;
    static bool configured = false;
    if (!configured) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024) != cudaSuccess) return TFF_ERR_LAUNCH;
        configured = true;
    }
    const int rows = max_nodes * (p.nq / p.nkv);
    if (smem > 200 * 1024) return TFF_ERR_UNSUPPORTED;
    return tff_launch_pdl(kern, dim3((rows + WARPS * RW - 1) / (WARPS * RW), p.nkv, requests * p.splits), dim3(WARPS * 32), smem, s,
                          (const T*)q, (const T*)cache, (T*)out, p);
}

template <typename T>
int dispatch(const void* q, const void* cache, void* out, const TreeParams& p, int requests, int max_nodes, cudaStream_t s) {
    const int rows = max_nodes * (p.nq / p.nkv);
    int st;
    // Tiles of 32 rows: 16 warps of two rows where there is at most a CTA an SM (26 rows a kv head behind 550 keys, two requests: 24 us, with
    // 8 warps of four 29), else two CTAs of 8 warps (72 tiles behind 900: 75 us, with 16 warps 86).
    const long long ctas = (long long)((rows + 31) / 32) * p.nkv * requests * p.splits;
    if (p.dv <= 128) st = rows <= 8 ? launch<T, 8, 1, 1>(q, cache, out, p, requests, max_nodes, s)
                          : rows <= 16 ? launch<T, 8, 2, 1>(q, cache, out, p, requests, max_nodes, s)
                          : ctas <= tff_num_sms() ? launch<T, 16, 2, 1>(q, cache, out, p, requests, max_nodes, s)
                                                  : launch<T, 8, 4, 1>(q, cache, out, p, requests, max_nodes, s);
    else if (p.dv <= 256) st = launch<T, 8, 2, 2>(q, cache, out, p, requests, max_nodes, s);
    else st = launch<T, 8, 1, 4>(q, cache, out, p, requests, max_nodes, s);
    if (st == TFF_OK && p.splits > 1)
        st = tff_launch_pdl(attention_tree_join_kernel<T>, dim3(max_nodes * p.nq, requests), dim3(JOIN_THREADS), (size_t)0, s, (T*)out, p);
    return st;
}

// Rows of a tile of the general kernel.
int tile_rows(int rows, int dv) { return dv <= 128 ? (rows <= 8 ? 8 : rows <= 16 ? 16 : 32) : dv <= 256 ? 16 : 8; }

}  // namespace

// In how many shares the general kernel's key blocks go to different CTAs: as many as fill the SMs, at least 2 blocks a share.
// ``max_kv`` bounds the cached tokens and nodes of a request.  With s > 1 shares the call needs num_tokens * nq * s * (dv + 2) floats.
TFF_API int tff_attention_tree_splits(int requests, int max_nodes, int max_kv, int nq, int nkv, int dv, int window, int keep, int sms) {
    if (requests <= 0 || max_nodes <= 0 || max_kv <= 0 || nkv <= 0 || nq <= 0 || nq % nkv || dv <= 0 || sms <= 0) return 1;
    const long long rows = (long long)max_nodes * (nq / nkv), tile = tile_rows((int)(rows < 64 ? rows : 64), dv);
    const long long ctas = (rows + tile - 1) / tile * nkv * requests;
    long long keys = max_kv;
    if (window > 0 && (long long)window + keep + max_nodes < keys) keys = (long long)window + keep + max_nodes;
    // A CTA an SM where that makes four shares or more of 32 rows (of 16 warps then: dispatch), else two; for smaller tiles two where their
    // stages leave room for both (one request of 8 nodes behind 4,000 tokens, 16/8 heads: 31 us, with one 40; of 4 behind 16,000, 8/8: 56 and 85)
    long long s = sms / ctas;
    if (s < 4 || (tile < 32 && dv <= 128)) s = 2ll * sms / ctas;
    if (s > keys / (2 * BLOCK)) s = keys / (2 * BLOCK);
    if (s > 32) s = 32;
    return s < 1 || requests * s > 65535 ? 1 : (int)s;
}

TFF_API int tff_attention_tree(const void* q, int is_bf16, const int* q_start, const int* pos_start, const int* parents,
                               const int* block_table, int table_width, const void* cache, long long cache_pages, int cache_layers, int layer,
                               int page_size, void* out, int num_tokens, int requests, int max_nodes, int nq, int nkv, int d, int dv, int dc,
                               float scale, int window, float softcap, int sink, const float* sink_val, const float* gate, int keep,
                               int splits, float* ws, cudaStream_t stream) {
    if (num_tokens <= 0 || requests <= 0 || max_nodes <= 0) return TFF_OK;
    if (!q || !q_start || !pos_start || !parents || !block_table || !cache || !out || nq <= 0 || nkv <= 0 || nq % nkv || d <= 0 ||
        dv <= 0 || dc < d || dc < dv || page_size <= 0 || cache_pages < 0 || softcap < 0.f || keep < 0 || splits < 1 || (splits > 1 && !ws))
        return TFF_ERR_BAD_ARGUMENT;
    if (d > 512 || dv > 512 || max_nodes > TREE_MAX_NODES || (long long)requests * splits > 65535 || nkv > 65535)
        return TFF_ERR_UNSUPPORTED;
    TreeParams p = {};
    p.q_start = q_start; p.pos_start = pos_start; p.parents = parents; p.block_table = block_table; p.tokens = num_tokens; p.table_width = table_width;
    p.pages = (int)(cache_pages < 0x7fffffff ? cache_pages : 0x7fffffff);
    p.layer = layer; p.nq = nq; p.nkv = nkv; p.d = d; p.dv = dv;
    p.window = window > 0 ? window : 0; p.keep = window > 0 ? keep : 0;
    p.sink = sink; p.sink_val = sink_val; p.gate = gate; p.scale = scale; p.softcap = softcap; p.splits = splits;
    p.L = make_kv_layout(cache_layers, nkv, page_size, dc);
    if (splits > 1) { p.part_ml = ws; p.part_o = ws + (size_t)num_tokens * nq * splits * 2; }
    // 4 elements are read at a time where rows and slots are whole groups at aligned addresses
    p.q_vec = d % 4 == 0 && ((uintptr_t)q & 15) == 0;
    p.vec = d % 4 == 0 && dv % 4 == 0 && dc % 4 == 0 && ((uintptr_t)cache & 15) == 0;
    return is_bf16 ? dispatch<bf16>(q, cache, out, p, requests, max_nodes, stream)
                   : dispatch<float>(q, cache, out, p, requests, max_nodes, stream);
}
