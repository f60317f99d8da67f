// Attention of trees of drafted tokens over the paged cache on the 5th-generation tensor cores: bfloat16, heads of 64 or 128, pages of
// 8 to 64 slots.  What a node sees and what a padding node gives is said in attention_tree.cu.
//
// The rows of a request and kv head (node, query head of the group) are one or a few tiles of 128 (QT = 2: pairs of tiles) that walk
// the same keys, context and nodes, in blocks of 64.  The walks of all requests and kv heads, one behind the other, are one
// line of blocks, of which every CTA takes an equal share, wherever that begins and ends: a share is pieces of one or
// more walks.  A piece that is a whole walk writes its rows' outputs; the others leave (maximum, sum, weighted values), which a second
// kernel joins.  Contexts of any lengths are so shared out evenly, and the division is made on the device from
// the step's arrays: a captured step follows its requests.
//
// A block of a piece (as in attention_prefill.cu, whose measurements the layout rests on):
//   S = Q K^T     tcgen05.mma, M = 128, N = 64; both operands K-major in 128-byte-swizzled shared memory; S in tensor memory
//   softmax       two groups of four warps a tile, one thread a row, which take a piece's blocks in turn: S row from tensor memory,
//                 maximum and sum in float32, probabilities to tensor memory as bfloat16 pairs
//   O += P V      tcgen05.mma, M = 128, N = head size, K = 64; P the A operand in tensor memory, V as the pages lie
// O is rescaled when a row's maximum has grown by more than 2^8.  Only blocks with nodes, a window's first and the kept
// tokens' last are masked: a row builds a word of 64 bits from its chain of parents, which lie in shared memory.
//   warps 0-7     softmax, rescale, outputs of the first tile (tensor memory lanes 32 * (warp % 4) ..)
//   warps 8-15    the same for the second tile (QT = 2)
//   then          TMA producer: one box a page into a ring of stages, without a pause between pieces; an issuing warp a tile
// Every mbarrier wait is bounded; a timeout raises the library's error word.
#define TFF_SUSPENDED_WAITS
#include "tcgen05.cuh"
#include "attention_common.h"
#include "attention_tc.cuh"
#include "attention_tree.cuh"
#include <type_traits>

namespace {

using tc5::smem_u32;
using tc5::mbar_init;
using tc5::mbar_expect_tx;
using tc5::mbar_arrive;
using tc5::mbar_wait_warp;
using tc5::umma4_bf16_elected;
using tc5::umma_commit_elected;
using tc5::fence_async_smem;
using tc5::tmem_alloc;
using tc5::tmem_dealloc;
using tc5::tc_fence_before;
using tc5::tc_fence_after;
using tc5::tmem_ld16;
using tc5::tmem_ld_wait;

constexpr int BLOCK_M = 128, BLOCK_N = 64, BARS_PER_TILE = 16, JOIN_ROWS = 16;
constexpr float RESCALE_THRESHOLD = 8.0f;            // in log2 units

struct TreeTcParams {
    const bf16* q; bf16* out;
    const int *q_start, *pos_start, *parents, *block_table;
    int requests, table_width, cache_layers, layer, page_shift, nq, nkv, window, keep, least;
    float scale_log2, scale_over_cap, cap_log2;
    int sink; const float *sink_val, *gate;
    float *part_o, *part_ml; int4* joins;
    int* error_flag;
};

// A box of tff_tensor_map_kv_groups: a page's keys and values of a kv head, from its first group of 8 rows.
__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* tm, uint32_t bar, int group) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %3, %3, %3, %4}], [%2];"
        ::"r"(dst), "l"(tm), "r"(bar), "r"(0), "r"(group) : "memory");
}

template <int D, int QT>
struct TreeCfg {
    static constexpr int kQBytes = BLOCK_M * D * 2;                 // [64-column half][128 rows][128 B]
    static constexpr int kStageBytes = BLOCK_N * 2 * D * 2;
    static constexpr int kStages = D > 64 ? 5 : 8;
    static constexpr int kExchange = QT * 2 * BLOCK_M * 4;          // a float of every row from either group
    static constexpr int kParents = TREE_MAX_NODES * 2;
    static constexpr int kBars = 2 * kStages + BARS_PER_TILE * QT;
    static constexpr int kSmem = QT * kQBytes + kStages * kStageBytes + kExchange + kParents + 8 * kBars + 16;
    static constexpr int kThreads = (8 * QT + 1 + QT) * 32;
    static_assert(kSmem <= 227 * 1024, "shared memory of the tree attention kernel");
};

// A request's walk.
struct Walk {
    int q0, nodes, ctx, lo, tiles, count;
    template <typename P>
    __device__ __forceinline__ Walk(const P& p, int b, int tile_rows) {
        q0 = p.q_start[b];
        nodes = max(0, min(p.q_start[b + 1] - q0, TREE_MAX_NODES));
        ctx = p.pos_start[b];
        lo = p.window > 0 ? max(0, ctx - p.window + 1) : 0;         // the first position that a root sees
        tiles = (nodes * (p.nq / p.nkv) + tile_rows - 1) / tile_rows;
        count = tiles > 0 ? keys(p.keep).count : 0;
    }
    __device__ __forceinline__ int hi() const { return ctx + nodes - 1; }
    __device__ __forceinline__ KeyWalk keys(int keep) const { return KeyWalk(keep, BLOCK_N, lo / BLOCK_N, hi() / BLOCK_N); }
    __device__ __forceinline__ long long blocks() const { return (long long)tiles * count; }
};

// A CTA's share of the line of blocks, piece by piece.  Every warp goes through it by itself, with all its lanes.
template <int ROWS>
struct Pieces {
    const TreeTcParams& p;
    long long first, left, line;                     // the share's first block, blocks behind the present piece, blocks a kv head
    int ctas;                                        // that have a share
    int b, kvh, tile, at, nb;                        // the piece: request, kv head, tile; its first block of the walk, its blocks
    Walk w;
    __device__ __forceinline__ Pieces(const TreeTcParams& p_) : p(p_), b(0), kvh(0), tile(0), at(0), nb(0), w(p_, 0, ROWS) {
        const int lane = threadIdx.x & 31;
        auto sum_of = [&](int r0) -> long long {     // inclusive sums of 32 requests' blocks
            long long s = r0 + lane < p.requests ? Walk(p, r0 + lane, ROWS).blocks() : 0;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const long long before = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s += before;
            }
            return s;
        };
        const long long head = sum_of(0);
        line = __shfl_sync(0xffffffffu, head, 31);
        for (int r0 = 32; r0 < p.requests; r0 += 32) line += __shfl_sync(0xffffffffu, sum_of(r0), 31);
        const long long all = line * p.nkv;
        ctas = (int)min((long long)gridDim.x, max(1ll, all / p.least));
        first = share(blockIdx.x);
        left = (int)blockIdx.x < ctas ? share(blockIdx.x + 1) - first : 0;
        if (left <= 0) { left = 0; return; }
        kvh = (int)(first / line);
        long long rest = first % line;
        for (int r0 = 0; r0 < p.requests; r0 += 32) {
            const long long s = r0 == 0 ? head : sum_of(r0);
            const unsigned behind = __ballot_sync(0xffffffffu, rest < s);
            if (behind) {
                const int src = __ffs(behind) - 1;
                b = r0 + src;
                const long long before = __shfl_sync(0xffffffffu, s, max(src - 1, 0));
                rest -= src > 0 ? before : 0;
                break;
            }
            rest -= __shfl_sync(0xffffffffu, s, 31);
        }
        w = Walk(p, b, ROWS);
        tile = (int)(rest / w.count);
        at = (int)(rest % w.count);
    }
    __device__ __forceinline__ long long share(int cta) const { return line * p.nkv * cta / ctas; }
    // The next piece; false behind the last.
    __device__ __forceinline__ bool next() {
        at += nb;
        if (nb > 0 && at == w.count) {
            at = 0;
            if (++tile == w.tiles) {
                tile = 0;
                if (left > 0) {
                    do {
                        if (++b == p.requests) { b = 0; ++kvh; }
                        w = Walk(p, b, ROWS);
                    } while (w.count == 0);
                }
            }
        }
        if (left <= 0) return false;
        nb = (int)min(left, (long long)(w.count - at));
        left -= nb;
        return true;
    }
    __device__ __forceinline__ bool whole() const { return at == 0 && nb == w.count; }
};

// below(k): the first k of 64 bits.
__device__ __forceinline__ uint64_t below(int k) { return k <= 0 ? 0ull : k >= 64 ? ~0ull : (1ull << k) - 1; }

// QT: query tiles a CTA walks with at once, two where some request has more rows than one.
template <int D, int QT>
__global__ void __launch_bounds__(TreeCfg<D, QT>::kThreads, 1)
attn_tree_tc_kernel(const __grid_constant__ CUtensorMap tm_cache, const TreeTcParams p) {
    using Cfg = TreeCfg<D, QT>;
    constexpr int HALVES = D / 64, CH = D / 8;                   // 64-column halves, 16-byte chunks of a key or value row
    constexpr int NSTAGES = Cfg::kStages, STAGE_BYTES = Cfg::kStageBytes;
    constexpr int GROUP = 2 * HALVES * 1024;                     // of a stage, [8 keys][K, V][half]: from 8 keys to the next 8
    constexpr int V_AT = HALVES * 1024;
    constexpr int ROWS = QT * BLOCK_M, SOFT = QT * 256;          // rows of a piece, softmax threads
    constexpr int TMEM_COLS = 512;                               // all of it: the allocation starts at column 0
    constexpr int LOAD_WARP = 8 * QT, ISSUE_WARP = LOAD_WARP + 1;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t sQ = smem_u32(smem), sKV = sQ + QT * Cfg::kQBytes;
    uint8_t* gKV = smem + QT * Cfg::kQBytes;
    volatile float* exchange = (volatile float*)(gKV + NSTAGES * STAGE_BYTES);       // [tile][group][row]
    short* parent = (short*)(gKV + NSTAGES * STAGE_BYTES + Cfg::kExchange);          // of the piece's request
    constexpr int BARS_AT = QT * Cfg::kQBytes + NSTAGES * STAGE_BYTES + Cfg::kExchange + Cfg::kParents;
    const uint32_t bars = sQ + BARS_AT;
    auto kv_full = [&](int s) { return bars + 8u * s; };
    auto kv_empty = [&](int s) { return bars + 8u * (NSTAGES + s); };
    // S(j), P(j), PV(j) and the reference of block j report to a barrier of the group that has block j of its piece (group j % 2)
    auto tile_bar = [&](int x, int i) { return bars + 8u * (2 * NSTAGES + BARS_PER_TILE * x + i); };
    auto s_full = [&](int x, int g) { return tile_bar(x, g); };
    auto s_free = [&](int x) { return tile_bar(x, 2); };
    auto p_full = [&](int x, int g) { return tile_bar(x, 3 + g); };
    auto pv_done = [&](int x, int g) { return tile_bar(x, 5 + g); };
    auto q_ready = [&](int x) { return tile_bar(x, 7); };
    auto ref_bar = [&](int x, int g, int q) { return tile_bar(x, 8 + 4 * g + q); };
    volatile uint32_t* tmem_slot = (volatile uint32_t*)(smem + BARS_AT + 8 * Cfg::kBars);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = p.nq / p.nkv;

    if (tid == 0) {
        for (int s = 0; s < NSTAGES; ++s) { mbar_init(kv_full(s), 1); mbar_init(kv_empty(s), QT); }
        for (int x = 0; x < QT; ++x) {
            for (int g = 0; g < 2; ++g) {
                mbar_init(s_full(x, g), 1); mbar_init(p_full(x, g), 4); mbar_init(pv_done(x, g), 1);
                for (int q = 0; q < 4; ++q) mbar_init(ref_bar(x, g, q), 1);
            }
            mbar_init(s_free(x), 4); mbar_init(q_ready(x), 8);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tm_cache) : "memory");
    }
    if (warp == ISSUE_WARP) tmem_alloc(smem_u32((const void*)tmem_slot), TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    constexpr uint32_t tmem_base = 0;
    pdl_launch_dependents();
    pdl_wait();
    Pieces<ROWS> piece(p);

    if (warp == LOAD_WARP) {
        // ------------------------------------------------------------ TMA producer
        if (lane == 0) {
            // the walk that this share's first piece ends, if others began it: joined by the second kernel
            int4 join = make_int4(-1, 0, 0, 0);
            if (piece.left > 0 && piece.at > 0 && piece.w.count - piece.at <= piece.left) {
                const long long start = piece.first - piece.at;
                int c = (int)(start * piece.ctas / (piece.line * p.nkv));
                while (c > 0 && piece.share(c) > start) --c;
                while (piece.share(c + 1) <= start) ++c;
                join = make_int4(piece.b, piece.kvh, piece.tile, c);
            }
            p.joins[blockIdx.x] = join;
        }
        __syncwarp();
        const int ppb = BLOCK_N >> p.page_shift;
        int s = 0;
        uint32_t round = 0;
        bool ok = true;
        while (ok && piece.next()) {
            const KeyWalk walk = piece.w.keys(p.keep);
            const int* table = p.block_table + (size_t)piece.b * p.table_width;
            const int table_end = piece.w.hi() >> p.page_shift;
            // the block table's entries of 32 pages, one a lane, and those of the next 32
            int chunk = -1, held = -1, ahead = -1;
            auto entry = [&](int c) {
                const int i = c * 32 + lane;
                return i <= table_end && i < p.table_width ? table[i] : -1;
            };
            for (int i = 0; i < piece.nb; ++i) {
                if (round > 0 && !(ok = mbar_wait_warp(kv_empty(s), (round - 1) & 1, abort_flag))) break;
                const int first = walk.block(piece.at + i) * BLOCK_N >> p.page_shift;       // (a block's pages lie in one run of 32)
                if (first >> 5 != chunk) {
                    held = first >> 5 == chunk + 1 && chunk >= 0 ? ahead : entry(first >> 5);
                    chunk = first >> 5;
                    ahead = entry(chunk + 1);
                }
                const bool valid = lane >= (first & 31) && lane < (first & 31) + ppb && held >= 0;
                const unsigned mask = __ballot_sync(0xffffffffu, valid);
                if (lane == 0) mbar_expect_tx(kv_full(s), (uint32_t)__popc(mask) * (uint32_t)(GROUP << (p.page_shift - 3)));
                __syncwarp();
                if (valid) {
                    const long long row = ((((long long)held * p.cache_layers + p.layer) * 2) * p.nkv + piece.kvh) << p.page_shift;
                    tma_load_5d(sKV + s * STAGE_BYTES + (uint32_t)((lane - (first & 31)) * (GROUP << (p.page_shift - 3))), &tm_cache, kv_full(s),
                                (int)(row >> 3));
                }
                if (++s == NSTAGES) { s = 0; ++round; }
            }
        }
    } else if (warp >= ISSUE_WARP) {
        // -------------------------------------------------------------- MMA issuers, one per tile
        auto issue = [&](auto which) {
            constexpr int x = decltype(which)::value;
            constexpr uint32_t t_s = tmem_base + x * 256, t_o = t_s + 128;
            const uint64_t qdesc = make_smem_desc(sQ + x * Cfg::kQBytes, 16, 1024);
            const uint64_t kdesc = make_smem_desc(sKV, 16, GROUP);             // + stage * STAGE_BYTES
            const uint64_t vdesc = make_smem_desc(sKV + V_AT, 1024, GROUP);
            constexpr uint32_t idesc_pv = make_idesc(BLOCK_M, D, 1);
            constexpr uint32_t idesc_s = make_idesc(BLOCK_M, BLOCK_N, 0);
            bool ok = true;
            uint32_t phase = 0, phase_q = 0, phase_s = 1;          // of the ring, the queries, s_free (nothing to wait for at first)
            uint32_t phase_p[2] = {0, 0};
            int st = 0, st_pv = 0;                                 // stages of S(n) and of PV(n - 2)
            while (ok && piece.next()) {
                if (piece.tile * ROWS + x * BLOCK_M >= piece.w.nodes * G) {
                    // a tile without rows gives the stages back as they arrive
                    for (int n = 0; n < piece.nb && ok; ++n) {
                        ok = mbar_wait_warp(kv_full(st), phase, abort_flag);
                        __syncwarp();
                        if (lane == 0) mbar_arrive(kv_empty(st));
                        if (++st == NSTAGES) { st = 0; phase ^= 1; }
                    }
                    st_pv = st;
                    continue;
                }
                ok = mbar_wait_warp(q_ready(x), phase_q, abort_flag);
                phase_q ^= 1;
                // S runs two blocks ahead of PV: a group that has written P(j) finds S(j + 2) finished
                for (int n = 0; n < piece.nb + 2 && ok; ++n) {
                    if (n < piece.nb) {
                        ok = mbar_wait_warp(kv_full(st), phase, abort_flag);
                        if (ok) ok = mbar_wait_warp(s_free(x), phase_s, abort_flag);         // the S before is in registers
                        if (!ok) break;
                        phase_s ^= 1;
                        tc_fence_after();
                        const uint64_t kd = kdesc + (uint64_t)(st * (STAGE_BYTES >> 4));
#pragma unroll
                        for (int h = 0; h < HALVES; ++h)
                            umma4_bf16_elected(t_s, qdesc + (uint64_t)(h * (BLOCK_M * 128) >> 4), kd + (uint64_t)(h * 1024 >> 4), idesc_s, h > 0 ? 1u : 0u);
                        umma_commit_elected(s_full(x, n & 1));
                        if (++st == NSTAGES) { st = 0; phase ^= 1; }
                    }
                    const int j = n - 2;
                    if (j >= 0) {
                        ok = mbar_wait_warp(p_full(x, j & 1), phase_p[j & 1], abort_flag);   // P(j) is in tensor memory
                        if (!ok) break;
                        phase_p[j & 1] ^= 1;
                        tc_fence_after();
                        const uint64_t vd = vdesc + (uint64_t)(st_pv * (STAGE_BYTES >> 4));
                        umma4_ts<(2 * GROUP >> 4)>(t_o, t_s + 64 + (j & 1) * 32, vd, idesc_pv, j > 0 ? 1u : 0u);
                        umma_commit_elected(pv_done(x, j & 1));                // O holds block j; that P buffer is free
                        umma_commit_elected(kv_empty(st_pv));                  // and this tile has read the stage
                        if (++st_pv == NSTAGES) st_pv = 0;
                    }
                }
            }
        };
        if (warp == ISSUE_WARP) issue(std::integral_constant<int, 0>());
        else if constexpr (QT == 2) issue(std::integral_constant<int, 1>());
    } else {
        // ------------------------------------------------- softmax / rescale / outputs
        const int x = warp >> 3, g = (warp >> 2) & 1;              // query tile and group of this warp: it has a piece's blocks g, g + 2, ...
        const int q = warp & 3;                                    // TMEM lane quarter this warp may touch
        const int r = q * 32 + lane;                               // row of the tile = TMEM lane
        const int tt = tid & 127;                                  // within the group
        const uint32_t t_row = tmem_base + ((uint32_t)(q * 32) << 16) + x * 256;
        const uint32_t t_s = t_row, t_p = t_row + 64 + g * 32, t_o = t_row + 128;
        // the two warps that have a row between them; all that read the parents and the queries' place
        auto pair_sync = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(1 + x * 4 + q) : "memory"); };
        auto soft_sync = [&]() { asm volatile("bar.sync 9, %0;" ::"n"(SOFT) : "memory"); };
        volatile float* mine = exchange + (x * 2 + g) * BLOCK_M + r;
        volatile float* other = exchange + (x * 2 + (g ^ 1)) * BLOCK_M + r;
        const float scale_log2 = p.cap_log2 > 0.f ? p.cap_log2 : p.scale_log2;
        // completions so far, mod 2: of the barriers of the own group, and of the other's
        uint32_t n_own = 0, n_other = 0;
        int stage = 0;                                             // of the piece's first block
        int parents_of = -1;
        bool ok = true;
        while (piece.next()) {
            const int q0 = piece.w.q0, ctx = piece.w.ctx, nodes = piece.w.nodes, hi = piece.w.hi(), nb = piece.nb;
            const KeyWalk walk = piece.w.keys(p.keep);
            const int R0 = piece.tile * ROWS + x * BLOCK_M, R = R0 + r, rows_total = nodes * G;
            const bool tile_active = R0 < rows_total;
            const int tok = R / G, head = piece.kvh * G + R % G;
            const int rows_left = min(32, rows_total - (R - lane));            // rows of this warp's 32 that exist
            // ---------------------------------- queries and parents; half of the columns of this warp's rows a group
            constexpr int RC = D / 16;                             // 16-byte chunks of a row that a group has
            uint4 u[RC];
            if (tile_active) {
#pragma unroll
                for (int i = 0; i < RC; ++i) {
                    const int row = (i * 32 + lane) / RC, c = g * RC + (i * 32 + lane) % RC;
                    const int t = __shfl_sync(0xffffffffu, tok, row), h = __shfl_sync(0xffffffffu, head, row);
                    u[i] = make_uint4(0u, 0u, 0u, 0u);
                    if (row < rows_left)
                        u[i] = __ldcg(reinterpret_cast<const uint4*>(p.q + ((size_t)(q0 + t) * p.nq + h) * D + c * 8));
                }
            }
            if (parents_of != piece.b) {
                // (every softmax thread goes through the same pieces)
                for (int i = tid; i < nodes; i += SOFT) parent[i] = tree_parent(__ldcg(p.parents + q0 + i), i);
                soft_sync();
                const bool gone = tid < nodes && tree_depth(parent, tid) < 0;
                static_assert(SOFT >= TREE_MAX_NODES, "a thread a node");
                soft_sync();
                if (gone) parent[tid] = -2;                        // whoever follows it is marked as well
                soft_sync();
                parents_of = piece.b;
            }
            const int depth = tile_active && R < rows_total ? tree_depth(parent, tok) : -1;
            const bool rv = depth >= 0;                            // a row of a node that is there
            const int pr = ctx + depth;
            const int lo_r = p.window > 0 ? max(0, pr - p.window + 1) : 0;
            if (tile_active) {
                uint8_t* dst = smem + x * Cfg::kQBytes + q * 32 * 128;
#pragma unroll
                for (int i = 0; i < RC; ++i) {
                    const int row = (i * 32 + lane) / RC, c = g * RC + (i * 32 + lane) % RC;
                    // padding has queries of zeros: whatever it brought, its scores are finite
                    if (!__shfl_sync(0xffffffffu, (int)rv, row)) u[i] = make_uint4(0u, 0u, 0u, 0u);
                    *reinterpret_cast<uint4*>(dst + (c >> 3) * (BLOCK_M * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = u[i];
                }
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(q_ready(x));
            }
            float m_used = -INFINITY, l = 0.f;
            const int nb_x = tile_active ? nb : 0;
            for (int j = g; j < nb_x && ok; j += 2) {
                ok = mbar_wait_warp(s_full(x, g), n_own, abort_flag);
                if (!ok) break;
                tc_fence_after();
                const int n_first = walk.block(piece.at + j) * BLOCK_N;
                // Masked or capped scores are written back over the raw ones, so that the pass below is the same for every block.
                // Rows that are not there are not stored: they need no mask.
                const bool some_nodes = n_first + BLOCK_N > ctx;
                const bool masked = some_nodes || !__all_sync(0xffffffffu, !rv || n_first >= lo_r || n_first + BLOCK_N <= p.keep);
                if (masked || p.cap_log2 > 0.f) {
                    uint64_t seen = ~0ull;
                    if (masked && rv) {
                        seen = below(ctx - n_first) & (~below(lo_r - n_first) | below(p.keep - n_first));
                        if (some_nodes) {
                            int pos = pr;
                            for (int a = tok; a >= 0 && ctx + a >= n_first; a = parent[a], --pos)
                                if (ctx + a < n_first + BLOCK_N && (pos >= lo_r || pos < p.keep)) seen |= 1ull << (ctx + a - n_first);
                        }
                    }
                    const uint32_t seen_lo = (uint32_t)seen, seen_hi = (uint32_t)(seen >> 32);
                    uint32_t v[BLOCK_N];
#pragma unroll
                    for (int h = 0; h < BLOCK_N / 16; ++h) tmem_ld16(t_s + h * 16, v + h * 16);
                    tmem_ld_wait();
                    if (p.cap_log2 > 0.f) {
#pragma unroll
                        for (int i = 0; i < BLOCK_N; ++i) v[i] = __float_as_uint(attn_tanh(__uint_as_float(v[i]) * p.scale_over_cap));
                    }
#pragma unroll
                    for (int i = 0; i < BLOCK_N; ++i)
                        v[i] = (i < 32 ? seen_lo >> i : seen_hi >> (i - 32)) & 1u ? v[i] : 0xff800000u;     // -infinity
#pragma unroll
                    for (int h = 0; h < BLOCK_N / 16; ++h) tmem_st16(t_s + h * 16, v + h * 16);
                    tmem_st_wait();
                }
                uint32_t s[BLOCK_N];
#pragma unroll
                for (int h = 0; h < BLOCK_N / 16; ++h) tmem_ld16(t_s + h * 16, s + h * 16);
                tmem_ld_wait();
                tc_fence_before();                                 // the scores are in registers: the buffer may
                __syncwarp();                                      // take the next block's
                if (lane == 0) mbar_arrive(s_free(x));
                float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < BLOCK_N; i += 2) m4[(i >> 1) & 3] = fmax3(m4[(i >> 1) & 3], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
                const float m_blk = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * scale_log2;
                // The reference that the exponentials use goes from block to block, and so from group to group.
                float m_prev = m_used;
                if (j > 0) {
                    ok = mbar_wait_warp(ref_bar(x, g ^ 1, q), n_other, abort_flag);
                    if (!ok) break;
                    n_other ^= 1;
                    m_prev = *other;
                }
                const bool grow = m_blk > m_prev + RESCALE_THRESHOLD || (m_prev == -INFINITY && m_blk > -INFINITY);
                const float m_new = grow ? m_blk : m_prev;
                *mine = m_new;
                const bool moved = __any_sync(0xffffffffu, m_new != m_used);
                __syncwarp();                                      // (a vote orders no memory: every lane's reference, then the arrival)
                if (lane == 0) mbar_arrive(ref_bar(x, g, q));
                // the product of the block before last must have read the P buffer that this block writes
                if (j > 1) {
                    ok = mbar_wait_warp(pv_done(x, g), n_own ^ 1, abort_flag);
                    if (!ok) break;
                    tc_fence_after();
                }
                if (some_nodes || walk.ragged(piece.at + j)) {
                    // value rows that no row may see (behind the last node, between the kept ones and the first window, of
                    // padding) are cleared, since slots and unfetched shared memory may hold anything; the warps of both tiles
                    // do it (the same zeros), so that each tile's products wait for its own warps only
                    uint8_t* rows = gKV + ((stage + j) % NSTAGES) * STAGE_BYTES + V_AT;
                    for (int idx = tt; idx < BLOCK_N * CH; idx += 128) {
                        const int kr = idx / CH, c = idx % CH;
                        const int n = n_first + kr;
                        if (n > hi || (n < piece.w.lo && n >= p.keep) || (n >= ctx && parent[n - ctx] == -2))
                            *reinterpret_cast<uint4*>(rows + (c >> 3) * 1024 + (kr >> 3) * GROUP + (kr & 7) * 128 + (((c & 7) ^ (kr & 7)) << 4)) =
                                make_uint4(0u, 0u, 0u, 0u);
                    }
                    fence_async_smem();
                }
                if (moved) {
                    const bool any_grow = __any_sync(0xffffffffu, grow);
                    if (any_grow && j > 0) {
                        // O must hold every earlier block before it is rescaled
                        ok = mbar_wait_warp(pv_done(x, g ^ 1), n_other ^ 1, abort_flag);
                        if (!ok) break;
                        tc_fence_after();
                        const float alpha = !grow ? 1.f : m_prev == -INFINITY ? 0.f : exp2f(m_prev - m_new);
#pragma unroll 1
                        for (int c0 = 0; c0 < D; c0 += 16) {
                            uint32_t v[16];
                            tmem_ld16(t_o + c0, v);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
                            tmem_st16(t_o + c0, v);
                        }
                    }
                    if (m_new != m_used) l = m_used == -INFINITY ? 0.f : l * exp2f(m_used - m_new);
                    m_used = m_new;
                }
                const float ms = m_used == -INFINITY ? 0.f : m_used;
                uint64_t lsum2[2] = {0ull, 0ull};
                const uint64_t scale2 = pack2(scale_log2, scale_log2), negms2 = pack2(-ms, -ms);
                // the probabilities, two a column
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t wd[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float a0, a1;
                        unpack2(fma2(pack2(__uint_as_float(s[c * 32 + 2 * i]), __uint_as_float(s[c * 32 + 2 * i + 1])), scale2, negms2), a0, a1);
                        const float e0 = ex2_approx(a0), e1 = ex2_approx(a1);
                        __nv_bfloat162 b2 = __floats2bfloat162_rn(e0, e1);
                        lsum2[i & 1] = add2(lsum2[i & 1], pack2(e0, e1));
                        wd[i] = *reinterpret_cast<uint32_t*>(&b2);
                    }
                    tmem_st16(t_p + c * 16, wd);
                }
                {
                    float s0, s1;
                    unpack2(add2(lsum2[0], lsum2[1]), s0, s1);
                    l += s0 + s1;
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full(x, g));
                n_own ^= 1;
            }
            // ---------------------------------------------------------------- outputs: half of the columns a group
            // The group that does not have the last block takes the last reference; the groups' sums then meet in shared memory.
            // (With a block fewer than the other group, or as many: what it has waited for and what it has not.)
            const int gl = (nb_x - 1) & 1;                         // the group of the last block
            if (ok && nb_x > 0 && g != gl) {
                ok = mbar_wait_warp(ref_bar(x, gl, q), n_other, abort_flag);
                n_other ^= 1;
                const float m_last = *other;
                if (m_used != m_last) l = m_used == -INFINITY ? 0.f : l * exp2f(m_used - m_last);
                m_used = m_last;
                // (its own last product first: the other barrier's completion before the one that is waited for is then in the past)
                if (ok && nb_x > 1) ok = mbar_wait_warp(pv_done(x, g), n_own ^ 1, abort_flag);
                if (ok) ok = mbar_wait_warp(pv_done(x, gl), n_other ^ 1, abort_flag);
            } else if (ok && nb_x > 0) {
                ok = mbar_wait_warp(pv_done(x, gl), n_own ^ 1, abort_flag);
            }
            pair_sync();                                           // both have read the last references
            *mine = l;
            pair_sync();
            l = g == 0 ? l + *other : *other + l;
            if (ok && nb_x > 0) {
                tc_fence_after();
                // through shared memory, where the queries lay (every S is finished), 32 rows a warp
                uint8_t* rows = smem + x * Cfg::kQBytes + (g * 4 + q) * (32 * D);
                if (piece.whole()) {
                    if (p.sink && l > 0.f) l += exp2f(attn_sink_log2(p.sink_val, head) - m_used);       // a key without a value
                    const bool some = rv && l > 0.f;               // (a padding row's sums may be anything)
                    float inv = some ? 1.f / l : 0.f;
                    if (p.gate && some) inv *= __ldcg(p.gate + (size_t)(q0 + tok) * p.nq + head);
                    auto cell = [&](int row, int c) { return rows + row * D + ((c ^ (RC == 8 ? row & 7 : (row >> 1) & 3)) << 4); };
#pragma unroll
                    for (int half = 0; half < RC / 4; ++half) {
                        uint32_t v[32];
                        tmem_ld16(t_o + g * (D / 2) + half * 32, v);
                        tmem_ld16(t_o + g * (D / 2) + half * 32 + 16, v + 16);
                        tmem_ld_wait();
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            uint32_t wd[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                __nv_bfloat162 b2 = __floats2bfloat162_rn(__uint_as_float(v[8 * c + 2 * i]) * inv, __uint_as_float(v[8 * c + 2 * i + 1]) * inv);
                                wd[i] = some ? *reinterpret_cast<uint32_t*>(&b2) : 0u;
                            }
                            *reinterpret_cast<uint4*>(cell(lane, half * 4 + c)) = make_uint4(wd[0], wd[1], wd[2], wd[3]);
                        }
                    }
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < RC; ++i) {
                        const int row = (i * 32 + lane) / RC, c = (i * 32 + lane) % RC;
                        const int t = __shfl_sync(0xffffffffu, tok, row), h = __shfl_sync(0xffffffffu, head, row);
                        if (row < rows_left)
                            *reinterpret_cast<uint4*>(p.out + ((size_t)(q0 + t) * p.nq + h) * D + (g * RC + c) * 8) =
                                *reinterpret_cast<const uint4*>(cell(row, c));
                    }
                } else {
                    // slot 0 of the CTA: a piece of a walk that another one began; slot 1: of one that this one begins
                    const size_t slot = ((size_t)blockIdx.x * 2 + (piece.at > 0 ? 0 : 1)) * ROWS + x * BLOCK_M + q * 32;
                    if (g == 0 && lane < rows_left)
                        *reinterpret_cast<float2*>(p.part_ml + (slot + lane) * 2) = make_float2(m_used, rv ? l : 0.f);
                    constexpr int W = D / 4;                       // columns at a time: 32 rows of them are what a warp's place holds
                    auto cell = [&](int row, int c) { return rows + row * (W * 4) + ((c ^ (row & (W / 4 - 1))) << 4); };
#pragma unroll 1
                    for (int half = 0; half < 2; ++half) {
                        uint32_t v[W];
#pragma unroll
                        for (int c = 0; c < W / 16; ++c) tmem_ld16(t_o + g * (D / 2) + half * W + c * 16, v + c * 16);
                        tmem_ld_wait();
#pragma unroll
                        for (int c = 0; c < W / 4; ++c)
                            *reinterpret_cast<uint4*>(cell(lane, c)) = make_uint4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < W / 4; ++i) {
                            const int row = (i * 32 + lane) / (W / 4), c = (i * 32 + lane) % (W / 4);
                            if (row < rows_left)
                                *reinterpret_cast<uint4*>(p.part_o + (slot + row) * D + g * (D / 2) + half * W + c * 4) =
                                    *reinterpret_cast<const uint4*>(cell(row, c));
                        }
                        __syncwarp();
                    }
                }
            }
            tc_fence_before();
            soft_sync();                                           // O, the queries' place and the parents may be written again
            stage = (stage + nb) % NSTAGES;
        }
    }
    // ------------------------------------------------------------------ teardown
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {
        for (int i = 0; i < 64; ++i) __nanosleep(1000);
        if (tid == 0) atomicExch(p.error_flag, 1);
        __syncthreads();
    }
    if (warp == ISSUE_WARP) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem_base, TMEM_COLS);
    }
}

// Joins the pieces of the walks that are more than one share's: blocks (c, y) take JOIN_ROWS rows of the walk that ends in share c.
template <int D, int QT>
__global__ void __launch_bounds__(128) attn_tree_join_kernel(const TreeTcParams p) {
    constexpr int ROWS = QT * BLOCK_M, W = D / 4;
    pdl_launch_dependents();
    pdl_wait();
    const int4 join = __ldcg(p.joins + blockIdx.x);                // request, kv head, tile, the first share
    if (join.x < 0) return;
    const int G = p.nq / p.nkv, b = join.x, last = blockIdx.x;
    const int q0 = p.q_start[b], rows_total = min(p.q_start[b + 1] - q0, TREE_MAX_NODES) * G;
    for (int idx = threadIdx.x; idx < JOIN_ROWS * W; idx += 128) {
        const int row = blockIdx.y * JOIN_ROWS + idx / W, c = idx % W;
        const int R = join.z * ROWS + row;
        if (R >= rows_total) return;
        auto slot = [&](int s) { return ((size_t)s * 2 + (s == join.w ? 1 : 0)) * ROWS + row; };
        float m = -INFINITY;
#pragma unroll 4
        for (int s = join.w; s <= last; ++s) {
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(p.part_ml) + slot(s));
            if (ml.y > 0.f) m = fmaxf(m, ml.x);
        }
        const float ms = m == -INFINITY ? 0.f : m;
        float l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int s = join.w; s <= last; ++s) {
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(p.part_ml) + slot(s));
            const float4 v = __ldcg(reinterpret_cast<const float4*>(p.part_o + slot(s) * D) + c);
            if (!(ml.y > 0.f)) continue;                           // a piece that the row saw nothing of counts for nothing
            const float f = exp2f(ml.x - ms);
            l = fmaf(ml.y, f, l);
            o.x = fmaf(v.x, f, o.x); o.y = fmaf(v.y, f, o.y); o.z = fmaf(v.z, f, o.z); o.w = fmaf(v.w, f, o.w);
        }
        const int t = q0 + R / G, h = join.y * G + R % G;
        float inv = 0.f;
        if (l > 0.f) inv = (p.gate ? __ldcg(p.gate + (size_t)t * p.nq + h) : 1.f) / (p.sink ? l + exp2f(attn_sink_log2(p.sink_val, h) - ms) : l);
        __nv_bfloat162 lo = __floats2bfloat162_rn(o.x * inv, o.y * inv), hi = __floats2bfloat162_rn(o.z * inv, o.w * inv);
        if (!(l > 0.f)) lo = hi = __floats2bfloat162_rn(0.f, 0.f);
        *reinterpret_cast<uint2*>(p.out + ((size_t)t * p.nq + h) * D + c * 4) =
            make_uint2(*reinterpret_cast<uint32_t*>(&lo), *reinterpret_cast<uint32_t*>(&hi));
    }
}

template <int D, int QT>
int launch(const CUtensorMap& tm, const TreeTcParams& p, int ctas, bool join, cudaStream_t stream) {
    constexpr int smem = TreeCfg<D, QT>::kSmem;
    auto kern = attn_tree_tc_kernel<D, QT>;
    static bool configured = false;
    if (!configured) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return TFF_ERR_LAUNCH;
        configured = true;
    }
    const int st = tff_launch_pdl(kern, dim3(ctas), dim3(TreeCfg<D, QT>::kThreads), (size_t)smem, stream, tm, p);
    if (st != TFF_OK || !join) return st;
    return tff_launch_pdl(attn_tree_join_kernel<D, QT>, dim3(ctas, QT * BLOCK_M / JOIN_ROWS), dim3(128), (size_t)0, stream, p);
}

int tiles_at_once(int max_nodes, int nq, int nkv) { return max_nodes * (nq / nkv) > BLOCK_M ? 2 : 1; }

}  // namespace

// Bytes of workspace of a call whose largest request brings max_nodes nodes.
TFF_API long long tff_attention_tree_tc_workspace(int max_nodes, int nq, int nkv, int d) {
    if (max_nodes <= 0 || nkv <= 0 || nq <= 0 || nq % nkv || d <= 0) return 0;
    const long long rows = (long long)tff_num_sms() * 2 * tiles_at_once(max_nodes, nq, nkv) * BLOCK_M;
    return rows * (d + 2) * 4 + (long long)tff_num_sms() * 16;
}

// TFF_ERR_UNSUPPORTED, with nothing launched, for what the general kernel (attention_tree.cu) has to take.
TFF_API int tff_attention_tree_tc(const void* q, const int* q_start, const int* pos_start, const int* parents, const int* block_table,
                                  int table_width, const void* cache, long long cache_pages, int cache_layers, int layer, int page_size,
                                  void* out, int num_tokens, int requests, int max_nodes, int nq, int nkv, int d, float scale, int window,
                                  float softcap, int sink, const float* sink_val, const float* gate, int keep, void* ws,
                                  cudaStream_t stream) {
    if (num_tokens <= 0 || requests <= 0 || max_nodes <= 0) return TFF_OK;
    if (!q || !q_start || !pos_start || !parents || !block_table || !cache || !out || nq <= 0 || nkv <= 0 || nq % nkv || softcap < 0.f ||
        keep < 0 || !ws)
        return TFF_ERR_BAD_ARGUMENT;
    if ((d != 64 && d != 128) || (page_size != 8 && page_size != 16 && page_size != 32 && page_size != 64)) return TFF_ERR_UNSUPPORTED;
    if (cache_pages <= 0 || !(scale > 0.f) || max_nodes > TREE_MAX_NODES) return TFF_ERR_UNSUPPORTED;   // (a positive scale is folded into the exponent)
    if (((uintptr_t)cache & 15) || ((uintptr_t)q & 15) || ((uintptr_t)out & 15) || ((uintptr_t)ws & 15)) return TFF_ERR_UNSUPPORTED;
    const long long rows = cache_pages * cache_layers * 2 * nkv * page_size;
    const int sms = tff_num_sms();
    if (rows >= (1ll << 31) || sms <= 0) return TFF_ERR_UNSUPPORTED;
    CUtensorMap tm;
    if (!tff_tensor_map_kv_groups(cache, rows, d, page_size, nkv, &tm)) return TFF_ERR_DRIVER;
    const int qt = tiles_at_once(max_nodes, nq, nkv);
    TreeTcParams p = {};
    p.q = (const bf16*)q; p.out = (bf16*)out;
    p.q_start = q_start; p.pos_start = pos_start; p.parents = parents; p.block_table = block_table;
    p.requests = requests; p.table_width = table_width; p.cache_layers = cache_layers; p.layer = layer;
    p.page_shift = page_size == 8 ? 3 : page_size == 16 ? 4 : page_size == 32 ? 5 : 6;
    p.nq = nq; p.nkv = nkv; p.window = window > 0 ? window : 0; p.keep = window > 0 ? keep : 0;
    p.least = 4;
    p.scale_log2 = scale * 1.4426950408889634f;
    p.scale_over_cap = softcap > 0.f ? scale / softcap : 0.f;
    p.cap_log2 = softcap > 0.f ? softcap * 1.4426950408889634f : 0.f;
    p.sink = sink; p.sink_val = sink_val; p.gate = gate;
    p.joins = (int4*)ws;
    p.part_o = (float*)((char*)ws + (size_t)sms * 16);
    p.part_ml = p.part_o + (size_t)sms * 2 * qt * BLOCK_M * d;
    p.error_flag = tff_device_error_flag();
    if (p.error_flag == nullptr) return TFF_ERR_LAUNCH;
    if (d == 128) return qt == 2 ? launch<128, 2>(tm, p, sms, true, stream) : launch<128, 1>(tm, p, sms, true, stream);
    return qt == 2 ? launch<64, 2>(tm, p, sms, true, stream) : launch<64, 1>(tm, p, sms, true, stream);
}
