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
//                 (both operands of a product have one type; the sum takes them unrounded: half steps of 2^-9 of a weight that do
//                 not add up one way, an output's error 0.0023 of its norm, 0.0017 of which its own rounding makes)
//   O += P V      tcgen05.mma, M = 128, N = head size, K = 64; P the A operand in tensor memory, V as the pages lie
// O is rescaled when a row's maximum has grown by more than 2^8.  Only blocks with nodes, a window's first and the kept
// tokens' last are masked: a row builds a word of 64 bits from its chain of parents, which lie in shared memory.
//   warps 0-7     softmax, rescale, outputs of the first tile (tensor memory lanes 32 * (warp % 4) ..)
//   warps 8-15    the same for the second tile (QT = 2)
//   then          TMA producer: one box a page into a ring of stages, without a pause between pieces; an issuing warp a tile, which
//                 asks for the queries of the next piece as soon as the products have read the last one's
// What bounds it (cycles counted in the kernel on a B200, heads of 128): with one tile a CTA a block of keys and values, 32 KB, takes 1,150
// cycles, about what the memory gives an SM: 64 trees of 8 nodes behind 200 to 6,000 tokens (32/8 heads) 148 us, 5.4 TB/s.  With two tiles it takes
// 1,590, the products' and exponentials' time: a tree of 64 nodes behind 32,000 tokens (64/8 heads) 83 to 95 us by the clock
// that the power cap leaves.  Around that, a CTA's first scores come 7,500 to 10,000 cycles after its start (2,900 for its place in the line, 3,500 for the
// first keys), and a second piece costs about six blocks: 8 trees of 32 nodes behind 2,048 tokens 25.4 us, 71 MB.  Two tiles leave a thread 96
// registers, and 68 bytes are spilled (heads of 128; 72 with heads of 64, none with one tile).
//   - The queries go ahead of all but two blocks of keys: behind a full ring of every CTA's they came 7,000 cycles later.
//   - A walk counts ``extra`` = 6 units more than its blocks: 3 gives 94.4 / 27.8 us (the long tree / the 8 trees), 5 and 7 92.3, 91.2 / 27.2, 27.3, and
//     12 91.2 / 28.7.
//   - A share has at least ``least`` = 4 units: one request of 32/8 heads behind 800 tokens 11.8 us, with 1 14.3, with 12 16.1; behind 2,048 14.9, 16.8, 16.3.
//   - Short walks are not divided (CudaKernels.TREE_WHOLE_BLOCKS).
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

constexpr int BLOCK_M = 128, BLOCK_N = 64, BARS_PER_TILE = 17, JOIN_ROWS = 16;
constexpr float RESCALE_THRESHOLD = 8.0f;            // in log2 units

struct TreeTcParams {
    bf16* out;
    const int *q_start, *pos_start, *parents, *block_table;
    int tokens, requests, table_width, cache_layers, layer, page_shift, nq, nkv, window, keep, least, extra, whole;
    int group; unsigned group_inverse;               // query heads a kv head, and what a row number is multiplied by for its node
    int tile_rows;                                   // of 128: whole nodes
    int pages, no_group;                             // of the cache; a group of rows behind its last, which reads as zeros
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

// A box of tff_tensor_map_heads: 64 columns (of a half) of the heads of a group, of a tile's nodes.
__device__ __forceinline__ void tma_load_queries(uint32_t dst, const CUtensorMap* tm, uint32_t bar, int half, int kvh, int token) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %3, %4, %5, %6}], [%2];"
        ::"r"(dst), "l"(tm), "r"(bar), "r"(0), "r"(half), "r"(kvh), "r"(token) : "memory");
}

template <int D, int QT>
struct TreeCfg {
    static constexpr int kQBytes = BLOCK_M * D * 2;                 // [64-column half][128 rows][128 B]
    static constexpr int kStageBytes = BLOCK_N * 2 * D * 2;
    static constexpr int kStages = D > 64 ? 5 : 8;
    static constexpr int kExchange = QT * 2 * BLOCK_M * 4;          // a float of every row from either group
    static constexpr int kParents = TREE_MAX_NODES * 2;
    static constexpr int kBars = 2 * kStages + BARS_PER_TILE * QT;
    static constexpr int kSmem = QT * kQBytes + kStages * kStageBytes + kExchange + kParents + 8 * kBars + 8 + 2 * 76;
    static constexpr int kThreads = (8 * QT + 1 + QT) * 32;
    static_assert(kSmem <= 227 * 1024, "shared memory of the tree attention kernel");
};

// A request's walk: the blocks of 64 keys that its rows see, for each of its tiles.
struct Walk {
    int q0 = 0, nodes = 0, ctx = 0, lo = 0, tiles = 0, count = 0;
    __device__ __forceinline__ void read(const TreeTcParams& p, int b, int tile_rows) {
        q0 = p.q_start[b];
        nodes = max(0, min(min(p.q_start[b + 1], p.tokens) - q0, TREE_MAX_NODES));      // (no rows behind the step's)
        ctx = p.pos_start[b];
        lo = p.window > 0 ? max(0, ctx - p.window + 1) : 0;         // the first position that a root sees
        tiles = (nodes * p.group + tile_rows - 1) / tile_rows;
        count = tiles > 0 ? keys(p.keep).count : 0;
    }
    __device__ __forceinline__ int hi() const { return ctx + nodes - 1; }
    __device__ __forceinline__ KeyWalk keys(int keep) const { return KeyWalk(keep, BLOCK_N, lo / BLOCK_N, hi() / BLOCK_N); }
};

// How a line of ``all`` units is shared out: the first ``rest`` CTAs have one unit more than the others.
struct Shares {
    int ctas, each, rest;
    __device__ __forceinline__ Shares(int all, int least) {
        ctas = min((int)gridDim.x, max(1, all / least));
        each = all / ctas;
        rest = all - each * ctas;
    }
    __device__ __forceinline__ int begin(int cta) const { return cta >= ctas ? each * ctas + rest : cta * each + min(cta, rest); }
    __device__ __forceinline__ int owner(int unit) const {
        const int more = rest * (each + 1);
        return unit < more ? unit / (each + 1) : rest + (unit - more) / each;
    }
};

// A CTA's share, piece by piece.  A walk has ``extra`` units ahead of its blocks, for what a piece costs beside them: a CTA of
// several pieces has fewer blocks.  ``whole``: a share is the walks that begin in it.
struct Pieces {
    int left = 0;                                    // units of the share behind the present piece
    int b = 0, kvh = 0, tile = 0, at = 0, nb = 0;    // the piece: request, kv head, tile; its first block of the walk, its blocks
    int unit = 0;                                    // of the walk, behind the present piece
    Walk w;
    // A warp's, with all its lanes; returns the line's units and the share's first one.
    __device__ __forceinline__ int2 start(const TreeTcParams& p, int rows) {
        const int lane = threadIdx.x & 31;
        Walk v;
        auto sum_of = [&](int r0) -> int {           // inclusive sums of 32 requests' units
            v = Walk();
            if (r0 + lane < p.requests) v.read(p, r0 + lane, rows);
            int s = v.count > 0 ? v.tiles * (v.count + p.extra) : 0;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const int before = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s += before;
            }
            return s;
        };
        const int head = sum_of(0);
        int line = __shfl_sync(0xffffffffu, head, 31);                 // units a kv head
        for (int r0 = 32; r0 < p.requests; r0 += 32) line += __shfl_sync(0xffffffffu, sum_of(r0), 31);
        const Shares sh(line * p.nkv, p.least);
        const int first = sh.begin(blockIdx.x);
        left = sh.begin(blockIdx.x + 1) - first;
        if (left <= 0) { left = 0; return make_int2(line * p.nkv, first); }
        kvh = first / line;
        int rest = first - kvh * line;
        for (int r0 = 0; r0 < p.requests; r0 += 32) {
            const int s = r0 == 0 && p.requests <= 32 ? head : sum_of(r0);
            const unsigned behind = __ballot_sync(0xffffffffu, rest < s);
            if (behind) {
                const int src = __ffs(behind) - 1;
                b = r0 + src;
                const int before = __shfl_sync(0xffffffffu, s, max(src - 1, 0));
                rest -= src > 0 ? before : 0;
                w.q0 = __shfl_sync(0xffffffffu, v.q0, src); w.nodes = __shfl_sync(0xffffffffu, v.nodes, src);
                w.ctx = __shfl_sync(0xffffffffu, v.ctx, src); w.lo = __shfl_sync(0xffffffffu, v.lo, src);
                w.tiles = __shfl_sync(0xffffffffu, v.tiles, src); w.count = __shfl_sync(0xffffffffu, v.count, src);
                break;
            }
            rest -= __shfl_sync(0xffffffffu, s, 31);
        }
        const int span = w.count + p.extra;
        tile = rest / span;
        unit = rest - tile * span;
        if (p.whole && unit > 0) {                   // (that walk is another CTA's)
            left -= span - unit;
            unit = span;
        }
        at = max(0, unit - p.extra);
        return make_int2(line * p.nkv, first);
    }
    // The next piece; false behind the last.
    __device__ __forceinline__ bool next(const TreeTcParams& p, int rows) {
        if (left <= 0) return false;
        if (unit == w.count + p.extra) {
            unit = 0;
            if (++tile == w.tiles) {
                tile = 0;
                do {
                    if (++b == p.requests) { b = 0; ++kvh; }
                    w.read(p, b, rows);
                } while (w.count == 0);
            }
        }
        const int end = p.whole ? w.count + p.extra : min(unit + left, w.count + p.extra);
        at = max(0, unit - p.extra);
        nb = max(0, end - p.extra) - at;
        left -= end - unit;
        unit = end;
        return nb > 0;                               // (none: the share ends ahead of the walk's first block)
    }
    __device__ __forceinline__ bool all() const { return at == 0 && nb == w.count; }
};

// A piece that the softmax warps are at, in shared memory: they have no registers for it.
struct Present {
    Pieces p;
    KeyWalk keys;
    int go, stage, fresh;                            // whether there is a piece; the stage of its first block; whether its request is another than before
};

// A row's node.
__device__ __forceinline__ int node_of(const TreeTcParams& p, int row) { return p.group == 1 ? row : (int)__umulhi((unsigned)row, p.group_inverse); }

// below(k): the first k of 64 bits.
__device__ __forceinline__ uint64_t below(int k) { return k <= 0 ? 0ull : k >= 64 ? ~0ull : (1ull << k) - 1; }

// QT: query tiles a CTA walks with at once, two where some request has more rows than one.
template <int D, int QT>
__global__ void __launch_bounds__(TreeCfg<D, QT>::kThreads, 1)
attn_tree_tc_kernel(const __grid_constant__ CUtensorMap tm_cache, const __grid_constant__ CUtensorMap tm_q, const TreeTcParams p) {
    using Cfg = TreeCfg<D, QT>;
    constexpr int HALVES = D / 64, CH = D / 8;                   // 64-column halves, 16-byte chunks of a key or value row
    constexpr int NSTAGES = Cfg::kStages, STAGE_BYTES = Cfg::kStageBytes;
    constexpr int GROUP = 2 * HALVES * 1024;                     // of a stage, [8 keys][K, V][half]: from 8 keys to the next 8
    constexpr int V_AT = HALVES * 1024;
    constexpr int ROWS = QT * BLOCK_M, SOFT = QT * 256;          // places of a piece's rows, softmax threads
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
    auto q_free = [&](int x) { return tile_bar(x, 16); };
    volatile uint32_t* tmem_slot = (volatile uint32_t*)(smem + BARS_AT + 8 * Cfg::kBars);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
    Present* present = (Present*)(tmem_slot + 2);                // [2]: the piece, and the next one
    static_assert(sizeof(Present) <= 76, "a piece's place");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = p.group, rows = QT * p.tile_rows;

    if (tid == 0) {
        for (int s = 0; s < NSTAGES; ++s) { mbar_init(kv_full(s), 1); mbar_init(kv_empty(s), QT); }
        for (int x = 0; x < QT; ++x) {
            for (int g = 0; g < 2; ++g) {
                mbar_init(s_full(x, g), 1); mbar_init(p_full(x, g), 4); mbar_init(pv_done(x, g), 1);
                for (int q = 0; q < 4; ++q) mbar_init(ref_bar(x, g, q), 1);
            }
            mbar_init(s_free(x), 4); mbar_init(q_ready(x), 1); mbar_init(q_free(x), 1);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tm_cache) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tm_q) : "memory");
    }
    if (warp == ISSUE_WARP) tmem_alloc(smem_u32((const void*)tmem_slot), TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    constexpr uint32_t tmem_base = 0;
    pdl_launch_dependents();
    pdl_wait();
    Pieces piece;                                                // (the other softmax warps read it from shared memory)
    int2 line = make_int2(0, 0);
    if (warp == 0 || warp >= LOAD_WARP) line = piece.start(p, rows);

    if (warp == LOAD_WARP) {
        // ------------------------------------------------------------ TMA producer
        // the walk that this share's first piece ends, if others began it: joined by the second kernel
        int4 join = make_int4(-1, 0, 0, 0);
        int begun = -1;
        if (piece.left > 0 && piece.at > 0 && piece.w.count - piece.at <= piece.left) {
            join = make_int4(piece.b, piece.kvh, piece.tile, 0);
            begun = line.y - piece.unit + p.extra;           // (the unit of the walk's first block)
        }
        const int ppb = BLOCK_N >> p.page_shift;
        int s = 0;
        uint32_t round = 0;
        bool ok = true;
        while (ok && piece.next(p, rows)) {
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
                // the first queries are on their way before more than two blocks are asked for: every CTA begins with both
                if (round == 0 && i == 2 && s == 2 && !(ok = mbar_wait_warp(q_ready(0), 0, abort_flag))) break;
                const int first = walk.block(piece.at + i) * BLOCK_N >> p.page_shift;       // (a block's pages lie in one run of 32)
                if (first >> 5 != chunk) {
                    held = first >> 5 == chunk + 1 && chunk >= 0 ? ahead : entry(first >> 5);
                    chunk = first >> 5;
                    ahead = entry(chunk + 1);
                }
                // (a page that the table lacks reads as zeros)
                const bool valid = lane >= (first & 31) && lane < (first & 31) + ppb && chunk * 32 + lane <= table_end;
                const unsigned mask = __ballot_sync(0xffffffffu, valid);
                if (lane == 0) mbar_expect_tx(kv_full(s), (uint32_t)__popc(mask) * (uint32_t)(GROUP << (p.page_shift - 3)));
                __syncwarp();
                if (valid) {
                    const long long row = ((((long long)held * p.cache_layers + p.layer) * 2) * p.nkv + piece.kvh) << p.page_shift;
                    tma_load_5d(sKV + s * STAGE_BYTES + (uint32_t)((lane - (first & 31)) * (GROUP << (p.page_shift - 3))), &tm_cache, kv_full(s),
                                (unsigned)held < (unsigned)p.pages ? (int)(row >> 3) : p.no_group);
                }
                if (++s == NSTAGES) { s = 0; ++round; }
            }
        }
        if (!p.whole && lane == 0) {
            if (begun >= 0) join.w = Shares(line.x, p.least).owner(begun);
            p.joins[blockIdx.x] = join;
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
            uint32_t phase_p = 0;                                  // of p_full, a bit a group
            int st = 0, st_pv = 0;                                 // stages of S(n) and of PV(n - 2)
            while (ok && piece.next(p, rows)) {
                if (piece.tile * rows + x * p.tile_rows >= piece.w.nodes * G) {
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
                // the queries, once the products of the piece before have read theirs; padding and rows of other requests among them
                // make rows of their own, which are not stored
                ok = mbar_wait_warp(q_free(x), phase_q ^ 1, abort_flag);
                if (!ok) break;
                if (lane == 0) {
                    mbar_expect_tx(q_ready(x), (uint32_t)(HALVES * p.tile_rows * 128));
                    const int token = piece.w.q0 + (piece.tile * QT + x) * (p.tile_rows / G);
#pragma unroll
                    for (int h = 0; h < HALVES; ++h)
                        tma_load_queries(sQ + x * Cfg::kQBytes + h * (BLOCK_M * 128), &tm_q, q_ready(x), h, piece.kvh, token);
                }
                __syncwarp();
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
                        if (n == piece.nb - 1) umma_commit_elected(q_free(x));
                        if (++st == NSTAGES) { st = 0; phase ^= 1; }
                    }
                    const int j = n - 2;
                    if (j >= 0) {
                        ok = mbar_wait_warp(p_full(x, j & 1), phase_p >> (j & 1) & 1u, abort_flag);   // P(j) is in tensor memory
                        if (!ok) break;
                        phase_p ^= 1u << (j & 1);
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
        bool ok = true;
        if (tid == 0) {
            present->go = piece.next(p, rows);
            present->p = piece;
            present->keys = piece.w.keys(p.keep);
            present->stage = 0;
            present->fresh = 1;
        }
        soft_sync();
        for (const Present* now = present;; now = present + (now == present)) {
            if (!now->go) break;
            auto row_of = [&]() { return (now->p.tile * QT + x) * p.tile_rows + r; };
            auto exists = [&]() { return r < p.tile_rows && row_of() < now->p.w.nodes * G; };
            const int tok = node_of(p, row_of());
            const bool tile_active = row_of() - r < now->p.w.nodes * G;
            if (now->fresh) {
                const int nodes = now->p.w.nodes;
                for (int i = tid; i < nodes; i += SOFT) parent[i] = tree_parent(__ldcg(p.parents + now->p.w.q0 + i), i);
                soft_sync();
            }
            const int depth = exists() ? tree_depth(parent, tok) : -1;         // (-1: a row of no node that is there)
            if (warp == 7) {                                       // the next piece, while the first products run (block 1 is this warp's first)
                Pieces next = now->p;
                const bool go = next.next(p, rows);
                Present* to = present + (now == present);
                if (lane == 0) {
                    to->fresh = next.b != now->p.b;
                    to->stage = (now->stage + now->p.nb) % NSTAGES;
                    to->go = go;
                    to->p = next;
                    to->keys = next.w.keys(p.keep);
                }
                __syncwarp();
            }
            const int tail = now->p.w.ctx - BLOCK_N;               // blocks that begin behind it hold nodes
            int n_first = (now->p.at + g) * BLOCK_N;
            float m_used = -INFINITY, l = 0.f;
            const int nb_x = tile_active ? now->p.nb : 0;
            for (int j = g; j < nb_x && ok; j += 2, n_first += 2 * BLOCK_N) {
                ok = mbar_wait_warp(s_full(x, g), n_own, abort_flag);
                if (!ok) break;
                tc_fence_after();
                if (p.window > 0) n_first = now->keys.block(now->p.at + j) * BLOCK_N;
                // Masked or capped scores are written back over the raw ones, so that the pass below is the same for every block.
                // Rows that are not there are not stored: they need no mask.
                const bool some_nodes = n_first > tail;
                bool masked = some_nodes;
                if (p.window > 0 && !some_nodes)
                    masked = !__all_sync(0xffffffffu, depth < 0 || n_first > now->p.w.ctx + depth - p.window || n_first + BLOCK_N <= p.keep);
                if (masked || p.cap_log2 > 0.f) {
                    uint64_t seen = ~0ull;
                    if (masked && depth >= 0) {
                        const int ctx = now->p.w.ctx;
                        int pos = ctx + depth;
                        const int lo = p.window > 0 ? pos - p.window + 1 : 0;
                        seen = below(ctx - n_first) & (~below(lo - n_first) | below(p.keep - n_first));
                        if (some_nodes) {
                            for (int a = tok; a >= 0 && ctx + a >= n_first; a = parent[a], --pos)
                                if (ctx + a < n_first + BLOCK_N && (pos >= lo || pos < p.keep)) seen |= 1ull << (ctx + a - n_first);
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
                if (some_nodes || (p.window > 0 && now->keys.ragged(now->p.at + j))) {      // (the last block holds nodes)
                    // value rows that no row may see (behind the last node, between the kept ones and the first window, of
                    // padding) are cleared, since slots and unfetched shared memory may hold anything; the warps of both tiles
                    // do it (the same zeros), so that each tile's products wait for its own warps only
                    uint8_t* rows = gKV + ((now->stage + j) % NSTAGES) * STAGE_BYTES + V_AT;
                    const int ctx = now->p.w.ctx, hi = now->p.w.hi(), lo = now->p.w.lo;
                    auto unseen = [&](int n) { return n > hi || (n < lo && n >= p.keep) || (n >= ctx && tree_depth(parent, n - ctx) < 0); };
                    const unsigned first = __ballot_sync(0xffffffffu, unseen(n_first + lane)), second = __ballot_sync(0xffffffffu, unseen(n_first + 32 + lane));
                    // a quarter of the rows a warp of the group, two rows at a time
#pragma unroll 1
                    for (int i = 0; i < BLOCK_N / 4; i += 32 / CH) {
                        const int kr = q * (BLOCK_N / 4) + i + lane / CH, c = lane % CH;
                        if ((kr < 32 ? first >> kr : second >> (kr - 32)) & 1u)
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
                if (now->p.all()) {
                    const int t = now->p.w.q0 + tok, head = now->p.kvh * G + (row_of() - tok * G);
                    if (p.sink && l > 0.f) l += exp2f(attn_sink_log2(p.sink_val, head) - m_used);       // a key without a value
                    const bool some = depth >= 0 && l > 0.f;       // (a padding row's sums may be anything)
                    float inv = some ? 1.f / l : 0.f;
                    if (p.gate && some) inv *= __ldcg(p.gate + (size_t)t * p.nq + head);
                    uint4* to = reinterpret_cast<uint4*>(p.out + ((size_t)t * p.nq + head) * D + g * (D / 2));
#pragma unroll
                    for (int c0 = 0; c0 < D / 2; c0 += 32) {
                        uint32_t v[32];
                        tmem_ld16(t_o + g * (D / 2) + c0, v);
                        tmem_ld16(t_o + g * (D / 2) + c0 + 16, v + 16);
                        tmem_ld_wait();
                        if (!exists()) continue;
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            uint32_t wd[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                __nv_bfloat162 b2 = __floats2bfloat162_rn(__uint_as_float(v[8 * c + 2 * i]) * inv, __uint_as_float(v[8 * c + 2 * i + 1]) * inv);
                                wd[i] = some ? *reinterpret_cast<uint32_t*>(&b2) : 0u;
                            }
                            to[c0 / 8 + c] = make_uint4(wd[0], wd[1], wd[2], wd[3]);
                        }
                    }
                } else {
                    // slot 0 of the CTA: a piece of a walk that another one began; slot 1: of one that this one begins
                    const size_t slot = ((size_t)blockIdx.x * 2 + (now->p.at > 0 ? 0 : 1)) * ROWS + x * BLOCK_M + q * 32;
                    if (g == 0 && exists())
                        *reinterpret_cast<float2*>(p.part_ml + (slot + lane) * 2) = make_float2(m_used, depth >= 0 ? l : 0.f);
                    // four columns of a row at a time, those of all rows side by side: what 32 lanes write is one run
                    float4* to = reinterpret_cast<float4*>(p.part_o) + (slot / ROWS) * (D / 4 * ROWS) + slot % ROWS + lane;
#pragma unroll
                    for (int c0 = 0; c0 < D / 8; c0 += 8) {
                        uint32_t v[32];
                        tmem_ld16(t_o + g * (D / 2) + c0 * 4, v);
                        tmem_ld16(t_o + g * (D / 2) + c0 * 4 + 16, v + 16);
                        tmem_ld_wait();
                        if (exists()) {
#pragma unroll
                            for (int c = 0; c < 8; ++c)
                                to[(g * (D / 8) + c0 + c) * ROWS] = make_float4(__uint_as_float(v[4 * c]), __uint_as_float(v[4 * c + 1]),
                                                                                __uint_as_float(v[4 * c + 2]), __uint_as_float(v[4 * c + 3]));
                        }
                    }
                }
            }
            tc_fence_before();
            soft_sync();                                           // O, the parents and the piece may be written again
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

// Joins the pieces of the walks that are more than one share's: a block takes JOIN_ROWS rows of the walk that ends in share
// blockIdx.x; eight threads a row, each an eighth of its columns.  Neighbouring threads have neighbouring rows, whose fours of columns lie
// side by side (with neighbouring columns instead, at 16 bytes of a line each, the loads came at a quarter of the rate).  Four pieces'
// loads together, none of them twice: 8 trees of 32 nodes behind 2,048 tokens 25.4 us; eight together 27, the last one repeated in
// place of the pieces that are not there 25.9.
template <int D, int QT>
__global__ void __launch_bounds__(JOIN_ROWS * 8) attn_tree_join_kernel(const TreeTcParams p) {
    constexpr int ROWS = QT * BLOCK_M, FOURS = D / 32, AHEAD = 4;
    pdl_launch_dependents();
    pdl_wait();
    const int4 join = __ldcg(p.joins + blockIdx.x);                // request, kv head, tile, the first share
    if (join.x < 0) return;
    const int b = join.x, last = blockIdx.x;
    const int row = blockIdx.y * JOIN_ROWS + threadIdx.x % JOIN_ROWS, c = threadIdx.x / JOIN_ROWS * FOURS;
    const int R = (join.z * QT + row / BLOCK_M) * p.tile_rows + row % BLOCK_M;
    const int q0 = p.q_start[b], rows_total = min(min(p.q_start[b + 1], p.tokens) - q0, TREE_MAX_NODES) * p.group;
    if (row % BLOCK_M >= p.tile_rows || R >= rows_total) return;
    float m = -INFINITY, l = 0.f;
    float4 o[FOURS];
#pragma unroll
    for (int k = 0; k < FOURS; ++k) o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = join.w; s0 <= last; s0 += AHEAD) {
        float2 ml[AHEAD];
        float4 v[AHEAD][FOURS];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int s = s0 + i;
            if (s > last) continue;
            const size_t slot = (size_t)s * 2 + (s == join.w ? 1 : 0);
            ml[i] = __ldcg(reinterpret_cast<const float2*>(p.part_ml) + slot * ROWS + row);
#pragma unroll
            for (int k = 0; k < FOURS; ++k) v[i][k] = __ldcg(reinterpret_cast<const float4*>(p.part_o) + (slot * (D / 4) + c + k) * ROWS + row);
        }
        // (a piece that the row saw nothing of counts for nothing)
        float most = m;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) if (s0 + i <= last && ml[i].y > 0.f) most = fmaxf(most, ml[i].x);
        const float f0 = m == -INFINITY ? 0.f : exp2f(m - most);
        l *= f0;
#pragma unroll
        for (int k = 0; k < FOURS; ++k) { o[k].x *= f0; o[k].y *= f0; o[k].z *= f0; o[k].w *= f0; }
        m = most;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (s0 + i > last || !(ml[i].y > 0.f)) continue;
            const float f = exp2f(ml[i].x - m);
            l = fmaf(ml[i].y, f, l);
#pragma unroll
            for (int k = 0; k < FOURS; ++k) {
                o[k].x = fmaf(v[i][k].x, f, o[k].x); o[k].y = fmaf(v[i][k].y, f, o[k].y);
                o[k].z = fmaf(v[i][k].z, f, o[k].z); o[k].w = fmaf(v[i][k].w, f, o[k].w);
            }
        }
    }
    const int tok = node_of(p, R), t = q0 + tok, h = join.y * p.group + (R - tok * p.group);
    float inv = 0.f;
    if (l > 0.f) inv = (p.gate ? __ldcg(p.gate + (size_t)t * p.nq + h) : 1.f) / (p.sink ? l + exp2f(attn_sink_log2(p.sink_val, h) - m) : l);
    uint4* to = reinterpret_cast<uint4*>(p.out + ((size_t)t * p.nq + h) * D + c * 4);
    auto pair = [&](float a, float b2) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a * inv, b2 * inv);
        return l > 0.f ? *reinterpret_cast<const uint32_t*>(&v) : 0u;
    };
#pragma unroll
    for (int k = 0; k < FOURS; k += 2)
        to[k / 2] = make_uint4(pair(o[k].x, o[k].y), pair(o[k].z, o[k].w), pair(o[k + 1].x, o[k + 1].y), pair(o[k + 1].z, o[k + 1].w));
}

template <int D, int QT>
int launch(const CUtensorMap& tm, const CUtensorMap& tq, const TreeTcParams& p, int ctas, int rows, cudaStream_t stream) {
    constexpr int smem = TreeCfg<D, QT>::kSmem;
    auto kern = attn_tree_tc_kernel<D, QT>;
    static bool configured = false;
    if (!configured) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return TFF_ERR_LAUNCH;
        configured = true;
    }
    const int st = tff_launch_pdl(kern, dim3(ctas), dim3(TreeCfg<D, QT>::kThreads), (size_t)smem, stream, tm, tq, p);
    if (st != TFF_OK || p.whole) return st;
    return tff_launch_pdl(attn_tree_join_kernel<D, QT>, dim3(ctas, (rows + JOIN_ROWS - 1) / JOIN_ROWS), dim3(JOIN_ROWS * 8), (size_t)0, stream, p);
}

}  // namespace

// TFF_ERR_UNSUPPORTED, with nothing launched, for what the general kernel (attention_tree.cu) has to take.  A CTA's share has at least
// ``least`` units, a walk ``extra`` of them ahead of its blocks; ``whole``: no walk is divided, and there is no second kernel.  ``ws``: an
// SM has 4 words and room for two pieces of 128 rows (256 where some request may have more rows than a tile) of d + 2 floats.
TFF_API int tff_attention_tree_tc(const void* q, const int* q_start, const int* pos_start, const int* parents, const int* block_table,
                                  int table_width, const void* cache, long long cache_pages, int cache_layers, int layer, int page_size,
                                  void* out, int num_tokens, int requests, int max_nodes, int nq, int nkv, int d, float scale, int window,
                                  float softcap, int sink, const float* sink_val, const float* gate, int keep, int least, int extra, int whole, void* ws,
                                  long long ws_floats, cudaStream_t stream) try {
    if (num_tokens <= 0 || requests <= 0 || max_nodes <= 0) return TFF_OK;
    if (!q || !q_start || !pos_start || !parents || !block_table || !cache || !out || nq <= 0 || nkv <= 0 || nq % nkv || softcap < 0.f ||
        keep < 0 || least <= 0 || extra < 0 || extra > 64 || table_width <= 0 || (!whole && !ws))
        return TFF_ERR_BAD_ARGUMENT;
    if ((d != 64 && d != 128) || (page_size != 8 && page_size != 16 && page_size != 32 && page_size != 64)) return TFF_ERR_UNSUPPORTED;
    if (nq / nkv > BLOCK_M) return TFF_ERR_UNSUPPORTED;          // a tile holds whole nodes
    if (cache_pages <= 0 || !(scale > 0.f) || max_nodes > TREE_MAX_NODES) return TFF_ERR_UNSUPPORTED;   // (a positive scale is folded into the exponent)
    if (((uintptr_t)cache & 15) || ((uintptr_t)q & 15) || ((uintptr_t)out & 15) || ((uintptr_t)ws & 15)) return TFF_ERR_UNSUPPORTED;
    const long long rows = cache_pages * cache_layers * 2 * nkv * page_size;
    const int sms = tff_num_sms();
    if (rows >= (1ll << 31) || sms <= 0) return TFF_ERR_UNSUPPORTED;
    const int group = nq / nkv, tile_rows = BLOCK_M / group * group;
    const int qt = (long long)max_nodes * group > tile_rows ? 2 : 1;
    // (the line's units are counted in 32 bits)
    if ((((long long)table_width * page_size + TREE_MAX_NODES) / BLOCK_N + 2 + extra) * requests * nkv * ((long long)TREE_MAX_NODES * group / tile_rows + 1) >= (1ll << 31))
        return TFF_ERR_UNSUPPORTED;
    if (!whole && ws_floats < (long long)sms * (4 + 2 * qt * BLOCK_M * (d + 2))) return TFF_ERR_BAD_ARGUMENT;
    CUtensorMap tm, tq;
    if (!tff_tensor_map_kv_groups(cache, rows, d, page_size, nkv, &tm)) return TFF_ERR_DRIVER;
    if (!tff_tensor_map_heads(q, num_tokens, nkv, group, d, tile_rows / group, &tq)) return TFF_ERR_DRIVER;
    TreeTcParams p = {};
    p.out = (bf16*)out;
    p.q_start = q_start; p.pos_start = pos_start; p.parents = parents; p.block_table = block_table;
    p.tokens = num_tokens; p.requests = requests; p.table_width = table_width; p.cache_layers = cache_layers; p.layer = layer;
    p.page_shift = page_size == 8 ? 3 : page_size == 16 ? 4 : page_size == 32 ? 5 : 6;
    p.nq = nq; p.nkv = nkv; p.window = window > 0 ? window : 0; p.keep = window > 0 ? keep : 0;
    p.least = least; p.extra = extra; p.whole = whole;
    p.pages = (int)(cache_pages < 0x7fffffff ? cache_pages : 0x7fffffff); p.no_group = (int)(rows >> 3);
    p.group = group; p.tile_rows = tile_rows; p.group_inverse = (unsigned)(((1ull << 32) + p.group - 1) / p.group);
    p.scale_log2 = scale * 1.4426950408889634f;
    p.scale_over_cap = softcap > 0.f ? scale / softcap : 0.f;
    p.cap_log2 = softcap > 0.f ? softcap * 1.4426950408889634f : 0.f;
    p.sink = sink; p.sink_val = sink_val; p.gate = gate;
    p.joins = (int4*)ws;
    p.part_o = (float*)((char*)ws + (size_t)sms * 16);
    p.part_ml = p.part_o + (size_t)sms * 2 * qt * BLOCK_M * d;
    p.error_flag = tff_device_error_flag();
    if (p.error_flag == nullptr) return TFF_ERR_LAUNCH;
    const int rows_at_most = qt == 2 ? 2 * BLOCK_M : max_nodes * group;
    if (d == 128) return qt == 2 ? launch<128, 2>(tm, tq, p, sms, rows_at_most, stream) : launch<128, 1>(tm, tq, p, sms, rows_at_most, stream);
    return qt == 2 ? launch<64, 2>(tm, tq, p, sms, rows_at_most, stream) : launch<64, 1>(tm, tq, p, sms, rows_at_most, stream);
} catch (...) {                                                  // (the tensor maps' tables: no memory for another)
    return TFF_ERR_DRIVER;
}
