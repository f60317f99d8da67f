// What a step that checks a tree of drafted tokens does with its result: the walk down the tree along the tokens that were
// drawn, and the accepted nodes' keys and values moved to where the next step expects them.
//
// Node i of request b is row q_start[b] + i of the step and has cache slot pos_start[b] + i; its parent is an earlier node,
// node 0 (the token drawn last, parent -1) the root.
//
// Measured in a captured run: the walk 1.7 us for one tree of 8 nodes, 2.6 for 64 of 64 (a launch and two trips to memory; 11 to 16
// votes of the warp are a fraction of that); the move 1.9 us for one path in 8 layers, 14.6 for 64 paths in 36 layers of 8 heads of 128 (60 MB
// read and written, 4.1 TB/s).  Registers for four CTAs an SM count: 16.9 with 80 of them; 18.9 with the places divided in 64 bits, 25 with
// four loads ahead and the places looked up by every thread, 16.4 with two items a thread.
#include "common.cuh"

namespace {

constexpr int MAX_NODES = 256;                       // of a request's tree
constexpr int PER_LANE = MAX_NODES / 32;

// From the root on, the path goes to the first child whose token is the one that was drawn behind the node; path[b] gets its
// nodes, emitted[b] the tokens drawn behind them (the request's new tokens), -1 beyond, count[b] their number.  A warp a
// request: a lane holds the parents and tokens of every 32nd node in registers, so that a step of the walk is a
// vote a 32 nodes.
__global__ void __launch_bounds__(32)
accept_tree_kernel(const int* tokens, const int* parents, const int* drawn, const int* q_start, int num_tokens,
                   int* __restrict__ path, int* __restrict__ emitted, int* __restrict__ count, int width) {
    __shared__ int draws[MAX_NODES];
    pdl_launch_dependents();
    pdl_wait();
    const int b = blockIdx.x, lane = threadIdx.x;
    const int q0 = __ldcg(q_start + b), n = min(min(__ldcg(q_start + b + 1), num_tokens) - q0, MAX_NODES);
    int up[PER_LANE], word[PER_LANE];
#pragma unroll
    for (int u = 0; u < PER_LANE; ++u) {
        const int i = u * 32 + lane;
        up[u] = -2; word[u] = -1;
        if (i < n) {
            up[u] = __ldcg(parents + q0 + i);
            word[u] = __ldcg(tokens + q0 + i);
            draws[i] = __ldcg(drawn + q0 + i);
            if (up[u] >= i) up[u] = -2;              // a parent is an earlier node
        }
    }
    __syncwarp();
    int at = __shfl_sync(0xffffffffu, up[0], 0) == -1 ? 0 : -1, k = 0;
    while (at >= 0 && k < width) {
        const int t = draws[at];
        if (lane == 0) { path[(size_t)b * width + k] = at; emitted[(size_t)b * width + k] = t; }
        ++k;
        int next = -1;
#pragma unroll
        for (int u = 0; u < PER_LANE; ++u) {
            const unsigned hit = __ballot_sync(0xffffffffu, up[u] == at && word[u] == t);
            if (hit && next < 0) next = u * 32 + __ffs(hit) - 1;
        }
        at = next;
    }
    for (int i = k + lane; i < width; i += 32) { path[(size_t)b * width + i] = -1; emitted[(size_t)b * width + i] = -1; }
    if (lane == 0) count[b] = k;
}

constexpr int KEEP_THREADS = 256, AHEAD = 8;

struct KeepParams {
    char* cache; long long page_bytes, layer_bytes, plane_bytes, head_bytes;
    int pages; unsigned layers, planes, heads, page_size, row_bytes;
    const int *pos_start, *block_table; unsigned table_width;
    const int *path, *count; int width;
};

// Slot pos + path[j] -> slot pos + j, for j < count, in every layer, plane and head.  A thread takes one V of a row for all j in
// order, eight loads ahead of their stores: a path's nodes ascend, so what is stored at j is never read at a later j.  The slots'
// places in a (layer, plane, head) are worked out once a block.
template <typename V>
__global__ void __launch_bounds__(KEEP_THREADS) keep_path_kernel(const KeepParams p) {
    __shared__ long long from[AHEAD], to[AHEAD];     // -1: nothing to move
    __shared__ int kept;
    pdl_launch_dependents();
    pdl_wait();
    const int b = blockIdx.y;
    // The first warp alone asks for what all blocks of a request read, all at once.
    int pos = 0, n = 0, next = 0;
    if (threadIdx.x < 32) {
        const int j = 1 + threadIdx.x % AHEAD;
        n = min(__ldcg(p.count + b), p.width);
        pos = __ldcg(p.pos_start + b);
        next = j < p.width ? __ldcg(p.path + (size_t)b * p.width + j) : j;
        if (threadIdx.x == 0) kept = n;
    }
    const unsigned row = p.row_bytes / (unsigned)sizeof(V);
    const unsigned item = blockIdx.x * KEEP_THREADS + threadIdx.x;
    const unsigned r = item / row, plane = r / p.heads, layer = plane / p.planes;
    char* base = layer < p.layers ? p.cache + layer * p.layer_bytes + (plane - layer * p.planes) * p.plane_bytes + (r - plane * p.heads) * p.head_bytes +
                 (item - r * row) * (unsigned)sizeof(V) : nullptr;
    for (int j0 = 1;; j0 += AHEAD) {
        if (threadIdx.x < 2 * AHEAD) {
            const int j = j0 + threadIdx.x % AHEAD;
            if (j0 > 1 && j < n) next = __ldcg(p.path + (size_t)b * p.width + j);
            const int i = j < n ? next : j;
            const long long at = (long long)pos + (threadIdx.x < AHEAD ? i : j);
            const unsigned entry = (unsigned)at / p.page_size;           // (at least 0, and below 2^32)
            long long place = -1;
            if (i != j && i >= 0 && at >= 0 && entry < p.table_width) {
                const int page = __ldcg(p.block_table + (size_t)b * p.table_width + entry);
                if (page >= 0 && page < p.pages) place = page * p.page_bytes + (long long)((unsigned)at - entry * p.page_size) * p.row_bytes;
            }
            (threadIdx.x < AHEAD ? from : to)[threadIdx.x % AHEAD] = place;
        }
        __syncthreads();
        V v[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
            if (from[u] >= 0 && to[u] >= 0 && base) v[u] = __ldcg((const V*)(base + from[u]));
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
            if (from[u] >= 0 && to[u] >= 0 && base) *(V*)(base + to[u]) = v[u];
        if (j0 + AHEAD >= kept) break;
        __syncthreads();                             // (the slots have been read)
    }
}

}  // namespace

TFF_API int tff_accept_tree(const int* tokens, const int* parents, const int* drawn, const int* q_start, int num_tokens,
                            int requests, int* path, int* emitted, int* count, int width, cudaStream_t stream) {
    if (requests <= 0) return TFF_OK;
    if (!q_start || !path || !emitted || !count || width <= 0 || (num_tokens > 0 && (!tokens || !parents || !drawn)))
        return TFF_ERR_BAD_ARGUMENT;
    return tff_launch_pdl(accept_tree_kernel, dim3(requests), dim3(32), (size_t)0, stream, tokens, parents, drawn, q_start, num_tokens,
                          path, emitted, count, width);
}

// Strides in bytes; a slot's row of a head is row_bytes long, the rows of a page lie one behind the other.
TFF_API int tff_keep_path(void* cache, int pages, int layers, int planes, int heads, int page_size, int row_bytes,
                          long long page_bytes, long long layer_bytes, const int* pos_start, const int* block_table,
                          int table_width, const int* path, const int* count, int requests, int width, cudaStream_t stream) {
    if (requests <= 0 || layers <= 0 || width <= 1) return TFF_OK;
    if (!cache || pages <= 0 || planes <= 0 || heads <= 0 || page_size <= 0 || row_bytes <= 0 || (row_bytes & 1) || !pos_start ||
        !block_table || table_width <= 0 || !path || !count || requests > 65535)
        return TFF_ERR_BAD_ARGUMENT;
    KeepParams p;
    p.cache = (char*)cache; p.page_bytes = page_bytes; p.layer_bytes = layer_bytes;
    p.head_bytes = (long long)page_size * row_bytes; p.plane_bytes = p.head_bytes * heads;
    p.pages = pages; p.layers = layers; p.planes = planes; p.heads = heads; p.page_size = page_size; p.row_bytes = row_bytes;
    p.pos_start = pos_start; p.block_table = block_table; p.table_width = table_width;
    p.path = path; p.count = count; p.width = width;
    const unsigned long long align = (uintptr_t)cache | (unsigned long long)page_bytes | (unsigned long long)layer_bytes | (unsigned long long)row_bytes;
    const int v = align % 16 == 0 ? 16 : align % 4 == 0 ? 4 : 2;
    const long long items = (long long)layers * planes * heads * (row_bytes / v);
    const long long blocks = (items + KEEP_THREADS - 1) / KEEP_THREADS;
    if (items > 0x7fffffff) return TFF_ERR_UNSUPPORTED;           // (counted in 32 bits)
    const dim3 grid((unsigned)blocks, requests);
    if (v == 16) return tff_launch_pdl(keep_path_kernel<uint4>, grid, dim3(KEEP_THREADS), (size_t)0, stream, p);
    if (v == 4) return tff_launch_pdl(keep_path_kernel<unsigned>, grid, dim3(KEEP_THREADS), (size_t)0, stream, p);
    return tff_launch_pdl(keep_path_kernel<unsigned short>, grid, dim3(KEEP_THREADS), (size_t)0, stream, p);
}
