// Trees of drafted tokens as the attention kernels read them: a request's parents in shared memory.
#pragma once

constexpr int TREE_MAX_NODES = 256;                  // of a request's tree

// A node's parent: an earlier node, -1 (the node follows the cached tokens), or -2 for what is neither (the node is not there).
__device__ __forceinline__ short tree_parent(int parent, int node) { return (short)(parent < -1 || parent >= node ? -2 : parent); }

// A node's ancestors, or -1 where the chain of its parents does not end at -1 (or node is -1).
__device__ __forceinline__ int tree_depth(const short* parent, int node) {
    if (node < 0) return -1;
    int depth = -1;
    while (node >= 0) { node = parent[node]; ++depth; }
    return node == -1 ? depth : -1;
}

// What a row's weighted sum of values is multiplied by: one over the sum of its weights, the sink's among them; 0 for a row that
// sees nothing.  ``m`` is the maximum that the weights are relative to.
__device__ __forceinline__ float tree_weight(float l, float m, int sink, const float* sink_val, int head) {
    if (!(l > 0.f)) return 0.f;
    if (sink) l += expf((sink_val ? sink_val[head] : 0.f) - m);
    return 1.f / l;
}
