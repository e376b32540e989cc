// A tree of drafted tokens: parents[i] < i is the node that node i continues, -1 the committed
// history (several roots are allowed).  At most 64 nodes, so that the ancestors of a node (itself
// included) are one 64-bit word; the words of all nodes come out of six doubling rounds in one warp:
// word |= word of the node `jump` points at, jump = jump of that node.
#pragma once
#include "common.cuh"

namespace rl {
namespace tree {

constexpr int kMaxNodes = 64;

// value of node i, when lane l holds those of the nodes l (lo) and l + 32 (hi)
template <class T>
__device__ __forceinline__ T of_node(T lo, T hi, int i) {
    const T a = __shfl_sync(0xffffffffu, lo, i & 31), b = __shfl_sync(0xffffffffu, hi, i & 31);
    return i & 32 ? b : a;
}

// parent of node i < n of one sequence's row (null: a chain); one that is not in [-1, i) records DEV_ERR_BAD_TREE and
// counts as -1
__device__ __forceinline__ int checked_parent(const int32_t* parents, int i, int n, int* err) {
    if (i >= n) return -1;
    if (!parents) return i - 1;
    const int p = parents[i];
    if (p >= -1 && p < i) return p;
    set_err(err, DEV_ERR_BAD_TREE);
    return -1;
}

// Called by one full warp.  parents: one sequence's row, or null for a chain; n nodes.  Returns the
// ancestor words of the nodes lane (lo) and lane + 32 (hi), and their checked parents (-1 for a
// root).
struct Words {
    unsigned long long lo, hi;
    int parent_lo, parent_hi;
};
__device__ __forceinline__ Words ancestors(const int32_t* parents, int n, int lane, int* err) {
    Words w;
    w.parent_lo = checked_parent(parents, lane, n, err);
    w.parent_hi = checked_parent(parents, lane + 32, n, err);
    w.lo = 1ull << lane;
    w.hi = 1ull << (lane + 32);
    int jl = w.parent_lo, jh = w.parent_hi;
    while (__any_sync(0xffffffffu, jl >= 0 || jh >= 0)) {
        const unsigned long long a = of_node(w.lo, w.hi, jl & 63), b = of_node(w.lo, w.hi, jh & 63);
        const int ja = of_node(jl, jh, jl & 63), jb = of_node(jl, jh, jh & 63);
        if (jl >= 0) {
            w.lo |= a;
            jl = ja;
        }
        if (jh >= 0) {
            w.hi |= b;
            jh = jb;
        }
    }
    return w;
}

// nodes of sequence b in a call of max_nodes rows per sequence
__device__ __forceinline__ int node_count(const int32_t* n_nodes, int b, int max_nodes, int* err) {
    if (!n_nodes) return max_nodes;
    const int n = n_nodes[b];
    if (n >= 0 && n <= max_nodes) return n;
    set_err(err, DEV_ERR_BAD_TREE);
    return 0;
}

// last node of the path to keep, -1: none; one that is not in [-1, nodes) records DEV_ERR_BAD_TREE and counts as -1
__device__ __forceinline__ int checked_leaf(const int32_t* leaf, const int32_t* n_nodes, int b, int max_nodes, int* err) {
    const int i = leaf[b], n = node_count(n_nodes, b, max_nodes, err);
    if (i >= -1 && i < n) return i;
    set_err(err, DEV_ERR_BAD_TREE);
    return -1;
}

}  // namespace tree
}  // namespace rl
