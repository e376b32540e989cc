// From the projections of the gated attention to its operands in one pass: q/gate split, head
// RMSNorm (1 + gamma) of q and k, rotation of the first rotary_dim dims, K and V rows into the
// paged F16 cache.
//
//   q_h = R(p) [ x / rms(x) (1 + gamma_q) ],   k_h likewise,   row t of sequence b -> cache row pos[b] + t
//   p = pos[b] + t, or with a draft tree pos[b] + depth of node t (siblings share a position, not a row)
//   R(p) turns the pair (d, d + rotary_dim / 2) by p theta^(-2 d / rotary_dim)
//
// What attn_qk_prepare and kv_append do in two passes with k going out to memory and back; here k
// leaves the registers as the fp16 row of its page.  The angle is formed in 64 bits, as a fraction of
// a turn: at position 100 000 the fp32 product of position and frequency is 4e-3 rad off, more than
// the rounding of K to fp16.  In a cache whose other rows attn_qk_prepare rotated, angle_f32 takes its fp32
// product instead: q, K and V are then those of attn_qk_prepare and kv_append bit for bit.
//
// Bound by bandwidth (a row of 24 + 4 heads reads 57 KB and writes 16 to 52 KB).  A warp takes one
// row of one head, 8 consecutive dims per lane, so that every load and store is 16 bytes wide and
// the norm is five shuffles; the heads of a row share the 32 sines and cosines of its position,
// which one warp of the block computes while the others' rows are on their way.
#include "common.cuh"
#include "kernels.h"
#include "tree.cuh"

namespace rl {

namespace {

constexpr int kWarps = 8;

__device__ __forceinline__ double sum_warp(double v) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
}

struct Row8 {
    float v[8];
};
__device__ __forceinline__ Row8 load8(const float* p) {
    const float4 a = __ldcs(reinterpret_cast<const float4*>(p)), b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
    return {{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
}
__device__ __forceinline__ uint4 pack_f16(const Row8& x) {
    return make_uint4(pack_h2(x.v[0], x.v[1]), pack_h2(x.v[2], x.v[3]), pack_h2(x.v[4], x.v[5]), pack_h2(x.v[6], x.v[7]));
}
__device__ __forceinline__ uint32_t pack_b2(float lo, float hi) {
    __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&b);
}

// the rounding of q to q_type is the caller's choice
__device__ __forceinline__ void store_q(void* out, int q_type, size_t i, const Row8& x) {
    if (q_type == 0) {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(out) + i);
        p[0] = make_float4(x.v[0], x.v[1], x.v[2], x.v[3]);
        p[1] = make_float4(x.v[4], x.v[5], x.v[6], x.v[7]);
    } else if (q_type == 1) {
        *reinterpret_cast<uint4*>(static_cast<__half*>(out) + i) = pack_f16(x);
    } else {
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(out) + i) =
            make_uint4(pack_b2(x.v[0], x.v[1]), pack_b2(x.v[2], x.v[3]), pack_b2(x.v[4], x.v[5]), pack_b2(x.v[6], x.v[7]));
    }
}

}  // namespace

// grid (rows, ceil(units / 8)); a row's units are its n_q query heads, n_kv K rows, n_kv V rows.
__global__ void __launch_bounds__(kWarps * 32) attn_qk_append_kernel(AttnQkAppendArgs a) {
    __shared__ float2 turn[kHeadDim / 2];          // cos, sin of each pair
    const int row = blockIdx.x, b = row / a.n_tok, t = row - b * a.n_tok;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int unit = blockIdx.y * kWarps + warp;
    if (t >= (a.n_nodes ? tree::node_count(a.n_nodes, b, a.n_tok, a.err) : a.n_tok)) return;
    const bool is_q = unit < a.n_q, is_k = !is_q && unit < a.n_q + a.n_kv, is_v = !is_q && !is_k && unit < a.n_q + 2 * a.n_kv;
    const int head = is_q ? unit : (is_k ? unit - a.n_q : unit - a.n_q - a.n_kv);
    const int d = lane * 8;
    Row8 x = {}, gate = {};
    if (is_q) {
        const float* src = a.qg + row * a.qg_stride + size_t(head) * (2 * kHeadDim) + d;
        x = load8(src);
        if (a.gate_out) gate = load8(src + kHeadDim);
    } else if (is_k) {
        x = load8(a.k + row * a.k_stride + size_t(head) * kHeadDim + d);
    } else if (is_v) {
        x = load8(a.v + row * a.v_stride + size_t(head) * kHeadDim + d);
    }
    const int base = a.pos[b];
    const int pairs = a.rotary_dim / 2;
    if (warp == 0) {
        int depth = t;
        if (a.parents) {
            const tree::Words w = tree::ancestors(a.parents + size_t(b) * a.n_tok, t + 1, lane, a.err);
            depth = __popcll(tree::of_node(w.lo, w.hi, t)) - 1;
        }
        for (int i = lane; i < pairs; i += 32) {
            if (a.angle_f32) {
                const float angle = float((long long)base + depth) * float(a.rate[i]);
                turn[i] = make_float2(cosf(angle), sinf(angle));
            } else {
                const double turns = (double(base) + depth) * a.rate[i];
                float s, c;
                sincospif(2.f * float(turns - rint(turns)), &s, &c);
                turn[i] = make_float2(c, s);
            }
        }
    }
    __syncthreads();
    if (is_q || is_k) {
        double ss = 0.0;                                      // as attn_qk_prepare sums (4 096 rows: 75.6 us, in 32 bits 74.1)
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fma(double(x.v[e]), double(x.v[e]), ss);
        const float inv = 1.f / sqrtf(float(sum_warp(ss) / kHeadDim) + a.eps);
        const float* gamma = is_q ? a.q_norm : a.k_norm;
#pragma unroll
        for (int e = 0; e < 8; ++e) x.v[e] *= inv;
        if (gamma) {
            const float4 g0 = *reinterpret_cast<const float4*>(gamma + d), g1 = *reinterpret_cast<const float4*>(gamma + d + 4);
            const float g[8] = {g0.x, g0.y, g0.z, g0.w, g1.x, g1.y, g1.z, g1.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) x.v[e] *= 1.f + g[e];
        }
        // rotary_dim is a multiple of 16: the partner of a lane's dims is all in one other lane
        const int hop = pairs / 8;
        const bool low = lane < hop, high = lane >= hop && lane < 2 * hop;
        const int partner = low ? lane + hop : (high ? lane - hop : lane);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float y = __shfl_sync(0xffffffffu, x.v[e], partner);
            if (low || high) {
                const float2 cs = turn[(low ? d : d - pairs) + e];
                x.v[e] = fmaf(x.v[e], cs.x, low ? -(y * cs.y) : y * cs.y);     // the roundings of attn_qk_prepare
            }
        }
    }
    if (is_q) {
        const size_t i = (size_t(row) * a.n_q + head) * kHeadDim + d;
        store_q(a.q_out, a.q_type, i, x);
        if (a.gate_out) {
            float4* p = reinterpret_cast<float4*>(a.gate_out + i);
            p[0] = make_float4(gate.v[0], gate.v[1], gate.v[2], gate.v[3]);
            p[1] = make_float4(gate.v[4], gate.v[5], gate.v[6], gate.v[7]);
        }
    } else if (is_k || is_v) {
        const long long at = (long long)base + t;
        if (base < 0 || at >= (long long)a.max_pages_per_seq * kPageTokens) {
            if (lane == 0) set_err(a.err, DEV_ERR_BAD_LEN);
            return;
        }
        const int page = a.page_table[size_t(b) * a.max_pages_per_seq + at / kPageTokens];
        if (page < 0 || page >= a.n_pages) {
            if (lane == 0) set_err(a.err, DEV_ERR_BAD_PAGE);
            return;
        }
        const size_t dst = (size_t(page) * a.n_kv + head) * kv_slice_elems() + kv_slice_offset(int(at % kPageTokens), d);
        *reinterpret_cast<uint4*>((is_k ? a.k_pool : a.v_pool) + dst) = pack_f16(x);
    }
}

void launch_attn_qk_append(const AttnQkAppendArgs& a, int batch, cudaStream_t st) {
    const int units = a.n_q + 2 * a.n_kv;
    attn_qk_append_kernel<<<dim3(unsigned(batch) * unsigned(a.n_tok), unsigned((units + kWarps - 1) / kWarps)), kWarps * 32, 0, st>>>(a);
}

// K and V rows of the path to a leaf -> consecutive cache rows base, base + 1, ...  Node i of the path
// lies at row base + i and goes to base + (its depth) <= base + i.  grid (n_kv, batch, 2: K, V): a
// block holds all rows of its path in registers before it writes the first, so the moves may overlap.
// A few tens of KB per sequence: the time is that of the launch and of three dependent loads.
constexpr int kCommitWarps = 16, kCommitRows = tree::kMaxNodes / kCommitWarps;
__global__ void __launch_bounds__(kCommitWarps * 32) kv_tree_commit_kernel(KvTreeCommitArgs a) {
    const int h = blockIdx.x, b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int leaf = tree::checked_leaf(a.leaf, a.n_nodes, b, a.max_nodes, threadIdx.x == 0 ? a.err : nullptr);
    unsigned long long path = 0;
    if (leaf >= 0) {
        const tree::Words w =
            tree::ancestors(a.parents ? a.parents + size_t(b) * a.max_nodes : nullptr, leaf + 1, lane, a.err);
        path = tree::of_node(w.lo, w.hi, leaf);
    }
    // A sequence with a row that has no place is left as it is, in both pools and every head, and accepts nothing.  64 rows
    // lie in two pages at most, the first's and the leaf's.
    const int base = a.base_len[b];
    const int32_t* table = a.page_table + size_t(b) * a.max_pages_per_seq;
    int page0 = 0, page1 = 0;
    if (path) {
        int bad = DEV_OK;
        if (base < 0 || (long long)base + leaf >= (long long)a.max_pages_per_seq * kPageTokens) {
            bad = DEV_ERR_BAD_LEN;
        } else {
            page0 = table[base / kPageTokens];
            page1 = table[(base + leaf) / kPageTokens];
            if (page0 < 0 || page0 >= a.n_pages || page1 < 0 || page1 >= a.n_pages) bad = DEV_ERR_BAD_PAGE;
        }
        if (bad) {
            if (threadIdx.x == 0) set_err(a.err, bad);
            path = 0;
        }
    }
    if (a.n_accept && threadIdx.x == 0 && h == 0 && blockIdx.z == 0) a.n_accept[b] = __popcll(path);
    if (!path) return;
    __half* pool = blockIdx.z ? a.v_pool : a.k_pool;
    auto row_at = [&](int at) -> __half* {
        const int page = at / kPageTokens == base / kPageTokens ? page0 : page1;
        return pool + (size_t(page) * a.n_kv + h) * kv_slice_elems() + kv_slice_offset(at % kPageTokens, lane * 8);
    };
    uint4 rows[kCommitRows];
    bool got[kCommitRows];
#pragma unroll
    for (int j = 0; j < kCommitRows; ++j) {
        const int i = warp + j * kCommitWarps;
        got[j] = false;
        // a node whose depth is its index stays where it is
        if ((path >> i & 1) && __popcll(path & ((1ull << i) - 1)) != i) {
            got[j] = true;
            rows[j] = *reinterpret_cast<const uint4*>(row_at(base + i));
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kCommitRows; ++j) {
        const int i = warp + j * kCommitWarps;
        if (!got[j]) continue;
        *reinterpret_cast<uint4*>(row_at(base + __popcll(path & ((1ull << i) - 1)))) = rows[j];
    }
}

void launch_kv_tree_commit(const KvTreeCommitArgs& a, int batch, cudaStream_t st) {
    kv_tree_commit_kernel<<<dim3(unsigned(a.n_kv), unsigned(batch), 2), kCommitWarps * 32, 0, st>>>(a);
}

}  // namespace rl
