// Gated DeltaNet over a tree of drafted tokens: the conv window and the delta rule of every node along
// its own path from the root, with the slot's state only read; and the commit of one path.
//
// With c_i the sum of the log decays on the path of node i, A(i) its strict ancestors and k, q of unit
// length, the rule  S_i = e^{g_i} S_parent + k_i u_i^T,  o_i = S_i^T q_i  has the closed form
//
//   u_i = beta_i (v_i - e^{c_i} S0^T k_i) - sum_{j in A(i)} beta_i e^{c_i - c_j} (k_i . k_j) u_j
//   o_i = e^{c_i} S0^T q_i + sum_{j in A(i) + i} e^{c_i - c_j} (q_i . k_j) u_j
//
// so no node needs a state of its own: 64 KiB per value head are read once, whatever the tree.
#include "common.cuh"
#include "kernels.h"
#include "launch.cuh"
#include "tree.cuh"

namespace rl {

namespace {

constexpr int kDk = 128, kDv = 128, kTaps = 4;
using tree::kMaxNodes;

__device__ __forceinline__ int key_head_of(int h, int n_v, int n_qk, int head_map) {
    return head_map == 0 ? h : (head_map == 1 ? h / (n_v / n_qk) : h % n_qk);
}

// The conv of four consecutive channels: weights and the slot's window, oldest tap first.
struct Conv4 {
    float4 w[4], win[4];             // [channel]
    __device__ __forceinline__ void load(const GdnTreeArgs& a, int slot, int c0) {
        const int ph = a.conv_phase ? a.conv_phase[slot] & 3 : 0;
        const float4* wp = reinterpret_cast<const float4*>(a.w) + c0;
        const float4* sp = reinterpret_cast<const float4*>(a.conv) + size_t(slot) * a.conv_dim + c0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = wp[i];
            float4 r = sp[i];
            if (ph & 1) r = make_float4(r.y, r.z, r.w, r.x);
            if (ph & 2) r = make_float4(r.z, r.w, r.x, r.y);
            win[i] = r;
        }
    }
};
__device__ __forceinline__ float comp(const float4& v, int i) { return i == 0 ? v.x : (i == 1 ? v.y : (i == 2 ? v.z : v.w)); }

// SiLU(conv) of channels c0 .. c0+3 at a node: taps are the node, its parent, ... (src[0..3]; src[k] < 0:
// that tap is window entry ~src[k]).
__device__ __forceinline__ float4 conv_node(const Conv4& cv, const float* x, size_t row_stride, int4 src) {
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    const int s[4] = {src.w, src.z, src.y, src.x};       // oldest first
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        float4 t;
        if (s[k] >= 0) {
            t = *reinterpret_cast<const float4*>(x + s[k] * row_stride);
        } else {
            const int j = ~s[k];
            t = make_float4(comp(cv.win[0], j), comp(cv.win[1], j), comp(cv.win[2], j), comp(cv.win[3], j));
        }
        acc[0] = fmaf(comp(cv.w[0], k), t.x, acc[0]);
        acc[1] = fmaf(comp(cv.w[1], k), t.y, acc[1]);
        acc[2] = fmaf(comp(cv.w[2], k), t.z, acc[2]);
        acc[3] = fmaf(comp(cv.w[3], k), t.w, acc[3]);
    }
    auto silu = [](float v) { return v / (1.f + expf(-v)); };
    return make_float4(silu(acc[0]), silu(acc[1]), silu(acc[2]), silu(acc[3]));
}

// taps of a node: itself and its next three ancestors, then the window from its newest entry (3) down
__device__ __forceinline__ int4 conv_sources(int i, const int* parents) {
    int s[4];
    int at = i, past = 3;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (at >= 0) {
            s[k] = at;
            at = parents[at];
        } else {
            s[k] = ~past;
            --past;
        }
    }
    return make_int4(s[0], s[1], s[2], s[3]);
}

__device__ __forceinline__ float sum_warp(float v) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
}
__device__ __forceinline__ float4 unit(float4 y, float eps, float extra) {
    const float inv = extra / sqrtf(sum_warp(y.x * y.x + y.y * y.y + y.z * y.z + y.w * y.w) + eps);
    return make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
}
__device__ __forceinline__ float dot4(float4 a, float4 b, float acc) {
    return fmaf(a.x, b.x, fmaf(a.y, b.y, fmaf(a.z, b.z, fmaf(a.w, b.w, acc))));
}

struct TreeSmem {
    float q[kMaxNodes][kDk], k[kMaxNodes][kDk], u[kMaxNodes][kDv];
    float low[kMaxNodes][kMaxNodes], mix[kMaxNodes][kMaxNodes];      // coefficients of u_j in u_i and in o_i
    float decay[kMaxNodes], beta[kMaxNodes];                          // c_i
    unsigned long long word[kMaxNodes];
    int parents[kMaxNodes];
    int4 src[kMaxNodes];
};

constexpr int kThreads = 128;

}  // namespace

// grid (n_v, batch): one CTA per (sequence, value head), thread = column of the state.
__global__ void __launch_bounds__(kThreads) gdn_tree_kernel(GdnTreeArgs a) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    TreeSmem& s = *reinterpret_cast<TreeSmem*>(smem_raw);
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int n = tree::node_count(a.n_nodes, b, a.max_nodes, a.err);
    const int slot = a.slot_ids ? a.slot_ids[b] : b;
    if (slot < 0 || slot >= a.n_slots) {
        if (tid == 0) set_err(a.err, DEV_ERR_BAD_SLOT);
        return;
    }
    if (n == 0) return;
    if (warp == 0) {
        const tree::Words w = tree::ancestors(a.parents ? a.parents + size_t(b) * a.max_nodes : nullptr, n, lane, a.err);
        s.word[lane] = w.lo;
        s.word[lane + 32] = w.hi;
        s.parents[lane] = w.parent_lo;
        s.parents[lane + 32] = w.parent_hi;
    }
    __syncthreads();
    if (tid < n) {
        s.src[tid] = conv_sources(tid, s.parents);
        float c = 0.f;
        for (unsigned long long m = s.word[tid]; m; m &= m - 1)
            c += a.g_log[(size_t(b) * a.max_nodes + (__ffsll(m) - 1)) * a.n_v + h];
        s.decay[tid] = c;
        s.beta[tid] = a.beta[(size_t(b) * a.max_nodes + tid) * a.n_v + h];
    }
    __syncthreads();
    const int hs = key_head_of(h, a.n_v, a.n_qk, a.head_map);
    const float* x = a.x + size_t(b) * a.max_nodes * a.x_stride;
#pragma unroll 1
    for (int role = 0; role < 3; ++role) {
        const int c0 = (role == 0 ? hs * kDk : (role == 1 ? (a.n_qk + hs) * kDk : 2 * a.n_qk * kDk + h * kDv)) + lane * 4;
        Conv4 cv;
        cv.load(a, slot, c0);
        for (int i = warp; i < n; i += kThreads / 32) {
            float4 y = conv_node(cv, x + c0, a.x_stride, s.src[i]);
            if (role == 0) y = unit(y, a.eps_l2, 1.f / sqrtf(float(kDk)));
            if (role == 1) y = unit(y, a.eps_l2, 1.f);
            *reinterpret_cast<float4*>(role == 0 ? &s.q[i][lane * 4] : (role == 1 ? &s.k[i][lane * 4] : &s.u[i][lane * 4])) = y;
        }
    }
    __syncthreads();
    for (int p = tid; p < n * n; p += kThreads) {
        const int i = p / n, j = p - i * n;
        if (!(s.word[i] >> j & 1)) continue;
        float kk = 0.f, qk = 0.f;
        for (int d = 0; d < kDk; d += 4) {
            const float4 kj = *reinterpret_cast<const float4*>(&s.k[j][d]);
            kk = dot4(*reinterpret_cast<const float4*>(&s.k[i][d]), kj, kk);
            qk = dot4(*reinterpret_cast<const float4*>(&s.q[i][d]), kj, qk);
        }
        const float e = expf(s.decay[i] - s.decay[j]);
        s.low[i][j] = s.beta[i] * e * kk;
        s.mix[i][j] = e * qk;
    }
    __syncthreads();
    const float* S = a.S + (size_t(slot) * a.n_v + h) * (kDk * kDv) + tid;
    constexpr int kStep = 8;
    for (int i0 = 0; i0 < n; i0 += kStep) {
        float ks[kStep] = {}, qs[kStep] = {};
        for (int d = 0; d < kDk; ++d) {
            const float sv = S[d * kDv];
#pragma unroll
            for (int r = 0; r < kStep; ++r) {
                const int i = min(i0 + r, n - 1);
                ks[r] = fmaf(s.k[i][d], sv, ks[r]);
                qs[r] = fmaf(s.q[i][d], sv, qs[r]);
            }
        }
#pragma unroll
        for (int r = 0; r < kStep; ++r) {
            const int i = i0 + r;
            if (i >= n) break;
            const float e = expf(s.decay[i]);
            float u = s.beta[i] * (s.u[i][tid] - e * ks[r]), o = e * qs[r];
            for (unsigned long long m = s.word[i] & ~(1ull << i); m; m &= m - 1) {
                const int j = __ffsll(m) - 1;
                const float uj = s.u[j][tid];
                u = fmaf(-s.low[i][j], uj, u);
                o = fmaf(s.mix[i][j], uj, o);
            }
            s.u[i][tid] = u;
            a.o[((size_t(b) * a.max_nodes + i) * a.n_v + h) * kDv + tid] = fmaf(s.mix[i][i], u, o);
        }
    }
}

// ------------------------------------------------------------------------------------------------
// Commit: the path to the leaf, up to 8 tokens at a time in the closed form above with the state in
// registers.  grid (4 slices of 32 columns, n_v, batch).
namespace {

constexpr int kSliceCols = 32, kSlices = kDv / kSliceCols, kCommitThreads = 256, kChunk = 8;

struct CommitSmem {
    float k[kChunk][kDk], v[kChunk][kSliceCols];
    float kk[kChunk][kChunk];
    float g[kChunk], beta[kChunk];
    float red[kCommitThreads / 32][kChunk][kSliceCols];
    float u[kChunk][kSliceCols];
    int parents[kMaxNodes];
    int path[kMaxNodes];
    int len;
};

}  // namespace

__global__ void __launch_bounds__(kCommitThreads) gdn_tree_commit_kernel(GdnTreeArgs a) {
    __shared__ CommitSmem s;
    griddep_launch();
    const int slice = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int slot = a.slot_ids ? a.slot_ids[b] : b;
    if (slot < 0 || slot >= a.n_slots) {
        if (tid == 0) set_err(a.err, DEV_ERR_BAD_SLOT);
        return;
    }
    const int leaf = a.leaf[b];
    if (leaf < 0 || leaf >= a.max_nodes) {
        if (leaf != -1 && tid == 0) set_err(a.err, DEV_ERR_BAD_TREE);
        return;
    }
    float* Sp = a.S_out + (size_t(slot) * a.n_v + h) * (kDk * kDv);
    const int rg = tid >> 3, cg = tid & 7;               // rows 4rg.., slice columns 4cg..
    const int col0 = slice * kSliceCols + cg * 4;
    float4 st[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) st[r] = *reinterpret_cast<const float4*>(Sp + (4 * rg + r) * kDv + col0);
    if (warp == 0) {
        const tree::Words w = tree::ancestors(a.parents ? a.parents + size_t(b) * a.max_nodes : nullptr, leaf + 1, lane, a.err);
        s.parents[lane] = w.parent_lo;
        s.parents[lane + 32] = w.parent_hi;
        const unsigned long long path = tree::of_node(w.lo, w.hi, leaf);
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            const int i = lane + 32 * z;
            if (path >> i & 1) s.path[__popcll(path & ((1ull << i) - 1))] = i;
        }
        if (lane == 0) s.len = __popcll(path);
    }
    __syncthreads();
    const int hs = key_head_of(h, a.n_v, a.n_qk, a.head_map);
    const float* x = a.x + size_t(b) * a.max_nodes * a.x_stride;
    const int len = s.len;
    for (int t0 = 0; t0 < len; t0 += kChunk) {
        const int m = min(kChunk, len - t0);
        if (warp < m) {
            const int i = s.path[t0 + warp];
            const int4 src = conv_sources(i, s.parents);
            const int ck = (a.n_qk + hs) * kDk + lane * 4;
            Conv4 cv;
            cv.load(a, slot, ck);
            const float4 y = unit(conv_node(cv, x + ck, a.x_stride, src), a.eps_l2, 1.f);
            *reinterpret_cast<float4*>(&s.k[warp][lane * 4]) = y;
            if (lane < kSliceCols / 4) {
                const int c = 2 * a.n_qk * kDk + h * kDv + slice * kSliceCols + lane * 4;
                cv.load(a, slot, c);
                *reinterpret_cast<float4*>(&s.v[warp][lane * 4]) = conv_node(cv, x + c, a.x_stride, src);
            } else if (lane == 31) {
                s.g[warp] = a.g_log[(size_t(b) * a.max_nodes + i) * a.n_v + h];
                s.beta[warp] = a.beta[(size_t(b) * a.max_nodes + i) * a.n_v + h];
            }
        } else {
            *reinterpret_cast<float4*>(&s.k[warp][lane * 4]) = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        __syncthreads();
        // k_i . k_j for j < i (warp i), and S0^T k of all tokens: 4 rows x 4 columns per thread
        if (warp < m) {
            const float4 ki = *reinterpret_cast<const float4*>(&s.k[warp][lane * 4]);
            for (int j = 0; j < warp; ++j) {
                const float d = sum_warp(dot4(ki, *reinterpret_cast<const float4*>(&s.k[j][lane * 4]), 0.f));
                if (lane == 0) s.kk[warp][j] = d;
            }
        }
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
            if (i >= m) break;
            const float4 k4 = *reinterpret_cast<const float4*>(&s.k[i][4 * rg]);
            float4 kv;
            kv.x = st[0].x * k4.x + st[1].x * k4.y + st[2].x * k4.z + st[3].x * k4.w;
            kv.y = st[0].y * k4.x + st[1].y * k4.y + st[2].y * k4.z + st[3].y * k4.w;
            kv.z = st[0].z * k4.x + st[1].z * k4.y + st[2].z * k4.z + st[3].z * k4.w;
            kv.w = st[0].w * k4.x + st[1].w * k4.y + st[2].w * k4.z + st[3].w * k4.w;
#pragma unroll
            for (int off = 8; off <= 16; off <<= 1) {
                kv.x += __shfl_xor_sync(0xffffffffu, kv.x, off);
                kv.y += __shfl_xor_sync(0xffffffffu, kv.y, off);
                kv.z += __shfl_xor_sync(0xffffffffu, kv.z, off);
                kv.w += __shfl_xor_sync(0xffffffffu, kv.w, off);
            }
            if (lane < 8) *reinterpret_cast<float4*>(&s.red[warp][i][lane * 4]) = kv;
        }
        __syncthreads();
        if (warp == 0) {
            // the solve, one column per lane
            float c = 0.f;
            for (int i = 0; i < m; ++i) {
                c += s.g[i];
                float t = 0.f;
#pragma unroll
                for (int w = 0; w < kCommitThreads / 32; ++w) t += s.red[w][i][lane];
                float u = s.v[i][lane] - expf(c) * t;
                float cj = 0.f;
                for (int j = 0; j < i; ++j) {
                    cj += s.g[j];
                    u = fmaf(-expf(c - cj) * s.kk[i][j], s.u[j][lane], u);
                }
                s.u[i][lane] = s.beta[i] * u;
            }
        }
        __syncthreads();
        float c = 0.f;
        for (int i = 0; i < m; ++i) c += s.g[i];
        const float e = expf(c);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            st[r].x *= e; st[r].y *= e; st[r].z *= e; st[r].w *= e;
        }
        float ci = 0.f;
        for (int i = 0; i < m; ++i) {
            ci += s.g[i];
            const float f = expf(c - ci);
            const float4 k4 = *reinterpret_cast<const float4*>(&s.k[i][4 * rg]);
            const float4 u4 = *reinterpret_cast<const float4*>(&s.u[i][cg * 4]);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float kr = comp(k4, r) * f;
                st[r].x = fmaf(kr, u4.x, st[r].x);
                st[r].y = fmaf(kr, u4.y, st[r].y);
                st[r].z = fmaf(kr, u4.z, st[r].z);
                st[r].w = fmaf(kr, u4.w, st[r].w);
            }
        }
        __syncthreads();                                 // k, u, red are rewritten by the next chunk
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) *reinterpret_cast<float4*>(Sp + (4 * rg + r) * kDv + col0) = st[r];
}

// The conv windows after the path: entry w (oldest first) is input len + w of the old window followed by
// the path's rows.  The ring keeps its phase: rewriting the four taps of a channel is one 16-byte store
// either way, and a phase that every block reads could only be advanced by another launch.
// grid (ceil(conv_dim / 256), batch), thread = channel; behind gdn_tree_commit_kernel, which reads the
// windows.
__global__ void __launch_bounds__(256) gdn_tree_window_kernel(GdnTreeArgs a) {
    __shared__ int last[kTaps];                          // node of the new entry w, or ~(old entry)
    griddep_wait();
    const int b = blockIdx.y, lane = threadIdx.x & 31;
    const int slot = a.slot_ids ? a.slot_ids[b] : b, leaf = a.leaf[b];
    if (slot < 0 || slot >= a.n_slots || leaf < 0 || leaf >= a.max_nodes) return;
    if (threadIdx.x < 32) {
        const tree::Words w = tree::ancestors(a.parents ? a.parents + size_t(b) * a.max_nodes : nullptr, leaf + 1, lane, nullptr);
        const unsigned long long path = tree::of_node(w.lo, w.hi, leaf);
        const int len = __popcll(path);
        if (lane < kTaps && len + lane < kTaps) last[lane] = ~(len + lane);
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            const int i = lane + 32 * z;
            const int at = __popcll(path & ((1ull << i) - 1)) + kTaps - len;     // entry this node becomes
            if ((path >> i & 1) && at >= 0) last[at] = i;
        }
    }
    __syncthreads();
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= a.conv_dim) return;
    const int ph = a.conv_phase ? a.conv_phase[slot] & 3 : 0;
    float4* ring = reinterpret_cast<float4*>(a.conv_out) + size_t(slot) * a.conv_dim + c;
    const float4 old = *ring;
    const float* x = a.x + size_t(b) * a.max_nodes * a.x_stride + c;
    float out[4];
#pragma unroll
    for (int w = 0; w < kTaps; ++w) {
        const int i = last[w];
        const float v = i >= 0 ? x[i * a.x_stride] : comp(old, (ph + ~i) & 3);
#pragma unroll
        for (int p = 0; p < kTaps; ++p)
            if (((ph + w) & 3) == p) out[p] = v;
    }
    *ring = make_float4(out[0], out[1], out[2], out[3]);
}

size_t gdn_tree_smem_bytes() { return sizeof(TreeSmem); }
const void* gdn_tree_kernel_ptr() { return reinterpret_cast<const void*>(&gdn_tree_kernel); }

void launch_gdn_tree(const GdnTreeArgs& a, cudaStream_t st) {
    gdn_tree_kernel<<<dim3(unsigned(a.n_v), unsigned(a.batch)), kThreads, gdn_tree_smem_bytes(), st>>>(a);
}

cudaError_t launch_gdn_tree_commit(const GdnTreeArgs& a, cudaStream_t st) {
    gdn_tree_commit_kernel<<<dim3(kSlices, unsigned(a.n_v), unsigned(a.batch)), kCommitThreads, 0, st>>>(a);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned((a.conv_dim + 255) / 256), unsigned(a.batch));
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, gdn_tree_window_kernel, a);
}

}  // namespace rl
