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
#include "tcgen05.cuh"
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

// v / (1 + e^-v) by the hardware exponential and reciprocal: within 2^-21 for the magnitudes that matter, in five
// instructions (far below, e^-v = inf makes it -0).  With expf and a division 32 chains of 64 take 171 us instead of 162,
// 16 trees of 21 53 instead of 50, one of 8 18.3 instead of 15.2, at the same error against 64 bits (4.1e-7; commit 4.3e-8).
__device__ __forceinline__ float silu(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + fast_exp2(v * -1.4426950408889634f)));
    return v * r;
}

// SiLU(conv) of channels c0 .. c0+3 at M nodes, all their taps requested before the first is used: taps are the
// node, its parent, ... (src.x .. src.w: offsets of their rows in floats; negative: window entry ~src).
template <int M>
__device__ __forceinline__ void conv_nodes(const Conv4& cv, const float* x, const int4 (&src)[M], float4 (&y)[M]) {
    float4 t[M][4];
#pragma unroll
    for (int m = 0; m < M; ++m) {
        t[m][3] = *reinterpret_cast<const float4*>(x + src[m].x);
        t[m][2] = *reinterpret_cast<const float4*>(x + max(src[m].y, 0));
        t[m][1] = *reinterpret_cast<const float4*>(x + max(src[m].z, 0));
        t[m][0] = *reinterpret_cast<const float4*>(x + max(src[m].w, 0));
    }
#pragma unroll
    for (int m = 0; m < M; ++m) {
        if (src[m].w < 0) {                                   // near a root
            const int s[3] = {src[m].w, src[m].z, src[m].y};
#pragma unroll
            for (int k = 0; k < 3; ++k)
                if (s[k] < 0) t[m][k] = make_float4(comp(cv.win[0], ~s[k]), comp(cv.win[1], ~s[k]), comp(cv.win[2], ~s[k]), comp(cv.win[3], ~s[k]));
        }
        float a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            a[0] = fmaf(comp(cv.w[0], k), t[m][k].x, a[0]);
            a[1] = fmaf(comp(cv.w[1], k), t[m][k].y, a[1]);
            a[2] = fmaf(comp(cv.w[2], k), t[m][k].z, a[2]);
            a[3] = fmaf(comp(cv.w[3], k), t[m][k].w, a[3]);
        }
        y[m] = make_float4(silu(a[0]), silu(a[1]), silu(a[2]), silu(a[3]));
    }
}

// taps of a node: itself and its next three ancestors, then the window from its newest entry (3) down
__device__ __forceinline__ int4 conv_sources(int i, const int* parents, int row_stride) {
    int s[4];
    int at = i, past = 3;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (at >= 0) {
            s[k] = at * row_stride;
            at = parents[at];
        } else {
            s[k] = ~past;
            --past;
        }
    }
    return make_int4(s[0], s[1], s[2], s[3]);
}

// Decays along a path are sums of up to 64 logs whose differences are exponentiated: summed in 64 bits, so that one
// strongly closed gate does not cost the nodes behind it their digits; e^-10000 is 0 as e^-inf is, and has differences.  NaN stays NaN.
__device__ __forceinline__ float log_decay(float g) { return g < -1e4f ? -1e4f : g; }

__device__ __forceinline__ float sum_warp(float v) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
}
__device__ __forceinline__ float4 unit(float4 y, float eps, float extra) {
    const float inv = extra * rsqrtf(sum_warp(y.x * y.x + y.y * y.y + y.z * y.z + y.w * y.w) + eps);
    return make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
}
__device__ __forceinline__ float dot4(float4 a, float4 b, float acc) {
    return fmaf(a.x, b.x, fmaf(a.y, b.y, fmaf(a.z, b.z, fmaf(a.w, b.w, acc))));
}

// x0, x1 as fp16 pairs: hi, and what hi leaves
__device__ __forceinline__ void split2(float x0, float x1, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x0, x1);
    const float2 f = __half22float2(h);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = pack_h2(x0 - f.x, x1 - f.y);
}
// the larger one, NaN if either is
__device__ __forceinline__ float max_or_nan(float x, float y) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(x), "f"(y));
    return m;
}
// the power of two that brings a largest magnitude mx into [2^14, 2^15), and its inverse
__device__ __forceinline__ float lift(float mx, float& back) {
    const int e = int(__float_as_uint(mx) >> 23) - 127;
    const int up = mx > 0.f && e < 128 ? min(max(14 - e, -112), 112) : 0;
    back = __uint_as_float(uint32_t(127 - up) << 23);
    return __uint_as_float(uint32_t(127 + up) << 23);
}
// scale of the unit vectors k, q and of the coefficients (all at most 1) under their split
constexpr float kLift = 4096.f, kBack = 1.f / 4096.f;

constexpr int kThreads = 256, kHalf = kThreads / 2;

template <int NB>
struct TreeSmem {
    static constexpr int kSub = 2 * NB * 128;                 // 64 dims of the rows [k; q], 128 bytes each
    static constexpr int kPitch = NB + 4;                     // of the fp32 triangle: 16-byte rows on all banks
    alignas(1024) unsigned char kq[4][kSub];                  // hi dims 0-63, 64-127, lo dims 0-63, 64-127
    alignas(1024) unsigned char inv[2][NB * 128];             // scratch of the inversion; then T as tiles, hi and lo
    union {
        float tri[NB][kPitch];                                // L, inverted in place
        alignas(1024) unsigned char mix[2][NB * 128];         // then: coefficients of u_j in o_i as tiles
    };
    float decay[NB], decay_lo[NB];                            // c_i log2 e in two terms
    float grow[NB], beta[NB], in[NB];                         // e^{c_i}, beta_i, -beta_i e^{c_i} / lift
    float amax[2][kDv];
    unsigned long long word[kMaxNodes];
    uint32_t bad[2][kDv];                                     // [half of the nodes][column]: W, U that are not finite, a bit each
    uint32_t hole[2][kDv];                                    // [half of the columns][row]: [k; q] k^T that are not finite
    int parents[kMaxNodes];
    uint64_t bar_rows, bar_gram, bar_half, bar_in, bar_u, bar_out;
    uint32_t tmem_base;
};
template <int NB>
constexpr size_t tree_smem_bytes() {
    // the Gram product takes its A operand as 128 rows, past the last tile's where there are fewer
    return (sizeof(TreeSmem<NB>) > 3 * TreeSmem<NB>::kSub + 128 * 128 ? sizeof(TreeSmem<NB>) : 3 * TreeSmem<NB>::kSub + 128 * 128) + 1024;
}

// t = (I + t)^-1 in place, t unit lower triangular with its strict lower part given; what lies above the 16 x 16
// blocks of the diagonal is neither read nor written.  x: scratch of NB / 2 * 32 floats.  All threads; ends synchronised.
//   [T1 0; -T2 L T1, T2] joins the inverses T1, T2 of two diagonal blocks with L below the first.
template <int NB, int P>
__device__ __forceinline__ float4 row_times(const float (&)[NB][P], const float* arow, const float* b, int b_pitch, int k0, int k1) {
    float4 c = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int k = k0; k < k1; k += 4) {
        const float4 x = *reinterpret_cast<const float4*>(arow + k);
        const float xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float4 y = *reinterpret_cast<const float4*>(b + (k + e) * b_pitch);
            c.x = fmaf(xs[e], y.x, c.x); c.y = fmaf(xs[e], y.y, c.y); c.z = fmaf(xs[e], y.z, c.z); c.w = fmaf(xs[e], y.w, c.w);
        }
    }
    return c;
}
template <int NB, int P>
__device__ __forceinline__ void invert_triangle(float (&t)[NB][P], float* x, int tid) {
    if (tid < (NB + 31) / 32 * 32) {                          // a thread per column of a diagonal block
        const int r0 = min(tid, NB - 1) & ~15, c = tid & 15;
        float y[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float r[4] = {i == c ? 1.f : 0.f, 0.f, 0.f, 0.f};       // four sums: no 15-step chain
#pragma unroll
            for (int j = 0; j < i; j += 4) {
                const float4 l = *reinterpret_cast<const float4*>(&t[r0 + i][r0 + j]);
                r[0] = fmaf(-l.x, y[j], r[0]);
                if (j + 1 < i) r[1] = fmaf(-l.y, y[j + 1], r[1]);
                if (j + 2 < i) r[2] = fmaf(-l.z, y[j + 2], r[2]);
                if (j + 3 < i) r[3] = fmaf(-l.w, y[j + 3], r[3]);
            }
            y[i] = (r[0] + r[1]) + (r[2] + r[3]);
        }
        __syncwarp();
        if (tid < NB) {
#pragma unroll
            for (int i = 0; i < 16; ++i) t[r0 + i][r0 + c] = y[i];
        }
    }
    __syncthreads();
    if constexpr (NB >= 32) {                                 // 16 + 16
        const int p = tid >> 6, i = (tid & 63) >> 2, j = (tid & 3) * 4, c0 = 32 * p, r0 = c0 + 16;
        const bool mine = p < NB / 32;
        if (mine) *reinterpret_cast<float4*>(x + p * 256 + i * 16 + j) = row_times(t, &t[r0 + i][c0], &t[c0][c0 + j], P, 0, 16);
        __syncthreads();
        if (mine) {
            const float4 r = row_times(t, &t[r0 + i][r0], x + p * 256 + j, 16, 0, 16);
            *reinterpret_cast<float4*>(&t[r0 + i][c0 + j]) = make_float4(-r.x, -r.y, -r.z, -r.w);
        }
        __syncthreads();
    }
    if constexpr (NB > 32) {                                  // 32 + the rest
        constexpr int kRest = NB - 32;
        const int i = tid >> 3, j = (tid & 7) * 4;
        const bool mine = i < kRest;
        if (mine) *reinterpret_cast<float4*>(x + i * 32 + j) = row_times(t, &t[32 + i][0], &t[0][j], P, j & ~15, 32);
        __syncthreads();
        if (mine) {
            const float4 r = row_times(t, &t[32 + i][32], x + j, 32, 0, i < 16 ? 16 : kRest);
            *reinterpret_cast<float4*>(&t[32 + i][j]) = make_float4(-r.x, -r.y, -r.z, -r.w);
        }
        __syncthreads();
    }
}

// byte offset of fp16 element (row, d < 64) in a tile of 128-byte rows under the 128-byte swizzle
__device__ __forceinline__ int tile_at(int row, int d) { return row * 128 + (((d >> 3) ^ (row & 7)) << 4) + (d & 7) * 2; }

// Workspace of the verify: the rows [k; q] of every (sequence, key head) as the main kernel's shared memory holds
// them (4 parts of 2 nb rows of 128 bytes), then v [batch][max_nodes][n_v][128].
struct VerifyWorkspace {
    unsigned char* kq;
    float* v;
    size_t bytes;
};
__host__ __device__ __forceinline__ int rounded_nodes(int max_nodes) { return (max_nodes + 15) / 16 * 16; }
__host__ __device__ __forceinline__ VerifyWorkspace verify_workspace(void* base, int batch, int max_nodes, int n_v, int n_qk) {
    VerifyWorkspace w;
    const size_t kq = size_t(batch) * n_qk * rounded_nodes(max_nodes) * 1024;
    w.kq = static_cast<unsigned char*>(base);
    w.v = reinterpret_cast<float*>(static_cast<char*>(base) + kq);
    w.bytes = kq + size_t(batch) * max_nodes * n_v * kDv * 4;
    return w;
}
constexpr int kPrepWarps = 4, kPrepNodes = 16, kPrepAhead = 2;

}  // namespace

// Conv, SiLU, unit length and split of all rows, before the states are touched: a warp per head (k, q or v) and 16
// nodes, the taps of two nodes in flight.  grid (ceil((2 n_qk + n_v) / 4), batch, nb / 16).  Inside the main kernel,
// where few warps share an SM with the states, the same work took more than half of its time (32 chains of 64: 187 us).
__global__ void __launch_bounds__(kPrepWarps * 32, 6) gdn_tree_rows_kernel(GdnTreeArgs a) {
    __shared__ int parents[kMaxNodes];
    __shared__ int4 sources[kPrepNodes];
    griddep_launch();
    const int b = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, i0 = blockIdx.z * kPrepNodes;
    const int n = tree::node_count(a.n_nodes, b, a.max_nodes, a.err);
    const int slot = a.slot_ids ? a.slot_ids[b] : b;
    if (slot < 0 || slot >= a.n_slots || n == 0) return;      // recorded by the main kernel
    const int role = blockIdx.x * kPrepWarps + warp;          // k heads, q heads, value heads
    const bool is_v = role >= 2 * a.n_qk, is_q = !is_v && role >= a.n_qk;
    const int h = is_v ? min(role - 2 * a.n_qk, a.n_v - 1) : (is_q ? role - a.n_qk : role);
    const int ch = (is_v ? 2 * a.n_qk * kDk + h * kDv : (is_q ? h * kDk : (a.n_qk + h) * kDk)) + lane * 4;
    const float* x = a.x + size_t(b) * a.max_nodes * a.x_stride + ch;
    // the warp's own rows, 4 lines each, are requested before the tree and the weights are known
#pragma unroll
    for (int z = 0; z < kPrepNodes / 8; ++z)
        if (i0 + z * 8 + (lane >> 2) < n) asm volatile("prefetch.global.L2 [%0];" ::"l"(x - lane * 4 + (i0 + z * 8 + (lane >> 2)) * a.x_stride + (lane & 3) * 32));
    Conv4 cv;
    cv.load(a, slot, ch);
    if (tid < kMaxNodes) parents[tid] = tree::checked_parent(a.parents ? a.parents + size_t(b) * a.max_nodes : nullptr, tid, n, a.err);
    __syncthreads();
    if (tid < kPrepNodes) sources[tid] = conv_sources(min(i0 + tid, n - 1), parents, int(a.x_stride));
    __syncthreads();
    if (role >= 2 * a.n_qk + a.n_v || (is_v && i0 >= n)) return;
    const int nb = rounded_nodes(a.max_nodes);
    const VerifyWorkspace ws = verify_workspace(a.workspace, a.batch, a.max_nodes, a.n_v, a.n_qk);
    for (int i = i0; i < i0 + kPrepNodes; i += kPrepAhead) {
        int4 src[kPrepAhead];
        float4 y[kPrepAhead];
#pragma unroll
        for (int m = 0; m < kPrepAhead; ++m) src[m] = sources[i - i0 + m];
        conv_nodes(cv, x, src, y);
#pragma unroll
        for (int m = 0; m < kPrepAhead; ++m) {
            if (is_v) {
                if (i + m < n) *reinterpret_cast<float4*>(ws.v + ((size_t(b) * a.max_nodes + i + m) * a.n_v + h) * kDv + lane * 4) = y[m];
            } else {
                y[m] = unit(y[m], a.eps_l2, kLift);
                if (i + m >= n) y[m] = make_float4(0.f, 0.f, 0.f, 0.f);
                uint2 hi, lo;
                split2(y[m].x, y[m].y, hi.x, lo.x);
                split2(y[m].z, y[m].w, hi.y, lo.y);
                unsigned char* part = ws.kq + (size_t(b) * a.n_qk + h) * nb * 1024 + (lane >> 4) * (nb * 256);
                const int at = tile_at((is_q ? nb : 0) + i + m, (lane * 4) & 63);
                *reinterpret_cast<uint2*>(part + at) = hi;
                *reinterpret_cast<uint2*>(part + nb * 512 + at) = lo;
            }
        }
    }
}

// The rest, behind gdn_tree_rows_kernel: one CTA per (key head, sequence) with that key head's value heads one after
// the other (a.heads > 1), or per (value head, sequence).  Node count rounded up to NB.
//
// S0^T k and S0^T q of all nodes are one product per value head, D[v][row] = sum_d S0[d][v] [k; q][row][d],
// with the state as the A operand in tensor memory (a thread reads column v of the state with coalesced loads
// and stores it as TMEM lane v) and the rows [k; q] as the K-major B operand in shared memory.  With
// W = beta (V - e^c S0^T k) and T = (I + L)^-1, U = T W and the last term of o are products of the same form.
// All must keep fp32's precision: operands are split into two fp16 terms (22 bits, rows scaled by powers of two
// so that neither term leaves fp16's range) and hi lo + lo hi + hi hi accumulate in fp32, the small ones first.
// T is formed in fp32 (16 x 16 blocks by substitution, then joined): n^3 / 6 products once instead of n^2 / 2
// for each of the 128 columns, and no thread walks 64 dependent steps.  Its entries are k_i^T (a product of
// contractions) k_j beta, at most max beta in magnitude, so a fixed scale serves them.
//
// A node whose inputs are not finite would reach its siblings as 0 * inf through T and U.  Its row of W shows it,
// whichever input it was (k by S0^T k, gates by e^c): that entry of W is replaced by 0, the coefficients that are NaN
// too, and the outputs of the column at the node and its descendants become NaN at the end.  A bad q stays in its row.
// (Two CTAs per SM leave 128 registers a thread, 64 of which hold the state: 120 to 332 bytes of spill stores a thread.)
template <int NB>
__global__ void __launch_bounds__(kThreads, 2) gdn_tree_kernel(GdnTreeArgs a) {
    using Smem = TreeSmem<NB>;
    extern __shared__ unsigned char smem_raw[];
    // (aligned by an offset, not by integer arithmetic on the pointer: the compiler keeps the loads shared-space ones)
    Smem& s = *reinterpret_cast<Smem*>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
    // tensor memory: A (32 columns hi, 32 lo: half the state's dims, later W and U), D, and [k; q] k^T (lane = row)
    constexpr uint32_t kColA = 0, kColD = 64, kColG = 64 + 2 * NB;
    constexpr uint32_t kCols = 64 + 3 * NB <= 128 ? 128 : 256;
    constexpr int kMine = NB / 2;                             // nodes of a thread's group
    const int b = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int grp = warp >> 2;                                // which half of the state's dims, of the nodes
    const int v = tid & (kDv - 1);                            // column of the state = TMEM lane
    const int slot = a.slot_ids ? a.slot_ids[b] : b;
    const int n = tree::node_count(a.n_nodes, b, a.max_nodes, a.err);
    if (slot < 0 || slot >= a.n_slots || n == 0) {
        if (tid == 0 && n) set_err(a.err, DEV_ERR_BAD_SLOT);
        griddep_wait();                                       // on every path: what follows this kernel follows the one in front too
        return;
    }
    const int ratio = a.n_v / a.n_qk;
    const int h0 = a.heads == 1 ? int(blockIdx.x) : (a.head_map == 1 ? int(blockIdx.x) * ratio : int(blockIdx.x));
    const int h_step = a.head_map == 1 ? 1 : a.n_qk;
    const int hs = a.heads == 1 ? key_head_of(h0, a.n_v, a.n_qk, a.head_map) : int(blockIdx.x);

    // the first head's half column of the state, on its way while the rows are prepared
    float st[kDk / 2];
    auto fetch = [&](int h) {
        const float* S = a.S + (size_t(slot) * a.n_v + h) * (kDk * kDv) + size_t(grp) * (kDk / 2) * kDv + v;
#pragma unroll
        for (int d = 0; d < kDk / 2; ++d) st[d] = __ldcs(S + d * kDv);
    };

    // the other heads' states start on their way into L2
    for (int i = tid; i < (a.heads - 1) * 512; i += kThreads)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(a.S + (size_t(slot) * a.n_v + h0 + ((i >> 9) + 1) * h_step) * (kDk * kDv) + (i & 511) * 32));
    fetch(h0);
    if (warp == 0) {
        const tree::Words w = tree::ancestors(a.parents ? a.parents + size_t(b) * a.max_nodes : nullptr, n, lane, a.err);
        s.word[lane] = w.lo;
        s.word[lane + 32] = w.hi;
        s.parents[lane] = w.parent_lo;
        s.parents[lane + 32] = w.parent_hi;
    } else if (warp == 1) {
        tc::tmem_alloc(&s.tmem_base, kCols);
    } else if (tid == 64) {
        mbar_init(&s.bar_rows, 1);
        mbar_init(&s.bar_gram, 1);
        mbar_init(&s.bar_half, 1);
        mbar_init(&s.bar_in, 1);
        mbar_init(&s.bar_u, 1);
        mbar_init(&s.bar_out, 1);
        mbar_fence_init();
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = s.tmem_base, lanes = tmem + (uint32_t((warp & 3) * 32) << 16);
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {         // `ok` is the same in all lanes of a warp
        if (ok && !__all_sync(0xffffffffu, mbar_wait(bar, parity))) {
            set_err(a.err, DEV_ERR_WAIT_TIMEOUT);
            ok = false;
        }
    };

    const VerifyWorkspace ws = verify_workspace(a.workspace, a.batch, a.max_nodes, a.n_v, a.n_qk);
    auto kq_desc = [&](int part) { return tc::smem_desc(smem_u32(s.kq[part]), 16, 1024); };
    // one thread: the rows into shared memory, then [k; q] k^T (lane = row).  Everything in front of it reads inputs that
    // were there before the rows kernel started, and runs beside it.
    auto gram = [&]() {
        griddep_wait();
        mbar_arrive_expect_tx(&s.bar_rows, sizeof(s.kq));
        bulk_g2s(s.kq, ws.kq + (size_t(b) * a.n_qk + hs) * sizeof(s.kq), sizeof(s.kq), &s.bar_rows);
        if (!mbar_wait(&s.bar_rows, 0)) set_err(a.err, DEV_ERR_WAIT_TIMEOUT);
        constexpr uint32_t idesc = tc::idesc_f16(128, NB, false, false);
#pragma unroll 1
        for (int pass = 0; pass < 3; ++pass) {
            const int pa = pass == 0 ? 2 : 0, pb = pass == 1 ? 2 : 0;     // lo hi, hi lo, hi hi
#pragma unroll
            for (int kk = 0; kk < 8; ++kk)
                tc::mma_ss(tmem + kColG, kq_desc(pa + (kk >> 2)) + (kk & 3) * 2, kq_desc(pb + (kk >> 2)) + (kk & 3) * 2, idesc,
                           pass > 0 || kk > 0);
        }
        tc::commit(&s.bar_gram);
    };

#pragma unroll 1
    for (int hi = 0; hi < a.heads; ++hi) {
        const int h = h0 + hi * h_step;
        const uint32_t par = hi & 1;
        // ---- decays along the paths ----
        if (warp == 4) {
            const size_t at = size_t(b) * a.max_nodes * a.n_v + h;
            const float g0 = lane < n ? a.g_log[at + size_t(lane) * a.n_v] : 0.f;
            const float g1 = NB > 32 && lane + 32 < n ? a.g_log[at + size_t(lane + 32) * a.n_v] : 0.f;
            const float b0 = lane < n ? a.beta[at + size_t(lane) * a.n_v] : 0.f;
            const float b1 = NB > 32 && lane + 32 < n ? a.beta[at + size_t(lane + 32) * a.n_v] : 0.f;
            const bool bad0 = !(g0 < INFINITY) || !(fabsf(b0) < INFINITY), bad1 = !(g1 < INFINITY) || !(fabsf(b1) < INFINITY);
            double c0 = bad0 ? 0.f : log_decay(g0), c1 = bad1 ? 0.f : log_decay(g1);
            int j0 = s.parents[lane], j1 = s.parents[lane + 32];
            while (__any_sync(0xffffffffu, j0 >= 0 || j1 >= 0)) {
                const double x0 = tree::of_node(c0, c1, j0 & 63), x1 = tree::of_node(c0, c1, j1 & 63);
                const int y0 = tree::of_node(j0, j1, j0 & 63), y1 = tree::of_node(j0, j1, j1 & 63);
                if (j0 >= 0) {
                    c0 += x0;
                    j0 = y0;
                }
                if (j1 >= 0) {
                    c1 += x1;
                    j1 = y1;
                }
            }
#pragma unroll
            for (int z = 0; z < 2; ++z) {
                const int i = lane + 32 * z;
                if (i >= NB) break;
                const double c = (z ? c1 : c0) * 1.4426950408889634;
                const bool bad = z ? bad1 : bad0;             // NaN in W alone
                const float bt = bad ? 0.f : (z ? b1 : b0), e = fast_exp2(float(c));
                s.decay[i] = float(c);
                s.decay_lo[i] = float(c - double(float(c)));
                s.grow[i] = e;
                s.beta[i] = bt;
                s.in[i] = bad ? __uint_as_float(0x7fc00000u) : -bt * e * kBack;
            }
        }
        // ---- the state's column -> A, 64 dims at a time ----
        {
            float mx = 0.f;
#pragma unroll
            for (int d = 0; d < kDk / 2; ++d) mx = fmaxf(mx, fabsf(st[d]));
            s.amax[grp][v] = mx;
        }
        __syncthreads();
        float back;
        const float f = lift(fmaxf(s.amax[0][v], s.amax[1][v]), back);
        {
            uint32_t th[32], tl[32];
#pragma unroll
            for (int c = 0; c < 32; ++c) split2(st[2 * c] * f, st[2 * c + 1] * f, th[c], tl[c]);
            if (grp == 1) wait(&s.bar_half, par);             // the first half's products are done with A
            tc::tmem_st32(lanes + kColA, th);
            tc::tmem_st32(lanes + kColA + 32, tl);
            tc::tmem_wait_st();
        }
        tc::fence_before_sync();
        named_bar_sync(1 + grp, kHalf);
        if ((tid & (kHalf - 1)) == 0) {
            tc::fence_after_sync();
            if (hi == 0 && grp == 0) gram();
            if (hi == 0 && grp == 1 && !mbar_wait(&s.bar_rows, 0)) set_err(a.err, DEV_ERR_WAIT_TIMEOUT);
            constexpr uint32_t idesc = tc::idesc_f16(128, 2 * NB, false, false);
#pragma unroll 1
            for (int pass = 0; pass < 3; ++pass) {
                const uint32_t acol = tmem + kColA + (pass == 0 ? 32 : 0);
                const uint64_t bd = kq_desc((pass == 1 ? 2 : 0) + grp);
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                    tc::mma_ts(tmem + kColD, acol + kk * 8, bd + kk * 2, idesc, grp > 0 || pass > 0 || kk > 0);
            }
            tc::commit(grp ? &s.bar_in : &s.bar_half);
        }
        float u[kMine];                                       // column v of W, later of U, at this group's nodes
        {
            __syncwarp();
            if (hi == 0) griddep_wait();
            const float* vp = ws.v + (size_t(b) * a.max_nodes * a.n_v + h) * kDv + v;
#pragma unroll
            for (int e = 0; e < kMine; ++e) {
                const int i = grp * kMine + e;
                u[e] = i < n ? vp[size_t(i) * a.n_v * kDv] : 0.f;
            }
        }
        // ---- this head's coefficients, half a row of [k; q] k^T per thread: L to shared memory, those of o kept ----
        float m[kMine];
        if (hi == 0) {
            wait(&s.bar_gram, 0);
            tc::fence_after_sync();
        }
        {
            const bool is_q = v >= NB;
            const int i = is_q ? v - NB : v;
            const bool row = v < 2 * NB && i < n;
            // this half's columns that count: ancestors, and for o the node itself
            const unsigned long long word = row ? (is_q ? s.word[i] : s.word[i] & ~(1ull << i)) : 0ull;
            uint32_t on = uint32_t(word >> (grp * kMine));
            if (hi == 0) {
                uint32_t hole = 0;
#pragma unroll
                for (int c = 0; c < kMine; c += 8) {
                    uint32_t g[8];
                    tc::tmem_ld8(lanes + kColG + grp * kMine + c, g);
                    tc::tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 8; ++e) hole |= uint32_t(!(fabsf(__uint_as_float(g[e])) < INFINITY)) << (c + e);
                }
                s.hole[grp][v] = hole;                        // read by this thread alone
                on &= ~hole;
            } else {
                on &= ~s.hole[grp][v];
            }
            const float ci = row ? s.decay[i] : 0.f, ci_lo = row ? s.decay_lo[i] : 0.f;
            const float f_ = is_q ? kBack * 0.08838834764831845f : (row ? s.beta[i] * kBack * kBack : 0.f);      // 1 / sqrt(128)
#pragma unroll
            for (int c = 0; c < kMine; c += 8) {
                const int j0 = grp * kMine + c;
                uint32_t g[8];
                tc::tmem_ld8(lanes + kColG + j0, g);
                tc::tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 8; e += 4) {
                    const float4 d4 = *reinterpret_cast<const float4*>(&s.decay[j0 + e]), l4 = *reinterpret_cast<const float4*>(&s.decay_lo[j0 + e]);
                    const float cj[4] = {d4.x, d4.y, d4.z, d4.w}, cj_lo[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
                    for (int z = 0; z < 4; ++z) {
                        const float y = fast_exp2((ci - cj[z]) + (ci_lo - cj_lo[z])) * (f_ * __uint_as_float(g[e + z]));     // no branch: what does not count is dropped
                        m[c + e + z] = on >> (c + e + z) & 1 ? y : 0.f;
                    }
                }
                if (v < NB) {
                    *reinterpret_cast<float4*>(&s.tri[i][j0]) = make_float4(m[c], m[c + 1], m[c + 2], m[c + 3]);
                    *reinterpret_cast<float4*>(&s.tri[i][j0 + 4]) = make_float4(m[c + 4], m[c + 5], m[c + 6], m[c + 7]);
                }
                __syncwarp();
            }
        }
        __syncthreads();
        invert_triangle<NB>(s.tri, reinterpret_cast<float*>(s.inv[0]), tid);
        // ---- T -> tiles; W = beta v - beta e^c S0^T k -> A ----
        for (int idx = tid; idx < NB * (NB / 8); idx += kThreads) {
            const int i = idx % NB, j0 = (idx / NB) * 8;
            float r[8];
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const float4 q = *reinterpret_cast<const float4*>(&s.tri[i][j0 + e]);
                r[e] = q.x; r[e + 1] = q.y; r[e + 2] = q.z; r[e + 3] = q.w;
            }
            uint32_t th[4], tl[4];
#pragma unroll
            for (int e = 0; e < 8; e += 2)
                split2(j0 + e <= i ? r[e] * kLift : 0.f, j0 + e + 1 <= i ? r[e + 1] * kLift : 0.f, th[e / 2], tl[e / 2]);
            const int at = tile_at(i, j0);
            *reinterpret_cast<uint4*>(s.inv[0] + at) = make_uint4(th[0], th[1], th[2], th[3]);
            *reinterpret_cast<uint4*>(s.inv[1] + at) = make_uint4(tl[0], tl[1], tl[2], tl[3]);
        }
        tc::fence_async_smem();
        wait(&s.bar_in, par);
        tc::fence_after_sync();
#pragma unroll
        for (int c = 0; c < kMine; c += 8) {
            uint32_t d[8];
            tc::tmem_ld8(lanes + kColD + grp * kMine + c, d);
            tc::tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 8; ++e)
                u[c + e] = fmaf(__uint_as_float(d[e]) * back, s.in[grp * kMine + c + e], u[c + e] * s.beta[grp * kMine + c + e]);
        }
        // column v of W or U, both halves' largest magnitude scaled into place -> A; returns the scale's inverse
        uint32_t bad = 0;
        auto store_column = [&]() {
            float mx = 0.f;
#pragma unroll
            for (int e = 0; e < kMine; ++e) mx = max_or_nan(mx, fabsf(u[e]));
            if (!(mx < INFINITY)) {
                mx = 0.f;
#pragma unroll
                for (int e = 0; e < kMine; ++e) {
                    if (!(fabsf(u[e]) < INFINITY)) {
                        bad |= 1u << e;
                        u[e] = 0.f;
                    }
                    mx = fmaxf(mx, fabsf(u[e]));
                }
            }
            s.bad[grp][v] = bad;
            s.amax[grp][v] = mx;
            __syncthreads();
            float bk;
            const float sc = lift(fmaxf(s.amax[0][v], s.amax[1][v]), bk);
#pragma unroll
            for (int c = 0; c < kMine / 2; c += 4) {
                uint32_t h4[4], l4[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) split2(u[2 * (c + e)] * sc, u[2 * (c + e) + 1] * sc, h4[e], l4[e]);
                tc::tmem_st4(lanes + kColA + grp * (kMine / 2) + c, h4);
                tc::tmem_st4(lanes + kColA + 32 + grp * (kMine / 2) + c, l4);
            }
            tc::tmem_wait_st();
            tc::fence_before_sync();
            __syncthreads();
            return bk;
        };
        // D's k columns = A x tiles, both split: lo hi, hi lo, hi hi
        auto product = [&](const unsigned char (&tiles)[2][NB * 128], uint64_t* done) {
            tc::fence_after_sync();
            constexpr uint32_t idesc = tc::idesc_f16(128, NB, false, false);
#pragma unroll 1
            for (int pass = 0; pass < 3; ++pass) {
                const uint32_t acol = tmem + kColA + (pass == 0 ? 32 : 0);
                const uint64_t bd = tc::smem_desc(smem_u32(tiles[pass == 1 ? 1 : 0]), 16, 1024);
#pragma unroll
                for (int kk = 0; kk < NB / 16; ++kk) tc::mma_ts(tmem + kColD, acol + kk * 8, bd + kk * 2, idesc, pass > 0 || kk > 0);
            }
            tc::commit(done);
        };
        const float wback = store_column() * kBack;
        if (tid == 0) product(s.inv, &s.bar_u);
        if (v >= NB && v < 2 * NB) {
#pragma unroll
            for (int c = 0; c < kMine; c += 8) {
                uint32_t mh[4], ml[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) split2(m[c + 2 * e], m[c + 2 * e + 1], mh[e], ml[e]);
                const int at = tile_at(v - NB, grp * kMine + c);
                *reinterpret_cast<uint4*>(s.mix[0] + at) = make_uint4(mh[0], mh[1], mh[2], mh[3]);
                *reinterpret_cast<uint4*>(s.mix[1] + at) = make_uint4(ml[0], ml[1], ml[2], ml[3]);
            }
        }
        tc::fence_async_smem();
        __syncwarp();
        wait(&s.bar_u, par);
        tc::fence_after_sync();
#pragma unroll
        for (int c = 0; c < kMine; c += 8) {
            uint32_t d[8];
            tc::tmem_ld8(lanes + kColD + grp * kMine + c, d);
            tc::tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 8; ++e) u[c + e] = __uint_as_float(d[e]) * wback;
        }
        const float uback = store_column() * kBack;
        if (tid == 0) product(s.mix, &s.bar_out);
        if (hi + 1 < a.heads) fetch(h + h_step);
        __syncwarp();
        wait(&s.bar_out, par);
        tc::fence_after_sync();
        // ---- o = e^c S0^T q / sqrt(128) + sum mix u ----
        const float qs = back * (kBack * 0.08838834764831845f);
        float* o = a.o + (size_t(b) * a.max_nodes * a.n_v + h) * kDv + v;
#pragma unroll
        for (int c = 0; c < kMine; c += 8) {
            const int i0 = grp * kMine + c;
            if (i0 >= n) break;
            uint32_t dq[8], du[8];
            tc::tmem_ld8(lanes + kColD + NB + i0, dq);
            tc::tmem_ld8(lanes + kColD + i0, du);
            tc::tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (ok && i0 + e < n)
                    __stcs(o + size_t(i0 + e) * a.n_v * kDv,
                           fmaf(__uint_as_float(dq[e]) * qs, s.grow[i0 + e], __uint_as_float(du[e]) * uback));
        }
        if (const unsigned long long hit = s.bad[0][v] | (unsigned long long)s.bad[1][v] << kMine; hit && ok) {
#pragma unroll 1
            for (int i = grp * kMine; i < min(n, (grp + 1) * kMine); ++i)
                if (s.word[i] & hit) o[size_t(i) * a.n_v * kDv] = __uint_as_float(0x7fc00000u);
        }
        tc::fence_before_sync();
        __syncthreads();                                      // D, A and the head's tables may be rewritten
        tc::fence_after_sync();
    }
    if (warp == 1) tc::tmem_dealloc(tmem, kCols);
}

// ------------------------------------------------------------------------------------------------
// Commit, in two kernels.  The first (gdn_tree_path_kernel) walks the path to the leaf and leaves its tokens' k
// (unit length), v, log decays and betas in the workspace, in path order; the second moves the state, 128 KiB in and
// out per head, which is the bound, and rewrites the conv windows, which nothing reads any more.  Together in one
// kernel every CTA waits for leaf, parents, rows and taps one after the other before it can touch the state (32
// paths in trees of 32: 93 us).
namespace {

constexpr int kPathWarps = 4, kCommitThreads = 256, kCommitCols = 64, kParts = kDv / kCommitCols, kChunk = 16;

struct CommitSmem {
    float k[kChunk][kDk], v[kChunk][kCommitCols];             // v, then u
    float low[kChunk][kChunk];                                // coefficient of u_j in u_i
    float red[4][kChunk][kCommitCols];                        // S0^T k by row blocks
    double c[kMaxNodes];                                      // log decay from the state to the path's token
    float beta[kMaxNodes];
};
// workspace: path lengths, then the path's nodes [batch][max_nodes], c and beta [batch][n_v][max_nodes], k
// [batch][max_nodes][n_qk][128], v [batch][max_nodes][n_v][128]
struct CommitWorkspace {
    int* len;
    int* path;
    double* c;
    float* beta;
    float *k, *v;
    size_t bytes;
};
__host__ __device__ __forceinline__ CommitWorkspace commit_workspace(void* base, int batch, int max_nodes, int n_v, int n_qk) {
    CommitWorkspace w;
    size_t at = 0;
    char* p = static_cast<char*>(base);
    auto take = [&](size_t bytes) {
        char* q = p + at;
        at += (bytes + 255) / 256 * 256;
        return q;
    };
    const size_t rows = size_t(batch) * max_nodes;
    w.len = reinterpret_cast<int*>(take(size_t(batch) * 4));
    w.path = reinterpret_cast<int*>(take(rows * 4));
    w.c = reinterpret_cast<double*>(take(rows * n_v * 8));
    w.beta = reinterpret_cast<float*>(take(rows * n_v * 4));
    w.k = reinterpret_cast<float*>(take(rows * n_qk * kDk * 4));
    w.v = reinterpret_cast<float*>(take(rows * n_v * kDv * 4));
    w.bytes = at;
    return w;
}

}  // namespace

// grid (ceil((n_qk + n_v) / 4), batch): a warp per key head (its k) or value head (its v, decays, betas).
__global__ void __launch_bounds__(kPathWarps * 32) gdn_tree_path_kernel(GdnTreeArgs a) {
    __shared__ int parents[kMaxNodes], path[kMaxNodes];
    __shared__ int path_len;
    griddep_launch();
    const int b = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int slot = a.slot_ids ? a.slot_ids[b] : b;
    const int leaf = tree::checked_leaf(a.leaf, a.n_nodes, b, a.max_nodes, tid == 0 ? a.err : nullptr);
    const CommitWorkspace ws = commit_workspace(a.workspace, a.batch, a.max_nodes, a.n_v, a.n_qk);
    const bool bad_slot = slot < 0 || slot >= a.n_slots;
    if (bad_slot || leaf < 0) {
        if (tid == 0) {
            if (bad_slot) set_err(a.err, DEV_ERR_BAD_SLOT);
            if (blockIdx.x == 0) ws.len[b] = 0;
        }
        return;
    }
    const int role = blockIdx.x * kPathWarps + warp;          // key heads, then value heads
    const bool is_k = role < a.n_qk, is_v = !is_k && role < a.n_qk + a.n_v;
    const int h = is_k ? role : role - a.n_qk;
    const int ch = (is_k ? (a.n_qk + h) * kDk : 2 * a.n_qk * kDk + (is_v ? h : 0) * kDv) + lane * 4;
    Conv4 cv;
    cv.load(a, slot, ch);
    if (warp == 0) {
        const tree::Words w = tree::ancestors(a.parents ? a.parents + size_t(b) * a.max_nodes : nullptr, leaf + 1, lane, a.err);
        parents[lane] = w.parent_lo;
        parents[lane + 32] = w.parent_hi;
        const unsigned long long on = tree::of_node(w.lo, w.hi, leaf);
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            const int i = lane + 32 * z, at = __popcll(on & ((1ull << i) - 1));
            if (on >> i & 1) {
                path[at] = i;
                if (blockIdx.x == 0) ws.path[size_t(b) * a.max_nodes + at] = i;
            }
        }
        if (lane == 0) {
            path_len = __popcll(on);
            if (blockIdx.x == 0) ws.len[b] = path_len;
        }
    }
    __syncthreads();
    if (!is_k && !is_v) return;
    const int len = path_len;
    const float* x = a.x + size_t(b) * a.max_nodes * a.x_stride;
    for (int t0 = 0; t0 < len; t0 += 4) {
        int4 src[4];
        float4 y[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) src[m] = conv_sources(path[min(t0 + m, len - 1)], parents, int(a.x_stride));
        conv_nodes(cv, x + ch, src, y);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const size_t at = size_t(b) * a.max_nodes + t0 + m;
            if (is_k) y[m] = unit(y[m], a.eps_l2, 1.f);
            if (t0 + m < len) *reinterpret_cast<float4*>(is_k ? ws.k + (at * a.n_qk + h) * kDk + lane * 4 : ws.v + (at * a.n_v + h) * kDv + lane * 4) = y[m];
        }
    }
    if (is_v) {
        double carry = 0.0;
        for (int t0 = 0; t0 < len; t0 += 32) {
            const int t = t0 + lane;
            const size_t at = t < len ? (size_t(b) * a.max_nodes + path[t]) * a.n_v + h : 0;
            double g = t < len ? log_decay(a.g_log[at]) : 0.f;
            const float bt = t < len ? a.beta[at] : 0.f;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const double up = __shfl_up_sync(0xffffffffu, g, off);
                if (lane >= off) g += up;
            }
            if (t < len) {
                ws.c[(size_t(b) * a.n_v + h) * a.max_nodes + t] = carry + g;
                ws.beta[(size_t(b) * a.n_v + h) * a.max_nodes + t] = bt;
            }
            carry += __shfl_sync(0xffffffffu, g, 31);
        }
    }
}

// grid (2 n_v + ceil(conv_dim / 256), batch).
// x < 2 n_v: 64 columns of one value head's state, in registers: warp w holds rows 32 (w / 2) .. and columns 32 (w % 2)
// .., a lane 8 rows x 4 columns, requested before the wait for the path kernel (only this kernel writes states).  Four
// such CTAs fit an SM, so that one's exchanges run under the others' loads and stores (two CTAs of 128 columns: 75
// against 68 us).  Up to 16 tokens at a time in the closed form above.
// The other blocks, a thread per channel: entry w (oldest first) of the new conv window is input len + w of the old
// window followed by the path's rows.  The ring keeps its phase: rewriting the four taps of a channel is one 16-byte
// store either way, and a phase that every block reads could only be advanced by another launch.
__global__ void __launch_bounds__(kCommitThreads, 4) gdn_tree_commit_kernel(GdnTreeArgs a) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    CommitSmem& s = *reinterpret_cast<CommitSmem*>(smem_raw);
    const int b = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const CommitWorkspace ws = commit_workspace(a.workspace, a.batch, a.max_nodes, a.n_v, a.n_qk);
    const int slot = a.slot_ids ? a.slot_ids[b] : b;
    if (slot < 0 || slot >= a.n_slots || tree::checked_leaf(a.leaf, a.n_nodes, b, a.max_nodes, nullptr) < 0) {
        griddep_wait();                                       // on every path: what follows this kernel follows the one in front too
        return;
    }
    if (int(blockIdx.x) >= kParts * a.n_v) {
        const int c = (blockIdx.x - kParts * a.n_v) * kCommitThreads + tid;
        griddep_wait();
        if (c >= a.conv_dim) return;
        const int len = ws.len[b], ph = a.conv_phase ? a.conv_phase[slot] & 3 : 0;
        float4* ring = reinterpret_cast<float4*>(a.conv_out) + size_t(slot) * a.conv_dim + c;
        const float4 old = *ring;
        const float* x = a.x + size_t(b) * a.max_nodes * a.x_stride + c;
        float out[kTaps];
#pragma unroll
        for (int w = 0; w < kTaps; ++w) {
            const int t = len + w - kTaps;                    // of the path; negative: old entry len + w
            const float y = t >= 0 ? x[ws.path[size_t(b) * a.max_nodes + t] * a.x_stride] : comp(old, (ph + len + w) & 3);
#pragma unroll
            for (int p = 0; p < kTaps; ++p)
                if (((ph + w) & 3) == p) out[p] = y;
        }
        *ring = make_float4(out[0], out[1], out[2], out[3]);
        return;
    }
    const int h = blockIdx.x / kParts, part0 = blockIdx.x % kParts * kCommitCols;
    float* Sh = a.S_out + (size_t(slot) * a.n_v + h) * (kDk * kDv) + part0;
    const int row0 = (warp >> 1) * 32 + (lane >> 3) * 8, col0 = (warp & 1) * 32 + (lane & 7) * 4;
    float4 st[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) st[r] = __ldcs(reinterpret_cast<const float4*>(Sh + (row0 + r) * kDv + col0));
    griddep_wait();
    const int len = ws.len[b], hs = key_head_of(h, a.n_v, a.n_qk, a.head_map);
    if (tid < len) {
        s.c[tid] = ws.c[(size_t(b) * a.n_v + h) * a.max_nodes + tid];
        s.beta[tid] = ws.beta[(size_t(b) * a.n_v + h) * a.max_nodes + tid];
    }
    for (int t0 = 0; t0 < len; t0 += kChunk) {
        const int m = min(kChunk, len - t0);
        for (int i = warp; i < m; i += kCommitThreads / 32) {
            const size_t at = size_t(b) * a.max_nodes + t0 + i;
            *reinterpret_cast<float4*>(&s.k[i][lane * 4]) = *reinterpret_cast<const float4*>(ws.k + (at * a.n_qk + hs) * kDk + lane * 4);
            if (lane < kCommitCols / 4)
                *reinterpret_cast<float4*>(&s.v[i][lane * 4]) = *reinterpret_cast<const float4*>(ws.v + (at * a.n_v + h) * kDv + part0 + lane * 4);
        }
        __syncthreads();
        const double c_in = t0 ? s.c[t0 - 1] : 0.0;           // decays are taken from the chunk's start
        // coefficients: pair (i, j < i) per warp; S0^T k: 8 rows x 4 columns per thread
        for (int p = warp; p < m * (m - 1) / 2; p += kCommitThreads / 32) {
            int i = 1, j = p;
            while (j >= i) j -= i++;
            const float d = sum_warp(dot4(*reinterpret_cast<const float4*>(&s.k[i][lane * 4]), *reinterpret_cast<const float4*>(&s.k[j][lane * 4]), 0.f));
            if (lane == 0) s.low[i][j] = s.beta[t0 + i] * expf(float(s.c[t0 + i] - s.c[t0 + j])) * d;
        }
#pragma unroll 2
        for (int i = 0; i < m; ++i) {
            const float4 ka = *reinterpret_cast<const float4*>(&s.k[i][row0]), kb = *reinterpret_cast<const float4*>(&s.k[i][row0 + 4]);
            const float kr[8] = {ka.x, ka.y, ka.z, ka.w, kb.x, kb.y, kb.z, kb.w};
            float4 kv = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                kv.x = fmaf(st[r].x, kr[r], kv.x); kv.y = fmaf(st[r].y, kr[r], kv.y);
                kv.z = fmaf(st[r].z, kr[r], kv.z); kv.w = fmaf(st[r].w, kr[r], kv.w);
            }
#pragma unroll
            for (int off = 8; off <= 16; off <<= 1) {
                kv.x += __shfl_xor_sync(0xffffffffu, kv.x, off);
                kv.y += __shfl_xor_sync(0xffffffffu, kv.y, off);
                kv.z += __shfl_xor_sync(0xffffffffu, kv.z, off);
                kv.w += __shfl_xor_sync(0xffffffffu, kv.w, off);
            }
            if (lane < 8) *reinterpret_cast<float4*>(&s.red[warp >> 1][i][col0]) = kv;
        }
        __syncthreads();
        // the solve, one column per thread
        if (tid < kCommitCols) {
            for (int i = 0; i < m; ++i) {
                const float kv = (s.red[0][i][tid] + s.red[1][i][tid]) + (s.red[2][i][tid] + s.red[3][i][tid]);
                float r = s.beta[t0 + i] * (s.v[i][tid] - expf(float(s.c[t0 + i] - c_in)) * kv);
                for (int j = 0; j < i; ++j) r = fmaf(-s.low[i][j], s.v[j][tid], r);
                s.v[i][tid] = r;
            }
        }
        __syncthreads();
        const double c_out = s.c[t0 + m - 1];
        const float e = expf(float(c_out - c_in));
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            st[r].x *= e; st[r].y *= e; st[r].z *= e; st[r].w *= e;
        }
        for (int i = 0; i < m; ++i) {
            const float f = expf(float(c_out - s.c[t0 + i]));
            const float4 ka = *reinterpret_cast<const float4*>(&s.k[i][row0]), kb = *reinterpret_cast<const float4*>(&s.k[i][row0 + 4]);
            const float kr[8] = {ka.x, ka.y, ka.z, ka.w, kb.x, kb.y, kb.z, kb.w};
            float4 u4 = *reinterpret_cast<const float4*>(&s.v[i][col0]);
            u4.x *= f; u4.y *= f; u4.z *= f; u4.w *= f;
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                st[r].x = fmaf(kr[r], u4.x, st[r].x); st[r].y = fmaf(kr[r], u4.y, st[r].y);
                st[r].z = fmaf(kr[r], u4.z, st[r].z); st[r].w = fmaf(kr[r], u4.w, st[r].w);
            }
        }
        if (t0 + kChunk < len) __syncthreads();               // k, v, red are rewritten by the next chunk
    }
#pragma unroll
    for (int r = 0; r < 8; ++r) __stcs(reinterpret_cast<float4*>(Sh + (row0 + r) * kDv + col0), st[r]);
}

size_t gdn_tree_commit_workspace_bytes(int batch, int max_nodes, int n_v, int n_qk) {
    return commit_workspace(nullptr, batch, max_nodes, n_v, n_qk).bytes;
}

namespace {
// a launch that may become resident while the kernel before it runs (both call griddep_*)
cudaError_t launch_behind(void (*kernel)(GdnTreeArgs), dim3 grid, int threads, size_t smem, cudaStream_t st, const GdnTreeArgs& a) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(unsigned(threads));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}
template <int NB>
cudaError_t set_attr() {
    return cudaFuncSetAttribute(gdn_tree_kernel<NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(tree_smem_bytes<NB>()));
}
template <int NB>
cudaError_t launch(const GdnTreeArgs& a, cudaStream_t st) {
    gdn_tree_rows_kernel<<<dim3(unsigned((2 * a.n_qk + a.n_v + kPrepWarps - 1) / kPrepWarps), unsigned(a.batch), NB / kPrepNodes),
                           kPrepWarps * 32, 0, st>>>(a);
    return launch_behind(gdn_tree_kernel<NB>, dim3(unsigned(a.n_v / a.heads), unsigned(a.batch)), kThreads, tree_smem_bytes<NB>(), st, a);
}
}  // namespace

cudaError_t gdn_tree_setup() {
    cudaError_t e = set_attr<16>();
    if (e == cudaSuccess) e = set_attr<32>();
    if (e == cudaSuccess) e = set_attr<48>();
    if (e == cudaSuccess) e = set_attr<64>();
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(gdn_tree_commit_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(sizeof(CommitSmem)));
    return e;
}

cudaError_t launch_gdn_tree(GdnTreeArgs a, int sms, cudaStream_t st) {
    // one CTA per value head while that leaves SMs without a second CTA; else a key head's value heads share its rows
    // and their products (16 trees of 21: 49.8 us shared, 51.3 not; 32 chains of 64: 161.6 and 169.8; one of 8: 26.0 and 15.1)
    a.heads = a.batch * a.n_v <= 2 * sms ? 1 : a.n_v / a.n_qk;
    switch (rounded_nodes(a.max_nodes)) {
        case 16: return launch<16>(a, st);
        case 32: return launch<32>(a, st);
        case 48: return launch<48>(a, st);
        default: return launch<64>(a, st);
    }
}

size_t gdn_tree_workspace_bytes(int batch, int max_nodes, int n_v, int n_qk) {
    return verify_workspace(nullptr, batch, max_nodes, n_v, n_qk).bytes;
}

cudaError_t launch_gdn_tree_commit(const GdnTreeArgs& a, cudaStream_t st) {
    gdn_tree_path_kernel<<<dim3(unsigned((a.n_qk + a.n_v + kPathWarps - 1) / kPathWarps), unsigned(a.batch)), kPathWarps * 32, 0, st>>>(a);
    return launch_behind(gdn_tree_commit_kernel, dim3(unsigned(kParts * a.n_v + (a.conv_dim + kCommitThreads - 1) / kCommitThreads), unsigned(a.batch)),
                         kCommitThreads, sizeof(CommitSmem), st, a);
}

}  // namespace rl
