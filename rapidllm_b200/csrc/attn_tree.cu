// Attention of a tree of drafted tokens over the paged F16 cache, for a ragged batch, on tcgen05 / TMEM.
//
//   o_i = sigmoid(gate_i) sum_t softmax_t(q_i . k_t / 16) v_t   over the rows t < base_len[b] of the cache
//         and the rows base_len[b] + j of node i's ancestors j and its own
//
// All query rows of a KV head -- (node, query head of the group) pairs, up to 64 x 8 -- share its K and V,
// so the 128 rows of an MMA tile are such pairs and a sequence's pages are read once per 128 rows (at 24 / 4
// heads: once for up to 21 nodes).  Up to there the cache's bandwidth is the bound (16 trees of 21 over 16K, 16-bit
// queries: 779 MB in 151 us at burst clocks, boundaries included; 171 us a call sustained).  Beyond it no unit is (4 trees
// of 64 over 32K: 189 us at burst clocks, 212 a call sustained; HBM 32 % busy, L2 26 %, tensor pipe 42 %, issue slots 33 %):
// a page's time is the chain S -> tensor-memory loads -> exponentials -> P -> P V with two pages in it, S being
// M 128 x N 64 products of about 45 clocks instead of 32; half of the warps' waits are for loads.  The 16 softmax warps
// have 96 registers a thread and spill (288 bytes of stores a thread, 494 with fp32 queries), about as the prefill kernel.
//
// Work division: the (sequence, KV head, row tile, page) units of the whole batch form one list, computed on
// the device from base_len and n_nodes (a captured step may advance them), and every CTA of a persistent
// grid takes a contiguous share of equal cost, cut into segments at (sequence, head, row tile) boundaries; a
// boundary is charged as some pages.  The page ring runs on across segments.  A segment's (unnormalised o, max,
// sum) go to slot `CTA + segment index`, distinct because a CTA's last segment is the next one's first at most;
// attn_tree_merge_kernel joins them, applies the gate and rounds.  Segments that hold all pages of their rows go
// the same way: here a lane has a row, whose gate it would read 16 bytes from a line at a time (all outputs written
// by the merge: 1 x 8 nodes over 120 tokens 14.1 us against 20.2, 16 x 64 over 2000 123 against 146).
//
// Inside a segment: S = Q K^T (M 128, N 64) and O += P V (M 128, N 256) with Q, P, S and O in tensor memory and the
// pages consumed as they lie in HBM (their slices are stored in the tensor cores' tile format).  16 softmax warps in
// two groups take alternate pages, so that one page's exponentials run under the other's MMAs; the row maximum is
// handed from page to page and only raised by more than 2^8.  P is rounded to fp16, as the cache's V is and as prefill
// and decode hold it: 2^-11 of a weight at most, which a sum over many tokens averages (against 64 bits 2.6e-4 instead
// of 2.1e-4 with fp16 outputs, 1.67e-3 instead of 1.66e-3 with bf16; a second term of P would take 204 us instead of
// 173 on the 16 trees, 258 instead of 212 on the 4).  Sums, maxima and O are fp32.  Q is scaled per row by a power of
// two before its rounding to fp16, so that no magnitude of a query overflows it; the score takes the scale back.  An
// fp32 query is two such terms, whatever the output's type, the second from shared memory in the place of a third page
// of the ring: an error of the scores is one of the weights, which no rounding of the output hides where values of
// both signs all but cancel.  It costs a quarter of the time (16 trees of 21 over 16K: 180 us against 154 at burst
// clocks, 212 against 170 sustained), which a caller saves by asking rl_attn_qk_append for 16-bit queries.
// Positions past the committed rows are visible by a bit of the node's ancestor word; K columns that are
// not are replaced, not added to, so that what an unused row of the last page holds cannot matter, and V
// rows past the last node are cleared for the same reason.  A drafted V row that is not finite would reach the
// node's siblings as 0 * inf: it is cleared too, and the rows that see it get NaN through their sum.
#include "common.cuh"
#include "kernels.h"
#include "launch.cuh"
#include "tcgen05.cuh"
#include "tree.cuh"

namespace rl {

namespace {

constexpr int kRows = 128;                        // MMA rows: (node, query head of the group)
constexpr int kTile = kPageTokens;
constexpr int kMaxStages = 3;                     // K and V pages in shared memory; 2 where the queries' second term takes the third's place
constexpr int kSliceBytes = kPageTokens * kHeadDim * 2;
constexpr int kGroupThreads = 256, kSoftmaxThreads = 512, kThreads = 608;
constexpr int kWarpLoader = 16, kWarpQK = 17, kWarpPV = 18;
constexpr uint32_t kTmemCols = 512;
// tensor memory columns: two S buffers [0,128), O [128,384), Q (fp16 pairs) [384,512).  The P of a page replaces the
// first 32 columns of its own S, so that the next page's S is computed while this one is exponentiated.
constexpr uint32_t kColS = 0, kColO = 128, kColQ = 384;
constexpr float kRescaleThreshold = 8.f;          // log2 units
// P is held times 2^kWeightLift, the largest weight in [2^kWeightLift, 2^15]: fp16's last step, 2^-24, is then 2^-31 of that
// weight or less (without the factor tokens of weight e^-17.5 counted as 0, however many).
// Sums and O carry the same factor, which the division takes out.  A lower threshold leaves room for a larger factor, but
// every raise waits for O (4 x 64 nodes over 32K sustained: 210 us with 8, 224 with 4, 230 with 2).
constexpr float kWeightLift = 15.f - kRescaleThreshold;
constexpr float kNoMax = -1e30f;                   // of a row that has seen nothing; scores are below 2^8 * 65504 * 256
constexpr int kMaxBatch = 512;

struct Segment {
    int b, h, rt, index;                          // index: running number of (b, h, rt)
    int j0, n_tiles, tiles;                       // page(0) .. page(n_tiles - 1) of the sequence's `tiles`; n_tiles 0: only the charge
    int base, nodes;
    int next;                                     // position of the next segment
    __device__ __forceinline__ int page(int j) const { return j0 + j < tiles ? j0 + j : j0 + j - tiles; }
};

// cost and segments of the sequences before b; entry `batch` holds the totals
struct Prefix {
    int unit[kMaxBatch + 1], seg[kMaxBatch + 1];
    int base[kMaxBatch], nodes[kMaxBatch];
};

struct Seq {
    int base, nodes, tiles, row_tiles;
};
__device__ __forceinline__ Seq sequence(const AttnTreeArgs& a, int base, int nodes, int* err) {
    Seq q;
    q.nodes = nodes;
    q.base = base;
    if (q.base < 0 || (long long)q.base + q.nodes > a.max_len) {
        set_err(err, DEV_ERR_BAD_LEN);
        q.nodes = 0;
    }
    q.tiles = q.nodes ? (q.base + q.nodes + kTile - 1) / kTile : 0;
    q.row_tiles = (q.nodes * (a.n_q / a.n_kv) + kRows - 1) / kRows;
    return q;
}
// one warp; every CTA computes the same table
__device__ __forceinline__ void build_prefix(Prefix& p, const AttnTreeArgs& a, int lane, int* err) {
    int units = 0, segs = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 32) {
        const int b = b0 + lane;
        int u = 0, g = 0;
        if (b < a.batch) {
            const Seq q = sequence(a, a.base_len[b], tree::node_count(a.n_nodes, b, a.max_nodes, err), err);
            p.base[b] = q.base;
            p.nodes[b] = q.nodes;
            g = a.n_kv * q.row_tiles;
            u = g * (q.tiles + a.boundary);
        }
        int su = u, sg = g;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, su, off), y = __shfl_up_sync(0xffffffffu, sg, off);
            if (lane >= off) {
                su += x;
                sg += y;
            }
        }
        if (b < a.batch) {
            p.unit[b] = units + su - u;
            p.seg[b] = segs + sg - g;
        }
        units += __shfl_sync(0xffffffffu, su, 31);
        segs += __shfl_sync(0xffffffffu, sg, 31);
    }
    if (lane == 0) {
        p.unit[a.batch] = units;
        p.seg[a.batch] = segs;
    }
}
// cost per CTA
__device__ __forceinline__ int share_of(int units, const AttnTreeArgs& a) {
    return max((units + a.grid - 1) / a.grid, a.min_share);
}
// the segment at position `pos` of a share that ends at `end`; b: a sequence at or before it.  A (sequence, head, row
// tile) spans `boundary` positions of charge, then its pages.  Row tiles of a head take the pages in an order rotated so
// that those at the same place of two shares, which run at the same time, are the same ones: read from HBM once, not
// once per row tile.
__device__ __forceinline__ Segment segment_at(const Prefix& p, const AttnTreeArgs& a, int share, int pos, int end, int& b) {
    while (p.unit[b + 1] <= pos) ++b;
    Segment s;
    const Seq q = sequence(a, p.base[b], p.nodes[b], nullptr);
    const int span = q.tiles + a.boundary, in = pos - p.unit[b], hr = in / span, at = in - hr * span - a.boundary;
    s.b = b;
    s.h = hr / q.row_tiles;
    s.rt = hr - s.h * q.row_tiles;
    s.index = p.seg[b] + hr;
    s.j0 = max(at, 0);
    s.next = min(end, pos + q.tiles - at);
    s.n_tiles = max(at + s.next - pos - s.j0, 0);
    s.tiles = q.tiles;
    if (s.rt) s.j0 = (s.j0 + s.rt * span % share) % q.tiles;
    s.base = q.base;
    s.nodes = q.nodes;
    return s;
}

struct Smem {
    alignas(1024) unsigned char k[kMaxStages][kSliceBytes];
    alignas(1024) unsigned char v[kMaxStages][kSliceBytes];
    Prefix prefix;
    uint64_t k_full[kMaxStages], k_empty[kMaxStages], v_full[kMaxStages], v_empty[kMaxStages];
    // rows of Q's second term, 64 dims per tile of 128 rows x 128 bytes (128-byte swizzle), in the last stage's place
    __device__ __forceinline__ unsigned char* q_lo(int sub) { return (sub < 2 ? k : v)[kMaxStages - 1] + (sub & 1) * (kRows * 128); }
    uint64_t bar_s[2], bar_p[2], bar_pv[2], bar_m[2], bar_q;
    float xch[2][2][kRows][2];                    // [group][use parity] row maxima of the two column halves
    float mrow[2][kRows];                         // [page parity] running row maximum, in units of S
    alignas(8) unsigned char v_bad[2][8];         // [group][warp] drafted V rows of its page that are not finite
    alignas(16) float part[kRows][4];             // per row: the four threads' query maxima, later their sums
    uint32_t tmem_base;
    int failed;
};

__device__ __forceinline__ float sigmoid(float g) { return __frcp_rn(1.f + fast_exp2(g * -1.4426950408889634f)); }
__device__ __forceinline__ uint32_t pack_b2(float lo, float hi) {
    __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&b);
}
// 32 bytes per thread: a whole sector of a row that is the thread's own
__device__ __forceinline__ void ld_sector(const void* p, uint32_t (&r)[8]) {
    asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "l"(p));
}
__device__ __forceinline__ void st_sector(void* p, const uint32_t (&r)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]),
                 "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
// 64 query values of type q_type from src, as floats
__device__ __forceinline__ void load_q(float (&x)[64], const void* q, int q_type, size_t at) {
    if (q_type == 0) {
        const float* p = static_cast<const float*>(q) + at;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            uint32_t w[8];
            ld_sector(p + 8 * i, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[8 * i + e] = __uint_as_float(w[e]);
        }
    } else {
        const uint16_t* p = static_cast<const uint16_t*>(q) + at;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t w[8];
            ld_sector(p + 16 * i, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float2 f = q_type == 1 ? __half22float2(*reinterpret_cast<const __half2*>(&w[e]))
                                             : __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[e]));
                x[16 * i + 2 * e] = f.x;
                x[16 * i + 2 * e + 1] = f.y;
            }
        }
    }
}
// an infinity or a NaN in a pair of fp16
__device__ __forceinline__ bool has_special(uint32_t x) { return (x & 0x7c00u) == 0x7c00u || (x & 0x7c000000u) == 0x7c000000u; }

}  // namespace

template <bool kTwoTerms>
__global__ void __launch_bounds__(kThreads, 1) attn_tree_kernel(AttnTreeArgs a) {
    constexpr int kStages = kTwoTerms ? kMaxStages - 1 : kMaxStages;
    extern __shared__ unsigned char smem_raw[];
    // (aligned by an offset, not by integer arithmetic on the pointer: the compiler keeps the loads shared-space ones)
    Smem& s = *reinterpret_cast<Smem*>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = a.n_q / a.n_kv;
    griddep_launch();
    if (warp == 0) build_prefix(s.prefix, a, lane, a.err);
    if (tid == 32) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&s.k_full[i], 1);
            mbar_init(&s.k_empty[i], 1);
        }
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&s.v_full[i], 1);
            mbar_init(&s.v_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s.bar_s[i], 1);
            mbar_init(&s.bar_p[i], kGroupThreads);
            mbar_init(&s.bar_pv[i], 1);
            mbar_init(&s.bar_m[i], kGroupThreads);
        }
        mbar_init(&s.bar_q, kSoftmaxThreads);
        s.failed = 0;
        mbar_fence_init();
    }
    if (warp == kWarpQK) tc::tmem_alloc(&s.tmem_base, kTmemCols);
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = s.tmem_base;
    const int units = s.prefix.unit[a.batch], share = share_of(units, a);
    const int u_begin = int(min((long long)units, (long long)share * blockIdx.x)), u_end = min(units, u_begin + share);

    if (warp == kWarpLoader) {
        // ------------------------------ page loader ------------------------------
        // The warp starts a segment's query rows (but the first's) and its sequence's parents on their way into L2
        // when it starts on its pages, several pages ahead of the softmax warps; then lane 0 waits and copies.
        int b = 0, it = 0;
        bool ok = true;
        for (int pos = u_begin; pos < u_end && ok;) {
            const Segment g = segment_at(s.prefix, a, share, pos, u_end, b);
            const bool first = pos == u_begin;
            pos = g.next;
            if (!g.n_tiles) continue;
            if (!first) {
                const int row_bytes = kHeadDim * (a.q_type == 0 ? 4 : 2), lines = row_bytes / 128;
                const int rows = min(kRows, g.nodes * G - g.rt * kRows);
                for (int i = lane; i < rows * lines; i += 32) {
                    const int row = g.rt * kRows + i / lines, node = row / G;
                    const size_t flat = (size_t(g.b) * a.max_nodes + node) * a.n_q + g.h * G + row - node * G;
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const char*>(a.q) + flat * row_bytes + (i % lines) * 128));
                }
                if (a.parents && lane < 2) asm volatile("prefetch.global.L2 [%0];" ::"l"(a.parents + size_t(g.b) * a.max_nodes + min(lane * 32, a.max_nodes - 1)));
            }
            const int32_t* table = a.page_table + size_t(g.b) * a.max_pages_per_seq;
            for (int j0 = 0; j0 < g.n_tiles && ok; j0 += 32) {
                // 32 page ids at a time: the table's latency is paid once per 32 pages
                int mine = 0;
                if (j0 + lane < g.n_tiles) {
                    mine = table[g.page(j0 + lane)];
                    if (mine < 0 || mine >= a.n_pages) {
                        set_err(a.err, DEV_ERR_BAD_PAGE);
                        mine = 0;
                    }
                }
                const int count = min(32, g.n_tiles - j0);
                for (int j = 0; j < count; ++j, ++it) {
                    const int page = __shfl_sync(0xffffffffu, mine, j);
                    if (lane != 0 || !ok) continue;
                    const int ks = it % kStages, vs = it % kStages;
                    const size_t slice = (size_t(page) * a.n_kv + g.h) * kv_slice_elems();
                    if (!mbar_wait(&s.k_empty[ks], ((it / kStages) & 1) ^ 1)) { ok = false; continue; }
                    mbar_arrive_expect_tx(&s.k_full[ks], kSliceBytes);
                    bulk_g2s(s.k[ks], a.k_pool + slice, kSliceBytes, &s.k_full[ks]);
                    if (!mbar_wait(&s.v_empty[vs], ((it / kStages) & 1) ^ 1)) { ok = false; continue; }
                    mbar_arrive_expect_tx(&s.v_full[vs], kSliceBytes);
                    bulk_g2s(s.v[vs], a.v_pool + slice, kSliceBytes, &s.v_full[vs]);
                }
                ok = __shfl_sync(0xffffffffu, int(ok), 0);
            }
        }
        if (!ok && lane == 0) {
            set_err(a.err, DEV_ERR_WAIT_TIMEOUT);
            s.failed = 1;
        }
    } else if (warp == kWarpQK) {
        // ------------------------------ S = Q K^T issuer ------------------------------
        if (lane == 0) {
            constexpr uint32_t idesc_qk = tc::idesc_f16(kRows, kTile, false, false);
            uint64_t k_desc[kStages];
#pragma unroll
            for (int i = 0; i < kStages; ++i) k_desc[i] = tc::smem_desc(smem_u32(s.k[i]), 16, 1024);
            const uint32_t q_tmem = tmem + kColQ;
            uint64_t lo_desc[4] = {};
            if (kTwoTerms) {
#pragma unroll
                for (int i = 0; i < 4; ++i) lo_desc[i] = tc::smem_desc(smem_u32(s.q_lo(i)), 16, 1024);
            }
            int b = 0, it = 0, sg = 0;
            bool ok = true;
            for (int pos = u_begin; pos < u_end && ok;) {
                const Segment g = segment_at(s.prefix, a, share, pos, u_end, b);
                pos = g.next;
                if (!g.n_tiles) continue;
                ok = mbar_wait(&s.bar_q, sg & 1);
                ++sg;
                for (int j = 0; j < g.n_tiles && ok; ++j, ++it) {
                    const int st = it % kStages;
                    if (!mbar_wait(&s.k_full[st], (it / kStages) & 1)) { ok = false; break; }
                    // this S buffer held the P of two pages before
                    if (it >= 2 && !mbar_wait(&s.bar_pv[it & 1], ((it - 2) >> 1) & 1)) { ok = false; break; }
                    tc::fence_after_sync();
                    const uint32_t s_tmem = tmem + kColS + (it & 1) * 64;
                    const uint64_t kd = st == 0 ? k_desc[0] : (st == 1 ? k_desc[1] : k_desc[kStages - 1]);
#pragma unroll
                    for (int kk = 0; kk < 16; ++kk) {
                        const uint64_t kd16 = kd + uint64_t(((kk >> 2) * (kTile * 128) + (kk & 3) * 32) >> 4);
                        if (kTwoTerms) tc::mma_ss(s_tmem, lo_desc[kk >> 2] + (kk & 3) * 2, kd16, idesc_qk, kk > 0);
                        tc::mma_ts(s_tmem, q_tmem + kk * 8, kd16, idesc_qk, kTwoTerms || kk > 0);
                    }
                    tc::commit(&s.k_empty[st]);
                    tc::commit(&s.bar_s[it & 1]);
                }
            }
            if (!ok) {
                set_err(a.err, DEV_ERR_WAIT_TIMEOUT);
                s.failed = 1;
            }
        }
    } else if (warp == kWarpPV) {
        // ------------------------------ O += P V issuer ------------------------------
        if (lane == 0) {
            constexpr uint32_t idesc_pv = tc::idesc_f16(kRows, kHeadDim, false, true);
            uint64_t v_desc[kStages];
#pragma unroll
            for (int i = 0; i < kStages; ++i) v_desc[i] = tc::smem_desc(smem_u32(s.v[i]), kTile * 128, 1024);
            int b = 0, it = 0;
            bool ok = true;
            for (int pos = u_begin; pos < u_end && ok;) {
                const Segment g = segment_at(s.prefix, a, share, pos, u_end, b);
                pos = g.next;
                if (!g.n_tiles) continue;
                for (int j = 0; j < g.n_tiles; ++j, ++it) {
                    const int st = it % kStages;
                    if (!mbar_wait(&s.v_full[st], (it / kStages) & 1)) { ok = false; break; }
                    // P of a segment's first page is published after every thread has read the segment before's O
                    if (!mbar_wait(&s.bar_p[it & 1], (it >> 1) & 1)) { ok = false; break; }
                    tc::fence_after_sync();
                    const uint64_t vd = st == 0 ? v_desc[0] : (st == 1 ? v_desc[1] : v_desc[kStages - 1]);
                    const uint32_t p_tmem = tmem + kColS + (it & 1) * 64;
                    tc::mma_ts(tmem + kColO, p_tmem, vd, idesc_pv, j > 0);
#pragma unroll
                    for (int kk = 1; kk < 4; ++kk)
                        tc::mma_ts(tmem + kColO, p_tmem + kk * 8, vd + uint64_t((kk * 16 * 128) >> 4), idesc_pv, 1);
                    tc::commit(&s.v_empty[st]);
                    tc::commit(&s.bar_pv[it & 1]);
                }
            }
            if (!ok) {
                set_err(a.err, DEV_ERR_WAIT_TIMEOUT);
                s.failed = 1;
            }
        }
    } else {
        // ------------------------------ softmax warps ------------------------------
        const int grp = warp >> 3, half = (warp >> 2) & 1, quad = warp & 3, quarter = warp >> 2;
        const int r = quad * 32 + lane;                       // row of the tile = TMEM lane
        const uint32_t lane_addr = tmem + (uint32_t(quad * 32) << 16);
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t parity) {     // `ok` is the same in all lanes of a warp
            if (ok && !__all_sync(0xffffffffu, mbar_wait(bar, parity))) {
                set_err(a.err, DEV_ERR_WAIT_TIMEOUT);
                ok = false;
            }
        };
        int b = 0, it0 = 0;                                   // it0: pages of the segments before
        for (int pos = u_begin; pos < u_end;) {
            const Segment g = segment_at(s.prefix, a, share, pos, u_end, b);
            pos = g.next;
            if (!g.n_tiles) continue;
            const int row = g.rt * kRows + r, node = row / G, hq = g.h * G + row - node * G;
            const bool live = node < g.nodes;
            const size_t flat = (size_t(g.b) * a.max_nodes + (live ? node : 0)) * a.n_q + hq;
            // ---- Q -> tensor memory: 64 dims per thread, the row scaled to a largest magnitude in [128, 256) ----
            float scale_log2 = a.scale * 1.4426950408889634f;
            {
                float x[64];
                if (live) {
                    load_q(x, a.q, a.q_type, flat * kHeadDim + quarter * 64);
                } else {
#pragma unroll
                    for (int i = 0; i < 64; ++i) x[i] = 0.f;
                }
                float mx = 0.f;
#pragma unroll
                for (int i = 0; i < 64; ++i) mx = fmaxf(mx, fabsf(x[i]));
                s.part[r][quarter] = mx;
                named_bar_sync(9, kSoftmaxThreads);
                const float4 m4 = *reinterpret_cast<const float4*>(s.part[r]);
                mx = fmaxf(fmaxf(m4.x, m4.y), fmaxf(m4.z, m4.w));
                const int e = int(__float_as_uint(mx) >> 23) - 127;
                const int up = mx > 0.f && e < 128 ? min(max(7 - e, -120), 120) : 0;
                const float f = __uint_as_float(uint32_t(127 + up) << 23);
                scale_log2 *= __uint_as_float(uint32_t(127 - up) << 23);
                uint32_t regs[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) regs[i] = pack_h2(x[2 * i] * f, x[2 * i + 1] * f);
                if (kTwoTerms) {
                    unsigned char* row_lo = s.q_lo(quarter) + r * 128;
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        uint32_t w[4];
#pragma unroll
                        for (int z = 0; z < 4; ++z) {
                            const float2 hi = __half22float2(*reinterpret_cast<const __half2*>(&regs[i + z]));
                            w[z] = pack_h2(fmaf(x[2 * (i + z)], f, -hi.x), fmaf(x[2 * (i + z) + 1], f, -hi.y));
                        }
                        *reinterpret_cast<uint4*>(row_lo + (((i / 4) ^ (r & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                    tc::fence_async_smem();
                }
                tc::tmem_st32(lane_addr + kColQ + quarter * 32, regs);
                tc::tmem_wait_st();
                tc::fence_before_sync();
                mbar_arrive(&s.bar_q);
            }
            // ---- this row's visible nodes ----
            unsigned long long seen = 0;
            if (min(g.j0 + g.n_tiles, g.tiles) * kTile > g.base) {        // the segment reaches the drafted rows
                const tree::Words w = tree::ancestors(a.parents ? a.parents + size_t(g.b) * a.max_nodes : nullptr, g.nodes, lane, a.err);
                seen = tree::of_node(w.lo, w.hi, node & 63);
            }
            const int last_pos = g.base + g.nodes - 1;
            float m_known = kNoMax, l_part = 0.f;             // maxima are kept as the scores they are, unscaled
            for (int j = (grp ^ it0) & 1; j < g.n_tiles; j += 2) {
                const int it = it0 + j;                       // it & 1 == grp
                const uint32_t par = (it >> 1) & 1;
                wait(&s.bar_s[grp], par);
                tc::fence_after_sync();
                uint32_t raw[32];
                if (ok) {
                    tc::tmem_ld32(lane_addr + kColS + grp * 64 + half * 32, raw);
                    tc::tmem_wait_ld();
                }
                const int tok0 = g.page(j) * kTile;
                const bool drafted = tok0 + kTile > g.base;   // rows behind the committed ones
                const int first = max(g.base - tok0, 0);
                if (drafted) {
                    // each warp clears its share of the V rows past the last node, and of the drafted ones that are not finite
                    wait(&s.v_full[it % kStages], (it / kStages) & 1);
                    const int end = last_pos + 1 - tok0;
                    uint32_t found = 0;
                    for (int vr = first + (warp & 7), bit = 1; vr < kTile; vr += 8, bit <<= 1) {
                        uint4* at = reinterpret_cast<uint4*>(s.v[it % kStages] + (lane >> 3) * (kTile * 128) + vr * 128 + (lane & 7) * 16);
                        bool clear = vr >= end;
                        if (!clear) {
                            const uint4 x = *at;
                            clear = __any_sync(0xffffffffu, has_special(x.x) || has_special(x.y) || has_special(x.z) || has_special(x.w));
                            if (clear) found |= bit;
                        }
                        if (clear) *at = make_uint4(0, 0, 0, 0);
                    }
                    if (lane == 0) s.v_bad[grp][warp & 7] = static_cast<unsigned char>(found);
                    tc::fence_async_smem();
                }
                float mx = kNoMax;
                if (drafted) {
                    // bit i of `vis`: token tok0 + 32 half + i is committed, or a node that this row sees
                    const int rel = tok0 + half * 32 - g.base;
                    uint32_t vis;
                    if (rel >= 0) vis = rel < 64 ? uint32_t(seen >> rel) : 0u;
                    else vis = rel <= -32 ? 0xffffffffu : (uint32_t(seen << -rel) | ((1u << -rel) - 1));
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        if (!(vis >> i & 1)) raw[i] = 0xff800000u;         // -inf
                        mx = fmaxf(mx, __uint_as_float(raw[i]));
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) mx = fmaxf(mx, __uint_as_float(raw[i]));
                }
                s.xch[grp][par][r][half] = mx;
                named_bar_sync(1 + grp * 4 + quad, 64);
                mx = fmaxf(mx, s.xch[grp][par][r][half ^ 1]);
                float m_prev = kNoMax;
                if (j > 0) {
                    wait(&s.bar_m[grp ^ 1], ((it - 1) >> 1) & 1);
                    m_prev = s.mrow[grp ^ 1][r];
                }
                float m_new = m_prev, alpha = 1.f;
                if (mx > m_prev && (m_prev == kNoMax || (mx - m_prev) * scale_log2 > kRescaleThreshold)) {
                    alpha = fast_exp2((m_prev - mx) * scale_log2);
                    m_new = mx;
                }
                if (half == 0) s.mrow[grp][r] = m_new;
                mbar_arrive(&s.bar_m[grp]);
                if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
                    wait(&s.bar_pv[grp ^ 1], ((it - 1) >> 1) & 1);         // O must not be in use
                    tc::fence_after_sync();
                    if (ok) {
#pragma unroll 1
                        for (int c0 = 0; c0 < kHeadDim / 2; c0 += 32) {
                            uint32_t o[32];
                            tc::tmem_ld32(lane_addr + kColO + half * 128 + c0, o);
                            tc::tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                            tc::tmem_st32(lane_addr + kColO + half * 128 + c0, o);
                        }
                        tc::tmem_wait_st();
                    }
                }
                if (m_new != m_known) {
                    l_part *= fast_exp2((m_known - m_new) * scale_log2);
                    m_known = m_new;
                }
                // p = 2^((s - m) scale) as one FFMA and one EX2.  m scale is rounded, the same for the whole row; only
                // where that rounding is itself a large exponent (|m scale| > 2^20) is the difference taken first.
                float m_log2 = m_new == kNoMax ? 0.f : m_new * scale_log2;
                if (__any_sync(0xffffffffu, fabsf(m_log2) > 1048576.f)) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) raw[i] = __float_as_uint(__uint_as_float(raw[i]) - m_new);
                    m_log2 = 0.f;
                }
                m_log2 -= kWeightLift;
                uint32_t ph[16];
                float lsum0 = 0.f, lsum1 = 0.f;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float p0 = fast_exp2(fmaf(__uint_as_float(raw[2 * i]), scale_log2, -m_log2));
                    const float p1 = fast_exp2(fmaf(__uint_as_float(raw[2 * i + 1]), scale_log2, -m_log2));
                    lsum0 += p0;
                    lsum1 += p1;
                    ph[i] = pack_h2(p0, p1);
                }
                l_part += lsum0 + lsum1;
                if (drafted) {
                    named_bar_sync(10 + grp, kGroupThreads);
                    if (unsigned long long bad = *reinterpret_cast<const unsigned long long*>(s.v_bad[grp])) {
                        for (; bad; bad &= bad - 1) {         // bit 8 w + z: row first + w + 8 z
                            const int bit = __ffsll(bad) - 1, rel = tok0 + first + (bit >> 3) + 8 * (bit & 7) - g.base;
                            if (seen >> rel & 1) l_part = __uint_as_float(0x7fc00000u);
                        }
                    }
                }
                if (ok) {                                     // both halves' scores left the buffer before the maxima met
                    tc::tmem_st16(lane_addr + kColS + grp * 64 + half * 16, ph);
                    tc::tmem_wait_st();
                }
                tc::fence_before_sync();
                mbar_arrive(&s.bar_p[grp]);
            }
            // ---- end of the segment ----
            it0 += g.n_tiles;
            const int it_last = it0 - 1;
            wait(&s.bar_m[it_last & 1], (it_last >> 1) & 1);
            const float m_fin = s.mrow[it_last & 1][r];
            s.part[r][quarter] = l_part * fast_exp2((m_known - m_fin) * scale_log2);
            named_bar_sync(9, kSoftmaxThreads);
            const float4 lp = *reinterpret_cast<const float4*>(s.part[r]);
            const float l_run = (lp.x + lp.y) + (lp.z + lp.w);
            wait(&s.bar_pv[it_last & 1], (it_last >> 1) & 1);              // every P.V of the segment is done
            tc::fence_after_sync();
            const size_t slot = size_t(blockIdx.x) + g.index;
            const int col0 = quarter * 64;
            if (ok && __all_sync(0xffffffffu, !*const_cast<volatile int*>(&s.failed))) {
#pragma unroll 1
                for (int c0 = 0; c0 < 64; c0 += 32) {
                    uint32_t raw[32];
                    __syncwarp();
                    tc::tmem_ld32(lane_addr + kColO + col0 + c0, raw);
                    tc::tmem_wait_ld();
                    if (!live) continue;
                    // [slot][dims / 8][row][8]: a warp's 32 rows of 32 bytes are contiguous
                    float* dst = a.part_o + (slot * (kHeadDim / 8) + (col0 + c0) / 8) * (kRows * 8) + r * 8;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t w[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) w[e] = raw[8 * i + e];
                        st_sector(dst + i * (kRows * 8), w);
                    }
                }
                if (live && quarter == 0) *reinterpret_cast<float2*>(a.part_ml + (slot * kRows + r) * 2) = make_float2(m_fin == kNoMax ? kNoMax : m_fin * scale_log2, l_run);
            }
            tc::fence_before_sync();
            named_bar_sync(9, kSoftmaxThreads);               // O, Q and `part` may be rewritten
        }
    }
    __syncthreads();
    if (warp == kWarpQK) tc::tmem_dealloc(tmem, kTmemCols);
}

// Log-sum-exp over a row's slots (log2 domain), gate, rounding.  A thread takes 4 dims of one row (32 bytes of 16 rows
// are contiguous in a slot) with four slots in flight, a block 16 rows; its 4 warps take 4 x 8 dims, or with kSplit a
// quarter of the slots each of the same 8.  Blocks this small fit beside a CTA of the main kernel (56 registers a thread
// are left there), so that they stand ready when its last CTA ends (512 threads: 1 x 8 nodes over 9 000 tokens 30.8 us
// against 26.2, before kSplit).
// grid (n_kv * row tiles * merge_blocks(kSplit), batch).
constexpr int kMergeRows = 16, kAhead = 4, kMergeWarps = 4;
constexpr int merge_chunks(bool split) { return kHeadDim / 8 / (split ? 1 : kMergeWarps); }
constexpr int merge_blocks(bool split) { return kRows / kMergeRows * merge_chunks(split); }     // of a row tile
template <bool kSplit>
__global__ void __launch_bounds__(kMergeWarps * 32, 9) attn_tree_merge_kernel(AttnTreeArgs a) {
    __shared__ Prefix prefix;
    __shared__ float quarter[kMergeWarps - 1][6][32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, b = blockIdx.y;
    const int G = a.n_q / a.n_kv;
    if (tid < 32) build_prefix(prefix, a, tid, nullptr);
    __syncthreads();
    const Seq q = sequence(a, prefix.base[b], prefix.nodes[b], nullptr);
    const int hr = blockIdx.x / merge_blocks(kSplit), part = blockIdx.x % merge_blocks(kSplit);
    const int group = part / merge_chunks(kSplit) * kMergeRows, r = group + (lane >> 1);
    const int d0 = (kSplit ? part % merge_chunks(kSplit) : part % merge_chunks(kSplit) * kMergeWarps + warp) * 8 + (lane & 1) * 4;
    int h = 0, node = 0, hq = 0, first = 0, parts = 0;
    if (hr < a.n_kv * q.row_tiles) {
        h = hr / q.row_tiles;
        const int tr0 = (hr - h * q.row_tiles) * kRows, share = share_of(prefix.unit[a.batch], a);
        node = (tr0 + r) / G;
        hq = h * G + tr0 + r - node * G;
        const int u0 = prefix.unit[b] + hr * (q.tiles + a.boundary) + a.boundary;
        first = u0 / share;
        parts = (tr0 + group) / G < q.nodes ? (u0 + q.tiles - 1) / share - first + 1 : 0;
    }
    // nothing to do.  The grid's first block waits all the same: what follows this kernel then follows the one in front.
    if (parts == 0) {
        if (blockIdx.x == 0 && b == 0) griddep_wait();
        return;
    }
    const bool live = node < q.nodes;
    if (!live) parts = node = hq = 0;
    const size_t row = (size_t(b) * a.max_nodes + node) * a.n_q + hq;
    float4 gate = make_float4(0.f, 0.f, 0.f, 0.f);
    if (a.gate) gate = __ldcs(reinterpret_cast<const float4*>(a.gate + (size_t(b) * a.max_nodes + node) * a.gate_row + size_t(hq) * a.gate_head + d0));
    griddep_wait();
    const size_t slot0 = size_t(first) + prefix.seg[b] + hr;
    const float* ml_at = a.part_ml + (slot0 * kRows + r) * 2;
    const float* o_at = a.part_o + (slot0 * (kHeadDim / 8) + d0 / 8) * (kRows * 8) + r * 8 + (d0 & 7);
    float m = kNoMax, l = 0.f, x[4] = {};
    for (int p0 = kSplit ? warp * kAhead : 0; p0 < parts; p0 += kSplit ? kMergeWarps * kAhead : kAhead) {
        float2 ml[kAhead];
        float4 o[kAhead];
#pragma unroll
        for (int z = 0; z < kAhead; ++z) {
            ml[z] = make_float2(kNoMax, 0.f);
            o[z] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (p0 + z < parts) {
                ml[z] = *reinterpret_cast<const float2*>(ml_at + size_t(p0 + z) * (kRows * 2));
                o[z] = *reinterpret_cast<const float4*>(o_at + size_t(p0 + z) * (kRows * kHeadDim));
            }
        }
        float mx = m;
#pragma unroll
        for (int z = 0; z < kAhead; ++z) mx = fmaxf(mx, ml[z].x);
        const float back = fast_exp2(m - mx);
        m = mx;
        l *= back;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] *= back;
#pragma unroll
        for (int z = 0; z < kAhead; ++z) {
            const float w = fast_exp2(ml[z].x - m);
            l = fmaf(ml[z].y, w, l);
            x[0] = fmaf(o[z].x, w, x[0]);
            x[1] = fmaf(o[z].y, w, x[1]);
            x[2] = fmaf(o[z].z, w, x[2]);
            x[3] = fmaf(o[z].w, w, x[3]);
        }
    }
    if constexpr (kSplit) {
        if (warp) {
            float* to = &quarter[warp - 1][0][lane];
            to[0] = m;
            to[32] = l;
#pragma unroll
            for (int e = 0; e < 4; ++e) to[64 + 32 * e] = x[e];
        }
        __syncthreads();
        if (warp) return;
        float mx = m;
#pragma unroll
        for (int z = 0; z < kMergeWarps - 1; ++z) mx = fmaxf(mx, quarter[z][0][lane]);
        const float back = fast_exp2(m - mx);
        l *= back;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] *= back;
#pragma unroll
        for (int z = 0; z < kMergeWarps - 1; ++z) {
            const float w = fast_exp2(quarter[z][0][lane] - mx);
            l = fmaf(quarter[z][1][lane], w, l);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = fmaf(quarter[z][2 + e][lane], w, x[e]);
        }
    }
    if (!live) return;
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    const float g[4] = {gate.x, gate.y, gate.z, gate.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] *= a.gate ? inv * sigmoid(g[e]) : inv;
    uint32_t w[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) w[e] = a.o_type == 1 ? pack_h2(x[2 * e], x[2 * e + 1]) : pack_b2(x[2 * e], x[2 * e + 1]);
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.o) + row * kHeadDim + d0) = make_uint2(w[0], w[1]);
}

namespace {
constexpr size_t kSmemBytes = sizeof(Smem) + 1024;
}

cudaError_t attn_tree_setup() {
    cudaError_t e = cudaFuncSetAttribute(attn_tree_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kSmemBytes));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(attn_tree_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kSmemBytes));
    return e;
}
int attn_tree_rows() { return kRows; }
int attn_tree_max_batch() { return kMaxBatch; }

cudaError_t launch_attn_tree(const AttnTreeArgs& a, cudaStream_t st) {
    // One term holds 16-bit queries: the row's largest element is scaled into [2^7, 2^8), so that fp16 elements down to 2^-21
    // of it (bf16 to 2^-24) are exact and smaller ones off by 2^-32 of it at most.
    if (a.q_type == 0) attn_tree_kernel<true><<<a.grid, kThreads, kSmemBytes, st>>>(a);
    else attn_tree_kernel<false><<<a.grid, kThreads, kSmemBytes, st>>>(a);
    cudaLaunchConfig_t cfg = {};
    const int row_tiles = (a.max_nodes * (a.n_q / a.n_kv) + kRows - 1) / kRows;
    // Many slots per row: their loads, four at a time, are the merge's time (1 x 8 nodes over 5 000 tokens, 37 slots:
    // 17.9 us split, 23.2 not).  Few: blocks are, and a split has four times as many (4 x 8 over 1 000, 9: 21.1 and 17.5).
    const bool split = a.grid >= 16 * a.batch * a.n_kv * row_tiles;
    cfg.gridDim = dim3(unsigned(a.n_kv * row_tiles * merge_blocks(split)), unsigned(a.batch));
    cfg.blockDim = dim3(kMergeWarps * 32);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return split ? cudaLaunchKernelEx(&cfg, attn_tree_merge_kernel<true>, a) : cudaLaunchKernelEx(&cfg, attn_tree_merge_kernel<false>, a);
}

}  // namespace rl
