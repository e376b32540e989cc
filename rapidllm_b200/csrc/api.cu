// C ABI of the library (include/rl_b200.h): argument checks, launches, the
// device-side cache object and the layer_types[] dispatch.  No exception and no
// C++ type crosses this boundary.
#include "../../include/rl_b200.h"

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <mutex>
#include <new>
#include <string>
#include <vector>

#include "comm.h"
#include "common.cuh"
#include "kernels.h"
#include "launch.cuh"

namespace {

thread_local char g_err[512] = "";

int fail(rl_status st, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof g_err, fmt, ap);
    va_end(ap);
    return st;
}

#define RL_CUDA(call)                                                                    \
    do {                                                                                 \
        cudaError_t e_ = (call);                                                         \
        if (e_ != cudaSuccess)                                                           \
            return fail(e_ == cudaErrorMemoryAllocation ? RL_ERR_NOMEM : RL_ERR_DEVICE,  \
                        "%s: %s", #call, cudaGetErrorString(e_));                        \
    } while (0)

__device__ int g_dev_err;   // device error word (one per device that loads the library)

struct DevInfo {
    bool ready = false;
    int sms = 0;
    int cc_major = 0;
    int* err_ptr = nullptr;
    bool attn_attr = false;
    // second streams + events for the calls that overlap two of their own kernels
    // (rl_delta_chunk_prefill): a pool, one set per call in flight (aux_acquire)
    std::vector<struct AuxSet*> aux_pool;
};
// One side stream with its fork/join events.  A set belongs to one call from aux_acquire()
// until the join event that call recorded last has completed, so two host threads (or two
// streams) running such calls on one device never share events.
struct AuxSet {
    cudaStream_t stream = nullptr;
    cudaEvent_t fork[32] = {};
    cudaEvent_t join = nullptr;
    bool used = false;              // join has been recorded at least once
};
std::mutex g_mu;
}  // namespace
namespace rl {
thread_local bool g_step_overlap = false;
thread_local bool g_step_first = false;
}
namespace {
// SMs the persistent kernels of the step in flight leave free (for the exchange kernels of a sharded step)
thread_local int g_sm_reserve = 0;
// set by the decode step around an append whose rows are the caller's own (KvWriteArgs::early)
thread_local bool g_append_early = false;
// set by the decode step around a decode over the caller's own page table (AttnDecodeArgs::stream_before_wait)
thread_local bool g_decode_early = false;
// set by the decode step around a fused DeltaNet step whose inputs are the caller's (GdnDecodeArgs::early)
thread_local bool g_gdn_early = false;
struct SmReserve {
    int prev;
    explicit SmReserve(int n) : prev(g_sm_reserve) { g_sm_reserve = n; }
    ~SmReserve() { g_sm_reserve = prev; }
};
inline int step_sms(int sms) { return std::max(1, sms - g_sm_reserve); }
}  // namespace
namespace {
DevInfo g_dev[64];

int dev_info(DevInfo** out) {
    int dev = 0;
    RL_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return fail(RL_ERR_RANGE, "device ordinal %d out of range", dev);
    std::lock_guard<std::mutex> lk(g_mu);
    DevInfo& d = g_dev[dev];
    if (!d.ready) {
        cudaDeviceProp prop;
        RL_CUDA(cudaGetDeviceProperties(&prop, dev));
        d.sms = prop.multiProcessorCount;
        d.cc_major = prop.major;
        if (prop.major != 10)
            return fail(RL_ERR_UNSUPPORTED, "device %d is sm_%d%d; this library is built for sm_100a only",
                        dev, prop.major, prop.minor);
        RL_CUDA(cudaGetSymbolAddress(reinterpret_cast<void**>(&d.err_ptr), g_dev_err));
        RL_CUDA(cudaMemset(d.err_ptr, 0, sizeof(int)));
        RL_CUDA(cudaFuncSetAttribute(rl::attn_decode_f16_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     int(rl::attn_decode_f16_smem_bytes())));
        RL_CUDA(cudaFuncSetAttribute(rl::delta_decode_stream_kernel_ptr(), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     int(rl::delta_decode_stream_smem_bytes())));
        RL_CUDA(cudaFuncSetAttribute(rl::gdn_decode_stream_kernel_ptr(), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     int(rl::gdn_decode_stream_smem_bytes())));
        RL_CUDA(cudaFuncSetAttribute(rl::delta_chunk_prepare_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     int(rl::delta_chunk_prepare_smem_bytes())));
        RL_CUDA(cudaFuncSetAttribute(rl::delta_chunk_keys_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     int(rl::delta_chunk_prepare_smem_bytes())));
        RL_CUDA(cudaFuncSetAttribute(rl::delta_chunk_scan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     int(rl::delta_chunk_scan_smem_bytes())));
        RL_CUDA(cudaFuncSetAttribute(rl::attn_prefill_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     int(rl::attn_prefill_smem_bytes())));
        RL_CUDA(cudaFuncSetAttribute(rl::attn_decode_tq_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     int(rl::attn_decode_tq_smem_bytes())));
        RL_CUDA(rl::attn_tree_setup());
        RL_CUDA(rl::gdn_tree_setup());
        d.ready = true;
    }
    *out = &d;
    return RL_OK;
}

// A side-stream set no earlier call is still using: one whose last join event has completed,
// else a new one (the pool only grows to the number of such calls in flight at once).
int aux_acquire(DevInfo* d, AuxSet** out) {
    std::lock_guard<std::mutex> lk(g_mu);
    for (AuxSet* a : d->aux_pool) {
        if (!a->used) { *out = a; return RL_OK; }
        const cudaError_t q = cudaEventQuery(a->join);
        if (q == cudaSuccess) { *out = a; return RL_OK; }
        if (q != cudaErrorNotReady) cudaGetLastError();   // e.g. recorded inside a capture: treat as busy
    }
    AuxSet* a = new (std::nothrow) AuxSet();
    if (!a) return fail(RL_ERR_NOMEM, "host allocation failed");
    int lo = 0, hi = 0;
    cudaError_t e = cudaDeviceGetStreamPriorityRange(&lo, &hi);
    if (e == cudaSuccess) e = cudaStreamCreateWithPriority(&a->stream, cudaStreamNonBlocking, hi);
    for (cudaEvent_t& ev : a->fork)
        if (e == cudaSuccess) e = cudaEventCreateWithFlags(&ev, cudaEventDisableTiming);
    if (e == cudaSuccess) e = cudaEventCreateWithFlags(&a->join, cudaEventDisableTiming);
    if (e != cudaSuccess) {
        for (cudaEvent_t ev : a->fork) if (ev) cudaEventDestroy(ev);
        if (a->join) cudaEventDestroy(a->join);
        if (a->stream) cudaStreamDestroy(a->stream);
        delete a;
        return fail(RL_ERR_DEVICE, "creating a side stream: %s", cudaGetErrorString(e));
    }
    d->aux_pool.push_back(a);
    *out = a;
    return RL_OK;
}

// Marks the launches of a step for programmatic dependent launch while it is alive.
struct StepOverlap {
    bool prev;
    explicit StepOverlap(bool on) : prev(rl::g_step_overlap) { rl::g_step_overlap = on; }
    ~StepOverlap() { rl::g_step_overlap = prev; }
};

inline cudaStream_t as_stream(void* s) { return static_cast<cudaStream_t>(s); }
inline size_t align_up(size_t x, size_t a) { return (x + a - 1) / a * a; }
inline int ceil_div(int a, int b) { return (a + b - 1) / b; }

// ---- split-KV plan: a pure function of the parameters ----------------------------
struct AttnPlan {
    int grid, G;
    size_t part_o_bytes, part_ml_bytes, total_bytes;
};

int attn_check(const rl_attn_decode_params* p) {
    if (!p) return fail(RL_ERR_RANGE, "params is NULL");
    if (p->head_dim != rl::kHeadDim) return fail(RL_ERR_UNSUPPORTED, "head_dim %d: only 256", p->head_dim);
    if (p->page_tokens != rl::kPageTokens) return fail(RL_ERR_UNSUPPORTED, "page_tokens %d: only 64", p->page_tokens);
    if (p->n_kv <= 0 || p->n_q <= 0 || p->n_q % p->n_kv != 0 || p->n_q / p->n_kv > 8)
        return fail(RL_ERR_UNSUPPORTED, "n_q %d / n_kv %d: group must divide and be <= 8", p->n_q, p->n_kv);
    if (p->batch < 0 || p->batch > rl::attn_decode_max_batch())
        return fail(RL_ERR_RANGE, "batch %d outside [0, %d]", p->batch, rl::attn_decode_max_batch());
    if (p->n_pages <= 0 || p->max_pages_per_seq <= 0) return fail(RL_ERR_RANGE, "empty page pool or table");
    if (p->max_seq_len <= 0 || p->max_seq_len > p->max_pages_per_seq * p->page_tokens)
        return fail(RL_ERR_RANGE, "max_seq_len %d outside (0, max_pages_per_seq*page_tokens]", p->max_seq_len);
    if (p->kv_dtype != RL_KV_F16 && p->kv_dtype != RL_KV_Q8K_TQ3V)
        return fail(RL_ERR_UNSUPPORTED, "kv_dtype %d unknown", p->kv_dtype);
    if (p->kv_dtype == RL_KV_Q8K_TQ3V && p->wht_len != 128 && p->wht_len != 256)
        return fail(RL_ERR_UNSUPPORTED, "wht_len %d: only 128 or 256", p->wht_len);
    return RL_OK;
}

// One persistent CTA per SM; fewer when the work is small (a CTA should own at least
// chunk_pages pages, default 1).  One partial slot per CTA plus one per (sequence, KV head).
AttnPlan attn_plan(const rl_attn_decode_params* p, int sms) {
    AttnPlan pl;
    pl.G = p->n_q / p->n_kv;
    const int batch = p->batch > 0 ? p->batch : 1;
    const long long page_heads = 1LL * batch * ceil_div(p->max_seq_len, p->page_tokens) * p->n_kv;
    const int per_cta = p->chunk_pages > 0 ? p->chunk_pages : 1;
    long long grid = (page_heads + per_cta - 1) / per_cta;
    if (grid > sms) grid = sms;
    if (grid < 1) grid = 1;
    pl.grid = int(grid);
    const size_t slots = size_t(pl.grid) + size_t(batch) * p->n_kv;
    pl.part_o_bytes = align_up(slots * pl.G * rl::kHeadDim * sizeof(float), 256);
    pl.part_ml_bytes = align_up(slots * pl.G * 2 * sizeof(float), 256);
    pl.total_bytes = pl.part_o_bytes + pl.part_ml_bytes;
    return pl;
}

// Tuning constants.  The shipped library never looks at the environment; a development build
// (-DRL_B200_DEV_KNOBS) lets a measurement override them once, at load time.
int knob(const char* name, int dflt) {
#ifdef RL_B200_DEV_KNOBS
    if (const char* e = std::getenv(name)) return std::max(0, atoi(e));
#endif
    (void)name;
    return dflt;
}
const int kTqSegWeight = knob("RL_B200_TQ_SEG_WEIGHT", 23);
const int kF16SegWeight = knob("RL_B200_F16_SEG_WEIGHT", 6);
// heads per launch from which the fused DeltaNet step streams whole heads through persistent CTAs
const int kGdnStreamMin = knob("RL_B200_GDN_STREAM_MIN", 96);
const int kGdnGrid = knob("RL_B200_GDN_GRID", 0);       // development builds: force the streaming form's grid
const int kDeltaChunkSegs = knob("RL_B200_DELTA_SEGS", 0);   // development builds: force the segment count of the chunked prefill

int attn_decode_impl(const void* k_pool, const void* v_pool, const int32_t* page_table,
                     const int32_t* seq_lens, const float* q, const float* gate, float* o, float* out_ml,
                     void* workspace, size_t workspace_bytes, const rl_attn_decode_params* p, void* stream,
                     cudaEvent_t after_main = nullptr) {
    if (int st = attn_check(p)) return st;
    if (p->batch == 0) return RL_OK;
    const bool tq = p->kv_dtype == RL_KV_Q8K_TQ3V;
    if (!k_pool || (!v_pool && !tq) || !page_table || !seq_lens || !q || !o || !workspace)
        return fail(RL_ERR_RANGE, "NULL pointer argument");
    DevInfo* d;
    if (int st = dev_info(&d)) return st;
    const AttnPlan pl = attn_plan(p, step_sms(d->sms));
    if (workspace_bytes < pl.total_bytes)
        return fail(RL_ERR_RANGE, "workspace %zu bytes < %zu required", workspace_bytes, pl.total_bytes);
    if (reinterpret_cast<uintptr_t>(k_pool) % 128 || (!tq && reinterpret_cast<uintptr_t>(v_pool) % 128) ||
        reinterpret_cast<uintptr_t>(q) % 16 || reinterpret_cast<uintptr_t>(workspace) % 16)
        return fail(RL_ERR_RANGE, "pools must be 128-byte aligned, q and workspace 16-byte aligned");
    rl::AttnDecodeArgs a;
    a.k_pool = static_cast<const __half*>(k_pool);
    a.v_pool = static_cast<const __half*>(v_pool);
    a.page_table = page_table;
    a.seq_lens = seq_lens;
    a.q = q;
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = reinterpret_cast<float*>(static_cast<char*>(workspace) + pl.part_o_bytes);
    a.err = d->err_ptr;
    a.batch = p->batch;
    a.n_q = p->n_q;
    a.n_kv = p->n_kv;
    a.n_pages = p->n_pages;
    a.max_pages_per_seq = p->max_pages_per_seq;
    a.len_add = p->len_add;
    a.scale = 1.f / sqrtf(float(p->head_dim));
    // A CTA that closes one (sequence, head) segment and opens the next spends a few microseconds on
    // it (compact KV: ~6 us, the time of ~23 records of 32 tokens at 44 GB/s per SM; F16: the time of
    // ~6 half pages).  While only a minority of the CTAs have a boundary in their range, those CTAs
    // are the last to finish, so their share of the units is cut by that much; once nearly every CTA
    // has one (segments > CTAs / 4) the division stays equal in units, which measured faster there.
    a.seg_weight = p->batch * p->n_kv * 4 <= pl.grid ? (tq ? kTqSegWeight : kF16SegWeight) : 0;
    a.stream_before_wait = !tq && g_decode_early && rl::g_step_overlap && !rl::g_step_first ? 1 : 0;
    const int grid = pl.grid;
    if (tq)
        rl::attn_decode_tq_kernel<<<grid, rl::attn_decode_tq_threads(), rl::attn_decode_tq_smem_bytes(),
                                    as_stream(stream)>>>(a);
    else
        RL_CUDA(rl::launch_step(rl::attn_decode_f16_kernel, dim3(grid), dim3(rl::attn_decode_f16_threads()),
                                rl::attn_decode_f16_smem_bytes(), as_stream(stream), a));
    if (after_main) cudaEventRecord(after_main, as_stream(stream));
    rl::AttnCombineArgs c;
    c.part_o = a.part_o;
    c.part_ml = a.part_ml;
    c.seq_lens = seq_lens;
    c.gate = gate;
    c.o = o;
    c.out_ml = out_ml;
    c.batch = p->batch;
    c.n_q = p->n_q;
    c.n_kv = p->n_kv;
    c.len_add = p->len_add;
    c.n_ctas = grid;
    c.seg_weight = a.seg_weight;
    c.max_len = p->max_pages_per_seq * p->page_tokens;
    c.wht_len = (tq && !out_ml) ? p->wht_len : 0;      // partial outputs stay in the rotated domain
    c.signs = (tq && p->wht_len == 256) ? p->tq_signs : nullptr;
    {
        // the merge always follows its decode kernel, which lets dependents in at its top: scheduled
        // early, the merge starts the moment the partials are complete
        StepOverlap merge_behind_decode(true);
        RL_CUDA(rl::launch_step(rl::attn_combine_kernel, dim3(p->n_q, p->batch), dim3(256), 0, as_stream(stream), c));
    }
    RL_CUDA(cudaGetLastError());
    return RL_OK;
}

}  // namespace

// ======================================================================================
struct rl_cache {
    rl_cache_config cfg;
    std::vector<int> types;
    int n_attn = 0, n_delta = 0, conv_dim = 0;
    size_t pool_elems = 0;          // halves per (layer, K or V) pool
    __half* kv = nullptr;           // [n_attn][2][pool_elems]
    float* S = nullptr;             // [n_delta][n_slots][n_v][dk][dv]
    float* conv = nullptr;          // [n_delta][n_slots][conv_dim][conv_k] ring windows (gdn_decode.cu)
    int32_t* conv_phase = nullptr;  // [n_delta][n_slots] ring position of each slot's next token
    int* dev_err = nullptr;         // the device error word
    // scratch of the optional element-wise steps inside the step (rl_stack_glue)
    float *g_q = nullptr, *g_gate = nullptr;      // [max_batch][n_q][256]
    float *g_beta = nullptr, *g_g = nullptr;      // [max_batch][n_v]
    rl_stack_glue gglue = {};       // contents of the glue the captured graph was built with
    void* attn_ws = nullptr;
    size_t attn_ws_bytes = 0;
    size_t bytes = 0;
    // compact cache (kv_dtype == RL_KV_Q8K_TQ3V): record pools, the F16 window and the prefill scratch
    unsigned char* kvc = nullptr;   // [n_attn][cpool_bytes] q8-K / TQ3-V records of every page
    size_t cpool_bytes = 0;
    int win_pages = 0;              // window pages per slot
    size_t wpool_elems = 0;         // halves per (layer, K or V) window pool = n_slots * win_pages pages
    __half* kvw = nullptr;          // [n_attn][2][wpool_elems]
    int32_t* win_table = nullptr;   // [n_slots][win_pages]: slot s owns window pages s * win_pages ..
    int32_t* win_rows = nullptr;    // [max_batch][win_pages] rows of the sequences of the step in flight
    float* d_signs = nullptr;       // [256] or null
    __half* scratch = nullptr;      // [2][max_pages_per_seq pages] F16 pages a prefill chunk past the window reads
    int32_t* scratch_table = nullptr;   // [max_pages_per_seq] identity
    bool compact() const { return cfg.kv_dtype == RL_KV_Q8K_TQ3V; }
    // host-call staging
    bool staging = false;
    float *d_attn_q = nullptr, *d_attn_gate = nullptr, *d_attn_k = nullptr, *d_attn_v = nullptr,
          *d_attn_o = nullptr, *d_delta_qkv = nullptr, *d_delta_beta = nullptr, *d_delta_g = nullptr,
          *d_delta_o = nullptr, *d_conv_w = nullptr;
    int32_t *d_page_table = nullptr, *d_pos = nullptr, *d_slot_ids = nullptr;
    cudaStream_t s_h2d = nullptr, s_run = nullptr, s_d2h = nullptr;
    std::vector<cudaEvent_t> ev_in, ev_out;
    // optional per-kernel timing of the last step (rl_stack_set_timing)
    bool timing = false;
    std::vector<cudaEvent_t> tev;   // 4 per layer: boundaries between the layer's kernels
    int tev_used = 0;
    // graph replay of rl_stack_decode: the step's launches are captured once per distinct io
    // (same pointers, same batch) and replayed afterwards; positions, page table and slots are
    // read from device memory by the kernels, so the captured step stays valid as they advance
    bool overlap = true;            // dependent launch between the step's kernels
    bool graph_enabled = true;
    cudaGraphExec_t gexec = nullptr;
    rl_stack_io gkey;               // io of the captured graph / of the last eager step
    int gkey_seen = 0;              // 0 none, 1 ran eagerly once, 2 captured
    cudaStream_t s_cap = nullptr;
    // the same for rl_stack_decode_host: copies in, layers and copies out as one graph over the
    // three internal streams (needs pinned host buffers; pageable ones cannot be captured)
    cudaGraphExec_t hexec = nullptr;
    rl_stack_io hkey;
    int hkey_seen = 0;
    bool host_graph_failed = false;
    cudaEvent_t ev_fork = nullptr, ev_join_a = nullptr, ev_join_b = nullptr;
    // sharded step: where the gathered outputs go, the side stream the exchanges run on and the
    // events that fork it from / join it to the step's stream (rl_stack_set_gather)
    rl_stack_gather gather = {};
    cudaStream_t s_comm = nullptr;
    cudaEvent_t ev_xfork = nullptr, ev_xjoin = nullptr;
    rl_attn_decode_params attn_params(int batch) const {
        rl_attn_decode_params p;
        std::memset(&p, 0, sizeof p);
        p.n_q = cfg.n_q;
        p.n_kv = cfg.n_kv;
        p.head_dim = cfg.head_dim;
        p.kv_dtype = cfg.kv_dtype;
        p.batch = batch;
        p.page_tokens = cfg.page_tokens;
        p.n_pages = cfg.n_pages;
        p.max_pages_per_seq = cfg.max_pages_per_seq;
        p.max_seq_len = cfg.max_seq_len;
        p.len_add = 1;
        p.chunk_pages = 0;
        p.wht_len = cfg.wht_len;
        p.tq_signs = d_signs;
        return p;
    }
    // the same over the F16 window pools (rows from win_rows / win_table)
    rl_attn_decode_params window_params(int batch) const {
        rl_attn_decode_params p = attn_params(batch);
        p.kv_dtype = RL_KV_F16;
        p.n_pages = cfg.n_slots * win_pages;
        p.max_pages_per_seq = win_pages;
        p.max_seq_len = std::min(cfg.max_seq_len, win_pages * cfg.page_tokens);
        return p;
    }
};

namespace {

template <class T>
int dev_alloc(T** p, size_t n, size_t* total) {
    *p = nullptr;
    if (n == 0) return RL_OK;
    RL_CUDA(cudaMalloc(reinterpret_cast<void**>(p), n * sizeof(T)));
    *total += n * sizeof(T);
    return RL_OK;
}

// layers per synchronisation with the copy streams in rl_stack_decode_host
const int kHostGroup = std::max(1, knob("RL_B200_HOST_GROUP", 4));

int stack_decode_layers(rl_cache* c, const rl_stack_io* io, cudaStream_t run, bool host_mode) {
    // not with per-kernel timing: an event between two kernels is what the overlap removes
    StepOverlap overlap(c->overlap && !c->timing);
    rl::g_step_first = true;      // the step's first kernel waits for all earlier work in the stream (launch.cuh)
    const rl_cache_config& f = c->cfg;
    const int B = io->batch;
    const size_t q_sz = size_t(B) * f.n_q * f.head_dim, kv_sz = size_t(B) * f.n_kv * f.head_dim;
    const size_t qkv_sz = size_t(B) * c->conv_dim, hv_sz = size_t(B) * f.n_v, do_sz = size_t(B) * f.n_v * f.dv;
    const size_t st_elems = size_t(f.n_slots) * f.n_v * f.dk * f.dv;
    const size_t cv_elems = size_t(f.n_slots) * c->conv_dim * f.conv_k;
    int ai = 0, di = 0;
    const bool tm = c->timing && !c->tev.empty();
    auto mark = [&](int L, int i) {
        if (tm) cudaEventRecord(c->tev[size_t(L) * 4 + i], run);
    };
    // Sharded step: the outputs of the layers since the last exchange are all-gathered on the side
    // stream (one grouped NCCL call), beside the layers that follow; split-KV partials are merged
    // and gated there too, straight out of the gather buffer.
    const rl_stack_glue* glue = io->glue;
    const rl_stack_gather& gx = c->gather;
    // a sharded step leaves a few SMs to the exchange kernels, which otherwise find no room beside
    // persistent CTAs that fill every SM's shared memory and run only in the gaps between kernels
    SmReserve reserve(gx.comm ? gx.reserve_sms : 0);
    rl::Comm* comm = reinterpret_cast<rl::Comm*>(gx.comm);
    const int n_ranks = comm ? rl::comm_ranks(comm) : 1;
    const int per_x = gx.layers_per_exchange > 0 ? gx.layers_per_exchange : 4;
    int sent_a = 0, sent_d = 0;
    auto exchange = [&]() -> int {
        if (sent_a == ai && sent_d == di) return RL_OK;
        RL_CUDA(cudaEventRecord(c->ev_xfork, run));
        RL_CUDA(cudaStreamWaitEvent(c->s_comm, c->ev_xfork, 0));
        const size_t ml_sz = size_t(B) * f.n_q * 2;
        int bad = rl::comm_group_start();
        for (int a = sent_a; a < ai && !bad; ++a) {
            bad = rl::comm_all_gather_f32(comm, io->attn_o + a * q_sz, gx.attn_o_all + size_t(a) * n_ranks * q_sz, q_sz, c->s_comm);
            if (!bad && io->attn_ml)
                bad = rl::comm_all_gather_f32(comm, io->attn_ml + a * ml_sz, gx.attn_ml_all + size_t(a) * n_ranks * ml_sz, ml_sz,
                                              c->s_comm);
        }
        for (int d = sent_d; d < di && !bad; ++d)
            bad = rl::comm_all_gather_f32(comm, io->delta_o + d * do_sz, gx.delta_o_all + size_t(d) * n_ranks * do_sz, do_sz,
                                          c->s_comm);
        const int bad_end = rl::comm_group_end();
        if (bad || bad_end) return fail(RL_ERR_DEVICE, "exchange of the step's outputs: %s", rl::comm_last_error());
        if (io->attn_ml)
            for (int a = sent_a; a < ai; ++a)
                rl::lse_combine_kernel<<<unsigned(B * f.n_q), 256, 0, c->s_comm>>>(
                    gx.attn_o_all + size_t(a) * n_ranks * q_sz, gx.attn_ml_all + size_t(a) * n_ranks * ml_sz,
                    io->attn_gate ? io->attn_gate + a * q_sz : nullptr, gx.attn_o_final + a * q_sz, n_ranks, B * f.n_q, 0,
                    nullptr);
        sent_a = ai;
        sent_d = di;
        return RL_OK;
    };
    if (c->compact() && c->win_pages && c->n_attn) {
        if (host_mode) RL_CUDA(cudaStreamWaitEvent(run, c->ev_in[std::min(kHostGroup, f.n_layers) - 1], 0));
        RL_CUDA(rl::launch_step(rl::kv_slot_rows_kernel, dim3(B), dim3(128), 0, run, c->win_rows, io->slot_ids, c->win_pages,
                                f.n_slots, c->dev_err));
    }
    for (int L = 0; L < f.n_layers; ++L) {
        // host buffers: the layers synchronise with the copy streams once per group of layers, not per
        // layer (every wait costs the run stream a few microseconds and the dependent launch behind it)
        if (host_mode && L % kHostGroup == 0)
            RL_CUDA(cudaStreamWaitEvent(run, c->ev_in[std::min(L + kHostGroup, f.n_layers) - 1], 0));
        mark(L, 0);
        if (c->types[L] == RL_LAYER_FULL_ATTENTION) {
            rl_kv_append_params ap;
            ap.n_kv = f.n_kv;
            ap.head_dim = f.head_dim;
            ap.batch = B;
            ap.n_tok = 1;
            ap.page_tokens = f.page_tokens;
            ap.n_pages = f.n_pages;
            ap.max_pages_per_seq = f.max_pages_per_seq;
            ap.pos0 = 0;
            ap.rows_fp16 = 0;
            ap.wht_len = 0;
            ap.pos_limit = 0;
            ap.pos_limit = 0;
            void* kp = rl_cache_k_pool(c, ai);
            void* vp = rl_cache_v_pool(c, ai);
            const float* q_l = glue ? c->g_q : io->attn_q + ai * q_sz;
            const float* gate_l = glue ? (io->attn_ml ? nullptr : c->g_gate)
                                       : ((io->attn_gate && !io->attn_ml) ? io->attn_gate + ai * q_sz : nullptr);
            const float* k_new = glue ? glue->attn_k_raw + ai * kv_sz : io->attn_k + ai * kv_sz;
            if (glue) {
                rl_attn_qk_prepare_params qp;
                qp.n_q = f.n_q, qp.n_kv = f.n_kv, qp.head_dim = f.head_dim, qp.rotary_dim = glue->rotary_dim, qp.rows = B;
                qp.pos0 = 0, qp.theta = glue->theta, qp.eps = glue->rms_eps;
                if (int st = rl_attn_qk_prepare(glue->attn_qg + size_t(ai) * B * f.n_q * 2 * f.head_dim,
                                                glue->attn_k_raw + ai * kv_sz,
                                                glue->q_norm ? glue->q_norm + size_t(ai) * f.head_dim : nullptr,
                                                glue->k_norm ? glue->k_norm + size_t(ai) * f.head_dim : nullptr, io->pos,
                                                c->g_q, c->g_gate, &qp, run))
                    return st;
            }
            float* ml_l = io->attn_ml ? io->attn_ml + size_t(ai) * B * f.n_q * 2 : nullptr;
            cudaEvent_t after_main = tm ? c->tev[size_t(L) * 4 + 3] : nullptr;
            if (!c->compact()) {
                if (!io->no_append) {
                    // rows straight from the caller (no in-step kernel made them), pages of this layer only: the
                    // append need not wait for the kernel of the layer in front before it works
                    g_append_early = !glue;
                    const int st = rl_kv_append(kp, vp, io->page_table, io->pos, k_new, io->attn_v + ai * kv_sz, &ap, run);
                    g_append_early = false;
                    if (st) return st;
                }
                mark(L, 1);
                rl_attn_decode_params dp = c->attn_params(B);
                dp.len_add = io->no_append ? 0 : 1;
                g_decode_early = true;        // the caller's page table and lengths; only the append in front writes pages
                const int st = attn_decode_impl(kp, vp, io->page_table, io->pos, q_l, gate_l, io->attn_o + ai * q_sz, ml_l,
                                                c->attn_ws, c->attn_ws_bytes, &dp, run, after_main);
                g_decode_early = false;
                if (st) return st;
            } else {
                // every token persists in the compact pages; the F16 window rows of the sequences still
                // inside it are kept current whichever of the two this step reads
                void* kw = rl_cache_window_k_pool(c, ai);
                void* vw = rl_cache_window_v_pool(c, ai);
                if (!io->no_append) {
                    ap.wht_len = f.wht_len;
                    if (int st = rl_kv_compact_append(kp, io->page_table, io->pos, k_new, io->attn_v + ai * kv_sz, c->d_signs,
                                                      &ap, run))
                        return st;
                    if (c->win_pages) {
                        rl_kv_append_params wp = ap;
                        wp.n_pages = f.n_slots * c->win_pages;
                        wp.max_pages_per_seq = c->win_pages;
                        wp.pos_limit = f.window_tokens;
                        if (int st = rl_kv_append(kw, vw, c->win_rows, io->pos, k_new, io->attn_v + ai * kv_sz, &wp, run))
                            return st;
                    }
                }
                mark(L, 1);
                const bool over_window = io->kv_window_ok && c->win_pages;
                rl_attn_decode_params dp = over_window ? c->window_params(B) : c->attn_params(B);
                dp.len_add = io->no_append ? 0 : 1;
                if (int st = attn_decode_impl(over_window ? kw : kp, over_window ? vw : nullptr,
                                              over_window ? c->win_rows : io->page_table, io->pos, q_l, gate_l,
                                              io->attn_o + ai * q_sz, ml_l, c->attn_ws, c->attn_ws_bytes, &dp, run, after_main))
                    return st;
            }
            mark(L, 2);
            ++ai;
        } else {
            // conv window + SiLU + l2 norms + delta rule in one kernel
            mark(L, 1);
            rl_gdn_decode_params gp;
            gp.n_v = f.n_v;
            gp.n_qk = f.n_k;
            gp.dk = f.dk;
            gp.dv = f.dv;
            gp.conv_k = f.conv_k;
            gp.batch = B;
            gp.n_slots = f.n_slots;
            gp.head_map = f.head_map;
            gp.eps_l2 = 1e-6f;
            const float* beta_l = glue ? c->g_beta : io->delta_beta + di * hv_sz;
            const float* g_l = glue ? c->g_g : io->delta_g + di * hv_sz;
            if (glue)
                if (int st = rl_delta_gates(glue->delta_a + di * hv_sz, glue->delta_b + di * hv_sz,
                                            glue->A_log + size_t(di) * f.n_v, glue->dt_bias + size_t(di) * f.n_v, c->g_beta,
                                            c->g_g, B, f.n_v, run))
                    return st;
            // caller-made inputs, state and conv ring of this layer only: no kernel in front of it in the step touches
            // anything it does, so it need not wait before it works
            g_gdn_early = !glue;
            const int gst = rl_gdn_decode(c->S + di * st_elems, c->conv + di * cv_elems, c->conv_phase + size_t(di) * f.n_slots,
                                          io->slot_ids, io->delta_qkv + di * qkv_sz,
                                          io->conv_w + size_t(di) * c->conv_dim * f.conv_k, beta_l, g_l,
                                          io->delta_o + di * do_sz, &gp, run);
            g_gdn_early = false;
            if (gst) return gst;
            if (glue && glue->delta_z)
                if (int st = rl_gated_rmsnorm(io->delta_o + di * do_sz, glue->delta_z + di * do_sz,
                                              glue->gnorm ? glue->gnorm + size_t(di) * f.dv : nullptr, io->delta_o + di * do_sz, B,
                                              f.n_v, f.dv, glue->rms_eps, run))
                    return st;
            mark(L, 2);
            ++di;
        }
        if (host_mode && ((L + 1) % kHostGroup == 0 || L + 1 == f.n_layers)) RL_CUDA(cudaEventRecord(c->ev_out[L], run));
        // one layer before each multiple of the group size, so that the last call of the step, the only one whose
        // time the step waits for in full, carries the last layer alone (in qwen3_5's period of three DeltaNet layers
        // and an attention layer: one tensor instead of four)
        if (comm && ((L + 2) % per_x == 0 || L + 1 == f.n_layers))
            if (int st = exchange()) return st;
    }
    // every layer's window has taken this step's token: move the rings on
    if (c->n_delta)
        if (int st = rl_gdn_phase_advance(c->conv_phase, io->slot_ids, c->n_delta, f.n_slots, B, 1, run)) return st;
    if (comm) {
        // the step is complete on `run` only when every rank's outputs have arrived
        RL_CUDA(cudaEventRecord(c->ev_xjoin, c->s_comm));
        RL_CUDA(cudaStreamWaitEvent(run, c->ev_xjoin, 0));
    }
    return RL_OK;
}

}  // namespace

// ======================================================================================
extern "C" {

int rl_b200_abi_version(void) { return RL_B200_ABI_VERSION; }

int rl_b200_available(void) {
    int n = 0;
    if (cudaGetDeviceCount(&n) != cudaSuccess || n <= 0) {
        cudaGetLastError();
        return 0;
    }
    int dev = 0;
    cudaDeviceProp prop;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaGetDeviceProperties(&prop, dev) != cudaSuccess) return 0;
    return prop.major == 10 ? 1 : 0;
}

const char* rl_last_error(void) { return g_err; }

const char* rl_device_error_string(int code) {
    switch (code) {
        case rl::DEV_OK: return "ok";
        case rl::DEV_ERR_BAD_PAGE: return "page-table entry outside the pool";
        case rl::DEV_ERR_WAIT_TIMEOUT: return "a bounded barrier wait gave up";
        case rl::DEV_ERR_WORKSPACE: return "more split-KV chunks than the workspace holds";
        case rl::DEV_ERR_BAD_SLOT: return "state slot outside the cache";
        case rl::DEV_ERR_BAD_LEN: return "sequence length or position outside the page table";
        case rl::DEV_ERR_BAD_TREE: return "draft tree: parent, node count or leaf out of range";
        default: return "unknown device error";
    }
}

int rl_device_error(void* stream) {
    DevInfo* d;
    if (dev_info(&d)) return -1;
    int code = 0;
    if (cudaStreamSynchronize(as_stream(stream)) != cudaSuccess ||
        cudaMemcpy(&code, d->err_ptr, sizeof(int), cudaMemcpyDeviceToHost) != cudaSuccess) {
        fail(RL_ERR_DEVICE, "reading the device error word: %s", cudaGetErrorString(cudaGetLastError()));
        return -1;
    }
    if (code) cudaMemset(d->err_ptr, 0, sizeof(int));
    return code;
}

size_t rl_attn_decode_workspace_bytes(const rl_attn_decode_params* p) {
    if (attn_check(p)) return 0;
    DevInfo* d;
    int sms = 148;
    if (dev_info(&d) == RL_OK) sms = d->sms;
    return attn_plan(p, sms).total_bytes;
}

int rl_attn_decode(const void* k_pool, const void* v_pool, const int32_t* page_table,
                   const int32_t* seq_lens, const float* q, const float* gate, float* o, void* workspace,
                   size_t workspace_bytes, const rl_attn_decode_params* p, void* stream) {
    return attn_decode_impl(k_pool, v_pool, page_table, seq_lens, q, gate, o, nullptr, workspace,
                            workspace_bytes, p, stream);
}

int rl_attn_decode_partial(const void* k_pool, const void* v_pool, const int32_t* page_table,
                           const int32_t* seq_lens, const float* q, float* part_o, float* part_ml,
                           void* workspace, size_t workspace_bytes, const rl_attn_decode_params* p,
                           void* stream) {
    if (!part_ml) return fail(RL_ERR_RANGE, "part_ml is NULL");
    return attn_decode_impl(k_pool, v_pool, page_table, seq_lens, q, nullptr, part_o, part_ml, workspace,
                            workspace_bytes, p, stream);
}

// ---- rl_attn_decode without any allocation: scratch in the library's device image -------------
namespace {
constexpr size_t kStaticScratchBytes = size_t(4) << 20;
// Split-KV partials of rl_attn_decode_noalloc.  One copy per GPU that loads this library.
static __device__ __align__(256) unsigned char g_attn_scratch[kStaticScratchBytes];
struct StaticScratch {
    bool ready = false;
    void* ptr = nullptr;
};
StaticScratch g_static_scratch[64];

// The array's name is only a host-side handle: the kernels need its device address, looked
// up once per device with that device current.
int static_scratch(void** out) {
    int dev = 0;
    RL_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return fail(RL_ERR_RANGE, "device ordinal %d out of range", dev);
    std::lock_guard<std::mutex> lk(g_mu);
    StaticScratch& sc = g_static_scratch[dev];
    if (!sc.ready) {
        void* ptr = nullptr;
        RL_CUDA(cudaGetSymbolAddress(&ptr, g_attn_scratch));
        if (!ptr) return fail(RL_ERR_DEVICE, "cudaGetSymbolAddress returned a null address for the scratch array");
        sc.ptr = ptr;
        sc.ready = true;
    }
    *out = sc.ptr;
    return RL_OK;
}
}  // namespace

int rl_attn_decode_noalloc(const void* k_pool, const void* v_pool, const int32_t* page_table,
                           const int32_t* seq_lens, const float* q, const float* gate, float* o,
                           const rl_attn_decode_params* p, void* stream) {
    if (int st = attn_check(p)) return st;
    DevInfo* d;
    if (int st = dev_info(&d)) return st;
    const size_t need = attn_plan(p, d->sms).total_bytes;
    if (need > kStaticScratchBytes)
        return fail(RL_ERR_RANGE,
                    "rl_attn_decode_noalloc: batch %d x %d KV heads needs %zu bytes of split-KV scratch, the "
                    "built-in array holds %zu; use rl_attn_decode with a caller workspace",
                    p->batch, p->n_kv, need, kStaticScratchBytes);
    void* scratch = nullptr;
    if (int st = static_scratch(&scratch)) return st;
    return attn_decode_impl(k_pool, v_pool, page_table, seq_lens, q, gate, o, nullptr, scratch, kStaticScratchBytes,
                            p, stream);
}

int rl_lse_combine(const float* part_o, const float* part_ml, const float* gate, float* o, int n_parts,
                   int rows, int head_dim, int wht_len, const float* tq_signs, void* stream) {
    if (head_dim != rl::kHeadDim) return fail(RL_ERR_UNSUPPORTED, "head_dim %d: only 256", head_dim);
    if (wht_len != 0 && wht_len != 128 && wht_len != 256)
        return fail(RL_ERR_UNSUPPORTED, "wht_len %d: only 0, 128 or 256", wht_len);
    if (n_parts <= 0 || rows < 0) return fail(RL_ERR_RANGE, "n_parts %d rows %d", n_parts, rows);
    if (rows == 0) return RL_OK;
    if (!part_o || !part_ml || !o) return fail(RL_ERR_RANGE, "NULL pointer argument");
    rl::lse_combine_kernel<<<rows, 256, 0, as_stream(stream)>>>(part_o, part_ml, gate, o, n_parts, rows, wht_len,
                                                                wht_len == 256 ? tq_signs : nullptr);
    RL_CUDA(cudaGetLastError());
    return RL_OK;
}

int rl_kv_append(void* k_pool, void* v_pool, const int32_t* page_table, const int32_t* pos,
                 const void* k_rows, const void* v_rows, const rl_kv_append_params* p, void* stream) {
    if (!p) return fail(RL_ERR_RANGE, "params is NULL");
    if (p->head_dim != rl::kHeadDim || p->page_tokens != rl::kPageTokens)
        return fail(RL_ERR_UNSUPPORTED, "head_dim %d / page_tokens %d: only 256 / 64", p->head_dim, p->page_tokens);
    if (p->batch < 0 || p->n_tok < 0 || p->n_kv <= 0 || p->n_kv > 65535 || p->batch > 65535)
        return fail(RL_ERR_RANGE, "batch %d n_tok %d n_kv %d", p->batch, p->n_tok, p->n_kv);
    if (p->batch == 0 || p->n_tok == 0) return RL_OK;
    if (!k_pool || !v_pool || !page_table || !k_rows || !v_rows) return fail(RL_ERR_RANGE, "NULL pointer argument");
    DevInfo* d;
    if (int st = dev_info(&d)) return st;
    rl::KvWriteArgs a;
    a.k_pool = static_cast<__half*>(k_pool);
    a.v_pool = static_cast<__half*>(v_pool);
    a.page_table = page_table;
    a.pos = pos;
    a.k_rows = k_rows;
    a.v_rows = v_rows;
    a.err = d->err_ptr;
    a.batch = p->batch;
    a.n_tok = p->n_tok;
    a.n_kv = p->n_kv;
    a.n_pages = p->n_pages;
    a.max_pages_per_seq = p->max_pages_per_seq;
    a.pos0 = p->pos0;
    a.rows_fp16 = p->rows_fp16;
    a.pos_limit = p->pos_limit;
    a.early = g_append_early && rl::g_step_overlap && !rl::g_step_first ? 1 : 0;
    const int rows_per_block = p->n_tok >= 8 ? 8 : 1;
    RL_CUDA(rl::launch_step(rl::kv_write_kernel, dim3((p->n_tok + rows_per_block - 1) / rows_per_block, p->n_kv, p->batch),
                            dim3(32, rows_per_block), 0, as_stream(stream), a));
    RL_CUDA(cudaGetLastError());
    return RL_OK;
}

// How the (query tile, head) items of a prefill call are divided among CTAs.
//  * fewer items than SMs (short chunks, verify rows): every item's KV range is shared by `parts`
//    CTAs, enough to fill the device twice over, each part keeping at least 8 KV tiles;
//  * a last wave that is at most half full (192 items of a 1 024-row chunk on 148 SMs): the first
//    n_full items run whole, the items of the last wave are divided among tail_parts CTAs each, so
//    that its work is spread over every SM (dividing EVERY item of such a chunk in two measured
//    slower than not dividing: the partials and second prologues cost more than the wave);
//  * otherwise nothing is divided.
static bool prefill_packed(const rl_attn_prefill_params* p) {
    // few enough rows that (token, query head of a group) pairs fit one 128-row tile per KV head
    return p->seq * (p->n_q / p->n_kv) <= rl::attn_prefill_q_rows();
}

struct PrefillSplit {
    int parts = 1;                   // uniform division of every item
    int n_full = 0, tail_parts = 1;  // or: items from n_full on divided in tail_parts
    long long items = 0;
    size_t ws_bytes(const rl_attn_prefill_params* p) const {
        if (tail_parts > 1) {
            const size_t units = size_t(items - n_full) * tail_parts, rows = rl::attn_prefill_q_rows();
            return align_up(units * rows * rl::kHeadDim * sizeof(float), 256) + units * rows * 2 * sizeof(float);
        }
        if (parts <= 1) return 0;
        const size_t rows_total = size_t(p->seq) * p->n_q;
        return align_up(size_t(parts) * rows_total * rl::kHeadDim * sizeof(float), 256) +
               size_t(parts) * rows_total * 2 * sizeof(float);
    }
};

static PrefillSplit prefill_split(const rl_attn_prefill_params* p, int sms) {
    PrefillSplit sp;
    const int rows = rl::attn_prefill_q_rows();
    const int n_qtiles = (p->seq + rows - 1) / rows;
    sp.items = prefill_packed(p) ? p->n_kv : 1LL * n_qtiles * p->n_q;
    if (sp.items <= 0) return sp;
    if (sp.items < sms) {
        const long long tiles = (1LL * p->pos0 + p->seq + p->page_tokens - 1) / p->page_tokens;   // of the last query tile
        long long parts = prefill_packed(p) ? sms / sp.items : (2LL * sms + sp.items - 1) / sp.items;
        parts = std::min(parts, std::max(1LL, tiles / 8));
        sp.parts = int(std::min(parts, 64LL));
        return sp;
    }
    const long long rest = sp.items % sms;
    if (rest == 0 || 2 * rest > sms) return sp;
    // the items of the last wave are the last of the launch order: the lowest query tiles of the
    // last KV head; the shortest of them attends to this many KV tiles
    const long long tiles_min = (1LL * p->pos0 + std::min<long long>(p->seq, rows) + p->page_tokens - 1) / p->page_tokens;
    const long long tp = std::min({1LL * sms / rest, 8LL, tiles_min / 8});
    if (tp > 1) {
        sp.n_full = int(sp.items - rest);
        sp.tail_parts = int(tp);
    }
    return sp;
}

static int attn_prefill_impl(void* k_pool, void* v_pool, const int32_t* page_table_row, const void* q_bf16,
                             const void* k_rows_bf16, const void* v_rows_bf16, const float* gate, float* o,
                             void* workspace, size_t workspace_bytes, const rl_attn_prefill_params* p, void* stream) {
    if (!p) return fail(RL_ERR_RANGE, "params is NULL");
    if (p->head_dim != rl::kHeadDim || p->page_tokens != rl::kPageTokens)
        return fail(RL_ERR_UNSUPPORTED, "head_dim %d / page_tokens %d: only 256 / 64", p->head_dim, p->page_tokens);
    if (p->n_kv <= 0 || p->n_q <= 0 || p->n_q % p->n_kv != 0 || p->n_q > 65535)
        return fail(RL_ERR_UNSUPPORTED, "n_q %d / n_kv %d", p->n_q, p->n_kv);
    if (p->seq < 0 || p->pos0 < 0 || p->n_pages <= 0) return fail(RL_ERR_RANGE, "seq %d pos0 %d n_pages %d", p->seq, p->pos0, p->n_pages);
    if ((long long)p->pos0 + p->seq > (long long)p->n_table * p->page_tokens)
        return fail(RL_ERR_RANGE, "pos0 %d + seq %d exceeds the %d pages of the table row", p->pos0, p->seq, p->n_table);
    if (p->seq == 0) return RL_OK;
    if (!k_pool || !v_pool || !page_table_row || !q_bf16 || !o) return fail(RL_ERR_RANGE, "NULL pointer argument");
    if ((k_rows_bf16 == nullptr) != (v_rows_bf16 == nullptr)) return fail(RL_ERR_RANGE, "k_rows and v_rows go together");
    if (reinterpret_cast<uintptr_t>(k_pool) % 128 || reinterpret_cast<uintptr_t>(v_pool) % 128 ||
        reinterpret_cast<uintptr_t>(q_bf16) % 16 || reinterpret_cast<uintptr_t>(o) % 16 ||
        reinterpret_cast<uintptr_t>(gate) % 16)
        return fail(RL_ERR_RANGE, "pools must be 128-byte aligned, q, gate and o 16-byte aligned");
    DevInfo* d;
    if (int st = dev_info(&d)) return st;
    if (k_rows_bf16) {
        rl_kv_append_params ap;
        ap.n_kv = p->n_kv;
        ap.head_dim = p->head_dim;
        ap.batch = 1;
        ap.n_tok = p->seq;
        ap.page_tokens = p->page_tokens;
        ap.n_pages = p->n_pages;
        ap.max_pages_per_seq = p->n_table;
        ap.pos0 = p->pos0;
        ap.rows_fp16 = 2;
        ap.wht_len = 0;
            ap.pos_limit = 0;
        if (int st = rl_kv_append(k_pool, v_pool, page_table_row, nullptr, k_rows_bf16, v_rows_bf16, &ap, stream))
            return st;
    }
    rl::AttnPrefillArgs a;
    a.k_pool = static_cast<const __half*>(k_pool);
    a.v_pool = static_cast<const __half*>(v_pool);
    a.page_table = page_table_row;
    a.q = static_cast<const __nv_bfloat16*>(q_bf16);
    a.gate = gate;
    a.o = o;
    a.err = d->err_ptr;
    a.T = p->seq;
    a.pos0 = p->pos0;
    a.n_q = p->n_q;
    a.n_kv = p->n_kv;
    a.n_pages = p->n_pages;
    a.scale = 1.f / sqrtf(float(p->head_dim));
    const int n_qtiles = (p->seq + rl::attn_prefill_q_rows() - 1) / rl::attn_prefill_q_rows();
    // a workspace lets short chunks (or a handful of verify rows over a long cache) spread every
    // (query tile, head) over several CTAs; without one the call runs unsplit
    PrefillSplit sp = workspace ? prefill_split(p, d->sms) : PrefillSplit();
    if (workspace_bytes < sp.ws_bytes(p) || reinterpret_cast<uintptr_t>(workspace) % 16) sp = PrefillSplit();
    const int parts = sp.parts;
    const size_t rows_total = size_t(p->seq) * p->n_q;
    const size_t units = sp.tail_parts > 1 ? size_t(sp.items - sp.n_full) * sp.tail_parts : 0;
    const size_t o_bytes = sp.tail_parts > 1
                               ? align_up(units * rl::attn_prefill_q_rows() * rl::kHeadDim * sizeof(float), 256)
                               : align_up(size_t(parts) * rows_total * rl::kHeadDim * sizeof(float), 256);
    const bool divided = parts > 1 || sp.tail_parts > 1;
    a.packed = prefill_packed(p) ? 1 : 0;
    a.kv_parts = parts;
    a.n_full = sp.tail_parts > 1 ? sp.n_full : 0;
    a.tail_parts = sp.tail_parts;
    a.by_size = sp.items < 2LL * d->sms ? 1 : 0;
    a.wave = d->sms;
    a.part_o = divided ? static_cast<float*>(workspace) : nullptr;
    a.part_ml = divided ? reinterpret_cast<float*>(static_cast<char*>(workspace) + o_bytes) : nullptr;
    const unsigned n_items = a.packed ? unsigned(p->n_kv) : unsigned(n_qtiles) * unsigned(p->n_q);
    {
        // both kernels wait for the kernel before them (griddepcontrol.wait) ahead of their first global access
        StepOverlap overlap(true);
        RL_CUDA(rl::launch_step(rl::attn_prefill_kernel,
                                dim3(sp.tail_parts > 1 ? unsigned(sp.n_full) + unsigned(units) : n_items * unsigned(parts)),
                                dim3(unsigned(rl::attn_prefill_threads())), rl::attn_prefill_smem_bytes(), as_stream(stream), a));
        if (sp.tail_parts > 1 && parts <= 1)
            RL_CUDA(rl::launch_step(rl::attn_prefill_tail_merge_kernel,
                                    dim3(unsigned(rl::attn_prefill_q_rows() / 8), unsigned(sp.items - sp.n_full)),
                                    dim3(256), 0, as_stream(stream), a));   // 8 rows per block, a warp each
    }
    if (parts > 1)
        rl::lse_combine_kernel<<<unsigned(rows_total), 256, 0, as_stream(stream)>>>(a.part_o, a.part_ml, gate, o, parts,
                                                                                  int(rows_total), 0, nullptr);

    RL_CUDA(cudaGetLastError());
    return RL_OK;
}

int rl_attn_prefill(void* k_pool, void* v_pool, const int32_t* page_table_row, const void* q_bf16,
                    const void* k_rows_bf16, const void* v_rows_bf16, const float* gate, float* o,
                    const rl_attn_prefill_params* p, void* stream) {
    return attn_prefill_impl(k_pool, v_pool, page_table_row, q_bf16, k_rows_bf16, v_rows_bf16, gate, o, nullptr, 0, p,
                             stream);
}

size_t rl_attn_prefill_workspace_bytes(const rl_attn_prefill_params* p) {
    if (!p || p->seq <= 0 || p->n_q <= 0 || p->page_tokens <= 0) return 0;
    DevInfo* d;
    if (dev_info(&d)) return 0;
    return prefill_split(p, d->sms).ws_bytes(p);
}

int rl_attn_prefill_ws(void* k_pool, void* v_pool, const int32_t* page_table_row, const void* q_bf16,
                       const void* k_rows_bf16, const void* v_rows_bf16, const float* gate, float* o, void* workspace,
                       size_t workspace_bytes, const rl_attn_prefill_params* p, void* stream) {
    return attn_prefill_impl(k_pool, v_pool, page_table_row, q_bf16, k_rows_bf16, v_rows_bf16, gate, o, workspace,
                             workspace_bytes, p, stream);
}


int rl_kv_gather(const void* pool, const int32_t* page_table_row, void* out_f16, int n_tok, int n_kv,
                 int head_dim, int n_pages, void* stream) {
    if (head_dim != rl::kHeadDim) return fail(RL_ERR_UNSUPPORTED, "head_dim %d: only 256", head_dim);
    if (n_tok < 0 || n_kv <= 0 || n_kv > 65535) return fail(RL_ERR_RANGE, "n_tok %d n_kv %d", n_tok, n_kv);
    if (n_tok == 0) return RL_OK;
    if (!pool || !page_table_row || !out_f16) return fail(RL_ERR_RANGE, "NULL pointer argument");
    DevInfo* d;
    if (int st = dev_info(&d)) return st;
    rl::kv_gather_kernel<<<dim3(n_tok, n_kv), 32, 0, as_stream(stream)>>>(
        static_cast<const __half*>(pool), page_table_row, static_cast<__half*>(out_f16), n_tok, n_kv, n_pages,
        d->err_ptr);
    RL_CUDA(cudaGetLastError());
    return RL_OK;
}

size_t rl_kv_compact_page_bytes(void) { return 2 * size_t(rl::kCompactRecordBytes); }

int rl_kv_compact_append(void* pool, const int32_t* page_table, const int32_t* pos, const void* k_rows,
                         const void* v_rows, const float* tq_signs, const rl_kv_append_params* p,
                         void* stream) {
    if (!p) return fail(RL_ERR_RANGE, "params is NULL");
    if (p->head_dim != rl::kHeadDim || p->page_tokens != rl::kPageTokens)
        return fail(RL_ERR_UNSUPPORTED, "head_dim %d / page_tokens %d: only 256 / 64", p->head_dim, p->page_tokens);
    if (p->wht_len != 128 && p->wht_len != 256) return fail(RL_ERR_UNSUPPORTED, "wht_len %d: only 128 or 256", p->wht_len);
    if (p->rows_fp16 != 0 && p->rows_fp16 != 2) return fail(RL_ERR_UNSUPPORTED, "the compact cache quantises fp32 or bf16 rows");
    if (p->batch < 0 || p->n_tok < 0 || p->n_kv <= 0 || p->n_kv > 65535 || p->batch > 65535)
        return fail(RL_ERR_RANGE, "batch %d n_tok %d n_kv %d", p->batch, p->n_tok, p->n_kv);
    if (p->batch == 0 || p->n_tok == 0) return RL_OK;
    if (!pool || !page_table || !k_rows || !v_rows) return fail(RL_ERR_RANGE, "NULL pointer argument");
    if (reinterpret_cast<uintptr_t>(pool) % 16) return fail(RL_ERR_RANGE, "pool must be 16-byte aligned");
    DevInfo* d;
    if (int st = dev_info(&d)) return st;
    rl::KvCompactWriteArgs a;
    a.pool = static_cast<unsigned char*>(pool);
    a.page_table = page_table;
    a.pos = pos;
    a.k_rows = k_rows;
    a.v_rows = v_rows;
    a.signs = tq_signs;
    a.err = d->err_ptr;
    a.batch = p->batch;
    a.n_tok = p->n_tok;
    a.n_kv = p->n_kv;
    a.n_pages = p->n_pages;
    a.max_pages_per_seq = p->max_pages_per_seq;
    a.pos0 = p->pos0;
    a.wht_len = p->wht_len;
    a.rows_bf16 = p->rows_fp16 == 2;
    rl::kv_compact_write_kernel<<<dim3(p->n_tok, p->n_kv, p->batch), 256, 0, as_stream(stream)>>>(a);
    RL_CUDA(cudaGetLastError());
    return RL_OK;
}

int rl_kv_compact_gather(const void* pool, const int32_t* page_table_row, void* k_q, void* k_sc, void* v_codes,
                         void* v_sc, int n_tok, int n_kv, int n_pages, int wht_len, void* stream) {
    if (wht_len != 128 && wht_len != 256) return fail(RL_ERR_UNSUPPORTED, "wht_len %d: only 128 or 256", wht_len);
    if (n_tok < 0 || n_kv <= 0 || n_kv > 65535) return fail(RL_ERR_RANGE, "n_tok %d n_kv %d", n_tok, n_kv);
    if (n_tok == 0) return RL_OK;
    if (!pool || !page_table_row || !k_q || !k_sc || !v_codes || !v_sc) return fail(RL_ERR_RANGE, "NULL pointer argument");
    DevInfo* d;
    if (int st = dev_info(&d)) return st;
    rl::kv_compact_gather_kernel<<<dim3(n_tok, n_kv), 256, 0, as_stream(stream)>>>(
        static_cast<const unsigned char*>(pool), page_table_row, static_cast<signed char*>(k_q),
        static_cast<__half*>(k_sc), static_cast<unsigned char*>(v_codes), static_cast<__half*>(v_sc), n_tok, n_kv,
        n_pages, wht_len, d->err_ptr);
    RL_CUDA(cudaGetLastError());
    return RL_OK;
}

int rl_kv_compact_to_f16(const void* pool, const int32_t* src_table_row, int src_pos0, int n_src_pages, void* k_pool,
                         void* v_pool, const int32_t* dst_table_row, int dst_pos0, int n_dst_pages, int n_tok,
                         int n_kv, int wht_len, const float* tq_signs, void* stream) {
    if (wht_len != 128 && wht_len != 256) return fail(RL_ERR_UNSUPPORTED, "wht_len %d: only 128 or 256", wht_len);
    if (n_tok < 0 || n_kv <= 0 || n_kv > 65535 || src_pos0 < 0 || dst_pos0 < 0 || n_src_pages <= 0 || n_dst_pages <= 0)
        return fail(RL_ERR_RANGE, "n_tok %d n_kv %d src_pos0 %d dst_pos0 %d", n_tok, n_kv, src_pos0, dst_pos0);
    if (n_tok == 0) return RL_OK;
    if (!pool || !src_table_row || !k_pool || !v_pool || !dst_table_row) return fail(RL_ERR_RANGE, "NULL pointer argument");
    DevInfo* d;
    if (int st = dev_info(&d)) return st;
    rl::kv_compact_to_f16_kernel<<<dim3(n_tok, n_kv), 256, 0, as_stream(stream)>>>(
        static_cast<const unsigned char*>(pool), src_table_row, src_pos0, n_src_pages, static_cast<__half*>(k_pool),
        static_cast<__half*>(v_pool), dst_table_row, dst_pos0, n_dst_pages, n_kv, wht_len, tq_signs, d->err_ptr);
    RL_CUDA(cudaGetLastError());
    return RL_OK;
}

// shared by the one-token and the several-token entry points; n_tok scales the dense strides
static int delta_decode_args(rl::DeltaDecodeArgs* out, float* S, const int32_t* slot_ids, const float* q,
                             const float* k, const float* v, const float* beta, const float* g_log, float* o,
                             const rl_delta_recurrent_params* p, int n_tok, DevInfo** dev) {
    if (!p) return fail(RL_ERR_RANGE, "params is NULL");
    if (p->dk != 128 || p->dv != 128) return fail(RL_ERR_UNSUPPORTED, "dk %d dv %d: only 128 x 128", p->dk, p->dv);
    if (p->n_v <= 0 || p->n_v > 65535 || p->batch < 0 || p->batch > 65535 || p->n_slots <= 0)
        return fail(RL_ERR_RANGE, "n_v %d batch %d n_slots %d", p->n_v, p->batch, p->n_slots);
    if (p->head_map == RL_HEADS_PER_VALUE ? p->n_qk != p->n_v
                                          : (p->n_qk <= 0 || p->n_v % p->n_qk != 0 || p->head_map > RL_HEADS_TILED))
        return fail(RL_ERR_RANGE, "n_qk %d does not fit n_v %d with head_map %d", p->n_qk, p->n_v, p->head_map);
    if (p->batch == 0) return RL_OK;
    if (!S || !q || !k || !v || !beta || !g_log || !o) return fail(RL_ERR_RANGE, "NULL pointer argument");
    if (int st = dev_info(dev)) return st;
    rl::DeltaDecodeArgs& a = *out;
    a.S = S;
    a.slot_ids = slot_ids;
    a.q = q;
    a.k = k;
    a.v = v;
    a.beta = beta;
    a.g_log = g_log;
    a.o = o;
    a.err = (*dev)->err_ptr;
    a.batch = p->batch;
    a.n_v = p->n_v;
    a.n_qk = p->n_qk;
    a.n_slots = p->n_slots;
    a.head_map = p->head_map;
    a.eps_l2 = p->eps_l2;
    a.q_stride = p->q_stride ? p->q_stride : 1LL * n_tok * p->n_qk * p->dk;
    a.k_stride = p->k_stride ? p->k_stride : 1LL * n_tok * p->n_qk * p->dk;
    a.v_stride = p->v_stride ? p->v_stride : 1LL * n_tok * p->n_v * p->dv;
    if ((a.q_stride | a.k_stride | a.v_stride) % 4 || reinterpret_cast<uintptr_t>(q) % 16 ||
        reinterpret_cast<uintptr_t>(k) % 16 || reinterpret_cast<uintptr_t>(v) % 16 ||
        reinterpret_cast<uintptr_t>(S) % 16)
        return fail(RL_ERR_RANGE, "S, q, k, v must be 16-byte aligned with strides a multiple of 4 floats");
    return RL_OK;
}

int rl_delta_recurrent(float* S, const int32_t* slot_ids, const float* q, const float* k, const float* v,
                       const float* beta, const float* g_log, float* o, const rl_delta_recurrent_params* p,
                       void* stream) {
    rl::DeltaDecodeArgs a;
    DevInfo* d = nullptr;
    if (int st = delta_decode_args(&a, S, slot_ids, q, k, v, beta, g_log, o, p, 1, &d)) return st;
    if (p->batch == 0) return RL_OK;
    rl::launch_delta_decode(a, d->sms, as_stream(stream));
    RL_CUDA(cudaGetLastError());
    return RL_OK;
}

int rl_delta_recurrent_multi(float* S, float* S_backup, const int32_t* slot_ids, const float* q, const float* k,
                             const float* v, const float* beta, const float* g_log, float* o,
                             const rl_delta_recurrent_params* p, int n_tok, long long qk_tok_stride,
                             long long v_tok_stride, void* stream) {
    if (n_tok < 0 || n_tok > 64) return fail(RL_ERR_RANGE, "n_tok %d outside [0, 64]", n_tok);
    if (n_tok == 0) return RL_OK;
    rl::DeltaDecodeArgs a;
    DevInfo* d = nullptr;
    if (int st = delta_decode_args(&a, S, slot_ids, q, k, v, beta, g_log, o, p, n_tok, &d)) return st;
    if (p->batch == 0) return RL_OK;
    const long long qk_t = qk_tok_stride ? qk_tok_stride : 1LL * p->n_qk * p->dk;
    const long long v_t = v_tok_stride ? v_tok_stride : 1LL * p->n_v * p->dv;
    if ((qk_t | v_t) % 4 || reinterpret_cast<uintptr_t>(S_backup) % 16)
        return fail(RL_ERR_RANGE, "token strides must be a multiple of 4 floats, S_backup 16-byte aligned");
    if (S_backup == S) return fail(RL_ERR_RANGE, "S_backup must not alias S");
    rl::launch_delta_decode_multi(a, S_backup, n_tok, qk_t, v_t, as_stream(stream));
    RL_CUDA(cudaGetLastError());
    return RL_OK;
}

static int delta_chunk_check(const rl_delta_chunk_params* p) {
    if (!p) return fail(RL_ERR_RANGE, "params is NULL");
    if (p->dk != 128 || p->dv != 128 || p->chunk != 64)
        return fail(RL_ERR_UNSUPPORTED, "dk %d dv %d chunk %d: only 128 x 128, chunk 64", p->dk, p->dv, p->chunk);
    if (p->n_v <= 0 || p->n_v > 65535 || p->seq < 0) return fail(RL_ERR_RANGE, "n_v %d seq %d", p->n_v, p->seq);
    if (p->head_map == RL_HEADS_PER_VALUE ? p->n_qk != p->n_v
                                          : (p->n_qk <= 0 || p->n_v % p->n_qk != 0 || p->head_map > RL_HEADS_TILED))
        return fail(RL_ERR_RANGE, "n_qk %d does not fit n_v %d with head_map %d", p->n_qk, p->n_v, p->head_map);
    return RL_OK;
}

int rl_attn_qk_prepare(const float* qg, float* k, const float* q_norm, const float* k_norm, const int32_t* pos,
                       float* q_out, float* gate_out, const rl_attn_qk_prepare_params* p, void* stream) {
    if (!p) return fail(RL_ERR_RANGE, "params is NULL");
    if (p->head_dim != rl::kHeadDim) return fail(RL_ERR_UNSUPPORTED, "head_dim %d: only 256", p->head_dim);
    if (p->n_q <= 0 || p->n_kv <= 0 || p->n_q + p->n_kv > 65535 || p->rows < 0 || p->rows > 65535)
        return fail(RL_ERR_RANGE, "n_q %d n_kv %d rows %d", p->n_q, p->n_kv, p->rows);
    if (p->rotary_dim < 0 || p->rotary_dim > p->head_dim || (p->rotary_dim & 1))
        return fail(RL_ERR_RANGE, "rotary_dim %d must be even and at most head_dim", p->rotary_dim);
    if (p->rotary_dim > 0 && !(p->theta > 0.f)) return fail(RL_ERR_RANGE, "theta must be positive");
    if (p->rows == 0) return RL_OK;
    if (!qg || !k || !q_out || !gate_out) return fail(RL_ERR_RANGE, "NULL pointer argument");
    DevInfo* d;
    if (int st = dev_info(&d)) return st;
    rl::AttnQkPrepareArgs a;
    a.qg = qg;
    a.k = k;
    a.q_norm = q_norm;
    a.k_norm = k_norm;
    a.pos = pos;
    a.q_out = q_out;
    a.gate_out = gate_out;
    a.n_q = p->n_q;
    a.n_kv = p->n_kv;
    a.rotary_dim = p->rotary_dim;
    a.pos0 = p->pos0;
    a.eps = p->eps;
    const int pairs = p->rotary_dim / 2;
    for (int i = 0; i < pairs; ++i) a.inv_freq[i] = 1.f / powf(p->theta, float(i) / float(pairs));
    rl::attn_qk_prepare_kernel<<<dim3(p->n_q + p->n_kv, p->rows), rl::kHeadDim, 0, as_stream(stream)>>>(a);
    RL_CUDA(cudaGetLastError());
    return RL_OK;
}

int rl_rmsnorm(const float* x, const float* gamma, float* y, int rows, int n, float eps, void* stream) {
    if (rows < 0 || n <= 0) return fail(RL_ERR_RANGE, "rows %d n %d", rows, n);
    if (rows == 0) return RL_OK;
    if (!x || !y) return fail(RL_ERR_RANGE, "NULL pointer argument");
    DevInfo* d;
    if (int st = dev_info(&d)) return st;
    rl::rmsnorm_kernel<<<rows, 256, 0, as_stream(stream)>>>(x, gamma, y, n, eps);
    RL_CUDA(cudaGetLastError());
    return RL_OK;
}

int rl_gated_rmsnorm(const float* x, const float* z, const float* gamma, float* y, int rows, int n_heads,
                     int head_dim, float eps, void* stream) {
    if (head_dim != 128) return fail(RL_ERR_UNSUPPORTED, "head_dim %d: only 128", head_dim);
    if (rows < 0 || rows > 65535 || n_heads <= 0 || n_heads > 65535) return fail(RL_ERR_RANGE, "rows %d n_heads %d", rows, n_heads);
    if (rows == 0) return RL_OK;
    if (!x || !z || !y) return fail(RL_ERR_RANGE, "NULL pointer argument");
    DevInfo* d;
    if (int st = dev_info(&d)) return st;
    rl::GatedRmsnormArgs a;
    a.x = x;
    a.z = z;
    a.gamma = gamma;
    a.y = y;
    a.n_heads = n_heads;
    a.head_dim = head_dim;
    a.eps = eps;
    rl::gated_rmsnorm_kernel<<<dim3(n_heads, rows), head_dim, 0, as_stream(stream)>>>(a);
    RL_CUDA(cudaGetLastError());
    return RL_OK;
}

int rl_cast_f32_to_bf16(const float* x, void* y_bf16, size_t n, void* stream) {
    if (n == 0) return RL_OK;
    if (!x || !y_bf16) return fail(RL_ERR_RANGE, "NULL pointer argument");
    if (reinterpret_cast<uintptr_t>(x) % 16 || reinterpret_cast<uintptr_t>(y_bf16) % 8)
        return fail(RL_ERR_RANGE, "x must be 16-byte and y 8-byte aligned");
    const size_t blocks = (n + 1023) / 1024;
    if (blocks > 0x7fffffffull) return fail(RL_ERR_RANGE, "n too large");
    rl::cast_f32_bf16_kernel<<<unsigned(blocks), 256, 0, as_stream(stream)>>>(x, static_cast<__nv_bfloat16*>(y_bf16), n);
    RL_CUDA(cudaGetLastError());
    return RL_OK;
}

int rl_delta_gates(const float* a, const float* b, const float* A_log, const float* dt_bias, float* beta,
                   float* g_log, int rows, int n_v, void* stream) {
    if (rows < 0 || n_v <= 0 || 1LL * rows * n_v > (1LL << 30)) return fail(RL_ERR_RANGE, "rows %d n_v %d", rows, n_v);
    if (rows == 0) return RL_OK;
    if (!a || !b || !A_log || !dt_bias || !beta || !g_log) return fail(RL_ERR_RANGE, "NULL pointer argument");
    DevInfo* d;
    if (int st = dev_info(&d)) return st;
    const int n = rows * n_v;
    rl::delta_gates_kernel<<<(n + 255) / 256, 256, 0, as_stream(stream)>>>(a, b, A_log, dt_bias, beta, g_log, n_v, rows);
    RL_CUDA(cudaGetLastError());
    return RL_OK;
}

size_t rl_delta_chunk_workspace_bytes(const rl_delta_chunk_params* p) {
    if (delta_chunk_check(p)) return 0;
    const size_t n_chunks = (size_t(p->seq) + 63) / 64;
    return align_up(n_chunks * p->n_v * rl::delta_chunk_record_bytes(), 256) + align_up(n_chunks * p->n_v * sizeof(float), 256) +
           align_up(n_chunks * p->n_qk * rl::delta_chunk_keys_bytes(), 256);
}

double rl_delta_chunk_mma_flops(void) { return rl::delta_chunk_scan_mma_flops(); }

int rl_delta_chunk_prefill(float* S, const float* q, const float* k, const float* v, const float* beta,
                           const float* g_log, float* o, void* workspace, size_t workspace_bytes,
                           const rl_delta_chunk_params* p, void* stream) {
    if (int st = delta_chunk_check(p)) return st;
    if (p->seq == 0) return RL_OK;
    if (!S || !q || !k || !v || !beta || !g_log || !o || !workspace) return fail(RL_ERR_RANGE, "NULL pointer argument");
    const size_t need = rl_delta_chunk_workspace_bytes(p);
    if (workspace_bytes < need) return fail(RL_ERR_RANGE, "workspace %zu bytes < %zu required", workspace_bytes, need);
    if (reinterpret_cast<uintptr_t>(workspace) % 256 || reinterpret_cast<uintptr_t>(q) % 16 ||
        reinterpret_cast<uintptr_t>(k) % 16 || reinterpret_cast<uintptr_t>(v) % 16)
        return fail(RL_ERR_RANGE, "workspace must be 256-byte aligned, q, k, v 16-byte aligned");
    DevInfo* d;
    if (int st = dev_info(&d)) return st;
    const int n_chunks = (p->seq + 63) / 64;
    rl::DeltaChunkArgs a;
    a.S = S;
    a.q = q;
    a.k = k;
    a.v = v;
    a.beta = beta;
    a.g_log = g_log;
    a.o = o;
    a.work = static_cast<unsigned char*>(workspace);
    a.chunk_decay = reinterpret_cast<float*>(a.work + align_up(size_t(n_chunks) * p->n_v * rl::delta_chunk_record_bytes(), 256));
    a.keys = reinterpret_cast<float*>(reinterpret_cast<unsigned char*>(a.chunk_decay) + align_up(size_t(n_chunks) * p->n_v * sizeof(float), 256));
    a.err = d->err_ptr;
    a.T = p->seq;
    a.n_v = p->n_v;
    a.n_qk = p->n_qk;
    a.head_map = p->head_map;
    a.eps_l2 = p->eps_l2;
    a.qk_tok_stride = p->qk_tok_stride ? p->qk_tok_stride : 1LL * p->n_qk * p->dk;
    a.v_tok_stride = p->v_tok_stride ? p->v_tok_stride : 1LL * p->n_v * p->dv;
    if ((a.qk_tok_stride | a.v_tok_stride) % 4 || a.qk_tok_stride < 0 || a.v_tok_stride < 0)
        return fail(RL_ERR_RANGE, "token strides must be non-negative multiples of 4 floats");
    // The scan of a value head walks its chunks in order on one SM (n_v CTAs), the chunk-local
    // precompute fills the device.  Long sequences are cut into a few segments so that the scan of one
    // segment (second stream, higher priority) runs beside the precompute of the next.  The two compete
    // for the same SMs, so the gain is modest (T 8192: 1.11 -> 0.97 ms with four segments) and below 32
    // chunks the extra launches cost more than the overlap returns.  What the key heads share is computed
    // for all chunks first.
    int n_seg = n_chunks < 32 ? 1 : (n_chunks < 64 ? 2 : (n_chunks < 128 ? 3 : 4));
    if (kDeltaChunkSegs > 0) n_seg = std::max(1, std::min({kDeltaChunkSegs, int(sizeof(AuxSet::fork) / sizeof(AuxSet::fork[0])), n_chunks}));
    cudaStream_t run = as_stream(stream);
    // All three kernels wait for the kernel in front (griddepcontrol.wait) before their first global access, so
    // on the caller's stream they are launched for programmatic dependent launch; the scans of a segmented call
    // follow an event on the second stream and are launched plainly.
    auto prepare = [&](int c0, int n, cudaStream_t st) {
        a.chunk0 = c0;
        a.chunks = n;
        return rl::launch_step(rl::delta_chunk_prepare_kernel, dim3(n, p->n_v), dim3(rl::delta_chunk_prepare_threads()),
                               rl::delta_chunk_prepare_smem_bytes(), st, a);
    };
    auto scan = [&](int c0, int n, cudaStream_t st) {
        a.chunk0 = c0;
        a.chunks = n;
        return rl::launch_step(rl::delta_chunk_scan_kernel, dim3(p->n_v), dim3(rl::delta_chunk_scan_threads()),
                               rl::delta_chunk_scan_smem_bytes(), st, a);
    };
    a.chunk0 = 0;
    a.chunks = n_chunks;
    {
        StepOverlap overlap(true);
        RL_CUDA(rl::launch_step(rl::delta_chunk_keys_kernel, dim3(n_chunks, p->n_qk), dim3(rl::delta_chunk_prepare_threads()),
                                rl::delta_chunk_prepare_smem_bytes(), run, a));
    }
    if (n_seg == 1) {
        StepOverlap overlap(true);
        RL_CUDA(prepare(0, n_chunks, run));
        RL_CUDA(scan(0, n_chunks, run));
    } else {
        AuxSet* aux = nullptr;
        if (int st = aux_acquire(d, &aux)) return st;
        for (int i = 0; i < n_seg; ++i) {
            const int c0 = int(1LL * i * n_chunks / n_seg), c1 = int(1LL * (i + 1) * n_chunks / n_seg);
            {
                StepOverlap overlap(true);
                RL_CUDA(prepare(c0, c1 - c0, run));
            }
            RL_CUDA(cudaEventRecord(aux->fork[i], run));
            RL_CUDA(cudaStreamWaitEvent(aux->stream, aux->fork[i], 0));   // also orders the first scan after the caller's work
            StepOverlap plain(false);
            RL_CUDA(scan(c0, c1 - c0, aux->stream));
        }
        RL_CUDA(cudaEventRecord(aux->join, aux->stream));
        aux->used = true;
        RL_CUDA(cudaStreamWaitEvent(run, aux->join, 0));
    }
    RL_CUDA(cudaGetLastError());
    return RL_OK;
}

int rl_gdn_decode(float* S, float* conv_ring, const int32_t* conv_phase, const int32_t* slot_ids, const float* qkv,
                  const float* conv_w, const float* beta, const float* g_log, float* o, const rl_gdn_decode_params* p,
                  void* stream) {
    if (!p) return fail(RL_ERR_RANGE, "params is NULL");
    if (p->dk != 128 || p->dv != 128 || p->conv_k != 4)
        return fail(RL_ERR_UNSUPPORTED, "dk %d dv %d conv_k %d: only 128 x 128, 4 taps", p->dk, p->dv, p->conv_k);
    if (p->n_v <= 0 || p->n_v > 65535 || p->batch < 0 || p->batch > 65535 || p->n_slots <= 0)
        return fail(RL_ERR_RANGE, "n_v %d batch %d n_slots %d", p->n_v, p->batch, p->n_slots);
    if (p->head_map == RL_HEADS_PER_VALUE ? p->n_qk != p->n_v
                                          : (p->n_qk <= 0 || p->n_v % p->n_qk != 0 || p->head_map > RL_HEADS_TILED))
        return fail(RL_ERR_RANGE, "n_qk %d does not fit n_v %d with head_map %d", p->n_qk, p->n_v, p->head_map);
    if (p->batch == 0) return RL_OK;
    if (!S || !conv_ring || !conv_phase || !qkv || !conv_w || !beta || !g_log || !o) return fail(RL_ERR_RANGE, "NULL pointer argument");
    if (reinterpret_cast<uintptr_t>(S) % 16 || reinterpret_cast<uintptr_t>(conv_ring) % 16 ||
        reinterpret_cast<uintptr_t>(qkv) % 16 || reinterpret_cast<uintptr_t>(conv_w) % 16)
        return fail(RL_ERR_RANGE, "S, conv_ring, qkv and conv_w must be 16-byte aligned");
    DevInfo* d;
    if (int st = dev_info(&d)) return st;
    rl::GdnDecodeArgs a;
    a.S = S;
    a.conv = conv_ring;
    a.conv_phase = conv_phase;
    a.slot_ids = slot_ids;
    a.x = qkv;
    a.w = conv_w;
    a.beta = beta;
    a.g_log = g_log;
    a.o = o;
    a.err = d->err_ptr;
    a.batch = p->batch;
    a.n_v = p->n_v;
    a.n_qk = p->n_qk;
    a.n_slots = p->n_slots;
    a.head_map = p->head_map;
    a.conv_dim = 2 * p->n_qk * p->dk + p->n_v * p->dv;
    a.eps_l2 = p->eps_l2;
    a.early = g_gdn_early && rl::g_step_overlap && !rl::g_step_first ? 1 : 0;
    rl::launch_gdn_decode(a, step_sms(d->sms), as_stream(stream), kGdnStreamMin, kGdnGrid);
    RL_CUDA(cudaGetLastError());
    return RL_OK;
}

int rl_gdn_phase_advance(int32_t* conv_phase, const int32_t* slot_ids, int n_layers, int n_slots, int batch, int n_tok,
                         void* stream) {
    if (n_layers < 0 || n_slots <= 0 || batch < 0 || n_tok < 0) return fail(RL_ERR_RANGE, "n_layers %d n_slots %d batch %d n_tok %d", n_layers, n_slots, batch, n_tok);
    if (n_layers == 0 || batch == 0) return RL_OK;
    if (!conv_phase) return fail(RL_ERR_RANGE, "NULL pointer argument");
    DevInfo* d;
    if (int st = dev_info(&d)) return st;
    rl::launch_gdn_phase_advance(conv_phase, slot_ids, n_layers, n_slots, batch, n_tok, d->err_ptr, as_stream(stream));
    RL_CUDA(cudaGetLastError());
    return RL_OK;
}

static int ring_args_check(const void* ring, const void* phase, const void* canon, int n_layers, int n_slots, int slot, int dim) {
    if (n_layers < 0 || n_slots <= 0 || n_slots > 65535 || n_layers > 65535 || slot >= n_slots || dim <= 0)
        return fail(RL_ERR_RANGE, "n_layers %d n_slots %d slot %d conv_dim %d", n_layers, n_slots, slot, dim);
    if (n_layers && (!ring || !phase || !canon)) return fail(RL_ERR_RANGE, "NULL pointer argument");
    if (reinterpret_cast<uintptr_t>(ring) % 16 || reinterpret_cast<uintptr_t>(canon) % 16)
        return fail(RL_ERR_RANGE, "windows must be 16-byte aligned");
    return RL_OK;
}

int rl_conv_ring_export(const float* conv_ring, const int32_t* conv_phase, float* canon, int n_layers, int n_slots,
                        int slot, int conv_dim, void* stream) {
    if (int st = ring_args_check(conv_ring, conv_phase, canon, n_layers, n_slots, slot, conv_dim)) return st;
    rl::launch_conv_ring_export(conv_ring, conv_phase, canon, n_layers, n_slots, slot, conv_dim, as_stream(stream));
    RL_CUDA(cudaGetLastError());
    return RL_OK;
}

int rl_conv_ring_import(float* conv_ring, int32_t* conv_phase, const float* canon, int n_layers, int n_slots, int slot,
                        int conv_dim, void* stream) {
    if (int st = ring_args_check(conv_ring, conv_phase, canon, n_layers, n_slots, slot, conv_dim)) return st;
    rl::launch_conv_ring_import(conv_ring, conv_phase, canon, n_layers, n_slots, slot, conv_dim, as_stream(stream));
    RL_CUDA(cudaGetLastError());
    return RL_OK;
}

int rl_conv1d_update(const float* x, const float* w, float* state, const int32_t* slot_ids, float* y,
                     const rl_conv1d_params* p, void* stream) {
    if (!p) return fail(RL_ERR_RANGE, "params is NULL");
    if (!p->silu) return fail(RL_ERR_UNSUPPORTED, "conv1d without SiLU is not on this path");
    if (p->dim <= 0 || p->k < 1 || p->k > 8 || p->batch < 0 || p->batch > 65535 || p->n_slots <= 0)
        return fail(RL_ERR_RANGE, "dim %d k %d batch %d n_slots %d", p->dim, p->k, p->batch, p->n_slots);
    if (p->batch == 0) return RL_OK;
    if (!x || !w || !state || !y) return fail(RL_ERR_RANGE, "NULL pointer argument");
    DevInfo* d;
    if (int st = dev_info(&d)) return st;
    rl::ConvUpdateArgs a;
    a.x = x;
    a.w = w;
    a.state = state;
    a.slot_ids = slot_ids;
    a.y = y;
    a.err = d->err_ptr;
    a.batch = p->batch;
    a.dim = p->dim;
    a.k = p->k;
    a.n_slots = p->n_slots;
    if (p->k == 4 && (reinterpret_cast<uintptr_t>(w) % 16 || reinterpret_cast<uintptr_t>(state) % 16))
        return fail(RL_ERR_RANGE, "w and state must be 16-byte aligned");
    rl::launch_conv1d_update(a, as_stream(stream));
    RL_CUDA(cudaGetLastError());
    return RL_OK;
}

int rl_conv1d_causal(const float* x, const float* w, float* y, float* state_io, int seq,
                     const rl_conv1d_params* p, int use_state_in, void* stream) {
    if (!p) return fail(RL_ERR_RANGE, "params is NULL");
    if (!p->silu) return fail(RL_ERR_UNSUPPORTED, "conv1d without SiLU is not on this path");
    if (p->dim <= 0 || p->k < 1 || p->k > 8 || seq < 0) return fail(RL_ERR_RANGE, "dim %d k %d seq %d", p->dim, p->k, seq);
    if (seq == 0) return RL_OK;
    if (!x || !w || !y) return fail(RL_ERR_RANGE, "NULL pointer argument");
    rl::launch_conv1d_prefill(x, w, y, state_io, seq, p->dim, p->k, use_state_in, as_stream(stream));
    RL_CUDA(cudaGetLastError());
    return RL_OK;
}

// ------------------------------------------------------------------------------------
// ---- trees of drafted tokens ----------------------------------------------------------------------

static int tree_shape_check(int n_kv, int head_dim, int batch, int max_nodes, int page_tokens, int n_pages,
                            int max_pages_per_seq) {
    if (head_dim != rl::kHeadDim || page_tokens != rl::kPageTokens)
        return fail(RL_ERR_UNSUPPORTED, "head_dim %d / page_tokens %d: only 256 / 64", head_dim, page_tokens);
    if (n_kv <= 0 || n_kv > 65535 || batch < 0 || batch > 65535) return fail(RL_ERR_RANGE, "n_kv %d batch %d", n_kv, batch);
    if (max_nodes < 0 || max_nodes > RL_TREE_MAX_NODES)
        return fail(RL_ERR_RANGE, "%d nodes per sequence: at most %d", max_nodes, RL_TREE_MAX_NODES);
    if (n_pages <= 0 || max_pages_per_seq <= 0 || max_pages_per_seq > 0x7fffffff / rl::kPageTokens)
        return fail(RL_ERR_RANGE, "n_pages %d max_pages_per_seq %d", n_pages, max_pages_per_seq);
    return RL_OK;
}
static bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
// the distance of a caller's rows: 0 = dense; else at least a row, in units that keep 16-byte loads aligned
static bool row_stride(long long given, long long dense, size_t* out) {
    *out = size_t(given ? given : dense);
    return given == 0 || (given >= dense && given % 4 == 0);
}

int rl_attn_qk_append(void* k_pool, void* v_pool, const int32_t* page_table, const int32_t* pos, const int32_t* parents,
                      const int32_t* n_nodes, const float* qg, const float* k, const float* v, const float* q_norm,
                      const float* k_norm, void* q_out, float* gate_out, const rl_attn_qk_append_params* p, void* stream) {
    if (!p) return fail(RL_ERR_RANGE, "params is NULL");
    if (int st = tree_shape_check(p->n_kv, p->head_dim, p->batch, 0, p->page_tokens, p->n_pages, p->max_pages_per_seq)) return st;
    if (p->n_q <= 0 || p->n_q > 65535 || p->n_tok < 0 || 1LL * p->batch * p->n_tok > 0x7fffffff)
        return fail(RL_ERR_RANGE, "n_q %d batch %d n_tok %d", p->n_q, p->batch, p->n_tok);
    if (parents && p->n_tok > RL_TREE_MAX_NODES)
        return fail(RL_ERR_RANGE, "%d nodes per sequence: at most %d", p->n_tok, RL_TREE_MAX_NODES);
    if (p->rotary_dim < 0 || p->rotary_dim > p->head_dim || p->rotary_dim % 16)
        return fail(RL_ERR_RANGE, "rotary_dim %d must be a multiple of 16 and at most head_dim", p->rotary_dim);
    if (p->rotary_dim > 0 && !(p->theta > 0.f)) return fail(RL_ERR_RANGE, "theta must be positive");
    if (p->q_type != RL_TYPE_F32 && p->q_type != RL_TYPE_F16 && p->q_type != RL_TYPE_BF16)
        return fail(RL_ERR_UNSUPPORTED, "q_type %d unknown", p->q_type);
    rl::AttnQkAppendArgs a;
    if (!row_stride(p->qg_stride, 2LL * p->n_q * rl::kHeadDim, &a.qg_stride) ||
        !row_stride(p->k_stride, 1LL * p->n_kv * rl::kHeadDim, &a.k_stride) ||
        !row_stride(p->v_stride, 1LL * p->n_kv * rl::kHeadDim, &a.v_stride))
        return fail(RL_ERR_RANGE, "row strides %lld %lld %lld: at least a row, multiples of 4", p->qg_stride, p->k_stride, p->v_stride);
    if (p->batch == 0 || p->n_tok == 0) return RL_OK;
    if (!k_pool || !v_pool || !page_table || !pos || !qg || !k || !v || !q_out) return fail(RL_ERR_RANGE, "NULL pointer argument");
    if (!aligned16(k_pool) || !aligned16(v_pool) || !aligned16(qg) || !aligned16(k) || !aligned16(v) || !aligned16(q_norm) ||
        !aligned16(k_norm) || !aligned16(q_out) || !aligned16(gate_out))
        return fail(RL_ERR_RANGE, "pools, rows and norms must be 16-byte aligned");
    DevInfo* d;
    if (int st = dev_info(&d)) return st;
    a.k_pool = static_cast<__half*>(k_pool);
    a.v_pool = static_cast<__half*>(v_pool);
    a.page_table = page_table;
    a.pos = pos;
    a.parents = parents;
    a.n_nodes = n_nodes;
    a.qg = qg;
    a.k = k;
    a.v = v;
    a.q_norm = q_norm;
    a.k_norm = k_norm;
    a.q_out = q_out;
    a.gate_out = gate_out;
    a.err = d->err_ptr;
    a.n_q = p->n_q;
    a.n_kv = p->n_kv;
    a.n_tok = p->n_tok;
    a.n_pages = p->n_pages;
    a.max_pages_per_seq = p->max_pages_per_seq;
    a.rotary_dim = p->rotary_dim;
    a.q_type = p->q_type;
    a.eps = p->eps;
    const int pairs = p->rotary_dim / 2;
    for (int i = 0; i < pairs; ++i)
        a.rate[i] = p->angle_f32 ? double(1.f / powf(p->theta, float(i) / float(pairs))) : pow(double(p->theta), -double(i) / pairs) / 6.283185307179586476925;
    a.angle_f32 = p->angle_f32;
    rl::launch_attn_qk_append(a, p->batch, as_stream(stream));
    RL_CUDA(cudaGetLastError());
    return RL_OK;
}

static int attn_tree_check(const rl_attn_tree_params* p) {
    if (!p) return fail(RL_ERR_RANGE, "params is NULL");
    if (int st = tree_shape_check(p->n_kv, p->head_dim, p->batch, p->max_nodes, p->page_tokens, p->n_pages, p->max_pages_per_seq))
        return st;
    if (p->n_q <= 0 || p->n_q % p->n_kv != 0 || p->n_q / p->n_kv > 8)
        return fail(RL_ERR_UNSUPPORTED, "n_q %d / n_kv %d: group must divide and be <= 8", p->n_q, p->n_kv);
    if (p->batch > rl::attn_tree_max_batch()) return fail(RL_ERR_RANGE, "batch %d above %d", p->batch, rl::attn_tree_max_batch());
    if (p->max_seq_len <= 0 || p->max_seq_len > p->max_pages_per_seq * p->page_tokens)
        return fail(RL_ERR_RANGE, "max_seq_len %d outside (0, max_pages_per_seq*page_tokens]", p->max_seq_len);
    if (p->q_type != RL_TYPE_F32 && p->q_type != RL_TYPE_F16 && p->q_type != RL_TYPE_BF16)
        return fail(RL_ERR_UNSUPPORTED, "q_type %d unknown", p->q_type);
    if (p->o_type != RL_TYPE_F16 && p->o_type != RL_TYPE_BF16)
        return fail(RL_ERR_UNSUPPORTED, "o_type %d: only RL_TYPE_F16 and RL_TYPE_BF16", p->o_type);
    const long long row_tiles = (1LL * p->max_nodes * (p->n_q / p->n_kv) + rl::attn_tree_rows() - 1) / rl::attn_tree_rows();
    if (1LL * p->batch * p->n_kv * row_tiles * (p->max_pages_per_seq + 64LL) > 0x3fffffff)
        return fail(RL_ERR_RANGE, "batch %d, n_kv %d, max_pages_per_seq %d: too many pages in one call", p->batch, p->n_kv, p->max_pages_per_seq);
    return RL_OK;
}

// One persistent CTA per SM, fewer when the batch has less than kTreeMinShare pages for each: 8 nodes over 2 000
// tokens take 15.3 us with 1 page, 14.8 with 2, 16.2 with 3, 16.5 with 4 (more CTAs leave more partials to merge).
static const int kTreeMinShare = knob("RL_B200_TREE_MIN_SHARE", 2);
// What a CTA pays to close one (sequence, head, row tile) and open the next (partial out, queries in, behind the pages
// already requested), in pages.  Sustained, with 8, 12, 16 and 24: 16 trees of 21 over 16K (16-bit queries) 179, 173, 171 and
// 177 us, over 2 000 tokens 50.7, 48.0, 49.3 and 53.2, 4 trees of 64 over 32K 217, 213, 214 and 218 (+- 2).
static const int kTreeBoundary = knob("RL_B200_TREE_BOUNDARY", 16);
struct AttnTreePlan {
    int grid;
    size_t o_bytes, total_bytes;
};
static AttnTreePlan attn_tree_plan(const rl_attn_tree_params* p, int sms) {
    AttnTreePlan pl;
    const int rows = rl::attn_tree_rows();
    const long long segs = 1LL * p->batch * p->n_kv * ((p->max_nodes * (p->n_q / p->n_kv) + rows - 1) / rows);
    const long long units = segs * (ceil_div(p->max_seq_len, p->page_tokens) + kTreeBoundary);
    pl.grid = int(std::max(1LL, std::min(1LL * sms, (units + kTreeMinShare - 1) / kTreeMinShare)));
    const size_t slots = size_t(pl.grid) + size_t(segs);
    pl.o_bytes = align_up(slots * rows * rl::kHeadDim * sizeof(float), 256);
    pl.total_bytes = pl.o_bytes + align_up(slots * rows * 2 * sizeof(float), 256);
    return pl;
}

size_t rl_attn_tree_workspace_bytes(const rl_attn_tree_params* p) {
    if (attn_tree_check(p)) return 0;
    DevInfo* d;
    if (dev_info(&d)) return 0;
    return attn_tree_plan(p, step_sms(d->sms)).total_bytes;
}

int rl_attn_tree(const void* k_pool, const void* v_pool, const int32_t* page_table, const int32_t* base_len,
                 const int32_t* parents, const int32_t* n_nodes, const void* q, const float* gate, void* o, void* workspace,
                 size_t workspace_bytes, const rl_attn_tree_params* p, void* stream) {
    if (int st = attn_tree_check(p)) return st;
    rl::AttnTreeArgs a;
    const long long head = p->gate_head ? p->gate_head : rl::kHeadDim;
    if (head < rl::kHeadDim || head % 4 || !row_stride(p->gate_row, head * p->n_q, &a.gate_row))
        return fail(RL_ERR_RANGE, "gate strides %lld %lld: at least a row and a head, multiples of 4", p->gate_row, p->gate_head);
    if (p->batch == 0 || p->max_nodes == 0) return RL_OK;
    if (!k_pool || !v_pool || !page_table || !base_len || !q || !o || !workspace) return fail(RL_ERR_RANGE, "NULL pointer argument");
    if (reinterpret_cast<uintptr_t>(k_pool) % 128 || reinterpret_cast<uintptr_t>(v_pool) % 128 ||
        reinterpret_cast<uintptr_t>(q) % 32 || reinterpret_cast<uintptr_t>(o) % 32 || reinterpret_cast<uintptr_t>(workspace) % 32 ||
        !aligned16(gate))
        return fail(RL_ERR_RANGE, "pools must be 128-byte aligned, q, o and workspace 32-byte, gate 16-byte");
    DevInfo* d;
    if (int st = dev_info(&d)) return st;
    const AttnTreePlan pl = attn_tree_plan(p, step_sms(d->sms));
    if (workspace_bytes < pl.total_bytes)
        return fail(RL_ERR_RANGE, "workspace %zu bytes < %zu required", workspace_bytes, pl.total_bytes);
    a.k_pool = static_cast<const __half*>(k_pool);
    a.v_pool = static_cast<const __half*>(v_pool);
    a.page_table = page_table;
    a.base_len = base_len;
    a.parents = parents;
    a.n_nodes = n_nodes;
    a.q = q;
    a.gate = gate;
    a.o = o;
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = reinterpret_cast<float*>(static_cast<char*>(workspace) + pl.o_bytes);
    a.err = d->err_ptr;
    a.gate_head = size_t(head);
    a.batch = p->batch;
    a.max_nodes = p->max_nodes;
    a.n_q = p->n_q;
    a.n_kv = p->n_kv;
    a.n_pages = p->n_pages;
    a.max_pages_per_seq = p->max_pages_per_seq;
    a.max_len = p->max_seq_len;
    a.q_type = p->q_type;
    a.o_type = p->o_type;
    a.grid = pl.grid;
    a.min_share = kTreeMinShare;
    a.boundary = kTreeBoundary;
    a.scale = 1.f / sqrtf(float(p->head_dim));
    RL_CUDA(rl::launch_attn_tree(a, as_stream(stream)));
    RL_CUDA(cudaGetLastError());
    return RL_OK;
}

int rl_kv_tree_commit(void* k_pool, void* v_pool, const int32_t* page_table, const int32_t* base_len, const int32_t* parents,
                      const int32_t* leaf, int32_t* n_accept, const rl_kv_tree_commit_params* p, void* stream) {
    if (!p) return fail(RL_ERR_RANGE, "params is NULL");
    if (int st = tree_shape_check(p->n_kv, p->head_dim, p->batch, p->max_nodes, p->page_tokens, p->n_pages, p->max_pages_per_seq))
        return st;
    if (p->batch == 0) return RL_OK;
    if (!k_pool || !v_pool || !page_table || !base_len || !leaf) return fail(RL_ERR_RANGE, "NULL pointer argument");
    if (!aligned16(k_pool) || !aligned16(v_pool)) return fail(RL_ERR_RANGE, "pools must be 16-byte aligned");
    DevInfo* d;
    if (int st = dev_info(&d)) return st;
    rl::KvTreeCommitArgs a;
    a.k_pool = static_cast<__half*>(k_pool);
    a.v_pool = static_cast<__half*>(v_pool);
    a.page_table = page_table;
    a.base_len = base_len;
    a.parents = parents;
    a.n_nodes = p->n_nodes;
    a.leaf = leaf;
    a.n_accept = n_accept;
    a.err = d->err_ptr;
    a.n_kv = p->n_kv;
    a.max_nodes = p->max_nodes;
    a.n_pages = p->n_pages;
    a.max_pages_per_seq = p->max_pages_per_seq;
    rl::launch_kv_tree_commit(a, p->batch, as_stream(stream));
    RL_CUDA(cudaGetLastError());
    return RL_OK;
}

static int gdn_tree_check(const rl_gdn_tree_params* p, rl::GdnTreeArgs* a) {
    if (!p) return fail(RL_ERR_RANGE, "params is NULL");
    if (p->dk != 128 || p->dv != 128 || p->conv_k != 4)
        return fail(RL_ERR_UNSUPPORTED, "dk %d dv %d conv_k %d: only 128 x 128, 4 taps", p->dk, p->dv, p->conv_k);
    if (p->n_v <= 0 || p->n_v > 65535 || p->batch < 0 || p->batch > 65535 || p->n_slots <= 0)
        return fail(RL_ERR_RANGE, "n_v %d batch %d n_slots %d", p->n_v, p->batch, p->n_slots);
    if (p->head_map == RL_HEADS_PER_VALUE
            ? p->n_qk != p->n_v
            : (p->n_qk <= 0 || p->n_v % p->n_qk != 0 || p->head_map < 0 || p->head_map > RL_HEADS_TILED))
        return fail(RL_ERR_RANGE, "n_qk %d does not fit n_v %d with head_map %d", p->n_qk, p->n_v, p->head_map);
    if (p->max_nodes < 0 || p->max_nodes > RL_TREE_MAX_NODES)
        return fail(RL_ERR_RANGE, "%d nodes per sequence: at most %d", p->max_nodes, RL_TREE_MAX_NODES);
    a->conv_dim = 2 * p->n_qk * p->dk + p->n_v * p->dv;
    if (!row_stride(p->qkv_stride, a->conv_dim, &a->x_stride))
        return fail(RL_ERR_RANGE, "qkv_stride %lld: at least a row, a multiple of 4", p->qkv_stride);
    if (a->x_stride > 0x7fffffff / RL_TREE_MAX_NODES) return fail(RL_ERR_RANGE, "qkv_stride %lld: rows too far apart", p->qkv_stride);
    return RL_OK;
}
static int gdn_tree_args(rl::GdnTreeArgs* a, const float* S, const float* conv_window, const int32_t* conv_phase,
                         const int32_t* slot_ids, const int32_t* parents, const float* qkv, const float* conv_w,
                         const float* beta, const float* g_log, const rl_gdn_tree_params* p) {
    if (int st = gdn_tree_check(p, a)) return st;
    if (p->batch == 0 || p->max_nodes == 0) return RL_OK;
    if (!S || !conv_window || !qkv || !conv_w || !beta || !g_log) return fail(RL_ERR_RANGE, "NULL pointer argument");
    if (!aligned16(S) || !aligned16(conv_window) || !aligned16(qkv) || !aligned16(conv_w))
        return fail(RL_ERR_RANGE, "S, conv_window, qkv and conv_w must be 16-byte aligned");
    DevInfo* d;
    if (int st = dev_info(&d)) return st;
    a->S = S;
    a->conv = conv_window;
    a->conv_phase = conv_phase;
    a->slot_ids = slot_ids;
    a->parents = parents;
    a->x = qkv;
    a->w = conv_w;
    a->beta = beta;
    a->g_log = g_log;
    a->err = d->err_ptr;
    a->batch = p->batch;
    a->max_nodes = p->max_nodes;
    a->n_v = p->n_v;
    a->n_qk = p->n_qk;
    a->n_slots = p->n_slots;
    a->head_map = p->head_map;
    a->eps_l2 = p->eps_l2;
    return RL_OK;
}

size_t rl_gdn_tree_workspace_bytes(const rl_gdn_tree_params* p) {
    rl::GdnTreeArgs a = {};
    if (gdn_tree_check(p, &a)) return 0;
    return std::max<size_t>(256, rl::gdn_tree_workspace_bytes(p->batch, p->max_nodes, p->n_v, p->n_qk));
}

int rl_gdn_tree(const float* S, const float* conv_window, const int32_t* conv_phase, const int32_t* slot_ids,
                const int32_t* parents, const int32_t* n_nodes, const float* qkv, const float* conv_w, const float* beta,
                const float* g_log, float* o, void* workspace, size_t workspace_bytes, const rl_gdn_tree_params* p, void* stream) {
    rl::GdnTreeArgs a = {};
    if (int st = gdn_tree_args(&a, S, conv_window, conv_phase, slot_ids, parents, qkv, conv_w, beta, g_log, p)) return st;
    if (p->batch == 0 || p->max_nodes == 0) return RL_OK;
    if (!o || !workspace) return fail(RL_ERR_RANGE, "NULL pointer argument");
    if (!aligned16(o) || !aligned16(workspace)) return fail(RL_ERR_RANGE, "o and workspace must be 16-byte aligned");
    const size_t need = rl::gdn_tree_workspace_bytes(p->batch, p->max_nodes, p->n_v, p->n_qk);
    if (workspace_bytes < need) return fail(RL_ERR_RANGE, "workspace %zu bytes < %zu required", workspace_bytes, need);
    a.n_nodes = n_nodes;
    a.o = o;
    a.workspace = workspace;
    DevInfo* d;
    if (int st = dev_info(&d)) return st;
    RL_CUDA(rl::launch_gdn_tree(a, d->sms, as_stream(stream)));
    RL_CUDA(cudaGetLastError());
    return RL_OK;
}

size_t rl_gdn_tree_commit_workspace_bytes(const rl_gdn_tree_params* p) {
    rl::GdnTreeArgs a = {};
    if (gdn_tree_check(p, &a)) return 0;
    return std::max<size_t>(256, rl::gdn_tree_commit_workspace_bytes(p->batch, p->max_nodes, p->n_v, p->n_qk));
}

int rl_gdn_tree_commit(float* S, float* conv_window, const int32_t* conv_phase, const int32_t* slot_ids,
                       const int32_t* parents, const int32_t* leaf, const float* qkv, const float* conv_w, const float* beta,
                       const float* g_log, void* workspace, size_t workspace_bytes, const rl_gdn_tree_params* p, void* stream) {
    rl::GdnTreeArgs a = {};
    if (int st = gdn_tree_args(&a, S, conv_window, conv_phase, slot_ids, parents, qkv, conv_w, beta, g_log, p)) return st;
    if (p->batch == 0 || p->max_nodes == 0) return RL_OK;
    if (!leaf || !workspace) return fail(RL_ERR_RANGE, "NULL pointer argument");
    if (!aligned16(workspace)) return fail(RL_ERR_RANGE, "workspace must be 16-byte aligned");
    const size_t need = rl::gdn_tree_commit_workspace_bytes(p->batch, p->max_nodes, p->n_v, p->n_qk);
    if (workspace_bytes < need) return fail(RL_ERR_RANGE, "workspace %zu bytes < %zu required", workspace_bytes, need);
    a.n_nodes = p->commit_nodes;
    a.leaf = leaf;
    a.S_out = S;
    a.conv_out = conv_window;
    a.workspace = workspace;
    RL_CUDA(rl::launch_gdn_tree_commit(a, as_stream(stream)));
    RL_CUDA(cudaGetLastError());
    return RL_OK;
}

int rl_plan_cache(const rl_plan_input* in, rl_plan_result* out) {
    if (!in || !out) return fail(RL_ERR_RANGE, "NULL argument");
    if (in->ctx <= 0 || in->max_batch <= 0 || in->page_tokens <= 0 || in->n_attn_layers < 0 || in->n_delta_layers < 0 ||
        in->n_kv < 0 || in->head_dim < 0 || in->kv_policy < RL_KV_POLICY_AUTO || in->kv_policy > RL_KV_POLICY_COMPACT)
        return fail(RL_ERR_RANGE, "ctx %d max_batch %d page_tokens %d kv_policy %d", in->ctx, in->max_batch,
                    in->page_tokens, in->kv_policy);
    std::memset(out, 0, sizeof *out);
    typedef unsigned long long u64;
    // bytes of one page over all attention layers (K and V)
    const u64 f16_page = u64(in->n_attn_layers) * in->n_kv * in->page_tokens * in->head_dim * 2 * 2;
    const u64 compact_page = u64(in->n_attn_layers) * in->n_kv * rl_kv_compact_page_bytes();
    out->state_bytes = u64(in->max_batch) * in->n_delta_layers *
                       (u64(in->n_v) * in->dk * in->dv * 4 + u64(in->conv_dim) * in->conv_k * 4);
    const u64 fixed = in->weight_bytes + out->state_bytes + in->pad_bytes;
    auto pages_for = [&](int ctx) { return u64((ctx + in->page_tokens - 1) / in->page_tokens); };
    // the compact cache carries an F16 window over the first tokens of every sequence
    auto window_of = [&](int ctx) { return std::min(ctx, std::max(8192, 2 * (in->prefill_chunk > 0 ? in->prefill_chunk : 1024))); };
    auto kv_bytes_of = [&](int dtype, int ctx) {
        if (dtype == RL_KV_F16) return f16_page * pages_for(ctx) * in->max_batch;
        return (compact_page * pages_for(ctx) + f16_page * pages_for(window_of(ctx))) * in->max_batch;
    };
    auto fits = [&](int dtype, int ctx) {
        return !in->available_bytes || fixed + kv_bytes_of(dtype, ctx) <= in->available_bytes;
    };
    int dtype = in->kv_policy == RL_KV_POLICY_COMPACT ? RL_KV_Q8K_TQ3V : RL_KV_F16;
    if (in->kv_policy == RL_KV_POLICY_AUTO && !fits(RL_KV_F16, in->ctx)) dtype = RL_KV_Q8K_TQ3V;
    if (dtype == RL_KV_Q8K_TQ3V && in->head_dim != rl::kHeadDim && in->n_attn_layers > 0) {
        if (in->kv_policy == RL_KV_POLICY_COMPACT)
            return fail(RL_ERR_UNSUPPORTED, "the compact cache needs head_dim 256, got %d", in->head_dim);
        dtype = RL_KV_F16;
    }
    int ctx = in->ctx;
    if (!fits(dtype, ctx) && in->allow_shrink) {
        // largest whole number of pages per sequence that fits (the window makes the cost piecewise linear)
        int lo = 0, hi = int(pages_for(in->ctx));
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (fits(dtype, mid * in->page_tokens)) lo = mid;
            else hi = mid - 1;
        }
        ctx = int(std::min<u64>(u64(lo) * in->page_tokens, u64(in->ctx)));
    }
    out->kv_dtype = dtype;
    out->ctx = ctx;
    out->max_pages_per_seq = int(pages_for(std::max(ctx, 1)));
    out->n_pages = out->max_pages_per_seq * in->max_batch;
    if (dtype != RL_KV_F16 && ctx > 0) {
        out->window_tokens = window_of(ctx);
        out->window_pages_per_seq = int(pages_for(out->window_tokens));
        out->window_bytes = f16_page * u64(out->window_pages_per_seq) * in->max_batch;
    }
    out->kv_bytes = ctx > 0 ? kv_bytes_of(dtype, ctx) : 0;
    out->need_bytes = fixed + out->kv_bytes;
    out->ok = ctx > 0 && (!in->available_bytes || out->need_bytes <= in->available_bytes);
    if (out->ok)
        std::snprintf(out->message, sizeof out->message, ctx == in->ctx ? "ok" : "ok: ctx reduced from %d to %d", in->ctx, ctx);
    else
        std::snprintf(out->message, sizeof out->message, "OOM: need %llu bytes, available %llu (ctx=%d)",
                      out->need_bytes, in->available_bytes, in->ctx);
    return RL_OK;
}

int rl_cache_create(const rl_cache_config* cfg, rl_cache** out) {
    if (!cfg || !out) return fail(RL_ERR_RANGE, "NULL argument");
    *out = nullptr;
    if (cfg->n_layers <= 0 || !cfg->layer_types) return fail(RL_ERR_RANGE, "no layers");
    if (cfg->head_dim != rl::kHeadDim || cfg->page_tokens != rl::kPageTokens || cfg->dk != 128 || cfg->dv != 128)
        return fail(RL_ERR_UNSUPPORTED, "shapes: head_dim 256, page_tokens 64, dk = dv = 128 only");
    if (cfg->kv_dtype != RL_KV_F16 && cfg->kv_dtype != RL_KV_Q8K_TQ3V) return fail(RL_ERR_UNSUPPORTED, "kv_dtype %d unknown", cfg->kv_dtype);
    const bool compact = cfg->kv_dtype == RL_KV_Q8K_TQ3V;
    if (compact && ((cfg->wht_len != 128 && cfg->wht_len != 256) || cfg->window_tokens < 0 ||
                    cfg->window_tokens > cfg->max_pages_per_seq * cfg->page_tokens || (cfg->wht_len == 256 && !cfg->tq_signs)))
        return fail(RL_ERR_RANGE, "compact cache: wht_len %d (128 or 256, 256 with tq_signs), window_tokens %d within the context",
                    cfg->wht_len, cfg->window_tokens);
    if (cfg->conv_k != 4) return fail(RL_ERR_UNSUPPORTED, "conv_k %d: the cache keeps 4-tap ring windows", cfg->conv_k);
    if (cfg->n_slots <= 0 || cfg->max_batch <= 0 || cfg->n_pages <= 0 || cfg->max_pages_per_seq <= 0 ||
        cfg->n_k <= 0 || cfg->n_v % cfg->n_k)
        return fail(RL_ERR_RANGE, "bad cache sizes");
    DevInfo* d;
    if (int st = dev_info(&d)) return st;
    rl_cache* c = new (std::nothrow) rl_cache();
    if (!c) return fail(RL_ERR_NOMEM, "host allocation failed");
    c->cfg = *cfg;
    c->types.assign(cfg->layer_types, cfg->layer_types + cfg->n_layers);
    c->cfg.layer_types = c->types.data();
    for (int t : c->types) (t == RL_LAYER_FULL_ATTENTION ? c->n_attn : c->n_delta)++;
    c->conv_dim = 2 * cfg->n_k * cfg->dk + cfg->n_v * cfg->dv;
    c->dev_err = d->err_ptr;
    c->cfg.tq_signs = nullptr;                 // the host vector is copied below, not kept
    if (!compact) c->cfg.wht_len = c->cfg.window_tokens = 0;
    c->pool_elems = compact ? 0 : size_t(cfg->n_pages) * cfg->n_kv * rl::kv_slice_elems();
    c->cpool_bytes = compact ? size_t(cfg->n_pages) * cfg->n_kv * rl_kv_compact_page_bytes() : 0;
    c->win_pages = compact ? ceil_div(cfg->window_tokens, cfg->page_tokens) : 0;
    c->wpool_elems = size_t(cfg->n_slots) * c->win_pages * cfg->n_kv * rl::kv_slice_elems();
    const rl_attn_decode_params ap = c->attn_params(cfg->max_batch);
    if (int st = attn_check(&ap)) {
        delete c;
        return st;
    }
    c->attn_ws_bytes = attn_plan(&ap, d->sms).total_bytes;
    if (c->win_pages) {
        const rl_attn_decode_params wp = c->window_params(cfg->max_batch);
        c->attn_ws_bytes = std::max(c->attn_ws_bytes, attn_plan(&wp, d->sms).total_bytes);
    }
    int st = RL_OK;
    if (!st) st = dev_alloc(&c->kv, size_t(c->n_attn) * 2 * c->pool_elems, &c->bytes);
    if (!st && compact) {
        st = dev_alloc(&c->kvc, size_t(c->n_attn) * c->cpool_bytes, &c->bytes);
        if (!st) st = dev_alloc(&c->kvw, size_t(c->n_attn) * 2 * c->wpool_elems, &c->bytes);
        if (!st) st = dev_alloc(&c->win_table, size_t(cfg->n_slots) * c->win_pages, &c->bytes);
        if (!st) st = dev_alloc(&c->win_rows, size_t(cfg->max_batch) * c->win_pages, &c->bytes);
        if (!st) st = dev_alloc(&c->scratch, 2 * size_t(cfg->max_pages_per_seq) * cfg->n_kv * rl::kv_slice_elems(), &c->bytes);
        if (!st) st = dev_alloc(&c->scratch_table, size_t(cfg->max_pages_per_seq), &c->bytes);
        if (!st && cfg->wht_len == 256) {
            st = dev_alloc(&c->d_signs, 256, &c->bytes);
            if (!st && cudaMemcpy(c->d_signs, cfg->tq_signs, 256 * sizeof(float), cudaMemcpyHostToDevice) != cudaSuccess)
                st = fail(RL_ERR_DEVICE, "copying the sign vector failed");
        }
        if (!st) {
            // identity tables: window pages by slot, scratch pages in order
            std::vector<int32_t> ids(std::max(size_t(cfg->n_slots) * c->win_pages, size_t(cfg->max_pages_per_seq)));
            for (size_t i = 0; i < ids.size(); ++i) ids[i] = int32_t(i);
            if ((c->win_table && cudaMemcpy(c->win_table, ids.data(), size_t(cfg->n_slots) * c->win_pages * sizeof(int32_t),
                                            cudaMemcpyHostToDevice) != cudaSuccess) ||
                cudaMemcpy(c->scratch_table, ids.data(), size_t(cfg->max_pages_per_seq) * sizeof(int32_t),
                           cudaMemcpyHostToDevice) != cudaSuccess)
                st = fail(RL_ERR_DEVICE, "writing the page tables failed");
        }
    }
    if (!st) st = dev_alloc(&c->S, size_t(c->n_delta) * cfg->n_slots * cfg->n_v * cfg->dk * cfg->dv, &c->bytes);
    if (!st) st = dev_alloc(&c->conv, size_t(c->n_delta) * cfg->n_slots * c->conv_dim * cfg->conv_k, &c->bytes);
    if (!st) st = dev_alloc(&c->conv_phase, size_t(c->n_delta) * cfg->n_slots, &c->bytes);
    if (!st && c->n_attn) st = dev_alloc(&c->g_q, size_t(cfg->max_batch) * cfg->n_q * cfg->head_dim, &c->bytes);
    if (!st && c->n_attn) st = dev_alloc(&c->g_gate, size_t(cfg->max_batch) * cfg->n_q * cfg->head_dim, &c->bytes);
    if (!st && c->n_delta) st = dev_alloc(&c->g_beta, size_t(cfg->max_batch) * cfg->n_v, &c->bytes);
    if (!st && c->n_delta) st = dev_alloc(&c->g_g, size_t(cfg->max_batch) * cfg->n_v, &c->bytes);
    if (!st) {
        char* ws = nullptr;
        st = dev_alloc(&ws, c->attn_ws_bytes, &c->bytes);
        c->attn_ws = ws;
    }
    if (!st) st = rl_cache_zero(c, nullptr);
    if (!st && cudaDeviceSynchronize() != cudaSuccess) st = fail(RL_ERR_DEVICE, "zeroing the cache failed");
    if (st) {
        rl_cache_destroy(c);
        return st;
    }
    *out = c;
    return RL_OK;
}

void rl_cache_destroy(rl_cache* c) {
    if (!c) return;
    void* ptrs[] = {c->g_q, c->g_gate, c->g_beta, c->g_g, c->kvc, c->kvw, c->win_table, c->win_rows, c->d_signs, c->scratch, c->scratch_table,
                    c->kv, c->S, c->conv, c->conv_phase, c->attn_ws, c->d_attn_q, c->d_attn_gate, c->d_attn_k,
                    c->d_attn_v, c->d_attn_o, c->d_delta_qkv, c->d_delta_beta, c->d_delta_g, c->d_delta_o,
                    c->d_conv_w, c->d_page_table, c->d_pos, c->d_slot_ids};
    for (void* p : ptrs)
        if (p) cudaFree(p);
    for (cudaEvent_t e : c->ev_in) cudaEventDestroy(e);
    for (cudaEvent_t e : c->ev_out) cudaEventDestroy(e);
    for (cudaEvent_t e : c->tev) cudaEventDestroy(e);
    if (c->gexec) cudaGraphExecDestroy(c->gexec);
    if (c->hexec) cudaGraphExecDestroy(c->hexec);
    for (cudaEvent_t e : {c->ev_fork, c->ev_join_a, c->ev_join_b})
        if (e) cudaEventDestroy(e);
    for (cudaEvent_t e : {c->ev_xfork, c->ev_xjoin})
        if (e) cudaEventDestroy(e);
    if (c->s_comm) cudaStreamDestroy(c->s_comm);
    if (c->s_cap) cudaStreamDestroy(c->s_cap);
    if (c->s_h2d) cudaStreamDestroy(c->s_h2d);
    if (c->s_run) cudaStreamDestroy(c->s_run);
    if (c->s_d2h) cudaStreamDestroy(c->s_d2h);
    delete c;
}

size_t rl_cache_bytes(const rl_cache* c) { return c ? c->bytes : 0; }
void* rl_cache_k_pool(rl_cache* c, int i) {
    if (!c || i < 0 || i >= c->n_attn) return nullptr;
    if (c->compact()) return c->kvc + size_t(i) * c->cpool_bytes;
    return c->kv + (size_t(i) * 2) * c->pool_elems;
}
void* rl_cache_v_pool(rl_cache* c, int i) {
    return (c && !c->compact() && i >= 0 && i < c->n_attn) ? c->kv + (size_t(i) * 2 + 1) * c->pool_elems : nullptr;
}
void* rl_cache_window_k_pool(rl_cache* c, int i) {
    return (c && c->win_pages && i >= 0 && i < c->n_attn) ? c->kvw + (size_t(i) * 2) * c->wpool_elems : nullptr;
}
void* rl_cache_window_v_pool(rl_cache* c, int i) {
    return (c && c->win_pages && i >= 0 && i < c->n_attn) ? c->kvw + (size_t(i) * 2 + 1) * c->wpool_elems : nullptr;
}
float* rl_cache_state(rl_cache* c, int i) {
    return (c && i >= 0 && i < c->n_delta)
               ? c->S + size_t(i) * c->cfg.n_slots * c->cfg.n_v * c->cfg.dk * c->cfg.dv : nullptr;
}
float* rl_cache_conv(rl_cache* c, int i) {
    return (c && i >= 0 && i < c->n_delta)
               ? c->conv + size_t(i) * c->cfg.n_slots * c->conv_dim * c->cfg.conv_k : nullptr;
}

int32_t* rl_cache_conv_phase(rl_cache* c, int i) {
    return (c && i >= 0 && i < c->n_delta) ? c->conv_phase + size_t(i) * c->cfg.n_slots : nullptr;
}

int rl_cache_conv_export(rl_cache* c, int i, float* canon, void* stream) {
    if (!c || i < 0 || i >= c->n_delta) return fail(RL_ERR_RANGE, "no such DeltaNet layer");
    return rl_conv_ring_export(rl_cache_conv(c, i), c->conv_phase + size_t(i) * c->cfg.n_slots, canon, 1, c->cfg.n_slots, -1,
                               c->conv_dim, stream);
}

int rl_cache_conv_import(rl_cache* c, int i, const float* canon, void* stream) {
    if (!c || i < 0 || i >= c->n_delta) return fail(RL_ERR_RANGE, "no such DeltaNet layer");
    return rl_conv_ring_import(rl_cache_conv(c, i), c->conv_phase + size_t(i) * c->cfg.n_slots, canon, 1, c->cfg.n_slots, -1,
                               c->conv_dim, stream);
}

int rl_cache_zero(rl_cache* c, void* stream) {
    if (!c) return fail(RL_ERR_RANGE, "cache is NULL");
    const rl_cache_config& f = c->cfg;
    if (c->kv) RL_CUDA(cudaMemsetAsync(c->kv, 0, size_t(c->n_attn) * 2 * c->pool_elems * sizeof(__half), as_stream(stream)));
    if (c->kvc) RL_CUDA(cudaMemsetAsync(c->kvc, 0, size_t(c->n_attn) * c->cpool_bytes, as_stream(stream)));
    if (c->kvw) RL_CUDA(cudaMemsetAsync(c->kvw, 0, size_t(c->n_attn) * 2 * c->wpool_elems * sizeof(__half), as_stream(stream)));
    if (c->S) RL_CUDA(cudaMemsetAsync(c->S, 0, size_t(c->n_delta) * f.n_slots * f.n_v * f.dk * f.dv * sizeof(float), as_stream(stream)));
    if (c->conv) RL_CUDA(cudaMemsetAsync(c->conv, 0, size_t(c->n_delta) * f.n_slots * c->conv_dim * f.conv_k * sizeof(float), as_stream(stream)));
    if (c->conv_phase) RL_CUDA(cudaMemsetAsync(c->conv_phase, 0, size_t(c->n_delta) * f.n_slots * sizeof(int32_t), as_stream(stream)));
    return RL_OK;
}

int rl_stack_set_timing(rl_cache* c, int enable) {
    if (!c) return fail(RL_ERR_RANGE, "cache is NULL");
    if (enable && c->tev.empty()) {
        c->tev.resize(size_t(c->cfg.n_layers) * 4);
        for (auto& e : c->tev) RL_CUDA(cudaEventCreate(&e));
    }
    c->timing = enable != 0;
    return RL_OK;
}

int rl_stack_timing(rl_cache* c, float* ms) {
    if (!c || !ms) return fail(RL_ERR_RANGE, "NULL argument");
    if (c->tev.empty()) return fail(RL_ERR_RANGE, "timing was never enabled");
    for (int i = 0; i < 5; ++i) ms[i] = 0.f;
    RL_CUDA(cudaEventSynchronize(c->tev[size_t(c->cfg.n_layers - 1) * 4 + 2]));
    for (int L = 0; L < c->cfg.n_layers; ++L) {
        float a = 0.f, b = 0.f;
        RL_CUDA(cudaEventElapsedTime(&a, c->tev[size_t(L) * 4], c->tev[size_t(L) * 4 + 1]));
        RL_CUDA(cudaEventElapsedTime(&b, c->tev[size_t(L) * 4 + 1], c->tev[size_t(L) * 4 + 2]));
        if (c->types[L] == RL_LAYER_FULL_ATTENTION) {
            float m = 0.f;
            RL_CUDA(cudaEventElapsedTime(&m, c->tev[size_t(L) * 4 + 1], c->tev[size_t(L) * 4 + 3]));
            ms[0] += a;       // KV append
            ms[1] += m;       // split-KV decode kernel
            ms[2] += b - m;   // merge + gate
        } else {
            ms[3] += a;       // conv1d update
            ms[4] += b;       // delta rule
        }
    }
    return RL_OK;
}

int rl_stack_launches_per_step(const rl_cache* c) {
    if (!c) return 0;
    // attention layer: append, decode, merge (+ the window append and one row-table kernel per step with a compact cache)
    const int per_attn = 3 + ((c->compact() && c->win_pages) ? 1 : 0);
    return c->n_attn * per_attn + ((c->compact() && c->win_pages && c->n_attn) ? 1 : 0) + c->n_delta + (c->n_delta ? 1 : 0);
}

static bool same_io(const rl_stack_io& k, const rl_stack_io* io) {
    return k.attn_q == io->attn_q && k.attn_gate == io->attn_gate && k.attn_k == io->attn_k &&
           k.attn_v == io->attn_v && k.attn_o == io->attn_o && k.delta_qkv == io->delta_qkv &&
           k.delta_beta == io->delta_beta && k.delta_g == io->delta_g && k.delta_o == io->delta_o &&
           k.conv_w == io->conv_w && k.page_table == io->page_table && k.pos == io->pos &&
           k.slot_ids == io->slot_ids && k.batch == io->batch && k.attn_ml == io->attn_ml &&
           k.no_append == io->no_append && k.kv_window_ok == io->kv_window_ok && (k.glue != nullptr) == (io->glue != nullptr);
}

namespace {

struct StackPrefillPlan {
    rl_attn_prefill_params ap;
    rl_delta_chunk_params dp;
    size_t mixed_bytes, delta_ws, attn_ws, canon_bytes, total;
};

int stack_prefill_plan(const rl_cache* c, int pos0, int T, StackPrefillPlan* pl) {
    if (!c) return fail(RL_ERR_RANGE, "cache is NULL");
    const rl_cache_config& f = c->cfg;
    if (T < 0 || pos0 < 0 || 1LL * pos0 + T > 1LL * f.max_pages_per_seq * f.page_tokens)
        return fail(RL_ERR_RANGE, "pos0 %d + T %d exceeds the page table (%d pages)", pos0, T, f.max_pages_per_seq);
    std::memset(pl, 0, sizeof *pl);
    pl->ap.n_q = f.n_q;
    pl->ap.n_kv = f.n_kv;
    pl->ap.head_dim = f.head_dim;
    pl->ap.seq = T;
    pl->ap.br = 128;
    pl->ap.bc = 64;
    pl->ap.pos0 = pos0;
    pl->ap.page_tokens = f.page_tokens;
    pl->ap.n_pages = f.n_pages;
    pl->ap.n_table = f.max_pages_per_seq;
    pl->dp.n_v = f.n_v;
    pl->dp.dk = f.dk;
    pl->dp.dv = f.dv;
    pl->dp.seq = T;
    pl->dp.chunk = 64;
    pl->dp.eps_l2 = 1e-6f;
    pl->dp.n_qk = f.n_k;
    pl->dp.head_map = f.head_map;
    pl->dp.qk_tok_stride = pl->dp.v_tok_stride = c->conv_dim;
    pl->mixed_bytes = c->n_delta ? align_up(size_t(T) * c->conv_dim * sizeof(float), 256) : 0;
    pl->delta_ws = c->n_delta && T ? align_up(rl_delta_chunk_workspace_bytes(&pl->dp), 256) : 0;
    pl->attn_ws = c->n_attn && T ? align_up(rl_attn_prefill_workspace_bytes(&pl->ap), 256) : 0;
    // the slot's conv windows of every DeltaNet layer in the reference's shifted form, for the chunk
    pl->canon_bytes = c->n_delta ? align_up(size_t(c->n_delta) * c->conv_dim * f.conv_k * sizeof(float), 256) : 0;
    pl->total = pl->mixed_bytes + pl->delta_ws + pl->attn_ws + pl->canon_bytes;
    return RL_OK;
}

}  // namespace

size_t rl_stack_prefill_workspace_bytes(const rl_cache* c, int pos0, int T) {
    StackPrefillPlan pl;
    if (stack_prefill_plan(c, pos0, T, &pl)) return 0;
    return pl.total;
}

int rl_stack_prefill(rl_cache* c, const rl_stack_prefill_io* io, void* workspace, size_t workspace_bytes, void* stream) {
    if (!c || !io) return fail(RL_ERR_RANGE, "NULL argument");
    StackPrefillPlan pl;
    if (int st = stack_prefill_plan(c, io->pos0, io->T, &pl)) return st;
    const rl_cache_config& f = c->cfg;
    if (io->slot < 0 || io->slot >= f.n_slots) return fail(RL_ERR_RANGE, "slot %d outside [0, %d)", io->slot, f.n_slots);
    if (io->T == 0) return RL_OK;
    if (!io->page_table_row && c->n_attn) return fail(RL_ERR_RANGE, "page_table_row is NULL");
    if (c->n_attn && (!io->attn_q || !io->attn_k || !io->attn_v || !io->attn_o)) return fail(RL_ERR_RANGE, "attention tensors are NULL");
    if (c->n_delta && (!io->delta_qkv || !io->delta_beta || !io->delta_g || !io->delta_o || !io->conv_w))
        return fail(RL_ERR_RANGE, "DeltaNet tensors are NULL");
    if (workspace_bytes < pl.total || (pl.total && !workspace))
        return fail(RL_ERR_RANGE, "workspace %zu bytes < %zu required", workspace_bytes, pl.total);
    // the chunk's kernels that wait for the kernel in front themselves (launch_step) overlap their heads with its tail
    StepOverlap overlap(true);
    if (reinterpret_cast<uintptr_t>(workspace) % 256) return fail(RL_ERR_RANGE, "workspace must be 256-byte aligned");
    cudaStream_t run = as_stream(stream);
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    float* mixed = reinterpret_cast<float*>(ws);
    void* delta_ws = ws + pl.mixed_bytes;
    void* attn_ws = ws + pl.mixed_bytes + pl.delta_ws;
    float* canon = reinterpret_cast<float*>(ws + pl.mixed_bytes + pl.delta_ws + pl.attn_ws);
    const int T = io->T;
    const size_t q_sz = size_t(T) * f.n_q * f.head_dim, kv_sz = size_t(T) * f.n_kv * f.head_dim;
    const size_t qkv_sz = size_t(T) * c->conv_dim, hv_sz = size_t(T) * f.n_v, do_sz = size_t(T) * f.n_v * f.dv;
    const size_t slot_S = size_t(f.n_v) * f.dk * f.dv, slot_cv = size_t(c->conv_dim) * f.conv_k;
    const size_t st_elems = size_t(f.n_slots) * slot_S, cv_elems = size_t(f.n_slots) * slot_cv;
    const uint16_t* aq = static_cast<const uint16_t*>(io->attn_q);
    const uint16_t* ak = static_cast<const uint16_t*>(io->attn_k);
    const uint16_t* av = static_cast<const uint16_t*>(io->attn_v);
    int ai = 0, di = 0;
    // a later chunk starts from the windows the previous chunk (or decode steps) left in the rings
    if (c->n_delta && io->pos0 > 0)
        rl::launch_conv_ring_export(c->conv, c->conv_phase, canon, c->n_delta, f.n_slots, io->slot, c->conv_dim, run);
    for (int L = 0; L < f.n_layers; ++L) {
        if (c->types[L] == RL_LAYER_FULL_ATTENTION) {
            const float* gate_l = io->attn_gate ? io->attn_gate + ai * q_sz : nullptr;
            if (!c->compact()) {
                if (int st = attn_prefill_impl(rl_cache_k_pool(c, ai), rl_cache_v_pool(c, ai), io->page_table_row, aq + ai * q_sz,
                                               ak + ai * kv_sz, av + ai * kv_sz, gate_l, io->attn_o + ai * q_sz,
                                               pl.attn_ws ? attn_ws : nullptr, pl.attn_ws, &pl.ap, run))
                    return st;
            } else {
                // the chunk's rows persist in the compact pages; it attends over the F16 window when it ends
                // inside it, else over F16 scratch pages rebuilt from the compact pages
                rl_kv_append_params cp;
                std::memset(&cp, 0, sizeof cp);
                cp.n_kv = f.n_kv, cp.head_dim = f.head_dim, cp.batch = 1, cp.n_tok = T, cp.page_tokens = f.page_tokens;
                cp.n_pages = f.n_pages, cp.max_pages_per_seq = f.max_pages_per_seq, cp.pos0 = io->pos0, cp.rows_fp16 = 2;
                cp.wht_len = f.wht_len;
                if (int st = rl_kv_compact_append(rl_cache_k_pool(c, ai), io->page_table_row, nullptr, ak + ai * kv_sz,
                                                  av + ai * kv_sz, c->d_signs, &cp, run))
                    return st;
                rl_attn_prefill_params ap = pl.ap;
                if (io->pos0 + T <= f.window_tokens) {
                    ap.n_pages = f.n_slots * c->win_pages;
                    ap.n_table = c->win_pages;
                    if (int st = attn_prefill_impl(rl_cache_window_k_pool(c, ai), rl_cache_window_v_pool(c, ai),
                                                   c->win_table + size_t(io->slot) * c->win_pages, aq + ai * q_sz, ak + ai * kv_sz,
                                                   av + ai * kv_sz, gate_l, io->attn_o + ai * q_sz,
                                                   pl.attn_ws ? attn_ws : nullptr, pl.attn_ws, &ap, run))
                        return st;
                } else {
                    __half* sk = c->scratch;
                    __half* sv = c->scratch + size_t(f.max_pages_per_seq) * f.n_kv * rl::kv_slice_elems();
                    if (int st = rl_kv_compact_to_f16(rl_cache_k_pool(c, ai), io->page_table_row, 0, f.n_pages, sk, sv,
                                                      c->scratch_table, 0, f.max_pages_per_seq, io->pos0 + T, f.n_kv, f.wht_len,
                                                      c->d_signs, run))
                        return st;
                    ap.n_pages = f.max_pages_per_seq;
                    if (int st = attn_prefill_impl(sk, sv, c->scratch_table, aq + ai * q_sz, nullptr, nullptr, gate_l,
                                                   io->attn_o + ai * q_sz, pl.attn_ws ? attn_ws : nullptr, pl.attn_ws, &ap, run))
                        return st;
                }
            }
            ++ai;
        } else {
            float* S = c->S + di * st_elems + io->slot * slot_S;
            float* cv = canon + size_t(di) * slot_cv;
            // a sequence that starts here starts from a zero state and an empty conv window
            if (io->pos0 == 0) RL_CUDA(cudaMemsetAsync(S, 0, slot_S * sizeof(float), run));
            rl_conv1d_params cp;
            cp.dim = c->conv_dim;
            cp.k = f.conv_k;
            cp.silu = 1;
            cp.batch = 1;
            cp.n_slots = 1;
            if (int st = rl_conv1d_causal(io->delta_qkv + di * qkv_sz, io->conv_w + size_t(di) * slot_cv, mixed, cv, T, &cp,
                                          io->pos0 > 0, run))
                return st;
            if (int st = rl_delta_chunk_prefill(S, mixed, mixed + size_t(f.n_k) * f.dk, mixed + 2 * size_t(f.n_k) * f.dk,
                                                io->delta_beta + di * hv_sz, io->delta_g + di * hv_sz, io->delta_o + di * do_sz,
                                                delta_ws, pl.delta_ws, &pl.dp, run))
                return st;
            ++di;
        }
    }
    if (c->n_delta) {
        rl::launch_conv_ring_import(c->conv, c->conv_phase, canon, c->n_delta, f.n_slots, io->slot, c->conv_dim, run);
        RL_CUDA(cudaGetLastError());
    }
    return RL_OK;
}

size_t rl_cache_delta_prefill_workspace_bytes(const rl_cache* c, int T) {
    StackPrefillPlan pl;
    if (!c || !c->n_delta || stack_prefill_plan(c, 0, T, &pl)) return 0;
    return pl.mixed_bytes + pl.delta_ws + align_up(size_t(c->conv_dim) * c->cfg.conv_k * sizeof(float), 256);
}

int rl_cache_delta_prefill(rl_cache* c, int di, int slot, int pos0, int T, const float* qkv, const float* conv_w,
                           const float* beta, const float* g_log, float* o, void* workspace, size_t workspace_bytes,
                           void* stream) {
    if (!c || di < 0 || di >= c->n_delta) return fail(RL_ERR_RANGE, "no such DeltaNet layer");
    StackPrefillPlan pl;
    if (int st = stack_prefill_plan(c, pos0, T, &pl)) return st;
    const rl_cache_config& f = c->cfg;
    if (slot < 0 || slot >= f.n_slots) return fail(RL_ERR_RANGE, "slot %d outside [0, %d)", slot, f.n_slots);
    if (T == 0) return RL_OK;
    if (!qkv || !conv_w || !beta || !g_log || !o || !workspace) return fail(RL_ERR_RANGE, "NULL pointer argument");
    const size_t need = rl_cache_delta_prefill_workspace_bytes(c, T);
    if (workspace_bytes < need) return fail(RL_ERR_RANGE, "workspace %zu bytes < %zu required", workspace_bytes, need);
    if (reinterpret_cast<uintptr_t>(workspace) % 256) return fail(RL_ERR_RANGE, "workspace must be 256-byte aligned");
    cudaStream_t run = as_stream(stream);
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    float* mixed = reinterpret_cast<float*>(ws);
    void* delta_ws = ws + pl.mixed_bytes;
    float* canon = reinterpret_cast<float*>(ws + pl.mixed_bytes + pl.delta_ws);
    const size_t slot_S = size_t(f.n_v) * f.dk * f.dv;
    float* S = rl_cache_state(c, di) + size_t(slot) * slot_S;
    float* ring = rl_cache_conv(c, di);
    int32_t* phase = rl_cache_conv_phase(c, di);
    if (pos0 == 0) RL_CUDA(cudaMemsetAsync(S, 0, slot_S * sizeof(float), run));
    else rl::launch_conv_ring_export(ring, phase, canon, 1, f.n_slots, slot, c->conv_dim, run);
    rl_conv1d_params cp;
    cp.dim = c->conv_dim;
    cp.k = f.conv_k;
    cp.silu = 1;
    cp.batch = 1;
    cp.n_slots = 1;
    if (int st = rl_conv1d_causal(qkv, conv_w, mixed, canon, T, &cp, pos0 > 0, run)) return st;
    if (int st = rl_delta_chunk_prefill(S, mixed, mixed + size_t(f.n_k) * f.dk, mixed + 2 * size_t(f.n_k) * f.dk, beta, g_log,
                                        o, delta_ws, pl.delta_ws, &pl.dp, run))
        return st;
    rl::launch_conv_ring_import(ring, phase, canon, 1, f.n_slots, slot, c->conv_dim, run);
    RL_CUDA(cudaGetLastError());
    return RL_OK;
}

int rl_stack_decode(rl_cache* c, const rl_stack_io* io, void* stream) {
    if (!c || !io) return fail(RL_ERR_RANGE, "NULL argument");
    if (io->batch < 0 || io->batch > c->cfg.max_batch)
        return fail(RL_ERR_RANGE, "batch %d outside [0, max_batch %d]", io->batch, c->cfg.max_batch);
    if (io->batch == 0) return RL_OK;
    const rl_stack_glue* gl = io->glue;
    if ((c->n_attn && (!(gl ? (const void*)gl->attn_qg : (const void*)io->attn_q) || !io->attn_o || !io->page_table || !io->pos ||
                       (!io->no_append && (!(gl ? (const void*)gl->attn_k_raw : (const void*)io->attn_k) || !io->attn_v)))) ||
        (c->n_delta && (!io->delta_qkv || !io->delta_o || !io->conv_w ||
                        (gl ? (!gl->delta_a || !gl->delta_b || !gl->A_log || !gl->dt_bias) : (!io->delta_beta || !io->delta_g)))))
        return fail(RL_ERR_RANGE, "NULL tensor in rl_stack_io");
    if (c->compact() && io->attn_ml) return fail(RL_ERR_UNSUPPORTED, "split-KV partials over the compact cache are offered by rl_attn_decode_partial only");
    if (c->gather.comm && io->attn_ml && c->n_attn && (!c->gather.attn_ml_all || !c->gather.attn_o_final))
        return fail(RL_ERR_RANGE, "split-KV partials need attn_ml_all and attn_o_final in rl_stack_gather");
    if (!c->graph_enabled || c->timing) return stack_decode_layers(c, io, as_stream(stream), false);
    const bool same = c->gkey_seen > 0 && same_io(c->gkey, io) &&
                      (!io->glue || std::memcmp(&c->gglue, io->glue, sizeof(rl_stack_glue)) == 0);
    if (same && c->gkey_seen == 2) {
        RL_CUDA(cudaGraphLaunch(c->gexec, as_stream(stream)));
        return RL_OK;
    }
    if (io->glue) c->gglue = *io->glue;
    if (!same) {
        // first step with this io: run it eagerly (also finishes every lazy set-up outside capture)
        if (c->gexec) {
            cudaGraphExecDestroy(c->gexec);
            c->gexec = nullptr;
        }
        c->gkey = *io;
        c->gkey_seen = 1;
        return stack_decode_layers(c, io, as_stream(stream), false);
    }
    // second step with the same io: capture on an internal stream, then replay on the caller's
    if (!c->s_cap) RL_CUDA(cudaStreamCreateWithFlags(&c->s_cap, cudaStreamNonBlocking));
    cudaGraph_t graph = nullptr;
    if (cudaStreamBeginCapture(c->s_cap, cudaStreamCaptureModeRelaxed) == cudaSuccess) {
        const int st = stack_decode_layers(c, io, c->s_cap, false);
        const cudaError_t ce = cudaStreamEndCapture(c->s_cap, &graph);
        if (st == RL_OK && ce == cudaSuccess && graph &&
            cudaGraphInstantiate(&c->gexec, graph, 0) == cudaSuccess) {
            cudaGraphDestroy(graph);
            c->gkey_seen = 2;
            RL_CUDA(cudaGraphLaunch(c->gexec, as_stream(stream)));
            return RL_OK;
        }
        if (graph) cudaGraphDestroy(graph);
    }
    cudaGetLastError();
    c->gexec = nullptr;
    c->graph_enabled = false;       // capture is not possible here: stay on plain launches
    return stack_decode_layers(c, io, as_stream(stream), false);
}

int rl_comm_unique_id(void* id) {
    if (!id) return fail(RL_ERR_RANGE, "id is NULL");
    if (rl::comm_unique_id(id)) return fail(RL_ERR_UNSUPPORTED, "%s", rl::comm_last_error());
    return RL_OK;
}

int rl_comm_create(const void* id, int rank, int n_ranks, rl_comm** out) {
    if (!id || !out) return fail(RL_ERR_RANGE, "NULL argument");
    *out = nullptr;
    if (n_ranks < 1 || rank < 0 || rank >= n_ranks) return fail(RL_ERR_RANGE, "rank %d outside [0, %d)", rank, n_ranks);
    DevInfo* d;
    if (int st = dev_info(&d)) return st;
    rl::Comm* c = nullptr;
    if (rl::comm_create(id, rank, n_ranks, &c)) return fail(RL_ERR_DEVICE, "%s", rl::comm_last_error());
    *out = reinterpret_cast<rl_comm*>(c);
    return RL_OK;
}

void rl_comm_destroy(rl_comm* comm) { rl::comm_destroy(reinterpret_cast<rl::Comm*>(comm)); }

int rl_stack_set_gather(rl_cache* c, const rl_stack_gather* g) {
    if (!c) return fail(RL_ERR_RANGE, "cache is NULL");
    if (g && g->comm) {
        if ((c->n_attn && !g->attn_o_all) || (c->n_delta && !g->delta_o_all))
            return fail(RL_ERR_RANGE, "gather buffers are NULL");
        if (g->layers_per_exchange < 0) return fail(RL_ERR_RANGE, "layers_per_exchange %d", g->layers_per_exchange);
        if (g->reserve_sms < 0 || g->reserve_sms > 64) return fail(RL_ERR_RANGE, "reserve_sms %d outside [0, 64]", g->reserve_sms);
        if (!c->s_comm) {
            int lo = 0, hi = 0;
            RL_CUDA(cudaDeviceGetStreamPriorityRange(&lo, &hi));
            RL_CUDA(cudaStreamCreateWithPriority(&c->s_comm, cudaStreamNonBlocking, hi));
            RL_CUDA(cudaEventCreateWithFlags(&c->ev_xfork, cudaEventDisableTiming));
            RL_CUDA(cudaEventCreateWithFlags(&c->ev_xjoin, cudaEventDisableTiming));
        }
        c->gather = *g;
    } else {
        c->gather = rl_stack_gather{};
    }
    // a captured step holds the old setting: start over
    if (c->gexec) {
        cudaGraphExecDestroy(c->gexec);
        c->gexec = nullptr;
    }
    if (c->hexec) {
        cudaGraphExecDestroy(c->hexec);
        c->hexec = nullptr;
    }
    c->gkey_seen = c->hkey_seen = 0;
    return RL_OK;
}

int rl_stack_set_graph(rl_cache* c, int enable) {
    if (!c) return fail(RL_ERR_RANGE, "cache is NULL");
    c->graph_enabled = enable != 0;
    if (!enable && c->gexec) {
        cudaGraphExecDestroy(c->gexec);
        c->gexec = nullptr;
    }
    if (!enable) c->gkey_seen = 0;
    return RL_OK;
}

static int ensure_staging(rl_cache* c) {
    if (c->staging) return RL_OK;
    const rl_cache_config& f = c->cfg;
    const size_t B = f.max_batch;
    size_t unused = 0;
    int st = RL_OK;
    const size_t q_sz = size_t(c->n_attn) * B * f.n_q * f.head_dim, kv_sz = size_t(c->n_attn) * B * f.n_kv * f.head_dim;
    if (!st) st = dev_alloc(&c->d_attn_q, q_sz, &unused);
    if (!st) st = dev_alloc(&c->d_attn_gate, q_sz, &unused);
    if (!st) st = dev_alloc(&c->d_attn_o, q_sz, &unused);
    if (!st) st = dev_alloc(&c->d_attn_k, kv_sz, &unused);
    if (!st) st = dev_alloc(&c->d_attn_v, kv_sz, &unused);
    if (!st) st = dev_alloc(&c->d_delta_qkv, size_t(c->n_delta) * B * c->conv_dim, &unused);
    if (!st) st = dev_alloc(&c->d_delta_beta, size_t(c->n_delta) * B * f.n_v, &unused);
    if (!st) st = dev_alloc(&c->d_delta_g, size_t(c->n_delta) * B * f.n_v, &unused);
    if (!st) st = dev_alloc(&c->d_delta_o, size_t(c->n_delta) * B * f.n_v * f.dv, &unused);
    if (!st && !c->d_conv_w) st = dev_alloc(&c->d_conv_w, size_t(c->n_delta) * c->conv_dim * f.conv_k, &unused);
    if (!st) st = dev_alloc(&c->d_page_table, B * f.max_pages_per_seq, &unused);
    if (!st) st = dev_alloc(&c->d_pos, B, &unused);
    if (!st) st = dev_alloc(&c->d_slot_ids, B, &unused);
    if (st) return st;
    c->bytes += unused;
    RL_CUDA(cudaStreamCreateWithFlags(&c->s_h2d, cudaStreamNonBlocking));
    RL_CUDA(cudaStreamCreateWithFlags(&c->s_run, cudaStreamNonBlocking));
    RL_CUDA(cudaStreamCreateWithFlags(&c->s_d2h, cudaStreamNonBlocking));
    c->ev_in.resize(f.n_layers);
    c->ev_out.resize(f.n_layers);
    for (int i = 0; i < f.n_layers; ++i) {
        RL_CUDA(cudaEventCreateWithFlags(&c->ev_in[i], cudaEventDisableTiming));
        RL_CUDA(cudaEventCreateWithFlags(&c->ev_out[i], cudaEventDisableTiming));
    }
    c->staging = true;
    return RL_OK;
}

int rl_stack_set_conv_w(rl_cache* c, const float* host_conv_w) {
    if (!c || !host_conv_w) return fail(RL_ERR_RANGE, "NULL argument");
    const size_t n = size_t(c->n_delta) * c->conv_dim * c->cfg.conv_k;
    if (!c->d_conv_w) {
        size_t t = 0;
        if (int st = dev_alloc(&c->d_conv_w, n, &t)) return st;
        c->bytes += t;
    }
    RL_CUDA(cudaMemcpy(c->d_conv_w, host_conv_w, n * sizeof(float), cudaMemcpyHostToDevice));
    return RL_OK;
}

// everything rl_stack_decode_host enqueues (copies in, layers, copies out), without waiting
static int host_step_enqueue(rl_cache* c, const rl_stack_io* h) {
    const rl_cache_config& f = c->cfg;
    const size_t B = h->batch;
    const size_t q_sz = B * f.n_q * f.head_dim, kv_sz = B * f.n_kv * f.head_dim;
    const size_t qkv_sz = B * c->conv_dim, hv_sz = B * f.n_v, do_sz = B * f.n_v * f.dv;
    const cudaMemcpyKind H2D = cudaMemcpyHostToDevice, D2H = cudaMemcpyDeviceToHost;
    RL_CUDA(cudaMemcpyAsync(c->d_page_table, h->page_table, B * f.max_pages_per_seq * sizeof(int32_t), H2D, c->s_h2d));
    RL_CUDA(cudaMemcpyAsync(c->d_pos, h->pos, B * sizeof(int32_t), H2D, c->s_h2d));
    if (h->slot_ids) RL_CUDA(cudaMemcpyAsync(c->d_slot_ids, h->slot_ids, B * sizeof(int32_t), H2D, c->s_h2d));
    int ai = 0, di = 0;
    for (int L = 0; L < f.n_layers; ++L) {
        if (c->types[L] == RL_LAYER_FULL_ATTENTION) {
            RL_CUDA(cudaMemcpyAsync(c->d_attn_q + ai * q_sz, h->attn_q + ai * q_sz, q_sz * 4, H2D, c->s_h2d));
            if (h->attn_gate)
                RL_CUDA(cudaMemcpyAsync(c->d_attn_gate + ai * q_sz, h->attn_gate + ai * q_sz, q_sz * 4, H2D, c->s_h2d));
            RL_CUDA(cudaMemcpyAsync(c->d_attn_k + ai * kv_sz, h->attn_k + ai * kv_sz, kv_sz * 4, H2D, c->s_h2d));
            RL_CUDA(cudaMemcpyAsync(c->d_attn_v + ai * kv_sz, h->attn_v + ai * kv_sz, kv_sz * 4, H2D, c->s_h2d));
            ++ai;
        } else {
            RL_CUDA(cudaMemcpyAsync(c->d_delta_qkv + di * qkv_sz, h->delta_qkv + di * qkv_sz, qkv_sz * 4, H2D, c->s_h2d));
            RL_CUDA(cudaMemcpyAsync(c->d_delta_beta + di * hv_sz, h->delta_beta + di * hv_sz, hv_sz * 4, H2D, c->s_h2d));
            RL_CUDA(cudaMemcpyAsync(c->d_delta_g + di * hv_sz, h->delta_g + di * hv_sz, hv_sz * 4, H2D, c->s_h2d));
            ++di;
        }
        if ((L + 1) % kHostGroup == 0 || L + 1 == f.n_layers) RL_CUDA(cudaEventRecord(c->ev_in[L], c->s_h2d));
    }
    rl_stack_io d = *h;
    d.attn_q = c->d_attn_q;
    d.attn_gate = h->attn_gate ? c->d_attn_gate : nullptr;
    d.attn_k = c->d_attn_k;
    d.attn_v = c->d_attn_v;
    d.attn_o = c->d_attn_o;
    d.delta_qkv = c->d_delta_qkv;
    d.delta_beta = c->d_delta_beta;
    d.delta_g = c->d_delta_g;
    d.delta_o = c->d_delta_o;
    d.conv_w = c->d_conv_w;
    d.page_table = c->d_page_table;
    d.pos = c->d_pos;
    d.slot_ids = h->slot_ids ? c->d_slot_ids : nullptr;
    if (int st = stack_decode_layers(c, &d, c->s_run, true)) return st;
    ai = di = 0;
    for (int L = 0; L < f.n_layers; ++L) {
        if (L % kHostGroup == 0)
            RL_CUDA(cudaStreamWaitEvent(c->s_d2h, c->ev_out[std::min(L + kHostGroup, f.n_layers) - 1], 0));
        if (c->types[L] == RL_LAYER_FULL_ATTENTION) {
            RL_CUDA(cudaMemcpyAsync(h->attn_o + ai * q_sz, c->d_attn_o + ai * q_sz, q_sz * 4, D2H, c->s_d2h));
            ++ai;
        } else {
            RL_CUDA(cudaMemcpyAsync(h->delta_o + di * do_sz, c->d_delta_o + di * do_sz, do_sz * 4, D2H, c->s_d2h));
            ++di;
        }
    }
    return RL_OK;
}

int rl_stack_decode_host(rl_cache* c, const rl_stack_io* h) {
    if (!c || !h) return fail(RL_ERR_RANGE, "NULL argument");
    if (h->batch < 0 || h->batch > c->cfg.max_batch)
        return fail(RL_ERR_RANGE, "batch %d outside [0, max_batch %d]", h->batch, c->cfg.max_batch);
    if (h->batch == 0) return RL_OK;
    if ((c->n_attn && (!h->attn_q || !h->attn_k || !h->attn_v || !h->attn_o || !h->page_table || !h->pos)) ||
        (c->n_delta && (!h->delta_qkv || !h->delta_beta || !h->delta_g || !h->delta_o)))
        return fail(RL_ERR_RANGE, "NULL tensor in rl_stack_io");
    if (h->attn_ml || h->no_append || h->glue)
        return fail(RL_ERR_UNSUPPORTED, "split-KV partials and the fused element-wise steps are offered by rl_stack_decode (device pointers) only");
    if (c->n_delta && !c->d_conv_w) return fail(RL_ERR_RANGE, "call rl_stack_set_conv_w first");
    if (int st = ensure_staging(c)) return st;
    if (c->graph_enabled && !c->timing && !c->host_graph_failed) {
        const bool same = c->hkey_seen > 0 && same_io(c->hkey, h);
        if (same && c->hkey_seen == 2) {
            RL_CUDA(cudaGraphLaunch(c->hexec, c->s_run));
            RL_CUDA(cudaStreamSynchronize(c->s_run));
            return RL_OK;
        }
        if (!same) {
            if (c->hexec) {
                cudaGraphExecDestroy(c->hexec);
                c->hexec = nullptr;
            }
            c->hkey = *h;
            c->hkey_seen = 1;                     // this call runs as plain launches
        } else {
            // second call with the same host buffers: capture the three streams as one graph
            if (!c->ev_fork) {
                RL_CUDA(cudaEventCreateWithFlags(&c->ev_fork, cudaEventDisableTiming));
                RL_CUDA(cudaEventCreateWithFlags(&c->ev_join_a, cudaEventDisableTiming));
                RL_CUDA(cudaEventCreateWithFlags(&c->ev_join_b, cudaEventDisableTiming));
            }
            cudaGraph_t graph = nullptr;
            bool ok = cudaStreamBeginCapture(c->s_run, cudaStreamCaptureModeRelaxed) == cudaSuccess;
            if (ok) {
                ok = cudaEventRecord(c->ev_fork, c->s_run) == cudaSuccess &&
                     cudaStreamWaitEvent(c->s_h2d, c->ev_fork, 0) == cudaSuccess &&
                     cudaStreamWaitEvent(c->s_d2h, c->ev_fork, 0) == cudaSuccess;
                ok = ok && host_step_enqueue(c, h) == RL_OK;
                ok = ok && cudaEventRecord(c->ev_join_a, c->s_h2d) == cudaSuccess &&
                     cudaStreamWaitEvent(c->s_run, c->ev_join_a, 0) == cudaSuccess &&
                     cudaEventRecord(c->ev_join_b, c->s_d2h) == cudaSuccess &&
                     cudaStreamWaitEvent(c->s_run, c->ev_join_b, 0) == cudaSuccess;
                const cudaError_t ce = cudaStreamEndCapture(c->s_run, &graph);
                ok = ok && ce == cudaSuccess && graph &&
                     cudaGraphInstantiate(&c->hexec, graph, 0) == cudaSuccess;
                if (graph) cudaGraphDestroy(graph);
            }
            cudaGetLastError();
            if (ok) {
                c->hkey_seen = 2;
                RL_CUDA(cudaGraphLaunch(c->hexec, c->s_run));
                RL_CUDA(cudaStreamSynchronize(c->s_run));
                return RL_OK;
            }
            c->hexec = nullptr;
            c->host_graph_failed = true;          // e.g. pageable host memory: stay on plain launches
        }
    }
    if (int st = host_step_enqueue(c, h)) return st;
    RL_CUDA(cudaStreamSynchronize(c->s_d2h));
    RL_CUDA(cudaStreamSynchronize(c->s_run));
    return RL_OK;
}

}  // extern "C"
