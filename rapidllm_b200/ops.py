"""Operator-level mirror of rapidllm::ops for torch CUDA tensors.

Same names and argument meaning as include/rapidllm/kernels/ops.h:118-131;
every function enqueues on the current torch stream through the C ABI and
raises RlError on a bad argument.  No CPU path exists here.
"""
from __future__ import annotations

import ctypes as C
import functools

import torch

from . import _lib
from ._lib import (AttnDecodeParams, AttnPrefillParams, Conv1dParams, DeltaChunkParams,
                   DeltaRecurrentParams, KvAppendParams, check, lib)

PAGE_TOKENS = 64
HEAD_DIM = 256


def _stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _p(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _need(t, dtype, name):
    if t is None:
        return
    if not (t.is_cuda and t.dtype == dtype and t.is_contiguous()):
        raise _lib.RlError(6, f"{name}: need a contiguous CUDA tensor of {dtype}")


def kv_slice_index(tok: torch.Tensor, d: torch.Tensor) -> torch.Tensor:
    """Offset (in halves) of element (tok, d) inside one (page, head) slice."""
    sub = d >> 6
    chunk = ((d & 63) >> 3) ^ (tok & 7)
    return sub * (PAGE_TOKENS * 64) + tok * 64 + chunk * 8 + (d & 7)


def new_pool(n_pages: int, n_kv: int, device="cuda") -> torch.Tensor:
    """A zeroed fp16 pool [n_pages][n_kv][64*256] for K or V."""
    return torch.zeros(n_pages, n_kv, PAGE_TOKENS * HEAD_DIM, dtype=torch.float16, device=device)


def kv_append(k_pool, v_pool, page_table, k_rows, v_rows, pos=None, pos0=0):
    """Write rows [batch][n_tok][n_kv][256] (fp32 -> fp16 RNE, or fp16) at pos[b] (+0..n_tok-1)."""
    n_pages, n_kv = k_pool.shape[0], k_pool.shape[1]
    if k_rows.dim() == 3:
        k_rows, v_rows = k_rows.unsqueeze(0), v_rows.unsqueeze(0)
    if page_table.dim() == 1:
        page_table = page_table.unsqueeze(0)
    kind = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}.get(k_rows.dtype)
    if kind is None:
        raise _lib.RlError(6, "k_rows: need fp32, fp16 or bf16")
    _need(k_rows, k_rows.dtype, "k_rows")
    _need(v_rows, k_rows.dtype, "v_rows")
    _need(page_table, torch.int32, "page_table")
    _need(pos, torch.int32, "pos")
    p = KvAppendParams(n_kv=n_kv, head_dim=HEAD_DIM, batch=k_rows.shape[0], n_tok=k_rows.shape[1],
                       page_tokens=PAGE_TOKENS, n_pages=n_pages,
                       max_pages_per_seq=page_table.shape[1], pos0=pos0, rows_fp16=kind)
    check(lib().rl_kv_append(_p(k_pool), _p(v_pool), _p(page_table), _p(pos), _p(k_rows),
                             _p(v_rows), C.byref(p), _stream()))


def kv_gather(pool, page_table_row, n_tok):
    """Tokens [0, n_tok) of one sequence as contiguous fp16 [n_tok][n_kv][256]."""
    n_pages, n_kv = pool.shape[0], pool.shape[1]
    _need(page_table_row, torch.int32, "page_table_row")
    out = torch.empty(n_tok, n_kv, HEAD_DIM, dtype=torch.float16, device=pool.device)
    check(lib().rl_kv_gather(_p(pool), _p(page_table_row), _p(out), n_tok, n_kv, HEAD_DIM, n_pages,
                             _stream()))
    return out


def new_compact_pool(n_pages: int, n_kv: int, device="cuda") -> torch.Tensor:
    """A zeroed byte pool [n_pages][n_kv][page bytes] for the q8-K / TQ3-V cache."""
    return torch.zeros(n_pages, n_kv, lib().rl_kv_compact_page_bytes(), dtype=torch.uint8, device=device)


def kv_compact_append(pool, page_table, k_rows, v_rows, wht_len=128, signs=None, pos=None, pos0=0):
    """Quantise fp32 rows [batch][n_tok][n_kv][256] into the compact cache at pos[b] (+0..n_tok-1)."""
    n_pages, n_kv = pool.shape[0], pool.shape[1]
    if k_rows.dim() == 3:
        k_rows, v_rows = k_rows.unsqueeze(0), v_rows.unsqueeze(0)
    if page_table.dim() == 1:
        page_table = page_table.unsqueeze(0)
    for t, n in ((k_rows, "k_rows"), (v_rows, "v_rows"), (signs, "signs")):
        _need(t, torch.float32, n)
    _need(page_table, torch.int32, "page_table")
    _need(pos, torch.int32, "pos")
    p = KvAppendParams(n_kv=n_kv, head_dim=HEAD_DIM, batch=k_rows.shape[0], n_tok=k_rows.shape[1],
                       page_tokens=PAGE_TOKENS, n_pages=n_pages,
                       max_pages_per_seq=page_table.shape[1], pos0=pos0, rows_fp16=0, wht_len=wht_len)
    check(lib().rl_kv_compact_append(_p(pool), _p(page_table), _p(pos), _p(k_rows), _p(v_rows),
                                     _p(signs), C.byref(p), _stream()))


def kv_compact_gather(pool, page_table_row, n_tok, wht_len=128):
    """Codes and scales of tokens [0, n_tok) in the reference's packing:
    (k_q int8 [n,n_kv,256], k_sc fp16 [n,n_kv], v_codes u8 [n,n_kv,96], v_sc fp16 [n,n_kv,256/wht])."""
    n_pages, n_kv = pool.shape[0], pool.shape[1]
    dev = pool.device
    k_q = torch.empty(n_tok, n_kv, HEAD_DIM, dtype=torch.int8, device=dev)
    k_sc = torch.empty(n_tok, n_kv, dtype=torch.float16, device=dev)
    v_codes = torch.empty(n_tok, n_kv, 96, dtype=torch.uint8, device=dev)
    v_sc = torch.empty(n_tok, n_kv, HEAD_DIM // wht_len, dtype=torch.float16, device=dev)
    check(lib().rl_kv_compact_gather(_p(pool), _p(page_table_row), _p(k_q), _p(k_sc), _p(v_codes),
                                     _p(v_sc), n_tok, n_kv, n_pages, wht_len, _stream()))
    return k_q, k_sc, v_codes, v_sc


def attn_params(n_q, n_kv, batch, n_pages, max_pages_per_seq, max_seq_len, len_add=0,
                chunk_pages=0, kv_dtype=_lib.RL_KV_F16, wht_len=128, signs=None):
    return AttnDecodeParams(n_q=n_q, n_kv=n_kv, head_dim=HEAD_DIM, kv_dtype=kv_dtype,
                            batch=batch, page_tokens=PAGE_TOKENS, n_pages=n_pages,
                            max_pages_per_seq=max_pages_per_seq, max_seq_len=max_seq_len,
                            len_add=len_add, chunk_pages=chunk_pages, wht_len=wht_len,
                            tq_signs=None if signs is None else signs.data_ptr())


def attn_decode(q, k_pool, v_pool, page_table, seq_lens, gate=None, max_seq_len=None,
                chunk_pages=0, workspace=None, out=None, partial=False, wht_len=128, signs=None):
    """ops::attn_decode for a ragged batch over the paged F16 cache, then o *= sigmoid(gate).

    q, gate [batch][n_q][256] fp32; page_table int32 [batch][max_pages]; seq_lens int32
    [batch] on the device.  With partial=True returns (part_o, part_ml) per (sequence,
    head) for a cross-GPU merge with lse_combine.  A uint8 k_pool (new_compact_pool) selects
    the q8-K / TQ3-V cache (v_pool is then ignored; wht_len 128 or 256, signs for 256).
    """
    _need(q, torch.float32, "q")
    _need(gate, torch.float32, "gate")
    _need(page_table, torch.int32, "page_table")
    _need(seq_lens, torch.int32, "seq_lens")
    batch, n_q, _ = q.shape
    n_pages, n_kv = k_pool.shape[0], k_pool.shape[1]
    if max_seq_len is None:
        max_seq_len = page_table.shape[1] * PAGE_TOKENS
    compact = k_pool.dtype == torch.uint8
    _need(signs, torch.float32, "signs")
    p = attn_params(n_q, n_kv, batch, n_pages, page_table.shape[1], max_seq_len, 0, chunk_pages,
                    _lib.RL_KV_Q8K_TQ3V if compact else _lib.RL_KV_F16, wht_len, signs)
    need = lib().rl_attn_decode_workspace_bytes(C.byref(p))
    if need == 0 and batch > 0:
        raise _lib.RlError(6, lib().rl_last_error().decode())
    if workspace is None or workspace.numel() < need:
        workspace = torch.empty(max(need, 16), dtype=torch.uint8, device=q.device)
    o = out if out is not None else torch.empty_like(q)
    if partial:
        ml = torch.empty(batch, n_q, 2, dtype=torch.float32, device=q.device)
        check(lib().rl_attn_decode_partial(_p(k_pool), _p(v_pool), _p(page_table), _p(seq_lens),
                                           _p(q), _p(o), _p(ml), _p(workspace), workspace.numel(),
                                           C.byref(p), _stream()))
        return o, ml
    check(lib().rl_attn_decode(_p(k_pool), _p(v_pool), _p(page_table), _p(seq_lens), _p(q),
                               _p(gate), _p(o), _p(workspace), workspace.numel(), C.byref(p),
                               _stream()))
    return o


def attn_prefill(q, k_pool, v_pool, page_table_row, pos0=0, k_rows=None, v_rows=None, gate=None, split=True,
                 workspace=None):
    """ops::attn_prefill for one chunk of one sequence over the paged F16 cache.

    q bf16 [T][n_q][256]; k_rows, v_rows bf16 [T][n_kv][256] are appended at pos0 first (or the
    cache already holds them); row t attends to cache rows [0, pos0 + t]; o *= sigmoid(gate).
    """
    _need(q, torch.bfloat16, "q")
    _need(k_rows, torch.bfloat16, "k_rows")
    _need(v_rows, torch.bfloat16, "v_rows")
    _need(gate, torch.float32, "gate")
    _need(page_table_row, torch.int32, "page_table_row")
    T, n_q, _ = q.shape
    n_pages, n_kv = k_pool.shape[0], k_pool.shape[1]
    o = torch.empty(T, n_q, HEAD_DIM, dtype=torch.float32, device=q.device)
    p = AttnPrefillParams(n_q=n_q, n_kv=n_kv, head_dim=HEAD_DIM, seq=T, br=128, bc=64, pos0=pos0,
                          page_tokens=PAGE_TOKENS, n_pages=n_pages, n_table=page_table_row.numel())
    need = lib().rl_attn_prefill_workspace_bytes(C.byref(p))
    ws = None
    if need and split:
        ws = workspace if workspace is not None and workspace.numel() >= need else \
            torch.empty(need, dtype=torch.uint8, device=q.device)
    check(lib().rl_attn_prefill_ws(_p(k_pool), _p(v_pool), _p(page_table_row), _p(q), _p(k_rows),
                                   _p(v_rows), _p(gate), _p(o), _p(ws), 0 if ws is None else ws.numel(),
                                   C.byref(p), _stream()))
    return o


def lse_combine(part_o, part_ml, gate=None, wht_len=0, signs=None):
    """Merge partials [n_parts][rows][256] / [n_parts][rows][2] -> o [rows][256]
    (wht_len 128/256: partials of the compact cache, still in the rotated domain)."""
    _need(part_o, torch.float32, "part_o")
    _need(part_ml, torch.float32, "part_ml")
    n_parts, rows, hd = part_o.shape
    o = torch.empty(rows, hd, dtype=torch.float32, device=part_o.device)
    check(lib().rl_lse_combine(_p(part_o), _p(part_ml), _p(gate), _p(o), n_parts, rows, hd,
                               wht_len, _p(signs), _stream()))
    return o


def delta_recurrent_step(S, q, k, v, beta, g_log, eps_l2=1e-6, slot_ids=None, head_map=None,
                         out=None):
    """ops::delta_recurrent_step for a batch; S [n_slots][n_v][128][128] fp32 in place.

    q,k [batch][n_qk][128]; v [batch][n_v][128]; beta,g_log [batch][n_v]; returns o.
    A 3-D S / 2-D q,k,v (the reference's single-sequence shapes) are accepted.
    """
    single = S.dim() == 3
    if single:
        S, q, k, v = S.unsqueeze(0), q.unsqueeze(0), k.unsqueeze(0), v.unsqueeze(0)
        beta, g_log = beta.unsqueeze(0), g_log.unsqueeze(0)
    for t, n in ((S, "S"), (q, "q"), (k, "k"), (v, "v"), (beta, "beta"), (g_log, "g_log")):
        _need(t, torch.float32, n)
    _need(slot_ids, torch.int32, "slot_ids")
    n_slots, n_v, dk, dv = S.shape
    batch, n_qk = q.shape[0], q.shape[1]
    if head_map is None:
        head_map = _lib.RL_HEADS_PER_VALUE if n_qk == n_v else _lib.RL_HEADS_GROUPED
    o = out if out is not None else torch.empty(batch, n_v, dv, dtype=torch.float32, device=S.device)
    p = DeltaRecurrentParams(n_v=n_v, dk=dk, dv=dv, eps_l2=eps_l2, batch=batch, n_slots=n_slots,
                             n_qk=n_qk, head_map=head_map, q_stride=0, k_stride=0, v_stride=0)
    check(lib().rl_delta_recurrent(_p(S), _p(slot_ids), _p(q), _p(k), _p(v), _p(beta), _p(g_log),
                                   _p(o), C.byref(p), _stream()))
    return o[0] if single else o


def delta_recurrent_multi(S, q, k, v, beta, g_log, eps_l2=1e-6, slot_ids=None, head_map=None, backup=None):
    """n_tok consecutive delta-rule steps per sequence in one pass (speculative verify).

    S [n_slots][n_v][128][128] in place; q,k [batch][n_tok][n_qk][128]; v [batch][n_tok][n_v][128];
    beta,g_log [batch][n_tok][n_v]; backup (same shape as S) receives the touched heads' state
    before the first token.  Returns o [batch][n_tok][n_v][128]."""
    for t, n in ((S, "S"), (q, "q"), (k, "k"), (v, "v"), (beta, "beta"), (g_log, "g_log"), (backup, "backup")):
        _need(t, torch.float32, n)
    _need(slot_ids, torch.int32, "slot_ids")
    n_slots, n_v, dk, dv = S.shape
    batch, n_tok, n_qk = q.shape[0], q.shape[1], q.shape[2]
    if head_map is None:
        head_map = _lib.RL_HEADS_PER_VALUE if n_qk == n_v else _lib.RL_HEADS_GROUPED
    o = torch.empty(batch, n_tok, n_v, dv, dtype=torch.float32, device=S.device)
    p = DeltaRecurrentParams(n_v=n_v, dk=dk, dv=dv, eps_l2=eps_l2, batch=batch, n_slots=n_slots,
                             n_qk=n_qk, head_map=head_map, q_stride=0, k_stride=0, v_stride=0)
    check(lib().rl_delta_recurrent_multi(_p(S), _p(backup), _p(slot_ids), _p(q), _p(k), _p(v), _p(beta),
                                         _p(g_log), _p(o), C.byref(p), n_tok, 0, 0, _stream()))
    return o


def delta_chunk_prefill(S, q, k, v, beta, g_log, eps_l2=1e-6, head_map=None, workspace=None):
    """T delta-rule steps of one sequence in chunked (WY) form: the result of T calls of
    ops::delta_recurrent_step.  S [n_v][128][128] fp32 in place; q,k [T][n_qk][128];
    v [T][n_v][128]; beta,g_log [T][n_v]; returns o [T][n_v][128]."""
    for t, n in ((S, "S"), (q, "q"), (k, "k"), (v, "v"), (beta, "beta"), (g_log, "g_log")):
        _need(t, torch.float32, n)
    n_v, dk, dv = S.shape
    T, n_qk = q.shape[0], q.shape[1]
    if head_map is None:
        head_map = _lib.RL_HEADS_PER_VALUE if n_qk == n_v else _lib.RL_HEADS_GROUPED
    p = DeltaChunkParams(n_v=n_v, dk=dk, dv=dv, seq=T, chunk=64, eps_l2=eps_l2, n_qk=n_qk, head_map=head_map)
    need = lib().rl_delta_chunk_workspace_bytes(C.byref(p))
    if need == 0 and T > 0:
        raise _lib.RlError(6, lib().rl_last_error().decode())
    if workspace is None or workspace.numel() < need:
        workspace = torch.empty(max(need, 256), dtype=torch.uint8, device=S.device)
    o = torch.empty(T, n_v, dv, dtype=torch.float32, device=S.device)
    check(lib().rl_delta_chunk_prefill(_p(S), _p(q), _p(k), _p(v), _p(beta), _p(g_log), _p(o), _p(workspace),
                                       workspace.numel(), C.byref(p), _stream()))
    return o


def conv1d_update(x_t, w, state, slot_ids=None):
    """ops::conv1d_update: state [n_slots][dim][k] (or [dim][k]) in place; x_t [batch][dim]."""
    single = x_t.dim() == 1
    if single:
        x_t, state = x_t.unsqueeze(0), state.unsqueeze(0)
    for t, n in ((x_t, "x_t"), (w, "w"), (state, "state")):
        _need(t, torch.float32, n)
    batch, dim = x_t.shape
    y = torch.empty_like(x_t)
    p = Conv1dParams(dim=dim, k=w.shape[1], silu=1, batch=batch, n_slots=state.shape[0])
    check(lib().rl_conv1d_update(_p(x_t), _p(w), _p(state), _p(slot_ids), _p(y), C.byref(p),
                                 _stream()))
    return y[0] if single else y


def conv1d_causal_prefill(x, w, state=None, use_state_in=False):
    """ops::conv1d_causal_prefill over x [seq][dim]; optional [dim][k] window in/out."""
    _need(x, torch.float32, "x")
    _need(w, torch.float32, "w")
    _need(state, torch.float32, "state")
    seq, dim = x.shape
    y = torch.empty_like(x)
    p = Conv1dParams(dim=dim, k=w.shape[1], silu=1, batch=1, n_slots=1)
    check(lib().rl_conv1d_causal(_p(x), _p(w), _p(y), _p(state), seq, C.byref(p),
                                 int(use_state_in), _stream()))
    return y


def attn_qk_prepare(qg, k, q_norm=None, k_norm=None, pos=None, pos0=0, rotary_dim=64, theta=1e7, eps=1e-6):
    """The steps of fused_attn_decode between the projections and the cache append: split
    qg [rows][n_q][512] into q and gate, head RMSNorm (1 + gamma) of q and k, partial RoPE at
    pos [rows] (int32) or pos0 + row.  k [rows][n_kv][256] is updated in place; returns q, gate."""
    for t, n in ((qg, "qg"), (k, "k"), (q_norm, "q_norm"), (k_norm, "k_norm")):
        _need(t, torch.float32, n)
    _need(pos, torch.int32, "pos")
    rows, n_q, two_hd = qg.shape
    q = torch.empty(rows, n_q, two_hd // 2, dtype=torch.float32, device=qg.device)
    gate = torch.empty_like(q)
    p = _lib.AttnQkPrepareParams(n_q=n_q, n_kv=k.shape[1], head_dim=two_hd // 2, rotary_dim=rotary_dim,
                                 rows=rows, pos0=pos0, theta=theta, eps=eps)
    check(lib().rl_attn_qk_prepare(_p(qg), _p(k), _p(q_norm), _p(k_norm), _p(pos), _p(q), _p(gate),
                                   C.byref(p), _stream()))
    return q, gate


def rmsnorm(x, gamma=None, eps=1e-6, out=None):
    """ops::qwen3_rmsnorm over the last dimension: x / rms(x) * (1 + gamma)."""
    _need(x, torch.float32, "x")
    _need(gamma, torch.float32, "gamma")
    y = torch.empty_like(x) if out is None else out
    n = x.shape[-1]
    check(lib().rl_rmsnorm(_p(x), _p(gamma), _p(y), x.numel() // n, n, eps, _stream()))
    return y


def gated_rmsnorm(x, z, gamma=None, eps=1e-6):
    """ops::gated_rmsnorm per head: x, z [rows][n_heads][128], gamma [128] -> y."""
    for t, n in ((x, "x"), (z, "z"), (gamma, "gamma")):
        _need(t, torch.float32, n)
    rows, n_heads, hd = x.shape
    y = torch.empty_like(x)
    check(lib().rl_gated_rmsnorm(_p(x), _p(z), _p(gamma), _p(y), rows, n_heads, hd, eps, _stream()))
    return y


def delta_gates(a, b, A_log, dt_bias):
    """beta = sigmoid(b), g_log = -exp(A_log) * softplus(a + dt_bias); a, b [rows][n_v]."""
    for t, n in ((a, "a"), (b, "b"), (A_log, "A_log"), (dt_bias, "dt_bias")):
        _need(t, torch.float32, n)
    rows, n_v = a.shape
    beta, g = torch.empty_like(a), torch.empty_like(a)
    check(lib().rl_delta_gates(_p(a), _p(b), _p(A_log), _p(dt_bias), _p(beta), _p(g), rows, n_v, _stream()))
    return beta, g


def kv_compact_to_f16(pool, src_table_row, k_pool, v_pool, dst_table_row, n_tok, src_pos0=0, dst_pos0=0,
                      wht_len=128, signs=None):
    """Dequantise n_tok tokens of one sequence of the compact cache into paged F16 pools (the
    F16 compute window for prefill chunks / verify rows over a compact cache)."""
    _need(src_table_row, torch.int32, "src_table_row")
    _need(dst_table_row, torch.int32, "dst_table_row")
    _need(signs, torch.float32, "signs")
    check(lib().rl_kv_compact_to_f16(_p(pool), _p(src_table_row), src_pos0, pool.shape[0], _p(k_pool), _p(v_pool),
                                     _p(dst_table_row), dst_pos0, k_pool.shape[0], n_tok, pool.shape[1], wht_len,
                                     _p(signs), _stream()))


def gdn_decode(S, conv_ring, conv_phase, qkv, conv_w, beta, g_log, n_qk, slot_ids=None, head_map=None,
               eps_l2=1e-6, advance=True):
    """The fused Gated DeltaNet decode step of one layer (rl_gdn_decode): conv window + SiLU + l2
    norms + delta rule.  S [n_slots][n_v][128][128], conv_ring [n_slots][conv_dim][4] (ring windows),
    conv_phase int32 [n_slots], qkv [batch][conv_dim], conv_w [conv_dim][4]; returns o.  With
    advance the rings' phases move on afterwards (rl_gdn_phase_advance), as after a layer's step."""
    for t, n in ((S, "S"), (conv_ring, "conv_ring"), (qkv, "qkv"), (conv_w, "conv_w"), (beta, "beta"), (g_log, "g_log")):
        _need(t, torch.float32, n)
    _need(conv_phase, torch.int32, "conv_phase")
    _need(slot_ids, torch.int32, "slot_ids")
    n_slots, n_v, dk, dv = S.shape
    batch = qkv.shape[0]
    if head_map is None:
        head_map = _lib.RL_HEADS_PER_VALUE if n_qk == n_v else _lib.RL_HEADS_GROUPED
    o = torch.empty(batch, n_v, dv, dtype=torch.float32, device=S.device)
    p = _lib.GdnDecodeParams(n_v=n_v, n_qk=n_qk, dk=dk, dv=dv, conv_k=conv_w.shape[1], batch=batch, n_slots=n_slots,
                             head_map=head_map, eps_l2=eps_l2)
    check(lib().rl_gdn_decode(_p(S), _p(conv_ring), _p(conv_phase), _p(slot_ids), _p(qkv), _p(conv_w), _p(beta),
                              _p(g_log), _p(o), C.byref(p), _stream()))
    if advance:
        check(lib().rl_gdn_phase_advance(_p(conv_phase), _p(slot_ids), 1, n_slots, batch, 1, _stream()))
    return o


def conv_ring_export(conv_ring, conv_phase):
    """Ring windows [n_slots][conv_dim][4] -> the reference's shifted windows, oldest tap first."""
    out = torch.empty_like(conv_ring)
    check(lib().rl_conv_ring_export(_p(conv_ring), _p(conv_phase), _p(out), 1, conv_ring.shape[0], -1,
                                    conv_ring.shape[1], _stream()))
    return out


# ---- trees of drafted tokens: append, verify, commit (rl_b200.h has the format of parents, n_nodes, leaf) ----
#
# These calls take microseconds on the device, so their host side is kept short: one test per tensor, addresses
# passed as plain integers.

_TYPES = {torch.float32: _lib.RL_TYPE_F32, torch.float16: _lib.RL_TYPE_F16, torch.bfloat16: _lib.RL_TYPE_BF16}
_F32, _I32 = torch.float32, torch.int32


def _stream_of(dev):
    return torch._C._cuda_getCurrentRawStream(dev)


def _arg(t, dtype, shape, dev, name):
    """Address of a contiguous tensor of that type and shape on device `dev` (the current one, whose current stream
    the call goes to); None for None."""
    if t is None:
        return None
    if t.get_device() == dev and t.dtype is dtype and t.shape == shape and t.is_contiguous():
        return t.data_ptr()
    raise _lib.RlError(6, f"{name}: need a contiguous {dtype} tensor of shape {tuple(shape)} on the current device cuda:{dev}, "
                          f"got {t.dtype} {tuple(t.shape)} on {t.device}")


def _needed(t, *rest):
    if t is None:
        raise _lib.RlError(6, f"{rest[-1]}: is None")
    return _arg(t, *rest)


def _rows(t, shape, dev, name):
    """Address of fp32 [batch][rows]..., dense inside a row, rows at one distance; and that distance in floats."""
    if t is None or t.get_device() != dev or t.dtype is not _F32 or t.shape != shape:
        raise _lib.RlError(6, f"{name}: need a {_F32} tensor of shape {tuple(shape)} on the current device cuda:{dev}")
    strides, inner = t.stride(), 1
    for d in range(len(shape) - 1, 1, -1):
        if shape[d] > 1 and strides[d] != inner:
            raise _lib.RlError(6, f"{name}: a row must be contiguous")
        inner *= shape[d]
    return t.data_ptr(), _row_distance(shape, strides, inner, name)


def _row_distance(shape, strides, inner, name):
    """Floats between the rows of [batch][rows]...  Rows that share memory (an expanded tensor has them 0 apart, which
    the C ABI takes as "dense") are refused here: the kernels would read behind the one row that exists."""
    row = strides[1] if shape[1] > 1 else (strides[0] if shape[0] > 1 else inner)
    if row < inner:
        raise _lib.RlError(6, f"{name}: rows {row} floats apart share memory, a row has {inner}")
    if shape[0] > 1 and shape[1] > 1 and strides[0] != shape[1] * row:
        raise _lib.RlError(6, f"{name}: the rows of all sequences must be at one distance")
    return row


def _gate(gate, shape, dev):
    """Address of fp32 [batch][nodes][heads][256], contiguous inside a head; floats between its rows and its heads."""
    if gate.get_device() != dev or gate.dtype is not _F32 or gate.shape != shape or gate.stride(3) != 1:
        raise _lib.RlError(6, f"gate: need a {_F32} tensor of shape {tuple(shape)} on the current device cuda:{dev}, contiguous inside a head")
    strides = gate.stride()
    head = strides[2] if shape[2] > 1 else shape[3]
    if head < shape[3]:
        raise _lib.RlError(6, f"gate: heads {head} floats apart share memory, a head has {shape[3]}")
    return gate.data_ptr(), _row_distance(shape, strides, head * shape[2], "gate"), head


def _scratch(workspace, need, device):
    """The caller's workspace where it is large enough, else a new one; and its size."""
    if workspace is not None:
        size = workspace.numel() * workspace.element_size()
        if size >= need:
            return workspace, size
    return torch.empty(need, dtype=torch.uint8, device=device), need


def _pools(k_pool, v_pool, page_table, batch, dev):
    shape = k_pool.shape
    if len(shape) != 3 or shape[2] != PAGE_TOKENS * HEAD_DIM:
        raise _lib.RlError(6, "k_pool: need [n_pages][n_kv][64 * 256] (new_pool)")
    if page_table.dim() != 2:
        raise _lib.RlError(6, f"page_table: need [{batch}][max_pages]")
    pages = page_table.shape[1]
    return (shape[0], shape[1], pages, _needed(k_pool, torch.float16, shape, dev, "k_pool"),
            _needed(v_pool, torch.float16, shape, dev, "v_pool"), _needed(page_table, _I32, (batch, pages), dev, "page_table"))


def attn_qk_append(qg, k, v, k_pool, v_pool, page_table, pos, q_norm=None, k_norm=None, parents=None, n_nodes=None,
                   rotary_dim=64, theta=1e7, eps=1e-6, q_dtype=torch.float32, want_gate=True, q_out=None, gate_out=None,
                   angle_f32=False):
    """From the projections to the operands of the attention in one pass: q/gate split, head RMSNorm
    (1 + gamma), rotation, K and V rows into the paged F16 cache at pos[b] + t.

    qg fp32 [batch][n_tok][n_q][512] ([q | gate] per head), k, v fp32 [batch][n_tok][n_kv][256], column
    ranges of one projection or dense; pos int32 [batch].  Row t is rotated by pos[b] + t, with parents
    [batch][n_tok] (n_tok <= 64) by pos[b] + the node's depth; the angle is formed in 64 bits, or with angle_f32 as
    attn_qk_prepare forms it (for a cache that holds its rows too).  Returns q of q_dtype (or of q_out) and the
    gate, None without want_gate.  Rows behind n_nodes[b] are left as they are."""
    dev = torch.cuda.current_device()
    batch, n_tok, n_q, two_hd = qg.shape
    if two_hd != 2 * HEAD_DIM:
        raise _lib.RlError(4, f"qg: rows of {two_hd} per head, only 512")
    n_pages, n_kv, pages, kp, vp, table = _pools(k_pool, v_pool, page_table, batch, dev)
    qg_p, qg_row = _rows(qg, qg.shape, dev, "qg")
    k_p, k_row = _rows(k, (batch, n_tok, n_kv, HEAD_DIM), dev, "k")
    v_p, v_row = _rows(v, (batch, n_tok, n_kv, HEAD_DIM), dev, "v")
    shape = (batch, n_tok, n_q, HEAD_DIM)
    if q_out is None:
        q_out = torch.empty(shape, dtype=q_dtype, device=qg.device)
    if q_out.dtype not in _TYPES:
        raise _lib.RlError(4, f"q_out: {q_out.dtype} unknown")
    if not want_gate:
        gate_out = None
    elif gate_out is None:
        gate_out = torch.empty(shape, dtype=_F32, device=qg.device)
    p = _lib.AttnQkAppendParams(n_q, n_kv, HEAD_DIM, rotary_dim, batch, n_tok, PAGE_TOKENS, n_pages, pages,
                                _TYPES[q_out.dtype], theta, eps, qg_row, k_row, v_row, angle_f32)
    check(lib().rl_attn_qk_append(kp, vp, table, _needed(pos, _I32, (batch,), dev, "pos"),
                                  _arg(parents, _I32, (batch, n_tok), dev, "parents"), _arg(n_nodes, _I32, (batch,), dev, "n_nodes"),
                                  qg_p, k_p, v_p, _arg(q_norm, _F32, (HEAD_DIM,), dev, "q_norm"),
                                  _arg(k_norm, _F32, (HEAD_DIM,), dev, "k_norm"), _arg(q_out, q_out.dtype, shape, dev, "q_out"),
                                  _arg(gate_out, _F32, shape, dev, "gate_out"), p, _stream_of(dev)))
    return q_out, gate_out


@functools.lru_cache(maxsize=256)
def _attn_tree_plan(dev, *fields):
    p = _lib.AttnTreeParams(*fields)
    need = lib().rl_attn_tree_workspace_bytes(p)
    if need == 0:
        raise _lib.RlError(6, lib().rl_last_error().decode())
    return p, need


def attn_tree(q, k_pool, v_pool, page_table, base_len, parents=None, n_nodes=None, gate=None, max_seq_len=None, out=None,
              out_dtype=None, workspace=None):
    """Attention of every node of a draft tree over the paged F16 cache: node i of sequence b sees the rows
    [0, base_len[b]) and base_len[b] + j for its ancestors j and itself; o *= sigmoid(gate).

    q fp32, fp16 or bf16 [batch][nodes][n_q][256]; gate fp32 of that shape, dense or strided (qg[..., 256:] as
    it lies); out fp16 or bf16 (default: q's type, fp16 for fp32).  parents None = chains."""
    dev = torch.cuda.current_device()
    shape = q.shape
    batch, nodes, n_q, hd = shape
    n_pages, n_kv, pages, kp, vp, table = _pools(k_pool, v_pool, page_table, batch, dev)
    if q.dtype not in _TYPES:
        raise _lib.RlError(4, f"q: {q.dtype} unknown")
    if out is None:
        out = torch.empty(shape, dtype=out_dtype or (torch.float16 if q.dtype is _F32 else q.dtype), device=q.device)
    if out.dtype not in _TYPES:
        raise _lib.RlError(4, f"out: {out.dtype} unknown")
    row = head = 0
    gate_p = None
    if gate is not None:
        gate_p, row, head = _gate(gate, shape, dev)
    p, need = _attn_tree_plan(dev, n_q, n_kv, hd, batch, nodes, PAGE_TOKENS, n_pages, pages,
                              pages * PAGE_TOKENS if max_seq_len is None else max_seq_len, _TYPES[q.dtype], _TYPES[out.dtype], row, head)
    workspace, size = _scratch(workspace, need, q.device)
    check(lib().rl_attn_tree(kp, vp, table, _needed(base_len, _I32, (batch,), dev, "base_len"),
                             _arg(parents, _I32, (batch, nodes), dev, "parents"), _arg(n_nodes, _I32, (batch,), dev, "n_nodes"),
                             _arg(q, q.dtype, shape, dev, "q"), gate_p, _arg(out, out.dtype, shape, dev, "out"),
                             _arg(workspace, workspace.dtype, workspace.shape, dev, "workspace"), size, p, _stream_of(dev)))
    return out


def kv_tree_commit(k_pool, v_pool, page_table, base_len, parents, leaf, n_nodes=None):
    """Keep the path to node leaf[b] (int32 [batch], -1 = nothing) of each sequence's tree: its K and V rows move
    to positions base_len[b], base_len[b] + 1, ...  Returns the paths' lengths, int32 [batch].  parents int32
    [batch][nodes], or the number of nodes for chains; n_nodes int32 [batch] as the verify had them: a leaf behind
    them counts as -1."""
    dev = torch.cuda.current_device()
    batch = leaf.shape[0]
    chain = isinstance(parents, int)
    if parents is None:
        raise _lib.RlError(6, "parents: is None (chains: the number of nodes)")
    nodes = parents if chain else parents.shape[1]
    n_pages, n_kv, pages, kp, vp, table = _pools(k_pool, v_pool, page_table, batch, dev)
    n_accept = torch.empty_like(leaf)
    p = _lib.KvTreeCommitParams(n_kv, HEAD_DIM, batch, nodes, PAGE_TOKENS, n_pages, pages, _arg(n_nodes, _I32, (batch,), dev, "n_nodes"))
    check(lib().rl_kv_tree_commit(kp, vp, table, _needed(base_len, _I32, (batch,), dev, "base_len"),
                                  None if chain else _needed(parents, _I32, (batch, nodes), dev, "parents"),
                                  _needed(leaf, _I32, (batch,), dev, "leaf"), n_accept.data_ptr(), p, _stream_of(dev)))
    return n_accept


def _gdn_tree_args(dev, S, conv_window, conv_phase, qkv, conv_w, beta, g_log, parents, third, name, n_qk, slot_ids, head_map,
                   eps_l2):
    n_slots, n_v, dk, dv = S.shape
    batch, nodes, dim = qkv.shape
    if dim != 2 * n_qk * dk + n_v * dv:
        raise _lib.RlError(6, f"qkv: rows of {dim} channels, {n_qk} key and {n_v} value heads need {2 * n_qk * dk + n_v * dv}")
    if slot_ids is None and batch > n_slots:
        raise _lib.RlError(6, f"{batch} sequences in {n_slots} slots")
    if head_map is None:
        head_map = _lib.RL_HEADS_PER_VALUE if n_qk == n_v else _lib.RL_HEADS_GROUPED
    qkv_p, row = _rows(qkv, qkv.shape, dev, "qkv")
    gates = (batch, nodes, n_v)
    return (_lib.GdnTreeParams(n_v, n_qk, dk, dv, 4, batch, nodes, n_slots, head_map, eps_l2, row),
            (_needed(S, _F32, S.shape, dev, "S"), _needed(conv_window, _F32, (n_slots, dim, 4), dev, "conv_window"),
             _arg(conv_phase, _I32, (n_slots,), dev, "conv_phase"), _arg(slot_ids, _I32, (batch,), dev, "slot_ids"),
             _arg(parents, _I32, (batch, nodes), dev, "parents"), _arg(third, _I32, (batch,), dev, name), qkv_p,
             _needed(conv_w, _F32, (dim, 4), dev, "conv_w"), _needed(beta, _F32, gates, dev, "beta"),
             _needed(g_log, _F32, gates, dev, "g_log")))


def gdn_tree(S, conv_window, conv_phase, qkv, conv_w, beta, g_log, parents, n_qk, n_nodes=None, slot_ids=None,
             head_map=None, eps_l2=1e-6, out=None, workspace=None):
    """The Gated DeltaNet step of every node of a draft tree, each along its own path; S [n_slots][n_v][128][128]
    and conv_window [n_slots][conv_dim][4] are only read.  conv_phase int32 [n_slots] (rings, see gdn_decode) or
    None (shifted windows, conv1d_update's state).  qkv fp32 [batch][nodes][conv_dim] (rows may be a column range),
    beta, g_log [batch][nodes][n_v].  Returns o fp32 [batch][nodes][n_v][128]."""
    dev = torch.cuda.current_device()
    p, args = _gdn_tree_args(dev, S, conv_window, conv_phase, qkv, conv_w, beta, g_log, parents, n_nodes, "n_nodes", n_qk,
                             slot_ids, head_map, eps_l2)
    shape = (qkv.shape[0], qkv.shape[1], S.shape[1], S.shape[3])
    if out is None:
        out = torch.empty(shape, dtype=_F32, device=S.device)
    workspace, size = _scratch(workspace, lib().rl_gdn_tree_workspace_bytes(p), S.device)
    check(lib().rl_gdn_tree(*args, _arg(out, _F32, shape, dev, "out"), _arg(workspace, workspace.dtype, workspace.shape, dev, "workspace"),
                            size, p, _stream_of(dev)))
    return out


def gdn_tree_commit(S, conv_window, conv_phase, qkv, conv_w, beta, g_log, parents, leaf, n_qk, slot_ids=None,
                    head_map=None, eps_l2=1e-6, workspace=None, n_nodes=None):
    """Advance S and conv_window of each sequence's slot by the path to node leaf[b] (-1 = nothing), in place, with
    gdn_tree's inputs; conv_phase stays.  slot_ids must be distinct; a leaf behind n_nodes[b] counts as -1."""
    dev = torch.cuda.current_device()
    p, args = _gdn_tree_args(dev, S, conv_window, conv_phase, qkv, conv_w, beta, g_log, parents, leaf, "leaf", n_qk, slot_ids,
                             head_map, eps_l2)
    if leaf is None:
        raise _lib.RlError(6, "leaf: is None")
    p.commit_nodes = _arg(n_nodes, _I32, (qkv.shape[0],), dev, "n_nodes")
    workspace, size = _scratch(workspace, lib().rl_gdn_tree_commit_workspace_bytes(p), S.device)
    check(lib().rl_gdn_tree_commit(*args, _arg(workspace, workspace.dtype, workspace.shape, dev, "workspace"), size, p, _stream_of(dev)))
