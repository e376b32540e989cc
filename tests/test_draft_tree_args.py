"""Refusals of the draft-tree entry points: before anything touches a device, with the status codes and a message."""
import ctypes as C

import pytest

from rapidllm_b200 import _lib

RANGE, UNSUPPORTED = 6, 4


def _err():
    return _lib.lib().rl_last_error().decode()


def _append(**kw):
    p = _lib.AttnQkAppendParams(n_q=24, n_kv=4, head_dim=256, rotary_dim=64, batch=1, n_tok=4, page_tokens=64, n_pages=4,
                                max_pages_per_seq=4, q_type=0, theta=1e7, eps=1e-6)
    parents = kw.pop("parents", None)
    for k, v in kw.items():
        setattr(p, k, v)
    return _lib.lib().rl_attn_qk_append(None, None, None, None, parents, None, None, None, None, None, None, None, None,
                                        C.byref(p), None)


def _attn(**kw):
    p = _lib.AttnTreeParams(n_q=24, n_kv=4, head_dim=256, batch=1, max_nodes=8, page_tokens=64, n_pages=4, max_pages_per_seq=4,
                            max_seq_len=256, q_type=0, o_type=1)
    for k, v in kw.items():
        setattr(p, k, v)
    return _lib.lib().rl_attn_tree(None, None, None, None, None, None, None, None, None, None, 0, C.byref(p), None)


def _kv(**kw):
    p = _lib.KvTreeCommitParams(n_kv=4, head_dim=256, batch=1, max_nodes=8, page_tokens=64, n_pages=4, max_pages_per_seq=4)
    for k, v in kw.items():
        setattr(p, k, v)
    return _lib.lib().rl_kv_tree_commit(None, None, None, None, None, None, None, C.byref(p), None)


def _gdn(commit=False, **kw):
    p = _lib.GdnTreeParams(n_v=48, n_qk=16, dk=128, dv=128, conv_k=4, batch=1, max_nodes=8, n_slots=1, head_map=1, eps_l2=1e-6)
    for k, v in kw.items():
        setattr(p, k, v)
    if commit:
        return _lib.lib().rl_gdn_tree_commit(*[None] * 11, 0, C.byref(p), None)
    return _lib.lib().rl_gdn_tree(*[None] * 12, 0, C.byref(p), None)


@pytest.mark.parametrize("call,status,kw", [
    (_append, UNSUPPORTED, dict(head_dim=128)), (_append, UNSUPPORTED, dict(page_tokens=32)), (_append, RANGE, dict(rotary_dim=24)),
    (_append, RANGE, dict(rotary_dim=272)), (_append, RANGE, dict(theta=0.0)), (_append, UNSUPPORTED, dict(q_type=3)),
    (_append, RANGE, dict(qg_stride=100)), (_append, RANGE, dict(k_stride=1026)), (_append, RANGE, dict(v_stride=-1024)),
    (_append, RANGE, dict(n_tok=65, parents=C.c_void_p(16))), (_append, RANGE, dict(n_tok=-1)), (_append, RANGE, dict(n_q=0)),
    (_append, RANGE, dict(batch=65535, n_tok=65535)), (_append, RANGE, dict()),
    (_attn, UNSUPPORTED, dict(head_dim=64)), (_attn, UNSUPPORTED, dict(n_q=25)), (_attn, UNSUPPORTED, dict(n_q=36)),
    (_attn, RANGE, dict(max_nodes=65)), (_attn, RANGE, dict(batch=513)), (_attn, RANGE, dict(max_seq_len=257)),
    (_attn, RANGE, dict(max_seq_len=0)), (_attn, UNSUPPORTED, dict(o_type=0)), (_attn, UNSUPPORTED, dict(q_type=-1)),
    (_attn, RANGE, dict(gate_head=128)), (_attn, RANGE, dict(gate_head=512, gate_row=512)), (_attn, RANGE, dict(gate_row=24 * 256 + 2)),
    (_attn, RANGE, dict(batch=512, n_kv=64, n_q=512, max_nodes=64, max_pages_per_seq=1 << 20, max_seq_len=1 << 20)), (_attn, RANGE, dict()),
    (_kv, UNSUPPORTED, dict(head_dim=64)), (_kv, RANGE, dict(max_nodes=65)), (_kv, RANGE, dict(n_pages=0)), (_kv, RANGE, dict()),
    (_gdn, UNSUPPORTED, dict(dk=64)), (_gdn, UNSUPPORTED, dict(conv_k=3)), (_gdn, RANGE, dict(max_nodes=65)), (_gdn, RANGE, dict(n_qk=7)),
    (_gdn, RANGE, dict(head_map=3)), (_gdn, RANGE, dict(head_map=-1)), (_gdn, RANGE, dict(qkv_stride=10238)), (_gdn, RANGE, dict(n_slots=0)),
    (_gdn, RANGE, dict()),
    (_gdn, UNSUPPORTED, dict(commit=True, dv=64)), (_gdn, RANGE, dict(commit=True, max_nodes=-1)), (_gdn, RANGE, dict(commit=True)),
])
def test_refused_with_a_message(call, status, kw):
    assert call(**kw) == status and _err()


def test_null_params_and_empty_calls():
    L = _lib.lib()
    assert L.rl_attn_qk_append(*[None] * 15) == RANGE
    assert L.rl_attn_tree(*[None] * 10, 0, None, None) == RANGE
    assert L.rl_attn_tree_workspace_bytes(None) == 0
    assert L.rl_kv_tree_commit(*[None] * 9) == RANGE
    assert L.rl_gdn_tree(*[None] * 12, 0, None, None) == RANGE and L.rl_gdn_tree_workspace_bytes(None) == 0 and L.rl_gdn_tree_commit(*[None] * 11, 0, None, None) == RANGE
    assert L.rl_gdn_tree_commit_workspace_bytes(None) == 0
    assert _append(batch=0) == 0 and _append(n_tok=0) == 0
    assert _attn(batch=0) == 0 and _attn(max_nodes=0) == 0
    assert _kv(batch=0) == 0
    assert _gdn(batch=0) == 0 and _gdn(max_nodes=0) == 0 and _gdn(commit=True, batch=0) == 0
