"""Draft-tree operators where a call is easily got wrong: expanded inputs, sequences that are refused inside a batch, leaves
of ragged drafts, chains, odd head counts, rounding of queries and weights, many heads at once.  Shapes, 64-bit forms and
tolerances are those of test_gpu_draft_tree.py unless a test derives its own."""
import math

import pytest
import torch

from helpers import STATE_REL_L2, rel_l2
from test_gpu_draft_tree import (DK, HALF_STEP, HD, _attn_exact, _gdn_exact, _gdn_inputs, _pages, _path, _pool_row, _tree,
                                 _weights)

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def test_expanded_inputs_are_refused():
    """A tensor whose rows or heads share memory is an RlError before anything is launched."""
    from rapidllm_b200 import _lib, ops
    gen = torch.Generator().manual_seed(41)
    B, n = 2, 8
    kp, vp, table, _ = _pages(gen, [10, 70], [n, n], 4, 0.0)
    base, parents, leaf = _i32([10, 70]), _tree(gen, B, n, 2).cuda(), _i32([1, 2])
    q = torch.zeros(B, n, 24, HD, device="cuda")
    qg, k = torch.zeros(B, n, 24, 512, device="cuda"), torch.zeros(B, n, 4, HD, device="cuda")
    S, win, qkv, w, beta, g = (t.cuda() for t in _gdn_inputs(gen, B, n, 6, 2, B))
    kept = kp.clone(), S.clone(), win.clone()
    gdn = dict(S=S, conv_window=win, conv_phase=None, conv_w=w, beta=beta, g_log=g, parents=parents, n_qk=2)
    app = dict(k_pool=kp, v_pool=vp, page_table=table, pos=base, parents=parents)
    calls = [lambda x=x: ops.attn_tree(q, kp, vp, table, base, parents, gate=x.expand(B, n, 24, HD))
             for x in (q[:1, :1], q[:1], q[:, :1], q[:, :, :1], q[:, :, :, :1])]
    calls += [lambda: ops.attn_qk_append(qg[:1, :1].expand(B, n, 24, 512), k, k, **app),
              lambda: ops.attn_qk_append(qg, k[:1, :1].expand(B, n, 4, HD), k, **app),
              lambda: ops.attn_qk_append(qg, k, k[:, :, :1].expand(B, n, 4, HD), **app),
              lambda: ops.gdn_tree(qkv=qkv[:1, :1].expand(B, n, -1), **gdn),
              lambda: ops.gdn_tree_commit(qkv=qkv[:1, :1].expand(B, n, -1), leaf=leaf, **gdn)]
    for call in calls:
        with pytest.raises(_lib.RlError):
            call()
    _lib.check_device()
    for t, was in zip((kp, S, win), kept):
        assert torch.equal(t, was)
