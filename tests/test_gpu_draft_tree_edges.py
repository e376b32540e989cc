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


def test_kv_commit_accepts_nothing_where_it_moves_nothing():
    """A base outside the table and a bad page under the rows up to the leaf: the sequence's rows stay, its accepted length
    is 0 (the caller adds it to base_len); the other sequences are served."""
    from rapidllm_b200 import _lib, ops
    gen = torch.Generator().manual_seed(42)
    base, n = [60, 60, 62, 130, 70, 10, 40], 8
    kp, vp, table, _ = _pages(gen, base, [n] * 7, 4, 0.0)
    parents = torch.tensor([[-1, -1, 1, 0, 2, 4, 3, 5]] * 7, dtype=torch.int32)
    parents[5] = torch.arange(n) - 1                          # a chain, whose rows stay where they are
    leaf = [7] * 7
    table[1, 1] = -1                                          # the page of the leaf
    table[2, 0] = kp.shape[0]                                 # the page of the first row
    table[5, 0] = -7
    bases = [60, 60, 62, table.shape[1] * 64 - 7, -1, 10, 40]
    want = [pool.clone() for pool in (kp, vp)]
    for b in (0, 6):
        for w, src in zip(want, (kp, vp)):
            for j, i in enumerate(_path(parents[b].tolist(), 7)):
                page, at = int(table[b, (base[b] + j) // 64]), (base[b] + j) % 64
                w[page][:, ops.kv_slice_index(torch.full((HD,), at), torch.arange(HD)).cuda()] = _pool_row(src, table, b, base[b] + i)
    taken = ops.kv_tree_commit(kp, vp, table, _i32(bases), parents.cuda(), _i32(leaf))
    assert _lib.device_error() in (1, 5)
    assert taken.tolist() == [5, 0, 0, 0, 0, 0, 5]
    assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])
