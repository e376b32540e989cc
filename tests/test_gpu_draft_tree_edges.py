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


def _gdn_tree_exact(S, win, qkv, w, beta, g, parents, n, n_qk, tiled):
    """o of the first n nodes of one sequence in 64 bits on the device, each node from its parent's state and window."""
    n_v, qd = S.shape[0], n_qk * DK
    hs = torch.tensor([h % n_qk if tiled else h // (n_v // n_qk) for h in range(n_v)], device="cuda")
    S, win, w, qkv, beta, g = (t.cuda().double() for t in (S, win, w, qkv, beta, g))
    at, out = {-1: (S, win)}, []
    for i in range(n):
        state, window = at[parents[i]]
        window = torch.cat([window[:, 1:], qkv[i].unsqueeze(1)], 1)
        y = (window * w).sum(1)
        y = y / (1 + torch.exp(-y))
        q, k, v = y[:qd].view(-1, DK)[hs], y[qd:2 * qd].view(-1, DK)[hs], y[2 * qd:].view(-1, DK)
        q = q / (q.square().sum(1, keepdim=True) + 1e-6).sqrt() / DK ** 0.5
        k = k / (k.square().sum(1, keepdim=True) + 1e-6).sqrt()
        state = state * g[i].exp().view(-1, 1, 1)
        state = state + k.unsqueeze(2) * (beta[i].unsqueeze(1) * (v - (k.unsqueeze(2) * state).sum(1))).unsqueeze(1)
        at[i] = state, window
        out.append((q.unsqueeze(2) * state).sum(1))
    return torch.stack(out).cpu() if out else None


def _full_batch(n_v):
    """Sequences at which the value heads of a key head share a CTA of gdn_tree: more than two heads per SM."""
    return 2 * torch.cuda.get_device_properties(0).multi_processor_count // n_v + 1


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


def test_a_leaf_behind_the_last_node_keeps_nothing():
    """Of a ragged draft: rows behind n_nodes[b] are neither read nor written, so a leaf there is recorded and counts as
    -1, in both commits and through the mixers; the last node itself is a leaf."""
    from rapidllm_b200 import _lib, ops
    gen = torch.Generator().manual_seed(43)
    B, n, n_v, n_qk = 5, 12, 6, 2
    counts, leaf = [5, 5, 0, 12, 13], [5, 4, 0, 11, 3]        # the last count is itself out of range: an empty draft
    parents = _tree(gen, B, n, 3)
    parents[0, 5:] = 77                                       # not validated by a verify, and not followed here
    S, win, qkv, w, beta, g = _gdn_inputs(gen, B, n, n_v, n_qk, B)
    qkv[0, 5:] = float("nan")
    dev = [t.cuda() for t in (S, win)]
    ops.gdn_tree_commit(*dev, None, *(t.cuda() for t in (qkv, w, beta, g, parents)), _i32(leaf), n_qk, n_nodes=_i32(counts))
    assert _lib.device_error() == 6
    for b in range(B):
        if b in (1, 3):
            path = _path(parents[b].tolist(), leaf[b])
            _, state, window = _gdn_exact(S[b], win[b], qkv[b], w, beta[b], g[b], path, n_v, n_qk, False)
            assert rel_l2(dev[0][b].cpu(), state) <= STATE_REL_L2 and torch.equal(dev[1][b].cpu(), window.float())
        else:
            assert torch.equal(dev[0][b].cpu(), S[b]) and torch.equal(dev[1][b].cpu(), win[b])
    base = [60, 61, 62, 63, 10]
    kp, vp, table, _ = _pages(gen, base, [n] * B, 4, 0.0)
    before = [[_pool_row(kp, table, b, base[b] + i).clone() for i in range(n)] for b in range(B)]
    taken = ops.kv_tree_commit(kp, vp, table, _i32(base), parents.cuda(), _i32(leaf), n_nodes=_i32(counts))
    assert _lib.device_error() == 6
    paths = [_path(parents[b].tolist(), leaf[b]) if b in (1, 3) else [] for b in range(B)]
    assert taken.tolist() == [len(p) for p in paths]
    for b in range(B):
        for i in range(n):
            src = paths[b][i] if i < len(paths[b]) else i
            assert torch.equal(_pool_row(kp, table, b, base[b] + i), before[b][src])


def test_the_stack_remembers_the_nodes_of_a_draft():
    """A commit through the mixers refuses the leaves that its verify did not run."""
    from rapidllm_b200 import _lib
    from rapidllm_b200.mixer import MixerStack
    gen = torch.Generator().manual_seed(44)
    attn, delta = _weights(gen, 128)
    stack = MixerStack([_lib.RL_LAYER_LINEAR_ATTENTION, _lib.RL_LAYER_FULL_ATTENTION], [delta, attn], n_pages=2, n_slots=2, n_q=6,
                       n_kv=1, n_k=2, n_v=6)
    table, base, parents = _i32([[0], [1]]), _i32([0, 0]), _tree(gen, 2, 6, 2).cuda()
    _, pending = stack.verify_tree(torch.randn(2, 6, 128, generator=gen).cuda(), table, base, parents, _i32([3, 6]))
    _lib.check_device()
    taken = stack.commit_tree(pending, table, base, parents, _i32([3, 5]))
    assert _lib.device_error() == 6
    assert taken.tolist() == [0, len(_path(parents[1].tolist(), 5))]
    assert not stack.layers[0].S[0].any() and not stack.layers[0].conv_state[0].any() and stack.layers[0].S[1].any()


@pytest.mark.parametrize("attn_first", [False, True])
def test_chains_through_a_stack(attn_first):
    """parents None in verify and commit of a stack with both kinds of layer is the chain written out."""
    from rapidllm_b200 import _lib, ops
    from rapidllm_b200.mixer import MixerStack
    gen = torch.Generator().manual_seed(45)
    attn, delta = _weights(gen, 128)
    B, n = 2, 7
    kinds = [(_lib.RL_LAYER_FULL_ATTENTION, attn), (_lib.RL_LAYER_LINEAR_ATTENTION, delta)]
    if not attn_first:
        kinds.reverse()
    x = torch.randn(B, n, 128, generator=gen).cuda()
    chain = (torch.arange(n) - 1).int().expand(B, n).contiguous().cuda()
    table, base, counts, leaf = _i32([[1, 2], [3, 0]]), _i32([61, 5]), _i32([7, 4]), _i32([5, 3])
    results = []
    for parents in (chain, None):
        stack = MixerStack([k for k, _ in kinds], [w for _, w in kinds], n_pages=4, n_slots=B, n_q=6, n_kv=1, n_k=2, n_v=6)
        y, pending = stack.verify_tree(x, table, base, parents, counts)
        taken = stack.commit_tree(pending, table, base, parents, leaf)
        _lib.check_device()
        assert taken.tolist() == [6, 4]
        d, a = stack.layers[attn_first], stack.layers[not attn_first]
        results.append([y[0], y[1, :4], d.S, d.conv_state, a.k_pool, a.v_pool])
        with pytest.raises(_lib.RlError):
            stack.commit_tree(pending[:1], table, base, parents, leaf)
        with pytest.raises(_lib.RlError):                     # before the first layer has moved
            stack.commit_tree(pending, table, base, n, leaf)
    for a, b in zip(*results):
        assert torch.equal(a, b)
    with pytest.raises(_lib.RlError):
        ops.kv_tree_commit(results[0][4], results[0][5], table, base, None, leaf)


@pytest.mark.parametrize("n_v,n_k", [(3, 1), (5, 5), (2, 1)])
def test_delta_mixer_with_odd_head_counts(n_v, n_k):
    """A chain through verify_tree and commit_tree equals decode steps, whatever the row of the projection (a multiple of 4
    floats or not)."""
    from rapidllm_b200 import _lib
    from rapidllm_b200.mixer import DeltaNetMixer
    torch.backends.cuda.matmul.allow_tf32 = False
    gen = torch.Generator().manual_seed(46)
    _, delta = _weights(gen, 128, nk=n_k, nv=n_v)
    B, n = 2, 5
    x = torch.randn(B, n, 128, generator=gen).cuda()
    a, b = (DeltaNetMixer(delta, n_k=n_k, n_v=n_v, n_slots=B) for _ in range(2))
    y, pending = a.verify_tree(x, None)
    a.commit_tree(pending, None, _i32([n - 1, n - 1]))
    want = torch.stack([b.decode(x[:, i].contiguous()) for i in range(n)], 1)
    _lib.check_device()
    assert rel_l2(y.cpu(), want.cpu()) <= STATE_REL_L2
    assert rel_l2(a.S.cpu(), b.S.cpu()) <= STATE_REL_L2 and rel_l2(a.conv_state.cpu(), b.conv_state.cpu()) <= STATE_REL_L2


def test_drafts_of_no_nodes():
    """A round in which nothing was drafted goes through verify and commit and changes nothing."""
    from rapidllm_b200 import _lib
    from rapidllm_b200.mixer import MixerStack
    gen = torch.Generator().manual_seed(47)
    attn, delta = _weights(gen, 128)
    stack = MixerStack([_lib.RL_LAYER_LINEAR_ATTENTION, _lib.RL_LAYER_FULL_ATTENTION], [delta, attn], n_pages=2, n_slots=2, n_q=6,
                       n_kv=1, n_k=2, n_v=6)
    table, base = _i32([[0], [1]]), _i32([3, 9])
    for B, n in ((2, 0), (0, 3)):
        parents = torch.zeros(B, n, dtype=torch.int32, device="cuda")
        y, pending = stack.verify_tree(torch.zeros(B, n, 128, device="cuda"), table[:B], base[:B], parents)
        assert y.shape == (B, n, 128)
        taken = stack.commit_tree(pending, table[:B], base[:B], parents, _i32([-1] * B))
        assert taken.tolist() == [0] * B
    _lib.check_device()
    assert not stack.layers[0].S.any() and not stack.layers[1].k_pool.any()


@pytest.mark.parametrize("o_type", [torch.float16, torch.bfloat16])
def test_fp32_queries_keep_their_digits(o_type):
    """Two tokens of all but equal scores, which meet different halves of the query: one half is 0.98 half steps of fp16
    above a value of fp16, the other on it.  A query of one fp16 term would lose the difference of the scores, 64 x 0.98 x
    2^-11, of which the output is a quarter each way (V is 1 and -1).  Two terms of 2^-22 and the sums of 256 products in
    fp32 leave at most 2^-16 of the score, whatever the output's type."""
    from rapidllm_b200 import _lib, ops
    n_q, n_kv, n = 24, 4, 3
    k, v = torch.zeros(2 + n, n_kv, HD), torch.zeros(2 + n, n_kv, HD)
    k[0, :, :128], k[1, :, 128:], k[2:] = 1.0, 1.0, -1.0
    v[0], v[1], v[2:] = 1.0, -1.0, 1.0
    kp, vp, table = ops.new_pool(2, n_kv), ops.new_pool(2, n_kv), _i32([[1]])
    ops.kv_append(kp, vp, table[0], k.half().cuda(), v.half().cuda(), pos0=0)
    q = torch.full((1, n, n_q, HD), 8.0)
    q[..., :128] *= 1 + 0.98 * 2.0 ** -11
    got = ops.attn_tree(q.cuda(), kp, vp, table, _i32([2]), out_dtype=o_type)
    _lib.check_device()
    o, mag, _ = _attn_exact(q[0], None, (k.half(), v.half()), 2, [-1, 0, 1], n, n_q, n_kv)
    assert (o > 0.015).all()
    bound = (2 * math.expm1(64 * 2.0 ** -16) + 2.0 ** -11 + 2.0 ** -15) * mag + HALF_STEP[o_type] * o.abs()
    assert ((got[0].cpu().double() - o).abs() <= bound).all()


@pytest.mark.parametrize("gap", [12.0, 17.5, 22.0])
@pytest.mark.parametrize("base,batch,n_kv", [(700, 1, 1), (40000, 1, 1), (3000, 40, 4)])      # the last: a CTA has whole sequences
def test_many_small_weights_count(gap, base, batch, n_kv):
    """One token takes all but a little of the weight and has V = 0; the output is what is left for the many others, whose
    weights e^-gap are below fp16's range for a largest weight of 1 (2^-17, 2^-25, 2^-32).  Weights are held as fp16 under a
    scale of at least 2^7, an absolute error of 2^-32 of the largest each."""
    from rapidllm_b200 import _lib, ops
    n_q, n = 6 * n_kv, 2
    k, v = torch.zeros(base + n, n_kv, HD), torch.ones(base + n, n_kv, HD)
    k[base // 3] = gap / 16
    v[base // 3] = 0.0
    pages = (base + n + 63) // 64
    kp, vp = ops.new_pool(pages, n_kv), ops.new_pool(pages, n_kv)
    table = torch.arange(pages, dtype=torch.int32, device="cuda").flip(0).repeat(batch, 1)     # one cache, many drafts
    ops.kv_append(kp, vp, table[0], k.half().cuda(), v.half().cuda(), pos0=0)
    q = torch.ones(batch, n, n_q, HD, dtype=torch.float16)
    got = ops.attn_tree(q.cuda(), kp, vp, table, _i32([base] * batch))
    _lib.check_device()
    o, mag, _ = _attn_exact(q[0], None, (k.half(), v.half()), base, [-1, 0], n, n_q, n_kv)
    bound = (2.0 ** -11 + 2.0 ** -15) * mag + base * 2.0 ** -32 + HALF_STEP[torch.float16] * o + 2.0 ** -25
    assert ((got.cpu().double() - o).abs() <= bound).all(), (got[0, 0, 0, 0].item(), o[0, 0, 0].item())


@pytest.mark.parametrize("rot", [64, 256])
def test_append_can_rotate_as_qk_prepare_does(rot):
    """With angle_f32, q, K and V are those of attn_qk_prepare and kv_append at any position, bit for bit: the same sum of
    the norm, the same angle, the same roundings."""
    from rapidllm_b200 import _lib, ops
    gen = torch.Generator().manual_seed(48)
    pos, n, n_q, n_kv = [0, 63, 130001, 16777300], 6, 12, 2
    B = len(pos)
    table = torch.full((B, max(pos) // 64 + 2), -1, dtype=torch.int32)
    for b, p in enumerate(pos):
        table[b, p // 64], table[b, p // 64 + 1] = 2 * b, 2 * b + 1
    table = table.cuda()
    qg, k, v = (torch.randn(B, n, h, d, generator=gen).cuda() for h, d in ((n_q, 512), (n_kv, HD), (n_kv, HD)))
    qn, kn = (0.2 * torch.randn(HD, generator=gen).cuda() for _ in range(2))
    pools = [ops.new_pool(2 * B, n_kv) for _ in range(4)]
    q, gate = ops.attn_qk_append(qg, k, v, *pools[:2], table, _i32(pos), qn, kn, rotary_dim=rot, angle_f32=True)
    at = (_i32(pos).unsqueeze(1) + torch.arange(n, dtype=torch.int32, device="cuda")).reshape(-1).contiguous()
    rotated = k.reshape(B * n, n_kv, HD).clone()
    want, want_gate = ops.attn_qk_prepare(qg.reshape(B * n, n_q, 512), rotated, qn, kn, pos=at, rotary_dim=rot)
    for b, p in enumerate(pos):
        ops.kv_append(*pools[2:], table[b], rotated.view(B, n, n_kv, HD)[b].contiguous(), v[b].contiguous(), pos0=p)
    _lib.check_device()
    assert torch.equal(gate.view_as(want_gate), want_gate) and torch.equal(q.view_as(want), want)
    assert torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3])


def test_attention_mixer_far_into_a_context():
    """A chain through verify_tree behind 100 003 tokens writes the cache rows of as many decode steps and gives their
    outputs: queries of 16 times the usual norm, so that scores spread over +- 50 and their rounding counts (P and the
    output in fp16, 2^-11 each, remain).  The rows differ by what the projections do, whose GEMMs have another number of
    rows: sums of 128 products in another order, 2 x 128 x 2^-24 of magnitudes that are 5 times the sum, 1e-4 of a row's
    root mean square, and the step of fp16 that this may move (an angle of another rule, 4e-3 rad, is far above)."""
    from rapidllm_b200 import _lib
    from rapidllm_b200.mixer import GatedAttentionMixer
    torch.backends.cuda.matmul.allow_tf32 = False
    gen = torch.Generator().manual_seed(49)
    weights, _ = _weights(gen, 128)
    weights["q_norm"] = torch.full((HD,), 15.0)
    base, n = 100003, 5
    pages = (base + n + 63) // 64
    table = torch.randperm(pages, generator=gen).int().view(1, -1).cuda()
    x = torch.randn(1, n, 128, generator=gen).cuda()
    mixers = [GatedAttentionMixer(weights, n_pages=pages, n_q=6, n_kv=1) for _ in range(2)]
    for m in mixers:
        fill = torch.Generator(device="cuda").manual_seed(50)
        for pool in (m.k_pool, m.v_pool):
            pool.copy_(torch.randn(pool.shape, generator=fill, device="cuda"))
    y = mixers[0].verify_tree(x, table, _i32([base]), None)
    want = torch.stack([mixers[1].decode(x[:, i].contiguous(), table, _i32([base + i])) for i in range(n)], 1)
    _lib.check_device()
    for a, b in zip(*([m.k_pool, m.v_pool] for m in mixers)):
        for i in range(n):
            got, ref = (_pool_row(p, table, 0, base + i).float() for p in (a, b))
            assert ((got - ref).abs() <= 2.0 ** -10 * ref.abs() + 1e-4 * ref.square().mean().sqrt()).all(), i
    assert rel_l2((y - x).cpu(), (want - x).cpu()) <= 2.0 ** -10


@pytest.mark.parametrize("n_v,n_qk,tiled,nodes,width", [
    (48, 16, False, 13, 3), (48, 16, True, 16, 1), (48, 16, False, 21, 4), (32, 16, True, 32, 6), (48, 16, False, 40, 3),
    (64, 16, True, 48, 8), (48, 16, False, 64, 1), (48, 16, True, 63, 5), (64, 64, False, 20, 2),
])
def test_gdn_tree_of_a_full_batch(n_v, n_qk, tiled, nodes, width):
    """Value heads one after the other in a CTA (every size of the kernel, both orders of heads): ragged counts, an empty
    draft and one of a single node among them."""
    from rapidllm_b200 import _lib, ops
    gen = torch.Generator().manual_seed(nodes * 10 + n_v + tiled)
    batch = _full_batch(n_v)
    S, win, qkv, w, beta, g = _gdn_inputs(gen, batch, nodes, n_v, n_qk, batch)
    parents = _tree(gen, batch, nodes, width)
    counts = [max(1, nodes - 5 * b) for b in range(batch)]
    counts[1], counts[2] = 0, 1
    out = torch.full((batch, nodes, n_v, DK), 5.0, device="cuda")
    ops.gdn_tree(*(t.cuda() for t in (S, win)), None, *(t.cuda() for t in (qkv, w, beta, g, parents)), n_qk, n_nodes=_i32(counts),
                 head_map=_lib.RL_HEADS_TILED if tiled else _lib.RL_HEADS_GROUPED, out=out)
    _lib.check_device()
    for b in range(batch):
        assert (out[b, counts[b]:] == 5.0).all()
        if counts[b]:
            want = _gdn_tree_exact(S[b], win[b], qkv[b], w, beta[b], g[b], parents[b].tolist(), counts[b], n_qk, tiled)
            got = out[b, :counts[b]].cpu()
            for h in range(n_v):
                assert rel_l2(got[:, h], want[:, h]) <= STATE_REL_L2, (b, h)


@pytest.mark.parametrize("n_v,n_qk,tiled,nodes", [(48, 16, False, 14), (48, 16, True, 30), (48, 16, False, 45), (32, 16, False, 64)])
def test_gdn_tree_bad_nodes_and_closed_gates_of_a_full_batch(n_v, n_qk, tiled, nodes):
    """In every head of a CTA, the first and the later ones: inputs that are not finite reach their node's descendants in
    the heads concerned alone, and gates that forget everything cost no digits behind them."""
    from rapidllm_b200 import _lib, ops
    gen = torch.Generator().manual_seed(51)
    batch, ratio = _full_batch(n_v), n_v // n_qk
    S, win, qkv, w, beta, g = _gdn_inputs(gen, batch, nodes, n_v, n_qk, batch)
    parents = _tree(gen, batch, nodes, 6)
    heads = [h for h in range(n_v) if (h % n_qk if tiled else h // ratio) == 2]       # those of key head 2, in a CTA's order
    qkv[0, 5, 2 * DK + 3] = math.inf                          # q of key head 2
    qkv[1, 7, n_qk * DK + 2 * DK + 9] = math.nan              # its k
    for z, h in enumerate(heads):
        qkv[2, 3 + z, 2 * n_qk * DK + h * DK + 17 * z] = math.nan                     # a column of each value head
        beta[3, 4 + z, h] = math.nan
        g[3, 8 + z, h] = math.inf
        g[4, 1 + 2 * z::5, h] = (-60.0, -5000.0, -math.inf, -90.0)[z]
    o = ops.gdn_tree(*(t.cuda() for t in (S, win)), None, *(t.cuda() for t in (qkv, w, beta, g, parents)), n_qk,
                     head_map=_lib.RL_HEADS_TILED if tiled else _lib.RL_HEADS_GROUPED).cpu()
    _lib.check_device()
    for b in range(batch):
        want = _gdn_tree_exact(S[b], win[b], qkv[b], w, beta[b], g[b], parents[b].tolist(), nodes, n_qk, tiled)
        fine = torch.isfinite(want)
        assert fine.all() == (b > 3) and torch.equal(torch.isfinite(o[b]), fine), b
        for h in range(n_v):
            assert rel_l2(o[b, :, h][fine[:, h]], want[:, h][fine[:, h]]) <= STATE_REL_L2, (b, h)


@pytest.mark.parametrize("up", [10, 20])
@pytest.mark.parametrize("full", [False, True])
def test_gdn_tree_of_siblings_of_unequal_size(up, full):
    """One sibling's v 2^up times the others'.  A value is held to 2^-22 of itself or 2^-39 of the largest of its column (two
    fp16 terms under one scale), twice: in W and in U.  With 2^20 that is 2 x 2^-19 = 4e-6 of the others' v, within the
    tolerance of a node's whole output; their outputs are of v's size, since the state is small here."""
    from rapidllm_b200 import _lib, ops
    gen = torch.Generator().manual_seed(52)
    n_v, n_qk, nodes = (48, 16, 24) if full else (6, 2, 24)
    batch = _full_batch(n_v) if full else 2
    S, win, qkv, w, beta, g = _gdn_inputs(gen, batch, nodes, n_v, n_qk, batch)
    S *= 0.1
    parents = torch.full((batch, nodes), -1, dtype=torch.int32)
    parents[:, 12:] = torch.arange(12).int()                  # twelve roots, a child each
    v0 = 2 * n_qk * DK
    qkv[:, 4, v0:] = qkv[:, 4, v0:].abs() * 2.0 ** up         # (SiLU takes large positive values as they are)
    w[v0:] = w[v0:].abs()
    qkv[:, 16, v0:] = qkv[:, 3, v0:]
    o = ops.gdn_tree(*(t.cuda() for t in (S, win)), None, *(t.cuda() for t in (qkv, w, beta, g, parents)), n_qk).cpu()
    _lib.check_device()
    for b in range(batch):
        want = _gdn_tree_exact(S[b], win[b], qkv[b], w, beta[b], g[b], parents[b].tolist(), nodes, n_qk, False)
        small = [i for i in range(nodes) if i not in (4, 16)]
        assert want[4].abs().mean() > 2.0 ** (up - 4) * want[small].abs().mean()
        for h in range(n_v):
            assert rel_l2(o[b, small, h], want[small, h]) <= STATE_REL_L2, (b, h)
            assert rel_l2(o[b, [4, 16], h], want[[4, 16], h]) <= STATE_REL_L2, (b, h)


def test_a_tree_on_the_device_cache():
    """Pools, states, conv rings and their phases of a HybridCache: a tree verified and one path committed through its views
    equal the cache's own decode steps along that path, and the next decode step goes on from there."""
    from rapidllm_b200 import _lib, ops
    from rapidllm_b200.cache import HybridCache
    gen = torch.Generator().manual_seed(53)
    kinds = [_lib.RL_LAYER_LINEAR_ATTENTION, _lib.RL_LAYER_FULL_ATTENTION]
    B, n, history, lens = 2, 9, 3, [60, 130]
    cache = HybridCache(kinds, n_pages=6, n_slots=3, max_batch=2, max_pages_per_seq=3)
    table, slots = _i32([[4, 0, -1], [2, 5, 1]]), _i32([2, 0])
    sh = cache.io_shapes(B)
    conv_w = torch.randn(sh["conv_w"], generator=gen).cuda() * 0.5
    parents = _tree(gen, 1, n, 3).repeat(B, 1)
    path = _path(parents[0].tolist(), n - 1)

    def token():
        t = {x: torch.randn(sh[x], generator=gen).cuda() for x in ("attn_q", "attn_gate", "attn_k", "attn_v", "delta_qkv")}
        t["delta_beta"] = torch.sigmoid(torch.randn(sh["delta_beta"], generator=gen)).cuda()
        t["delta_g"] = -0.3 * torch.rand(sh["delta_g"], generator=gen).cuda()
        return t

    def step(t, at):
        io = dict(t, attn_o=torch.zeros(sh["attn_o"], device="cuda"), delta_o=torch.zeros(sh["delta_o"], device="cuda"),
                  conv_w=conv_w, page_table=table, slot_ids=slots, pos=_i32(at))
        cache.decode(io, B)
        torch.cuda.synchronize()
        return io["attn_o"][0].clone(), io["delta_o"][0].clone()

    for pool in (cache.k_pool(0), cache.v_pool(0)):
        pool.copy_(torch.randn(pool.shape, generator=gen))
    for d in range(history):                                  # the rings' phases leave 0
        step(token(), [x + d for x in lens])
    base = [x + history for x in lens]
    views = [cache.k_pool(0), cache.v_pool(0), cache.state(0), cache.conv(0), cache.conv_phase(0)]
    kept = [v.clone() for v in views]
    assert views[4][slots.long()].tolist() == [history % 4] * B
    nodes, nxt = [token() for _ in range(n)], token()
    want = [step(nodes[i], [x + d for x in base]) for d, i in enumerate(path)]
    after = [cache.state(0).clone(), cache.conv_windows(0)]
    want_next = step(nxt, [x + len(path) for x in base])
    for v, was in zip(views, kept):
        v.copy_(was)

    rows = lambda x: torch.stack([t[x][0] for t in nodes], 1).contiguous()  # noqa: E731
    k, v = rows("attn_k"), rows("attn_v")
    for b in range(B):
        ops.kv_append(*views[:2], table[b], k[b], v[b], pos0=base[b])
    o = ops.attn_tree(rows("attn_q"), *views[:2], table, _i32(base), parents.cuda(), gate=rows("attn_gate"))
    gdn = (*views[2:], rows("delta_qkv"), conv_w[0], rows("delta_beta"), rows("delta_g"), parents.cuda())
    do = ops.gdn_tree(*gdn, n_qk=16, slot_ids=slots)
    leaf = _i32([n - 1] * B)
    taken = ops.kv_tree_commit(*views[:2], table, _i32(base), parents.cuda(), leaf)
    ops.gdn_tree_commit(*gdn, leaf, n_qk=16, slot_ids=slots)
    _lib.check_device()
    assert taken.tolist() == [len(path)] * B
    for d, i in enumerate(path):
        assert rel_l2(o[:, i].float().cpu(), want[d][0].cpu()) <= 1e-3
        assert rel_l2(do[:, i].cpu(), want[d][1].cpu()) <= STATE_REL_L2
    assert rel_l2(cache.state(0).cpu(), after[0].cpu()) <= STATE_REL_L2
    assert torch.equal(cache.conv_windows(0), after[1])
    got = step(nxt, [x + len(path) for x in base])
    assert rel_l2(got[0].cpu(), want_next[0].cpu()) <= 1e-3 and rel_l2(got[1].cpu(), want_next[1].cpu()) <= STATE_REL_L2
    cache.close()


def test_attn_tree_of_the_largest_batch():
    """512 sequences, most of them short: every eighth against 64 bits; 513 are refused.  The same call again gives the same
    bits; a tight bound of the lengths (another division of the work) the same values."""
    from rapidllm_b200 import _lib, ops
    gen = torch.Generator().manual_seed(54)
    B, n, n_q, n_kv = 512, 5, 12, 2
    base = [(b * 37) % 150 for b in range(B)]
    base[100], base[511] = 3000, 1100
    counts = [(b * 3) % (n + 1) for b in range(B)]
    kp, vp, table, rows = _pages(gen, base, counts, n_kv, float("nan"))
    parents, q = _tree(gen, B, n, 3), torch.randn(B, n, n_q, HD, generator=gen).half()
    args = (q.cuda(), kp, vp, table, _i32(base), parents.cuda())
    out = [torch.full((B, n, n_q, HD), 5.0, dtype=torch.float16, device="cuda") for _ in range(3)]
    ops.attn_tree(*args, n_nodes=_i32(counts), out=out[0])
    ops.attn_tree(*args, n_nodes=_i32(counts), out=out[1])
    ops.attn_tree(*args, n_nodes=_i32(counts), out=out[2], max_seq_len=max(x + c for x, c in zip(base, counts)))
    _lib.check_device()
    assert torch.equal(out[0], out[1])
    assert rel_l2(out[2].float().cpu(), out[0].float().cpu()) <= 2.0 ** -11
    for b in [*range(0, B, 8), 100, 511]:
        assert (out[0][b, counts[b]:] == 5.0).all()
        if counts[b]:
            o, _, _ = _attn_exact(q[b], None, rows[b], base[b], parents[b].tolist(), counts[b], n_q, n_kv)
            assert rel_l2(out[0][b, :counts[b]].float().cpu(), o) <= 1e-3, b
    with pytest.raises(_lib.RlError):
        ops.attn_tree(torch.cat([args[0], args[0][:1]]), kp, vp, torch.cat([table, table[:1]]), _i32(base + [0]), None)


def test_rounds_on_two_streams():
    """Delta rule and commits of two groups of slots on streams of their own, round after round, give what one stream
    gives."""
    from rapidllm_b200 import _lib, ops
    gen = torch.Generator().manual_seed(55)
    n_v, n_qk, n, half = 6, 2, 11, 3
    S, win, qkv, w, beta, g = (t.cuda() for t in _gdn_inputs(gen, 2 * half, n, n_v, n_qk, 2 * half))
    parents, leaf, counts = _tree(gen, 2 * half, n, 3).cuda(), _i32([10, 4, -1, 0, 6, 3]), _i32([11, 5, 3, 1, 7, 4])
    slots = _i32([4, 0, 2, 5, 1, 3])

    def rounds(state, window, part):
        cut = [t[part].contiguous() for t in (qkv, beta, g, parents, leaf, counts, slots)]
        got = []
        for _ in range(6):
            got.append(ops.gdn_tree(state, window, None, cut[0], w, cut[1], cut[2], cut[3], n_qk, slot_ids=cut[6]))
            ops.gdn_tree_commit(state, window, None, cut[0], w, cut[1], cut[2], cut[3], cut[4], n_qk, slot_ids=cut[6], n_nodes=cut[5])
        return got

    parts = [slice(0, half), slice(half, 2 * half)]
    one = [S.clone(), win.clone()]
    want = [rounds(*one, p) for p in parts]
    two = [S.clone(), win.clone()]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in parts], []
    for s, p in zip(streams, parts):
        with torch.cuda.stream(s):
            got.append(rounds(*two, p))
    torch.cuda.synchronize()
    _lib.check_device()
    for a, b in zip(one, two):
        assert torch.equal(a, b)
    for a, b in zip(want, got):
        for x, y in zip(a, b):
            assert torch.equal(x, y)
