"""Trees of drafted tokens (attn_qk_append, attn_tree, kv_tree_commit, gdn_tree, gdn_tree_commit) against
plain implementations in 64 bits, node by node along each path.

Tolerances, from the arithmetic:
  * fp32 results of attn_qk_append: the square sum of 256 values in fp32 (8 fused steps and 5 pairwise
    additions, halved by the root), about 8 more roundings, sine and cosine within 2 ulp: 32 * 2^-24 of the
    row's largest value.  Rounded results add half a step: fp16 2^-11, bf16 2^-8 of the value.
  * attn_tree: P rounded to fp16 (2^-11), the query rounded to fp16 (2^-11 of each product: the score is off by
    at most e = 2^-11 sum |q k| / 16, both numerator and denominator by a factor exp(e)), exponential, sums and
    gate within 2^-16; all of it relative to sum p |v|.  Computed per row from the inputs.
  * the delta rule: fp32 sums of 128 terms, at worst 128 * 2^-24 = 7.6e-6 of the magnitudes; relative L2 1e-5,
    as for the other forms of the rule.
"""
import math

import pytest
import torch

from helpers import ATTN_MAX_ABS, ATTN_REL_L2, STATE_REL_L2, rel_l2

pytestmark = pytest.mark.gpu

HD, DK = 256, 128
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 0.0}


def _path(parents, i):
    p = []
    while i >= 0:
        p.append(i)
        i = parents[i]
    return p[::-1]


def _tree(gen, batch, nodes, width):
    rows = []
    for _ in range(batch):
        rows.append([i - 1 - int(torch.randint(0, min(width, i) or 1, (1,), generator=gen)) if i else -1 for i in range(nodes)])
        if nodes > 4 and width > 1:
            rows[-1][3] = -1                                  # a second root
    return torch.tensor(rows, dtype=torch.int32)


def _pages(gen, base, extra, n_kv, fill):
    """Pools of random rows; `fill` in every row behind a sequence's last.  Returns pools, table and the rows."""
    from rapidllm_b200 import ops
    counts = [(b + e + 63) // 64 for b, e in zip(base, extra)]
    total = sum(counts) + 2
    perm = torch.randperm(total, generator=gen).int()
    table = torch.full((len(base), max(1, max(counts))), -1, dtype=torch.int32)
    at = 0
    kp, vp = ops.new_pool(total, n_kv), ops.new_pool(total, n_kv)
    kp.fill_(fill)
    vp.fill_(fill)
    rows = []
    for b, c in enumerate(counts):
        table[b, :c] = perm[at:at + c]
        at += c
    table = table.cuda()
    for b in range(len(base)):
        n = base[b] + extra[b]
        k = torch.randn(n, n_kv, HD, generator=gen).half()
        v = torch.randn(n, n_kv, HD, generator=gen).half()
        rows.append((k, v))
        if n:
            ops.kv_append(kp, vp, table[b], k.cuda(), v.cuda(), pos0=0)
    return kp, vp, table, rows


def _rotated(x, position, rot, theta):
    half = rot // 2
    if half:
        ang = position.double().view(-1, 1, 1) * theta ** (-torch.arange(half, dtype=torch.float64) / half)
        a, b = x[..., :half].clone(), x[..., half:rot].clone()
        x[..., :half] = a * ang.cos() - b * ang.sin()
        x[..., half:rot] = a * ang.sin() + b * ang.cos()
    return x


@pytest.mark.parametrize("n_q,n_kv,batch,n_tok,rot,q_type,tree,norms,pos", [
    (24, 4, 1, 1, 64, torch.float32, False, True, [0]),
    (24, 4, 3, 1, 64, torch.float16, False, True, [63, 64, 130001]),
    (24, 4, 2, 64, 64, torch.float16, True, True, [17, 100000]),
    (24, 4, 3, 21, 64, torch.bfloat16, True, False, [5, 0, 999]),
    (6, 1, 2, 13, 128, torch.float32, True, True, [1, 40]),
    (8, 8, 1, 130, 256, torch.float32, False, True, [31]),
    (12, 2, 1, 70, 0, torch.float16, False, True, [0]),
    (16, 2, 1, 33, 16, torch.bfloat16, False, True, [7]),
    (1, 1, 2, 3, 32, torch.float32, True, True, [62, 126]),
])
def test_append(n_q, n_kv, batch, n_tok, rot, q_type, tree, norms, pos):
    from rapidllm_b200 import _lib, ops
    gen = torch.Generator().manual_seed(n_q * 1000 + n_tok)
    theta, eps = 1e7, 1e-6
    extra = [n_tok] * batch
    n_pages = sum((p + n_tok - 1) // 64 - p // 64 + 1 for p in pos) + 1
    table = torch.full((batch, max((p + n_tok + 63) // 64 for p in pos)), -1, dtype=torch.int32)
    perm, at = torch.randperm(n_pages, generator=gen).int(), 0
    for b, p in enumerate(pos):
        for i in range(p // 64, (p + n_tok - 1) // 64 + 1):
            table[b, i] = perm[at]
            at += 1
    table = table.cuda()
    proj = torch.randn(batch, n_tok, (2 * n_q + 2 * n_kv) * HD, generator=gen)
    pc = proj.cuda()
    cut = lambda t, lo, heads, w: t[..., lo * HD:lo * HD + heads * w].view(batch, n_tok, heads, w)  # noqa: E731
    parts = [(0, n_q, 2 * HD), (2 * n_q, n_kv, HD), (2 * n_q + n_kv, n_kv, HD)]
    qg, k, v = (cut(pc, *x) for x in parts)
    qn, kn = (torch.randn(HD, generator=gen) * 0.2, torch.randn(HD, generator=gen) * 0.2) if norms else (None, None)
    parents = _tree(gen, batch, n_tok, 4) if tree else None
    counts = [max(1, n_tok - 2 * b) for b in range(batch)] if tree else [n_tok] * batch
    kp, vp = ops.new_pool(n_pages, n_kv), ops.new_pool(n_pages, n_kv)
    kp.fill_(7.0)
    vp.fill_(7.0)
    q_out = torch.full((batch, n_tok, n_q, HD), 3.0, dtype=q_type, device="cuda")
    gate_out = torch.full((batch, n_tok, n_q, HD), 3.0, device="cuda")
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    args = (qg, k, v, kp, vp, table, torch.tensor(pos, dtype=torch.int32, device="cuda"), dev(qn), dev(kn))
    kw = dict(parents=dev(parents), n_nodes=torch.tensor(counts, dtype=torch.int32, device="cuda") if tree else None,
              rotary_dim=rot, theta=theta, eps=eps)
    ops.attn_qk_append(*args, q_out=q_out, gate_out=gate_out, **kw)
    _lib.check_device()
    assert torch.equal(pc.cpu(), proj)                        # the projection is only read
    touched = torch.zeros(n_pages, 64, dtype=torch.bool)
    for b in range(batch):
        n = counts[b]
        depth = [len(_path(parents[b].tolist(), i)) - 1 for i in range(n)] if tree else list(range(n))
        position = torch.tensor([pos[b] + d for d in depth])
        qg64, k64, v64 = (cut(proj, *x)[b, :n].double() for x in parts)
        got_k = torch.stack([_pool_row(kp, table, b, pos[b] + t) for t in range(n)]).cpu().double()
        got_v = torch.stack([_pool_row(vp, table, b, pos[b] + t) for t in range(n)]).cpu()
        for t in range(n):
            touched[int(table[b, (pos[b] + t) // 64]), (pos[b] + t) % 64] = True
        for x, w, got, step in ((qg64[..., :HD], qn, q_out[b, :n].cpu().double(), HALF_STEP[q_type]),
                                (k64, kn, got_k, HALF_STEP[torch.float16])):
            y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
            y = _rotated(y * (1 + w.double()) if w is not None else y.clone(), position, rot, theta)
            bound = step * y.abs() + 32 * 2.0 ** -24 * y.abs().amax(-1, keepdim=True)
            assert ((got - y).abs() <= bound * (1 + 1e-3) + 2.0 ** -25).all(), (b, ((got - y).abs() / bound).max())
        assert torch.equal(got_v, v64.half())
        assert torch.equal(gate_out[b, :n].cpu(), qg64[..., HD:].float())
        assert (q_out[b, n:] == 3.0).all() and (gate_out[b, n:] == 3.0).all()
    untouched = ~touched
    for pool in (kp, vp):
        assert (_unswizzled(pool).cpu().permute(0, 2, 1, 3)[untouched] == 7.0).all()
    q2, g2 = ops.attn_qk_append(*args, q_dtype=q_type, want_gate=False, **kw)
    assert g2 is None
    for b in range(batch):
        assert torch.equal(q2[b, :counts[b]], q_out[b, :counts[b]])


def _unswizzled(pool):
    """[pages][n_kv][64][256] of a pool."""
    from rapidllm_b200 import ops
    tok, d = torch.arange(64).view(64, 1), torch.arange(HD).view(1, HD)
    return pool[:, :, ops.kv_slice_index(tok, d).to(pool.device)]


def _pool_row(pool, table, b, position):
    from rapidllm_b200 import ops
    page = int(table[b, position // 64])
    return pool[page][:, ops.kv_slice_index(torch.full((HD,), position % 64), torch.arange(HD)).to(pool.device)]


def _attn_exact(q, gate, rows, base, parents, n, n_q, n_kv):
    """(o, sum p|v| gate, score error bound) of one sequence in 64 bits."""
    k, v = rows[0].double(), rows[1].double()
    G = n_q // n_kv
    hidden = torch.ones(n, base + n, dtype=torch.bool)
    hidden[:, :base] = False
    for i in range(n):
        hidden[i, [base + j for j in _path(parents, i)]] = False
    o, mag, err = [], [], []
    for h in range(n_q):
        s = q[:n, h].double() @ k[:base + n, h // G].T / 16
        p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
        gt = torch.sigmoid(gate[:n, h].double()) if gate is not None else 1.0
        vv = v[:base + n, h // G]
        o.append(torch.where(p > 0, p, 0.0) @ vv * gt)
        mag.append(p @ vv.abs() * gt)
        err.append((q[:n, h].double().abs() @ k[:base + n, h // G].abs().T / 16).masked_fill(hidden, 0.0).amax(-1) * 2.0 ** -11)
    return torch.stack(o, 1), torch.stack(mag, 1), torch.stack(err, 1)


@pytest.mark.parametrize("n_q,n_kv,nodes,base,counts,width,q_type,o_type,gated", [
    (24, 4, 1, [0], [1], 1, torch.float32, torch.float16, False),            # nothing committed, one node
    (24, 4, 8, [100], [8], 3, torch.float16, torch.float16, True),
    (24, 4, 21, [63, 0, 4001], [21, 20, 0], 4, torch.bfloat16, torch.bfloat16, True),   # one row tile; an empty draft
    (24, 4, 22, [64, 42, 43], [22, 1, 21], 4, torch.float32, torch.bfloat16, True),     # a second row tile; page edges
    (24, 4, 64, [700, 1], [64, 63], 6, torch.float32, torch.float16, True),  # three row tiles, two pages of nodes
    (16, 2, 64, [129, 0], [64, 33], 8, torch.float16, torch.float16, False),  # group of 8: four row tiles
    (8, 8, 5, [3000], [5], 2, torch.float32, torch.float16, True),            # group of 1
    (6, 1, 13, [20000], [13], 1, torch.bfloat16, torch.float16, True),        # a chain, one head over many CTAs
    (12, 2, 40, [50] * 37, [40 - b for b in range(37)], 3, torch.float16, torch.bfloat16, True),   # more heads than CTAs
])
def test_attn_tree(n_q, n_kv, nodes, base, counts, width, q_type, o_type, gated):
    from rapidllm_b200 import _lib, ops
    gen = torch.Generator().manual_seed(nodes * 100 + n_q)
    batch = len(base)
    kp, vp, table, rows = _pages(gen, base, counts, n_kv, float("nan"))
    parents = _tree(gen, batch, nodes, width)
    q = (torch.randn(batch, nodes, n_q, HD, generator=gen) * 2).to(q_type)
    qg = torch.randn(batch, nodes, n_q, 2 * HD, generator=gen)
    gate = qg[..., HD:]
    out = torch.full((batch, nodes, n_q, HD), 5.0, dtype=o_type, device="cuda")
    dev = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    got = ops.attn_tree(q.cuda(), kp, vp, table, dev(*base), None if width == 1 else parents.cuda(), n_nodes=dev(*counts),
                        gate=qg.cuda()[..., HD:] if gated else None, out=out)
    _lib.check_device()
    assert got is out
    for b in range(batch):
        n = counts[b]
        assert (out[b, n:] == 5.0).all()
        if n:
            o, mag, err = _attn_exact(q[b], gate[b] if gated else None, rows[b], base[b], parents[b].tolist(), n, n_q, n_kv)
            bound = (2 * torch.expm1(err).unsqueeze(2) + 2.0 ** -11 + 2.0 ** -15) * mag + HALF_STEP[o_type] * o.abs() + 2.0 ** -25
            diff = (out[b, :n].cpu().double() - o).abs()
            assert (diff <= bound).all(), (b, (diff / bound).max())
            # the bound adds up worst cases; the errors do not
            assert rel_l2(out[b, :n].float().cpu(), o) <= (1e-3 if o_type == torch.float16 else 4e-3)


def test_attn_tree_large_and_tiny_queries():
    """The scale that a row is rounded under follows its magnitude: 1e-30 and 1e30 times a query give what they should
    (equal weights, and the largest score alone), rows of zeros are fine."""
    from rapidllm_b200 import ops
    gen = torch.Generator().manual_seed(5)
    kp, vp, table, rows = _pages(gen, [190], [4], 4, 0.0)
    q = torch.randn(1, 4, 24, HD, generator=gen)
    q[0, 0] *= 1e-30
    q[0, 1] *= 1e30
    q[0, 2] = 0
    parents = torch.tensor([[-1, 0, 1, 2]], dtype=torch.int32)
    got = ops.attn_tree(q.cuda(), kp, vp, table, torch.tensor([190], dtype=torch.int32, device="cuda"), parents.cuda()).cpu().double()
    k, v = rows[0][0].double(), rows[0][1].double()
    for h in range(24):
        for i in (0, 2):
            assert (got[0, i, h] - v[:191 + i, h // 6].mean(0)).abs().max() <= 2e-3
        best = (q[0, 1, h].double() @ k[:192, h // 6].T).argmax()
        assert torch.equal(got[0, 1, h], v[best, h // 6])
    o, mag, err = _attn_exact(q[0], None, rows[0], 190, parents[0].tolist(), 4, 24, 4)
    assert rel_l2(got[0, 3], o[3]) <= 1e-3


@pytest.mark.parametrize("nodes,base,leaf,width", [
    (1, [0], [0], 1),
    (8, [60, 0, 5], [7, -1, 0], 3),
    (64, [1000, 63, 1], [63, 40, 2], 2),
    (64, [10], [63], 1),                                                       # a chain stays where it is
    (33, [127, 64], [32, 31], 8),
])
def test_kv_commit(nodes, base, leaf, width):
    from rapidllm_b200 import _lib, ops
    gen = torch.Generator().manual_seed(nodes)
    batch = len(base)
    kp, vp, table, rows = _pages(gen, base, [nodes] * batch, 4, 9.0)
    parents = _tree(gen, batch, nodes, width)
    if nodes == 64 and width == 2:
        parents[0] = torch.tensor([-1] + [max(0, i - 2) for i in range(1, 64)])
    want = [pool.clone() for pool in (kp, vp)]
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    for b in range(batch):
        path = _path(parents[b].tolist(), leaf[b])
        for w, src in zip(want, (kp, vp)):
            taken = [_pool_row(src, table, b, base[b] + i).clone() for i in path]
            for j, row in enumerate(taken):
                page, at = int(table[b, (base[b] + j) // 64]), (base[b] + j) % 64
                w[page][:, ops.kv_slice_index(torch.full((HD,), at), torch.arange(HD)).cuda()] = row
    n = ops.kv_tree_commit(kp, vp, table, dev(base), parents.cuda(), dev(leaf))
    _lib.check_device()
    assert n.tolist() == [len(_path(parents[b].tolist(), leaf[b])) for b in range(batch)]
    assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])


def _gdn_inputs(gen, batch, nodes, n_v, n_qk, slots, pad=0):
    dim = 2 * n_qk * DK + n_v * DK
    S = torch.randn(slots, n_v, DK, DK, generator=gen) * 0.3
    win = torch.randn(slots, dim, 4, generator=gen)
    qkv = torch.randn(batch, nodes, dim + pad, generator=gen)
    w = torch.randn(dim, 4, generator=gen) * 0.5
    beta = torch.sigmoid(torch.randn(batch, nodes, n_v, generator=gen))
    g = -0.3 * torch.rand(batch, nodes, n_v, generator=gen)
    return S, win, qkv, w, beta, g


def _gdn_exact(S, win, qkv, w, beta, g, path, n_v, n_qk, tiled):
    """(o of the last node, state, window) after the path's steps, 64 bits; win oldest tap first."""
    qd = n_qk * DK
    hs = torch.tensor([h % n_qk if tiled else h // (n_v // n_qk) for h in range(n_v)])
    S, win, w = S.double(), win.double(), w.double()
    o = None
    for i in path:
        win = torch.cat([win[:, 1:], qkv[i].double().unsqueeze(1)], 1)
        y = (win * w).sum(1)
        y = y / (1 + torch.exp(-y))
        q, k, v = y[:qd].view(-1, DK)[hs], y[qd:2 * qd].view(-1, DK)[hs], y[2 * qd:].view(-1, DK)
        q = q / (q.square().sum(1, keepdim=True) + 1e-6).sqrt() / DK ** 0.5
        k = k / (k.square().sum(1, keepdim=True) + 1e-6).sqrt()
        S = S * g[i].double().exp().view(-1, 1, 1)
        u = beta[i].double().unsqueeze(1) * (v - torch.einsum("hd,hdv->hv", k, S))
        S = S + k.unsqueeze(2) * u.unsqueeze(1)
        o = torch.einsum("hd,hdv->hv", q, S)
    return o, S, win


GDN_SHAPES = [
    (48, 16, False, 1, [1], 1),
    (48, 16, False, 8, [8, 5], 3),
    (6, 2, True, 21, [21, 0, 17], 4),
    (4, 4, False, 64, [64, 33], 1),
    (6, 2, False, 64, [64, 63], 5),
    (3, 1, False, 16, [16, 15, 9, 1], 2),
    (2, 1, True, 33, [33, 32], 8),
    (5, 5, False, 48, [47], 3),
]


@pytest.mark.parametrize("ring", [True, False])
@pytest.mark.parametrize("n_v,n_qk,tiled,nodes,counts,width", GDN_SHAPES)
def test_gdn_tree(n_v, n_qk, tiled, nodes, counts, width, ring):
    from rapidllm_b200 import _lib, ops
    gen = torch.Generator().manual_seed(nodes * 10 + n_v)
    batch, slots = len(counts), len(counts) + 2
    S, win, qkv, w, beta, g = _gdn_inputs(gen, batch, nodes, n_v, n_qk, slots, pad=8)
    dim = w.shape[0]
    parents = _tree(gen, batch, nodes, width)
    ids = torch.randperm(slots, generator=gen)[:batch].int()
    phase = torch.randint(0, 4, (slots,), generator=gen).int() if ring else torch.zeros(slots, dtype=torch.int32)
    stored = torch.stack([torch.roll(win[s], int(phase[s]), 1) for s in range(slots)])
    head_map = _lib.RL_HEADS_TILED if tiled else _lib.RL_HEADS_GROUPED
    out = torch.full((batch, nodes, n_v, DK), 5.0, device="cuda")
    Sc, wc = S.cuda(), stored.cuda()
    ops.gdn_tree(Sc, wc, phase.cuda() if ring else None, qkv.cuda()[..., :dim], w.cuda(), beta.cuda(), g.cuda(), parents.cuda(),
                 n_qk, n_nodes=torch.tensor(counts, dtype=torch.int32, device="cuda"), slot_ids=ids.cuda(), head_map=head_map, out=out)
    _lib.check_device()
    assert torch.equal(Sc.cpu(), S) and torch.equal(wc.cpu(), stored)
    for b in range(batch):
        par = parents[b].tolist()
        want = [_gdn_exact(S[ids[b]], win[ids[b]], qkv[b, :, :dim], w, beta[b], g[b], _path(par, i), n_v, n_qk, tiled)[0]
                for i in range(counts[b])]
        assert (out[b, counts[b]:] == 5.0).all()
        if want:
            got, want = out[b, :counts[b]].cpu(), torch.stack(want)
            assert rel_l2(got, want) <= STATE_REL_L2
            for h in range(n_v):
                assert rel_l2(got[:, h], want[:, h]) <= STATE_REL_L2, (b, h)


@pytest.mark.parametrize("ring", [True, False])
@pytest.mark.parametrize("n_v,n_qk,tiled,nodes,counts,width", GDN_SHAPES)
def test_gdn_commit(n_v, n_qk, tiled, nodes, counts, width, ring):
    from rapidllm_b200 import _lib, ops
    gen = torch.Generator().manual_seed(nodes * 10 + n_v + 1)
    batch, slots = len(counts), len(counts) + 2
    S, win, qkv, w, beta, g = _gdn_inputs(gen, batch, nodes, n_v, n_qk, slots, pad=4)
    dim = w.shape[0]
    parents = _tree(gen, batch, nodes, width)
    leaf = [c - 1 for c in counts]
    ids = torch.randperm(slots, generator=gen)[:batch].int()
    phase = torch.randint(0, 4, (slots,), generator=gen).int() if ring else torch.zeros(slots, dtype=torch.int32)
    stored = torch.stack([torch.roll(win[s], int(phase[s]), 1) for s in range(slots)])
    Sc, wc, pc = S.cuda(), stored.cuda(), phase.cuda() if ring else None
    ops.gdn_tree_commit(Sc, wc, pc, qkv.cuda()[..., :dim], w.cuda(), beta.cuda(), g.cuda(), parents.cuda(),
                        torch.tensor(leaf, dtype=torch.int32, device="cuda"), n_qk, slot_ids=ids.cuda(),
                        head_map=_lib.RL_HEADS_TILED if tiled else _lib.RL_HEADS_GROUPED)
    _lib.check_device()
    want_S, want_w = S.double(), stored.clone()
    for b in range(batch):
        path = _path(parents[b].tolist(), leaf[b])
        _, s, wn = _gdn_exact(S[ids[b]], win[ids[b]], qkv[b, :, :dim], w, beta[b], g[b], path, n_v, n_qk, tiled)
        want_S[ids[b]] = s
        want_w[ids[b]] = torch.roll(wn.float(), int(phase[ids[b]]), 1)
    assert torch.equal(wc.cpu(), want_w)
    for s in range(slots):
        if s in ids.tolist() and leaf[ids.tolist().index(s)] >= 0:
            assert rel_l2(Sc[s].cpu(), want_S[s]) <= STATE_REL_L2
        else:
            assert torch.equal(Sc[s].cpu(), S[s])
    if ring:
        assert torch.equal(pc.cpu(), phase)


def test_gdn_closed_gates_do_not_cost_digits():
    """Gates that forget everything in between (log decays of -60, -5000 and -inf): the nodes behind them keep the
    tolerance, in the verify and in the commit."""
    from rapidllm_b200 import _lib, ops
    gen = torch.Generator().manual_seed(77)
    n_v, n_qk, nodes = 4, 2, 40
    S, win, qkv, w, beta, g = _gdn_inputs(gen, 2, nodes, n_v, n_qk, 2)
    g[:, 3::7, 0] = -60.0
    g[:, 2::9, 1] = -5000.0
    g[:, 4::11, 2] = -math.inf
    parents = torch.stack([torch.arange(nodes) - 1, _tree(gen, 1, nodes, 3)[0]]).int()
    dev = [t.cuda() for t in (S, win)]
    rest = [t.cuda() for t in (qkv, w, beta, g, parents)]
    o = ops.gdn_tree(*dev, None, *rest, n_qk).cpu()
    leaf = torch.tensor([nodes - 1, nodes - 1], dtype=torch.int32)
    ops.gdn_tree_commit(*dev, None, *rest, leaf.cuda(), n_qk)
    _lib.check_device()
    for b in range(2):
        par = parents[b].tolist()
        want = torch.stack([_gdn_exact(S[b], win[b], qkv[b], w, beta[b], g[b], _path(par, i), n_v, n_qk, False)[0] for i in range(nodes)])
        for h in range(n_v):
            assert rel_l2(o[b, :, h], want[:, h]) <= STATE_REL_L2, (b, h)
            for i in range(nodes):
                assert rel_l2(o[b, i, h], want[i, h]) <= 1e-4, (b, h, i)
        state = _gdn_exact(S[b], win[b], qkv[b], w, beta[b], g[b], _path(par, nodes - 1), n_v, n_qk, False)[1]
        for h in range(n_v):
            assert rel_l2(dev[0][b, h].cpu(), state[h]) <= STATE_REL_L2, (b, h)


def test_refusals_of_the_wrappers():
    """Wrong device, type, shape or stride of a tensor is an RlError with the argument's name; nothing is launched."""
    from rapidllm_b200 import _lib, ops
    gen = torch.Generator().manual_seed(4)
    B, n = 2, 5
    kp, vp, table, _ = _pages(gen, [10, 70], [n, n], 4, 0.0)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    base, parents, leaf = i32(10, 70), _tree(gen, B, n, 2).cuda(), i32(1, 2)
    q = torch.zeros(B, n, 24, HD, device="cuda")
    qg, k = torch.zeros(B, n, 24, 512, device="cuda"), torch.zeros(B, n, 4, HD, device="cuda")
    S, win, qkv, w, beta, g = (t.cuda() for t in _gdn_inputs(gen, B, n, 6, 2, B))
    attn = dict(q=q, k_pool=kp, v_pool=vp, page_table=table, base_len=base, parents=parents)
    app = dict(qg=qg, k=k, v=k, k_pool=kp, v_pool=vp, page_table=table, pos=base, parents=parents)
    kv = dict(k_pool=kp, v_pool=vp, page_table=table, base_len=base, parents=parents, leaf=leaf)
    gdn = dict(S=S, conv_window=win, conv_phase=None, qkv=qkv, conv_w=w, beta=beta, g_log=g, parents=parents, n_qk=2)
    before = kp.clone(), S.clone(), win.clone()
    for call, good, bad in (
        (ops.attn_tree, attn, dict(q=q.cpu())), (ops.attn_tree, attn, dict(q=q.double())), (ops.attn_tree, attn, dict(parents=parents.long())),
        (ops.attn_tree, attn, dict(base_len=None)), (ops.attn_tree, attn, dict(base_len=base[:1])), (ops.attn_tree, attn, dict(page_table=table[:1])),
        (ops.attn_tree, attn, dict(out=torch.zeros_like(q))), (ops.attn_tree, attn, dict(gate=q.half())), (ops.attn_tree, attn, dict(v_pool=vp[:1])),
        (ops.attn_tree, attn, dict(gate=torch.zeros(B, n, 24, 2 * HD, device="cuda")[..., ::2])),
        (ops.attn_tree, attn, dict(q=torch.zeros(B, 65, 24, HD, device="cuda"), parents=None)),
        (ops.attn_tree, attn, dict(q=torch.zeros(B, n, HD, 24, device="cuda").transpose(2, 3))),
        (ops.attn_tree, attn, dict(max_seq_len=10 ** 6)), (ops.attn_tree, attn, dict(q=torch.zeros(B, n, 6, HD, device="cuda"))),
        (ops.attn_qk_append, app, dict(qg=qg[..., :256])), (ops.attn_qk_append, app, dict(k=k[:, :, ::2])), (ops.attn_qk_append, app, dict(v=k.half())),
        (ops.attn_qk_append, app, dict(qg=torch.zeros(n, B, 24, 512, device="cuda").transpose(0, 1))), (ops.attn_qk_append, app, dict(q_norm=base)),
        (ops.attn_qk_append, app, dict(q_dtype=torch.float64)), (ops.attn_qk_append, app, dict(rotary_dim=40)),
        (ops.kv_tree_commit, kv, dict(leaf=leaf.long())), (ops.kv_tree_commit, kv, dict(parents=parents[:1])), (ops.kv_tree_commit, kv, dict(parents=65)),
        (ops.gdn_tree, gdn, dict(n_qk=3)), (ops.gdn_tree, gdn, dict(S=S.half())), (ops.gdn_tree, gdn, dict(conv_window=win[:1])),
        (ops.gdn_tree, gdn, dict(S=S[:1], conv_window=win[:1])), (ops.gdn_tree, gdn, dict(beta=beta[:, :, :2])), (ops.gdn_tree, gdn, dict(g_log=None)),
        (ops.gdn_tree_commit, dict(gdn, leaf=leaf), dict(leaf=None)), (ops.gdn_tree_commit, dict(gdn, leaf=leaf), dict(parents=parents.cpu())),
        (ops.gdn_tree_commit, dict(gdn, leaf=leaf), dict(slot_ids=i32(0, 1, 1))),
    ):
        with pytest.raises(_lib.RlError):
            call(**{**good, **bad})
    torch.cuda.synchronize()
    assert _lib.device_error() == 0
    for t, was in zip((kp, S, win), before):
        assert torch.equal(t, was)
    # a workspace that is large enough is used, one that is not is replaced
    want = ops.gdn_tree(**gdn)
    for size in (16, 1 << 24):
        assert torch.equal(ops.gdn_tree(**gdn, workspace=torch.empty(size, dtype=torch.uint8, device="cuda")), want)


def test_bad_trees_are_recorded_and_skipped():
    """A parent that is not in [-1, i) counts as a root, a bad count as an empty draft, a bad leaf as none."""
    from rapidllm_b200 import _lib, ops
    gen = torch.Generator().manual_seed(3)
    S, win, qkv, w, beta, g = (t.cuda() for t in _gdn_inputs(gen, 3, 4, 2, 1, 3))
    dev = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    bad, good = dev([-1, 0, 2, 9], [-1, 0, -5, 1], [-1, 0, 1, 2]), dev([-1, 0, -1, -1], [-1, 0, -1, 1], [-1, 0, 1, 2])
    o = ops.gdn_tree(S, win, None, qkv, w, beta, g, bad, 1)
    assert _lib.device_error() == 6 and b"tree" in _lib.lib().rl_device_error_string(6)
    assert torch.equal(o, ops.gdn_tree(S, win, None, qkv, w, beta, g, good, 1))
    assert _lib.device_error() == 0
    out = torch.full_like(o, 2.0)
    ops.gdn_tree(S, win, None, qkv, w, beta, g, good, 1, n_nodes=dev(4, 5, -1), out=out)
    assert _lib.device_error() == 6
    assert torch.equal(out[0], o[0]) and (out[1:] == 2.0).all()
    kept = S.clone(), win.clone()
    ops.gdn_tree_commit(S, win, None, qkv, w, beta, g, good, dev(-1, 4, -2), 1)
    assert _lib.device_error() == 6
    assert torch.equal(S, kept[0]) and torch.equal(win, kept[1])
    ops.gdn_tree(S, win, None, qkv, w, beta, g, good, 1, slot_ids=dev(0, 3, -1), out=out)
    assert _lib.device_error() == 4
    kp, vp, table, _ = _pages(gen, [70, 3], [4, 4], 4, 0.0)
    q = torch.randn(2, 4, 24, HD, generator=gen).cuda()
    out = torch.full((2, 4, 24, HD), 2.0, dtype=torch.float16, device="cuda")
    # a base beyond the table's pages: that sequence is left out, the other is served
    ops.attn_tree(q, kp, vp, table, dev(125, 3), good[:2].contiguous(), out=out)
    assert _lib.device_error() == 5
    assert (out[0] == 2.0).all() and not (out[1] == 2.0).any()
    before = kp.clone()
    n = ops.kv_tree_commit(kp, vp, table, dev(70, 3), good[:2].contiguous(), dev(7, -3))
    assert _lib.device_error() == 6 and n.tolist() == [0, 0] and torch.equal(kp, before)
    table[0, 1] = kp.shape[0] + 3
    ops.attn_tree(q, kp, vp, table, dev(70, 3), good[:2].contiguous())
    assert _lib.device_error() == 1
    ops.kv_tree_commit(kp, vp, table, dev(70, 3), dev([-1, 0, 0, 2], [-1, 0, 0, 2]), dev(3, -1))
    assert _lib.device_error() == 1 and torch.equal(kp, before)
    ops.attn_qk_append(torch.randn(2, 4, 24, 512, device="cuda"), torch.randn(2, 4, 4, HD, device="cuda"),
                       torch.randn(2, 4, 4, HD, device="cuda"), kp, vp, table, dev(70, -1), parents=good[:2].contiguous())
    assert _lib.device_error() in (1, 5) and torch.equal(kp, before)


def test_a_captured_round_replays_with_new_lengths():
    """Append, attention, delta rule and commits of one round in a CUDA graph; lengths, tree and leaf are read when it
    runs.  Two graphs with one workspace, replayed in turn on one stream."""
    from rapidllm_b200 import _lib, ops
    gen = torch.Generator().manual_seed(11)
    B, n = 3, 12
    base = [500, 64, 0]
    kp, vp, table, _ = _pages(gen, [600, 200, 80], [n] * B, 4, 0.0)
    S, win, qkv, w, beta, g = (t.cuda() for t in _gdn_inputs(gen, B, n, 6, 2, B))
    qg, k, v = torch.randn(B, n, 24, 512).cuda(), torch.randn(B, n, 4, HD).cuda(), torch.randn(B, n, 4, HD).cuda()
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    base_len, leaf, parents, counts = dev(base), dev([11, 3, -1]), _tree(gen, B, n, 3).cuda(), dev([12, 5, 7])
    ws = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    out = [torch.zeros(B, n, 24, HD, dtype=torch.float16, device="cuda") for _ in range(2)]
    og = torch.zeros(B, n, 6, DK, device="cuda")

    def step(o):
        q, _ = ops.attn_qk_append(qg, k, v, kp, vp, table, base_len, parents=parents, n_nodes=counts, want_gate=False)
        ops.attn_tree(q, kp, vp, table, base_len, parents, n_nodes=counts, gate=qg[..., HD:], out=o, workspace=ws)
        ops.gdn_tree(S, win, None, qkv, w, beta, g, parents, 2, n_nodes=counts, out=og)
        ops.gdn_tree_commit(S, win, None, qkv, w, beta, g, parents, leaf, 2)
        return ops.kv_tree_commit(kp, vp, table, base_len, parents, leaf)

    keep = [t.clone() for t in (kp, vp, S, win)]

    def restore():
        for t, was in zip((kp, vp, S, win), keep):
            t.copy_(was)

    step(out[0])
    _lib.check_device()
    graphs = []
    for o in out:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(o)
        graphs.append(graph)
    for trial, (new_base, new_leaf) in enumerate((([500, 64, 0], [11, 3, -1]), ([601, 130, 17], [2, -1, 6]))):
        base_len.copy_(dev(new_base))
        leaf.copy_(dev(new_leaf))
        parents.copy_(_tree(gen, B, n, 3).cuda())
        restore()
        step(out[0])
        want = [t.clone() for t in (out[0], og, kp, vp, S, win)]
        for graph, o in zip(graphs, out):
            restore()
            o.zero_()
            graph.replay()
            _lib.check_device()
            for t, x in zip((o, og, kp, vp, S, win), want):
                assert torch.equal(t, x), trial


def test_calls_on_two_streams():
    from rapidllm_b200 import ops
    gen = torch.Generator().manual_seed(12)
    kp, vp, table, _ = _pages(gen, [900, 333], [16, 16], 4, 0.0)
    q = torch.randn(2, 16, 24, HD, generator=gen).cuda()
    parents = _tree(gen, 2, 16, 3).cuda()
    base = torch.tensor([900, 333], dtype=torch.int32, device="cuda")
    want = ops.attn_tree(q, kp, vp, table, base, parents)
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(8):
        with torch.cuda.stream(side[i % 2]):
            got.append(ops.attn_tree(q, kp, vp, table, base, parents))
    torch.cuda.synchronize()
    for o in got:
        assert torch.equal(o, want)


def _weights(gen, hidden, n_q=6, n_kv=1, nk=2, nv=6):
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    cd = 2 * nk * DK + nv * DK
    attn = dict(rms_w=r(hidden) * 0.1, Wq=r(n_q * 2 * HD, hidden) / 20, Wk=r(n_kv * HD, hidden) / 20, Wv=r(n_kv * HD, hidden) / 20,
                Wo=r(hidden, n_q * HD) / 80, q_norm=r(HD) * 0.1, k_norm=r(HD) * 0.1)
    delta = dict(rms_w=r(hidden) * 0.1, Wqkv=r(cd, hidden) / 20, Wz=r(nv * DK, hidden) / 20, Wa=r(nv, hidden) / 20,
                 Wb=r(nv, hidden) / 20, Wo=r(hidden, nv * DK) / 80, A_log=r(nv) * 0.5, dt_bias=r(nv), conv_w=r(cd, 4) * 0.5, gnorm=r(DK))
    return attn, delta


def test_a_tree_through_the_mixers_equals_decode_along_each_path():
    """Two delta layers and one attention layer: a history by decode steps, a verify pass over a tree, compared with
    decode steps along every node's path; then a commit, and one more decode step from there."""
    from rapidllm_b200 import _lib
    from rapidllm_b200.mixer import MixerStack
    torch.backends.cuda.matmul.allow_tf32 = False
    gen = torch.Generator().manual_seed(21)
    hidden, B, n, history = 256, 2, 10, 5
    attn, delta = _weights(gen, hidden)
    _, delta2 = _weights(gen, hidden)
    kinds = [_lib.RL_LAYER_LINEAR_ATTENTION, _lib.RL_LAYER_FULL_ATTENTION, _lib.RL_LAYER_LINEAR_ATTENTION]
    stack = MixerStack(kinds, [delta, attn, delta2], n_pages=5, n_slots=3, n_q=6, n_kv=1, n_k=2, n_v=6)
    table = torch.tensor([[3, 0], [1, 4]], dtype=torch.int32, device="cuda")
    slots = torch.tensor([2, 0], dtype=torch.int32, device="cuda")
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    base = [history + 57, history]                            # the first tree crosses a page edge

    # sequence 0 starts at position 57 over rows of zeros, as a longer history would leave some
    def decode(x, at, live):
        return stack.decode(x, table, dev(at), slots if live is None else live)

    for t in range(history):
        decode(torch.randn(B, hidden, generator=gen).cuda(), [57 + t, t], None)

    def state():
        out = []
        for layer in stack.layers:
            out += [layer.S, layer.conv_state] if hasattr(layer, "S") else [layer.k_pool, layer.v_pool]
        return out

    kept = [t.clone() for t in state()]

    def restore():
        for t, was in zip(state(), kept):
            t.copy_(was)

    x = torch.randn(B, n, hidden, generator=gen)
    parents = _tree(gen, B, n, 3)
    counts = [n, n - 3]
    y, pending = stack.verify_tree(x.cuda(), table, dev(base), parents.cuda(), dev(counts), slots)
    _lib.check_device()
    verified = [t.clone() for t in state()]
    leaf = [max(range(counts[b]), key=lambda i: len(_path(parents[b].tolist(), i))) for b in range(B)]
    ends = {}
    for b in range(B):
        for i in range(counts[b]):
            restore()
            path = _path(parents[b].tolist(), i)
            for d, node in enumerate(path):
                both = torch.randn(B, hidden)
                both[b] = x[b, node]
                at = [base[0] + d, base[1] + d]
                h = decode(both.cuda(), at, None)[b].cpu()
            got = y[b, i].cpu()
            assert (got - h).abs().max() <= ATTN_MAX_ABS and rel_l2(got, h) <= ATTN_REL_L2, (b, i)
            if i == leaf[b]:
                ends[b] = [t.clone() for t in state()], len(path)
    for t, was in zip(state(), verified):
        t.copy_(was)
    taken = stack.commit_tree(pending, table, dev(base), parents.cuda(), dev(leaf), slots)
    _lib.check_device()
    assert taken.tolist() == [ends[0][1], ends[1][1]]
    nxt = torch.randn(B, hidden, generator=gen)
    for b in range(B):
        for i, (t, w) in enumerate(zip(state(), ends[b][0])):
            if t.dim() > 3 or t.shape[0] == 3:                # state or window of this sequence's slot
                assert rel_l2(t[slots[b]].cpu(), w[slots[b]].cpu()) <= ATTN_REL_L2, (b, i)
    committed = [t.clone() for t in state()]
    got = decode(nxt.cuda(), [base[0] + ends[0][1], base[1] + ends[1][1]], None).cpu()
    for b in range(B):
        for t, w in zip(state(), ends[b][0]):
            t.copy_(w)
        want = decode(nxt.cuda(), [base[0] + ends[0][1], base[1] + ends[1][1]], None)[b].cpu()
        assert (got[b] - want).abs().max() <= ATTN_MAX_ABS and rel_l2(got[b], want) <= ATTN_REL_L2
    del committed


def test_chains_without_parents():
    """parents None (a number of nodes for the KV commit) is the tree whose every node continues the one before."""
    from rapidllm_b200 import _lib, ops
    gen = torch.Generator().manual_seed(31)
    B, n = 2, 9
    chain = (torch.arange(n) - 1).int().expand(B, n).contiguous().cuda()
    base = torch.tensor([61, 200], dtype=torch.int32, device="cuda")
    counts, leaf = torch.tensor([9, 4], dtype=torch.int32, device="cuda"), torch.tensor([8, 2], dtype=torch.int32, device="cuda")
    results = []
    for parents in (chain, None):
        gen.manual_seed(31)
        kp, vp, table, _ = _pages(gen, [61, 200], [n, n], 4, 0.0)
        S, win, qkv, w, beta, g = (t.cuda() for t in _gdn_inputs(gen, B, n, 6, 2, B))
        qg, k, v = (torch.randn(B, n, h, d, generator=gen).cuda() for h, d in ((24, 512), (4, HD), (4, HD)))
        out = torch.zeros(B, n, 24, HD, dtype=torch.float16, device="cuda")
        o = torch.zeros(B, n, 6, DK, device="cuda")
        q, gate = ops.attn_qk_append(qg, k, v, kp, vp, table, base, parents=parents, q_dtype=torch.float16)
        ops.attn_tree(q, kp, vp, table, base, parents, n_nodes=counts, gate=gate, out=out)
        ops.gdn_tree(S, win, None, qkv, w, beta, g, parents, 2, n_nodes=counts, out=o)
        ops.gdn_tree_commit(S, win, None, qkv, w, beta, g, parents, leaf, 2)
        taken = ops.kv_tree_commit(kp, vp, table, base, n if parents is None else parents, leaf)
        _lib.check_device()
        assert taken.tolist() == [9, 3]
        results.append((q, gate, kp, vp, out, o, S, win))
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_pages_far_into_a_large_pool():
    """Pages whose offset in the pool passes 2^32 bytes and 2^31 values."""
    from rapidllm_b200 import _lib, ops
    gen = torch.Generator().manual_seed(32)
    n, base, n_pages = 12, 130, 33000
    kp, vp = ops.new_pool(n_pages, 4), ops.new_pool(n_pages, 4)
    table = torch.tensor([[n_pages - 1, 5, n_pages - 7]], dtype=torch.int32, device="cuda")
    rows = [torch.randn(base + n, 4, HD, generator=gen).half() for _ in range(2)]
    ops.kv_append(kp, vp, table[0], rows[0][:base].cuda(), rows[1][:base].cuda(), pos0=0)
    parents = _tree(gen, 1, n, 3)
    at = torch.tensor([base], dtype=torch.int32, device="cuda")
    qg = torch.randn(1, n, 24, 512, generator=gen)
    k, v = (r[base:].float().unsqueeze(0).cuda() for r in rows)
    q, _ = ops.attn_qk_append(qg.cuda(), k, v, kp, vp, table, at, parents=parents.cuda(), rotary_dim=0, q_dtype=torch.float16, want_gate=False)
    rows[0][base:] = torch.stack([_pool_row(kp, table, 0, base + i) for i in range(n)]).cpu()
    assert torch.equal(torch.stack([_pool_row(vp, table, 0, base + i) for i in range(n)]).cpu(), rows[1][base:])
    got = ops.attn_tree(q, kp, vp, table, at, parents.cuda())
    o, _, _ = _attn_exact(q[0].cpu(), None, rows, base, parents[0].tolist(), n, 24, 4)
    assert rel_l2(got[0].float().cpu(), o) <= 1e-3
    path = _path(parents[0].tolist(), n - 1)
    ops.kv_tree_commit(kp, vp, table, at, parents.cuda(), torch.tensor([n - 1], dtype=torch.int32, device="cuda"))
    _lib.check_device()
    for j, i in enumerate(path):
        assert torch.equal(_pool_row(kp, table, 0, base + j).cpu(), rows[0][base + i])
        assert torch.equal(_pool_row(vp, table, 0, base + j).cpu(), rows[1][base + i])


@pytest.mark.parametrize("base,q_type", [([40, 3], torch.float16), ([6000, 64], torch.float32)])
def test_attn_tree_bad_rows_stay_with_their_descendants(base, q_type):
    """K, V or a query that is not finite: NaN in the rows that see it, nothing else changes by a bit (what a row does not
    see has weight 0 and is replaced by 0 before the product)."""
    from rapidllm_b200 import _lib, ops
    gen = torch.Generator().manual_seed(33)
    B, n = 2, 40
    kp, vp, table, _ = _pages(gen, base, [n, n], 4, float("nan"))
    parents = _tree(gen, B, n, 6)
    q = torch.randn(B, n, 24, HD, generator=gen).to(q_type)
    at = torch.tensor(base, dtype=torch.int32, device="cuda")
    clean = ops.attn_tree(q.cuda(), kp, vp, table, at, parents.cuda())
    hit = torch.zeros(B, n, 4, dtype=torch.bool)
    for b, pool, node, head, value in ((0, vp, 4, 1, math.inf), (0, vp, 25, 3, math.nan), (0, kp, 11, 0, math.nan), (1, vp, 30, 2, -math.inf)):
        page, row = int(table[b, (base[b] + node) // 64]), (base[b] + node) % 64
        pool[page, head, int(ops.kv_slice_index(torch.tensor(row), torch.tensor(77)))] = value
        for i in range(n):
            hit[b, i, head] |= node in _path(parents[b].tolist(), i)
    q[1, 7, 20, 200] = math.nan
    got = ops.attn_tree(q.cuda(), kp, vp, table, at, parents.cuda())
    _lib.check_device()
    rows = hit.repeat_interleave(6, 2)
    rows[1, 7, 20] = True
    assert rows.any() and not rows.all()
    assert torch.isnan(got.cpu()[rows]).all()
    assert torch.equal(got.cpu()[~rows], clean.cpu()[~rows])


@pytest.mark.parametrize("n_v,n_qk,nodes", [(4, 2, 14), (6, 2, 30), (3, 3, 64)])
def test_gdn_tree_bad_nodes_stay_with_their_descendants(n_v, n_qk, nodes):
    """Projections and gates that are not finite: the outputs that the formula makes so are not finite, all others keep
    their tolerance."""
    from rapidllm_b200 import _lib, ops
    gen = torch.Generator().manual_seed(34)
    S, win, qkv, w, beta, g = _gdn_inputs(gen, 2, nodes, n_v, n_qk, 2)
    parents = _tree(gen, 2, nodes, 6)
    qkv[0, 5, 3] = math.inf                                   # q of head 0
    qkv[0, 7, n_qk * DK + DK + 9] = math.nan                  # k of head 1
    qkv[1, 6, 2 * n_qk * DK + 2 * DK + 50] = math.nan         # v of head 2, one column
    qkv[1, nodes - 2, 2 * n_qk * DK + 100] = -math.inf
    beta[1, 9, 0] = math.nan
    g[1, 8, 1] = math.inf
    g[1, 4, 1] = -math.inf                                    # a closed gate
    o = ops.gdn_tree(S.cuda(), win.cuda(), None, *(t.cuda() for t in (qkv, w, beta, g, parents)), n_qk).cpu()
    _lib.check_device()
    for b in range(2):
        par = parents[b].tolist()
        want = torch.stack([_gdn_exact(S[b], win[b], qkv[b], w, beta[b], g[b], _path(par, i), n_v, n_qk, False)[0] for i in range(nodes)])
        fine = torch.isfinite(want)
        assert not fine.all() and fine.double().mean() > 0.3
        assert torch.equal(torch.isfinite(o[b]), fine)
        for h in range(n_v):
            assert rel_l2(o[b, :, h][fine[:, h]], want[:, h][fine[:, h]]) <= STATE_REL_L2, (b, h)


def test_gdn_commit_of_paths_with_bad_nodes():
    """Nodes off the path leave no trace, whatever they hold; on the path they spoil what the formula says and no more."""
    from rapidllm_b200 import _lib, ops
    gen = torch.Generator().manual_seed(35)
    B, n_v, n_qk, nodes = 2, 6, 2, 20
    S, win, qkv, w, beta, g = _gdn_inputs(gen, B, nodes, n_v, n_qk, B)
    parents = torch.full((B, nodes), -1, dtype=torch.int32)
    parents[:, 2::2] = torch.arange(0, nodes - 2, 2)           # two chains: even and odd nodes
    parents[:, 3::2] = torch.arange(1, nodes - 2, 2)
    leaf = torch.tensor([nodes - 2, nodes - 1], dtype=torch.int32)

    def run(qkv, beta, g):
        dev = [t.cuda() for t in (S, win)]
        ops.gdn_tree_commit(*dev, None, *(t.cuda() for t in (qkv, w, beta, g, parents, leaf)), n_qk)
        _lib.check_device()
        return [t.cpu() for t in dev]

    clean = run(qkv, beta, g)
    bad = [t.clone() for t in (qkv, beta, g)]
    bad[0][:, 5], bad[1][:, 7], bad[2][:, 9] = math.nan, math.inf, math.nan         # on the second sequence's path
    got = run(*bad)
    assert torch.equal(got[0][0], clean[0][0]) and torch.equal(got[1][0], clean[1][0])
    assert not torch.isfinite(got[0][1]).any()
    one = [t.clone() for t in (qkv, beta, g)]
    one[0][1, 15, n_qk * DK + DK + 4] = math.inf              # k of head 1: value heads 3, 4, 5
    one[0][1, 11, 2 * n_qk * DK + 7] = math.nan               # a column of value head 0
    one[1][1, 13, 1] = math.nan
    one[2][0, 8, 2] = math.nan
    got = run(*one)
    for b in range(B):
        path = _path(parents[b].tolist(), int(leaf[b]))
        _, state, window = _gdn_exact(S[b], win[b], one[0][b], w, one[1][b], one[2][b], path, n_v, n_qk, False)
        fine = torch.isfinite(state)
        assert fine.any() and not fine.all()
        assert torch.equal(torch.isfinite(got[0][b]), fine)
        assert rel_l2(got[0][b][fine], state[fine]) <= STATE_REL_L2
        assert torch.equal(got[1][b].isnan(), window.isnan())


@pytest.mark.parametrize("n_q,n_kv,nodes,base,counts,q_type,o_type", [
    (24, 4, 64, [3000, 1500, 900], [64, 50, 30], torch.float16, torch.float16),    # 3, 3 and 2 row tiles in 11 pages a CTA
    (16, 2, 64, [5000, 0, 2111], [64, 64, 17], torch.float32, torch.float16),      # 4, 4 and 2
    (24, 4, 43, [9000], [43], torch.bfloat16, torch.bfloat16),                     # 3, the last one of one node
])
def test_attn_tree_row_tiles_over_long_caches(n_q, n_kv, nodes, base, counts, q_type, o_type):
    """Row tiles start at different pages of a sequence and wrap around its end."""
    test_attn_tree(n_q, n_kv, nodes, base, counts, 5, q_type, o_type, True)
