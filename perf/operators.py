"""The operators that verify and commit a tree of drafted tokens in the hybrid stack, as cases that can be timed.

A draft proposes up to 64 tokens per sequence as a tree: parents[b][i] < i is the node that token i
continues, -1 the committed history.  One verify pass runs every node through the mixers, a commit
keeps one path:

    attn_qk_append    q/gate split, head norms, rotation at the node's depth, K and V into the pages
    attn_tree         attention of every node over the cache and its own ancestors, gated
    gdn_tree          conv + delta rule of every node along its own path; the state is only read
    gdn_tree_commit   state and conv window advanced along the path to the chosen leaf (the ring's phase stays)
    kv_tree_commit    the K and V rows of that path moved to consecutive positions

`run` computes them in plain torch, or, with `own` set, through rapidllm_b200.ops.  Sizes are those
of the hybrid model (24 query / 4 KV heads of 256, 48 value / 16 key heads of 128 x 128), lengths
are a function of the case, values come from the seed.
"""
import math

import torch

own = False

HD, DK, PAGE, TAPS = 256, 128, 64, 4
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------

def listed():
    attn = {"n_q": 24, "n_kv": 4}
    gdn = {"n_v": 48, "n_qk": 16, "tiled": False}
    return [
        # one user's small draft: the call's latency
        dict(op="append", name="append-tree-1x8", batch=1, nodes=8, ctx=2000, width=3, tree=True, rot=64, q="fp16",
             gate=False, **attn),
        # a chunk of a long prompt: bandwidth over the projections' rows
        dict(op="append", name="append-prompt-4096", batch=1, nodes=4096, ctx=100000, width=1, tree=False, rot=64,
             q="bf16", gate=True, **attn),
        # one user, short chat: latency
        dict(op="attn", name="attn-1x8-2k", batch=1, nodes=8, ctx=2000, width=3, q="fp16", o="fp16", **attn),
        # a serving batch at ragged contexts: bandwidth of the cache
        dict(op="attn", name="attn-16x21-16k", batch=16, nodes=21, ctx=16384, width=4, q="fp32", o="bf16", **attn),
        # wide trees over long documents: the tensor cores' rate
        dict(op="attn", name="attn-4x64-32k", batch=4, nodes=64, ctx=32768, width=6, q="bf16", o="bf16", **attn),
        dict(op="gdn", name="gdn-1x8", batch=1, nodes=8, width=3, **gdn),
        dict(op="gdn", name="gdn-16x21", batch=16, nodes=21, width=4, **gdn),
        # a chain of 64 in every sequence: the most work a node can have
        dict(op="gdn", name="gdn-32x64-chain", batch=32, nodes=64, width=1, **gdn),
        dict(op="gdn_commit", name="gdn-commit-1x8", batch=1, nodes=8, width=3, **gdn),
        dict(op="gdn_commit", name="gdn-commit-32x32", batch=32, nodes=32, width=6, **gdn),
        dict(op="kv_commit", name="kv-commit-1x8", batch=1, nodes=8, ctx=2000, width=3, **attn),
        dict(op="kv_commit", name="kv-commit-32x64", batch=32, nodes=64, ctx=1000, width=2, **attn),
    ]


def draw(rng):
    def log_int(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["append", "attn", "attn", "gdn", "gdn", "gdn_commit", "kv_commit"])
    n_q, n_kv = rng.choice([(24, 4), (24, 4), (12, 2), (6, 1), (16, 2), (8, 8)])
    n_v, n_qk = rng.choice([(48, 16), (48, 16), (24, 8), (32, 16), (16, 16)])
    nodes, width = rng.choice([1, 2, 5, 8, 13, 16, 21, 27, 32, 48, 63, 64]), rng.randint(1, 8)
    if op == "append":
        tree = rng.random() < 0.5
        if not tree:
            nodes = log_int(1, 4000)
        batch = log_int(1, max(1, min(32, 4000 // nodes)))
        return dict(op=op, batch=batch, nodes=nodes, ctx=log_int(1, min(131072, 400000 // batch)), width=width, tree=tree,
                    rot=rng.choice([64, 64, 128, 32]), q=rng.choice(["fp32", "fp16", "bf16"]), gate=rng.random() < 0.5,
                    n_q=n_q, n_kv=n_kv)
    if op == "attn":
        batch = log_int(1, 16)
        ctx = log_int(1, min(131072, 131072 * 21 // (batch * max(21, nodes))))
        q = rng.choice(["fp32", "fp16", "bf16"])
        return dict(op=op, batch=batch, nodes=nodes, ctx=ctx, width=width, q=q, o="bf16" if q == "bf16" else rng.choice(["fp16", "bf16"]),
                    n_q=n_q, n_kv=n_kv)
    if op == "kv_commit":
        return dict(op=op, batch=log_int(1, 32), nodes=nodes, ctx=log_int(1, 1000), width=width, n_q=n_q, n_kv=n_kv)
    return dict(op=op, batch=log_int(1, 31), nodes=nodes if op == "gdn" else min(nodes, 32), width=width, n_v=n_v,
                n_qk=n_qk, tiled=rng.random() < 0.3)


def _base(c):
    """Committed tokens of each sequence: ragged, from ctx down to 3/8 of it."""
    return [max(1, c["ctx"] - (c["ctx"] * 5 * b) // (8 * c["batch"])) for b in range(c["batch"])]


def _counts(c):
    """Nodes of each sequence: from the case's number down to half of it."""
    return [max(1, c["nodes"] - (c["nodes"] * b) // (2 * c["batch"])) for b in range(c["batch"])]


def work(case):
    c, n = case, sum(_counts(case))
    size = {"fp32": 4, "fp16": 2, "bf16": 2}
    if c["op"] == "append":
        n = n if c["tree"] else c["batch"] * c["nodes"]
        row_in = c["n_q"] * (2 if c["gate"] else 1) * HD * 4 + 2 * c["n_kv"] * HD * 4
        row_out = c["n_q"] * HD * (size[c["q"]] + (4 if c["gate"] else 0)) + 2 * c["n_kv"] * HD * 2
        return {"bytes": n * (row_in + row_out), "flops": n * (c["n_q"] + c["n_kv"]) * HD * 6}
    if c["op"] == "attn":
        kv = sum(a + b for a, b in zip(_base(c), _counts(c))) * c["n_kv"] * HD * 2 * 2
        rows = n * c["n_q"] * HD
        pairs = sum((a + 1) * b for a, b in zip(_base(c), _counts(c)))
        return {"bytes": kv + rows * (size[c["q"]] + size[c["o"]] + 4), "flops": 4 * HD * c["n_q"] * pairs}
    if c["op"] == "kv_commit":
        # the rows of the path to a leaf in the middle, read and written
        rows = sum(max(1, k // (c["width"] + 1)) for k in _counts(c))
        return {"bytes": rows * c["n_kv"] * HD * 2 * 2 * 2, "flops": 0}
    conv_dim = 2 * c["n_qk"] * DK + c["n_v"] * DK
    state = c["batch"] * c["n_v"] * DK * DK * 4
    if c["op"] == "gdn":
        return {"bytes": state + n * (conv_dim + c["n_v"] * DK + 2 * c["n_v"]) * 4 + c["batch"] * conv_dim * TAPS * 4 + conv_dim * TAPS * 4,
                "flops": n * c["n_v"] * DK * DK * 4}
    path = sum(max(1, k // (c["width"] + 1)) for k in _counts(c))
    return {"bytes": 2 * state + path * (conv_dim - c["n_qk"] * DK + 2 * c["n_v"]) * 4 + 2 * c["batch"] * conv_dim * TAPS * 4,
            "flops": path * c["n_v"] * DK * DK * 4}


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------

def _tree(c, gen, dev):
    """parents [batch][nodes]: each node continues one of the `width` nodes before it (width 1: a chain)."""
    i = torch.arange(c["nodes"], device=dev).expand(c["batch"], -1)
    back = (torch.rand(c["batch"], c["nodes"], generator=gen, device=dev) * torch.minimum(i, torch.full_like(i, c["width"]))).long()
    return (i - 1 - back).to(torch.int32)


def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device=dev) * scale

    B, n = c["batch"], c["nodes"]
    s = {"case": dict(c), "parents": _tree(c, gen, dev) if c.get("tree", True) else None,
         "n_nodes": torch.tensor(_counts(c), dtype=torch.int32, device=dev) if c.get("tree", True) else None}
    if c["op"] in ("append", "attn", "kv_commit"):
        base = _base(c)
        pages = [(x + n + PAGE - 1) // PAGE for x in base]
        total = sum(pages) + 1
        perm = torch.randperm(total, generator=gen, device=dev).to(torch.int32)
        table = torch.zeros(B, max(pages), dtype=torch.int32)
        at = 0
        where = torch.zeros(B, max(pages), dtype=torch.long)
        for b, p in enumerate(pages):
            where[b, :p] = torch.arange(at, at + p)
            at += p
        table = perm[where.to(dev)].contiguous()
        s["table"], s["base"] = table, torch.tensor(base, dtype=torch.int32, device=dev)
        s["k_pool"] = normal(total, c["n_kv"], PAGE * HD).half()
        s["v_pool"] = normal(total, c["n_kv"], PAGE * HD).half()
    if c["op"] == "append":
        # one projection's rows: [q | gate] of every head, then k, then v, as columns
        nq, nk = c["n_q"] * 2 * HD, c["n_kv"] * HD
        proj = normal(B, n, nq + 2 * nk)
        s["qg"] = proj[..., :nq].view(B, n, c["n_q"], 2 * HD)
        s["k"] = proj[..., nq:nq + nk].view(B, n, c["n_kv"], HD)
        s["v"] = proj[..., nq + nk:].view(B, n, c["n_kv"], HD)
        s["q_norm"], s["k_norm"] = normal(HD, scale=0.2), normal(HD, scale=0.2)
        s["q_out"] = torch.zeros(B, n, c["n_q"], HD, dtype=TYPES[c["q"]], device=dev)
        s["gate_out"] = torch.zeros(B, n, c["n_q"], HD, device=dev) if c["gate"] else None
    elif c["op"] == "attn":
        s["q"] = normal(B, n, c["n_q"], HD, scale=2.0).to(TYPES[c["q"]])
        # the gate is read where the projection left it: the second half of every head's columns
        s["gate"] = normal(B, n, c["n_q"], 2 * HD)[..., HD:]
        s["o"] = torch.zeros(B, n, c["n_q"], HD, dtype=TYPES[c["o"]], device=dev)
    else:
        # a leaf anywhere in the tree; in a batch, the second sequence rejects its draft
        leaf = (torch.rand(B, generator=gen, device=dev) * s["n_nodes"]).to(torch.int32)
        if B > 1:
            leaf[1] = -1
        s["leaf"] = leaf
    if c["op"] in ("gdn", "gdn_commit"):
        dim = 2 * c["n_qk"] * DK + c["n_v"] * DK
        slots = B + 1
        s["slots"] = torch.randperm(slots, generator=gen, device=dev)[:B].to(torch.int32)
        s["S"] = normal(slots, c["n_v"], DK, DK, scale=0.3)
        s["ring"] = normal(slots, dim, TAPS)
        s["phase"] = torch.randint(0, TAPS, (slots,), generator=gen, device=dev, dtype=torch.int32)
        s["conv_w"] = normal(dim, TAPS, scale=0.5)
        s["qkv"] = normal(B, n, dim)
        s["beta"] = torch.sigmoid(normal(B, n, c["n_v"]))
        s["g_log"] = -0.2 * torch.rand(B, n, c["n_v"], generator=gen, device=dev)
        if c["op"] == "gdn":
            s["o"] = torch.zeros(B, n, c["n_v"], DK, device=dev)
    return s


# ------------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------------

def _reach(parents):
    """[B][n][n] 1.0 where column j is row i or one of its ancestors: (I - P)^-1 of the parent matrix."""
    n = parents.shape[1]
    ids = torch.arange(n, device=parents.device)
    p = (parents.unsqueeze(2) == ids).double()
    eye = torch.eye(n, dtype=torch.float64, device=parents.device)
    r = eye + p
    for _ in range(max(1, (n - 1).bit_length())):
        p = p @ p
        r = r + p @ r
    return (r > 0.5).double()


def _slices(pool, n_kv):
    """A pool as [pages][heads][token][256]; the 16-byte chunks of token t are stored at index (chunk ^ (t & 7))."""
    x = pool.view(-1, n_kv, HD // 64, PAGE, 8, 8)
    t = torch.arange(PAGE, device=pool.device).unsqueeze(1)
    j = torch.arange(8, device=pool.device).unsqueeze(0) ^ (t & 7)
    return x[:, :, :, t, j].permute(0, 1, 3, 2, 4, 5).reshape(x.shape[0], n_kv, PAGE, HD)


def _row_index(table, position, n_kv):
    """Flat pool index of every value of the rows at `position` [B][n]: [B][n][n_kv][256]."""
    page = torch.gather(table.long(), 1, position // PAGE)
    row = position % PAGE
    d = torch.arange(HD, device=table.device)
    off = (d // 64) * (PAGE * 64) + row.unsqueeze(2) * 64 + (((d % 64) // 8) ^ (row.unsqueeze(2) & 7)) * 8 + d % 8
    head = torch.arange(n_kv, device=table.device).view(1, 1, n_kv, 1)
    return (page.view(*page.shape, 1, 1) * n_kv + head) * (PAGE * HD) + off.unsqueeze(2)


def _live(s, n):
    if s["n_nodes"] is None:
        return torch.ones(s["case"]["batch"], n, dtype=torch.bool, device="cuda")
    return torch.arange(n, device="cuda") < s["n_nodes"].unsqueeze(1)


def _normed(x, w):
    x = x.float()
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (1.0 + w)


def _rotated(x, position, rot):
    half = rot // 2
    inv = torch.pow(torch.tensor(1e7, dtype=torch.float64, device=x.device), -torch.arange(half, device=x.device, dtype=torch.float64) / half)
    angle = position.double().unsqueeze(2) * inv
    cos, sin = torch.cos(angle).float().unsqueeze(2), torch.sin(angle).float().unsqueeze(2)
    a, b = x[..., :half], x[..., half:rot]
    return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., rot:]], -1)


def _append(s):
    c, n = s["case"], s["case"]["nodes"]
    slot = s["base"].long().unsqueeze(1) + torch.arange(n, device="cuda")
    position = slot if s["parents"] is None else s["base"].long().unsqueeze(1) + _reach(s["parents"]).sum(2).long() - 1
    live = _live(s, n)
    q = _rotated(_normed(s["qg"][..., :HD], s["q_norm"]), position, c["rot"])
    k = _rotated(_normed(s["k"], s["k_norm"]), position, c["rot"])
    s["q_out"][live] = q.to(s["q_out"].dtype)[live]
    if s["gate_out"] is not None:
        s["gate_out"][live] = s["qg"][..., HD:][live]
    at = _row_index(s["table"], slot, c["n_kv"])[live].reshape(-1)
    s["k_pool"].view(-1)[at] = k.half()[live].reshape(-1)
    s["v_pool"].view(-1)[at] = s["v"].half()[live].reshape(-1)
    return [s["q_out"], s["gate_out"], s["k_pool"], s["v_pool"]] if c["gate"] else [s["q_out"], s["k_pool"], s["v_pool"]]


def _attn(s):
    c, B, n = s["case"], s["case"]["batch"], s["case"]["nodes"]
    G = c["n_q"] // c["n_kv"]
    pages = s["table"].long()
    L = pages.shape[1] * PAGE
    k = _slices(s["k_pool"], c["n_kv"])[pages].permute(0, 2, 1, 3, 4).reshape(B, c["n_kv"], L, HD).float()
    q = s["q"].float().view(B, n, c["n_kv"], G, HD).permute(0, 2, 3, 1, 4).reshape(B, c["n_kv"], G * n, HD)
    score = (q @ k.transpose(2, 3)) / math.sqrt(HD)
    del k
    at = torch.arange(L, device="cuda").view(1, 1, L)
    base = s["base"].long().view(B, 1, 1)
    node = (at - base).clamp(0, n - 1).expand(B, n, L)
    seen = (at < base) | ((at - base < n) & (at >= base) & (torch.gather(_reach(s["parents"]), 2, node) > 0.5))
    score = score.view(B, c["n_kv"], G, n, L).masked_fill(~seen.view(B, 1, 1, n, L), float("-inf"))
    score = torch.exp(score - score.amax(-1, keepdim=True))
    total = score.sum(-1, keepdim=True)
    v = _slices(s["v_pool"], c["n_kv"])[pages].permute(0, 2, 1, 3, 4).reshape(B, c["n_kv"], L, HD).float()
    o = (score.view(B, c["n_kv"], G * n, L) @ v).view(B, c["n_kv"], G, n, HD) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(B, n, c["n_q"], HD) * torch.sigmoid(s["gate"])
    live = _live(s, n)
    s["o"][live] = o.to(s["o"].dtype)[live]
    return [s["o"]]


def _key_heads(c):
    h = torch.arange(c["n_v"], device="cuda")
    return h % c["n_qk"] if c["tiled"] else h // (c["n_v"] // c["n_qk"])


def _conv(s):
    """SiLU of the four taps of every node: itself and its three nearest ancestors, then the slot's window."""
    c, n = s["case"], s["case"]["nodes"]
    slots = s["slots"].long()
    order = (s["phase"][slots].long().unsqueeze(1) + torch.arange(TAPS, device="cuda")) % TAPS
    past = torch.gather(s["ring"][slots], 2, order.unsqueeze(1).expand(-1, s["ring"].shape[1], -1)).transpose(1, 2)
    rows = torch.cat([past, s["qkv"]], 1)                   # the window's inputs, oldest first, then the nodes'
    # a step back from row r: r - 1 inside the window, the parent's row (the newest input for a root) in the tree
    back = torch.cat([torch.arange(-1, TAPS - 1, device="cuda").clamp(min=0).expand(slots.numel(), -1),
                      s["parents"].long() + TAPS], 1)
    r0 = torch.arange(TAPS, TAPS + n, device="cuda").expand(slots.numel(), -1)
    r1 = torch.gather(back, 1, r0)
    r2 = torch.gather(back, 1, r1)
    r3 = torch.gather(back, 1, r2)
    pick = lambda r: torch.gather(rows, 1, r.unsqueeze(2).expand(-1, -1, rows.shape[2]))  # noqa: E731
    w = s["conv_w"]
    y = pick(r3) * w[:, 0] + pick(r2) * w[:, 1] + pick(r1) * w[:, 2] + pick(r0) * w[:, 3]
    return y * torch.sigmoid(y)


def _heads(c, y):
    """q, k (unit length) and v of every value head: [B][n_v][n][128]."""
    B, n = y.shape[:2]
    qd = c["n_qk"] * DK
    unit = lambda x: x * torch.rsqrt((x * x).sum(-1, keepdim=True) + EPS)  # noqa: E731
    hs = _key_heads(c)
    q = unit(y[..., :qd].view(B, n, c["n_qk"], DK))[:, :, hs].transpose(1, 2) / math.sqrt(DK)
    k = unit(y[..., qd:2 * qd].view(B, n, c["n_qk"], DK))[:, :, hs].transpose(1, 2)
    return q, k, y[..., 2 * qd:].view(B, n, c["n_v"], DK).transpose(1, 2)


def _updates(S, k, v, beta, g, reach):
    """u of every node, (I + L) u = beta (v - decay S^T k) with L over strict ancestors, and the decays."""
    total = reach.unsqueeze(1) @ g.double().unsqueeze(3)                     # log decay from the state to the node
    between = torch.exp(torch.where(reach.unsqueeze(1) > 0, total - total.transpose(2, 3), -math.inf))
    strict = reach - torch.eye(reach.shape[1], dtype=torch.float64, device="cuda")
    low = -(beta.double().unsqueeze(3) * between * strict.unsqueeze(1) * (k.double() @ k.double().transpose(2, 3)))
    inverse = torch.eye(reach.shape[1], dtype=torch.float64, device="cuda") + low
    for _ in range(max(1, (reach.shape[1] - 1).bit_length())):
        low = low @ low
        inverse = inverse + low @ inverse
    rhs = beta.unsqueeze(3) * (v - torch.exp(total).float() * (k @ S))
    return inverse.float() @ rhs, total, between


def _gdn(s):
    c, n = s["case"], s["case"]["nodes"]
    S = s["S"][s["slots"].long()]
    q, k, v = _heads(c, _conv(s))
    u, total, between = _updates(S, k, v, s["beta"].transpose(1, 2), s["g_log"].transpose(1, 2), _reach(s["parents"]))
    o = torch.exp(total).float() * (q @ S) + ((q @ k.transpose(2, 3)) * between.float()) @ u
    live = _live(s, n)
    s["o"][live] = o.transpose(1, 2)[live]
    return [s["o"]]


def _gdn_commit(s):
    c, n, B = s["case"], s["case"]["nodes"], s["case"]["batch"]
    slots = s["slots"].long()
    S = s["S"][slots]
    _, k, v = _heads(c, _conv(s))
    reach = _reach(s["parents"])
    u, total, _ = _updates(S, k, v, s["beta"].transpose(1, 2), s["g_log"].transpose(1, 2), reach)
    leaf = s["leaf"].long()
    on = torch.gather(reach, 1, leaf.clamp(min=0).view(B, 1, 1).expand(-1, 1, n)).view(B, 1, n, 1)
    end = torch.gather(total, 2, leaf.clamp(min=0).view(B, 1, 1, 1).expand(-1, c["n_v"], 1, 1))
    weight = torch.where(on > 0, torch.exp(end - total), 0.0).float()
    new = torch.exp(end).float() * S + (k * weight).transpose(2, 3) @ u
    s["S"][slots] = torch.where((leaf >= 0).view(B, 1, 1, 1), new, S)
    # the window: the last four inputs up to the leaf, kept as a ring that starts at the slot's phase
    depth = torch.where(leaf >= 0, torch.gather(reach.sum(2), 1, leaf.clamp(min=0).unsqueeze(1)).squeeze(1).long(), 0)
    step = torch.where(on.view(B, n) > 0, reach.sum(2).long(), -1)
    age = depth.unsqueeze(1) + torch.arange(1 - TAPS, 1, device="cuda")                  # oldest first; <= 0: the old window's
    hit = (step.unsqueeze(1) == age.unsqueeze(2)) & (age.unsqueeze(2) > 0)
    fresh = torch.gather(s["qkv"], 1, hit.long().argmax(2).unsqueeze(2).expand(-1, -1, s["ring"].shape[1])).transpose(1, 2)
    order = (s["phase"][slots].long().unsqueeze(1) + torch.arange(TAPS, device="cuda")) % TAPS
    dim = s["ring"].shape[1]
    past = torch.gather(s["ring"][slots], 2, order.unsqueeze(1).expand(-1, dim, -1))
    kept = torch.gather(past, 2, (age + TAPS - 1).clamp(0, TAPS - 1).unsqueeze(1).expand(-1, dim, -1))
    s["ring"][slots] = torch.zeros_like(past).scatter(2, order.unsqueeze(1).expand(-1, dim, -1),
                                                      torch.where((age > 0).unsqueeze(1), fresh, kept))
    return [s["S"], s["ring"]]


def _kv_commit(s):
    c, n, B = s["case"], s["case"]["nodes"], s["case"]["batch"]
    reach = _reach(s["parents"])
    leaf = s["leaf"].long()
    on = (torch.gather(reach, 1, leaf.clamp(min=0).view(B, 1, 1).expand(-1, 1, n)).view(B, n) > 0) & (leaf >= 0).unsqueeze(1)
    base = s["base"].long().unsqueeze(1)
    src = _row_index(s["table"], base + torch.arange(n, device="cuda"), c["n_kv"])[on].reshape(-1)
    dst = _row_index(s["table"], base + reach.sum(2).long() - 1, c["n_kv"])[on].reshape(-1)
    for pool in (s["k_pool"].view(-1), s["v_pool"].view(-1)):
        pool[dst] = pool[src]
    return [s["k_pool"], s["v_pool"], on.sum(1).to(torch.int32)]


def run(state):
    s = state
    if own:
        from rapidllm_b200 import _lib, ops
        c = s["case"]
        if c["op"] == "append":
            q, gate = ops.attn_qk_append(s["qg"], s["k"], s["v"], s["k_pool"], s["v_pool"], s["table"], s["base"], s["q_norm"],
                                         s["k_norm"], parents=s["parents"], n_nodes=s["n_nodes"], rotary_dim=c["rot"], theta=1e7,
                                         eps=EPS, q_out=s["q_out"], gate_out=s["gate_out"], want_gate=c["gate"])
            return [q, gate, s["k_pool"], s["v_pool"]] if c["gate"] else [q, s["k_pool"], s["v_pool"]]
        if c["op"] == "attn":
            return [ops.attn_tree(s["q"], s["k_pool"], s["v_pool"], s["table"], s["base"], s["parents"], n_nodes=s["n_nodes"],
                                  gate=s["gate"], out=s["o"])]
        if c["op"] == "kv_commit":
            return [s["k_pool"], s["v_pool"], ops.kv_tree_commit(s["k_pool"], s["v_pool"], s["table"], s["base"], s["parents"], s["leaf"])]
        head_map = _lib.RL_HEADS_TILED if c["tiled"] else _lib.RL_HEADS_GROUPED
        args = (s["S"], s["ring"], s["phase"], s["qkv"], s["conv_w"], s["beta"], s["g_log"], s["parents"])
        if c["op"] == "gdn":
            return [ops.gdn_tree(*args, n_qk=c["n_qk"], n_nodes=s["n_nodes"], slot_ids=s["slots"], head_map=head_map, eps_l2=EPS, out=s["o"])]
        ops.gdn_tree_commit(*args, s["leaf"], n_qk=c["n_qk"], slot_ids=s["slots"], head_map=head_map, eps_l2=EPS)
        return [s["S"], s["ring"]]
    return {"append": _append, "attn": _attn, "gdn": _gdn, "gdn_commit": _gdn_commit, "kv_commit": _kv_commit}[s["case"]["op"]](s)


# ------------------------------------------------------------------------------------------------
# 64-bit values, node by node from the definitions
# ------------------------------------------------------------------------------------------------

def _path(parents, i):
    p = []
    while i >= 0:
        p.append(i)
        i = parents[i]
    return p[::-1]


def _token_rows(pool, table_row, n_kv, first, count):
    """Tokens [first, first + count) of one sequence, [count][n_kv][256] in 64 bits, and the index that found them."""
    t = torch.arange(first, first + count, device=pool.device)
    page, r = table_row.long()[t.div(PAGE, rounding_mode="floor")], t.remainder(PAGE)
    sub, chunk, e = torch.meshgrid(torch.arange(4, device=pool.device), torch.arange(8, device=pool.device),
                                   torch.arange(8, device=pool.device), indexing="ij")
    inside = sub * 4096 + r.view(-1, 1, 1, 1) * 64 + torch.bitwise_xor(chunk, r.view(-1, 1, 1, 1) % 8) * 8 + e
    return pool[page][:, :, :].gather(2, inside.reshape(count, 1, HD).expand(-1, n_kv, -1)).double(), (page, inside.reshape(count, HD))


def _put_rows(pool, found, rows):
    page, inside = found
    h = torch.arange(pool.shape[1], device=pool.device).view(1, -1, 1)
    pool[page.view(-1, 1, 1), h, inside.unsqueeze(1)] = rows


def exact(case, seed):
    s = prepare(case, seed)
    c, n = case, case["nodes"]
    parents = s["parents"].tolist() if s["parents"] is not None else None
    counts = s["n_nodes"].tolist() if s["n_nodes"] is not None else [n] * c["batch"]
    if c["op"] in ("gdn", "gdn_commit"):
        return _exact_gdn(s, parents, counts)
    base = s["base"].tolist()
    kp, vp = s["k_pool"].double(), s["v_pool"].double()
    if c["op"] == "append":
        q_out = s["q_out"].double()
        gate_out = s["gate_out"].double() if c["gate"] else None
        half = c["rot"] // 2
        for b in range(c["batch"]):
            m = counts[b]
            depth = list(range(m)) if parents is None else [len(_path(parents[b], i)) - 1 for i in range(m)]
            angle = torch.tensor([base[b] + d for d in depth], dtype=torch.float64, device="cuda").view(m, 1, 1) / \
                torch.tensor([1e7 ** (i / half) for i in range(half)], dtype=torch.float64, device="cuda")
            for x, w, put in ((s["qg"][b, :m, :, :HD], s["q_norm"], None), (s["k"][b, :m], s["k_norm"], kp)):
                x = x.double()
                x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * (1 + w.double())
                turn = torch.polar(torch.ones_like(angle), angle) * torch.complex(x[..., :half], x[..., half:c["rot"]])
                x[..., :half], x[..., half:c["rot"]] = turn.real, turn.imag
                if put is None:
                    q_out[b, :m] = x
                else:
                    _put_rows(put, _token_rows(put, s["table"][b], c["n_kv"], base[b], m)[1], x)
            _put_rows(vp, _token_rows(vp, s["table"][b], c["n_kv"], base[b], m)[1], s["v"][b, :m].double())
            if gate_out is not None:
                gate_out[b, :m] = s["qg"][b, :m, :, HD:].double()
        return [q_out, gate_out, kp, vp] if c["gate"] else [q_out, kp, vp]
    if c["op"] == "kv_commit":
        taken = []
        for b in range(c["batch"]):
            path = _path(parents[b], int(s["leaf"][b]))
            taken.append(len(path))
            for pool in (kp, vp):
                rows, _ = _token_rows(pool, s["table"][b], c["n_kv"], base[b], n)
                if path:
                    _put_rows(pool, _token_rows(pool, s["table"][b], c["n_kv"], base[b], len(path))[1], rows[path])
        return [kp, vp, torch.tensor(taken, dtype=torch.int32, device="cuda")]
    o, G = s["o"].double(), c["n_q"] // c["n_kv"]
    for b in range(c["batch"]):
        m = counts[b]
        k, _ = _token_rows(s["k_pool"], s["table"][b], c["n_kv"], 0, base[b] + m)
        v, _ = _token_rows(s["v_pool"], s["table"][b], c["n_kv"], 0, base[b] + m)
        hidden = torch.ones(m, m, dtype=torch.bool)
        for i in range(m):
            hidden[i, _path(parents[b], i)] = False
        for h in range(c["n_q"]):
            x = s["q"][b, :m, h].double() @ k[:, h // G].T / 16.0
            x[:, base[b]:].masked_fill_(hidden.cuda(), -math.inf)
            o[b, :m, h] = (torch.softmax(x, -1) @ v[:, h // G]) / (1 + torch.exp(-s["gate"][b, :m, h].double()))
    return [o]


def _exact_gdn(s, parents, counts):
    c, dim = s["case"], s["qkv"].shape[2]
    qd, w = c["n_qk"] * DK, s["conv_w"].double()
    hs = torch.tensor([h % c["n_qk"] if c["tiled"] else h // (c["n_v"] // c["n_qk"]) for h in range(c["n_v"])], device="cuda")
    S_all, ring_all = s["S"].double() if c["op"] == "gdn_commit" else None, s["ring"].double()
    o = torch.zeros(c["batch"], c["nodes"], c["n_v"], DK, dtype=torch.float64, device="cuda")
    for b in range(c["batch"]):
        slot = int(s["slots"][b])
        phase = int(s["phase"][slot])
        window = [s["ring"][slot][:, (phase + j) % TAPS].double() for j in range(TAPS)]    # oldest first
        states = {-1: (s["S"][slot].double(), window)}
        nodes = range(counts[b]) if c["op"] == "gdn" else _path(parents[b], int(s["leaf"][b]))
        left = [0] * (c["nodes"] + 1)
        for i in nodes:
            left[parents[b][i]] += 1
        for i in nodes:
            p = parents[b][i]
            S, win = states[p]
            left[p] -= 1
            if not left[p] and p >= 0:
                del states[p]
            win = win[1:] + [s["qkv"][b, i].double()]
            y = sum(win[j] * w[:, j] for j in range(TAPS))
            y = y / (1 + torch.exp(-y))
            q, k, v = y[:qd].view(-1, DK)[hs], y[qd:2 * qd].view(-1, DK)[hs], y[2 * qd:].view(-1, DK)
            q = q / (q.square().sum(-1, keepdim=True) + EPS).sqrt() / DK ** 0.5
            k = k / (k.square().sum(-1, keepdim=True) + EPS).sqrt()
            S = S * torch.exp(s["g_log"][b, i].double()).view(-1, 1, 1)
            delta = s["beta"][b, i].double().view(-1, 1) * (v - (k.unsqueeze(1) @ S).squeeze(1))
            S = S + k.unsqueeze(2) * delta.unsqueeze(1)
            o[b, i] = (q.unsqueeze(1) @ S).squeeze(1)
            if left[i] or c["op"] == "gdn_commit":
                states[i] = (S, win)
        if c["op"] == "gdn_commit" and len(nodes):
            S, win = states[nodes[-1]]
            S_all[slot] = S
            for j in range(TAPS):
                ring_all[slot][:, (phase + j) % TAPS] = win[j]
    return [o] if c["op"] == "gdn" else [S_all, ring_all]
