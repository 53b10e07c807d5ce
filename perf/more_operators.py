"""Performance cases of a speculative decoding step's operators, through the C ABI.

A case is a dict of plain values. `listed()` gives the cases that are always measured, `draw()` more of the same
ranges; `prepare()` makes what a program has in hand before the call, `run()` is one pass, `exact()` the same pass in
64 bits, `work()` what the pass cannot do without. With `own` false, `run()` computes the operators in elementary
torch operations; with `own` true it makes the framework's calls.

Kinds of cases:
  plan    ancestor masks and positions of a tree of drafted tokens, from their parents
  tree    attention of the tree's tokens over a cache that holds their own keys in its last rows
  sample  a token for each row of logits: temperature, top-k, top-p and min-p, with given random numbers
  commit  the path through the tree that the drawn tokens accept, and its rows' move to their places in the cache

Layer dimensions are those of efm_setup's model shapes.
"""
import math
import os
import sys

import torch

own = False

# (layers, heads, kv heads, head_dim)
MODELS = {"0p5b": (24, 14, 2, 64), "1p5b": (28, 12, 2, 128), "vl3b": (36, 16, 2, 128), "7b": (28, 28, 4, 128)}
VOCAB = 151936
ONE = 2.0 ** 44   # a sampler's mass of the likeliest token


def _capi():
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "edge-fm-x_amd"))
    import efm_capi

    return efm_capi


def listed():
    return [
        # the smallest tree of a step: a root and a few drafts
        dict(name="plan_small", kind="plan", nodes=7, depth=3, prefix=300),
        # the largest tree that is planned
        dict(name="plan_large", kind="plan", nodes=1000, depth=24, prefix=20000),
        # a few drafted tokens of a short chat on the narrow model (head_dim 64): latency counts
        dict(name="tree_small", kind="tree", model="0p5b", nodes=5, depth=4, prefix=300),
        # an ordinary tree in the middle of a chat
        dict(name="tree_chat", kind="tree", model="1p5b", nodes=24, depth=6, prefix=2003),
        # a tree over a long cached context
        dict(name="tree_long", kind="tree", model="7b", nodes=33, depth=7, prefix=32000),
        # many candidates at once, a draft model's wide beams
        dict(name="tree_wide", kind="tree", model="vl3b", nodes=250, depth=9, prefix=3900),
        # one row of a pruned vocabulary, min-p alone
        dict(name="sample_compact", kind="sample", rows=1, vocab=8192, bf16=False, t=0.7, k=0, p=1.0, min_p=0.05, pad=0),
        # a decode step's row, every filter on
        dict(name="sample_row", kind="sample", rows=1, vocab=VOCAB, bf16=False, t=0.8, k=50, p=0.95, min_p=0.02, pad=0),
        # the rows of a tree, nucleus sampling
        dict(name="sample_tree", kind="sample", rows=33, vocab=VOCAB, bf16=False, t=1.0, k=0, p=0.9, min_p=0.0, pad=0),
        # the rows of a wide tree, 16-bit logits in a buffer of padded rows
        dict(name="sample_wide", kind="sample", rows=250, vocab=VOCAB, bf16=True, t=1.0, k=200, p=0.98, min_p=0.0, pad=64),
        # the end of a step with few drafts on the narrow model
        dict(name="commit_small", kind="commit", model="0p5b", nodes=7, depth=3, accepted=3, prefix=300),
        # the end of a step with a large tree on the model with the most cache
        dict(name="commit_large", kind="commit", model="7b", nodes=120, depth=12, accepted=9, prefix=4000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "tree", "tree", "tree", "tree", "sample", "sample", "sample", "commit"])
    if kind == "plan":
        nodes = _log(rng, 1, 1000)
        return dict(kind=kind, nodes=nodes, depth=rng.randint(0, min(nodes - 1, 40)), prefix=_log(rng, 1, 60000))
    if kind == "tree":
        model, nodes = rng.choice(sorted(MODELS)), _log(rng, 1, 250)
        prefix = rng.choice([0, _log(rng, 1, 32000), _log(rng, 1, 32000)])
        prefix = min(prefix, 28 * 33 * 32000 // (nodes * MODELS[model][1]))   # no more work than the largest listed case's
        return dict(kind=kind, model=model, nodes=nodes, depth=rng.randint(0, min(nodes - 1, 12)), prefix=prefix)
    if kind == "sample":
        return dict(kind=kind, rows=rng.choice([1, _log(rng, 2, 250)]), vocab=_log(rng, 1000, VOCAB), bf16=rng.random() < 0.4,
                    t=rng.uniform(0.3, 1.5), k=rng.choice([0, _log(rng, 1, 1000)]), p=rng.choice([1.0, rng.uniform(0.5, 0.99)]),
                    min_p=rng.choice([0.0, rng.uniform(0.005, 0.2)]), pad=rng.choice([0, 8 * rng.randint(1, 16)]))
    accepted = rng.randint(1, 10)
    nodes = _log(rng, 2 * accepted + 2, 250)
    return dict(kind=kind, model=rng.choice(sorted(MODELS)), nodes=nodes, depth=rng.randint(max(1, accepted - 1), accepted + 1),
                accepted=accepted, prefix=_log(rng, 1, 16000))


# Inputs, from the seed alone: activations and cached values N(0, 1), a few channels of the keys several times larger;
# logits of a bulk and a few likely tokens; trees level by level, every node's parent drawn from the level above.

def _rng(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *size):
    return torch.randn(*size, generator=g, device="cuda").to(torch.bfloat16)


def _keys(g, *size):
    k = torch.randn(*size, generator=g, device="cuda")
    k[..., torch.randperm(size[-1], generator=g, device="cuda")[:3]] *= 6.0
    return k.to(torch.bfloat16)


def _levels(case):
    """Nodes of each level: one root, then `depth` levels, the first with as many nodes at least as a path accepts."""
    nodes, depth = case["nodes"], case["depth"]
    if depth == 0 or nodes == 1:
        return [nodes]   # roots alone
    rest, sizes = nodes - 1, []
    for level in range(depth):
        left = depth - level - 1
        take = rest if left == 0 else max(1, min(rest - left, (2 * rest) // (left + 2)))
        if level == 0 and left > 0:
            take = max(take, min(rest - left, case.get("accepted", 1) - 1))
        sizes.append(take)
        rest -= take
    return [1] + sizes


def _parents(case, seed):
    """Parents of the nodes, -1 for a root; a list."""
    cpu = torch.Generator().manual_seed(seed)
    sizes, parents, first = _levels(case), [], 0
    for level, size in enumerate(sizes):
        if level == 0:
            parents += [-1] * size
            continue
        above = sizes[level - 1]
        # the first node of a level, its likeliest, always has a child
        parents += sorted([first] + (first + torch.randint(0, above, (size - 1,), generator=cpu)).tolist())
        first += above
    return parents


def _lines(parents):
    """For each node the nodes from its root to itself."""
    lines = []
    for i, p in enumerate(parents):
        lines.append((lines[p] if p >= 0 else []) + [i])
    return lines


def _plan_inputs(case, seed):
    cached = case["prefix"] + int(torch.randint(0, 4096, (1,), generator=torch.Generator().manual_seed(seed)))
    return dict(parents=torch.tensor(_parents(case, seed), dtype=torch.int32, device="cuda"),
                length=torch.tensor([cached + case["nodes"]], dtype=torch.int32, device="cuda"))


def _tree_inputs(case, seed):
    _, hq, hkv, hd = MODELS[case["model"]]
    g, n = _rng(seed), case["nodes"]
    rows = case["prefix"] + n
    return dict(q=_randn(g, n, hq, hd), k=_keys(g, rows, hkv, hd), v=_randn(g, rows, hkv, hd),
                parents=torch.tensor(_parents(case, seed), dtype=torch.int32, device="cuda"))


def _sample_inputs(case, seed):
    g, n, vocab = _rng(seed), case["rows"], case["vocab"]
    stride = vocab + case["pad"]
    x = 2.5 * torch.randn(n, stride, generator=g, device="cuda")
    likely = torch.randint(0, vocab, (n, 24), generator=g, device="cuda")
    top = 8.0 + 3.0 * torch.empty(n, 24, device="cuda").exponential_(generator=g)
    x.scatter_(1, likely, top)
    x = x.to(torch.bfloat16) if case["bf16"] else x
    return dict(logits=x, u=torch.rand(n, generator=g, device="cuda"))


def _commit_inputs(case, seed):
    layers, _, hkv, hd = MODELS[case["model"]]
    g, cpu, n = _rng(seed), torch.Generator().manual_seed(seed + 1), case["nodes"]
    parents = _parents(case, seed)
    # a path of which no moved row is written over by another, so that a pass can be repeated on the same cache
    paths = [p for p in _lines(parents) if len(p) == case["accepted"] and all(i == x or x >= len(p) for i, x in enumerate(p))]
    path = paths[int(torch.randint(0, len(paths), (1,), generator=cpu))]
    # drafts are below VOCAB - 1000 and differ among siblings; a draw that accepts no draft is above
    drafts = torch.randperm(VOCAB - 1000, generator=cpu)[:n].to(torch.int32)
    drawn = torch.randint(VOCAB - 1000, VOCAB, (n,), generator=cpu, dtype=torch.int32)
    for a, b in zip(path, path[1:]):
        drawn[a] = drafts[b]
    room = _rows(case["prefix"] + n)
    cache = torch.randn(layers, 2, 1, hkv * hd, generator=g, device="cuda").to(torch.bfloat16).repeat(1, 1, room, 1)
    base = case["prefix"]
    cache[:, :, base:base + n] = _randn(g, layers, 2, n, hkv * hd)
    return dict(parents=torch.tensor(parents, dtype=torch.int32, device="cuda"), drafts=drafts.cuda(), drawn=drawn.cuda(),
                cache=cache, length=torch.tensor([base + n], dtype=torch.int32, device="cuda"))


def _rows(n):
    return -(-n // 128) * 128   # the engine's row bound: whole 128-row buckets


def _f32(x):
    return float(torch.tensor(x, dtype=torch.float32))


def prepare(case, seed):
    kind = case["kind"]
    if kind == "plan":
        t = _plan_inputs(case, seed)
    elif kind == "tree":
        t = _tree_inputs(case, seed)
        t["mask"] = _plain_masks(t["parents"])[0]   # planned once a step, for all of its layers
    elif kind == "sample":
        t = _sample_inputs(case, seed)
    else:
        t = _commit_inputs(case, seed)
    state = dict(case=case, **t)
    if own:
        _prepare_own(case, state)
    torch.cuda.synchronize()
    return state


def _prepare_own(case, state):
    """The contexts, outputs and workspaces that a program keeps, and the calls of a pass."""
    C = _capi()
    lib, kind, sh = C.load(), case["kind"], torch.cuda.current_stream().cuda_stream

    def empty(*size, dtype=torch.int32):
        return torch.empty(*size, dtype=dtype, device="cuda")

    def buf(nbytes):
        return torch.zeros(max(int(nbytes), 256), dtype=torch.uint8, device="cuda")

    if kind == "sample":
        n, vocab = case["rows"], case["vocab"]
        out, ws = empty(n), buf(lib.efm_sampler_filtered_workspace_bytes(n, vocab))
        calls = [("efm_sampler_filtered", n, vocab, state["logits"].data_ptr(),
                  C.EFM_DTYPE_BF16 if case["bf16"] else C.EFM_DTYPE_F32, vocab + case["pad"], case["t"], case["k"], case["p"],
                  case["min_p"], state["u"].data_ptr(), out.data_ptr(), ws.data_ptr(), ws.numel(), sh)]
        state.update(C=C, calls=calls, out=dict(token=out), keep=(ws,))
        return
    n = case["nodes"]
    if kind == "plan":
        mask, pos = empty(n, -(-n // 64), dtype=torch.int64), empty(3, n)
        calls = [("efm_draft_tree_plan", n, state["parents"].data_ptr(), 0, state["length"].data_ptr(), 0, mask.data_ptr(),
                  pos.data_ptr(), n, sh)]
        state.update(C=C, calls=calls, out=dict(mask=mask, pos=pos))
        return
    layers, hq, hkv, hd = MODELS[case["model"]]
    ctx = C.make_attention_ctx(hq, hkv, hd, rope=False)
    if kind == "tree":
        rows = case["prefix"] + n
        bound, d_len = _rows(rows), torch.tensor([rows], dtype=torch.int32, device="cuda")
        cache = empty(2, bound, hkv, hd, dtype=torch.bfloat16)
        cache[0, :rows], cache[1, :rows] = state["k"], state["v"]
        o, ws = empty(n, hq * hd, dtype=torch.bfloat16), buf(lib.efm_attention_tree_workspace_bytes(ctx, n, bound))
        calls = [("efm_attention_tree", ctx, state["q"].data_ptr(), cache[0].data_ptr(), cache[1].data_ptr(),
                  state["mask"].data_ptr(), o.data_ptr(), n, 0, d_len.data_ptr(), bound, ws.data_ptr(), ws.numel(), sh)]
        state.update(C=C, calls=calls, out=dict(o=o), keep=(ctx, cache, d_len, ws))
        del state["k"], state["v"]
        return
    cache, base = state["cache"], case["prefix"]
    room, layer = cache.shape[2], 2 * cache.shape[2] * hkv * hd
    length, commit, tokens = empty(1), empty(n + 2), empty(n)
    calls = [("efm_draft_tree_accept", n, state["parents"].data_ptr(), state["drafts"].data_ptr(), state["drawn"].data_ptr(),
              state["length"].data_ptr(), 0, length.data_ptr(), commit.data_ptr(), tokens.data_ptr(), sh),
             ("efm_draft_tree_move_kv", ctx, layers, layer, cache[0, 0].data_ptr(), cache[0, 1].data_ptr(), room, n,
              commit.data_ptr(), sh)]
    state.update(C=C, calls=calls, keep=(ctx,),
                 out=dict(tokens=tokens, commit=commit, length=length, rows=cache[:, :, base:base + n]))


def _words(bits):
    """Bits [n, n] as 64-bit words [n, ceil(n / 64)], bit j of a row in word j / 64."""
    n = bits.shape[1]
    wide = torch.nn.functional.pad(bits.long(), (0, -n % 64)).unflatten(1, (-1, 64))
    return (wide << torch.arange(64, device=bits.device)).sum(-1)


def _plain_masks(parents):
    """(ancestor words, depths): a node's set is its own bit and its parent's set; each pass doubles the generations."""
    n = parents.shape[0]
    bits, up = torch.eye(n, dtype=torch.bool, device=parents.device), parents.long()
    depth = (up >= 0).long()
    for _ in range(max(1, n.bit_length())):
        has, at = up >= 0, up.clamp(min=0)
        bits = bits | (bits[at] & has[:, None])
        depth = depth + torch.where(has, depth[at], 0)
        up = torch.where(has, up[at], -1)
    return _words(bits), depth


def _plain_tree(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    n, hq, hd = q.shape
    rows, hkv, _ = k.shape
    group = hq // hkv
    q = q.view(n, hkv, group, hd).permute(1, 2, 0, 3).reshape(hkv, group * n, hd)
    scores = torch.bmm(q, k.permute(1, 2, 0).contiguous()).view(hkv, group, n, rows) / math.sqrt(hd)
    bits = (s["mask"].unsqueeze(-1) >> torch.arange(64, device=q.device) & 1).flatten(1)[:, :n].bool()
    scores[..., rows - n:].masked_fill_(~bits, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))   # every node sees itself
    p /= p.sum(-1, keepdim=True)
    o = torch.bmm(p.view(hkv, group * n, rows), v.permute(1, 0, 2).contiguous())
    return dict(o=o.view(hq, n, hd).permute(1, 0, 2).reshape(n, hq * hd).bfloat16())


def _plain_sample(s):
    case = s["case"]
    x = s["logits"][:, :case["vocab"]].double()
    w = torch.round(torch.exp((x - x.amax(-1, keepdim=True)) / _f32(case["t"])) * ONE).long()
    kept = w >= math.ceil(_f32(case["min_p"]) * ONE)
    if case["k"] > 0 or case["p"] < 1:
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices   # of equal logits the lowest id first
        ranked = torch.where(kept, w, 0).gather(1, order)
        if case["k"] > 0:
            ranked[:, case["k"]:] = 0
        if case["p"] < 1:
            mass = ranked.cumsum(-1)
            need = torch.ceil(mass[:, -1:].double() * _f32(case["p"])).long().clamp(min=1)
            ranked = torch.where(mass - ranked < need, ranked, 0)
        w = torch.zeros_like(w).scatter_(1, order, ranked)
    else:
        w = torch.where(kept, w, 0)
    mass = w.cumsum(-1)
    total = mass[:, -1:]
    r = torch.minimum(torch.floor(total.double() * s["u"].double()[:, None]).long(), total - 1)
    return dict(token=(mass <= r).sum(-1).int())


def _plain_plan(s):
    words, depth = _plain_masks(s["parents"])
    return dict(mask=words, pos=(s["length"] - depth.shape[0] + depth).int().expand(3, -1).contiguous())


def _plain_commit(s):
    parents, drafts, drawn, base = s["parents"].long(), s["drafts"], s["drawn"], s["case"]["prefix"]
    n = parents.shape[0]
    index = torch.arange(n, device=parents.device)
    accepts = (parents[None] == index[:, None]) & (drafts[None] == drawn[:, None])   # [node, child]
    after = torch.where(accepts, index[None], n).amin(-1)
    after = torch.cat([after, torch.full_like(after[:1], n)])
    at, path = torch.zeros_like(after[:1]), []
    for _ in range(n):
        path.append(at)
        at = after[at]
    path = torch.cat(path)
    on = path < n
    count = on.sum(0, keepdim=True)
    tokens = torch.where(on, drawn[path.clamp(max=n - 1)].long(), -1).int()
    rows = s["cache"][:, :, base:base + n]
    moved = rows[:, :, torch.where(on, path, index)]
    rows.copy_(moved)
    commit = torch.cat([s["length"] - n, count, torch.where(on, path, -1)]).int()
    return dict(tokens=tokens, commit=commit, length=(s["length"] - n + count).int(), rows=rows)


def run(state):
    if own:
        call = state["C"].call
        for args in state["calls"]:
            call(*args)
        return state["out"]
    return dict(plan=_plain_plan, tree=_plain_tree, sample=_plain_sample, commit=_plain_commit)[state["case"]["kind"]](state)


def work(case):
    kind = case["kind"]
    if kind == "sample":
        n = case["rows"] * case["vocab"]
        return dict(bytes=n * (2 if case["bf16"] else 4) + 8 * case["rows"], flops=3 * n)
    n = case["nodes"]
    if kind == "plan":
        return dict(bytes=16 * n + 8 * n * -(-n // 64), flops=n * (case["depth"] + 1))
    layers, hq, hkv, hd = MODELS[case["model"]]
    if kind == "commit":
        moved = max(case["accepted"] - 1, 0)
        return dict(bytes=layers * 2 * moved * hkv * hd * 4 + 20 * n, flops=n)
    seen = n * case["prefix"] + n * (case["depth"] // 2 + 1)
    return dict(bytes=4 * (case["prefix"] + n) * hkv * hd + 4 * n * hq * hd + 8 * n * -(-n // 64), flops=4 * hq * hd * seen)


# The passes in 64 bits, from the operators' definitions.

def _exact_sample(case, seed):
    t = _sample_inputs(case, seed)
    tokens = []
    for row, u in zip(t["logits"], t["u"].tolist()):
        x = row[:case["vocab"]].double()
        top = x.max()
        w = torch.round(ONE * torch.exp((x - top) / _f32(case["t"]))).long()
        w[w < math.ceil(ONE * _f32(case["min_p"]))] = 0
        if case["k"] > 0 or case["p"] < 1:
            # the likely tokens in order: by logit, then by id
            many = min(case["k"] or case["vocab"], case["vocab"])
            cut = torch.topk(x, many).values[-1]
            sure, border = (x > cut).nonzero().flatten(), (x == cut).nonzero().flatten()
            ids = torch.cat([sure[torch.argsort(-x[sure], stable=True)], border])[:many]
            if case["p"] < 1:
                total = int(w[ids].sum())
                need = max(1, math.ceil(float(total) * _f32(case["p"])))
                count = int((w[ids].cumsum(0) < need).sum()) + 1
                ids = ids[:count]
            ids = ids.sort().values
        else:
            ids = torch.arange(case["vocab"], device=x.device)
        mass = w[ids].cumsum(0)
        total = int(mass[-1])
        r = min(total - 1, int(float(total) * u))
        tokens.append(int(ids[int(torch.searchsorted(mass, torch.tensor(r, device=x.device), right=True))]))
    return dict(token=torch.tensor(tokens, dtype=torch.int32, device="cuda"))


def exact(case, seed):
    kind = case["kind"]
    if kind == "sample":
        return _exact_sample(case, seed)
    n = case["nodes"]
    if kind == "plan":
        t, mask = _plan_inputs(case, seed), []
        lines = _lines(t["parents"].tolist())
        for line in lines:
            bits = sum(1 << j for j in line)
            words = [bits >> 64 * i & (1 << 64) - 1 for i in range(-(-n // 64))]
            mask.append([w - (1 << 64) if w >> 63 else w for w in words])
        pos = torch.tensor([int(t["length"]) - n + len(line) - 1 for line in lines], dtype=torch.int32, device="cuda")
        return dict(mask=torch.tensor(mask, dtype=torch.int64, device="cuda"), pos=pos.repeat(3, 1))
    if kind == "commit":
        t = _commit_inputs(case, seed)
        parents, drafts, drawn = (t[x].tolist() for x in ("parents", "drafts", "drawn"))
        path = [0]
        while True:
            child = [c for c in range(n) if parents[c] == path[-1] and drafts[c] == drawn[path[-1]]]
            if not child:
                break
            path.append(child[0])
        rows = t["cache"][:, :, case["prefix"]:case["prefix"] + n].clone()
        for i, p in enumerate(path):
            rows[:, :, i] = rows[:, :, p]
        fill = [-1] * (n - len(path))
        return dict(tokens=torch.tensor([drawn[p] for p in path] + fill, dtype=torch.int32, device="cuda"),
                    commit=torch.tensor([case["prefix"], len(path)] + path + fill, dtype=torch.int32, device="cuda"),
                    length=torch.tensor([case["prefix"] + len(path)], dtype=torch.int32, device="cuda"), rows=rows)
    t = _tree_inputs(case, seed)
    q, k, v = t["q"].double(), t["k"].double(), t["v"].double()
    rows, hq, hd = k.shape[0], q.shape[1], q.shape[2]
    hidden = torch.zeros(n, rows, dtype=torch.bool)
    hidden[:, rows - n:] = True
    for i, line in enumerate(_lines(t["parents"].tolist())):
        hidden[i, rows - n + torch.tensor(line)] = False
    hidden = hidden.cuda()
    heads = []
    for h in range(hq):
        own_k, own_v = k[:, h * k.shape[1] // hq], v[:, h * k.shape[1] // hq]
        s = (q[:, h] @ own_k.T.contiguous() / hd ** 0.5).masked_fill(hidden, -math.inf)
        heads.append(torch.softmax(s, -1) @ own_v)
    return dict(o=torch.stack(heads, 1).flatten(1))
