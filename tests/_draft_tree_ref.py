"""Plain 64-bit forms of a speculative decoding step's operators, for the tests."""
import math

import torch

ONE = 2.0 ** 44


def used(parents):
    """Whether each node is part of the tree: its parent is -1 or an earlier node that is."""
    out = []
    for i, p in enumerate(parents):
        out.append(p == -1 or (0 <= p < i and out[p]))
    return out


def lines(parents):
    """For each node the list of its ancestors and itself; unused nodes: empty."""
    out, ok = [], used(parents)
    for i, p in enumerate(parents):
        out.append([] if not ok[i] else (out[p] if p >= 0 else []) + [i])
    return out


def bits(parents):
    n = len(parents)
    m = torch.zeros(n, n, dtype=torch.bool)
    for i, line in enumerate(lines(parents)):
        m[i, line] = True
    return m


def words(m):
    """Bits [rows, n] as int64 words [rows, ceil(n / 64)]."""
    rows, n = m.shape
    wide = torch.zeros(rows, -(-n // 64) * 64, dtype=torch.bool)
    wide[:, :n] = m
    return (wide.view(rows, -1, 64).long() << torch.arange(64)).sum(-1)


def attention(q, k, v, m):
    """(outputs, bound of their error) of q [n, Hq, hd] over k, v [L, Hkv, hd] (float64) with m [n, n] for the last n
    rows. Bound: a weight's rounding to bf16 is 2^-8 relative at most and moves a row by 2^-8 of its weighted distance from
    the values; scores carry fp32 sums of hd products, a multiplication and an exponential; sums and outputs fp32 sums
    over L keys in chains; the output is rounded to bf16."""
    n, hq, hd = q.shape
    rows, hkv, _ = k.shape
    sees = torch.ones(n, rows, dtype=torch.bool, device=q.device)
    sees[:, rows - n:] = m.to(q.device)
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    for h in range(hq):
        kh, vh = k[:, h * hkv // hq], v[:, h * hkv // hq]
        s = (q[:, h] @ kh.T.contiguous()) / math.sqrt(hd)
        mag = (q[:, h].abs() @ kh.abs().T.contiguous()) / math.sqrt(hd)
        s = s.masked_fill(~sees, -math.inf)
        p = torch.softmax(s, -1)
        p = torch.where(sees.any(-1, keepdim=True), p, torch.zeros_like(p))
        o = p @ vh
        err = torch.where(sees, mag, torch.zeros_like(mag)).amax(-1, keepdim=True) * (hd + 4) * 2.0 ** -24 * 2 + 2.0 ** -20
        far = torch.stack([(p[i][:, None] * (vh - o[i]).abs()).sum(0) for i in range(n)])
        size = p @ vh.abs()
        tol[:, h] = (2.0 ** -8 * 1.01 + err) * far + (2.0 ** -8 * 1.01) * o.abs() + (rows / 32 + 64) * 2.0 ** -24 * size + 1e-30
        out[:, h] = o
    return out, tol


def f32(x):
    return float(torch.tensor(x, dtype=torch.float32))


def masses(x, t):
    """x [rows, vocab] float64 without NaN."""
    top = x.amax(-1, keepdim=True)
    d = torch.where(x == top, torch.zeros_like(x), x - top)
    w = torch.round(torch.exp(d / f32(t)) * ONE).long()
    return torch.where(top == -math.inf, torch.zeros_like(w), w)


def sample(logits, u, t=1.0, k=0, p=1.0, min_p=0.0):
    """Tokens of logits [rows, vocab] (fp32 or bf16) with random numbers u [rows]."""
    x = logits.double()
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    w = masses(x, t)
    least = max(1, math.ceil(f32(min_p) * ONE))
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    ranked = w.gather(1, order)
    ranked = torch.where(ranked >= least, ranked, torch.zeros_like(ranked))
    if k > 0:
        ranked[:, k:] = 0
    if p < 1:
        mass = ranked.cumsum(-1)
        need = torch.ceil(mass[:, -1:].double() * f32(p)).long().clamp(min=1)
        ranked = torch.where(mass - ranked < need, ranked, torch.zeros_like(ranked))
    w = torch.zeros_like(w).scatter_(1, order, ranked)
    mass = w.cumsum(-1)
    total = mass[:, -1:]
    ud = torch.nan_to_num(u.double(), nan=0.0).clamp(0, 1)[:, None]
    r = torch.minimum(torch.floor(total.double() * ud).long(), total - 1)
    token = (mass <= r).sum(-1)
    return torch.where(total[:, 0] > 0, token, torch.full_like(token, -1)).int()


def accept(parents, draft, target):
    """The accepted path."""
    path = [0]
    while True:
        child = [c for c in range(path[-1] + 1, len(parents))
                 if parents[c] == path[-1] and draft[c] >= 0 and draft[c] == target[path[-1]]]
        if not child:
            return path
        path.append(child[0])


def random_tree(n, gen, roots=1, reach=None):
    """Parents of n nodes, each drawn from the `reach` nodes before it (all)."""
    out = [-1] * min(roots, n)
    for i in range(len(out), n):
        low = 0 if reach is None else max(0, i - reach)
        out.append(int(torch.randint(low, i, (1,), generator=gen)))
    return out
