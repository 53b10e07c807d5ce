"""GPU tests of a speculative decoding step's operators against plain 64-bit forms (_draft_tree_ref).

Tolerances of the attention are derived there; everything else has to be equal."""
import math

import pytest
import torch

import _draft_tree_ref as R
import efm_capi as C
from _util import ptr, stream

pytestmark = pytest.mark.gpu

HEADS = [pytest.param(14, 2, 64, id="0p5b"), pytest.param(12, 2, 128, id="1p5b"), pytest.param(28, 4, 128, id="7b")]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _bf(g, *size, std=1.0):
    return (torch.randn(*size, generator=g) * std).to(torch.bfloat16)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _buf(nbytes, fill=0xff):
    return torch.full((max(int(nbytes), 256),), fill, dtype=torch.uint8, device="cuda")


# ---------------------------------------------------------------- plan

def _plan(parents, rows, device_len=True, off=0, stride=None, want=(True, True)):
    n = len(parents)
    stride = stride or n
    par, d = _i32(parents), _i32([rows])
    mask = torch.full((n, -(-n // 64)), 0x5a, dtype=torch.int64, device="cuda")
    pos = torch.full((3, stride), -7, dtype=torch.int32, device="cuda")
    C.call("efm_draft_tree_plan", n, ptr(par), 0 if device_len else rows, ptr(d) if device_len else None, off,
           ptr(mask) if want[0] else None, ptr(pos) if want[1] else None, stride, stream())
    torch.cuda.synchronize()
    return mask.cpu(), pos.cpu()


def _check_plan(parents, rows, off=0, **kw):
    n = len(parents)
    mask, pos = _plan(parents, rows, off=off, **kw)
    assert torch.equal(mask, R.words(R.bits(parents)))
    want = torch.tensor([rows - n + max(len(x) - 1, 0) + off for x in R.lines(parents)], dtype=torch.int32)
    assert torch.equal(pos[:, :n], want.expand(3, -1))
    assert (pos[:, n:] == -7).all()


@pytest.mark.parametrize("n", [1, 2, 3, 63, 64, 65, 127, 128, 500, 1000, 1024])
@pytest.mark.parametrize("shape", ["chain", "star", "random", "near", "forest"])
def test_plan(gpu, n, shape):
    g = _gen(n)
    parents = dict(chain=list(range(-1, n - 1)), star=[-1] + [0] * (n - 1), random=R.random_tree(n, g),
                   near=R.random_tree(n, g, reach=3), forest=R.random_tree(n, g, roots=min(n, 5)))[shape]
    _check_plan(parents, 3000 + n, off=-17)


@pytest.mark.parametrize("device_len", [False, True])
def test_plan_unused_nodes(gpu, device_len):
    """Parents that are neither -1 nor earlier nodes, and their descendants; rows right at the nodes' number."""
    parents = [-1, 0, -2, 2, 3, 5, 9, 1, 2 ** 31 - 1, -2 ** 31, 9, 7, 8, 3]
    _check_plan(parents, len(parents), device_len=device_len, stride=20)
    chain = [-5] + list(range(700))
    _check_plan(chain, 5000, device_len=device_len)


def test_plan_single_outputs_and_short_lengths(gpu):
    parents = [-1, 0, 0, 1]
    mask, pos = _plan(parents, 104, want=(True, False))
    assert torch.equal(mask, R.words(R.bits(parents))) and (pos == -7).all()
    mask, pos = _plan(parents, 104, want=(False, True))
    assert (mask == 0x5a).all() and pos[0].tolist() == [100, 101, 101, 102]
    mask, pos = _plan(parents, 3, off=11)   # fewer rows than nodes: every node is unused
    assert (mask == 0).all() and (pos == 11).all()


# ---------------------------------------------------------------- attention

class _Attn:
    """Inputs of a call, on the host; `call` runs it with the layout asked for."""

    def __init__(self, g, hq, hkv, hd, n, prefix, mask=None):
        self.hq, self.hkv, self.hd, self.n, self.rows = hq, hkv, hd, n, prefix + n
        self.q, self.k, self.v = _bf(g, n, hq, hd), _bf(g, self.rows, hkv, hd), _bf(g, self.rows, hkv, hd)
        self.k[..., 3] *= 5
        self.mask = mask if mask is not None else R.bits(R.random_tree(n, g))

    def ref(self):
        return R.attention(self.q.double().cuda(), self.k.double().cuda(), self.v.double().cuda(), self.mask)

    def call(self, device_len=True, bound=None, ws=None, words=None):
        n, hq, hkv, hd = self.n, self.hq, self.hkv, self.hd
        bound = bound or (self.rows + 50 if device_len else self.rows)
        c = C.make_attention_ctx(hq, hkv, hd, rope=False)
        k = torch.full((bound, hkv, hd), math.nan, dtype=torch.bfloat16, device="cuda")   # rows past the end: NaN
        v = torch.full_like(k, math.nan)
        k[:self.rows], v[:self.rows] = self.k.cuda(), self.v.cuda()
        q, mask, d = self.q.cuda(), (R.words(self.mask) if words is None else words).cuda(), _i32([self.rows])
        o = torch.full((n + 1, hq * hd), 7.0, dtype=torch.bfloat16, device="cuda")
        size = C.load().efm_attention_tree_workspace_bytes(c, n, bound)
        ws = _buf(size) if ws is None else ws
        C.call("efm_attention_tree", c, ptr(q), ptr(k), ptr(v), ptr(mask), ptr(o), n, 0 if device_len else self.rows,
               ptr(d) if device_len else None, bound if device_len else 0, ptr(ws), ws.numel(), stream())
        torch.cuda.synchronize()
        assert (o[n] == 7).all()   # the row behind the last is left as it was
        return o[:n].view(n, hq, hd)


def _close(got, ref, tol, what=""):
    got, ref, tol = got.double().cpu(), ref.cpu(), tol.cpu()
    assert torch.equal(torch.isfinite(got), torch.isfinite(ref)), f"{what}: not finite in other places"
    ok = torch.isfinite(ref)
    err = (got - ref).abs()[ok]
    assert bool((err <= tol[ok]).all()), f"{what}: worst {float((err - tol[ok]).max())} past its tolerance"


@pytest.mark.parametrize("hq,hkv,hd", HEADS)
@pytest.mark.parametrize("n,prefix", [(1, 0), (1, 1), (1, 700), (2, 31), (5, 300), (7, 33), (16, 2003), (31, 64), (33, 8001), (64, 0),
                                      (65, 127), (70, 1000), (130, 63), (250, 3900), (600, 17)])
def test_attention(gpu, hq, hkv, hd, n, prefix):
    a = _Attn(_gen(n + prefix), hq, hkv, hd, n, prefix)
    ref, tol = a.ref()
    _close(a.call(), ref, tol, "device length")
    _close(a.call(device_len=False), ref, tol, "host length")


@pytest.mark.parametrize("hq,hkv,hd", [(1, 1, 128), (8, 8, 64), (4, 2, 128), (6, 2, 64), (8, 2, 128), (12, 2, 64), (16, 2, 128), (64, 8, 128),
                                       (14, 14, 128), (9, 3, 128)])
@pytest.mark.parametrize("n,prefix", [(3, 95), (40, 1500)])
def test_attention_head_layouts(gpu, hq, hkv, hd, n, prefix):
    a = _Attn(_gen(hq), hq, hkv, hd, n, prefix)
    _close(a.call(), *a.ref())


@pytest.mark.parametrize("hq,hkv,hd,n,prefix", [(28, 4, 128, 33, 17000), (14, 2, 64, 250, 9300), (12, 2, 128, 1000, 400), (28, 4, 128, 1000, 30),
                                                (4, 2, 128, 1024, 7001), (9, 3, 64, 700, 8333), (28, 4, 128, 1024, 2500)])
def test_attention_much_work(gpu, hq, hkv, hd, n, prefix):
    """Sizes at which 128 rows share a tile, with and without splits."""
    a = _Attn(_gen(n), hq, hkv, hd, n, prefix)
    _close(a.call(), *a.ref())


@pytest.mark.parametrize("hq,hkv,hd", HEADS)
@pytest.mark.parametrize("n,prefix,bound", [(40, 0, 60000), (75, 1000, 40000), (64, 8000, 70000), (130, 63, 9000)])
def test_attention_far_below_the_bound(gpu, hq, hkv, hd, n, prefix, bound):
    """The splits are laid out for the bound: most of them have no keys here."""
    a = _Attn(_gen(n + 1), hq, hkv, hd, n, prefix)
    _close(a.call(bound=bound), *a.ref())


def test_attention_largest_tree(gpu):
    a = _Attn(_gen(4), 12, 2, 128, 1024, 100)
    _close(a.call(), *a.ref())


@pytest.mark.parametrize("hq,hkv,hd", HEADS)
@pytest.mark.parametrize("prefix,bound", [(0, None), (5, None), (1000, None), (0, 60000), (5, 60000), (1000, 60000)])
def test_attention_any_mask(gpu, hq, hkv, hd, prefix, bound):
    """Masks that are no tree's: random bits, later nodes seen, rows without a bit (zeros without a prefix), all bits; and
    bits past the nodes in the mask's words, which are not looked at."""
    g = _gen(prefix)
    n = 75
    m = torch.rand(n, n, generator=g) < 0.3
    m[3], m[74], m[10], m[40, :64], m[41, 64:] = False, False, True, False, False
    a = _Attn(g, hq, hkv, hd, n, prefix, mask=m)
    ref, tol = a.ref()
    got = a.call(bound=bound)
    _close(got, ref, tol)
    if prefix == 0:
        assert (got[3] == 0).all() and (got[74] == 0).all()
    words = R.words(m)
    words[:, 1] |= -1 << (n - 64)
    assert torch.equal(a.call(words=words, bound=bound), got)


@pytest.mark.parametrize("hq,hkv,hd", HEADS)
@pytest.mark.parametrize("prefix,bound", [(0, None), (3, None), (700, None), (0, 60000), (3, 60000), (700, 60000)])
def test_attention_not_finite_where_masked(gpu, hq, hkv, hd, prefix, bound):
    """A node's key and value hold NaN or infinities: the nodes that do not see it are as without it, and those that do
    are not finite in the channels of a value, or everywhere for a NaN key."""
    g = _gen(7)
    n = 40
    parents = R.random_tree(n, g)
    clean = _Attn(g, hq, hkv, hd, n, prefix, mask=R.bits(parents))
    ref, tol = clean.ref()
    a = _Attn(g, hq, hkv, hd, n, prefix, mask=clean.mask)
    a.q, a.k, a.v = clean.q.clone(), clean.k.clone(), clean.v.clone()
    bad = {5: math.nan, 17: math.inf, 29: -math.inf, 39: math.nan}
    sees = torch.zeros(n, hd, dtype=torch.bool)
    for node, x in bad.items():
        a.v[prefix + node, :, 1:hd:node] = x
        sees[:, 1:hd:node] |= clean.mask[:, node, None]
    for node in (11, 38):
        a.k[prefix + node] = math.nan
        sees |= clean.mask[:, node, None]
    got = a.call(bound=bound).double().cpu()
    for h in range(hq):
        assert not torch.isfinite(got[:, h][sees]).any()
        ok = ~sees
        assert bool(((got[:, h] - ref[:, h].cpu()).abs()[ok] <= tol[:, h].cpu()[ok]).all())


@pytest.mark.parametrize("bound", [None, 140000])
def test_attention_prefix_not_finite(gpu, bound):
    """Every node sees the rows before the tree: an infinite value there reaches its channel of every node."""
    a = _Attn(_gen(9), 12, 2, 128, 9, 500)
    ref, tol = a.ref()
    a.v[100, 1, 7] = math.inf
    got = a.call(bound=bound).double().cpu()
    assert not torch.isfinite(got[:, 6:, 7]).any()
    got[:, 6:, 7], ref, tol = 0, ref.cpu(), tol.cpu()
    ref[:, 6:, 7] = 0
    _close(got, ref, tol)


@pytest.mark.parametrize("bound", [None, 140000])
def test_attention_score_extremes(gpu, bound):
    """Scores far apart, and equal ones: large keys, and keys of zeros."""
    a = _Attn(_gen(10), 12, 2, 128, 20, 3000)
    a.k[:1000] *= 30
    a.k[1000:2000] = 0
    a.q[3] = 0
    _close(a.call(bound=bound), *a.ref())


@pytest.mark.parametrize("bound", [None, 600000])
def test_attention_minus_infinity_scores(gpu, bound):
    """All of a row's visible scores are -inf: zeros, as in the other attention operators."""
    a = _Attn(_gen(11), 4, 2, 128, 3, 0, mask=torch.eye(3, dtype=torch.bool))
    a.q[1], a.k[1] = 1, 0
    a.k[1, :, 0] = -math.inf
    got = a.call(bound=bound)
    assert (got[1] == 0).all() and torch.isfinite(got).all()


@pytest.mark.parametrize("hq,hkv,hd", HEADS)
@pytest.mark.parametrize("past", [9, 120000])
def test_attention_strides(gpu, hq, hkv, hd, past):
    """Queries inside a fused q/k/v buffer; a cache with the heads outermost; a cache with wide rows."""
    g = _gen(12)
    n, prefix = 21, 1111
    a = _Attn(g, hq, hkv, hd, n, prefix)
    ref, tol = a.ref()
    rows, bound, width = a.rows, a.rows + past, (hq + 2 * hkv) * hd
    fused = torch.full((n, width), math.nan, dtype=torch.bfloat16, device="cuda")
    fused[:, :hq * hd] = a.q.cuda().flatten(1)
    mask, d = R.words(a.mask).cuda(), _i32([rows])
    for layout in ("heads", "wide"):
        if layout == "heads":
            k = torch.full((hkv, bound, hd), math.nan, dtype=torch.bfloat16, device="cuda")
            v = torch.full((hkv, bound + 3, hd), math.nan, dtype=torch.bfloat16, device="cuda")
            k[:, :rows], v[:, :rows] = a.k.cuda().transpose(0, 1), a.v.cuda().transpose(0, 1)
            st = dict(k_stride_n=hd, k_stride_h=bound * hd, kv_stride_n=hd, kv_stride_h=(bound + 3) * hd)
        else:
            k = torch.full((bound, hkv * hd + 24), math.nan, dtype=torch.bfloat16, device="cuda")
            v = torch.full((bound, hkv * hd + 8), math.nan, dtype=torch.bfloat16, device="cuda")
            k[:rows, :hkv * hd], v[:rows, :hkv * hd] = a.k.cuda().flatten(1), a.v.cuda().flatten(1)
            st = dict(k_stride_n=hkv * hd + 24, kv_stride_n=hkv * hd + 8)
        c = C.make_attention_ctx(hq, hkv, hd, rope=False, q_stride_n=width, **st)
        o = torch.empty(n, hq, hd, dtype=torch.bfloat16, device="cuda")
        ws = _buf(C.load().efm_attention_tree_workspace_bytes(c, n, bound))
        C.call("efm_attention_tree", c, ptr(fused), ptr(k), ptr(v), ptr(mask), ptr(o), n, 0, ptr(d), bound, ptr(ws), ws.numel(), stream())
        torch.cuda.synchronize()
        _close(o, ref, tol, layout)


def test_attention_cache_past_32_bits(gpu):
    """Rows more than 2^32 elements from the cache's start."""
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    hq, hkv, hd, n, prefix, stride = 12, 2, 128, 10, 2300, 1 << 22
    a = _Attn(_gen(13), hq, hkv, hd, n, prefix)
    rows = a.rows
    # one buffer: K, and V 1024 elements on in each row
    both = torch.empty((rows - 1) * stride + 1024 + hkv * hd, dtype=torch.bfloat16, device="cuda")
    kd, vd = both.as_strided((rows, hkv, hd), (stride, hd, 1)), both[1024:].as_strided((rows, hkv, hd), (stride, hd, 1))
    kd.copy_(a.k), vd.copy_(a.v)
    c = C.make_attention_ctx(hq, hkv, hd, rope=False, k_stride_n=stride, kv_stride_n=stride)
    q, mask, o = a.q.cuda(), R.words(a.mask).cuda(), torch.empty(n, hq, hd, dtype=torch.bfloat16, device="cuda")
    ws = _buf(C.load().efm_attention_tree_workspace_bytes(c, n, rows))
    C.call("efm_attention_tree", c, ptr(q), ptr(kd), ptr(vd), ptr(mask), ptr(o), n, rows, None, 0, ptr(ws), ws.numel(), stream())
    torch.cuda.synchronize()
    _close(o, *a.ref())
    # the move of rows that far
    commit = _i32([prefix, 3, 0, 4, 9] + [-1] * (n - 3))
    C.call("efm_draft_tree_move_kv", c, 1, 0, ptr(kd), ptr(vd), rows, n, ptr(commit), stream())
    torch.cuda.synchronize()
    assert torch.equal(kd[prefix + 1].cpu(), a.k[prefix + 4]) and torch.equal(vd[prefix + 2].cpu(), a.v[prefix + 9])
    assert torch.equal(kd[prefix + 3:].cpu(), a.k[prefix + 3:]) and torch.equal(vd[:prefix + 1].cpu(), a.v[:prefix + 1])


@pytest.mark.parametrize("length", [0, 6, -1, 2 ** 31, 2 ** 32 - 1])
@pytest.mark.parametrize("bound", [1000, 140000])
def test_attention_device_length_out_of_range(gpu, length, bound):
    """Lengths below the nodes' number and past the bound: zeros."""
    a = _Attn(_gen(14), 12, 2, 128, 7, 900)
    length = bound + 1 if length == -1 else length
    c = C.make_attention_ctx(12, 2, 128, rope=False)
    k = torch.zeros(bound, 2, 128, dtype=torch.bfloat16, device="cuda")
    q, mask = a.q.cuda(), R.words(a.mask).cuda()
    d = torch.tensor([length - (1 << 32) if length >= 1 << 31 else length], dtype=torch.int32, device="cuda")
    o = torch.full((7, 12 * 128), 5.0, dtype=torch.bfloat16, device="cuda")
    ws = _buf(C.load().efm_attention_tree_workspace_bytes(c, 7, bound))
    C.call("efm_attention_tree", c, ptr(q), ptr(k), ptr(k), ptr(mask), ptr(o), 7, 0, ptr(d), bound, ptr(ws), ws.numel(), stream())
    torch.cuda.synchronize()
    assert (o == 0).all()


def test_attention_one_workspace_serves_smaller_calls(gpu):
    """The largest call's workspace, filled with NaN, under calls of fewer nodes and rows."""
    c = C.make_attention_ctx(28, 4, 128, rope=False)
    ws = _buf(C.load().efm_attention_tree_workspace_bytes(c, 64, 9000))
    for n, prefix in ((64, 8936), (1, 8999), (2, 8000), (9, 5000), (17, 8983), (40, 300), (64, 1000)):
        a = _Attn(_gen(n), 28, 4, 128, n, prefix)
        _close(a.call(ws=ws, bound=n + prefix), *a.ref(), f"{n} nodes behind {prefix}")


@pytest.mark.parametrize("prefix", [9000, 19000])
def test_attention_repeats(gpu, prefix):
    a = _Attn(_gen(15), 28, 4, 128, 33, prefix)
    first = a.call()
    for _ in range(3):
        assert torch.equal(a.call(), first)


def test_attention_chain_is_causal_prefill(gpu):
    """A chain of nodes sees what the rows of a causal prompt see."""
    n, prefix = 45, 2000
    a = _Attn(_gen(16), 28, 4, 128, n, prefix, mask=torch.ones(n, n, dtype=torch.bool).tril())
    got = a.call()
    c = C.make_attention_ctx(28, 4, 128, rope=False)
    q, k, v = a.q.cuda(), a.k.cuda(), a.v.cuda()
    o = torch.empty(n, 28, 128, dtype=torch.bfloat16, device="cuda")
    C.call("efm_attention_prefill", c, ptr(q), ptr(k), ptr(v), ptr(o), n, n + prefix, 1, stream())
    torch.cuda.synchronize()
    ref, tol = a.ref()
    _close(got, ref, tol)
    assert bool(((got.double() - o.double()).abs() <= 2 * tol + 2.0 ** -8 * 3 * ref.abs()).all())


# ---------------------------------------------------------------- sampling

def _sample(x, u, t=1.0, k=0, p=1.0, min_p=0.0, stride=0, vocab=None, rows=None, data=None, ws=None):
    rows, vocab = rows or x.shape[0], vocab or x.shape[1]
    out = torch.full((rows + 1,), -77, dtype=torch.int32, device="cuda")
    ws = _buf(C.load().efm_sampler_filtered_workspace_bytes(rows, vocab)) if ws is None else ws
    dt = C.EFM_DTYPE_BF16 if x.dtype == torch.bfloat16 else C.EFM_DTYPE_F32
    C.call("efm_sampler_filtered", rows, vocab, data or ptr(x), dt, stride, t, k, p, min_p, ptr(u), ptr(out), ptr(ws), ws.numel(), stream())
    torch.cuda.synchronize()
    assert int(out[rows]) == -77
    return out[:rows]


def _logits(seed, rows, vocab, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = 2.5 * torch.randn(rows, vocab, generator=g, device="cuda")
    x.scatter_(1, torch.randint(0, vocab, (rows, 12), generator=g, device="cuda"),
               7 + 3 * torch.rand(rows, 12, generator=g, device="cuda"))
    return x.to(dtype), torch.rand(rows, generator=g, device="cuda")


FILTERS = [dict(), dict(t=0.5), dict(k=1), dict(k=50), dict(k=1000), dict(p=0.9), dict(p=0.3, t=1.4), dict(min_p=0.05), dict(min_p=1.0),
           dict(k=40, p=0.95), dict(k=300, min_p=0.01), dict(p=0.999, min_p=0.002), dict(k=64, p=0.8, min_p=0.1, t=0.7), dict(p=1e-9),
           dict(t=1e-6), dict(t=1e6), dict(t=1e6, p=0.5), dict(t=1e6, k=700, p=0.5), dict(k=2 ** 31 - 1, p=0.99)]


@pytest.mark.parametrize("f", FILTERS, ids=str)
@pytest.mark.parametrize("rows,vocab,dtype", [(1, 151936, torch.float32), (5, 8192, torch.float32), (3, 151936, torch.bfloat16),
                                              (70, 3001, torch.float32), (40, 1000, torch.bfloat16)])
def test_sampler(gpu, f, rows, vocab, dtype):
    x, u = _logits(rows + vocab, rows, vocab, dtype)
    assert torch.equal(_sample(x, u, **f), R.sample(x, u, **f))


@pytest.mark.parametrize("f", [dict(), dict(k=50, p=0.9), dict(p=0.95), dict(min_p=0.03)], ids=str)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (4, 2), (3, 63), (2, 65), (9, 1023), (9, 1025), (2, 32768), (2, 32769), (2, (1 << 20) - 1),
                                        (260, 40000), (600, 700), (1100, 15000), (3, 16384), (3, 16385), (1500, 20000), (127, 50000), (128, 50000)])
def test_sampler_sizes(gpu, f, rows, vocab):
    for dtype in (torch.float32, torch.bfloat16):
        x, u = _logits(vocab, rows, vocab, dtype)
        assert torch.equal(_sample(x, u, **f), R.sample(x, u, **f))


@pytest.mark.parametrize("f", [dict(k=7), dict(k=700), dict(p=0.5), dict(k=900, p=0.6), dict(p=0.999), dict()], ids=str)
@pytest.mark.parametrize("values", [1, 2, 5])
@pytest.mark.parametrize("vocab", [3000, 151936])
def test_sampler_ties(gpu, f, values, vocab):
    """Few different logits, both zeros among them: ties go to the lowest ids."""
    g = torch.Generator(device="cuda").manual_seed(values)
    table = torch.tensor([0.0, -0.0, 1.0, -1.5, -40.0], device="cuda")
    x = table[torch.randint(0, values, (6, vocab), generator=g, device="cuda")]
    u = torch.rand(6, generator=g, device="cuda")
    assert torch.equal(_sample(x, u, **f), R.sample(x, u, **f))


@pytest.mark.parametrize("f", [dict(p=0.9), dict(p=0.5, t=3.0), dict(p=0.999), dict(k=5000), dict(k=2500, p=0.7), dict(k=9000, p=0.99, min_p=0.02),
                               dict(min_p=0.3), dict(p=0.8, min_p=0.2)], ids=str)
@pytest.mark.parametrize("shift", [0.0, 1e4, -1e4])
@pytest.mark.parametrize("rows,vocab", [(1, 151936), (4, 16000), (7, 4097), (257, 16000)])
def test_sampler_flat_rows(gpu, f, shift, rows, vocab):
    """Thousands of ids of nearly the same mass at the place where the choice ends; logits far from zero."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = 0.6 * torch.randn(rows, vocab, generator=g, device="cuda") + shift
    u = torch.rand(rows, generator=g, device="cuda")
    for y in (x, x.bfloat16()):
        assert torch.equal(_sample(y, u, **f), R.sample(y, u, **f))


@pytest.mark.parametrize("f", [dict(p=0.9), dict(p=0.3), dict(k=700), dict(k=2000, p=0.5), dict(p=0.95, min_p=0.9)], ids=str)
@pytest.mark.parametrize("rows,width", [(1, 9600), (5, 1500), (3, 40), (130, 9600)])
def test_sampler_clusters(gpu, f, rows, width):
    """Neighbouring ids hold nearly all of the mass: few runs of many kept ids."""
    vocab = 151936
    g = torch.Generator(device="cuda").manual_seed(width)
    x = torch.randn(rows, vocab, generator=g, device="cuda")
    for r in range(rows):
        at = (r * 7919 + 1001) % (vocab - width)
        x[r, at:at + width] = 25 + 0.05 * x[r, at:at + width]
    u = torch.rand(rows, generator=g, device="cuda")
    for y in (x, x.bfloat16()):
        assert torch.equal(_sample(y, u, **f), R.sample(y, u, **f))


@pytest.mark.parametrize("f", [dict(), dict(k=20), dict(p=0.9), dict(min_p=0.1), dict(k=30, p=0.7, min_p=0.01)], ids=str)
@pytest.mark.parametrize("vocab", [2000, 100000])
def test_sampler_rows_that_are_not_finite(gpu, f, vocab):
    """NaN and infinities among the logits; rows with one finite logit, one +inf, several, and none (-1)."""
    x, u = _logits(3, 9, vocab)
    x[0, ::3], x[1, 1::2] = math.nan, -math.inf
    x[2], x[3] = -math.inf, math.nan
    x[4] = -math.inf
    x[4, vocab - 7] = -1e30
    x[5, 1234], x[6, 100:1500:9] = math.inf, math.inf
    x[7, 5], x[7, 6] = 3.4e38, -3.4e38
    x[8, vocab // 2:] = torch.finfo(torch.float32).min
    got = _sample(x, u, **f)
    assert torch.equal(got, R.sample(x, u, **f))
    assert got[2] == -1 and got[3] == -1 and got[4] == vocab - 7 and got[5] == 1234


@pytest.mark.parametrize("f", [dict(k=20), dict(k=3000), dict(k=50, p=0.9), dict(p=0.9), dict(min_p=0.02), dict()], ids=str)
@pytest.mark.parametrize("rows,vocab", [(3, 10000), (2, 151936), (140, 30000)])
def test_sampler_masked_rows(gpu, f, rows, vocab):
    """Rows with -inf for all but some ids, as a grammar leaves them: in one run, every 1000th, and all below zero."""
    x, u = _logits(5, rows, vocab)
    keep = torch.zeros(rows, vocab, dtype=torch.bool, device="cuda")
    keep[0, 64:90], keep[1:, 13::1000] = True, True
    x = torch.where(keep, x, -math.inf)
    x[1:] -= 60
    assert torch.equal(_sample(x, u, **f), R.sample(x, u, **f))


def test_sampler_random_numbers_at_the_ends(gpu):
    x, _ = _logits(4, 8, 5000)
    x[:] = x[0]
    u = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, 5.0, math.inf, -1.0, math.nan, 2.0 ** -140], device="cuda")
    for f in (dict(), dict(k=9), dict(p=0.5)):
        got = _sample(x, u, **f)
        assert torch.equal(got, R.sample(x, u, **f))
        first, last = int(got[0]), int(got[1])
        assert got.tolist() == [first, last, last, last, last, first, first, first] and first <= last


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [8192, 60001])
def test_sampler_strides_and_offsets(gpu, dtype, vocab):
    """Padded rows whose padding would win, and rows that start at any element."""
    for pad, shift in ((1, 0), (64, 1), (7, 3), (0, 5)):
        x, u = _logits(pad, 5, vocab, dtype)
        flat = torch.full((shift + 5 * (vocab + pad) + 8,), 1e4, dtype=dtype, device="cuda")
        flat[shift:shift + 5 * (vocab + pad)].view(5, -1)[:, :vocab] = x
        got = _sample(x, u, t=0.8, k=60, p=0.95, stride=vocab + pad, data=flat.data_ptr() + shift * flat.element_size())
        assert torch.equal(got, R.sample(x, u, t=0.8, k=60, p=0.95)), (pad, shift)


def test_sampler_row_offsets_past_32_bits(gpu):
    rows, vocab, stride = 3, 5000, 1 << 31
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 30 GB")
    x, u = _logits(6, rows, vocab)
    flat = torch.empty(2 * stride + vocab, device="cuda")
    for r in range(rows):
        flat[r * stride:r * stride + vocab] = x[r]
    for f in (dict(p=0.9), dict(k=40), dict(min_p=0.05)):
        assert torch.equal(_sample(x, u, stride=stride, data=flat.data_ptr(), **f), R.sample(x, u, **f))


def test_sampler_rows_do_not_meet(gpu):
    """A row's token is the same alone and among others, and with a workspace that held other calls."""
    x, u = _logits(8, 90, 151936)
    for f in (dict(k=50, p=0.9), dict(p=0.95, t=1.3), dict(min_p=0.02)):
        all_rows = _sample(x, u, **f)
        for r in (0, 41, 89):
            assert torch.equal(_sample(x[r:r + 1], u[r:r + 1], **f), all_rows[r:r + 1])


def test_sampler_workspace_serves_calls_of_any_size(gpu):
    """One workspace under calls of other sizes, filters and types, overflowing lists among them."""
    ws = _buf(C.load().efm_sampler_filtered_workspace_bytes(64, 1 << 19))
    for i in range(3):
        for rows, vocab, f in ((64, 20000, dict(p=0.9)), (1, 151936, dict(k=50)), (7, 500000, dict(p=0.99, t=1.5)), (33, 151936, dict(k=900, p=0.9)),
                               (2, 40000, dict()), (5, 30000, dict(t=1e6, p=0.5)), (5, 30000, dict(t=1e6, k=9)), (64, 15000, dict(min_p=0.1))):
            x, u = _logits(i, rows, vocab, (torch.float32, torch.bfloat16)[i % 2])
            if i == 2:
                x[:, ::2] = 1.0
            assert torch.equal(_sample(x, u, ws=ws, **f), R.sample(x, u, **f)), (rows, vocab, f)


def test_sampler_draws_the_distribution(gpu):
    """Evenly spaced random numbers draw each id as often as its probability says, to one draw."""
    vocab, rows = 50, 4096
    x, _ = _logits(9, 1, vocab)
    u = (torch.arange(rows, device="cuda") + 0.5) / rows
    got = _sample(x.expand(rows, -1).contiguous(), u, t=0.9)
    p = torch.softmax(x[0].double() / 0.9, -1)
    count = torch.bincount(got.long(), minlength=vocab)
    assert bool(((count - p * rows).abs() <= 1.01).all())


# ---------------------------------------------------------------- accept and move

def _accept(parents, draft, target, rows, next_nodes=0, in_place=False):
    n = len(parents)
    args = [_i32(x) for x in (parents, draft, target)]
    d = _i32([rows])
    out = d if in_place else _i32([-9])
    commit, tokens = torch.full((n + 3,), -77, dtype=torch.int32, device="cuda"), torch.full((n + 1,), -77, dtype=torch.int32, device="cuda")
    C.call("efm_draft_tree_accept", n, *[ptr(x) for x in args], ptr(d), next_nodes, ptr(out), ptr(commit), ptr(tokens), stream())
    torch.cuda.synchronize()
    assert int(commit[n + 2]) == -77 and int(tokens[n]) == -77
    return commit[:n + 2].tolist(), tokens[:n].tolist(), int(out[0])


def _check_accept(parents, draft, target, rows, **kw):
    n = len(parents)
    path = R.accept(parents, draft, target)
    commit, tokens, length = _accept(parents, draft, target, rows, **kw)
    fill = [-1] * (n - len(path))
    assert commit == [rows - n, len(path)] + path + fill
    assert tokens == [target[p] for p in path] + fill
    assert length == rows - n + len(path) + kw.get("next_nodes", 0)
    return path


@pytest.mark.parametrize("n", [1, 2, 5, 64, 65, 300, 1024])
@pytest.mark.parametrize("in_place", [False, True])
def test_accept(gpu, n, in_place):
    for seed in range(4):
        g = _gen(seed)
        parents = R.random_tree(n, g, reach=(None, 4, 30, 2)[seed])
        draft = torch.randint(0, 3, (n,), generator=g).tolist()   # few tokens: siblings often agree, the lowest index wins
        target = torch.randint(0, 3, (n,), generator=g).tolist()
        _check_accept(parents, draft, target, 500 + n, next_nodes=seed * 7, in_place=in_place)


def test_accept_whole_chain(gpu):
    n = 1024
    assert len(_check_accept(list(range(-1, n - 1)), list(range(n)), list(range(1, n + 1)), n)) == n


def test_accept_unused_nodes_and_missing_tokens(gpu):
    parents = [-1, 0, 0, -2, 2, 4, 9, 5, -1]
    # node 1 has no token (-1) and neither has node 0's row: they do not match; node 2 is accepted, then 4, 5
    assert _check_accept(parents, [9, -1, 3, 3, 4, 5, 6, 7, 3], [-1] * 9, 100) == [0]
    assert _check_accept(parents, [9, -1, 3, 3, 4, 5, 6, 7, 3], [3, 1, 4, 4, 5, 8, 6, 7, 3], 100) == [0, 2, 4, 5]
    # fewer rows than nodes: nothing
    commit, tokens, length = _accept(parents, [0] * 9, [0] * 9, 8, next_nodes=5)
    assert commit == [0, 0] + [-1] * 9 and tokens == [-1] * 9 and length == 8


@pytest.mark.parametrize("hq,hkv,hd", HEADS)
@pytest.mark.parametrize("path", [[0], [0, 1, 2], [0, 3, 4, 9], [0, 2, 3, 5, 6, 7, 8, 9, 10, 11, 13, 14, 18, 19], list(range(20)), [5, 19], []],
                         ids=str)
def test_move(gpu, hq, hkv, hd, path):
    g = _gen(len(path))
    layers, rows, n, base = 3, 70, 20, 41
    cache = _bf(g, layers, 2, rows, hkv * hd)
    dev = cache.cuda()
    c = C.make_attention_ctx(hq, hkv, hd, rope=False)
    commit = _i32([base, len(path)] + path + [-1] * (n - len(path)))
    C.call("efm_draft_tree_move_kv", c, layers, 2 * rows * hkv * hd, ptr(dev[0, 0]), ptr(dev[0, 1]), rows, n, ptr(commit), stream())
    torch.cuda.synchronize()
    want = cache.clone()
    for i, p in enumerate(path):
        want[:, :, base + i] = cache[:, :, base + p]
    assert torch.equal(dev.cpu(), want)


def test_move_with_the_heads_outermost(gpu):
    hkv, hd, layers, rows, n = 4, 64, 2, 50, 8
    k, v = _bf(_gen(1), layers, hkv, rows, hd).cuda(), _bf(_gen(2), layers, hkv, rows, hd).cuda()
    k0, v0 = k.clone(), v.clone()
    c = C.make_attention_ctx(8, hkv, hd, rope=False, k_stride_n=hd, k_stride_h=rows * hd, kv_stride_n=hd, kv_stride_h=rows * hd)
    commit = _i32([rows - n, 3, 0, 2, 7] + [-1] * 5)
    C.call("efm_draft_tree_move_kv", c, layers, hkv * rows * hd, ptr(k), ptr(v), rows, n, ptr(commit), stream())
    torch.cuda.synchronize()
    for i, p in enumerate((0, 2, 7)):
        k0[:, :, rows - n + i], v0[:, :, rows - n + i] = k0[:, :, rows - n + p].clone(), v0[:, :, rows - n + p].clone()
    assert torch.equal(k, k0) and torch.equal(v, v0)


@pytest.mark.parametrize("commit", [[43, 3, 0, 2, 3], [-1, 3, 0, 2, 3], [10, -4, 0, 2, 3], [2 ** 31 - 1, 3, 0, 2, 3]], ids=str)
def test_move_that_would_leave_the_cache(gpu, commit):
    """A base past the cache (here 43 + 8 of 50 rows) and a negative count move nothing."""
    k = _bf(_gen(3), 50, 256).cuda()
    v, k0 = k.clone(), k.clone()
    c = C.make_attention_ctx(12, 2, 128, rope=False)
    d = _i32(commit + [-1] * 5)
    C.call("efm_draft_tree_move_kv", c, 1, 0, ptr(k), ptr(v), 50, 8, ptr(d), stream())
    torch.cuda.synchronize()
    assert torch.equal(k, k0) and torch.equal(v, k0)


@pytest.mark.parametrize("path,moved", [([0, 3, 2, 6], 2), ([0, 3, 8, 9], 2), ([0, 4, -1, 5], 2), ([0, 4, 4, 5], 2), ([0, 2, 5, 7, 1, 1, 1, 1, 7], 4)], ids=str)
def test_move_of_a_path_that_does_not_rise(gpu, path, moved):
    """The move ends where the path falls, repeats itself or leaves the tree's 8 nodes."""
    k = _bf(_gen(4), 50, 256).cuda()
    v, want = k.clone(), k.clone()
    for i, p in enumerate(path[:moved]):
        want[20 + i] = k[20 + p]
    c = C.make_attention_ctx(12, 2, 128, rope=False)
    d = _i32([20, len(path)] + path + [-1] * 8)
    C.call("efm_draft_tree_move_kv", c, 1, 0, ptr(k), ptr(v), 50, 8, ptr(d), stream())
    torch.cuda.synchronize()
    assert torch.equal(k, want) and torch.equal(v, want)


@pytest.mark.parametrize("hq,hkv,hd", [(9, 9, 128), (6, 3, 64)])
@pytest.mark.parametrize("end", [None, 1, 63, 64, 65, 127, 128, 200])
def test_move_of_long_paths(gpu, hq, hkv, hd, end):
    """Hundreds of accepted nodes, whole or up to entry `end`, which repeats the one before it."""
    n, base, g = 700, 5, _gen(hkv)
    path = torch.cat([torch.arange(70), 70 + torch.randperm(n - 70, generator=g)[:190].sort().values]).tolist()
    moved = len(path) if end is None else end
    if end is not None:
        path[end] = path[end - 1]
    k, v = _bf(g, base + n, hkv * hd).cuda(), _bf(g, base + n, hkv * hd).cuda()
    k0, v0 = k.clone(), v.clone()
    at = torch.tensor(path[:moved], device="cuda") + base
    k0[base:base + moved], v0[base:base + moved] = k[at], v[at]
    c = C.make_attention_ctx(hq, hkv, hd, rope=False)
    commit = _i32([base, len(path)] + path + [-1] * (n - len(path)))
    C.call("efm_draft_tree_move_kv", c, 1, 0, ptr(k), ptr(v), base + n, n, ptr(commit), stream())
    torch.cuda.synchronize()
    assert torch.equal(k, k0) and torch.equal(v, v0)


# ---------------------------------------------------------------- a step

class _Step:
    """Steps of a model of one layer whose qkv rows depend on the token alone: its cache has to hold, bit for bit, what a
    prefill of the accepted text writes."""
    VOCAB, MAX = 16, 1600

    def __init__(self, hq, hkv, hd, n, prefix, seed=5, ws=None):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.hq, self.hkv, self.hd, self.n = hq, hkv, hd, n
        bf = lambda *s, std: (torch.randn(*s, generator=g, device="cuda") * std).bfloat16()
        self.table = bf(self.VOCAB, (hq + 2 * hkv) * hd, std=1.0)
        self.head, self.qw, self.kw = bf(self.VOCAB, hq * hd, std=2 / math.sqrt(hd)), bf(hd, std=1.0), bf(hd, std=1.0)
        self.ctx = C.make_attention_ctx(hq, hkv, hd, rope=True)
        self.plain = C.make_attention_ctx(hq, hkv, hd, rope=False)
        self.text = torch.randint(0, self.VOCAB, (prefix,), generator=g, device="cuda").tolist()
        self.cache = torch.full((2, self.MAX, hkv, hd), math.nan, dtype=torch.bfloat16, device="cuda")
        self.write(self.text, self.cache)
        # every node but the root guesses a token; the children of a node guess different ones
        self.parents = [-1] + [(i - 1) // 3 for i in range(1, n)]
        i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
        self.d_parents, self.drafts, self.len = _i32(self.parents), i32(n), _i32([prefix + n])
        self.mask, self.pos = torch.zeros(n, -(-n // 64), dtype=torch.int64, device="cuda"), i32(3, n)
        self.qkv, self.o = self.table.new_zeros(n, self.table.shape[1]), self.table.new_zeros(n, hq * hd)
        self.q = self.table.new_zeros(n, hq, hd)
        self.logits, self.u = torch.zeros(n, self.VOCAB, device="cuda"), torch.zeros(n, device="cuda")
        self.drawn, self.commit, self.tokens = i32(n), i32(n + 2), i32(n)
        size = max(C.load().efm_attention_tree_workspace_bytes(self.plain, n, self.MAX),
                   C.load().efm_sampler_filtered_workspace_bytes(n, self.VOCAB))
        self.ws = _buf(size) if ws is None else ws
        self.last = int(torch.randint(0, self.VOCAB, (1,), generator=g, device="cuda"))
        self.g = torch.Generator().manual_seed(seed)

    def write(self, text, cache):
        qkv = self.table[torch.tensor(text, device="cuda")]
        C.call("efm_qk_norm_rope_write_kv", self.ctx, ptr(qkv), 0, ptr(self.qw), ptr(self.kw), 1e-6, None, ptr(cache[0]), ptr(cache[1]),
               self.MAX, len(text), 0, None, None, 0, 0, 0, 0, stream())

    def feed(self):
        """The next tree's tokens and random numbers."""
        guess = [self.last] + [(int(torch.randint(0, self.VOCAB, (1,), generator=self.g)) // 3 * 3 + i) % self.VOCAB for i in range(1, self.n)]
        self.drafts.copy_(_i32(guess))
        self.u.copy_(torch.rand(self.n, generator=self.g))

    def launch(self):
        n, hq, hkv, hd = self.n, self.hq, self.hkv, self.hd
        torch.index_select(self.table, 0, self.drafts, out=self.qkv)
        C.call("efm_draft_tree_plan", n, ptr(self.d_parents), 0, ptr(self.len), 0, ptr(self.mask), ptr(self.pos), n, stream())
        C.call("efm_qk_norm_rope_write_kv", self.ctx, ptr(self.qkv), 0, ptr(self.qw), ptr(self.kw), 1e-6, ptr(self.q), ptr(self.cache[0]),
               ptr(self.cache[1]), self.MAX, n, 0, ptr(self.len), ptr(self.pos), n, hd // 8, hd // 8, hd // 4, stream())
        C.call("efm_attention_tree", self.plain, ptr(self.q), ptr(self.cache[0]), ptr(self.cache[1]), ptr(self.mask), ptr(self.o), n, 0,
               ptr(self.len), self.MAX, ptr(self.ws), self.ws.numel(), stream())
        C.call("efm_linear", n, hq * hd, self.VOCAB, ptr(self.o), ptr(self.head), None, ptr(self.logits), C.EFM_DTYPE_F32, stream())
        C.call("efm_sampler_filtered", n, self.VOCAB, ptr(self.logits), C.EFM_DTYPE_F32, 0, 0.8, 12, 0.95, 0.0, ptr(self.u), ptr(self.drawn),
               ptr(self.ws), self.ws.numel(), stream())
        C.call("efm_draft_tree_accept", n, ptr(self.d_parents), ptr(self.drafts), ptr(self.drawn), ptr(self.len), n, ptr(self.len),
               ptr(self.commit), ptr(self.tokens), stream())
        C.call("efm_draft_tree_move_kv", self.plain, 1, 0, ptr(self.cache[0]), ptr(self.cache[1]), self.MAX, n, ptr(self.commit), stream())

    def take(self):
        """Reads what the step emitted; returns it with the cache's rows of the text."""
        torch.cuda.synchronize()
        before, count = self.commit[:2].tolist()
        new = self.tokens[:count].tolist()
        assert before == len(self.text) and count >= 1
        self.text += [self.last] + new[:-1]
        self.last = new[-1]
        assert int(self.len) == len(self.text) + self.n
        return new, self.cache[:, :len(self.text)].clone()


@pytest.mark.parametrize("hq,hkv,hd", HEADS)
@pytest.mark.parametrize("n,prefix", [(1, 1), (13, 3), (40, 700), (70, 1100)])
def test_steps(gpu, hq, hkv, hd, n, prefix):
    """plan, rows, attention, logits, tokens, walk and move, step after step."""
    st, accepted = _Step(hq, hkv, hd, n, prefix), 0
    for _ in range(30):
        st.feed()
        st.launch()
        torch.cuda.synchronize()
        rows = len(st.text) + n
        # the nodes' rows are overwritten by the move: q and the text's rows give what the attention saw
        keys = torch.full_like(st.cache, math.nan)
        keys[:, :len(st.text)] = st.cache[:, :len(st.text)]
        C.call("efm_qk_norm_rope_write_kv", st.ctx, ptr(st.qkv), 0, ptr(st.qw), ptr(st.kw), 1e-6, None, ptr(keys[0]), ptr(keys[1]), st.MAX, n,
               len(st.text), None, ptr(st.pos), n, hd // 8, hd // 8, hd // 4, stream())
        ref, tol = R.attention(st.q.double(), keys[0, :rows].double(), keys[1, :rows].double(), R.bits(st.parents))
        _close(st.o.view(n, hq, hd), ref, tol)
        assert torch.equal(st.drawn, R.sample(st.logits, st.u, t=0.8, k=12, p=0.95))
        path = R.accept(st.parents, st.drafts.tolist(), st.drawn.tolist())
        drawn = st.drawn.tolist()
        new, cache = st.take()
        assert new == [drawn[i] for i in path]
        accepted += len(path)
        text = torch.full_like(st.cache, math.nan)
        st.write(st.text, text)
        assert torch.equal(cache, text[:, :len(st.text)])
    # Some guess was right: a root has three, of 16 ids, so that none is in 30 steps with a chance of (13 / 16)^30 = 0.2%
    # (of 5 steps 35%).
    assert n < 13 or accepted > 30


@pytest.mark.parametrize("hq,hkv,hd", HEADS)
def test_captured_steps_that_share_a_workspace(gpu, hq, hkv, hd):
    """Graphs of steps of two sizes over one workspace, replayed in turn, with eager work between."""
    sizes = [(40, 700), (9, 900)]
    ws = _buf(max(C.load().efm_attention_tree_workspace_bytes(C.make_attention_ctx(hq, hkv, hd, rope=False), n, _Step.MAX) for n, _ in sizes))
    eager = [_Step(hq, hkv, hd, n, prefix) for n, prefix in sizes]
    graphed = [_Step(hq, hkv, hd, n, prefix, ws=ws) for n, prefix in sizes]
    side, graphs = torch.cuda.Stream(), []
    torch.cuda.synchronize()
    for st in graphed:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
            st.launch()
        graphs.append(graph)
    for step in range(6):
        for a, b, graph in zip(eager, graphed, graphs):
            a.feed()
            a.launch()
            b.feed()
            graph.replay()
            (new, cache), (new_b, cache_b) = a.take(), b.take()
            assert new == new_b and torch.equal(cache, cache_b) and torch.equal(a.o, b.o) and torch.equal(a.drawn, b.drawn)


def test_two_streams_at_once(gpu):
    """Steps of two texts on streams of their own, their launches in turn."""
    args = [(14, 2, 64, 40, 700), (28, 4, 128, 24, 900)]
    alone, both = [_Step(*a) for a in args], [_Step(*a) for a in args]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for step in range(4):
        for st in alone:
            st.feed()
            st.launch()
        for st in both:
            st.feed()
        torch.cuda.synchronize()
        for st, s in zip(both, streams):
            with torch.cuda.stream(s):
                st.launch()
        for a, b in zip(alone, both):
            (new, cache), (new_b, cache_b) = a.take(), b.take()
            assert new == new_b and torch.equal(cache, cache_b) and torch.equal(a.o, b.o)


@pytest.mark.parametrize("rows,vocab,f", [(2, 3000, dict(p=0.9)), (3, 151936, dict(k=40, p=0.9)), (5, 151936, dict(p=0.9)), (5, 50000, dict(min_p=0.01))],
                         ids=str)
def test_captured_sampler_that_shares_a_workspace(gpu, rows, vocab, f):
    """A graph replayed over new logits, with eager calls of other sizes over the same workspace between."""
    ws = _buf(C.load().efm_sampler_filtered_workspace_bytes(9, 200000))
    x, u = _logits(1, rows, vocab)
    other, ou = _logits(2, 9, 200000)
    out = torch.zeros(rows, dtype=torch.int32, device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
        C.call("efm_sampler_filtered", rows, vocab, ptr(x), C.EFM_DTYPE_F32, 0, 1.0, f.get("k", 0), f.get("p", 1.0), f.get("min_p", 0.0), ptr(u),
               ptr(out), ptr(ws), ws.numel(), stream())
    for seed in range(5):
        y, v = _logits(10 + seed, rows, vocab)
        x.copy_(y), u.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, R.sample(x, u, **f))
        assert torch.equal(_sample(other, ou, ws=ws, p=0.8), R.sample(other, ou, p=0.8))
