"""CPU tests of the argument checks of a speculative decoding step's operators: they run on the host before any launch."""
import math

import pytest

import efm_capi as C

P, ODD = 4096, 4098   # addresses on and off a 4-byte boundary; never read
BAD, UNSUP, WS = C.EFM_ERR_INVALID_ARGUMENT, C.EFM_ERR_UNSUPPORTED, C.EFM_ERR_WORKSPACE


def _ctx(hq=12, hkv=2, hd=128, rope=False, **kw):
    return C.make_attention_ctx(hq, hkv, hd, rope=rope, **kw)


def _rc(name, *args):
    lib = C.load()
    rc = getattr(lib, name)(*args)
    if rc != C.EFM_OK:
        assert lib.efm_last_error().decode().startswith(name[4:])
    return rc


def _plan(n=8, parents=P, kv=100, d=None, off=0, mask=P, pos=P, stride=8):
    return _rc("efm_draft_tree_plan", n, parents, kv, d, off, mask, pos, stride, None)


@pytest.mark.parametrize("kw,want", [
    (dict(n=0), BAD), (dict(n=1025, stride=1025, kv=2000), UNSUP), (dict(parents=None), BAD), (dict(mask=None, pos=None), BAD),
    (dict(kv=7), BAD), (dict(stride=7), BAD), (dict(parents=ODD), BAD), (dict(mask=4100), BAD), (dict(pos=ODD), BAD),
    (dict(d=ODD), BAD), (dict(stride=-1), BAD),
])
def test_plan_refusals(kw, want):
    assert _plan(**kw) == want


def _tree(ctx=None, q=P, k=P, v=P, mask=P, o=P, n=8, kv=100, d=None, bound=0, ws=None, nbytes=0):
    return _rc("efm_attention_tree", ctx if ctx is not None else _ctx(), q, k, v, mask, o, n, kv, d, bound, ws, nbytes, None)


@pytest.mark.parametrize("kw,want", [
    (dict(ctx=_ctx(10, 2)), UNSUP), (dict(ctx=_ctx(hd=96)), UNSUP), (dict(ctx=_ctx(rope=True)), UNSUP), (dict(ctx=_ctx(7, 2)), BAD),
    (dict(q=None), BAD), (dict(k=None), BAD), (dict(v=None), BAD), (dict(mask=None), BAD), (dict(o=None), BAD),
    (dict(q=4104), BAD), (dict(k=4104), BAD), (dict(v=4104), BAD), (dict(o=4104), BAD), (dict(mask=4100), BAD),
    (dict(n=0), BAD), (dict(n=1025, kv=2000), UNSUP), (dict(kv=7), BAD), (dict(kv=0, d=P, bound=7), BAD),
    (dict(kv=0, d=P, bound=0), BAD), (dict(kv=0, d=ODD, bound=100), BAD), (dict(kv=(1 << 24) + 1), UNSUP),
    (dict(ctx=_ctx(k_stride_n=1 << 24)), UNSUP), (dict(ctx=_ctx(kv_stride_n=1 << 24)), UNSUP), (dict(ctx=_ctx(k_stride_n=260)), UNSUP),
    (dict(ctx=_ctx(1 << 15, 1 << 15)), UNSUP), (dict(kv=30000), WS), (dict(kv=30000, ws=P, nbytes=1024), WS),
    (dict(kv=30000, ws=4104, nbytes=1 << 40), BAD),
])
def test_attention_refusals(kw, want):
    assert _tree(**kw) == want


def test_attention_workspace():
    lib = C.load()
    size = lib.efm_attention_tree_workspace_bytes
    assert size(_ctx(), 8, 100) == 0
    assert size(_ctx(), 8, 30000) > 0
    assert size(_ctx(hd=96), 8, 30000) == 0 and size(_ctx(), 1025, 30000) == 0
    # what a call needs is never more than what a larger call asks for
    for n in (1, 3, 17, 100, 1024):
        assert size(_ctx(), n, 30000) <= size(_ctx(), 1024, 30000)


def _sample(rows=2, vocab=100, x=P, dt=C.EFM_DTYPE_F32, stride=0, t=1.0, k=0, p=1.0, mp=0.0, u=P, out=P, ws=None, nbytes=0):
    return _rc("efm_sampler_filtered", rows, vocab, x, dt, stride, t, k, p, mp, u, out, ws, nbytes, None)


@pytest.mark.parametrize("kw,want", [
    (dict(rows=-1), BAD), (dict(vocab=0), BAD), (dict(vocab=1 << 20), BAD), (dict(dt=C.EFM_DTYPE_F16), UNSUP), (dict(stride=99), BAD),
    (dict(t=0.0), BAD), (dict(t=1e-7), BAD), (dict(t=math.inf), BAD), (dict(t=math.nan), BAD), (dict(t=-1.0), BAD),
    (dict(p=0.0), BAD), (dict(p=math.nan), BAD), (dict(p=-0.5), BAD), (dict(mp=1.5), BAD), (dict(mp=math.nan), BAD),
    (dict(x=None), BAD), (dict(u=None), BAD), (dict(out=None), BAD), (dict(x=ODD), BAD), (dict(x=4097, dt=C.EFM_DTYPE_BF16), BAD),
    (dict(u=ODD), BAD), (dict(out=ODD), BAD), (dict(rows=0), C.EFM_OK), (dict(rows=65536), UNSUP),
    (dict(vocab=151936), WS), (dict(vocab=151936, ws=P, nbytes=1000), WS), (dict(vocab=151936, ws=4104, nbytes=1 << 40), BAD),
])
def test_sampler_refusals(kw, want):
    assert _sample(**kw) == want


def _accept(n=8, parents=P, draft=P, target=P, d=P, nxt=0, out=P, commit=P, tokens=P):
    return _rc("efm_draft_tree_accept", n, parents, draft, target, d, nxt, out, commit, tokens, None)


@pytest.mark.parametrize("kw,want", [
    (dict(n=0), BAD), (dict(n=1025), UNSUP), (dict(nxt=1025), UNSUP), (dict(parents=None), BAD), (dict(draft=None), BAD),
    (dict(target=None), BAD), (dict(d=None), BAD), (dict(out=None), BAD), (dict(commit=None), BAD), (dict(parents=ODD), BAD),
    (dict(tokens=ODD), BAD), (dict(d=ODD), BAD),
])
def test_accept_refusals(kw, want):
    assert _accept(**kw) == want


def _move(ctx=None, layers=2, stride=4096, k=P, v=P, rows=64, n=8, commit=P):
    return _rc("efm_draft_tree_move_kv", ctx if ctx is not None else _ctx(), layers, stride, k, v, rows, n, commit, None)


@pytest.mark.parametrize("kw,want", [
    (dict(ctx=_ctx(10, 2)), UNSUP), (dict(n=0), BAD), (dict(n=1025, rows=2000), UNSUP), (dict(k=None), BAD), (dict(v=None), BAD),
    (dict(commit=None), BAD), (dict(k=4104), BAD), (dict(v=4104), BAD), (dict(commit=ODD), BAD), (dict(stride=-8), BAD),
    (dict(stride=0), BAD), (dict(stride=4100), UNSUP), (dict(rows=7), BAD), (dict(layers=4097), UNSUP),
    (dict(ctx=_ctx(5000, 5000)), UNSUP), (dict(layers=0), C.EFM_OK),
])
def test_move_refusals(kw, want):
    assert _move(**kw) == want
