"""CPU tests of the FP4 operators' argument checks: they run on the host before any launch."""
import pytest

import efm_capi as C

P, ODD = 4096, 4104   # addresses on and off a 16-byte boundary; never read


def _ctx(hq=12, hkv=2, hd=128, **kw):
    return C.make_attention_ctx(hq, hkv, hd, **kw)


def _rc(name, *args):
    return getattr(C.load(), name)(*args)


BAD, UNSUP, WS = C.EFM_ERR_INVALID_ARGUMENT, C.EFM_ERR_UNSUPPORTED, C.EFM_ERR_WORKSPACE


@pytest.mark.parametrize("args,want", [
    ((0, 64, P, P, P, None), BAD), ((64, 0, P, P, P, None), BAD), ((-32, 64, P, P, P, None), BAD),
    ((48, 64, P, P, P, None), UNSUP), ((1 << 21, 64, P, P, P, None), UNSUP), ((64, 1 << 25, P, P, P, None), UNSUP),
    ((64, 64, None, P, P, None), BAD), ((64, 64, P, None, P, None), BAD), ((64, 64, P, P, None, None), BAD),
])
@pytest.mark.parametrize("name", ["efm_fp4_quantize", "efm_fp4_pack"])
def test_weight_layout_refusals(name, args, want):
    assert _rc(name, *args) == want
    assert C.load().efm_last_error().decode().startswith(name[4:])


def test_weight_layout_alignment():
    assert _rc("efm_fp4_quantize", 64, 64, ODD, P, P, None) == BAD
    assert _rc("efm_fp4_quantize", 64, 64, P, ODD, P, None) == BAD
    assert _rc("efm_fp4_pack", 64, 64, ODD, P, P, None) == BAD
    assert _rc("efm_fp4_pack", 64, 64, P, P, ODD, None) == BAD


def test_packed_bytes():
    lib = C.load()
    assert lib.efm_fp4_packed_bytes(128, 16) == 1024 + 64
    assert lib.efm_fp4_packed_bytes(160, 17) == 4 * (1024 + 64)
    assert lib.efm_fp4_packed_bytes(48, 16) == 0 and lib.efm_fp4_packed_bytes(0, 16) == 0


@pytest.mark.parametrize("args,want", [
    ((-1, 64, 64, P, P, None, P, 2, None, 0, None), BAD), ((1, 0, 64, P, P, None, P, 2, None, 0, None), BAD),
    ((1, 40, 64, P, P, None, P, 2, None, 0, None), UNSUP), ((1 << 21, 64, 64, P, P, None, P, 2, None, 0, None), UNSUP),
    ((1, 64, 64, None, P, None, P, 2, None, 0, None), BAD), ((1, 64, 64, P, None, None, P, 2, None, 0, None), BAD),
    ((1, 64, 64, P, P, None, None, 2, None, 0, None), BAD), ((1, 64, 64, ODD, P, None, P, 2, None, 0, None), BAD),
    ((1, 64, 64, P, ODD, None, P, 2, None, 0, None), BAD), ((1, 64, 64, P, P, None, P, 1, None, 0, None), UNSUP),
    ((0, 64, 64, P, P, None, P, 2, None, 0, None), C.EFM_OK),
])
def test_linear_refusals(args, want):
    assert _rc("efm_linear_fp4", *args) == want


@pytest.mark.parametrize("args,want", [
    ((-1, 64, 64, P, P, P, None, 0, None), BAD), ((1, 64, 0, P, P, P, None, 0, None), BAD),
    ((1, 64, 40, P, P, P, None, 0, None), UNSUP), ((1, 40, 64, P, P, P, None, 0, None), UNSUP),
    ((1, 64, 64, None, P, P, None, 0, None), BAD), ((1, 64, 64, P, ODD, P, None, 0, None), BAD),
    ((0, 64, 64, P, P, P, None, 0, None), C.EFM_OK),
])
def test_swiglu_refusals(args, want):
    assert _rc("efm_fused_gate_up_swiglu_fp4", *args) == want


def _write(fp4, ctx=None, qkv=P, stride=0, qw=P, kw=P, eps=1e-6, q_out=P, k=P, v=P, max_rows=64, seq=4, base=0, d_len=None,
           pos=None, pos_stride=0, sec=(0, 0, 0)):
    ctx = ctx if ctx is not None else _ctx()
    dst = (k,) if fp4 else (k, v)
    return _rc("efm_qk_norm_rope_write_kv" + ("_fp4" if fp4 else ""), ctx, qkv, stride, qw, kw, eps, q_out, *dst, max_rows,
               seq, base, d_len, pos, pos_stride, *sec, None)


@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("kw,want", [
    (dict(ctx=_ctx(10, 2)), UNSUP), (dict(ctx=_ctx(hd=96)), UNSUP), (dict(qkv=None), BAD), (dict(k=None), BAD),
    (dict(stride=2040), BAD), (dict(stride=2052), BAD), (dict(qkv=ODD), BAD), (dict(qw=ODD), BAD), (dict(kw=ODD), BAD),
    (dict(q_out=ODD), BAD), (dict(k=ODD), BAD), (dict(eps=-1.0), BAD), (dict(eps=float("nan")), BAD),
    (dict(max_rows=1 << 25), UNSUP), (dict(seq=65), BAD), (dict(base=61), BAD), (dict(base=0xffffffff), BAD),
    (dict(pos=P, pos_stride=3, sec=(16, 24, 24)), BAD), (dict(pos=P, pos_stride=4, sec=(16, 24, 20)), BAD),
    (dict(pos=P, pos_stride=4, sec=(-16, 40, 40)), BAD), (dict(ctx=_ctx(rope=False), pos=P, pos_stride=4, sec=(16, 24, 24)), BAD),
    (dict(seq=0), C.EFM_OK),
])
def test_write_refusals(fp4, kw, want):
    assert _write(fp4, **kw) == want


def test_write_bf16_needs_a_value_cache():
    assert _write(False, v=None) == BAD


def test_cache_bytes_and_read_refusals():
    lib, ctx = C.load(), _ctx()
    assert lib.efm_kv_fp4_bytes(ctx, 64) == 64 * 2 * 128 * 17 // 16
    assert lib.efm_kv_fp4_bytes(ctx, 65) == lib.efm_kv_fp4_bytes(ctx, 96)
    assert lib.efm_kv_fp4_bytes(_ctx(10, 2), 64) == 0
    read = lambda cache=P, room=64, first=0, rows=64, k=P, v=P, c=ctx: _rc("efm_kv_fp4_read", c, cache, room, first, rows, k, v, None)  # noqa: E731
    assert read(cache=None) == BAD and read(k=None, v=None) == BAD and read(k=ODD) == BAD and read(cache=ODD) == BAD
    assert read(first=1) == BAD and read(first=0xffffffff, rows=1) == BAD and read(rows=65) == BAD
    assert read(room=1 << 25) == UNSUP and read(c=_ctx(10, 2)) == UNSUP
    assert read(rows=0) == C.EFM_OK


def _decode(ctx=None, q=P, cache=P, room=4096, o=P, n=4096, d_len=None, bound=0, ws=P, nbytes=1 << 30):
    return _rc("efm_attention_decode_kv_fp4", ctx or _ctx(rope=False), q, cache, room, o, n, d_len, bound, ws, nbytes, None)


@pytest.mark.parametrize("kw,want", [
    (dict(ctx=_ctx()), UNSUP), (dict(ctx=_ctx(10, 2, rope=False)), UNSUP), (dict(ctx=_ctx(hd=256, rope=False)), UNSUP),
    (dict(q=None), BAD), (dict(cache=None), BAD), (dict(o=None), BAD), (dict(q=ODD), BAD), (dict(cache=ODD), BAD),
    (dict(o=ODD), BAD), (dict(n=4097), BAD), (dict(d_len=P, bound=0), BAD), (dict(d_len=P, bound=4097), BAD),
    (dict(room=1 << 25), UNSUP), (dict(ws=None), WS), (dict(nbytes=64), WS), (dict(ws=ODD), BAD),
])
def test_decode_refusals(kw, want):
    assert _decode(**kw) == want


def _rows(ctx=None, q=P, cache=P, room=4096, o=P, n=4, kv=4096, ws=P, nbytes=1 << 30):
    return _rc("efm_attention_prefill_kv_fp4", ctx or _ctx(rope=False), q, cache, room, o, n, kv, 1, ws, nbytes, None)


@pytest.mark.parametrize("kw,want", [
    (dict(ctx=_ctx()), UNSUP), (dict(q=None), BAD), (dict(cache=None), BAD), (dict(o=None), BAD), (dict(n=5, kv=4), BAD),
    (dict(kv=4097), BAD), (dict(ws=None), WS), (dict(nbytes=64), WS), (dict(ws=ODD), BAD),
    (dict(n=(1 << 20) + 1, kv=1 << 21, room=1 << 21), UNSUP), (dict(n=0), C.EFM_OK),
])
def test_rows_refusals(kw, want):
    assert _rows(**kw) == want
    assert C.load().efm_attention_prefill_kv_fp4_workspace_bytes(_ctx(10, 2, rope=False), 4, 64) == 0
    assert C.load().efm_attention_decode_kv_fp4_workspace_bytes(_ctx(rope=False), 4096) > 64


def test_workspaces_serve_every_smaller_call():
    """The bytes never fall as rows or keys grow; none for a few tiles of keys."""
    lib = C.load()
    for ctx in (_ctx(rope=False), _ctx(28, 4, rope=False), _ctx(14, 2, hd=64, rope=False)):
        lens = [1, 200, 257, 900, 4000, 8192, 8193, 8300, 40000, 1 << 24, (1 << 32) - 1]
        one = [lib.efm_attention_decode_kv_fp4_workspace_bytes(ctx, n) for n in lens]
        assert one == sorted(one) and one[0] == 0
        for rows in (1, 2, 40, 600, 5000):
            many = [lib.efm_attention_prefill_kv_fp4_workspace_bytes(ctx, rows, n) for n in lens]
            more = [lib.efm_attention_prefill_kv_fp4_workspace_bytes(ctx, rows + 1, n) for n in lens]
            assert many == sorted(many) and all(a <= b for a, b in zip(many, more))


def test_more_heads_than_an_index_holds():
    big = _ctx(1 << 17, 1 << 17, rope=False)
    assert _decode(ctx=big) == UNSUP and _rows(ctx=big) == UNSUP
    assert _rows(ctx=_ctx(1 << 15, 1 << 15, rope=False), n=1 << 16, kv=1 << 16, room=1 << 16) == UNSUP
    assert C.load().efm_kv_fp4_bytes(big, 64) == 0 and C.load().efm_kv_fp4_bytes(_ctx(), 1 << 25) == 0


def test_every_operator_of_the_cache_takes_the_same_heads():
    most, more = _ctx(1 << 16, 1 << 16, hd=64, rope=False), _ctx(1 << 17, 1 << 17, hd=64, rope=False)
    read = lambda c: _rc("efm_kv_fp4_read", c, P, 64, 0, 0, P, P, None)  # noqa: E731
    write = lambda c: _write(True, ctx=c, seq=0)  # noqa: E731
    rows = lambda c: _rows(ctx=c, n=0)  # noqa: E731
    for call in (read, write, rows):
        assert call(most) == C.EFM_OK
    assert read(more) == UNSUP and write(more) == UNSUP
    assert C.load().efm_kv_fp4_bytes(most, 64) > 0 and C.load().efm_kv_fp4_bytes(more, 64) == 0


def test_more_threads_than_a_grid_holds():
    assert _rows(ctx=_ctx(512, 64, hd=64, rope=False), n=1 << 20, kv=1 << 20, room=1 << 20) == UNSUP
    assert "rows of 512 query heads" in C.load().efm_last_error().decode()
    assert _rc("efm_linear_fp4", 1 << 20, 32, 1 << 24, P, P, None, P, 2, None, 0, None) == UNSUP
    assert "too many tiles" in C.load().efm_last_error().decode()
