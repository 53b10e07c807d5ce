"""GPU tests of the FP4 weights and cache and of the per-head norms, against plain 64-bit forms (_fp4_ref).

Tolerances are derived: half a step of the output's type (bf16 2^-8, relative), what the documented roundings inside an
operator can move, and the rounding of fp32 sums. Quantised values have to be equal."""
import math

import pytest
import torch

import _fp4_ref as R
import efm_capi as C
from _fp4_sizes import LINEAR_LONG, SWIGLU_LONG
from _util import ptr, stream

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -8   # bf16
HEADS = [pytest.param(14, 2, 64, id="0p5b"), pytest.param(12, 2, 128, id="1p5b"), pytest.param(28, 4, 128, id="7b")]


def _buf(nbytes, fill=0):
    return torch.full((max(int(nbytes), 256),), fill, dtype=torch.uint8, device="cuda")


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _bf(g, *size, std=1.0):
    return (torch.randn(*size, generator=g) * std).to(torch.bfloat16)


def _within(got, ref, tol, what=""):
    got, err = got.double().cpu(), None
    assert got.shape == ref.shape
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{what}: NaN in other places"
    err = (got - ref).abs()
    bad = ~(err <= tol) & ~torch.isnan(ref)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err - tol)[bad].max())} past its tolerance"


# ---------------------------------------------------------------- weights

def _quantize(w):
    out, k = w.shape
    codes = torch.zeros(out, k // 2, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(out, k // 32, dtype=torch.uint8, device="cuda")
    wd = w.cuda()
    C.call("efm_fp4_quantize", k, out, ptr(wd), ptr(codes), ptr(scales), stream())
    torch.cuda.synchronize()
    return codes, scales


def _pack(codes, scales):
    out, k = codes.shape[0], codes.shape[1] * 2
    packed = _buf(C.load().efm_fp4_packed_bytes(k, out), 0xff)
    cd, sd = codes.cuda().contiguous(), scales.cuda().contiguous()
    C.call("efm_fp4_pack", k, out, ptr(cd), ptr(sd), ptr(packed), stream())
    torch.cuda.synchronize()
    return packed


def test_quantize_equals_the_definition(gpu):
    """Random rows of several magnitudes, borders of the grid under every scale's mantissa, zeros, the smallest and the
    largest bf16 values, and groups with NaN and infinities."""
    g = _gen(1)
    w = _bf(g, 24, 96) * torch.exp2(torch.randint(-130, 125, (24, 3), generator=g).float()).repeat_interleave(32, 1).bfloat16()
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, 6, 7] * 2)
    w[0, :32], w[1, :32], w[2, :32] = ties, ties * 2.0 ** -120, ties * 2.0 ** 100
    w[3, :32] = 0
    w[4, :32] = 2.0 ** -133
    w[5, :32] = torch.finfo(torch.bfloat16).max
    w[6, 0], w[6, 32], w[6, 64] = math.nan, math.inf, -math.inf
    w[7, :32] = torch.linspace(-7.03125, 7.03125, 32).bfloat16()   # 7.03125 is past 7: the next scale
    codes, scales = _quantize(w)
    code, byte = R.quantize(w)
    assert torch.equal(scales.cpu(), byte)
    assert torch.equal(codes.cpu(), R.halves(code))


def test_quantize_many_groups(gpu):
    """More values than a pass of the grid takes: the parts by themselves give the same."""
    g = torch.Generator(device="cuda").manual_seed(2)
    w = torch.randn(8200, 4128, generator=g, device="cuda").bfloat16()
    codes, scales = _quantize(w)
    for lo, hi in ((0, 2000), (2000, 6000), (6000, 8200)):
        c, s = _quantize(w[lo:hi].contiguous())
        assert torch.equal(codes[lo:hi], c) and torch.equal(scales[lo:hi], s)
    at = torch.tensor([0, 4063, 4064, 8199])   # the grid's first pass ends in row 4064
    code, byte = R.quantize(w[at.cuda()])
    assert torch.equal(scales.cpu()[at], byte) and torch.equal(codes.cpu()[at], R.halves(code))


@pytest.mark.parametrize("k,out", [(1 << 20, (1 << 17) + 24)])
def test_pack_past_32_bits_of_threads(gpu, k, out):
    """The first, a middle and the last tile of 73 GB of weights, equal to the packing of their rows alone."""
    lib = C.load()
    if torch.cuda.mem_get_info()[0] < 200 << 30:
        pytest.skip("needs 160 GB")
    torch.cuda.empty_cache()
    codes, scales = (torch.empty(out, k // n, dtype=torch.uint8, device="cuda") for n in (2, 32))
    packed = torch.empty(lib.efm_fp4_packed_bytes(k, out), dtype=torch.uint8, device="cuda")
    tiles, of_tile = -(-out // 16), k * 8
    rows = {t: slice(16 * t, min(16 * t + 16, out)) for t in (0, tiles // 2, tiles - 1)}
    for t, at in rows.items():
        half, byte = _weights_on_device(t, at.stop - at.start, k)
        codes[at], scales[at] = half, byte
        packed[t * of_tile:(t + 1) * of_tile] = 0xff
    C.call("efm_fp4_pack", k, out, ptr(codes), ptr(scales), ptr(packed), stream())
    torch.cuda.synchronize()
    for t, at in rows.items():
        alone, s0 = _pack(codes[at], scales[at]), tiles * of_tile + t * of_tile // 16
        assert torch.equal(packed[t * of_tile:(t + 1) * of_tile], alone[:of_tile]), t
        assert torch.equal(packed[s0:s0 + of_tile // 16], alone[of_tile:]), t
    del codes, scales, packed
    torch.cuda.empty_cache()


def _linear(x, packed, k, out, bias=None, f32=False, fill_ws=0xff):
    m = x.shape[0]
    y = torch.full((m, out), math.nan, dtype=torch.float32 if f32 else torch.bfloat16, device="cuda")
    ws = _buf(C.load().efm_linear_fp4_workspace_bytes(m, k, out), fill_ws)
    C.call("efm_linear_fp4", m, k, out, ptr(x), ptr(packed), ptr(bias), ptr(y), C.EFM_DTYPE_F32 if f32 else C.EFM_DTYPE_BF16,
           ptr(ws), ws.numel(), stream())
    torch.cuda.synchronize()
    return y


def _weights(g, out, k):
    """Codes and scales of any bit pattern with scales around 2^-7, as a checkpoint of the format may hold."""
    code = torch.randint(0, 16, (out, k), generator=g).to(torch.uint8)
    byte = torch.randint(117, 123, (out, k // 32), generator=g).to(torch.uint8)
    return code, byte


def _product(x, w):
    """(x w^T, bound of its fp32 error): chains of K / 32 products of 32 terms, 2^-23 an addition, of the sum of
    magnitudes; sums of waves and slices of K are 64 additions more at most."""
    k = x.shape[1]
    return x @ w.T, (k / 32 + 32 + 64) * 2.0 ** -23 * (x.abs() @ w.abs().T)


def _swiglu(x, w):
    """(bf16(silu(bf16(gate)) * bf16(up)) in 64 bits, its bound): both products' errors through the activation."""
    (up, gate), (eu, eg) = (t.chunk(2, 1) for t in _product(x.double(), w))
    silu = gate * torch.sigmoid(gate)
    du, dg = eu + HALF * (up.abs() + eu), eg + HALF * (gate.abs() + eg)
    tol = 1.1 * dg * (up.abs() + du) + silu.abs() * du   # |silu'| < 1.1
    return silu * up, tol + (HALF + 2.0 ** -20) * ((silu * up).abs() + tol)


SHAPES = [(1, 32, 1), (1, 896, 1152), (1, 160, 17), (1, 18944, 100), (2, 96, 33), (5, 4864, 896), (16, 1536, 300), (17, 544, 48),
          (31, 992, 130), (33, 288, 64), (64, 2048, 272), (100, 160, 4608), (129, 896, 257), (300, 1536, 640), (1000, 512, 384)]


@pytest.mark.parametrize("m,k,out", SHAPES)
@pytest.mark.parametrize("bias,f32", [(False, False), (True, True)])
def test_linear(gpu, m, k, out, bias, f32):
    g = _gen(m * 7 + k + out)
    code, byte = _weights(g, out, k)
    x, b = _bf(g, m, k), _bf(g, out)
    y = _linear(x.cuda(), _pack(R.halves(code), byte), k, out, b.cuda() if bias else None, f32)
    ref, tol = _product(x.double(), R.values(code, byte))
    if bias:
        ref = ref + b.double()
        tol = tol + 2.0 ** -23 * ref.abs()
    _within(y, ref, tol if f32 else tol + HALF * (ref.abs() + tol), f"{m} x {k} -> {out}")


@pytest.mark.parametrize("m,hidden,inter", [(1, 896, 4864), (1, 32, 16), (3, 1536, 64), (16, 160, 112), (24, 1536, 8960),
                                            (40, 544, 48), (70, 896, 80), (200, 256, 272), (600, 512, 320)])
def test_swiglu(gpu, m, hidden, inter):
    g = _gen(m + hidden + inter)
    code, byte = _weights(g, 2 * inter, hidden)
    x = _bf(g, m, hidden)
    packed, y = _pack(R.halves(code), byte), torch.full((m, inter), math.nan, dtype=torch.bfloat16, device="cuda")
    ws = _buf(C.load().efm_fused_gate_up_swiglu_fp4_workspace_bytes(m, hidden, inter), 0xff)
    xd = x.cuda()
    C.call("efm_fused_gate_up_swiglu_fp4", m, hidden, inter, ptr(xd), ptr(packed), ptr(y), ptr(ws), ws.numel(), stream())
    torch.cuda.synchronize()
    (up, gate), (eu, eg) = (t.chunk(2, 1) for t in _product(x.double(), R.values(code, byte)))
    silu = gate * torch.sigmoid(gate)
    du, dg = eu + HALF * (up.abs() + eu), eg + HALF * (gate.abs() + eg)
    tol = 1.1 * dg * (up.abs() + du) + silu.abs() * du   # |silu'| < 1.1
    _within(y, silu * up, tol + (HALF + 2.0 ** -20) * ((silu * up).abs() + tol), f"{m} {hidden} {inter}")


# sizes that between them take every shape of workgroup, with widths and lengths that end inside its tiles
WIDE = [(7, 32, 50), (5, 32, 4177), (5, 1664, 4303), (17, 32, 4481), (19, 1568, 8650), (19, 5184, 4250), (17, 928, 34530),
        (35, 672, 15219), (5, 32, 16530), (97, 160, 41515), (33, 1824, 64960), (71, 1088, 57690), (6, 544, 50), (5, 288, 17), (3001, 672, 270),
        (65, 32, 53179), (723, 32, 57850), (5, 864, 4460), (17, 800, 4351), (17, 1440, 8410),
        (17, 704, 20401), (3, 8224, 70), (4, 6176, 65530),
        (4, 1056, 65601), (2, 32, 65537)]


def _columns(g, n):
    return torch.cat([torch.arange(min(n, 150)), torch.randint(0, n, (200,), generator=g), torch.arange(max(0, n - 150), n)])


def _weights_on_device(seed, out, k):
    g = torch.Generator(device="cuda").manual_seed(seed)
    half = torch.randint(0, 256, (out, k // 2), generator=g, dtype=torch.uint8, device="cuda")
    return half, torch.randint(117, 123, (out, k // 32), generator=g, dtype=torch.uint8, device="cuda")


def _values_of(half, byte, rows):
    half, byte = half[rows.cuda()].cpu(), byte[rows.cuda()].cpu()
    return R.values(torch.stack([half & 15, half >> 4], 2).flatten(1), byte)


@pytest.mark.parametrize("m,k,out", WIDE)
@pytest.mark.parametrize("f32", [False, True])
def test_linear_every_shape(gpu, m, k, out, f32):
    """Against 64 bits in the first and last columns and 200 others, equal to a second call in all."""
    g = _gen(m + k + out)
    half, byte = _weights_on_device(m + k, out, k)
    packed, x = _pack(half, byte), _bf(g, m, k)
    y = _linear(x.cuda(), packed, k, out, None, f32)
    at = _columns(g, out)
    ref, tol = _product(x.double(), _values_of(half, byte, at))
    _within(y[:, at.cuda()], ref, tol if f32 else tol + HALF * (ref.abs() + tol), f"{m} x {k} -> {out}")
    assert not y.isnan().any() and torch.equal(y, _linear(x.cuda(), packed, k, out, None, f32))


@pytest.mark.parametrize("m,hidden,inter", [(5, 32, 16), (5, 544, 16), (17, 32, 2144), (18, 1504, 4160), (18, 5024, 2160),
                                            (42, 992, 8272), (35, 672, 7936), (5, 32, 8288), (33, 32, 43248), (33, 1088, 56288),
                                            (72, 1120, 28112), (5, 1568, 16), (1667, 672, 288), (66, 32, 25200), (871, 32, 22256),
                                            (5, 800, 16), (21, 800, 2144), (17, 832, 7216), (17, 672, 9392),
                                            (4, 4192, 80), (4, 8224, 48), (2, 2080, 33040)])
def test_swiglu_every_shape(gpu, m, hidden, inter):
    g = _gen(m + hidden + inter)
    half, byte = _weights_on_device(m + hidden, 2 * inter, hidden)
    packed, x = _pack(half, byte), _bf(g, m, hidden)
    xd, ys = x.cuda(), []
    for _ in range(2):
        ys.append(torch.full((m, inter), math.nan, dtype=torch.bfloat16, device="cuda"))
        C.call("efm_fused_gate_up_swiglu_fp4", m, hidden, inter, ptr(xd), ptr(packed), ptr(ys[-1]), None, 0, stream())
    torch.cuda.synchronize()
    at = _columns(g, inter)
    up, eu = _product(x.double(), _values_of(half, byte, at))
    gate, eg = _product(x.double(), _values_of(half, byte, at + inter))
    silu = gate * torch.sigmoid(gate)
    du, dg = eu + HALF * (up.abs() + eu), eg + HALF * (gate.abs() + eg)
    tol = 1.1 * dg * (up.abs() + du) + silu.abs() * du   # |silu'| < 1.1
    _within(ys[0][:, at.cuda()], silu * up, tol + (HALF + 2.0 ** -20) * ((silu * up).abs() + tol), f"{m} {hidden} {inter}")
    assert not ys[0].isnan().any() and torch.equal(*ys)


@pytest.mark.parametrize("m,k,out", LINEAR_LONG)
def test_linear_every_shape_over_long_k(gpu, m, k, out):
    g = _gen(m + k + out)
    half, byte = _weights_on_device(m + k, out, k)
    packed, x = _pack(half, byte), _bf(g, m, k)
    y, at = _linear(x.cuda(), packed, k, out, None, True), _columns(g, out).unique()
    _within(y[:, at.cuda()], *_product(x.double(), _values_of(half, byte, at)), f"{m} x {k} -> {out}")
    assert not y.isnan().any() and torch.equal(y, _linear(x.cuda(), packed, k, out, None, True))


@pytest.mark.parametrize("m,hidden,inter", SWIGLU_LONG)
def test_swiglu_every_shape_over_long_k(gpu, m, hidden, inter):
    g = _gen(m + hidden + inter)
    half, byte = _weights_on_device(m + hidden, 2 * inter, hidden)
    packed, x = _pack(half, byte), _bf(g, m, hidden)
    xd, at, ys = x.cuda(), _columns(g, inter).unique(), []
    for _ in range(2):
        ys.append(torch.full((m, inter), math.nan, dtype=torch.bfloat16, device="cuda"))
        C.call("efm_fused_gate_up_swiglu_fp4", m, hidden, inter, ptr(xd), ptr(packed), ptr(ys[-1]), None, 0, stream())
    torch.cuda.synchronize()
    _within(ys[0][:, at.cuda()], *_swiglu(x, _values_of(half, byte, torch.cat([at, at + inter]))), f"{m} {hidden} {inter}")
    assert not ys[0].isnan().any() and torch.equal(*ys)


def _ahead_of_nan(x):
    """x in a larger buffer that holds NaN behind it."""
    wide = torch.full((x.numel() + 512,), math.nan, dtype=torch.bfloat16, device="cuda")
    wide[:x.numel()] = x.flatten().cuda()
    return wide[:x.numel()].view(x.shape)


@pytest.mark.parametrize("m,k,out", [(1, 24608, 17), (1, 24672, 40), (1, 24736, 130), (2, 24608, 33), (5, 160, 50), (17, 544, 48),
                                     (100, 672, 300), (500, 416, 1024)])
def test_linear_whose_last_columns_end_inside_a_load(gpu, m, k, out):
    """Lengths of K that end inside the last block or slab, one row of x past LDS among them: what lies behind x stays out."""
    g = _gen(m + k + out)
    code, byte = _weights(g, out, k)
    x = _bf(g, m, k)
    y = _linear(_ahead_of_nan(x), _pack(R.halves(code), byte), k, out, None, True)
    _within(y, *_product(x.double(), R.values(code, byte)), f"{m} x {k} -> {out}")


@pytest.mark.parametrize("m,hidden,inter", [(1, 16416, 16), (1, 16480, 48), (1, 16928, 48), (3, 5472, 32), (40, 160, 80)])
def test_swiglu_whose_last_columns_end_inside_a_load(gpu, m, hidden, inter):
    g = _gen(m + hidden + inter)
    code, byte = _weights(g, 2 * inter, hidden)
    x, packed = _bf(g, m, hidden), _pack(R.halves(code), byte)
    y, xd = torch.full((m, inter), math.nan, dtype=torch.bfloat16, device="cuda"), _ahead_of_nan(x)
    C.call("efm_fused_gate_up_swiglu_fp4", m, hidden, inter, ptr(xd), ptr(packed), ptr(y), None, 0, stream())
    torch.cuda.synchronize()
    _within(y, *_swiglu(x, R.values(code, byte)), f"{m} {hidden} {inter}")


@pytest.mark.parametrize("m,k", [(m, k) for m, last in ((1, 24544), (2, 12256), (3, 8160), (4, 6112)) for k in (last, last + 32)])
def test_linear_where_x_leaves_lds(gpu, m, k):
    """The longest rows of x that LDS holds, and the next."""
    g = _gen(m + k)
    code, byte = _weights(g, 50, k)
    x = _bf(g, m, k)
    _within(_linear(x.cuda(), _pack(R.halves(code), byte), k, 50, None, True), *_product(x.double(), R.values(code, byte)))


@pytest.mark.parametrize("m,hidden", [(m, k) for m, last in ((1, 16352), (4, 4064)) for k in (last, last + 32)])
def test_swiglu_where_x_leaves_lds(gpu, m, hidden):
    g = _gen(m + hidden)
    code, byte = _weights(g, 96, hidden)
    x, packed = _bf(g, m, hidden), _pack(R.halves(code), byte)
    y, xd = torch.full((m, 48), math.nan, dtype=torch.bfloat16, device="cuda"), x.cuda()
    C.call("efm_fused_gate_up_swiglu_fp4", m, hidden, 48, ptr(xd), ptr(packed), ptr(y), None, 0, stream())
    torch.cuda.synchronize()
    _within(y, *_swiglu(x, R.values(code, byte)))


@pytest.mark.parametrize("m", [1, 20, 200])
@pytest.mark.parametrize("low,high,power", [(0, 4, 120), (250, 255, -120)])
def test_linear_smallest_and_largest_scales(gpu, m, low, high, power):
    """Scales at both ends of the format, where values are subnormal in bf16, or close to its largest and, from 2^128 on,
    infinite, with rows of x that bring the products back."""
    g = _gen(m)
    k, out = 256, 40
    code = torch.randint(0, 16, (out, k), generator=g).to(torch.uint8)
    code = torch.where((code & 7) > 5, code & 13, code) if low else code
    byte = torch.randint(low, high, (out, k // 32), generator=g).to(torch.uint8)
    x = _bf(g, m, k) * 2.0 ** power
    y = _linear(x.cuda(), _pack(R.halves(code), byte), k, out, None, True).cpu()
    w = R.values(code, byte)
    w[w.abs() >= 2.0 ** 128] *= math.inf
    ref, tol = _product(x.double(), w)
    assert torch.equal(y.isnan(), ref.isnan()) and torch.equal(y[ref.isinf()].double(), ref[ref.isinf()])
    assert (ref[ref.isfinite()].abs() > 2.0 ** -30).any()
    _within(y[ref.isfinite()], ref[ref.isfinite()], tol[ref.isfinite()])


@pytest.mark.parametrize("m", [1, 20, 200])
def test_linear_nan_stays_in_its_place(gpu, m):
    """A NaN group reaches its own output column alone, a NaN row of x its own row; rows and columns that pad the tiles
    reach nothing."""
    g = _gen(3)
    k, out = 160, 19
    code, byte = _weights(g, out, k)
    byte[7, 4] = 255
    x = _bf(g, m, k)
    y = _linear(x.cuda(), _pack(R.halves(code), byte), k, out).cpu()
    bad = torch.isnan(y)
    assert bad[:, 7].all() and int(bad.sum()) == m
    if m > 1:
        x[m - 1, 3] = math.inf
        x[m - 1, 4] = math.nan
        bad = torch.isnan(_linear(x.cuda(), _pack(R.halves(code), byte), k, out).cpu())
        assert bad[m - 1].all() and bad[:, 7].all() and int(bad.sum()) == m + out - 1


@pytest.mark.parametrize("m,k,out", [(1, 4864, 896), (24, 8960, 512), (200, 1024, 640)])
def test_linear_repeats_and_runs_in_a_graph(gpu, m, k, out):
    """Captured on a side stream and replayed with other inputs, eager work between: bit for bit the eager result."""
    g = _gen(m + 5)
    code, byte = _weights(g, out, k)
    packed, x = _pack(R.halves(code), byte), _bf(g, m, k).cuda()
    y = torch.empty(m, out, dtype=torch.bfloat16, device="cuda")
    ws = _buf(C.load().efm_linear_fp4_workspace_bytes(m, k, out))
    s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s, capture_error_mode="thread_local"):
        C.call("efm_linear_fp4", m, k, out, ptr(x), ptr(packed), None, ptr(y), C.EFM_DTYPE_BF16, ptr(ws), ws.numel(), s.cuda_stream)
    for rep in range(3):
        x.copy_(_bf(g, m, k))
        y.fill_(math.nan)
        torch.randn(1 << 18, device="cuda").sum()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, _linear(x, packed, k, out)), f"replay {rep}"


# ---------------------------------------------------------------- norm, rotation, write

def _positions(base, S, half, off=0):
    return (base + off + torch.arange(S, dtype=torch.int64))[:, None].expand(S, half)


def _write(ctx, fp4, qkv, qw, kw, q_out, dst, room, S, base, d_len=None, pos=None, sec=(0, 0, 0), eps=1e-6, stride=0, on=None):
    C.call("efm_qk_norm_rope_write_kv" + ("_fp4" if fp4 else ""), ctx, ptr(qkv), stride, ptr(qw), ptr(kw), eps, ptr(q_out),
           *[ptr(d) for d in dst], room, S, base, ptr(d_len), ptr(pos), 0 if pos is None else pos.shape[1], *sec,
           on if on is not None else stream())


def _read(ctx, cache, room, first, rows, hkv, hd):
    k, v = (torch.empty(rows, hkv, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    C.call("efm_kv_fp4_read", ctx, ptr(cache), room, first, rows, ptr(k), ptr(v), stream())
    torch.cuda.synchronize()
    return k.cpu().double(), v.cpu().double()


def _y_tol(y, x, w, eps):
    """fp32 work on a pair: sums of hd squares, sqrt, division, sine and cosine, products: 2^-18 of the pair's larger
    magnitude covers some 30 roundings; then half a step of bf16."""
    n = R.norm_rope(x, w, eps, None, 1.0).abs()
    pair = n + n.roll(x.shape[-1] // 2, -1)
    return HALF * y.abs() + 2.0 ** -18 * pair


@pytest.mark.parametrize("hq,hkv,hd", HEADS)
@pytest.mark.parametrize("S,base", [(1, 0), (1, 63), (5, 3), (33, 31), (130, 1000000), (2051, 13)])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("fp4", [False, True])
def test_write(gpu, hq, hkv, hd, S, base, norm, fp4):
    """Queries, keys and values of a prompt or a step; rows of the cache around the written ones stay as they were."""
    g = _gen(S + base + hd)
    width = (hq + 2 * hkv) * hd
    qkv = _bf(g, S, width + 8, std=1.5)
    qkv[:, :hd] *= 100.0
    qw, kw = (1 + _bf(g, hd, std=0.2), 1 + _bf(g, hd, std=0.2)) if norm else (None, None)
    room = base + S + 40
    ctx = C.make_attention_ctx(hq, hkv, hd, rope_theta=1e6)
    x = qkv[:, :width].double().view(S, -1, hd)
    q_out = torch.full((S, hq, hd), math.nan, dtype=torch.bfloat16, device="cuda")
    dev = [None if t is None else t.cuda() for t in (qkv, qw, kw)]
    pos = _positions(base, S, hd // 2)
    q = R.norm_rope(x[:, :hq], qw, 1e-6, pos, 1e6)
    k = R.norm_rope(x[:, hq:hq + hkv], kw, 1e-6, pos, 1e6)
    if fp4:
        cache = _buf(C.load().efm_kv_fp4_bytes(ctx, room), 0x5a)
        _write(ctx, True, *dev, q_out, [cache], room, S, base, stride=width + 8)
        kk, vv = _read(ctx, cache, room, base, S, hkv, hd)
        assert torch.equal(kk, R.rounded(k)) and torch.equal(vv, R.rounded(x[:, hq + hkv:]))
        fresh = _buf(C.load().efm_kv_fp4_bytes(ctx, room), 0x5a)
        lo, n = max(0, base - 40), min(base, 40)
        for first, rows in ((lo, n), (base + S, room - base - S)):
            if rows:
                for a, b in zip(_read(ctx, cache, room, first, rows, hkv, hd), _read(ctx, fresh, room, first, rows, hkv, hd)):
                    assert torch.equal(a, b), "a row beside the written ones changed"
    else:
        kc, vc = (torch.full((room, hkv, hd), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        _write(ctx, False, *dev, q_out, [kc, vc], room, S, base, stride=width + 8)
        torch.cuda.synchronize()
        _within(kc[base:base + S], k, _y_tol(k, x[:, hq:hq + hkv], kw, 1e-6), "keys")
        assert torch.equal(vc[base:base + S].cpu(), qkv[:, (hq + hkv) * hd:width].reshape(S, hkv, hd))
        for c in (kc, vc):
            assert (c[:base] == 7).all() and (c[base + S:] == 7).all()
    torch.cuda.synchronize()
    _within(q_out, q, _y_tol(q, x[:, :hq], qw, 1e-6), "queries")


@pytest.mark.parametrize("S", [37, 2051])
@pytest.mark.parametrize("fp4", [False, True])
def test_write_mrope_offsets_strides_and_in_place(gpu, fp4, S):
    """M-RoPE ids with sections; without ids, offsets of queries and keys that differ; a strided bf16 cache; the queries
    written over their own columns."""
    g = _gen(9)
    hq, hkv, hd, base, room = 16, 2, 128, 11, S + 27
    width = (hq + 2 * hkv) * hd
    qkv, qw, kw = _bf(g, S, width), 1 + _bf(g, hd, std=0.2), 1 + _bf(g, hd, std=0.2)
    x = qkv.double().view(S, -1, hd)
    ids = torch.randint(0, 5000, (3, S + 3), generator=g, dtype=torch.int32)
    sec = (16, 24, 24)
    by_id = torch.cat([ids[i, :S, None].expand(S, n) for i, n in enumerate(sec)], 1)
    for pos, qp, kp, off in ((ids, by_id, by_id, (0, 0)), (None, _positions(base, S, 64, 5), _positions(base, S, 64, 70000), (5, 70000))):
        ctx = C.make_attention_ctx(hq, hkv, hd, rope_theta=1e4, rope_scale=2.0, q_rope_pos_offset=off[0], k_rope_pos_offset=off[1],
                                   q_stride_n=width, k_stride_n=2 * hkv * hd, kv_stride_n=2 * hkv * hd, k_stride_h=2 * hd,
                                   kv_stride_h=2 * hd)
        q, k = R.norm_rope(x[:, :hq], qw, 1e-5, qp, 1e4, 2.0), R.norm_rope(x[:, hq:hq + hkv], kw, 1e-5, kp, 1e4, 2.0)
        d = qkv.cuda()
        pd = None if pos is None else pos.cuda()
        s = sec if pos is not None else (0, 0, 0)
        kv = torch.full((room, hkv, 2, hd), 7.0, dtype=torch.bfloat16, device="cuda")
        cache = _buf(C.load().efm_kv_fp4_bytes(ctx, room))
        dst = [cache] if fp4 else [kv[:, :, 0], kv[:, :, 1]]
        _write(ctx, fp4, d, qw.cuda(), kw.cuda(), d, dst, room, S, base, pos=pd, sec=s, eps=1e-5)
        torch.cuda.synchronize()
        got = d.cpu().view(S, -1, hd)
        _within(got[:, :hq], q, _y_tol(q, x[:, :hq], qw, 1e-5), "queries")
        assert torch.equal(got[:, hq:], qkv.view(S, -1, hd)[:, hq:])
        if fp4:
            kk, vv = _read(ctx, cache, room, base, S, hkv, hd)
            assert torch.equal(kk, R.rounded(k)) and torch.equal(vv, R.rounded(x[:, hq + hkv:]))
        else:
            _within(kv[base:base + S, :, 0], k, _y_tol(k, x[:, hq:hq + hkv], kw, 1e-5), "keys")
            assert torch.equal(kv[base:base + S, :, 1].cpu(), qkv.view(S, -1, hd)[:, hq + hkv:])


@pytest.mark.parametrize("S", [3, 1500])
@pytest.mark.parametrize("fp4", [False, True])
def test_write_at_offsets_below_zero(gpu, fp4, S):
    """Positions that lie before the cache rows, the first of them below zero."""
    g = _gen(S)
    hq, hkv, hd, base = 12, 2, 128, 40
    qkv, w = _bf(g, S, (hq + 2 * hkv) * hd), 1 + _bf(g, hd, std=0.2)
    x, room = qkv.double().view(S, -1, hd), base + S
    ctx = C.make_attention_ctx(hq, hkv, hd, q_rope_pos_offset=2 ** 32 - 41, k_rope_pos_offset=2 ** 32 - 7)
    q = torch.empty(S, hq, hd, dtype=torch.bfloat16, device="cuda")
    dst = [_buf(C.load().efm_kv_fp4_bytes(ctx, room))] if fp4 else \
        [torch.empty(room, hkv, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    _write(ctx, fp4, qkv.cuda(), w.cuda(), w.cuda(), q, dst, room, S, base)
    torch.cuda.synchronize()
    ref = R.norm_rope(x[:, :hq], w, 1e-6, _positions(base, S, 64, -41), 1e6)
    _within(q, ref, _y_tol(ref, x[:, :hq], w, 1e-6), "queries")
    k = R.norm_rope(x[:, hq:hq + hkv], w, 1e-6, _positions(base, S, 64, -7), 1e6)
    if fp4:
        assert torch.equal(_read(ctx, dst[0], room, base, S, hkv, hd)[0], R.rounded(k))
    else:
        _within(dst[0][base:], k, _y_tol(k, x[:, hq:hq + hkv], w, 1e-6), "keys")


@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("length", [0, 2, 3, 50, 64, 65])
def test_write_at_a_device_length(gpu, fp4, length):
    """Three rows that end at *d_kv_len; a length outside [3, 64] writes nothing. Equal to the call with the host's base."""
    g = _gen(2)
    hq, hkv, hd, S, room = 12, 2, 128, 3, 64
    ctx = C.make_attention_ctx(hq, hkv, hd)
    qkv, w = _bf(g, S, (hq + 2 * hkv) * hd).cuda(), (1 + _bf(g, hd, std=0.2)).cuda()
    d_len = torch.tensor([length], dtype=torch.int32, device="cuda")
    outs = []
    for by_device in (True, False):
        q = torch.full((S, hq, hd), 7.0, dtype=torch.bfloat16, device="cuda")
        dst = [_buf(C.load().efm_kv_fp4_bytes(ctx, room), 0x11)] if fp4 else \
            [torch.full((room, hkv, hd), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        if by_device:
            _write(ctx, fp4, qkv, w, w, q, dst, room, S, 0, d_len=d_len)
        elif S <= length <= room:
            _write(ctx, fp4, qkv, w, w, q, dst, room, S, length - S)
        torch.cuda.synchronize()
        outs.append([q] + dst)
    for a, b in zip(*outs):
        assert torch.equal(a, b)


@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("length", [1601, 1602, 1700, 1701])
def test_write_many_rows_at_a_device_length(gpu, fp4, length):
    """1602 rows, equal to blocks of 89 by the host's base; too short or long a length writes nothing."""
    g = _gen(2)
    hq, hkv, hd, S, room = 12, 2, 128, 1602, 1700
    ctx = C.make_attention_ctx(hq, hkv, hd)
    qkv, w = _bf(g, S, (hq + 2 * hkv) * hd).cuda(), (1 + _bf(g, hd, std=0.2)).cuda()
    d_len = torch.tensor([length], dtype=torch.int32, device="cuda")
    outs = []
    for by_device in (True, False):
        q = torch.full((S, hq, hd), 7.0, dtype=torch.bfloat16, device="cuda")
        dst = [_buf(C.load().efm_kv_fp4_bytes(ctx, room), 0x11)] if fp4 else \
            [torch.full((room, hkv, hd), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        if by_device:
            _write(ctx, fp4, qkv, w, w, q, dst, room, S, 0, d_len=d_len)
        elif S <= length <= room:
            for i in range(0, S, 89):
                _write(ctx, fp4, qkv[i:i + 89], w, w, q[i:i + 89], dst, room, 89, length - S + i)
        torch.cuda.synchronize()
        outs.append([q] + dst)
    for a, b in zip(*outs):
        assert torch.equal(a, b)


@pytest.mark.parametrize("n", [40, 4200])
def test_write_without_queries_in_many_rows(gpu, n):
    """Keys and values alone, wide enough for rows together; nothing but the cache changes."""
    g = _gen(n)
    hq, hkv, hd = 14, 2, 64
    ctx = C.make_attention_ctx(hq, hkv, hd)
    qkv, w = _bf(g, n, 18 * 64), 1 + _bf(g, hd, std=0.2)
    cache, dev = _buf(C.load().efm_kv_fp4_bytes(ctx, n)), qkv.cuda()
    _write(ctx, True, dev, None, w.cuda(), None, [cache], n, n, 0)
    k, v = _read(ctx, cache, n, 0, n, hkv, hd)
    x = qkv.double().view(n, 18, 64)
    assert torch.equal(k, R.rounded(R.norm_rope(x[:, 14:16], w, 1e-6, _positions(0, n, 32), 1e6)))
    assert torch.equal(v, R.rounded(x[:, 16:])) and torch.equal(dev.cpu(), qkv)


def test_write_without_queries_and_read_of_one_side(gpu):
    g = _gen(4)
    ctx = C.make_attention_ctx(14, 2, 64, rope=False)
    qkv = _bf(g, 9, 18 * 64)
    x = qkv.double().view(9, 18, 64)
    cache = _buf(C.load().efm_kv_fp4_bytes(ctx, 9))
    _write(ctx, True, qkv.cuda(), None, None, None, [cache], 9, 9, 0, eps=0.0)
    k = torch.empty(4, 2, 64, dtype=torch.bfloat16, device="cuda")
    C.call("efm_kv_fp4_read", ctx, ptr(cache), 9, 5, 4, ptr(k), None, stream())
    v = torch.empty(4, 2, 64, dtype=torch.bfloat16, device="cuda")
    C.call("efm_kv_fp4_read", ctx, ptr(cache), 9, 5, 4, None, ptr(v), stream())
    torch.cuda.synchronize()
    assert torch.equal(k.cpu().double(), R.rounded(x[5:, 14:16])) and torch.equal(v.cpu().double(), R.rounded(x[5:, 16:]))


@pytest.mark.parametrize("heads", [65535, 65536])
def test_the_most_heads(gpu, heads):
    """Written, read back and attended: a row of one key is its value."""
    g = _gen(heads)
    ctx = C.make_attention_ctx(heads, heads, 64, rope=False)
    qkv = _bf(g, 2, 3 * heads * 64)
    x = qkv.view(2, 3 * heads, 64)
    cache, q = _buf(C.load().efm_kv_fp4_bytes(ctx, 3), 0xff), torch.empty(2, heads, 64, dtype=torch.bfloat16, device="cuda")
    _write(ctx, True, qkv.cuda(), None, None, q, [cache], 3, 2, 0)
    k, v = _read(ctx, cache, 3, 0, 2, heads, 64)
    at = torch.cat([torch.arange(40), torch.randint(0, heads, (500,), generator=g), torch.arange(heads - 40, heads)])
    assert torch.equal(q.cpu(), x[:, :heads])
    assert torch.equal(k[:, at], R.rounded(x[:, heads + at])) and torch.equal(v[:, at], R.rounded(x[:, 2 * heads + at]))
    assert torch.equal(_decode(ctx, q[:1], cache, 3, 1).cpu().double(), v[:1])
    assert torch.equal(_rows(ctx, q, cache, 3, 2, 2)[0].cpu().double(), v[0])


@pytest.mark.parametrize("n,kv", [(1, 70), (40, 100), (600, 900)])
def test_the_largest_values_reach_the_rows_that_see_them(gpu, n, kv):
    """Values up to 7 * 2^125 are stored as finite ones, larger as NaN: neither reaches a row before their key."""
    hq, hkv, hd = 12, 2, 128
    q, k, v = _qkv(n, n, kv, hq, hkv, hd)
    at = kv - max(1, n // 2)
    v[at, 0, 3], v[at, 1, 70] = 7 * 2.0 ** 125, torch.finfo(torch.bfloat16).max
    ctx = C.make_attention_ctx(hq, hkv, hd, rope=False)
    cache = _fill(ctx, k, v, kv)
    got = _read(ctx, cache, kv, at, 1, hkv, hd)[1]
    assert got[0, 0, 3] == 6 * 2.0 ** 125 and got[0, 1].isnan().sum() == 32
    o = _rows(ctx, q.cuda(), cache, kv, n, kv).cpu()
    before = torch.arange(n) + kv - n < at
    assert torch.isfinite(o[before]).all() and o[~before, hq // 2:, 64:96].isnan().all()
    rv = R.rounded(v)
    ref, tol = R.attention(q.double(), R.rounded(k), rv.nan_to_num(0), True)
    _within(o[before], ref[before], tol[before])


def test_write_fp4_groups_that_are_not_finite(gpu):
    g = _gen(6)
    hq, hkv, hd = 12, 2, 128
    ctx = C.make_attention_ctx(hq, hkv, hd, rope=False)
    qkv = _bf(g, 4, (hq + 2 * hkv) * hd)
    x = qkv.view(4, -1, hd)
    x[1, hq, 40], x[2, hq + 1, 0], x[3, hq + 2, 127], x[0, hq + 3, 64] = math.nan, math.inf, -math.inf, math.nan
    cache = _buf(C.load().efm_kv_fp4_bytes(ctx, 4))
    _write(ctx, True, qkv.cuda(), None, None, None, [cache], 4, 4, 0)
    k, v = _read(ctx, cache, 4, 0, 4, hkv, hd)
    for got, ref in ((k, R.rounded(x[:, hq:hq + hkv])), (v, R.rounded(x[:, hq + hkv:]))):
        assert int(torch.isnan(ref).sum()) == 64
        assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(got.nan_to_num(0), ref.nan_to_num(0))


# ---------------------------------------------------------------- attention

def _fill(ctx, k, v, room, stale=0xff):
    """A cache of `room` rows whose first hold k, v [kv, hkv, hd]; the rest holds `stale` bytes (0xff: NaN groups)."""
    kv, hkv, hd = k.shape
    hq = ctx.num_qo_heads
    cache = _buf(C.load().efm_kv_fp4_bytes(ctx, room), stale)
    if kv:
        rows = torch.cat([torch.zeros(kv, hq * hd, dtype=torch.bfloat16), k.flatten(1), v.flatten(1)], 1).cuda()
        none = C.make_attention_ctx(hq, hkv, hd, rope=False)
        _write(none, True, rows, None, None, None, [cache], room, kv, 0)
    torch.cuda.synchronize()
    return cache


def _decode(ctx, q, cache, room, kv, d_len=None, bound=0):
    ws = _buf(C.load().efm_attention_decode_kv_fp4_workspace_bytes(ctx, bound or kv), 0xff)
    o = torch.full((1, ctx.num_qo_heads, ctx.head_dim), 9.0, dtype=torch.bfloat16, device="cuda")
    C.call("efm_attention_decode_kv_fp4", ctx, ptr(q), ptr(cache), room, ptr(o), kv, ptr(d_len), bound, ptr(ws), ws.numel(), stream())
    torch.cuda.synchronize()
    return o


def _rows(ctx, q, cache, room, n, kv, causal=True):
    ws = _buf(C.load().efm_attention_prefill_kv_fp4_workspace_bytes(ctx, n, kv), 0xff)
    o = torch.full((n, ctx.num_qo_heads, ctx.head_dim), 9.0, dtype=torch.bfloat16, device="cuda")
    C.call("efm_attention_prefill_kv_fp4", ctx, ptr(q), ptr(cache), room, ptr(o), n, kv, int(causal), ptr(ws), ws.numel(), stream())
    torch.cuda.synchronize()
    return o


def _qkv(seed, n, kv, hq, hkv, hd):
    g = _gen(seed)
    k = _bf(g, kv, hkv, hd)
    k[..., 5] *= 6
    return _bf(g, n, hq, hd), k, _bf(g, kv, hkv, hd)


@pytest.mark.parametrize("hq,hkv,hd", HEADS + [pytest.param(2, 2, 128, id="mha"), pytest.param(16, 2, 64, id="8of64"),
                                                pytest.param(3, 1, 64, id="3of64")])
@pytest.mark.parametrize("kv", [0, 1, 31, 32, 33, 257, 1000, 4099])
def test_decode(gpu, hq, hkv, hd, kv):
    """Host length, and the same with the length on the device under a larger bound; rows past it hold NaN groups."""
    q, k, v = _qkv(kv + hd, 1, kv, hq, hkv, hd)
    room = kv + 77
    ctx = C.make_attention_ctx(hq, hkv, hd, rope=False)
    cache = _fill(ctx, k, v, room)
    ref, tol = R.attention(q.double(), R.rounded(k), R.rounded(v), False)
    _within(_decode(ctx, q.cuda(), cache, room, kv), ref, tol, "host length")
    d_len = torch.tensor([kv], dtype=torch.int32, device="cuda")
    _within(_decode(ctx, q.cuda(), cache, room, 0, d_len, room), ref, tol, "device length")


def test_decode_long(gpu):
    q, k, v = _qkv(1, 1, 40001, 28, 4, 128)
    ctx = C.make_attention_ctx(28, 4, 128, rope=False)
    cache = _fill(ctx, k, v, 65536)
    ref, tol = R.attention(q.double(), R.rounded(k), R.rounded(v), False)
    _within(_decode(ctx, q.cuda(), cache, 65536, 40001), ref, tol)
    d_len = torch.tensor([40001], dtype=torch.int32, device="cuda")
    _within(_decode(ctx, q.cuda(), cache, 65536, 0, d_len, 65536), ref, tol)


@pytest.mark.parametrize("kv", [8161, 16400, 65536, 70001])
def test_decode_of_one_kv_head(gpu, kv):
    """Up to as many splits as a joining workgroup has threads, the last ones short or, by a smaller length on the device,
    without keys."""
    q, k, v = _qkv(kv, 1, kv, 7, 1, 128)
    ctx = C.make_attention_ctx(7, 1, 128, rope=False)
    cache = _fill(ctx, k, v, kv + 3)
    ref, tol = R.attention(q.double(), R.rounded(k), R.rounded(v), False)
    _within(_decode(ctx, q.cuda(), cache, kv + 3, kv), ref, tol)
    n = kv // 3
    d_len = torch.tensor([n], dtype=torch.int32, device="cuda")
    ref, tol = R.attention(q.double(), R.rounded(k[:n]), R.rounded(v[:n]), False)
    _within(_decode(ctx, q.cuda(), cache, kv + 3, 0, d_len, kv), ref, tol)


def test_decode_length_beyond_the_bound(gpu):
    """*d_kv_len past max_kv_len attends max_kv_len rows."""
    q, k, v = _qkv(8, 1, 200, 12, 2, 128)
    ctx = C.make_attention_ctx(12, 2, 128, rope=False)
    cache = _fill(ctx, k, v, 200)
    d_len = torch.tensor([4000000], dtype=torch.int32, device="cuda")
    ref, tol = R.attention(q.double(), R.rounded(k[:150]), R.rounded(v[:150]), False)
    _within(_decode(ctx, q.cuda(), cache, 200, 0, d_len, 150), ref, tol)


ROWS = [(1, 1), (1, 40), (2, 2), (7, 7), (16, 100), (33, 33), (37, 800), (5, 3001), (130, 130), (200, 1111), (515, 515), (700, 1500)]


@pytest.mark.parametrize("hq,hkv,hd", HEADS)
@pytest.mark.parametrize("n,kv", ROWS)
@pytest.mark.parametrize("causal", [True, False])
def test_rows(gpu, hq, hkv, hd, n, kv, causal):
    q, k, v = _qkv(n + kv, n, kv, hq, hkv, hd)
    room = kv + 5
    ctx = C.make_attention_ctx(hq, hkv, hd, rope=False)
    ref, tol = R.attention(q.double(), R.rounded(k), R.rounded(v), causal)
    _within(_rows(ctx, q.cuda(), _fill(ctx, k, v, room), room, n, kv, causal), ref, tol)


@pytest.mark.parametrize("hq,hkv,hd", [(1, 1, 128), (8, 4, 64), (24, 6, 128), (16, 2, 128)])
@pytest.mark.parametrize("n,kv", [(19, 150), (300, 400)])
def test_rows_head_layouts(gpu, hq, hkv, hd, n, kv):
    q, k, v = _qkv(n, n, kv, hq, hkv, hd)
    ctx = C.make_attention_ctx(hq, hkv, hd, rope=False)
    ref, tol = R.attention(q.double(), R.rounded(k), R.rounded(v), True)
    _within(_rows(ctx, q.cuda(), _fill(ctx, k, v, kv), kv, n, kv), ref, tol)


# Many blocks of 128 rows: workgroups that share the unpacked keys
SHARED = [(64, 64, 1000, 1501, True), (64, 64, 1000, 1000, False), (96, 96, 900, 900, True), (256, 32, 340, 340, True),
          (320, 320, 130, 333, True), (320, 320, 130, 131, False), (224, 32, 366, 397, True), (640, 640, 2, 77, True),
          (640, 640, 2, 2, True), (648, 648, 65, 65, True)]


@pytest.mark.parametrize("hq,hkv,n,kv,causal", SHARED)
def test_rows_of_many_blocks(gpu, hq, hkv, n, kv, causal):
    """Rows past the end hold NaN groups; strided queries; every third head is checked, and a second call's equality."""
    g = _gen(hq + n + kv)
    k, v, q = _bf(g, kv, hkv, 128), _bf(g, kv, hkv, 128), _bf(g, n, hq, 128)
    k[..., 5] *= 6
    room = kv + 100
    wide = torch.full((n, hq, 136), math.nan, dtype=torch.bfloat16, device="cuda")
    wide[..., :128] = q.cuda()
    ctx = C.make_attention_ctx(hq, hkv, 128, rope=False, q_stride_n=hq * 136, q_stride_h=136)
    cache = _fill(ctx, k, v, room)
    o = _rows(ctx, wide, cache, room, n, kv, causal)
    kvh = torch.arange(0, hkv, 3)
    qh = (kvh[:, None] * (hq // hkv) + torch.arange(hq // hkv)).flatten()
    ref, tol = R.attention(q[:, qh].double(), R.rounded(k[:, kvh]), R.rounded(v[:, kvh]), causal)
    _within(o[:, qh.cuda()], ref, tol)
    assert not o.isnan().any() and torch.equal(o, _rows(ctx, wide, cache, room, n, kv, causal))


@pytest.mark.parametrize("what", ["key", "value"])
def test_nan_groups_of_many_blocks(gpu, what):
    hq = hkv = 320
    n, kv, at = 130, 300, 221
    q, k, v = _qkv(n, n, kv, hq, hkv, 128)
    (k if what == "key" else v)[at, 7, 40] = math.nan
    ctx = C.make_attention_ctx(hq, hkv, 128, rope=False)
    heads = torch.tensor([0, 6, 7, 8, 319])
    o = _rows(ctx, q.cuda(), _fill(ctx, k, v, kv), kv, n, kv)
    ref, tol = R.attention(q[:, heads].double(), R.rounded(k[:, heads]).nan_to_num(0), R.rounded(v[:, heads]).nan_to_num(0), True)
    sees = torch.arange(n) + kv - n >= at
    if what == "key":
        ref[sees, 2] = math.nan
    else:
        ref[sees, 2, 32:64] = math.nan
    _within(o[:, heads.cuda()], ref, tol, what)
    others = torch.arange(hq) != 7
    assert not o[:, others.cuda()].isnan().any()


def test_a_workspace_serves_fewer_rows_and_keys(gpu):
    """One workspace of the largest call's bytes is enough for every smaller call."""
    lib, ctx = C.load(), C.make_attention_ctx(28, 4, 128, rope=False)
    kv = 8300
    q, k, v = _qkv(3, 40, kv, 28, 4, 128)
    cache, q = _fill(ctx, k, v, kv), q.cuda()
    ws = _buf(lib.efm_attention_prefill_kv_fp4_workspace_bytes(ctx, 40, kv))
    wd = _buf(lib.efm_attention_decode_kv_fp4_workspace_bytes(ctx, kv))
    for n in (40, 17, 5, 1):
        for L in (8300, 8192, 4096, 1000, 600, 300, 40):
            o = torch.empty(n, 28, 128, dtype=torch.bfloat16, device="cuda")
            C.call("efm_attention_prefill_kv_fp4", ctx, ptr(q), ptr(cache), kv, ptr(o), n, L, 1, ptr(ws), ws.numel(), stream())
            assert torch.equal(o, _rows(ctx, q, cache, kv, n, L))
            if n == 1:
                C.call("efm_attention_decode_kv_fp4", ctx, ptr(q), ptr(cache), kv, ptr(o), L, None, 0, ptr(wd), wd.numel(), stream())
                assert torch.equal(o, _decode(ctx, q, cache, kv, L))


@pytest.mark.parametrize("n", [1, 21, 600])
def test_rows_strided_queries(gpu, n):
    """Queries inside a wider buffer with the heads apart: strides of ctx."""
    hq, hkv, hd, kv = 12, 2, 128, n + 90
    q, k, v = _qkv(n, n, kv, hq, hkv, hd)
    wide = torch.full((n, hq, 2, hd), math.nan, dtype=torch.bfloat16)
    wide[:, :, 1] = q
    wide = wide.cuda()
    ctx = C.make_attention_ctx(hq, hkv, hd, rope=False, q_stride_n=hq * 2 * hd, q_stride_h=2 * hd)
    ref, tol = R.attention(q.double(), R.rounded(k), R.rounded(v), True)
    _within(_rows(ctx, wide[:, :, 1], _fill(ctx, k, v, kv), kv, n, kv), ref, tol)
    if n == 1:
        _within(_decode(ctx, wide[:, :, 1], _fill(ctx, k, v, kv), kv, kv), ref, tol)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,kv", [(1, 300), (40, 300), (700, 900)])
def test_nan_groups_reach_the_rows_that_see_them(gpu, hd, n, kv):
    """A NaN group of a key makes NaN of every row that sees the key, one of a value of that head's channels of the group
    in those rows; rows before it, and the other KV head, keep their results."""
    hq, hkv, at = 12, 2, kv - max(1, n // 2)
    q, k, v = _qkv(n, n, kv, hq, hkv, hd)
    ctx = C.make_attention_ctx(hq, hkv, hd, rope=False)
    for what in ("key", "value"):
        kk, vv = k.clone(), v.clone()
        if what == "key":
            kk[at, 1, 3] = math.nan
        else:
            vv[at, 0, 33] = math.inf
        rk, rv = R.rounded(kk), R.rounded(vv)
        ref, tol = R.attention(q.double(), rk.nan_to_num(0), rv.nan_to_num(0), True)
        clean = torch.arange(n) + kv - n < at
        if what == "key":
            ref[~clean, hq // 2:] = math.nan
        else:
            ref[~clean, :hq // 2, 32:64] = math.nan
        assert n == 1 or clean.any()
        _within(_rows(ctx, q.cuda(), _fill(ctx, kk, vv, kv), kv, n, kv), ref, tol, what)
        if n == 1:
            _within(_decode(ctx, q.cuda(), _fill(ctx, kk, vv, kv + 9), kv + 9, kv), ref, tol, what + ", decode")


@pytest.mark.parametrize("hq,hkv,hd", [(12, 2, 128), (14, 2, 64), (320, 320, 128)])
@pytest.mark.parametrize("n,kv", [(1, 700), (40, 300), (130, 333)])
def test_queries_that_are_not_finite(gpu, hq, hkv, hd, n, kv):
    """A NaN or an infinity in a query makes NaN of its own row and head alone."""
    q, k, v = _qkv(n, n, kv, hq, hkv, hd)
    heads = torch.tensor([0, 1, hq // 2, hq - 1])
    ctx = C.make_attention_ctx(hq, hkv, hd, rope=False)
    kvh = heads // (hq // hkv)
    ref, tol = R.attention(q[:, heads].double(), R.rounded(k[:, kvh]), R.rounded(v[:, kvh]), True)
    for bad in (math.nan, math.inf):
        x = q.clone()
        x[n // 2, 1, 7] = bad
        want = ref.clone()
        want[n // 2, 1] = math.nan
        cache = _fill(ctx, k, v, kv)
        o = _rows(ctx, x.cuda(), cache, kv, n, kv)
        _within(o[:, heads.cuda()], want, tol, str(bad))
        assert int(o.isnan().sum()) == hd
        if n == 1:
            assert torch.equal(_decode(ctx, x.cuda(), cache, kv, kv).isnan(), o.isnan())


@pytest.mark.parametrize("n", [1, 50, 600])
def test_large_scores(gpu, n):
    """Scores of thousands: one key takes all the weight, whichever wave or split holds it."""
    hq, hkv, hd, kv = 12, 2, 128, n + 1200
    q, k, v = _qkv(5, n, kv, hq, hkv, hd)
    q, k = q * 16, k * 16
    ctx = C.make_attention_ctx(hq, hkv, hd, rope=False)
    ref, tol = R.attention(q.double(), R.rounded(k), R.rounded(v), True)
    _within(_rows(ctx, q.cuda(), _fill(ctx, k, v, kv), kv, n, kv), ref, tol)


def test_decode_in_a_graph(gpu):
    """Two captured steps of different heads share a workspace, and follow the length on the device."""
    lib = C.load()
    shapes = [(28, 4, 128, 5000), (14, 2, 64, 900)]
    bufs = []
    for hq, hkv, hd, room in shapes:
        q, k, v = _qkv(room, 1, room, hq, hkv, hd)
        ctx = C.make_attention_ctx(hq, hkv, hd, rope=False)
        bufs.append((ctx, q.cuda(), _fill(ctx, k, v, room), room, torch.empty(1, hq, hd, dtype=torch.bfloat16, device="cuda")))
    d_len = torch.tensor([1], dtype=torch.int32, device="cuda")
    ws = _buf(max(lib.efm_attention_decode_kv_fp4_workspace_bytes(b[0], b[3]) for b in bufs))
    s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s, capture_error_mode="thread_local"):
        for ctx, q, cache, room, o in bufs:
            C.call("efm_attention_decode_kv_fp4", ctx, ptr(q), ptr(cache), room, ptr(o), 0, ptr(d_len), room, ptr(ws), ws.numel(), s.cuda_stream)
    for length in (700, 33, 900, 1):
        d_len.fill_(length)
        ws.fill_(0xff)
        torch.randn(1 << 18, device="cuda").sum()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for ctx, q, cache, room, o in bufs:
            assert torch.equal(o, _decode(ctx, q, cache, room, 0, d_len, room))


# ---------------------------------------------------------------- together

def test_layer_step_and_prompt(gpu):
    """A layer with FP4 weights over an FP4 cache, as a program runs it: a prompt of 45 rows, then steps of one row with the
    length on the device. Each operator's output is checked against 64 bits on the inputs that it was given."""
    g = _gen(12)
    hidden, hq, hkv, hd, inter, room, S = 512, 8, 2, 64, 1024, 64, 45
    width = (hq + 2 * hkv) * hd
    mats = {n: _weights(g, o, k) for n, o, k in (("qkv", width, hidden), ("o", hidden, hq * hd), ("gu", 2 * inter, hidden), ("down", hidden, inter))}
    packed = {n: _pack(R.halves(c), b) for n, (c, b) in mats.items()}
    w64 = {n: R.values(c, b) for n, (c, b) in mats.items()}
    qw, kw, bias = 1 + _bf(g, hd, std=0.2), 1 + _bf(g, hd, std=0.2), _bf(g, width)
    rope, ctx = C.make_attention_ctx(hq, hkv, hd), C.make_attention_ctx(hq, hkv, hd, rope=False)
    cache = _buf(C.load().efm_kv_fp4_bytes(ctx, room), 0xff)
    d_len = torch.tensor([S], dtype=torch.int32, device="cuda")
    dev = [t.cuda() for t in (qw, kw, bias)]
    keys, vals = torch.zeros(0, hkv, hd, dtype=torch.float64), torch.zeros(0, hkv, hd, dtype=torch.float64)

    def check_linear(y, x, name, b=None):
        ref, tol = _product(x.cpu().double(), w64[name])
        if b is not None:
            ref = ref + b.double()
        _within(y, ref, tol + 2.0 ** -23 * ref.abs() + HALF * (ref.abs() + tol), name)

    base = 0
    for n in (S, 1, 1, 1):
        x = _bf(g, n, hidden).cuda()
        qkv = _linear(x, packed["qkv"], hidden, width, dev[2])
        check_linear(qkv, x, "qkv", bias)
        q = torch.empty(n, hq, hd, dtype=torch.bfloat16, device="cuda")
        if n == 1:
            d_len += 1
            _write(rope, True, qkv, dev[0], dev[1], q, [cache], room, 1, 0, d_len=d_len)
        else:
            _write(rope, True, qkv, dev[0], dev[1], q, [cache], room, n, 0)
        rows = qkv.cpu().double().view(n, -1, hd)
        pos = _positions(base, n, hd // 2)
        keys = torch.cat([keys, R.rounded(R.norm_rope(rows[:, hq:hq + hkv], kw, 1e-6, pos, 1e6))])
        vals = torch.cat([vals, R.rounded(rows[:, hq + hkv:])])
        base += n
        att = _rows(ctx, q, cache, room, n, base) if n > 1 else _decode(ctx, q, cache, room, 0, d_len, room)
        ref, tol = R.attention(q.cpu().double(), keys, vals, True)
        _within(att, ref, tol, "attention")
        check_linear(_linear(att.view(n, -1), packed["o"], hq * hd, hidden), att.view(n, -1), "o")
        mid = torch.empty(n, inter, dtype=torch.bfloat16, device="cuda")
        ws = _buf(C.load().efm_fused_gate_up_swiglu_fp4_workspace_bytes(n, hidden, inter))
        C.call("efm_fused_gate_up_swiglu_fp4", n, hidden, inter, ptr(x), ptr(packed["gu"]), ptr(mid), ptr(ws), ws.numel(), stream())
        check_linear(_linear(mid, packed["down"], inter, hidden), mid, "down")


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [1, 3, 1100])
def test_queries_at_a_device_length_and_the_activation(gpu, n, hd):
    """Queries of rows that end at the device's length, and what the down projection is given, against 64 bits: the outputs
    of a layer that its attention and its down projection take as they are."""
    g = _gen(n + hd)
    hidden, hq, hkv, inter, room, length = 512, 8, 2, 1024, 1400, 1331
    width = (hq + 2 * hkv) * hd
    code, byte = _weights(g, 2 * inter, hidden)
    qkv, x, qw, kw = _bf(g, n, width), _bf(g, n, hidden), 1 + _bf(g, hd, std=0.2), 1 + _bf(g, hd, std=0.2)
    ctx = C.make_attention_ctx(hq, hkv, hd)
    d_len = torch.tensor([length], dtype=torch.int32, device="cuda")
    pos = _positions(length - n, n, hd // 2)
    heads = qkv.double().view(n, -1, hd)
    ref = R.norm_rope(heads[:, :hq], qw, 1e-6, pos, 1e6)
    tol = _y_tol(ref, heads[:, :hq], qw, 1e-6)
    dev = [t.cuda() for t in (qkv, qw, kw)]
    for fp4 in (True, False):
        dst = [_buf(C.load().efm_kv_fp4_bytes(ctx, room))] if fp4 else \
            [torch.zeros(room, hkv, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        q = torch.full((n, hq, hd), math.nan, dtype=torch.bfloat16, device="cuda")
        _write(ctx, fp4, *dev, q, dst, room, n, 0, d_len=d_len)
        torch.cuda.synchronize()
        _within(q, ref, tol, "queries")
    packed, xd = _pack(R.halves(code), byte), x.cuda()
    mid = torch.full((n, inter), math.nan, dtype=torch.bfloat16, device="cuda")
    C.call("efm_fused_gate_up_swiglu_fp4", n, hidden, inter, ptr(xd), ptr(packed), ptr(mid), None, 0, stream())
    torch.cuda.synchronize()
    _within(mid, *_swiglu(x, R.values(code, byte)), "activation")


def test_same_stream_order_on_a_side_stream(gpu):
    """Write, read and attention queued on a side stream follow each other without host waits."""
    hq, hkv, hd, kv = 12, 2, 128, 400
    q, k, v = _qkv(3, 1, kv, hq, hkv, hd)
    ctx = C.make_attention_ctx(hq, hkv, hd, rope=False)
    rows = torch.cat([torch.zeros(kv, hq * hd, dtype=torch.bfloat16), k.flatten(1), v.flatten(1)], 1).cuda()
    cache, qd = _buf(C.load().efm_kv_fp4_bytes(ctx, kv), 0xff), q.cuda()
    ws = _buf(C.load().efm_attention_decode_kv_fp4_workspace_bytes(ctx, kv))
    o = torch.empty(1, hq, hd, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    _write(ctx, True, rows, None, None, None, [cache], kv, kv, 0, on=s.cuda_stream)
    C.call("efm_attention_decode_kv_fp4", ctx, ptr(qd), ptr(cache), kv, ptr(o), kv, None, 0, ptr(ws), ws.numel(), s.cuda_stream)
    s.synchronize()
    ref, tol = R.attention(q.double(), R.rounded(k), R.rounded(v), False)
    _within(o, ref, tol)


def test_layer_step_in_a_graph(gpu):
    """A decode step of a layer captured once and replayed for several rows, the workspaces shared by its operators: bit
    for bit the eager step, cache included."""
    g = _gen(21)
    lib = C.load()
    hidden, hq, hkv, hd, inter, room = 512, 8, 2, 128, 768, 1300
    width = (hq + 2 * hkv) * hd
    packed = {n: _pack(*_weights_on_device(i, o, k)) for i, (n, o, k) in
              enumerate((("qkv", width, hidden), ("o", hidden, hq * hd), ("gu", 2 * inter, hidden), ("down", hidden, inter)))}
    qw, kw, bias = ((1 + _bf(g, n, std=0.2)).cuda() for n in (hd, hd, width))
    rope, ctx = C.make_attention_ctx(hq, hkv, hd), C.make_attention_ctx(hq, hkv, hd, rope=False)
    start = 1200
    prompt = _bf(g, start, width).cuda()
    ws = _buf(lib.efm_attention_decode_kv_fp4_workspace_bytes(ctx, room))

    def state():
        cache = _buf(lib.efm_kv_fp4_bytes(ctx, room), 0xff)
        _write(rope, True, prompt, qw, kw, None, [cache], room, start, 0)
        return dict(cache=cache, x=torch.empty(1, hidden, dtype=torch.bfloat16, device="cuda"), n=torch.tensor([start], dtype=torch.int32, device="cuda"),
                    qkv=torch.empty(1, width, dtype=torch.bfloat16, device="cuda"), q=torch.empty(1, hq, hd, dtype=torch.bfloat16, device="cuda"),
                    att=torch.empty(1, hq * hd, dtype=torch.bfloat16, device="cuda"), out=torch.empty(1, hidden, dtype=torch.bfloat16, device="cuda"),
                    mid=torch.empty(1, inter, dtype=torch.bfloat16, device="cuda"), y=torch.empty(1, hidden, dtype=torch.float32, device="cuda"))

    def step(t, on):
        lin = lambda k, n, x, w, b, y, dt: C.call("efm_linear_fp4", 1, k, n, ptr(x), ptr(w), ptr(b), ptr(y), dt, None, 0, on)
        lin(hidden, width, t["x"], packed["qkv"], bias, t["qkv"], C.EFM_DTYPE_BF16)
        _write(rope, True, t["qkv"], qw, kw, t["q"], [t["cache"]], room, 1, 0, d_len=t["n"], on=on)
        C.call("efm_attention_decode_kv_fp4", ctx, ptr(t["q"]), ptr(t["cache"]), room, ptr(t["att"]), 0, ptr(t["n"]), room, ptr(ws), ws.numel(), on)
        lin(hq * hd, hidden, t["att"], packed["o"], None, t["out"], C.EFM_DTYPE_BF16)
        C.call("efm_fused_gate_up_swiglu_fp4", 1, hidden, inter, ptr(t["out"]), ptr(packed["gu"]), ptr(t["mid"]), None, 0, on)
        lin(inter, hidden, t["mid"], packed["down"], None, t["y"], C.EFM_DTYPE_F32)

    eager, captured = state(), state()
    s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s, capture_error_mode="thread_local"):
        step(captured, s.cuda_stream)
    for rep in range(4):
        x = _bf(g, 1, hidden)
        for t in (eager, captured):
            t["x"].copy_(x)
            t["n"] += 1
        ws.fill_(0xff)
        step(eager, stream())
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.isfinite(eager["y"]).all()
        for name in eager:
            assert torch.equal(eager[name], captured[name]), (rep, name)


def test_prompt_in_a_graph(gpu):
    """Write and attention of a prompt's rows behind others, captured and replayed with other rows."""
    g = _gen(22)
    hq, hkv, hd, base, n = 12, 2, 128, 500, 70
    room = base + n
    rope, ctx = C.make_attention_ctx(hq, hkv, hd), C.make_attention_ctx(hq, hkv, hd, rope=False)
    cache = _buf(C.load().efm_kv_fp4_bytes(ctx, room), 0xff)
    w = (1 + _bf(g, hd, std=0.2)).cuda()
    _write(rope, True, _bf(g, base, (hq + 2 * hkv) * hd).cuda(), w, w, None, [cache], room, base, 0)
    qkv = torch.empty(n, (hq + 2 * hkv) * hd, dtype=torch.bfloat16, device="cuda")
    q, o = (torch.empty(n, hq, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ws = _buf(C.load().efm_attention_prefill_kv_fp4_workspace_bytes(ctx, n, room))

    def both(on):
        _write(rope, True, qkv, w, w, q, [cache], room, n, base, on=on)
        C.call("efm_attention_prefill_kv_fp4", ctx, ptr(q), ptr(cache), room, ptr(o), n, room, 1, ptr(ws), ws.numel(), on)

    s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s, capture_error_mode="thread_local"):
        both(s.cuda_stream)
    for rep in range(3):
        qkv.copy_(_bf(g, *qkv.shape))
        ws.fill_(0xff)
        graph.replay()
        torch.randn(1 << 18, device="cuda").sum()
        torch.cuda.synchronize()
        got = o.clone()
        o.fill_(math.nan)
        both(stream())
        torch.cuda.synchronize()
        assert torch.isfinite(o).all() and torch.equal(got, o), f"replay {rep}"


def test_two_streams_at_once(gpu):
    """Calls on two streams, each with a workspace of its own, do not disturb each other."""
    hq, hkv, hd, kv = 28, 4, 128, 6000
    ctx = C.make_attention_ctx(hq, hkv, hd, rope=False)
    sets = []
    for seed in (1, 2):
        q, k, v = _qkv(seed, 1, kv, hq, hkv, hd)
        sets.append([q.cuda(), _fill(ctx, k, v, kv), _buf(C.load().efm_attention_decode_kv_fp4_workspace_bytes(ctx, kv)),
                     torch.empty(20, 1, hq, hd, dtype=torch.bfloat16, device="cuda"), torch.cuda.Stream()])
    torch.cuda.synchronize()
    for i in range(20):
        for q, cache, ws, o, s in sets:
            C.call("efm_attention_decode_kv_fp4", ctx, ptr(q), ptr(cache), kv, ptr(o[i]), kv, None, 0, ptr(ws), ws.numel(), s.cuda_stream)
    torch.cuda.synchronize()
    for q, cache, ws, o, s in sets:
        alone = _decode(ctx, q, cache, kv, kv)
        assert all(torch.equal(x, alone) for x in o)


def test_cache_past_32_bits(gpu):
    """The largest cache, 9 GB of 2^24 rows: zeros but for rows at both ends whose scores outweigh the rest."""
    hq, hkv, hd, room, n = 28, 4, 128, 1 << 24, 24
    g = _gen(31)
    ctx = C.make_attention_ctx(hq, hkv, hd, rope=False)
    cache = torch.zeros(C.load().efm_kv_fp4_bytes(ctx, room), dtype=torch.uint8, device="cuda")
    q, k, v = _bf(g, 1, hq, hd), _bf(g, 2 * n, hkv, hd), _bf(g, 2 * n, hkv, hd)
    k[::5] = q.view(hkv, hq // hkv, hd)[:, 0] * 2.5   # scores of 28 for a head of each group
    rows = torch.cat([torch.zeros(2 * n, hq * hd, dtype=torch.bfloat16), k.flatten(1), v.flatten(1)], 1).cuda()
    _write(ctx, True, rows[:n].contiguous(), None, None, None, [cache], room, n, 0)
    _write(ctx, True, rows[n:].contiguous(), None, None, None, [cache], room, n, room - n)
    kk, vv = R.rounded(k), R.rounded(v)
    for at, part in ((0, slice(0, n)), (room - n, slice(n, 2 * n))):
        a, b = _read(ctx, cache, room, at, n, hkv, hd)
        assert torch.equal(a, kk[part]) and torch.equal(b, vv[part])
    o = _decode(ctx, q.cuda(), cache, room, room)
    rep = lambda t: t.repeat_interleave(hq // hkv, 1)
    s = (q.double() * rep(kk)).sum(-1) / math.sqrt(hd)                       # [rows, heads]
    mag = (q.double() * rep(kk)).abs().sum(-1).amax(0) / math.sqrt(hd)
    top = s.amax(0).clamp(min=0)
    w = (s - top).exp()
    den = w.sum(0) + (room - 2 * n) * (-top).exp()
    ref = (w[..., None] * rep(vv)).sum(0) / den[:, None]
    # as for shorter lengths: output and weights to bf16, scores in fp32; and a sum's chain, 2^19 tiles over 2^8 workgroups at
    # least and their partial sums: under 2^13 additions of 2^-23
    d = (hd / 32 + 40) * 2.0 ** -23 * mag[:, None]
    share = (w[..., None] * rep(vv).abs()).sum(0) / den[:, None]
    tol = HALF * ref.abs() + share * (HALF + 2 * d + 2.0 ** -18 + 2.0 ** -10)
    _within(o[0], ref, tol)
    assert (ref[:: hq // hkv].abs().amax(-1) > 0.1).all()
