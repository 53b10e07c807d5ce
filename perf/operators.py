"""Performance cases of the 4-bit operators and of the per-head norms with the rotation, through the C ABI.

A case is a dict of plain values. `listed()` gives the cases that are always measured, `draw()` more of the same
ranges; `prepare()` makes what a program has in hand before the call, `run()` is one pass, `exact()` the same pass in
64 bits, `work()` what the pass cannot do without. With `own` false, `run()` computes the operators in elementary
torch operations; with `own` true it makes the framework's calls.

Kinds of cases:
  linear   y = x W^T (+ b) with FP4 weights
  swiglu   silu(x Wg^T) * (x Wu^T) with FP4 weights, W = [up; gate]
  write    norm of queries and keys per head, position rotation and cache write; the cache holds bf16 or FP4
  decode   one query row over an FP4 cache
  rows     several query rows, causal, over an FP4 cache that holds their own keys too

FP4 is the microscaling format: groups of 32 values share a scale 2^e, a value is one of 0, 0.5, 1, 1.5, 2, 3, 4, 6
with a sign. Layer dimensions are those of efm_setup's model shapes.
"""
import math
import os
import sys

import torch

own = False

# (hidden, heads, kv heads, head_dim, intermediate, M-RoPE sections)
MODELS = {"0p5b": (896, 14, 2, 64, 4864, None), "1p5b": (1536, 12, 2, 128, 8960, None),
          "vl3b": (2048, 16, 2, 128, 11008, (16, 24, 24)), "7b": (3584, 28, 4, 128, 18944, None)}
THETA, EPS = 1.0e6, 1e-6
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _capi():
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "edge-fm-x_amd"))
    import efm_capi

    return efm_capi


def listed():
    return [
        # the smallest projection of a decode step, with its bias: latency counts
        dict(name="linear_decode_small", kind="linear", rows=1, inp=896, out=1152, bias=True, f32=False),
        # the fused q/k/v projection of a prompt on the largest model
        dict(name="linear_prompt", kind="linear", rows=1000, inp=3584, out=4608, bias=True, f32=False),
        # the widest weight stream of a decode step
        dict(name="swiglu_decode_large", kind="swiglu", rows=1, hidden=3584, inter=18944),
        # the MLP of a chat turn's few new rows
        dict(name="swiglu_turn", kind="swiglu", rows=24, hidden=1536, inter=8960),
        # a decode step's row into the bf16 cache
        dict(name="write_bf16_decode", kind="write", cache="bf16", model="1p5b", rows=1, base=640, norm=True, mrope=False),
        # a multimodal prompt into the bf16 cache: vision positions on a grid, then text
        dict(name="write_bf16_vision", kind="write", cache="bf16", model="vl3b", rows=1344, base=0, norm=True, mrope=True),
        # a decode step's row into the FP4 cache, far into a long context
        dict(name="write_fp4_decode", kind="write", cache="fp4", model="7b", rows=1, base=16400, norm=True, mrope=False),
        # a long prompt into the FP4 cache
        dict(name="write_fp4_prompt", kind="write", cache="fp4", model="7b", rows=4096, base=13, norm=True, mrope=False),
        # a decode step of a short chat on the narrow model (head_dim 64)
        dict(name="decode_short", kind="decode", model="0p5b", context=700),
        # a decode step of a long context
        dict(name="decode_long", kind="decode", model="7b", context=32771),
        # a turn's few new rows against a long cached prefix
        dict(name="rows_turn", kind="rows", model="1p5b", rows=37, prefix=8000),
        # a long prompt's second half
        dict(name="rows_long", kind="rows", model="7b", rows=2048, prefix=2048),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "swiglu", "write", "write", "decode", "decode", "rows", "rows"])
    if kind == "linear":
        rows = 1 if rng.random() < 0.4 else _log(rng, 2, 1000)
        return dict(kind=kind, rows=rows, inp=32 * _log(rng, 4, 592 if rows < 64 else 112), out=_log(rng, 100, 4608),
                    bias=rng.random() < 0.5, f32=rng.random() < 0.25)
    if kind == "swiglu":
        return dict(kind=kind, rows=rng.choice([1, 1, _log(rng, 2, 100)]), hidden=32 * _log(rng, 8, 112),
                    inter=16 * _log(rng, 20, 1184))
    model = rng.choice(sorted(MODELS))
    if kind == "write":
        mrope = model == "vl3b" and rng.random() < 0.7
        return dict(kind=kind, cache=rng.choice(["bf16", "fp4"]), model=model, rows=rng.choice([1, _log(rng, 2, 4000)]),
                    base=rng.choice([0, _log(rng, 1, 60000)]), norm=rng.random() < 0.7, mrope=mrope)
    if kind == "decode":
        return dict(kind=kind, model=model, context=_log(rng, 1, 32000))
    rows = _log(rng, 2, 2000)
    return dict(kind=kind, model=model, rows=rows, prefix=rng.choice([0, _log(rng, 1, min(16000, 4000000 // rows))]))


# Inputs, from the seed alone: weights N(0, 0.02) as the benchmark's, activations and cached values N(0, 1), a few
# channels of the keys several times larger, norm weights around one.

def _rng(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *size, std=1.0):
    return (torch.randn(*size, generator=g, device="cuda") * std).to(torch.bfloat16)


def _keys(g, *size):
    k = torch.randn(*size, generator=g, device="cuda")
    k[..., torch.randperm(size[-1], generator=g, device="cuda")[:3]] *= 6.0
    return k.to(torch.bfloat16)


def _codes(x):
    """FP4 codes (one to a byte) and scale bytes of x [..., K] in groups of 32 along K; 64 bits, so that no value next
    to a border falls on its other side."""
    x = x.double().unflatten(-1, (-1, 32))
    frac, exp = torch.frexp(x.abs().amax(-1, keepdim=True))
    e = (exp - 3 + (frac > 0.875)).clamp(min=-125)
    a = torch.ldexp(x.abs(), -e)
    code = ((a > 0.25).byte() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5)
            + 8 * (x < 0).byte())
    return code.flatten(-2), (e.squeeze(-1) + 127).to(torch.uint8)


def _halves(code):
    """Two codes to a byte, the even one in the low half."""
    return code[..., 0::2] | code[..., 1::2] << 4


def _values(packed, scale):
    """fp32 values of packed codes [..., K / 2] with scale bytes [..., K / 32]."""
    table = torch.tensor(GRID + tuple(-v for v in GRID), device=packed.device)
    code = torch.stack([packed & 15, packed >> 4], -1).flatten(-2)
    v = table[code.int()].unflatten(-1, (-1, 32))
    return (v * torch.exp2(scale.float() - 127).unsqueeze(-1)).flatten(-2)


def _linear_inputs(case, seed):
    g = _rng(seed)
    n, k, out = case["rows"], case.get("inp") or case["hidden"], case.get("out") or 2 * case["inter"]
    t = dict(x=_randn(g, n, k))
    w = torch.randn(out, k, generator=g, device="cuda") * 0.02
    parts = [_codes(p) for p in w.split(4096)]
    t["codes"], t["scales"] = (torch.cat([_halves(p[0]) for p in parts]), torch.cat([p[1] for p in parts]))
    if case.get("bias"):
        t["bias"] = _randn(g, out, std=0.5)
    return t


def _positions(case):
    """int32 [3, rows]: a grid of vision rows, then text positions past its largest."""
    n = case["rows"]
    grid = (n * 20 // 21) // 32 * 32
    i = torch.arange(grid, device="cuda", dtype=torch.int32)
    text = torch.arange(n - grid, device="cuda", dtype=torch.int32) + max(32, grid // 32)
    return case["base"] + torch.stack([torch.cat([torch.zeros_like(i), text]), torch.cat([i // 32, text]),
                                       torch.cat([i % 32, text])]).contiguous()


def _write_inputs(case, seed):
    _, hq, hkv, hd, _, _ = MODELS[case["model"]]
    g, n = _rng(seed), case["rows"]
    t = dict(qkv=torch.cat([_randn(g, n, hq * hd), _keys(g, n, hkv, hd).flatten(1), _randn(g, n, hkv * hd)], 1).contiguous())
    if case["norm"]:
        t["qw"], t["kw"] = 1 + _randn(g, hd, std=0.1), 1 + _randn(g, hd, std=0.1)
    if case["mrope"]:
        t["pos"] = _positions(case)
    return t


def _attention_inputs(case, seed):
    _, hq, hkv, hd, _, _ = MODELS[case["model"]]
    n = case.get("rows", 1)
    kv = case["context"] if case["kind"] == "decode" else n + case["prefix"]
    g = _rng(seed)
    return dict(q=_randn(g, n, hq, hd), k=_keys(g, kv, hkv, hd), v=_randn(g, kv, hkv, hd))


def _rows(n):
    return -(-n // 128) * 128   # the engine's row bound: whole 128-row buckets


def prepare(case, seed):
    kind = case["kind"]
    if kind in ("linear", "swiglu"):
        state = dict(case=case, **_linear_inputs(case, seed))
    elif kind == "write":
        state = dict(case=case, **_write_inputs(case, seed))
    else:
        t = _attention_inputs(case, seed)
        state = dict(case=case, q=t["q"], kv=t["k"].shape[0])
        if not own:   # the cache as packed codes and scales
            for name in ("k", "v"):
                code, scale = _codes(t[name])
                state[name] = (_halves(code), scale)
    if own:
        _prepare_own(case, state, t if kind in ("decode", "rows") else None)
    torch.cuda.synchronize()
    return state


def _prepare_own(case, state, t):
    """The packed weights, caches and workspaces that a program keeps, and the calls of a pass."""
    C = _capi()
    lib, kind, sh = C.load(), case["kind"], torch.cuda.current_stream().cuda_stream
    def empty(*size, dtype=torch.bfloat16):
        return torch.empty(*size, dtype=dtype, device="cuda")
    def buf(nbytes):
        return torch.zeros(max(int(nbytes), 256), dtype=torch.uint8, device="cuda")
    if kind in ("linear", "swiglu"):
        n, k = state["x"].shape
        out = state["codes"].shape[0]
        packed = buf(lib.efm_fp4_packed_bytes(k, out))
        C.call("efm_fp4_pack", k, out, state["codes"].data_ptr(), state["scales"].data_ptr(), packed.data_ptr(), sh)
        if kind == "linear":
            y = empty(n, out, dtype=torch.float32 if case["f32"] else torch.bfloat16)
            ws = buf(lib.efm_linear_fp4_workspace_bytes(n, k, out))
            bias = state["bias"].data_ptr() if case["bias"] else None
            calls = [("efm_linear_fp4", n, k, out, state["x"].data_ptr(), packed.data_ptr(), bias, y.data_ptr(),
                      C.EFM_DTYPE_F32 if case["f32"] else C.EFM_DTYPE_BF16, ws.data_ptr(), ws.numel(), sh)]
        else:
            y = empty(n, case["inter"])
            ws = buf(lib.efm_fused_gate_up_swiglu_fp4_workspace_bytes(n, k, case["inter"]))
            calls = [("efm_fused_gate_up_swiglu_fp4", n, k, case["inter"], state["x"].data_ptr(), packed.data_ptr(),
                      y.data_ptr(), ws.data_ptr(), ws.numel(), sh)]
        torch.cuda.synchronize()
        del state["codes"], state["scales"]
        state.update(C=C, calls=calls, out=dict(y=y), keep=(packed, ws))
        return
    _, hq, hkv, hd, _, sections = MODELS[case["model"]]
    if kind == "write":
        n, base = case["rows"], case["base"]
        room, width = _rows(base + n), (hq + 2 * hkv) * hd
        q, k, v = empty(n, hq, hd), empty(n, hkv, hd), empty(n, hkv, hd)
        ctx = C.make_attention_ctx(hq, hkv, hd, rope_theta=THETA)
        norms = [state[w].data_ptr() if case["norm"] else None for w in ("qw", "kw")]
        place = (base, None) if n > 1 else (0, torch.tensor([base + 1], dtype=torch.int32, device="cuda"))
        at = (n, place[0], place[1] if place[1] is None else place[1].data_ptr())
        pos = (state["pos"].data_ptr(), n, *sections) if case["mrope"] else (None, 0, 0, 0, 0)
        head = (ctx, state["qkv"].data_ptr(), width, *norms, EPS, q.data_ptr())
        if case["cache"] == "bf16":
            cache = empty(2, room, hkv, hd)
            calls = [("efm_qk_norm_rope_write_kv", *head, cache[0].data_ptr(), cache[1].data_ptr(), room, *at, *pos, sh)]
            k, v = cache[0, base:base + n], cache[1, base:base + n]
        else:
            cache = buf(lib.efm_kv_fp4_bytes(ctx, room))
            calls = [("efm_qk_norm_rope_write_kv_fp4", *head, cache.data_ptr(), room, *at, *pos, sh),
                     ("efm_kv_fp4_read", ctx, cache.data_ptr(), room, base, n, k.data_ptr(), v.data_ptr(), sh)]
        state.update(C=C, calls=calls, out=dict(q=q, k=k, v=v), keep=(ctx, cache, place))
        return
    n, kv = t["q"].shape[0], state["kv"]
    room = _rows(kv)
    ctx = C.make_attention_ctx(hq, hkv, hd, rope=False)
    cache, o = buf(lib.efm_kv_fp4_bytes(ctx, room)), empty(n, hq * hd)
    rows = torch.cat([empty(kv, hq * hd), t["k"].flatten(1), t["v"].flatten(1)], 1)
    C.call("efm_qk_norm_rope_write_kv_fp4", ctx, rows.data_ptr(), rows.shape[1], None, None, 0.0, None, cache.data_ptr(),
           room, kv, 0, None, None, 0, 0, 0, 0, sh)
    if kind == "decode":
        d_len = torch.tensor([kv], dtype=torch.int32, device="cuda")
        ws = buf(lib.efm_attention_decode_kv_fp4_workspace_bytes(ctx, room))
        calls = [("efm_attention_decode_kv_fp4", ctx, state["q"].data_ptr(), cache.data_ptr(), room, o.data_ptr(), 0,
                  d_len.data_ptr(), room, ws.data_ptr(), ws.numel(), sh)]
    else:
        d_len, ws = None, buf(lib.efm_attention_prefill_kv_fp4_workspace_bytes(ctx, n, kv))
        calls = [("efm_attention_prefill_kv_fp4", ctx, state["q"].data_ptr(), cache.data_ptr(), room, o.data_ptr(), n, kv, 1,
                  ws.data_ptr(), ws.numel(), sh)]
    torch.cuda.synchronize()
    state.update(C=C, calls=calls, out=dict(o=o), keep=(ctx, cache, d_len, ws))


def _plain_rotate(x, pos, sections):
    """Rotate-half of x [rows, heads, hd] at int positions pos [rows] (or [3, rows]: one row for each section)."""
    half = x.shape[-1] // 2
    freq = THETA ** (-torch.arange(half, device=x.device, dtype=torch.float64) / half)
    if sections is None:
        ang = pos.double()[:, None] * freq
    else:
        ang = torch.repeat_interleave(pos.double(), torch.tensor(sections, device=x.device), 0).T * freq
    cos, sin = ang.cos().unsqueeze(1), ang.sin().unsqueeze(1)
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_write(s):
    case = s["case"]
    _, hq, hkv, hd, _, sections = MODELS[case["model"]]
    n = case["rows"]
    q, k, v = s["qkv"].double().view(n, hq + 2 * hkv, hd).split([hq, hkv, hkv], 1)
    if case["norm"]:
        q = q / torch.sqrt(q.square().mean(-1, keepdim=True) + EPS) * s["qw"].double()
        k = k / torch.sqrt(k.square().mean(-1, keepdim=True) + EPS) * s["kw"].double()
    if case["mrope"]:
        q, k = _plain_rotate(q, s["pos"], sections), _plain_rotate(k, s["pos"], sections)
    else:
        pos = torch.arange(case["base"], case["base"] + n, device=q.device)
        q, k = _plain_rotate(q, pos, None), _plain_rotate(k, pos, None)
    if case["cache"] == "fp4":
        kc, vc = _codes(k), _codes(v)
        k, v = _values(_halves(kc[0]), kc[1]), _values(_halves(vc[0]), vc[1])
    return dict(q=q.bfloat16(), k=k.bfloat16(), v=v.bfloat16())


def _plain_attention(s):
    n, hq, hd = s["q"].shape
    k, v = _values(*s["k"]), _values(*s["v"])
    kv, hkv, _ = k.shape
    group = hq // hkv
    q = s["q"].float().view(n, hkv, group, hd).permute(1, 2, 0, 3).reshape(hkv, group * n, hd)
    scores = torch.bmm(q, k.permute(1, 2, 0).contiguous()).view(hkv, group, n, kv) / math.sqrt(hd)
    row = torch.arange(n, device=q.device)[:, None] + (kv - n)
    scores.masked_fill_(torch.arange(kv, device=q.device) > row, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p /= p.sum(-1, keepdim=True)
    o = torch.bmm(p.view(hkv, group * n, kv), v.permute(1, 0, 2).contiguous())
    return dict(o=o.view(hq, n, hd).permute(1, 0, 2).reshape(n, hq * hd).bfloat16())


def _plain_linear(s):
    case = s["case"]
    y = s["x"].float() @ _values(s["codes"], s["scales"]).T
    if case["kind"] == "swiglu":   # the products are rounded to 16 bits before the activation
        up, gate = y.bfloat16().float().chunk(2, -1)
        return dict(y=(gate / (1 + torch.exp(-gate)) * up).bfloat16())
    if case["bias"]:
        y = y + s["bias"].float()
    return dict(y=y if case["f32"] else y.bfloat16())


def run(state):
    if own:
        call = state["C"].call
        for args in state["calls"]:
            call(*args)
        return state["out"]
    kind = state["case"]["kind"]
    if kind in ("linear", "swiglu"):
        return _plain_linear(state)
    return _plain_write(state) if kind == "write" else _plain_attention(state)


def _pairs(case):
    n, base = case.get("rows", 1), case.get("prefix", 0)
    return case["context"] if case["kind"] == "decode" else n * base + n * (n + 1) // 2


def work(case):
    kind, n = case["kind"], case.get("rows", 1)
    if kind == "linear":
        k, out = case["inp"], case["out"]
        return dict(bytes=out * k * 17 / 32 + 2 * n * k + (4 if case["f32"] else 2) * n * out, flops=2 * n * k * out)
    if kind == "swiglu":
        k, out = case["hidden"], 2 * case["inter"]
        return dict(bytes=out * k * 17 / 32 + 2 * n * k + n * out, flops=2 * n * k * out)
    _, hq, hkv, hd, _, _ = MODELS[case["model"]]
    if kind == "write":
        rows = 2 * hkv * hd
        # an FP4 cache's rows are written, and read back into the bf16 values that are returned
        cached = 2 * rows if case["cache"] == "bf16" else rows * (2 * 17 / 32 + 2)
        return dict(bytes=n * (2 * (2 * hq + 2 * hkv) * hd + cached), flops=n * 10 * (hq + hkv) * hd)
    kv = case["context"] if kind == "decode" else n + case["prefix"]
    return dict(bytes=2 * kv * hkv * hd * 17 / 32 + 4 * n * hq * hd, flops=4 * hq * hd * _pairs(case))


# The passes in 64 bits, from the operators' definitions.

def _fp4_64(x):
    """Values of x [..., 32 g] after FP4 quantisation: the scale is the least power of two with max |x| <= 7 * scale (at
    least 2^-125), an element the nearest multiple on the grid, of two as near the one with the even code."""
    g = x.reshape(*x.shape[:-1], -1, 32)
    top = g.abs().max(-1, keepdim=True).values
    e = torch.ceil(torch.log2(torch.where(top > 0, top / 7, torch.ones_like(top))))
    e = e - (top <= 7 * torch.exp2(e - 1)).double() + (top > 7 * torch.exp2(e)).double()
    e = torch.where(top > 0, e, torch.full_like(e, -125)).clamp(min=-125)
    scale = torch.exp2(e)
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    borders = (grid[1:] + grid[:-1]) / 2
    a = g.abs() / scale
    low, high = torch.bucketize(a, borders), torch.bucketize(a, borders, right=True)
    code = torch.where(low % 2 == 0, low, high)   # they differ on a border alone
    return (torch.sign(g) * grid[code] * scale).reshape(x.shape)


def _weights64(t):
    low, high = t["codes"].long() % 16, t["codes"].long() // 16
    code = torch.empty(low.shape[0], 2 * low.shape[1], dtype=torch.int64, device=low.device)
    code[:, 0::2], code[:, 1::2] = low, high
    grid = torch.tensor(GRID, dtype=torch.float64, device=low.device)
    w = grid[code % 8] * (1 - 2 * (code // 8)).double()
    return w * torch.exp2(t["scales"].double() - 127).repeat_interleave(32, 1)


def _turned64(x, ang):
    """Each pair (d, d + hd / 2) of x [rows, heads, hd] as a complex number, turned by ang [rows, hd / 2]."""
    half = x.shape[-1] // 2
    z = torch.complex(x[..., :half], x[..., half:]) * torch.polar(torch.ones_like(ang), ang)[:, None]
    return torch.cat([z.real, z.imag], -1)


def exact(case, seed):
    kind = case["kind"]
    if kind in ("linear", "swiglu"):
        t = _linear_inputs(case, seed)
        x = t["x"].double()
        y = torch.cat([x @ _weights64(dict(codes=c, scales=s)).T
                       for c, s in zip(t["codes"].split(4096), t["scales"].split(4096))], 1)
        if kind == "swiglu":
            up, gate = y[:, :case["inter"]], y[:, case["inter"]:]
            return dict(y=gate * torch.sigmoid(gate) * up)
        return dict(y=y + t["bias"].double() if case["bias"] else y)
    _, hq, hkv, hd, _, sections = MODELS[case["model"]]
    if kind == "write":
        t, n = _write_inputs(case, seed), case["rows"]
        x = t["qkv"].double().reshape(n, -1, hd)
        q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
        if case["norm"]:
            q = q * torch.rsqrt((q * q).sum(-1, keepdim=True) / hd + EPS) * t["qw"].double()
            k = k * torch.rsqrt((k * k).sum(-1, keepdim=True) / hd + EPS) * t["kw"].double()
        half = hd // 2
        pos = torch.arange(n, device=x.device)[:, None].expand(n, half) + case["base"]
        if case["mrope"]:
            pos = torch.cat([t["pos"][i][:, None].expand(n, s) for i, s in enumerate(sections)], 1)
        ang = pos.double() * torch.exp(-math.log(THETA) * torch.arange(half, device=x.device, dtype=torch.float64) / half)
        q, k = _turned64(q, ang), _turned64(k, ang)
        return dict(q=q, k=_fp4_64(k), v=_fp4_64(v)) if case["cache"] == "fp4" else dict(q=q, k=k, v=v)
    t = _attention_inputs(case, seed)
    q, k, v = t["q"].double(), _fp4_64(t["k"].double()), _fp4_64(t["v"].double())
    n, kv = q.shape[0], k.shape[0]
    hidden = torch.ones(n, kv, dtype=torch.bool, device=q.device).triu(kv - n + 1)
    heads = []
    for h in range(hq):
        s = (q[:, h] @ k[:, h * hkv // hq].T.contiguous() / hd ** 0.5).masked_fill(hidden, -math.inf)
        heads.append(torch.softmax(s, -1) @ v[:, h * hkv // hq])
    return dict(o=torch.stack(heads, 1).flatten(1))
