"""The 4-bit KV cache's operators and the per-head norms with rotation, as cases that can be timed and checked.

Four operators of the C ABI (include/am_gfx950.h):

  qk_norm_rope   per-head RMSNorm of queries and keys with the rotation in the same pass
  kv_append      a padded batch of sequences: (norm,) rotation and the cache write in one launch, the cache in
                 the activation type or in 4 bits, in planes or in blocks
  kv4_read       rows of a 4-bit cache back as values
  kv4_attention  causal grouped-query attention over a 4-bit cache

A 4-bit row holds E2M1 codes (low nibble = even dimension) and one E8M0 scale for each 32 dimensions:
value = code * 2^(scale - 127), scale 255 = NaN.  The scale is the smallest with max|x| < 7 * 2^e (e at most 125),
a code the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the even code).
"""

import math

import torch

own = False

THETA = 500000.0
EPS = 1e-5
# Head layouts: the 8B shape of the benchmark, the 2048-wide one of the tests, the tiny configuration's.
SHAPES = {"8b": (32, 8, 128), "2k": (16, 4, 128), "tiny": (8, 2, 64)}
TICKET_BYTES = 1 << 14  # attention workspace: tickets, then records of at most 4096 slots
WORKSPACE = 1 << 26


def listed():
    return [
        # One token of one sequence, the step where launch latency is all there is.
        {"name": "qk_norm_rope_1", "kind": "norm", "shape": "8b", "dtype": "bf16", "rows": 1, "norm": True},
        # A long prefill chunk; q and k are views into the rows of one q|k|v product.
        {"name": "qk_norm_rope_2048", "kind": "norm", "shape": "8b", "dtype": "bf16", "rows": 2048, "norm": True},
        # An odd number of fp32 rows of 64-wide heads.
        {"name": "qk_norm_rope_f32_777", "kind": "norm", "shape": "tiny", "dtype": "f32", "rows": 777, "norm": True},
        # A decode step of the widest batch: one token of each sequence into a paged bf16 cache.
        {"name": "append_bf16_b16", "kind": "append", "shape": "8b", "dtype": "bf16", "fmt": "plain", "batch": 16, "seq": 1,
         "start": 777, "block": 64, "norm": False, "ragged": False},
        # The same step into a paged 4-bit cache, with the norms, and the written rows read back.
        {"name": "append_kv4_b16", "kind": "append", "shape": "8b", "dtype": "bf16", "fmt": "kv4", "batch": 16, "seq": 1,
         "start": 777, "block": 64, "norm": True, "ragged": False},
        # The last 2048-token chunk of an 8192-token prompt into a contiguous 4-bit cache.
        {"name": "append_kv4_2048", "kind": "append", "shape": "8b", "dtype": "bf16", "fmt": "kv4", "batch": 1, "seq": 2048,
         "start": 6144, "block": 0, "norm": False, "ragged": False},
        # A short prefix of a paged sequence taken out of the 4-bit cache.
        {"name": "read_kv4_37", "kind": "read", "shape": "8b", "dtype": "bf16", "batch": 1, "seq": 37, "start": 600, "block": 64},
        # Four 8k sequences taken out whole.
        {"name": "read_kv4_b4_8k", "kind": "read", "shape": "8b", "dtype": "bf16", "batch": 4, "seq": 8192, "start": 0, "block": 0},
        # One token over a short context: single-sequence decode.
        {"name": "attention_b1_640", "kind": "attention", "shape": "8b", "dtype": "bf16", "batch": 1, "seq": 1, "start": 639,
         "block": 0, "ragged": False},
        # The widest batch over contexts of several lengths, paged.
        {"name": "attention_b16_8k", "kind": "attention", "shape": "8b", "dtype": "bf16", "batch": 16, "seq": 1, "start": 8319,
         "block": 64, "ragged": False},
        # One token over a very long context.
        {"name": "attention_b1_131072", "kind": "attention", "shape": "8b", "dtype": "bf16", "batch": 1, "seq": 1,
         "start": 131071, "block": 0, "ragged": False},
        # The last 2048-token chunk of an 8192-token prompt.
        {"name": "attention_2048_at_6144", "kind": "attention", "shape": "8b", "dtype": "bf16", "batch": 1, "seq": 2048,
         "start": 6144, "block": 0, "ragged": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    shape, dtype = rng.choice(["8b", "8b", "2k", "tiny"]), rng.choice(["bf16", "bf16", "bf16", "f32"])
    block = rng.choice([0, 32, 64, 256])
    what = rng.random()
    if what < 0.2:
        return {"kind": "norm", "shape": shape, "dtype": dtype, "rows": _log_int(rng, 1, 2048), "norm": rng.random() < 0.8}
    batch = _log_int(rng, 1, 16)
    if what < 0.45:
        return {"kind": "append", "shape": shape, "dtype": dtype, "fmt": rng.choice(["plain", "kv4", "kv4"]), "batch": batch,
                "seq": rng.choice([1, _log_int(rng, 2, max(2, 2048 // batch))]), "start": rng.randrange(0, 4096), "block": block,
                "norm": rng.random() < 0.5, "ragged": rng.random() < 0.5}
    if what < 0.55:
        return {"kind": "read", "shape": shape, "dtype": dtype, "batch": batch, "seq": _log_int(rng, 1, 8192 // batch),
                "start": rng.randrange(0, 1024), "block": block}
    if what < 0.8:
        return {"kind": "attention", "shape": shape, "dtype": dtype, "batch": batch, "seq": 1,
                "start": _log_int(rng, 1, 131072 // batch) - 1, "block": block, "ragged": False}
    seq = _log_int(rng, 2, max(2, 1024 // batch))
    return {"kind": "attention", "shape": shape, "dtype": dtype, "batch": batch, "seq": seq,
            "start": rng.choice([0, rng.randrange(0, max(1, 6144 // batch))]), "block": block, "ragged": rng.random() < 0.5}


# ------------------------------------------------------------------ the case's sizes
def _starts(case):
    """First position of each sequence: from start down to about half of it."""
    b, s = case["batch"], case["start"]
    return [s - i * (s // (2 * b)) for i in range(b)] if case["kind"] != "read" else [s] * b


def _lens(case):
    """Live rows of each sequence of a padded batch."""
    b, s = case["batch"], case["seq"]
    return [s - i * s // (2 * b) for i in range(b)] if case.get("ragged") else [s] * b


def _capacity(case):
    return -(-(case["start"] + case["seq"]) // 256) * 256


def _esz(case):
    return 2 if case["dtype"] == "bf16" else 4


def work(case):
    hq, hkv, d = SHAPES[case["shape"]]
    e, kind = _esz(case), case["kind"]
    row4 = d / 2 + d / 32  # bytes of one 4-bit row
    if kind == "norm":
        n, v = case["rows"], case["rows"] * (hq + hkv) * d
        return {"bytes": 2 * v * e + n * (8 + 4 * d) + (2 * d * e if case["norm"] else 0), "flops": 3 * v + (4 * v if case["norm"] else 0)}
    if kind == "append":
        n = sum(_lens(case))
        q, kv = n * hq * d, 2 * n * hkv * d
        moved = (2 * q + kv) * e + n * 4 * d
        # the rows written; in 4 bits they are also read back as bf16 values
        moved += kv * e if case["fmt"] == "plain" else 2 * n * 2 * hkv * row4 + kv * 2
        return {"bytes": moved, "flops": 3 * (q + kv / 2) + (4 * (q + kv / 2) if case["norm"] else 0)}
    if kind == "read":
        rows = 2 * case["batch"] * case["seq"] * hkv
        return {"bytes": rows * (row4 + 2 * d), "flops": rows * d}
    starts, lens = _starts(case), _lens(case)
    keys = sum(s + n for s, n in zip(starts, lens))
    pairs = sum(n * s + n * (n + 1) // 2 for s, n in zip(starts, lens))
    return {"bytes": 2 * keys * hkv * row4 + 2 * sum(lens) * hq * d * e, "flops": 4 * pairs * hq * d}


# ------------------------------------------------------------------ the 4-bit format
def _e2m1(dev, dtype):
    v = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=dev, dtype=dtype)
    return torch.cat([v, -v])


def _e8m0(dev, dtype):
    t = torch.pow(2.0, torch.arange(256, device=dev, dtype=torch.float64) - 127)
    t[255] = math.nan
    return t.to(dtype)


def _encode(x):
    """E2M1 codes [..., d] and E8M0 scales [..., d / 32] (uint8, one code a byte) of fp32 values."""
    g = x.reshape(*x.shape[:-1], -1, 32)
    top = g.abs().amax(-1)
    e = (((top.view(torch.int32) + 0x200000) >> 23) - 2).clamp(0, 252)
    t = (g * torch.pow(2.0, (127 - e).to(torch.float32))[..., None]).abs()
    code = (t > 0.25).to(torch.uint8) + (t >= 0.75) + (t > 1.25) + (t >= 1.75) + (t > 2.5) + (t >= 3.5) + (t > 5)
    code = code + 8 * torch.signbit(g)
    fine = torch.isfinite(g).all(-1)
    return (code * fine[..., None]).reshape(x.shape).to(torch.uint8), torch.where(fine, e, 255).to(torch.uint8)


def _values(code, scale, dtype=torch.float32):
    """The values that codes (one a byte) and scales stand for."""
    v = _e2m1(code.device, dtype)[code.long()].reshape(*scale.shape, 32)
    return (v * _e8m0(code.device, dtype)[scale.long()][..., None]).reshape(code.shape)


def _unpack(packed):
    return torch.stack([packed & 15, packed >> 4], -1).flatten(-2)


def _pack(code):
    return code[..., 0::2] | (code[..., 1::2] << 4)


# ------------------------------------------------------------------ inputs
def _dt(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _tables(n, d):
    inv = THETA ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
    a = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * inv[None, :]
    return a.cos().float(), a.sin().float()


def _blocks(t, block):
    """Pools [blocks][hkv][block][...] and the block table of [batch][hkv][capacity][...], the sequences' blocks
    interleaved as growing sequences take them."""
    b, hkv, cap, w = t.shape
    per = cap // block
    pool = t.view(b, hkv, per, block, w).permute(2, 0, 1, 3, 4).reshape(per * b, hkv, block, w).contiguous()
    table = (torch.arange(per, device="cuda")[None, :] * b + torch.arange(b, device="cuda")[:, None]).to(torch.int32)
    return pool, table.contiguous()


def prepare(case, seed):
    hq, hkv, d = SHAPES[case["shape"]]
    dt, kind = _dt(case), case["kind"]
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    x = {"case": case}
    if kind in ("norm", "append"):
        rows = case["rows"] if kind == "norm" else case["batch"] * case["seq"]
        x["qkv"] = normal(rows, (hq + 2 * hkv) * d).to(dt)  # one product's rows, q then k then v
        x["q_w"], x["k_w"] = ((1 + 0.25 * normal(d)).to(dt) for _ in range(2))
        x["q_out"] = torch.zeros(rows, hq * d, device="cuda", dtype=dt)
    if kind == "norm":
        x["cos"], x["sin"] = _tables(8192, d)
        x["pos"] = torch.arange(case["rows"], device="cuda") + int(torch.randint(0, 6145, (1,), generator=gen, device="cuda"))
        x["k_out"] = torch.zeros(case["rows"], hkv * d, device="cuda", dtype=dt)
        return x
    b, cap, block = case["batch"], _capacity(case), case["block"]
    x["start"] = torch.tensor(_starts(case), device="cuda")
    x["lens"] = torch.tensor(_lens(case), device="cuda", dtype=torch.int32)
    if kind == "append":
        x["cos"], x["sin"] = _tables(cap, d)
    plain = case.get("fmt") == "plain"
    for n in ("k", "v"):
        # some channels are larger than the others, keys' more than values'
        wide = 1 + (3 if n == "k" else 1) * torch.rand(hkv, 1, d, generator=gen, device="cuda") ** 4
        t = normal(b, hkv, cap, d) * wide
        if plain:
            held = {n: t.to(dt)}
        else:
            code, scale = _encode(t)
            held = {n: _pack(code), n + "_scale": scale}
        for m, c in held.items():
            if block:
                c, x["table"] = _blocks(c, block)
            x[m] = c
    if kind == "attention":
        x["q"] = normal(b * case["seq"], hq * d).to(dt)
        x["out"] = torch.zeros(b * case["seq"], hq * d, device="cuda", dtype=dt)
        x["ws"] = torch.zeros(WORKSPACE, device="cuda", dtype=torch.uint8)  # a serving program's, kept over its calls
    elif not plain:
        x["k_out"], x["v_out"] = (torch.zeros(b * case["seq"], hkv * d, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    return x


# ------------------------------------------------------------------ the plain forms
def _plain_rotate(x, w, c, s, wide=False):
    """x [rows][heads][d], norm gain w or None, tables' rows c, s [rows][d / 2]; 64 bits where the result is
    rounded to 4 bits next to a border"""
    x = x.double() if wide else x.float()
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.to(x.dtype)
    a, b = x.chunk(2, -1)
    c, s = c[:, None].to(x.dtype), s[:, None].to(x.dtype)
    return torch.cat([a * c - b * s, b * c + a * s], -1).float()


def _split(x):
    hq, hkv, d = SHAPES[x["case"]["shape"]]
    q, k, v = x["qkv"].split([hq * d, hkv * d, hkv * d], -1)
    return q.unflatten(-1, (hq, d)), k.unflatten(-1, (hkv, d)), v.unflatten(-1, (hkv, d))


def _plain_whole(x, name):
    """[batch][hkv][capacity][...] of a cache held in planes or blocks"""
    t = x[name]
    if not x["case"]["block"]:
        return t
    t = t[x["table"].long()]  # [batch][per][hkv][block][...]
    return t.transpose(1, 2).flatten(2, 3)


def _plain_norm(x):
    q, k, _ = _split(x)
    norm = x["case"]["norm"]
    c, s = x["cos"][x["pos"]], x["sin"][x["pos"]]
    qo = _plain_rotate(q, x["q_w"] if norm else None, c, s)
    ko = _plain_rotate(k, x["k_w"] if norm else None, c, s)
    return {"q": qo.flatten(1).to(x["qkv"].dtype), "k": ko.flatten(1).to(x["qkv"].dtype)}


def _plain_append(x):
    case = x["case"]
    q, k, v = _split(x)
    step = torch.arange(case["seq"], device="cuda")
    pos = (x["start"][:, None] + step).flatten()
    live = (step < x["lens"][:, None]).flatten()
    at = pos.clamp(max=x["cos"].shape[0] - 1)
    c, s = x["cos"][at], x["sin"][at]
    four = case["fmt"] == "kv4"
    qo = _plain_rotate(q, x["q_w"] if case["norm"] else None, c, s)
    ko = _plain_rotate(k, x["k_w"] if case["norm"] else None, c, s, wide=four)
    out = {"q": torch.where(live[:, None], qo.flatten(1), 0).to(x["qkv"].dtype)}
    if four:
        for n, t in (("k", ko), ("v", v.float())):
            out[n] = torch.where(live[:, None], _values(*_encode(t.contiguous())).flatten(1), 0).to(torch.bfloat16)
        return out
    row = live.nonzero()[:, 0]
    seq, p = row // case["seq"], pos[row]
    if case["block"]:
        first, second = x["table"][seq, p // case["block"]].long(), p % case["block"]
    else:
        first, second = seq, p
    for n, t in (("k", ko), ("v", v)):
        x[n][first, :, second] = t[row].to(x[n].dtype)
        out[n] = x[n]
    return out


def _plain_read(x):
    case, out = x["case"], {}
    for n in ("k", "v"):
        code = _unpack(_plain_whole(x, n)[:, :, case["start"]:case["start"] + case["seq"]])
        scale = _plain_whole(x, n + "_scale")[:, :, case["start"]:case["start"] + case["seq"]]
        out[n] = _values(code, scale).transpose(1, 2).flatten(0, 1).flatten(1).to(torch.bfloat16)
    return out


def _plain_attention(x):
    case = x["case"]
    hq, hkv, d = SHAPES[case["shape"]]
    b, n = case["batch"], case["seq"]
    k, v = (_values(_unpack(_plain_whole(x, m)), _plain_whole(x, m + "_scale")) for m in ("k", "v"))
    q = x["q"].float().view(b, n, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) / math.sqrt(d)
    step = torch.arange(n, device="cuda")
    last = (x["start"][:, None] + step).repeat(1, hq // hkv)  # [batch][heads of the group, rows]
    score.masked_fill_(torch.arange(k.shape[2], device="cuda") > last[:, None, :, None], -math.inf)
    score = (score - score.amax(-1, keepdim=True)).exp_()
    out = torch.matmul(score, v) / score.sum(-1, keepdim=True)
    out = out.view(b, hkv, hq // hkv, n, d).permute(0, 3, 1, 2, 4)
    out = torch.where((step < x["lens"][:, None])[:, :, None, None, None], out, 0)
    return {"out": out.reshape(b * n, hq * d).to(x["q"].dtype)}


# ------------------------------------------------------------------ the framework's calls
def _own_calls(x):
    """The argument blocks of a case, filled once over the buffers that the program keeps."""
    import ctypes as C

    import aethermind_amd.native as N

    case = x["case"]
    hq, hkv, d = SHAPES[case["shape"]]
    kind, dt = case["kind"], N.AM_DT_BF16 if case["dtype"] == "bf16" else N.AM_DT_F32
    p = {n: t.data_ptr() for n, t in x.items() if isinstance(t, torch.Tensor)}
    e, width = _esz(case), (hq + 2 * hkv) * d
    if kind in ("norm", "append"):
        q, k, v = p["qkv"], p["qkv"] + hq * d * e, p["qkv"] + (hq + hkv) * d * e
        qw, kw = (p["q_w"], p["k_w"]) if case["norm"] else (None, None)
    if kind == "norm":
        return [("am_gfx950_qk_norm_rope", N.QkNormRopeArgs(q, k, p["q_out"], p["k_out"], case["rows"], hq, hkv, d, width, width,
                                                            hq * d, hkv * d, qw, kw, EPS, p["pos"], p["cos"], p["sin"], 8192, dt))]
    b, n, cap = case["batch"], case["seq"], _capacity(case)
    cbs = hkv * cap * d
    pages = None
    if case["block"]:
        pages = C.pointer(N.KvPages(p["table"], case["block"], x["table"].shape[1], x["k"].shape[0], None))
    lens = p["lens"] if case.get("ragged") else None
    if kind == "read":
        return [("am_gfx950_kv4_read", N.Kv4ReadArgs(p["k"], p["k_scale"], p["v"], p["v_scale"], p["k_out"], p["v_out"], b, n, hkv,
                                                     d, cap, cbs, p["start"], lens, N.AM_DT_BF16, pages))]
    if kind == "append":
        four = case["fmt"] == "kv4"
        calls = [("am_gfx950_kv_append", N.KvAppendArgs(
            q, k, v, p["q_out"], b, n, hq, hkv, d, width, width, width, hq * d, qw, kw, EPS, p["cos"], p["sin"], cap, p["start"],
            lens, p["k"], p["v"], p.get("k_scale"), p.get("v_scale"), cap, cbs, N.AM_KV_MXFP4 if four else N.AM_KV_PLAIN, dt, None,
            pages))]
        if four:
            calls.append(("am_gfx950_kv4_read", N.Kv4ReadArgs(p["k"], p["k_scale"], p["v"], p["v_scale"], p["k_out"], p["v_out"], b,
                                                              n, hkv, d, cap, cbs, p["start"], lens, N.AM_DT_BF16, pages)))
        return calls
    return [("am_gfx950_kv4_attention", N.Kv4AttentionArgs(p["q"], p["out"], p["k"], p["k_scale"], p["v"], p["v_scale"], b, n, hq,
                                                           hkv, d, cap, cbs, p["start"], lens, 0.0, dt, p["ws"], WORKSPACE, pages))]


def _own_run(x):
    import aethermind_amd.native as N

    if "calls" not in x:
        x["calls"] = _own_calls(x)
    lib, stream = N.lib(), torch.cuda.current_stream().cuda_stream
    for name, args in x["calls"]:
        lib.call(name, args, stream)
    case = x["case"]
    if case["kind"] == "norm":
        return {"q": x["q_out"], "k": x["k_out"]}
    if case["kind"] == "append":
        return {"q": x["q_out"], "k": x["k"], "v": x["v"]} if case["fmt"] == "plain" else {"q": x["q_out"], "k": x["k_out"], "v": x["v_out"]}
    return {"k": x["k_out"], "v": x["v_out"]} if case["kind"] == "read" else {"out": x["out"]}


def run(state):
    if own:
        return _own_run(state)
    return {"norm": _plain_norm, "append": _plain_append, "read": _plain_read, "attention": _plain_attention}[state["case"]["kind"]](state)


# ------------------------------------------------------------------ 64 bits, from the definitions
def _exact_heads(rows, gain, cos, sin):
    """Norm and rotation of [rows][heads][d] by complex products."""
    z = rows.double()
    if gain is not None:
        z = z / ((z ** 2).sum(-1, keepdim=True) / z.shape[-1] + EPS).sqrt() * gain.double()
    half = z.shape[-1] // 2
    turn = torch.complex(cos.double(), sin.double())[:, None, :]
    z = torch.complex(z[..., :half], z[..., half:]) * turn
    return torch.cat([z.real, z.imag], -1)


def _exact_four(t):
    """The values that the 4-bit rows of `t` stand for: nearest of the grid at the group's scale."""
    g = t.float().double().reshape(-1, 32)
    top = g.abs().amax(1)
    e = torch.where(top > 0, torch.floor(torch.log2(top / 7)) + 1, -127.0)
    e = torch.where(top >= 7 * torch.exp2(e), e + 1, e)
    e = torch.where(top < 7 * torch.exp2(e - 1), e - 1, e).clamp(-127, 125)
    unit = g / torch.exp2(e)[:, None]
    grid = _e2m1(t.device, torch.float64)[:8]
    far = (unit.abs()[..., None] - grid).abs()
    near = far.amin(-1, keepdim=True)
    # ties to the even code
    order = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7], device=t.device)
    pick = order[(far == near)[..., order].to(torch.uint8).argmax(-1)]
    return (grid[pick] * torch.sign(unit) * torch.exp2(e)[:, None]).reshape(t.shape)


def _exact_cache(x, name, b):
    """[hkv][capacity][d] of sequence b, 64 bits, block after block"""
    case = x["case"]
    if case["block"]:
        ids = x["table"][b].tolist()
        code = torch.cat([x[name][i] for i in ids], 1)
        scale = torch.cat([x[name + "_scale"][i] for i in ids], 1)
    else:
        code, scale = x[name][b], x[name + "_scale"][b]
    lo, hi = code.int() % 16, code.int() // 16
    nib = torch.empty(*code.shape[:-1], 2 * code.shape[-1], dtype=torch.int32, device=code.device)
    nib[..., 0::2], nib[..., 1::2] = lo, hi
    mag = _e2m1(code.device, torch.float64)[(nib % 8).long()]
    return mag * torch.where(nib >= 8, -1.0, 1.0) * torch.exp2(scale.double() - 127).repeat_interleave(32, -1)


def exact(case, seed):
    x = prepare(case, seed)
    hq, hkv, d = SHAPES[case["shape"]]
    kind = case["kind"]
    if kind == "norm":
        q, k, _ = _split(x)
        c, s = x["cos"].index_select(0, x["pos"]), x["sin"].index_select(0, x["pos"])
        gains = (x["q_w"], x["k_w"]) if case["norm"] else (None, None)
        return {"q": _exact_heads(q, gains[0], c, s).flatten(1), "k": _exact_heads(k, gains[1], c, s).flatten(1)}
    starts, lens, n = _starts(case), _lens(case), case["seq"]
    if kind == "append":
        q, k, v = _split(x)
        gains = (x["q_w"], x["k_w"]) if case["norm"] else (None, None)
        four = case["fmt"] == "kv4"
        qo = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
        ko, vo = (torch.zeros(k.shape, dtype=torch.float64, device="cuda") for _ in range(2))
        held = {} if four else {m: x[m].double() for m in ("k", "v")}
        for b, (p0, m) in enumerate(zip(starts, lens)):
            r = slice(b * n, b * n + m)
            c, s = x["cos"][p0:p0 + m], x["sin"][p0:p0 + m]
            qo[r] = _exact_heads(q[r], gains[0], c, s)
            ko[r] = _exact_heads(k[r], gains[1], c, s)
            vo[r] = v[r].double()
            if four:
                ko[r], vo[r] = _exact_four(ko[r]), _exact_four(vo[r])
                continue
            for i in range(m):
                p = p0 + i
                at = (int(x["table"][b, p // case["block"]]), slice(None), p % case["block"]) if case["block"] else (b, slice(None), p)
                held["k"][at], held["v"][at] = ko[b * n + i], vo[b * n + i]
        return {"q": qo.flatten(1), **({"k": ko.flatten(1), "v": vo.flatten(1)} if four else held)}
    if kind == "read":
        p0 = case["start"]
        return {m: torch.cat([_exact_cache(x, m, b)[:, p0:p0 + n].transpose(0, 1).flatten(1) for b in range(case["batch"])])
                for m in ("k", "v")}
    out = torch.zeros(case["batch"], n, hq, d, dtype=torch.float64, device="cuda")
    q = x["q"].double().view(case["batch"], n, hq, d)
    for b, (p0, m) in enumerate(zip(starts, lens)):
        k, v = _exact_cache(x, "k", b)[:, :p0 + m], _exact_cache(x, "v", b)[:, :p0 + m]
        after = torch.arange(p0 + m, device="cuda") > (p0 + torch.arange(m, device="cuda"))[:, None]
        for h in range(hq):
            s = q[b, :m, h] @ k[h // (hq // hkv)].t() * d ** -0.5
            out[b, :m, h] = torch.softmax(s.masked_fill(after, -math.inf), -1) @ v[h // (hq // hkv)]
    return {"out": out.reshape(-1, hq * d)}
