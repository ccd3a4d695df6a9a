"""The 4-bit KV cache (am_gfx950_kv_append, am_gfx950_kv4_read, am_gfx950_kv4_attention) and the per-head norms with
rotation (am_gfx950_qk_norm_rope) against plain 64-bit forms (kv4_ref.py): formats, odd sizes, strides, pages, padded
batches, rows without keys, NaN in and behind the keys, split contexts, graphs, and a decode loop of all of them.

Codes and scales are compared exactly; bounds of the computed outputs are derived in kv4_ref.py and beside the tests."""

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a GPU", allow_module_level=True)

import ctypes as C  # noqa: E402

import aethermind_amd.native as N  # noqa: E402
import kv4_ref as R  # noqa: E402
from kv4_ref import DTYPES, HALF, Cache, i32, i64  # noqa: E402

L = N.lib()


def randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def gen_of(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ------------------------------------------------------------------ qk_norm_rope
def norm_rope(q, k, qo, ko, rows, hq, hkv, d, pos, cos, sin, qw=None, kw=None, eps=1e-5, dtype="bf16"):
    pt = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    st = lambda t: 0 if t is None else t.stride(0)  # noqa: E731
    a = N.QkNormRopeArgs(pt(q), pt(k), pt(qo), pt(ko), rows, hq, hkv, d, st(q), st(k), st(qo), st(ko), pt(qw), pt(kw), eps,
                         pos.data_ptr(), cos.data_ptr(), sin.data_ptr(), cos.shape[0], DTYPES[dtype][1])
    L.call("am_gfx950_qk_norm_rope", a, R.stream())


def check_rows(got, x, w, eps, cos, sin, pos, dtype, what):
    """Bound: the rounding of the result, and fp32 work on the pair (y1, y2): a sum of squares of at most 20 roundings a
    term, a root, a quotient, two products and three roundings of the rotation, below 32 * 2^-24 of the pair's length."""
    ok = (pos >= 0) & (pos < cos.shape[0])
    at = pos.clamp(0, cos.shape[0] - 1)
    y = R.norm(x, w, eps)
    want = R.rotate(y, cos[at], sin[at], ok)
    a, b = y.chunk(2, -1)
    length = (a.square() + b.square()).sqrt().repeat(1, 1, 2)
    tol = HALF[dtype] * want.abs() * 1.001 + 2.0**-19 * length + 1e-37
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} values off, first at {bad.nonzero()[0].tolist()}"


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [2, 10, 64, 80, 128, 256, 1024])
@pytest.mark.parametrize("rows,hq,hkv", [(1, 32, 8), (37, 5, 3), (300, 8, 1)])
@pytest.mark.parametrize("gains", [True, False])
def test_qk_norm_rope(dtype, d, rows, hq, hkv, gains):
    g, dt = gen_of(d + rows), DTYPES[dtype][0]
    qkv = (randn(g, rows, (hq + 2 * hkv) * d) * 3).to(dt)
    q, k = qkv[:, : hq * d], qkv[:, hq * d : (hq + hkv) * d]
    w = [(1 + randn(g, d) / 4).to(dt) for _ in range(2)] if gains else [None, None]
    cos, sin = R.tables(512, d)
    pos = torch.randint(0, 512, (rows,), generator=g, device="cuda")
    if rows > 2:
        pos[1], pos[2] = -1, 512  # outside: normed, not rotated
    qo, ko = torch.empty(rows, hq * d, dtype=dt, device="cuda"), torch.empty(rows, hkv * d, dtype=dt, device="cuda")
    norm_rope(q, k, qo, ko, rows, hq, hkv, d, pos, cos, sin, *w, dtype=dtype)
    check_rows(qo.view(rows, hq, d), q.reshape(rows, hq, d), w[0], 1e-5, cos, sin, pos, dtype, "q")
    check_rows(ko.view(rows, hkv, d), k.reshape(rows, hkv, d), w[1], 1e-5, cos, sin, pos, dtype, "k")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128, 48])
def test_qk_norm_rope_without_gains_is_rope(dtype, d):
    g, dt, rows, hq, hkv = gen_of(d), DTYPES[dtype][0], 61, 6, 2
    q, k = randn(g, rows, hq * d).to(dt), randn(g, rows, hkv * d).to(dt)
    cos, sin = R.tables(4096, d)
    pos = torch.randint(0, 4096, (rows,), generator=g, device="cuda")
    qo, ko, q1, k1 = (torch.empty_like(t) for t in (q, k, q, k))
    norm_rope(q, k, qo, ko, rows, hq, hkv, d, pos, cos, sin, dtype=dtype)
    L.call("am_gfx950_rope", N.RopeArgs(q.data_ptr(), k.data_ptr(), q1.data_ptr(), k1.data_ptr(), pos.data_ptr(), cos.data_ptr(),
                                        sin.data_ptr(), rows, hq, hkv, d, 4096, DTYPES[dtype][1]), R.stream())
    assert torch.equal(qo, q1) and torch.equal(ko, k1)


@pytest.mark.parametrize("d", [64, 128, 80])
@pytest.mark.parametrize("off", [0, 1, 3])
def test_qk_norm_rope_in_place_and_unaligned(d, off):
    """in place on views whose first element and stride are not vector-aligned; one of q and k alone"""
    g, rows, hq, hkv = gen_of(off), 19, 4, 2
    width = (hq + hkv) * d + 2 * off + (off > 0)
    buf = randn(g, rows, width).to(torch.bfloat16)
    before = buf.clone()
    q, k = buf[:, off : off + hq * d], buf[:, off + hq * d : off + (hq + hkv) * d]
    w = (1 + randn(g, d + 1) / 4).to(torch.bfloat16)[off % 2 :][:d]
    cos, sin = R.tables(128, d)
    pos = torch.arange(rows, device="cuda") * 5
    want = torch.empty(rows, hq * d, dtype=torch.bfloat16, device="cuda"), torch.empty(rows, hkv * d, dtype=torch.bfloat16, device="cuda")
    norm_rope(q, None, want[0], None, rows, hq, 0, d, pos, cos, sin, w, None)
    norm_rope(None, k, None, want[1], rows, 0, hkv, d, pos, cos, sin, None, w)
    assert torch.equal(buf, before)
    check_rows(want[0].view(rows, hq, d), q.reshape(rows, hq, d), w, 1e-5, cos, sin, pos, "bf16", "q")
    norm_rope(q, k, q, k, rows, hq, hkv, d, pos, cos, sin, w, w)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(buf[:, :off], before[:, :off]) and torch.equal(buf[:, off + (hq + hkv) * d :], before[:, off + (hq + hkv) * d :])


def test_qk_norm_rope_large_and_small_values():
    """squares that pass fp32 are infinite (zeros out, as the formula in fp32); tiny rows keep eps"""
    d, rows = 128, 4
    x = torch.ones(rows, d, device="cuda")
    x[0] *= 1e-30
    x[1] *= 1e18
    x[2, 5] = float("nan")
    x[3, 7] = float("inf")
    cos, sin = R.tables(8, d)
    out = torch.empty_like(x)
    w = torch.ones(d, device="cuda")
    norm_rope(x, None, out, None, rows, 1, 0, d, i64(0, 0, 0, 0), cos, sin, w, None, dtype="f32")
    assert torch.allclose(out[0], x[0] / (1e-5**0.5), rtol=1e-5, atol=0)
    assert torch.allclose(out[1], torch.ones_like(out[1]), rtol=1e-5, atol=0)
    assert torch.isnan(out[2]).all() and torch.isnan(out[3, [7, 7 + 64]]).any()


# ------------------------------------------------------------------ the format
def test_read_every_code_and_scale():
    d, cap = 128, 256  # row = scale, all byte values in two rows of 64 + ... bytes
    for first in range(0, 256, 64):
        c = Cache(1, 1, cap, d)
        codes = torch.arange(first, first + 64, device="cuda").to(torch.uint8).expand(cap, 64)
        scale = torch.arange(256, device="cuda").to(torch.uint8)[:, None].expand(cap, 4)
        for n in ("k", "v"):
            c.put(n, codes[None, None])
            c.put(n + "s", scale[None, None])
        want = c.values("k")[0, 0]
        for dtype in ("bf16", "f32"):
            for got in R.read(c, 1, cap, i64(0), dtype=dtype):
                got = got.double()
                assert torch.equal(torch.isnan(got), torch.isnan(want))
                assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))


SPECIAL = [0.0, -0.0, 1.0, -1.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 6.96875, 7.0, 7.25, -7.0, -2.5, 1e-3, 2.0**-126,
           2.0**-133, 2.0**-130, 3e38, -3.3e38, 2.0**127, 1e-20, 100.0, 0.2499, 0.251]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128])
def test_append_encodes_special_groups(dtype, d):
    """groups whose largest value sits on and beside the rule's border, ties, subnormals, the ends of the range, a NaN or an
    infinity in one place"""
    dt = DTYPES[dtype][0]
    g = gen_of(5)
    groups = []
    for top in SPECIAL:
        for spread in (1.0, 0.4, 1.0 / 6, 1e-3):
            t = randn(g, 32).clamp(-1, 1) * abs(top) * spread
            t[11] = top
            groups.append(t)
    steps = torch.tensor(sorted(set(R.GRID + [(a + b) / 2 for a, b in zip(R.GRID, R.GRID[1:])])), device="cuda")
    for e in (-126, -3, 0, 7, 120):  # every grid value and every tie, with the top that sets the scale
        t = torch.zeros(32, device="cuda")
        t[: len(steps)] = steps
        t[16 : 16 + len(steps)] = -steps
        groups.append(t * 2.0**e)
    for bad in (float("nan"), float("inf"), -float("inf")):
        t = randn(g, 32)
        t[31] = bad
        groups.append(t)
    n = -(-len(groups) * 32 // d)
    x = torch.zeros(n * d, device="cuda")
    x[: len(groups) * 32] = torch.cat(groups)
    x = x.view(n, d).to(dt)
    c = Cache(1, 1, -(-n // 32) * 32, d)
    cos, sin = torch.ones(c.cap, d // 2, device="cuda"), torch.zeros(c.cap, d // 2, device="cuda")
    R.append(c, None, x, x, None, 1, n, 0, i64(0), cos=cos, sin=sin, dtype=dtype)
    code, scale = R.encode(x)
    assert torch.equal(c.whole("vs")[0, 0, :n], scale)
    assert torch.equal(c.whole("v")[0, 0, :n], R.pack(code))
    # keys pass the rotation by 0 (x * 1 - y * 0): the same where the pair is finite, signs of zeros aside
    both = torch.isfinite(x).all(-1)
    assert torch.equal(c.whole("ks")[0, 0, :n][both], scale[both])
    assert torch.equal(c.values("k")[0, 0, :n][both], c.values("v")[0, 0, :n][both])


# ------------------------------------------------------------------ kv_append
def append_reference(c, qkv, hq, start, lens, n, cos, sin, qw, kw):
    """(q rows in 64 bits, code and scale planes after the append, rows written) of a 4-bit append"""
    hkv, d, b = c.hkv, c.d, c.b
    q, k, v = qkv.split([hq * d, hkv * d, hkv * d], -1)
    pos = torch.tensor([start[i] + s for i in range(b) for s in range(n)], device="cuda")
    live = torch.tensor([s < lens[i] for i in range(b) for s in range(n)], device="cuda")
    ok = (pos >= 0) & (pos < c.cap)
    at = pos.clamp(0, cos.shape[0] - 1)
    qy = R.norm(q.reshape(-1, hq, d), qw, 1e-5) if hq else None
    k_rot = R.rotate(R.norm(k.reshape(-1, hkv, d), kw, 1e-5), cos[at], sin[at], ok).float()
    planes = {m: c.whole(m) for m in ("k", "ks", "v", "vs")}
    for m, t in (("k", k_rot), ("v", v.reshape(-1, hkv, d).float())):
        code, scale = R.encode(t)
        for r in (live & ok).nonzero()[:, 0].tolist():
            planes[m][r // n, :, pos[r]] = R.pack(code[r])
            planes[m + "s"][r // n, :, pos[r]] = scale[r]
    return qy, planes, pos, live, ok


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d,hq,hkv", [(128, 32, 8), (64, 6, 3), (128, 1, 1), (64, 0, 2)])
@pytest.mark.parametrize("block", [0, 32, 64])
@pytest.mark.parametrize("b,n,start,lens", [(1, 1, [0], None), (3, 1, [95, 0, 40], None), (2, 37, [10, 50], [37, 20]),
                                            (4, 5, [94, -3, 2, 96], [5, 5, 0, 5])])
@pytest.mark.parametrize("gains", [True, False])
def test_append_kv4(dtype, d, hq, hkv, block, b, n, start, lens, gains):
    g, dt, cap = gen_of(b * 100 + n + d), DTYPES[dtype][0], 96
    qkv = randn(g, b * n, (hq + 2 * hkv) * d).to(dt)
    qw, kw = [(1 + randn(g, d) / 4).to(dt) for _ in range(2)] if gains else (None, None)
    cos, sin = R.tables(cap, d)
    c = Cache(b, hkv, cap, d, block, seed=b)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    live_rows = lens or [n] * b
    qy, want, pos, live, ok = append_reference(c, qkv, hq, start, live_rows, n, cos, sin, qw, kw)
    q = qkv[:, : hq * d] if hq else None
    q_out = torch.full((b * n, hq * d), -7.0, dtype=dt, device="cuda") if hq else None
    before = {m: t.clone() for m, t in c.t.items()}
    R.append(c, q, qkv[:, hq * d : (hq + hkv) * d], qkv[:, (hq + hkv) * d :], q_out, b, n, hq, i64(*start),
             i32(*lens) if lens else None, qw, kw, cos=cos, sin=sin, err=err, dtype=dtype)
    for m in want:
        assert torch.equal(c.whole(m), want[m]), m
    if block:  # blocks that belong to no sequence
        used = set(c.table.flatten().tolist())
        for m, t in c.t.items():
            assert all(torch.equal(t[i], before[m][i]) for i in range(c.nb) if i not in used)
    assert int(err[0]) == int((live & ~ok).any()) and int(c.err[0]) == 0
    if hq:
        assert (q_out[~live] == -7.0).all()
        rows = live & (pos < 512)
        if rows.any():
            check_rows(q_out.view(-1, hq, d)[rows], q.reshape(-1, hq, d)[rows], qw, 1e-5, cos, sin, pos[rows], dtype, "q_out")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128])
def test_append_kv4_unaligned_inputs(dtype, d):
    """inputs that are not vector-aligned give the codes of aligned ones"""
    g, b, n, hq, hkv, cap = gen_of(d), 2, 9, 3, 2, 64
    wide = randn(g, b * n, (hq + 2 * hkv) * d + 1).to(DTYPES[dtype][0])
    w = (1 + randn(g, d + 1) / 4).to(DTYPES[dtype][0])
    cos, sin = R.tables(cap, d)
    got = []
    for x, gain in ((wide[:, 1:], w[1:]), (wide[:, 1:].contiguous(), w[1:].clone())):
        c = Cache(b, hkv, cap, d)
        q_out = torch.zeros(b * n, hq * d, dtype=wide.dtype, device="cuda")
        R.append(c, x[:, : hq * d], x[:, hq * d : (hq + hkv) * d], x[:, (hq + hkv) * d :], q_out, b, n, hq, i64(3, 40), q_w=gain, k_w=gain,
                 cos=cos, sin=sin, dtype=dtype)
        got.append((q_out, *c.t.values()))
    assert all(torch.equal(x, y) for x, y in zip(*got))


def test_append_kv4_unassigned_blocks():
    """table entries outside the pool: those rows are not written and the pages' flag is set"""
    g, b, n, hkv, d, cap = gen_of(2), 1, 96, 2, 64, 128
    c = Cache(b, hkv, cap, d, 32)
    c.table[0, 1], c.table[0, 2] = -1, c.nb
    before = {m: t.clone() for m, t in c.t.items()}
    kv = randn(g, n, 2 * hkv * d).to(torch.bfloat16)
    cos, sin = R.tables(cap, d)
    R.append(c, None, kv[:, : hkv * d], kv[:, hkv * d :], None, b, n, 0, i64(0), cos=cos, sin=sin)
    assert int(c.err[0]) == 1
    code, scale = R.encode(kv[:32, hkv * d :].reshape(32, hkv, d))
    blk = int(c.table[0, 0])
    assert torch.equal(c.t["v"][blk], R.pack(code).transpose(0, 1)) and torch.equal(c.t["vs"][blk], scale.transpose(0, 1))
    for m, t in c.t.items():
        others = [i for i in range(c.nb) if i != blk]
        assert torch.equal(t[others], before[m][others])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128, 256, 40])
@pytest.mark.parametrize("block", [0, 64])
@pytest.mark.parametrize("shift", [0, 1])
def test_append_plain_is_rope_then_kv_update(dtype, d, block, shift):
    """a plain cache: the bits of am_gfx950_rope and am_gfx950_kv_update, sequence by sequence (v's bits, NaN included);
    shift: inputs that are not vector-aligned"""
    g, dt, b, n, hq, hkv, cap = gen_of(d), DTYPES[dtype][0], 3, 21, 4, 2, 192
    width = (hq + 2 * hkv) * d + shift
    qkv = randn(g, b * n, width).to(dt)[:, shift:]
    qkv[3, (hq + hkv) * d + 5] = float("nan")
    q, k, v = qkv[:, : hq * d], qkv[:, hq * d : (hq + hkv) * d], qkv[:, (hq + hkv) * d :]
    cos, sin = R.tables(cap, d)
    start = [0, 100, 171]
    shape = (b, hkv, cap, d)
    pages = [None] * (b + 1)
    if block:
        per = cap // block
        table = torch.randperm(b * per, generator=torch.Generator().manual_seed(1)).view(b, per).to(torch.int32).cuda()
        shape = (b * per, hkv, block, d)
        pages = [C.pointer(N.KvPages(table.data_ptr() + 4 * per * i, block, per, b * per, None)) for i in range(b)]
        pages.append(C.pointer(N.KvPages(table.data_ptr(), block, per, b * per, None)))
    want, got = ([torch.full(shape, 9.0, dtype=dt, device="cuda") for _ in range(2)] for _ in range(2))
    qc, kc, vc = q.contiguous(), k.contiguous(), v.contiguous()
    qr, kr = torch.empty_like(qc), torch.empty_like(kc)
    pos = torch.cat([torch.arange(s, s + n, device="cuda") for s in start])
    L.call("am_gfx950_rope", N.RopeArgs(qc.data_ptr(), kc.data_ptr(), qr.data_ptr(), kr.data_ptr(), pos.data_ptr(), cos.data_ptr(),
                                        sin.data_ptr(), b * n, hq, hkv, d, cap, DTYPES[dtype][1]), R.stream())
    e = dt.itemsize
    for i in range(b):
        to = [t.data_ptr() + (0 if block else i * hkv * cap * d * e) for t in want]
        L.call("am_gfx950_kv_update", N.KvUpdateArgs(kr.data_ptr() + i * n * hkv * d * e, vc.data_ptr() + i * n * hkv * d * e, *to, n,
                                                     hkv, d, cap, start[i], None, DTYPES[dtype][1], None, pages[i]), R.stream())
    qo, sd = torch.empty_like(qc), i64(*start)
    a = N.KvAppendArgs(q.data_ptr(), k.data_ptr(), v.data_ptr(), qo.data_ptr(), b, n, hq, hkv, d, qkv.stride(0), qkv.stride(0),
                       qkv.stride(0), hq * d, None, None, 0.0, cos.data_ptr(), sin.data_ptr(), cap, sd.data_ptr(), None,
                       got[0].data_ptr(), got[1].data_ptr(), None, None, cap, hkv * cap * d, N.AM_KV_PLAIN, DTYPES[dtype][1], None,
                       pages[b])
    L.call("am_gfx950_kv_append", a, R.stream())
    bits = torch.int16 if e == 2 else torch.int32
    assert torch.equal(qo, qr)
    for x, y in zip(got, want):
        assert torch.equal(x.view(bits), y.view(bits))


def test_append_rows_alone_equal_rows_together():
    """a row's codes do not depend on the call that writes it: one call of 40 rows, and 40 calls of one"""
    g, hq, hkv, d, cap, n = gen_of(9), 8, 2, 128, 64, 40
    qkv = randn(g, n, (hq + 2 * hkv) * d).to(torch.bfloat16)
    cos, sin = R.tables(cap, d)
    w = (1 + randn(g, d) / 4).to(torch.bfloat16)
    outs = []
    for step in (n, 1):
        c = Cache(1, hkv, cap, d)
        q_out = torch.zeros(n, hq * d, dtype=torch.bfloat16, device="cuda")
        for r in range(0, n, step):
            x = qkv[r : r + step]
            R.append(c, x[:, : hq * d], x[:, hq * d : (hq + hkv) * d], x[:, (hq + hkv) * d :], q_out[r : r + step], 1, step, hq, i64(r),
                     q_w=w, k_w=w, cos=cos, sin=sin)
        outs.append((q_out, *(c.t[m] for m in ("k", "ks", "v", "vs"))))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


# ------------------------------------------------------------------ kv4_read
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("block", [0, 32])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_read_rows(d, block, dtype):
    g, b, hkv, cap, n = gen_of(d), 3, 3, 96, 23
    c = Cache(b, hkv, cap, d, block)
    for m in ("k", "v"):
        c.put_values(m, randn(g, b, hkv, cap, d))
    start, lens = [80, -4, 3], [23, 23, 7]
    out = [torch.full((b * n, hkv * d), 3.5, dtype=DTYPES[dtype][0], device="cuda") for _ in range(2)]
    R.read(c, b, n, i64(*start), i32(*lens), dtype, out)
    for m, got in zip(("k", "v"), out):
        vals = c.values(m)
        want = torch.full((b, n, hkv, d), 3.5, dtype=torch.float64, device="cuda")
        for i in range(b):
            for s in range(lens[i]):
                p = start[i] + s
                want[i, s] = vals[i, :, p] if 0 <= p < cap else 0.0
        assert torch.equal(got.double(), want.view(b * n, hkv * d)), m


# ------------------------------------------------------------------ kv4_attention
def attention_case(seed, b, n, hq, hkv, d, cap, start, lens=None, block=0, dtype="bf16", scale=0.0, behind="nan", ws=None, twice=True,
                   spread=1.0):
    g, dt = gen_of(seed), DTYPES[dtype][0]
    c = Cache(b, hkv, cap, d, block, seed=seed)
    live = lens or [n] * b
    for m in ("k", "v"):
        c.put_values(m, randn(g, b, hkv, cap, d) * spread)
        if behind == "nan":  # past the last live row's keys the cache holds anything
            code, sc = c.whole(m), c.whole(m + "s")
            for i in range(b):
                end = min(max(start[i] + live[i], 0), cap) if live[i] else 0
                code[i, :, end:], sc[i, :, end:] = 0x7F, 0xFF
            c.put(m, code)
            c.put(m + "s", sc)
    q = randn(g, b * n, hq * d).to(dt)
    out = torch.full((b * n, hq * d), 4.25, dtype=dt, device="cuda")
    ws = R.workspace(b, n, hq, hkv, d, cap) if ws is None else ws
    args = (c, q, out, b, n, hq, i64(*start), ws, i32(*lens) if lens else None, scale, dtype)
    R.attend(*args)
    if twice:
        first = out.clone()
        out.fill_(4.25)
        R.attend(*args)
        assert torch.equal(out.view(torch.uint8), first.view(torch.uint8)), "two calls differ"
    assert not ws[:16384].any(), "tickets left"
    s = scale or R.softmax_scale(d)
    want, mag, top = R.attention(q.double().view(b, n, hq, d), c.values("k").nan_to_num(0.0), c.values("v").nan_to_num(0.0), start, live, s)
    got = out.view(b, n, hq, d)
    rows = torch.tensor([[r < live[i] for r in range(n)] for i in range(b)], device="cuda")
    assert (got[~rows] == 4.25).all(), "rows behind the last were written"
    bound = R.attention_bound(want, mag, top, cap, d, dtype)
    off = (got.double() - want).abs()[rows]
    assert not torch.isnan(off).any(), "NaN"
    assert (off <= bound[rows]).all(), f"off by {float((off / bound[rows]).max()):.2f} of the bound"


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 1), (8, 2), (14, 2), (8, 1), (16, 1), (10, 2)])
@pytest.mark.parametrize("n,start", [(1, 0), (1, 31), (1, 32), (1, 200), (2, 7), (5, 0), (17, 90), (40, 0)])
def test_attention_shapes(dtype, d, hq, hkv, n, start):
    attention_case(n + d, 1, n, hq, hkv, d, 288, [start], dtype=dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("block", [0, 32, 128])
@pytest.mark.parametrize("ctx", [[1], [33], [640], [1000, 5, 0, 300], [2047] * 3])
def test_attention_decode(dtype, block, ctx):
    """contexts from nothing (a row before position 0 gives zeros) to several pieces; paged and not"""
    attention_case(len(ctx), len(ctx), 1, 32, 8, 128, 2080, [t - 1 for t in ctx], block=block, dtype=dtype)


@pytest.mark.parametrize("n", [1, 3, 400])
def test_attention_paged_capacity_inside_a_block(n):
    """a capacity that ends inside a block, and inside a step of 32 keys: rows at and past it"""
    attention_case(n, 1, n, 64, 16, 64, 405, [404 - n // 2], block=64, behind="nan" if n == 1 else "")


def test_attention_one_long_row():
    attention_case(1, 1, 1, 8, 2, 128, 20000 - 20000 % 32, [19900])


@pytest.mark.parametrize("b", [17, 63, 64, 65, 130, 300])
def test_attention_many_rows_of_uneven_contexts(b):
    """units over several lanes' worth of the plan, one of them far longer than the others"""
    start = [(37 * i) % 90 for i in range(b)]
    start[b // 2] = 1500
    attention_case(b, b, 1, 2, 1, 64, 1536, start)


def test_attention_more_blocks_than_a_plan():
    attention_case(3, 40, 1, 64, 16, 64, 128, [(29 * i) % 127 for i in range(40)])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n", [1, 6, 33])
def test_attention_padded_batch(dtype, n):
    """rows behind a sequence's last are left; a sequence of none; one that starts before 0; one past the cache"""
    attention_case(n, 5, n, 8, 2, 128, 128, [100, 3, 0, -4, 126], lens=[n, max(n - 2, 0), 0, n, n], dtype=dtype, block=64)


def test_attention_scale_and_peaked_scores():
    attention_case(4, 2, 3, 8, 2, 128, 512, [500, 77], scale=0.5)
    attention_case(5, 2, 3, 8, 2, 128, 512, [500, 77], scale=3.0, dtype="f32")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n,hq,hkv", [(1, 8, 2), (5, 8, 2), (400, 64, 16)])
@pytest.mark.parametrize("rise", [0.02, 0.12, 0.5, -0.1])
def test_attention_rising_scores(dtype, n, hq, hkv, rise):
    """scores that rise (or fall) by `rise` a key, beside noise: every step of keys passes the ones before by little or much"""
    g, d, cap, start = gen_of(n), 64, 800, 380
    c = Cache(1, hkv, cap, d, 32)
    u = randn(g, d).sign()
    k = u * (torch.arange(cap, device="cuda")[:, None] * rise / d) + randn(g, 1, hkv, cap, d) * 0.05
    c.put_values("k", k)
    c.put_values("v", randn(g, 1, hkv, cap, d))
    q = (u * d**0.5 + randn(g, n, hq, d)).view(n, hq * d).to(DTYPES[dtype][0])
    out = torch.empty_like(q)
    R.attend(c, q, out, 1, n, hq, i64(start), R.workspace(1, n, hq, hkv, d, cap), dtype=dtype)
    want, mag, top = R.attention(q.double().view(1, n, hq, d), c.values("k"), c.values("v"), [start], [n], R.softmax_scale(d))
    bound = R.attention_bound(want, mag, top, cap, d, dtype)
    if N.last_launch().kernel.startswith(b"kv4_attention_wide<bf16"):
        # f16 probabilities: a reference that a score passes by less than 2^4 stands for 2^11, and f16 has steps of 2^-24 at its
        # least, so a probability is off by at most 2^-25 / 2^11 = 2^-36 of the row's largest beside its 11 bits.  (Where the
        # keys near the largest score hold zeros in a dimension, `mag` there is smaller than that.)
        bound = bound + 2.0**-36 * c.values("v").abs().sum(2).amax()
    assert ((out.double().view_as(want) - want).abs() <= bound).all()


@pytest.mark.parametrize("n", [1, 4, 40])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_nan_keys_and_values(n, dtype):
    """a NaN value spoils its own 32 dimensions of the rows that see it, a NaN key whole rows, and no others; of two
    rows in one tile the earlier one must not meet the later one's key"""
    g, b, hq, hkv, d, cap, start = gen_of(n), 1, 8, 2, 128, 128, 50
    for which in ("k", "v"):
        c = Cache(b, hkv, cap, d)
        for m in ("k", "v"):
            c.put_values(m, randn(g, b, hkv, cap, d))
        clean = {m: c.values(m) for m in ("k", "v")}
        key = start + n // 2  # seen by rows n // 2 and later
        c.t[which + "s"][0, 1, key, 2] = 255
        q = randn(g, n, hq * d).to(DTYPES[dtype][0])
        out = torch.empty_like(q)
        R.attend(c, q, out, b, n, hq, i64(start), R.workspace(b, n, hq, hkv, d, cap), dtype=dtype)
        want, mag, top = R.attention(q.double().view(b, n, hq, d), clean["k"], clean["v"], [start], [n], R.softmax_scale(d))
        bad = torch.zeros(n, hq, d, dtype=torch.bool, device="cuda")
        bad[n // 2 :, 4:, 64:96 if which == "v" else None] = True
        if which == "k":
            bad[n // 2 :, 4:] = True
        got = out.view(n, hq, d)
        assert torch.equal(torch.isnan(got), bad)
        ok = (got.double() - want[0]).abs() <= R.attention_bound(want, mag, top, cap, d, dtype)[0]
        assert (ok | bad).all()


def test_attention_extreme_scales():
    """the largest and the smallest groups a writer makes"""
    g, d, cap = gen_of(3), 128, 64
    c = Cache(1, 1, cap, d)
    k, v = randn(g, 1, 1, cap, d), randn(g, 1, 1, cap, d)
    k[..., :32] *= 1e-38
    v[..., 32:64] *= 1e37
    v[..., 64:96] *= 1e-37
    c.put_values("k", k)
    c.put_values("v", v)
    q = randn(g, 1, 4 * d)
    out = torch.empty_like(q)
    R.attend(c, q, out, 1, 1, 4, i64(cap - 1), R.workspace(1, 1, 4, 1, d, cap), dtype="f32")
    want, mag, top = R.attention(q.double().view(1, 1, 4, d), c.values("k"), c.values("v"), [cap - 1], [1], R.softmax_scale(d))
    assert ((out.double().view(1, 1, 4, d) - want).abs() <= R.attention_bound(want, mag, top, cap, d, "f32") + 1e-42).all()


def test_attention_shared_prefix_stride_zero():
    """sequences that read one cache (stride 0)"""
    g, b, hq, hkv, d, cap = gen_of(8), 3, 8, 2, 64, 96
    c = Cache(1, hkv, cap, d)
    for m in ("k", "v"):
        c.put_values(m, randn(g, 1, hkv, cap, d))
    q = randn(g, b, hq * d).to(torch.bfloat16)
    out, ws, start = torch.empty_like(q), R.workspace(b, 1, hq, hkv, d, cap), i64(95, 10, 40)
    c.cbs = lambda: 0
    R.attend(c, q, out, b, 1, hq, start, ws)
    for i in range(b):
        one = torch.empty(1, hq * d, dtype=torch.bfloat16, device="cuda")
        R.attend(c, q[i : i + 1], one, 1, 1, hq, start[i : i + 1].clone(), ws)
        want, mag, top = R.attention(q[i : i + 1].double().view(1, 1, hq, d), c.values("k"), c.values("v"), [int(start[i])], [1],
                                     R.softmax_scale(d))
        bound = R.attention_bound(want, mag, top, cap, d, "bf16").flatten()
        assert ((out[i].double() - want.flatten()).abs() <= bound).all() and ((one[0].double() - want.flatten()).abs() <= bound).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("hq,hkv,d,b,n,start,lens,block", [
    (64, 16, 128, 2, 200, [0, 70], None, 0),
    (64, 16, 64, 2, 200, [0, 70], [200, 77], 32),
    (32, 32, 128, 1, 800, [5], None, 64),               # heads of their own
    (48, 16, 128, 1, 490, [33], None, 0),               # three heads a group: columns to spare
    (80, 16, 64, 1, 300, [0], None, 0),                 # five
    (14, 2, 64, 9, 180, [0, 3, 90, 0, 50, 7, 8, 9, -40], [180, 1, 180, 0, 44, 180, 2, 33, 90], 32),
    (64, 64, 128, 1, 300, [-30], None, 0),              # rows before position 0
    (64, 64, 64, 1, 300, [20], None, 0),                # past the cache
    (256, 16, 64, 1, 100, [0], None, 0),                # sixteen heads a group
    (64, 16, 64, 1, 400, [2300], None, 32),             # more blocks than a wave holds of the table
    (32, 8, 128, 16, 33, [31 * i for i in range(16)], [33 - 2 * i for i in range(16)], 32),  # a second block of one row
])
def test_attention_many_rows(dtype, hq, hkv, d, b, n, start, lens, block):
    cap = 160 if start == [20] else max(max(s + n for s in start), 32) + 31
    attention_case(n, b, n, hq, hkv, d, cap - cap % 32, start, lens=lens, block=block, dtype=dtype)
    assert N.last_launch().kernel.startswith(b"kv4_attention_wide")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("hq,hkv,d,b,n,start,lens,block", [
    (64, 16, 64, 1, 100, [2300], None, 32),              # two pieces of four
    (64, 16, 128, 1, 97, [4181], None, 64),              # four pieces, the last one short
    (32, 16, 64, 3, 64, [2100, 0, 1100], [64, 33, 0], 0),  # sequences of two, one and no pieces
    (16, 16, 128, 2, 200, [1990, 980], [200, 7], 32),    # rows on both sides of a further piece
    (96, 16, 64, 1, 60, [-20], None, 0),                 # no keys for some
    (64, 16, 64, 1, 128, [6000], None, 0),               # past the cache
])
def test_attention_many_rows_in_pieces(dtype, hq, hkv, d, b, n, start, lens, block):
    cap = 3000 if start == [6000] else max(max(s + n for s in start), 64) + 31
    attention_case(n, b, n, hq, hkv, d, cap - cap % 32, start, lens=lens, block=block, dtype=dtype)
    assert N.last_launch().kernel.startswith(b"kv4_attention_wide") and b"splits=1>" not in N.last_launch().kernel


@pytest.mark.parametrize("which", ["k", "v"])
def test_attention_many_rows_in_pieces_nan_and_distant_values(which):
    """a NaN in one piece's keys and values of 2^40 times the others' in another's"""
    g, hq, hkv, n, start, cap, d = gen_of(5), 64, 16, 100, 2400, 2528, 64
    c = Cache(1, hkv, cap, d, 32)
    k, v = randn(g, 1, hkv, cap, d), randn(g, 1, hkv, cap, d)
    v[:, 2, 2470, :32] *= 2.0**40
    c.put_values("k", k)
    c.put_values("v", v)
    clean = {m: c.values(m) for m in ("k", "v")}
    marks = c.whole(which + "s")
    marks[0, 3, 2450, 1] = 255  # seen by rows 50 and later of kv head 3
    marks[0, 7, 100, 0] = 254   # by all rows of kv head 7
    c.put(which + "s", marks)
    q = randn(g, n, hq * d).to(torch.bfloat16)
    out, ws = torch.empty_like(q), R.workspace(1, n, hq, hkv, d, cap)
    R.attend(c, q, out, 1, n, hq, i64(start), ws)
    assert N.last_launch().kernel.startswith(b"kv4_attention_wide") and not ws[:16384].any()
    want, mag, top = R.attention(q.double().view(1, n, hq, d), clean["k"], clean["v"], [start], [n], R.softmax_scale(d))
    bad = torch.zeros(n, hq, d, dtype=torch.bool, device="cuda")
    bad[50:, 12:16, slice(32, 64) if which == "v" else slice(None)] = True
    bad[:, 28:32, slice(0, 32) if which == "v" else slice(None)] = True
    got = out.view(n, hq, d)
    assert torch.equal(torch.isnan(got), bad)
    assert (((got.double() - want[0]).abs() <= R.attention_bound(want, mag, top, cap, d, "bf16")[0]) | bad).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_many_rows_spread_values(dtype):
    """values whose scales differ widely between keys and between groups, rows that meet only the small ones"""
    g, n, hq, hkv, d, cap = gen_of(3), 400, 64, 16, 128, 416
    c = Cache(1, hkv, cap, d)
    k, v = randn(g, 1, hkv, cap, d), randn(g, 1, hkv, cap, d)
    v *= torch.exp2(torch.randint(-12, 13, (1, hkv, cap, 4), generator=g, device="cuda").double()).float().repeat_interleave(32, -1)
    v[..., :32] *= 2.0**60
    v[..., 32:64] *= 2.0**-60
    v[:, :, :50, 64:96] = 0  # a group of zeros first
    c.put_values("k", k)
    c.put_values("v", v)
    q = randn(g, n, hq * d).to(DTYPES[dtype][0])
    out, ws = torch.empty_like(q), R.workspace(1, n, hq, hkv, d, cap)
    R.attend(c, q, out, 1, n, hq, i64(0), ws, dtype=dtype)
    assert N.last_launch().kernel.startswith(b"kv4_attention_wide")
    want, mag, top = R.attention(q.double().view(1, n, hq, d), c.values("k"), c.values("v"), [0], [n], R.softmax_scale(d))
    assert ((out.double().view_as(want) - want).abs() <= R.attention_bound(want, mag, top, cap, d, dtype)).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("up", [0, 8, 16, 17, 18, 40, 120])
def test_attention_many_rows_distant_later_values(d, up):
    """a later key's value of 2^up times the others', inside the rows of one block: the rows before it do not notice"""
    g, n, hq, hkv, cap, b = gen_of(d), 400, 64, 16, 416, 1
    c = Cache(1, hkv, cap, d)
    k, v = randn(g, 1, hkv, cap, d), randn(g, 1, hkv, cap, d) * 2.0**-50
    v[:, :, 77] *= 2.0**up
    v[:, :, 251, :32] = 0
    c.put_values("k", k)
    c.put_values("v", v)
    q = randn(g, n, hq * d).to(torch.bfloat16)
    out, ws = torch.empty_like(q), R.workspace(1, n, hq, hkv, d, cap)
    R.attend(c, q, out, 1, n, hq, i64(0), ws)
    assert N.last_launch().kernel.startswith(b"kv4_attention_wide")
    want, mag, top = R.attention(q.double().view(1, n, hq, d), c.values("k"), c.values("v"), [0], [n], R.softmax_scale(d))
    got = out.double().view_as(want)
    assert (got.abs().amax((0, 2, 3)) > 0).all()
    # attention_bound with its floor (1e-30) scaled as the values are
    assert ((got - want).abs() * 2.0**50 <= R.attention_bound(want * 2.0**50, mag * 2.0**50, top, cap, d, "bf16")).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_many_rows_nan(dtype, d):
    """as test_attention_nan_keys_and_values, for the kernel of many rows"""
    g, hq, hkv, n, start, cap = gen_of(7), 64, 16, 400, 40, 480
    for which in ("k", "v"):
        c = Cache(1, hkv, cap, d, 32)
        for m in ("k", "v"):
            c.put_values(m, randn(g, 1, hkv, cap, d))
        clean = {m: c.values(m) for m in ("k", "v")}
        marks = {m: c.whole(m + "s") for m in ("k", "v")}
        marks[which][0, 3, 100, 1] = 253  # seen by rows 60 and later of kv head 3
        marks[which][0, 5, start + n :] = 255  # behind every row
        c.put(which + "s", marks[which])
        q = randn(g, n, hq * d).to(DTYPES[dtype][0])
        out = torch.empty_like(q)
        R.attend(c, q, out, 1, n, hq, i64(start), R.workspace(1, n, hq, hkv, d, cap), dtype=dtype)
        want, mag, top = R.attention(q.double().view(1, n, hq, d), clean["k"], clean["v"], [start], [n], R.softmax_scale(d))
        bad = torch.zeros(n, hq, d, dtype=torch.bool, device="cuda")
        bad[60:, 12:16, slice(32, 64) if which == "v" else slice(None)] = True
        got = out.view(n, hq, d)
        assert torch.equal(torch.isnan(got), bad)
        assert (((got.double() - want[0]).abs() <= R.attention_bound(want, mag, top, cap, d, dtype)[0]) | bad).all()


@pytest.mark.parametrize("block", [0, 4096])
def test_offsets_past_32_bits(block):
    """caches of 2^34 values: rows written, read and attended to where offsets in values (and in bytes) pass 2^32; scores of
    the rows before them are 0 beside ones near 60, values 0, so that they add nothing"""
    g, b, hq, hkv, d, cap, n = gen_of(4), 2, 8, 2, 128, 2**25 + 96, 40
    c = Cache(b, hkv, cap, d, block, fill=0, scale_fill=0)
    start = [cap - n, cap - 4000]
    kv = randn(g, b * n, 2 * hkv * d).to(torch.bfloat16)
    code, scale = R.encode(kv.view(b, n, 2, hkv, d))
    cos, sin = torch.ones(cap, d // 2, device="cuda"), torch.zeros(cap, d // 2, device="cuda")
    R.append(c, None, kv[:, : hkv * d], kv[:, hkv * d :], None, b, n, 0, i64(*start), cos=cos, sin=sin)
    del cos, sin
    for i in range(b):
        for m, t in (("k", 0), ("v", 1)):
            for r in (0, n - 1):
                at = start[i] + r
                row = c.t[m][i, :, at] if not block else c.t[m][int(c.table[i, at // block]), :, at % block]
                assert torch.equal(row, R.pack(code[i, r, t])), (m, i, r)
    k, v = R.read(c, b, n, i64(*start))
    values = R.decode(R.pack(code), scale)  # [b][n][2][hkv][d]
    assert torch.equal(k.double().view(b, n, hkv, d), values[:, :, 0]) and torch.equal(v.double().view(b, n, hkv, d), values[:, :, 1])
    # a row at the end of each sequence's keys: q along its first key, 60 in the exponent
    q = torch.empty(b, hq, d, device="cuda")
    for h in range(hq):
        key = values[:, 0, 0, h // (hq // hkv)].float()
        q[:, h] = key * (60 * d**0.5 / key.square().sum(-1, keepdim=True))
    q = q.to(torch.bfloat16)
    out, at = torch.empty(b, hq, d, dtype=torch.bfloat16, device="cuda"), i64(*[s + n - 1 for s in start])
    R.attend(c, q, out, b, 1, hq, at, R.workspace(b, 1, hq, hkv, d, cap))
    planes = values.permute(2, 0, 3, 1, 4)  # [2][b][hkv][n][d]
    want, mag, top = R.attention(q.double().view(b, 1, hq, d), planes[0], planes[1], [n - 1] * b, [1] * b, R.softmax_scale(d))
    # the other keys' share: 2^26 e^-60 < 2^-60
    assert ((out.double().view_as(want) - want).abs() <= R.attention_bound(want, mag, top, 2 * n, d, "bf16")).all()
    # the kernel of many rows, at the front of each sequence's planes (the second head's start past 2^32)
    c.t["k"].zero_(), c.t["v"].zero_()
    m, hd = 1024, 64
    kv = randn(g, b * m, 2 * hkv * d).to(torch.bfloat16)
    cos, sin = torch.ones(cap, hd, device="cuda"), torch.zeros(cap, hd, device="cuda")
    R.append(c, None, kv[:, : hkv * d], kv[:, hkv * d :], None, b, m, 0, i64(0, 0), cos=cos, sin=sin)
    q = randn(g, b * m, hq * d).to(torch.bfloat16)
    out = torch.empty_like(q)
    R.attend(c, q, out, b, m, hq, i64(0, 0), R.workspace(b, m, hq, hkv, d, cap))
    assert N.last_launch().kernel.startswith(b"kv4_attention_wide")
    code, scale = R.encode(kv.view(b, m, 2, hkv, d))
    planes = R.decode(R.pack(code), scale).permute(2, 0, 3, 1, 4)
    rows = [0, 31, 500, m - 1]
    for r in rows:
        want, mag, top = R.attention(q.double().view(b, m, hq, d)[:, r : r + 1], planes[0], planes[1], [r] * b, [1] * b, R.softmax_scale(d))
        got = out.double().view(b, m, hq, d)[:, r : r + 1]
        assert ((got - want).abs() <= R.attention_bound(want, mag, top, m, d, "bf16")).all()


# ------------------------------------------------------------------ together
class Model:
    """One attention layer of a decode: append of a token of each sequence, then attention over the cache."""

    def __init__(self, b, hq, hkv, d, cap, block):
        self.c = Cache(b, hkv, cap, d, block)
        self.b, self.hq = b, hq
        self.cos, self.sin = R.tables(cap, d)
        g = gen_of(1)
        self.w = (1 + randn(g, d) / 4).to(torch.bfloat16)
        self.qkv = torch.zeros(b, (hq + 2 * hkv) * d, dtype=torch.bfloat16, device="cuda")
        self.q = torch.zeros(b, hq * d, dtype=torch.bfloat16, device="cuda")
        self.out = torch.zeros_like(self.q)
        self.start = torch.zeros(b, dtype=torch.int64, device="cuda")

    def step(self, ws):
        hq, hkv, d = self.hq, self.c.hkv, self.c.d
        x = self.qkv
        R.append(self.c, x[:, : hq * d], x[:, hq * d : (hq + hkv) * d], x[:, (hq + hkv) * d :], self.q, self.b, 1, hq, self.start,
                 q_w=self.w, k_w=self.w, cos=self.cos, sin=self.sin)
        R.attend(self.c, self.q, self.out, self.b, 1, hq, self.start, ws)


@pytest.mark.parametrize("block", [0, 32])
def test_decode_loop_of_append_and_attention(block):
    """a prompt appended in one call, then token by token; every step's output against the cache's own values, which are
    checked against the encoding of the rotated keys"""
    b, hq, hkv, d, cap, prompt = 2, 8, 2, 128, 96, 40
    m = Model(b, hq, hkv, d, cap, block)
    g = gen_of(12)
    pre = randn(g, b * prompt, (hq + 2 * hkv) * d).to(torch.bfloat16)
    q_pre, o_pre = (torch.zeros(b * prompt, hq * d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    _, want, *_ = append_reference(m.c, pre, hq, [0, 0], [prompt, 33], prompt, m.cos, m.sin, m.w, m.w)
    R.append(m.c, pre[:, : hq * d], pre[:, hq * d : (hq + hkv) * d], pre[:, (hq + hkv) * d :], q_pre, b, prompt, hq, i64(0, 0),
             i32(prompt, 33), m.w, m.w, cos=m.cos, sin=m.sin)
    ws = R.workspace(b, prompt, hq, hkv, d, cap)
    R.attend(m.c, q_pre, o_pre, b, prompt, hq, i64(0, 0), ws, i32(prompt, 33))
    assert all(torch.equal(m.c.whole(n), want[n]) for n in want)
    k, v = (m.c.values(n).nan_to_num(0.0) for n in ("k", "v"))
    ref, mag, top = R.attention(q_pre.double().view(b, prompt, hq, d), k, v, [0, 0], [prompt, 33], R.softmax_scale(d))
    assert ((o_pre.double().view_as(ref) - ref).abs() <= R.attention_bound(ref, mag, top, cap, d, "bf16")).all()
    at = [prompt, 33]
    for _ in range(6):
        m.qkv.copy_(randn(g, *m.qkv.shape))
        m.start.copy_(i64(*at))
        _, want, *_ = append_reference(m.c, m.qkv, hq, at, [1, 1], 1, m.cos, m.sin, m.w, m.w)
        m.step(ws)
        assert all(torch.equal(m.c.whole(n), want[n]) for n in want)
        k, v = (m.c.values(n).nan_to_num(0.0) for n in ("k", "v"))
        ref, mag, top = R.attention(m.q.double().view(b, 1, hq, d), k, v, at, [1, 1], R.softmax_scale(d))
        assert ((m.out.double().view_as(ref) - ref).abs() <= R.attention_bound(ref, mag, top, cap, d, "bf16")).all()
        kr, vr = R.read(m.c, b, 1, m.start)
        for i in range(b):
            assert torch.equal(kr[i].double().view(hkv, d), k[i, :, at[i]]) and torch.equal(vr[i].double().view(hkv, d), v[i, :, at[i]])
        at = [t + 1 for t in at]


def test_graphs_that_share_a_workspace():
    """two captured steps of different shapes on one workspace, replayed in turn with eager work between; every replay equals
    the eager call of the same inputs"""
    models = [Model(3, 32, 8, 128, 4096, 64), Model(1, 16, 4, 128, 8192, 0)]
    g = gen_of(3)
    need = max(R.workspace(m.b, 1, m.hq, m.c.hkv, m.c.d, m.c.cap).numel() for m in models)
    ws = torch.zeros(need, dtype=torch.uint8, device="cuda")
    for m in models:
        for n in ("k", "v"):
            m.c.put_values(n, randn(g, m.b, m.c.hkv, m.c.cap, m.c.d))
    side = torch.cuda.Stream()
    graphs = []
    for m in models:
        m.start.copy_(torch.arange(m.b, device="cuda") * 500 + 3000)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            m.step(ws)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            m.step(ws)
        graphs.append(graph)
    for turn in range(4):
        for m, graph in zip(models, graphs):
            m.qkv.copy_(randn(g, *m.qkv.shape))
            m.start.copy_(torch.arange(m.b, device="cuda") * 400 + 100 + 700 * turn)
            m.out.zero_()
            graph.replay()
            got = m.out.clone()
            torch.cuda.synchronize()
            m.out.zero_()
            m.step(ws)
            assert torch.equal(got, m.out)
            torch.cuda.synchronize()
    assert not ws[:16384].any()


def test_graph_of_pieces_beside_decode():
    """a captured call of many rows in pieces and one of single rows, on one workspace, at other positions in every replay"""
    g, hq, hkv, d, cap, n = gen_of(31), 64, 16, 64, 4096, 100
    c = Cache(1, hkv, cap, d, 64)
    for m in ("k", "v"):
        c.put_values(m, randn(g, 1, hkv, cap, d))
    ws = torch.zeros(max(R.workspace(1, r, hq, hkv, d, cap).numel() for r in (n, 1)), dtype=torch.uint8, device="cuda")
    q = [torch.zeros(r, hq * d, dtype=torch.bfloat16, device="cuda") for r in (n, 1)]
    out = [torch.zeros_like(t) for t in q]
    start = [i64(0), i64(0)]

    def step():
        for x, y, s in zip(q, out, start):
            R.attend(c, x, y, 1, x.shape[0], hq, s, ws)

    start[0].fill_(2200)
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for first in (3900, 0, 2048, 700):
        for x in q:
            x.copy_(randn(g, *x.shape))
        start[0].fill_(first), start[1].fill_(first + n)
        for y in out:
            y.zero_()
        graph.replay()
        got = [y.clone() for y in out]
        torch.cuda.synchronize()
        for y in out:
            y.zero_()
        step()
        assert all(torch.equal(x, y) for x, y in zip(got, out))
        assert out[0].any(-1).all() and not ws[:16384].any()


def test_other_stream():
    m = Model(2, 8, 2, 64, 256, 32)
    g = gen_of(6)
    for n in ("k", "v"):
        m.c.put_values(n, randn(g, 2, 2, 256, 64))
    m.qkv.copy_(randn(g, *m.qkv.shape))
    m.start.copy_(i64(200, 31))
    ws = R.workspace(2, 1, 8, 2, 64, 256)
    m.step(ws)
    want = m.out.clone()
    m.out.zero_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m.step(ws)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(m.out, want)


def test_two_streams_at_once():
    """calls that overlap, each with a workspace and a cache of its own, give what they give alone"""
    g, models, alone = gen_of(14), [Model(2, 32, 8, 128, 16384, 64), Model(1, 16, 4, 128, 32768, 0)], []
    spaces = [R.workspace(m.b, 1, m.hq, m.c.hkv, m.c.d, m.c.cap) for m in models]
    for m, ws in zip(models, spaces):
        for n in ("k", "v"):
            m.c.put_values(n, randn(g, m.b, m.c.hkv, m.c.cap, m.c.d))
        m.qkv.copy_(randn(g, *m.qkv.shape))
        m.start.copy_(torch.arange(m.b, device="cuda") * 500 + 15000)
        m.step(ws)
        alone.append(m.out.clone())
        m.out.zero_()
    streams = [torch.cuda.Stream() for _ in models]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for m, ws, s in zip(models, spaces, streams):
            with torch.cuda.stream(s):
                m.step(ws)
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for m, ws, want in zip(models, spaces, alone):
        assert torch.equal(m.out, want)
        assert not ws[:16384].any()


@pytest.mark.parametrize("n", [1, 100, 400])
def test_attention_refuses_a_smaller_workspace(n):
    """single rows over many keys, many rows in pieces, many rows: 16 bytes less than the size asked for"""
    hq, hkv, d, cap = 64, 16, 64, 4096
    c = Cache(1, hkv, cap, d, fill=0, scale_fill=0)
    q = torch.zeros(n, hq * d, dtype=torch.bfloat16, device="cuda")
    out, ws = torch.full_like(q, 2.0), R.workspace(1, n, hq, hkv, d, cap)
    with pytest.raises(N.NativeError):
        R.attend(c, q, out, 1, n, hq, i64(cap - n), ws[:-16])
    assert (out == 2.0).all()
    R.attend(c, q, out, 1, n, hq, i64(cap - n), ws)
    assert (out == 0.0).all()
