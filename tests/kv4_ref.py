"""Plain 64-bit forms of the 4-bit KV cache's operators, and plumbing their GPU tests share."""

from __future__ import annotations

import ctypes as C
import math

import torch

import aethermind_amd.native as N

GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
DTYPES = {"f32": (torch.float32, N.AM_DT_F32), "bf16": (torch.bfloat16, N.AM_DT_BF16)}
# half a step of a rounding to the type, relative to the value
HALF = {"f32": 2.0**-24, "bf16": 2.0**-8}


def encode(x):
    """Codes (one a byte) and scales of values [..., d], by search over the definition: the
    smallest exponent with max|x| < 7 * 2^e, the nearest code, ties to the even one."""
    g = x.double().reshape(*x.shape[:-1], -1, 32)
    top = g.abs().amax(-1)
    fine = torch.isfinite(g).all(-1)
    e = torch.full_like(top, -127)
    todo = fine & (top > 0)
    guess = torch.floor(torch.log2(torch.where(todo, top, 1.0))) - 4
    for k in range(8):  # the first that holds, from below
        guess = torch.where(top < 7 * torch.exp2(guess), guess, guess + 1)
    e = torch.where(todo, guess, e).clamp(-127, 125)
    u = (torch.where(fine[..., None], g, 0.0) / torch.exp2(e)[..., None]).abs()
    code = torch.zeros_like(u, dtype=torch.uint8)
    for c in range(7):
        mid = (GRID[c] + GRID[c + 1]) / 2
        # a tie goes to the even one of c and c + 1
        code = torch.where((u > mid) if c % 2 == 0 else (u >= mid), torch.tensor(c + 1, dtype=torch.uint8, device=x.device), code)
    code = torch.where(fine[..., None], code + 8 * torch.signbit(g).to(torch.uint8), torch.zeros_like(code))
    scale = torch.where(fine, e + 127, 255.0).to(torch.uint8)
    return code.reshape(x.shape), scale


def decode(packed, scale):
    """float64 values of packed codes [..., d/2] and scales [..., d/32]"""
    code = torch.stack([packed & 15, packed >> 4], -1).flatten(-2)
    v = torch.tensor(GRID + [-t for t in GRID], dtype=torch.float64, device=packed.device)[code.long()]
    s = torch.exp2(scale.double() - 127)
    s = torch.where(scale >= 253, torch.nan, s)
    return v * s.repeat_interleave(32, -1)


def pack(code):
    return code[..., 0::2] | (code[..., 1::2] << 4)


def norm(x, w, eps):
    x = x.double()
    if w is None:
        return x
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()


def rotate(y, cos, sin, ok):
    """[rows][heads][d] at table rows cos, sin [rows][d/2]; rows that are not ok stay"""
    a, b = y.chunk(2, -1)
    c, s = cos.double()[:, None], sin.double()[:, None]
    z = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.where(ok[:, None, None], z, y)


def tables(n, d, theta=10000.0):
    inv = theta ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    a = torch.arange(n, dtype=torch.float64)[:, None] * inv
    return a.cos().float().cuda(), a.sin().float().cuda()


def attention(q, k, v, start, lens, scale):
    """q [b][s][hq][d], k and v [b][hkv][cap][d] (float64); rows behind lens and rows without keys: zeros.
    Returns out and sum p |v| / sum p, and the largest sum |q k| scale, for bounds."""
    b, n, hq, d = q.shape
    hkv, cap = k.shape[1], k.shape[2]
    out = torch.zeros(b, n, hq, d, dtype=torch.float64, device=q.device)
    mag, top = torch.zeros_like(out), 0.0
    for i in range(b):
        for s in range(lens[i]):
            keys = min(max(start[i] + s + 1, 0), cap)
            if keys == 0:
                continue
            for h in range(hkv):
                g = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
                kk, vv = k[i, h, :keys], v[i, h, :keys]
                p = torch.softmax(q[i, s, g] @ kk.t().contiguous() * scale, -1)
                out[i, s, g] = p @ vv
                mag[i, s, g] = p @ vv.abs()
                top = max(top, float((q[i, s, g].abs() @ kk.abs().t().contiguous()).amax().nan_to_num(0.0)) * scale)
    return out, mag, top


def attention_bound(out, mag, top, keys, d, dtype):
    """What |kernel - out| may be: the rounding of out, and relative errors of the probabilities: fp32
    sums of d products in the scores (each off by at most (d + 4) 2^-24 sum|qk|, in the exponent, in numerator and
    denominator), exp2 (2 ulp), their parts and fp32 sums over the keys.  Parts: bf16 hi + lo 2^-16, three parts 2^-23;
    the kernel for many rows takes bf16 calls' probabilities in f16, off by at most half a step, 2^-11, each, in the
    numerator and in the row sum, which adds the same rounded values."""
    wide = N.last_launch().kernel.startswith(b"kv4_attention_wide")
    parts = (2 * 2.0**-11 if wide else 2.0**-16) if dtype == "bf16" else 2.0**-23
    rel = 2 * (d + 4) * 2.0**-24 * top + 4 * 2.0**-23 + parts + 2 * (keys + 64) * 2.0**-24
    return HALF[dtype] * out.abs() * 1.001 + rel * mag + 1e-30


class Cache:
    """A 4-bit cache [b][hkv][cap] in planes or, with `block`, in scattered blocks; `whole` gives planes back."""

    def __init__(self, b, hkv, cap, d, block=0, fill=0xAB, scale_fill=0xFF, spare=2, seed=0):
        self.b, self.hkv, self.cap, self.d, self.block = b, hkv, cap, d, block
        self.err = torch.zeros(1, dtype=torch.int32, device="cuda")
        if block:
            per = -(-cap // block)
            self.nb = b * per + spare
            gen = torch.Generator().manual_seed(seed)
            self.table = torch.randperm(self.nb, generator=gen)[: b * per].view(b, per).to(torch.int32).cuda()
            lead = (self.nb, hkv, block)
            self.pages = N.KvPages(self.table.data_ptr(), block, per, self.nb, self.err.data_ptr())
        else:
            lead, self.pages = (b, hkv, cap), None
        self.t = {}
        for n in ("k", "v"):
            self.t[n] = torch.full((*lead, d // 2), fill, dtype=torch.uint8, device="cuda")
            self.t[n + "s"] = torch.full((*lead, d // 32), scale_fill, dtype=torch.uint8, device="cuda")

    def ptr(self):
        return self.t["k"].data_ptr(), self.t["ks"].data_ptr(), self.t["v"].data_ptr(), self.t["vs"].data_ptr()

    def cbs(self):
        return self.hkv * self.cap * self.d

    def page_arg(self):
        return C.pointer(self.pages) if self.pages is not None else None

    def whole(self, name):
        t = self.t[name]
        if not self.block:
            return t.clone()
        t = t[self.table.long()]
        return t.transpose(1, 2).flatten(2, 3)[:, :, : self.cap]

    def put(self, name, planes):
        """planes [b][hkv][cap][...] into the cache"""
        if not self.block:
            self.t[name].copy_(planes)
            return
        per = self.table.shape[1]
        padded = torch.zeros(self.b, self.hkv, per * self.block, planes.shape[-1], dtype=torch.uint8, device="cuda")
        padded[:, :, : self.cap] = planes
        blocks = padded.view(self.b, self.hkv, per, self.block, -1).transpose(1, 2)
        self.t[name][self.table.long()] = blocks

    def put_values(self, name, x):
        code, scale = encode(x)
        self.put(name, pack(code))
        self.put(name + "s", scale)

    def values(self, name):
        return decode(self.whole(name), self.whole(name + "s"))


def i64(*v):
    return torch.tensor(v, dtype=torch.int64, device="cuda")


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def stream():
    return torch.cuda.current_stream().cuda_stream


def append(cache, q, k, v, q_out, b, n, hq, start, lens=None, q_w=None, k_w=None, eps=1e-5, cos=None, sin=None, err=None, dtype="bf16"):
    """am_gfx950_kv_append into a 4-bit cache; q, k, v may be views (row strides are taken from them)"""
    pt = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    kc, ks, vc, vs = cache.ptr()
    a = N.KvAppendArgs(pt(q), pt(k), pt(v), pt(q_out), b, n, hq, cache.hkv, cache.d, q.stride(0) if q is not None else 0,
                       k.stride(0), v.stride(0), q_out.stride(0) if q_out is not None else 0, pt(q_w), pt(k_w), eps, pt(cos),
                       pt(sin), cos.shape[0], pt(start), pt(lens), kc, vc, ks, vs, cache.cap, cache.cbs(), N.AM_KV_MXFP4,
                       DTYPES[dtype][1], pt(err), cache.page_arg())
    N.lib().call("am_gfx950_kv_append", a, stream())


def read(cache, b, n, start, lens=None, dtype="bf16", out=None):
    if out is None:
        out = [torch.zeros(b * n, cache.hkv * cache.d, dtype=DTYPES[dtype][0], device="cuda") for _ in range(2)]
    kc, ks, vc, vs = cache.ptr()
    a = N.Kv4ReadArgs(kc, ks, vc, vs, out[0].data_ptr(), out[1].data_ptr(), b, n, cache.hkv, cache.d, cache.cap, cache.cbs(),
                      start.data_ptr(), None if lens is None else lens.data_ptr(), DTYPES[dtype][1], cache.page_arg())
    N.lib().call("am_gfx950_kv4_read", a, stream())
    return out


def workspace(b, n, hq, hkv, d, cap):
    return torch.zeros(N.lib().am_gfx950_kv4_attention_workspace_bytes(b, n, hq, hkv, d, cap), dtype=torch.uint8, device="cuda")


def attend(cache, q, out, b, n, hq, start, ws, lens=None, scale=0.0, dtype="bf16"):
    kc, ks, vc, vs = cache.ptr()
    a = N.Kv4AttentionArgs(q.data_ptr(), out.data_ptr(), kc, ks, vc, vs, b, n, hq, cache.hkv, cache.d, cache.cap, cache.cbs(),
                           start.data_ptr(), None if lens is None else lens.data_ptr(), scale, DTYPES[dtype][1], ws.data_ptr(),
                           ws.numel(), cache.page_arg())
    N.lib().call("am_gfx950_kv4_attention", a, stream())


def softmax_scale(d):
    return 1.0 / math.sqrt(d)
