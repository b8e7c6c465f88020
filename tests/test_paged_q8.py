"""The 8-bit paged KV cache: writing, reading back and attention against the formulas in 64 bits.

Tolerances.  Codes and scales of unrotated 16-bit rows are exact (the quantiser's quotient is correctly rounded and
16-bit inputs keep away from its rounding points).  A rotated or 32-bit row differs by at most one code at a rounding
point: value tolerance one step of the code.  Attention: fp16 / bf16 outputs carry the output's rounding (2^-11 / 2^-8
of the value) and q and P rounded to 11 bits, 2^-11 each of a mean of values below max |v|: 3 * 2^-11 max |v| for fp16,
(2^-8 + 2^-10) max |v| for bf16; 32-bit rows keep 22 bits of q and P and sums in fp32: 2^-17 max |v|."""

from __future__ import annotations

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

F = {"int8": 127.0, "e4m3": 448.0}
CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


@pytest.fixture(scope="module")
def ops():
    from onnxruntime_ep_b200 import ops as _ops

    return _ops


@pytest.fixture(autouse=True)
def _device_error_clean(request):
    if "gpu" not in request.keywords:
        yield
        return
    from onnxruntime_ep_b200 import ops as _ops

    _ops.device_error(clear=True)
    yield
    torch.cuda.synchronize()
    code, detail = _ops.device_error(clear=True)
    assert code == 0, f"device error {code} ({detail})"


# ---- the formulas in 64 bits ------------------------------------------------------------------------
E4M3 = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
E4M3_POS = E4M3[:127]  # 0 .. 448, ascending


def nearest_e4m3(t):
    """Nearest e4m3 value, ties to the even code."""
    a = np.abs(t)
    i = np.clip(np.searchsorted(E4M3_POS, a), 1, 126)
    lo, hi = E4M3_POS[i - 1], E4M3_POS[i]
    up = (a - lo > hi - a) | ((a - lo == hi - a) & (i % 2 == 0))
    return np.where(up, hi, lo) * np.where(np.signbit(t), -1.0, 1.0)


def quantise(x, code):
    """(codes as values, scale) of rows x [..., D] in 64 bits."""
    a = np.abs(x).max(-1, keepdims=True)
    t = np.divide(x * F[code], a, out=np.zeros_like(x), where=a > 0)  # exact products: ties stay ties
    return (np.rint(t) if code == "int8" else nearest_e4m3(t)), a[..., 0] / F[code]


def rotate(x, cos, sin, pos, inter):
    """x [T, heads, D] at positions pos [T]; cos / sin [max_seq, half]."""
    half = cos.shape[1]
    c, s = cos[pos][:, None], sin[pos][:, None]
    y = x.copy()
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if inter else (x[..., :half], x[..., half:2 * half])
    ra, rb = a * c - b * s, b * c + a * s
    if inter:
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = ra, rb
    else:
        y[..., :half], y[..., half:2 * half] = ra, rb
    return y


class Case:
    """Sequences of `new` rows behind `past` cached ones, pages scattered at random."""

    def __init__(self, rng, *, H, HK, D, bs, new, past, dt, code, rotary=True, inter=0, half=None, spread=1.0):
        self.H, self.HK, self.D, self.bs, self.code, self.dt, self.inter = H, HK, D, bs, code, dt, inter
        self.new, self.past = list(new), list(past)
        B, T = len(new), sum(new)
        total = [a + b for a, b in zip(new, past)]
        need = [-(-t // bs) for t in total]
        self.nb = sum(need) + 2
        order = rng.permutation(self.nb).astype(np.int32)
        self.bt = np.full((B, max(max(need), 1) + 1), -1, np.int32)
        o = 0
        for b, n in enumerate(need):
            self.bt[b, :n] = order[o:o + n]
            o += n
        self.cum = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.T, self.total = T, total
        # the packed projection [T, (H + 2 HK) D]; inputs are what the type holds
        x = rng.standard_normal((T, (H + 2 * HK) * D)) * spread
        x[:, rng.integers(0, x.shape[1], 3)] *= 8
        self.qkv = torch.from_numpy(x).to(DT[dt])
        xs = self.qkv.double().numpy()
        self.q = xs[:, :H * D].reshape(T, H, D)
        self.k = xs[:, H * D:(H + HK) * D].reshape(T, HK, D)
        self.v = xs[:, (H + HK) * D:].reshape(T, HK, D)
        self.cos = self.sin = None
        self.seq = np.repeat(np.arange(B), new)
        self.pos = np.concatenate([np.arange(p, p + n) for p, n in zip(past, new)] + [np.zeros(0)]).astype(np.int64)
        if rotary:
            half = half or D // 2
            ang = np.arange(max(total) + 1)[:, None] / 10000.0 ** (np.arange(half) / half)[None, :]
            self.cos, self.sin = (torch.from_numpy(f(ang)).to(DT[dt]) for f in (np.cos, np.sin))
        # a cache whose past is filled, and garbage (NaN scales) wherever nothing was written
        shape = (self.nb, HK, bs)
        self.codes = []
        for _ in range(2):
            c, s = quantise(rng.standard_normal(shape + (D,)).astype(np.float16).astype(np.float64), code)
            s = s.astype(np.float32).astype(np.float64)
            used = np.zeros(shape, bool)
            for b in range(B):
                for t in range(past[b]):
                    used[self.bt[b, t // bs], :, t % bs] = True
            s[~used] = np.nan
            self.codes.append((c, s))

    def cuda(self):
        t = {}
        for n, (c, s) in zip("kv", self.codes):
            x = torch.from_numpy(c)
            t[n + "c"] = (x.to(torch.int8) if self.code == "int8" else x.to(torch.float32).to(CODE[self.code])).cuda()
            t[n + "s"] = torch.from_numpy(s).to(torch.float32).cuda()
        qkv = self.qkv.cuda()
        H, HK, D = self.H, self.HK, self.D
        t["q"], t["k"], t["v"] = qkv.split([H * D, HK * D, HK * D], 1)
        for n in ("cum", "bt"):
            t[n] = torch.from_numpy(getattr(self, n)).cuda()
        t["past"] = torch.tensor(self.past, dtype=torch.int32).cuda()
        t["total"] = torch.tensor(self.total, dtype=torch.int32).cuda()
        t["cos"] = t["sin"] = None
        if self.cos is not None:
            t["cos"], t["sin"] = self.cos.cuda(), self.sin.cuda()
        return t

    def written(self):
        """Codes and scales of the new rows [T, HK, D], [T, HK] in 64 bits: (key, value)."""
        k = self.k
        if self.cos is not None:
            k = rotate(k, self.cos.double().numpy(), self.sin.double().numpy(), self.pos, self.inter)
        return quantise(k, self.code), quantise(self.v, self.code)

    def values(self, which, b, n):
        """Values [n, HK, D] of the first n positions, taken from the cache arrays in 64 bits."""
        c, s = self.codes[which]
        t = np.arange(n)
        page, off = self.bt[b, t // self.bs], t % self.bs
        return c[page, :, off] * s[page, :, off][..., None]

    def put(self, kv):
        for which, (c, s) in enumerate(kv):
            for i in range(self.T):
                p = int(self.pos[i])
                page = self.bt[self.seq[i], p // self.bs]
                self.codes[which][0][page, :, p % self.bs] = c[i]
                self.codes[which][1][page, :, p % self.bs] = s[i]

    def attend(self, scale=None):
        q = self.q
        if self.cos is not None:
            q = rotate(q, self.cos.double().numpy(), self.sin.double().numpy(), self.pos, self.inter)
        out = np.zeros((self.T, self.H, self.D))
        G = self.H // self.HK
        for i in range(self.T):
            n = int(self.pos[i]) + 1
            k, v = (self.values(w, self.seq[i], n) for w in (0, 1))
            s = np.einsum("hgd,nhd->hgn", q[i].reshape(self.HK, G, self.D), k) * (scale or self.D ** -0.5)
            p = np.exp(s - s.max(-1, keepdims=True))
            out[i] = np.einsum("hgn,nhd->hgd", p / p.sum(-1, keepdims=True), v).reshape(self.H, self.D)
        return out.reshape(self.T, -1)


def cache_of(t, case):
    return [(t[n + "c"].float().double().cpu().numpy(), t[n + "s"].double().cpu().numpy()) for n in "kv"]


def write(ops, t, case):
    ops.paged_kv_quantize(t["k"], t["v"], t["kc"], t["vc"], t["ks"], t["vs"], t["cum"], t["past"], t["bt"], t["cos"],
                          t["sin"], interleaved=case.inter)


# ---- writing ------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("HK,D,bs,new,past", [
    (8, 128, 16, [1], [0]),
    (2, 64, 24, [5, 1, 0, 33], [7, 0, 9, 100]),       # pages of 24; a sequence without new rows
    (3, 32, 4, [2, 9], [1, 3]),
    (1, 256, 64, [70], [63]),
])
def test_write_codes_exact(ops, code, dt, HK, D, bs, new, past):
    """Unrotated rows: 16-bit inputs give the codes and scales of the formula, all else in the cache stays."""
    c = Case(np.random.default_rng(D + bs), H=HK, HK=HK, D=D, bs=bs, new=new, past=past, dt=dt, code=code,
             rotary=False)
    t = c.cuda()
    before = cache_of(t, c)
    write(ops, t, c)
    got = cache_of(t, c)
    kv = c.written()
    for which in (0, 1):
        codes, scales = kv[which]
        touched = np.zeros(before[which][1].shape, bool)
        for i in range(c.T):
            page, off = c.bt[c.seq[i], c.pos[i] // bs], c.pos[i] % bs
            touched[page, :, off] = True
            if dt == "f32":  # x F is rounded: a code may fall on the other side of a rounding point
                step = np.maximum(np.abs(codes[i]) / 8, 1.0 if code == "int8" else 2.0 ** -9)
                assert (np.abs(got[which][0][page, :, off] - codes[i]) <= step).all()
                assert np.mean(got[which][0][page, :, off] != codes[i]) < 0.01
            else:
                np.testing.assert_array_equal(got[which][0][page, :, off], codes[i])
            np.testing.assert_allclose(got[which][1][page, :, off], scales[i], rtol=2.0 ** -23)
        np.testing.assert_array_equal(got[which][0][~touched], before[which][0][~touched])
        np.testing.assert_array_equal(got[which][1][~touched], before[which][1][~touched])


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dt,D,half,inter", [("f16", 128, 64, 0), ("bf16", 64, 32, 1), ("f32", 64, 16, 0),
                                             ("f16", 64, 12, 0), ("f16", 256, 100, 1), ("bf16", 32, 16, 0)])
def test_write_rotated(ops, code, dt, D, half, inter):
    """Rotated keys: each value within one code step of the rotated row (rotation is rounded in fp32)."""
    c = Case(np.random.default_rng(D + half), H=4, HK=2, D=D, bs=16, new=[9, 1], past=[11, 40], dt=dt, code=code,
             inter=inter, half=half)
    t = c.cuda()
    write(ops, t, c)
    got = cache_of(t, c)
    k, v = c.written()
    flips = 0
    for i in range(c.T):
        page, off = c.bt[c.seq[i], c.pos[i] // c.bs], c.pos[i] % c.bs
        for which, (codes, scales) in ((0, k), (1, v)):
            np.testing.assert_allclose(got[which][1][page, :, off], scales[i], rtol=1e-6)
            d = np.abs(got[which][0][page, :, off] - codes[i])
            step = np.maximum(np.abs(codes[i]) / 8, 1.0 if code == "int8" else 2.0 ** -9)
            assert (d <= step).all()
            flips += (d > 0).sum()
    assert flips <= 0.01 * c.T * 2 * c.HK * D


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_write_extreme_rows(ops, code, dt):
    """Rows of zeros, of the type's largest and smallest values, and with an infinity or a NaN."""
    D = 64
    x = torch.zeros(6, D, dtype=torch.float64)
    x[1] = torch.linspace(-1, 1, D) * 3e38
    x[2] = torch.linspace(-1, 1, D) * 2e-36
    x[3, 5], x[4, 7] = math.inf, math.nan
    x[5, 0] = -1.0
    rows = x.to(DT[dt]).cuda()
    kc = torch.zeros(1, 1, 8, D, device="cuda").to(CODE[code])
    vc, ks = kc.clone(), torch.full((1, 1, 8), 7.0, device="cuda")
    vs = ks.clone()
    i32 = dict(dtype=torch.int32, device="cuda")
    bt, cum, past = torch.zeros(1, 1, **i32), torch.tensor([0, 6], **i32), torch.zeros(1, **i32)
    ops.paged_kv_quantize(rows, rows, kc, vc, ks, vs, cum, past, bt)
    k, v = ops.paged_kv_dequantize(kc, vc, ks, vs, torch.tensor([6], **i32), bt, cap=6, dtype=torch.float32)
    assert torch.equal(torch.nan_to_num(k), torch.nan_to_num(v))
    got, src = k[0, 0].double().cpu(), rows.double().cpu()
    assert (got[0] == 0).all() and ks[0, 0, 0] == 0
    assert torch.isnan(got[3]).all() and torch.isnan(got[4]).all()
    for r in (1, 2, 5):
        step = src[r].abs().max() / F[code] * (1.0 if code == "int8" else 32.0)
        assert ((got[r] - src[r]).abs() <= 0.501 * step).all()
    assert got[5, 0] == -1.0 and (got[5, 1:] == 0).all()


# ---- reading back ---------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("HK,D,bs,past,extra", [
    (8, 128, 16, [1], 0), (2, 64, 24, [100, 0, 47, 1], 5), (1, 256, 8, [65, 64], 0), (5, 32, 3, [31, 32, 33], 31)])
def test_read_back(ops, code, dt, HK, D, bs, past, extra):
    c = Case(np.random.default_rng(D), H=HK, HK=HK, D=D, bs=bs, new=[0] * len(past), past=past, dt=dt, code=code,
             rotary=False)
    t = c.cuda()
    cap = max(past) + extra
    k, v = ops.paged_kv_dequantize(t["kc"], t["vc"], t["ks"], t["vs"], t["total"], t["bt"], cap=cap, dtype=DT[dt])
    for which, got in ((0, k), (1, v)):
        assert got.shape == (len(past), HK, cap, D) and got.dtype == DT[dt]
        for b, n in enumerate(past):
            want = torch.from_numpy(c.values(which, b, n).astype(np.float32)).transpose(0, 1)  # exact in fp32 and back
            assert torch.equal(got[b, :, :n].cpu(), want.to(DT[dt]))
            assert (got[b, :, n:] == 0).all()
    # into given buffers
    k2, v2 = torch.full_like(k, 9.0), torch.full_like(v, 9.0)
    ops.paged_kv_dequantize(t["kc"], t["vc"], t["ks"], t["vs"], t["total"], t["bt"], key=k2, value=v2)
    assert torch.equal(k, k2) and torch.equal(v, v2)


# ---- attention --------------------------------------------------------------------------------------------
def bound(dt, v):
    top = np.abs(v).max()
    return {"f16": 3 * 2.0 ** -11, "bf16": 2.0 ** -8 + 2.0 ** -10, "f32": 2.0 ** -17}[dt] * top


def run_attention(ops, t, c, append, **kw):
    return ops.paged_attention_quantized(
        t["q"], t["k"] if append else None, t["v"] if append else None, t["kc"], t["vc"], t["ks"], t["vs"], t["cum"],
        t["past"], t["bt"], t["cos"], t["sin"], num_heads=c.H, kv_heads=c.HK, interleaved=c.inter, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("H,HK,D,bs,new,past", [
    (32, 8, 128, 16, [1], [0]),                             # one key: the row itself
    (32, 8, 128, 16, [1, 1, 1], [1023, 31, 32]),            # unit borders
    (64, 8, 128, 32, [1, 1], [2047, 500]),                  # groups of 8
    (6, 2, 64, 24, [1, 1, 1, 1], [0, 300, 23, 24]),         # groups of 3, pages of 24
    (4, 4, 32, 5, [1, 1], [63, 200]),                       # one query head per kv head, pages of 5
    (16, 1, 64, 16, [1, 1], [777, 2]),                      # 16 heads share one kv head
    (28, 4, 128, 64, [1], [4999]),                          # groups of 7
    (48, 2, 128, 16, [1], [130]),                           # 24 heads: two chunks of 16
    (16, 2, 256, 16, [1, 1], [700, 0]),                     # head size 256
    (24, 1, 256, 8, [1], [90]),                             # head size 256, three chunks of 8
    (8, 2, 128, 16, [3, 1, 0, 40], [100, 9, 5, 0]),         # several new rows; a sequence without any
])
def test_attention(ops, code, dt, H, HK, D, bs, new, past):
    rng = np.random.default_rng(H * 131 + D + sum(past))
    c = Case(rng, H=H, HK=HK, D=D, bs=bs, new=new, past=past, dt=dt, code=code)
    t = c.cuda()
    out = run_attention(ops, t, c, True)
    c.codes = [(a, s) for a, s in cache_of(t, c)]  # what was written is tested above: attend to what the cache holds
    want = c.attend()
    used = np.concatenate([c.values(1, b, n).reshape(-1) for b, n in enumerate(c.total) if n])
    assert np.abs(out.double().cpu().numpy() - want).max() <= bound(dt, used)
    # the rows are in the cache by now: the same call without them, on scratch of its own
    ws = torch.full((ops.paged_attention_quantized_workspace_size(num_heads=H, kv_heads=HK, head_size=D),), 255,
                    dtype=torch.uint8, device="cuda")
    assert torch.equal(out, run_attention(ops, t, c, False, workspace=ws))
    assert torch.equal(out, run_attention(ops, t, c, False, workspace=ws))


@pytest.mark.gpu
@pytest.mark.parametrize("dt,D,half,inter,rotary", [
    ("f16", 64, 32, 1, True),      # pairs
    ("bf16", 128, 16, 0, True),    # part of the head rotated
    ("f16", 64, 12, 0, True),      # cos / sin rows off 16 bytes
    ("f32", 256, 100, 1, True),
    ("f16", 128, 64, 0, False),    # no RoPE
])
def test_attention_rotary_forms(ops, dt, D, half, inter, rotary):
    c = Case(np.random.default_rng(half), H=4, HK=2, D=D, bs=16, new=[1, 2], past=[37, 150], dt=dt, code="int8",
             inter=inter, half=half, rotary=rotary)
    t = c.cuda()
    out = run_attention(ops, t, c, True)
    c.codes = cache_of(t, c)
    v = np.concatenate([c.values(1, b, n).reshape(-1) for b, n in enumerate(c.total)])
    assert np.abs(out.double().cpu().numpy() - c.attend()).max() <= bound(dt, v)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f16", "f32"])
def test_rows_off_alignment(ops, dt):
    """Query, key and value rows that start off a 16-byte boundary, with an odd row stride; scales off one as well."""
    c = Case(np.random.default_rng(21), H=4, HK=2, D=64, bs=16, new=[1, 1, 1], past=[90, 3, 300], dt=dt, code="e4m3")
    t = c.cuda()
    want = {n: t[n].clone() for n in ("kc", "vc", "ks", "vs")}
    out = ops.paged_attention_quantized(t["q"].contiguous(), t["k"].contiguous(), t["v"].contiguous(), want["kc"],
                                        want["vc"], want["ks"], want["vs"], t["cum"], t["past"], t["bt"], t["cos"],
                                        t["sin"], num_heads=4, kv_heads=2)
    wide = torch.zeros(3, 8 * 64 + 7, dtype=DT[dt], device="cuda")
    wide[:, 1:8 * 64 + 1] = c.qkv.cuda()
    q, k, v = wide[:, 1:257], wide[:, 257:385], wide[:, 385:513]
    shifted = {}
    for n in ("ks", "vs"):
        flat = torch.zeros(t[n].numel() + 1, device="cuda")
        flat[1:] = t[n].reshape(-1)
        shifted[n] = flat[1:].view(t[n].shape)
    got = ops.paged_attention_quantized(q, k, v, t["kc"], t["vc"], shifted["ks"], shifted["vs"], t["cum"], t["past"],
                                        t["bt"], t["cos"], t["sin"], num_heads=4, kv_heads=2)
    assert torch.equal(out, got)
    assert torch.equal(want["kc"].view(torch.int8), t["kc"].view(torch.int8))
    assert torch.equal(torch.nan_to_num(want["ks"]), torch.nan_to_num(shifted["ks"]))


@pytest.mark.gpu
def test_cache_past_32_bit_offsets(ops):
    """Pages at the end of a cache of more than 2^32 bytes (and rows past 2^25): written, read back, attended to."""
    HK, D, bs = 4, 256, 32
    blocks = (1 << 32) // (HK * bs * D) + 40
    kc = torch.empty(blocks, HK, bs, D, dtype=torch.int8, device="cuda")
    vc, ks = torch.empty_like(kc), torch.empty(blocks, HK, bs, device="cuda")
    vs = torch.empty_like(ks)
    n = 70
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.randn(n, HK * D, device="cuda", generator=g).half() for _ in range(2))
    q = torch.randn(n, 2 * HK * D, device="cuda", generator=g).half()
    i32 = dict(dtype=torch.int32, device="cuda")
    bt = torch.tensor([[blocks - 1, 0, blocks - 20]], **i32)
    cum, past = torch.tensor([0, n], **i32), torch.zeros(1, **i32)
    out = ops.paged_attention_quantized(q, k, v, kc, vc, ks, vs, cum, past, bt, num_heads=2 * HK, kv_heads=HK)
    kr, vr = ops.paged_kv_dequantize(kc, vc, ks, vs, torch.tensor([n], **i32), bt, cap=n, dtype=torch.float32)
    for got, src in ((kr, k), (vr, v)):
        rows = src.float().view(n, HK, D).transpose(0, 1)
        assert ((got[0] - rows).abs() <= rows.abs().amax(-1, keepdim=True) * (0.5 / 127 + 1e-6)).all()
    x = q[-1].double().view(HK, 2, D)
    p = torch.softmax(torch.einsum("hgd,hnd->hgn", x, kr[0].double()) / 16.0, -1)
    o = torch.einsum("hgn,hnd->hgd", p, vr[0].double()).reshape(-1)
    assert (out[-1].double() - o).abs().max().item() <= bound("f16", vr.cpu().numpy())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f16", "f32"])
def test_attention_many_ragged_rows(ops, dt):
    """More rows than a CTA has threads, lengths from 1 to several units: every kind of split."""
    rng = np.random.default_rng(3)
    past = [int(x) for x in rng.integers(0, 150, 300)]
    c = Case(rng, H=4, HK=2, D=64, bs=16, new=[1] * 300, past=past, dt=dt, code="int8")
    t = c.cuda()
    out = run_attention(ops, t, c, True)
    c.codes = cache_of(t, c)
    v = np.concatenate([c.values(1, b, n).reshape(-1) for b, n in enumerate(c.total)])
    assert np.abs(out.double().cpu().numpy() - c.attend()).max() <= bound(dt, v)


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_attention_long(ops, code):
    """One sequence over every CTA (each row's parts are joined), scores with a wide spread, a given scale."""
    rng = np.random.default_rng(11)
    c = Case(rng, H=8, HK=1, D=128, bs=64, new=[1], past=[30011], dt="f16", code=code, spread=3.0)
    t = c.cuda()
    out = run_attention(ops, t, c, True, scale=0.2)
    c.codes = cache_of(t, c)
    assert np.abs(out.double().cpu().numpy() - c.attend(scale=0.2)).max() <= bound("f16", c.values(1, 0, 30012))


@pytest.mark.gpu
def test_attention_value_scales_far_apart(ops):
    """Value rows whose scales differ by many powers of two (the running exponent moves both ways)."""
    rng = np.random.default_rng(5)
    c = Case(rng, H=8, HK=2, D=64, bs=16, new=[1], past=[400], dt="f32", code="int8")
    c.codes[1][1][:] *= np.exp2(rng.integers(-40, 20, c.codes[1][1].shape)).astype(np.float32)
    t = c.cuda()
    out = run_attention(ops, t, c, True)
    c.codes = cache_of(t, c)
    assert np.abs(out.double().cpu().numpy() - c.attend()).max() <= bound("f32", c.values(1, 0, 401))


@pytest.mark.gpu
def test_attention_on_a_side_stream_and_in_a_graph(ops):
    rng = np.random.default_rng(6)
    c = Case(rng, H=32, HK=8, D=128, bs=16, new=[1, 1], past=[900, 77], dt="f16", code="int8")
    t = c.cuda()
    want = run_attention(ops, t, c, True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run_attention(ops, t, c, True)
        out = torch.zeros_like(got)
        ws = torch.empty(ops.paged_attention_quantized_workspace_size(num_heads=32, kv_heads=8, head_size=128),
                         dtype=torch.uint8, device="cuda")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            run_attention(ops, t, c, True, out=out, workspace=ws)
        graph.replay()
        graph.replay()
    s.synchronize()
    assert torch.equal(want, got) and torch.equal(want, out)


@pytest.mark.gpu
def test_bad_pages_and_positions_are_reported(ops, request):
    """A page outside the cache is skipped; a row past the table or the cos rows gives zeros."""
    rng = np.random.default_rng(7)
    c = Case(rng, H=4, HK=2, D=64, bs=8, new=[1, 1, 1], past=[20, 30, 9], dt="f16", code="int8")
    t = c.cuda()
    run_attention(ops, t, c, True)
    c.codes = cache_of(t, c)
    torch.cuda.synchronize()
    assert ops.device_error(clear=True)[0] == 0
    t["bt"][0, 1] = c.nb + 3                    # keys 8 .. 15 of sequence 0
    t["past"][1] = c.bt.shape[1] * 8 + 5        # past the table
    out = run_attention(ops, t, c, False)
    torch.cuda.synchronize()
    assert ops.device_error(clear=True)[0] == 122
    assert (out[1] == 0).all()
    want = c.attend().reshape(3, 4, 64)
    assert np.abs(out[2].double().cpu().numpy() - want[2].reshape(-1)).max() <= bound("f16", c.values(1, 2, 10))
    keep = [j for j in range(21) if not 8 <= j < 16]
    k, v = c.values(0, 0, 21)[keep], c.values(1, 0, 21)[keep]
    q = rotate(c.q, c.cos.double().numpy(), c.sin.double().numpy(), c.pos, 0)[0].reshape(2, 2, 64)
    s = np.einsum("hgd,nhd->hgn", q, k) / 8.0
    p = np.exp(s - s.max(-1, keepdims=True))
    o = np.einsum("hgn,nhd->hgd", p / p.sum(-1, keepdims=True), v).reshape(-1)
    assert np.abs(out[0].double().cpu().numpy() - o).max() <= bound("f16", v)
    t["past"][1] = c.cos.shape[0]               # inside the table, past the cos rows
    ops.paged_kv_quantize(t["k"], t["v"], t["kc"], t["vc"], t["ks"], t["vs"], t["cum"], t["past"], t["bt"], t["cos"],
                          t["sin"])
    torch.cuda.synchronize()
    assert ops.device_error(clear=True)[0] == 122


@pytest.mark.gpu
def test_prompt_in_chunks_matches_one_pass(ops):
    """A prompt taken in pieces (write, read back, GroupQueryAttention over the values) and a decode step over
    the pages see the same cache."""
    rng = np.random.default_rng(8)
    c = Case(rng, H=8, HK=2, D=64, bs=16, new=[50], past=[0], dt="f16", code="int8")
    t = c.cuda()
    whole = {n: t[n].clone() for n in ("kc", "vc", "ks", "vs")}
    ops.paged_kv_quantize(t["k"], t["v"], whole["kc"], whole["vc"], whole["ks"], whole["vs"], t["cum"], t["past"],
                          t["bt"], t["cos"], t["sin"])
    i32 = dict(dtype=torch.int32, device="cuda")
    for a, b in ((0, 7), (7, 8), (8, 50)):
        ops.paged_kv_quantize(t["k"][a:b], t["v"][a:b], t["kc"], t["vc"], t["ks"], t["vs"],
                              torch.tensor([0, b - a], **i32), torch.tensor([a], **i32), t["bt"], t["cos"], t["sin"])
    a = ops.paged_kv_dequantize(t["kc"], t["vc"], t["ks"], t["vs"], t["total"], t["bt"], cap=50)
    b = ops.paged_kv_dequantize(*(whole[n] for n in ("kc", "vc", "ks", "vs")), t["total"], t["bt"], cap=50)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


# ---- refusals (no GPU work: the checks come first) -----------------------------------------------------------
def _args(**kw):
    a = dict(q=torch.zeros(2, 4 * 64, dtype=torch.float16), k=torch.zeros(2, 2 * 64, dtype=torch.float16),
             kc=torch.zeros(4, 2, 8, 64, dtype=torch.int8), ks=torch.zeros(4, 2, 8),
             cum=torch.tensor([0, 1, 2], dtype=torch.int32), past=torch.zeros(2, dtype=torch.int32),
             bt=torch.zeros(2, 2, dtype=torch.int32), heads=4, kv=2, cos=None, sin=None)
    a.update(kw)
    return a


def _call(ops, a):
    return ops.paged_attention_quantized(a["q"], a["k"], a.get("v", a["k"]), a["kc"], a.get("vc", a["kc"]), a["ks"],
                                         a["ks"], a["cum"], a["past"], a["bt"], a["cos"], a["sin"],
                                         num_heads=a["heads"], kv_heads=a["kv"])


@pytest.mark.parametrize("kw,match", [
    (dict(kc=torch.zeros(4, 2, 8, 64, dtype=torch.float16)), "int8 or float8"),
    (dict(vc=torch.zeros(4, 2, 8, 64).to(torch.float8_e4m3fn)), "int8 or float8"),
    (dict(kc=torch.zeros(4, 2, 512, dtype=torch.int8)), "num_blocks, kv_heads"),
    (dict(ks=torch.zeros(4, 8, 2)), "scales"),
    (dict(ks=torch.zeros(4, 2, 8, dtype=torch.float16)), "scales"),
    (dict(kv=4), "kv heads"),
    (dict(q=torch.zeros(2, 100, dtype=torch.float16)), "query"),
    (dict(k=torch.zeros(3, 128, dtype=torch.float16)), "key"),
    (dict(k=torch.zeros(2, 128)), "key"),
    (dict(k=torch.zeros(2, 256, dtype=torch.float16)[:, ::2]), "contiguous"),
    (dict(v=None), "together"),
    (dict(bt=torch.zeros(2, 2, dtype=torch.int64)), "block_table"),
    (dict(cum=torch.tensor([0, 2], dtype=torch.int32)), "one entry more"),
    (dict(past=torch.zeros(2, dtype=torch.int64)), "past_seqlens"),
    (dict(cos=torch.zeros(9, 32, dtype=torch.float16)), "come together"),
    (dict(cos=torch.zeros(9, 32), sin=torch.zeros(9, 32)), "cos / sin"),
    (dict(), "one CUDA device"),
])
def test_refusals_of_the_binding(ops, kw, match):
    with pytest.raises(ValueError, match=match):
        _call(ops, _args(**kw))


def test_refusals_of_the_entry_points(ops):
    """The C entry points check before they launch: reachable without a GPU."""
    import ctypes

    from onnxruntime_ep_b200 import load_library

    L = ops._lib()
    assert L is load_library()

    def params(**kw):
        p = ops.PagedQ8Params()
        base = dict(batch=1, num_tokens=1, num_heads=4, kv_heads=2, head_size=64, num_blocks=4, block_size=8,
                    max_blocks=2, cache_type=3)
        base.update(kw)
        for k, v in base.items():
            setattr(p, k, v)
        return p

    def last():
        return L.b200ep_last_error().decode()

    one = ctypes.c_void_p(16)
    for kw, dtype, word in ((dict(head_size=80), 10, "head_size"), (dict(cache_type=2), 10, "cache_type"),
                            (dict(), 7, "dtype"), (dict(block_size=0), 10, "geometry"),
                            (dict(num_blocks=1 << 20, block_size=1 << 10, kv_heads=4), 10, "geometry"),
                            (dict(do_rotary=1, rotary_half=33, max_seq=9), 10, "rotary"),
                            (dict(num_heads=3), 10, "multiple"), (dict(batch=0), 10, "sequence"),
                            (dict(query_stride=10), 10, "strides"), (dict(), 10, "workspace")):
        p = params(**kw)
        rc = L.b200ep_paged_attention_quantized(ctypes.byref(p), *([one] * 13), dtype, None, 0, None)
        assert rc == 1 and word in last(), (kw, last())
    p = params()
    assert L.b200ep_paged_kv_quantize(ctypes.byref(p), *([None] * 11), 10, None) == 1 and "null" in last()
    assert L.b200ep_paged_kv_dequantize(ctypes.byref(p), *([one] * 8), -1, 10, None) == 1 and "cap" in last()
    assert L.b200ep_paged_attention_quantized(None, *([one] * 13), 10, None, 0, None) == 1
    p = params(num_tokens=0)
    assert L.b200ep_paged_kv_quantize(ctypes.byref(p), *([None] * 11), 10, None) == 0
    size = ops.paged_attention_quantized_workspace_size(num_heads=4, kv_heads=2, head_size=64)
    assert size > 0 and ops.paged_attention_quantized_workspace_size(num_heads=3, kv_heads=2, head_size=64) == 0
