"""Cases for the serving operators over an 8-bit paged key-value cache, and for the choice of the
next token: what each pass is given, what it returns, and the operators in plain torch.

Operators (the library's entry points in onnxruntime_ep_b200.ops):
  paged_kv_quantize          rotates new key rows, quantises key and value rows to 8 bits with one
                             scale per token and kv head, and writes them into their cache pages
  paged_kv_dequantize        gathers sequences out of the pages as floating rows [B, HK, cap, D]
  paged_attention_quantized  attention of packed query rows over the pages
  sample                     temperature / top-k / top-p / min-p and the draw, from given noise

Cache layout: codes [num_blocks, HK, block_size, D] (int8 or float8_e4m3fn), scales float32
[num_blocks, HK, block_size]; value = code * scale, scale = amax / 127 (or 448).

Kinds of case:
  chunk   a chunk of new tokens is written, then the sequences are read back, as a prompt that is
          taken in pieces does; the outputs are the values that the cache stands for
  read    sequences are read back (for a prompt kernel, or to move them elsewhere)
  attend  one new token of each sequence attends to its cached keys
  sample  one token per row is drawn from the logits
"""

import math
import random

import numpy as np
import torch

own = False

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}
QMAX = {"int8": 127.0, "e4m3": 448.0}
CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def _ops():
    import os
    import sys

    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "onnxruntime-mlx_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    from onnxruntime_ep_b200 import ops

    return ops


# ---- the cases -----------------------------------------------------------------------------------
def listed():
    chunk = {"kind": "chunk", "heads": 32, "kv_heads": 8, "head": 128, "block": 16}
    attend = {"kind": "attend", "heads": 32, "kv_heads": 8, "head": 128, "block": 16}
    return [
        # a five-token question on a short past: the smallest write, where latency counts
        dict(chunk, name="chunk 5 on 12", batch=1, new=5, past=12, ragged=False, dtype="f16", code="int8"),
        # eight prompts of uneven lengths taken in chunks of up to 1024 behind pasts of up to 4096
        dict(chunk, name="chunk 8 x 1024 ragged", batch=8, new=1024, past=4096, ragged=True, dtype="bf16",
             code="e4m3", block=32),
        # one sequence of odd length read back, interactive use
        {"kind": "read", "name": "read 1 x 1000", "batch": 1, "kv_heads": 8, "head": 128, "block": 16, "past": 1000,
         "ragged": False, "dtype": "f16", "code": "int8"},
        # sixteen long sequences read back
        {"kind": "read", "name": "read 16 x 8192", "batch": 16, "kv_heads": 8, "head": 128, "block": 16,
         "past": 8192, "ragged": False, "dtype": "bf16", "code": "e4m3"},
        # one user, short context: latency
        dict(attend, name="attend 1 x 1024", batch=1, past=1024, ragged=False, dtype="f16", code="int8"),
        # a served batch with lengths all over the range, eight query heads to a kv head
        dict(attend, name="attend 16 x 4096 ragged", batch=16, heads=64, past=4096, ragged=True, dtype="bf16",
             code="e4m3", block=32),
        # one very long sequence: all the work lies along the cache
        dict(attend, name="attend 1 x 131072", batch=1, past=131072, ragged=False, dtype="f16", code="int8"),
        # a full serving batch at a long context: bandwidth
        dict(attend, name="attend 64 x 8192", batch=64, past=8192, ragged=False, dtype="f16", code="e4m3"),
        # 32-bit activations, head size 64, three query heads to a kv head, pages of 24 rows
        dict(attend, name="attend f32 7 x 1531", batch=7, heads=12, kv_heads=4, head=64, past=1531, ragged=True,
             dtype="f32", code="int8", block=24),
        # one user's next token from the 128256-word vocabulary of the decoder shape
        {"kind": "sample", "name": "sample 1 x 128256", "batch": 1, "vocab": 128256, "dtype": "f16",
         "mix": "k50p90"},
        # a served batch whose requests ask for different filters
        {"kind": "sample", "name": "sample 64 x 128256", "batch": 64, "vocab": 128256, "dtype": "f16",
         "mix": "mixed"},
        # a large batch over a smaller vocabulary, 32-bit logits
        {"kind": "sample", "name": "sample 256 x 32000", "batch": 256, "vocab": 32000, "dtype": "f32",
         "mix": "mixed"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    kind = rng.choice(["chunk", "read", "attend", "attend", "sample"])
    if kind == "sample":
        vocab = _log(rng, 1000, 128256)
        batch = _log(rng, 1, max(1, min(256, 8200000 // vocab)))
        return {"kind": kind, "batch": batch, "vocab": vocab, "dtype": rng.choice(["f16", "bf16", "f32"]),
                "mix": rng.choice(["k50p90", "p95", "minp", "plain", "mixed"])}
    kv = rng.choice([1, 2, 4, 8])
    head = rng.choice([64, 128, 128, 256])
    c = {"kind": kind, "kv_heads": kv, "head": head, "block": rng.choice([8, 16, 24, 32, 64, 128]),
         "ragged": rng.random() < 0.6, "dtype": rng.choice(["f16", "bf16", "f32"]),
         "code": rng.choice(["int8", "e4m3"]), "batch": _log(rng, 1, 64)}
    # tokens of a sequence, so that the whole cache stays below the largest listed one
    row = c["batch"] * kv * head
    most = {"chunk": 30e6, "read": 100e6, "attend": 400e6}[kind] / row
    c["past"] = _log(rng, 1, max(2, min(131072, most)))
    if kind == "read":
        return c
    c["heads"] = kv * rng.choice([1, 2, 3, 4, 7, 8, 16])
    if kind == "chunk":
        c["new"] = _log(rng, 1, max(2, min(2048, most / 2)))
    return c


# ---- inputs ----------------------------------------------------------------------------------------
def _lengths(case, g, most, least):
    if not case["ragged"]:
        return torch.full((case["batch"],), most, dtype=torch.int32)
    n = torch.empty(case["batch"]).uniform_(0, 1, generator=g).mul_(most - least + 1).long().clamp_(0, most - least)
    n = n.to(torch.int32) + least
    n[-1] = most
    return n


def _rows(shape, g, dtype=torch.float32):
    """Rows as projections give them: normal, with a few channels that are much larger."""
    x = torch.randn(shape, device="cuda", generator=g, dtype=torch.float32)
    lift = 1.0 + 6.0 * (torch.rand(shape[-1], device="cuda", generator=g) < 0.03)
    return x.mul_(lift).to(dtype)


def _codes(x, code):
    amax = x.abs().amax(-1)
    t = (x * QMAX[code]) / torch.where(amax > 0, amax, torch.ones_like(amax)).unsqueeze(-1)
    return (torch.round(t) if code == "int8" else t).to(CODE[code]), amax / QMAX[code]


def _cache(case, blocks, g):
    shape = (blocks, case["kv_heads"], case["block"], case["head"])
    parts = [[], []]
    step = max(1, (1 << 26) // (shape[1] * shape[2] * shape[3]))
    for i in range(2):
        for a in range(0, blocks, step):
            parts[i].append(_codes(_rows((min(step, blocks - a),) + shape[1:], g), case["code"]))
    (kc, ks), (vc, vs) = ((torch.cat([p[0].view(torch.int8) for p in q]).view(CODE[case["code"]]),
                           torch.cat([p[1] for p in q])) for q in parts)
    return kc, vc, ks, vs


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    h = torch.Generator().manual_seed(int(seed))
    if case["kind"] == "sample":
        return _prepare_sample(case, g, h)
    B, hk, D, bs = case["batch"], case["kv_heads"], case["head"], case["block"]
    dtype = DT[case["dtype"]]
    past = _lengths(case, h, case["past"], 1 if case["kind"] == "read" else 0)
    new = _lengths(case, h, case["new"], 1) if case["kind"] == "chunk" else torch.ones(B, dtype=torch.int32)
    if case["kind"] == "attend":  # `past` counts the keys that a row sees, its own among them
        past = (past - 1).clamp_(min=0)
    total = past + new if case["kind"] != "read" else past
    pages = (total + bs - 1) // bs
    width = int(pages.max())
    blocks = int(pages.sum()) + 1
    order = torch.randperm(blocks, generator=h)[: blocks - 1].to(torch.int32)
    table = torch.zeros(B, width, dtype=torch.int32)
    table[torch.arange(width)[None, :] < pages[:, None]] = order
    kc, vc, ks, vs = _cache(case, blocks, g)
    cap = int(total.max())
    s = {"case": case, "kc": kc, "vc": vc, "ks": ks, "vs": vs, "table": table.cuda(), "cap": cap,
         "total": total.cuda(), "past": past.cuda(), "dtype": dtype}
    if case["kind"] == "read":
        return s
    cum = torch.zeros(B + 1, dtype=torch.int32)
    cum[1:] = new.cumsum(0)
    s["cum"] = cum.cuda()
    T, H = int(cum[-1]), case["heads"]
    # the projections' packed output [T, (H + 2 HK) D]: query, key and value are slices of its rows
    qkv = _rows((T, (H + 2 * hk) * D), g, dtype)
    s["q"], s["k"], s["v"] = qkv.split([H * D, hk * D, hk * D], dim=1)
    angle = torch.arange(cap, device="cuda", dtype=torch.float64)[:, None] / (
        10000.0 ** (torch.arange(D // 2, device="cuda", dtype=torch.float64) / (D // 2)))[None, :]
    s["cos"], s["sin"] = angle.cos().to(dtype), angle.sin().to(dtype)
    # scratch that a serving loop keeps
    s["scratch"] = torch.empty(16 << 20, dtype=torch.uint8, device="cuda")
    return s


MIX = {"k50p90": [(0.8, 50, 0.9, 0.0)], "p95": [(1.0, 0, 0.95, 0.0)], "minp": [(1.2, 0, 1.0, 0.05)],
       "plain": [(1.0, 0, 1.0, 0.0)],
       "mixed": [(0.8, 50, 0.9, 0.0), (1.0, 0, 0.95, 0.0), (0.7, 40, 1.0, 0.0), (0.0, 0, 1.0, 0.0),
                 (1.2, 0, 1.0, 0.05), (1.0, 200, 0.8, 0.02), (1.0, 0, 1.0, 0.0), (0.6, 0, 0.9, 0.0)]}


def _prepare_sample(case, g, h):
    B, V = case["batch"], case["vocab"]
    # logits: a broad normal body with a few dozen candidates above it
    x = 2.0 * torch.randn(B, V, device="cuda", generator=g)
    at = torch.randint(0, V, (B, 40), device="cuda", generator=g)
    # (the largest where two fall on one token, so that the order of the writes does not matter)
    x.scatter_reduce_(1, at, 6.0 + 3.0 * torch.randn(B, 40, device="cuda", generator=g), "amax")
    rows = [MIX[case["mix"]][b % len(MIX[case["mix"]])] for b in range(B)]
    col = [torch.tensor(c, device="cuda") for c in zip(*rows)]
    noise = torch.empty(B, V, device="cuda").exponential_(generator=g).clamp_(min=1e-10)
    return {"case": case, "logits": x.to(DT[case["dtype"]]), "noise": noise, "temperature": col[0].float(),
            "top_k": col[1].to(torch.int32), "top_p": col[2].float(), "min_p": col[3].float()}


# ---- one pass ------------------------------------------------------------------------------------
def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    ops, case = _ops(), s["case"]
    if case["kind"] == "sample":
        return ops.sample(s["logits"], s["noise"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    if case["kind"] == "attend":
        return ops.paged_attention_quantized(
            s["q"], None, None, s["kc"], s["vc"], s["ks"], s["vs"], s["cum"], s["past"], s["table"], s["cos"],
            s["sin"], num_heads=case["heads"], kv_heads=case["kv_heads"], workspace=s["scratch"])
    if case["kind"] == "chunk":
        ops.paged_kv_quantize(s["k"], s["v"], s["kc"], s["vc"], s["ks"], s["vs"], s["cum"], s["past"], s["table"],
                              s["cos"], s["sin"])
    return ops.paged_kv_dequantize(s["kc"], s["vc"], s["ks"], s["vs"], s["total"], s["table"], cap=s["cap"],
                                   dtype=s["dtype"])


def _run_plain(s):
    kind = s["case"]["kind"]
    if kind == "sample":
        return _plain_sample(s)
    if kind == "attend":
        return _plain_attend(s)
    if kind == "chunk":
        _plain_write(s)
    return _plain_read(s)


def _rotate(x, s, pos):
    """x [T, heads, D] in 32 bits, halves (i, i + D/2) rotated by the angles of `pos`."""
    half = x.shape[-1] // 2
    c, d = s["cos"].float()[pos][:, None], s["sin"].float()[pos][:, None]
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * c - b * d, b * c + a * d], -1)


def _positions(s):
    at = torch.arange(s["q"].shape[0], device="cuda")
    seq = (at[:, None] >= s["cum"][None, 1:]).sum(1)
    return seq, (s["past"][seq] + at - s["cum"][seq]).long()


def _plain_write(s):
    hk, D, bs = s["case"]["kv_heads"], s["case"]["head"], s["case"]["block"]
    seq, pos = _positions(s)
    page, off = s["table"][seq, pos // bs].long(), pos % bs
    k = _rotate(s["k"].float().view(-1, hk, D), s, pos)
    for x, cache, scales in ((k, s["kc"], s["ks"]), (s["v"].float().view(-1, hk, D), s["vc"], s["vs"])):
        codes, scale = _codes(x, s["case"]["code"])
        cache.view(torch.int8)[page, :, off] = codes.view(torch.int8)
        scales[page, :, off] = scale


def _gather(s, cache, scales, n):
    """Values [B, HK, n, D] in 32 bits of the pages that the table names."""
    B, hk, D = s["table"].shape[0], cache.shape[1], cache.shape[3]
    at = s["table"].long()
    x = cache.view(torch.int8)[at].view(cache.dtype).float() * scales[at].unsqueeze(-1)
    return x.transpose(1, 2).reshape(B, hk, -1, D)[:, :, :n]


def _plain_read(s):
    inside = (torch.arange(s["cap"], device="cuda")[None, :] < s["total"][:, None])[:, None, :, None]
    return [torch.where(inside, _gather(s, c, f, s["cap"]), 0.0).to(s["dtype"])
            for c, f in ((s["kc"], s["ks"]), (s["vc"], s["vs"]))]


def _plain_attend(s):
    case, B = s["case"], s["q"].shape[0]
    hk, D = case["kv_heads"], case["head"]
    q = _rotate(s["q"].float().view(B, -1, D), s, s["past"].long()).view(B, hk, -1, D)
    score = torch.matmul(q, _gather(s, s["kc"], s["ks"], s["cap"]).transpose(2, 3)) / math.sqrt(D)
    hidden = torch.arange(s["cap"], device="cuda")[None, :] > s["past"][:, None]
    score = score.masked_fill(hidden[:, None, None, :], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    return torch.matmul(p, _gather(s, s["vc"], s["vs"], s["cap"])).view(B, -1).to(s["dtype"])


def _plain_sample(s):
    x = s["logits"].float()
    V = x.shape[1]
    value, index = torch.sort(x, dim=1, descending=True, stable=True)
    top = value[:, :1]
    greedy = s["temperature"] == 0
    t = torch.where(greedy, torch.ones_like(s["temperature"]), s["temperature"])
    k = torch.where(greedy, torch.ones_like(s["top_k"]), torch.where(s["top_k"] > 0, s["top_k"], V))
    rank = torch.arange(V, device=x.device)[None, :]
    w = torch.exp((value - top) / t[:, None])
    within = torch.where(rank < k[:, None], w, 0.0)
    before = within.cumsum(1) - within
    p = s["top_p"][:, None]
    keep = (rank < k[:, None]) & ((p >= 1) | (rank == 0) | (before < p * within.sum(1, keepdim=True)))
    keep &= w >= s["min_p"][:, None]
    key = torch.where(keep, w / s["noise"].gather(1, index), -1.0)
    best = key.amax(1, keepdim=True)
    token = torch.where(key == best, index, V).amin(1)
    logz = torch.log(torch.exp(x - top).sum(1))
    return token, x.gather(1, token[:, None])[:, 0] - top[:, 0] - logz


# ---- the work a pass cannot do without -------------------------------------------------------------
def _mean_total(case):
    """Tokens of all sequences; of ragged ones the mean (lengths are uniform, the last one is the longest)."""
    B = case["batch"]
    return lambda most, least: B * most if not case["ragged"] else (B - 1) * (most + least) / 2 + most


def work(case):
    if case["kind"] == "sample":
        B, V = case["batch"], case["vocab"]
        noise = [(k if k > 0 else V if p >= 1 and m == 0 else 0) if t > 0 else 0 for t, k, p, m in MIX[case["mix"]]]
        noise = sum(noise[b % len(noise)] for b in range(B))
        return {"bytes": B * V * SIZE[case["dtype"]] + 4 * noise + B * 28, "flops": 4 * B * V}
    B, hk, D, size = case["batch"], case["kv_heads"], case["head"], SIZE[case["dtype"]]
    count = _mean_total(case)
    row = 2 * hk * (D + 4)  # a token's codes and scales
    if case["kind"] == "attend":
        n = count(case["past"], 1)
        return {"bytes": n * row + 2 * B * case["heads"] * D * size, "flops": 4 * case["heads"] * D * n}
    if case["kind"] == "read":
        n = count(case["past"], 1)
        return {"bytes": n * row + 2 * B * hk * case["past"] * D * size, "flops": 2 * n * hk * D}
    new = count(case["new"], 1)
    n = new + count(case["past"], 0)
    values = 2 * B * hk * (case["past"] + case["new"]) * D * size
    return {"bytes": new * (2 * hk * D * size + row) + n * row + values, "flops": 10 * new * hk * D + 2 * n * hk * D}


# ---- the definitions in 64 bits ----------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"sample": _exact_sample, "attend": _exact_attend, "read": _exact_read, "chunk": _exact_read}[
        case["kind"]](s)


def _turned(x, s, pos):
    """Rows x [n, heads, D] at positions pos [n], as complex numbers turned by their angles, in 64 bits."""
    half = x.shape[-1] // 2
    turn = torch.complex(s["cos"].double(), s["sin"].double())[pos][:, None]
    z = torch.complex(x[..., :half].double(), x[..., half:].double()) * turn
    return torch.cat([z.real, z.imag], -1)


def _sequence(s, cache, scales, b, n):
    """Values [n, HK, D] of sequence b, in 64 bits."""
    pos = torch.arange(n, device="cuda")
    bs = cache.shape[2]
    page = s["table"][b, pos // bs].long()
    code = cache.view(torch.int8)[page, :, pos % bs].view(cache.dtype)
    return code.to(torch.float32).double() * scales[page, :, pos % bs].double()[..., None]


def _nearest_code(t, code):
    """t / qmax scaled values rounded to what 8 bits hold, ties to even, in 64 bits."""
    if code == "int8":
        return torch.round(t)
    _, e = torch.frexp(t)  # |t| in [2^(e-1), 2^e): steps of 2^(e-4), and of 2^-9 below 2^-6
    step = torch.exp2((e.double() - 4).clamp(min=-9))
    return torch.round(t / step) * step


def _exact_read(s):
    case = s["case"]
    B, hk, D, cap = case["batch"], case["kv_heads"], case["head"], s["cap"]
    out = []
    for x, cache, scales in (("k", s["kc"], s["ks"]), ("v", s["vc"], s["vs"])):
        y = torch.zeros(B, hk, cap, D, dtype=torch.float64, device="cuda")
        for b in range(B):
            past, total = int(s["past"][b]), int(s["total"][b])
            if case["kind"] == "chunk":
                lo, hi = int(s["cum"][b]), int(s["cum"][b + 1])
                rows = s[x][lo:hi].reshape(hi - lo, hk, D).double()
                if x == "k":
                    rows = _turned(rows, s, torch.arange(past, total, device="cuda"))
                amax = rows.abs().amax(-1, keepdim=True)
                full = QMAX[case["code"]]
                y[b, :, past:total] = (_nearest_code(rows / amax * full, case["code"]) * amax / full).transpose(0, 1)
            if past:
                y[b, :, :past] = _sequence(s, cache, scales, b, past).transpose(0, 1)
        out.append(y)
    return out


def _exact_attend(s):
    case = s["case"]
    hk, D, H = case["kv_heads"], case["head"], case["heads"]
    out = torch.empty(case["batch"], H * D, dtype=torch.float64, device="cuda")
    for b in range(case["batch"]):
        n = int(s["past"][b]) + 1
        q = _turned(s["q"][b].reshape(1, H, D), s, torch.tensor([n - 1], device="cuda"))[0].view(hk, H // hk, D)
        a = torch.einsum("hgd,nhd->hgn", q, _sequence(s, s["kc"], s["ks"], b, n)) * D ** -0.5
        out[b] = torch.einsum("hgn,nhd->hgd", torch.softmax(a, -1), _sequence(s, s["vc"], s["vs"], b, n)).reshape(-1)
    return out


def _exact_sample(s):
    x = s["logits"].double().cpu().numpy()
    noise = s["noise"].double().cpu().numpy()
    t, k, p, m = (s[n].cpu().numpy().astype(np.float64) for n in ("temperature", "top_k", "top_p", "min_p"))
    B, V = x.shape
    tokens, logp = np.empty(B, np.int64), np.empty(B)
    for b in range(B):
        order = np.argsort(-x[b], kind="stable")
        if t[b] == 0:
            token = order[0]
        else:
            count = V if k[b] <= 0 else min(V, int(k[b]))
            order = order[:count]
            mass = np.exp((x[b, order] - x[b, order[0]]) / t[b])
            if p[b] < 1:
                run_up = np.cumsum(mass)
                order = order[: max(1, int(np.searchsorted(run_up, p[b] * run_up[-1], side="left")) + 1)]
            order = np.sort(order[mass[: len(order)] >= m[b]])
            token = order[np.argmax(np.exp((x[b, order] - x[b].max()) / t[b]) / noise[b, order])]
        tokens[b] = token
        logp[b] = x[b, token] - x[b].max() - np.log(np.exp(x[b] - x[b].max()).sum())
    return torch.from_numpy(tokens), torch.from_numpy(logp)
