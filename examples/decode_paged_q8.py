"""Generate from a Llama-shaped int4 decoder over an 8-bit paged KV cache, with the kernel-level bindings.

    python examples/decode_paged_q8.py [--layers 4 --batch 4 --prompt 100 --new 32 --code int8]

Per layer: RMS norm and int4 projections (MatMulNBits); a prompt is taken in chunks — the sequence's past is read back
from its pages (paged_kv_dequantize), GroupQueryAttention attends to it and the chunk, and the chunk's rows are quantised
into the pages (paged_kv_quantize).  A decode step writes each sequence's new row and attends over the pages
(paged_attention_quantized).  The next tokens come from sample(), whose int64 ids are the next step's input.  Weights are
random, of the configuration's shape.
"""

from __future__ import annotations

import argparse
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if os.path.join(ROOT, "onnxruntime-mlx_b200") not in sys.path:
    sys.path.insert(0, os.path.join(ROOT, "onnxruntime-mlx_b200"))

import numpy as np  # noqa: E402
import torch  # noqa: E402

from onnxruntime_ep_b200 import ops  # noqa: E402
from onnxruntime_ep_b200.decoder import DecoderConfig, quantize_params, rotary_caches  # noqa: E402

CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


class PagedQ8Decoder:
    """Weights, pages and the lengths of `batch` sequences of up to `capacity` tokens."""

    def __init__(self, cfg: DecoderConfig, batch: int, capacity: int, block: int = 16, code: str = "int8"):
        self.cfg, self.batch, self.block = cfg, batch, block
        rng = np.random.default_rng(cfg.seed)
        H, HK, D, hid = cfg.heads, cfg.kv_heads, cfg.head_dim, cfg.hidden
        dev = "cuda"

        def linear(n, k):
            b, s, z = (torch.from_numpy(x.copy()).to(dev) for x in quantize_params(rng, n, k, cfg.block, np.float16))
            return ops.matmulnbits_prepack(b, s, z, K=k, N=n, block_size=cfg.block), n, k

        def norm():
            return torch.from_numpy(rng.uniform(0.8, 1.2, hid).astype(np.float16)).to(dev)

        self.layers = [dict(ln1=norm(), qkv=linear((H + 2 * HK) * D, hid), o=linear(hid, H * D), ln2=norm(),
                            gate_up=linear(2 * cfg.ffn, hid), down=linear(hid, cfg.ffn)) for _ in range(cfg.layers)]
        self.norm, self.lm_head = norm(), linear(cfg.vocab, hid)
        self.embed = torch.from_numpy(rng.standard_normal((cfg.vocab, hid)).astype(np.float16)).to(dev)
        self.cos, self.sin = (torch.from_numpy(x).to(dev) for x in rotary_caches(cfg.max_seq, D, cfg.rope_base, np.float16))
        # pages of all sequences, scattered over one pool
        width = -(-capacity // block)
        self.table = torch.from_numpy(rng.permutation(batch * width).astype(np.int32)).to(dev).view(batch, width)
        shape = (batch * width, HK, block, D)
        for layer in self.layers:
            for name in ("k", "v"):
                layer[name + "_cache"] = torch.zeros(shape, dtype=torch.int8, device=dev).view(CODES[code])
                layer[name + "_scales"] = torch.zeros(shape[:3], device=dev)
        self.past = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.one_each = torch.arange(batch + 1, dtype=torch.int32, device=dev)
        self.workspace = torch.empty(
            ops.paged_attention_quantized_workspace_size(num_heads=H, kv_heads=HK, head_size=D), dtype=torch.uint8,
            device=dev)

    def _linear(self, x, w):
        packed, n, k = w
        return ops.matmulnbits_prepacked(x, packed, K=k, N=n, block_size=self.cfg.block)

    def _cache(self, layer):
        return layer["k_cache"], layer["v_cache"], layer["k_scales"], layer["v_scales"]

    def _stack(self, ids, attend):
        """Rows of `ids` through all layers; attend(layer, qkv) -> attention rows.  Returns the normed hidden rows."""
        x, cfg = self.embed[ids], self.cfg
        residual = None
        for layer in self.layers:
            if residual is None:
                residual, h = x, ops.rms_norm(x, layer["ln1"], cfg.eps)
            else:
                h, residual = ops.skip_rms_norm(x, residual, layer["ln1"], cfg.eps)
            x = self._linear(attend(layer, self._linear(h, layer["qkv"])), layer["o"])
            h, residual = ops.skip_rms_norm(x, residual, layer["ln2"], cfg.eps)
            gate, up = self._linear(h, layer["gate_up"]).chunk(2, dim=-1)
            x = self._linear(torch.nn.functional.silu(gate) * up, layer["down"])
        return ops.skip_rms_norm(x, residual, self.norm, cfg.eps)[0]

    def prompt(self, sequence: int, ids, chunk: int = 64):
        """Take a prompt in chunks; returns the logits [vocab] after its last token."""
        cfg = self.cfg
        H, HK, D = cfg.heads, cfg.kv_heads, cfg.head_dim
        past = int(self.past[sequence])
        table = self.table[sequence:sequence + 1].contiguous()
        i32 = dict(dtype=torch.int32, device="cuda")
        for part in ids.split(chunk):
            S = part.numel()
            before, rows = torch.tensor([past], **i32), torch.tensor([0, S], **i32)
            last = torch.tensor([past + S - 1], **i32)

            def attend(layer, qkv):
                k, v = qkv[:, H * D:(H + HK) * D], qkv[:, (H + HK) * D:]
                keys, values = ops.paged_kv_dequantize(*self._cache(layer), before, table, cap=past + S)
                ops.paged_kv_quantize(k, v, *self._cache(layer), rows, before, table, self.cos, self.sin)
                return ops.group_query_attention(qkv[None], None, None, keys, values, last, self.cos, self.sin,
                                                 num_heads=H, kv_heads=HK)[0]

            hidden = self._stack(part, attend)
            past += S
        self.past[sequence] = past
        return self._linear(hidden[-1:], self.lm_head)[0]

    def step(self, ids):
        """One new token of every sequence; returns the logits [batch, vocab]."""
        cfg = self.cfg
        H, HK, D = cfg.heads, cfg.kv_heads, cfg.head_dim

        def attend(layer, qkv):
            q, k, v = qkv.split([H * D, HK * D, HK * D], dim=1)
            return ops.paged_attention_quantized(q, k, v, *self._cache(layer), self.one_each, self.past, self.table,
                                                 self.cos, self.sin, num_heads=H, kv_heads=HK,
                                                 workspace=self.workspace)

        hidden = self._stack(ids, attend)
        self.past += 1
        return self._linear(hidden, self.lm_head)


def generate(model: PagedQ8Decoder, prompts, new: int, temperature=0.8, top_k=50, top_p=0.95, min_p=0.0, seed=0):
    """`new` tokens after each prompt: (ids [batch, new], log-probabilities [batch, new])."""
    B, V = model.batch, model.cfg.vocab
    g = torch.Generator(device="cuda").manual_seed(seed)
    noise = torch.empty(B, V, device="cuda")
    rows = [torch.full((B,), v, dtype=t, device="cuda") for v, t in (
        (temperature, torch.float32), (top_k, torch.int32), (top_p, torch.float32), (min_p, torch.float32))]
    logits = torch.stack([model.prompt(b, ids) for b, ids in enumerate(prompts)])
    ids, logp = [], []
    for i in range(new):
        token, lp = ops.sample(logits, noise.exponential_(generator=g), *rows)
        ids.append(token)
        logp.append(lp)
        if i + 1 < new:
            logits = model.step(token)
    return torch.stack(ids, 1), torch.stack(logp, 1)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=100)
    ap.add_argument("--new", type=int, default=32)
    ap.add_argument("--code", choices=sorted(CODES), default="int8")
    a = ap.parse_args()
    cfg = DecoderConfig(layers=a.layers, hidden=1024, heads=16, kv_heads=4, head_dim=64, ffn=2816, vocab=32000)
    model = PagedQ8Decoder(cfg, a.batch, a.prompt + a.new, code=a.code)
    g = torch.Generator(device="cuda").manual_seed(1)
    prompts = torch.randint(0, cfg.vocab, (a.batch, a.prompt), device="cuda", generator=g)
    ids, logp = generate(model, prompts, a.new)
    for b in range(a.batch):
        print(f"sequence {b}: {ids[b].tolist()}  mean log-probability {logp[b].mean().item():.3f}")


if __name__ == "__main__":
    main()
