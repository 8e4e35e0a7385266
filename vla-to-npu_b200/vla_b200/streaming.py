"""Text layers over a stream of observations, on a quantised key/value cache.

The model's prefix (image, instruction and state tokens) is recomputed for every
observation, and each sees itself alone.  Here the text layers keep what they
saw: the new tokens' keys and values are quantised into a ``KVCache`` as the
layer makes them, and its queries attend over the cache, over everything or over
the instruction's first tokens and a window of recent ones.  The layers' weights,
products and norms are those of ``vla_llama_self_layer_bf16`` (RMSNorm, QKV with
RoPE, attention, output projection, RMSNorm, SwiGLU), with positions that go on
from step to step.  All streams take the same number of tokens in a step; the
cache holds ``max_len`` tokens of each, also those that a window has left behind.
The position is the host's, so a step is not one to capture and replay (the
cache's own calls are).

    python -m vla_b200.streaming --batch 8 --steps 20 --window 1130 --sinks 48
"""
from __future__ import annotations

from typing import Dict, Optional, Sequence

import torch

from . import _lib
from . import device as dev
from .configs import TextCfg
from .kvcache import KVCache
from .model import LlamaLayerWeights, rope_table

BF16 = torch.bfloat16


class StreamingText:
    """``layers`` text layers for ``batch`` streams that advance together.

    ``window`` = 0 keeps every token visible; otherwise a token sees the last
    ``window`` ones and the first ``sinks``.  ``max_len`` tokens fit a stream.
    Steps run on ``device``, on its current stream, whichever device is current."""

    def __init__(self, cfg: TextCfg, layers: Sequence[Dict[str, torch.Tensor]], batch: int, max_len: int, bits: int = 4,
                 window: int = 0, sinks: int = 0, device="cuda"):
        d = torch.device(device)
        self.cfg, self.batch, self.max_len, self.window, self.sinks = cfg, batch, max_len, window, sinks
        self.layers = [LlamaLayerWeights(p, cfg, d) for p in layers]
        self.cache = KVCache(batch, max_len, kv_heads=cfg.kv_heads, layers=len(self.layers), bits=bits, device=d)
        self.rope = rope_table(max_len, cfg.head_dim, cfg.rope_theta).to(d)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=d)
        self.pos = 0
        self.rows = 0

    def reset(self) -> None:
        self.lens.zero_()
        self.pos = 0

    def _allocate(self, rows: int) -> None:
        if rows == self.rows:
            return
        c, d = self.cfg, self.lens.device
        self.rows = rows
        self.h = torch.empty(rows, c.hidden, dtype=BF16, device=d)
        self.qkv = torch.empty(rows, c.q_dim + 2 * c.kv_dim, dtype=BF16, device=d)
        self.o = torch.empty(rows, c.q_dim, dtype=BF16, device=d)
        self.gu = torch.empty(rows, c.ffn, dtype=BF16, device=d)

    def step(self, x: torch.Tensor) -> torch.Tensor:
        """The next n tokens of every stream: x bfloat16 [batch * n, hidden] in
        place through all layers."""
        c, B, d = self.cfg, self.batch, self.lens.device
        if x.dim() != 2 or x.shape[1] != c.hidden or x.shape[0] % B or x.dtype != BF16 or x.device != d:
            raise ValueError(f"x: need bfloat16 [{B} * n, {c.hidden}] on {d}, got {x.dtype} {tuple(x.shape)} on {x.device}")
        n = x.shape[0] // B
        if self.pos + n > self.max_len:
            raise ValueError(f"{self.pos} + {n} tokens do not fit max_len {self.max_len}")
        if n == 0:
            return x
        with torch.cuda.device(d):  # the products and norms launch on the current device
            lens = self._advance(x, n)
        self.lens = lens
        self.pos += n
        return x

    def _advance(self, x: torch.Tensor, n: int) -> torch.Tensor:
        c, B = self.cfg, self.batch
        self._allocate(B * n)
        lens = self.lens + n
        q = self.qkv.view(B, n, -1)[:, :, :c.q_dim]
        k, v = self.qkv[:, c.q_dim:c.q_dim + c.kv_dim], self.qkv[:, c.q_dim + c.kv_dim:]
        rope = dev.make_epilogue(act=_lib.ACT_ROPE, rope_cs=self.rope[self.pos:self.pos + n], rope_seq=n,
                                 rope_ncols=c.q_dim + c.kv_dim, b_static=True)
        add = dev.make_epilogue(residual=x, b_static=True)
        for i, lw in enumerate(self.layers):
            dev.rms_norm(x, lw.norm1, c.eps, out=self.h)
            dev.gemm(self.h, lw.w_qkv, self.qkv, rope)
            self.cache.append(k, v, self.lens, n, layer=i)
            self.cache.attend(q, lens, window=self.window, sinks=self.sinks, max_len=self.pos + n, layer=i,
                              out=self.o.view(B, n, -1))
            dev.gemm(self.o, lw.w_o, x, add)
            dev.rms_norm(x, lw.norm2, c.eps, out=self.h)
            dev.gemm(self.h, lw.w_gu, self.gu, dev.make_epilogue(act=_lib.ACT_SWIGLU, b_static=True))
            dev.gemm(self.gu, lw.w_down, x, add)
        return lens

    def held(self, layer: int, first: int = 0, n: Optional[int] = None):
        """The keys and values that a layer's cache stands for, bfloat16
        [batch, n, kv_dim] each, tokens first .. first + n (all up to now)."""
        n = self.pos - first if n is None else n
        if first < 0 or n < 0 or first + n > self.pos:
            raise ValueError(f"tokens {first} .. {first + n}: {self.pos} are held")
        return self.cache.read(n, start=torch.full_like(self.lens, first), layer=layer)


def main(argv=None) -> None:
    """Streams random prefixes through seeded text layers on cuda:0 and reports the
    time per step, the cache's size against bfloat16, and how far the last layer's
    held keys are from the ones written."""
    import argparse
    from . import weights as W
    ap = argparse.ArgumentParser(description=main.__doc__)
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--tokens", type=int, default=113, help="tokens of one observation's prefix")
    ap.add_argument("--layers", type=int, default=16)
    ap.add_argument("--bits", type=int, default=4, choices=(4, 8))
    ap.add_argument("--window", type=int, default=0)
    ap.add_argument("--sinks", type=int, default=0)
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args(argv)
    cfg = TextCfg()
    text = StreamingText(cfg, [W.text_block_params(cfg, seed=a.seed, layer=i) for i in range(a.layers)], a.batch,
                         a.tokens * a.steps, a.bits, a.window, a.sinks)
    gen = torch.Generator(device="cuda").manual_seed(a.seed)
    ms = []
    for _ in range(a.steps):
        x = torch.randn(a.batch * a.tokens, cfg.hidden, generator=gen, device="cuda", dtype=BF16)
        t0, t1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        t0.record()
        text.step(x)
        t1.record()
        t1.synchronize()
        ms.append(t0.elapsed_time(t1))
    dev.sync_check()
    held = text.held(a.layers - 1, text.pos - a.tokens)[0].flatten(0, 1).float()
    wrote = text.qkv[:, cfg.q_dim:cfg.q_dim + cfg.kv_dim].float()
    plain = 2 * 2 * cfg.kv_dim * a.batch * text.pos * a.layers
    mine = text.cache.pool.numel()
    print(f"{a.batch} streams x {text.pos} tokens, {a.layers} layers, {a.bits} bits: {sorted(ms)[len(ms) // 2]:.2f} ms a step (median), "
          f"last {ms[-1]:.2f} ms; cache {mine / 2**20:.1f} MiB ({plain / 2**20:.1f} in bfloat16); "
          f"held keys off by {(held - wrote).norm() / wrote.norm():.4f}")


if __name__ == "__main__":
    main()
