"""Plain restatement of the text layers that stream through the quantised cache:
the whole sequence at once in 64 bits, keys and values as the cache holds them,
and bf16 where the layers store a tensor (norms, QKV, attention, the residual
stream, the SwiGLU product)."""
import numpy as np
import torch

from . import kvcache_ref as R
from . import smolvla_ref as S

F64 = torch.float64

# Largest 2-norm of the error of what the layers add to their input, over the 2-norm of what
# they add, for two layers whose attention is as large as their input.  A layer stores six
# tensors in bf16, each off by at most 2^-9 of an element where two sums of other order round
# apart, about 2^-9 / sqrt(3) in the mean: sqrt(12) of these, and the scores double them at a
# spread of 2: 0.008.  A key that is one bf16 step off may round to the next code: in 8 bits
# (a step of about the group's largest value / 90) that is as small again, in 4 bits (a step
# of 1/7.5 of it, 0.3 of an element's rms) it happens to about 2^-9 / 0.3 = 0.7 % of the
# elements and costs sqrt(0.007) * 0.3 = 0.025 in keys, and the same in values.
LIMIT = {8: 0.02, 4: 0.05}


def strong_layers(params):
    """Layers whose scores spread (by about 2) and whose attention adds as much as their input."""
    grow = {"Wq": 5, "Wk": 5, "Wv": 4, "Wo": 4}
    return [{k: v * grow.get(k, 1) for k, v in p.items()} for p in params]


def _bf16(x):
    return x.to(torch.bfloat16).to(F64)


def seen(n, window, sinks):
    """[n, n]: whether the token of a row sees the key of a column."""
    i, j = torch.arange(n)[:, None], torch.arange(n)[None, :]
    return (j <= i) & ((j > i - window) | (j < sinks) if window else torch.ones(n, n, dtype=torch.bool))


def layers(x, params, cfg, bits, visible, positions=None):
    """x bf16 [B, n, hidden] through the layers: float64 [B, n, hidden]."""
    B, n, _ = x.shape
    G = cfg.heads // cfg.kv_heads
    x = x.to(F64)
    positions = torch.arange(n) if positions is None else positions
    held = lambda t: torch.from_numpy(R.held(t.numpy(), bits))  # noqa: E731
    for p in params:
        h = _bf16(S.rms_norm(x, p["W_norm_1"], cfg.eps, F64))
        q, k, v = (S.linear(h, p[w], dt=F64).view(B, n, -1, cfg.head_dim) for w in ("Wq", "Wk", "Wv"))
        q, k = (_bf16(S.apply_rope(t, cfg.rope_theta, positions.expand(B, n))) for t in (q, k))
        k, v = held(k), held(_bf16(v))
        k, v = (t.repeat_interleave(G, 2) for t in (k, v))
        s = torch.einsum("bihd,bjhd->bhij", q, k) / np.sqrt(cfg.head_dim)
        s = s.masked_fill(~visible, -torch.inf)
        o = _bf16(torch.einsum("bhij,bjhd->bihd", torch.softmax(s, -1), v).reshape(B, n, -1))
        x = _bf16(x + S.linear(o, p["Wo"], dt=F64))
        h = _bf16(S.rms_norm(x, p["W_norm_2"], cfg.eps, F64))
        gate = S.linear(h, p["W_gate"], dt=F64)
        x = _bf16(x + S.linear(_bf16(gate * torch.sigmoid(gate) * S.linear(h, p["W_up"], dt=F64)), p["W_down"], dt=F64))
    return x


def off(got, want, x):
    """The error of what was added to x, over what is to be added."""
    x = x.to(F64)
    return float((got.to(F64) - want).norm() / (want - x).norm())
