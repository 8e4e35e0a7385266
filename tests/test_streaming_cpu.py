"""The streaming text layers without a GPU: where their calls go, by stand-ins that
record the device that is current when each is made."""
from types import SimpleNamespace

import pytest
import torch

from vla_b200 import streaming
from vla_b200.configs import TextCfg

BF16 = torch.bfloat16


class Devices:
    """torch.cuda.device in place of the real one: the devices entered, innermost last."""

    def __init__(self):
        self.entered = ["the caller's"]

    def __call__(self, d):
        outer = self

        class Guard:
            def __enter__(self):
                outer.entered.append(d)

            def __exit__(self, *_):
                outer.entered.pop()
        return Guard()


@pytest.fixture
def stream(monkeypatch):
    """A StreamingText of two layers on stand-ins, and the list of its calls with their device."""
    devices, calls = Devices(), []
    note = lambda name: lambda *a, **k: calls.append((name, devices.entered[-1]))  # noqa: E731
    cache = SimpleNamespace(append=note("append"), attend=note("attend"), read=note("read"))
    layer = SimpleNamespace(**{w: None for w in ("norm1", "norm2", "w_qkv", "w_o", "w_gu", "w_down")})
    monkeypatch.setattr(torch.cuda, "device", devices)
    monkeypatch.setattr(streaming, "KVCache", lambda *a, **k: cache)
    monkeypatch.setattr(streaming, "LlamaLayerWeights", lambda *a, **k: layer)
    monkeypatch.setattr(streaming, "dev", SimpleNamespace(
        rms_norm=note("rms_norm"), gemm=note("gemm"), make_epilogue=lambda **k: None))
    cfg = TextCfg(hidden=192, heads=6, kv_heads=2, head_dim=64, ffn=320, layers=2)
    return streaming.StreamingText(cfg, [{}, {}], 2, 10, device="cpu"), calls, devices


def test_every_launch_of_a_step_is_made_under_its_own_device(stream):
    text, calls, devices = stream
    text.step(torch.zeros(2 * 3, 192, dtype=BF16))
    assert [c for c, _ in calls].count("gemm") == 8 and [c for c, _ in calls].count("attend") == 2
    assert {d for _, d in calls} == {torch.device("cpu")}, "a launch went to the device that was current"
    assert devices.entered == ["the caller's"] and text.pos == 3 and text.lens.tolist() == [3, 3]


def test_rows_of_another_device_are_refused(stream):
    text, calls, _ = stream
    with pytest.raises(ValueError, match="meta"):
        text.step(torch.zeros(2 * 3, 192, dtype=BF16, device="meta"))
    assert not calls and text.pos == 0


def test_tokens_that_are_not_held_are_refused(stream):
    text, calls, _ = stream
    text.step(torch.zeros(2 * 3, 192, dtype=BF16))
    for first, n in ((0, 4), (2, 2), (-1, 2), (4, None), (0, -1)):
        with pytest.raises(ValueError, match="tokens"):
            text.held(0, first, n)
    assert "read" not in [c for c, _ in calls]
    text.held(0, 1)
    text.held(1, 3, 0)
    assert [c for c, _ in calls].count("read") == 2


STEPS = (1, 49, 1, 98, 1)


def strong():
    from oracle import streaming_ref as O
    from vla_b200 import weights as W
    cfg = TextCfg(hidden=192, heads=6, kv_heads=2, head_dim=64, ffn=320, layers=2)
    gen = torch.Generator().manual_seed(2)
    return cfg, O.strong_layers([W.text_block_params(cfg, seed=4, layer=i) for i in range(2)]), \
        torch.randn(3, sum(STEPS), cfg.hidden, generator=gen).to(BF16)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 10)])
def test_mistakes_of_a_streaming_step_exceed_the_limit(bits, window, sinks):
    """Mistakes planted in the restatement are far above the limit that the layers are held to on the GPU."""
    from oracle import streaming_ref as O
    cfg, params, x = strong()
    n = x.shape[1]
    visible = O.seen(n, window, sinks)
    want = O.layers(x, params, cfg, bits, visible)
    assert 0.5 < float((want - x.double()).norm() / x.double().norm()) < 4  # the layers' part is no trifle
    step = torch.repeat_interleave(torch.arange(len(STEPS)), torch.tensor(STEPS))
    first = torch.cat([torch.tensor([0]), torch.tensor(STEPS).cumsum(0)[:-1]])[step]
    same = step[:, None] == step[None, :]
    i, j = torch.arange(n)[:, None], torch.arange(n)[None, :]
    swapped = [{**p, "Wk": p["Wk"].roll(64, 1), "Wv": p["Wv"].roll(64, 1)} for p in params]
    mistakes = {
        "positions from 0 in every step": O.layers(x, params, cfg, bits, visible, torch.arange(n) - first),
        "own step only": O.layers(x, params, cfg, bits, visible & same),
        "own step not causal": O.layers(x, params, cfg, bits, visible | (same & (j < i + 20))),
        "a token later": O.layers(x, params, cfg, bits, visible & (j < i) | (i == j) & (i == 0)),
        "equal scores": O.layers(x, [{**p, "Wq": p["Wq"] * 0} for p in params], cfg, bits, visible),
        "heads swapped": O.layers(x, swapped, cfg, bits, visible),
        "no attention": O.layers(x, [{**p, "Wo": p["Wo"] * 0} for p in params], cfg, bits, visible),
    }
    if window:
        mistakes["no window"] = O.layers(x, params, cfg, bits, O.seen(n, 0, 0))
        mistakes["no sinks"] = O.layers(x, params, cfg, bits, O.seen(n, window, 0))
    offs = {name: O.off(got, want, x) for name, got in mistakes.items()}
    assert min(offs.values()) > 2 * O.LIMIT[bits], offs
