"""Text layers that stream through the quantised cache, against the same layers
over the whole sequence at once."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def small():
    from vla_b200 import weights as W
    from vla_b200.configs import TextCfg
    cfg = TextCfg(hidden=192, heads=6, kv_heads=2, head_dim=64, ffn=320, layers=2)
    return cfg, [W.text_block_params(cfg, seed=4, layer=i) for i in range(2)]


def whole(cfg, params, x, batch, seq):
    from vla_b200 import device as dev
    from vla_b200.model import LlamaLayerWeights, rope_table
    ws, rope = dev.Workspace("cuda"), rope_table(seq, 64, cfg.rope_theta).cuda()
    x = x.clone()
    for p in params:
        lw = LlamaLayerWeights(p, cfg, "cuda")
        dev.llama_self_layer(lw.struct, x, batch, seq, rope, ws)
    return x


# A group's values lie within its largest magnitude a; the step of its codes is at most a / 63.5 (8 bits: the
# power of two may be up to twice a / 127) or a / 7.5 (4 bits: a / 8 rounded up to 5 significant bits).  A rounding
# is off by at most half of it, for 32 normal values (a about 2.2 rms) 0.9 % and 9 % of the values' rms in the mean.
# What the layer adds to its input is off by no more than that in keys and values together; the residual shrinks it.
@pytest.mark.parametrize("bits,most", [(8, 0.02), (4, 0.2)])
def test_steps_agree_with_the_whole_sequence(cuda, bits, most):
    from vla_b200 import device as dev
    from vla_b200.streaming import StreamingText
    cfg, params = small()
    B, seq = 3, 150
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(B, seq, cfg.hidden, generator=gen).to(BF16).cuda()
    want = whole(cfg, params, x.view(B * seq, -1), B, seq).view(B, seq, -1).float()
    text = StreamingText(cfg, params, B, seq, bits=bits)
    for _ in range(2):  # again after a reset
        got, at = [], 0
        for n in (1, 49, 1, 98, 1):
            part = x[:, at:at + n].reshape(B * n, -1).clone()
            got.append(text.step(part).view(B, n, -1))
            at += n
        got = torch.cat(got, 1).float()
        assert (got - want).norm() / want.norm() < most
        assert (got[:, :1] - want[:, :1]).norm() / want[:, :1].norm() < most
        text.reset()
    dev.sync_check()


def test_a_window_as_long_as_the_stream_changes_nothing_and_a_short_one_does(cuda):
    from vla_b200.streaming import StreamingText
    cfg, params = small()
    gen = torch.Generator().manual_seed(3)
    xs = [torch.randn(2 * 40, cfg.hidden, generator=gen).to(BF16).cuda() for _ in range(3)]

    def run(**kw):
        text = StreamingText(cfg, params, 2, 120, bits=8, **kw)
        return torch.cat([text.step(x.clone()) for x in xs])

    full = run()
    assert torch.equal(full, run(window=120))
    assert torch.equal(full, run(window=40, sinks=120))
    short = run(window=20)
    assert torch.equal(full[:40][:20], short[:40][:20])  # stream 0's first 20 tokens lose nothing
    assert not torch.equal(full, short)


def test_streaming_refusals_and_held(cuda):
    from vla_b200.streaming import StreamingText
    cfg, params = small()
    text = StreamingText(cfg, params, 2, 10)
    x = torch.zeros(2 * 6, cfg.hidden, dtype=BF16, device="cuda")
    text.step(x)
    k, v = text.held(1, 2)
    assert k.shape == (2, 4, 128) and v.shape == (2, 4, 128)
    for bad in (x, x.float()[:4], x[:3], x[:4, :8]):
        with pytest.raises(ValueError):
            text.step(bad)
    assert text.step(x[:0]).shape == (0, cfg.hidden) and text.pos == 6


def test_command_line_example_runs(cuda, capsys):
    from vla_b200 import streaming
    streaming.main(["--batch", "2", "--steps", "3", "--layers", "2", "--window", "200", "--sinks", "48"])
    out = capsys.readouterr().out
    assert "2 streams x 339 tokens" in out and "held keys off by 0.0" in out


def test_held_refuses_tokens_that_are_not_there(cuda):
    from vla_b200.streaming import StreamingText
    cfg, params = small()
    text = StreamingText(cfg, params, 2, 10)
    text.step(torch.zeros(2 * 6, cfg.hidden, dtype=BF16, device="cuda"))
    assert text.held(0)[0].shape == (2, 6, 128) and text.held(0, 6)[0].shape == (2, 0, 128)
    for first, n in ((0, 7), (5, 2), (-1, 3), (7, None), (0, -1)):
        with pytest.raises(ValueError, match="tokens"):
            text.held(0, first, n)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 10)])
def test_what_steps_add_is_what_the_restatement_adds(cuda, bits, window, sinks):
    """Layers whose attention weighs as much as their input, in uneven steps, against the whole sequence at once with
    the cache's rounding; the limit is far below what a mistake costs (test_streaming_cpu.py)."""
    from oracle import streaming_ref as O
    from test_streaming_cpu import STEPS, strong
    from vla_b200 import device as dev
    from vla_b200.streaming import StreamingText
    cfg, params, x = strong()
    B, seq = x.shape[:2]
    want = O.layers(x, params, cfg, bits, O.seen(seq, window, sinks))
    text = StreamingText(cfg, params, B, seq, bits=bits, window=window, sinks=sinks)
    got, at = [], 0
    for n in STEPS:
        got.append(text.step(x[:, at:at + n].reshape(B * n, -1).cuda()).view(B, n, -1))
        at += n
    assert O.off(torch.cat(got, 1).cpu(), want, x) < O.LIMIT[bits]
    dev.sync_check()
