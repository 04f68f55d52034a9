"""FusedDecoderStack's calls of its layers, with stand-ins for them (no GPU needed)."""
import pytest
import torch

import decoder
import ds_kernels


class Attn:
    """An attention object with the call that the bf16 decode step has always made."""

    def __init__(self):
        self.calls = []

    def decode(self, hidden_states, cache, events=None):
        self.calls.append(cache)
        return hidden_states


class Attn4(Attn):
    def decode(self, hidden_states, cache, events=None, mass_decay=None):
        self.calls.append((cache, mass_decay))
        return hidden_states


def stack(attn, monkeypatch):
    monkeypatch.setattr(ds_kernels, "rms_norm", lambda x, w, eps: x)
    monkeypatch.setattr(ds_kernels, "rms_norm_residual", lambda a, x, w, eps: (a, x))
    w = torch.ones(4)
    return decoder.FusedDecoderStack([decoder.FusedDecoderLayer(attn, lambda x: x, w, w)])


def test_a_step_without_accumulation_makes_the_call_that_it_always_made(monkeypatch):
    attn = Attn()
    s = stack(attn, monkeypatch)
    x = torch.ones(2, 4)
    assert torch.equal(s.decode_step(x, ["cache"]), x)
    assert attn.calls == ["cache"]
    with pytest.raises(TypeError, match="mass_decay"):
        s.decode_step(x, ["cache"], mass_decay=1.0)


def test_a_step_with_accumulation_passes_the_decay_on(monkeypatch):
    attn = Attn4()
    s = stack(attn, monkeypatch)
    s.decode_step(torch.ones(2, 4), ["c"], mass_decay=0.5)
    s.decode_step(torch.ones(2, 4), ["c"], mass_decay=0.0)
    s.decode_step(torch.ones(2, 4), ["c"])
    assert attn.calls == [("c", 0.5), ("c", 0.0), ("c", None)]


def fused_mla():
    from mla import FusedMLA
    g = torch.Generator().manual_seed(1)

    def w(*shape):
        return torch.randn(*shape, generator=g).to(torch.bfloat16)

    return FusedMLA.from_weights(w(2 * 192, 32), w(576, 32), torch.ones(512), w(2 * 256, 512), w(32, 2 * 128),
                                 torch.ones(8, 64), torch.zeros(8, 64), 1.0, heads=2)


def test_the_8_bit_decode_weights_do_not_keep_the_bf16_ones_alive(monkeypatch):
    monkeypatch.setattr(ds_kernels, "int8_quantize", lambda w: [w.to(torch.int8), w[:, 0].float()])
    attn = fused_mla()
    q = attn.quantized_decode_weights()
    assert attn._dec_w is None and attn.quantized_decode_weights() is q
    # ones that a bf16 step (or its graph) already uses stay where they are
    attn = fused_mla()
    w = attn.decode_weights()
    attn.quantized_decode_weights()
    assert attn.decode_weights() is w
    assert all(torch.equal(a, b) for a, b in zip(fused_mla().quantized_decode_weights(), q))
