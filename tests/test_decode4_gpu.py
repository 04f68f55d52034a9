"""The decode step over a 4-bit cache with 8-bit weights: the public operators one after the other
give the same bits; through FusedMLA and FusedDecoderStack, eagerly, captured and with evictions.
"""
import pytest
import torch

import ds_kernels
from mla_cache import LatentKVCache, LatentKVCache4

pytestmark = pytest.mark.gpu
bf16 = torch.bfloat16


def attn_weights(hidden, heads, positions, seed):
    from mla import FusedMLA
    import decoder
    g = torch.Generator(device="cuda").manual_seed(seed)
    cos, sin, scale = decoder.yarn_tables(positions, 40.0, "cuda")

    def w(*shape):
        return (torch.randn(*shape, generator=g, device="cuda") * 0.05).to(bf16)

    return FusedMLA.from_weights(w(heads * 192, hidden), w(576, hidden),
                                 torch.rand(512, generator=g, device="cuda") + 0.5,
                                 w(heads * 256, 512), w(hidden, heads * 128), cos, sin, scale, heads)


def by_operators(attn, x, cache, mass_decay):
    """The step from the public operators, the query's rotation in elementary ones."""
    w_dec, s_dec, w_out, s_out = attn.quantized_decode_weights()
    H, B = attn.heads, x.shape[0]
    proj = ds_kernels.int8_linear(x, w_dec, s_dec)
    q_pe = proj[:, H * 512:H * 576].view(B, H, 64).float()
    pos = cache.next_pos.long()
    c, s = attn.cos[pos].float()[:, None], attn.sin[pos].float()[:, None]
    a, b = q_pe[..., 0::2], q_pe[..., 1::2]
    rot = torch.cat([a * c[..., :32] - b * s[..., :32], b * c[..., 32:] + a * s[..., 32:]], -1).to(bf16)
    q = torch.cat([proj[:, :H * 512].view(B, H, 512), rot], -1)
    ds_kernels.mla_cache4_append(proj[:, None, H * 576:H * 576 + 512], proj[:, None, H * 576 + 512:], cache,
                                 attn.cos, attn.sin, attn.eps)
    o = ds_kernels.mla_decode_attention4(q, cache, attn.softmax_scale, mass_decay=mass_decay)
    return ds_kernels.int8_linear(o, w_out, s_out)


@pytest.mark.parametrize("heads,hidden,b", [(16, 256, 3), (1, 64, 1), (20, 512, 17), (16, 2048, 64)])
@pytest.mark.parametrize("mass_decay", [None, 0.5])
def test_step_is_its_operators(heads, hidden, b, mass_decay):
    attn = attn_weights(hidden, heads, 512, heads)
    g = torch.Generator(device="cuda").manual_seed(b)
    caches = [LatentKVCache4(b, 400) for _ in range(2)]
    lat = torch.randn(b, 300, 512, generator=g, device="cuda").to(bf16)
    kpe = torch.randn(b, 300, 64, generator=g, device="cuda").to(bf16)
    lens = torch.randint(0, 301, (b,), generator=g, device="cuda").to(torch.int32)
    for c in caches:
        ds_kernels.mla_cache4_append(lat, kpe, c, attn.cos, attn.sin, new_lens=lens)
    for _ in range(3):
        x = torch.randn(b, hidden, generator=g, device="cuda").to(bf16)
        y = attn.decode(x, caches[0], mass_decay=mass_decay)
        assert torch.equal(y, by_operators(attn, x, caches[1], mass_decay))
        for f in ("codes", "scales", "rstd", "pos", "mass", "state"):
            assert torch.equal(getattr(caches[0], f), getattr(caches[1], f)), f
    assert caches[0].next_pos.tolist() == (lens + 3).tolist() and caches[0].current_len == 303
    assert torch.isfinite(y).all()


def test_prefill_fills_the_cache_with_the_forward_s_latents():
    attn = attn_weights(256, 16, 512, 7)
    x = torch.randn(3, 200, 256, device="cuda").to(bf16)
    exact, c = LatentKVCache(3, 200), LatentKVCache4(3, 256)
    want = attn.prefill(x, exact)
    lens = torch.tensor([200, 1, 77], dtype=torch.int32, device="cuda")
    assert torch.equal(attn.prefill(x, c, prompt_lens=lens), want)
    ref = LatentKVCache4(3, 256)
    ds_kernels.mla_cache4_append(exact.kv_latent, exact.k_pe_cache, ref, attn.cos, attn.sin, attn.eps, new_lens=lens)
    for f in ("codes", "scales", "rstd", "pos", "state"):
        assert torch.equal(getattr(c, f), getattr(ref, f))
    with pytest.raises(RuntimeError, match="empty"):
        attn.prefill(x, c)
    with pytest.raises(NotImplementedError, match="4-bit"):
        attn.prefill(x, LatentKVCache(3, 200), prompt_lens=lens)
    with pytest.raises(NotImplementedError, match="4-bit"):
        attn.decode(x[:, 0], exact, mass_decay=1.0)


def test_refusals_of_the_step():
    attn = attn_weights(64, 4, 128, 8)
    c = LatentKVCache4(2, 128)
    x = torch.zeros(2, 64, dtype=bf16, device="cuda")
    w = attn.quantized_decode_weights()

    def step(x=x, w=w, cache=c, **kw):
        return ds_kernels.mla_decode4_step(x, *w, attn.cos, attn.sin, cache, 1.0, heads=4, **kw)

    for bad in (x.float(), x[:1], torch.zeros(2, 128, dtype=bf16, device="cuda")[:, ::2], x.cpu()):
        with pytest.raises(RuntimeError, match="mla_decode4_step"):
            step(x=bad)
    with pytest.raises(RuntimeError, match="w_dec"):
        step(w=(w[0][:-8], w[1], w[2], w[3]))
    with pytest.raises(RuntimeError, match="int8"):
        step(w=(w[0], w[1].half(), w[2], w[3]))
    with pytest.raises(RuntimeError, match="mass_decay"):
        step(mass_decay=1.5)
    c._bound = 128
    with pytest.raises(RuntimeError, match="overflow"):
        step()
    c._bound, c._seen = 5, 128
    with pytest.raises(RuntimeError, match="RoPE"):
        step()


@pytest.fixture(scope="module")
def stack():
    import decoder
    return decoder.random_stack(3, torch.device("cuda"), hidden=256, dense_inter=512, moe_inter=128, experts=8,
                                top_k=2, n_shared=1, positions=512, seed=3)


def test_stack_decodes_captures_and_evicts(stack):
    b = 3
    x = torch.randn(b, 64, 256, device="cuda").to(bf16)
    steps = [torch.randn(b, 256, device="cuda").to(bf16) for _ in range(40)]
    eager, graphed = (stack.new_caches(b, 96, bits=4) for _ in range(2))
    assert all(isinstance(c, LatentKVCache4) for c in eager)
    assert torch.equal(stack.prefill(x, eager), stack.prefill(x, graphed))
    with pytest.raises(ValueError, match="bits"):
        stack.new_caches(b, 8, bits=8)
    first = stack.capture_decode(steps[0], graphed, mass_decay=1.0)
    assert torch.equal(first, stack.decode_step(steps[0], eager, mass_decay=1.0))
    for i, s in enumerate(steps[1:]):
        if eager[0].remaining_capacity == 0:
            for caches in (eager, graphed):
                stack.evict(caches, 70, 16)
            assert eager[0].lens.tolist() == [70] * b
        want = stack.decode_step(s, eager, mass_decay=1.0)
        got = stack.replay_decode(s)
        # the same products, cut into other segments: 2^-7 of rounding
        assert (got.float() - want.float()).norm() <= 2.0 ** -6 * want.float().norm()
        assert torch.isfinite(got).all()
    assert graphed[0].current_len == eager[0].current_len and graphed[0].next_pos.tolist() == [64 + 40] * b
    with pytest.raises(RuntimeError, match="full"):
        for s in steps:
            stack.replay_decode(s)


def test_replays_stop_at_the_end_of_the_rope_tables(stack):
    caches = stack.new_caches(1, 32, bits=4)
    stack.prefill(torch.randn(1, 8, 256, device="cuda").to(bf16), caches)
    x = torch.randn(1, 256, device="cuda").to(bf16)
    stack.capture_decode(x, caches)
    for c in caches:                    # as many evictions later
        c._seen = 511
        c.next_pos.fill_(511)
    stack.replay_decode(x)
    with pytest.raises(RuntimeError, match="RoPE"):
        stack.replay_decode(x)
    caches[0].reset()
    caches[0]._seen = 3
    with pytest.raises(RuntimeError, match="empty"):
        stack.layers[0].attn.prefill(torch.randn(1, 4, 256, device="cuda").to(bf16), caches[0])


def test_steps_of_two_caches_captured_on_forked_streams():
    """Kernels that are set up under their predecessors, behind forks and joins of a capture."""
    b, heads, hidden = 4, 16, 256
    attn = attn_weights(hidden, heads, 512, 11)
    g = torch.Generator(device="cuda").manual_seed(12)
    x = torch.randn(2, b, hidden, generator=g, device="cuda").to(bf16)
    lat = torch.randn(b, 200, 512, generator=g, device="cuda").to(bf16)
    kpe = torch.randn(b, 200, 64, generator=g, device="cuda").to(bf16)
    w, s = attn.quantized_decode_weights()[2:]
    w2, s2 = ds_kernels.int8_quantize(torch.randn(hidden, hidden, generator=g, device="cuda").to(bf16))

    def caches():
        out = [LatentKVCache4(b, 400) for _ in range(2)]
        for c in out:
            ds_kernels.mla_cache4_append(lat, kpe, c, attn.cos, attn.sin)
        return out

    def both(cs, side):
        main = torch.cuda.current_stream()
        if side is not None:
            side.wait_stream(main)
        y0 = attn.decode(x[0], cs[0], mass_decay=1.0)
        with torch.cuda.stream(side if side is not None else main):
            cs[1].evict(150, 10)
            if side is None:    # a recorded call is cut for all slots: so is the eager one here
                cs[0]._bound = cs[1]._bound = 399
            y1 = attn.decode(x[1], cs[1], mass_decay=1.0)
        if side is not None:
            main.wait_stream(side)
        return ds_kernels.int8_linear(y0 + y1, w2, s2), y0, y1

    plain, forked = caches(), caches()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = both(forked, side)
    for _ in range(4):
        graph.replay()
        plain[0]._bound = 399
        for a, c in zip(got, both(plain, None)):
            assert torch.isfinite(a).all() and torch.equal(a, c)
        assert torch.equal(forked[0].state, plain[0].state) and torch.equal(forked[1].state, plain[1].state)
        assert torch.equal(forked[0].codes, plain[0].codes)
    assert forked[0].lens.tolist() == [204] * b and forked[1].lens.tolist() == [151] * b
    assert ds_kernels.device_status() == ds_kernels.DS_OK
