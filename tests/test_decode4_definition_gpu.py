"""The decode step over a 4-bit cache with 8-bit weights against the attention's definition in 64 bits, from
the raw (unabsorbed) weights: what the step composes, not only how well its parts do.

Weights and inputs are chosen so that every quantisation but one is exact, and the step may be held to the
definition instead of to the quantisation's noise:

* inputs have one entry that is not zero, a power of two: 127 in 8 bits, zeros elsewhere;
* projection rows are whole numbers of up to 7 and one entry of 127 (in a column that no input touches), so
  8 bits hold them exactly, as do the absorbed rows: w_uk and w_uv pick one row for each latent dimension, with
  a sign, and the latent norm's weights are 1 and 2;
* so latents and k_pe are whole numbers up to 7 times a power of two with a 7 in each group of each token, and
  the rotations are quarter turns, other ones at every position and frequency: 4 bits hold them exactly;
* output rows have three entries that are not zero, the largest 127, the others even and below 63.

What is left: the latent outputs o = sum p v and A = sum p |v| carry the attention's error (the tolerance at the
head of test_cache4_gpu.py, and 2^-18 A for the row scale rstd); they go to 8 bits, off by at most a / 254 with a
the row's largest, and the result is rounded to bf16 once (2^-8).
"""
import pytest
import torch

import ds_kernels
import oracle
from mla_cache import LatentKVCache4

pytestmark = pytest.mark.gpu
bf16, f64 = torch.bfloat16, torch.float64
SCALE = 1 / 64


def whole(g, *shape):
    return torch.randint(-7, 8, shape, generator=g).double()


def with_sevens(n, g):
    """n [..., 576] with a 7 or -7 in each group of each token"""
    flat = n.view(-1, 576)
    for lo, size in ((0, 128), (128, 128), (256, 128), (384, 128), (512, 64)):
        at = lo + torch.randint(0, size, (flat.shape[0],), generator=g)
        flat[torch.arange(flat.shape[0]), at] = 7 * signs(g, flat.shape[0])
    return flat.view(n.shape)


def signs(g, *shape):
    return torch.randint(0, 2, shape, generator=g).double() * 2 - 1


def layer(heads, hidden, positions, seed):
    """The raw weights in 64 bits, as FusedMLA.from_weights takes them."""
    g = torch.Generator().manual_seed(seed)
    norm = 1.0 + torch.randint(0, 2, (128,), generator=g).double().repeat_interleave(4)       # [512]
    w_q = whole(g, heads * 192, hidden)
    w_kva = with_sevens(whole(g, hidden, 576), g).t().contiguous()
    w_q[:, -1], w_kva[:, -1] = 127, 127
    w_kvb = torch.zeros(heads, 256, 512, dtype=f64)
    d = torch.arange(512)
    for h in range(heads):
        for base in (0, 128):                  # w_uk, w_uv: four latent dimensions a row
            pick = torch.randperm(128, generator=g)[d // 4]
            w_kvb[h, base + pick, d] = signs(g, 512)
    w_o = torch.zeros(hidden, heads * 128, dtype=f64)
    for n in range(hidden):
        at = torch.randperm(heads * 128, generator=g)[:3]
        w_o[n, at] = torch.tensor([127.0, 2.0 * torch.randint(1, 32, (1,), generator=g).item(),
                                   -2.0 * torch.randint(1, 32, (1,), generator=g).item()], dtype=f64)
    turn = torch.randint(0, 4, (positions, 32), generator=g)
    cos = torch.tensor([1.0, 0.0, -1.0, 0.0])[turn].repeat(1, 2)
    sin = torch.tensor([0.0, 1.0, 0.0, -1.0])[turn].repeat(1, 2)
    return w_q, w_kva, norm, w_kvb.view(-1, 512), w_o, cos, sin


def step64(x, past, w, heads, eps):
    """One sequence: x [hidden], past [n, 576] (raw latent, raw k_pe): probabilities, latent outputs and
    their tolerance, by elementary operations."""
    w_q, w_kva, norm, w_kvb, _, cos, sin = w
    raw = torch.cat([past, (w_kva @ x)[None]])
    n = raw.shape[0]

    def rot(v, pos):
        a, b, c, s = v[..., 0::2], v[..., 1::2], cos[pos].double(), sin[pos].double()
        return torch.cat([a * c[..., :32] - b * s[..., :32], b * c[..., 32:] + a * s[..., 32:]], -1)

    lat = raw[:, :512] * (raw[:, :512].square().mean(1, keepdim=True) + eps).rsqrt()
    kpe = rot(raw[:, 512:], torch.arange(n))
    q = (w_q @ x).view(heads, 192)
    uk, uv = w_kvb.view(heads, 256, 512)[:, :128], w_kvb.view(heads, 256, 512)[:, 128:]
    k = torch.einsum("hjd,td->htj", uk, lat * norm)
    qpe = rot(q[:, 128:], torch.full((heads,), n - 1))
    s = SCALE * (torch.einsum("hj,htj->ht", q[:, :128], k) + qpe @ kpe.t())
    p = torch.softmax(s, 1)
    absorbed = torch.einsum("hj,hjd->hd", q[:, :128], uk) * norm
    size = SCALE * (absorbed.abs() @ lat.abs().t() + qpe.abs() @ kpe.abs().t())
    moved = 2 * ((40 * 2.0 ** -23 + 2.0 ** -18) * size.amax(1, keepdim=True) + 2.0 ** -21)
    o, a = p @ lat, p @ lat.abs()
    fac = lat.abs().amax() / 7
    tol = (2.0 ** -8 * (o.abs() + a) + (moved + 2.0 ** -18) * a + n * 7 * fac * 2.0 ** -31)
    w_out = torch.einsum("nhv,hvd->nhd", w[4].view(-1, heads, 128), uv) * norm
    out = torch.einsum("nhd,hd->n", w_out, o)
    most = (o.abs() + tol).max()
    err = torch.einsum("nhd,hd->n", w_out.abs(), tol + most / 254 * (1 + 2.0 ** -20))
    return out, err + (2.0 ** -8 + 2.0 ** -20) * (out.abs() + err), p.sum(0), (p * moved).sum(0) + heads * 2.0 ** -22, raw[-1]


@pytest.mark.parametrize("heads,hidden,lens", [(16, 256, [0, 1, 150, 64, 127]), (4, 64, [33, 0]), (20, 128, [130, 5, 70])])
def test_the_step_is_the_attention_s_definition(heads, hidden, lens, monkeypatch):
    from mla import FusedMLA
    monkeypatch.setattr("oracle.mla_oracle.F32", f64)
    b, steps, eps = len(lens), 8, 1e-6
    w = layer(heads, hidden, 256, heads)
    attn = FusedMLA.from_weights(*(t.cuda() for t in w[:7]), SCALE, heads, eps)
    g = torch.Generator().manual_seed(7)
    cache = LatentKVCache4(b, 200)
    top = max(lens)
    prompt = with_sevens(whole(g, b, top, 576), g) * 2.0 ** torch.randint(-1, 2, (b, top, 1), generator=g)
    ds_kernels.mla_cache4_append(prompt[..., :512].to(bf16).cuda(), prompt[..., 512:].to(bf16).cuda(), cache, attn.cos,
                                 attn.sin, eps, new_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    past = [prompt[i, :n] for i, n in enumerate(lens)]
    mass = [torch.zeros(200, dtype=f64) for _ in lens]
    mtol = [torch.zeros(200, dtype=f64) for _ in lens]
    for step in range(steps):
        x = torch.zeros(b, hidden, dtype=f64)
        x[torch.arange(b), torch.randint(0, hidden - 1, (b,), generator=g)] = \
            signs(g, b) * 2.0 ** torch.randint(-1, 2, (b,), generator=g)
        out = attn.decode(x.to(bf16).cuda(), cache, mass_decay=1.0).cpu().double()
        for i in range(b):
            want, tol, p, ptol, new = step64(x[i], past[i], w, heads, eps)
            ref = oracle.mla_decode_step(x[i:i + 1], past[i][None, :, :512], past[i][None, :, 512:], *w[:7], SCALE, heads,
                                         eps)[0]
            assert (ref - want).abs().max() <= 1e-9 * want.abs().max()      # two statements of one definition
            err = (out[i] - ref).abs()
            assert (err <= tol).all(), (step, i, (err / tol).max())
            # the tolerance tells a mistake from a rounding
            assert tol.norm() <= 0.1 * want.norm()
            past[i] = torch.cat([past[i], new[None]])
            n = past[i].shape[0]
            mass[i][:n] += p
            mtol[i][:n] += ptol
            assert ((cache.mass[i].cpu().double()[:200] - mass[i]).abs() <= mtol[i]).all()
    lat, _ = cache.get(200)
    for i in range(b):
        n = past[i].shape[0]
        assert n == cache.lens[i].item() == cache.next_pos[i].item()
        assert torch.equal(lat[i, :n].cpu().double(), past[i][:, :512])     # nothing was lost on the way
        assert (lat[i, n:] == 0).all()
