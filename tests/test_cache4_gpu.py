"""The 4-bit latent cache: filling, reading back, attention over it and eviction from it, against
their definitions in 64 bits on the CPU.

Codes, scales, positions and what eviction keeps are exact and compared bit for bit.

Attention: with A = sum_t p |v| (per output), the probabilities times a group's factor (scale *
rstd) are rounded once to 16 bits (2^-8 of A at most) and the output once (2^-8 |o|).  In f16 that
first rounding has a floor: the products are scaled so that the group's largest factor F meets [2^6,
2^7) when it is set, and weights are taken against a maximum that the largest weight reaches, so a
weight p (of a sum of 1 or more) becomes p f 2^6 / F or more, and below 2^-14 its error is 2^-25:
2^-31 F of a value's factor, 7 of them a code at most: n 7 F 2^-31 for n slots.  A score is a sum of 576 products, exact
one by one, added up in f32 by at most 40 dependent additions of 2^-23 relative to sum |q k|; it
and the exponentials (2^-21) move a probability by twice that at most (numerator and sum).
"""
import math

import pytest
import torch

import ds_kernels
from mla_cache import LatentKVCache4

pytestmark = pytest.mark.gpu
bf16 = torch.bfloat16
SCALE = 192 ** -0.5


def tables(n):
    freq = 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    a = torch.outer(torch.arange(n, dtype=torch.float64), freq)
    a = torch.cat([a, a], 1)
    return a.cos().to(bf16), a.sin().to(bf16)


def tokens(b, n, seed):
    g = torch.Generator().manual_seed(seed)
    lat = torch.randn(b, n, 512, generator=g) * torch.exp(torch.randn(b, n, 1, generator=g))
    kpe = torch.randn(b, n, 64, generator=g) * 3
    return lat.to(bf16), kpe.to(bf16)


def quant64(v, group):
    """bf16 [..., d] -> codes (0..15), scales bf16 [..., d/group]"""
    w = v.double().unflatten(-1, (-1, group))
    a = w.abs().amax(-1)
    bad = ~torch.isfinite(a)
    s = torch.where(bad, torch.full_like(a, float("nan")), a / 7).to(bf16)
    sd = s.double()[..., None]
    q = torch.where(sd > 0, torch.round(w / torch.where(sd > 0, sd, torch.ones_like(sd))).clamp(-7, 7),
                    torch.zeros_like(w))
    return (q + 8).to(torch.uint8).flatten(-2), s


def rotate(kpe, pos, cos, sin):
    x, y = kpe.double()[..., 0::2], kpe.double()[..., 1::2]
    c, s = cos.double()[pos], sin.double()[pos]
    return torch.cat([x * c[..., :32] - y * s[..., :32], y * c[..., 32:] + x * s[..., 32:]], -1).to(bf16)


def pack(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def unpack(packed):
    return torch.stack([packed & 15, packed >> 4], -1).flatten(-2)


def random_cache(b, max_seq, lens, seed, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    cache = LatentKVCache4(b, max_seq, device)
    n = cache.slots
    st = {"codes": torch.randint(0, 256, (b, n, 288), generator=g, dtype=torch.uint8),
          "scales": (0.1 + 0.3 * torch.rand(b, 5, n, generator=g)).to(bf16),
          "rstd": 0.3 + torch.rand(b, n, generator=g), "lens": torch.tensor(lens, dtype=torch.int32)}
    cache.load_state_dict({k: v.to(device) for k, v in st.items()})
    return cache, st


def values64(st, b, n):
    sig = st["scales"][b, :, :n].double()
    c = unpack(st["codes"][b, :n]).double() - 8
    lat = c[:, :512].unflatten(1, (4, 128)) * sig[:4].t()[:, :, None]
    return lat.flatten(1) * st["rstd"][b, :n, None].double(), c[:, 512:] * sig[4][:, None]


def attend64(st, q, lens, scale=SCALE):
    """out, its tolerance, mass, its tolerance"""
    B, H, _ = q.shape
    out, tol = torch.zeros(B, H * 512, dtype=torch.float64), torch.zeros(B, H * 512, dtype=torch.float64)
    mass = torch.zeros(B, st["rstd"].shape[1], dtype=torch.float64)
    mtol = torch.zeros_like(mass)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        lat, rope = values64(st, b, n)
        k = torch.cat([lat, rope], 1)
        qd = q[b].double()
        p = torch.softmax(scale * qd @ k.t(), 1)
        size = scale * qd.abs() @ k.abs().t()
        moved = 2 * (40 * 2.0 ** -23 * size.amax(1, keepdim=True) + 2.0 ** -21)
        o, a = p @ lat, p @ lat.abs()
        fac = (st["scales"][b, :4, :n].double() * st["rstd"][b, :n].double()).amax(1).repeat_interleave(128)
        out[b] = o.flatten()
        tol[b] = (2.0 ** -8 * (o.abs() + a) + moved * a + n * 7 * fac * 2.0 ** -31).flatten()
        mass[b, :n], mtol[b, :n] = p.sum(0), (p * moved).sum(0) + 2.0 ** -23 * p.sum(0) * H
    return out, tol, mass, mtol


def check(got, want, tol):
    err = (got.cpu().double() - want).abs()
    assert (err <= tol + 1e-30).all(), (err / (tol + 1e-30)).max()


# ---- filling and reading back -----------------------------------------------------------------
@pytest.mark.parametrize("b,sizes", [(1, [1]), (3, [1, 1, 1]), (2, [7, 1, 8, 9]), (5, [64, 3]), (1, [65, 130])])
def test_append_is_exact(b, sizes):
    cos, sin = tables(256)
    cache = LatentKVCache4(b, 200)
    at = 0
    for i, n in enumerate(sizes):
        lat, kpe = tokens(b, n, 10 * i + b)
        cache.mass.fill_(3.0)
        ds_kernels.mla_cache4_append(lat.cuda(), kpe.cuda(), cache, cos.cuda(), sin.cuda(), 1e-6)
        pos = torch.arange(at, at + n)
        lc, ls = quant64(lat, 128)
        kc, ks = quant64(rotate(kpe, pos, cos, sin), 64)
        sl = slice(at, at + n)
        assert torch.equal(cache.codes[:, sl].cpu(), pack(torch.cat([lc, kc], -1)))
        assert torch.equal(cache.scales[:, :, sl].cpu(), torch.cat([ls, ks], -1).transpose(1, 2))
        assert torch.equal(cache.pos[:, sl].cpu(), pos.int().expand(b, -1))
        assert (cache.mass[:, sl] == 0).all()
        want = (lat.double().square().mean(-1) + 1e-6).rsqrt()
        assert ((cache.rstd[:, sl].cpu().double() - want).abs() <= want * 2.0 ** -19).all()
        got_l, got_k = cache.get()
        vl = ((lc.double() - 8).unflatten(-1, (4, 128)) * ls.double()[..., None]).flatten(-2).to(bf16)
        vk = ((kc.double() - 8) * ks.double()).to(bf16)
        assert torch.equal(got_l[:, sl].cpu(), vl) and torch.equal(got_k[:, sl].cpu(), vk)
        at += n
        assert cache.lens.tolist() == [at] * b and cache.next_pos.tolist() == [at] * b
        assert cache.current_len == at


@pytest.mark.parametrize("n", [5, 40])
def test_ragged_append_touches_nothing_else(n):
    b = 4
    lens = [0, 1, n - 2, n]
    cos, sin = tables(64)
    lat, kpe = tokens(b, n, 2)
    cache = LatentKVCache4(b, 64)
    for t in (cache.codes, cache.scales, cache.rstd, cache.pos, cache.mass):
        t.fill_(99)
    new = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ds_kernels.mla_cache4_append(lat.cuda(), kpe.cuda(), cache, cos.cuda(), sin.cuda(), new_lens=new)
    assert cache.lens.tolist() == lens
    lc, ls = quant64(lat, 128)
    for i, m in enumerate(lens):
        assert torch.equal(unpack(cache.codes[i, :m].cpu())[:, :512], lc[i, :m])
        for t in (cache.codes[i, m:], cache.scales[i, :, m:], cache.rstd[i, m:], cache.pos[i, m:], cache.mass[i, m:]):
            assert (t == 99).all()
    got, _ = cache.get(n)
    for i, m in enumerate(lens):
        assert (got[i, m:] == 0).all()


def test_append_of_many_tokens():
    """Enough for the kernel that takes four tokens a warp; ragged, behind what is there, more tokens than
    one sequence has slots for in its padding."""
    b, n, had = 3, 3001, 70
    cos, sin = (t for t in tables(4000))
    cache = LatentKVCache4(b, n + had)
    lat0, kpe0 = tokens(b, had, 70)
    ds_kernels.mla_cache4_append(lat0.cuda(), kpe0.cuda(), cache, cos.cuda(), sin.cuda())
    for f in ("codes", "rstd", "mass"):
        getattr(cache, f)[:, had:].fill_(77)
    lat, kpe = tokens(b, n, 71)
    lens = [n, 0, 1777]
    ds_kernels.mla_cache4_append(lat.cuda(), kpe.cuda(), cache, cos.cuda(), sin.cuda(),
                                 new_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    assert cache.lens.tolist() == [had + m for m in lens] == cache.next_pos.tolist()
    assert cache.state[2].tolist() == [0] * b
    at = torch.arange(had, had + n)
    want = torch.cat([quant64(lat, 128)[0], quant64(rotate(kpe, at.expand(b, -1), cos, sin), 64)[0]], -1)
    for i, m in enumerate(lens):
        assert torch.equal(unpack(cache.codes[i, had:had + m].cpu()), want[i, :m])
        assert torch.equal(cache.pos[i, had:had + m].cpu().long(), at[:m])
        assert (cache.codes[i, had + m:] == 77).all() and (cache.rstd[i, had + m:] == 77).all()
        assert (cache.mass[i, had + m:] == 77).all() and (cache.mass[i, :had + m] == 0).all()


def test_append_takes_strided_rows_and_odd_views():
    cos, sin = tables(64)
    proj = torch.randn(3, 9792 + 8, dtype=torch.float32).to(bf16).cuda()
    lat, kpe = proj[:, None, 9216:9728], proj[:, None, 9728:9792]
    odd = proj[:, 1:577].contiguous().view(3, 1, 576)[:, :, :]
    for l, k in ((lat, kpe), (odd[..., :512], odd[..., 512:]), (proj[:, None, 3:515], proj[:, None, 520:584])):
        cache = LatentKVCache4(3, 8)
        ds_kernels.mla_cache4_append(l, k, cache, cos.cuda(), sin.cuda())
        assert torch.equal(unpack(cache.codes[:, :1].cpu())[..., :512], quant64(l.cpu(), 128)[0])
        kc = quant64(rotate(k.cpu(), torch.zeros(1, dtype=torch.long), cos, sin), 64)[0]
        assert torch.equal(unpack(cache.codes[:, :1].cpu())[..., 512:], kc)
    wide = tokens(2, 12, 3)
    cache = LatentKVCache4(2, 8)
    ds_kernels.mla_cache4_append(wide[0].cuda()[:, 4:10], wide[1].cuda()[:, 4:10], cache, cos.cuda(), sin.cuda())
    assert torch.equal(unpack(cache.codes[:, :6].cpu())[..., :512], quant64(wide[0][:, 4:10], 128)[0])


@pytest.mark.parametrize("size", [0.0, 2.0 ** -133, 2.0 ** -130, 1e-36, 1e-30, 1e30, 3.3e38])
def test_append_at_the_ends_of_the_range(size):
    cos, sin = tables(8)
    g = torch.Generator().manual_seed(4)
    lat = ((torch.rand(1, 4, 512, generator=g, dtype=torch.float64) * 2 - 1) * size).to(bf16)
    kpe = ((torch.rand(1, 4, 64, generator=g, dtype=torch.float64) * 2 - 1) * size * 0.5).to(bf16)
    cache = LatentKVCache4(1, 4)
    ds_kernels.mla_cache4_append(lat.cuda(), kpe.cuda(), cache, cos.cuda(), sin.cuda())
    lc, ls = quant64(lat, 128)
    assert torch.equal(cache.scales[0, :4, :4].cpu().t(), ls[0])
    assert torch.equal(unpack(cache.codes[0, :4].cpu())[:, :512], lc[0])


def test_every_pair_of_mantissas_goes_to_its_side():
    cos, sin = tables(1)
    m = 1 + torch.arange(128) / 128.0
    lat = torch.zeros(128, 1, 512)
    for e in range(4):
        v = m[None] * 2.0 ** -e
        lat[:, 0, 128 * e:128 * e + 128] = torch.where(v <= m[:, None], v, torch.zeros(()))
        lat[:, 0, 128 * e] = m
    lat = lat.to(bf16)
    cache = LatentKVCache4(128, 1)
    ds_kernels.mla_cache4_append(lat.cuda(), torch.zeros(128, 1, 64, dtype=bf16).cuda(), cache, cos.cuda(), sin.cuda())
    lc, ls = quant64(lat, 128)
    assert torch.equal(cache.scales[:, :4, 0].cpu(), ls[:, 0])
    assert torch.equal(unpack(cache.codes[:, :1].cpu())[..., :512], lc)


def test_a_token_that_is_not_finite_spoils_its_own_sequence_alone():
    cos, sin = tables(8)
    lat, kpe = tokens(2, 3, 5)
    lat[0, 1, 130] = float("inf")
    cache = LatentKVCache4(2, 4)
    ds_kernels.mla_cache4_append(lat.cuda(), kpe.cuda(), cache, cos.cuda(), sin.cuda())
    assert torch.isnan(cache.scales[0, 1, 1]) and not torch.isnan(cache.scales[1]).any()
    q = torch.randn(2, 16, 576).to(bf16).cuda()
    out = ds_kernels.mla_decode_attention4(q, cache, SCALE)
    assert torch.isnan(out[0]).any() and torch.isfinite(out[1]).all()


# ---- attention --------------------------------------------------------------------------------
@pytest.mark.parametrize("heads", [1, 3, 8, 16, 17, 24, 40, 128])
@pytest.mark.parametrize("lens", [[0], [1], [5, 0, 64], [63, 65, 127], [129, 200, 1, 0]])
def test_attention(heads, lens):
    b = len(lens)
    cache, st = random_cache(b, 203, lens, heads)
    q = torch.randn(b, heads, 576, generator=torch.Generator().manual_seed(heads)).to(bf16)
    out = ds_kernels.mla_decode_attention4(q.cuda(), cache, SCALE)
    ref, tol, _, _ = attend64(st, q, lens)
    check(out, ref, tol)


@pytest.mark.parametrize("b,lens", [(1, [5000]), (2, [4097, 1]), (3, [1, 2047, 3000]), (160, None)])
def test_attention_over_many_splits(b, lens):
    lens = lens or [(37 * i) % 300 for i in range(b)]
    cache, st = random_cache(b, 5000 if b < 100 else 300, lens, b)
    q = torch.randn(b, 16, 576, generator=torch.Generator().manual_seed(b)).to(bf16)
    cache.mass.fill_(2.0)
    out = ds_kernels.mla_decode_attention4(q.cuda(), cache, SCALE, mass_decay=0.5)
    ref, tol, mass, mtol = attend64(st, q, lens)
    check(out, ref, tol)
    for i, n in enumerate(lens):
        check(cache.mass[i, :n], 1.0 + mass[i, :n], mtol[i, :n] + 2.0 ** -22)
        assert (cache.mass[i, n:] == 2.0).all()          # slots behind the sequence stay
    cache.mass.fill_(float("nan"))
    again = ds_kernels.mla_decode_attention4(q.cuda(), cache, SCALE, mass_decay=0.0)
    assert torch.equal(again, out)                       # the same bits, with the weights or without
    assert torch.equal(ds_kernels.mla_decode_attention4(q.cuda(), cache, SCALE), out)
    for i, n in enumerate(lens):
        check(cache.mass[i, :n], mass[i, :n], mtol[i, :n])


@pytest.mark.parametrize("scale", [0.0, 3.0, 40.0])
def test_attention_flat_and_peaked(scale):
    lens = [300, 77]
    cache, st = random_cache(2, 320, lens, 9)
    q = torch.randn(2, 16, 576, generator=torch.Generator().manual_seed(9)).to(bf16)
    cache.mass.zero_()
    out = ds_kernels.mla_decode_attention4(q.cuda(), cache, scale, mass_decay=1.0)
    ref, tol, mass, mtol = attend64(st, q, lens, scale)
    check(out, ref, tol)
    check(cache.mass, mass, mtol)


def test_what_lies_behind_a_sequence_does_not_matter():
    lens = [70, 0, 129]
    cache, st = random_cache(3, 256, lens, 12)
    q = torch.randn(3, 16, 576).to(bf16).cuda()
    want = ds_kernels.mla_decode_attention4(q, cache, SCALE)
    for i, n in enumerate(lens):
        cache.codes[i, n:] = 255
        cache.scales[i, :, n:] = float("nan")
        cache.rstd[i, n:] = float("inf")
    assert torch.equal(ds_kernels.mla_decode_attention4(q, cache, SCALE, mass_decay=0.0), want)
    assert torch.isfinite(want).all()


def test_the_cache_may_hold_more_than_two_to_the_31_bytes():
    # 8 sequences of 2^20 slots: 2.4 GB of codes; only the last slots of the last ones are looked at
    b, n = 8, 1 << 20
    cache = LatentKVCache4(b, n)
    cos, sin = tables(4)
    cache.state[0].fill_(n - 3)
    cache._bound = n - 3
    lat, kpe = tokens(b, 3, 20)
    ds_kernels.mla_cache4_append(lat.cuda(), kpe.cuda(), cache, cos.cuda(), sin.cuda())
    lc, _ = quant64(lat, 128)
    assert torch.equal(unpack(cache.codes[:, n - 3:].cpu())[..., :512], lc)
    # all other slots are zeros with scale 0: their scores are 0, and so are their values
    cache.codes[:, :n - 3] = 0x88
    q = torch.zeros(b, 16, 576, dtype=bf16, device="cuda")
    out = ds_kernels.mla_decode_attention4(q, cache, SCALE, mass_decay=0.0)
    sig = quant64(lat, 128)[1].double()
    v = ((lc.double() - 8).unflatten(-1, (4, 128)) * sig[..., None]).flatten(-2)
    v = v * (lat.double().square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    want = v.sum(1) / n
    err = (out.cpu().double().view(b, 16, 512) - want[:, None]).abs()
    assert (err <= 2.0 ** -8 * (want.abs() + v.abs().sum(1) / n)[:, None] + want.abs()[:, None] * 2.0 ** -15).all()
    m = cache.mass[:, n - 3:].cpu().double()
    assert ((m - 16 / n).abs() <= 16 / n * 2.0 ** -10).all()


# ---- eviction ---------------------------------------------------------------------------------
def evict_ref(mass, pos, n, nxt, budget, recent):
    """slot j of the result -> source slot"""
    if n <= budget:
        return list(range(n))
    m = [-math.inf if math.isnan(x) else x for x in mass[:n].tolist()]
    nan = torch.isnan(mass[:n]).tolist()
    order = sorted(range(n), key=lambda t: (0 if pos[t] >= nxt - recent else 1, nan[t], -m[t], t))
    kept = sorted(order[:budget])
    holes = [j for j in range(budget) if j not in set(kept)]
    late = [t for t in kept if t >= budget]
    src = list(range(budget))
    for j, t in zip(holes, late):
        src[j] = t
    return src


def masses(kind, b, n, seed):
    g = torch.Generator().manual_seed(seed)
    if kind == "ties":
        return torch.randint(0, 4, (b, n), generator=g).float()
    if kind == "equal":
        return torch.zeros(b, n)
    m = torch.rand(b, n, generator=g) ** 4 * 100
    if kind == "odd":
        m[:, ::7], m[:, 1::7], m[:, 2::7], m[:, 3::7] = float("nan"), float("inf"), -float("inf"), -0.0
        m[:, 4::7] = 0.0
        m[:, 5::7] = 1e-42
    return m


FIELDS = ("codes", "scales", "rstd", "pos", "mass")


@pytest.mark.parametrize("kind", ["random", "ties", "equal", "odd"])
@pytest.mark.parametrize("lens,budget,recent", [([10], 1, 0), ([10], 1, 1), ([130, 64, 0, 1], 64, 16),
                                                ([300, 299, 5], 65, 65), ([2500, 1023, 1025], 1000, 100),
                                                ([200], 200, 3), ([777], 776, 0)])
@pytest.mark.parametrize("in_place", [True, False])
def test_evict(kind, lens, budget, recent, in_place):
    b, top = len(lens), max(lens)
    cache, _ = random_cache(b, top, lens, budget)
    cache.mass[:, :].copy_(masses(kind, b, cache.slots, recent))
    g = torch.Generator().manual_seed(7)
    for i, n in enumerate(lens):    # positions in another order, as earlier evictions leave them
        cache.pos[i, :n] = torch.randperm(n, generator=g).int().cuda()
    before = {f: getattr(cache, f).cpu().clone() for f in FIELDS}
    out = cache if in_place else LatentKVCache4(b, budget)
    if not in_place:
        for f in FIELDS:
            getattr(out, f).fill_(99)
    got = ds_kernels.mla_cache4_evict(cache, budget, recent, None if in_place else out)
    assert got is out and out.current_len == min(top, budget)
    assert out.lens.tolist() == [min(n, budget) for n in lens] and out.next_pos.tolist() == lens
    for i, n in enumerate(lens):
        src = evict_ref(before["mass"][i], before["pos"][i].tolist(), n, n, budget, recent)
        for f in FIELDS:
            have, was = getattr(out, f)[i].cpu(), before[f][i]
            if f == "scales":
                have, was = have.t(), was.t()
            assert torch.equal(have[:len(src)].nan_to_num(-5), was[src].nan_to_num(-5)), f
            if not in_place:
                assert (have[len(src):] == 99).all(), f
    if not in_place:
        for f in FIELDS:
            assert torch.equal(getattr(cache, f).cpu().nan_to_num(-5), before[f].nan_to_num(-5))
        assert cache.lens.tolist() == lens


@pytest.mark.parametrize("kind", ["random", "ties", "equal"])
@pytest.mark.parametrize("lens,budget,recent", [([9000, 20000, 3000], 3000, 64), ([32768, 2049], 2048, 0),
                                                ([8192, 8191], 8191, 8191), ([1024, 600], 300, 17)])
def test_evict_sizes_of_every_kernel(kind, lens, budget, recent):
    b = len(lens)
    cache, _ = random_cache(b, max(lens), lens, budget)
    cache.mass.copy_(masses(kind, b, cache.slots, budget))
    mass, pos, codes = cache.mass.cpu().clone(), cache.pos.cpu().clone(), cache.codes.cpu().clone()
    ds_kernels.mla_cache4_evict(cache, budget, recent)
    for i, n in enumerate(lens):
        src = evict_ref(mass[i], pos[i].tolist(), n, n, budget, recent)
        assert cache.pos[i, :len(src)].cpu().tolist() == pos[i][src].tolist()
        assert torch.equal(cache.codes[i, :len(src)].cpu(), codes[i][src])


def test_evict_long():
    cache, _ = random_cache(2, 40000, [40000, 39999], 3)
    cache.mass.copy_(masses("random", 2, cache.slots, 1))
    mass, pos = cache.mass.cpu().clone(), cache.pos.cpu().clone()
    out = ds_kernels.mla_cache4_evict(cache, 4096, 128, LatentKVCache4(2, 4096))
    for i, n in enumerate((40000, 39999)):
        src = evict_ref(mass[i], pos[i].tolist(), n, n, 4096, 128)
        assert out.pos[i].cpu().tolist() == pos[i][src].tolist()


def evict_ref_long(mass, pos, n, nxt, budget, recent):
    """evict_ref by arrays"""
    if n <= budget:
        return torch.arange(n)
    m = mass[:n].double()
    nan = torch.isnan(m)
    m = torch.where(nan, -math.inf, m)
    order = torch.argsort(m, descending=True, stable=True)          # (-0 and 0 are equal)
    order = order[torch.argsort(nan[order].int(), stable=True)]
    order = order[torch.argsort((pos[:n] < nxt - recent)[order].int(), stable=True)]
    kept = torch.zeros(n, dtype=torch.bool)
    kept[order[:budget]] = True
    src = torch.arange(budget)
    src[~kept[:budget]] = budget + kept[budget:].nonzero().flatten()
    return src


@pytest.mark.parametrize("kind", ["random", "ties", "equal", "odd"])
@pytest.mark.parametrize("lens,budget,recent", [([16000, 5, 8193], 1000, 10), ([65536, 40000, 0], 20000, 300),
                                                ([100000, 65537, 1], 30000, 0), ([262208], 5000, 5000)])
@pytest.mark.parametrize("in_place", [True, False])
def test_evict_by_clusters_and_beyond(kind, lens, budget, recent, in_place):
    b = len(lens)
    cache, _ = random_cache(b, max(lens), lens, budget)
    cache.mass.copy_(masses(kind, b, cache.slots, budget))
    g = torch.Generator().manual_seed(9)
    for i, n in enumerate(lens):
        cache.pos[i, :n] = torch.randperm(n, generator=g).int().cuda()
    mass, pos = cache.mass.cpu().clone(), cache.pos.cpu().clone()
    rows = {i: cache.codes[i].cpu() for i in range(b)}
    out = ds_kernels.mla_cache4_evict(cache, budget, recent, None if in_place else LatentKVCache4(b, budget))
    assert out.lens.tolist() == [min(n, budget) for n in lens] and out.next_pos.tolist() == lens
    for i, n in enumerate(lens):
        src = evict_ref_long(mass[i], pos[i], n, n, budget, recent)
        assert torch.equal(out.pos[i, :len(src)].cpu(), pos[i][src])
        assert torch.equal(out.codes[i, :len(src)].cpu(), rows[i][src])


def test_attention_of_few_long_sequences_among_many():
    """More partials of a sequence than the joining kernels take by a warp a head, in few and in many
    rows."""
    for lens in ([20000], [9000, 0, 300], [30000] + [5] * 70):
        b = len(lens)
        cache, st = random_cache(b, max(lens), lens, b)
        q = torch.randn(b, 16, 576, generator=torch.Generator().manual_seed(b)).to(bf16)
        few = [i for i in range(b) if lens[i] > 0][:3] + [b - 1]
        o = ds_kernels.mla_decode_attention4(q.cuda(), cache, SCALE, mass_decay=0.0)
        part = {k: v[few] for k, v in st.items()}
        want, tol, mass, mtol = attend64(part, q[few], [lens[i] for i in few])
        check(o.view(b, -1)[few], want, tol)
        check(cache.mass[few], mass, mtol)


# ---- together ---------------------------------------------------------------------------------
def test_a_run_of_steps_with_evictions():
    """Append, attend with accumulation and evict, step after step, against the same in 64 bits on
    what the cache then holds."""
    b, heads, budget, recent = 3, 16, 48, 8
    cos, sin = tables(256)
    cache = LatentKVCache4(b, 64)
    lat, kpe = tokens(b, 40, 30)
    new = torch.tensor([40, 17, 1], dtype=torch.int32, device="cuda")
    ds_kernels.mla_cache4_append(lat.cuda(), kpe.cuda(), cache, cos.cuda(), sin.cuda(), new_lens=new)
    seen = new.tolist()
    g = torch.Generator().manual_seed(31)
    for step in range(40):
        lat, kpe = tokens(b, 1, 100 + step)
        if cache.remaining_capacity < 1:
            held = {f: getattr(cache, f).cpu().clone() for f in FIELDS}
            lens = cache.lens.tolist()
            cache.evict(budget, recent)
            for i, n in enumerate(lens):
                src = evict_ref(held["mass"][i], held["pos"][i].tolist(), n, seen[i], budget, recent)
                assert cache.pos[i, :len(src)].cpu().tolist() == held["pos"][i][src].tolist()
        ds_kernels.mla_cache4_append(lat.cuda(), kpe.cuda(), cache, cos.cuda(), sin.cuda())
        seen = [n + 1 for n in seen]
        assert cache.next_pos.tolist() == seen
        st = {k: v.cpu() for k, v in cache.state_dict().items()}
        q = torch.randn(b, heads, 576, generator=g).to(bf16)
        was = cache.mass.cpu().double()
        out = ds_kernels.mla_decode_attention4(q.cuda(), cache, SCALE, mass_decay=1.0)
        lens = st["lens"].tolist()
        ref, tol, mass, mtol = attend64(st, q, lens)
        check(out, ref, tol)
        check(cache.mass, was + mass, mtol + 2.0 ** -22 * (was + 1))
        for i, n in enumerate(lens):   # the newest position is there, at its rotary position
            assert seen[i] - 1 in st["pos"][i, :n].tolist()
    assert ds_kernels.device_status() == ds_kernels.DS_OK


def test_captured_steps_replay_past_the_length_they_were_recorded_at():
    b, heads = 2, 16
    cos, sin = (t.cuda() for t in tables(512))
    lat, kpe = tokens(b, 30, 40)
    graphed, eager = LatentKVCache4(b, 300), LatentKVCache4(b, 300)
    for c in (graphed, eager):
        ds_kernels.mla_cache4_append(lat.cuda(), kpe.cuda(), c, cos, sin)
    sl, sk = (t.cuda() for t in tokens(b, 1, 41))
    sq = torch.randn(b, heads, 576).to(bf16).cuda()

    def step(cache, l, k, q):
        ds_kernels.mla_cache4_append(l, k, cache, cos, sin)
        return ds_kernels.mla_decode_attention4(q, cache, SCALE, mass_decay=0.75)

    ds_kernels.mla_decode_attention4(sq, eager, SCALE)          # warm up
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(graphed, sl, sk, sq)
    assert graphed.current_len == 31 and graphed.lens.tolist() == [30, 30]
    graphed.note_replay(-1)                                     # recording appended nothing
    for i in range(150):
        l, k = tokens(b, 1, 50 + i)
        sl.copy_(l)
        sk.copy_(k)
        graph.replay()
        graphed.note_replay()
        want = step(eager, l.cuda(), k.cuda(), sq)
        if i % 30 == 0 or i == 149:
            assert (out.float() - want.float()).norm() <= 2.0 ** -7 * want.float().norm()
            assert torch.allclose(graphed.mass, eager.mass, rtol=1e-4, atol=1e-6)
    assert graphed.lens.tolist() == [180, 180] and graphed.current_len == 180
    assert torch.equal(graphed.codes, eager.codes) and torch.equal(graphed.pos, eager.pos)


def test_calls_on_another_stream_and_two_at_once():
    caches = [random_cache(4, 3000, [3000, 10, 0, 1500], s) for s in (1, 2)]
    qs = [torch.randn(4, 16, 576, generator=torch.Generator().manual_seed(s)).to(bf16).cuda() for s in (1, 2)]
    want = [ds_kernels.mla_decode_attention4(q, c, SCALE, mass_decay=0.0) for q, (c, _) in zip(qs, caches)]
    mass = [c.mass.clone() for c, _ in caches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        outs = []
        for s, q, (c, _) in zip(streams, qs, caches):
            with torch.cuda.stream(s):
                outs.append(ds_kernels.mla_decode_attention4(q, c, SCALE, mass_decay=0.0))
        torch.cuda.synchronize()
        for o, w, m, (c, _) in zip(outs, want, mass, caches):
            assert torch.equal(o, w) and torch.equal(c.mass, m)


def test_state_dict_round_trip_into_a_larger_cache():
    cache, _ = random_cache(2, 100, [100, 31], 50)
    cache.evict(40, 4)
    big = LatentKVCache4(2, 500)
    big.load_state_dict(cache.state_dict())
    assert big.lens.tolist() == cache.lens.tolist() and big.next_pos.tolist() == [100, 31]
    assert big.current_len == 40 and big._seen == 100
    q = torch.randn(2, 16, 576).to(bf16).cuda()
    a, b = (ds_kernels.mla_decode_attention4(q, c, SCALE) for c in (cache, big))
    assert (a.float() - b.float()).norm() <= 2.0 ** -7 * a.float().norm()


def test_a_captured_eviction_replays():
    b = 2
    cos, sin = (t.cuda() for t in tables(512))
    lat, kpe = (t.cuda() for t in tokens(b, 150, 60))
    graphed, eager = LatentKVCache4(b, 200), LatentKVCache4(b, 200)
    q = torch.randn(b, 16, 576).to(bf16).cuda()
    for c in (graphed, eager):
        ds_kernels.mla_cache4_append(lat, kpe, c, cos, sin)
        ds_kernels.mla_decode_attention4(q, c, SCALE, mass_decay=0.0)
    sl, sk = (t.cuda() for t in tokens(b, 1, 61))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        graphed.evict(100, 8)
        ds_kernels.mla_cache4_append(sl, sk, graphed, cos, sin)
        out = ds_kernels.mla_decode_attention4(q, graphed, SCALE, mass_decay=1.0)
    graphed.note_replay(-1)                                     # recording appended nothing
    # nothing has run: an eager call still sees all 150 positions
    assert graphed.current_len == 150
    a, w = (ds_kernels.mla_decode_attention4(q, c, SCALE) for c in (graphed, eager))
    assert torch.equal(a, w)
    for _ in range(3):
        graph.replay()
        graphed.note_replay(1, budget=100)
        eager.evict(100, 8)
        ds_kernels.mla_cache4_append(sl, sk, eager, cos, sin)
        want = ds_kernels.mla_decode_attention4(q, eager, SCALE, mass_decay=1.0)
        assert graphed.current_len == eager.current_len == 101
        assert graphed.lens.tolist() == eager.lens.tolist() == [101] * b
        # the same sums, cut into other segments
        assert (out.float() - want.float()).norm() <= 2.0 ** -7 * want.float().norm()
    assert graphed.next_pos.tolist() == [153] * b


def test_a_captured_eviction_into_another_cache_replays_over_a_grown_source():
    b, heads = 2, 16
    cos, sin = (t.cuda() for t in tables(2048))
    lat, kpe = (t.cuda() for t in tokens(b, 1000, 80))
    src, dst = LatentKVCache4(b, 1500), LatentKVCache4(b, 1000)
    q = torch.randn(b, heads, 576).to(bf16).cuda()
    ds_kernels.mla_cache4_append(lat[:, :200], kpe[:, :200], src, cos, sin)
    ds_kernels.mla_cache4_append(lat[:, :40], kpe[:, :40], dst, cos, sin)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        src.evict(800, 8, out=dst)
    # nothing has run yet: dst holds its 40 tokens, and takes more
    assert dst.current_len == 40
    ds_kernels.mla_cache4_append(lat[:, 40:60], kpe[:, 40:60], dst, cos, sin)
    assert dst.current_len == 60 and dst.lens.tolist() == [60] * b
    ds_kernels.mla_cache4_append(lat[:, 200:], kpe[:, 200:], src, cos, sin)
    ds_kernels.mla_decode_attention4(q, src, SCALE, mass_decay=0.0)
    want = src.evict(800, 8, out=LatentKVCache4(b, 1000))
    graph.replay()
    dst.note_replay(0, budget=800)
    assert dst.lens.tolist() == [800] * b and dst.current_len == 800 and dst.next_pos.tolist() == [1000] * b
    dst.mass.zero_()
    want.mass.zero_()
    got, ref = (ds_kernels.mla_decode_attention4(q, c, SCALE, mass_decay=0.0) for c in (dst, want))
    assert torch.equal(got, ref)                         # all 800 slots, with and without the graph
    assert torch.equal(dst.mass[:, :800], want.mass[:, :800])
    assert ((dst.mass[:, :800].sum(1) - heads).abs() <= heads * 2.0 ** -14).all()
    with pytest.raises(RuntimeError, match="overflow"):
        ds_kernels.mla_cache4_append(lat[:, :201], kpe[:, :201], dst, cos, sin)
    with pytest.raises(RuntimeError, match="RoPE"):
        ds_kernels.mla_cache4_append(lat[:, :5], kpe[:, :5], dst, cos[:1004], sin[:1004])


def test_eager_steps_behind_a_recorded_eviction_see_every_token():
    b, n, more = 2, 200, 150
    cos, sin = (t.cuda() for t in tables(512))
    lat, kpe = (t.cuda() for t in tokens(b, n + more, 81))
    c, eager = LatentKVCache4(b, 400), LatentKVCache4(b, 400)
    q = torch.randn(b, 16, 576).to(bf16).cuda()
    for x in (c, eager):
        ds_kernels.mla_cache4_append(lat[:, :n], kpe[:, :n], x, cos, sin)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.evict(100, 8)
    for x in (c, eager):
        ds_kernels.mla_cache4_append(lat[:, n:], kpe[:, n:], x, cos, sin)
    assert c.current_len == eager.current_len == n + more == c.lens[0].item()
    got, want = (ds_kernels.mla_decode_attention4(q, x, SCALE, mass_decay=0.0) for x in (c, eager))
    assert torch.equal(got, want) and torch.equal(c.mass, eager.mass)
    graph.replay()
    c.note_replay(0, budget=100)
    eager.evict(100, 8)
    assert c.current_len == 100 and torch.equal(c.pos[:, :100], eager.pos[:, :100])


@pytest.mark.parametrize("start", [-5, -2 ** 31, 62, 2 ** 31 - 2])
def test_positions_outside_the_tables_take_their_first_or_last_row(start):
    """next_pos is an array that the caller may write (the host's bound does not see it)."""
    b, n, rows = 2, 7, 64
    cos, sin = tables(rows)
    lat, kpe = tokens(b, n, 82)
    cache = LatentKVCache4(b, 64)
    cache.next_pos.fill_(start)
    ds_kernels.mla_cache4_append(lat.cuda(), kpe.cuda(), cache, cos.cuda(), sin.cuda())
    at = torch.arange(start, start + n)
    at = (at + 2 ** 31) % 2 ** 32 - 2 ** 31                # as int32 counts
    want = quant64(rotate(kpe, at.clamp(0, rows - 1).expand(b, -1), cos, sin), 64)[0]
    assert torch.equal(unpack(cache.codes[:, :n].cpu())[..., 512:], want)
    assert torch.equal(cache.pos[:, :n].cpu().long(), at.expand(b, -1))


@pytest.mark.parametrize("heads", [1, 5, 15, 17, 24, 40, 48, 128])
@pytest.mark.parametrize("lens", [[1, 0, 700], [129, 64, 1000, 5]])
def test_weights_of_any_number_of_heads(heads, lens):
    b = len(lens)
    cache, st = random_cache(b, 1000, lens, heads)
    q = torch.randn(b, heads, 576, generator=torch.Generator().manual_seed(heads)).to(bf16)
    ref, tol, mass, mtol = attend64(st, q, lens)
    cache.mass.fill_(3.0)
    check(ds_kernels.mla_decode_attention4(q.cuda(), cache, SCALE, mass_decay=0.25), ref, tol)
    for i, n in enumerate(lens):
        check(cache.mass[i, :n], 0.75 + mass[i, :n], mtol[i, :n] + 2.0 ** -22 * (0.75 + mass[i, :n]))
        assert (cache.mass[i, n:] == 3.0).all()


@pytest.mark.parametrize("b,heads,top", [(330, 16, 700), (50, 128, 400), (301, 1, 129)])
def test_more_rows_than_ctas(b, heads, top):
    """More non-empty (sequence, head tile) rows than CTAs run at once: a CTA takes several, whole, one
    after the other, of other lengths each."""
    lens = [(97 * i) % (top + 1) for i in range(b)]
    lens[3], lens[-1] = 0, top
    cache, st = random_cache(b, top, lens, b)
    q = torch.randn(b, heads, 576, generator=torch.Generator().manual_seed(b)).to(bf16)
    ref, tol, mass, mtol = attend64(st, q, lens)
    out = ds_kernels.mla_decode_attention4(q.cuda(), cache, SCALE)
    check(out, ref, tol)
    cache.mass.fill_(float("nan"))
    assert torch.equal(ds_kernels.mla_decode_attention4(q.cuda(), cache, SCALE, mass_decay=0.0), out)
    for i, n in enumerate(lens):
        check(cache.mass[i, :n], mass[i, :n], mtol[i, :n])
        assert torch.isnan(cache.mass[i, n:]).all()
    assert ds_kernels.device_status() == ds_kernels.DS_OK


@pytest.mark.parametrize("kind", ["random", "equal", "odd"])
@pytest.mark.parametrize("in_place", [True, False])
def test_evict_by_the_largest_clusters(kind, in_place):
    """131073 to 262144 slots: eight blocks a sequence, 32 keys a thread."""
    lens, budget, recent = [200000, 262144, 131073, 7], 30000, 77
    b = len(lens)
    cache = LatentKVCache4(b, max(lens))
    cache.lens.copy_(torch.tensor(lens, dtype=torch.int32))
    cache.next_pos.copy_(cache.lens)
    cache._bound = cache._seen = max(lens)
    g = torch.Generator().manual_seed(9)
    mass = masses(kind, b, cache.slots, budget)
    pos = torch.stack([torch.cat([torch.randperm(n, generator=g), torch.full((cache.slots - n,), -1)]) for n in lens])
    cache.mass.copy_(mass)
    cache.pos.copy_(pos)
    cache.codes[:, :, 0] = (pos % 251).to(torch.uint8).cuda()       # rows that tell where they came from
    cache.codes[:, :, 287] = (pos % 253).to(torch.uint8).cuda()
    out = ds_kernels.mla_cache4_evict(cache, budget, recent, None if in_place else LatentKVCache4(b, budget))
    assert out.lens.tolist() == [min(n, budget) for n in lens] and out.next_pos.tolist() == lens
    for i, n in enumerate(lens):
        src = evict_ref_long(mass[i], pos[i], n, n, budget, recent)
        assert torch.equal(out.pos[i, :len(src)].cpu().long(), pos[i][src])
        assert torch.equal(out.mass[i, :len(src)].cpu().nan_to_num(-5), mass[i][src].nan_to_num(-5))
        assert torch.equal(out.codes[i, :len(src), 0].cpu().long(), pos[i][src] % 251)
        assert torch.equal(out.codes[i, :len(src), 287].cpu().long(), pos[i][src] % 253)
