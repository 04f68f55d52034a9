"""Cases of the quantised decode operators: the 8-bit integer linear, the 4-bit latent cache (filling and reading
it, attention over it) and eviction from it by accumulated attention weight.

`run` computes each case in elementary torch operations (`own` false) or through the package's public calls
(`own` true).  Sizes are those of the decode and prefill paths (hidden 2048, 16 heads, 512-wide latent, 64-wide
k_pe: projections 2048 -> 9792, 8192 -> 2048, 2048 -> 3648) and generic ones around them.
"""
import math
import sys

import torch

own = False

LATENT, ROPE, GROUPS, GROUP = 512, 64, 5, 128
SCALE = 192 ** -0.5
EPS = 1e-6
MOST_MACS = 16384 * 2048 * 3648
MOST_TOKENS = 32 * 16384


def listed():
    return [
        # one token through the absorbed query projection of a decode step
        {"name": "linear-one-token", "op": "linear", "m": 1, "k": 2048, "n": 9792},
        # 64 sequences through the absorbed output projection
        {"name": "linear-decode", "op": "linear", "m": 64, "k": 8192, "n": 2048},
        # sizes that fill no tile: a ragged batch of prompts through an odd-sized layer
        {"name": "linear-odd", "op": "linear", "m": 333, "k": 1424, "n": 2840},
        # a 4 x 4096-token prefill through the fused q | kv_a projection
        {"name": "linear-prefill", "op": "linear", "m": 16384, "k": 2048, "n": 3648},
        # a short conversation with one user
        {"name": "attend-one", "op": "attend", "b": 1, "h": 16, "len": 711, "ragged": False, "mass": False},
        # a ragged batch, empty sequences among them, with the weights accumulated
        {"name": "attend-ragged", "op": "attend", "b": 17, "h": 24, "len": 4001, "ragged": True, "mass": True},
        # the decode benchmark's batch: 64 sequences of 2048 positions
        {"name": "attend-batch", "op": "attend", "b": 64, "h": 16, "len": 2048, "ragged": False, "mass": False},
        # long documents, with the weights accumulated for a later eviction
        {"name": "attend-long", "op": "attend", "b": 32, "h": 16, "len": 16384, "ragged": False, "mass": True},
        # one new token for each of 64 sequences
        {"name": "fill-step", "op": "fill", "b": 64, "n": 1, "ragged": False},
        # prompts of different lengths, padded to the longest
        {"name": "fill-prompt", "op": "fill", "b": 4, "n": 4096, "ragged": True},
        # two chats trimmed to a small window
        {"name": "evict-short", "op": "evict", "b": 2, "len": 333, "budget": 128, "recent": 32, "ragged": False},
        # long prompts compressed into a small cache
        {"name": "evict-long", "op": "evict", "b": 32, "len": 8192, "budget": 1024, "recent": 64, "ragged": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(("linear", "attend", "fill", "evict"))
    if op == "linear":
        while True:
            m, k, n = _log(rng, 1, 16384), 16 * _log(rng, 1, 640), 8 * _log(rng, 1, 1400)
            if m * k * n <= MOST_MACS:
                return {"op": op, "m": m, "k": k, "n": n}
    if op == "attend":
        while True:
            b, h, n = _log(rng, 1, 64), _log(rng, 1, 64), _log(rng, 1, 32768)
            if b * n * -(-h // 16) <= MOST_TOKENS:
                return {"op": op, "b": b, "h": h, "len": n, "ragged": rng.random() < 0.6, "mass": rng.random() < 0.5}
    if op == "fill":
        while True:
            b, n = _log(rng, 1, 64), _log(rng, 1, 4096)
            if b * n <= 16384:
                return {"op": op, "b": b, "n": n, "ragged": rng.random() < 0.6}
    while True:
        b, n = _log(rng, 1, 64), _log(rng, 1, 32768)
        if b * n <= 32 * 8192:
            budget = _log(rng, 1, n)
            return {"op": op, "b": b, "len": n, "budget": budget, "recent": rng.randint(0, budget),
                    "ragged": rng.random() < 0.6}


def _slots(n):
    return -(-max(n, 1) // 64) * 64


def _lens(case, g, most):
    if not case["ragged"]:
        return torch.full((case["b"],), most, dtype=torch.int32, device="cuda")
    lens = torch.randint(0, most + 1, (case["b"],), generator=g, device="cuda").to(torch.int32)
    lens[-1:] = most                    # the longest fills its slots; with several, one is empty and one has one token
    if case["b"] > 2:
        lens[0], lens[1] = 0, min(1, most)
    return lens


def _rows(g, *shape):
    """bf16 values whose rows differ in size, as activations do."""
    x = torch.randn(*shape, generator=g, device="cuda")
    return (x * (0.25 + 1.5 * torch.rand(*shape[:-1], 1, generator=g, device="cuda"))).to(torch.bfloat16)


def _cache(case, g, b, n):
    """What a cache of n positions a sequence holds: codes 0..15 (value + 8), scales by group, the norm's row scale."""
    slots = _slots(n)
    s = {"codes": torch.randint(1, 16, (b, slots, LATENT + ROPE), generator=g, device="cuda", dtype=torch.uint8)}
    size = 0.25 + 1.5 * torch.rand(b, 1, slots, generator=g, device="cuda")
    s["scales"] = (size * (0.35 + 0.2 * torch.rand(b, GROUPS, slots, generator=g, device="cuda"))).to(torch.bfloat16)
    s["rstd"] = (1.0 / (size[:, 0] * 2.0)).contiguous()
    s["lens"] = _lens(case, g, n)
    return s


def _pack(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": case}
    op = case["op"]
    if op == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        s["x"] = _rows(g, m, k)
        s["wq"] = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
        s["ws"] = (0.5 + torch.rand(n, generator=g, device="cuda")) * (0.06 / 127)
    elif op == "attend":
        s.update(_cache(case, g, case["b"], case["len"]))
        s["q"] = torch.randn(case["b"], case["h"], LATENT + ROPE, generator=g, device="cuda").to(torch.bfloat16)
    elif op == "fill":
        b, n = case["b"], case["n"]
        s["latent"], s["k_pe"] = _rows(g, b, n, LATENT), _rows(g, b, n, ROPE)
        s["lens"] = _lens(case, g, n)
        freq = 10000.0 ** (-torch.arange(0, ROPE, 2, device="cuda", dtype=torch.float64) / ROPE)
        ang = torch.outer(torch.arange(n, device="cuda", dtype=torch.float64), freq)
        ang = torch.cat([ang, ang], dim=1)
        s["cos"], s["sin"] = ang.cos().to(torch.bfloat16), ang.sin().to(torch.bfloat16)
    else:
        b, n = case["b"], case["len"]
        s.update(_cache(case, g, b, n))
        # a few positions gather most of the weight; whole multiples of 2^-12, so that some are equal
        u = torch.rand(b, _slots(n), generator=g, device="cuda")
        s["mass"] = torch.floor(4096 * 8 * u ** 6) / 4096
        s["codes"] = _pack(s["codes"])
        s["pos"] = torch.arange(_slots(n), device="cuda", dtype=torch.int32).expand(b, -1).contiguous()
    if own:
        sys.path.insert(0, "deepseek-v2-lite-cuda_b200")
        import mla_cache
        if op == "attend":
            b, n = case["b"], case["len"]
            s["cache"] = mla_cache.LatentKVCache4(b, n)
            s["cache"].load_state_dict({"codes": _pack(s["codes"]), "scales": s["scales"], "rstd": s["rstd"],
                                        "lens": s["lens"]})
        elif op == "fill":
            s["cache"] = mla_cache.LatentKVCache4(case["b"], case["n"])
        elif op == "evict":
            s["cache"] = mla_cache.LatentKVCache4(case["b"], case["len"])
            s["cache"].load_state_dict({k: s[k] for k in ("codes", "scales", "rstd", "lens", "mass", "pos")})
            s["out"] = mla_cache.LatentKVCache4(case["b"], case["budget"])
    return s


# ---- the plain forms ------------------------------------------------------------------------------------------
def _linear(x, wq, ws):
    """Rows of x to 8-bit integers by their largest value, an exact product, one scaling.  The division and the sum
    are in 64 bits: a value next to a border has to go to its own side, and a long sum passes 2^24."""
    x = x.double()
    a = x.abs().amax(1, keepdim=True)
    q = torch.where(a > 0, torch.round(127 * x / a), 0.0)
    acc = (q @ wq.double().t()).float()
    return (acc * ((a.float() / 127) * ws)).to(torch.bfloat16)


def _by_dim(scales):
    """[b, 5, slots] scales -> [b, slots, 576], one for each dimension."""
    s = scales.float().transpose(1, 2)
    return torch.cat([s[..., :4].repeat_interleave(GROUP, dim=2), s[..., 4:].expand(-1, -1, ROPE)], dim=2)


def _attend(codes, scales, rstd, lens, q, mass):
    k = (codes.float() - 8) * _by_dim(scales)
    k[..., :LATENT] *= rstd[..., None]
    seen = torch.arange(k.shape[1], device=k.device) < lens[:, None]
    k = torch.where(seen[..., None], k, 0.0)
    s = (q.float() @ k.transpose(1, 2)) * SCALE
    s = torch.where(seen[:, None], s, -math.inf)
    e = torch.where(seen[:, None], torch.exp(s - s.amax(2, keepdim=True)), 0.0)
    p = e / e.sum(2, keepdim=True).clamp_min(1e-30)
    o = (p @ k[..., :LATENT]).flatten(1).to(torch.bfloat16)
    return (o, p.sum(1)) if mass else o


def _fill(latent, k_pe, lens, cos, sin):
    """Positions 0 .. of each sequence quantised, and read back as the values that the codes stand for."""
    b, n, _ = latent.shape
    seen = torch.arange(n, device=lens.device) < lens[:, None]
    lat, kp = latent.float(), k_pe.float()
    rstd = torch.rsqrt((lat * lat).mean(2) + EPS)
    x, y = kp[..., 0::2], kp[..., 1::2]
    c, s = cos.float(), sin.float()
    half = ROPE // 2
    rot = torch.cat([x * c[:, :half] - y * s[:, :half], y * c[:, half:] + x * s[:, half:]], dim=2).to(torch.bfloat16)

    def back(v, group):
        v = v.double().unflatten(2, (-1, group))  # 64 bits: a value next to a border goes to its own side
        sigma = (v.abs().amax(3, keepdim=True).float() / 7).to(torch.bfloat16).double()
        codes = torch.where(sigma > 0, torch.round(v / sigma).clamp(-7, 7), 0.0)
        return torch.where(seen[..., None], (codes * sigma).flatten(2).to(torch.bfloat16), 0.0)

    full = torch.zeros(b, _slots(n), device=lens.device)
    full[:, :n] = torch.where(seen, rstd, 0.0)
    return back(lat, GROUP), back(rot, ROPE), full, lens.clone()


def _evict(st, budget, recent):
    slots, dev = st["mass"].shape[1], st["mass"].device
    at = torch.arange(slots, device=dev).expand(st["mass"].shape[0], -1)
    lens = st["lens"].long()[:, None]
    valid = at < lens
    newest = valid & (st["pos"] >= lens - recent)
    # by weight, the lowest slot first among equals; then what is protected before all else
    order = torch.argsort(torch.where(valid, st["mass"], -1.0), dim=1, descending=True, stable=True)
    rank = torch.where(valid.gather(1, order), torch.where(newest.gather(1, order), 0, 1), 2)
    order = order.gather(1, torch.argsort(rank, dim=1, stable=True))
    kept = torch.zeros_like(valid).scatter_(1, order[:, :budget], True) & valid
    # slot j of the result: its own row if it stays, else the next survivor from behind the budget
    hole = (at < budget) & ~kept & valid
    late = (at >= budget) & kept
    into = torch.argsort(torch.where(late, at, slots), dim=1, stable=True)
    nth = (hole.cumsum(1) - 1).clamp_min(0)
    src = torch.where(hole, into.gather(1, nth), at)[:, :min(budget, slots)]
    have = torch.arange(src.shape[1], device=dev) < lens.clamp_max(budget)
    width = _slots(budget)

    def move(v, extra):
        idx = src.reshape(src.shape + (1,) * extra).expand(src.shape + v.shape[2:])
        m = have.reshape(have.shape + (1,) * extra)
        out = torch.zeros((v.shape[0], width) + v.shape[2:], dtype=v.dtype, device=dev)
        out[:, :src.shape[1]] = torch.where(m, v.gather(1, idx), torch.zeros((), dtype=v.dtype, device=dev))
        return out

    return {"codes": move(st["codes"], 1), "scales": move(st["scales"].transpose(1, 2), 1).transpose(1, 2),
            "rstd": move(st["rstd"], 0), "mass": move(st["mass"], 0), "pos": move(st["pos"], 0),
            "lens": st["lens"].clamp_max(budget)}


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        import ds_kernels
        if op == "linear":
            return ds_kernels.int8_linear(state["x"], state["wq"], state["ws"])
        cache = state["cache"]
        if op == "attend":
            if not case["mass"]:
                return ds_kernels.mla_decode_attention4(state["q"], cache, SCALE)
            # decay 0: the weights of this step alone, so that every pass gives the same
            o = ds_kernels.mla_decode_attention4(state["q"], cache, SCALE, mass_decay=0.0)
            return o, cache.mass
        if op == "fill":
            cache.reset()
            ds_kernels.mla_cache4_append(state["latent"], state["k_pe"], cache, state["cos"], state["sin"], EPS,
                                         new_lens=state["lens"])
            lat, k_pe = ds_kernels.mla_cache4_get(cache, case["n"])
            return lat, k_pe, cache.rstd, cache.lens
        out = ds_kernels.mla_cache4_evict(cache, case["budget"], case["recent"], out=state["out"])
        return {"codes": out.codes, "scales": out.scales, "rstd": out.rstd, "mass": out.mass, "pos": out.pos,
                "lens": out.lens}
    if op == "linear":
        return _linear(state["x"], state["wq"], state["ws"])
    if op == "attend":
        return _attend(state["codes"], state["scales"], state["rstd"], state["lens"], state["q"], case["mass"])
    if op == "fill":
        return _fill(state["latent"], state["k_pe"], state["lens"], state["cos"], state["sin"])
    return _evict(state, case["budget"], case["recent"])


def work(case):
    op = case["op"]
    if op == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": 2 * m * k + n * k + 4 * n + 2 * m * n, "flops": 2 * m * n * k}
    share = 0.5 if case["ragged"] else 1.0  # ragged lengths are uniform up to the longest
    if op == "attend":
        b, h = case["b"], case["h"]
        tokens = share * b * case["len"]
        return {"bytes": tokens * (288 + 10 + 4 + (4 if case["mass"] else 0)) + b * h * 2 * (576 + 512),
                "flops": tokens * h * 2 * (576 + 512)}
    if op == "fill":
        # latent and k_pe in; codes, scales, row scale and position into the cache; the values read back
        tokens = share * case["b"] * case["n"]
        return {"bytes": tokens * (1152 + 306) + case["b"] * case["n"] * 1152, "flops": tokens * 6 * 576}
    tokens = share * case["b"] * case["len"]
    kept = case["b"] * case["budget"] * (1.0 if not case["ragged"] else 1 - 0.5 * case["budget"] / case["len"])
    return {"bytes": tokens * 8 + kept * 2 * 310, "flops": tokens}


# ---- from the definitions, in 64 bits -------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "linear":
        x, w = st["x"].to(torch.float64), st["wq"].to(torch.float64)
        top = x.abs().max(dim=1).values
        step = top / 127
        # nearest whole number of 127 x / top, the even one of two
        t = x * 127 / torch.where(top > 0, top, 1.0)[:, None]
        return torch.mm(torch.round(t), w.T) * step[:, None] * st["ws"].to(torch.float64)
    if op == "attend":
        outs = torch.zeros(case["b"], case["h"] * LATENT, dtype=torch.float64, device="cuda")
        mass = torch.zeros(case["b"], _slots(case["len"]), dtype=torch.float64, device="cuda")
        for i, n in enumerate(st["lens"].tolist()):
            if n == 0:
                continue
            sig = st["scales"][i, :, :n].double()
            val = st["codes"][i, :n].double() - 8.0
            lat = (val[:, :LATENT].reshape(n, 4, GROUP) * sig[:4].T[:, :, None]).reshape(n, LATENT)
            lat = lat * st["rstd"][i, :n, None].double()
            rope = val[:, LATENT:] * sig[4][:, None]
            q = st["q"][i].double()
            z = SCALE * (q[:, :LATENT] @ lat.T + q[:, LATENT:] @ rope.T)
            p = torch.softmax(z, dim=1)
            outs[i] = (p @ lat).reshape(-1)
            mass[i, :n] = p.sum(0)
        return (outs, mass) if case["mass"] else outs
    if op == "fill":
        b, n = case["b"], case["n"]
        lat, kp = st["latent"].double(), st["k_pe"].double()
        pairs = kp.reshape(b, n, ROPE // 2, 2)
        c, s = st["cos"].double(), st["sin"].double()
        turned = torch.empty_like(kp)
        turned[..., :32] = pairs[..., 0] * c[:, :32] - pairs[..., 1] * s[:, :32]
        turned[..., 32:] = pairs[..., 1] * c[:, 32:] + pairs[..., 0] * s[:, 32:]
        turned = turned.to(torch.bfloat16).double()
        vals = []
        for v, group in ((lat, GROUP), (turned, ROPE)):
            w = v.reshape(b, n, -1, group)
            sigma = (w.abs().max(dim=3).values / 7).to(torch.bfloat16).double()[..., None]
            codes = torch.round(w / torch.where(sigma > 0, sigma, 1.0))
            vals.append((codes.clamp(-7, 7) * sigma).reshape(b, n, -1))
        rstd = torch.zeros(b, _slots(n), dtype=torch.float64, device="cuda")
        rstd[:, :n] = 1 / torch.sqrt(lat.square().mean(dim=2) + EPS)
        for i, m in enumerate(st["lens"].tolist()):
            vals[0][i, m:], vals[1][i, m:], rstd[i, m:] = 0, 0, 0
        return vals[0], vals[1], rstd, None
    return None  # rows that move as they are
